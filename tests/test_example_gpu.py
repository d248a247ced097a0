"""The example's step against the same layer written with torch operations in
64 bits and differentiated by torch: the loss and every gradient."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                    "routed_distill_step.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("routed_distill_step", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def plain(x, ws, teacher, chosen, tau):
    x, router, up, down, head = (t.double().detach().requires_grad_() for t in (x, *ws))
    best = (x @ router.t()).gather(1, chosen)
    gates = torch.softmax(best, 1)
    y = x
    for e in range(up.shape[0]):
        out = torch.relu(x @ up[e].t()) @ down[e].t()
        y = y + (gates * (chosen == e)).sum(1, keepdim=True) * out
    lq = torch.log_softmax(y @ head.t() / tau, 1)
    ptr, col, val = teacher
    k = int(ptr[1])
    p = torch.softmax(val.double().view(-1, k) / tau, 1)
    loss = (p * (torch.log(p) - lq.gather(1, col.long().view(-1, k)))).sum(1).mean()
    loss.backward()
    return loss.detach(), [t.grad for t in (router, up, down, head, x)]


@pytest.mark.parametrize("tokens,width,inner,experts,vocab", [(96, 64, 128, 4, 1000),
                                                              (61, 40, 72, 5, 333)])
def test_step_against_torch(pf, example, tokens, width, inner, experts, vocab):
    """f16 values: every stored intermediate is rounded to 2^-11 of its size, and
    about a dozen of them lie between an input and a gradient, whose errors are
    independent: 5 * 2^-11 * sqrt(12) = 1 % of the gradient's norm bounds them."""
    x, ws, teacher = example.random_problem(tokens, width, inner, experts, vocab, 16, 3,
                                            torch.float16)
    ws = [ws[0]] + [w.half() for w in ws[1:]]
    h = pf.Handle()
    example_loss, grads = example.step(pf, h, x, *ws, teacher, 1.5)
    assert h.device_error() == 0
    chosen = (x.float() @ ws[0].t()).topk(2, dim=1)[1]
    loss, want = plain(x, ws, teacher, chosen, 1.5)
    assert abs(float(example_loss) - float(loss)) <= 0.01 * abs(float(loss))
    for got, ref, what in zip(grads, want, ("router", "up", "down", "head", "x")):
        off = float((got.double() - ref).norm() / ref.norm())
        assert off <= 0.01, (what, off)
    h.close()
