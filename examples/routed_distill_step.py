"""A training step of a routed layer whose head learns from a teacher's kept
logits, with the library's operators in the places where they belong:

    dispatch    spmm with the slots x tokens matrix
    experts     grouped_mm, twice
    combine     spmm with the tokens x slots matrix of the gates
    loss        distill, which also turns the logits into their gradient, in place
    backward    grouped_mm (inputs), grouped_wgrad (weights), spmm (slots,
                tokens), sddmm (gates)

    python examples/routed_distill_step.py [--steps N]

prints the loss of each step on one fixed random batch. The router's choice and
the dense head are plain torch.
"""
import argparse
import importlib
import os
import sys
from dataclasses import dataclass

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


@dataclass
class Routing:
    """The chosen experts as two CSR matrices over the same slots: `tokens`
    (tokens x slots, the gates its values) and `slots` (slots x tokens). Slots
    are in the experts' order; expert e owns slots group_ptr[e] .. group_ptr[e+1]."""
    token_ptr: torch.Tensor
    token_col: torch.Tensor
    slot_ptr: torch.Tensor
    slot_col: torch.Tensor
    slot_of: torch.Tensor    # slot of each (token, choice)
    group_ptr: torch.Tensor
    gates: torch.Tensor      # (tokens, top), differentiable


def route(scores: torch.Tensor, top: int) -> Routing:
    tokens, experts = scores.shape
    best, expert = scores.topk(top, dim=1)
    order = torch.argsort(expert.flatten(), stable=True)
    slot_of = torch.empty_like(order)
    slot_of[order] = torch.arange(order.numel(), device=order.device)
    group_ptr = torch.zeros(experts + 1, dtype=torch.int32, device=scores.device)
    group_ptr[1:] = torch.bincount(expert.flatten(), minlength=experts).cumsum(0)
    ptr = torch.arange(0, tokens * top + 1, top, dtype=torch.int32, device=scores.device)
    return Routing(ptr, slot_of.int(),
                   torch.arange(tokens * top + 1, dtype=torch.int32, device=scores.device),
                   (order // top).int(), slot_of, group_ptr, torch.softmax(best, dim=1))


def step(pf, handle, x, w_router, w_up, w_down, head, teacher, temperature=1.0, top=2):
    """Mean loss over the tokens, and the gradients of (w_router, w_up, w_down,
    head, x). x: tokens x width; w_router: experts x width (float32); w_up:
    experts x inner x width, w_down: experts x width x inner; head: vocabulary x
    width; teacher: CSR (row_ptr, col, val) over tokens x vocabulary."""
    tokens, width = x.shape
    experts, inner, _ = w_up.shape
    like = dict(dtype=x.dtype, device=x.device)
    # the router is small: torch differentiates it
    router_w = w_router.detach().requires_grad_()
    router_x = x.detach().float().requires_grad_()
    with torch.enable_grad():
        r = route(router_x @ router_w.t(), top)
    slots = tokens * top
    gates = r.gates.detach().flatten().to(x.dtype)
    gate_of_slot = torch.empty_like(gates)
    gate_of_slot[r.slot_of] = gates
    ones = torch.ones(slots, **like)

    # forward
    xs = torch.empty(slots, width, **like)
    pf.spmm(handle, slots, tokens, slots, r.slot_ptr, r.slot_col, ones, x, xs)
    up = torch.empty(slots, inner, **like)
    pf.grouped_mm(handle, r.group_ptr, xs, w_up, up)
    act = torch.relu(up)
    ys = torch.empty(slots, width, **like)
    pf.grouped_mm(handle, r.group_ptr, act, w_down, ys)
    y = x.clone()  # residual
    pf.spmm(handle, tokens, slots, slots, r.token_ptr, r.token_col, gates, ys, y, beta=1.0)
    z = y @ head.t()

    # loss, and the logits' gradient in their place
    loss = torch.empty(tokens, device=x.device)
    weight = torch.full((tokens,), 1.0 / tokens, device=x.device)
    pf.distill(handle, tokens, head.shape[0], teacher[1].numel(), *teacher, z, loss, dZ=z,
               weight=weight, temperature=temperature)

    # backward
    d_head = z.t() @ y
    dy = z @ head
    dys = torch.empty_like(ys)
    pf.spmm(handle, slots, tokens, slots, r.slot_ptr, r.slot_col, gate_of_slot, dy, dys)
    d_gates = torch.empty_like(gates)
    pf.sddmm(handle, tokens, slots, slots, r.token_ptr, r.token_col, dy, ys, d_gates)
    d_down = torch.empty(experts, width, inner, device=x.device)  # float32
    pf.grouped_wgrad(handle, r.group_ptr, dys, act, d_down)
    d_up_out = torch.empty_like(up)
    pf.grouped_mm(handle, r.group_ptr, dys, w_down, d_up_out, transpose_w=False)
    d_up_out.mul_(up > 0)
    d_up = torch.empty(experts, inner, width, device=x.device)
    pf.grouped_wgrad(handle, r.group_ptr, d_up_out, xs, d_up)
    dxs = torch.empty_like(xs)
    pf.grouped_mm(handle, r.group_ptr, d_up_out, w_up, dxs, transpose_w=False)
    dx = dy.clone()  # residual
    pf.spmm(handle, tokens, slots, slots, r.token_ptr, r.token_col, ones, dxs, dx, beta=1.0)
    r.gates.backward(d_gates.view_as(r.gates).float())
    return loss.sum(), (router_w.grad, d_up, d_down, d_head, dx + router_x.grad.to(x.dtype))


def random_problem(tokens=512, width=256, inner=512, experts=8, vocab=4000, keep=32, seed=0,
                   dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std):
        return torch.randn(*shape, generator=g, device="cuda") * std

    x = normal(tokens, width, std=1.0).to(dtype)
    weights = [normal(experts, width, std=width ** -0.5),
               normal(experts, inner, width, std=width ** -0.5),
               normal(experts, width, inner, std=inner ** -0.5),
               normal(vocab, width, std=width ** -0.5)]
    top_logits, col = normal(tokens, vocab, std=3.0).topk(keep, dim=1)
    ptr = torch.arange(0, tokens * keep + 1, keep, dtype=torch.int32, device="cuda")
    return x, weights, (ptr, col.flatten().int(), top_logits.flatten().to(dtype))


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--steps", type=int, default=10)
    a = ap.parse_args()
    pf = importlib.import_module("prefree-public_b200")
    handle = pf.Handle()
    x, masters, teacher = random_problem()
    for i in range(a.steps):
        w = [masters[0]] + [m.to(x.dtype) for m in masters[1:]]
        loss, grads = step(pf, handle, x, *w, teacher)
        for m, d in zip(masters, grads):
            m -= 5.0 * d.float()
        print(f"step {i}: loss {float(loss):.4f}")
    if handle.device_error():
        raise SystemExit("a kernel flagged an error")
    handle.close()


if __name__ == "__main__":
    main()
