"""Measured cases of the framework's operators for routed models and sparse targets.

Three operators, all on a CSR matrix:

* ``distill``  the loss of a student's dense logits against a teacher's kept logits
  (CSR rows), alone (``fwd``) or with the gradient of the logits (``train``);
* ``grouped``  matrix products of ragged row groups with one weight matrix each:
  ``fwd`` (X W^T), ``dx`` (dY W) and ``dw`` (dY^T X);
* ``combine``  the wide 16-bit sparse-dense product that weighs and sums expert
  outputs (``fwd``), and its gradients (``bwd``: of the expert outputs, a product
  with the transposed CSR, and of the gates, the sampled dense-dense product).

``run`` computes each with elementary torch operations in 32 bits, or, with ``own``
set, with the calls that a user of the framework makes.
"""
import importlib
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}

_kept = {}


def _framework():
    """The package and one handle for the stream that the passes run on."""
    if "pf" not in _kept:
        _kept["pf"] = importlib.import_module("prefree-public_b200")
        _kept["handle"] = _kept["pf"].Handle()
    return _kept["pf"], _kept["handle"]


def listed():
    return [
        # scoring a handful of positions while serving or validating: latency
        dict(name="distill_fwd_few", op="distill", dir="fwd", rows=16, vocab=32000, keep=32,
             ragged=False, dtype="bf16", temperature=1.0),
        # validation over a batch with 32-bit logits
        dict(name="distill_fwd_f32", op="distill", dir="fwd", rows=2048, vocab=65536, keep=64,
             ragged=True, dtype="f32", temperature=2.0),
        # a micro-batch with an odd vocabulary: no row but the first is aligned
        dict(name="distill_train_odd", op="distill", dir="train", rows=1500, vocab=49999, keep=50,
             ragged=True, dtype="f16", temperature=1.5),
        # a full training batch over a large vocabulary
        dict(name="distill_train_large", op="distill", dir="train", rows=4096, vocab=131072,
             keep=64, ragged=False, dtype="bf16", temperature=1.0),
        # decoding a few sequences: a row or two for some experts, none for others
        dict(name="grouped_fwd_decode", op="grouped", dir="fwd", rows=24, groups=32, n=2048,
             k=1024, skew=0.0, dtype="bf16"),
        # a long prompt or training batch through the experts' first product
        dict(name="grouped_fwd_prompt", op="grouped", dir="fwd", rows=16384, groups=16, n=4096,
             k=2048, skew=0.5, dtype="bf16"),
        # backward through the same product, many small experts, strongly uneven
        dict(name="grouped_dx_ragged", op="grouped", dir="dx", rows=5003, groups=64, n=1000,
             k=2008, skew=1.0, dtype="f16"),
        # gradients of the experts' weights
        dict(name="grouped_dw_small", op="grouped", dir="dw", rows=777, groups=8, n=768, k=512,
             skew=0.5, dtype="f16"),
        dict(name="grouped_dw_batch", op="grouped", dir="dw", rows=16384, groups=16, n=2048,
             k=2048, skew=0.5, dtype="bf16"),
        # one decoding step's outputs
        dict(name="combine_fwd_decode", op="combine", dir="fwd", tokens=8, top=2, width=4096,
             dtype="bf16"),
        # a batch's expert outputs, eight to a token, some dropped
        dict(name="combine_fwd_batch", op="combine", dir="fwd", tokens=8192, top=8, width=2048,
             dtype="bf16"),
        # its gradients, with a width that is no multiple of anything
        dict(name="combine_bwd_odd", op="combine", dir="bwd", tokens=3001, top=4, width=1531,
             dtype="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["distill", "grouped", "combine"])
    if op == "distill":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        vocab = _log(rng, 1000, 131072)
        if rng.random() < 0.5:
            vocab = max(1024, vocab // 128 * 128)
        most = 4096 * 131072 * 2 // (SIZE[dtype] * vocab)
        return dict(op=op, dir=rng.choice(["fwd", "train"]), rows=_log(rng, 1, min(4096, most)),
                    vocab=vocab, keep=_log(rng, 1, 128), ragged=rng.random() < 0.5, dtype=dtype,
                    temperature=rng.choice([0.7, 1.0, 2.0, 4.0]))
    if op == "grouped":
        n, k = 8 * _log(rng, 32, 512), 8 * _log(rng, 32, 512)
        groups = _log(rng, 1, min(128, 16 * 4096 * 4096 // (n * k)))
        most = 16384 * 4096 * 2048 // (n * k)
        return dict(op=op, dir=rng.choice(["fwd", "dx", "dw"]), rows=_log(rng, 1, min(16384, most)),
                    groups=groups, n=n, k=k, skew=rng.choice([0.0, 0.5, 1.0]),
                    dtype=rng.choice(["bf16", "f16"]))
    top = rng.randint(1, 8)
    width = _log(rng, 256, 4096)
    if rng.random() < 0.7:
        width = max(256, width // 8 * 8)
    most = 65536 * 2048 // (top * width)
    return dict(op=op, dir=rng.choice(["fwd", "bwd"]), tokens=_log(rng, 1, min(8192, most)),
                top=top, width=width, dtype=rng.choice(["bf16", "f16"]))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _pointers(lengths):
    ptr = torch.zeros(lengths.numel() + 1, dtype=torch.int32, device=lengths.device)
    ptr[1:] = torch.cumsum(lengths, 0)
    return ptr


def _prepare_distill(c, g):
    m, v, dt = c["rows"], c["vocab"], DTYPES[c["dtype"]]
    keep = min(c["keep"], v)
    z = torch.empty(m, v, dtype=dt, device="cuda").normal_(0.0, 2.5, generator=g)
    # one column out of each of `keep` equal ranges, in the order of the teacher's logits
    wide = v // keep
    col = torch.randint(0, wide, (m, keep), generator=g, device="cuda")
    col += torch.arange(keep, device="cuda") * wide
    order = torch.rand(m, keep, generator=g, device="cuda").argsort(1)
    col = col.gather(1, order)
    # a student on its way to the teacher: high logits where the teacher has them
    top = torch.empty(m, keep, device="cuda").normal_(8.0, 3.0, generator=g)
    top = top.sort(1, descending=True)[0]
    near = top + torch.empty(m, keep, device="cuda").normal_(0.0, 1.5, generator=g)
    z.scatter_(1, col, near.to(dt))
    lengths = torch.full((m,), keep, device="cuda")
    if c["ragged"]:
        lengths = torch.randint(0, keep + 1, (m,), generator=g, device="cuda")
        lengths[m // 2] = keep
    stored = torch.arange(keep, device="cuda") < lengths[:, None]
    # the mean over the positions, scaled up where gradients are kept in binary16
    weight = torch.full((m,), (4096.0 if c["dtype"] == "f16" else 1.0) / m, device="cuda")
    weight[5::16] = 0.0  # positions that do not count: padding, prompts
    return dict(ptr=_pointers(lengths), col=col[stored].to(torch.int32), val=top[stored].to(dt),
                z=z, weight=weight, longest=keep,
                loss=torch.empty(m, dtype=torch.float32, device="cuda"),
                dz=torch.empty_like(z) if c["dir"] == "train" else None)


def _prepare_grouped(c, g):
    rows, groups, n, k, dt = c["rows"], c["groups"], c["n"], c["k"], DTYPES[c["dtype"]]
    share = torch.exp(c["skew"] * torch.randn(groups, generator=g, device="cuda"))
    to = torch.multinomial(share, rows, replacement=True, generator=g)
    lengths = torch.bincount(to, minlength=groups)
    s = dict(ptr=_pointers(lengths), longest=int(lengths.max()))

    def normal(*shape, std=1.0):
        return torch.empty(*shape, dtype=dt, device="cuda").normal_(0.0, std, generator=g)

    if c["dir"] == "fwd":
        s.update(x=normal(rows, k), w=normal(groups, n, k, std=k ** -0.5),
                 out=torch.empty(rows, n, dtype=dt, device="cuda"))
    elif c["dir"] == "dx":
        s.update(dy=normal(rows, n), w=normal(groups, n, k, std=k ** -0.5),
                 out=torch.empty(rows, k, dtype=dt, device="cuda"))
    else:
        s.update(dy=normal(rows, n), x=normal(rows, k),
                 out=torch.empty(groups, n, k, dtype=dt, device="cuda"))
    return s


def _prepare_combine(c, g):
    t, top, width, dt = c["tokens"], c["top"], c["width"], DTYPES[c["dtype"]]
    # a token loses some of its slots where an expert was full
    gone = torch.randperm(t * top, generator=g, device="cuda")[:t * top // 20]
    lengths = top - torch.bincount(gone // top, minlength=t)
    ptr = _pointers(lengths)
    nnz = t * top - t * top // 20
    col = torch.randperm(nnz, generator=g, device="cuda")
    val = torch.rand(nnz, generator=g, device="cuda").to(dt)
    token = torch.repeat_interleave(torch.arange(t, device="cuda"), lengths, output_size=nnz)
    # the transposed CSR, which the routing has too: one token to a slot
    to = torch.empty(nnz, dtype=torch.int32, device="cuda")
    to[col] = token.to(torch.int32)
    gate = torch.empty_like(val)
    gate[col] = val
    s = dict(ptr=ptr, col=col.to(torch.int32), val=val, nnz=nnz,
             x=torch.empty(nnz, width, dtype=dt, device="cuda").normal_(generator=g))
    if c["dir"] == "fwd":
        s["out"] = torch.empty(t, width, dtype=dt, device="cuda")
    else:
        s.update(dy=torch.empty(t, width, dtype=dt, device="cuda").normal_(generator=g),
                 slot_ptr=torch.arange(nnz + 1, dtype=torch.int32, device="cuda"), slot_col=to,
                 slot_val=gate, dx=torch.empty_like(s["x"]), dval=torch.empty_like(val))
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    make = {"distill": _prepare_distill, "grouped": _prepare_grouped, "combine": _prepare_combine}
    return dict(make[case["op"]](case, g), case=case)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _padded(ptr, longest):
    """For each row of a CSR its elements' places, and which of them exist."""
    at = ptr[:-1, None].long() + torch.arange(longest, device=ptr.device)
    there = at < ptr[1:, None]
    return torch.where(there, at, 0), there


def _plain_distill(s, c):
    tau = c["temperature"]
    z = s["z"].float() / tau
    at, there = _padded(s["ptr"], s["longest"])
    if s["val"].numel() == 0:
        p = torch.zeros(at.shape, device=z.device)
        col, t = torch.zeros_like(at), p
    else:
        col = s["col"][at].long()
        t = (s["val"].float() / tau)[at]
        high = torch.where(there, t, -math.inf).amax(1, keepdim=True)
        e = torch.where(there, torch.exp(t - torch.where(high > -math.inf, high, 0.0)), 0.0)
        total = e.sum(1, keepdim=True)
        p = e / torch.where(total > 0, total, 1.0)
    high = z.amax(1, keepdim=True)
    e = torch.exp(z - high)
    total = e.sum(1, keepdim=True)
    log_q = z.gather(1, col) - high - torch.log(total)
    term = torch.where(p > 0, p * (torch.log(torch.where(p > 0, p, 1.0)) - log_q), 0.0)
    live = (s["weight"] != 0) & (p.sum(1) > 0)
    loss = torch.where(live, s["weight"] * term.sum(1), 0.0)
    if c["dir"] == "fwd":
        return {"loss": loss}
    e = e / total
    e.scatter_add_(1, col, -p)
    e *= torch.where(live, s["weight"] / tau, 0.0)[:, None]
    return {"loss": loss, "dz": e.to(s["z"].dtype)}


def _plain_grouped(s, c):
    at, there = _padded(s["ptr"], s["longest"])

    def padded(v):  # groups x longest x width, rows past a group's end zero
        return torch.where(there[:, :, None], v[at].float(), 0.0)

    if c["dir"] == "dw":
        return torch.bmm(padded(s["dy"]).transpose(1, 2), padded(s["x"])).to(s["x"].dtype)
    if c["dir"] == "fwd":
        full = torch.bmm(padded(s["x"]), s["w"].float().transpose(1, 2))
    else:
        full = torch.bmm(padded(s["dy"]), s["w"].float())
    return full[there].to(s["w"].dtype)  # groups in order: the rows in order


def _plain_combine(s, c):
    t = s["ptr"].numel() - 1
    lengths = (s["ptr"][1:] - s["ptr"][:-1]).long()
    token = torch.repeat_interleave(torch.arange(t, device=lengths.device), lengths,
                                    output_size=s["nnz"])
    col = s["col"].long()
    if c["dir"] == "fwd":
        y = torch.zeros(t, c["width"], device=token.device)
        y.index_add_(0, token, s["val"].float()[:, None] * s["x"].float()[col])
        return y.to(s["x"].dtype)
    dy = s["dy"].float()[token]
    dx = s["slot_val"].float()[:, None] * s["dy"].float()[s["slot_col"].long()]
    dval = (dy * s["x"].float()[col]).sum(1)
    return {"dx": dx.to(s["x"].dtype), "dval": dval.to(s["val"].dtype)}


def _own_distill(s, c):
    pf, h = _framework()
    m, n = s["z"].shape
    pf.distill(h, m, n, s["col"].numel(), s["ptr"], s["col"], s["val"], s["z"], s["loss"],
               dZ=s["dz"], weight=s["weight"], temperature=c["temperature"])
    return {"loss": s["loss"]} if c["dir"] == "fwd" else {"loss": s["loss"], "dz": s["dz"]}


def _own_grouped(s, c):
    pf, h = _framework()
    if c["dir"] == "fwd":
        pf.grouped_mm(h, s["ptr"], s["x"], s["w"], s["out"], transpose_w=True)
    elif c["dir"] == "dx":
        pf.grouped_mm(h, s["ptr"], s["dy"], s["w"], s["out"], transpose_w=False)
    else:
        pf.grouped_wgrad(h, s["ptr"], s["dy"], s["x"], s["out"])
    return s["out"]


def _own_combine(s, c):
    pf, h = _framework()
    t, nnz = s["ptr"].numel() - 1, s["nnz"]
    if c["dir"] == "fwd":
        pf.spmm(h, t, nnz, nnz, s["ptr"], s["col"], s["val"], s["x"], s["out"])
        return s["out"]
    pf.spmm(h, nnz, t, nnz, s["slot_ptr"], s["slot_col"], s["slot_val"], s["dy"], s["dx"])
    pf.sddmm(h, t, nnz, nnz, s["ptr"], s["col"], s["dy"], s["x"], s["dval"])
    return {"dx": s["dx"], "dval": s["dval"]}


def run(state):
    c = state["case"]
    if own:
        return {"distill": _own_distill, "grouped": _own_grouped,
                "combine": _own_combine}[c["op"]](state, c)
    return {"distill": _plain_distill, "grouped": _plain_grouped,
            "combine": _plain_combine}[c["op"]](state, c)


# ---------------------------------------------------------------------------
# what a pass cannot do without, and its exact result
# ---------------------------------------------------------------------------
def work(case):
    c, size = case, SIZE[case["dtype"]]
    if c["op"] == "distill":
        m = c["rows"]
        live = m - len(range(5, m, 16))  # rows of weight 0 are not read
        nnz = m * min(c["keep"], c["vocab"]) * (0.5 if c["ragged"] else 1.0)
        moved = live * c["vocab"] * size + nnz * (size + 4) + m * 12
        if c["dir"] == "train":
            moved += m * c["vocab"] * size
        return {"bytes": moved, "flops": live * c["vocab"] * (4 if c["dir"] == "fwd" else 8)}
    if c["op"] == "grouped":
        rows, g, n, k = c["rows"], c["groups"], c["n"], c["k"]
        live = g if c["dir"] == "dw" else g * (1.0 - (1.0 - 1.0 / g) ** rows)
        return {"bytes": size * (rows * (n + k) + live * n * k) + 4 * (g + 1),
                "flops": 2.0 * rows * n * k}
    t, width, nnz = c["tokens"], c["width"], c["tokens"] * c["top"]
    nnz -= nnz // 20
    matrix = 4 * (t + 1) + nnz * (4 + size)
    if c["dir"] == "fwd":
        return {"bytes": size * width * (nnz + t) + matrix, "flops": 2.0 * nnz * width}
    return {"bytes": size * width * (2 * nnz + t) + 2 * matrix + nnz * size,
            "flops": 3.0 * nnz * width}


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    ptr = s["ptr"].tolist()
    if c["op"] == "distill":
        m, v = s["z"].shape
        tau = c["temperature"]
        row = torch.repeat_interleave(torch.arange(m), torch.tensor(ptr).diff()).cuda()
        col = s["col"].long()
        t = s["val"].double() / tau
        e = torch.exp(t - t.max()) if t.numel() else t
        total = torch.zeros(m, dtype=torch.float64, device="cuda").index_add_(0, row, e)
        p = e / total[row]
        loss = torch.zeros(m, dtype=torch.float64, device="cuda")
        dz = torch.zeros(m, v, dtype=torch.float64, device="cuda") if c["dir"] == "train" else None
        wt = torch.where(total > 0, s["weight"].double(), 0.0)
        for r0 in range(0, m, 512):
            r1 = min(m, r0 + 512)
            a, b = ptr[r0], ptr[r1]
            lq = torch.log_softmax(s["z"][r0:r1].double() / tau, 1)
            rr = row[a:b] - r0
            part = p[a:b] * (torch.log(p[a:b]) - lq[rr, col[a:b]])
            loss[r0:r1].index_add_(0, rr, part)
            if dz is not None:
                q = torch.exp(lq)
                q.index_put_((rr, col[a:b]), -p[a:b], accumulate=True)
                dz[r0:r1] = q * (wt[r0:r1] / tau)[:, None]
        loss = loss * wt
        return {"loss": loss} if dz is None else {"loss": loss, "dz": dz}
    if c["op"] == "grouped":
        if 2.0 * c["rows"] * c["n"] * c["k"] > 4e14:
            return None
        out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
        for i in range(c["groups"]):
            rows = slice(ptr[i], ptr[i + 1])
            if c["dir"] == "fwd":
                out[rows] = torch.einsum("rk,nk->rn", s["x"][rows].double(), s["w"][i].double())
            elif c["dir"] == "dx":
                out[rows] = torch.einsum("rn,nk->rk", s["dy"][rows].double(), s["w"][i].double())
            else:
                out[i] = torch.einsum("rn,rk->nk", s["dy"][rows].double(), s["x"][rows].double())
        return out
    t = c["tokens"]
    a = torch.sparse_csr_tensor(s["ptr"].long(), s["col"].long(), s["val"].double(),
                                size=(t, s["nnz"]))
    if c["dir"] == "fwd":
        return a @ s["x"].double()
    row = torch.repeat_interleave(torch.arange(t), torch.tensor(ptr).diff()).cuda()
    dx = torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda")
    dx[s["col"].long()] = s["val"].double()[:, None] * s["dy"].double()[row]
    dval = torch.einsum("jc,jc->j", s["dy"].double()[row], s["x"].double()[s["col"].long()])
    return {"dx": dx, "dval": dval}
