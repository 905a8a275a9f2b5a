"""The operators around the experts' products, measured one case at a time: tokens sorted by expert
and back, with their gradients, and products with 4-bit weights and group scales.

Kinds of case:
  sort    kt_moe_sort.moe_sort: the rows of x copied in expert order, with the offsets of the
          experts' segments and both permutations; with grad, the gradient of x too
  unsort  kt_moe_sort.moe_unsort: the sorted rows back in token order, weighted and summed; with
          grad, the gradients of the rows and of the weights too
  dense   kt_w4_vec.w4_vec: one 4-bit matrix against a few tokens
  routed  kt_w4_vec.moe_w4_vec: each route's rows from the 4-bit matrix of its expert
  sorted  kt_w4_vec.moe_w4_sorted: the same for rows already sorted by expert

With `own` false, `run` computes them in elementary torch operations in 32 bits; with `own` true it
calls the framework. `exact` computes them in 64 bits.

Shapes are those of the package's own workloads (synth.WORKLOADS) and generic ones. Inputs:
activations ~ N(0, 1), Zipf expert popularity, top-k of Gumbel-perturbed logits, 4-bit codes
distributed as quantised normals.
"""
from __future__ import annotations

import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

_ROOT = Path(__file__).resolve().parent.parent
_ops = None


def _framework():
    """(kt_moe_sort, kt_w4_vec) of this repository's package."""
    global _ops
    if _ops is None:
        name = "kt_prefill_lend_amd"
        if name not in sys.modules:
            root = _ROOT / "kt-prefill-lend_amd"
            spec = importlib.util.spec_from_file_location(name, root / "__init__.py",
                                                          submodule_search_locations=[str(root)])
            mod = importlib.util.module_from_spec(spec)
            sys.modules[name] = mod
            spec.loader.exec_module(mod)
        import kt_prefill_lend_amd.kt_moe_sort as S
        import kt_prefill_lend_amd.kt_w4_vec as W

        _ops = (S, W)
    return _ops


_DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one user's decode step of a small-expert model, part of whose experts are on the CPU
        dict(name="sort-1", kind="sort", tokens=1, top_k=8, experts=256, cold=0.4, cols=2048, dtype="bf16", grad=False),
        # a decode batch with ten experts a token, in fp16
        dict(name="sort-77-f16", kind="sort", tokens=77, top_k=10, experts=512, cold=0.0, cols=2048, dtype="f16",
             grad=False),
        # a training step's sequence, with the gradient of the tokens
        dict(name="sort-2047-grad", kind="sort", tokens=2047, top_k=8, experts=128, cold=0.0, cols=2048, dtype="bf16",
             grad=True),
        # a full prefill chunk on a rank that holds most of the experts
        dict(name="sort-16384", kind="sort", tokens=16384, top_k=8, experts=256, cold=0.3, cols=2048, dtype="bf16",
             grad=False),
        # a small decode batch of a large-expert model
        dict(name="unsort-5", kind="unsort", tokens=5, top_k=8, experts=256, cold=0.0, cols=7168, dtype="bf16",
             grad=False),
        # a router and adapters trained in fp32 on a ragged sequence
        dict(name="unsort-1021-f32-grad", kind="unsort", tokens=1021, top_k=4, experts=64, cold=0.0, cols=1000,
             dtype="f32", grad=True),
        # a training step's batch in bf16, with the gradients of the experts' outputs and the weights
        dict(name="unsort-4096-grad", kind="unsort", tokens=4096, top_k=8, experts=128, cold=0.2, cols=2048,
             dtype="bf16", grad=True),
        # a dense projection of one token
        dict(name="w4-1", kind="dense", tokens=1, rows=4096, cols=7168, group=128, zeros=False, dtype="bf16",
             sdtype="bf16"),
        # a dense projection of a decode batch, fp16 with zero points
        dict(name="w4-24-f16", kind="dense", tokens=24, rows=7168, cols=2048, group=64, zeros=True, dtype="f16",
             sdtype="f16"),
        # the gate and up rows of one user's decode step, groups of 32
        dict(name="moe-w4-1", kind="routed", tokens=1, top_k=8, experts=256, cold=0.0, rows=1024, cols=2048, group=32,
             zeros=False, dtype="bf16", sdtype="bf16"),
        # a decode window of a large-expert model, a third of its routes on the CPU
        dict(name="moe-w4-13", kind="routed", tokens=13, top_k=8, experts=24, cold=0.3, rows=4096, cols=7168, group=128,
             zeros=False, dtype="bf16", sdtype="bf16"),
        # the down products of a batch's sorted routes, with zero points
        dict(name="w4-sorted-64", kind="sorted", tokens=64, top_k=8, experts=128, cold=0.0, rows=2048, cols=768,
             group=128, zeros=True, dtype="bf16", sdtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["sort", "sort", "unsort", "unsort", "dense", "routed", "routed", "sorted"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind in ("sort", "unsort"):
        cols = rng.choice([512, 1000, 1021, 2048, 2048, 4096, 7168])
        top_k = rng.choice([1, 2, 4, 6, 8, 10])
        grad = rng.random() < 0.5
        # the bytes of tokens and sorted rows (twice with a gradient) at most the largest listed case's
        most = 16384 * 9 * 2048 * 2 // (cols * (top_k + 1) * _SIZE[dtype] * (2 if grad else 1))
        return dict(kind=kind, tokens=_log_int(rng, 1, min(16384, most)), top_k=top_k,
                    experts=rng.choice([16, 64, 128, 256, 512]), cold=rng.choice([0.0, 0.0, 0.3, 0.9]), cols=cols,
                    dtype=dtype, grad=grad)
    group = rng.choice([32, 64, 128, 128])
    rows, cols = rng.choice([(1024, 2048), (2048, 512), (2048, 768), (1536, 2048), (7168, 2048), (4096, 7168),
                             (1000, 1000), (515, 1111), (2048, 2080)])
    case = dict(kind=kind, tokens=_log_int(rng, 1, 64))
    if kind != "dense":
        # experts * rows * cols at most the largest listed case's
        case.update(top_k=rng.choice([1, 2, 4, 8]), experts=min(rng.choice([8, 16, 32, 64, 128, 256]),
                                                              24 * 4096 * 7168 // (rows * cols)),
                    cold=rng.choice([0.0, 0.3]))
    case.update(rows=rows, cols=cols, group=group, zeros=rng.random() < 0.5, dtype=dtype,
                sdtype=rng.choice([dtype, dtype, "f32"]))
    return case


# ---------------------------------------------------------------- inputs

def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + salt * 7919) % (1 << 62))
    return g


def _randn(seed, salt, shape, dtype):
    return torch.randn(shape, generator=_gen(seed, salt), device="cuda").to(dtype)


def _routing(case, seed):
    """(ids int32 [T, k], a share of them -1; weights fp32 [T, k])."""
    g = _gen(seed, 1)
    E, shape = case["experts"], (case["tokens"], case["top_k"])
    logp = -1.1 * torch.log(torch.arange(1, E + 1, device="cuda", dtype=torch.float32))
    logp = logp[torch.randperm(E, generator=g, device="cuda")]
    u = torch.rand((shape[0], E), generator=g, device="cuda").clamp_(1e-9, 1 - 1e-7)
    sel, ids = torch.topk(logp - torch.log(-torch.log(u)), shape[1], dim=1)
    cold = torch.rand(shape, generator=g, device="cuda") < case["cold"]
    return ids.masked_fill(cold, -1).to(torch.int32), torch.softmax(sel, dim=1)


def _order(ids, n_experts):
    """(offsets int32 [E + 1], perm int32 [R], pos int32 [T, k]) of a stable sort by expert; the routes
    without one come last and carry the complement of their index or place."""
    flat = ids.reshape(-1)
    key = torch.where((flat >= 0) & (flat < n_experts), flat, n_experts)
    order = torch.argsort(key, stable=True)
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device=order.device)
    counts = (key[:, None] == torch.arange(n_experts, device=key.device)).sum(0)
    offsets = torch.cat([counts.new_zeros(1), torch.cumsum(counts, 0)]).to(torch.int32)
    perm = torch.where(key[order] < n_experts, order, ~order).to(torch.int32)
    pos = torch.where(key < n_experts, place, ~place).to(torch.int32)
    return offsets, perm, pos.reshape(ids.shape)


def _weights(case, seed):
    """(codes uint8 [E, N, ceil(K / 2)], scales [E, N, groups], zero points uint8 or None); no E if dense."""
    g = _gen(seed, 2)
    N, K = case["rows"], case["cols"]
    lead = () if case["kind"] == "dense" else (case["experts"],)
    half, groups = (K + 1) // 2, -(-K // case["group"])

    def codes():
        v = torch.randn(lead + (N, half), generator=g, device="cuda", dtype=torch.float32)
        return v.mul_(3.0).add_(7.5).round_().clamp_(0, 15).to(torch.uint8)

    q = codes() | (codes() << 4)
    s = (torch.rand(lead + (N, groups), generator=g, device="cuda") * 0.007 + 0.003).to(_DTYPE[case["sdtype"]])
    z = torch.randint(6, 10, lead + (N, groups), generator=g, device="cuda", dtype=torch.uint8) if case["zeros"] else None
    return q, s, z


def prepare(case, seed):
    state = dict(case)
    dtype, kind = _DTYPE[case["dtype"]], case["kind"]
    T, K = case["tokens"], case["cols"]
    if kind == "dense":
        state.update(x=_randn(seed, 3, (T, K), dtype))
        state["q"], state["s"], state["z"] = _weights(case, seed)
        return state
    ids, w = _routing(case, seed)
    R = T * case["top_k"]
    if kind == "sort":
        state.update(ids=ids, x=_randn(seed, 3, (T, K), dtype), drows=_randn(seed, 4, (R, K), dtype))
        state["x"].requires_grad_(case["grad"])
    elif kind == "unsort":
        # the rows as the experts' products leave them, those past the last expert's segment zero
        offsets, _, pos = _order(ids, case["experts"])
        rows = _randn(seed, 3, (R, K), dtype)
        rows.masked_fill_(torch.arange(R, device="cuda")[:, None] >= offsets[-1], 0.0)
        state.update(pos=pos, rows=rows.requires_grad_(case["grad"]), w=w.requires_grad_(case["grad"]),
                     dy=_randn(seed, 4, (T, K), dtype))
    else:
        state["q"], state["s"], state["z"] = _weights(case, seed)
        if kind == "routed":
            state.update(x=_randn(seed, 3, (T, K), dtype), ids=ids.reshape(-1))
        else:
            state.update(x=_randn(seed, 3, (R, K), dtype), offsets=_order(ids, case["experts"])[0])
    return state


# ---------------------------------------------------------------- the plain forms

def _plain_sort(state):
    x, ids = state["x"].detach(), state["ids"]
    T, k = ids.shape
    offsets, perm, pos = _order(ids, state["experts"])
    route = torch.where(perm >= 0, perm, ~perm).long()
    rows = torch.where((perm >= 0)[:, None], x[route // k], torch.zeros((), dtype=x.dtype, device=x.device))
    out = dict(rows=rows, offsets=offsets, perm=perm, pos=pos)
    if state["grad"]:
        d = state["drows"][torch.where(pos >= 0, pos, 0).long()].float()
        out["dx"] = (d * (pos >= 0)[:, :, None]).sum(1).to(x.dtype)
    return out


def _plain_unsort(state):
    rows, w, pos = state["rows"].detach(), state["w"].detach(), state["pos"]
    placed = pos >= 0
    at = torch.where(placed, pos, ~pos).long()
    w = torch.where(placed, w, torch.zeros((), device=w.device))
    picked = rows[at].float()
    out = dict(y=(picked * w[:, :, None]).sum(1).to(rows.dtype))
    if state["grad"]:
        dy = state["dy"].float()
        out["drows"] = torch.empty_like(rows)
        out["drows"][at.reshape(-1)] = (dy[:, None, :] * w[:, :, None]).reshape(-1, rows.shape[1]).to(rows.dtype)
        out["dw"] = torch.where(placed, (picked * dy[:, None, :]).sum(2), torch.zeros((), device=w.device))
    return out


def _dequant(q, s, z, group, cols):
    """The 4-bit weights in fp32 [..., N, K]."""
    v = torch.stack([q & 15, q >> 4], dim=-1).flatten(-2)[..., :cols].float()
    at = torch.arange(cols, device=q.device) // group
    v -= 8.0 if z is None else z.float()[..., at]
    v *= s.float()[..., at]
    return v


def _plain_w4(state):
    x, q, s, z = state["x"], state["q"], state["s"], state["z"]
    G, K = state["group"], state["cols"]
    if state["kind"] == "dense":
        return torch.matmul(x.float(), _dequant(q, s, z, G, K).t()).to(x.dtype)
    E = state["experts"]
    if state["kind"] == "routed":
        e = state["ids"].long()
        rows = x.float()[torch.arange(e.numel(), device=e.device) // state["top_k"]]
    else:
        at = torch.arange(x.shape[0], device=x.device)
        e = (at[:, None] >= state["offsets"][None, 1:]).sum(1)
        rows = x.float()
    valid = (e >= 0) & (e < E)
    e = torch.where(valid, e, 0)
    if e.numel() < E:  # the routes' own matrices
        w = _dequant(q[e], s[e], None if z is None else z[e], G, K)
        y = torch.matmul(w, rows[:, :, None])[:, :, 0]
    else:  # every expert's products, of which the routes' own are kept
        y = torch.matmul(rows[None], _dequant(q, s, z, G, K).transpose(1, 2))
        y = y[e, torch.arange(e.numel(), device=e.device)]
    return torch.where(valid[:, None], y, torch.zeros((), device=y.device)).to(x.dtype)


def run(state):
    kind = state["kind"]
    if own:
        S, W = _framework()
        if kind == "sort":
            r = S.moe_sort(state["x"], state["ids"], state["experts"])
            out = dict(rows=r.rows, offsets=r.offsets, perm=r.perm, pos=r.pos)
            if state["grad"]:
                out["dx"], = torch.autograd.grad(r.rows, state["x"], state["drows"])
            return out
        if kind == "unsort":
            out = dict(y=S.moe_unsort(state["rows"], state["w"], state["pos"]))
            if state["grad"]:
                out["drows"], out["dw"] = torch.autograd.grad(out["y"], (state["rows"], state["w"]), state["dy"])
            return out
        if kind == "dense":
            return W.w4_vec(state["x"], state["q"], state["s"], state["z"], state["group"])
        if kind == "routed":
            return W.moe_w4_vec(state["x"], state["q"], state["s"], state["ids"], state["top_k"], state["z"],
                                state["group"])
        return W.moe_w4_sorted(state["x"], state["q"], state["s"], state["offsets"], state["z"], state["group"])
    if kind == "sort":
        return _plain_sort(state)
    if kind == "unsort":
        return _plain_unsort(state)
    return _plain_w4(state)


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    kind, k = case["kind"], case.get("top_k", 1)
    if kind == "sort":
        x, ids, E = st["x"].detach().double(), st["ids"], case["experts"]
        T = x.shape[0]
        rows = torch.zeros((T * k, x.shape[1]), dtype=torch.float64, device="cuda")
        dx = torch.zeros_like(x)
        at = 0
        for e in range(E):
            route = (ids.reshape(-1) == e).nonzero().reshape(-1)
            n = route.numel()
            rows[at:at + n] = x[route // k]
            if case["grad"]:
                dx.index_add_(0, route // k, st["drows"][at:at + n].double())
            at += n
        out = dict(rows=rows, offsets=None, perm=None, pos=None)
        return dict(out, dx=dx) if case["grad"] else out
    if kind == "unsort":
        rows, w, pos = st["rows"].detach(), st["w"].detach().double(), st["pos"]
        T, K = pos.shape[0], rows.shape[1]
        y = torch.zeros((T, K), dtype=torch.float64, device="cuda")
        drows = torch.zeros(rows.shape, dtype=torch.float64, device="cuda")
        dw = torch.zeros((T, k), dtype=torch.float64, device="cuda")
        dy = st["dy"].double()
        for j in range(k):
            t = (pos[:, j] >= 0).nonzero().reshape(-1)
            p = pos[t, j].long()
            y[t] += w[t, j, None] * rows[p].double()
            drows[p] = w[t, j, None] * dy[t]
            dw[t, j] = (dy[t] * rows[p].double()).sum(1)
        return dict(y=y, drows=drows, dw=dw) if case["grad"] else dict(y=y)
    N, K, G = case["rows"], case["cols"], case["group"]
    x = st["x"].double()

    def matrix(q, s, z):
        w = torch.empty((N, q.shape[1], 2), dtype=torch.float64, device="cuda")
        w[:, :, 0], w[:, :, 1] = (q % 16).double(), (q // 16).double()
        w = w.reshape(N, -1)[:, :K].contiguous()
        for i, k0 in enumerate(range(0, K, G)):
            w[:, k0:k0 + G] -= 8.0 if z is None else z[:, i, None].double()
            w[:, k0:k0 + G] *= s[:, i, None].double()
        return w

    if kind == "dense":
        return x @ matrix(st["q"], st["s"], st["z"]).t()
    y = torch.zeros((case["tokens"] * k, N), dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        if kind == "routed":
            r = (st["ids"] == e).nonzero().reshape(-1)
            rows = x[r // k]
        else:
            r = torch.arange(int(st["offsets"][e]), int(st["offsets"][e + 1]), device="cuda")
            rows = x[r]
        if r.numel():
            y[r] = rows @ matrix(st["q"][e], st["s"][e], None if st["z"] is None else st["z"][e]).t()
    return y


# ---------------------------------------------------------------- what a pass cannot do without

def _touched(case):
    """Experts with a route, expected over the routing's distribution."""
    E, k = case["experts"], case["top_k"]
    p = [(e + 1) ** -1.1 for e in range(E)]
    total = sum(p)
    draws = case["tokens"] * k * (1 - case["cold"])
    return sum(1 - (1 - v / total) ** draws for v in p)


def work(case):
    T, K, es, k = case["tokens"], case["cols"], _SIZE[case["dtype"]], case.get("top_k", 1)
    R = T * k
    if case["kind"] in ("sort", "unsort"):
        hot = R * (1 - case["cold"])
        if case["kind"] == "sort":
            b = T * K * es + R * K * es + 12 * R + 4 * (case["experts"] + 1)
            f = 0
            if case["grad"]:
                b += hot * K * es + T * K * es
                f += hot * K
        else:
            b = hot * K * es + T * K * es + 8 * R
            f = 2 * hot * K
            if case["grad"]:
                b += T * K * es + R * K * es + 4 * R
                f += 3 * hot * K
        return dict(bytes=b, flops=f)
    N = case["rows"]
    matrix = N * ((K + 1) // 2 + -(-K // case["group"]) * (_SIZE[case["sdtype"]] + case["zeros"]))
    if case["kind"] == "dense":
        return dict(bytes=matrix + T * (K + N) * es, flops=2 * T * N * K)
    rows_in = T if case["kind"] == "routed" else R
    return dict(bytes=_touched(case) * matrix + rows_in * K * es + R * N * es + 4 * (R if case["kind"] == "routed" else case["experts"]),
                flops=2 * R * (1 - case["cold"]) * N * K)
