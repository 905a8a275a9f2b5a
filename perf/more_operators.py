"""More operators around the experts' products, measured one case at a time: products in 8-bit floating
point with a scale for each block of 128, gated feed-forward products and experts' products with their
gradients.

Kinds of case:
  fp8           kt_fp8_block.fp8_linear: rows of x, quantised in groups of 128, by one e4m3 matrix
  fp8_routed    kt_fp8_block.moe_fp8_vec: each route's row by the e4m3 matrix of its expert
  fp8_sorted    kt_fp8_block.moe_fp8_sorted: the same for rows already sorted by expert
  gated         kt_gated.gated: act(x Wg^T) * (x Wu^T) of one matrix [gate; up]; with grad, the
                gradients of x and of the matrix too
  gated_sorted  kt_gated.moe_gated_sorted: the same for rows sorted by expert
  linear_sorted kt_gated.moe_linear_sorted: rows sorted by expert by their expert's matrix; with grad,
                the gradients of the rows and of the matrices too

With `own` false, `run` computes them in elementary torch operations in 32 bits; with `own` true it
calls the framework. `exact` computes them in 64 bits.

Shapes are those of the package's own workloads (synth.WORKLOADS) and generic ones. Inputs:
activations ~ N(0, 1), Zipf expert popularity, top-k of Gumbel-perturbed logits, weights ~ N(0, 0.02),
e4m3 codes distributed as quantised normals.
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
    """(kt_fp8_block, kt_gated) of this repository's package."""
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
        import kt_prefill_lend_amd.kt_fp8_block as F
        import kt_prefill_lend_amd.kt_gated as G

        _ops = (F, G)
    return _ops


_DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
_BLOCK = 128  # values of a group of x, and rows and columns of a block of weights
_TOP = 448.0  # e4m3's largest value
_LEAST = 2.0 ** -116  # a group's largest value counts as at least this


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # a dense projection of one user's token
        dict(name="fp8-1", kind="fp8", tokens=1, rows=4096, cols=7168, dtype="bf16"),
        # the same projection of a prefill chunk
        dict(name="fp8-2047", kind="fp8", tokens=2047, rows=4096, cols=7168, dtype="bf16"),
        # the gate and up rows of one user's decode step of a small-expert model, in fp16
        dict(name="moe-fp8-1-f16", kind="fp8_routed", tokens=1, top_k=8, experts=256, cold=0.0, rows=1024, cols=2048,
             dtype="f16"),
        # a decode window of a large-expert model, a third of its routes on the CPU
        dict(name="moe-fp8-13", kind="fp8_routed", tokens=13, top_k=8, experts=24, cold=0.3, rows=4096, cols=7168,
             dtype="bf16"),
        # the down products of a decode batch's sorted routes
        dict(name="fp8-sorted-77", kind="fp8_sorted", tokens=77, top_k=8, experts=128, cold=0.0, rows=2048, cols=768,
             dtype="bf16"),
        # the gate and up products of a full prefill chunk on a rank that holds most of the experts
        dict(name="fp8-sorted-16384", kind="fp8_sorted", tokens=16384, top_k=8, experts=256, cold=0.3, rows=1024,
             cols=2048, dtype="bf16"),
        # a dense layer's gate and up of one user's token
        dict(name="gated-1", kind="gated", tokens=1, inter=2048, cols=7168, act="silu", dtype="bf16", grad=False),
        # a training step of that layer
        dict(name="gated-4096-grad", kind="gated", tokens=4096, inter=2048, cols=7168, act="silu", dtype="bf16", grad=True),
        # a decode batch's sorted routes, in fp16, with the other activation
        dict(name="moe-gated-24-f16", kind="gated_sorted", tokens=24, top_k=8, experts=128, cold=0.0, inter=768,
             cols=2048, act="gelu_tanh", dtype="f16", grad=False),
        # a training step's sequence over experts, some of whose routes are on another rank
        dict(name="moe-gated-2047-grad", kind="gated_sorted", tokens=2047, top_k=8, experts=128, cold=0.2, inter=768,
             cols=2048, act="silu", dtype="bf16", grad=True),
        # small experts trained in fp32 on a ragged sequence
        dict(name="moe-linear-1021-f32-grad", kind="linear_sorted", tokens=1021, top_k=4, experts=64, cold=0.0, rows=1000,
             cols=515, dtype="f32", grad=True),
        # the down products of a training step's batch
        dict(name="moe-linear-4096-grad", kind="linear_sorted", tokens=4096, top_k=8, experts=128, cold=0.0, rows=2048,
             cols=768, dtype="bf16", grad=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["fp8", "fp8_routed", "fp8_sorted", "gated", "gated_sorted", "linear_sorted"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    rows, cols = rng.choice([(1024, 2048), (2048, 512), (2048, 768), (7168, 2048), (4096, 7168), (1000, 1000),
                             (515, 1111), (2048, 2080), (96, 4096)])
    case = dict(kind=kind, dtype=dtype, cols=cols)
    if kind in ("gated", "gated_sorted"):
        case.update(inter=rows // 2, act=rng.choice(["silu", "silu", "gelu_tanh"]))
        rows = rows // 2 * 2
    else:
        case.update(rows=rows)
    grad = kind in ("gated", "gated_sorted", "linear_sorted") and rng.random() < 0.5
    if kind in ("gated", "gated_sorted", "linear_sorted"):
        case.update(grad=grad)
    # the operations of a pass at most a share of the largest listed case's (in fp32 a small one), and
    # at most as many bytes of matrices
    most = (2 * 3 * 4096 * 4096 * 7168) // ((6 if grad else 2) * rows * cols * (16 if dtype == "f32" else 1))
    if kind in ("fp8", "gated"):
        return dict(case, tokens=_log_int(rng, 1, max(1, min(8192, most))))
    top_k = rng.choice([1, 2, 4, 8])
    size = _SIZE[dtype] * (2 if grad else 1) if kind in ("gated_sorted", "linear_sorted") else 1
    experts = max(1, min(rng.choice([8, 16, 32, 64, 128, 256]), 24 * 4096 * 7168 // (rows * cols * size)))
    top_k = min(top_k, experts)
    highest = 64 if kind == "fp8_routed" else max(1, min(16384, most // top_k, (1 << 28) // (top_k * max(rows, cols))))
    return dict(case, tokens=_log_int(rng, 1, highest), top_k=top_k, experts=experts, cold=rng.choice([0.0, 0.0, 0.3, 0.9]))


# ---------------------------------------------------------------- inputs

def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + salt * 7919) % (1 << 62))
    return g


def _randn(seed, salt, shape, dtype, sigma=1.0):
    g = _gen(seed, salt)
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    for i in range(0, flat.numel(), 1 << 27):  # no fp32 copy of all the experts' weights at once
        n = min(1 << 27, flat.numel() - i)
        flat[i:i + n] = torch.randn(n, generator=g, device="cuda").mul_(sigma).clamp_(-_TOP, _TOP)  # e4m3's range
    return out


def _routing(case, seed):
    """ids int32 [T, k], a share of them -1."""
    g = _gen(seed, 1)
    E, shape = case["experts"], (case["tokens"], case["top_k"])
    logp = -1.1 * torch.log(torch.arange(1, E + 1, device="cuda", dtype=torch.float32))
    logp = logp[torch.randperm(E, generator=g, device="cuda")]
    u = torch.rand((shape[0], E), generator=g, device="cuda").clamp_(1e-9, 1 - 1e-7)
    ids = torch.topk(logp - torch.log(-torch.log(u)), shape[1], dim=1).indices
    cold = torch.rand(shape, generator=g, device="cuda") < case["cold"]
    return ids.masked_fill(cold, -1).to(torch.int32)


def _offsets(ids, n_experts):
    counts = (ids.reshape(-1, 1) == torch.arange(n_experts, device=ids.device)).sum(0)
    return torch.cat([counts.new_zeros(1), torch.cumsum(counts, 0)]).to(torch.int32)


def prepare(case, seed):
    state = dict(case)
    kind, dtype, T, K = case["kind"], _DTYPE[case["dtype"]], case["tokens"], case["cols"]
    N = 2 * case["inter"] if "inter" in case else case["rows"]
    lead = (case["experts"],) if "experts" in case else ()
    if kind.startswith("fp8"):
        state["w"] = _randn(seed, 2, lead + (N, K), torch.float8_e4m3fn, 110.0)
        blocks = lead + (-(-N // _BLOCK), -(-K // _BLOCK))
        state["s"] = torch.rand(blocks, generator=_gen(seed, 5), device="cuda").mul_(0.5).add_(0.75).mul_(0.02 / 110.0)
    else:
        state["w"] = _randn(seed, 2, lead + (N, K), dtype, 0.02)
    R = T
    if lead:
        ids = _routing(case, seed)
        if kind == "fp8_routed":
            state["ids"] = ids.reshape(-1)
        else:
            R = T * case["top_k"]
            state["offsets"] = _offsets(ids, case["experts"])
    state["x"] = _randn(seed, 3, (R, K), dtype)
    if "offsets" in state:  # rows past the last expert's, as the sort leaves them
        state["x"].masked_fill_(torch.arange(R, device="cuda")[:, None] >= state["offsets"][-1], 0.0)
    if case.get("grad"):
        state["dy"] = _randn(seed, 4, (R, case.get("inter", N)), dtype)
        state["x"].requires_grad_(True)
        state["w"].requires_grad_(True)
    return state


# ---------------------------------------------------------------- the plain forms

def _rounded_rows(x):
    """The rows as their 8-bit codes and scales stand for them, in fp32."""
    R, K = x.shape
    pad = -K % _BLOCK
    v = torch.nn.functional.pad(x.float(), (0, pad)).reshape(R, -1, _BLOCK)
    top = v.abs().amax(2, keepdim=True).clamp_min(_LEAST)
    most = torch.full_like(top, _TOP)  # a tensor: by a number torch multiplies by its reciprocal, rounded twice
    v = (v * (most / top)).to(torch.float8_e4m3fn).float() * (top / most)
    return v.reshape(R, -1)[:, :K]


def _matrices(w, s):
    """The 8-bit weights in fp32."""
    N, K = w.shape[-2:]
    at_n = torch.arange(N, device=w.device) // _BLOCK
    at_k = torch.arange(K, device=w.device) // _BLOCK
    return w.float() * s[..., at_n, :][..., at_k]


_TILE = 128


def _tiles(offsets, n_rows):
    """Sorted rows as padded tiles of one expert each: (expert [n], row [n, tile], whether it is one [n, tile])."""
    counts = (offsets[1:] - offsets[:-1]).long()
    ends = torch.cumsum((counts + _TILE - 1) // _TILE, 0)
    n = n_rows // _TILE + counts.numel()
    t = torch.arange(n, device=offsets.device)
    e = torch.searchsorted(ends, t, right=True)
    there = e < counts.numel()
    e = torch.where(there, e, 0)
    first = t - torch.where(e > 0, ends[e - 1], 0)
    row = (first * _TILE)[:, None] + torch.arange(_TILE, device=offsets.device)
    valid = there[:, None] & (row < counts[e][:, None])
    row = torch.where(valid, row + offsets.long()[e][:, None], 0)
    return e, row, valid


def _take(rows, tiles):
    return rows[tiles[1]].float() * tiles[2][:, :, None]


def _put(products, tiles, n_rows):
    """The tiles' rows in their places, zeros where no expert has a row."""
    y = torch.zeros((n_rows, products.shape[2]), dtype=products.dtype, device=products.device)
    y[tiles[1][tiles[2]]] = products[tiles[2]]
    return y


def _by_expert(products, tiles, n_experts):
    y = torch.zeros((n_experts,) + products.shape[1:], dtype=products.dtype, device=products.device)
    return y.index_add_(0, tiles[0], products)


def _act(kind, g):
    """(act(g), its derivative)."""
    if kind == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)


def _plain_fp8(state):
    x, w, s = state["x"], state["w"], state["s"]
    v = _rounded_rows(x)
    if state["kind"] == "fp8":
        return torch.matmul(v, _matrices(w, s).t()).to(x.dtype)
    if state["kind"] == "fp8_sorted":
        tiles = _tiles(state["offsets"], x.shape[0])
        m = _matrices(w, s)
        return _put(torch.bmm(_take(v, tiles), m[tiles[0]].transpose(1, 2)), tiles, x.shape[0]).to(x.dtype)
    e = state["ids"].long()
    valid = e >= 0
    e = torch.where(valid, e, 0)
    rows = v[torch.arange(e.numel(), device=e.device) // state["top_k"]]
    if e.numel() < state["experts"]:  # the routes' own matrices
        y = torch.matmul(_matrices(w[e], s[e]), rows[:, :, None])[:, :, 0]
    else:  # every expert's products, of which the routes' own are kept
        y = torch.matmul(rows[None], _matrices(w, s).transpose(1, 2))[e, torch.arange(e.numel(), device=e.device)]
    return (y * valid[:, None]).to(x.dtype)


def _plain_products(state):
    """The gated and the linear products, dense or by expert, with their gradients."""
    x, w = state["x"].detach(), state["w"].detach()
    tiles = _tiles(state["offsets"], x.shape[0]) if "offsets" in state else None
    if tiles is None:
        a, m = x.float()[None], w.float()[None]
    else:
        a, m = _take(x, tiles), w.float()[tiles[0]]
    y = torch.bmm(a, m.transpose(1, 2))
    if "inter" in state:
        g, u = y[:, :, :state["inter"]], y[:, :, state["inter"]:]
        f, df = _act(state["act"], g)
        y = f * u
    out = dict(y=(y[0] if tiles is None else _put(y, tiles, x.shape[0])).to(x.dtype))
    if state["grad"]:
        d = state["dy"].float()[None] if tiles is None else _take(state["dy"], tiles)
        if "inter" in state:
            d = torch.cat([d * u * df, d * f], dim=2)
        dx, dw = torch.bmm(d, m), torch.bmm(d.transpose(1, 2), a)
        out["dx"] = (dx[0] if tiles is None else _put(dx, tiles, x.shape[0])).to(x.dtype)
        out["dw"] = (dw[0] if tiles is None else _by_expert(dw, tiles, w.shape[0])).to(x.dtype)
    return out


def run(state):
    kind = state["kind"]
    if own:
        F, G = _framework()
        if kind == "fp8":
            return F.fp8_linear(state["x"], state["w"], state["s"])
        if kind == "fp8_routed":
            return F.moe_fp8_vec(state["x"], state["w"], state["s"], state["ids"], state["top_k"])
        if kind == "fp8_sorted":
            return F.moe_fp8_sorted(state["x"], state["w"], state["s"], state["offsets"])
        if kind == "gated":
            y = G.gated(state["x"], state["w"], state["act"])
        elif kind == "gated_sorted":
            y = G.moe_gated_sorted(state["x"], state["w"], state["offsets"], state["act"])
        else:
            y = G.moe_linear_sorted(state["x"], state["w"], state["offsets"])
        if not state["grad"]:
            return dict(y=y)
        dx, dw = torch.autograd.grad(y, (state["x"], state["w"]), state["dy"])
        return dict(y=y, dx=dx, dw=dw)
    return _plain_fp8(state) if kind.startswith("fp8") else _plain_products(state)


# ---------------------------------------------------------------- the definition in 64 bits

def _e4m3(v):
    """fp32 values rounded to e4m3's, to nearest, ties to even, in 64 bits."""
    v = v.double()
    exponent = torch.frexp(v).exponent - 1
    step = torch.ldexp(torch.ones_like(v), exponent.clamp_min(-6) - 3)
    return (torch.round(v / step) * step).clamp(-_TOP, _TOP)


def exact(case, seed):
    st = prepare(case, seed)
    kind, dev = case["kind"], "cuda"
    x, w = st["x"].detach().double(), st["w"].detach()
    R, K = x.shape
    if kind.startswith("fp8"):
        # the scale and its inverse are fp32 numbers by definition, and so is the quotient that is rounded to 8 bits
        for k0 in range(0, K, _BLOCK):
            v = x[:, k0:k0 + _BLOCK]
            top = v.abs().amax(1, keepdim=True).clamp_min(_LEAST)
            inverse, scale = (_TOP / top).float().double(), (top / _TOP).float().double()
            x[:, k0:k0 + _BLOCK] = _e4m3((v * inverse).float()) * scale

    def matrix(e):
        m = (w if e is None else w[e]).double()
        if kind.startswith("fp8"):
            s = st["s"] if e is None else st["s"][e]
            for n, n0 in enumerate(range(0, m.shape[0], _BLOCK)):
                for k, k0 in enumerate(range(0, K, _BLOCK)):
                    m[n0:n0 + _BLOCK, k0:k0 + _BLOCK] *= s[n, k].double()
        return m

    if kind == "fp8":
        return x @ matrix(None).t()
    if kind == "fp8_routed":
        y = torch.zeros((R * case["top_k"], case["rows"]), dtype=torch.float64, device=dev)
        for e in range(case["experts"]):
            r = (st["ids"] == e).nonzero().reshape(-1)
            if r.numel():
                y[r] = x[r // case["top_k"]] @ matrix(e).t()
        return y
    if kind == "fp8_sorted":
        y = torch.zeros((R, case["rows"]), dtype=torch.float64, device=dev)
        ends = st["offsets"].tolist()
        for e in range(case["experts"]):
            if ends[e + 1] > ends[e]:
                y[ends[e]:ends[e + 1]] = x[ends[e]:ends[e + 1]] @ matrix(e).t()
        return y
    width = case.get("inter", case.get("rows"))
    y = torch.zeros((R, width), dtype=torch.float64, device=dev)
    dx, dw = torch.zeros_like(x), torch.zeros(w.shape, dtype=torch.float64, device=dev) if case["grad"] else None
    parts = [(None, 0, R)]
    if "experts" in case:
        ends = st["offsets"].tolist()
        parts = [(e, ends[e], ends[e + 1]) for e in range(case["experts"]) if ends[e + 1] > ends[e]]
    for e, a, b in parts:
        m = matrix(e)
        v = x[a:b] @ m.t()
        if "inter" in case:
            g, u = v[:, :width], v[:, width:]
            if case["act"] == "silu":
                sig = torch.sigmoid(g)
                f, df = g * sig, sig + g * sig * (1 - sig)
            else:
                z = math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
                dz = math.sqrt(2 / math.pi) * (1 + 0.134145 * g ** 2)
                f, df = g * (1 + torch.tanh(z)) / 2, (1 + torch.tanh(z)) / 2 + g * dz / (2 * torch.cosh(z) ** 2)
            v = f * u
        y[a:b] = v
        if case["grad"]:
            d = st["dy"][a:b].double()
            if "inter" in case:
                d = torch.cat([d * u * df, d * f], 1)
            dx[a:b] = d @ m
            (dw if e is None else dw[e]).copy_(d.t() @ x[a:b])
    return dict(y=y, dx=dx, dw=dw) if case["grad"] else dict(y=y)


# ---------------------------------------------------------------- what a pass cannot do without

def _touched(case):
    """Experts with a route, expected over the routing's distribution."""
    E, k = case["experts"], case["top_k"]
    p = [(e + 1) ** -1.1 for e in range(E)]
    total = sum(p)
    draws = case["tokens"] * k * (1 - case["cold"])
    return sum(1 - (1 - v / total) ** draws for v in p)


def work(case):
    kind, K, es = case["kind"], case["cols"], _SIZE[case["dtype"]]
    N = 2 * case["inter"] if "inter" in case else case["rows"]
    width = case.get("inter", N)
    rows_out = case["tokens"] * case.get("top_k", 1)
    rows_in = case["tokens"] if kind in ("fp8", "fp8_routed") else rows_out
    active = rows_out * (1 - case.get("cold", 0.0))
    read_in = rows_in if kind in ("fp8", "fp8_routed", "gated") else active
    touched = _touched(case) if "experts" in case else 1
    ints = 4 * (rows_out if kind == "fp8_routed" else case.get("experts", -1) + 1)
    flops = 2 * active * N * K
    if kind.startswith("fp8"):
        matrix = N * K + 4 * (-(-N // _BLOCK)) * (-(-K // _BLOCK))
        return dict(bytes=touched * matrix + read_in * K * es + rows_out * N * es + ints, flops=flops)
    b = touched * N * K * es + read_in * K * es + rows_out * width * es + ints
    if case["grad"]:
        b += active * width * es + rows_out * K * es + case.get("experts", 1) * N * K * es
        flops *= 3
    return dict(bytes=b, flops=flops)
