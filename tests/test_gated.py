"""Gated and linear products by expert and their gradients (kt_gated).

The linear products are tested with small integers: every product and partial sum is exact in fp32 whatever the
order of the sums, so outputs and gradients have to be equal bit for bit. The gate is not exact: its values
are tested against 64 bits, with the roundings counted, and its gradients against the formula and against differences."""
import ctypes
import math

import pytest
import torch

import kt_prefill_lend_amd.kt_gated as G
import kt_prefill_lend_amd.kt_moe_sort as S
from helpers import check_refused_records, wrapped
from kt_prefill_lend_amd import _lib

gpu = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
ACTS = ["silu", "gelu_tanh"]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def ints(shape, dtype, seed, dev, top=3):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-top, top + 1, shape, generator=g).to(dtype).to(dev)


def randn(shape, dtype, seed, dev, sigma=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * sigma).to(dtype).to(dev)


def segments(counts, tail, dev):
    offsets = torch.tensor([0] + counts).cumsum(0).to(torch.int32).to(dev)
    return offsets, sum(counts) + tail


def spans(offsets, R):
    o = offsets.tolist()
    return [(e, min(max(o[e], 0), R), min(max(o[e + 1], 0), R)) for e in range(len(o) - 1)]


def act64(act, g):
    """(act(g), its derivative) in 64 bits."""
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    c = 2 * math.sqrt(2 / math.pi)  # (1 + tanh z) / 2 = sigmoid(2 z), without tanh's cancellation at -1
    s = torch.sigmoid(c * (g + 0.044715 * g ** 3))
    return g * s, s + g * s * torch.sigmoid(-c * (g + 0.044715 * g ** 3)) * c * (1 + 3 * 0.044715 * g ** 2)


def linear64(x, w, offsets, dy=None):
    """y, dx, dw of the linear products in 64 bits."""
    y = torch.zeros((x.shape[0], w.shape[1]), dtype=torch.float64, device=x.device)
    dx, dw = torch.zeros(x.shape, dtype=torch.float64, device=x.device), torch.zeros(w.shape, dtype=torch.float64, device=x.device)
    for e, a, b in spans(offsets, x.shape[0]):
        if b > a:
            y[a:b] = x[a:b].double() @ w[e].double().t()
            if dy is not None:
                dx[a:b] = dy[a:b].double() @ w[e].double()
                dw[e] = dy[a:b].double().t() @ x[a:b].double()
    return y, dx, dw


def gated64(x, w13, offsets, act, dh=None):
    """h, dx, dw13 in 64 bits; offsets None: dense."""
    w = w13[None] if offsets is None else w13
    off = torch.tensor([0, x.shape[0]]) if offsets is None else offsets
    n = w.shape[1] // 2
    v = linear64(x, w, off)[0]
    g, u = v[:, :n], v[:, n:]
    f, df = act64(act, g)
    if dh is None:
        return f * u, None, None
    d = torch.cat([dh.double() * u * df, dh.double() * f], 1)
    _, dx, dw = linear64(x, w, off, d)
    return f * u, dx, dw[0] if offsets is None else dw


def same(got, want64):
    assert torch.equal(got, want64.float().to(got.dtype)), (got.double() - want64).abs().max()


def grads(fn, leaves, d):
    y = fn(*leaves)
    return [y.detach(), *torch.autograd.grad(y, leaves, d)]


# rows of each expert, rows behind the last, N, K
LINEAR = [([1], 0, 1, 1), ([2], 0, 5, 7), ([0, 3, 0, 0, 17, 1, 0], 4, 72, 384), ([0, 0, 0], 7, 9, 96), ([70, 0, 33], 0, 40, 130),
          ([5] * 60, 3, 16, 96), ([300, 2], 1, 24, 256), ([0] * 500 + [2, 1], 2, 33, 64), ([1] * 2048, 5, 3, 8),
          ([129, 0, 257, 64], 130, 300, 144), ([90, 400], 3, 129, 515), ([700, 500], 300, 1030, 520), ([1111], 0, 515, 1111),
          ([260, 230, 200, 250], 9, 2048, 1536), ([3], 0, 33000, 1100), ([2], 1, 33000, 200), ([25, 20], 1, 200, 600)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts,tail,N,K", LINEAR)
def test_linear_exact(dev, counts, tail, N, K, dtype):
    offsets, R = segments(counts, tail, dev)
    x, w, dy = ints((R, K), dtype, 1, dev), ints((len(counts), N, K), dtype, 2, dev), ints((R, N), dtype, 3, dev)
    want = linear64(x, w, offsets, dy)
    same(G.moe_linear_sorted(x, w, offsets), want[0])
    got = grads(lambda x, w: G.moe_linear_sorted(x, w, offsets), [x.requires_grad_(True), w.requires_grad_(True)], dy)
    for a, b in zip(got, want):
        same(a, b)


# the gate and up of whole tiles, of parts of them, of few rows
GATED = [(1, 1, 1), (3, 5, 7), (16, 8, 64), (17, 33, 130), (64, 20, 515), (65, 1, 8), (100, 130, 256), (200, 257, 1000), (1000, 1100, 144),
         (2, 17000, 1100), (3, 17000, 130), (30, 300, 500)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("T,N,K", GATED)
def test_gated_and_gradients(dev, T, N, K, act, dtype):
    check_gated(randn((T, K), dtype, 1, dev), randn((2 * N, K), dtype, 2, dev, 1 / math.sqrt(K)), None, act,
                randn((T, N), dtype, 3, dev))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("counts,tail,N,K", [([1], 0, 5, 64), ([0, 3, 0, 17, 1, 0], 4, 72, 384), ([0, 0], 7, 9, 96),
                                             ([70, 0, 33], 5, 40, 130), ([129, 0, 257, 64], 130, 300, 144), ([90, 400], 3, 129, 515)])
def test_gated_sorted_and_gradients(dev, counts, tail, N, K, act, dtype):
    offsets, R = segments(counts, tail, dev)
    check_gated(randn((R, K), dtype, 1, dev), randn((len(counts), 2 * N, K), dtype, 2, dev, 1 / math.sqrt(K)), offsets, act,
                randn((R, N), dtype, 3, dev))


def check_gated(x, w, offsets, act, dh):
    """Each sum of K products is off by at most (K + 4) 2^-24 of the terms' size (a chain of K additions, each of a partial sum below
    it), which with weights of size 1 / sqrt(K) and normal rows is about sqrt(K) as large as the sum's
    own; as a whole roundings of independent sign are off by 3 sqrt(K) 2^-24 of it. act has slope up to 1.13, its derivative up to
    0.8, and __expf and the quotient are off by 2^-21 of the value, so h's share of that is below 2^-18. h is rounded once; dx and dw take the
    projections' gradients rounded once (half a step of each, of independent sign over the sums: half a step as a whole)
    and are rounded once themselves."""
    dtype, K = x.dtype, x.shape[1]
    want = gated64(x, w, offsets, act, dh)
    fn = (lambda x, w: G.gated(x, w, act)) if offsets is None else (lambda x, w: G.moe_gated_sorted(x, w, offsets, act))
    h = fn(x, w)
    got = grads(fn, [x.requires_grad_(True), w.requires_grad_(True)], dh)
    assert torch.equal(h, got[0])
    u = half_step(dtype)
    noise = 8 * 3 * math.sqrt(max(K, 2 * dh.shape[1], x.shape[0])) * 2.0 ** -24 + 2.0 ** -18
    tiny = 2.0 ** -25 * math.sqrt(want[2].numel()) if dtype == torch.float16 else 0.0  # f16's subnormal steps
    for a, b, roundings in zip(got, want, (1, 2, 2)):
        assert a.dtype == dtype and a.shape == b.shape
        assert (a.double() - b).norm() <= (roundings * u + noise) * b.norm() + tiny, roundings
    for e, a, b in ([] if offsets is None else spans(offsets, x.shape[0])):
        if a == b:
            assert (got[2][e] == 0).all()
    if offsets is not None:
        end = int(offsets[-1])
        assert (got[0][end:] == 0).all() and (got[1][end:] == 0).all()


def kernel_of(what, dtype, N, K, E, R):
    k = _lib.ktmi_prod_kernel()
    assert _lib.lib().ktmi_linear_kernel_of(what, _lib.dtype_code(dtype), N, K, E, R, ctypes.byref(k)) == 0
    return k.tile_rows, k.tile_cols, k.splits


# what, rows of each expert, N, K -> the tile of 16-bit and of fp32 rows and whether blocks share its k; K with whole steps,
# with a last chunk, with a word in it
FWD, DX, DW = _lib.PROD_LINEAR, _lib.PROD_GRAD_X, _lib.PROD_GRAD_W
SHAPES = [(FWD, [30, 3], 40, 192, (0, 0), (0, 0), False), (FWD, [40, 70], 300, 128, (64, 128), (64, 128), False),
          (FWD, [40, 70], 300, 136, (64, 128), (64, 128), False), (FWD, [40, 70], 300, 134, (64, 128), (64, 128), False),
          (FWD, [250], 12300, 128, (128, 128), (64, 128), False), (FWD, [250], 12300, 138, (128, 128), (64, 128), False),
          (FWD, [250, 252], 12300, 128, (128, 256), (64, 128), False), (FWD, [250, 252], 12300, 130, (128, 256), (64, 128), False),
          (FWD, [1000], 12300, 128, (256, 256), (256, 256), False), (FWD, [1000], 12300, 150, (256, 256), (256, 256), False),
          (FWD, [40, 70], 130, 4096, (64, 128), (64, 128), True), (FWD, [600], 200, 4100, (64, 128), (64, 128), True),
          (DX, [40, 70], 128, 300, (64, 128), (64, 128), False), (DX, [250], 128, 12300, (128, 128), (64, 128), False),
          (DX, [250], 138, 12300, (128, 128), (64, 128), False), (DX, [1000], 128, 12300, (256, 256), (256, 256), False),
          (DX, [1000], 150, 12300, (256, 256), (256, 256), False), (DX, [70, 90], 4100, 130, (64, 128), (64, 128), True),
          (DW, [40, 70], 200, 300, (128, 128), (128, 128), False), (DW, [60], 3300, 4100, (256, 256), (128, 128), False),
          (DW, [5000], 200, 300, (128, 128), (128, 128), True), (DW, [2500, 2400], 100, 90, (128, 128), (128, 128), True)]


def test_kernel_shapes_are_all_reached():
    reached = set()
    for what, counts, N, K, narrow, wide, split in SHAPES:
        for dtype in DTYPES:
            *tile, splits = kernel_of(what, dtype, N, K, len(counts), sum(counts) + 5)
            assert tuple(tile) == (wide if dtype == torch.float32 else narrow) and (splits > 1) == split, (what, counts, N, K, dtype, tile, splits)
            reached.add((what, *tile, splits > 1))
    tiles = {(64, 128), (128, 128), (256, 256)}
    assert {(w, *t, False) for w in (FWD, DX) for t in tiles} | {(FWD, 128, 256, False), (FWD, 0, 0, False), (DW, 256, 256, False),
                                                                 (DW, 128, 128, False)} <= reached
    k = ctypes.byref(_lib.ktmi_prod_kernel())
    for args in [(4, 2, 8, 8, 1, 1, k), (-1, 2, 8, 8, 1, 1, k), (0, 3, 8, 8, 1, 1, k), (0, 2, 0, 8, 1, 1, k), (0, 2, 8, 0, 1, 1, k),
                 (0, 2, 8, 8, 0, 1, k), (0, 2, 8, 8, 1, 0, k), (0, 2, 8, 8, 1, 1, None)]:
        assert _lib.lib().ktmi_linear_kernel_of(*args) == -1


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("what,counts,N,K,narrow,wide,split", SHAPES)
def test_shapes_exact(dev, what, counts, N, K, narrow, wide, split, dtype):
    offsets, R = segments(counts, 5, dev)
    x, w, dy = ints((R, K), dtype, 1, dev, 2), ints((len(counts), N, K), dtype, 2, dev, 2), ints((R, N), dtype, 3, dev, 2)
    want = linear64(x, w, offsets, dy)
    got = grads(lambda x, w: G.moe_linear_sorted(x, w, offsets), [x.requires_grad_(True), w.requires_grad_(True)], dy)
    for a, b in zip(got, want):
        same(a, b)


# rows, I, K: the gate's tiles, with splits and without
@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,N,K,tile,split", [(256, 6150, 128, (128, 128), False), (300, 12300, 192, (128, 256), False),
                                              (1000, 6150, 130, (256, 256), False), (100, 90, 4100, (64, 128), True),
                                              (70, 3, 8192, (64, 128), True)])
def test_gated_shapes(dev, T, N, K, tile, split, dtype):
    *got, splits = kernel_of(_lib.PROD_GATED, dtype, N, K, 1, T)
    assert (dtype == torch.float32 or tuple(got) == tile) and (splits > 1) == split
    check_gated(randn((T, K), dtype, 1, dev), randn((2 * N, K), dtype, 2, dev, 1 / math.sqrt(K)), None, "silu", randn((T, N), dtype, 3, dev))


@gpu
@pytest.mark.parametrize("act", ACTS)
def test_gate_over_its_range(dev, act):
    """One row and column: h = act(g) u at g from -200 to 200, in fp32, and the gradients' factors. Of sigmoid(v): gelu's v takes
    four products and a sum, each off by 2^-24 of itself and all of one sign, so v is off by at most 5 |v| 2^-24; its product with log2 e by
    |v| 2^-24 more; these are sigmoid's relative error where it is small, and the power, sum, quotient and products add at
    most 8 2^-24. Past |v| = 72 the values are below 1e-30, so the relative error is at most (8 + 6 72) 2^-24 < 2^-15."""
    g = torch.cat([torch.linspace(-200, 200, 4001), torch.linspace(-6, 6, 1201), torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1e20, -1e20])])
    x = g[:, None].to(dev).requires_grad_(True)
    w = torch.tensor([[1.0], [0.5]], device=dev).requires_grad_(True)
    h, dx = grads(lambda x: G.gated(x, w.detach(), act), [x], torch.ones((g.numel(), 1), device=dev))
    v = x.detach().double()
    f, df = act64(act, v.clamp(-1e4, 1e4))
    f = torch.where(v.abs() > 1e4, v.clamp_min(0), f)
    want_h, want_dx = f * 0.5 * v, 0.5 * v * df + 0.5 * f
    tol = 2.0 ** -15
    over = want_h.float().isinf()  # 1e20 * 5e19
    assert torch.equal(h[over], want_h.float()[over])
    assert ((h.double() - want_h).abs() <= tol * want_h.abs() + 1e-30)[~over].all()
    # dx = dg + du / 2: both terms are rounded and may cancel
    assert ((dx.double() - want_dx).abs() <= tol * (0.5 * v * df).abs() + tol * (0.5 * f).abs() + 2.0 ** -20 * torch.exp(-v.abs() / 2) + 1e-30).all()


@gpu
@pytest.mark.parametrize("rows,cols,tile,split", [(20, 2, (0, 0), False), (400, 2, (64, 128), False), (100, 4096, (64, 128), True)])
def test_silu_keeps_fp32(dev, rows, cols, tile, split):
    """h, dg and du in fp32 for g from -87, where the sigmoid is a normal number yet, to 87, and u = 1: in units of 2^-24 of their values
    the power is off by 2 at most (a step), the sum and the quotient by 1 each, so the sigmoid s by 4, f = g s by 5, h = f u
    by 6 and du = dh f too. 1 - s is off by 4 s and its own rounding; act' = s + f (1 - s) by 4 s + |f| (4 s + 7 (1 - s))
    and the sum's rounding, dg by one more. The products with w are by 1 and 0. Terms of second order are below 2^-20 of these."""
    N = 90
    *got, splits = kernel_of(_lib.PROD_GATED, torch.float32, N, cols, 1, rows)
    assert tuple(got) == tile and (splits > 1) == split
    u = 2.0 ** -24 * (1 + 2.0 ** -18)
    g = torch.linspace(-87, 87, 400 * 3, device=dev)
    w = torch.zeros((2 * N, cols), device=dev)
    w[:N, 0], w[N:, cols - 1] = 1, 1
    for part in torch.cat([g, torch.linspace(-6, 6, 400, device=dev)]).split(rows):
        x = torch.zeros((rows, cols), device=dev)
        x[:, cols - 1] = 1
        x[:part.numel(), 0] = part
        dh = torch.zeros((rows, N), device=dev)
        dh[:, N - 1] = 1
        h, dx = grads(lambda x: G.gated(x, w), [x.requires_grad_(True)], dh)
        v = x.detach()[:, 0].double()
        s, r = torch.sigmoid(v), torch.sigmoid(-v)  # r = 1 - s
        f, df = v * s, s * (1 + v * r)
        assert ((h.double() - f[:, None]).abs() <= 6 * u * f.abs()[:, None]).all()
        assert ((dx[:, cols - 1].double() - f).abs() <= 6 * u * f.abs()).all()
        assert ((dx[:, 0].double() - df).abs() <= u * (4 * s + f.abs() * (4 * s + 7 * r) + 2 * df.abs())).all()


@gpu
@pytest.mark.parametrize("act", ACTS)
def test_gradients_against_differences(dev, act):
    """Central differences of the forward pass itself, in fp32: of a sum over h weighted with dh, along random
    directions. The step's truncation error is of order eps^2 and the values' roundings are divided by eps: with
    eps = 2^-6 both are below 2^-10 of the sum over 30 x 24 terms."""
    offsets, R = segments([11, 0, 15], 4, dev)
    x, w = randn((R, 32), torch.float32, 1, dev), randn((3, 48, 32), torch.float32, 2, dev, 0.2)
    w2, dy = randn((3, 20, 24), torch.float32, 5, dev, 0.2), randn((R, 20), torch.float32, 3, dev)

    def forward(x, w, w2):
        return G.moe_linear_sorted(G.moe_gated_sorted(x, w, offsets, act), w2, offsets)

    leaves = [t.clone().requires_grad_(True) for t in (x, w, w2)]
    _, *gs = grads(forward, leaves, dy)
    eps = 2.0 ** -6
    for i, g in enumerate(gs):
        for seed in range(3):
            d = randn(g.shape, torch.float32, 10 + seed, dev)
            d /= d.norm()
            up, down = [x, w, w2], [x, w, w2]
            up[i], down[i] = up[i] + eps * d, down[i] - eps * d
            diff = ((forward(*up).double() - forward(*down).double()) * dy.double()).sum() / (2 * eps)
            assert abs(float(diff - (g.double() * d.double()).sum())) <= 2.0 ** -9 * float(g.norm()) + 2.0 ** -10


@gpu
def test_only_the_wanted_gradients(dev):
    offsets, R = segments([40, 90], 3, dev)
    x, w, dh = randn((R, 64), torch.bfloat16, 1, dev), randn((2, 48, 64), torch.bfloat16, 2, dev), randn((R, 24), torch.bfloat16, 3, dev)
    fn = lambda x, w: G.moe_gated_sorted(x, w, offsets)  # noqa: E731
    both = grads(fn, [x.clone().requires_grad_(True), w.clone().requires_grad_(True)], dh)
    assert torch.equal(grads(lambda x: fn(x, w), [x.clone().requires_grad_(True)], dh)[1], both[1])
    assert torch.equal(grads(lambda w: fn(x, w), [w.clone().requires_grad_(True)], dh)[1], both[2])
    with torch.no_grad():
        assert torch.equal(fn(x.clone().requires_grad_(True), w), both[0])
    lin = lambda x, w: G.moe_linear_sorted(x, w, offsets)  # noqa: E731
    dy = randn((R, 48), torch.bfloat16, 4, dev)
    both = grads(lin, [x.clone().requires_grad_(True), w.clone().requires_grad_(True)], dy)
    assert torch.equal(grads(lambda x: lin(x, w), [x.clone().requires_grad_(True)], dy)[1], both[1])
    assert torch.equal(grads(lambda w: lin(x, w), [w.clone().requires_grad_(True)], dy)[1], both[2])
    leaf = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(lin(leaf, w).sum(), leaf, create_graph=True)  # an expanded gradient
    assert torch.equal(g, grads(lambda x: lin(x, w), [leaf], torch.ones_like(dy))[1])
    with pytest.raises(RuntimeError):
        g.sum().backward()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("counts", [[2, 3], [150, 140]])
def test_what_is_in_no_segment_does_not_leak(dev, counts, bad, dtype):
    """Rows behind the last segment, in x and in the gradients, and an expert without rows: whatever they hold."""
    counts = counts + [0]
    offsets, R = segments(counts, 7, dev)
    end = R - 7
    x, w, dh = randn((R, 72), dtype, 1, dev), randn((3, 40, 72), dtype, 2, dev), randn((R, 20), dtype, 3, dev)
    fn = lambda x, w: G.moe_gated_sorted(x, w, offsets)  # noqa: E731
    lin = lambda x, w: G.moe_linear_sorted(x, w, offsets)  # noqa: E731
    dy = randn((R, 40), dtype, 4, dev)
    clean = [grads(f, [x.clone().requires_grad_(True), w.clone().requires_grad_(True)], d) for f, d in ((fn, dh), (lin, dy))]
    for t in (x, dh, dy):
        t[end:] = bad
    w[2] = bad
    for (f, d), want in zip(((fn, dh), (lin, dy)), clean):
        got = grads(f, [x.clone().requires_grad_(True), w.clone().requires_grad_(True)], d)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # a value that is not finite stays in its own row of y and dx
    x[1, 5] = bad
    got = grads(lin, [x.clone().requires_grad_(True), w.clone().requires_grad_(True)], dy)
    rest = torch.arange(R, device=dev) != 1
    assert torch.equal(got[0][rest], clean[1][0][rest]) and torch.equal(got[1], clean[1][1])
    assert not got[0][1].isfinite().any() and not got[2][0][:, 5].isfinite().all()
    assert torch.equal(got[2][1], clean[1][2][1])


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [6, 150])
def test_strides_and_alignment(dev, rows, dtype):
    N, K = 40, 144
    offsets, R = segments([rows, rows // 2], 3, dev)
    x, w, dy = ints((R, K), dtype, 1, dev), ints((2, N, K), dtype, 2, dev), ints((R, N), dtype, 3, dev)
    want = grads(lambda x, w: G.moe_linear_sorted(x, w, offsets), [x.requires_grad_(True), w.requires_grad_(True)], dy)
    x, w = x.detach(), w.detach()
    wide = torch.zeros((R, 2 * K + 3), dtype=dtype, device=dev)
    wide[:, 1:K + 1] = x
    flat = torch.zeros(2 * N * K + 1, dtype=dtype, device=dev)
    flat[1:] = w.reshape(-1)
    dwide = torch.zeros((R, N + 5), dtype=dtype, device=dev)
    dwide[:, 3:N + 3] = dy
    strided = torch.zeros(6, dtype=torch.int32, device=dev)
    strided[::2] = offsets
    for xx in (wide[:, 1:K + 1], x.t().contiguous().t()):
        for ww in (flat[1:].view(2, N, K), w.transpose(1, 2).contiguous().transpose(1, 2)):
            for dd in (dwide[:, 3:N + 3], dy.t().contiguous().t()):
                xx, ww = xx.detach().requires_grad_(True), ww.detach().requires_grad_(True)
                got = grads(lambda x, w: G.moe_linear_sorted(x, w, strided[::2]), [xx, ww], dd)
                assert all(torch.equal(a, b) for a, b in zip(got, want))
    # rows that end inside a word or a chunk, at strides that are multiples of 16 bytes; what lies behind them is not read
    for n in (K - 1, K - 3):
        xx, ww, dd = [torch.full((t.shape[0], t.shape[1] + 24), float("nan"), dtype=dtype, device=dev)[:, :m]
                      for t, m in ((x, n), (w.reshape(2 * N, K), n), (dy, N - 1))]
        xx.copy_(x[:, :n]), dd.copy_(dy[:, :N - 1])
        wp = w[:, :N - 1, :n].contiguous()
        got = grads(lambda x, w: G.moe_linear_sorted(x, w, offsets), [xx.requires_grad_(True), wp.requires_grad_(True)], dd)
        for a, b in zip(got, linear64(x[:, :n], wp.detach(), offsets, dy[:, :N - 1])):
            same(a, b)
    # the gate's gradient from a strided dh
    dh = dwide[:, 3:N // 2 + 3]
    fn = lambda x, w: G.moe_gated_sorted(x, w, offsets)  # noqa: E731
    a = grads(fn, [x.clone().requires_grad_(True), w.clone().requires_grad_(True)], dh)
    b = grads(fn, [wide[:, 1:K + 1].detach().requires_grad_(True), flat[1:].view(2, N, K).detach().requires_grad_(True)], dh.contiguous())
    for p, q in zip(a, b):
        assert (p.double() - q.double()).norm() <= half_step(dtype) * q.double().norm()
    one = x[:1].expand(R, K)
    assert torch.equal(G.moe_linear_sorted(one, w, offsets), G.moe_linear_sorted(one.contiguous(), w, offsets))


@gpu
@pytest.mark.parametrize("rows", [12, 600])
def test_offsets_outside_the_range(dev, rows):
    dtype, N, K = torch.bfloat16, 48, 64
    x, w, dy = ints((rows, K), dtype, 1, dev), ints((3, N, K), dtype, 2, dev), ints((rows, N), dtype, 3, dev)
    for off in ([-7, 3, rows - 5, rows + 100], [2, 4, 6, 8], [0, 0, 0, 0], [rows] * 4, [5, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1]):
        offsets = torch.tensor(off, dtype=torch.int32, device=dev)
        want = linear64(x, w, offsets, dy)
        got = grads(lambda x, w: G.moe_linear_sorted(x, w, offsets), [x.clone().requires_grad_(True), w.clone().requires_grad_(True)], dy)
        for a, b in zip(got, want):
            same(a, b)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_no_rows(dev, dtype):
    w, w1 = randn((2, 8, 16), dtype, 1, dev).requires_grad_(True), randn((8, 16), dtype, 1, dev).requires_grad_(True)
    x = torch.zeros((0, 16), device=dev, dtype=dtype).requires_grad_(True)
    offsets = torch.zeros(3, dtype=torch.int32, device=dev)
    for fn, m, n in ((lambda x, w: G.moe_gated_sorted(x, w, offsets), w, 4), (lambda x, w: G.moe_linear_sorted(x, w, offsets), w, 8),
                     (G.gated, w1, 4)):
        y, dx, dw = grads(fn, [x, m], torch.zeros((0, n), device=dev, dtype=dtype))
        assert y.shape == (0, n) and dx.shape == (0, 16) and dw.shape == m.shape and (dw == 0).all()


@gpu
def test_offsets_past_32_bits(dev):
    """Rows, weights and their gradients past 4 GiB; rows are cheap in columns, so that 64 bits check the last ones."""
    dtype, K = torch.bfloat16, 2048
    R = (1 << 31) // K + 500
    x = torch.zeros((R, K), dtype=dtype, device=dev)
    x[-400:] = ints((400, K), dtype, 1, dev)
    w, dy = ints((2, 8, K), dtype, 2, dev), torch.zeros((R, 8), dtype=dtype, device=dev)
    dy[-400:] = ints((400, 8), dtype, 3, dev)
    offsets = torch.tensor([0, R - 300, R], dtype=torch.int32, device=dev)
    got = grads(lambda x, w: G.moe_linear_sorted(x, w, offsets), [x.requires_grad_(True), w.requires_grad_(True)], dy)
    want = linear64(x.detach()[-400:], w.detach(), torch.tensor([0, 100, 400]), dy[-400:])
    same(got[0][-400:], want[0])
    same(got[1][-400:], want[1])
    same(got[2], want[2])
    assert (got[0][:-400] == 0).all() and (got[1][:1000] == 0).all()
    del x, got
    E, N = 600, 1800
    w = torch.zeros((E, N, K), dtype=dtype, device=dev)
    w[-1] = ints((N, K), dtype, 4, dev)
    for n in (5, 200):  # few rows, and tiles
        x, dy = ints((n, K), dtype, 5, dev).requires_grad_(True), ints((n, N), dtype, 6, dev)
        offsets = torch.zeros(E + 1, dtype=torch.int32, device=dev)
        offsets[-1] = n
        y, dx, dw = grads(lambda x, w: G.moe_linear_sorted(x, w, offsets), [x, w.requires_grad_(True)], dy)
        want = linear64(x.detach(), w.detach()[-1:], torch.tensor([0, n]), dy)
        same(y, want[0])
        same(dx, want[1])
        same(dw[-1:], want[2])
        assert not dw[:-1].any()


@gpu
def test_repeats_bit_for_bit(dev):
    offsets, R = segments([200, 3, 0, 511], 20, dev)
    x, w, dh = randn((R, 520), torch.bfloat16, 1, dev), randn((4, 600, 520), torch.bfloat16, 2, dev, 0.05), randn((R, 300), torch.bfloat16, 3, dev)
    step = lambda: grads(lambda x, w: G.moe_gated_sorted(x, w, offsets), [x.clone().requires_grad_(True), w.clone().requires_grad_(True)], dh)  # noqa: E731
    want = step()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(want, step()))


@gpu
@pytest.mark.parametrize("T", [3, 80])
def test_graph_and_streams(dev, T):
    """The whole layer, forward and backward: two captured graphs replayed between eager calls and on another stream."""
    k, E, K, N = 4, 8, 136, 96
    ids = [torch.randint(-1, E, (T, k), dtype=torch.int32, generator=torch.Generator().manual_seed(i)).to(dev) for i in range(2)]
    x = [randn((T, K), torch.bfloat16, i, dev).requires_grad_(True) for i in range(2)]
    w13, w2 = [randn(s, torch.bfloat16, 7, dev, 0.1).requires_grad_(True) for s in ((E, 2 * N, K), (E, K, N))]
    tw = torch.softmax(randn((T, k), torch.float32, 9, dev), 1)
    dy = randn((T, K), torch.bfloat16, 20, dev)

    def step(i):
        s = S.moe_sort(x[i], ids[i], E)
        y = S.moe_unsort(G.moe_linear_sorted(G.moe_gated_sorted(s.rows, w13, s.offsets), w2, s.offsets), tw, s.pos)
        return [y.detach(), *torch.autograd.grad(y, (x[i], w13, w2), dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in range(2):
            step(i)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(i))
        graphs.append(g)
    for turn in range(4):
        with torch.no_grad():
            for i in range(2):
                x[i].copy_(randn((T, K), torch.bfloat16, 30 + turn + i, dev))
                ids[i].copy_(torch.randint(-1, E, (T, k), dtype=torch.int32, generator=torch.Generator().manual_seed(turn + i)))
        for i in ((0, 1) if turn % 2 else (1, 0)):
            graphs[i].replay()
        for i in range(2):
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs[i], step(i)))
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = step(0)
    b = step(1)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(a, step(0))) and all(torch.equal(p, q) for p, q in zip(b, step(1)))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [9, 300])
def test_a_trained_layer(dev, T, dtype):
    """A run as it would be used: sort, gate, down products, back with weights, and every gradient, against 64 bits. Each
    of the stages rounds once, forward (gate, down, sum) and back (rows of the sum's gradient, the down products', the projections', the
    rows', the sum over routes); each at most half a step, so the distance is below the number of roundings before an output."""
    k, E, K, N = 3, 7, 128, 72
    g = torch.Generator().manual_seed(5)
    ids = torch.stack([torch.randperm(E + 2, generator=g)[:k] - 2 for _ in range(T)]).to(torch.int32).to(dev)
    x = randn((T, K), dtype, 1, dev).requires_grad_(True)
    w13 = randn((E, 2 * N, K), dtype, 2, dev, 0.1).requires_grad_(True)
    w2 = randn((E, K, N), dtype, 3, dev, 0.1).requires_grad_(True)
    tw = torch.softmax(randn((T, k), torch.float32, 4, dev), 1).requires_grad_(True)
    dy = randn((T, K), dtype, 6, dev)
    s = S.moe_sort(x, ids, E)
    y = S.moe_unsort(G.moe_linear_sorted(G.moe_gated_sorted(s.rows, w13, s.offsets), w2, s.offsets), tw, s.pos)
    got = [y.detach(), *torch.autograd.grad(y, (x, w13, w2, tw), dy)]
    leaves = [t.detach().double().requires_grad_(True) for t in (x, w13, w2, tw)]
    X, A, B, W = leaves
    parts = []
    for t in range(T):
        total = torch.zeros(K, dtype=torch.float64, device=dev)
        for j in range(k):
            e = int(ids[t, j])
            if e >= 0:
                v = A[e] @ X[t]
                total = total + W[t, j] * (B[e] @ (v[:N] * torch.sigmoid(v[:N]) * v[N:]))
        parts.append(total)
    ref = torch.stack(parts)
    want = [ref.detach(), *torch.autograd.grad(ref, leaves, dy.double())]
    for a, b, n in zip(got, want, (3, 6, 5, 4, 3)):
        assert (a.double() - b).norm() <= (n * half_step(dtype) + 2.0 ** -17) * b.norm(), n


@gpu
@pytest.mark.parametrize("how", ["aot_eager", "checkpoint"])
def test_compiled_and_checkpointed(dev, how):
    offsets, R = segments([40, 90], 3, dev)
    x, w, dh = randn((R, 64), torch.bfloat16, 1, dev), randn((2, 48, 64), torch.bfloat16, 2, dev), randn((R, 24), torch.bfloat16, 3, dev)
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    forward = lambda x, w: G.moe_gated_sorted(x * 1, w, offsets) + 1  # noqa: E731
    want = grads(forward, leaves, dh)
    if how == "checkpoint":
        from torch.utils.checkpoint import checkpoint

        other = lambda x, w: checkpoint(forward, x, w, use_reentrant=False)  # noqa: E731
    else:
        torch._dynamo.reset()
        other = torch.compile(forward, backend=how)
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(want, grads(other, leaves, dh)))


@gpu
def test_threads(dev):
    """Calls of several host threads, each on a stream of its own, with refusals between them."""
    import threading

    offsets, R = segments([40, 90], 3, dev)
    x, w, dh = randn((R, 64), torch.bfloat16, 1, dev), randn((2, 48, 64), torch.bfloat16, 2, dev), randn((R, 24), torch.bfloat16, 3, dev)
    step = lambda: grads(lambda x, w: G.moe_gated_sorted(x, w, offsets), [x.clone().requires_grad_(True), w.clone().requires_grad_(True)], dh)  # noqa: E731
    want, wrong = step(), []
    torch.cuda.synchronize()

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for n in range(10):
                    got = step()
                    stream.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(want, got)):
                        wrong.append((i, n))
                    with pytest.raises(ValueError, match="act 'tanh'"):
                        G.gated(x, w[0], "tanh")
        except BaseException as e:  # a thread's failure is the test's
            wrong.append((i, repr(e)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong


# ---------------------------------------------------------------- refusals (no GPU)

def test_refusals():
    x, w, off = torch.zeros(2, 64), torch.zeros(6, 64), torch.zeros(2, dtype=torch.int32)
    for args, error in [((x.double(), w), TypeError), ((x, w.half()), TypeError), ((x[0], w), ValueError), ((x[:, :63], w), ValueError),
                        ((x, w[:5]), ValueError), ((x, w[:0]), ValueError), ((x, w[None]), ValueError), ((x, w, "tanh"), ValueError),
                        ((x[:, :0], w[:, :0]), ValueError), ((x, w), ValueError)]:  # the last: not on the GPU
        with pytest.raises(error, match="gated"):
            G.gated(*args)
    we = w[None]
    for fn in (G.moe_gated_sorted, G.moe_linear_sorted):
        for args, error in [((x, we, off.long()), TypeError), ((x, we, off[:1]), ValueError), ((x, we, off[None]), ValueError),
                            ((x, w, off), ValueError), ((x, we[:0], off[:1]), ValueError), ((x, we, None), TypeError),
                            ((x, torch.zeros(2049, 2, 64), torch.zeros(2050, dtype=torch.int32)), ValueError), ((x, we, off), ValueError)]:
            with pytest.raises(error, match=fn.__name__):
                fn(*args)


def test_c_refusals():
    """Argument errors of the entry points come before any device work (the pointers are never read)."""
    L = _lib.lib()
    p = 4096

    def gated(x=p, dt=2, xs=64, K=64, w=p, N=8, E=4, off=p, R=2, act=0, h=p, sums=0, ws=p, n=1 << 50):
        return L.ktmi_gated(x, dt, xs, K, w, N, E, off, R, act, h, sums, ws, n, 0)

    for kw in [dict(dt=3), dict(K=0), dict(N=0), dict(R=-1), dict(x=0), dict(w=0), dict(h=0), dict(x=p + 1), dict(w=p + 1), dict(h=p + 1),
               dict(sums=p + 4), dict(xs=63), dict(K=1 << 25, xs=1 << 25), dict(R=1 << 31), dict(E=0), dict(E=2049), dict(off=0),
               dict(act=2), dict(act=-1), dict(N=(1 << 23) + 1)]:
        assert gated(**kw) == -1 and b"gated" in L.ktmi_last_error(), kw
    assert gated(R=0) == 0

    def grad(sums=p, dh=p, dt=2, st=8, N=8, R=2, act=0, out=p):
        return L.ktmi_gated_grad(sums, dh, dt, st, N, R, act, out, 0)

    for kw in [dict(sums=0), dict(dh=0), dict(dt=7), dict(st=7), dict(N=0), dict(R=-1), dict(act=2), dict(out=0), dict(sums=p + 4)]:
        assert grad(**kw) == -1 and b"gated_grad" in L.ktmi_last_error(), kw
    assert grad(R=0) == 0

    def linear(x=p, dt=2, xs=64, K=64, w=p, N=8, E=4, off=p, R=2, y=p, ws=p, n=1 << 50):
        return L.ktmi_linear(x, dt, xs, K, w, N, E, off, R, y, ws, n, 0)

    def grad_x(x=p, dt=2, xs=64, K=8, w=p, N=64, E=4, off=p, R=2, y=p, ws=p, n=1 << 50):
        return L.ktmi_linear_grad_x(x, dt, xs, N, w, K, E, off, R, y, ws, n, 0)

    def grad_w(x=p, dt=2, xs=64, K=64, N=64, E=4, off=p, R=2, y=p, dy=p, ds=64, ws=p, n=1 << 50):
        return L.ktmi_linear_grad_w(dy, dt, ds, N, x, xs, K, E, off, R, y, ws, n, 0)

    for fn, name in ((linear, b"linear"), (grad_x, b"linear_grad_x"), (grad_w, b"linear_grad_w")):
        for kw in [dict(dt=3), dict(K=0), dict(N=0), dict(R=-1), dict(x=0), dict(y=0), dict(x=p + 1), dict(y=p + 1), dict(xs=63),
                   dict(R=1 << 31), dict(E=0), dict(E=2049), dict(off=0)]:
            assert fn(**kw) == -1 and name in L.ktmi_last_error(), (name, kw)
        if fn is not grad_w:  # an expert without rows has a gradient too
            assert fn(R=0) == 0
    assert grad_w(dy=0) == -1 and grad_w(ds=63) == -1 and grad_w(R=0, y=0) == -1
    # workspaces: what splits of a long k ask for
    need = L.ktmi_linear_workspace(_lib.PROD_LINEAR, 2, 64, 8192, 1, 70)
    assert need > 0 and linear(K=8192, xs=8192, N=64, E=1, R=70, n=need - 1) == -4 and linear(K=8192, xs=8192, N=64, E=1, R=70, ws=0) == -4
    assert linear(K=8192, xs=8192, N=64, E=1, R=70, ws=p + 4) == -4
    assert L.ktmi_linear_workspace(_lib.PROD_LINEAR, 2, 64, 64, 1, 70) == 0 and L.ktmi_linear_workspace(9, 2, 64, 8192, 1, 70) == 0
    # grids past 2^32 threads
    assert linear(E=2048, R=1 << 30, N=1 << 24) == -1 and b"grid" in L.ktmi_last_error()
    assert grad_x(E=2048, R=1 << 30, K=1 << 24) == -1 and b"grid" in L.ktmi_last_error()
    assert grad_w(E=2048, R=1 << 30, N=1 << 24, ds=1 << 24, K=1 << 20, xs=1 << 20) == -1 and b"grid" in L.ktmi_last_error()


def record_calls(dev):
    x, w = torch.ones((4, 16), device=dev), torch.ones((2, 8, 16), device=dev)
    off = torch.tensor([0, 2, 4], dtype=torch.int32, device=dev)
    return {"gated": (lambda x, w: G.gated(x, w), (x, w[0])), "moe_gated_sorted": (lambda x, w: G.moe_gated_sorted(x, w, off), (x, w)),
            "moe_linear_sorted": (lambda x, w: G.moe_linear_sorted(x, w, off), (x, w))}


NAMES = ["gated", "moe_gated_sorted", "moe_linear_sorted"]


@pytest.mark.filterwarnings("ignore:Converting a tensor")
@pytest.mark.parametrize("name", NAMES)
def test_records_without_the_kernels_are_refused(monkeypatch, name):
    monkeypatch.setattr(G, "_check_gpu", lambda *a: None)
    check_refused_records(name, *record_calls("cpu")[name])


@gpu
@pytest.mark.filterwarnings("ignore:Converting a tensor")
@pytest.mark.parametrize("name", NAMES)
def test_records_without_the_kernels_are_refused_on_the_gpu(dev, name):
    check_refused_records(name, *record_calls(dev)[name])


def test_tensors_without_memory_are_refused():
    """Where the library takes a null pointer for an argument left out, a wrapper's must not pass for one."""
    x, w, dy = torch.ones(4, 16), torch.ones(1, 8, 16), torch.ones(4, 8)
    off = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(TypeError, match="moe_gated_sorted: a Wrapped"):
        G._launch_gated(0, "moe_gated_sorted", x, w, wrapped(off), 0, False)
    with pytest.raises(TypeError, match="moe_linear_sorted: a Wrapped"):
        G._launch_linear(0, "moe_linear_sorted", x, w, wrapped(off))
    for d, o in ((wrapped(dy), off), (dy, wrapped(off))):
        with pytest.raises(TypeError, match="a Wrapped"):
            G._launch_grads(0, "gradient", d, x, w, o, True, True)
