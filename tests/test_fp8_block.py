"""Products in 8-bit floating point with block scales (kt_fp8_block).

Most cases use integers for x with one 448 (times a power of two) in each row's block, so that the quantised
codes are x itself, small integers for w and powers of two for the scales: every product and partial sum is
exact in fp32 whatever the order of the sums, and no term is more than 2^13 times another, so the
outputs have to be equal bit for bit. Others use general values against 64 bits."""
import ctypes
import math

import pytest
import torch

import kt_prefill_lend_amd.kt_fp8_block as F
from helpers import check_refused_records, wrapped
from kt_prefill_lend_amd import _lib

gpu = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
E4M3 = torch.float8_e4m3fn


def blocks_of(n):
    return -(-n // 128)


def make_w(lead, N, K, seed, dev, exact=True):
    g = torch.Generator().manual_seed(seed)
    if exact:
        w = torch.randint(-3, 4, (*lead, N, K), generator=g).float()
        s = 2.0 ** torch.randint(-6, -3, (*lead, blocks_of(N), blocks_of(K)), generator=g).float()
    else:
        w = (torch.randn((*lead, N, K), generator=g) * 110).clamp(-448, 448)
        s = torch.rand((*lead, blocks_of(N), blocks_of(K)), generator=g) * 2e-4 + 1e-4
    return w.to(E4M3).to(dev), s.to(dev)


def make_x(T, K, dtype, seed, dev, exact=True):
    g = torch.Generator().manual_seed(seed)
    if not exact:
        return torch.randn((T, K), generator=g).to(dtype).to(dev)
    x = torch.randint(-2, 3, (T, K), generator=g).float()
    for k0 in range(0, K, 128):  # each row's block its own power of two
        at = torch.randint(0, min(128, K - k0), (T,), generator=g)
        x[torch.arange(T), k0 + at] = 448.0 * (1 - 2 * torch.randint(0, 2, (T,), generator=g).float())
        x[:, k0:k0 + 128] *= 2.0 ** torch.randint(-2, 2, (T, 1), generator=g).float()
    return x.to(dtype).to(dev)


def e4m3(v):
    """fp32 values rounded to e4m3's, in 64 bits."""
    v = v.double()
    step = torch.ldexp(torch.ones_like(v), (torch.frexp(v).exponent - 1).clamp_min(-6) - 3)
    return torch.round(v / step) * step


def quantised(x):
    """x as its codes and scales stand for it, in 64 bits."""
    out = x.double()
    for k0 in range(0, x.shape[1], 128):
        v = out[:, k0:k0 + 128].clone()
        a = v.abs().amax(1, keepdim=True).clamp_min(2.0 ** -116)
        out[:, k0:k0 + 128] = e4m3((v * (448.0 / a).float().double()).float()) * (a / 448.0).float().double()
    return out


def matrix(w, s):
    N, K = w.shape[-2:]
    at_n, at_k = torch.arange(N, device=w.device) // 128, torch.arange(K, device=w.device) // 128
    return w.double() * s.double()[..., at_n, :][..., at_k]


def routed(x, w, s, ids, top_k):
    """y [R, N] and the sums of the terms' sizes, in 64 bits."""
    xq = quantised(x)
    y = torch.zeros((ids.numel(), w.shape[1]), dtype=torch.float64, device=x.device)
    size = torch.zeros_like(y)
    for e in range(w.shape[0]):
        r = (ids == e).nonzero().reshape(-1)
        if r.numel():
            m = matrix(w[e], s[e])
            y[r] = xq[r // top_k] @ m.t()
            size[r] = xq[r // top_k].abs() @ m.abs().t()
    return y, size


def same(got, want64):
    assert torch.equal(got, want64.float().to(got.dtype)), (got.double() - want64).abs().max()


# tokens, N, K: few rows, then tiles; rows of w at any alignment; ends inside a block, a chunk, a tile
DENSE = [(1, 1, 1), (1, 5, 127), (2, 17, 128), (3, 130, 129), (1, 515, 1111), (7, 64, 1000), (16, 128, 256), (17, 96, 384),
         (33, 20, 2080), (64, 300, 130), (65, 1, 1), (65, 129, 128), (66, 515, 1111), (100, 260, 1000), (129, 128, 144),
         (255, 257, 640), (300, 600, 272), (1100, 4200, 256), (1000, 4097, 400), (513, 8192, 130),
         # few rows by many: more rows of w a wave, short rows
         (3, 8200, 2100), (16, 16500, 2050), (2, 8200, 256), (1, 33000, 2176)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,N,K", DENSE)
def test_dense_exact(dev, T, N, K, dtype):
    w, s = make_w((), N, K, N + K, dev)
    x = make_x(T, K, dtype, T, dev)
    assert torch.equal(quantised(x), x.double())
    same(F.fp8_linear(x, w, s), x.double() @ matrix(w, s).t())


# routed or not, rows of x, top_k, experts, N, K -> the tile, and whether blocks share its k
SHAPES = [(0, 20, 1, 1, 40, 200, (0, 0), False), (1, 20, 2, 3, 40, 200, (0, 0), False), (0, 100, 1, 1, 300, 256, (64, 128), False),
          (0, 256, 1, 1, 12300, 256, (128, 128), False), (0, 256, 1, 1, 12300, 200, (128, 128), False),
          (0, 1000, 1, 1, 12300, 256, (256, 256), False), (0, 1000, 1, 1, 12300, 144, (256, 256), False),
          (0, 100, 1, 1, 130, 8192, (64, 128), True), (0, 90, 1, 1, 131, 8197, (64, 128), True),
          (1, 90, 2, 2, 70, 8192, (64, 128), True), (1, 300, 4, 2, 12300, 128, (256, 256), False)]


def test_kernel_shapes_are_all_reached():
    k = _lib.ktmi_prod_kernel()
    for ids, T, top_k, E, N, K, tile, split in SHAPES:
        assert _lib.lib().ktmi_fp8_kernel_of(ids, N, K, E, top_k, T, ctypes.byref(k)) == 0
        assert ((k.tile_rows, k.tile_cols), k.splits > 1) == (tile, split), (ids, T, top_k, E, N, K, k.tile_rows, k.tile_cols, k.splits)
    for args in [(0, 0, 8, 1, 1, 1), (0, 8, 0, 1, 1, 1), (0, 8, 8, 0, 1, 1), (0, 8, 8, 1, 0, 1), (0, 8, 8, 1, 1, 0)]:
        assert _lib.lib().ktmi_fp8_kernel_of(*args, ctypes.byref(k)) == -1
    assert _lib.lib().ktmi_fp8_kernel_of(0, 8, 8, 1, 1, 1, None) == -1


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ids,T,top_k,E,N,K,tile,split", SHAPES)
def test_shapes_exact(dev, ids, T, top_k, E, N, K, tile, split, dtype):
    w, s = make_w((E,), N, K, N + K, dev)
    x = make_x(T, K, dtype, T, dev)
    if ids:
        r = routes(T, top_k, E, 0.1, T, dev)
        same(F.moe_fp8_vec(x, w, s, r, top_k), routed(x, w, s, r, top_k)[0])
    else:
        same(F.fp8_linear(x, w[0], s[0]), x.double() @ matrix(w[0], s[0]).t())


# columns that are no multiple of 16, whose codes go through registers: no tiles of 256 rows there
RAGGED = [(0, 1000, 1, 1, 12300, 132, (128, 128)), (0, 1000, 1, 1, 12300, 130, (128, 128)), (0, 256, 1, 1, 12300, 137, (128, 128)),
          (1, 300, 4, 2, 12300, 132, (128, 128)), (0, 100, 1, 1, 300, 132, (64, 128)), (0, 20, 1, 1, 300, 132, (0, 0))]


def test_kernels_of_ragged_columns():
    k = _lib.ktmi_prod_kernel()
    for ids, T, top_k, E, N, K, tile in RAGGED:
        assert _lib.lib().ktmi_fp8_kernel_of(ids, N, K, E, top_k, T, ctypes.byref(k)) == 0
        assert (k.tile_rows, k.tile_cols, k.splits) == (*tile, 1), (ids, T, top_k, E, N, K, k.tile_rows, k.tile_cols, k.splits)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ids,T,top_k,E,N,K,tile", RAGGED)
def test_ragged_columns_exact(dev, ids, T, top_k, E, N, K, tile, dtype):
    test_shapes_exact(dev, ids, T, top_k, E, N, K, tile, False, dtype)


def routes(T, k, E, cold, seed, dev):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, E, (T * k,), generator=g, dtype=torch.int32)
    ids[torch.rand(T * k, generator=g) < cold] = -1
    return ids.to(dev)


ROUTED = [(1, 1, 1, 5, 64, 0.0), (1, 8, 40, 64, 256, 0.3), (5, 3, 7, 72, 130, 0.2), (64, 1, 1, 33, 160, 0.0), (21, 3, 2, 48, 384, 0.1),
          (40, 8, 300, 16, 96, 0.0), (6, 2, 4, 20, 77, 1.0), (64, 8, 3, 130, 288, 0.1), (70, 4, 2, 200, 1000, 0.2),
          (600, 2, 3, 300, 272, 0.3), (300, 4, 64, 40, 144, 0.0), (90, 1, 1, 140, 515, 0.5),
          (60, 1, 2, 17000, 300, 0.1), (20, 3, 2, 17000, 2100, 0.1)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,E,N,K,cold", ROUTED)
def test_routed_exact(dev, T, k, E, N, K, cold, dtype):
    w, s = make_w((E,), N, K, N + K, dev)
    x, ids = make_x(T, K, dtype, T, dev), routes(T, k, E, cold, T, dev)
    y = F.moe_fp8_vec(x, w, s, ids, k)
    same(y, routed(x, w, s, ids, k)[0])
    assert (y[ids < 0] == 0).all()


SORTED = [([1], 0, 5, 64), ([0, 3, 0, 0, 17, 1, 0], 4, 72, 384), ([0, 0, 0], 7, 9, 96), ([70, 0, 33], 0, 40, 130),
          ([5] * 60, 3, 16, 96), ([300, 2], 1, 24, 256), ([0] * 500 + [2, 1], 2, 33, 64), ([1] * 2048, 5, 3, 16),
          ([129, 0, 257, 64], 130, 300, 144), ([700, 500, 1], 300, 4100, 128), ([90, 400], 3, 129, 515)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts,tail,N,K", SORTED)
def test_sorted_exact(dev, counts, tail, N, K, dtype):
    E, R = len(counts), sum(counts) + tail
    w, s = make_w((E,), N, K, N + K, dev)
    ids = torch.repeat_interleave(torch.arange(E + 1), torch.tensor(counts + [tail])).to(dev)
    offsets = torch.tensor([0] + counts).cumsum(0).to(torch.int32).to(dev)
    x = make_x(R, K, dtype, 5, dev)
    y = F.moe_fp8_sorted(x, w, s, offsets)
    same(y, routed(x, w, s, ids, 1)[0])
    assert (y[R - tail:] == 0).all()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,N,K", [(1, 300, 2048), (5, 129, 1000), (20, 64, 1111), (50, 100, 512), (200, 260, 2048), (300, 4200, 515)])
def test_general_values(dev, T, N, K, dtype):
    """Against 64 bits: the codes are the definition's, so what is left are the sums' roundings. In fp32 each of the K
    additions and two products by a scale is off by 2^-24 of a partial sum at most, as a whole by
    3 sqrt(2 K) 2^-24 for roundings of independent sign of partial sums up to three times the final ones'. Of y in 16 bits the
    matrix cores add 8-bit products with about 16 bits below the largest of an instruction: 1.5e-5 of the sums' norm
    measured for normal values, bounded here by 2^-14, and each by 2^-12 of the terms' size."""
    w, s = make_w((), N, K, 3, dev, exact=False)
    x = make_x(T, K, dtype, 4, dev, exact=False)
    xq, m = quantised(x), matrix(w, s)
    want, size = xq @ m.t(), xq.abs() @ m.abs().t()
    got = F.fp8_linear(x, w, s).double()
    u = torch.finfo(dtype).eps / 2
    cores = 0.0 if dtype == torch.float32 else 1.0
    each = (K + 4) * 2.0 ** -24 + cores * 2.0 ** -12
    whole = 3 * math.sqrt(2 * K) * 2.0 ** -24 + cores * 2.0 ** -14
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0  # half a step below f16's normal numbers
    assert ((got - want).abs() <= u * want.abs() + (1 + u) * each * size + tiny).all()
    assert (got - want).norm() <= (u + whole) * want.norm()


@gpu
@pytest.mark.parametrize("T", [1, 100])
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_code(dev, T, dtype):
    """Each finite code of w against each of x, one product an output: exact, the last rounding aside."""
    K = 128
    codes = torch.arange(256, dtype=torch.uint8)
    w = torch.zeros((256, K), dtype=torch.uint8)
    w[:, 1] = codes
    x = torch.zeros((max(T, 1), K))
    values = codes.view(E4M3).float()
    values = values[~values.isnan()]
    x[:, 0] = 448
    x[:, 1] = values[torch.arange(x.shape[0]) * 53 % values.numel()]
    finite = ~codes.view(E4M3).float().isnan()
    for _ in range(1 if T > 1 else values.numel()):
        y = F.fp8_linear(x.to(dtype).to(dev), w.to(dev), torch.ones((2, 1), device=dev)).cpu()
        want = x[:, 1:2].double() * codes.view(E4M3).float().double()
        # f16 has e4m3's values, and their products below 65504 to 2^-11
        assert torch.equal(y[:, finite], want[:, finite].float().to(dtype))
        assert y[:, ~finite].isnan().all()
        x = x.clone()
        x[:, 1] = values[int((values == x[0, 1]).nonzero()[0, 0] + 1) % values.numel()]


@gpu
@pytest.mark.parametrize("T", [1, 17, 100])
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_pair_of_codes(dev, T, dtype):
    """All 254 finite codes of x, by their bytes, against all of w: one product an output, exact, the last rounding aside. (The
    walk of test_every_code finds its place by value: at -0 it finds 0, and starts over.)"""
    K = 128
    codes = torch.arange(256, dtype=torch.uint8)
    value = codes.view(E4M3).float()
    finite = ~value.isnan()
    of_x = codes[finite]
    w = torch.zeros((256, K), dtype=torch.uint8)
    w[:, 1] = codes
    w, scales, done = w.to(dev), torch.ones((2, 1), device=dev), []
    for i in range(-(-of_x.numel() // T)):
        c = of_x[(torch.arange(T) * 53 + i * T * 53) % of_x.numel()]
        x = torch.zeros((T, K))
        x[:, 0], x[:, 1] = 448, c.view(E4M3).float()
        y = F.fp8_linear(x.to(dtype).to(dev), w, scales).cpu()
        want = c.view(E4M3).double()[:, None] * value.double()
        assert torch.equal(y[:, finite], want[:, finite].float().to(dtype))
        assert y[:, ~finite].isnan().all()
        done.append(c)
    assert torch.cat(done).unique().numel() == 254


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [3, 100])
def test_ends_of_the_range(dev, T, dtype):
    """Rows of zeros, of values below 2^-116, of a type's largest; one block large and the next small. The two scales' product
    is rounded to fp32: below 2^-126 by at most 2^-150, half a step of its subnormal numbers, and the codes that it is a factor of
    sum to at most K 448^2."""
    K, N = 256, 40
    f = torch.finfo(dtype)
    w, s = make_w((), N, K, 3, dev, exact=False)
    x = make_x(T, K, dtype, 4, dev, exact=False)
    x[0] = 0
    x[1, :128] *= f.max / 64
    x[1, 128:] *= f.tiny * 8
    x[2] = f.tiny / 2 if dtype != torch.float16 else f.tiny
    got = F.fp8_linear(x, w, s * 2.0 ** -20).double()
    m = matrix(w, s * 2.0 ** -20)
    want, size = quantised(x) @ m.t(), quantised(x).abs() @ m.abs().t()
    assert (got[0] == 0).all() and got.isfinite().all()
    u = torch.finfo(dtype).eps / 2
    tiny = f.tiny * f.eps / 2 + (2.0 ** -149 if dtype != torch.float16 else 0)  # half a step of the type's smallest
    scales = 2.0 ** -150 * K * 448 ** 2
    assert ((got - want).abs() <= u * want.abs() + 2.0 ** -11 * size + tiny + scales).all()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [3, 90])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_scales_whose_product_is_past_the_range(dev, T, sign, dtype):
    """A block of the type's largest values by a scale of 2^125: their product is no fp32 number, and a row of w with zeros there
    adds 0 all the same, so that the other blocks' sums are left, bit for bit. One with codes there is infinite; a scale
    that is not finite makes its rows so."""
    N, K = 300, 640
    w, s = make_w((), N, K, 3, dev)
    x = make_x(T, K, dtype, 4, dev)
    want = x.double()
    want[:, 128:256] = 0
    want = want @ matrix(w, s).t()
    x[:, 128:256] = 0
    x[:, 130] = torch.finfo(dtype).max
    s[:, 1] = sign * 2.0 ** 125
    w = w.view(torch.uint8)
    w[:, 130] = 0
    got = F.fp8_linear(x, w, s)
    same(got, want)
    ids = (torch.arange(T, device=dev) % 2).to(torch.int32)
    assert torch.equal(F.moe_fp8_vec(x, torch.stack([w, w]), torch.stack([s, s]), ids, 1), got)
    w[7, 130] = torch.tensor(448.0).to(E4M3).view(torch.uint8)
    y = F.fp8_linear(x, w, s)
    assert (y[:, 7] == sign * math.inf).all()
    rest = torch.arange(N, device=dev) != 7
    assert torch.equal(y[:, rest], got[:, rest])
    w[:, 130] = w[7, 130]
    for bad in (math.inf, -math.inf, math.nan):
        s[1, 1] = bad
        y = F.fp8_linear(x, w, s)
        assert y[:, 128:256].isnan().all() if math.isnan(bad) else (y[:, 128:256] == bad).all()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [5, 90])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_not_finite(dev, T, dtype, bad):
    """A value of x that is not finite makes its own row NaN and leaves the others' bits alone."""
    w, s = make_w((), 40, 384, 3, dev, exact=False)
    x = make_x(T, 384, dtype, 4, dev, exact=False)
    clean = F.fp8_linear(x, w, s)
    x[2, 77] = bad
    got = F.fp8_linear(x, w, s)
    rest = torch.arange(T, device=dev) != 2
    assert got[2].isnan().all() and torch.equal(got[rest], clean[rest])
    y = F.moe_fp8_sorted(x, w[None], s[None], torch.tensor([0, 2], dtype=torch.int32, device=dev))
    assert torch.equal(y[:2], clean[:2]) and (y[2:] == 0).all()  # rows of no expert, whatever they hold


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [3, 80])
def test_strides_and_alignment(dev, T, dtype):
    N, K = 140, 272
    w, s = make_w((2,), N, K, 3, dev)
    x = make_x(T, K, dtype, 4, dev)
    off = torch.tensor([0, T // 2, T], dtype=torch.int32, device=dev)
    want = F.moe_fp8_sorted(x, w, s, off)
    wide = torch.zeros((T, 2 * K + 3), dtype=dtype, device=dev)
    wide[:, 1:K + 1] = x
    flat = torch.zeros(2 * N * K + 1, dtype=torch.uint8, device=dev)
    flat[1:] = w.view(torch.uint8).reshape(-1)
    odd = flat[1:].view(2, N, K)  # rows of codes at odd addresses
    wt = w.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2)
    st = s.transpose(1, 2).contiguous().transpose(1, 2)
    for xx in (wide[:, 1:K + 1], x.t().contiguous().t(), x):
        for ww in (w, w.view(torch.uint8), odd, wt, odd.view(E4M3)):
            assert torch.equal(F.moe_fp8_sorted(xx, ww, st, off), want)
    ids = torch.zeros((T, 2), dtype=torch.int32, device=dev)
    assert torch.equal(F.moe_fp8_vec(wide[:, 1:K + 1], odd, s, ids[:, 0], 1), F.fp8_linear(x, w[0], s[0]))
    assert torch.equal(F.fp8_linear(x[:1].expand(T, K), w[0], s[0])[T - 1], F.fp8_linear(x[:1].expand(T, K), w[0], s[0])[0])


@gpu
@pytest.mark.parametrize("rows", [12, 900])
def test_ids_and_offsets_outside_the_range(dev, rows):
    N, K, E = 40, 272, 3
    w, s = make_w((E,), N, K, 3, dev)
    x = make_x(rows, K, torch.bfloat16, 4, dev)
    g = torch.Generator().manual_seed(1)
    ids = torch.tensor([-2 ** 31, -5, -1, 0, 1, 2, 3, 4, 1000, 2 ** 31 - 1], dtype=torch.int32)
    ids = ids[torch.randint(0, 10, (rows,), generator=g)].to(dev)
    y = F.moe_fp8_vec(x, w, s, ids, 1)
    same(y, routed(x, w, s, ids, 1)[0])
    off = torch.tensor([-7, 3, rows - 5, rows + 100], dtype=torch.int32, device=dev)
    at = torch.arange(rows, device=dev)
    ids = torch.where(at < 3, 0, torch.where(at < rows - 5, 1, 2))
    same(F.moe_fp8_sorted(x, w, s, off), routed(x, w, s, ids, 1)[0])
    off = torch.tensor([2, 4, 6, 8], dtype=torch.int32, device=dev)  # rows in front of the first segment too
    ids = torch.where((at < 2) | (at >= 8), -1, (at - 2) // 2)
    same(F.moe_fp8_sorted(x, w, s, off), routed(x, w, s, ids, 1)[0])


@gpu
def test_no_rows(dev):
    w, s = make_w((2,), 8, 64, 1, dev)
    x = torch.zeros((0, 64), device=dev, dtype=torch.bfloat16)
    ids = torch.zeros(0, dtype=torch.int32, device=dev)
    assert F.fp8_linear(x, w[0], s[0]).shape == (0, 8)
    assert F.moe_fp8_vec(x, w, s, ids, 4).shape == (0, 8)
    assert F.moe_fp8_sorted(x, w, s, torch.zeros(3, dtype=torch.int32, device=dev)).shape == (0, 8)


@gpu
def test_codes_past_32_bits(dev):
    """Experts whose codes start past 4 GiB, for few rows and for tiles; rows of y past 4 GiB."""
    E, N, K = 530, 2048, 4096
    w = torch.zeros((E, N, K), dtype=torch.uint8, device=dev)
    s = torch.ones((E, N // 128, K // 128), device=dev)
    one = int(torch.tensor(1.0).to(E4M3).view(torch.uint8))
    w[E - 1, :, 7] = one
    w[E - 1, N - 1, K - 1] = one
    for rows in (3, E * 70):
        x = torch.zeros((rows, K), dtype=torch.bfloat16, device=dev)
        x[:, 7] = 448
        x[:, K - 1] = 448
        off = torch.zeros(E + 1, dtype=torch.int32, device=dev)
        off[E] = rows
        y = F.moe_fp8_sorted(x, w, s, off)
        assert (y[:, :N - 1] == 448).all() and (y[:, N - 1] == 896).all()
    del x, y
    rows = (1 << 31) // 2048 + 300
    x = torch.zeros((rows, 128), dtype=torch.bfloat16, device=dev)
    x[-1, 3] = 448
    w = torch.full((2048, 128), one, dtype=torch.uint8, device=dev)
    y = F.fp8_linear(x, w, torch.ones((16, 1), device=dev))
    assert (y[-1] == 448).all() and (y[:-1] == 0).all()


@gpu
@pytest.mark.parametrize("K", [(1 << 23) + 128, 1 << 24])
def test_longest_rows(dev, K):
    """Tiles of rows whose codes lie up to 2 GiB apart."""
    T, N = 140, 3
    x = torch.zeros((T, K), dtype=torch.bfloat16, device=dev)
    w = torch.zeros((N, K), dtype=torch.uint8, device=dev)
    w[:, K - 1] = w[:, 3] = int(torch.tensor(1.0).to(E4M3).view(torch.uint8))
    x[:, K - 1], x[::2, 3] = 448, 448
    y = F.fp8_linear(x, w, torch.ones((1, K // 128), device=dev))
    assert (y[::2] == 896).all() and (y[1::2] == 448).all()


@gpu
def test_routed_tokens_past_32_bits_of_codes(dev):
    """More than 2 GiB of quantised tokens: slices of them, the last one short."""
    K, N, E, T = 1 << 17, 16, 2, (1 << 14) + 70
    w = torch.zeros((E, N, K), device=dev).to(E4M3)
    w[0, :, 5], w[1, :, K - 1] = 1, 2
    x = torch.zeros((T, K), dtype=torch.bfloat16, device=dev)
    x[:, 5], x[:, K - 1] = 448, 448
    x[-3:] *= -1
    ids = (torch.arange(T, device=dev) % 3 - 1).to(torch.int32)
    y = F.moe_fp8_vec(x, w, torch.ones((E, 1, K // 128), device=dev), ids, 1)
    want = torch.where(ids < 0, 0, 448 * (ids + 1)).to(torch.bfloat16)
    want[-3:] *= -1
    assert torch.equal(y, want[:, None].expand(T, N))


@gpu
@pytest.mark.parametrize("T", [1, 30, 400])
def test_graphs_and_streams(dev, T):
    """Two captured graphs replayed between eager calls, and calls on two streams at once."""
    k, E, N, K = 4, 6, 80, 512
    w, s = make_w((E,), N, K, 8, dev, exact=False)
    x = [make_x(T, K, torch.bfloat16, i, dev, exact=False) for i in range(2)]
    ids = [routes(T, k, E, 0.2, i, dev) for i in range(2)]

    def step(i):
        return [F.moe_fp8_vec(x[i], w, s, ids[i], k), F.fp8_linear(x[i], w[i], s[i])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(0)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(i))
        graphs.append(g)
    for turn in range(4):
        for i in range(2):
            x[i].copy_(make_x(T, K, torch.bfloat16, 10 + turn + i, dev, exact=False))
            ids[i].copy_(routes(T, k, E, 0.2 * turn, 20 + turn + i, dev))
        for i in ((0, 1) if turn % 2 else (1, 0)):
            graphs[i].replay()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[i], step(i)))
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = step(0)
    b = step(1)
    torch.cuda.synchronize()
    assert all(torch.equal(p, r) for p, r in zip(a + b, step(0) + step(1)))


def test_refusals():
    x, w, s = torch.zeros(2, 64), torch.zeros(3, 64).to(E4M3), torch.zeros(1, 1)
    for args, error in [
            ((x.double(), w, s), TypeError), ((x, w.float(), s), TypeError), ((x, w.to(torch.float8_e5m2), s), TypeError),
            ((x, w, s.half()), TypeError), ((x[0], w, s), ValueError), ((x[:, :63], w, s), ValueError), ((x, w[None], s), ValueError),
            ((x, w[:0], s), ValueError), ((x, w, s[:, :0]), ValueError), ((x, w, s[0]), ValueError),
            ((x.requires_grad_(True), w, s), RuntimeError), ((torch.zeros(2, 64), w, s), ValueError)]:  # the last: not on the GPU
        with pytest.raises(error, match="fp8_linear"):
            F.fp8_linear(*args)
    x, we, se, ids = torch.zeros(2, 64), w[None], s[None], torch.zeros(4, dtype=torch.int32)
    for args, error in [((x, we, se, ids.long(), 2), TypeError), ((x, we, se, ids, 3), ValueError), ((x, we, se, ids, 0), ValueError),
                        ((x, w, s, ids, 2), ValueError), ((x, we[:0], se[:0], ids, 2), ValueError), ((x, we, se, ids, 2), ValueError)]:
        with pytest.raises(error, match="moe_fp8_vec"):
            F.moe_fp8_vec(*args)
    off = torch.zeros(2, dtype=torch.int32)
    for args, error in [((x, we, se, off.long()), TypeError), ((x, we, se, off[:1]), ValueError), ((x, we, se, off[None]), ValueError),
                        ((x, we, se, off), ValueError)]:
        with pytest.raises(error, match="moe_fp8_sorted"):
            F.moe_fp8_sorted(*args)


def test_c_refusals():
    """Argument errors of the entry points come before any device work (the pointers are never read)."""
    L = _lib.lib()
    p = 4096

    def dense(x=p, dt=2, xs=64, K=64, w=p, s=p, N=8, T=2, y=p, ws=p, n=1 << 40):
        return L.ktmi_fp8_linear(x, dt, xs, K, w, s, N, T, y, ws, n, 0)

    for kw in [dict(dt=3), dict(K=0), dict(N=0), dict(T=-1), dict(x=0), dict(w=0), dict(s=0), dict(y=0), dict(x=p + 1), dict(s=p + 1),
               dict(y=p + 1), dict(xs=63), dict(K=1 << 25, xs=1 << 25), dict(T=1 << 31)]:
        assert dense(**kw) == -1 and b"fp8_linear" in L.ktmi_last_error(), kw
    need = L.ktmi_fp8_linear_workspace(8, 64, 1000)
    assert need >= 1000 * 128 and dense(T=1000, n=need - 1) == -4 and dense(T=1000, ws=0) == -4 and dense(T=1000, ws=p + 4) == -4
    assert dense(T=0) == 0 and L.ktmi_fp8_linear_workspace(8, 0, 5) == 0 and L.ktmi_fp8_linear_workspace(8, 64, -1) == 0

    def routed_(E=4, ids=p, k=2, T=2, ws=p, n=1 << 40, x=p, N=8):
        return L.ktmi_moe_fp8_vec(x, 2, 64, 64, p, p, N, E, ids, k, T, p, ws, n, 0)

    for kw in [dict(E=0), dict(E=F.MAX_EXPERTS + 1), dict(ids=0), dict(k=0), dict(k=65536), dict(T=-1), dict(T=1 << 31), dict(x=0)]:
        assert routed_(**kw) == -1 and b"moe_fp8_vec" in L.ktmi_last_error(), kw
    need = L.ktmi_moe_fp8_vec_workspace(8, 64, 100, 8, 4)
    assert need > 0 and routed_(T=100, k=8, n=need - 1) == -4 and routed_(T=100, k=8, ws=0) == -4
    assert routed_(T=0) == 0

    def sorted_(E=4, off=p, R=2, N=8, ws=p, n=1 << 40):
        return L.ktmi_moe_fp8_sorted(p, 2, 64, 64, p, p, N, E, off, R, p, ws, n, 0)

    for kw in [dict(E=0), dict(off=0), dict(R=-1), dict(N=0), dict(R=1 << 31)]:
        assert sorted_(**kw) == -1 and b"moe_fp8_sorted" in L.ktmi_last_error(), kw
    need = L.ktmi_moe_fp8_sorted_workspace(8, 64, 4, 1000)
    assert need > 0 and sorted_(R=1000, n=need - 1) == -4
    assert sorted_(R=0) == 0
    # a grid past 2^32 threads
    assert sorted_(E=2048, R=1 << 24, N=1 << 24) == -1 and b"grid" in L.ktmi_last_error()


def record_calls(dev):
    x, w, s = torch.ones((4, 128), device=dev), torch.ones((2, 8, 128), device=dev).to(E4M3), torch.ones((2, 1, 1), device=dev)
    ids = torch.zeros(4, dtype=torch.int32, device=dev)
    off = torch.tensor([0, 2, 4], dtype=torch.int32, device=dev)
    return {"fp8_linear": (lambda x: F.fp8_linear(x, w[0], s[0]), (x,)), "moe_fp8_vec": (lambda x: F.moe_fp8_vec(x, w, s, ids, 1), (x,)),
            "moe_fp8_sorted": (lambda x: F.moe_fp8_sorted(x, w, s, off), (x,))}


@pytest.mark.filterwarnings("ignore:Converting a tensor")
@pytest.mark.parametrize("name", ["fp8_linear", "moe_fp8_vec", "moe_fp8_sorted"])
def test_records_without_the_kernels_are_refused(monkeypatch, name):
    monkeypatch.setattr(F, "_check_gpu", lambda *a: None)
    check_refused_records(name, *record_calls("cpu")[name])


@gpu
@pytest.mark.filterwarnings("ignore:Converting a tensor")
@pytest.mark.parametrize("name", ["fp8_linear", "moe_fp8_vec", "moe_fp8_sorted"])
def test_records_without_the_kernels_are_refused_on_the_gpu(dev, name):
    check_refused_records(name, *record_calls(dev)[name])


@gpu
def test_tensors_without_memory_are_refused(dev):
    call, (x,) = record_calls(dev)["moe_fp8_sorted"]
    with pytest.raises(RuntimeError, match="null pointer"):
        call(wrapped(x))
