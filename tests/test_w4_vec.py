"""Products with 4-bit weights and group scales (kt_w4_vec).

Most cases use small integers for x and powers of two for the scales: every product and partial sum
is then exact in fp32 whatever the order of the sums, so the only rounding is the last one and the
outputs have to be equal bit for bit. Others use general values against 64 bits."""
import ctypes
import math

import pytest
import torch

import kt_prefill_lend_amd.kt_w4_vec as W
from helpers import check_refused_records
from kt_prefill_lend_amd import _lib

gpu = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def groups_of(K, G):
    return -(-K // G)


def make_weights(lead, N, K, G, zeros, sdtype, seed, dev, exact=True):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(0, 256, (*lead, N, (K + 1) // 2), generator=g, dtype=torch.uint8)
    shape = (*lead, N, groups_of(K, G))
    s = 2.0 ** torch.randint(-3, 1, shape, generator=g).float() if exact else torch.randn(shape, generator=g) * 0.01
    z = torch.randint(0, 16, shape, generator=g, dtype=torch.uint8) if zeros else None
    return q.to(dev), s.to(sdtype).to(dev), None if z is None else z.to(dev)


def make_x(T, K, dtype, seed, dev, exact=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-2, 3, (T, K), generator=g).float() if exact else torch.randn((T, K), generator=g)
    return x.to(dtype).to(dev)


def matrix(q, s, z, G, K):
    """(the weights, their size (code + zero point) * scale) in 64 bits."""
    v = torch.stack([q & 15, q >> 4], -1).flatten(-2)[..., :K].double()
    at = torch.arange(K, device=q.device) // G
    zz = torch.full_like(v, 8.0) if z is None else z.double()[..., at]
    sc = s.double()[..., at]
    return (v - zz) * sc, (v + zz) * sc.abs()


def routed(x, q, s, z, G, ids, top_k):
    """y [R, N] and the sums of the terms' sizes, in 64 bits."""
    K = x.shape[1]
    y = torch.zeros((ids.numel(), q.shape[1]), dtype=torch.float64, device=x.device)
    size = torch.zeros_like(y)
    xd = x.double()
    for e in range(q.shape[0]):
        r = (ids == e).nonzero().reshape(-1)
        if r.numel():
            w, m = matrix(q[e], s[e], None if z is None else z[e], G, K)
            y[r] = xd[r // top_k] @ w.t()
            size[r] = xd[r // top_k].abs() @ m.t()
    return y, size


def same(got, want64):
    """got is the exact result rounded once to its type (exact in fp32 before that)."""
    assert torch.equal(got, want64.float().to(got.dtype)), (got.double() - want64).abs().max()


# tokens, N, K, group
SHAPES = [
    (1, 1, 1, 32), (1, 3, 2, 32), (2, 17, 31, 64), (3, 16, 32, 32), (1, 64, 128, 128), (4, 33, 96, 32), (5, 65, 130, 64),
    (1, 515, 1111, 128), (16, 48, 256, 32), (17, 80, 192, 64), (33, 16, 640, 128), (64, 100, 513, 32), (65, 31, 384, 128),
    (1, 256, 2048, 128), (7, 40, 1024, 1024), (9, 24, 1000, 1000), (3, 20, 520, 4096), (2, 130, 4096, 256), (130, 70, 288, 32),
]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("T,N,K,G", SHAPES)
def test_dense_exact(dev, T, N, K, G, zeros, dtype):
    q, s, z = make_weights((), N, K, G, zeros, dtype, N + K, dev)
    x = make_x(T, K, dtype, T, dev)
    same(W.w4_vec(x, q, s, z, G), x.double() @ matrix(q, s, z, G, K)[0].t())


def routes(T, k, E, cold, seed, dev):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, E, (T * k,), generator=g, dtype=torch.int32)
    ids[torch.rand(T * k, generator=g) < cold] = -1
    return ids.to(dev)


# tokens, top_k, experts, N, K, group, share of routes without an expert
ROUTED = [
    (1, 1, 1, 5, 64, 32, 0.0), (1, 8, 40, 64, 256, 128, 0.3), (5, 3, 7, 72, 130, 64, 0.2), (13, 10, 9, 48, 384, 128, 0.4),
    (64, 8, 3, 33, 160, 32, 0.1), (40, 8, 300, 16, 96, 32, 0.0), (6, 2, 4, 20, 77, 64, 1.0),
    # more routes than a window's: past 1024, and one expert with most of them
    (260, 4, 5, 24, 64, 32, 0.1), (1100, 1, 2, 17, 40, 64, 0.0),
]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("T,k,E,N,K,G,cold", ROUTED)
def test_routed_exact(dev, T, k, E, N, K, G, cold, zeros, dtype):
    q, s, z = make_weights((E,), N, K, G, zeros, dtype, N + K, dev)
    x, ids = make_x(T, K, dtype, T, dev), routes(T, k, E, cold, T, dev)
    y = W.moe_w4_vec(x, q, s, ids, k, z, G)
    same(y, routed(x, q, s, z, G, ids, k)[0])
    assert (y[ids < 0] == 0).all()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("counts,tail,N,K,G", [
    ([1], 0, 5, 64, 32), ([0, 3, 0, 0, 17, 1, 0], 4, 72, 384, 128), ([0, 0, 0], 7, 9, 96, 64), ([70, 0, 33], 0, 40, 130, 64),
    ([5] * 60, 3, 16, 96, 32), ([300, 2], 1, 24, 256, 128), ([0] * 500 + [2, 1], 2, 33, 64, 32)])
def test_sorted_exact(dev, counts, tail, N, K, G, zeros, dtype):
    E, R = len(counts), sum(counts) + tail
    q, s, z = make_weights((E,), N, K, G, zeros, dtype, N + K, dev)
    ids = torch.cat([torch.full((n,), e) for e, n in enumerate(counts)] + [torch.full((tail,), -1)]).to(dev)
    offsets = torch.tensor([0] + counts).cumsum(0).to(torch.int32).to(dev)
    x = make_x(R, K, dtype, 5, dev)
    y = W.moe_w4_sorted(x, q, s, offsets, z, G)
    same(y, routed(x, q, s, z, G, ids, 1)[0])
    assert (y[R - tail:] == 0).all()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sdtype", DTYPES)
@pytest.mark.parametrize("T,N,K,G,zeros", [(1, 64, 2048, 128, False), (3, 48, 1000, 64, True), (24, 32, 512, 32, True)])
def test_general_values(dev, T, N, K, G, zeros, dtype, sdtype):
    """Against 64 bits. Every element: K products and the zero points' share of them, each addition off by
    2^-24 of a partial sum at most, then the group's scale and sum, then the last rounding. And as a
    whole: a chain of 2 K roundings of independent sign, of partial sums at most about three times the
    final ones' size, is off by 3 sqrt(2 K) 2^-24 of it."""
    q, s, z = make_weights((), N, K, G, zeros, sdtype, 3, dev, exact=False)
    x = make_x(T, K, dtype, 4, dev, exact=False)
    w, m = matrix(q, s, z, G, K)
    want, size = x.double() @ w.t(), x.double().abs() @ m.t()
    got = W.w4_vec(x, q, s, z, G).double()
    u = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0  # half a step below f16's normal numbers
    assert ((got - want).abs() <= u * want.abs() + (1 + u) * (2 * K + 4) * 2.0 ** -24 * size + tiny).all()
    assert (got - want).norm() <= (u + 3 * math.sqrt(2 * K) * 2.0 ** -24) * want.norm()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_code_and_zero_point(dev, dtype):
    """Each of the 16 codes against each of the 256 zero points a byte can hold, at every place of a group."""
    N, K, G = 256, 32, 32
    q = torch.arange(N * 16, dtype=torch.int64).reshape(N, 16)
    q = ((q * 7 + q // 16) % 256).to(torch.uint8).to(dev)
    z = torch.arange(256, dtype=torch.uint8).reshape(N, 1).to(dev)
    s = torch.ones((N, 1), dtype=dtype, device=dev)
    x = torch.eye(K).to(dtype).to(dev)
    y = W.w4_vec(x, q, s, z, G)
    same(y, matrix(q, s, z, G, K)[0].t())


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_infinities_and_nan(dev, dtype, bad):
    """A value of x that is not finite gives what the products' plain sum gives (an infinity where the weight
    is not zero, NaN where it is), in its own row alone."""
    T, N, K, G = 5, 40, 384, 64
    q, s, z = make_weights((), N, K, G, True, dtype, 3, dev)
    x = make_x(T, K, dtype, 4, dev)
    clean = W.w4_vec(x, q, s, z, G)
    x[2, 77] = bad
    got = W.w4_vec(x, q, s, z, G)
    assert torch.equal(got[[0, 1, 3, 4]], clean[[0, 1, 3, 4]])
    weight = matrix(q, s, z, G, K)[0][:, 77]
    want = weight * bad
    assert (weight == 0).any() and (weight > 0).any() and (weight < 0).any()
    assert torch.equal(got[2].double().isnan(), want.isnan())
    assert torch.equal(got[2].double()[~want.isnan()], want[~want.isnan()])
    # the same row as one of an expert's routes
    ids = torch.zeros(T, dtype=torch.int32, device=dev)
    again = W.moe_w4_vec(x, q[None], s[None], ids, 1, z[None], G)
    assert torch.equal(again.nan_to_num(7.0), got.nan_to_num(7.0))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_large_and_small_values(dev, dtype):
    """Values near the ends of x's range keep their bits: each output is one product."""
    f = torch.finfo(dtype)
    K = 64
    vals = torch.tensor([f.max / 8, -f.max / 16, f.tiny, -f.tiny * 1.5, f.tiny / 2, 1.0, f.eps, 1 + f.eps], dtype=dtype)
    x = torch.zeros((8, K), dtype=dtype)
    x[torch.arange(8), torch.arange(8) * 7] = vals
    x = x.to(dev)
    q = torch.full((4, K // 2), 0x99, dtype=torch.uint8, device=dev)  # code 9, weight 1
    q[1] = 0x77  # weight -1
    q[2] = 0x88  # weight 0
    q[3] = 0xCC  # weight 4
    s = torch.ones((4, 1), dtype=dtype, device=dev)
    y = W.w4_vec(x, q, s, None, 64)
    want = (vals.double()[:, None] * torch.tensor([1.0, -1.0, 0.0, 4.0], dtype=torch.float64)).to(dev)
    assert torch.equal(y.double(), want)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(dev, dtype):
    T, k, E, N, K, G = 6, 2, 5, 37, 256, 64
    q, s, z = make_weights((E,), N, K, G, True, dtype, 8, dev)
    x, ids = make_x(T, K, dtype, 9, dev), routes(T, k, E, 0.2, 9, dev)
    want = W.moe_w4_vec(x, q, s, ids, k, z, G)
    same(want, routed(x, q, s, z, G, ids, k)[0])
    wide = torch.full((T, K + 9), float("nan"), dtype=dtype, device=dev)
    wide[:, 3:K + 3] = x
    odd = torch.empty(q.numel() + 1, dtype=torch.uint8, device=dev)[1:]
    odd.copy_(q.reshape(-1))
    odd_s = torch.empty(s.numel() + 1, dtype=dtype, device=dev)[1:]
    odd_s.copy_(s.reshape(-1))
    odd_z = torch.empty(z.numel() + 1, dtype=torch.uint8, device=dev)[1:]
    odd_z.copy_(z.reshape(-1))
    assert torch.equal(W.moe_w4_vec(wide[:, 3:K + 3], odd.view(q.shape), odd_s.view(s.shape), ids, k, odd_z.view(z.shape), G), want)
    assert torch.equal(W.moe_w4_vec(x, q.view(torch.int32), s, ids, k, z, G), want)
    part = torch.cat([q, q], 1)[:, :N]  # experts apart
    assert not part.is_contiguous()
    assert torch.equal(W.moe_w4_vec(x.t().contiguous().t(), part, s, torch.stack([ids, ids], 1)[:, 0], k, z, G), want)
    one = make_x(1, K, dtype, 3, dev).expand(T, K)
    same(W.moe_w4_vec(one, q, s, ids, k, z, G), routed(one, q, s, z, G, ids, k)[0])


@gpu
def test_ids_and_offsets_outside_the_range(dev):
    E, N, K, G = 3, 20, 64, 32
    q, s, z = make_weights((E,), N, K, G, False, torch.bfloat16, 8, dev)
    x = make_x(6, K, torch.bfloat16, 9, dev)
    ids = torch.tensor([0, 3, 2, -1, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=dev)
    y = W.moe_w4_vec(x, q, s, ids, 1, z, G)
    same(y, routed(x, q, s, z, G, ids, 1)[0])
    # segments past the rows are cut at them
    offsets = torch.tensor([-5, 2, 4, 900], dtype=torch.int32, device=dev)
    y = W.moe_w4_sorted(x, q, s, offsets, z, G)
    same(y, routed(x, q, s, z, G, torch.tensor([0, 0, 1, 1, 2, 2], device=dev), 1)[0])


@gpu
def test_no_rows(dev):
    q, s, z = make_weights((2,), 8, 64, 32, False, torch.bfloat16, 8, dev)
    x = torch.empty((0, 64), dtype=torch.bfloat16, device=dev)
    ids = torch.empty((0,), dtype=torch.int32, device=dev)
    assert W.w4_vec(x, q[0], s[0], None, 32).shape == (0, 8)
    assert W.moe_w4_vec(x, q, s, ids, 4, None, 32).shape == (0, 8)
    assert W.moe_w4_sorted(x, q, s, torch.zeros(3, dtype=torch.int32, device=dev), None, 32).shape == (0, 8)


@gpu
def test_codes_past_32_bits(dev):
    """A matrix behind more than 4 GiB of codes."""
    E, N, K, G = 5, 32768, 65536, 65536
    q = torch.zeros((E, N, K // 2), dtype=torch.uint8, device=dev)
    q[4] = 0x99
    q[4, N - 1, K // 2 - 1] = 0xA9
    s = torch.ones((E, N, 1), dtype=torch.float32, device=dev)
    x = torch.zeros((2, K), dtype=torch.float32, device=dev)
    x[0, :64], x[0, K - 1], x[1, 5] = 1.0, 1.0, 3.0
    ids = torch.tensor([4, 4], dtype=torch.int32, device=dev)
    for y in (W.moe_w4_vec(x, q, s, ids, 1, None, G),
              W.moe_w4_sorted(x, q, s, torch.tensor([0, 0, 0, 0, 0, 2], dtype=torch.int32, device=dev), None, G)):
        assert (y[0, :N - 1] == 65).all() and y[0, N - 1] == 66 and (y[1] == 3).all()


@gpu
@pytest.mark.parametrize("T", [1, 20])
def test_graphs_and_streams(dev, T):
    """Two captured graphs replayed between eager calls, and calls on two streams at once."""
    k, E, N, K, G = 4, 12, 80, 512, 128
    q, s, z = make_weights((E,), N, K, G, True, torch.bfloat16, 8, dev, exact=False)
    x = [make_x(T, K, torch.bfloat16, i, dev, exact=False) for i in range(2)]
    ids = [routes(T, k, E, 0.2, i, dev) for i in range(2)]

    def step(i):
        return [W.moe_w4_vec(x[i], q, s, ids[i], k, z, G), W.w4_vec(x[i], q[i], s[i], z[i], G)]

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


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("T,N,K,G", [(64, 4113, 256, 128), (33, 8192, 130, 64), (40, 4200, 512, 32), (200, 1100, 392, 392),
                                     (70, 3000, 4480, 128)])
def test_dense_exact_of_many_weight_rows(dev, T, N, K, G, zeros, dtype):
    """More blocks of 32 weight rows than CUs, fewer of 64 for 17 rows of x and more."""
    q, s, z = make_weights((), N, K, G, zeros, dtype, 3, dev)
    x = make_x(T, K, dtype, 5, dev)
    same(W.w4_vec(x, q, s, z, G), x.double() @ matrix(q, s, z, G, K)[0].t())


LARGE_GROUPS = [2 ** 31, 2 ** 32, 2 ** 40, 2 ** 64 + 32]


@pytest.mark.parametrize("G", LARGE_GROUPS)
def test_group_sizes_past_32_bits_reach_c_as_one_group(G):
    x, q, s = torch.ones(1, 64), torch.zeros((3, 32), dtype=torch.uint8), torch.ones(3, 1)
    assert W._args(x, q, s, None, G)[1][-1] == 64


@gpu
@pytest.mark.parametrize("K", [1, 64, 127, 128, 200])
@pytest.mark.parametrize("G", LARGE_GROUPS)
def test_group_sizes_past_32_bits(dev, G, K):
    q, s, z = make_weights((2,), 21, K, K, True, torch.bfloat16, 8, dev)
    x = make_x(3, K, torch.bfloat16, 9, dev)
    same(W.w4_vec(x, q[1], s[1], z[1], G), x.double() @ matrix(q[1], s[1], z[1], K, K)[0].t())
    ids = torch.tensor([1, 0, -1], dtype=torch.int32, device=dev)
    same(W.moe_w4_vec(x, q, s, ids, 1, z, G), routed(x, q, s, z, K, ids, 1)[0])
    # the C entry by itself
    if G < 2 ** 63:
        y = torch.empty((3, 21), dtype=torch.bfloat16, device=dev)
        L = _lib.lib()
        assert L.ktmi_w4_vec(x.data_ptr(), _lib.KTMI_BF16, K, K, q.data_ptr(), s.data_ptr(), _lib.KTMI_BF16, z.data_ptr(), G,
                             21, 3, y.data_ptr(), _lib.stream_ptr()) == 0
        same(y, x.double() @ matrix(q[0], s[0], z[0], K, K)[0].t())


# ---------------------------------------------------------------- refusals (no GPU)


def test_refusals():
    x, q, s = torch.zeros(2, 64), torch.zeros(3, 32, dtype=torch.uint8), torch.zeros(3, 2)
    z = torch.zeros(3, 2, dtype=torch.uint8)
    for args, error in [
            ((x.double(), q, s, z, 32), TypeError), ((x, q.long(), s, z, 32), TypeError), ((x, q, s.double(), z, 32), TypeError),
            ((x, q, s, z.int(), 32), TypeError), ((x[0], q, s, z, 32), ValueError), ((x[:, :63], q[:, :31], s, z, 32), ValueError),
            ((x, q, s, z, 48), ValueError), ((x, q, s, z, 0), ValueError), ((x, q, s, z, 63), ValueError),
            ((x, q, s[:, :1], z, 32), ValueError), ((x, q, s, z[:2], 32), ValueError), ((x, q[None], s, z, 32), ValueError),
            ((x, q, s, z, 64), ValueError), ((x.requires_grad_(True), q, s, z, 32), RuntimeError),
            ((x.detach()[:, :60], torch.zeros(3, 8, dtype=torch.int32), s, z, 32), ValueError),
            ((torch.zeros(2, 64), q, s, z, 32), ValueError)]:  # the last: not on the GPU
        with pytest.raises(error, match="w4_vec"):
            W.w4_vec(*args)
    x, qe, se = torch.zeros(2, 64), q[None], s[None]
    ids = torch.zeros(4, dtype=torch.int32)
    for args, error in [((x, qe, se, ids.long(), 2), TypeError), ((x, qe, se, ids, 3), ValueError), ((x, qe, se, ids, 0), ValueError),
                        ((x, q, s, ids, 2), ValueError), ((x, qe[:0], se[:0], ids, 2), ValueError), ((x, qe, se, ids, 2), ValueError)]:
        with pytest.raises(error, match="moe_w4_vec"):
            W.moe_w4_vec(*args, group_size=32)
    off = torch.zeros(2, dtype=torch.int32)
    for args, error in [((x, qe, se, off.long()), TypeError), ((x, qe, se, off[:1]), ValueError), ((x, qe, se, off[None]), ValueError),
                        ((x, qe, se, off), ValueError)]:
        with pytest.raises(error, match="moe_w4_sorted"):
            W.moe_w4_sorted(*args, group_size=32)


def test_c_refusals():
    """Argument errors of the entry points come before any device work (the pointers are never read)."""
    L = _lib.lib()
    p = 4096

    def dense(x=p, dt=2, xs=64, K=64, q=p, s=p, st=2, z=0, G=32, N=8, T=2, y=p):
        return L.ktmi_w4_vec(x, dt, xs, K, q, s, st, z, G, N, T, y, 0)

    for kw in [dict(dt=3), dict(st=5), dict(K=0), dict(N=0), dict(T=-1), dict(G=48), dict(G=0), dict(G=63), dict(x=0), dict(q=0),
               dict(s=0), dict(y=0), dict(x=p + 1), dict(s=p + 1), dict(y=p + 1), dict(xs=63), dict(K=1 << 25, xs=1 << 25)]:
        assert dense(**kw) == -1 and b"w4_vec" in L.ktmi_last_error(), kw
    assert dense(T=0) == 0

    def routed_(E=4, ids=p, k=2, T=2, ws=p, n=1 << 30, **kw):
        a = dict(x=p, dt=2, xs=64, K=64, q=p, s=p, st=2, z=0, G=32, N=8, y=p) | kw
        return L.ktmi_moe_w4_vec(a["x"], a["dt"], a["xs"], a["K"], a["q"], a["s"], a["st"], a["z"], a["G"], a["N"], E, ids, k, T,
                                 a["y"], ws, n, 0)

    for kw in [dict(E=0), dict(E=W.MAX_EXPERTS + 1), dict(ids=0), dict(k=0), dict(k=65536), dict(T=-1), dict(T=1 << 31), dict(G=33)]:
        assert routed_(**kw) == -1 and b"moe_w4_vec" in L.ktmi_last_error(), kw
    need = L.ktmi_moe_w4_vec_workspace(100000, 8, 4)
    if need:
        assert routed_(T=100000, k=8, n=need - 1) == -4 and routed_(T=100000, k=8, ws=0) == -4
    assert routed_(T=0) == 0

    def sorted_(E=4, off=p, R=2, N=8, y=p):
        return L.ktmi_moe_w4_sorted(p, 2, 64, 64, p, p, 2, 0, 32, N, E, off, R, y, 0)

    for kw in [dict(E=0), dict(off=0), dict(R=-1), dict(N=0), dict(y=0)]:
        assert sorted_(**kw) == -1 and b"moe_w4_sorted" in L.ktmi_last_error(), kw
    assert sorted_(R=0) == 0


def test_c_refuses_grids_past_32_bits():
    L = _lib.lib()
    p, most = 4096, 1 << 23
    for K in (64, 128):
        assert L.ktmi_w4_vec(p, 2, K, K, p, p, 2, 0, 32, 8, most + 1, p, 0) == -1 and b"2^23" in L.ktmi_last_error()
        assert L.ktmi_moe_w4_sorted(p, 2, K, K, p, p, 2, 0, 32, 8, 4, p, most + 1, p, 0) == -1
        assert b"2^23" in L.ktmi_last_error()
        assert L.ktmi_moe_w4_vec(p, 2, K, K, p, p, 2, 0, 32, 8, 4, p, 2, most // 2 + 1, p, p, 1 << 40, 0) == -1
        assert b"2^23" in L.ktmi_last_error()
    assert L.ktmi_w4_vec(p, 2, 128, 128, p, p, 2, 0, 32, 1 << 24, most, p, 0) == -1 and b"2^32" in L.ktmi_last_error()


# ---------------------------------------------------------------- what torch would record without the kernels


def record_calls(dev):
    """name -> (call, its tensors that could carry a derivative)."""
    x, q, s = torch.ones(2, 64, device=dev), torch.zeros((3, 32), dtype=torch.uint8, device=dev), torch.ones(3, 2, device=dev)
    ids, offsets = torch.zeros(2, dtype=torch.int32, device=dev), torch.tensor([0, 2], dtype=torch.int32, device=dev)
    return {"w4_vec": (lambda x, s: W.w4_vec(x, q, s, None, 32), (x, s)),
            "moe_w4_vec": (lambda x, s: W.moe_w4_vec(x, q[None], s, ids, 1, None, 32), (x, s[None])),
            "moe_w4_sorted": (lambda x, s: W.moe_w4_sorted(x, q[None], s, offsets, None, 32), (x, s[None]))}


@pytest.mark.filterwarnings("ignore:Converting a tensor")
@pytest.mark.parametrize("name", ["w4_vec", "moe_w4_vec", "moe_w4_sorted"])
def test_records_without_the_kernels_are_refused(monkeypatch, name):
    monkeypatch.setattr(W, "_check_gpu", lambda *a: None)
    check_refused_records(name, *record_calls("cpu")[name])


@gpu
@pytest.mark.filterwarnings("ignore:Converting a tensor")
@pytest.mark.parametrize("name", ["w4_vec", "moe_w4_vec", "moe_w4_sorted"])
def test_records_without_the_kernels_are_refused_on_the_gpu(dev, name):
    call, tensors = record_calls(dev)[name]
    want = call(*tensors)
    check_refused_records(name, call, tensors)
    assert torch.equal(call(*tensors), want)


# ---------------------------------------------------------------- every kernel shape of the products


def kernel_of(by, dtype, K, G, N, E, R):
    """(x_rows, col_waves, weight_rows, tiles, staged) of the kernel that the call takes."""
    k = _lib.ktmi_w4_kernel()
    _lib.check(_lib.lib().ktmi_w4_kernel_of(by, _lib.dtype_code(dtype), K, G, N, E, R, ctypes.byref(k)), "w4_kernel_of")
    return tuple(getattr(k, name) for name, _ in k._fields_)


def test_kernel_of_refusals():
    L, k = _lib.lib(), _lib.ktmi_w4_kernel()
    good = dict(by=_lib.W4_SORTED, dt=2, K=256, G=128, N=64, E=4, R=8)
    for kw in [dict(), dict(by=3), dict(by=-1), dict(dt=5), dict(K=0), dict(G=48), dict(N=0), dict(E=0), dict(R=0), dict(R=1 << 24)]:
        a = good | kw
        rc = L.ktmi_w4_kernel_of(a["by"], a["dt"], a["K"], a["G"], a["N"], a["E"], a["R"], ctypes.byref(k))
        assert rc == (-1 if kw else 0), kw
    assert L.ktmi_w4_kernel_of(0, 2, 256, 128, 64, 1, 8, None) == -1


# rows of x, N, K, group; with the shapes above: the kernel that bf16 rows take
DENSE_SHAPES = [
    (16, 20000, 2080, 32, (16, 1, 64, 1, 1)), (64, 40000, 2080, 32, (32, 1, 64, 2, 1)), (1, 16390, 2048, 128, (16, 1, 64, 1, 0)),
    (33, 16400, 768, 64, (32, 1, 64, 1, 0)), (2, 100000, 1280, 256, (16, 1, 64, 2, 0)), (5, 1030, 2080, 32, (16, 4, 16, 1, 0)),
    (40, 1030, 2080, 64, (32, 4, 32, 1, 1)), (40, 1030, 768, 64, (32, 4, 32, 1, 0)), (64, 6000, 768, 128, (32, 2, 64, 1, 0)),
    (64, 6000, 7168, 128, (32, 2, 64, 1, 1)), (64, 6000, 2080, 32, (32, 2, 64, 1, 1)),
]
# mean rows of an expert, experts, N, K, group: uneven counts, some none
SORTED_SHAPES = [
    (8, 48, 2050, 768, 128, (16, 1, 64, 2, 0)), (3, 128, 1050, 4480, 32, (16, 1, 64, 4, 1)), (20, 64, 1050, 4096, 64, (32, 1, 64, 2, 1)),
    (2, 400, 1030, 640, 128, (16, 1, 64, 8, 0)), (21, 150, 520, 1280, 256, (32, 1, 64, 2, 1)), (24, 90, 2050, 2080, 32, (32, 1, 64, 5, 1)),
    (2, 300, 33, 384, 64, (16, 1, 64, 1, 0)), (1, 140, 20, 256, 32, (16, 4, 16, 1, 0)), (25, 130, 20, 640, 128, (32, 4, 32, 1, 0)),
]
# tokens, routes of each, experts, N, K, group: up to 64 ids looked at by every wave, more ordered in one launch,
# in chunks, in more chunks than add up their counts by themselves
ROUTED_SHAPES = [
    (8, 8, 200, 2050, 768, 128, (16, 1, 64, 2, 0)), (13, 8, 18, 3000, 4096, 64, (16, 1, 64, 1, 1)),
    (625, 8, 200, 200, 256, 32, (32, 1, 64, 1, 0)), (17000, 8, 130, 40, 128, 128, (32, 2, 64, 1, 0)),
    (60, 17, 150, 130, 384, 64, (16, 1, 64, 1, 0)), (5000, 1, 300, 70, 256, 64, (16, 1, 64, 1, 0)),
]


def test_kernel_shapes_are_all_reached():
    """The lists hold every split of the waves, several row tiles a block, and stages, for each group size class."""
    bf16, reached = torch.bfloat16, set()
    for T, N, K, G, want in DENSE_SHAPES:
        assert kernel_of(_lib.W4_DENSE, bf16, K, G, N, 1, T) == want, (T, N, K, G)
        reached.add((min(G, 128), *want))
    for n, E, N, K, G, want in SORTED_SHAPES:
        assert kernel_of(_lib.W4_SORTED, bf16, K, G, N, E, n * E) == want, (n, E, N, K, G)
        reached.add((min(G, 128), *want))
    for T, k, E, N, K, G, want in ROUTED_SHAPES:
        assert kernel_of(_lib.W4_IDS, bf16, K, G, N, E, T * k) == want, (T, k, E, N, K, G)
        reached.add((min(G, 128), *want))
    splits = {(rows, waves, at_once) for _, rows, waves, at_once, _, _ in reached}
    assert splits == {(16, 1, 64), (16, 4, 16), (32, 1, 64), (32, 4, 32), (32, 2, 64)}
    for G in (32, 64, 128):
        whole = [r for r in reached if r[0] == G and r[2] == 1]
        assert {r[1] for r in whole} == {16, 32} and any(r[4] > 1 for r in whole)
    assert any(r[5] and r[4] > 1 and r[1] == 16 for r in reached) and any(r[5] and r[4] > 1 and r[1] == 32 for r in reached)


def uneven(mean, E, seed):
    """Rows of each of E experts, mean * E in all."""
    g = torch.Generator().manual_seed(seed)
    at = torch.multinomial(torch.rand(E, generator=g) ** 2, mean * E, replacement=True, generator=g)
    return torch.bincount(at, minlength=E)


def scale_types(dtype):
    return {"own": dtype, "other": torch.bfloat16 if dtype == torch.float32 else torch.float32}


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("stype", ["own", "other"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("T,N,K,G,shape", DENSE_SHAPES)
def test_dense_shapes_exact(dev, T, N, K, G, shape, zeros, stype, dtype):
    q, s, z = make_weights((), N, K, G, zeros, scale_types(dtype)[stype], N + K, dev)
    x = make_x(T, K, dtype, T, dev)
    same(W.w4_vec(x, q, s, z, G), x.double() @ matrix(q, s, z, G, K)[0].t())


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("stype", ["own", "other"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("n,E,N,K,G,shape", SORTED_SHAPES)
def test_sorted_shapes_exact(dev, n, E, N, K, G, shape, zeros, stype, dtype):
    """Rows before the first segment and behind the last are zeros."""
    before, after = 3, 2
    counts = uneven(n, E, N)
    R = before + int(counts.sum()) + after
    q, s, z = make_weights((E,), N, K, G, zeros, scale_types(dtype)[stype], N + K, dev)
    ids = torch.full((R,), -1)
    ids[before:R - after] = torch.repeat_interleave(torch.arange(E), counts)
    offsets = (before + torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)])).to(torch.int32).to(dev)
    x = make_x(R, K, dtype, 5, dev)
    y = W.moe_w4_sorted(x, q, s, offsets, z, G)
    same(y, routed(x, q, s, z, G, ids.to(dev), 1)[0])
    assert (y[:before] == 0).all() and (y[R - after:] == 0).all()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("stype", ["own", "other"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("T,k,E,N,K,G,shape", ROUTED_SHAPES)
def test_routed_shapes_exact(dev, T, k, E, N, K, G, shape, zeros, stype, dtype):
    q, s, z = make_weights((E,), N, K, G, zeros, scale_types(dtype)[stype], N + K, dev)
    x, ids = make_x(T, K, dtype, T, dev), routes(T, k, E, 0.2, T, dev)
    same(W.moe_w4_vec(x, q, s, ids, k, z, G), routed(x, q, s, z, G, ids, k)[0])


# K, group: rows that end with a word of codes and rows that do not
WIDE = [(128, 32), (130, 64), (256, 128), (192, 64), (131, 128)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("again", [False, True])
@pytest.mark.parametrize("K,G", WIDE)
def test_every_code_and_zero_point_on_the_matrix_cores(dev, K, G, again, dtype):
    """Each of the 256 bytes of codes against each of the 256 zero points, at every place of a step. With an
    infinity in another row of the block its sums are made again another way."""
    N, groups = 256, groups_of(K, G)
    half = (K + 1) // 2
    n, j = torch.arange(N)[:, None], torch.arange(half)[None]
    x = torch.eye(K).to(dtype).to(dev)
    if again:
        x = torch.cat([x, torch.full((1, K), float("inf")).to(dtype).to(dev)])
        x = x[torch.randperm(K + 1, generator=torch.Generator().manual_seed(2)).to(dev)]
    s = torch.ones((N, groups), dtype=dtype, device=dev)
    finite = torch.isfinite(x).all(1)
    for shift in range(0, 256, 16):
        q = ((j * 16 + n * 1 + n * shift) % 256).to(torch.uint8).to(dev)
        z = ((n * 3 + torch.arange(groups)[None] * 85 + shift) % 256).to(torch.uint8).to(dev)
        y = W.w4_vec(x, q, s, z, G)
        w = matrix(q, s, z, G, K)[0]
        same(y[finite], x[finite].double() @ w.t())


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("large", [False, True])
@pytest.mark.parametrize("K,G", WIDE)
def test_large_and_small_values_on_the_matrix_cores(dev, K, G, large, dtype):
    """Values near the ends of x's range keep their bits, subnormal ones too: each output is one product. Large
    ones times a code pass fp32, times the code less the zero point they do not."""
    f = torch.finfo(dtype)
    vals = [f.max / 8, -f.max / 16, f.max / 16, -f.max / 8] if large else []
    vals = torch.tensor(vals + [f.tiny, -f.tiny * 1.5, f.tiny / 2, -f.tiny / 4, 1.0, f.eps, 1 + f.eps, -f.tiny * (1 + f.eps)],
                        dtype=dtype)
    n = vals.numel()
    x = torch.zeros((n, K), dtype=dtype)
    x[torch.arange(n), torch.arange(n) * 10] = vals
    x = x.to(dev)
    q = torch.full((4, (K + 1) // 2), 0x99, dtype=torch.uint8, device=dev)  # code 9, weight 1
    q[1] = 0x77  # weight -1
    q[2] = 0x88  # weight 0
    q[3] = 0xCC  # weight 4
    s = torch.ones((4, groups_of(K, G)), dtype=dtype, device=dev)
    y = W.w4_vec(x, q, s, None, G)
    weight = torch.tensor([1.0, -1.0, 0.0, 4.0], dtype=torch.float64)
    want, off = (vals.double()[:, None] * weight).to(dev), torch.zeros(n, 4, dtype=torch.float64)
    if dtype == torch.float32:  # its three bf16 parts end at 2^-133: what is below is less than one such step
        off[vals.abs() < 2.0 ** -109] = 2.0 ** -133 * weight.abs()
        # Values of 24 bits: of the parts h, m, l (|m| < 2^-7 |v|, |l| < 2^-15 |v|) the sum runs over c h, -8 h (both
        # exact: 8 bits times 4), c m, -8 m, c l, -8 l, whose partial sums are at most (|c - 8| + 12 2^-7) |v|, below
        # 1.1 |c - 8| |v| (all of it exact for c = 8): four additions, each off by 2^-24 of that.
        full = vals.abs() > 1e30
        off[full] = 4 * 2.0 ** -24 * 1.1 * vals.double().abs()[full, None] * weight.abs()
    assert ((y.double() - want).abs() <= off.to(dev)).all()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [20, 17000])
@pytest.mark.parametrize("K,G", WIDE)
def test_ids_and_offsets_outside_the_range_on_the_matrix_cores(dev, K, G, N, dtype):
    E = 3
    q, s, z = make_weights((E,), N, K, G, True, dtype, 8, dev)
    x = make_x(6, K, dtype, 9, dev)
    ids = torch.tensor([0, 3, 2, -1, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=dev)
    same(W.moe_w4_vec(x, q, s, ids, 1, z, G), routed(x, q, s, z, G, ids, 1)[0])
    more = ids.repeat(12)  # past the ids that a wave holds
    same(W.moe_w4_vec(x, q, s, more, 12, z, G), routed(x, q, s, z, G, more, 12)[0])
    # segments past the rows are cut at them, rows in none are zeros
    for offsets, of in [([-5, 2, 4, 900], [0, 0, 1, 1, 2, 2]), ([2, 2, 5, 5], [-1, -1, 1, 1, 1, -1]), ([9, 9, 9, 9], [-1] * 6),
                        ([-9, -9, -9, -1], [-1] * 6), ([0, 6, 6, 2 ** 31 - 1], [0] * 6), ([-2 ** 31, 1, 1, 6], [0, 2, 2, 2, 2, 2])]:
        y = W.moe_w4_sorted(x, q, s, torch.tensor(offsets, dtype=torch.int32, device=dev), z, G)
        same(y, routed(x, q, s, z, G, torch.tensor(of, device=dev), 1)[0])


# rows of x, N, K, group: the columns shared by four waves, by two, whole rows a wave, several row tiles, stages
NEIGHBOURS = [(5, 40, 384, 64), (20, 70, 640, 128), (64, 6000, 768, 128), (7, 20000, 2080, 32), (24, 40000, 2080, 64), (9, 40, 130, 64)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("T,N,K,G", NEIGHBOURS)
def test_rows_beside_one_that_is_not_finite_keep_their_bits(dev, T, N, K, G, zeros, dtype):
    """General values: a row's sums do not depend on what another row of the call holds, by a bit."""
    q, s, z = make_weights((), N, K, G, zeros, dtype, 3, dev, exact=False)
    x = make_x(T, K, dtype, 4, dev, exact=False)
    clean = W.w4_vec(x, q, s, z, G)
    f = torch.finfo(dtype)
    w, m = matrix(q, s, z, G, K)
    for bad in (float("inf"), float("nan"), f.max, f.max / 12):
        other = x.clone()
        other[2, K - 2] = other[T - 1, 1] = bad
        got = W.w4_vec(other, q, s, z, G)
        rest = [t for t in range(T) if t not in (2, T - 1)]
        assert torch.equal(got[rest], clean[rest])
        ids = torch.zeros(T, dtype=torch.int32, device=dev)
        again = W.moe_w4_vec(other, q[None], s[None], ids, 1, None if z is None else z[None], G)
        first = W.moe_w4_vec(x, q[None], s[None], ids, 1, None if z is None else z[None], G)
        assert torch.equal(again[rest], first[rest])
        # the rows themselves: what 64 bits give where they are not finite; else, where the groups' sums
        # stay within fp32, as near as a plain sum
        plain = matrix(q, torch.ones_like(s), z, G, K)[0].abs()
        for t in (2, T - 1):
            want = other[t].double() @ w.t()
            if abs(bad) < float("inf"):
                near = (other[t].double().abs() @ plain.t() < 2.0 ** 127) & (want.abs() < 0.9 * f.max)
                size = other[t].double().abs() @ m.t()
                tol = f.eps / 2 * want.abs() + (1 + f.eps / 2) * (2 * K + 4) * 2.0 ** -24 * size
                tol += 2.0 ** -25 if dtype == torch.float16 else 0.0  # half a step below f16's normal numbers
                assert near.any() and ((got[t].double() - want).abs() <= tol)[near].all()
            else:
                assert torch.equal(got[t].isnan(), want.isnan())
                assert torch.equal(got[t][~want.isnan()].double(), want[~want.isnan()])


@gpu
@pytest.mark.parametrize("E", [1, 2, 63, 64, 65, 127, 640, 2047, 2048])
@pytest.mark.parametrize("K", [1, 96, 127, 130])
def test_sorted_exact_of_many_experts(dev, E, K):
    """Empty segments in front, between and behind, a first segment past row 0, offsets past the rows."""
    g = torch.Generator().manual_seed(E + K)
    R, N, G = 301, 3, 32
    q, s, z = make_weights((E,), N, K, G, True, torch.bfloat16, 8, dev)
    x = make_x(R, K, torch.bfloat16, 9, dev)
    for offsets in (torch.sort(torch.randint(-20, R + 20, (E + 1,), generator=g)).values,
                    torch.sort(torch.randint(7, R - 7, (E + 1,), generator=g) // 40 * 40).values,
                    torch.full((E + 1,), R // 2), torch.arange(E + 1) - 3, R - E - 1 + torch.arange(E + 1)):
        ids = torch.searchsorted(offsets, torch.arange(R), right=True) - 1
        ids[ids >= E] = -1
        y = W.moe_w4_sorted(x, q, s, offsets.to(torch.int32).to(dev), z, G)
        same(y, routed(x, q, s, z, G, ids.to(dev), 1)[0])


def test_zeros_without_memory_are_refused():
    from helpers import wrapped

    x, q, s = torch.ones(2, 64), torch.zeros((3, 32), dtype=torch.uint8), torch.ones(3, 2)
    with pytest.raises(TypeError, match="zeros: a Wrapped"):
        W._args(x, q, s, wrapped(torch.zeros((3, 2), dtype=torch.uint8)), 32)
