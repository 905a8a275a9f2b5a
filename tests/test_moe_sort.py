"""Tokens sorted by expert and back (kt_moe_sort): places and copies exactly, sums and gradients
against 64 bits. Tolerances count roundings: an fp32 step is off by 2^-24 of its result at most,
the final rounding by half a step of the output type."""
import numpy as np
import pytest
import torch

import kt_prefill_lend_amd.kt_moe_sort as S
from helpers import check_refused_records
from kt_prefill_lend_amd import _lib

gpu = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
U24 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def plain_order(ids, E):
    """(offsets, perm, pos) of ids [T, k] by the definition, in numpy."""
    flat = ids.cpu().numpy().reshape(-1).astype(np.int64)
    key = np.where((flat >= 0) & (flat < E), flat, E)
    order = np.argsort(key, kind="stable")
    pos = np.empty_like(order)
    pos[order] = np.arange(order.size)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(key, minlength=E + 1)[:E])])
    valid = key < E
    return (offsets.astype(np.int32), np.where(valid[order], order, ~order).astype(np.int32),
            np.where(valid, pos, ~pos).astype(np.int32).reshape(ids.shape))


def make_ids(T, k, E, cold, seed, dev):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, E, (T, k), generator=g, dtype=torch.int32)  # an expert may come twice in a token
    ids[torch.rand((T, k), generator=g) < cold] = -1
    return ids.to(dev)


def make_x(shape, dtype, seed, dev):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(dev)


def check_sorted(s, x, ids, E):
    offsets, perm, pos = plain_order(ids, E)
    assert np.array_equal(s.offsets.cpu().numpy(), offsets)
    assert np.array_equal(s.perm.cpu().numpy(), perm)
    assert np.array_equal(s.pos.cpu().numpy(), pos)
    route = torch.from_numpy(np.where(perm >= 0, perm, 0).astype(np.int64)).to(x.device)
    want = x.detach()[route // ids.shape[1]]
    want[torch.from_numpy(perm < 0).to(x.device)] = 0
    bits = torch.int32 if x.dtype == torch.float32 else torch.int16
    assert torch.equal(s.rows.detach().view(bits), want.contiguous().view(bits))


# tokens, top_k, experts, cols, share of routes without an expert
SHAPES = [
    (1, 1, 1, 1, 0.0), (1, 8, 256, 2048, 0.4), (3, 2, 5, 7, 0.3), (5, 3, 2, 9, 0.0), (7, 17, 33, 130, 0.2),
    (64, 8, 512, 515, 0.5), (77, 10, 512, 1000, 0.0), (13, 8, 40, 520, 1.0),
    # one route more and less than the blocks of the order take
    (255, 4, 16, 64, 0.1), (1025, 1, 2048, 8, 0.0), (2047, 1, 3, 24, 0.1), (2049, 1, 300, 16, 0.1),
    (683, 6, 64, 33, 0.9), (4097, 8, 129, 40, 0.3),
    (512, 8, 2048, 12, 0.2), (4097, 1, 2047, 10, 0.1), (6144, 1, 3, 8, 0.0), (2049, 3, 300, 16, 0.1),
]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,E,K,cold", SHAPES)
def test_sort(dev, T, k, E, K, cold, dtype):
    ids, x = make_ids(T, k, E, cold, T + K, dev), make_x((T, K), dtype, 3, dev)
    check_sorted(S.moe_sort(x, ids, E), x, ids, E)


def unsort_exact(rows, w, pos):
    """(y, sum of |terms|) in 64 bits."""
    placed = (pos >= 0).double()
    r = rows.detach().double()[pos.clamp(min=0).long()]
    r = torch.where(pos[:, :, None] >= 0, r, torch.zeros((), dtype=torch.float64, device=r.device))
    ww = placed if w is None else torch.where(pos >= 0, w.detach().double(), placed)
    return (r * ww[:, :, None]).sum(1), (r * ww[:, :, None]).abs().sum(1)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,E,K,cold", SHAPES)
@pytest.mark.parametrize("weighted", [True, False])
def test_unsort_and_gradients(dev, T, k, E, K, cold, dtype, weighted):
    ids = make_ids(T, k, E, cold, T + K, dev)
    pos = torch.from_numpy(plain_order(ids, E)[2]).to(dev)
    rows = make_x((T * k, K), dtype, 4, dev).requires_grad_(True)
    w = make_x((T, k), torch.float32, 5, dev).requires_grad_(True) if weighted else None
    dy = make_x((T, K), dtype, 6, dev)
    y = S.moe_unsort(rows, w, pos)
    want, size = unsort_exact(rows, w, pos)
    u = half_step(dtype)
    tiny = 1e-7 if dtype == torch.float16 else 1e-37  # below the type's normal numbers steps stop shrinking
    assert ((y.detach().double() - want).abs() <= u * want.abs() + (1 + u) * k * U24 * size + tiny).all()
    drows, *dw = torch.autograd.grad(y, (rows, w) if weighted else (rows,), dy)
    placed = (pos >= 0).reshape(-1)
    ww = torch.ones((T, k), dtype=torch.float64, device=dev) if w is None else w.detach().double()
    at = torch.where(pos >= 0, pos, ~pos).reshape(-1).long()
    want = torch.zeros((T * k, K), dtype=torch.float64, device=dev)
    want[at] = torch.where(placed[:, None], (ww[:, :, None] * dy.double()[:, None]).reshape(-1, K), want)
    assert ((drows.double() - want).abs() <= (u + U24 + u * U24) * want.abs() + tiny).all()
    if weighted:
        terms = rows.detach().double()[pos.clamp(min=0).long()] * dy.double()[:, None]
        want = torch.where(pos >= 0, terms.sum(2), torch.zeros((), dtype=torch.float64, device=dev))
        depth = K / 64 + 32  # additions of a lane's own values, then of lanes and waves
        assert ((dw[0].double() - want).abs() <= depth * U24 * terms.abs().sum(2) + 1e-37).all()
        assert (dw[0][pos < 0] == 0).all()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,E,K,cold", [(1, 8, 16, 64, 0.5), (9, 3, 4, 21, 0.3), (130, 8, 32, 1000, 0.0)])
def test_sort_gradient(dev, T, k, E, K, cold, dtype):
    ids = make_ids(T, k, E, cold, 8, dev)
    x = make_x((T, K), dtype, 9, dev).requires_grad_(True)
    s = S.moe_sort(x, ids, E)
    check_sorted(s, x, ids, E)
    d = make_x((T * k, K), dtype, 10, dev)
    dx, = torch.autograd.grad(s.rows, x, d)
    want, size = unsort_exact(d, None, s.pos)
    u = half_step(dtype)
    assert ((dx.double() - want).abs() <= u * want.abs() + (1 + u) * k * U24 * size + 1e-7).all()


@gpu
def test_gradients_against_differences(dev):
    """Both operators are linear in each argument, so a difference of two calls is the derivative times
    the step up to the rounding of the calls; inputs are small integers, where all is exact in fp32."""
    T, k, E, K = 6, 3, 4, 40
    g = torch.Generator().manual_seed(3)

    def ints(*shape):
        return torch.randint(-8, 9, shape, generator=g).float().to(dev)

    ids = make_ids(T, k, E, 0.25, 2, dev)
    x, w, c = ints(T, K).requires_grad_(True), ints(T, k).requires_grad_(True), ints(T, K)

    def loss(x, w):
        s = S.moe_sort(x, ids, E)
        return (S.moe_unsort(s.rows * 2, w, s.pos) * c).sum()

    dx, dw = torch.autograd.grad(loss(x, w), (x, w))
    for _ in range(4):
        hx, hw = ints(T, K), ints(T, k)
        with torch.no_grad():
            assert (loss(x + hx, w) - loss(x, w)).item() == (dx * hx).sum().item()
            assert (loss(x, w + hw) - loss(x, w)).item() == (dw * hw).sum().item()


@gpu
def test_only_the_wanted_gradients(dev):
    T, k, E, K = 5, 2, 3, 16
    ids = make_ids(T, k, E, 0.2, 2, dev)
    pos = S.moe_sort(make_x((T, K), torch.float32, 1, dev), ids, E).pos
    rows, w, dy = (make_x(s, torch.float32, i, dev) for i, s in enumerate([(T * k, K), (T, k), (T, K)]))
    r2, w2 = rows.clone().requires_grad_(True), w.clone().requires_grad_(True)
    both = torch.autograd.grad(S.moe_unsort(r2, w2, pos), (r2, w2), dy)
    assert torch.equal(torch.autograd.grad(S.moe_unsort(r2, w, pos), r2, dy)[0], both[0])
    assert torch.equal(torch.autograd.grad(S.moe_unsort(rows, w2, pos), w2, dy)[0], both[1])
    # a gradient that is broadcast (a plain sum's) and one of several uses
    loss = S.moe_unsort(r2, w2, pos).sum()
    loss.backward()
    assert torch.equal(r2.grad, torch.autograd.grad(S.moe_unsort(r2, w2, pos), r2, torch.ones_like(dy))[0])
    with pytest.raises(RuntimeError):
        d, = torch.autograd.grad(S.moe_unsort(r2, w2, pos).sum(), r2, create_graph=True)
        d.sum().backward()


@gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_what_no_route_names_does_not_leak(dev, bad):
    """Rows and weights of routes without an expert are not read: NaN and infinities there change nothing,
    in the sums and in the gradients; a token without any route gives zeros."""
    T, k, E, K = 12, 4, 8, 72
    ids = make_ids(T, k, E, 0.4, 5, dev)
    ids[3] = -1
    pos = torch.from_numpy(plain_order(ids, E)[2]).to(dev)
    rows, w = make_x((T * k, K), torch.float32, 6, dev), make_x((T, k), torch.float32, 7, dev)
    tail, dropped = (~pos[pos < 0]).long(), pos < 0
    dy = make_x((T, K), torch.float32, 8, dev)

    def all_of(rows, w):
        rows, w = rows.clone().requires_grad_(True), w.clone().requires_grad_(True)
        y = S.moe_unsort(rows, w, pos)
        return [y.detach(), *torch.autograd.grad(y, (rows, w), dy)]

    clean = all_of(rows, w)
    rows[tail], w[dropped] = bad, bad
    for a, b in zip(clean, all_of(rows, w)):
        assert torch.equal(a, b)
    assert (clean[0][3] == 0).all() and (clean[1][tail] == 0).all()
    x = make_x((T, K), torch.float32, 9, dev)
    x[3] = bad  # no route reads token 3
    assert torch.isfinite(S.moe_sort(x, ids, E).rows).all()


@gpu
def test_ids_outside_the_experts(dev):
    ids = torch.tensor([[0, 4, -1], [5, 2 ** 31 - 1, -2 ** 31], [3, 3, 3]], dtype=torch.int32, device=dev)
    x = make_x((3, 24), torch.bfloat16, 2, dev)
    check_sorted(S.moe_sort(x, ids, 4), x, ids, 4)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dev, dtype):
    """Rows apart from each other, starting off any vector's alignment, and columns apart."""
    T, k, E, K = 33, 4, 6, 250
    ids = make_ids(T, 2 * k, E, 0.2, 4, dev)[:, ::2]
    for x in (make_x((T, K + 3), dtype, 5, dev)[:, 1:K + 1], make_x((K, T), dtype, 5, dev).t(),
              make_x((1, K), dtype, 5, dev).expand(T, K)):
        s = S.moe_sort(x, ids, E)
        check_sorted(s, x, ids, E)
        rows = make_x((T * k, K + 5), dtype, 6, dev)[:, 3:K + 3]
        w = make_x((T, 2 * k), torch.float32, 7, dev)[:, 1::2]
        assert torch.equal(S.moe_unsort(rows, w, s.pos), S.moe_unsort(rows.contiguous(), w.contiguous(), s.pos))


@gpu
def test_no_tokens(dev):
    x, ids = torch.empty((0, 64), dtype=torch.bfloat16, device=dev), torch.empty((0, 4), dtype=torch.int32, device=dev)
    s = S.moe_sort(x, ids, 7)
    assert s.rows.shape == (0, 64) and s.pos.shape == (0, 4) and (s.offsets == 0).all()
    assert S.moe_unsort(s.rows, torch.empty((0, 4), device=dev), s.pos).shape == (0, 64)


@gpu
def test_offsets_past_32_bits(dev):
    """Rows whose elements and bytes lie past 2^32: the copies, the sums and the gradients reach them."""
    T, k, E, K = 65537, 16, 5, 2056
    ids = make_ids(T, k, E, 0.1, 11, dev)
    x = torch.randn((T, K), device=dev).to(torch.bfloat16)
    s = S.moe_sort(x, ids, E)
    assert s.rows.numel() > 2 ** 31
    _, perm, pos = plain_order(ids, E)
    assert np.array_equal(s.perm.cpu().numpy(), perm) and np.array_equal(s.pos.cpu().numpy(), pos)
    for p in (0, T * k // 2, int(s.offsets[-1]) - 1):
        assert torch.equal(s.rows[p], x[perm[p] // k])
    assert (s.rows[int(s.offsets[-1]):] == 0).all()
    for a in range(0, T * k, 1 << 18):  # in parts, to bound the check's memory
        part = s.perm[a:a + (1 << 18)]
        want = x[torch.where(part >= 0, part, 0).long() // k]
        want[part < 0] = 0
        assert torch.equal(s.rows[a:a + (1 << 18)], want)
    del want
    y = S.moe_unsort(s.rows, None, s.pos)
    n = (s.pos >= 0).sum(1)
    assert torch.equal(y, (x.float() * n[:, None]).to(torch.bfloat16))  # n <= 16 times a bf16 value is exact in fp32
    w = torch.ones((T, k), device=dev, requires_grad=True)
    rows = s.rows.requires_grad_(True)
    drows, = torch.autograd.grad(S.moe_unsort(rows, w, s.pos), rows, x)
    assert torch.equal(drows, s.rows.detach())


@gpu
@pytest.mark.parametrize("routes", [65536, 65537, 64 * 2048, 64 * 2048 + 1, 65 * 2048, 300001, 1 << 22])
@pytest.mark.parametrize("E,cold", [(1, 0.5), (63, 0.0), (64, 0.1), (2048, 0.3)])
def test_order_of_many_routes(dev, routes, E, cold):
    """Chunks few and many, whose counts are added up in one way or the other."""
    ids = make_ids(routes, 1, E, cold, 21, dev)
    x = torch.arange(routes, dtype=torch.float32, device=dev)[:, None]
    check_sorted(S.moe_sort(x, ids, E), x, ids, E)


@gpu
@pytest.mark.parametrize("K,dtype", [(4, torch.float32), (2, torch.bfloat16)])
def test_more_tokens_than_a_launch_takes(dev, K, dtype):
    T, k, E = (1 << 23) + 3, 2, 9
    ids = torch.randint(-1, E, (T, k), dtype=torch.int32, device=dev)
    x = torch.randn((T, K), device=dev).to(dtype).requires_grad_(True)
    s = S.moe_sort(x, ids, E)
    _, order = torch.sort(torch.where(ids >= 0, ids, E).reshape(-1), stable=True)
    hot = ids.reshape(-1)[order] >= 0
    assert torch.equal(s.perm.long(), torch.where(hot, order, ~order))
    want = torch.where(hot[:, None], x.detach()[order // k], 0)
    assert torch.equal(s.rows.detach(), want)
    # integer weights and values: sums of two terms that are exact in every type
    rows = torch.randint(-3, 4, s.rows.shape, device=dev).to(dtype).requires_grad_(True)
    w = torch.randint(-2, 3, (T, k), device=dev).float().requires_grad_(True)
    dy = torch.randint(-3, 4, (T, K), device=dev).to(dtype)
    y = S.moe_unsort(rows, w, s.pos)
    drows, dw = torch.autograd.grad(y, (rows, w), dy)
    at, there = torch.where(s.pos >= 0, s.pos, ~s.pos).long(), (s.pos >= 0)[..., None]
    picked = torch.where(there, rows.detach()[at], 0).float()
    assert torch.equal(y.detach().float(), (picked * w.detach()[..., None]).sum(1))
    assert torch.equal(dw, (picked * dy[:, None].float()).sum(2))
    assert torch.equal(drows[at].float(), torch.where(there, w.detach()[..., None] * dy[:, None].float(), 0))
    dx, = torch.autograd.grad(s.rows, x, rows.detach())
    assert torch.equal(dx.float(), picked.sum(1))


@gpu
def test_repeats_bit_for_bit(dev):
    T, k, E, K = 300, 8, 32, 1000
    ids, x = make_ids(T, k, E, 0.1, 1, dev), make_x((T, K), torch.float32, 2, dev)
    s = S.moe_sort(x, ids, E)
    rows, w = s.rows.detach().requires_grad_(True), make_x((T, k), torch.float32, 3, dev).requires_grad_(True)
    first = None
    for _ in range(5):
        y = S.moe_unsort(rows, w, s.pos)
        now = [y.detach(), *torch.autograd.grad(y, (rows, w), x)]
        first = first or now
        assert all(torch.equal(a, b) for a, b in zip(first, now))


@gpu
@pytest.mark.parametrize("T", [4, 700])
def test_graph_and_streams(dev, T):
    """Two captured graphs replayed between eager calls and on another stream, forward and backward."""
    k, E, K = 8, 64, 520
    ids = [make_ids(T, k, E, 0.2, i, dev) for i in range(2)]
    x = [make_x((T, K), torch.bfloat16, i, dev).requires_grad_(True) for i in range(2)]
    w = [make_x((T, k), torch.float32, 9 + i, dev).requires_grad_(True) for i in range(2)]
    dy = make_x((T, K), torch.bfloat16, 20, dev)

    def step(i):
        s = S.moe_sort(x[i], ids[i], E)
        y = S.moe_unsort(s.rows, w[i], s.pos)
        return [s.rows.detach(), s.offsets, s.perm, s.pos, y.detach(), *torch.autograd.grad(y, (x[i], w[i]), dy)]

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
                x[i].copy_(make_x((T, K), torch.bfloat16, 30 + turn + i, dev))
                ids[i].copy_(make_ids(T, k, E, 0.1 * turn, 40 + turn + i, dev))
        for i in ((0, 1) if turn % 2 else (1, 0)):
            graphs[i].replay()
        if turn == 2:
            torch.cuda.synchronize()
        for i in range(2):
            torch.cuda.synchronize()
            for a, b in zip(outs[i], step(i)):
                assert torch.equal(a, b)
    # eager work on a stream of its own, while the first stream is busy with other inputs
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = step(0)
    b = step(1)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(a, step(0))) and all(torch.equal(p, q) for p, q in zip(b, step(1)))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_sorted_products_with_the_layer_neighbours(dev, dtype):
    """A run as it would be used: the hot cache's slot ids, the sort, products of the sorted rows, silu * mul
    (the library's entry point), products again, back with weights; against 64 bits. One rounding a stage."""
    import kt_prefill_lend_amd.kt_hot_cache as C
    import kt_prefill_lend_amd.kt_w4_vec as W

    T, k, E, hot, H, N, G = 19, 4, 24, 9, 256, 96, 32
    g = torch.Generator().manual_seed(12)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).to(torch.int32).to(dev)
    table = torch.full((E,), -1, dtype=torch.int32)
    table[torch.randperm(E, generator=g)[:hot]] = torch.arange(hot, dtype=torch.int32)
    table = table.to(dev)
    slots, _ = C.route_native(ids, table, torch.where(table >= 0, -1, torch.arange(E, dtype=torch.int32, device=dev)).to(torch.int32),
                              torch.zeros(E, device=dev))
    x = make_x((T, H), dtype, 1, dev)
    w = torch.softmax(make_x((T, k), torch.float32, 2, dev), 1)

    def codes(*shape):
        return torch.randint(0, 256, shape, generator=g, dtype=torch.uint8).to(dev)

    def scales(*shape):
        return (torch.rand(shape, generator=g) * 0.01 + 0.005).to(dtype).to(dev)

    q13, s13 = codes(hot, 2 * N, H // 2), scales(hot, 2 * N, H // G)
    q2, s2 = codes(hot, H, N // 2), scales(hot, H, N // G)
    s = S.moe_sort(x, slots, hot)
    h13 = W.moe_w4_sorted(s.rows, q13, s13, s.offsets, group_size=G)
    h = torch.empty((T * k, N), dtype=dtype, device=dev)
    _lib.check(_lib.lib().ktmi_silu_and_mul(h13.data_ptr(), _lib.dtype_code(dtype), T * k, N, h.data_ptr(),
                                            _lib.stream_ptr(dev)))
    y = S.moe_unsort(W.moe_w4_sorted(h, q2, s2, s.offsets, group_size=G), w, s.pos)
    # the same by the routes' ids, as a decode window calls it
    flat = slots.reshape(-1)
    by_id = W.moe_w4_vec(x, q13, s13, flat, k, group_size=G)
    at = torch.where(s.pos >= 0, s.pos, ~s.pos).reshape(-1).long()
    # the two may sum in another order, which moves a value over a rounding's border now and then
    assert (by_id.double() - h13[at].double()).norm() <= half_step(dtype) * by_id.double().norm()

    def dequant(q, sc):
        v = torch.stack([q & 15, q >> 4], -1).flatten(-2).double() - 8
        return v * sc.double().repeat_interleave(G, -1)

    w13, w2 = dequant(q13, s13), dequant(q2, s2)
    want = torch.zeros((T, H), dtype=torch.float64, device=dev)
    for t in range(T):
        for j in range(k):
            e = int(slots[t, j])
            if e >= 0:
                a = w13[e] @ x[t].double()
                want[t] += w[t, j].double() * (w2[e] @ (a[:N] * torch.sigmoid(a[:N]) * a[N:]))
    # four roundings to the type on the way (gate and up, h, the down product, y), each at most half a
    # step of its value and independent over the sums: the relative distance stays below their sum
    assert (y.double() - want).norm() <= 5 * half_step(dtype) * want.norm()


# ---------------------------------------------------------------- refusals (no GPU)

def test_refusals():
    x, ids = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    for bad_x, bad_ids, n, error in [
            (x, ids.long(), 3, TypeError), (x.double(), ids, 3, TypeError), (x, ids[:3], 3, ValueError),
            (x[0], ids, 3, ValueError), (x, ids.reshape(-1), 3, ValueError), (x, ids, 0, ValueError),
            (x, ids, S.MAX_EXPERTS + 1, ValueError), (x, ids[:, :0], 3, ValueError), (x[:, :0], ids, 3, ValueError),
            (x, ids, 3, ValueError)]:  # the last: not on the GPU
        with pytest.raises(error, match="moe_sort"):
            S.moe_sort(bad_x, bad_ids, n)
    rows, w, pos = torch.zeros(8, 8), torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int32)
    for r, v, p, error in [
            (rows, w, pos.long(), TypeError), (rows, w.double(), pos, TypeError), (rows.double(), w, pos, TypeError),
            (rows[:7], w, pos, ValueError), (rows, w[:3], pos, ValueError), (rows, w.t(), pos, ValueError),
            (rows, w, pos.reshape(-1), ValueError), (rows, w, pos, ValueError)]:
        with pytest.raises(error, match="moe_unsort"):
            S.moe_unsort(r, v, p)


def test_c_refusals():
    """Argument errors of the entry points come before any device work (the pointers are never read)."""
    L = _lib.lib()
    p = 4096

    def sort(x=p, dt=2, stride=8, cols=8, ids=p, T=4, k=2, E=3, rows=p, off=p, perm=p, pos=p, ws=p, n=1 << 20):
        return L.ktmi_moe_sort(x, dt, stride, cols, ids, T, k, E, rows, off, perm, pos, ws, n, 0)

    assert L.ktmi_moe_sort_workspace(70000, 2, 3) > 0 and L.ktmi_moe_sort_workspace(0, 2, 3) == 0
    for kw, code in [(dict(dt=3), -1), (dict(cols=0), -1), (dict(cols=1 << 25, stride=1 << 25), -1), (dict(T=-1), -1),
                     (dict(k=0), -1), (dict(T=1 << 31), -1), (dict(T=1 << 62, k=4), -1), (dict(E=0), -1),
                     (dict(E=S.MAX_EXPERTS + 1), -1), (dict(x=0), -1), (dict(ids=0), -1), (dict(off=0), -1),
                     (dict(perm=0), -1), (dict(pos=0), -1), (dict(x=p + 1), -1), (dict(rows=p + 1), -1),
                     (dict(stride=7), -1), (dict(T=70000, ws=0), -4), (dict(T=70000, n=1), -4)]:
        assert sort(**kw) == code and b"moe_sort" in L.ktmi_last_error(), kw

    def unsort(rows=p, dt=2, stride=8, cols=8, w=p, pos=p, T=4, k=2, y=p):
        return L.ktmi_moe_unsort(rows, dt, stride, cols, w, pos, T, k, y, 0)

    for kw in [dict(dt=7), dict(cols=0), dict(T=-1), dict(k=0), dict(rows=0), dict(pos=0), dict(y=0), dict(stride=7),
               dict(y=p + 1), dict(T=1 << 31)]:
        assert unsort(**kw) == -1 and b"moe_unsort" in L.ktmi_last_error(), kw
    assert unsort(T=0) == 0

    def grad(dy=p, ds=8, rows=p, rs=8, dt=2, cols=8, w=p, pos=p, T=4, k=2, drows=p, dw=p):
        return L.ktmi_moe_unsort_grad(dy, ds, rows, rs, dt, cols, w, pos, T, k, drows, dw, 0)

    for kw in [dict(dt=7), dict(cols=0), dict(dy=0), dict(rows=0), dict(pos=0), dict(ds=7), dict(rs=7),
               dict(drows=p + 1), dict(k=0)]:
        assert grad(**kw) == -1 and b"moe_unsort_grad" in L.ktmi_last_error(), kw
    assert grad(T=0) == 0 and grad(drows=0, dw=0) == 0


def test_c_refuses_more_routes_a_token_than_a_block_takes():
    L = _lib.lib()
    p, k = 4096, 65536
    assert L.ktmi_moe_sort(p, 2, 8, 8, p, 1, k, 3, p, p, p, p, p, 1 << 30, 0) == -1 and b"65535" in L.ktmi_last_error()
    assert L.ktmi_moe_unsort(p, 2, 8, 8, p, p, 1, k, p, 0) == -1 and b"65535" in L.ktmi_last_error()
    assert L.ktmi_moe_unsort_grad(p, 8, p, 8, 2, 8, p, p, 1, k, p, p, 0) == -1 and b"65535" in L.ktmi_last_error()


# ---------------------------------------------------------------- what torch would record without the kernels

def calls_of_tensors(dev):
    """name -> (call, its tensors that could carry a derivative); sizes are the smallest."""
    x, rows = torch.ones(2, 4, device=dev), torch.ones(4, 4, device=dev)
    ids, w = torch.zeros(2, 2, dtype=torch.int32, device=dev), torch.ones(2, 2, device=dev)
    pos = torch.arange(4, dtype=torch.int32, device=dev).reshape(2, 2)
    return {"moe_sort": (lambda x: S.moe_sort(x, ids, 3).rows, (x,)),
            "moe_unsort": (lambda rows, w: S.moe_unsort(rows, w, pos), (rows, w))}


@pytest.mark.filterwarnings("ignore:Converting a tensor")
@pytest.mark.parametrize("name", ["moe_sort", "moe_unsort"])
def test_records_without_the_kernels_are_refused(monkeypatch, name):
    monkeypatch.setattr(S, "_check_gpu", lambda *a: None)
    check_refused_records(name, *calls_of_tensors("cpu")[name])


@gpu
@pytest.mark.filterwarnings("ignore:Converting a tensor")
@pytest.mark.parametrize("name", ["moe_sort", "moe_unsort"])
def test_records_without_the_kernels_are_refused_on_the_gpu(dev, name):
    from torch.autograd import forward_ad

    call, tensors = calls_of_tensors(dev)[name]
    want = call(*tensors)
    check_refused_records(name, call, tensors)
    with forward_ad.dual_level():  # a level by itself changes nothing
        assert torch.equal(call(*tensors), want)
        # a tangent of what comes back through the gradient
        leaves = [t.clone().requires_grad_(True) for t in tensors]
        y = call(*leaves)
        with pytest.raises(NotImplementedError, match=f"{name}'s gradient"):
            torch.autograd.grad(y, leaves, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))
    assert torch.equal(call(*tensors), want)


# ---------------------------------------------------------------- few routes a token, wide rows

def test_workspace_follows_the_order_work():
    """Few routes a token make every block of the one launch dearer: such calls may take the chunked order, so
    they have its workspace; decode-sized calls have none."""
    L = _lib.lib()
    for T, k in [(1, 8), (64, 8), (77, 10), (512, 1), (0, 4)]:
        assert L.ktmi_moe_sort_workspace(T, k, 256) == 0, (T, k)
    for T, k in [(4096, 1), (2048, 2), (1025, 1), (1024, 4), (4097, 1), (1, 4096), (3, 17)]:
        assert L.ktmi_moe_sort_workspace(T, k, 256) >= 4 * 257 * 2, (T, k)
    assert L.ktmi_moe_sort(4096, 2, 8, 8, 4096, 4096, 1, 256, 4096, 4096, 4096, 4096, None, 0, 0) == -4


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,E,K,cold", [
    (4096, 1, 256, 40, 0.2), (4095, 1, 2048, 2050, 0.0), (2048, 2, 300, 1030, 0.1), (1025, 1, 5, 9000, 0.3),
    (1024, 4, 129, 7001, 0.0), (513, 1, 16, 4100, 0.1), (512, 8, 64, 5000, 0.2), (256, 16, 33, 3000, 0.0),
    (200, 20, 40, 2100, 0.1), (400, 10, 40, 2100, 0.1), (1, 4096, 2000, 100, 0.1), (3, 17, 5, 50, 0.3)])
def test_sort_few_routes_a_token(dev, T, k, E, K, cold, dtype):
    ids, x = make_ids(T, k, E, cold, T + K, dev), make_x((T, K), dtype, 3, dev)
    check_sorted(S.moe_sort(x, ids, E), x, ids, E)


@gpu
@pytest.mark.parametrize("T,k", [(1, 8), (512, 1), (513, 1), (1448, 1), (1449, 1), (2048, 2), (4096, 1), (512, 8), (1365, 3),
                                 (1, 17), (240, 17), (1, 4096), (256, 16)])
def test_order_alone(dev, T, k):
    """Without rows, with exactly the workspace that the query names."""
    E, L = 130, _lib.lib()
    ids = make_ids(T, k, E, 0.1, T, dev)
    need = L.ktmi_moe_sort_workspace(T, k, E)
    off, perm, pos = (torch.full((n,), 77, dtype=torch.int32, device=dev) for n in (E + 1, T * k, T * k))
    ws = torch.full((need + 64,), 93, dtype=torch.uint8, device=dev)
    _lib.check(L.ktmi_moe_sort(None, 2, 0, 8, ids.data_ptr(), T, k, E, None, off.data_ptr(), perm.data_ptr(), pos.data_ptr(),
                               ws.data_ptr(), need, _lib.stream_ptr(dev)))
    for got, want in zip((off, perm, pos.reshape(T, k)), plain_order(ids, E)):
        assert np.array_equal(got.cpu().numpy(), want)
    assert (ws[need:] == 93).all()


def test_tensors_without_memory_are_refused():
    """Where the library takes a null pointer for an argument left out, a wrapper's must not pass for one."""
    from helpers import wrapped

    x, w, ids = torch.ones(2, 4), torch.ones(2, 2), torch.zeros(2, 2, dtype=torch.int32)
    rows, pos = torch.ones(4, 4), torch.arange(4, dtype=torch.int32).reshape(2, 2)
    with pytest.raises(TypeError, match="moe_sort: a Wrapped"):
        S._launch_sort(0, wrapped(x), ids, 3)
    with pytest.raises(TypeError, match="moe_unsort: a Wrapped"):
        S._launch_unsort(0, rows, wrapped(w), pos)
    for dy, v in [(wrapped(x), w), (x, wrapped(w))]:
        with pytest.raises(TypeError, match="moe_unsort's gradient: a Wrapped"):
            S._launch_unsort_grad(0, dy, rows, v, pos, True, True)


# ---------------------------------------------------------------- compiled, checkpointed, from several threads

def a_run(dev, ids, E):
    """A sort, an operation on the rows and the way back, as a function of (x, w), with its gradients."""
    def forward(x, w):
        s = S.moe_sort(x * 1, ids, E)
        return S.moe_unsort(s.rows * 2, w, s.pos) + 1

    def all_of(fn, x, w):
        y = fn(x, w)
        return [y.detach(), *torch.autograd.grad(y, (x, w), torch.ones_like(y))]

    return forward, all_of


@gpu
@pytest.mark.parametrize("how", ["eager", "aot_eager", "checkpoint"])
def test_compiled_and_checkpointed(dev, how):
    T, k, E, K = 77, 8, 16, 256
    ids = make_ids(T, k, E, 0.1, 1, dev)
    x, w = make_x((T, K), torch.bfloat16, 2, dev).requires_grad_(True), make_x((T, k), torch.float32, 3, dev).requires_grad_(True)
    forward, all_of = a_run(dev, ids, E)
    want = all_of(forward, x, w)
    if how == "checkpoint":
        from torch.utils.checkpoint import checkpoint

        other = lambda x, w: checkpoint(forward, x, w, use_reentrant=False)  # noqa: E731
    else:
        torch._dynamo.reset()
        other = torch.compile(forward, backend=how)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(want, all_of(other, x, w)))


@gpu
def test_threads(dev):
    """Calls of several host threads, each on a stream of its own, with refusals between them."""
    import threading

    import kt_prefill_lend_amd.kt_w4_vec as W

    T, k, E, K, N = 77, 8, 16, 256, 128
    ids = make_ids(T, k, E, 0.1, 1, dev)
    x, w = make_x((T, K), torch.bfloat16, 2, dev).requires_grad_(True), make_x((T, k), torch.float32, 3, dev).requires_grad_(True)
    g = torch.Generator().manual_seed(4)
    q = torch.randint(0, 256, (E, N, K // 2), generator=g, dtype=torch.uint8).to(dev)
    sc = torch.rand((E, N, K // 128), generator=g).to(torch.bfloat16).to(dev)
    forward, all_of = a_run(dev, ids, E)

    def step():
        with torch.no_grad():
            y = W.moe_w4_vec(x, q, sc, ids.reshape(-1), k)
        return [y, *all_of(forward, x, w)]

    want, wrong = step(), []
    torch.cuda.synchronize()

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for n in range(20):
                    got = step()
                    stream.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(want, got)):
                        wrong.append((i, n))
                    with pytest.raises(ValueError, match="4000 experts"):
                        S.moe_sort(x.detach(), ids, 4000)
        except BaseException as e:  # a thread's failure is the test's
            wrong.append((i, repr(e)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong
