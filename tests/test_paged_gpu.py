"""The paged key/value cache: append and one-token attention against the formulas in f64.

Every cache here holds NaN and infinities wherever no live position is, so a
kernel that reads past a length, or multiplies a masked value by zero, shows.

Tolerances, from the arithmetic. A result rounded to type T is off by at most
eps(T)/2 of itself. Append: the fraction of a turn is rounded to f32 (2^-24 of
at most pi) and sincospif is good to 2 ulp, so each product is off by less than
2^-21 and the rotated value by less than 2^-20 (|x0| + |x1|). Attention: a score
sums D products in f32, off by D 2^-24 sum|q k| scale at most; that and the
exponential's 2^-21 move each probability by as much of itself (twice, through
the sum of the probabilities); the sums over len keys add len 2^-24, and the bf16
kernel carries probabilities as two bf16 numbers, off by 2^-16 of themselves.
"""
import threading

import pytest
import torch

import haelixe_b200 as hx
from haelixe_b200 import _native as N

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
DT = [pytest.param(F32, id="f32"), pytest.param(BF16, id="bf16")]
BASE = 10000.0


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _garbage(shape, dtype):
    """NaN, +inf and -inf in turn."""
    n = 1
    for s in shape:
        n *= s
    t = torch.tensor([float("nan"), float("inf"), float("-inf")], device="cuda", dtype=dtype)
    return t.repeat(-(-n // 3))[:n].view(shape)


def _filled(seed, dtype, lens, page, hk, dim, heads_first=False, spare=2, columns=None):
    """A cache with random values at the live positions alone, its table, and the values as lists of [len, hk, dim]."""
    g = _gen(seed)
    need = [-(-max(n, 0) // page) for n in lens]
    columns = columns or max(1, max(need))
    pages = sum(need) + spare
    perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), columns), -12345, dtype=torch.int32, device="cuda")  # unused entries: no page
    shape = (pages, hk, page, dim) if heads_first else (pages, page, hk, dim)
    kc, vc = _garbage(shape, dtype), _garbage(shape, dtype)
    if heads_first:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    ks, vs, at = [], [], 0
    for s, n in enumerate(lens):
        table[s, :need[s]] = perm[at:at + need[s]]
        at += need[s]
        n = max(n, 0)
        k, v = (torch.randn(n, hk, dim, generator=g, device="cuda", dtype=dtype) for _ in range(2))
        j = torch.arange(n, device="cuda")
        rows = table[s].long()[j // page]
        kc[rows, j % page], vc[rows, j % page] = k, v
        ks.append(k)
        vs.append(v)
    return hx.PagedKVCache(kc, vc, table), ks, vs


def _reference(q, ks, vs, scale):
    """f64 o and lse of each sequence, and the bound on the error besides the rounding of o."""
    n, hq, dim = q.shape
    o = torch.zeros(n, hq, dim, dtype=torch.float64, device="cuda")
    lse = torch.full((n, hq), float("-inf"), dtype=torch.float64, device="cuda")
    off, off_lse = torch.zeros_like(o), torch.zeros_like(lse)
    for s in range(n):
        k, v = ks[s].double(), vs[s].double()
        m = k.shape[0]
        if m == 0:
            continue
        group = hq // k.shape[1]
        k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
        sc = torch.einsum("hd,lhd->hl", q[s].double(), k) * scale
        p = torch.softmax(sc, -1)
        o[s] = torch.einsum("hl,lhd->hd", p, v)
        lse[s] = torch.logsumexp(sc, -1)
        ds = (dim + 4) * 2.0 ** -24 * (torch.einsum("hd,lhd->hl", q[s].double().abs(), k.abs()) * abs(scale)).amax(-1) + 2.0 ** -20
        rel = 2 * ds + m * 2.0 ** -24 + (2.0 ** -16 if q.dtype == BF16 else 0.0)
        off[s] = rel[:, None] * torch.einsum("hl,lhd->hd", p, v.abs())
        off_lse[s] = ds + m * 2.0 ** -24 + 2.0 ** -22 * lse[s].abs()
    return o, lse, off, off_lse


def _check(q, ks, vs, scale, o, lse):
    ro, rl, off, off_lse = _reference(q, ks, vs, scale)
    err = (o.double() - ro).abs()
    assert torch.isfinite(o).all()
    assert (err <= torch.finfo(q.dtype).eps / 2 * (ro.abs() + off) + off).all(), float((err - off).max())
    empty = rl == float("-inf")
    assert (lse[empty] == float("-inf")).all() and (o.double()[empty] == 0).all()
    assert ((lse.double() - rl).abs()[~empty] <= off_lse[~empty] + 2.0 ** -24 * rl.abs()[~empty]).all()


def _lens(*a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


EDGES = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("hk,group,dim,page", [
    (1, 1, 64, 16), (2, 4, 128, 16), (3, 1, 128, 24), (2, 3, 80, 1), (2, 8, 64, 7), (1, 5, 8, 64), (2, 16, 128, 32),
    (1, 13, 64, 16), (1, 20, 128, 8), (2, 2, 256, 16), (1, 11, 192, 16), (4, 7, 96, 128), (1, 33, 40, 16),
])
def test_attention_at_the_edges_of_pages_and_tiles(dtype, heads_first, hk, group, dim, page):
    cache, ks, vs = _filled(hk * 1000 + dim + page, dtype, EDGES, page, hk, dim, heads_first)
    q = torch.randn(len(EDGES), hk * group, dim, generator=_gen(5), device="cuda", dtype=dtype)
    o, lse = hx.paged_attention(cache, q, _lens(*EDGES), dim ** -0.5)
    _check(q, ks, vs, dim ** -0.5, o, lse)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("lens", [[20011], [5, 17000, 0, 0, 3, 64, 9000], [0, 0, 0], [1] * 700, [0] * 300 + [40] * 3])
def test_attention_split_over_long_and_many_sequences(dtype, lens):
    cache, ks, vs = _filled(11, dtype, lens, 16, 2, 64)
    q = torch.randn(len(lens), 8, 64, generator=_gen(6), device="cuda", dtype=dtype)
    o, lse = hx.paged_attention(cache, q, _lens(*lens), 0.125)
    _check(q, ks, vs, 0.125, o, lse)


@pytest.mark.parametrize("dtype", DT)
def test_attention_is_the_same_each_time_and_close_to_alone(dtype):
    lens = [777, 4000, 64]
    cache, ks, vs = _filled(12, dtype, lens, 16, 4, 128)
    q = torch.randn(3, 16, 128, generator=_gen(7), device="cuda", dtype=dtype)
    a = hx.paged_attention(cache, q, _lens(*lens), 0.1)
    for _ in range(3):
        b = hx.paged_attention(cache, q, _lens(*lens), 0.1)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
@pytest.mark.parametrize("dtype", DT)
def test_attention_scales(dtype, scale):
    """A scale of 4 spreads the scores over hundreds: the maximum moves, most probabilities vanish."""
    lens = [500, 33]
    cache, ks, vs = _filled(13, dtype, lens, 16, 2, 64)
    q = torch.randn(2, 4, 64, generator=_gen(8), device="cuda", dtype=dtype)
    o, lse = hx.paged_attention(cache, q, _lens(*lens), scale)
    _check(q, ks, vs, scale, o, lse)


@pytest.mark.parametrize("dtype", DT)
def test_attention_of_growing_scores(dtype):
    """Each key scores higher than the one before, so the running maximum moves all the way."""
    n, dim = 600, 64
    cache, ks, vs = _filled(14, dtype, [n], 16, 1, dim)
    j = torch.arange(n, device="cuda")
    k = torch.zeros(n, 1, dim, device="cuda", dtype=dtype)
    k[:, 0, 0] = (j / 4).to(dtype)
    cache.k[cache.block_table[0].long()[j // 16], j % 16] = k
    q = torch.ones(1, 3, dim, device="cuda", dtype=dtype)
    o, lse = hx.paged_attention(cache, q, _lens(n), 1.0)
    _check(q, [k], vs, 1.0, o, lse)


@pytest.mark.parametrize("dtype", DT)
def test_values_that_are_not_finite(dtype):
    """A NaN or an infinite score inside the length gives what the formula gives; -inf scores weigh nothing."""
    lens = [200, 200, 200, 200]
    cache, ks, vs = _filled(15, dtype, lens, 16, 1, 64)
    t = cache.block_table.long()
    q = torch.zeros(4, 2, 64, device="cuda", dtype=dtype)
    q[:, :, 0] = 1.0
    inf = float("inf")
    for s, (at, value) in enumerate([(150, float("nan")), (150, inf), (150, -inf), (None, -inf)]):
        for p in ([at] if at is not None else range(200)):
            cache.k[t[s, p // 16], p % 16, 0, 0] = value
            ks[s][p, 0, 0] = value
    # The other products with an infinity are 0 * x; only element 0 of q is not zero.
    o, lse = hx.paged_attention(cache, q, _lens(*lens), 1.0)
    assert torch.isnan(o[0]).all() and torch.isnan(lse[0]).all()
    assert torch.isnan(o[1]).all()
    assert torch.isnan(o[3]).all() and (lse[3] == -inf).all()
    keep = torch.arange(200, device="cuda") != 150
    ro, rl, off, _ = _reference(q[2:3], [ks[2][keep]], [vs[2][keep]], 1.0)
    err = (o[2:3].double() - ro).abs()
    assert (err <= torch.finfo(dtype).eps / 2 * (ro.abs() + off) + off).all()


@pytest.mark.parametrize("dtype", DT)
def test_bad_pages_and_lengths(dtype):
    lens = [100, 100, 100, 100, 100]
    cache, ks, vs = _filled(16, dtype, lens, 16, 2, 64)
    q = torch.randn(5, 4, 64, generator=_gen(9), device="cuda", dtype=dtype)
    good, good_lse = hx.paged_attention(cache, q, _lens(*lens), 0.125)
    cache.block_table[1, 3] = -1
    cache.block_table[2, 6] = cache.k.shape[0]  # holds positions 96..99
    o, lse = hx.paged_attention(cache, q, _lens(100, 100, 100, 113, -7), 0.125)
    for s in (1, 2, 3):
        assert torch.isnan(o[s]).all() and torch.isnan(lse[s]).all()
    assert (o[4] == 0).all() and (lse[4] == float("-inf")).all()
    _check(q[:1], ks[:1], vs[:1], 0.125, o[:1], lse[:1])
    # The same entries past the length are not looked at.
    o, lse = hx.paged_attention(cache, q, _lens(100, 48, 96, 100, 100), 0.125)
    _check(q, [k[:n] for k, n in zip(ks, (100, 48, 96, 100, 100))],
           [v[:n] for v, n in zip(vs, (100, 48, 96, 100, 100))], 0.125, o, lse)


def test_strided_queries_and_outputs():
    lens = [70, 5]
    cache, ks, vs = _filled(17, BF16, lens, 16, 2, 64)
    qkv = torch.randn(2, 3, 8, 64, generator=_gen(10), device="cuda", dtype=BF16)
    q = qkv[:, 1]
    wide = torch.full((2, 8, 96), 7.0, device="cuda", dtype=BF16)
    o, lse = hx.paged_attention(cache, q, _lens(*lens), 0.125, out=wide[:, :, 16:80])
    _check(q, ks, vs, 0.125, o, lse)
    assert (wide[:, :, :16] == 7).all() and (wide[:, :, 80:] == 7).all()


def test_shared_pages():
    """Two sequences that share their first pages (a common prompt)."""
    cache, ks, vs = _filled(18, BF16, [64, 64], 16, 2, 64)
    cache.block_table[1, :2] = cache.block_table[0, :2]
    ks[1], vs[1] = torch.cat([ks[0][:32], ks[1][32:]]), torch.cat([vs[0][:32], vs[1][32:]])
    q = torch.randn(2, 2, 64, generator=_gen(11), device="cuda", dtype=BF16)
    _check(q, ks, vs, 0.125, *hx.paged_attention(cache, q, _lens(64, 64), 0.125))


def test_offsets_past_32_bits():
    """A cache of more than 2^32 bytes and 2^31 elements, used at its far end."""
    pages, page, hk, dim = 9000, 64, 32, 128  # 2.36e9 elements
    kc, vc = (torch.empty(pages, page, hk, dim, device="cuda", dtype=BF16) for _ in range(2))
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32, device="cuda")
    cache = hx.PagedKVCache(kc, vc, table)
    n = 150
    k, v = (torch.randn(n, hk, dim, generator=_gen(s), device="cuda", dtype=BF16) for s in (1, 2))
    seq, pos = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda")
    hx.paged_append(cache, k, v, seq, pos)
    assert torch.equal(kc[pages - 1], k[:64]) and torch.equal(vc[3], v[64:128]) and torch.equal(kc[pages - 2, :22], k[128:])
    q = torch.randn(1, hk, dim, generator=_gen(3), device="cuda", dtype=BF16)
    _check(q, [k], [v], 0.1, *hx.paged_attention(cache, q, _lens(n), 0.1))


def _rotated(x, pos, base=BASE):
    d = x.shape[-1]
    ang = pos.double()[:, None] * base ** (-torch.arange(0, d, 2, device=x.device, dtype=torch.float64) / d)
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    a, b = x.double()[..., 0::2], x.double()[..., 1::2]
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2), (a.abs() + b.abs()).repeat_interleave(2, -1)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("hk,hq,dim,page,heads_first", [(1, 1, 8, 1, False), (4, 12, 128, 16, False), (3, 3, 80, 24, True),
                                                       (2, 32, 256, 64, True), (8, 0, 64, 16, False)])
@pytest.mark.parametrize("rope", [None, BASE, 500000.0])
def test_append(dtype, hk, hq, dim, page, heads_first, rope):
    """Tokens of three sequences in mixed order, positions up to the end of the table, with padding."""
    g = _gen(21)
    columns = 7
    table = torch.randperm(30, generator=g, device="cuda")[:3 * columns].to(torch.int32).view(3, columns)
    shape = (30, hk, page, dim) if heads_first else (30, page, hk, dim)
    kc, vc = (torch.full(shape, 3.0, device="cuda", dtype=dtype) for _ in range(2))
    if heads_first:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    want_k, want_v = kc.double(), vc.double()
    last = columns * page - 1
    seq = _lens(0, 2, -1, 1, 2, -5, 0)
    pos = _lens(0, last, 4, min(17, last), 0, 0, last)
    T = 7
    k, v = (torch.randn(T, hk, dim, generator=g, device="cuda", dtype=dtype) for _ in range(2))
    q = torch.randn(T, hq, dim, generator=g, device="cuda", dtype=dtype) if hq else None
    out = torch.full((T, hq, dim), 9.0, device="cuda", dtype=dtype) if hq else None
    got = hx.paged_append(hx.PagedKVCache(kc, vc, table), k, v, seq, pos, rope_base=rope, q=q, out_q=out)
    assert got is out
    rk, mag = (_rotated(k, pos, rope) if rope else (k.double(), torch.zeros_like(k.double())))
    tol = torch.full_like(want_k, 0.0)
    for t in range(T):
        if seq[t] >= 0:
            at = (table[seq[t], pos[t] // page].long(), pos[t].long() % page)
            want_k[at], want_v[at] = rk[t], v[t].double()
            tol[at] = torch.finfo(dtype).eps / 2 * rk[t].abs() * (1 if rope else 0) + 2.0 ** -20 * mag[t]
    assert ((kc.double() - want_k).abs() <= tol).all()
    assert torch.equal(vc.double(), want_v)
    if hq:
        rq, mag = (_rotated(q, pos, rope) if rope else (q.double(), torch.zeros_like(q.double())))
        live = seq >= 0
        tol = torch.finfo(dtype).eps / 2 * rq.abs() * (1 if rope else 0) + 2.0 ** -20 * mag
        assert ((out.double() - rq).abs() <= tol)[live].all()
        assert (out[~live] == 9).all()  # padding rows are left as they were


def test_append_agrees_with_the_rotation_of_whole_sequences():
    """Positions 0..S-1 give what rope_forward gives, within the angle error of its f32 product (S 2^-24 twice over)."""
    S, H, D = 64, 2, 64
    x = torch.randn(S, H, D, generator=_gen(30), device="cuda")
    table = torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4)
    cache = hx.PagedKVCache.allocate(4, 16, H, D, table, dtype=F32)
    q = hx.paged_append(cache, x, x, torch.zeros(S, dtype=torch.int32, device="cuda"),
                        torch.arange(S, dtype=torch.int32, device="cuda"), rope_base=BASE, q=x)
    want = hx.rope_forward(x.transpose(0, 1), BASE).transpose(0, 1)
    mag = (x[..., 0::2].abs() + x[..., 1::2].abs()).repeat_interleave(2, -1)
    # freq off by 2 ulp of powf and the product by half an ulp of the angle: 2.5 S 2^-23.
    assert ((q - want).abs() <= (2.5 * S * 2.0 ** -23 + 2.0 ** -19) * mag).all()
    assert torch.equal(cache.k.view(S, H, D), q) and torch.equal(cache.v.view(S, H, D), x)


@pytest.mark.parametrize("dtype", DT)
def test_append_at_far_positions(dtype):
    """Positions of 10^9: the table alone is that wide, one page is in memory."""
    page, columns, D = 1 << 20, 2000, 128
    table = torch.zeros(1, columns, dtype=torch.int32, device="cuda")
    kc = torch.zeros(1, page, 1, D, device="cuda", dtype=dtype)
    vc = torch.zeros_like(kc)
    pos = _lens(1_000_000_007, 999_999_999, (1 << 20) * 2000 - 1)
    x = torch.randn(3, 1, D, generator=_gen(31), device="cuda", dtype=dtype)
    q = hx.paged_append(hx.PagedKVCache(kc, vc, table), x, x, _lens(0, 0, 0), pos, rope_base=500000.0, q=x)
    want, mag = _rotated(x, pos, 500000.0)
    # The frequency is good to 2^-49 or so in both, times 2^31 positions: 2^-18 radians.
    tol = torch.finfo(dtype).eps / 2 * want.abs() + (2.0 ** -18 + 2.0 ** -20) * mag
    assert ((q.double() - want).abs() <= tol).all()
    assert torch.equal(kc[0, pos.long() % page], q)


def test_append_without_a_slot():
    table = torch.tensor([[0, 99, -3]], dtype=torch.int32, device="cuda")
    cache = hx.PagedKVCache.allocate(2, 16, 1, 64, table)
    x = torch.randn(7, 1, 64, generator=_gen(32), device="cuda", dtype=BF16)
    seq, pos = _lens(0, 0, 0, 0, 0, 1, 7), _lens(15, 16, 32, 48, -1, 0, 0)
    q = hx.paged_append(cache, x, x, seq, pos, q=x)
    assert torch.equal(q[0], x[0]) and torch.isnan(q[1:]).all()
    want = torch.zeros_like(cache.k)
    want[0, 15] = x[0]
    assert torch.equal(cache.k, want) and torch.equal(cache.v, want)


@pytest.mark.parametrize("dtype", DT)
def test_append_from_unaligned_and_strided_rows(dtype):
    """Rows cut from a fused projection, at an odd element offset; q rotated in place."""
    T, H, D = 5, 2, 64
    base = torch.randn(T, 3 * H * D + 1, generator=_gen(33), device="cuda", dtype=dtype)
    q, k, v = base[:, 1:].unflatten(1, (3, H, D)).unbind(1)
    before = base.clone()
    q0, k0, v0 = before[:, 1:].unflatten(1, (3, H, D)).unbind(1)
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    caches = [hx.PagedKVCache.allocate(1, 16, H, D, table, dtype=dtype) for _ in range(2)]
    zero = torch.zeros_like(pos)
    assert hx.paged_append(caches[0], k, v, zero, pos, rope_base=BASE, q=q, out_q=q) is q
    want = hx.paged_append(caches[1], k0.contiguous(), v0.contiguous(), zero, pos, rope_base=BASE, q=q0.contiguous())
    assert torch.equal(q, want) and torch.equal(caches[0].k, caches[1].k) and torch.equal(caches[0].v, caches[1].v)
    assert torch.equal(base[:, 0], before[:, 0]) and torch.equal(k, k0) and torch.equal(v, v0)


def test_empty_calls():
    table = torch.zeros(0, 4, dtype=torch.int32, device="cuda")
    cache = hx.PagedKVCache.allocate(2, 16, 2, 64, table)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    x = torch.zeros(0, 2, 64, device="cuda", dtype=BF16)
    assert hx.paged_append(cache, x, x, none, none, rope_base=BASE, q=x).shape == (0, 2, 64)
    o, lse = hx.paged_attention(cache, x, none, 1.0)
    assert o.shape == (0, 2, 64) and lse.shape == (0, 2)


def _step(cache, q, k, v, seq, pos, lens):
    q = hx.paged_append(cache, k, v, seq, pos, rope_base=BASE, q=q)
    return hx.paged_attention(cache, q, lens, 0.125)


def test_graphs_and_streams():
    """Two captured decode steps of different shapes, replayed at once on two streams with new inputs each time."""
    steps = []
    for n, hk, hq, dim in ((3, 2, 8, 64), (5, 4, 4, 128)):
        lens = [400 + 37 * i for i in range(n)]
        cache, ks, vs = _filled(40 + n, BF16, lens, 16, hk, dim, columns=40)
        cache.block_table[cache.block_table < 0] = 0
        st = dict(cache=cache, q=torch.zeros(n, hq, dim, device="cuda", dtype=BF16),
                  k=torch.zeros(n, hk, dim, device="cuda", dtype=BF16), v=torch.zeros(n, hk, dim, device="cuda", dtype=BF16),
                  seq=torch.arange(n, dtype=torch.int32, device="cuda"), pos=_lens(*lens) - 1, lens=_lens(*lens))
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            _step(**st)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = _step(**st)
        steps.append((st, graph, out, stream))
    for turn in range(4):
        for i, (st, _, _, _) in enumerate(steps):
            for name in "qkv":
                st[name].copy_(torch.randn(st[name].shape, generator=_gen(turn * 10 + i), device="cuda", dtype=BF16))
            st["lens"] -= 50
            st["pos"] -= 50
        torch.cuda.synchronize()
        for _, graph, _, stream in steps:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for st, _, out, _ in steps:
            got = [t.clone() for t in out]
            want = _step(**st)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_calls_from_several_threads():
    work = []
    for i in range(3):
        cache, ks, vs = _filled(50 + i, BF16, [300 + 500 * i, 20], 16, 2, 64)
        work.append((cache, ks, vs, torch.randn(2, 4, 64, generator=_gen(i), device="cuda", dtype=BF16),
                     _lens(300 + 500 * i, 20)))
    torch.cuda.synchronize()
    found = [None] * 3

    def go(i):
        cache, ks, vs, q, lens = work[i]
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(50):
                r = hx.paged_attention(cache, q, lens, 0.125)
            stream.synchronize()
        found[i] = r

    threads = [threading.Thread(target=go, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for (cache, ks, vs, q, lens), r in zip(work, found):
        _check(q, ks, vs, 0.125, *r)


def test_refusals():
    table = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    k = torch.zeros(4, 16, 2, 64, device="cuda", dtype=BF16)
    cache = hx.PagedKVCache(k, k.clone(), table)
    lens = _lens(1, 1)
    q = torch.zeros(2, 4, 64, device="cuda", dtype=BF16)
    x = torch.zeros(2, 2, 64, device="cuda", dtype=BF16)
    for bad in (lambda: hx.PagedKVCache(k.half(), k.half(), table), lambda: hx.PagedKVCache(k, k, table.long()),
                lambda: hx.paged_attention(cache, q, lens.long(), 1.0),
                lambda: hx.paged_append(cache, x, x, lens.long(), lens)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: hx.PagedKVCache(k, k[:3], table), lambda: hx.PagedKVCache(k, k.float(), table),
                lambda: hx.PagedKVCache(k, k.transpose(0, 1).contiguous().transpose(0, 1), table),
                lambda: hx.PagedKVCache(k.transpose(2, 3), k.transpose(2, 3), table),
                lambda: hx.PagedKVCache(k, k, table.t()),
                lambda: hx.paged_attention(cache, q[:1], lens, 1.0), lambda: hx.paged_attention(cache, q.float(), lens, 1.0),
                lambda: hx.paged_attention(cache, q, lens[:1], 1.0),
                lambda: hx.paged_attention(cache, q, lens, 1.0, out=q[:, :2]),
                lambda: hx.paged_attention(cache, q, lens, 1.0, lse=torch.zeros(2, 4, device="cuda", dtype=BF16)),
                lambda: hx.paged_append(cache, q, q, lens, lens), lambda: hx.paged_append(cache, x, x, lens, lens, rope_base=0.0),
                lambda: hx.paged_append(cache, x, x, lens, lens, out_q=q),
                lambda: hx.paged_append(cache, x, x.cpu(), lens, lens)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: hx.paged_attention(cache, q[:, :3], lens, 1.0), lambda: hx.paged_attention(cache, q, lens, float("nan")),
                lambda: hx.paged_append(cache, x, x, lens, lens, rope_base=float("inf")),
                lambda: hx.PagedKVCache(k[..., :60], k[..., :60], table),
                lambda: hx.PagedKVCache(*(torch.zeros(4, 16, 2, 264, device="cuda", dtype=BF16) for _ in range(2)), table)):
        with pytest.raises(N.HxError):
            bad()
    unaligned = torch.zeros(2 * 4 * 64 + 1, device="cuda", dtype=BF16)[1:].view(2, 4, 64)
    with pytest.raises(N.HxError):
        hx.paged_attention(cache, unaligned, lens, 1.0)
    with pytest.raises(RuntimeError):
        hx.paged_attention(cache, q.requires_grad_(), lens, 1.0)
    with torch.no_grad():
        hx.paged_attention(cache, q, lens, 1.0)


def test_capture_without_a_workspace_is_refused():
    import ctypes

    cache, _, _ = _filled(60, BF16, [20], 16, 1, 64)
    q = torch.zeros(1, 1, 64, device="cuda", dtype=BF16)
    o, lens = torch.empty_like(q), _lens(20)
    ctx = hx.context()
    rows = [N.Rows(t.data_ptr(), 64, 64) for t in (q, o)]

    def call():
        ctx.use_stream()
        return N.lib().hx_paged_attention(ctx.handle, N.HX_BF16, cache._ref, 1, ctypes.byref(rows[0]),
                                          ctypes.byref(rows[1]), None, lens.data_ptr(), 1.0, None, 0)

    assert call() == N.HX_OK
    torch.cuda.synchronize()
    one = torch.zeros(1, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one += 1  # a graph of its own, beside the refused call
        assert call() == N.HX_ERR_INVALID


@pytest.mark.parametrize("dtype", DT)
def test_outputs_at_any_element(dtype):
    """An output that starts at an odd element, with rows of an odd stride."""
    lens = [90, 700, 0]
    cache, ks, vs = _filled(70, dtype, lens, 16, 2, 64)
    q = torch.randn(3, 4, 64, generator=_gen(1), device="cuda", dtype=dtype)
    wide = torch.full((3, 4, 67), 5.0, device="cuda", dtype=dtype)
    o, lse = hx.paged_attention(cache, q, _lens(*lens), 0.125, out=wide[:, :, 1:65])
    _check(q, ks, vs, 0.125, o, lse)
    assert (wide[:, :, 0] == 5).all() and (wide[:, :, 65:] == 5).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("hk,group,dim", [(16, 1, 64), (16, 1, 40), (8, 2, 72), (5, 5, 128), (4, 16, 64)])
def test_more_tiles_than_workers(dtype, hk, group, dim):
    """Runs that end one item and begin the next, so that workers leave both of their parts."""
    lens = [1500 - 97 * i for i in range(14)] + [3, 0, 700]
    cache, ks, vs = _filled(71, dtype, lens, 24, hk, dim)
    q = torch.randn(len(lens), hk * group, dim, generator=_gen(2), device="cuda", dtype=dtype)
    o, lse = hx.paged_attention(cache, q, _lens(*lens), dim ** -0.5)
    _check(q, ks, vs, dim ** -0.5, o, lse)


def test_steps_that_follow_each_other_see_each_others_writes():
    """Append and attention in turn on one stream, with nothing between them: every step attends to
    the token that the call before it wrote, to pages that earlier calls read."""
    H, D, n = 4, 64, 300
    table = torch.randperm(60, generator=_gen(3), device="cuda")[:40].to(torch.int32).view(2, 20)
    cache = hx.PagedKVCache.allocate(60, 16, H, D, table, dtype=F32)
    k, v, q = (torch.randn(n, 2, H, D, generator=_gen(s), device="cuda") for s in (4, 5, 6))
    seq = _lens(0, 1)
    at = [_lens(i, i) for i in range(n + 1)]
    torch.cuda.synchronize()
    outs = []
    for i in range(n):
        hx.paged_append(cache, k[i], v[i], seq, at[i])
        outs.append(hx.paged_attention(cache, q[i], at[i + 1], 0.125))
    for i in range(0, n, 23):
        ks, vs = ([t[:i + 1, s] for s in range(2)] for t in (k, v))
        _check(q[i], ks, vs, 0.125, *outs[i])


def test_lengths_near_the_largest_integer():
    """A table row of 2^31 positions on one page: lengths past 2^31 - 256 are refused with NaN."""
    page = 1 << 20
    table = torch.zeros(3, 2048, dtype=torch.int32, device="cuda")
    cache = hx.PagedKVCache(*(torch.zeros(1, page, 1, 8, device="cuda", dtype=BF16) for _ in range(2)), table)
    o, lse = hx.paged_attention(cache, torch.zeros(3, 1, 8, device="cuda", dtype=BF16), _lens(2**31 - 1, 5, 2**31 - 255), 1.0)
    assert torch.isnan(o[[0, 2]]).all() and (o[1] == 0).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("lens", [[40, 0, 7], [9000, 1, 333]])
def test_attention_over_its_own_queries(dtype, lens):
    """out may be q, for items that one worker has and for items that many share."""
    cache, ks, vs = _filled(71, dtype, lens, 16, 2, 64)
    q = torch.randn(len(lens), 6, 64, device="cuda", dtype=dtype, generator=_gen(72))
    first = q.clone()
    o, lse = hx.paged_attention(cache, q, _lens(*lens), 0.125, out=q)
    assert o is q
    _check(first, ks, vs, 0.125, o, lse)


def test_outputs_that_share_memory_are_refused():
    table = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    k = torch.zeros(2, 16, 2, 64, device="cuda", dtype=BF16)
    cache, lens, x = hx.PagedKVCache(k, k.clone(), table), _lens(1, 1), torch.zeros(2, 2, 64, device="cuda", dtype=BF16)
    shared = torch.zeros(1, 2, 64, device="cuda", dtype=BF16).expand(2, 2, 64)
    near = torch.zeros(2, 2, 128, device="cuda", dtype=BF16).as_strided((2, 2, 64), (96, 64, 1))
    for out in (shared, near, x.transpose(0, 1)):  # the last is x at other strides
        with pytest.raises(N.HxError):
            hx.paged_attention(cache, x, lens, 1.0, out=out)
        with pytest.raises(N.HxError):
            hx.paged_append(cache, x, x, lens, lens, q=x, out_q=out)
    # One set of keys for all heads: to read, not to write.
    one = hx.PagedKVCache(k[:, :, :1].expand(2, 16, 2, 64), k[:, :, :1].expand(2, 16, 2, 64), table)
    hx.paged_attention(one, x, lens, 1.0)
    with pytest.raises(N.HxError):
        hx.paged_append(one, x, x, lens, lens)
    flat = torch.zeros(16, 2, 64, device="cuda", dtype=BF16).expand(2, 16, 2, 64)
    with pytest.raises(N.HxError):
        hx.paged_append(hx.PagedKVCache(flat, flat, table), x, x, lens, lens)
    across = torch.empty(2, 2, 64, device="cuda", dtype=BF16).transpose(0, 1)  # strides in another order do not overlap
    hx.paged_append(cache, x, x, _lens(0, 1), _lens(0, 1), q=x, out_q=across)
    assert (across == 0).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dim,group", [(64, 2), (128, 12), (256, 1)])
def test_infinite_values_keep_their_sign(dtype, dim, group):
    """An infinite value makes its element infinite whatever its weight (from 1 to 2^-86 here); both signs, or NaN, give NaN."""
    inf, nan = float("inf"), float("nan")
    lens = [1, 200, 200, 5000, 200, 90]
    cache, ks, vs = _filled(81, dtype, lens, 16, 1, dim)
    t = cache.block_table.long()
    q = torch.randn(len(lens), group, dim, generator=_gen(82), device="cuda", dtype=dtype)
    q[1] = 0  # equal weights, each one bf16 number exactly
    q[5] = 0
    q[5, :, 0] = 1
    k = ks[5].clone()
    k[:, 0, 0] = 0
    k[7, 0, 0] = -60.0 * dim ** 0.5  # this key weighs e^-60 of the others
    j = torch.arange(90, device="cuda")
    cache.k[t[5][j // 16], j % 16], ks[5] = k, k
    for s, at, d, value in [(0, 0, 3, inf), (1, 150, 3, inf), (1, 0, 9, -inf), (2, 150, 3, inf), (2, 77, 9, -inf),
                            (2, 150, 17, nan), (3, 4321, 3, inf), (3, 0, 9, -inf), (3, 17, 21, inf), (3, 4900, 21, -inf),
                            (4, 10, 21, inf), (4, 20, 21, -inf), (5, 7, 3, inf), (5, 7, 9, -inf)]:
        cache.v[t[s, at // 16], at % 16, 0, d] = value
        vs[s][at, 0, d] = value
    o, lse = hx.paged_attention(cache, q, _lens(*lens), dim ** -0.5)
    want, rl, off, off_lse = _reference(q, ks, vs, dim ** -0.5)
    assert torch.equal(torch.isnan(o), torch.isnan(want))
    assert torch.equal(torch.isinf(o), torch.isinf(want)) and torch.isinf(want).sum() == group * 9
    assert torch.equal(o[torch.isinf(want)].double(), want[torch.isinf(want)])
    live = torch.isfinite(want)
    assert ((o.double() - want).abs() <= torch.finfo(dtype).eps / 2 * (want.abs() + off) + off)[live].all()
    assert ((lse.double() - rl).abs() <= off_lse + 2.0 ** -24 * rl.abs()).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("dim,group", [(64, 1), (128, 4), (128, 12), (256, 1)])
@pytest.mark.parametrize("lens", [[1, 40, 700], [30000, 5]])
def test_values_near_the_largest(dtype, dim, group, lens):
    """The result is a mean of the values, so it is finite where they are, however large: sums of weights
    that are not yet divided by their total must not overflow."""
    cache, ks, vs = _filled(83, dtype, lens, 16, 2, dim)
    t = cache.block_table.long()
    for s, n in enumerate(lens):
        j = torch.arange(n, device="cuda")
        # Of one sign in every second element, of both in the others.
        v = (1 + torch.rand(n, 2, dim, generator=_gen(84 + s), device="cuda")) * 2.0 ** 126
        v[..., 1::2] *= torch.sign(torch.randn(n, 2, dim // 2, generator=_gen(94 + s), device="cuda"))
        vs[s] = v.to(dtype)
        cache.v[t[s][j // 16], j % 16] = vs[s]
    q = torch.randn(len(lens), 2 * group, dim, generator=_gen(85), device="cuda", dtype=dtype)
    o, lse = hx.paged_attention(cache, q, _lens(*lens), 4 * dim ** -0.5)
    _check(q, ks, vs, 4 * dim ** -0.5, o, lse)
    again = hx.paged_attention(cache, q, _lens(*lens), 4 * dim ** -0.5)
    assert torch.equal(o, again[0]) and torch.equal(lse, again[1])


@pytest.mark.parametrize("mode", [torch.enable_grad, torch.no_grad])
def test_forward_mode_is_refused(mode):
    """A dual tensor does not require a gradient, but its tangent must not be lost."""
    table = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    k = torch.zeros(2, 16, 2, 64, device="cuda", dtype=BF16)
    cache, lens, x = hx.PagedKVCache(k, k.clone(), table), _lens(1, 1), torch.zeros(2, 2, 64, device="cuda", dtype=BF16)
    with mode(), torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for bad in (lambda: hx.paged_attention(cache, dual, lens, 1.0), lambda: hx.paged_append(cache, dual, x, lens, lens),
                    lambda: hx.paged_append(cache, x, dual, lens, lens),
                    lambda: hx.paged_append(cache, x, x, lens, lens, q=dual)):
            with pytest.raises(RuntimeError):
                bad()
        hx.paged_append(cache, x, x, _lens(0, 1), _lens(0, 0), q=x)  # without a tangent
        hx.paged_attention(cache, x, lens, 1.0)


def test_caches_and_outputs_that_need_a_gradient_are_refused():
    table = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    k = torch.zeros(2, 16, 2, 64, device="cuda", dtype=BF16)
    lens, x = _lens(1, 1), torch.zeros(2, 2, 64, device="cuda", dtype=BF16)
    leaf = x.clone().requires_grad_()
    cache = hx.PagedKVCache(k, k.clone(), table)
    for kv in ((k.clone().requires_grad_(), k.clone()), (k.clone(), k.clone().requires_grad_())):
        c = hx.PagedKVCache(*kv, table)
        for call in (lambda: hx.paged_attention(c, x, lens, 1.0), lambda: hx.paged_append(c, x, x, lens, lens)):
            with pytest.raises(RuntimeError):
                call()
            with torch.no_grad():
                call()
    for call in (lambda: hx.paged_attention(cache, x, lens, 1.0, out=leaf),
                 lambda: hx.paged_append(cache, x, x, lens, lens, q=x, out_q=leaf),
                 lambda: hx.paged_attention(cache, x, lens, 1.0, lse=torch.zeros(2, 2, device="cuda", requires_grad=True))):
        with pytest.raises(RuntimeError):
            call()
        with torch.no_grad():
            call()


def test_outputs_that_overlap_their_inputs_in_part_are_refused():
    """An output may be its input; it may not begin inside it."""
    table = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    k = torch.zeros(2, 16, 2, 64, device="cuda", dtype=BF16)
    cache, lens = hx.PagedKVCache(k, k.clone(), table), _lens(1, 1)
    buf = torch.zeros(4, 2, 64, device="cuda", dtype=BF16)
    wide = torch.zeros(2, 4, 64, device="cuda", dtype=BF16)
    flat = torch.zeros(1024, device="cuda", dtype=BF16)
    for q, out in ((buf[:2], buf[1:3]), (buf[1:3], buf[:2]), (wide[:, :2], wide[:, 1:3]),
                   (flat[:256].view(2, 2, 64), flat[64:320].view(2, 2, 64)), (flat[:256].view(2, 2, 64), flat[8:264].view(2, 2, 64)),
                   (flat[128:384].view(2, 2, 64), flat.as_strided((2, 2, 64), (256, 64, 1)))):
        with pytest.raises(N.HxError):
            hx.paged_attention(cache, q, lens, 1.0, out=out)
        with pytest.raises(N.HxError):
            hx.paged_append(cache, q, q, lens, lens, q=q, out_q=out)
    # Heads of one buffer side by side do not overlap.
    wide.normal_(generator=_gen(1))
    want = wide[:, :2].clone()
    hx.paged_append(cache, want, want, _lens(0, 1), _lens(0, 1), q=wide[:, :2], out_q=wide[:, 2:])
    assert torch.equal(wide[:, 2:], want) and torch.equal(wide[:, :2], want)
    out = torch.zeros(2, 2, 192, device="cuda", dtype=BF16)
    hx.paged_attention(cache, out[:, :, :64], lens, 1.0, out=out[:, :, 64:128])


def test_keys_and_values_in_the_same_memory_are_for_reading():
    table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    k = torch.randn(2, 16, 2, 64, generator=_gen(2), device="cuda", dtype=BF16)
    x, one = torch.zeros(1, 2, 64, device="cuda", dtype=BF16), _lens(0)
    both = torch.zeros(2, 16, 4, 64, device="cuda", dtype=BF16)
    pages = torch.zeros(3, 16, 2, 64, device="cuda", dtype=BF16)
    for kv in ((k, k), (both[:, :, :2], both[:, :, 1:3]), (pages[:2], pages[1:])):
        cache = hx.PagedKVCache(*kv, table)
        hx.paged_attention(cache, x, _lens(1), 1.0)
        with pytest.raises(N.HxError):
            hx.paged_append(cache, x, x, one, one)
    for kv in ((both[:, :, :2], both[:, :, 2:]), (pages[:1], pages[1:2]), (pages[:, :, :, :32], pages[:, :, :, 32:])):
        cache = hx.PagedKVCache(*kv, table)
        y = torch.ones(1, 2, kv[0].shape[3], device="cuda", dtype=BF16)
        hx.paged_append(cache, y, 2 * y, one, one)
        assert (kv[0][0, 0] == 1).all() and (kv[1][0, 0] == 2).all()


def test_sizes_past_an_int_are_refused():
    """2^32 + 1 pages (one, at stride 0) or sequences would otherwise be taken for one."""
    k = torch.zeros(1, 16, 1, 8, device="cuda", dtype=BF16)
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    for kv, t in ((k.expand(2**32 + 1, 16, 1, 8), table), (k, table.expand(2**32 + 1, 1))):
        with pytest.raises(ValueError):
            hx.PagedKVCache(kv, kv, t)
    cache = hx.PagedKVCache(k, k.clone(), table)
    with pytest.raises(ValueError):
        hx.paged_append(cache, k[0, :1].expand(2**32 + 1, 1, 8), k[0, :1].expand(2**32 + 1, 1, 8), _lens(0), _lens(0))


def test_scales_of_any_number_type():
    import numpy as np

    cache, ks, vs = _filled(90, BF16, [33], 16, 2, 64)
    q = torch.randn(1, 2, 64, generator=_gen(91), device="cuda", dtype=BF16)
    want = hx.paged_attention(cache, q, _lens(33), 0.25)
    for scale in (np.float32(0.25), np.float64(0.25), torch.tensor(0.25)):
        got = hx.paged_attention(cache, q, _lens(33), scale)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
