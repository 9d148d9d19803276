"""Log probabilities of given tokens, entropy, alternatives and gradients, against the formulas in f64.

Tolerances, from the arithmetic, for a row with z = x - max, s = sum e^z: an
exponential is good to 2^-22 and its argument is rounded twice (2^-23 |z|), a
thread adds V/512 of them (in each of two halves) and a tree of 1 + 5 + 3 levels,
with up to 8 CTAs after it, joins them, each at 2^-24 and 2^-22 for the weights of the
joins. So ln s is off by less than
rel = 2^-21 + (V/512 + 64) 2^-23 + 2^-22 E|z|, a log probability by that and 2^-23
(|z| + |ln s|), the entropy by rel (1 + H) and 2^-22 E(z^2 + |z|).
"""
import pytest
import torch

import haelixe_b200 as hx
from haelixe_b200 import _native as N

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
DT = [pytest.param(F32, id="f32"), pytest.param(BF16, id="bf16")]
INF = float("inf")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _logits(rows, classes, dtype, seed=0, spread=2.5):
    return (torch.randn(rows, classes, generator=_gen(seed), device="cuda") * spread).to(dtype)


def _targets(rows, classes, seed=1):
    return torch.randint(classes, (rows,), generator=_gen(seed), device="cuda")


class Ref:
    def __init__(self, x, t):
        x = x.double()
        self.z = x - x.amax(1, keepdim=True)
        e = torch.exp(self.z)
        self.s = e.sum(1, keepdim=True)
        self.p = e / self.s
        self.ls = torch.log(self.s)
        zz = torch.where(self.p > 0, self.z, 0.0)
        self.entropy = (self.p * (self.ls - zz)).sum(1)
        self.logp = (self.z - self.ls).gather(1, t[:, None]).squeeze(1)
        V = x.shape[1]
        self.rel = 2.0 ** -21 + (V / 512 + 64) * 2.0 ** -23 + 2.0 ** -22 * (self.p * zz.abs()).sum(1)
        zt = self.z.gather(1, t[:, None]).squeeze(1)
        self.off_logp = self.rel + 2.0 ** -23 * (zt.abs() + self.ls.squeeze(1).abs())
        self.off_h = self.rel * (1 + self.entropy) + 2.0 ** -22 * (self.p * (zz * zz + zz.abs())).sum(1)
        self.t = t

    def grad(self, gl, gh):
        """dlogits and the bound on its error besides the rounding to its type."""
        lp = torch.where(self.p > 0, self.z - self.ls, 0.0)
        gl = torch.zeros_like(self.logp) if gl is None else gl.double()
        gh = torch.zeros_like(self.logp) if gh is None else gh.double()
        gl, gh, h = gl[:, None], gh[:, None], self.entropy[:, None]
        d = -self.p * (gl + gh * (lp + h))
        d.scatter_add_(1, self.t[:, None], gl)
        off_z = self.rel[:, None] + 2.0 ** -22 * (lp.abs() + self.ls.abs())
        size = self.p * (gl.abs() + gh.abs() * (lp.abs() + h))
        off = size * (off_z + 2.0 ** -21) + self.p * gh.abs() * (off_z + self.off_h[:, None])
        off.scatter_add_(1, self.t[:, None], 2.0 ** -23 * gl.abs())
        return d, off


def _close(got, want, off):
    bad = (got.double() - want).abs() > off
    assert torch.isfinite(got).all() and not bad.any(), float(((got.double() - want).abs() - off).max())


def _check(r, x, t):
    ref = Ref(x, t)
    _close(r.logprob, ref.logp, ref.off_logp)
    _close(r.entropy, ref.entropy, ref.off_h)
    return ref


def _order(x):
    """Stable: equal values keep the order of their indices."""
    return torch.sort(torch.where(torch.isnan(x.float()), -INF, x.float()), dim=1, descending=True, stable=True).indices


def _check_top(r, x, k):
    ids = _order(x)[:, :k]
    assert torch.equal(r.top_ids.long(), ids)
    ref = Ref(x, ids[:, 0])
    # From the maximum: at logits of 10^38 even f64 would lose the sum's logarithm next to them.
    lp = (ref.z - ref.ls).gather(1, ids)
    live = torch.isfinite(lp)
    assert torch.equal(torch.isfinite(r.top_logprobs), live)
    zs = ref.z.gather(1, ids)
    off = ref.rel[:, None] + 2.0 ** -23 * (zs.abs() + ref.ls.abs())
    assert ((r.top_logprobs.double() - lp).abs() <= off)[live].all()
    assert (r.top_logprobs[~live] == -INF).all()


SIZES = [1, 2, 7, 8, 9, 33, 511, 513, 4095, 4099, 32000, 50001, 131071]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("classes", SIZES)
@pytest.mark.parametrize("rows", [1, 5])
def test_forward_and_top(dtype, classes, rows):
    x, t = _logits(rows, classes, dtype, classes), _targets(rows, classes)
    _check(hx.nn.token_logprobs(x, t), x, t)
    for k in sorted({1, min(5, classes), min(32, classes)}):
        r = hx.nn.token_logprobs(x, t.to(torch.int32), k)
        _check(r, x, t)
        _check_top(r, x, k)


@pytest.mark.parametrize("dtype", DT)
def test_many_rows(dtype):
    x, t = _logits(3001, 515, dtype), _targets(3001, 515)
    r = hx.nn.token_logprobs(x, t, 3)
    _check(r, x, t)
    _check_top(r, x, 3)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,classes", [(1200, 5003), (1201, 20000), (160, 70001), (1185, 34007), (70, 9001)])
def test_rows_and_lengths_of_each_kernel(dtype, rows, classes):
    x, t = _logits(rows, classes, dtype), _targets(rows, classes)
    _check(hx.nn.token_logprobs(x, t), x, t)
    for k in (1, 20, 32):
        r = hx.nn.token_logprobs(x, t, k)
        _check(r, x, t)
        _check_top(r, x, k)
    # Ties all over: the slow way of putting the alternatives in order.
    x = (x * 0.5).round()
    r = hx.nn.token_logprobs(x, t, 32)
    _check(r, x, t)
    _check_top(r, x, 32)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("lead", [0, 1, 3, 8])
def test_rows_cut_from_a_wider_buffer(dtype, lead):
    """What surrounds the rows is NaN, and each row starts at its own offset from a 16-byte boundary."""
    wide = torch.full((6, 1000 + 13), float("nan"), device="cuda", dtype=dtype)
    x = wide[:, lead:lead + 1000]
    x.copy_(_logits(6, 1000, dtype))
    t = _targets(6, 1000)
    r = hx.nn.token_logprobs(x, t, 7)
    ref = _check(r, x, t)
    _check_top(r, x, 7)
    xg = x.detach().requires_grad_()
    r = hx.nn.token_logprobs(xg, t)
    gl, gh = (torch.randn(6, generator=_gen(s), device="cuda") for s in (1, 2))
    (d,) = torch.autograd.grad([r.logprob, r.entropy], [xg], [gl, gh])
    want, off = ref.grad(gl, gh)
    _close(d, want, off + torch.finfo(dtype).eps / 2 * (want.abs() + off))


@pytest.mark.parametrize("dtype", DT)
def test_ties_and_orders(dtype):
    V = 20000
    j = torch.arange(V, device="cuda")
    E = 8 if dtype == BF16 else 4
    rows = [torch.zeros(V, device="cuda"), (j // 157).float(), -(j // 157).float(), (j % 2).float(),
            ((j // E) % 512 == 300).float() * (1 + j / V), ((j // E) % 512 < 3).float(),
            torch.where(j % 2 == 0, 0.0, -0.0), torch.where(j == V - 1, 5.0, 0.0)]
    x = torch.stack(rows).to(dtype)
    t = _targets(len(rows), V)
    for k in (1, 20, 32):
        r = hx.nn.token_logprobs(x, t, k)
        _check(r, x, t)
        _check_top(r, x, k)


@pytest.mark.parametrize("dtype", DT)
def test_masked_logits(dtype):
    """-inf and the type's lowest value over most of the row, a single live logit, a row of the lowest value."""
    V = 3000
    low = torch.finfo(dtype).min
    x = _logits(6, V, dtype)
    x[0, 100:] = -INF
    x[1, 1:] = -INF
    x[2, :-2] = low
    x[3, :] = low
    x[4, ::2] = -INF
    x[5, 5:] = -INF
    t = torch.tensor([50, 0, V - 1, 17, 1, 2], device="cuda")
    r = hx.nn.token_logprobs(x, t, 8)
    ref = _check(r, x, t)
    _check_top(r, x, 8)
    assert r.logprob[1] == 0 and r.entropy[1] == 0
    xg = x.detach().requires_grad_()
    r = hx.nn.token_logprobs(xg, t)
    gl, gh = (torch.randn(6, generator=_gen(s), device="cuda") for s in (1, 2))
    (d,) = torch.autograd.grad([r.logprob, r.entropy], [xg], [gl, gh])
    want, off = ref.grad(gl, gh)
    _close(d, want, off + torch.finfo(dtype).eps / 2 * (want.abs() + off))
    # A masked target has no probability.
    assert hx.nn.token_logprobs(x[1:2], torch.tensor([5], device="cuda")).logprob.item() == -INF


@pytest.mark.parametrize("dtype", DT)
def test_large_logits(dtype):
    """Logits near +-10^4 and 10^38: only their differences count."""
    x = torch.stack([_logits(1, 777, F32)[0] + 1e4, _logits(1, 777, F32)[0] * 1e3, _logits(1, 777, F32)[0] * 1e37]).to(dtype)
    t = _targets(3, 777)
    t[2] = x[2].argmax()
    _check(hx.nn.token_logprobs(x, t, 4), x, t)


@pytest.mark.parametrize("dtype", DT)
def test_rows_that_are_not_finite(dtype):
    x = _logits(5, 600, dtype)
    x[0, 3], x[1, 599], x[2, :], x[3, 7] = float("nan"), INF, -INF, 100.0
    t = torch.tensor([9, 9, 9, 600, 4], device="cuda")
    r = hx.nn.token_logprobs(x, t, 2)
    assert torch.isnan(r.logprob[:3]).all() and torch.isnan(r.entropy[:3]).all()
    assert torch.isnan(r.logprob[3]) and torch.isfinite(r.entropy[3])  # a target outside the classes
    assert torch.equal(r.top_ids.long()[[0, 2, 3, 4]], _order(x)[[0, 2, 3, 4], :2])
    _check(hx.nn.token_logprobs(x[4:], t[4:]), x[4:], t[4:])
    xg = x.detach().requires_grad_()
    hx.nn.token_logprobs(xg, t).logprob.backward(torch.ones(5, device="cuda"))
    assert torch.isnan(xg.grad[:4]).all(1).all() and torch.isfinite(xg.grad[4]).all()
    assert torch.isnan(hx.nn.token_logprobs(x[4:], torch.tensor([-100], device="cuda")).logprob).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("classes", [1, 8, 513, 4099, 32000])
@pytest.mark.parametrize("which", ["both", "logprob", "entropy"])
def test_gradient(dtype, classes, which):
    x, t = _logits(7, classes, dtype).requires_grad_(), _targets(7, classes)
    gl, gh = (torch.randn(7, generator=_gen(s), device="cuda") for s in (3, 4))
    r = hx.nn.token_logprobs(x, t, min(3, classes))
    assert not r.top_logprobs.requires_grad
    outs = {"both": [(r.logprob, gl), (r.entropy, gh)], "logprob": [(r.logprob, gl)], "entropy": [(r.entropy, gh)]}[which]
    (d,) = torch.autograd.grad([o for o, _ in outs], [x], [g for _, g in outs])
    want, off = Ref(x.detach(), t).grad(gl if which != "entropy" else None, gh if which != "logprob" else None)
    assert d.dtype == dtype
    _close(d, want, off + torch.finfo(dtype).eps / 2 * (want.abs() + off))


def test_gradient_against_differences():
    """Central differences of the f64 formula (h = 1e-5: off by h^2 and 1e-16 / h) along random directions."""
    x, t = _logits(4, 40, F32), _targets(4, 40)
    gl, gh = (torch.randn(4, generator=_gen(s), device="cuda") for s in (5, 6))
    xg = x.clone().requires_grad_()
    r = hx.nn.token_logprobs(xg, t)
    ((r.logprob * gl).sum() + (r.entropy * gh).sum()).backward()

    def value(y):
        lp = y - torch.logsumexp(y, 1, keepdim=True)
        return (lp.gather(1, t[:, None]).squeeze(1) * gl).sum() - ((lp.exp() * lp).sum(1) * gh).sum()

    for s in range(5):
        v = torch.randn(x.shape, generator=_gen(10 + s), device="cuda").double()
        h = 1e-5
        want = (value(x.double() + h * v) - value(x.double() - h * v)) / (2 * h)
        got = (xg.grad.double() * v).sum()
        assert abs(float(got - want)) < 1e-5 * float((xg.grad.double() * v).abs().sum() + 1)


def test_gradient_of_a_mean_and_beside_cross_entropy():
    """Expanded upstream gradients; the mean of -logprob is cross_entropy, with its gradient."""
    x, t = _logits(64, 1000, F32), _targets(64, 1000)
    a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
    la, lb = -hx.nn.token_logprobs(a, t).logprob.mean(), hx.nn.cross_entropy(b, t)
    la.backward()
    lb.backward()
    assert abs(float(la.detach() - lb.detach())) < 64 * 2.0 ** -23 * float(lb.detach())
    assert (a.grad - b.grad).abs().max() < 2.0 ** -20 / 64


def test_same_bits_and_graph():
    """Forward and backward captured while an eager graph of the same logits lives. The captured step
    differentiates a leaf of its own: autograd ties a leaf to the stream of its first live graph, and
    joining that stream would end any capture, whatever the operator."""
    x, t = _logits(33, 5003, BF16).requires_grad_(), _targets(33, 5003).to(torch.int32)
    g = torch.randn(33, generator=_gen(1), device="cuda")

    def step():
        leaf = x.detach().requires_grad_()
        r = hx.nn.token_logprobs(leaf, t, 4)
        return (*(f.detach() for f in r), torch.autograd.grad([r.logprob, r.entropy], [leaf], [g, g])[0])

    alive = hx.nn.token_logprobs(x, t)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        first = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step()
    for seed in (0, 7):
        with torch.no_grad():
            x.copy_(_logits(33, 5003, BF16, seed))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        if seed == 0:
            assert all(torch.equal(a, b) for a, b in zip(first, want))
    del alive


def test_offsets_past_32_bits():
    """More than 2^31 logits: the last rows are right."""
    V = 131072
    x = torch.zeros(16500, V, device="cuda", dtype=BF16)
    x[-2:] = _logits(2, V, BF16)
    t = torch.zeros(16500, dtype=torch.int32, device="cuda")
    t[-2:] = 77
    xg = x.requires_grad_()
    r = hx.nn.token_logprobs(xg, t, 2)
    part = xg.detach()[-2:]
    ref = Ref(part, t[-2:].long())
    _close(r.logprob.detach()[-2:], ref.logp, ref.off_logp)
    g = torch.ones(16500, device="cuda")
    (d,) = torch.autograd.grad([r.logprob, r.entropy], [xg], [g, g])
    want, off = ref.grad(g[-2:], g[-2:])
    _close(d[-2:], want, off + 2.0 ** -8 * (want.abs() + off))


def test_refusals_and_empty():
    x, t = _logits(3, 10, F32), _targets(3, 10)
    for bad in (lambda: hx.nn.token_logprobs(x[0], t), lambda: hx.nn.token_logprobs(x.t(), t),
                lambda: hx.nn.token_logprobs(x, t[:2]), lambda: hx.nn.token_logprobs(x, t, 11),
                lambda: hx.nn.token_logprobs(_logits(3, 100, F32), t, 33), lambda: hx.nn.token_logprobs(x, t, -1),
                lambda: hx.nn.token_logprobs(x, t.cpu())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        hx.nn.token_logprobs(x.half(), t)
    with pytest.raises(TypeError):
        hx.nn.token_logprobs(x, t.float())
    with pytest.raises(RuntimeError):
        hx.nn.token_logprobs(x.cpu(), t.cpu())
    r = hx.nn.token_logprobs(x[:0].requires_grad_(), t[:0], 2)
    assert r.logprob.shape == (0,) and r.top_ids.shape == (0, 2)
    e = x[:1].expand(3, 10)  # rows that share memory
    _check(hx.nn.token_logprobs(e, t, 2), e, t)
    L, c = N.lib(), hx.context()
    p = x.data_ptr()
    assert L.hx_token_logprobs_fwd(c.handle, 0, p, 9, p, p, p, None, 0, None, None, 3, 10) == N.HX_ERR_INVALID
    assert L.hx_token_logprobs_fwd(c.handle, 0, p, 10, p, p, p, None, 2, None, None, 3, 10) == N.HX_ERR_INVALID
    assert L.hx_token_logprobs_fwd(c.handle, 5, p, 10, p, p, p, None, 0, None, None, 3, 10) == N.HX_ERR_INVALID
    assert L.hx_token_logprobs_bwd(c.handle, 0, p, 10, p, None, p, p, p, 10, 3, 10) == N.HX_ERR_INVALID
    assert L.hx_token_logprobs_bwd(c.handle, 0, p, 10, p, p, p, p, p, 9, 3, 10) == N.HX_ERR_INVALID
    assert L.hx_token_logprobs_fwd(None, 0, p, 10, p, p, p, None, 0, None, None, 3, 10) == N.HX_ERR_INVALID


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("classes", [5, 4099, 40000])
def test_gradient_written_over_the_logits(dtype, classes):
    """The library's backward with dlogits on the logits themselves gives what it gives beside them."""
    x, t = _logits(9, classes, dtype), _targets(9, classes).to(torch.int32)
    g = torch.randn(9, generator=_gen(1), device="cuda")
    leaf = x.clone().requires_grad_()
    r = hx.nn.token_logprobs(leaf, t)
    (want,) = torch.autograd.grad([r.logprob, r.entropy], [leaf], [g, g])
    stats, lp, h = (torch.empty(9, n, device="cuda") for n in (3, 1, 1))
    c = hx.context()
    c.use_stream()
    d = 0 if dtype == F32 else 1
    p = x.data_ptr()
    N.check(N.lib().hx_token_logprobs_fwd(c.handle, d, p, classes, t.data_ptr(), lp.data_ptr(), h.data_ptr(), stats.data_ptr(),
                                          0, None, None, 9, classes), c.handle)
    N.check(N.lib().hx_token_logprobs_bwd(c.handle, d, p, classes, t.data_ptr(), stats.data_ptr(), g.data_ptr(), g.data_ptr(),
                                          p, classes, 9, classes), c.handle)
    assert torch.equal(x, want)


def test_gradient_of_shared_rows():
    """Rows that are one row expanded: its gradient is the sum."""
    row = _logits(1, 50, F32).requires_grad_()
    t, g = _targets(4, 50), torch.randn(4, generator=_gen(2), device="cuda")
    (hx.nn.token_logprobs(row.expand(4, 50), t).logprob * g).sum().backward()
    ref = Ref(row.detach().expand(4, 50), t)
    want, off = ref.grad(g, None)
    _close(row.grad, want.sum(0, keepdim=True), off.sum(0, keepdim=True) + 2.0 ** -22 * want.abs().sum(0, keepdim=True))


def test_gradient_over_the_logits_at_another_stride_is_refused():
    x, t = torch.randn(3, 12, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    L, c, f = N.lib(), hx.context(), torch.zeros(9, device="cuda")
    p, q = x.data_ptr(), f.data_ptr()
    assert L.hx_token_logprobs_bwd(c.handle, 0, p, 12, t.data_ptr(), q, q, None, p, 10, 3, 10) == N.HX_ERR_INVALID


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,classes", [(1300, 300), (1300, 1000), (1300, 2100), (700, 5003), (150, 4001), (40, 400), (600, 60), (1, 129)])
def test_rows_and_lengths_where_the_kernel_changes(dtype, rows, classes):
    test_rows_and_lengths_of_each_kernel(dtype, rows, classes)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,classes", [(5, 5003), (1, 131072), (160, 20000), (1200, 5003), (1300, 300), (515, 131071)])
def test_pieces_made_of_nan(dtype, rows, classes):
    """Whole 16-byte pieces of NaN, among them the first that a thread reads, with the likeliest classes in later
    pieces of the same threads (every kernel steps by a power of two of pieces): NaN ranks as -inf."""
    E = 8 if dtype == BF16 else 4
    x = _logits(rows, classes, dtype)
    x[:, :41 * E] = float("nan")
    for r in range(min(rows, 6)):
        at = torch.arange(5 * E + E // 2, classes, (32 << r) * E, device="cuda")[1:]
        x[r, at] = 20 + torch.arange(len(at), device="cuda").to(dtype)
    t = _targets(rows, classes)
    for k in (1, 20):
        r = hx.nn.token_logprobs(x, t, k)
        assert torch.equal(r.top_ids.long(), _order(x)[:, :k])
        assert torch.isnan(r.logprob).all() and torch.isnan(r.entropy).all() and torch.isnan(r.top_logprobs).all()


def test_forward_mode_is_refused():
    """A dual tensor does not require a gradient, but its tangent must not be lost."""
    x, t = _logits(3, 10, F32), _targets(3, 10)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), pytest.raises(NotImplementedError):
                hx.nn.token_logprobs(dual, t, 2)
        _check(hx.nn.token_logprobs(x, t), x, t)  # without a tangent
