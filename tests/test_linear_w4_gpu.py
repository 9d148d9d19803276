"""Linear products with 4-bit weights, against the formula in f64.

Tolerance, from the arithmetic: the products are exact (4-bit integers times
bf16, f32 as three bf16 that sum to it), so only sums and the scale round. A
unit of 128 k is up to 24 tensor products in a chain, each off by at most 2^-23 of
the partial sum it adds to; then a group of warps adds its scaled units (in / 128 at
most), 8 groups and 8 CTAs are joined, bias and residual added, each at 2^-24.
Altogether (24 + in / 256 + 20) 2^-23 of the sum of magnitudes, and half a
step of the type.
"""
import pytest
import torch

import haelixe_b200 as hx
from haelixe_b200 import _native as N

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
DT = [pytest.param(F32, id="f32"), pytest.param(BF16, id="bf16")]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _make(rows, in_f, out_f, group, dtype, seed=0):
    g = _gen(seed)
    x = torch.randn(rows, in_f, generator=g, device="cuda").to(dtype)
    packed = torch.randint(-2**31, 2**31, (-(-in_f // 8), out_f), generator=g, device="cuda").to(torch.int32)
    scales = (torch.rand(-(-in_f // group), out_f, generator=g, device="cuda") * 0.02 - 0.005).to(dtype)
    return x, packed, scales


def _weight(packed, scales, group, in_f):
    q = torch.stack([(packed.long() >> (4 * i)) & 15 for i in range(8)], 1).flatten(0, 1)[:in_f]
    return (q - 8).double() * scales.double()[torch.arange(in_f, device="cuda") // group]


def _check(y, x, w, bias=None, residual=None):
    x = x.double()
    want, size = x @ w, x.abs() @ w.abs()
    for t in (bias, residual):
        if t is not None:
            want, size = want + t.double(), size + t.double().abs()
    off = (44 + x.shape[-1] / 256) * 2.0 ** -23 * size
    err = (y.double() - want).abs()
    assert torch.isfinite(y).all()
    assert (err <= off + torch.finfo(y.dtype).eps / 2 * (want.abs() + off)).all(), float((err - off).max())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("in_f,out_f,group", [
    (1, 1, 32), (7, 5, 32), (8, 4, 64), (31, 33, 32), (32, 32, 32), (33, 64, 32), (100, 130, 64), (256, 31, 256),
    (1000, 36, 128), (1024, 96, 1024), (2048, 257, 128), (4104, 64, 96), (8192, 40, 64), (16388, 32, 4096),
])
@pytest.mark.parametrize("rows", [1, 3, 8, 9, 16, 17, 33])
def test_sizes(dtype, in_f, out_f, group, rows):
    x, packed, scales = _make(rows, in_f, out_f, group, dtype, rows + in_f)
    w = _weight(packed, scales, group, in_f)
    g = _gen(3)
    bias, res = (torch.randn(s, generator=g, device="cuda").to(dtype) for s in ((out_f,), (rows, out_f)))
    _check(hx.nn.linear_w4(x, packed, scales, group), x, w)
    _check(hx.nn.linear_w4(x, packed, scales, group, bias, res), x, w, bias, res)


@pytest.mark.parametrize("dtype", DT)
def test_many_rows_and_leading_dimensions(dtype):
    x, packed, scales = _make(150, 512, 64, 128, dtype)
    y = hx.nn.linear_w4(x.view(3, 50, 512), packed, scales, 128)
    assert y.shape == (3, 50, 64)
    _check(y.view(150, 64), x, _weight(packed, scales, 128, 512))


@pytest.mark.parametrize("dtype", DT)
def test_each_nibble_and_column(dtype):
    """One-hot rows read single weights back exactly."""
    in_f, out_f = 64, 48
    _, packed, scales = _make(1, in_f, out_f, 32, dtype)
    w = _weight(packed, scales, 32, in_f)
    x = torch.eye(in_f, device="cuda", dtype=dtype)
    assert torch.equal(hx.nn.linear_w4(x, packed, scales, 32), w.to(dtype))


def test_f32_activations_keep_their_bits():
    """x of 24 significant bits, and far apart in size: nothing is lost to the tensor products' 8 bits."""
    x = torch.tensor([[1 + 2.0 ** -23, 2.0 ** 20 + 2.0 ** -3, -(1 - 2.0 ** -24), 3.0 ** -20]], device="cuda")
    packed = torch.tensor([[0x9999]], dtype=torch.int32, device="cuda")  # weights 1, 1, 1, 1
    for i in range(4):
        one = torch.zeros_like(x)
        one[0, i] = x[0, i]
        assert hx.nn.linear_w4(one, packed, torch.ones(1, 1, device="cuda"), 32).item() == x[0, i].item()


@pytest.mark.parametrize("dtype", DT)
def test_values_that_are_not_finite_stay_in_their_row(dtype):
    x, packed, scales = _make(4, 96, 40, 32, dtype)
    w = _weight(packed, scales, 32, 96)
    x[1, 5], x[2, 40], x[3, 95] = float("nan"), float("inf"), -float("inf")
    y = hx.nn.linear_w4(x, packed, scales, 32)
    _check(y[:1], x[:1], w)
    assert torch.isnan(y[1]).all()
    for r, k in ((2, 40), (3, 95)):
        want = x[r, k].double() * w[k]  # inf * 0 is NaN
        assert torch.equal(torch.isnan(y[r]), torch.isnan(want))
        assert torch.equal(y[r].double()[~torch.isnan(want)], want[~torch.isnan(want)])
    top = torch.full((1, 8), torch.finfo(dtype).max, device="cuda", dtype=dtype)
    one = torch.full((1, 1), 0x9, dtype=torch.int32, device="cuda")  # weights 1, -8 ...: only the first counts
    top[0, 1:] = 0
    assert hx.nn.linear_w4(top, one, torch.ones(1, 1, device="cuda", dtype=dtype), 32).item() == top[0, 0].item()


def test_nibbles_past_the_inputs_are_ignored():
    x, packed, scales = _make(2, 13, 8, 32, BF16)
    a = hx.nn.linear_w4(x, packed, scales, 32)
    packed[1] ^= torch.tensor(-(1 << 20), dtype=torch.int32, device="cuda")  # q of k = 13, 14, 15
    assert torch.equal(a, hx.nn.linear_w4(x, packed, scales, 32))


def test_residual_may_be_the_output_buffer_and_x_strided():
    x, packed, scales = _make(6, 256, 64, 64, BF16)
    w = _weight(packed, scales, 64, 256)
    wide = torch.randn(6, 300, generator=_gen(1), device="cuda").to(BF16)
    wide[:, 20:276] = x
    _check(hx.nn.linear_w4(wide[:, 20:276], packed, scales, 64), x, w)
    res = torch.randn(6, 64, generator=_gen(2), device="cuda").to(BF16)
    want = hx.nn.linear_w4(x, packed, scales, 64, residual=res)
    c = hx.context()
    c.use_stream()
    N.check(N.lib().hx_linear_w4_fwd(c.handle, N.HX_BF16, x.data_ptr(), packed.data_ptr(), scales.data_ptr(), None,
                                     res.data_ptr(), res.data_ptr(), 6, 256, 64, 64), c.handle)
    assert torch.equal(res, want)


def test_unaligned_operands():
    x, packed, scales = _make(5, 64, 32, 32, BF16)
    want = hx.nn.linear_w4(x, packed, scales, 32)

    def shifted(t):
        return torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)

    assert torch.equal(hx.nn.linear_w4(shifted(x), packed, scales, 32), want)
    assert torch.equal(hx.nn.linear_w4(x, shifted(packed), scales, 32), want)
    assert torch.equal(hx.nn.linear_w4(x, packed, shifted(scales), 32), want)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("in_f,out_f,group", [(1, 1, 32), (64, 40, 32), (100, 7, 64), (2048, 300, 128)])
def test_quantize(dtype, in_f, out_f, group):
    w = torch.randn(in_f, out_f, generator=_gen(4), device="cuda").to(dtype)
    w[:, 0] = 0
    packed, scales = hx.nn.quantize_w4(w, group)
    pad = -in_f % group
    wp = torch.nn.functional.pad(w.float(), (0, 0, 0, pad)).view(-1, group, out_f)
    # In f64 first: torch divides an f32 tensor by a scalar with a rounded reciprocal.
    s = (wp.abs().amax(1).double() / 7).float().to(dtype)
    assert torch.equal(scales, s)
    q = torch.where(s.float()[:, None] > 0, torch.round(wp / s.float()[:, None]), 0.0).clamp(-8, 7).view(-1, out_f)[:in_f]
    want = q.double() * s.double().repeat_interleave(group, 0)[:in_f]
    got = _weight(packed, scales, group, in_f)
    assert torch.equal(got, want)
    # Half a step of the scale, and bf16's rounding of the scale over 7 of them.
    assert ((got - w.double()).abs() <= s.double().repeat_interleave(group, 0)[:in_f] * (0.5 + 8 * torch.finfo(dtype).eps)).all()


def test_graph_and_same_bits():
    x, packed, scales = _make(9, 1024, 320, 128, BF16)
    first = hx.nn.linear_w4(x, packed, scales, 128)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = hx.nn.linear_w4(x, packed, scales, 128)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, first)
    x.mul_(-1)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, -first)


def test_refusals_and_empty():
    x, packed, scales = _make(2, 64, 32, 32, BF16)
    bias = torch.zeros(32, device="cuda", dtype=BF16)
    for bad in (lambda: hx.nn.linear_w4(x, packed, scales, 16), lambda: hx.nn.linear_w4(x, packed, scales, 64),
                lambda: hx.nn.linear_w4(x, packed[:-1], scales, 32), lambda: hx.nn.linear_w4(x, packed.long(), scales, 32),
                lambda: hx.nn.linear_w4(x, packed, scales.float(), 32), lambda: hx.nn.linear_w4(x, packed.t().contiguous().t(), scales, 32),
                lambda: hx.nn.linear_w4(x, packed, scales, 32, bias[:31]), lambda: hx.nn.linear_w4(x, packed, scales, 32, bias.float()),
                lambda: hx.nn.linear_w4(x, packed, scales, 32, residual=x), lambda: hx.nn.linear_w4(x, packed, scales.cpu(), 32),
                lambda: hx.nn.quantize_w4(x, 20), lambda: hx.nn.quantize_w4(x[0])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        hx.nn.linear_w4(x.half(), packed, scales.half(), 32)
    with pytest.raises(RuntimeError):
        hx.nn.linear_w4(x.clone().requires_grad_(), packed, scales, 32)
    assert hx.nn.linear_w4(x[:0], packed, scales, 32).shape == (0, 32)
    L, c, p = N.lib(), hx.context(), x.data_ptr()
    for rows, in_f, out_f, group in ((0, 64, 32, 32), (2, 0, 32, 32), (2, 64, 0, 32), (2, 64, 32, 0), (2, 64, 32, 48)):
        assert L.hx_linear_w4_fwd(c.handle, 1, p, p, p, None, None, p, rows, in_f, out_f, group) == N.HX_ERR_INVALID
    assert L.hx_linear_w4_fwd(c.handle, 1, p, p, p, None, None, p, 16 * 65535 + 1, 64, 32, 32) == N.HX_ERR_UNSUPPORTED
    assert L.hx_linear_w4_fwd(c.handle, 1, p, None, p, None, None, p, 2, 64, 32, 32) == N.HX_ERR_INVALID
    assert L.hx_quantize_w4(c.handle, 1, p, None, p, 64, 32, 32) == N.HX_ERR_INVALID
    assert L.hx_quantize_w4(None, 1, p, p, p, 64, 32, 32) == N.HX_ERR_INVALID


def test_sizes_past_the_limits_are_refused():
    L, c, p = N.lib(), hx.context(), torch.zeros(64, device="cuda").data_ptr()
    big = (1 << 30) + 32
    for rows, i, o, group in ((1, big, 1, 32), (1, 32, big, 32), (1, 32, 32, big), (16 * 65535 + 1, 32, 32, 32)):
        assert L.hx_linear_w4_fwd(c.handle, 0, p, p, p, None, None, p, rows, i, o, group) == N.HX_ERR_UNSUPPORTED
    assert L.hx_quantize_w4(c.handle, 0, p, p, p, 32, 32, big) == N.HX_ERR_UNSUPPORTED


@pytest.mark.parametrize("mode", [torch.enable_grad, torch.no_grad])
def test_forward_mode_is_refused(mode):
    """A dual tensor does not require a gradient, but its tangent must not be lost."""
    x, packed, scales = _make(2, 64, 32, 32, BF16)
    bias, res = torch.zeros(32, device="cuda", dtype=BF16), torch.zeros(2, 32, device="cuda", dtype=BF16)
    args = dict(x=x, scales=scales, bias=bias, residual=res)
    with mode(), torch.autograd.forward_ad.dual_level():
        for name, a in args.items():
            dual = torch.autograd.forward_ad.make_dual(a, torch.ones_like(a))
            with pytest.raises(RuntimeError):
                hx.nn.linear_w4(packed=packed, group=32, **{**args, name: dual})
        hx.nn.linear_w4(packed=packed, group=32, **args)  # without a tangent


def test_first_calls_of_two_contexts_at_once():
    """In a process of its own: two threads with a context each make a kernel's first calls, one of a form that needs
    less shared memory than the other's. Both are launched, then and later."""
    import subprocess
    import sys

    code = """
import threading, torch
import haelixe_b200 as hx
from haelixe_b200 import _native as N
L, bad = N.lib(), []
ctx = [hx.CudaContext(0), hx.CudaContext(0)]
stream = torch.cuda.Stream()
for c in ctx:
    c.use_stream(stream)
x = torch.zeros(33, 512, device="cuda")
y = [torch.zeros(33, 8192, device="cuda") for _ in ctx]
packed, scales = torch.zeros(64, 8192, dtype=torch.int32, device="cuda"), torch.zeros(16, 8192, device="cuda")
torch.cuda.synchronize()
def call(i, dtype, rows, group):
    out = (8192, 64)[i]
    st = L.hx_linear_w4_fwd(ctx[i].handle, dtype, x.data_ptr(), packed.data_ptr(), scales.data_ptr(), None, None,
                            y[i].data_ptr(), rows, 512, out, group)
    if st:
        bad.append((out, dtype, rows, group, N.last_error(ctx[i].handle)))
for dtype in (0, 1):
    for rows in (8, 16, 33):
        for group in (32, 64, 128):
            start = threading.Barrier(2)
            def go(i):
                start.wait()
                call(i, dtype, rows, group)
            ts = [threading.Thread(target=go, args=(i,)) for i in range(2)]
            [t.start() for t in ts]
            [t.join() for t in ts]
            for i in (0, 1, 0):
                call(i, dtype, rows, group)
torch.cuda.synchronize()
assert not bad, bad
"""
    root = __file__.rsplit("/tests/", 1)[0]
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("in_f,out_f,group", [
    (100, 4612, 32), (136, 8192, 64), (1000, 4612, 96), (2048, 8196, 128), (4104, 4612, 192), (5000, 8192, 32),
    (8192, 4864, 64), (16384, 4612, 128),
])
@pytest.mark.parametrize("rows", [1, 8, 9, 16, 17, 33])
def test_wide_outputs(dtype, in_f, out_f, group, rows):
    """Outputs wide enough that two warps share each unit of k, with units that do and do not divide among the
    groups of warps and the CTAs of a cluster."""
    x, packed, scales = _make(rows, in_f, out_f, group, dtype, rows + in_f)
    w = _weight(packed, scales, group, in_f)
    g = _gen(3)
    bias, res = (torch.randn(s, generator=g, device="cuda").to(dtype) for s in ((out_f,), (rows, out_f)))
    y = hx.nn.linear_w4(x, packed, scales, group, bias, res)
    _check(y, x, w, bias, res)
    for _ in range(3):
        assert torch.equal(hx.nn.linear_w4(x, packed, scales, group, bias, res), y)


@pytest.mark.parametrize("in_f,group", [(1000, 64), (8200, 128)])
@pytest.mark.parametrize("rows", [17, 32, 33])
def test_wide_outputs_of_many_rows(in_f, group, rows):
    """Over 16 rows in bf16 a CTA is half as wide, so two warps share a unit from half as many columns on."""
    x, packed, scales = _make(rows, in_f, 2400, group, BF16, rows)
    y = hx.nn.linear_w4(x, packed, scales, group)
    _check(y, x, _weight(packed, scales, group, in_f))
    assert torch.equal(hx.nn.linear_w4(x, packed, scales, group), y)


def test_sizes_past_an_int_are_refused():
    x, packed, scales = _make(1, 64, 32, 32, BF16)
    with pytest.raises(ValueError):
        hx.nn.linear_w4(x.expand(2**32 + 1, 64), packed, scales, 32)
    with pytest.raises(ValueError):
        hx.nn.linear_w4(x, packed, scales[:1], 2**32 + 64)  # would be a group of 64
    with pytest.raises(ValueError):
        hx.nn.quantize_w4(x[:, :1].expand(1, 2**32 + 1))
