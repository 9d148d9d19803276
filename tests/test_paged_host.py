"""CPU checks of the paged cache's entry points: what they refuse, without a GPU call."""
import ctypes

import pytest
import torch

import haelixe_b200 as hx
from haelixe_b200 import _native as N


def _cache(**over):
    f = dict(k=4096, v=8192, block_table=256, stride_page=16 * 4 * 64, stride_slot=4 * 64, stride_head=64,
             table_stride=8, num_pages=10, page_size=16, H=4, D=64, num_seqs=3, max_pages=8)
    f.update(over)
    return N.PagedCache(*(f[n] for n, _ in N.PagedCache._fields_))


def _size(cache, dtype=N.HX_BF16, heads=8):
    out = ctypes.c_uint64()
    return N.lib().hx_paged_attention_workspace_size(dtype, ctypes.byref(cache), heads, ctypes.byref(out)), out.value


def test_workspace_size_of_a_good_cache():
    st, n = _size(_cache())
    # A 256-byte multiple for 3 sequences, then two parts for each of up to 1024 workers, of 8 heads
    # of head_dim floats, the maximum and the sum, in 16-byte pieces.
    assert st == N.HX_OK and n == 256 + 2 * 1024 * 8 * (64 + 4) * 4


@pytest.mark.parametrize("over,status", [
    (dict(num_pages=0), N.HX_ERR_INVALID),
    (dict(page_size=0), N.HX_ERR_INVALID),
    (dict(H=0), N.HX_ERR_INVALID),
    (dict(D=0), N.HX_ERR_INVALID),
    (dict(max_pages=0), N.HX_ERR_INVALID),
    (dict(num_seqs=-1), N.HX_ERR_INVALID),
    (dict(D=60), N.HX_ERR_UNSUPPORTED),
    (dict(D=264), N.HX_ERR_UNSUPPORTED),
    (dict(k=None), N.HX_ERR_INVALID),
    (dict(v=None), N.HX_ERR_INVALID),
    (dict(block_table=None), N.HX_ERR_INVALID),
    (dict(k=4098), N.HX_ERR_INVALID),
    (dict(stride_slot=4 * 64 + 4), N.HX_ERR_INVALID),
    (dict(stride_slot=32), N.HX_ERR_INVALID),
    (dict(stride_head=-64), N.HX_ERR_INVALID),
    (dict(stride_page=-64), N.HX_ERR_INVALID),
    (dict(table_stride=7), N.HX_ERR_INVALID),
])
def test_bad_caches_are_refused(over, status):
    assert _size(_cache(**over))[0] == status


@pytest.mark.parametrize("heads", [0, -4, 6])
def test_query_heads_must_divide(heads):
    assert _size(_cache(), heads=heads)[0] == N.HX_ERR_INVALID


def test_unknown_dtype_and_missing_outputs():
    assert _size(_cache(), dtype=7)[0] == N.HX_ERR_INVALID
    assert N.lib().hx_paged_attention_workspace_size(N.HX_BF16, ctypes.byref(_cache()), 4, None) == N.HX_ERR_INVALID
    assert N.lib().hx_paged_attention_workspace_size(N.HX_BF16, None, 4, ctypes.byref(ctypes.c_uint64())) \
        == N.HX_ERR_INVALID


def test_null_context():
    L = N.lib()
    c = _cache()
    assert L.hx_paged_append(None, N.HX_BF16, ctypes.byref(c), 1, None, None, None, None, 0, None, None, 0.0) \
        == N.HX_ERR_INVALID
    assert L.hx_paged_attention(None, N.HX_BF16, ctypes.byref(c), 4, None, None, None, None, 1.0, None, 0) \
        == N.HX_ERR_INVALID


def test_cpu_tensors_are_refused():
    k = torch.zeros(2, 16, 1, 64)
    with pytest.raises(RuntimeError):
        hx.PagedKVCache(k, k, torch.zeros(1, 2, dtype=torch.int32))


def test_a_tangent_is_seen():
    x = torch.ones(3)
    assert not hx.attention.has_tangent(x, None)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, x)
        assert not dual.requires_grad and not hx.attention.has_tangent(x, None)
        assert hx.attention.has_tangent(None, dual) and hx.attention.has_tangent(dual[1:], x)
    assert not hx.attention.has_tangent(x)


def test_sizes_past_an_int_are_refused():
    """ctypes keeps the low 32 bits of a larger one, so 2^32 + 1 rows would be one."""
    assert ctypes.c_int(2**32 + 1).value == 1
    N.check_sizes("x", 0, 1, 2**31 - 1)
    for n in (2**31, 2**32 + 1):
        with pytest.raises(ValueError):
            N.check_sizes("x", 5, n)
    with pytest.raises(ValueError):
        hx.nn.token_logprobs(torch.zeros(1, 4).expand(2**32 + 1, 4), torch.zeros(1, dtype=torch.int32).expand(2**32 + 1))
