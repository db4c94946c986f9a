"""What the entry points of the per-head norm and rotation and of the paged cache refuse, before any launch (no GPU)."""
import ctypes as C

import pytest

from dfdx_b200 import _lib

P = 0x1000          # an address that is never followed: every call below is refused


@pytest.fixture(scope="module")
def lib():
    from dfdx_b200 import build
    build.build()
    return _lib.load()


def st(*s):
    return _lib.strides(s)


def op(pairs=(32, 0, 0), norm=1, freq=P, q_gain=None, k_gain=None):
    o = _lib.HeadOp()
    o.frequencies, o.normalize, o.epsilon, o.q_gain, o.k_gain = freq, norm, 1e-6, q_gain, k_gain
    for i, n in enumerate(pairs):
        o.axis_pairs[i] = n
    return o


def cache(page=64, d=64, heads=2, pages=8, k=P):
    return _lib.KvCacheView(k, P, P, P, pages, heads, page, d)


def batch(seqs=2, tokens=4, max_new=2, cu=P, table_stride=4, max_pages=4):
    return _lib.KvBatch(seqs, tokens, max_new, cu, P, P, table_stride, max_pages)


def forward(lib, o, dtype=_lib.F16, d=64, q=P, qs=None, out=P, outs=None, b=1, s=4):
    qs = qs or st(s * 2 * d, 2 * d, d, 1)
    return lib.b200_qk_norm_rotary_forward(dtype, o, b, s, 2, 2, d, q, qs, q, qs, None, out, outs or qs, out, outs or qs, None)


def test_norm_rotary_forward(lib):
    assert forward(lib, op(), dtype=17) == _lib.ERR_DTYPE
    assert forward(lib, op(), dtype=_lib.F64) == _lib.ERR_UNSUPPORTED
    assert forward(lib, op(), d=63) == _lib.ERR_UNSUPPORTED
    assert forward(lib, op(), d=258) == _lib.ERR_UNSUPPORTED
    assert forward(lib, op(pairs=(33, 0, 0))) == _lib.ERR_SHAPE          # 66 of 64 elements
    assert forward(lib, op(pairs=(16, 16, 1))) == _lib.ERR_SHAPE
    assert forward(lib, op(freq=None)) == _lib.ERR_NULL
    assert forward(lib, op(norm=0, q_gain=P)) == _lib.ERR_UNSUPPORTED
    assert forward(lib, op(), q=None) == _lib.ERR_NULL
    assert forward(lib, op(), out=None) == _lib.ERR_NULL
    assert forward(lib, op(), qs=st(512, 128, 1, 2)) == _lib.ERR_UNSUPPORTED   # unit stride is not the last
    assert forward(lib, op(), outs=st(512, 0, 64, 1)) == _lib.ERR_STRIDE       # tokens would share their output
    assert forward(lib, op(), b=1 << 20, s=1 << 20) == _lib.ERR_LIMIT


def test_norm_rotary_backward(lib):
    s = st(512, 128, 64, 1)

    def backward(o, ggq=P, ws=P, nbytes=1 << 30):
        return lib.b200_qk_norm_rotary_backward(_lib.F16, o, 1, 4, 2, 2, 64, P, s, P, s, None, P, s, P, s, P, s, P, s, ggq, ggq, 0,
                                                ws, nbytes, None)

    need = lib.b200_qk_norm_rotary_backward_workspace_bytes(64)
    assert need == 1024 * 2 * 64 * 4 and lib.b200_qk_norm_rotary_backward_workspace_bytes(1000) == 0
    assert backward(op(), nbytes=need - 1) == _lib.ERR_WORKSPACE
    assert backward(op(), ws=None) == _lib.ERR_NULL
    assert backward(op(norm=0)) == _lib.ERR_UNSUPPORTED                         # no norm, no gain's gradient
    assert backward(op()) == _lib.ERR_STRIDE                                    # one buffer for both gains' gradients


def append(lib, c=None, b=None, o=None, dtype=_lib.F16, q=P, q_heads=4, q_out=P, k=P, ks=None):
    ks = ks or st(128, 64, 1)
    return lib.b200_kv_cache_append(dtype, c or cache(), b or batch(), o, q_heads, q, st(256, 64, 1), k, ks, P, ks, None, q_out,
                                    st(256, 64, 1), None)


def test_append(lib):
    assert append(lib, dtype=99) == _lib.ERR_DTYPE
    assert append(lib, dtype=_lib.F64) == _lib.ERR_UNSUPPORTED
    for page in (0, 8, 24, 256):
        assert append(lib, c=cache(page=page)) == _lib.ERR_UNSUPPORTED
    for d in (0, 16, 80, 160):
        assert append(lib, c=cache(d=d)) == _lib.ERR_UNSUPPORTED
    assert append(lib, c=cache(heads=0)) == _lib.ERR_SHAPE
    assert append(lib, c=cache(k=None)) == _lib.ERR_NULL
    assert append(lib, c=cache(k=P + 8)) == _lib.ERR_UNSUPPORTED                # codes not 16-byte aligned
    assert append(lib, b=batch(cu=None)) == _lib.ERR_NULL
    assert append(lib, b=batch(max_new=5)) == _lib.ERR_SHAPE                    # more new tokens than tokens
    assert append(lib, b=batch(table_stride=3)) == _lib.ERR_STRIDE
    assert append(lib, b=batch(seqs=1 << 31)) == _lib.ERR_LIMIT
    assert append(lib, k=None) == _lib.ERR_NULL
    assert append(lib, ks=st(128, 1, 64)) == _lib.ERR_UNSUPPORTED
    assert append(lib, q_heads=0) == _lib.ERR_SHAPE
    assert append(lib, q_out=None) == _lib.ERR_NULL
    assert append(lib, o=op(pairs=(40, 0, 0))) == _lib.ERR_SHAPE


def test_read(lib):
    assert lib.b200_kv_cache_read(_lib.F64, cache(), 1, P, P, P, None) == _lib.ERR_UNSUPPORTED
    assert lib.b200_kv_cache_read(_lib.F16, cache(), 1, None, P, P, None) == _lib.ERR_NULL
    assert lib.b200_kv_cache_read(_lib.F16, cache(), 1, P, P + 2, P, None) == _lib.ERR_UNSUPPORTED
    assert lib.b200_kv_cache_read(_lib.F16, cache(page=48), 1, P, P, P, None) == _lib.ERR_UNSUPPORTED


def test_attention(lib):
    def attend(c=None, b=None, dtype=_lib.F16, heads=4, q=P, qs=None, causal=1, window=0, os=None, ws=P, nbytes=1 << 40):
        return lib.b200_kv_cache_attention(dtype, c or cache(), b or batch(), heads, q, qs or st(256, 64, 1), 0.125, causal, window,
                                           P, os or st(256, 64, 1), None, ws, nbytes, None)

    assert attend(dtype=_lib.F32) == _lib.ERR_UNSUPPORTED
    assert attend(heads=3) == _lib.ERR_SHAPE and attend(heads=0) == _lib.ERR_SHAPE
    assert attend(causal=0, window=8) == _lib.ERR_UNSUPPORTED
    assert attend(window=1 << 40) == _lib.ERR_LIMIT
    assert attend(q=None) == _lib.ERR_NULL
    assert attend(qs=st(256, 64, 2)) == _lib.ERR_UNSUPPORTED
    assert attend(os=st(0, 64, 1)) == _lib.ERR_STRIDE
    assert attend(c=cache(d=48)) == _lib.ERR_UNSUPPORTED


def test_nothing_to_do_is_no_error(lib):
    assert append(lib, b=batch(seqs=0, tokens=0, max_new=0)) == _lib.OK
    assert lib.b200_kv_cache_attention(_lib.F16, cache(), batch(seqs=0, tokens=0, max_new=0), 4, P, st(256, 64, 1), 1.0, 1, 0, P,
                                       st(256, 64, 1), None, None, 0, None) == _lib.OK
    assert lib.b200_kv_cache_read(_lib.F16, cache(), 0, None, None, None, None) == _lib.OK
    assert lib.b200_kv_cache_attention_workspace_bytes(cache(), batch(), 3, 1, 0) == 0


def test_struct_layouts():
    assert C.sizeof(_lib.HeadOp) == 64 and C.sizeof(_lib.KvCacheView) == 64 and C.sizeof(_lib.KvBatch) == 64
