"""What the 8-bit cache, windowed and tree attention refuse, before any device
work: through the C ABI with made-up addresses, and through the public functions
on the CPU."""

import ctypes

import pytest
import torch

from tests.test_abi import _call, _v
from tinyserver_amd import _lib
from tinyserver_amd import kernels as K

R = ctypes.byref
INVALID, UNSUPPORTED = _lib.TSA_ERR_INVALID, _lib.TSA_ERR_UNSUPPORTED
E4, I8, BF, F32 = torch.float8_e4m3fn, torch.int8, torch.bfloat16, torch.float32


def _store(**kw):
    v = dict(k=_v((2, 5, 128)), v=_v((2, 5, 128)), kc=_v((9, 2, 16, 128), E4), vc=_v((9, 2, 16, 128), E4),
             ks=_v((9, 2, 16), F32), vs=_v((9, 2, 16), F32), bt=_v((3, 4), torch.int32), cu=_v((4,), torch.int32), pos=None)
    v.update(kw)
    return _call("tsa_store_kv_quantized", *(R(x) if x is not None else None for x in v.values()), None)


@pytest.mark.parametrize("kw,word", [
    (dict(k=None), "3D"), (dict(k=_v((2, 5, 128), torch.int32)), "floating"), (dict(v=_v((2, 5, 128), F32)), "floating"),
    (dict(v=_v((2, 4, 128))), "same shape"), (dict(kc=_v((9, 2, 16, 128), BF)), "8-bit"), (dict(vc=_v((9, 2, 16, 128), I8)), "8-bit"),
    (dict(vc=_v((8, 2, 16, 128), E4)), "same shape"), (dict(ks=_v((9, 2, 16))), "float32"), (dict(vs=_v((9, 2, 15), F32)), "head_dim"),
    (dict(ks=None), "3D"), (dict(k=_v((3, 5, 128)), v=_v((3, 5, 128))), "kv heads"),
    (dict(k=_v((2, 5, 64)), v=_v((2, 5, 64))), "head_dim"), (dict(bt=_v((3, 4), torch.int64)), "int32"),
    (dict(cu=_v((3,), torch.int32)), "cu_seqlens"), (dict(pos=_v((4,), torch.int32)), "positions"),
])
def test_store(kw, word):
    rc, msg = _store(**kw)
    assert rc == INVALID and word in msg


def test_load():
    o, kc, sc = _v((5, 2, 128)), _v((9, 2, 16, 128), I8), _v((9, 2, 16), F32)
    bt, cu = _v((3, 4), torch.int32), _v((4,), torch.int32)
    rc, msg = _call("tsa_load_kv_quantized", R(o), R(_v((5, 2, 128), F32)), R(kc), R(kc), R(sc), R(sc), R(bt), R(cu), None, None)
    assert rc == INVALID and "floating" in msg
    rc, msg = _call("tsa_load_kv_quantized", R(_v((2, 5, 128))), R(_v((2, 5, 128))), R(kc), R(kc), R(sc), R(sc), R(bt), R(cu), None, None)
    assert rc == INVALID and "kv heads" in msg
    rc, msg = _call("tsa_load_kv_quantized", R(o), R(o), R(o), R(kc), R(sc), R(sc), R(bt), R(cu), None, None)
    assert rc == INVALID and "4D" in msg


def _decode(window=8, sinks=0, **kw):
    q = _v((4, 8, 128))
    v = dict(out=q, q=q, kc=_v((9, 2, 16, 128)), vc=_v((9, 2, 16, 128)), ks=None, vs=None, bt=_v((4, 3), torch.int32),
             sl=_v((4,), torch.int32))
    v.update(kw)
    return _call("tsa_paged_decode_window", *(R(x) if x is not None else None for x in v.values()), window, sinks, 0.1, None, 0, None)


@pytest.mark.parametrize("kw,code,word", [
    (dict(q=_v((4, 128))), INVALID, "3D"), (dict(kc=_v((9, 3, 16, 128)), vc=_v((9, 3, 16, 128))), INVALID, "multiple"),
    (dict(kc=_v((9, 2, 16, 64)), vc=_v((9, 2, 16, 64))), INVALID, "head_dim"), (dict(vc=_v((8, 2, 16, 128))), INVALID, "match"),
    (dict(kc=_v((9, 2, 16, 128), F32)), INVALID, "floating"), (dict(out=_v((4, 8, 64))), INVALID, "shape"),
    (dict(bt=_v((3, 3), torch.int32)), INVALID, "rows"), (dict(sl=_v((4,), torch.int64)), INVALID, "seq_lens"),
    (dict(window=-1), INVALID, "window"), (dict(sinks=-1), INVALID, "sinks"),
    (dict(kc=_v((9, 2, 16, 128), E4), vc=_v((9, 2, 16, 128), E4)), INVALID, "floating"),
    (dict(ks=_v((9, 2, 16), F32), vs=_v((9, 2, 16), F32)), INVALID, "8-bit"),
    (dict(kc=_v((9, 2, 16, 128), E4), vc=_v((9, 2, 16, 128), E4), ks=_v((9, 2, 16), F32)), INVALID, "scale"),
    (dict(bt=_v((4, 1 << 26), torch.int32)), INVALID, "too long"),
    (dict(q=_v((4, 8, 1024)), out=_v((4, 8, 1024)), kc=_v((9, 2, 16, 1024)), vc=_v((9, 2, 16, 1024))), UNSUPPORTED, "512"),
])
def test_decode(kw, code, word):
    rc, msg = _decode(**kw)
    assert rc == code and word in msg


def _tree(max_nodes=4, **kw):
    q = _v((7, 8, 128))
    v = dict(out=q, q=q, kc=_v((9, 2, 16, 128)), vc=_v((9, 2, 16, 128)), bt=_v((3, 3), torch.int32), sl=_v((3,), torch.int32),
             cu=_v((4,), torch.int32), mask=_v((7, 1), torch.int64))
    v.update(kw)
    return _call("tsa_paged_tree", *(R(x) if x is not None else None for x in v.values()), max_nodes, 0.1, None, 0, None)


@pytest.mark.parametrize("kw,word", [
    (dict(cu=None), "cu_nodes"), (dict(cu=_v((3,), torch.int32)), "cu_nodes"), (dict(mask=None), "tree_mask"),
    (dict(mask=_v((6, 1), torch.int64)), "tree_mask"), (dict(mask=_v((7, 1), torch.int32)), "tree_mask"),
    (dict(mask=_v((7, 0), torch.int64)), "word"), (dict(max_nodes=8), "max_nodes"), (dict(max_nodes=-1), "max_nodes"),
    (dict(sl=_v((2,), torch.int32)), "context_lens"), (dict(kc=_v((9, 2, 16, 128), I8), vc=_v((9, 2, 16, 128), I8)), "floating"),
])
def test_tree(kw, word):
    rc, msg = _tree(**kw)
    assert rc == INVALID and word in msg


@pytest.mark.parametrize("window,sinks,word", [(0, 0, "window"), (-3, 0, "window"), (4, -1, "sinks")])
def test_prefill(window, sinks, word):
    q, k, cu = _v((10, 8, 128)), _v((10, 2, 128)), _v((3,), torch.int32)
    rc, msg = _call("tsa_varlen_prefill_window", R(q), R(q), R(k), R(k), R(cu), R(cu), 6, 6, window, sinks, 0.1, None)
    assert rc == INVALID and word in msg
    rc, msg = _call("tsa_varlen_prefill_window", R(q), R(q), R(_v((10, 3, 128))), R(_v((10, 3, 128))), R(cu), R(cu), 6, 6, 4, 0,
                    0.1, None)
    assert rc == INVALID and "divisible" in msg


def test_public_functions():
    """Their own checks come before the device's; tensors on the CPU are refused, whatever they hold."""
    q, kc = torch.zeros(3, 8, 128, dtype=BF), torch.zeros(9, 2, 16, 128, dtype=BF)
    bt, sl = torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="window"):
        K.paged_attention_window(q, kc, kc, bt, 16, sl, 0)
    with pytest.raises(ValueError, match="sinks"):
        K.paged_attention_window(q, kc, kc, bt, 16, sl, 4, -1)
    with pytest.raises(ValueError, match="block_size"):
        K.paged_attention_window(q, kc, kc, bt, 8, sl, 4)
    with pytest.raises(ValueError, match="3D"):
        K.paged_attention_quantized(q[0], kc, kc, kc, kc, bt, 16, sl)
    with pytest.raises(ValueError, match="2D"):
        K.paged_attention_tree(q, kc, kc, bt[0], 16, sl, sl, sl.long())
    with pytest.raises(ValueError, match="int64"):
        K.paged_attention_tree(q, kc, kc, bt, 16, sl, sl, sl)
    with pytest.raises(ValueError, match="window"):
        K.flash_attn_varlen_window(q, q, q, sl, sl, 3, 3, 0)
    with pytest.raises(ValueError, match="sinks"):
        K.flash_attn_varlen_window(q, q, q, sl, sl, 3, 3, 4, -2)
    with pytest.raises(ValueError, match="3D"):
        K.flash_attn_varlen_window(q[0], q, q, sl, sl, 3, 3, 4)
    with pytest.raises(ValueError, match="same shape"):
        K.store_kv_cache_quantized(q, q[:2], kc, kc, kc, kc, bt, sl)
    with pytest.raises(ValueError, match="4D"):
        K.load_kv_cache_quantized(q, q, q, q, bt, sl, 3)
    for call in (lambda: K.paged_attention_window(q, kc, kc, bt, 16, sl, 4),
                 lambda: K.paged_attention_tree(q, kc, kc, bt, 16, sl, torch.zeros(4, dtype=torch.int32), sl.long()),
                 lambda: K.flash_attn_varlen_window(q, q[:, :2], q[:, :2], sl, sl, 3, 3, 4),
                 lambda: K.load_kv_cache_quantized(kc, kc, kc, kc, bt, sl, 3)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_argument_counts_of_the_extension():
    """The entry points beyond the reference's path take what their bindings say."""
    names = _lib.host().extra_entries()
    assert len(names) == 5 and not set(names) & set(_lib.host().entries())
    for name in names:
        with pytest.raises(TypeError, match=name):
            _lib.call(name)
        kinds = _lib.SIGNATURES[name][1]
        with pytest.raises(TypeError, match=f"{name} takes"):
            _lib.call(name, *([None] * (len(kinds) + 1)))
    q, kc = torch.zeros(4, 7, 128, dtype=BF), torch.zeros(9, 2, 16, 128, dtype=I8)
    sc, bt, sl = torch.zeros(9, 2, 16), torch.zeros(4, 3, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    rc = _lib.call("tsa_paged_decode_window", q, q, kc, kc, sc, sc, bt, sl, 0, 0, 0.1, 0, 0, 0)
    assert rc == INVALID and b"multiple" in _lib.load().tsa_last_error()
    rc = _lib.call("tsa_paged_decode", q, q, kc, kc, bt, sl, 0.1, 0, 0, 0, 0)  # the 16-bit decode takes no 8-bit cache
    assert rc == INVALID and b"floating" in _lib.load().tsa_last_error()


@pytest.mark.parametrize("shape", [
    (65535, 1, 65535, 65535, 128, 1 << 20, 64, 0, 0),
    (65535, 1, 65535, 1, 512, (1 << 27) - 1, 1, 0, 0),
    (65535, 1 << 40, 65535, 1, 128, 1 << 20, 64, 0, 0),
    (1, 1 << 30, 64, 8, 128, 1 << 26, 1, 0, 0),
    (4097, 1, 32, 8, 128, 1024, 16, 0, 0),
    (8193, 1, 32, 8, 128, 1024, 16, 1000, 70000),
])
def test_workspace_of_large_calls(shape):
    """Sizes stay within what the sequences of one launch need, however large the batch and the table."""
    size = _lib.load().tsa_paged_rows_workspace_bytes(*shape)
    b, _, hq, hkv, d = shape[:5]
    g = min(hq // hkv, 16)
    units = min(1 << 22, min(b, 4096) * hkv * -(-(hq // hkv) // 16)) + 65536
    assert 0 <= size <= max(units * g, 1 << 22) * (d + 4) * 4 + (1 << 20)
