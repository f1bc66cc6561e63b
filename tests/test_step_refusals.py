"""What step tables, attention of a chunk and log probabilities refuse, before any
device work: through the C ABI with made-up addresses, and through the public
functions on the CPU."""

import ctypes

import pytest
import torch

from tests.test_abi import _call, _v
from tinyserver_amd import _lib
from tinyserver_amd import kernels as K

R = ctypes.byref
INVALID, UNSUPPORTED = _lib.TSA_ERR_INVALID, _lib.TSA_ERR_UNSUPPORTED
BF, F32, I32, I64 = torch.bfloat16, torch.float32, torch.int32, torch.int64


def _views(v):
    return (R(x) if x is not None else None for x in v.values())


def _chunk(max_seqlen=4, **kw):
    q = _v((7, 8, 128))
    v = dict(out=q, q=q, kc=_v((9, 2, 16, 128)), vc=_v((9, 2, 16, 128)), bt=_v((3, 3), I32), ctx=_v((3,), I32),
             cu=_v((4,), I32))
    v.update(kw)
    return _call("tsa_paged_chunk", *_views(v), max_seqlen, 0.1, None, 0, None)


@pytest.mark.parametrize("kw,code,word", [
    (dict(q=_v((7, 128))), INVALID, "3D"), (dict(out=_v((7, 8, 64))), INVALID, "shape"), (dict(out=None), INVALID, "3D"),
    (dict(kc=_v((9, 16, 128))), INVALID, "4D"), (dict(vc=_v((8, 2, 16, 128))), INVALID, "match"),
    (dict(kc=_v((9, 2, 16, 128), F32)), INVALID, "floating"), (dict(out=_v((7, 8, 128), F32)), INVALID, "floating"),
    (dict(kc=_v((9, 2, 16, 128), torch.int8), vc=_v((9, 2, 16, 128), torch.int8)), INVALID, "floating"),
    (dict(kc=_v((9, 3, 16, 128)), vc=_v((9, 3, 16, 128))), INVALID, "multiple"),
    (dict(kc=_v((9, 2, 16, 64)), vc=_v((9, 2, 16, 64))), INVALID, "head_dim"),
    (dict(kc=_v((9, 2, 0, 128)), vc=_v((9, 2, 0, 128))), INVALID, "block_size"),
    (dict(bt=_v((3, 3), I64)), INVALID, "int32"), (dict(bt=_v((3,), I32)), INVALID, "2D"),
    (dict(bt=_v((3, 1 << 26), I32)), INVALID, "too long"), (dict(ctx=_v((2,), I32)), INVALID, "context_lens"),
    (dict(ctx=_v((3,), I64)), INVALID, "context_lens"), (dict(cu=_v((3,), I32)), INVALID, "cu_seqlens"),
    (dict(cu=None), INVALID, "cu_seqlens"), (dict(max_seqlen=-1), INVALID, "max_seqlen"),
    (dict(q=_v((7, 8, 1024)), out=_v((7, 8, 1024)), kc=_v((9, 2, 16, 1024)), vc=_v((9, 2, 16, 1024))), UNSUPPORTED, "512"),
])
def test_chunk(kw, code, word):
    rc, msg = _chunk(**kw)
    assert rc == code and word in msg


def _step(block_size=16, **kw):
    v = dict(bt=_v((3, 5), I32), cu=_v((4,), I32), seq=_v((3,), I32), pos=_v((9,), I32), blk=_v((9,), I32),
             slot=_v((9,), I32), left=_v((1,), I32), tables=_v((6, 5), I32), rows=_v((3,), I32), ctx=_v((3,), I32),
             q=_v((3,), I32), free=_v((20,), I32), num=_v((1,), I32))
    v["left"].data += 64
    v.update(kw)
    return _call("tsa_step_tables", *_views(v), block_size, None)


@pytest.mark.parametrize("kw,word", [
    (dict(tables=_v((6,), I32)), "tables"), (dict(tables=_v((6, 5), I64)), "tables"), (dict(ctx=_v((3,), I64)), "context_lens"),
    (dict(q=_v((2,), I32)), "query_lens"), (dict(rows=_v((2,), I32)), "rows"), (dict(rows=None, tables=_v((2, 5), I32)), "row for each"),
    (dict(bt=_v((2, 5), I32)), "block_tables"), (dict(cu=_v((3,), I32)), "cu_seqlens"), (dict(seq=_v((4,), I32)), "seq_lens"),
    (dict(pos=_v((9,), I64)), "positions"), (dict(blk=_v((8,), I32)), "block_mapping"), (dict(slot=None), "slot_mapping"),
    (dict(free=_v((20,), I64)), "free_blocks"), (dict(num=_v((2,), I32)), "num_free"), (dict(left=None), "free_left"),
    (dict(free=None), "free_blocks"), (dict(free=None, num=None), "free_blocks"), (dict(block_size=0), "block_size"),
    (dict(num=_v((1,), I32), left=_v((1,), I32)), "may not be"),
])
def test_step(kw, word):
    rc, msg = _step(**kw)
    assert rc == INVALID and word in msg


def _logprobs(**kw):
    v = dict(lp=_v((4,), F32), en=_v((4,), F32), tl=_v((4, 5), F32), tt=_v((4, 5), I64), x=_v((4, 100)), tok=_v((4,), I64))
    v.update(kw)
    return _call("tsa_token_logprobs", *_views(v), None, 0, None)


@pytest.mark.parametrize("kw,code,word", [
    (dict(x=_v((4,))), INVALID, "logits"), (dict(x=_v((4, 100), I32)), INVALID, "logits"), (dict(x=_v((4, 0))), INVALID, "vocabulary"),
    (dict(tok=_v((3,), I64)), INVALID, "tokens"), (dict(tok=_v((4,), F32)), INVALID, "tokens"), (dict(lp=_v((4,))), INVALID, "logprobs"),
    (dict(en=_v((3,), F32)), INVALID, "entropy"), (dict(tl=_v((4, 5))), INVALID, "top_logprobs"), (dict(tt=_v((4, 5), I32)), INVALID, "top_tokens"),
    (dict(tt=_v((4, 4), I64)), INVALID, "top_tokens"), (dict(x=_v((4, 3))), INVALID, "larger"),
    (dict(tl=_v((4, 65), F32), tt=_v((4, 65), I64)), UNSUPPORTED, "64"),
])
def test_logprobs(kw, code, word):
    rc, msg = _logprobs(**kw)
    assert rc == code and word in msg


def test_public_functions():
    """Their own checks come before the device's; tensors on the CPU are refused, whatever they hold."""
    q, kc = torch.zeros(3, 8, 128, dtype=BF), torch.zeros(9, 2, 16, 128, dtype=BF)
    bt, n = torch.zeros(3, 2, dtype=I32), torch.ones(3, dtype=I32)
    cu = torch.zeros(4, dtype=I32)
    with pytest.raises(ValueError, match="3D"):
        K.paged_attention_chunk(q[0], kc, kc, bt, 16, n, cu)
    with pytest.raises(ValueError, match="block_size"):
        K.paged_attention_chunk(q, kc, kc, bt, 8, n, cu)
    with pytest.raises(ValueError, match="2D"):
        K.paged_attention_chunk(q, kc, kc, bt[0], 16, n, cu)
    with pytest.raises(ValueError, match="tables"):
        K.step_tables(bt.long(), n, n, 16, 3)
    with pytest.raises(ValueError, match="query_lens"):
        K.step_tables(bt, n, bt, 16, 3)
    with pytest.raises(ValueError, match="num_free"):
        K.step_tables(bt, n, n, 16, 3, num_free=n[:1])
    with pytest.raises(ValueError, match="num_tokens"):
        K.step_tables(bt, n, n, 16, -1)
    with pytest.raises(ValueError, match="logits"):
        K.token_logprobs(q, n)
    with pytest.raises(ValueError, match="tokens"):
        K.token_logprobs(bt.float(), bt)
    with pytest.raises(ValueError, match="num_top"):
        K.token_logprobs(bt.float(), n, -1)
    for call in (lambda: K.paged_attention_chunk(q, kc, kc, bt, 16, n, cu), lambda: K.step_tables(bt, n, n, 16, 3),
                 lambda: K.token_logprobs(bt.float(), n, 2)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_argument_counts_of_the_extension():
    names = _lib.host().step_entries()
    assert set(names) == {"tsa_step_tables", "tsa_paged_chunk", "tsa_token_logprobs"}
    assert not set(names) & {*_lib.host().entries(), *_lib.host().extra_entries()}
    for name in names:
        with pytest.raises(TypeError, match=name):
            _lib.call(name)
        with pytest.raises(TypeError, match=f"{name} takes"):
            _lib.call(name, *([None] * (len(_lib.SIGNATURES[name][1]) + 1)))
    x, n = torch.zeros(4, 9), torch.zeros(4)
    rc = _lib.call("tsa_token_logprobs", n, n, x, x, x, n, 0, 0, 0)
    assert rc == INVALID and b"tokens" in _lib.load().tsa_last_error()


def test_workspace_sizes():
    """Nothing for sizes that are refused or have nothing to do; within bounds for the largest."""
    lib = _lib.load()
    assert lib.tsa_paged_chunk_workspace_bytes(0, 5, 5, 8, 2, 128, 4, 16) == 0
    assert lib.tsa_paged_chunk_workspace_bytes(3, 0, 0, 8, 2, 128, 4, 16) == 0
    assert lib.tsa_paged_chunk_workspace_bytes(3, 5, 5, 8, 3, 128, 4, 16) == 0
    assert lib.tsa_token_logprobs_workspace_bytes(0, 100, 5) == 0
    for shape in ((65535, (1 << 27) - 1, (1 << 27) - 1, 65535, 65535, 128, (1 << 26) - 1, 1),
                  (65535, 1 << 26, 1, 65535, 1, 128, 1 << 20, 64), (1, 1, 1, 1, 1, 128, 1, 16)):
        assert 0 <= lib.tsa_paged_chunk_workspace_bytes(*shape) <= 1 << 28
    for shape in ((1 << 30, 1 << 29, 64), (1, 1 << 29, 64), (1, 151936, 64), (1 << 20, 8, 8)):
        assert 0 <= lib.tsa_token_logprobs_workspace_bytes(*shape) <= 1 << 28
