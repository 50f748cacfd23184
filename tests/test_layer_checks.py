"""Argument checks of the layer operators: what the host refuses, without a GPU
(the C entry points check before any device call)."""

import ctypes

import pytest
import torch

import cube_awq_b200 as cawq
from cube_awq_b200 import _lib
from cube_awq_b200.errors import CubeAwqError, DTypeError, ShapeError

P = ctypes.c_void_p(64)


def _kv(**over):
    kv = _lib.PagedKVC()
    base = dict(k=64, v=64, pages=10, n_kv=2, page_size=16, head_dim=128, stride_page=4096,
                stride_head=2048, stride_token=128, block_table=64, batch=3, table_width=4,
                ld_table=4, seq_lens=64, q_start=None)
    for name, value in {**base, **over}.items():
        setattr(kv, name, value)
    return kv


def _decode(kv, n_q=4, ld_q=0, ld_out=0, dtype=_lib.CAWQ_F16, q=P, out=P, ws=P, nbytes=1 << 30):
    return _lib.lib().cawq_attention_decode(q, out, ctypes.byref(kv) if kv else None, n_q, ld_q,
                                            ld_out, 1.0, 0, 0, dtype, ws, nbytes, None)


def _rope(kv, n_q=4, tokens=3, dtype=_lib.CAWQ_F16, rope=P, rows=100, ld_q=0, q=P):
    return _lib.lib().cawq_rope_append(q, P, P, rope, rows, P, ctypes.byref(kv), tokens, n_q, ld_q,
                                       0, 0, 0, dtype, None)


@pytest.mark.parametrize("over,status,text", [
    (dict(head_dim=96), _lib.CAWQ_ERR_INVALID_SHAPE, "head_dim"),
    (dict(page_size=12), _lib.CAWQ_ERR_INVALID_SHAPE, "page_size"),
    (dict(page_size=0), _lib.CAWQ_ERR_INVALID_SHAPE, "page_size"),
    (dict(n_kv=3), _lib.CAWQ_ERR_INVALID_SHAPE, "multiple of n_kv"),
    (dict(n_kv=0), _lib.CAWQ_ERR_INVALID_SHAPE, "multiple of n_kv"),
    (dict(stride_token=132), _lib.CAWQ_ERR_ALIGNMENT, "multiples of 8"),
    (dict(ld_table=3), _lib.CAWQ_ERR_INVALID_SHAPE, "ld_table"),
    (dict(table_width=1 << 28), _lib.CAWQ_ERR_INVALID_SHAPE, "below 2^31"),
    (dict(pages=1 << 31), _lib.CAWQ_ERR_INVALID_SHAPE, "below 2^31"),
    (dict(k=72), _lib.CAWQ_ERR_ALIGNMENT, "16-byte"),
    (dict(v=None), _lib.CAWQ_ERR_NULL_POINTER, "non-null"),
    (dict(seq_lens=None), _lib.CAWQ_ERR_NULL_POINTER, "non-null"),
    (dict(block_table=None), _lib.CAWQ_ERR_NULL_POINTER, "non-null"),
])
def test_cache_rules(over, status, text):
    kv = _kv(**over)
    assert _decode(kv) == status and text in _lib.last_error()
    assert _rope(kv) == status and text in _lib.last_error()


def test_attention_entry_rules():
    assert _decode(None) == _lib.CAWQ_ERR_NULL_POINTER
    assert _decode(_kv(), dtype=_lib.CAWQ_F32) == _lib.CAWQ_ERR_DTYPE
    assert _decode(_kv(), ld_q=500) == _lib.CAWQ_ERR_INVALID_SHAPE and "q:" in _lib.last_error()
    assert _decode(_kv(), ld_out=516) == _lib.CAWQ_ERR_INVALID_SHAPE
    assert _decode(_kv(), q=None) == _lib.CAWQ_ERR_NULL_POINTER
    assert _decode(_kv(), out=ctypes.c_void_p(72)) == _lib.CAWQ_ERR_ALIGNMENT
    assert _decode(_kv(n_kv=1), n_q=129) == _lib.CAWQ_ERR_INVALID_SHAPE
    assert _decode(_kv(batch=0)) == _lib.CAWQ_OK
    need = _lib.lib().cawq_attention_workspace(ctypes.byref(_kv()), 3, 4)
    if need:
        assert _decode(_kv(), nbytes=need - 1) == _lib.CAWQ_ERR_INVALID_ARGUMENT
        assert _decode(_kv(), ws=None) == _lib.CAWQ_ERR_INVALID_ARGUMENT
    L = _lib.lib()
    st = L.cawq_attention_prefill(P, P, ctypes.byref(_kv()), 9, 4, 0, 0, 1.0, 0, 0, _lib.CAWQ_F16,
                                  P, 1 << 30, None)
    assert st == _lib.CAWQ_ERR_NULL_POINTER and "q_start" in _lib.last_error()


def test_rope_entry_rules():
    assert _rope(_kv(), dtype=_lib.CAWQ_F32) == _lib.CAWQ_ERR_DTYPE
    assert _rope(_kv(), tokens=5) == _lib.CAWQ_ERR_INVALID_SHAPE
    assert "one new token" in _lib.last_error()
    assert _rope(_kv(), rope=ctypes.c_void_p(8)) == _lib.CAWQ_ERR_ALIGNMENT
    assert _rope(_kv(), ld_q=8) == _lib.CAWQ_ERR_INVALID_SHAPE
    assert _rope(_kv(), q=ctypes.c_void_p(24)) == _lib.CAWQ_ERR_ALIGNMENT
    assert _rope(_kv(batch=0), tokens=0) == _lib.CAWQ_OK


def test_norm_entry_rules():
    L = _lib.lib()
    norm = lambda d=64, ld=0, eps=1e-6, dtype=_lib.CAWQ_F16, x=P, res=None, ro=None, rows=2: \
        L.cawq_rms_norm(x, P, res, P, ro, rows, d, ld, 0, 0, 0, eps, dtype, None)  # noqa: E731
    assert norm(dtype=7) == _lib.CAWQ_ERR_DTYPE
    assert norm(d=0) == _lib.CAWQ_ERR_INVALID_SHAPE
    assert norm(ld=63) == _lib.CAWQ_ERR_INVALID_SHAPE
    assert norm(eps=-1.0) == _lib.CAWQ_ERR_INVALID_ARGUMENT
    assert norm(eps=float("nan")) == _lib.CAWQ_ERR_INVALID_ARGUMENT
    assert norm(x=None) == _lib.CAWQ_ERR_NULL_POINTER
    assert norm(ro=P) == _lib.CAWQ_ERR_INVALID_ARGUMENT
    assert norm(rows=0, x=None) == _lib.CAWQ_OK
    st = L.cawq_rms_norm_fp8(P, P, None, P, None, None, 2, 64, 0, 0, 0, 0, 1e-6, _lib.CAWQ_F16, None)
    assert st == _lib.CAWQ_ERR_NULL_POINTER and "scales" in _lib.last_error()


def test_python_layer_refuses_cpu_tensors():
    x = torch.zeros(2, 64, dtype=torch.float16)
    with pytest.raises(CubeAwqError, match="no CPU fallback"):
        cawq.rms_norm(x, x[0])
    kv = torch.zeros(2, 1, 16, 64, dtype=torch.float16)
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(CubeAwqError, match="no CPU fallback"):
        cawq.attention_decode(x.view(1, 2, 64), kv, kv, table, lens)


@pytest.mark.gpu
def test_python_layer_refusals(cuda_device):
    z = lambda *s, dt=torch.float16: torch.zeros(s, dtype=dt, device=cuda_device)  # noqa: E731
    i32 = lambda *s: z(*s, dt=torch.int32)  # noqa: E731
    kv, q, table, lens = z(4, 2, 16, 128), z(3, 4, 128), i32(3, 2), i32(3)
    att = lambda q=q, k=kv, v=kv, t=table, n=lens, **kw: \
        cawq.attention_decode(q, k, v, t, n, **kw)  # noqa: E731
    att()
    for bad, kind in [
            (dict(q=q.float()), DTypeError), (dict(k=kv.bfloat16(), v=kv.bfloat16()), DTypeError),
            (dict(q=q[:2]), ShapeError), (dict(q=z(3, 4, 64)), ShapeError),
            (dict(q=z(3, 5, 128)), ShapeError), (dict(v=kv[:3]), ShapeError),
            (dict(v=z(4, 16, 2, 128).transpose(1, 2)), ShapeError),
            (dict(t=table.long()), DTypeError), (dict(t=i32(2, 2)), ShapeError),
            (dict(n=lens.float()), DTypeError), (dict(out=z(3, 4, 64)), ShapeError),
            (dict(out=q.float()), DTypeError), (dict(window=-1), CubeAwqError),
            (dict(sinks=-1), CubeAwqError), (dict(q=z(3, 128, 4).transpose(1, 2)), ShapeError),
            (dict(k=z(4, 2, 12, 128), v=z(4, 2, 12, 128)), ShapeError),
            (dict(k=z(4, 2, 16, 96), v=z(4, 2, 16, 96), q=z(3, 4, 96)), ShapeError)]:
        with pytest.raises(kind):
            att(**bad)
    with pytest.raises(ShapeError):
        cawq.attention_prefill(q, kv, kv, table, lens, None)
    with pytest.raises(ShapeError):
        cawq.attention_prefill(q, kv, kv, table, lens, i32(3))
    rope, k = z(100, 128, dt=torch.float32), z(3, 2, 128)
    cawq.rope_append(q, k, k, rope, kv, kv.clone(), table, lens)
    for bad in (dict(k=z(3, 4, 128)), dict(rope=z(100, 64, dt=torch.float32)),
                dict(rope=rope.half()), dict(k=z(2, 2, 128))):
        a = {**dict(q=q, k=k, v=k, rope=rope), **bad}
        with pytest.raises(ShapeError):
            cawq.rope_append(a["q"], a["k"], a["v"], a["rope"], kv, kv.clone(), table, lens)
    x, w = z(3, 64), z(64)
    for a, kw, kind in [((x, z(32)), {}, ShapeError), ((x, w.float()), {}, DTypeError),
                        ((x.int(), w.int()), {}, DTypeError),
                        ((x, w), dict(residual=z(2, 64)), ShapeError),
                        ((x, w), dict(residual=x.float()), DTypeError),
                        ((x, w), dict(out=x.float()), DTypeError),
                        ((x, w), dict(residual_out=x), CubeAwqError),
                        ((x, w), dict(eps=-1.0), CubeAwqError),
                        ((z(3, 0), z(0)), {}, ShapeError)]:
        with pytest.raises(kind):
            cawq.rms_norm(*a, **kw)


@pytest.mark.parametrize("over,tokens", [(dict(), 3), (dict(batch=1), 1), (dict(q_start=64), 9),
                                         (dict(table_width=1), 3)])
def test_short_workspaces_are_refused(over, tokens):
    kv = _kv(**over)
    need = _lib.lib().cawq_attention_workspace(ctypes.byref(kv), tokens, 4)
    assert need > 0
    for ws, nbytes in ((P, need - 1), (P, 0), (None, need), (ctypes.c_void_p(72), need)):
        if kv.q_start is None:
            st = _decode(kv, ws=ws, nbytes=nbytes)
        else:
            st = _lib.lib().cawq_attention_prefill(P, P, ctypes.byref(kv), tokens, 4, 0, 0, 1.0, 0, 0,
                                                   _lib.CAWQ_F16, ws, nbytes, None)
        assert st == _lib.CAWQ_ERR_INVALID_ARGUMENT and "workspace" in _lib.last_error()
