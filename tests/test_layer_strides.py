"""Operands whose rows share memory (a broadcast one has a row stride of 0,
which means "dense" to the C entry points) are refused before any launch."""

import pytest
import torch

import cube_awq_b200 as cawq
from cube_awq_b200 import layer_ops
from cube_awq_b200.errors import ShapeError

F16, F32, F8 = torch.float16, torch.float32, torch.float8_e4m3fn


def test_rows_that_share_memory_are_refused():
    row = torch.zeros(64, dtype=F16)
    for bad in (row.expand(8, 64), torch.zeros(200, dtype=F16).as_strided((3, 64), (63, 1)),
                row[:1].expand(8, 1)):
        with pytest.raises(ShapeError):
            layer_ops._rows("x", bad, bad.shape, F16)
    for good in (row.expand(1, 64), row.expand(0, 64), row.view(1, 64), row.view(64, 1),
                 torch.zeros(3, 80, dtype=F16)[:, 8:72], row.as_strided((1, 64), (0, 1))):
        layer_ops._rows("x", good, good.shape, F16)


def test_tokens_that_share_memory_are_refused():
    one = torch.zeros(1, 4, 128, dtype=F16)
    for bad in (one.expand(8, 4, 128), torch.zeros(2000, dtype=F16).as_strided((3, 4, 128), (504, 128, 1))):
        with pytest.raises(ShapeError):
            layer_ops._heads("q", bad, 4, 128, F16)
    assert layer_ops._heads("q", one.expand(1, 4, 128), 4, 128, F16) == 512
    assert layer_ops._heads("q", one.as_strided((1, 4, 128), (0, 128, 1)), 4, 128, F16) == 512
    assert layer_ops._heads("q", torch.zeros(3, 6, 128, dtype=F16)[:, :4], 4, 128, F16) == 768
    assert layer_ops._heads("q", one.expand(0, 4, 128), 4, 128, F16) == 512


@pytest.mark.gpu
@pytest.mark.parametrize("compiled", [True, False])
def test_calls_refuse_broadcast_operands(cuda_device, compiled, monkeypatch):
    if not compiled:
        monkeypatch.setattr(layer_ops, "_torch_ext", lambda: None)
    z = lambda *s, dt=F16: torch.zeros(s, dtype=dt, device=cuda_device)  # noqa: E731
    n, d = 8, 64
    x, w, row = z(n, d), z(d), z(d).expand(n, d)
    for args, kw in (((row, w), {}), ((x, w), dict(residual=row)), ((x, w), dict(out=row)),
                     ((x, w), dict(residual=x, residual_out=row))):
        with pytest.raises(ShapeError):
            cawq.rms_norm(*args, **kw)
        if "out" not in kw:
            with pytest.raises(ShapeError):
                cawq.rms_norm_fp8(*args, **kw)
    with pytest.raises(ShapeError):
        cawq.rms_norm_fp8(x, w, out=z(d, dt=F8).expand(n, d))
    with pytest.raises(ShapeError):
        cawq.rms_norm_fp8(x, w, scales=z(1, dt=F32).expand(n))
    kc, vc, q, k = z(4, 2, 16, 128), z(4, 2, 16, 128), z(n, 4, 128), z(n, 2, 128)
    q1, k1 = z(1, 4, 128).expand(n, 4, 128), z(1, 2, 128).expand(n, 2, 128)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda_device)  # noqa: E731
    table, lens, rope = torch.zeros((n, 1), dtype=torch.int32, device=cuda_device), i32([1] * n), \
        z(16, 128, dt=F32)
    each = (kc, vc, table, lens)
    one = (kc, vc, table[:1], i32([n]), i32([0, n]))
    for a, kw in ((dict(q=q1), {}), (dict(), dict(out=q1))):
        qq = a.get("q", q)
        for call in (lambda: cawq.attention_decode(qq, *each, **kw),
                     lambda: cawq.attention_prefill(qq, *one, **kw),
                     lambda: cawq.rope_append(qq, k, k, rope, *each, **kw)):
            with pytest.raises(ShapeError):
                call()
    for kk, vv in ((k1, k), (k, k1)):
        with pytest.raises(ShapeError):
            cawq.rope_append(q, kk, vv, rope, *each)
    # a table of all sequences in one row has no row stride of its own either
    with pytest.raises(ShapeError):
        cawq.attention_decode(q, kc, vc, table[:1].expand(n, 1), lens)
    # one row has no stride: what broadcasting made of it does not matter
    y, h = cawq.rms_norm(z(d).expand(1, d), w, residual=x[:1])
    assert y.shape == (1, d) and torch.equal(h, x[:1])
    assert cawq.attention_decode(z(4, 128).expand(1, 4, 128), kc, vc, table[:1], lens[:1]).shape == (1, 4, 128)
    assert cawq.device_error() == 0
