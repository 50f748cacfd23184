"""AWQDecoderLayer against the layer in 64 bits: prompts of several lengths in
one call, then single tokens, over one paged cache.

Bound: every stage rounds to F once (norm, qkv, rotary, attention twice, o,
residual, norm, gate_up, down: ten roundings, each at most u = half a unit in
the last place in relative size, and the attention's and the linears' gains
are about one), so outputs are within 16 u in the 2-norm."""

import pytest
import torch

import cube_awq_b200 as cawq
from cube_awq_b200.errors import ShapeError
from cube_awq_b200.synth import make_weights
from layer_ref import ROUND

pytestmark = pytest.mark.gpu

HIDDEN, INTER, NQ, NKV, D, G = 512, 1024, 4, 2, 128, 128


def _layer(dtype, dev, window, sinks, seed=0):
    def linear(k, n, s):
        w = make_weights(k, n, G, dtype, dev, seed=seed + s)
        return cawq.AWQGEMMLinear(w.qweight, w.qzeros, w.scales * 0.1)

    q, k, v = linear(HIDDEN, NQ * D, 1), linear(HIDDEN, NKV * D, 2), linear(HIDDEN, NKV * D, 3)
    o, gate, up, down = (linear(NQ * D, HIDDEN, 4), linear(HIDDEN, INTER, 5),
                         linear(HIDDEN, INTER, 6), linear(INTER, HIDDEN, 7))
    g = torch.Generator(device=dev).manual_seed(seed)
    n1, n2 = ((1 + 0.1 * torch.randn(HIDDEN, generator=g, device=dev)).to(dtype) for _ in range(2))
    layer = cawq.AWQDecoderLayer(n1, cawq.AWQQKVLinear(q, k, v), o, n2,
                                 cawq.AWQGateUpSiluMul(gate, up), down, NQ, NKV, D, 1e-6, window,
                                 sinks)
    deq = lambda l: cawq.dequantize_awq(l.qweight, l.qzeros, l.scales, G, order="awq").double()  # noqa: E731
    return layer, [deq(l) for l in (q, k, v, o, gate, up, down)], n1.double(), n2.double()


def _reference(x, r, ws, n1, n2, rope, window, sinks):
    """The layer over one whole sequence x [n, hidden] with residual r, in fp64."""
    norm = lambda t, w: t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w  # noqa: E731
    wq, wk, wv, wo, wg, wu, wd = ws
    n = x.shape[0]
    h = x + r
    y = norm(h, n1)
    c, s = rope[:n, None, :D // 2].double(), rope[:n, None, D // 2:].double()

    def turn(t):
        a, b = t[..., :D // 2], t[..., D // 2:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    q, k = turn((y @ wq).view(n, NQ, D)), turn((y @ wk).view(n, NKV, D))
    v = (y @ wv).view(n, NKV, D)
    k, v = (t.repeat_interleave(NQ // NKV, 1) for t in (k, v))
    i, j = torch.arange(n, device=x.device)[:, None], torch.arange(n, device=x.device)[None]
    seen = j <= i
    if window:
        seen &= (j > i - window) | (j < sinks)
    a = torch.einsum("qhd,khd->hqk", q, k) * D ** -0.5
    a = torch.softmax(a.masked_fill(~seen, float("-inf")), -1)
    h = h + torch.einsum("hqk,khd->qhd", a, v).reshape(n, -1) @ wo
    y = norm(h, n2)
    return (torch.nn.functional.silu(y @ wg) * (y @ wu)) @ wd, h


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("window,sinks", [(None, 0), (48, 4)])
def test_prompts_then_tokens(cuda_device, dtype, window, sinks):
    dev = cuda_device
    layer, ws, n1, n2 = _layer(dtype, dev, window, sinks)
    lens, page, steps = [37, 150, 5], 16, 3
    g = torch.Generator(device=dev).manual_seed(9)
    xs = [torch.randn((n + steps, HIDDEN), generator=g, device=dev).to(dtype) for n in lens]
    rs = [torch.randn((n + steps, HIDDEN), generator=g, device=dev).to(dtype) for n in lens]
    width = -(-(max(lens) + steps) // page)
    table = torch.randperm(width * len(lens), generator=g, device=dev).int().view(len(lens), width)
    kc = torch.full((width * len(lens), NKV, page, D), float("nan"), dtype=dtype, device=dev)
    vc = kc.clone()
    rope = cawq.rope_table(256, D, device=dev)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    cawq.device_error()
    outs = [[] for _ in lens]
    x, r = (torch.cat([t[:n] for t, n in zip(ts, lens)]) for ts in (xs, rs))
    y, h = layer(x, r, rope, kc, vc, table, i32(lens), q_start=i32(starts))
    for b, n in enumerate(lens):
        outs[b].append((y[starts[b]:starts[b + 1]], h[starts[b]:starts[b + 1]]))
    for step in range(steps):
        x, r = (torch.stack([t[n + step] for t, n in zip(ts, lens)]) for ts in (xs, rs))
        y, h = layer(x, r, rope, kc, vc, table, i32([n + step + 1 for n in lens]))
        for b in range(len(lens)):
            outs[b].append((y[b:b + 1], h[b:b + 1]))
    assert cawq.device_error() == 0
    for b in range(len(lens)):
        want = _reference(xs[b].double(), rs[b].double(), ws, n1, n2, rope, window, sinks)
        for k in range(2):
            got = torch.cat([o[k] for o in outs[b]]).double()
            rel = float((got - want[k]).norm() / want[k].norm())
            assert rel <= 16 * ROUND[dtype], (b, k, rel)


def test_first_layer_has_no_residual(cuda_device):
    layer, ws, n1, n2 = _layer(torch.float16, cuda_device, None, 0)
    x = torch.randn((1, HIDDEN), device=cuda_device).half()
    kc = torch.zeros((2, NKV, 16, D), dtype=torch.float16, device=cuda_device)
    rope = cawq.rope_table(32, D, device=cuda_device)
    table = torch.tensor([[1]], dtype=torch.int32, device=cuda_device)
    one = torch.ones(1, dtype=torch.int32, device=cuda_device)
    keep = x.clone()
    y, h = layer(x, None, rope, kc, kc.clone(), table, one)
    want = _reference(x.double(), torch.zeros_like(x).double(), ws, n1, n2, rope, None, 0)
    for got, ref in zip((y, h), want):
        assert float((got.double() - ref).norm() / ref.norm()) <= 16 * ROUND[torch.float16]
    assert torch.equal(x, keep)


def test_sizes_that_do_not_fit_are_refused(cuda_device):
    layer, *_ = _layer(torch.float16, cuda_device, None, 0)
    args = (layer.input_norm, layer.qkv, layer.o, layer.post_norm, layer.gate_up, layer.down)
    for heads in ((NQ * 2, NKV, D), (NQ, NKV * 2, D), (NQ, NKV, 64)):
        with pytest.raises(ShapeError):
            cawq.AWQDecoderLayer(*args, *heads)
    with pytest.raises(ShapeError):
        cawq.AWQDecoderLayer(layer.input_norm[:256], *args[1:], NQ, NKV, D)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_no_tokens(cuda_device, dtype):
    # an empty batch, and a batch whose sequences have no new tokens
    layer, *_ = _layer(dtype, cuda_device, None, 0)
    x = torch.empty((0, HIDDEN), dtype=dtype, device=cuda_device)
    kc = torch.ones((4, NKV, 16, D), dtype=dtype, device=cuda_device)
    vc, rope = kc.clone(), cawq.rope_table(32, D, device=cuda_device)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=cuda_device)  # noqa: E731
    for r in (x, None):
        for table, lens, starts in ((i32(0, 2), i32(0), None), (i32(0, 2), i32(0), i32(1)),
                                    (i32(2, 2), i32(2) + 3, i32(3))):
            y, h = layer(x, r, rope, kc, vc, table, lens, q_start=starts)
            assert y.shape == h.shape == (0, HIDDEN) and y.dtype == h.dtype == dtype
    assert (kc == 1).all() and (vc == 1).all() and cawq.device_error() == 0
