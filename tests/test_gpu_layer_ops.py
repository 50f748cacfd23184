"""The operators between a decoder layer's linears on the GPU, each against its
definition in 64 bits (layer_ref.py, whose bounds follow from the arithmetic)."""

import pytest
import torch

import cube_awq_b200 as cawq
from cube_awq_b200.errors import CubeAwqError
from layer_ref import FLOOR, ROUND, Cache, F32, assert_within, attention_ref, norm_ref, norm_rel

pytestmark = pytest.mark.gpu

F16, BF16, FP32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _no_device_error(cuda_device):
    cawq.device_error()
    yield
    assert cawq.device_error() == 0


def _randn(shape, dtype, dev, seed, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=dev) * scale).to(dtype)


# ----------------------------------------------------------------- RMS norm
NORM_SIZES = [(1, 4096), (1, 1), (3, 7), (5, 129), (17, 3584), (4, 8200), (2, 16385), (300, 64),
              (1, 40000), (2, 8191), (300, 8192), (2, 16383), (3, 16384), (2, 32768), (300, 1000),
              (301, 20000), (2, 12000)]


def _check_norm(x, w, eps, r, y, h):
    hr, yr = norm_ref(x, w, eps, r)
    u = ROUND[x.dtype]
    assert_within(y, yr, yr.abs() * (u + norm_rel(x.shape[-1]) + 2 * F32) * (1 + u) + FLOOR[x.dtype], "y")
    if r is not None:
        assert_within(h, hr, hr.abs() * (u + 2 * F32) + FLOOR[x.dtype], "h")
    else:
        assert h is None


@pytest.mark.parametrize("dtype", [FP32, F16, BF16])
@pytest.mark.parametrize("rows,d", NORM_SIZES)
@pytest.mark.parametrize("res", [False, True])
def test_rms_norm(cuda_device, dtype, rows, d, res):
    x = _randn((rows, d), dtype, cuda_device, 1)
    r = _randn((rows, d), dtype, cuda_device, 2, 4.0) if res else None
    w = _randn((d,), dtype, cuda_device, 3)
    y, h = cawq.rms_norm(x, w, 1e-5, residual=r)
    _check_norm(x, w, 1e-5, r, y, h)


@pytest.mark.parametrize("dtype", [FP32, F16, BF16])
@pytest.mark.parametrize("rows,d", NORM_SIZES)
@pytest.mark.parametrize("res", [False, True])
def test_rms_norm_fp8(cuda_device, dtype, rows, d, res):
    x = _randn((rows, d), dtype, cuda_device, 4)
    r = _randn((rows, d), dtype, cuda_device, 5) if res else None
    w = _randn((d,), dtype, cuda_device, 6)
    y8, s, h = cawq.rms_norm_fp8(x, w, 1e-6, residual=r)
    assert y8.dtype == torch.float8_e4m3fn and y8.shape == x.shape and s.shape == (rows,)
    hr, yr = norm_ref(x, w, 1e-6, r)
    rel = norm_rel(d) + 8 * F32
    sr = yr.abs().amax(dim=1) / 448
    assert_within(s, sr, sr * rel + 1e-38, "scale")
    # e4m3 has 4 significant bits: half a step is 2^-4 of the value, 2^-10 below the normal range
    tol = torch.maximum(yr.abs() * 2.0 ** -4, sr[:, None] * 2.0 ** -10)
    assert_within(y8.double() * s.double()[:, None], yr, tol * (1 + 2.0 ** -9) + yr.abs() * rel, "y8")
    if res:
        assert_within(h, hr, hr.abs() * (ROUND[dtype] + 2 * F32) + FLOOR[dtype], "h")


def test_rms_norm_rows_of_zeros_and_strides_and_in_place(cuda_device):
    d = 520
    buf = _randn((6, 1024), F16, cuda_device, 7)
    x, w = buf[:, 8:8 + d], _randn((d,), F16, cuda_device, 8)
    odd = buf[:, 1:1 + d]  # off every vector's alignment
    for v in (x, odd):
        y, _ = cawq.rms_norm(v, w, 1e-6)
        _check_norm(v, w, 1e-6, None, y, None)
    z = torch.zeros((3, d), dtype=BF16, device=cuda_device)
    y8, s, _ = cawq.rms_norm_fp8(z, w.to(BF16), 1e-6)
    assert not y8.float().any() and not s.any()
    y, _ = cawq.rms_norm(z, w.to(BF16), 0.0)  # 0 / 0
    assert y.isnan().all()
    # residual stream and x updated in place
    a, r = _randn((9, d), BF16, cuda_device, 9), _randn((9, d), BF16, cuda_device, 10)
    wb = w.to(BF16)
    a0, r0 = a.clone(), r.clone()
    y, h = cawq.rms_norm(a, wb, 1e-6, residual=r, out=a, residual_out=r)
    assert y is a and h is r
    _check_norm(a0, wb, 1e-6, r0, y, h)
    # leading dimensions, no rows
    y, h = cawq.rms_norm(a0.view(3, 3, d), wb, 1e-6, residual=r0.view(3, 3, d))
    assert y.shape == (3, 3, d) and torch.equal(y.view(9, d), a) and torch.equal(h.view(9, d), r)
    y, _ = cawq.rms_norm(a0[:0], wb)
    assert y.shape == (0, d)


def test_rms_norm_large_values(cuda_device):
    # squares that overflow 16 bits, and a row holding an infinity
    x = torch.full((2, 256), 60000.0, dtype=F16, device=cuda_device)
    x[1, 3] = float("inf")
    w = torch.ones(256, dtype=F16, device=cuda_device)
    y, _ = cawq.rms_norm(x, w, 1e-6)
    assert torch.equal(y[0], torch.ones_like(y[0]))
    assert y[1, 3].isnan() and not y[1, 4:].any()


# -------------------------------------------------------------- rotary append
def _rope_case(dev, dtype, seqs, hq, hkv, d, page, layout, seed=0, decode=False):
    c = Cache(seqs, hkv, d, page, dtype, dev, seed=seed, layout=layout)
    tokens = c.starts[-1]
    wide = _randn((tokens, (hq + 2 * hkv) * d + 8), dtype, dev, seed + 1, 2.0)
    q = wide[:, :hq * d].unflatten(1, (hq, d))
    k = wide[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
    v = wide[:, (hq + hkv) * d:(hq + 2 * hkv) * d].unflatten(1, (hkv, d))
    rope = cawq.rope_table(max(t for _, t in seqs) + 1, d, 10000.0, dev)
    return c, q, k, v, rope


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,d,page,layout", [(4, 4, 128, 16, "head"), (7, 1, 64, 24, "token"),
                                                  (28, 4, 128, 64, "pair"), (64, 8, 128, 8, "head")])
@pytest.mark.parametrize("seqs", [[(1, 1), (1, 77), (1, 0), (1, 300)],
                                  [(5, 5), (0, 40), (1, 129), (33, 90), (3, 0), (140, 300)]])
def test_rope_append(cuda_device, dtype, hq, hkv, d, page, layout, seqs):
    c, q, k, v, rope = _rope_case(cuda_device, dtype, seqs, hq, hkv, d, page, layout, seed=page)
    decode = all(n == 1 for n, _ in seqs)
    kc, vc = c.k.clone(), c.v.clone()
    out = cawq.rope_append(q, k, v, rope, c.k, c.v, c.table, c.lens,
                           q_start=None if decode else c.q_start)
    half = d // 2
    u = ROUND[dtype]

    def turn(x, pos):
        cs, sn = rope.double()[pos, None, :half], rope.double()[pos, None, half:]
        a, b = x.double()[..., :half], x.double()[..., half:]
        r = torch.cat([a * cs - b * sn, b * cs + a * sn], -1)
        size = torch.cat([(a * cs).abs() + (b * sn).abs(), (b * cs).abs() + (a * sn).abs()], -1)
        return r, r.abs() * u + 3 * F32 * size + FLOOR[dtype]

    for i, (n, total) in enumerate(seqs):
        rows = slice(c.starts[i], c.starts[i] + n)
        if total == 0:
            assert not out[rows].any()
            continue
        pos = torch.arange(total - n, total, device=cuda_device)
        r, tol = turn(q[rows], pos)
        assert_within(out[rows], r, tol, "q")
        pg = c.table[i].long()[pos // page]
        r, tol = turn(k[rows], pos)
        assert_within(c.k[pg, :, pos % page], r, tol, "k")
        assert torch.equal(c.v[pg, :, pos % page], v[rows])
        kc[pg, :, pos % page] = c.k[pg, :, pos % page]
        vc[pg, :, pos % page] = c.v[pg, :, pos % page]
    # nothing else was written
    assert torch.equal(kc.nan_to_num(nan=7.0), c.k.nan_to_num(nan=7.0))
    assert torch.equal(vc.nan_to_num(nan=7.0), c.v.nan_to_num(nan=7.0))
    # q in place gives the same
    want = out.clone()
    got = cawq.rope_append(q, k, v, rope, c.k, c.v, c.table, c.lens,
                           q_start=None if decode else c.q_start, out=q)
    assert got is q and torch.equal(got, want)


# ------------------------------------------------------------------ attention
def _attend(dev, dtype, seqs, hq, hkv, d, page, window=0, sinks=0, layout="head", seed=0,
            decode=False, evict=False, scale=None, qscale=1.5, check=True):
    c = Cache(seqs, hkv, d, page, dtype, dev, seed=seed, layout=layout,
              evict_window=window if evict else None, sinks=sinks)
    q = _randn((c.starts[-1], hq, d), dtype, dev, seed + 1, qscale)
    if decode:
        out = cawq.attention_decode(q, c.k, c.v, c.table, c.lens, window=window, sinks=sinks,
                                    scale=scale)
    else:
        out = cawq.attention_prefill(q, c.k, c.v, c.table, c.lens, c.q_start, window=window,
                                     sinks=sinks, scale=scale)
    if check:
        ref, tol = attention_ref(q, c, window, sinks, scale)
        assert_within(out, ref, tol)
    return c, q, out


HEADS = [(1, 1, 128), (4, 4, 128), (28, 4, 128), (64, 8, 128), (14, 2, 64), (16, 1, 128),
         (40, 2, 64), (96, 1, 128)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("page", [8, 16, 24, 256])
def test_decode_lengths(cuda_device, dtype, hq, hkv, d, page):
    lens = [1, 0, 2, 15, 16, 17, 63, 64, 65, 127, 129, 500, 1023, 3]
    _attend(cuda_device, dtype, [(1, t) for t in lens], hq, hkv, d, page, decode=True,
            seed=hq + page)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,d,page,length", [(32, 32, 128, 16, 1000), (8, 1, 128, 64, 20011),
                                                  (28, 4, 128, 16, 4096), (14, 2, 64, 128, 9999),
                                                  (2, 1, 128, 32, 1)])
def test_decode_one_sequence(cuda_device, dtype, hq, hkv, d, page, length):
    _attend(cuda_device, dtype, [(1, length)], hq, hkv, d, page, decode=True, seed=length)


@pytest.mark.parametrize("batch", [1, 7, 200])
def test_decode_batches(cuda_device, batch):
    lens = [(37 * i * i + 5 * i) % 700 for i in range(batch)]
    _attend(cuda_device, BF16, [(1, t) for t in lens], 8, 2, 128, 16, decode=True, seed=batch)


WINDOWS = [(1, 0), (16, 4), (100, 0), (128, 1), (300, 130), (5000, 4), (7, 600)]


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("evict", [False, True])
def test_decode_window_and_sinks(cuda_device, window, sinks, evict):
    lens = [1, 5, 0, 64, 101, 128, 129, 333, 600, 1500]
    _attend(cuda_device, F16, [(1, t) for t in lens], 7, 1, 128, 16, window, sinks, decode=True,
            evict=evict, seed=window)
    _attend(cuda_device, BF16, [(1, t) for t in lens], 8, 8, 64, 24, window, sinks, decode=True,
            evict=evict, seed=window, layout="token")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("page", [8, 16, 24, 256])
def test_prefill_lengths(cuda_device, dtype, hq, hkv, d, page):
    seqs = [(1, 1), (3, 0), (2, 2), (0, 9), (17, 40), (64, 64), (65, 300), (1, 700), (130, 131),
            (257, 400)]
    _attend(cuda_device, dtype, seqs, hq, hkv, d, page, seed=hq + page)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,d,page,new,total", [
    (4, 2, 128, 16, 1100, 1100), (7, 1, 128, 64, 513, 2049), (2, 2, 64, 16, 1500, 1501),
    (1, 1, 128, 16, 127, 128), (8, 1, 128, 128, 2000, 4000), (12, 12, 128, 16, 5, 3000),
    (4, 1, 64, 32, 16, 5000)])
def test_prefill_one_sequence(cuda_device, dtype, hq, hkv, d, page, new, total):
    _attend(cuda_device, dtype, [(new, total)], hq, hkv, d, page, seed=new)


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("evict", [False, True])
def test_prefill_window_and_sinks(cuda_device, window, sinks, evict):
    seqs = [(1, 5), (40, 40), (3, 700), (200, 1500), (300, 300), (2, 0), (129, 900)]
    _attend(cuda_device, F16, seqs, 7, 1, 128, 16, window, sinks, evict=evict, seed=window)
    _attend(cuda_device, BF16, seqs, 4, 2, 64, 24, window, sinks, evict=evict, seed=window,
            layout="pair")


def test_prefill_more_new_tokens_than_the_cache_holds(cuda_device):
    # positions below zero see nothing and give zeros
    seqs = [(10, 4), (300, 100), (5, 5)]
    c = Cache(seqs, 2, 128, 16, F16, cuda_device)
    q = _randn((c.starts[-1], 4, 128), F16, cuda_device, 3)
    out = cawq.attention_prefill(q, c.k, c.v, c.table, c.lens, c.q_start)
    ref, tol = attention_ref(q, c)
    assert_within(out, ref, tol)
    assert not out[:6].any() and not out[10:210].any()


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("layout", ["head", "token", "pair"])
def test_attention_layouts_views_and_scale(cuda_device, decode, layout):
    seqs = [(1, 300), (1, 20)] if decode else [(70, 300), (33, 40)]
    _attend(cuda_device, F16, seqs, 14, 2, 128, 16, layout=layout, decode=decode, scale=0.3)
    _attend(cuda_device, BF16, seqs, 14, 2, 128, 16, layout=layout, decode=decode, scale=0.0)
    c = Cache(seqs, 2, 128, 16, F16, cuda_device, layout=layout)
    t = c.starts[-1]
    buf, obuf = _randn((t, 3000), F16, cuda_device, 5), torch.zeros((t, 2048), dtype=F16, device=cuda_device)
    q, out = buf[:, 16:16 + 512].unflatten(1, (4, 128)), obuf[:, 8:8 + 512].unflatten(1, (4, 128))
    table = torch.full((2, c.table.shape[1] + 3), -1, dtype=torch.int32, device=cuda_device)
    table[:, :c.table.shape[1]] = c.table
    args = (q, c.k, c.v, table[:, :c.table.shape[1]], c.lens)
    got = cawq.attention_decode(*args, out=out) if decode else \
        cawq.attention_prefill(*args, c.q_start, out=out)
    assert got is out
    ref, tol = attention_ref(q, c)
    assert_within(out, ref, tol)
    assert not obuf[:, :8].any() and not obuf[:, 8 + 512:].any()


@pytest.mark.parametrize("decode", [True, False])
def test_attention_large_scores_and_growing_maximum(cuda_device, decode):
    # scores that grow along the cache by hundreds, and a first key above all
    # others: the running maximum moves at every step, or never again
    for sign in (1.0, -1.0):
        seqs = [(1, 700)] if decode else [(300, 700)]
        c = Cache(seqs, 1, 128, 16, BF16, cuda_device)
        ramp = torch.linspace(-1, 1, 700, device=cuda_device)[:, None, None] * sign
        kd = (ramp.expand(700, 1, 128) * 4 + 0.01 * c.kd[0].float()).to(BF16)
        pos = torch.arange(700, device=cuda_device)
        c.k[c.table[0].long()[pos // 16], :, pos % 16] = kd
        c.kd[0] = kd
        q = _randn((c.starts[-1], 8, 128), BF16, cuda_device, 2, 0.5).abs() + 1
        args = (q, c.k, c.v, c.table, c.lens)
        out = cawq.attention_decode(*args) if decode else cawq.attention_prefill(*args, c.q_start)
        ref, tol = attention_ref(q, c)
        assert_within(out, ref, tol)


@pytest.mark.parametrize("decode", [True, False])
def test_attention_same_bits_again_on_another_stream_and_in_a_graph(cuda_device, decode):
    seqs = [(1, 5000), (1, 33), (1, 900)] if decode else [(300, 1000), (1, 3000), (40, 41)]
    c = Cache(seqs, 4, 128, 16, BF16, cuda_device)
    q = _randn((c.starts[-1], 28, 128), BF16, cuda_device, 2)
    fn = (lambda: cawq.attention_decode(q, c.k, c.v, c.table, c.lens)) if decode else \
        (lambda: cawq.attention_prefill(q, c.k, c.v, c.table, c.lens, c.q_start))
    want = fn()
    assert torch.equal(fn(), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [fn() for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(g, want) for g in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g = fn()
    q.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(g, fn()) and not torch.equal(g, want)
    del graph


@pytest.mark.parametrize("decode", [True, False])
def test_attention_cache_past_32_bits(cuda_device, decode):
    # pages 160 MB apart: the used ones lie past 2^32 bytes
    seqs = [(1, 100)] if decode else [(40, 100)]
    src = Cache(seqs, 1, 128, 16, F16, cuda_device, spare=0, table_extra=0)
    pages, step = 64, 80 * 1024 * 1024
    pool = torch.empty(pages * step, dtype=F16, device=cuda_device)
    k = pool.as_strided((pages, 1, 16, 128), (step, 2048, 128, 1))
    v = pool.as_strided((pages, 1, 16, 128), (step, 2048, 128, 1), 4096)
    n = src.table.shape[1]
    table = torch.arange(pages - n, pages, dtype=torch.int32, device=cuda_device)[None]
    k[table[0].long()], v[table[0].long()] = src.k[src.table[0].long()], src.v[src.table[0].long()]
    q = _randn((src.starts[-1], 8, 128), F16, cuda_device, 2)
    args = (q, k, v, table, src.lens)
    out = cawq.attention_decode(*args) if decode else cawq.attention_prefill(*args, src.q_start)
    ref, tol = attention_ref(q, src)
    assert_within(out, ref, tol)


def test_bad_pages_and_positions_are_skipped_and_reported(cuda_device):
    seqs = [(1, 100), (1, 60)]
    c = Cache(seqs, 2, 128, 16, F16, cuda_device, table_extra=0)
    q = _randn((2, 4, 128), F16, cuda_device, 2)
    bad = c.table.clone()
    bad[0, 2] = c.pages          # past the cache: positions 32 .. 47 are not seen
    out = cawq.attention_decode(q, c.k, c.v, bad, c.lens)
    assert cawq.device_error() == 4
    keep = torch.ones(100, dtype=torch.bool, device=cuda_device)
    keep[32:48] = False
    c.kd[0], c.vd[0], c.seqs = c.kd[0][keep], c.vd[0][keep], [(1, 84), (1, 60)]
    ref, tol = attention_ref(q, c)
    assert_within(out, ref, tol)
    out2 = cawq.attention_prefill(q, c.k, c.v, bad, c.lens, c.q_start)
    assert cawq.device_error() == 4
    assert_within(out2, ref, tol)
    # a length past the table is cut to it
    lens = torch.tensor([100, 5000], dtype=torch.int32, device=cuda_device)
    out = cawq.attention_decode(q, c.k, c.v, c.table, lens)
    assert cawq.device_error() == 4 and out.shape == q.shape
    # rope: a position past the table of angles, and a bad page
    rope = cawq.rope_table(64, 128, device=cuda_device)
    kn, vn = _randn((2, 2, 128), F16, cuda_device, 3), _randn((2, 2, 128), F16, cuda_device, 4)
    before = c.k.clone()
    o = cawq.rope_append(q, kn, vn, rope, c.k, c.v, c.table, c.lens)
    assert cawq.device_error() == 4
    assert not o[0].any() and o[1].any()
    pg = int(c.table[1, 59 // 16])
    before[pg, :, 59 % 16] = c.k[pg, :, 59 % 16]
    assert torch.equal(before.nan_to_num(nan=7.0), c.k.nan_to_num(nan=7.0))


def test_empty_calls(cuda_device):
    c = Cache([(1, 5)], 2, 128, 16, F16, cuda_device)
    q = torch.empty((0, 4, 128), dtype=F16, device=cuda_device)
    none = torch.empty((0,), dtype=torch.int32, device=cuda_device)
    table = torch.empty((0, 3), dtype=torch.int32, device=cuda_device)
    assert cawq.attention_decode(q, c.k, c.v, table, none).shape == (0, 4, 128)
    zero = torch.zeros(2, dtype=torch.int32, device=cuda_device)
    assert cawq.attention_prefill(q, c.k, c.v, c.table, c.lens, zero).shape == (0, 4, 128)


@pytest.mark.parametrize("compiled", [True, False])
def test_both_host_paths(cuda_device, compiled, monkeypatch):
    # the compiled host path, and the one in Python where it was not built
    from cube_awq_b200 import layer_ops
    if not compiled:
        monkeypatch.setattr(layer_ops, "_torch_ext", lambda: None)
    x, w = _randn((5, 640), BF16, cuda_device, 1), _randn((640,), BF16, cuda_device, 2)
    y, h = cawq.rms_norm(x, w, 1e-6, residual=x)
    _check_norm(x, w, 1e-6, x, y, h)
    y8, s, h8 = cawq.rms_norm_fp8(x, w, 1e-6, residual=x)
    assert torch.equal(h, h8) and y8.dtype == torch.float8_e4m3fn and s.shape == (5,)
    _attend(cuda_device, BF16, [(1, 300), (1, 2)], 8, 2, 128, 16, 50, 3, decode=True)
    _attend(cuda_device, BF16, [(30, 300), (2, 2)], 8, 2, 128, 16, 50, 3)
    c, q, k, v, rope = _rope_case(cuda_device, F16, [(3, 40), (1, 1)], 4, 2, 64, 16, "pair")
    out = cawq.rope_append(q, k, v, rope, c.k, c.v, c.table, c.lens, q_start=c.q_start)
    assert out.shape == q.shape and torch.equal(c.v[int(c.table[1, 0]), :, 0], v[3])
    with pytest.raises(CubeAwqError):
        cawq.attention_decode(q[:2], c.k, c.v, c.table, c.lens, window=-1)


def test_prefill_many_sequences(cuda_device):
    # more sequences than the kernels have threads; runs of empty ones
    seqs = [((i * 7) % 4, (i * 7) % 4 + (i % 5) * 30) if i % 3 else (0, 0) for i in range(1500)]
    _attend(cuda_device, BF16, seqs, 4, 1, 64, 16, seed=3)


def test_decode_many_sequences(cuda_device):
    _attend(cuda_device, F16, [(1, (i * 37) % 90) for i in range(1000)], 4, 1, 64, 16, seed=4,
            decode=True)


@pytest.mark.parametrize("window,sinks", [(0, 0), (2000, 7)])
def test_prefill_batches_of_long_and_short_and_prompts(cuda_device, window, sinks):
    # single tokens and short runs behind long caches (split) beside prompts (tiles)
    seqs = [(1, 9000), (300, 300), (3, 4001), (16, 7000), (1, 1), (0, 50), (1, 1024), (1, 1023),
            (100, 5000), (2, 0)]
    _attend(cuda_device, BF16, seqs, 8, 1, 128, 16, window, sinks, seed=5)
    _attend(cuda_device, F16, seqs, 14, 2, 64, 24, window, sinks, seed=6, layout="token",
            evict=bool(window))


@pytest.mark.parametrize("long", [900, 6000])
@pytest.mark.parametrize("batch", [5, 32, 33, 70])
@pytest.mark.parametrize("prompt", [0, 33, 600])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1500, 4)])
def test_prefill_of_many_short_runs_and_a_long_one(cuda_device, long, batch, prompt, window, sinks):
    # what one sequence has decides which kernel takes the others' rows, empty
    # sequences and 128 rows (of a kv head) among them, 132 and a prompt left out
    seqs = [(0, 30) if i % 4 == 3 else (1 + i % 3, 1 + i % 3 + (i * i * 29) % 300) for i in range(batch)]
    seqs[1], seqs[2], seqs[batch - 1] = (32, 700), (33, 700), (3, long)
    if prompt:
        seqs[4] = (prompt, prompt + 11)
    _attend(cuda_device, BF16, seqs, 8, 2, 64, 16, window=window, sinks=sinks, seed=batch + long)


@pytest.mark.parametrize("new,total", [(1, 3000), (5, 2500), (18, 6000), (19, 800), (40, 9000)])
def test_prefill_of_one_sequence_with_few_rows(cuda_device, new, total):
    _attend(cuda_device, F16, [(new, total)], 7, 1, 128, 16, seed=new)


@pytest.mark.parametrize("decode", [True, False])
def test_attention_pages_between_whole_heads(cuda_device, decode):
    # a page stride that is no whole number of head strides
    seqs = [(1, 300), (1, 20)] if decode else [(70, 300), (33, 40)]
    c = Cache(seqs, 3, 128, 16, F16, cuda_device)
    sh, sp = 16 * 128, 3 * 16 * 128 + 8
    pool = torch.full((2, c.pages * sp), float("nan"), dtype=F16, device=cuda_device)
    k, v = (pool[i].as_strided((c.pages, 3, 16, 128), (sp, sh, 128, 1), i * c.pages * sp)
            for i in range(2))
    k.copy_(c.k)
    v.copy_(c.v)
    q = _randn((c.starts[-1], 12, 128), F16, cuda_device, 2)
    args = (q, k, v, c.table, c.lens)
    out = cawq.attention_decode(*args) if decode else cawq.attention_prefill(*args, c.q_start)
    ref, tol = attention_ref(q, c)
    assert_within(out, ref, tol)


@pytest.mark.parametrize("batch,hq,hkv,length", [(1, 1, 1, 1000), (1, 8, 8, 65), (3, 48, 3, 300),
                                                 (20, 8, 2, 500), (40, 32, 8, 100), (1, 6, 2, 4096),
                                                 (2, 64, 64, 129)])
@pytest.mark.parametrize("d", [64, 128])
def test_decode_few_row_tiles(cuda_device, batch, hq, hkv, length, d):
    # calls small enough for a cluster per row tile, of every size, with row
    # tiles that have fewer keys than the cluster has CTAs
    lens = [max(0, length - 17 * i * i) for i in range(batch)]
    _attend(cuda_device, BF16, [(1, t) for t in lens], hq, hkv, d, 16, decode=True, seed=length)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("batch,hq,hkv,d", [(400, 8, 8, 64), (300, 64, 4, 128), (70, 5, 5, 128),
                                            (257, 9, 3, 64), (150, 24, 2, 128)])
@pytest.mark.parametrize("page,longest", [(16, 256), (8, 256), (24, 250), (16, 17), (64, 64), (16, 257)])
def test_decode_many_short_sequences(cuda_device, dtype, batch, hq, hkv, d, page, longest):
    # tables short enough for a warp per row tile, more of them than warps; and
    # one page past that
    lens = [longest if i == 7 else (i * i * 13 + 5 * i) % (longest + 1) for i in range(batch)]
    _attend(cuda_device, dtype, [(1, t) for t in lens], hq, hkv, d, page, decode=True, seed=batch)


@pytest.mark.parametrize("batch,hq,hkv", [(296, 3, 1), (297, 16, 1), (64, 32, 8), (37, 56, 8), (148, 20, 4)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("longest", [128, 129, 190, 512, 513])
def test_decode_one_or_two_row_tiles_for_each_cta(cuda_device, batch, hq, hkv, d, longest):
    lens = [longest if i == 3 else (i * i * 7 + 11 * i) % (longest + 1) for i in range(batch)]
    _attend(cuda_device, BF16, [(1, t) for t in lens], hq, hkv, d, 16, decode=True, seed=longest)


@pytest.mark.parametrize("layout", ["head", "token", "pair"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (17, 0), (200, 56), (250, 7)])
def test_decode_many_sequences_in_short_windows(cuda_device, layout, window, sinks):
    lens = [(i * 131) % 1500 for i in range(160)]
    _attend(cuda_device, BF16, [(1, t) for t in lens], 16, 8, 128, 16, decode=True, evict=True,
            window=window, sinks=sinks, layout=layout)


def test_attention_scales(cuda_device):
    seqs = [(130, 200), (3, 2000)]
    for scale in (-0.2, 1e-3, 2.0):
        _attend(cuda_device, F16, seqs, 8, 2, 128, 16, scale=scale, qscale=0.5)
        _attend(cuda_device, F16, [(1, 700)], 8, 2, 128, 16, scale=scale, qscale=0.5, decode=True)
