"""The layer operators at the edges of their contracts: caches that end inside
a copied box, rows of no sequence, lengths past the table, values that are not
finite or hardly there."""

import pytest
import torch

import cube_awq_b200 as cawq
from layer_ref import Cache, assert_within, attention_ref

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _no_device_error(cuda_device):
    cawq.device_error()
    yield
    assert cawq.device_error() == 0


def _randn(shape, dtype, dev, seed, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=dev) * scale).to(dtype)


def _i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("d", [64, 128])
def test_prefill_of_caches_that_end_inside_a_box(cuda_device, page, d):
    # the values of the last box are written by a warp's threads, with zeros
    # past the end, where the cache holds NaN; every remainder, again and again
    seqs = [(70, 128 * (1 + r % 3) + r) for r in range(1, page if page < 128 else 100, 2)]
    c = Cache(seqs, 2, d, page, BF16, cuda_device, seed=page + d)
    q = _randn((c.starts[-1], 8, d), BF16, cuda_device, 1)
    call = lambda: cawq.attention_prefill(q, c.k, c.v, c.table, c.lens, c.q_start)  # noqa: E731
    out = call()
    ref, tol = attention_ref(q, c)
    assert_within(out, ref, tol)
    for _ in range(30):
        assert torch.equal(call(), out)


def _rope_args(dev, tokens, hq=4, hkv=2, d=64, seed=0):
    q, k, v = (_randn((tokens, h, d), F16, dev, seed + i) for i, h in enumerate((hq, hkv, hkv)))
    return q, k, v, cawq.rope_table(200, d, device=dev)


def test_rows_outside_all_sequences_are_left_out(cuda_device):
    # a part of a batch on the tensors of the whole: rows before q_start[0] and
    # from q_start[batch] on are no sequence's
    seqs = [(3, 100), (2, 9)]
    c = Cache(seqs, 2, 64, 16, F16, cuda_device)
    q_start = c.q_start + 5
    q, k, v, rope = _rope_args(cuda_device, 13)
    out = cawq.rope_append(q, k, v, rope, c.k, c.v, c.table, c.lens, q_start=q_start)
    want = Cache(seqs, 2, 64, 16, F16, cuda_device)
    mine = slice(5, 10)
    got = cawq.rope_append(q[mine], k[mine], v[mine], rope, want.k, want.v, want.table, want.lens,
                           q_start=want.q_start)
    assert torch.equal(out[mine], got) and not out[:5].any() and not out[10:].any()
    for a, b in ((c.k, want.k), (c.v, want.v)):
        assert torch.equal(a.nan_to_num(nan=7.0), b.nan_to_num(nan=7.0))
    keep = torch.full_like(q, 3.0)
    att = cawq.attention_prefill(q, c.k, c.v, c.table, c.lens, q_start, out=keep)
    assert (att[:5] == 3).all() and (att[10:] == 3).all()
    assert torch.equal(att[mine], cawq.attention_prefill(q[mine], c.k, c.v, c.table, c.lens, c.q_start))


def test_row_starts_that_do_not_ascend_stay_inside_the_cache(cuda_device):
    # such starts break a precondition; what they name is then undefined, but
    # no token goes past its sequence's length. The table's rows lie in a wider
    # one, whose other entries name a page that nothing may touch.
    g = torch.Generator().manual_seed(0)
    batch, tokens, page = 6, 24, 8
    starts = [[0, 9, 1, 2, 8, 3, 24]] + [torch.randint(0, tokens + 1, (batch + 1,), generator=g).tolist()
                                         for _ in range(60)]
    q, k, v, rope = _rope_args(cuda_device, tokens)
    for s in starts:
        kc = torch.zeros((2 * batch + 1, 2, page, 64), dtype=F16, device=cuda_device)
        vc = kc.clone()
        wide = torch.full((batch, 8), 2 * batch, dtype=torch.int32, device=cuda_device)
        wide[:, :2] = torch.arange(2 * batch, device=cuda_device).view(batch, 2)
        lens = _i32([13, 16, 1, 5, 0, 9], cuda_device)
        out = cawq.rope_append(q, k, v, rope, kc, vc, wide[:, :2], lens, q_start=_i32(s, cuda_device))
        assert out.shape == q.shape and not kc[-1].any() and not vc[-1].any()
        for b, n in enumerate(lens.tolist()):  # nor past a length inside the table
            flat = kc[2 * b:2 * b + 2].transpose(1, 2).reshape(2 * page, -1)
            assert not flat[n:].any()


@pytest.mark.parametrize("window,sinks", [(2 ** 31 - 1, 0), (2 ** 31 - 1, 4), (2 ** 40, 2 ** 40),
                                          (2 ** 31 - 8, 2 ** 31 - 1)])
@pytest.mark.parametrize("seqs", [[(10, 4), (300, 100), (5, 5)], [(40, 4), (1, 4000), (6, 1000)]])
def test_windows_as_wide_as_can_be(cuda_device, window, sinks, seqs):
    # as good as none, also for new tokens whose positions lie below zero
    c = Cache(seqs, 2, 128, 16, F16, cuda_device)
    q = _randn((c.starts[-1], 4, 128), F16, cuda_device, 3)
    out = cawq.attention_prefill(q, c.k, c.v, c.table, c.lens, c.q_start, window=window, sinks=sinks)
    ref, tol = attention_ref(q, c)
    assert_within(out, ref, tol)
    one = cawq.attention_decode(q[:len(seqs)], c.k, c.v, c.table, c.lens, window=window, sinks=sinks)
    assert torch.equal(one, cawq.attention_decode(q[:len(seqs)], c.k, c.v, c.table, c.lens))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("seqs", [[(300, 300), (70, 500)], [(2, 3000)], [(1, 5000), (300, 310), (0, 4)],
                                  [(1, 700), (1, 60), (1, 3000)]])
def test_queries_that_are_not_finite_give_nan(cuda_device, dtype, d, seqs):
    # whichever kernel takes the row, and no other row
    c = Cache(seqs, 2, d, 16, dtype, cuda_device, seed=d)
    q = _randn((c.starts[-1], 8, d), dtype, cuda_device, 1)
    calls = [lambda x: cawq.attention_prefill(x, c.k, c.v, c.table, c.lens, c.q_start)]
    if all(n == 1 for n, _ in seqs):
        calls.append(lambda x: cawq.attention_decode(x, c.k, c.v, c.table, c.lens))
    nan, inf = float("nan"), float("inf")
    tokens = c.starts[-1]
    hit = torch.zeros((tokens, 8), dtype=torch.bool, device=cuda_device)
    bad = q.clone()
    # (token, head, value): past the first tokens, so that the infinite scores
    # of a row have both signs
    for t, h, x in ((tokens - 1, 0, nan), (tokens - 1, 7, inf), (0 if seqs[0][1] > 600 else 90, 3, -inf),
                    (tokens // 2, 5, nan)):
        t = min(t, tokens - 1)
        bad[t, h, (7 * h + 5) % d] = x
        hit[t, h] = True
    for call in calls:
        want, got = call(q), call(bad)
        assert got[hit].isnan().all()
        assert torch.equal(got[~hit], want[~hit])


def test_rope_past_the_table_is_skipped(cuda_device):
    # a table of 4 pages of 16: position 64 and later have no slot
    q, k, v, rope = _rope_args(cuda_device, 3)
    kc = _randn((13, 2, 16, 64), F16, cuda_device, 7)
    vc = _randn((13, 2, 16, 64), F16, cuda_device, 8)
    table = torch.arange(12, dtype=torch.int32, device=cuda_device).view(3, 4)
    kk, vv = kc.clone(), vc.clone()
    out = cawq.rope_append(q, k, v, rope, kc, vc, table, _i32([65, 64, 100], cuda_device))
    assert cawq.device_error() == 4
    for a, b in ((kc, kk), (vc, vv)):  # the second one's slot alone is written
        b[7, :, 15] = a[7, :, 15]
        assert torch.equal(a, b)
    assert torch.equal(vc[7, :, 15], v[1])
    # q turns by its true position
    far = torch.zeros((3, 13), dtype=torch.int32, device=cuda_device)
    far[:, :4] = 12
    want = cawq.rope_append(q, k, v, rope, kk, vv, far, _i32([65, 64, 100], cuda_device))
    assert torch.equal(out, want)
    # of a run of new tokens those that have a slot are stored in it
    kc2, vc2 = kk.clone(), vv.clone()
    cawq.rope_append(q, k, v, rope, kc2, vc2, table[:1], _i32([66], cuda_device), q_start=_i32([0, 3], cuda_device))
    assert cawq.device_error() == 4
    assert torch.equal(vc2[3, :, 15], v[0])
    kc2[3, :, 15], vc2[3, :, 15] = kk[3, :, 15], vv[3, :, 15]
    assert torch.equal(kc2, kk) and torch.equal(vc2, vv)


class _Cut(Cache):
    """A cache whose tables hold `slots` positions, given to calls whose
    sequences are longer: their other keys and values do not exist."""

    def __init__(self, seqs, slots, hkv, d, page, dtype, device, seed=0):
        super().__init__([(n, min(t, slots)) for n, t in seqs], hkv, d, page, dtype, device, seed=seed,
                         table_extra=0)
        assert self.table.shape[1] * page == slots
        self.true = [t for _, t in seqs]
        self.lens = _i32(self.true, device)


def _cut_ref(q, c, window, sinks):
    """attention_ref with the queries at their true positions, keys up to the table's end."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for i, ((n, have), true) in enumerate(zip(c.seqs, c.true)):
        rows = slice(c.starts[i], c.starts[i] + n)
        for t in range(n):
            pos = true - n + t
            seen = [j for j in range(min(pos + 1, have)) if not window or j > pos - window or j < sinks]
            one = Cache.__new__(Cache)
            one.seqs, one.starts, one.k = [(1, len(seen))], [0, 1], c.k
            one.kd, one.vd = [c.kd[i][seen]], [c.vd[i][seen]]
            r = rows.start + t
            out[r:r + 1], tol[r:r + 1] = attention_ref(q[r:r + 1], one)
    return out, tol


@pytest.mark.parametrize("page,slots", [(16, 336), (8, 72), (64, 640)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 0), (40, 7), (700, 100)])
def test_attention_past_the_table(cuda_device, page, slots, d, window, sinks):
    # positions are the true ones, keys end with the table
    seqs = [(3, slots + 1), (20, slots + 6), (40, slots + 40), (2, slots + 1000), (70, slots), (5, 9),
            (1, 2 ** 31 - 1), (33, 2 ** 30)]
    c = _Cut(seqs, slots, 2, d, page, BF16, cuda_device, seed=slots)
    q = _randn((c.starts[-1], 8, d), BF16, cuda_device, 1)
    out = cawq.attention_prefill(q, c.k, c.v, c.table, c.lens, c.q_start, window=window, sinks=sinks)
    assert cawq.device_error() == 4
    ref, tol = _cut_ref(q, c, window, sinks)
    assert_within(out, ref, tol)
    for part in ([1], [2], [3], [7]):  # alone, so that either kernel takes them
        i = part[0]
        rows = slice(c.starts[i], c.starts[i + 1])
        out = cawq.attention_prefill(q[rows], c.k, c.v, c.table[i:i + 1], c.lens[i:i + 1],
                                     _i32([0, seqs[i][0]], cuda_device), window=window, sinks=sinks)
        assert_within(out, ref[rows], tol[rows])
    assert cawq.device_error() == 4
    one = _Cut([(1, t) for _, t in seqs], slots, 2, d, page, BF16, cuda_device, seed=slots + 1)
    out = cawq.attention_decode(q[:len(seqs)], one.k, one.v, one.table, one.lens, window=window, sinks=sinks)
    assert cawq.device_error() == 4
    ref, tol = _cut_ref(q[:len(seqs)], one, window, sinks)
    assert_within(out, ref, tol)


def test_many_rows_past_the_table(cuda_device):
    # a long run whose first tokens have slots and whose last ones have none
    c = _Cut([(500, 800), (300, 700)], 640, 1, 128, 16, F16, cuda_device)
    q = _randn((c.starts[-1], 4, 128), F16, cuda_device, 1)
    for window, sinks in ((0, 0), (100, 5)):
        out = cawq.attention_prefill(q, c.k, c.v, c.table, c.lens, c.q_start, window=window, sinks=sinks)
        assert cawq.device_error() == 4
        ref, tol = _cut_ref(q, c, window, sinks)
        assert_within(out, ref, tol)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 520, 1001, 8192, 17001])
@pytest.mark.parametrize("size", [1e-40, 1e-38, 1e-36, 1.3e-36, 1.4e-36])
def test_rms_norm_fp8_of_rows_that_are_hardly_there(cuda_device, dtype, d, size):
    # 448 / max |y| passes the largest fp32 below 1.3e-36. eps is large, so that
    # y = x * weight to fp32's precision, and the weights put |y| near `size`.
    x = _randn((5, d), dtype, cuda_device, 1)
    x[:, ::7] = 0
    x[4] = 0
    w = (torch.rand(d, generator=torch.Generator(device=cuda_device).manual_seed(2),
                    device=cuda_device) + 0.5).mul_(size).to(dtype)
    y8, s, _ = cawq.rms_norm_fp8(x, w, 1.0)
    h = x.double()
    y = h / (h.square().mean(dim=1, keepdim=True) + 1.0).sqrt() * w.double()
    scale = y.abs().amax(dim=1) / 448
    tiny = 2.0 ** -149  # the grid of fp32 values this small: y, the largest, the scale
    assert_within(s, scale, scale * 1e-4 + 1.1 * tiny, "scale")
    assert not s[4].any() and not y8[4].float().any()
    ratio = torch.where(scale[:, None] > 0, y / scale[:, None], 0.0)
    # e4m3: half a step is 2^-4 of the value, 2^-10 below the normal range; y and
    # the maximum are off by up to a step of their grid each, which the ratio scales
    grid = torch.where(scale > 0, 1.1 * tiny / scale, 0.0)[:, None]
    tol = torch.maximum(ratio.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10, dtype=torch.float64)) * 1.01 \
        + ratio.abs() * (1e-4 + grid / 448) + grid
    assert_within(y8.double(), ratio, tol, "y8")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,d", [(6, 64), (600, 64), (600, 1000), (6, 4096), (6, 1001), (6, 17001)])
def test_rms_norm_fp8_of_rows_that_are_not_finite(cuda_device, dtype, rows, d):
    # the largest |y| of a row that holds a NaN is NaN, and so is its scale
    x, w = _randn((rows, d), dtype, cuda_device, 1), _randn((d,), dtype, cuda_device, 2)
    clean = cawq.rms_norm_fp8(x, w)
    bad = x.clone()
    bad[1, d - 1], bad[3, d // 2], bad[5, 0] = float("nan"), float("inf"), -float("inf")
    y8, s, _ = cawq.rms_norm_fp8(bad, w)
    hit = torch.zeros(rows, dtype=torch.bool, device=cuda_device)
    hit[[1, 3, 5]] = True
    assert s[hit].isnan().all() and y8[1].float().isnan().all()
    assert y8[3, d // 2].float().isnan() and y8[5, 0].float().isnan()
    assert torch.equal(s[~hit], clean[1][~hit])
    assert torch.equal(y8[~hit].view(torch.uint8), clean[0][~hit].view(torch.uint8))


@pytest.mark.parametrize("pages,hkv", [(1, 2), (1, 1), (5, 1), (5, 2)])
@pytest.mark.parametrize("what", ["heads", "pages", "slots"])
def test_broadcast_caches(cuda_device, pages, hkv, what):
    # views with a stride of 0: they may be read, whichever kernel takes the call
    page, d = 64, 128
    shape = dict(heads=(pages, 1, page, d), pages=(1, hkv, page, d), slots=(pages, hkv, 1, d))[what]
    k, v = (_randn(shape, F16, cuda_device, s).expand(pages, hkv, page, d) for s in (1, 2))
    total = pages * page - 3
    q = _randn((min(total, 200), 4 * hkv, d), F16, cuda_device, 3)
    n = q.shape[0]
    table = torch.arange(pages, dtype=torch.int32, device=cuda_device)[None]
    lens, q_start = _i32([total], cuda_device), _i32([0, n], cuda_device)
    c = Cache.__new__(Cache)
    c.seqs, c.starts, c.k = [(n, total)], [0, n], k
    c.kd, c.vd = ([x.transpose(1, 2).reshape(pages * page, hkv, d)[:total]] for x in (k, v))
    ref, tol = attention_ref(q, c)
    assert_within(cawq.attention_prefill(q, k, v, table, lens, q_start), ref, tol)
    out = cawq.attention_decode(q[-1:], k, v, table, lens)
    assert_within(out, ref[-1:], tol[-1:])


@pytest.mark.parametrize("pages,width", [(0, 0), (0, 3), (4, 0)])
def test_caches_and_tables_that_hold_nothing(cuda_device, pages, width):
    kc = torch.ones((pages, 2, 16, 64), dtype=F16, device=cuda_device)
    vc = kc.clone()
    table = torch.zeros((3, width), dtype=torch.int32, device=cuda_device)
    q, k, v, rope = _rope_args(cuda_device, 3)
    for lens, error in (([0, 0, 0], 0), ([0, 20, 1], 4)):
        lens = _i32(lens, cuda_device)
        assert not cawq.attention_decode(q, kc, vc, table, lens).any()
        assert cawq.device_error() == error
        for starts in ([0, 1, 2, 3], [0, 0, 3, 3]):
            assert not cawq.attention_prefill(q, kc, vc, table, lens, _i32(starts, cuda_device)).any()
            assert cawq.device_error() == error
        out = cawq.rope_append(q, k, v, rope, kc, vc, table, lens)
        assert cawq.device_error() == error
        assert out[1].any() == bool(error) and not out[0].any()
        assert (kc == 1).all() and (vc == 1).all()
