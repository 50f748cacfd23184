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
