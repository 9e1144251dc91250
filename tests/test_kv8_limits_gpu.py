"""GPU: the 8-bit paged KV cache at the limits of its scales and lengths."""
import math

import numpy as np
import pytest
import torch
from test_kv8_gpu import D, Held, attend64, filled

pytestmark = pytest.mark.gpu

# rows per request, kv heads, query heads per kv head: one token, a few, a prompt chunk (the kernels differ)
SHAPES = [(1, 2, 3), (5, 2, 3), (300, 10, 3)]


def held_by(cache, scales):
    """What the cache holds, with the K scales moved into the K values: the exponents left are those of V, by which the
    roundings of the weights are counted."""
    held = Held(cache, scales)
    held.x[:, :, :, 0] *= np.exp2(held.e[:, :, 0].astype(np.float64))[:, :, None, None]
    held.e[:, :, 0] = 0
    return held


def bounds(n, batch):
    return None if n == 1 else torch.arange(0, n * batch + 1, n, dtype=torch.int32)


@pytest.mark.parametrize("n,heads,group", SHAPES)
def test_pages_of_the_lowest_scale(cuda_device, n, heads, group):
    """V so small that every page has the lowest scale there is, 2^-127: the outputs are small, not 0."""
    from prime_kernels_b200 import kv8

    g = torch.Generator().manual_seed(n)
    cache, scales, table, lens = filled(g, [n + 90, n + 7], heads, 16, False, cuda_device, lambda k, v: (k, v * 2.0 ** -122))
    held = held_by(cache, scales)
    live = [int(p) for p in table.flatten() if p >= 0]
    assert (held.e[live] == 0).all()
    q, cu = torch.randn(2 * n, heads * group, D, generator=g).bfloat16(), bounds(n, 2)
    out = kv8.attention(q.to(cuda_device), cache, scales, table.to(cuda_device), lens.to(cuda_device), None if cu is None else cu.to(cuda_device))
    want, _, tol, _, _ = attend64(q, held, table.numpy(), lens.numpy(), np.arange(3) if cu is None else cu.numpy(), D ** -0.5)
    # bf16 below 2^-126 has steps of 2^-133: half of one more than the relative roundings that attend64 counts
    assert (np.abs(out.double().cpu().numpy() - want) <= tol + 2.0 ** -134).all()
    assert (np.abs(want) > 2.0 ** -126).mean() > 0.5


@pytest.mark.parametrize("n,heads,group", SHAPES)
def test_nan_among_zeros(cuda_device, n, heads, group):
    """Pages of zeros have the lowest scale; NaN does not count for it and reaches the rows that see it all the same."""
    from prime_kernels_b200 import kv8

    g = torch.Generator().manual_seed(n + 1)

    def gain(k, v):
        v = torch.zeros_like(v)
        v[8, 1, 5] = math.nan                              # position 8 of the first request
        return k, v

    cache, scales, table, lens = filled(g, [n + 90, n + 7], heads, 16, False, cuda_device, gain)
    q, cu = torch.randn(2 * n, heads * group, D, generator=g).bfloat16(), bounds(n, 2)
    out = kv8.attention(q.to(cuda_device), cache, scales, table.to(cuda_device), lens.to(cuda_device), None if cu is None else cu.to(cuda_device))
    want = torch.zeros(2 * n, heads * group, D)
    want[:n, group: 2 * group, 5] = math.nan
    out = out.float().cpu()
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and (out[~torch.isnan(want)] == 0).all()


@pytest.mark.parametrize("n,heads,group", SHAPES)
@pytest.mark.parametrize("ratio", [0, 8, 13, 20, 24, 30])
@pytest.mark.parametrize("alike", [True, False])
def test_what_pages_of_small_scales_add(cuda_device, n, heads, group, ratio, alike):
    """V in dims 0..31 of every third page, 2^-ratio of it in dims 32..63 of the others: the weights of those are f16 relative
    to the row's largest product of weight and V scale, off by 2^-11 of themselves or 2^-25 of that product."""
    from prime_kernels_b200 import kv8

    g = torch.Generator().manual_seed(n + ratio)

    def gain(k, v):
        big = (torch.arange(len(v)) // 16 % 3 == 0)[:, None, None]
        upper = torch.arange(D) >= 32
        v = torch.where(big, v * ~upper, v * upper * 2.0 ** -ratio)
        return (k * 0 if alike else k), v

    cache, scales, table, lens = filled(g, [n + 91, n + 21], heads, 16, False, cuda_device, gain)
    q, cu = torch.randn(2 * n, heads * group, D, generator=g).bfloat16(), bounds(n, 2)
    out = kv8.attention(q.to(cuda_device), cache, scales, table.to(cuda_device), lens.to(cuda_device), None if cu is None else cu.to(cuda_device))
    want, _, tol, _, _ = attend64(q, held_by(cache, scales), table.numpy(), lens.numpy(), np.arange(3) if cu is None else cu.numpy(), D ** -0.5)
    off = np.abs(out.double().cpu().numpy() - want)
    assert (off <= tol).all()
    if alike and ratio <= 13:
        # equal scores: weights are powers of two, exact in f16 down to 2^-24 (2^8 of them are the prompt kernel's to lose,
        # a page's scale varies by another 2^2): nothing but the roundings of the sums (fp32) and of the output (bf16) is left
        held = held_by(cache, scales)
        held.x[:, :, :, 1] = np.abs(held.x[:, :, :, 1])
        spread, _, _, _, _ = attend64(q, held, table.numpy(), lens.numpy(), np.arange(3) if cu is None else cu.numpy(), D ** -0.5)
        assert (off <= 2.0 ** -8 * np.abs(want) + 2.0 ** -17 * spread).all()
