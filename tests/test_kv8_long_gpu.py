"""GPU: attention over the 8-bit cache at contexts where a warp looks pages up more than once, against the definition.

The kernel for few tokens holds the pages of 16 steps of a warp (one CTA of eight warps: 4096 keys), the one for prompt
chunks those of 32 steps (2048 keys); behind them the next ones are read while the last of the old ones are in use."""
import numpy as np
import pytest
import torch
from test_kv8_gpu import D, attend64, filled
from test_kv8_limits_gpu import held_by

pytestmark = pytest.mark.gpu


def check(dev, g, seq, new, heads, group, size, planes, holes=()):
    """Page scales differ from page to page in K and V; ``holes``: (request, position) of pages taken out of the pool."""
    from prime_kernels_b200 import kv8

    def gain(k, v):
        i = torch.arange(len(k)) // 16
        return k * torch.exp2((i * 5 % 4 - 2).float())[:, None, None], v * torch.exp2((i * 3 % 7 - 3).float())[:, None, None]

    cache, scales, table, lens = filled(g, seq, heads, size, planes, dev, gain)
    for r, at in holes:
        table[r, at // size] = -1
    cu = torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32))
    q = torch.randn(sum(new), heads * group, D, generator=g).bfloat16()
    out, lse = kv8.attention(q.to(dev), cache, scales, table.to(dev), lens.to(dev), None if max(new) == 1 else cu.to(dev),
                             max_query_len=max(new), return_lse=True)
    want, wlse, tol, tol_lse, _ = attend64(q, held_by(cache, scales), table.numpy(), lens.numpy(), cu.numpy(), D ** -0.5)
    out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    some = np.isfinite(wlse)
    assert np.array_equal(np.isneginf(lse), ~some) and (out[~some] == 0).all()
    assert (np.abs(out - want) <= tol).all(), np.abs(out - want).max()
    assert (np.abs(lse - np.where(some, wlse, 0.0))[some] <= tol_lse[some]).all()


@pytest.mark.parametrize("n", [1, 5])
@pytest.mark.parametrize("long,size,planes", [(4095, 16, False), (4097, 16, True), (4200, 64, False), (8190, 16, False), (8192, 256, True)])
def test_few_tokens_in_one_cta(cuda_device, long, size, planes, n):
    """64 requests of 5 heads, so that an item has one CTA; one of them long, with holes around the second look-up."""
    g = torch.Generator().manual_seed(long + n)
    seq = [n + 3 + i % 40 for i in range(64)]
    seq[7] = long
    holes = [(7, 4095 - size), (7, min(4096 + size, long - 1))] if long > 4097 else [(7, 100)]
    check(cuda_device, g, seq, [n] * 64, 5, 3, size, planes, holes)


@pytest.mark.parametrize("n", [1, 6])
@pytest.mark.parametrize("long", [33000, 65537])
def test_few_tokens_in_a_cluster(cuda_device, long, n):
    """One request: eight CTAs a head, each with more than 4096 keys."""
    g = torch.Generator().manual_seed(long)
    check(cuda_device, g, [long], [n], 2, 3, 64, False, [(0, 16500), (0, long - 70)])


@pytest.mark.parametrize("long", [2048, 2049, 2112, 4096, 4200, 6500])
@pytest.mark.parametrize("size,planes", [(16, False), (64, True), (256, False)])
def test_prompt_chunks(cuda_device, long, size, planes):
    """Three chunks of which one is long, holes in the pages next to the second look-up and in the last one."""
    g = torch.Generator().manual_seed(long + size)
    holes = [(0, 2047), (0, long - 301)] + ([(0, 2048 + size)] if long > 4000 else [])
    check(cuda_device, g, [long, 305, 400], [300, 290, 310], 10, 3, size, planes, holes)
