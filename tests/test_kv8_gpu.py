"""GPU: the 8-bit paged KV cache (store, attention) against its definition in 64 bits."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
D = 64


# ------------------------------------------------------------------------------------------------ 64-bit definition
def e4m3(x):
    """Nearest e4m3 value (ties to even, largest 448), as doubles; NaN stays."""
    with np.errstate(invalid="ignore"):
        y = np.clip(x, -448.0, 448.0)
        _, e = np.frexp(np.abs(np.where(np.isnan(y), 0.0, y)))
        step = np.exp2(np.maximum(e - 1, -6) - 3.0)
        return np.clip(np.rint(y / step) * step, -448.0, 448.0)


def exponent(amax):
    """Biased exponent of the scale: round-up of fp32 amax * fl(1/448) to a power of two."""
    x = (amax.astype(np.float32) * np.float32(1 / 448)).astype(np.float64)
    m, e = np.frexp(x)
    return np.where(x > 0, np.clip(np.where(m == 0.5, e - 1, e) + 127, 0, 254), 0).astype(np.int64)


class Held:
    """What a cache holds, [pages, heads, slots, 2, 64] e4m3 values and [pages, heads, 2] exponents, in doubles."""

    def __init__(self, cache, scales):
        c = cache.float().cpu().numpy().astype(np.float64)
        self.planes = c.ndim == 5
        self.x = (c.transpose(1, 3, 2, 0, 4) if self.planes else c.reshape(*c.shape[:3], 2, D)).copy()
        self.e = scales.view(torch.uint8).cpu().numpy().astype(np.int64)

    def append(self, k, v, table, seq, cu):
        new = np.stack([k.double().cpu().numpy(), v.double().cpu().numpy()], 2)     # [T, heads, 2, 64]
        size = self.x.shape[2]
        for r in range(len(seq)):
            a, b = int(cu[r]), min(int(cu[r + 1]), len(new))
            n = b - a
            pos = int(seq[r]) - n
            t = max(0, -pos)
            while t < n:
                col, slot = divmod(pos + t, size)
                m = min(size - slot, n - t)
                if col < table.shape[1] and 0 <= table[r, col] < len(self.x):
                    page = int(table[r, col])
                    part = new[a + t: a + t + m]
                    size_of = np.abs(np.where(np.isfinite(part), part, 0.0)).max(axis=(0, 3))
                    e = exponent(size_of)
                    if slot:
                        e = np.maximum(e, self.e[page])
                        self.x[page, :, :slot] = e4m3(self.x[page, :, :slot] * np.exp2(self.e[page] - e)[:, None, :, None])
                    with np.errstate(over="ignore"):
                        self.x[page, :, slot: slot + m] = e4m3(part * np.exp2(127.0 - e)[None, :, :, None]).transpose(1, 0, 2, 3)
                    self.e[page] = e
                t += m

    def same(self, cache, scales):
        other = Held(cache, scales)
        assert np.array_equal(self.e, other.e)
        assert np.array_equal(self.x, other.x, equal_nan=True)

    def values(self, pages):
        """K and V of a list of pages, [tokens, heads, 64] each; a page outside the pool gives None tokens (NaN marks)."""
        x, ok = [], []
        for p in pages:
            inside = 0 <= p < len(self.x)
            q = self.x[p] * np.exp2(self.e[p] - 127.0)[:, None, :, None] if inside else np.zeros(self.x.shape[1:])
            x.append(q.transpose(1, 0, 2, 3))
            ok += [inside] * self.x.shape[2]
        if not x:
            return np.zeros((0, self.x.shape[1], D)), np.zeros((0, self.x.shape[1], D)), np.zeros(0, bool)
        x = np.concatenate(x)
        return x[:, :, 0], x[:, :, 1], np.array(ok)


def attend64(q, held, table, seq, cu, scale):
    """(out, lse, tolerance of out, tolerance of lse) of every row, in doubles.

    Tolerances count the kernel's roundings.  Scores: products are exact (bf16 x e4m3 bits) and sums of 64 of them
    in fp32 are off by at most 64 * 2^-22 of the sum of magnitudes (an adder that truncates), plus three fp32
    products: ds = 2^-15 * sum|q k| * scale, in the exponent.  Weights: f16, 2^-11 of each, or 2^-25 of the largest
    (s + scale exponent) one where they are subnormal, and ex2 2^-22: the second gives n * 2^-25 * 448 * 2^(e - 127)
    over the sum.  Output: bf16, 2^-8."""
    q = q.double().cpu().numpy()
    tokens, heads, _ = q.shape
    group = heads // held.x.shape[1]
    size = held.x.shape[2]
    out, lse = np.zeros_like(q), np.full((tokens, heads), -np.inf)
    tol, tol_lse, mine = np.zeros_like(q), np.zeros((tokens, heads)), np.zeros(tokens, bool)
    for r in range(len(seq)):
        a, b = max(int(cu[r]), 0), min(int(cu[r + 1]), tokens)
        n, length = b - a, min(max(int(seq[r]), 0), table.shape[1] * size)
        if n <= 0:
            continue
        mine[a:b] = True
        pages = [int(p) for p in table[r, : -(-length // size)]]
        k, v, ok = held.values(pages)
        k, v, ok = k[:length], v[:length], ok[:length]
        top = np.array([2.0 ** float(held.e[p].max() - 127) for p in pages if 0 <= p < len(held.x)] or [0.0]).max()
        upto = np.clip(int(seq[r]) - n + 1 + np.arange(n), 0, length)
        sees = (np.arange(length) < upto[:, None]) & ok                                    # [n, length]
        some = sees.any(1)
        for h in range(heads):
            kk, vv, qq = k[:, h // group], v[:, h // group], q[a:b, h]
            s = np.where(sees, qq @ kk.T * scale, -np.inf)
            ds = 2.0 ** -15 * np.where(sees, np.abs(qq) @ np.abs(kk).T, 0.0).max(1, initial=0.0) * abs(scale)
            m = np.where(some, s.max(1, initial=-np.inf), 0.0)
            w = np.exp(s - m[:, None])
            z = np.where(some, w.sum(1), 1.0)
            out[a:b, h] = w @ vv / z[:, None]
            lse[a:b, h] = np.where(some, m + np.log(z), -np.inf)
            spread = w @ np.abs(vv) / z[:, None]
            tol[a:b, h] = (2.0 ** -8 * np.abs(out[a:b, h]) + spread * (2.0 ** -11 + 2.0 ** -18 + 2 * ds)[:, None] +
                           (sees.sum(1) * 2.0 ** -25 * 448 * top / z)[:, None])
            tol_lse[a:b, h] = ds + 2.0 ** -21 * (1 + np.abs(m) + np.log(z))
    return out, lse, tol, tol_lse, mine


# ------------------------------------------------------------------------------------------------ set-up
def pool(g, pages, heads, size, planes, dev, spread=1.0):
    """A cache with content, every dead byte a NaN: pages are filled by the caller's appends."""
    from prime_kernels_b200 import kv8

    cache, scales = kv8.empty_cache(pages, heads, size, planes=planes, device=dev)
    cache.view(torch.uint8).fill_(0x7f)
    scales.view(torch.uint8).fill_(0xff)
    return cache, scales


def tables(g, seq, size, cols=None, spare=3):
    need = [-(-max(s, 0) // size) for s in seq]
    cols = max(max(need), 1) if cols is None else cols
    order = torch.randperm(sum(need) + spare, generator=g).tolist()
    t = torch.full((len(seq), cols), -1, dtype=torch.int32)
    for r, n in enumerate(need):
        for c in range(min(n, cols)):
            t[r, c] = order.pop()
        del order[: max(0, n - cols)]
    return t, sum(need) + spare


def filled(g, seq, heads, size, planes, dev, gain=None):
    """Cache, scales, table of requests with ``seq`` tokens each; dead slots and dead pages hold NaN bytes."""
    from prime_kernels_b200 import kv8

    table, pages = tables(g, seq, size)
    cache, scales = pool(g, pages, heads, size, planes, dev)
    total = sum(seq)
    k = torch.randn(total, heads, D, generator=g)
    v = torch.randn(total, heads, D, generator=g)
    if gain is not None:
        k, v = gain(k, v)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(seq)]), dtype=torch.int32)
    lens = torch.tensor(seq, dtype=torch.int32)
    if total:
        kv8.append(k.bfloat16().to(dev), v.bfloat16().to(dev), cache, scales, table.to(dev), lens.to(dev), cu.to(dev))
    return cache, scales, table, lens


def run_attention(dev, cache, scales, table, lens, q, cu=None, scale=None, **kw):
    from prime_kernels_b200 import kv8

    batch = len(lens)
    bounds = np.arange(batch + 1) if cu is None else cu.numpy()
    out, lse = kv8.attention(q.to(dev), cache, scales, table.to(dev), lens.to(dev), None if cu is None else cu.to(dev),
                             scale=scale, return_lse=True, **kw)
    want, wlse, tol, tol_lse, mine = attend64(q, Held(cache, scales), table.numpy(), lens.numpy(), bounds,
                                              D ** -0.5 if scale is None else scale)
    got, glse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    assert np.isfinite(got[mine]).all()
    bad = np.abs(got - want)[mine] > tol[mine]
    assert not bad.any(), (np.argwhere(bad)[:5], np.abs(got - want)[mine].max())
    live = np.isfinite(wlse) & mine[:, None]
    assert np.array_equal(glse[~live & mine[:, None]], wlse[~live & mine[:, None]])
    off = np.abs(glse[live] - wlse[live])
    assert (off <= tol_lse[live]).all(), off.max()
    return out, lse


# ------------------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("planes", [False, True])
@pytest.mark.parametrize("size", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("heads", [1, 3, 5])
def test_append_in_pieces(cuda_device, planes, size, heads):
    """Ragged pieces, the scale of a begun page growing and not growing, K and V out of one projection's rows."""
    from prime_kernels_b200 import kv8

    g = torch.Generator().manual_seed(size + heads)
    counts = [[1, 17, 300, 0, 5], [1, 1, 1, 1, 1], [31, 2, 0, 64, 200], [1, 16, 16, 1, 3]]
    table, pages = tables(g, [sum(c[r] for c in counts) for r in range(5)], size)
    cache, scales = pool(g, pages, heads, size, planes, cuda_device)
    held = Held(cache, scales)
    seq = np.zeros(5, np.int64)
    for i, c in enumerate(counts):
        total = sum(c)
        qkv = (torch.randn(total, (2 * heads + 2) * D, generator=g) * 4.0 ** ((i * 3) % 4 - 1)).bfloat16()
        k = qkv[:, D: D + heads * D].view(total, heads, D)
        v = qkv[:, (heads + 1) * D: (2 * heads + 1) * D].view(total, heads, D)
        cu = np.concatenate([[0], np.cumsum(c)]).astype(np.int32)
        seq += np.array(c)
        qd = qkv.to(cuda_device)
        kd, vd = qd[:, D: D + heads * D].view(total, heads, D), qd[:, (heads + 1) * D: (2 * heads + 1) * D].view(total, heads, D)
        one = c == [1] * 5
        kv8.append(kd, vd, cache, scales, table.to(cuda_device), torch.tensor(seq, dtype=torch.int32, device=cuda_device),
                   None if one else torch.from_numpy(cu).to(cuda_device))
        held.append(k, v, table.numpy(), seq, cu)
        held.same(cache, scales)


def test_append_special_values(cuda_device):
    from prime_kernels_b200 import kv8

    g = torch.Generator().manual_seed(1)
    cache, scales = pool(g, 6, 2, 16, False, cuda_device)
    held = Held(cache, scales)
    x = torch.randn(5, 16, 2, D, generator=g)
    x[0, 3, 0, 7], x[0, 4, 1, 0], x[0, 5, 0, 1] = math.inf, -math.inf, math.nan
    x[1] = 0.0
    x[2] *= 2.0 ** -130                                  # subnormal
    x[3] *= 2.0 ** 126
    x[4, :, 0] = torch.tensor([448.0] + [1.0] * 63)
    k = x.reshape(80, 2, D).bfloat16()
    v = x.flip(1).reshape(80, 2, D).bfloat16()
    table = torch.arange(5, dtype=torch.int32)[:, None]
    lens, cu = torch.full((5,), 16, dtype=torch.int32), torch.arange(0, 96, 16, dtype=torch.int32)
    kv8.append(k.to(cuda_device), v.to(cuda_device), cache, scales, table.to(cuda_device), lens.to(cuda_device), cu.to(cuda_device))
    held.append(k, v, table.numpy(), lens.numpy(), cu.numpy())
    held.same(cache, scales)
    assert torch.equal(torch.isnan(kv8.dequantise(cache, scales)[0, :, :, :D]).cpu().sum(), torch.tensor(1))


def test_append_leaves_the_rest_alone(cuda_device):
    """Rows of no request, pages outside the pool, positions behind the table and before 0 store nothing."""
    from prime_kernels_b200 import kv8

    g = torch.Generator().manual_seed(2)
    cache, scales = pool(g, 5, 3, 16, True, cuda_device)
    held = Held(cache, scales)
    table = torch.tensor([[0, 1], [-1, 2], [3, 99]], dtype=torch.int32)
    seq = torch.tensor([40, 20, 30], dtype=torch.int32)         # 40 > two pages
    cu = torch.tensor([2, 20, 40, 72], dtype=torch.int32)       # the last request has more rows than positions
    k, v = torch.randn(90, 3, D, generator=g).bfloat16(), torch.randn(90, 3, D, generator=g).bfloat16()
    # page 0 of request 0 was begun before: give its scales a value
    scales.view(torch.uint8)[1] = 127
    cache.view(torch.uint8)[:, 1] = 0x38
    held = Held(cache, scales)
    kv8.append(k.to(cuda_device), v.to(cuda_device), cache, scales, table.to(cuda_device), seq.to(cuda_device), cu.to(cuda_device))
    held.append(k, v, table.numpy(), seq.numpy(), cu.numpy())
    held.same(cache, scales)
    before = cache.clone()
    kv8.append(k[:0].to(cuda_device), v[:0].to(cuda_device), cache, scales, table.to(cuda_device), seq.to(cuda_device),
               torch.zeros(4, dtype=torch.int32, device=cuda_device))
    assert torch.equal(cache.view(torch.uint8), before.view(torch.uint8))


# ------------------------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("planes", [False, True])
@pytest.mark.parametrize("size", [16, 64, 256])
@pytest.mark.parametrize("heads,group", [(1, 1), (3, 3), (2, 8), (1, 20), (5, 1)])
def test_decode_attention(cuda_device, planes, size, heads, group):
    g = torch.Generator().manual_seed(size + heads * 10 + group)
    seq = [1, 15, 16, 17, 0, 130, 700]
    cache, scales, table, lens = filled(g, seq, heads, size, planes, cuda_device)
    q = torch.randn(len(seq), heads * group, D, generator=g).bfloat16()
    run_attention(cuda_device, cache, scales, table, lens, q)


@pytest.mark.parametrize("batch,length", [(1, 6000), (2, 2500), (70, 40)])
def test_decode_attention_spread_over_ctas(cuda_device, batch, length):
    """One long request takes a whole cluster per head, many short ones none."""
    g = torch.Generator().manual_seed(length)
    seq = [length - 3 * i % length for i in range(batch)]
    cache, scales, table, lens = filled(g, seq, 3, 16, False, cuda_device)
    q = (3 * torch.randn(batch, 9, D, generator=g)).bfloat16()
    run_attention(cuda_device, cache, scales, table, lens, q)


@pytest.mark.parametrize("heads,group", [(1, 1), (3, 3), (2, 5)])
@pytest.mark.parametrize("new", [[2, 5, 0, 1, 9], [33, 16, 0, 130, 7], [1, 1, 300, 64, 65], [700, 3, 0, 260, 515], [128, 64, 0, 1200, 641]])
@pytest.mark.parametrize("known", [True, False])
def test_ragged_queries(cuda_device, heads, group, new, known):
    """Several query tokens each, causal among themselves; rows behind the last request are left alone."""
    g = torch.Generator().manual_seed(sum(new) + heads)
    seq = [new[0], new[1] + 40, 9, new[3] + 333, new[4] + 16]
    cache, scales, table, lens = filled(g, seq, heads, 16, heads == 2, cuda_device)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32)
    q = torch.randn(sum(new) + 6, heads * group + 2, D, generator=g).bfloat16()[:, 1:-1]
    out = torch.full(q.shape, 77.0, dtype=torch.bfloat16, device=cuda_device)
    run_attention(cuda_device, cache, scales, table, lens, q, cu, max_query_len=max(new) if known else None, out=out)
    assert (out[sum(new):] == 77).all()
    # a max_query_len that is too small: every row is computed all the same
    run_attention(cuda_device, cache, scales, table, lens, q, cu, max_query_len=1)


@pytest.mark.parametrize("heads,group,first,second", [(2, 2, 12, 8), (4, 4, 700, 600)])
def test_more_queries_than_positions(cuda_device, heads, group, first, second):
    """Rows before position 0 see nothing: zeros and -inf."""
    g = torch.Generator().manual_seed(3)
    cache, scales, table, lens = filled(g, [5, 40], heads, 16, False, cuda_device)
    cu = torch.tensor([0, first, first + second], dtype=torch.int32)
    q = torch.randn(first + second, heads * group, D, generator=g).bfloat16()
    out, lse = run_attention(cuda_device, cache, scales, table, lens, q, cu)
    assert (out[: first - 5] == 0).all() and (lse[: first - 5] == -math.inf).all()
    run_attention(cuda_device, cache, scales, table, lens, q, cu, max_query_len=max(first, second))


@pytest.mark.parametrize("n,heads", [(1, 2), (40, 2), (333, 12)])
def test_scales_that_differ_from_page_to_page(cuda_device, n, heads):
    """V scales over 60 binades, pages of zeros, large scores: no page's scale may hurt another's tokens."""
    g = torch.Generator().manual_seed(4)

    def gain(k, v):
        i = torch.arange(len(v)) // 16
        v = v * torch.exp2((i * 37 % 61 - 40).float())[:, None, None]
        v[(i % 5) == 2] = 0.0
        k = k * torch.exp2((i % 4 - 2).float())[:, None, None]
        return k, v

    cache, scales, table, lens = filled(g, [400, 333], heads, 16, False, cuda_device, gain)
    cu = None if n == 1 else torch.tensor([0, n, 2 * n], dtype=torch.int32)
    q = (4 * torch.randn(2 * n, 2 * heads, D, generator=g)).bfloat16()
    run_attention(cuda_device, cache, scales, table, lens, q, cu)


@pytest.mark.parametrize("n,heads,group", [(1, 1, 2), (40, 1, 2), (100, 12, 10)])
def test_low_scale_pages_under_a_masked_high_scale_one(cuda_device, n, heads, group):
    """All the weight lies on pages whose V scale is 2^-30 of another page's that gets next to none of it."""
    from prime_kernels_b200 import kv8

    g = torch.Generator().manual_seed(5)

    def gain(k, v):
        v[:16] *= 2.0 ** 30
        k[:16] = -k[:16].abs() - 6.0                     # scores near -250 on the first page
        k[16:] = k[16:].abs()
        return k, v

    cache, scales, table, lens = filled(g, [100 + n - 1], heads, 16, False, cuda_device, gain)
    q = torch.rand(n, heads * group, D, generator=g).add(4.0).bfloat16()
    cu = None if n == 1 else torch.tensor([0, n], dtype=torch.int32)
    out = kv8.attention(q.to(cuda_device), cache, scales, table.to(cuda_device), lens.to(cuda_device),
                        None if cu is None else cu.to(cuda_device))
    want, _, tol, _, _ = attend64(q, Held(cache, scales), table.numpy(), lens.numpy(),
                                  np.arange(2) if cu is None else cu.numpy(), D ** -0.5)
    # the first page's share is below 2^-100: the tolerance may not count its scale
    tight = 2.0 ** -8 * np.abs(want) + 2.0 ** -9 * 4.0
    assert (np.abs(out.double().cpu().numpy() - want) <= np.minimum(tol, tight)).all()


@pytest.mark.parametrize("n,heads", [(1, 1), (400, 10)])
@pytest.mark.parametrize("size", [1e-30, 1.0, 1e30, -1.0, 0.0])
def test_q_of_any_size(cuda_device, size, n, heads):
    """q is brought into f16's range by a power of two per row; a row of zeros weighs all keys alike, and so does a scale
    of 0; a negative scale turns the order round."""
    g = torch.Generator().manual_seed(6)
    cache, scales, table, lens = filled(g, [76 + n, 449 + n], heads, 16, False, cuda_device)
    q = torch.randn(2 * n, 3 * heads, D, generator=g)
    q[0, 1] = 0.0
    cu = None if n == 1 else torch.tensor([0, n, 2 * n], dtype=torch.int32)
    run_attention(cuda_device, cache, scales, table, lens, (q * (abs(size) or 1.0)).bfloat16(), cu, scale=0.125 / size if size else 0.0)


@pytest.mark.parametrize("n,heads", [(1, 2), (16, 2), (300, 10)])
def test_pages_outside_the_pool_are_masked(cuda_device, n, heads):
    g = torch.Generator().manual_seed(7)
    cache, scales, table, lens = filled(g, [390, 368, 16], heads, 16, False, cuda_device)
    table[0, 2], table[1, 0], table[2, 0] = -1, 10 ** 6, -5          # the last request has nothing left
    q = torch.randn(3 * n, 3 * heads, D, generator=g).bfloat16()
    cu = None if n == 1 else torch.tensor([0, n, 2 * n, 3 * n], dtype=torch.int32)
    out, lse = run_attention(cuda_device, cache, scales, table, lens, q, cu)
    assert (out[2 * n:] == 0).all() and (lse[2 * n:] == -math.inf).all()
    lens[1] = 10 ** 6                                                # longer than its table: clamped to it
    run_attention(cuda_device, cache, scales, table, lens, q, cu)
    lens[0] = -4
    run_attention(cuda_device, cache, scales, table, lens, q, cu)


@pytest.mark.parametrize("n,heads", [(1, 1), (400, 10)])
def test_nan_is_not_hidden(cuda_device, n, heads):
    from prime_kernels_b200 import kv8

    g = torch.Generator().manual_seed(9)
    cache, scales, table, lens = filled(g, [400, 410], heads, 16, False, cuda_device)
    q = torch.randn(2 * n, 3 * heads, D, generator=g).bfloat16()
    q[0, 0, 5] = math.nan
    cu = None if n == 1 else torch.tensor([0, n, 2 * n], dtype=torch.int32, device=cuda_device)
    out = kv8.attention(q.to(cuda_device), cache, scales, table.to(cuda_device), lens.to(cuda_device), cu)
    assert torch.isnan(out[0, 0]).all()
    out[0, 0] = 0
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("planes", [False, True])
@pytest.mark.parametrize("n,group,heads,size", [(3, 2, 2, 16), (4, 5, 1, 32), (40, 3, 2, 16), (77, 4, 10, 64), (260, 3, 10, 16), (300, 7, 3, 256)])
def test_nan_of_later_tokens(cuda_device, n, group, heads, size, planes):
    """NaN among the V values (or in the K) of a token reaches the rows that see it, and only those."""
    from prime_kernels_b200 import kv8

    g = torch.Generator().manual_seed(n)
    seq = [n + 201, n, n + 990]
    table, pages = tables(g, seq, size)
    cache, scales = pool(g, pages, heads, size, planes, cuda_device)
    total, starts = sum(seq), np.concatenate([[0], np.cumsum(seq)])
    k, v = torch.randn(total, heads, D, generator=g), torch.randn(total, heads, D, generator=g)
    marks = [(0, 200, 0, 3), (0, 203, 0, 63), (1, 1, heads - 1, 17), (1, n - 1, 0, 0), (2, 990 + n // 2, heads - 1, 32),
             (2, 990 + n // 2, heads - 1, 35)]                            # request, position, kv head, dim
    lens, cu_all = torch.tensor(seq, dtype=torch.int32), torch.from_numpy(starts.astype(np.int32))
    for bad in (False, True):
        kb, vb = k.bfloat16(), v.bfloat16()
        for r, at, h, d in marks:
            vb[starts[r] + at, h, d] = math.nan if bad else 0.0
        if bad:
            kb[starts[2] + 990 + n - 1, 0, 9] = math.nan                  # the last token of all
        kv8.append(kb.to(cuda_device), vb.to(cuda_device), cache, scales, table.to(cuda_device), lens.to(cuda_device), cu_all.to(cuda_device))
        q = torch.randn(3 * n, group * heads, D, generator=torch.Generator().manual_seed(1)).bfloat16()
        cu = torch.arange(0, 3 * n + 1, n, dtype=torch.int32)
        if not bad:
            want, want_lse, tol, tol_lse, _ = attend64(q, Held(cache, scales), table.numpy(), lens.numpy(), cu.numpy(), D ** -0.5)
    out, lse = kv8.attention(q.to(cuda_device), cache, scales, table.to(cuda_device), lens.to(cuda_device), cu.to(cuda_device),
                             max_query_len=n, return_lse=True)
    out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    for r, at, h, d in marks:
        sees = r * n + max(at - (seq[r] - n), 0)
        want[sees: (r + 1) * n, h * group: (h + 1) * group, d] = math.nan
    want[-1, :group] = want_lse[-1, :group] = math.nan
    for got, ref, t in ((out, want, tol), (lse, want_lse, tol_lse)):
        assert np.array_equal(np.isnan(got), np.isnan(ref))
        assert (np.abs(got - ref)[~np.isnan(ref)] <= t[~np.isnan(ref)]).all()


@pytest.mark.parametrize("known", [False, True])
@pytest.mark.parametrize("new", [[300] + [1] * 599, [800] + [30] * 49])
def test_one_long_among_many(cuda_device, new, known):
    """A request with far more rows than the mean: its tiles are taken in turns."""
    g = torch.Generator().manual_seed(len(new))
    cache, scales, table, lens = filled(g, [n + 20 for n in new], 10, 16, False, cuda_device)
    q = torch.randn(sum(new), 30, D, generator=g).bfloat16()
    cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32)
    run_attention(cuda_device, cache, scales, table, lens, q, cu, max_query_len=max(new) if known else None)


def test_no_wait_gave_up(cuda_device):
    """After everything above: no bounded wait of the prompt kernel has expired."""
    from prime_kernels_b200 import _cabi

    assert _cabi.library().pk_kv8_wait_timeouts() == 0


def test_strides_and_shared_pages(cuda_device):
    """q and out as views of wider rows; two requests that read the same pages; a cache that is a slice of a larger one."""
    from prime_kernels_b200 import kv8

    g = torch.Generator().manual_seed(10)
    cache, scales, table, lens = filled(g, [64, 100], 3, 16, False, cuda_device)
    table = torch.stack([table[1], table[1]])
    lens = torch.tensor([64, 100], dtype=torch.int32)
    wide = torch.zeros(len(cache), 3, 16, 4 * D, dtype=torch.uint8, device=cuda_device)
    wide[..., D: 3 * D] = cache.view(torch.uint8)
    cache = wide.view(torch.float8_e4m3fn)[..., D: 3 * D]
    qkv = torch.randn(2, 15 * D, generator=g).bfloat16()
    q = qkv[:, : 9 * D].view(2, 9, D)
    want, wlse = run_attention(cuda_device, cache, scales, table, lens, q)
    qd = qkv.to(cuda_device)[:, : 9 * D].view(2, 9, D)
    buf = torch.full((2, 9, 2 * D), 5.0, dtype=torch.bfloat16, device=cuda_device)
    kv8.attention(qd, cache, scales, table.to(cuda_device), lens.to(cuda_device), out=buf[..., :D])
    assert torch.equal(buf[..., :D], want) and (buf[..., D:] == 5).all()


def test_offsets_past_32_bits(cuda_device):
    """A pool of more than 2^32 bytes: pages behind the border are stored and read where they are."""
    from prime_kernels_b200 import kv8

    pages = (1 << 32) // (32 * 16 * 128) + 40
    cache = torch.empty((pages, 32, 16, 128), dtype=torch.uint8, device=cuda_device).view(torch.float8_e4m3fn)
    scales = torch.zeros((pages, 32, 2), dtype=torch.uint8, device=cuda_device).view(torch.float8_e8m0fnu)
    g = torch.Generator().manual_seed(11)
    table = torch.tensor([[pages - 1, 3, pages - 30]], dtype=torch.int32)
    lens = torch.tensor([41], dtype=torch.int32)
    k, v = torch.randn(41, 32, D, generator=g).bfloat16(), torch.randn(41, 32, D, generator=g).bfloat16()
    cu = torch.tensor([0, 41], dtype=torch.int32)
    kv8.append(k.to(cuda_device), v.to(cuda_device), cache, scales, table.to(cuda_device), lens.to(cuda_device), cu.to(cuda_device))
    small = torch.stack([cache.view(torch.uint8)[p] for p in table[0].tolist()]).view(torch.float8_e4m3fn)
    se = torch.stack([scales.view(torch.uint8)[p] for p in table[0].tolist()]).view(torch.float8_e8m0fnu)
    held = Held(torch.zeros_like(small.view(torch.uint8)).view(torch.float8_e4m3fn), se)
    here = torch.tensor([[0, 1, 2]])
    held.e[:] = 0
    held.append(k, v, here.numpy(), lens.numpy(), cu.numpy())
    assert np.array_equal(held.e, Held(small, se).e)
    q = torch.randn(1, 32, D, generator=g).bfloat16()
    out = kv8.attention(q.to(cuda_device), cache, scales, table.to(cuda_device), lens.to(cuda_device))
    again = kv8.attention(q.to(cuda_device), small, se, here.int().to(cuda_device), lens.to(cuda_device))
    assert torch.equal(out, again)


def test_refusals(cuda_device):
    from prime_kernels_b200 import kv8

    cache, scales = kv8.empty_cache(4, 2, 16, device=cuda_device)
    table = torch.zeros(2, 2, dtype=torch.int32, device=cuda_device)
    lens = torch.ones(2, dtype=torch.int32, device=cuda_device)
    q = torch.zeros(2, 4, D, dtype=torch.bfloat16, device=cuda_device)
    k = torch.zeros(2, 2, D, dtype=torch.bfloat16, device=cuda_device)
    cu = torch.zeros(3, dtype=torch.int32, device=cuda_device)
    wide = torch.zeros(2, 4, 2 * D + 4, dtype=torch.bfloat16, device=cuda_device)
    kv8.attention(q, cache, scales, table, lens, cu)
    attend = [(q.half(), cache, scales, table, lens), (q[:, :3], cache, scales, table, lens), (q[:1], cache, scales, table, lens),
              (q[..., :32], cache, scales, table, lens), (wide[..., 4: 4 + D], cache, scales, table, lens), (q.transpose(0, 2), cache, scales, table, lens),
              (q, cache.float(), scales, table, lens), (q, cache[:, :, :, :64], scales, table, lens), (q, cache[:, :, :8], scales, table, lens),
              (q, cache, scales[:3], table, lens), (q, cache, scales.float(), table, lens), (q, cache, scales, table.long(), lens),
              (q, cache, scales, table[:1], lens), (q, cache, scales, table.t().contiguous().t(), lens), (q, cache, scales, table, lens.long()),
              (q, cache, scales, table, lens, cu[:2]), (q, cache, scales, table, lens, cu.long()), (q, cache, scales, table, lens.cpu()),
              (q, cache, scales, table.cpu(), lens), (q.cpu(), cache, scales, table, lens)]
    for args in attend:
        with pytest.raises(RuntimeError):
            kv8.attention(*args)
    with pytest.raises(RuntimeError):
        kv8.attention(q, cache, scales, table, lens, out=q[:1])
    with pytest.raises(RuntimeError):
        kv8.attention(q, cache, scales, table, lens, out=q.float())
    for a, b in ((k[:, :1], k), (k, k[:1]), (k.float(), k), (k, k.float()), (wide[:, :2, 4: 4 + D], k)):
        with pytest.raises(RuntimeError):
            kv8.append(a, b, cache, scales, table, lens)
    with pytest.raises(ValueError):
        kv8.empty_cache(4, 2, 24)


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("n,heads", [(1, 5), (5, 3), (300, 10)])
def test_graphs_and_streams(cuda_device, n, heads):
    """Append and attention captured twice and replayed with other lengths and pages, and beside each other on two streams."""
    from prime_kernels_b200 import kv8

    dev, size = cuda_device, 16
    g = torch.Generator().manual_seed(n + heads)
    seq = [n + 37, n + 250, n, 0 if n == 1 else n + 3]                     # a padded batch: the last decode row has no token
    table, pages = tables(g, [s + 100 for s in seq], size)
    x = torch.randn(4 * n, 5 * heads, D, generator=g).bfloat16().to(dev)
    q, k, v = x[:, : 3 * heads], x[:, 3 * heads: 4 * heads], x[:, 4 * heads:]
    cu = None if n == 1 else torch.arange(0, 4 * n + 1, n, dtype=torch.int32, device=dev)
    start = torch.randint(0, 127, (pages, heads, size, 2 * D), generator=g, dtype=torch.uint8)
    lens, bt = torch.tensor(seq, dtype=torch.int32, device=dev), table.to(dev)

    def held():
        cache, scales = kv8.empty_cache(pages, heads, size, device=dev)
        cache.view(torch.uint8).copy_(start)
        scales.view(torch.uint8).fill_(120)
        return cache, scales

    def both(cache, scales):
        kv8.append(k, v, cache, scales, bt, lens, cu)
        return kv8.attention(q, cache, scales, bt, lens, cu, max_query_len=n)

    def eager():
        cache, scales = held()
        return both(cache, scales), cache

    kept = [held() for _ in range(2)]
    both(*kept[0])
    graphs, outs = [], []
    for cache, scales in kept:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(both(cache, scales))
        graphs.append(graph)
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    for shift in (0, 20, -9):
        lens.copy_(torch.tensor([max(s + shift, 0) if s else 0 for s in seq], dtype=torch.int32))
        bt.copy_(table[:, torch.arange(table.shape[1])] if shift == 0 else table.flip(0))
        for cache, scales in kept:
            cache.view(torch.uint8).copy_(start)
            scales.view(torch.uint8).fill_(120)
        want, want_cache = eager()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for out, (cache, _) in zip(outs, kept):
            assert torch.equal(out.view(torch.int16), want.view(torch.int16))
            assert torch.equal(cache.view(torch.uint8), want_cache.view(torch.uint8))


def test_a_decode_loop_of_all_three(cuda_device):
    """Prompt chunk, then steps of append -> attention -> logits -> sample, eager and replayed from one CUDA graph on a side
    stream: the same ids; every step checked against the definition."""
    from prime_kernels_b200 import kv8
    from prime_kernels_b200 import sampling as S

    dev, batch, heads, group, vocab, steps = cuda_device, 3, 5, 3, 999, 20
    g = torch.Generator().manual_seed(12)
    emb = torch.randn(vocab, (heads * group + 2 * heads) * D, generator=g).bfloat16().to(dev)
    head = (torch.randn(heads * group * D, vocab, generator=g) * 0.1).bfloat16().to(dev)
    prompt = [20, 1, 33]
    uniform = torch.rand(steps, batch, generator=g).to(dev)
    table, pages = tables(g, [p + steps for p in prompt], 16)

    def rows(x):
        n = len(x)
        return (x[:, : heads * group * D].view(n, heads * group, D), x[:, heads * group * D: -heads * D].view(n, heads, D),
                x[:, -heads * D:].view(n, heads, D))

    def loop(graphed):
        cache, scales = pool(g, pages, heads, 16, False, dev)
        tab, lens = table.to(dev), torch.tensor(prompt, dtype=torch.int32, device=dev)
        cu = torch.tensor(np.concatenate([[0], np.cumsum(prompt)]), dtype=torch.int32, device=dev)
        _, k, v = rows(emb[torch.arange(sum(prompt)) % vocab])
        kv8.append(k, v, cache, scales, tab, lens, cu)
        ids, u = torch.arange(batch, device=dev), uniform[0].clone()
        out = torch.zeros(batch, heads * group, D, dtype=torch.bfloat16, device=dev)

        def step():
            lens.add_(1)
            q, k, v = rows(emb[ids])
            kv8.append(k, v, cache, scales, tab, lens)
            kv8.attention(q, cache, scales, tab, lens, out=out)
            S.sample(out.view(batch, -1) @ head, u, temperature=0.8, top_k=40, top_p=0.95, out=ids)

        seen = []
        if graphed:
            side, graph = torch.cuda.Stream(dev), torch.cuda.CUDAGraph()
            keep = [t.clone() for t in (cache.view(torch.uint8), scales.view(torch.uint8), lens, ids)]
            side.wait_stream(torch.cuda.current_stream(dev))
            with torch.cuda.stream(side):
                step()
                with torch.cuda.graph(graph, stream=side):
                    step()
                for t, old in zip((cache.view(torch.uint8), scales.view(torch.uint8), lens, ids), keep):
                    t.copy_(old)
                for i in range(steps):
                    u.copy_(uniform[i])
                    graph.replay()
                    seen.append(ids.clone())
            torch.cuda.current_stream(dev).wait_stream(side)
            return torch.stack(seen)
        for i in range(steps):
            u.copy_(uniform[i])
            fed = ids.clone()
            step()
            seen.append(ids.clone())
            if i % 7 == 0:
                q = rows(emb[fed])[0].cpu()
                want, _, tol, _, _ = attend64(q, Held(cache, scales), table.numpy(), lens.cpu().numpy(), np.arange(batch + 1), D ** -0.5)
                assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()
        return torch.stack(seen)

    eager = loop(False)
    assert torch.equal(eager, loop(True))
    assert len(eager.unique()) > 5
