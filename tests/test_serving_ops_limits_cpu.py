"""CPU: refusals at the C entries of the 8-bit cache and of sampling (no device is touched)."""
import pytest
from test_serving_ops_cpu import P, append, attend, cache, sample


@pytest.mark.parametrize("name", ["block_table", "seq_lens", "cu_seqlens"])
@pytest.mark.parametrize("off", [1, 2])
def test_cache_arrays_are_aligned(name, off):
    """int32 arrays that the kernels read word by word."""
    assert append(cache(**{name: (1 << 18) + off})) == 9107
    assert attend(cache(**{name: (1 << 18) + off})) == 9107


@pytest.mark.parametrize("name", ["uniform", "temperature", "top_k", "top_p", "min_p", "logprobs"])
@pytest.mark.parametrize("off", [1, 2])
def test_sample_arrays_are_aligned(name, off):
    assert sample(**{name: P + off}) == 9107


def test_lengths_next_to_32_bits_are_refused():
    """The kernels look up to 32 steps of 64 keys ahead of a row's last key: a table that ends within that of 2^31 would
    wrap the index of a page.  The same for rows (tokens x query heads of a kv head), of which a tile more is counted."""
    most = 2 ** 31 - 2 ** 16
    for size in (16, 256):
        for cols in (most // size + 1, (2 ** 31 - size) // size):
            assert append(cache(page_size=size, bt_cols=cols)) == 9102
            assert attend(cache(page_size=size, bt_cols=cols)) == 9102
        # the longest that is taken: refused for its tokens, not its length
        assert append(cache(page_size=size, bt_cols=most // size), tokens=-1) == 9111
        assert attend(cache(page_size=size, bt_cols=most // size), heads=5) == 9111
    cu = dict(cu_seqlens=1 << 18, kv_heads=1)
    assert attend(cache(**cu), tokens=2 ** 25, heads=64, longest=1) == 9111
    assert attend(cache(**cu), tokens=2 ** 30 - 255, heads=1, longest=1) == 9111
