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
