"""GPU: sampling with numbers beyond the kernel's own types."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("top_k", [-1, -(2 ** 31) - 1, -(2 ** 32) + 1, -(2 ** 63), 2 ** 32 + 1, 2 ** 63 - 1])
def test_top_k_beyond_32_bits(cuda_device, top_k):
    """The operator takes 64 bits, the kernel 32: below 0 is off and above the vocabulary everything stays, as far as numbers go."""
    import prime_kernels_b200.sampling  # noqa: F401  (registers the operator)

    x = torch.zeros(3, 100, device=cuda_device)
    u = torch.tensor([0.105, 0.505, 0.905], device=cuda_device)
    ids = torch.ops.prime_sampling.sample(x, u, None, 1.0, None, top_k, None, 1.0, None, 0.0)
    assert ids.tolist() == [10, 50, 90]
