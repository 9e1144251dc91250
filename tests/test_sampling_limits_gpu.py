"""GPU: sampling with numbers beyond the kernel's own types."""
import math

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


FLAT = [100, 250, 256, 300, 777, 1000, 5000, 49152, 100003, 262144]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", FLAT)
@pytest.mark.parametrize("rows", [1, 160])
def test_draws_at_exact_borders(cuda_device, dtype, vocab, rows):
    """n equal tokens: the running sum behind token i is i + 1 of n, so u = a / 2^b draws floor(u n), to the token where
    u n is a whole number.  Whole numbers throughout, nothing is rounded."""
    from prime_kernels_b200 import sampling as S

    x = torch.full((1, vocab), 1.5, dtype=dtype, device=cuda_device).expand(rows, vocab)
    for top_k in (0, 64, 200, 400, 3000):
        n = min(top_k or vocab, vocab)
        for num, bits in ((1, 1), (1, 2), (3, 2), (5, 3), (11, 4), (63, 6), (1, 6), (2 ** 24 - 1, 24), (1, 24), (3, 40)):
            ids = S.sample(x, torch.full((rows,), num / 2 ** bits, device=cuda_device), top_k=top_k)
            assert ids.tolist() == [num * n >> bits] * rows, (top_k, num, bits)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", FLAT)
@pytest.mark.parametrize("rows", [1, 160])
def test_top_p_at_exact_borders(cuda_device, dtype, vocab, rows):
    """n equal tokens with top_p = a / 2^b: ceil(p n) of them stay, the ones that come first."""
    from prime_kernels_b200 import sampling as S

    x = torch.full((1, vocab), -0.25, dtype=dtype, device=cuda_device).expand(rows, vocab)
    u = torch.full((rows,), 1 - 2 ** -24, device=cuda_device)
    for top_k in (0, 64, 200, 400, 3000):
        n = min(top_k or vocab, vocab)
        for num, bits in ((1, 1), (1, 2), (3, 2), (7, 3), (61, 6), (1, 20)):
            stay = max(-(-num * n >> bits), 1)
            ids, lp = S.sample(x, u, top_k=top_k, top_p=num / 2 ** bits, return_logprobs=True)
            assert ids.tolist() == [stay - 1] * rows, (top_k, num, bits)
            assert (lp.double() + math.log(stay)).abs().max() <= 2 ** -23 * math.log(stay) + 1e-9
