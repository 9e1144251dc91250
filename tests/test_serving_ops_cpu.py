"""CPU: refusals and fake kernels of the 8-bit cache and of sampling (no device is touched)."""
import ctypes

import pytest
import torch

from prime_kernels_b200 import _cabi


def cache(**kw):
    base = dict(cache=1 << 20, scales=1 << 16, k_off=0, v_off=64, page_stride=4096, token_stride=128, head_stride=2048, pages=8,
                page_size=16, kv_heads=2, block_table=1 << 18, bt_stride=4, bt_cols=4, seq_lens=1 << 19, cu_seqlens=None, batch=2)
    return _cabi.PkKv8Cache(**{**base, **kw})


P = 1 << 22


def append(c, k=P, v=P, strides=(128, 64, 128, 64), tokens=2):
    return _cabi.library().pk_kv8_append(ctypes.byref(c), k, strides[0], strides[1], v, strides[2], strides[3], tokens, None)


def attend(c, q=P, out=P, strides=(256, 64, 256, 64), lse=None, tokens=2, heads=4, longest=0):
    return _cabi.library().pk_kv8_attention(ctypes.byref(c), q, strides[0], strides[1], out, strides[2], strides[3], lse, tokens,
                                            heads, longest, 0.125, None)


@pytest.mark.parametrize("kw,status", [
    ({"page_size": 8}, 9109), ({"page_size": 24}, 9109), ({"page_size": 512}, 9109), ({"kv_heads": 0}, 9111),
    ({"batch": -1}, 9111), ({"batch": 65536}, 9111), ({"pages": -1}, 9111), ({"bt_cols": 1 << 28}, 9102), ({"cache": None}, 9103),
    ({"scales": None}, 9103), ({"seq_lens": None}, 9103), ({"block_table": None}, 9103), ({"cache": (1 << 20) + 8}, 9107),
    ({"v_off": 8}, 9107), ({"token_stride": 72}, 9107), ({"head_stride": 2056}, 9107), ({"page_stride": 4100}, 9107),
    ({"batch": 3}, 9111)])
def test_cache_descriptions_are_checked(kw, status):
    assert append(cache(**kw)) == status
    assert attend(cache(**kw)) == status


def test_rows_are_checked():
    assert append(cache(), k=None) == 9103 and append(cache(), v=None) == 9103
    assert append(cache(), k=P + 8) == 9107 and append(cache(), strides=(128, 60, 128, 64)) == 9107
    assert append(cache(), tokens=-1) == 9111
    assert attend(cache(), q=None) == 9103 and attend(cache(), out=None) == 9103
    assert attend(cache(), out=P + 2) == 9107 and attend(cache(), lse=P + 2) == 9107
    assert attend(cache(), heads=5) == 9111 and attend(cache(), heads=0) == 9111 and attend(cache(), longest=-1) == 9111
    # nothing to do is no error and reaches no device
    assert append(cache(batch=0)) == 0 and append(cache(), tokens=0) == 0
    assert attend(cache(batch=0)) == 0 and attend(cache(), tokens=0) == 0
    assert _cabi.library().pk_kv8_append(None, P, 64, 64, P, 64, 64, 1, None) == 9103


def sample(**kw):
    base = dict(stream=None, logits=P, row_stride=100, rows=2, vocab=100, dtype=0, uniform=P, temperature=None, top_k=None,
                top_p=None, min_p=None, temperature_value=1.0, top_k_value=0, top_p_value=1.0, min_p_value=0.0, ids=P, logprobs=None)
    return _cabi.library().pk_sample(ctypes.byref(_cabi.PkSampleArgs(**{**base, **kw})))


def test_sample_arguments_are_checked():
    assert sample(rows=-1) == 9111 and sample(vocab=0) == 9111 and sample(vocab=262145) == 9111 and sample(dtype=3) == 9111
    assert sample(logits=None) == 9103 and sample(uniform=None) == 9103 and sample(ids=None) == 9103
    assert sample(logits=P + 1) == 9107 and sample(ids=P + 4) == 9107
    assert sample(rows=0, logits=None) == 0
    assert _cabi.library().pk_sample(None) == 9103


def test_settings_are_checked_before_the_device():
    from prime_kernels_b200 import sampling as S

    x, u = torch.zeros(2, 16), torch.zeros(2)
    for kw in ({"temperature": -1.0}, {"temperature": float("nan")}, {"top_k": -1}, {"top_p": 0.0}, {"top_p": 1.01}, {"min_p": 1.5}):
        with pytest.raises(ValueError):
            S.sample(x, u, **kw)
        with pytest.raises(ValueError):
            S.Sampler(**kw)
    with pytest.raises(NotImplementedError):            # no CPU fallback
        S.sample(x, u)


def test_fake_kernels():
    from prime_kernels_b200 import kv8
    from prime_kernels_b200 import sampling as S

    x, u = torch.empty(3, 1000, dtype=torch.bfloat16, device="meta"), torch.empty(3, device="meta")
    ids, lp = S.sample(x, u, return_logprobs=True)
    assert ids.shape == lp.shape == (3,) and ids.dtype == torch.int64 and lp.dtype == torch.float32
    q = torch.empty(5, 15, 64, dtype=torch.bfloat16, device="meta")
    c, s = kv8.empty_cache(4, 5, 16, device="meta")
    t, n = torch.empty(5, 4, dtype=torch.int32, device="meta"), torch.empty(5, dtype=torch.int32, device="meta")
    out, lse = kv8.attention(q, c, s, t, n, return_lse=True)
    assert out.shape == q.shape and out.dtype == torch.bfloat16 and lse.shape == (5, 15)
    kv8.append(q[:, :5], q[:, 5:10], c, s, t, n)


def test_dequantise_of_both_layouts():
    from prime_kernels_b200 import kv8

    for planes in (False, True):
        c, s = kv8.empty_cache(2, 3, 16, planes=planes, device="cpu")
        c.view(torch.uint8).fill_(0x38)                 # 1.0
        s.view(torch.uint8).copy_(torch.arange(12, dtype=torch.uint8).view(2, 3, 2) + 120)
        d = kv8.dequantise(c, s)
        want = torch.exp2(torch.arange(12.0).view(2, 3, 2) - 7)
        for h in range(3):
            for i in range(2):
                got = d[i, 1, :, h] if planes else d[1, h, :, 64 * i: 64 * i + 64]
                assert (got == want[1, h, i]).all()
