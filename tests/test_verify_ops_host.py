"""The cache, attention and log-probability calls on the CPU: argument checks that need no
device, and the Python wrappers' checks of shapes and strides."""
import ctypes

import pytest
import torch

import dflash_qmm


def cpu_cache(**kw):
    a = dict(slots=2, heads=2, capacity=8, head_dim=64, bits=4, group_size=32, device="cpu")
    a.update(kw)
    return dflash_qmm.KVCache(**a)


def test_calls_without_a_context_are_refused():
    lib = dflash_qmm.load_library()
    cache = cpu_cache()
    n = ctypes.c_size_t(7)
    assert lib.dfq_cache_append(None, cache.desc, None, None, 128, 1, 1, 0, None, None) == 1
    assert lib.dfq_cache_read(None, cache.desc, None, None, 0, 1, 1, 0, None, None) == 1
    assert lib.dfq_cache_attention(None, None, 0, cache.desc, None, 8, None, None, 256, None, None,
                                   1, 1, 4, 1.0, None, 0, None) == 1
    assert lib.dfq_cache_attention_workspace_bytes(None, None, 0, cache.desc, 8, 1, 1, 4,
                                                   ctypes.byref(n)) == 1 and n.value == 0
    assert lib.dfq_token_logprobs(None, None, 9, 1, 9, 0, None, 0, None, None, None, None, None, 0,
                                  None) == 1
    assert lib.dfq_token_logprobs_workspace_bytes(None, 1, 9, 0, None) == 1
    assert b"null" in lib.dfq_last_error()


def test_cache_shapes():
    cache = cpu_cache(head_dim=128, bits=8, group_size=64, dtype=torch.float16)
    assert cache.k[0].shape == (2, 2, 8, 32) and cache.v[2].shape == (2, 2, 8, 2)
    assert cache.head_dim == 128 and cache.dtype == torch.float16
    k, v = cache.k, cache.v
    again = dflash_qmm.KVCache.from_arrays(k, v, 8, 64)
    assert again._desc.k_codes == k[0].data_ptr() and again._desc.capacity == 8
    for bad in ((k[0][:1], k[1], k[2]), (k[0], k[1].bfloat16(), k[2]), (k[0], k[1], k[2][..., :1]),
                (k[0].transpose(0, 1), k[1], k[2])):
        with pytest.raises(ValueError):
            dflash_qmm.KVCache.from_arrays(bad, v, 8, 64)


def test_row_strides():
    x = torch.zeros(3, 4, 100)
    stride = dflash_qmm._row_stride
    assert stride(x) == 100 and stride(x[:, :, 7:50]) == 100
    assert stride(x[:1]) == 100 and stride(x[:, :1, :9]) == 400 and stride(x[:1, :1, :9]) == 9
    for bad in (x[:, :, ::2], x[:, :2], x.transpose(0, 1)):
        with pytest.raises(ValueError):
            stride(bad)
