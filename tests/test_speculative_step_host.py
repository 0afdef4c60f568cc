"""The speculative step's entry points without a device: null handles, and a
context that keeps its books on the host alone."""
import ctypes as C

import pytest

import slmkv


def test_null_handles_are_refused():
    lib = slmkv.lib()
    assert lib.slm_batch_append_layer_normed(None, 0, None, None, None, 0, 0, 0, None, None, 1e-5, 1,
                                             None) == slmkv.ERR_INVALID_INPUT
    assert lib.slm_batch_shared_attention(None, 0, None, 0, None) == slmkv.ERR_INVALID_INPUT
    assert lib.slm_batch_token_probabilities(None, None, 1, 1, 1, None, None) == slmkv.ERR_INVALID_INPUT
    assert lib.slm_batch_verify_drafts(None, 1, None, None, None, None, None, None) == slmkv.ERR_INVALID_INPUT
    assert lib.slm_pool_storage(None, None, None, None) == slmkv.ERR_INVALID_INPUT
    assert lib.slm_model_score(None, None, None, None, None) == slmkv.ERR_INVALID_INPUT


def test_a_pool_without_a_device_has_no_storage():
    pool = slmkv.KvPool(num_layers=1, num_query_heads=4, num_key_value_heads=2, context_length=64, num_blocks=8,
                        max_sequences=2, device=-1)
    a = [C.c_int64(-5) for _ in range(3)]
    assert slmkv.lib().slm_pool_storage(pool.handle, *map(C.byref, a)) == slmkv.ERR_NO_DEVICE
    assert [x.value for x in a] == [-5] * 3
    with pytest.raises(slmkv.EngineError):
        pool.storage()
