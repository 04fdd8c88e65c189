"""Argument checks of the decoding operators that need no GPU."""
import ctypes

from tinygpt_b200 import _lib


def test_null_handles_and_arguments(cuda_lib):
    L = cuda_lib
    h = ctypes.c_void_p()
    cfg = _lib.CacheConfig(1, 1, 64, 16, 4, 2, 2, _lib.TG_DTYPE_BF16)
    pool = ctypes.c_void_p(4096)
    bad = _lib.TG_ERR_INVALID_ARG
    assert L.tg_cache_create(0, ctypes.byref(cfg), pool, pool, None) == bad
    assert L.tg_cache_create(0, None, pool, pool, ctypes.byref(h)) == bad
    assert L.tg_cache_create(0, ctypes.byref(cfg), None, pool, ctypes.byref(h)) == bad
    for field, value, code in (("layers", 0, bad), ("num_pages", -1, bad), ("head_dim", 68, _lib.TG_ERR_UNSUPPORTED),
                               ("head_dim", 256, _lib.TG_ERR_UNSUPPORTED), ("page_size", 24, _lib.TG_ERR_UNSUPPORTED),
                               ("dtype", _lib.TG_DTYPE_F32, _lib.TG_ERR_UNSUPPORTED), ("num_pages", 1 << 25, _lib.TG_ERR_UNSUPPORTED)):
        other = _lib.CacheConfig(1, 1, 64, 16, 4, 2, 2, _lib.TG_DTYPE_BF16)
        setattr(other, field, value)
        assert L.tg_cache_create(0, ctypes.byref(other), pool, pool, ctypes.byref(h)) == code, field
        assert not h.value
    assert L.tg_cache_create(0, ctypes.byref(cfg), ctypes.c_void_p(4104), pool, ctypes.byref(h)) == bad
    assert b"aligned" in L.tg_last_error_string()
    assert L.tg_cache_destroy(None) == _lib.TG_OK and L.tg_beam_destroy(None) == _lib.TG_OK
    assert L.tg_cache_extend(None, 1, None, None, None) == bad and b"cache is NULL" in L.tg_last_error_string()
    assert L.tg_cache_fork(None, 1, None, None, None) == bad
    assert L.tg_cache_truncate(None, 1, None, None, None) == bad
    assert L.tg_cache_commit(None, 1, None, None, None) == bad
    assert L.tg_cache_append(None, 0, 1, None, None, 1, None, 0, 0, 0, None, 0, 0, 0, None) == bad
    assert L.tg_cache_accept(None, 1, None, 1, None, None, None, None, None, None, None) == bad
    assert L.tg_cache_get_state(None, None) == bad and L.tg_cache_device_status(None, None) == bad
    assert L.tg_tree_attention(None, 0, 1, None, 1, None, None, 1, None, 0, 0, 0, None, 0, 0, 0, None, 0, 0, 0,
                               ctypes.c_float(1.0), None, None, None) == bad
    assert L.tg_tree_masks(1, 4, None, None, None, None) == bad
    assert L.tg_tree_masks(1, 65, None, None, None, None) == _lib.TG_ERR_UNSUPPORTED
    assert L.tg_tree_masks(0, 4, None, None, None, None) == _lib.TG_OK
    assert L.tg_beam_create(0, 100, 4, 1, None) == bad
    assert L.tg_beam_create(0, _lib.TG_MAX_VOCAB + 1, 4, 1, ctypes.byref(h)) == _lib.TG_ERR_UNSUPPORTED
    assert L.tg_beam_create(0, 100, 0, 1, ctypes.byref(h)) == _lib.TG_ERR_UNSUPPORTED
    assert L.tg_beam_create(0, 100, 32, 4000, ctypes.byref(h)) == _lib.TG_ERR_UNSUPPORTED
    assert L.tg_beam_select(None, None, 0, 0, 1, None, None, None, 0, None, -1, 0, None, None, 0, None, None, None, None,
                            None, None, None) == bad
    assert L.tg_beam_device_status(None, None) == bad


def test_config_layout():
    assert ctypes.sizeof(_lib.CacheConfig) == 32 and ctypes.sizeof(_lib.CacheState) == 32
