"""A cache whose keys and values share memory is refused by sltx_kv_append, which would
write both to the same places: on the CPU, with pointers that are never read."""
import ctypes

import pytest

K, SIZE = 0x1000000, 2 * 3 * 2 * 256 * 64 * 2     # bytes of k: layers, batch, heads, slots, head_dim
FAR = 0x4000000000


def _append(pkg, v):
    c = pkg.CKVCache(k=K, v=v, length=FAR, next_position=FAR, layers=2, batch=3, kv_heads=2, capacity=256, head_dim=64,
                     dtype=0)
    strides = (ctypes.c_int64 * 3)(1024, 256, 64)
    return pkg.lib().sltx_kv_append(2 * FAR, strides, 2 * FAR, strides, 2 * FAR, strides, ctypes.byref(c), 0, 4, 4, FAR, 32,
                                    0, None, 3 * FAR, None)


@pytest.mark.parametrize("v", [K, K + SIZE - 16, K - SIZE + 16, K + 1024])
def test_shared_keys_and_values(pkg, v):
    assert _append(pkg, v) == -1
    assert "k and v of the cache overlap" in pkg.last_error()
