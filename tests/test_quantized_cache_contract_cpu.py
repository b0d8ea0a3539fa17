"""What the C entry points of the 8-bit cache refuse of a `start` from the host, without and with lengths of padded calls."""
import ctypes

from qwen3_triton import _abi


def test_a_start_from_the_host_with_counts():
    lib = _abi.lib()
    fields = dict(keys=16, values=16, key_scales=16, value_scales=16, recent_keys=16, recent_values=16, marks=16, batch=2, heads=2,
                  capacity=100, head_dim=64, dtype=_abi.Q3_BF16)
    cache = ctypes.byref(_abi.QuantizedCacheView(*fields.values()))
    for s, start, counts in [(10, 91, None), (10, -1, 16), (10, 101, 16), (101, 0, 16), (10, 2 ** 62, 16), (2 ** 62, 2 ** 62, 16)]:
        assert lib.q3_qcache_append(cache, 16, 16, s, start, None, counts, None, None) == -2
        assert lib.q3_qcache_attention(cache, 16, 16, 16, 2 ** 40, s, 4, start, None, counts, 0.125, None, None) == -2
    # the workspace of such a call is that of the longest sequence
    long = dict(fields, capacity=10 ** 6)
    cache = ctypes.byref(_abi.QuantizedCacheView(*long.values()))
    need = lib.q3_qcache_attention_workspace_bytes
    assert need(cache, 16, 4, 10 ** 6 - 16) > 0
    assert need(cache, 16, 4, 10 ** 6 - 3) == need(cache, 16, 4, 10 ** 6 - 16)
    assert need(cache, 16, 4, 10 ** 6 + 1) == 0
