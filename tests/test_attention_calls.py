"""The attention operators' C ABI where no GPU is: calls without a handle, and the ranges that a decode call cuts its sequences into.  No GPU."""
import ctypes as C

import pytest

from rustingbrain_amd import TransformerBuilder, InvalidConfig
from rustingbrain_amd import _lib as L

NAMES = [n for n in L.SIGNATURES if n.startswith(("rbmoe_attention_", "rbmoe_kv_cache_", "rbmoe_decode_"))]


@pytest.mark.parametrize("name", NAMES)
def test_calls_without_a_handle(name):
    restype, argtypes = L.SIGNATURES[name]
    zero = [None if a in (C.c_void_p, C.POINTER(C.c_void_p)) else a(0) for a in argtypes]
    got = getattr(L.load(), name)(*zero)
    if restype is None:
        return  # destroying nothing
    assert got == L.NULL_POINTER
    assert L.load().rbmoe_last_global_error().decode()


def ranges(sequences, kv_heads, group, longest):
    fn = L.load().rbmoe_internal_decode_ranges
    fn.restype, fn.argtypes = C.c_int, [C.c_int32] * 4
    return fn(sequences, kv_heads, group, longest)


def test_ranges_of_a_decode_call():
    assert ranges(1, 2, 4, 1024) == 0 and ranges(1, 2, 4, 1025) > 1  # one workgroup a group of heads, or ranges
    assert ranges(1024, 8, 4, 4000) > 1 and ranges(1025, 8, 4, 4000) == 0
    for sequences in (1, 3, 64, 1000):
        for kv_heads, group in ((1, 1), (2, 4), (8, 4), (1, 40), (1024, 1)):
            for longest in (1025, 5000, 1 << 20, 1 << 30):
                n = ranges(sequences, kv_heads, group, longest)
                blocks = (group + 15) // 16
                # the workspace holds `n` + `sequences` parts of every head: so many are accounted for
                assert 1 <= n and n * kv_heads * group <= 512 * min(group, 16) or n == 1
                assert n * kv_heads * blocks <= 512 or n == 1


def test_the_builder_checks_its_heads_first():
    for build in ("build_attention", "build_caches", "build_decode_attention"):
        more = {"build_caches": dict(sequences=1), "build_decode_attention": dict(max_sequences=1)}.get(build, {})
        with pytest.raises(InvalidConfig, match="multiple"):
            getattr(TransformerBuilder().heads(8, 3, 64), build)(None, **more)
