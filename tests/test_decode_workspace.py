"""The workspace of a decode attention holds every part that a call may write: part range + sequence of each head, for any call of the handle.  No GPU."""
import ctypes as C

import pytest

from rustingbrain_amd import _lib as L


def internal(name, restype, *args):
    fn = getattr(L.load(), name)
    fn.restype, fn.argtypes = restype, [C.c_int32] * len(args)
    return fn(*args)


@pytest.mark.parametrize("kv_heads,group", [(1, 1), (2, 4), (8, 4), (1, 15), (1, 16), (1, 17), (3, 40), (1, 1024), (16, 64), (512, 2), (600, 1), (1024, 1), (33, 31)])
def test_parts_of_every_call_have_room(kv_heads, group):
    heads = kv_heads * group
    shared = 0
    for most in (1, 2, 7, 64, 511, 512, 513, 1023, 1024, 1025, 3000, 65535):
        room = internal("rbmoe_internal_decode_parts", C.c_int64, most, kv_heads, group)
        for n in {1, 2, 3, 64, 500, 512, 1000, 1023, 1024, 1025, most - 1, most}:
            if not 0 < n <= most:
                continue
            for longest in (1, 1024, 1025, 1100, 5000, 1 << 17, 1 << 30):
                ranges = internal("rbmoe_internal_decode_ranges", C.c_int, n, kv_heads, group, longest)
                if ranges <= 1:
                    continue  # one range, or a workgroup a sequence: rows are written whole
                shared += 1
                # the last part of the last range: range ranges - 1 within sequence n - 1
                assert (ranges - 1 + n - 1 + 1) * heads <= room, (most, n, longest, ranges)
    assert shared or kv_heads * -(-group // 16) > 256
