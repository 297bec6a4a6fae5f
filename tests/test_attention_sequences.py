"""Which rows and keys of a sequence an attention call finds inside its arrays, whatever the begins and counts are: those that the sequence names and the
arrays have, each row with the keys that it would see if all were there.  No GPU."""
import ctypes as C
import itertools
import random

import pytest

from rustingbrain_amd import _lib as L


def found(*args):
    fn = L.load().rbmoe_internal_attention_sequence
    fn.restype, fn.argtypes = None, [C.c_int32] * 8 + [C.POINTER(C.c_int32)]
    out = (C.c_int32 * 5)()
    fn(*args, out)
    return list(out)


def limit(r, nk, ahead):  # of causal rows, as the kernels form it in 32 bits
    assert -2 ** 31 <= r + ahead + 1 < 2 ** 31
    return min(max(r + ahead + 1, 0), nk)


def check(query_begin, query_count, key_begin, key_count, query_rows, key_rows, longest_queries, longest_keys):
    args = (query_begin, query_count, key_begin, key_count, query_rows, key_rows, longest_queries, longest_keys)
    nq, nk = min(max(query_count, 0), longest_queries), min(max(key_count, 0), longest_keys)
    there = lambda begin, n, rows: range(max(begin, 0), max(max(begin, 0), min(begin + n, rows)))  # noqa: E731
    queries, keys = there(query_begin, nq, query_rows), there(key_begin, nk, key_rows)
    q0, got_q, k0, got_k, ahead = found(*args)
    assert (got_q, got_k) == (len(queries), len(keys)), args
    assert 0 <= q0 <= query_rows - got_q and 0 <= k0 <= key_rows - got_k, args
    assert (got_q == 0 or q0 == queries[0]) and (got_k == 0 or k0 == keys[0]), args
    for row in {queries[0], queries[len(queries) // 2], queries[-1]} if got_q > 50 else queries:
        last = key_begin + (row - query_begin) + nk - nq  # the last key that this row sees, where it is there
        assert limit(row - q0, got_k, ahead) == min(max(last + 1 - keys.start, 0), got_k), (args, row)


def test_small_sequences_all_ways():
    for args in itertools.product((-3, 0, 2, 5), (-1, 0, 1, 4), (-2, 0, 3), (0, 2, 5), (0, 3, 6), (2, 6), (2, 6), (1, 6)):
        check(*args)


@pytest.mark.parametrize("args,want", [
    ((-5, 10, -5, 10, 50, 50, 10, 10), [0, 5, 0, 5, 0]),    # five rows in front of the arrays: rows 0 .. 4, not 0 .. 9
    ((40, 20, 0, 20, 50, 50, 20, 20), [40, 10, 0, 20, 0]),  # ten rows behind the queries' array: the others see what they saw
    ((0, 20, -8, 20, 50, 50, 20, 20), [0, 20, 0, 12, -8]),  # eight keys in front of theirs
])
def test_rows_and_keys_that_are_not_there(args, want):
    assert found(*args) == want
    check(*args)


def test_largest_numbers():
    rng = random.Random(1)
    numbers = [-2 ** 31, -2 ** 31 + 1, -2 ** 30, -1, 0, 1, 7, 2 ** 30 - 1, 2 ** 30, 2 ** 31 - 1]
    counts = [0, 1, 100, 2 ** 30 - 1, 2 ** 30]
    for _ in range(20000):
        check(*(rng.choice(numbers) for _ in range(4)), rng.choice(counts), rng.choice(counts), rng.choice(counts + [2 ** 31 - 1]),
              rng.choice(counts + [2 ** 31 - 1]))
