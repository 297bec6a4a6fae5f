"""The attention operators give the same bits from the same call whatever lies in the outputs, the cache's places and the handles' workspaces before it:
everything is overwritten between the calls, and calls of other shapes go through the same handles."""
import numpy as np

import pytest

from test_gpu_attention import Ints
from test_gpu_attention_calls import Step, same
from test_gpu_graph import Capture, hip  # noqa: F401  (a fixture)
from test_gpu_join import Array

pytestmark = pytest.mark.gpu


class Disturbed(Step):
    """A step whose outputs hold 0xA5 and whose handles have served other calls."""

    def __init__(self, device, seed=3):
        super().__init__(device, seed)
        p = self.p
        self.other_rows = [Ints(device, v) for v in ([0], [p.rows], [5, 90], [80, 250])]
        self.other = {n: Array(device, a.shape, a.dtype) for n, a in (("out", self.out), ("lse", self.lse), ("new", self.new))}
        self.other_grads = [Array(device, a.shape, a.dtype) for a in self.grads]
        self.other_tables = Ints(device, np.arange(200)[::-1].reshape(2, 100))
        self.other_lengths = Ints(device, [3, 1599])

    def outputs(self):
        return [self.out, self.lse, *self.grads, *self.back, self.new]

    def disturb(self):
        p, o = self.p, self.other
        q, k, v = p.inputs()
        self.device.synchronize()
        for begin, count, n in ((self.other_rows[0], self.other_rows[1], 1), (self.other_rows[2], self.other_rows[3], 2)):
            where = {**p.where(), "query_begin_ptr": begin.ptr, "query_count_ptr": count.ptr, "longest_queries": p.rows, "longest_keys": p.rows, "scale": 0.7}
            p.op.forward_device(n, q, k, v, o["out"].ptr, lse_ptr=o["lse"].ptr, **where)
            p.op.backward_device(n, q, k, v, o["out"].ptr, o["lse"].ptr, p.dgo.ptr, *(g.ptr for g in self.other_grads), **where)
        self.cache.write_device(p.rows, p.dv.ptr, p.dk.ptr, self.slots.ptr)  # (other rows in the step's places)
        self.decode.forward_device(self.cache, 2, q, o["new"].ptr, self.other_tables.ptr, 100, self.other_lengths.ptr, longest=1600)
        self.decode.forward_device(self.cache, 1, q, o["new"].ptr, self.other_tables.ptr, 100, self.other_lengths.ptr, longest=40)
        self.device.synchronize()
        for a in self.outputs():
            a.buf.upload(np.full(a.buf.nbytes, 0xA5, np.uint8))


def test_the_same_call_again(device):
    s = Disturbed(device)
    s.run()
    want = s.results()
    assert all(np.isfinite(a).all() for a in want)
    for _ in range(2):
        s.disturb()
        s.run()
        assert same(s.results(), want)


def test_replays_write_everything_again(device, hip):  # noqa: F811
    eager, captured = Disturbed(device), Disturbed(device)
    cap = Capture(hip, device, captured.run)
    device.set_stream(None)
    eager.run()
    want = eager.results()
    for _ in range(3):
        device.set_stream(None)
        captured.disturb()
        cap.replay()
        assert same(captured.results(), want)
    cap.close()
