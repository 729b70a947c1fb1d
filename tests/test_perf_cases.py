"""The performance cases' own calls go to the stream that their inputs are made on (no GPU: streams and library are stand-ins)."""
import importlib.util
import os
import types

import pytest


class Stream:
    made = 0

    def __init__(self, handle=None):
        Stream.made += handle is None
        self.cuda_stream = 4096 + Stream.made if handle is None else handle
        self.waited = []

    def wait_stream(self, other):
        self.waited.append(other)


@pytest.fixture
def ops(monkeypatch):
    import torch  # (not where the GPU tests are collected: it brings a HIP runtime of its own)
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "operators.py")
    spec = importlib.util.spec_from_file_location("perf_operators", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.own, m.device = True, "cpu"
    m.now, m.calls = [Stream(0)], []
    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: m.now[-1])
    monkeypatch.setattr(torch.cuda, "set_stream", m.now.append)
    real = m._lib()

    def draco_kv_plan(args, stream):
        m.calls.append((stream, m.now[-1].cuda_stream))
        return 0
    fake = types.SimpleNamespace(KvPlan=real.KvPlan, load=lambda: types.SimpleNamespace(draco_kv_plan=draco_kv_plan), check=real.check)
    monkeypatch.setattr(m, "_lib", lambda: fake)
    return m


def test_the_loops_stream_is_the_current_one(ops):
    """Where the null stream is current, which the library takes for its own, the loop's stream becomes the current one, behind it."""
    null, case = ops.now[0], ops.listed()[0]
    inputs = ops._ints
    made_on = []
    ops._ints = lambda v: made_on.append(ops.now[-1].cuda_stream) or inputs(v)
    for seed in range(3):
        s = ops.prepare(case, seed)
        loop = ops.now[-1]
        assert loop.cuda_stream != 0 and null in loop.waited
        ops.run(s)
        ops.run(s)
    assert set(made_on) == {loop.cuda_stream}
    assert ops.calls == [(loop.cuda_stream, loop.cuda_stream)] * 6
    # another part of the program goes back to the null stream: the next inputs come behind its work
    ops.now.append(null)
    n = len(loop.waited)
    ops.run(ops.prepare(case, 9))
    assert ops.now[-1] is loop and len(loop.waited) == n + 1 and ops.calls[-1] == (loop.cuda_stream, loop.cuda_stream)


def test_a_stream_of_the_callers_is_used_as_it_is(ops):
    mine = Stream(77)
    ops.now.append(mine)
    ops.run(ops.prepare(ops.listed()[0], 1))
    assert ops.now[-1] is mine and ops.calls == [(77, 77)] and not mine.waited
