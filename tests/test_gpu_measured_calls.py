"""The measured cases' calls of the library from programs that never synchronise: inputs still being made, results read at
once, results dropped while they are read.  The delays are longer than the calls, so a missing wait would show."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CASES = [
    {"op": "xent", "train": True, "n": 40, "v": 700, "d": 64},
    {"op": "distill", "t": "f16", "n": 30, "v": 3000, "k": 9, "tau": 2.0},
    {"op": "router", "t": "f32", "n": 500, "e": 24, "k": 3},
]
INPUT = {"xent": "x", "distill": "s", "router": "r"}
DELAY = 20_000_000                                     # clocks, about 10 ms


@pytest.fixture(scope="module")
def ops():
    spec = importlib.util.spec_from_file_location("measured_operators", os.path.join(ROOT, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.own = True
    yield m
    import gc
    gc.collect()
    if m._ctx is not None:
        m._ctx.close()


def expected(ops, state):
    import torch
    torch.cuda.synchronize()
    out = [o.clone() for o in ops.run(state)]
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("case", CASES, ids=lambda c: c["op"])
@pytest.mark.parametrize("side", [False, True])
def test_inputs_still_being_made_and_results_read_at_once(ops, case, side):
    import torch
    state = ops.prepare(case, 1)
    want = expected(ops, state)
    x = state[INPUT[case["op"]]]
    kept = x.clone()
    x.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream() if side else torch.cuda.current_stream()):
        torch.cuda._sleep(DELAY)
        x.copy_(kept)
        got = [o.clone() for o in ops.run(state)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("case", CASES, ids=lambda c: c["op"])
def test_results_dropped_while_they_are_read(ops, case):
    import torch
    state, other = ops.prepare(case, 1), ops.prepare(case, 2)
    want = expected(ops, state)
    out = ops.run(state)
    torch.cuda._sleep(DELAY)
    got = [o.clone() for o in out]
    del out
    for _ in range(3):
        ops.run(other)                                 # has the same blocks of the pool
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
