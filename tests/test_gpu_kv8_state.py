"""What calls on one context share: its scratch and arrival counters, under graphs, on several streams, and the state of a
cache that works on a stream of its own."""
import numpy as np
import pytest
import torch

from aihost_b200.kv8 import Kv8Ops
from aihost_b200.ops import Context
from test_gpu_kv8 import DEV, I32, World

pytestmark = pytest.mark.gpu


@pytest.fixture
def own():
    """A context of this test's own: its scratch starts empty."""
    c = Context(0)
    yield c
    torch.cuda.synchronize()
    c.close()


def _args(w):
    return [w.dev(x, I32) for x in (w.start, w.kv_len, w.table)] + [w.dev(x) for x in (w.k, w.v, w.ks, w.vs)]


def test_a_captured_call_outlives_the_growth_of_the_scratch(own):
    """A captured decode step whose chunks are merged in the scratch, replayed after a longer prompt has made the scratch
    grow, and grow again: the replays still give the eager result, and write to nobody else's memory."""
    w = World(own, [3000, 40, 700], [1, 1, 1], D=128, P=64)
    q = w.rows(w.Hq)[0].to(DEV)
    args, out, side = _args(w), torch.empty_like(q), torch.cuda.Stream()
    want = w.ops.attend(q, *args, 1, 3001).clone()
    torch.cuda.synchronize()
    graph, ops = torch.cuda.CUDAGraph(), Kv8Ops(own, w.spec, side)
    with torch.cuda.graph(graph, stream=side):
        ops.attend(q, *args, 1, 3001, out=out)
    for new, bound in ((64, 20000), (64, 200000)):  # either needs more scratch than the call before it
        p = World(own, [2500], [new], D=128, P=64)
        pq = p.rows(p.Hq)[0].to(DEV)
        p.ops.attend(pq, *_args(p), new, bound)
        torch.cuda.synchronize()
        # memory that the growth may have given back, in other hands now
        others = [torch.full((1 << 20,), 7.0, device=DEV) for _ in range(64)]
        for _ in range(3):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
        assert all((x == 7.0).all() for x in others)
        assert torch.equal(w.ops.attend(q, *args, 1, 3001), want)
    own.sync_status()
