"""What calls on one context share: its scratch and arrival counters, under graphs, on several streams, and the state of a
cache that works on a stream of its own."""
import numpy as np
import pytest
import torch

from aihost_b200 import ROPE_NONE
from aihost_b200.kv8 import Kv8Cache, Kv8Ops, Kv8Spec, StepMap
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


def _busy(stream, ms=3):
    """Keeps a stream at work for some milliseconds, so that what follows on it runs late."""
    with torch.cuda.stream(stream):
        torch.cuda._sleep(int(ms * 2_000_000))


def test_attention_on_several_streams_of_one_context(own):
    """Calls of different chunk counts, enqueued on three streams at once, merge their chunks in one scratch with one
    set of counters: each gives what it gives alone, and so does a call on a single stream afterwards."""
    worlds = [World(own, [3000, 40, 700], [1, 1, 1], D=128, P=64), World(own, [9000] * 8, [1] * 8, D=128, P=128, H=4, Hq=32),
              World(own, [2500], [64], D=64, P=16)]
    bounds = [(1, 3001), (1, 9001), (64, 20000)]
    calls = []
    for w, (new, most) in zip(worlds, bounds):
        q, args = w.rows(w.Hq)[0].to(DEV), _args(w)
        calls.append((w, (q, *args, new, most), w.ops.attend(q, *args, new, most).clone()))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for turn in range(6):
        got = []
        for i, (w, args, _) in enumerate(calls):
            _busy(streams[(i + turn) % 3])
        for _ in range(3):
            for i, (w, args, want) in enumerate(calls):
                ops = Kv8Ops(own, w.spec, streams[(i + turn) % 3])
                got.append((ops.attend(*args), want))
        torch.cuda.synchronize()
        assert all(torch.equal(x, want) for x, want in got)
    for w, args, want in calls:
        assert torch.equal(w.ops.attend(*args), want)
    own.sync_status()


def test_page_maps_on_several_streams_of_one_context(own):
    """Maps of several blocks that write their lengths in place, on two streams at once."""
    P, batch, T = 16, 700, 30000
    g = np.random.default_rng(0)
    t = lambda x, dt=I32: torch.tensor(x, dtype=dt, device=DEV)  # noqa: E731
    streams, states = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        n_pages = 6000
        ops = Kv8Ops(own, Kv8Spec(8, 2, 64, P, n_pages, 40), s)
        states.append((ops, t([0] * batch), t(list(range(n_pages))), t([n_pages]), t([[-1] * 40] * batch), [0] * batch,
                       torch.zeros(T, dtype=torch.int64, device=DEV), t([0] * T), t([0] * (batch + 1))))
    torch.cuda.synchronize()
    for turn in range(5):
        news = [g.integers(0, 30, batch).tolist() for _ in states]
        dev = [t(n) for n in news]
        torch.cuda.synchronize()
        for (ops, lens, stack, count, table, host, slots, pos, start), n in zip(states, dev):
            for _ in range(4):
                ops.map_pages(lens, n, stack, count, table, T, into=StepMap(lens, start, slots, pos, count))
        torch.cuda.synchronize()
        for i, n in enumerate(news):
            state = states[i]
            state[5][:] = [c + 4 * x for c, x in zip(state[5], n)]
            assert state[1].tolist() == state[5]
            assert state[3].item() == 6000 - sum(-(-c // P) for c in state[5])
            for b, c in enumerate(state[5]):
                state[5][b] = 0
            state[0].release_pages(t([1] * batch), state[1], state[2], state[3], state[4])
            torch.cuda.synchronize()
            assert state[3].item() == 6000 and sorted(state[2].tolist()) == list(range(6000))
    own.sync_status()


def test_a_cache_on_a_stream_of_its_own_needs_no_wait(own):
    """A cache made and used on a side stream while the current stream is busy gives what one on the current stream
    gives, also with tensors of the current stream coming and going in between."""
    B, H, Hq, D, P, steps = 5, 2, 8, 64, 16, 12
    spec = Kv8Spec(Hq, H, D, P, 60, 8, rope_mode=ROPE_NONE)
    new = [torch.tensor([(3 * i + b) % 4 for b in range(B)], dtype=I32, device=DEV) for i in range(steps)]
    g = torch.Generator().manual_seed(5)
    rows = [[torch.randn(16, h, D, generator=g).half().to(DEV) for h in (Hq, H, H)] for _ in range(steps)]
    want = []

    def run(cache, got):
        for n, (q, k, v) in zip(new, rows):
            m = cache.begin(n, 16)
            cache.append(0, k, v)
            got.append((cache.attend(0, q, 4, 128), m))
            cache.end()
            for _ in range(4):  # where a tensor that the step let go would be handed out again
                torch.full((B,), -7, dtype=I32, device=DEV)
                torch.full((1,), -7, dtype=I32, device=DEV)

    run(Kv8Cache(own, spec, B), want)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for late in (torch.cuda.current_stream(), side):
        got = []
        _busy(late, 20)
        cache = Kv8Cache(own, spec, B, stream=side)
        run(cache, got)
        torch.cuda.synchronize()
        for (a, m), (b, n) in zip(got, want):
            T = n.row_start[-1].item()
            assert T and all(torch.equal(x, y) for x, y in zip(m, n)) and torch.equal(a[:T], b[:T])
    own.sync_status()
