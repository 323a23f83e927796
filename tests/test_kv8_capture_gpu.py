"""GPU: rope, the int8 cache and attention recorded into CUDA graphs.  A replay gives what a direct call gives,
whatever was called since the recording, and recording leaves nothing half done for direct calls."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import kv8_plain as P

pytestmark = pytest.mark.gpu

CASES = [  # q_heads, heads, dim, page, new, length, window
    (8, 8, 64, 16, [1], [90], 0),                          # one block per head
    (8, 2, 128, 64, [1, 1, 3], [9000, 64, 5000], 0),       # streamed, keys divided
    (8, 2, 128, 64, [60], [9000], 0),                      # tiled, keys divided
    (48, 1, 128, 64, [140], [900], 0),                     # key tiles made before
    (8, 2, 64, 32, [1, 200, 4, 1], [9000, 200, 700, 3], 0),   # both kernels
    (12, 4, 64, 32, [1, 300, 9], [5000, 2000, 700], 333)]


class Step:
    def __init__(self, acf, case, seed):
        self.acf, (self.hq, heads, dim, page, new, length, self.window) = acf, case
        self.b = P.Batch(acf, new, length, page, seed=seed)
        self.cache = P.random_cache(acf, self.b.pages, heads, dim, page, seed + 1)
        self.state = (self.cache.k, self.cache.v, self.cache.k_scale, self.cache.v_scale)
        self.spec = acf.Rope(torch.from_numpy(acf.rope_frequencies(dim)[0]).cuda())
        self.kv = torch.empty((self.b.tokens, 2, heads, dim), dtype=torch.bfloat16, device="cuda")
        self.q = torch.empty((self.b.tokens, self.hq, dim), dtype=torch.bfloat16, device="cuda")
        self.pos = torch.cat([torch.arange(n - k, n, dtype=torch.int32) for k, n in zip(new, length)]).cuda()
        self.turned, self.out = torch.empty_like(self.q), torch.empty_like(self.q)
        self.lse = torch.empty((self.b.tokens, self.hq), device="cuda")

    def fill(self, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.kv.copy_(torch.randn(self.kv.shape, generator=g, device="cuda"))
        self.q.copy_(torch.randn(self.q.shape, generator=g, device="cuda"))
        for t in self.state[:2]:
            t.copy_(torch.randint(-127, 128, t.shape, generator=g, device="cuda"))
        for t in self.state[2:]:
            t.fill_(0.01)
        self.out.fill_(7.0), self.lse.fill_(7.0)

    def __call__(self):
        self.acf.rope(self.q, self.pos, self.spec, out=self.turned)
        self.cache.append(self.kv[:, 0], self.kv[:, 1], self.b.h, rope=self.spec)
        self.cache.attention(self.turned, self.b.h, window=self.window, out=self.out, lse=self.lse)
        return self.cache.read(self.b.h, torch.float16)

    def results(self, read):
        torch.cuda.synchronize()
        return [t.clone() for t in (self.turned, self.out, self.lse, *read, *self.state)]


def on(acf, stream, f):
    acf.lib().acfun_set_stream(stream)
    try:
        return f()
    finally:
        acf.lib().acfun_set_stream(None)


def record(acf, f):
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        got = on(acf, stream.cuda_stream, f)
    return graph, got


@pytest.mark.parametrize("case", CASES, ids=str)
def test_replays_equal_direct_calls(acf, case):
    s = Step(acf, case, 101)
    want = []
    for seed in (1, 2):
        s.fill(seed)
        want.append(s.results(s()))
    acf.synchronize()
    graph, read = record(acf, s)
    for seed in (1, 2, 1):
        s.fill(seed)
        torch.cuda.synchronize()
        graph.replay()
        for x, y in zip(s.results(read), want[seed - 1]):
            assert torch.equal(x, y)
        # direct calls in between that make the library's scratch grow and move
        big = Step(acf, (32, 8, 128, 64, [1] * 3 + [200] * seed, [40000 * seed] * 3 + [300] * seed, 0), 103)
        big.fill(3)
        for _ in range(2):
            big()
        acf.synchronize()
        del big
    s.fill(2)
    for x, y in zip(s.results(s()), want[1]):
        assert torch.equal(x, y)
    acf.synchronize()


def test_two_graphs_replayed_side_by_side(acf):
    steps = [Step(acf, CASES[i], 105 + i) for i in (1, 4)]
    want = []
    for i, s in enumerate(steps):
        s.fill(i)
        want.append(s.results(s()))
    graphs = [record(acf, s) for s in steps]
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(5):
        for i, s in enumerate(steps):
            s.fill(i)
        torch.cuda.synchronize()
        for (graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for s, (_, read), w in zip(steps, graphs, want):
            for x, y in zip(s.results(read), w):
                assert torch.equal(x, y)
    acf.synchronize()


def test_host_memory_is_refused_while_recording(acf):
    s = Step(acf, CASES[0], 107)
    s.fill(1)
    s()
    acf.synchronize()
    hb = acf.KvBatch(s.b.table.numpy(), np.array(s.b.start, np.int32), np.array(s.b.length, np.int32), s.b.tokens, 1, 90)
    refusals = []

    def calls():
        for f in (lambda: acf.rope(s.q, s.pos.cpu(), s.spec, out=s.turned), lambda: s.cache.attention(s.q, hb, out=s.out)):
            with pytest.raises(acf.AcfunError, match="host memory"):
                f()
            refusals.append(f)
        s()

    pos = s.pos.cpu()
    s.pos.cpu = lambda: pos
    graph, _ = record(acf, calls)
    assert len(refusals) == 2
    graph.replay()           # what was recorded beside the refused calls
    torch.cuda.synchronize()
    assert torch.isfinite(s.out).all()


def test_recording_before_any_direct_call_of_attention():
    """What attention sets up at its first call must not be left to the graph."""
    here = os.path.dirname(os.path.abspath(__file__))
    code = (f"import sys; sys.path[:0] = [{os.path.dirname(here)!r}, {here!r}]\n"
            "import torch, acfun_b200 as acf, test_kv8_capture_gpu as t\n"
            "acf.rope(torch.zeros((1, 1, 8), device='cuda'), torch.zeros(1, dtype=torch.int32, device='cuda'), acf.Rope(torch.ones(4, device='cuda')))\n"
            "acf.synchronize()\n"
            "s = t.Step(acf, t.CASES[1], 109)\n"
            "graph, read = t.record(acf, s)\n"
            "s.fill(1); direct = s.results(s())\n"
            "s.fill(1); torch.cuda.synchronize(); graph.replay(); replayed = s.results(read)\n"
            "acf.synchronize()\n"
            "assert all(torch.equal(x, y) for x, y in zip(direct, replayed))\n"
            "t.P.check_attention(s.out, s.lse, t.P.attention64(s.cache, s.b, s.turned, 128 ** -0.5, True, 0), 'bf16')\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
