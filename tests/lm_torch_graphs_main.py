"""Graphs of the serving operators' calls on torch tensors, several at a time, in a process of its own: started by
test_gpu_lm_torch_graphs.py with the name of one check."""
import sys

import torch

from lm_torch_main import Step, same


def eager(*steps):
    out = []
    for s in steps:
        s.run()
        out.append(s.results())
    return out


def captured(s, **kw):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, **kw):
        s.run()
    return g


def check(s, want):
    same(s.results(), want)
    s.clear()


def order():
    """Two graphs captured one after the other on a stream that no call ran on before, the second replayed first."""
    a, b = Step(10), Step(11, long=2500, V=30011)
    wa, wb = eager(a, b)
    ga, gb = captured(a), captured(b)
    for _ in range(3):
        for s, g, want in ((b, gb, wb), (a, ga, wa), (a, ga, wa)):
            s.clear()
            g.replay()
            check(s, want)
            other = torch.randn(1 << 20, device="cuda")       # torch's own work between the replays
            assert torch.isfinite(other.sum())


def together():
    """Two graphs replayed on two streams at a time, and eager calls on the stream that they were captured on."""
    a, b, c = Step(12), Step(13, long=2800), Step(14, long=2600)
    wa, wb, wc = eager(a, b, c)
    cap, one, two = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.Stream()
    ga, gb = captured(a, stream=cap), captured(b, stream=cap)
    for _ in range(10):
        for s in (a, b, c):
            s.clear()
        torch.cuda.synchronize()
        for _ in range(20):
            with torch.cuda.stream(one):
                ga.replay()
            with torch.cuda.stream(two):
                gb.replay()
            with torch.cuda.stream(cap):
                c.run()
        for s, want in ((a, wa), (b, wb), (c, wc)):
            same(s.results(), want)


def given():
    """A stream that is captured but not torch's current one, given by its handle."""
    a = Step(15)
    want, = eager(a)
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        side.wait_stream(torch.cuda.current_stream())
        a.run(stream=side.cuda_stream)
        torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        a.clear()
        g.replay()
        check(a, want)
    a.run(stream=side.cuda_stream)
    check(a, want)


def grown():
    """A graph whose second call wants a larger workspace than its first, and a first eager call on the capture's stream
    after the capture."""
    a, b = Step(16, long=1500, V=17000), Step(17, long=6000, V=60011)
    wa, wb = eager(a, b)
    cap = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=cap):
        a.run()
        b.run()
        a.run()
    with torch.cuda.stream(cap):
        b.clear()
        b.run()
    check(b, wb)
    for _ in range(3):
        a.clear()
        b.clear()
        g.replay()
        check(a, wa)
        check(b, wb)


if __name__ == "__main__":
    globals()[sys.argv[1]]()
    torch.cuda.synchronize()
    print("ok", sys.argv[1], flush=True)
