"""GPU: the draw, the 4-bit products and the gradient norm as several users at once have them: first calls inside a capture, threads, graphs that
follow one another on memory of their own, lists of other kinds."""
import os
import subprocess
import sys
import threading

import pytest
import torch

import albatross_b200 as ab
from conftest import ROOT

pytestmark = pytest.mark.gpu

FIRST = """
import torch
import albatross_b200 as ab
g = torch.Generator(device="cuda").manual_seed(1)
rand = lambda *s: torch.randn(*s, device="cuda", generator=g)
x, u = rand(5, {V}).to(torch.{dtype}), torch.rand(5, device="cuda", generator=g)
w = ab.quantize_int4(rand(300, 1024), 64, True)
a, grads = rand(3, 1024).half(), [rand(1000, 7), rand(3).half()]
keep = [t.clone() for t in grads]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    drawn = [ab.sampler_batch(x, u, **f) for f in (dict(top_p=0.9), dict(top_k=20), dict(top_k=torch.full((5,), 20, device="cuda")), dict(min_p=0.1))]
    y = ab.linear_int4(a, *w)
    norm = ab.clip_grad_norm(grads, 0.5)
for _ in range(2):
    for t, k in zip(grads, keep):
        t.copy_(k)
    graph.replay()
torch.cuda.synchronize()
for (ids, logp), f in zip(drawn, (dict(top_p=0.9), dict(top_k=20), dict(top_k=20), dict(min_p=0.1))):
    i, p = ab.sampler_batch(x, u, **f)
    assert torch.equal(i, ids) and torch.allclose(p, logp, rtol=0, atol=4e-6)
assert torch.equal(ab.linear_int4(a, *w), y)
got = [t.clone() for t in grads]
assert torch.equal(ab.clip_grad_norm(keep, 0.5), norm) and all(torch.equal(s, t) for s, t in zip(keep, got))
print("FINE")
"""


@pytest.mark.parametrize("dtype,V", [("float16", 5000), ("float32", 70000)])
def test_the_first_calls_of_a_process_may_be_captured(dtype, V):
    res = subprocess.run([sys.executable, "-c", FIRST.format(dtype=dtype, V=V)], cwd=ROOT, env=dict(os.environ), capture_output=True, text=True, timeout=300)
    assert "FINE" in res.stdout, (res.stdout + res.stderr)[-2000:]


def inputs(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(20, 33001, device="cuda", generator=g) * 2
    u = torch.rand(20, device="cuda", generator=g)
    w = ab.quantize_int4(torch.randn(700, 2048, device="cuda", generator=g), 32, True)
    a = torch.randn(6, 2048, device="cuda", generator=g).half()
    grads = [torch.randn(n, device="cuda", generator=g) for n in (100, 5000, 77777)]
    k = 1 + torch.arange(20, device="cuda") * 3
    return x, u, w, a, grads, k


def calls(x, u, w, a, grads, k):
    out = [torch.empty_like(t) for t in grads]
    return [*ab.sampler_batch(x, u, top_p=0.9), *ab.sampler_batch(x, u, top_k=k), *ab.sampler_batch(x.half(), u, top_p=0.9), *ab.sampler_batch(x, u, top_k=50), ab.linear_int4(a, *w),
            ab.clip_grad_norm(grads, 0.3, out=out), *out]


def test_threads_on_streams_of_their_own():
    data = [inputs(s) for s in range(4)]
    want = [calls(*d) for d in data]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(25):
                    got = calls(*data[i])
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(s, t) for s, t in zip(got, want[i])):
                        wrong.append(i)
        except Exception as e:      # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:3]


def test_graphs_on_two_streams_at_once():
    data = [inputs(s) for s in (5, 6)]
    want = [calls(*d) for d in data]
    graphs, outs = [], []
    for d in data:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(calls(*d))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(10):
        for t in (*outs[0], *outs[1]):
            t.zero_()
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for got, w in zip(outs, want):
            assert all(torch.equal(s, t) for s, t in zip(got, w))


def test_lists_of_other_kinds():
    """A generator, a tuple, the rows of a tensor; the same gradient twice, into two places."""
    g = torch.randn(6, 50, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    want = float(g.double().norm())
    f = min(1.0, 0.5 / want)
    for kind in (lambda t: (r for r in t), tuple, lambda t: t):
        t = g.clone()
        assert float(ab.clip_grad_norm(kind(t), 0.5)) == pytest.approx(want, rel=1e-6) and torch.allclose(t, g * f, rtol=1e-6)
    two = [torch.empty_like(g), torch.empty_like(g)]
    norm = ab.clip_grad_norm([g, g], 0.5, out=two)
    assert float(norm) == pytest.approx(want * 2 ** 0.5, rel=1e-6) and torch.equal(two[0], two[1])
    for bad in (3, None, [None], [g, 1.0], [[g]]):
        with pytest.raises((RuntimeError, TypeError)):
            ab.clip_grad_norm(bad, 1.0)


def test_empty_batches_of_several_dimensions():
    for shape in ((0, 3, 40), (3, 0, 40)):
        ids, logp = ab.sampler_batch(torch.zeros(shape, device="cuda"), torch.zeros(shape[:-1], device="cuda"))
        assert ids.shape == logp.shape == (*shape[:-1], 1)
        m = ab.quantize_int4(torch.ones(8, 128, device="cuda"))
        assert ab.linear_int4(torch.zeros(*shape[:-1], 128, device="cuda", dtype=torch.float16), *m).shape == (*shape[:-1], 8)
