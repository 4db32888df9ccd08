"""Workspaces of captured calls: a graph's own, never kept with the OpEnv, whose kept ones serve the
eager calls of their stream."""
import gc

import numpy as np
import pytest
import torch

from oracle.lans_f64 import LansHParams
from tests.helpers import lans_inputs

DEV = "cuda:0"


def test_a_captured_call_keeps_no_workspace(monkeypatch):
    """Without a GPU: under capture the chunk is torch's and new at every call; otherwise it is the memory
    pool's, once per stream."""
    from raf_amd import op

    class Env:
        workspace_bytes = 1000
        workspaces = {}

    made = []

    class Memory:
        def __init__(self, *args, **kw):
            made.append(args)
            self.data = 4096 * len(made)

    monkeypatch.setattr(op.runtime, "Memory", Memory)
    like, capturing = torch.zeros(3), False
    monkeypatch.setattr(op, "_capturing", lambda device: capturing)
    first = op._workspace(Env, like, 7)
    capturing = True
    chunks = [op._workspace(Env, like, s) for s in (7, 7, 8)]
    assert len({c.data for c in chunks}) == 3 and all(c.data != first.data for c in chunks)
    assert list(Env.workspaces) == [7] and len(made) == 1
    capturing = False
    assert op._workspace(Env, like, 7) is first and op._workspace(Env, like, 8).data == 8192
    assert list(Env.workspaces) == [7, 8]


def _to_dev(arrs):
    return [torch.from_numpy(np.ascontiguousarray(a)).to(DEV) for a in arrs]


@pytest.mark.gpu
def test_lans_captured_on_a_stream_that_has_no_workspace(native_libs, capfd):
    """The step is captured without a warm-up on the capture's stream; when the graph is gone, eager steps on
    that stream and the end of the OpEnv find nothing of it."""
    from raf_amd import op

    op.clear_op_env_cache()
    gc.collect()
    capfd.readouterr()
    sizes = [70001, 5, 8192, 1]
    g, w, m, v = lans_inputs(sizes, cfg=85)
    hp = LansHParams()
    args = (hp.learning_rate, hp.beta1, hp.beta2, hp.eps, hp.bias_correction, hp.weight_decay, hp.grad_averaging, hp.mode,
            hp.normalize_grad)
    one, two = op.TensorList(_to_dev(g + w + m + v)), op.TensorList(_to_dev(g + w + m + v))
    step = torch.ones((), device=DEV)
    op.lans(one, step, *args)  # the plan and its pointer table
    op.lans(two, step, *args)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        op.lans(one, step, *args)
    (env,) = op._env_cache.values()
    assert stream.cuda_stream not in env.workspaces
    step.fill_(2.0)
    graph.replay()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        op.lans(two, step, *args)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(one, two))
    del graph
    gc.collect()
    torch.cuda.empty_cache()
    step.fill_(3.0)
    op.lans(one, step, *args)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        op.lans(two, step, *args)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(one, two))
    del env
    op.clear_op_env_cache()
    gc.collect()
    torch.cuda.synchronize()
    assert "releasing memory failed" not in capfd.readouterr().err


@pytest.mark.gpu
def test_two_captured_norms_replayed_side_by_side(native_libs):
    """Both captured on one stream, replayed on two at once, over and over: neither sums into the other's
    partial sums."""
    from raf_amd import op

    n = 5_000_000
    xs = [torch.full((n,), float(k + 1), device=DEV) for k in range(2)]
    want = [float(k + 1) * np.sqrt(n) for k in range(2)]
    capture, graphs, outs = torch.cuda.Stream(), [], []
    with torch.cuda.stream(capture):
        op.l2norm(xs[0])
    torch.cuda.synchronize()
    for x in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=capture):
            outs.append(op.l2norm(x))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(50):
        for _ in range(4):
            for graph, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        for out, value in zip(outs, want):
            assert float(out) == pytest.approx(value, rel=1e-5)
