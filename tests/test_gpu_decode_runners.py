"""Several runners of one DecodeGraph object, and buffers that a runner is given later: every node works on
the buffers of the runner that runs it."""
import numpy as np
import pytest

import einsummable_amd as ea
from einsummable_amd.llama_layer import DeviceRunner
from helpers import assert_bits_equal, normal, rng
from serving_oracle import Paged
from test_gpu_decode_layer import DIM, HEADS, batch_inputs, graph_of, set_all, weights

pytestmark = pytest.mark.gpu

N_POS = 96
READ = ("values", "q.rotated", "cache.k", "cache.v")


def inputs(seed, group):
    b = Paged(seed, ea.F16, HEADS, 2, DIM // HEADS, 16, [1, 3, 1], [40, 33, 70], 32)
    vals = weights(seed, 2, N_POS, group)
    vals.update(batch_inputs(b))
    vals["x"] = normal(rng(seed + 1), (b.tokens, DIM), np.float16, 1.0)
    return b, vals


def result(run):
    import torch

    torch.cuda.synchronize()
    return [run.get(n, np.uint8).copy() for n in (run.g.output,) + READ]


def alone(km, b, vals, group):
    run = DeviceRunner(km, graph_of(b, N_POS, group, 2, 32))
    set_all(run, vals)
    run.run()
    return result(run)


def same(got, want, what):
    for g, w, name in zip(got, want, ("output",) + READ):
        assert_bits_equal(g, w, "%s: %s" % (what, name))


@pytest.mark.parametrize("group", [None, 64])
def test_two_runners_of_one_graph(km, group):
    import torch

    (b, vals), (b2, vals2) = inputs(5, group), inputs(6, group)
    want, want2 = alone(km, b, vals, group), alone(km, b2, vals2, group)
    g = graph_of(b, N_POS, group, 2, 32)
    first, second = DeviceRunner(km, g), DeviceRunner(km, g)
    set_all(first, vals)
    set_all(second, vals2)
    for _ in range(2):   # the appended positions are the same: a second run repeats the first
        first.run()
        same(result(first), want, "first")
        second.run()
        same(result(second), want2, "second")
    graphs = first.capture(), second.capture()
    for run, graph, w in ((first, graphs[0], want), (second, graphs[1], want2)):
        for name in (g.output,) + READ[:2]:
            run.mem[name].zero_()
        graph.replay()
        same(result(run), w, "captured")
    torch.cuda.synchronize()


def test_a_runner_leaves_the_graph_as_it_was(km):
    """The graph's nodes hold nothing of a runner."""
    b, vals = inputs(7, 64)
    g = graph_of(b, N_POS, 64, 2, 32)
    before = [dict(n) for n in g.nodes]
    DeviceRunner(km, g)
    assert [sorted(n) for n in g.nodes] == [sorted(n) for n in before]


def test_buffers_exchanged_after_construction(km):
    """A cache and activations that the runner gets later are the ones its next run uses."""
    import torch

    b, vals = inputs(8, 64)
    want = alone(km, b, vals, 64)
    run = DeviceRunner(km, graph_of(b, N_POS, 64, 2, 32))
    set_all(run, vals)
    kept = {n: run.mem[n] for n in READ + ("lens", "page_table", "wo.scales")}
    bytes_of = {n: t.clone() for n, t in kept.items()}
    for n in kept:
        run.mem[n] = kept[n].clone()
    run.run()
    same(result(run), want, "exchanged")
    torch.cuda.synchronize()
    for n, t in kept.items():
        assert torch.equal(t, bytes_of[n]), n
