"""The decoder layer over a paged cache: apply nodes and serving operators together, eager and as
HIP graphs, against the 64-bit oracles node by node and against the layer on whole sequences."""
import numpy as np
import pytest

import einsummable_amd as ea
import oracle
from einsummable_amd.llama_layer import (DecodeGraph, DeviceRunner, LayerGraph, freqs_cis_table,
                                         quantize_int4)
from helpers import NP, assert_bits_equal, assert_close, normal, rng
from serving_oracle import Paged, assert_within, attention64, int4_64, rotate64, rotate_bound

pytestmark = pytest.mark.gpu

DIM, HEADS, FFN = 256, 4, 352
WEIGHTS = {"wq": "d", "wk": "kv", "wv": "kv", "wo": "d", "w1": "f", "w3": "f", "w2": "d"}


def weights(seed, n_kv, n_pos, group):
    r = rng(seed)
    rows = {"d": DIM, "kv": n_kv * (DIM // HEADS), "f": FFN}
    vals = {"full_freqs_cis": freqs_cis_table(n_pos, DIM // HEADS // 2)}
    for name in ("attention_norm.weight", "ffn_norm.weight"):
        vals[name] = (1.0 + normal(r, DIM, np.float32, 0.02)).astype(np.float16)
    for name, n in WEIGHTS.items():
        w = normal(r, (rows[n], FFN if name == "w2" else DIM), np.float16, 0.05)
        if group is None:
            vals[name] = w
        else:
            vals[name + ".q"], vals[name + ".scales"], vals[name + ".zeros"] = \
                quantize_int4(w.astype(np.float32), group)
    return vals


def graph_of(b, n_pos, group, n_kv, shared):
    return DecodeGraph(b.tokens, b.n_seqs, b.n_pages, b.page, b.table.shape[1], n_pos, shared,
                       dim=DIM, n_heads=HEADS, n_kv_heads=n_kv, ffn=FFN, int4_group=group,
                       scale=(DIM // HEADS) ** -0.5)


def batch_inputs(b):
    return {"cache.k": b.k, "cache.v": b.v, "offsets": b.offsets,
            "lens": np.asarray(b.lens, np.int32), "page_table": b.table}


def set_all(run, vals):
    for name, v in vals.items():
        run.set_input(name, v)


def f16(run, name, *shape):
    return run.get(name, np.float16).reshape(*shape)


def check_append(run, n, b, freqs):
    hd, x = DIM // HEADS, n["inns"]
    q, k, v = (f16(run, name, b.tokens, -1, hd) for name in x)
    got_q = f16(run, n["out"], b.tokens, HEADS, hd)
    kc, vc = f16(run, "cache.k", *b.k.shape), f16(run, "cache.v", *b.v.shape)
    for s in range(b.n_seqs):
        rows = np.arange(b.offsets[s], b.offsets[s + 1])
        if rows.size == 0:
            continue
        pos = b.lens[s] - (b.offsets[s + 1] - rows)
        for got, x in ((got_q[rows], q[rows]), (b.rows(kc, s, pos), k[rows])):
            want = rotate64(x, freqs[pos], ea.ROPE_PAIRS)
            assert_within(got, want, rotate_bound(x, want, ea.F16, ea.ROPE_PAIRS), "append")
        assert_bits_equal(b.rows(vc, s, pos), v[rows], "cache.v")


def check_nodes(run, b, vals):
    """Every node against its oracle on what the device read."""
    g, used = run.g, slice(0, b.used)
    for n in g.nodes:
        label = n["label"]
        if n["kind"] == "einsummable":
            od, dts = oracle.scalarop_info(n["e"].join)
            ins = [run.get(x, NP[dt]) for x, dt in zip(n["inns"], dts)]
            e = n["e"]
            want = oracle.einsummable(e.join_shape, e.inns, e.out_rank, e.join, e.castable, ins,
                                      oracle.WIDE)
            assert_close(run.get(n["out"], NP[od]), want, od, what=label)
        elif n["kind"] == "touch":
            assert_bits_equal(run.get(n["out"], np.uint8), run.get(n["inn"], np.uint8), label)
        elif n["kind"] == "kv_append":
            check_append(run, n, b, vals["full_freqs_cis"])
        elif n["kind"] == "prefix_attention":
            now = f16(run, "cache.k", *b.k.shape), f16(run, "cache.v", *b.v.shape)
            (b.k, b.v), old = now, (b.k, b.v)
            hd = DIM // HEADS
            want, bound = attention64(b, f16(run, n["inn"], b.tokens, HEADS, hd), g.scale)
            b.k, b.v = old
            assert_within(f16(run, n["out"], b.tokens, HEADS, hd)[used], want[used], bound[used],
                          label)
        else:
            m, n_out, n_in = n["shape"]
            packed, scales, zeros = (vals[x] for x in n["w"])
            q = np.stack([packed & 15, packed >> 4], -1).reshape(n_out, n_in)
            want, bound = int4_64(q, scales, zeros, f16(run, n["inn"], m, n_in), n["group"], ea.F16)
            assert_within(f16(run, n["out"], m, n_out), want, bound, label)


@pytest.mark.parametrize("group,n_kv", [(None, 4), (None, 2), (32, 4), (128, 1)])
@pytest.mark.parametrize("new,lens,shared", [
    ([1], [37], 0),                                  # one token
    ([1, 1, 1, 1, 1], [90, 71, 64, 65, 130], 64),    # a step of a batch behind a prefix
    ([20, 0, 7], [20, 11, 30], 0)])                  # prompts, one sequence waiting
def test_decode_layer_node_by_node(km, group, n_kv, new, lens, shared):
    import torch

    n_pos = 160
    b = Paged(5, ea.F16, HEADS, n_kv, DIM // HEADS, 16, new, lens, shared)
    vals = weights(3, n_kv, n_pos, group)
    vals.update(batch_inputs(b))
    vals["x"] = normal(rng(4), (b.tokens, DIM), np.float16, 1.0)
    run = DeviceRunner(km, graph_of(b, n_pos, group, n_kv, shared))
    set_all(run, vals)
    run.run()
    torch.cuda.synchronize()
    check_nodes(run, b, vals)


def test_padded_batch_keeps_the_cache_and_its_rows(km):
    """Rows behind the last sequence belong to nobody: the operators over the cache leave their
    outputs and the cache as they were."""
    import torch

    b = Paged(6, ea.F16, HEADS, 2, DIM // HEADS, 16, [1, 2], [33, 47], 0, tokens=8)
    vals = weights(3, 2, 64, 64)
    vals.update(batch_inputs(b))
    vals["x"] = normal(rng(4), (b.tokens, DIM), np.float16, 1.0)
    run = DeviceRunner(km, graph_of(b, 64, 64, 2, 0))
    set_all(run, vals)
    for name in ("q.rotated", "values"):
        run.mem[name].fill_(0x3c)
    run.run()
    torch.cuda.synchronize()
    for name in ("q.rotated", "values"):
        assert (run.get(name, np.uint8).reshape(8, -1)[3:] == 0x3c).all(), name
    written = np.zeros(b.k.shape[:2], bool)
    for s in range(2):
        pos = np.arange(b.lens[s] - b.new[s], b.lens[s])
        written[b.table[s][pos // 16], pos % 16] = True
    for name, before in (("cache.k", b.k), ("cache.v", b.v)):
        assert_bits_equal(f16(run, name, *before.shape)[~written], before[~written], name)


def test_prompt_then_tokens_match_the_layer_on_the_whole_sequence(km):
    """A prompt in one call and the rest token by token give what the layer gives for the sequence
    at once.  The whole layer rounds its scores to f16 and this one does not; scores are below 4
    here, so weights differ by 4 * 2^-11, inside the contract of f16 tensors."""
    import torch

    seq, prompt, page = 48, 41, 8
    whole = LayerGraph(dim=DIM, n_heads=HEADS, ffn=FFN, seq=seq)
    vals = weights(8, HEADS, 2 * seq, None)
    x = normal(rng(9), (seq, DIM), np.float16, 1.0)
    ref = DeviceRunner(km, whole)
    set_all(ref, dict(vals, x=x))
    ref.run()
    torch.cuda.synchronize()
    want = ref.get(whole.output, np.float16).reshape(seq, DIM)

    def step(n, mem):
        g = DecodeGraph(n, 1, 8, page, 8, 2 * seq, dim=DIM, n_heads=HEADS, ffn=FFN)
        return DeviceRunner(km, g, mem)

    first = step(prompt, None)
    kept = [name for name in first.g.inputs if name not in ("x", "offsets", "lens")]
    single = step(1, {name: first.mem[name] for name in kept})
    set_all(first, vals)
    table = np.random.RandomState(1).permutation(8).astype(np.int32)
    first.set_input("page_table", table)
    first.mem["cache.k"].fill_(0xff)   # NaN wherever nothing was appended
    first.mem["cache.v"].fill_(0xff)
    for run, n in ((first, prompt), (single, 1)):
        run.set_input("offsets", np.array([0, n], np.int32))
    at = 0
    while at < seq:
        run, n = (first, prompt) if at == 0 else (single, 1)
        run.set_input("x", x[at:at + n])
        run.set_input("lens", np.array([at + n], np.int32))
        run.run()
        torch.cuda.synchronize()
        got = run.get(run.g.output, np.float16).reshape(n, DIM)
        assert_close(got, want[at:at + n], ea.F16, what="tokens from %d" % at)
        at += n


def test_captured_steps_follow_lengths_and_tables(km):
    """Two steps of different sizes, captured once each over one cache and one workspace, replayed
    in turn with fresh tokens, lengths and tables, eager work in between: the bytes of eager runs."""
    import torch

    n_pos, group = 128, 32
    vals = weights(11, 2, n_pos, group)
    r = rng(12)
    cases = [([1, 1, 1], [50, 33, 70], 32), ([4, 1], [36, 80], 0)]
    batches = [Paged(13, ea.F16, HEADS, 2, DIM // HEADS, 16, new, [n_pos] * len(new), shared)
               for new, lens, shared in cases]
    pages = max(b.n_pages for b in batches)
    first = None
    runs = []
    for b, (new, lens, shared) in zip(batches, cases):
        b.n_pages = pages
        g = graph_of(b, n_pos, group, 2, shared)
        kept = [] if first is None else [n for n in g.inputs if n.startswith(("w", "cache"))]
        run = DeviceRunner(km, g, {n: first.mem[n] for n in kept})
        if first is None:
            first = run
        set_all(run, {n: v for n, v in vals.items() if n in g.inputs and n not in kept})
        run.set_input("offsets", b.offsets)
        run.set_input("page_table", b.table)
        run.set_input("lens", np.asarray(lens, np.int32))
        run.mem["x"].zero_()
        runs.append(run)
    shape = (pages, 16, 2, DIM // HEADS)
    cache = [normal(r, shape, np.float16, 1.0) for _ in range(2)]
    big = max((run.workspace for run in runs), key=lambda w: w.numel())
    for run in runs:
        run.workspace = big
    first.set_input("cache.k", cache[0])
    first.set_input("cache.v", cache[1])
    graphs = [run.capture() for run in runs]
    for turn in range(6):
        run, graph, (new, lens, shared) = [(x[turn % 2]) for x in (runs, graphs, cases)]
        b = batches[turn % 2]
        run.set_input("x", normal(r, (b.tokens, DIM), np.float16, 1.0))
        lens = np.asarray(lens, np.int32) + 3 * turn
        run.set_input("lens", lens)
        table = b.table.copy()
        common = shared // 16   # the pages behind the prefix change places
        for s in range(b.n_seqs):
            table[s, common:-1] = np.roll(table[s, common:-1], turn)
        run.set_input("page_table", table)
        got = []
        for go in (run.run, graph.replay):
            first.set_input("cache.k", cache[0])
            first.set_input("cache.v", cache[1])
            run.mem[run.g.output].zero_()
            torch.cuda.synchronize()
            go()
            torch.cuda.synchronize()
            got.append([run.get(n, np.uint8).copy()
                        for n in (run.g.output, "values", "cache.k", "cache.v")])
        for a, c in zip(*got):
            assert_bits_equal(a, c, "turn %d" % turn)
        assert np.isfinite(got[0][0].view(np.float16)).all()
        cache = [got[0][2].view(np.float16).reshape(shape), got[0][3].view(np.float16).reshape(shape)]
