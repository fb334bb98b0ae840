"""The serving operators' checks of their arguments, which need no device: without a handle a call
gets its checks and, when they all pass, "null handle".  No pointer below is ever followed."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import einsummable_amd as ea
from einsummable_amd.llama_layer import DecodeGraph, quantize_int4
from serving_oracle import int4_pack

OK, UNSUPPORTED, INVALID, WORKSPACE = 0, 1, -1, -3
A = 1 << 20   # an address on a 256-byte boundary


def cache(**kw):
    a = dict(dtype=ea.F16, n_heads=8, n_kv_heads=2, head_dim=64, n_pages=10, page_size=16, k=A, v=A)
    strides = kw.pop("strides", None)
    a.update(kw)
    return ea.KvCache(**a, strides=strides)


def batch(**kw):
    a = dict(n_seqs=2, n_tokens=3, offsets=A, lens=A, page_table=A, max_pages=4)
    a.update(kw)
    return ea.KvBatch(**a)


def weight(**kw):
    a = dict(dtype=ea.F16, n=40, k=128, group=64, w=A, scales=A, zeros=0)
    a.update(kw)
    return ea.Int4Weight(**a)


def outcome(rc):
    return rc, ea.load_library().es_km_last_error(None).decode()


def append(c=None, b=None, q_out=A, q=A, k=A, v=A, strides=(512, 512, 128, 128),
           rope=ea.ROPE_PAIRS, freqs=A, n_pos=9):
    c, b = c or cache(), b or batch()
    return outcome(ea.load_library().es_km_kv_append(None, c._at, b._at, None, q_out, q, k, v,
                                                     *strides, rope, freqs, n_pos))


def attend(c=None, b=None, shared=0, scale=0.1, out=2 * A, q=A, strides=(512, 512), ws=A,
           ws_bytes=1 << 40):
    c, b = c or cache(), b or batch()
    return outcome(ea.load_library().es_km_prefix_attention(None, c._at, b._at, shared, scale,
                                                            None, out, q, *strides, ws, ws_bytes))


def linear(w=None, m=3, y=2 * A, x=A, strides=(40, 128), ws=None, ws_bytes=0):
    w = w or weight()
    return outcome(ea.load_library().es_km_int4_linear(None, w._at, m, None, y, x, *strides, ws,
                                                       ws_bytes))


def test_valid_calls_only_miss_the_handle():
    for rc, why in (append(), append(q=0, q_out=0), append(rope=ea.ROPE_NONE, freqs=0, n_pos=0),
                    append(q_out=A, strides=(512, 512, 128, 128)),
                    append(c=cache(dtype=ea.F32, n_heads=3, n_kv_heads=3, head_dim=8),
                           strides=(24, 24, 24, 24)),
                    append(b=batch(n_tokens=0), k=0, v=0, q=0, q_out=0),
                    attend(), attend(shared=1 << 20), attend(c=cache(dtype=ea.F32)),
                    linear(), linear(m=0, y=0, x=0), linear(w=weight(zeros=A)),
                    linear(w=weight(dtype=ea.F32), ws=A, ws_bytes=1 << 30)):
        assert rc == INVALID and why == "null handle", (rc, why)


BAD_CACHES = [
    (dict(n_heads=7), INVALID), (dict(n_kv_heads=0), INVALID), (dict(n_heads=0), INVALID),
    (dict(dtype=9), INVALID), (dict(dtype=-1), INVALID), (dict(dtype=ea.F64), UNSUPPORTED),
    (dict(dtype=ea.C64), UNSUPPORTED), (dict(head_dim=0), INVALID),
    (dict(head_dim=60), UNSUPPORTED), (dict(head_dim=264), UNSUPPORTED),
    (dict(page_size=0), INVALID), (dict(page_size=-4), INVALID), (dict(n_pages=0), INVALID),
    (dict(n_pages=1 << 31), INVALID), (dict(k=0), INVALID), (dict(v=0), INVALID),
    (dict(k=A + 8), INVALID), (dict(v=A + 2), INVALID), (dict(strides=(2048, 132, 64)), INVALID),
    (dict(strides=(1 << 40, 128, 64)), INVALID)]


@pytest.mark.parametrize("kw,code", BAD_CACHES, ids=[str(kw) for kw, _ in BAD_CACHES])
def test_bad_caches(kw, code):
    for rc, why in (append(c=cache(**kw)), attend(c=cache(**kw))):
        assert rc == code and why != "null handle" and why, (rc, why)


BAD_BATCHES = [dict(n_seqs=-1), dict(n_tokens=-1), dict(n_seqs=(1 << 20) + 1),
               dict(n_tokens=(1 << 22) + 1), dict(max_pages=0), dict(table_stride=3),
               dict(offsets=0), dict(lens=0), dict(page_table=0), dict(offsets=A + 2),
               dict(max_pages=(1 << 26) + 1)]


@pytest.mark.parametrize("kw", BAD_BATCHES, ids=str)
def test_bad_batches(kw):
    for rc, why in (append(b=batch(**kw)), attend(b=batch(**kw))):
        assert rc == INVALID and why != "null handle" and why, (rc, why)


@pytest.mark.parametrize("kw", [
    dict(q=0), dict(q_out=0), dict(k=0), dict(v=0), dict(k=A + 8), dict(q=A + 8), dict(v=A + 8),
    dict(q_out=A + 8), dict(rope=3), dict(rope=-1), dict(freqs=0), dict(n_pos=0),
    dict(freqs=A + 4), dict(rope=ea.ROPE_NONE), dict(n_pos=(1 << 31) + 1),
    dict(strides=(511, 512, 128, 128)), dict(strides=(512, 520, 128, 128)),
    dict(strides=(512, 512, 120, 128)), dict(strides=(512, 512, 128, 132)),
    dict(strides=(512, 512, 128, 1 << 41))], ids=str)
def test_bad_appends(kw):
    rc, why = append(**kw)
    assert rc == INVALID and why != "null handle" and why, (rc, why)


@pytest.mark.parametrize("kw,code", [
    (dict(q=0), INVALID), (dict(out=0), INVALID), (dict(q=A + 8), INVALID),
    (dict(out=2 * A + 8), INVALID), (dict(out=A), INVALID), (dict(strides=(512, 508)), INVALID),
    (dict(strides=(500, 512)), INVALID), (dict(scale=float("nan")), INVALID),
    (dict(scale=float("inf")), INVALID), (dict(shared=(1 << 30) + 1), INVALID),
    (dict(ws=0), WORKSPACE), (dict(ws_bytes=100), WORKSPACE), (dict(ws=A + 16), INVALID)], ids=str)
def test_bad_attentions(kw, code):
    rc, why = attend(**kw)
    assert rc == code and why != "null handle" and why, (rc, why)


@pytest.mark.parametrize("kw,code", [
    (dict(w=weight(dtype=ea.F64)), UNSUPPORTED), (dict(w=weight(dtype=ea.C64)), UNSUPPORTED),
    (dict(w=weight(dtype=7)), INVALID), (dict(w=weight(n=0)), INVALID),
    (dict(w=weight(k=0)), INVALID), (dict(w=weight(k=100)), UNSUPPORTED),
    (dict(w=weight(group=48)), UNSUPPORTED), (dict(w=weight(group=16)), UNSUPPORTED),
    (dict(w=weight(k=(1 << 20) + 32)), UNSUPPORTED), (dict(w=weight(w=0)), INVALID),
    (dict(w=weight(scales=0)), INVALID), (dict(w=weight(w=A + 8)), INVALID),
    (dict(w=weight(scales=A + 1)), INVALID), (dict(w=weight(w_stride=48)), INVALID),
    (dict(w=weight(w_stride=72)), INVALID), (dict(w=weight(scale_stride=1)), INVALID),
    (dict(m=65537), INVALID), (dict(x=0), INVALID), (dict(y=0), INVALID), (dict(x=A + 8), INVALID),
    (dict(y=A + 1), INVALID), (dict(y=A), INVALID), (dict(strides=(39, 128)), INVALID),
    (dict(strides=(40, 132)), INVALID), (dict(strides=(40, 120)), INVALID),
    (dict(w=weight(dtype=ea.F32)), WORKSPACE),
    (dict(w=weight(dtype=ea.F32), ws=A, ws_bytes=64), WORKSPACE),
    (dict(w=weight(dtype=ea.F32), ws=A + 4, ws_bytes=1 << 20), INVALID)],
    ids=lambda v: str(v) if isinstance(v, int) else str(sorted(v)))
def test_bad_products(kw, code):
    rc, why = linear(**kw)
    assert rc == code and why != "null handle" and why, (rc, why)


def test_null_descriptors():
    lib, ws = ea.load_library(), ctypes.c_uint64()
    at = ctypes.addressof(ws)
    c, b, w = cache(), batch(), weight()
    assert lib.es_km_kv_append(None, None, b._at, None, A, A, A, A, 0, 0, 0, 0, 0, 0, 0) == INVALID
    assert lib.es_km_kv_append(None, c._at, None, None, A, A, A, A, 0, 0, 0, 0, 0, 0, 0) == INVALID
    assert lib.es_km_prefix_attention(None, c._at, None, 0, 1.0, None, A, A, 0, 0, A, 0) == INVALID
    assert lib.es_km_int4_linear(None, None, 1, None, A, A, 0, 0, None, 0) == INVALID
    assert lib.es_km_prefix_attention_workspace(None, None, 1, 1, 0, at) == INVALID
    assert lib.es_km_prefix_attention_workspace(None, c._at, 1, 1, 0, None) == INVALID
    assert lib.es_km_prefix_attention_workspace(None, c._at, -1, 1, 0, at) == INVALID
    assert lib.es_km_int4_linear_workspace(None, None, 1, at) == INVALID
    assert lib.es_km_int4_linear_workspace(None, w._at, 1, None) == INVALID
    assert lib.es_km_int4_linear_workspace(None, w._at, 1 << 17, at) == INVALID


def test_workspaces():
    lib, ws = ea.load_library(), ctypes.c_uint64()
    at = ctypes.addressof(ws)
    w16, w32 = weight(), weight(dtype=ea.F32)
    assert lib.es_km_int4_linear_workspace(None, w16._at, 5, at) == OK and ws.value == 0
    assert lib.es_km_int4_linear_workspace(None, w32._at, 5, at) == OK
    assert ws.value >= 5 * 3 * 128 * 2 + 5 * 4
    c = cache()
    assert lib.es_km_prefix_attention_workspace(None, c._at, 0, 0, 0, at) == OK and ws.value == 0
    sizes = []
    for tokens in (1, 64, 4096):
        assert lib.es_km_prefix_attention_workspace(None, c._at, min(tokens, 64), tokens, 512,
                                                    at) == OK
        # at least one partial result per row of the shared part
        assert ws.value >= tokens * 8 * 64 * 4
        sizes.append(ws.value)
    assert sizes == sorted(sizes)


@pytest.mark.parametrize("heads,kv,seqs,tokens", [
    (64, 64, 1 << 20, 1 << 20),     # rows that the join's launch does not hold
    (65536, 1, 1, 1 << 22),         # nor 32 bits
    (32, 32, 1 << 20, 1 << 20)])    # a tile per sequence and head
def test_batches_beyond_a_launch_are_refused(heads, kv, seqs, tokens):
    lib, ws = ea.load_library(), ctypes.c_uint64()
    c = cache(n_heads=heads, n_kv_heads=kv)
    assert lib.es_km_prefix_attention_workspace(None, c._at, seqs, tokens, 0,
                                                ctypes.addressof(ws)) == INVALID
    assert b"than a launch holds" in lib.es_km_last_error(None)
    assert lib.es_km_prefix_attention_workspace(None, c._at, 1 << 8, 1 << 8, 0,
                                                ctypes.addressof(ws)) == OK


# ------------------------------------------------------------------------------ C++ and the layer

def test_cxx_members_compile(tmp_path):
    """The header's members take what the C entries take."""
    src = tmp_path / "serving.cc"
    src.write_text("""
#include "es_km.hpp"
void step(eskm::kernel_manager_t const& km, es_km_kv_cache_t const& c, es_km_kv_batch_t const& b,
          es_km_int4_weight_t const& w, void* p)
{
    km.kv_append(c, b, nullptr, p, p, p, p, 8, 8, 8, 8);
    km.kv_append(c, b, nullptr, nullptr, nullptr, p, p, 0, 0, 8, 8, ES_KM_ROPE_PAIRS, p, 16);
    uint64_t const n = km.prefix_attention_workspace(c, 1, 1, 64);
    km.prefix_attention(c, b, 64, 0.5f, nullptr, p, p, 8, 8, std::make_tuple(p, n));
    km.prefix_attention(c, b, 0, 0.5f, nullptr, p, p, 8, 8);
    uint64_t const m = km.int4_linear_workspace(w, 1);
    km.int4_linear(w, 1, nullptr, p, p, 8, 32, std::make_tuple(p, m));
    km.int4_linear(w, 1, nullptr, p, p, 8, 32);
}
""")
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["g++", "-std=c++17", "-fsyntax-only", "-Wall", "-Werror", "-I", include,
                    str(src)], check=True)


@pytest.mark.parametrize("k,group", [(64, 32), (160, 64), (96, 128)])
def test_quantize_int4(k, group):
    """Within half a step of the weight (and what rounding the step to f16 moves the 15 steps:
    15 * 2^-11), zero kept exactly, ranges without zero and empty ones included."""
    r = np.random.RandomState(k)
    w = r.normal(0, 1, (6, k)).astype(np.float32)
    w[1] = np.abs(w[1]) + 1
    w[2] = -np.abs(w[2])
    w[3] = 0
    w[4, ::3] = 0
    packed, scales, zeros = quantize_int4(w, group)
    assert packed.dtype == zeros.dtype == np.uint8 and scales.dtype == np.float16
    assert packed.shape == (6, k // 2) and scales.shape == zeros.shape == (6, -(-k // group))
    q = np.stack([packed & 15, packed >> 4], -1).reshape(6, k)
    assert np.array_equal(int4_pack(q), packed)
    of = np.arange(k) // group
    step = scales.astype(np.float64)[:, of]
    back = (q - zeros.astype(np.float64)[:, of]) * step
    assert (np.abs(back - w) <= step * (0.5 + 15 * 2.0 ** -11 + 2.0 ** -20)).all()
    assert not back[w == 0].any()


def test_decode_graph_inputs():
    g = DecodeGraph(5, 3, 11, 16, 4, 64, dim=256, n_heads=4, n_kv_heads=2, ffn=352, int4_group=64)
    assert g.inputs["wk.q"] == ("u8", (128, 128)) and g.buffers["wk.q"] == 128 * 128
    assert g.inputs["w2.scales"] == (ea.F16, (256, 6)) and g.inputs["w2.zeros"] == ("u8", (256, 6))
    assert g.inputs["cache.k"] == (ea.F16, (11, 16, 2, 64))
    assert g.buffers["page_table"] == 3 * 4 * 4 and g.buffers["offsets"] == 16
    kinds = [n["kind"] for n in g.nodes]
    assert kinds.count("int4_linear") == 7
    assert kinds.index("kv_append") < kinds.index("prefix_attention")
    dense = DecodeGraph(1, 1, 2, 16, 2, 64, dim=256, n_heads=4, ffn=352)
    assert dense.inputs["wk"] == (ea.F16, (256, 256))
    assert "int4_linear" not in [n["kind"] for n in dense.nodes]
