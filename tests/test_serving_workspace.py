"""What prefix_attention asks of its caller: room for partial results where there are any.  No device."""
import ctypes

import pytest

import einsummable_amd as ea

A = 1 << 20
OK, WORKSPACE = 0, -3


def need(dtype, heads, kv, dim, n_seqs, n_tokens, shared=0):
    lib, ws = ea.load_library(), ctypes.c_uint64()
    c = ea.KvCache(dtype, heads, kv, dim, 10, 16, A, A)
    assert lib.es_km_prefix_attention_workspace(None, c._at, n_seqs, n_tokens, shared,
                                                ctypes.addressof(ws)) == OK
    return ws.value


# at least 2048 workgroups of whole tiles: nothing is cut, results go straight to the output
@pytest.mark.parametrize("args", [
    (ea.F16, 32, 32, 128, 1, 16384), (ea.F16, 32, 32, 128, 1, 131072),
    (ea.F16, 32, 8, 128, 4, 32768), (ea.F16, 32, 32, 256, 2, 8192), (ea.F32, 32, 32, 128, 1, 4096),
    (ea.F16, 8, 8, 64, 1024, 1024)], ids=str)
def test_nothing_is_asked_where_nothing_is_joined(args):
    assert need(*args) == 0
    dtype, heads, kv, dim, n_seqs, n_tokens = args
    c = ea.KvCache(dtype, heads, kv, dim, 10, 16, A, A)
    b = ea.KvBatch(n_seqs, n_tokens, A, A, A, 4)
    width = heads * dim
    lib = ea.load_library()
    lib.es_km_prefix_attention(None, c._at, b._at, 0, 0.1, None, 2 * A, A, width, width, None, 0)
    assert lib.es_km_last_error(None) == b"null handle"


@pytest.mark.parametrize("args", [
    (ea.F16, 32, 32, 128, 1, 1), (ea.F16, 32, 32, 128, 1, 2048), (ea.F32, 32, 32, 128, 1, 1024),
    (ea.F16, 8, 8, 64, 1024, 1024, 64), (ea.F16, 8, 8, 64, 500, 500)], ids=str)
def test_parts_that_are_joined_have_room(args):
    heads, dim, n_tokens = args[1], args[3], args[5]
    # a row of the result, its reference and sum, and where its parts are
    assert need(*args) >= n_tokens * heads * (dim * 4 + 8 + 16)
