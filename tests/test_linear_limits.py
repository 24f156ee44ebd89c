"""Sizes beyond what a launch can have, and gradients written over what is still read, are refused
as such, before anything is enqueued.

Every call here is refused: the addresses belong to nothing.
"""
import pytest

from avelang_amd import _native

P = [(i + 1) << 42 for i in range(16)]


@pytest.mark.parametrize("rows,D,dt", [(1 << 28, 8, 1), ((1 << 28) - 15, 128, 2), (1 << 28, 64, 0),
                                       (1 << 27, 256, 1), (1 << 26, 2048, 1), (1 << 24, 4096, 1),
                                       ((1 << 24) + 1, 20001, 0)])
def test_norm_rows(rows, D, dt):
    lib = _native.lib()
    assert lib.gdn_layer_norm_fwd(P[0], None, None, P[1], None, rows, 1, D, 1e-5, dt, 0, None) == -2
    assert "too large" in _native.last_error()


def test_norm_backward():
    lib = _native.lib()

    def bwd(rows, heads, D, dw):
        return lib.gdn_layer_norm_bwd(P[0], None, P[1], P[2], P[3], dw, None, rows, heads, D, 1, 0, P[4],
                                      1 << 60, None)
    assert bwd(1 << 24, 1, 20001, None) == -2      # a workgroup per row
    assert bwd(4, 1 << 20, 256, P[5]) == -2        # a lane per column and slice of the sums
    assert bwd(0, 1 << 20, 256, P[5]) == -2


@pytest.mark.parametrize("N,Hqk,Hv,K,V", [(1 << 20, 16, 16, 64, 64), (1 << 20, 8, 16, 64, 128),
                                          (1 << 19, 32, 32, 128, 128)])
def test_many_sequences(N, Hqk, Hv, K, V):
    """A workgroup per sequence and v-head (backward: pair of them)."""
    lib = _native.lib()
    rows = (Hqk * K, Hqk * K, Hv * V)
    assert lib.gdn_linear_chunk_fwd(P[0], P[1], P[2], *rows, P[3], 0, 0, None, None, P[5], P[4], 1, N, Hqk,
                                    Hv, K, V, N, 0.1, None, P[11], 1 << 60, None) == -2
    assert "too large" in _native.last_error()
    # (a pair of v-heads per workgroup: twice as many sequences)
    M = N * (Hv // Hqk)
    assert lib.gdn_linear_chunk_bwd(P[0], P[1], P[2], *rows, P[3], 0, 0, P[5], None, P[6], P[7], P[8], P[9],
                                    P[10], None, P[4], 1, M, Hqk, Hv, K, V, M, 0.1, P[11], 1 << 60,
                                    None) == -2
    assert "too large" in _native.last_error()


NAMES = ("q", "k", "v", "g", "dO", "states", "cu", "dht", "dq", "dk", "dv", "dg", "dh0")
OUT = NAMES[8:]


@pytest.mark.parametrize("out", OUT)
@pytest.mark.parametrize("other", NAMES)
@pytest.mark.parametrize("sliced", [False, True])
def test_gradients_apart(out, other, sliced):
    if out == other or (out, other) == ("dh0", "dht"):
        return
    lib = _native.lib()
    at = dict(zip(NAMES, P))
    at[out] = at[other] + 16   # within both, at these sizes
    if sliced and other in "qkv":   # beyond a contiguous tensor's end, within the slices' rows
        at[out] = at[other] + 99 * 1024 * 2
    rows = (1024,) * 3 if sliced else (128, 128, 256)
    rc = lib.gdn_linear_chunk_bwd(at["q"], at["k"], at["v"], *rows, at["g"], 0, 0, at["dO"], at["dht"],
                                  at["states"], at["dq"], at["dk"], at["dv"], at["dg"], at["dh0"], at["cu"],
                                  1, 100, 2, 4, 64, 64, 7, 0.1, P[14], 1 << 60, None)
    assert rc == -5 and len(_native.last_error()) > 0
