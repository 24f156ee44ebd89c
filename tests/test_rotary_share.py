"""Rotary positions on the CPU: q and k that share elements are refused in place, and outputs that do."""
import pytest

from avelang_amd import _native
from avelang_amd.rotary import _STRIDES

BF = 1
BASE = 1 << 40   # an address that no call below reaches: every one is refused


def _in_place(q, k, qs, ks, B, T, Hq, Hk, D, apart=0):
    """q and k at these elements of a bf16 buffer, in place or (``apart``) as outputs of other inputs."""
    q, k = BASE + 2 * q, BASE + 2 * k
    args = (q + apart, k + 2 * apart, q, k, _STRIDES(*qs, *ks, *qs, *ks))
    return _native.lib().gdn_rotary(*args, B, T, Hq, Hk, D, 1 << 44, 1, 0, 1 << 45, D, 1.0, 0, 0, BF, None)


@pytest.mark.parametrize("apart", [0, 1 << 42])
@pytest.mark.parametrize("q,k,qs,ks,B,T,Hq,Hk,D", [
    (0, 0, (0, 192, 64), (0, 192, 64), 1, 4, 2, 1, 64),         # k is q's first head
    (0, 64, (0, 192, 64), (0, 192, 64), 1, 4, 2, 1, 64),        # its second
    (0, 127, (0, 192, 64), (0, 192, 64), 1, 4, 2, 1, 64),       # one element of it
    (0, 192, (0, 192, 64), (0, 192, 64), 1, 4, 2, 1, 64),       # the next token's
    (192, 0, (0, 192, 64), (0, 192, 64), 1, 4, 2, 1, 64),
    (0, 191, (0, 192, 64), (0, 192, 64), 1, 4, 2, 1, 64),       # the next token's first element
    (0, 3 * 192, (0, 192, 64), (0, 192, 64), 1, 4, 2, 1, 64),   # q's last token, k's first
    (0, 32, (4096, 128, 64), (4096, 128, 64), 3, 5, 2, 2, 64),
    (0, 4096 + 512, (4096, 128, 64), (4096, 64, 4096), 3, 5, 2, 1, 64),   # q's second batch's last token
    (0, 7, (0, 100, 10), (0, 77, 11), 1, 9, 3, 2, 6),           # strides that have nothing in common
])
def test_refused(q, k, qs, ks, B, T, Hq, Hk, D, apart):
    shared = {q + b * qs[0] + t * qs[1] + h * qs[2] + e for b in range(B) for t in range(T) for h in range(Hq)
              for e in range(D)} & {k + b * ks[0] + t * ks[1] + h * ks[2] + e for b in range(B) for t in range(T)
                                    for h in range(Hk) for e in range(D)}
    assert shared   # (a case that shares nothing would be launched)
    assert _in_place(q, k, qs, ks, B, T, Hq, Hk, D, apart) == -5
    assert "share no element" in _native.last_error()
