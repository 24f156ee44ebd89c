"""Outputs that overlap what other workgroups still read or write are refused by the entry points (on the CPU: no
call below launches anything)."""
import pytest

from avelang_amd import _native
from test_attn_host import E4M3, P, attn, rms, write


@pytest.mark.parametrize("kw", [
    dict(kc=P[3], vc=P[3]), dict(vc=P[3] + 4096), dict(ks=P[5], vs=P[5]), dict(vs=P[5] + 256), dict(k=P[3]),
    dict(k=P[4] + 512), dict(v=P[3] + 64), dict(v=P[4]),
])
def test_cache_write(kw):
    assert write(**kw) == -5 and "overlap" in _native.last_error()


@pytest.mark.parametrize("kw", [dict(o=P[1]), dict(o=P[2] + 4096), dict(o=P[2] - 64)])
def test_attention(kw):
    assert attn(**kw) == -5 and "overlap" in _native.last_error()


@pytest.mark.parametrize("kw", [
    dict(y=P[2]), dict(h=P[2]), dict(y=P[2] + 16), dict(y=P[2] - 512 + 2), dict(h=P[2], rows=1),
    dict(y=P[2], rows=1), dict(h=P[2], rows=1, wt=1), dict(out=E4M3, scale=P[6], y=P[2] + 8, rows=1)])
def test_norm(kw):
    assert rms(**kw) == -5 and "weight" in _native.last_error()
