"""What the learning operators refuse (bundlesdf_amd/learn_ops.py and their C entry points): an error with a text, nothing launched.
No GPU: the checks come before any device work."""
import ctypes as C

import pytest
import torch

from bundlesdf_amd import learn_ops as L
from bundlesdf_amd import lib

PTR = C.c_void_p(256)                                            # never dereferenced


def refused(f, *a, **k):
    with pytest.raises(lib.NofError) as e:
        f(*a, **k)
    return str(e.value)


def test_embed_refusals():
    t, i = torch.zeros(4, 3), torch.zeros(5, dtype=torch.int64)
    assert 'GPU' in refused(L.embed_lookup, t, i)
    assert 'float32' in refused(L.embed_lookup, t.double(), i)
    assert '[V, D]' in refused(L.embed_lookup, t[0], i)
    assert 'int32 or int64' in refused(L.embed_lookup, t, i.float())
    assert 'int32 or int64' in refused(L.embed_lookup_grad, torch.zeros(5, 3), i.to(torch.int16), 4)
    assert 'ids.shape' in refused(L.embed_lookup_grad, torch.zeros(4, 3), i, 4)
    assert 'n_rows' in refused(L.embed_lookup_grad, torch.zeros(5, 3), i, -1)
    assert 'n_rows' in refused(L.embed_lookup_grad, torch.zeros(5, 3), i, 1 << 30)
    assert 'GPU' in refused(L.embed_lookup_grad, torch.zeros(5, 3), i, 4)


def test_embed_entry_points_refuse():
    so = lib.load()

    def fwd(type=0, ids64=0, N=4, V=4, D=4, stride=4, ids=PTR, out=PTR, table=PTR):
        return so.nof_embed_fwd(table, stride, type, ids, ids64, 1.0, out, N, V, D, None)

    def bwd(type=0, ids64=0, N=4, V=4, D=4, stride=4, ids=PTR, grad=PTR, dout=PTR, ws=PTR, size=1 << 20):
        return so.nof_embed_bwd(dout, stride, type, ids, ids64, 1.0, grad, ws, size, N, V, D, None)

    for f in (fwd, bwd):
        for bad in ({'type': 3}, {'type': -1}, {'ids64': 2}, {'N': -1}, {'N': 1 << 31}, {'V': -1}, {'V': 1 << 30}, {'D': -1}, {'D': (1 << 20) + 1},
                    {'stride': -1}, {'ids': None}):
            assert f(**bad) < 0 and b'argument check' in so.nof_last_error(), bad
    assert fwd(out=None) < 0 and fwd(table=None) < 0
    assert bwd(grad=None) < 0 and bwd(dout=None) < 0 and bwd(ws=None) < 0 and bwd(size=0) < 0 and bwd(ws=C.c_void_p(8)) < 0
    assert fwd(N=0) == 0 and fwd(D=0) == 0 and bwd(V=0) == 0 and bwd(D=0) == 0           # nothing to do, nothing touched
    assert so.nof_embed_bwd_workspace_bytes(-1, 4, 4) == -1 and so.nof_embed_bwd_workspace_bytes(0, 4, 4) == 0
    assert so.nof_embed_bwd_workspace_bytes(70001, 1 << 20, 2) > 16 * 70001
