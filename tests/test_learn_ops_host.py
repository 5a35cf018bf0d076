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


def test_scan_refusals():
    g, v, s = torch.zeros(2, 5, 3), torch.zeros(2, 5, 6), torch.zeros(2, 6)
    n = torch.zeros(2, dtype=torch.int32)
    assert 'GPU' in refused(L.gated_scan, g, v)
    assert 'B, T, D' in refused(L.gated_scan, g, v[0])
    assert 'B, T, D' in refused(L.gated_scan, g, v.double())
    assert 'but for the channels' in refused(L.gated_scan, g[:, :4], v)
    assert "float32 or of value's type" in refused(L.gated_scan, g.half(), v)
    assert "float32 or of value's type" in refused(L.gated_scan, g.half(), v.bfloat16())
    assert 'divide' in refused(L.gated_scan, torch.zeros(2, 5, 4), v)
    assert 'divide' in refused(L.gated_scan, torch.zeros(2, 5, 0), v)
    assert 'divide' in refused(L.gated_scan, torch.zeros(2, 5, 12), v)
    assert 'state' in refused(L.gated_scan, g, v, s[:1])
    assert 'state' in refused(L.gated_scan, g, v, s.half())
    assert 'lengths' in refused(L.gated_scan, g, v, s, n.long())
    assert 'lengths' in refused(L.gated_scan, g, v, s, n[:1])
    assert 'dh' in refused(L.gated_scan_grad, g, v, v[:, :4])
    assert 'dh' in refused(L.gated_scan_grad, g, v, v.half())
    assert 'dlast' in refused(L.gated_scan_grad, g, v, v, s[:, :2])
    assert 'marks' in refused(L.gated_scan_grad, g, v, v, s, s, torch.zeros(3))
    assert 'GPU' in refused(L.gated_scan_grad, g, v, v, s, s)
    assert 'state' in refused(L.gated_scan_step, g[:, 0], v[:, 0], None)
    assert 'B, D' in refused(L.gated_scan_step, g, v, s)
    assert 'new_state' in refused(L.gated_scan_step, g[:, 0], v[:, 0], s, s[:1])
    assert 'GPU' in refused(L.gated_scan_step, g[:, 0], v[:, 0], s)


def test_scan_entry_points_refuse():
    so = lib.load()
    null = C.c_void_p(None)

    def fwd(gt=0, t=0, rev=0, B=2, T=5, D=4, G=4, sb=20, st=4, gate=PTR, value=PTR, ws=null, size=0):
        return so.nof_gated_scan_fwd(gate, sb, st, gt, value, sb, st, t, null, null, rev, PTR, PTR, null, ws, size, B, T, D, G, None)

    def bwd(gt=0, t=0, rev=0, B=2, T=5, D=4, G=4, sb=20, st=4, gate=PTR, value=PTR, dh=PTR, marks=PTR, dgate=PTR, dvalue=PTR, ws=null, size=0):
        return so.nof_gated_scan_bwd(gate, sb, st, gt, value, sb, st, t, dh, sb, st, null, marks, null, rev, dgate, dvalue, PTR, ws, size, B, T, D, G, None)

    def step(gt=0, t=0, B=2, D=4, G=4, sb=4, gate=PTR, value=PTR, state=PTR, h=PTR):
        return so.nof_gated_scan_step(gate, sb, gt, value, sb, t, state, PTR, h, B, D, G, None)

    common = [{'t': 3}, {'gt': 1}, {'gt': 2, 't': 1}, {'B': -1}, {'B': 1 << 24}, {'D': -1}, {'D': (1 << 20) + 1}, {'G': 3}, {'G': 0}, {'G': 8}, {'sb': -1},
              {'gate': None}, {'value': None}, {'t': 1, 'gt': 1, 'value': C.c_void_p(258)}, {'t': 1, 'gt': 1, 'sb': 21}]
    for f in (fwd, bwd, step):
        for bad in common:
            assert f(**bad) < 0 and b'argument check' in so.nof_last_error(), (f.__name__, bad)
        assert f(B=0) == 0 and f(D=0) == 0
    for f in (fwd, bwd):
        for bad in ({'rev': 2}, {'T': -1}, {'T': 1 << 31}, {'st': -1}, {'T': 100000}):          # the last needs a workspace
            assert f(**bad) < 0 and b'argument check' in so.nof_last_error(), (f.__name__, bad)
    for bad in ({'dh': None}, {'marks': None}, {'dgate': None}, {'dvalue': None}):
        assert bwd(**bad) < 0
    assert step(state=None) < 0 and step(h=None) < 0
    assert so.nof_gated_scan_marks_bytes(2, 5, 4, 3, 0) == -1 and so.nof_gated_scan_workspace_bytes(2, 5, 4, 4, 7) == -1
    assert so.nof_gated_scan_marks_bytes(0, 5, 4, 4, 0) == 0 and so.nof_gated_scan_marks_bytes(2, 0, 4, 4, 0) == 0
    assert so.nof_gated_scan_marks_bytes(2, 5, 4, 4, 0) == 2 * 4 * 4


def test_orthogonalize_refusals():
    u = torch.zeros(4, 6)
    assert 'GPU' in refused(L.orthogonalize, u)
    assert 'm, n' in refused(L.orthogonalize, u[0])
    assert 'm, n' in refused(L.orthogonalize, u.double())
    assert '16384' in refused(L.orthogonalize, torch.zeros(1, 1).expand(16385, 1))
    assert '65535' in refused(L.orthogonalize, torch.zeros(1, 1, 1).expand(65536, 1, 1))
    assert 'steps' in refused(L.orthogonalize, u, steps=0)
    assert 'steps' in refused(L.orthogonalize, u, steps=33)
    assert 'triple' in refused(L.orthogonalize, u, coefficients=(1.0, 2.0))
    assert 'triple' in refused(L.orthogonalize, u, steps=3, coefficients=((1.5, -0.5, 0.0),) * 2)
    assert 'out' in refused(L.orthogonalize, u, out=torch.zeros(6, 4))
    assert 'out' in refused(L.orthogonalize, u, out=torch.zeros(6, 4).t())


def test_orthogonalize_entry_point_refuses():
    so = lib.load()
    quintic = (C.c_float * 15)(*L.QUINTIC * 5)

    def call(type=0, steps=5, coef=quintic, eps=1e-30, ws=None, size=0, batch=2, m=4, n=6, u=PTR, out=PTR):
        return so.nof_orthogonalize(u, out, type, steps, coef, eps, ws, size, batch, m, n, None)

    for bad in ({'type': 3}, {'steps': 0}, {'steps': 33}, {'coef': None}, {'eps': -1.0}, {'eps': float('nan')}, {'batch': -1}, {'batch': 65536},
                {'m': 16385}, {'n': -1}, {'u': None}, {'out': None}, {'m': 200}, {'m': 200, 'ws': PTR, 'size': 8}, {'m': 200, 'ws': C.c_void_p(8), 'size': 1 << 30},
                {'steps': 1, 'coef': (C.c_float * 3)(2.5, 0.0, 0.0)}, {'steps': 1, 'coef': (C.c_float * 3)(float('nan'), 0.0, 0.0)},
                {'steps': 2, 'coef': (C.c_float * 6)(1.9, 0.0, 0.0, 1.9, 0.0, 0.0)}, {'steps': 1, 'coef': (C.c_float * 3)(-16.0, 0.0, 15.0)}):
        assert call(**bad) < 0 and b'argument check' in so.nof_last_error(), bad
    assert call(batch=0) == 0 and call(m=0) == 0 and call(n=0) == 0
    assert so.nof_orthogonalize_workspace_bytes(1, 16385, 4) == -1 and so.nof_orthogonalize_workspace_bytes(1, 128, 128) == 0
    assert so.nof_orthogonalize_workspace_bytes(3, 129, 20) > 3 * 2 * 3 * 129 * 20 * 2


def test_overlap_of_results_and_inputs():
    x = torch.zeros(100)
    assert L._apart(x[:50], x[50:]) and L._apart(x[:50], x[:50]) and L._apart(x[:0], x[:9]) and L._apart(x[50:], x[:50])
    assert not L._apart(x[:50], x[49:]) and not L._apart(x[:50], x[:49]) and not L._apart(x[10:20], x)
