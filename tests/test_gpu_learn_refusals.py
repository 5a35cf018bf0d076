"""Tensors that the learning operators (bundlesdf_amd/learn_ops.py) refuse or read as what they stand for."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu
R = dict(device='cuda')


def calls(L):
    """(name, function, its float arguments)"""
    ids = torch.tensor([2, 0, 2, 5], **R)
    return [('embed_lookup', lambda t: L.embed_lookup(t, ids), [torch.randn(6, 3, **R)]),
            ('embed_lookup_grad', lambda d: L.embed_lookup_grad(d, ids, 6), [torch.randn(4, 3, **R)]),
            ('gated_scan', lambda g, v, s: L.gated_scan(g, v, s), [torch.rand(2, 9, 1, **R), torch.randn(2, 9, 4, **R), torch.randn(2, 4, **R)]),
            ('gated_scan_grad', lambda g, v, d, dl, s: L.gated_scan_grad(g, v, d, dl, s),
             [torch.rand(2, 9, 1, **R), torch.randn(2, 9, 4, **R), torch.randn(2, 9, 4, **R), torch.randn(2, 4, **R), torch.randn(2, 4, **R)]),
            ('gated_scan_step', lambda g, v, s: L.gated_scan_step(g, v, s), [torch.rand(2, 4, **R), torch.randn(2, 4, **R), torch.randn(2, 4, **R)]),
            ('orthogonalize', lambda u: L.orthogonalize(u), [torch.randn(5, 7, **R)])]


def test_tangents_are_refused(nof):
    from bundlesdf_amd import learn_ops as L
    for name, f, args in calls(L):
        want = f(*args)
        with forward_ad.dual_level():
            for k in range(len(args)):
                dual = list(args)
                dual[k] = forward_ad.make_dual(args[k], torch.ones_like(args[k]))
                with pytest.raises(nof.NofError, match=f'{name} carries no forward-mode tangents'):
                    f(*dual)
            got = f(*args)                                            # without one: as ever
        for a, b in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
            assert torch.equal(a, b)


def negated(x, **k):
    """x as a view of memory that holds -x"""
    y = torch.complex(torch.zeros_like(x), -x).conj().imag
    assert y.is_neg() and torch.equal(y, x)
    return y


@pytest.mark.parametrize('as_view', [negated, lambda x: torch._neg_view(-x)], ids=['conj', 'neg_view'])
def test_negated_views_are_read_as_what_they_stand_for(nof, as_view):
    """one channel, one element, one row: where nothing else makes a copy of them"""
    from bundlesdf_amd import learn_ops as L
    ids = torch.tensor([1, 0, 1], **R)
    more = calls(L) + [('lookup', lambda t: L.embed_lookup(t, ids), [torch.randn(2, 1, **R)]), ('grad', lambda d: L.embed_lookup_grad(d, ids, 2), [torch.randn(3, 1, **R)]),
                       ('scan', lambda g, v, s: L.gated_scan(g, v, s), [torch.rand(2, 9, 1, **R), torch.randn(2, 9, 1, **R), torch.randn(2, 1, **R)]),
                       ('scan grad', lambda g, v, d, dl, s: L.gated_scan_grad(g, v, d, dl, s),
                        [torch.rand(2, 9, 1, **R), torch.randn(2, 9, 1, **R), torch.randn(2, 9, 1, **R), torch.randn(2, 1, **R), torch.randn(2, 1, **R)]),
                       ('step', lambda g, v, s: L.gated_scan_step(g, v, s), [torch.rand(2, 1, **R), torch.randn(2, 1, **R), torch.randn(2, 1, **R)]),
                       ('update', lambda u: L.orthogonalize(u), [torch.randn(1, 1, **R)])]
    for name, f, args in more:
        want = f(*args)
        for k in range(len(args)):
            view = list(args)
            view[k] = as_view(args[k])
            assert view[k].is_neg() and torch.equal(view[k], args[k])
            got = f(*view)
            for a, b in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
                assert torch.equal(a, b), (name, k)
    u, s = torch.randn(4, 4, **R), torch.randn(2, 4, **R)
    with pytest.raises(nof.NofError, match='negated'):
        L.orthogonalize(u, out=torch._neg_view(u.clone()))
    with pytest.raises(nof.NofError, match='negated'):
        L.gated_scan_step(torch.rand(2, 4, **R), torch.randn(2, 4, **R), s, torch._neg_view(s.clone()))


def test_a_new_state_that_another_lane_reads_is_refused(nof):
    from bundlesdf_amd import learn_ops as L
    line, state = torch.zeros(400, **R), torch.randn(4, 8, **R)
    gate, value = torch.rand(4, 8, **R), torch.randn(4, 8, **R)
    for shift in (1, 8, 31):
        at = line[shift:shift + 32].view(4, 8)
        with pytest.raises(nof.NofError, match='apart from gate and value'):
            L.gated_scan_step(gate, line[:32].view(4, 8), state, at)
        with pytest.raises(nof.NofError, match='apart from gate and value'):
            L.gated_scan_step(line[:32].view(4, 8), value, state, at)
        with pytest.raises(nof.NofError, match='apart from gate and value'):
            L.gated_scan_step(line[:4].view(4, 1) if shift < 4 else line[shift + 3:shift + 7].view(4, 1), value, state, at)
    with pytest.raises(nof.NofError, match='apart from gate and value'):                  # rows of a wider tensor
        L.gated_scan_step(gate, line[:400].view(4, 100)[:, 90:98], state, line[100:132].view(4, 8))
    with pytest.raises(nof.NofError, match='apart from gate and value'):                  # of another type
        L.gated_scan_step(gate, line[:16].view(torch.bfloat16).view(4, 8), state, line[:32].view(4, 8))
    want = L.gated_scan_step(gate, value, state)
    for which in (0, 1):                                                                  # in the very place of one of them: each lane its own element
        g, v = gate.clone(), value.clone()
        h, new = L.gated_scan_step(g, v, state, (g, v)[which])
        assert new.data_ptr() == (g, v)[which].data_ptr() and torch.equal(new, want[1]) and torch.equal(h, want[0])
    h, new = L.gated_scan_step(gate, line[:32].view(4, 8).copy_(value), state, line[32:64].view(4, 8))       # side by side
    assert torch.equal(new, want[1]) and torch.equal(h, want[0])


def test_behind_an_infinity_its_channel_is_not_finite(nof):
    from bundlesdf_amd import learn_ops as L
    gate, value, state = torch.full((2, 4000, 1), 0.5, **R), torch.randn(2, 4000, 3, **R), torch.zeros(2, 3, **R)
    want, last = L.gated_scan(gate, value, state)
    for at, sign in ((0, 1.0), (17, -1.0), (1500, -1.0)):
        bad = value.clone()
        bad[1, at, 2] = sign * float('inf')
        h, end = L.gated_scan(gate, bad, state)
        assert not h[1, at:, 2].isfinite().any() and not end[1, 2].isfinite() and h[1, at, 2] == sign * float('inf')
        assert torch.equal(h[0], want[0]) and torch.equal(h[1, :, :2], want[1, :, :2]) and torch.equal(h[1, :at], want[1, :at])
