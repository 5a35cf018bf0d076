"""The gradients of the learning operators as a field with learnt codes uses them together -- code per frame, features through a weight matrix,
blended back to front along the ray, loss, and back --, bounded closely enough that a wrong one is seen.  (The check of the same chain in
tests/test_gpu_learn_train.py uses 64 samples a ray and 1 + opacity for the gates' magnitude, 1.1^64 of what it bounds: gradients of zero pass it.)

Tolerance: u = 2^-24 times the roundings of a chain times M, the same chain on absolute values with the gates |1 - opacity|.  A term goes through the
code's product (1), a feature's sum of 3 + C products (3 + C + 1), opacity times it and 1 - opacity (2), the scan (3 per sample and 64 for the levels
of its composition, as tests/test_gpu_learn_scan.py has it), the residual (1), the scan backward (as much again), the products of the gradients (3),
and the sum that its gradient is: H channels for an opacity, R S samples for a weight, H channels and the samples of all rays of its frame for a
code (scaled: 1)."""
import pytest
import torch

R, S, F, C, H = 240, 6, 12, 5, 16
SCALE = 2.0


def scene(seed):
    gen = torch.Generator().manual_seed(seed)
    return {'frame': torch.randint(-1, F, (R,), generator=gen), 'pts': torch.rand(R, S, 3, generator=gen) * 2 - 1, 'alpha': torch.rand(R, S, 1, generator=gen) * 0.4,
            'count': torch.randint(0, S + 1, (R,), generator=gen).to(torch.int32), 'want': torch.randn(R, H, generator=gen) * 0.3,
            'codes': torch.randn(F, C, generator=gen), 'weight': torch.randn(H, 3 + C, generator=gen) * 0.5}


def plain(s, absolute=False):
    """in 64 bits by autograd: blend, and the gradients of codes, weight, and of the opacity through the values and through the gates"""
    s = {k: v.double() if v.is_floating_point() else v for k, v in s.items()}
    size = torch.abs if absolute else torch.clone
    pts, want = size(s['pts']), -s['want'].abs() if absolute else s['want']
    codes, weight, alpha, gate = (size(x).requires_grad_(True) for x in (s['codes'], s['weight'], s['alpha'], 1 - s['alpha']))
    code = torch.where((s['frame'] >= 0)[:, None], codes[s['frame'].clamp_min(0)], torch.zeros(()).double()) * SCALE
    feature = torch.cat((pts, code[:, None].expand(R, S, C)), 2) @ weight.T
    blend = torch.zeros(R, H).double()
    for t in reversed(range(S)):
        here = (t < s['count'])[:, None]
        blend = torch.where(here, gate[:, t] * blend + alpha[:, t] * feature[:, t], blend)
    (0.5 * (blend - want).square().sum()).backward()
    return {'blend': blend.detach(), 'codes': codes.grad, 'weight': weight.grad, 'value': alpha.grad, 'gate': gate.grad}


def bounds(s):
    m = plain(s, absolute=True)
    m['alpha'] = m['value'] + m['gate']
    forward = 1 + 3 + C + 1 + 2 + 3 * S + 64
    back = forward + 1 + 3 * S + 64 + 3
    rays = int(torch.bincount(s['frame'].clamp_min(0), minlength=F).max())
    count = {'blend': forward, 'alpha': back + H, 'weight': back + R * S, 'codes': back + H + rays * S + 1}
    return {k: n * 2.0 ** -24 * m[k] for k, n in count.items()}


def gradients(s):
    want = plain(s)
    return {'blend': want['blend'], 'codes': want['codes'], 'weight': want['weight'], 'alpha': want['value'] - want['gate']}


@pytest.mark.parametrize('seed', range(3))
def test_wrong_gradients_exceed_the_bounds(seed):
    s = scene(seed)
    want, tol, parts = gradients(s), bounds(s), plain(s)
    for name, w in want.items():
        there = w != 0
        for wrong, share in ((0 * w, 0.9), (-w, 0.9), (2 * w, 0.9), (w * 1.01, 0.5)):      # of its elements (some are near zero themselves)
            seen = (wrong - w).abs() > tol[name]
            assert seen[there].double().mean() > share, (name, seen[there].double().mean())
    for wrong in (parts['value'], -parts['gate'], parts['value'] + parts['gate']):        # a term dropped, the other one, its sign
        seen = ((wrong - want['alpha']).abs() > tol['alpha'])[want['alpha'] != 0]
        assert seen.double().mean() > 0.6
    shifted = want['codes'].roll(1, 0)                                                    # the neighbour's code
    assert ((shifted - want['codes']).abs() > tol['codes']).double().mean() > 0.9


@pytest.mark.gpu
@pytest.mark.parametrize('seed', range(3))
def test_gradients_of_the_whole(nof, seed):
    from bundlesdf_amd import learn_ops as L
    host = scene(seed)
    s = {k: v.cuda() for k, v in host.items()}
    code = L.embed_lookup(s['codes'], s['frame'], SCALE)
    x = torch.cat((s['pts'], code[:, None].expand(R, S, C)), 2)
    feature = (x.view(-1, 3 + C) @ s['weight'].T).view(R, S, H)
    gate, value = 1 - s['alpha'], s['alpha'] * feature
    h, blend, marks = L.gated_scan(gate, value, lengths=s['count'], reverse=True, want_marks=True)
    dgate, dvalue, _ = L.gated_scan_grad(gate, value, torch.zeros_like(h), blend - s['want'], marks=marks, lengths=s['count'], reverse=True)
    df = (s['alpha'] * dvalue).view(-1, H)
    dcode = (df @ s['weight'][:, 3:]).view(R, S, C).sum(1)
    got = {'blend': blend, 'codes': L.embed_lookup_grad(dcode, s['frame'], F, SCALE), 'weight': df.T @ x.view(-1, 3 + C),
           'alpha': (dvalue * feature).sum(2, keepdim=True) - dgate}
    want, tol = gradients(host), bounds(host)
    for name, w in want.items():
        bad = (got[name].double().cpu() - w).abs() > tol[name]
        assert got[name].shape == w.shape and not bad.any(), (name, int(bad.sum()))
