"""The learning operators together, as a field with learnt codes trains: a code per frame looked up for every ray, features of every sample
through a weight matrix, blended back to front along the ray, a loss, and all the way back -- codes by their gradient, the matrix by its
orthogonalised gradient.

Tolerance of the gradients: every one is a chain of sums and products whose magnitudes M come from the same program on absolute values; no
chain has more than R * S + 1000 roundings of 2^-24 each in binary32."""
import pytest
import torch

pytestmark = pytest.mark.gpu
R, S, F, C, H = 300, 64, 12, 8, 16


def scene(seed=0):
    gen = torch.Generator().manual_seed(seed)
    return {'frame': torch.randint(-1, F, (R,), generator=gen), 'pts': torch.rand(R, S, 3, generator=gen) * 2 - 1, 'alpha': torch.rand(R, S, 1, generator=gen) * 0.2,
            'count': torch.randint(0, S + 1, (R,), generator=gen).to(torch.int32), 'want': torch.randn(R, H, generator=gen),
            'codes': torch.randn(F, C, generator=gen), 'weight': torch.randn(H, 3 + C, generator=gen) * 0.3}


def plain(s, absolute=False):
    """blend and gradients in 64 bits by autograd; `absolute`: of the magnitudes (a chain of sums and products of non-negative values)"""
    s = {k: v.double() if v.is_floating_point() else v for k, v in s.items()}
    pts, want = (s['pts'].abs(), -s['want'].abs()) if absolute else (s['pts'], s['want'])
    codes, weight, alpha = ((s[k].abs() if absolute else s[k].clone()).requires_grad_(True) for k in ('codes', 'weight', 'alpha'))
    code = torch.where((s['frame'] >= 0)[:, None], codes[s['frame'].clamp_min(0)], torch.zeros(()).double()) * 2.0
    x = torch.cat((pts, code[:, None].expand(R, S, C)), 2)
    feature = x @ weight.T
    here = (torch.arange(S)[None] < s['count'][:, None])[..., None]
    a = torch.where(here, alpha, torch.zeros(()).double())
    blend = torch.zeros(R, H).double()
    for t in reversed(range(S)):
        blend = (1 + a[:, t] if absolute else 1 - a[:, t]) * blend + a[:, t] * feature[:, t]
    (0.5 * (blend - want).square().sum()).backward()
    return blend.detach(), codes.grad, weight.grad, alpha.grad


def step(s, L):
    """the same through the framework, on the GPU"""
    code = L.embed_lookup(s['codes'], s['frame'], 2.0)
    x = torch.cat((s['pts'], code[:, None].expand(R, S, C)), 2)
    feature = (x.view(-1, 3 + C) @ s['weight'].T).view(R, S, H)
    h, blend, marks = L.gated_scan(1 - s['alpha'], s['alpha'] * feature, lengths=s['count'], reverse=True, want_marks=True)
    dgate, dvalue, _ = L.gated_scan_grad(1 - s['alpha'], s['alpha'] * feature, torch.zeros_like(h), blend - s['want'], marks=marks, lengths=s['count'], reverse=True)
    dalpha = (dvalue * feature).sum(2, keepdim=True) - dgate
    df = (s['alpha'] * dvalue).view(-1, H)
    dweight = df.T @ x.view(-1, 3 + C)
    dcode = (df @ s['weight'][:, 3:]).view(R, S, C).sum(1)
    dcodes = L.embed_lookup_grad(dcode, s['frame'], F, 2.0)
    return blend, dcodes, dweight, dalpha, L.orthogonalize(dweight)


def test_gradients_of_the_whole(nof):
    from bundlesdf_amd import learn_ops as L
    s = scene()
    want, mag = plain(s), plain(s, absolute=True)
    got = step({k: v.cuda() for k, v in s.items()}, L)
    for name, a, b, m in zip(('blend', 'codes', 'weight', 'alpha'), got, want, mag):
        bad = (a.double().cpu() - b).abs() > (R * S + 1000) * 2.0 ** -24 * m.abs()
        assert a.shape == b.shape and not bad.any(), (name, int(bad.sum()))
    # its singular values are the quintic's, five times, of the gradient's: not all near 1 (3.4445^5 = 485 lifts what is above a
    # thousandth of the norm), so they are compared one by one; products of 2^-22 of the norm, lifted by at most 1 + a + ... + a^4 = 197
    sv = torch.linalg.svdvals(got[2].double().cpu())
    sv = sv / sv.norm()
    for _ in range(5):
        sv = sv * (3.4445 + sv ** 2 * (-4.7750 + 2.0315 * sv ** 2))
    off = torch.linalg.svdvals(got[4].double().cpu()) - sv.sort(descending=True).values
    assert off.abs().max() < 4 * 197 * 2.0 ** -22


def test_trains_captured_as_it_does_eagerly(nof):
    """five steps of both kinds of update, eager and as one replayed graph: the same bits; the loss is a number all along"""
    from bundlesdf_amd import learn_ops as L
    a, b = ({k: v.cuda() for k, v in scene(1).items()} for _ in range(2))

    def update(s):
        blend, dcodes, dweight, _, direction = step(s, L)
        s['codes'].sub_(dcodes, alpha=1e-4)
        s['weight'].sub_(direction, alpha=1e-2)
        return 0.5 * (blend - s['want']).square().mean()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        keep = b['codes'].clone(), b['weight'].clone()
        update(b)                                                         # (a library's first call allocates: not inside the capture)
        b['codes'].copy_(keep[0])
        b['weight'].copy_(keep[1])
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        loss = update(b)
    for _ in range(5):
        want = update(a)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, want) and torch.isfinite(want)
        assert torch.equal(a['codes'], b['codes']) and torch.equal(a['weight'], b['weight'])
