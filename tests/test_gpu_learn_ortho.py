"""The orthogonalised update (bundlesdf_amd/learn_ops.py: orthogonalize) against the singular value decomposition in 64 bits: the quintic
moves each singular value by itself.

Tolerance.  Write q = p o ... o p for the composed polynomial.  An operand pair holds its value to 2^-23, the sums over K terms are
binary32: each product of a step is off by at most (2 * 2^-23 + sqrt(K) 2^-24 + 2^-22) of the operands' Frobenius norms (hi lo products
that are left out: 2^-24; sums taken as a random walk, with a factor 4 in hand).  A perturbation E of X (Frobenius, against |X| <= sqrt(r))
grows per later step by at most the polynomial's steepest slope, a = 3.4445 near zero, less elsewhere: summed over five steps at
most (1 + a + ... + a^4) = 197 at the first step's |X| = 1, after which |X| has grown with it.  Relative to |result| >= 0.6 sqrt(rank):
bound = 4 * 197 * 2^-22 / (0.6 sqrt(rank)) * (1 + sqrt(K) / 8) + eps/2 of the type (3e-4 for one full-rank direction, 6e-6 for rank 1000)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def exact(u, steps=5, coef=(3.4445, -4.7750, 2.0315)):
    x = u.double()
    left, s, right = torch.linalg.svd(x, full_matrices=False)
    s = s / torch.sqrt((s * s).sum(-1, keepdim=True))
    for i in range(steps):
        a, b, c = coef[i] if isinstance(coef[0], tuple) else coef
        s = s * (a + s ** 2 * (b + c * s ** 2))
    return (left * s[..., None, :]) @ right


def make(kind, shape, dtype, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    g = torch.randn(*shape, device='cuda', generator=gen)
    if kind == 'decay':                                               # singular values 1, 1/2, 1/3, ...
        left, s, right = torch.linalg.svd(g.double().cpu(), full_matrices=False)
        s = 1.0 / torch.arange(1, s.shape[-1] + 1, dtype=torch.float64).expand(s.shape)
        g = ((left * s[..., None, :]) @ right).float().cuda()
    elif kind == 'tiny':
        g = g * (1e-20 if dtype != torch.float16 else 1e-4)
    elif kind == 'huge':
        g = g * (1e20 if dtype != torch.float16 else 1e3)
    return g.to(dtype)


def check(got, u, **k):
    want = exact(u.cpu(), **k)
    K, rank = max(u.shape[-2:]), min(u.shape[-2:])
    tol = 4 * 197 * 2.0 ** -22 / (0.6 * rank ** 0.5) * (1 + K ** 0.5 / 8) + torch.finfo(u.dtype).eps / 2
    if u.dtype == torch.float16:
        tol += 2.0 ** -25 * K ** 0.5 / 0.6                            # fp16's subnormal spacing over |result| / sqrt(r K)
    err = (got.double().cpu() - want).flatten(-2).norm(dim=-1) / want.flatten(-2).norm(dim=-1)
    assert got.shape == u.shape and got.dtype == u.dtype and bool((err <= tol).all()), (err.max().item(), tol)


SHAPES = [(1, 1), (1, 7), (5, 1), (3, 64), (16, 64), (64, 31), (64, 32), (64, 64), (33, 65), (128, 128), (127, 100), (128, 1), (129, 128), (4, 130),
          (130, 130), (1, 300), (300, 1), (256, 128), (257, 385), (600, 130), (333, 1001), (512, 512),
          (20, 2000), (3000, 50), (90, 700), (128, 4200), (2500, 97), (32, 129), (300, 64), (140, 2300)]


@pytest.mark.parametrize('m,n', SHAPES)
@pytest.mark.parametrize('kind', ['noise', 'decay', 'tiny', 'huge'])
def test_matrices(nof, m, n, kind):
    from bundlesdf_amd import learn_ops as L
    for q, dtype in enumerate(TYPES):
        u = make(kind, (2, m, n), dtype, m + n + q)
        got = L.orthogonalize(u)
        check(got, u)
        assert torch.equal(got, L.orthogonalize(u)) and torch.equal(got[1], L.orthogonalize(u[1]))     # the same bits, alone or in a batch


@pytest.mark.parametrize('dtype', TYPES)
def test_a_large_one(nof, dtype):
    from bundlesdf_amd import learn_ops as L
    u = make('noise', (1500, 2000), dtype, 1)
    got = L.orthogonalize(u)
    x = u.double()
    x = x / x.norm()
    for _ in range(5):
        a = x @ x.mT.contiguous()
        x = 3.4445 * x + (-4.7750 * a + 2.0315 * (a @ a)) @ x
    err = ((got.double() - x).norm() / x.norm()).item()
    assert err < 4 * 197 * 2.0 ** -22 / (0.6 * 1500 ** 0.5) * (1 + 2000 ** 0.5 / 8) + torch.finfo(dtype).eps / 2, err


@pytest.mark.parametrize('m,n', [(40, 96), (96, 40), (200, 300), (300, 200)])
def test_steps_coefficients_layout_and_place(nof, m, n):
    from bundlesdf_amd import learn_ops as L
    u = make('noise', (3, 2, m, n), torch.float32, 3)
    check(L.orthogonalize(u, steps=1), u, steps=1)
    cubic = (1.5, -0.5, 0.0)
    check(L.orthogonalize(u, steps=3, coefficients=cubic), u, steps=3, coef=cubic)
    plan = ((3.0, -3.2, 1.2), (2.0, -1.5, 0.5), (1.5, -0.5, 0.0))
    check(L.orthogonalize(u, steps=3, coefficients=plan), u, steps=3, coef=plan)
    want = L.orthogonalize(u)
    assert torch.equal(L.orthogonalize(u.mT.contiguous().mT), want)                       # any strides
    out = torch.full_like(u, 7.0)
    assert L.orthogonalize(u, out=out).data_ptr() == out.data_ptr() and torch.equal(out, want)
    v = u.clone()
    L.orthogonalize(v, out=v)                                                             # in place
    assert torch.equal(v, want)
    line = torch.zeros(u.numel() + 8, device='cuda')
    with pytest.raises(nof.NofError, match='apart'):
        L.orthogonalize(line[:u.numel()].view(u.shape), out=line[8:].view(u.shape))
    assert L.orthogonalize(u[:0]).shape == (0, 2, m, n) and L.orthogonalize(u[..., :0]).shape == (3, 2, m, 0)


@pytest.mark.parametrize('m,n', [(50, 60), (150, 60)])
def test_zero_and_not_finite(nof, m, n):
    from bundlesdf_amd import learn_ops as L
    u = make('noise', (4, m, n), torch.float32, 5)
    want = L.orthogonalize(u)
    u[1] = 0.0
    u[2, 3, 4] = float('inf')
    u[3, 5, 6] = float('nan')
    for eps in (1e-30, 0.0, 1e-7):
        got = L.orthogonalize(u, eps=eps)
        assert torch.equal(got[0], want[0]) and (got[1] == 0).all()                       # neighbours in a batch do not mix
        assert got[2].isnan().all() and got[3].isnan().all()
    small = L.orthogonalize(u[:1] * 1e-6, steps=1, eps=1.0)                               # below eps: not blown up
    x = u[:1].double() * 1e-6
    ref = 3.4445 * x - 4.7750 * (x @ x.mT.contiguous()) @ x
    assert ((small.double() - ref).norm() / ref.norm()).item() < 2.0 ** -10               # 4096 * 1e-6 in fp16 pairs: lo is subnormal


def test_stream_and_graph(nof):
    from bundlesdf_amd import learn_ops as L
    a, b = make('noise', (6, 100, 128), torch.float32, 1), make('noise', (300, 140), torch.bfloat16, 2)
    want = L.orthogonalize(a), L.orthogonalize(b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = L.orthogonalize(a), L.orthogonalize(b)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = L.orthogonalize(a), L.orthogonalize(b)
    gen = torch.Generator(device='cuda').manual_seed(0)
    for _ in range(4):
        a.normal_(generator=gen)
        b.normal_(generator=gen)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], L.orthogonalize(a)) and torch.equal(out[1], L.orthogonalize(b))


@pytest.mark.parametrize('m,n', [(9, 20), (20, 9), (31, 128), (9, 300), (32, 2100), (300, 17), (40, 64), (33, 100), (128, 50), (64, 300), (700, 41), (100, 100), (90, 300),
                                 (140, 300), (140, 2300), (1100, 333)])
@pytest.mark.parametrize('dtype', TYPES)
def test_every_way_of_computing_it(nof, m, n, dtype):
    """one, two and five steps, in place, a zero matrix and one that is not finite between others, and captured: replays with the program's own calls between"""
    from bundlesdf_amd import learn_ops as L
    u = make('noise', (4, m, n), dtype, m + n)
    for steps in (1, 2):
        check(L.orthogonalize(u, steps=steps), u, steps=steps)
    want = L.orthogonalize(u)
    check(want, u)
    v = u.clone()
    assert L.orthogonalize(v, out=v) is v and torch.equal(v, want)
    v = u.clone()
    v[1] = 0.0
    v[2, m // 2, n // 2] = float('nan')
    got = L.orthogonalize(v)
    assert torch.equal(got[0], want[0]) and torch.equal(got[3], want[3]) and (got[1] == 0).all() and got[2].isnan().all()
    v[2, m // 2, n // 2] = float('-inf')
    got = L.orthogonalize(v)
    assert torch.equal(got[3], want[3]) and got[2].isnan().all()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = L.orthogonalize(v)
    for seed in range(3):
        v.copy_(make('decay', (4, m, n), dtype, seed))
        g.replay()
        eager = L.orthogonalize(v)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
    check(out, v)
