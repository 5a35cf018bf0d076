"""How exact the orthogonalised update is (bundlesdf_amd/learn_ops.py: orthogonalize), beyond tests/test_gpu_learn_ortho.py's bound for
whole matrices of noise."""
import pytest
import torch

pytestmark = pytest.mark.gpu
QUINTIC = (3.4445, -4.7750, 2.0315)


def randn(*shape, seed):
    return torch.randn(*shape, device='cuda', generator=torch.Generator(device='cuda').manual_seed(seed))


def iterate(x, steps, coef=QUINTIC):
    """the definition on a normalised x, in x's type"""
    a, b, c = coef
    for _ in range(steps):
        g = x @ x.mT.contiguous() if x.shape[-2] <= x.shape[-1] else x.mT.contiguous() @ x
        p = b * g + c * (g @ g)
        x = a * x + (p @ x if x.shape[-2] <= x.shape[-1] else x @ p)
    return x


def normalised(u):
    x = u.double()
    return x / x.flatten(-2).norm(dim=-1)[..., None, None]


def half_step(x, dtype):
    """half a step of `dtype` at x: its bits of mantissa below x's binade, not below its smallest one's"""
    bits, least = {torch.bfloat16: (8, -134), torch.float16: (11, -25)}[dtype]
    return torch.maximum(torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(1e-300))) - bits), torch.full_like(x, 2.0 ** least))


# A result of 16 bits is the binary32 result rounded once: no product on the way to it has fewer bits because of the result's type.  Both
# calls get the same values; only the norm's sum (64 bits) may run in another order, which moves single elements of X by a rounding
# of binary32 (2^-24 of them, together at most 2^-24 of |X| = 1), and five steps amplify it by at most (largest slope of the quintic, 4)^5 =
# 2^10: an error of at most 2^-14 before the rounding, at most twice that beyond half a step behind it (a value that crosses into the next binade).
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('m,n,rank', [(333, 1001, 1), (1001, 333, 1), (700, 900, 16), (1024, 1024, 16), (256, 512, 2), (140, 2300, 3), (200, 1100, 4), (20, 700, 1), (100, 90, 2)])
def test_sixteen_bits_are_the_binary32_result_rounded_once(nof, dtype, m, n, rank):
    from bundlesdf_amd import learn_ops as L
    u = (randn(m, rank, seed=m) @ randn(rank, n, seed=n)).to(dtype)
    for steps, coef in ((5, QUINTIC), (2, QUINTIC), (1, QUINTIC), (1, (8.2872, -23.5959, 17.3004))):
        got, want = L.orthogonalize(u, steps=steps, coefficients=coef), L.orthogonalize(u.float(), steps=steps, coefficients=coef).double()
        beyond = ((got.double() - want).abs() - half_step(want, dtype)).clamp_min(0.0)
        assert got.dtype == dtype and float(beyond.norm()) <= 2.0 ** -13, (steps, coef, float(beyond.norm()), float(want.norm()))


# Beside a binary32 computation of the same products.  There a product of two elements is rounded once, 2^-24 of it; here its operands are held to
# 2^-23 each and lo lo, at most 2^-24 (2^-12 of either), is left out: five times as much.  The sums are binary32's in both.  So an error is at most five
# times the binary32 computation's -- of a row, or a column, where those differ in size --, as long as what carries it lies above the smallest
# that pairs hold, 2^-48 of the norm: P (|a| + |b| + |c| = s of magnitudes, r elements a row) and X bring s (1 + sqrt(r)) of those to a row of size `size`.
def check_beside_binary32(got, u, steps, dim, coef=QUINTIC):
    x = normalised(u)
    want = iterate(x, steps, coef)
    plain = iterate(x.float(), steps, coef).double()
    size = x.norm(dim=dim).clamp_min(1e-300)
    floor = 2.0 ** -48 * sum(abs(c) for c in coef) * (1 + min(u.shape[-2:]) ** 0.5) / size
    off, ref = ((y - want).norm(dim=dim) / want.norm(dim=dim).clamp_min(1e-300) for y in (got.double(), plain))
    bad = off > 5 * ref.amax(-1, keepdim=True) + floor
    assert not bad.any(), (u.shape, steps, int(bad.sum()), float((off / (5 * ref.amax(-1, keepdim=True) + floor)).max()), float(off.max()), float(ref.max()))


SHAPES = [(8, 4096), (8, 100), (40, 96), (64, 1000), (100, 120), (96, 96), (90, 700), (200, 400), (333, 1001), (130, 2300), (1024, 4096)]


@pytest.mark.parametrize('m,n', SHAPES + [(n, m) for m, n in SHAPES])
def test_rows_and_columns_of_very_different_size(nof, m, n):
    """an embedding's seldom rows, units that are almost dead: 1e-5, 1e-7 of the others, and so many steps that they become part of the result"""
    from bundlesdf_amd import learn_ops as L
    for small in (1e-3, 1e-5, 1e-7):
        rows, cols = randn(2, m, n, seed=m + n), randn(2, m, n, seed=m + n + 1)
        rows[:, ::2] *= small
        cols[:, :, 1::2] *= small
        for steps in (5, 12):
            check_beside_binary32(L.orthogonalize(rows, steps=steps), rows, steps, -1)
            check_beside_binary32(L.orthogonalize(cols, steps=steps), cols, steps, -2)


@pytest.mark.parametrize('m,n', [(8, 8), (50, 50), (120, 120), (20, 300), (150, 150), (300, 200)])
def test_single_values_down_to_1e_9(nof, m, n):
    from bundlesdf_amd import learn_ops as L
    u = torch.zeros(m, n, device='cuda')
    k = min(m, n)
    u[torch.arange(k), torch.arange(k)] = torch.logspace(0, -9, k, device='cuda')
    for steps in (5, 12):
        check_beside_binary32(L.orthogonalize(u, steps=steps)[:k, :k], u[:k, :k], steps, -1)


@pytest.mark.parametrize('m,n', SHAPES + [(2048, 2048), (4001, 1100)])
def test_low_rank_and_noise(nof, m, n):
    """few strong directions over weak ones, which the steps lift: where single fp16 products are off by percents"""
    from bundlesdf_amd import learn_ops as L
    for noise in (0.0, 1e-4, 1e-2):
        u = randn(m, 4, seed=m) @ randn(4, n, seed=n) + noise * randn(m, n, seed=m + n)
        for steps in (1, 5):
            x = normalised(u)
            want = iterate(x, steps)
            got, plain = L.orthogonalize(u, steps=steps).double(), iterate(x.float(), steps).double()
            assert float((got - want).norm()) <= 5 * float((plain - want).norm()), (noise, steps, float((got - want).norm()), float((plain - want).norm()))


# A multiple of the identity has one singular value, 1 / sqrt(k), and every product one term: the error is no average.  Of the value s, with
# eta = 5 * 2^-24 a product, A is off by eta s^2 and A A by 4 eta s^4 at most (its two factors, itself, its storing), b A by 2, P by its storing and
# its product with X: eta s (2 |b| s^2 + 4 |c| s^4 + 2 (|a| + |b| s^2 + |c| s^4)); a former error is multiplied by the slope.
@pytest.mark.parametrize('k', [5, 30, 64, 100, 128, 200, 333, 1024, 2048])
def test_multiple_of_the_identity(nof, k):
    from bundlesdf_amd import learn_ops as L
    a, b, c = QUINTIC
    for steps in (1, 2, 5):
        s, tol, eta = k ** -0.5, k ** -0.5 * 2.0 ** -22, 5 * 2.0 ** -24
        for _ in range(steps):
            tol = abs(a + 3 * b * s ** 2 + 5 * c * s ** 4) * tol * 1.01 + eta * s * (2 * abs(b) * s ** 2 + 4 * abs(c) * s ** 4 + 2 * abs(a) + 2 * abs(b) * s ** 2 + 2 * abs(c) * s ** 4)
            s = s * (a + s ** 2 * (b + c * s ** 2))
        got = L.orthogonalize(torch.eye(k, device='cuda') * 0.37, steps=steps).double()
        assert float((got.diagonal() - s).abs().max()) <= tol, (steps, float((got.diagonal() - s).abs().max()), tol)
        assert float((got - torch.diag(got.diagonal())).abs().max()) == 0.0


# The products by tiles of 128 x 128: of X one tile a compute unit at most (2500 x 1024, 2048 x 2048 and its A and P), more (4001 x 1100; the last
# two, of whose A and P too), of either orientation; padded to whole tiles or not; one matrix and several.
@pytest.mark.parametrize('batch,m,n', [(1, 2500, 1024), (1, 1024, 2500), (1, 2048, 2048), (1, 4096, 1024), (1, 1024, 4096), (4, 1024, 1024), (1, 4001, 1100),
                                       (1, 1100, 4001), (3, 1153, 1400), (9, 600, 900), (2, 2048, 2048), (1, 2950, 2900)])
def test_large_tiles(nof, batch, m, n):
    from bundlesdf_amd import learn_ops as L
    u = randn(batch, m, n, seed=m + n) + randn(batch, m, 4, seed=m) @ randn(batch, 4, n, seed=n)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        v = u.to(dtype)
        for steps in (1, 2, 5):
            x = normalised(v)
            want = iterate(x, steps)
            off = (iterate(x.float(), steps).double() - want).flatten(1).norm(dim=1)
            got = L.orthogonalize(v, steps=steps)
            err = (got.double() - want).abs()
            if dtype != torch.float32:                                # (beyond half a step at most twice what there was before the rounding)
                err, off = (err - half_step(want, dtype)).clamp_min(0.0), 2 * off
            assert (err.flatten(1).norm(dim=1) <= 5 * off).all(), (dtype, steps, err.flatten(1).norm(dim=1).tolist(), off.tolist())
            assert torch.equal(got, L.orthogonalize(v, steps=steps))
            w = v.clone()
            L.orthogonalize(w, steps=steps, out=w)
            assert torch.equal(got, w)
