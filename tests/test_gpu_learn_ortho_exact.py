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
