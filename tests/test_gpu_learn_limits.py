"""The learning operators (bundlesdf_amd/learn_ops.py) at the far end of the sizes that they take."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def poisoned(*shape, dtype):
    """the next tensor of this size lies where this one of NaN lay"""
    x = torch.full(shape, float('nan'), dtype=dtype, device='cuda')
    torch.cuda.synchronize()
    del x


@pytest.mark.parametrize('N', [0, 3000, 5000])
def test_gradient_of_the_largest_table(nof, N):
    """2^30 - 1 rows: every row that no id names is zero"""
    from bundlesdf_amd import learn_ops as L
    V = (1 << 30) - 1
    gen = torch.Generator(device='cuda').manual_seed(N)
    ids = torch.randint(0, V, (N,), device='cuda', generator=gen, dtype=torch.int64)
    if N:
        ids[:4] = torch.tensor([0, V - 1, V - 1, V // 2], device='cuda')
    dout = torch.randint(1, 9, (N, 1), device='cuda', generator=gen).to(torch.bfloat16)
    poisoned(V, 1, dtype=torch.bfloat16)
    grad = L.embed_lookup_grad(dout, ids, V)
    unique, where = torch.unique(ids, return_inverse=True)
    want = torch.zeros(unique.numel(), device='cuda').index_add_(0, where, dout[:, 0].float())       # whole numbers of at most 8 bits: exact
    assert torch.equal(grad[unique, 0].float(), want)
    assert int(torch.count_nonzero(grad)) == unique.numel()


def test_gradient_of_more_than_2_30_positions(nof):
    """every id holds some thousand positions: runs up to the last are joined"""
    from bundlesdf_amd import learn_ops as L
    N, V = (1 << 30) + 70001, 1 << 20
    ids, dout = torch.empty(N, dtype=torch.int32, device='cuda'), torch.empty(N, 1, device='cuda')
    for lo in range(0, N, 1 << 27):
        i = torch.arange(lo, min(lo + (1 << 27), N), device='cuda')
        ids[lo:lo + (1 << 27)] = i % V
        dout[lo:lo + (1 << 27), 0] = (i // V + i) % 7
    poisoned(V, 1, dtype=torch.float32)
    grad = L.embed_lookup_grad(dout, ids, V)
    v = torch.arange(V, device='cuda')
    want = torch.zeros(V, dtype=torch.int64, device='cuda')
    for k in range(-(-N // V)):
        want += torch.where(k * V + v < N, (k + k * V + v) % 7, 0)
    assert torch.equal(grad[:, 0].long(), want)                       # whole numbers below 2^24: exact in any order


@pytest.mark.parametrize('gdtype', [torch.float32, torch.bfloat16])
def test_gates_of_no_channel_have_no_gradient(nof, gdtype):
    from bundlesdf_amd import learn_ops as L
    B, T, G = 3, 700, 100
    gate, value = torch.ones(B, T, G, dtype=gdtype, device='cuda'), torch.ones(B, T, 0, dtype=torch.bfloat16, device='cuda')
    h, last, marks = L.gated_scan(gate, value, want_marks=True)
    assert h.shape == (B, T, 0) and last.shape == (B, 0)
    poisoned(B, T, G, dtype=gdtype)
    dgate, dvalue, dstate = L.gated_scan_grad(gate, value, value, marks=marks)
    assert dgate.shape == gate.shape and dgate.dtype == gdtype and (dgate == 0).all()
    assert dvalue.shape == value.shape and dstate.shape == (B, 0)
