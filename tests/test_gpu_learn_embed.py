"""Row lookup with scaling and its gradient by sorted ids (bundlesdf_amd/learn_ops.py) against plain sums in 64 bits.

Tolerances: the lookup is a product of two binary32 values rounded to the tensor's type, at most once on the way (the compiler may fuse
the product and the rounding to 16 bits, which drops the first): off by at most 2^-24 + eps/2 of the product, relative.  An own first
form of this check asked for the bits of two roundings in a row, which the fused form need not give: near a tie of the 16-bit type the
binary32 rounding moves the product onto the tie.  A gradient row is
a sum of n terms in binary32 (each addition off by at most 2^-24 of the partial sum, itself at most the sum of the terms' magnitudes),
times scale (a rounding of scale, one of the product), rounded once to the tensor's type: (n + 2) 2^-24 * scale * sum|dout| + eps/2 |row|."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make_ids(kind, N, V, dtype, rng):
    if kind == 'same':
        ids = np.full(N, V // 2)
    elif kind == 'random':
        ids = rng.integers(0, V, N)
    elif kind == 'skewed':                                        # a few ids hold most positions
        ids = np.minimum((V ** rng.random(N)).astype(np.int64), V) - 1
    else:                                                         # 'absent': ids outside the table among them
        ids = rng.integers(0, V, N)
        bad = rng.random(N) < 0.4
        far = np.array([-1, V, -2 ** 31, 2 ** 31 - 1] if dtype == torch.int32 else [-1, V, 2 ** 40, -2 ** 40, 2 ** 32])
        ids = np.where(bad, far[rng.integers(0, len(far), N)], ids)
    return torch.from_numpy(ids.astype(np.int64)).to(dtype)


def check_grad(got, dout, ids, V, scale):
    d, i = dout.double().cpu(), ids.long().cpu().reshape(-1)
    there = (i >= 0) & (i < V)
    d, i = d.reshape(len(i), got.shape[1])[there], i[there]
    want = torch.zeros(V, d.shape[1], dtype=torch.float64).index_add_(0, i, d) * scale
    mag = torch.zeros(V, d.shape[1], dtype=torch.float64).index_add_(0, i, d.abs()) * abs(scale)
    n = torch.bincount(i, minlength=V)[:, None].double()
    tol = (n + 2) * 2.0 ** -24 * mag + torch.finfo(got.dtype).eps / 2 * want.abs()
    if got.dtype == torch.float16:
        tol += 2.0 ** -25                                         # half the spacing of the type's subnormals
    assert got.shape == want.shape
    bad = (got.double().cpu() - want).abs() > tol * (1 + 1e-6)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4])


@pytest.mark.parametrize('N,V,D', [(0, 5, 3), (1, 1, 1), (1, 1000, 2048), (63, 2, 2), (65, 33, 3), (1000, 7, 16), (4096, 64, 16), (4096, 70000, 5),
                                   (4097, 1023, 8), (4097, 1024, 100), (20000, 3, 1), (9000, 40000, 1001), (70001, 1050000, 2), (8192, 300, 2056),
                                   (200000, 1, 4), (300, 50, 8200)])
@pytest.mark.parametrize('kind', ['same', 'random', 'skewed', 'absent'])
def test_lookup_and_gradient(nof, N, V, D, kind):
    from bundlesdf_amd import learn_ops as L
    rng = np.random.default_rng(N + V + D)
    k = ['same', 'random', 'skewed', 'absent'].index(kind) + N + D
    dtype, idt = TYPES[k % 3], (torch.int32, torch.int64)[k % 2]
    ids = make_ids(kind, N, V, idt, rng).cuda()
    gen = torch.Generator(device='cuda').manual_seed(k)
    table = torch.randn(V, D, device='cuda', generator=gen).to(dtype)
    dout = torch.randn(N, D, device='cuda', generator=gen).to(dtype)
    scale = 1.7
    out = L.embed_lookup(table, ids, scale)
    i = ids.long()
    there = ((i >= 0) & (i < V))[:, None]
    want = torch.where(there, table[torch.where(there[:, 0], i, 0 * i)].double() * float(np.float32(scale)), 0.0)
    fine = (out.double() - want).abs() <= (2.0 ** -24 + torch.finfo(dtype).eps / 2) * want.abs() * (1 + 1e-6) + (2.0 ** -25 if dtype == torch.float16 else 0)
    assert out.dtype == dtype and out.shape == want.shape and fine.all()
    assert (out[~there[:, 0]] == 0).all()
    grad = L.embed_lookup_grad(dout, ids, V, scale)
    check_grad(grad, dout, ids, V, scale)
    for _ in range(3):
        assert torch.equal(grad, L.embed_lookup_grad(dout, ids, V, scale))      # the same bits every time


def test_gradient_against_differences(nof):
    """d sum(w * lookup) / d table, by steps of the table (the lookup is linear: the step's size does not matter)"""
    from bundlesdf_amd import learn_ops as L
    gen = torch.Generator(device='cuda').manual_seed(4)
    table = torch.randn(6, 5, device='cuda', generator=gen)
    ids = torch.tensor([3, 3, -1, 0, 5, 3, 6, 1], device='cuda')
    w = torch.randn(8, 5, device='cuda', generator=gen)
    grad = L.embed_lookup_grad(w, ids, 6, 0.5)
    for r in range(6):
        for c in range(5):
            up, down = table.clone(), table.clone()
            up[r, c] += 4.0
            down[r, c] -= 4.0
            diff = ((L.embed_lookup(up, ids, 0.5).double() - L.embed_lookup(down, ids, 0.5).double()) * w.double()).sum() / 8.0
            assert abs(float(diff) - float(grad[r, c])) < 1e-5


@pytest.mark.parametrize('dtype', TYPES)
def test_strides_and_alignment(nof, dtype):
    """rows apart, rows that start off every vector's border, a transposed table, one row read by all (stride 0), ids of two dimensions"""
    from bundlesdf_amd import learn_ops as L
    gen = torch.Generator(device='cuda').manual_seed(1)
    big = torch.randn(300, 67, device='cuda', generator=gen).to(dtype)
    ids = torch.randint(0, 300, (7, 11), device='cuda', generator=gen)
    for table in (big, big[:, 1:65], big[:, 3:], big[::2][:, :64], big.t().contiguous().t(), big[:1].expand(300, 67)):
        V = table.shape[0]
        assert torch.equal(L.embed_lookup(table, ids % V, 1.0), table[ids % V])
        d = table[(ids * 7) % V].reshape(7, 11, -1)
        for dout in (d, d.transpose(0, 1).contiguous().transpose(0, 1), d[:, :1].expand_as(d)):
            check_grad(L.embed_lookup_grad(dout, ids % V, V, 2.0), dout.reshape(77, -1), (ids % V).reshape(-1), V, 2.0)
    flat = torch.randn(64 * 40 + 1, device='cuda', generator=gen).to(dtype)[1:].view(40, 64)       # the whole table off the border
    assert torch.equal(L.embed_lookup(flat, ids % 40, 1.0), flat[ids % 40])


def test_values_that_are_not_finite_stay_in_their_rows(nof):
    from bundlesdf_amd import learn_ops as L
    ids = torch.tensor([1, 2, 2, -1, 4], device='cuda')
    dout = torch.ones(5, 8, device='cuda')
    dout[2, 0], dout[3, 1], dout[4, 2] = float('inf'), float('nan'), float('-inf')      # row 3 is absent: its NaN reaches nobody
    grad = L.embed_lookup_grad(dout, ids, 5, 1.0)
    want = torch.zeros(5, 8, device='cuda')
    want[1], want[2], want[4] = 1.0, 2.0, 1.0
    want[2, 0], want[4, 2] = float('inf'), float('-inf')
    assert torch.equal(grad, want)


def test_stream_and_graph(nof):
    """on a stream of its own, and captured: every replay on new inputs gives the eager call's bits"""
    from bundlesdf_amd import learn_ops as L
    gen = torch.Generator(device='cuda').manual_seed(2)
    ids = torch.randint(-1, 900, (6000,), device='cuda', generator=gen)
    dout = torch.randn(6000, 24, device='cuda', generator=gen)
    want = L.embed_lookup_grad(dout, ids, 900, 1.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = L.embed_lookup_grad(dout, ids, 900, 1.0)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = L.embed_lookup(want, ids, 0.5)
        grad = L.embed_lookup_grad(dout, ids, 900, 1.0)
    for _ in range(4):
        ids.copy_(torch.randint(-1, 900, (6000,), device='cuda', generator=gen))
        dout.normal_(generator=gen)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(grad, L.embed_lookup_grad(dout, ids, 900, 1.0)) and torch.equal(out, L.embed_lookup(want, ids, 0.5))


def test_offsets_past_32_bits(nof):
    """a table and a gradient of more than 2^32 bytes and 2^31 elements"""
    from bundlesdf_amd import learn_ops as L
    V, D = 1100000, 2048
    table = torch.empty(V, D, dtype=torch.bfloat16, device='cuda')
    ids = torch.tensor([V - 1, 0, V - 2, V // 2, V - 1, -1, V], device='cuda')
    gen = torch.Generator(device='cuda').manual_seed(0)
    rows = torch.randn(7, D, device='cuda', generator=gen).to(torch.bfloat16)
    table[ids[:4]] = rows[:4]
    out = L.embed_lookup(table, ids)
    assert torch.equal(out[:4], rows[:4]) and torch.equal(out[4], rows[0]) and (out[5:] == 0).all()
    del table
    grad = L.embed_lookup_grad(rows, ids, V)
    assert torch.equal(grad[V - 1], (rows[0].float() + rows[4].float()).to(torch.bfloat16)) and torch.equal(grad[V - 2], rows[2])
    grad[ids[:4]] = 0
    assert all(int(torch.count_nonzero(part)) == 0 for part in grad.split(1 << 17))


def big_of(V, D, N, dtype, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    return torch.randn(N, D, device='cuda', generator=gen).to(dtype), gen


@pytest.mark.parametrize('N,V,D', [(4096, 4096, 32), (4096, 4097, 32), (4096, 64, 33), (4097, 64, 16), (257, 300, 9), (1, 19000, 33), (63, 5, 1001), (2049, 2, 24),
                                   (1000, 40000, 16), (4000, 90000, 40)])
@pytest.mark.parametrize('kind', ['same', 'random', 'skewed', 'absent'])
def test_the_gradient_on_either_side_of_one_launch(nof, N, V, D, kind):
    """few positions of few rows are added in one launch, others sorted: either side of the border, at odd sizes, rows apart, ids and dout not finite"""
    from bundlesdf_amd import learn_ops as L
    rng = np.random.default_rng(N * 3 + V + D)
    for q, dtype in enumerate(TYPES):
        ids = make_ids(kind, N, V, (torch.int32, torch.int64)[(q + N) % 2], rng).cuda()
        dout, _ = big_of(V, D + 3, N, dtype, q)
        for d in (dout[:, 3:], dout[:1, :D].expand(N, D)):
            grad = L.embed_lookup_grad(d, ids, V, -0.3)
            check_grad(grad, d, ids, V, -0.3)
            assert torch.equal(grad, L.embed_lookup_grad(d.clone(), ids, V, -0.3))
        inside = ids.long().clamp(-1, V)
        dout[N // 2, :] = float('nan')
        grad = L.embed_lookup_grad(dout[:, :D], ids, V)
        hit = torch.zeros(V + 2, dtype=torch.bool, device='cuda')
        hit[inside[N // 2] + 1] = True
        assert torch.equal(grad.isnan().any(1), hit[1:V + 1])                      # in the row that it is added to, and there alone


def test_one_launch_captured(nof):
    from bundlesdf_amd import learn_ops as L
    dout, gen = big_of(40, 20, 700, torch.bfloat16, 3)
    ids = torch.randint(-1, 41, (700,), device='cuda', generator=gen)
    L.embed_lookup_grad(dout, ids, 40)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        grad = L.embed_lookup_grad(dout, ids, 40, 2.0)
    for _ in range(4):
        ids.copy_(torch.randint(-1, 41, (700,), device='cuda', generator=gen))
        dout.normal_(generator=gen)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(grad, L.embed_lookup_grad(dout, ids, 40, 2.0))
        check_grad(grad, dout, ids, 40, 2.0)


@pytest.mark.parametrize('N,V,D', [(5000, 60000, 1000), (300, 30000, 1001), (4999, 131000, 7)])
def test_rows_that_nobody_names_are_zeros_wherever_they_lie(nof, N, V, D):
    """a table larger than the stretch that the sort's launches clear, over memory that held something else"""
    from bundlesdf_amd import learn_ops as L
    for q, dtype in enumerate(TYPES):
        dout, gen = big_of(V, D, N, dtype, 7 + q)
        ids = torch.randint(-1, V, (N,), device='cuda', generator=gen)
        ids[:N // 3] = V - 1
        stale = torch.full((V, D), float('nan'), dtype=dtype, device='cuda')
        del stale
        grad = L.embed_lookup_grad(dout, ids, V, 0.5)
        named = torch.zeros(V, dtype=torch.bool, device='cuda')
        named[ids[ids >= 0]] = True
        assert not grad[~named].any() and not grad.isnan().any()
        rows = torch.unique(ids[ids >= 0])
        check_grad(grad[rows], dout[ids >= 0], torch.searchsorted(rows, ids[ids >= 0]), len(rows), 0.5)
