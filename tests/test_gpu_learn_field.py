"""The orthogonalised update on the field's own weight matrices, by the hook that a training step calls between its backward and Adam: matrices
move by it, everything else by Adam, and the next step runs on the new weights."""
import numpy as np
import pytest
import torch

from tests import util as U
from tests.test_gpu_step import _pair

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('precision,hidden', [('fp32', 64), ('bf16', 64), ('bf16', 128)])
def test_matrices_of_the_field(nof, precision, hidden):
    from bundlesdf_amd import learn_ops as L
    cfg, fld, _, batch, rng = _pair(nof, precision, hidden=hidden)
    R = batch.shape[0]
    u = [U.dev(rng.random((R, cfg[k])).astype(np.float32)) for k in ('N_samples', 'N_samples_around_depth')]
    momentum = [torch.zeros(o, i, device='cuda') for o, i in fld.layer_dims]
    seen = []

    def orthogonal(grads):
        weights, g = fld.mlp, grads[fld.n_table:fld.n_table + fld.n_mlp]
        seen.append((grads.clone(), fld.params.clone()))
        for l, (o, i) in enumerate(fld.layer_dims):
            at = slice(fld.desc.w_off[l], fld.desc.w_off[l] + o * i)
            momentum[l].mul_(0.95).add_(g[at].view(o, i))
            weights[at].view(o, i).sub_(L.orthogonalize(momentum[l]), alpha=0.01)
            g[at].zero_()

    expected = [torch.zeros(o, i, device='cuda') for o, i in fld.layer_dims]
    lr = fld.learning_rates()[0]
    for step in range(3):
        fld.train_step(U.dev(batch), None, R, *u, grad_sync=orthogonal)
        torch.cuda.synchronize()
        grads, before = seen[-1]
        assert len(seen) == step + 1 and torch.isfinite(fld.params).all()
        moved = torch.zeros(fld.n_mlp, dtype=torch.bool, device='cuda')
        for l, (o, i) in enumerate(fld.layer_dims):
            lo = fld.desc.w_off[l]
            moved[lo:lo + o * i] = True
            at = slice(fld.n_table + lo, fld.n_table + lo + o * i)
            expected[l].mul_(0.95).add_(grads[at].view(o, i))
            want = before[at].view(o, i) - 0.01 * L.orthogonalize(expected[l])
            assert float(grads[at].abs().max()) > 0.0
            assert float((fld.params[at].view(o, i) - want).abs().max()) <= 2.0 ** -22 * float(want.abs().max() + 0.1), (step, l)       # two roundings
        if step == 0:                                                     # Adam's first step: lr times the gradient's sign
            for lo, g, p, q in ((0, *(x[:fld.n_table] for x in (grads, before, fld.params))),
                                (fld.n_table, *(x[fld.n_table:fld.n_table + fld.n_mlp][~moved] for x in (grads, before, fld.params)))):
                clear = g.abs() > 1e-9
                assert clear.any() and float((q - (p - lr * g.sign()))[clear].abs().max()) <= 1e-5 * lr + 2.0 ** -23 * float(p.abs().max()), lo
        assert float(fld.grads.abs().max()) == 0.0
    # the next step's forward is that of a field that is given these parameters
    other = _pair(nof, precision, hidden=hidden)[1]
    other.load_parameters(table=fld.table, mlp=fld.mlp, pose=fld.pose)
    for f in (fld, other):
        f.train_step(U.dev(batch), None, R, *u, do_step=False)
    a, b = fld.losses(), other.losses()
    assert all(a[k] == b[k] or abs(a[k] - b[k]) <= 1e-5 * abs(b[k]) for k in ('rgb_loss', 'sdf_loss', 'fs_loss')), (a, b)
