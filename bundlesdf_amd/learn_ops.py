"""Learning operators on device tensors (csrc/nof_embed.hip, nof_scan.hip, nof_ortho.hip; the last section of include/nof_hip.h): what
a field with learnt codes, blended features and matrix-shaped weights trains with, next to the hash grid, the SDF compositing and Adam.

    embed_lookup, embed_lookup_grad        rows of a table by id, scaled; the table's gradient summed in a fixed order
    gated_scan, gated_scan_grad, gated_scan_step
                                           h[t] = gate[t] h[t-1] + value[t] along samples or tokens; its gradients; one step of it
    orthogonalize                          the orthogonalised update of weight matrices (Newton-Schulz products on MFMA)

Like the rest of the framework they are explicit forward and backward calls, launched on torch's current stream of the tensors'
device, without a host synchronisation: every one can be captured into a graph.  Tensors are float32, bfloat16 or float16; sums, states
and norms are float32 or wider and a result is rounded to its type once.  They record no autograd history -- a tensor that would need it
is refused -- and they raise lib.NofError on anything they do not take; there is no fallback.
"""
import torch

from . import lib
from .lib import NofError

_TYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}        # NOF_TYPE_*
_INT64 = {torch.int32: 0, torch.int64: 1}


def _need(ok, what):
    if not ok:
        raise NofError(what)


def _on_device(what, *tensors):
    """one CUDA device for all of them, no autograd history lost"""
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise NofError(f'{what}: tensors must be on the GPU')
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise NofError(f'{what}: tensors are on different devices ({dev}, {t.device})')
        if t.requires_grad and torch.is_grad_enabled():
            raise NofError(f'{what} records no autograd history: call it under torch.no_grad() or with detached tensors, '
                           'and its gradient function for the gradients')
    return dev


def _call(dev, name, *args):
    """the C call on the current stream of `dev`, whichever device is current"""
    if dev.index == torch.cuda.current_device():
        lib.call(name, *args)
    else:
        with torch.cuda.device(dev):
            lib.call(name, *args)


def _rows(x):
    """x [N, D] with its elements side by side in a row: (tensor, elements between rows)"""
    if x.shape[1] > 1 and x.stride(1) != 1:
        x = x.contiguous()
    return x, x.stride(0) if x.shape[0] > 1 else x.shape[1]


# ---- rows of a table ------------------------------------------------------------------------------------------------------------------
def embed_lookup(table, ids, scale=1.0):
    """table [V, D], ids int32 or int64 of any shape -> scale * table[ids], [*ids.shape, D] in the table's type.  An id outside [0, V)
    -- padding, a ray without a frame -- gives zeros."""
    _need(table.dim() == 2 and table.dtype in _TYPE, 'embed_lookup: table must be [V, D] float32, bfloat16 or float16')
    _need(ids.dtype in _INT64, 'embed_lookup: ids must be int32 or int64')
    dev = _on_device('embed_lookup', table, ids)
    table, stride = _rows(table)
    ids = ids.contiguous()
    V, D = table.shape
    out = torch.empty((*ids.shape, D), dtype=table.dtype, device=dev)
    _call(dev, 'nof_embed_fwd', table.data_ptr(), stride, _TYPE[table.dtype], ids, _INT64[ids.dtype], float(scale), out, ids.numel(), V, D)
    return out


def embed_lookup_grad(dout, ids, n_rows, scale=1.0):
    """The gradient of embed_lookup's table: dout [*ids.shape, D] -> [n_rows, D] in dout's type, row v = scale * the sum of dout where
    ids = v (zeros where nobody asks for v; ids outside [0, n_rows) contribute nothing).  The sum's order depends on the ids alone:
    equal inputs give equal bits."""
    n_rows = int(n_rows)
    _need(dout.dtype in _TYPE, 'embed_lookup_grad: dout must be float32, bfloat16 or float16')
    _need(ids.dtype in _INT64, 'embed_lookup_grad: ids must be int32 or int64')
    _need(dout.dim() >= 1 and dout.shape[:-1] == ids.shape, 'embed_lookup_grad: dout must be [*ids.shape, D]')
    _need(0 <= n_rows < 1 << 30, 'embed_lookup_grad: n_rows must be in [0, 2^30)')
    dev = _on_device('embed_lookup_grad', dout, ids)
    N, D = ids.numel(), dout.shape[-1]
    dout, stride = _rows(dout.reshape(N, D))
    ids = ids.contiguous()
    grad = torch.empty((n_rows, D), dtype=dout.dtype, device=dev)
    nbytes = lib.load().nof_embed_bwd_workspace_bytes(N, n_rows, D)
    _need(nbytes >= 0, f'embed_lookup_grad: sizes out of range (N = {N}, n_rows = {n_rows}, D = {D})')
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _call(dev, 'nof_embed_bwd', dout.data_ptr(), stride, _TYPE[dout.dtype], ids, _INT64[ids.dtype], float(scale), grad, ws, nbytes, N, n_rows, D)
    return grad
