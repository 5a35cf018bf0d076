"""Learning operators on device tensors (csrc/nof_embed.hip, nof_scan.hip, nof_ortho.hip; the last section of include/nof_hip.h): what
a field with learnt codes, blended features and matrix-shaped weights trains with, next to the hash grid, the SDF compositing and Adam.

    embed_lookup, embed_lookup_grad        rows of a table by id, scaled; the table's gradient summed in a fixed order
    gated_scan, gated_scan_grad, gated_scan_step
                                           h[t] = gate[t] h[t-1] + value[t] along samples or tokens; its gradients; one step of it
    orthogonalize                          the orthogonalised update of weight matrices (Newton-Schulz products on MFMA)

Like the rest of the framework they are explicit forward and backward calls, launched on torch's current stream of the tensors'
device, without a host synchronisation: every one can be captured into a graph.  Tensors are float32, bfloat16 or float16; sums, states
and norms are float32 or wider and a result is rounded to its type once.  They record no autograd history and carry no tangents -- a tensor
that would need either is refused -- and they raise lib.NofError on anything they do not take; there is no fallback.
"""
import ctypes as C
import functools

import torch
from torch.autograd import forward_ad

from . import lib
from .lib import NofError

_TYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}        # NOF_TYPE_*
_INT64 = {torch.int32: 0, torch.int64: 1}


def _on_device(what, *tensors):
    """the index of the one CUDA device of all of them; no autograd history lost.  (These run a few times per call that takes a few
    microseconds on the GPU: plain loops, integers.)"""
    dev = -2
    for t in tensors:
        if t is None:
            continue
        d = t.get_device()
        if d != dev:
            if d < 0:
                raise NofError(f'{what}: tensors must be on the GPU')
            if dev >= 0:
                raise NofError(f'{what}: tensors are on different devices (cuda:{dev}, cuda:{d})')
            dev = d
        if t.requires_grad and torch.is_grad_enabled():
            raise NofError(f'{what} records no autograd history: call it under torch.no_grad() or with detached tensors, '
                           'and its gradient function for the gradients')
        if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
            raise NofError(f'{what} carries no forward-mode tangents: call it with the primal tensors')
    return dev


_fn = {}
_device = getattr(torch._C, '_cuda_getDevice', None) or torch.cuda.current_device
_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None) or (lambda dev: torch.cuda.current_stream(dev).cuda_stream)     # (no Stream object)


def _call(dev, name, *args):
    """the C call (addresses and numbers) on the current stream of device `dev`, whichever device is current"""
    fn = _fn.get(name)
    if fn is None:
        fn = _fn[name] = getattr(lib.load(), name)
    if dev == _device():
        rc = fn(*args, _stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _stream(dev))
    if rc != 0:
        raise NofError(f'{name} failed with code {rc}: {lib.load().nof_last_error().decode()}')


def _at(x):
    return None if x is None else x.data_ptr()


def _apart(a, b):
    """whether two contiguous tensors share no memory, or all of it (same start, same length)"""
    n, m = a.numel() * a.element_size(), b.numel() * b.element_size()
    x, y = a.data_ptr(), b.data_ptr()
    return x + n <= y or y + m <= x or (x == y and n == m) or n == 0 or m == 0


def _clear_of(lo, hi, D, x, at, row):
    """whether what is written to a contiguous [B, D] float32 at the addresses lo to hi cannot be read from x [B, C], `row` elements between rows,
    by another lane: x lies apart, or each element of it is the written one's own"""
    if hi <= at or lo == hi:
        return True
    rows, cols = x.shape
    if at + ((rows - 1) * row + cols) * x.element_size() <= lo or cols == 0:
        return True
    return at == lo and cols == D and x.dtype == torch.float32 and rows * D * 4 == hi - lo and (row == D or rows == 1)


def _rows(x):
    """x [N, D] with its elements side by side in a row: (tensor, elements between rows)"""
    if x.is_neg():                                                       # (a view like z.conj().imag holds the other sign)
        x = x.resolve_neg()
    if x.shape[1] > 1 and x.stride(1) != 1:
        x = x.contiguous()
    return x, x.stride(0) if x.shape[0] > 1 else x.shape[1]


@functools.lru_cache(maxsize=1024)
def _bytes(name, *sizes):
    """a size query of the library: of the sizes alone"""
    n = getattr(lib.load(), name)(*sizes)
    if not (n >= 0):
        raise NofError(f'{name}: sizes out of range {sizes}')
    return n


def _scratch(like, nbytes):
    return like.new_empty(nbytes, dtype=torch.uint8) if nbytes else None


# ---- rows of a table ------------------------------------------------------------------------------------------------------------------
def embed_lookup(table, ids, scale=1.0):
    """table [V, D], ids int32 or int64 of any shape -> scale * table[ids], [*ids.shape, D] in the table's type.  An id outside [0, V)
    -- padding, a ray without a frame -- gives zeros."""
    if not (table.dim() == 2 and table.dtype in _TYPE):
        raise NofError('embed_lookup: table must be [V, D] float32, bfloat16 or float16')
    if not (ids.dtype in _INT64):
        raise NofError('embed_lookup: ids must be int32 or int64')
    dev, scale = _on_device('embed_lookup', table, ids), float(scale)
    table, stride = _rows(table)
    ids = ids.contiguous()
    V, D = table.shape
    out = table.new_empty((*ids.shape, D))
    _call(dev, 'nof_embed_fwd', table.data_ptr(), stride, _TYPE[table.dtype], ids.data_ptr(), _INT64[ids.dtype], scale, out.data_ptr(), ids.numel(), V, D)
    return out


def embed_lookup_grad(dout, ids, n_rows, scale=1.0):
    """The gradient of embed_lookup's table: dout [*ids.shape, D] -> [n_rows, D] in dout's type, row v = scale * the sum of dout where
    ids = v (zeros where nobody asks for v; ids outside [0, n_rows) contribute nothing).  The sum's order depends on the ids alone:
    equal inputs give equal bits."""
    n_rows = int(n_rows)
    if not (dout.dtype in _TYPE):
        raise NofError('embed_lookup_grad: dout must be float32, bfloat16 or float16')
    if not (ids.dtype in _INT64):
        raise NofError('embed_lookup_grad: ids must be int32 or int64')
    if not (dout.dim() >= 1 and dout.shape[:-1] == ids.shape):
        raise NofError('embed_lookup_grad: dout must be [*ids.shape, D]')
    if not (0 <= n_rows < 1 << 30):
        raise NofError('embed_lookup_grad: n_rows must be in [0, 2^30)')
    dev, scale = _on_device('embed_lookup_grad', dout, ids), float(scale)
    N, D = ids.numel(), dout.shape[-1]
    dout, stride = _rows(dout.reshape(N, D))
    ids = ids.contiguous()
    grad = dout.new_empty((n_rows, D))
    nbytes = _bytes('nof_embed_bwd_workspace_bytes', N, n_rows, D)
    ws = _scratch(dout, nbytes)
    _call(dev, 'nof_embed_bwd', dout.data_ptr(), stride, _TYPE[dout.dtype], ids.data_ptr(), _INT64[ids.dtype], scale, grad.data_ptr(), _at(ws), nbytes,
          N, n_rows, D)
    return grad


# ---- gated recurrence along time ------------------------------------------------------------------------------------------------------
def _scan_even(dtype, D, G):
    """whether the kernels take two channels per lane (csrc/nof_scan.hip: scan_vec)"""
    return dtype != torch.float32 and (D if G == D else D // G) % 2 == 0


def _scan_strided(x, even):
    """x [B, T, C] (or [B, C]) as the kernels take it -- channels side by side, two-channel loads on their border -- and its strides"""
    if x.is_neg():
        x = x.resolve_neg()
    if x.is_contiguous():
        n = x.shape
        st = (n[1],) if len(n) == 2 else (n[1] * n[2], n[2])
        if not even or x.data_ptr() % (2 * x.element_size()) == 0:         # (even: so are the strides)
            return x, st
        return x.clone(), st
    st = x.stride()
    if st[-1] != 1 and x.shape[-1] > 1:
        x = x.contiguous()
        st = x.stride()
    st = tuple([s if n > 1 else 0 for s, n in zip(st[:-1], x.shape)])
    if even and (x.data_ptr() % (2 * x.element_size()) or any([s % 2 for s in st])):
        x = x.clone(memory_format=torch.contiguous_format)
        st = tuple([s if n > 1 else 0 for s, n in zip(x.stride()[:-1], x.shape)])
    return x, st


def _flat(x, even):
    """a [B, D] float32 argument as the kernels take it, or None"""
    if x is None:
        return None
    if x.is_neg():
        x = x.resolve_neg()
    if not x.is_contiguous():
        x = x.contiguous()
    return x.clone() if even and x.data_ptr() % 8 else x


def _state_ok(what, name, x, B, D):
    if not (x is None or (x.dtype == torch.float32 and x.shape == (B, D))):
        raise NofError(f'{what}: {name} must be [B, D] float32')


def _scan_args(what, gate, value, lengths, dims):
    vs, gs = value.shape, gate.shape
    if len(vs) != dims or value.dtype not in _TYPE:
        raise NofError(f'{what}: value must be [{"B, T, D" if dims == 3 else "B, D"}] float32, bfloat16 or float16')
    if not (len(gs) == dims and gs[:-1] == vs[:-1]):
        raise NofError(f"{what}: gate must have value's shape but for the channels")
    if not (gate.dtype is value.dtype or gate.dtype is torch.float32):
        raise NofError(f"{what}: gate must be float32 or of value's type")
    D, G = vs[-1], gs[-1]
    if not (D == 0 or (G > 0 and D % G == 0)):
        raise NofError(f'{what}: the number of gates per position must divide the number of channels')
    if not (D <= 1 << 20 and vs[0] < 1 << 24 and (dims == 2 or vs[1] < 1 << 31)):
        raise NofError(f'{what}: sizes out of range')
    if lengths is not None:
        if not (lengths.dtype == torch.int32 and lengths.shape == vs[:1]):
            raise NofError(f'{what}: lengths must be [B] int32')
    return D, G


def gated_scan(gate, value, state=None, lengths=None, reverse=False, want_marks=False):
    """h[:, t] = gate[:, t] * h[:, t-1] + value[:, t] with h[:, -1] = state (None: zeros) -> (h [B, T, D] in value's type, the last h
    [B, D] float32), and with want_marks the float32 states that gated_scan_grad starts from.

    gate [B, T, G] (value's type or float32), value [B, T, D]; G divides D: channel d uses gate d // (D // G) -- G = D is a gate per
    channel, G = 1 one for all.  lengths [B] int32: rows from lengths[b] on do not exist (not read; zeros in h).  reverse: from the last
    existing row to the first -- with gate = 1 - opacity and value = opacity * feature, h[:, 0] is the ray's blend, back to front.
    Gates compose over positions in float32: their products must stay in its range (|gate| <= 1 always does).  Behind an infinity a channel
    is infinite or NaN (a product of gates that has become zero meets it)."""
    D, G = _scan_args('gated_scan', gate, value, lengths, 3)
    B, T = value.shape[:2]
    _state_ok('gated_scan', 'state', state, B, D)
    dev = _on_device('gated_scan', gate, value, state, lengths)
    return _scan_forward(dev, gate, value, state, lengths, reverse, want_marks, True)


def _scan_forward(dev, gate, value, state, lengths, reverse, want_marks, want_h):
    B, T, D = value.shape
    G, dt = gate.shape[-1], value.dtype
    even, ty = _scan_even(dt, D, G), _TYPE[dt]
    (value, vst), (gate, gst), state = _scan_strided(value, even), _scan_strided(gate, even and G == D), _flat(state, even)
    lengths = lengths.contiguous() if lengths is not None else None
    h = value.new_empty((B, T, D)) if want_h else None
    last = value.new_empty((B, D), dtype=torch.float32) if want_h else None
    marks = value.new_empty(_bytes('nof_gated_scan_marks_bytes', B, T, D, G, ty) // 4, dtype=torch.float32) if want_marks else None
    nbytes = _bytes('nof_gated_scan_workspace_bytes', B, T, D, G, ty)
    ws = _scratch(value, nbytes)
    _call(dev, 'nof_gated_scan_fwd', gate.data_ptr(), *gst, _TYPE[gate.dtype], value.data_ptr(), *vst, ty, _at(state), _at(lengths),
          1 if reverse else 0, _at(h), _at(last), _at(marks), _at(ws), nbytes, B, T, D, G)
    return (h, last, marks) if want_marks else (h, last)


def gated_scan_grad(gate, value, dh, dlast=None, state=None, marks=None, lengths=None, reverse=False):
    """The gradients of gated_scan: dh [B, T, D] and dlast [B, D] float32 (None: zeros) are the loss's gradients of its two results; the
    other arguments are the forward's.  -> (dgate in gate's type, summed over the channels that share it, dvalue, dstate [B, D] float32).
    marks: what gated_scan(..., want_marks=True) gave for the same gate, value, state, lengths and reverse; None recomputes them."""
    D, G = _scan_args('gated_scan_grad', gate, value, lengths, 3)
    B, T = value.shape[:2]
    dt = value.dtype
    if not (dh.shape == value.shape and dh.dtype == dt):
        raise NofError("gated_scan_grad: dh must have value's shape and type")
    _state_ok('gated_scan_grad', 'state', state, B, D)
    _state_ok('gated_scan_grad', 'dlast', dlast, B, D)
    if marks is not None:
        if not (marks.dtype == torch.float32 and marks.dim() == 1 and marks.numel() * 4 == _bytes('nof_gated_scan_marks_bytes', B, T, D, G, _TYPE[dt])):
            raise NofError('gated_scan_grad: marks are not those of a forward pass of these sizes')
    dev = _on_device('gated_scan_grad', gate, value, dh, dlast, state, marks, lengths)
    if marks is None:
        marks = _scan_forward(dev, gate, value, state, lengths, reverse, True, False)[2]
    even, ty = _scan_even(dt, D, G), _TYPE[dt]
    (value, vst), (gate, gst), (dh, dst) = _scan_strided(value, even), _scan_strided(gate, even and G == D), _scan_strided(dh, even)
    dlast, marks = _flat(dlast, even), _flat(marks, even)
    lengths = lengths.contiguous() if lengths is not None else None
    if D == 0:                                                            # no channel shares the gates
        return gate.new_zeros((B, T, G)), value.new_empty((B, T, 0)), value.new_empty((B, 0), dtype=torch.float32)
    dgate, dvalue, dstate = gate.new_empty((B, T, G)), value.new_empty((B, T, D)), value.new_empty((B, D), dtype=torch.float32)
    nbytes = _bytes('nof_gated_scan_workspace_bytes', B, T, D, G, ty)
    ws = _scratch(value, nbytes)
    _call(dev, 'nof_gated_scan_bwd', gate.data_ptr(), *gst, _TYPE[gate.dtype], value.data_ptr(), *vst, ty, dh.data_ptr(), *dst, _at(dlast),
          marks.data_ptr(), _at(lengths), 1 if reverse else 0, dgate.data_ptr(), dvalue.data_ptr(), dstate.data_ptr(), _at(ws), nbytes, B, T, D, G)
    return dgate, dvalue, dstate


def gated_scan_step(gate, value, state, new_state=None):
    """One position of gated_scan: gate [B, G], value [B, D], state [B, D] float32 -> (h [B, D] in value's type, the new state).
    new_state: where the new state goes (`state` itself for an update in place, apart from gate and value); None allocates it."""
    D, G = _scan_args('gated_scan_step', gate, value, None, 2)
    B = value.shape[0]
    if not (state is not None):
        raise NofError('gated_scan_step: state must be [B, D] float32')
    _state_ok('gated_scan_step', 'state', state, B, D)
    _state_ok('gated_scan_step', 'new_state', new_state, B, D)
    dev = _on_device('gated_scan_step', gate, value, state, new_state)
    if not (new_state is None or (new_state.is_contiguous() and not new_state.is_neg())):
        raise NofError('gated_scan_step: new_state must be contiguous and no negated view')
    dt = value.dtype
    even = _scan_even(dt, D, G)
    (value, vst), (gate, gst), state = _scan_strided(value, even), _scan_strided(gate, even and G == D), _flat(state, even)
    gate_at, value_at = gate.data_ptr(), value.data_ptr()
    if new_state is None:
        new_state = state.new_empty((B, D))
        lo = new_state.data_ptr()
    else:
        lo = new_state.data_ptr()
        hi = lo + 4 * B * D
        if even and lo % 8:
            raise NofError('gated_scan_step: new_state must start on an 8-byte border')
        if state is not new_state and not _apart(new_state, state):
            raise NofError('gated_scan_step: new_state must be state itself or lie apart from it')
        if not (_clear_of(lo, hi, D, value, value_at, vst[0]) and _clear_of(lo, hi, D, gate, gate_at, gst[0])):
            raise NofError('gated_scan_step: new_state must lie apart from gate and value')
    h = value.new_empty((B, D))
    _call(dev, 'nof_gated_scan_step', gate_at, *gst, _TYPE[gate.dtype], value_at, *vst, _TYPE[dt], state.data_ptr(), lo, h.data_ptr(), B, D, G)
    return h, new_state


# ---- the orthogonalised update --------------------------------------------------------------------------------------------------------
QUINTIC = (3.4445, -4.7750, 2.0315)     # steep at 0 (a small singular value grows 3.4 times a step), within about [0.7, 1.2] from there on


@functools.lru_cache(maxsize=64)
def _coefficients(steps, coefficients):
    if not (1 <= steps <= 32):
        raise NofError('orthogonalize: steps must be in [1, 32]')
    flat = coefficients if len(coefficients) > 0 and isinstance(coefficients[0], (tuple, list)) else (coefficients,) * steps
    if not (len(flat) == steps and all(len(c) == 3 for c in flat)):
        raise NofError('orthogonalize: coefficients must be (a, b, c) or one such triple per step')
    return (C.c_float * (3 * steps))(*[float(x) for c in flat for x in c])


def orthogonalize(update, steps=5, coefficients=QUINTIC, eps=1e-30, out=None):
    """The orthogonalised form of weight updates [..., m, n]: X = update / max(|update|_F, eps), then `steps` times
    X <- (a + b A + c A A) X, A = X X^T (over the shorter side), with coefficients (a, b, c) -- one triple, or a tuple of `steps` of them.
    The singular vectors stay, the singular values go to the quintic's fixed band around 1.  Result in the update's type, in `out` (which
    may be `update`) where given.  Products hold their operands to 2^-23 of themselves or 2^-48 of the norm and add in
    binary32.  Equal calls give equal bits; how many matrices share a call may change a matrix's last bits.  Coefficients that let a singular
    value leave [0, 2] are refused."""
    if not (update.dim() >= 2 and update.dtype in _TYPE):
        raise NofError('orthogonalize: update must be [..., m, n] float32, bfloat16 or float16')
    m, n = update.shape[-2:]
    if not (m <= 16384 and n <= 16384):
        raise NofError('orthogonalize: m and n must be at most 16384')
    batch = update.shape[:-2].numel()
    if not (batch < 65536):
        raise NofError('orthogonalize: at most 65535 matrices')
    coef = _coefficients(int(steps), tuple(tuple(c) if isinstance(c, (tuple, list)) else c for c in coefficients))
    if not (out is None or (out.shape == update.shape and out.dtype == update.dtype and out.is_contiguous() and not out.is_neg())):
        raise NofError("orthogonalize: out must be contiguous, of update's shape and type and no negated view")
    dev = _on_device('orthogonalize', update, out)
    update = update.resolve_neg().contiguous()
    if out is None:
        out = update.new_empty(update.shape)
    elif not _apart(out, update):
        raise NofError('orthogonalize: out must be update itself or lie apart from it')
    nbytes = _bytes('nof_orthogonalize_workspace_bytes', batch, m, n)
    ws = _scratch(update, nbytes)
    _call(dev, 'nof_orthogonalize', update.data_ptr(), out.data_ptr(), _TYPE[update.dtype], int(steps), coef, float(eps), _at(ws), nbytes, batch, m, n)
    return out
