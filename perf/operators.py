"""The learning operators of bundlesdf_amd/learn_ops.py on their own: cases, inputs, the plain torch forms and the 64-bit values.

    embed   out[i] = scale * table[ids[i]] and, for training, the table's gradient (an id outside the table: a zero row, no gradient)
    scan    h[t] = gate[t] * h[t-1] + value[t] along the samples of a ray or the tokens of a sequence, its gradients, its single step
    ortho   the orthogonalised update of a weight matrix: five Newton-Schulz products of the normalised update

`run` computes them in elementary torch operations, or through the framework where `own` is true.
"""
import math

import torch

own = False

TYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
SIZE = {'fp32': 4, 'bf16': 2, 'fp16': 2}
NS = (3.4445, -4.7750, 2.0315)          # the quintic's coefficients: what an orthogonalised update commonly runs, five times


def _embed(name, mode, V, N, D, dtype, ids='int64', absent=0.0):
    return {'name': name, 'op': 'embed', 'mode': mode, 'V': V, 'N': N, 'D': D, 'dtype': dtype, 'ids': ids, 'absent': absent}


def _scan(name, mode, B, T, D, G, dtype, reverse=False, ragged=False, gate='same'):
    return {'name': name, 'op': 'scan', 'mode': mode, 'B': B, 'T': T, 'D': D, 'G': G, 'dtype': dtype, 'reverse': reverse,
            'ragged': ragged, 'gate': gate}


def _ortho(name, batch, m, n, dtype):
    return {'name': name, 'op': 'ortho', 'batch': batch, 'm': m, 'n': n, 'dtype': dtype}


def listed():
    return [
        # a learnt code per keyframe, gathered by the frame of each ray of a training batch; and its gradient
        _embed('embed frame codes', 'train', 64, 4096, 16, 'fp32', ids='int32'),
        # one position each of a few sequences being answered, a row length that no vector width divides
        _embed('embed single tokens', 'lookup', 50000, 32, 1001, 'fp16'),
        # a training batch of four sequences, a tenth of it padding
        _embed('embed training batch', 'train', 32768, 8192, 1024, 'bf16', absent=0.1),
        # a large vocabulary and a large batch
        _embed('embed large table', 'train', 131072, 65536, 2048, 'bf16'),
        # 16 feature channels blended back to front along the 192 samples of a batch's rays, one opacity per sample
        _scan('scan along rays', 'train', 4096, 192, 16, 1, 'fp32', reverse=True),
        # one token each of a batch being answered: state in, state out
        _scan('scan single tokens', 'step', 96, 1, 2048, 2048, 'bf16'),
        # prompts of different lengths (one empty) padded to the longest, eight heads with one gate each, going on from a state
        _scan('scan padded prompts', 'forward', 24, 1777, 520, 8, 'fp16', ragged=True, gate='fp32'),
        # few long sequences, a gate per channel
        _scan('scan long training', 'train', 4, 16384, 1024, 1024, 'bf16'),
        # the hidden matrices of the 128-wide networks
        _ortho('ortho field networks', 6, 128, 128, 'fp32'),
        # odd matrices, wider than tall
        _ortho('ortho odd', 3, 333, 1001, 'bf16'),
        # a tall matrix in full precision
        _ortho('ortho tall', 1, 4096, 1024, 'fp32'),
        # the largest matrix
        _ortho('ortho large', 1, 4096, 4096, 'bf16'),
    ]


def _between(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(('embed', 'scan', 'ortho'))
    dtype = rng.choice(('fp32', 'bf16', 'fp16'))
    if op == 'embed':
        mode = rng.choice(('lookup', 'train', 'train'))
        V, N, D = _between(rng, 16, 131072), _between(rng, 1, 65536), _between(rng, 1, 2048)
        cap = (1 << 28) // SIZE[dtype]
        c = _embed('', mode, min(V, cap // D), min(N, cap // 2 // D), D, dtype, rng.choice(('int32', 'int64')), rng.choice((0.0, 0.0, 0.2)))
    elif op == 'scan':
        mode = rng.choice(('step', 'forward', 'train', 'train'))
        B, T, D = _between(rng, 1, 4096), 1 if mode == 'step' else _between(rng, 1, 16384), _between(rng, 1, 4096)
        T = max(1, min(T, (1 << 26) // (B * D)))
        G = rng.choice((1, D, max(g for g in range(1, 17) if D % g == 0)))
        ragged = mode != 'step' and rng.random() < 0.4
        c = _scan('', mode, B, T, D, G, dtype, mode != 'step' and rng.random() < 0.5, ragged, rng.choice(('same', 'fp32')))
    else:
        m, n = _between(rng, 8, 4096), _between(rng, 8, 4096)
        most = max(1, int(2e11 / _ortho_flops(1, m, n)))
        c = _ortho('', min(most, _between(rng, 1, 16)), m, n, dtype)
    del c['name']
    return c


def _ortho_flops(batch, m, n):
    r, k = min(m, n), max(m, n)
    # X X^T and its square are symmetric: half of each is computed
    return batch * len(NS_STEPS) * (r * (r + 1) * k + r * (r + 1) * r + 2 * r * r * k)


NS_STEPS = range(5)


def work(case):
    c, s = case, SIZE[case['dtype']]
    if c['op'] == 'embed':
        i = 4 if c['ids'] == 'int32' else 8
        read = min(c['V'], c['N']) * c['D'] * s              # the rows looked up, each once
        b = c['N'] * (i + c['D'] * s) + read
        f = c['N'] * c['D']
        if c['mode'] == 'train':
            b += c['N'] * (i + c['D'] * s) + c['V'] * c['D'] * s
            f *= 3
        return {'bytes': b, 'flops': f}
    if c['op'] == 'scan':
        v = c['B'] * c['T'] * c['D']
        g = c['B'] * c['T'] * c['G'] * (4 if c['gate'] == 'fp32' else s)
        if c['ragged']:                                       # lengths spread evenly between none and all
            v, g = v // 2, g // 2
        st = c['B'] * c['D'] * 4
        b, f = g + 2 * v * s + 2 * st, 2 * v
        if c['mode'] == 'train':                              # backward: gate, value, dh in, dgate, dvalue out, the states' gradients
            b += 2 * g + 3 * v * s + 3 * st
            f += 4 * v
        return {'bytes': b, 'flops': f}
    return {'bytes': 2 * c['batch'] * c['m'] * c['n'] * s, 'flops': _ortho_flops(c['batch'], c['m'], c['n'])}


def prepare(case, seed):
    c, t = case, TYPES[case['dtype']]
    gen = torch.Generator(device='cuda').manual_seed(seed)

    def normal(*shape, dtype=t):
        return torch.randn(*shape, device='cuda', generator=gen).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, device='cuda', generator=gen)

    s = dict(c)
    if c['op'] == 'embed':
        # tokens are distributed by Zipf's law over a shuffled vocabulary: rank ~ V^u; rays over frames likewise, only milder
        rank = (torch.exp(uniform(c['N']) * math.log(c['V'] + 1.0)) - 1.0).long().clamp_(0, c['V'] - 1)
        ids = torch.randperm(c['V'], device='cuda', generator=gen)[rank]
        if c['absent']:
            ids = torch.where(uniform(c['N']) < c['absent'], torch.full_like(ids, -1), ids)
        s['ids'] = ids.to(torch.int32 if c['ids'] == 'int32' else torch.int64)
        s['table'] = normal(c['V'], c['D'])
        s['scale'] = math.sqrt(c['D'])
        s['dout'] = normal(c['N'], c['D']) if c['mode'] == 'train' else None
    elif c['op'] == 'scan':
        B, T, D, G = c['B'], c['T'], c['D'], c['G']
        # a gate per sample that lets most of the past through: 1 - opacity along a ray, a decay along a sequence
        s['gate'] = torch.sigmoid(torch.randn(B, T, G, device='cuda', generator=gen) + 2.0).to(torch.float32 if c['gate'] == 'fp32' else t)
        s['value'] = normal(B, T, D)
        s['state'] = normal(B, D, dtype=torch.float32)
        s['lengths'] = None
        if c['ragged']:
            n = (uniform(B) * (T + 1)).floor().clamp_(0, T).to(torch.int32)
            n[0] = T
            if B > 1:
                n[B - 1] = 0
            s['lengths'] = n
        if c['mode'] == 'train':
            s['dh'], s['dlast'] = normal(B, T, D), normal(B, D, dtype=torch.float32)
        elif c['mode'] == 'step':
            s['gate'], s['value'] = s['gate'][:, 0].contiguous(), s['value'][:, 0].contiguous()
    else:
        # the momentum of a weight gradient: a few strong directions over noise
        b, m, n = c['batch'], c['m'], c['n']
        k = min(4, m, n)
        g = torch.randn(b, m, n, device='cuda', generator=gen)
        g += torch.matmul(torch.randn(b, m, k, device='cuda', generator=gen), torch.randn(b, k, n, device='cuda', generator=gen))
        s['update'] = (g * 1e-3).to(t)
    return s


def run(state):
    s = state
    if own:
        from bundlesdf_amd import learn_ops as L
        if s['op'] == 'embed':
            out = L.embed_lookup(s['table'], s['ids'], s['scale'])
            if s['mode'] == 'lookup':
                return out
            return out, L.embed_lookup_grad(s['dout'], s['ids'], s['V'], s['scale'])
        if s['op'] == 'ortho':
            return L.orthogonalize(s['update'])
        if s['mode'] == 'step':
            return L.gated_scan_step(s['gate'], s['value'], s['state'])
        if s['mode'] == 'forward':
            return L.gated_scan(s['gate'], s['value'], s['state'], lengths=s['lengths'], reverse=s['reverse'])
        h, last, marks = L.gated_scan(s['gate'], s['value'], s['state'], lengths=s['lengths'], reverse=s['reverse'], want_marks=True)
        dgate, dvalue, dstate = L.gated_scan_grad(s['gate'], s['value'], s['dh'], s['dlast'], s['state'], marks,
                                                  lengths=s['lengths'], reverse=s['reverse'])
        return h, last, dgate, dvalue, dstate
    return {'embed': _plain_embed, 'scan': _plain_scan, 'ortho': _plain_ortho}[s['op']](s)


# ---- plain forms ------------------------------------------------------------------------------------------------------------------
def _plain_embed(s):
    t, V, D = s['table'], s['V'], s['D']
    ids = s['ids'].long()
    there = (ids >= 0) & (ids < V)
    row = torch.where(there, ids, torch.zeros_like(ids))
    keep = there[:, None]
    out = torch.where(keep, t[row].float() * s['scale'], torch.zeros((), device=t.device)).to(t.dtype)
    if s['mode'] == 'lookup':
        return out
    d = torch.where(keep, s['dout'].float() * s['scale'], torch.zeros((), device=t.device))
    grad = torch.zeros(V, D, device=t.device).index_add_(0, row, d)
    return out, grad.to(t.dtype)


def _double(a, b):
    """b[t] = a[t] b[t-1] + b[t] over dim 1, by doubling the distance that every position has taken in"""
    T, k = b.shape[1], 1
    while k < T:
        b = torch.cat((b[:, :k], a[:, k:] * b[:, :-k] + b[:, k:]), 1)
        a = torch.cat((a[:, :k], a[:, k:] * a[:, :-k]), 1)
        k *= 2
    return b


def _turn(x, n, reverse):
    """the first n[b] positions of each row, last first where `reverse`; an own inverse"""
    if not reverse:
        return x
    t = torch.arange(x.shape[1], device=x.device)[None]
    at = torch.where(t < n[:, None], n[:, None] - 1 - t, t)
    return torch.gather(x, 1, at[..., None].expand_as(x))


def _plain_scan(s):
    v = s['value']
    if s['mode'] == 'step':
        B, D = v.shape
        g = s['gate'].float()
        new = (g[..., None] * s['state'].reshape(B, g.shape[1], -1)).reshape(B, D) + v.float()
        return new.to(v.dtype), new
    B, T, D = v.shape
    G, rev = s['gate'].shape[2], s['reverse']
    n = s['lengths'].long() if s['lengths'] is not None else torch.full((B,), T, device=v.device)
    inside = (torch.arange(T, device=v.device)[None] < n[:, None])[..., None]
    zero, one = torch.zeros((), device=v.device), torch.ones((), device=v.device)
    g = torch.where(inside, _turn(s['gate'].float(), n, rev), one)
    x = torch.where(inside, _turn(v.float(), n, rev), zero)
    wide = g.repeat_interleave(D // G, 2)
    x = torch.cat(((wide[:, :1] * s['state'][:, None] + x[:, :1]), x[:, 1:]), 1)
    h = _double(wide, x)                                     # rows behind a sequence's end keep its last state
    last = h[:, -1].clone()
    out = _turn(torch.where(inside, h, zero), n, rev).to(v.dtype)
    if s['mode'] == 'forward':
        return out, last
    d = torch.where(inside, _turn(s['dh'].float(), n, rev), zero)
    d = torch.cat((d[:, :-1], d[:, -1:] + s['dlast'][:, None]), 1)
    after = torch.cat((wide[:, 1:], torch.ones_like(wide[:, :1])), 1)
    dv = _double(after.flip(1), d.flip(1)).flip(1)
    before = torch.cat((s['state'][:, None], h[:, :-1]), 1)
    dg = (dv * before).reshape(B, T, G, D // G).sum(3)
    dstate = dv[:, 0] * wide[:, 0]
    dg = _turn(torch.where(inside, dg, zero), n, rev).to(s['gate'].dtype)
    return out, last, dg, _turn(torch.where(inside, dv, zero), n, rev).to(v.dtype), dstate


def _plain_ortho(s):
    u = s['update']
    x = u.double()
    x = (x / torch.sqrt((x * x).sum((1, 2), keepdim=True)).clamp_min(1e-30)).float()     # the norm is a long sum: in 64 bits
    tall = x.shape[1] > x.shape[2]
    x = x.mT.contiguous() if tall else x
    a, b, c = NS
    for _ in NS_STEPS:
        g = torch.matmul(x, x.mT.contiguous())
        x = a * x + torch.matmul(b * g + c * torch.matmul(g, g), x)
    return (x.mT.contiguous() if tall else x).to(u.dtype)


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {'embed': _exact_embed, 'scan': _exact_scan, 'ortho': _exact_ortho}[s['op']](s)


def _exact_embed(s):
    V, D, ids = s['V'], s['D'], s['ids'].long()
    dev = ids.device
    ids = torch.where((ids < 0) | (ids >= V), torch.full_like(ids, V), ids)              # one zero row behind the table
    out = torch.cat((s['table'].double(), torch.zeros(1, D, dtype=torch.float64, device=dev)))[ids] * s['scale']
    if s['mode'] == 'lookup':
        return out
    order = torch.argsort(ids, stable=True)
    at = ids[order]
    sums = torch.cumsum(s['dout'].double()[order], 0)
    ends = torch.searchsorted(at, torch.arange(V, device=dev), right=True)
    sums = torch.cat((torch.zeros(1, D, dtype=torch.float64, device=dev), sums))[ends]
    first = torch.zeros(1, D, dtype=torch.float64, device=dev)
    return out, (sums - torch.cat((first, sums[:-1]))) * s['scale']


def _exact_scan(s):
    v = s['value'].double()
    if s['mode'] == 'step':
        g = s['gate'].double().repeat_interleave(v.shape[1] // s['gate'].shape[1], 1)
        new = g * s['state'].double() + v
        return new, new
    B, T, D = v.shape
    G = s['gate'].shape[2]
    g = s['gate'].double().repeat_interleave(D // G, 2)
    n = torch.full((B,), T, device=v.device) if s['lengths'] is None else s['lengths'].long()
    inside = (torch.arange(T, device=v.device)[None] < n[:, None])[..., None]            # [B, T, 1]
    order = range(T - 1, -1, -1) if s['reverse'] else range(T)
    h, state = torch.zeros_like(v), s['state'].double()
    before = torch.zeros_like(v)
    for t in order:
        before[:, t] = state
        state = torch.where(inside[:, t], g[:, t] * state + v[:, t], state)
        h[:, t] = torch.where(inside[:, t], state, torch.zeros_like(state))
    if s['mode'] == 'forward':
        return h, state
    carry, dv, dh = s['dlast'].double(), torch.zeros_like(v), s['dh'].double()
    for t in reversed(order):
        r = carry + dh[:, t]
        dv[:, t] = torch.where(inside[:, t], r, torch.zeros_like(r))
        carry = torch.where(inside[:, t], r * g[:, t], carry)
    return h, state, (dv * before).reshape(B, T, G, D // G).sum(3), dv, carry


def _exact_ortho(s):
    """p(X) X applied through the singular values, which the quintic moves one by one: U diag(p(...p(s))) V^T -- for matrices whose
    decomposition takes long, the same polynomial of the Gram matrix in 64 bits"""
    u = s['update'].double()
    norm = u.flatten(1).norm(dim=1).clamp_min(1e-30)[:, None, None]
    x = u / norm
    a, b, c = NS
    if min(x.shape[1:]) <= 128:
        left, sv, right = torch.linalg.svd(x, full_matrices=False)
        for _ in NS_STEPS:
            sv = sv * (a + sv ** 2 * (b + sv ** 2 * c))
        return torch.matmul(left * sv[:, None, :], right.contiguous())
    side = x.shape[1] <= x.shape[2]
    eye = torch.eye(min(x.shape[1:]), dtype=torch.float64, device=x.device)
    for _ in NS_STEPS:
        other = x.mT.contiguous()
        gram = torch.matmul(x, other) if side else torch.matmul(other, x)
        p = a * eye + torch.matmul(gram, b * eye + c * gram)
        x = torch.matmul(p, x) if side else torch.matmul(x, p)
    return x
