"""Cases of the packed-row operators: key spans of documents, rotary positions over several axes, and attention with a capped score, a
distance bias and key spans, each with its gradient.  `run` computes them in elementary torch operations, or, where `own` is true, by this
package's operators.

A packed row holds documents one behind another: an image of height x width tokens, with or without its text in front.  Rows behind the last
document are padding: they see no key."""
import math
import random

import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}


def listed():
    return [
        # one image and its text, masks made anew for every request
        dict(name='spans_one_image', kind='spans', tokens=310, text=48, side=16, mask='prefix'),
        # a training batch packed into one row: image tokens that read their own texts' tokens
        dict(name='spans_cross_batch', kind='spans', tokens=131000, text=77, side=32, mask='cross'),
        # one position of each of 32 requests, as a step of a decoder with a cache takes it
        dict(name='rotary_step', kind='rotary', b=32, n=1, hq=8, hk=8, d=64, sections='16+16', norm=True, interleaved=False, far=700, dtype='bf16'),
        # queries and keys of 32 images of 32 x 32 tokens, straight out of the projection
        dict(name='rotary_superres', kind='rotary', b=32, n=1024, hq=8, hk=8, d=64, sections='16+16', norm=True, interleaved=False, far=0, dtype='bf16'),
        # the same in training: gradients of queries, keys and both scales
        dict(name='rotary_bwd_superres', kind='rotary_bwd', b=32, n=1024, hq=8, hk=8, d=64, sections='16+16', norm=True, interleaved=False, far=0, dtype='bf16'),
        # a video of odd length, time / height / width, wide heads with a part that is not turned, shared keys, positions far out
        dict(name='rotary_bwd_video', kind='rotary_bwd', b=1, n=12345, hq=16, hk=4, d=128, sections='8+20+20', norm=False, interleaved=True, far=1000000, dtype='fp16'),
        # one image of 16 x 16 tokens, one request: latency
        dict(name='attend_image', kind='attend', b=1, n=256, j=256, hq=8, hk=8, d=64, mask='none', text=0, side=16, cap=0.0, axes=2, layout=0, dtype='bf16'),
        # one new position of 16 requests over caches of different lengths
        dict(name='attend_token', kind='attend', b=16, n=1, j=16384, hq=16, hk=4, d=128, mask='ragged', text=0, side=0, cap=30.0, axes=0, layout=1, dtype='fp16'),
        # a packed batch of images of many sizes, bias by rows and columns
        dict(name='attend_packed', kind='attend', b=1, n=16300, j=16300, hq=8, hk=8, d=64, mask='docs', text=0, side=32, cap=0.0, axes=2, layout=2, dtype='bf16'),
        # long documents, text prefix read both ways and image tokens in order, shared keys, capped scores
        dict(name='attend_prefix', kind='attend', b=1, n=8192, j=8192, hq=16, hk=4, d=128, mask='prefix', text=512, side=64, cap=30.0, axes=0, layout=3, dtype='bf16'),
        # the packed batch in training, slopes learned
        dict(name='attend_bwd_packed', kind='attend_bwd', b=1, n=8150, j=8150, hq=8, hk=8, d=64, mask='docs', text=0, side=32, cap=0.0, axes=2, layout=4, dtype='bf16'),
        # the long documents in training
        dict(name='attend_bwd_prefix', kind='attend_bwd', b=1, n=6100, j=6100, hq=16, hk=4, d=128, mask='prefix', text=512, side=64, cap=30.0, axes=0, layout=5, dtype='bf16'),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(['spans', 'rotary', 'rotary_bwd', 'attend', 'attend', 'attend_bwd', 'attend_bwd'])
    if kind == 'spans':
        return dict(kind=kind, tokens=_log(rng, 40, 131000), text=_log(rng, 4, 77), side=_log(rng, 4, 32), mask=rng.choice(['docs', 'causal', 'prefix', 'cross']))
    d = rng.choice([32, 64, 64, 128])
    hk = rng.choice([1, 2, 4, 8])
    if kind in ('rotary', 'rotary_bwd'):
        axes = rng.choice([1, 2, 3])
        sections = [rng.randint(1, d // (2 * axes)) for _ in range(axes)] if rng.random() < 0.5 else [d // 2 // axes // 8 * 8 or d // 2 // axes] * axes
        hq = hk * rng.choice([1, 1, 2, 4])
        b = _log(rng, 1, 32)
        dtype = rng.choice(['bf16', 'bf16', 'fp16', 'fp32'])
        n = _log(rng, 1, max(1, (16000000 if dtype == 'fp32' else 33000000) // (b * (hq + hk) * d)))
        return dict(kind=kind, b=b, n=n, hq=hq, hk=hk, d=d, sections='+'.join(map(str, sections)), norm=rng.random() < 0.6, interleaved=rng.random() < 0.4,
                    far=rng.choice([0, 0, 5000, 1000000]), dtype=dtype)
    mask = rng.choice(['none', 'docs', 'prefix', 'cross'] + (['ragged'] if kind == 'attend' else []))
    hq = min(16, hk * rng.choice([1, 2, 4]))
    text, side = _log(rng, 4, 512), _log(rng, 4, 48)
    b = 1
    if mask == 'ragged':
        b, n, j = _log(rng, 1, 16), rng.choice([1, 1, 1, 2, 5]), _log(rng, 16, 16384)
    elif mask == 'none':
        side = _log(rng, 3, 40)
        b, n = _log(rng, 1, 8), side * side
        j = n if rng.random() < 0.6 else _log(rng, 1, 600)
        b = max(1, min(b, 24000000 // (n * j * hq)))
    else:
        top = 7500 if kind == 'attend' else 5500
        n = j = max(_log(rng, 60, top), text + 16)
        if mask == 'cross':
            j = max(8, n // 2)
    return dict(kind=kind, b=b, n=n, j=j, hq=hq, hk=hk, d=d, mask=mask, text=text, side=side, cap=rng.choice([0.0, 0.0, 30.0, 50.0]),
                axes=rng.choice([0, 1, 2, 3]) if mask != 'ragged' else rng.choice([0, 1]), layout=rng.randint(1, 10 ** 6),
                dtype='bf16' if kind == 'attend_bwd' else rng.choice(['bf16', 'bf16', 'fp16']))


# ------------------------------------------------------------------------------------------------ what lies in a packed row

def _documents(rng, tokens, keys, text, side, mask):
    """(text, height, width) of the documents, as many as fit into `tokens` query rows (and `keys` key rows where texts are read across)"""
    docs, used, used_k = [], 0, 0
    while True:
        t = rng.randint(max(1, text // 4), text) if text else 0
        h, w = rng.randint(max(1, side // 4), side), rng.randint(max(1, side // 4), side)
        own_rows = h * w if mask == 'cross' else t + h * w
        if used + own_rows > tokens or (mask == 'cross' and used_k + t > keys):
            break
        docs.append((t, h, w))
        used, used_k = used + own_rows, used_k + t
    return docs or [(0, 1, 1) if mask != 'cross' else (1, 1, 1)]


def _bounds(lengths):
    return torch.tensor([0] + lengths, dtype=torch.int64).cumsum(0).to(torch.int32)


def _rows(docs, mask):
    """cu_q, cu_k, prefix of the documents"""
    nq = [h * w if mask == 'cross' else t + h * w for t, h, w in docs]
    nk = [t for t, h, w in docs] if mask == 'cross' else nq
    return _bounds(nq), _bounds(nk), torch.tensor([t for t, h, w in docs], dtype=torch.int32)


def _places(docs, rows, mask, keys):
    """int64 [rows, 3]: (time, height, width) of every row; text runs along the diagonal, an image lies behind its text"""
    out = torch.zeros(rows, 3, dtype=torch.int64)
    at = 0
    for t, h, w in docs:
        if mask != 'cross' or keys:
            out[at:at + t] = torch.arange(t)[:, None]
            at += t
        if mask != 'cross' or not keys:
            g = torch.arange(h * w)
            out[at:at + h * w] = torch.stack([torch.full_like(g, t), t + g // w, t + g % w], 1)
            at += h * w
    return out


def _layout(case):
    """documents of an attention case, or lengths of its caches"""
    rng = random.Random(case['layout'])
    if case['mask'] == 'ragged':
        return [rng.randint(max(case['n'], case['j'] // 2), max(case['n'], case['j'])) if i else max(case['n'], case['j']) for i in range(case['b'])]
    if case['mask'] == 'none':
        return None
    return _documents(rng, case['n'], case['j'], case['text'], case['side'], case['mask'])


def _pairs(case):
    """(query, key) pairs that are visible, over the batch, and key rows that are read"""
    lay = _layout(case)
    if case['mask'] == 'none':
        return case['b'] * case['n'] * case['j'], case['b'] * case['j']
    if case['mask'] == 'ragged':
        return case['n'] * sum(min(x, case['j']) for x in lay), sum(min(x, case['j']) for x in lay)
    if case['mask'] == 'cross':
        return sum(t * h * w for t, h, w in lay), sum(t for t, h, w in lay)
    m = [(t, t + h * w) for t, h, w in lay]
    if case['mask'] == 'docs':
        return sum(x * x for t, x in m), sum(x for t, x in m)
    return sum(t * t + (x * (x + 1) - t * (t + 1)) // 2 for t, x in m), sum(x for t, x in m)


# ------------------------------------------------------------------------------------------------ inputs

def _sections(case):
    """pairs that turn with each axis"""
    return [int(s) for s in case['sections'].split('+')]


def _freqs(sections, dev):
    return torch.cat([10000.0 ** (-torch.arange(s, dtype=torch.float64) / s) for s in sections]).to(dev)


def prepare(case, seed):
    dev = torch.device('cuda')
    gen = torch.Generator(device=dev).manual_seed(seed)
    kind = case['kind']
    if kind == 'spans':
        keys = max(8, case['tokens'] // 2) if case['mask'] == 'cross' else case['tokens']
        docs = _documents(random.Random(seed), case['tokens'], keys, case['text'], case['side'], case['mask'])
        cu_q, cu_k, prefix = _rows(docs, case['mask'])
        return dict(case=case, n=case['tokens'], j=keys, cu_q=cu_q.to(dev), cu_k=cu_k.to(dev) if case['mask'] == 'cross' else None,
                    prefix=prefix.to(dev) if case['mask'] == 'prefix' else None, causal=case['mask'] in ('causal', 'prefix'))
    dt, d, hq, hk, b, n = DTYPES[case['dtype']], case['d'], case['hq'], case['hk'], case['b'], case['n']
    if kind in ('rotary', 'rotary_bwd'):
        rows = torch.randn(b, n, hq + 2 * hk, d, generator=gen, device=dev).to(dt)
        q, k = rows[:, :, :hq].transpose(1, 2), rows[:, :, hq:hq + hk].transpose(1, 2)
        axes = len(_sections(case))
        side = max(1, math.isqrt(n))
        t = torch.arange(n, device=dev)
        pos = torch.stack([t, t // side, t % side], 1)[:, {1: [0], 2: [1, 2], 3: [0, 1, 2]}[axes]]
        pos = pos[None] + torch.randint(0, case['far'] + 1, (b, 1, axes), generator=gen, device=dev)
        st = dict(case=case, q=q, k=k, positions=pos.to(torch.int32), freqs=_freqs(_sections(case), dev), sections=_sections(case), q_scale=None, k_scale=None)
        if case['norm']:
            st['q_scale'] = 1 + 0.2 * torch.randn(d, generator=gen, device=dev)
            st['k_scale'] = 1 + 0.2 * torch.randn(d, generator=gen, device=dev)
        if kind == 'rotary_bwd':
            st['dq'] = torch.randn(b, n, hq, d, generator=gen, device=dev).to(dt).transpose(1, 2)
            st['dk'] = torch.randn(b, n, hk, d, generator=gen, device=dev).to(dt).transpose(1, 2)
        return st
    j, axes, lay = case['j'], case['axes'], _layout(case)
    cols = {0: [0], 1: [0], 2: [1, 2], 3: [0, 1, 2]}[axes]
    unit = case['cap'] == 0.0                    # without a cap the queries and keys are normalised, as the model's are
    rows = torch.randn(b, n, hq, d, generator=gen, device=dev)
    keys = torch.randn(b, j, 2 * hk, d, generator=gen, device=dev)
    if unit:
        rows = rows / rows.norm(dim=-1, keepdim=True)
        keys[:, :, :hk] /= keys[:, :, :hk].norm(dim=-1, keepdim=True)
    q, keys = rows.to(dt).transpose(1, 2), keys.to(dt)
    st = dict(case=case, q=q, k=keys[:, :, :hk].transpose(1, 2), v=keys[:, :, hk:].transpose(1, 2), scale=8.0 if unit else 2.0 * d ** -0.5,
              softcap=case['cap'], spans=None, slopes=None, positions=None, key_positions=None)
    if case['mask'] == 'ragged':
        ends = torch.tensor(lay, device=dev)
        at = ends[:, None] - n + torch.arange(n, device=dev)          # the new positions are the last ones of their caches
        st['spans'] = torch.stack([torch.zeros_like(at), at + 1], 2).to(torch.int32)
        pos_q, pos_k = at[:, :, None].expand(b, n, 3), torch.arange(j, device=dev)[:, None].expand(j, 3)
    elif case['mask'] == 'none':
        t, u = torch.arange(n, device=dev), torch.arange(j, device=dev)
        pos_q = torch.stack([t, t // case['side'], t % case['side']], 1)
        pos_k = torch.stack([u, u // case['side'], u % case['side']], 1)
    else:
        cu_q, cu_k, prefix = _rows(lay, case['mask'])
        st['spans'] = _plain_spans(cu_q.to(dev), cu_k.to(dev), prefix.to(dev) if case['mask'] == 'prefix' else None, n, j, case['mask'] == 'prefix')
        pos_q = _places(lay, n, case['mask'], False).to(dev)
        pos_k = _places(lay, j, case['mask'], True).to(dev)
    if axes:
        st['positions'], st['key_positions'] = pos_q[..., cols].to(torch.int32).contiguous(), pos_k[..., cols].to(torch.int32).contiguous()
        st['slopes'] = 0.02 + 0.2 * torch.rand(hq, axes, generator=gen, device=dev)
    if kind == 'attend_bwd':
        st['out'], st['lse'] = _plain_attend(st)
        st['dout'] = torch.randn(b, n, hq, d, generator=gen, device=dev).to(dt).transpose(1, 2)
    return st


# ------------------------------------------------------------------------------------------------ plain forms

def _plain_spans(cu_q, cu_k, prefix, n, j, causal):
    i = torch.arange(n, device=cu_q.device)
    doc = torch.searchsorted(cu_q.long(), i, right=True) - 1
    inside = (doc >= 0) & (doc < cu_q.numel() - 1)
    doc = doc.clamp(0, cu_q.numel() - 2)
    q0, lq, k0, lk = cu_q[doc], cu_q[doc + 1] - cu_q[doc], cu_k[doc], cu_k[doc + 1] - cu_k[doc]
    seen = lk
    if causal:
        seen = i - q0 + 1 + lk - lq
        if prefix is not None:
            seen = torch.maximum(seen, prefix[doc])
        seen = torch.minimum(seen.clamp(min=0), lk)
    zero = torch.zeros_like(i)
    return torch.stack([torch.where(inside, k0, zero), torch.where(inside, k0 + seen, zero)], 1).to(torch.int32)


def _plain_angles(st):
    sections = st['sections']
    axis = torch.arange(len(sections), device=st['freqs'].device).repeat_interleave(torch.tensor(sections, device=st['freqs'].device))
    angle = st['positions'].double()[..., axis] * st['freqs']                # [b, n, pairs]
    return angle.cos().float()[:, None], angle.sin().float()[:, None]


def _plain_turn(x, cos, sin, interleaved):
    p = cos.shape[-1]
    a, b = (x[..., 0:2 * p:2], x[..., 1:2 * p:2]) if interleaved else (x[..., :p], x[..., p:2 * p])
    a, b = a * cos - b * sin, a * sin + b * cos
    y = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([y, x[..., 2 * p:]], -1)


def _plain_rotary(x, scale, cos, sin, interleaved):
    y = x.float()
    if scale is not None:
        y = y / (y * y).sum(-1, keepdim=True).sqrt().clamp(min=1e-12) * scale
    return _plain_turn(y, cos, sin, interleaved).to(x.dtype)


def _plain_rotary_bwd(dy, x, scale, cos, sin, interleaved):
    g = _plain_turn(dy.float(), cos, -sin, interleaved)
    if scale is None:
        return g.to(dy.dtype), None
    x = x.float()
    norm = (x * x).sum(-1, keepdim=True).sqrt().clamp(min=1e-12)
    xh, gs = x / norm, g * scale
    return ((gs - xh * (xh * gs).sum(-1, keepdim=True)) / norm).to(dy.dtype), (g * xh).sum((0, 1, 2))


def _plain_scores(st):
    """scores [b, hk, hq / hk, n, j] in 32 bits, the derivative of the cap, and which pairs are visible"""
    q, k = st['q'].float(), st['k'].float()
    b, hq, n, d = q.shape
    hk, j = k.shape[1], k.shape[2]
    s = torch.matmul(q.reshape(b, hk, hq // hk * n, d), k.transpose(-1, -2)).reshape(b, hk, hq // hk, n, j) * st['scale']
    slope = None
    if st['softcap']:
        t = torch.tanh(s / st['softcap'])
        s, slope = st['softcap'] * t, 1 - t * t
    if st['slopes'] is not None:
        far = (st['positions'][..., :, None, :] - st['key_positions'][..., None, :, :]).abs().float()       # [(b,) n, j, axes]
        bias = torch.matmul(far, st['slopes'].t()).movedim(-1, -3)                                           # [(b,) hq, n, j]
        s = s - bias.reshape(-1, hk, hq // hk, n, j)
    seen = torch.ones(n, j, dtype=torch.bool, device=q.device)
    if st['spans'] is not None:
        key = torch.arange(j, device=q.device)
        seen = (key >= st['spans'][..., :1]) & (key < st['spans'][..., 1:])
    return s, slope, (seen[:, None, None] if seen.dim() == 3 else seen)


def _plain_attend(st):
    s, _, seen = _plain_scores(st)
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = (s - top.clamp(min=-1e30)).exp()
    total = p.sum(-1, keepdim=True)
    b, hk, group, n, j = s.shape
    out = torch.matmul(p.reshape(b, hk, group * n, j), st['v'].float()).reshape(b, hk, group, n, -1) / total.clamp(min=1e-30)
    lse = torch.where(total > 0, top + total.clamp(min=1e-30).log(), torch.full_like(top, -math.inf))
    return out.reshape(st['q'].shape).to(st['q'].dtype), lse.reshape(b, hk * group, n)


def _plain_attend_bwd(st):
    s, slope, seen = _plain_scores(st)
    b, hk, group, n, j = s.shape
    d = st['q'].shape[-1]
    lse = st['lse'].reshape(b, hk, group, n, 1)
    p = (s - lse.clamp(min=-1e30)).masked_fill(~seen, -math.inf).exp()
    del s
    dout = st['dout'].float()
    delta = (dout * st['out'].float()).sum(-1).reshape(b, hk, group, n, 1)
    dout = dout.reshape(b, hk, group * n, d)
    ds = p * (torch.matmul(dout, st['v'].float().transpose(-1, -2)).reshape(p.shape) - delta)
    dv = torch.matmul(p.reshape(b, hk, group * n, j).transpose(-1, -2).contiguous(), dout)
    del p
    dslopes = None
    if st['slopes'] is not None:
        far = (st['positions'][..., :, None, :] - st['key_positions'][..., None, :, :]).abs().float()
        dslopes = -torch.matmul(ds.reshape(b, hk * group, n, j).transpose(1, 2), far).double().sum((0, 1)).float()
    if slope is not None:
        ds = ds * slope
    ds = (ds * st['scale']).reshape(b, hk, group * n, j)
    dq = torch.matmul(ds, st['k'].float()).reshape(st['q'].shape)
    dk = torch.matmul(ds.transpose(-1, -2).contiguous(), st['q'].float().reshape(b, hk, group * n, d))
    dt = st['q'].dtype
    return dq.to(dt), dk.to(dt), dv.to(dt), dslopes


def run(state):
    st, case = state, state['case']
    kind = case['kind']
    if kind == 'spans':
        if own:
            from muse_maskgit_pytorch_amd import ops
            return ops.attention_spans(st['cu_q'], st['n'], cu_k=st['cu_k'], j=st['j'], prefix=st['prefix'], causal=st['causal'])
        return _plain_spans(st['cu_q'], st['cu_q'] if st['cu_k'] is None else st['cu_k'], st['prefix'], st['n'], st['j'], st['causal'])
    if kind == 'rotary':
        if own:
            from muse_maskgit_pytorch_amd import ops
            return ops.rotary_axes(st['q'], st['k'], st['positions'], st['freqs'], st['sections'], q_scale=st['q_scale'], k_scale=st['k_scale'],
                                   interleaved=case['interleaved'])
        cos, sin = _plain_angles(st)
        return (_plain_rotary(st['q'], st['q_scale'], cos, sin, case['interleaved']), _plain_rotary(st['k'], st['k_scale'], cos, sin, case['interleaved']))
    if kind == 'rotary_bwd':
        if own:
            from muse_maskgit_pytorch_amd import ops
            got = ops.rotary_axes_bwd(st['dq'], st['dk'], st['positions'], st['freqs'], st['sections'], q=st['q'], k=st['k'], q_scale=st['q_scale'],
                                      k_scale=st['k_scale'], interleaved=case['interleaved'])
        else:
            cos, sin = _plain_angles(st)
            dq, dqs = _plain_rotary_bwd(st['dq'], st['q'], st['q_scale'], cos, sin, case['interleaved'])
            dk, dks = _plain_rotary_bwd(st['dk'], st['k'], st['k_scale'], cos, sin, case['interleaved'])
            got = dq, dk, dqs, dks
        return got if case['norm'] else got[:2]
    if kind == 'attend':
        if own:
            from muse_maskgit_pytorch_amd import ops
            return ops.attend_spans(st['q'], st['k'], st['v'], st['spans'], scale=st['scale'], softcap=st['softcap'], slopes=st['slopes'],
                                    positions=st['positions'], key_positions=st['key_positions'], return_lse=True)
        return _plain_attend(st)
    if own:
        from muse_maskgit_pytorch_amd import ops
        got = ops.attend_spans_bwd(st['q'], st['k'], st['v'], st['out'], st['lse'], st['dout'], st['spans'], scale=st['scale'], softcap=st['softcap'],
                                   slopes=st['slopes'], positions=st['positions'], key_positions=st['key_positions'])
    else:
        got = _plain_attend_bwd(st)
    return got if case['axes'] else got[:3]


# ------------------------------------------------------------------------------------------------ what a pass cannot do without

def work(case):
    kind = case['kind']
    if kind == 'spans':
        return dict(bytes=8 * case['tokens'], flops=8 * case['tokens'])
    size = 4 if case['dtype'] == 'fp32' else 2
    if kind in ('rotary', 'rotary_bwd'):
        rows, pairs = case['b'] * case['n'], sum(_sections(case))
        values = rows * (case['hq'] + case['hk']) * case['d']
        passes = 3 if kind == 'rotary_bwd' and case['norm'] else 2
        return dict(bytes=passes * size * values + 4 * rows * len(_sections(case)) + 8 * pairs,
                    flops=rows * (case['hq'] + case['hk']) * 6 * pairs + (values * (8 if kind == 'rotary_bwd' else 4) if case['norm'] else 0))
    pairs, keys = _pairs(case)
    q = case['b'] * case['n'] * case['hq'] * case['d'] * size
    kv = 2 * keys * case['hk'] * case['d'] * size
    small = 4 * case['b'] * case['n'] * case['hq'] + (0 if case['mask'] == 'none' else 8 * case['n'] * (case['b'] if case['mask'] == 'ragged' else 1))
    small += 4 * case['axes'] * (case['n'] + case['j'])
    if kind == 'attend':
        return dict(bytes=2 * q + kv + small, flops=4 * case['d'] * case['hq'] * pairs)
    return dict(bytes=4 * q + 2 * kv + small, flops=10 * case['d'] * case['hq'] * pairs)


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits

def _exact_rotary(x, scale, pos, freqs, sections, interleaved, dy=None):
    x = x.double()
    size = x.norm(dim=-1, keepdim=True).clamp(min=1e-12)
    y = dy.double() if dy is not None else (x if scale is None else x / size * scale.double())
    out, p0, total = y.clone(), 0, sum(sections)
    for axis, s in enumerate(sections):
        z = pos[:, None, :, axis, None].double() * freqs[p0:p0 + s]
        turn = torch.polar(torch.ones_like(z), -z if dy is not None else z)
        ia = torch.arange(p0, p0 + s, device=x.device) * (2 if interleaved else 1)
        ib = ia + (1 if interleaved else total)
        w = torch.complex(y[..., ia], y[..., ib]) * turn
        out[..., ia], out[..., ib] = w.real, w.imag
        p0 += s
    if dy is None or scale is None:
        return out, None
    xh, gs = x / size, out * scale.double()
    return (gs - xh * (xh * gs).sum(-1, keepdim=True)) / size, (out * xh).sum((0, 1, 2))


def _exact_attend(st, grads):
    case, dev = st['case'], st['q'].device
    b, hq, n, d = st['q'].shape
    hk, j = st['k'].shape[1:3]
    group = hq // hk
    out, lse = torch.zeros(b, hq, n, d, dtype=torch.float64, device=dev), torch.zeros(b, hq, n, dtype=torch.float64, device=dev)
    dq, dk, dv = (torch.zeros(t.shape, dtype=torch.float64, device=dev) for t in (st['q'], st['k'], st['v']))
    dslopes = torch.zeros(hq, case['axes'], dtype=torch.float64, device=dev)
    key = torch.arange(j, device=dev)
    for x in range(b):
        of = lambda t, dims: t[x] if t.dim() == dims else t
        hidden = None
        if st['spans'] is not None:
            sp = of(st['spans'], 3)
            hidden = (key[None] < sp[:, :1]) | (key[None] >= sp[:, 1:])
        for h in range(hq):
            q, k, v = st['q'][x, h].double(), st['k'][x, h // group].double(), st['v'][x, h // group].double()
            s = (q @ k.T) * st['scale']
            t = None
            if case['cap']:
                t = (s / case['cap']).tanh_()
                s = t * case['cap']
            for a in range(case['axes']):
                far = (of(st['positions'], 3)[:, None, a] - of(st['key_positions'], 3)[None, :, a]).abs()
                s -= st['slopes'][h, a].double() * far
            if hidden is not None:
                s.masked_fill_(hidden, -math.inf)
            if not grads:
                lse[x, h] = torch.logsumexp(s, -1)
                p = (s - lse[x, h].clamp(min=-1e300)[:, None]).exp_()
                out[x, h] = p @ v
                continue
            do, o = st['dout'][x, h].double(), st['out'][x, h].double()
            p = (s - st['lse'][x, h].double().clamp(min=-1e300)[:, None]).exp_()
            dv[x, h // group] += p.T @ do
            ds = (do @ v.T - (do * o).sum(-1, keepdim=True)) * p
            for a in range(case['axes']):
                far = (of(st['positions'], 3)[:, None, a] - of(st['key_positions'], 3)[None, :, a]).abs()
                dslopes[h, a] -= (ds * far).sum()
            if t is not None:
                ds *= 1 - t * t
            ds *= st['scale']
            dq[x, h] = ds @ k
            dk[x, h // group] += ds.T @ q
    if not grads:
        return out, lse
    return (dq, dk, dv, dslopes) if case['axes'] else (dq, dk, dv)


def exact(case, seed):
    st = prepare(case, seed)
    kind = case['kind']
    if kind == 'spans':
        cu_q, cu_k = st['cu_q'].tolist(), (st['cu_q'] if st['cu_k'] is None else st['cu_k']).tolist()
        want = torch.zeros(st['n'], 2, dtype=torch.int32)
        for doc in range(len(cu_q) - 1):
            lq, lk = cu_q[doc + 1] - cu_q[doc], cu_k[doc + 1] - cu_k[doc]
            want[cu_q[doc]:cu_q[doc + 1], 0] = cu_k[doc]
            first = 0 if st['prefix'] is None else int(st['prefix'][doc])
            want[cu_q[doc]:cu_q[doc + 1], 1] = torch.tensor([cu_k[doc] + (max(0, min(lk, max(first, i + 1 + lk - lq))) if st['causal'] else lk) for i in range(lq)],
                                                             dtype=torch.int32)
        return want.to(st['cu_q'].device)
    if kind in ('rotary', 'rotary_bwd'):
        dq, dk = st.get('dq'), st.get('dk')
        q, dqs = _exact_rotary(st['q'], st['q_scale'], st['positions'], st['freqs'], st['sections'], case['interleaved'], dq)
        k, dks = _exact_rotary(st['k'], st['k_scale'], st['positions'], st['freqs'], st['sections'], case['interleaved'], dk)
        return (q, k, dqs, dks) if kind == 'rotary_bwd' and case['norm'] else (q, k)
    return _exact_attend(st, kind == 'attend_bwd')
