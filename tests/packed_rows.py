"""Plain 64-bit forms of the packed-row operators (ops.attention_spans, rotary_axes, attend_spans and the gradients), written from their definitions, and the bounds
within which the kernels have to stay.  Bounds count roundings: one rounding to a type t is off by at most eps(t) / 2 of the value."""
import math

import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
F32 = 2.0 ** -24


def spans_of(cu_q, cu_k, prefix, n, causal):
    out = torch.zeros(n, 2, dtype=torch.int32)
    cu_q, cu_k = [int(x) for x in cu_q], [int(x) for x in cu_k]
    for doc in range(len(cu_q) - 1):
        lq, lk = cu_q[doc + 1] - cu_q[doc], cu_k[doc + 1] - cu_k[doc]
        for x in range(lq):
            seen = lk
            if causal:
                seen = min(lk, max(0, x + 1 + lk - lq, 0 if prefix is None else int(prefix[doc])))
            if 0 <= cu_q[doc] + x < n:
                out[cu_q[doc] + x] = torch.tensor([cu_k[doc], cu_k[doc] + seen], dtype=torch.int32)
    return out


def turn(x, pos, freqs, sections, interleaved, back=False):
    """x float64 (b, h, n, d), pos (b, n, axes)"""
    P = sum(sections)
    axis = [a for a, s in enumerate(sections) for _ in range(s)]
    y = x.clone()
    for p in range(P):
        ang = pos[:, None, :, axis[p]].double() * freqs[p]
        c, s = ang.cos(), ang.sin() * (-1 if back else 1)
        ia, ib = (2 * p, 2 * p + 1) if interleaved else (p, P + p)
        y[..., ia] = x[..., ia] * c - x[..., ib] * s
        y[..., ib] = x[..., ia] * s + x[..., ib] * c
    return y


def rotary(x, pos, freqs, sections, scale=None, interleaved=False):
    x = x.double()
    if scale is not None:
        x = x / x.norm(dim=-1, keepdim=True).clamp(min=1e-12) * scale.double()
    return turn(x, pos, freqs, sections, interleaved)


def visible(n, j, spans=None, key_mask=None, b=1):
    """bool (b, n, j)"""
    key = torch.arange(j)
    seen = torch.ones(b, n, j, dtype=torch.bool)
    if spans is not None:
        sp = spans if spans.dim() == 3 else spans[None]
        seen = seen & (key >= sp[..., :1]) & (key < sp[..., 1:])
    if key_mask is not None:
        seen = seen & key_mask[:, None, :].bool()
    return seen


def attention(q, k, v, seen, scale, cap=0.0, slopes=None, pos_q=None, pos_k=None, dout=None, out=None, lse=None, tight_cap=False):
    """float64 results and their bounds: forward {out, lse}, with dout (and the forward's out / lse, taken as they are) {dq, dk, dv, dslopes}; each with a tensor
    of what the kernel's roundings may change.  Hidden keys and rows are taken out of the operands (their values, NaN among them, take no part)."""
    dt, half = q.dtype, HALF[q.dtype]
    b, hq, n, d = q.shape
    hk, j = k.shape[1], k.shape[2]
    g = hq // hk
    q, k, v = q.double(), k.double(), v.double()
    r = {}

    def new(*s):
        return torch.zeros(*s, dtype=torch.float64)
    fwd = dout is None
    if fwd:
        r['out'], r['out_tol'], r['lse'], r['lse_tol'] = new(b, hq, n, d), new(b, hq, n, d), new(b, hq, n), new(b, hq, n)
    else:
        for name, like in (('dq', q), ('dk', k), ('dv', v)):
            r[name], r[name + '_tol'] = new(*like.shape), new(*like.shape)
        if slopes is not None:
            r['dslopes'], r['dslopes_tol'] = new(*slopes.shape), new(*slopes.shape)
    for x in range(b):
        sv = seen[x]
        keys, rows = sv.any(0), sv.any(1)
        for h in range(hq):
            Q, K, V = (torch.where(m[:, None], t, torch.zeros_like(t)) for m, t in ((rows, q[x, h]), (keys, k[x, h // g]), (keys, v[x, h // g])))
            raw = Q @ K.T * scale
            # fp32 sums of d products, then a handful of roundings of the score
            serr = F32 * ((d + 4) * (Q.abs() @ K.abs().T) * scale)
            s, slope = raw, torch.ones_like(raw)
            if cap:
                t = torch.tanh(raw / cap)
                s, slope = cap * t, 1 - t * t
                serr = serr + F32 * 8 * (s.abs() if tight_cap else cap)      # a few roundings, of the cap's size or (tight_cap) of the score's own
            far = []
            if slopes is not None:
                pq, pk = (p if p.dim() == 3 else p[None].expand(b, -1, -1) for p in (pos_q, pos_k))
                for a in range(slopes.shape[1]):
                    far.append((pq[x, :, None, a].long() - pk[x, None, :, a].long()).abs().double())
                    s = s - slopes[h, a].double() * far[-1]
                    serr = serr + 3 * F32 * (slopes[h, a].double().abs() * far[-1] + s.abs())
            serr = serr + 4 * F32 * s.abs()
            s = s.masked_fill(~sv, -math.inf)
            serr = serr.masked_fill(~sv, 0)
            if fwd:
                L = torch.logsumexp(s, -1)
                p = torch.where(sv, (s - L.clamp(min=-1e300)[:, None]).exp(), torch.zeros_like(s))
                worst = 2 * (serr.max(-1).values if j else torch.zeros(n, dtype=torch.float64)) + (8 + 4 * math.sqrt(j)) * F32       # of a probability: its score, the sum's, exp2's and the sum's additions
                r['out'][x, h], r['lse'][x, h] = p @ V, L
                r['out_tol'][x, h] = half * 1.02 * (p @ V.abs() + (p @ V).abs()) + worst[:, None] * (p @ V.abs()) + (2.0 ** -24 if dt == torch.float16 else 1e-30)
                r['lse_tol'][x, h] = worst + 4 * F32 * L.abs().nan_to_num(posinf=0, neginf=0)
                continue
            O, DO = (torch.where(rows[:, None], t[x, h].double(), torch.zeros(1, dtype=torch.float64)) for t in (out, dout))
            L = lse[x, h].double().clamp(min=-1e300)
            p = torch.where(sv, (s - L[:, None]).exp(), torch.zeros_like(s))
            perr = p * (serr + F32 * (8 + 4 * L.clamp(min=-1e6).abs()[:, None]))
            dp = DO @ V.T
            delta = (DO * O).sum(-1, keepdim=True)
            dperr = F32 * (d + 4) * (DO.abs() @ V.abs().T + (DO * O).abs().sum(-1, keepdim=True))
            ds = p * (dp - delta)
            dserr = perr * (dp - delta).abs() + p * dperr + 4 * F32 * ds.abs()
            hh = h // g
            r['dv'][x, hh] += p.T @ DO
            r['dv_tol'][x, hh] += (half * 1.02 * p + perr).T @ DO.abs()
            for a in range(len(far)):
                r['dslopes'][h, a] -= (ds * far[a]).sum()
                r['dslopes_tol'][h, a] += ((dserr + 16 * F32 * ds.abs()) * far[a]).sum()
            cerr = 16 * F32 * (slope < 1) if cap else 0.0       # 1 - tanh^2 near the flat ends
            g2 = ds * slope * scale
            g2err = (dserr * slope + ds.abs() * cerr) * scale + 4 * F32 * g2.abs()
            r['dq'][x, h] = g2 @ K
            r['dq_tol'][x, h] = (half * 1.02 * g2.abs() + g2err) @ K.abs()
            r['dk'][x, hh] += g2.T @ Q
            r['dk_tol'][x, hh] += (half * 1.02 * g2.abs() + g2err).T @ Q.abs()
    if not fwd:
        for name in ('dq', 'dk', 'dv'):
            r[name + '_tol'] += half * 1.02 * r[name].abs() + 1e-30
            r[name + '_tol'] += 4 * math.sqrt(max(n, j) * g) * F32 * r[name + '_tol'] / half       # additions in fp32
        if slopes is not None:
            r['dslopes_tol'] += 1e-30
    return r


def check(got, want, tol, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, f'{what}: shape {tuple(got.shape)}, not {tuple(want.shape)}'
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, torch.zeros_like(want), (got - want).abs())
    bad = ~(off <= tol)
    assert not bad.any(), f'{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / tol.clamp(min=1e-300)).nan_to_num(1e9).max()):.3g} of its bound, at {bad.nonzero()[0].tolist()}: {float(got[bad][0])} for {float(want[bad][0])}'
