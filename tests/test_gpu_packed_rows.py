"""The packed-row operators on the GPU against their plain forms in 64 bits (tests/packed_rows.py): spans of documents, rotary positions, attention with spans, capped
scores and a distance bias, their gradients."""
import math
import random

import pytest
import torch

import packed_rows as R
from muse_maskgit_pytorch_amd import ops

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
DT = dict(bf16=torch.bfloat16, fp16=torch.float16, fp32=torch.float32)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def bounds(rng, docs, total):
    cuts = sorted(rng.randint(0, total) for _ in range(docs))
    return torch.tensor([0] + cuts, dtype=torch.int32)


# ------------------------------------------------------------------------------------------------ spans
@pytest.mark.parametrize('docs,n', [(0, 5), (1, 1), (1, 256), (3, 310), (40, 257), (5000, 9000)])
@pytest.mark.parametrize('mode', ['all', 'causal', 'prefix', 'cross', 'cross_prefix'])
def test_spans(docs, n, mode):
    rng = random.Random(docs * 7 + n)
    cu_q = bounds(rng, docs, max(0, n - 3))
    cross = mode.startswith('cross')
    j = n // 2 + 1 if cross else n
    cu_k = bounds(rng, docs, j) if cross else None
    prefix = torch.tensor([rng.randint(0, 50) for _ in range(docs)], dtype=torch.int32) if 'prefix' in mode else None
    causal = mode in ('causal', 'prefix', 'cross_prefix')
    got = ops.attention_spans(cu_q.to(DEV), n, cu_k=cu_k.to(DEV) if cross else None, j=j, prefix=prefix.to(DEV) if prefix is not None else None, causal=causal)
    assert got.dtype == torch.int32 and torch.equal(got.cpu(), R.spans_of(cu_q, cu_k if cross else cu_q, prefix, n, causal))


def test_spans_of_a_batch_and_of_bounds_that_do_not_start_at_zero():
    cu = torch.tensor([[0, 3, 3, 10], [2, 4, 9, 12]], dtype=torch.int32)
    got = ops.attention_spans(cu.to(DEV), 14, causal=True)
    assert got.shape == (2, 14, 2)
    for x in range(2):
        assert torch.equal(got[x].cpu(), R.spans_of(cu[x], cu[x], None, 14, True))
    # strided tables; bounds behind the keys are cut off
    wide = torch.zeros(4, 6, dtype=torch.int32)
    wide[:, ::2][:, :3] = torch.tensor([0, 4, 20], dtype=torch.int32)
    got = ops.attention_spans(wide.to(DEV)[0, ::2], 8, cu_k=wide.to(DEV)[1, ::2], j=10)
    assert got.cpu().tolist() == [[0, 4]] * 4 + [[4, 10]] * 4


CUT = [  # cu_q, cu_k, prefix, n, j: bounds behind the rows and keys or in front of them (a window of a longer packing), the last document cut off inside
    ([0, 4, 20], None, None, 8, 8), ([0, 4, 20], None, None, 10, 10), ([0, 4, 20], None, [0, 3], 10, 10), ([0, 4, 20], None, [2, 9], 10, 7), ([-5, 3, 6], None, None, 9, 9),
    ([-5, 3, 6], None, [4, 2], 9, 9), ([0, 3, 9], [0, 5, 40], None, 9, 12), ([0, 3, 9], [-4, 5, 40], [3, 20], 9, 12), ([0, 3, 9], [-4, -2, 6], [1, 1], 9, 12),
    ([0, 3, 9], [14, 20, 30], None, 9, 12), ([0, 6, 2 ** 31 - 1], None, None, 300, 290), ([-2 ** 31, 6, 2 ** 31 - 1], None, [5, 7], 300, 300)]


@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('case', CUT, ids=lambda c: f'{c[0]}-{c[1]}-{c[2]}-{c[3]}-{c[4]}')
def test_spans_of_documents_that_are_cut_off(case, causal):
    """what a row sees goes by the whole document; then what lies outside the j keys is cut off"""
    cu_q, cu_k, prefix, n, j = case
    if prefix is not None and not causal:
        prefix = None
    ck = cu_q if cu_k is None else cu_k
    want = []
    for i in range(n):
        doc = max((d for d in range(len(cu_q)) if cu_q[d] <= i), default=-1)
        if not 0 <= doc < len(cu_q) - 1:
            want.append([0, 0])
            continue
        lq, lk = cu_q[doc + 1] - cu_q[doc], ck[doc + 1] - ck[doc]
        seen = lk
        if causal:
            seen = min(lk, max(0, i - cu_q[doc] + 1 + lk - lq, prefix[doc] if prefix else 0))
        want.append([min(max(ck[doc], 0), j), min(max(ck[doc] + seen, 0), j)])
    t = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device=DEV)
    got = ops.attention_spans(t(cu_q), n, cu_k=t(cu_k), j=j, prefix=t(prefix), causal=causal)
    assert got.tolist() == want
    two = lambda x: None if x is None else torch.stack([t(x)] * 2)
    assert ops.attention_spans(two(cu_q), n, cu_k=two(cu_k), j=j, prefix=two(prefix), causal=causal).tolist() == [want] * 2


# ------------------------------------------------------------------------------------------------ rotary
ROT = [  # b, n, hq, hk, d, sections, interleaved
    (1, 1, 1, 1, 32, [16], False), (2, 37, 8, 8, 64, [16, 16], False), (3, 65, 4, 1, 128, [8, 20, 20], False), (2, 19, 6, 2, 64, [8, 8, 8], True),
    (1, 300, 8, 2, 128, [64], True), (2, 33, 3, 3, 20, [3, 2], False), (1, 9, 2, 1, 24, [1, 2, 3, 4], True), (1, 70, 2, 2, 256, [32, 32, 64], False),
    (1, 17, 2, 2, 256, [1, 2, 7], True), (2, 5, 1, 5, 128, [5, 7], False), (1, 4, 2, 2, 2, [1], False), (1, 130, 40, 40, 64, [32], False), (1, 6, 2, 1, 64, [0, 0], False)]


def rot_inputs(b, n, hq, hk, d, sections, dtype, seed, far=3000):
    g = gen(seed)
    rows = torch.randn(b, n, hq + 2 * hk, d, generator=g).to(DT[dtype])
    q, k = rows[:, :, :hq].transpose(1, 2), rows[:, :, hq:hq + hk].transpose(1, 2)
    pos = torch.randint(-far, far + 1, (b, n, len(sections)), generator=g).to(torch.int32)
    freqs = torch.cat([1000.0 ** (-torch.arange(s, dtype=torch.float64) / max(1, s)) for s in sections])
    return rows, q, k, pos, freqs, 1 + 0.3 * torch.randn(d, generator=g), 1 + 0.3 * torch.randn(d, generator=g), g


def rot_tol(want, mag, half):
    """one rounding of the result; before it a few fp32 roundings of terms of the size of the pair (`mag`)"""
    return half * 1.02 * want.abs() + 24 * R.F32 * mag + (2.0 ** -24 if half == R.HALF[torch.float16] else 1e-30)


def pair_size(x, sections, interleaved):
    """largest magnitude of a pair (of the element itself behind the pairs)"""
    P = sum(sections)
    y = x.abs().clone()
    for p in range(P):
        a, b = (2 * p, 2 * p + 1) if interleaved else (p, P + p)
        m = torch.maximum(x[..., a].abs(), x[..., b].abs())
        y[..., a] = y[..., b] = m
    return y


@pytest.mark.parametrize('dtype', ['bf16', 'fp16', 'fp32'])
@pytest.mark.parametrize('norm', [False, True])
@pytest.mark.parametrize('shape', ROT)
def test_rotary(shape, norm, dtype):
    b, n, hq, hk, d, sections, inter = shape
    rows, q, k, pos, freqs, qs, ks, _ = rot_inputs(*shape[:6], dtype, 11)
    dev_rows = rows.to(DEV)
    dq_, dk_ = dev_rows[:, :, :hq].transpose(1, 2), dev_rows[:, :, hq:hq + hk].transpose(1, 2)
    got = ops.rotary_axes(dq_, dk_, pos.to(DEV), freqs.to(DEV), sections, *((qs.to(DEV), ks.to(DEV)) if norm else ()), interleaved=inter)
    for x, s, y, name in ((q, qs, got[0], 'q'), (k, ks, got[1], 'k')):
        assert y.dtype == x.dtype and y.shape == x.shape
        want = R.rotary(x, pos, freqs, sections, s if norm else None, inter)
        z = x.double()
        if norm:
            z = z / z.norm(dim=-1, keepdim=True) * s.double()
        R.check(y, want, rot_tol(want, pair_size(z, sections, inter) * (d / 8 if norm else 1), R.HALF[x.dtype]), name)


@pytest.mark.parametrize('dtype', ['bf16', 'fp16', 'fp32'])
@pytest.mark.parametrize('norm', [False, True])
@pytest.mark.parametrize('shape', ROT)
def test_rotary_bwd(shape, norm, dtype):
    b, n, hq, hk, d, sections, inter = shape
    rows, q, k, pos, freqs, qs, ks, g = rot_inputs(*shape[:6], dtype, 12)
    dq = torch.randn(b, n, hq, d, generator=g).to(DT[dtype]).transpose(1, 2)
    dk = torch.randn(b, hk, n, d, generator=g).to(DT[dtype])
    args = dict(q=q.to(DEV), k=k.to(DEV), q_scale=qs.to(DEV), k_scale=ks.to(DEV)) if norm else {}
    got = ops.rotary_axes_bwd(dq.to(DEV), dk.to(DEV), pos.to(DEV), freqs.to(DEV), sections, interleaved=inter, **args)
    again = ops.rotary_axes_bwd(dq.to(DEV), dk.to(DEV), pos.to(DEV), freqs.to(DEV), sections, interleaved=inter, **args)
    for x, s, dy, dx, ds, name in ((q, qs, dq, got[0], got[2], 'q'), (k, ks, dk, got[1], got[3], 'k')):
        gr = R.turn(dy.double(), pos, freqs, sections, inter, back=True)
        half, size = R.HALF[x.dtype], pair_size(dy.double(), sections, inter)
        if not norm:
            assert ds is None
            R.check(dx, gr, rot_tol(gr, size, half), name)
            continue
        x, s = x.double(), s.double()
        ln = x.norm(dim=-1, keepdim=True)
        xh, gs = x / ln, gr * s
        want = (gs - xh * (xh * gs).sum(-1, keepdim=True)) / ln
        mag = (size * s.abs() + xh.abs() * (xh.abs() * size * s.abs()).sum(-1, keepdim=True)) / ln
        R.check(dx, want, rot_tol(want, mag * d / 8, half), name)
        R.check(ds, (gr * xh).sum((0, 1, 2)), (R.F32 * (24 + d + 2 * math.sqrt(b * n * hq))) * (size * xh.abs()).sum((0, 1, 2)), name + ' scale')
    for x, y in zip(got, again):
        assert x is None and y is None or torch.equal(x, y)


@pytest.mark.parametrize('dtype', ['bf16', 'fp16', 'fp32'])
@pytest.mark.parametrize('shape', [(2, 37, 3, 1, 128, [8, 20, 20], False), (2, 33, 3, 3, 20, [3, 2], False), (1, 40, 4, 2, 64, [8, 8, 7], True), (1, 9, 2, 1, 24, [1, 2, 3, 4], True),
                                   (1, 6, 2, 1, 64, [0, 0], False)], ids=str)
def test_rotary_elements_behind_the_pairs_pass_as_they_are(shape, dtype):
    """infinities, NaN and zeros of either sign behind the pairs, alone and beside each other: bit for bit the same in both directions, and the pairs in front know nothing of them"""
    b, n, hq, hk, d, sections, inter = shape
    rows, q, k, pos, freqs, _, _, g = rot_inputs(*shape[:6], dtype, 13)
    P = sum(sections)
    odd = torch.tensor([math.inf, -math.inf, math.nan, 0.0, -0.0, 3.0, -2.0], dtype=rows.dtype)
    rows[..., 2 * P:] = odd[torch.randint(0, 7, rows[..., 2 * P:].shape, generator=g)]
    r = rows.to(DEV)
    bits = {2: torch.int16, 4: torch.int32}[rows.element_size()]
    a, c = r[:, :, :hq].transpose(1, 2), r[:, :, hq:hq + hk].transpose(1, 2)
    fwd = ops.rotary_axes(a, c, pos.to(DEV), freqs.to(DEV), sections, interleaved=inter)
    bwd = ops.rotary_axes_bwd(a, c, pos.to(DEV), freqs.to(DEV), sections, interleaved=inter)
    for back, got in ((False, fwd), (True, bwd[:2])):
        for x, y in ((q, got[0]), (k, got[1])):
            y = y.cpu()
            same = y[..., 2 * P:].contiguous().view(bits) == x[..., 2 * P:].contiguous().view(bits)
            assert (same | (x[..., 2 * P:].isnan() & y[..., 2 * P:].isnan())).all()
            z = x.double()[..., :2 * P]
            want = R.turn(z, pos, freqs, sections, inter, back=back)
            R.check(y[..., :2 * P], want, rot_tol(want, pair_size(z, sections, inter), R.HALF[x.dtype]), 'pairs')


LONG_ROT = [  # several tokens a workgroup (tokens / 1024, in the gradient behind the norm / 512), a ragged last group, groups over two rows of the batch
    (1, 5003, 3, 2, 64, [16, 16], False), (3, 1671, 2, 3, 32, [5, 7], True), (1, 5003, 3, 2, 20, [3, 2], False), (1, 2100, 70, 1, 64, [8, 24], False), (2, 1300, 1, 70, 24, [1, 2, 3, 4], True),
    # more tokens than 2048 workgroups hold at a time: k makes its turns again
    (1, 33001, 1, 1, 256, [32, 32, 64], False), (2, 33001, 1, 2, 128, [9, 20, 20], False)]


@pytest.mark.parametrize('dtype', ['bf16', 'fp32'])
@pytest.mark.parametrize('norm', [False, True])
@pytest.mark.parametrize('shape', LONG_ROT, ids=str)
def test_rotary_of_several_tokens_a_workgroup(shape, norm, dtype):
    test_rotary(shape, norm, dtype)


@pytest.mark.parametrize('dtype', ['bf16', 'fp32'])
@pytest.mark.parametrize('norm', [False, True])
@pytest.mark.parametrize('shape', LONG_ROT, ids=str)
def test_rotary_bwd_of_several_tokens_a_workgroup(shape, norm, dtype):
    test_rotary_bwd(shape, norm, dtype)


def test_rotary_far_positions_keep_their_angle():
    n, d = 64, 64
    pos = (2 ** 30 - 1 - 977 * torch.arange(n)).to(torch.int32)[:, None]
    freqs = 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    x = torch.randn(1, 2, n, d, generator=gen(3))
    got, none = ops.rotary_axes(x.to(DEV), None, pos.to(DEV), freqs.to(DEV), [32])
    assert none is None
    want = R.rotary(x, pos[None], freqs, [32])
    # the product of position and frequency in 64 bits: 2^30 * 2^-53 radians
    R.check(got, want, rot_tol(want, pair_size(x.double(), [32], False), R.HALF[torch.float32]) + 2.0 ** -22 * pair_size(x.double(), [32], False), 'far')


def test_rotary_gradient_against_differences():
    b, n, h, d, sections = 1, 3, 2, 16, [3, 4]
    _, q, _, pos, freqs, qs, _, g = rot_inputs(b, n, h, 1, d, sections, 'fp32', 5)
    q = q.contiguous()
    w = torch.randn(b, h, n, d, generator=g)
    dq, _, ds, _ = ops.rotary_axes_bwd(w.to(DEV), None, pos.to(DEV), freqs.to(DEV), sections, q=q.to(DEV), q_scale=qs.to(DEV))
    f = lambda x, s: float((R.rotary(x, pos, freqs, sections, s) * w.double()).sum())
    q, qs, eps = q.double(), qs.double(), 1e-6
    for idx in [(0, 0, 0, 0), (0, 1, 2, 7), (0, 0, 1, 15), (0, 1, 0, 9)]:
        e = torch.zeros_like(q)
        e[idx] = eps
        assert abs((f(q + e, qs) - f(q - e, qs)) / (2 * eps) - float(dq[idx])) < 2e-5
    for c in (0, 8, 15):
        e = torch.zeros_like(qs)
        e[c] = eps
        assert abs((f(q, qs + e) - f(q, qs - e)) / (2 * eps) - float(ds[c])) < 2e-5


def test_rotary_of_nothing_and_of_a_zero_row():
    freqs = torch.ones(16, dtype=torch.float64, device=DEV)
    z = torch.zeros(1, 2, 0, 32, device=DEV, dtype=torch.bfloat16)
    p0 = torch.zeros(0, 1, dtype=torch.int32, device=DEV)
    assert ops.rotary_axes(z, z, p0, freqs, [16])[0].shape == z.shape
    s = torch.ones(32, device=DEV)
    _, _, ds, dks = ops.rotary_axes_bwd(z, z, p0, freqs, [16], q=z, k=z, q_scale=s, k_scale=s)
    assert ds.tolist() == [0.0] * 32 and dks.tolist() == [0.0] * 32
    x = torch.zeros(1, 1, 1, 32, device=DEV)
    y, _ = ops.rotary_axes(x, None, torch.zeros(1, 1, dtype=torch.int32, device=DEV), freqs, [16], q_scale=s)
    assert torch.equal(y, x)


def test_rotary_gradient_of_no_heads():
    """scales whose q or k has no heads: their gradients are zeros, whatever the workspace held"""
    freqs, pos, s = torch.ones(16, dtype=torch.float64, device=DEV), torch.zeros(700, 1, dtype=torch.int32, device=DEV), torch.ones(32, device=DEV)
    none, some = torch.zeros(1, 0, 700, 32, device=DEV), torch.randn(1, 2, 700, 32, generator=gen(14)).to(DEV)
    want = ops.rotary_axes_bwd(some, None, pos, freqs, [16], q=some, q_scale=s)[2]
    for q, k in ((none, None), (none, none), (none, some), (some, none)):
        held = [torch.full((1 << 18,), math.nan, device=DEV) for _ in range(4)]
        torch.cuda.synchronize()
        del held
        dq, dk, ds, dks = ops.rotary_axes_bwd(q, k, pos, freqs, [16], q=q, k=k, q_scale=s, k_scale=None if k is None else s)
        assert dq.shape == q.shape and (k is None or dk.shape == k.shape)
        for x, y in ((q, ds), (k, dks)):
            assert y is None and x is None or torch.equal(y, want if x is some else torch.zeros_like(s))


@pytest.mark.parametrize('dtype', ['bf16', 'fp32'])
@pytest.mark.parametrize('d,sections,inter', [(64, [16, 16], False), (20, [3, 2], False), (64, [8, 8, 7], True)])
def test_rotary_gradient_of_rows_below_the_norms_floor(d, sections, inter, dtype):
    """rows shorter than 1e-12 are divided by that constant: no projection in their gradient; against autograd of the formula in 64 bits"""
    sizes = torch.tensor([0.0, 1e-20, 1e-14, 3e-13, 8e-13, 9.8e-13, 1.03e-12, 3e-12, 1.0])
    n, g = len(sizes), gen(15)
    x = torch.randn(1, 2, n, d, generator=g)
    x = (x / x.norm(dim=-1, keepdim=True) * sizes[:, None]).to(DT[dtype])
    dy = torch.randn(1, 2, n, d, generator=g).to(DT[dtype])
    pos = torch.randint(0, 50, (n, len(sections)), generator=g).to(torch.int32)
    freqs = torch.cat([100.0 ** (-torch.arange(s, dtype=torch.float64) / s) for s in sections])
    s = 1 + 0.3 * torch.randn(d, generator=g)
    dx, _, ds, _ = ops.rotary_axes_bwd(dy.to(DEV), None, pos.to(DEV), freqs.to(DEV), sections, q=x.to(DEV), q_scale=s.to(DEV), interleaved=inter)
    leaf, scale = x.double().requires_grad_(), s.double().requires_grad_()
    ln = leaf.norm(dim=-1, keepdim=True).clamp(min=1e-12)
    gr = R.turn(dy.double(), pos[None], freqs, sections, inter, back=True)
    want, want_s = torch.autograd.grad((leaf / ln * scale * gr).sum(), (leaf, scale))
    ln, xh, size = ln.detach(), (leaf / ln).detach().abs(), pair_size(dy.double(), sections, inter)
    mag = (size * s.double().abs() + xh * (xh * size * s.double().abs()).sum(-1, keepdim=True)) / ln
    R.check(dx, want, rot_tol(want, mag * d / 8, R.HALF[x.dtype]), 'dx')
    R.check(ds[None], want_s[None], (R.F32 * (24 + d + 2 * math.sqrt(2 * n)) * (size * xh).sum((0, 1, 2)))[None], 'scale')


# ------------------------------------------------------------------------------------------------ attention
def att_inputs(b, hq, hk, n, j, d, dtype, mask, cap, axes, seed, unit=None):
    """operands on the CPU, spans, key mask, positions; the key rows are views of wider rows, as a projection leaves them"""
    g, rng = gen(seed), random.Random(seed)
    t = DT[dtype]
    unit = cap == 0.0 if unit is None else unit
    q = torch.randn(b, n, hq, d, generator=g)
    kv = torch.randn(b, j, 2 * hk, d, generator=g)
    if unit:
        q = q / q.norm(dim=-1, keepdim=True)
        kv[:, :, :hk] /= kv[:, :, :hk].norm(dim=-1, keepdim=True).clamp(min=1e-3)
    scale = 8.0 if unit else 2.0 * d ** -0.5
    spans = key_mask = None
    if mask in ('docs', 'prefix', 'causal', 'cross'):
        docs = max(1, n // 40)
        cu = bounds(rng, docs, n - n // 20)
        cu_k = cu if n == j else bounds(rng, docs, j)
        prefix = torch.tensor([rng.randint(0, 30) for _ in range(docs)], dtype=torch.int32) if mask == 'prefix' else None
        spans = R.spans_of(cu, cu_k, prefix, n, mask in ('prefix', 'causal'))
    elif mask == 'any':          # per row of the batch, in no order, empty and out of range ones among them
        lo = torch.randint(-5, j + 5, (b, n), generator=g)
        spans = torch.stack([lo, lo + torch.randint(-3, max(2, j), (b, n), generator=g)], 2).to(torch.int32)
    elif mask == 'keys':
        key_mask = torch.rand(b, j, generator=g) < 0.6
        key_mask[0] = False
    elif mask == 'both':
        key_mask = torch.rand(b, j, generator=g) < 0.7
        lo = torch.randint(0, max(1, j // 2), (n,), generator=g)
        spans = torch.stack([lo, lo + torch.randint(0, j // 2 + 1, (n,), generator=g)], 1).to(torch.int32)
    slopes = pos_q = pos_k = None
    if axes:
        slopes = 0.02 + 0.2 * torch.rand(hq, axes, generator=g)
        shape = (b, n, axes) if mask == 'any' else (n, axes)
        pos_q = torch.randint(0, 40, shape, generator=g).to(torch.int32)
        pos_k = torch.randint(0, 40, (j, axes), generator=g).to(torch.int32)
    return dict(q=q.to(t).transpose(1, 2), kv=kv.to(t), scale=scale, cap=cap, spans=spans, key_mask=key_mask, slopes=slopes, pos_q=pos_q, pos_k=pos_k, hk=hk)


def on_gpu(x):
    mv = lambda t: None if t is None else t.to(DEV)
    kv = x['kv'].to(DEV)
    return (x['q'].to(DEV), kv[:, :, :x['hk']].transpose(1, 2), kv[:, :, x['hk']:].transpose(1, 2), mv(x['spans'])), \
        dict(scale=x['scale'], softcap=x['cap'], slopes=mv(x['slopes']), positions=mv(x['pos_q']), key_positions=mv(x['pos_k']), key_mask=mv(x['key_mask']))


def plain(x, **more):
    b, _, n, _ = x['q'].shape
    k, v = x['kv'][:, :, :x['hk']].transpose(1, 2), x['kv'][:, :, x['hk']:].transpose(1, 2)
    seen = R.visible(n, k.shape[2], x['spans'], x['key_mask'], b)
    return R.attention(x['q'], k, v, seen, x['scale'], x['cap'], x['slopes'], x['pos_q'], x['pos_k'], **more)


ATT = [  # b, hq, hk, n, j, d, dtype, mask, cap, axes        -- few rows (keys split over waves and workgroups)
    (1, 1, 1, 1, 1, 64, 'bf16', 'none', 0.0, 0), (2, 8, 2, 1, 2000, 128, 'fp16', 'none', 30.0, 0), (3, 4, 4, 1, 700, 64, 'bf16', 'any', 0.0, 1),
    (1, 8, 8, 256, 256, 64, 'bf16', 'none', 0.0, 2), (1, 8, 8, 33, 65, 32, 'bf16', 'none', 0.0, 0), (2, 6, 3, 5, 999, 32, 'fp16', 'keys', 0.0, 3),
    (1, 16, 1, 3, 4097, 128, 'bf16', 'both', 20.0, 1), (2, 2, 1, 129, 31, 64, 'fp16', 'any', 0.0, 0), (1, 4, 2, 300, 300, 128, 'bf16', 'prefix', 30.0, 2),
    (1, 2, 2, 200, 90, 64, 'bf16', 'cross', 0.0, 0), (1, 3, 1, 64, 0, 64, 'bf16', 'none', 0.0, 0), (4, 12, 4, 2, 128, 64, 'bf16', 'keys', 50.0, 0),
    # many rows (128 queries a workgroup)
    (8, 16, 4, 200, 200, 32, 'bf16', 'docs', 0.0, 0), (8, 16, 16, 130, 257, 64, 'bf16', 'none', 0.0, 0), (4, 16, 8, 400, 400, 64, 'bf16', 'docs', 0.0, 2),
    (2, 16, 4, 1000, 1000, 128, 'bf16', 'prefix', 30.0, 0), (8, 16, 2, 256, 191, 64, 'fp16', 'any', 0.0, 1), (4, 32, 32, 256, 64, 128, 'fp16', 'keys', 0.0, 3),
    (4, 16, 16, 512, 63, 32, 'bf16', 'both', 10.0, 3), (2, 64, 1, 250, 250, 64, 'bf16', 'causal', 0.0, 1), (4, 32, 4, 129, 1, 128, 'bf16', 'none', 0.0, 0),
    (16, 16, 16, 129, 0, 32, 'fp16', 'none', 0.0, 0)]


@pytest.mark.parametrize('case', ATT, ids=lambda c: '-'.join(map(str, c)))
def test_attend_spans(case):
    x = att_inputs(*case, seed=21)
    args, kw = on_gpu(x)
    out, lse = ops.attend_spans(*args, **kw, return_lse=True)
    want = plain(x)
    R.check(lse, want['lse'], want['lse_tol'], 'lse')
    R.check(out, want['out'], want['out_tol'], 'out')
    rows = ops.attend_spans(*args, **kw, out_rows=True)
    b, hq, n, d = out.shape
    assert torch.equal(rows, out.permute(0, 2, 1, 3).reshape(b * n, hq * d))


@pytest.mark.parametrize('case', [(1, 2, 1, 300, 300, 64, 'bf16', 'docs', 0.0, 0), (8, 16, 16, 200, 200, 64, 'bf16', 'docs', 0.0, 2), (8, 16, 4, 200, 200, 128, 'fp16', 'both', 30.0, 0),
                                  (2, 8, 2, 1, 3000, 128, 'fp16', 'any', 0.0, 1), (2, 4, 4, 40, 200, 32, 'bf16', 'both', 0.0, 0)], ids=lambda c: '-'.join(map(str, c)))
@pytest.mark.parametrize('where', ['sevenths', 'second half'])
@pytest.mark.parametrize('value', [math.nan, math.inf])
def test_attend_spans_what_is_hidden_stays_out(case, value, where):
    """infinities and NaN in keys and values that a row does not see, rows of other documents and rows behind the last document among them, never reach it"""
    x = att_inputs(*case, seed=22)
    b, _, n, _ = x['q'].shape
    j = x['kv'].shape[1]
    seen = R.visible(n, j, x['spans'], x['key_mask'], b)
    want = plain(x)
    broken = ~seen.any(1)                                # keys that nothing sees, and every seventh, or all that the first half of the rows does not see
    if where == 'second half' or n == 1:                 # (a single long row sees some of the sevenths)
        broken = ~seen[:, :(n + 1) // 2].any(1)
    else:
        broken[:, ::7] = True
    x['kv'][broken] = value
    args, kw = on_gpu(x)
    out, lse = ops.attend_spans(*args, **kw, return_lse=True)
    clean = ~(seen & broken[:, None]).any(-1)            # rows that see no broken key
    assert clean.any()
    c = clean[:, None].expand(lse.shape)
    R.check(lse.cpu()[c], want['lse'][c], want['lse_tol'][c], 'lse')
    R.check(out.cpu()[c], want['out'][c], want['out_tol'][c], 'out')
    rest = ~c
    if rest.any():
        assert not out.cpu()[rest].isfinite().all(-1).any()


@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
@pytest.mark.parametrize('hq,n,j,drop', [(1, 1, 1 << 19, 17.6), (1, 1, 1 << 19, 20.0), (8, 1, 1 << 16, 15.0), (1, 40, 1 << 17, 17.6), (128, 129, 1 << 17, 17.6), (128, 129, 1 << 13, 14.0)])
def test_a_long_tail_of_small_weights(hq, n, j, drop, dtype):
    """one key that takes nearly everything before a long cache of keys whose weights are each below the smallest fp16 number (2^-24 of it) but together some
    thousandths: they count, in the narrow and the wide form"""
    d, t = 32, DT[dtype]
    q, k, v = torch.zeros(1, hq, n, d, dtype=t), torch.zeros(1, 1, j, d, dtype=t), torch.ones(1, 1, j, d, dtype=t)
    q[..., 0] = 1.0
    v[:, :, 5, ::2] = 0.0                                     # the one key's value: 0 in the even elements, 1 in the odd ones
    k[:, :, 5, 0] = drop
    k, v, q = k.to(DEV), v.to(DEV), q.to(DEV)
    out, lse = ops.attend_spans(q, k, v, scale=1.0, return_lse=True)
    top = float(torch.tensor(drop, dtype=t))
    tail = (j - 1) * math.exp(-top)
    want = torch.full(out.shape, tail / (1 + tail), dtype=torch.float64)
    want[..., 1::2] = 1.0
    # P and the result rounded once each; the sum in 32 bits: a lane has every other group of 4 keys, half of them, and adds them 8 at a time, so j / 16 additions to
    # a sum of about 1, each off by at most 2^-24 of it
    tol = want * (2.04 * R.HALF[t] + R.F32 * (64 + j / 16)) + 2.0 ** -24
    R.check(out, want, tol, 'out')
    R.check(lse, torch.full(lse.shape, top + math.log1p(tail), dtype=torch.float64), torch.full(lse.shape, R.F32 * (64 + j / 16 + 8 * top), dtype=torch.float64), 'lse')


@pytest.mark.parametrize('hq,n', [(2, 3), (128, 129)])
def test_subnormal_fp16_values_count(hq, n):
    """values below 2^-14 in fp16, as they are"""
    v = (torch.randint(-1000, 1001, (1, 1, 300, 64), generator=gen(97)) * 2.0 ** -24).to(torch.float16)
    q, k = torch.zeros(1, hq, n, 64, dtype=torch.float16), torch.zeros(1, 1, 300, 64, dtype=torch.float16)
    out = ops.attend_spans(q.to(DEV), k.to(DEV), v.to(DEV), scale=1.0)
    want = v.double().mean(2, keepdim=True).expand(1, hq, n, 64)
    R.check(out, want, 2.0 ** -25 * 1.01 + want.abs() * (2.0 ** -11 + 64 * R.F32), 'out')      # (P is 1: the result's rounding alone, to whole 2^-24)


@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
@pytest.mark.parametrize('hq,n', [(2, 3), (128, 129)])
@pytest.mark.parametrize('sign', [1.0, -1.0])
def test_scores_of_1e7(sign, hq, n, dtype):
    """the largest scores that are taken: 63 keys of the same score of 9e6 in size and 64 far below them; the weights are 1 / 63, whatever the score's last bit is worth"""
    t = DT[dtype]
    q, k = torch.zeros(1, hq, n, 32, dtype=t), torch.zeros(1, 1, 127, 32, dtype=t)
    q[..., 3], q[..., 7] = 3008.0, 256.0
    k[..., 3] = 3008.0 * sign
    k[:, :, 1::2, 7] = -2.0                                     # scores 512 lower: products of 8 bits each, exact in fp32
    v = torch.randn(1, 1, 127, 32, generator=gen(98)).to(t)
    k[:, :, 0, 7] = -2.0
    out, lse = ops.attend_spans(q.to(DEV), k.to(DEV), v.to(DEV), scale=1.0, return_lse=True)
    best = k[0, 0, :, 7] == 0
    assert int(best.sum()) == 63
    w = v[0, 0, best].double()
    want = w.mean(0).expand(out.shape)
    # P is the same number for all of them (2^0 .. 2^16, one rounding), and so is the sum's share; the result's rounding
    R.check(out, want, w.abs().mean(0).expand(out.shape) * (2.04 * R.HALF[t] + 64 * R.F32), 'out')
    top = 3008.0 ** 2 * sign
    R.check(lse, torch.full(lse.shape, top + math.log(63), dtype=torch.float64), torch.full(lse.shape, 4 * R.F32 * abs(top), dtype=torch.float64), 'lse')


@pytest.mark.parametrize('dtype', ['fp16', 'bf16'])
@pytest.mark.parametrize('hq,n', [(1, 1), (128, 129)])
def test_lse_of_few_keys_keeps_its_bits(hq, n, dtype):
    """rows that see 1 .. 40 keys of score 0: lse is log(keys), whatever the weights are scaled by for their 16 bits"""
    t, j = DT[dtype], 40
    q, k = torch.zeros(j, hq, n, 32, dtype=t, device=DEV), torch.zeros(j, 1, j, 32, dtype=t, device=DEV)
    spans = torch.stack([torch.zeros(j, n), (torch.arange(j) + 1.0)[:, None].expand(j, n)], 2).to(torch.int32)
    _, lse = ops.attend_spans(q, k, k, spans.to(DEV), scale=1.0, return_lse=True)
    want = torch.arange(1, j + 1).double().log()[:, None, None].expand(j, hq, n)
    # the logarithm of a whole number (an ulp of up to 5.4), the reference beside it (0 or a power of two away), ln 2 and its product
    R.check(lse, want, 5 * R.F32 * want + 1e-30, 'lse')


def test_attend_spans_sees_through_strides_and_expanded_operands():
    """keys shared by a batch (batch stride 0), token-major and head-major operands, a slice of a longer cache"""
    g = gen(9)
    cache = torch.randn(2, 4, 500, 64, generator=g).to(torch.bfloat16).to(DEV)
    q = torch.randn(3, 8, 70, 64, generator=g).to(torch.bfloat16).to(DEV)
    k, v = cache[0, :, 17:317].expand(3, 4, 300, 64), cache[1, :, 17:317].expand(3, 4, 300, 64)
    a = ops.attend_spans(q, k, v, scale=0.125)
    b = ops.attend_spans(q.contiguous(), k.contiguous(), v.contiguous(), scale=0.125)
    assert torch.equal(a, b)


def test_attend_spans_wide_and_narrow_agree_and_repeat():
    """the same rows alone (keys split) and among many (128 queries a workgroup): within two roundings of P and of the result, and each the same bits every time"""
    x = att_inputs(16, 16, 16, 150, 150, 64, 'bf16', 'docs', 0.0, 2, seed=31)
    args, kw = on_gpu(x)
    many = ops.attend_spans(*args, **kw)
    assert torch.equal(many, ops.attend_spans(*args, **kw))
    one = ops.attend_spans(args[0][:1], args[1][:1], args[2][:1], args[3], **kw)
    assert torch.equal(one, ops.attend_spans(args[0][:1], args[1][:1], args[2][:1], args[3], **kw))
    want = plain(x)
    R.check(one - many[:1].float(), torch.zeros_like(want['out'][:1]), 2 * want['out_tol'][:1], 'difference')


BWD = [c for c in ATT if c[6] == 'bf16'] + [(2, 4, 1, 700, 130, 128, 'bf16', 'any', 20.0, 1), (1, 2, 2, 17000, 40, 32, 'bf16', 'none', 0.0, 1), (1, 3, 3, 60, 700, 64, 'bf16', 'both', 0.0, 3),
                                            (2, 8, 2, 257, 257, 128, 'bf16', 'docs', 0.0, 3)]


def bwd_inputs(case, seed):
    x = att_inputs(*case, seed=seed)
    f = plain(x)
    dt = DT[case[6]]
    out, lse = f['out'].to(dt), f['lse'].float()
    dout = torch.randn(out.shape, generator=gen(seed + 1)).to(dt)
    return x, out, lse, dout


@pytest.mark.parametrize('case', BWD, ids=lambda c: '-'.join(map(str, c)))
def test_attend_spans_bwd(case):
    x, out, lse, dout = bwd_inputs(case, 41)
    args, kw = on_gpu(x)
    # gradients arrive as a projection's rows: (b, n, h, d)
    rows = dout.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
    got = ops.attend_spans_bwd(*args[:3], out.to(DEV), lse.to(DEV), rows, args[3], **kw)
    want = plain(x, dout=dout, out=out, lse=lse)
    for name, t in zip(('dq', 'dk', 'dv', 'dslopes'), got):
        if name == 'dslopes' and x['slopes'] is None:
            assert t is None
            continue
        R.check(t, want[name], want[name + '_tol'], name)
    again = ops.attend_spans_bwd(*args[:3], out.to(DEV), lse.to(DEV), rows, args[3], **kw)
    for a, c in zip(got, again):
        assert a is None or torch.equal(a, c)


@pytest.mark.parametrize('case', [(1, 2, 1, 300, 300, 64, 'bf16', 'docs', 0.0, 0), (2, 4, 2, 200, 200, 128, 'bf16', 'both', 30.0, 1), (2, 2, 2, 150, 90, 32, 'bf16', 'any', 0.0, 0)],
                         ids=lambda c: '-'.join(map(str, c)))
@pytest.mark.parametrize('value', [math.nan, math.inf])
def test_attend_spans_bwd_what_is_hidden_stays_out(case, value):
    """broken keys and broken gradient rows: queries that see no broken key and keys that no broken row sees have the gradients of a clean batch"""
    x, out, lse, dout = bwd_inputs(case, 42)
    b, _, n, _ = x['q'].shape
    j = x['kv'].shape[1]
    seen = R.visible(n, j, x['spans'], x['key_mask'], b)
    want = plain(x, dout=dout, out=out, lse=lse)
    keys = ~seen[:, :n // 2].any(1)                          # keys that the first half of the rows does not see
    x['kv'][keys] = value
    rows = ~seen.any(-1)                                     # rows that see nothing, and a few of the second half
    rows[:, n // 2 + 3::17] = True
    dout.transpose(1, 2)[rows] = value
    x['q'].transpose(1, 2)[~seen.any(-1)] = value
    out.transpose(1, 2)[~seen.any(-1)] = value
    args, kw = on_gpu(x)
    dq, dk, dv, ds = ops.attend_spans_bwd(*args[:3], out.to(DEV), lse.to(DEV), dout.to(DEV), args[3], **kw)
    cq = ~(seen & keys[:, None]).any(-1) & (~rows | ~seen.any(-1))
    ck = ~(seen & rows[:, :, None]).any(1) & ~(keys & seen.any(1))
    assert cq.any() and ck.any()
    cq, ck = cq[:, None].expand(dq.shape[:3]), ck[:, None].expand(dk.shape[:3])
    R.check(dq.cpu()[cq], want['dq'][cq], want['dq_tol'][cq], 'dq')
    R.check(dk.cpu()[ck], want['dk'][ck], want['dk_tol'][ck], 'dk')
    R.check(dv.cpu()[ck], want['dv'][ck], want['dv_tol'][ck], 'dv')


def test_attend_spans_gradients_against_differences():
    """scale 1, two heads over one key head, capped, biased: the kernel's gradients against central differences of the 64-bit forward along random directions"""
    case = (1, 2, 1, 24, 24, 32, 'bf16', 'causal', 5.0, 2)
    x = att_inputs(*case, seed=51)
    f = plain(x)
    out, lse = f['out'].to(torch.bfloat16), f['lse'].float()
    g = gen(52)
    dout = torch.randn(out.shape, generator=g).to(torch.bfloat16)
    args, kw = on_gpu(x)
    got = ops.attend_spans_bwd(*args[:3], out.to(DEV), lse.to(DEV), dout.to(DEV), args[3], **kw)
    seen = R.visible(24, 24, x['spans'])
    q, k, v, s = x['q'].double(), x['kv'][:, :, :1].transpose(1, 2).double(), x['kv'][:, :, 1:].transpose(1, 2).double(), x['slopes'].double()

    def value(q, k, v, s):
        t = q @ k.transpose(2, 3) * x['scale']
        t = 5.0 * torch.tanh(t / 5.0)
        t = t - torch.einsum('ha,nja->hnj', s, (x['pos_q'][:, None] - x['pos_k'][None]).abs().double())
        p = torch.softmax(t.masked_fill(~seen[:, None], -1e300), -1) * seen[:, None]
        return float(((p @ v) * dout.double()).sum())
    eps = 1e-6
    for n, t in enumerate((q, k, v, s)):
        e = torch.randn(t.shape, generator=g).double()
        up, down = [q, k, v, s], [q, k, v, s]
        up[n], down[n] = t + eps * e, t - eps * e
        diff = (value(*up) - value(*down)) / (2 * eps)
        grad = got[n].detach().cpu().double()
        # three roundings to bf16 (out, an operand, the result) of every term
        assert abs(float((grad * e).sum()) - diff) < 3 * 2.0 ** -8 * float((grad * e).abs().sum()) + 1e-6, ('q', 'k', 'v', 'slopes')[n]


CAPS = [(1e-3, 1.0), (1.0, 0.125), (30.0, 1.0), (50.0, 8.0), (1e4, 1.0)]


@pytest.mark.parametrize('cap,scale', CAPS)
@pytest.mark.parametrize('hq,n,d', [(1, 400, 64), (2, 400, 32), (1, 400, 128)])
@pytest.mark.parametrize('axes', [0, 1])
def test_a_capped_score_keeps_the_bits_of_its_own_size(axes, hq, n, d, cap, scale):
    """few rows: a row that sees one key has that score as its lse, within a few fp32 roundings of the score itself, from 1e-6 of the cap to far beyond it, either sign, on tiles of
    small scores alone and beside large ones"""
    u = torch.cat([torch.logspace(-6, -0.05, 200), torch.logspace(-6, 1.5, 200)]).double()      # the first tiles stay below the cap, the others do not
    u = u * torch.where(torch.arange(400) % 3 == 0, -1.0, 1.0)
    q, k = torch.zeros(1, hq, n, d), torch.zeros(1, 1, n, d)
    q[..., 5], k[..., 5] = 1.0, (u * cap / scale).float()
    q, k = q.to(torch.bfloat16), k.to(torch.bfloat16)
    at = torch.arange(n, dtype=torch.int32)
    spans = torch.stack([at, at + 1], 1)
    kw = {}
    if axes:
        kw = dict(slopes=torch.full((hq, 1), 0.25 * cap), positions=at[:, None] * 3, key_positions=at[:, None] * 3 - 1)
    g = lambda t: t.to(DEV) if isinstance(t, torch.Tensor) else t
    _, lse = ops.attend_spans(g(q), g(k), g(k), g(spans), scale=scale, softcap=cap, return_lse=True, **{a: g(b) for a, b in kw.items()})
    want = cap * torch.tanh(k[0, 0, :, 5].double() * scale / cap)
    size = want.abs()
    if axes:
        size = size + 0.25 * cap
        want = want - 0.25 * cap
    # scale / cap, its product, four roundings in tanh, the cap in units of log2, the product with it, back to natural units; log2 of the sum (exact: 1) -- a dozen at most
    R.check(lse, want.expand(1, hq, n), (12 * R.F32 * size + 1e-37).expand(1, hq, n), 'lse')


@pytest.mark.parametrize('d,hk', [(32, 2), (64, 4), (128, 2)])
@pytest.mark.parametrize('cap,axes', [(1000.0, 1), (10000.0, 2)])
@pytest.mark.parametrize('big', [False, True])
def test_slope_gradients_behind_a_cap_far_above_the_scores(d, hk, cap, axes, big):
    """the slopes' gradient, which no rounding to 16 bits follows, of scores of a few units under a large cap, and (big) of a few beyond it among them: within fp32 roundings of the
    scores' own size, not of the cap's"""
    x = att_inputs(2, 4, hk, 5, 6, d, 'bf16', 'none', cap, axes, seed=99)
    # one element a head: the products are exact, so that the bound is that of the cap alone; few pairs, whose errors do not cancel
    keep = x['q'][..., :1].clone()
    x['q'].zero_()
    x['q'][..., :1] = keep
    x['kv'][..., 1:] = 0
    x['scale'] = 2.0
    if big:
        x['q'][:, :, 0, 0], x['kv'][:, 3, :hk, 0] = 1.5, 1.25 * cap
    f = plain(x)
    out, lse = f['out'].to(torch.bfloat16), f['lse'].float()
    args, kw = on_gpu(x)
    dout = torch.randn(out.shape, generator=gen(100)).to(torch.bfloat16)
    dout[..., 1:] = 0
    got = ops.attend_spans_bwd(*args[:3], out.to(DEV), lse.to(DEV), dout.to(DEV), args[3], **kw)
    want = plain(x, dout=dout, out=out, lse=lse)
    for name, t in zip(('dq', 'dk', 'dv'), got):
        R.check(t, want[name], want[name + '_tol'], name)
    want = plain(x, dout=dout, out=out, lse=lse, tight_cap=True)
    R.check(got[3], want['dslopes'], want['dslopes_tol'], 'dslopes')


def test_packed_training_pass_of_all_operators_together():
    """a layer's attention over a packed row, as a model runs it: projection rows -> l2norm, scales and positions -> attention by document with a distance bias, and
    the way back; against the same chain in 64 bits"""
    rng, g = random.Random(7), gen(7)
    h, d, n = 4, 64, 331
    sections, freqs = [16, 16], torch.cat([100.0 ** (-torch.arange(16, dtype=torch.float64) / 16)] * 2)
    cu = torch.tensor([0, 64, 64, 180, 316], dtype=torch.int32)
    prefix = torch.tensor([10, 0, 30, 0], dtype=torch.int32)
    pos = torch.stack([torch.arange(n) // 16, torch.arange(n) % 16], 1).to(torch.int32)
    rows = torch.randn(1, n, 3 * h, d, generator=g).to(torch.bfloat16)
    qs, ks = 1 + 0.2 * torch.randn(d, generator=g), 1 + 0.2 * torch.randn(d, generator=g)
    slopes = 0.05 + 0.1 * torch.rand(h, 2, generator=g)
    w = torch.randn(1, n, h, d, generator=g).to(torch.bfloat16).transpose(1, 2)
    r = rows.to(DEV)
    q, k, v = (r[:, :, x * h:(x + 1) * h].transpose(1, 2) for x in range(3))
    p, f, s = pos.to(DEV), freqs.to(DEV), slopes.to(DEV)
    spans = ops.attention_spans(cu.to(DEV), n, prefix=prefix.to(DEV), causal=True)
    qr, kr = ops.rotary_axes(q, k, p, f, sections, q_scale=qs.to(DEV), k_scale=ks.to(DEV))
    out, lse = ops.attend_spans(qr, kr, v, spans, slopes=s, positions=p, return_lse=True)
    dqr, dkr, dv, dsl = ops.attend_spans_bwd(qr, kr, v, out, lse, w.to(DEV), spans, slopes=s, positions=p)
    dq, dk, dqs, dks = ops.rotary_axes_bwd(dqr, dkr, p, f, sections, q=q, k=k, q_scale=qs.to(DEV), k_scale=ks.to(DEV))
    leaves = [t.double().requires_grad_() for t in (rows, qs, ks, slopes)]
    x = leaves[0]
    z = [x[:, :, a * h:(a + 1) * h].transpose(1, 2) for a in range(3)]
    z[0], z[1] = (turn_autograd(t / t.norm(dim=-1, keepdim=True) * sc, pos, freqs) for t, sc in ((z[0], leaves[1]), (z[1], leaves[2])))
    seen = R.visible(n, n, R.spans_of(cu, cu, prefix, n, True))
    t = z[0] @ z[1].transpose(2, 3) * 8 - torch.einsum('ha,nja->hnj', leaves[3], (pos[:, None] - pos[None]).abs().double())
    pr = torch.softmax(t.masked_fill(~seen[:, None], -1e300), -1) * seen[:, None]
    o = pr @ z[2]
    grads = torch.autograd.grad((o * w.double()).sum(), leaves)
    # bf16 between the operators: the scores (|s| up to 8 |q_scale k_scale|) move by a few 2^-8 of themselves, everything behind them by as much in relation to its size
    rel = lambda a, b: float((a.cpu().double() - b).norm() / b.norm())
    bound = 8 * 2.0 ** -8
    assert rel(out, o.detach()) < bound
    assert rel(torch.cat([dq, dk, dv], 1).transpose(1, 2), grads[0]) < bound
    assert rel(dqs, grads[1]) < bound and rel(dks, grads[2]) < bound and rel(dsl, grads[3]) < bound
    assert not out[:, :, 316:].any() and not dq[:, :, 316:].any() and not dk[:, :, 316:].any() and not dv[:, :, 316:].any()


def turn_autograd(x, pos, freqs):
    ang = pos.double()[:, [0] * 16 + [1] * 16] * freqs
    a, b = x[..., :32], x[..., 32:]
    return torch.cat([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()], -1)


def test_packed_rows_in_a_captured_graph():
    """the whole chain captured once and replayed over new inputs, with eager work between the replays; a second graph of the same operators beside it"""
    g = gen(61)
    h, d, n = 8, 64, 400
    f, s = torch.ones(32, dtype=torch.float64, device=DEV) * 0.1, torch.rand(h, 1, generator=g).to(DEV) * 0.1
    pos = torch.arange(n, dtype=torch.int32, device=DEV)[:, None]
    cu = torch.tensor([0, 100, 250, 390], dtype=torch.int32, device=DEV)
    scale = torch.ones(d, device=DEV)

    def chain(rows, w):
        q, k, v = (rows[:, :, x * h:(x + 1) * h].transpose(1, 2) for x in range(3))
        spans = ops.attention_spans(cu, n)
        qr, kr = ops.rotary_axes(q, k, pos, f, [32], q_scale=scale, k_scale=scale)
        out, lse = ops.attend_spans(qr, kr, v, spans, slopes=s, positions=pos, return_lse=True)
        one = ops.attend_spans(qr[:, :, -20:-19], kr, v, slopes=s, positions=pos[-20:-19], key_positions=pos, softcap=9.0)
        return (out, lse, one) + ops.attend_spans_bwd(qr, kr, v, out, lse, w, spans, slopes=s, positions=pos)

    new = lambda: (torch.randn(1, n, 3 * h, d, generator=g).to(torch.bfloat16).to(DEV), torch.randn(1, n, h, d, generator=g).to(torch.bfloat16).to(DEV).transpose(1, 2))
    graphs = []
    for _ in range(2):
        rows, w = new()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            chain(rows, w)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            got = chain(rows, w)
        graphs.append((gr, rows, w, got))
    for turn in range(4):
        for gr, rows, w, got in graphs:
            a, b = new()
            rows.copy_(a)
            w.copy_(b)
            gr.replay()
            want = chain(a, b)
            torch.cuda.synchronize()
            for x, y in zip(got, want):
                assert torch.equal(x, y), turn


def test_packed_rows_on_a_stream_of_their_own():
    g = gen(71)
    x = torch.randn(2, 200, 12, 64, generator=g).to(torch.bfloat16).to(DEV)
    q, k, v = (x[:, :, a * 4:(a + 1) * 4].transpose(1, 2) for a in range(3))
    want, wl = ops.attend_spans(q, k, v, return_lse=True)
    wb = ops.attend_spans_bwd(q, k, v, want, wl, q)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out, lse = ops.attend_spans(q, k, v, return_lse=True)
        got = ops.attend_spans_bwd(q, k, v, out, lse, q)
    side.synchronize()
    assert torch.equal(out, want) and torch.equal(lse, wl) and all(torch.equal(a, c) for a, c in zip(got[:3], wb[:3]))


@pytest.mark.parametrize('d,cap,axes', [(32, 0.0, 1), (64, 0.0, 0), (128, 20.0, 2)])
def test_one_broken_element_in_many_rows(d, cap, axes):
    """one NaN in v, seen by all, and one in dout: every row and key is computed again on its own, and only what the formula reaches is NaN"""
    x, out, lse, dout = bwd_inputs((1, 4, 2, 1100, 1100, d, 'bf16', 'none', cap, axes), 91)
    want = {**plain(x), **plain(x, dout=dout, out=out, lse=lse)}
    args, kw = on_gpu(x)
    v = args[2].clone()
    v[0, 1, 700, 3] = math.nan
    got = ops.attend_spans(args[0], args[1], v, args[3], **kw)
    assert got[:, 2:, :, 3].isnan().all() and got.isnan().sum() == 2 * 1100
    clean = ~got.isnan().cpu()
    R.check(got.cpu()[clean], want['out'][clean], want['out_tol'][clean], 'out')
    g = dout.clone()
    g[0, 3, 50, 5] = math.nan                                   # row 50 of head 3 (key head 1)
    dq, dk, dv, ds = ops.attend_spans_bwd(*args[:3], out.to(DEV), lse.to(DEV), g.to(DEV), args[3], **kw)
    assert dq[0, 3, 50].isnan().all() and dq.isnan().sum() == d
    assert dk[0, 1].isnan().all() and dk.isnan().sum() == 1100 * d
    assert dv[0, 1, :, 5].isnan().all() and dv.isnan().sum() == 1100
    for name, t in (('dq', dq), ('dk', dk), ('dv', dv)):
        clean = ~t.isnan().cpu()
        R.check(t.cpu()[clean], want[name][clean], want[name + '_tol'][clean], name)
    if axes:
        assert ds[3].isnan().all() and ds.isnan().sum() == axes


def test_everything_broken_ends_soon():
    """a diverged step: all of dout NaN.  Rows and keys stop at their first NaN sum instead of walking every pair"""
    g = gen(92)
    q, k, v = (torch.randn(1, 4, 4096, 64, generator=g).to(torch.bfloat16).to(DEV) for _ in range(3))
    out, lse = ops.attend_spans(q, k, v, return_lse=True)
    dq, dk, dv, _ = ops.attend_spans_bwd(q, k, v, out, lse, torch.full_like(out, math.nan))
    assert dq.isnan().all() and dk.isnan().all() and dv.isnan().all()
    out, lse = ops.attend_spans(q, k, torch.full_like(v, math.nan), return_lse=True)
    assert out.isnan().all() and lse.isfinite().all()


@pytest.mark.parametrize('hq,hk,d', [(8, 1, 128), (4, 2, 64)])
def test_rows_behind_the_last_document_on_a_poisoned_workspace(hq, hk, d):
    """300 rows of documents in 900: whole key tiles that nothing sees get zeros from every split, whatever the workspace and those rows held"""
    g = gen(93)
    n = 900
    q = torch.randn(1, n, hq, d, generator=g).to(torch.bfloat16).to(DEV).transpose(1, 2)
    k, v = (torch.randn(1, n, hk, d, generator=g).to(torch.bfloat16).to(DEV).transpose(1, 2) for _ in range(2))
    spans = ops.attention_spans(torch.tensor([0, 120, 300], dtype=torch.int32, device=DEV), n, causal=True)
    s, pos = torch.rand(hq, 1, generator=g).to(DEV), torch.arange(n, dtype=torch.int32, device=DEV)[:, None]
    kw = dict(scale=d ** -0.5, slopes=s, positions=pos)
    out, lse = ops.attend_spans(q, k, v, spans, return_lse=True, **kw)
    dout = torch.randn(out.shape, generator=g).to(torch.bfloat16).to(DEV)
    short = [t[:, :, :300] for t in (q, k, v, out, lse, dout)]
    want = ops.attend_spans_bwd(*short, spans[:300], scale=d ** -0.5, slopes=s, positions=pos[:300])
    for t in (q, k, v, dout):
        t[:, :, 300:] = math.nan
    for _ in range(3):
        held = [torch.full((1 << 23,), math.nan, device=DEV) for _ in range(2)]
        torch.cuda.synchronize()
        del held
        got = ops.attend_spans_bwd(q, k, v, out, lse, dout, spans, **kw)
        for a, b in zip(got[:3], want[:3]):
            assert (a[:, :, 300:] == 0).all()
            # other splits and tiles than the short call's: the sums' order, one rounding to bf16 apart, and that of the terms' sizes
            torch.testing.assert_close(a[:, :, :300].float(), b.float(), rtol=2 ** -7, atol=2 ** -7 * float(b.float().abs().max()))
        torch.testing.assert_close(got[3], want[3], rtol=1e-4, atol=1e-4 * float(want[3].abs().max()))


@pytest.mark.parametrize('n,j', [(0, 50), (50, 0), (0, 0)])
def test_attention_of_nothing(n, j):
    q = torch.ones(2, 4, n, 64, dtype=torch.bfloat16, device=DEV)
    k, v = (torch.ones(2, 2, j, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    pq, pk = (torch.zeros(x, 2, dtype=torch.int32, device=DEV) for x in (n, j))
    kw = dict(slopes=torch.ones(4, 2, device=DEV), positions=pq, key_positions=pk)
    out, lse = ops.attend_spans(q, k, v, return_lse=True, **kw)
    assert out.shape == q.shape and (out == 0).all() and (lse == -math.inf).all()
    dq, dk, dv, ds = ops.attend_spans_bwd(q, k, v, out, lse, q, **kw)
    assert dq.shape == q.shape and dk.shape == k.shape and dv.shape == v.shape
    for t in (dq, dk, dv, ds):
        assert (t == 0).all()


@pytest.mark.parametrize('n', [1, 600])
def test_a_cache_whose_offsets_pass_32_bits(n):
    """the last 700 of 2^19 rows, 4608 elements apart: byte offsets above 2^32, element offsets above 2^31; the rows before hold NaN and are not seen"""
    g = gen(94)
    j, seen, hq, d = 1 << 19, 700, 64, 128
    rows = torch.full((1, j, 4608), math.nan, dtype=torch.bfloat16, device=DEV)
    kv = torch.randn(1, seen, 2, d, generator=g).to(torch.bfloat16).to(DEV)
    rows[:, -seen:, :d], rows[:, -seen:, 4352:4352 + d] = kv[:, :, 0], kv[:, :, 1]
    k, v = rows[:, None, :, :d], rows[:, None, :, 4352:4352 + d]
    q, dout = (torch.randn(1, hq, n, d, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    at = torch.arange(n, dtype=torch.int32, device=DEV)
    near = torch.stack([at * 0, at + seen - n + 1], 1).to(torch.int32)
    far = near + (j - seen)
    kw = dict(scale=d ** -0.5, softcap=20.0)
    close = lambda a, b: torch.testing.assert_close(a.float(), b.float(), rtol=2 ** -7, atol=2 ** -7 * float(b.float().abs().max()))      # (one rounding to bf16 each, and that of P)
    kc, vc = kv[:, None, :, 0].contiguous(), kv[:, None, :, 1].contiguous()
    out, lse = ops.attend_spans(q, k, v, far, return_lse=True, **kw)
    want, want_lse = ops.attend_spans(q, kc, vc, near, return_lse=True, **kw)
    close(out, want)
    torch.testing.assert_close(lse, want_lse, rtol=1e-5, atol=1e-5)
    dq, dk, dv, _ = ops.attend_spans_bwd(q, k, v, want, want_lse, dout, far, **kw)
    wq, wk, wv, _ = ops.attend_spans_bwd(q, kc, vc, want, want_lse, dout, near, **kw)
    close(dq, wq)
    close(dk[:, :, -seen:], wk)
    close(dv[:, :, -seen:], wv)
    assert (dk[:, :, :-seen] == 0).all() and (dv[:, :, :-seen] == 0).all()


def test_two_streams_at_once():
    """gradients with slopes on two streams side by side, over and over: each call's workspace and counts are its own"""
    g = gen(95)
    n, h, d = 1500, 8, 64
    s, pos = torch.rand(h, 2, generator=g).to(DEV), torch.stack([torch.arange(n) // 40, torch.arange(n) % 40], 1).to(torch.int32).to(DEV)
    spans = ops.attention_spans(torch.tensor([0, 500, 1300], dtype=torch.int32, device=DEV), n)
    kw = dict(slopes=s, positions=pos)
    sets = []
    for _ in range(2):
        q, k, v, w = (torch.randn(1, n, h, d, generator=g).to(torch.bfloat16).to(DEV).transpose(1, 2) for _ in range(4))
        out, lse = ops.attend_spans(q, k, v, spans, return_lse=True, **kw)
        sets.append(((q, k, v, out, lse, w, spans), ops.attend_spans_bwd(q, k, v, out, lse, w, spans, **kw), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for a, _, stream in sets:
            with torch.cuda.stream(stream):
                got.append(ops.attend_spans_bwd(*a, **kw))
        torch.cuda.synchronize()
        for (_, want, _), x in zip(sets, got):
            assert all(torch.equal(c, e) for c, e in zip(x, want))


MANY = [  # tiles sorted longest first (batch x tiles x heads >= 512 with spans), too many of them to sort (more than 4096), documents that end inside tiles
    (16, 16, 4, 257, 257, 64, 'bf16', 'docs', 0.0, 2), (16, 16, 4, 257, 257, 128, 'bf16', 'docs', 30.0, 1), (16, 16, 16, 150, 150, 64, 'bf16', 'docs', 0.0, 2),
    (8, 32, 8, 300, 300, 32, 'bf16', 'prefix', 0.0, 0), (16, 16, 16, 260, 90, 64, 'bf16', 'any', 20.0, 0), (2100, 1, 1, 130, 130, 32, 'bf16', 'any', 0.0, 0)]


@pytest.mark.parametrize('case', MANY, ids=lambda c: '-'.join(map(str, c)))
def test_attend_spans_of_many_tiles(case):
    test_attend_spans(case)


MANY_BWD = MANY + [
    # heads that share a key head: two workgroups of two heads each, one of all four, three of two (batch x key heads x key tiles against 512)
    (8, 16, 4, 70, 1100, 64, 'bf16', 'none', 0.0, 2), (8, 16, 4, 70, 1100, 128, 'bf16', 'both', 30.0, 1), (16, 16, 4, 50, 1100, 128, 'bf16', 'any', 0.0, 0),
    (16, 16, 4, 50, 1100, 32, 'bf16', 'keys', 0.0, 1), (9, 24, 4, 40, 700, 64, 'bf16', 'any', 20.0, 3),
    # more than 256 tiles of 64 queries: the list of a key tile in two stretches
    (1, 2, 2, 16500, 40, 128, 'bf16', 'none', 0.0, 0), (1, 2, 1, 16500, 140, 128, 'bf16', 'any', 20.0, 2), (1, 2, 2, 16500, 200, 64, 'bf16', 'docs', 0.0, 1)]


@pytest.mark.parametrize('case', MANY_BWD, ids=lambda c: '-'.join(map(str, c)))
def test_attend_spans_bwd_of_many_tiles(case):
    test_attend_spans_bwd(case)


def test_everything_broken_in_bounded_time():
    """a diverged step of 4096 x 4096, gradients and forward: every row and key is looked at again, each until its first sum that is not finite -- milliseconds; a walk over all
    of its pairs would take each 64 times as long and the call seconds"""
    g = gen(92)
    q, k, v = (torch.randn(1, 4, 4096, 64, generator=g).to(torch.bfloat16).to(DEV) for _ in range(3))
    out, lse = ops.attend_spans(q, k, v, return_lse=True)
    bad = torch.full_like(out, math.nan)
    for call in (lambda: ops.attend_spans(q, k, bad), lambda: ops.attend_spans_bwd(q, k, v, out, lse, bad)):
        call()
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        call()
        b.record()
        b.synchronize()
        assert a.elapsed_time(b) < 200, 'ms'
