"""What the packed-row operators refuse, and their plain forms against autograd (CPU)."""
import pytest
import torch

import packed_rows as R
from muse_maskgit_pytorch_amd import _lib, ops

BF = torch.bfloat16


def refuses(match, fn, *a, **k):
    with pytest.raises(_lib.MuseHipError, match=match):
        fn(*a, **k)


def test_spans_refusals():
    cu = torch.tensor([0, 4, 9], dtype=torch.int32)
    for match, a, k in [('int32', (cu.long(), 9), {}), ('at least one bound', (cu[:0], 9), {}), ('one length', (cu, 9), dict(cu_k=cu[:2], j=9)),
                        ('number of keys', (cu, 9), dict(cu_k=cu)), ('one prefix', (cu, 9), dict(prefix=cu, causal=True)),
                        ('without causal', (cu, 9), dict(prefix=cu[:2])), ('0 to', (cu, -1), {}), ('batch sizes', (cu[None], 9), dict(cu_k=torch.stack([cu, cu]), j=9)),
                        ('one or two', (cu[None, None], 9), {})]:
        refuses(match, ops.attention_spans, *a, **k)


def test_rotary_refusals():
    q, k = torch.zeros(2, 4, 5, 64, dtype=BF), torch.zeros(2, 2, 5, 64, dtype=BF)
    pos, f = torch.zeros(5, 2, dtype=torch.int32), torch.zeros(32, dtype=torch.float64)
    s = torch.ones(64)
    ok = dict(q=q, k=k, positions=pos, freqs=f, sections=[16, 16])
    for match, change in [('float64', dict(freqs=f.float())), ('one per pair', dict(freqs=f[:31])), ('int32', dict(positions=pos.long())), ('shape', dict(positions=pos[:4])),
                          ('shape', dict(positions=pos[:, :1])), ('both scales', dict(q_scale=s)), ('both scales', dict(k_scale=s)), ('fp32', dict(q_scale=s.double(), k_scale=s)),
                          ('fp32', dict(q_scale=s, k_scale=s[:32])), ('sections', dict(sections=[])), ('sections', dict(sections=[7] * 5)), ('twice the sum', dict(sections=[16, 17], freqs=torch.zeros(33).double())),
                          ('beside', dict(k=k.float())), ('beside', dict(k=k[:, :, :4])), ('contiguous', dict(q=torch.zeros(2, 4, 64, 5, dtype=BF).transpose(2, 3))),
                          ('bf16, fp16', dict(q=q.double(), k=k.double())), ('even', dict(q=q[..., :63], k=k[..., :63], sections=[3, 3], freqs=torch.zeros(6).double())),
                          ('k_scale without k', dict(k=None, q_scale=s, k_scale=s)), ('tensors', dict(q=q[0]))]:
        refuses(match, ops.rotary_axes, **{**ok, **change})
    refuses('needs q', ops.rotary_axes_bwd, q, k, pos, f, [16, 16], k=k, q_scale=s, k_scale=s)
    refuses('needs k', ops.rotary_axes_bwd, q, k, pos, f, [16, 16], q=q, q_scale=s, k_scale=s)


def att(**change):
    q, k = torch.zeros(2, 4, 5, 64, dtype=BF), torch.zeros(2, 2, 7, 64, dtype=BF)
    return {**dict(q=q, k=k, v=k.clone()), **change}


ATT_REFUSALS = [
    ('one type', dict(k=torch.zeros(2, 2, 7, 64, dtype=torch.float16))), ('bf16 or fp16', dict(q=torch.zeros(2, 4, 5, 64))), ('query heads', dict(q=torch.zeros(2, 3, 5, 64, dtype=BF))),
    ('width', dict(q=torch.zeros(2, 4, 5, 96, dtype=BF), k=torch.zeros(2, 2, 7, 96, dtype=BF), v=torch.zeros(2, 2, 7, 96, dtype=BF))), ('k ', dict(v=torch.zeros(2, 2, 8, 64, dtype=BF))),
    ('not positive', dict(scale=0.0)), ('not positive', dict(scale=float('nan'))), ('softcap', dict(softcap=-1.0)), ('softcap', dict(softcap=float('inf'))),
    ('spans', dict(spans=torch.zeros(4, 2, dtype=torch.int32))), ('int32', dict(spans=torch.zeros(5, 2))), ('key_mask', dict(key_mask=torch.ones(2, 6, dtype=torch.bool))),
    ('key_mask', dict(key_mask=torch.ones(2, 7))), ('slopes and positions', dict(slopes=torch.ones(4, 1))), ('slopes and positions', dict(positions=torch.zeros(5, 1, dtype=torch.int32))),
    ('differ in number', dict(slopes=torch.ones(4, 1), positions=torch.zeros(5, 1, dtype=torch.int32))), ('fp32', dict(slopes=torch.ones(2, 1), positions=torch.zeros(5, 1, dtype=torch.int32))),
    ('without positions', dict(key_positions=torch.zeros(7, 1, dtype=torch.int32))), ('1 .. 3', dict(slopes=torch.ones(4, 4), positions=torch.zeros(5, 4, dtype=torch.int32))),
    ('contiguous', dict(q=torch.zeros(2, 4, 64, 5, dtype=BF).transpose(2, 3)))]


@pytest.mark.parametrize('match,change', ATT_REFUSALS)
def test_attention_refusals(match, change):
    refuses(match, ops.attend_spans, **att(**change))


def test_attention_bwd_refusals():
    a = att()
    lse = torch.zeros(2, 4, 5)
    for match, change in [('out', dict(out=a['q'][:, :2])), ('dout', dict(dout=a['q'].float())), ('lse', dict(lse=lse.double())), ('lse', dict(lse=lse[:, :2])),
                          ('contiguous', dict(dout=torch.zeros(2, 4, 64, 5, dtype=BF).transpose(2, 3)))]:
        refuses(match, ops.attend_spans_bwd, **{**a, **dict(out=a['q'], lse=lse, dout=a['q']), **change})
    h = {n: t.half() for n, t in a.items()}
    refuses('bf16, not', ops.attend_spans_bwd, **h, out=h['q'], lse=lse, dout=h['q'])
    for match, change in ATT_REFUSALS[2:]:
        if 'q' not in change:
            refuses(match, ops.attend_spans_bwd, **{**a, **dict(out=a['q'], lse=lse, dout=a['q']), **change})


def test_packed_descriptors_have_the_fields_of_the_c_structs():
    for packer, cls in ((ops._ROTARY, _lib.Rotary), (ops._SPAN, _lib.SpanAttn)):
        assert packer.size == _lib.C.sizeof(cls)
        d = cls.from_buffer_copy(packer.pack(*range(1, len(packer.unpack(bytes(packer.size))) + 1)))

        def flat(x):
            for f, t in x._fields_:
                v = getattr(x, f)
                if isinstance(v, _lib.C.Structure):
                    yield from flat(v)
                elif isinstance(v, _lib.C.Array):
                    yield from v
                else:
                    yield v
        assert list(flat(d)) == list(range(1, len(list(flat(d))) + 1))


def span_desc(**change):
    """a descriptor whose pointers are never followed: the C checks come first"""
    d = _lib.SpanAttn()
    for f in ('q', 'k', 'v', 'out', 'lse', 'dout', 'dq', 'dk', 'dv'):
        setattr(d, f, 4096)
    for f in ('q', 'k', 'v', 'out', 'dout', 'dq', 'dk', 'dv'):
        setattr(d, f + '_stride', (64 * 64, 64 * 16, 64))
    d.batch, d.heads_q, d.heads_k, d.nq, d.nk, d.dim, d.scale = 2, 4, 2, 16, 16, 64, 1.0
    for f, v in change.items():
        setattr(d, f, v)
    return d


@pytest.mark.parametrize('change,code', [
    (dict(q=None), -1), (dict(k=4104), -3), (dict(v_stride=(64 * 64, 64 * 16, 60)), -3), (dict(k_stride=(64 * 64, 64 * 16, 32)), -1), (dict(k_stride=(0, 0, 1 << 23)), -1),
    (dict(q_stride=(-64, 64, 64)), -3), (dict(dim=48), -7), (dict(dtype=2), -2), (dict(heads_k=3), -1), (dict(batch=-1), -1), (dict(scale=0.0), -1), (dict(scale=float('nan')), -1),
    (dict(softcap=-1.0), -1), (dict(axes=4), -1), (dict(slopes=4096, axes=0), -1), (dict(slopes=4096, axes=1), -1), (dict(spans=4100), -3), (dict(spans=4096, spans_sb=3), -3),
    (dict(nq=1 << 29), -1), (dict(batch=1 << 19, nq=1 << 20), -1), (dict(out=None), -1)])
def test_c_entries_refuse_before_they_launch(change, code):
    lib = _lib.lib()
    d = span_desc(**change)
    ref = _lib.C.byref(d)
    assert lib.mm_span_attention(None, ref, None, 0) == code and lib.mm_last_error()
    assert lib.mm_span_attention_workspace_bytes(ref) == 0
    assert lib.mm_span_attention_bwd(None, ref, None, 0) == code and lib.mm_span_attention_bwd_workspace_bytes(ref) == 0


def test_c_entries_of_nothing_and_null():
    lib = _lib.lib()
    assert lib.mm_span_attention(None, None, None, 0) == -1 and lib.mm_rotary_axes(None, None) == -1 and lib.mm_rotary_axes_bwd(None, None, None, None, 0) == -1
    assert lib.mm_span_attention(None, _lib.C.byref(span_desc(batch=0)), None, 0) == 0
    assert lib.mm_span_attention_bwd(None, _lib.C.byref(span_desc(dtype=1)), None, 0) == -2          # fp16: the forward only
    # a single position over a long cache: partial results need a workspace
    long = span_desc(nq=1, nk=100000)
    assert lib.mm_span_attention_workspace_bytes(_lib.C.byref(long)) > 0 and lib.mm_span_attention(None, _lib.C.byref(long), None, 0) == -6
    assert lib.mm_attention_spans(None, None, 0, None, 0, None, 0, 0, 3, 5, 5, 0, None) == 0
    assert lib.mm_attention_spans(None, None, 0, None, 0, None, 0, 1, 3, 5, 5, 0, None) == -1
    r = _lib.Rotary()
    r.axes, r.dim, r.batch, r.n = 1, 64, 1, 1
    r.q.heads = 1
    for f, v, code in [('dim', 63, -1), ('axes', 5, -1), ('dtype', 9, -2), ('batch', -1, -1), ('positions', None, -1)]:
        s = _lib.Rotary.from_buffer_copy(r)
        setattr(s, f, v)
        assert lib.mm_rotary_axes(None, _lib.C.byref(s)) == code
    s = _lib.Rotary.from_buffer_copy(r)      # 160 wide, rows that do not allow 16-byte accesses
    s.dim, s.positions = 160, 4096
    s.q.x, s.q.out, s.q.x_stride = 4098, 4096, (0, 0, 160)
    assert lib.mm_rotary_axes(None, _lib.C.byref(s)) == -7


# ------------------------------------------------------------------------------------------------ the plain forms themselves
@pytest.mark.parametrize('cap,axes', [(0.0, 0), (3.0, 0), (0.0, 2), (2.0, 3)])
def test_plain_attention_gradients_are_autograds(cap, axes):
    g = torch.Generator().manual_seed(1)
    b, hq, hk, n, j, d = 2, 4, 2, 9, 11, 32
    q, k, v = (torch.randn(b, h, m, d, generator=g).to(BF) for h, m in ((hq, n), (hk, j), (hk, j)))
    lo = torch.randint(0, 6, (b, n), generator=g)
    spans = torch.stack([lo, lo + torch.randint(0, 7, (b, n), generator=g)], 2).to(torch.int32)
    seen = R.visible(n, j, spans, torch.rand(b, j, generator=g) < 0.8, b)
    slopes = torch.rand(hq, axes, generator=g) if axes else None
    pq, pk = (torch.randint(0, 9, (m, axes), generator=g).to(torch.int32) if axes else None for m in (n, j))
    f = R.attention(q, k, v, seen, 0.3, cap, slopes, pq, pk)
    leaves = [t.double().requires_grad_() for t in (q, k, v)] + ([slopes.double().requires_grad_()] if axes else [])
    s = leaves[0] @ leaves[1].repeat_interleave(2, 1).transpose(2, 3) * 0.3
    if cap:
        s = cap * torch.tanh(s / cap)
    if axes:
        s = s - torch.einsum('ha,nja->hnj', leaves[3], (pq[:, None] - pk[None]).abs().double())
    p = torch.softmax(s.masked_fill(~seen[:, None], -1e300), -1) * seen[:, None]
    out = p @ leaves[2].repeat_interleave(2, 1)
    assert torch.allclose(out, f['out'], rtol=0, atol=1e-12)
    w = torch.randn(b, hq, n, d, generator=g).double()
    grads = torch.autograd.grad((out * w).sum(), leaves)
    got = R.attention(q, k, v, seen, 0.3, cap, slopes, pq, pk, dout=w, out=f['out'], lse=f['lse'])
    for name, want in zip(('dq', 'dk', 'dv', 'dslopes'), grads):
        assert torch.allclose(got[name], want, rtol=0, atol=1e-9), name


@pytest.mark.parametrize('match,change', [('not positive', dict(scale=1e-30)), ('not positive', dict(scale=1e30)), ('softcap', dict(softcap=1e-9)), ('softcap', dict(softcap=1e6))])
def test_attention_refuses_numbers_that_leave_32_bits(match, change):
    refuses(match, ops.attend_spans, **att(**change))
    lib = _lib.lib()
    for f, v in change.items():
        assert lib.mm_span_attention(None, _lib.C.byref(span_desc(**{f: v})), None, 0) == -1


def test_spans_refuse_tables_of_no_rows_beside_tables_of_some():
    cu, none = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(0, 4, dtype=torch.int32)
    refuses('batch sizes', ops.attention_spans, none, 5, cu, 5)
    refuses('batch sizes', ops.attention_spans, cu, 5, none, 5)
    refuses('2\\^30', ops.attention_spans, cu, 2 ** 31 - 1)
    assert _lib.lib().mm_attention_spans(None, 4096, 0, 4096, 0, None, 0, 1, 3, 2 ** 31 - 1, 5, 0, 4096) == -1


def test_c_sizes_of_a_long_cache_are_taken_forward_alone():
    """64 sequences of one new position over 2^22 keys: the blocks of 32 keys count only where a launch has threads for each (the backward)"""
    lib = _lib.lib()
    d = span_desc(batch=64, heads_q=32, heads_k=4, nq=1, nk=1 << 22)      # (256 workgroups: the keys are split in two)
    assert lib.mm_span_attention_workspace_bytes(_lib.C.byref(d)) == 2 * 256 * 32 * (64 + 2) * 4
    assert lib.mm_span_attention_bwd_workspace_bytes(_lib.C.byref(d)) == 0
    assert lib.mm_span_attention_bwd(None, _lib.C.byref(d), None, 0) == -1
