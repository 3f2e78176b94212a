// Attention of packed rows, backward, from q, k, v, out, lse and dout.  With p = exp(s - lse) and delta_i = sum_d dout_id out_id:
//     dv = p^T dout,   ds = p (dout v^T - delta),   dslope_a = - sum ds |distance_a|,   dq = scale (ds cap') k,   dk = scale (ds cap')^T q
// Three launches and no atomics, so every sum has one order:
//   span_bwd_pre : delta per row (one read of out and dout) and, per 32 queries, the keys they see (lowest, highest bound; and whether all see the same whole range)
//   span_bwd_dq  : 128 queries of a head (4 waves x 32), key tiles of 64: the forward's S^T form -- lse and delta belong to the lane; ds goes into dQ^T = K^T dS^T
//   span_bwd_dkv : 128 keys of a key head (4 waves x 32), query tiles of 64 of every head that shares it: S = Q K^T puts a KEY into the lane's column, so dV^T = dO^T P
//                  and dK^T = Q^T dS take P and dS from the accumulators as they are; only the query tiles whose keys meet this tile are visited
// Recomputing S and dP in both kernels makes 7 products where 5 would do with atomic sums of dQ.  P and dS are rounded to bf16 as operands of the products; everything
// else (scores, exp, ds, delta, slopes' gradients) is fp32.
#include <string.h>

#include "span_attn.h"

void span_args(const mm_span_attn* a, SpanArgs& p);
long span_order_tiles(const mm_span_attn* a);
int span_order_run(hipStream_t s, const mm_span_attn* a, int32_t* order);

namespace {

constexpr int BQ = 128, BK = 128, BT = 64;

__device__ __forceinline__ int2 row_span(const SpanArgs& p, int b, int h, int i) {      // empty where the row sees nothing or its lse says so
    int lo = 0, hi = p.nk;
    if (p.spans) {
        const int2 sp = reinterpret_cast<const int2*>(p.spans + b * p.spans_sb)[i];
        lo = max(sp.x, 0); hi = min(sp.y, p.nk);
    }
    if (lo >= hi || p.lse[((long)b * p.Hq + h) * p.nq + i] == -INFINITY) lo = hi = 0;
    return make_int2(lo, hi);
}

// one wave per 64 / (D / 8) rows: D / 8 lanes a row, 16 bytes of out and of dout each
template <int D>
__global__ __launch_bounds__(256) void span_bwd_pre(const SpanArgs p) {
    constexpr int TPR = D / 8, RPB = 256 / TPR;
    const int c = threadIdx.x % TPR;
    const long row = (long)blockIdx.x * RPB + threadIdx.x / TPR, rows = (long)p.B * p.Hq * p.nq;
    if (row < rows) {
        const int i = (int)(row % p.nq), h = (int)(row / p.nq % p.Hq), b = (int)(row / p.nq / p.Hq);
        const u32x4_t x = *reinterpret_cast<const u32x4_t*>(p.out + b * p.o_s[0] + h * p.o_s[1] + (long)i * p.o_s[2] + c * 8);
        const u32x4_t y = *reinterpret_cast<const u32x4_t*>(p.dout + b * p.do_s[0] + h * p.do_s[1] + (long)i * p.do_s[2] + c * 8);
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) s = __builtin_fmaf(bf16lo(x[e]), bf16lo(y[e]), __builtin_fmaf(bf16hi(x[e]), bf16hi(y[e]), s));
#pragma unroll
        for (int o = 1; o < TPR; o <<= 1) s += __shfl_xor(s, o, 64);
        if (c == 0) p.delta[row] = s;
    }
}

// per 32 queries: .x lowest, .y highest key bound (x >= y: nobody sees anything), .z / .w highest low and lowest high bound (a tile inside them needs no mask).  By the
// spans alone: a row whose lse is -inf although its span is not empty (all of its keys masked) is found per key tile by the mask.
__global__ __launch_bounds__(256) void span_bwd_hulls(const SpanArgs p) {
    const int lane = threadIdx.x & 63;
    const long seg = ((long)blockIdx.x * 256 + threadIdx.x) / 32;
    const long tiles = (long)p.hull_tiles;
    const int b = (int)(seg / tiles), i = (int)(seg % tiles) * 32 + (lane & 31);
    int lo = INT32_MAX, hi = 0, lx = INT32_MAX, hn = 0;      // a row that is not there or sees nothing: no part of the hull, and no tile without a mask
    if (b < p.B && i < p.nq) {
        int a = 0, e = p.nk;
        if (p.spans) {
            const int2 sp = reinterpret_cast<const int2*>(p.spans + b * p.spans_sb)[i];
            a = max(sp.x, 0); e = min(sp.y, p.nk);
        }
        if (a < e) { lo = lx = a; hi = hn = e; }
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        lo = min(lo, __shfl_xor(lo, o, 64)); hi = max(hi, __shfl_xor(hi, o, 64));
        lx = max(lx, __shfl_xor(lx, o, 64)); hn = min(hn, __shfl_xor(hn, o, 64));
    }
    if (b < p.B && (lane & 31) == 0) p.hulls[seg] = make_int4(lo, hi, lx, hn);
}

// gradient of one query row from its own keys alone, by one wave (lane = key, then lane = element)
template <int D, int AX>
__device__ __forceinline__ void query_again(const SpanArgs& p, int b, int h, int i, int k0, int k1, float lse2, float delta, int lane, float (&o)[2]) {
    const uint16_t* q = p.q + b * p.q_s[0] + h * p.q_s[1] + (long)i * p.q_s[2];
    const uint16_t* g = p.dout + b * p.do_s[0] + h * p.do_s[1] + (long)i * p.do_s[2];
    const int hk = h / (p.Hq / p.Hk);
    const uint16_t* kb = p.k + b * p.k_s[0] + hk * p.k_s[1];
    const uint16_t* vb = p.v + b * p.v_s[0] + hk * p.v_s[1];
    o[0] = o[1] = 0.f;
#pragma nounroll
    for (int t0 = k0; t0 < k1; t0 += 64) {
        const int key = t0 + lane;
        float w = 0.f, slope;
        if (key < k1 && (!p.kmask || p.kmask[b * p.km_sb + key])) {
            const float s = pair_score<D, false, AX>(p, q, kb + (long)key * p.k_s[2], b, h, i, key, &slope);
            w = __builtin_amdgcn_exp2f(s - lse2) * (row_dot<D, false>(g, vb + (long)key * p.v_s[2]) - delta) * slope;
        }
#pragma nounroll
        for (int e = 0; e < min(64, k1 - t0); ++e) {
            const float we = __shfl(w, e, 64);
            if (p.kmask && !p.kmask[b * p.km_sb + t0 + e]) continue;
            const uint16_t* k = kb + (long)(t0 + e) * p.k_s[2];
            if (lane < D) o[0] = __builtin_fmaf(we, bf16_to_f32(k[lane]), o[0]);
            if (D > 64) o[1] = __builtin_fmaf(we, bf16_to_f32(k[lane + 64]), o[1]);
        }
    }
}

// gradients of one key row from the queries that see it alone, by one wave (lane = query, then lane = element)
template <int D, int AX>
__device__ __forceinline__ void key_again(const SpanArgs& p, int b, int hk, int h0, int h1, int key, int lane, float (&dk)[2], float (&dv)[2]) {
    const uint16_t* k = p.k + b * p.k_s[0] + hk * p.k_s[1] + (long)key * p.k_s[2];
    const uint16_t* v = p.v + b * p.v_s[0] + hk * p.v_s[1] + (long)key * p.v_s[2];
    dk[0] = dk[1] = dv[0] = dv[1] = 0.f;
#pragma nounroll
    for (int h = h0; h < h1; ++h)
#pragma nounroll
        for (int t0 = 0; t0 < p.nq; t0 += 64) {
            const int i = t0 + lane;
            float w = 0.f, ds = 0.f, slope;
            bool sees = false;
            if (i < p.nq) {
                const int2 sp = row_span(p, b, h, i);
                sees = sp.x <= key && key < sp.y;
            }
            if (sees) {
                const long row = ((long)b * p.Hq + h) * p.nq + i;
                const float s = pair_score<D, false, AX>(p, p.q + b * p.q_s[0] + h * p.q_s[1] + (long)i * p.q_s[2], k, b, h, i, key, &slope);
                w = __builtin_amdgcn_exp2f(s - p.lse[row] * SPAN_LOG2E);
                ds = w * (row_dot<D, false>(p.dout + b * p.do_s[0] + h * p.do_s[1] + (long)i * p.do_s[2], v) - p.delta[row]) * slope;
            }
            unsigned long long todo = __ballot(sees);
#pragma nounroll
            while (todo) {
                const int e = __builtin_ctzll(todo);
                todo &= todo - 1;
                const float we = __shfl(w, e, 64), de = __shfl(ds, e, 64);
                const uint16_t* q = p.q + b * p.q_s[0] + h * p.q_s[1] + (long)(t0 + e) * p.q_s[2];
                const uint16_t* g = p.dout + b * p.do_s[0] + h * p.do_s[1] + (long)(t0 + e) * p.do_s[2];
                if (lane < D) { dk[0] = __builtin_fmaf(de, bf16_to_f32(q[lane]), dk[0]); dv[0] = __builtin_fmaf(we, bf16_to_f32(g[lane]), dv[0]); }
                if (D > 64) { dk[1] = __builtin_fmaf(de, bf16_to_f32(q[lane + 64]), dk[1]); dv[1] = __builtin_fmaf(we, bf16_to_f32(g[lane + 64]), dv[1]); }
            }
        }
}

template <int D, int AX, bool CAP>
__global__ __launch_bounds__(256, 2) void span_bwd_dq(const SpanArgs p) {
    typedef Tile<D, BT> T;
    extern __shared__ __attribute__((aligned(128))) unsigned char smem[];
    constexpr int POS = AX * BT * 4, STAGE = 2 * T::BYTES + POS;
    int* red = reinterpret_cast<int*>(smem + 2 * STAGE);
    const int t = threadIdx.x, lane = t & 63, half = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(t >> 6);
    const int tiles = (p.nq + BQ - 1) / BQ;
    int rt, h;
    if (!span_item(p.order, p.Hq, p.B * tiles, rt, h)) return;
    const int tile = rt % tiles, b = rt / tiles, hk = h / (p.Hq / p.Hk);
    const int i = tile * BQ + w * 32 + (lane & 31);
    const bool ok = i < p.nq;
    int lo = 0, hi = 0;
    float lse2 = 0.f, delta = 0.f;
    if (ok) {
        const int2 sp = row_span(p, b, h, i);
        lo = sp.x; hi = sp.y;
        const long row = ((long)b * p.Hq + h) * p.nq + i;
        lse2 = hi > lo ? p.lse[row] * SPAN_LOG2E : 0.f;
        delta = hi > lo ? p.delta[row] : 0.f;      // (a row that sees nothing may hold anything)
    }
    int h0 = hi > lo ? lo : INT32_MAX, h1 = hi;
    for (int o = 16; o > 0; o >>= 1) { h0 = min(h0, __shfl_xor(h0, o, 64)); h1 = max(h1, __shfl_xor(h1, o, 64)); }
    if (lane == 0) { red[w] = h0; red[4 + w] = h1; }
    u32x4_t qf[D / 16], gf[D / 16];
    {
        const uint16_t* qp = p.q + b * p.q_s[0] + h * p.q_s[1] + (long)(ok ? i : 0) * p.q_s[2] + half * 8;
        const uint16_t* gp = p.dout + b * p.do_s[0] + h * p.do_s[1] + (long)(ok ? i : 0) * p.do_s[2] + half * 8;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) { qf[c] = *reinterpret_cast<const u32x4_t*>(qp + c * 16); gf[c] = *reinterpret_cast<const u32x4_t*>(gp + c * 16); }
    }
    float sl[AX ? AX : 1], ds_sl[AX ? AX : 1]; int pq[AX ? AX : 1];
#pragma unroll
    for (int a = 0; a < AX; ++a) {
        sl[a] = p.slopes[h * AX + a] * SPAN_LOG2E;
        pq[a] = ok ? p.pos_q[b * p.pq_sb + (long)i * AX + a] : 0;
        ds_sl[a] = 0.f;
    }
    __syncthreads();
    const int k0 = __builtin_amdgcn_readfirstlane(min(min(red[0], red[1]), min(red[2], red[3])));
    const int k1 = __builtin_amdgcn_readfirstlane(max(max(red[4], red[5]), max(red[6], red[7])));
    const int nt = k1 > k0 ? (k1 - k0 + BT - 1) / BT : 0;
    const uint16_t* kp = p.k + b * p.k_s[0] + hk * p.k_s[1];
    const uint16_t* vp = p.v + b * p.v_s[0] + hk * p.v_s[1];
    const uint8_t* km = p.kmask ? p.kmask + b * p.km_sb : nullptr;
    const int* pkp = AX ? p.pos_k + b * p.pk_sb : nullptr;
    const float c1 = CAP ? 2.f * p.scale * SPAN_LOG2E / p.cap : p.scale * SPAN_LOG2E, c2 = p.cap * SPAN_LOG2E;

#define SPAN_ISSUE(it_)                                                                                                \
    {                                                                                                                  \
        const int t0_ = k0 + (it_) * BT;                                                                               \
        unsigned char* st_ = smem + ((it_) & 1) * STAGE;                                                               \
        T::template fill<4>(st_, kp + (long)t0_ * p.k_s[2], min(BT, k1 - t0_), (int)p.k_s[2], w, lane);                \
        T::template fill<4>(st_ + T::BYTES, vp + (long)t0_ * p.v_s[2], min(BT, k1 - t0_), (int)p.v_s[2], w, lane);     \
    }
#define SPAN_POS_LOAD(it_) \
    if constexpr (AX > 0) { if (t < BT * AX) { const int key_ = k0 + (it_) * BT + t / AX; posv = key_ < k1 ? pkp[(long)key_ * AX + t % AX] : 0; } }
#define SPAN_POS_STORE(it_) \
    if constexpr (AX > 0) { if (t < BT * AX) reinterpret_cast<int*>(smem + ((it_) & 1) * STAGE + 2 * T::BYTES)[(t % AX) * BT + t / AX] = posv; }
    f32x16_t dq[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) dq[c][r] = 0.f;
    int posv = 0;
    if (nt > 0) { SPAN_ISSUE(0); SPAN_POS_LOAD(0); SPAN_POS_STORE(0); }
    for (int it = 0; it < nt; ++it) {
        const int t0 = k0 + it * BT;
        unsigned char* Ks = smem + (it & 1) * STAGE;
        unsigned char* Vs = Ks + T::BYTES;
        const int* pks = reinterpret_cast<const int*>(Ks + 2 * T::BYTES);
        unsigned long long keep = ~0ull;
        if (km) keep = __ballot(t0 + lane < k1 && km[t0 + lane]);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (it + 1 < nt) { SPAN_ISSUE(it + 1); SPAN_POS_LOAD(it + 1); }
        if (keep != ~0ull) {
            T::clear_rows(Ks, keep, t, 256);
            __syncthreads();
        }
        if (__any(lo < t0 + BT && hi > t0)) {
            const bool masked = keep != ~0ull || !__all(lo <= t0 && hi >= t0 + BT);
            const unsigned long long bits = masked ? (bit_range(lo - t0, hi - t0) & keep) >> (4 * half) : ~0ull;
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                f32x16_t s, g;
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = g[r] = 0.f;
#pragma unroll
                for (int c = 0; c < D / 16; ++c) {
                    s = mfma32<false>(T::rows(Ks, c, n, lane), qf[c], s);
                    g = mfma32<false>(T::rows(Vs, c, n, lane), gf[c], g);
                }
                const uint32_t wb = (uint32_t)(bits >> (32 * n));
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4) {
                    int4 kq[AX ? AX : 1];
#pragma unroll
                    for (int a = 0; a < AX; ++a) kq[a] = *reinterpret_cast<const int4*>(pks + a * BT + n * 32 + g4 * 8 + half * 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = g4 * 4 + e;
                        float x = s[r], slope = 1.f, far[AX ? AX : 1];
                        if constexpr (CAP) { const float th = span_tanh(x, c1); slope = __builtin_fmaf(-th, th, 1.f); x = th * c2; }
                        else x *= c1;
#pragma unroll
                        for (int a = 0; a < AX; ++a) {
                            const int kv = e == 0 ? kq[a].x : (e == 1 ? kq[a].y : (e == 2 ? kq[a].z : kq[a].w));
                            far[a] = fabsf((float)(pq[a] - kv));
                            x = __builtin_fmaf(-sl[a], far[a], x);
                        }
                        float d = __builtin_amdgcn_exp2f(x - lse2) * (g[r] - delta);
                        if (!(wb & (1u << (8 * g4 + e)))) d = 0.f;
#pragma unroll
                        for (int a = 0; a < AX; ++a) ds_sl[a] = __builtin_fmaf(d, far[a], ds_sl[a]);
                        s[r] = CAP ? d * slope : d;
                    }
                    asm volatile("" ::: "memory");      // (four scores at a time: all sixteen at once cost 60 registers more, and the second workgroup of a CU)
                }
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const u32x4_t f = pack_slots<false>(s, x);      // dS rounded to bf16: an operand of the product with K
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) dq[c] = mfma32<false>(T::cols(Ks, 2 * n + x, c, lane), f, dq[c]);
                }
            }
        }
        if (it + 1 < nt) SPAN_POS_STORE(it + 1);
    }
#undef SPAN_ISSUE
#undef SPAN_POS_LOAD
#undef SPAN_POS_STORE
    float bad = 0.f;
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) bad = __builtin_fmaf(dq[c][r], 0.f, bad);
    bad = both_halves_sum(bad);
    const bool redo = ok && bad != 0.f && (lse2 + delta) * 0.f == 0.f;      // (a row whose own numbers are not finite is what it is)
    if (ok && !redo) {
        uint16_t* op = p.dq + b * p.dq_s[0] + h * p.dq_s[1] + (long)i * p.dq_s[2] + half * 4;
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<uint2*>(op + c * 32 + g * 8) = make_uint2(pack_bf16x2(dq[c][4 * g] * p.scale, dq[c][4 * g + 1] * p.scale), pack_bf16x2(dq[c][4 * g + 2] * p.scale, dq[c][4 * g + 3] * p.scale));
    }
    unsigned long long todo = __ballot(redo) & 0xFFFFFFFFull;
#pragma nounroll
    while (todo) {
        const int r = __builtin_ctzll(todo);
        todo &= todo - 1;
        const int ri = tile * BQ + w * 32 + r;
        float ro[2];
        query_again<D, AX>(p, b, h, ri, __shfl(lo, r, 64), __shfl(hi, r, 64), __shfl(lse2, r, 64), __shfl(delta, r, 64), lane, ro);
        uint16_t* op = p.dq + b * p.dq_s[0] + h * p.dq_s[1] + (long)ri * p.dq_s[2];
        if (lane < D) op[lane] = f32_to_bf16(ro[0] * p.scale);
        if (D > 64) op[lane + 64] = f32_to_bf16(ro[1] * p.scale);
    }
    if constexpr (AX > 0) {
        if (p.dsl_part) {      // the workgroup's part of the slopes' gradients: lanes in a fixed tree, then the waves in order
            float* fr = reinterpret_cast<float*>(red);
            __syncthreads();
#pragma unroll
            for (int a = 0; a < AX; ++a) {
                const float v = wave_sum(ds_sl[a]);
                if (lane == 0) fr[w * 4 + a] = -v;
            }
            __syncthreads();
            if (t < AX) p.dsl_part[((long)b * tiles + tile) * p.Hq * AX + h * AX + t] = ((fr[t] + fr[4 + t]) + fr[8 + t]) + fr[12 + t];
        }
    }
}

template <int D, int AX, bool CAP>
__global__ __launch_bounds__(256, D == 128 ? 1 : 2) void span_bwd_dkv(const SpanArgs p) {
    typedef Tile<D, BT> T;
    extern __shared__ __attribute__((aligned(128))) unsigned char smem[];
    constexpr int ROWB = (4 + AX) * BT * 4, STAGE = 2 * T::BYTES + ROWB;      // Q, dO, then per row: lse (log2 units), delta, lo, hi, positions
    int* list = reinterpret_cast<int*>(smem + 2 * STAGE);                     // [256] query tiles
    int4* hull = reinterpret_cast<int4*>(list + 256);                         // [256][2] bounds of their two 32-row halves
    int* cnt = reinterpret_cast<int*>(hull + 512);                            // [4]
    const int t = threadIdx.x, lane = t & 63, half = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(t >> 6);
    const int tiles = (p.nk + BK - 1) / BK, total = p.B * p.Hk * p.splits * tiles, per = (total + 7) / 8;
    const int item = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || item >= total) return;
    const int tile = item % tiles, part = (item / tiles) % p.splits, hk = (item / tiles / p.splits) % p.Hk, b = item / tiles / p.splits / p.Hk;
    const int heads = p.Hq / p.Hk / p.splits, h0 = (hk * p.splits + part) * heads, h1 = h0 + heads;      // the query heads of this workgroup
    const int t0 = tile * BK, t1 = min(t0 + BK, p.nk), w0 = t0 + w * 32;      // the wave's keys: w0 .. w0 + 31
    const int key = w0 + (lane & 31);
    const bool live = key < p.nk && (!p.kmask || p.kmask[b * p.km_sb + key]);      // a key that is not there or masked: zeros, no weight
    const bool all_live = __all(live);
    u32x4_t kf[D / 16], vf[D / 16];
    {
        const uint16_t* kp = p.k + b * p.k_s[0] + hk * p.k_s[1] + (long)(live ? key : 0) * p.k_s[2] + half * 8;
        const uint16_t* vp = p.v + b * p.v_s[0] + hk * p.v_s[1] + (long)(live ? key : 0) * p.v_s[2] + half * 8;
        const u32x4_t z = {0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
            const u32x4_t x = *reinterpret_cast<const u32x4_t*>(kp + c * 16), y = *reinterpret_cast<const u32x4_t*>(vp + c * 16);
            kf[c] = live ? x : z; vf[c] = live ? y : z;
        }
    }
    int pk[AX ? AX : 1];
#pragma unroll
    for (int a = 0; a < AX; ++a) pk[a] = key < p.nk ? p.pos_k[b * p.pk_sb + (long)key * AX + a] : 0;
    const float c1 = CAP ? 2.f * p.scale * SPAN_LOG2E / p.cap : p.scale * SPAN_LOG2E, c2 = p.cap * SPAN_LOG2E;
    f32x16_t dk[D / 32], dv[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) dk[c][r] = dv[c][r] = 0.f;

    const int qtiles = (p.nq + BT - 1) / BT;
    float lsev = 0.f, delv = 0.f;
    int2 spv = make_int2(0, 0);
    int posv[AX ? AX : 1];
    // the tile being fetched: entry f_at of the list, head f_h (its rows: lane = row of the 64, every wave the same; wave 0 writes them to LDS)
    int f_at = 0, f_h = h0, f_stage = 0;
    const uint16_t *f_q = p.q + b * p.q_s[0] + f_h * p.q_s[1], *f_g = p.dout + b * p.do_s[0] + f_h * p.do_s[1];
#define SPAN_ISSUE()                                                                                                              \
    {                                                                                                                             \
        unsigned char* st_ = smem + f_stage * STAGE;                                                                              \
        const int q0_ = __builtin_amdgcn_readfirstlane(list[f_at]) * BT, ok_ = min(BT, p.nq - q0_);                               \
        T::template fill<4>(st_, f_q + (long)q0_ * p.q_s[2], ok_, (int)p.q_s[2], w, lane);                                        \
        T::template fill<4>(st_ + T::BYTES, f_g + (long)q0_ * p.do_s[2], ok_, (int)p.do_s[2], w, lane);                           \
        const int i_ = q0_ + lane;                                                                                                \
        spv = make_int2(0, 0); lsev = 0.f; delv = 0.f;                                                                            \
        if (i_ < p.nq) {                                                                                                          \
            const long row_ = ((long)b * p.Hq + f_h) * p.nq + i_;                                                                 \
            spv = row_span(p, b, f_h, i_);                                                                                        \
            lsev = p.lse[row_] * SPAN_LOG2E; delv = p.delta[row_];                                                                \
            _Pragma("unroll") for (int a = 0; a < AX; ++a) posv[a] = p.pos_q[b * p.pq_sb + (long)i_ * AX + a];                    \
        }                                                                                                                         \
    }
#define SPAN_ROW_STORE()                                                                                     \
    if (w == 0) {                                                                                            \
        float* rw_ = reinterpret_cast<float*>(smem + f_stage * STAGE + 2 * T::BYTES);                        \
        rw_[lane] = lsev; rw_[BT + lane] = delv;                                                             \
        reinterpret_cast<int*>(rw_)[2 * BT + lane] = spv.x; reinterpret_cast<int*>(rw_)[3 * BT + lane] = spv.y; \
        _Pragma("unroll") for (int a = 0; a < AX; ++a) reinterpret_cast<int*>(rw_)[(4 + a) * BT + lane] = posv[a]; \
    }
    for (int base = 0; base < qtiles; base += 256) {
        // ---- the query tiles of this stretch that see keys of this tile, in order
        __syncthreads();
        int n_list;
        {
            const int qt = base + t;
            int4 a = make_int4(INT32_MAX, 0, INT32_MAX, 0), e = a;
            if (qt < qtiles) {
                const int4* hp = p.hulls + (long)b * p.hull_tiles + 2 * qt;
                a = hp[0];
                if (2 * qt + 1 < p.hull_tiles) e = hp[1];
            }
            const bool in = (a.x < t1 && a.y > t0) || (e.x < t1 && e.y > t0);
            const unsigned long long m = __ballot(in);
            if (lane == 0) cnt[w] = __popcll(m);
            __syncthreads();
            int to = __popcll(m & ((1ull << lane) - 1ull));
            for (int x = 0; x < w; ++x) to += cnt[x];
            n_list = __builtin_amdgcn_readfirstlane(cnt[0] + cnt[1] + cnt[2] + cnt[3]);
            if (in) { list[to] = qt; hull[2 * to] = a; hull[2 * to + 1] = e; }
            __syncthreads();
        }
        if (n_list == 0) continue;
        f_at = 0; f_h = h0; f_stage = 0;
        f_q = p.q + b * p.q_s[0] + f_h * p.q_s[1]; f_g = p.dout + b * p.do_s[0] + f_h * p.do_s[1];
        SPAN_ISSUE();
        SPAN_ROW_STORE();
        for (bool more = true; more;) {
            const int at = f_at, stage = f_stage, h = f_h;
            unsigned char* Qs = smem + stage * STAGE;
            unsigned char* Gs = Qs + T::BYTES;
            const float* rw = reinterpret_cast<const float*>(Gs + T::BYTES);
            const int* ri = reinterpret_cast<const int*>(rw);
            const unsigned long long keep = __ballot(spv.x < t1 && spv.y > t0);      // rows that see some key of the tile
            float sl[AX ? AX : 1];
#pragma unroll
            for (int a = 0; a < AX; ++a) sl[a] = p.slopes[h * AX + a] * SPAN_LOG2E;
            if (++f_at == n_list) { f_at = 0; ++f_h; f_q += p.q_s[1]; f_g += p.do_s[1]; }
            more = f_h < h1;
            f_stage ^= 1;
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (more) SPAN_ISSUE();
            if (keep != ~0ull) {      // the others' values take no part, whatever they hold (rows behind the last document)
                T::clear_rows(Qs, keep, t, 256);
                T::clear_rows(Gs, keep, t, 256);
                __syncthreads();
            }
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const int4 hl = hull[2 * at + n];
                if (!(hl.x < min(w0 + 32, t1) && hl.y > w0)) continue;
                const bool masked = !all_live || !(hl.z <= w0 && hl.w >= w0 + 32) || (uint32_t)(keep >> (32 * n)) != 0xFFFFFFFFu;
                f32x16_t s, g;
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = g[r] = 0.f;
#pragma unroll
                for (int c = 0; c < D / 16; ++c) {
                    s = mfma32<false>(T::rows(Qs, c, n, lane), kf[c], s);
                    g = mfma32<false>(T::rows(Gs, c, n, lane), vf[c], g);
                }
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4) {
                    const int o4 = n * 32 + g4 * 8 + half * 4;
                    const float4 ls = *reinterpret_cast<const float4*>(rw + o4), de = *reinterpret_cast<const float4*>(rw + BT + o4);
                    int4 lo4 = make_int4(0, 0, 0, 0), hi4 = lo4;
                    if (masked) { lo4 = *reinterpret_cast<const int4*>(ri + 2 * BT + o4); hi4 = *reinterpret_cast<const int4*>(ri + 3 * BT + o4); }
                    int4 qq[AX ? AX : 1];
#pragma unroll
                    for (int a = 0; a < AX; ++a) qq[a] = *reinterpret_cast<const int4*>(ri + (4 + a) * BT + o4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = g4 * 4 + e;
#define SPAN_E4(v_) (e == 0 ? v_.x : (e == 1 ? v_.y : (e == 2 ? v_.z : v_.w)))
                        float x = s[r], slope = 1.f;
                        if constexpr (CAP) { const float th = span_tanh(x, c1); slope = __builtin_fmaf(-th, th, 1.f); x = th * c2; }
                        else x *= c1;
#pragma unroll
                        for (int a = 0; a < AX; ++a) x = __builtin_fmaf(-sl[a], fabsf((float)(SPAN_E4(qq[a]) - pk[a])), x);
                        float pr = __builtin_amdgcn_exp2f(x - SPAN_E4(ls)), d = pr * (g[r] - SPAN_E4(de));
                        if (masked && !(live && SPAN_E4(lo4) <= key && key < SPAN_E4(hi4))) { pr = 0.f; d = 0.f; }
#undef SPAN_E4
                        s[r] = pr;
                        g[r] = CAP ? d * slope : d;
                    }
                    asm volatile("" ::: "memory");
                }
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const u32x4_t pf = pack_slots<false>(s, x), df = pack_slots<false>(g, x);      // P and dS rounded to bf16: operands
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) {
                        dv[c] = mfma32<false>(T::cols(Gs, 2 * n + x, c, lane), pf, dv[c]);
                        dk[c] = mfma32<false>(T::cols(Qs, 2 * n + x, c, lane), df, dk[c]);
                    }
                }
            }
            if (more) SPAN_ROW_STORE();
        }
    }
#undef SPAN_ISSUE
#undef SPAN_ROW_STORE
    float bad = 0.f;
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) bad = __builtin_fmaf(dk[c][r], 0.f, __builtin_fmaf(dv[c][r], 0.f, bad));
    bad = both_halves_sum(bad);
    const bool redo = live && bad != 0.f;
    const long prow = ((long)b * p.Hk + hk) * p.nk, pall = (long)p.B * p.Hk * p.nk;      // partial sums: [splits][dk, dv][rows][D]
    if (p.splits > 1) {
        if (key < p.nk && !redo) {
            float* kp = p.part_o + ((long)part * 2 * pall + prow + key) * D + half * 4;
            float* vp = kp + pall * D;
#pragma unroll
            for (int c = 0; c < D / 32; ++c)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
                    *reinterpret_cast<float4*>(kp + c * 32 + g * 8) = live ? make_float4(dk[c][4 * g], dk[c][4 * g + 1], dk[c][4 * g + 2], dk[c][4 * g + 3]) : z;
                    *reinterpret_cast<float4*>(vp + c * 32 + g * 8) = live ? make_float4(dv[c][4 * g], dv[c][4 * g + 1], dv[c][4 * g + 2], dv[c][4 * g + 3]) : z;
                }
        }
    } else if (key < p.nk && !redo) {
        uint16_t* kp = p.dk + b * p.dk_s[0] + hk * p.dk_s[1] + (long)key * p.dk_s[2] + half * 4;
        uint16_t* vp = p.dv + b * p.dv_s[0] + hk * p.dv_s[1] + (long)key * p.dv_s[2] + half * 4;
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const uint2 x = make_uint2(pack_bf16x2(dk[c][4 * g] * p.scale, dk[c][4 * g + 1] * p.scale), pack_bf16x2(dk[c][4 * g + 2] * p.scale, dk[c][4 * g + 3] * p.scale));
                const uint2 y = make_uint2(pack_bf16x2(dv[c][4 * g], dv[c][4 * g + 1]), pack_bf16x2(dv[c][4 * g + 2], dv[c][4 * g + 3]));
                *reinterpret_cast<uint2*>(kp + c * 32 + g * 8) = live ? x : make_uint2(0, 0);
                *reinterpret_cast<uint2*>(vp + c * 32 + g * 8) = live ? y : make_uint2(0, 0);
            }
    }
    unsigned long long todo = __ballot(redo) & 0xFFFFFFFFull;
#pragma nounroll
    while (todo) {
        const int r = __builtin_ctzll(todo);
        todo &= todo - 1;
        float a[2], c[2];
        key_again<D, AX>(p, b, hk, h0, h1, w0 + r, lane, a, c);
        if (p.splits > 1) {
            float* kp = p.part_o + ((long)part * 2 * pall + prow + w0 + r) * D;
            float* vp = kp + pall * D;
            if (lane < D) { kp[lane] = a[0]; vp[lane] = c[0]; }
            if (D > 64) { kp[lane + 64] = a[1]; vp[lane + 64] = c[1]; }
            continue;
        }
        uint16_t* kp = p.dk + b * p.dk_s[0] + hk * p.dk_s[1] + (long)(w0 + r) * p.dk_s[2];
        uint16_t* vp = p.dv + b * p.dv_s[0] + hk * p.dv_s[1] + (long)(w0 + r) * p.dv_s[2];
        if (lane < D) { kp[lane] = f32_to_bf16(a[0] * p.scale); vp[lane] = f32_to_bf16(c[0]); }
        if (D > 64) { kp[lane + 64] = f32_to_bf16(a[1] * p.scale); vp[lane + 64] = f32_to_bf16(c[1]); }
    }
}

// adds the head splits of a key row in split order; masked keys' parts are zeros.  4 elements a thread
template <int D>
__global__ __launch_bounds__(256) void span_bwd_join(const SpanArgs p) {
    const long pall = (long)p.B * p.Hk * p.nk, x = (long)blockIdx.x * 256 + threadIdx.x;
    const long row = x / (D / 4);
    const int c = (int)(x % (D / 4)) * 4;
    if (row >= 2 * pall) return;
    float4 v = *reinterpret_cast<const float4*>(p.part_o + row * D + c);
    for (int s = 1; s < p.splits; ++s) {
        const float4 y = *reinterpret_cast<const float4*>(p.part_o + (s * 2 * pall + row) * D + c);
        v.x += y.x; v.y += y.y; v.z += y.z; v.w += y.w;
    }
    const bool is_v = row >= pall;
    const long r = is_v ? row - pall : row;
    const int key = (int)(r % p.nk), hk = (int)(r / p.nk % p.Hk), b = (int)(r / p.nk / p.Hk);
    const float f = is_v ? 1.f : p.scale;
    uint16_t* o = is_v ? p.dv + b * p.dv_s[0] + hk * p.dv_s[1] + (long)key * p.dv_s[2] : p.dk + b * p.dk_s[0] + hk * p.dk_s[1] + (long)key * p.dk_s[2];
    *reinterpret_cast<uint2*>(o + c) = make_uint2(pack_bf16x2(v.x * f, v.y * f), pack_bf16x2(v.z * f, v.w * f));
}

// Query heads that share a key head go to workgroups of their own, fp32 partial sums joined in order, as far as that fills the card: the smallest divisor of the group
// that gives 512 workgroups (two per CU), or the whole group.
int head_splits(const mm_span_attn* a) {
    const int group = a->heads_q / a->heads_k;
    const long wgs = (long)a->batch * a->heads_k * ((a->nk + BK - 1) / BK);
    for (int s = 1; s < group; ++s)
        if (group % s == 0 && wgs * s >= 512) return s;
    return group;
}

template <int D, int AX, bool CAP>
int launch_bwd(hipStream_t s, const SpanArgs& a) {
    int rc;
    if (a.nq > 0) {
        const long rows = (long)a.B * a.Hq * a.nq;
        hipLaunchKernelGGL(span_bwd_pre<D>, dim3((unsigned)((rows + 256 / (D / 8) - 1) / (256 / (D / 8)))), dim3(256), 0, s, a);
        if ((rc = mm_check_launch("span_bwd_pre"))) return rc;
        hipLaunchKernelGGL(span_bwd_hulls, dim3((unsigned)(((long)a.B * a.hull_tiles + 7) / 8)), dim3(256), 0, s, a);
        if ((rc = mm_check_launch("span_bwd_hulls"))) return rc;
        constexpr int sm = 2 * (2 * Tile<D, BT>::BYTES + AX * BT * 4) + 64;
        static std::atomic<unsigned long long> lds{0};
        if ((rc = span_allow_lds(reinterpret_cast<const void*>(span_bwd_dq<D, AX, CAP>), sm, lds))) return rc;
        hipLaunchKernelGGL((span_bwd_dq<D, AX, CAP>), dim3((unsigned)(a.B * a.Hq * ((a.nq + BQ - 1) / BQ))), dim3(256), sm, s, a);
        if ((rc = mm_check_launch("span_bwd_dq"))) return rc;
    }
    if (a.nk > 0) {
        constexpr int sm = 2 * (2 * Tile<D, BT>::BYTES + (4 + AX) * BT * 4) + 256 * 4 + 512 * 16 + 16;
        static std::atomic<unsigned long long> lds{0};
        if ((rc = span_allow_lds(reinterpret_cast<const void*>(span_bwd_dkv<D, AX, CAP>), sm, lds))) return rc;
        const long total = (long)a.B * a.Hk * a.splits * ((a.nk + BK - 1) / BK);
        hipLaunchKernelGGL((span_bwd_dkv<D, AX, CAP>), dim3((unsigned)((total + 7) / 8 * 8)), dim3(256), sm, s, a);
        if ((rc = mm_check_launch("span_bwd_dkv"))) return rc;
        if (a.splits > 1) {
            const long work = 2L * a.B * a.Hk * a.nk * (D / 4);
            hipLaunchKernelGGL(span_bwd_join<D>, dim3((unsigned)((work + 255) / 256)), dim3(256), 0, s, a);
            if ((rc = mm_check_launch("span_bwd_join"))) return rc;
        }
    }
    return MM_OK;
}

template <int D, bool CAP>
int launch_bwd_axes(hipStream_t s, const SpanArgs& a) {
    switch (a.axes) {
        case 0: return launch_bwd<D, 0, CAP>(s, a);
        case 1: return launch_bwd<D, 1, CAP>(s, a);
        case 2: return launch_bwd<D, 2, CAP>(s, a);
        default: return launch_bwd<D, 3, CAP>(s, a);
    }
}
template <int D>
int launch_bwd_dim(hipStream_t s, const SpanArgs& a) { return a.cap > 0.f ? launch_bwd_axes<D, true>(s, a) : launch_bwd_axes<D, false>(s, a); }

struct BwdLayout { size_t hulls, delta, order, slopes, parts, bytes; int hull_tiles, splits; long slope_parts; };
BwdLayout bwd_layout(const mm_span_attn* a) {
    BwdLayout r;
    r.hull_tiles = (a->nq + 31) / 32;
    r.slope_parts = a->slopes && a->dslopes ? (long)a->batch * ((a->nq + BQ - 1) / BQ) : 0;
    size_t at = 0;
    r.hulls = at; at += (size_t)a->batch * r.hull_tiles * sizeof(int4);
    r.delta = at; at += ((size_t)a->batch * a->heads_q * a->nq * sizeof(float) + 15) / 16 * 16;
    r.order = at; at += span_order_tiles(a) * sizeof(int32_t);
    r.slopes = at; at += (size_t)r.slope_parts * a->heads_q * a->axes * sizeof(float);
    at = (at + 15) / 16 * 16;
    r.splits = head_splits(a);
    r.parts = at; at += r.splits > 1 ? (size_t)r.splits * 2 * a->batch * a->heads_k * a->nk * a->dim * sizeof(float) : 0;
    r.bytes = at;
    return r;
}

}  // namespace

size_t k_span_attn_bwd_workspace_bytes(const mm_span_attn* a) { return bwd_layout(a).bytes; }

int k_span_attn_bwd(hipStream_t s, const mm_span_attn* a, void* ws) {
    SpanArgs p;
    span_args(a, p);
    const BwdLayout l = bwd_layout(a);
    p.hulls = reinterpret_cast<int4*>((char*)ws + l.hulls);
    p.hull_tiles = l.hull_tiles;
    p.delta = reinterpret_cast<float*>((char*)ws + l.delta);
    p.splits = l.splits;
    if (span_order_tiles(a)) {
        p.order = reinterpret_cast<int32_t*>((char*)ws + l.order);
        if (const int rc = span_order_run(s, a, reinterpret_cast<int32_t*>((char*)ws + l.order))) return rc;
    }
    p.part_o = reinterpret_cast<float*>((char*)ws + l.parts);
    p.dsl_part = l.slope_parts ? reinterpret_cast<float*>((char*)ws + l.slopes) : nullptr;
    const int rc = a->dim == 32 ? launch_bwd_dim<32>(s, p) : (a->dim == 64 ? launch_bwd_dim<64>(s, p) : launch_bwd_dim<128>(s, p));
    if (rc || !a->slopes || !a->dslopes) return rc;
    return k_colsum(s, p.dsl_part, (int)l.slope_parts, (long)a->heads_q * a->axes, a->dslopes);      // (no rows: zeros)
}
