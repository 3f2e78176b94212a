// Attention of packed rows, backward, from q, k, v, out, lse and dout.  With p = exp(s - lse) and delta_i = sum_d dout_id out_id:
//     dv = p^T dout,   ds = p (dout v^T - delta),   dslope_a = - sum ds |distance_a|,   dq = scale (ds cap') k,   dk = scale (ds cap')^T q
// Two launches (three where heads share keys), and every sum in one order:
//   span_bwd_pre  : delta per row (one read of out and dout) and, per 32 queries, the keys they see (lowest, highest bound; and whether all see the same whole range)
//   span_bwd_main : dq_tile,  128 queries of a head, key tiles of 64: the forward's S^T form -- lse and delta belong to the lane; ds goes into dQ^T = K^T dS^T
//                   dkv_tile, 128 keys of a key head, query tiles of 64 of every head that shares it: S = Q K^T puts a KEY into the lane's column, so dV^T = dO^T P and
//                   dK^T = Q^T dS take P and dS from the accumulators as they are; only the query tiles whose keys meet this tile are visited
//   span_bwd_join : the parts of dk and dv of the heads that share a key head, in order
// Recomputing S and dP in both makes 7 products where 5 would do with atomic sums of dQ.  P and dS are rounded to bf16 as operands of the products; everything
// else (scores, exp, ds, delta, slopes' gradients) is fp32.
#include <string.h>

#include "span_attn.h"

void span_args(const mm_span_attn* a, SpanArgs& p);

namespace {

constexpr int BQ = SPAN_TILE, BK = 128, BT = 64;

__device__ __forceinline__ int2 row_span(const SpanArgs& p, int b, int h, int i) {      // empty where the row sees nothing or its lse says so
    int lo = 0, hi = p.nk;
    if (p.spans) {
        const int2 sp = reinterpret_cast<const int2*>(p.spans + b * p.spans_sb)[i];
        lo = max(sp.x, 0); hi = min(sp.y, p.nk);
    }
    if (lo >= hi || p.lse[((long)b * p.Hq + h) * p.nq + i] == -INFINITY) lo = hi = 0;
    return make_int2(lo, hi);
}

// In one launch, all of it read by the next:
//   the first workgroup (where the order is wanted): the order of the query tiles
//   then 8 blocks of 32 queries a workgroup: .x lowest, .y highest key bound (x >= y: nobody sees anything), .z / .w highest low and lowest high bound (a key tile
//   inside them needs no mask).  By the spans alone: a row whose lse is -inf although its span is not empty (all of its keys masked) is found per tile
//   then delta: D / 8 lanes a row, 16 bytes of out and of dout each
template <int D>
__global__ __launch_bounds__(256) void span_bwd_pre(const SpanArgs p) {
    constexpr int TPR = D / 8, RPB = 256 / TPR;
    __shared__ SpanOrderLds m;
    long block = blockIdx.x;
    if (block == 0 && threadIdx.x == 0 && p.done) *p.done = 0;
    if (p.order_out) {
        if (block == 0) { span_order_tiles<256>(m, p.spans, p.spans_sb, p.B, p.nq, p.nk, p.order_out); return; }
        --block;
    }
    const long hull_blocks = ((long)p.B * p.hull_tiles + 7) / 8;
    if (block < hull_blocks) {
        const int lane = threadIdx.x & 63;
        const long seg = (block * 256 + threadIdx.x) / 32, tiles = p.hull_tiles;
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
        return;
    }
    block -= hull_blocks;
    const int c = threadIdx.x % TPR;
    const long row = block * RPB + threadIdx.x / TPR, rows = (long)p.B * p.Hq * p.nq;
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

// the slopes' gradients: the parts of the query tiles (and rows of the batch) in 32 chains, the chains in order; by the workgroup of dq that is done last
__device__ __forceinline__ void sum_slope_parts(const SpanArgs& p, int threads, float* red) {
    const int n = p.Hq * p.axes, t = threadIdx.x, lanes = threads / 32;      // threads / 32 columns at a time, 32 chains each
    const long parts = (long)p.B * ((p.nq + BQ - 1) / BQ);
    for (int c0 = 0; c0 < n; c0 += lanes) {
        const int c = c0 + t % lanes, chain = t / lanes;
        float v = 0.f;
        if (c < n)
            for (long x = chain; x < parts; x += 32) v += __hip_atomic_load(&p.dsl_part[x * n + c], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        red[chain * lanes + t % lanes] = v;
        __syncthreads();
        if (chain == 0 && c < n) {
            v = 0.f;
            for (int x = 0; x < 32; ++x) v += red[x * lanes + t];
            p.dslopes[c] = v;
        }
    }
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
    for (int t0 = k0; t0 < k1 && !all_nan<D>(o, lane); t0 += 64) {
        const int key = t0 + lane;
        const bool sees = key < k1 && (!p.kmask || p.kmask[b * p.km_sb + key]);
        float w = 0.f, slope;
        if (sees) {
            const float s = pair_score<D, false, AX, false>(p, q, kb + (long)key * p.k_s[2], b, h, i, key, &slope);
            w = __builtin_amdgcn_exp2f(s - lse2) * (row_dot<D, false>(g, vb + (long)key * p.v_s[2]) - delta) * slope;
        }
        rows_add<D, false>(o, __ballot(sees), w, kb + (long)t0 * p.k_s[2], p.k_s[2], min(64, k1 - t0), lane);
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
                const float s = pair_score<D, false, AX, false>(p, p.q + b * p.q_s[0] + h * p.q_s[1] + (long)i * p.q_s[2], k, b, h, i, key, &slope);
                w = __builtin_amdgcn_exp2f(s - p.lse[row] * SPAN_LOG2E);
                ds = w * (row_dot<D, false>(p.dout + b * p.do_s[0] + h * p.do_s[1] + (long)i * p.do_s[2], v) - p.delta[row]) * slope;
            }
            const unsigned long long seen = __ballot(sees);
            if (!seen) continue;
            rows_add<D, false>(dk, seen, ds, p.q + b * p.q_s[0] + h * p.q_s[1] + (long)t0 * p.q_s[2], p.q_s[2], min(64, p.nq - t0), lane);
            rows_add<D, false>(dv, seen, w, p.dout + b * p.do_s[0] + h * p.do_s[1] + (long)t0 * p.do_s[2], p.do_s[2], min(64, p.nq - t0), lane);
            if (all_nan<D>(dk, lane) && all_nan<D>(dv, lane)) return;
        }
}

// GROUPS (two for 128 wide heads, where one workgroup fills a CU): waves 0 .. 3 take the even key tiles of the same 128 queries, waves 4 .. 7 the odd ones, joined at the end
template <int D, int AX, int GROUPS>
struct DqLds {
    static constexpr int STAGE = 2 * Tile<D, BT>::BYTES + AX * BT * 4, BYTES = 2 * GROUPS * STAGE + 128;
};
template <int D, int AX, bool CAP, int GROUPS>
__device__ __forceinline__ void dq_tile(const SpanArgs& p, unsigned id, unsigned char* smem) {
    typedef Tile<D, BT> T;
    constexpr int STAGE = DqLds<D, AX, GROUPS>::STAGE;
    int* red = reinterpret_cast<int*>(smem + 2 * GROUPS * STAGE);
    const int t = threadIdx.x & 255, lane = t & 63, half = lane >> 5;      // (t: of the 256 threads of a group)
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), w = wave & 3, grp = GROUPS > 1 ? wave >> 2 : 0;
    const int tiles = (p.nq + BQ - 1) / BQ;
    int rt, h;
    if (!span_item(id, p.order, p.Hq, p.B * tiles, rt, h)) return;
    const int tile = rt % tiles, b = rt / tiles, hk = h / (p.Hq / p.Hk);
    const int i = tile * BQ + w * 32 + (lane & 31);
    const bool ok = i < p.nq;
    int lo = 0, hi = 0;
    float lse2 = 0.f, delta = 0.f;
    if (ok) {      // (all of a row's numbers at once: they come one memory latency later, not three)
        const long row = ((long)b * p.Hq + h) * p.nq + i;
        const float l = p.lse[row], dl = p.delta[row];
        lo = 0; hi = p.nk;
        if (p.spans) {
            const int2 sp = reinterpret_cast<const int2*>(p.spans + b * p.spans_sb)[i];
            lo = max(sp.x, 0); hi = min(sp.y, p.nk);
        }
        if (lo >= hi || l == -INFINITY) lo = hi = 0;
        lse2 = hi > lo ? l * SPAN_LOG2E : 0.f;
        delta = hi > lo ? dl : 0.f;      // (a row that sees nothing may hold anything)
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
    float sl[AX ? AX : 1], ds_sl[AX ? AX : 1], pq[AX ? AX : 1];
#pragma unroll
    for (int a = 0; a < AX; ++a) {
        sl[a] = p.slopes[h * AX + a] * SPAN_LOG2E;
        pq[a] = ok ? (float)p.pos_q[b * p.pq_sb + (long)i * AX + a] : 0.f;
        ds_sl[a] = 0.f;
    }
    __syncthreads();
    const int k0 = __builtin_amdgcn_readfirstlane(min(min(red[0], red[1]), min(red[2], red[3])));
    const int k1 = __builtin_amdgcn_readfirstlane(max(max(red[4], red[5]), max(red[6], red[7])));
    const int nt = k1 > k0 ? (k1 - k0 + GROUPS * BT - 1) / (GROUPS * BT) : 0;
    const uint16_t* kp = p.k + b * p.k_s[0] + hk * p.k_s[1];
    const uint16_t* vp = p.v + b * p.v_s[0] + hk * p.v_s[1];
    const uint8_t* km = p.kmask ? p.kmask + b * p.km_sb : nullptr;
    const int* pkp = AX ? p.pos_k + b * p.pk_sb : nullptr;
    constexpr bool SLOPES = CAP && AX > 0;      // fp32 gradients of slopes behind a cap: span_tanh_block
    const float c1 = SLOPES ? p.scale / p.cap : (CAP ? 2.f * p.scale * SPAN_LOG2E / p.cap : p.scale * SPAN_LOG2E), c2 = p.cap * SPAN_LOG2E;

#define SPAN_ISSUE(it_)                                                                                                \
    {                                                                                                                  \
        const int t0_ = k0 + ((it_) * GROUPS + grp) * BT;                                                              \
        unsigned char* st_ = smem + (((it_) & 1) * GROUPS + grp) * STAGE;                                              \
        T::template fill<4>(st_, kp + (long)t0_ * p.k_s[2], min(BT, k1 - t0_), (int)p.k_s[2], w, lane);                \
        T::template fill<4>(st_ + T::BYTES, vp + (long)t0_ * p.v_s[2], min(BT, k1 - t0_), (int)p.v_s[2], w, lane);     \
    }
#define SPAN_POS_LOAD(it_) \
    if constexpr (AX > 0) { if (t < BT * AX) { const int key_ = k0 + ((it_) * GROUPS + grp) * BT + t / AX; posv = key_ < k1 ? pkp[(long)key_ * AX + t % AX] : 0; } }
#define SPAN_POS_STORE(it_) \
    if constexpr (AX > 0) { if (t < BT * AX) reinterpret_cast<float*>(smem + (((it_) & 1) * GROUPS + grp) * STAGE + 2 * T::BYTES)[(t % AX) * BT + t / AX] = (float)posv; }
    f32x16_t dq[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) dq[c][r] = 0.f;
    int posv = 0;
    if (nt > 0) { SPAN_ISSUE(0); SPAN_POS_LOAD(0); SPAN_POS_STORE(0); }
    for (int it = 0; it < nt; ++it) {
        const int t0 = k0 + (it * GROUPS + grp) * BT;
        unsigned char* Ks = smem + ((it & 1) * GROUPS + grp) * STAGE;
        unsigned char* Vs = Ks + T::BYTES;
        unsigned long long keep = ~0ull, all = ~0ull;
        if (km) {
            keep = all = __ballot(t0 + lane < k1 && km[t0 + lane]);
            if constexpr (GROUPS > 1) {      // (the same answer in every wave: there is a barrier behind it)
                const int t1 = k0 + (it * GROUPS + 1 - grp) * BT;
                all &= __ballot(t1 + lane < k1 && km[t1 + lane]);
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (it + 1 < nt) { SPAN_ISSUE(it + 1); SPAN_POS_LOAD(it + 1); }
        if (all != ~0ull) {
            T::clear_rows(Ks, keep, t, 256);
            lds_barrier();
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
                SpanTanh tanh;
                if constexpr (SLOPES) tanh = span_tanh_block(s, c1);
                const uint32_t wb = (uint32_t)(bits >> (32 * n));
                int pos = ((it & 1) * GROUPS + grp) * STAGE + 2 * T::BYTES + (n * 32 + half * 4) * 4;
                f32x4_t kq[AX ? AX : 1], kn[AX ? AX : 1];      // positions of four keys, and of the next four
#pragma unroll
                for (int a = 0; a < AX; ++a) kq[a] = lds_f4(smem + pos + a * BT * 4);
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4) {
                    float d4[4], far[AX ? AX : 1][4], slope[4];
                    if (g4 < 3)
#pragma unroll
                        for (int a = 0; a < AX; ++a) kn[a] = lds_f4(smem + pos + a * BT * 4 + (g4 + 1) * 32);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = g4 * 4 + e;
                        float x;
                        if constexpr (CAP) { const float th = SLOPES ? span_tanh_poly(s[r] * tanh.k, tanh.c) : span_tanh(s[r], c1); slope[e] = __builtin_fmaf(-th, th, 1.f); x = __builtin_fmaf(th, c2, -lse2); }
                        else x = __builtin_fmaf(s[r], c1, -lse2);
#pragma unroll
                        for (int a = 0; a < AX; ++a) {
                            far[a][e] = pq[a] - kq[a][e];
                            x = __builtin_fmaf(-sl[a], fabsf(far[a][e]), x);
                        }
                        d4[e] = __builtin_amdgcn_exp2f(x) * (g[r] - delta);
                    }
                    if (masked) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) d4[e] = __uint_as_float(__float_as_uint(d4[e]) & (uint32_t)((int)(wb << (31 - (8 * g4 + e))) >> 31));
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
#pragma unroll
                        for (int a = 0; a < AX; ++a) ds_sl[a] = __builtin_fmaf(d4[e], fabsf(far[a][e]), ds_sl[a]);
                        s[g4 * 4 + e] = CAP ? d4[e] * slope[e] : d4[e];
                    }
                    // (four scores at a time: all sixteen at once cost 60 registers more)
                    asm volatile("" : "+v"(pos), "+v"(s[g4 * 4]), "+v"(s[g4 * 4 + 1]), "+v"(s[g4 * 4 + 2]), "+v"(s[g4 * 4 + 3]) :: "memory");
#pragma unroll
                    for (int a = 0; a < AX; ++a) { asm volatile("" : "+v"(ds_sl[a])); kq[a] = kn[a]; }
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
    if constexpr (GROUPS > 1) {      // the second group's sums to the first
        float* sum = reinterpret_cast<float*>(smem);
        __syncthreads();
        if (grp == 1) {
#pragma unroll
            for (int c = 0; c < D / 32; ++c)
#pragma unroll
                for (int r = 0; r < 16; ++r) sum[(c * 16 + r) * 256 + t] = dq[c][r];
        }
        __syncthreads();
        if (grp == 0) {
#pragma unroll
            for (int c = 0; c < D / 32; ++c)
#pragma unroll
                for (int r = 0; r < 16; ++r) dq[c][r] += sum[(c * 16 + r) * 256 + t];
        }
    }
    float bad = 0.f;
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) bad = __builtin_fmaf(dq[c][r], 0.f, bad);
    bad = both_halves_sum(bad);
    const bool here = ok && grp == 0, redo = here && bad != 0.f && (lse2 + delta) * 0.f == 0.f;      // (a row whose own numbers are not finite is what it is)
    if (here && !redo) {
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
        if (p.dsl_part) {      // the workgroup's part of the slopes' gradients: lanes in a fixed tree, then the waves in order; the last workgroup adds the parts
            float* fr = reinterpret_cast<float*>(red);
            __syncthreads();
#pragma unroll
            for (int a = 0; a < AX; ++a) {
                const float v = wave_sum(ds_sl[a]);
                if (lane == 0) fr[wave * 4 + a] = -v;
            }
            __syncthreads();
            if (threadIdx.x < AX) {
                float v = ((fr[t] + fr[4 + t]) + fr[8 + t]) + fr[12 + t];
                if constexpr (GROUPS > 1) v += ((fr[16 + t] + fr[20 + t]) + fr[24 + t]) + fr[28 + t];
                __hip_atomic_store(&p.dsl_part[((long)b * tiles + tile) * p.Hq * AX + h * AX + t], v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            // the parts are stored and loaded at the scope of the card (past the XCD's L2), so that the count only has to wait until its workgroup's are there; a release
            // would write back the whole L2, once a workgroup (8150 rows of packed images: 89 us, 78 so)
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (threadIdx.x == 0) red[0] = __hip_atomic_fetch_add(p.done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u == (unsigned)(p.B * p.Hq * tiles);
            __syncthreads();
            if (red[0]) {
                sum_slope_parts(p, GROUPS * 256, reinterpret_cast<float*>(smem));
            }
        }
    }
}

// The order of LDS reads and matrix instructions of a product in the instruction stream: the operands of two steps ahead.  Left alone the compiler often reads one
// operand, waits for it and multiplies, eight times over.  (0x100: LDS read, 0x008: matrix instruction)
template <int PER, int STEPS>
__device__ __forceinline__ void paced() {
    __builtin_amdgcn_sched_group_barrier(0x100, 2 * PER, 0);
#pragma unroll
    for (int c = 0; c < STEPS; ++c) {
        __builtin_amdgcn_sched_group_barrier(0x008, PER, 0);
        if (c + 2 < STEPS) __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);
    }
}
template <int STEPS>      // transposed operands: two reads each
__device__ __forceinline__ void paced_cols() {
    __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
    for (int c = 0; c < STEPS; ++c) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if (c + 3 < STEPS) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
}

struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };

// What turns a raw product q.k into p and into the factor of ds (compare Form in attention_spans.hip: one fused multiply-add in front of exp2):
//     p = exp2(ka y - lse'),   ds = p (dout.v - delta) w
//   no cap:  y = raw - sum (slope / scale) |distance|,  ka = scale log2 e,                          lse' = lse log2 e,        w = 1
//   cap:     r = 1 / (exp(2 raw scale / cap) + 1),      tanh = 1 - 2 r,  1 - tanh^2 = 4 r (1 - r),  w = r (1 - r), the 4 in the factor at the end
//            without a bias y = r, ka = -2 cap log2 e, lse' = lse log2 e - cap log2 e;  with one y = cap log2 e (1 - 2 r) - sum slope log2 e |distance|, ka = 1
template <bool CAP, int AX>
struct BwdForm {
    float pre, ka, kb, c2, end, per;      // per: units of y in one of a slope
    __device__ __forceinline__ void init(const SpanArgs& p) {
        const float c1 = p.scale * SPAN_LOG2E;
        pre = CAP ? 2.f * c1 / p.cap : 1.f;
        c2 = p.cap * SPAN_LOG2E;
        ka = CAP ? (AX ? 1.f : -2.f * c2) : c1;
        kb = CAP && !AX ? c2 : 0.f;
        end = CAP ? 4.f * p.scale : p.scale;
        per = CAP ? SPAN_LOG2E : 1.f / p.scale;
    }
    // raw -> y (in front of the bias); w: factor of ds
    __device__ __forceinline__ float y(float raw, float& w) const {
        w = 1.f;
        if constexpr (!CAP) return raw;
        const float r = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(raw * pre) + 1.f);
        w = __builtin_fmaf(-r, r, r);
        return AX ? __builtin_fmaf(r, -2.f * c2, c2) : r;
    }
};

// 128 keys of a key head against the query tiles that see them: a wave holds 32 keys as operands (K, V) and their gradients as accumulators.
// ROLES (128 wide heads): 8 waves, the first four take dV, the others dK of the same keys -- both gradients and both operands are 192 registers, which leaves one wave
// per SIMD and every latency in the open.  The two waves of 32 keys make the scores, P and dS of half a query tile's rows each; what the other one multiplies by goes
// through LDS and is taken a tile later, dV's wave in front of its next scores, dK's behind them (Q and dO have three stages for it).  2 x 16 heads of 4096 x 4096, dq, dk
// and dv: S twice in waves of their own 1.10 ms (dk and dv alone 695 us; both in one wave 942), P handed over 1.05, scores shared 1.00 (capped, where the scores cost more:
// 1.31, 1.23 and 1.15).  Narrower heads take both gradients in one wave, two or three of which fit a SIMD.
template <int D, int AX>
struct DkvLds {
    // [ST] Q, [ST] dO, [2] per row: lse', delta, lo, hi, positions; with pairs [2] the operand that each of the eight waves has for its partner; the list
    static constexpr int T = Tile<D, BT>::BYTES, ST = D == 128 ? 3 : 2, G = ST * T, R = 2 * ST * T, ROWB = (4 + AX) * BT * 4, X = R + 2 * ROWB, LIST = X + (D == 128 ? 2 * 8 * 2048 : 0);
    static constexpr int BYTES = LIST + 256 * 4 + 512 * 16 + 16;
};
template <int D, int AX, bool CAP>
__device__ __forceinline__ void dkv_tile(const SpanArgs& p, unsigned id, unsigned char* smem) {
    typedef Tile<D, BT> T;
    constexpr bool ROLES = D == 128;
    constexpr int NW = ROLES ? 8 : 4, NT = NW * 64;
    typedef DkvLds<D, AX> M;
    int* list = reinterpret_cast<int*>(smem + M::LIST);                       // [256] query tiles
    int4* hull = reinterpret_cast<int4*>(list + 256);                         // [256][2] bounds of their two 32-row halves
    int* cnt = reinterpret_cast<int*>(hull + 512);                            // [4]
    const int t = threadIdx.x, lane = t & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6), w = ROLES ? wave & 3 : wave;
    const int tiles = (p.nk + BK - 1) / BK, total = p.B * p.Hk * p.splits * tiles, per = (total + 7) / 8;
    const int item = (id & 7) * per + (id >> 3);      // (a contiguous part of (row, key head, split, tile) per XCD)
    if (item >= total) return;
    const int tile = item % tiles, part = (item / tiles) % p.splits, hk = (item / tiles / p.splits) % p.Hk, b = item / tiles / p.splits / p.Hk;
    const int heads = p.Hq / p.Hk / p.splits, h0 = (hk * p.splits + part) * heads, h1 = h0 + heads;      // the query heads of this workgroup
    const int t0 = tile * BK, t1 = min(t0 + BK, p.nk), w0 = t0 + w * 32;      // the wave's keys: w0 .. w0 + 31
    const int key = w0 + (lane & 31);
    const bool live = key < p.nk && (!p.kmask || p.kmask[b * p.km_sb + key]);      // a key that is not there or masked: zeros, no weight
    const bool all_live = __all(live);
    const int mkey = live ? key : -1;      // (no span holds key -1)
    float pk[AX ? AX : 1];
#pragma unroll
    for (int a = 0; a < AX; ++a) pk[a] = key < p.nk ? (float)p.pos_k[b * p.pk_sb + (long)key * AX + a] : 0.f;
    BwdForm<CAP, AX> F;
    F.init(p);

    const int qtiles = (p.nq + BT - 1) / BT;
    // the tile being fetched: entry f_at of the list, head f_h, stages f_g (Q, dO) and f_st (its rows' numbers); its rows' numbers (lane = row of the 64, every wave the same; wave 0 writes them to LDS)
    float lsev = 0.f, delv = 0.f;
    int2 spv = make_int2(0, 0);
    int posv[AX ? AX : 1];
    float f_sl[AX ? AX : 1];
    int n_list = 0, f_at = 0, f_h = h0, f_st = 0, f_g = 0, f_rows = 0;
    const auto fetch = [&]() {      // (nothing here waits: the rows' numbers are looked at in settle(), a tile later)
        const int q0 = __builtin_amdgcn_readfirstlane(list[f_at]) * BT, i = min(q0 + lane, p.nq - 1);
        const long row = ((long)b * p.Hq + f_h) * p.nq + i;
        lsev = p.lse[row];
        delv = p.delta[row];
        spv = make_int2(0, p.nk);
        if (p.spans) spv = reinterpret_cast<const int2*>(p.spans + b * p.spans_sb)[i];
#pragma unroll
        for (int a = 0; a < AX; ++a) { posv[a] = p.pos_q[b * p.pq_sb + (long)i * AX + a]; f_sl[a] = p.slopes[f_h * AX + a]; }
        f_rows = p.nq - q0;
        const int ok = min(BT, f_rows);
        T::template fill<NW>(smem + f_g * M::T, p.q + b * p.q_s[0] + f_h * p.q_s[1] + (long)q0 * p.q_s[2], ok, (int)p.q_s[2], wave, lane);
        T::template fill<NW>(smem + M::G + f_g * M::T, p.dout + b * p.do_s[0] + f_h * p.do_s[1] + (long)q0 * p.do_s[2], ok, (int)p.do_s[2], wave, lane);
    };
    // rows that are not there, see nothing or whose lse says so: an empty span; which of the 64 see a key of this tile
    const auto settle = [&]() {
        const bool out = lane >= f_rows || lsev == -INFINITY;
        spv = out ? make_int2(0, 0) : make_int2(max(spv.x, 0), min(spv.y, p.nk));
        const bool in = spv.x < t1 && spv.y > t0;
        if (!in) spv = make_int2(0, 0);
        lsev = in ? __builtin_fmaf(lsev, SPAN_LOG2E, -F.kb) : 0.f;
        delv = in ? delv : 0.f;
        return __ballot(in);
    };
    const auto store_rows = [&]() {
        if (wave == 0) {
            float* rw = reinterpret_cast<float*>(smem + M::R + f_st * M::ROWB);
            int* ri = reinterpret_cast<int*>(rw);
            rw[lane] = lsev; rw[BT + lane] = delv;
            ri[2 * BT + lane] = spv.x; ri[3 * BT + lane] = spv.y;
#pragma unroll
            for (int a = 0; a < AX; ++a) rw[(4 + a) * BT + lane] = (float)posv[a];
        }
    };
    const auto pass = [&](auto take_v, auto take_k) {      // the whole walk over the query tiles, for the gradients that this wave takes
        constexpr bool DV = decltype(take_v)::value, DK = decltype(take_k)::value;
        u32x4_t kf[D / 16], vf[D / 16], own[2];      // own: the operand that this wave made of the tile before, for its own product
        const auto load_keys = [&]() {
            const uint16_t* kp = p.k + b * p.k_s[0] + hk * p.k_s[1] + (long)(live ? key : 0) * p.k_s[2] + half * 8;
            const uint16_t* vp = p.v + b * p.v_s[0] + hk * p.v_s[1] + (long)(live ? key : 0) * p.v_s[2] + half * 8;
            const u32x4_t z = {0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
                const u32x4_t x = *reinterpret_cast<const u32x4_t*>(kp + c * 16);
                const u32x4_t y = *reinterpret_cast<const u32x4_t*>(vp + c * 16);
                kf[c] = live ? x : z;
                vf[c] = live ? y : z;
            }
        };
        f32x16_t dk[DK ? D / 32 : 1], dv[DV ? D / 32 : 1];
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                if constexpr (DK) dk[c][r] = 0.f;
                if constexpr (DV) dv[c][r] = 0.f;
            }
        bool any = false;      // does any query see this tile
        const auto meets = [&](int at, int n) {      // do rows 32 n .. + 31 of a listed tile see one of the wave's keys
            const i32x4_t hl = lds_i4(hull + 2 * at + n);
            return __builtin_amdgcn_readfirstlane((int)(hl[0] < min(w0 + 32, t1) && hl[1] > w0)) != 0;
        };
        for (int base = 0; base < qtiles; base += 256) {
            // ---- the query tiles of this stretch that see keys of this tile, in order
            __syncthreads();
            {
                const int qt = base + t;
                int4 x = make_int4(INT32_MAX, 0, INT32_MAX, 0), y = x;
                if (t < 256 && qt < qtiles) {
                    const int4* hp = p.hulls + (long)b * p.hull_tiles + 2 * qt;
                    x = hp[0];
                    if (2 * qt + 1 < p.hull_tiles) y = hp[1];
                }
                const bool in = (x.x < t1 && x.y > t0) || (y.x < t1 && y.y > t0);
                const unsigned long long m = __ballot(in);
                if (lane == 0 && wave < 4) cnt[wave] = __popcll(m);
                __syncthreads();
                int to = __popcll(m & ((1ull << lane) - 1ull));
                for (int z = 0; z < min(wave, 4); ++z) to += cnt[z];
                n_list = __builtin_amdgcn_readfirstlane(cnt[0] + cnt[1] + cnt[2] + cnt[3]);
                if (in) { list[to] = qt; hull[2 * to] = x; hull[2 * to + 1] = y; }
                __syncthreads();
            }
            if (n_list == 0) continue;
            f_at = 0; f_h = h0; f_st = 0; f_g = 0;
            fetch();
            if (!any) load_keys();      // (behind the first tile's DMA, and not at all for keys that nobody sees)
            any = true;
            int p_at = -1, p_st = 0, p_g = 0;      // pairs: the tile whose operands are made
            const auto product = [&]() {
                if constexpr (ROLES) {
                    if (p_at < 0) return;
                    const unsigned char* As = smem + p_g * M::T + (DV ? M::G : 0);
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        if (!meets(p_at, n)) continue;
                        const unsigned char* xs = smem + M::X + ((p_st * 4 + w) * 2 + n) * 2048 + lane * 16;
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const u32x4_t f = n == (DV ? 0 : 1) ? own[x] : *reinterpret_cast<const u32x4_t*>(xs + x * 1024);
#pragma unroll
                            for (int c = 0; c < D / 32; ++c) {
                                if constexpr (DV) dv[c] = mfma32<false>(T::cols(As, 2 * n + x, c, lane), f, dv[c]);
                                else dk[c] = mfma32<false>(T::cols(As, 2 * n + x, c, lane), f, dk[c]);
                            }
                        }
                        paced_cols<D / 16>();
                    }
                }
            };
            for (bool more = true; more;) {
                const int at = f_at, st = f_st, gs = f_g;
                float sl[AX ? AX : 1];
#pragma unroll
                for (int a = 0; a < AX; ++a) sl[a] = f_sl[a] * F.per;
                const unsigned long long keep = settle();
                store_rows();
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();      // the tile and its rows' numbers are there for every wave; every wave is done with the other stage
                if (++f_at == n_list) { f_at = 0; ++f_h; }
                f_st ^= 1;
                f_g = f_g + 1 == M::ST ? 0 : f_g + 1;
                more = f_h < h1;
                if (more) fetch();
                const unsigned char* Qs = smem + gs * M::T;
                const unsigned char* Gs = smem + M::G + gs * M::T;
                if (keep != ~0ull) {      // rows that see no key of this tile take no part, whatever they hold (rows behind the last document)
                    T::clear_rows(smem + gs * M::T, keep, t, NT);
                    T::clear_rows(smem + M::G + gs * M::T, keep, t, NT);
                    lds_barrier();
                }
                if constexpr (DV) product();      // (dV's wave first, dK's behind its scores: one has the matrix pipe while the other has the vector pipe)
                u32x4_t made[2];
#pragma unroll
                for (int n = ROLES ? (DV ? 0 : 1) : 0; n < (ROLES ? (DV ? 1 : 2) : 2); ++n) {
                    if (!meets(at, n)) continue;
                    const i32x4_t hl = lds_i4(hull + 2 * at + n);
                    const bool masked = !all_live || __builtin_amdgcn_readfirstlane((int)!(hl[2] <= w0 && hl[3] >= w0 + 32)) != 0 || (uint32_t)(keep >> (32 * n)) != 0xFFFFFFFFu;
                    f32x16_t s, g;
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = g[r] = 0.f;
                    u32x4_t q0 = T::rows(Qs, 0, n, lane), q1 = T::rows(Qs, 1, n, lane), g0 = T::rows(Gs, 0, n, lane), g1 = T::rows(Gs, 1, n, lane);
#pragma unroll
                    for (int c = 0; c < D / 16; ++c) {
                        const u32x4_t x = q0, y = g0;
                        q0 = q1; g0 = g1;
                        if (c + 2 < D / 16) {
                            q1 = T::rows(Qs, c + 2, n, lane);
                            g1 = T::rows(Gs, c + 2, n, lane);
                        }
                        s = mfma32<false>(x, kf[c], s);
                        g = mfma32<false>(y, vf[c], g);
                    }
                    paced<2, D / 16>();
                    int rows = M::R + st * M::ROWB + (n * 32 + half * 4) * 4;
                    f32x4_t l4, d4, k4[AX ? AX : 1], ln, dn, kn[AX ? AX : 1];      // numbers of four rows, and of the next four
                    l4 = ln = lds_f4(smem + rows);
                    d4 = dn = lds_f4(smem + rows + BT * 4);
#pragma unroll
                    for (int a = 0; a < AX; ++a) k4[a] = kn[a] = lds_f4(smem + rows + (4 + a) * BT * 4);
#pragma unroll
                    for (int g4 = 0; g4 < 4; ++g4) {
                        if (g4 < 3) {
                            ln = lds_f4(smem + rows + (g4 + 1) * 32);
                            dn = lds_f4(smem + rows + BT * 4 + (g4 + 1) * 32);
#pragma unroll
                            for (int a = 0; a < AX; ++a) kn[a] = lds_f4(smem + rows + (4 + a) * BT * 4 + (g4 + 1) * 32);
                        }
                        float y4[4], w4[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) y4[e] = F.y(s[g4 * 4 + e], w4[e]);
#pragma unroll
                        for (int a = 0; a < AX; ++a) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) y4[e] = __builtin_fmaf(-sl[a], fabsf(k4[a][e] - pk[a]), y4[e]);
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) y4[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(y4[e], F.ka, -l4[e]));
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float d = y4[e] * (g[g4 * 4 + e] - d4[e]);
                            if constexpr (CAP) d *= w4[e];
                            w4[e] = d;
                        }
                        if constexpr (AX > 0) asm volatile("" : "+v"(rows), "+v"(w4[0]), "+v"(w4[1]), "+v"(w4[2]), "+v"(w4[3]));      // (done with these four before the next are fetched)
#pragma unroll
                        for (int e = 0; e < 4; ++e) g[g4 * 4 + e] = w4[e];
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[g4 * 4 + e] = y4[e];
                        l4 = ln; d4 = dn;
#pragma unroll
                        for (int a = 0; a < AX; ++a) k4[a] = kn[a];
                    }
                    if (masked) {
                        const int* ri = reinterpret_cast<const int*>(smem + M::R + st * M::ROWB) + 2 * BT + n * 32 + half * 4;
#pragma unroll
                        for (int g4 = 0; g4 < 4; ++g4) {
                            const i32x4_t lo = lds_i4(ri + g4 * 8), hi = lds_i4(ri + BT + g4 * 8);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {      // all ones: the row sees this key (spans are 0 <= lo <= hi)
                                const uint32_t z = (uint32_t)-(int)((uint32_t)(mkey - lo[e]) < (uint32_t)(hi[e] - lo[e]));
                                s[g4 * 4 + e] = __uint_as_float(__float_as_uint(s[g4 * 4 + e]) & z);
                                g[g4 * 4 + e] = __uint_as_float(__float_as_uint(g[g4 * 4 + e]) & z);
                            }
                        }
                    }
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const u32x4_t pf = pack_slots<false>(s, x), df = pack_slots<false>(g, x);      // P and dS rounded to bf16: operands
                        if constexpr (ROLES) {
                            made[x] = DV ? pf : df;
                            *reinterpret_cast<u32x4_t*>(smem + M::X + ((st * 4 + w) * 2 + n) * 2048 + x * 1024 + lane * 16) = DV ? df : pf;
                        } else {
#pragma unroll
                            for (int c = 0; c < D / 32; ++c) {
                                dv[c] = mfma32<false>(T::cols(Gs, 2 * n + x, c, lane), pf, dv[c]);
                                dk[c] = mfma32<false>(T::cols(Qs, 2 * n + x, c, lane), df, dk[c]);
                            }
                        }
                    }
                    if constexpr (!ROLES) paced_cols<D / 8>();
                }
                if constexpr (!DV) product();
                if constexpr (ROLES) {
                    own[0] = made[0]; own[1] = made[1];
                    p_at = at; p_st = st; p_g = gs;
                }
            }
            if constexpr (ROLES) {
                __syncthreads();
                product();
            }
        }
        // ---- out; a key whose gradient is not finite -- another key's infinity or NaN met its zero weight in the matrix instruction -- is computed again from its own rows
        const long prow = ((long)b * p.Hk + hk) * p.nk, pall = (long)p.B * p.Hk * p.nk;      // partial sums: [splits][dk, dv][rows][D]
        if (p.splits > 1) {      // (a tile that nothing sees has no parts)
            if (t == 0) p.seen[b * tiles + tile] = any;
            if (!any) return;
        }
        const auto put = [&](f32x16_t* acc, int which, float f) {
            float bad = 0.f;
#pragma unroll
            for (int c = 0; c < D / 32; ++c)
#pragma unroll
                for (int r = 0; r < 16; ++r) bad = __builtin_fmaf(acc[c][r], 0.f, bad);
            bad = both_halves_sum(bad);
            const bool redo = live && bad != 0.f;
            if (!live) f = 0.f;
            if (key < p.nk && !redo) {
                uint16_t* o = which ? p.dv + b * p.dv_s[0] + hk * p.dv_s[1] + (long)key * p.dv_s[2] : p.dk + b * p.dk_s[0] + hk * p.dk_s[1] + (long)key * p.dk_s[2];
                float* po = p.part_o + (((long)part * 2 + which) * pall + prow + key) * D;
#pragma unroll
                for (int c = 0; c < D / 32; ++c)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const float4 v = live ? make_float4(acc[c][4 * g] * f, acc[c][4 * g + 1] * f, acc[c][4 * g + 2] * f, acc[c][4 * g + 3] * f) : make_float4(0.f, 0.f, 0.f, 0.f);
                        if (p.splits > 1) *reinterpret_cast<float4*>(po + c * 32 + g * 8 + half * 4) = v;
                        else *reinterpret_cast<uint2*>(o + c * 32 + g * 8 + half * 4) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
                    }
            }
            unsigned long long todo = __ballot(redo) & 0xFFFFFFFFull;
#pragma nounroll
            while (todo) {
                const int r = __builtin_ctzll(todo);
                todo &= todo - 1;
                float a[2], c[2];
                key_again<D, AX>(p, b, hk, h0, h1, w0 + r, lane, a, c);
                if (which) { a[0] = c[0]; a[1] = c[1]; }
                else { a[0] *= p.scale; a[1] *= p.scale; }
                if (p.splits > 1) {
                    float* po = p.part_o + (((long)part * 2 + which) * pall + prow + w0 + r) * D;
                    if (lane < D) po[lane] = a[0];
                    if (D > 64) po[lane + 64] = a[1];
                } else {
                    uint16_t* o = which ? p.dv + b * p.dv_s[0] + hk * p.dv_s[1] + (long)(w0 + r) * p.dv_s[2] : p.dk + b * p.dk_s[0] + hk * p.dk_s[1] + (long)(w0 + r) * p.dk_s[2];
                    if (lane < D) o[lane] = f32_to_bf16(a[0]);
                    if (D > 64) o[lane + 64] = f32_to_bf16(a[1]);
                }
            }
        };
        if constexpr (DK) put(dk, 0, F.end);
        if constexpr (DV) put(dv, 1, 1.f);
    };
    if constexpr (!ROLES) pass(Yes(), Yes());
    else if (wave < 4) pass(Yes(), No());
    else pass(No(), Yes());
}

// dq and dk / dv read the same and need nothing of each other: one launch, the key tiles first, so that the end of one fills up with the other (a launch each: 6100 rows
// with one document of 2462, 16 / 4 heads of 128, capped: 256 us, 206 so; 8150 rows of packed images, 8 heads of 64, two axes: 114 and 91; 2 x 16 heads of 4096 x 4096,
// where both fill the card by themselves: 1.11 ms and 1.10)
template <int D, int AX, bool CAP>
__global__ __launch_bounds__(D == 128 ? 512 : 256, D == 32 ? 3 : 2) void span_bwd_main(const SpanArgs p) {
    extern __shared__ __attribute__((aligned(128))) unsigned char smem[];
    const int keys = (p.B * p.Hk * p.splits * ((p.nk + BK - 1) / BK) + 7) / 8 * 8;
    if ((int)blockIdx.x < keys) dkv_tile<D, AX, CAP>(p, blockIdx.x, smem);
    else dq_tile<D, AX, CAP, D == 128 ? 2 : 1>(p, blockIdx.x - keys, smem);
}

// adds the head splits of a key row in split order; masked keys' parts are zeros, tiles that nothing sees have none.  4 elements a thread
template <int D>
__global__ __launch_bounds__(256) void span_bwd_join(const SpanArgs p) {
    const long pall = (long)p.B * p.Hk * p.nk, x = (long)blockIdx.x * 256 + threadIdx.x;
    const long row = x / (D / 4);
    const int c = (int)(x % (D / 4)) * 4;
    if (row >= 2 * pall) return;
    const bool is_v = row >= pall;
    const long r = is_v ? row - pall : row;
    const int key = (int)(r % p.nk), hk = (int)(r / p.nk % p.Hk), b = (int)(r / p.nk / p.Hk);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (p.seen[b * ((p.nk + BK - 1) / BK) + key / BK]) {
        v = *reinterpret_cast<const float4*>(p.part_o + row * D + c);
        for (int s = 1; s < p.splits; ++s) {
            const float4 y = *reinterpret_cast<const float4*>(p.part_o + (s * 2 * pall + row) * D + c);
            v.x += y.x; v.y += y.y; v.z += y.z; v.w += y.w;
        }
    }
    uint16_t* o = is_v ? p.dv + b * p.dv_s[0] + hk * p.dv_s[1] + (long)key * p.dv_s[2] : p.dk + b * p.dk_s[0] + hk * p.dk_s[1] + (long)key * p.dk_s[2];
    *reinterpret_cast<uint2*>(o + c) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
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
        const long rows = (long)a.B * a.Hq * a.nq, rpb = 256 / (D / 8);
        const long blocks = (a.order_out ? 1 : 0) + ((long)a.B * a.hull_tiles + 7) / 8 + (rows + rpb - 1) / rpb;
        hipLaunchKernelGGL(span_bwd_pre<D>, dim3((unsigned)blocks), dim3(256), 0, s, a);
        if ((rc = mm_check_launch("span_bwd_pre"))) return rc;
    }
    if (a.nk > 0 || a.nq > 0) {
        constexpr int dq = DqLds<D, AX, D == 128 ? 2 : 1>::BYTES, dkv = DkvLds<D, AX>::BYTES, sm = dq > dkv ? dq : dkv;
        static std::atomic<unsigned long long> lds{0};
        if ((rc = span_allow_lds(reinterpret_cast<const void*>(span_bwd_main<D, AX, CAP>), sm, lds))) return rc;
        const long keys = ((long)a.B * a.Hk * a.splits * ((a.nk + BK - 1) / BK) + 7) / 8 * 8, rows = (long)a.B * a.Hq * ((a.nq + BQ - 1) / BQ);
        hipLaunchKernelGGL((span_bwd_main<D, AX, CAP>), dim3((unsigned)(keys + rows)), dim3(D == 128 ? 512 : 256), sm, s, a);
        if ((rc = mm_check_launch("span_bwd_main"))) return rc;
        if (a.splits > 1 && a.nk > 0) {
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

struct BwdLayout { size_t hulls, delta, done, seen, order, slopes, parts, bytes; int hull_tiles, splits; long slope_parts; };
BwdLayout bwd_layout(const mm_span_attn* a) {
    BwdLayout r;
    r.hull_tiles = (a->nq + 31) / 32;
    r.slope_parts = a->slopes && a->dslopes ? (long)a->batch * ((a->nq + BQ - 1) / BQ) : 0;
    size_t at = 0;
    r.hulls = at; at += (size_t)a->batch * r.hull_tiles * sizeof(int4);
    r.delta = at; at += ((size_t)a->batch * a->heads_q * a->nq * sizeof(float) + 15) / 16 * 16;
    r.done = at; at += 16;
    r.splits = head_splits(a);
    r.seen = at; at += r.splits > 1 ? (size_t)a->batch * ((a->nk + BK - 1) / BK) * sizeof(int) : 0;
    r.order = at; at += span_order_count(a) * sizeof(int32_t);
    r.slopes = at; at += (size_t)r.slope_parts * a->heads_q * a->axes * sizeof(float);
    at = (at + 15) / 16 * 16;
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
    if (span_order_count(a)) p.order = p.order_out = reinterpret_cast<int32_t*>((char*)ws + l.order);
    p.part_o = reinterpret_cast<float*>((char*)ws + l.parts);
    p.dsl_part = l.slope_parts ? reinterpret_cast<float*>((char*)ws + l.slopes) : nullptr;
    p.done = l.slope_parts ? reinterpret_cast<unsigned*>((char*)ws + l.done) : nullptr;
    p.seen = reinterpret_cast<int*>((char*)ws + l.seen);
    p.dslopes = a->dslopes;
    if (a->slopes && a->dslopes && !l.slope_parts)      // (no rows: zeros)
        if (const int rc = k_colsum(s, a->dslopes, 0, (long)a->heads_q * a->axes, a->dslopes)) return rc;
    return a->dim == 32 ? launch_bwd_dim<32>(s, p) : (a->dim == 64 ? launch_bwd_dim<64>(s, p) : launch_bwd_dim<128>(s, p));
}
