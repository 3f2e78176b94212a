// Attention of packed rows, forward:   out_i = sum over the keys lo_i <= key < hi_i of softmax(s)_key v_key,   s = cap(scale q.k) - sum_a slope_a |pos_q - pos_k|
// One pass over the keys with a running maximum and sum per query.  S^T = K Q^T puts a query into a lane's column (common layout in span_attn.h): its scores, maximum,
// sum and the rescaling of its output stay in that lane (and its partner in the other half wave), P needs no LDS, O^T = V^T P^T.
//   span_attn_wide   : 128 queries of one head (4 waves x 32), key tiles of 64 shared by the waves, double-buffered by LDS-DMA.  A wave passes over tiles that none of
//                      its rows sees; tiles that all of its rows see whole take no mask.
//   span_attn_narrow : few rows (a new position over a cache, one image): 32 rows = (heads that share a key head) x queries; the four waves take every fourth 32-key tile
//                      each, on their own, and are joined through LDS; longer key ranges are split over workgroups as well and joined by span_attn_join in split order.
// What a row does not see never reaches it: rows behind the workgroup's key range are not read (zeros), rows that the key mask hides are cleared in LDS, and a row whose
// output is not finite although its sum is -- another row's infinity or NaN met its zero weight in the matrix instruction -- is computed again from its own keys alone.
#include <string.h>

#include "span_attn.h"

namespace {

constexpr int WQ = SPAN_TILE, KT = 64;

// sum over this row's visible keys in [k0, k1) of exp2(s - m) v, by one wave: lane = key for the scores, lane = element for the sum
template <int D, bool F16, int AX, bool TANH>
__device__ __forceinline__ void row_again(const SpanArgs& p, int b, int h, int i, int k0, int k1, float m, int lane, float (&o)[2]) {
    const uint16_t* q = p.q + b * p.q_s[0] + h * p.q_s[1] + (long)i * p.q_s[2];
    const int hk = h / (p.Hq / p.Hk);
    const uint16_t* kb = p.k + b * p.k_s[0] + hk * p.k_s[1];
    const uint16_t* vb = p.v + b * p.v_s[0] + hk * p.v_s[1];
    o[0] = o[1] = 0.f;
#pragma nounroll
    for (int t0 = k0; t0 < k1 && !all_nan<D>(o, lane); t0 += 64) {
        const int key = t0 + lane;
        const bool sees = key < k1 && (!p.kmask || p.kmask[b * p.km_sb + key]);
        float w = 0.f, unused;
        if (sees) w = __builtin_amdgcn_exp2f(pair_score<D, F16, AX, TANH>(p, q, kb + (long)key * p.k_s[2], b, h, i, key, &unused) - m);
        rows_add<D, F16>(o, __ballot(sees), w, vb + (long)t0 * p.v_s[2], p.v_s[2], min(64, k1 - t0), lane);
    }
}

// A score passes through three forms.  raw: the product q.k.  y: what the maximum is taken of --
//     no cap:          raw - sum (slope / scale) |distance|,     score = ka y,       ka = scale log2 e
//     cap, no bias:    r = 1 / (exp(2 raw scale / cap) + 1),     score = ka y + kb,  ka = -2 cap log2 e, kb = cap log2 e   (cap tanh(x) = cap - 2 cap r: smallest r)
//     cap and bias:    cap tanh(..) - sum slope |distance|,      score = y           (all in units of log2)
// and p = exp2(ka y + (kb - m)): one fused multiply-add in front of exp2 whatever the form.
// TANH: the tanh itself comes in (span_tanh_block: a score to a few roundings of its own size, not of the cap's, and so the lse of a row of few keys); the cap without a bias
// is then y = tanh, ka = cap log2 e, kb = 0.
template <bool CAP, int AX, bool TANH = false>
struct Form {
    static constexpr bool falls = CAP && AX == 0 && !TANH;      // the score falls with y
    float pre, ka, kb, sl[AX ? AX : 1];
    __device__ __forceinline__ void init(const SpanArgs& p, int h) {
        const float c1 = p.scale * SPAN_LOG2E;
        pre = CAP ? 2.f * c1 / p.cap : 1.f;
        c2 = p.cap * SPAN_LOG2E;
        ka = CAP ? (AX ? 1.f : (TANH ? c2 : -2.f * c2)) : c1;
        kb = falls ? c2 : 0.f;
#pragma unroll
        for (int a = 0; a < AX; ++a) sl[a] = CAP ? p.slopes[h * AX + a] * SPAN_LOG2E : p.slopes[h * AX + a] / p.scale;
    }
    float c2;
    // 4 consecutive keys (k: their positions).  Positions are whole numbers below 2^24 in size, exact in fp32; a distance is too up to 2^24, and rounded once above (signs
    // apart): a subtraction and a multiply-add with |.| an axis and score
    __device__ __forceinline__ void y4(f32x16_t& s, int r, const float (&pq)[AX ? AX : 1], const f32x4_t (&k)[AX ? AX : 1]) const {
        float v[4] = {s[r], s[r + 1], s[r + 2], s[r + 3]};
        if constexpr (CAP && TANH) {
            if constexpr (AX > 0)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] *= c2;
        } else if constexpr (CAP) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(v[e] * pre) + 1.f);
                if constexpr (AX > 0) v[e] = __builtin_fmaf(v[e], -2.f * c2, c2);
            }
        }
#pragma unroll
        for (int a = 0; a < AX; ++a) {
            v[0] = __builtin_fmaf(-sl[a], fabsf(pq[a] - k[a].x), v[0]);
            v[1] = __builtin_fmaf(-sl[a], fabsf(pq[a] - k[a].y), v[1]);
            v[2] = __builtin_fmaf(-sl[a], fabsf(pq[a] - k[a].z), v[2]);
            v[3] = __builtin_fmaf(-sl[a], fabsf(pq[a] - k[a].w), v[3]);
        }
        s[r] = v[0]; s[r + 1] = v[1]; s[r + 2] = v[2]; s[r + 3] = v[3];
    }
    // hidden keys out: w bit 8 (r >> 2) + (r & 3) of block n for register r (already shifted by the half)
    __device__ __forceinline__ void hide(f32x16_t& s, uint32_t w) const {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const uint32_t t = (uint32_t)((int)(w << (31 - (8 * (r >> 2) + (r & 3)))) >> 31);      // all ones: visible
            s[r] = __uint_as_float((t & __float_as_uint(s[r])) | (~t & (falls ? 0x7F800000u : 0xFF800000u)));
        }
    }
    __device__ __forceinline__ float extreme(const f32x16_t& s, float m) const {
#pragma unroll
        for (int r = 0; r < 16; ++r) m = falls ? fminf(m, s[r]) : fmaxf(m, s[r]);
        return m;
    }
    static __device__ __forceinline__ float worst() { return falls ? INFINITY : -INFINITY; }
    __device__ __forceinline__ float score(float y) const { return __builtin_fmaf(y, ka, kb); }
};

// The weights' reference m follows the running maximum: it moves only when some row's maximum passes m + TOP, and then to UP below it.  Most tiles rescale nothing.
// bf16: P stays below 2^8.  fp16 has no exponents to spare: weights below 2^-24 would vanish as operands, though a long cache of them counts (131072 keys of 2^-25 beside one
// key of 1: 0 for 0.003), and those below 2^-14 lose bits.  There P lies between 2^10 and 2^14 at a row's maximum, so that weights down to 2^-24 of it keep all their bits.
template <bool F16> constexpr float UP = F16 ? 10.f : 0.f;
template <bool F16> constexpr float TOP = F16 ? 14.f : 8.f;
template <int D, bool F16>
__device__ __forceinline__ void rescale(float tmax, float& m, float& l, f32x16_t (&o)[D / 32]) {
    tmax = both_halves_max(tmax);
    if (__any(tmax > m + TOP<F16>)) {
        const float mn = fmaxf(m, tmax - UP<F16>), f = __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= f;
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[c][r] *= f;
    }
}

// lse of a row from its reference and its sum (the sum back in the maximum's units first: its logarithm is rounded at its own size); nothing seen: -inf
template <bool F16>
__device__ __forceinline__ float row_lse(float m, float l) {
    constexpr float down = F16 ? 1.f / 1024.f : 1.f;      // 2^-UP
    return l > 0.f ? (m + UP<F16> + __builtin_amdgcn_logf(l * down)) * SPAN_LN2 : (l == 0.f ? -INFINITY : l);
}

// 8 probabilities of a lane -> an operand.  Rounding of P to 16 bits: the product with V needs it; the sum takes the unrounded values
template <bool F16>
__device__ __forceinline__ u32x4_t probs(const f32x16_t& s, int x, float ka, float kbm, float& l) {
    float q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * x + e], ka, kbm));
    l += ((q[0] + q[1]) + (q[2] + q[3])) + ((q[4] + q[5]) + (q[6] + q[7]));
    return u32x4_t{pack2<F16>(q[0], q[1]), pack2<F16>(q[2], q[3]), pack2<F16>(q[4], q[5]), pack2<F16>(q[6], q[7])};
}

struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };

// AHEAD (128 wide heads): the product of tile it + 1's keys with the queries is issued between the instructions that turn tile it's scores into probabilities
// (independent work for the matrix and the vector pipe from one wave); K then runs one tile ahead of V in the two stages.  It needs a second set of scores: narrower
// heads lose their third wave per SIMD to it and are slower (16300 rows of packed images, 64 wide, two axes: 81 against 66 us; 128 wide, capped: 138 against 155).
template <int D, bool F16, int AX, bool CAP>
__global__ __launch_bounds__(256, 2) void span_attn_wide(const SpanArgs p) {
    typedef Tile<D, KT> T;
    constexpr bool AHEAD = D == 128;
    extern __shared__ __attribute__((aligned(128))) unsigned char smem[];
    constexpr int POS = AX * KT * 4, STAGE = 2 * T::BYTES + POS;
    int* red = reinterpret_cast<int*>(smem + 2 * STAGE);
    const int t = threadIdx.x, lane = t & 63, half = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(t >> 6);
    const int tiles = (p.nq + WQ - 1) / WQ;
    int rt, h;
    if (!span_item(blockIdx.x, p.order, p.Hq, p.B * tiles, rt, h)) return;
    const int tile = rt % tiles, b = rt / tiles, hk = h / (p.Hq / p.Hk);
    const int i = tile * WQ + w * 32 + (lane & 31);
    const bool ok = i < p.nq;

    int lo = 0, hi = 0;
    if (ok) {
        hi = p.nk;
        if (p.spans) {
            const int2 sp = reinterpret_cast<const int2*>(p.spans + b * p.spans_sb)[i];
            lo = max(sp.x, 0); hi = min(sp.y, p.nk);
        }
        if (lo >= hi) lo = hi = 0;
    }
    int h0 = hi > lo ? lo : INT32_MAX, h1 = hi;
    for (int o = 16; o > 0; o >>= 1) { h0 = min(h0, __shfl_xor(h0, o, 64)); h1 = max(h1, __shfl_xor(h1, o, 64)); }
    if (lane == 0) { red[w] = h0; red[4 + w] = h1; }
    u32x4_t qf[D / 16];
    {
        const uint16_t* qp = p.q + b * p.q_s[0] + h * p.q_s[1] + (long)(ok ? i : 0) * p.q_s[2] + half * 8;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) qf[c] = *reinterpret_cast<const u32x4_t*>(qp + c * 16);
    }
    float pq[AX ? AX : 1];
#pragma unroll
    for (int a = 0; a < AX; ++a) pq[a] = ok ? (float)p.pos_q[b * p.pq_sb + (long)i * AX + a] : 0.f;
    Form<CAP, AX> F;
    F.init(p, h);
    __syncthreads();
    const int k0 = __builtin_amdgcn_readfirstlane(min(min(red[0], red[1]), min(red[2], red[3])));
    const int k1 = __builtin_amdgcn_readfirstlane(max(max(red[4], red[5]), max(red[6], red[7])));
    const int nt = k1 > k0 ? (k1 - k0 + KT - 1) / KT : 0;

    const uint16_t* kp = p.k + b * p.k_s[0] + hk * p.k_s[1];
    const uint16_t* vp = p.v + b * p.v_s[0] + hk * p.v_s[1];
    const uint8_t* km = p.kmask ? p.kmask + b * p.km_sb : nullptr;
    const int* pkp = AX ? p.pos_k + b * p.pk_sb : nullptr;

    float m = SPAN_LOW, l = 0.f;
    f32x16_t o[D / 32], sa[2], sb[2];
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[c][r] = 0.f;
    int posv = 0;
    const auto fill_k = [&](int it) {
        const int t0 = k0 + it * KT;
        T::template fill<4>(smem + (it & 1) * STAGE, kp + (long)t0 * p.k_s[2], min(KT, k1 - t0), (int)p.k_s[2], w, lane);
    };
    const auto fill_v = [&](int it) {
        const int t0 = k0 + it * KT;
        T::template fill<4>(smem + (it & 1) * STAGE + T::BYTES, vp + (long)t0 * p.v_s[2], min(KT, k1 - t0), (int)p.v_s[2], w, lane);
    };
    const auto pos_load = [&](int it) {
        if constexpr (AX > 0) {
            if (t < KT * AX) { const int key = k0 + it * KT + t / AX; posv = key < k1 ? pkp[(long)key * AX + t % AX] : 0; }
        }
    };
    const auto pos_store = [&](int it) {
        if constexpr (AX > 0) {
            if (t < KT * AX) reinterpret_cast<float*>(smem + (it & 1) * STAGE + 2 * T::BYTES)[(t % AX) * KT + t / AX] = (float)posv;
        }
    };
    const auto sees = [&](int it) { return it < nt && __any(lo < k0 + it * KT + KT && hi > k0 + it * KT); };
    constexpr int NC = D / 16, E = 8 / NC;      // product steps; groups of 4 scores beside each
    // scores of the next tile (into sn) and y of this tile's (s), together or one of them
    const auto mix = [&](int it, f32x16_t (&s)[2], f32x16_t (&sn)[2], auto with_next, auto with_this) {
        const unsigned char* Kn = smem + ((it + 1) & 1) * STAGE;
        int pos = (it & 1) * STAGE + 2 * T::BYTES + half * 16;
        // positions of this group of four keys and of the next (their read waits in the open otherwise: 2 x 16 heads of 4096 x 4096, 64 wide, two axes 279 us, 256 so)
        f32x4_t pk[AX ? AX : 1], pn[AX ? AX : 1];
        if constexpr (with_this.value && AX > 0)
#pragma unroll
            for (int a = 0; a < AX; ++a) pk[a] = lds_f4(smem + pos + a * KT * 4);
        u32x4_t f0, f1;
        if constexpr (with_next.value) {
#pragma unroll
            for (int r = 0; r < 16; ++r) sn[0][r] = sn[1][r] = 0.f;
            f0 = T::rows(Kn, 0, 0, lane); f1 = T::rows(Kn, 0, 1, lane);
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            if constexpr (with_next.value) {
                const u32x4_t a0 = f0, a1 = f1;
                if (c + 1 < NC) { f0 = T::rows(Kn, c + 1, 0, lane); f1 = T::rows(Kn, c + 1, 1, lane); }
                sn[0] = mfma32<F16>(a0, qf[c], sn[0]);
                sn[1] = mfma32<F16>(a1, qf[c], sn[1]);
            }
            if constexpr (with_this.value && (CAP || AX > 0)) {
#pragma unroll
                for (int x = 0; x < E; ++x) {
                    const int g = c * E + x;
                    if constexpr (AX > 0)
                        if (g < 7)
#pragma unroll
                            for (int a = 0; a < AX; ++a) pn[a] = lds_f4(smem + pos + a * KT * 4 + ((g + 1) >> 2) * 128 + ((g + 1) & 3) * 32);
                    F.y4(s[g >> 2], (g & 3) * 4, pq, pk);
                    // y of these four now, the next group's positions behind it: left alone, the compiler moves three of the four behind the branch on the mask and keeps
                    // the positions of all 64 keys until then (32 registers an axis: a wave per SIMD)
                    if constexpr (AX > 0) {
                        f32x16_t& y = s[g >> 2];
                        const int r = (g & 3) * 4;
                        float y0 = y[r], y1 = y[r + 1], y2 = y[r + 2], y3 = y[r + 3];
                        asm volatile("" : "+v"(pos), "+v"(y0), "+v"(y1), "+v"(y2), "+v"(y3));
                        y[r] = y0; y[r + 1] = y1; y[r + 2] = y2; y[r + 3] = y3;
#pragma unroll
                        for (int a = 0; a < AX; ++a) pk[a] = pn[a];
                    }
                }
            }
        }
    };
    const auto step = [&](int it, f32x16_t (&s)[2], f32x16_t (&sn)[2]) {
        const int t0 = k0 + it * KT;
        unsigned char* Vs = smem + (it & 1) * STAGE + T::BYTES;
        unsigned long long keep = ~0ull;
        if (km) keep = __ballot(t0 + lane < k1 && km[t0 + lane]);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();      // V of tile it and K of tile it (+ 1: AHEAD) have landed for every wave, and every wave is done with what the fills below write over
        if (it + 1 < nt) {
            if constexpr (!AHEAD) fill_k(it + 1);
            fill_v(it + 1);
            pos_load(it + 1);
        }
        if (AHEAD && it + 2 < nt) fill_k(it + 2);
        if (keep != ~0ull) {
            T::clear_rows(Vs, keep, t, 256);
            lds_barrier();
        }
        const bool now = sees(it);
        if constexpr (AHEAD) {
            const bool next = sees(it + 1);
            if (now && next) mix(it, s, sn, Yes(), Yes());
            else if (next) mix(it, s, sn, Yes(), No());
            else if (now) mix(it, s, sn, No(), Yes());
        } else if (now) {
            mix(it - 1, s, s, Yes(), No());
            mix(it, s, s, No(), Yes());
        }
        if (now) {
            if (keep != ~0ull || !__all(lo <= t0 && hi >= t0 + KT)) {
                const unsigned long long bits = (bit_range(lo - t0, hi - t0) & keep) >> (4 * half);
                F.hide(s[0], (uint32_t)bits);
                F.hide(s[1], (uint32_t)(bits >> 32));
            }
            rescale<D, F16>(F.score(F.extreme(s[1], F.extreme(s[0], Form<CAP, AX>::worst()))), m, l, o);
            const float kbm = F.kb - m;
            u32x4_t pf = probs<F16>(s[0], 0, F.ka, kbm, l);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                u32x4_t vf[D / 32];
#pragma unroll
                for (int c = 0; c < D / 32; ++c) vf[c] = T::cols(Vs, ks, c, lane);
                const u32x4_t pc = pf;
#pragma unroll
                for (int c = 0; c < D / 32; ++c) o[c] = mfma32<F16>(vf[c], pc, o[c]);
                if (ks < 3) pf = probs<F16>(s[(ks + 1) >> 1], (ks + 1) & 1, F.ka, kbm, l);
            }
        }
        if (it + 1 < nt) pos_store(it + 1);
    };
    if (nt > 0) {
        fill_k(0);
        pos_load(0);
        pos_store(0);
        if constexpr (AHEAD) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            fill_v(0);
            if (nt > 1) fill_k(1);
            if (sees(0)) mix(-1, sb, sa, Yes(), No());
            for (int it = 0; it < nt; it += 2) {
                step(it, sa, sb);
                if (it + 1 < nt) step(it + 1, sb, sa);
            }
        } else {
            fill_v(0);
            for (int it = 0; it < nt; ++it) step(it, sa, sa);
        }
    }

    l = both_halves_sum(l);
    const float inv = l > 0.f ? 1.f / l : 0.f;
    if (p.lse && ok && half == 0) p.lse[((long)b * p.Hq + h) * p.nq + i] = row_lse<F16>(m, l);
    float bad = 0.f;
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) bad = __builtin_fmaf(o[c][r], 0.f, bad);
    bad = both_halves_sum(bad);
    const bool redo = ok && bad != 0.f && l * 0.f == 0.f;      // (bad is 0 or NaN; NaN != 0)
    if (ok && !redo) {
        const float f = l != l ? l : inv;
        uint16_t* op = p.out + b * p.o_s[0] + h * p.o_s[1] + (long)i * p.o_s[2] + half * 4;
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<uint2*>(op + c * 32 + g * 8) = make_uint2(pack2<F16>(o[c][4 * g] * f, o[c][4 * g + 1] * f), pack2<F16>(o[c][4 * g + 2] * f, o[c][4 * g + 3] * f));
    }
    unsigned long long todo = __ballot(redo) & 0xFFFFFFFFull;
#pragma nounroll
    while (todo) {
        const int r = __builtin_ctzll(todo);
        todo &= todo - 1;
        const int ri = tile * WQ + w * 32 + r;
        float ro[2];
        row_again<D, F16, AX, false>(p, b, h, ri, __shfl(lo, r, 64), __shfl(hi, r, 64), __shfl(m, r, 64), lane, ro);
        const float rinv = __shfl(inv, r, 64);
        uint16_t* op = p.out + b * p.o_s[0] + h * p.o_s[1] + (long)ri * p.o_s[2];
        if (lane < D) op[lane] = (uint16_t)pack2<F16>(ro[0] * rinv, 0.f);
        if (D > 64) op[lane + 64] = (uint16_t)pack2<F16>(ro[1] * rinv, 0.f);
    }
}

template <int D, bool F16, int AX, bool CAP>
__global__ __launch_bounds__(256, 2) void span_attn_narrow(const SpanArgs p) {
    typedef Tile<D, 32> T;
    constexpr int POS = AX * 32 * 4, STAGE = 2 * T::BYTES + POS, OS = D + 4;      // OS: row of the joined output in floats
    extern __shared__ __attribute__((aligned(128))) unsigned char smem[];
    float* ml = reinterpret_cast<float*>(smem + (8 * STAGE > 4 * 32 * OS * 4 ? 8 * STAGE : 4 * 32 * OS * 4));      // [4][32][2]
    float* os = reinterpret_cast<float*>(smem);                                                                     // [4][32][OS], over the tiles
    const int t = threadIdx.x, lane = t & 63, half = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(t >> 6);
    const int group = p.Hq / p.Hk, rows = group * p.nq;
    const int rt = blockIdx.x % p.row_tiles, hk = (blockIdx.x / p.row_tiles) % p.Hk, b = blockIdx.x / p.row_tiles / p.Hk, split = blockIdx.y;
    const int row = rt * 32 + (lane & 31);
    const bool ok = row < rows;
    const int h = hk * group + (ok ? row / p.nq : 0), i = ok ? row % p.nq : 0;
    int lo = 0, hi = 0;
    if (ok) {
        hi = p.nk;
        if (p.spans) {
            const int2 sp = reinterpret_cast<const int2*>(p.spans + b * p.spans_sb)[i];
            lo = max(sp.x, 0); hi = min(sp.y, p.nk);
        }
        if (lo >= hi) lo = hi = 0;
    }
    int k0 = hi > lo ? lo : INT32_MAX, k1 = hi;
    for (int o = 16; o > 0; o >>= 1) { k0 = min(k0, __shfl_xor(k0, o, 64)); k1 = max(k1, __shfl_xor(k1, o, 64)); }
    k0 = __builtin_amdgcn_readfirstlane(k0); k1 = __builtin_amdgcn_readfirstlane(k1);
    if (k1 > k0) {      // this split's keys: whole rounds of the four waves
        const int chunk = ((k1 - k0 + p.splits - 1) / p.splits + 127) / 128 * 128;
        k0 = (int)min((long)k0 + (long)split * chunk, (long)k1);
        k1 = (int)min((long)k0 + chunk, (long)k1);
    } else k0 = k1 = 0;
    const int nt = (k1 - k0 + 31) / 32;      // tiles of 32; this wave takes w, w + 4, ...

    u32x4_t qf[D / 16];
    {
        const uint16_t* qp = p.q + b * p.q_s[0] + h * p.q_s[1] + (long)i * p.q_s[2] + half * 8;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) qf[c] = *reinterpret_cast<const u32x4_t*>(qp + c * 16);
    }
    float pq[AX ? AX : 1];
#pragma unroll
    for (int a = 0; a < AX; ++a) pq[a] = (float)p.pos_q[b * p.pq_sb + (long)i * AX + a];
    Form<CAP, AX, true> F;      // (memory and latency are what bounds this form: tanh to its own size costs nothing here)
    F.init(p, h);
    const float cap_k = CAP ? p.scale / p.cap : 0.f;
    const uint16_t* kp = p.k + b * p.k_s[0] + hk * p.k_s[1];
    const uint16_t* vp = p.v + b * p.v_s[0] + hk * p.v_s[1];
    const uint8_t* km = p.kmask ? p.kmask + b * p.km_sb : nullptr;
    const int* pkp = AX ? p.pos_k + b * p.pk_sb : nullptr;
    unsigned char* mine = smem + w * 2 * STAGE;

    float m = SPAN_LOW, l = 0.f;
    f32x16_t o[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[c][r] = 0.f;
#define SPAN_ISSUE(tt_, st_)                                                                                           \
    {                                                                                                                  \
        const int t0_ = k0 + (tt_) * 32;                                                                               \
        unsigned char* sp_ = mine + (st_) * STAGE;                                                                     \
        T::template fill<1>(sp_, kp + (long)t0_ * p.k_s[2], min(32, k1 - t0_), (int)p.k_s[2], 0, lane);                \
        T::template fill<1>(sp_ + T::BYTES, vp + (long)t0_ * p.v_s[2], min(32, k1 - t0_), (int)p.v_s[2], 0, lane);     \
    }
    int st = 0;
    if (w < nt) SPAN_ISSUE(w, 0);
    for (int tt = w; tt < nt; tt += 4, st ^= 1) {
        const int t0 = k0 + tt * 32;
        unsigned char* Ks = mine + st * STAGE;
        unsigned char* Vs = Ks + T::BYTES;
        float* pks = reinterpret_cast<float*>(Ks + 2 * T::BYTES);
        if constexpr (AX > 0) {
            if (lane < 32) {
#pragma unroll
                for (int a = 0; a < AX; ++a) pks[a * 32 + lane] = t0 + lane < k1 ? (float)pkp[(long)(t0 + lane) * AX + a] : 0.f;
            }
        }
        uint32_t keep = 0xFFFFFFFFu;
        if (km) keep = (uint32_t)__ballot(lane < 32 && t0 + lane < k1 && km[t0 + lane]);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");      // (the wave's own tile: no barrier)
        if (tt + 4 < nt) SPAN_ISSUE(tt + 4, st ^ 1);
        if (keep != 0xFFFFFFFFu) T::clear_rows(Vs, keep, lane, 64);
        __builtin_amdgcn_wave_barrier();
        f32x16_t s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) s = mfma32<F16>(T::rows(Ks, c, 0, lane), qf[c], s);
        if constexpr (CAP) {
            const SpanTanh tanh = span_tanh_block(s, cap_k);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = span_tanh_poly(s[r] * tanh.k, tanh.c);
        }
        if constexpr (AX > 0)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                f32x4_t pk[AX ? AX : 1];
#pragma unroll
                for (int a = 0; a < AX; ++a) pk[a] = lds_f4(pks + a * 32 + g * 8 + half * 4);
                F.y4(s, g * 4, pq, pk);
            }
        if (keep != 0xFFFFFFFFu || !__all(lo <= t0 && hi >= t0 + 32)) F.hide(s, (uint32_t)((bit_range(lo - t0, hi - t0) & (unsigned long long)keep) >> (4 * half)));
        rescale<D, F16>(F.score(F.extreme(s, Form<CAP, AX, true>::worst())), m, l, o);
        const float kbm = F.kb - m;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            const u32x4_t pf = probs<F16>(s, ks, F.ka, kbm, l);
#pragma unroll
            for (int c = 0; c < D / 32; ++c) o[c] = mfma32<F16>(T::cols(Vs, ks, c, lane), pf, o[c]);
        }
    }
#undef SPAN_ISSUE
    // ---- join the four waves: common maximum, then the sums in wave order
    l = both_halves_sum(l);
    if (half == 0) { ml[(w * 32 + lane) * 2] = m; ml[(w * 32 + lane) * 2 + 1] = l; }
    __syncthreads();      // (also: every wave is done with its tiles)
    {
        const int r = lane & 31;
        const float M = fmaxf(fmaxf(ml[r * 2], ml[(32 + r) * 2]), fmaxf(ml[(64 + r) * 2], ml[(96 + r) * 2]));
        const float f = __builtin_amdgcn_exp2f(m - M);
        float* dst = os + (w * 32 + r) * OS + half * 4;
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
            for (int g = 0; g < 4; ++g) *reinterpret_cast<float4*>(dst + c * 32 + g * 8) = make_float4(o[c][4 * g] * f, o[c][4 * g + 1] * f, o[c][4 * g + 2] * f, o[c][4 * g + 3] * f);
    }
    __syncthreads();
    // thread t: row t >> 3 of the tile, every 8th group of 4 elements
    const int r = t >> 3, rr = rt * 32 + r;
    float M = SPAN_LOW, L = 0.f;
#pragma unroll
    for (int x = 0; x < 4; ++x) M = fmaxf(M, ml[(x * 32 + r) * 2]);
#pragma unroll
    for (int x = 0; x < 4; ++x) L += ml[(x * 32 + r) * 2 + 1] * __builtin_amdgcn_exp2f(ml[(x * 32 + r) * 2] - M);
    float4 v[D / 32];
    float bad = 0.f;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
        v[c] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const float4 y = *reinterpret_cast<const float4*>(os + (x * 32 + r) * OS + (c * 8 + (t & 7)) * 4);
            v[c].x += y.x; v[c].y += y.y; v[c].z += y.z; v[c].w += y.w;
        }
        bad += (v[c].x + v[c].y + v[c].z + v[c].w) * 0.f;
    }
#pragma unroll
    for (int x = 1; x < 8; x <<= 1) bad += __shfl_xor(bad, x, 64);
    const bool live = rr < rows, redo = live && bad != 0.f && L * 0.f == 0.f;
    const int rh = hk * group + (live ? rr / p.nq : 0), ri = live ? rr % p.nq : 0;
    const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
    const long prow = (((long)b * p.Hk + hk) * p.row_tiles + rt) * 32 + r, prows = (long)p.B * p.Hk * p.row_tiles * 32;
    if (live && p.splits == 1) {
        uint16_t* op = p.out + b * p.o_s[0] + rh * p.o_s[1] + (long)ri * p.o_s[2];
        if (!redo)
#pragma unroll
            for (int c = 0; c < D / 32; ++c)
                *reinterpret_cast<uint2*>(op + (c * 8 + (t & 7)) * 4) = make_uint2(pack2<F16>(v[c].x * inv, v[c].y * inv), pack2<F16>(v[c].z * inv, v[c].w * inv));
        if (p.lse && (t & 7) == 0) p.lse[((long)b * p.Hq + rh) * p.nq + ri] = row_lse<F16>(M, L);
    } else if (live) {
        float* po = p.part_o + (split * prows + prow) * D;
        if (!redo)
#pragma unroll
            for (int c = 0; c < D / 32; ++c) *reinterpret_cast<float4*>(po + (c * 8 + (t & 7)) * 4) = v[c];
        if ((t & 7) == 0) { p.part_ml[(split * prows + prow) * 2] = M; p.part_ml[(split * prows + prow) * 2 + 1] = L; }
    }
    unsigned long long todo = __ballot(redo && (t & 7) == 0);
#pragma nounroll
    while (todo) {
        const int src = __builtin_ctzll(todo);
        todo &= todo - 1;
        const int xr = rt * 32 + w * 8 + (src >> 3), xh = hk * group + xr / p.nq, xi = xr % p.nq;
        int xlo = 0, xhi = p.nk;
        if (p.spans) {
            const int2 sp = reinterpret_cast<const int2*>(p.spans + b * p.spans_sb)[xi];
            xlo = max(sp.x, 0); xhi = min(sp.y, p.nk);
        }
        float ro[2];
        row_again<D, F16, AX, true>(p, b, xh, xi, max(xlo, k0), min(xhi, k1), __shfl(M, src, 64), lane, ro);
        const float rinv = __shfl(inv, src, 64);
        if (p.splits == 1) {
            uint16_t* op = p.out + b * p.o_s[0] + xh * p.o_s[1] + (long)xi * p.o_s[2];
            if (lane < D) op[lane] = (uint16_t)pack2<F16>(ro[0] * rinv, 0.f);
            if (D > 64) op[lane + 64] = (uint16_t)pack2<F16>(ro[1] * rinv, 0.f);
        } else {
            float* po = p.part_o + (split * prows + (((long)b * p.Hk + hk) * p.row_tiles + rt) * 32 + w * 8 + (src >> 3)) * D;
            if (lane < D) po[lane] = ro[0];
            if (D > 64) po[lane + 64] = ro[1];
        }
    }
}

// joins the splits of a row in split order: D / 4 threads a row
template <int D, bool F16>
__global__ __launch_bounds__(256) void span_attn_join(const SpanArgs p) {
    constexpr int TPR = D / 4, JOIN = 8;
    const long rows = (long)p.B * p.Hk * p.row_tiles * 32;
    const long r = (long)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
    const int c = threadIdx.x % TPR;
    if (r >= rows) return;
    const int group = p.Hq / p.Hk;
    const int in_head = (int)(r % (p.row_tiles * 32));
    if (in_head >= group * p.nq) return;
    const int hk = (int)(r / (p.row_tiles * 32)) % p.Hk, b = (int)(r / (p.row_tiles * 32) / p.Hk);
    const int h = hk * group + in_head / p.nq, i = in_head % p.nq;
    float M = SPAN_LOW, L = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = 0; s0 < p.splits; s0 += JOIN) {      // JOIN splits' reads go out together (one by one, each waits for the one before: 8 us for 8 splits of 64 x 4 rows, 5 so)
        float2 ml[JOIN];
        float4 y[JOIN];
#pragma unroll
        for (int x = 0; x < JOIN; ++x) {
            const long at = min(s0 + x, p.splits - 1) * rows + r;
            ml[x] = *reinterpret_cast<const float2*>(p.part_ml + at * 2);
            y[x] = *reinterpret_cast<const float4*>(p.part_o + at * D + c * 4);
        }
        float mn = M;
#pragma unroll
        for (int x = 0; x < JOIN; ++x) mn = fmaxf(mn, ml[x].x);
        float f = __builtin_amdgcn_exp2f(M - mn);
        M = mn;
        L *= f;
        v.x *= f; v.y *= f; v.z *= f; v.w *= f;
#pragma unroll
        for (int x = 0; x < JOIN; ++x) {
            if (s0 + x >= p.splits) break;
            f = __builtin_amdgcn_exp2f(ml[x].x - M);
            L = __builtin_fmaf(ml[x].y, f, L);
            v.x = __builtin_fmaf(y[x].x, f, v.x); v.y = __builtin_fmaf(y[x].y, f, v.y); v.z = __builtin_fmaf(y[x].z, f, v.z); v.w = __builtin_fmaf(y[x].w, f, v.w);
        }
    }
    const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
    *reinterpret_cast<uint2*>(p.out + b * p.o_s[0] + h * p.o_s[1] + (long)i * p.o_s[2] + c * 4) =
        make_uint2(pack2<F16>(v.x * inv, v.y * inv), pack2<F16>(v.z * inv, v.w * inv));
    if (p.lse && c == 0) p.lse[((long)b * p.Hq + h) * p.nq + i] = row_lse<F16>(M, L);
}

__global__ __launch_bounds__(1024) void span_order(const int32_t* __restrict__ spans, long sb, int B, int n, int nk, int32_t* __restrict__ order) {
    __shared__ SpanOrderLds m;
    span_order_tiles<1024>(m, spans, sb, B, n, nk, order);
}

struct SpanPlan { bool narrow; int row_tiles, splits; };

// The narrow form where the wide one would leave CUs without a workgroup (< 256 of them) or most of a workgroup's 128 rows empty (up to 32 queries: 16 new positions
// over caches of 16384 keys, 16 / 4 heads of 128: 505 us wide, 99 narrow).  There the keys are split for one to four rounds of the workgroups that the card holds (one a CU
// 128 wide, two narrower: their LDS), at least 256 keys each (two tiles a wave), whichever is least in keys a workgroup passes over, its start and the join counted as 512 each.
// (8 heads of 1089 x 1089, 128 wide: 32 us whole, 37 in two splits and a round more; 8 key heads of 60000 keys, one position: 55 us in one round, 64 in two; 130 positions
// of 2 x 16 / 4 heads over 5000 keys: 47 in three splits, two rounds, 52 whole on half the CUs)
SpanPlan span_plan(const mm_span_attn* a) {
    SpanPlan r;
    const long wide = (long)a->batch * a->heads_q * ((a->nq + WQ - 1) / WQ);
    const long rows = (long)(a->heads_q / a->heads_k) * a->nq;
    r.row_tiles = (int)((rows + 31) / 32);
    r.narrow = wide < 256 || a->nq <= 32;
    r.splits = 1;
    if (!r.narrow) return r;
    const long wgs = (long)a->batch * a->heads_k * r.row_tiles, slots = a->dim == 128 ? 256 : 512, most = (a->nk + 255) / 256;
    const auto cost = [&](long s) { return (wgs * s + slots - 1) / slots * ((a->nk + s - 1) / s + 512) + (s > 1 ? 512 : 0); };
    for (long rounds = 1; rounds <= 4; ++rounds) {
        const long s = rounds * slots / wgs < most ? rounds * slots / wgs : most;
        if (s > 1 && cost(s) < cost(r.splits)) r.splits = (int)s;
    }
    return r;
}

template <int D, bool F16, int AX, bool CAP>
int launch_fwd(hipStream_t s, const SpanArgs& a, const SpanPlan& pl) {
    if (!pl.narrow) {
        constexpr int sm = 2 * (2 * Tile<D, KT>::BYTES + AX * KT * 4) + 64;
        static std::atomic<unsigned long long> lds{0};
        if (const int rc = span_allow_lds(reinterpret_cast<const void*>(span_attn_wide<D, F16, AX, CAP>), sm, lds)) return rc;
        hipLaunchKernelGGL((span_attn_wide<D, F16, AX, CAP>), dim3((unsigned)(a.B * a.Hq * ((a.nq + WQ - 1) / WQ))), dim3(256), sm, s, a);
        return mm_check_launch("span_attn_wide");
    }
    constexpr int st = 8 * (2 * Tile<D, 32>::BYTES + AX * 32 * 4), jo = 4 * 32 * (D + 4) * 4;
    constexpr int sm = (st > jo ? st : jo) + 4 * 32 * 2 * 4;
    static std::atomic<unsigned long long> lds{0};
    if (const int rc = span_allow_lds(reinterpret_cast<const void*>(span_attn_narrow<D, F16, AX, CAP>), sm, lds)) return rc;
    hipLaunchKernelGGL((span_attn_narrow<D, F16, AX, CAP>), dim3((unsigned)(a.B * a.Hk * pl.row_tiles), pl.splits), dim3(256), sm, s, a);
    const int rc = mm_check_launch("span_attn_narrow");
    if (rc || pl.splits == 1) return rc;
    const long rows = (long)a.B * a.Hk * pl.row_tiles * 32, blocks = (rows + 256 / (D / 4) - 1) / (256 / (D / 4));
    hipLaunchKernelGGL((span_attn_join<D, F16>), dim3((unsigned)blocks), dim3(256), 0, s, a);
    return mm_check_launch("span_attn_join");
}

template <int D, bool F16, bool CAP>
int launch_axes(hipStream_t s, const SpanArgs& a, const SpanPlan& pl) {
    switch (a.axes) {
        case 0: return launch_fwd<D, F16, 0, CAP>(s, a, pl);
        case 1: return launch_fwd<D, F16, 1, CAP>(s, a, pl);
        case 2: return launch_fwd<D, F16, 2, CAP>(s, a, pl);
        default: return launch_fwd<D, F16, 3, CAP>(s, a, pl);
    }
}
template <int D>
int launch_dim(hipStream_t s, const SpanArgs& a, const SpanPlan& pl, bool f16) {
    if (a.cap > 0.f) return f16 ? launch_axes<D, true, true>(s, a, pl) : launch_axes<D, false, true>(s, a, pl);
    return f16 ? launch_axes<D, true, false>(s, a, pl) : launch_axes<D, false, false>(s, a, pl);
}

}  // namespace

void span_args(const mm_span_attn* a, SpanArgs& p) {
    memset(&p, 0, sizeof(p));
    p.q = (const uint16_t*)a->q; p.k = (const uint16_t*)a->k; p.v = (const uint16_t*)a->v; p.out = (uint16_t*)a->out; p.lse = a->lse;
    p.spans = a->spans; p.spans_sb = a->spans_sb; p.kmask = a->key_mask; p.km_sb = a->key_mask_sb;
    p.slopes = a->slopes; p.pos_q = a->positions_q; p.pq_sb = a->positions_q_sb; p.pos_k = a->positions_k; p.pk_sb = a->positions_k_sb;
    for (int i = 0; i < 3; ++i) {
        p.q_s[i] = a->q_stride[i]; p.k_s[i] = a->k_stride[i]; p.v_s[i] = a->v_stride[i]; p.o_s[i] = a->out_stride[i];
        p.do_s[i] = a->dout_stride[i]; p.dq_s[i] = a->dq_stride[i]; p.dk_s[i] = a->dk_stride[i]; p.dv_s[i] = a->dv_stride[i];
    }
    if (a->nk == 1) p.k_s[2] = p.v_s[2] = a->dim;      // (one key: its stride says nothing)
    p.B = a->batch; p.Hq = a->heads_q; p.Hk = a->heads_k; p.nq = a->nq; p.nk = a->nk; p.axes = a->slopes ? a->axes : 0;
    p.scale = a->scale; p.cap = a->softcap;
    p.dout = (const uint16_t*)a->dout; p.dq = (uint16_t*)a->dq; p.dk = (uint16_t*)a->dk; p.dv = (uint16_t*)a->dv;
}

size_t k_span_attn_workspace_bytes(const mm_span_attn* a) {
    const SpanPlan pl = span_plan(a);
    if (!pl.narrow) return (size_t)span_order_count(a) * sizeof(int32_t);
    if (pl.splits == 1) return 0;
    return (size_t)pl.splits * a->batch * a->heads_k * pl.row_tiles * 32 * (a->dim + 2) * sizeof(float);
}

int k_span_attn(hipStream_t s, const mm_span_attn* a, void* ws) {
    SpanArgs p;
    span_args(a, p);
    const SpanPlan pl = span_plan(a);
    p.splits = pl.splits; p.row_tiles = pl.row_tiles;
    if (!pl.narrow && span_order_count(a)) {
        hipLaunchKernelGGL(span_order, dim3(1), dim3(1024), 0, s, a->spans, a->spans_sb, a->batch, a->nq, a->nk, (int32_t*)ws);
        if (const int rc = mm_check_launch("span_order")) return rc;
        p.order = (const int32_t*)ws;
    }
    p.part_o = (float*)ws;
    p.part_ml = p.part_o ? p.part_o + (size_t)pl.splits * a->batch * a->heads_k * pl.row_tiles * 32 * a->dim : nullptr;
    const bool f16 = a->dtype == MM_DT_F16;
    if (a->dim == 32) return launch_dim<32>(s, p, pl, f16);
    if (a->dim == 64) return launch_dim<64>(s, p, pl, f16);
    return launch_dim<128>(s, p, pl, f16);
}
