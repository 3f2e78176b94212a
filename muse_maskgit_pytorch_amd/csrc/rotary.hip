// Positions and masks of packed rows (documents = images of several sizes, with or without their text, one behind another):
//   attention_spans : per query row the interval [lo, hi) of keys it sees, from document bounds, causal order and prefix lengths
//   rotary_axes     : rotary positions over up to four axes (time / height / width ...), with or without l2norm * scale in front (mmp.py:151-153), and the gradient
#include <string.h>

#include "common.h"
#include "muse_hip_internal.h"

namespace {

// ------------------------------------------------------------------------------------------------ spans
// Row i belongs to the last document with cu_q[doc] <= i (empty documents are passed over); rows in front of the first or behind the last document see nothing.
// One thread per row, the bounds in LDS (a binary search is log2(docs) DEPENDENT reads: 64 cycles each there, an L2 round trip each from memory).  Bounded by
// latency: 310 rows and 131000 rows take about the same time.
constexpr int SPAN_LDS_DOCS = 4096;

__global__ __launch_bounds__(256) void attention_spans_kernel(const int32_t* __restrict__ cu_q, long q_sb, const int32_t* __restrict__ cu_k, long k_sb,
                                                              const int32_t* __restrict__ prefix, long p_sb, int docs, int n, int j, int causal, int2* __restrict__ out) {
    __shared__ int32_t cu[SPAN_LDS_DOCS + 1];
    const int b = blockIdx.y;
    const int32_t* cq = cu_q + b * q_sb;
    const int32_t* ck = cu_k + b * k_sb;
    const bool in_lds = docs <= SPAN_LDS_DOCS;
    if (in_lds) {
        for (int t = threadIdx.x; t <= docs; t += 256) cu[t] = cq[t];
        __syncthreads();
    }
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    int a = 0, e = docs + 1;      // number of bounds <= i
    while (a < e) {
        const int m = (a + e) >> 1;
        const int v = in_lds ? cu[m] : cq[m];
        if (v <= i) a = m + 1;
        else e = m;
    }
    int2 r = make_int2(0, 0);
    const int doc = a - 1;
    if (doc >= 0 && doc < docs) {
        // by the document's own lengths, in 64 bits (bounds may be any int32); what lies outside the j keys is cut off at the end: cut first, a document that goes on
        // behind the row would lose keys but no queries, and its causal diagonal would move
        const long k0 = ck[doc], lk = max((long)ck[doc + 1] - k0, 0L);
        long seen = lk;
        if (causal) {
            seen = i + 1 + lk - cq[doc + 1];      // the last row of a document sees all of its keys
            if (prefix) seen = max(seen, (long)prefix[b * p_sb + doc]);
            seen = min(max(seen, 0L), lk);
        }
        r = make_int2((int)min(max(k0, 0L), (long)j), (int)min(max(k0 + seen, 0L), (long)j));
    }
    out[(long)b * n + i] = r;
}

// ------------------------------------------------------------------------------------------------ rotary positions
// Pair p of a head (p < P = sum of the sections) belongs to axis a(p) and turns by the angle  pos_a * freq_p:   a' = a cos - b sin,  b' = a sin + b cos,  with
// (a, b) = elements (p, P + p), or (2p, 2p + 1) interleaved; elements from 2P on pass.  The gradient turns back.  The angle is formed in 64 bits and reduced to one
// turn there (far positions: an fp32 product is 0.03 rad off at position 10^6), then sin / cos in fp32.
// HBM-bound: one read + one write of every element (the backward with the norm reads two).  A workgroup takes TB tokens: first their turns into LDS, one pair a thread
// (the 64-bit products and sincospif of eight pairs side by side in a lane take 130 registers, and the loads need the occupancy), then their heads, G lanes a head, VEC
// pairs a lane.
struct RotT {      // one of q / k
    const void* x; long x_sb, x_sh, x_sn;      // forward: the input; backward: the forward's input (NORM only)
    const void* dy; long d_sb, d_sh, d_sn;     // backward: the gradient of the output
    void* out;                                 // [B][n][H][d] contiguous
    const float* scale;                        // fp32 [d]
    int H;
};
struct RotArgs {
    RotT t[2];
    const int32_t* pos; long pos_sb; int A;
    const double* freq;
    int P, c1, c2, c3;                         // axis of pair p = (p >= c1) + (p >= c2) + (p >= c3)
    int B, n, d, G, TB, interleaved;
    float* part;                               // backward with the norm: [gridDim.x][2][d]
};

template <typename T> __device__ __forceinline__ float rot_ld(T v);
template <> __device__ __forceinline__ float rot_ld<float>(float v) { return v; }
template <> __device__ __forceinline__ float rot_ld<_Float16>(_Float16 v) { return (float)v; }
template <> __device__ __forceinline__ float rot_ld<__bf16>(__bf16 v) { return (float)v; }

template <typename T, int VEC> struct alignas(sizeof(T) * VEC > 16 ? 16 : sizeof(T) * VEC) RotVec { T v[VEC]; };

template <typename T, int VEC>
__device__ __forceinline__ void rot_store(T* p, const float (&f)[VEC]) {
    RotVec<T, VEC> r;
#pragma unroll
    for (int e = 0; e < VEC; ++e) r.v[e] = (T)f[e];
    *reinterpret_cast<RotVec<T, VEC>*>(p) = r;
}

// the lane's pairs from `turned` on lie behind the P that turn: they pass as they are (a turn by 0 would not do: 0 times a neighbour's infinity is NaN)
template <int VEC, bool INTER>
__device__ __forceinline__ void rot_turn(float (&a)[VEC], float (&b)[VEC], const float (&c)[VEC], const float (&s)[VEC], int turned) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        // interleaved: the unit's 2 VEC consecutive elements hold its VEC pairs, (a0 a1) (a2 a3) .. (b0 b1) ..
        constexpr bool beside = INTER && VEC > 1;
        float& x_ = !beside ? a[e] : (2 * e < VEC ? a[(2 * e) % VEC] : b[(2 * e) % VEC]);
        float& y_ = !beside ? b[e] : (2 * e < VEC ? a[(2 * e + 1) % VEC] : b[(2 * e + 1) % VEC]);
        const float x = x_, y = y_;
        const bool on = (beside ? e : 0) < turned;
        x_ = on ? __builtin_fmaf(x, c[e], -(y * s[e])) : x;
        y_ = on ? __builtin_fmaf(x, s[e], y * c[e]) : y;
    }
}

__device__ __forceinline__ float rot_group_sum(float v, int G) {
    for (int o = G >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

constexpr int ROT_TURNS = 2048;      // (cos, sin) pairs a workgroup holds: ROT_TURNS / (d / 2) tokens at most

template <typename T, int VEC, bool NORM, bool BWD, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(const RotArgs p) {
    constexpr int HB = VEC == 8 && !(NORM && BWD) ? 2 : 1;      // heads whose loads go out together
    __shared__ __attribute__((aligned(16))) float2 turns[ROT_TURNS];
    const int G = p.G, u = threadIdx.x & (G - 1), slots = 256 / G, slot = threadIdx.x / G, pairs = p.d / 2;
    const bool live = u < p.d / (2 * VEC);
    const int turned = p.P - u * VEC;      // how many of the lane's pairs turn (none or all of them unless interleaved)
    int offa, offb;
    if (INTER) { offa = 2 * VEC * u; offb = offa + VEC; }
    else if (u * VEC < p.P) { offa = u * VEC; offb = p.P + u * VEC; }
    else { offa = 2 * p.P + 2 * (u * VEC - p.P); offb = offa + VEC; }
    const long tokens = (long)p.B * p.n;
#pragma unroll
    for (int w = 0; w < 2; ++w) {      // q, then k
        const RotT& t = p.t[w];
        float acc[2][VEC];             // backward with the norm: gradient of the scale
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[0][e] = acc[1][e] = 0.f;
        for (long tok0 = (long)blockIdx.x * p.TB; tok0 < tokens && t.H > 0; tok0 += (long)gridDim.x * p.TB) {
            const int here = (int)min((long)p.TB, tokens - tok0);
            if (w == 0 || p.t[0].H == 0 || (long)gridDim.x * p.TB < tokens) {      // (one group of tokens: k finds q's turns)
                __syncthreads();
#pragma nounroll
                for (int x = threadIdx.x; x < here * pairs; x += 256) {
                    const long tk = tok0 + x / pairs;
                    const int pr = x % pairs;
                    float2 cs = make_float2(1.f, 0.f);
                    if (pr < p.P) {
                        const int ax = (pr >= p.c1) + (pr >= p.c2) + (pr >= p.c3);
                        const double turn = (double)p.pos[tk / p.n * p.pos_sb + tk % p.n * p.A + ax] * p.freq[pr] * 0.15915494309189533577;      // / (2 pi)
                        sincospif((float)(2.0 * (turn - rint(turn))), &cs.y, &cs.x);
                        if (BWD) cs.y = -cs.y;
                    }
                    turns[x] = cs;
                }
                __syncthreads();
            }
            float sa[VEC], sb[VEC];
            if constexpr (NORM) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) { sa[e] = live ? t.scale[offa + e] : 0.f; sb[e] = live ? t.scale[offb + e] : 0.f; }
            }
            // heads of one token beside each other in the workgroup: its reads and writes are whole rows, token after token
            const int all = here * t.H, qt = slots / t.H, rh = slots % t.H;
            int tk = slot / t.H, h = slot % t.H;
#pragma nounroll
            for (int v0 = 0; v0 < all; v0 += slots * HB) {
                RotVec<T, VEC> rx[HB][2], rd[HB][2];
                int ti[HB], hi[HB];
#pragma unroll
                for (int y = 0; y < HB; ++y) {
                    const bool ok = live && v0 + y * slots + slot < all;
                    ti[y] = ok ? tk : -1; hi[y] = h;
                    if (ok) {
                        const long token = tok0 + tk;
                        const int b = (int)(token / p.n), i = (int)(token - (long)b * p.n);
                        if constexpr (!BWD || NORM) {
                            const T* xp = reinterpret_cast<const T*>(t.x) + b * t.x_sb + (long)h * t.x_sh + (long)i * t.x_sn;
                            rx[y][0] = *reinterpret_cast<const RotVec<T, VEC>*>(xp + offa); rx[y][1] = *reinterpret_cast<const RotVec<T, VEC>*>(xp + offb);
                        }
                        if constexpr (BWD) {
                            const T* dp = reinterpret_cast<const T*>(t.dy) + b * t.d_sb + (long)h * t.d_sh + (long)i * t.d_sn;
                            rd[y][0] = *reinterpret_cast<const RotVec<T, VEC>*>(dp + offa); rd[y][1] = *reinterpret_cast<const RotVec<T, VEC>*>(dp + offb);
                        }
                    }
                    h += rh; tk += qt;
                    if (h >= t.H) { h -= t.H; ++tk; }
                }
#pragma unroll
                for (int y = 0; y < HB; ++y) {
                    const bool ok = ti[y] >= 0;
                    float xa[VEC], xb[VEC], ga[VEC], gb[VEC], c[VEC], s[VEC];
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        xa[e] = xb[e] = ga[e] = gb[e] = 0.f;
                        const float2 cs = ok ? turns[ti[y] * pairs + u * VEC + e] : make_float2(1.f, 0.f);
                        c[e] = cs.x; s[e] = cs.y;
                        if (ok) {
                            if constexpr (!BWD || NORM) { xa[e] = rot_ld<T>(rx[y][0].v[e]); xb[e] = rot_ld<T>(rx[y][1].v[e]); }
                            if constexpr (BWD) { ga[e] = rot_ld<T>(rd[y][0].v[e]); gb[e] = rot_ld<T>(rd[y][1].v[e]); }
                        }
                    }
                    float inv = 1.f;
                    bool below = false;      // the row is divided by the constant, whose derivative is 0: no projection in its gradient
                    if constexpr (NORM) {
                        float ss = 0.f;
#pragma unroll
                        for (int e = 0; e < VEC; ++e) ss = __builtin_fmaf(xa[e], xa[e], __builtin_fmaf(xb[e], xb[e], ss));
                        ss = rot_group_sum(ss, G);
                        const float len = sqrtf(ss);
                        below = len < 1e-12f;
                        inv = 1.f / fmaxf(len, 1e-12f);      // F.normalize eps (mmp.py:41-42)
                    }
                    if constexpr (!BWD) {
                        if constexpr (NORM) {
#pragma unroll
                            for (int e = 0; e < VEC; ++e) { xa[e] = xa[e] * inv * sa[e]; xb[e] = xb[e] * inv * sb[e]; }
                        }
                        rot_turn<VEC, INTER>(xa, xb, c, s, turned);
                    } else {
                        rot_turn<VEC, INTER>(ga, gb, c, s, turned);
                        if constexpr (NORM) {
                            float dot = 0.f;
#pragma unroll
                            for (int e = 0; e < VEC; ++e) {
                                xa[e] *= inv; xb[e] *= inv;
                                acc[0][e] = __builtin_fmaf(ga[e], xa[e], acc[0][e]);
                                acc[1][e] = __builtin_fmaf(gb[e], xb[e], acc[1][e]);
                                ga[e] *= sa[e]; gb[e] *= sb[e];
                                dot = __builtin_fmaf(xa[e], ga[e], __builtin_fmaf(xb[e], gb[e], dot));
                            }
                            dot = rot_group_sum(dot, G);
                            if (below) dot = 0.f;
#pragma unroll
                            for (int e = 0; e < VEC; ++e) { xa[e] = __builtin_fmaf(-xa[e], dot, ga[e]) * inv; xb[e] = __builtin_fmaf(-xb[e], dot, gb[e]) * inv; }
                        } else {
#pragma unroll
                            for (int e = 0; e < VEC; ++e) { xa[e] = ga[e]; xb[e] = gb[e]; }
                        }
                    }
                    if (ok) {
                        T* op = reinterpret_cast<T*>(t.out) + ((tok0 + ti[y]) * t.H + hi[y]) * p.d;
                        rot_store<T, VEC>(op + offa, xa); rot_store<T, VEC>(op + offb, xb);
                    }
                }
            }
        }
        if constexpr (NORM && BWD) {      // the workgroup's part of the scale's gradient: its slots added in order
            extern __shared__ float sm[];      // [slots][d]
            if (w == 1) __syncthreads();
            if (live) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) { sm[slot * p.d + offa + e] = acc[0][e]; sm[slot * p.d + offb + e] = acc[1][e]; }
            }
            __syncthreads();
            float* part = p.part + ((long)blockIdx.x * 2 + w) * p.d;
            for (int col = threadIdx.x; col < p.d; col += 256) {
                float v = 0.f;
                for (int sl = 0; sl < slots; ++sl) v += sm[sl * p.d + col];
                part[col] = v;
            }
        }
    }
}

struct RotPlan { int vec, G, TB, gx; };

// VEC = 8 where rows and pairs allow 16-byte accesses, else one pair per lane.  Tokens a workgroup: as many as leave four workgroups a CU, two where each has parts of the
// scales' gradients to add up (32 x 1024 tokens, 16 heads of 64, forward: 36 us with two and 31 with four; gradient behind the norm: 53 and 59); one for a step of a
// decoder, at most what the turns have room for.  Up to 2048 workgroups, which then take several such groups.
RotPlan rot_plan(int B, int n, int d, int vec, bool sums) {
    RotPlan r;
    r.vec = vec;
    int g = 1;
    while (g < d / (2 * vec)) g *= 2;
    r.G = g;
    const long tokens = (long)B * n;
    const long most = ROT_TURNS / (d / 2), tb = tokens / (sums ? 512 : 1024);
    r.TB = (int)(tb < 1 ? 1 : (tb > most ? most : tb));
    const long blocks = (tokens + r.TB - 1) / r.TB;
    r.gx = (int)(blocks < 2048 ? blocks : 2048);
    return r;
}

template <typename T, int VEC, bool INTER>
void rot_launch_pairs(hipStream_t s, const RotArgs& a, const RotPlan& pl, bool norm, bool bwd) {
    const dim3 g(pl.gx), blk(256);
    const size_t sm = norm && bwd ? (size_t)(256 / pl.G) * a.d * sizeof(float) : 0;
    if (norm && bwd) hipLaunchKernelGGL((rotary_kernel<T, VEC, true, true, INTER>), g, blk, sm, s, a);
    else if (bwd) hipLaunchKernelGGL((rotary_kernel<T, VEC, false, true, INTER>), g, blk, 0, s, a);
    else if (norm) hipLaunchKernelGGL((rotary_kernel<T, VEC, true, false, INTER>), g, blk, 0, s, a);
    else hipLaunchKernelGGL((rotary_kernel<T, VEC, false, false, INTER>), g, blk, 0, s, a);
}
template <typename T, int VEC>
void rot_launch(hipStream_t s, const RotArgs& a, const RotPlan& pl, bool norm, bool bwd) {
    if (a.interleaved) rot_launch_pairs<T, VEC, true>(s, a, pl, norm, bwd);
    else rot_launch_pairs<T, VEC, false>(s, a, pl, norm, bwd);
}

bool rot_wide(const mm_rotary* r) {
    int P = 0;
    for (int a = 0; a < r->axes; ++a) P += r->sections[a];
    const int per16 = r->dtype == MM_DT_F32 ? 4 : 8;
    if (r->dim % 16 || (!r->interleaved && (P % 8 || (r->dim - 2 * P) % 16))) return false;
    for (int w = 0; w < 2; ++w) {
        const mm_rotary_side* t = w ? &r->k : &r->q;
        if (t->heads == 0) continue;
        if (((uintptr_t)t->x | (uintptr_t)t->dy | (uintptr_t)t->out) & 15) return false;
        const int size[3] = {r->batch, t->heads, r->n};      // (a dimension of one element has no stride)
        for (int i = 0; i < 3; ++i)
            if (size[i] > 1 && ((t->x && t->x_stride[i] % per16) || (t->dy && t->dy_stride[i] % per16))) return false;
    }
    return true;
}

}  // namespace

int k_attention_spans(hipStream_t s, const int32_t* cu_q, long q_sb, const int32_t* cu_k, long k_sb, const int32_t* prefix, long p_sb, int B, int docs, int n, int j,
                      int causal, int32_t* out) {
    if (B == 0 || n == 0) return MM_OK;
    hipLaunchKernelGGL(attention_spans_kernel, dim3((n + 255) / 256, B), dim3(256), 0, s, cu_q, q_sb, cu_k, k_sb, prefix, p_sb, docs, n, j, causal, reinterpret_cast<int2*>(out));
    return mm_check_launch("attention_spans_kernel");
}

// rows [2 dim] of the scales' partial gradients; -1: a head too long for one pair per lane (64 lanes) whose rows do not allow 16-byte accesses
long k_rotary_parts(const mm_rotary* r) {
    if (r->dim > 128 && !rot_wide(r)) return -1;
    const RotPlan pl = rot_plan(r->batch, r->n, r->dim, rot_wide(r) ? 8 : 1, true);
    return pl.gx;
}

int k_rotary(hipStream_t s, const mm_rotary* r, bool bwd, float* ws, float* dscales) {
    RotArgs a;
    memset(&a, 0, sizeof(a));
    for (int w = 0; w < 2; ++w) {
        const mm_rotary_side* t = w ? &r->k : &r->q;
        a.t[w].x = t->x; a.t[w].x_sb = t->x_stride[0]; a.t[w].x_sh = t->x_stride[1]; a.t[w].x_sn = t->x_stride[2];
        a.t[w].dy = t->dy; a.t[w].d_sb = t->dy_stride[0]; a.t[w].d_sh = t->dy_stride[1]; a.t[w].d_sn = t->dy_stride[2];
        a.t[w].out = t->out; a.t[w].scale = t->scale; a.t[w].H = t->heads;
    }
    a.pos = r->positions; a.pos_sb = r->pos_sb; a.A = r->axes; a.freq = r->freqs;
    int cum[4] = {0, 0, 0, 0}, P = 0;
    for (int i = 0; i < r->axes; ++i) { P += r->sections[i]; cum[i] = P; }
    for (int i = r->axes; i < 4; ++i) cum[i] = P;
    a.P = P; a.c1 = cum[0]; a.c2 = cum[1]; a.c3 = cum[2];
    a.B = r->batch; a.n = r->n; a.d = r->dim; a.interleaved = r->interleaved;
    const bool wide = rot_wide(r);
    const bool norm = r->normalize != 0;
    const RotPlan pl = rot_plan(r->batch, r->n, r->dim, wide ? 8 : 1, norm && bwd);
    a.G = pl.G; a.TB = pl.TB; a.part = ws;
    const bool any = pl.gx > 0 && r->q.heads + r->k.heads > 0;
    if (any) {
        if (r->dtype == MM_DT_F32) { if (wide) rot_launch<float, 8>(s, a, pl, norm, bwd); else rot_launch<float, 1>(s, a, pl, norm, bwd); }
        else if (r->dtype == MM_DT_F16) { if (wide) rot_launch<_Float16, 8>(s, a, pl, norm, bwd); else rot_launch<_Float16, 1>(s, a, pl, norm, bwd); }
        else { if (wide) rot_launch<__bf16, 8>(s, a, pl, norm, bwd); else rot_launch<__bf16, 1>(s, a, pl, norm, bwd); }
        const int rc = mm_check_launch("rotary_kernel");
        if (rc) return rc;
    }
    return norm && bwd ? k_colsum(s, ws, any ? pl.gx : 0, 2 * r->dim, dscales) : MM_OK;      // (no rows or no heads: zeros)
}
