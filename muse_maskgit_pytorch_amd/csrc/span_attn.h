// Shared by the forward and the backward of the packed-row attention (attention_spans.hip, attention_spans_bwd.hip): arguments, tiles in LDS, masks, scores.
#pragma once
#include <atomic>

#include "common.h"
#include "muse_hip_internal.h"

struct SpanArgs {
    const uint16_t *q, *k, *v;
    uint16_t* out;
    float* lse;
    const int32_t* spans; long spans_sb;
    const uint8_t* kmask; long km_sb;
    const float* slopes;
    const int32_t *pos_q, *pos_k; long pq_sb, pk_sb;
    long q_s[3], k_s[3], v_s[3], o_s[3];
    int B, Hq, Hk, nq, nk, axes;
    float scale, cap;
    const int32_t* order;      // [B * tiles] tiles of 128 rows, the longest first (NULL: as they come, last first)
    // forward, keys split over workgroups
    int splits, row_tiles; float* part_o; float* part_ml;
    // backward
    const uint16_t* dout; long do_s[3];
    uint16_t *dq, *dk, *dv; long dq_s[3], dk_s[3], dv_s[3];
    float* delta; float* dsl_part; float* dslopes; unsigned* done; int* seen; int4* hulls; int hull_tiles; int32_t* order_out;
};

namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short sp_v4i16_t __attribute__((ext_vector_type(4)));
// reads of LDS beside a DMA in flight: through native vectors.  HIP's int4 / float4 carry no alias information, and without any the compiler waits for every DMA first
typedef int i32x4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ i32x4_t lds_i4(const void* p) { return *reinterpret_cast<const i32x4_t*>(p); }
__device__ __forceinline__ f32x4_t lds_f4(const void* p) { return *reinterpret_cast<const f32x4_t*>(p); }

constexpr float SPAN_LOG2E = 1.4426950408889634f, SPAN_LN2 = 0.6931471805599453f;
constexpr float SPAN_LOW = -1.0e30f;      // start of a running maximum: finite, so that a masked score (-inf) minus it is -inf, not NaN

// v_mfma_f32_32x32x16: A lane l holds row l & 31, contraction 8 (l >> 5) .. + 7; B the same with columns; C lane l holds column l & 31, rows 8 (r >> 2) + 4 (l >> 5)
// + (r & 3).  A C fragment's registers 8 s .. 8 s + 7 are therefore a B operand over 16 of its rows, in the order (slot j of half h) = row 16 s + 8 (j >> 2) + 4 h +
// (j & 3) -- the order in which two transposing LDS reads deliver the other operand.  No value crosses lanes between the two products.
template <bool F16>
__device__ __forceinline__ f32x16_t mfma32(u32x4_t a, u32x4_t b, f32x16_t c) {
    if constexpr (F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
template <bool F16> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (F16) return (uint32_t)f32_to_f16_bits(a) | ((uint32_t)f32_to_f16_bits(b) << 16);
    else return pack_bf16x2(a, b);
}
template <bool F16> __device__ __forceinline__ float to_f32(uint16_t v) {
    if constexpr (F16) return f16_bits_to_f32(v);
    else return bf16_to_f32(v);
}
template <bool F16> __device__ __forceinline__ u32x4_t pack_slots(const f32x16_t& c, int s) {      // (s: a constant after unrolling)
    return u32x4_t{pack2<F16>(c[8 * s], c[8 * s + 1]), pack2<F16>(c[8 * s + 2], c[8 * s + 3]), pack2<F16>(c[8 * s + 4], c[8 * s + 5]), pack2<F16>(c[8 * s + 6], c[8 * s + 7])};
}
__device__ __forceinline__ float both_halves_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float both_halves_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// ds_read_b64_tr_b16.  __restrict__: the access gets alias information of its own; without any the compiler takes every LDS-DMA in flight (the NEXT tile's, into the
// other stage) for a write to it and waits for all of them in the middle of a tile (s_waitcnt vmcnt(0)).  The kernels wait for a tile themselves, before its barrier.
__device__ __forceinline__ sp_v4i16_t tr_read(const unsigned char* __restrict__ p) {
    typedef __attribute__((address_space(3))) sp_v4i16_t* lds_v4_t;
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4_t)p);
}

// A tile of ROWS rows x D elements in LDS as [D / 16][ROWS][16] (32-byte rows; 128 bytes between blocks keep the two column blocks of a transposing read on
// different banks).  ONE image serves both operand forms: rows as they are (ds_read_b128: the wave reads 1 KiB in a row) and transposed (ds_read_b64_tr_b16).  Filled
// by LDS-DMA, 32 rows x 16 columns per wave instruction; rows at or behind rows_ok are outside the descriptor and come as zeros.
template <int D, int ROWS>
struct Tile {
    static constexpr int NB = D / 16, BS = ROWS * 32 + 128, BYTES = NB * BS;
    template <int NW>      // waves that share the work, this one being w
    static __device__ __forceinline__ void fill(unsigned char* lds, const uint16_t* base, int rows_ok, int stride, int w, int lane) {
        typedef __attribute__((address_space(3))) void* lds_ptr_t;
        const int sb = stride * 2;
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(base), 0, rows_ok > 0 ? (unsigned)((rows_ok - 1) * sb + D * 2) : 0u, 0x00020000);
        const int v0 = (lane >> 1) * sb + (lane & 1) * 16;
#pragma unroll
        for (int i = 0; i < NB * (ROWS / 32) / NW; ++i) {
            const int idx = i * NW + w, cb = idx % NB, rb = idx / NB;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr_t)(lds + cb * BS + rb * 1024), 16, v0, rb * 32 * sb + cb * 32, 0, 0);
        }
    }
    // operand over columns 16 cb .. + 15, rows 32 rb .. + 31
    static __device__ __forceinline__ u32x4_t rows(const unsigned char* lds, int cb, int rb, int lane) {
        return *reinterpret_cast<const u32x4_t*>(lds + cb * BS + (rb * 32 + (lane & 31)) * 32 + (lane >> 5) * 16);
    }
    // operand over rows 16 s .. + 15 (in the slot order above), columns 32 cd .. + 31
    static __device__ __forceinline__ u32x4_t cols(const unsigned char* lds, int s, int cd, int lane) {
        const unsigned char* p = lds + (2 * cd + ((lane >> 4) & 1)) * BS + (s * 16 + (lane >> 5) * 4 + ((lane & 15) >> 2)) * 32 + (lane & 3) * 8;
        const uint2 x = __builtin_bit_cast(uint2, tr_read(p)), y = __builtin_bit_cast(uint2, tr_read(p + 256));
        return u32x4_t{x.x, x.y, y.x, y.y};
    }
    // rows whose bit is clear become zeros (all threads of the workgroup; the caller's barriers)
    static __device__ __forceinline__ void clear_rows(unsigned char* lds, unsigned long long keep, int t, int threads) {
        for (int c = t; c < NB * ROWS * 2; c += threads) {
            const int row = (c >> 1) % ROWS;
            if (!((keep >> row) & 1ull)) *reinterpret_cast<u32x4_t*>(lds + (c / (2 * ROWS)) * BS + row * 32 + (c & 1) * 16) = u32x4_t{0, 0, 0, 0};
        }
    }
};

// Which (tile, head) a workgroup takes.  Workgroups go to the 8 XCDs in turn: with a multiple of 8 heads each XCD keeps its own heads (their keys are read into one
// L2), neighbours among them; otherwise heads in turn.  Tiles in the order of `order`, heads innermost, so the long ones of every head start first.
__device__ __forceinline__ bool span_item(unsigned id, const int32_t* order, int heads, int rows, int& row_tile, int& head) {      // rows: tiles over the batch
    int rank;
    if (heads % 8 == 0) {
        const unsigned own = heads / 8, slot = id >> 3;
        rank = slot / own; head = (id & 7) * own + slot % own;
    } else { rank = id / heads; head = id % heads; }
    if (rank >= rows) return false;
    row_tile = order ? order[rank] : rows - 1 - rank;
    return true;
}

// a barrier for what was written to LDS alone (__syncthreads waits for the next tile's DMA too)
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// bits a .. e - 1 of 64, both clamped
__device__ __forceinline__ unsigned long long bit_range(int a, int e) {
    a = max(a, 0); e = min(e, 64);
    return e > a ? (~0ull >> (64 - (e - a))) << a : 0ull;
}

// s in units of log2: cap(scale q.k) * log2 e.  cap tanh(x / cap) = cap (1 - 2 / (exp(2 x / cap) + 1)): one exp2 and one reciprocal; the absolute error is an fp32
// rounding of cap, enough in front of weights that are rounded to 16 bits (in 2 x 16 heads of 4096 x 4096 the forward takes 338 us with it, 128 wide, and 353 with the polynomial
// below; long documents 99 and 109).  c1 = scale * log2 e without a cap, 2 * scale * log2 e / cap with one; c2 = cap * log2 e.
__device__ __forceinline__ float span_tanh(float x, float c1) {
    return __builtin_fmaf(-2.f, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * c1) + 1.f), 1.f);
}

// tanh(u) to a few fp32 roundings of its own size, for what is fp32 behind it, the slopes' gradients and the lse of few rows: a score that is off by a rounding of its cap
// leaves them 3 - 15 times as far from the 64-bit form as a plain fp32 form is, a row of few keys 60 times (scores of a few units under caps of 30 and 50).
// |u| <= 1/2: u times a polynomial in u^2 (the minimax of the relative error, 1.5e-8, with 1 in front; Remez's exchange); beyond, the exponential.  A wave whose scores are all
// below takes the polynomial alone; otherwise the scores become their tanh first and the polynomial leaves them as they are (its coefficients are 0): one code for both, whose
// scores stay in their product's registers, and a score's value is the same either way, whatever stands beside it.
struct SpanTanh { float k, c[4]; };
constexpr float SPAN_TANH[4] = {-0.333331436f, 0.133258790f, -0.0530454926f, 0.0172414910f};
__device__ __forceinline__ float span_tanh_poly(float u, const float (&c)[4]) {
    const float v = u * u;
    float t = __builtin_fmaf(c[3], v, c[2]);
    t = __builtin_fmaf(t, v, c[1]);
    t = __builtin_fmaf(t, v, c[0]);
    return u * __builtin_fmaf(t, v, 1.f);
}
__device__ __forceinline__ float span_tanh_one(float u) {
    const float far = span_tanh(u, 2.f * SPAN_LOG2E);
    return fabsf(u) <= 0.5f ? span_tanh_poly(u, SPAN_TANH) : far;
}
// a block of raw scores in front of span_tanh_poly(raw * .k, .c) = tanh(raw k)
__device__ __forceinline__ SpanTanh span_tanh_block(f32x16_t& s, float k) {
    float m[4] = {0.f, 0.f, 0.f, 0.f};      // (a NaN is passed over: the polynomial keeps it)
#pragma unroll
    for (int r = 0; r < 16; ++r) m[r & 3] = fmaxf(m[r & 3], fabsf(s[r]));
    const bool near = __all(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])) * k <= 0.5f);
    if (!near)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = span_tanh_one(s[r] * k);
    SpanTanh t;
    t.k = near ? k : 1.f;
#pragma unroll
    for (int x = 0; x < 4; ++x) t.c[x] = near ? SPAN_TANH[x] : 0.f;
    return t;
}

// dot product of two rows by one lane
template <int D, bool F16>
__device__ __forceinline__ float row_dot(const uint16_t* x, const uint16_t* y) {
    float s = 0.f;
#pragma unroll 4
    for (int c = 0; c < D; c += 8) {
        const u32x4_t a = *reinterpret_cast<const u32x4_t*>(x + c), b = *reinterpret_cast<const u32x4_t*>(y + c);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            s = __builtin_fmaf(to_f32<F16>((uint16_t)a[e]), to_f32<F16>((uint16_t)b[e]), s);
            s = __builtin_fmaf(to_f32<F16>((uint16_t)(a[e] >> 16)), to_f32<F16>((uint16_t)(b[e] >> 16)), s);
        }
    }
    return s;
}

// o += sum over the set bits e of `sees` of w[lane e] * (row e of x)[lane], lane = element (o[1]: element lane + 64): eight rows' loads at a time.  Rows whose bit is clear
// are read where they lie (below `rows`) but not added, whatever they hold
template <int D, bool F16>
__device__ __forceinline__ void rows_add(float (&o)[2], unsigned long long sees, float w, const uint16_t* x, long stride, int rows, int lane) {
#pragma nounroll
    for (int e0 = 0; e0 < rows; e0 += 8) {
        if (((sees >> e0) & 0xFFull) == 0) continue;
        float a[8], c[8];
#pragma unroll
        for (int y = 0; y < 8; ++y) {
            const uint16_t* r = x + (long)min(e0 + y, rows - 1) * stride;
            a[y] = to_f32<F16>(r[D >= 64 ? lane : lane & (D - 1)]);
            c[y] = D > 64 ? to_f32<F16>(r[lane + 64]) : 0.f;
        }
#pragma unroll
        for (int y = 0; y < 8; ++y) {
            const float we = __shfl(w, e0 + y, 64);      // (e0 + y <= 63)
            if ((sees >> (e0 + y)) & 1ull) { o[0] = __builtin_fmaf(we, a[y], o[0]); o[1] = __builtin_fmaf(we, c[y], o[1]); }
        }
    }
}
// nothing finite can come back: every element of the sum is NaN
template <int D>
__device__ __forceinline__ bool all_nan(const float (&o)[2], int lane) { return __all((lane >= D || o[0] != o[0]) && (D <= 64 || o[1] != o[1])); }

// score (log2 units) of one visible pair by one lane; *slope: derivative of the cap; TANH: to its own size
template <int D, bool F16, int AX, bool TANH>
__device__ __forceinline__ float pair_score(const SpanArgs& p, const uint16_t* q, const uint16_t* k, int b, int h, int i, int key, float* slope) {
    float x = row_dot<D, F16>(q, k);
    *slope = 1.f;
    if (p.cap > 0.f) {
        const float t = TANH ? span_tanh_one(x * (p.scale / p.cap)) : span_tanh(x, 2.f * p.scale * SPAN_LOG2E / p.cap);
        *slope = 1.f - t * t;
        x = t * (p.cap * SPAN_LOG2E);
    } else x *= p.scale * SPAN_LOG2E;
#pragma unroll
    for (int a = 0; a < AX; ++a)
        x -= p.slopes[h * AX + a] * SPAN_LOG2E * fabsf((float)p.pos_q[b * p.pq_sb + (long)i * AX + a] - (float)p.pos_k[b * p.pk_sb + (long)key * AX + a]);
    return x;
}

// Tiles of 128 query rows, those that see the most keys first.  Documents differ in length: in their own order the long ones meet on some CUs and the others wait
// (16300 rows of packed images, 8 heads: 67 us, 60 so; long documents in order, 16 heads of 128: 137 and 107).  The length comes from four rows of a tile; it decides an
// order, no result.  One workgroup, a counting sort in LDS, up to SPAN_ORDER_MAX tiles; ITEMS = SPAN_ORDER_MAX / threads.
constexpr int SPAN_ORDER_MAX = 4096, SPAN_TILE = 128;
struct SpanOrderLds { int hist[1024], part[16]; };
template <int THREADS>
__device__ __forceinline__ void span_order_tiles(SpanOrderLds& m, const int32_t* __restrict__ spans, long sb, int B, int n, int nk, int32_t* __restrict__ order) {
    constexpr int ITEMS = SPAN_ORDER_MAX / THREADS, PER = 1024 / THREADS;
    const int t = threadIdx.x, lane = t & 63, w = t >> 6, tiles = (n + SPAN_TILE - 1) / SPAN_TILE, N = B * tiles;
#pragma unroll
    for (int y = 0; y < PER; ++y) m.hist[t * PER + y] = 0;
    __syncthreads();
    int bucket[ITEMS];
#pragma unroll
    for (int x = 0; x < ITEMS; ++x) {
        const int item = t + x * THREADS;
        bucket[x] = 0;
        if (item >= N) continue;
        const int2* sp = reinterpret_cast<const int2*>(spans + (item / tiles) * sb);
        const int r0 = item % tiles * SPAN_TILE;
        int lo = INT32_MAX, hi = 0;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            const int2 v = sp[min(r0 + y * (SPAN_TILE - 1) / 3, n - 1)];
            const int a = max(v.x, 0), e = min(v.y, nk);
            if (a < e) { lo = min(lo, a); hi = max(hi, e); }
        }
        const long len = hi > lo ? hi - lo : 0;
        bucket[x] = 1023 - (int)(len * 1023 / max(nk, 1));
        atomicAdd(&m.hist[bucket[x]], 1);
    }
    __syncthreads();
    int own[PER], v = 0;
#pragma unroll
    for (int y = 0; y < PER; ++y) { own[y] = m.hist[t * PER + y]; v += own[y]; }
    const int mine = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) { const int u = __shfl_up(v, o, 64); if (lane >= o) v += u; }
    if (lane == 63) m.part[w] = v;
    __syncthreads();
    int base = v - mine;
    for (int x = 0; x < w; ++x) base += m.part[x];
#pragma unroll
    for (int y = 0; y < PER; ++y) { m.hist[t * PER + y] = base; base += own[y]; }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < ITEMS; ++x)
        if (t + x * THREADS < N) order[atomicAdd(&m.hist[bucket[x]], 1)] = t + x * THREADS;
}
// the order pays from two workgroups per CU on (below, all of them start at once)
inline long span_order_count(const mm_span_attn* a) {
    const long n = (long)a->batch * ((a->nq + SPAN_TILE - 1) / SPAN_TILE);
    return a->spans && n <= SPAN_ORDER_MAX && n * a->heads_q >= 512 ? n : 0;
}

// more than 64 KiB of dynamic LDS has to be allowed once per kernel and device (`done`: a bit per device)
inline int span_allow_lds(const void* kernel, int bytes, std::atomic<unsigned long long>& done) {
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e == hipSuccess && (dev > 63 || !((done.load() >> dev) & 1ull))) {
        e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == hipSuccess && dev < 64) done.fetch_or(1ull << dev);
    }
    return e == hipSuccess ? MM_OK : mm_set_hip_error(e, "span attention LDS");
}

}  // namespace
