// rsx_logprob.h -- what the full-catalog log-probability (rsx_logprob.hip) and its gradient (rsx_logprob_grad.hip) share.
//
// fp32 tables go through the 16-bit matrix cores: v_mfma_f32_32x32x16_f16 does 16 times the products of v_mfma_f32_32x32x2_f32, and
// x = hi + lo with hi = half(x), lo = half(x - hi) holds x to 2^-24 of itself (11 + 11 bits and a sign) as long as lo is not
// subnormal.  x y = hi hi' + hi lo' + lo hi' (lo lo' is below 2^-24 |x y|): three instructions instead of sixteen.  A row of P, and
// 32 rows of Q together, are scaled by a power of two that puts their largest element into [2^13, 2^14): elements down to 2^-27 of the
// largest keep their 24 bits.  Where the largest elements of 32 rows of Q lie more than 2^12 apart, each has a scale of its own: a row that shares one
// is then off by 2^-26 of its own largest element at most, whatever its neighbours are.  bf16 tables are multiplied as they are.
#pragma once
#include "rsx_common.h"

namespace lp {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.69314718055994530942;
constexpr int kTile = 32;                 // items (or rows) of one matrix instruction

// eight 16-bit elements, the operand of one lane
union Frag {
    half8 h;
    bf16x8 b;
    uint4 u;
};

template <bool F32>
__device__ __forceinline__ f32x16 mfma32(const Frag &a, const Frag &b, f32x16 c)
{
    if constexpr (F32) return __builtin_amdgcn_mfma_f32_32x32x16_f16(a.h, b.h, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.b, b.b, c, 0, 0, 0);
}

__device__ __forceinline__ float bf16_f32(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
__device__ __forceinline__ uint16_t f32_bf16(float v)        // nearest even; NaN stays NaN
{
    const uint32_t u = __float_as_uint(v);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (uint16_t)((u >> 16) | 0x40u);
    return (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}

// geometry of a [rows x d] operand as 16-bit planes: a row is hi[d] lo[d] (fp32) or [d] (bf16)
template <int D, bool F32>
struct Geo {
    static constexpr int NP = F32 ? 2 : 1, ROWB = D * NP * 2, TILEB = kTile * ROWB, KS = D / 16;
    // 16-byte slots of a row are XORed with this, so that the 16 rows a quarter of a fragment read touches fall on 16 different slots of
    // the 256 bytes the LDS delivers a cycle (rows of 64 and 128 bytes: 4 and 2 of them share a line)
    __device__ static __forceinline__ int swz(int row) { return ROWB >= 256 ? row & 15 : ROWB == 128 ? (row >> 1) & 7 : (row >> 2) & 3; }
};

// 64 lanes x 16 (or 4) bytes from global memory straight into LDS, lane-linear from a wavefront-uniform base.
// (functions of their own: called from a kernel's body, the builtin costs the kernel its host stub)
__device__ __forceinline__ void copy_to_lds(const char *src, char *dst) { __builtin_amdgcn_global_load_lds(src, dst, 16, 0, 0); }
__device__ __forceinline__ void copy4_to_lds(const char *src, char *dst) { __builtin_amdgcn_global_load_lds(src, dst, 4, 0, 0); }
// wait for this wavefront's copies (and other accesses to memory): vmcnt(0)
__device__ __forceinline__ void wait_memory() { __builtin_amdgcn_s_waitcnt(0x0F70); }
// Every wavefront's copies have landed, and everybody is done with what they will be followed by.  The wait is written out: a barrier alone orders
// LDS and waits for the copies only where the compiler happens to have a reason to, and the others' copies are not its concern.
__device__ __forceinline__ void barrier_after_copies()
{
    wait_memory();
    __syncthreads();
}

// power of two that brings a largest magnitude m into [2^13, 2^14), and its inverse.  Below 2^-112 as for 2^-112, where both are still normal
__device__ __forceinline__ void scale_for(float m, float *up, float *down)
{
    int e = (int)((__float_as_uint(m) >> 23) & 0xFF) - 126;      // m in [2^(e-1), 2^e)
    e = e < -112 ? -112 : e;
    *up = ldexpf(1.0f, 14 - e);
    *down = ldexpf(1.0f, e - 14);
}
__device__ __forceinline__ float finite_abs(float v) { const float a = fabsf(v); return a < INFINITY ? a : 0.0f; }     // NaN and infinities: 0

// a value the compiler does not look behind.  half(a * b) becomes one fused instruction that rounds the exact product once, and where the same half
// is also needed in fp32 (to form its remainder) the unfused one is used beside it: at a tie of the two roundings hi and lo would not belong
// to each other (errors of 2^-11 of an element, one in some thousand).
__device__ __forceinline__ float opaque(float v)
{
    asm("" : "+v"(v));
    return v;
}

// eight scaled floats -> the two planes' fragments, two at a time (v_cvt_pk_f16_f32, to nearest)
typedef float float2v __attribute__((ext_vector_type(2)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void split8(const float *x, Frag *hi, Frag *lo)
{
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const float2v v = {opaque(x[j]), opaque(x[j + 1])};
        const half2v h = __builtin_convertvector(v, half2v);
        const float2v r = {v[0] - (float)h[0], v[1] - (float)h[1]};
        const half2v l = __builtin_convertvector(r, half2v);
        hi->h[j] = h[0]; hi->h[j + 1] = h[1];
        lo->h[j] = l[0]; lo->h[j + 1] = l[1];
    }
}

// ... of x times k, the product not rounded before it is split
__device__ __forceinline__ void split8_times(const float *x, double k, Frag *hi, Frag *lo)
{
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const double y = (double)x[j] * k;
        const _Float16 h = (_Float16)opaque((float)y);
        hi->h[j] = h;
        lo->h[j] = (_Float16)opaque((float)(y - (double)(float)h));
    }
}

// eight consecutive elements of a table row in fp32
template <bool F32>
__device__ __forceinline__ void load8(const void *base, int64_t at, float *x)
{
    if constexpr (F32) {
        const float4 *p = reinterpret_cast<const float4 *>((const float *)base + at);
        const float4 a = p[0], b = p[1];
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
        const uint4 v = *reinterpret_cast<const uint4 *>((const uint16_t *)base + at);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) { x[2 * j] = __uint_as_float(w[j] << 16); x[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u); }
    }
}

// rows of the call: a position whose user id is outside the table names no row
__device__ __forceinline__ bool row_ok(int32_t u, int64_t num_users) { return u >= 0 && u < num_users; }

// words a row of the bit mask holds: four tiles of 32 items at a time
__host__ __device__ __forceinline__ int64_t mask_words(int64_t num_items) { return (num_items + 127) / 128 * 4; }

// seen items of the call's rows as bits, [rows][words]: bit i & 31 of word i >> 5.  One workgroup per row builds 32 KB of it at a time in LDS and
// writes it out whole: no clearing pass, no atomics on memory.  A position that names no row sees everything.
constexpr int kBitWords = 8192;
__device__ __forceinline__ void write_seen_bits(int32_t u, bool ok, const int64_t *__restrict__ indptr, const int32_t *__restrict__ indices, int64_t num_items,
                                                uint32_t *__restrict__ row, uint32_t *lds)
{
    const int64_t words = mask_words(num_items);
    const int64_t lo = ok ? indptr[u] : 0, hi = ok ? indptr[u + 1] : 0;
    for (int64_t w0 = 0; w0 < words; w0 += kBitWords) {
        const int n = (int)(words - w0 < kBitWords ? words - w0 : kBitWords);             // (a multiple of four)
        for (int t = threadIdx.x; t < n / 4; t += blockDim.x) reinterpret_cast<uint4 *>(lds)[t] = ok ? make_uint4(0u, 0u, 0u, 0u) : make_uint4(~0u, ~0u, ~0u, ~0u);
        __syncthreads();
        for (int64_t p = lo + threadIdx.x; p < hi; p += blockDim.x) {
            const int32_t i = indices[p];
            const int64_t w = (i >> 5) - w0;
            if (i >= 0 && i < num_items && w >= 0 && w < n) atomicOr(lds + w, 1u << (i & 31));
        }
        __syncthreads();
        for (int t = threadIdx.x; t < n / 4; t += blockDim.x) reinterpret_cast<uint4 *>(row + w0)[t] = reinterpret_cast<const uint4 *>(lds)[t];
        __syncthreads();
    }
}

// rows of a tile share a scale while their largest elements lie within this; rows of zeros do not count.  (Every tile with scales of its rows' own: 1024 x 100K x 128
// fp32 115 -> 128 us, the gradient 372 -> 378, in bf16 186 -> 193)
constexpr float kUneven = 4096.0f;
constexpr float kOwnScales = -1.0f;       // in place of a tile's factor: every row has its own

// largest element of this thread's row (held by its TPR neighbours), and of the 32 rows the largest and smallest of those
template <int TPR>
__device__ __forceinline__ float row_max(float m)
{
#pragma unroll
    for (int o = TPR / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, TPR));
    return m;
}
__device__ __forceinline__ void tile_range(float *most, float *least, float *lds)      // by 256 threads, over their values; lds: 8 words
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) { *most = fmaxf(*most, __shfl_xor(*most, o, 64)); *least = fminf(*least, __shfl_xor(*least, o, 64)); }
    if ((threadIdx.x & 63) == 0) { lds[threadIdx.x >> 6] = *most; lds[4 + (threadIdx.x >> 6)] = *least; }
    __syncthreads();
    *most = fmaxf(fmaxf(lds[0], lds[1]), fmaxf(lds[2], lds[3]));
    *least = fminf(fminf(lds[4], lds[5]), fminf(lds[6], lds[7]));
}

// a tile of fp32 item rows -> scaled planes [tiles padded to a multiple of 4][32][hi d, lo d] and the tile's factor (or kOwnScales and its rows'), by 256
// threads.  Rows behind the last item are zero.
template <int D>
__device__ __forceinline__ void split_items(const float *__restrict__ Q, int64_t num_items, int64_t tile, uint4 *__restrict__ planes, float *__restrict__ factor,
                                            float *__restrict__ row_factor, float *lds)
{
    constexpr int TPR = D / 8, RPP = 256 / TPR, N = kTile / RPP > 0 ? kTile / RPP : 1;       // threads a row, rows a pass, passes
    const int tid = threadIdx.x;
    float x[N][8], big[N];
    float most = 0.0f, least = INFINITY;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int r = n * RPP + tid / TPR;
        const int64_t i = tile * kTile + r;
        const bool live = r < kTile && i < num_items;
        const float4 *src = reinterpret_cast<const float4 *>(Q + (size_t)(live ? i : 0) * D + 8 * (tid % TPR));
        const float4 a = live ? src[0] : make_float4(0.f, 0.f, 0.f, 0.f), b = live ? src[1] : make_float4(0.f, 0.f, 0.f, 0.f);
        x[n][0] = a.x; x[n][1] = a.y; x[n][2] = a.z; x[n][3] = a.w; x[n][4] = b.x; x[n][5] = b.y; x[n][6] = b.z; x[n][7] = b.w;
        float m = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, finite_abs(x[n][j]));
        big[n] = row_max<TPR>(m);
        most = fmaxf(most, big[n]);
        least = big[n] > 0.0f ? fminf(least, big[n]) : least;
    }
    tile_range(&most, &least, lds);
    const bool own = least * kUneven < most;
    float up, down;
    scale_for(most, &up, &down);
    if (tid == 0) factor[tile] = own ? kOwnScales : down;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int r = n * RPP + tid / TPR;
        if (r >= kTile) continue;
        if (own) {
            scale_for(big[n], &up, &down);
            if (tid % TPR == 0) row_factor[tile * kTile + r] = down;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) x[n][j] *= up;
        Frag h, l;
        split8(x[n], &h, &l);
        uint4 *dst = planes + (size_t)(tile * kTile + r) * (2 * TPR) + tid % TPR;
        dst[0] = h.u;
        dst[TPR] = l.u;
    }
}

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline int64_t a256(int64_t x) { return (x + 255) / 256 * 256; }

}  // namespace lp
