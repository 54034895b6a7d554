// rsx_ortho.hip -- Newton-Schulz orthogonalisation of a tall [rows x d] matrix and the optimizer step built on it, for gfx950 (MI355X).
//
//   X_0 = X / (|X|_F + eps);   X_{k+1} = a X_k + X_k (b A_k + c A_k^2),   A_k = X_k^T X_k          (`steps` times)
//
// Every X_k is X times a polynomial of G = X^T X, so only the first Gram matrix and the last product touch the rows:
//   with s = 1 / (|X|_F + eps), A_0 = s^2 G, M_0 = s I:   T = a I + b A + c A^2,   M <- M T,   A <- T A T = (A T) T,   X_steps = X M.
// All these matrices are symmetric and commute.  |X|_F^2 is the trace of G: it costs no pass of its own.
//
// The [d x d] part is held in 64 bits.  A step amplifies A's small eigenvalues by a^2 (about 12): noise of 2^-24 |A| in G would have
// grown to 12^4 * 6e-8 = 1e-3 by the fifth step, and decide the small directions of X.  v_mfma_f64_16x16x4_f64 does the products.
//
// Four launches of row work and [d x d] work:
//   gram_kernel    rows -> partial Gram matrices (upper triangle of 16 x 16 blocks), with the momentum update of the optimizer step
//   gram_reduce    partials in a fixed order -> G
//   ns_*           the iteration in [d x d]
//   project_kernel rows times M (fp32 MFMA), with the weight update of the optimizer step
#include <type_traits>

#include "rsx_common.h"

namespace {

typedef double f64x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// round to nearest even; NaN stays NaN
__device__ __forceinline__ uint16_t f32_bf16(float v)
{
    const uint32_t u = __float_as_uint(v);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (uint16_t)((u >> 16) | 0x40u);
    return (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}

// what is orthogonalised: X itself, or the optimizer's momentum (M <- mu M + G, U = G + mu M or M)
template <typename T, bool MUON>
struct Rows {
    const T *X;       // X, or the gradient G
    float *M;         // MUON: the momentum
    float mu;
    int nesterov;
};

// four elements of it, asked for early and used late
template <typename T, bool MUON>
struct Piece {
    typename std::conditional<sizeof(T) == 2, uint2, uint4>::type x;
    float4 m;
    __device__ __forceinline__ void load(const Rows<T, MUON> &in, int64_t at, int64_t end)
    {
        if (at >= end) return;
        x = *reinterpret_cast<const decltype(x) *>(in.X + at);
        if constexpr (MUON) m = *reinterpret_cast<const float4 *>(in.M + at);
    }
    // UPDATE: this is the pass that advances M
    template <bool UPDATE>
    __device__ __forceinline__ float4 take(const Rows<T, MUON> &in, int64_t at, int64_t end)
    {
        if (at >= end) return make_float4(0.f, 0.f, 0.f, 0.f);
        float4 g;
        if constexpr (sizeof(T) == 2) g = make_float4(__uint_as_float(x.x << 16), __uint_as_float(x.x & 0xFFFF0000u), __uint_as_float(x.y << 16), __uint_as_float(x.y & 0xFFFF0000u));
        else g = make_float4(__uint_as_float(x.x), __uint_as_float(x.y), __uint_as_float(x.z), __uint_as_float(x.w));
        if constexpr (MUON) {
            const float mu = in.mu;
            if constexpr (UPDATE) {
                m = make_float4(fmaf(mu, m.x, g.x), fmaf(mu, m.y, g.y), fmaf(mu, m.z, g.z), fmaf(mu, m.w, g.w));
                *reinterpret_cast<float4 *>(in.M + at) = m;
            }
            if (!in.nesterov) return m;
            g = make_float4(fmaf(mu, m.x, g.x), fmaf(mu, m.y, g.y), fmaf(mu, m.z, g.z), fmaf(mu, m.w, g.w));
        }
        return g;
    }
};

// ---- the Gram matrix -------------------------------------------------------------------------------------------------------------
// Column groups of 16: what a lane's 16-byte (d = 32: 8-byte) piece of a row holds for m = lane & 15 -- no transpose.  group_col maps (group, m) back.
__host__ __device__ constexpr int n_groups(int D) { return D / 16; }
__device__ __forceinline__ int group_col(int D, int b, int m) { return D == 32 ? 2 * m + b : 64 * (b >> 2) + 4 * m + (b & 3); }
__host__ __device__ constexpr int n_blocks(int D) { return n_groups(D) * (n_groups(D) + 1) / 2; }
__host__ __device__ constexpr int block_at(int D, int p, int q) { return p * n_groups(D) - p * (p - 1) / 2 + (q - p); }   // q >= p

// Eight wavefronts; the 16 x 16 blocks of the upper triangle are dealt to SETS of them (8 registers a block: 72 at d = 128, 136 at d = 256, so that two
// wavefronts share a SIMD), the rows of a tile to the 8 / SETS wavefronts of a set.  16 KB tiles pass through LDS; two tiles of G and M are on their way
// in registers (64 KB a CU: what HBM's latency takes).  Bound by HBM with the momentum (1M x 128: 1.5 GB in 0.39 ms), by the fp64 matrix
// rate without (36 instructions of 64 cycles per four rows: 0.27 ms).
// d = 256 without the momentum (whose update one workgroup has to make): four workgroups share a row range and its blocks, two sets each, so that there
// are a quarter of the partials (20011 rows: 37 us and 5 to add them up; 256 workgroups with all 136 blocks each: 35 and 15).
template <int D, bool MUON>
struct Gram {
    static constexpr int SHARE = D == 256 && !MUON ? 4 : 1;
    static constexpr int SETS = D == 256 ? 8 : D == 128 ? 4 : 1, MINE = SETS / SHARE, KSPLIT = 8 / MINE, TR = 4096 / D, NB = n_blocks(D), PER = (NB + SETS - 1) / SETS;
};

template <int D, int SET, typename F>
__device__ __forceinline__ void set_blocks(F f)          // f(index of the accumulator, block, column group p, column group q)
{
    int a = 0, n = 0;
#pragma unroll
    for (int p = 0; p < n_groups(D); ++p)
#pragma unroll
        for (int q = p; q < n_groups(D); ++q, ++n)
            if (n / Gram<D, true>::PER == SET) f(a++, n, p, q);
}

template <int D, int SET, typename T, bool MUON>
__device__ __forceinline__ void gram_body(const Rows<T, MUON> &in, int64_t rows, int piece, int pieces, double *__restrict__ part, char *lds)
{
    using C = Gram<D, MUON>;
    constexpr int LW = D == 32 ? 2 : 4;                                 // elements of a lane's piece
    const int tid = threadIdx.x, lane = tid & 63, ks = (tid >> 6) % C::KSPLIT;
    f64x4 acc[C::PER];
#pragma unroll
    for (int b = 0; b < C::PER; ++b) acc[b] = f64x4{0.0, 0.0, 0.0, 0.0};
    const int64_t stride = (int64_t)pieces * C::TR, first = (int64_t)piece * C::TR;
    Piece<T, MUON> a[2], b[2];                                          // this thread's two pieces of the next tile, and of the one after
    auto at = [&](int64_t r0, int n) { return r0 * D + 4 * (tid + 512 * n); };
    auto fetch = [&](Piece<T, MUON> (&p)[2], int64_t r0) {
#pragma unroll
        for (int n = 0; n < 2; ++n) p[n].load(in, at(r0, n), rows * D);
    };
    auto tile = [&](Piece<T, MUON> (&p)[2], int64_t r0, float *t) {     // pieces of tile r0 -> LDS, then the next but one is asked for
#pragma unroll
        for (int n = 0; n < 2; ++n) *reinterpret_cast<float4 *>(t + 4 * (tid + 512 * n)) = p[n].template take<true>(in, at(r0, n), rows * D);
        fetch(p, r0 + 2 * stride);
        __syncthreads();                                                // (two tiles: a slow wavefront still reads the last one)
#pragma unroll 1
        for (int k = 4 * ks; k < C::TR; k += 4 * C::KSPLIT) {
            const float *row = t + (k + (lane >> 4)) * D + LW * (lane & 15);
            double v[n_groups(D)];
            if constexpr (D == 32) {
                const float2 x = *reinterpret_cast<const float2 *>(row);
                v[0] = x.x; v[1] = x.y;
            } else {
#pragma unroll
                for (int q = 0; q < D / 64; ++q) {
                    const float4 x = *reinterpret_cast<const float4 *>(row + 64 * q);
                    v[4 * q] = x.x; v[4 * q + 1] = x.y; v[4 * q + 2] = x.z; v[4 * q + 3] = x.w;
                }
            }
            set_blocks<D, SET>([&](int i, int, int p, int q) { acc[i] = __builtin_amdgcn_mfma_f64_16x16x4f64(v[p], v[q], acc[i], 0, 0, 0); });
        }
    };
    fetch(a, first);
    fetch(b, first + stride);
    float *const t0 = reinterpret_cast<float *>(lds), *const t1 = t0 + 4096;
    for (int64_t r0 = first; r0 < rows; r0 += 2 * stride) {             // (every wavefront of the workgroup runs the same rounds and barriers)
        tile(a, r0, t0);
        if (r0 + stride < rows) tile(b, r0 + stride, t1);
    }
    // the KSPLIT wavefronts of a set one after the other (a fixed order), through LDS four blocks a set at a time; then the workgroup's partial
    // (f64 result layout: register pair i of lane l is row 4 i + (l >> 4), column l & 15)
    double *dst = part + (size_t)piece * (C::NB * 256);
    auto cell = [&](int i) { return (4 * i + (lane >> 4)) * 16 + (lane & 15); };
    if constexpr (C::KSPLIT == 1) {
        set_blocks<D, SET>([&](int i, int n, int, int) {
#pragma unroll
            for (int e = 0; e < 4; ++e) dst[n * 256 + cell(e)] = acc[i][e];
        });
    } else {
        double *red = reinterpret_cast<double *>(lds) + SET % C::MINE * 4 * 256;  // (sets x 4 blocks of 2 KB: 32 KB at most)
#pragma unroll
        for (int i0 = 0; i0 < C::PER; i0 += 4) {
            for (int w = 0; w < C::KSPLIT; ++w) {
                __syncthreads();
                if (ks != w) continue;
                set_blocks<D, SET>([&](int i, int n, int, int) {
                    if (i < i0 || i >= i0 + 4) return;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        double *c = red + (i - i0) * 256 + cell(e);
                        const double v = w == 0 ? acc[i][e] : *c + acc[i][e];
                        if (w + 1 < C::KSPLIT) *c = v; else dst[n * 256 + cell(e)] = v;
                    }
                });
            }
        }
    }
}

template <int D, typename T, bool MUON>
__global__ __launch_bounds__(512, (D == 256 ? 2 : 4)) void gram_kernel(Rows<T, MUON> in, int64_t rows, double *__restrict__ part)
{
    using C = Gram<D, MUON>;
    __shared__ __attribute__((aligned(16))) char lds[32768];
    // workgroups of one row range 8 apart: on one XCD, whose L2 they share
    const int share = C::SHARE == 1 ? 0 : blockIdx.x / 8 % C::SHARE, pieces = gridDim.x / C::SHARE;
    const int piece = C::SHARE == 1 ? blockIdx.x : blockIdx.x / (8 * C::SHARE) * 8 + blockIdx.x % 8;
    const int set = __builtin_amdgcn_readfirstlane(share * C::MINE + (threadIdx.x >> 6) / C::KSPLIT);
    if (set == 0) gram_body<D, 0, T, MUON>(in, rows, piece, pieces, part, lds);
    if constexpr (C::SETS >= 4) {
        if (set == 1) gram_body<D, 1, T, MUON>(in, rows, piece, pieces, part, lds);
        if (set == 2) gram_body<D, 2, T, MUON>(in, rows, piece, pieces, part, lds);
        if (set == 3) gram_body<D, 3, T, MUON>(in, rows, piece, pieces, part, lds);
    }
    if constexpr (C::SETS >= 8) {
        if (set == 4) gram_body<D, 4, T, MUON>(in, rows, piece, pieces, part, lds);
        if (set == 5) gram_body<D, 5, T, MUON>(in, rows, piece, pieces, part, lds);
        if (set == 6) gram_body<D, 6, T, MUON>(in, rows, piece, pieces, part, lds);
        if (set == 7) gram_body<D, 7, T, MUON>(in, rows, piece, pieces, part, lds);
    }
}

// partials -> the full symmetric matrix in column order.  32 elements x 16 slices of the partials per workgroup, eight loads of two elements on their
// way (512 partials of d = 128, 38 MB: 7.5 us; one element a load, as many as the compiler unrolls: 13).
template <int D>
__global__ __launch_bounds__(256) void gram_reduce_kernel(const double *__restrict__ part, int n_part, double *__restrict__ G)
{
    constexpr int NB = n_blocks(D);
    __shared__ double s[16][34];
    const int e = threadIdx.x & 15, sl = threadIdx.x >> 4;
    const int at = blockIdx.x * 32 + 2 * e;                   // element of [NB][16][16]
    double2 sum = make_double2(0.0, 0.0);
    for (int p0 = sl; p0 < n_part; p0 += 128) {
        double2 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int p = p0 + 16 * k;
            v[k] = p < n_part ? *reinterpret_cast<const double2 *>(part + (size_t)p * (NB * 256) + at) : make_double2(0.0, 0.0);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) { sum.x += v[k].x; sum.y += v[k].y; }
    }
    s[sl][2 * e] = sum.x;
    s[sl][2 * e + 1] = sum.y;
    __syncthreads();
    if (threadIdx.x < 32) {
        double v = 0.0;
#pragma unroll
        for (int i = 0; i < 16; ++i) v += s[i][threadIdx.x];
        const int cell = blockIdx.x * 32 + threadIdx.x, blk = cell >> 8;
        int p = 0;
        while (p + 1 < n_groups(D) && block_at(D, p + 1, p + 1) <= blk) ++p;
        const int q = p + blk - block_at(D, p, p);
        const int r = group_col(D, p, (cell >> 4) & 15), c = group_col(D, q, cell & 15);
        G[(size_t)r * D + c] = v;
        G[(size_t)c * D + r] = v;
    }
}

// ---- the iteration in [d x d] ------------------------------------------------------------------------------------------------------
struct Coeffs { double a, b, c, eps; };

// 1 / (|X|_F + eps): every workgroup sums the diagonal in the same order
__device__ __forceinline__ double norm_scale(const double *G, int D, double eps, double *lds)
{
    if (threadIdx.x < 64) {
        double t = 0.0;
        for (int i = threadIdx.x; i < D; i += 64) t += G[(size_t)i * D + i];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
        if (threadIdx.x == 0) *lds = 1.0 / (sqrt(t) + eps);
    }
    __syncthreads();
    return *lds;
}

// one 16 x 16 block of X Y (both symmetric): four wavefronts share the contraction.  Operands are read as rows k, columns of the block.
template <int D, typename FX, typename FY>
__device__ __forceinline__ double ns_block(FX fx, FY fy, int p, int q, double (*red)[64][4])
{
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    constexpr int KS = D / 16;
    double x[KS], y[KS];
#pragma unroll
    for (int i = 0; i < KS; ++i) {
        const int k = w * (D / 4) + 4 * i + (lane >> 4);
        x[i] = fx(k, 16 * p + (lane & 15));
        y[i] = fy(k, 16 * q + (lane & 15));
    }
    f64x4 acc = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
    for (int i = 0; i < KS; ++i) acc = __builtin_amdgcn_mfma_f64_16x16x4f64(x[i], y[i], acc, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) red[w][lane][i] = acc[i];
    __syncthreads();
    const int r = threadIdx.x >> 4, c = threadIdx.x & 15, l = (r & 3) * 16 + c;
    return red[0][l][r >> 2] + red[1][l][r >> 2] + red[2][l][r >> 2] + red[3][l][r >> 2];
}

template <int D>
__device__ __forceinline__ void ns_pq(int b, int *p, int *q)
{
    int i = 0;
    while (i + 1 < n_groups(D) && block_at(D, i + 1, i + 1) <= b) ++i;
    *p = i; *q = i + b - block_at(D, i, i);
}

// both triangles from the upper one.  (On the diagonal X Y's (r, c) and (c, r) are sums of other roundings: one of them, always the same
// one, stands for both.)
template <int D>
__device__ __forceinline__ void ns_store(double *out, int p, int q, double v)
{
    const int r = 16 * p + (threadIdx.x >> 4), c = 16 * q + (threadIdx.x & 15);
    if (r > c) return;
    out[(size_t)r * D + c] = v;
    out[(size_t)c * D + r] = v;
}

// the result: fp32 for the fp32 products, or three bf16 planes that add up to it in the operand order of project_bf16_kernel:
// [32 columns][16 rows][plane][lane][8]
template <int D>
__device__ __forceinline__ void put_result(float *out, int r, int c, double v) { out[(size_t)r * D + c] = (float)v; }
template <int D>
__device__ __forceinline__ void put_result(uint16_t *out, int r, int c, double v)
{
    float m = (float)v;
    uint16_t *dst = out + ((((size_t)(c / 32) * (D / 16) + r / 16) * 3) * 64 + 32 * ((r % 16) / 8) + c % 32) * 8 + r % 8;
#pragma unroll
    for (int n = 0; n < 3; ++n) {
        const uint16_t h = f32_bf16(m);
        dst[n * 512] = h;
        m -= __uint_as_float((uint32_t)h << 16);
    }
}
template <int D, typename O>
__device__ __forceinline__ void ns_result(O *out, int p, int q, double v)
{
    const int r = 16 * p + (threadIdx.x >> 4), c = 16 * q + (threadIdx.x & 15);
    if (r > c) return;
    put_result<D>(out, r, c, v);
    put_result<D>(out, c, r, v);
}

// T = a I + b A + c A A, for the two kernels behind it.  FIRST: A = s^2 G is formed here and stored
template <int D, bool FIRST>
__global__ __launch_bounds__(256) void ns_square_kernel(const double *__restrict__ G, double *__restrict__ A, double *__restrict__ T, Coeffs k)
{
    __shared__ double red[4][64][4], s_norm;
    int p, q;
    ns_pq<D>(blockIdx.x, &p, &q);
    const int r = 16 * p + (threadIdx.x >> 4), c = 16 * q + (threadIdx.x & 15);
    double here = G[(size_t)r * D + c];
    auto f = [&](int i, int j) { return G[(size_t)i * D + j]; };
    double v = ns_block<D>(f, f, p, q, red);
    if constexpr (FIRST) {
        const double s = norm_scale(G, D, k.eps, &s_norm), s2 = s * s;
        here *= s2;
        v *= s2 * s2;
        ns_store<D>(A, p, q, here);
    }
    ns_store<D>(T, p, q, fma(k.c, v, fma(k.b, here, r == c ? k.a : 0.0)));
}

// blockIdx.y == 0: out_m = M T (FIRST: s T, no product);  1: W = A T
template <int D, bool FIRST, typename O>
__global__ __launch_bounds__(256) void ns_times_t_kernel(const double *__restrict__ G, const double *__restrict__ A, const double *__restrict__ T,
                                                         const double *__restrict__ M, O *__restrict__ out_m, double *__restrict__ W, double eps)
{
    __shared__ double red[4][64][4], s_norm;
    int p, q;
    ns_pq<D>(blockIdx.x, &p, &q);
    auto t = [&](int r, int c) { return T[(size_t)r * D + c]; };
    if (blockIdx.y == 0) {
        double v;
        if constexpr (FIRST) v = norm_scale(G, D, eps, &s_norm) * t(16 * p + (threadIdx.x >> 4), 16 * q + (threadIdx.x & 15));
        else v = ns_block<D>([&](int r, int c) { return M[(size_t)r * D + c]; }, t, p, q, red);
        if constexpr (std::is_same<O, double>::value) ns_store<D>(out_m, p, q, v);
        else ns_result<D>(out_m, p, q, v);
    } else {
        ns_store<D>(W, p, q, ns_block<D>([&](int r, int c) { return A[(size_t)r * D + c]; }, t, p, q, red));
    }
}

// A' = W T
template <int D>
__global__ __launch_bounds__(256) void ns_next_kernel(const double *__restrict__ W, const double *__restrict__ T, double *__restrict__ A2)
{
    __shared__ double red[4][64][4];
    int p, q;
    ns_pq<D>(blockIdx.x, &p, &q);
    ns_store<D>(A2, p, q, ns_block<D>([&](int r, int c) { return W[(size_t)r * D + c]; }, [&](int r, int c) { return T[(size_t)r * D + c]; }, p, q, red));
}

// d <= 64: the whole iteration in one workgroup, the four matrices in LDS (128 KB at d = 64).  Blocks of the upper triangles are dealt to 16 wavefronts
// (M T and A T together: 20 blocks, five a SIMD); both triangles are written.  Bound by one CU's fp64 matrix rate and the
// LDS reads before it (five steps at d = 64: 33 us, about 22 of them products; 38 before the addresses were one place and constant offsets).
// Columns are XORed by row: the two rows of a half-wavefront's read lie in different halves of the 256 bytes the LDS delivers a cycle, and the 16 rows
// of a transposed store in eight different places.
constexpr int kSmallThreads = 1024;      // (512: fewer wavefronts to cover the LDS reads, a 1682 x 64 step 54 us for 52)
template <int D, typename O>
__global__ __launch_bounds__(kSmallThreads) void ns_small_kernel(const double *__restrict__ G, O *__restrict__ out, int steps, Coeffs k)
{
    constexpr int NB = n_blocks(D), NW = kSmallThreads / 64, ONE = (NB + NW - 1) / NW, TWO = (2 * NB + NW - 1) / NW;      // a wavefront's blocks of one product, of a pair
    __shared__ __attribute__((aligned(16))) double A[D * D], T[D * D], W[D * D], M[D * D];
    __shared__ double s_norm;
    auto el = [](int r, int c) { return r * D + (c ^ (((r & 1) << 4) | ((r & 6) << 1))); };
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const double s = norm_scale(G, D, k.eps, &s_norm);
    for (int t = tid; t < D * D; t += kSmallThreads) {
        const int r = t / D, c = t % D;
        A[el(r, c)] = s * s * G[t];
    }
    __syncthreads();
    // el(4 i + (lane >> 4), 16 p + (lane & 15)) less 4 i D: one place for the even i, one for the odd ones
    auto place = [&](int p, int odd) { const int r = lane >> 4; return r * D + ((16 * p) ^ ((r & 1) << 4)) + ((lane & 15) ^ ((r & 2) << 1) ^ (odd << 3)); };
    auto mul = [&](const double *x, const double *y, int p, int q) {
        const int bx[2] = {place(p, 0), place(p, 1)}, by[2] = {place(q, 0), place(q, 1)};
        f64x4 acc = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
        for (int h = 0; h < D / 32; ++h) {                                // (eight steps' operands on their way before the first product)
            double fx[8], fy[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) { fx[i] = x[bx[i & 1] + (32 * h + 4 * i) * D]; fy[i] = y[by[i & 1] + (32 * h + 4 * i) * D]; }
#pragma unroll
            for (int i = 0; i < 8; ++i) acc = __builtin_amdgcn_mfma_f64_16x16x4f64(fx[i], fy[i], acc, 0, 0, 0);
        }
        return acc;
    };
    auto put = [&](double *x, int p, int q, int i, double v) {           // (on the diagonal one of (r, c) and (c, r) stands for both)
        const int r = 16 * p + 4 * i + (lane >> 4), c = 16 * q + (lane & 15);
        if (r > c) return;
        x[el(r, c)] = v;
        x[el(c, r)] = v;
    };
    for (int step = 0; step < steps; ++step) {
        const bool last = step + 1 == steps;
        f64x4 x[TWO];                                                      // (results leave the registers when everybody has read what they replace)
        int p, q;
#pragma unroll
        for (int n = 0; n < ONE; ++n) {
            if (w + NW * n >= NB) continue;
            ns_pq<D>(w + NW * n, &p, &q);
            const f64x4 sq = mul(A, A, p, q);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 16 * p + 4 * i + (lane >> 4), c = 16 * q + (lane & 15);
                put(T, p, q, i, fma(k.c, sq[i], fma(k.b, A[el(r, c)], r == c ? k.a : 0.0)));
            }
        }
        __syncthreads();
        // blocks of A T, then of M T (not of A T in the last step, nor of M T in the first: M = s I)
        const int first = last ? NB : 0, end = step == 0 ? NB : 2 * NB;
#pragma unroll
        for (int n = 0; n < TWO; ++n) {
            const int b = first + w + NW * n;
            if (b >= end) continue;
            ns_pq<D>(b % NB, &p, &q);
            x[n] = mul(b < NB ? A : M, T, p, q);
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < TWO; ++n) {
            const int b = first + w + NW * n;
            if (b >= end) continue;
            ns_pq<D>(b % NB, &p, &q);
#pragma unroll
            for (int i = 0; i < 4; ++i) put(b < NB ? W : M, p, q, i, x[n][i]);
        }
        if (step == 0)
#pragma unroll 1
            for (int t = tid; t < D * D; t += kSmallThreads) M[t] = s * T[t];
        __syncthreads();
        if (!last) {
#pragma unroll
            for (int n = 0; n < ONE; ++n) {                                // (A was last read before the barrier above)
                if (w + NW * n >= NB) continue;
                ns_pq<D>(w + NW * n, &p, &q);
                const f64x4 y = mul(W, T, p, q);
#pragma unroll
                for (int i = 0; i < 4; ++i) put(A, p, q, i, y[i]);
            }
        }
        __syncthreads();
    }
    for (int t = tid; t < D * D; t += kSmallThreads) put_result<D>(out, t / D, t % D, M[el(t / D, t % D)]);
}

template <int D, typename O>
__global__ __launch_bounds__(256) void ns_identity_kernel(const double *__restrict__ G, O *__restrict__ out, double eps)   // steps == 0
{
    __shared__ double s_norm;
    const double s = norm_scale(G, D, eps, &s_norm);
    for (int t = threadIdx.x; t < D * D; t += 256) put_result<D>(out, t / D, t % D, t / D == t % D ? s : 0.0);
}

// ---- rows times the [d x d] result ---------------------------------------------------------------------------------------------------
// v_mfma_f32_32x32x2_f32, exact fp32 products.  A wavefront owns 32 output columns and keeps its 32 columns of the [d x d] matrix in registers
// (d / 2 of them) for all its rows; rows pass through LDS, and so does the result, so that every access to memory is 16 bytes a lane.  The rows of the
// next tile and the weights of this one are on their way during the products.  The contraction index is permuted so that a lane
// reads its row four elements at a time: step 4 j + e multiplies k = 8 j + 4 (lane >> 5) + e.  Bound by HBM (optimizer step, 1M x 128: 2.6 GB in 0.47 ms).
template <int D>
struct Proj {
    static constexpr int WAVES = D == 256 ? 8 : 4, CG = D / 32, RG = WAVES / CG, TR = 32 * RG, LD = D + 4, NT = 64 * WAVES, NP = TR * D / 4 / NT;
};

template <int D, typename T, bool MUON>
__global__ __launch_bounds__(Proj<D>::NT) void project_kernel(Rows<T, MUON> in, T *out, float *__restrict__ W, int64_t rows,      // (out may be in.X)
                                                              const float *__restrict__ Mt, float keep, float step)
{
    using C = Proj<D>;
    __shared__ __attribute__((aligned(16))) float tile[C::TR * C::LD], res[C::TR * C::LD];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, cg = w % C::CG, rg = w / C::CG, hi = lane >> 5, l31 = lane & 31;
    const int64_t stride = (int64_t)gridDim.x * C::TR, first = (int64_t)blockIdx.x * C::TR, end = rows * D;
    Piece<T, MUON> p[C::NP];
    float4 wt[MUON ? C::NP : 1];
    auto spot = [&](int n) { const int t = tid + C::NT * n; return (t / (D / 4)) * C::LD + 4 * (t % (D / 4)); };
    auto at = [&](int64_t r0, int n) { return r0 * D + 4 * (int64_t)(tid + C::NT * n); };
    auto fetch = [&](int64_t r0) {
#pragma unroll
        for (int n = 0; n < C::NP; ++n) p[n].load(in, at(r0, n), end);
    };
    auto weights = [&](int64_t r0) {
        if constexpr (MUON) {
#pragma unroll
            for (int n = 0; n < C::NP; ++n)
                if (at(r0, n) < end) wt[n] = *reinterpret_cast<const float4 *>(W + at(r0, n));
        }
    };
    fetch(first);
    weights(first);
    float b[D / 2];
#pragma unroll
    for (int j = 0; j < D / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) b[4 * j + e] = Mt[(8 * j + 4 * hi + e) * D + 32 * cg + l31];
    for (int64_t r0 = first; r0 < rows; r0 += stride) {
#pragma unroll
        for (int n = 0; n < C::NP; ++n) *reinterpret_cast<float4 *>(tile + spot(n)) = p[n].template take<false>(in, at(r0, n), end);
        __syncthreads();
        fetch(r0 + stride);
        f32x16 acc;
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[i] = 0.0f;
        const float *a = tile + (32 * rg + l31) * C::LD + 4 * hi;
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
            const float4 x = *reinterpret_cast<const float4 *>(a + 8 * j);
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x.x, b[4 * j], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x.y, b[4 * j + 1], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x.z, b[4 * j + 2], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x.w, b[4 * j + 3], acc, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) res[(32 * rg + (i & 3) + 8 * (i >> 2) + 4 * hi) * C::LD + 32 * cg + l31] = acc[i];
        __syncthreads();                // (every wavefront has read its rows, also before any of them is written where out == X)
#pragma unroll
        for (int n = 0; n < C::NP; ++n) {
            if (at(r0, n) >= end) continue;
            const float4 o = *reinterpret_cast<const float4 *>(res + spot(n));
            if constexpr (MUON) {
                *reinterpret_cast<float4 *>(W + at(r0, n)) = make_float4(fmaf(-step, o.x, keep * wt[n].x), fmaf(-step, o.y, keep * wt[n].y), fmaf(-step, o.z, keep * wt[n].z),
                                                                         fmaf(-step, o.w, keep * wt[n].w));
                if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2 *>(out + at(r0, n)) = make_uint2(0u, 0u);      // out is the gradient: zero for the next step
                else *reinterpret_cast<float4 *>(out + at(r0, n)) = make_float4(0.f, 0.f, 0.f, 0.f);
            } else {
                *reinterpret_cast<float4 *>(out + at(r0, n)) = o;
            }
        }
        weights(r0 + stride);
    }
}

// bf16 rows alone (no optimizer step): v_mfma_f32_32x32x16_bf16 with the matrix in three bf16 planes (24 bits of it: exact products, as good as fp32's; six
// times its rate).  A wavefront holds the planes of its 32 columns (192 registers at d = 256).  20011 x 256: 14 us, 37 with fp32 products.
template <int D>
__global__ __launch_bounds__(Proj<D>::NT, 2) void project_bf16_kernel(const uint16_t *X, uint16_t *out, int64_t rows, const uint4 *__restrict__ Mt)
{
    using C = Proj<D>;
    typedef short bf16x8 __attribute__((ext_vector_type(8)));
    typedef __bf16 frag __attribute__((ext_vector_type(8)));
    constexpr int LD = D + 8, KS = D / 16, NP = C::TR * D / 8 / C::NT;
    __shared__ __attribute__((aligned(16))) uint16_t tile[C::TR * LD], res[C::TR * LD];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, cg = w % C::CG, rg = w / C::CG, hi = lane >> 5, l31 = lane & 31;
    const int64_t stride = (int64_t)gridDim.x * C::TR, first = (int64_t)blockIdx.x * C::TR, end = rows * D;
    uint4 p[NP];
    auto spot = [&](int n) { const int t = tid + C::NT * n; return (t / (D / 8)) * LD + 8 * (t % (D / 8)); };
    auto at = [&](int64_t r0, int n) { return r0 * D + 8 * (int64_t)(tid + C::NT * n); };
    auto fetch = [&](int64_t r0) {
#pragma unroll
        for (int n = 0; n < NP; ++n) p[n] = at(r0, n) < end ? *reinterpret_cast<const uint4 *>(X + at(r0, n)) : make_uint4(0u, 0u, 0u, 0u);
    };
    fetch(first);
    bf16x8 b[KS][3];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int n = 0; n < 3; ++n) b[s][n] = __builtin_bit_cast(bf16x8, Mt[((size_t)cg * KS + s) * 192 + n * 64 + lane]);
    for (int64_t r0 = first; r0 < rows; r0 += stride) {
#pragma unroll
        for (int n = 0; n < NP; ++n) *reinterpret_cast<uint4 *>(tile + spot(n)) = p[n];
        __syncthreads();
        fetch(r0 + stride);
        f32x16 acc;
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[i] = 0.0f;
        const uint16_t *a = tile + (32 * rg + l31) * LD + 8 * hi;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const frag x = __builtin_bit_cast(frag, *reinterpret_cast<const bf16x8 *>(a + 16 * s));
#pragma unroll
            for (int n = 2; n >= 0; --n) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, __builtin_bit_cast(frag, b[s][n]), acc, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) res[(32 * rg + (i & 3) + 8 * (i >> 2) + 4 * hi) * LD + 32 * cg + l31] = f32_bf16(acc[i]);
        __syncthreads();                // (every wavefront has read its rows, also before any of them is written where out == X)
#pragma unroll
        for (int n = 0; n < NP; ++n)
            if (at(r0, n) < end) *reinterpret_cast<uint4 *>(out + at(r0, n)) = *reinterpret_cast<const uint4 *>(res + spot(n));
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------------------
struct OrthoWs {
    double *part, *G, *A, *A2, *P, *W, *M, *M2;      // P: the polynomial T of a step
    void *T;                                     // the result, float or planes (put_result)
    int n_part;
    int64_t bytes;
};

// row ranges: one for every two tiles of 4096 / d rows, at most two workgroups per CU (d = 256: one, by its registers; shared by four: a quarter, whole
// groups of eight)
int gram_pieces(int64_t rows, int d, bool muon)
{
    const int64_t per = 2 * (4096 / d), want = (rows + per - 1) / per;
    if (d == 256 && !muon) return want >= 64 ? 64 : (int)((want + 7) / 8 * 8);
    const int64_t most = d == 256 ? 256 : 512;
    return (int)(want > most ? most : want);
}

OrthoWs ortho_carve(void *ws, int64_t rows, int d, bool muon)
{
    OrthoWs w;
    char *base = (char *)ws;
    int64_t off = 0;
    auto take = [&](int64_t n) { char *q = base + off; off += (n + 255) / 256 * 256; return q; };
    w.n_part = gram_pieces(rows, d, muon);
    const int64_t mat = (int64_t)d * d * 8;
    w.part = (double *)take((int64_t)w.n_part * n_blocks(d) * 2048);
    w.G = (double *)take(mat); w.A = (double *)take(mat); w.A2 = (double *)take(mat); w.P = (double *)take(mat);
    w.W = (double *)take(mat); w.M = (double *)take(mat); w.M2 = (double *)take(mat);
    w.T = take(mat);
    w.bytes = off;
    return w;
}

template <int D, typename O>
void newton_schulz(const OrthoWs &w, O *out, int steps, const Coeffs &k, hipStream_t st)
{
    if (steps == 0) { hipLaunchKernelGGL((ns_identity_kernel<D, O>), dim3(1), dim3(256), 0, st, w.G, out, k.eps); return; }
    if constexpr (D <= 64) {
        hipLaunchKernelGGL((ns_small_kernel<D, O>), dim3(1), dim3(kSmallThreads), 0, st, w.G, out, steps, k);
    } else {
        constexpr int NB = n_blocks(D);
        double *A = w.A, *A2 = w.A2, *M = w.M, *M2 = w.M2;
        for (int s = 0; s < steps; ++s) {
            const bool last = s + 1 == steps;
            if (s == 0) hipLaunchKernelGGL((ns_square_kernel<D, true>), dim3(NB), dim3(256), 0, st, w.G, A, w.P, k);
            else hipLaunchKernelGGL((ns_square_kernel<D, false>), dim3(NB), dim3(256), 0, st, A, (double *)nullptr, w.P, k);
            const dim3 grid(NB, last ? 1 : 2);
            if (s == 0 && last) hipLaunchKernelGGL((ns_times_t_kernel<D, true, O>), grid, dim3(256), 0, st, w.G, A, w.P, M, out, w.W, k.eps);
            else if (s == 0) hipLaunchKernelGGL((ns_times_t_kernel<D, true, double>), grid, dim3(256), 0, st, w.G, A, w.P, M, M2, w.W, k.eps);
            else if (last) hipLaunchKernelGGL((ns_times_t_kernel<D, false, O>), grid, dim3(256), 0, st, w.G, A, w.P, M, out, w.W, k.eps);
            else hipLaunchKernelGGL((ns_times_t_kernel<D, false, double>), grid, dim3(256), 0, st, w.G, A, w.P, M, M2, w.W, k.eps);
            if (!last) hipLaunchKernelGGL(ns_next_kernel<D>, dim3(NB), dim3(256), 0, st, w.W, w.P, A2);
            double *x = A; A = A2; A2 = x;
            x = M; M = M2; M2 = x;
        }
    }
}

template <int D, typename T, bool MUON>
void orthogonalize_d(const Rows<T, MUON> &in, T *out, float *W, int64_t rows, int steps, const Coeffs &k, float keep, float step, const OrthoWs &w, hipStream_t st)
{
    hipLaunchKernelGGL((gram_kernel<D, T, MUON>), dim3(w.n_part * Gram<D, MUON>::SHARE), dim3(512), 0, st, in, rows, w.part);
    hipLaunchKernelGGL(gram_reduce_kernel<D>, dim3(n_blocks(D) * 8), dim3(256), 0, st, w.part, w.n_part, w.G);
    using C = Proj<D>;
    const int64_t tiles = (rows + C::TR - 1) / C::TR;
    auto grid = [&](int per_cu) { const int64_t most = (int64_t)rsx_num_cus() * per_cu; return dim3((unsigned)(tiles < most ? tiles : most)); };
    if constexpr (sizeof(T) == 2 && !MUON) {
        newton_schulz<D>(w, (uint16_t *)w.T, steps, k, st);
        hipLaunchKernelGGL(project_bf16_kernel<D>, grid(D == 256 ? 1 : 3), dim3(C::NT), 0, st, in.X, out, rows, (const uint4 *)w.T);
    } else {
        newton_schulz<D>(w, (float *)w.T, steps, k, st);
        hipLaunchKernelGGL((project_kernel<D, T, MUON>), grid(D == 256 ? 2 : 3), dim3(C::NT), 0, st, in, out, W, rows, (const float *)w.T, keep, step);
    }
}

template <typename T, bool MUON>
void orthogonalize_any(const Rows<T, MUON> &in, T *out, float *W, int64_t rows, int d, int steps, const Coeffs &k, float keep, float step, const OrthoWs &w,
                       hipStream_t st)
{
    switch (d) {
    case 32: orthogonalize_d<32, T, MUON>(in, out, W, rows, steps, k, keep, step, w, st); break;
    case 64: orthogonalize_d<64, T, MUON>(in, out, W, rows, steps, k, keep, step, w, st); break;
    case 128: orthogonalize_d<128, T, MUON>(in, out, W, rows, steps, k, keep, step, w, st); break;
    default: orthogonalize_d<256, T, MUON>(in, out, W, rows, steps, k, keep, step, w, st); break;
    }
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool finite64(double v) { return v - v == 0.0; }

}  // namespace

RSX_API int64_t rsx_orthogonalize_workspace(int64_t rows, int d)
{
    if (rows < 0 || !rsx_dim_ok(d)) return RSX_E_INVALID;
    const int64_t a = ortho_carve(nullptr, rows < 1 ? 1 : rows, d, false).bytes, b = ortho_carve(nullptr, rows < 1 ? 1 : rows, d, true).bytes;
    return a > b ? a : b;
}

RSX_API int rsx_orthogonalize(const void *X, void *out, int64_t rows, int d, int dtype, int steps, double a, double b, double c, double eps, void *ws,
                              int64_t ws_bytes, rsx_stream_t stream)
{
    RSX_CHECK_ARG(X && out, "null pointer");
    RSX_CHECK_ARG(rsx_dim_ok(d), "d must be 32, 64, 128 or 256");
    RSX_CHECK_ARG(rows >= 0, "bad shape");
    RSX_CHECK_ARG(dtype == RSX_F32 || dtype == RSX_BF16, "dtype must be RSX_F32 or RSX_BF16");
    RSX_CHECK_ARG(steps >= 0 && steps <= 32, "steps must be in [0, 32]");
    RSX_CHECK_ARG(finite64(a) && finite64(b) && finite64(c) && finite64(eps) && eps >= 0.0, "coefficients must be finite, eps >= 0");
    RSX_CHECK_ARG(aligned16(X) && aligned16(out), "rows must be 16-byte aligned");
    if (rows == 0) return RSX_OK;
    const OrthoWs w = ortho_carve(ws, rows, d, false);
    if (ws == nullptr || ws_bytes < w.bytes || !aligned16(ws)) {
        rsx_set_error("rsx_orthogonalize: workspace of %lld bytes (16-byte aligned) required, got %lld", (long long)w.bytes, (long long)ws_bytes);
        return RSX_E_WORKSPACE;
    }
    const Coeffs k{a, b, c, eps};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == RSX_F32)
        orthogonalize_any<float, false>({(const float *)X, nullptr, 0.f, 0}, (float *)out, nullptr, rows, d, steps, k, 0.f, 0.f, w, st);
    else
        orthogonalize_any<uint16_t, false>({(const uint16_t *)X, nullptr, 0.f, 0}, (uint16_t *)out, nullptr, rows, d, steps, k, 0.f, 0.f, w, st);
    RSX_CHECK_LAUNCH();
    return RSX_OK;
}

RSX_API int rsx_muon_apply(float *W, float *M, void *G, int64_t rows, int d, int g_dtype, double lr, double momentum, int nesterov, int steps, double a,
                           double b, double c, double eps, double weight_decay, double update_scale, void *ws, int64_t ws_bytes, rsx_stream_t stream)
{
    RSX_CHECK_ARG(W && M && G, "null pointer");
    RSX_CHECK_ARG(rsx_dim_ok(d), "d must be 32, 64, 128 or 256");
    RSX_CHECK_ARG(rows >= 0, "bad shape");
    RSX_CHECK_ARG(g_dtype == RSX_F32 || g_dtype == RSX_BF16, "g_dtype must be RSX_F32 or RSX_BF16");
    RSX_CHECK_ARG(steps >= 0 && steps <= 32, "steps must be in [0, 32]");
    RSX_CHECK_ARG(finite64(a) && finite64(b) && finite64(c) && finite64(eps) && eps >= 0.0, "coefficients must be finite, eps >= 0");
    RSX_CHECK_ARG(finite64(lr) && finite64(weight_decay) && finite64(update_scale) && momentum >= 0.0 && momentum < 1.0, "momentum must be in [0, 1), the rest finite");
    RSX_CHECK_ARG(aligned16(W) && aligned16(M) && aligned16(G), "rows must be 16-byte aligned");
    if (rows == 0) return RSX_OK;
    const OrthoWs w = ortho_carve(ws, rows, d, true);
    if (ws == nullptr || ws_bytes < w.bytes || !aligned16(ws)) {
        rsx_set_error("rsx_muon_apply: workspace of %lld bytes (16-byte aligned) required, got %lld", (long long)w.bytes, (long long)ws_bytes);
        return RSX_E_WORKSPACE;
    }
    const Coeffs k{a, b, c, eps};
    const float keep = (float)(1.0 - lr * weight_decay), step = (float)(lr * update_scale);
    hipStream_t st = (hipStream_t)stream;
    if (g_dtype == RSX_F32)
        orthogonalize_any<float, true>({(const float *)G, M, (float)momentum, nesterov}, (float *)G, W, rows, d, steps, k, keep, step, w, st);
    else
        orthogonalize_any<uint16_t, true>({(const uint16_t *)G, M, (float)momentum, nesterov}, (uint16_t *)G, W, rows, d, steps, k, keep, step, w, st);
    RSX_CHECK_LAUNCH();
    return RSX_OK;
}
