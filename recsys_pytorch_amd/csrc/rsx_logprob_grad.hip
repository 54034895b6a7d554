// rsx_logprob_grad.hip -- gradient of the full-catalog log-probabilities (rsx_logprob.hip) for gfx950 (MI355X).
//
//   dz_ri = scale (sum_t g_rt [i = items_rt] - p_ri (sum_t g_rt + h_r (log p_ri + H_r))),   p_ri = exp(z_ri - lse_r)
//   GP_r = sum_i dz_ri Q_i,   GQ_i = sum_r dz_ri P_r
//
// Neither the scores nor dz exist in memory.  Two passes of one kernel, each recomputing the scores it needs:
//   users stay, items stream   -> GP: the p part; the T rows of Q that the positions name are added when the partial sums are joined
//   items stay, users stream   -> GQ, with the named items inside the tile
// A wavefront keeps 32 columns (users or items) in registers: their operands for the scores and their d sums of the gradient.  Tiles of 32
// streaming rows come through LDS in two forms, copied asynchronously: row-major for the scores, and in the operand order of the
// second product (transposed once, before the pass).  The scores come out of the first product with a column in a lane, which is the
// layout the second product takes its operand in: dz goes from one to the other in registers.  The order of the contraction that this
// fixes (register i of half h is row (i & 3) + 8 (i >> 2) + 4 h) is built into the transposed tiles.
//
// 8 n I d operations instead of the 6 that a stored dz would take, against 3 n I of stored and twice read halves: recomputing is the
// cheaper side from d = 128 down (4096 x 100 000 x 128: 0.4 TFLOP against 2.4 GB).  No atomics: every sum has one order.
//
// dz goes into the second product as halves, one (bf16 tables: 2^-11 of itself, an eighth of what rounding the result to bf16 may take; dz in bf16, as far off
// as the result's rounding, was measured at 2.3e-3 instead of 1.7e-3 of GP) or two (fp32 tables: three products, rsx_logprob.h, on both sides).  A half ends
// at 2^-25 (half its last step), a row's sum may be of probabilities near 1 or of 2^-60: every column keeps a power of two M of its own, and dz |y| / 2^M is
// what is split, y scaled to its row's (32 item rows': rsx_logprob.h) largest element.  M follows the first terms and is raised, with the sums, where a tile
// exceeds it: the largest term of a sum is held at 2^7 or more, the others to 2^-32 of it, whatever other columns, rows or weights are.  Rising costs a maximum of
// the tile's exponents a score and a branch a tile that is hardly taken after the first.  A tile's shares of exponent and sign are in the
// row's parameters: the scores' exponential delivers dz |y| / 2^M as it is.  bf16 rows in scaled halves are what they were down to 2^-31 of their scale.
#include "rsx_logprob.h"

namespace {
using namespace lp;

constexpr float kFar = 1.0e30f;           // log-normaliser of a row without probabilities: every p is 0
// exponents of dz |y| / 2^M: where one is above kTop, M is raised in every column of the wavefront whose largest is above kSet, to that (six binades of room: every
// raise multiplies the sums; kSet 12: 4096 x 100K x 128 1.21 ms, 8: 1.19).  With the entropy's part the exponent is that of p |y| alone, which has to
// stay within fp32's (kGuard, then kGuardSet), and the products' own magnitude is looked at after it
constexpr float kTop = 14.0f, kSet = 8.0f, kGuard = 100.0f, kGuardSet = 90.0f;
constexpr float kNothing = -250.0f;       // exponents below it are not looked at: no sum of such terms is a number of fp32
constexpr int kUnit = 14;                 // rows' scaled elements are in units of 2^-14 of their exponent

struct Args {
    const void *P, *Q;
    const int32_t *user_ids, *items;
    const float *lse, *ent, *g, *h;
    int64_t rows, users, cat;             // positions, user rows, items
    int T;
    float scale;
};

// per tile of 32 positions: [0] factor of its scores (bf16: the same in every row), [1] what is added to them, [2] [3] dz = 2^t (A + B t), [4] .. [7] the first
// four named items (as integers; -1: none): 1 KB, one wavefront's copy.  Without the entropy's part B = 0: [1] is log2 |A| - lse, so that the
// exponential is |dz|, and the sign of A goes with the row's weight (GP) and into the streaming rows (GQ): the same products with one parameter of a row
// instead of three and a multiplication less a score (4096 x 100K x 128 fp32: 1.173 -> 1.161 ms).  The row's exponent is in [1], and taken out of A t.
constexpr int kHeld = 4;
struct Prm {
    float v[4 + kHeld][kTile];
};
// the same of a position that stays: without its row's exponent; w: the exponent of its weight, out of A and B (with the entropy's part)
struct Stay {
    float f, off, A, B, w, pad[3];
};

// e with m in [2^(e - 1), 2^e), and the one of a power of two 2^(e - kUnit) that scale_for made
__device__ __forceinline__ int exponent_of(float m) { return (int)((__float_as_uint(m) >> 23) & 0xFF) - 126; }
__device__ __forceinline__ float exponent_of_factor(float down) { return (float)((int)(__float_as_uint(down) >> 23) - 127 + kUnit); }

// ---- what the passes need -------------------------------------------------------------------------------------------------------------
// one wavefront per position (padded to 128), positions dealt round: coefficients, named items with theirs
template <int D, bool F32>
__global__ __launch_bounds__(256) void rows_kernel(Args a, const uint32_t *__restrict__ bits, int64_t padded, Prm *__restrict__ prm, Stay *__restrict__ stay, float *__restrict__ weight,
                                                   int32_t *__restrict__ named, float *__restrict__ coef)
{
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    for (int64_t r = (int64_t)blockIdx.x * 4 + wid; r < padded; r += (int64_t)gridDim.x * 4) {
        const int32_t u = r < a.rows ? a.user_ids[r] : -1;
        const bool ok = row_ok(u, a.users);
        auto listed = [&](int32_t i) { return (bits[r * mask_words(a.cat) + (i >> 5)] >> (i & 31)) & 1u; };        // is item i among the row's seen items?
        Prm &out = prm[r / kTile];
        const int c = (int)(r % kTile);
        // the row's weight: one order of summation, every lane the same
        double sum = 0.0, mag = 0.0;
        for (int t = 0; t < a.T; ++t) {
            const int32_t i = r < a.rows ? a.items[r * a.T + t] : -1;
            const bool in = ok && i >= 0 && i < a.cat && !(bits != nullptr && listed(i));
            const float g = in ? a.g[r * a.T + t] : 0.0f;
            sum += g;
            mag += fabs((double)g);
            if (lane == 0) {
                if (r < a.rows) named[r * a.T + t] = in ? i : -1;
                if (t < kHeld) out.v[4 + t][c] = __int_as_float(in ? i : -1);
            }
        }
        const float h = ok && a.h != nullptr ? a.h[r] : 0.0f;
        const float lse = ok ? a.lse[r] : -INFINITY;
        const bool live = ok && lse != -INFINITY;
        const float sign = a.h == nullptr && sum > 0.0 ? -1.0f : 1.0f;
        const double w = mag + fabs((double)h);
        float factor = live ? F32 ? 1.0f : a.scale * kLog2e : 0.0f;
        int e_row = 0, e_w = 0;                // exponents of the row and (with the entropy's part) of its weight
        float big = 0.0f, up, down;
        if (ok && lane < D / 8) {
            float x[8];
            load8<F32>(a.P, (int64_t)u * D + 8 * lane, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) big = fmaxf(big, finite_abs(x[j]));
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor(big, o, 64));
        if constexpr (F32) {
            scale_for(big * (a.scale * kLog2e), &up, &down);
            factor *= down;
        }
        scale_for(big, &up, &down);
        e_row = (int)exponent_of_factor(down);
        if (a.h != nullptr) e_w = exponent_of((float)w);
        // dz = p (A + B log2 p), p = 2^(z - lse2).  Without the entropy's part |dz| = 2^(z + off), off = log2 |A| - lse2 in whole 2^-15, to which whole exponents
        // add exactly; what is left (`fix`) goes where the sign goes (bf16 rows stay as they are: rounded to fp32 is enough there).  With it, by t = z + off, off the rounded e - lse2: what the rounding (half a
        // step at 24 is 1e-6 of every p) and e change goes into the coefficients
        const double lse2 = (double)lse * 1.4426950408889634074;
        const double H = a.h != nullptr ? (double)h * a.ent[r < a.rows ? r : 0] : 0.0;
        const double A = live ? ldexp(-(sum + H), -e_w) : 0.0, B = live ? ldexp(-(double)h * kLn2, -e_w) : 0.0;
        const bool none = !live || (a.h == nullptr && sum == 0.0);
        const double exact = log2(fabs(sum)) - lse2;
        const float near = (float)(F32 ? rint(exact * 32768.0) * 0x1p-15 : exact);
        const double fix = F32 && a.h == nullptr && !none ? exp2(exact - (double)near) : 1.0;
        auto params = [&](int e, float *off, float *pa, float *pb) {
            *off = none ? -kFar : near + (float)e;
            *pa = *pb = 0.0f;
            if (a.h == nullptr || none) return;
            const double want = e - lse2;
            *off = (float)want;
            const double d = (double)*off - want, turn = exp2(-d);
            *pa = (float)((A - B * (e + d)) * turn);
            *pb = (float)(B * turn);
        };
        for (int t = lane; t < a.T && r < a.rows; t += 64) {              // (a masked item is not looked up)
            const int32_t i = a.items[r * a.T + t];
            coef[r * a.T + t] = ok && i >= 0 && i < a.cat ? (float)ldexp((double)a.g[r * a.T + t] * sign / fix, e_row) : 0.0f;
        }
        if (lane == 0) {
            Stay q{};
            q.f = factor;
            q.w = (float)e_w;
            params(0, &q.off, &q.A, &q.B);
            stay[r] = q;
            out.v[0][c] = factor;
            params(e_row + e_w, &out.v[1][c], &out.v[2][c], &out.v[3][c]);
            for (int k = a.T; k < kHeld; ++k) out.v[4 + k][c] = __int_as_float(-1);
            weight[r] = live && !(w == 0.0) ? sign * (float)fix : 0.0f;   // (no weight, no gradient; NaN stays NaN)
        }
    }
}

// element order of a transposed tile: [plane][block of 32 columns][half of the rows][lane][8]: lane l, element j is column 32 kb + (l & 31) of
// row (i & 3) + 8 (i >> 2) + 4 (l >> 5), i = 8 half + j
template <int D>
__device__ __forceinline__ int tile_row(int half, int hi, int j) { const int i = 8 * half + j; return (i & 3) + 8 * (i >> 2) + 4 * hi; }

// a tile of 32 rows by 256 threads: row-major planes (bf16 items: the table is that) and the transposed tile.  USERS: rows gathered by user id, each times scale log2 e and with its own
// power of two in the row-major planes, times its own and its sign (0: no weight) in the transposed ones.  Items: the tile's power of two in both, or each row's own
// where they are too unequal (rsx_logprob.h).
template <int D>
struct TileLds {
    float x[kTile][D + 1];
    float range[8], big[kTile], mul[kTile];
};

template <int D, bool F32, bool USERS>
__device__ __forceinline__ void lay_tile(const Args &a, int64_t tile, const float *__restrict__ weight, uint4 *__restrict__ rowm, uint4 *__restrict__ tr, float *__restrict__ factor,
                                         float *__restrict__ row_factor, TileLds<D> &lds)
{
    constexpr int TPR = D / 8;
    auto &x = lds.x;
    float *const s_mul = lds.mul;
    const int tid = threadIdx.x;
    const int64_t n = USERS ? a.rows : a.cat;
    float most = 0.0f, least = INFINITY;  // items: the rows' largest elements, the largest and the smallest of them
    for (int t = tid; t < kTile * TPR; t += 256) {
        const int r = t / TPR, c = 8 * (t % TPR);
        const int64_t at = tile * kTile + r;
        int64_t row = at < n ? at : -1;
        if constexpr (USERS) { const int32_t u = row >= 0 ? a.user_ids[row] : -1; row = row_ok(u, a.users) ? u : -1; }
        const void *src = USERS ? a.P : a.Q;
        float v[8], big = 0.0f, up, down;
        load8<F32>(src, (row < 0 ? 0 : row) * D + c, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) { v[j] = row < 0 ? 0.0f : v[j]; big = fmaxf(big, finite_abs(v[j])); x[r][c + j] = v[j]; }
        big = row_max<TPR>(big);
        if constexpr (USERS) {
            if constexpr (F32) {
                scale_for(big * (a.scale * kLog2e), &up, &down);
                Frag h, l;
                split8_times(v, (double)a.scale * 1.4426950408889634074 * up, &h, &l);
                rowm[(size_t)at * (2 * TPR) + t % TPR] = h.u;
                rowm[(size_t)at * (2 * TPR) + TPR + t % TPR] = l.u;
            } else {
                uint4 y = *reinterpret_cast<const uint4 *>((const uint16_t *)src + (row < 0 ? 0 : row) * D + c);
                if (row < 0) y = make_uint4(0u, 0u, 0u, 0u);
                rowm[(size_t)at * TPR + t % TPR] = y;
            }
            scale_for(big, &up, &down);
            if (c == 0) s_mul[r] = weight[at] * up;
        } else {
            most = fmaxf(most, big);
            least = big > 0.0f ? fminf(least, big) : least;
            if (c == 0) lds.big[r] = big;
        }
    }
    if constexpr (!USERS) {
        tile_range(&most, &least, lds.range);
        const bool own = least * kUneven < most;
        if (tid < kTile) {
            float up, down;
            scale_for(own ? lds.big[tid] : most, &up, &down);
            s_mul[tid] = up;
            row_factor[tile * kTile + tid] = down;
            if (tid == 0) factor[tile] = own ? kOwnScales : down;
        }
        __syncthreads();
        for (int t = tid; F32 && t < kTile * TPR; t += 256) {
            const int r = t / TPR, c = 8 * (t % TPR);
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = x[r][c + j] * s_mul[r];
            Frag h, l;
            split8(v, &h, &l);
            rowm[(size_t)(tile * kTile + r) * (2 * TPR) + t % TPR] = h.u;
            rowm[(size_t)(tile * kTile + r) * (2 * TPR) + TPR + t % TPR] = l.u;
        }
    }
    __syncthreads();
    // the second product multiplies by dz = 0 where a cell is masked: what is not finite is 0 there (where it is not masked, lse is NaN already)
    constexpr int NF = D / 32 * 2 * 64;
    uint4 *dst = tr + (size_t)tile * (NF * (F32 ? 2 : 1));
    for (int t = tid; t < NF; t += 256) {
        const int lane = t & 63, half = (t >> 6) & 1, kb = t >> 7, col = 32 * kb + (lane & 31);
        Frag h, l;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int r = tile_row<D>(half, lane >> 5, j);
            const float y = x[r][col];
            v[j] = (fabsf(y) < INFINITY ? y : 0.0f) * s_mul[r];
        }
        split8(v, &h, &l);
        if constexpr (F32) dst[NF + t] = l.u;
        dst[t] = h.u;
    }
}

// everything before the positions' coefficients, in one launch: workgroups [0, tiles) lay out the item tiles (in the first pass), the rest write a
// position's seen bits each
template <int D, bool F32>
__global__ __launch_bounds__(256) void items_kernel(Args a, const int64_t *__restrict__ indptr, const int32_t *__restrict__ indices, int64_t tiles, uint4 *__restrict__ rowm,
                                                    uint4 *__restrict__ tr, float *__restrict__ factor, float *__restrict__ row_factor, uint32_t *__restrict__ bits)
{
    __shared__ __attribute__((aligned(16))) union { TileLds<D> tile; uint32_t bits[kBitWords]; } lds;
    const int64_t at = blockIdx.x;
    if (at < tiles) {
        lay_tile<D, F32, false>(a, at, nullptr, rowm, tr, factor, row_factor, lds.tile);
        return;
    }
    const int32_t u = a.user_ids[at - tiles];
    write_seen_bits(u, row_ok(u, a.users), indptr, indices, a.cat, bits + (size_t)(at - tiles) * mask_words(a.cat), lds.bits);
}

template <int D, bool F32>
__global__ __launch_bounds__(256) void users_kernel(Args a, const float *__restrict__ weight, uint4 *__restrict__ rowm, uint4 *__restrict__ tr)
{
    __shared__ __attribute__((aligned(16))) TileLds<D> lds;
    lay_tile<D, F32, true>(a, blockIdx.x, weight, rowm, tr, nullptr, nullptr, lds);
}

// ---- the pass -------------------------------------------------------------------------------------------------------------------------
struct Pass {
    const char *stay, *flow;              // row-major planes of what stays in registers and of what streams
    const char *flow_t;                   // transposed tiles of what streams
    const float *tile_factor, *row_factor;      // items: a tile's scale (or kOwnScales), a row's
    const Prm *prm;
    const Stay *stay_prm;
    const uint32_t *bits;
    const int32_t *named;
    const float *coef;
    int64_t stay_rows, flow_tiles;        // valid rows of what stays; tiles that stream
    int64_t flow_valid;                   // valid rows of what streams
    int64_t positions;                    // rows of named / coef / bits
    int64_t cat;
    int T;
    float factor;                         // bf16: scale log2 e
    float *part;                          // [segments][padded rows that stay][d]
    int64_t part_rows;
    int pieces;                           // workgroups of this pass
};

// The work of a pass is a line of (block of 128 columns, streaming tile) cut into equal pieces, one per workgroup of a full device: no ragged last
// round (782 item blocks on 512 slots were two rounds for 1.53).  A block's pieces are its segments, numbered from the first.
__host__ __device__ __forceinline__ int64_t piece_begin(int64_t total, int pieces, int64_t w) { return total * w / pieces; }
// the piece that holds position x of the line: the largest w with piece_begin(w) <= x
__host__ __device__ __forceinline__ int64_t piece_of(int64_t total, int pieces, int64_t x) { return ((x + 1) * pieces - 1) / total; }

template <int D, bool F32>
struct GradGeo : Geo<D, F32> {
    using G = Geo<D, F32>;
    static constexpr int KB = D / 32;
    static constexpr int ST = 16384 / G::TILEB >= 4 ? 4 : 16384 / G::TILEB >= 1 ? 16384 / G::TILEB : 1;       // tiles of one LDS buffer
    // a buffer: row-major tiles, transposed tiles, parameter blocks, and 1 KB of seen bits a tile
    static constexpr int PRM = 2 * ST * G::TILEB, BITS = PRM + ST * 1024, STAGE = BITS + ST * 1024;
    // Workgroups a CU holds, and wavefronts that share 32 columns.  d = 256: the sums of 256 elements are half of a lane's registers at two wavefronts a
    // SIMD.  bf16: two wavefronts take 128 each, and both form the scores (24 products a tile and wavefront instead of 32, two on a SIMD:
    // 1000 x 50021: GP 104 -> 92, GQ 175 -> 157 us); fp32, whose operands take another 128 registers: one a SIMD.
    static constexpr int WGS = D == 256 ? 1 : 2, HS = D == 256 && !F32 ? 2 : 1, NW = 4 * HS, NT = 64 * NW;
};

template <int D, bool F32, bool ITEMS_STAY, bool MASK, bool ENT>
__device__ __forceinline__ void grad_body(const Pass &a, int64_t piece, char *lds0, char *lds1)
{
    using G = GradGeo<D, F32>;
    constexpr int KS = G::KS, NP = G::NP, ST = G::ST, KB = G::KB / G::HS;              // KB: this wavefront's blocks of 32 elements
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wid = wave & 3, half = wave >> 2, hi = lane >> 5, l31 = lane & 31;
    const int64_t total = a.part_rows / 128 * a.flow_tiles;
    int64_t at = piece_begin(total, a.pieces, piece);
    const int64_t end = piece_begin(total, a.pieces, piece + 1);
    const int64_t words = mask_words(a.cat);
    const int sw = G::swz(l31) * 16;

    // Copies of the next ST tiles, 1 KB a wavefront instruction: uniform bases and lane offsets that stay (an address computed per copy
    // would be half of the loop's vector instructions)
    constexpr int NC = ST * G::TILEB / (1024 * G::NW);
    uint32_t off[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        const int o = (n * G::NW + wave) * 1024 + lane * 16, row = o / G::ROWB, c = ((o % G::ROWB) / 16) ^ G::swz(row & 31);
        off[n] = (uint32_t)(row * G::ROWB + 16 * c);
    }
    const uint32_t lane16 = (uint32_t)(lane * 16);
    constexpr bool TABLE = !ITEMS_STAY && !F32;                  // bf16 item rows are the table itself: its last tile may be short
    auto stage = [&](int64_t tile, char *lds, int64_t block, int64_t colc) __attribute__((always_inline)) {
        const char *rows = a.flow + (size_t)tile * G::TILEB, *turned = a.flow_t + (size_t)tile * G::TILEB;
        const int64_t tiles = a.flow_tiles - tile;
        const int64_t left = (a.flow_valid - tile * kTile) * G::ROWB;
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const int k = n * G::NW + wave;
            if (ST > 1 && k * 1024 / G::TILEB >= tiles) continue;
            uint32_t o = off[n];
            if constexpr (TABLE) o = (int64_t)o < left ? o : o % G::ROWB;           // (rows behind the last item: any valid row, they are masked)
            copy_to_lds(rows + o, lds + k * 1024);
            copy_to_lds(turned + k * 1024 + lane16, lds + ST * G::TILEB + k * 1024);
        }
        if constexpr (ITEMS_STAY) {
            if (wave < ST && wave < tiles) copy_to_lds((const char *)(a.prm + tile + wave) + lane16, lds + G::PRM + wave * 1024);
        }
        if constexpr (MASK) {
            if constexpr (ITEMS_STAY) {              // four words of each of the tile's 32 positions: the workgroup's blocks (both halves of a wavefront the same)
                if (wave < ST && wave < tiles) {
                    int64_t r = (tile + wave) * kTile + l31;
                    r = r < a.positions ? r : a.positions - 1;
                    if (hi == 0) copy_to_lds((const char *)(a.bits + (size_t)r * words + 4 * block), lds + G::BITS + wave * 1024);
                }
            } else if (half == 0) {                                  // this wavefront's columns, a word a tile
#pragma unroll
                for (int j = 0; j < ST; ++j) {
                    const int64_t t = tile + j < words ? tile + j : words - 1;
                    copy4_to_lds((const char *)(a.bits + (size_t)(colc < a.positions ? colc : a.positions - 1) * words + t), lds + G::BITS + j * 1024 + wid * 256);
                }
            }
        }
    };
    while (at < end) {
    const int64_t block = at / a.flow_tiles, t0 = at - block * a.flow_tiles;                        // this segment: tiles [t0, t1) of a block
    const int64_t t1 = end - at < a.flow_tiles - t0 ? t0 + (end - at) : a.flow_tiles;
    const int64_t segment = piece - piece_of(total, a.pieces, block * a.flow_tiles);
    const int64_t col = block * 128 + wid * 32 + l31;                                                // this lane's column
    const int64_t colc = col < a.stay_rows ? col : a.stay_rows - 1;
    const int32_t my_block = (int32_t)(block * 4 + wid);                                             // items stay: the block of 32 this wavefront holds
    __syncthreads();                      // (the last segment's tiles are read)
    stage(t0, lds0, block, colc);
    Frag b[KS][NP];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int p = 0; p < NP; ++p) b[s][p].u = *reinterpret_cast<const uint4 *>(a.stay + (size_t)colc * G::ROWB + 16 * (p * (D / 8) + 2 * s + hi));
    f32x16 out[KB];
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
        for (int i = 0; i < 16; ++i) out[k][i] = 0.0f;
    float sf = 0.0f, slse = 0.0f, sA = 0.0f, sB = 0.0f, sE = 0.0f, my_factor = 1.0f;               // users stay: this lane's row; items stay: its row's factor
    if constexpr (!ITEMS_STAY) {
        const Stay &p = a.stay_prm[colc];
        sf = p.f; slse = p.off; sA = p.A; sB = p.B; sE = p.w;
    } else if constexpr (F32) {
        my_factor = a.row_factor[colc];
    }
    float M = 0.0f;                       // this column's: what dz |y| is divided by, as an exponent (a whole number; the same in both lanes of a column)
    float limit = kNothing;               // an exponent above this changes M (until the column has met a term: any)
    // M up by k binades, the sums down.  (fp32 rows of 256: the sums are in accumulation registers, and said to stay there; else the whole loop moves
    // them to and fro for this branch: 1000 x 50021 512 us instead of 411)
    auto raise = [&](float k) __attribute__((always_inline)) {
        const float f = k > 0.0f ? ldexpf(1.0f, -(int)k) : 1.0f;       // (down only before the first term)
#pragma unroll
        for (int q = 0; q < KB; ++q) {
            if constexpr (F32 && D == 256) asm volatile("" : "+a"(out[q]));
#pragma unroll
            for (int i = 0; i < 16; ++i) out[q][i] *= f;
            if constexpr (F32 && D == 256) asm volatile("" : "+a"(out[q]));
        }
        M += k;
    };
    wait_memory();                        // (the operands' loads end here: left to their first use, that wait would stand in the loop, for every stage's copies)
    auto step = [&](int64_t s0, const char *lds, char *next) __attribute__((always_inline)) {
        barrier_after_copies();
        if (s0 + ST < t1) stage(s0 + ST, next, block, colc);
        for (int j = 0; j < ST && s0 + j < t1; ++j) {
            const int64_t tile = s0 + j;
            // (hardly anything in this loop loads into registers from memory: loads return in order, and one waits for the next stage's copies.  What does: the
            // coefficient of a named item that is found, the factors of rows with scales of their own, and, from the fifth of T on, the names: 1024 x 100K x 128
            // fp32 381 us with T = 4, 418 with 10)
            uint32_t seen = 0u;
            if constexpr (MASK) {
                const char *sb = lds + G::BITS + j * 1024;
                seen = ITEMS_STAY ? *reinterpret_cast<const uint32_t *>(sb + l31 * 16 + wid * 4) : *reinterpret_cast<const uint32_t *>(sb + wid * 256 + lane * 4);
            }
            const float tf = ITEMS_STAY ? my_factor : a.tile_factor[tile];
            const char *rm = lds + j * G::TILEB + l31 * G::ROWB;
            const char *tr = lds + ST * G::TILEB + j * G::TILEB + lane * 16;
            __builtin_amdgcn_s_setprio(1);         // (a wavefront in its products goes first: the two of a SIMD fall into step otherwise; 1.19 -> 1.16 ms)
            f32x16 acc;
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[i] = 0.0f;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                Frag x[NP];
#pragma unroll
                for (int p = 0; p < NP; ++p) x[p].u = *reinterpret_cast<const uint4 *>(rm + ((16 * (p * (D / 8) + 2 * s + hi)) ^ sw));
                acc = mfma32<F32>(x[0], b[s][0], acc);
                if constexpr (F32) {
                    acc = mfma32<F32>(x[0], b[s][NP - 1], acc);
                    acc = mfma32<F32>(x[NP - 1], b[s][0], acc);
                }
            }
            __builtin_amdgcn_s_setprio(0);
            // dz of this lane's column and rows (i & 3) + 8 (i >> 2) + 4 hi of the tile: 2^s, or with the entropy's part 2^s (A + B t)
            float v[16];
            float s[16], t[ENT ? 16 : 1];
            float need = 0.0f;                     // sum of the named items' |dz| |y| of this column
            uint64_t hit = 0;                      // which of the T names have one here (bit k & 63)
            if constexpr (!ITEMS_STAY) {
                if (tf < 0.0f) {                   // (kOwnScales: rare, and loads in the loop)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float4 y = *reinterpret_cast<const float4 *>(a.row_factor + tile * kTile + 8 * q + 4 * hi);
                        const float ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float by = exponent_of_factor(ys[e]) + sE - M;
                            const float f = F32 ? sf * ys[e] : sf;
                            if constexpr (ENT) { t[4 * q + e] = fmaf(acc[4 * q + e], f, slse); s[4 * q + e] = t[4 * q + e] + by; }
                            else s[4 * q + e] = fmaf(acc[4 * q + e], f, slse + by);
                        }
                    }
                } else {
                    const float f = F32 ? sf * tf : sf, by = exponent_of_factor(tf) + sE - M, off = slse + by;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        if constexpr (ENT) { t[i] = fmaf(acc[i], f, slse); s[i] = t[i] + by; }
                        else s[i] = fmaf(acc[i], f, off);
                    }
                }
                const int64_t left = a.flow_valid - tile * kTile;
                uint32_t w = left >= 32 ? 0u : 0xFFFFFFFFu << left;
                if constexpr (MASK) w |= seen;
                w >>= 4 * hi;
                if (__builtin_amdgcn_ballot_w64((w & 0x0F0F0F0Fu) != 0u) != 0ull) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const bool none = (w >> ((i & 3) + 8 * (i >> 2))) & 1u;
                        s[i] = none ? -1.0e4f : s[i];
                        if constexpr (ENT) t[i] = none ? 0.0f : t[i];
                    }
                }
            } else {
                const Prm *prm = reinterpret_cast<const Prm *>(lds + G::PRM + j * 1024);
                if (MASK && tile * kTile + l31 >= a.positions) seen = 0xFFFFFFFFu;            // nobody's rows behind the last
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int r0 = 8 * q + 4 * hi;
                    const float4 f4 = F32 ? *reinterpret_cast<const float4 *>(&prm->v[0][r0]) : make_float4(a.factor, a.factor, a.factor, a.factor), l4 = *reinterpret_cast<const float4 *>(&prm->v[1][r0]);
                    const float fs[4] = {f4.x, f4.y, f4.z, f4.w}, ls[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if constexpr (ENT) { t[4 * q + e] = fmaf(acc[4 * q + e], fs[e] * tf, ls[e]); s[4 * q + e] = t[4 * q + e] - M; }
                        else s[4 * q + e] = fmaf(acc[4 * q + e], fs[e] * tf, ls[e] - M);
                    }
                }
                if (MASK && __builtin_amdgcn_ballot_w64(seen != 0u) != 0ull) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const bool none = (__shfl(seen, (i & 3) + 8 * (i >> 2) + 4 * hi, 64) >> l31) & 1u;
                        s[i] = none ? -1.0e4f : s[i];
                        if constexpr (ENT) t[i] = none ? 0.0f : t[i];
                    }
                }
            }
            // named items of the tile's positions that are in this wavefront's block: f(position in the tile, column, what is added to its dz)
            auto named = [&](bool add, auto f) __attribute__((always_inline)) {
                const Prm *prm = reinterpret_cast<const Prm *>(lds + G::PRM + j * 1024);
                for (int k = 0; k < a.T; ++k) {
                    if (add && !((hit >> (k & 63)) & 1)) continue;
                    const int64_t r = tile * kTile + l31;
                    const int32_t it = k < kHeld ? __float_as_int(prm->v[4 + k][l31]) : r < a.positions ? a.named[r * a.T + k] : -1;
                    const bool mine = hi == 0 && (it >> 5) == my_block;          // (-1 >> 5 is nobody's block)
                    unsigned long long hits = __builtin_amdgcn_ballot_w64(mine);
                    if (hits == 0ull) continue;
                    hit |= 1ull << (k & 63);
                    const float c = mine ? a.coef[r * a.T + k] : 0.0f;
                    while (hits) {
                        const int row = __builtin_ctzll(hits);
                        hits &= hits - 1;
                        f(row, __builtin_amdgcn_readlane(it, row) & 31, __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(c), row)));
                    }
                }
            };
            {
                if constexpr (ITEMS_STAY) named(false, [&](int, int at, float c) { need += l31 == at ? fabsf(c) : 0.0f; });
                float most = s[0];
#pragma unroll
                for (int i = 1; i < 16; ++i) most = fmaxf(most, s[i]);
                if (need > 0.0f) most = fmaxf(most, (float)exponent_of(need) - M);
                if (__builtin_amdgcn_ballot_w64(most > limit) != 0ull) {
                    most = fmaxf(most, __shfl_xor(most, 32, 64));
                    constexpr float set = ENT ? kGuardSet : kSet;
                    const float k = most > fminf(limit, set) ? fminf(ceilf(most) - set, 600.0f) : 0.0f;
                    if (most > kNothing) limit = ENT ? kGuard : kTop;
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[i] -= k;
                    raise(k);
                }
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const Prm *prm = reinterpret_cast<const Prm *>(lds + G::PRM + j * 1024);
                float4 a4 = make_float4(sA, sA, sA, sA), b4 = make_float4(sB, sB, sB, sB);
                if constexpr (ENT && ITEMS_STAY) { a4 = *reinterpret_cast<const float4 *>(&prm->v[2][8 * q + 4 * hi]); b4 = *reinterpret_cast<const float4 *>(&prm->v[3][8 * q + 4 * hi]); }
                const float as[4] = {a4.x, a4.y, a4.z, a4.w}, bs[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[4 * q + e] = __builtin_amdgcn_exp2f(s[4 * q + e]);
                    if constexpr (ENT) v[4 * q + e] *= fmaf(bs[e], t[4 * q + e], as[e]);
                }
            }
            if (ITEMS_STAY && hit != 0)
                named(true, [&](int row, int at, float c) {
                    const float add = ldexpf(c, -(int)M);
                    const int reg = (row & 3) | ((row >> 3) << 2);
                    const bool here = lane == at + 32 * ((row >> 2) & 1);
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] += here && i == reg ? add : 0.0f;
                });
            if constexpr (ENT) {
                float most = fabsf(v[0]);
#pragma unroll
                for (int i = 1; i < 16; ++i) most = fmaxf(most, fabsf(v[i]));
                constexpr float over = 32768.0f;       // 2^(kTop + 1)
                if (__builtin_amdgcn_ballot_w64(most > over) != 0ull) {
                    most = fmaxf(most, __shfl_xor(most, 32, 64));
                    const int e = exponent_of(most) - (int)kSet, k = e > 0 ? e : 0;
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] = ldexpf(v[i], -k);
                    raise((float)k);
                }
            }
            // second product: registers 8 h .. 8 h + 7 are the operand of its half h
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                Frag z[NP];
                if constexpr (F32) {
                    split8(v + 8 * h, &z[0], &z[NP - 1]);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const float2v w = {v[8 * h + e], v[8 * h + e + 1]};
                        const half2v y = __builtin_convertvector(w, half2v);
                        z[0].h[e] = y[0]; z[0].h[e + 1] = y[1];
                    }
                }
#pragma unroll
                for (int k = 0; k < KB; ++k) {
                    Frag y[NP];
#pragma unroll
                    for (int p = 0; p < NP; ++p) y[p].u = *reinterpret_cast<const uint4 *>(tr + ((p * G::KB + half * KB + k) * 2 + h) * 1024);
                    out[k] = mfma32<true>(y[0], z[0], out[k]);
                    if constexpr (F32) {
                        out[k] = mfma32<true>(y[0], z[NP - 1], out[k]);
                        out[k] = mfma32<true>(y[NP - 1], z[0], out[k]);
                    }
                }
            }
        }
    };
    // Written out for both buffers, as objects of their own: where one buffer is read and the other filled through the same pointer, the compiler may
    // wait for the copies before it reads.  (fp32 rows of 256: the second copy would spill, and it does not wait there.)
    if constexpr (F32 && D == 256) {
        char *cur = lds0, *next = lds1;
        for (int64_t s0 = t0; s0 < t1; s0 += ST) {
            step(s0, cur, next);
            char *x = cur; cur = next; next = x;
        }
    } else {
        for (int64_t s0 = t0; s0 < t1; s0 += 2 * ST) {
            step(s0, lds0, lds1);
            if (s0 + ST < t1) step(s0 + ST, lds1, lds0);
        }
    }
    float *dst = a.part + ((size_t)segment * a.part_rows + col) * D + 32 * KB * half + 4 * hi;
    const int e = (int)M - kUnit;
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *reinterpret_cast<float4 *>(dst + 32 * k + 8 * q) = make_float4(ldexpf(out[k][4 * q], e), ldexpf(out[k][4 * q + 1], e), ldexpf(out[k][4 * q + 2], e), ldexpf(out[k][4 * q + 3], e));
    at += t1 - t0;
    }
}

// both passes in one launch, the users' first: neither waits for the other's last workgroups (256 x 1682 x 64: 9.6 us for 17 in two)
template <int D, bool F32, bool MASK, bool ENT>
__global__ __launch_bounds__((GradGeo<D, F32>::NT), (GradGeo<D, F32>::WGS * GradGeo<D, F32>::HS)) void grad_kernel(Pass p, Pass q)
{
    __shared__ __attribute__((aligned(1024))) char lds0[GradGeo<D, F32>::STAGE], lds1[GradGeo<D, F32>::STAGE];
    if ((int)blockIdx.x < p.pieces) grad_body<D, F32, false, MASK, ENT>(p, blockIdx.x, lds0, lds1);
    else grad_body<D, F32, true, MASK, ENT>(q, blockIdx.x - p.pieces, lds0, lds1);
}

// segments of a block of 128 columns
__device__ __forceinline__ int segments_of(int64_t block, int64_t flow_tiles, int pieces, int64_t part_rows)
{
    const int64_t total = part_rows / 128 * flow_tiles;
    return (int)(piece_of(total, pieces, (block + 1) * flow_tiles - 1) - piece_of(total, pieces, block * flow_tiles)) + 1;
}

// ---- the partial sums -> the gradients ------------------------------------------------------------------------------------------------------
// GP: four elements a thread; the partials in order, the row's sign (and what its exponent was rounded by), the named rows of Q
template <int D, bool F32>
__device__ __forceinline__ void join_rows(int64_t t, const Args &a, const float *__restrict__ part, int64_t flow_tiles, int pieces, int64_t part_rows, const float *__restrict__ weight,
                                                        const int32_t *__restrict__ named, void *__restrict__ GP)
{
    const int64_t r = t / (D / 4);
    const int c = 4 * (int)(t % (D / 4));
    if (r >= a.rows) return;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    const int segments = weight[r] != 0.0f ? segments_of(r / 128, flow_tiles, pieces, part_rows) : 0;         // (no weight, no gradient, whatever the products were)
#pragma unroll 8
    for (int k = 0; k < segments; ++k) {
        const float4 p = *reinterpret_cast<const float4 *>(part + ((size_t)k * part_rows + r) * D + c);
        s[0] += p.x; s[1] += p.y; s[2] += p.z; s[3] += p.w;
    }
    const float f = weight[r];
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] *= f;
    for (int k = 0; k < a.T; ++k) {
        const int32_t i = named[r * a.T + k];
        if (i < 0) continue;
        const float g = a.g[r * a.T + k];
        if constexpr (F32) {
            const float4 q = *reinterpret_cast<const float4 *>((const float *)a.Q + (size_t)i * D + c);
            s[0] = fmaf(g, q.x, s[0]); s[1] = fmaf(g, q.y, s[1]); s[2] = fmaf(g, q.z, s[2]); s[3] = fmaf(g, q.w, s[3]);
        } else {
            const ushort4 q = *reinterpret_cast<const ushort4 *>((const uint16_t *)a.Q + (size_t)i * D + c);
            s[0] = fmaf(g, bf16_f32(q.x), s[0]); s[1] = fmaf(g, bf16_f32(q.y), s[1]); s[2] = fmaf(g, bf16_f32(q.z), s[2]); s[3] = fmaf(g, bf16_f32(q.w), s[3]);
        }
    }
    if constexpr (F32) *reinterpret_cast<float4 *>((float *)GP + r * D + c) = make_float4(s[0] * a.scale, s[1] * a.scale, s[2] * a.scale, s[3] * a.scale);
    else *reinterpret_cast<ushort4 *>((uint16_t *)GP + r * D + c) = make_ushort4(f32_bf16(s[0] * a.scale), f32_bf16(s[1] * a.scale), f32_bf16(s[2] * a.scale), f32_bf16(s[3] * a.scale));
}

// GQ: the passes' sums in order
struct Passes {
    int64_t flow_tiles, last_tiles;       // streaming tiles of a pass, of the last one
    int passes, pieces, last_pieces;
    int64_t stride;                       // elements of a pass' partial sums
};
template <int D, bool F32>
__device__ __forceinline__ void join_items(int64_t t, int64_t cat, const float *__restrict__ part, const Passes &ps, int64_t part_rows, float scale, void *__restrict__ GQ)
{
    const int64_t r = t / (D / 4);
    const int c = 4 * (int)(t % (D / 4));
    if (r >= cat) return;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    for (int pass = 0; pass < ps.passes; ++pass) {
        const bool last = pass + 1 == ps.passes;
        const int segments = segments_of(r / 128, last ? ps.last_tiles : ps.flow_tiles, last ? ps.last_pieces : ps.pieces, part_rows);
#pragma unroll 4
        for (int k = 0; k < segments; ++k) {
            const float4 p = *reinterpret_cast<const float4 *>(part + (size_t)pass * ps.stride + ((size_t)k * part_rows + r) * D + c);
            s[0] += p.x; s[1] += p.y; s[2] += p.z; s[3] += p.w;
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] *= scale;
    if constexpr (F32) *reinterpret_cast<float4 *>((float *)GQ + r * D + c) = make_float4(s[0], s[1], s[2], s[3]);
    else *reinterpret_cast<ushort4 *>((uint16_t *)GQ + r * D + c) = make_ushort4(f32_bf16(s[0]), f32_bf16(s[1]), f32_bf16(s[2]), f32_bf16(s[3]));
}

// workgroups [0, row_wgs): GP; the rest (after the last pass): GQ
template <int D, bool F32>
__global__ __launch_bounds__(256) void join_kernel(Args a, Pass p, const float *__restrict__ weight, void *__restrict__ GP, int64_t row_wgs, Passes ps, const float *__restrict__ part_q,
                                                   int64_t pad_q, void *__restrict__ GQ)
{
    const int64_t at = blockIdx.x;
    if (at < row_wgs) join_rows<D, F32>(at * 256 + threadIdx.x, a, p.part, p.flow_tiles, p.pieces, p.part_rows, weight, p.named, GP);
    else join_items<D, F32>((at - row_wgs) * 256 + threadIdx.x, a.cat, part_q, ps, pad_q, a.scale, GQ);
}

// ---- T[ids[r]] += R[r] in the order of r -----------------------------------------------------------------------------------------------
// One wavefront per position of a block of kAddRows: the first of the block that names a row adds up all of the block's for it.  Every wavefront looks through
// the block's ids, so the work grows with the square of a block (128 elements a row: 256 rows 11 us, 4096 16, 16384 129, where the bytes take 5).
constexpr int kAddRows = 16384;

template <bool F32>
__global__ __launch_bounds__(256) void add_rows_kernel(float *__restrict__ T, int64_t table_rows, int d, const int32_t *__restrict__ ids, const void *__restrict__ R, int n)
{
    const int r = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (r >= n) return;
    const int32_t id = ids[r];
    if (!row_ok(id, table_rows)) return;
    for (int q = 0; q < r; q += 64)                     // somebody before me?
        if (__builtin_amdgcn_ballot_w64(q + lane < r && ids[q + lane] == id) != 0ull) return;
    float acc[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = 64 * j + lane < d ? T[(size_t)id * d + 64 * j + lane] : 0.0f;
    for (int q = r & ~63; q < n; q += 64) {
        unsigned long long m = __builtin_amdgcn_ballot_w64(q + lane >= r && q + lane < n && ids[q + lane < n ? q + lane : n - 1] == id);
        while (m) {
            const int k = q + __builtin_ctzll(m);
            m &= m - 1;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (64 * j + lane < d) {
                    const size_t at = (size_t)k * d + 64 * j + lane;
                    acc[j] += F32 ? ((const float *)R)[at] : bf16_f32(((const uint16_t *)R)[at]);
                }
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (64 * j + lane < d) T[(size_t)id * d + 64 * j + lane] = acc[j];
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------------
struct Ws {
    char *user_rm, *user_t, *item_rm, *item_t;
    float *tile_factor, *row_factor, *weight, *coef, *part_p, *part_q;
    Prm *prm;
    Stay *stay;
    int32_t *named;
    uint32_t *bits;
    int64_t pass, passes, seg_q, pad_p, pad_q, bytes;
    int wgs, st;
};

int64_t pad128(int64_t n) { return (n + 127) / 128 * 128; }

// workgroups of rows_kernel: four positions each while the chip has room (a chain of loads a position: as many at once as it holds)
int row_groups(int64_t padded)
{
    const int64_t most = 4 * (int64_t)rsx_num_cus();
    return (int)(padded / 4 < most ? padded / 4 : most);
}

// Pieces of a pass, of at least `st` tiles: each of the two passes fills the device, so that the device deals their pieces out as it gets through them; with
// fewer than 16 tiles a piece, where a piece's start and its partial sums cost as much as its tiles, both together (315 x 8135 x 256 fp32, three
// tiles a piece and then six: 90 -> 69 us, 1000 x 20000 x 128 bf16 71 -> 58).
int grad_pieces(int64_t stay, int64_t flow_tiles, int wgs, int st)
{
    const int64_t units = pad128(stay) / 128 * flow_tiles, most = (units + st - 1) / st;
    int64_t slots = (int64_t)wgs * rsx_num_cus();
    if (units < 16 * slots) slots /= 2;
    return (int)(most < slots ? most : slots);
}
// and the segments a block of 128 columns may have then
int64_t grad_segments(int64_t stay, int64_t flow_tiles, int pieces)
{
    const int64_t per = pad128(stay) / 128 * flow_tiles / pieces;            // tiles of a piece, at least
    const int64_t s = (flow_tiles + per - 1) / per + 1;
    return s < pieces ? s : pieces;
}

// geometry the host needs of GradGeo
void grad_geo(int d, bool f32, int *wgs, int *st)
{
    const int tileb = kTile * d * (f32 ? 4 : 2), s = 16384 / tileb;
    *st = s >= 4 ? 4 : s >= 1 ? s : 1;
    *wgs = d == 256 ? 1 : 2;
}

Ws carve(void *ws, int64_t rows, int64_t cat, int d, int dtype, bool mask, int T)
{
    Ws w;
    char *base = (char *)ws;
    int64_t off = 0;
    auto take = [&](int64_t n) { char *q = base + off; off += a256(n); return q; };
    const bool f32 = dtype == RSX_F32;
    const int rowb = d * (f32 ? 4 : 2);
    grad_geo(d, f32, &w.wgs, &w.st);
    // a pass' bits are held to 1 GB (without a mask: one pass)
    int64_t most = (1ll << 30) / (mask_words(cat) * 4) / 128 * 128;
    most = most < 128 ? 128 : most;
    w.pass = mask && rows > most ? most : rows;
    w.passes = (rows + w.pass - 1) / w.pass;
    w.pad_p = pad128(w.pass);
    w.pad_q = pad128(cat);
    const int64_t item_tiles = w.pad_q / kTile, user_tiles = w.pad_p / kTile;
    const int64_t flow = (cat + kTile - 1) / kTile;
    // (the last, shorter pass: fewer tiles in no fewer pieces, so a block has no more segments of items; of users it may have more, over fewer blocks)
    const int64_t tail = rows - (w.passes - 1) * w.pass;
    auto cells_p = [&](int64_t n) { return grad_segments(n, flow, grad_pieces(n, flow, w.wgs, w.st)) * pad128(n); };
    auto seg_q = [&](int64_t n) { return grad_segments(cat, pad128(n) / kTile, grad_pieces(cat, pad128(n) / kTile, w.wgs, w.st)); };
    const int64_t cells = cells_p(w.pass) > cells_p(tail) ? cells_p(w.pass) : cells_p(tail);
    w.seg_q = seg_q(w.pass) > seg_q(tail) ? seg_q(w.pass) : seg_q(tail);
    w.user_rm = take(w.pad_p * rowb);
    w.user_t = take(w.pad_p * rowb);
    w.item_rm = take(f32 ? w.pad_q * rowb : 0);
    w.item_t = take(w.pad_q * rowb);
    w.tile_factor = (float *)take(item_tiles * 4);
    w.row_factor = (float *)take(w.pad_q * 4);
    w.weight = (float *)take(w.pad_p * 4);
    w.coef = (float *)take(w.pass * T * 4);
    w.named = (int32_t *)take(w.pass * T * 4);
    w.prm = (Prm *)take(user_tiles * (int64_t)sizeof(Prm));
    w.stay = (Stay *)take(w.pad_p * (int64_t)sizeof(Stay));
    w.bits = (uint32_t *)take(mask ? w.pass * mask_words(cat) * 4 : 0);
    w.part_p = (float *)take(cells * d * 4);
    w.part_q = (float *)take(w.passes * w.seg_q * w.pad_q * d * 4);
    w.bytes = off;
    return w;
}

template <int D, bool F32>
void run(const Args &all, const int64_t *indptr, const int32_t *indices, const Ws &w, void *GP, void *GQ, hipStream_t st)
{
    const int es = F32 ? 4 : 2;
    Passes ps{0, 0, (int)w.passes, 0, 0, w.seg_q * w.pad_q * D};
    for (int64_t k = 0; k < w.passes; ++k) {
        Args a = all;
        const int64_t r0 = k * w.pass;
        a.rows = all.rows - r0 < w.pass ? all.rows - r0 : w.pass;
        a.user_ids += r0; a.lse += r0; a.g += r0 * a.T; a.items += r0 * a.T;
        if (a.ent) a.ent += r0;
        if (a.h) a.h += r0;
        const int64_t pad = pad128(a.rows), user_tiles = pad / kTile, item_tiles = k == 0 ? w.pad_q / kTile : 0, bit_rows = indptr ? a.rows : 0;
        if (item_tiles + bit_rows > 0)
            hipLaunchKernelGGL((items_kernel<D, F32>), dim3((unsigned)(item_tiles + bit_rows)), dim3(256), 0, st, a, indptr, indices, item_tiles, (uint4 *)w.item_rm, (uint4 *)w.item_t,
                               w.tile_factor, w.row_factor, w.bits);
        hipLaunchKernelGGL((rows_kernel<D, F32>), dim3((unsigned)row_groups(pad)), dim3(256), 0, st, a, indptr ? w.bits : (const uint32_t *)nullptr, pad, w.prm, w.stay, w.weight, w.named, w.coef);
        hipLaunchKernelGGL((users_kernel<D, F32>), dim3((unsigned)user_tiles), dim3(256), 0, st, a, w.weight, (uint4 *)w.user_rm, (uint4 *)w.user_t);
        Pass p;                               // users stay
        p.tile_factor = w.tile_factor; p.row_factor = w.row_factor; p.prm = w.prm; p.stay_prm = w.stay; p.bits = w.bits; p.named = w.named; p.coef = w.coef;
        p.positions = a.rows; p.cat = a.cat; p.T = a.T; p.factor = a.scale * kLog2e;
        p.stay = w.user_rm; p.flow = F32 ? w.item_rm : (const char *)a.Q; p.flow_t = w.item_t;
        p.stay_rows = pad; p.flow_tiles = (a.cat + kTile - 1) / kTile; p.flow_valid = a.cat;
        p.part = w.part_p; p.part_rows = pad;
        p.pieces = grad_pieces(a.rows, p.flow_tiles, w.wgs, w.st);
        Pass q = p;                           // items stay
        q.stay = F32 ? w.item_rm : (const char *)a.Q; q.flow = w.user_rm; q.flow_t = w.user_t;
        q.stay_rows = F32 ? w.pad_q : a.cat; q.flow_tiles = user_tiles; q.flow_valid = a.rows;
        q.part = w.part_q + (size_t)k * w.seg_q * w.pad_q * D; q.part_rows = w.pad_q;
        q.pieces = grad_pieces(a.cat, user_tiles, w.wgs, w.st);
#define RSX_GRAD(M_, E_) hipLaunchKernelGGL((grad_kernel<D, F32, M_, E_>), dim3((unsigned)(p.pieces + q.pieces)), dim3(GradGeo<D, F32>::NT), 0, st, p, q)
        if (indptr) { if (a.h) RSX_GRAD(true, true); else RSX_GRAD(true, false); }
        else { if (a.h) RSX_GRAD(false, true); else RSX_GRAD(false, false); }
#undef RSX_GRAD
        if (k == 0) { ps.flow_tiles = user_tiles; ps.pieces = q.pieces; }
        ps.last_tiles = user_tiles; ps.last_pieces = q.pieces;
        const int64_t joins = (a.rows * (D / 4) + 255) / 256, item_joins = k + 1 == w.passes ? (a.cat * (D / 4) + 255) / 256 : 0;
        hipLaunchKernelGGL((join_kernel<D, F32>), dim3((unsigned)(joins + item_joins)), dim3(256), 0, st, a, p, w.weight, (char *)GP + r0 * D * es, joins, ps, w.part_q, w.pad_q,
                           GQ);
    }
}

}  // namespace

RSX_API int64_t rsx_score_logprobs_grad_workspace(int64_t num_rows, int64_t num_items, int d, int dtype, int masked, int T)
{
    if (num_rows < 0 || num_rows >= (1ll << 31) - 128 || num_items <= 0 || num_items >= (1ll << 31) - 128 || !rsx_dim_ok(d) || (dtype != RSX_F32 && dtype != RSX_BF16) || T < 0)
        return RSX_E_INVALID;
    return carve(nullptr, num_rows < 1 ? 1 : num_rows, num_items, d, dtype, masked != 0, T).bytes;
}

RSX_API int rsx_score_logprobs_grad(const void *P, int64_t num_users, const int32_t *user_ids_dev, int64_t num_rows, const void *Q, int64_t num_items, int d,
                                    int dtype, const int64_t *mask_indptr_dev, const int32_t *mask_indices_dev, float scale, const int32_t *items_dev, int T,
                                    const float *lse_dev, const float *g_logp_dev, const float *entropy_dev, const float *g_entropy_dev, void *GP_out,
                                    void *GQ_out, void *ws, int64_t ws_bytes, rsx_stream_t stream)
{
    RSX_CHECK_ARG(P && Q && user_ids_dev && lse_dev && GP_out && GQ_out, "null pointer");
    RSX_CHECK_ARG(rsx_dim_ok(d), "d must be 32, 64, 128 or 256");
    RSX_CHECK_ARG(dtype == RSX_F32 || dtype == RSX_BF16, "dtype must be RSX_F32 or RSX_BF16");
    RSX_CHECK_ARG(num_rows >= 1 && num_rows < (1ll << 31) - 128 && num_users > 0 && num_items > 0 && num_items < (1ll << 31) - 128, "bad shape");
    RSX_CHECK_ARG((mask_indptr_dev == nullptr) == (mask_indices_dev == nullptr), "mask needs both CSR arrays");
    RSX_CHECK_ARG((entropy_dev == nullptr) == (g_entropy_dev == nullptr), "the entropies and their gradients come together");
    RSX_CHECK_ARG(scale > 0.0f && scale < INFINITY, "scale must be positive and finite");
    RSX_CHECK_ARG(T >= 0 && (T == 0 || (items_dev && g_logp_dev)), "T items per row need their ids and gradients");
    RSX_CHECK_ARG(T > 0 || g_entropy_dev != nullptr, "nothing to differentiate");
    RSX_CHECK_ARG(aligned16(P) && aligned16(Q) && aligned16(GP_out) && aligned16(GQ_out), "table rows must be 16-byte aligned");
    RSX_CHECK_ARG(GP_out != GQ_out && GP_out != P && GP_out != Q && GQ_out != P && GQ_out != Q, "the gradients need memory of their own");
    const Ws w = carve(ws, num_rows, num_items, d, dtype, mask_indptr_dev != nullptr, T);
    if (ws == nullptr || ws_bytes < w.bytes || !aligned16(ws)) {
        rsx_set_error("rsx_score_logprobs_grad: workspace of %lld bytes (16-byte aligned) required, got %lld", (long long)w.bytes, (long long)ws_bytes);
        return RSX_E_WORKSPACE;
    }
    const Args a{P, Q, user_ids_dev, items_dev, lse_dev, entropy_dev, g_logp_dev, g_entropy_dev, num_rows, num_users, num_items, T, scale};
    hipStream_t st = (hipStream_t)stream;
#define RSX_GRAD_RUN(D_) do { if (dtype == RSX_F32) run<D_, true>(a, mask_indptr_dev, mask_indices_dev, w, GP_out, GQ_out, st); \
                              else run<D_, false>(a, mask_indptr_dev, mask_indices_dev, w, GP_out, GQ_out, st); } while (0)
    switch (d) {
    case 32: RSX_GRAD_RUN(32); break;
    case 64: RSX_GRAD_RUN(64); break;
    case 128: RSX_GRAD_RUN(128); break;
    default: RSX_GRAD_RUN(256); break;
    }
#undef RSX_GRAD_RUN
    RSX_CHECK_LAUNCH();
    return RSX_OK;
}

RSX_API int rsx_add_rows(float *T, int64_t table_rows, int d, const int32_t *ids_dev, const void *R, int dtype, int64_t n, rsx_stream_t stream)
{
    RSX_CHECK_ARG(T && ids_dev && R, "null pointer");
    RSX_CHECK_ARG(rsx_dim_ok(d), "d must be 32, 64, 128 or 256");
    RSX_CHECK_ARG(dtype == RSX_F32 || dtype == RSX_BF16, "dtype must be RSX_F32 or RSX_BF16");
    RSX_CHECK_ARG(table_rows > 0 && n >= 0, "bad shape");
    if (n == 0) return RSX_OK;
    for (int64_t r0 = 0; r0 < n; r0 += kAddRows) {
        const int m = (int)(n - r0 < kAddRows ? n - r0 : kAddRows);
        const void *src = (const char *)R + (size_t)r0 * d * (dtype == RSX_F32 ? 4 : 2);
        if (dtype == RSX_F32) hipLaunchKernelGGL(add_rows_kernel<true>, dim3((m + 3) / 4), dim3(256), 0, (hipStream_t)stream, T, table_rows, d, ids_dev + r0, src, m);
        else hipLaunchKernelGGL(add_rows_kernel<false>, dim3((m + 3) / 4), dim3(256), 0, (hipStream_t)stream, T, table_rows, d, ids_dev + r0, src, m);
    }
    RSX_CHECK_LAUNCH();
    return RSX_OK;
}
