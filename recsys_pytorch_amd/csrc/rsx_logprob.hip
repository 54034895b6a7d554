// rsx_logprob.hip -- log-probabilities of given items under the softmax over the whole catalog, with entropy and the K most probable
// items, for gfx950 (MI355X).
//
//   z_ri = scale <P[u_r], Q_i>  (-inf where masked),  lse_r = log sum_i exp z_ri,  logp_rt = z_r,items[r,t] - lse_r,
//   H_r = lse_r - sum_i p_ri z_ri,  top = the K largest z_ri (ties: lowest id)
//
// The [rows x items] scores never exist in memory.  One pass over the catalog keeps, per row, a running reference m, the sum of
// 2^(t - m) and the sum of (t - m) 2^(t - m) with t = z log2 e; they are rescaled only when a tile exceeds m by 2^16, so the common
// path is one fused multiply-add, one v_exp_f32 and two accumulations per score.  The products are laid out so that a lane holds
// scores of ONE row (items are the matrix instruction's rows, users its columns): all of this is lane-local.
//
// Top-K: the pass also stores the largest score of every 8 items as a half (relative to a score of the same row, so that halves
// resolve it; -inf only where all 8 are masked).  The K best items lie in chunks whose maximum is at least the K-th largest maximum, less what halves and fast
// products are off by; finish_kernel takes the chunks from there up, computes their items' products again in 64 bits and orders those.  What the fast
// products' rounding could swap is decided by the 64-bit ones.
//
// Two forms of the pass:
//   thin_kernel  few rows: the catalog is read once, straight into registers (v_mfma_f32_16x16x4_f32 / 16x16x32_bf16), bound by HBM (16 rows, 1M x 128
//                bf16: 256 MB in 42 us)
//   wide_kernel  many rows: item tiles through LDS (asynchronous copies, two buffers), users' operands held in registers for the whole
//                pass (up to 128 registers a lane), bound by the matrix cores (fp32: three f16 products, rsx_logprob.h) or, for bf16
//                rows of 128, by the five vector instructions a score needs after its product (8192 x 100K: 0.34 ms, 0.16 of it
//                products; 1024 x 100K fp32: 94 us, 55 of it products)
#include "rsx_logprob.h"

namespace {
using namespace lp;

constexpr int kMaxK = 128;
// Blocks of 32 users a wavefront holds: two in bf16, where an item operand read from LDS then serves two products; one in fp32, where it
// serves two of the three products anyway, twice the workgroups fill the chip better, and a wavefront leaves registers to spare (1024 x 100K x
// 128 fp32: 182 us with two, 166 with one; 8192 x 100K x 128 bf16: 493 with two, 520 with one and twice the wavefronts a SIMD)
constexpr int users_block(bool f32) { return f32 ? 1 : 2; }
constexpr int kWaves = 2;                // wavefronts a SIMD that the registers are cut for (three: 169 us in fp32)
constexpr float kNone = -3.0e38f;        // reference of a row that has met no score yet
constexpr float kLazy = 16.0f;           // a tile's maximum may exceed the reference by this much before the sums are rescaled

struct Shape {
    const int32_t *user_ids;
    int64_t rows, users, items;
    float scale;
};

// running sums of one row, in units of log2: in fp32 over a tile or a group of tiles, in 64 bits over those (equal terms round the same way: a
// few hundred groups in fp32 were off by 3e-6)
template <typename T>
struct StatOf {
    float m;
    T sum, ent;
};
typedef StatOf<float> Stat;
typedef StatOf<double> LongStat;

template <typename T>
__device__ __forceinline__ void stat_lift(StatOf<T> &s, float top)      // new reference max(m, top)
{
    const float m = fmaxf(s.m, top);
    const float r = __builtin_amdgcn_exp2f(s.m - m);
    s.ent = s.sum > 0 ? (T)r * fma(s.sum, (T)(s.m - m), s.ent) : s.ent;      // (0 * inf for a row that has met nothing: skipped.  NaN sums: kept)
    s.sum = s.sum * (T)r;
    s.m = m;
}

// reference score of a row for the chunk maxima: the median of three items' scores, 0 if that is not finite
__device__ __forceinline__ float pick_reference(float a, float b, float c)
{
    const float m = __builtin_amdgcn_fmed3f(a, b, c);
    return fabsf(m) < 1.0e30f ? m : 0.0f;
}

// chunk maxima as halves, two at a time.  Rounded towards zero: what lies beyond a half's range stays finite (+-65504; the ties this makes are told apart by
// their products in 64 bits), and -inf is left to the chunks that hold nothing
__device__ __forceinline__ uint32_t key_bits(float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b)); }

// the reference a row's chunk maxima are stored against: a score of its own, so that an offset common to a row's scores does not eat the halves'
// eleven bits; and how far apart two of its fast products may be off: twice 3 (d + 1) 2^-24 sum |x||y|, of the middle one of the same three items (a
// bound that no roundings reach, with room for items a few times as long).  One wavefront per row.
template <int D, bool F32>
__device__ __forceinline__ void row_reference(const void *__restrict__ P, const void *__restrict__ Q, const Shape &sh, int64_t r, float *__restrict__ ref, float *__restrict__ slack)
{
    const int lane = threadIdx.x & 63;
    if (r >= sh.rows) return;
    const int32_t u = sh.user_ids[r];
    if (!row_ok(u, sh.users)) return;
    float d[3] = {0.0f, 0.0f, 0.0f}, size[3] = {0.0f, 0.0f, 0.0f};
    if (lane < D / 8) {
        float x[8], q[8];
        load8<F32>(P, (int64_t)u * D + 8 * lane, x);
#pragma unroll
        for (int n = 0; n < 3; ++n) {
            load8<F32>(Q, (n == 0 ? 0 : n == 1 ? sh.items / 2 : sh.items - 1) * D + 8 * lane, q);
#pragma unroll
            for (int j = 0; j < 8; ++j) { d[n] = fmaf(x[j], q[j], d[n]); size[n] = fmaf(fabsf(x[j]), fabsf(q[j]), size[n]); }
        }
    }
#pragma unroll
    for (int n = 0; n < 3; ++n)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) { d[n] += __shfl_xor(d[n], o, 64); size[n] += __shfl_xor(size[n], o, 64); }
    if (lane == 0) {
        ref[r] = sh.scale * kLog2e * pick_reference(d[0], d[1], d[2]);
        slack[r] = sh.scale * kLog2e * (6 * (D + 1) * 0x1p-24f) * pick_reference(size[0], size[1], size[2]);
    }
}

// what the pass needs, in one launch: workgroups [0, tiles) split the item tiles (fp32), the next bit_rows write a row's seen bits each, the rest
// the references of four rows each.  (As three launches: 943 x 1682 x 64 took 5 us longer, of 50.)
template <int D, bool F32>
__global__ __launch_bounds__(256) void prepare_kernel(const void *__restrict__ P, const void *__restrict__ Q, Shape sh, const int64_t *__restrict__ indptr,
                                                      const int32_t *__restrict__ indices, int64_t tiles, int64_t bit_rows, uint4 *__restrict__ planes, float *__restrict__ factor,
                                                      float *__restrict__ row_factor, uint32_t *__restrict__ bits, float *__restrict__ ref, float *__restrict__ slack)
{
    __shared__ __attribute__((aligned(16))) uint32_t lds[kBitWords];
    int64_t at = blockIdx.x;
    if (at < tiles) {
        if constexpr (F32) split_items<D>((const float *)Q, sh.items, at, planes, factor, row_factor, reinterpret_cast<float *>(lds));
        return;
    }
    at -= tiles;
    if (at < bit_rows) {
        const int32_t u = sh.user_ids[at];
        write_seen_bits(u, row_ok(u, sh.users), indptr, indices, sh.items, bits + (size_t)at * mask_words(sh.items), lds);
        return;
    }
    row_reference<D, F32>(P, Q, sh, (at - bit_rows) * 4 + (threadIdx.x >> 6), ref, slack);
}

// ---- many rows ------------------------------------------------------------------------------------------------------------------------
template <int D, bool F32>
struct WideGeo : Geo<D, F32> {
    using G = Geo<D, F32>;
    // 32-user blocks a wavefront holds: their operands take KS * NP * 4 registers each
    static constexpr int UB = users_block(F32), WGU = 128 * UB, OCC = kWaves;
    // item tiles of one of the two LDS buffers
    static constexpr int ST = 16384 / G::TILEB >= 4 ? 4 : 16384 / G::TILEB >= 1 ? 16384 / G::TILEB : 1;
};

// chunk maxima of a row, 16 halves per group of four tiles: [hi][tile & 3][h] holds items 32 tile + 16 h + 4 hi + {0..3, 8..11}
__device__ __forceinline__ int64_t chunk_item0(int64_t c)
{
    return (4 * (c >> 4) + ((c >> 1) & 3)) * kTile + 16 * (c & 1) + 4 * ((c >> 3) & 1);
}

template <int D, bool F32, bool MASK, bool TOP>
struct WideLds {
    using G = WideGeo<D, F32>;
    __attribute__((aligned(1024))) char tile[2][G::ST * G::TILEB];
    char bits[MASK ? 2 : 1][MASK ? 4 : 1][G::UB][512];        // a group's seen bits, 16 bytes a row of the wavefront's
    uint32_t key[G::UB][TOP ? 4 : 1][256];                    // a group's chunk maxima, this lane's own slots
    float top[G::UB][256];                                    // reference and sums of all groups before this one, this lane's own slots
    double sum[G::UB][256], ent[G::UB][256];
};

// the products' 16 scores of one row (register i: item (i & 3) + 8 (i >> 2) + 4 hi of the tile) into the group's sums.  SOME: bits of w mask some.
// (Two whole versions rather than a masked copy of the scores before one: merging the copies would cost the common path 16 moves.)
template <bool SOME, bool TOP>
__device__ __forceinline__ void absorb(const f32x16 &acc, float f, uint32_t w, Stat &st, float ref, uint32_t *key)
{
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = SOME && ((w >> ((i & 3) + 8 * (i >> 2))) & 1u) ? -INFINITY : acc[i];
    float c0 = x[0], c1 = x[8];
#pragma unroll
    for (int i = 1; i < 8; ++i) { c0 = __builtin_elementwise_maximum(c0, x[i]); c1 = __builtin_elementwise_maximum(c1, x[8 + i]); }
    const float top = __builtin_elementwise_maximum(c0, c1) * f;
    if constexpr (TOP) *key = key_bits(fmaf(c0, f, -ref), fmaf(c1, f, -ref));
    if (__builtin_amdgcn_ballot_w64(top > st.m + kLazy) != 0ull) {
        if (top > st.m) stat_lift(st, top);
    }
    float sum = 0.0f, ent = 0.0f;         // of the tile; then of the group, then (in 64 bits) of all
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float t = fmaf(x[i], f, -st.m);
        if constexpr (SOME) t = x[i] == -INFINITY ? -1.0e4f : t;
        const float e = __builtin_amdgcn_exp2f(t);
        sum += e;
        ent = fmaf(e, t, ent);
    }
    st.sum += sum;
    st.ent += ent;
}

template <int D, bool F32, bool MASK, bool TOP>
__device__ __forceinline__ void wide_body(const void *__restrict__ P, const char *__restrict__ rows, const float *__restrict__ factor, const float *__restrict__ row_factor, const Shape &sh,
                                          const uint32_t *__restrict__ bits, const float *__restrict__ row_ref, int splits, float4 *__restrict__ part,
                                          uint4 *__restrict__ keys, WideLds<D, F32, MASK, TOP> &lds)
{
    using G = WideGeo<D, F32>;
    constexpr int UB = G::UB, KS = G::KS, NP = G::NP, ST = G::ST;
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, hi = lane >> 5, l31 = lane & 31;
    const int64_t groups = (sh.items + 127) / 128;
    const int64_t g0 = groups * blockIdx.x / splits, g1 = groups * (blockIdx.x + 1) / splits;
    const int64_t row0 = (int64_t)blockIdx.y * G::WGU + wid * (32 * UB);

    // this wavefront's users: operands, scale, reference
    Frag b[UB][KS][NP];
    float rowf[UB], ref[UB];
    Stat st[UB];                          // of the current group of tiles
#pragma unroll
    for (int ub = 0; ub < UB; ++ub) {
        const int64_t r = row0 + 32 * ub + l31;
        const int32_t u = sh.user_ids[r < sh.rows ? r : sh.rows - 1];
        const bool ok = row_ok(u, sh.users);
        const int64_t at = (int64_t)(ok ? u : 0) * D + 8 * hi;
        float up = 1.0f, down = 1.0f;
        if constexpr (F32) {
            float m = 0.0f;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                float x[8];
                load8<F32>(P, at + 16 * s, x);
#pragma unroll
                for (int j = 0; j < 8; ++j) m = fmaxf(m, finite_abs(x[j]));
            }
            scale_for(fmaxf(m, __shfl_xor(m, 32, 64)) * (sh.scale * kLog2e), &up, &down);
        }
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            if constexpr (F32) {
                float x[8];
                load8<F32>(P, at + 16 * s, x);
                split8_times(x, (double)sh.scale * 1.4426950408889634074 * up, &b[ub][s][0], &b[ub][s][NP - 1]);
            } else {
                b[ub][s][0].u = *reinterpret_cast<const uint4 *>((const uint16_t *)P + at + 16 * s);
            }
        }
        rowf[ub] = !ok ? 0.0f : F32 ? down : sh.scale * kLog2e;      // (fp32: scale log2 e is in the operands, the factor a power of two)
        ref[ub] = TOP && ok ? row_ref[r < sh.rows ? r : sh.rows - 1] : 0.0f;
        st[ub] = {kNone, 0.0f, 0.0f};
        lds.top[ub][tid] = kNone;
        lds.sum[ub][tid] = lds.ent[ub][tid] = 0.0;
    }

    // copies of the next ST tiles: 1 KB a wavefront instruction, lane-linear in LDS, the swizzle in the source address.  (Nothing in the loop loads into
    // registers from memory: loads return in order, and one would wait for the next stage's copies.)
    constexpr int NC = (ST * G::TILEB / 1024 + 3) / 4;
    uint32_t off[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        const int o = ((n * 4 + wid) * 1024 + lane * 16) % (ST * G::TILEB), row = o / G::ROWB, c = ((o % G::ROWB) / 16) ^ G::swz(row & 31);
        off[n] = (uint32_t)(row * G::ROWB + 16 * c);
    }
    const int64_t words = mask_words(sh.items), tiles = (sh.items + kTile - 1) / kTile;
    auto stage = [&](int64_t tile, int buf) {
        const int64_t t = F32 || tile < tiles ? tile : tiles - 1;                // (the planes of fp32 tables are padded to groups)
        const char *base = rows + (size_t)t * G::TILEB;
        const int64_t left = (sh.items - t * kTile) * G::ROWB;
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            if ((NC * 4 - 3) * 1024 > ST * G::TILEB && (n * 4 + wid) * 1024 >= ST * G::TILEB) break;
            uint32_t o = off[n];
            if constexpr (!F32) o = (int64_t)o < left ? o : o % G::ROWB;          // rows behind the last item: any valid row, they are masked
            copy_to_lds(base + o, lds.tile[buf] + (n * 4 + wid) * 1024);
        }
        if constexpr (MASK) {
            if ((tile & 3) == 0) {
#pragma unroll
                for (int ub = 0; ub < UB; ++ub) {
                    const int64_t r = row0 + 32 * ub + l31;
                    if (hi == 0) copy_to_lds((const char *)(bits + (size_t)(r < sh.rows ? r : sh.rows - 1) * words + tile), lds.bits[(tile >> 2) & 1][wid][ub]);
                }
            }
        }
    };
    const int hs = (16 * hi) ^ (G::swz(l31) * 16);
    if (g0 < g1) stage(4 * g0, 0);
    int buf = 0;
    for (int64_t g = g0; g < g1; ++g) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t tile = 4 * g + j;
            if (j % ST == 0) {
                barrier_after_copies();  // this stage's tiles are there; everyone is done with the other buffer
                if (TOP && j == 0 && g > g0) {        // the last group's maxima, ahead of the copies so that the next barrier finds them done
#pragma unroll
                    for (int ub = 0; ub < UB; ++ub) {
                        const int64_t r = row0 + 32 * ub + l31;
                        if (r < sh.rows)
                            keys[(size_t)r * (2 * groups) + 2 * (g - 1) + hi] = make_uint4(lds.key[ub][0][tid], lds.key[ub][1 % (TOP ? 4 : 1)][tid], lds.key[ub][2 % (TOP ? 4 : 1)][tid], lds.key[ub][3 % (TOP ? 4 : 1)][tid]);
                    }
                }
                if (j + ST < 4 || g + 1 < g1) stage(tile + ST, buf ^ 1);
                buf ^= 1;
            }
            const char *t0 = lds.tile[buf ^ 1] + (j % ST) * G::TILEB + l31 * G::ROWB;
            f32x16 acc[UB];
#pragma unroll
            for (int ub = 0; ub < UB; ++ub)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[ub][i] = 0.0f;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                Frag a[NP];
#pragma unroll
                for (int p = 0; p < NP; ++p) a[p].u = *reinterpret_cast<const uint4 *>(t0 + ((p * (2 * D) + 32 * s) ^ hs));
#pragma unroll
                for (int ub = 0; ub < UB; ++ub) acc[ub] = mfma32<F32>(a[0], b[ub][s][0], acc[ub]);
                if constexpr (F32) {
#pragma unroll
                    for (int ub = 0; ub < UB; ++ub) acc[ub] = mfma32<F32>(a[0], b[ub][s][1], acc[ub]);
#pragma unroll
                    for (int ub = 0; ub < UB; ++ub) acc[ub] = mfma32<F32>(a[1], b[ub][s][0], acc[ub]);
                }
            }
            // the tile's operands are read from LDS AHEAD steps before their products
            constexpr int AHEAD = 2;
            __builtin_amdgcn_sched_group_barrier(0x100, (KS < AHEAD ? KS : AHEAD) * NP, 0);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                __builtin_amdgcn_sched_group_barrier(0x008, (F32 ? 3 : 1) * UB, 0);
                if (s + AHEAD < KS) __builtin_amdgcn_sched_group_barrier(0x100, NP, 0);
            }
            const float tf = F32 ? factor[tile] : 1.0f;
            const int64_t left = sh.items - tile * kTile;
            const uint32_t none = left >= 32 ? 0u : left <= 0 ? 0xFFFFFFFFu : 0xFFFFFFFFu << left;
#pragma unroll
            for (int ub = 0; ub < UB; ++ub) {
                uint32_t w = none;
                if constexpr (MASK) w |= *reinterpret_cast<const uint32_t *>(lds.bits[g & 1][wid][ub] + l31 * 16 + j * 4);
                w >>= 4 * hi;
                uint32_t *key = &lds.key[ub][j % (TOP ? 4 : 1)][tid];
                if (F32 && tf < 0.0f) {       // (kOwnScales: rare, and the only loads of the loop)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float4 v = *reinterpret_cast<const float4 *>(row_factor + tile * kTile + 8 * q + 4 * hi);
                        acc[ub][4 * q] *= rowf[ub] * v.x; acc[ub][4 * q + 1] *= rowf[ub] * v.y; acc[ub][4 * q + 2] *= rowf[ub] * v.z; acc[ub][4 * q + 3] *= rowf[ub] * v.w;
                    }
                    absorb<true, TOP>(acc[ub], 1.0f, w, st[ub], ref[ub], key);
                } else if (__builtin_amdgcn_ballot_w64((w & 0x0F0F0F0Fu) != 0u) == 0ull) absorb<false, TOP>(acc[ub], rowf[ub] * tf, 0u, st[ub], ref[ub], key);
                else absorb<true, TOP>(acc[ub], rowf[ub] * tf, w, st[ub], ref[ub], key);
            }
        }
#pragma unroll
        for (int ub = 0; ub < UB; ++ub) {
            LongStat all = {lds.top[ub][tid], lds.sum[ub][tid], lds.ent[ub][tid]};
            if (__builtin_amdgcn_ballot_w64(st[ub].m > all.m) != 0ull) stat_lift(all, st[ub].m);
            lds.top[ub][tid] = all.m;
            lds.sum[ub][tid] = all.sum + (double)st[ub].sum;
            lds.ent[ub][tid] = all.ent + (double)st[ub].ent;
            st[ub].sum = st[ub].ent = 0.0f;
        }
    }
    // the two halves of a row, then the row's partial of this split
#pragma unroll
    for (int ub = 0; ub < UB; ++ub) {
        const int64_t r = row0 + 32 * ub + l31;
        if (TOP && g1 > g0 && r < sh.rows)
            keys[(size_t)r * (2 * groups) + 2 * (g1 - 1) + hi] = make_uint4(lds.key[ub][0][tid], lds.key[ub][1 % (TOP ? 4 : 1)][tid], lds.key[ub][2 % (TOP ? 4 : 1)][tid], lds.key[ub][3 % (TOP ? 4 : 1)][tid]);
        LongStat all = {lds.top[ub][tid], lds.sum[ub][tid], lds.ent[ub][tid]};
        LongStat o = {__shfl_xor(all.m, 32, 64), __shfl_xor(all.sum, 32, 64), __shfl_xor(all.ent, 32, 64)};
        const float m = fmaxf(all.m, o.m);
        stat_lift(all, m);
        stat_lift(o, m);
        if (hi == 0 && r < sh.rows) part[(size_t)r * splits + blockIdx.x] = make_float4(m, (float)(all.sum + o.sum), (float)(all.ent + o.ent), 0.0f);
    }
}

template <int D, bool F32, bool MASK, bool TOP>
__global__ __launch_bounds__(256, (WideGeo<D, F32>::OCC)) void wide_kernel(const void *__restrict__ P, const char *__restrict__ rows, const float *__restrict__ factor,
                                                                           const float *__restrict__ row_factor, Shape sh, const uint32_t *__restrict__ bits, const float *__restrict__ row_ref, int splits,
                                                                           float4 *__restrict__ part, uint4 *__restrict__ keys)
{
    __shared__ WideLds<D, F32, MASK, TOP> lds;
    wide_body<D, F32, MASK, TOP>(P, rows, factor, row_factor, sh, bits, row_ref, splits, part, keys, lds);
}

// ---- few rows ---------------------------------------------------------------------------------------------------------------------------
// A wavefront takes 32-item tiles in two halves of 16 rows.  Row m of half h of a tile is item 16 (m >> 3) + 4 ((m >> 2) & 1) + (m & 3) + 8 h:
// lane (user l & 15, g = l >> 4) then holds, over both halves, exactly one chunk of wide_kernel's numbering (h = g >> 1, hi = g & 1).
template <int D, bool F32, int UB, bool MASK, bool TOP>
__global__ __launch_bounds__(256) void thin_kernel(const void *__restrict__ P, const void *__restrict__ Q, Shape sh, const uint32_t *__restrict__ bits,
                                                   const float *__restrict__ row_ref, float4 *__restrict__ part, uint16_t *__restrict__ keys)
{
    constexpr int NL = F32 ? D / 16 : D / 32;              // 16-byte loads of a lane per item row
    constexpr int EPL = F32 ? 4 : 8;                       // elements of one
    __shared__ float4 s_part[4][16 * UB];
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, g = lane >> 4, l15 = lane & 15;
    const int64_t tiles = (sh.items + kTile - 1) / kTile;

    auto load = [&](const void *t, int64_t row, int n) { return *reinterpret_cast<const u32x4 *>((const char *)t + (size_t)row * (D * (F32 ? 4 : 2)) + n * 64 + g * 16); };
    u32x4 b[UB][NL];
    float rowf[UB], ref[UB];
    LongStat st[UB];
#pragma unroll
    for (int ub = 0; ub < UB; ++ub) {
        const int64_t r = 16 * ub + l15;
        const int32_t u = sh.user_ids[r < sh.rows ? r : sh.rows - 1];
        const bool ok = row_ok(u, sh.users);
#pragma unroll
        for (int n = 0; n < NL; ++n) b[ub][n] = load(P, ok ? u : 0, n);
        rowf[ub] = ok ? sh.scale * kLog2e : 0.0f;
        ref[ub] = TOP && ok ? row_ref[r < sh.rows ? r : sh.rows - 1] : 0.0f;
        st[ub] = {kNone, 0.0f, 0.0f};
    }
    const int64_t words = mask_words(sh.items), groups = (sh.items + 127) / 128;
    const int irow = 16 * (l15 >> 3) + 4 * ((l15 >> 2) & 1) + (l15 & 3);
    const int64_t step = (int64_t)gridDim.x * 4;
    const int64_t first = (int64_t)blockIdx.x * 4 + wid;
    u32x4 a[2][NL];
    auto fetch = [&](int64_t tile, int h) {
        int64_t i = tile * kTile + irow + 8 * h;
        i = i < sh.items ? i : sh.items - 1;
#pragma unroll
        for (int n = 0; n < NL; ++n) a[h][n] = load(Q, i, n);
    };
    if (first < tiles) { fetch(first, 0); fetch(first, 1); }
    for (int64_t tile = first; tile < tiles; tile += step) {
        uint32_t w[UB];
        const int64_t left = sh.items - tile * kTile;
        const uint32_t none = left >= 32 ? 0u : 0xFFFFFFFFu << left;
#pragma unroll
        for (int ub = 0; ub < UB; ++ub) {
            w[ub] = none;
            if constexpr (MASK) {
                const int64_t r = 16 * ub + l15;
                w[ub] |= bits[(size_t)(r < sh.rows ? r : sh.rows - 1) * words + tile];
            }
        }
        f32x4 acc[2][UB];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int ub = 0; ub < UB; ++ub) acc[h][ub] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int n = 0; n < NL; ++n) {
#pragma unroll
                for (int ub = 0; ub < UB; ++ub) {
                    if constexpr (F32) {
#pragma unroll
                        for (int e = 0; e < EPL; ++e)
                            acc[h][ub] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[h][n][e]), __uint_as_float(b[ub][n][e]), acc[h][ub], 0, 0, 0);
                    } else {
                        acc[h][ub] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[h][n]), __builtin_bit_cast(bf16x8, b[ub][n]), acc[h][ub], 0, 0, 0);
                    }
                }
            }
            if (tile + step < tiles) fetch(tile + step, h);        // (into the half that was just used up)
        }
#pragma unroll
        for (int ub = 0; ub < UB; ++ub) {
            const float f = rowf[ub];
            // result layout of the 16 x 16 instruction: register i of lane l is row 4 (l >> 4) + i
            const uint32_t ws = w[ub] >> (16 * (g >> 1) + 4 * (g & 1));
            const bool any = __builtin_amdgcn_ballot_w64((ws & 0x0F0Fu) != 0u) != 0ull;
            float x[8];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) x[4 * h + i] = any && ((ws >> (8 * h + i)) & 1u) ? -INFINITY : acc[h][ub][i];
            float c = x[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) c = fmaxf(c, x[i]);
            const float top = c * f;
            if constexpr (TOP) {
                const int64_t r = 16 * ub + l15;
                if (r < sh.rows) keys[(size_t)r * (16 * groups) + 16 * (tile >> 2) + 8 * (g & 1) + 2 * (tile & 3) + (g >> 1)] = (uint16_t)key_bits(fmaf(c, f, -ref[ub]), 0.0f);
            }
            if (__builtin_amdgcn_ballot_w64(top > st[ub].m + kLazy) != 0ull) {
                if (top > st[ub].m) stat_lift(st[ub], top);
            }
            float sum = 0.0f, ent = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float t = x[i] == -INFINITY ? -1.0e4f : fmaf(x[i], f, -st[ub].m);
                const float e = __builtin_amdgcn_exp2f(t);
                sum += e;
                ent = fmaf(e, t, ent);
            }
            st[ub].sum += (double)sum;
            st[ub].ent += (double)ent;
        }
    }
    // four lanes and four wavefronts hold a row
#pragma unroll
    for (int ub = 0; ub < UB; ++ub) {
#pragma unroll
        for (int o = 16; o <= 32; o <<= 1) {
            LongStat q = {__shfl_xor(st[ub].m, o, 64), __shfl_xor(st[ub].sum, o, 64), __shfl_xor(st[ub].ent, o, 64)};
            const float m = fmaxf(st[ub].m, q.m);
            stat_lift(st[ub], m);
            stat_lift(q, m);
            st[ub].sum += q.sum;
            st[ub].ent += q.ent;
        }
        if (g == 0) s_part[wid][16 * ub + l15] = make_float4(st[ub].m, (float)st[ub].sum, (float)st[ub].ent, 0.f);
    }
    __syncthreads();
    if (tid < 16 * UB && tid < sh.rows) {
        Stat s = {kNone, 0.f, 0.f};
        float m = kNone;
        for (int q = 0; q < 4; ++q) m = fmaxf(m, s_part[q][tid].x);
        s.m = m;
        for (int q = 0; q < 4; ++q) {
            Stat o = {s_part[q][tid].x, s_part[q][tid].y, s_part[q][tid].z};
            stat_lift(o, m);
            s.sum += o.sum;
            s.ent += o.ent;
        }
        part[(size_t)tid * gridDim.x + blockIdx.x] = make_float4(s.m, s.sum, s.ent, 0.f);
    }
    // chunk maxima behind the last tile of a group: none
    if constexpr (TOP) {
        if (blockIdx.x == 0) {
            const int spare = (int)(4 * groups - tiles);
            for (int64_t t = tid; t < sh.rows * spare * 4; t += 256) {
                const int64_t r = t / (spare * 4), q = t % (spare * 4), tile = tiles + q / 4;
                keys[(size_t)r * (16 * groups) + 16 * (tile >> 2) + 8 * (q & 1) + 2 * (tile & 3) + ((q >> 1) & 1)] = 0xFC00u;      // -inf
            }
        }
    }
}

// ---- one workgroup per row: join the partials, the given items, the K best -------------------------------------------------------------
constexpr int kMaxChunks = 256;                   // chunks whose items are computed again; more (a row of zeros, ties by the thousand): the whole row is, by its one
                                                  // workgroup (100K x 128: 1.5 ms, ten times what 1024 rows without such a one take)
constexpr int kCand = 8 * kMaxChunks;
constexpr int kListed = 4096;                     // chunks looked at more closely for that choice
static_assert(kListed * 4 <= kCand * 8 && kListed * 2 <= kCand * 4, "the list of chunks lies in the candidates' memory");

// (score, id) order: larger score first, then lower id
__device__ __forceinline__ bool before(double sa, int32_t ia, double sb, int32_t ib) { return sa > sb || (sa == sb && ia < ib); }

template <int NT>
__device__ void sort_candidates(double *s, int32_t *id, int n)          // descending; n <= kCand entries, padded here to a power of two
{
    int n2 = 1;
    while (n2 < n) n2 <<= 1;
    for (int t = n + threadIdx.x; t < n2; t += NT) { s[t] = -INFINITY; id[t] = 0x7FFFFFFF; }
    __syncthreads();
    for (int size = 2; size <= n2; size <<= 1)
        for (int stride = size >> 1; stride > 0; stride >>= 1) {
            for (int t = threadIdx.x; t < n2 / 2; t += NT) {
                const int lo = 2 * t - (t & (stride - 1)), hi = lo + stride;
                const bool down = (lo & size) == 0;
                if (before(s[hi], id[hi], s[lo], id[lo]) == down) {
                    const double x = s[lo]; s[lo] = s[hi]; s[hi] = x;
                    const int32_t y = id[lo]; id[lo] = id[hi]; id[hi] = y;
                }
            }
            __syncthreads();
        }
}

__device__ __forceinline__ half2v max2(half2v a, half2v b) { return __builtin_elementwise_max(a, b); }      // (NaN: the other)
__device__ __forceinline__ half2v as_half2(uint32_t w) { return __builtin_bit_cast(half2v, w); }
__device__ __forceinline__ uint32_t half_order(_Float16 v)                                                  // halves -> ordered integers
{
    const uint32_t h = __builtin_bit_cast(uint16_t, v);
    return (h & 0x8000u) ? (~h & 0xFFFFu) : (h | 0x8000u);
}
__device__ __forceinline__ float half_value(uint32_t order)
{
    const uint16_t h = (uint16_t)((order & 0x8000u) ? order & 0x7FFFu : ~order);
    return (float)__builtin_bit_cast(_Float16, h);
}

// a stored maximum less what it may be off by: a half's last place twice (the maximum's, and the bound's own) and the fast products
__device__ __forceinline__ float surely_above(float h, float slack) { return h - (fabsf(h) * 0.003f + 0x1p-23f + slack); }

// EPL elements of a table row as they lie in memory
template <bool F32, int EPL>
struct RowPiece {
    uint4 lo, hi;                                             // (16 bytes: lo alone)
    __device__ __forceinline__ float at(int j) const
    {
        const uint32_t a[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        return F32 ? __uint_as_float(a[j]) : __uint_as_float(j & 1 ? a[j / 2] & 0xFFFF0000u : a[j / 2] << 16);
    }
};
template <bool F32, int EPL>
__device__ __forceinline__ RowPiece<F32, EPL> load_piece(const void *base, int64_t at)
{
    RowPiece<F32, EPL> v{};
    const uint4 *src = reinterpret_cast<const uint4 *>((const char *)base + at * (F32 ? 4 : 2));
    v.lo = src[0];
    if constexpr (F32 && EPL == 8) v.hi = src[1];
    return v;
}

// sum over groups of LPI neighbouring lanes, in their last one
template <int LPI>
__device__ __forceinline__ float group_sum(float v)
{
#define RSX_DPP_ADD(ctrl_) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl_, 0xF, 0xF, true))
    RSX_DPP_ADD(0x111);                                       // row_shr:1
    RSX_DPP_ADD(0x112);
    if constexpr (LPI >= 8) RSX_DPP_ADD(0x114);
    if constexpr (LPI >= 16) RSX_DPP_ADD(0x118);
#undef RSX_DPP_ADD
    if constexpr (LPI >= 32) v += __shfl_up(v, 16, 64);
    if constexpr (LPI >= 64) v += __shfl_up(v, 32, 64);
    return v;
}

// NT threads a row: 1024 where rows are few and one row's chain of loads is the time, 512 up to two rows a CU, 256 where more rows share a CU (whole call,
// 300 x 50K x 256: 144 us with 256, 130 with 512, 154 with 1024; 943 x 1682 x 64: 46 with 256, 60 with 512)
template <int D, bool F32, int NT>
__global__ __launch_bounds__(NT, (NT >= 512 ? 4 : F32 ? 5 : 6)) void finish_kernel(const void *__restrict__ P, const void *__restrict__ Q, Shape sh, const uint32_t *__restrict__ bits,
                                                    const float4 *__restrict__ part, int splits, double skew, const uint16_t *__restrict__ keys,
                                                    const float *__restrict__ row_ref, const float *__restrict__ row_slack, const int32_t *__restrict__ given, int T, int K, float *__restrict__ logp,
                                                    float *__restrict__ lse_out, float *__restrict__ ent_out, int32_t *__restrict__ top_idx, float *__restrict__ top_logp)
{
    // elements of an item's row a lane takes, lanes a row, items a pass.  fp32: eight where the work of many rows is the time (fewer additions between lanes:
    // 943 x 1682 x 64 48 -> 43 us, 600 x 50K x 256 167 -> 149), four where one row's chain is (34.1 us a call against 35.4)
    constexpr int EPL = F32 && NT == 1024 ? 4 : 8, LPI = D / EPL, IPP = NT / LPI;
    // the maxima from the bound up are read again, by the few threads that have any, instead of kept: a sixth wavefront a SIMD fits (4000 x 20K x 64 bf16 102 ->
    // 97 us; fp32, whose rows take more registers, would spill: 2000 x 50K x 128 150 -> 158)
    constexpr bool AGAIN = !F32 && NT == 256;
    constexpr int NW = NT / 64, KR = NT == 1024 ? 16 : 8, FL = NT == 1024 ? 8 : 4;                               // wavefronts; 16-byte loads of maxima a thread keeps; item rows on the way together
    __shared__ __attribute__((aligned(16))) double c_s[kCand];
    __shared__ __attribute__((aligned(16))) int32_t c_id[kCand];
    __shared__ double s_red[3][NW];
    __shared__ __attribute__((aligned(16))) uint16_t s_max[256];
    __shared__ int32_t s_list[kMaxChunks];
    int32_t *const s_item = c_id;                  // (item e is read where its id is written back: the same value)
    __shared__ int s_n, s_count;
    __shared__ uint32_t s_tau;
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    const int64_t r = blockIdx.x;
    const int32_t u = sh.user_ids[r];
    if (!row_ok(u, sh.users)) {                    // no row: nothing is probable, nothing has a log-probability
        for (int t = tid; t < T; t += NT) logp[r * T + t] = 0.0f;
        for (int t = tid; t < K; t += NT) { top_idx[r * K + t] = -1; top_logp[r * K + t] = -INFINITY; }
        if (tid == 0) { if (lse_out) lse_out[r] = -INFINITY; if (ent_out) ent_out[r] = 0.0f; }
        return;
    }
    // everything that is known to be needed is asked for at once: the maxima of the chunks, the user's row, the partials
    const int64_t chunks = (sh.items + 127) / 128 * 16;
    const uint16_t *key = keys + (size_t)r * chunks;
    uint4 kept[KR];
    auto fetch = [&](int64_t base) {               // maxima base + 8 (tid + NT n) ..
#pragma unroll
        for (int n = 0; n < KR; ++n) {
            const int64_t c = base + 8 * ((int64_t)tid + NT * n);
            kept[n] = c < chunks ? *reinterpret_cast<const uint4 *>(key + c) : make_uint4(0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u);
        }
    };
    if (K > 0) fetch(0);
    const int li = tid % LPI;
    double p[EPL];
    auto piece = [&](const void *base, int64_t row) { return load_piece<F32, EPL>(base, row * D + EPL * li); };
    {
        const RowPiece<F32, EPL> v = piece(P, u);
#pragma unroll
        for (int j = 0; j < EPL; ++j) p[j] = (double)v.at(j);
    }
    float pf[EPL];
#pragma unroll
    for (int j = 0; j < EPL; ++j) pf[j] = (float)p[j];

    // the partials, in 64 bits
    float4 mine = make_float4(kNone, 0.f, 0.f, 0.f);
    if (tid < splits) mine = part[r * splits + tid];
    double m = mine.x, sum = 0.0, ent = 0.0;
    for (int s = tid + NT; s < splits; s += NT) m = fmax(m, (double)part[r * splits + s].x);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmax(m, __shfl_xor(m, o, 64));
    if (lane == 0) s_red[0][wid] = m;
    if (tid == 0) s_n = 0;
    __syncthreads();
    m = s_red[0][0];
#pragma unroll
    for (int w = 1; w < NW; ++w) m = fmax(m, s_red[0][w]);
    for (int s = tid; s < splits; s += NT) {
        const float4 q = s == tid ? mine : part[r * splits + s];
        if (q.y == 0.0f) continue;                 // (met nothing; NaN sums are kept)
        const double w = exp2((double)q.x - m);
        sum += w * q.y;
        ent += w * ((double)q.z + (double)q.y * ((double)q.x - m));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) { sum += __shfl_xor(sum, o, 64); ent += __shfl_xor(ent, o, 64); }
    if (lane == 0) { s_red[1][wid] = sum; s_red[2][wid] = ent; }
    __syncthreads();
    sum = ent = 0.0;
#pragma unroll
    for (int w = 0; w < NW; ++w) { sum += s_red[1][w]; ent += s_red[2][w]; }
    const double l2 = log2(sum);
    // the pass multiplied by a factor that is off by `skew` of itself: to first order (skew^2 is 2^-46) the normaliser is off by that of the mean score
    const double mean = m + ent / sum, late = mean - mean == 0.0 ? skew * mean : 0.0;
    const double lse = sum == 0.0 ? -INFINITY : kLn2 * (m + l2 - late);
    if (tid == 0) {
        if (lse_out) lse_out[r] = (float)lse;
        if (ent_out) ent_out[r] = sum == 0.0 ? 0.0f : (float)(kLn2 * (l2 - ent / sum));
    }

    const int64_t words = mask_words(sh.items);
    const uint32_t *seen = bits ? bits + (size_t)r * words : nullptr;
    auto masked = [&](int32_t i) { return seen != nullptr && ((seen[i >> 5] >> (i & 31)) & 1u); };
    // FL items at a time
    auto dots = [&](const int32_t (&i)[FL], double (&z)[FL]) {
        RowPiece<F32, EPL> v[FL];
#pragma unroll
        for (int n = 0; n < FL; ++n) v[n] = piece(Q, i[n]);
#pragma unroll
        for (int n = 0; n < FL; ++n) {
            z[n] = 0.0;
#pragma unroll
            for (int j = 0; j < EPL; ++j) z[n] = fma(p[j], (double)v[n].at(j), z[n]);
        }
#pragma unroll
        for (int o = LPI / 2; o > 0; o >>= 1)
#pragma unroll
            for (int n = 0; n < FL; ++n) z[n] += __shfl_xor(z[n], o, LPI);
#pragma unroll
        for (int n = 0; n < FL; ++n) z[n] *= (double)sh.scale;
    };

    // The chunks whose maximum may be among the K largest: those from a little below the K-th largest up.  First a lower bound of that maximum: the K-th largest of the
    // threads' own (no fewer chunks can be above it); then the chunks from a little below the bound up, the K-th largest among them, and those from there up
    int n = 0;                                     // entries: T given items, then 8 for each chosen chunk
    float cut = -INFINITY;                         // a score that K items reach, by the stored maxima
    bool whole = false;                            // too many ties: every item of the row is computed
    if (K > 0) {
        const half2v none = as_half2(0xFC00FC00u);                                                  // -inf: nothing in the chunk
        const uint32_t lowest = half_order(none[0]);
        half2v top8 = none;
        for (int64_t base = 0; base < chunks; base += 8ll * NT * KR) {
            if (base > 0) fetch(base);
#pragma unroll
            for (int n_ = 0; n_ < KR; ++n_)
                top8 = max2(top8, max2(max2(as_half2(kept[n_].x), as_half2(kept[n_].y)), max2(as_half2(kept[n_].z), as_half2(kept[n_].w))));
        }
        uint32_t best = half_order(top8[0]);       // this thread's largest (NT > 256: that of NT / 256 threads)
        { const uint32_t x = half_order(top8[1]); best = x > best ? x : best; }
        if constexpr (NT > 256) {                  // 256 maxima, of NT / 256 threads each
#pragma unroll
            for (int o = 1; o < NT / 256; o <<= 1) { const uint32_t x = __shfl_xor(best, o, 64); best = x > best ? x : best; }
        }
        if (tid % (NT / 256) == 0) s_max[tid / (NT / 256)] = (uint16_t)best;
        __syncthreads();
        const float slack = row_slack[r];
        // a maximum's order -> that of the smallest one that may belong to a larger score (-inf, a chunk with nothing in it, never does)
        auto from = [&](uint32_t order) {
            const uint32_t low = half_order((_Float16)__builtin_bit_cast(half2v, key_bits(surely_above(half_value(order), slack), 0.0f))[0]);
            return order <= lowest || low <= lowest ? lowest + 1 : low < order ? low : order;        // (NaN and infinities: themselves)
        };
        if (wid == 0) {                            // the K-th largest of 256, bit by bit, in one wavefront
            const uint2 v = reinterpret_cast<const uint2 *>(s_max)[lane];
            const uint32_t x[4] = {v.x & 0xFFFFu, v.x >> 16, v.y & 0xFFFFu, v.y >> 16};
            uint32_t t = 0;
            for (int bit = 15; bit >= 0; --bit) {
                const uint32_t u_ = t | (1u << bit);
                int c = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) c += __builtin_popcountll(__builtin_amdgcn_ballot_w64(x[j] >= u_));
                if (c >= K) t = u_;
            }
            if (lane == 0) s_tau = from(t);
        }
        __syncthreads();
        int32_t *const l_chunk = reinterpret_cast<int32_t *>(c_s);
        uint16_t *const l_key = reinterpret_cast<uint16_t *>(c_id);
        const uint32_t bound = s_tau;
        const _Float16 bound_h = (_Float16)half_value(bound);
        for (int64_t base = 0; base < chunks; base += 8ll * NT * KR) {
            if (AGAIN ? best >= bound : chunks > 8ll * NT * KR) fetch(base);
            else if (AGAIN) continue;
#pragma unroll
            for (int n_ = 0; n_ < KR; ++n_) {
                const half2v m2 = max2(max2(as_half2(kept[n_].x), as_half2(kept[n_].y)), max2(as_half2(kept[n_].z), as_half2(kept[n_].w)));
                if (m2[0] < bound_h && m2[1] < bound_h) continue;
                const uint32_t w[4] = {kept[n_].x, kept[n_].y, kept[n_].z, kept[n_].w};
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t k = half_order(as_half2(w[j / 2])[j & 1]);
                    if (k >= bound) {
                        const int at = atomicAdd(&s_n, 1);
                        if (at < kListed) { l_chunk[at] = (int32_t)(base + 8 * ((int64_t)tid + NT * n_) + j); l_key[at] = (uint16_t)k; }
                    }
                }
            }
        }
        __syncthreads();
        const int listed = s_n;
        __syncthreads();                           // (s_n is counted anew below)
        if (tid == 0) { s_n = listed <= kListed ? 0 : listed; s_tau = 0xFFFFu; }
        if (tid < 8 && listed <= 1024) l_key[listed + tid] = 0;              // (read eight at a time)
        __syncthreads();
        if (listed <= 1024) {
            for (int q = tid; q < listed; q += NT) {
                const uint32_t k = l_key[q];
                int over = 0;
                for (int t = 0; t < listed; t += 8) {
                    const uint4 v = *reinterpret_cast<const uint4 *>(l_key + t);
                    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) over += ((w[j] & 0xFFFFu) > k) + ((w[j] >> 16) > k);
                }
                if (over < K) atomicMin(&s_tau, k);                      // the K-th largest maximum, from above
            }
        } else if (listed <= kListed) {            // (the best items' chunks were few threads': the K-th bit by bit)
            uint32_t tau = 0;
            for (int bit = 15; bit >= 0; --bit) {
                const uint32_t t = tau | (1u << bit);
                if (tid == 0) s_count = 0;
                __syncthreads();
                int c = 0;
                for (int q = tid; q < listed; q += NT) c += l_key[q] >= t;
                if (c) atomicAdd(&s_count, c);
                __syncthreads();
                if (s_count >= K) tau = t;
                __syncthreads();
            }
            if (tid == 0) s_tau = tau;
        }
        __syncthreads();
        if (listed <= kListed) {
            const uint32_t least = from(s_tau);
            for (int q = tid; q < listed; q += NT)
                if (l_key[q] >= least) {
                    const int at = atomicAdd(&s_n, 1);
                    if (at < kMaxChunks) s_list[at] = l_chunk[q];
                }
        }
        __syncthreads();
        whole = s_n > kMaxChunks;
        n = whole ? 0 : 8 * s_n;
        // K items reach the K-th maximum.  (How much lower the cut is taken does not matter: if fewer than K scores certainly reach it, nothing is left out.)
        if (!whole && s_n >= K) cut = (row_ref[r] + surely_above(half_value(s_tau), slack)) * (float)kLn2;
        __syncthreads();
        if (tid == 0) s_n = s_count = 0;
        __syncthreads();
    }
    // The items of the chosen chunks in fp32 with a bound of what that is off: those that can reach `cut` are computed in 64 bits.  If K of them
    // certainly do, the K best are among them.
    int reach = 0;
    if (n > 0) {
        for (int q0 = tid / LPI; q0 < n; q0 += FL * IPP) {
            int32_t i[FL];
            RowPiece<F32, EPL> v[FL];
#pragma unroll
            for (int k = 0; k < FL; ++k) {
                const int e = q0 + k * IPP;
                const int64_t at = e < n ? chunk_item0(s_list[e >> 3]) + (e & 3) + 2 * (e & 4) : sh.items;
                i[k] = at < sh.items ? (int32_t)at : -1;
                v[k] = piece(Q, i[k] < 0 ? 0 : i[k]);
            }
            auto reaches = [&](int k, float z, float err) {
                if (li == LPI - 1 && i[k] >= 0 && z + err >= cut && !masked(i[k])) {
                    const int at = atomicAdd(&s_n, 1);
                    if (at < kMaxChunks) s_item[at] = i[k];
                    if (z - err >= cut) atomicAdd(&s_count, 1);
                }
            };
            auto bound = [&](float size) { return group_sum<LPI>(size) * (sh.scale * (D + 8) * 0x1p-24f) + fabsf(cut) * 0x1p-22f; };
            float size = 0.0f, err = 0.0f;   // sums of |x||y|
            if constexpr (F32 && EPL == 8) { // (one for the FL items, with the largest of their elements in every place)
#pragma unroll
                for (int j = 0; j < EPL; ++j) {
                    float most = fabsf(v[0].at(j));
#pragma unroll
                    for (int k = 1; k < FL; ++k) most = fmaxf(most, fabsf(v[k].at(j)));
                    size = fmaf(fabsf(pf[j]), fminf(most, 3.0e38f), size);      // (an infinity of a masked item is not to make its neighbours' bound a NaN)
                }
                err = bound(size);
            }
#pragma unroll
            for (int k = 0; k < FL; ++k) {
                float z = 0.0f;
                if constexpr (!(F32 && EPL == 8)) size = 0.0f;
#pragma unroll
                for (int j = 0; j < EPL; ++j) {
                    z = fmaf(pf[j], v[k].at(j), z);
                    if constexpr (!(F32 && EPL == 8)) size = fmaf(fabsf(pf[j]), fabsf(v[k].at(j)), size);
                }
                z = group_sum<LPI>(z) * sh.scale;
                if constexpr (!(F32 && EPL == 8)) err = bound(size);
                reaches(k, z, err);
            }
        }
        __syncthreads();
        reach = s_n;
        if (s_count < K || reach > kMaxChunks) reach = 0;      // no: all of them in 64 bits
    }
    const int all = reach > 0 ? reach : n;
    for (int q0 = tid / LPI; q0 < T + all; q0 += FL * IPP) {
        int32_t i[FL];
        double z[FL];
        bool ok[FL];
#pragma unroll
        for (int k = 0; k < FL; ++k) {
            const int q = q0 + k * IPP, e = q - T;
            const int64_t at = q < T ? given[r * T + q] : e >= all ? -1 : reach > 0 ? s_item[e] : chunk_item0(s_list[e >> 3]) + (e & 3) + 2 * (e & 4);
            ok[k] = at >= 0 && at < sh.items;
            i[k] = ok[k] ? (int32_t)at : 0;
        }
        dots(i, z);
        if (li == 0) {
#pragma unroll
            for (int k = 0; k < FL; ++k) {
                const int q = q0 + k * IPP;
                if (q >= T + all) continue;
                const bool out = ok[k] && masked(i[k]);
                if (q < T) logp[r * T + q] = !ok[k] ? 0.0f : out ? -INFINITY : (float)(z[k] - lse);
                else { c_s[q - T] = ok[k] && !out && z[k] == z[k] ? z[k] : -INFINITY; c_id[q - T] = i[k]; }
            }
        }
    }
    if (K == 0) return;
    __syncthreads();
    if (reach > 0) {
        for (int q = tid; q < reach; q += NT) {      // each one's place is the number of those before it
            const double z = c_s[q];
            const int32_t id = c_id[q];
            int place = 0;
            for (int t = 0; t < reach; ++t) place += before(c_s[t], c_id[t], z, id);
            if (place < K) { top_idx[r * K + place] = id; top_logp[r * K + place] = (float)(z - lse); }
        }
        return;
    }
    if (!whole) {
        sort_candidates<NT>(c_s, c_id, n);
    } else {
        // the row in blocks of half the list: what exceeds the K-th best so far is added, and the list cut to K when it is half full
        double least = -INFINITY;
        for (int64_t base = 0; base < sh.items; base += kCand / 2) {
            const int64_t end = base + kCand / 2 < sh.items ? base + kCand / 2 : sh.items;
            for (int64_t q0 = base + tid / LPI; q0 < base + kCand / 2; q0 += FL * IPP) {      // (whole groups of lanes stay together)
                int32_t i[FL];
                double z[FL];
#pragma unroll
                for (int k = 0; k < FL; ++k) i[k] = q0 + k * IPP < end ? (int32_t)(q0 + k * IPP) : 0;
                dots(i, z);
#pragma unroll
                for (int k = 0; k < FL; ++k) {
                    if (li == 0 && q0 + k * IPP < end && z[k] > least && !masked(i[k])) {
                        const int at = atomicAdd(&s_n, 1);
                        c_s[at] = z[k];
                        c_id[at] = i[k];
                    }
                }
            }
            __syncthreads();
            const int have = s_n;
            __syncthreads();
            if (have > kCand / 2 || end == sh.items) {
                sort_candidates<NT>(c_s, c_id, have);
                if (have >= K) least = c_s[K - 1];
                if (tid == 0) s_n = have < K ? have : K;
                __syncthreads();
            }
        }
        n = s_n;
    }
    for (int t = tid; t < K; t += NT) {
        const bool in = t < n && c_s[t] > -INFINITY;
        top_idx[r * K + t] = in ? c_id[t] : -1;
        top_logp[r * K + t] = in ? (float)(c_s[t] - lse) : -INFINITY;
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------------
int thin_rows(int d, int dtype)                // rows the thin form takes: operands of 16 rows cost d / 4 (fp32) or d / 8 registers
{
    const int ub = dtype == RSX_F32 ? 256 / d : 512 / d;
    return 16 * (ub > 4 ? 4 : ub);
}

int thin_groups(int64_t items)
{
    const int64_t tiles = (items + kTile - 1) / kTile, want = (tiles + 3) / 4, most = (int64_t)rsx_num_cus() * 4;
    return (int)(want < most ? want : most);
}

struct Ws {
    char *planes;
    float *factor, *row_factor;
    uint32_t *bits;
    float *ref, *slack;
    float4 *part;
    uint16_t *keys;
    int64_t pass, bytes;      // rows of one pass over the catalog
};

int wide_users(int dtype) { return 128 * users_block(dtype == RSX_F32); }

int64_t wide_splits(int64_t rows, int64_t items, int dtype)
{
    const int64_t slots = kWaves * (int64_t)rsx_num_cus(), ut = (rows + wide_users(dtype) - 1) / wide_users(dtype), groups = (items + 127) / 128;
    const int64_t s = slots / ut;
    return s < 1 ? 1 : s > groups ? groups : s;
}

// a pass' bits and chunk maxima are held to 768 MB, its blocks of rows to what a grid's second dimension takes
int64_t pass_rows(int64_t rows, int64_t items)
{
    const int64_t per = mask_words(items) * 4 + (items + 127) / 128 * 32;
    int64_t most = (768ll << 20) / per / 256 * 256;
    most = most < 256 ? 256 : most > (1ll << 22) ? 1ll << 22 : most;
    return rows < most ? rows : most;
}

Ws carve(void *ws, int64_t rows, int64_t items, int d, int dtype, bool mask, int K)
{
    Ws w;
    char *base = (char *)ws;
    int64_t off = 0;
    auto take = [&](int64_t n) { char *q = base + off; off += a256(n); return q; };
    const int64_t tiles4 = (items + 127) / 128 * 4;
    const bool thin = rows <= thin_rows(d, dtype);
    w.pass = pass_rows(rows, items);
    const int64_t parts = thin ? thin_groups(items) : wide_splits(w.pass, items, dtype);
    // (the last, shorter pass takes more splits over fewer rows: rows x splits never exceeds this)
    const int64_t cells = thin ? rows * parts : w.pass * parts + kWaves * (int64_t)rsx_num_cus() * wide_users(dtype);
    w.planes = take(!thin && dtype == RSX_F32 ? tiles4 * kTile * (int64_t)d * 4 : 0);
    w.factor = (float *)take(!thin && dtype == RSX_F32 ? tiles4 * 4 : 0);
    w.row_factor = (float *)take(!thin && dtype == RSX_F32 ? tiles4 * kTile * 4 : 0);
    w.bits = (uint32_t *)take(mask ? w.pass * mask_words(items) * 4 : 0);
    w.ref = (float *)take(w.pass * 4);
    w.slack = (float *)take(w.pass * 4);
    w.part = (float4 *)take(cells * 16);
    w.keys = (uint16_t *)take(K > 0 ? w.pass * ((items + 127) / 128) * 32 : 0);
    w.bytes = off;
    return w;
}

struct Call {
    const void *P, *Q;
    Shape sh;
    const int64_t *indptr;
    const int32_t *indices;
    const int32_t *given;
    int T, K;
    float *logp, *lse, *ent;
    int32_t *top_idx;
    float *top_logp;
};

template <int D, bool F32, int UB>
void launch_thin(const Call &c, const Shape &sh, const Ws &w, int groups, hipStream_t st)
{
#define RSX_LP_THIN(M_, T_) hipLaunchKernelGGL((thin_kernel<D, F32, UB, M_, T_>), dim3(groups), dim3(256), 0, st, c.P, c.Q, sh, w.bits, w.ref, w.part, w.keys)
    if (c.indptr) { if (c.K) RSX_LP_THIN(true, true); else RSX_LP_THIN(true, false); }
    else { if (c.K) RSX_LP_THIN(false, true); else RSX_LP_THIN(false, false); }
#undef RSX_LP_THIN
}

template <int D, bool F32>
void run(const Call &c, const Ws &w, hipStream_t st)
{
    const bool thin = c.sh.rows <= thin_rows(D, F32 ? RSX_F32 : RSX_BF16);
    const int64_t items = c.sh.items;
    const double off_by = (double)(c.sh.scale * kLog2e) / (c.sh.scale * 1.4426950408889634074) - 1.0;      // of the fp32 factor scale log2 e
    for (int64_t r0 = 0; r0 < c.sh.rows; r0 += w.pass) {
        Shape sh = c.sh;
        sh.user_ids += r0;
        sh.rows = c.sh.rows - r0 < w.pass ? c.sh.rows - r0 : w.pass;
        const int64_t tiles = F32 && !thin && r0 == 0 ? (items + 127) / 128 * 4 : 0, bit_rows = c.indptr ? sh.rows : 0, refs = c.K ? (sh.rows + 3) / 4 : 0;
        if (tiles + bit_rows + refs > 0)
            hipLaunchKernelGGL((prepare_kernel<D, F32>), dim3((unsigned)(tiles + bit_rows + refs)), dim3(256), 0, st, c.P, c.Q, sh, c.indptr, c.indices, tiles, bit_rows,
                               (uint4 *)w.planes, w.factor, w.row_factor, w.bits, w.ref, w.slack);
        int parts;
        double skew;
        if (thin) {
            parts = thin_groups(items);
            constexpr int MOST = F32 ? 256 / D : 512 / D;
            if (sh.rows <= 16) launch_thin<D, F32, 1>(c, sh, w, parts, st);
            else if constexpr (MOST >= 2) {
                if (sh.rows <= 32) launch_thin<D, F32, 2>(c, sh, w, parts, st);
                else if constexpr (MOST >= 4) launch_thin<D, F32, 4>(c, sh, w, parts, st);
            }
            skew = off_by;
        } else {
            skew = F32 ? 0.0 : off_by;          // (fp32: scale log2 e is in the operands)
            parts = (int)wide_splits(sh.rows, items, F32 ? RSX_F32 : RSX_BF16);
            const dim3 grid((unsigned)parts, (unsigned)((sh.rows + WideGeo<D, F32>::WGU - 1) / WideGeo<D, F32>::WGU));
#define RSX_LP_WIDE(M_, T_) hipLaunchKernelGGL((wide_kernel<D, F32, M_, T_>), grid, dim3(256), 0, st, c.P, F32 ? w.planes : (const char *)c.Q, w.factor, w.row_factor, sh, w.bits, w.ref, parts, w.part, (uint4 *)w.keys)
            if (c.indptr) { if (c.K) RSX_LP_WIDE(true, true); else RSX_LP_WIDE(true, false); }
            else { if (c.K) RSX_LP_WIDE(false, true); else RSX_LP_WIDE(false, false); }
#undef RSX_LP_WIDE
        }
#define RSX_LP_FINISH(NT_) hipLaunchKernelGGL((finish_kernel<D, F32, NT_>), dim3((unsigned)sh.rows), dim3(NT_), 0, st, c.P, c.Q, sh, c.indptr ? w.bits : (const uint32_t *)nullptr, \
                                              w.part, parts, skew, w.keys, w.ref, w.slack, c.given + (c.T ? r0 * c.T : 0), c.T, c.K, c.logp + (c.T ? r0 * c.T : 0), \
                                              c.lse ? c.lse + r0 : nullptr, c.ent ? c.ent + r0 : nullptr, c.top_idx + (c.K ? r0 * c.K : 0), c.top_logp + (c.K ? r0 * c.K : 0))
        if (sh.rows <= rsx_num_cus()) RSX_LP_FINISH(1024); else if (sh.rows <= 2 * rsx_num_cus()) RSX_LP_FINISH(512); else RSX_LP_FINISH(256);
#undef RSX_LP_FINISH
    }
}

}  // namespace

RSX_API int64_t rsx_score_logprobs_workspace(int64_t num_rows, int64_t num_items, int d, int dtype, int masked, int K)
{
    if (num_rows < 0 || num_items <= 0 || num_items >= (1ll << 31) - 128 || !rsx_dim_ok(d) || (dtype != RSX_F32 && dtype != RSX_BF16) || K < 0 || K > kMaxK)
        return RSX_E_INVALID;
    return carve(nullptr, num_rows < 1 ? 1 : num_rows, num_items, d, dtype, masked != 0, K).bytes;
}

RSX_API int rsx_score_logprobs(const void *P, int64_t num_users, const int32_t *user_ids_dev, int64_t num_rows, const void *Q, int64_t num_items, int d,
                               int dtype, const int64_t *mask_indptr_dev, const int32_t *mask_indices_dev, float scale, const int32_t *items_dev, int T, int K,
                               float *logp_out, float *lse_out, float *entropy_out, int32_t *topk_idx_out, float *topk_logp_out, void *ws, int64_t ws_bytes,
                               rsx_stream_t stream)
{
    RSX_CHECK_ARG(P && Q && user_ids_dev, "null pointer");
    RSX_CHECK_ARG(rsx_dim_ok(d), "d must be 32, 64, 128 or 256");
    RSX_CHECK_ARG(dtype == RSX_F32 || dtype == RSX_BF16, "dtype must be RSX_F32 or RSX_BF16");
    RSX_CHECK_ARG(num_rows >= 0 && num_users > 0 && num_items > 0 && num_items < (1ll << 31) - 128, "bad shape");
    RSX_CHECK_ARG((mask_indptr_dev == nullptr) == (mask_indices_dev == nullptr), "mask needs both CSR arrays");
    RSX_CHECK_ARG(scale > 0.0f && scale < INFINITY, "scale must be positive and finite");
    RSX_CHECK_ARG(T >= 0 && (T == 0 || (items_dev && logp_out)), "T items per row need their ids and an output");
    RSX_CHECK_ARG(K >= 0 && K <= kMaxK && K <= num_items && (K == 0 || (topk_idx_out && topk_logp_out)), "K must be in [0, min(128, num_items)], with both outputs");
    RSX_CHECK_ARG(aligned16(P) && aligned16(Q), "table rows must be 16-byte aligned");
    if (num_rows == 0) return RSX_OK;
    const Ws w = carve(ws, num_rows, num_items, d, dtype, mask_indptr_dev != nullptr, K);
    if (ws == nullptr || ws_bytes < w.bytes || !aligned16(ws)) {
        rsx_set_error("rsx_score_logprobs: workspace of %lld bytes (16-byte aligned) required, got %lld", (long long)w.bytes, (long long)ws_bytes);
        return RSX_E_WORKSPACE;
    }
    const Call c{P, Q, {user_ids_dev, num_rows, num_users, num_items, scale}, mask_indptr_dev, mask_indices_dev, items_dev, T, K,
                 logp_out, lse_out, entropy_out, topk_idx_out, topk_logp_out};
    hipStream_t st = (hipStream_t)stream;
#define RSX_LP_RUN(D_) do { if (dtype == RSX_F32) run<D_, true>(c, w, st); else run<D_, false>(c, w, st); } while (0)
    switch (d) {
    case 32: RSX_LP_RUN(32); break;
    case 64: RSX_LP_RUN(64); break;
    case 128: RSX_LP_RUN(128); break;
    default: RSX_LP_RUN(256); break;
    }
#undef RSX_LP_RUN
    RSX_CHECK_LAUNCH();
    return RSX_OK;
}
