// paged_attention.hip — attention over a paged K/V cache (aq_paged_attention): the choice of kernel, the kernel for few
// rows (single tokens, verify batches, and f32 rows of any number), the plan and the join of split sequences. Many
// 16-bit rows take paged_chunk.hip.
//
// The kernel for few rows. Single tokens are bound by reading the cache: a wave takes 32 positions at a time straight
// from the pages into registers, in the matrix cores' operand layout, with no LDS on the way:
//   S^T = K Q^T  A = K: lane (r = lane & 15, g = lane >> 4) holds position r (+ 16 t), 16 bytes of its row at dimension
//                32 s + 8 g; B = Q^T from the LDS, where the work-group's rows lie in the same order. Lane (n, g) then has
//                row n's scores of positions 16 t + 4 g + i.
//   O^T = V^T P^T  those scores' exponentials are already B's layout if k-slot (g, e) stands for position 16 (e / 4) + 4 g
//                + e % 4, so A = V^T takes the V rows in that order: each lane loads 16 bytes (8 dimensions) of its 8
//                positions and turns the 8 x 8 block in registers (one v_perm per dword).
// One running maximum and sum per row; a wave's four lane groups share the maximum, the sum is joined at the end.
//
// f32 rows over a 16-bit cache keep 32-bit accuracy: q, scaled to its row's exponent, and the probabilities go in as two
// f16 or three bf16 pieces whose sum has 22 or 24 bits. f32 over f32 takes the f32 matrix cores (16x16x4).
#include <algorithm>
#include <atomic>
#include <cmath>
#include <mutex>

#include "paged_attn.h"

namespace aq {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));

template <int CT>
__device__ __forceinline__ f4 mfma16(u4 a, u4 b, f4 c) {
    if constexpr (CT == AQ_TYPE_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

// The sum of v over pieces: v as NP values of the type, each the rounding of what the ones before left.
template <int CT, int NP>
__device__ __forceinline__ void pieces(const float *v, u4 *out) { // 8 values -> NP operands
    using E = typename RowType<CT>::type;
    typedef E vec __attribute__((ext_vector_type(8)));
    float rest[8];
#pragma unroll
    for (int i = 0; i < 8; i++) rest[i] = v[i];
#pragma unroll
    for (int p = 0; p < NP; p++) {
        vec x;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            x[i] = (E)rest[i];
            if (p + 1 < NP) rest[i] -= (float)x[i];
        }
        out[p] = __builtin_bit_cast(u4, x);
    }
}

// An infinity or a NaN.
__device__ __forceinline__ bool odd_f32(unsigned w) { return (w & 0x7F800000u) == 0x7F800000u; }

constexpr int WAVES = 4, TILE = 32, UNIT = WAVES * TILE; // positions of a wave's tile and of a work-group's step

// What the few-row kernel keeps where, for one cache type, row type and padded head size.
template <int CT, bool FQ, int D, int NR>
struct FewShape {
    static constexpr bool F = CT == AQ_TYPE_F32;
    static constexpr int NP = !FQ || F ? 1 : (CT == AQ_TYPE_F16 ? 2 : 3); // pieces of q and of the probabilities
    static constexpr int STEPS = F ? D / 16 : D / 32;                     // 16-byte K operands of a row per lane
    static constexpr int VB = F || D == 64 ? 4 : 8;                       // dimensions of a V row per lane and chunk
    static constexpr int CHUNKS = D / (16 * VB);
    static constexpr int ACC = CHUNKS * VB; // accumulators (4 values each) per row tile
    static constexpr int R = 16 * NR;
    static constexpr int PASSES = D / 64, CROW = 68; // the waves' outputs meet 64 dimensions at a time
    static constexpr int QF = NR * STEPS * NP * 64;  // 16-byte operands of q
    static constexpr int LDS = QF * 16 + WAVES * R * CROW * 4 + WAVES * R * 8;
    static constexpr bool AHEAD = D <= 128 || NR == 1; // the next tile's K rows loaded while this one is summed
};

template <int CT, bool FQ, int D, int NR>
__global__ void __launch_bounds__(256, 2) few_rows_kernel(AttnPagedArgs a) {
    using S = FewShape<CT, FQ, D, NR>;
    constexpr bool F = S::F;
    constexpr int QT = FQ ? AQ_TYPE_F32 : CT, NP = S::NP, STEPS = S::STEPS, CHUNKS = S::CHUNKS, VB = S::VB, R = S::R;
    constexpr int ES = F ? 4 : 2;
    // f16 probabilities are kept at 2^14 times their size (and so are the sums): their small ones stay normal numbers
    constexpr float P_SHIFT = CT == AQ_TYPE_F16 ? 14.0f : 0.0f;
    extern __shared__ __align__(16) char smem[];
    u4 *qf = reinterpret_cast<u4 *>(smem);
    float *comb = reinterpret_cast<float *>(smem + S::QF * 16);        // [WAVES][R][CROW]
    float *ml = reinterpret_cast<float *>(smem + S::QF * 16 + WAVES * R * S::CROW * 4); // [WAVES][R][2]
    __shared__ uint32_t pre[INLINE_SEQS + 1], wsum[WAVES], qmax[R], found;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int hd = a.kv.hd, G = a.G;

    const Share sh = take_share(a, R, UNIT, pre, wsum, &found);
    uint32_t u = sh.begin, j = sh.j;
    while (u < sh.end) { // uniform
        const Segment sg = next_segment(a, R, pre, sh, u, j);
        const uint32_t kvh = sg.kvh, seq = sg.seq, t0 = sg.t0, t1 = sg.t1;
        const int32_t r0 = sg.r0;
        const SeqRows sr = paged_seq(a.b, seq);
        const int32_t n_rows = sr.n * G, base = sr.len - sr.n;
        const UnitRange range = tile_units(sr, G, a.window, a.cap, r0, R, UNIT);
        const int32_t tok0 = r0 / G, tok1 = (min(r0 + R, n_rows) - 1) / G;
        const int32_t kend = min(max(base + tok1 + 1, 0), (int32_t)a.cap);
        const int32_t min_hi = base + tok0 + 1;
        const int64_t max_lo = a.window ? (int64_t)base + tok1 + 1 - (int64_t)a.window : INT64_MIN;
        const int32_t *table = a.b.pages + (size_t)seq * a.b.max_pages;
        const uint64_t head_off = (uint64_t)kvh * a.kv.head_bytes;

        // this lane's rows: the positions they see are lo .. hi - 1
        int32_t hi[NR], lo[NR];
#pragma unroll
        for (int nr = 0; nr < NR; nr++) {
            const int32_t rr = r0 + 16 * nr + r, tok = rr / G;
            hi[nr] = rr < n_rows ? base + tok + 1 : 0;
            const int64_t l = a.window ? (int64_t)base + tok + 1 - (int64_t)a.window : 0;
            lo[nr] = l > 0 ? (int32_t)l : 0;
        }

        __syncthreads(); // the LDS of the segment before is read
        // ---- queries into the LDS, operand order; 16 rows x 16 units of 8 (4) dimensions at a time
        float rscale[NR]; // what this lane's rows' scores are multiplied by
        {
            constexpr int QV = F ? 4 : 8, ALL = NR * (D / QV), UNITS = (ALL + 15) / 16; // 16 at a time
            float v[UNITS][QV];
            if (tid < R) qmax[tid] = 0;
            if constexpr (NP == 2) __syncthreads();
#pragma unroll
            for (int i = 0; i < UNITS; i++) {
                const int unit = i * 16 + (tid >> 4), nr = unit / (D / QV), at = unit % (D / QV) * QV, n = tid & 15;
                if (ALL % 16 && unit >= ALL) continue;
                const int32_t rr = r0 + 16 * nr + n, tok = rr / G;
                const int head = (int)kvh * G + (rr - tok * G);
                const char *row = a.q.p + ((int64_t)(sr.first + tok) * a.q.row + (int64_t)head * a.q.head) *
                                              (int64_t)sizeof(typename RowType<QT>::type);
                load_row<QT, QV>(row, at, rr < n_rows ? hd : 0, a.q_wide, v[i]);
                if constexpr (NP == 2) {
                    float m = 0.0f;
#pragma unroll
                    for (int e = 0; e < QV; e++) m = fmaxf(m, fabsf(v[i][e]));
                    atomicMax(&qmax[16 * nr + n], __float_as_uint(m));
                }
            }
            if constexpr (NP == 2) __syncthreads();
            // two f16 pieces: the row is scaled so that its largest value lies in [1, 2)
            auto exponent = [&](int row) { return min(max(qmax[row] >> 23, 1u), 253u); };
#pragma unroll
            for (int i = 0; i < UNITS; i++) {
                const int unit = i * 16 + (tid >> 4), nr = unit / (D / QV), at = unit % (D / QV), n = tid & 15;
                if (ALL % 16 && unit >= ALL) continue;
                if constexpr (F) { // operand s = at / 4, lane (n, g = at % 4)
                    qf[(nr * STEPS + at / 4) * 64 + (at % 4) * 16 + n] =
                        u4{__float_as_uint(v[i][0]), __float_as_uint(v[i][1]), __float_as_uint(v[i][2]),
                           __float_as_uint(v[i][3])};
                } else {
                    if constexpr (NP == 2) {
                        const float up = __uint_as_float((254u - exponent(16 * nr + n)) << 23);
#pragma unroll
                        for (int e = 0; e < QV; e++) v[i][e] *= up;
                    }
                    u4 piece[NP];
                    pieces<CT, NP>(v[i], piece);
#pragma unroll
                    for (int p = 0; p < NP; p++)
                        qf[((nr * STEPS + at / 4) * NP + p) * 64 + (at % 4) * 16 + n] = piece[p];
                }
            }
#pragma unroll
            for (int nr = 0; nr < NR; nr++)
                rscale[nr] = NP == 2 ? a.scale_log2 * __uint_as_float(exponent(16 * nr + r) << 23) : a.scale_log2;
        }
        __syncthreads();

        // ---- the wave's tiles of 32 positions
        f4 o[NR][S::ACC];
        float m[NR], l[NR];
#pragma unroll
        for (int nr = 0; nr < NR; nr++) {
            m[nr] = -INFINITY;
            l[nr] = 0.0f;
#pragma unroll
            for (int i = 0; i < S::ACC; i++) o[nr][i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        const int32_t last_tile = min((int32_t)((range.lo + t1) * WAVES), (kend + TILE - 1) / TILE);
        int32_t tile = (int32_t)(range.lo + t0) * WAVES + wave;

        // where the tile's rows are: lane (and lane + 32) holds position `lane & 31`'s
        auto locate = [&](int32_t t, uint32_t *units) {
            const int32_t p = t * TILE + (lane & 31);
            const bool ok = p < kend && paged_slot(a.kv, table, a.b.max_pages, (uint32_t)p, units);
            if (!ok) *units = 0;
            return (uint32_t)__ballot(ok);
        };
        auto row_ptr = [&](const char *pool, uint32_t units, int pos) {
            return pool + (((uint64_t)(uint32_t)__shfl((int)units, pos) << a.kv.unit_shift) + head_off);
        };
        auto load_k = [&](uint32_t units, int t, u4 *k) { // one 16-position half
            const char *p = row_ptr(a.kv.k, units, 16 * t + r);
#pragma unroll
            for (int s = 0; s < STEPS; s++) {
                // dimensions past the head repeat its last ones: q is 0 there
                const int at = min((F ? 16 : 32) * s + (F ? 4 : 8) * g, hd - (F ? 4 : 8));
                k[s] = *reinterpret_cast<const u4 *>(p + at * ES);
            }
        };

        constexpr int KH = F ? 1 : 2; // 16-position halves of K in registers at once
        u4 k[KH][STEPS];
        uint32_t units = 0, okm = 0;
        if (tile < last_tile) {
            okm = locate(tile, &units);
            if constexpr (S::AHEAD && !F) {
#pragma unroll
                for (int t = 0; t < 2; t++) load_k(units, t, k[t]);
            }
        }
        for (; tile < last_tile; tile += WAVES) {
            asm volatile("" ::: "memory"); // q's operands are read from the LDS each time, not kept in registers
            const int32_t kb = tile * TILE;
            const uint32_t here = units, ok = okm;
            // the next tile's page entries, ahead of its rows
            if (tile + WAVES < last_tile) okm = locate(tile + WAVES, &units);
            f4 s[NR][2];
#pragma unroll
            for (int nr = 0; nr < NR; nr++)
#pragma unroll
                for (int t = 0; t < 2; t++) s[nr][t] = f4{0.0f, 0.0f, 0.0f, 0.0f};

            // ---- V rows of 8 (f32: 4 per half) positions: lane (r, g) has dimensions VB r .. of chunk c
            auto load_v = [&](int e, int c, auto *dst) {
                const int pos = 16 * (e / 4) + 4 * g + e % 4;
                const char *p = row_ptr(a.kv.v, here, pos);
                const int at = min(c * 16 * VB + VB * r, hd - VB); // past the head: outputs that are not stored
                if constexpr (VB * ES == 8) *dst = *reinterpret_cast<const u2 *>(p + at * ES);
                else *dst = *reinterpret_cast<const u4 *>(p + at * ES);
            };

            if constexpr (!F) {
                using VV = typename std::conditional<VB * ES == 8, u2, u4>::type;
                constexpr int VW = VB * ES / 4; // dwords
                if constexpr (!S::AHEAD) {
#pragma unroll
                    for (int t = 0; t < 2; t++) load_k(here, t, k[t]);
                }
                VV v[CHUNKS][8];
#pragma unroll
                for (int c = 0; c < (S::AHEAD ? CHUNKS : 1); c++)
#pragma unroll
                    for (int e = 0; e < 8; e++) load_v(e, c, &v[c][e]);
#pragma unroll
                for (int st = 0; st < STEPS; st++)
#pragma unroll
                    for (int nr = 0; nr < NR; nr++)
#pragma unroll
                        for (int p = 0; p < NP; p++) {
                            const u4 q = qf[((nr * STEPS + st) * NP + p) * 64 + lane];
#pragma unroll
                            for (int t = 0; t < 2; t++) s[nr][t] = mfma16<CT>(k[t][st], q, s[nr][t]);
                        }
                if constexpr (NP > 1) { // an infinite key times the pieces of one number is a NaN: by the first piece alone
                    bool nan = false;
#pragma unroll
                    for (int nr = 0; nr < NR; nr++)
#pragma unroll
                        for (int e = 0; e < 8; e++) nan |= s[nr][e / 4][e % 4] != s[nr][e / 4][e % 4];
                    if (__any(nan)) {
#pragma unroll
                        for (int nr = 0; nr < NR; nr++)
#pragma unroll
                            for (int t = 0; t < 2; t++) {
                                f4 one = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                                for (int st = 0; st < STEPS; st++)
                                    one = mfma16<CT>(k[t][st], qf[(nr * STEPS + st) * NP * 64 + lane], one);
#pragma unroll
                                for (int i = 0; i < 4; i++) s[nr][t][i] = s[nr][t][i] == s[nr][t][i] ? s[nr][t][i] : one[i];
                            }
                    }
                }
                if constexpr (S::AHEAD) {
                    if (tile + WAVES < last_tile) {
#pragma unroll
                        for (int t = 0; t < 2; t++) load_k(units, t, k[t]);
                    }
                } else {
#pragma unroll
                    for (int c = 1; c < CHUNKS; c++)
#pragma unroll
                        for (int e = 0; e < 8; e++) load_v(e, c, &v[c][e]);
                }
                const bool edge = kb + TILE > min_hi || (int64_t)kb < max_lo || ok != 0xFFFFFFFFu; // uniform
                u4 pf[NR][NP];
#pragma unroll
                for (int nr = 0; nr < NR; nr++) {
                    float x[8], mt = -INFINITY;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const int pos = 16 * (e / 4) + 4 * g + e % 4;
                        x[e] = s[nr][e / 4][e % 4] * rscale[nr];
                        if (edge && !(kb + pos < hi[nr] && kb + pos >= lo[nr] && ((ok >> pos) & 1))) x[e] = -INFINITY;
                        mt = fmaxf(mt, x[e]);
                    }
                    mt = fmaxf(mt, __shfl_xor(mt, 16));
                    mt = fmaxf(mt, __shfl_xor(mt, 32));
                    const float mn = fmaxf(m[nr], mt), mu = mn == -INFINITY ? 0.0f : mn;
                    if (__any(mn > m[nr])) {
                        const float alpha = fast_exp2(m[nr] - mu);
                        l[nr] *= alpha;
#pragma unroll
                        for (int i = 0; i < S::ACC; i++)
#pragma unroll
                            for (int e = 0; e < 4; e++) o[nr][i][e] *= alpha;
                        m[nr] = mn;
                    }
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        x[e] = fast_exp2((x[e] - mu) + P_SHIFT);
                        l[nr] += x[e];
                    }
                    pieces<CT, NP>(x, pf[nr]);
                }
#pragma unroll
                for (int c = 0; c < CHUNKS; c++) {
                    auto product = [&](int jj) { // V^T operand of dimension jj of each lane's VB
                        u4 t;
                        const unsigned sel = jj & 1 ? 0x07060302u : 0x05040100u;
#pragma unroll
                        for (int h = 0; h < 4; h++)
                            t[h] = __builtin_amdgcn_perm(v[c][2 * h + 1][jj / 2], v[c][2 * h][jj / 2], sel);
                        return t;
                    };
                    if (edge) { // rows of positions that no page holds are not numbers that may be multiplied by 0
#pragma unroll
                        for (int e = 0; e < 8; e++)
#pragma unroll
                            for (int x = 0; x < VW; x++)
                                v[c][e][x] = (ok >> (16 * (e / 4) + 4 * g + e % 4)) & 1 ? v[c][e][x] : 0u;
                    }
                    if ((edge && tok0 < tok1) || NP > 1) {
                        // Nor are infinities and NaN of positions that only some of the rows see, and an infinity times
                        // the pieces of one number is a NaN: such values are added position by position, to the rows
                        // that see them, by the probability's first piece, and taken out of the product of the others.
                        unsigned any = 0;
#pragma unroll
                        for (int e = 0; e < 8; e++)
#pragma unroll
                            for (int x = 0; x < VW; x++) any |= odd_bits<CT>(v[c][e][x]);
                        uint32_t odd = 0;
                        if (__any(any & 0x80008000u)) {
#pragma unroll
                            for (int e = 0; e < 8; e++) {
                                unsigned bits = 0;
#pragma unroll
                                for (int x = 0; x < VW; x++) bits |= odd_bits<CT>(v[c][e][x]);
                                const uint64_t b = __ballot(bits & 0x80008000u);
#pragma unroll
                                for (int gg = 0; gg < 4; gg++)
                                    if ((b >> (16 * gg)) & 0xFFFFu) odd |= 1u << (16 * (e / 4) + 4 * gg + e % 4);
                            }
                        }
                        if (odd) {
#pragma unroll 1
                            for (uint32_t rest = odd; rest; rest &= rest - 1) {
                                const int pos = __ffs(rest) - 1, e = 4 * (pos / 16) + pos % 4; // its k-slot
                                u4 only = u4{0u, 0u, 0u, 0u};
                                if (pos % 16 / 4 == g) only[e / 2] = e & 1 ? 0xFFFF0000u : 0x0000FFFFu;
#pragma unroll
                                for (int nr = 0; nr < NR; nr++) {
                                    const bool sees = kb + pos < hi[nr] && kb + pos >= lo[nr];
#pragma unroll
                                    for (int jj = 0; jj < VB; jj++) {
                                        u4 vt = product(jj) & only;
#pragma unroll
                                        for (int x = 0; x < 4; x++) vt[x] &= odd_mask<CT>(vt[x]);
                                        const f4 t = mfma16<CT>(vt, pf[nr][0], o[nr][c * VB + jj]);
#pragma unroll
                                        for (int x = 0; x < 4; x++)
                                            o[nr][c * VB + jj][x] = sees ? t[x] : o[nr][c * VB + jj][x];
                                    }
                                }
                            }
#pragma unroll
                            for (int e = 0; e < 8; e++)
#pragma unroll
                                for (int x = 0; x < VW; x++) v[c][e][x] &= ~odd_mask<CT>(v[c][e][x]);
                        }
                    }
#pragma unroll
                    for (int jj = 0; jj < VB; jj++) {
                        const u4 vt = product(jj);
#pragma unroll
                        for (int nr = 0; nr < NR; nr++)
#pragma unroll
                            for (int p = 0; p < NP; p++)
                                o[nr][c * VB + jj] = mfma16<CT>(vt, pf[nr][p], o[nr][c * VB + jj]);
                    }
                }
            } else {
                // ---- f32 cache: 16 positions at a time, k-slot g of step i stands for position 16 t + 4 g + i
                auto mul = [](unsigned x, unsigned y, f4 c) {
                    return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(x), __uint_as_float(y), c, 0, 0, 0);
                };
                u4 v[4][CHUNKS];
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    load_k(here, t, k[0]);
                    if (t == 0) {
#pragma unroll
                        for (int i = 0; i < 4; i++)
#pragma unroll
                            for (int c = 0; c < CHUNKS; c++) load_v(i, c, &v[i][c]);
                    }
#pragma unroll
                    for (int st = 0; st < STEPS; st++)
#pragma unroll
                        for (int nr = 0; nr < NR; nr++) {
                            const u4 q = qf[(nr * STEPS + st) * 64 + lane];
#pragma unroll
                            for (int i = 0; i < 4; i++) s[nr][t] = mul(k[0][st][i], q[i], s[nr][t]);
                        }
                }
                const bool edge = kb + TILE > min_hi || (int64_t)kb < max_lo || ok != 0xFFFFFFFFu; // uniform
                float x[NR][8];
#pragma unroll
                for (int nr = 0; nr < NR; nr++) {
                    float mt = -INFINITY;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const int pos = 16 * (e / 4) + 4 * g + e % 4;
                        x[nr][e] = s[nr][e / 4][e % 4] * rscale[nr];
                        if (edge && !(kb + pos < hi[nr] && kb + pos >= lo[nr] && ((ok >> pos) & 1))) x[nr][e] = -INFINITY;
                        mt = fmaxf(mt, x[nr][e]);
                    }
                    mt = fmaxf(mt, __shfl_xor(mt, 16));
                    mt = fmaxf(mt, __shfl_xor(mt, 32));
                    const float mn = fmaxf(m[nr], mt), mu = mn == -INFINITY ? 0.0f : mn;
                    if (__any(mn > m[nr])) {
                        const float alpha = fast_exp2(m[nr] - mu);
                        l[nr] *= alpha;
#pragma unroll
                        for (int i = 0; i < S::ACC; i++)
#pragma unroll
                            for (int e = 0; e < 4; e++) o[nr][i][e] *= alpha;
                        m[nr] = mn;
                    }
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        x[nr][e] = fast_exp2(x[nr][e] - mu);
                        l[nr] += x[nr][e];
                    }
                }
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    if (t == 1) {
#pragma unroll
                        for (int i = 0; i < 4; i++)
#pragma unroll
                            for (int c = 0; c < CHUNKS; c++) load_v(4 + i, c, &v[i][c]);
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int pos0 = 16 * t + i; // + 4 g
                        if (edge) {
                            const bool keep = (ok >> (pos0 + 4 * g)) & 1;
                            bool is_odd = false;
#pragma unroll
                            for (int c = 0; c < CHUNKS; c++)
#pragma unroll
                                for (int y = 0; y < 4; y++) {
                                    v[i][c][y] = keep ? v[i][c][y] : 0u;
                                    is_odd |= odd_f32(v[i][c][y]);
                                }
                            const uint64_t b = __ballot(is_odd);
                            if (b && tok0 < tok1) {
#pragma unroll 1
                                for (int gg = 0; gg < 4; gg++) {
                                    if (!((b >> (16 * gg)) & 0xFFFFu)) continue; // uniform
                                    const int pos = kb + pos0 + 4 * gg;
#pragma unroll
                                    for (int nr = 0; nr < NR; nr++) {
                                        const bool sees = pos < hi[nr] && pos >= lo[nr];
#pragma unroll
                                        for (int c = 0; c < CHUNKS; c++)
#pragma unroll
                                            for (int y = 0; y < 4; y++) {
                                                const f4 n = mul(g == gg ? v[i][c][y] : 0u,
                                                                 __float_as_uint(x[nr][4 * t + i]), o[nr][c * 4 + y]);
#pragma unroll
                                                for (int z = 0; z < 4; z++)
                                                    o[nr][c * 4 + y][z] = sees ? n[z] : o[nr][c * 4 + y][z];
                                            }
                                    }
                                }
                                const bool out = (b >> (16 * g)) & 0xFFFFu;
#pragma unroll
                                for (int c = 0; c < CHUNKS; c++)
#pragma unroll
                                    for (int y = 0; y < 4; y++) v[i][c][y] = out ? 0u : v[i][c][y];
                            }
                        }
#pragma unroll
                        for (int nr = 0; nr < NR; nr++)
#pragma unroll
                            for (int c = 0; c < CHUNKS; c++)
#pragma unroll
                                for (int y = 0; y < 4; y++)
                                    o[nr][c * 4 + y] = mul(v[i][c][y], __float_as_uint(x[nr][4 * t + i]), o[nr][c * 4 + y]);
                    }
                }
            }
        }

        // ---- the four waves' rows joined: each scaled to the common maximum, then added, 64 dimensions a pass
#pragma unroll
        for (int nr = 0; nr < NR; nr++) {
            l[nr] += __shfl_xor(l[nr], 16);
            l[nr] += __shfl_xor(l[nr], 32);
            if (g == 0) {
                ml[(wave * R + 16 * nr + r) * 2] = m[nr];
                ml[(wave * R + 16 * nr + r) * 2 + 1] = l[nr];
            }
        }
        __syncthreads();
        float mine[NR];
#pragma unroll
        for (int nr = 0; nr < NR; nr++) {
            float mx = -INFINITY;
#pragma unroll
            for (int x = 0; x < WAVES; x++) mx = fmaxf(mx, ml[(x * R + 16 * nr + r) * 2]);
            mine[nr] = fast_exp2(m[nr] - (mx == -INFINITY ? 0.0f : mx));
        }
        const bool cut = t1 - t0 < sg.cnt;
        const uint32_t slot = 2 * sh.w + (t0 == 0 ? 1 : 0);
#pragma unroll
        for (int pass = 0; pass < S::PASSES; pass++) {
            if (pass) __syncthreads();
#pragma unroll
            for (int nr = 0; nr < NR; nr++) {
                float *c = comb + (size_t)(wave * R + 16 * nr + r) * S::CROW + 16 * g;
                if constexpr (VB == 4) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        f4 t;
#pragma unroll
                        for (int y = 0; y < 4; y++) t[y] = o[nr][pass * 4 + y][i] * mine[nr];
                        *reinterpret_cast<f4 *>(c + 4 * i) = t;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 2; i++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            f4 t;
#pragma unroll
                            for (int y = 0; y < 4; y++)
                                t[y] = o[nr][(pass / 2) * 8 + 4 * h + y][2 * (pass & 1) + i] * mine[nr];
                            *reinterpret_cast<f4 *>(c + 8 * i + 4 * h) = t;
                        }
                }
            }
            __syncthreads();
#pragma unroll
            for (int it = 0; it < NR; it++) {
                const int row = it * 16 + (tid >> 4), v0 = (tid & 15) * 4;
                const int32_t rr = r0 + row;
                const int dim = VB == 4 ? 64 * pass + v0
                                        : 128 * (pass >> 1) + 8 * (4 * (v0 >> 4) + 2 * (pass & 1) + ((v0 >> 3) & 1)) + (v0 & 7);
                if (rr >= n_rows || dim >= hd) continue;
                f4 sum = *reinterpret_cast<const f4 *>(comb + (size_t)row * S::CROW + v0);
                float mx = ml[row * 2];
#pragma unroll
                for (int x = 1; x < WAVES; x++) {
                    const f4 t = *reinterpret_cast<const f4 *>(comb + (size_t)(x * R + row) * S::CROW + v0);
#pragma unroll
                    for (int y = 0; y < 4; y++) sum[y] += t[y];
                    mx = fmaxf(mx, ml[(x * R + row) * 2]);
                }
                float lt = 0.0f;
#pragma unroll
                for (int x = 0; x < WAVES; x++)
                    lt += ml[(x * R + row) * 2 + 1] * fast_exp2(ml[(x * R + row) * 2] - (mx == -INFINITY ? 0.0f : mx));
                if (cut) {
                    *reinterpret_cast<f4 *>(a.part_o + ((size_t)slot * R + row) * D + dim) = sum;
                    if (dim == 0) {
                        a.part_ml[((size_t)slot * R + row) * 2] = mx;
                        a.part_ml[((size_t)slot * R + row) * 2 + 1] = lt;
                    }
                } else {
                    const int32_t tok = rr / G;
                    float out[4];
#pragma unroll
                    for (int y = 0; y < 4; y++) out[y] = lt == 0.0f ? 0.0f : sum[y] / lt;
                    store_out<QT>(a, sr.first + tok, (int)kvh * G + (rr - tok * G), dim, out);
                }
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------------- the join
// One work-group per row of a segment: a group of D / 4 threads takes every so many parts, each part's outputs times
// 2^(its maximum - the running one); the groups meet in the LDS.
template <int QT>
__global__ void __launch_bounds__(256) join_kernel(AttnPagedArgs a, int R, int D) {
    __shared__ f4 os[256];
    __shared__ float ms[256], ls[256];
    const uint32_t nkv = (uint32_t)a.kv.nkv, j = blockIdx.x / nkv, kvh = blockIdx.x % nkv;
    const uint32_t chunk = a.plan[1];
    if (j >= a.plan[2]) return;
    const uint32_t p0 = a.plan[PLAN_HEAD + j], cnt = a.plan[PLAN_HEAD + j + 1] - p0;
    if (cnt == 0) return;
    const uint32_t s0 = p0 * nkv + kvh * cnt, w0 = s0 / chunk, w1 = (s0 + cnt - 1) / chunk;
    if (w0 == w1) return; // one share had it all
    const uint32_t seq = a.planned ? a.seg_seq[j] : j;
    const int32_t r0 = a.planned ? (int32_t)a.seg_rt[j] * R : 0;
    const SeqRows sr = paged_seq(a.b, seq);
    const int row = blockIdx.y;
    const int32_t rr = r0 + row;
    if (rr >= sr.n * a.G) return;
    const int tid = threadIdx.x, quads = D / 4, grp = tid / quads, groups = 256 / quads, dim = tid % quads * 4;
    float m = -INFINITY, l = 0.0f;
    f4 o = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (uint32_t w = w0 + grp; w <= w1; w += groups) {
        const size_t at = (size_t)(2 * w + (w == w0 ? 1 : 0)) * R + row;
        const float pm = a.part_ml[at * 2], pl = a.part_ml[at * 2 + 1];
        const f4 po = dim < a.kv.hd ? *reinterpret_cast<const f4 *>(a.part_o + at * D + dim) : f4{0.0f, 0.0f, 0.0f, 0.0f};
        const float mn = fmaxf(m, pm), mu = mn == -INFINITY ? 0.0f : mn;
        const float x = fast_exp2(m - mu), y = fast_exp2(pm - mu);
        m = mn;
        l = l * x + pl * y;
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = o[i] * x + po[i] * y;
    }
    os[tid] = o;
    ms[tid] = m;
    ls[tid] = l;
    __syncthreads();
    if (grp || dim >= a.kv.hd) return;
    float mx = m;
    for (int x = 1; x < groups; x++) mx = fmaxf(mx, ms[x * quads + tid]);
    const float mu = mx == -INFINITY ? 0.0f : mx;
    const float x0 = fast_exp2(m - mu);
    l *= x0;
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] *= x0;
    for (int x = 1; x < groups; x++) {
        const float y = fast_exp2(ms[x * quads + tid] - mu);
        l += ls[x * quads + tid] * y;
        const f4 t = os[x * quads + tid];
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] += t[i] * y;
    }
    float out[4];
#pragma unroll
    for (int i = 0; i < 4; i++) out[i] = l == 0.0f ? 0.0f : o[i] / l;
    const int32_t tok = rr / a.G;
    store_out<QT>(a, sr.first + tok, (int)kvh * a.G + (rr - tok * a.G), dim, out);
}

// ---------------------------------------------------------------------------------------------------- the plan
// Row tiles of all sequences in order, and the prefix sums of their units; one work-group.
__global__ void __launch_bounds__(1024) plan_kernel(AttnPagedArgs a, int R, uint32_t tk) {
    __shared__ uint32_t wsum[16], carry;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // the inclusive prefix sum of v over the work-group, plus what came before; uniform calls
    auto scan = [&](uint32_t v) {
        uint32_t s = v;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const uint32_t x = __shfl_up(s, d);
            if (lane >= d) s += x;
        }
        if (lane == 63) wsum[wave] = s;
        __syncthreads();
        uint32_t before = carry;
        for (int i = 0; i < wave; i++) before += wsum[i];
        s += before;
        __syncthreads();
        if (tid == 1023) carry = s;
        __syncthreads();
        return s;
    };
    if (tid == 0) carry = 0;
    __syncthreads();
    // row tiles: each sequence writes its own
    for (uint32_t s0 = 0; s0 < a.b.n_seq; s0 += 1024) {
        const uint32_t s = s0 + tid;
        uint32_t n = 0;
        if (s < a.b.n_seq) n = (uint32_t)(((int64_t)paged_seq(a.b, s).n * a.G + R - 1) / R);
        const uint32_t at = scan(n) - n;
        for (uint32_t i = 0; i < n && at + i < a.n_seg; i++) {
            a.seg_seq[at + i] = s;
            a.seg_rt[at + i] = i;
        }
    }
    const uint32_t n_seg = min(carry, a.n_seg);
    __syncthreads();
    if (tid == 0) carry = 0;
    __syncthreads();
    for (uint32_t j0 = 0; j0 < n_seg; j0 += 1024) {
        const uint32_t j = j0 + tid;
        uint32_t n = 0;
        if (j < n_seg) {
            const UnitRange u = tile_units(paged_seq(a.b, a.seg_seq[j]), a.G, a.window, a.cap,
                                           (int32_t)a.seg_rt[j] * R, R, tk);
            n = u.hi - u.lo;
        }
        const uint32_t end = scan(n);
        if (j < n_seg) a.plan[PLAN_HEAD + j + 1] = end;
    }
    if (tid == 0) {
        const uint32_t total = carry * (uint32_t)a.kv.nkv;
        a.plan[0] = total;
        a.plan[1] = share_chunk(total, a.shares, a.min_chunk);
        a.plan[2] = n_seg;
        a.plan[PLAN_HEAD] = 0;
    }
}

// ------------------------------------------------------------------------------------------------- the choice
int compute_units(int device) {
    static std::mutex mu;
    static int cus[64];
    if (device < 0 || device >= 64) return 256;
    std::lock_guard<std::mutex> lock(mu);
    if (!cus[device]) {
        int n = 0;
        if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || n <= 0) n = 256;
        cus[device] = n;
    }
    return cus[device];
}

// Which kernel, its row tile and padded head size, and how its work is split.
struct Choice {
    bool many = false; // paged_chunk.hip
    int R = 16, D = 64;
    uint32_t unit = UNIT, shares = 0, min_chunk = 1, n_seg = 0, cap = 0;
    bool planned = false, join = false;
    PagedSpace space;
};

template <int CT, bool FQ, int D, int NR>
int few_launch(const AttnPagedArgs &a, hipStream_t stream) {
    using S = FewShape<CT, FQ, D, NR>;
    const auto kernel = few_rows_kernel<CT, FQ, D, NR>;
    if constexpr (S::LDS > 56 * 1024) { // with the static arrays past the 64 KiB that need no asking
        static std::atomic<uint64_t> raised{0}; // bit d: done on device d
        int dev = 0;
        AQ_HIP(hipGetDevice(&dev));
        if (!(raised.load() & (1ull << (dev & 63)))) {
            AQ_HIP(hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, S::LDS));
            raised.fetch_or(1ull << (dev & 63));
        }
    }
    kernel<<<a.shares, 256, S::LDS, stream>>>(a);
    AQ_HIP(hipGetLastError());
    return 0;
}
template <int CT, bool FQ>
int few_pick(const AttnPagedArgs &a, int D, int R, hipStream_t stream) {
    if (R == 16) {
        if (D == 64) return few_launch<CT, FQ, 64, 1>(a, stream);
        if (D == 128) return few_launch<CT, FQ, 128, 1>(a, stream);
        return few_launch<CT, FQ, 256, 1>(a, stream);
    }
    if (D == 64) return few_launch<CT, FQ, 64, 2>(a, stream);
    if (D == 128) return few_launch<CT, FQ, 128, 2>(a, stream);
    return few_launch<CT, FQ, 256, 2>(a, stream);
}

int choose(const char *call, const aq_paged_kv *kv, const aq_paged_batch *b, uint32_t n_head, bool f32_rows, int device,
           Choice *c) {
    const uint32_t G = n_head / kv->n_head_kv;
    const uint64_t rows = (uint64_t)b->max_rows * G;
    c->D = kv->head_dim <= 64 ? 64 : kv->head_dim <= 128 ? 128 : 256;
    c->cap = (uint32_t)std::min<uint64_t>((uint64_t)b->max_pages * kv->page_size, b->max_len);
    // 16-bit rows past what one pass of the few-row kernel holds
    c->many = !f32_rows && rows > 32;
    c->R = c->many ? CHUNK_ROWS : rows <= 16 ? 16 : 32;
    c->unit = c->many ? chunk_keys(c->D) : UNIT;
    c->min_chunk = c->many ? 256 / c->unit : 1;
    c->planned = rows > (uint64_t)c->R || b->n_seq > INLINE_SEQS;
    // row tiles: a whole one per R rows of all sequences together, and one begun per sequence
    const uint64_t n_seg = c->planned ? ((uint64_t)b->n_rows * G) / c->R + b->n_seq : b->n_seq;
    const int cu = compute_units(device);
    c->shares = (uint32_t)cu * 2;
    const uint64_t per = (c->cap + c->unit - 1) / c->unit + 1;
    if ((double)n_seg * (double)per * kv->n_head_kv >= 2147483648.0 || n_seg * kv->n_head_kv >= (1u << 31))
        return fail(AQ_EUNSUP, std::string(call) + ": batch of more than 2^31 units of work");
    c->n_seg = (uint32_t)n_seg;
    c->join = c->cap > c->unit; // else no segment has a second unit
    c->space = paged_space(c->shares, c->n_seg, (size_t)c->R, (size_t)c->D);
    return 0;
}

int check_attention(const char *call, aq_ctx *ctx, const aq_paged_kv *kv, const aq_paged_batch *batch, uint32_t n_head,
                    PagedKv *pk, PagedBatch *pb) {
    AQ_REQUIRE(ctx, std::string(call) + ": null ctx");
    const int rc = check_paged(call, kv, batch, pk, pb);
    if (rc) return rc;
    AQ_REQUIRE(n_head > 0 && n_head <= 65535 && n_head % kv->n_head_kv == 0,
               std::string(call) + ": n_head " + std::to_string(n_head) + " is not a multiple of n_head_kv " +
                   std::to_string(kv->n_head_kv));
    AQ_REQUIRE((uint64_t)batch->n_rows * (n_head / kv->n_head_kv) < (1ull << 31), std::string(call) + ": batch size");
    return 0;
}

} // namespace

int launch_paged_plan(const AttnPagedArgs &a, int R, uint32_t tk, hipStream_t stream) {
    plan_kernel<<<1, 1024, 0, stream>>>(a, R, tk);
    AQ_HIP(hipGetLastError());
    return 0;
}

int launch_paged_combine(const AttnPagedArgs &a, int R, int D, hipStream_t stream) {
    const dim3 grid(a.n_seg * (uint32_t)a.kv.nkv, (uint32_t)R);
    switch (a.q.type) {
    case AQ_TYPE_F32: join_kernel<AQ_TYPE_F32><<<grid, 256, 0, stream>>>(a, R, D); break;
    case AQ_TYPE_F16: join_kernel<AQ_TYPE_F16><<<grid, 256, 0, stream>>>(a, R, D); break;
    default: join_kernel<AQ_TYPE_BF16><<<grid, 256, 0, stream>>>(a, R, D); break;
    }
    AQ_HIP(hipGetLastError());
    return 0;
}

} // namespace aq

using namespace aq;

extern "C" {

int aq_paged_attention_workspace(aq_ctx *ctx, const aq_paged_kv *kv, const aq_paged_batch *batch, uint32_t n_head,
                                 size_t *bytes) {
    AQ_REQUIRE(bytes, "aq_paged_attention_workspace: null bytes");
    int rc = check_attention("aq_paged_attention_workspace", ctx, kv, batch, n_head, nullptr, nullptr);
    if (rc) return rc;
    size_t most = 0;
    for (int f32_rows = 0; f32_rows < 2; f32_rows++) { // enough for either type of rows
        Choice c;
        rc = choose("aq_paged_attention_workspace", kv, batch, n_head, f32_rows != 0, ctx->device, &c);
        if (rc) return rc;
        most = std::max(most, c.space.bytes);
    }
    *bytes = most;
    return 0;
}

int aq_paged_attention(aq_ctx *ctx, const aq_paged_kv *kv, const aq_paged_batch *batch, uint32_t n_head,
                       const aq_heads *q, const aq_heads *out, float scale, uint32_t window, const aq_heads *gate,
                       void *workspace, size_t workspace_bytes, void *stream) {
    const char *call = "aq_paged_attention";
    AttnPagedArgs a;
    int rc = check_attention(call, ctx, kv, batch, n_head, &a.kv, &a.b);
    if (rc) return rc;
    const uint32_t rows = batch->n_rows, hd = kv->head_dim;
    rc = check_heads(call, "q", q, rows, n_head, hd);
    if (!rc) rc = check_heads(call, "out", out, rows, n_head, hd);
    if (!rc && gate) rc = check_heads(call, "gate", gate, rows, n_head, hd);
    if (rc) return rc;
    AQ_REQUIRE(q->type == AQ_TYPE_F32 || q->type == kv->type, "aq_paged_attention: rows are F32 or of the cache's type");
    AQ_REQUIRE(out->type == q->type && (!gate || gate->type == q->type),
               "aq_paged_attention: q, gate and out of different types");
    AQ_REQUIRE(std::isfinite(scale) && scale > 0.0f, "aq_paged_attention: scale");
    if (rows == 0 || batch->n_seq == 0 || batch->max_rows == 0) return 0;
    Choice c;
    rc = choose(call, kv, batch, n_head, q->type == AQ_TYPE_F32, ctx->device, &c);
    if (rc) return rc;
    AQ_REQUIRE(workspace && (uintptr_t)workspace % 16 == 0, "aq_paged_attention: workspace is null or not 16-byte aligned");
    AQ_REQUIRE(workspace_bytes >= c.space.bytes, "aq_paged_attention: workspace of " + std::to_string(workspace_bytes) +
                                                     " bytes, " + std::to_string(c.space.bytes) + " needed");
    a.q = heads_view(q);
    a.out = heads_view(out);
    if (gate) a.gate = heads_view(gate);
    a.n_head = (int)n_head;
    a.G = (int)(n_head / kv->n_head_kv);
    a.window = window;
    a.cap = c.cap;
    a.scale_log2 = scale * 1.44269504088896340736f;
    a.q_wide = heads_aligned(q, rows, n_head);
    a.out_wide = heads_aligned(out, rows, n_head) && (!gate || heads_aligned(gate, rows, n_head));
    a.shares = c.shares;
    a.min_chunk = c.min_chunk;
    a.n_seg = c.n_seg;
    a.planned = c.planned;
    char *ws = (char *)workspace;
    a.plan = (uint32_t *)(ws + c.space.plan);
    a.seg_seq = (uint32_t *)(ws + c.space.seg);
    a.seg_rt = a.seg_seq + c.n_seg;
    a.part_o = (float *)(ws + c.space.o);
    a.part_ml = (float *)(ws + c.space.ml);
    AQ_HIP(hipSetDevice(ctx->device));
    const hipStream_t st = stream ? (hipStream_t)stream : ctx->stream;
    if (c.planned) {
        rc = launch_paged_plan(a, c.R, c.unit, st);
        if (rc) return rc;
    }
    if (c.many) {
        rc = launch_paged_chunk(a, c.D, st);
    } else if (q->type == AQ_TYPE_F32) {
        if (kv->type == AQ_TYPE_F32) rc = few_pick<AQ_TYPE_F32, true>(a, c.D, c.R, st);
        else if (kv->type == AQ_TYPE_F16) rc = few_pick<AQ_TYPE_F16, true>(a, c.D, c.R, st);
        else rc = few_pick<AQ_TYPE_BF16, true>(a, c.D, c.R, st);
    } else if (kv->type == AQ_TYPE_F16) {
        rc = few_pick<AQ_TYPE_F16, false>(a, c.D, c.R, st);
    } else {
        rc = few_pick<AQ_TYPE_BF16, false>(a, c.D, c.R, st);
    }
    if (rc || !c.join) return rc;
    return launch_paged_combine(a, c.R, c.D, st);
}

} // extern "C"
