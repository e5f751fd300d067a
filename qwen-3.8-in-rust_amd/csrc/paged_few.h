// paged_few.h — attention of few rows over a paged cache (paged_attn.h): single tokens, verify batches, and f32 rows of any
// number. Instantiated per cache type in paged_few_*.hip.
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
// 16-bit rows: the exponentials are rounded to the rows' type for the second product, once, and summed as rounded. Largest
// error against 64 bits, relative to the largest output, where the output's rounding alone gives 0.0017 (bf16) and 0.00020
// (f16): 0.0020 and 0.00022. A second piece of them, as f32 rows have, would take that away: single tokens of 48 sequences
// at 6000 1% slower, at 3000 with heads of 64 5%, of 64 at 130 5%, verify batches 1 to 2%. Callers to whom it matters have
// f32 rows.
//
// Measured: single tokens of 48 sequences at 6000 (bf16, 32 heads on 8 of 128) 215 to 223 us by card, 5.5 to 5.3 TB/s, where
// a plain read reaches 6.3; of one sequence at 8000 (f16, 24 heads on 4 of 256) 17.8 us, two launches of latencies; four
// new tokens of eight sequences at 3000 (f32 over f16, the same heads) 42.5 to 44.1 us, 2.5 TB/s: its 16 rows of 256
// outputs leave registers for two waves a SIMD, which wait for loads 55% of their time. Eight waves to a work-group there:
// 40.4 us for 42.7, but contexts below 1000 1 to 2 us slower and single tokens 5 to 8%.
//
// f32 rows over a 16-bit cache keep 32-bit accuracy: q, scaled to its row's exponent, and the probabilities go in as two
// f16 or three bf16 pieces whose sum has 22 or 24 bits. f32 over f32 takes the f32 matrix cores (16x16x4).
#pragma once

#include <type_traits>

#include "paged_attn.h"

namespace aq {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));

__device__ const u4 zeros = {0, 0, 0, 0};

template <int CT>
__device__ __forceinline__ f4 mfma16(u4 a, u4 b, f4 c) {
    if constexpr (CT == AQ_TYPE_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

// O^T += V^T P^T over 32 positions (16-byte operands) or 16 (8-byte ones).
template <int CT>
__device__ __forceinline__ f4 mfma_pv(u4 a, u4 b, f4 c) {
    return mfma16<CT>(a, b, c);
}
template <int CT>
__device__ __forceinline__ f4 mfma_pv(u2 a, u2 b, f4 c) {
    if constexpr (CT == AQ_TYPE_F16)
        return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(h4, a), __builtin_bit_cast(h4, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s4, a), __builtin_bit_cast(s4, b), c, 0, 0, 0);
}

// v as NP operands of the type: each the rounding of what the ones before left.
template <int CT, int NP, typename V>
__device__ __forceinline__ void pieces(const float *v, V *out) {
    using T = typename RowType<CT>::type;
    constexpr int N = sizeof(V) / 2;
    typedef T vec __attribute__((ext_vector_type(N)));
    float rest[N];
#pragma unroll
    for (int i = 0; i < N; i++) rest[i] = v[i];
#pragma unroll
    for (int p = 0; p < NP; p++) {
        vec x;
#pragma unroll
        for (int i = 0; i < N; i++) {
            x[i] = (T)rest[i];
            if (p + 1 < NP) rest[i] -= (float)x[i];
        }
        out[p] = __builtin_bit_cast(V, x);
    }
}

// An infinity or a NaN.
__device__ __forceinline__ bool odd_f32(unsigned w) { return (w & 0x7F800000u) == 0x7F800000u; }

// What the kernel keeps where.
template <int CT, bool FQ, int D, int ROWS>
struct FewShape {
    static constexpr int R = ROWS, RG = few_groups(CT, D, R), KW = WAVES / RG, NT = R / 16, NR = NT / RG;
    static constexpr bool F = CT == AQ_TYPE_F32;
    static constexpr int NP = !FQ || F ? 1 : (CT == AQ_TYPE_F16 ? 2 : 3); // pieces of q and of the probabilities
    static constexpr int TILE = few_tile(D);  // positions of a wave's step
    static constexpr int E = TILE / 4;                // of them a lane's: 16 (e / 4) + 4 g + e % 4
    static constexpr int STEPS = F ? D / 16 : D / 32; // 16-byte K operands of a row per lane
    static constexpr int VB = F || D == 64 ? 4 : 8;   // dimensions of a V row per lane and chunk
    static constexpr int CHUNKS = D / (16 * VB);
    static constexpr int ACC = CHUNKS * VB; // accumulators (4 values each) per row tile
    static constexpr int PASSES = D / 64, CROW = 68;  // the waves' outputs meet 64 dimensions at a time
    static constexpr int QF = NT * STEPS * NP * 64 * 16, CB = KW * R * CROW * 4; // bytes of q; of the meeting
    static constexpr int LDS = (QF > CB ? QF : CB) + KW * R * 8;
};

// EXACT: the head fills D, so that a row's loads differ by constants only.
template <int CT, bool FQ, int D, int R, bool EXACT>
__global__ void __launch_bounds__(256, 2) few_rows_kernel(AttnPagedArgs a) {
    using S = FewShape<CT, FQ, D, R>;
    constexpr bool F = S::F;
    constexpr int QT = FQ ? AQ_TYPE_F32 : CT, NP = S::NP, STEPS = S::STEPS, CHUNKS = S::CHUNKS, VB = S::VB;
    constexpr int RG = S::RG, KW = S::KW, NT = S::NT, NR = S::NR;
    constexpr int TILE = S::TILE, UNIT = KW * TILE, E = S::E, HT = TILE / 16, ES = F ? 4 : 2;
    // f16 probabilities are kept at 2^14 times their size (and so are the sums): their small ones stay normal numbers
    constexpr float P_SHIFT = CT == AQ_TYPE_F16 ? 14.0f : 0.0f;
    extern __shared__ __align__(16) char smem[];
    u4 *qf = reinterpret_cast<u4 *>(smem);
    float *comb = reinterpret_cast<float *>(smem);                           // [KW][R][CROW], after the last tile
    float *ml = reinterpret_cast<float *>(smem + S::LDS - KW * R * 8); // [KW][R][2]
    __shared__ PlanLds plan;
    __shared__ uint32_t qmax[R];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4, rg = wave % RG, kg = wave / RG; // which rows, which positions
    const int hd = EXACT ? D : a.kv.hd, G = a.G;

    const Share sh = take_share(a, R, UNIT, plan);
    uint32_t u = sh.begin, j = sh.j, kv_at = sh.kvh;
    while (u < sh.end) { // uniform
        const Segment sg = next_segment(a, R, UNIT, plan, sh, u, j, kv_at);
        if (sg.t1 <= sg.t0) continue;
        const uint32_t kvh = sg.kvh;
        const int32_t r0 = sg.r0;
        const SeqRows sr = paged_seq(a.b, sg.seq);
        const int32_t n_rows = sr.n * G, base = sr.base;
        const UnitRange range = tile_units(a, sr, r0, R, UNIT);
        const int32_t tok0 = (int32_t)a.by_g.quot(r0), tok1 = (int32_t)a.by_g.quot(min(r0 + R, n_rows) - 1);
        const int32_t kend = min(max(base + tok1 + 1, 0), (int32_t)a.cap);
        // before this position nobody of the tile looks: there is no page there, whatever it holds
        const int32_t kbegin = a.window ? (int32_t)max((int64_t)base + tok0 + 1 - (int64_t)a.window, (int64_t)0) : 0;
        const int32_t min_hi = base + tok0 + 1;
        const int64_t max_lo = a.window ? (int64_t)base + tok1 + 1 - (int64_t)a.window : INT64_MIN;
        const int32_t *table = a.b.pages + (size_t)sg.seq * a.b.max_pages;
        const uint64_t head_off = (uint64_t)kvh * a.kv.head_bytes;
        const char *const kpool = a.kv.k + head_off, *const vpool = a.kv.v + head_off;

        const int32_t last_tile = min((int32_t)((range.lo + sg.t1) * KW), (kend + TILE - 1) / TILE);
        int32_t tile = (int32_t)(range.lo + sg.t0) * KW + kg;
        // where a tile's rows are: lane l has position l % TILE's page entry, then its place; bit l: it has a page
        auto entry = [&](int32_t t) {
            const int32_t p = t * TILE + lane % TILE;
            return t < last_tile && p >= kbegin && p < kend ? paged_entry(a.kv, table, a.b.max_pages, (uint32_t)p) : 0xFFFFFFFFu;
        };
        auto locate = [&](int32_t t, uint32_t e, uint32_t *units) {
            const bool ok = paged_units(a.kv, e, (uint32_t)(t * TILE + lane % TILE), units);
            return (uint32_t)__ballot(ok) & (uint32_t)((1ull << TILE) - 1);
        };
        constexpr uint32_t ALL = (uint32_t)((1ull << TILE) - 1);
        auto row_off = [&](uint32_t units, int pos) {
            return (uint64_t)(uint32_t)__shfl((int)units, pos) << a.kv.unit_shift;
        };
        // 16 rows of K as operands; dimensions past the head are zeros like q's there (0 times an infinity would be a NaN),
        // chosen by the address, so that nothing waits for the load
        auto load_k = [&](uint32_t units, int t, u4 *k) {
            const char *p = kpool + (row_off(units, 16 * t + r) + 16 * g);
#pragma unroll
            for (int s = 0; s < STEPS; s++)
                k[s] = *reinterpret_cast<const u4 *>(EXACT || 64 * s + 16 * g < hd * ES ? p + 64 * s : (const char *)&zeros);
        };
        using VV = typename std::conditional<VB * ES == 8, u2, u4>::type;
        using VP = typename std::conditional<HT == 1, u2, u4>::type; // probabilities, V^T: E 16-bit values
        constexpr int VW = VB * ES / 4; // dwords
        // the row of this lane's e-th position: dimensions VB r .. of each chunk; past the head: outputs not stored
        auto load_v = [&](uint32_t units, int e, VV *v, int stride) {
            const char *p = vpool + (row_off(units, 16 * (e / 4) + 4 * g + e % 4) + (EXACT ? VB * ES * r : 0));
#pragma unroll
            for (int c = 0; c < CHUNKS; c++) {
                const int at = EXACT ? c * 16 * VB * ES : min(c * 16 * VB + VB * r, hd - VB) * ES;
                v[c * stride] = *reinterpret_cast<const VV *>(p + at);
            }
        };

        u4 k[HT][STEPS];
        uint32_t units = 0, okm = 0;
        uint32_t next = entry(tile); // page entries of the tile after this one, on their way for a tile's time
        if (tile < last_tile) {
            okm = locate(tile, next, &units);
            next = entry(tile + KW);
        }

        // this lane's rows: the positions they see are lo .. hi - 1
        int32_t hi[NR], lo[NR];
#pragma unroll
        for (int nr = 0; nr < NR; nr++) {
            const int32_t rr = r0 + 16 * (rg * NR + nr) + r, tok = (int32_t)a.by_g.quot(rr);
            hi[nr] = rr < n_rows ? base + tok + 1 : 0;
            const int64_t l = a.window ? (int64_t)base + tok + 1 - (int64_t)a.window : 0;
            lo[nr] = l > 0 ? (int32_t)l : 0;
        }

        __syncthreads(); // the LDS of the segment before is read
        // ---- queries into the LDS, operand order; 16 rows x 16 units of 8 (4) dimensions at a time
        float rscale[NR]; // what this lane's rows' scores are multiplied by
        {
            constexpr int QV = F ? 4 : 8, UN = NT * (D / QV), UNITS = (UN + 15) / 16;
            const int th = here(tid), n = th & 15;
            float v[UNITS][QV];
            if constexpr (NP == 2) {
                if (th < R) qmax[th] = 0;
                __syncthreads();
            }
#pragma unroll
            for (int i = 0; i < UNITS; i++) {
                const int unit = i * 16 + (th >> 4), nr = unit / (D / QV), at = unit % (D / QV) * QV;
                if (UN % 16 && unit >= UN) continue;
                const int32_t rr = r0 + 16 * nr + n, tok = (int32_t)a.by_g.quot(rr);
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
                const int unit = i * 16 + (th >> 4), nr = unit / (D / QV), at = unit % (D / QV);
                if (UN % 16 && unit >= UN) continue;
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
                rscale[nr] = NP == 2 ? a.scale_log2 * __uint_as_float(exponent(16 * (rg * NR + nr) + r) << 23) : a.scale_log2;
        }
        if (tile < last_tile) {
#pragma unroll
            for (int t = 0; t < HT; t++) load_k(units, t, k[t]);
        }
        __syncthreads();

        // ---- the wave's tiles
        f4 o[NR][S::ACC];
        float m[NR], l[NR];
#pragma unroll
        for (int nr = 0; nr < NR; nr++) {
            m[nr] = -INFINITY;
            l[nr] = 0.0f;
#pragma unroll
            for (int i = 0; i < S::ACC; i++) o[nr][i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        // The scores of one tile, in place: scaled, hidden ones taken out, then their exponentials against the running
        // maximum, which the sums and outputs follow.
        auto soften = [&](int nr, float *x, int32_t kb, uint32_t ok, bool edge) {
            float mt = -INFINITY;
#pragma unroll
            for (int e = 0; e < E; e++) x[e] *= rscale[nr];
            if (edge) {
                const int gh = here(4 * g);
                const int hr = hi[nr] - kb - gh, lr = lo[nr] - kb - gh; // of the lane's first position
                const uint32_t mine = ok >> gh;
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const int pos = 16 * (e / 4) + e % 4;
                    x[e] = pos < hr && pos >= lr && ((mine >> pos) & 1) ? x[e] : -INFINITY;
                }
            }
#pragma unroll
            for (int e = 0; e < E; e++) mt = fmaxf(mt, x[e]);
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
            for (int e = 0; e < E; e++) {
                x[e] = fast_exp2((x[e] - mu) + P_SHIFT);
                if (F || NP > 1) l[nr] += x[e];
            }
        };

        for (; tile < last_tile; tile += KW) {
            asm volatile("" ::: "memory"); // q's operands are read from the LDS each time, not kept in registers
            const int32_t kb = tile * TILE;
            const uint32_t now = units, ok = okm;
            const bool edge = kb + TILE > min_hi || (int64_t)kb < max_lo || ok != ALL; // uniform
            f4 s[NR][HT];
#pragma unroll
            for (int nr = 0; nr < NR; nr++)
#pragma unroll
                for (int t = 0; t < HT; t++) s[nr][t] = f4{0.0f, 0.0f, 0.0f, 0.0f};

            if constexpr (!F) {
                VV v[CHUNKS][E];
                okm = locate(tile + KW, next, &units);
                next = entry(tile + 2 * KW);
#pragma unroll
                for (int e = 0; e < E; e++) load_v(now, e, &v[0][e], E);
                const u4 *ql = qf + rg * NR * STEPS * NP * 64 + here(lane);
#pragma unroll
                for (int st = 0; st < STEPS; st++)
#pragma unroll
                    for (int nr = 0; nr < NR; nr++)
#pragma unroll
                        for (int p = 0; p < NP; p++) {
                            const u4 q = ql[((nr * STEPS + st) * NP + p) * 64];
#pragma unroll
                            for (int t = 0; t < HT; t++) s[nr][t] = mfma16<CT>(k[t][st], q, s[nr][t]);
                            if (nr == NR - 1 && p == NP - 1 && st % 2 == 1) __builtin_amdgcn_sched_barrier(0);
                        }
                if constexpr (NP > 1) { // an infinite key times the pieces of one number is a NaN: by the first piece alone
                    bool nan = false;
#pragma unroll
                    for (int nr = 0; nr < NR; nr++)
#pragma unroll
                        for (int e = 0; e < E; e++) nan |= s[nr][e / 4][e % 4] != s[nr][e / 4][e % 4];
                    if (__any(nan)) {
#pragma unroll
                        for (int nr = 0; nr < NR; nr++)
#pragma unroll
                            for (int t = 0; t < HT; t++) {
                                f4 one = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                                for (int st = 0; st < STEPS; st++)
                                    one = mfma16<CT>(k[t][st], ql[(nr * STEPS + st) * NP * 64], one);
#pragma unroll
                                for (int i = 0; i < 4; i++) s[nr][t][i] = s[nr][t][i] == s[nr][t][i] ? s[nr][t][i] : one[i];
                            }
                    }
                }
                if (tile + KW < last_tile) { // the next tile's K rows, while this one is summed
#pragma unroll
                    for (int t = 0; t < HT; t++) load_k(units, t, k[t]);
                }
                VP pf[NR][NP];
#pragma unroll
                for (int nr = 0; nr < NR; nr++) {
                    float x[E];
#pragma unroll
                    for (int e = 0; e < E; e++) x[e] = s[nr][e / 4][e % 4];
                    soften(nr, x, kb, ok, edge);
                    pieces<CT, NP>(x, pf[nr]);
                    if constexpr (NP == 1) { // the sum is of what the product takes, so that roundings weigh on both alike
#pragma unroll
                        for (int h = 0; h < E / 2; h++) l[nr] = add2<CT>(pf[nr][0][h], l[nr]);
                    }
                }
                if (edge) { // rows of positions that no page holds are not numbers that may be multiplied by 0
                    const uint32_t mine = ok >> here(4 * g);
#pragma unroll
                    for (int e = 0; e < E; e++)
#pragma unroll
                        for (int c = 0; c < CHUNKS; c++)
#pragma unroll
                            for (int x = 0; x < VW; x++)
                                v[c][e][x] = (mine >> (16 * (e / 4) + e % 4)) & 1 ? v[c][e][x] : 0u;
                }
#pragma unroll
                for (int c = 0; c < CHUNKS; c++) {
                    auto product = [&](int jj) { // V^T operand of dimension jj of each lane's VB
                        VP t;
                        const unsigned sel = jj & 1 ? 0x07060302u : 0x05040100u;
#pragma unroll
                        for (int h = 0; h < E / 2; h++)
                            t[h] = __builtin_amdgcn_perm(v[c][2 * h + 1][jj / 2], v[c][2 * h][jj / 2], sel);
                        return t;
                    };
                    if ((edge && tok0 < tok1) || NP > 1) { // one token's rows all see what has a page
                        // Nor are infinities and NaN of positions that only some of the rows see, and an infinity times
                        // the pieces of one number is a NaN: such values are added position by position, to the rows
                        // that see them, by the probability's first piece, and taken out of the product of the others.
                        unsigned any = 0;
#pragma unroll
                        for (int e = 0; e < E; e++)
#pragma unroll
                            for (int x = 0; x < VW; x++) any |= odd_bits<CT>(v[c][e][x]);
                        if (__any(any & 0x80008000u)) {
#pragma unroll 1
                            for (int pos = 0; pos < TILE; pos++) {
                                const int e = 4 * (pos / 16) + pos % 4; // its k-slot
#pragma unroll
                                for (int i = 0; i < E; i++) // nothing of the operands is kept from before the loop
#pragma unroll
                                    for (int x = 0; x < VW; x++) asm volatile("" : "+v"(v[c][i][x]));
                                VP only = {};
                                if (pos % 16 / 4 == g) only[e / 2] = e & 1 ? 0xFFFF0000u : 0x0000FFFFu;
#pragma unroll
                                for (int nr = 0; nr < NR; nr++) {
                                    const bool sees = kb + pos < hi[nr] && kb + pos >= lo[nr];
#pragma unroll
                                    for (int jj = 0; jj < VB; jj++) {
                                        VP vt = product(jj) & only;
#pragma unroll
                                        for (int x = 0; x < E / 2; x++) vt[x] &= odd_mask<CT>(vt[x]);
                                        const f4 t = mfma_pv<CT>(vt, pf[nr][0], o[nr][c * VB + jj]);
#pragma unroll
                                        for (int x = 0; x < 4; x++)
                                            o[nr][c * VB + jj][x] = sees ? t[x] : o[nr][c * VB + jj][x];
                                    }
                                }
                            }
#pragma unroll
                            for (int e = 0; e < E; e++)
#pragma unroll
                                for (int x = 0; x < VW; x++) v[c][e][x] &= ~odd_mask<CT>(v[c][e][x]);
                        }
                    }
#pragma unroll
                    for (int jj = 0; jj < VB; jj++) {
                        const VP vt = product(jj);
#pragma unroll
                        for (int nr = 0; nr < NR; nr++)
#pragma unroll
                            for (int p = 0; p < NP; p++)
                                o[nr][c * VB + jj] = mfma_pv<CT>(vt, pf[nr][p], o[nr][c * VB + jj]);
                        if (jj % 2 == 1) __builtin_amdgcn_sched_barrier(0);
                    }
                }
            } else {
                // ---- f32 cache: 16 positions at a time, k-slot g of step i stands for position 16 t + 4 g + i
                auto mul = [](unsigned x, unsigned y, f4 c) {
                    return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(x), __uint_as_float(y), c, 0, 0, 0);
                };
                constexpr int VI = D == 64 ? 8 : 4; // V rows in registers at once
                okm = locate(tile + KW, next, &units);
                next = entry(tile + 2 * KW);
                VV v[CHUNKS][VI];
                const u4 *ql = qf + rg * NR * STEPS * NP * 64 + here(lane);
#pragma unroll
                for (int i = 0; i < VI; i++) load_v(now, i, &v[0][i], VI);
#pragma unroll
                for (int st = 0; st < STEPS; st++)
#pragma unroll
                    for (int nr = 0; nr < NR; nr++) {
                        const u4 q = ql[(nr * STEPS + st) * 64];
#pragma unroll
                        for (int i = 0; i < 4; i++)
#pragma unroll
                            for (int t = 0; t < HT; t++) s[nr][t] = mul(k[t][st][i], q[i], s[nr][t]);
                    }
                if (tile + KW < last_tile) { // the next tile's K rows, while this one is summed
#pragma unroll
                    for (int t = 0; t < HT; t++) load_k(units, t, k[t]);
                }
                float x[NR][E];
#pragma unroll
                for (int nr = 0; nr < NR; nr++) {
#pragma unroll
                    for (int e = 0; e < E; e++) x[nr][e] = s[nr][e / 4][e % 4];
                    soften(nr, x[nr], kb, ok, edge);
                }
#pragma unroll
                for (int t = 0; t < HT; t++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        if (VI == 4 && i == 0 && t) {
#pragma unroll
                            for (int y = 0; y < 4; y++) load_v(now, 4 * t + y, &v[0][y], VI);
                        }
                        if (edge) { // as above
                            const int pos0 = 16 * t + i; // + 4 g
                            const bool keep = (ok >> (pos0 + here(4 * g))) & 1;
                            bool is_odd = false;
#pragma unroll
                            for (int c = 0; c < CHUNKS; c++)
#pragma unroll
                                for (int y = 0; y < 4; y++) {
                                    v[c][(4 * t + i) % VI][y] = keep ? v[c][(4 * t + i) % VI][y] : 0u;
                                    is_odd |= odd_f32(v[c][(4 * t + i) % VI][y]);
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
                                                const f4 n = mul(g == gg ? v[c][(4 * t + i) % VI][y] : 0u,
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
                                    for (int y = 0; y < 4; y++) v[c][(4 * t + i) % VI][y] = out ? 0u : v[c][(4 * t + i) % VI][y];
                            }
                        }
#pragma unroll
                        for (int c = 0; c < CHUNKS; c++)
#pragma unroll
                            for (int y = 0; y < 4; y++)
#pragma unroll
                                for (int nr = 0; nr < NR; nr++)
                                    o[nr][c * 4 + y] = mul(v[c][(4 * t + i) % VI][y], __float_as_uint(x[nr][4 * t + i]), o[nr][c * 4 + y]);
                    }
                }
            }
        }

        // ---- the waves' rows joined: each scaled to the common maximum, then added, 64 dimensions a pass
#pragma unroll
        for (int nr = 0; nr < NR; nr++) {
            l[nr] += __shfl_xor(l[nr], 16);
            l[nr] += __shfl_xor(l[nr], 32);
            if (g == 0) {
                ml[(kg * R + 16 * (rg * NR + nr) + r) * 2] = m[nr];
                ml[(kg * R + 16 * (rg * NR + nr) + r) * 2 + 1] = l[nr];
            }
        }
        __syncthreads(); // every wave is past its tiles: q's place is the meeting's now
        const int th = here(tid);
        float *const cw = comb + (size_t)(kg * R + 16 * rg * NR + (th & 15)) * S::CROW + 16 * (th >> 4 & 3);
        float mine[NR];
#pragma unroll
        for (int nr = 0; nr < NR; nr++) {
            float mx = -INFINITY;
#pragma unroll
            for (int x = 0; x < KW; x++) mx = fmaxf(mx, ml[(x * R + 16 * (rg * NR + nr) + (th & 15)) * 2]);
            mine[nr] = fast_exp2(m[nr] - (mx == -INFINITY ? 0.0f : mx));
        }
        const bool cut = is_cut(sg);
        const uint32_t slot = part_slot(sg, sh);
        // this thread's row (+ 16 it) and its values of a pass: the waves' sums, their maximum
        const int row0 = th >> 4, v0 = (th & 15) * 4;
        float lt[NT], mx[NT];
#pragma unroll
        for (int it = 0; it < NT; it++) {
            const float *p = ml + (it * 16 + row0) * 2;
            mx[it] = p[0];
#pragma unroll
            for (int x = 1; x < KW; x++) mx[it] = fmaxf(mx[it], p[x * R * 2]);
            lt[it] = 0.0f;
#pragma unroll
            for (int x = 0; x < KW; x++)
                lt[it] += p[x * R * 2 + 1] * fast_exp2(p[x * R * 2] - (mx[it] == -INFINITY ? 0.0f : mx[it]));
            if (cut && v0 == 0 && r0 + it * 16 + row0 < n_rows) {
                float *d = a.part_ml + ((size_t)slot * R + it * 16 + row0) * 2;
                d[0] = mx[it];
                d[1] = lt[it];
            }
        }
#pragma unroll
        for (int pass = 0; pass < S::PASSES; pass++) {
            if (pass) __syncthreads();
#pragma unroll
            for (int nr = 0; nr < NR; nr++) {
                float *c = cw + 16 * nr * S::CROW;
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
            const int dim = VB == 4 ? 64 * pass + v0
                                    : 128 * (pass >> 1) + 8 * (4 * (v0 >> 4) + 2 * (pass & 1) + ((v0 >> 3) & 1)) + (v0 & 7);
#pragma unroll
            for (int it = 0; it < NT; it++) {
                const int row = it * 16 + row0;
                const int32_t rr = r0 + row;
                if (rr >= n_rows || dim >= hd) continue;
                f4 sum = *reinterpret_cast<const f4 *>(comb + (size_t)row * S::CROW + v0);
#pragma unroll
                for (int x = 1; x < KW; x++) {
                    const f4 t = *reinterpret_cast<const f4 *>(comb + (size_t)(x * R + row) * S::CROW + v0);
#pragma unroll
                    for (int y = 0; y < 4; y++) sum[y] += t[y];
                }
                if (cut) {
                    *reinterpret_cast<f4 *>(a.part_o + ((size_t)slot * R + row) * D + dim) = sum;
                } else {
                    const int32_t tok = (int32_t)a.by_g.quot(rr);
                    float out[4];
#pragma unroll
                    for (int y = 0; y < 4; y++) out[y] = lt[it] == 0.0f ? 0.0f : sum[y] / lt[it];
                    store_out<QT>(a, sr.first + tok, (int)kvh * G + (rr - tok * G), dim, out);
                }
            }
        }
    }
}

template <int CT, bool FQ, int D, int R, bool EXACT>
int few_launch(const AttnPagedArgs &a, hipStream_t stream) {
    using S = FewShape<CT, FQ, D, R>;
    const auto kernel = few_rows_kernel<CT, FQ, D, R, EXACT>;
    static_assert(S::LDS + sizeof(PlanLds) + R * 4 <= 64 * 1024, "more LDS than a launch has without asking for it");
    kernel<<<a.shares, 256, S::LDS, stream>>>(a);
    AQ_HIP(hipGetLastError());
    return 0;
}
template <int CT, bool FQ, int D>
int few_rows(const AttnPagedArgs &a, int R, hipStream_t stream) {
    if (a.kv.hd == D) return R == 16 ? few_launch<CT, FQ, D, 16, true>(a, stream) : few_launch<CT, FQ, D, 32, true>(a, stream);
    return R == 16 ? few_launch<CT, FQ, D, 16, false>(a, stream) : few_launch<CT, FQ, D, 32, false>(a, stream);
}
template <int CT, bool FQ>
int few_pick(const AttnPagedArgs &a, int D, int R, hipStream_t stream) {
    if (D == 64) return few_rows<CT, FQ, 64>(a, R, stream);
    if (D == 128) return few_rows<CT, FQ, 128>(a, R, stream);
    return few_rows<CT, FQ, 256>(a, R, stream);
}

} // namespace
} // namespace aq
