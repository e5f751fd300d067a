// paged_chunk.hip — attention of many 16-bit rows (prompt chunks, whole prompts) over a paged cache of their type: bound
// by the matrix cores (4 D flops a row and position).
//
// A work-group's 128 rows lie on four waves of 32; the keys come in tiles of 64 (heads past 128: 32), K and V through
// the LDS, the next tile loaded while this one is summed:
//   S^T = K Q^T   32x32x16: A = K from the LDS, B = Q^T in registers for the whole segment. Lane (n, h) = (lane & 31,
//                 lane >> 5) then holds row n's scores of positions 8 (i / 4) + 4 h + i % 4, so that a row's maximum and
//                 sum are in two lanes: one exchange (v_permlane32_swap) per tile.
//   O^T = V^T P^T the exponentials, rounded, are B's layout as they stand if k-slot (h, e) stands for position 8 (e / 4) +
//                 4 h + e % 4; A = V^T comes from the row-major V tile by transposing LDS reads (ds_read_b64_tr_b16).
//                 Rounded to the rows' type, once, and summed as rounded: a second piece would be half as many products
//                 again in a kernel that they bound. Largest error against 64 bits, relative to the largest output: bf16
//                 0.0023, f16 0.00026, where the output's rounding alone gives 0.0017 and 0.00020.
// The maximum a row's exponentials are taken against moves only when it grows by more than 2^7 (their scale leaves room
// for that), so that outputs are rarely rescaled.
//
// Tiles are loaded straight into the LDS (16 bytes a lane, consecutive lanes consecutive addresses), each lane choosing
// which 16 bytes of its row it fetches: the row's chunks are swapped by an exclusive or with the row's low bits, so that
// neither kind of read meets a bank twice. Rows without a page come from a row of zeros.
//
// Measured, by card: 512 rows of 24 heads on 4 of 256 at 32,000 (bf16) 472 to 492 us, 860 to 825 TFLOP/s, where a library
// product of 8192^3 reaches 1121; prompts of three requests of 3500, 32 heads on 8 of 128 (f16), 411 to 433 us, 736 to 698.
// Heads that do not fill their padded size load by an address each: 512 rows at 8000, heads of 192, 98 us for 95 without
// the zeros past the head. Products and softmax (per score a product, an exponential, a rounding, half a sum) take turns on
// two waves a SIMD; at heads of 256 the next tile's products beside this one's softmax need the registers that hold the
// rows (770 for 792 TFLOP/s). Heads of 128 and 64 leave some (198 and 150 registers); it was not tried there.
#include <atomic>
#include <type_traits>

#include "paged_attn.h"

namespace aq {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef short s4 __attribute__((ext_vector_type(4)));

__device__ const u4 zeros = {0, 0, 0, 0};

template <int CT>
__device__ __forceinline__ f16v mfma32(u4 a, u4 b, f16v c) {
    if constexpr (CT == AQ_TYPE_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

template <int CT>
__device__ __forceinline__ unsigned pack2(float x, float y) {
    using E = typename RowType<CT>::type;
    typedef E e2 __attribute__((ext_vector_type(2)));
    typedef float f2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, __builtin_convertvector(f2{x, y}, e2));
}

// The larger of x's two halves (lanes l and l + 32).
__device__ __forceinline__ float both_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

template <int D>
struct ChunkShape {
    static constexpr int RB = D * 2, CPR = D / 8;             // bytes and 16-byte chunks of a row
    static constexpr int KEYS = chunk_keys(D), HALVES = KEYS / 32; // positions of a tile; 32 x 32 score tiles
    static constexpr int TILE_BYTES = KEYS * RB;
    static constexpr int LOADS = TILE_BYTES / (256 * 16);     // 16-byte loads per thread and tile, of K and of V
    static constexpr int OROW = 68;                           // floats of a row of 64 outputs there
    static constexpr int OUT = CHUNK_ROWS * OROW * 4, LDS = 4 * TILE_BYTES > OUT ? 4 * TILE_BYTES : OUT; // two buffers of each
    // Which chunk of row r lies at place p: p ^ swizzle(r). A clock serves 256 bytes: of K 16 bytes of 16 rows, which all
    // have another value; of V 64 bytes of four rows, whose values differ above those four chunks. Linear: swizzle(x ^ y) =
    // swizzle(x) ^ swizzle(y).
    static __host__ __device__ constexpr uint32_t swizzle(uint32_t r) {
        return D == 64 ? (r >> 1 & 1) << 2 | (r >> 2 & 3) : (r & 3) << 2 | (r >> 2 & 3);
    }
};

#define AQ_LDS __attribute__((address_space(3)))
#define AQ_GLB __attribute__((address_space(1)))

// Rows row0 + 8 i (i < 4) of a wave's 32, from w0 on: eight outputs each, at x + row * stride; times the gate, rounded,
// stored. All four gates are on their way before the first is used.
template <int CT>
__device__ __forceinline__ void store_rows(const AttnPagedArgs &a, const SeqRows &sr, int kvh, int32_t w0, int32_t n_rows,
                                           int dim, int row0, const float *x, int stride) {
    using E = typename RowType<CT>::type;
    typedef E vec __attribute__((ext_vector_type(8)));
    int64_t row[4], head[4];
    bool have[4];
    vec gate[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int32_t rr = w0 + row0 + 8 * i, tok = (int32_t)a.by_g.quot(rr);
        have[i] = rr < n_rows && dim < a.kv.hd;
        row[i] = sr.first + tok;
        head[i] = kvh * a.G + (rr - tok * a.G);
        if (a.gate.p && have[i]) {
            const E *g = (const E *)a.gate.p + row[i] * a.gate.row + head[i] * a.gate.head + dim;
            if (a.out_wide) {
                gate[i] = *reinterpret_cast<const vec *>(g);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) gate[i][e] = g[e];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const f4 u = *reinterpret_cast<const f4 *>(x + (row0 + 8 * i) * stride),
                 v = *reinterpret_cast<const f4 *>(x + (row0 + 8 * i) * stride + 4);
        vec y;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            float z = e < 4 ? u[e & 3] : v[e & 3];
            if (a.gate.p) z *= 1.0f / (1.0f + expf(-(float)gate[i][e]));
            y[e] = (E)z;
        }
        if (!have[i]) continue;
        E *o = (E *)a.out.p + row[i] * a.out.row + head[i] * a.out.head + dim;
        if (a.out_wide) {
            *reinterpret_cast<vec *>(o) = y;
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) o[e] = y[e];
        }
    }
}

template <int CT, int D>
__global__ void __launch_bounds__(256, 2) chunk_kernel(AttnPagedArgs a) {
    using S = ChunkShape<D>;
    constexpr int R = CHUNK_ROWS, KEYS = S::KEYS, HALVES = S::HALVES, STEPS = D / 16, DB = D / 32;
    // Exponentials lie up to 2^GROW over those of the maximum they are taken against. f16: between 2^7 and 2^14, so that small
    // ones stay normal numbers; bf16, whose values may be as large as sums are: never above 1.
    constexpr float GROW = 7.0f, P_SHIFT = CT == AQ_TYPE_F16 ? 7.0f : -GROW;
    extern __shared__ __align__(16) char smem[];
    __shared__ PlanLds plan;
    char *kbuf = smem, *vbuf = smem + 2 * S::TILE_BYTES;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hd = a.kv.hd, G = a.G;

    // LDS addresses of this lane's reads of K (operand step 0) and V (dimensions 0 .. 31); the other steps by an exclusive
    // or, rows and chunks from 16 on by constant offsets
    const int n0 = lane & 31, h0 = lane >> 5, vi = lane & 15, vkey = 4 * h0 + vi / 4;
    const int kaddr0 = n0 * S::RB + (int)((h0 ^ S::swizzle(n0)) << 4);
    const int vaddr0 = vkey * S::RB + (int)(((2 * ((lane >> 4) & 1) + (vi % 4) / 2) ^ S::swizzle(vkey)) << 4) + (vi % 2) * 8;

    const Share sh = take_share(a, R, KEYS, plan);
    uint32_t u = sh.begin, j = sh.j, kv_at = sh.kvh;
    while (u < sh.end) { // uniform
        const Segment sg = next_segment(a, R, 0, plan, sh, u, j, kv_at);
        if (sg.t1 <= sg.t0) continue;
        const int n = here(n0), h = here(h0);
        const SeqRows sr = paged_seq(a.b, sg.seq);
        const int32_t n_rows = sr.n * G, base = sr.base;
        const UnitRange range = tile_units(a, sr, sg.r0, R, KEYS);
        const int32_t *table = a.b.pages + (size_t)sg.seq * a.b.max_pages;
        const uint64_t head_off = (uint64_t)sg.kvh * a.kv.head_bytes;
        const int32_t seg_last = (int32_t)a.by_g.quot(min(sg.r0 + R, n_rows) - 1);
        const int32_t kend = min(max(base + seg_last + 1, 0), (int32_t)a.cap); // positions from here on: nobody's

        // this lane's row, and what the wave's rows see between them
        const int32_t rr = sg.r0 + 32 * wave + n, tok = (int32_t)a.by_g.quot(rr);
        const bool have = rr < n_rows;
        const int32_t hi = have ? base + tok + 1 : 0;
        const int64_t lo64 = a.window ? (int64_t)base + tok + 1 - (int64_t)a.window : 0;
        const int32_t lo = lo64 > 0 ? (int32_t)lo64 : 0;
        const int32_t w0 = sg.r0 + 32 * wave, w1 = min(w0 + 32, n_rows) - 1;
        const bool idle = w0 >= n_rows; // a wave without rows only loads
        const int32_t tok0 = (int32_t)a.by_g.quot(w0), tok1 = idle ? tok0 : (int32_t)a.by_g.quot(w1);
        const int32_t min_hi = base + tok0 + 1, max_hi = idle ? 0 : base + tok1 + 1;
        const int64_t min_lo = a.window ? (int64_t)base + tok0 + 1 - (int64_t)a.window : INT64_MIN,
                      max_lo = a.window ? (int64_t)base + tok1 + 1 - (int64_t)a.window : INT64_MIN;

        constexpr uint64_t ALL = KEYS == 64 ? ~0ull : (1ull << (KEYS & 63)) - 1;
        // where a tile's rows are: lane l has position l's page entry, then its place; bit l of the result: it has a page
        auto entry = [&](int32_t tile) {
            const int32_t p = tile * KEYS + lane;
            return p < kend && lane < KEYS ? paged_entry(a.kv, table, a.b.max_pages, (uint32_t)p) : 0xFFFFFFFFu;
        };
        auto locate = [&](int32_t tile, uint32_t e, uint32_t *units) {
            return (uint64_t)__ballot(paged_units(a.kv, e, (uint32_t)(tile * KEYS + lane), units));
        };
        // a load's rows lie in one page, and near enough for 32 bits
        const bool runs = a.kv.page_size.d % (64 / S::CPR) == 0 && ((uint64_t)a.kv.slot_units << a.kv.unit_shift) < (1u << 27);
        const char *const kpool = a.kv.k + head_off, *const vpool = a.kv.v + head_off;
        // One wave's loads of its rows of a tile, RPI rows each.
        auto load_tile = [&](uint32_t units, uint64_t ok, int buf) __attribute__((always_inline)) {
            constexpr uint32_t RPI = 64 / S::CPR;
            const uint32_t ln = (uint32_t)here(lane) & 63, first = wave * S::LOADS * RPI, row0 = first + ln / S::CPR;
            const uint32_t c0 = (ln % S::CPR) ^ S::swizzle(row0);
            char *kd = kbuf + buf * S::TILE_BYTES + wave * S::LOADS * 1024, *vd = vbuf + (kd - kbuf);
            // the lane's 16 bytes of row row0 + i RPI (whose low bits row0 has none of)
            auto chunk = [&](uint32_t i) { return (c0 ^ S::swizzle(i * RPI)) * 16; };
            if (ok == ALL && runs && hd == D) { // a load's rows are one run of a page: one address for the wave
                const uint32_t lead = (ln / S::CPR) * (a.kv.slot_units << a.kv.unit_shift);
#pragma unroll
                for (uint32_t i = 0; i < S::LOADS; i++) {
                    const uint64_t off = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)units, first + i * RPI) << a.kv.unit_shift;
                    const uint32_t at = lead + chunk(i);
                    __builtin_amdgcn_global_load_lds((const AQ_GLB void *)(kpool + off + at), (AQ_LDS void *)(kd + i * 1024), 16, 0, 0);
                    __builtin_amdgcn_global_load_lds((const AQ_GLB void *)(vpool + off + at), (AQ_LDS void *)(vd + i * 1024), 16, 0, 0);
                }
            } else { // rows without a page are zeros, and dimensions past the head like the queries' there: 0 times an infinity
                     // would be a NaN
#pragma unroll
                for (uint32_t i = 0; i < S::LOADS; i++) {
                    const uint32_t un = (uint32_t)__builtin_amdgcn_ds_bpermute((int)(row0 * 4 + i * RPI * 4), (int)units);
                    const uint64_t off = ((uint64_t)un << a.kv.unit_shift) + chunk(i);
                    const bool has = ((ok >> (row0 + i * RPI)) & 1) && chunk(i) < (uint32_t)hd * 2;
                    const char *kp = has ? kpool + off : (const char *)&zeros, *vp = has ? vpool + off : (const char *)&zeros;
                    __builtin_amdgcn_global_load_lds((const AQ_GLB void *)kp, (AQ_LDS void *)(kd + i * 1024), 16, 0, 0);
                    __builtin_amdgcn_global_load_lds((const AQ_GLB void *)vp, (AQ_LDS void *)(vd + i * 1024), 16, 0, 0);
                }
            }
        };

        // ---- queries
        u4 q[STEPS];
        {
            const char *row = a.q.p + ((int64_t)(sr.first + tok) * a.q.row + (int64_t)((int)sg.kvh * G + (rr - tok * G)) * a.q.head) * 2;
#pragma unroll
            for (int s = 0; s < STEPS; s++) {
                const int at = 16 * s + 8 * h;
                u4 x = u4{0u, 0u, 0u, 0u};
                if (have && at < hd) {
                    if (a.q_wide) {
                        x = *reinterpret_cast<const u4 *>(row + at * 2);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const uint16_t *y = reinterpret_cast<const uint16_t *>(row) + at + 2 * e;
                            x[e] = y[0] | ((uint32_t)y[1] << 16);
                        }
                    }
                }
                q[s] = x;
            }
        }

        f16v o[DB];
#pragma unroll
        for (int db = 0; db < DB; db++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[db][i] = 0.0f;
        float mc = -INFINITY, l = 0.0f; // the maximum times scale_log2; this lane's part of the sum
        bool big = false;               // some row's is past 2^20: products and difference are rounded apart

        int32_t t = (int32_t)(range.lo + sg.t0);
        const int32_t t_end = (int32_t)(range.lo + sg.t1);
        uint32_t units;
        uint64_t ok = locate(t, entry(t), &units);
        __syncthreads(); // the segment before has read its tiles
        load_tile(units, ok, 0);
        uint32_t next = t + 1 < t_end ? entry(t + 1) : 0; // the next tile's page entries, on their way for a tile's time
        int buf = 0;
        for (; t < t_end; t++) {
            const int32_t kb = t * KEYS;
            const char *kt = kbuf + buf * S::TILE_BYTES, *vt = vbuf + buf * S::TILE_BYTES;
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            const uint64_t ok_now = ok;
            if (t + 1 < t_end) {
                ok = locate(t + 1, next, &units);
                load_tile(units, ok, buf ^ 1);
                if (t + 2 < t_end) next = entry(t + 2);
            }
            const bool work = kb < max_hi && (int64_t)kb + KEYS > min_lo; // uniform in the wave
            const bool edge = kb + KEYS > min_hi || (int64_t)kb < max_lo || ok_now != ALL;
            // One tile; CAREFUL: with what only tiles at an edge, with holes or with huge scores need. False: nothing done,
            // the scores are huge.
            auto sum_tile = [&](auto careful) __attribute__((always_inline)) {
                constexpr bool CAREFUL = decltype(careful)::value;
                f16v s[HALVES];
                const int ka = here(kaddr0), va = here(vaddr0);
#pragma unroll
                for (int k = 0; k < HALVES; k++)
#pragma unroll
                    for (int i = 0; i < 16; i++) s[k][i] = 0.0f;
#pragma unroll
                for (int st = 0; st < STEPS; st++)
#pragma unroll
                    for (int k = 0; k < HALVES; k++) {
                        const u4 x = *reinterpret_cast<const u4 *>(kt + (ka ^ (st % 8 * 32)) + 32 * k * S::RB + (st / 8) * 256);
                        s[k] = mfma32<CT>(x, q[st], s[k]);
                        if (D == 256 && st % 8 == 7) __builtin_amdgcn_sched_barrier(0);
                    }
                if (CAREFUL && edge) {
                    const int hr = hi - kb - 4 * h, lr = lo - kb - 4 * h; // of position 0 of this lane's
#pragma unroll
                    for (int k = 0; k < HALVES; k++)
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const int pos = 32 * k + 8 * (i / 4) + i % 4;
                            s[k][i] = pos < hr && pos >= lr ? s[k][i] : -INFINITY;
                        }
                    if (ok_now != ALL) {
                        const uint64_t mine = ok_now >> (4 * here(h));
#pragma unroll
                        for (int k = 0; k < HALVES; k++)
#pragma unroll
                            for (int i = 0; i < 16; i++)
                                s[k][i] = (mine >> (32 * k + 8 * (i / 4) + i % 4)) & 1 ? s[k][i] : -INFINITY;
                    }
                }
                float mt = s[0][0];
#pragma unroll
                for (int i = 1; i < 16 * HALVES; i++) mt = fmaxf(mt, s[i / 16][i % 16]);
                mt = both_max(mt) * a.scale_log2;
                if (!CAREFUL && __any(!(fabsf(mt) < 1048576.0f))) return false;
                if (__any(mt > mc + GROW)) {
                    const float mn = fmaxf(mc, mt), mu = mn == -INFINITY ? 0.0f : mn;
                    const float alpha = fast_exp2(mc - mu);
                    l *= alpha;
#pragma unroll
                    for (int db = 0; db < DB; db++)
#pragma unroll
                        for (int i = 0; i < 16; i++) o[db][i] *= alpha;
                    mc = mn;
                    big = __any(!(fabsf(mc) < 1048576.0f) && mc != -INFINITY);
                }
                const float mu = mc == -INFINITY ? 0.0f : mc;
                if (CAREFUL && big) {
#pragma unroll
                    for (int k = 0; k < HALVES; k++)
#pragma unroll
                        for (int i = 0; i < 16; i++) s[k][i] = fast_exp2((s[k][i] * a.scale_log2 - mu) + P_SHIFT);
                } else {
                    const float off = P_SHIFT - mu;
#pragma unroll
                    for (int k = 0; k < HALVES; k++)
#pragma unroll
                        for (int i = 0; i < 16; i++) s[k][i] = fast_exp2(fmaf(s[k][i], a.scale_log2, off));
                }
                u4 p[2 * HALVES]; // of 16 positions each
#pragma unroll
                for (int kk = 0; kk < 2 * HALVES; kk++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                    {
                        p[kk][e] = pack2<CT>(s[kk / 2][8 * (kk % 2) + 2 * e], s[kk / 2][8 * (kk % 2) + 2 * e + 1]);
                        l = add2<CT>(p[kk][e], l);
                    }

                auto v_operand = [&](int kk, int db) {
                    u4 x;
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const char *at = vt + (va ^ (db % 4 * 64 + e * 32)) + (16 * kk + 8 * e) * S::RB + (db / 4) * 256;
                        const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((AQ_LDS s4 *)at);
                        const u2 z = __builtin_bit_cast(u2, y);
                        x[2 * e] = z[0];
                        x[2 * e + 1] = z[1];
                    }
                    return x;
                };
#pragma unroll
                for (int kk = 0; kk < 2 * HALVES; kk++)
#pragma unroll
                    for (int db = 0; db < DB; db++) {
                        u4 x = v_operand(kk, db);
                        if (CAREFUL) {
#pragma unroll
                            for (int y = 0; y < 4; y++) x[y] &= ~odd_mask<CT>(x[y]);
                        }
                        o[db] = mfma32<CT>(x, p[kk], o[db]);
                        if (CAREFUL || (D == 256 && db % 4 == 3)) __builtin_amdgcn_sched_barrier(0);
                    }
                if (CAREFUL) {
                    // A position that only some rows see must not reach the others as a 0 times an infinity or a NaN: such
                    // values were left out above, and are added here to the rows that see them.
                    unsigned any = 0;
                    const int ln = here(lane);
#pragma unroll 4
                    for (int c = 0; c < S::CPR; c++) {
                        const u4 x = *reinterpret_cast<const u4 *>(vt + (ln % KEYS) * S::RB + ((c + ln) % S::CPR) * 16);
#pragma unroll
                        for (int e = 0; e < 4; e++) any |= odd_bits<CT>(x[e]);
                    }
#pragma unroll 1
                    for (uint64_t rest = __ballot(any & 0x80008000u) & ALL; rest; rest &= rest - 1) {
                        const int pos = __builtin_ctzll(rest);
                        unsigned w = 0; // the word of p that has the position's, in the lanes of its half
#pragma unroll
                        for (int kk = 0; kk < 2 * HALVES; kk++)
#pragma unroll
                            for (int e = 0; e < 4; e++) w = pos / 16 * 4 + pos / 8 % 2 * 2 + pos % 4 / 2 == 4 * kk + e ? p[kk][e] : w;
                        w = (unsigned)__shfl((int)w, here(n) + 32 * (pos / 4 % 2));
                        using T = typename RowType<CT>::type;
                        const float pv = (float)__builtin_bit_cast(T, (uint16_t)(pos & 1 ? w >> 16 : w));
                        const bool sees = kb + pos < hi && kb + pos >= lo;
                        const char *row = vt + pos * S::RB + here(8 * h);
#pragma unroll
                        for (int db = 0; db < DB; db++)
#pragma unroll
                            for (int i = 0; i < 4; i++) { // dimensions 32 db + 8 i + 4 h ..
                                const u2 v = *reinterpret_cast<const u2 *>(row + ((4 * db + i) ^ (int)S::swizzle(pos)) * 16);
#pragma unroll
                                for (int e = 0; e < 4; e++) {
                                    const uint16_t x = (uint16_t)(e & 1 ? v[e / 2] >> 16 : v[e / 2]);
                                    if (sees && (odd_bits<CT>(x) & 0x8000u)) o[db][4 * i + e] += pv * (float)__builtin_bit_cast(T, x);
                                }
                            }
                    }
                }
                return true;
            };
            if (work && (edge || big || !sum_tile(std::false_type{}))) sum_tile(std::true_type{});
            buf ^= 1;
        }

        // ---- out: the whole segment's rows, or this share's part, through the LDS so that neighbouring lanes have
        // neighbouring values; each wave its own 32 rows, 64 dimensions a pass
        {
            const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
            l = __uint_as_float(r[0]) + __uint_as_float(r[1]);
        }
        const bool cut = is_cut(sg);
        const uint32_t slot = part_slot(sg, sh);
        const int ln = here(lane);
        if (cut && have && h == 0) {
            float *ml = a.part_ml + ((size_t)slot * R + 32 * wave + n) * 2;
            ml[0] = mc;
            ml[1] = l;
        }
        const float inv = cut ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
        constexpr int OROW = S::OROW;
        float *mine = reinterpret_cast<float *>(smem) + wave * 32 * OROW;
        __syncthreads(); // every wave is past its tiles
#pragma unroll
        for (int pass = 0; pass < D / 64; pass++) {
            asm volatile("" ::: "memory");
#pragma unroll
            for (int i = 0; i < 8; i++) { // dimensions 8 i + 4 h .. of the pass
                f4 x;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float y = o[2 * pass + i / 4][4 * (i % 4) + e];
                    x[e] = inv == 0.0f ? 0.0f : y * inv;
                }
                *reinterpret_cast<f4 *>(mine + (ln & 31) * OROW + 8 * i + 4 * (ln >> 5)) = x;
            }
            asm volatile("" ::: "memory");
            if (cut) { // 16 lanes a row
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int row = 4 * i + (ln >> 4), dim = 64 * pass + 4 * (ln & 15);
                    const f4 x = *reinterpret_cast<const f4 *>(mine + row * OROW + 4 * (ln & 15));
                    if (w0 + row < n_rows && dim < hd)
                        *reinterpret_cast<f4 *>(a.part_o + ((size_t)slot * R + 32 * wave + row) * D + dim) = x;
                }
            } else { // 8 lanes a row
                store_rows<CT>(a, sr, (int)sg.kvh, w0, n_rows, 64 * pass + 8 * (ln & 7), ln >> 3, mine + 8 * (ln & 7), OROW);
            }
        }
    }
}

template <int CT, int D>
int chunk_launch(const AttnPagedArgs &a, hipStream_t stream) {
    using S = ChunkShape<D>;
    static std::atomic<uint64_t> raised{0}; // bit d: done on device d
    int dev = 0;
    AQ_HIP(hipGetDevice(&dev));
    if (!(raised.load() & (1ull << (dev & 63)))) {
        AQ_HIP(hipFuncSetAttribute((const void *)chunk_kernel<CT, D>, hipFuncAttributeMaxDynamicSharedMemorySize, S::LDS));
        raised.fetch_or(1ull << (dev & 63));
    }
    chunk_kernel<CT, D><<<a.shares, 256, S::LDS, stream>>>(a);
    AQ_HIP(hipGetLastError());
    return 0;
}

} // namespace

int launch_paged_chunk(const AttnPagedArgs &a, int D, hipStream_t stream) {
    if (a.kv.type == AQ_TYPE_F16) {
        if (D == 64) return chunk_launch<AQ_TYPE_F16, 64>(a, stream);
        if (D == 128) return chunk_launch<AQ_TYPE_F16, 128>(a, stream);
        return chunk_launch<AQ_TYPE_F16, 256>(a, stream);
    }
    if (D == 64) return chunk_launch<AQ_TYPE_BF16, 64>(a, stream);
    if (D == 128) return chunk_launch<AQ_TYPE_BF16, 128>(a, stream);
    return chunk_launch<AQ_TYPE_BF16, 256>(a, stream);
}

} // namespace aq
