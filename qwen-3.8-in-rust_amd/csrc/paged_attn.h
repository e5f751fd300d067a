// paged_attn.h — what the two paged attention kernels (paged_few.h: few rows, pages streamed through registers;
// paged_chunk.hip: many rows, tiles in the LDS) share: the division of the work, the partial results, the outputs.
//
// Rows. The G = n_head / n_head_kv query heads that share a K/V head, times a sequence's new tokens, are its rows over
// that head's keys: row = token * G + head in the group. A segment is one row tile (R rows) of one sequence on one K/V
// head; its keys are counted in units of TK positions from position 0, and only the units that some row of the tile
// sees are work.
//
// Split. All segments' units in order (sequence, K/V head, row tile, key unit: row tiles that read the same keys side by
// side, on one XCD at one time), each segment's with `lead` places before them for what a segment costs besides its units,
// form one line of `total` places, cut into work-group shares of `chunk` places each, however long or short the sequences
// are (short contexts: every segment has `whole` places and is a share). A share that holds a whole segment writes its
// output; where a segment is cut, each share writes its part (row maxima, sums and unnormalised outputs, in f32) to the
// workspace, slot 2w for the segment that began before share w, slot 2w + 1 for the one that goes on after it, and a second
// launch joins the parts in order. Which share has which part follows from the lengths alone, so the same call gives the
// same bits.
#pragma once

#include "paged.h"

namespace aq {

// A row tile: its sequence, its index there, and the prefix sums where the sequence's row tiles begin and end.
struct RowTile {
    uint32_t seq, rt, p0, p1;
};

struct AttnPagedArgs {
    PagedKv kv;
    PagedBatch b;
    HeadsView q, out, gate;  // gate.p null: none
    int n_head, G;
    FastDiv by_g; // rows to tokens
    uint32_t window; // 0: all
    uint32_t cap;    // positions from here on are not attended: the table's reach, or max_len
    float scale_log2;          // scale * log2(e)
    uint32_t q_wide, out_wide; // 16-byte loads of q; 4-value stores of out and loads of gate
    uint32_t shares, min_chunk, lead; // work-groups; least places of a share; places before a segment's units
    uint32_t whole;   // places of every segment, where each share is one whole segment; 0: as many as it has units, and cut
    uint32_t n_seg;   // row tiles of all sequences at most
    uint32_t planned; // 1: a plan launch has filled plan and tiles; 0: the work-groups divide by themselves
    // workspace
    uint32_t *plan;    // [0] total places (of all K/V heads), [1] chunk, [2] row tiles; then prefix sums of their places
    RowTile *tiles;    // of each row tile
    float *part_o;  // [2 * shares][R][D]
    float *part_ml; // [2 * shares][R][2]
};
constexpr uint32_t PLAN_HEAD = 4;

// The units of a row tile: rows r0 .. r0 + R - 1 of a sequence of `sr.n` rows; first unit and one past the last. A tile
// whose rows see nothing has one unit all the same: the one that writes its zeros.
struct UnitRange {
    uint32_t lo, hi;
};
__device__ __forceinline__ UnitRange tile_units(const AttnPagedArgs &a, const SeqRows &sr, int32_t r0, int32_t R, uint32_t tk) {
    const int32_t last = min(r0 + R, sr.n * a.G) - 1;
    const int32_t t0 = (int32_t)a.by_g.quot(r0), t1 = (int32_t)a.by_g.quot(last), base = sr.base; // row tokens' positions are base + token
    const int32_t end = min(max(base + t1 + 1, 0), (int32_t)a.cap);
    const int64_t begin = a.window ? max((int64_t)base + t0 + 1 - (int64_t)a.window, (int64_t)0) : 0;
    UnitRange u;
    u.lo = (uint32_t)begin / tk;
    u.hi = ((uint32_t)end + tk - 1) / tk;
    if (u.hi <= u.lo) u.hi = u.lo + 1;
    return u;
}

// Units per share: at least min_chunk, and so many that no more than `shares` shares are needed.
__device__ __forceinline__ uint32_t share_chunk(uint32_t total, uint32_t shares, uint32_t min_chunk) {
    return max((total + shares - 1) / shares, min_chunk);
}

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// x, of which the compiler knows nothing more: what is computed from it stays where it is used, instead of waiting in a
// register from before a loop.
__device__ __forceinline__ int here(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// x, which all lanes have: in a scalar register.
__device__ __forceinline__ uint32_t same(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }

constexpr int INLINE_TILES = 1024; // sequences, and row tiles, that a work-group of 256 divides by itself

// The plan in a work-group's LDS: of each row tile its sequence, of each sequence its first row tile, and the prefix sums
// of the row tiles' places.
struct PlanLds {
    uint32_t pre[INLINE_TILES + 1], first[INLINE_TILES + 1], seq[INLINE_TILES], wsum[4], found;
};

// A work-group's share of the line: its number, its places begin .. end - 1 (none: begin == end); the row tile and K/V head
// that begin lies in.
struct Share {
    uint32_t w, begin, end, j, kvh, n_seg;
};

// Row tile j of the plan, wherever that is.
__device__ __forceinline__ RowTile row_tile(const AttnPagedArgs &a, const PlanLds &lds, uint32_t n_seg, uint32_t j) {
    if (a.planned) return a.tiles[j];
    RowTile t;
    t.seq = lds.seq[j];
    const uint32_t j0 = lds.first[t.seq], j1 = t.seq + 1 < a.b.n_seq ? min(lds.first[t.seq + 1], n_seg) : n_seg;
    t.rt = j - j0;
    t.p0 = lds.pre[j0];
    t.p1 = lds.pre[j1];
    return t;
}
// The first place of row tile j on a K/V head (pre: its prefix sum).
__device__ __forceinline__ uint32_t tile_place(const RowTile &t, uint32_t pre, uint32_t nkv, uint32_t kvh) {
    return t.p0 * nkv + kvh * (t.p1 - t.p0) + (pre - t.p0);
}
// Whether place x lies in row tile j (its prefix sums pre .. end), and on which K/V head.
__device__ __forceinline__ bool tile_holds(const RowTile &t, uint32_t pre, uint32_t end, uint32_t nkv, uint32_t x, uint32_t *kvh) {
    if (x < t.p0 * nkv || x >= t.p1 * nkv) return false;
    const uint32_t rel = x - t.p0 * nkv, size = t.p1 - t.p0;
    *kvh = rel / size;
    const uint32_t at = rel - *kvh * size + t.p0;
    return pre <= at && at < end;
}

// Inclusive prefix sums over a wave, and over a work-group of 256 (wsum: 4 words; two barriers).
__device__ __forceinline__ uint32_t wave_scan(uint32_t v, int lanes = 64) { // the first `lanes` lanes'
    const int lane = threadIdx.x & 63;
    for (int d = 1; d < lanes; d *= 2) {
        const uint32_t x = __shfl_up(v, d);
        if (lane >= d) v += x;
    }
    return v;
}
__device__ __forceinline__ uint32_t group_scan(uint32_t v, uint32_t *wsum) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v = wave_scan(v);
    __syncthreads(); // the last call's sums are read
    if (lane == 63) wsum[wave] = v;
    __syncthreads();
    for (int w = 0; w < wave; w++) v += wsum[w];
    return v;
}

__device__ __forceinline__ uint32_t seq_tiles(const AttnPagedArgs &a, uint32_t s, int R) {
    return s < a.b.n_seq ? (uint32_t)((paged_seq(a.b, s).n * a.G + R - 1) / R) : 0u;
}
__device__ __forceinline__ uint32_t tile_count(const AttnPagedArgs &a, uint32_t s, uint32_t rt, int R, uint32_t tk) {
    if (a.whole) return a.whole;
    const UnitRange u = tile_units(a, paged_seq(a.b, s), (int32_t)rt * R, R, tk);
    return u.hi - u.lo + a.lead;
}

__device__ __forceinline__ Share take_share(const AttnPagedArgs &a, int R, uint32_t tk, PlanLds &lds) {
    const int tid = threadIdx.x, lane = tid & 63;
    const uint32_t nkv = (uint32_t)a.kv.nkv;
    Share sh;
    // neighbouring shares on one XCD: work-groups go round the 8 XCDs, and neighbours read the same pages' lines
    sh.w = a.shares % 8 ? blockIdx.x : (blockIdx.x % 8) * (a.shares / 8) + blockIdx.x / 8;
    sh.begin = sh.end = sh.j = sh.kvh = 0;
    uint32_t total, chunk, n_seg;
    bool one_wave = false;
    if (a.planned) {
        total = a.plan[0];
        chunk = a.plan[1];
        n_seg = a.plan[2];
    } else {
        // Few: every wave for itself, without a barrier (all write the same words).
        uint32_t cnt = 0, incl = 0;
        if (a.b.n_seq <= 64) {
            cnt = min(seq_tiles(a, lane, R), 65u);
            incl = wave_scan(cnt, (int)a.b.n_seq);
            n_seg = __builtin_amdgcn_readlane(incl, a.b.n_seq - 1);
            one_wave = n_seg <= min(64u, a.n_seg);
        }
        if (one_wave) {
            lds.first[lane] = incl - cnt;
            for (uint32_t i = 0; i < cnt; i++) lds.seq[incl - cnt + i] = lane;
            __builtin_amdgcn_wave_barrier();
            uint32_t units = 0;
            if ((uint32_t)lane < n_seg) {
                const uint32_t s = lds.seq[lane];
                units = tile_count(a, s, lane - lds.first[s], R, tk);
            }
            const uint32_t sum = wave_scan(units, (int)n_seg);
            if (lane == 0) lds.pre[0] = 0;
            lds.pre[lane + 1] = sum;
            total = n_seg ? (uint32_t)__builtin_amdgcn_readlane(sum, n_seg - 1) * nkv : 0u;
            __builtin_amdgcn_wave_barrier();
        } else {
            constexpr int PER = INLINE_TILES / 256;
            uint32_t mine[PER], sum = 0;
#pragma unroll
            for (int i = 0; i < PER; i++) sum += mine[i] = min(seq_tiles(a, tid * PER + i, R), (uint32_t)INLINE_TILES);
            uint32_t at = group_scan(sum, lds.wsum) - sum;
#pragma unroll
            for (int i = 0; i < PER; i++) {
                lds.first[tid * PER + i] = at;
                for (uint32_t k = 0; k < mine[i] && at + k < (uint32_t)INLINE_TILES; k++) lds.seq[at + k] = tid * PER + i;
                at += mine[i];
            }
            if (tid == 255) lds.first[INLINE_TILES] = at;
            __syncthreads();
            n_seg = min(min(lds.first[INLINE_TILES], (uint32_t)INLINE_TILES), a.n_seg);
            sum = 0;
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const uint32_t j = tid * PER + i;
                mine[i] = 0;
                if (j < n_seg) mine[i] = tile_count(a, lds.seq[j], j - lds.first[lds.seq[j]], R, tk);
                sum += mine[i];
            }
            at = group_scan(sum, lds.wsum) - sum;
            if (tid == 0) lds.pre[0] = 0;
#pragma unroll
            for (int i = 0; i < PER; i++) {
                at += mine[i];
                lds.pre[tid * PER + i + 1] = at;
            }
            __syncthreads();
            n_seg = same(n_seg);
            total = same(lds.pre[n_seg]) * nkv;
        }
        chunk = a.whole ? a.whole : share_chunk(total, a.shares, a.min_chunk);
        if (blockIdx.x == 0) { // for the join
            if (tid == 0) {
                a.plan[0] = total;
                a.plan[1] = chunk;
                a.plan[2] = n_seg;
                a.plan[PLAN_HEAD] = 0;
            }
            for (uint32_t j = tid; j < n_seg; j += 256) {
                a.plan[PLAN_HEAD + j + 1] = lds.pre[j + 1];
                a.tiles[j] = row_tile(a, lds, n_seg, j);
            }
        }
    }
    const uint64_t first = (uint64_t)sh.w * chunk;
    if (first >= total) return sh;
    sh.begin = (uint32_t)first;
    sh.end = min(total, sh.begin + chunk);
    // the row tile that the share begins in
    uint32_t kvh = 0;
    if (one_wave) {
        if (n_seg > 1) {
            const bool in = (uint32_t)lane < n_seg && tile_holds(row_tile(a, lds, n_seg, lane), lds.pre[lane],
                                                                 lds.pre[lane + 1], nkv, sh.begin, &kvh);
            sh.j = (uint32_t)__builtin_ctzll(__ballot(in));
        }
    } else {
        for (uint32_t j = tid; j < n_seg; j += 256) {
            const uint32_t p = a.planned ? a.plan[PLAN_HEAD + j] : lds.pre[j];
            const uint32_t e = a.planned ? a.plan[PLAN_HEAD + j + 1] : lds.pre[j + 1];
            if (tile_holds(row_tile(a, lds, n_seg, j), p, e, nkv, sh.begin, &kvh)) lds.found = j;
        }
        __syncthreads();
        sh.j = same(lds.found);
    }
    const RowTile t = row_tile(a, lds, n_seg, sh.j);
    sh.kvh = (sh.begin - same(t.p0) * nkv) / (same(t.p1) - same(t.p0));
    sh.n_seg = n_seg;
    return sh;
}

// The next segment of a share, from place u on (row tile j on K/V head kvh, or the one after it): the sequence, its first
// row, the units t0 .. t1 - 1 of the segment's cnt that are the share's (none: t1 <= t0). Advances u, j and kvh. All uniform.
// tk: the unit, 0 where a share is never a whole segment by itself.
struct Segment {
    uint32_t kvh, seq, cnt;
    int32_t t0, t1, r0;
};
__device__ __forceinline__ Segment next_segment(const AttnPagedArgs &a, int R, uint32_t tk, const PlanLds &lds, const Share &sh,
                                                uint32_t &u, uint32_t &j, uint32_t &kvh) {
    const uint32_t nkv = (uint32_t)a.kv.nkv;
    auto line = [&](uint32_t i) { return same(a.planned ? a.plan[PLAN_HEAD + i] : lds.pre[i]); };
    RowTile t = row_tile(a, lds, sh.n_seg, j);
    t.p0 = same(t.p0);
    t.p1 = same(t.p1);
    t.rt = same(t.rt);
    uint32_t p = line(j), e = line(j + 1);
    if (u >= tile_place(t, p, nkv, kvh) + (e - p)) { // past it: the sequence's next row tile, next head, or the next sequence
        if (e < t.p1) {
            j++;
            t.rt++;
        } else if (kvh + 1 < nkv) {
            kvh++;
            j -= t.rt;
            t.rt = 0;
        } else {
            kvh = 0;
            j++;
            t = row_tile(a, lds, sh.n_seg, j);
            t.p0 = same(t.p0);
            t.p1 = same(t.p1);
            t.rt = 0;
        }
        p = line(j);
        e = line(j + 1);
    }
    Segment s;
    s.kvh = kvh;
    const uint32_t places = e - p, from = u - tile_place(t, p, nkv, kvh), to = min(places, from + (sh.end - u));
    s.cnt = places - a.lead;
    s.t0 = max((int32_t)(from - a.lead), 0);
    s.t1 = (int32_t)(to - a.lead);
    u += to - from;
    s.seq = same(t.seq);
    s.r0 = (int32_t)t.rt * R;
    if (tk && a.whole) {
        const UnitRange range = tile_units(a, paged_seq(a.b, s.seq), s.r0, R, tk);
        s.t0 = 0;
        s.t1 = (int32_t)(s.cnt = range.hi - range.lo);
    }
    return s;
}
// Whether other shares have units of it too, and then the slot of this share's part.
__device__ __forceinline__ bool is_cut(const Segment &s) { return s.t1 - s.t0 < (int32_t)s.cnt; }
__device__ __forceinline__ uint32_t part_slot(const Segment &s, const Share &sh) { return 2 * sh.w + (s.t0 == 0 ? 1 : 0); }

// N consecutive values of a row as f32, of which `have` exist (the others 0).
template <int QT, int N>
__device__ __forceinline__ void load_row(const char *row, int at, int have, bool wide, float *v) {
    using E = typename RowType<QT>::type;
    if (at >= have) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = 0.0f;
    } else if (wide) {
        constexpr int C = 16 / (int)sizeof(E) < N ? 16 / (int)sizeof(E) : N;
        typedef E vec __attribute__((ext_vector_type(C)));
#pragma unroll
        for (int i = 0; i < N / C; i++) {
            const vec x = *reinterpret_cast<const vec *>(row + (size_t)(at + i * C) * sizeof(E));
#pragma unroll
            for (int j = 0; j < C; j++) v[i * C + j] = (float)x[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = (float)reinterpret_cast<const E *>(row)[at + i];
    }
}

// Four outputs of a row: times the gate, rounded, stored.
template <int QT>
__device__ __forceinline__ void store_out(const AttnPagedArgs &a, int64_t row, int head, int dim, float *v) {
    using E = typename RowType<QT>::type;
    if (a.gate.p) {
        const char *gp = a.gate.p + (row * a.gate.row + (int64_t)head * a.gate.head + dim) * (int64_t)sizeof(E);
        float g[4];
        load_row<QT, 4>(gp, 0, 4, a.out_wide, g);
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] *= 1.0f / (1.0f + expf(-g[i]));
    }
    E *o = (E *)a.out.p + row * a.out.row + (int64_t)head * a.out.head + dim;
    typedef E vec __attribute__((ext_vector_type(4)));
    if (a.out_wide) {
        vec x;
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = (E)v[i];
        *reinterpret_cast<vec *>(o) = x;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = (E)v[i];
    }
}

// Bits 15 and 31 of the result: the low and high 16-bit value of w is an infinity or a NaN (its exponent plus one carries).
template <int CT>
__device__ __forceinline__ unsigned odd_bits(unsigned w) {
    return (w & 0x7FFF7FFFu) + (CT == AQ_TYPE_F16 ? 0x04000400u : 0x00800080u);
}
// All bits of such a value, none of others.
template <int CT>
__device__ __forceinline__ unsigned odd_mask(unsigned w) {
    return ((odd_bits<CT>(w) & 0x80008000u) >> 15) * 0xFFFFu;
}

// l plus the two values of a packed word, in 32 bits.
template <int CT>
__device__ __forceinline__ float add2(unsigned w, float l) {
    if constexpr (CT == AQ_TYPE_F16) {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, w), h2{1, 1}, l, false);
    } else {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, w), b2{(__bf16)1.0f, (__bf16)1.0f}, l, false);
    }
}

// Workspace layout, the same in the size query and in the launch.
struct PagedSpace {
    size_t plan = 0, seg = 0, o = 0, ml = 0, bytes = 0;
};
inline PagedSpace paged_space(size_t shares, size_t n_seg, size_t R, size_t D) {
    PagedSpace s;
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    s.seg = up((PLAN_HEAD + n_seg + 1) * 4);
    s.o = s.seg + up(n_seg * sizeof(RowTile));
    s.ml = s.o + up(2 * shares * R * D * 4);
    s.bytes = s.ml + up(2 * shares * R * 2 * 4);
    return s;
}

int launch_paged_plan(const AttnPagedArgs &a, int R, uint32_t tk, hipStream_t stream);
// The few-row kernel (paged_few.h): a cache of this type, rows of its type or f32; D the padded head size, R 16 or 32 rows.
int launch_paged_few_f32(const AttnPagedArgs &a, int D, int R, hipStream_t stream);
int launch_paged_few_f16(const AttnPagedArgs &a, int D, int R, hipStream_t stream);
int launch_paged_few_bf16(const AttnPagedArgs &a, int D, int R, hipStream_t stream);
int launch_paged_chunk(const AttnPagedArgs &a, int D, hipStream_t stream); // 16-bit rows and cache
int launch_paged_combine(const AttnPagedArgs &a, int R, int D, int rows, hipStream_t stream);

constexpr int WAVES = 4;

// Positions that a wave of the few-row kernel takes at once: 32, and 16 of a wide head, whose rows fill the registers.
constexpr int few_tile(int D) { return D == 256 ? 16 : 32; }
// The rows (16 or 32) lie on a wave's NR accumulator tiles; 32 rows of a wide head would not fit its registers, so there two
// waves take 16 rows each over the same positions (RG = 2: the second reads them from the cache the first filled).
constexpr int few_groups(int CT, int D, int R) { return R == 32 && (D == 256 || (CT == AQ_TYPE_F32 && D == 128)) ? 2 : 1; }
constexpr int few_unit(int CT, int D, int R) { return WAVES / few_groups(CT, D, R) * few_tile(D); }

constexpr int CHUNK_ROWS = 128;                                   // paged_chunk.hip's row tile
constexpr int chunk_keys(int D) { return D == 256 ? 32 : 64; } // and its unit

} // namespace aq
