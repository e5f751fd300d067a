// paged_attn.h — what the paged attention kernels (paged_attention.hip) share: the division of the work, the partial
// results, their argument block.
//
// Rows. The G = n_head / n_head_kv query heads that share a K/V head, times a sequence's new tokens, are its rows over
// that head's keys: row = token * G + head in the group. A segment is one row tile (R rows) of one sequence on one K/V
// head; its keys are counted in units of TK positions from position 0, and only the units that some row of the tile
// sees are work.
//
// Split. All segments' units in order (sequence, row tile, K/V head, key unit) form one line of `total` units, cut into
// work-group shares of `chunk` units each, however long or short the sequences are. A share that holds a whole segment
// writes its output; where a segment is cut, each share writes its part (row maxima, sums and unnormalised outputs, in
// f32) to the workspace, slot 2w for the segment that began before share w, slot 2w + 1 for the one that goes on after
// it, and a second launch joins the parts in order. Which share has which part follows from the lengths alone, so the
// same call gives the same bits.
#pragma once

#include "paged.h"

namespace aq {

struct AttnPagedArgs {
    PagedKv kv;
    PagedBatch b;
    HeadsView q, out, gate;  // gate.p null: none
    int n_head, G;
    uint32_t window; // 0: all
    uint32_t cap;    // positions from here on are not attended: the table's reach, or max_len
    float scale_log2;          // scale * log2(e)
    uint32_t q_wide, out_wide; // 16-byte loads of q; 4-value stores of out and loads of gate
    uint32_t shares, min_chunk; // work-groups; least units of a share
    uint32_t n_seg;   // row tiles of all sequences at most (one per sequence where planned is 0)
    uint32_t planned; // 1: a plan launch has filled plan, seg_seq, seg_rt; 0: one row tile per sequence
    // workspace
    uint32_t *plan;    // [0] total units (of all K/V heads), [1] chunk, [2] row tiles; then prefix sums of their units
    uint32_t *seg_seq; // of each row tile: its sequence and its index there (kernels with a plan launch)
    uint32_t *seg_rt;
    float *part_o;  // [2 * shares][R][D]
    float *part_ml; // [2 * shares][R][2]
};
constexpr uint32_t PLAN_HEAD = 4;

// The units of a row tile: rows r0 .. r0 + R - 1 of a sequence of `sr.n` rows; first unit and one past the last. A tile
// whose rows see nothing has one unit all the same: the one that writes its zeros.
struct UnitRange {
    uint32_t lo, hi;
};
__device__ __forceinline__ UnitRange tile_units(const SeqRows &sr, int G, uint32_t window, uint32_t cap, int32_t r0,
                                                int32_t R, uint32_t tk) {
    const int32_t last = min(r0 + R, sr.n * G) - 1;
    const int32_t t0 = r0 / G, t1 = last / G, base = sr.len - sr.n; // row tokens' positions are base + token
    const int32_t end = min(max(base + t1 + 1, 0), (int32_t)cap);
    const int64_t begin = window ? max((int64_t)base + t0 + 1 - (int64_t)window, (int64_t)0) : 0;
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

// Workspace layout, the same in the size query and in the launch.
struct PagedSpace {
    size_t plan = 0, seg = 0, o = 0, ml = 0, bytes = 0;
};
inline PagedSpace paged_space(size_t shares, size_t n_seg, size_t R, size_t D) {
    PagedSpace s;
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    s.seg = up((PLAN_HEAD + n_seg + 1) * 4);
    s.o = s.seg + up(n_seg * 8);
    s.ml = s.o + up(2 * shares * R * D * 4);
    s.bytes = s.ml + up(2 * shares * R * 2 * 4);
    return s;
}

int launch_paged_plan(const AttnPagedArgs &a, int R, uint32_t tk, hipStream_t stream);
int launch_paged_combine(const AttnPagedArgs &a, int R, int D, hipStream_t stream);

} // namespace aq
