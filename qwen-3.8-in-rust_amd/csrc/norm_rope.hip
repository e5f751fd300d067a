// norm_rope.hip — the norms of queries and keys head by head with their rotation in the same pass, over rows of heads
// (aq_qk_norm_rope) and on the way into the pages (aq_paged_append_norm).
//
// y = x / sqrt(mean(x^2) + eps) * weight over the head's values, in 32 bits, then its pairs turned as rope.hip turns them, and
// one rounding at the store. A head's values lie on a group of lanes, one unit each, so that both values of a pair are in one
// lane and the sum of squares is one exchange per doubling of the group. A wave has as many heads of one row as fit it,
// computes the row's angles once, one a lane, and hands them over in the LDS: no work-group to wait for, and the values are
// on their way meanwhile.
//
// Bound by their bytes, with about as many cycles of arithmetic: 8191 rows of 40 heads of 128 (bf16) 33.6 us, 5.0 TB/s, what a
// large copy reaches; with the angles over a work-group behind a barrier 42.2, with work-groups that go on from row to row
// 46.6 (too few waves); with a branch for every lane that has no unit or no pair 36.0. 5342 rows of 24 query and 4 K/V heads
// of 256 (f32 into f16) appended in 61.9 us, 5.3 TB/s. Single tokens: an empty launch and three latencies.
#include <cmath>

#include "rope.h"

namespace aq {
namespace {

constexpr int MAX_HEAD = 256;
// Heads of a lane, so that it has 32 bytes to load. One and two heads: 8191 rows of 40 heads of 128 (bf16), 32 bytes of each
// (half layout) 33.6 and 39.8 us, 16 (neighbours) 38.0 and 35.3; 5342 rows of 32 heads of 256 (f32 into f16), 32 bytes,
// 61.9 and 66.5.
constexpr uint32_t heads_per_lane(uint32_t bytes) { return bytes < 32 ? 2 : 1; }

struct NormArgs {
    PagedKv kv;
    PagedBatch b;
    HeadsView q, qo, k, ko, v;
    const float *qw, *kw;
    const double *freq;
    const int32_t *pos; // of each row; null: its place in its sequence
    uint32_t n_rows, dim, rot_units, pass_units, pass_seconds, units, lane_shift;
    uint32_t nq, nqk, jobs; // heads of a row: queries, keys after them, values after those
    uint32_t parts;         // waves of a row
    FastDiv by_parts;
    float eps, inv_hd, gain;
};

// A unit's N values as they are stored.
template <int T, int N>
struct Raw {
    using E = typename RowType<T>::type;
    typedef E vec __attribute__((ext_vector_type(N)));
    vec x;
};
// V values at p: into x[at ..], and back from v, at most 16 bytes at a time where W.
template <int V, bool W, typename E, typename VEC>
__device__ __forceinline__ void load_raw(const E *p, VEC &x, int at) {
    constexpr int C = !W ? 1 : V * (int)sizeof(E) > 16 ? 16 / (int)sizeof(E) : V;
    typedef E vec __attribute__((ext_vector_type(C)));
#pragma unroll
    for (int i = 0; i < V / C; i++) {
        const vec y = *reinterpret_cast<const vec *>(p + i * C);
#pragma unroll
        for (int e = 0; e < C; e++) x[at + i * C + e] = y[e];
    }
}
template <int V, bool W, typename E>
__device__ __forceinline__ void store_raw(E *p, const float *v) {
    constexpr int C = !W ? 1 : V * (int)sizeof(E) > 16 ? 16 / (int)sizeof(E) : V;
    typedef E vec __attribute__((ext_vector_type(C)));
#pragma unroll
    for (int i = 0; i < V / C; i++) {
        vec y;
#pragma unroll
        for (int e = 0; e < C; e++) y[e] = (E)v[i * C + e];
        *reinterpret_cast<vec *>(p + i * C) = y;
    }
}

// One wave has one row's heads `part * HB * heads a wave` and on, of `parts` waves a row; a head lies on 2^lane_shift lanes,
// and a wave takes HB times as many heads as fit it. NU: units a lane has at most (one where 16 bytes are moved at a time).
// A unit: VEC values of either half of what is turned (half layout), of either half of what passes through, or VEC neighbours.
// Little of it branches: a lane past the head's units has the first one's once more, a unit without second values its first
// ones twice, a head past the last is the last one again (its values, its weight), and only the stores are left out.
template <int TI, int TO, bool INTER, int VEC, bool W, int NU, bool PAGED>
__global__ void __launch_bounds__(256, 8) norm_kernel(NormArgs a) {
    using EI = typename RowType<TI>::type;
    using EO = typename RowType<TO>::type;
    constexpr int N = INTER ? VEC : 2 * VEC, PAIRS = N / 2;
    constexpr uint32_t HB = heads_per_lane(N * sizeof(EI));
    __shared__ __align__(16) float turns[4][2][MAX_HEAD / 2]; // each wave's cosines and sines
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lanes = 1u << a.lane_shift;
    const uint32_t id = (uint32_t)__builtin_amdgcn_readfirstlane((int)((blockIdx.y * gridDim.x + blockIdx.x) * 4 + wave));
    const uint32_t row = a.by_parts.quot(id), part = id - row * a.parts;
    if (row >= a.n_rows) return;

    // Where each of this lane's units begins, its second values and its angles; whether it has them, and turns them.
    uint32_t at[NU], two[NU], pair[NU];
    bool have[NU], both[NU], rot[NU];
#pragma unroll
    for (int i = 0; i < NU; i++) {
        const uint32_t u = (lane & (lanes - 1)) + ((uint32_t)i << a.lane_shift);
        have[i] = u < a.units;
        rot[i] = u < a.rot_units;
        at[i] = rot[i] ? u * VEC : have[i] ? a.dim + (u - a.rot_units) * VEC : 0;
        both[i] = !INTER && (rot[i] || (have[i] && u - a.rot_units < a.pass_seconds));
        two[i] = at[i] + (both[i] ? (rot[i] ? a.dim / 2 : a.pass_units * VEC) : 0);
        pair[i] = rot[i] ? (INTER ? at[i] / 2 : at[i]) : 0;
    }
    // A job: one head of the row's queries, keys or values. What is not there has null pointers, so a job past the last is
    // the last one again wherever it chooses between them.
    const uint32_t per = 64u >> a.lane_shift, j0 = part * HB * per + (lane >> a.lane_shift);
    auto job = [&](int h) { return min(j0 + h * per, a.jobs - 1); };
    Raw<TI, N> raw[HB][NU];
#pragma unroll
    for (int h = 0; h < (int)HB; h++) {
        const uint32_t j = job(h);
        const bool q = j < a.nq, k = j < a.nqk;
        const EI *p = (const EI *)(q ? a.q.p : k ? a.k.p : a.v.p) + row * (q ? a.q.row : k ? a.k.row : a.v.row) +
                      (int64_t)(j - (q ? 0 : k ? a.nq : a.nqk)) * (q ? a.q.head : k ? a.k.head : a.v.head);
#pragma unroll
        for (int i = 0; i < NU; i++) {
            load_raw<VEC, W>(p + at[i], raw[h][i].x, 0);
            if (!INTER) load_raw<VEC, W>(p + two[i], raw[h][i].x, N - VEC);
        }
    }

    // Where the row is rotated and stored; a row of no sequence is left alone.
    int32_t pos = 0;
    bool store = true;
    uint32_t off = 0;
    if constexpr (PAGED) {
        const uint32_t seq = paged_seq_of(a.b, row);
        if (seq >= a.b.n_seq) return; // uniform in the wave, as all of this
        const SeqRows sr = paged_seq(a.b, seq);
        if ((int32_t)row < sr.first) return; // before the first sequence's rows
        pos = sr.base + ((int32_t)row - sr.first);
        store = pos >= 0 && paged_slot(a.kv, a.b.pages + (size_t)seq * a.b.max_pages, a.b.max_pages, (uint32_t)pos, &off);
    }
    if (a.pos) pos = a.pos[row];
    float *const cosines = turns[wave][0], *const sines = turns[wave][1];
    for (uint32_t i = lane; i < a.dim / 2; i += 64) {
        float sn, cs;
        rope_angle(a.freq[i], pos, &sn, &cs);
        cosines[i] = cs * a.gain;
        sines[i] = sn * a.gain;
    }
    // Written and read by one wave: the hardware keeps its order, the fences make the compiler keep it (no instruction comes
    // of them).
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");

#pragma unroll
    for (int h = 0; h < (int)HB; h++) {
        const uint32_t j = job(h);
        const bool q = j < a.nq, k = j < a.nqk;
        float v[NU][N];
#pragma unroll
        for (int i = 0; i < NU; i++)
#pragma unroll
            for (int e = 0; e < N; e++) v[i][e] = (float)raw[h][i].x[e];
        if (!PAGED || k) { // values pass as they are
            const float *w = q ? a.qw : a.kw;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < NU; i++) {
                float one = 0.0f, second = 0.0f;
#pragma unroll
                for (int e = 0; e < VEC; e++) one = fmaf(v[i][e], v[i][e], one);
                if (!INTER) {
#pragma unroll
                    for (int e = VEC; e < N; e++) second = fmaf(v[i][e], v[i][e], second);
                }
                sum += (have[i] ? one : 0.0f) + (both[i] ? second : 0.0f);
            }
            for (uint32_t d = 1; d < lanes; d *= 2) sum += __shfl_xor(sum, (int)d);
            const float scale = rsqrtf(sum * a.inv_hd + a.eps);
#pragma unroll
            for (int i = 0; i < NU; i++) {
                float x[N], c[PAIRS], s[PAIRS];
                load_n<AQ_TYPE_F32, VEC, W>(w + at[i], x);
                if (!INTER) load_n<AQ_TYPE_F32, VEC, W>(w + two[i], x + N - VEC);
#pragma unroll
                for (int e = 0; e < PAIRS; e++) {
                    c[e] = cosines[pair[i] + e];
                    s[e] = sines[pair[i] + e];
                }
#pragma unroll
                for (int e = 0; e < N; e++) x[e] *= v[i][e] * scale;
#pragma unroll
                for (int e = 0; e < PAIRS; e++) {
                    const int ia = INTER ? 2 * e : e, ib = INTER ? 2 * e + 1 : VEC + e;
                    const float p = fmaf(x[ia], c[e], -(x[ib] * s[e])), r = fmaf(x[ib], c[e], x[ia] * s[e]);
                    v[i][ia] = rot[i] ? p : x[ia];
                    v[i][ib] = rot[i] ? r : x[ib];
                }
            }
        }
        if (j0 + h * per >= a.jobs) continue;
        auto put = [&](auto *to) {
#pragma unroll
            for (int i = 0; i < NU; i++) {
                if (have[i]) store_raw<VEC, W>(to + at[i], v[i]);
                if (both[i]) store_raw<VEC, W>(to + two[i], v[i] + N - VEC);
            }
        };
        if (q) {
            put((EI *)a.qo.p + row * a.qo.row + (int64_t)j * a.qo.head);
        } else if constexpr (PAGED) {
            char *to = const_cast<char *>(k ? a.kv.k : a.kv.v) + ((uint64_t)off << a.kv.unit_shift) +
                       (uint64_t)(k ? j - a.nq : j - a.nqk) * a.kv.head_bytes;
            if (store) put((EO *)to);
        } else {
            put((EI *)a.ko.p + row * a.ko.row + (int64_t)(j - a.nq) * a.ko.head);
        }
    }
}

// vec: values moved at a time, 0: one (two neighbours) after the other.
template <int TI, int TO, bool PAGED>
int norm_pick(const NormArgs &a, bool inter, uint32_t vec, dim3 grid, hipStream_t stream) {
    constexpr int WIDE = TI == AQ_TYPE_F32 && TO == AQ_TYPE_F32 ? 4 : 8;
    if (inter) {
        if (vec == WIDE) norm_kernel<TI, TO, true, WIDE, true, 1, PAGED><<<grid, 256, 0, stream>>>(a);
        else if (vec) norm_kernel<TI, TO, true, 4, true, 1, PAGED><<<grid, 256, 0, stream>>>(a);
        else norm_kernel<TI, TO, true, 2, false, 2, PAGED><<<grid, 256, 0, stream>>>(a);
    } else {
        if (vec == WIDE) norm_kernel<TI, TO, false, WIDE, true, 1, PAGED><<<grid, 256, 0, stream>>>(a);
        else if (vec) norm_kernel<TI, TO, false, 4, true, 1, PAGED><<<grid, 256, 0, stream>>>(a);
        else norm_kernel<TI, TO, false, 1, false, 2, PAGED><<<grid, 256, 0, stream>>>(a);
    }
    AQ_HIP(hipGetLastError());
    return 0;
}

// What both calls check of the norm and the rotation.
int check_norm(const char *call, aq_ctx *ctx, const aq_rope *rope, const int32_t *pos, uint32_t hd, float eps) {
    auto who = [&] { return std::string(call); };
    AQ_REQUIRE((uintptr_t)pos % 4 == 0, who() + ": pos_dev is not aligned to its type");
    AQ_REQUIRE(std::isfinite(eps) && eps > 0.0f, who() + ": eps");
    if (rope) {
        AQ_REQUIRE(rope->ctx->device == ctx->device, who() + ": the rope is on another device");
        AQ_REQUIRE(rope->dim <= hd, who() + ": head_dim " + std::to_string(hd) + " is less than the rotated " +
                                        std::to_string(rope->dim));
    }
    return 0;
}
int check_weight(const char *call, const char *what, const float *w) {
    AQ_REQUIRE(w && (uintptr_t)w % 4 == 0, std::string(call) + ": " + what + " is null or not aligned to its type");
    return 0;
}
bool weight_aligned(const float *w) { return (uintptr_t)w % 16 == 0; }
int check_in_place(const char *call, const aq_heads *x, const aq_heads *y) {
    AQ_REQUIRE(x->type == y->type, std::string(call) + ": rows and outputs of different types");
    AQ_REQUIRE(x->data != y->data || (x->row_stride == y->row_stride && x->head_stride == y->head_stride),
               std::string(call) + ": in place needs the same strides");
    return 0;
}

// Values moved at a time: as many as 16 bytes of the rows or of the cache hold, or 4, where the units and all that is read and
// written allow it (6000 rows of 32 heads of 80 of which 40 are turned, bf16: 4 a time 17.8 us, 1 a time 59.8).
uint32_t values_at_once(const aq_rope *rope, uint32_t hd, bool f32, bool aligned) {
    const uint32_t layout = rope ? rope->layout : (uint32_t)AQ_ROPE_HALF, dim = rope ? rope->dim : 0;
    if (aligned && !f32 && wide_fits(layout, dim, hd, 8)) return 8;
    return aligned && wide_fits(layout, dim, hd, 4) ? 4 : 0;
}

// The units, the lanes of a head, and the launch (row_bytes: of a value of the rows); false: more waves than a launch has.
bool shape(NormArgs &a, const aq_rope *rope, uint32_t hd, uint32_t vec, uint32_t row_bytes, float eps, dim3 *grid) {
    const bool inter = rope && rope->layout == AQ_ROPE_INTERLEAVED;
    a.dim = rope ? rope->dim : 0;
    a.freq = rope ? rope->freq : nullptr;
    a.gain = rope ? rope->gain : 1.0f;
    a.eps = eps;
    a.inv_hd = 1.0f / (float)hd;
    const uint32_t v = vec ? vec : inter ? 2 : 1, pass = (hd - a.dim) / v;
    a.rot_units = a.dim / v / (inter ? 1 : 2);
    a.pass_units = inter ? pass : (pass + 1) / 2;
    a.pass_seconds = pass - a.pass_units;
    a.units = a.rot_units + a.pass_units;
    a.lane_shift = 0;
    while (a.lane_shift < 6 && (1u << a.lane_shift) < a.units) a.lane_shift++;
    const uint32_t per = heads_per_lane((inter ? v : 2 * v) * row_bytes) * (64u >> a.lane_shift);
    a.parts = (a.jobs + per - 1) / per;
    a.by_parts = FastDiv(a.parts);
    const uint64_t waves = (uint64_t)a.parts * a.n_rows;
    if (waves >= (1ull << 31) - (1u << 23)) return false;
    const uint32_t groups = (uint32_t)((waves + 3) / 4), most = 1u << 20;
    *grid = groups <= most ? dim3(groups) : dim3(most, (groups + most - 1) / most);
    return true;
}

} // namespace
} // namespace aq

using namespace aq;

extern "C" {

int aq_qk_norm_rope(aq_ctx *ctx, const aq_heads *q, const aq_heads *q_out, uint32_t n_head, const aq_heads *k,
                    const aq_heads *k_out, uint32_t n_head_kv, uint32_t head_dim, size_t n_rows, const float *q_weight,
                    const float *k_weight, float eps, const aq_rope *rope, const int32_t *pos_dev, void *stream) {
    const char *call = "aq_qk_norm_rope";
    AQ_REQUIRE(ctx, "aq_qk_norm_rope: null ctx");
    AQ_REQUIRE(q || k, "aq_qk_norm_rope: neither q nor k");
    AQ_REQUIRE(!q == !q_out && !k == !k_out, "aq_qk_norm_rope: rows and their outputs go together");
    AQ_REQUIRE(n_rows < (1u << 24) && (!q || (n_head > 0 && n_head <= 65535)) && (!k || (n_head_kv > 0 && n_head_kv <= 65535)),
               "aq_qk_norm_rope: size");
    if (head_dim == 0 || head_dim > MAX_HEAD)
        return fail(AQ_EUNSUP, "aq_qk_norm_rope: head_dim " + std::to_string(head_dim) + " (1 to 256)");
    int rc = check_norm(call, ctx, rope, pos_dev, head_dim, eps);
    if (!rc && q) rc = check_heads(call, "q", q, n_rows, n_head, head_dim);
    if (!rc && q) rc = check_heads(call, "q_out", q_out, n_rows, n_head, head_dim);
    if (!rc && k) rc = check_heads(call, "k", k, n_rows, n_head_kv, head_dim);
    if (!rc && k) rc = check_heads(call, "k_out", k_out, n_rows, n_head_kv, head_dim);
    if (!rc && q) rc = check_weight(call, "q_weight", q_weight);
    if (!rc && k) rc = check_weight(call, "k_weight", k_weight);
    if (!rc && q) rc = check_in_place(call, q, q_out);
    if (!rc && k) rc = check_in_place(call, k, k_out);
    if (rc) return rc;
    AQ_REQUIRE(!q || !k || q->type == k->type, "aq_qk_norm_rope: q and k of different types");
    AQ_REQUIRE(!rope == !pos_dev, "aq_qk_norm_rope: a rope and positions go together");
    if (n_rows == 0) return 0;
    const int type = q ? q->type : k->type;
    const bool inter = rope && rope->layout == AQ_ROPE_INTERLEAVED;
    const bool aligned =
        (!q || (heads_aligned(q, n_rows, n_head) && heads_aligned(q_out, n_rows, n_head) && weight_aligned(q_weight))) &&
        (!k || (heads_aligned(k, n_rows, n_head_kv) && heads_aligned(k_out, n_rows, n_head_kv) && weight_aligned(k_weight)));
    const uint32_t vec = values_at_once(rope, head_dim, type == AQ_TYPE_F32, aligned);
    AQ_REQUIRE(vec || !inter || head_dim % 2 == 0, "aq_qk_norm_rope: head_dim is odd");
    NormArgs a = {};
    if (q) {
        a.q = heads_view(q);
        a.qo = heads_view(q_out);
        a.qw = q_weight;
    }
    if (k) {
        a.k = heads_view(k);
        a.ko = heads_view(k_out);
        a.kw = k_weight;
    }
    a.pos = pos_dev;
    a.n_rows = (uint32_t)n_rows;
    a.nq = q ? n_head : 0;
    a.jobs = a.nqk = a.nq + (k ? n_head_kv : 0);
    dim3 grid;
    if (!shape(a, rope, head_dim, vec, (uint32_t)type_bytes(type), eps, &grid))
        return fail(AQ_EUNSUP, "aq_qk_norm_rope: more than 2^31 pieces of rows");
    AQ_HIP(hipSetDevice(ctx->device));
    const hipStream_t st = stream ? (hipStream_t)stream : ctx->stream;
    switch (type) {
    case AQ_TYPE_F32: return norm_pick<AQ_TYPE_F32, AQ_TYPE_F32, false>(a, inter, vec, grid, st);
    case AQ_TYPE_F16: return norm_pick<AQ_TYPE_F16, AQ_TYPE_F16, false>(a, inter, vec, grid, st);
    default: return norm_pick<AQ_TYPE_BF16, AQ_TYPE_BF16, false>(a, inter, vec, grid, st);
    }
}

int aq_paged_append_norm(aq_ctx *ctx, const aq_paged_kv *kv, const aq_paged_batch *batch, const aq_heads *k,
                         const aq_heads *v, const aq_heads *q, const aq_heads *q_out, uint32_t n_head, const float *q_weight,
                         const float *k_weight, float eps, const aq_rope *rope, const int32_t *pos_dev, void *stream) {
    const char *call = "aq_paged_append_norm";
    AQ_REQUIRE(ctx, "aq_paged_append_norm: null ctx");
    NormArgs a = {};
    int rc = check_paged(call, kv, batch, &a.kv, &a.b);
    if (rc) return rc;
    const uint32_t hd = kv->head_dim, rows = batch->n_rows;
    rc = check_norm(call, ctx, rope, pos_dev, hd, eps);
    if (!rc) rc = check_heads(call, "k", k, rows, kv->n_head_kv, hd);
    if (!rc) rc = check_heads(call, "v", v, rows, kv->n_head_kv, hd);
    if (!rc) rc = check_weight(call, "k_weight", k_weight);
    if (rc) return rc;
    AQ_REQUIRE(k->type == v->type, "aq_paged_append_norm: k and v of different types");
    AQ_REQUIRE(k->type == AQ_TYPE_F32 || k->type == kv->type, "aq_paged_append_norm: rows are F32 or of the cache's type");
    AQ_REQUIRE(!q == !q_out, "aq_paged_append_norm: q and q_out go together");
    if (q) {
        AQ_REQUIRE(n_head > 0 && n_head <= 65535, "aq_paged_append_norm: n_head");
        rc = check_heads(call, "q", q, rows, n_head, hd);
        if (!rc) rc = check_heads(call, "q_out", q_out, rows, n_head, hd);
        if (!rc) rc = check_weight(call, "q_weight", q_weight);
        if (!rc) rc = check_in_place(call, q, q_out);
        if (rc) return rc;
        AQ_REQUIRE(q->type == k->type, "aq_paged_append_norm: q and k of different types");
    }
    AQ_REQUIRE(rope || !pos_dev, "aq_paged_append_norm: positions without a rope");
    if (rows == 0 || batch->n_seq == 0) return 0;
    const bool inter = rope && rope->layout == AQ_ROPE_INTERLEAVED;
    const bool aligned =
        heads_aligned(k, rows, kv->n_head_kv) && heads_aligned(v, rows, kv->n_head_kv) && weight_aligned(k_weight) &&
        (!q || (heads_aligned(q, rows, n_head) && heads_aligned(q_out, rows, n_head) && weight_aligned(q_weight)));
    const uint32_t vec = values_at_once(rope, hd, kv->type == AQ_TYPE_F32, aligned);
    a.k = heads_view(k);
    a.v = heads_view(v);
    a.kw = k_weight;
    if (q) {
        a.q = heads_view(q);
        a.qo = heads_view(q_out);
        a.qw = q_weight;
    }
    a.pos = pos_dev;
    a.n_rows = rows;
    a.nq = q ? n_head : 0;
    a.nqk = a.nq + kv->n_head_kv;
    a.jobs = a.nqk + kv->n_head_kv;
    dim3 grid;
    if (!shape(a, rope, hd, vec, (uint32_t)type_bytes(k->type), eps, &grid))
        return fail(AQ_EUNSUP, "aq_paged_append_norm: more than 2^31 pieces of rows");
    AQ_HIP(hipSetDevice(ctx->device));
    const hipStream_t st = stream ? (hipStream_t)stream : ctx->stream;
    if (k->type == AQ_TYPE_F32) {
        if (kv->type == AQ_TYPE_F32) return norm_pick<AQ_TYPE_F32, AQ_TYPE_F32, true>(a, inter, vec, grid, st);
        if (kv->type == AQ_TYPE_F16) return norm_pick<AQ_TYPE_F32, AQ_TYPE_F16, true>(a, inter, vec, grid, st);
        return norm_pick<AQ_TYPE_F32, AQ_TYPE_BF16, true>(a, inter, vec, grid, st);
    }
    if (kv->type == AQ_TYPE_F16) return norm_pick<AQ_TYPE_F16, AQ_TYPE_F16, true>(a, inter, vec, grid, st);
    return norm_pick<AQ_TYPE_BF16, AQ_TYPE_BF16, true>(a, inter, vec, grid, st);
}

} // extern "C"
