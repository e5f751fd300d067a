// norm_rope.hip — the norms of queries and keys head by head with their rotation in the same pass, over rows of heads
// (aq_qk_norm_rope) and on the way into the pages (aq_paged_append_norm).
//
// y = x / sqrt(mean(x^2) + eps) * weight over the head's values, in 32 bits, then its pairs turned as rope.hip turns them, and
// one rounding at the store. A head's values lie on a group of lanes, one unit (rope.h) each, so that both values of a pair are
// in one lane and the sum of squares is one exchange per doubling of the group. A row's angles are computed once for all of
// its heads, one a thread, and handed over in the LDS; the first heads' values are on their way meanwhile.
#include <cmath>
#include <type_traits>

#include "rope.h"

namespace aq {
namespace {

constexpr int MAX_HEAD = 256, MAX_THREADS = 512;

struct NormArgs {
    PagedKv kv;
    PagedBatch b;
    HeadsView q, qo, k, ko, v;
    const float *qw, *kw;
    const double *freq;
    const int32_t *pos; // of each row; null: its place in its sequence
    uint32_t n_rows, dim, rot_units, units, lane_shift;
    uint32_t nq, nqk, jobs; // heads of a row: queries, keys after them, values after those
    float eps, inv_hd, gain;
};

// One row per blockIdx.x, its heads over blockIdx.y and the threads' groups of 2^lane_shift lanes, two at a time. NU: units a
// lane has at most (one where 16 bytes are moved at a time).
template <int TI, int TO, bool INTER, int VEC, bool W, int NU, bool PAGED>
__global__ void __launch_bounds__(MAX_THREADS) norm_kernel(NormArgs a) {
    using EI = typename RowType<TI>::type;
    using EO = typename RowType<TO>::type;
    constexpr int N = INTER ? VEC : 2 * VEC, PAIRS = N / 2, HB = 2;
    __shared__ float cosines[MAX_HEAD / 2], sines[MAX_HEAD / 2];
    const uint32_t row = blockIdx.x, lanes = 1u << a.lane_shift;
    int32_t pos = 0;
    bool store = true;
    uint32_t off = 0;
    if constexpr (PAGED) {
        const uint32_t seq = paged_seq_of(a.b, row);
        if (seq >= a.b.n_seq) return; // uniform in the work-group, as all of this
        const SeqRows sr = paged_seq(a.b, seq);
        if ((int32_t)row < sr.first) return; // before the first sequence's rows
        pos = sr.base + ((int32_t)row - sr.first);
        store = pos >= 0 && paged_slot(a.kv, a.b.pages + (size_t)seq * a.b.max_pages, a.b.max_pages, (uint32_t)pos, &off);
    }
    if (a.pos) pos = a.pos[row];

    const uint32_t lane0 = threadIdx.x & (lanes - 1);
    uint32_t at[NU]; // where each of this lane's units begins; bit i: it is there, it is turned
    uint32_t have = 0, rot = 0;
#pragma unroll
    for (int i = 0; i < NU; i++) {
        const uint32_t u = lane0 + ((uint32_t)i << a.lane_shift);
        have |= u < a.units ? 1u << i : 0u;
        rot |= u < a.rot_units ? 1u << i : 0u;
        at[i] = u < a.rot_units ? u * VEC : a.dim + (u - a.rot_units) * VEC;
    }
    // A job: one head of the row's queries, keys or values.
    float v[HB][NU][N];
    auto source = [&](uint32_t j) {
        const HeadsView &s = j < a.nq ? a.q : j < a.nqk ? a.k : a.v;
        const uint32_t head = j < a.nq ? j : j < a.nqk ? j - a.nq : j - a.nqk;
        return (const EI *)s.p + (int64_t)row * s.row + (int64_t)head * s.head;
    };
    auto fetch = [&](uint32_t j, float (*x)[N]) {
        const EI *p = source(j);
#pragma unroll
        for (int i = 0; i < NU; i++) {
            if (!((have >> i) & 1)) continue;
            load_n<TI, VEC, W>(p + at[i], x[i]);
            if (!INTER && ((rot >> i) & 1)) load_n<TI, VEC, W>(p + at[i] + a.dim / 2, x[i] + N - VEC);
        }
    };
    const uint32_t group = (blockIdx.y * blockDim.x + threadIdx.x) >> a.lane_shift,
                   groups = (gridDim.y * blockDim.x) >> a.lane_shift;
#pragma unroll
    for (int h = 0; h < HB; h++)
        if (group + h * groups < a.jobs) fetch(group + h * groups, v[h]);

    for (uint32_t i = threadIdx.x; i < a.dim / 2; i += blockDim.x) {
        float sn, cs;
        rope_angle(a.freq[i], pos, &sn, &cs);
        cosines[i] = cs * a.gain;
        sines[i] = sn * a.gain;
    }
    __syncthreads();
    float c[NU][PAIRS], s[NU][PAIRS];
#pragma unroll
    for (int i = 0; i < NU; i++)
#pragma unroll
        for (int e = 0; e < PAIRS; e++) {
            const uint32_t pair = (rot >> i) & 1 ? (INTER ? at[i] / 2 : at[i]) + e : 0;
            c[i][e] = cosines[pair];
            s[i][e] = sines[pair];
        }

    for (uint32_t j0 = group; j0 < a.jobs; j0 += HB * groups) {
        if (j0 != group) {
#pragma unroll
            for (int h = 0; h < HB; h++)
                if (j0 + h * groups < a.jobs) fetch(j0 + h * groups, v[h]);
        }
#pragma unroll
        for (int h = 0; h < HB; h++) {
            const uint32_t j = j0 + h * groups;
            if (j >= a.jobs) continue;
            if (j < a.nqk) {
                const float *w = j < a.nq ? a.qw : a.kw;
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < NU; i++) {
                    if (!((have >> i) & 1)) continue;
#pragma unroll
                    for (int e = 0; e < N; e++)
                        if (INTER || e < VEC || ((rot >> i) & 1)) sum = fmaf(v[h][i][e], v[h][i][e], sum);
                }
                for (uint32_t d = 1; d < lanes; d *= 2) sum += __shfl_xor(sum, (int)d);
                const float scale = rsqrtf(sum * a.inv_hd + a.eps);
#pragma unroll
                for (int i = 0; i < NU; i++) {
                    if (!((have >> i) & 1)) continue;
                    const bool turned = (rot >> i) & 1;
                    float x[N];
                    load_n<AQ_TYPE_F32, VEC, W>(w + at[i], x);
                    if (!INTER && turned) load_n<AQ_TYPE_F32, VEC, W>(w + at[i] + a.dim / 2, x + N - VEC);
#pragma unroll
                    for (int e = 0; e < N; e++)
                        if (INTER || e < VEC || turned) x[e] = v[h][i][e] * scale * x[e];
#pragma unroll
                    for (int e = 0; e < PAIRS; e++) {
                        const int ia = INTER ? 2 * e : e, ib = INTER ? 2 * e + 1 : VEC + e;
                        const float p = x[ia], r = x[ib];
                        v[h][i][ia] = turned ? fmaf(p, c[i][e], -(r * s[i][e])) : p;
                        v[h][i][ib] = turned ? fmaf(r, c[i][e], p * s[i][e]) : r;
                    }
                }
            }
            auto put = [&](auto *p, auto type) {
                constexpr int T = decltype(type)::value;
#pragma unroll
                for (int i = 0; i < NU; i++) {
                    if (!((have >> i) & 1)) continue;
                    store_n<T, VEC, W>(p + at[i], v[h][i]);
                    if (!INTER && ((rot >> i) & 1)) store_n<T, VEC, W>(p + at[i] + a.dim / 2, v[h][i] + N - VEC);
                }
            };
            if (j < a.nq) {
                put((EI *)a.qo.p + (int64_t)row * a.qo.row + (int64_t)j * a.qo.head, std::integral_constant<int, TI>());
            } else if constexpr (PAGED) {
                const bool key = j < a.nqk;
                char *p = const_cast<char *>(key ? a.kv.k : a.kv.v) + ((uint64_t)off << a.kv.unit_shift) +
                          (uint64_t)(key ? j - a.nq : j - a.nqk) * a.kv.head_bytes;
                if (store) put((EO *)p, std::integral_constant<int, TO>());
            } else {
                put((EI *)a.ko.p + (int64_t)row * a.ko.row + (int64_t)(j - a.nq) * a.ko.head,
                    std::integral_constant<int, TI>());
            }
        }
    }
}

template <int TI, int TO, bool PAGED>
int norm_pick(const NormArgs &a, bool inter, bool wide, dim3 grid, uint32_t threads, hipStream_t stream) {
    constexpr int VW = TI == AQ_TYPE_F32 && TO == AQ_TYPE_F32 ? 4 : 8;
    if (inter) {
        if (wide) norm_kernel<TI, TO, true, VW, true, 1, PAGED><<<grid, threads, 0, stream>>>(a);
        else norm_kernel<TI, TO, true, 2, false, 2, PAGED><<<grid, threads, 0, stream>>>(a);
    } else {
        if (wide) norm_kernel<TI, TO, false, VW, true, 1, PAGED><<<grid, threads, 0, stream>>>(a);
        else norm_kernel<TI, TO, false, 1, false, 4, PAGED><<<grid, threads, 0, stream>>>(a);
    }
    AQ_HIP(hipGetLastError());
    return 0;
}

// What both calls check of the norm and the rotation.
int check_norm(const char *call, aq_ctx *ctx, const aq_rope *rope, uint32_t hd, float eps) {
    auto who = [&] { return std::string(call); };
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

// The units, the lanes of a head, and the launch. `vec`: values moved at a time where `wide`.
void shape(NormArgs &a, const aq_rope *rope, uint32_t hd, uint32_t vec, bool wide, float eps, dim3 *grid, uint32_t *threads) {
    const bool inter = rope && rope->layout == AQ_ROPE_INTERLEAVED;
    a.dim = rope ? rope->dim : 0;
    a.freq = rope ? rope->freq : nullptr;
    a.gain = rope ? rope->gain : 1.0f;
    a.eps = eps;
    a.inv_hd = 1.0f / (float)hd;
    unit_shape(inter ? AQ_ROPE_INTERLEAVED : AQ_ROPE_HALF, a.dim, hd, wide ? vec : inter ? 2 : 1, &a.rot_units, &a.units);
    a.lane_shift = 0;
    while (a.lane_shift < 6 && (1u << a.lane_shift) < a.units) a.lane_shift++;
    const uint32_t items = a.jobs << a.lane_shift; // lanes that a row needs at once
    // Few rows: a work-group to each wave's heads; many: a row to a work-group, two heads a group of lanes.
    uint32_t t = 64;
    if ((uint64_t)a.n_rows * items > (1u << 18)) {
        while (t < MAX_THREADS && t * 2 < items && (uint64_t)(t + 64) * a.n_rows < (1ull << 32)) t += 64;
        *grid = dim3(a.n_rows);
    } else {
        *grid = dim3(a.n_rows, (items + t - 1) / t);
    }
    *threads = t;
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
    int rc = check_norm(call, ctx, rope, head_dim, eps);
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
    const uint32_t vec = 16 / (uint32_t)type_bytes(type);
    const bool wide = (!q || (heads_aligned(q, n_rows, n_head) && heads_aligned(q_out, n_rows, n_head) && weight_aligned(q_weight))) &&
                      (!k || (heads_aligned(k, n_rows, n_head_kv) && heads_aligned(k_out, n_rows, n_head_kv) && weight_aligned(k_weight))) &&
                      wide_fits(inter ? AQ_ROPE_INTERLEAVED : AQ_ROPE_HALF, rope ? rope->dim : 0, head_dim, vec);
    AQ_REQUIRE(wide || !inter || head_dim % 2 == 0, "aq_qk_norm_rope: head_dim is odd");
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
    uint32_t threads;
    shape(a, rope, head_dim, vec, wide, eps, &grid, &threads);
    AQ_HIP(hipSetDevice(ctx->device));
    const hipStream_t st = stream ? (hipStream_t)stream : ctx->stream;
    switch (type) {
    case AQ_TYPE_F32: return norm_pick<AQ_TYPE_F32, AQ_TYPE_F32, false>(a, inter, wide, grid, threads, st);
    case AQ_TYPE_F16: return norm_pick<AQ_TYPE_F16, AQ_TYPE_F16, false>(a, inter, wide, grid, threads, st);
    default: return norm_pick<AQ_TYPE_BF16, AQ_TYPE_BF16, false>(a, inter, wide, grid, threads, st);
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
    rc = check_norm(call, ctx, rope, hd, eps);
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
    const uint32_t vec = k->type == AQ_TYPE_F32 && kv->type == AQ_TYPE_F32 ? 4 : 8;
    const bool wide = heads_aligned(k, rows, kv->n_head_kv) && heads_aligned(v, rows, kv->n_head_kv) && weight_aligned(k_weight) &&
                      (!q || (heads_aligned(q, rows, n_head) && heads_aligned(q_out, rows, n_head) && weight_aligned(q_weight))) &&
                      wide_fits(inter ? AQ_ROPE_INTERLEAVED : AQ_ROPE_HALF, rope ? rope->dim : 0, hd, vec);
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
    uint32_t threads;
    shape(a, rope, hd, vec, wide, eps, &grid, &threads);
    AQ_HIP(hipSetDevice(ctx->device));
    const hipStream_t st = stream ? (hipStream_t)stream : ctx->stream;
    if (k->type == AQ_TYPE_F32) {
        if (kv->type == AQ_TYPE_F32) return norm_pick<AQ_TYPE_F32, AQ_TYPE_F32, true>(a, inter, wide, grid, threads, st);
        if (kv->type == AQ_TYPE_F16) return norm_pick<AQ_TYPE_F32, AQ_TYPE_F16, true>(a, inter, wide, grid, threads, st);
        return norm_pick<AQ_TYPE_F32, AQ_TYPE_BF16, true>(a, inter, wide, grid, threads, st);
    }
    if (kv->type == AQ_TYPE_F16) return norm_pick<AQ_TYPE_F16, AQ_TYPE_F16, true>(a, inter, wide, grid, threads, st);
    return norm_pick<AQ_TYPE_BF16, AQ_TYPE_BF16, true>(a, inter, wide, grid, threads, st);
}

} // extern "C"
