// paged_attention.hip — attention over a paged K/V cache (aq_paged_attention): the choice of kernel (paged_few.h for
// few rows and for f32 rows, paged_chunk.hip for many 16-bit rows), the plan and the join of split sequences.
#include <algorithm>
#include <cmath>
#include <mutex>

#include "paged_attn.h"

namespace aq {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------------------------------------------- the join
// The rows of one cut segment: segment blockIdx.x of all, or, BY_SHARE, the one that begins in share blockIdx.x and goes on
// past it (where there are more segments than shares). Threads of a group of D / 4 have four dimensions each; ROWS groups
// side by side take a row each, and GROUPS of them every so many parts of it, whose outputs, each times 2^(its maximum -
// the running one), meet in the LDS.
template <int QT, int THREADS, int D, int GROUPS, bool BY_SHARE>
__global__ void __launch_bounds__(THREADS) join_kernel(AttnPagedArgs a, int R) {
    constexpr int QUADS = D / 4, ROWS = THREADS / (QUADS * GROUPS);
    __shared__ uint32_t found;
    __shared__ f4 os[GROUPS > 1 ? THREADS : 1];
    __shared__ float ms[GROUPS > 1 ? THREADS : 1], ls[GROUPS > 1 ? THREADS : 1];
    const int tid = threadIdx.x;
    const uint32_t nkv = (uint32_t)a.kv.nkv, total = a.plan[0], chunk = a.plan[1], n_seg = a.plan[2];
    const uint32_t *line = a.plan + PLAN_HEAD;
    uint32_t j, kvh, s0, cnt;
    RowTile t;
    if constexpr (BY_SHARE) {
        const uint64_t end64 = (uint64_t)(blockIdx.x + 1) * chunk;
        if (end64 >= total) return; // the last share, or none
        const uint32_t end = (uint32_t)end64;
        for (uint32_t i = tid; i < n_seg; i += THREADS)
            if (tile_holds(a.tiles[i], line[i], line[i + 1], nkv, end, &kvh)) found = i;
        __syncthreads();
        j = found;
        t = a.tiles[j];
        kvh = (end - t.p0 * nkv) / (t.p1 - t.p0);
        s0 = tile_place(t, line[j], nkv, kvh) + a.lead; // the first unit's place
        cnt = line[j + 1] - line[j] - a.lead;
        if (s0 >= end || s0 / chunk != blockIdx.x) return; // begins there, or before this share
    } else {
        j = blockIdx.x / nkv;
        kvh = blockIdx.x % nkv;
        const uint32_t p0 = line[j], p1 = line[j + 1]; // one latency for all of the plan
        t = a.tiles[j];
        if (j >= n_seg) return;
        s0 = tile_place(t, p0, nkv, kvh) + a.lead;
        cnt = p1 - p0 - a.lead;
    }
    const uint32_t w0 = s0 / chunk, w1 = (s0 + cnt - 1) / chunk;
    if (w0 == w1) return; // one share had it all
    const SeqRows sr = paged_seq(a.b, t.seq);
    const int row = (int)blockIdx.y * ROWS + tid / (QUADS * GROUPS), grp = tid / QUADS % GROUPS, dim = tid % QUADS * 4;
    const int32_t rr = (int32_t)t.rt * R + row;
    const bool have = row < R && rr < sr.n * a.G && dim < a.kv.hd;
    float m = -INFINITY, l = 0.0f;
    f4 o = f4{0.0f, 0.0f, 0.0f, 0.0f};
    if (have) {
#pragma unroll 4
        for (uint32_t w = w0 + grp; w <= w1; w += GROUPS) {
            const size_t at = (size_t)(2 * w + (w == w0 ? 1 : 0)) * R + row;
            const float pm = a.part_ml[at * 2], pl = a.part_ml[at * 2 + 1];
            const f4 po = *reinterpret_cast<const f4 *>(a.part_o + at * D + dim);
            const float mn = fmaxf(m, pm), mu = mn == -INFINITY ? 0.0f : mn;
            const float x = fast_exp2(m - mu), y = fast_exp2(pm - mu);
            m = mn;
            l = l * x + pl * y;
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] = o[i] * x + po[i] * y;
        }
    }
    if constexpr (GROUPS > 1) {
        os[tid] = o;
        ms[tid] = m;
        ls[tid] = l;
        __syncthreads();
        if (grp) return;
        float mx = m;
#pragma unroll 4
        for (int x = 1; x < GROUPS; x++) mx = fmaxf(mx, ms[x * QUADS + tid]);
        const float mu = mx == -INFINITY ? 0.0f : mx, x0 = fast_exp2(m - mu);
        l *= x0;
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] *= x0;
#pragma unroll 4
        for (int x = 1; x < GROUPS; x++) {
            const float y = fast_exp2(ms[x * QUADS + tid] - mu);
            l += ls[x * QUADS + tid] * y;
            const f4 t = os[x * QUADS + tid];
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] += t[i] * y;
        }
    }
    if (!have) return;
    float out[4];
#pragma unroll
    for (int i = 0; i < 4; i++) out[i] = l == 0.0f ? 0.0f : o[i] / l;
    const int32_t tok = (int32_t)a.by_g.quot(rr);
    store_out<QT>(a, sr.first + tok, (int)kvh * a.G + (rr - tok * a.G), dim, out);
}

// Few rows: a work-group per row, of 1024 threads where a row has many parts (a long context of one sequence has hundreds:
// 24 rows of 63 parts of 256 dimensions take 5.9 us, with 256 threads 9.9); with more segments than shares 512 threads on
// 512 / D rows, most of which have two parts or are whole (work-groups of 256 on a row each: f32 prompts of four requests of
// 500, 16 heads on 2 of 64, 71.4 us in all for 55.1). Many rows: 256 threads, a row per D / 4 of them, its two to a few
// parts one after the other.
template <int QT, int D>
void join_launch(const AttnPagedArgs &a, int R, int rows, hipStream_t stream) {
    const uint32_t segs = a.n_seg * (uint32_t)a.kv.nkv;
    if (R > 32) {
        constexpr int ROWS = 256 / (D / 4);
        const uint32_t y = (uint32_t)((rows + ROWS - 1) / ROWS);
        if (segs <= a.shares) join_kernel<QT, 256, D, 1, false><<<dim3(segs, y), 256, 0, stream>>>(a, R);
        else join_kernel<QT, 256, D, 1, true><<<dim3(a.shares, y), 256, 0, stream>>>(a, R);
    } else if (segs <= a.shares / 16) {
        join_kernel<QT, 1024, D, 1024 / (D / 4), false><<<dim3(segs, (uint32_t)rows), 1024, 0, stream>>>(a, R);
    } else if (segs <= a.shares) {
        join_kernel<QT, 256, D, 256 / (D / 4), false><<<dim3(segs, (uint32_t)rows), 256, 0, stream>>>(a, R);
    } else {
        constexpr int ROWS = 512 / D;
        join_kernel<QT, 512, D, 4, true><<<dim3(a.shares, (uint32_t)((rows + ROWS - 1) / ROWS)), 512, 0, stream>>>(a, R);
    }
}
template <int QT>
void join_pick(const AttnPagedArgs &a, int R, int D, int rows, hipStream_t stream) {
    if (D == 64) join_launch<QT, 64>(a, R, rows, stream);
    else if (D == 128) join_launch<QT, 128>(a, R, rows, stream);
    else join_launch<QT, 256>(a, R, rows, stream);
}

// ---------------------------------------------------------------------------------------------------- the plan
// Of batches of more sequences or row tiles than a work-group divides by itself: all row tiles in order, and the prefix
// sums of their units; one work-group. Around the border (single tokens at 200, 32 heads on 8 of 128, bf16): 1020 sequences
// 260 us, 1030 265.
__global__ void __launch_bounds__(1024) plan_kernel(AttnPagedArgs a, int R, uint32_t tk) {
    __shared__ uint32_t wsum[16], carry, first[1024];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // the inclusive prefix sum of v over the work-group, plus what came before; uniform calls
    auto scan = [&](uint32_t v) {
        uint32_t s = wave_scan(v);
        if (lane == 63) wsum[wave] = s;
        __syncthreads();
        for (int i = 0; i < wave; i++) s += wsum[i];
        s += carry;
        __syncthreads();
        if (tid == 1023) carry = s;
        __syncthreads();
        return s;
    };
    if (tid == 0) carry = 0;
    __syncthreads();
    // the row tiles of 1024 sequences at a time, each found by its number
    for (uint32_t s0 = 0; s0 < a.b.n_seq; s0 += 1024) {
        const uint32_t from = carry, n = min(seq_tiles(a, s0 + tid, R), a.n_seg);
        first[tid] = scan(n) - n;
        __syncthreads();
        const uint32_t to = min(carry, a.n_seg);
        for (uint32_t j = from + tid; j < to; j += 1024) {
            uint32_t lo = 0, hi = min(1024u, a.b.n_seq - s0); // the last sequence that begins at or before j
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) / 2;
                if (first[mid] <= j) lo = mid;
                else hi = mid;
            }
            a.tiles[j].seq = s0 + lo;
            a.tiles[j].rt = j - first[lo];
        }
        __syncthreads();
        if (carry > a.n_seg) break; // sequences that overlap: not a batch
    }
    const uint32_t n_seg = min(carry, a.n_seg);
    __syncthreads();
    if (tid == 0) carry = 0;
    __syncthreads();
    for (uint32_t j0 = 0; j0 < n_seg; j0 += 1024) {
        const uint32_t j = j0 + tid;
        uint32_t n = 0;
        if (j < n_seg) n = tile_count(a, a.tiles[j].seq, a.tiles[j].rt, R, tk); // its own, or ordered by the barriers above
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
    __syncthreads(); // the prefix sums are written
    for (uint32_t j = tid; j < n_seg; j += 1024) {
        const uint32_t j0 = j - a.tiles[j].rt, j1 = min(j0 + seq_tiles(a, a.tiles[j].seq, R), n_seg);
        a.tiles[j].p0 = a.plan[PLAN_HEAD + j0];
        a.tiles[j].p1 = a.plan[PLAN_HEAD + j1];
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
    uint32_t unit = 0, per = 0, shares = 0, min_chunk = 1, lead = 0, whole = 0, n_seg = 0, cap = 0;
    bool planned = false, join = false;
    PagedSpace space;
};

// Rows of a K/V head of the longest sequence, and the positions a batch can reach.
uint64_t longest_rows(const aq_paged_kv *kv, const aq_paged_batch *b, uint32_t n_head) {
    return (uint64_t)b->max_rows * (n_head / kv->n_head_kv);
}
uint32_t reach_of(const aq_paged_kv *kv, const aq_paged_batch *b) {
    return (uint32_t)std::min<uint64_t>((uint64_t)b->max_pages * kv->page_size, b->max_len);
}
// Paged chunks for 16-bit rows past one row tile of the few-row kernel, once there is enough to do: its start (code,
// 128-row blocks) takes 12 to 30 us whatever the work, each further row tile of the other reads K and V again. Few-row
// and chunk kernel, by rows x heads x positions (bf16, us): heads of 256: 0.04M 13.6 and 29.2, 3.1M 37.7 and 43.3, 4.6M
// 40.7 and 43.9, 7.4M 54.6 and 48.7; of 128: 0.05M 9.8 and 18.2, 4.1M 27.4 and 30.0, 4.4M 30.9 and 30.0, 7.7M 41.9 and
// 38.5, 46M 211 and 136; of 64: 5.0M 22.2 and 24.2, 10M 30.0 and 26.1, 31M 81 and 59.
bool takes_chunks(const aq_paged_kv *kv, const aq_paged_batch *b, uint32_t n_head) {
    return longest_rows(kv, b, n_head) > 32 && (double)b->n_rows * n_head * reach_of(kv, b) > 5.0 * (1 << 20);
}

// The work on row tiles of R rows, and the workspace it takes: that grows with each of the batch's bounds.
Choice on_tiles(const aq_paged_kv *kv, const aq_paged_batch *b, uint32_t n_head, bool many, int R, int device) {
    Choice c;
    const uint32_t G = n_head / kv->n_head_kv;
    c.many = many;
    c.R = R;
    c.D = kv->head_dim <= 64 ? 64 : kv->head_dim <= 128 ? 128 : 256;
    c.cap = reach_of(kv, b);
    c.unit = c.many ? chunk_keys(c.D) : few_unit(kv->type, c.D, c.R);
    c.min_chunk = c.many ? 256 / c.unit : 1;
    // What a segment costs besides its positions (queries, first loads, the waves' meeting, its output), in units. Prompts
    // of three requests (9733 rows of 32 heads of 128), of 64 positions: 0: 794 us, 2: 532, 4: 459, 6: 459, 8: 467. Eight
    // verify batches of 32 rows (f32 over f16, heads of 256), of 32: 0: 46.4, 2: 42.5, 4: 42.6. Single tokens: none to gain;
    // nor where a unit takes as long as that (f32 products).
    c.lead = c.many ? 320 / c.unit : c.R == 32 && kv->type != AQ_TYPE_F32 ? 2 : 0;
    // row tiles: a whole one per R rows of all sequences together, and one begun per sequence
    const uint64_t n_seg = std::min<uint64_t>((uint64_t)b->n_rows * G / c.R + b->n_seq, (uint64_t)b->n_rows * G);
    c.planned = n_seg > INLINE_TILES || b->n_seq > INLINE_TILES;
    // places of a segment at most (a window may begin inside a unit)
    c.per = (c.cap + c.unit - 1) / c.unit + 1 + c.lead;
    c.n_seg = (uint32_t)n_seg;
    // Two work-groups per CU; one of up to 16 rows over 16-bit pages, bound by the memory alone (48 sequences at 6000, 32
    // heads on 8 of 128: one 215 us, two 228, three 223; one sequence at 8000, 24 heads on 4 of 256: 17.7 and 19.0; but f32
    // pages, 64 rows at 4001: 131 and 101). Chunks at heads of 64 fit three: prompts 3 x 3500 of 16 heads 152 us with two,
    // 148 with three, 512 rows at 8000 of 16 heads 45 and 45, 128 rows at 4000 of 16 heads on 4 23.7 and 25.3. No more than
    // there can be units.
    const uint32_t per_cu = !c.many && c.R == 16 && kv->type != AQ_TYPE_F32 ? 1 : 2;
    const uint32_t most = (uint32_t)compute_units(device) * per_cu;
    const double units = (double)n_seg * kv->n_head_kv * c.per;
    const uint32_t shares = units < most ? (uint32_t)units : most;
    c.shares = shares > 8 ? (shares + 7) / 8 * 8 : std::max(shares, 1u);
    c.space = paged_space(c.shares, c.n_seg, (size_t)c.R, (size_t)c.D);
    return c;
}

int choose(const char *call, const aq_paged_kv *kv, const aq_paged_batch *b, uint32_t n_head, bool f32_rows, int device,
           Choice *c) {
    const bool many = !f32_rows && takes_chunks(kv, b, n_head);
    *c = on_tiles(kv, b, n_head, many, many ? CHUNK_ROWS : longest_rows(kv, b, n_head) <= 16 ? 16 : 32, device);
    const uint64_t segs = (uint64_t)c->n_seg * kv->n_head_kv, cus = (uint64_t)compute_units(device);
    if ((double)segs * c->per >= 2147483648.0)
        return fail(AQ_EUNSUP, std::string(call) + ": batch of more than 2^31 units of work");
    // Short contexts: a share to each segment, and no join, whose launch costs as much as three or four units. Line and whole
    // segments (us): one sequence of 32 heads on 8 of 128 (bf16) at 150: 11.2 and 8.4, at 300: 11.2 and 10.1, at 500: 11.3
    // and 11.5; 64 of them at 150: 27.5 and 16.6, at 300: 37.2 and 26.2, at 500: 44.6 and 43.9, at 800: 59.0 and 65.0; 24
    // heads on 4 of 256 (f16), one at 150: 12.1 and 11.0, at 300: 13.2 and 13.5. Not where two waves share a unit (32 rows
    // of 256 at 150: 14.3 and 18.2), nor with more segments than measured, eight a CU (128 sequences of 16 heads of 80 at
    // 130: 74.3 and 35.7, of 64 at 285: 94.0 and 43.8).
    if (!c->many && !c->planned && few_groups(kv->type, c->D, c->R) == 1 && segs <= 8 * cus &&
        c->cap <= (c->D == 256 ? 256u : segs >= cus ? 512u : 384u)) {
        c->whole = c->per;
        c->shares = (uint32_t)(segs > 8 ? (segs + 7) / 8 * 8 : segs);
    }
    c->join = !c->whole && c->cap > c->unit; // else no segment has a second unit
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
    AQ_REQUIRE((uint64_t)batch->n_rows * (n_head / kv->n_head_kv) <= (1ull << 31) - 1024,
               std::string(call) + ": batch size (rows of a K/V head)");
    return 0;
}

} // namespace

int launch_paged_plan(const AttnPagedArgs &a, int R, uint32_t tk, hipStream_t stream) {
    plan_kernel<<<1, 1024, 0, stream>>>(a, R, tk);
    AQ_HIP(hipGetLastError());
    return 0;
}

int launch_paged_combine(const AttnPagedArgs &a, int R, int D, int rows, hipStream_t stream) {
    switch (a.q.type) {
    case AQ_TYPE_F32: join_pick<AQ_TYPE_F32>(a, R, D, rows, stream); break;
    case AQ_TYPE_F16: join_pick<AQ_TYPE_F16>(a, R, D, rows, stream); break;
    default: join_pick<AQ_TYPE_BF16>(a, R, D, rows, stream); break;
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
    // Enough for either type of rows, and for every batch within these bounds: one with shorter sequences may take smaller
    // row tiles, of which there are more.
    Choice c;
    rc = choose("aq_paged_attention_workspace", kv, batch, n_head, true, ctx->device, &c);
    if (rc && kv->type != AQ_TYPE_F32) rc = choose("aq_paged_attention_workspace", kv, batch, n_head, false, ctx->device, &c);
    if (rc) return rc;
    size_t most = on_tiles(kv, batch, n_head, false, 16, ctx->device).space.bytes;
    if (longest_rows(kv, batch, n_head) > 16)
        most = std::max(most, on_tiles(kv, batch, n_head, false, 32, ctx->device).space.bytes);
    if (kv->type != AQ_TYPE_F32 && takes_chunks(kv, batch, n_head))
        most = std::max(most, on_tiles(kv, batch, n_head, true, CHUNK_ROWS, ctx->device).space.bytes);
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
    auto apart = [&](const aq_heads *x) { // each output where its own input is, or in memory of its own
        return out->data != x->data || ((rows <= 1 || out->row_stride == x->row_stride) &&
                                        (n_head <= 1 || out->head_stride == x->head_stride));
    };
    AQ_REQUIRE(apart(q) && (!gate || apart(gate)), "aq_paged_attention: in place needs the same strides");
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
    a.by_g = FastDiv((uint32_t)a.G);
    a.window = window;
    a.cap = c.cap;
    a.scale_log2 = scale * 1.44269504088896340736f;
    a.q_wide = heads_aligned(q, rows, n_head);
    a.out_wide = heads_aligned(out, rows, n_head) && (!gate || heads_aligned(gate, rows, n_head));
    a.shares = c.shares;
    a.min_chunk = c.min_chunk;
    a.lead = c.lead;
    a.whole = c.whole;
    a.n_seg = c.n_seg;
    a.planned = c.planned;
    char *ws = (char *)workspace;
    a.plan = (uint32_t *)(ws + c.space.plan);
    a.tiles = (RowTile *)(ws + c.space.seg);
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
    } else if (kv->type == AQ_TYPE_F32) {
        rc = launch_paged_few_f32(a, c.D, c.R, st);
    } else if (kv->type == AQ_TYPE_F16) {
        rc = launch_paged_few_f16(a, c.D, c.R, st);
    } else {
        rc = launch_paged_few_bf16(a, c.D, c.R, st);
    }
    if (rc || !c.join) return rc;
    return launch_paged_combine(a, c.R, c.D, (int)std::min<uint64_t>((uint64_t)c.R, (uint64_t)batch->max_rows * a.G), st);
}

} // extern "C"
