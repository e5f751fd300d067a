// rope.hip — rotary positions over rows of heads (aq_rope_*), and new K/V rows written into pages with the rotation on
// the way (aq_paged_append).
//
// A pair (a, b) of a head at position p turns by p * f: (a cos - b sin, b cos + a sin). The angle is counted in turns in
// 64 bits (p up to 2^31 times f <= 1 / 2 pi leaves 2^-24 of a turn), cut to one turn, and only then taken in 32 bits:
// f32 angles lose 2^-7 of a radian at position 200,000. One thread computes the pairs of one 16-byte unit once and
// applies them to several heads of the row, so the 64-bit work (a product, a floor, a difference per pair) stays
// below the memory time from four heads on.
//
// Bound by their bytes: 8191 rows of 40 heads of 128 (bf16) 34.1 us, 4.9 TB/s where a copy reaches 5.3; 5342 new rows of 24
// query and 4 K/V heads of 256 (f32 into f16) appended in 65.5 us, 5.0 TB/s; 48 single tokens 5.2 us, an empty launch 2.4.
#include <cmath>
#include <memory>
#include <new>

#include "paged.h"

struct aq_rope {
    aq_ctx *ctx = nullptr;
    uint32_t dim = 0, layout = 0;
    float gain = 1.0f;
    double *freq = nullptr; // dim / 2 turns per position
};

namespace aq {

int check_heads(const char *call, const char *what, const aq_heads *h, size_t n_rows, size_t n_heads, size_t head_dim) {
    auto who = [&] { return std::string(call) + ": " + what; };
    AQ_REQUIRE(h && (h->data || n_rows == 0), who() + ": null");
    AQ_REQUIRE(row_type(h->type), who() + ": type " + std::to_string(h->type) + " is not F32, F16 or BF16");
    AQ_REQUIRE((uintptr_t)h->data % type_bytes(h->type) == 0, who() + ": data is not aligned to its type");
    AQ_REQUIRE(h->row_stride >= 0 && h->head_stride >= 0 && h->row_stride < ((int64_t)1 << 40) &&
                   h->head_stride < ((int64_t)1 << 40),
               who() + ": strides");
    AQ_REQUIRE(n_heads <= 1 || h->head_stride >= (int64_t)head_dim, who() + ": heads overlap");
    AQ_REQUIRE(n_rows <= 1 || h->row_stride >= (int64_t)head_dim, who() + ": rows overlap");
    return 0;
}

bool heads_aligned(const aq_heads *h, size_t n_rows, size_t n_heads) {
    const size_t v = 16 / type_bytes(h->type);
    return (uintptr_t)h->data % 16 == 0 && (n_rows <= 1 || h->row_stride % v == 0) &&
           (n_heads <= 1 || h->head_stride % v == 0);
}

int check_paged(const char *call, const aq_paged_kv *kv, const aq_paged_batch *b, PagedKv *out, PagedBatch *bout) {
    auto who = [&] { return std::string(call); };
    AQ_REQUIRE(kv && b, who() + ": null argument");
    AQ_REQUIRE(kv->k && kv->v, who() + ": null k or v pages");
    AQ_REQUIRE(row_type(kv->type), who() + ": cache type " + std::to_string(kv->type) + " is not F32, F16 or BF16");
    AQ_REQUIRE(kv->n_pages > 0 && kv->n_pages < (1u << 31) && kv->page_size > 0 && kv->page_size < (1u << 31),
               who() + ": pages");
    AQ_REQUIRE(kv->n_head_kv > 0 && kv->n_head_kv <= 65535, who() + ": n_head_kv");
    if (kv->head_dim == 0 || kv->head_dim > 256 || kv->head_dim % 8)
        return fail(AQ_EUNSUP, who() + ": head_dim " + std::to_string(kv->head_dim) + " (a multiple of 8, at most 256)");
    const int64_t tb = (int64_t)type_bytes(kv->type), lim = (int64_t)1 << 40;
    AQ_REQUIRE((uintptr_t)kv->k % 16 == 0 && (uintptr_t)kv->v % 16 == 0, who() + ": pages are not 16-byte aligned");
    const int64_t st[3] = {kv->page_stride, kv->slot_stride, kv->head_stride};
    for (int i = 0; i < 3; i++)
        AQ_REQUIRE(st[i] >= 0 && st[i] < lim && st[i] * tb % 16 == 0, who() + ": page strides (multiples of 16 bytes)");
    AQ_REQUIRE(kv->n_head_kv == 1 || kv->head_stride >= (int64_t)kv->head_dim, who() + ": heads of a page overlap");
    AQ_REQUIRE(kv->page_size == 1 || kv->slot_stride >= (int64_t)kv->head_dim, who() + ": slots of a page overlap");
    AQ_REQUIRE(kv->n_pages == 1 || kv->page_stride >= (int64_t)kv->head_dim, who() + ": pages overlap");
    const uint64_t pb = kv->n_pages > 1 ? (uint64_t)kv->page_stride * tb : 0,
                   sb = kv->page_size > 1 ? (uint64_t)kv->slot_stride * tb : 0;
    uint32_t sh = 4;
    while (sh < 40 && (pb | sb) && !(((pb | sb) >> sh) & 1)) sh++;
    const uint64_t pu = pb >> sh, su = sb >> sh;
    const double reach = (double)(kv->n_pages - 1) * (double)pu + (double)(kv->page_size - 1) * (double)su;
    if (reach >= 4294967295.0)
        return fail(AQ_EUNSUP, who() + ": the pool reaches past 2^32 units of " + std::to_string(1ull << sh) + " bytes");
    AQ_REQUIRE(b->n_rows < (1u << 24) && b->n_seq < (1u << 24), who() + ": batch size (fewer than 2^24 rows)");
    AQ_REQUIRE(b->n_seq == 0 || (b->row_start && b->kv_len && b->pages), who() + ": null batch array");
    AQ_REQUIRE(b->n_seq == 0 || b->max_pages > 0, who() + ": max_pages");
    AQ_REQUIRE((uint64_t)b->max_pages * kv->page_size <= (1ull << 31) - 1024,
               who() + ": the page table reaches past 2^31 positions");
    if (out) {
        out->k = (const char *)kv->k;
        out->v = (const char *)kv->v;
        out->n_pages = kv->n_pages;
        out->page_units = (uint32_t)pu;
        out->slot_units = (uint32_t)su;
        out->unit_shift = sh;
        out->head_bytes = (uint64_t)kv->head_stride * tb;
        out->page_size = FastDiv(kv->page_size);
        out->nkv = (int)kv->n_head_kv;
        out->hd = (int)kv->head_dim;
        out->type = kv->type;
    }
    if (bout) {
        bout->row_start = b->row_start;
        bout->kv_len = b->kv_len;
        bout->pages = b->pages;
        bout->n_seq = b->n_seq;
        bout->max_pages = b->max_pages;
        bout->n_rows = b->n_rows;
    }
    return 0;
}

namespace {

// N values at p as f32, and back with one rounding; 16 bytes at a time where W.
template <int T, int N, bool W>
__device__ __forceinline__ void load_n(const typename RowType<T>::type *p, float *v) {
    using E = typename RowType<T>::type;
    if constexpr (W) {
        constexpr int C = 16 / (int)sizeof(E);
        typedef E vec __attribute__((ext_vector_type(C)));
#pragma unroll
        for (int i = 0; i < N / C; i++) {
            const vec x = *reinterpret_cast<const vec *>(p + i * C);
#pragma unroll
            for (int j = 0; j < C; j++) v[i * C + j] = (float)x[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = (float)p[i];
    }
}

template <int T, int N, bool W>
__device__ __forceinline__ void store_n(typename RowType<T>::type *p, const float *v) {
    using E = typename RowType<T>::type;
    if constexpr (W) {
        constexpr int C = 16 / (int)sizeof(E);
        typedef E vec __attribute__((ext_vector_type(C)));
#pragma unroll
        for (int i = 0; i < N / C; i++) {
            vec x;
#pragma unroll
            for (int j = 0; j < C; j++) x[j] = (E)v[i * C + j];
            *reinterpret_cast<vec *>(p + i * C) = x;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) p[i] = (E)v[i];
    }
}

// The rotation of one unit: half layout VEC pairs (values u..u+VEC-1 with those dim/2 further), interleaved VEC / 2
// pairs of neighbours.
template <bool INTER, int VEC>
struct Unit {
    static constexpr int PAIRS = INTER ? VEC / 2 : VEC;
    float c[PAIRS], s[PAIRS];

    __device__ __forceinline__ void angles(const double *freq, uint32_t unit, int32_t pos, float gain, float sign) {
#pragma unroll
        for (int i = 0; i < PAIRS; i++) {
            const double t = (double)pos * freq[unit * PAIRS + i];
            float sn, cs;
            sincospif(2.0f * (float)(t - rint(t)), &sn, &cs);
            c[i] = cs * gain;
            s[i] = sn * gain * sign;
        }
    }
    // v: half layout the VEC first values, then the VEC second ones
    __device__ __forceinline__ void turn(float *v) const {
#pragma unroll
        for (int i = 0; i < PAIRS; i++) {
            const int ia = INTER ? 2 * i : i, ib = INTER ? 2 * i + 1 : VEC + i;
            const float a = v[ia], b = v[ib];
            v[ia] = fmaf(a, c[i], -(b * s[i]));
            v[ib] = fmaf(b, c[i], a * s[i]);
        }
    }
};

constexpr int HB = 4; // heads in flight in a thread's registers

// Heads h0 .. h1-1 of one row, one unit: rotated (rot) or copied. from / to: the row's head 0.
template <int TI, int TO, bool INTER, int VEC, bool W>
__device__ __forceinline__ void move_heads(const typename RowType<TI>::type *from, int64_t from_head,
                                           typename RowType<TO>::type *to, int64_t to_head, int h0, int h1, bool rot,
                                           uint32_t unit, uint32_t dim, uint32_t rot_units, const Unit<INTER, VEC> &u) {
    constexpr int N = INTER ? VEC : 2 * VEC; // values of a rotated unit
    const uint32_t at = rot ? unit * VEC : dim + (unit - rot_units) * VEC;
    for (int h = h0; h < h1; h += HB) {
        float v[HB][N];
#pragma unroll
        for (int i = 0; i < HB; i++) {
            if (h + i < h1) {
                const auto *p = from + (h + i) * from_head + at;
                load_n<TI, VEC, W>(p, v[i]);
                if (!INTER && rot) load_n<TI, VEC, W>(p + dim / 2, v[i] + N - VEC);
            }
        }
#pragma unroll
        for (int i = 0; i < HB; i++) {
            if (h + i < h1) {
                auto *p = to + (h + i) * to_head + at;
                if (rot) u.turn(v[i]);
                store_n<TO, VEC, W>(p, v[i]);
                if (!INTER && rot) store_n<TO, VEC, W>(p + dim / 2, v[i] + N - VEC);
            }
        }
    }
}

struct RopeArgs {
    HeadsView x, y;
    const double *freq;
    const int32_t *pos;
    uint32_t n_rows, n_heads, dim, rot_units, units, heads_per, items;
    FastDiv unit_div, item_div;
    float gain, sign;
};

// One (row, head group, unit) item per thread, in that order, 64 bytes or more in flight each. Items run on from row to row:
// with a row's items to a work-group, 80 items left most of its lanes idle (8191 rows of 40 heads of 128: 40.8 us for 34.1).
template <int T, bool INTER, int VEC, bool W>
__global__ void __launch_bounds__(256) rope_kernel(RopeArgs a) {
    using E = typename RowType<T>::type;
    const uint32_t at = blockIdx.x * 256u + threadIdx.x, row = a.item_div.quot(at), item = at - row * a.items;
    if (row >= a.n_rows) return;
    const uint32_t grp = a.unit_div.quot(item), unit = item - grp * a.units;
    const bool rot = unit < a.rot_units;
    Unit<INTER, VEC> u;
    if (rot) u.angles(a.freq, unit, a.pos[row], a.gain, a.sign);
    const int h0 = (int)(grp * a.heads_per), h1 = min(h0 + (int)a.heads_per, (int)a.n_heads);
    move_heads<T, T, INTER, VEC, W>((const E *)a.x.p + row * a.x.row, a.x.head, (E *)a.y.p + row * a.y.row, a.y.head, h0,
                                    h1, rot, unit, a.dim, a.rot_units, u);
}

struct AppendArgs {
    PagedKv kv;
    PagedBatch b;
    HeadsView k, v, q, qo;
    const double *freq;
    uint32_t dim, rot_units, units, vunits, heads_per, n_head;
    uint32_t qk_items, items, q_groups; // (query groups + key groups) * units, and the value groups' after them
    FastDiv unit_div, vunit_div;
    float gain;
};

// One row per wave at least (row = blockIdx.x; its (head group, unit) items over blockIdx.y and the threads), so the
// sequence is found by the wave together: the row's page is two dependent loads away from it.
template <int TI, int TO, bool INTER, int VEC, bool W>
__global__ void __launch_bounds__(256) append_kernel(AppendArgs a) {
    using EI = typename RowType<TI>::type;
    using EO = typename RowType<TO>::type;
    const uint32_t row = blockIdx.x, item = blockIdx.y * blockDim.x + threadIdx.x;
    const uint32_t seq = paged_seq_of(a.b, row);
    if (seq >= a.b.n_seq || row >= a.b.n_rows || item >= a.items) return;
    const SeqRows sr = paged_seq(a.b, seq);
    if ((int32_t)row < sr.first) return; // before the first sequence's rows
    const int32_t pos = sr.base + ((int32_t)row - sr.first);
    const bool isv = item >= a.qk_items;
    const uint32_t it = isv ? item - a.qk_items : item;
    const uint32_t grp = isv ? a.vunit_div.quot(it) : a.unit_div.quot(it);
    const uint32_t unit = it - grp * (isv ? a.vunits : a.units);
    const bool isq = !isv && grp < a.q_groups;
    const bool rot = !isv && unit < a.rot_units;
    Unit<INTER, VEC> u;
    if (rot) u.angles(a.freq, unit, pos, a.gain, 1.0f);
    const int h0 = (int)((isq || isv ? grp : grp - a.q_groups) * a.heads_per);
    if (isq) {
        move_heads<TI, TI, INTER, VEC, W>((const EI *)a.q.p + row * a.q.row, a.q.head, (EI *)a.qo.p + row * a.qo.row,
                                          a.qo.head, h0, min(h0 + (int)a.heads_per, (int)a.n_head), rot, unit, a.dim,
                                          a.rot_units, u);
        return;
    }
    uint32_t off;
    if (pos < 0 || !paged_slot(a.kv, a.b.pages + (size_t)seq * a.b.max_pages, a.b.max_pages, (uint32_t)pos, &off)) return;
    const HeadsView &src = isv ? a.v : a.k;
    char *dst = const_cast<char *>(isv ? a.kv.v : a.kv.k) + ((uint64_t)off << a.kv.unit_shift);
    move_heads<TI, TO, INTER, VEC, W>((const EI *)src.p + row * src.row, src.head, (EO *)dst,
                                      (int64_t)(a.kv.head_bytes / sizeof(EO)), h0,
                                      min(h0 + (int)a.heads_per, a.kv.nkv), rot, unit, isv ? 0u : a.dim,
                                      isv ? 0u : a.rot_units, u);
}

// How a head divides into units: `vec` values each (half layout: of either half), then the values that pass through.
void unit_shape(uint32_t layout, uint32_t dim, uint32_t hd, uint32_t vec, uint32_t *rot, uint32_t *all) {
    *rot = layout == AQ_ROPE_INTERLEAVED ? dim / vec : dim / 2 / vec;
    *all = *rot + (hd - dim) / vec;
}
bool wide_fits(uint32_t layout, uint32_t dim, uint32_t hd, uint32_t vec) {
    return hd % vec == 0 && dim % vec == 0 && (layout == AQ_ROPE_INTERLEAVED || (dim / 2) % vec == 0);
}

template <int T, bool INTER, bool W>
int rope_launch(const RopeArgs &a, dim3 grid, hipStream_t stream) {
    constexpr int VEC = W ? 16 / (int)sizeof(typename RowType<T>::type) : (INTER ? 2 : 1);
    rope_kernel<T, INTER, VEC, W><<<grid, 256, 0, stream>>>(a);
    AQ_HIP(hipGetLastError());
    return 0;
}
template <int T>
int rope_pick(const RopeArgs &a, bool inter, bool wide, dim3 grid, hipStream_t stream) {
    if (inter) return wide ? rope_launch<T, true, true>(a, grid, stream) : rope_launch<T, true, false>(a, grid, stream);
    return wide ? rope_launch<T, false, true>(a, grid, stream) : rope_launch<T, false, false>(a, grid, stream);
}

template <int TI, int TO, bool INTER, bool W>
int append_launch(const AppendArgs &a, dim3 grid, uint32_t threads, hipStream_t stream) {
    constexpr int VEC = W ? (TI == AQ_TYPE_F32 && TO == AQ_TYPE_F32 ? 4 : 8) : (INTER ? 2 : 1);
    append_kernel<TI, TO, INTER, VEC, W><<<grid, threads, 0, stream>>>(a);
    AQ_HIP(hipGetLastError());
    return 0;
}
template <int TI, int TO>
int append_pick(const AppendArgs &a, bool inter, bool wide, dim3 grid, uint32_t threads, hipStream_t stream) {
    if (inter)
        return wide ? append_launch<TI, TO, true, true>(a, grid, threads, stream)
                    : append_launch<TI, TO, true, false>(a, grid, threads, stream);
    return wide ? append_launch<TI, TO, false, true>(a, grid, threads, stream)
                : append_launch<TI, TO, false, false>(a, grid, threads, stream);
}

// Heads a thread carries through one set of angles. One where the launch has too few threads to fill the chip
// otherwise, else eight (the angles of a unit cost as much as four heads of it).
uint32_t heads_per_thread(uint64_t unit_heads) { return unit_heads <= (1u << 18) ? 1u : 8u; }

} // namespace
} // namespace aq

using namespace aq;

extern "C" {

int aq_rope_new(aq_ctx *ctx, const aq_rope_config *c, aq_rope **out) {
    AQ_REQUIRE(ctx && c && out, "aq_rope_new: null argument");
    AQ_REQUIRE(c->dim >= 2 && c->dim % 2 == 0 && c->dim <= 65536, "aq_rope_new: dim " + std::to_string(c->dim));
    AQ_REQUIRE(c->layout <= AQ_ROPE_INTERLEAVED, "aq_rope_new: layout " + std::to_string(c->layout));
    AQ_REQUIRE(c->scaling <= AQ_ROPE_YARN, "aq_rope_new: scaling " + std::to_string(c->scaling));
    AQ_REQUIRE(std::isfinite(c->theta) && c->theta >= 1.0f, "aq_rope_new: theta");
    AQ_REQUIRE(c->scaling == AQ_ROPE_PLAIN || (std::isfinite(c->factor) && c->factor >= 0.0009765625f), "aq_rope_new: factor");
    const double fast = c->beta_fast == 0.0f ? 32.0 : c->beta_fast, slow = c->beta_slow == 0.0f ? 1.0 : c->beta_slow;
    float gain = 1.0f;
    const double two_pi = 6.283185307179586476925;
    const uint32_t half = c->dim / 2;
    double lo = 0, hi = 0;
    if (c->scaling == AQ_ROPE_YARN) {
        AQ_REQUIRE(c->theta > 1.0f && c->orig_ctx > 0, "aq_rope_new: YARN needs theta > 1 and orig_ctx");
        AQ_REQUIRE(std::isfinite(fast) && std::isfinite(slow) && fast > 0 && slow > 0 && fast >= slow,
                   "aq_rope_new: beta_fast, beta_slow");
        AQ_REQUIRE(std::isfinite(c->attn_factor) && c->attn_factor >= 0.0f, "aq_rope_new: attn_factor");
        // the pair that makes `turns` turns over orig_ctx positions
        auto index = [&](double turns) {
            return c->dim * std::log(c->orig_ctx / (turns * two_pi)) / (2 * std::log((double)c->theta));
        };
        lo = std::fmax(std::floor(index(fast)), 0.0);
        hi = std::fmin(std::ceil(index(slow)), (double)c->dim - 1);
        gain = c->attn_factor > 0 ? c->attn_factor
                                  : (c->factor <= 1.0f ? 1.0f : (float)(0.1 * std::log((double)c->factor) + 1.0));
    }
    std::unique_ptr<double[]> f(new (std::nothrow) double[half]);
    if (!f) return fail(AQ_ENOMEM, "aq_rope_new: host memory");
    for (uint32_t i = 0; i < half; i++) {
        f[i] = std::pow((double)c->theta, -2.0 * i / c->dim);
        if (c->scaling == AQ_ROPE_LINEAR) f[i] /= (double)c->factor;
        if (c->scaling == AQ_ROPE_YARN) {
            const double slowed = std::fmin(std::fmax((i - lo) / std::fmax(hi - lo, 1e-3), 0.0), 1.0);
            f[i] = f[i] / (double)c->factor * slowed + f[i] * (1.0 - slowed);
        }
        f[i] /= two_pi;
    }
    AQ_HIP(hipSetDevice(ctx->device));
    aq_rope *r = new (std::nothrow) aq_rope();
    if (!r) return fail(AQ_ENOMEM, "aq_rope_new: host memory");
    r->ctx = ctx;
    r->dim = c->dim;
    r->layout = c->layout;
    r->gain = gain;
    if (dev_malloc(&r->freq, half * sizeof(double)) != hipSuccess) {
        delete r;
        return fail(AQ_ENOMEM, "aq_rope_new: hipMalloc");
    }
    hipError_t e = hipMemcpyAsync(r->freq, f.get(), half * sizeof(double), hipMemcpyHostToDevice, ctx->stream);
    if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
    if (e != hipSuccess) {
        (void)hipFree(r->freq);
        delete r;
        return fail(AQ_EHIP, std::string("aq_rope_new: ") + hipGetErrorString(e));
    }
    *out = r;
    return 0;
}

int aq_rope_free(aq_rope *r) {
    if (!r) return 0;
    (void)hipFree(r->freq);
    delete r;
    return 0;
}

int aq_rope_apply(const aq_rope *r, const aq_heads *x, const aq_heads *y, size_t n_rows, size_t n_heads, size_t head_dim,
                  const int32_t *pos_dev, int inverse, void *stream) {
    AQ_REQUIRE(r, "aq_rope_apply: null rope");
    AQ_REQUIRE(n_rows < (1u << 24) && n_heads <= 65535 && head_dim <= 65536, "aq_rope_apply: size");
    if (n_rows == 0 || n_heads == 0) return 0;
    AQ_REQUIRE(head_dim >= r->dim, "aq_rope_apply: head_dim " + std::to_string(head_dim) + " is less than the rotated " +
                                       std::to_string(r->dim));
    int rc = check_heads("aq_rope_apply", "x", x, n_rows, n_heads, head_dim);
    if (!rc) rc = check_heads("aq_rope_apply", "y", y, n_rows, n_heads, head_dim);
    if (rc) return rc;
    AQ_REQUIRE(x->type == y->type, "aq_rope_apply: x and y of different types");
    AQ_REQUIRE(x->data != y->data || (x->row_stride == y->row_stride && x->head_stride == y->head_stride),
               "aq_rope_apply: in place needs the same strides");
    AQ_REQUIRE(pos_dev, "aq_rope_apply: null pos_dev");
    const uint32_t vec = 16 / (uint32_t)type_bytes(x->type);
    const bool inter = r->layout == AQ_ROPE_INTERLEAVED;
    const bool wide = heads_aligned(x, n_rows, n_heads) && heads_aligned(y, n_rows, n_heads) &&
                      wide_fits(r->layout, r->dim, (uint32_t)head_dim, vec);
    AQ_REQUIRE(wide || !inter || head_dim % 2 == 0, "aq_rope_apply: head_dim is odd");
    RopeArgs a;
    a.x = heads_view(x);
    a.y = heads_view(y);
    a.freq = r->freq;
    a.pos = pos_dev;
    a.n_rows = (uint32_t)n_rows;
    a.n_heads = (uint32_t)n_heads;
    a.dim = r->dim;
    unit_shape(r->layout, r->dim, (uint32_t)head_dim, wide ? vec : (inter ? 2 : 1), &a.rot_units, &a.units);
    if (x->data == y->data) a.units = a.rot_units; // the rest of the head stays where it is
    a.heads_per = heads_per_thread((uint64_t)n_rows * n_heads * a.units);
    const uint64_t items = (uint64_t)a.units * ((n_heads + a.heads_per - 1) / a.heads_per), all = items * n_rows;
    if (all > (1ull << 31) - 256) return fail(AQ_EUNSUP, "aq_rope_apply: more than 2^31 pieces of rows");
    a.items = (uint32_t)items;
    a.unit_div = FastDiv(a.units);
    a.item_div = FastDiv(a.items);
    a.gain = r->gain;
    a.sign = inverse ? -1.0f : 1.0f;
    const dim3 grid((uint32_t)((all + 255) / 256));
    AQ_HIP(hipSetDevice(r->ctx->device));
    const hipStream_t st = stream ? (hipStream_t)stream : r->ctx->stream;
    switch (x->type) {
    case AQ_TYPE_F32: return rope_pick<AQ_TYPE_F32>(a, inter, wide, grid, st);
    case AQ_TYPE_F16: return rope_pick<AQ_TYPE_F16>(a, inter, wide, grid, st);
    default: return rope_pick<AQ_TYPE_BF16>(a, inter, wide, grid, st);
    }
}

int aq_paged_append(aq_ctx *ctx, const aq_paged_kv *kv, const aq_paged_batch *batch, const aq_heads *k,
                    const aq_heads *v, const aq_rope *rope, const aq_heads *q, const aq_heads *q_out, uint32_t n_head,
                    void *stream) {
    AQ_REQUIRE(ctx, "aq_paged_append: null ctx");
    AppendArgs a;
    int rc = check_paged("aq_paged_append", kv, batch, &a.kv, &a.b);
    if (rc) return rc;
    const uint32_t hd = kv->head_dim, rows = batch->n_rows;
    rc = check_heads("aq_paged_append", "k", k, rows, kv->n_head_kv, hd);
    if (!rc) rc = check_heads("aq_paged_append", "v", v, rows, kv->n_head_kv, hd);
    if (rc) return rc;
    AQ_REQUIRE(k->type == v->type, "aq_paged_append: k and v of different types");
    AQ_REQUIRE(k->type == AQ_TYPE_F32 || k->type == kv->type, "aq_paged_append: rows are F32 or of the cache's type");
    AQ_REQUIRE(!q || rope, "aq_paged_append: q without a rope");
    AQ_REQUIRE(!q == !q_out, "aq_paged_append: q and q_out go together");
    if (rope) {
        AQ_REQUIRE(rope->ctx->device == ctx->device, "aq_paged_append: the rope is on another device");
        AQ_REQUIRE(rope->dim <= hd, "aq_paged_append: head_dim " + std::to_string(hd) + " is less than the rotated " +
                                        std::to_string(rope->dim));
    }
    if (q) {
        AQ_REQUIRE(n_head > 0 && n_head <= 65535, "aq_paged_append: n_head");
        rc = check_heads("aq_paged_append", "q", q, rows, n_head, hd);
        if (!rc) rc = check_heads("aq_paged_append", "q_out", q_out, rows, n_head, hd);
        if (rc) return rc;
        AQ_REQUIRE(q->type == k->type && q_out->type == k->type, "aq_paged_append: q, q_out and k of different types");
        AQ_REQUIRE(q->data != q_out->data || (q->row_stride == q_out->row_stride && q->head_stride == q_out->head_stride),
                   "aq_paged_append: in place needs the same strides");
    }
    if (rows == 0 || batch->n_seq == 0) return 0;
    const bool inter = rope && rope->layout == AQ_ROPE_INTERLEAVED;
    const uint32_t layout = inter ? AQ_ROPE_INTERLEAVED : AQ_ROPE_HALF, dim = rope ? rope->dim : 0;
    const uint32_t vec = k->type == AQ_TYPE_F32 && kv->type == AQ_TYPE_F32 ? 4 : 8;
    const bool wide = heads_aligned(k, rows, kv->n_head_kv) && heads_aligned(v, rows, kv->n_head_kv) &&
                      (!q || (heads_aligned(q, rows, n_head) && heads_aligned(q_out, rows, n_head))) &&
                      wide_fits(layout, dim, hd, vec);
    const uint32_t vu = wide ? vec : (inter ? 2 : 1);
    a.k = heads_view(k);
    a.v = heads_view(v);
    if (q) {
        a.q = heads_view(q);
        a.qo = heads_view(q_out);
    }
    a.freq = rope ? rope->freq : nullptr;
    a.gain = rope ? rope->gain : 1.0f;
    a.dim = dim;
    unit_shape(layout, dim, hd, vu, &a.rot_units, &a.units);
    a.vunits = hd / vu;
    a.n_head = q ? n_head : 0;
    a.heads_per = heads_per_thread((uint64_t)rows * (a.n_head + 2 * kv->n_head_kv) * a.vunits);
    const uint32_t kv_groups = (kv->n_head_kv + a.heads_per - 1) / a.heads_per;
    a.q_groups = (a.n_head + a.heads_per - 1) / a.heads_per;
    a.qk_items = (a.q_groups + kv_groups) * a.units;
    a.items = a.qk_items + kv_groups * a.vunits;
    a.unit_div = FastDiv(a.units);
    a.vunit_div = FastDiv(a.vunits);
    uint32_t threads = 64;
    while (threads < 256 && threads < a.items) threads *= 2;
    const uint32_t gy = (a.items + threads - 1) / threads;
    AQ_REQUIRE(gy <= 65535, "aq_paged_append: size");
    const dim3 grid(rows, gy);
    AQ_HIP(hipSetDevice(ctx->device));
    const hipStream_t st = stream ? (hipStream_t)stream : ctx->stream;
    if (k->type == AQ_TYPE_F32) {
        if (kv->type == AQ_TYPE_F32) return append_pick<AQ_TYPE_F32, AQ_TYPE_F32>(a, inter, wide, grid, threads, st);
        if (kv->type == AQ_TYPE_F16) return append_pick<AQ_TYPE_F32, AQ_TYPE_F16>(a, inter, wide, grid, threads, st);
        return append_pick<AQ_TYPE_F32, AQ_TYPE_BF16>(a, inter, wide, grid, threads, st);
    }
    if (kv->type == AQ_TYPE_F16) return append_pick<AQ_TYPE_F16, AQ_TYPE_F16>(a, inter, wide, grid, threads, st);
    return append_pick<AQ_TYPE_BF16, AQ_TYPE_BF16>(a, inter, wide, grid, threads, st);
}

} // extern "C"
