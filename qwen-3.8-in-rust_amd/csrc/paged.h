// paged.h — the paged K/V cache and the batch over it as the kernels see them, and the host checks the paged entry
// points share (rope.hip: rotation and append; paged_attention.hip: attention).
#pragma once

#include "aq_common.h"

namespace aq {

// n / d for n < 2^31: m = ceil(2^(31 + k) / d) with 2^(k-1) < d <= 2^k exceeds 2^(31+k) / d by less than 1, so
// floor(n m / 2^(31+k)) is exact.
struct FastDiv {
    uint32_t d = 1, mul = 1u << 31, shift = 0;
    FastDiv() = default;
    explicit FastDiv(uint32_t div) : d(div) {
        while ((1ull << shift) < div) shift++;
        mul = (uint32_t)(((1ull << (31 + shift)) + div - 1) / div);
    }
    __host__ __device__ uint32_t quot(uint32_t n) const { return (uint32_t)(((uint64_t)n * mul) >> 31) >> shift; }
};

// The cache: K and V rows at base + ((page * page_units + slot * slot_units) << unit_shift) bytes, then the head.
// Offsets are counted in the largest power of two of bytes that divides both strides, so that 32 bits of it reach any
// pool a device can hold.
struct PagedKv {
    const char *k = nullptr, *v = nullptr;
    uint32_t n_pages = 0, page_units = 0, slot_units = 0, unit_shift = 0;
    uint64_t head_bytes = 0;
    FastDiv page_size;
    int nkv = 0, hd = 0, type = 0;
};

struct PagedBatch {
    const int32_t *row_start = nullptr, *kv_len = nullptr, *pages = nullptr;
    uint32_t n_seq = 0, max_pages = 0, n_rows = 0;
};

// [rows][heads][head_dim] values with strides, in elements.
struct HeadsView {
    char *p = nullptr;
    int64_t row = 0, head = 0;
    int type = 0;
};

inline size_t type_bytes(int t) { return t == AQ_TYPE_F32 ? 4 : 2; }
inline bool row_type(int t) { return t == AQ_TYPE_F32 || t == AQ_TYPE_F16 || t == AQ_TYPE_BF16; }

// The host checks; each names the call in its message.
int check_heads(const char *call, const char *what, const aq_heads *h, size_t n_rows, size_t n_heads, size_t head_dim);
int check_paged(const char *call, const aq_paged_kv *kv, const aq_paged_batch *b, PagedKv *out, PagedBatch *bout);
inline HeadsView heads_view(const aq_heads *h) {
    HeadsView v;
    v.p = (char *)h->data;
    v.row = h->row_stride;
    v.head = h->head_stride;
    v.type = h->type;
    return v;
}
// Whether every row of the view can be read and written 16 bytes at a time.
bool heads_aligned(const aq_heads *h, size_t n_rows, size_t n_heads);

// ------------------------------------------------------------------------------------------------ device side
template <int T> struct RowType;
template <> struct RowType<AQ_TYPE_F32> { using type = float; };
template <> struct RowType<AQ_TYPE_F16> { using type = _Float16; };
template <> struct RowType<AQ_TYPE_BF16> { using type = __bf16; };

// Byte offset (in units) of a position's K / V row and whether it has one: a position past the table or on a page
// outside 0..n_pages-1 has none. In two steps, so that the page's load need not be waited for at once.
__device__ __forceinline__ uint32_t paged_entry(const PagedKv &c, const int32_t *table, uint32_t max_pages, uint32_t pos) {
    const uint32_t col = c.page_size.quot(pos);
    return col < max_pages ? (uint32_t)table[col] : 0xFFFFFFFFu;
}
__device__ __forceinline__ bool paged_units(const PagedKv &c, uint32_t entry, uint32_t pos, uint32_t *units) {
    const uint32_t slot = pos - c.page_size.quot(pos) * c.page_size.d;
    const bool ok = entry < c.n_pages;
    *units = ok ? entry * c.page_units + slot * c.slot_units : 0u;
    return ok;
}
__device__ __forceinline__ bool paged_slot(const PagedKv &c, const int32_t *table, uint32_t max_pages, uint32_t pos,
                                           uint32_t *units) {
    return paged_units(c, paged_entry(c, table, max_pages, pos), pos, units);
}

// The sequence that row `row` belongs to, if any: the number of sequences that end at or before it (n_seq: all do). A row
// before the first one's row_start is in none all the same, which the caller looks at. row_start never falls, so the whole
// wave looks at the ends of 64 blocks of sequences, then inside the first that ends after the row.
__device__ __forceinline__ uint32_t paged_seq_of(const PagedBatch &b, uint32_t row) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t lo = 0, hi = b.n_seq; // the answer is one of lo .. hi
    while (lo < hi) {
        const uint32_t step = (hi - lo + 63) / 64, s = lo + lane * step;
        const bool before = s < hi && b.row_start[min(s + step, hi)] <= (int32_t)row;
        lo = min(lo + (uint32_t)__popcll(__ballot(before)) * step, hi);
        hi = min(lo + step - 1, hi);
    }
    return lo;
}

// A sequence's rows within the tensors' n_rows, whatever row_start holds, and the position of the first of them: a sequence
// that begins before the tensors or ends past them keeps its other rows' positions.
struct SeqRows {
    int32_t first, n, base;
};
__device__ __forceinline__ SeqRows paged_seq(const PagedBatch &b, uint32_t s) {
    const int32_t lo = b.row_start[s], hi = b.row_start[s + 1], len = b.kv_len[s];
    SeqRows r;
    r.first = lo < 0 ? 0 : lo;
    const int32_t end = hi < (int32_t)b.n_rows ? hi : (int32_t)b.n_rows;
    r.n = end > r.first ? end - r.first : 0;
    r.base = (len > 0 ? len : 0) - (hi > r.first ? hi - r.first : 0);
    return r;
}

} // namespace aq
