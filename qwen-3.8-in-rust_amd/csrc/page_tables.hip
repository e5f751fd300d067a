// page_tables.hip — the page tables of a step of a batch of sequences, on the device (aq_paged_tables), and the accepted path
// of a tree of drafts kept in the pages (aq_paged_tree_commit).
//
// Tables. A sequence that will have n positions wants ceil(n / page_size) pages. What it lacks it takes from the front of a
// ring of free pages, what it has too many it puts at the ring's end, and each knows its place in the ring from the sums over
// the sequences before it: the same call gives the same tables. Pages put back are for the next call, so that what is read
// (the ring's free pages, the tables' held entries) and what is written (the ring behind them, the entries past them) are
// apart, and every work-group can work all of it out by itself: each scans the sequences, 256 or 1024 at a time, then
// takes every so many of the rows, of the pages taken and of those put back. Only the lengths, the counts and the ring's state
// may be written over what the others still read: then the last work-group to arrive at a counter writes those. Bound by
// latency: lengths, scan, search, page entry, store. One row each of 48 requests 5.3 us, 50,044 rows of 700 requests 10.5, where
// an empty launch takes 2.4. In place a step that takes pages and one that puts them back, in turn, 6.4 and 18.6 us a call for
// 5.1 and 8.9 into other arrays: the counter, and 64 work-groups for 97.
//
// Commit. A path's rows rise, so its e-th row lies at or past place e, and moved in order none overwrites one that is still
// to move. A work-group has one sequence's K or V rows in one cache: its lanes find 64 entries' places at a time, then each
// thread moves its 16 bytes of a row for entry after entry, eight on their way. Bound by latency: lengths, path, page entries,
// rows. Paths of 48 trees of 8 in 16 caches (8 heads of 128, bf16), 24 MB: 6.6 us, of one of 5 (4 heads of 256, f16) 3.6.
#include <algorithm>
#include <climits>
#include <memory>
#include <new>

#include "paged.h"

namespace aq {
namespace {

struct TablesArgs {
    const int32_t *before, *fresh, *held, *state, *depth;
    int32_t *pages, *ring, *held_out, *state_out, *row_start, *kv_len, *missing, *pos;
    int64_t *slots;
    uint32_t n_seq, max_pages, n_pages, n_rows;
    uint32_t apart; // no output lies where an input does
    FastDiv page_size;
};

// Of a chunk of sequences: the sums of rows, of pages taken and of pages put back before each, and what each has and wants.
template <uint32_t SCAN>
struct TablesLds {
    uint32_t rows[SCAN + 1], take[SCAN + 1], back[SCAN + 1], held[SCAN], want[SCAN], wsum[3][8], taken, last;
    int32_t before[SCAN];
};

// One sequence: its new rows, the pages it holds, those it needs and those of them that its table has room for.
struct Request {
    uint32_t rows, held, want, need;
    int32_t before, len;
};
__device__ __forceinline__ Request request(const TablesArgs &a, uint32_t s) {
    Request r = {0, 0, 0, 0, 0, 0};
    if (s >= a.n_seq) return r;
    const int32_t fresh = a.fresh[s], before = a.before[s], held = a.held[s];
    r.held = (uint32_t)min(max(held, 0), (int32_t)a.max_pages);
    if (fresh < 0) return r; // ended: it needs nothing
    r.before = max(before, 0);
    r.rows = (uint32_t)fresh;
    r.len = (int32_t)min((uint32_t)r.before + r.rows, (uint32_t)INT_MAX);
    r.need = a.page_size.quot((uint32_t)r.len);
    r.need += r.need * a.page_size.d < (uint32_t)r.len;
    r.want = min(r.need, a.max_pages);
    return r;
}
__device__ __forceinline__ uint32_t over(uint32_t x, uint32_t y) { return x > y ? x - y : 0u; }
// Sums of rows stop at 2^32 - 1 (those of pages are at most the tables' entries, fewer than 2^32).
__device__ __forceinline__ uint32_t plus(uint32_t x, uint32_t y) { return __builtin_elementwise_add_sat(x, y); }

// PER: sequences a thread scans at a time.
template <uint32_t PER, uint32_t THREADS>
__global__ void __launch_bounds__(THREADS) tables_kernel(TablesArgs a) {
    constexpr uint32_t SCAN = PER * THREADS;
    __shared__ TablesLds<SCAN> lds;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int32_t state0 = a.state[0], state1 = a.state[1];
    const uint32_t me = blockIdx.x * THREADS + tid, all = gridDim.x * THREADS;

    // The chunk of sequences from s0 on, onto the sums of those before it.
    uint32_t sums0[3] = {0, 0, 0};
    Request r[PER];
    auto scan = [&](uint32_t s0) {
        uint32_t sum[3] = {0, 0, 0}, in[3];
#pragma unroll
        for (uint32_t i = 0; i < PER; i++) {
            r[i] = request(a, s0 + tid * PER + i);
            sum[0] = plus(sum[0], r[i].rows);
            sum[1] += over(r[i].want, r[i].held);
            sum[2] += over(r[i].held, r[i].want);
        }
#pragma unroll
        for (int k = 0; k < 3; k++) in[k] = sum[k];
#pragma unroll
        for (uint32_t d = 1; d < 64; d *= 2) {
#pragma unroll
            for (int k = 0; k < 3; k++) {
                const uint32_t x = __shfl_up(in[k], d);
                if (lane >= d) in[k] = plus(in[k], x);
            }
        }
        __syncthreads(); // the chunk before is read
        if (lane == 63) {
#pragma unroll
            for (int k = 0; k < 3; k++) lds.wsum[k][wave] = in[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 3; k++) {
            uint32_t at = __shfl_up(in[k], 1); // before this thread's
            at = lane ? at : 0u;
            for (uint32_t w = 0; w < wave; w++) at = plus(at, lds.wsum[k][w]);
            in[k] = plus(at, sums0[k]);
            for (uint32_t w = 0; w < THREADS / 64; w++) sums0[k] = plus(sums0[k], lds.wsum[k][w]);
        }
#pragma unroll
        for (uint32_t i = 0; i < PER; i++) {
            const uint32_t l = tid * PER + i;
            lds.rows[l] = in[0];
            lds.take[l] = in[1];
            lds.back[l] = in[2];
            lds.before[l] = r[i].before;
            lds.held[l] = r[i].held;
            lds.want[l] = r[i].want;
            in[0] = plus(in[0], r[i].rows);
            in[1] += over(r[i].want, r[i].held);
            in[2] += over(r[i].held, r[i].want);
        }
        if (tid == THREADS - 1) {
            lds.rows[SCAN] = in[0];
            lds.take[SCAN] = in[1];
            lds.back[SCAN] = in[2];
        }
        __syncthreads();
    };
    const uint32_t first = (uint32_t)state0 % a.n_pages, count = (uint32_t)min(max(state1, 0), (int32_t)a.n_pages);
    auto ring = [&](uint32_t i) -> int32_t & { // its i-th place; past the second turn only where the counts are wrong
        uint64_t at = (uint64_t)first + i;
        if (at >= a.n_pages) at -= a.n_pages;
        if (at >= a.n_pages) at %= a.n_pages;
        return a.ring[at];
    };
    // Whether all that the chunk's sequences up to l take is there.
    auto served = [&](uint32_t l) { return lds.take[l + 1] <= count; };
    // Every so many of the chunk's rows, of the pages it takes and of those it puts back, ROWS, PAGES and PAGES of them a round:
    // all searches side by side, then all loads, then all stores, so that a round waits once for each (with the searches one
    // after the other, 700 requests of 90 rows 4 us more).
    auto items = [&](uint32_t s0, uint32_t n) {
        constexpr int ROWS = 2, PAGES = 1, ALL = ROWS + 2 * PAGES;
        const uint32_t step0 = n > 1 ? 1u << (31 - __builtin_clz(n - 1)) : 0u;
        const uint32_t row_end = min(lds.rows[SCAN], a.n_rows), take_end = lds.take[SCAN], back_end = lds.back[SCAN];
        for (uint64_t row = (uint64_t)lds.rows[0] + me, take = (uint64_t)lds.take[0] + me, back = (uint64_t)lds.back[0] + me;
             row < row_end || take < take_end || back < back_end;
             row += (uint64_t)ROWS * all, take += (uint64_t)PAGES * all, back += (uint64_t)PAGES * all) {
            // each item's sequence: the last whose sum is at or below it (past n the sums are those of all)
            auto item = [&](int i) { return i < ROWS ? row + (uint64_t)i * all
                                            : i < ROWS + PAGES ? take + (uint64_t)(i - ROWS) * all
                                                               : back + (uint64_t)(i - ROWS - PAGES) * all; };
            auto sums = [&](int i) { return i < ROWS ? lds.rows : i < ROWS + PAGES ? lds.take : lds.back; };
            uint32_t seq[ALL];
#pragma unroll
            for (int i = 0; i < ALL; i++) seq[i] = 0;
            for (uint32_t step = step0; step; step /= 2) {
#pragma unroll
                for (int i = 0; i < ALL; i++) seq[i] += sums(i)[seq[i] + step] <= item(i) ? step : 0u;
            }
            const int32_t *from[ALL];
            uint32_t at[ROWS], slot[ROWS]; // a row's position, its slot in its page
#pragma unroll
            for (int i = 0; i < ALL; i++) {
                from[i] = nullptr;
                const uint32_t l = seq[i], x = (uint32_t)item(i) - sums(i)[l], held = lds.held[l], want = lds.want[l];
                const int32_t *const table = a.pages + (size_t)(s0 + l) * a.max_pages;
                if (i < ROWS) {
                    const uint32_t p = (uint32_t)lds.before[l] + x;
                    at[i] = min(p, (uint32_t)INT_MAX);
                    const uint32_t col = a.page_size.quot(at[i]);
                    slot[i] = at[i] - col * a.page_size.d;
                    if (item(i) >= row_end) continue;
                    if (a.depth) at[i] = (uint32_t)lds.before[l] + (uint32_t)a.depth[item(i)];
                    if (a.slots && col < want && p <= INT_MAX) { // in a page held before, or taken now
                        if (col < held) from[i] = table + col;
                        else if (served(l)) from[i] = &ring(lds.take[l] + (col - held));
                    }
                } else if (i < ROWS + PAGES) {
                    if (item(i) < take_end && served(l)) from[i] = &ring((uint32_t)item(i));
                } else if (item(i) < back_end) {
                    from[i] = table + want + x;
                }
            }
            int32_t page[ALL];
#pragma unroll
            for (int i = 0; i < ALL; i++) page[i] = from[i] ? *from[i] : -1;
#pragma unroll
            for (int i = 0; i < ALL; i++) {
                if (i < ROWS) {
                    if (item(i) >= row_end) continue;
                    if (a.pos) a.pos[item(i)] = (int32_t)at[i];
                    if (a.slots)
                        a.slots[item(i)] = (uint32_t)page[i] < a.n_pages ? (int64_t)page[i] * a.page_size.d + slot[i] : -1;
                } else if (i < ROWS + PAGES) {
                    const uint32_t l = seq[i];
                    if (item(i) < take_end)
                        a.pages[(size_t)(s0 + l) * a.max_pages + lds.held[l] + ((uint32_t)item(i) - lds.take[l])] = page[i];
                } else if (item(i) < back_end) {
                    ring(count + (uint32_t)item(i)) = page[i]; // behind the pages that were free
                }
            }
        }
    };
    auto sequences = [&](uint32_t s0) {
#pragma unroll
        for (uint32_t i = 0; i < PER; i++) {
            const uint32_t l = tid * PER + i, s = s0 + l;
            if (s >= a.n_seq) continue;
            const uint32_t take = over(r[i].want, r[i].held);
            a.row_start[s] = (int32_t)min(lds.rows[l], (uint32_t)INT_MAX);
            a.kv_len[s] = r[i].len;
            a.held_out[s] = (int32_t)(served(l) ? r[i].want : min(r[i].held, r[i].want));
            if (a.missing) a.missing[s] = (int32_t)(r[i].need - r[i].want + (served(l) ? 0u : take));
            if (served(l) && take) atomicMax(&lds.taken, lds.take[l + 1]);
        }
    };
    auto state = [&] { // after the last of them
        __syncthreads();
        if (tid) return;
        const uint32_t taken = lds.taken; // at most count
        a.row_start[a.n_seq] = (int32_t)min(sums0[0], (uint32_t)INT_MAX);
        a.state_out[0] = (int32_t)(((uint64_t)first + taken) % a.n_pages);
        a.state_out[1] = (int32_t)min((uint64_t)(count - taken) + sums0[2], (uint64_t)a.n_pages);
    };

    if (tid == 0) lds.taken = 0;
    for (uint32_t s0 = 0; s0 < a.n_seq; s0 += SCAN) {
        scan(s0);
        if (a.apart ? blockIdx.x == 0 : gridDim.x == 1) sequences(s0); // nobody else reads what this writes
        items(s0, min(a.n_seq - s0, SCAN));
    }
    for (uint64_t i = (uint64_t)sums0[0] + me; i < a.n_rows; i += all) { // behind the last sequence
        if (a.pos) a.pos[i] = 0;
        if (a.slots) a.slots[i] = -1;
    }
    if (a.apart || gridDim.x == 1) {
        if (blockIdx.x == 0) state();
        return;
    }
    __threadfence(); // what was read is read; the counter ends at 0 again
    __syncthreads();
    if (tid == 0) lds.last = atomicInc((unsigned *)&a.state_out[2], gridDim.x - 1) == gridDim.x - 1;
    __syncthreads();
    if (!lds.last) return;
    __threadfence();
    if (a.n_seq <= SCAN) {
        sequences(0); // the scan is still there
    } else {
        sums0[0] = sums0[1] = sums0[2] = 0;
        for (uint32_t s0 = 0; s0 < a.n_seq; s0 += SCAN) {
            scan(s0);
            sequences(s0);
        }
    }
    state();
}

// ------------------------------------------------------------------------------------------------- the commit
constexpr uint32_t MAX_CACHES = 64; // of a launch
typedef unsigned u4 __attribute__((ext_vector_type(4)));

struct CommitArgs {
    PagedKv kv; // the shape of all; k and v unused
    PagedBatch b;
    const int32_t *path, *path_len;
    int32_t *kv_len_out;
    uint32_t max_path, chunks; // 16-byte pieces of a row of all heads
    FastDiv per_head;          // of one head's
    char *pools[2 * MAX_CACHES];
};

__global__ void __launch_bounds__(256) commit_kernel(CommitArgs a) {
    constexpr int FLIGHT = 8;
    const uint32_t seq = blockIdx.x, lane = threadIdx.x & 63;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    char *const pool = a.pools[blockIdx.y];
    const int32_t *path = a.path + (size_t)seq * a.max_path, *table = a.b.pages + (size_t)seq * a.b.max_pages;
    const SeqRows sr = paged_seq(a.b, seq);
    const int32_t base = sr.before, fresh = sr.len - base; // all of its new rows
    const uint32_t len = (uint32_t)min(max(a.path_len[seq], 0), (int32_t)min(a.max_path, (uint32_t)INT_MAX));
    int32_t before = -1;  // the entry before the 64
    uint32_t kept = 0;
    bool whole = true;
    for (uint32_t e0 = 0; e0 < len && whole; e0 += 64) { // uniform
        const uint32_t e = e0 + lane;
        const int32_t from = e < len ? path[e] : -1;
        const int32_t prev = lane ? __shfl_up(from, 1) : before;
        const uint64_t good = __ballot(e < len && from > prev && from < fresh);
        const uint32_t n = good == ~0ull ? 64u : (uint32_t)__builtin_ctzll(~good); // up to the first that does not rise
        before = __shfl(from, 63);
        kept += n;
        whole = n == 64;
        const int32_t src = base + from, dst = base + (int32_t)e;
        uint32_t from_units = 0, to_units = 0;
        bool moves = lane < n && from != (int32_t)e && dst >= 0;
        if (moves) {
            const uint32_t x = paged_entry(a.kv, table, a.b.max_pages, (uint32_t)src),
                           y = paged_entry(a.kv, table, a.b.max_pages, (uint32_t)dst);
            moves = paged_units(a.kv, x, (uint32_t)src, &from_units);
            moves = paged_units(a.kv, y, (uint32_t)dst, &to_units) && moves;
        }
        const uint64_t todo = __ballot(moves);
        if (!todo) continue;
        // A wave's pieces, 64 at a time. All its lanes are on where a place is read from the lane that has it; only the moves
        // leave out lanes past the last piece.
        for (uint32_t c0 = wave * 64; c0 < a.chunks; c0 += blockDim.x) { // uniform
            const uint32_t c = c0 + lane, head = a.per_head.quot(c);
            char *const at = pool + (uint64_t)head * a.kv.head_bytes + (c - head * a.per_head.d) * 16;
            uint64_t rest = todo;
            while (rest) { // uniform
                uint32_t from_at[FLIGHT], to_at[FLIGHT];
                int flying = 0;
#pragma unroll
                for (int i = 0; i < FLIGHT; i++) {
                    if (!rest) break;
                    const int l = __builtin_ctzll(rest);
                    rest &= rest - 1;
                    from_at[i] = (uint32_t)__builtin_amdgcn_readlane((int)from_units, l);
                    to_at[i] = (uint32_t)__builtin_amdgcn_readlane((int)to_units, l);
                    flying++;
                }
                if (c < a.chunks) {
                    u4 x[FLIGHT];
#pragma unroll
                    for (int i = 0; i < FLIGHT; i++)
                        if (i < flying) x[i] = *reinterpret_cast<const u4 *>(at + ((uint64_t)from_at[i] << a.kv.unit_shift));
#pragma unroll
                    for (int i = 0; i < FLIGHT; i++)
                        if (i < flying) *reinterpret_cast<u4 *>(at + ((uint64_t)to_at[i] << a.kv.unit_shift)) = x[i];
                }
            }
        }
    }
    if (a.kv_len_out && blockIdx.y == 0 && threadIdx.x == 0) a.kv_len_out[seq] = max(base + (int32_t)kept, 0);
}

// What the host sees of an array: where it begins, and its bytes.
struct Span {
    const void *p;
    size_t bytes;
    bool meets(const Span &x) const {
        const uintptr_t a = (uintptr_t)p, b = (uintptr_t)x.p;
        return a && b && bytes && x.bytes && a < b + x.bytes && b < a + bytes;
    }
};

} // namespace
} // namespace aq

using namespace aq;

extern "C" {

int aq_paged_tables(aq_ctx *ctx, const aq_page_tables *t, const int32_t *kv_before, const int32_t *n_new, uint32_t n_rows,
                    int32_t *row_start, int32_t *kv_len, int32_t *missing, int32_t *pos, int64_t *slots,
                    const int32_t *row_depth, void *stream) {
    AQ_REQUIRE(ctx && t, "aq_paged_tables: null argument");
    AQ_REQUIRE(t->n_seq < (1u << 24) && n_rows < (1u << 24), "aq_paged_tables: batch size (fewer than 2^24 rows)");
    AQ_REQUIRE(t->n_pages > 0 && t->n_pages < (1u << 31) && t->page_size > 0 && t->page_size < (1u << 31),
               "aq_paged_tables: pages");
    AQ_REQUIRE(t->n_seq == 0 || t->max_pages > 0, "aq_paged_tables: max_pages");
    AQ_REQUIRE((uint64_t)t->max_pages * t->page_size <= (1ull << 31) - 1024,
               "aq_paged_tables: the page table reaches past 2^31 positions");
    if ((uint64_t)t->n_seq * t->max_pages >= (1ull << 32))
        return fail(AQ_EUNSUP, "aq_paged_tables: tables of 2^32 entries and more");
    AQ_REQUIRE(t->free_pages && t->free_state && t->free_state_out, "aq_paged_tables: null free pages");
    AQ_REQUIRE(t->n_seq == 0 || (t->pages && t->held && t->held_out && kv_before && n_new && kv_len),
               "aq_paged_tables: null array");
    AQ_REQUIRE(row_start, "aq_paged_tables: null row_start");
    AQ_REQUIRE(!row_depth || pos, "aq_paged_tables: depths without positions");
    const void *all[] = {t->pages, t->held,  t->held_out, t->free_pages, t->free_state, t->free_state_out, kv_before,
                         n_new,    row_start, kv_len,     missing,       pos,           row_depth};
    for (const void *p : all) AQ_REQUIRE((uintptr_t)p % 4 == 0, "aq_paged_tables: an array is not aligned to its type");
    AQ_REQUIRE((uintptr_t)slots % 8 == 0, "aq_paged_tables: an array is not aligned to its type");
    const size_t seqs = (size_t)t->n_seq * 4, rows = (size_t)n_rows * 4;
    const Span spans[] = {{t->held_out, seqs}, {t->free_state_out, 16}, {kv_len, seqs}, // these three may be an input's own array
                          {t->held, seqs}, {t->free_state, 16}, {kv_before, seqs}, {n_new, seqs}, {row_depth, rows},
                          {row_start, seqs + 4}, {missing, seqs}, {pos, rows}, {slots, 2 * rows}, {t->pages, seqs * t->max_pages},
                          {t->free_pages, (size_t)t->n_pages * 4}};
    constexpr int OUT = 3, READ = 8, ALL = sizeof(spans) / sizeof(spans[0]); // 3 .. 7 are only read
    for (int i = 0; i < ALL; i++)
        for (int j = i + 1; j < ALL; j++)
            AQ_REQUIRE(!spans[i].meets(spans[j]) || (i >= OUT && j < READ) || (j == i + OUT && i < OUT && spans[i].p == spans[j].p),
                       "aq_paged_tables: an output lies over another array");
    TablesArgs a;
    a.before = kv_before;
    a.fresh = n_new;
    a.held = t->held;
    a.state = t->free_state;
    a.depth = row_depth;
    a.pages = t->pages;
    a.ring = t->free_pages;
    a.held_out = t->held_out;
    a.state_out = t->free_state_out;
    a.row_start = row_start;
    a.kv_len = kv_len;
    a.missing = missing;
    a.pos = pos;
    a.slots = slots;
    a.n_seq = t->n_seq;
    a.max_pages = t->max_pages;
    a.n_pages = t->n_pages;
    a.n_rows = n_rows;
    a.apart = a.held_out != a.held && a.state_out != a.state && a.kv_len != a.before;
    a.page_size = FastDiv(t->page_size);
    // A row to a thread, or 16 threads to a sequence, whose pages put back are not known here: 700 requests of 90 rows with 49,
    // 98 and 197 work-groups of 256 17.7, 15.3 and 13.3 us, with 97 of 512 10.5; 300 of one row, some of which ended, with one
    // and 18 of 256 17.7 and 7.9. In place no more than 64: each arrives at the counter, 256 of them 6 us later.
    const uint64_t work = (uint64_t)t->n_seq * 16 > n_rows ? (uint64_t)t->n_seq * 16 : n_rows;
    const bool small = t->n_seq <= 256;
    const uint32_t threads = small ? 256 : 512, most = a.apart ? 65536 / threads : 64;
    const uint32_t grid = work < 2 * threads ? 1 : work / threads > most ? most : (uint32_t)(work / threads);
    AQ_HIP(hipSetDevice(ctx->device));
    const hipStream_t st = stream ? (hipStream_t)stream : ctx->stream;
    if (small) tables_kernel<1, 256><<<grid, threads, 0, st>>>(a);
    else tables_kernel<2, 512><<<grid, threads, 0, st>>>(a); // 1024 sequences a scan
    AQ_HIP(hipGetLastError());
    return 0;
}

int aq_paged_tree_commit(aq_ctx *ctx, const aq_paged_kv *kv, uint32_t n_kv, const aq_paged_batch *batch,
                         const int32_t *path_dev, const int32_t *path_len_dev, uint32_t max_path, int32_t *kv_len_out,
                         void *stream) {
    const char *call = "aq_paged_tree_commit";
    AQ_REQUIRE(ctx && kv && n_kv > 0, "aq_paged_tree_commit: null argument");
    CommitArgs a;
    for (uint32_t i = 0; i < n_kv; i++) {
        const int rc = check_paged(call, kv + i, batch, &a.kv, &a.b);
        if (rc) return rc;
        const aq_paged_kv &x = kv[i], &y = kv[0];
        AQ_REQUIRE(x.type == y.type && x.n_pages == y.n_pages && x.page_size == y.page_size && x.n_head_kv == y.n_head_kv &&
                       x.head_dim == y.head_dim && x.page_stride == y.page_stride && x.slot_stride == y.slot_stride &&
                       x.head_stride == y.head_stride,
                   "aq_paged_tree_commit: caches of different shapes");
    }
    AQ_REQUIRE(batch->n_seq == 0 || (path_dev && path_len_dev && max_path > 0), "aq_paged_tree_commit: null path");
    AQ_REQUIRE(max_path < (1u << 24), "aq_paged_tree_commit: max_path");
    AQ_REQUIRE((uintptr_t)path_dev % 4 == 0 && (uintptr_t)path_len_dev % 4 == 0 && (uintptr_t)kv_len_out % 4 == 0,
               "aq_paged_tree_commit: an array is not aligned to its type");
    const size_t seqs = (size_t)batch->n_seq * 4;
    const Span read[] = {{batch->kv_len, seqs}, {batch->row_start, seqs + 4}, {batch->pages, seqs * batch->max_pages},
                         {path_dev, seqs * max_path}, {path_len_dev, seqs}};
    for (const Span &x : read)
        AQ_REQUIRE(!x.meets({kv_len_out, seqs}), "aq_paged_tree_commit: kv_len_out lies over an input");
    // Rows that two of the call's work-groups move would be moved on by the second.
    std::unique_ptr<const void *[]> pools(new (std::nothrow) const void *[2 * (size_t)n_kv]);
    if (!pools) return fail(AQ_ENOMEM, "aq_paged_tree_commit: host allocation");
    for (uint32_t i = 0; i < n_kv; i++) {
        pools[2 * (size_t)i] = kv[i].k;
        pools[2 * (size_t)i + 1] = kv[i].v;
    }
    std::sort(&pools[0], &pools[0] + 2 * (size_t)n_kv);
    AQ_REQUIRE(std::adjacent_find(&pools[0], &pools[0] + 2 * (size_t)n_kv) == &pools[0] + 2 * (size_t)n_kv,
               "aq_paged_tree_commit: two of the caches' k and v are the same memory");
    if (batch->n_seq == 0) return 0;
    a.path = path_dev;
    a.path_len = path_len_dev;
    a.max_path = max_path;
    const uint32_t per_head = (uint32_t)(kv->head_dim * type_bytes(kv->type) / 16);
    a.chunks = per_head * kv->n_head_kv;
    a.per_head = FastDiv(per_head);
    uint32_t threads = 64;
    while (threads < 256 && threads < a.chunks) threads *= 2;
    AQ_HIP(hipSetDevice(ctx->device));
    const hipStream_t st = stream ? (hipStream_t)stream : ctx->stream;
    for (uint32_t i = 0; i < n_kv; i += MAX_CACHES) {
        const uint32_t n = n_kv - i < MAX_CACHES ? n_kv - i : MAX_CACHES;
        for (uint32_t j = 0; j < n; j++) {
            a.pools[2 * j] = (char *)kv[i + j].k;
            a.pools[2 * j + 1] = (char *)kv[i + j].v;
        }
        a.kv_len_out = i ? nullptr : kv_len_out;
        commit_kernel<<<dim3(batch->n_seq, 2 * n), threads, 0, st>>>(a);
        AQ_HIP(hipGetLastError());
    }
    return 0;
}

} // extern "C"
