// yl_pages.hip -- the pages of a pool: handing them out, sharing them between
// branches of a conversation, giving them back, moving them together.
// No counterpart in the reference, which holds one conversation.
//
// All state is on the device (tables, lengths, references), so that a step that
// branches and ends conversations can be captured.  "The free pages in rising
// order" is an exclusive scan over the references: a workgroup per 1024 pages
// counts, then each adds up the counts before its own and lists its pages by
// rank; pools of up to 16,384 pages by one workgroup.  Bound by the copies; the
// scans are launches of 2 to 5 us: four branches of a 600-token answer, 16 layers, f16:
// release 2.5, list 3.3, copy 5.1, reserve 2.9 us.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/yallma3.h"
#include "yl_device.h"
#include "yl_internal.h"
#include "yl_paged.h"

namespace yl {

namespace {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int kLayers = 128;           // pools of one call: their addresses are kernel arguments

// The pools of all layers: of every (page, kv head), page_size rows of row0
// bytes, then (MXFP4's scales) as many of row1.
struct Pools {
    char* at[2 * kLayers];             // keys and values in turn
    int n, n_kv, page_shift, row0, row1;
};
__host__ __device__ __forceinline__ size_t head_bytes(const Pools& p) { return (size_t)(p.row0 + p.row1) << p.page_shift; }

// The workspace, in ints (n_pages, sequences or forks).
struct Space {
    int* counts;                       // [1024] pages of a kind in each workgroup's share
    int* meta;                         // [16]
    int* need; int* first;             // [items]: pages that an item takes, and the rank of its first
    int* list;                         // [n_pages] pages by rank
    int* rank; int* holes;             // [n_pages] each (compact)
};
enum { kFree = 0, kMoved = 1 };        // meta: free (used) pages; pages that move

size_t space_ints(size_t n_pages, size_t items) { return 1024 + 16 + 2 * items + 3 * n_pages; }
Space space_of(void* w, size_t n_pages, size_t items) {
    int* p = static_cast<int*>(w);
    return Space{p, p + 1024, p + 1040, p + 1040 + items, p + 1040 + 2 * items, p + 1040 + 2 * items + n_pages,
                 p + 1040 + 2 * items + 2 * n_pages};
}

__device__ __forceinline__ int scan_add(int x) {       // inclusive, over the 64 lanes
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, true);
    return x;
}

// Exclusive scan of one value per thread over a workgroup of W wavefronts; *total: the sum.
template <int W>
__device__ __forceinline__ int scan_group(int x, int* total) {
    __shared__ int sums[W];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int upto = scan_add(x);
    __syncthreads();                                   // (the last scan's sums have been read)
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < W; w++) {
        const int s = sums[w];
        before += w < wave ? s : 0;
        all += s;
    }
    *total = all;
    return before + upto - x;
}

}  // namespace

// ----------------------------------------------------- counting and listing

// Of each workgroup's share of the pages, how many are in use (used) or free.
// Workgroups behind them count the entries that each sequence lacks (want_len).
__global__ __launch_bounds__(256) void k_pages_count(TableArgs t, Space sp, int used, const uint32_t* want_len, uint32_t* lacking) {
    const int groups = page_groups(t.n_pages), per = pages_per_group(t.n_pages), tid = threadIdx.x;
    if (blockIdx.x == 0 && tid == 0 && lacking) *lacking = 0;
    if ((int)blockIdx.x >= groups) {                   // a wavefront per sequence
        const int s = ((int)blockIdx.x - groups) * 4 + (tid >> 6), lane = tid & 63;
        if (s >= t.n_seqs) return;
        bool past;
        const int n = table_entries(t, want_len[s], &past);
        int missing = 0;
        for (int i = lane; i < n; i += 64) missing += paged_page(t.table[(size_t)s * t.max_pages + i], t.n_pages) < 0;
        missing = scan_add(missing);
        if (lane == 63) sp.need[s] = missing;
        return;
    }
    int n = 0;
    const int64_t begin = (int64_t)blockIdx.x * per, end = min(begin + per, (int64_t)t.n_pages);
    for (int64_t p = begin + tid; p < end; p += 256) n += (t.refs[p] > 0) == (used != 0);
    int total;
    scan_group<4>(n, &total);
    if (tid == 0) sp.counts[blockIdx.x] = total;
}

// Of all shares, the pages before this one's and all of them.
__device__ __forceinline__ int pages_before(const Space& sp, int groups, int group, int* all) {
    int before = 0, sum = 0;
    for (int i = threadIdx.x; i < groups; i += 256) {
        const int n = sp.counts[i];
        sum += n;
        before += i < group ? n : 0;
    }
    int b;
    scan_group<4>(sum, all);
    scan_group<4>(before, &b);
    return b;
}

// Whether child i of a fork takes a page, and of which parent's entry.
__device__ __forceinline__ bool fork_pair(const TableArgs& t, const uint32_t* parents, const uint32_t* children, int i, int* parent,
                                          int* child, int* full, int* slots, int* last) {
    const uint32_t p = parents[i], c = children[i];
    if (p >= (uint32_t)t.n_seqs || c >= (uint32_t)t.n_seqs || p == c) return false;
    *parent = (int)p;
    *child = (int)c;
    table_filled(t, t.kv_len[p], full, slots);
    *last = *slots ? paged_page(t.table[(size_t)p * t.max_pages + *full], t.n_pages) : -1;
    return true;
}

// Lists the free pages by rank, the first n_list of them.  The last workgroup
// adds up what the items (forks; or sequences, sp.need) take.
__global__ __launch_bounds__(256) void k_pages_list(TableArgs t, Space sp, int n_list, int items, const uint32_t* parents, const uint32_t* children) {
    const int groups = page_groups(t.n_pages), per = pages_per_group(t.n_pages), tid = threadIdx.x;
    if ((int)blockIdx.x == groups) {
        int before = 0;
        for (int b = 0; b < items; b += 256) {
            const int i = b + tid;
            int need = 0, p, c, f, s, last;
            if (i < items) {
                if (!parents) need = sp.need[i];
                else if (fork_pair(t, parents, children, i, &p, &c, &f, &s, &last)) need = last >= 0;
            }
            int total;
            const int first = before + scan_group<4>(need, &total);
            if (i < items) sp.first[i] = first;
            before += total;
        }
        return;
    }
    int all;
    int rank = pages_before(sp, groups, blockIdx.x, &all);
    if (blockIdx.x == 0 && tid == 0) sp.meta[kFree] = all;
    const int64_t begin = (int64_t)blockIdx.x * per, end = min(begin + per, (int64_t)t.n_pages);
    for (int64_t b = begin; b < end; b += 256) {
        const int64_t p = b + tid;
        const bool is = p < end && t.refs[p] <= 0;
        int total;
        const int r = rank + scan_group<4>(is, &total);
        if (is && r < n_list) sp.list[r] = (int)p;
        rank += total;
    }
}

// Page p, which `before` used pages precede, where `used` are in use: the j-th used page
// (from 0) moves if its id is not below `used`; the movers are the last kMoved of
// the ranks, and meet the free ids below `used` in order.
__device__ __forceinline__ void move_page(const Space& sp, int p, bool is, int before, int used) {
    if (p == used) sp.meta[kMoved] = used - before;
    if (p >= used) {
        sp.rank[p] = is ? before : -1;
        if (is) sp.list[before] = p;
    } else if (!is) {
        sp.holes[p - before] = p;
    }
}

// ---------------------------------------------------------------- reserving

// A wavefront per sequence fills the entries that name no page, in their order.
__global__ __launch_bounds__(256) void k_pages_reserve(TableArgs t, Space sp, const uint32_t* want_len, uint32_t* lacking) {
    const int s = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (s >= t.n_seqs) return;
    bool past;
    const int n = table_entries(t, want_len[s], &past), free_pages = sp.meta[kFree];
    int rank = sp.first[s], lacks = past;
    for (int b = 0; b < n; b += 64) {
        const int i = b + lane;
        const bool missing = i < n && paged_page(t.table[(size_t)s * t.max_pages + i], t.n_pages) < 0;
        const auto all = __ballot(missing);
        const int r = rank + __builtin_popcountll(all & ((1ull << lane) - 1));
        if (missing && r < free_pages) {
            const int page = sp.list[r];
            t.table[(size_t)s * t.max_pages + i] = page;
            t.refs[page] = 1;
        }
        rank += __builtin_popcountll(all);
        lacks += __builtin_popcountll(__ballot(missing && r >= free_pages));
    }
    if (lane == 0 && lacks && lacking) atomicAdd(lacking, (uint32_t)lacks);
}

// -------------------------------------------------------------- small pools

// One workgroup looks through up to kSmall things, C neighbouring ones per thread,
// all of their loads in flight: a launch less than counting and listing, two less
// than reserving.
constexpr int kSmallThreads = 1024, kSmallMost = 16, kSmall = kSmallThreads * kSmallMost;
// (320 sequences of 24 entries: 16 us by one workgroup, 13 by the three kernels)
constexpr int kSmallReserve = 4 * kSmallThreads;

// Ranks, in rising order, of those of n things that `is` picks from their values: put(index, rank).  Returns how many there are.
template <int C, typename Load, typename Is, typename Put>
__device__ __forceinline__ int rank_all(int n, const Load& load, const Is& is, const Put& put) {
    const int at = threadIdx.x * C;
    int v[C], mine = 0;
#pragma unroll
    for (int i = 0; i < C; i++) v[i] = n > 0 ? load(min(at + i, n - 1)) : 0;
#pragma unroll
    for (int i = 0; i < C; i++) mine += at + i < n && is(at + i, v[i]);
    int total, rank = scan_group<kSmallThreads / 64>(mine, &total);
#pragma unroll
    for (int i = 0; i < C; i++)
        if (at + i < n) {
            const bool yes = is(at + i, v[i]);
            put(at + i, yes ? rank : -1, rank);
            rank += yes;
        }
    return total;
}

// What k_pages_count and k_pages_list leave for a fork.
template <int C>
__global__ __launch_bounds__(kSmallThreads) void k_pages_list_small(TableArgs t, Space sp, int items, const uint32_t* parents, const uint32_t* children,
                                                                    uint32_t* lacking) {
    if (threadIdx.x == 0 && lacking) *lacking = 0;
    const int free_pages = rank_all<C>(t.n_pages, [&](int i) { return t.refs[i]; }, [](int, int r) { return r <= 0; },
                                       [&](int i, int r, int) { if (r >= 0) sp.list[r] = i; });
    if (threadIdx.x == 0) sp.meta[kFree] = free_pages;
    rank_all<C>(items,
                [&](int i) {
                    int p, c, f, s, last;
                    return (int)(fork_pair(t, parents, children, i, &p, &c, &f, &s, &last) && last >= 0);
                },
                [](int, int need) { return need != 0; }, [&](int i, int, int before) { sp.first[i] = before; });
}

// yl_paged_reserve: the entries that name no page, in the table's order, get the free pages.
template <int C>
__global__ __launch_bounds__(kSmallThreads) void k_pages_reserve_small(TableArgs t, const uint32_t* want_len, uint32_t* lacking) {
    __shared__ int list[kSmallThreads * C];
    __shared__ int past;
    if (threadIdx.x == 0) past = 0;
    const int free_pages = rank_all<C>(t.n_pages, [&](int i) { return t.refs[i]; }, [](int, int r) { return r <= 0; },
                                       [&](int i, int r, int) { if (r >= 0) list[r] = i; });
    __syncthreads();
    for (int s = threadIdx.x; s < t.n_seqs; s += kSmallThreads) {
        bool p;
        table_entries(t, want_len[s], &p);
        if (p) atomicAdd(&past, 1);
    }
    // (1: wanted and not there)
    const int missing = rank_all<C>(t.n_seqs * t.max_pages,
                                    [&](int i) {
                                        bool p;
                                        const int s = i / t.max_pages;
                                        return (int)(i - s * t.max_pages < table_entries(t, want_len[s], &p) && paged_page(t.table[i], t.n_pages) < 0);
                                    },
                                    [](int, int is) { return is != 0; },
                                    [&](int i, int r, int) {
                                        if (r < 0 || r >= free_pages) return;
                                        t.table[i] = list[r];
                                        t.refs[list[r]] = 1;
                                    });
    __syncthreads();
    if (threadIdx.x == 0 && lacking) *lacking = (uint32_t)(max(missing - free_pages, 0) + past);
}

// What k_pages_count and k_pages_moves leave for moving.
template <int C>
__global__ __launch_bounds__(kSmallThreads) void k_pages_moves_small(TableArgs t, Space sp, uint32_t* used_out) {
    int used = 0;
    {
        const int at = threadIdx.x * C;
        int v[C], mine = 0;
#pragma unroll
        for (int i = 0; i < C; i++) v[i] = t.refs[min(at + i, t.n_pages - 1)];
#pragma unroll
        for (int i = 0; i < C; i++) mine += at + i < t.n_pages && v[i] > 0;
        int before = scan_group<kSmallThreads / 64>(mine, &used);
#pragma unroll
        for (int i = 0; i < C; i++)
            if (at + i < t.n_pages) {
                move_page(sp, at + i, v[i] > 0, before, used);
                before += v[i] > 0;
            }
    }
    if (threadIdx.x == 0) {
        sp.meta[kFree] = used;
        *used_out = (uint32_t)used;
        if (used == t.n_pages) sp.meta[kMoved] = 0;
    }
}

// ------------------------------------------------------------------ copying

// `bytes` (a multiple of 16) from one 16-byte aligned place to another by the whole
// workgroup.  The stores are not kept in L2: 700 pages of 16 layers, 229 MB, 98 us with
// plain ones, 77 with these, 5.9 TB/s in and out (a large copy: 4.9).
__device__ __forceinline__ void copy16(char* dst, const char* src, size_t bytes) {
    const size_t n = bytes / 16;
    const u4* s = reinterpret_cast<const u4*>(src);
    u4* d = reinterpret_cast<u4*>(dst);
    size_t i = threadIdx.x;
    for (; i + 768 < n; i += 1024) {
        u4 x[4];
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = s[i + 256 * k];
#pragma unroll
        for (int k = 0; k < 4; k++) __builtin_nontemporal_store(x[k], d + i + 256 * k);
    }
    for (; i < n; i += 256) d[i] = s[i];
}

// The filled slots of a page, of one layer's keys or values.  (256 copies of some 16
// slots in 16 layers, 129 MB written: 41 us, 3.1 TB/s; all heads' stretches as one, or
// four layers per workgroup, the same.)
__device__ __forceinline__ void copy_slots(const Pools& pl, int which, int dst, int src, int slots) {
    const size_t head = head_bytes(pl), codes = (size_t)slots * pl.row0, scales = (size_t)slots * pl.row1;
    for (int h = 0; h < pl.n_kv; h++) {
        char* d = pl.at[which] + ((size_t)dst * pl.n_kv + h) * head;
        const char* s = pl.at[which] + ((size_t)src * pl.n_kv + h) * head;
        copy16(d, s, codes);
        const size_t at = (size_t)pl.row0 << pl.page_shift;
        for (size_t i = threadIdx.x; i < scales; i += 256) d[at + i] = s[at + i];
    }
}

// ------------------------------------------------------------------ forking

// Workgroups (which, child): the copy of the last page in one layer's keys or
// values; those of `which` = n also write the child's row.
__global__ __launch_bounds__(256) void k_pages_fork(TableArgs t, Space sp, Pools pl, const uint32_t* parents, const uint32_t* children,
                                                    int child0, uint32_t* lacking) {
    const int which = blockIdx.x, i = child0 + blockIdx.y, tid = threadIdx.x;
    int parent, child, full, slots, last;
    if (!fork_pair(t, parents, children, i, &parent, &child, &full, &slots, &last)) return;
    const bool takes = last >= 0;
    const int rank = sp.first[i];
    const bool made = !takes || rank < sp.meta[kFree];
    const int page = takes && made ? sp.list[rank] : -1;
    if (which < 2 * pl.n) {
        if (page >= 0) copy_slots(pl, which, page, last, slots);
        return;
    }
    const int32_t* from = t.table + (size_t)parent * t.max_pages;
    int32_t* to = t.table + (size_t)child * t.max_pages;
    for (int e = tid; e < t.max_pages; e += 256) {
        int x = -1;
        if (made && e < full) {
            x = paged_page(from[e], t.n_pages);
            if (x >= 0) atomicAdd(&t.refs[x], 1);
        } else if (e == full) {
            x = page;
        }
        to[e] = x;
    }
    if (tid == 0) {
        t.kv_len[child] = made ? t.kv_len[parent] : 0;
        if (page >= 0) t.refs[page] = 1;
        if (!made && lacking) atomicAdd(lacking, 1u);
    }
}

// ---------------------------------------------------------------- releasing

// A workgroup per sequence.  An entry is taken out once, so that a sequence that
// is there twice is ended once.
__global__ __launch_bounds__(256) void k_pages_release(TableArgs t, const uint32_t* seqs, int seq0) {
    const uint32_t s = seqs[seq0 + blockIdx.x];
    if (s >= (uint32_t)t.n_seqs) return;
    for (int e = threadIdx.x; e < t.max_pages; e += 256) {
        const int page = paged_page(atomicExch(&t.table[(size_t)s * t.max_pages + e], -1), t.n_pages);
        if (page >= 0) atomicSub(&t.refs[page], 1);
    }
    if (threadIdx.x == 0) t.kv_len[s] = 0;
}

// --------------------------------------------------------------- compacting

// Ranks of pages that move, -1 of free ones; where they go.
__global__ __launch_bounds__(256) void k_pages_moves(TableArgs t, Space sp, uint32_t* used_out) {
    const int groups = page_groups(t.n_pages), per = pages_per_group(t.n_pages), tid = threadIdx.x;
    int used;
    int rank = pages_before(sp, groups, blockIdx.x, &used);
    const int64_t begin = (int64_t)blockIdx.x * per, end = min(begin + per, (int64_t)t.n_pages);
    if (blockIdx.x == 0 && tid == 0) {
        sp.meta[kFree] = used;
        *used_out = (uint32_t)used;
        if (used == t.n_pages) sp.meta[kMoved] = 0;
    }
    for (int64_t b = begin; b < end; b += 256) {
        const int64_t p = b + tid;
        const bool is = p < end && t.refs[p] > 0;
        int total;
        const int before = rank + scan_group<4>(is, &total);
        if (p < end) move_page(sp, (int)p, is, before, used);
        rank += total;
    }
}

// Where the page of an entry has gone.
__device__ __forceinline__ int moved_to(const TableArgs& t, const Space& sp, int entry, int used, int moved) {
    const int page = paged_page(entry, t.n_pages);
    if (page < used) return entry;                     // (none, or one that stays)
    const int r = sp.rank[page];
    return r < 0 ? entry : sp.holes[r - (used - moved)];
}

// Workgroups deal the moves of all layers' keys and values among themselves, then
// the entries of the tables.
__global__ __launch_bounds__(256) void k_pages_move(TableArgs t, Space sp, Pools pl) {
    const int used = sp.meta[kFree], moved = sp.meta[kMoved], tid = threadIdx.x;
    if (moved == 0) return;
    const size_t bytes = head_bytes(pl) * pl.n_kv;
    const int64_t jobs = (int64_t)moved * 2 * pl.n;
    for (int64_t j = blockIdx.x; j < jobs; j += gridDim.x) {
        const int m = (int)(j / (2 * pl.n)), which = (int)(j % (2 * pl.n));
        const int src = sp.list[used - moved + m], dst = sp.holes[m];
        copy16(pl.at[which] + dst * bytes, pl.at[which] + src * bytes, bytes);
        if (which == 0 && tid == 0) {
            t.refs[dst] = t.refs[src];
            t.refs[src] = 0;
        }
    }
    const int64_t entries = (int64_t)t.n_seqs * t.max_pages;
    for (int64_t i = (int64_t)blockIdx.x * 256 + tid; i < entries + t.prefix_entries; i += (int64_t)gridDim.x * 256) {
        int32_t* e = i < entries ? t.table + i : t.prefix_pages + (i - entries);
        const int old = *e, now = moved_to(t, sp, old, used, moved);
        if (now != old) *e = now;
    }
}

// The keys and values, in turn, of some layers of two pools whose pages have `bytes`.
struct PoolPairs {
    static constexpr int kMost = 64;
    char* dst[2 * kMost];
    const char* src[2 * kMost];
    size_t bytes;
    int dst_pages, src_pages;
};

// Workgroups (which, pair): whole pages between pools.
__global__ __launch_bounds__(256) void k_pages_copy(PoolPairs pp, const int32_t* to, const int32_t* from, int pair0) {
    const int which = blockIdx.x, i = pair0 + blockIdx.y;
    const int d = paged_page(to[i], pp.dst_pages), s = paged_page(from[i], pp.src_pages);
    if (d < 0 || s < 0) return;
    copy16(pp.dst[which] + d * pp.bytes, pp.src[which] + s * pp.bytes, pp.bytes);
}

// --------------------------------------------------------------------- host

namespace {

yl_status refuse(const char* what, yl_status st = YL_ERR_ARG) {
    set_error(what);
    return st;
}

yl_status table_args(const yl_paged_tables* t, TableArgs* a) {
    if (!t) return refuse("paged tables: none");
    if (t->page_size != 16 && t->page_size != 32 && t->page_size != 64 && t->page_size != 128 && t->page_size != 256)
        return refuse("paged tables: page size 16, 32, 64, 128 or 256");
    if (!t->n_pages || (uint64_t)t->n_pages * t->page_size >= (1ull << 31))
        return refuse("paged tables: n_pages * page_size from 1 page to below 2^31");
    if (t->n_seqs > (1u << 22) || (uint64_t)t->n_seqs * t->max_pages >= (1ull << 31) ||
        (uint64_t)t->prefix_len + (uint64_t)t->max_pages * t->page_size >= (1ull << 30))
        return refuse("paged tables: n_seqs at most 2^22, n_seqs * max_pages below 2^31, a sequence's capacity below 2^30", YL_ERR_RANGE);
    if (!t->refs || (t->n_seqs && (!t->kv_len || (t->max_pages && !t->page_table)))) return refuse("paged tables: refs, kv_len and page_table have to be there");
    if (t->prefix_len && !t->prefix_pages) return refuse("paged tables: a prefix needs prefix_pages");
    *a = TableArgs{(int)t->n_seqs, (int)t->max_pages, (int)t->n_pages, __builtin_ctz(t->page_size), t->page_table, t->kv_len, t->refs,
                   (int)t->prefix_len, (int)((t->prefix_len + t->page_size - 1) / t->page_size), t->prefix_pages};
    return YL_OK;
}

// The pools of a call; `n_pages` 0: any number of pages, but the same of all.
yl_status pools_of(const yl_paged_cache* c, uint32_t n, uint32_t n_pages, uint32_t page_size, Pools* p) {
    if (!c || !n || n > (uint32_t)kLayers) return refuse("paged pages: 1 to 128 layers");
    for (uint32_t i = 0; i < n; i++) {
        const yl_status st = paged_cache_ok(c + i);
        if (st != YL_OK) return st;
        if (c[i].dtype != c->dtype || c[i].n_pages != c->n_pages || c[i].page_size != c->page_size || c[i].n_kv_heads != c->n_kv_heads ||
            c[i].head_size != c->head_size)
            return refuse("paged pages: layers of one type, size and number of pages");
        p->at[2 * i] = static_cast<char*>(c[i].keys);
        p->at[2 * i + 1] = static_cast<char*>(c[i].values);
    }
    if (n_pages && (c->n_pages != n_pages || c->page_size != page_size)) return refuse("paged pages: tables of other pools (n_pages, page_size)");
    p->n = (int)n;
    p->n_kv = (int)c->n_kv_heads;
    p->page_shift = __builtin_ctz(c->page_size);
    const int hd = (int)c->head_size;
    p->row0 = c->dtype == YL_T_F32 ? 4 * hd : c->dtype == YL_T_MXFP4 ? hd / 2 : 2 * hd;
    p->row1 = c->dtype == YL_T_MXFP4 ? hd / 32 : 0;
    return YL_OK;
}

size_t items_of(const TableArgs& t, uint32_t n) { return std::max<size_t>(n, (size_t)t.n_seqs); }

yl_status space_ok(const TableArgs& t, uint32_t n, void* w, size_t bytes) {
    if (!w || (uintptr_t)w % 16) return refuse("paged tables: the workspace has to be there, 16-byte aligned");
    if (bytes < 4 * space_ints(t.n_pages, items_of(t, n))) return refuse("paged tables: the workspace is smaller than yl_paged_tables_workspace says", YL_ERR_RANGE);
    return YL_OK;
}

yl_status launched(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return YL_OK;
    set_error(std::string(what) + ": " + hipGetErrorString(e));
    return YL_ERR_HIP;
}

constexpr uint32_t kGridY = 65535;

// Launches one of a kernel's forms for 1, 4 or 16 things per thread of a workgroup.
#define YL_SMALL(kernel, things, s, ...)                                                                           \
    do {                                                                                                           \
        auto k = (things) <= kSmallThreads ? kernel<1> : (things) <= 4 * kSmallThreads ? kernel<4> : kernel<16>;   \
        hipLaunchKernelGGL(k, dim3(1), dim3(kSmallThreads), 0, s, __VA_ARGS__);                                    \
    } while (0)

}  // namespace
}  // namespace yl

using namespace yl;

extern "C" {

size_t yl_paged_tables_workspace(const yl_paged_tables* tables, uint32_t n) {
    TableArgs t{};
    if (table_args(tables, &t) != YL_OK || n > (1u << 22)) return 0;
    return 4 * space_ints(t.n_pages, items_of(t, n));
}

yl_status yl_paged_reserve(const yl_paged_tables* tables, const uint32_t* want_len, uint32_t* lacking, void* workspace,
                           size_t workspace_bytes, void* stream) {
    TableArgs t{};
    yl_status st = table_args(tables, &t);
    if (st != YL_OK) return st;
    if ((st = space_ok(t, 0, workspace, workspace_bytes)) != YL_OK) return st;
    if (t.n_seqs && !want_len) return refuse("paged_reserve: no want_len");
    const Space sp = space_of(workspace, t.n_pages, items_of(t, 0));
    const hipStream_t s = (hipStream_t)stream;
    const int64_t things = std::max<int64_t>({t.n_pages, (int64_t)t.n_seqs * t.max_pages, 1});
    if (things <= kSmallReserve) {
        auto k = things <= kSmallThreads ? k_pages_reserve_small<1> : k_pages_reserve_small<4>;
        hipLaunchKernelGGL(k, dim3(1), dim3(kSmallThreads), 0, s, t, want_len, lacking);
        return launched("paged_reserve launch");
    }
    const int groups = page_groups(t.n_pages), by_seq = (t.n_seqs + 3) / 4;
    hipLaunchKernelGGL(k_pages_count, dim3(groups + by_seq), dim3(256), 0, s, t, sp, 0, want_len, lacking);
    if ((st = launched("paged_reserve launch")) != YL_OK || !t.n_seqs) return st;
    hipLaunchKernelGGL(k_pages_list, dim3(groups + 1), dim3(256), 0, s, t, sp, t.n_pages, t.n_seqs, (const uint32_t*)nullptr, (const uint32_t*)nullptr);
    if ((st = launched("paged_reserve launch")) != YL_OK) return st;
    hipLaunchKernelGGL(k_pages_reserve, dim3(by_seq), dim3(256), 0, s, t, sp, want_len, lacking);
    return launched("paged_reserve launch");
}

yl_status yl_paged_fork(const yl_paged_tables* tables, const yl_paged_cache* layers, uint32_t n_layers, const uint32_t* parents,
                        const uint32_t* children, uint32_t n, uint32_t* lacking, void* workspace, size_t workspace_bytes, void* stream) {
    TableArgs t{};
    Pools pl{};
    yl_status st = table_args(tables, &t);
    if (st != YL_OK || (st = pools_of(layers, n_layers, tables->n_pages, tables->page_size, &pl)) != YL_OK) return st;
    if (n > (1u << 22)) return refuse("paged_fork: at most 2^22 forks", YL_ERR_RANGE);
    if ((st = space_ok(t, n, workspace, workspace_bytes)) != YL_OK) return st;
    if (n && (!parents || !children)) return refuse("paged_fork: no parents or no children");
    const Space sp = space_of(workspace, t.n_pages, items_of(t, n));
    const hipStream_t s = (hipStream_t)stream;
    const int groups = page_groups(t.n_pages);
    const int64_t things = std::max<int64_t>(t.n_pages, n);
    if (things <= kSmall) {
        YL_SMALL(k_pages_list_small, things, s, t, sp, (int)n, parents, children, lacking);
        if ((st = launched("paged_fork launch")) != YL_OK || !n) return st;
    } else {
        hipLaunchKernelGGL(k_pages_count, dim3(groups), dim3(256), 0, s, t, sp, 0, (const uint32_t*)nullptr, lacking);
        if ((st = launched("paged_fork launch")) != YL_OK || !n) return st;
        hipLaunchKernelGGL(k_pages_list, dim3(groups + 1), dim3(256), 0, s, t, sp, (int)std::min<uint32_t>(n, t.n_pages), (int)n, parents, children);
    }
    for (uint32_t c = 0; c < n && (st = launched("paged_fork launch")) == YL_OK; c += kGridY)
        hipLaunchKernelGGL(k_pages_fork, dim3(2 * pl.n + 1, std::min(n - c, kGridY)), dim3(256), 0, s, t, sp, pl, parents, children, (int)c, lacking);
    return st != YL_OK ? st : launched("paged_fork launch");
}

yl_status yl_paged_release(const yl_paged_tables* tables, const uint32_t* seqs, uint32_t n, void* stream) {
    TableArgs t{};
    const yl_status st = table_args(tables, &t);
    if (st != YL_OK) return st;
    if (n > (1u << 22)) return refuse("paged_release: at most 2^22 sequences", YL_ERR_RANGE);
    if (!n) return YL_OK;
    if (!seqs) return refuse("paged_release: no seqs");
    hipLaunchKernelGGL(k_pages_release, dim3(n), dim3(256), 0, (hipStream_t)stream, t, seqs, 0);
    return launched("paged_release launch");
}

yl_status yl_paged_compact(const yl_paged_tables* tables, const yl_paged_cache* layers, uint32_t n_layers, uint32_t* used,
                           void* workspace, size_t workspace_bytes, void* stream) {
    TableArgs t{};
    Pools pl{};
    yl_status st = table_args(tables, &t);
    if (st != YL_OK || (st = pools_of(layers, n_layers, tables->n_pages, tables->page_size, &pl)) != YL_OK) return st;
    if ((st = space_ok(t, 0, workspace, workspace_bytes)) != YL_OK) return st;
    if (!used) return refuse("paged_compact: no used");
    const Space sp = space_of(workspace, t.n_pages, items_of(t, 0));
    const hipStream_t s = (hipStream_t)stream;
    const int groups = page_groups(t.n_pages);
    if (t.n_pages <= kSmall) {
        YL_SMALL(k_pages_moves_small, t.n_pages, s, t, sp, used);
    } else {
        hipLaunchKernelGGL(k_pages_count, dim3(groups), dim3(256), 0, s, t, sp, 1, (const uint32_t*)nullptr, (uint32_t*)nullptr);
        if ((st = launched("paged_compact launch")) != YL_OK) return st;
        hipLaunchKernelGGL(k_pages_moves, dim3(groups), dim3(256), 0, s, t, sp, used);
    }
    if ((st = launched("paged_compact launch")) != YL_OK) return st;
    // as many copies at most as half of the pages move, or the entries, in a grid that fills the GPU
    const int64_t copies = (int64_t)(t.n_pages / 2) * 2 * pl.n, entries = ((int64_t)t.n_seqs * t.max_pages + t.prefix_entries + 255) / 256;
    const unsigned grid = (unsigned)std::clamp<int64_t>(std::max(copies, entries), 1, 4096);
    hipLaunchKernelGGL(k_pages_move, dim3(grid), dim3(256), 0, s, t, sp, pl);
    return launched("paged_compact launch");
}

yl_status yl_paged_copy(const yl_paged_cache* dst, const yl_paged_cache* src, uint32_t n_layers, const int32_t* dst_pages,
                        const int32_t* src_pages, uint32_t n, void* stream) {
    Pools d{}, f{};
    yl_status st = pools_of(dst, n_layers, 0, 0, &d);
    if (st != YL_OK || (st = pools_of(src, n_layers, 0, 0, &f)) != YL_OK) return st;
    if (dst->dtype != src->dtype || dst->page_size != src->page_size || dst->n_kv_heads != src->n_kv_heads || dst->head_size != src->head_size)
        return refuse("paged_copy: pools of one type, page size and heads");
    if (n >= (1u << 31)) return refuse("paged_copy: fewer than 2^31 pairs", YL_ERR_RANGE);
    if (n && (!dst_pages || !src_pages)) return refuse("paged_copy: no dst_pages or no src_pages");
    for (int l = 0; l < d.n; l += PoolPairs::kMost) {
        PoolPairs pp{};
        const int layers = std::min(d.n - l, PoolPairs::kMost);
        std::copy(d.at + 2 * l, d.at + 2 * (l + layers), pp.dst);
        std::copy(f.at + 2 * l, f.at + 2 * (l + layers), pp.src);
        pp.bytes = head_bytes(d) * d.n_kv;
        pp.dst_pages = (int)dst->n_pages;
        pp.src_pages = (int)src->n_pages;
        for (uint32_t c = 0; c < n; c += kGridY) {
            hipLaunchKernelGGL(k_pages_copy, dim3(2 * layers, std::min(n - c, kGridY)), dim3(256), 0, (hipStream_t)stream, pp, dst_pages, src_pages, (int)c);
            if ((st = launched("paged_copy launch")) != YL_OK) return st;
        }
    }
    return YL_OK;
}

}  // extern "C"
