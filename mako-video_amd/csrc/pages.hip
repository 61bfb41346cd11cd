// Kept rows in pages: `pages_take`, `pages_free`, `pages_fork`, `pages_copy`, `pages_compact` and `pages_write`. A stream's
// kept row j lies in page table[stream][j / page_rows], at its row j % page_rows; an entry of -1 is no page. refs[p] counts
// the entries that name page p, and a page is free if that is zero, so the table and refs are all of the state.
//
// What the calls decide is a function of their inputs alone: free pages are taken lowest first, for the entries in the
// order (stream, entry); counts change by integer atomics, whose order does not show. (Only rows that one pages_write writes
// twice, into a page that two entries name, are any mixture of the two: finding them would take a look at the other streams'
// entries for each row.) Entries that are no page of the pool (negative, or past its end) are no page to any kernel, so a
// bad table reads and writes nothing outside the pool.
// A program calls them once a step (fork, free, compact: now and then), for all layers: what bounds them is the launches
// (take and write 4.5 us each, a fork of eight streams 4.3 to plan and 4.3 to do) and, where pages move, HBM: 512 pages of
// 262 KB copied in 54 us, 5 TB/s, two of five streams' pages freed and 510 MB moved in 96.
// Planning is one workgroup's for take and fork: 1024 entries and 8192 counts in each of its passes. The plan of a compaction
// is a workgroup's per 8192 pages, each of which counts all pages itself: pages^2 / 1024 bytes in all, mostly from L2, 0.1 MB
// for ten thousand pages and 1 GB for a million.
#include "mh3_common.hpp"

#include <algorithm>

namespace mh3 {
namespace {

struct Table {
    int32_t* entries;
    uint64_t stride; // ints from a stream's first entry to the next one's
    uint32_t streams, cols, pages;
    __device__ __forceinline__ int32_t& at(uint32_t s, uint32_t e) const { return entries[uint64_t(s) * stride + e]; }
    __device__ __forceinline__ bool page(int32_t p) const { return uint32_t(p) < pages; }
};

struct Pools {
    MH3Pool pool[MH3_MAX_POOLS];
    uint32_t first[MH3_MAX_POOLS + 1]; // chunks of a page in the pools before
    uint32_t n;
};

constexpr uint32_t kChunk = 32768; // bytes of a page that a workgroup copies at a time, eight vectors a thread

// Chunk c of page src to page dst, by 256 threads.
__device__ __forceinline__ void copy_chunk(const Pools& pools, uint32_t c, uint32_t src, uint32_t dst)
{
    uint32_t i = 0;
    while (c >= pools.first[i + 1u])
        ++i;
    const MH3Pool& p = pools.pool[i];
    const uint64_t at = uint64_t(c - pools.first[i]) * kChunk;
    const uint32_t n = uint32_t(min(uint64_t(kChunk), p.page_bytes - at)) / 16u;
    const uint4* const from = reinterpret_cast<const uint4*>(static_cast<const char*>(p.base) + src * p.page_stride + at);
    uint4* const to = reinterpret_cast<uint4*>(static_cast<char*>(p.base) + dst * p.page_stride + at);
    if (n == kChunk / 16u) {
        uint4 t[8];
#pragma unroll
        for (uint32_t u = 0; u < 8u; ++u)
            t[u] = ld_stream(from + 256u * u + threadIdx.x);
#pragma unroll
        for (uint32_t u = 0; u < 8u; ++u)
            st_stream(to + 256u * u + threadIdx.x, t[u]);
    } else {
        for (uint32_t u = threadIdx.x; u < n; u += 256u)
            to[u] = from[u];
    }
}

// ---- taking pages ----------------------------------------------------------------------------------------------------

constexpr uint32_t kTakers = 1024, kWaves = kTakers / 64;
constexpr uint32_t kScan = 8192; // counts looked at in one go, eight a thread

struct TakeShared {
    uint32_t wave[kWaves];
    int32_t queue[kTakers + kScan]; // the lowest free pages that are not given yet
};

// The exclusive sum of v over the workgroup's threads, and the total.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t& total, uint32_t* wave_sums)
{
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t before = wave_excl_scan_u32(v);
    if (lane == 63u)
        wave_sums[wave] = before + v;
    __syncthreads();
    uint32_t base = 0;
    total = 0;
#pragma unroll
    for (uint32_t i = 0; i < kWaves; ++i) {
        const uint32_t t = wave_sums[i];
        base += i < wave ? t : 0u;
        total += t;
    }
    __syncthreads();
    return base + before;
}

// Gives the lowest free pages to those of the items j < n that want(j) one, in order: give(j, page), by one workgroup of
// kTakers threads. Returns how many found none (give(j, -1)).
template <class Want, class Give>
__device__ __forceinline__ uint32_t take_lowest(const int32_t* refs, uint32_t pages, uint32_t n, TakeShared& sh,
                                                const Want& want, const Give& give)
{
    uint32_t scanned = 0, held = 0, missing = 0;
    for (uint32_t j0 = 0; j0 < n; j0 += kTakers) {
        const uint32_t j = j0 + threadIdx.x;
        const bool wants = j < n && want(j);
        uint32_t total;
        const uint32_t rank = block_scan(wants, total, sh.wave);
        while (held < total && scanned < pages) {
            const uint32_t first = scanned + 8u * threadIdx.x;
            uint32_t bits = 0;
#pragma unroll
            for (uint32_t u = 0; u < 8u; ++u)
                bits |= first + u < pages && refs[first + u] == 0 ? 1u << u : 0u;
            uint32_t found;
            uint32_t at = held + block_scan(__popc(bits), found, sh.wave);
            for (; bits; bits &= bits - 1u)
                sh.queue[at++] = int32_t(first + __builtin_ctz(bits));
            held += found, scanned += min(kScan, pages - scanned);
        }
        __syncthreads();
        if (wants)
            give(j, rank < held ? sh.queue[rank] : -1);
        const uint32_t given = min(held, total);
        missing += total - given;
        // The rest of the queue to its front. (held < kTakers + kScan: it grows only while it is below a block's wants.)
        int32_t keep[(kTakers + kScan) / kTakers];
        __syncthreads();
#pragma unroll
        for (uint32_t u = 0; u < (kTakers + kScan) / kTakers; ++u) {
            const uint32_t i = given + u * kTakers + threadIdx.x;
            keep[u] = i < held ? sh.queue[i] : -1;
        }
        __syncthreads();
        held -= given;
#pragma unroll
        for (uint32_t u = 0; u < (kTakers + kScan) / kTakers; ++u)
            if (u * kTakers + threadIdx.x < held)
                sh.queue[u * kTakers + threadIdx.x] = keep[u];
        __syncthreads();
    }
    return missing;
}

__device__ __forceinline__ void span_of(const Table& t, const int32_t* first, const int32_t* last, uint32_t s, uint32_t& a,
                                        uint32_t& b)
{
    a = uint32_t(min(max(first[s], 0), int32_t(t.cols)));
    b = uint32_t(min(max(last[s], int32_t(a)), int32_t(t.cols)));
}

// One workgroup: the entries of all streams' spans are one list, found in it through the sums of the spans' lengths.
__global__ __launch_bounds__(kTakers) void pages_take_kernel(Table t, int32_t* refs, const int32_t* first,
                                                             const int32_t* last, int32_t* missing)
{
    __shared__ TakeShared sh;
    __shared__ uint32_t begin[MH3_MAX_STREAMS + 1], start[MH3_MAX_STREAMS];
    uint32_t n = 0;
    for (uint32_t s0 = 0; s0 < t.streams; s0 += kTakers) {
        const uint32_t s = s0 + threadIdx.x;
        uint32_t a = 0, b = 0, total;
        if (s < t.streams)
            span_of(t, first, last, s, a, b);
        const uint32_t at = n + block_scan(b - a, total, sh.wave);
        if (s < t.streams)
            begin[s] = at, start[s] = a;
        n += total;
    }
    if (threadIdx.x == 0)
        begin[t.streams] = n;
    __syncthreads();
    const auto entry = [&](uint32_t j) -> int32_t& {
        uint32_t a = 0, b = t.streams; // begin[a] <= j < begin[b]
        while (b - a > 1u) {
            const uint32_t mid = (a + b) / 2u;
            if (begin[mid] <= j)
                a = mid;
            else
                b = mid;
        }
        return t.at(a, start[a] + j - begin[a]);
    };
    const uint32_t none = take_lowest(
        refs, t.pages, n, sh, [&](uint32_t j) { return !t.page(entry(j)); },
        [&](uint32_t j, int32_t page) {
            entry(j) = page;
            if (page >= 0)
                refs[page] = 1; // behind what has been scanned: it is not looked at again
        });
    if (threadIdx.x == 0 && missing)
        *missing = int32_t(none);
}

__global__ __launch_bounds__(256) void pages_free_kernel(Table t, int32_t* refs, const int32_t* first, const int32_t* last,
                                                         FastDiv div_cols)
{
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= t.streams * t.cols)
        return;
    const uint32_t s = div_cols.div(i), e = i - s * t.cols;
    uint32_t a, b;
    span_of(t, first, last, s, a, b);
    if (e < a || e >= b)
        return;
    int32_t& entry = t.at(s, e);
    if (t.page(entry))
        atomicSub(refs + entry, 1);
    entry = -1;
}

// ---- forking ---------------------------------------------------------------------------------------------------------

struct ForkParams {
    Table old, fresh; // fresh: the new table
    int32_t* refs;
    const int32_t* parents;
    const int32_t* rows;
    int2* moves; // each stream's page that was begun: from, to (-1: none)
    int32_t* missing;
    uint32_t page_rows;
    FastDiv div_rows, div_cols;
};

// Whether stream s goes on from another one's row (or from none: parent past the table).
__device__ __forceinline__ bool forks(const ForkParams& p, uint32_t s, uint32_t& parent)
{
    parent = uint32_t(p.parents[s]); // a negative one is past every table
    return parent != s;
}

// The full pages that stream s shares, and whether it has begun another.
__device__ __forceinline__ uint32_t full_pages(const ForkParams& p, uint32_t s, bool& begun)
{
    const uint32_t rows = uint32_t(max(p.rows[s], 0)), full = p.div_rows.div(rows);
    begun = rows != full * p.page_rows;
    return full;
}

__global__ __launch_bounds__(kTakers) void pages_fork_plan_kernel(ForkParams p)
{
    __shared__ TakeShared sh;
    const auto begun_page = [&](uint32_t s) {
        uint32_t parent;
        bool begun = false;
        if (!forks(p, s, parent) || parent >= p.old.streams)
            return -1;
        const uint32_t full = full_pages(p, s, begun);
        const int32_t page = begun && full < p.old.cols ? p.old.at(parent, full) : -1;
        return p.old.page(page) ? page : -1;
    };
    for (uint32_t s = threadIdx.x; s < p.old.streams; s += kTakers)
        p.moves[s] = int2{-1, -1};
    const uint32_t none = take_lowest(
        p.refs, p.old.pages, p.old.streams, sh, [&](uint32_t s) { return begun_page(s) >= 0; },
        [&](uint32_t s, int32_t page) {
            p.moves[s] = int2{begun_page(s), page}; // the same thread cleared it
            if (page >= 0)
                p.refs[page] = 1;
        });
    if (threadIdx.x == 0 && p.missing)
        *p.missing = int32_t(none);
}

// The first table_blocks workgroups write the new table and count, the others copy the pages that were begun. A page that
// this call leaves without an entry may be copied from here while its count falls to zero: no page that was in use before
// the call is taken by it.
__global__ __launch_bounds__(256) void pages_fork_kernel(ForkParams p, Pools pools, uint32_t table_blocks)
{
    if (blockIdx.x >= table_blocks) {
        const uint32_t chunks = pools.first[pools.n];
        for (uint64_t i = blockIdx.x - table_blocks; i < uint64_t(chunks) * p.old.streams; i += gridDim.x - table_blocks) {
            const uint32_t s = uint32_t(i / chunks);
            const int2 m = p.moves[s];
            if (m.y >= 0)
                copy_chunk(pools, uint32_t(i - uint64_t(s) * chunks), uint32_t(m.x), uint32_t(m.y));
        }
        return;
    }
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= p.old.streams * p.old.cols)
        return;
    const uint32_t s = p.div_cols.div(i), e = i - s * p.old.cols;
    const int32_t before = p.old.at(s, e);
    uint32_t parent;
    if (!forks(p, s, parent)) {
        p.fresh.at(s, e) = before;
        return;
    }
    int32_t now = -1;
    if (parent < p.old.streams) {
        bool begun;
        const uint32_t full = full_pages(p, s, begun);
        if (e < full) {
            now = p.old.at(parent, e);
            if (p.old.page(now))
                atomicAdd(p.refs + now, 1);
            else
                now = -1;
        } else if (e == full && begun) {
            now = p.moves[s].y;
        }
    }
    p.fresh.at(s, e) = now;
    if (p.old.page(before))
        atomicSub(p.refs + before, 1);
}

// ---- copying ---------------------------------------------------------------------------------------------------------

// A workgroup takes a run of the pairs' chunks. A pair whose destination is a page that the call also copies from, or an
// earlier pair's destination, is passed over: the lists are searched once for each pair that a workgroup meets (512 pairs:
// nothing measurable; 16,384: about as long as 32 KB of its copying).
__global__ __launch_bounds__(256) void pages_copy_kernel(Pools pools, const int32_t* src, const int32_t* dst, uint32_t n,
                                                         uint32_t pages)
{
    const uint32_t chunks = pools.first[pools.n];
    const uint64_t items = uint64_t(chunks) * n;
    const uint64_t begin = items * blockIdx.x / gridDim.x, end = items * (blockIdx.x + 1ull) / gridDim.x;
    for (uint64_t i = begin; i < end;) {
        const uint32_t pair = uint32_t(i / chunks);
        const uint32_t c0 = uint32_t(i - uint64_t(pair) * chunks);
        const uint32_t c1 = uint32_t(min(uint64_t(chunks), c0 + (end - i)));
        const int32_t from = src[pair], to = dst[pair];
        bool clash = uint32_t(from) >= pages || uint32_t(to) >= pages;
        for (uint32_t j = threadIdx.x; j < n; j += 256u)
            clash |= src[j] == to || (j < pair && dst[j] == to);
        if (!__syncthreads_or(clash))
            for (uint32_t c = c0; c < c1; ++c)
                copy_chunk(pools, c, uint32_t(from), uint32_t(to));
        i += c1 - c0;
    }
}

// ---- compacting ------------------------------------------------------------------------------------------------------

struct CompactParams {
    Table table;
    int32_t* refs;
    int32_t* map;    // int32 [pages]: each page's new number, -1 for a free one
    int32_t* used;   // how many are in use
    int32_t* moves;  // how many move
    int32_t* holes;  // the free pages below `used`, in order
    int32_t* strays; // the pages in use past it, in order
    FastDiv div_cols;
};

// Used pages among the counts [first, last), by all threads of the workgroup.
__device__ __forceinline__ uint32_t count_used(const int32_t* refs, uint32_t first, uint32_t last, uint32_t* wave_sums)
{
    uint32_t n = 0, total;
    for (uint32_t i = first + threadIdx.x; i < last; i += kTakers)
        n += refs[i] > 0 ? 1u : 0u;
    block_scan(n, total, wave_sums);
    return total;
}

// A workgroup plans the moves of kScan pages. It counts the pages before and behind its own by itself: the loads do not
// wait for each other, and nothing waits for another workgroup.
__global__ __launch_bounds__(kTakers) void pages_compact_plan_kernel(CompactParams p)
{
    __shared__ uint32_t wave_sums[kWaves];
    const uint32_t pages = p.table.pages, first = blockIdx.x * kScan, last = min(first + kScan, pages);
    const uint32_t before = count_used(p.refs, 0u, first, wave_sums);
    const uint32_t used = before + count_used(p.refs, first, pages, wave_sums);
    const uint32_t low = count_used(p.refs, 0u, used, wave_sums); // of them below `used`
    const uint32_t i0 = first + 8u * threadIdx.x;
    uint32_t bits = 0;
#pragma unroll
    for (uint32_t u = 0; u < 8u; ++u)
        bits |= i0 + u < last && p.refs[i0 + u] > 0 ? 1u << u : 0u;
    uint32_t total;
    uint32_t rank = before + block_scan(__popc(bits), total, wave_sums);
#pragma unroll
    for (uint32_t u = 0; u < 8u; ++u) {
        const uint32_t i = i0 + u;
        if (i >= last)
            break;
        if (bits >> u & 1u) {
            p.map[i] = i < used ? int32_t(i) : -2 - int32_t(rank - low); // past it: the hole's number, looked up later
            if (i >= used)
                p.strays[rank - low] = int32_t(i);
            ++rank;
        } else {
            p.map[i] = -1;
            if (i < used)
                p.holes[i - rank] = int32_t(i);
        }
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        *p.moves = int32_t(used - low);
        if (p.used)
            *p.used = int32_t(used);
    }
}

// The first table_blocks workgroups turn the table's entries, the next page_blocks move the counts and end the map, the
// others move the pages. What one of them reads of the map while another ends it says the same either way.
__global__ __launch_bounds__(256) void pages_compact_kernel(CompactParams p, Pools pools, uint32_t table_blocks,
                                                            uint32_t page_blocks)
{
    uint32_t block = blockIdx.x;
    const uint32_t moves = uint32_t(*p.moves);
    if (block < table_blocks) {
        const uint32_t i = block * 256u + threadIdx.x;
        if (i >= p.table.streams * p.table.cols)
            return;
        const uint32_t s = p.div_cols.div(i);
        int32_t& entry = p.table.at(s, i - s * p.table.cols);
        const int32_t old = entry;
        if (old == -1)
            return;
        int32_t now = p.table.page(old) ? __atomic_load_n(p.map + old, __ATOMIC_RELAXED) : -1;
        if (now <= -2)
            now = p.holes[-2 - now];
        if (now != old)
            entry = now;
        return;
    }
    block -= table_blocks;
    if (block < page_blocks) {
        const uint32_t i = block * 256u + threadIdx.x;
        if (i < moves) {
            const int32_t from = p.strays[i], to = p.holes[i];
            __atomic_store_n(p.map + from, to, __ATOMIC_RELAXED);
            p.refs[to] = p.refs[from];
            p.refs[from] = 0;
        }
        return;
    }
    block -= page_blocks;
    const uint32_t chunks = pools.first[pools.n], blocks = gridDim.x - table_blocks - page_blocks;
    for (uint64_t i = block; i < uint64_t(chunks) * moves; i += blocks) {
        const uint32_t move = uint32_t(i / chunks);
        copy_chunk(pools, uint32_t(i - uint64_t(move) * chunks), uint32_t(p.strays[move]), uint32_t(p.holes[move]));
    }
}

// ---- writing ---------------------------------------------------------------------------------------------------------

struct WriteParams {
    const uint16_t* k;
    const uint16_t* v;
    uint16_t* k_pages;
    uint16_t* v_pages;
    Table table;
    const int32_t* starts;
    const int32_t* off;
    const int32_t* rows;
    uint64_t khs, krs, vhs, vrs, kps, kphs, kprs, vps, vphs, vprs; // elements
    uint32_t kv_heads, n_rows, n, page_rows;
    FastDiv div_rows, div_heads;
};

// 16 threads a head's row of k and v.
__global__ __launch_bounds__(256) void pages_write_kernel(WriteParams p)
{
    const uint32_t i = blockIdx.x * 16u + threadIdx.x / 16u, c = 8u * (threadIdx.x % 16u);
    const uint32_t j = p.div_heads.div(i), head = i - j * p.kv_heads;
    if (j >= p.n)
        return;
    uint32_t a = 0, b = p.table.streams; // off[a - 1] <= j < off[b] in a sorted list
    while (a < b) {
        const uint32_t mid = (a + b) / 2u;
        if (p.off[mid + 1u] <= int32_t(j))
            a = mid + 1u;
        else
            b = mid;
    }
    if (a >= p.table.streams || p.off[a] > int32_t(j))
        return;
    const uint32_t row = p.rows ? uint32_t(p.rows[j]) : j;
    const int64_t place = int64_t(p.starts[a]) + j - p.off[a];
    if (row >= p.n_rows || place < 0 || place >= int64_t(p.table.cols) * p.page_rows)
        return;
    const uint32_t e = p.div_rows.div(uint32_t(place)), r = uint32_t(place) - e * p.page_rows;
    const int32_t page = p.table.at(a, e);
    if (!p.table.page(page))
        return;
    const uint4 k = *reinterpret_cast<const uint4*>(p.k + head * p.khs + row * p.krs + c);
    const uint4 v = *reinterpret_cast<const uint4*>(p.v + head * p.vhs + row * p.vrs + c);
    *reinterpret_cast<uint4*>(p.k_pages + uint32_t(page) * p.kps + head * p.kphs + r * p.kprs + c) = k;
    *reinterpret_cast<uint4*>(p.v_pages + uint32_t(page) * p.vps + head * p.vphs + r * p.vprs + c) = v;
}

} // namespace
} // namespace mh3

namespace {

using namespace mh3;

bool aligned4(const void* p) { return reinterpret_cast<uintptr_t>(p) % 4u == 0u; }

int check_table(const MH3PagesArgs* args)
{
    if (!args)
        return MH3_ERR_POINTER;
    const MH3PagesArgs& a = *args;
    if (a.streams == 0 || a.streams > MH3_MAX_STREAMS || a.cols == 0 || a.cols >= (1u << 24) || a.pages == 0 ||
        a.pages >= (1u << 24) || a.table_stride < a.cols || a.table_stride >= (1ull << 32) ||
        uint64_t(a.streams) * a.cols >= (1ull << 30))
        return MH3_ERR_SHAPE;
    return MH3_OK;
}

uint64_t table_bytes(const MH3PagesArgs& a) { return ((a.streams - 1ull) * a.table_stride + a.cols) * 4u; }

Table table_of(const MH3PagesArgs& a, int32_t* entries)
{
    return Table{entries, a.table_stride, a.streams, a.cols, a.pages};
}

uint64_t pool_span(const MH3Pool& p, uint32_t pages) { return (pages - 1ull) * p.page_stride + p.page_bytes; }

int check_pools(const MH3Pool* pools, uint32_t n, uint32_t pages, Pools& out)
{
    if (n > MH3_MAX_POOLS)
        return MH3_ERR_SHAPE;
    if (n && !pools)
        return MH3_ERR_POINTER;
    out = Pools{};
    out.n = n;
    uint64_t chunks = 0;
    for (uint32_t i = 0; i < n; ++i) {
        const MH3Pool& p = pools[i];
        if (!p.base)
            return MH3_ERR_POINTER;
        if (!host::aligned16(p.base) || p.page_bytes % 16u != 0 || p.page_stride % 16u != 0)
            return MH3_ERR_ALIGN;
        if (p.page_bytes == 0 || p.page_stride < p.page_bytes || p.page_stride >= (1ull << 39))
            return MH3_ERR_SHAPE;
        for (uint32_t j = 0; j < i; ++j)
            if (host::overlaps(p.base, pool_span(p, pages), pools[j].base, pool_span(pools[j], pages)))
                return MH3_ERR_PARAM;
        out.pool[i] = p;
        chunks += (p.page_bytes + kChunk - 1u) / kChunk;
        if (chunks >= (1ull << 31))
            return MH3_ERR_SHAPE;
        out.first[i + 1u] = uint32_t(chunks);
    }
    return MH3_OK;
}

// Whether any of the tables and lists lies in a pool.
template <size_t N>
bool in_pools(const Pools& pools, uint32_t pages, const host::Span (&spans)[N])
{
    for (uint32_t i = 0; i < pools.n; ++i)
        for (const host::Span& s : spans)
            if (s.p && host::overlaps(s.p, s.n, pools.pool[i].base, pool_span(pools.pool[i], pages)))
                return true;
    return false;
}

// How often something repeats, and elements from one to the next.
struct Repeat {
    uint64_t n, stride;
};

// Whether rows of 128 elements that repeat so lie apart: from the smallest stride to the largest, each steps over all that
// the smaller ones span. The other layouts without a shared element (strides that miss each other by their factors) are no
// nest of dimensions, and count as none.
template <size_t N>
bool rows_apart(Repeat (&dims)[N])
{
    std::sort(dims, dims + N, [](const Repeat& a, const Repeat& b) { return a.stride < b.stride; });
    uint64_t span = 128;
    for (const Repeat& d : dims) {
        if (d.n <= 1u)
            continue;
        if (d.stride < span)
            return false;
        span += (d.n - 1u) * d.stride;
    }
    return true;
}

// Whether two pools of the same strides, `offset` elements apart, share none: a pair of such rows repeats as they do, and
// seen from any repetition of the largest stride the other pool's rows are its remainder on, or as many short of the next.
bool pools_apart(uint64_t pages, uint64_t page, uint64_t heads, uint64_t head, uint64_t rows, uint64_t row, uint64_t offset)
{
    Repeat dims[] = {{pages, page}, {heads, head}, {rows, row}};
    uint64_t largest = 0, span = 128;
    for (const Repeat& d : dims)
        if (d.n > 1u)
            largest = std::max(largest, d.stride), span += (d.n - 1u) * d.stride;
    if (offset >= span)
        return true;
    const uint64_t on = largest ? offset % largest : offset;
    for (const uint64_t step : {on, largest > on ? largest - on : on}) {
        Repeat all[] = {{2u, step}, dims[0], dims[1], dims[2]};
        if (rows_apart(all))
            return true;
    }
    return false;
}

uint32_t copy_blocks(uint64_t items) { return uint32_t(std::min<uint64_t>(items, 8u * uint64_t(host::cu_count()))); }

} // namespace

extern "C" int mh3_pages_take(const MH3PagesArgs* args, int32_t* table, int32_t* refs, const int32_t* first,
                              const int32_t* last, int32_t* missing, mh3_stream_t stream)
{
    if (const int rc = check_table(args); rc != MH3_OK)
        return rc;
    if (!table || !refs || !first || !last)
        return MH3_ERR_POINTER;
    if (!aligned4(table) || !aligned4(refs) || !aligned4(first) || !aligned4(last) || !aligned4(missing))
        return MH3_ERR_ALIGN;
    const host::Span in[] = {{first, args->streams * 4ull}, {last, args->streams * 4ull}};
    const host::Span out[] = {{table, table_bytes(*args)}, {refs, args->pages * 4ull}, {missing, 4u}};
    if (host::any_overlap(in, out))
        return MH3_ERR_PARAM;
    hipLaunchKernelGGL(pages_take_kernel, dim3(1), dim3(kTakers), 0, static_cast<hipStream_t>(stream),
                       table_of(*args, table), refs, first, last, missing);
    return host::check_launch();
}

extern "C" int mh3_pages_free(const MH3PagesArgs* args, int32_t* table, int32_t* refs, const int32_t* first,
                              const int32_t* last, mh3_stream_t stream)
{
    if (const int rc = check_table(args); rc != MH3_OK)
        return rc;
    if (!table || !refs || !first || !last)
        return MH3_ERR_POINTER;
    if (!aligned4(table) || !aligned4(refs) || !aligned4(first) || !aligned4(last))
        return MH3_ERR_ALIGN;
    const host::Span in[] = {{first, args->streams * 4ull}, {last, args->streams * 4ull}};
    const host::Span out[] = {{table, table_bytes(*args)}, {refs, args->pages * 4ull}};
    if (host::any_overlap(in, out))
        return MH3_ERR_PARAM;
    hipLaunchKernelGGL(pages_free_kernel, dim3((args->streams * args->cols + 255u) / 256u), dim3(256), 0,
                       static_cast<hipStream_t>(stream), table_of(*args, table), refs, first, last,
                       FastDiv::make(args->cols));
    return host::check_launch();
}

extern "C" int64_t mh3_pages_fork_workspace_bytes(const MH3PagesArgs* args)
{
    if (const int rc = check_table(args); rc != MH3_OK)
        return rc;
    return int64_t(args->streams) * 8;
}

extern "C" int mh3_pages_fork(const MH3PagesArgs* args, const MH3Pool* pools, uint32_t n_pools, const int32_t* table,
                              int32_t* refs, const int32_t* parents, const int32_t* rows, int32_t* new_table,
                              int32_t* missing, void* workspace, uint64_t workspace_bytes, mh3_stream_t stream)
{
    if (const int rc = check_table(args); rc != MH3_OK)
        return rc;
    const MH3PagesArgs& a = *args;
    if (a.page_rows == 0 || a.page_rows >= (1u << 30))
        return MH3_ERR_SHAPE;
    if (!table || !refs || !parents || !rows || !new_table || !workspace)
        return MH3_ERR_POINTER;
    if (!aligned4(table) || !aligned4(refs) || !aligned4(parents) || !aligned4(rows) || !aligned4(new_table) ||
        !aligned4(missing) || !host::aligned16(workspace))
        return MH3_ERR_ALIGN;
    if (workspace_bytes < a.streams * 8ull)
        return MH3_ERR_SHAPE;
    Pools held;
    if (const int rc = check_pools(pools, n_pools, a.pages, held); rc != MH3_OK)
        return rc;
    const host::Span in[] = {{table, table_bytes(a)}, {parents, a.streams * 4ull}, {rows, a.streams * 4ull}};
    const host::Span out[] = {{new_table, table_bytes(a)}, {refs, a.pages * 4ull}, {missing, 4u},
                              {workspace, a.streams * 8ull}};
    if (host::any_overlap(in, out) || in_pools(held, a.pages, in) || in_pools(held, a.pages, out))
        return MH3_ERR_PARAM;
    ForkParams p{};
    p.old = table_of(a, const_cast<int32_t*>(table)), p.fresh = table_of(a, new_table);
    p.refs = refs, p.parents = parents, p.rows = rows, p.moves = static_cast<int2*>(workspace), p.missing = missing;
    p.page_rows = a.page_rows, p.div_rows = FastDiv::make(a.page_rows), p.div_cols = FastDiv::make(a.cols);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(pages_fork_plan_kernel, dim3(1), dim3(kTakers), 0, s, p);
    if (const int rc = host::check_launch(); rc != MH3_OK)
        return rc;
    const uint32_t table_blocks = (a.streams * a.cols + 255u) / 256u;
    const uint32_t blocks = table_blocks + copy_blocks(uint64_t(held.first[held.n]) * a.streams);
    hipLaunchKernelGGL(pages_fork_kernel, dim3(blocks), dim3(256), 0, s, p, held, table_blocks);
    return host::check_launch();
}

extern "C" int mh3_pages_copy(const MH3Pool* pools, uint32_t n_pools, uint32_t pages, const int32_t* src,
                              const int32_t* dst, uint32_t n, mh3_stream_t stream)
{
    if (pages == 0 || pages >= (1u << 24) || n > MH3_MAX_PAIRS)
        return MH3_ERR_SHAPE;
    Pools held;
    if (const int rc = check_pools(pools, n_pools, pages, held); rc != MH3_OK)
        return rc;
    if (n == 0 || n_pools == 0)
        return MH3_OK;
    if (!src || !dst)
        return MH3_ERR_POINTER;
    if (!aligned4(src) || !aligned4(dst))
        return MH3_ERR_ALIGN;
    const host::Span in[] = {{src, n * 4ull}, {dst, n * 4ull}};
    if (in_pools(held, pages, in))
        return MH3_ERR_PARAM;
    hipLaunchKernelGGL(pages_copy_kernel, dim3(copy_blocks(uint64_t(held.first[held.n]) * n)), dim3(256), 0,
                       static_cast<hipStream_t>(stream), held, src, dst, n, pages);
    return host::check_launch();
}

extern "C" int64_t mh3_pages_compact_workspace_bytes(const MH3PagesArgs* args)
{
    if (const int rc = check_table(args); rc != MH3_OK)
        return rc;
    return 16 + int64_t(args->pages / 2u) * 8; // as many holes below the end as pages past it: half of them at most
}

extern "C" int mh3_pages_compact(const MH3PagesArgs* args, const MH3Pool* pools, uint32_t n_pools, int32_t* table,
                                 int32_t* refs, int32_t* map, int32_t* used, void* workspace, uint64_t workspace_bytes,
                                 mh3_stream_t stream)
{
    const int64_t need = mh3_pages_compact_workspace_bytes(args);
    if (need < 0)
        return int(need);
    const MH3PagesArgs& a = *args;
    if (!table || !refs || !map || !workspace)
        return MH3_ERR_POINTER;
    if (!aligned4(table) || !aligned4(refs) || !aligned4(map) || !aligned4(used) || !host::aligned16(workspace))
        return MH3_ERR_ALIGN;
    if (workspace_bytes < uint64_t(need))
        return MH3_ERR_SHAPE;
    Pools held;
    if (const int rc = check_pools(pools, n_pools, a.pages, held); rc != MH3_OK)
        return rc;
    const host::Span in[] = {{nullptr, 0u}};
    const host::Span out[] = {{table, table_bytes(a)}, {refs, a.pages * 4ull}, {map, a.pages * 4ull}, {used, 4u},
                              {workspace, uint64_t(need)}};
    if (host::any_overlap(in, out) || in_pools(held, a.pages, out))
        return MH3_ERR_PARAM;
    int32_t* const ws = static_cast<int32_t*>(workspace);
    const CompactParams p{table_of(a, table), refs, map, used, ws, ws + 4, ws + 4 + a.pages / 2u, FastDiv::make(a.cols)};
    const hipStream_t s = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(pages_compact_plan_kernel, dim3((a.pages + kScan - 1u) / kScan), dim3(kTakers), 0, s, p);
    if (const int rc = host::check_launch(); rc != MH3_OK)
        return rc;
    const uint32_t table_blocks = (a.streams * a.cols + 255u) / 256u, page_blocks = (a.pages / 2u + 255u) / 256u;
    const uint32_t blocks = table_blocks + page_blocks + copy_blocks(uint64_t(held.first[held.n]) * (a.pages / 2u));
    hipLaunchKernelGGL(pages_compact_kernel, dim3(blocks), dim3(256), 0, s, p, held, table_blocks, page_blocks);
    return host::check_launch();
}

extern "C" int mh3_pages_write(const MH3PagesWriteArgs* args, const uint16_t* k, const uint16_t* v, uint16_t* k_pages,
                               uint16_t* v_pages, const int32_t* table, const int32_t* starts, const int32_t* off,
                               const int32_t* rows, mh3_stream_t stream)
{
    if (!args)
        return MH3_ERR_POINTER;
    const MH3PagesWriteArgs& a = *args;
    if (const int rc = check_table(&a.table); rc != MH3_OK)
        return rc;
    if (a.kv_heads == 0 || a.kv_heads > 4096u || a.head_dim == 0 || a.table.page_rows == 0 ||
        uint64_t(a.table.cols) * a.table.page_rows >= (1ull << 30) || a.n_rows >= (1u << 30) ||
        uint64_t(a.n) * a.kv_heads >= (1ull << 31))
        return MH3_ERR_SHAPE;
    if (a.head_dim != 128u)
        return MH3_ERR_UNSUPPORTED;
    for (const uint64_t s : {a.k_row_stride, a.v_row_stride, a.k_page_row_stride, a.v_page_row_stride}) {
        if (s % 8u != 0)
            return MH3_ERR_ALIGN;
        if (s < 128u || s >= (1ull << 23))
            return MH3_ERR_SHAPE;
    }
    for (const uint64_t s : {a.k_head_stride, a.v_head_stride, a.k_page_stride, a.v_page_stride, a.k_page_head_stride,
                             a.v_page_head_stride}) {
        if (s % 8u != 0)
            return MH3_ERR_ALIGN;
        if (s >= (1ull << 36))
            return MH3_ERR_SHAPE;
    }
    // A pool's rows apart from each other, as out's of the attention.
    Repeat kd[] = {{a.table.pages, a.k_page_stride}, {a.kv_heads, a.k_page_head_stride}, {a.table.page_rows, a.k_page_row_stride}};
    Repeat vd[] = {{a.table.pages, a.v_page_stride}, {a.kv_heads, a.v_page_head_stride}, {a.table.page_rows, a.v_page_row_stride}};
    if (!rows_apart(kd) || !rows_apart(vd))
        return MH3_ERR_PARAM;
    if (a.n == 0 || a.n_rows == 0)
        return MH3_OK;
    if (!k || !v || !k_pages || !v_pages || !table || !starts || !off)
        return MH3_ERR_POINTER;
    // And from the other pool's, where both have the same strides; else only the same pool twice is told.
    const uint64_t from = reinterpret_cast<uintptr_t>(k_pages), to = reinterpret_cast<uintptr_t>(v_pages);
    if (from == to || (a.k_page_stride == a.v_page_stride && a.k_page_head_stride == a.v_page_head_stride &&
                       a.k_page_row_stride == a.v_page_row_stride &&
                       !pools_apart(a.table.pages, a.k_page_stride, a.kv_heads, a.k_page_head_stride, a.table.page_rows,
                                    a.k_page_row_stride, (from < to ? to - from : from - to) / 2u)))
        return MH3_ERR_PARAM;
    if (!host::aligned16(k) || !host::aligned16(v) || !host::aligned16(k_pages) || !host::aligned16(v_pages) ||
        !aligned4(table) || !aligned4(starts) || !aligned4(off) || !aligned4(rows))
        return MH3_ERR_ALIGN;
    const auto pool = [&](uint64_t ps, uint64_t hs, uint64_t rs) {
        return ((a.table.pages - 1u) * ps + (a.kv_heads - 1u) * hs + (a.table.page_rows - 1u) * rs + 128u) * 2u;
    };
    const auto span = [&](uint64_t hs, uint64_t rs) { return ((a.kv_heads - 1u) * hs + (a.n_rows - 1u) * rs + 128u) * 2u; };
    const host::Span in[] = {{k, span(a.k_head_stride, a.k_row_stride)},
                             {v, span(a.v_head_stride, a.v_row_stride)},
                             {table, table_bytes(a.table)},
                             {starts, a.table.streams * 4ull},
                             {off, (a.table.streams + 1ull) * 4u},
                             {rows, a.n * 4ull}};
    // Each pool by itself: those of a layer's keys and values may lie in one another's gaps.
    const host::Span ko[] = {{k_pages, pool(a.k_page_stride, a.k_page_head_stride, a.k_page_row_stride)}};
    const host::Span vo[] = {{v_pages, pool(a.v_page_stride, a.v_page_head_stride, a.v_page_row_stride)}};
    if (host::any_overlap(in, ko) || host::any_overlap(in, vo))
        return MH3_ERR_PARAM;
    WriteParams p{};
    p.k = k, p.v = v, p.k_pages = k_pages, p.v_pages = v_pages;
    p.table = table_of(a.table, const_cast<int32_t*>(table)), p.starts = starts, p.off = off, p.rows = rows;
    p.khs = a.k_head_stride, p.krs = a.k_row_stride, p.vhs = a.v_head_stride, p.vrs = a.v_row_stride;
    p.kps = a.k_page_stride, p.kphs = a.k_page_head_stride, p.kprs = a.k_page_row_stride;
    p.vps = a.v_page_stride, p.vphs = a.v_page_head_stride, p.vprs = a.v_page_row_stride;
    p.kv_heads = a.kv_heads, p.n_rows = a.n_rows, p.n = a.n, p.page_rows = a.table.page_rows;
    p.div_rows = FastDiv::make(a.table.page_rows), p.div_heads = FastDiv::make(a.kv_heads);
    hipLaunchKernelGGL(pages_write_kernel, dim3((a.n * a.kv_heads + 15u) / 16u), dim3(256), 0,
                       static_cast<hipStream_t>(stream), p);
    return host::check_launch();
}
