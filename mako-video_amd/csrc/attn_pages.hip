// `flash_attn_pages_128`: attention of streams' new rows (a single one each, a tree of drafted ones, a chunk) over their kept
// rows in pages and over themselves, head_dim 128, bf16 in and out, with a window and first rows that stay in sight.
//   row i of a stream with L kept rows has place L + depth(i), depth the number of its ancestors (without parents: i);
//   it attends kept row j if j < L and (j < sinks or j > place_i - window), and new row i' if that is i or one of its
//   ancestors (without parents: i' <= i) and (place_i' < sinks or place_i' > place_i - window);
//   s = scale q.k, under a cap cap tanh(s / cap); out_i = sum softmax(s)[j] v_j.
//
// Design (the tiles, rows and softmax of attn_tiles.hpp, as attn_dense.hip describes them):
// - A stream's query heads that share a key head are rows of one list, f = row group + g; an item is 32 of them, a key head
//   and the tiles of 64 keys that they attend: those of the first rows, those of the window, those of the new rows, these
//   from the last to the first.
// - A tile is four groups of 16 rows, each in one page: four descriptors, of as many rows as there are and none where the
//   entry is no page, so that nothing else is read and what is missing is zeros. The page numbers of 16 tiles lie in the
//   lanes of one register, 16 entries read at once, and come out of it by readlane.
// - With few list rows a stream a workgroup is one wave with 32 of them; with more it is eight waves of 32, which share their
//   tiles and take turns at products and softmax as in attn_dense.hip.
// - What a row attends of a tile that is not whole is 64 bits: of ranges, or of the row's line of ancestors. Along it the
//   rows' numbers fall, and so do the tiles', so a row walks its line once, as far as each tile reaches.
// - Streams are of any lengths, which the host does not know. All items' tiles are one list, and each of as many workgroups
//   as the chip holds takes an equal run of it, whichever items that cuts: it writes the items that are its own and leaves
//   parts (O, the maximum, the sum) of the two at its ends. A second kernel joins those in the order of the tiles. Where the
//   cuts lie follows from the lengths alone. If all streams' items have as many row tiles, that many workgroups take the
//   same run, one row tile each, so that what one of them has read the others find in their XCD's L2 (two frames of 510
//   rows, 56 heads, 4080 rows back and the 435 first: 209 us, and 188 since).
// What bounds it, by what a call has most of (5 TB/s is what a copy of 1 GiB reaches here):
// - One new row a stream: the one pass over K and V. 129,536 kept rows of three streams, 40 heads on 8: 97 us, 5.5 TB/s, and 6
//   for the join; of 64 streams under a window of 1020 rows, 240 MB: 49 and 5.
// - Small trees: a part's begin (the streams' sums, the pages' numbers, the rows' lines) beside few turns: eight rows after
//   2985 kept, 56 heads, 24 us and 4 for the join, the pass over K and V alone 17.
// - Larger trees: the turns. Five of 63 rows after 129,536 kept in all, 40 heads on 8: 160 list rows an item leave three of
//   eight waves without rows; 136 turns of 1.5 us or more, by the card and its clock (with zeros for all values 203 us for
//   241), and some 25 to begin and to join: 226 .. 275.
// - Chunks: products and softmax in turn, K and V from HBM: those frames' 80 turns take 2 us each, the clock at 1.8 .. 2.1 GHz
//   and the matrix cores busy 38 .. 43% of it.
// Most of the eight-wave kernel's 38 registers in scratch are those of the list of parts; the loop of whole tiles reads none.
#include "attn_tiles.hpp"

namespace mh3 {
namespace {

struct PagesParams : DenseParams {
    const uint16_t* k_pages;
    const uint16_t* v_pages;
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* q_off;
    const int32_t* parents;
    const int32_t* first_rows;
    uint64_t kps, kphs, kprs, vps, vphs, vprs, table_stride; // elements
    uint32_t streams, cols, pages, page_rows, window, workers, slot_rows;
    uint32_t item_rows; // list rows of an item: a wave's 32, or up to eight waves'
    uint32_t begin;     // tiles that take as long as the begin of a part
    uint32_t zero_rest; // rows of no stream become zero
    FastDiv div_item;
    FastDiv div_page;
};

constexpr uint32_t kLeastTiles = 3; // of a workgroup: below it the join costs more than the tiles

// A stream: its new rows q0 .. q0 + rows - 1, kept rows, and the tiles of its items.
struct Stream {
    uint32_t q0, rows, kept, sinks;
    uint32_t front, near0, near; // tiles of the first rows; the first tile that the window reaches, and how many from it on
    uint32_t tiles, row_tiles;
    __device__ __forceinline__ Stream(const PagesParams& p, uint32_t first_q, uint32_t n, uint32_t kept_rows, uint32_t first)
        : q0(first_q), rows(n), kept(kept_rows), sinks(first)
    {
        const uint32_t all = (kept + 63u) / 64u;
        const uint32_t reach = p.window && p.window - 1u < kept ? kept - (p.window - 1u) : 0u; // of the first new rows
        near0 = reach < kept ? reach / 64u : all;
        near = all - near0;
        front = min((sinks + 63u) / 64u, near0);
        tiles = front + near + (rows + 63u) / 64u;
        row_tiles = p.div_item.div(rows * p.group + p.item_rows - 1u);
    }
    // The first key of kept tile u.
    __device__ __forceinline__ uint32_t key(uint32_t u) const { return 64u * (u < front ? u : near0 + u - front); }
    __device__ __forceinline__ bool is_kept(uint32_t u) const { return u < front + near; }
    // The first row of the tile of new rows u.
    __device__ __forceinline__ uint32_t fresh(uint32_t u) const { return 64u * (tiles - 1u - u); }
};

// A 64-bit value of one lane, for all of them.
__device__ __forceinline__ uint64_t lane_u64(uint64_t v, uint32_t lane)
{
    return uint64_t(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(v)), int(lane)))) |
           uint64_t(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(v >> 32)), int(lane)))) << 32;
}

// a / b and ceil(a / b), of 32 bits where a has no more: 64 take some hundred instructions.
__device__ __forceinline__ uint64_t quotient(uint64_t a, uint32_t b)
{
    return a >> 32 ? a / b : uint64_t(uint32_t(a) / b);
}

// The sum of v over the lanes up to this one.
__device__ __forceinline__ uint64_t wave_scan_u64(uint64_t v, uint32_t lane)
{
    if (!__ballot(v >> 26)) // so 64 of them are below 2^32
        return wave_excl_scan_u32(uint32_t(v)) + v;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const uint64_t o = __shfl_up(static_cast<unsigned long long>(v), d, kWave);
        v += lane >= uint32_t(d) ? o : 0u;
    }
    return v;
}

// Stream s of the table, as `sinks` gives it its first rows (which may be new ones too).
__device__ __forceinline__ Stream stream_of(const PagesParams& p, uint32_t s, uint32_t& sinks)
{
    const uint32_t q0 = uint32_t(min(max(p.q_off[s], 0), int32_t(p.q_rows)));
    const uint32_t rows = uint32_t(min(max(p.q_off[s + 1u], int32_t(q0)), int32_t(p.q_rows))) - q0;
    const uint32_t kept = uint32_t(min(max(p.lengths[s], 0), int32_t(p.cols * p.page_rows)));
    sinks = p.first_rows ? min(uint32_t(max(p.first_rows[s], 0)), 1u << 30) : 0u;
    return Stream(p, q0, rows, kept, min(sinks, kept));
}

// How the items' tiles are shared out: runs of `share` pieces, each taken by `together` workgroups, a row tile each (if all
// streams' items have as many row tiles; else 1, and row tiles count one by one). A piece is a tile, or with `size` an
// item's equal part of so many tiles at most.
// An item's tiles are its stream's: those that its own rows do not see (new rows behind its last one, and under a window kept
// and new ones that it has left behind) take masked turns that add nothing. That is little for the trees and frames that this
// is for, but long chunks grow with the square of their rows (40 heads on 8, 4096 kept, a window of 64, 510 / 1000 / 2000 /
// 4000 new rows 36 / 51 / 115 / 332 us, and in one piece through flash_attn_128 47 / 17 / 33 / 49). Nor do all
// workgroups have work where as many of a run's row tiles as go together do not divide them (without the window, 64 / 69 / 86 /
// 130 / 254 row tiles on 256 workgroups: 526 / 710 / 1177 / 3161 / 5301 us, 724 / 590 / 482 / 320 / 532 TFLOP/s).
struct Sharing {
    uint32_t together, size;
    __device__ __forceinline__ uint32_t pieces(uint32_t tiles) const { return size ? (tiles + size - 1u) / size : tiles; }
    // Those of a lane's stream, and of all lanes': 2^32 - 1 for more than a few million.
    __device__ __forceinline__ uint64_t of(const PagesParams& p, const Stream& t) const
    {
        return uint64_t(together > 1u ? min(t.row_tiles, 1u) : t.row_tiles) * p.kv_heads * pieces(t.tiles);
    }
    __device__ __forceinline__ uint32_t of_all(const PagesParams& p, const Stream& t) const
    {
        const uint64_t n = of(p, t);
        return __ballot(n >> 20) ? ~0u : wave_sum_u32(uint32_t(n));
    }
};

// The streams 64 at a time, one a lane, by the sums of their items' pieces.
struct Streams {
    uint32_t s0;
    uint64_t before, some, end; // pieces before the lane's stream; the streams that have any; those up to the 64's end
    __device__ __forceinline__ void sum(const PagesParams& p, uint32_t from, uint64_t base, const Stream& t,
                                        const Sharing& sharing, uint32_t lane)
    {
        s0 = from;
        const uint64_t pieces = sharing.of(p, t);
        some = __ballot(pieces != 0u);
        const uint64_t to = wave_scan_u64(pieces, lane);
        before = base + to - pieces;
        end = base + lane_u64(to, kWave - 1);
    }
    __device__ __forceinline__ static Stream of_lane(const PagesParams& p, uint32_t from, uint32_t lane)
    {
        uint32_t sinks;
        return from + lane < p.streams ? stream_of(p, from + lane, sinks) : Stream(p, 0u, 0u, 0u, 0u);
    }
    __device__ __forceinline__ void load(const PagesParams& p, uint32_t from, uint64_t base, const Sharing& sharing,
                                         uint32_t lane)
    {
        sum(p, from, base, of_lane(p, from, lane), sharing, lane);
    }
    // The last stream that begins at piece x or before it and has any, x one of the 64's.
    __device__ __forceinline__ uint32_t of(uint64_t x) const
    {
        return 63u - uint32_t(__builtin_clzll(__ballot(before <= x) & some));
    }
};

struct Shares : Sharing {
    uint64_t units, share;
    // Leaves the streams at their first 64.
    __device__ __forceinline__ Shares(const PagesParams& p, Streams& st, uint32_t lane)
    {
        const Stream mine = Streams::of_lane(p, 0u, lane);
        uint32_t least = wave_min_u32(mine.rows ? mine.row_tiles : ~0u), most = wave_max_u32(mine.row_tiles);
        for (uint32_t s0 = kWave; s0 < p.streams; s0 += kWave) {
            const Stream t = Streams::of_lane(p, s0, lane);
            least = min(least, wave_min_u32(t.rows ? t.row_tiles : ~0u)), most = max(most, wave_max_u32(t.row_tiles));
        }
        together = least == most && most <= p.workers ? most : 1u, size = 0u;
        st.sum(p, 0u, 0u, mine, *this, lane);
        while (st.s0 + kWave < p.streams)
            st.load(p, st.s0 + kWave, st.end, *this, lane);
        units = st.end;
        const uint32_t runs = p.workers / together;
        share = max(quotient(units + runs - 1u, runs), uint64_t(kLeastTiles));
        // Where cutting each item into equal parts gives every run one of them, hardly longer than its share: a run that
        // goes on into another item begins anew there, which takes as long as some tiles.
        for (uint32_t i = 0; i <= p.begin && size == 0u && share < (1u << 20); ++i) {
            const Sharing parts{together, uint32_t(share) + i};
            uint64_t n = parts.of_all(p, mine);
            for (uint32_t s0 = kWave; s0 < p.streams && n <= runs; s0 += kWave)
                n += parts.of_all(p, Streams::of_lane(p, s0, lane));
            if (n <= runs)
                size = parts.size;
        }
        if (size || st.s0 != 0u)
            st.sum(p, 0u, 0u, mine, *this, lane);
        while (size && st.s0 + kWave < p.streams)
            st.load(p, st.s0 + kWave, st.end, *this, lane);
        if (size) {
            units = st.end, share = 1u;
            if (st.s0 != 0u)
                st.sum(p, 0u, 0u, mine, *this, lane);
        }
    }
};

// What the join has to know of an item that runs cut, left by the workgroup whose run is the first to begin inside it.
struct Cut {
    uint32_t rows; // list rows, 0: the workgroup leaves none
    uint32_t q0, f0, kvh;
    uint32_t run, last; // the parts are those of runs run - 1 .. last
    uint32_t together, row_tile;
};

// Rows in one piece: where they begin and how many bytes a buffer over them has (none: nothing is read, and zeros come).
struct Piece {
    uint64_t at;
    uint32_t bytes;
};

// A wave's item, and what a lane has of it.
struct Item {
    Stream st;
    uint32_t stream, kvh;
    uint32_t begin, list, f0; // the item's list rows, up to `list`, and the wave's first one
    uint32_t sinks;   // as given: new rows may be among the first ones too
    uint32_t row, up; // the lane's row's number among the new ones; the row of its line that the walk is at (~0: at its end)
    uint32_t place;   // the row's
    uint32_t up_place; // that of `up`
    uint32_t lo;      // kept rows from it on are under the window
    uint32_t all_lo;  // of every row of the workgroup, or a bound of that
    const int32_t* parents; // in LDS, of streams of up to kParents rows
};

constexpr uint32_t kParents = 1024;

// The row's parent, ~0 for none: a parent lies before its row. (A line of them read from memory takes half a us a step.)
__device__ __forceinline__ uint32_t parent_of(const PagesParams& p, const Item& it, uint32_t row)
{
    uint32_t up = ~0u;
    if (row < it.st.rows)
        up = uint32_t(it.st.rows <= kParents ? it.parents[row] : p.parents[it.st.q0 + row]);
    return up < row ? up : ~0u;
}

// The parents of the item's stream into LDS, by all `threads` of the workgroup.
__device__ __forceinline__ void load_parents(const PagesParams& p, const Item& it, int32_t* to, uint32_t threads)
{
    if (p.parents && it.st.rows <= kParents)
        for (uint32_t i = threadIdx.x; i < it.st.rows; i += threads)
            to[i] = p.parents[it.st.q0 + i];
}

// A wave's rows of q as they lie in memory, so that they are on their way while other things are looked up.
struct RawRows {
    uint4 t[8];
    __device__ __forceinline__ RawRows(const PagesParams& p, const Item& it, uint32_t lane)
    {
        const uint32_t f = it.f0 + (lane & 31u), fc = min(f, it.list - 1u), row = p.div_group.div(fc);
        const uint32_t head = it.kvh * p.group + (fc - row * p.group);
        const uint16_t* const src = p.q + uint64_t(head) * p.qhs + uint64_t(it.st.q0 + row) * p.qrs + 8u * (lane >> 5);
#pragma unroll
        for (int dc = 0; dc < 8; ++dc)
            t[dc] = f < it.list ? *reinterpret_cast<const uint4*>(src + 16 * dc) : uint4{0u, 0u, 0u, 0u};
    }
};

// The kept rows that every row of the workgroup has under the window, at least: a row has as many ancestors as there are
// rows before it, at most.
__device__ __forceinline__ void bound_window(const PagesParams& p, Item& it)
{
    const uint32_t far = it.st.kept + p.div_group.div(it.list - 1u);
    it.all_lo = p.window && p.window - 1u < far ? far - (p.window - 1u) : 0u;
}

__device__ __forceinline__ void begin_item(const PagesParams& p, Item& it, const RawRows& raw, uint32_t lane, WaveRows& w)
{
    it.row = p.div_group.div(min(it.f0 + (lane & 31u), it.list - 1u));
#pragma unroll
    for (int dc = 0; dc < 8; ++dc) {
        uint32_t x[4] = {raw.t[dc].x, raw.t[dc].y, raw.t[dc].z, raw.t[dc].w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            x[e] = pack_bf16(bf16_lo(x[e]) * p.q_pow, bf16_hi(x[e]) * p.q_pow);
        w.qf[dc] = __builtin_bit_cast(bf16x8_t, uint4{x[0], x[1], x[2], x[3]});
    }
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e)
            w.o[b][e] = 0.0f;
    uint32_t depth = it.row;
    if (p.parents && p.window) { // only a window asks for the rows' places
        depth = 0;
        for (uint32_t up = parent_of(p, it, it.row); up != ~0u; up = parent_of(p, it, up))
            ++depth;
    }
    it.place = it.st.kept + depth;
    it.up = it.row, it.up_place = it.place;
    it.lo = p.window && p.window - 1u < it.place ? it.place - (p.window - 1u) : 0u;
    w.m_run = -kInf, w.l_run = 0.0f, w.settled = false, w.begun = false;
}

// The bits of the lane's row's keys among the 64 new rows from n0 on. Of a tree the tiles are asked for from the last to
// the first, each once, but need not begin with the last.
__device__ __forceinline__ uint64_t fresh_bits(const PagesParams& p, Item& it, uint32_t n0)
{
    const uint32_t none = it.st.kept < it.sinks ? it.sinks - it.st.kept : 0u; // new rows that are among the first ones
    if (!p.parents) {
        const uint32_t lo = it.lo > it.st.kept ? it.lo - it.st.kept : 0u;
        return key_bits(lo, it.row + 1u, n0) | key_bits(0u, min(none, it.row + 1u), n0);
    }
    uint64_t bits = 0;
    while (it.up != ~0u && it.up >= n0) {
        if (it.up < n0 + 64u && (!p.window || it.up_place >= it.lo || it.up_place < it.sinks))
            bits |= uint64_t(1) << (it.up - n0);
        it.up = parent_of(p, it, it.up), --it.up_place;
    }
    return bits;
}

// Rows r .. r + n - 1 (of tile u, `row` their first one there) of a part's K (VALUE false) or V, and whether they are there.
template <bool VALUE>
__device__ __forceinline__ Piece piece_of(const PagesParams& p, const Item& it, bool kept, uint32_t key, int32_t page,
                                          uint32_t n)
{
    if (kept) {
        const uint32_t r = key - p.div_page.div(key) * p.page_rows;
        const uint64_t at = uint64_t(uint32_t(max(page, 0))) * (VALUE ? p.vps : p.kps) +
                            uint64_t(r) * (VALUE ? p.vprs : p.kprs) + it.kvh * (VALUE ? p.vphs : p.kphs);
        const uint32_t rows = page >= 0 && key < it.st.kept ? min(n, it.st.kept - key) : 0u;
        return {reinterpret_cast<uint64_t>((VALUE ? p.v_pages : p.k_pages) + at),
                rows ? (rows - 1u) * uint32_t(VALUE ? p.vprs : p.kprs) * 2u + 256u : 0u};
    }
    const uint32_t rows = key < it.st.rows ? min(n, it.st.rows - key) : 0u;
    const uint64_t at = uint64_t(it.st.q0 + (rows ? key : 0u)) * (VALUE ? p.vrs : p.krs) + it.kvh * (VALUE ? p.vhs : p.khs);
    return {reinterpret_cast<uint64_t>((VALUE ? p.v : p.k) + at),
            rows ? (rows - 1u) * uint32_t(VALUE ? p.vrs : p.krs) * 2u + 256u : 0u};
}

// The page of kept row `key`, -1 for none.
__device__ __forceinline__ int32_t page_of(const PagesParams& p, const Item& it, uint32_t key)
{
    if (key >= it.st.kept)
        return -1;
    const int32_t page = p.table[uint64_t(it.stream) * p.table_stride + p.div_page.div(key)];
    return uint32_t(page) < p.pages ? page : -1;
}

// What a workgroup of one wave loads, tile by tile: four pieces of 16 rows, which each lie in one page. Lane 4 (u % 16) + g
// has those of group g of tile u, for 16 tiles at a time: a page's place takes some 40 scalar instructions to find.
struct PageFeed {
    char* lds; // K, V, the wave's scratch (1 KB)
    uint32_t k_key, k_chunk, v_key, v_chunk; // the lane's row and bytes of it in its instructions
    Piece k, v;
    uint64_t there_bits; // lanes whose page is there
    __device__ __forceinline__ PageFeed(char* memory, uint32_t lane)
        : lds(memory), k_key(lane >> 4), k_chunk(16u * ((lane & 15u) ^ (lane >> 4))), v_key((lane >> 2) & 3u),
          v_chunk(16u * (4u * (lane >> 4) + (lane & 3u)))
    {
    }
    __device__ __forceinline__ void numbers(const PagesParams& p, const Item& it, uint32_t u16, uint32_t lane)
    {
        const uint32_t u = u16 + lane / 4u, g = lane % 4u;
        const bool kept = it.st.is_kept(u);
        const uint32_t key = 16u * g + (kept ? it.st.key(u) : it.st.fresh(min(u, it.st.tiles - 1u)));
        const int32_t page = kept ? page_of(p, it, key) : -1;
        there_bits = __ballot(page >= 0);
        k = piece_of<false>(p, it, kept, key, page, 16u), v = piece_of<true>(p, it, kept, key, page, 16u);
    }
    // The bits of the tile's keys whose page is there.
    __device__ __forceinline__ uint64_t there(uint32_t u) const
    {
        uint64_t bits = 0;
#pragma unroll
        for (uint32_t g = 0; g < 4u; ++g)
            bits |= there_bits >> (4u * (u % 16u) + g) & 1u ? uint64_t(0xffff) << (16u * g) : 0u;
        return bits;
    }
    __device__ __forceinline__ bool all_there(uint32_t u) const { return (there_bits >> (4u * (u % 16u)) & 15u) == 15u; }
    template <bool VALUE>
    __device__ __forceinline__ void load(const PagesParams& p, const Item& it, uint32_t u) const
    {
        char* const dst = lds + (VALUE ? kTileBytes : 0u);
        const uint32_t row = 2u * uint32_t(it.st.is_kept(u) ? (VALUE ? p.vprs : p.kprs) : (VALUE ? p.vrs : p.krs));
        const Piece& t = VALUE ? v : k;
        uint32_t off[4];
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) // rows 4 i of the group, of K the chunks swizzled by the row
            off[i] = VALUE ? (v_key + 4u * i) * row + v_chunk : (k_key + 4u * i) * row + (k_chunk ^ (64u * i));
#pragma unroll
        for (uint32_t g = 0; g < 4u; ++g) {
            const int at = int(4u * (u % 16u) + g);
            const u32x4_t b{uint32_t(__builtin_amdgcn_readlane(int(uint32_t(t.at)), at)),
                            uint32_t(__builtin_amdgcn_readlane(int(uint32_t(t.at >> 32)), at)) & 0xffffu,
                            uint32_t(__builtin_amdgcn_readlane(int(t.bytes), at)), uint32_t(kRsrcFlags)};
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i)
                load_lds16(b, dst + 4096u * g + 1024u * i, off[i]);
        }
    }
};

// The keys of tile u that the lane's row attends.
template <class Feed>
__device__ __forceinline__ uint64_t bits_of(const PagesParams& p, Item& it, const Feed& feed, uint32_t u)
{
    if (!it.st.is_kept(u))
        return fresh_bits(p, it, it.st.fresh(u));
    const uint32_t t0 = it.st.key(u);
    return (key_bits(it.lo, it.st.kept, t0) | key_bits(0u, it.st.sinks, t0)) & feed.there(u);
}

// Whether every row attends all of tile u, if its pages are there.
__device__ __forceinline__ bool is_whole(const Item& it, uint32_t u)
{
    if (!it.st.is_kept(u))
        return false;
    const uint32_t t0 = it.st.key(u);
    return t0 + 64u <= it.st.kept && (t0 >= it.all_lo || t0 + 64u <= it.st.sinks);
}

// A turn of attn_pages_kernel, tile u, as few_turn of attn_dense.hip: a tile's K is on its way from the products before it
// to its own, its V from the output before. The page numbers of tile u + 1 are in the feed by its end.
template <bool CAP, bool MASKED>
__device__ __forceinline__ void pages_turn(const PagesParams& p, Item& it, WaveRows& w, PageFeed& feed, const TileReads& rd,
                                           uint32_t u, uint32_t last, uint32_t lane)
{
    uint16_t* const scratch = reinterpret_cast<uint16_t*>(feed.lds + 2u * kTileBytes);
    const char* const vt = feed.lds + kTileBytes;
    const bool more = u + 1u < last;
    const BitsSeen seen(MASKED ? bits_of(p, it, feed, u) : 0u, lane);
    floatx16 s[2];
    bf16x8_t frag[kAhead];
    TileP pt;
    wait_vm<16>(); // K; V may still be in flight
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
        frag[j] = rd.k(feed.lds, j);
    tile_products<false, false>(w, s, pt, frag, rd, feed.lds, nullptr, 0, nullptr, lane);
    wait_lds();
    if (more) {
        if ((u + 1u) % 16u == 0u)
            feed.numbers(p, it, u + 1u, lane);
        feed.load<false>(p, it, u + 1u);
        __builtin_amdgcn_sched_barrier(0);
    }
    tile_softmax<CAP, false, MASKED>(p, w, s, pt, 0u, seen, nullptr, nullptr, false, false, lane);
    if (more)
        wait_vm<16>(); // V, but not the next K
    else
        wait_vm<0>();
    if (MASKED && holds_nonfinite<16>(vt, lane))
        tile_output_masked(w, pt, rd, vt, seen, scratch, lane);
    else
        tile_output(w, pt, frag, rd, vt);
    wait_lds();
    if (more)
        feed.load<true>(p, it, u + 1u);
}

// The parts behind the cuts.
__device__ __forceinline__ float* parts_of(const PagesParams& p) { return p.part + uint64_t(p.workers) * (sizeof(Cut) / 4u); }

// Writes an item's rows, or with `slot` a part of them: O [slot][row][128], behind all slots' the maxima and sums.
__device__ __forceinline__ void store_item(const PagesParams& p, const Item& it, const WaveRows& w, uint32_t slot,
                                           uint32_t lane)
{
    const uint32_t hh = lane >> 5, f = it.f0 + (lane & 31u), n = f - it.begin;
    const float l = w.l_run + __shfl_xor(w.l_run, 32, kWave);
    if (f >= it.list)
        return;
    if (slot != ~0u) {
        const uint64_t at = uint64_t(slot) * p.slot_rows + n;
        float* const dst = parts_of(p) + at * 128u;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<float4*>(dst + 32 * db + 8 * g + 4u * hh) =
                    float4{w.o[db][4 * g], w.o[db][4 * g + 1], w.o[db][4 * g + 2], w.o[db][4 * g + 3]};
        if (hh == 0)
            *reinterpret_cast<float2*>(parts_of(p) + 2ull * p.workers * p.slot_rows * 128u + at * 2u) = float2{w.m_run, l};
        return;
    }
    const uint32_t row = p.div_group.div(f), head = it.kvh * p.group + (f - row * p.group);
    const float inv = 1.0f / l; // a row attends itself
    uint16_t* const dst = p.out + uint64_t(head) * p.ohs + uint64_t(it.st.q0 + row) * p.ors;
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<uint2*>(dst + 32 * db + 8 * g + 4u * hh) =
                uint2{pack_bf16(w.o[db][4 * g] * inv, w.o[db][4 * g + 1] * inv),
                      pack_bf16(w.o[db][4 * g + 2] * inv, w.o[db][4 * g + 3] * inv)};
}

// A workgroup's run of all items' tiles: part(item, first, last, slot) for each of its parts.
template <class Part>
__device__ __forceinline__ void for_parts(const PagesParams& p, uint32_t lane, const Part& part)
{
    // Blocks go to the 8 XCDs round-robin; each takes a contiguous part of the list, key head by key head.
    const uint32_t worker = (blockIdx.x % 8u) * (gridDim.x / 8u) + blockIdx.x / 8u;
    Streams streams;
    const Shares shares(p, streams, lane);
    const uint32_t run = worker / shares.together, row_tile = worker - run * shares.together;
    const uint64_t begin = shares.share * run, end = min(shares.units, begin + shares.share);
    Cut cut{};
    for (uint64_t x = begin; x < end;) {
        while (x >= streams.end)
            streams.load(p, streams.s0 + kWave, streams.end, shares, lane);
        const uint32_t at = streams.of(x), stream = streams.s0 + at;
        uint32_t sinks;
        const Stream st = stream_of(p, stream, sinks);
        const uint32_t pieces = shares.pieces(st.tiles);
        const uint64_t local = x - lane_u64(streams.before, at), number = quotient(local, pieces);
        const uint32_t a = uint32_t(local - number * pieces), b = uint32_t(min(uint64_t(pieces), a + (end - x)));
        const uint32_t kvh = uint32_t(shares.together > 1u ? number : quotient(number, st.row_tiles));
        const uint32_t from = p.item_rows * (shares.together > 1u ? row_tile : uint32_t(number - uint64_t(kvh) * st.row_tiles));
        Item it{st};
        it.stream = stream, it.kvh = kvh, it.sinks = sinks;
        it.begin = it.f0 = from, it.list = min(from + p.item_rows, st.rows * p.group);
        // The item that the run begins with, unless with its first piece, is the first of the workgroup's two parts.
        const bool whole = a == 0u && b == pieces;
        if (a > 0u && shares.share >= a) // the run before this one begins with the item or ahead of it
            cut = Cut{it.list - from,
                      st.q0,
                      from,
                      kvh,
                      run,
                      uint32_t(quotient(x - a + pieces - 1u, uint32_t(min(shares.share, uint64_t(~0u))))),
                      shares.together,
                      row_tile};
        const uint32_t first = shares.size ? uint32_t(uint64_t(st.tiles) * a / pieces) : a;
        const uint32_t last = shares.size ? uint32_t(uint64_t(st.tiles) * b / pieces) : b;
        part(it, first, last, whole ? ~0u : 2u * worker + (a > 0u ? 0u : 1u));
        x += b - a;
    }
    if (threadIdx.x == 0)
        reinterpret_cast<Cut*>(p.part)[worker] = cut;
}

// One wave a workgroup, with a tile of its own in LDS; four of them share a CU.
template <bool CAP>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(1, 1))) void attn_pages_kernel(PagesParams p)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const uint32_t lane = threadIdx.x;
    const TileReads rd(lane);
    PageFeed feed(lds, lane);
    int32_t* const parents = reinterpret_cast<int32_t*>(lds + 2u * kTileBytes + 1024u);
    for_parts(p, lane, [&](Item& it, uint32_t first, uint32_t last, uint32_t slot) {
        WaveRows w;
        bound_window(p, it);
        const RawRows raw(p, it, lane);
        load_parents(p, it, parents, kWave);
        it.parents = parents;
        feed.numbers(p, it, first & ~15u, lane);
        feed.load<false>(p, it, first);
        feed.load<true>(p, it, first);
        begin_item(p, it, raw, lane, w);
        for (uint32_t u = first; u < last;) {
#pragma unroll 1
            for (; u < last && !(is_whole(it, u) && feed.all_there(u)); ++u)
                pages_turn<CAP, true>(p, it, w, feed, rd, u, last, lane);
#pragma unroll 1
            for (; u < last && is_whole(it, u) && feed.all_there(u); ++u)
                pages_turn<CAP, false>(p, it, w, feed, rd, u, last, lane);
        }
        store_item(p, it, w, slot, lane);
    });
}

// What a wave of eight loads of a workgroup's tiles, K or V, each a quarter: a group of 16 rows, which lie in one page. Their
// places and sizes are found for 64 tiles at a time, one a lane, every 32 tiles, and lie in LDS: among the softmax's vector
// instructions there is no time for the some 40 scalar ones that each takes.
struct PairPageFeed {
    static constexpr int kLoads = 4; // of a turn
    const PagesParams& p;
    const Item& it;
    char* lds;
    u32x4_t* places; // of tile u at u % 64: address, bytes, bytes from a row to the next
    uint32_t first, tiles, wave; // the part's first tile, and how many
    uint32_t key, chunk; // the lane's row and bytes of it in its instructions
    uint32_t base;         // the places are those of tiles base .. base + 63
    uint64_t whole;        // bit u % 64: every row attends all of tile u
    uint64_t group_there[4]; // whether the page of each group of 16 rows is there

    __device__ __forceinline__ PairPageFeed(const PagesParams& params, const Item& item, char* memory, u32x4_t* list,
                                            uint32_t part_first, uint32_t part_tiles, uint32_t wave_number, uint32_t lane)
        : p(params), it(item), lds(memory), places(list), first(part_first), tiles(part_tiles), wave(wave_number)
    {
        key = wave < kHalf ? lane >> 4 : (lane >> 2) & 3u;
        chunk = 16u * (wave < kHalf ? (lane & 15u) ^ (lane >> 4) : 4u * (lane >> 4) + (lane & 3u));
    }
    __device__ __forceinline__ void find(uint32_t from)
    {
        const uint32_t lane = threadIdx.x & 63u;
        base = from;
        const uint32_t u = base + ((lane - base) & 63u);
        const bool kept = it.st.is_kept(u);
        const uint32_t k0 = kept ? it.st.key(u) : it.st.fresh(min(u, it.st.tiles - 1u));
        int32_t mine = -1;
        whole = __ballot(is_whole(it, u));
#pragma unroll
        for (uint32_t g = 0; g < 4u; ++g) {
            const int32_t page = kept ? page_of(p, it, k0 + 16u * g) : -1;
            mine = g == wave % kHalf ? page : mine;
            group_there[g] = __ballot(page >= 0);
            whole &= group_there[g];
        }
        const uint32_t k = k0 + 16u * (wave % kHalf);
        const Piece t = wave < kHalf ? piece_of<false>(p, it, kept, k, mine, 16u) : piece_of<true>(p, it, kept, k, mine, 16u);
        const uint64_t row = wave < kHalf ? (kept ? p.kprs : p.krs) : (kept ? p.vprs : p.vrs);
        places[lane] = u32x4_t{uint32_t(t.at), uint32_t(t.at >> 32) & 0xffffu, t.bytes, 2u * uint32_t(row)};
        asm volatile("" ::: "memory"); // a wave's LDS accesses are in order
    }
    __device__ __forceinline__ const char* k_tile(uint32_t t) const { return lds + (t % kRing) * kTileBytes; }
    __device__ __forceinline__ const char* v_tile(uint32_t t) const { return lds + (kRing + t % kRing) * kTileBytes; }
    __device__ __forceinline__ int32_t* positions(uint32_t) const { return nullptr; }
    // The part's tile t, past its end the last one again: every turn has the same count of loads.
    __device__ __forceinline__ void load(uint32_t t) const
    {
        const u32x4_t place = places[(first + min(t, tiles - 1u)) % 64u];
        char* const dst = const_cast<char*>(wave < kHalf ? k_tile(t) : v_tile(t)) + 4096u * (wave % kHalf);
        const u32x4_t b{uint32_t(__builtin_amdgcn_readfirstlane(int(place[0]))), // all lanes have the same
                        uint32_t(__builtin_amdgcn_readfirstlane(int(place[1]))),
                        uint32_t(__builtin_amdgcn_readfirstlane(int(place[2]))), uint32_t(kRsrcFlags)};
        const uint32_t four = 4u * uint32_t(__builtin_amdgcn_readfirstlane(int(place[3])));
        const uint32_t flip = wave < kHalf ? 64u : 0u; // of K the chunks are swizzled by the row, 4 u + key
        const uint32_t at = key * (four / 4u);
#pragma unroll
        for (uint32_t u = 0; u < 4u; ++u)
            load_lds16(b, dst + 1024u * u, at + u * four + (chunk ^ u * flip));
    }
    __device__ __forceinline__ void next(uint32_t t)
    {
        const uint32_t ahead = t + (wave < kHalf ? 3u : 2u);
        if (first + min(ahead, tiles - 1u) >= base + 64u)
            find(base + 32u);
        load(ahead);
    }
    // The bits of the tile's keys whose page is there.
    __device__ __forceinline__ uint64_t there(uint32_t u) const
    {
        uint64_t bits = 0;
#pragma unroll
        for (uint32_t g = 0; g < 4u; ++g)
            bits |= group_there[g] >> (u % 64u) & 1u ? uint64_t(0xffff) << (16u * g) : 0u;
        return bits;
    }
};

// A part's tiles, as pair_walk asks for them. What a lane has of its row lies in LDS: only masked turns ask for it.
struct PairPageWalk {
    const PagesParams& p;
    Item& it;
    const PairPageFeed& feed;
    uint4* rows; // the wave's: number, place in its line, that place, first kept row under the window
    uint32_t lane;
    __device__ __forceinline__ uint32_t key(uint32_t) const { return 0u; } // only a bias asks where a tile lies
    __device__ __forceinline__ bool whole(uint32_t t) const { return feed.whole >> ((feed.first + t) % 64u) & 1u; }
    __device__ __forceinline__ BitsSeen seen(uint32_t t)
    {
        const uint4 r = rows[lane & 31u];
        it.row = r.x, it.up = r.y, it.up_place = r.z, it.lo = r.w;
        const uint64_t bits = bits_of(p, it, feed, feed.first + t);
        if (p.parents)
            rows[lane & 31u] = uint4{it.row, it.up, it.up_place, it.lo}; // both of a row's lanes the same
        return BitsSeen(it.f0 + (lane & 31u) < it.list ? bits : 0u, lane);
    }
};

// Eight waves a workgroup: one to a CU.
constexpr uint32_t kPairWaveBytes = 1024u + 512u + 1024u; // a wave's scratch, its rows, its places

template <bool CAP>
__global__ __launch_bounds__(kPairWaves * 64) __attribute__((amdgpu_waves_per_eu(2))) void attn_pages_pair_kernel(PagesParams p)
{
    // K ring, V ring, the waves' own, for two tiles whether the waves' parts of V hold an infinity or a NaN, and a tree.
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    char* const own = lds + 2u * kRing * kTileBytes + kPairWaveBytes * wave;
    uint16_t* const scratch = reinterpret_cast<uint16_t*>(own);
    uint4* const rows = reinterpret_cast<uint4*>(own + 1024u);
    u32x4_t* const places = reinterpret_cast<u32x4_t*>(own + 1536u);
    uint32_t* const odd = reinterpret_cast<uint32_t*>(lds + 2u * kRing * kTileBytes + kPairWaveBytes * kPairWaves);
    int32_t* const parents = reinterpret_cast<int32_t*>(odd + 2u * kHalf);
    const TileReads rd(lane);
    for_parts(p, lane, [&](Item& it, uint32_t first, uint32_t last, uint32_t slot) {
        // Few rows go to as many waves of either group, and to each SIMD before one gets two.
        it.f0 += 32u * (wave < kHalf ? 2u * wave : 2u * (kPairWaves - 1u - wave) + 1u);
        bound_window(p, it);
        const RawRows raw(p, it, lane);
        PairPageFeed feed(p, it, lds, places, first, last - first, wave, lane);
        feed.find(first & ~31u);
        lds_barrier(); // the part before this one is read
        feed.load(0u);
        feed.load(1u);
        if (wave < kHalf)
            feed.load(2u);
        load_parents(p, it, parents, 64u * kPairWaves);
        it.parents = parents;
        lds_barrier();
        WaveRows w;
        begin_item(p, it, raw, lane, w);
        rows[lane & 31u] = uint4{it.row, it.up, it.up_place, it.lo};
        PairPageWalk walk{p, it, feed, rows, lane};
        pair_walk<CAP, false>(p, w, feed, walk, rd, scratch, odd, wave, last - first, it.f0 < it.list, lane);
        store_item(p, it, w, slot, lane);
    });
}

// Joins the parts of the items that the runs cut, in the order of the tiles. A workgroup takes 8 / SPLIT rows of a cut at a
// time, 32 lanes a row, four values of d each; with SPLIT 4 a row's parts are taken by four waves, every fourth each, and
// these meet in LDS. The host does not know the cuts: each workgroup sums up their rows and finds its own by itself. (A
// workgroup for each cut that there may be and some of its rows, most of which find none, takes 1.15 us a thousand: three
// streams' single rows over 129,536 kept ones 8.9 us for 6.2 now, eight drafts over 2985 8.9 and 4.2.)
template <uint32_t SPLIT>
__global__ __launch_bounds__(256) void attn_pages_join_kernel(PagesParams p)
{
    constexpr uint32_t kRows = 8u / SPLIT, kU = 8;
    __shared__ float met[SPLIT][kRows][6][32];
    __shared__ uint32_t wave_sums[4], found_row;
    __shared__ Cut found;
    const Cut* const cuts = reinterpret_cast<const Cut*>(p.part);
    const auto pieces = [&](uint32_t c) { return (cuts[c].rows + kRows - 1u) / kRows; };
    const uint32_t share = (p.workers + 255u) / 256u, c0 = threadIdx.x * share; // a thread's cuts
    uint32_t mine = 0;
    for (uint32_t c = c0; c < min(c0 + share, p.workers); ++c)
        mine += pieces(c);
    uint32_t before = wave_excl_scan_u32(mine), total = 0;
    if (threadIdx.x % 64u == 63u)
        wave_sums[threadIdx.x / 64u] = before + mine;
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) {
        before += i < threadIdx.x / 64u ? wave_sums[i] : 0u;
        total += wave_sums[i];
    }
    if (p.zero_rest) {
        const uint32_t from = uint32_t(min(max(p.q_off[p.streams], 0), int32_t(p.q_rows)));
        const uint32_t ahead = min(uint32_t(max(p.q_off[0], 0)), from), rest = ahead + p.q_rows - from;
        const uint32_t heads = p.kv_heads * p.group;
        for (uint64_t i = blockIdx.x * 8u + threadIdx.x / 32u; i < uint64_t(rest) * heads; i += gridDim.x * 8u) {
            const uint32_t n = uint32_t(i / heads), head = uint32_t(i - uint64_t(n) * heads);
            const uint32_t row = n < ahead ? n : from + (n - ahead);
            *reinterpret_cast<uint2*>(p.out + uint64_t(head) * p.ohs + uint64_t(row) * p.ors + 4u * (threadIdx.x & 31u)) =
                uint2{0u, 0u};
        }
    }
    const float* const parts = parts_of(p);
    const float2* const ml = reinterpret_cast<const float2*>(parts + 2ull * p.workers * p.slot_rows * 128u);
    const uint32_t sub = threadIdx.x / 32u, which = sub / kRows, d = 4u * (threadIdx.x & 31u);
    for (uint32_t piece = blockIdx.x; piece < total; piece += gridDim.x) {
        __syncthreads();
        if (piece - before < mine) {
            uint32_t left = piece - before, c = c0;
            for (uint32_t n = pieces(c); left >= n; n = pieces(c))
                left -= n, ++c;
            found = cuts[c], found_row = left * kRows;
        }
        __syncthreads();
        const Cut cut = found;
        const uint32_t n = found_row + sub % kRows;
        const bool here = n < cut.rows;
        float m = -kInf, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        const auto meet = [&](const float2* t, const float4* v, uint32_t count) {
            float m_new = m;
            for (uint32_t u = 0; u < count; ++u)
                m_new = fmaxf(m_new, t[u].x);
            // A part without a key of this row has left zeros and -inf. (A NaN of its scores is in its sum and its O.)
            const float old = m == -kInf ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
            l *= old, m = m_new;
            for (int c = 0; c < 4; ++c)
                o[c] *= old;
            for (uint32_t u = 0; u < count; ++u) {
                const float e = t[u].x == -kInf ? 1.0f : __builtin_amdgcn_exp2f(t[u].x - m_new);
                l = fmaf(t[u].y, e, l);
                o[0] = fmaf(v[u].x, e, o[0]), o[1] = fmaf(v[u].y, e, o[1]);
                o[2] = fmaf(v[u].z, e, o[2]), o[3] = fmaf(v[u].w, e, o[3]);
            }
        };
        for (uint32_t i0 = cut.run - 1u + which; i0 <= cut.last; i0 += SPLIT * kU) {
            float2 t[kU];
            float4 v[kU];
#pragma unroll
            for (uint32_t u = 0; u < kU; ++u) {
                const uint32_t i = i0 + SPLIT * u;
                t[u] = float2{-kInf, 0.0f}, v[u] = float4{0.0f, 0.0f, 0.0f, 0.0f};
                if (here && i <= cut.last) {
                    const uint64_t slot =
                        (2ull * (i * cut.together + cut.row_tile) + (i < cut.run ? 1u : 0u)) * p.slot_rows + n;
                    t[u] = ml[slot], v[u] = *reinterpret_cast<const float4*>(parts + slot * 128u + d);
                }
            }
            meet(t, v, kU);
        }
        if (SPLIT > 1u) {
            float(&mark)[6][32] = met[which][sub % kRows];
            mark[0][d / 4u] = m, mark[1][d / 4u] = l;
            for (int c = 0; c < 4; ++c)
                mark[2 + c][d / 4u] = o[c];
            __syncthreads();
            if (which == 0u) {
                float2 t[SPLIT];
                float4 v[SPLIT];
                for (uint32_t i = 0; i < SPLIT; ++i) {
                    const float(&from)[6][32] = met[i][sub % kRows];
                    t[i] = float2{from[0][d / 4u], from[1][d / 4u]};
                    v[i] = float4{from[2][d / 4u], from[3][d / 4u], from[4][d / 4u], from[5][d / 4u]};
                }
                m = -kInf, l = 0.0f, o[0] = o[1] = o[2] = o[3] = 0.0f;
                meet(t, v, SPLIT);
            }
            __syncthreads();
        }
        if (!here || which != 0u)
            continue;
        const float inv = 1.0f / l;
        const uint32_t f = cut.f0 + n, row = p.div_group.div(f), head = cut.kvh * p.group + (f - row * p.group);
        *reinterpret_cast<uint2*>(p.out + uint64_t(head) * p.ohs + uint64_t(cut.q0 + row) * p.ors + d) =
            uint2{pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv)};
    }
}

} // namespace
} // namespace mh3

namespace {

using namespace mh3;

// Tiles that take as long as the begin of a part, of one wave and of eight.
constexpr uint32_t kBegin = 3, kPairBegin = 12;

// Which kernel a call takes, and how many rows an item has, from the list rows that its streams have on average. (One wave a
// workgroup and eight, us, 40 heads on 8: five streams of 129,536 kept rows in all and 60 list rows each 118 and 128, 65 139
// and 128, 100 169 and 130; three of 14,925 and 60 rows 33 and 36, 90 36 and 37, 125 41 and 40; one of 2985 within 3 of each
// other up to 150.) Streams without new rows count too, as the host does not see them: two of 510 rows over 4515 kept ones take
// 171 us in a table of two and 337 in one of 64 (56 heads; 40 on 8 136 and 222).
struct PagesPlan {
    uint32_t item_rows, workers, slot_rows; // slot_rows: a part's, an item's or all of the call's where they are fewer
    uint64_t workspace;
};

PagesPlan pages_plan(const MH3PagesAttnArgs& a)
{
    const uint64_t list = uint64_t(a.q_rows) * (a.heads / a.kv_heads);
    const uint64_t rows = (list + a.table.streams - 1u) / a.table.streams; // of a stream
    const bool pair = rows > 64u;
    const uint32_t cus = uint32_t(std::max(host::cu_count(), 1));
    PagesPlan plan;
    const uint64_t items = (rows + 32u * kPairWaves - 1u) / (32u * kPairWaves);
    plan.item_rows = pair ? uint32_t((rows + items - 1u) / items + 31u) / 32u * 32u : 32u;
    plan.workers = ((pair ? 1u : 4u) * cus + 7u) / 8u * 8u;
    plan.slot_rows = uint32_t(std::min<uint64_t>(plan.item_rows, list));
    plan.workspace = uint64_t(plan.workers) * (sizeof(Cut) + 2ull * plan.slot_rows * 130u * 4u);
    return plan;
}

int check_pages_args(const MH3PagesAttnArgs* args)
{
    if (!args)
        return MH3_ERR_POINTER;
    const MH3PagesAttnArgs& a = *args;
    const MH3PagesArgs& t = a.table;
    if (a.heads == 0 || a.kv_heads == 0 || a.head_dim == 0 || a.heads % a.kv_heads != 0)
        return MH3_ERR_SHAPE;
    if (a.head_dim != 128u)
        return MH3_ERR_UNSUPPORTED;
    if (a.zero_rest > 1u || !(a.scale >= 0.0f && a.scale <= 0x1p100f) ||
        !(a.cap == 0.0f || (a.cap >= 0x1p-60f && a.cap <= 1024.0f)))
        return MH3_ERR_PARAM;
    if (t.streams == 0 || t.streams > MH3_MAX_STREAMS || t.cols == 0 || t.cols >= (1u << 24) || t.pages == 0 ||
        t.pages >= (1u << 24) || t.table_stride < t.cols || t.table_stride >= (1ull << 32) || t.page_rows == 0 ||
        t.page_rows % 16u != 0 || uint64_t(t.cols) * t.page_rows >= (1ull << 30))
        return MH3_ERR_SHAPE;
    if (a.heads > 4096u || uint64_t(a.q_rows) * (a.heads / a.kv_heads) >= (1u << 30) || a.q_rows >= (1u << 30))
        return MH3_ERR_SHAPE;
    for (const uint64_t s : {a.q_row_stride, a.k_row_stride, a.v_row_stride, a.out_row_stride, a.k_page_row_stride,
                             a.v_page_row_stride}) {
        if (s % 8u != 0)
            return MH3_ERR_ALIGN;
        if (s < 128u || s >= (1ull << 23)) // 64 rows of a tile in 32-bit byte offsets
            return MH3_ERR_SHAPE;
    }
    for (const uint64_t s : {a.q_head_stride, a.k_head_stride, a.v_head_stride, a.out_head_stride, a.k_page_stride,
                             a.k_page_head_stride, a.v_page_stride, a.v_page_head_stride}) {
        if (s % 8u != 0)
            return MH3_ERR_ALIGN;
        if (s >= (1ull << 36))
            return MH3_ERR_SHAPE;
    }
    return MH3_OK;
}

template <class Kernel>
int launch_items(Kernel kernel, uint32_t waves, size_t lds, const PagesParams& p, hipStream_t stream)
{
    if (const hipError_t e = host::allow_dynamic_lds(reinterpret_cast<const void*>(kernel), lds); e != hipSuccess)
        return host::hip_error(e);
    hipLaunchKernelGGL(kernel, dim3(p.workers), dim3(64u * waves), lds, stream, p);
    return host::check_launch();
}

template <bool CAP>
int launch_pages(const PagesParams& p, hipStream_t stream)
{
    if (p.item_rows > 32u)
        return launch_items(attn_pages_pair_kernel<CAP>, kPairWaves,
                            2u * kRing * kTileBytes + (kPairWaveBytes + 4u) * kPairWaves + 4u * kParents, p, stream);
    return launch_items(attn_pages_kernel<CAP>, 1u, 2u * kTileBytes + 1024u + 4u * kParents, p, stream);
}

} // namespace

extern "C" int64_t mh3_flash_attn_pages_128_workspace_bytes(const MH3PagesAttnArgs* args)
{
    if (const int rc = check_pages_args(args); rc != MH3_OK)
        return rc;
    return int64_t(pages_plan(*args).workspace);
}

extern "C" int mh3_flash_attn_pages_128(const MH3PagesAttnArgs* args, const uint16_t* q, const uint16_t* k,
                                        const uint16_t* v, const uint16_t* k_pages, const uint16_t* v_pages,
                                        const int32_t* table, const int32_t* lengths, const int32_t* q_off,
                                        const int32_t* parents, const int32_t* sinks, void* workspace,
                                        uint64_t workspace_bytes, uint16_t* out, mh3_stream_t stream)
{
    if (const int rc = check_pages_args(args); rc != MH3_OK)
        return rc;
    const MH3PagesAttnArgs& a = *args;
    const MH3PagesArgs& t = a.table;
    if (a.q_rows == 0)
        return MH3_OK;
    const PagesPlan plan = pages_plan(a);
    const uint64_t need = plan.workspace;
    if (!q || !k || !v || !k_pages || !v_pages || !table || !lengths || !q_off || !workspace || !out)
        return MH3_ERR_POINTER;
    if (workspace_bytes < need)
        return MH3_ERR_SHAPE;
    if (!host::aligned16(q) || !host::aligned16(k) || !host::aligned16(v) || !host::aligned16(k_pages) ||
        !host::aligned16(v_pages) || !host::aligned16(workspace) || !host::aligned16(out) ||
        (reinterpret_cast<uintptr_t>(table) | reinterpret_cast<uintptr_t>(lengths) | reinterpret_cast<uintptr_t>(q_off) |
         reinterpret_cast<uintptr_t>(parents) | reinterpret_cast<uintptr_t>(sinks)) %
                4u !=
            0u)
        return MH3_ERR_ALIGN;
    // out's rows apart from each other: heads one behind the other, or side by side in a row.
    const bool behind = a.heads == 1u || a.out_head_stride >= (a.q_rows - 1u) * a.out_row_stride + 128u;
    const bool beside = a.out_head_stride >= 128u &&
                        (a.q_rows == 1u || a.out_row_stride >= (a.heads - 1u) * a.out_head_stride + 128u);
    if (!behind && !beside)
        return MH3_ERR_PARAM;
    const auto span = [&](uint64_t heads, uint64_t hs, uint64_t rs) {
        return ((heads - 1u) * hs + (a.q_rows - 1ull) * rs + 128u) * 2u;
    };
    const auto pool = [&](uint64_t ps, uint64_t hs, uint64_t rs) {
        return ((t.pages - 1ull) * ps + (a.kv_heads - 1ull) * hs + (t.page_rows - 1ull) * rs + 128u) * 2u;
    };
    const host::Span in[] = {{q, span(a.heads, a.q_head_stride, a.q_row_stride)},
                             {k, span(a.kv_heads, a.k_head_stride, a.k_row_stride)},
                             {v, span(a.kv_heads, a.v_head_stride, a.v_row_stride)},
                             {k_pages, pool(a.k_page_stride, a.k_page_head_stride, a.k_page_row_stride)},
                             {v_pages, pool(a.v_page_stride, a.v_page_head_stride, a.v_page_row_stride)},
                             {table, ((t.streams - 1ull) * t.table_stride + t.cols) * 4u},
                             {lengths, t.streams * 4ull},
                             {q_off, (t.streams + 1ull) * 4u},
                             {parents, a.q_rows * 4ull},
                             {sinks, t.streams * 4ull}};
    const host::Span o[] = {{out, span(a.heads, a.out_head_stride, a.out_row_stride)}, {workspace, need}};
    if (host::any_overlap(in, o))
        return MH3_ERR_PARAM;
    PagesParams p{};
    p.q = q, p.k = k, p.v = v, p.out = out, p.k_pages = k_pages, p.v_pages = v_pages;
    p.table = table, p.lengths = lengths, p.q_off = q_off, p.parents = parents, p.first_rows = sinks;
    p.part = static_cast<float*>(workspace);
    p.qhs = a.q_head_stride, p.qrs = a.q_row_stride, p.khs = a.k_head_stride, p.krs = a.k_row_stride;
    p.vhs = a.v_head_stride, p.vrs = a.v_row_stride, p.ohs = a.out_head_stride, p.ors = a.out_row_stride;
    p.kps = a.k_page_stride, p.kphs = a.k_page_head_stride, p.kprs = a.k_page_row_stride;
    p.vps = a.v_page_stride, p.vphs = a.v_page_head_stride, p.vprs = a.v_page_row_stride;
    p.table_stride = t.table_stride, p.streams = t.streams, p.cols = t.cols, p.pages = t.pages;
    p.page_rows = t.page_rows, p.window = a.window, p.div_page = FastDiv::make(t.page_rows);
    p.kv_heads = a.kv_heads, p.group = a.heads / a.kv_heads, p.q_rows = a.q_rows, p.div_group = FastDiv::make(p.group);
    p.workers = plan.workers, p.slot_rows = plan.slot_rows, p.item_rows = plan.item_rows;
    p.zero_rest = a.zero_rest, p.div_item = FastDiv::make(plan.item_rows), p.begin = plan.item_rows > 32u ? kPairBegin : kBegin;
    score_factors(a.scale, a.cap, p);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (const int rc = a.cap > 0.0f ? launch_pages<true>(p, s) : launch_pages<false>(p, s); rc != MH3_OK)
        return rc;
    // Four waves to a row's parts where items have many (with two parts an item, 64 streams' single rows, 7.2 us, and 5.4 with
    // one wave), and as many workgroups as there may be pieces of rows, of one a CU to four (five cases at one, two and four,
    // us: 6.2, 6.4 and 7.1; 11.4, 8.0 and 7.3; 4.2, 4.4 and 5.0; 10.0, 7.9 and 7.0; 5.2, 5.2 and 5.3).
    const uint64_t cus = uint64_t(std::max(host::cu_count(), 1)), list = uint64_t(a.q_rows) * p.group;
    const uint64_t items = p.kv_heads * (list / p.item_rows + std::min(t.streams, a.q_rows));
    const bool split = p.workers > 8u * items;
    const uint64_t pieces = items + p.kv_heads * list / (split ? 2u : 8u);
    const uint32_t joiners = uint32_t(std::min(std::max(pieces, cus), 4u * cus));
    if (split)
        hipLaunchKernelGGL(attn_pages_join_kernel<4u>, dim3(joiners), dim3(256), 0, s, p);
    else
        hipLaunchKernelGGL(attn_pages_join_kernel<1u>, dim3(joiners), dim3(256), 0, s, p);
    return host::check_launch();
}
