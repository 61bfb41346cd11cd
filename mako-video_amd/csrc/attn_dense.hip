// `flash_attn_128`: flash attention over whole rows, head_dim 128, bf16 in and out: what a block runs without the sparse
// selection, for any count of query and key rows, shared key heads, a range of keys for each query row (documents packed
// into one batch, a prefix, causal rows), a second range (what a window has left behind and still keeps in sight), a tanh cap
// on the scores and a bias that falls with the distance.
//   s[i][j] = cap tanh(scale q_i . k_j / cap) - slope |q_pos_i - k_pos_j|   (without a cap: scale q_i . k_j)
//   out_i = sum_j softmax_j(s[i][j], j in [lo_i, hi_i) or [lo'_i, hi'_i)) v_j;   a row without keys is zero.
// The reference's counterpart of the plain case is mako-common's flash_attn_coop_128_32 (docs/performance.md).
//
// Design (gfx950, v_mfma_f32_32x32x16_bf16), the fragments and LDS images of attn.hip:
// - The query heads that share a key head are rows of one list, f = row group + g: a tile of such rows reads its K and V
//   once for all of them, and with one new row a stream fills the MFMA's columns with heads.
// - A wave takes 32 rows. Scores are transposed, S^T = K Q^T: a row's keys lie in one lane and its lane + 32 twin, so the
//   softmax's maximum and sum need one exchange, and P^T is the B operand of O^T += V^T P^T as it stands.
// - A workgroup walks the key tiles from its rows' lowest lo to their highest hi, under a bias from the last to the first:
//   a causal row's scores then fall from its own position on, and the first tile's maximum serves to the end (2 x 4096
//   causal rows, 40 heads on 8, slopes 2^-1 .. 2^-8: 571 us in rising order). A wave masks a tile only where its own
//   rows' ranges do not all cover it.
// - A masked probability is a zero, and zero times an infinite or NaN value of V would still be NaN in the rows that do
//   not attend it: masked tiles are searched for such values, and where there are any the matrix cores take zeros for
//   them, and they are added one key at a time to the rows that attend it. (All tiles masked, 40 heads, 14,080 rows on
//   11,264 keys: 3.75 ms, and 2.65 ms with none masked.)
// - Softmax in base 2. A row's running maximum is brought up to date only when a tile's probabilities sum up to more than
//   2^10 in a lane, so P stays below 2^10 and most tiles neither search a maximum nor rescale O. P rounds to bf16 for the
//   matrix cores (by up to 2^-8 of each probability, the sum takes them unrounded); maxima, sums and O are float.
// - A row's bits come from its own scores, its keys' values and the ranges. Waves and workgroups decide together what to
//   skip, never how a row rounds: that a neighbour attends an infinity or a far position leaves no trace. (One decision for
//   the wave's 32 rows instead: the same time within 2%.)
// - Of two ranges a workgroup walks the tiles of both, not those between them, and a row's keys of a masked tile are 64 bits
//   instead of two bounds: one pair of bounds is compared key by key in the scalar registers of each compare, and a second
//   pair's did not fit beside them. Which turns are masked is decided tile by tile: a walk's first and last of each range.
// - Eight waves load a tile together: the first four K three tiles ahead, the others V two, each a quarter, as soon as half
//   of a turn has made room (all eight waves loading K and then V: 945 rows of 56 heads 40.8 us for 39.6 now, 960 x 544
//   8,507 and 8,419, the packed clips below 1,503 and 1,474, 2 x 4096 causal rows of 40 heads on 8 under a bias 450 and 430).
// - Few rows leave the chip idle: their keys are then split over workgroups, each leaves its part of O, the maximum and the
//   sum in the workspace, and a second kernel joins them in a fixed order.
// What bounds it: many rows, the chip's power (960 x 544, 56 heads, 19,305 rows: 8.4 .. 8.9 ms, 1200 .. 1270 TFLOP/s, the
// clock at 1.65 to 1.7 GHz and the matrix cores busy 72% of it); under a cap also the vector unit's transcendentals (five
// clips packed into 14,925 rows of 40 heads 1475 us, without a cap 1230, with a multiplication in the place of the cap's
// exponential and reciprocal 1260); under a window also the turns that are masked and each workgroup's begin (960 x 544,
// 4080 keys back and the 435 first: 2160 .. 2290 us by card for 75 tiles a workgroup, 1.74 us a whole turn, 2.9 a masked one of
// which there are some nine, 4.7 the first, 5.8 before it, and 5 until the CU has its next workgroup); few rows, the one pass over K and V
// (129,536 keys of 8 heads in 95 us, 5.5 TB/s).
// Under a bias the eight-wave kernels hold six or seven registers in scratch, read between the loops, in masked turns and in
// rare paths, never in the loop of whole tiles; with a second range twenty, six of which each turn reads.
#include "attn_tiles.hpp"

#include <type_traits>

namespace mh3 {
namespace {

// Whether attn_few_kernel has less to do than attn_pair_kernel, from the key tiles that the rows of each one's workgroups
// span: in tenths of a us, a workgroup's start and its turns (plan_of's figures, and 2.0 and 2.8 us a turn of eight waves
// and of one whose rows do not attend the same keys), of the longest workgroup or of all of them over the CUs. Integers,
// so that both kernels find the same. A lane takes a tile of 32 rows, eight of them are a tile of 256.
__device__ __forceinline__ bool few_has_less(const DenseParams& p, uint32_t lane)
{
    uint32_t few_max = 0, pair_max = 0;
    uint64_t few_sum = 0, pair_sum = 0;
    for (uint32_t t0 = 0; t0 * 32u < p.list; t0 += 64u) {
        const uint32_t f0 = (t0 + lane) * 32u;
        uint32_t lo = ~0u, hi = 0u, all_lo = 0u, all_hi = ~0u;
        if (f0 < p.list) {
            const uint32_t r1 = p.div_group.div(min(f0 + 32u, p.list) - 1u);
            for (uint32_t r = p.div_group.div(f0); r <= r1; ++r) {
                uint32_t a, b;
                range_of(p, f0, r, a, b);
                if (a < b)
                    lo = min(lo, a), hi = max(hi, b);
                all_lo = max(all_lo, a), all_hi = min(all_hi, b);
            }
        }
        const auto alike = [&] { return all_lo < all_hi && uint64_t(all_hi - all_lo) * 8u >= uint64_t(hi - lo) * 7u; };
        const uint32_t few = lo < hi ? (hi - lo + 63u) / 64u * (alike() ? 15u : 28u) : 0u;
#pragma unroll
        for (int d = 1; d < 8; d *= 2) {
            lo = min(lo, uint32_t(__shfl_xor(int(lo), d, kWave))), hi = max(hi, uint32_t(__shfl_xor(int(hi), d, kWave)));
            all_lo = max(all_lo, uint32_t(__shfl_xor(int(all_lo), d, kWave)));
            all_hi = min(all_hi, uint32_t(__shfl_xor(int(all_hi), d, kWave)));
        }
        const uint32_t pair = (lane & 7u) == 0u && lo < hi ? (hi - lo + 63u) / 64u * (alike() ? 15u : 20u) : 0u;
        few_max = max(few_max, wave_max_u32(few)), pair_max = max(pair_max, wave_max_u32(pair));
        for (uint32_t i = 0; i < 64u; ++i)
            few_sum += uint32_t(__builtin_amdgcn_readlane(int(few), int(i)));
        for (uint32_t i = 0; i < 64u; i += 8u)
            pair_sum += uint32_t(__builtin_amdgcn_readlane(int(pair), int(i)));
    }
    const Contest& c = p.contest;
    const uint64_t few = 100u + max(uint64_t(few_max / c.few_splits), few_sum * p.kv_heads / (4u * c.cus));
    const uint64_t pair = 140u + max(uint64_t(pair_max / c.pair_splits), pair_sum * p.kv_heads / c.cus);
    return few < pair;
}

// Writes the wave's rows: normalized, or with splits the part of this split.
__device__ __forceinline__ void store_rows(const DenseParams& p, const WaveRows& w, uint32_t kvh, uint32_t f0,
                                           uint32_t split, uint32_t lane)
{
    const uint32_t n = lane & 31u, hh = lane >> 5, f = f0 + n;
    const float l = w.l_run + __shfl_xor(w.l_run, 32, kWave);
    if (f >= p.list)
        return;
    if (p.splits > 1u) {
        const uint64_t at = (uint64_t(split) * p.kv_heads + kvh) * p.list + f;
        float* const dst = p.part + at * 128u;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<float4*>(dst + 32 * db + 8 * g + 4u * hh) =
                    float4{w.o[db][4 * g], w.o[db][4 * g + 1], w.o[db][4 * g + 2], w.o[db][4 * g + 3]};
        if (hh == 0)
            *reinterpret_cast<float2*>(p.part + uint64_t(p.splits) * p.kv_heads * p.list * 128u + at * 2u) =
                float2{w.m_run, l};
        return;
    }
    const uint32_t row = p.div_group.div(f), head = kvh * p.group + (f - row * p.group);
    // A row without keys is zero; one whose scores are all -inf divides zero by zero.
    const float inv = w.lo < w.hi ? 1.0f / l : 0.0f;
    uint16_t* const dst = p.out + uint64_t(head) * p.ohs + uint64_t(row) * p.ors;
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<uint2*>(dst + 32 * db + 8 * g + 4u * hh) =
                uint2{pack_bf16(w.o[db][4 * g] * inv, w.o[db][4 * g + 1] * inv),
                      pack_bf16(w.o[db][4 * g + 2] * inv, w.o[db][4 * g + 3] * inv)};
}

// This workgroup's key head, row tile and split. Blocks go to the 8 XCDs round-robin; each XCD takes a contiguous part of
// the tiles, key head by key head, so that those running on it walk the same K and V. Within a head the last rows go
// first: under a causal mask they are the longest.
__device__ __forceinline__ bool block_of(const DenseParams& p, uint32_t& kvh, uint32_t& tile, uint32_t& split)
{
    const uint32_t per = gridDim.x / 8u, l = (blockIdx.x % 8u) * per + blockIdx.x / 8u;
    const uint32_t t = p.div_splits.div(l);
    split = l - t * p.splits;
    kvh = p.div_tiles.div(t);
    tile = p.tiles - 1u - (t - kvh * p.tiles);
    return kvh < p.kv_heads;
}

// The key tiles [first, last) of a workgroup's, for its split.
__device__ __forceinline__ void split_of(const DenseParams& p, uint32_t tiles, uint32_t split, uint32_t& first,
                                         uint32_t& last)
{
    first = uint32_t(uint64_t(tiles) * split / p.splits);
    last = uint32_t(uint64_t(tiles) * (split + 1u) / p.splits);
}

// The same where its rows' keys lie in [k0, k1).
__device__ __forceinline__ void tiles_of(const DenseParams& p, uint32_t k0, uint32_t k1, uint32_t split, uint32_t& first,
                                         uint32_t& last)
{
    split_of(p, k0 < k1 ? (k1 - k0 + 63u) / 64u : 0u, split, first, last);
}

template <bool SINKS>
using Seen = std::conditional_t<SINKS, BitsSeen, RangeSeen>;

// The key tiles of rows whose keys lie in [k0, k1), and of SINKS' in [s0, s1) before them: those of the front and, behind a
// gap, the others'; without room for a gap all of them as one.
struct Walk {
    uint32_t s0, front, k0, tiles;
    __device__ __forceinline__ Walk(uint32_t s_first, uint32_t s_last, uint32_t first, uint32_t last)
    {
        s0 = 0, front = 0, k0 = first;
        const uint32_t count = s_first < s_last ? (s_last - s_first + 63u) / 64u : 0u;
        if (count && first < last && s_first + 64u * count <= first)
            s0 = s_first, front = count;
        else if (count)
            k0 = min(first, s_first), last = max(last, s_last); // first is ~0 where no row has other keys
        tiles = front + (k0 < last ? (last - k0 + 63u) / 64u : 0u);
    }
    __device__ __forceinline__ uint32_t key(uint32_t i) const { return i < front ? s0 + 64u * i : k0 + 64u * (i - front); }
};

// What attn_few_kernel loads of a tile: K and, in the slot of its turn, the key positions; or V.
template <bool BIAS>
struct FewLoads {
    TileLoads<16, false> load_k;
    TileLoads<16, true> load_v;
    const uint16_t* kh;
    const uint16_t* vh;
    char* lds; // K, V, the wave's scratch (1 KB), two tiles' key positions
    __device__ __forceinline__ int32_t* positions(uint32_t t) const
    {
        return reinterpret_cast<int32_t*>(lds + 2u * kTileBytes + 1024u + 256u * (t & 1u));
    }
    __device__ __forceinline__ void k(const DenseParams& p, uint32_t t, uint32_t t0, uint32_t lane) const
    {
        load_k(lds, kh + uint64_t(t0) * p.krs, p.kv_rows - t0);
        if (BIAS) // no positions: no records, and zeros
            load_lds4(buffer_words(p.k_pos ? p.k_pos + t0 : nullptr, p.k_pos ? (p.kv_rows - t0) * 4u : 0u),
                      reinterpret_cast<char*>(positions(t)), 4u * lane);
    }
    __device__ __forceinline__ void v(const DenseParams& p, uint32_t t0) const
    {
        load_v(lds + kTileBytes, vh + uint64_t(t0) * p.vrs, p.kv_rows - t0);
    }
};

// A turn of attn_few_kernel, tile t at key t0; next: the next tile's key, if there is one (more). A tile's K is on its way
// from the products before it to its own, its V from the output before.
template <bool CAP, bool BIAS, bool SINKS, bool MASKED>
__device__ __forceinline__ void few_turn(const DenseParams& p, WaveRows& w, const FewLoads<BIAS>& feed,
                                         const TileReads& rd, uint32_t t, uint32_t t0, bool more, uint32_t next,
                                         uint32_t lane)
{
    const Seen<SINKS> seen(w, t0, lane);
    uint16_t* const scratch = reinterpret_cast<uint16_t*>(feed.lds + 2u * kTileBytes);
    const char* const vt = feed.lds + kTileBytes;
    floatx16 s[2];
    bf16x8_t frag[kAhead];
    TileP pt;
    wait_vm<16>(); // K and the positions; V may still be in flight
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
        frag[j] = rd.k(feed.lds, j);
    tile_products<false, false>(w, s, pt, frag, rd, feed.lds, nullptr, 0, nullptr, lane);
    wait_lds();
    if (more) {
        feed.k(p, t + 1u, next, lane);
        __builtin_amdgcn_sched_barrier(0);
    }
    tile_softmax<CAP, BIAS, MASKED>(p, w, s, pt, t0, seen, feed.positions(t), reinterpret_cast<float*>(scratch), false,
                                    false, lane);
    if (more)
        wait_vm<BIAS ? 17 : 16>(); // V, but not the next K
    else
        wait_vm<0>();
    if (MASKED && holds_nonfinite<16>(vt, lane))
        tile_output_masked(w, pt, rd, vt, seen, scratch, lane);
    else
        tile_output(w, pt, frag, rd, vt);
    wait_lds();
    if (more)
        feed.v(p, next);
}

// Few rows: one wave of 32 list rows a workgroup, with a tile of its own in LDS; four or five of them share a CU, and
// one's loads arrive while the others compute.
template <bool CAP, bool BIAS, bool SINKS>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(1, 1))) void attn_few_kernel(DenseParams p)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    uint32_t kvh, tile, split;
    if (!block_of(p, kvh, tile, split))
        return;
    const uint32_t lane = threadIdx.x;
    if (p.contest.few_splits) {
        if (!few_has_less(p, lane))
            return;
        if (blockIdx.x == 0 && lane == 0)
            *p.contest.winner = p.splits;
    }
    WaveRows w;
    load_rows<CAP, BIAS, SINKS>(p, kvh, tile * 32u, lane, w);
    uint32_t first, last;
    Walk walk(0u, 0u, 0u, 0u);
    if (SINKS) {
        walk = Walk(w.any_s_lo, w.any_s_hi, w.any_lo, w.any_hi);
        split_of(p, walk.tiles, split, first, last);
    } else {
        tiles_of(p, w.any_lo, w.any_hi, split, first, last);
    }
    const FewLoads<BIAS> feed{{p.krs, 0u, lane},
                              {p.vrs, 0u, lane},
                              p.k + uint64_t(kvh) * p.khs,
                              p.v + uint64_t(kvh) * p.vhs,
                              lds};
    const TileReads rd(lane);
    const uint32_t tiles = last - first;
    const auto key_of = [&](uint32_t t) {
        const uint32_t i = BIAS ? last - 1u - t : first + t;
        return SINKS ? walk.key(i) : w.any_lo + 64u * i;
    };
    const auto masks = [&](uint32_t t0) {
        return w.masks(t0) && !(SINKS && t0 >= w.all_s_lo && t0 + 64u <= w.all_s_hi);
    };
    if (tiles) {
        feed.k(p, 0u, key_of(0u), lane);
        feed.v(p, key_of(0u));
    }
    // Two loops, the masked tiles' and the whole ones': one body with both forms copies O between them at every tile.
    for (uint32_t t = 0; t < tiles;) {
#pragma unroll 1
        for (; t < tiles && masks(key_of(t)); ++t)
            few_turn<CAP, BIAS, SINKS, true>(p, w, feed, rd, t, key_of(t), t + 1u < tiles, key_of(t + 1u), lane);
#pragma unroll 1
        for (; t < tiles && !masks(key_of(t)); ++t)
            few_turn<CAP, BIAS, SINKS, false>(p, w, feed, rd, t, key_of(t), t + 1u < tiles, key_of(t + 1u), lane);
    }
    store_rows(p, w, kvh, tile * 32u, split, lane);
}

// What a wave loads of a workgroup's tiles, a call a tile: its quarter of K, or of V. After the workgroup's last tile the
// same again, so that every turn has the same count of loads; these are not read. The state is scalar and moves by
// additions.
// With JUMP, between the tile after which `jump` more are to come and the next one, the gap between the two parts of a walk.
template <bool JUMP>
struct PairStream {
    uint32_t row, off[4];     // bytes from a key to the next; the lane's in its four instructions
    char* quarter;            // of the ring's first tile
    uint32_t slot;            // byte offset in the ring
    const uint16_t* at;       // the next tile's first key
    int64_t step;             // elements to the one after it
    uint32_t left, left_step; // keys from it on
    uint32_t more;            // tiles after it
    uint32_t jump, gap;       // keys more to the next tile's
    __device__ __forceinline__ PairStream(bool value, uint64_t stride, uint32_t wave, uint32_t lane, char* ring,
                                          const uint16_t* first, uint32_t keys, bool back, uint32_t tiles, uint32_t jump_at,
                                          uint32_t gap_keys)
        : row(uint32_t(stride) * 2u), quarter(ring + 4096u * (wave % kHalf)), slot(0u), at(first),
          step((back ? -64 : 64) * int64_t(stride)), left(keys), left_step(back ? 64u : -64u), more(tiles - 1u), jump(jump_at),
          gap(gap_keys)
    {
        // As TileLoads: instruction i holds keys 4 i .. 4 i + 3, and 4 (wave % 4) is the first.
        const uint32_t key = value ? (lane >> 2) & 3u : lane >> 4;
#pragma unroll
        for (uint32_t u = 0; u < 4u; ++u) {
            const uint32_t chunk = value ? 4u * (lane >> 4) + (lane & 3u) : (lane & 15u) ^ (4u * u + key);
            off[u] = (16u * (wave % kHalf) + 4u * u + key) * row + 16u * chunk;
        }
    }
    __device__ __forceinline__ void operator()()
    {
        const u32x4_t r = buffer_words(at, (min(64u, left) - 1u) * row + 256u);
#pragma unroll
        for (uint32_t u = 0; u < 4u; ++u)
            load_lds16(r, quarter + slot + 1024u * u, off[u]);
        slot = (slot + kTileBytes) & (kRing * kTileBytes - 1u);
        at += more ? step : 0;
        left += more ? left_step : 0u;
        if (JUMP && more == jump) {
            const bool back = step < 0;
            at += (back ? -int64_t(gap) : int64_t(gap)) * int64_t(row / 2u);
            left += back ? gap : -gap;
        }
        more -= more ? 1u : 0u;
    }
};

// Under a bias each wave loads all of a tile's key positions into a ring of its own, a turn's with those of K.
template <bool JUMP>
struct PosStream {
    char* ring;
    uint32_t slot;
    const int32_t* pos; // null: no records, and zeros
    uint32_t left, more, jump, gap, lane;
    __device__ __forceinline__ void operator()()
    {
        load_lds4(buffer_words(pos, pos ? left * 4u : 0u), ring + slot, 4u * lane);
        slot = (slot + 256u) & (kRing * 256u - 1u);
        // From the last tile to the first.
        const uint32_t back = (more ? 64u : 0u) + (JUMP && more == jump ? gap : 0u);
        pos -= pos ? back : 0u;
        left += back;
        more -= more ? 1u : 0u;
    }
};

template <bool BIAS, bool SINKS>
struct PairFeed {
    static constexpr int kLoads = BIAS ? 5 : 4; // of a turn
    PairStream<SINKS> stream;
    PosStream<SINKS> pos;
    char* lds;
    __device__ __forceinline__ const char* k_tile(uint32_t t) const { return lds + (t % kRing) * kTileBytes; }
    __device__ __forceinline__ const char* v_tile(uint32_t t) const { return lds + (kRing + t % kRing) * kTileBytes; }
    __device__ __forceinline__ int32_t* positions(uint32_t t) const
    {
        return reinterpret_cast<int32_t*>(pos.ring + (t % kRing) * 256u);
    }
    // In turn t: K of tile t + 3 or V of tile t + 2, and the positions of tile t + 3.
    __device__ __forceinline__ void next(uint32_t)
    {
        stream();
        if (BIAS)
            pos();
    }
};

// The tiles of a workgroup's walk over two parts.
template <bool BIAS>
struct PairWalk {
    const Walk& walk;
    uint32_t first, last;
    uint32_t all_lo, all_hi, all_s_lo, all_s_hi;
    const uint4* rows; // the wave's rows' ranges
    uint32_t lane;
    __device__ __forceinline__ uint32_t key(uint32_t t) const { return walk.key(BIAS ? last - 1u - t : first + t); }
    __device__ __forceinline__ bool whole(uint32_t t) const
    {
        const uint32_t t0 = key(t);
        return (t0 >= all_lo && t0 + 64u <= all_hi) || (t0 >= all_s_lo && t0 + 64u <= all_s_hi);
    }
    __device__ __forceinline__ BitsSeen seen(uint32_t t) const
    {
        const uint4 r = rows[lane & 31u];
        const uint32_t t0 = key(t);
        return BitsSeen(key_bits(r.x, r.y, t0) | key_bits(r.z, r.w, t0), lane);
    }
};

template <bool CAP, bool BIAS, bool SINKS>
__global__ __launch_bounds__(kPairWaves * 64) __attribute__((amdgpu_waves_per_eu(2))) void attn_pair_kernel(DenseParams p)
{
    // K ring, V ring, then a wave's scratch (1 KB) and ring of key positions (1 KB), and the waves' spans.
    extern __shared__ __attribute__((aligned(16))) char lds[];
    uint32_t kvh, tile, split;
    if (!block_of(p, kvh, tile, split))
        return;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (p.contest.few_splits) {
        if (few_has_less(p, lane))
            return; // every wave finds the same
        if (blockIdx.x == 0 && tid == 0)
            *p.contest.winner = p.splits;
    }
    constexpr uint32_t kWaveBytes = SINKS ? 2048u + 512u : 2048u;
    uint16_t* const scratch = reinterpret_cast<uint16_t*>(lds + 2u * kRing * kTileBytes + kWaveBytes * wave);
    uint32_t* const span = reinterpret_cast<uint32_t*>(lds + 2u * kRing * kTileBytes + kWaveBytes * kPairWaves);
    const uint32_t f0 = (tile * kPairWaves + wave) * 32u;
    WaveRows w;
    if (SINKS)
        load_ranges<CAP, BIAS, true>(p, kvh, f0, lane, w); // the queries when the first tiles are on their way
    else
        load_rows<CAP, BIAS, false>(p, kvh, f0, lane, w);
    uint32_t* const odd = span + 4u * kPairWaves; // [2][kHalf]: a masked tile's V holds an infinity or a NaN
    uint32_t* const s_span = odd + 2u * kHalf;     // SINKS
    // SINKS: the rows' ranges, out of the registers: only masked turns ask for them.
    uint4* const rows = reinterpret_cast<uint4*>(scratch + 1024u);
    if (SINKS && lane < 32u)
        rows[lane] = uint4{w.lo, w.hi, w.s_lo, w.s_hi};
    if (lane == 0) {
        *reinterpret_cast<uint4*>(span + 4u * wave) = uint4{w.any_lo, w.any_hi, w.all_lo, w.all_hi};
        if (SINKS)
            *reinterpret_cast<uint4*>(s_span + 4u * wave) = uint4{w.any_s_lo, w.any_s_hi, w.all_s_lo, w.all_s_hi};
    }
    lds_barrier();
    uint32_t k0 = ~0u, k1 = 0u, all_lo = 0u, all_hi = ~0u; // of the workgroup's rows
#pragma unroll
    for (uint32_t i = 0; i < kPairWaves; ++i) {
        const uint4 t = *reinterpret_cast<const uint4*>(span + 4u * i);
        k0 = min(k0, t.x), k1 = max(k1, t.y), all_lo = max(all_lo, t.z), all_hi = min(all_hi, t.w);
    }
    k0 = __builtin_amdgcn_readfirstlane(k0), k1 = __builtin_amdgcn_readfirstlane(k1);
    all_lo = __builtin_amdgcn_readfirstlane(all_lo), all_hi = __builtin_amdgcn_readfirstlane(all_hi);
    uint32_t first, last;
    Walk walk(0u, 0u, 0u, 0u);
    uint32_t all_s_lo = 0u, all_s_hi = ~0u;
    if (SINKS) {
        uint32_t s0 = ~0u, s1 = 0u;
#pragma unroll
        for (uint32_t i = 0; i < kPairWaves; ++i) {
            const uint4 t = *reinterpret_cast<const uint4*>(s_span + 4u * i);
            s0 = min(s0, t.x), s1 = max(s1, t.y), all_s_lo = max(all_s_lo, t.z), all_s_hi = min(all_s_hi, t.w);
        }
        all_s_lo = __builtin_amdgcn_readfirstlane(all_s_lo), all_s_hi = __builtin_amdgcn_readfirstlane(all_s_hi);
        walk = Walk(__builtin_amdgcn_readfirstlane(s0), __builtin_amdgcn_readfirstlane(s1), k0, k1);
        split_of(p, walk.tiles, split, first, last);
    } else {
        tiles_of(p, k0, k1, split, first, last);
    }
    if (first >= last) { // the same for every wave
        if (SINKS)
            load_queries(p, kvh, f0, lane, w); // for its zeros
        store_rows(p, w, kvh, f0, split, lane);
        return;
    }
    k0 += 64u * first;
    const uint32_t tiles = last - first;
    // Turn t's tile.
    const auto key_of = [&](uint32_t t) {
        return SINKS ? walk.key(BIAS ? last - 1u - t : first + t) : k0 + 64u * (BIAS ? tiles - 1u - t : t);
    };
    // SINKS: the gap, and the tiles that are to come when the walk is at the last one before it.
    const bool both = SINKS && first < walk.front && last > walk.front;
    const uint32_t gap = both ? walk.k0 - walk.s0 - 64u * walk.front : 0u;
    const uint32_t jump = both ? (BIAS ? walk.front - first : last - walk.front) : ~0u;
    const TileReads rd(lane);
    const uint32_t from = key_of(0);
    const bool second = wave >= kHalf;
    const uint64_t head = uint64_t(kvh) * (second ? p.vhs : p.khs), row = second ? p.vrs : p.krs;
    PairFeed<BIAS, SINKS> feed{{second, row, wave, lane, lds + (second ? kRing * kTileBytes : 0u),
                                (second ? p.v : p.k) + head + uint64_t(from) * row, p.kv_rows - from, BIAS, tiles, jump, gap},
                               {reinterpret_cast<char*>(scratch) + 1024, 0u, p.k_pos ? p.k_pos + from : nullptr,
                                p.kv_rows - from, tiles - 1u, jump, gap, lane},
                               lds};
    // K of tiles 0, 1 and 2, or V of tiles 0 and 1, each turn's loads together.
    if (second) {
        if (BIAS)
            feed.pos();
        feed.next(0u);
        feed.next(0u);
    } else {
        feed.next(0u);
        feed.next(0u);
        feed.next(0u);
    }
    if (SINKS) {
        load_queries(p, kvh, f0, lane, w);
        PairWalk<BIAS> turns{walk, first, last, all_lo, all_hi, all_s_lo, all_s_hi, rows, lane};
        pair_walk<CAP, BIAS>(p, w, feed, turns, rd, scratch, odd, wave, tiles, f0 < p.list, lane);
        const uint4 r = rows[lane & 31u];
        w.lo = r.x, w.hi = r.y;
        store_rows(p, w, kvh, f0, split, lane);
        return;
    }
    wait_vm<2 * PairFeed<BIAS, SINKS>::kLoads>(); // K of tile 0
    lds_barrier();
    if (second)
        phase_barrier();
    floatx16 s[2];
    bf16x8_t frag[kAhead];
    TileP pt;
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
        frag[j] = rd.k(lds, j);
    // The turns in between, whose own tile and the one before are whole for every row of the workgroup, in a loop of their
    // own: one body with both forms copies O between them at every tile.
    uint32_t a = min(all_lo > k0 ? (all_lo - k0 + 63u) / 64u : 0u, tiles);
    uint32_t b = min(all_hi > k0 ? (all_hi - k0) / 64u : 0u, tiles);
    if (BIAS) {
        const uint32_t t = tiles - a;
        a = tiles - b, b = t;
    }
    a = min(a + 1u, tiles), b = max(a, b);
    const auto seen = [&](uint32_t t) { return RangeSeen(w, key_of(t), lane); };
#pragma unroll 1
    for (uint32_t t = 0; t < a; ++t)
        pair_turn<CAP, BIAS, true>(p, w, feed, rd, s, frag, pt, scratch, odd, true, wave, t, key_of(t), seen(t),
                                   seen(t - 1u), lane);
#pragma unroll 1
    for (uint32_t t = a; t < b; ++t)
        pair_turn<CAP, BIAS, false>(p, w, feed, rd, s, frag, pt, scratch, odd, true, wave, t, key_of(t), seen(t), seen(t),
                                    lane);
#pragma unroll 1
    for (uint32_t t = b; t < tiles; ++t)
        pair_turn<CAP, BIAS, true>(p, w, feed, rd, s, frag, pt, scratch, odd, t > b || a == b, wave, t, key_of(t), seen(t),
                                   seen(t - 1u), lane);
    const uint32_t end = tiles - 1u;
    if (!w.meets(key_of(end)))
        ; // nothing of it is this wave's
    else if (b < tiles || a == tiles) // the last turn was of the masked form
        masked_output(w, pt, frag, rd, feed.v_tile(end), seen(end), odd + kHalf * (end % 2u), scratch, lane);
    else
        tile_output(w, pt, frag, rd, feed.v_tile(end));
    if (!second)
        phase_barrier();
    wait_vm<0>(); // no load into this workgroup's LDS outlives it
    store_rows(p, w, kvh, f0, split, lane);
}

// Joins the splits of a list row, a workgroup of four waves each: every wave takes every fourth split, two values of d a
// lane, eight splits in flight, and the four sums meet in LDS in a fixed order.
__global__ __launch_bounds__(256) void attn_join_kernel(DenseParams p)
{
    __shared__ float part[4][4][64]; // a wave's maximum, sum and two values of O, by lane
    if (p.contest.few_splits) {
        p.splits = *p.contest.winner;
        if (p.splits == 1u)
            return; // the rows are written
    }
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint64_t item = blockIdx.x, items = uint64_t(p.kv_heads) * p.list;
    const uint32_t kvh = uint32_t(item / p.list), f = uint32_t(item - uint64_t(kvh) * p.list);
    const uint32_t row = p.div_group.div(f), head = kvh * p.group + (f - row * p.group);
    const float2* const ml = reinterpret_cast<const float2*>(p.part + uint64_t(p.splits) * items * 128u);
    constexpr uint32_t kU = 8;
    float m = -kInf, l = 0.0f, a = 0.0f, b = 0.0f;
    for (uint32_t s0 = wave; s0 < p.splits; s0 += 4u * kU) {
        float2 t[kU], o[kU];
#pragma unroll
        for (uint32_t u = 0; u < kU; ++u) {
            const uint32_t s = s0 + 4u * u;
            const bool in = s < p.splits;
            t[u] = in ? ml[s * items + item] : float2{-kInf, 0.0f};
            o[u] = in ? *reinterpret_cast<const float2*>(p.part + (s * items + item) * 128u + 2u * lane)
                      : float2{0.0f, 0.0f};
        }
        float m_new = m;
#pragma unroll
        for (uint32_t u = 0; u < kU; ++u)
            m_new = fmaxf(m_new, t[u].x);
        // A split without a key of this row has left zeros and -inf. (A NaN of its scores is in its sum and its O.)
        const float old = m == -kInf ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
        l *= old, a *= old, b *= old, m = m_new;
#pragma unroll
        for (uint32_t u = 0; u < kU; ++u) {
            const float e = t[u].x == -kInf ? 1.0f : __builtin_amdgcn_exp2f(t[u].x - m_new);
            l = fmaf(t[u].y, e, l), a = fmaf(o[u].x, e, a), b = fmaf(o[u].y, e, b);
        }
    }
    part[wave][0][lane] = m, part[wave][1][lane] = l, part[wave][2][lane] = a, part[wave][3][lane] = b;
    __syncthreads();
    if (wave != 0)
        return;
    uint32_t lo, hi;
    range_of(p, f, row, lo, hi);
    if (p.sinks) {
        uint32_t s_lo, s_hi;
        sinks_of(p, f, row, lo, hi, s_lo, s_hi);
    }
    float mm = m;
#pragma unroll
    for (int w = 1; w < 4; ++w)
        mm = fmaxf(mm, part[w][0][lane]);
    l = a = b = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float e = part[w][0][lane] == -kInf ? 1.0f : __builtin_amdgcn_exp2f(part[w][0][lane] - mm);
        l = fmaf(part[w][1][lane], e, l), a = fmaf(part[w][2][lane], e, a), b = fmaf(part[w][3][lane], e, b);
    }
    const float inv = lo < hi ? 1.0f / l : 0.0f;
    *reinterpret_cast<uint32_t*>(p.out + uint64_t(head) * p.ohs + uint64_t(row) * p.ors + 2u * lane) =
        pack_bf16(a * inv, b * inv);
}

struct RangeParams {
    const int32_t* q_off;
    const int32_t* k_off;
    const int32_t* prefix;
    int2* ranges;
    uint32_t q_rows, kv_rows, docs, causal;
};

// The last document whose first row is at most i (of empty ones that start together the last), `docs` for a row of none.
__device__ __forceinline__ uint32_t document_of(const int32_t* q_off, uint32_t docs, uint32_t i)
{
    uint32_t a = 0, b = docs; // q_off[a - 1] <= i < q_off[b] in a sorted list
    while (a < b) {
        const uint32_t mid = (a + b) / 2u;
        if (q_off[mid + 1u] <= int32_t(i))
            a = mid + 1u;
        else
            b = mid;
    }
    return a < docs && q_off[a] <= int32_t(i) ? a : docs;
}

__global__ __launch_bounds__(256) void attn_ranges_kernel(RangeParams p)
{
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= p.q_rows)
        return;
    const uint32_t a = document_of(p.q_off, p.docs, i);
    int2 r{0, 0};
    if (a < p.docs) {
        // Diagonal and prefix lie where the offsets say, wherever the keys end: the result is what is cut off.
        const int64_t start = p.k_off[a], end = p.k_off[a + 1u], n = p.kv_rows;
        int64_t hi = end;
        if (p.causal) {
            const int64_t own = end - p.q_off[a + 1u] + i; // the last query row sits on the last key row
            const int64_t seen = start + (p.prefix ? max(p.prefix[a], 0) : 0);
            hi = min(end, max(own + 1, seen));
        }
        const int64_t lo = min(max(start, int64_t(0)), n);
        r = int2{int32_t(lo), int32_t(min(max(hi, lo), n))};
    }
    p.ranges[i] = r;
}

struct WindowParams {
    const int32_t* q_off;
    const int32_t* k_off;
    const int32_t* sinks;
    int2* ranges;
    int2* first;
    uint32_t q_rows, kv_rows, docs, causal, window;
};

__global__ __launch_bounds__(256) void attn_window_ranges_kernel(WindowParams p)
{
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= p.q_rows)
        return;
    const uint32_t d = document_of(p.q_off, p.docs, i);
    int2 r{0, 0}, s{0, 0};
    if (d < p.docs) {
        const int64_t start = p.k_off[d], end = p.k_off[d + 1u], n = p.kv_rows;
        const int64_t own = end - p.q_off[d + 1u] + i; // the last query row sits on the last key row
        const int64_t stop = p.causal ? min(end, own + 1) : end;
        const auto cut = [&](int64_t x) { return int32_t(min(max(x, int64_t(0)), n)); };
        const int64_t lo = max(start, own - p.window + 1), hi = min(stop, own + p.window);
        const int64_t front = min(stop, start + (p.sinks ? max(p.sinks[d], 0) : 0));
        if (lo < hi)
            r = int2{cut(lo), cut(hi)};
        // What the window does not cover: up to it, or on both sides of it, where the row sees the keys behind it too.
        if (start < front && !(lo <= start && front <= hi))
            s = lo < hi && front > lo && front <= hi ? int2{cut(start), cut(lo)} : int2{cut(start), cut(front)};
    }
    p.ranges[i] = r, p.first[i] = s.x < s.y ? s : int2{0, 0};
}

} // namespace
} // namespace mh3

namespace {

using namespace mh3;

struct Plan {
    uint32_t waves, splits;
    uint64_t tiles;
    double us; // estimated
};

// The key splits of a call for the kernel of `waves` waves a workgroup: those of least estimated time, of none and as many
// as give the chip one, two or four workgroups a CU. In us, measured: a workgroup of eight waves takes 14 and 1.5 a key
// tile (it has a CU to itself), one of a single wave 10 and 1.5 (four share a CU); K and V come from HBM once at 6 TB/s,
// and for each further row tile from the MALL or L2 at some 16; the join takes 6 and its parts' bytes. Heads, query and
// key rows, eight waves and one, each at its best splits (us): 56, 945 x 945 44 and 68; 40, 212 x 212 20 and 15; 7,
// 700 x 700 30 and 24; 40, 64 x 20,000 125 and 93; 40 on 8 key heads, 1 x 5000 18 and 15, 3 x 129,536 108 and 94; 7 on 1,
// 500 x 16,000 52 and 71; 56 on 8, 64 x 100,000 198 and 324.
Plan plan_of(const MH3DenseAttnArgs& a, uint32_t waves)
{
    const uint64_t list = uint64_t(a.q_rows) * (a.heads / a.kv_heads), key_tiles = (uint64_t(a.kv_rows) + 63u) / 64u;
    const uint64_t cus = uint64_t(std::max(host::cu_count(), 1));
    const double head_us = double(a.kv_heads) * a.kv_rows * 512.0 * 1e-6; // us a pass over K and V at 1 TB/s
    const bool pair = waves == kPairWaves;
    const uint64_t tiles = (list + 32u * waves - 1u) / (32u * waves), blocks = tiles * a.kv_heads;
    Plan best{};
    for (const uint64_t fill : {uint64_t(0), cus, 2u * cus, 4u * cus}) {
        // At least four key tiles a split.
        const uint64_t splits = std::max<uint64_t>(1u, std::min<uint64_t>({fill / blocks, key_tiles / 4u, 256u}));
        const uint64_t rounds = (blocks * splits + (pair ? cus : 4u * cus) - 1u) / (pair ? cus : 4u * cus);
        const double turns = double((key_tiles + splits - 1u) / splits);
        double us = std::max(double(rounds) * (pair ? 14.0 + 1.5 * turns : 10.0 + 1.5 * turns),
                             head_us * (1.0 / 6.0 + double(tiles - 1u) / 16.0));
        if (splits > 1u)
            us += 6.0 + double(splits) * double(a.kv_heads) * double(list) * 1040.0 * 1e-6 / 4.0;
        if (best.waves == 0u || us < best.us)
            best = Plan{waves, uint32_t(splits), tiles, us};
    }
    return best;
}

// Both kernels' plans, the one to run first. With ranges, few rows against many keys may be of many documents, of which a
// workgroup of eight waves spans several and walks all of their keys with most of its waves idle; or of one, where it
// reads K and V once for more rows. So that is decided on the device (few_has_less; contest), where a call is long
// enough for the second launch and the look at the ranges, some 6 us. One-wave workgroups then take more splits, as those
// that span two documents are longer than the others, where there are many (4 x 28 rows below: 7 splits 422, 14 282).
// Heads, documents, query rows of each, keys in all, eight waves and one at their best splits (us): 40 on 8, 64 x 1,
// 129,536 162 and 107; 3 x 4, 129,536 139 and 99; 1 x 28, 116,105 118 and 152; 4 x 28 227 and 267; 56 on 8, 1 x 64,
// 100,000 198 and 335; 2 x 64 314 and 341; 40, 4 x 64, 20,000 136 and 102; 56, 5 x 18, 63,257 484 and 429.
// Calls of these sizes without ranges hold no contest, but take the same splits where one-wave workgroups are the first
// plan: more of them than plan_of's is faster there too, or costs little (us, plan_of's splits and these: 56, 51 x 14,922 4
// 100 and 9 90; 16, 39 x 29,920 16 54 and 32 45; 392 on 56, 9 x 11,066 4 79 and 9 70; 35 on 7, 11 x 69,694 36 67 and
// 73 70; 7, 34 x 75,312 36 72 and 73 74).
// Nor do calls with a second range of keys, as few_has_less counts one a row: they take the first plan, made as if each row
// attended all keys, where the same rows with one range may find the other kernel or be held up by the look (us, both ranges
// of a window of 1020 keys and 16 first ones, and the window's alone; documents of 1024 keys each, 40 on 8: 64 x 1 124 and 77,
// 8 x 64 69 and 85).
struct Plans {
    Plan first, second;
    uint64_t list;
    bool contest;
};

Plans plans_of(const MH3DenseAttnArgs& a)
{
    const Plan pair = plan_of(a, kPairWaves);
    Plan few = plan_of(a, 1u);
    const uint64_t list = uint64_t(a.q_rows) * (a.heads / a.kv_heads);
    const bool contest = list > 32u && list <= 8192u && uint64_t(a.q_rows) * 4u <= a.kv_rows &&
                         (pair.splits > 1u || few.splits > 1u) && std::min(pair.us, few.us) >= 60.0;
    if (!contest)
        return pair.us < few.us ? Plans{pair, few, list, false} : Plans{few, pair, list, false};
    const uint64_t fill = (few.tiles > 8u ? 8u : 4u) * uint64_t(std::max(host::cu_count(), 1));
    few.splits = uint32_t(std::max<uint64_t>(
        1u, std::min<uint64_t>({fill / (few.tiles * a.kv_heads), (uint64_t(a.kv_rows) + 255u) / 256u, 256u})));
    return pair.us < few.us ? Plans{pair, few, list, true} : Plans{few, pair, list, true};
}

constexpr uint64_t kHeader = 16u; // bytes before the parts: the contest's winner

uint64_t workspace_bytes(const MH3DenseAttnArgs& a, const Plans& p)
{
    const uint32_t splits = p.contest ? std::max(p.first.splits, p.second.splits) : p.first.splits;
    return splits > 1u ? kHeader + uint64_t(splits) * a.kv_heads * p.list * 130u * 4u : 0u;
}

int check_args(const MH3DenseAttnArgs* args)
{
    if (!args)
        return MH3_ERR_POINTER;
    const MH3DenseAttnArgs& a = *args;
    if (a.heads == 0 || a.kv_heads == 0 || a.head_dim == 0 || a.heads % a.kv_heads != 0)
        return MH3_ERR_SHAPE;
    if (a.head_dim != 128)
        return MH3_ERR_UNSUPPORTED;
    // The factors made of them stay ordinary floats (cap_in where it is made), and the capped scores' error (2^-23 of the
    // cap) below bf16's.
    if (!(a.scale >= 0.0f && a.scale <= 0x1p100f) || !(a.cap == 0.0f || (a.cap >= 0x1p-60f && a.cap <= 1024.0f)))
        return MH3_ERR_PARAM;
    if (a.heads > 4096u || a.q_rows >= (1u << 30) || a.kv_rows >= (1u << 30) ||
        uint64_t(a.q_rows) * (a.heads / a.kv_heads) >= (1u << 30))
        return MH3_ERR_SHAPE;
    for (const uint64_t s : {a.q_row_stride, a.k_row_stride, a.v_row_stride, a.out_row_stride}) {
        if (s % 8u != 0)
            return MH3_ERR_ALIGN;
        if (s < 128u || s >= (1ull << 23)) // 64 rows of a tile in 32-bit byte offsets
            return MH3_ERR_SHAPE;
    }
    if ((a.q_head_stride | a.k_head_stride | a.v_head_stride | a.out_head_stride) % 8u != 0)
        return MH3_ERR_ALIGN;
    return MH3_OK;
}

template <typename Kernel>
int launch_rows(Kernel kernel, size_t lds, const DenseParams& p, uint32_t waves, hipStream_t stream)
{
    if (const hipError_t e = host::allow_dynamic_lds(reinterpret_cast<const void*>(kernel), lds); e != hipSuccess)
        return host::hip_error(e);
    const uint32_t blocks = (p.kv_heads * p.tiles * p.splits + 7u) / 8u * 8u;
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(waves * 64u), lds, stream, p);
    return host::check_launch();
}

template <bool CAP, bool BIAS, bool SINKS>
int launch_form(const DenseParams& p, uint32_t waves, hipStream_t stream)
{
    if (waves == kPairWaves)
        return launch_rows(attn_pair_kernel<CAP, BIAS, SINKS>,
                           2u * kRing * kTileBytes + (2048u + 16u + 4u + (SINKS ? 512u + 16u : 0u)) * kPairWaves, p, waves,
                           stream);
    return launch_rows(attn_few_kernel<CAP, BIAS, SINKS>, 2u * kTileBytes + 1024u + 512u, p, waves, stream);
}

template <bool CAP, bool BIAS>
int launch_dense(const DenseParams& p, uint32_t waves, hipStream_t stream)
{
    return p.sinks ? launch_form<CAP, BIAS, true>(p, waves, stream) : launch_form<CAP, BIAS, false>(p, waves, stream);
}

} // namespace

extern "C" int64_t mh3_flash_attn_128_workspace_bytes(const MH3DenseAttnArgs* args)
{
    if (const int rc = check_args(args); rc != MH3_OK)
        return rc;
    if (args->q_rows == 0)
        return 0;
    return int64_t(workspace_bytes(*args, plans_of(*args)));
}

extern "C" int mh3_flash_attn_128(const MH3DenseAttnArgs* args, const uint16_t* q, const uint16_t* k, const uint16_t* v,
                                  const int32_t* ranges, const float* slopes, const int32_t* q_pos, const int32_t* k_pos,
                                  void* workspace, uint64_t workspace_bytes, uint16_t* out, mh3_stream_t stream)
{
    return mh3_flash_attn_128_sinks(args, q, k, v, ranges, nullptr, slopes, q_pos, k_pos, workspace, workspace_bytes, out,
                                    stream);
}

extern "C" int mh3_flash_attn_128_sinks(const MH3DenseAttnArgs* args, const uint16_t* q, const uint16_t* k,
                                        const uint16_t* v, const int32_t* ranges, const int32_t* sinks,
                                        const float* slopes, const int32_t* q_pos, const int32_t* k_pos, void* workspace,
                                        uint64_t workspace_bytes_given, uint16_t* out, mh3_stream_t stream)
{
    if (const int rc = check_args(args); rc != MH3_OK)
        return rc;
    const MH3DenseAttnArgs& a = *args;
    if (a.q_rows == 0)
        return MH3_OK;
    const Plans plans = plans_of(a);
    const uint64_t need = workspace_bytes(a, plans);
    if (!q || !out || (a.kv_rows && (!k || !v)) || (need && !workspace))
        return MH3_ERR_POINTER;
    if (!q_pos != !k_pos || (q_pos && !slopes) || (sinks && !ranges))
        return MH3_ERR_POINTER;
    if (workspace_bytes_given < need)
        return MH3_ERR_SHAPE;
    if (!host::aligned16(q) || !host::aligned16(k) || !host::aligned16(v) || !host::aligned16(out) ||
        !host::aligned16(workspace) ||
        (reinterpret_cast<uintptr_t>(ranges) | reinterpret_cast<uintptr_t>(sinks)) % 8u != 0u ||
        (reinterpret_cast<uintptr_t>(slopes) | reinterpret_cast<uintptr_t>(q_pos) | reinterpret_cast<uintptr_t>(k_pos)) %
                4u !=
            0u)
        return MH3_ERR_ALIGN;
    // out's rows apart from each other: heads one behind the other, or side by side in a row.
    const bool behind = a.heads == 1u || a.out_head_stride >= (a.q_rows - 1u) * a.out_row_stride + 128u;
    const bool beside = a.out_head_stride >= 128u &&
                        (a.q_rows == 1u || a.out_row_stride >= (a.heads - 1u) * a.out_head_stride + 128u);
    if (!behind && !beside)
        return MH3_ERR_PARAM;
    const auto span = [](uint64_t heads, uint64_t hs, uint64_t rows, uint64_t rs) {
        return rows ? ((heads - 1u) * hs + (rows - 1u) * rs + 128u) * 2u : 0u;
    };
    const host::Span in[] = {{q, span(a.heads, a.q_head_stride, a.q_rows, a.q_row_stride)},
                             {k, span(a.kv_heads, a.k_head_stride, a.kv_rows, a.k_row_stride)},
                             {v, span(a.kv_heads, a.v_head_stride, a.kv_rows, a.v_row_stride)},
                             {ranges, uint64_t(a.q_rows) * 8u},
                             {sinks, uint64_t(a.q_rows) * 8u},
                             {slopes, a.heads * 4ull},
                             {q_pos, uint64_t(a.q_rows) * 4u},
                             {k_pos, uint64_t(a.kv_rows) * 4u}};
    const host::Span o[] = {{out, span(a.heads, a.out_head_stride, a.q_rows, a.out_row_stride)}, {workspace, need}};
    if (host::any_overlap(in, o))
        return MH3_ERR_PARAM;
    for (const Plan& plan : {plans.first, plans.second})
        if (plan.tiles * a.kv_heads * plan.splits * plan.waves * 64u >= (1ull << 31))
            return MH3_ERR_SHAPE;
    DenseParams p{};
    p.q = q, p.k = k, p.v = v, p.out = out, p.ranges = ranges, p.sinks = sinks, p.slopes = slopes;
    p.q_pos = q_pos, p.k_pos = k_pos;
    p.part = need ? reinterpret_cast<float*>(static_cast<char*>(workspace) + kHeader) : nullptr;
    p.qhs = a.q_head_stride, p.qrs = a.q_row_stride, p.khs = a.k_head_stride, p.krs = a.k_row_stride;
    p.vhs = a.v_head_stride, p.vrs = a.v_row_stride, p.ohs = a.out_head_stride, p.ors = a.out_row_stride;
    p.kv_heads = a.kv_heads, p.group = a.heads / a.kv_heads, p.q_rows = a.q_rows, p.kv_rows = a.kv_rows;
    p.list = uint32_t(plans.list);
    p.div_group = FastDiv::make(p.group);
    score_factors(a.scale, a.cap, p);
    const bool contest = plans.contest && ranges && !sinks;
    if (contest) {
        const bool pair_first = plans.first.waves == kPairWaves;
        p.contest = Contest{(pair_first ? plans.first : plans.second).splits, (pair_first ? plans.second : plans.first).splits,
                            uint32_t(std::max(host::cu_count(), 1)), static_cast<uint32_t*>(workspace)};
    }
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const bool cap = a.cap > 0.0f, bias = slopes != nullptr;
    const auto run = [&](const Plan& plan) {
        p.tiles = uint32_t(plan.tiles), p.splits = plan.splits;
        p.div_tiles = FastDiv::make(p.tiles), p.div_splits = FastDiv::make(p.splits);
        return cap ? bias ? launch_dense<true, true>(p, plan.waves, s) : launch_dense<true, false>(p, plan.waves, s)
                   : bias ? launch_dense<false, true>(p, plan.waves, s)
                          : launch_dense<false, false>(p, plan.waves, s);
    };
    int rc = run(plans.first);
    if (rc == MH3_OK && contest)
        rc = run(plans.second);
    if (rc != MH3_OK || (!contest && p.splits == 1u))
        return rc;
    const uint64_t items = uint64_t(p.kv_heads) * p.list;
    hipLaunchKernelGGL(attn_join_kernel, dim3(uint32_t(items)), dim3(256), 0, s, p);
    return host::check_launch();
}

extern "C" int mh3_attn_ranges(const MH3RangeArgs* args, const int32_t* q_off, const int32_t* k_off,
                               const int32_t* prefix, int32_t* ranges, mh3_stream_t stream)
{
    if (!args)
        return MH3_ERR_POINTER;
    const MH3RangeArgs& a = *args;
    if (a.causal > 1u || (prefix && !a.causal))
        return MH3_ERR_PARAM;
    if (a.docs == 0 || a.docs >= (1u << 30) || a.q_rows >= (1u << 30) || a.kv_rows >= (1u << 30))
        return MH3_ERR_SHAPE;
    if (a.q_rows == 0)
        return MH3_OK;
    if (!q_off || !k_off || !ranges)
        return MH3_ERR_POINTER;
    if ((reinterpret_cast<uintptr_t>(q_off) | reinterpret_cast<uintptr_t>(k_off) | reinterpret_cast<uintptr_t>(prefix)) %
                4u !=
            0u ||
        reinterpret_cast<uintptr_t>(ranges) % 8u != 0u)
        return MH3_ERR_ALIGN;
    const host::Span in[] = {{q_off, (a.docs + 1ull) * 4u}, {k_off, (a.docs + 1ull) * 4u}, {prefix, a.docs * 4ull}};
    const host::Span o[] = {{ranges, uint64_t(a.q_rows) * 8u}};
    if (host::any_overlap(in, o))
        return MH3_ERR_PARAM;
    const RangeParams p{q_off, k_off, prefix, reinterpret_cast<int2*>(ranges), a.q_rows, a.kv_rows, a.docs, a.causal};
    hipLaunchKernelGGL(attn_ranges_kernel, dim3((a.q_rows + 255u) / 256u), dim3(256), 0,
                       static_cast<hipStream_t>(stream), p);
    return host::check_launch();
}

extern "C" int mh3_attn_window_ranges(const MH3WindowArgs* args, const int32_t* q_off, const int32_t* k_off,
                                      const int32_t* sinks, int32_t* ranges, int32_t* first, mh3_stream_t stream)
{
    if (!args)
        return MH3_ERR_POINTER;
    const MH3WindowArgs& a = *args;
    if (a.causal > 1u || a.window == 0u)
        return MH3_ERR_PARAM;
    if (a.docs == 0 || a.docs >= (1u << 30) || a.q_rows >= (1u << 30) || a.kv_rows >= (1u << 30))
        return MH3_ERR_SHAPE;
    if (a.q_rows == 0)
        return MH3_OK;
    if (!q_off || !k_off || !ranges || !first)
        return MH3_ERR_POINTER;
    if ((reinterpret_cast<uintptr_t>(q_off) | reinterpret_cast<uintptr_t>(k_off) | reinterpret_cast<uintptr_t>(sinks)) % 4u !=
            0u ||
        (reinterpret_cast<uintptr_t>(ranges) | reinterpret_cast<uintptr_t>(first)) % 8u != 0u)
        return MH3_ERR_ALIGN;
    const host::Span in[] = {{q_off, (a.docs + 1ull) * 4u}, {k_off, (a.docs + 1ull) * 4u}, {sinks, a.docs * 4ull}};
    const host::Span o[] = {{ranges, uint64_t(a.q_rows) * 8u}, {first, uint64_t(a.q_rows) * 8u}};
    if (host::any_overlap(in, o))
        return MH3_ERR_PARAM;
    const WindowParams p{q_off,    k_off,     sinks,  reinterpret_cast<int2*>(ranges), reinterpret_cast<int2*>(first),
                         a.q_rows, a.kv_rows, a.docs, a.causal,                        a.window};
    hipLaunchKernelGGL(attn_window_ranges_kernel, dim3((a.q_rows + 255u) / 256u), dim3(256), 0,
                       static_cast<hipStream_t>(stream), p);
    return host::check_launch();
}
