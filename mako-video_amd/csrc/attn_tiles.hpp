// What the attention kernels over tiles of 64 keys share (attn_dense.hip, attn_pages.hip): a tile's way into LDS, a wave's 32
// rows, and their products and softmax with a tile. attn_dense.hip says why they are as they are.
#pragma once

#include "mh3_common.hpp"

#include <algorithm>
#include <cmath>
#include <limits>

namespace mh3 {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float floatx4_t __attribute__((ext_vector_type(4)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef unsigned short ushortx2 __attribute__((ext_vector_type(2)));
typedef short v4i16 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInf = __builtin_inff();
constexpr uint32_t kTileBytes = 16384; // 64 keys of K, or of V

// Ranges that the host has not seen: both kernels are launched, and each of their workgroups finds out from the ranges
// which of the two has less to do. The other ends at once.
struct Contest {
    uint32_t pair_splits, few_splits; // 0: no contest
    uint32_t cus;
    uint32_t* winner; // its splits, for the join
};

struct DenseParams {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    uint16_t* out;
    const int32_t* ranges;
    const int32_t* sinks; // SINKS: a second range of each query row
    const float* slopes;
    const int32_t* q_pos;
    const int32_t* k_pos;
    float* part; // splits > 1: O [splits][kv_heads][list][128], then (maximum, sum) [splits][kv_heads][list][2]
    uint64_t qhs, qrs, khs, krs, vhs, vrs, ohs, ors; // elements
    uint32_t kv_heads, group, q_rows, kv_rows, list; // list = q_rows group
    uint32_t tiles, splits;                          // row tiles a key head, key splits
    FastDiv div_group, div_tiles, div_splits;
    Contest contest;
    // A score comes from the matrix cores of q times a power of two, q_pow (exact), which leaves the rest of the scale: so
    // a dot product overflows only where the scaled score nearly would.
    float q_pow;
    float scale_log2;      // the factor of such a product that gives base-2 units (without a cap)
    float cap_in, cap_out; // exp2(cap_in x) = exp(2 scale / q_pow x / cap); cap log2(e)
};

// s_waitcnt that waits for vmcnt <= n only (gfx9 encoding), with no memory access moved across it.
template <int N>
__device__ __forceinline__ void wait_vm()
{
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt((N & 0xF) | ((N >> 4) << 14) | 0x0F70);
    __builtin_amdgcn_sched_barrier(0);
}

__device__ __forceinline__ void lds_barrier()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F); // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// A wave's LDS reads done, with no memory access moved across it.
__device__ __forceinline__ void wait_lds()
{
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0xC07F); // lgkmcnt(0)
    __builtin_amdgcn_sched_barrier(0);
}

// A raw buffer of `bytes` at base, as the instructions below take it: reads past its end return zeros.
__device__ __forceinline__ u32x4_t buffer_words(const void* base, uint32_t bytes)
{
    const uint64_t a = reinterpret_cast<uint64_t>(base);
    return u32x4_t{uint32_t(a), uint32_t(a >> 32) & 0xffffu, bytes, uint32_t(kRsrcFlags)};
}

// The workgroup's barrier alone, with nothing moved across it: between phases whose LDS reads are used up, or are meant to
// stay in flight.
__device__ __forceinline__ void phase_barrier()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
}

// 16 or 4 bytes a lane from a buffer straight into LDS, lane L's at lds + 16 L or 4 L. Written as assembly for what the
// compiler would make of the builtin here: it waits for every such load in flight before each transposed LDS read, as
// if one might land under it, which made a turn half as long again (the tiles' slots and the waits in pair_turn and
// few_turn order them). No vector register is written, so nothing is in flight that the compiler has to know
// of, and M0 is used by nothing else in this file.
__device__ __forceinline__ void load_lds16(const u32x4_t& buffer, char* lds, uint32_t offset)
{
    const uint32_t at = uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds));
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(at), "v"(offset),
                 "s"(buffer)
                 : "memory");
}
__device__ __forceinline__ void load_lds4(const u32x4_t& buffer, char* lds, uint32_t offset)
{
    const uint32_t at = uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds));
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(at), "v"(offset),
                 "s"(buffer)
                 : "memory");
}

// The keys [lo, hi) of list row f, within [0, kv_rows]; none for a row past the list.
__device__ __forceinline__ void range_of(const DenseParams& p, uint32_t f, uint32_t row, uint32_t& lo, uint32_t& hi)
{
    lo = 0, hi = f < p.list ? p.kv_rows : 0u;
    if (p.ranges && f < p.list) {
        const int2 r = *reinterpret_cast<const int2*>(p.ranges + 2ull * row);
        lo = uint32_t(min(max(r.x, 0), int32_t(p.kv_rows)));
        hi = uint32_t(min(max(r.y, int32_t(lo)), int32_t(p.kv_rows)));
    }
}

// List row f's second range [s_lo, s_hi), and [lo, hi) as it is with it: the one that lies behind, with a gap between them,
// or both as one and [0, 0).
__device__ __forceinline__ void sinks_of(const DenseParams& p, uint32_t f, uint32_t row, uint32_t& lo, uint32_t& hi,
                                         uint32_t& s_lo, uint32_t& s_hi)
{
    s_lo = s_hi = 0;
    if (f < p.list) {
        const int2 r = *reinterpret_cast<const int2*>(p.sinks + 2ull * row);
        s_lo = uint32_t(min(max(r.x, 0), int32_t(p.kv_rows)));
        s_hi = uint32_t(min(max(r.y, int32_t(s_lo)), int32_t(p.kv_rows)));
    }
    if (lo >= hi)
        lo = s_lo, hi = s_hi, s_lo = s_hi = 0;
    if (s_lo < s_hi && s_lo > lo) {
        const uint32_t a = s_lo, b = s_hi;
        s_lo = lo, s_hi = hi, lo = a, hi = b;
    }
    if (s_lo < s_hi && s_hi >= lo)
        lo = s_lo, hi = max(hi, s_hi), s_lo = s_hi = 0;
    if (s_lo >= s_hi)
        s_lo = s_hi = 0;
}

// N of a tile's 16 DMA instructions of K (VALUE false) or V, the ones from i0 on. Instruction i fills the LDS kilobyte
// 1024 i with keys 4 i .. 4 i + 3: of K 256-byte rows whose 16-byte chunks are XOR-swizzled by the row, of V the four keys'
// 64-byte pieces interleaved (so that operand and transposed reads hit distinct banks); each quad of lanes fetches one
// aligned 64-byte piece of a row. The descriptor ends behind the last key, so keys past it read zeros.
template <int N, bool VALUE>
struct TileLoads {
    // Instructions i and i + 4 of K, any two of V, differ by a multiple of the row stride.
    static constexpr int kOff = VALUE ? 1 : N < 4 ? N : 4;
    uint32_t row, off[kOff], i0; // row: bytes from a key to the next
    __device__ __forceinline__ TileLoads(uint64_t stride, uint32_t first, uint32_t lane)
        : row(uint32_t(stride) * 2u), i0(first)
    {
#pragma unroll
        for (uint32_t u = 0; u < uint32_t(kOff); ++u) {
            const uint32_t i = first + u;
            const uint32_t key = VALUE ? (lane >> 2) & 3u : lane >> 4;
            const uint32_t chunk = VALUE ? 4u * (lane >> 4) + (lane & 3u) : (lane & 15u) ^ (4u * (i & 3u) + key);
            off[u] = (4u * i + key) * row + 16u * chunk;
        }
    }
    // The tile whose first key is at `base`, `keys` >= 1 of whose 64 exist.
    __device__ __forceinline__ void operator()(char* dst, const uint16_t* base, uint32_t keys) const
    {
        const u32x4_t r = buffer_words(base, (min(64u, keys) - 1u) * row + 256u);
        uint32_t step = 4u * row;
        asm volatile("" : "+s"(step)); // an addition a load, not registers kept through the products
#pragma unroll
        for (uint32_t u = 0; u < uint32_t(N); ++u)
            load_lds16(r, dst + 1024u * (i0 + u), off[u % uint32_t(kOff)] + u / uint32_t(kOff) * uint32_t(kOff) * step);
    }
};

// A wave's 32 rows: their query fragments, and the state of their softmax and output.
struct WaveRows {
    bf16x8_t qf[8];  // B operand of S^T: lane (n, hh) holds d 16 dc + 8 hh .. + 7 of row n
    floatx16 o[4];   // O^T: d 32 db + 8 (i / 4) + 4 hh + i % 4 of row n
    float m_run, l_run;
    bool settled;    // every row has a maximum, of no more than 2^20 (0 stands for one in rows without keys)
    uint32_t lo, hi;            // the lane's row's keys
    uint32_t s_lo, s_hi;        // SINKS: and those before them, [0, 0) or with a gap up to lo
    bool begun;                 // SINKS: a masked tile has held some of them
    uint32_t all_lo, all_hi;    // keys that every row with any attends: [all_lo, all_hi)
    uint32_t any_lo, any_hi;    // keys that some row attends lie in [any_lo, any_hi)
    uint32_t any_s_lo, any_s_hi, all_s_lo, all_s_hi; // SINKS: the same of [s_lo, s_hi)
    float slope_log2;           // BIAS: the row's head's slope, in base-2 units
    int32_t q_pos, q_base;      // BIAS: the row's position, the wave's first row's
    float q_rel;                // BIAS: their difference, if q_near: it is under 2^23 in all of the wave's rows
    bool q_near;                // (and none of them is steep)
    bool steep;                 // a slope of the wave's rows is beyond 2^80 units of a score
    float slope_unit;
    // Whether the wave has work in the tile at key t0, and whether some row's range does not cover it.
    __device__ __forceinline__ bool meets(uint32_t t0) const { return t0 < any_hi && t0 + 64u > any_lo; }
    __device__ __forceinline__ bool masks(uint32_t t0) const { return t0 < all_lo || t0 + 64u > all_hi; }
};

// The keys of a masked tile, at key t0, that a lane's row attends.
struct RangeSeen {
    uint32_t lo, hi, t0, from_lo; // from_lo modulo 2^32: below lo is past every count
    __device__ __forceinline__ RangeSeen(const WaveRows& w, uint32_t tile, uint32_t lane)
        : lo(w.lo), hi(w.hi), t0(tile), from_lo(tile + 4u * (lane >> 5) - w.lo)
    {
    }
    // The lane's score i of block b, -inf where its key is not one of them.
    __device__ __forceinline__ float score(float s, int b, int i) const
    {
        return from_lo + (32u * b + 8u * (i >> 2) + (i & 3)) < hi - lo ? s : -kInf;
    }
    // Whether a row of the wave attends not all of block b's 32 keys (not asked here).
    __device__ __forceinline__ bool masks(int) const { return true; }
    // Whether key j of the tile is.
    __device__ __forceinline__ bool key(uint32_t j) const { return t0 + j >= lo && t0 + j < hi; }
    __device__ __forceinline__ bool any() const { return max(lo, t0) < min(hi, t0 + 64u); }
    // Whether the row's range begins here, in a walk from the last tile to the first where BACKWARD.
    template <bool BACKWARD>
    __device__ __forceinline__ bool begins(const WaveRows&) const
    {
        return BACKWARD ? hi <= t0 + 64u : lo >= t0;
    }
    __device__ __forceinline__ void note(WaveRows&) const {}
    // Whether the wave has work in the tile.
    __device__ __forceinline__ bool meets(const WaveRows& w) const { return w.meets(t0); }
};

// The bits of a tile's 64 keys, at key t0, that lie in [lo, hi).
__device__ __forceinline__ uint64_t key_bits(uint32_t lo, uint32_t hi, uint32_t t0)
{
    const uint32_t a = lo > t0 ? min(lo - t0, 64u) : 0u, b = hi > t0 ? min(hi - t0, 64u) : 0u;
    if (a >= b)
        return 0;
    return (~uint64_t(0) >> (64u - (b - a))) << a;
}

// The same of any 64 bits, a key's each.
struct BitsSeen {
    uint32_t word[2];
    uint32_t shift;
    __device__ __forceinline__ BitsSeen(uint64_t bits, uint32_t lane)
        : word{uint32_t(bits), uint32_t(bits >> 32)}, shift(4u * (lane >> 5))
    {
    }
    __device__ __forceinline__ BitsSeen(const WaveRows& w, uint32_t t0, uint32_t lane)
        : BitsSeen(key_bits(w.lo, w.hi, t0) | key_bits(w.s_lo, w.s_hi, t0), lane)
    {
    }
    // A bit over a whole register selects: comparisons took two scalar registers each, and the kernels to scratch.
    __device__ __forceinline__ float score(float s, int b, int i) const
    {
        const uint32_t m = uint32_t(__builtin_amdgcn_sbfe(int(word[b] >> shift), 8 * (i >> 2) + (i & 3), 1));
        return __uint_as_float((__float_as_uint(s) & m) | (0xff800000u & ~m));
    }
    __device__ __forceinline__ bool masks(int b) const { return __ballot(word[b] != ~0u) != 0u; }
    __device__ __forceinline__ bool key(uint32_t j) const { return word[j >> 5] >> (j & 31u) & 1u; }
    __device__ __forceinline__ bool any() const { return (word[0] | word[1]) != 0u; }
    template <bool BACKWARD>
    __device__ __forceinline__ bool begins(const WaveRows& w) const
    {
        return !w.begun;
    }
    __device__ __forceinline__ void note(WaveRows& w) const { w.begun |= any(); }
    __device__ __forceinline__ bool meets(const WaveRows&) const { return __ballot(any()) != 0u; }
};

// What one of a score as the products (and cap_scores) leave it is in base 2.
template <bool CAP>
__device__ __forceinline__ float score_unit(const DenseParams& p)
{
    return CAP ? 2.0f * p.cap_out : p.scale_log2;
}

__device__ __forceinline__ bool is_near(int32_t rel) { return rel > -(1 << 23) && rel < (1 << 23); }

// The query fragments of a wave's rows, and zeros for their output.
__device__ __forceinline__ void load_queries(const DenseParams& p, uint32_t kvh, uint32_t f0, uint32_t lane, WaveRows& w)
{
    const uint32_t n = lane & 31u, hh = lane >> 5, f = f0 + n;
    const uint32_t fc = min(f, p.list - 1u), row = p.div_group.div(fc), head = kvh * p.group + (fc - row * p.group);
    const uint16_t* const src = p.q + uint64_t(head) * p.qhs + uint64_t(row) * p.qrs;
#pragma unroll
    for (int dc = 0; dc < 8; ++dc) {
        const uint4 t = f < p.list ? *reinterpret_cast<const uint4*>(src + 16 * dc + 8u * hh) : uint4{0u, 0u, 0u, 0u};
        uint32_t x[4] = {t.x, t.y, t.z, t.w};
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
}

// The keys of a wave's rows, and what their bias goes by.
template <bool CAP, bool BIAS, bool SINKS>
__device__ __forceinline__ void load_ranges(const DenseParams& p, uint32_t kvh, uint32_t f0, uint32_t lane, WaveRows& w)
{
    const uint32_t f = f0 + (lane & 31u);
    const uint32_t fc = min(f, p.list - 1u), row = p.div_group.div(fc), head = kvh * p.group + (fc - row * p.group);
    range_of(p, f, row, w.lo, w.hi);
    if (SINKS) {
        sinks_of(p, f, row, w.lo, w.hi, w.s_lo, w.s_hi);
        const bool some = w.s_lo < w.s_hi;
        w.begun = false;
        w.any_s_lo = wave_min_u32(some ? w.s_lo : ~0u), w.any_s_hi = wave_max_u32(some ? w.s_hi : 0u);
        w.all_s_lo = wave_max_u32(w.s_lo), w.all_s_hi = wave_min_u32(f < p.list ? w.s_hi : ~0u);
    }
    const bool any = w.lo < w.hi;
    w.m_run = any ? -kInf : 0.0f, w.l_run = 0.0f, w.settled = false;
    w.any_lo = wave_min_u32(any ? w.lo : ~0u);
    w.any_hi = wave_max_u32(any ? w.hi : 0u);
    w.all_lo = wave_max_u32(w.lo); // a row of the list without keys masks every tile, one past it none
    w.all_hi = wave_min_u32(f < p.list ? w.hi : ~0u);
    if (BIAS) {
        w.slope_log2 = p.slopes[head] * kLog2e;
        w.q_pos = p.q_pos ? p.q_pos[row] : int32_t(row);
        w.q_base = __builtin_amdgcn_readfirstlane(w.q_pos);
        const int32_t rel = __builtin_elementwise_sub_sat(w.q_pos, w.q_base);
        w.q_rel = float(rel);
        w.slope_unit = w.slope_log2 / score_unit<CAP>(p);
        w.steep = __ballot(!(fabsf(w.slope_unit) <= 0x1p80f)) != 0;
        w.q_near = !w.steep && !__ballot(!is_near(rel));
    }
}

template <bool CAP, bool BIAS, bool SINKS>
__device__ __forceinline__ void load_rows(const DenseParams& p, uint32_t kvh, uint32_t f0, uint32_t lane, WaveRows& w)
{
    load_queries(p, kvh, f0, lane, w);
    load_ranges<CAP, BIAS, SINKS>(p, kvh, f0, lane, w);
}

// Scores x under a cap, without their factor and but for a constant, which a softmax does not see: tanh(u) =
// 1 - 2 / (exp(2 u) + 1), so cap tanh(u) log2(e) is cap_out + 2 cap_out times -1 / (exp2(cap_in x) + 1). At either end the
// exponential gives +-cap, and the error near zero is 2^-23 of the cap, below what bf16 operands leave of the score.
__device__ __forceinline__ void cap_scores(const DenseParams& p, floatx16 (&s)[2])
{
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            s[b][i] = __builtin_amdgcn_rcpf(-1.0f - __builtin_amdgcn_exp2f(s[b][i] * p.cap_in));
}

// The key positions of a tile as floats from the wave's base, if they and the wave's rows are all under 2^23 from it: the
// float differences are then exact, and the bias takes two operations a score. pos: the position of the tile's key `lane`;
// near_pos (64 floats of LDS, the wave's own) takes the result, zeros if this is not so.
__device__ __forceinline__ bool near_positions(const WaveRows& w, int32_t pos, float* near_pos, uint32_t lane)
{
    const int32_t rel = __builtin_elementwise_sub_sat(pos, w.q_base);
    const bool near = w.q_near && !__ballot(!is_near(rel));
    near_pos[lane] = near ? float(rel) : 0.0f;
    asm volatile("" ::: "memory"); // a wave's LDS accesses are in order
    return near;
}

// The bias off a score, from its key's position as near_positions leaves it.
__device__ __forceinline__ float less_bias(const WaveRows& w, float x, float slope_unit, float key)
{
    return fmaf(-slope_unit, fabsf(w.q_rel - key), x);
}

__device__ __forceinline__ floatx4_t near_four(const float* near_pos, int g, uint32_t lane)
{
    return *reinterpret_cast<const floatx4_t*>(near_pos + 8 * g + 4u * (lane >> 5));
}

// The bias off the scores, from the distances of int32 positions (kp: the tile's; the keys' numbers without k_pos), which
// are exact before they round to float. That is less_bias' own operation, so a row's bits do not depend on the positions that
// made its wave come here; or with a steep slope in the wave in base-2 units, as what is returned, the factor of the scores
// as they then stand, says.
__device__ __forceinline__ float bias_scores_far(const DenseParams& p, const WaveRows& w, floatx16 (&s)[2], float unit,
                                                 uint32_t t0, const int32_t* kp, uint32_t lane)
{
    const uint32_t given = p.k_pos ? ~0u : 0u; // no branch a score
    const float scale = w.steep ? unit : 1.0f, slope = w.steep ? w.slope_log2 : w.slope_unit;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t key = 32u * b + 8u * (i >> 2) + 4u * (lane >> 5) + (i & 3);
            const int32_t pos = int32_t((uint32_t(kp[key]) & given) | ((t0 + key) & ~given));
            // The distance of two int32 positions fits 32 bits without a sign.
            const uint32_t d = w.q_pos > pos ? uint32_t(w.q_pos) - uint32_t(pos) : uint32_t(pos) - uint32_t(w.q_pos);
            s[b][i] = fmaf(-slope, float(d), s[b][i] * scale);
            if (i % 4 == 3)
                __builtin_amdgcn_sched_barrier(0); // four positions' registers at a time
        }
    return w.steep ? 1.0f : unit;
}

// Where a wave's lanes find their operands in a tile's LDS images.
struct TileReads {
    uint32_t k_lane, v_lane;
    __device__ __forceinline__ explicit TileReads(uint32_t lane)
    {
        const uint32_t n = lane & 31u, hh = lane >> 5, L = lane & 15u, grp = lane >> 4;
        k_lane = 256u * n + 16u * (hh ^ (n & 15u));
        v_lane = 1024u * (grp >> 1) + 32u * (grp & 1u) + 64u * (L >> 2) + 8u * (L & 3u);
    }
    // A operand of S^T, j < 16: key block j % 2, d chunk j / 2.
    __device__ __forceinline__ bf16x8_t k(const char* kt, int j) const
    {
        return *reinterpret_cast<const bf16x8_t*>(kt + 8192u * (j & 1) + (k_lane ^ (32u * (j >> 1))));
    }
    // A operand of O^T, j < 16: 16-key chunk j / 4, d block j % 4, two transposed reads.
    __device__ __forceinline__ bf16x8_t v(const char* vt, int j) const
    {
        const char* const at = vt + v_lane + 4096u * (j >> 2) + 256u * (j & 3);
        const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (v4i16 __attribute__((address_space(3)))*)(const_cast<char*>(at)));
        const v4i16 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (v4i16 __attribute__((address_space(3)))*)(const_cast<char*>(at) + 2048u));
        return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
};

constexpr int kAhead = 8; // fragments read ahead of their MFMAs

// P^T of a tile: chunk c's words (elements 8 (c % 2) .. + 7 of block c / 2) are 4 c .. 4 c + 3.
struct TileP {
    uint32_t w[16];
    __device__ __forceinline__ bf16x8_t chunk(int c) const
    {
        return __builtin_bit_cast(bf16x8_t, uint4{w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]});
    }
};

// s unit - m in two roundings.
__device__ __forceinline__ float rounded_difference(float s, float unit, float m)
{
#pragma clang fp contract(off)
    const float x = s * unit;
    return x - m;
}

// The larger of a lane's value and its lane +- 32 twin's.
__device__ __forceinline__ float both_halves_max(float v)
{
    const uint32_t u = __float_as_uint(v);
    const auto t = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(t[0]), __uint_as_float(t[1]));
}

// P^T of a tile from its scores, exp2(factor s - m), and a row's sum of them over the lane's keys.
__device__ __forceinline__ float tile_exponentials(const floatx16 (&s)[2], TileP& pt, float factor, float m)
{
    float sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const int b = e >> 3, i = 2 * (e & 7);
        const floatx2 t = {__builtin_amdgcn_exp2f(fmaf(s[b][i], factor, -m)),
                           __builtin_amdgcn_exp2f(fmaf(s[b][i + 1], factor, -m))};
        sum[0] += t[0], sum[1] += t[1];
        pt.w[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(t, bf16x2_t)); // one conversion for both
    }
    return sum[0] + sum[1];
}

// The softmax of a tile at key t0 (MASKED: not every row attends all of it, but the keys that `seen` says): P^T, and the
// rows' maxima, sums and (where a maximum moved) rescaled O. BIAS: kp and near_pos are LDS for the tile's positions; sloped:
// tile_products has taken the bias off, if the positions are near.
template <bool CAP, bool BIAS, bool MASKED, class Seen>
__device__ __forceinline__ void tile_softmax(const DenseParams& p, WaveRows& w, floatx16 (&s)[2], TileP& pt, uint32_t t0,
                                             const Seen& seen, const int32_t* kp, float* near_pos, bool sloped, bool near,
                                             uint32_t lane)
{
    float factor = score_unit<CAP>(p); // of the scores as they stand: base-2 units
    if (CAP)
        cap_scores(p, s);
    if (BIAS) {
        if (!sloped) {
            near = near_positions(w, p.k_pos ? kp[lane] : int32_t(t0 + lane), near_pos, lane);
            if (near) {
#pragma unroll
                for (int g = 0; g < 8; ++g) {
                    const floatx4_t key = near_four(near_pos, g, lane);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s[g >> 2][4 * (g & 3) + e] = less_bias(w, s[g >> 2][4 * (g & 3) + e], w.slope_unit, key[e]);
                    if (g % 2)
                        __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        if (!near)
            factor = bias_scores_far(p, w, s, factor, t0, kp, lane);
    }
    if (MASKED) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
            if (seen.masks(b))
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    s[b][i] = seen.score(s[b][i], b, i);
    }
    // Most tiles raise no maximum by much, and the sum over a lane's 32 keys of a row tells: up to 2^10 no key is above
    // that, and the old maximum serves. That spares the search for the new one in a phase whose vector instructions take 7
    // clocks each beside the other group's MFMAs. Rows without a maximum or with a large one take the tile's without the
    // look at their sums, and so do all rows in a tile where the range of one of the wave's begins. Each row thus goes by its
    // own scores and by the ranges: none of its bits depends on the scores of the rows beside it.
    const auto known = [&] { return fabsf(w.m_run) <= 0x1p20f; };
    float m_ref = w.m_run, sum;
    bool asks = false, looks = true; // the row asks for its maximum; some row of the wave goes by its sum
    uint64_t asking = 0, over = 0;   // rows that ask, and lanes whose row asks by its sum
    if (MASKED) {
        const bool here = seen.any();
        const bool begins = __ballot(here && seen.template begins<BIAS>(w)) != 0; // with its last key under a bias
        seen.note(w);
        m_ref = known() ? m_ref : 0.0f; // a row without a key here has zeros for probabilities
        asks = here && (begins || !known());
        asking = __ballot(asks), looks = asking == 0 || __ballot(here && !asks) != 0;
    } else if (__builtin_expect(!w.settled, false)) {
        asks = !known();
        asking = __ballot(asks), looks = ~asking != 0;
    }
    if (__builtin_expect(looks, !MASKED)) {
        sum = tile_exponentials(s, pt, factor, m_ref);
        over = __ballot(!(sum <= 0x1p10f));
    }
    if (__builtin_expect((asking | over) != 0, MASKED)) {
        asks |= ((over | over >> 32 | over << 32) >> lane & 1u) != 0;
        float mt = -kInf;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                mt = fmaxf(mt, s[b][i]);
        mt = both_halves_max(mt) * factor;
        const float m_new = asks ? fmaxf(w.m_run, mt) : w.m_run;
        const float alpha = w.m_run == -kInf ? 0.0f : __builtin_amdgcn_exp2f(w.m_run - m_new);
        if (__ballot(m_new > w.m_run)) {
            w.l_run *= alpha;
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    w.o[b][i] *= m_new > w.m_run ? alpha : 1.0f;
        }
        w.m_run = m_new;
        w.settled = !__ballot(!known());
        m_ref = m_new == -kInf ? 0.0f : m_new;
        // factor s - m in one fused operation keeps the rounding of m, 2^-24 of it, in the exponent: common to all of a
        // row's probabilities and harmless, until it leaves the exponent's range. Scores so large are rounded as m was.
        const bool large = fabsf(m_ref) > 0x1p20f;
        if (__ballot(large)) {
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    s[b][i] = large ? rounded_difference(s[b][i], factor, m_ref) : fmaf(s[b][i], factor, -m_ref);
            m_ref = 0.0f, factor = 1.0f;
        }
        sum = tile_exponentials(s, pt, factor, m_ref);
    }
    w.l_run += sum;
}

// S^T of a tile, and then with PV the O^T += V^T P^T of another (the one before it in a walk), in one run of MFMAs: frag
// holds the first kAhead K fragments, and each MFMA's slot takes the fragment of the MFMA kAhead on, so V's are on their
// way before the last scores are out. SLOPED: the bias comes off the scores in the slots of the V^T P^T, where the vector
// unit is idle, if the key positions (pos: that of key `lane`) are near, which is returned.
template <bool PV, bool SLOPED>
__device__ __forceinline__ bool tile_products(WaveRows& w, floatx16 (&s)[2], const TileP& pt, bf16x8_t (&frag)[kAhead],
                                              const TileReads& rd, const char* kt, const char* vt, int32_t pos,
                                              float* near_pos, uint32_t lane)
{
    static_assert(PV || !SLOPED);
    bool near = false;
    float slope = 0.0f;
    floatx4_t key[8];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            s[b][i] = 0.0f;
#pragma unroll
    for (int j = 0; j < (PV ? 32 : 16); ++j) {
        __builtin_amdgcn_sched_barrier(0);
        bf16x8_t& f = frag[j % kAhead];
        if (j < 16)
            s[j & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f, w.qf[j >> 1], s[j & 1], 0, 0, 0);
        else
            w.o[j & 3] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f, pt.chunk((j - 16) >> 2), w.o[j & 3], 0, 0, 0);
        if (j + kAhead < 16)
            f = rd.k(kt, j + kAhead);
        else if (PV && j + kAhead < 32)
            f = rd.v(vt, j + kAhead - 16);
        if (SLOPED && j == 5) {
            near = near_positions(w, pos, near_pos, lane);
            slope = near ? w.slope_unit : 0.0f;
        }
        if (SLOPED && j >= 12 && j % 2 == 0 && j < 28)
            key[(j - 12) / 2] = near_four(near_pos, (j - 12) / 2, lane);
        if (SLOPED && j >= 17)
#pragma unroll
            for (int e = 2 * (j - 17); e < (j == 31 ? 32 : 2 * (j - 16)); ++e)
                s[e >> 4][e & 15] = less_bias(w, s[e >> 4][e & 15], slope, key[e >> 2][e & 3]);
    }
    __builtin_amdgcn_sched_barrier(0);
    return near;
}

// O^T += V^T P^T of a tile alone.
__device__ __forceinline__ void tile_output(WaveRows& w, const TileP& pt, bf16x8_t (&frag)[kAhead], const TileReads& rd,
                                            const char* vt)
{
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
        frag[j] = rd.v(vt, j);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        __builtin_amdgcn_sched_barrier(0);
        w.o[j & 3] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag[j % kAhead], pt.chunk(j >> 2), w.o[j & 3], 0, 0, 0);
        if (j + kAhead < 16)
            frag[j % kAhead] = rd.v(vt, j + kAhead);
    }
    __builtin_amdgcn_sched_barrier(0);
}

// All ones in each half of a bf16 pair that is an infinity or a NaN: the sum carries out of an exponent field of ones.
__device__ __forceinline__ uint32_t not_finite(uint32_t w)
{
    return ((((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u) >> 15) * 0xffffu;
}

// A V fragment with zeros for its infinities and NaN; `any` collects whether it held one.
__device__ __forceinline__ bf16x8_t finite_only(const bf16x8_t& f, uint32_t& any)
{
    const uint4 t = __builtin_bit_cast(uint4, f);
    uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t m = not_finite(w[e]);
        any |= m;
        w[e] &= ~m;
    }
    return __builtin_bit_cast(bf16x8_t, uint4{w[0], w[1], w[2], w[3]});
}

// The same for a masked tile: the matrix cores take zeros for V's infinities and NaN, and where there were any these are
// added one key at a time to the rows that attend them. scratch: 1 KB of LDS of the wave's own, for the probabilities of
// 16 keys at a time ([row][key], as they entered the MFMA).
template <class Seen>
__device__ __forceinline__ void tile_output_masked(WaveRows& w, const TileP& pt, const TileReads& rd, const char* vt,
                                                   const Seen& seen, uint16_t* scratch, uint32_t lane)
{
    uint32_t any = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        w.o[j & 3] =
            __builtin_amdgcn_mfma_f32_32x32x16_bf16(finite_only(rd.v(vt, j), any), pt.chunk(j >> 2), w.o[j & 3], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    }
    if (!__ballot(any != 0u))
        return;
    const uint32_t n = lane & 31u, hh = lane >> 5;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        // Keys 16 c + 8 g + 4 hh + 0 .. 3 of row n: words 2 g and 2 g + 1 of chunk c.
#pragma unroll
        for (int g = 0; g < 2; ++g)
            *reinterpret_cast<uint2*>(scratch + 16u * n + 8 * g + 4u * hh) = uint2{pt.w[4 * c + 2 * g],
                                                                                 pt.w[4 * c + 2 * g + 1]};
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 1
        for (uint32_t jj = 0; jj < 16u; ++jj) {
            const uint32_t j = 16u * c + jj;
            const float pj = __uint_as_float(uint32_t(scratch[16u * n + jj]) << 16);
            const uint32_t in = seen.key(j) ? ~0u : 0u;
            const char* const row = vt + 1024u * (j >> 2) + 64u * (j & 3u) + 8u * hh;
#pragma unroll
            for (int db = 0; db < 4; ++db)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    uint2 t = *reinterpret_cast<const uint2*>(row + 256 * db + 16 * g);
                    t.x &= not_finite(t.x) & in, t.y &= not_finite(t.y) & in; // zeros but for those to be added
                    const float v[4] = {bf16_lo(t.x), bf16_hi(t.x), bf16_lo(t.y), bf16_hi(t.y)};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        w.o[db][4 * g + e] = fmaf(pj, v[e], w.o[db][4 * g + e]);
                    __builtin_amdgcn_sched_barrier(0);
                }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// Whether N KB of a V tile hold an infinity or a NaN.
template <int N>
__device__ __forceinline__ bool holds_nonfinite(const char* part, uint32_t lane)
{
    ushortx2 top{0, 0}; // the largest magnitudes: an exponent of ones is above every other
#pragma unroll
    for (uint32_t i = 0; i < uint32_t(N); ++i) {
        const u32x4_t t = *reinterpret_cast<const u32x4_t*>(part + 1024u * i + 16u * lane);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            top = __builtin_elementwise_max(top, __builtin_bit_cast(ushortx2, t[e] & 0x7fff7fffu));
    }
    return __ballot(top[0] >= 0x7f80u || top[1] >= 0x7f80u) != 0u;
}

// Many rows: eight waves of 32 list rows, in two groups of four, one wave of each group on a SIMD. A group's turn at a
// tile has two phases, the products (S of this tile, and O of the one before) and the softmax, and the groups are a phase
// apart, held there by the barriers: while one group's wave has the matrix core of a SIMD the other's has its vector unit.
// K and V lie in rings of four tiles. The first group loads K and the second V, each wave a quarter: a tile's loads go out
// three turns of K (two of V) ahead of its use and have a turn and a half to arrive, as the group that loads what the other
// reads first is the one that is ahead with K and behind with V. (Each wave an eighth of both: one turn. 256 heads of 256
// rows and 8192 keys each, K and V from HBM: 287 us and 277.)
constexpr uint32_t kPairWaves = 8, kHalf = kPairWaves / 2, kRing = 4;

// tile_output where the tile may have been masked; odd: four waves' words from holds_nonfinite for it (null: it was whole).
template <class Seen>
__device__ __forceinline__ void masked_output(WaveRows& w, const TileP& pt, bf16x8_t (&frag)[kAhead], const TileReads& rd,
                                              const char* vt, const Seen& seen, const uint32_t* odd, uint16_t* scratch,
                                              uint32_t lane)
{
    uint32_t any = 0;
    if (odd) {
        const u32x4_t a = *reinterpret_cast<const u32x4_t*>(odd);
        any = a[0] | a[1] | a[2] | a[3];
    }
    if (__builtin_amdgcn_readfirstlane(any))
        tile_output_masked(w, pt, rd, vt, seen, scratch, lane);
    else
        tile_output(w, pt, frag, rd, vt);
}

// A turn of the eight waves, tile t at key t0, of which a row attends the keys that `seen` says, and of the one before it
// those of `before`. MASKED: this tile or the one before it is not whole for every row of the
// workgroup, or there is none before it; checked: the turn before was of this form too.
template <bool CAP, bool BIAS, bool MASKED, class Feed, class Seen>
__device__ __forceinline__ void pair_turn(const DenseParams& p, WaveRows& w, Feed& feed, const TileReads& rd,
                                          floatx16 (&s)[2], bf16x8_t (&frag)[kAhead], TileP& pt, uint16_t* scratch,
                                          uint32_t* odd, bool checked, uint32_t wave, uint32_t t, uint32_t t0,
                                          const Seen& seen, const Seen& before, uint32_t lane, bool works = true)
{
    // The products.
    __builtin_amdgcn_s_setprio(1);
    constexpr bool kSloped = BIAS && !CAP && !MASKED;
    float* const near_pos = reinterpret_cast<float*>(scratch);
    int32_t pos = 0;
    if (kSloped)
        pos = feed.positions(t)[lane], pos = p.k_pos ? pos : int32_t(t0 + lane);
    bool near = false;
    if (MASKED ? seen.meets(w) : works)
        near = tile_products<!MASKED, kSloped>(w, s, pt, frag, rd, feed.k_tile(t), feed.v_tile(t - 1u), pos, near_pos, lane);
    if (MASKED) {
        if (t > 0 && before.meets(w))
            masked_output(w, pt, frag, rd, feed.v_tile(t - 1u), before,
                          checked ? odd + kHalf * ((t - 1u) % 2u) : nullptr, scratch, lane);
        wait_lds();
    }
    // The first group's K of tile t + 1 has arrived, the second's V of tile t, all but the last turn's loads: the first
    // reader of either is the first group, of K at this turn's end and of V at its next products, past the barrier here.
    wait_vm<Feed::kLoads>();
    if (MASKED && wave >= kHalf) { // the part of V that this wave loaded
        const bool any = holds_nonfinite<4>(feed.v_tile(t) + 4096u * (wave - kHalf), lane);
        if (lane == 0)
            odd[kHalf * (t % 2u) + wave - kHalf] = any;
        wait_lds();
    }
    __builtin_amdgcn_s_setprio(0);
    phase_barrier();
    // The softmax. With it go out the first group's K of tile t + 3, into the slot of tile t - 1, which both groups have
    // read, and the second's V of tile t + 2 into that of tile t - 2 (among the products they cost 10%: this phase is the
    // shorter one).
    feed.next(t);
    if (MASKED ? seen.meets(w) : works)
        tile_softmax<CAP, BIAS, MASKED>(p, w, s, pt, t0, seen, feed.positions(t), near_pos, kSloped, near, lane);
    // Past the last tile these are some tile's again, and not used.
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
        frag[j] = rd.k(feed.k_tile(t + 1u), j);
    phase_barrier();
}

// The turns of a workgroup's tiles, of which walk.whole(t) says whether every row of the workgroup attends all of tile t,
// walk.seen(t) a row's keys of another one (asked for once, in order) and walk.key(t) where it lies; and what is left of
// the last one's output. The feed has loaded K of three tiles, or V of two. works: the wave has rows; one without only
// loads.
template <bool CAP, bool BIAS, class Feed, class Walk>
__device__ __forceinline__ void pair_walk(const DenseParams& p, WaveRows& w, Feed& feed, Walk& walk, const TileReads& rd,
                                          uint16_t* scratch, uint32_t* odd, uint32_t wave, uint32_t tiles, bool works,
                                          uint32_t lane)
{
    wait_vm<2 * Feed::kLoads>(); // K of tile 0
    lds_barrier();
    const bool second = wave >= kHalf;
    if (second)
        phase_barrier();
    floatx16 s[2];
    bf16x8_t frag[kAhead];
    TileP pt;
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
        frag[j] = rd.k(feed.k_tile(0u), j);
    bool masked = true; // the last turn's form
    BitsSeen before(0u, lane);
    // Two loops: one body with both forms copies O between them at every tile.
    for (uint32_t t = 0; t < tiles;) {
#pragma unroll 1
        do {
            const BitsSeen seen = walk.seen(t);
            pair_turn<CAP, BIAS, true>(p, w, feed, rd, s, frag, pt, scratch, odd, masked, wave, t, walk.key(t), seen, before,
                                       lane);
            before = seen;
            masked = true, ++t;
        } while (t < tiles && !(walk.whole(t) && walk.whole(t - 1u)));
        if (t < tiles) {
#pragma unroll 1
            do {
                pair_turn<CAP, BIAS, false>(p, w, feed, rd, s, frag, pt, scratch, odd, true, wave, t, walk.key(t), before,
                                            before, lane, works);
                ++t;
            } while (t < tiles && walk.whole(t));
            masked = false, before = BitsSeen(works ? ~uint64_t(0) : 0u, lane);
        }
    }
    const uint32_t end = tiles - 1u;
    if (!before.meets(w))
        ; // nothing of it is this wave's
    else if (masked)
        masked_output(w, pt, frag, rd, feed.v_tile(end), before, odd + kHalf * (end % 2u), scratch, lane);
    else
        tile_output(w, pt, frag, rd, feed.v_tile(end));
    if (!second)
        phase_barrier();
    wait_vm<0>(); // no load into this workgroup's LDS outlives it
}

// The factors of the scores from `scale` (0: 1 / sqrt(128)) and `cap` (0: none).
inline void score_factors(float scale_given, float cap, DenseParams& p)
{
    const float scale = scale_given > 0.0f ? scale_given : 0.08838834764831845f; // 1 / sqrt(128)
    int pow = 0;
    std::frexp(scale, &pow);
    pow = std::min(std::max(pow, -16), 0);
    p.q_pow = std::ldexp(1.0f, pow);
    p.scale_log2 = scale / p.q_pow * kLog2e;
    // cap_in stays finite, for scores of zero to stay that. It leaves a float's range only where the cap is below 2^-26: no
    // score is then more than that from zero, whatever its product, and the probabilities are equal in float.
    if (cap > 0.0f)
        p.cap_in = std::min(2.0f * kLog2e * (scale / p.q_pow) / cap, std::numeric_limits<float>::max()),
        p.cap_out = cap * kLog2e;
}

} // namespace
} // namespace mh3
