// `flash_attn_128`: flash attention over whole rows, head_dim 128, bf16 in and out: what a block runs without the sparse
// selection, for any count of query and key rows, shared key heads, a range of keys for each query row (documents packed
// into one batch, a prefix, causal rows), a tanh cap on the scores and a bias that falls with the distance.
//   s[i][j] = cap tanh(scale q_i . k_j / cap) - slope |q_pos_i - k_pos_j|   (without a cap: scale q_i . k_j)
//   out_i = sum_j softmax_j(s[i][lo_i .. hi_i)) v_j;   a row without keys is zero.
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
// - Few rows leave the chip idle: their keys are then split over workgroups, each leaves its part of O, the maximum and the
//   sum in the workspace, and a second kernel joins them in a fixed order.
// What bounds it: many rows, the chip's power (960 x 544, 56 heads, 19,305 rows: 8.65 .. 8.9 ms, 1200 .. 1230 TFLOP/s, the
// clock at 1.65 to 1.7 GHz and the matrix cores busy 72% of it); under a cap also the vector unit's transcendentals (five
// clips packed into 14,925 rows of 40 heads 1490 us, without a cap 1230, with a multiplication in the place of the cap's
// exponential and reciprocal 1260); few rows, the one pass over K and V (129,536 keys of 8 heads in 95 us, 5.5 TB/s).
// Under a bias the eight-wave kernels hold five or six registers in scratch, read between the loops, in masked turns and in
// rare paths, never in the loop of whole tiles.
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
    uint32_t all_lo, all_hi;    // keys that every row with any attends: [all_lo, all_hi)
    uint32_t any_lo, any_hi;    // keys that some row attends lie in [any_lo, any_hi)
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

// What one of a score as the products (and cap_scores) leave it is in base 2.
template <bool CAP>
__device__ __forceinline__ float score_unit(const DenseParams& p)
{
    return CAP ? 2.0f * p.cap_out : p.scale_log2;
}

__device__ __forceinline__ bool is_near(int32_t rel) { return rel > -(1 << 23) && rel < (1 << 23); }

template <bool CAP, bool BIAS>
__device__ __forceinline__ void load_rows(const DenseParams& p, uint32_t kvh, uint32_t f0, uint32_t lane, WaveRows& w)
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
    range_of(p, f, row, w.lo, w.hi);
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

// The softmax of a tile at key t0 (MASKED: not every row attends all of it): P^T, and the rows' maxima, sums and (where a
// maximum moved) rescaled O. BIAS: kp and near_pos are LDS for the tile's positions; sloped: tile_products has taken the
// bias off, if the positions are near.
template <bool CAP, bool BIAS, bool MASKED>
__device__ __forceinline__ void tile_softmax(const DenseParams& p, WaveRows& w, floatx16 (&s)[2], TileP& pt, uint32_t t0,
                                             const int32_t* kp, float* near_pos, bool sloped, bool near, uint32_t lane)
{
    const uint32_t hh = lane >> 5;
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
        const uint32_t from_lo = t0 + 4u * hh - w.lo, keys = w.hi - w.lo; // modulo 2^32: below lo is past every count
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                s[b][i] = from_lo + (32u * b + 8u * (i >> 2) + (i & 3)) < keys ? s[b][i] : -kInf;
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
        const uint32_t end = t0 + 64u;
        const bool here = max(w.lo, t0) < min(w.hi, end);
        const bool begins = __ballot(here && (BIAS ? w.hi <= end : w.lo >= t0)) != 0; // with its last key under a bias
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
__device__ __forceinline__ void tile_output_masked(WaveRows& w, const TileP& pt, const TileReads& rd, const char* vt,
                                                   uint32_t t0, uint16_t* scratch, uint32_t lane)
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
            const uint32_t in = t0 + j >= w.lo && t0 + j < w.hi ? ~0u : 0u;
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

// The key tiles [first, last) of a workgroup whose rows' keys lie in [k0, k1), for its split.
__device__ __forceinline__ void tiles_of(const DenseParams& p, uint32_t k0, uint32_t k1, uint32_t split, uint32_t& first,
                                         uint32_t& last)
{
    const uint32_t tiles = k0 < k1 ? (k1 - k0 + 63u) / 64u : 0u;
    first = uint32_t(uint64_t(tiles) * split / p.splits);
    last = uint32_t(uint64_t(tiles) * (split + 1u) / p.splits);
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
template <bool CAP, bool BIAS, bool MASKED>
__device__ __forceinline__ void few_turn(const DenseParams& p, WaveRows& w, const FewLoads<BIAS>& feed,
                                         const TileReads& rd, uint32_t t, uint32_t t0, bool more, uint32_t next,
                                         uint32_t lane)
{
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
    tile_softmax<CAP, BIAS, MASKED>(p, w, s, pt, t0, feed.positions(t), reinterpret_cast<float*>(scratch), false, false,
                                    lane);
    if (more)
        wait_vm<BIAS ? 17 : 16>(); // V, but not the next K
    else
        wait_vm<0>();
    if (MASKED && holds_nonfinite<16>(vt, lane))
        tile_output_masked(w, pt, rd, vt, t0, scratch, lane);
    else
        tile_output(w, pt, frag, rd, vt);
    wait_lds();
    if (more)
        feed.v(p, next);
}

// Few rows: one wave of 32 list rows a workgroup, with a tile of its own in LDS; four or five of them share a CU, and
// one's loads arrive while the others compute.
template <bool CAP, bool BIAS>
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
    load_rows<CAP, BIAS>(p, kvh, tile * 32u, lane, w);
    uint32_t first, last;
    tiles_of(p, w.any_lo, w.any_hi, split, first, last);
    const FewLoads<BIAS> feed{{p.krs, 0u, lane},
                              {p.vrs, 0u, lane},
                              p.k + uint64_t(kvh) * p.khs,
                              p.v + uint64_t(kvh) * p.vhs,
                              lds};
    const TileReads rd(lane);
    const uint32_t tiles = last - first;
    const auto key_of = [&](uint32_t t) { return w.any_lo + 64u * (BIAS ? last - 1u - t : first + t); };
    if (tiles) {
        feed.k(p, 0u, key_of(0u), lane);
        feed.v(p, key_of(0u));
    }
    // Two loops, the masked tiles' and the whole ones': one body with both forms copies O between them at every tile.
    for (uint32_t t = 0; t < tiles;) {
#pragma unroll 1
        for (; t < tiles && w.masks(key_of(t)); ++t)
            few_turn<CAP, BIAS, true>(p, w, feed, rd, t, key_of(t), t + 1u < tiles, key_of(t + 1u), lane);
#pragma unroll 1
        for (; t < tiles && !w.masks(key_of(t)); ++t)
            few_turn<CAP, BIAS, false>(p, w, feed, rd, t, key_of(t), t + 1u < tiles, key_of(t + 1u), lane);
    }
    store_rows(p, w, kvh, tile * 32u, split, lane);
}

// Many rows: eight waves of 32 list rows, in two groups of four, one wave of each group on a SIMD. A group's turn at a
// tile has two phases, the products (S of this tile, and O of the one before) and the softmax, and the groups are a phase
// apart, held there by the barriers: while one group's wave has the matrix core of a SIMD the other's has its vector unit.
// K and V lie in rings of four tiles; a tile's loads go out three of its K (two of its V) ahead of its use, each wave an
// eighth.
constexpr uint32_t kPairWaves = 8, kRing = 4;

// What a wave loads of a workgroup's tiles, a call a tile: its eighth of K (with all of the tile's key positions, into the
// wave's own ring) or of V. After the workgroup's last tile the same again, so that every turn has the same count of loads;
// these are not read. The state is scalar and moves by additions.
template <bool VALUE, bool POS>
struct PairStream {
    TileLoads<2, VALUE> ld;
    const uint16_t* at;       // the next tile's first key
    int64_t step;             // elements to the one after it
    uint32_t left, left_step; // keys from it on
    uint32_t more;            // tiles after it
    char* ring;
    uint32_t slot; // byte offset in the ring
    const int32_t* pos;
    char* pos_ring;
    uint32_t lane;
    __device__ __forceinline__ void operator()()
    {
        ld(ring + slot, at, left);
        if (POS) // no positions: no records, and zeros
            load_lds4(buffer_words(pos, pos ? left * 4u : 0u), pos_ring + slot / 64u, 4u * lane);
        slot = (slot + kTileBytes) & (kRing * kTileBytes - 1u);
        at += more ? step : 0;
        left += more ? left_step : 0u;
        if (POS)
            pos -= more && pos ? int32_t(left_step) : 0;
        more -= more ? 1u : 0u;
    }
};

template <bool BIAS>
struct PairFeed {
    static constexpr int kLoads = BIAS ? 5 : 4; // of a turn
    PairStream<false, BIAS> k;
    PairStream<true, false> v;
    __device__ __forceinline__ const char* k_tile(uint32_t t) const { return k.ring + (t % kRing) * kTileBytes; }
    __device__ __forceinline__ const char* v_tile(uint32_t t) const { return v.ring + (t % kRing) * kTileBytes; }
    __device__ __forceinline__ int32_t* positions(uint32_t t) const
    {
        return reinterpret_cast<int32_t*>(k.pos_ring + (t % kRing) * 256u);
    }
};

// tile_output where the tile may have been masked; odd: the eight waves' words from holds_nonfinite for it (null: it was
// whole).
__device__ __forceinline__ void masked_output(WaveRows& w, const TileP& pt, bf16x8_t (&frag)[kAhead], const TileReads& rd,
                                              const char* vt, uint32_t t0, const uint32_t* odd, uint16_t* scratch,
                                              uint32_t lane)
{
    uint32_t any = 0;
    if (odd) {
        const u32x4_t a = *reinterpret_cast<const u32x4_t*>(odd), b = *reinterpret_cast<const u32x4_t*>(odd + 4);
        any = a[0] | a[1] | a[2] | a[3] | b[0] | b[1] | b[2] | b[3];
    }
    if (__builtin_amdgcn_readfirstlane(any))
        tile_output_masked(w, pt, rd, vt, t0, scratch, lane);
    else
        tile_output(w, pt, frag, rd, vt);
}

// A turn of attn_pair_kernel, tile t at key t0. MASKED: this tile or the one before it is not whole for every row of the
// workgroup, or there is none before it; checked: the turn before was of this form too.
template <bool CAP, bool BIAS, bool MASKED>
__device__ __forceinline__ void pair_turn(const DenseParams& p, WaveRows& w, PairFeed<BIAS>& feed, const TileReads& rd,
                                          floatx16 (&s)[2], bf16x8_t (&frag)[kAhead], TileP& pt, uint16_t* scratch,
                                          uint32_t* odd, bool checked, uint32_t wave, uint32_t t, uint32_t t0,
                                          uint32_t lane)
{
    // The products.
    __builtin_amdgcn_s_setprio(1);
    constexpr bool kSloped = BIAS && !CAP && !MASKED;
    float* const near_pos = reinterpret_cast<float*>(scratch);
    int32_t pos = 0;
    if (kSloped)
        pos = feed.positions(t)[lane], pos = p.k_pos ? pos : int32_t(t0 + lane);
    bool near = false;
    if (!MASKED || w.meets(t0))
        near = tile_products<!MASKED, kSloped>(w, s, pt, frag, rd, feed.k_tile(t), feed.v_tile(t - 1u), pos, near_pos, lane);
    if (MASKED) {
        if (t > 0 && w.meets(BIAS ? t0 + 64u : t0 - 64u))
            masked_output(w, pt, frag, rd, feed.v_tile(t - 1u), BIAS ? t0 + 64u : t0 - 64u,
                          checked ? odd + kPairWaves * ((t - 1u) % 2u) : nullptr, scratch, lane);
        // The part of V that this wave loaded: every wave's word is read at the next products, a barrier on.
        const bool any = holds_nonfinite<2>(feed.v_tile(t) + 2048u * wave, lane);
        if (lane == 0)
            odd[kPairWaves * (t % 2u) + wave] = any;
        wait_lds();
    }
    __builtin_amdgcn_s_setprio(0);
    phase_barrier();
    // The softmax. With it go out K of tile t + 3, into the slot of tile t - 1, which both groups have read, and V of tile
    // t + 2 into that of tile t - 2 (among the products they cost 10%: this phase is the shorter one).
    feed.k();
    feed.v();
    if (!MASKED || w.meets(t0))
        tile_softmax<CAP, BIAS, MASKED>(p, w, s, pt, t0, feed.positions(t), near_pos, kSloped, near, lane);
    // Past the last tile these are some tile's again, and not used.
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
        frag[j] = rd.k(feed.k_tile(t + 1u), j);
    // K of tile t + 2 and V of tile t + 1 have arrived, all but this turn's loads: both groups are past their barriers by
    // the time that either reads them.
    wait_vm<PairFeed<BIAS>::kLoads>();
    phase_barrier();
}

template <bool CAP, bool BIAS>
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
    uint16_t* const scratch = reinterpret_cast<uint16_t*>(lds + 2u * kRing * kTileBytes + 2048u * wave);
    uint32_t* const span = reinterpret_cast<uint32_t*>(lds + 2u * kRing * kTileBytes + 2048u * kPairWaves);
    const uint32_t f0 = (tile * kPairWaves + wave) * 32u;
    WaveRows w;
    load_rows<CAP, BIAS>(p, kvh, f0, lane, w);
    if (lane == 0)
        *reinterpret_cast<uint4*>(span + 4u * wave) = uint4{w.any_lo, w.any_hi, w.all_lo, w.all_hi};
    lds_barrier();
    uint32_t* const odd = span + 4u * kPairWaves; // [2][kPairWaves]: a masked tile's V holds an infinity or a NaN
    uint32_t k0 = ~0u, k1 = 0u, all_lo = 0u, all_hi = ~0u; // of the workgroup's rows
#pragma unroll
    for (uint32_t i = 0; i < kPairWaves; ++i) {
        const uint4 t = *reinterpret_cast<const uint4*>(span + 4u * i);
        k0 = min(k0, t.x), k1 = max(k1, t.y), all_lo = max(all_lo, t.z), all_hi = min(all_hi, t.w);
    }
    k0 = __builtin_amdgcn_readfirstlane(k0), k1 = __builtin_amdgcn_readfirstlane(k1);
    all_lo = __builtin_amdgcn_readfirstlane(all_lo), all_hi = __builtin_amdgcn_readfirstlane(all_hi);
    uint32_t first, last;
    tiles_of(p, k0, k1, split, first, last);
    if (first >= last) { // the same for every wave
        store_rows(p, w, kvh, f0, split, lane);
        return;
    }
    k0 += 64u * first;
    const uint32_t tiles = last - first;
    // Turn t's tile.
    const auto key_of = [&](uint32_t t) { return k0 + 64u * (BIAS ? tiles - 1u - t : t); };
    const TileReads rd(lane);
    const uint32_t from = key_of(0), left_step = BIAS ? 64u : -64u;
    const auto stride = [](uint64_t row) { return (BIAS ? -64 : 64) * int64_t(row); };
    PairFeed<BIAS> feed{{{p.krs, 2u * wave, lane},
                         p.k + uint64_t(kvh) * p.khs + uint64_t(from) * p.krs,
                         stride(p.krs),
                         p.kv_rows - from,
                         left_step,
                         tiles - 1u,
                         lds,
                         0u,
                         p.k_pos ? p.k_pos + from : nullptr,
                         reinterpret_cast<char*>(scratch) + 1024,
                         lane},
                        {{p.vrs, 2u * wave, lane},
                         p.v + uint64_t(kvh) * p.vhs + uint64_t(from) * p.vrs,
                         stride(p.vrs),
                         p.kv_rows - from,
                         left_step,
                         tiles - 1u,
                         lds + kRing * kTileBytes,
                         0u,
                         nullptr,
                         nullptr,
                         lane}};
    feed.k();
    feed.k();
    feed.v();
    feed.k();
    feed.v();
    wait_vm<PairFeed<BIAS>::kLoads>(); // K of tiles 0 and 1, V of tile 0
    lds_barrier();
    const bool second = wave >= kPairWaves / 2u;
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
#pragma unroll 1
    for (uint32_t t = 0; t < a; ++t)
        pair_turn<CAP, BIAS, true>(p, w, feed, rd, s, frag, pt, scratch, odd, true, wave, t, key_of(t), lane);
#pragma unroll 1
    for (uint32_t t = a; t < b; ++t)
        pair_turn<CAP, BIAS, false>(p, w, feed, rd, s, frag, pt, scratch, odd, true, wave, t, key_of(t), lane);
#pragma unroll 1
    for (uint32_t t = b; t < tiles; ++t)
        pair_turn<CAP, BIAS, true>(p, w, feed, rd, s, frag, pt, scratch, odd, t > b || a == b, wave, t, key_of(t),
                                    lane);
    const uint32_t end = tiles - 1u;
    if (!w.meets(key_of(end)))
        ; // nothing of it is this wave's
    else if (b < tiles || a == tiles) // the last turn was of the masked form
        masked_output(w, pt, frag, rd, feed.v_tile(end), key_of(end), odd + kPairWaves * (end % 2u), scratch, lane);
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

__global__ __launch_bounds__(256) void attn_ranges_kernel(RangeParams p)
{
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= p.q_rows)
        return;
    // The last document whose first row is at most i (of empty ones that start together the last).
    uint32_t a = 0, b = p.docs; // q_off[a - 1] <= i < q_off[b] in a sorted list
    while (a < b) {
        const uint32_t mid = (a + b) / 2u;
        if (p.q_off[mid + 1u] <= int32_t(i))
            a = mid + 1u;
        else
            b = mid;
    }
    int2 r{0, 0};
    if (a < p.docs && p.q_off[a] <= int32_t(i)) {
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

template <bool CAP, bool BIAS>
int launch_dense(const DenseParams& p, uint32_t waves, hipStream_t stream)
{
    if (waves == kPairWaves)
        return launch_rows(attn_pair_kernel<CAP, BIAS>, 2u * kRing * kTileBytes + (2048u + 16u + 8u) * kPairWaves, p, waves,
                           stream);
    return launch_rows(attn_few_kernel<CAP, BIAS>, 2u * kTileBytes + 1024u + 512u, p, waves, stream);
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
                                  void* workspace, uint64_t workspace_bytes_given, uint16_t* out, mh3_stream_t stream)
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
    if (!q_pos != !k_pos || (q_pos && !slopes))
        return MH3_ERR_POINTER;
    if (workspace_bytes_given < need)
        return MH3_ERR_SHAPE;
    if (!host::aligned16(q) || !host::aligned16(k) || !host::aligned16(v) || !host::aligned16(out) ||
        !host::aligned16(workspace) || reinterpret_cast<uintptr_t>(ranges) % 8u != 0u ||
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
    p.q = q, p.k = k, p.v = v, p.out = out, p.ranges = ranges, p.slopes = slopes, p.q_pos = q_pos, p.k_pos = k_pos;
    p.part = need ? reinterpret_cast<float*>(static_cast<char*>(workspace) + kHeader) : nullptr;
    p.qhs = a.q_head_stride, p.qrs = a.q_row_stride, p.khs = a.k_head_stride, p.krs = a.k_row_stride;
    p.vhs = a.v_head_stride, p.vrs = a.v_row_stride, p.ohs = a.out_head_stride, p.ors = a.out_row_stride;
    p.kv_heads = a.kv_heads, p.group = a.heads / a.kv_heads, p.q_rows = a.q_rows, p.kv_rows = a.kv_rows;
    p.list = uint32_t(plans.list);
    p.div_group = FastDiv::make(p.group);
    const float scale = a.scale > 0.0f ? a.scale : 0.08838834764831845f; // 1 / sqrt(128)
    int pow = 0;
    std::frexp(scale, &pow);
    pow = std::min(std::max(pow, -16), 0);
    p.q_pow = std::ldexp(1.0f, pow);
    p.scale_log2 = scale / p.q_pow * kLog2e;
    // cap_in stays finite, for scores of zero to stay that. It leaves a float's range only where the cap is below 2^-26: no
    // score is then more than that from zero, whatever its product, and the probabilities are equal in float.
    if (a.cap > 0.0f)
        p.cap_in = std::min(2.0f * kLog2e * (scale / p.q_pow) / a.cap, std::numeric_limits<float>::max()),
        p.cap_out = a.cap * kLog2e;
    const bool contest = plans.contest && ranges;
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
