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
// - A workgroup walks the key tiles from its rows' lowest lo to their highest hi. A wave masks a tile only where its own
//   rows' ranges do not all cover it.
// - A masked probability is a zero, and zero times an infinite or NaN value of V would still be NaN in the rows that do
//   not attend it: in a masked tile the wave looks for such values, and where there are any the matrix cores take zeros
//   for them, and they are added one key at a time to the rows that attend it.
// - Softmax in base 2. A row's running maximum moves only when a tile raises it by more than 8, so P stays below 2^8 and
//   most tiles skip the rescale of O. P rounds to bf16 for the matrix cores (2^-9 of each probability, below the output's
//   own rounding); maxima, sums and O are float.
// - Few rows leave the chip idle: their keys are then split over workgroups, each leaves its part of O, the maximum and the
//   sum in the workspace, and a second kernel joins them in a fixed order.
#include "mh3_common.hpp"

#include <algorithm>
#include <cmath>

namespace mh3 {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* lds_ptr_t;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInf = __builtin_inff();
constexpr uint32_t kPastEnd = 0x80000000u; // a buffer offset past num_records: the load reads zeros
constexpr uint32_t kRecords = 0x7fffffffu;
constexpr uint32_t kTileBytes = 16384; // 64 keys of K, or of V

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

// The sources of a wave's DMA instructions. Instruction i of a tile's 16 fills the LDS kilobyte 1024 i with keys
// 4 i .. 4 i + 3: of K 256-byte rows whose 16-byte chunks are XOR-swizzled by the row, of V the four keys' 64-byte
// pieces interleaved (so that operand and transposed reads hit distinct banks); each quad of lanes fetches one aligned
// 64-byte piece of a row.
struct TileLoads {
    uint32_t k_row, v_key, k_off[4], v_off;
    __device__ __forceinline__ TileLoads(const DenseParams& p, uint32_t lane)
    {
        k_row = lane >> 4, v_key = (lane >> 2) & 3u;
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u)
            k_off[u] = k_row * uint32_t(p.krs) * 2u + 16u * ((lane & 15u) ^ (4u * u + k_row));
        v_off = v_key * uint32_t(p.vrs) * 2u + 16u * (4u * (lane >> 4) + (lane & 3u));
    }
    // Instructions i0 .. i0 + N - 1 of the K or V tile at key t0, `live` of whose 64 keys exist.
    template <int N>
    __device__ __forceinline__ void k_tile(const DenseParams& p, const uint16_t* kh, char* dst, uint32_t t0, uint32_t i0,
                                           uint32_t live) const
    {
        const __amdgpu_buffer_rsrc_t r = buffer_rsrc(kh + uint64_t(t0) * p.krs, kRecords);
#pragma unroll
        for (uint32_t u = 0; u < uint32_t(N); ++u) {
            const uint32_t i = i0 + u;
            const int so = int(4u * i * uint32_t(p.krs) * 2u);
            const uint32_t off = N % 4 == 0 ? k_off[u & 3u] : (i & 1u) ? ((i & 2u) ? k_off[3] : k_off[1])
                                                                       : ((i & 2u) ? k_off[2] : k_off[0]);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr_t)(dst + 1024u * i), 16,
                                                     live >= 64u || 4u * i + k_row < live ? off : kPastEnd, so, 0, 0);
        }
    }
    template <int N>
    __device__ __forceinline__ void v_tile(const DenseParams& p, const uint16_t* vh, char* dst, uint32_t t0, uint32_t i0,
                                           uint32_t live) const
    {
        const __amdgpu_buffer_rsrc_t r = buffer_rsrc(vh + uint64_t(t0) * p.vrs, kRecords);
#pragma unroll
        for (uint32_t u = 0; u < uint32_t(N); ++u) {
            const uint32_t i = i0 + u;
            const int so = int(4u * i * uint32_t(p.vrs) * 2u);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr_t)(dst + 1024u * i), 16,
                                                     live >= 64u || 4u * i + v_key < live ? v_off : kPastEnd, so, 0, 0);
        }
    }
};

// A wave's 32 rows: their query fragments, and the state of their softmax and output.
struct WaveRows {
    bf16x8_t qf[8];  // B operand of S^T: lane (n, hh) holds d 16 dc + 8 hh .. + 7 of row n
    floatx16 o[4];   // O^T: d 32 db + 8 (i / 4) + 4 hh + i % 4 of row n
    float m_run, l_run;
    uint32_t lo, hi;            // the lane's row's keys
    uint32_t all_lo, all_hi;    // keys that every row with any attends: [all_lo, all_hi)
    uint32_t any_lo, any_hi;    // keys that some row attends lie in [any_lo, any_hi)
    float slope_log2;           // BIAS: the row's head's slope, in base-2 units
    int32_t q_pos;
};

template <bool BIAS>
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
    w.m_run = -kInf, w.l_run = 0.0f;
    range_of(p, f, row, w.lo, w.hi);
    const bool any = w.lo < w.hi;
    w.any_lo = wave_min_u32(any ? w.lo : ~0u);
    w.any_hi = wave_max_u32(any ? w.hi : 0u);
    w.all_lo = wave_max_u32(w.lo); // a row of the list without keys masks every tile, one past it none
    w.all_hi = wave_min_u32(f < p.list ? w.hi : ~0u);
    if (BIAS) {
        w.slope_log2 = p.slopes[head] * kLog2e;
        w.q_pos = p.q_pos ? p.q_pos[row] : int32_t(row);
    }
}

// Whether the V tile in LDS holds an infinity or a NaN (wave-uniform).
__device__ __forceinline__ bool tile_not_finite(const char* vt, uint32_t lane)
{
    uint32_t any = 0;
#pragma unroll 4
    for (uint32_t i = 0; i < kTileBytes / 1024u; ++i) {
        const uint4 t = *reinterpret_cast<const uint4*>(vt + 1024u * i + 16u * lane);
        const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) // the exponent field of either half all ones: the sum carries into its sign bit
            any |= ((w[e] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
    }
    return __ballot(any != 0u) != 0;
}

// Scores of a tile at key t0 to base-2 units where a cap or a bias needs every one changed; kp: the tile's key positions
// (LDS, or null: the keys' numbers).
template <bool CAP, bool BIAS>
__device__ __forceinline__ void shape_scores(const DenseParams& p, const WaveRows& w, floatx16 (&s)[2], uint32_t t0,
                                             uint32_t hh, const int32_t* kp)
{
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const uint32_t key = 32u * b + 8u * g + 4u * hh;
            int32_t pos[4];
            if (BIAS) {
                if (kp) {
                    const int4 t = *reinterpret_cast<const int4*>(kp + key);
                    pos[0] = t.x, pos[1] = t.y, pos[2] = t.z, pos[3] = t.w;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        pos[e] = int32_t(t0 + key) + e;
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x = s[b][4 * g + e];
                // tanh(u) = 1 - 2 / (exp(2 u) + 1): at either end the exponential gives +-1, and its error near zero is
                // 2^-23 of the cap, below what bf16 operands leave of the score.
                if (CAP)
                    x = fmaf(-2.0f * p.cap_out,
                             __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * p.cap_in) + 1.0f), p.cap_out);
                else
                    x *= p.scale_log2;
                // The distance of two int32 positions fits 32 bits without a sign.
                if (BIAS) {
                    const uint32_t d = w.q_pos > pos[e] ? uint32_t(w.q_pos) - uint32_t(pos[e])
                                                        : uint32_t(pos[e]) - uint32_t(w.q_pos);
                    x = fmaf(-w.slope_log2, float(d), x);
                }
                s[b][4 * g + e] = x;
            }
        }
}

// The non-finite values of a masked tile's V (the matrix cores took zeros for them), one key at a time into the rows that
// attend it. pl: the wave's probabilities as they entered the MFMA, [row][key] bf16.
__device__ __forceinline__ void add_not_finite(WaveRows& w, const char* vt, const uint16_t* pl, uint32_t t0, uint32_t lane)
{
    const uint32_t n = lane & 31u, hh = lane >> 5;
#pragma unroll 1
    for (uint32_t j = 0; j < 64u; ++j) {
        const float pj = __uint_as_float(uint32_t(pl[n * 64u + j]) << 16);
        const bool in = t0 + j >= w.lo && t0 + j < w.hi;
        const char* const row = vt + 1024u * (j >> 2) + 64u * (j & 3u) + 8u * hh;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const uint2 t = *reinterpret_cast<const uint2*>(row + 256 * db + 16 * g);
                const float v[4] = {bf16_lo(t.x), bf16_hi(t.x), bf16_lo(t.y), bf16_hi(t.y)};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool add = in && (__float_as_uint(v[e]) & 0x7f800000u) == 0x7f800000u;
                    w.o[db][4 * g + e] = add ? fmaf(pj, v[e], w.o[db][4 * g + e]) : w.o[db][4 * g + e];
                }
            }
    }
}

// A V fragment with zeros for its infinities and NaN.
__device__ __forceinline__ bf16x8_t finite_only(const bf16x8_t& f)
{
    uint4 t = __builtin_bit_cast(uint4, f);
    uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        w[e] = (w[e] & 0x7f80u) == 0x7f80u ? w[e] & 0xffff0000u : w[e];
        w[e] = (w[e] & 0x7f800000u) == 0x7f800000u ? w[e] & 0xffffu : w[e];
    }
    return __builtin_bit_cast(bf16x8_t, uint4{w[0], w[1], w[2], w[3]});
}

// s unit - m in two roundings.
__device__ __forceinline__ float rounded_difference(float s, float unit, float m)
{
#pragma clang fp contract(off)
    const float x = s * unit;
    return x - m;
}

// One tile of 64 keys at t0 for a wave: scores, softmax and its part of O. kt, vt: the tile in LDS; scratch: 4 KB of LDS
// of the wave's own.
template <bool CAP, bool BIAS>
__device__ __forceinline__ void attend_tile(const DenseParams& p, WaveRows& w, const char* kt, const char* vt, uint32_t t0,
                                            const int32_t* kp, uint16_t* scratch, uint32_t lane)
{
    constexpr int kAhead = 8;
    const uint32_t n = lane & 31u, hh = lane >> 5, L = lane & 15u, grp = lane >> 4;
    const uint32_t k_lane = 256u * n + 16u * (hh ^ (n & 15u));
    const char* const vs = vt + 1024u * (grp >> 1) + 32u * (grp & 1u) + 64u * (L >> 2) + 8u * (L & 3u);
    auto read_k = [&](int j) { // key block j % 2, d chunk j / 2
        return *reinterpret_cast<const bf16x8_t*>(kt + 8192u * (j & 1) + (k_lane ^ (32u * (j >> 1))));
    };
    auto read_v = [&](int j) { // 16-key chunk j / 4, d block j % 4
        const uint32_t off = 4096u * (j >> 2) + 256u * (j & 3);
        const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (v4i16 __attribute__((address_space(3)))*)(const_cast<char*>(vs) + off));
        const v4i16 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (v4i16 __attribute__((address_space(3)))*)(const_cast<char*>(vs) + off + 2048u));
        return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    floatx16 s[2];
    bf16x8_t frag[kAhead];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            s[b][i] = 0.0f;
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
        frag[j] = read_k(j);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        __builtin_amdgcn_sched_barrier(0);
        s[j & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag[j % kAhead], w.qf[j >> 1], s[j & 1], 0, 0, 0);
        if (j + kAhead < 16)
            frag[j % kAhead] = read_k(j + kAhead);
    }
    __builtin_amdgcn_sched_barrier(0);
    constexpr bool kShaped = CAP || BIAS;
    if (kShaped)
        shape_scores<CAP, BIAS>(p, w, s, t0, hh, kp);
    const float unit = kShaped ? 1.0f : p.scale_log2;
    const bool masked = t0 < w.all_lo || t0 + 64u > w.all_hi;
    if (masked) {
        asm volatile("" ::: "memory"); // kept a branch
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const uint32_t key = t0 + 32u * b + 8u * (i >> 2) + 4u * hh + (i & 3);
                s[b][i] = key >= w.lo && key < w.hi ? s[b][i] : -kInf;
            }
    }
    float mt = -kInf;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            mt = fmaxf(mt, s[b][i]);
    mt = fmaxf(mt, __shfl_xor(mt, 32, kWave)) * unit;
    if (__ballot(mt > w.m_run + 8.0f)) {
        const float m_new = fmaxf(w.m_run, mt);
        const float alpha = w.m_run == -kInf ? 0.0f : __builtin_amdgcn_exp2f(w.m_run - m_new);
        w.m_run = m_new;
        w.l_run *= alpha;
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                w.o[b][i] *= alpha;
    }
    float m_ref = w.m_run == -kInf ? 0.0f : w.m_run, factor = unit;
    // s unit - m in one fused operation keeps the rounding of m, 2^-24 of it, in the exponent: common to all of a row's
    // probabilities and harmless, until it leaves the exponent's range. Scores so large are rounded as m was first.
    if (__ballot(fabsf(m_ref) > 0x1p20f)) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                s[b][i] = rounded_difference(s[b][i], unit, m_ref);
        m_ref = 0.0f, factor = 1.0f;
    }
    uint32_t pw[4][4]; // P^T chunk c: elements 8 (c % 2) .. + 7 of block c / 2
    float ps = 0.0f;
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int b = c >> 1, i = 8 * (c & 1) + 2 * e;
            const float p0 = __builtin_amdgcn_exp2f(fmaf(s[b][i], factor, -m_ref));
            const float p1 = __builtin_amdgcn_exp2f(fmaf(s[b][i + 1], factor, -m_ref));
            ps += p0 + p1;
            pw[c][e] = pack_bf16(p0, p1);
        }
    w.l_run += ps;
    if (masked && tile_not_finite(vt, lane)) {
        // Keys 32 b + 8 g + 4 hh + 0 .. 3 of row n: words 2 (g % 2) and + 1 of chunk 2 b + g / 2.
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int g = 0; g < 2; ++g)
                *reinterpret_cast<uint2*>(scratch + n * 64u + 32 * (c >> 1) + 8 * (2 * (c & 1) + g) + 4u * hh) =
                    uint2{pw[c][2 * g], pw[c][2 * g + 1]};
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int c = j >> 2;
            const bf16x8_t pf = __builtin_bit_cast(bf16x8_t, uint4{pw[c][0], pw[c][1], pw[c][2], pw[c][3]});
            w.o[j & 3] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(finite_only(read_v(j)), pf, w.o[j & 3], 0, 0, 0);
        }
        add_not_finite(w, vt, scratch, t0, lane);
        return;
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
        frag[j] = read_v(j);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const bf16x8_t pf = __builtin_bit_cast(bf16x8_t, uint4{pw[c][0], pw[c][1], pw[c][2], pw[c][3]});
#pragma unroll
        for (int db = 0; db < 4; ++db) {
            const int j = 4 * c + db;
            __builtin_amdgcn_sched_barrier(0);
            w.o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag[j % kAhead], pf, w.o[db], 0, 0, 0);
            if (j + kAhead < 16)
                frag[j % kAhead] = read_v(j + kAhead);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
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

// W waves of 32 list rows each.
template <int W, bool CAP, bool BIAS>
__global__ __launch_bounds__(W * 64) __attribute__((amdgpu_waves_per_eu(2))) void attn_dense_kernel(DenseParams p)
{
    extern __shared__ __attribute__((aligned(16))) char lds[]; // K, V, key positions, the waves' scratch, 2 W words
    uint32_t kvh, tile, split;
    if (!block_of(p, kvh, tile, split))
        return;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int32_t* const kp = reinterpret_cast<int32_t*>(lds + 2u * kTileBytes);
    uint16_t* const scratch = reinterpret_cast<uint16_t*>(lds + 2u * kTileBytes + 256u + 4096u * wave);
    uint32_t* const span = reinterpret_cast<uint32_t*>(lds + 2u * kTileBytes + 256u + 4096u * W);
    const uint32_t f0 = (tile * W + wave) * 32u;
    WaveRows w;
    load_rows<BIAS>(p, kvh, f0, lane, w);
    uint32_t k0 = w.any_lo, k1 = w.any_hi;
    if (W > 1) {
        if (lane == 0)
            span[2u * wave] = k0, span[2u * wave + 1u] = k1;
        lds_barrier();
#pragma unroll
        for (int i = 0; i < W; ++i)
            k0 = min(k0, span[2 * i]), k1 = max(k1, span[2 * i + 1]);
        k0 = __builtin_amdgcn_readfirstlane(k0), k1 = __builtin_amdgcn_readfirstlane(k1);
    }
    const uint32_t tiles = k0 < k1 ? (k1 - k0 + 63u) / 64u : 0u;
    const uint32_t t_first = uint32_t(uint64_t(tiles) * split / p.splits);
    const uint32_t t_last = uint32_t(uint64_t(tiles) * (split + 1u) / p.splits);
    const uint16_t* const kh = p.k + uint64_t(kvh) * p.khs;
    const uint16_t* const vh = p.v + uint64_t(kvh) * p.vhs;
    const TileLoads ld(p, lane);
    for (uint32_t t = t_first; t < t_last; ++t) {
        const uint32_t t0 = k0 + 64u * t, live = min(64u, p.kv_rows - t0);
        ld.k_tile<16 / W>(p, kh, lds, t0, wave * (16u / W), live);
        ld.v_tile<16 / W>(p, vh, lds + kTileBytes, t0, wave * (16u / W), live);
        if (BIAS && p.k_pos && tid < 64u)
            kp[tid] = p.k_pos[min(t0 + tid, p.kv_rows - 1u)];
        wait_vm<0>();
        lds_barrier(); // the tile is in LDS for every wave
        if (t0 < w.any_hi && t0 + 64u > w.any_lo)
            attend_tile<CAP, BIAS>(p, w, lds, lds + kTileBytes, t0, p.k_pos ? kp : nullptr, scratch, lane);
        lds_barrier(); // every wave is done with it before it is overwritten
    }
    store_rows(p, w, kvh, f0, split, lane);
}

// Joins the splits of a list row: a wave a row, two values of d a lane.
__global__ __launch_bounds__(256) void attn_join_kernel(DenseParams p)
{
    const uint32_t lane = threadIdx.x & 63u;
    const uint64_t item = uint64_t(blockIdx.x) * 4u + (threadIdx.x >> 6), items = uint64_t(p.kv_heads) * p.list;
    if (item >= items)
        return;
    const uint32_t kvh = uint32_t(item / p.list), f = uint32_t(item - uint64_t(kvh) * p.list);
    const uint32_t row = p.div_group.div(f), head = kvh * p.group + (f - row * p.group);
    uint32_t lo, hi;
    range_of(p, f, row, lo, hi);
    const float2* const ml = reinterpret_cast<const float2*>(p.part + uint64_t(p.splits) * items * 128u);
    float m = -kInf;
    for (uint32_t s = 0; s < p.splits; ++s)
        m = fmaxf(m, ml[s * items + item].x);
    const float m_ref = m == -kInf ? 0.0f : m;
    float l = 0.0f, a = 0.0f, b = 0.0f;
    for (uint32_t s = 0; s < p.splits; ++s) {
        const float2 t = ml[s * items + item];
        const float2 o = *reinterpret_cast<const float2*>(p.part + (s * items + item) * 128u + 2u * lane);
        // A split without a key of this row has left zeros and -inf. (A NaN of its scores is in its sum and its O.)
        const float f = t.x == -kInf ? 1.0f : __builtin_amdgcn_exp2f(t.x - m_ref);
        l = fmaf(t.y, f, l), a = fmaf(o.x, f, a), b = fmaf(o.y, f, b);
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
        const int32_t n = int32_t(p.kv_rows);
        const int32_t lo = min(max(p.k_off[a], 0), n), end = min(max(p.k_off[a + 1u], lo), n);
        int32_t hi = end;
        if (p.causal) {
            const int64_t own = int64_t(end) - p.q_off[a + 1u] + i; // the last query row sits on the last key row
            const int64_t seen = int64_t(lo) + (p.prefix ? max(p.prefix[a], 0) : 0);
            hi = int32_t(max(int64_t(lo), min(int64_t(end), max(own + 1, seen))));
        }
        r = int2{lo, hi};
    }
    p.ranges[i] = r;
}

} // namespace
} // namespace mh3

namespace {

using namespace mh3;

struct Plan {
    uint32_t waves, splits;
    uint64_t list, tiles;
};

// The workgroup's waves and the key splits of a call.
Plan plan_of(const MH3DenseAttnArgs& a)
{
    Plan p{};
    p.list = uint64_t(a.q_rows) * (a.heads / a.kv_heads);
    const uint64_t cus = uint64_t(std::max(host::cu_count(), 1));
    p.waves = (p.list + 127u) / 128u * a.kv_heads >= cus ? 4u : 1u;
    p.tiles = (p.list + 32u * p.waves - 1u) / (32u * p.waves);
    const uint64_t blocks = p.tiles * a.kv_heads, key_tiles = (uint64_t(a.kv_rows) + 63u) / 64u;
    const uint64_t want = blocks >= 2u * cus ? 1u : (4u * cus + blocks - 1u) / blocks;
    p.splits = uint32_t(std::max<uint64_t>(1u, std::min<uint64_t>({want, key_tiles / 4u, 256u})));
    return p;
}

uint64_t workspace_bytes(const MH3DenseAttnArgs& a, const Plan& p)
{
    return p.splits > 1u ? uint64_t(p.splits) * a.kv_heads * p.list * 130u * 4u : 0u;
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
    if (!(a.scale >= 0.0f) || a.scale == __builtin_inff() || !(a.cap >= 0.0f) || a.cap == __builtin_inff())
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

template <int W, bool CAP, bool BIAS>
int launch_dense(const DenseParams& p, hipStream_t stream)
{
    const auto kernel = &attn_dense_kernel<W, CAP, BIAS>;
    const size_t lds = 2u * kTileBytes + 256u + 4096u * W + 8u * W;
    if (const hipError_t e = host::allow_dynamic_lds(reinterpret_cast<const void*>(kernel), lds); e != hipSuccess)
        return host::hip_error(e);
    const uint32_t blocks = (p.kv_heads * p.tiles * p.splits + 7u) / 8u * 8u;
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(W * 64), lds, stream, p);
    return host::check_launch();
}

template <int W>
int launch_by_score(const DenseParams& p, bool cap, bool bias, hipStream_t stream)
{
    if (cap)
        return bias ? launch_dense<W, true, true>(p, stream) : launch_dense<W, true, false>(p, stream);
    return bias ? launch_dense<W, false, true>(p, stream) : launch_dense<W, false, false>(p, stream);
}

} // namespace

extern "C" int64_t mh3_flash_attn_128_workspace_bytes(const MH3DenseAttnArgs* args)
{
    if (const int rc = check_args(args); rc != MH3_OK)
        return rc;
    if (args->q_rows == 0)
        return 0;
    return int64_t(workspace_bytes(*args, plan_of(*args)));
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
    const Plan plan = plan_of(a);
    const uint64_t need = workspace_bytes(a, plan);
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
    if (plan.tiles * a.kv_heads * plan.splits * plan.waves * 64u >= (1ull << 31))
        return MH3_ERR_SHAPE;
    DenseParams p{};
    p.q = q, p.k = k, p.v = v, p.out = out, p.ranges = ranges, p.slopes = slopes, p.q_pos = q_pos, p.k_pos = k_pos;
    p.part = static_cast<float*>(workspace);
    p.qhs = a.q_head_stride, p.qrs = a.q_row_stride, p.khs = a.k_head_stride, p.krs = a.k_row_stride;
    p.vhs = a.v_head_stride, p.vrs = a.v_row_stride, p.ohs = a.out_head_stride, p.ors = a.out_row_stride;
    p.kv_heads = a.kv_heads, p.group = a.heads / a.kv_heads, p.q_rows = a.q_rows, p.kv_rows = a.kv_rows;
    p.list = uint32_t(plan.list), p.tiles = uint32_t(plan.tiles), p.splits = plan.splits;
    p.div_group = FastDiv::make(p.group), p.div_tiles = FastDiv::make(p.tiles), p.div_splits = FastDiv::make(p.splits);
    const float scale = a.scale > 0.0f ? a.scale : 0.08838834764831845f; // 1 / sqrt(128)
    int pow = 0;
    std::frexp(scale, &pow);
    pow = std::min(std::max(pow, -16), 0);
    p.q_pow = std::ldexp(1.0f, pow);
    p.scale_log2 = scale / p.q_pow * kLog2e;
    if (a.cap > 0.0f)
        p.cap_in = 2.0f * kLog2e * (scale / p.q_pow) / a.cap, p.cap_out = a.cap * kLog2e;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const bool cap = a.cap > 0.0f, bias = slopes != nullptr;
    const int rc = plan.waves == 4u ? launch_by_score<4>(p, cap, bias, s) : launch_by_score<1>(p, cap, bias, s);
    if (rc != MH3_OK || p.splits == 1u)
        return rc;
    const uint64_t items = uint64_t(p.kv_heads) * p.list;
    hipLaunchKernelGGL(attn_join_kernel, dim3(uint32_t((items + 3u) / 4u)), dim3(256), 0, s, p);
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
