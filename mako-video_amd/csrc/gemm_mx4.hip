// The block's products on 4-bit microscaled operands (OCP MX: blocks of 32 e2m1 values that share a power of two), on
// v_mfma_scale_f32_16x16x128_f8f6f4, which takes both operands' block scales with them. The calls are those of the
// int8 and bf16 forms (gemm.hip) with the same epilogues: a plain store (qkv), SwiGLU (fc1), gate_add_rows (out, fc2).
//   y[r][c] = sum over the blocks b of 2^(sx[r][b] + sw[c][b] - 254) sum_{i in b} x[r][i] w[c][i], in float.
//
// Design (gfx950), the tile kernels:
// - The wave layout, the LDS swizzle and the XCD map are gemm_kernel's: a row of an LDS stage is 128 bytes of k, here 256
//   values, and one MFMA operand is 16 bytes a lane, here the 32 values of one block. So each lane has one scale byte an
//   operand, and a K-step of 256 k is 64 MFMAs a wave (256 x 256 tiles) with four times the bf16 kernel's products.
// - The scale bytes come eight blocks (a K-step) of all rows at a time, [k / 256][rows][8]: a tile's are then one
//   contiguous run a K-step, 4 bytes a lane of one DMA instruction a wave, and an operand's byte is one ds_read_u8 (a
//   row's eight bytes in one read and a shift: 1 to 2% slower; no scale reads at all: 5% faster).
// - A ring of stages holds a whole K-step each. x's loads of tile kt + kStages start as soon as every wave has read tile
//   kt, behind the barrier that publishes tile kt + 1; w's and the scales' with the next step's first products, since all at
//   once held the products up behind them (256 x 256 tiles, 2985 x 5376 x 7168: 68 us, now 63 to 65).
// What bounds them: large products, the chip's power (19,305 x 5376 -> 2 x 14,336: 1.42 ms, 4.2 PFLOP/s, the clock at 1.6 to
// 1.8 GHz and the matrix cores busy 58% of it; the bare MFMA in a loop reaches 6.0 at 1.5 GHz, this kernel without its
// loads 4.75; loads a tile ahead with stores straight from registers, or four waves of 128 x 128, were slower); middle ones
// the rounds of tiles; few rows the weights' bytes (3 rows, 5376 x 14,336: 11.3 us, 41 MB at 3.6 TB/s with the launch in it).
#include "gemm.hpp"

#include <algorithm>
#include <cmath>

namespace mh3 {
namespace {

typedef int int32x8 __attribute__((ext_vector_type(8)));

typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ u32x4_t load_b128(__amdgpu_buffer_rsrc_t buffer, uint32_t offset, int soffset)
{
    return __builtin_amdgcn_raw_buffer_load_b128(buffer, offset, soffset, 0);
}

__device__ __forceinline__ u32x2_t load_b64(__amdgpu_buffer_rsrc_t buffer, uint32_t offset, int soffset)
{
    return __builtin_amdgcn_raw_buffer_load_b64(buffer, offset, soffset, 0);
}

constexpr uint32_t kPastEnd = 0x80000000u; // a buffer offset past num_records: the load reads zeros

template <int BM, int BN, int WM, int WN, int S>
struct Mx4Ring {
    static constexpr uint32_t kWaves = WM * WN, kStages = S;
    static constexpr uint32_t kA = BM * 128u, kB = 2u * BN * 128u, kScale = kWaves * 256u; // bytes
    static constexpr uint32_t kStage = kA + kB + 2u * kScale;
    static constexpr size_t kEpi = size_t(BM) * gemm_epi_stride(BN) * sizeof(float);
    static constexpr size_t kBytes = S * size_t(kStage) > kEpi ? S * size_t(kStage) : kEpi;
    static_assert(BM * 8u <= kScale && 2u * BN * 8u <= kScale, "one scale DMA a wave covers a tile");
    static_assert(kBytes <= 160u * 1024u, "the LDS");
};

template <int BM, int BN, int WM, int WN, int S, int EPI>
__global__ __launch_bounds__(WM* WN * 64) void gemm_mx4_kernel(const uint8_t* __restrict__ x,
                                                               const uint8_t* __restrict__ xs,
                                                               const uint8_t* __restrict__ w,
                                                               const uint8_t* __restrict__ ws,
                                                               uint16_t* __restrict__ out, uint32_t M, uint32_t N,
                                                               uint32_t K, uint32_t mt, uint32_t nt, GemmGate gg)
{
    using Ring = Mx4Ring<BM, BN, WM, WN, S>;
    constexpr uint32_t kWaves = WM * WN;
    constexpr int TM = BM / WM / 16, TN = BN / WN / 16; // MFMA tiles: rows, and gate (= up) columns
    constexpr int FA = TM / 2;                          // row tiles a sub-step holds
    static_assert(TM % 2 == 0);
    extern __shared__ u32x4_t smem[];
    char* const lds = reinterpret_cast<char*>(smem);
    uint32_t tm, tn;
    tile_of<BM>(mt, nt, tm, tn);
    const uint32_t m0 = tm * uint32_t(BM);
    const uint32_t w_lo = EPI == kSwiGLU ? tn * uint32_t(BN) : tn * 2u * BN;
    const uint32_t w_hi = EPI == kSwiGLU ? N + w_lo : w_lo + uint32_t(BN);
    const uint32_t w_rows = EPI == kSwiGLU ? 2u * N : N;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t wm = wave / WN, wn = wave % WN;
    const uint32_t KB = K / 2u, KT = K / 256u; // bytes of a row, K-steps

    // Operand loads: lane L of a wave's instruction i lands in chunk (wave AI + i) 64 + L = 8 row + physical chunk of
    // the stage and fetches the logical chunk that the swizzle puts there. Rows past M read zeros.
    constexpr int AI = BM * 8 / 64 / int(kWaves), BI = 2 * BN * 8 / 64 / int(kWaves);
    static_assert(AI * 64 * int(kWaves) == BM * 8 && BI * 64 * int(kWaves) == 2 * BN * 8);
    const uint64_t a_left = uint64_t(M - m0) * KB;
    const __amdgpu_buffer_rsrc_t ra =
        buffer_rsrc(x + uint64_t(m0) * KB, uint32_t(a_left < 0x7fffffffu ? a_left : 0x7fffffffu));
    const __amdgpu_buffer_rsrc_t rb = buffer_rsrc(w, w_rows * KB);
    uint32_t a_off[AI], b_off[BI];
#pragma unroll
    for (int i = 0; i < AI; ++i) {
        const uint32_t row = (wave * AI + uint32_t(i)) * 8u + (lane >> 3), c = (lane & 7u) ^ ((row >> 1) & 7u);
        a_off[i] = m0 + row < M ? row * KB + c * 16u : kPastEnd;
    }
#pragma unroll
    for (int i = 0; i < BI; ++i) {
        const uint32_t row = (wave * BI + uint32_t(i)) * 8u + (lane >> 3), c = (lane & 7u) ^ ((row >> 1) & 7u);
        b_off[i] = (row < uint32_t(BN) ? w_lo + row : w_hi + (row - uint32_t(BN))) * KB + c * 16u;
    }
    // Scale loads: dword d = 64 wave + lane of the stage's scales is word d % 2 of row d / 2.
    const __amdgpu_buffer_rsrc_t rsa = buffer_rsrc(xs, KT * M * 8u), rsb = buffer_rsrc(ws, KT * w_rows * 8u);
    uint32_t sa_off, sb_off;
    {
        const uint32_t d = wave * 64u + lane, row = d >> 1;
        const uint32_t wrow = row < uint32_t(BN) ? w_lo + row : w_hi + (row - uint32_t(BN));
        sa_off = row < uint32_t(BM) && m0 + row < M ? (m0 + row) * 8u + (d & 1u) * 4u : kPastEnd;
        sb_off = row < 2u * BN ? wrow * 8u + (d & 1u) * 4u : kPastEnd;
    }
    constexpr int kLoads = AI + BI + 2; // a wave's loads of one K-step
    auto issue_x = [&](uint32_t kt) {
        char* const stage = lds + (kt % S) * Ring::kStage;
#pragma unroll
        for (int i = 0; i < AI; ++i)
            lds_dma16(ra, stage + (wave * AI + uint32_t(i)) * 1024u, a_off[i], int(kt * 128u));
        __builtin_amdgcn_sched_barrier(0); // the waits count these loads
    };
    auto issue_rest = [&](uint32_t kt) {
        char* const stage = lds + (kt % S) * Ring::kStage;
#pragma unroll
        for (int i = 0; i < BI; ++i)
            lds_dma16(rb, stage + Ring::kA + (wave * BI + uint32_t(i)) * 1024u, b_off[i], int(kt * 128u));
        char* const sc = stage + Ring::kA + Ring::kB + wave * 256u;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsa, (lds_ptr_t)sc, 4, sa_off, int(kt * M * 8u), 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsb, (lds_ptr_t)(sc + Ring::kScale), 4, sb_off, int(kt * w_rows * 8u), 0,
                                                 0);
        __builtin_amdgcn_sched_barrier(0);
    };

    // Operands of sub-step ks (k-half h = ks / 2, the wave's row tiles (ks % 2) FA ..): 16 bytes a lane, row
    // lane % 16 of a tile and block 4 h + lane / 16 of the K-step, and that block's scale byte.
    // Every row a lane reads has the same swizzle, so a tile is a constant of 16 rows on.
    const uint32_t rs = lane % 16u, kq = lane >> 4, fsx = (rs >> 1) & 7u;
    const uint32_t arow = wm * uint32_t(BM / WM) + rs, brow = wn * 16u * TN + rs;
    const uint32_t as_off = Ring::kA + Ring::kB + arow * 8u + kq;
    const uint32_t bs_off = Ring::kA + Ring::kB + Ring::kScale + brow * 8u + kq;
    uint32_t a_at[2], b_at[2];
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
        a_at[h] = arow * 128u + ((4u * h + kq) ^ fsx) * 16u;
        b_at[h] = Ring::kA + brow * 128u + ((4u * h + kq) ^ fsx) * 16u;
    }
    auto frags_a = [&](uint32_t kt, uint32_t ks, u32x4_t (&fa)[FA], int (&sa)[FA]) {
        const char* const stage = lds + (kt % S) * Ring::kStage;
        const char* const A = stage + a_at[ks >> 1];
        const char* const SA = stage + as_off;
#pragma unroll
        for (int t = 0; t < FA; ++t) {
            const int tile = int(ks & 1u) * FA + t;
            fa[t] = *reinterpret_cast<const u32x4_t*>(A + tile * 2048);
            sa[t] = *reinterpret_cast<const uint8_t*>(SA + tile * 128 + 4 * int(ks >> 1));
        }
    };
    auto frags_b = [&](uint32_t kt, uint32_t ks, u32x4_t (&fb)[2 * TN], int (&sb)[2 * TN]) {
        const char* const stage = lds + (kt % S) * Ring::kStage;
        const char* const B = stage + b_at[ks >> 1];
        const char* const SB = stage + bs_off;
#pragma unroll
        for (int t = 0; t < 2 * TN; ++t) {
            const int row = 16 * (t % TN) + (t >= TN ? BN : 0);
            fb[t] = *reinterpret_cast<const u32x4_t*>(B + row * 128);
            sb[t] = *reinterpret_cast<const uint8_t*>(SB + row * 8 + 4 * int(ks >> 1));
        }
    };

    floatx4 acc[TM][2 * TN];
#pragma unroll
    for (int a = 0; a < TM; ++a)
#pragma unroll
        for (int b = 0; b < 2 * TN; ++b)
            acc[a][b] = floatx4{};
    u32x4_t fa[2][FA], fb[2][2 * TN]; // double buffers: A by sub-step, B by k-half
    int sa[2][FA], sb[2][2 * TN];
    auto widen = [](const u32x4_t& v) { return int32x8{int(v[0]), int(v[1]), int(v[2]), int(v[3]), 0, 0, 0, 0}; };
    auto mfmas = [&](uint32_t ks, const u32x4_t (&a)[FA], const int (&as)[FA], const u32x4_t (&b)[2 * TN],
                     const int (&bs)[2 * TN]) {
        const int t0 = int(ks & 1u) * FA;
#pragma unroll
        for (int i = 0; i < FA; ++i)
#pragma unroll
            for (int j = 0; j < 2 * TN; ++j) // formats 4: e2m1
                acc[t0 + i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(widen(a[i]), widen(b[j]), acc[t0 + i][j],
                                                                                 4, 4, 0, as[i], 0, bs[j]);
    };

    for (uint32_t t = 0; t < uint32_t(S); ++t)
        if (t < KT) {
            issue_x(t);
            if (t + 1u < uint32_t(S))
                issue_rest(t); // the last stage's goes out with the first step
        }
    if (KT >= uint32_t(S))
        __builtin_amdgcn_s_waitcnt(waitcnt_vm((S - 2) * kLoads + AI));
    else
        __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
    asm volatile("" ::"s"(out), "s"(gg.gate), "s"(gg.set_of_row)); // no scalar load in flight in the loop
    lds_barrier();
    frags_a(0, 0, fa[0], sa[0]);
    frags_b(0, 0, fb[0], sb[0]);
    // One K-step of tile kt; more: tile kt + S exists; rest: tile kt + S - 1 does; last: there is no tile kt + 1. No branch lies between the MFMAs (the
    // compiler sinks them past one, to the step's end, and then spills the operands that all wait for it).
    auto kstep = [&](uint32_t kt, auto more, auto rest, auto last) {
        constexpr bool kMore = decltype(more)::value, kRest = decltype(rest)::value, kLast = decltype(last)::value;
        frags_a(kt, 1, fa[1], sa[1]);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (kRest)
            issue_rest(kt + uint32_t(S) - 1u);
        mfmas(0, fa[0], sa[0], fb[0], sb[0]);
        frags_a(kt, 2, fa[0], sa[0]);
        frags_b(kt, 2, fb[1], sb[1]);
        __builtin_amdgcn_sched_barrier(0);
        mfmas(1, fa[1], sa[1], fb[0], sb[0]);
        frags_a(kt, 3, fa[1], sa[1]);
        __builtin_amdgcn_sched_barrier(0);
        mfmas(2, fa[0], sa[0], fb[1], sb[1]);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (!kLast) {
            // Loads complete in order: tile kt + 1 is there once only the later tiles' loads are left.
            __builtin_amdgcn_s_waitcnt(waitcnt_vm(kMore ? (S - 2) * kLoads : 0));
            lds_barrier();
            frags_a(kt + 1, 0, fa[0], sa[0]);
            frags_b(kt + 1, 0, fb[0], sb[0]);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (kMore)
                issue_x(kt + uint32_t(S)); // into the stage that every wave has read
        }
        __builtin_amdgcn_sched_barrier(0);
        mfmas(3, fa[1], sa[1], fb[1], sb[1]);
    };
    using Yes = std::true_type;
    using No = std::false_type;
    uint32_t kt = 0;
    for (; kt + uint32_t(S) < KT; ++kt)
        kstep(kt, Yes{}, Yes{}, No{});
    if (KT >= uint32_t(S)) // S >= 2, so this step is not the last
        kstep(kt++, No{}, Yes{}, No{});
    for (; kt + 1u < KT; ++kt)
        kstep(kt, No{}, No{}, No{});
    kstep(kt, No{}, No{}, Yes{});

    gemm_epilogue<BM, BN, WM, WN, kBf16, EPI, TM, TN>(acc, smem, M, N, m0, w_lo, w_hi, nullptr, nullptr, out, gg);
}

// Up to 16 MT rows: the time is w's one pass from memory. A workgroup takes 32 rows of w (SwiGLU: 16 gate rows and their
// 16 up rows), its eight waves the K-steps in turn, from memory straight into registers; their sums are joined through LDS
// in the waves' order. The products are w x^T: a lane then holds four consecutive columns of one row of the result.
// (3 rows, 5376 x 14,336: 11.3 us. With 16 rows of w a workgroup 15.0, with 64 21.8; sixteen waves 13.2; two steps ahead
// 14.1, where the loads past the end cost as much as others; non-temporal loads 15.1; the 64 x 128 tiles 26.)
constexpr uint32_t kFewWaves = 8, kFewTiles = 2; // tiles of 16 rows of w

template <int MT, int EPI>
__global__ __launch_bounds__(kFewWaves * 64) void gemm_mx4_few_kernel(const uint8_t* __restrict__ x,
                                                                      const uint8_t* __restrict__ xs,
                                                                      const uint8_t* __restrict__ w,
                                                                      const uint8_t* __restrict__ ws,
                                                                      uint16_t* __restrict__ out, uint32_t M, uint32_t N,
                                                                      uint32_t K, GemmGate gg)
{
    constexpr uint32_t NT = kFewTiles, kPair = EPI == kSwiGLU ? 1u : NT; // column tiles of the result
    __shared__ floatx4 part[kFewWaves][MT * NT][64];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t KB = K / 2u, KT = K / 256u, w_rows = EPI == kSwiGLU ? 2u * N : N, n0 = blockIdx.x * 16u * kPair;
    const uint32_t r = lane % 16u, kq = lane >> 4, shift = kq * 8u;

    // A thread's four results: columns 16 j + 4 kq .. of row 16 i + r, for the wave's tile (i, j). What the epilogue adds
    // to is on its way while the products are made.
    const uint32_t ti = wave / kPair, tj = wave % kPair;
    const uint32_t row = 16u * ti + r, col = n0 + 16u * tj + kq * 4u;
    const bool stores = wave < MT * kPair && row < M;
    const uint64_t at = uint64_t(row) * N + col;
    floatx4 gate{}, res{};
    if constexpr (EPI == kGateAdd || EPI == kGateAddF32) {
        if (stores) {
            const uint32_t set = gg.set_of_row ? min(uint32_t(gg.set_of_row[row]), gg.n_sets - 1u) : 0u;
            const float* const g = gg.gate + uint64_t(set) * gg.gate_stride + col;
            gate = floatx4{g[0], g[1], g[2], g[3]};
            if constexpr (EPI == kGateAddF32) {
                res = *reinterpret_cast<const floatx4*>(reinterpret_cast<const float*>(out) + at);
            } else {
                const uint2 v = *reinterpret_cast<const uint2*>(out + at);
                res = floatx4{bf16_lo(v.x), bf16_hi(v.x), bf16_lo(v.y), bf16_hi(v.y)};
            }
        }
    }

    // A lane's 16 bytes of a K-step's half h are block 4 h + kq of its row. Rows past M repeat the last one.
    const __amdgpu_buffer_rsrc_t ra = buffer_rsrc(x, M * KB), rb = buffer_rsrc(w, w_rows * KB);
    const __amdgpu_buffer_rsrc_t rsa = buffer_rsrc(xs, KT * M * 8u), rsb = buffer_rsrc(ws, KT * w_rows * 8u);
    uint32_t a_row[MT], b_row[NT];
#pragma unroll
    for (uint32_t t = 0; t < MT; ++t)
        a_row[t] = min(16u * t + r, M - 1u);
#pragma unroll
    for (uint32_t t = 0; t < NT; ++t)
        b_row[t] = n0 + r + (EPI == kSwiGLU ? t * N : 16u * t);

    floatx4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < int(NT); ++j)
            acc[i][j] = floatx4{};
    auto widen = [](const u32x4_t& v) { return int32x8{int(v[0]), int(v[1]), int(v[2]), int(v[3]), 0, 0, 0, 0}; };
    struct Step {
        u32x4_t fa[MT][2], fb[NT][2];
        u32x2_t sa[MT], sb[NT];
    };
    auto load = [&](uint32_t kt, Step& p) {
#pragma unroll
        for (int t = 0; t < int(NT); ++t) {
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h)
                p.fb[t][h] = load_b128(rb, b_row[t] * KB + kq * 16u + h * 64u, int(kt * 128u));
            p.sb[t] = load_b64(rsb, b_row[t] * 8u, int(kt * w_rows * 8u));
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) {
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h)
                p.fa[t][h] = load_b128(ra, a_row[t] * KB + kq * 16u + h * 64u, int(kt * 128u));
            p.sa[t] = load_b64(rsa, a_row[t] * 8u, int(kt * M * 8u));
        }
        __builtin_amdgcn_sched_barrier(0); // before the products of the step before
    };
    auto multiply = [&](const Step& p) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < int(NT); ++j)
#pragma unroll
                for (int i = 0; i < MT; ++i)
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                        widen(p.fb[j][h]), widen(p.fa[i][h]), acc[i][j], 4, 4, 0, int(p.sb[j][h] >> shift), 0,
                        int(p.sa[i][h] >> shift));
        __builtin_amdgcn_sched_barrier(0);
    };
    // A step's loads go out before the products of the step before it.
    if (wave < KT) {
        Step p[2];
        load(wave, p[0]);
        uint32_t kt = wave;
        for (; kt + 2u * kFewWaves < KT; kt += 2u * kFewWaves) {
            load(kt + kFewWaves, p[1]);
            multiply(p[0]);
            load(kt + 2u * kFewWaves, p[0]);
            multiply(p[1]);
        }
        if (kt + kFewWaves < KT)
            load(kt + kFewWaves, p[1]);
        multiply(p[0]);
        if (kt + kFewWaves < KT)
            multiply(p[1]);
    }

#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < int(NT); ++j)
            part[wave][i * int(NT) + j][lane] = acc[i][j];
    __syncthreads();
    if (!stores)
        return;
    auto joined = [&](uint32_t tile) {
        floatx4 y = part[0][tile][lane];
#pragma unroll
        for (uint32_t v = 1; v < kFewWaves; ++v)
            y += part[v][tile][lane];
        return y;
    };
    floatx4 y = joined(ti * NT + tj);
    if constexpr (EPI == kSwiGLU) {
        const floatx4 up = joined(ti * NT + 1u);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            y[e] = y[e] * __builtin_amdgcn_rcpf(1.0f + __expf(-y[e])) * up[e];
    }
    if constexpr (EPI == kGateAdd || EPI == kGateAddF32)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            y[e] = fmaf(gate[e], y[e], res[e]);
    if constexpr (EPI == kGateAddF32)
        *reinterpret_cast<floatx4*>(reinterpret_cast<float*>(out) + at) = y;
    else
        *reinterpret_cast<uint2*>(out + at) = uint2{pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3])};
}

// The launch with tiles of BM rows and BN columns (2 BN where the epilogue pairs none).
template <int BM, int BN, int WM, int WN, int S, int EPI>
int launch_tile(const MH3GemmArgs* a, const uint8_t* x, const uint8_t* xs, const uint8_t* w, const uint8_t* ws,
                uint16_t* out, const GemmGate& gg, mh3_stream_t stream)
{
    const auto kernel = &gemm_mx4_kernel<BM, BN, WM, WN, S, EPI>;
    constexpr size_t kLds = Mx4Ring<BM, BN, WM, WN, S>::kBytes;
    if (const hipError_t e = host::allow_dynamic_lds(reinterpret_cast<const void*>(kernel), kLds); e != hipSuccess)
        return host::hip_error(e);
    const uint32_t mt = (a->m + uint32_t(BM) - 1u) / uint32_t(BM), nt = a->n / (EPI == kSwiGLU ? BN : 2 * BN);
    hipLaunchKernelGGL(kernel, dim3(mt * nt), dim3(WM * WN * 64), kLds, static_cast<hipStream_t>(stream), x, xs, w, ws,
                       out, a->m, a->n, a->k, mt, nt, gg);
    return host::check_launch();
}

template <int MT, int EPI>
int launch_few(const MH3GemmArgs* a, const uint8_t* x, const uint8_t* xs, const uint8_t* w, const uint8_t* ws,
               uint16_t* out, const GemmGate& gg, mh3_stream_t stream)
{
    hipLaunchKernelGGL((gemm_mx4_few_kernel<MT, EPI>), dim3(a->n / (EPI == kSwiGLU ? 16u : 32u)), dim3(kFewWaves * 64), 0,
                       static_cast<hipStream_t>(stream), x, xs, w, ws, out, a->m, a->n, a->k, gg);
    return host::check_launch();
}

// The kernels by their tiles: rows, and rows of w.
enum Mx4Tile { kFew, k64x64, k64x128, k128x128, k192x256, k256x256 };

// The kernel of least estimated time (us), from the sizes alone. A tile kernel: rounds of the 256 CUs, each the K-steps'
// time in one tile; measured on one round of 21 .. 56 steps, 0.34, 0.45 .. 0.55, 0.68 .. 0.75, 1.4 .. 1.6 and 1.55 .. 1.8
// us a step (64 x 64 to 256 x 256). The few-row kernel: its bytes, x's from the caches, at the rate that either reads w
// from memory with.
// At n 5376, k 14336, rows 1, 32, 128, 512, 1024: few 11.3, 17.1, -; 64 x 64 22.5, 22.3, 23.3, 52, 90; 64 x 128 25.8, 27.8,
// 31, 57, 84; 128 x 128 -, -, 41, 40, 79; 192 x 256 -, -, 85, 84, 84; 256 x 256 -, -, 88, 91, 90. At n 21504, k 5376, rows
// 1, 64, 192, 945: few 13.1, -; 64 x 64 15.8, 19.4, 31, 116; 64 x 128 14.1, 16.4, 27.6, 104; 128 x 128 -, 17.8, 33, 96;
// 192 x 256 -, 35, 37, 80; 256 x 256 -, 37, 39, 79. (A tile's K-steps split over two groups of waves: 43 for 31 at 128 rows
// of the first.)
Mx4Tile tile_of_sizes(uint32_t m, uint32_t w_rows, uint32_t k)
{
    const float steps = float(k / 256u), kStart = 4.0f, kRate = 6.2e6f; // bytes a us
    const float w_us = float(w_rows) * float(k) * (0.53125f / kRate);
    struct Tile {
        Mx4Tile tile;
        uint32_t rows, cols;
        float step_us;
    };
    constexpr Tile kTiles[] = {
        {k256x256, 256, 256, 1.65f}, {k192x256, 192, 256, 1.5f}, {k128x128, 128, 128, 0.71f}, {k64x128, 64, 128, 0.48f},
        {k64x64, 64, 64, 0.35f}};
    Mx4Tile best = k256x256;
    float least = INFINITY;
    for (const Tile& t : kTiles) {
        const uint64_t tiles = uint64_t((m + t.rows - 1u) / t.rows) * (w_rows / t.cols);
        const float us = kStart + std::max(float((tiles + 255u) / 256u) * steps * t.step_us, w_us);
        if (us < least)
            least = us, best = t.tile;
    }
    const float x_us = float(w_rows / 32u) * float(m) * float(k) * (0.5f * 0.7f / kRate);
    return m <= 32u && kStart + w_us + x_us <= least ? kFew : best;
}

// The checks of the four entry points and their launch.
template <int EPI>
int launch_mx4(const MH3GemmArgs* a, const uint8_t* x, const uint8_t* xs, const uint8_t* w, const uint8_t* ws,
               uint16_t* out, const GemmGate& gg, mh3_stream_t stream)
{
    constexpr uint32_t kCols = EPI == kSwiGLU ? kBN : 2u * kBN;
    if (!a)
        return MH3_ERR_POINTER;
    if (a->m == 0 || a->k == 0 || a->n == 0 || a->k % 256u != 0 || a->n % kCols != 0)
        return MH3_ERR_SHAPE;
    const uint64_t w_rows = EPI == kSwiGLU ? 2ull * a->n : a->n;
    if (a->m >= (1u << 31) || w_rows >= (uint64_t(1) << 31))
        return MH3_ERR_SHAPE;
    // 32-bit buffer offsets: a tile's rows of x, all of w, and all of either's scales.
    if (uint64_t(a->k) / 2u * kBM >= (uint64_t(1) << 31) || w_rows * a->k / 2u >= (uint64_t(1) << 31) ||
        uint64_t(a->m) * (a->k / 32u) >= (uint64_t(1) << 31))
        return MH3_ERR_UNSUPPORTED;
    if (!x || !xs || !w || !ws || !out)
        return MH3_ERR_POINTER;
    constexpr bool kGate = EPI == kGateAdd || EPI == kGateAddF32;
    if (kGate && (!gg.gate || gg.n_sets == 0 || gg.n_sets > 256 || gg.gate_stride < a->n))
        return gg.gate ? MH3_ERR_PARAM : MH3_ERR_POINTER;
    if (!host::aligned16(x) || !host::aligned16(xs) || !host::aligned16(w) || !host::aligned16(ws) ||
        !host::aligned16(out) || (kGate && reinterpret_cast<uintptr_t>(gg.gate) % 4u != 0u))
        return MH3_ERR_ALIGN;
    // The output may not overlap anything that other tiles still read.
    const uint64_t x_bytes = uint64_t(a->m) * (a->k / 2u), w_bytes = w_rows * (a->k / 2u);
    const host::Span in[] = {
        {x, x_bytes},
        {xs, x_bytes / 16u},
        {w, w_bytes},
        {ws, w_bytes / 16u},
        {gg.gate, kGate ? (uint64_t(gg.n_sets) - 1u) * gg.gate_stride * 4u + a->n * 4ull : 0u},
        {gg.set_of_row, kGate ? uint64_t(a->m) : 0u}};
    const host::Span o[] = {{out, uint64_t(a->m) * a->n * (EPI == kGateAddF32 ? 4u : 2u)}};
    if (host::any_overlap(in, o))
        return MH3_ERR_PARAM;
    const uint32_t nt = a->n / kCols;
    if (uint64_t((a->m + 63u) / 64u) * nt * 4u >= (uint64_t(1) << 23)) // a launch holds under 2^32 threads
        return MH3_ERR_SHAPE;
    switch (tile_of_sizes(a->m, uint32_t(w_rows), a->k)) {
    case kFew:
        return a->m <= 16u ? launch_few<1, EPI>(a, x, xs, w, ws, out, gg, stream)
                           : launch_few<2, EPI>(a, x, xs, w, ws, out, gg, stream);
    case k64x64:
        return launch_tile<64, 32, 2, 2, 4, EPI>(a, x, xs, w, ws, out, gg, stream);
    case k64x128:
        return launch_tile<64, 64, 2, 4, 4, EPI>(a, x, xs, w, ws, out, gg, stream);
    case k128x128:
        return launch_tile<128, 64, 2, 4, 3, EPI>(a, x, xs, w, ws, out, gg, stream);
    case k192x256:
        return launch_tile<192, 128, 2, 4, 2, EPI>(a, x, xs, w, ws, out, gg, stream);
    case k256x256:
        break;
    }
    return launch_tile<256, 128, 2, 4, 2, EPI>(a, x, xs, w, ws, out, gg, stream);
}

const GemmGate kNoGate{nullptr, nullptr, 0, 0};

GemmGate gate_of(const MH3GemmArgs* a, const float* gate, const uint8_t* set_of_row)
{
    const uint32_t n_sets = a && a->n_sets ? a->n_sets : 1u;
    const uint32_t stride = a && a->gate_stride ? a->gate_stride : (a ? a->n : 0u);
    return GemmGate{gate, set_of_row, stride, n_sets};
}

} // namespace
} // namespace mh3

extern "C" int mh3_gemm_mx4(const MH3GemmArgs* a, const uint8_t* x, const uint8_t* x_scale, const uint8_t* w,
                            const uint8_t* w_scale, uint16_t* out, mh3_stream_t stream)
{
    return mh3::launch_mx4<mh3::kStore>(a, x, x_scale, w, w_scale, out, mh3::kNoGate, stream);
}

extern "C" int mh3_gemm_mx4_swiglu(const MH3GemmArgs* a, const uint8_t* x, const uint8_t* x_scale, const uint8_t* w,
                                   const uint8_t* w_scale, uint16_t* out, mh3_stream_t stream)
{
    return mh3::launch_mx4<mh3::kSwiGLU>(a, x, x_scale, w, w_scale, out, mh3::kNoGate, stream);
}

extern "C" int mh3_gemm_mx4_gate_add(const MH3GemmArgs* a, const uint8_t* x, const uint8_t* x_scale, const uint8_t* w,
                                     const uint8_t* w_scale, const float* gate, const uint8_t* set_of_row,
                                     uint16_t* residual, mh3_stream_t stream)
{
    return mh3::launch_mx4<mh3::kGateAdd>(a, x, x_scale, w, w_scale, residual, mh3::gate_of(a, gate, set_of_row),
                                          stream);
}

extern "C" int mh3_gemm_mx4_gate_add_f32(const MH3GemmArgs* a, const uint8_t* x, const uint8_t* x_scale,
                                         const uint8_t* w, const uint8_t* w_scale, const float* gate,
                                         const uint8_t* set_of_row, float* residual, mh3_stream_t stream)
{
    return mh3::launch_mx4<mh3::kGateAddF32>(a, x, x_scale, w, w_scale, reinterpret_cast<uint16_t*>(residual),
                                             mh3::gate_of(a, gate, set_of_row), stream);
}
