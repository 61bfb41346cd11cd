// What the block's GEMM kernels share: LDS access, the workgroup-to-tile map and the epilogues (gemm.hip: bf16 and int8
// operands; gemm_mx4.hip: 4-bit microscaled ones).
#pragma once

#include "mh3_common.hpp"

#include <type_traits>

namespace mh3 {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kBM = 256, kBN = 128, kBK = 64; // kBM: the largest row tile

constexpr uint32_t kBandM = 4; // row tiles an XCD sweeps across all column tiles before moving on

typedef __attribute__((address_space(3))) void* lds_ptr_t;

// 16 bytes a lane from a buffer straight into LDS: lane L's bytes land at lds + 16 L (buffer_load_dwordx4 ... lds).
__device__ __forceinline__ void lds_dma16(__amdgpu_buffer_rsrc_t rsrc, void* lds, uint32_t voffset, int soffset)
{
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr_t)lds, 16, voffset, soffset, 0, 0);
}

// 16-byte chunk c of a 128-byte LDS row r sits at chunk c ^ ((r >> 1) & 7): the 16 rows an MFMA operand read touches
// per half-wave then cover all 64 banks once.
__device__ __forceinline__ uint32_t swz(uint32_t row, uint32_t chunk) { return row * 8u + (chunk ^ ((row >> 1) & 7u)); }

template <int BM>
__device__ __forceinline__ void tile_of(uint32_t mt, uint32_t nt, uint32_t& tm, uint32_t& tn)
{
    constexpr uint32_t kBand = kBandM * kBM / uint32_t(BM);
    const uint32_t nb = gridDim.x, b = blockIdx.x;
    const uint32_t logical = (nb % 8u == 0u) ? (b % 8u) * (nb / 8u) + b / 8u : b;
    const uint32_t band = logical / (kBand * nt), within = logical - band * kBand * nt;
    const uint32_t in_band = min(kBand, mt - band * kBand);
    tm = band * kBand + within % in_band;
    tn = within / in_band;
}

// s_waitcnt immediate that waits for vmcnt <= n only (gfx9 encoding: vmcnt in bits 3:0 and 15:14, expcnt 6:4,
// lgkmcnt 11:8).
constexpr int waitcnt_vm(int n) { return (n & 0xF) | (((n >> 4) & 3) << 14) | (0x7 << 4) | (0xF << 8); }

// All LDS accesses before it done, then the workgroup barrier; the asm statements keep the compiler from moving
// memory accesses across it.
__device__ __forceinline__ void lds_barrier()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F); // lgkmcnt(0), vmcnt and expcnt unconstrained
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

constexpr int kGemmWM = 2; // wavefronts along the tile's rows
constexpr int kGemmWN = 4; // wavefronts along its columns

// The three fc1 forms: int8 weights widened to bf16 with bf16 activations (weight-only), bf16 weights, and int8
// weights with int8 activations (each row of x with its own scale) on the int8 MFMA.
enum GemmMode { kW8A16 = 0, kBf16 = 1, kW8A8 = 2 };
// What the epilogue does with y = x w^T (scaled):
//   kSwiGLU:  out[m][N] = silu(y gate column) * y up column; w holds N gate rows then N up rows (fc1);
//   kStore:   out[m][N] = y; w holds N rows (the qkv projection);
//   kGateAdd: out[m][N] += gate[set(row)] * y, in place on the bf16 residual (the out projection and fc2, with the
//             reference's gate_add_rows folded in);
//   kGateAddF32: the same on a float residual (the reference's float residual stream), out read as float [m][N].
// With kSwiGLU a tile's 256 weight rows are 128 gate rows from n0 and the 128 matching up rows from N + n0; otherwise
// they are 256 consecutive rows, so both halves of the wave's accumulators are output columns.
enum GemmEpi { kSwiGLU = 0, kStore = 1, kGateAdd = 2, kGateAddF32 = 3 };

// The epilogue's extra operands (kGateAdd): gate vectors [n_sets][gate_stride] floats, a set per row (NULL: set 0).
struct GemmGate {
    const float* gate;
    const uint8_t* set_of_row;
    uint32_t gate_stride, n_sets;
};

typedef int int32x4 __attribute__((ext_vector_type(4)));

// Floats a row of the epilogue's staged half-tile: 4 rows apart = 32 banks apart. The kernel's LDS holds BM such rows.
constexpr uint32_t gemm_epi_stride(int bn) { return uint32_t(bn) + 8u; }

// The epilogue shared by the GEMM kernels, through the LDS (idle after the last K-step). acc[a][b][e] is y[r][c]
// with c = lane % 16 + 16 b + wn 16 TN within the tile's first BN w rows (b < TN) or, for acc[a][TN + b], the same
// position in its second BN, and tile row r = wm (BM / WM) + a 16 + 4 (lane / 16) + e. A
// BN-column half of the tile at a time, each wave writes its scaled results as floats into a [BM][kEpiStride] LDS
// tile (the two half-waves' rows, 4 apart, fall on disjoint banks); then each thread takes 8 consecutive columns of
// a row, so the output, and with kGateAdd the residual, moves in 16-byte accesses, BN / 8 threads to a row.
// The results round to bf16 once, at the end, as they would written straight from the registers.
template <int BM, int BN, int WM, int WN, int MODE, int EPI, int TM, int TN, typename Acc>
__device__ __forceinline__ void gemm_epilogue(Acc (&acc)[TM][2 * TN], u32x4_t* smem, uint32_t M, uint32_t N,
                                              uint32_t m0, uint32_t w_lo, uint32_t w_hi,
                                              const float* __restrict__ scale, const float* __restrict__ xscale,
                                              uint16_t* __restrict__ out, const GemmGate& gg)
{
    constexpr uint32_t kThreads = WM * WN * 64;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, wm = wave / WN, wn = wave % WN;
    const uint32_t rl = lane % 16u;
    constexpr uint32_t kEpiStride = gemm_epi_stride(BN);
    constexpr int kHalves = EPI == kSwiGLU ? 1 : 2;
    float* const stage = reinterpret_cast<float*>(smem);
    lds_barrier(); // every wave is done with the last K-step's fragments
#pragma unroll
    for (int hv = 0; hv < kHalves; ++hv) {
        if (hv)
            lds_barrier(); // the first half is read out
#pragma unroll
        for (int b = 0; b < TN; ++b) {
            const uint32_t c = wn * 16u * TN + uint32_t(b) * 16u + rl;
            const float s_lo = MODE != kBf16 ? scale[w_lo + c] : 1.0f, s_hi = MODE != kBf16 ? scale[w_hi + c] : 1.0f;
#pragma unroll
            for (int a = 0; a < TM; ++a) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t r = wm * (uint32_t(BM) / WM) + uint32_t(a) * 16u + 4u * (lane >> 4) + uint32_t(e);
                    const float sx = MODE == kW8A8 ? xscale[min(m0 + r, M - 1u)] : 1.0f;
                    float v;
                    if constexpr (EPI == kSwiGLU) {
                        const float lo = float(acc[a][b][e]) * s_lo * sx, hi = float(acc[a][TN + b][e]) * s_hi * sx;
                        v = lo * __builtin_amdgcn_rcpf(1.0f + __expf(-lo)) * hi;
                    } else {
                        v = hv == 0 ? float(acc[a][b][e]) * s_lo * sx : float(acc[a][TN + b][e]) * s_hi * sx;
                    }
                    stage[r * kEpiStride + c] = v;
                }
            }
        }
        lds_barrier();
        // Output column of staged column 0: the tile's gate columns (SwiGLU), else its first or second 128 columns.
        const uint32_t col0 = hv == 0 ? w_lo : w_hi;
        for (uint32_t q = tid; q < uint32_t(BM) * (BN / 8u); q += kThreads) {
            const uint32_t r = q / (BN / 8u), c8 = (q % (BN / 8u)) * 8u, row = m0 + r;
            if (row >= M)
                break; // rows grow with q
            const float4 v0 = *reinterpret_cast<const float4*>(stage + r * kEpiStride + c8);
            const float4 v1 = *reinterpret_cast<const float4*>(stage + r * kEpiStride + c8 + 4u);
            float o[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
            if constexpr (EPI == kGateAddF32) {
                // The float residual: 32 bytes a thread, x += gate * y with one float rounding.
                const uint32_t set = gg.set_of_row ? min(uint32_t(gg.set_of_row[row]), gg.n_sets - 1u) : 0u;
                const float* g = gg.gate + uint64_t(set) * gg.gate_stride + col0 + c8;
                float4* fdst = reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + uint64_t(row) * N + col0 + c8);
                const float4 r0 = fdst[0], r1 = fdst[1];
                fdst[0] = float4{fmaf(g[0], o[0], r0.x), fmaf(g[1], o[1], r0.y), fmaf(g[2], o[2], r0.z),
                                 fmaf(g[3], o[3], r0.w)};
                fdst[1] = float4{fmaf(g[4], o[4], r1.x), fmaf(g[5], o[5], r1.y), fmaf(g[6], o[6], r1.z),
                                 fmaf(g[7], o[7], r1.w)};
                continue;
            }
            uint4* dst = reinterpret_cast<uint4*>(out + uint64_t(row) * N + col0 + c8);
            if constexpr (EPI == kGateAdd) {
                const uint32_t set = gg.set_of_row ? min(uint32_t(gg.set_of_row[row]), gg.n_sets - 1u) : 0u;
                const float* g = gg.gate + uint64_t(set) * gg.gate_stride + col0 + c8;
                const uint4 res = *dst;
                const uint32_t rw[4] = {res.x, res.y, res.z, res.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    o[2 * i] = fmaf(g[2 * i], o[2 * i], bf16_lo(rw[i]));
                    o[2 * i + 1] = fmaf(g[2 * i + 1], o[2 * i + 1], bf16_hi(rw[i]));
                }
            }
            *dst = uint4{pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]), pack_bf16(o[4], o[5]), pack_bf16(o[6], o[7])};
        }
    }
}

} // namespace mh3
