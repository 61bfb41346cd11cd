// `quant_rows_mx4`: rows to 4-bit microscaled floats (OCP MX), the operands of gemm_mx4.hip. Each block of 32 columns
// shares a power of two, 2^(floor(log2 max|block|) - 2), which puts its largest value in [4, 8); each value is then
// rounded to the nearest of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6}, ties to the even code, 6 at most. Weights go through it once
// at load, activations every step.
//
// HBM-bound: 2 bytes read (bf16) and 17/32 of a byte written a value. Four lanes take a block, 8 values each, so a
// wave's 16-byte loads cover 1 KB without gaps; the block's maximum is two DPP steps within the quad, and a quad's codes
// go out as one 16-byte run. 19,305 x 5376 in 51 us, 5.2 TB/s.
#include "mh3_common.hpp"

namespace mh3 {
namespace {

constexpr uint32_t kMx4Threads = 256;
constexpr int kMx4U = 4; // groups of 8 values a thread has in flight

template <int DT>
__device__ __forceinline__ void load8(const void* x, uint64_t at, float (&v)[8])
{
    if constexpr (DT == MH3_BF16) {
        const uint4 t = ld_stream(static_cast<const uint4*>(x) + at);
        const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v[2 * i] = bf16_lo(w[i]), v[2 * i + 1] = bf16_hi(w[i]);
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint4 t = ld_stream(static_cast<const uint4*>(x) + 2u * at + h);
            v[4 * h] = __uint_as_float(t.x), v[4 * h + 1] = __uint_as_float(t.y);
            v[4 * h + 2] = __uint_as_float(t.z), v[4 * h + 3] = __uint_as_float(t.w);
        }
    }
}

// Thread t of the launch takes the groups t, t + threads, ... of 8 values; every lane of a wave takes part in each (the
// quads' exchanges), the ones past the end with zeros.
template <int DT>
__global__ __launch_bounds__(kMx4Threads) void quant_mx4_kernel(const void* __restrict__ x, uint8_t* __restrict__ q,
                                                                uint8_t* __restrict__ scale, uint32_t row0, uint32_t rows,
                                                                uint64_t all_rows, uint32_t groups, FastDiv div_groups)
{
    const uint32_t n = rows * groups, base = blockIdx.x * kMx4Threads * kMx4U + threadIdx.x;
    float v[kMx4U][8];
#pragma unroll
    for (int u = 0; u < kMx4U; ++u) {
        const uint32_t g = base + kMx4Threads * uint32_t(u);
        if (g < n) {
            load8<DT>(x, uint64_t(row0) * groups + g, v[u]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                v[u][i] = 0.0f;
        }
    }
#pragma unroll
    for (int u = 0; u < kMx4U; ++u) {
        const uint32_t g = base + kMx4Threads * uint32_t(u);
        // The largest magnitude as a bit pattern: non-negative floats order as theirs, and infinity and NaN above all.
        uint32_t mx = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            mx = max(mx, __float_as_uint(v[u][i]) & 0x7fffffffu);
        mx = max(mx, uint32_t(__builtin_amdgcn_mov_dpp(int(mx), 0xB1, 0xF, 0xF, true)));
        mx = max(mx, uint32_t(__builtin_amdgcn_mov_dpp(int(mx), 0x4E, 0xF, 0xF, true)));
        // floor(log2) of it, less 2, plus the byte's bias of 127: its exponent field less 2 (0 where that is below, among
        // them zero and subnormal blocks). A block with an infinity or a NaN is all NaN: scale byte 255.
        const uint32_t e = mx >> 23;
        const bool bad = e == 255u;
        const uint32_t byte = bad ? 255u : e < 2u ? 0u : e - 2u;
        uint32_t codes = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = ldexpf(v[u][2 * i], 127 - int(byte)), b = ldexpf(v[u][2 * i + 1], 127 - int(byte));
            switch (i) { // the destination byte is an immediate
            case 0: codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, a, b, 1.0f, 0); break;
            case 1: codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, a, b, 1.0f, 1); break;
            case 2: codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, a, b, 1.0f, 2); break;
            default: codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, a, b, 1.0f, 3); break;
            }
        }
        if (g < n) {
            reinterpret_cast<uint32_t*>(q)[uint64_t(row0) * groups + g] = bad ? 0u : codes;
            if ((g & 3u) == 0u) {
                const uint32_t r = div_groups.div(g), block = (g - r * groups) / 4u;
                scale[((block / 8u) * all_rows + row0 + r) * 8u + block % 8u] = uint8_t(byte);
            }
        }
    }
}

} // namespace
} // namespace mh3

extern "C" int mh3_quant_rows_mx4(const MH3QuantArgs* a, const void* x, uint8_t* q, uint8_t* scale, mh3_stream_t stream)
{
    using namespace mh3;
    if (!a)
        return MH3_ERR_POINTER;
    if (a->dtype != MH3_F32 && a->dtype != MH3_BF16)
        return MH3_ERR_PARAM;
    if (a->cols == 0 || a->cols % 256u != 0)
        return MH3_ERR_SHAPE;
    if (a->rows == 0)
        return MH3_OK;
    if (a->rows >= (1u << 31) || a->cols >= (1u << 30))
        return MH3_ERR_SHAPE;
    if (!x || !q || !scale)
        return MH3_ERR_POINTER;
    if (!host::aligned16(x) || !host::aligned16(q) || !host::aligned16(scale))
        return MH3_ERR_ALIGN;
    const uint64_t n = uint64_t(a->rows) * a->cols;
    const host::Span in[] = {{x, n * (a->dtype == MH3_BF16 ? 2u : 4u)}};
    const host::Span out[] = {{q, n / 2u}, {scale, n / 32u}};
    if (host::any_overlap(in, out))
        return MH3_ERR_PARAM;
    // A launch's group index stays below 2^31.
    const uint32_t groups = a->cols / 8u, step = (1u << 30) / groups;
    for (uint32_t row0 = 0; row0 < a->rows; row0 += step) {
        const uint32_t rows = a->rows - row0 < step ? a->rows - row0 : step;
        const dim3 grid((rows * groups + kMx4Threads * kMx4U - 1u) / (kMx4Threads * kMx4U));
        const auto kernel = a->dtype == MH3_BF16 ? &quant_mx4_kernel<MH3_BF16> : &quant_mx4_kernel<MH3_F32>;
        hipLaunchKernelGGL(kernel, grid, dim3(kMx4Threads), 0, static_cast<hipStream_t>(stream), x, q, scale, row0, rows,
                           uint64_t(a->rows), groups, FastDiv::make(groups));
        if (const int rc = host::check_launch(); rc != MH3_OK)
            return rc;
    }
    return MH3_OK;
}
