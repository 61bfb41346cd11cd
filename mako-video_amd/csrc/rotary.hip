// `rotary_axes`: the cos / sin tables that heads_partial and heads_partial_pool read, from integer positions on up to
// four axes (a video's time, height and width). The reference builds its tables on the host; here they are made where
// they are read. A thread takes one (row, pair): 8 bytes written for some 45 instructions, so a long table is bound by
// HBM and a short one by the launch (212 rows of 48 pairs: 3 us).
#include "rotary.hpp"

#include <cmath>

namespace mh3 {
namespace {

constexpr uint32_t kRotaryThreads = 256;

__global__ __launch_bounds__(kRotaryThreads) void rotary_axes_kernel(RotaryParams p, FastDiv div_half, uint32_t first,
                                                                     uint32_t rows, float* __restrict__ cos_t,
                                                                     float* __restrict__ sin_t)
{
    const uint32_t n = blockIdx.x * kRotaryThreads + threadIdx.x, r = div_half.div(n);
    if (r >= rows)
        return;
    const uint32_t i = n - r * p.half;
    const uint64_t row = uint64_t(first) + r;
    float c, s;
    row_cos_sin(p, row, i, c, s);
    cos_t[row * p.half + i] = c;
    sin_t[row * p.half + i] = s;
}

} // namespace

namespace host {

int rotary_setup(const MH3AxesArgs* args, const int32_t* pos, uint32_t half, RotaryParams& p)
{
    if (!args)
        return MH3_ERR_POINTER;
    const MH3AxesArgs& a = *args;
    if (a.axes == 0 || a.axes > 4u)
        return MH3_ERR_PARAM;
    p = RotaryParams{};
    p.pos = pos, p.axes = a.axes;
    uint64_t at = 0;
    long double power[kMaxRotPairs + 3];
    for (uint32_t x = 0; x < a.axes; ++x) {
        // Frequencies at most |step| (theta >= 1), so a position is below 2^18 turns and F keeps 46 bits of fraction
        // at the extreme, all 64 for steps of a turn or less.
        if (!(a.theta[x] >= 1.0) || !std::isfinite(a.theta[x]) || !(std::fabs(a.step[x]) <= 1e6) ||
            a.pairs[x] > kMaxRotPairs || at + a.pairs[x] > kMaxRotPairs)
            return MH3_ERR_PARAM;
        // theta^(-j / pairs) as exponentials (their argument, at most some 700, is within 2^-54: far below the bound): every
        // fourth, times the first four. Axes alike take the same.
        if (x == 0 || a.pairs[x] != a.pairs[x - 1] || a.theta[x] != a.theta[x - 1]) {
            const long double ln = a.pairs[x] ? logl((long double)a.theta[x]) / (long double)a.pairs[x] : 0.0L;
            long double low[4] = {1.0L, expl(-ln), expl(-2.0L * ln), expl(-3.0L * ln)};
            for (uint32_t j = 0; j < a.pairs[x]; j += 4) {
                const long double high = j ? expl(-(long double)j * ln) : 1.0L;
                for (uint32_t i = 0; i < 4; ++i)
                    power[j + i] = high * low[i];
            }
        }
        for (uint32_t j = 0; j < a.pairs[x]; ++j) {
            const long double f = (long double)a.step[x] * power[j] / 6.283185307179586476925286766559005768L;
            long double frac = f - (long double)int64_t(f); // |f| < 2^18
            frac += frac < 0.0L ? 1.0L : 0.0L;
            const long double fixed = frac * 0x1p64L + 0.5L;
            p.turn[at + j] = fixed >= 0x1p64L ? 0u : uint64_t(fixed);
        }
        at += a.pairs[x];
        if (x < 3u)
            p.end[x] = uint32_t(at);
    }
    for (uint32_t x = a.axes; x < 4u; ++x) {
        if (a.pairs[x] != 0)
            return MH3_ERR_PARAM;
        if (x < 3u)
            p.end[x] = uint32_t(at); // no pair lies on an axis past the last
    }
    if (half && at != half)
        return MH3_ERR_PARAM;
    p.half = uint32_t(at);
    return MH3_OK;
}

} // namespace host
} // namespace mh3

extern "C" int mh3_rotary_axes(const MH3AxesArgs* args, uint32_t rows, const int32_t* pos, float* cos_t, float* sin_t,
                               mh3_stream_t stream)
{
    using namespace mh3;
    RotaryParams p;
    if (const int rc = host::rotary_setup(args, pos, 0, p); rc != MH3_OK)
        return rc;
    if (rows == 0 || p.half == 0)
        return MH3_OK;
    if (rows >= (1u << 31))
        return MH3_ERR_SHAPE;
    if (!pos || !cos_t || !sin_t)
        return MH3_ERR_POINTER;
    if ((reinterpret_cast<uintptr_t>(pos) | reinterpret_cast<uintptr_t>(cos_t) | reinterpret_cast<uintptr_t>(sin_t)) &
        3u)
        return MH3_ERR_ALIGN;
    const uint64_t tab = uint64_t(rows) * p.half * 4u;
    const host::Span in[] = {{pos, uint64_t(rows) * p.axes * 4u}};
    const host::Span out[] = {{cos_t, tab}, {sin_t, tab}};
    if (host::any_overlap(in, out))
        return MH3_ERR_PARAM;
    // A launch's element index stays below 2^31.
    const uint32_t step = (1u << 31) / kMaxRotPairs / 2u;
    for (uint64_t first = 0; first < rows; first += step) {
        const uint32_t n = uint32_t(rows - first < step ? rows - first : step);
        const uint32_t blocks = (n * p.half + kRotaryThreads - 1u) / kRotaryThreads;
        hipLaunchKernelGGL(rotary_axes_kernel, dim3(blocks), dim3(kRotaryThreads), 0, static_cast<hipStream_t>(stream),
                           p, FastDiv::make(p.half), uint32_t(first), n, cos_t, sin_t);
        if (const int rc = host::check_launch(); rc != MH3_OK)
            return rc;
    }
    return MH3_OK;
}
