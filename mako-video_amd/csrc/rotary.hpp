// Rotary angles from integer positions on several axes, shared by rotary_axes and heads_partial_axes.
//
// The angle of pair j of axis a at position p is p step[a] theta[a]^(-j / pairs[a]) radians. In turns that is p F with
// F = step theta^(-j / pairs) / 2 pi, and only its fraction matters, so F is held as a 64-bit fixed-point fraction of a
// turn and p F is one wrapping 64-bit multiplication: exact modulo a turn but for F's own rounding (2^-65 a position,
// 2^-34 of a turn at the largest int32 position). A float product would lose the whole angle by position 2^24.
#pragma once

#include "mh3_common.hpp"

namespace mh3 {

constexpr uint32_t kMaxRotPairs = 64; // half a head of 128 values

struct RotaryParams {
    const int32_t* pos;      // [rows][axes]
    uint32_t axes, half;     // half: pairs in all
    uint32_t end[3];         // the first pair after axes 0, 1 and 2
    uint64_t turn[kMaxRotPairs]; // F of each pair
};

// cos and sin of t / 2^64 turns. The quarter turn nearest to it is taken off exactly; the rest lies within an eighth of
// a turn, where both Taylor series are cut below 2^-29, and its rounding to float and that of 2 pi are carried as a
// correction (cos and sin together within 1.5 float ulp of the exact values).
__device__ __forceinline__ void turn_cos_sin(uint64_t t, float& c, float& s)
{
    const uint64_t q = (t + (uint64_t(1) << 61)) >> 62;
    const int64_t r = int64_t(t - (q << 62)); // [-2^61, 2^61)
    // r / 2^64 in two floats: its upper 24 bits or so, and what they leave.
    const float hi = __ll2float_rn(r), lo = float(r - int64_t(hi)); // |hi| <= 2^61: the cast back is exact
    constexpr float kPi2Hi = 0x1.921fb6p+2f, kPi2Lo = -0x1.777a5cp-23f; // 2 pi
    const float y = hi * 0x1p-64f, yl = lo * 0x1p-64f;
    const float x = y * kPi2Hi;
    const float d = fmaf(y, kPi2Hi, -x) + fmaf(y, kPi2Lo, yl * kPi2Hi);
    const float z = x * x;
    float ps = fmaf(z, 1.0f / 362880.0f, -1.0f / 5040.0f);
    ps = fmaf(ps, z, 1.0f / 120.0f);
    ps = fmaf(ps, z, -1.0f / 6.0f);
    float pc = fmaf(z, -1.0f / 3628800.0f, 1.0f / 40320.0f);
    pc = fmaf(pc, z, -1.0f / 720.0f);
    pc = fmaf(pc, z, 1.0f / 24.0f);
    pc = fmaf(pc, z, -0.5f);
    const float sn0 = fmaf(x * z, ps, x), cs0 = fmaf(pc, z, 1.0f);
    const float sn = fmaf(cs0, d, sn0), cs = fmaf(-sn0, d, cs0);
    const uint32_t quarter = uint32_t(q) & 3u;
    const float a = quarter & 1u ? sn : cs, b = quarter & 1u ? cs : sn;
    c = (quarter == 1u || quarter == 2u) ? -a : a;
    s = quarter >= 2u ? -b : b;
}

// cos and sin of pair i (below half) at row `row`'s positions.
__device__ __forceinline__ void row_cos_sin(const RotaryParams& p, uint64_t row, uint32_t i, float& c, float& s)
{
    const uint32_t axis = uint32_t(i >= p.end[0]) + uint32_t(i >= p.end[1]) + uint32_t(i >= p.end[2]);
    const int64_t at = p.pos[row * p.axes + axis];
    turn_cos_sin(uint64_t(at) * p.turn[i], c, s);
}

namespace host {
// The checks of the axes and the parameters that they give (pos is set to what is passed; it may be null only where
// there is no pair). `half`: the pairs that the axes must sum up to, or 0 for any.
int rotary_setup(const MH3AxesArgs* args, const int32_t* pos, uint32_t half, RotaryParams& p);
} // namespace host

} // namespace mh3
