// The dense path's operators through the C++ host layer (mako_h3.hpp) on the GPU, against restatements in double on the
// host, one "ok"/"FAIL" line a check and the number of failures as the exit status: positions on several axes, attention
// over packed documents, and products of 4-bit microscaled operands. The inputs and bounds are small; the kernels'
// own tests cover their sizes.
#include "mako_h3.hpp"

#include <cmath>
#include <cstdio>
#include <cstring>
#include <functional>
#include <string>
#include <vector>

namespace {

using namespace mako::h3;

int failures = 0;

void check(bool ok, const std::string& what)
{
    std::printf("  %-4s %s\n", ok ? "ok" : "FAIL", what.c_str());
    std::fflush(stdout);
    failures += !ok;
}

struct Rng {
    uint64_t s;
    uint64_t next()
    {
        uint64_t z = (s += 0x9E3779B97F4A7C15ull);
        z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
        return z ^ (z >> 27);
    }
    double operator()() { return double(next() >> 11) * 0x1.0p-52 - 1.0; } // [-1, 1)
};

double of_bf16(uint16_t b)
{
    const uint32_t u = uint32_t(b) << 16;
    float f;
    std::memcpy(&f, &u, 4);
    return f;
}
uint16_t to_bf16(double d)
{
    const float f = float(d);
    uint32_t u;
    std::memcpy(&u, &f, 4);
    return uint16_t((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}
std::vector<uint16_t> bf16_values(Rng& r, size_t n)
{
    std::vector<uint16_t> v(n);
    for (auto& x : v)
        x = to_bf16(r());
    return v;
}

template <class T>
DeviceBuffer<T> on_device(const std::vector<T>& v)
{
    DeviceBuffer<T> d(v.size());
    d.upload(v);
    return d;
}

// Every element of a bf16 result within 2^-8 of the wanted value and its slack.
void compare(const std::string& what, const std::vector<uint16_t>& got, const std::vector<double>& want,
             const std::vector<double>& slack)
{
    size_t bad = got.size() != want.size();
    for (size_t i = 0; i < want.size() && i < got.size(); ++i)
        bad += !(std::fabs(of_bf16(got[i]) - want[i]) <= 0x1p-8 * std::fabs(want[i]) + slack[i]);
    check(bad == 0, what + ": " + std::to_string(bad) + " of " + std::to_string(want.size()) + " beyond tolerance");
}

constexpr uint32_t kRows = 70, kHeads = 3, kDim = 256;

void axes(const Kernels& k)
{
    std::printf("axes\n");
    Rng r{1};
    const Axes ax{{{16, 10000.0, 0.25}, {8, 500.0, 1.0}, {8, 10000.0, 1.0}}};
    std::vector<int32_t> pos(kRows * 3);
    for (auto& p : pos)
        p = int32_t(r() * 5000);
    const auto dpos = on_device(pos);
    DeviceBuffer<float> cos_t(kRows * 32), sin_t(kRows * 32);
    k.rotary_axes(ax, kRows, dpos.get(), cos_t.get(), sin_t.get());
    const auto c = cos_t.download(), s = sin_t.download();
    size_t bad = 0;
    for (uint32_t row = 0; row < kRows; ++row)
        for (uint32_t i = 0; i < 32; ++i) {
            const uint32_t a = i < 16 ? 0 : i < 24 ? 1 : 2, j = i - (a == 0 ? 0 : a == 1 ? 16 : 24);
            const long double angle = pos[row * 3 + a] * (long double)ax.axes[a].step *
                                      powl(ax.axes[a].theta, -(long double)j / ax.axes[a].pairs);
            // 1e-7 is the tables' bound; the angles here are within 2^-40 of the exact ones.
            bad += std::fabs(double(c[row * 32 + i] - cosl(angle))) > 1.01e-7;
            bad += std::fabs(double(s[row * 32 + i] - sinl(angle))) > 1.01e-7;
        }
    check(bad == 0, "tables of three axes");

    const auto qkv = on_device(bf16_values(r, size_t(kRows) * 3 * kHeads * 128));
    Heads hd;
    hd.rows = kRows, hd.heads = kHeads, hd.rot = 64;
    const size_t n = size_t(kRows) * kHeads * 128;
    DeviceBuffer<uint16_t> a[3] = {DeviceBuffer<uint16_t>(n), DeviceBuffer<uint16_t>(n), DeviceBuffer<uint16_t>(n)};
    DeviceBuffer<uint16_t> b[3] = {DeviceBuffer<uint16_t>(n), DeviceBuffer<uint16_t>(n), DeviceBuffer<uint16_t>(n)};
    k.heads_partial_axes(hd, ax, qkv.get(), nullptr, nullptr, dpos.get(), nullptr, a[0].get(), a[1].get(), a[2].get());
    k.heads_partial(hd, qkv.get(), nullptr, nullptr, cos_t.get(), sin_t.get(), nullptr, b[0].get(), b[1].get(),
                    b[2].get());
    bool same = true;
    for (int t = 0; t < 3; ++t)
        same = same && a[t].download() == b[t].download();
    check(same, "heads_partial_axes is rotary_axes and heads_partial");
}

void attention(const Kernels& k)
{
    std::printf("attention\n");
    Rng r{2};
    Dense d;
    d.heads = 4, d.kv_heads = 2, d.q_rows = d.kv_rows = kRows;
    d.cap = 5.0f;
    d.out = {128, 4 * 128}; // [rows][heads * 128]
    const auto hq = bf16_values(r, 4 * kRows * 128), hk = bf16_values(r, 2 * kRows * 128),
               hv = bf16_values(r, 2 * kRows * 128);
    const auto q = on_device(hq), kk = on_device(hk), v = on_device(hv);
    const std::vector<int32_t> off{0, 20, kRows - 5}; // two causal documents, five rows of none
    const std::vector<float> slopes{0.5f, 0.1f, 0.0f, -0.1f};
    const auto doff = on_device(off);
    const auto dslopes = on_device(slopes);
    DeviceBuffer<int32_t> ranges(2 * kRows);
    k.attn_ranges(kRows, kRows, 2, true, doff.get(), doff.get(), nullptr, ranges.get());
    const auto rg = ranges.download();
    bool right = true;
    for (int32_t i = 0; i < int32_t(kRows); ++i) {
        const bool none = i >= off[2];
        const int32_t lo = i < off[1] ? 0 : off[1];
        right = right && (none ? rg[2 * i] >= rg[2 * i + 1] : rg[2 * i] == lo && rg[2 * i + 1] == i + 1);
    }
    check(right, "ranges of two causal documents");
    const uint64_t bytes = Kernels::flash_attn_128_workspace_bytes(d);
    DeviceBuffer<uint8_t> ws(bytes ? bytes : 1);
    DeviceBuffer<uint16_t> out(4 * kRows * 128);
    Scores sc;
    sc.ranges = ranges.get(), sc.slopes = dslopes.get();
    k.flash_attn_128(d, q.get(), kk.get(), v.get(), sc, ws.get(), bytes, out.get());
    std::vector<double> want(4 * kRows * 128, 0.0), slack(want.size(), 0.0);
    for (uint32_t h = 0; h < 4; ++h)
        for (uint32_t i = 0; i < kRows; ++i) {
            std::vector<double> p;
            double sum = 0;
            for (int32_t j = rg[2 * i]; j < rg[2 * i + 1]; ++j) {
                double dot = 0;
                for (uint32_t x = 0; x < 128; ++x)
                    dot += of_bf16(hq[(h * kRows + i) * 128 + x]) * of_bf16(hk[(h / 2 * kRows + j) * 128 + x]);
                p.push_back(std::exp(5.0 * std::tanh(dot / std::sqrt(128.0) / 5.0) - double(slopes[h]) * std::fabs(double(i) - j)));
                sum += p.back();
            }
            for (uint32_t x = 0; x < 128; ++x) {
                const size_t at = (size_t(i) * 4 + h) * 128 + x;
                for (size_t j = 0; j < p.size(); ++j) {
                    const double t = p[j] / sum * of_bf16(hv[(h / 2 * kRows + rg[2 * i] + j) * 128 + x]);
                    want[at] += t, slack[at] += std::fabs(t) * (0x1p-8 + 0x1p-11); // P's rounding, and the scores'
                }
            }
        }
    compare("attention under ranges, cap and bias", out.download(), want, slack);
}

// The values of a 4-bit matrix.
std::vector<double> values(const std::vector<uint8_t>& q, const std::vector<uint8_t>& scale, uint32_t rows, uint32_t cols)
{
    const double mags[8] = {0, 0.5, 1, 1.5, 2, 3, 4, 6};
    std::vector<double> v(size_t(rows) * cols);
    for (uint32_t r = 0; r < rows; ++r)
        for (uint32_t c = 0; c < cols; ++c) {
            const uint32_t b = q[(size_t(r) * cols + c) / 2] >> (c % 2 * 4) & 15u;
            const int e = int(scale[(size_t(c / 256) * rows + r) * 8 + c % 256 / 32]) - 127;
            v[size_t(r) * cols + c] = std::ldexp(b & 8 ? -mags[b & 7] : mags[b & 7], e);
        }
    return v;
}

void products(const Kernels& k)
{
    std::printf("products\n");
    Rng r{3};
    constexpr uint32_t kN = 512;
    const auto x = on_device(bf16_values(r, kRows * kDim)), w = on_device(bf16_values(r, kN * kDim));
    DeviceBuffer<uint8_t> xq(kRows * kDim / 2), xs(kRows * kDim / 32), wq(kN * kDim / 2), wsc(kN * kDim / 32);
    k.quant_rows_mx4(kRows, kDim, MH3_BF16, x.get(), xq.get(), xs.get());
    k.quant_rows_mx4(kN, kDim, MH3_BF16, w.get(), wq.get(), wsc.get());
    const auto hx = x.download();
    const auto xv = values(xq.download(), xs.download(), kRows, kDim), wv = values(wq.download(), wsc.download(), kN, kDim);
    size_t bad = 0;
    for (size_t b = 0; b < hx.size(); b += 32) {
        double top = 0;
        for (size_t i = 0; i < 32; ++i)
            top = std::max(top, std::fabs(of_bf16(hx[b + i])));
        // The block's maximum lies in [4, 8) steps of its power of two: at most one away, where it saturates at 6 two.
        const double unit = top > 0 ? std::ldexp(1.0, std::ilogb(top) - 2) : 0;
        for (size_t i = 0; i < 32; ++i)
            bad += !(std::fabs(of_bf16(hx[b + i]) - xv[b + i]) <= 2 * unit);
    }
    check(bad == 0, "4-bit rows stand for their matrix");
    std::vector<double> y(size_t(kRows) * kN), tol(y.size());
    for (uint32_t i = 0; i < kRows; ++i)
        for (uint32_t j = 0; j < kN; ++j) {
            double s = 0, m = 0;
            for (uint32_t c = 0; c < kDim; ++c) {
                const double t = xv[size_t(i) * kDim + c] * wv[size_t(j) * kDim + c];
                s += t, m += std::fabs(t);
            }
            y[size_t(i) * kN + j] = s, tol[size_t(i) * kN + j] = m * 18 * 0x1p-22;
        }
    DeviceBuffer<uint16_t> out(y.size());
    k.gemm_mx4(kRows, kN, kDim, xq.get(), xs.get(), wq.get(), wsc.get(), out.get());
    compare("gemm_mx4", out.download(), y, tol);

    std::vector<double> want(size_t(kRows) * kN / 2), slack(want.size());
    for (uint32_t i = 0; i < kRows; ++i)
        for (uint32_t j = 0; j < kN / 2; ++j) {
            const size_t g = size_t(i) * kN + j, u = g + kN / 2, at = size_t(i) * (kN / 2) + j;
            const double silu = y[g] / (1 + std::exp(-y[g]));
            want[at] = silu * y[u];
            slack[at] = 1.1 * tol[g] * (std::fabs(y[u]) + tol[u]) + std::fabs(silu) * tol[u] +
                        0x1p-21 * (1 + std::fabs(y[g])) * std::fabs(want[at]);
        }
    DeviceBuffer<uint16_t> act(want.size());
    k.fc1_swiglu_mx4(kRows, kN / 2, kDim, xq.get(), xs.get(), wq.get(), wsc.get(), act.get());
    compare("fc1_swiglu_mx4", act.download(), want, slack);

    std::vector<float> gate(kN), res(y.size());
    for (auto& g : gate)
        g = float(r());
    for (auto& v : res)
        v = float(of_bf16(to_bf16(r())));
    std::vector<uint16_t> res16(res.size());
    std::vector<double> sum(res.size()), near(res.size());
    for (size_t i = 0; i < res.size(); ++i) {
        res16[i] = to_bf16(res[i]);
        const double g = gate[i % kN];
        sum[i] = res[i] + g * y[i], near[i] = std::fabs(g) * (tol[i] + 0x1p-24 * std::fabs(y[i]));
    }
    const auto dgate = on_device(gate);
    Modulation m;
    m.gate = dgate.get();
    auto r16 = on_device(res16);
    auto r32 = on_device(res);
    k.gemm_mx4_gate_add(kRows, kN, kDim, xq.get(), xs.get(), wq.get(), wsc.get(), m, r16.get());
    k.gemm_mx4_gate_add(kRows, kN, kDim, xq.get(), xs.get(), wq.get(), wsc.get(), m, r32.get());
    compare("gemm_mx4_gate_add, bf16 residual", r16.download(), sum, near);
    const auto f = r32.download();
    bad = 0;
    for (size_t i = 0; i < f.size(); ++i)
        bad += !(std::fabs(double(f[i]) - sum[i]) <= 0x1p-23 * std::fabs(sum[i]) + near[i]);
    check(bad == 0, "gemm_mx4_gate_add, float residual");
}

void errors(const Kernels& k)
{
    std::printf("errors\n");
    auto throws = [](const std::function<void()>& f) {
        try {
            f();
        } catch (const std::runtime_error&) {
            return true;
        }
        return false;
    };
    DeviceBuffer<float> a(4096), b(4096);
    DeviceBuffer<int32_t> pos(256);
    check(throws([&] { k.rotary_axes(Axes{}, 4, pos.get(), a.get(), b.get()); }), "no axes throw");
    check(throws([&] { k.rotary_axes(Axes{{{16, 0.5, 1.0}}}, 4, pos.get(), a.get(), b.get()); }), "theta below 1 throws");
    Dense d;
    d.heads = 3, d.kv_heads = 2, d.q_rows = d.kv_rows = 4;
    check(throws([&] { (void)Kernels::flash_attn_128_workspace_bytes(d); }), "key heads that do not divide the heads throw");
    DeviceBuffer<uint8_t> q(4096), s(4096);
    check(throws([&] { k.quant_rows_mx4(2, 96, MH3_F32, a.get(), q.get(), s.get()); }), "columns not of 256 throw");
    DeviceBuffer<uint16_t> out(4096);
    check(throws([&] { k.gemm_mx4(2, 64, 256, q.get(), s.get(), q.get(), s.get(), out.get()); }), "64 columns throw");
}

} // namespace

int main()
{
    int devices = 0;
    if (hipGetDeviceCount(&devices) != hipSuccess || devices == 0) {
        std::printf("no GPU: skipped\n");
        return 77;
    }
    try {
        const Kernels k;
        axes(k);
        attention(k);
        products(k);
        errors(k);
        k.finish();
    } catch (const std::exception& e) {
        std::printf("  FAIL %s\n", e.what());
        ++failures;
    }
    std::printf("%d failure%s\n", failures, failures == 1 ? "" : "s");
    return failures;
}
