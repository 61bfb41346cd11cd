// Streams' kept rows in pages and attention over them through the C++ host layer (mako_h3.hpp) on the GPU, against
// restatements in double on the host, one "ok"/"FAIL" line a check and the number of failures as the exit status. The
// inputs are small; the kernels' own tests cover their sizes.
#include "mako_h3.hpp"

#include <algorithm>
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

constexpr uint32_t kHeads = 4, kKv = 2, kDim = 128;

// out[row][head] of softmax(q k^T / sqrt(128)) v over the keys that each row has, in double; the slack holds the rounding
// of P to bf16 and the scores' error.
struct Keys {
    std::vector<const uint16_t*> k, v; // a key's row of 128, head by head: [key * kKv + head]
};
void attend(const uint16_t* q, const Keys& keys, uint32_t head, double* want, double* slack)
{
    const uint32_t g = head / (kHeads / kKv);
    std::vector<double> p;
    double sum = 0;
    for (size_t j = 0; j < keys.k.size() / kKv; ++j) {
        double dot = 0;
        for (uint32_t x = 0; x < kDim; ++x)
            dot += of_bf16(q[x]) * of_bf16(keys.k[j * kKv + g][x]);
        p.push_back(std::exp(dot / std::sqrt(128.0)));
        sum += p.back();
    }
    for (uint32_t x = 0; x < kDim; ++x)
        for (size_t j = 0; j < p.size(); ++j) {
            const double t = p[j] / sum * of_bf16(keys.v[j * kKv + g][x]);
            want[x] += t, slack[x] += std::fabs(t) * (0x1p-8 + 0x1p-11);
        }
}

void window(const Kernels& k)
{
    std::printf("window\n");
    Rng r{1};
    constexpr uint32_t kRows = 90;
    const int32_t kWindow = 12;
    const std::vector<int32_t> off{0, 50, 85}, sinks{4, 0};
    const auto doff = on_device(off), dsinks = on_device(sinks);
    DeviceBuffer<int32_t> ranges(2 * kRows), first(2 * kRows);
    k.attn_window_ranges(kRows, kRows, 2, kWindow, true, doff.get(), doff.get(), dsinks.get(), ranges.get(), first.get());
    Dense d;
    d.heads = kHeads, d.kv_heads = kKv, d.q_rows = d.kv_rows = kRows;
    d.out = {kDim, kHeads * kDim};
    const auto hq = bf16_values(r, kHeads * kRows * kDim), hk = bf16_values(r, kKv * kRows * kDim),
               hv = bf16_values(r, kKv * kRows * kDim);
    const auto q = on_device(hq), kk = on_device(hk), v = on_device(hv);
    const uint64_t bytes = Kernels::flash_attn_128_workspace_bytes(d);
    DeviceBuffer<uint8_t> ws(bytes ? bytes : 1);
    DeviceBuffer<uint16_t> out(kHeads * kRows * kDim);
    Scores sc;
    sc.ranges = ranges.get(), sc.sinks = first.get();
    k.flash_attn_128(d, q.get(), kk.get(), v.get(), sc, ws.get(), bytes, out.get());
    std::vector<double> want(out.size(), 0.0), slack(out.size(), 0.0);
    for (int32_t i = 0; i < off[2]; ++i) {
        const int doc = i >= off[1];
        Keys keys;
        for (int32_t j = off[doc]; j <= i; ++j)
            if (j - off[doc] < sinks[doc] || j > i - kWindow)
                for (uint32_t h = 0; h < kKv; ++h)
                    keys.k.push_back(&hk[(h * kRows + j) * kDim]), keys.v.push_back(&hv[(h * kRows + j) * kDim]);
        for (uint32_t h = 0; h < kHeads; ++h)
            attend(&hq[(h * kRows + i) * kDim], keys, h, &want[(i * kHeads + h) * kDim], &slack[(i * kHeads + h) * kDim]);
    }
    compare("attention of two documents under a window and first rows", out.download(), want, slack);
}

// Three streams over a pool of 12 pages of 32 rows, kept apart as one tensor of keys and one of values.
void streams(const Kernels& k)
{
    std::printf("streams\n");
    Rng r{2};
    constexpr uint32_t kPage = 32, kCols = 6, kPages = 12, kNew = 9;
    PagesAttn d;
    d.table.streams = 3, d.table.cols = kCols, d.table.pages = kPages, d.table.page_rows = kPage;
    d.heads = kHeads, d.kv_heads = kKv, d.q_rows = kNew + 2; // two rows of no stream
    d.window = 20, d.zero_rest = true;
    const size_t page = size_t(kKv) * kPage * kDim;
    std::vector<int32_t> lengths{70, 33, 0};
    DeviceBuffer<uint16_t> kp(kPages * page), vp(kPages * page);
    kp.upload(std::vector<uint16_t>(kp.size(), 0x7fc0)), vp.upload(std::vector<uint16_t>(vp.size(), 0x7fc0));
    auto table = on_device(std::vector<int32_t>(3 * kCols, -1));
    auto refs = on_device(std::vector<int32_t>(kPages, 0));
    DeviceBuffer<int32_t> missing(1), used(1), map(kPages);
    const auto none = on_device(std::vector<int32_t>{0, 0, 0});
    k.pages_take(d.table, table.get(), refs.get(), none.get(), on_device(std::vector<int32_t>{3, 2, 0}).get(),
                 missing.get());
    check(missing.download()[0] == 0 && refs.download() == std::vector<int32_t>{1, 1, 1, 1, 1, 0, 0, 0, 0, 0, 0, 0},
          "five pages taken");

    // Rows of both streams, then stream 2 goes on from the first 40 of stream 0.
    PagesAttn kept = d;
    kept.q_rows = 103;
    const auto hk = bf16_values(r, kKv * 103 * kDim), hv = bf16_values(r, kKv * 103 * kDim);
    k.pages_write(kept, on_device(hk).get(), on_device(hv).get(), kp.get(), vp.get(), table.get(), none.get(),
                  on_device(std::vector<int32_t>{0, 70, 103, 103}).get());
    const std::vector<MH3Pool> pools{{kp.get(), page * 2, page * 2}, {vp.get(), page * 2, page * 2}};
    {
        auto next = on_device(std::vector<int32_t>(3 * kCols, -1));
        const uint64_t bytes = Kernels::pages_fork_workspace_bytes(d.table);
        DeviceBuffer<uint8_t> ws(bytes);
        k.pages_fork(d.table, pools, table.get(), refs.get(), on_device(std::vector<int32_t>{0, 1, 0}).get(),
                     on_device(std::vector<int32_t>{70, 33, 40}).get(), next.get(), ws.get(), bytes, missing.get());
        table.upload(next.download());
    }
    lengths[2] = 40;
    check(missing.download()[0] == 0 && refs.download() == std::vector<int32_t>{2, 1, 1, 1, 1, 1, 0, 0, 0, 0, 0, 0},
          "a fork shares its full page and copies the begun one");

    // New rows: one, five in a tree, and three in order; stream s's kept row j is row of hk kept_at(s) + j.
    const std::vector<int32_t> off{0, 1, 6, 9}, sinks{3, 0, 1}, parents{-1, -1, 0, 0, 1, 2, -1, 0, 1, -1, -1};
    const auto nq = bf16_values(r, kHeads * d.q_rows * kDim), nk = bf16_values(r, kKv * d.q_rows * kDim),
               nv = bf16_values(r, kKv * d.q_rows * kDim);
    const auto q = on_device(nq), kk = on_device(nk), v = on_device(nv);
    const auto doff = on_device(off), dsinks = on_device(sinks), dparents = on_device(parents);
    const uint64_t bytes = Kernels::flash_attn_pages_128_workspace_bytes(d);
    DeviceBuffer<uint8_t> ws(bytes ? bytes : 1);
    auto attention = [&](const std::string& what) {
        DeviceBuffer<uint16_t> out(kHeads * d.q_rows * kDim);
        out.upload(std::vector<uint16_t>(out.size(), 0x7fc0));
        k.flash_attn_pages_128(d, q.get(), kk.get(), v.get(), kp.get(), vp.get(), table.get(), on_device(lengths).get(),
                               doff.get(), dparents.get(), dsinks.get(), ws.get(), bytes, out.get());
        std::vector<double> want(out.size(), 0.0), slack(out.size(), 0.0);
        for (int32_t s = 0; s < 3; ++s)
            for (int32_t i = off[s]; i < off[s + 1]; ++i) {
                std::vector<int32_t> line{i}; // i and its ancestors
                while (parents[line.back()] >= 0)
                    line.push_back(off[s] + parents[line.back()]);
                const int32_t n = int32_t(line.size()), place = lengths[s] + n - 1, low = place - int32_t(d.window);
                Keys keys;
                const int32_t base = s == 1 ? 70 : 0;
                for (int32_t j = 0; j < lengths[s]; ++j)
                    if (j < sinks[s] || j > low)
                        for (uint32_t h = 0; h < kKv; ++h)
                            keys.k.push_back(&hk[(h * 103 + base + j) * kDim]),
                                keys.v.push_back(&hv[(h * 103 + base + j) * kDim]);
                for (int32_t a = 0; a < n; ++a)
                    if (place - a < sinks[s] || place - a > low)
                        for (uint32_t h = 0; h < kKv; ++h)
                            keys.k.push_back(&nk[(h * d.q_rows + line[a]) * kDim]),
                                keys.v.push_back(&nv[(h * d.q_rows + line[a]) * kDim]);
                for (uint32_t h = 0; h < kHeads; ++h) {
                    const size_t at = (h * d.q_rows + i) * kDim;
                    attend(&nq[at], keys, h, &want[at], &slack[at]);
                }
            }
        compare(what, out.download(), want, slack);
    };
    attention("trees over pages under a window");

    // Stream 0 ends, the others' pages move together, and one of them is copied.
    k.pages_free(d.table, table.get(), refs.get(), none.get(), on_device(std::vector<int32_t>{kCols, 0, 0}).get());
    lengths[0] = 0;
    {
        const uint64_t n = Kernels::pages_compact_workspace_bytes(d.table);
        DeviceBuffer<uint8_t> space(n);
        k.pages_compact(d.table, pools, table.get(), refs.get(), map.get(), space.get(), n, used.get());
    }
    check(used.download()[0] == 4 && refs.download() == std::vector<int32_t>{1, 1, 1, 1, 0, 0, 0, 0, 0, 0, 0, 0},
          "four pages stay, the first ones");
    attention("the same rows after a compaction");
    const std::vector<int32_t> src{1, 2}, dst{8, 11};
    k.pages_copy(pools, kPages, on_device(src).get(), on_device(dst).get(), 2);
    bool same = true;
    for (const auto& h : {kp.download(), vp.download()})
        for (int i = 0; i < 2; ++i)
            same = same && std::equal(&h[src[i] * page], &h[src[i] * page] + page, &h[dst[i] * page]);
    check(same, "copies of two pages");

    // Drafted rows 0, 2 and 4 of stream 1 were right: they become kept rows 33 .. 35.
    const std::vector<int32_t> right{1, 3, 5};
    k.pages_write(d, kk.get(), v.get(), kp.get(), vp.get(), table.get(), on_device(lengths).get(),
                  on_device(std::vector<int32_t>{0, 0, 3, 3}).get(), on_device(right).get(), 3);
    const auto t = table.download();
    const auto pages = kp.download();
    same = true;
    for (uint32_t i = 0; i < 3; ++i)
        for (uint32_t h = 0; h < kKv; ++h) {
            const uint16_t* at = &pages[t[kCols + 1] * page + (h * kPage + 1 + i) * kDim];
            same = same && std::equal(at, at + kDim, &nk[(h * d.q_rows + right[i]) * kDim]);
        }
    check(same, "accepted rows are kept");
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
    PagesAttn d;
    d.table.streams = 1, d.table.cols = 1, d.table.pages = 1, d.table.page_rows = 24;
    d.heads = d.kv_heads = d.q_rows = 1;
    check(throws([&] { (void)Kernels::flash_attn_pages_128_workspace_bytes(d); }), "pages not of 16 rows throw");
    Pages t;
    check(throws([&] { (void)Kernels::pages_fork_workspace_bytes(t); }), "no streams throw");
    DeviceBuffer<int32_t> a(16);
    check(throws([&] { k.attn_window_ranges(4, 4, 1, 0, true, a.get(), a.get(), nullptr, a.get(), a.get()); }),
          "an empty window throws");
    check(throws([&] { k.pages_copy({{a.get(), 24, 32}}, 1, a.get(), a.get() + 8, 1); }), "pages not of 16 bytes throw");
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
        window(k);
        streams(k);
        errors(k);
        k.finish();
    } catch (const std::exception& e) {
        std::printf("  FAIL %s\n", e.what());
        ++failures;
    }
    std::printf("%d failure%s\n", failures, failures == 1 ? "" : "s");
    return failures;
}
