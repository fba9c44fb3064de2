// PagedKVCache and the launchers of paged_kernels.hpp against sums in double: a batch of
// three sequences grows token by token over four-row pages, one forks, one is cut, the pool
// is compacted; a 4-bit product against its own codes.  Prints PASS/FAIL lines and exits with
// the number of failures.
#include <cmath>
#include <cstdio>
#include <cstring>
#include <random>
#include <vector>

#include "../../include/paged_kv_cache.hpp"

namespace {

int g_failures = 0;
void report(const char* name, bool ok) {
    std::printf("%s %s\n", ok ? "PASS" : "FAIL", name);
    std::fflush(stdout);
    if (!ok) ++g_failures;
}

struct Config {
    size_t num_layers = 2, num_heads = 4, num_kv_heads = 2, head_dim = 64;
};
constexpr size_t kSeqs = 3, kHeads = 4, kKv = 2, kDim = 64, kQ = kHeads * kDim, kKvDim = kKv * kDim;

float to_float(uint16_t b) {
    _Float16 v;
    std::memcpy(&v, &b, 2);
    return (float)v;
}
uint16_t to_half(float x) {
    const _Float16 v = (_Float16)x;
    uint16_t b;
    std::memcpy(&b, &v, 2);
    return b;
}

template <class T>
struct Device {
    T* p = nullptr;
    size_t n;
    explicit Device(size_t count) : n(count) { HIP_CHECK(hipMalloc(&p, n * sizeof(T))); }
    Device(const std::vector<T>& v) : Device(v.size()) { put(v); }
    ~Device() { (void)hipFree(p); }
    void put(const std::vector<T>& v) {
        HIP_CHECK(hipMemcpy(p, v.data(), n * sizeof(T), hipMemcpyHostToDevice));
    }
    std::vector<T> get() const {
        std::vector<T> v(n);
        HIP_CHECK(hipMemcpy(v.data(), p, n * sizeof(T), hipMemcpyDeviceToHost));
        return v;
    }
    __half* half() const { return reinterpret_cast<__half*>(p); }
};

std::mt19937 g_rng(1);
std::vector<uint16_t> random_half(size_t n) {
    std::normal_distribution<float> d(0.f, 1.f);
    std::vector<uint16_t> v(n);
    for (auto& x : v) x = to_half(d(g_rng));
    return v;
}

using Rows = std::vector<std::vector<uint16_t>>;  // cached rows of one sequence and layer

// largest error over its bound: half a step of fp16, weights in fp16, fp32 sums
double attention_error(const uint16_t* q, const Rows& k, const Rows& v, const uint16_t* out) {
    double worst = 0;
    for (size_t h = 0; h < kHeads; ++h) {
        const size_t at = h / (kHeads / kKv) * kDim;
        std::vector<double> s(k.size());
        double most = -1e300, sum = 0;
        for (size_t j = 0; j < k.size(); ++j) {
            for (size_t d = 0; d < kDim; ++d)
                s[j] += (double)to_float(q[h * kDim + d]) * to_float(k[j][at + d]);
            s[j] /= 8.0;
            most = std::max(most, s[j]);
        }
        for (auto& x : s) sum += x = std::exp(x - most);
        for (size_t d = 0; d < kDim; ++d) {
            double o = 0, size = 0;
            for (size_t j = 0; j < v.size(); ++j) {
                o += s[j] / sum * to_float(v[j][at + d]);
                size += s[j] / sum * std::fabs(to_float(v[j][at + d]));
            }
            const double bound = 2.5 * 0x1p-11 * size + 0x1p-11 * std::fabs(o) + 0x1p-24;
            worst = std::max(worst, std::fabs(to_float(out[h * kDim + d]) - o) / bound);
        }
    }
    return worst;
}

}  // namespace

int main() {
    const Config config;
    const size_t layers = config.num_layers;
    PagedKVCache cache(config, 12, 4, kSeqs, 6);
    std::vector<Rows> k(kSeqs * layers), v(kSeqs * layers);
    std::vector<int32_t> lens(kSeqs, 0);
    Device<uint16_t> q(kSeqs * kQ), kn(kSeqs * kKvDim), vn(kSeqs * kKvDim), out(kSeqs * kQ);
    Device<int32_t> grow(kSeqs), pos(kSeqs);
    double worst = 0;
    bool status_ok = true;
    auto step = [&](const std::vector<int32_t>& which) {
        std::vector<int32_t> p(kSeqs);
        for (size_t b = 0; b < kSeqs; ++b) p[b] = which[b] ? lens[b] : -1;
        grow.put(which);
        pos.put(p);
        cache.grow(grow.p);
        for (size_t l = 0; l < layers; ++l) {
            const auto hq = random_half(kSeqs * kQ), hk = random_half(kSeqs * kKvDim),
                       hv = random_half(kSeqs * kKvDim);
            q.put(hq);
            kn.put(hk);
            vn.put(hv);
            cache.append(l, q.half(), kn.half(), vn.half(), nullptr, nullptr, nullptr, nullptr,
                         pos.p, kSeqs, 64, 0, 0, false);
            cache.decode(l, q.half(), out.half());
            HIP_CHECK(hipDeviceSynchronize());
            const auto o = out.get();
            for (size_t b = 0; b < kSeqs; ++b) {
                if (!which[b]) continue;
                auto row = [&](const std::vector<uint16_t>& x) {
                    return std::vector<uint16_t>(x.begin() + b * kKvDim,
                                                 x.begin() + (b + 1) * kKvDim);
                };
                k[b * layers + l].push_back(row(hk));
                v[b * layers + l].push_back(row(hv));
                worst = std::max(worst, attention_error(&hq[b * kQ], k[b * layers + l],
                                                        v[b * layers + l], &o[b * kQ]));
            }
        }
        int32_t lacks[2];
        HIP_CHECK(hipMemcpy(lacks, cache.status(), sizeof lacks, hipMemcpyDeviceToHost));
        status_ok = status_ok && lacks[0] == 0 && lacks[1] == 0;
        for (size_t b = 0; b < kSeqs; ++b) lens[b] += which[b];
    };
    for (int i = 0; i < 6; ++i) step({1, i % 2, 0});
    report("steps of a batch with padding", worst <= 1.0 && status_ok);
    worst = 0;
    Device<int32_t> parents(std::vector<int32_t>{-1, -1, 0});
    cache.fork(parents.p);
    for (size_t l = 0; l < layers; ++l) {
        k[2 * layers + l] = k[l];
        v[2 * layers + l] = v[l];
    }
    lens[2] = lens[0];
    for (int i = 0; i < 3; ++i) step({1, 0, 1});
    report("a fork and its parent go different ways", worst <= 1.0 && status_ok);
    worst = 0;
    Device<int32_t> keep(std::vector<int32_t>{5, 0, -1});
    cache.free(keep.p);
    cache.compact();
    for (size_t l = 0; l < layers; ++l) {
        k[l].resize(5);
        v[l].resize(5);
        k[layers + l].clear();
        v[layers + l].clear();
    }
    lens[0] = 5;
    lens[1] = 0;
    int32_t used = 0;
    HIP_CHECK(hipMemcpy(&used, cache.num_used(), 4, hipMemcpyDeviceToHost));
    step({1, 1, 1});
    // pages in use after the cut: sequence 0 two (one shared with the fork), the fork three
    report("cut, compaction and new tokens", worst <= 1.0 && status_ok && used == 4);

    // a pool that runs short says so and keeps the state
    grow.put({16, 16, 14});
    cache.grow(grow.p);
    HIP_CHECK(hipDeviceSynchronize());
    int32_t now[3], lacks[2];
    HIP_CHECK(hipMemcpy(lacks, cache.status(), sizeof lacks, hipMemcpyDeviceToHost));
    HIP_CHECK(hipMemcpy(now, cache.seq_lens(), sizeof now, hipMemcpyDeviceToHost));
    report("a pool that runs short", lacks[0] > 0 && lacks[1] == 0 && now[0] == lens[0] &&
                                         now[1] == lens[1] && now[2] == lens[2]);

    // 4-bit product: codes and scales as documented, two tokens with a residual
    constexpr size_t N = 40, K = 200, G = 64;
    const auto w = random_half(N * K), x = random_half(2 * K), r = random_half(2 * N);
    Device<uint16_t> dw(w), dx(x), dr(r), dy(2 * N),
        ds(attn_w4_scale_count(N, K, G));
    Device<uint32_t> dp(attn_w4_weight_bytes(N, K) / 4);
    launch_w4_pack(dw.half(), dp.p, ds.half(), N, K, G);
    launch_w4_matvec(dx.half(), dy.half(), dp.p, ds.half(), dr.half(), 2, K, N, G);
    HIP_CHECK(hipDeviceSynchronize());
    const auto packed = dp.get();
    const auto scales = ds.get(), y = dy.get();
    bool codes_ok = true, y_ok = true;
    for (size_t t = 0; t < 2; ++t)
        for (size_t n = 0; n < N; ++n) {
            double sum = to_float(r[t * N + n]), size = std::fabs(sum);
            for (size_t c = 0; c < K; ++c) {
                const size_t tile = n / 16 * ((K + 127) / 128) + c / 128;
                const size_t word = 4 * (16 * (c % 32 / 8) + n % 16) + c % 128 / 32;
                const size_t e = c % 8, bit = 4 * (e / 2) + 16 * (e % 2);
                const int code = (int)(packed[tile * 256 + word] >> bit & 15u) - 8;
                const double s = to_float(scales[c / G * 48 + n]);
                // rounded to nearest: within half a step
                codes_ok = codes_ok && std::fabs(code * s - to_float(w[n * K + c])) <= 0.5001 * s;
                sum += code * s * to_float(x[t * K + c]);
                size += std::fabs(code * s * to_float(x[t * K + c]));
            }
            y_ok = y_ok && std::fabs(to_float(y[t * N + n]) - sum) <=
                               0x1p-11 * std::fabs(sum) + (K + 16) * 0x1p-24 * size + 0x1p-24;
        }
    report("4-bit codes are within half a step", codes_ok);
    report("4-bit product", y_ok);

    bool thrown = false;
    try {
        launch_w4_matvec(dx.half(), dy.half(), dp.p, ds.half(), nullptr, 1, K, N, 20);
    } catch (const std::runtime_error& e) {
        thrown = std::strstr(e.what(), "launch_w4_matvec") != nullptr;
    }
    report("a refused call throws", thrown);
    return g_failures;
}
