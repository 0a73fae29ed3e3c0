// The paged key-value cache through the C++ host side (include/jitllm_hip.hpp): requests of several lengths
// through plan -> append -> attend, step by step, against a double-precision history kept here.
// Built by __graft_entry__.build() beside the library; run by tests/test_cpp_kv.py.
//
//   kv_check --no-device    argument checks and exception types only (no GPU needed)
//   kv_check                the check on device 0
#include <cmath>
#include <cstdio>
#include <cstring>
#include <random>
#include <vector>

#include "jitllm_hip.hpp"

using namespace jitllm;

namespace {

int failed = 0;
void report(const char *name, bool ok) {
    std::printf("[cpp-kv] %s %s\n", name, ok ? "ok" : "FAILED");
    std::fflush(stdout);
    failed += !ok;
}

void without_a_device() {
    bool thrown = false;
    try {
        Context ctx(0);
    } catch (const Error &) {
        thrown = true;
    }
    report("no device", thrown);
    report("bytes of a cache", jl_kv_cache_bytes(JL_KV_F16, 3, 2, 64, 16) == 2u * 3 * 2 * 16 * 64 * 2);
    report("bytes of no cache", jl_kv_cache_bytes(JL_KV_F16, 3, 2, 65, 16) == 0);
}

void steps(jl_kv_type type, double tolerance) {
    Context ctx(0);
    const int requests = 3, blocks = 5, page = 16, pages = 12, rows = 48, heads = 6, kv = 2, dim = 64;
    BlockTables tables(ctx, requests, blocks, pages, page, rows);
    PagedKvCache cache(ctx, type, pages, kv, dim, page);
    PagedAttention attention(ctx, heads, kv, dim);
    std::vector<double> frequencies;
    for (int i = 0; i < dim / 2; i++) frequencies.push_back(std::pow(10000.0, -2.0 * i / dim));
    Rope rope(ctx, frequencies, JL_ROPE_HALVES);
    std::mt19937 random(7);
    std::normal_distribution<float> normal;
    const int width = (heads + 2 * kv) * dim;
    std::vector<std::vector<std::vector<double>>> keys(requests), values(requests);
    const std::vector<std::vector<std::int32_t>> fresh = {{17, 3, 0}, {1, 1, 25}, {1, -1, 1}, {1, 9, 1}};
    double worst = 0;
    for (const auto &step : fresh) {
        std::vector<float> x(static_cast<std::size_t>(rows) * width);
        for (float &v : x) v = normal(random);
        FloatArray qkv(ctx, x), out(ctx, static_cast<std::size_t>(rows) * heads * dim);
        int used = 0;
        for (int f : step) used += f > 0 ? f : 0;
        tables.plan(IntArray(ctx, step));
        const FloatRows q(qkv, width);
        cache.append(FloatRows(qkv, width, heads * dim), FloatRows(qkv, width, (heads + kv) * dim), tables.positions, tables.slots, used, &rope,
                     &q, heads);
        attention.attend(cache, q, used, tables, FloatRows(out, heads * dim), 0.125f);
        ctx.sync();
        const std::vector<float> got = out.get();
        int row = 0;
        for (int r = 0; r < requests; r++) {
            if (step[r] < 0) keys[r].clear(), values[r].clear();
            for (int i = 0; i < step[r]; i++, row++) {
                const int position = static_cast<int>(keys[r].size());
                std::vector<double> turned(x.begin() + static_cast<std::ptrdiff_t>(row) * width, x.begin() + static_cast<std::ptrdiff_t>(row + 1) * width);
                for (int h = 0; h < heads + kv; h++)
                    for (int p = 0; p < dim / 2; p++) {
                        double &a = turned[h * dim + p], &b = turned[h * dim + p + dim / 2];
                        const double c = std::cos(position * frequencies[p]), s = std::sin(position * frequencies[p]), a0 = a;
                        a = a0 * c - b * s, b = a0 * s + b * c;
                    }
                keys[r].emplace_back(turned.begin() + heads * dim, turned.begin() + (heads + kv) * dim);
                values[r].emplace_back(turned.begin() + (heads + kv) * dim, turned.end());
                for (int h = 0; h < heads; h++) {
                    std::vector<double> weight;
                    double total = 0;
                    for (const auto &k : keys[r]) {
                        double s = 0;
                        for (int d = 0; d < dim; d++) s += 0.125 * turned[h * dim + d] * k[h / (heads / kv) * dim + d];
                        weight.push_back(std::exp(s));
                        total += weight.back();
                    }
                    for (int d = 0; d < dim; d++) {
                        double want = 0;
                        for (std::size_t t = 0; t < weight.size(); t++) want += weight[t] / total * values[r][t][h / (heads / kv) * dim + d];
                        worst = std::max(worst, std::fabs(want - got[(static_cast<std::size_t>(row) * heads + h) * dim + d]));
                    }
                }
            }
        }
    }
    std::printf("worst difference %.2e\n", worst);
    report(type == JL_KV_F16 ? "steps over binary16" : "steps over 8-bit blocks", worst <= tolerance);
    report("lengths", tables.lengths.get() == std::vector<std::int32_t>({20, 9, 27}));
}

}  // namespace

int main(int argc, char **argv) {
    if (argc > 1 && std::strcmp(argv[1], "--no-device") == 0) {
        without_a_device();
    } else {
        // Values are normal: k and v are off by half a step of binary16 (2^-11 of at most 5), scores by 2^-11 of
        // 0.125 sum |q k| (about 5) and weights by twice that: 0.01 together.  8-bit blocks: 1 / 254 of a block's
        // largest (3), likewise: 0.15.
        steps(JL_KV_F16, 0.01);
        steps(JL_KV_Q8_0, 0.15);
    }
    if (!failed) std::printf("[cpp-kv] all ok\n");
    return failed ? 1 : 0;
}
