// Attention with shaped scores and log probabilities through the C++ host side (include/jitllm_hip.hpp): a prompt of two
// documents and decoding over each type of cache, then probabilities of what came out, against double precision over what
// the cache holds.  Built by __graft_entry__.build() beside the library; run by tests/test_cpp_scores.py.
//
//   scores_check --no-device    sizes and exception types only (no GPU needed)
//   scores_check                the check on device 0
#include <algorithm>
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
    std::printf("[cpp-scores] %s %s\n", name, ok ? "ok" : "FAILED");
    std::fflush(stdout);
    failed += !ok;
}

template <typename E, typename F>
bool throws(F f) {
    try {
        f();
    } catch (const E &) {
        return true;
    }
    return false;
}

void without_a_device() {
    report("no device", throws<Error>([] { Context ctx(0); }));
    report("bytes of a cache of fours", jl_kv_cache_bytes(JL_KV_Q4_0, 3, 2, 64, 16) == 2u * 3 * 2 * 16 * 36);
    report("workspace", jl_logprobs_workspace_bytes(32000, 64) > 0);
    report("no workspace", jl_logprobs_workspace_bytes(32000, 65) == 0 && jl_logprobs_workspace_bytes(0, 0) == 0);
}

void attention(jl_kv_type type) {
    Context ctx(0);
    const int requests = 2, blocks = 6, page = 16, pages = 12, rows = 64, heads = 6, kv = 2, dim = 64, width = heads * dim;
    const float scale = 0.125f, cap = 20.f;
    BlockTables tables(ctx, requests, blocks, pages, page, rows);
    PagedKvCache cache(ctx, type, pages, kv, dim, page);
    PagedAttention attention(ctx, heads, kv, dim);
    std::vector<float> slope(heads);
    for (int h = 0; h < heads; h++) slope[h] = std::ldexp(1.f, -h - 1);
    FloatArray slopes(ctx, slope);
    std::mt19937 random(9);
    std::normal_distribution<float> normal;
    double worst = 0;
    const std::vector<std::vector<std::int32_t>> fresh = {{40, 17}, {1, 1}, {1, 30}};
    for (const auto &step : fresh) {
        std::vector<float> x(static_cast<std::size_t>(rows) * width), k(static_cast<std::size_t>(rows) * kv * dim), v(k.size());
        for (auto *a : {&x, &k, &v})
            for (float &e : *a) e = 2 * normal(random);
        FloatArray q(ctx, x), keys(ctx, k), values(ctx, v), out(ctx, x.size());
        tables.plan(IntArray(ctx, step));
        const int used = step[0] + step[1];
        cache.append(FloatRows(keys, kv * dim), FloatRows(values, kv * dim), tables.positions, tables.slots, used);
        const auto positions = tables.positions.get(), of = tables.rowRequests.get(), table = tables.table.get();
        std::vector<std::int32_t> begin(rows), end(rows);
        for (int i = 0; i < used; i++) begin[i] = positions[i] >= 25 ? 25 : 0, end[i] = std::max(positions[i] + 1, of[i] == 0 ? 30 : 0);
        IntArray first(ctx, begin), ends(ctx, end);
        Scores scores;
        scores.cap = cap, scores.slopes = &slopes, scores.firstTokens = &first, scores.endTokens = &ends;
        attention.attend(cache, FloatRows(q, width), used, tables, FloatRows(out, width), scale, 0, scores);
        std::vector<std::int32_t> slots;                           // what the cache holds of every token
        for (int r = 0; r < requests; r++)
            for (int j = 0; j < blocks * page; j++) {
                const int p = table[r * blocks + j / page];
                slots.push_back(p < 0 ? -1 : p * page + j % page);
            }
        const std::int64_t all = static_cast<std::int64_t>(slots.size());
        FloatArray held_k(ctx, slots.size() * kv * dim), held_v(ctx, slots.size() * kv * dim);
        const IntArray where(ctx, slots);
        cache.read(where, all, held_k, held_v);
        ctx.sync();
        const auto hk = held_k.get(), hv = held_v.get(), got = out.get();
        for (int i = 0; i < used; i++)
            for (int h = 0; h < heads; h++) {
                std::vector<double> s, o(dim);
                double most = -1e300, sum = 0;
                auto at = [&](const std::vector<float> &a, int j) { return a.data() + (static_cast<std::size_t>(of[i] * blocks * page + j) * kv + h / (heads / kv)) * dim; };
                for (int j = begin[i]; j < end[i]; j++) {
                    double dot = 0;
                    for (int e = 0; e < dim; e++) dot += static_cast<double>(at(hk, j)[e]) * x[static_cast<std::size_t>(i) * width + h * dim + e];
                    s.push_back(cap * std::tanh(scale * dot / cap) - slope[h] * std::abs(positions[i] - j));
                    most = std::max(most, s.back());
                }
                for (std::size_t n = 0; n < s.size(); n++) {
                    const double w = std::exp(s[n] - most);
                    sum += w;
                    for (int e = 0; e < dim; e++) o[e] += w * at(hv, begin[i] + static_cast<int>(n))[e];
                }
                for (int e = 0; e < dim; e++) worst = std::max(worst, std::fabs(o[e] / sum - got[static_cast<std::size_t>(i) * width + h * dim + e]));
            }
    }
    // A score is off by (2 dim + 8) half steps of fp32, 2^-24, of scale sum |q k| -- about 0.125 * 64 * 1.6^2 = 20 -- so by
    // 1.6e-4, a weight by twice that, and values are at most about 10: 3.3e-3.
    std::printf("[cpp-scores] type %d, largest difference %.2e\n", type, worst);
    report("scored attention", worst < 5e-3);
    FloatArray short_slopes(ctx, 1);
    IntArray few(ctx, 1);
    Scores bad;
    bad.slopes = &short_slopes;
    FloatArray q(ctx, static_cast<std::size_t>(2 * width)), out(ctx, static_cast<std::size_t>(2 * width));
    report("slopes of other heads", throws<std::invalid_argument>([&] { attention.attend(cache, FloatRows(q, width), 2, tables, FloatRows(out, width), 1.f, 0, bad); }));
    bad.slopes = nullptr, bad.endTokens = &few;
    report("too few ends", throws<std::out_of_range>([&] { attention.attend(cache, FloatRows(q, width), 2, tables, FloatRows(out, width), 1.f, 0, bad); }));
    bad.endTokens = nullptr, bad.cap = -1.f;
    report("a cap below 0", throws<Error>([&] { attention.attend(cache, FloatRows(q, width), 2, tables, FloatRows(out, width), 1.f, 0, bad); }));
}

void probabilities() {
    Context ctx(0);
    const int rows = 5, vocab = 5003, top = 8;
    const float scale = 0.8f;
    std::mt19937 random(4);
    std::normal_distribution<float> normal;
    std::vector<float> x(static_cast<std::size_t>(rows) * vocab);
    for (float &e : x) e = 3 * normal(random);
    FloatArray logits(ctx, x), lp(ctx, rows), entropy(ctx, rows), of_top(ctx, rows * top);
    IntArray tokens(ctx, {0, 5002, 17, -1, 4000}), list(ctx, rows * top);
    LogProbabilities answers(ctx, vocab, top);
    answers.compute(FloatRows(logits, vocab), rows, &tokens, &lp, &entropy, &list, &of_top, 1, scale);
    ctx.sync();
    const auto got = lp.get(), h = entropy.get(), got_top = of_top.get();
    const auto t = tokens.get(), best = list.get();
    double worst = 0;
    bool listed = true;
    for (int r = 0; r < rows; r++) {
        const float *row = x.data() + static_cast<std::size_t>(r) * vocab;
        const double most = *std::max_element(row, row + vocab);
        double sum = 0, spread = 0;
        for (int i = 0; i < vocab; i++) sum += std::exp(scale * (row[i] - most));
        auto log_p = [&](int i) { return scale * (row[i] - most) - std::log(sum); };
        for (int i = 0; i < vocab; i++) spread -= std::exp(log_p(i)) * log_p(i);
        worst = std::max({worst, std::fabs(h[r] - spread), std::fabs(got[r] - (t[r] < 0 ? 0 : log_p(t[r])))});
        std::vector<int> order(vocab);
        for (int i = 0; i < vocab; i++) order[i] = i;
        std::stable_sort(order.begin(), order.end(), [&](int a, int b) { return row[a] > row[b]; });
        for (int k = 0; k < top; k++) {
            listed = listed && best[r * top + k] == order[k];
            worst = std::max(worst, std::fabs(got_top[r * top + k] - log_p(order[k])));
        }
    }
    // (n / 64 + 30) half steps of fp32 of a log p of up to 40: 110 x 6e-8 x 40
    std::printf("[cpp-scores] log probabilities, largest difference %.2e\n", worst);
    report("log probabilities", worst < 3e-4);
    report("the list", listed);
    report("a list of one half", throws<std::invalid_argument>([&] { answers.compute(FloatRows(logits, vocab), rows, &tokens, &lp, nullptr, &list); }));
    report("too few places", throws<std::out_of_range>([&] { answers.compute(FloatRows(logits, vocab), rows, &tokens, &lp, nullptr, nullptr, nullptr, 2); }));
    report("a list of 65", throws<std::invalid_argument>([&] { LogProbabilities(ctx, vocab, 65); }));
}

}  // namespace

int main(int argc, char **argv) {
    if (argc > 1 && !std::strcmp(argv[1], "--no-device")) {
        without_a_device();
    } else {
        for (jl_kv_type type : {JL_KV_F16, JL_KV_Q8_0, JL_KV_Q4_0}) attention(type);
        probabilities();
    }
    if (!failed) std::printf("[cpp-scores] all ok\n");
    return failed != 0;
}
