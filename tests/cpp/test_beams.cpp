// Beam search through the engine-side mirror (kvengine::generate_beams): fork,
// decode over shared blocks, choice and reorder as one run.  The search itself is
// repeated here in 64 bits from the same synthetic logits, and what every beam's
// layers gave at the end is compared with a session that processes that beam's
// tokens alone.  Needs a HIP device.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <numeric>
#include <vector>

#include "../../include/kvc.h"
#include "../../qwen3.5-9b-bfp8b-1xn300_amd/engine/kv_engine.h"

using kvengine::Beam;
using kvengine::StepOutput;

static int g_checks = 0, g_failed = 0;
static void check_at(bool ok, const char* expr, int line) {
    g_checks++;
    if (ok) return;
    g_failed++;
    fprintf(stderr, "    check failed (line %d): %s\n", line, expr);
}
#define CHECK(cond) check_at((cond), #cond, __LINE__)

static float bf16f(uint16_t b) {
    const uint32_t u = (uint32_t)b << 16;
    float f;
    memcpy(&f, &u, 4);
    return f;
}
static uint64_t mix64(uint64_t z) {
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ULL;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBULL;
    return z ^ (z >> 31);
}
static std::vector<int> random_tokens(int n, uint64_t seed) {
    std::vector<int> t(n);
    for (int i = 0; i < n; i++) t[i] = (int)(mix64(seed * 1000003 + (uint64_t)i) % kvengine::kVocab);
    return t;
}

static bool load(int n_ssm, int max_beams, int max_ctx = 1024) {
    kvengine::EngineConfig cfg;
    cfg.n_attn_layers = 3;
    cfg.n_ssm_layers = n_ssm;
    cfg.pool_blocks = 512;
    cfg.snapshot_slots = 4;
    cfg.max_sessions = 2;
    cfg.max_beams = max_beams;
    cfg.seed = 77;
    kvengine::set_engine_config(cfg);
    return kvengine::load_model_and_tokenizer("synthetic/beams", max_ctx);
}

// the engine's synthetic log probabilities behind a history, in 64 bits
static uint64_t token_hash(const std::vector<int>& t) {
    uint64_t h = 0x6B76656E67696E65ULL;
    const uint8_t* b = reinterpret_cast<const uint8_t*>(t.data());
    const size_t n = t.size() * sizeof(int);
    size_t i = 0;
    for (; i + 8 <= n; i += 8) {
        uint64_t w;
        memcpy(&w, b + i, 8);
        h = mix64(h ^ w);
    }
    for (; i < n; i++) h = mix64(h ^ b[i]);
    return h;
}
static std::vector<double> log_probabilities(const std::vector<int>& history) {
    std::vector<uint16_t> x(kvengine::kVocab);
    uint16_t* d = nullptr;
    CHECK(hipMalloc((void**)&d, x.size() * 2) == hipSuccess);
    CHECK(kvc_fill_normal_bf16(kvengine::context(), d, kvengine::kVocab, mix64(77 ^ token_hash(history)), 3.0f, nullptr) == KVC_OK);
    CHECK(hipMemcpy(x.data(), d, x.size() * 2, hipMemcpyDeviceToHost) == hipSuccess);
    CHECK(hipFree(d) == hipSuccess);
    std::vector<double> p(x.size());
    double sum = 0;
    for (size_t i = 0; i < x.size(); i++) sum += std::exp((p[i] = bf16f(x[i])));
    for (double& v : p) v -= std::log(sum);
    return p;
}

static std::vector<Beam> search(const std::vector<int>& prompt, int n_beams, int n_tokens) {
    struct Node {
        std::vector<int> tokens;
        double score;
    };
    std::vector<Node> beams(1, Node{{}, 0.0});
    for (int n = 0; n < n_tokens; n++) {
        std::vector<Node> all;
        for (const Node& b : beams) {
            std::vector<int> h(prompt);
            h.insert(h.end(), b.tokens.begin(), b.tokens.end());
            const std::vector<double> p = log_probabilities(h);
            std::vector<int> order(p.size());
            std::iota(order.begin(), order.end(), 0);
            std::partial_sort(order.begin(), order.begin() + n_beams, order.end(),
                              [&](int x, int y) { return p[x] != p[y] ? p[x] > p[y] : x < y; });
            for (int i = 0; i < n_beams; i++) {
                all.push_back(Node{b.tokens, b.score + p[order[i]]});
                all.back().tokens.push_back(order[i]);
            }
        }
        std::stable_sort(all.begin(), all.end(), [](const Node& x, const Node& y) { return x.score > y.score; });
        all.resize(n_beams);
        beams = all;
    }
    std::vector<Beam> out;
    for (const Node& b : beams) out.push_back(Beam{b.tokens, (float)b.score});
    return out;
}

// |a - b| / |b| over a row of bf16 values
static double relative(const std::vector<uint16_t>& a, const std::vector<uint16_t>& b) {
    double d = 0, n = 0;
    for (size_t i = 0; i < b.size(); i++) {
        const double x = bf16f(a[i]), y = bf16f(b[i]);
        d += (x - y) * (x - y);
        n += y * y;
    }
    return a.size() == b.size() ? std::sqrt(d / n) : 1e9;
}

static void run(int n_ssm, int n_prompt, int n_beams, int n_tokens) {
    printf("  %d beams of %d tokens behind %d, %d recurrent layers\n", n_beams, n_tokens, n_prompt, n_ssm);
    CHECK(load(n_ssm, 8));
    const std::vector<int> prompt = random_tokens(n_prompt, 5 + (uint64_t)n_prompt);
    std::vector<Beam> got;
    CHECK(kvengine::generate_beams(0, prompt, n_beams, n_tokens, got) == n_tokens);
    CHECK((int)got.size() == n_beams && kvengine::pos() == n_prompt && kvengine::cached_tokens() == prompt);
    const std::vector<Beam> want = search(prompt, n_beams, n_tokens);
    for (int i = 0; i < n_beams && i < (int)got.size(); i++) {
        CHECK(got[i].tokens == want[i].tokens);
        // n_tokens sums of a 32-bit score and a log sum that is off by at most 200 x 2^-24
        CHECK(std::fabs(got[i].score - want[i].score) <= n_tokens * (200 + std::fabs(want[i].score)) * 0x1p-24);
    }
    const std::vector<StepOutput> steps = kvengine::beam_outputs();
    CHECK((int)steps.size() == (n_tokens > 1 ? n_beams : 0));
    // each beam alone, from a fresh engine's empty cache
    for (int i = 0; i < (int)steps.size(); i++) {
        CHECK(load(n_ssm, 0));
        std::vector<int> t(prompt);
        t.insert(t.end(), got[i].tokens.begin(), got[i].tokens.end() - 1);
        CHECK(kvengine::generate(t, 0, 0.f, nullptr) == 0);
        const StepOutput& alone = kvengine::step_outputs().back();
        CHECK(steps[i].pos == alone.pos && steps[i].token == alone.token && alone.pos == (int)t.size() - 1);
        // two roundings of the output to bf16 (2^-8 each) and two of the weights, whose errors
        // average over the keys; a wrong parent's state or keys give differences of order one
        for (int l = 0; l < 3; l++) CHECK(relative(steps[i].out[l], alone.out[l]) <= 4 * 0x1p-8);
        for (int l = 0; l < n_ssm; l++) CHECK(relative(steps[i].ssm_out[l], alone.ssm_out[l]) <= 4 * 0x1p-8);
    }
}

static void test_refusals_and_room() {
    printf("  refusals, and sequences given back\n");
    std::vector<Beam> b(3);
    kvengine::shutdown();
    CHECK(kvengine::generate_beams(0, {1, 2}, 2, 2, b) == 0 && b.empty());
    CHECK(load(0, 0));
    CHECK(kvengine::generate_beams(0, {1, 2}, 1, 2, b) == 0);  // none configured
    CHECK(load(1, 4, 40));
    CHECK(kvengine::generate_beams(0, {1, 2}, 5, 2, b) == 0);
    CHECK(kvengine::generate_beams(0, {1, 2}, 0, 2, b) == 0);
    CHECK(kvengine::generate_beams(0, {1, 2}, 2, 0, b) == 0);
    CHECK(kvengine::generate_beams(0, {}, 2, 2, b) == 0);
    CHECK(kvengine::generate_beams(1, {1, 2}, 2, 2, b) == 0);  // not open
    for (int i = 0; i < 3; i++) CHECK(kvengine::generate_beams(0, random_tokens(9, 3), 4, 3, b) == 3 && b.size() == 4);
    CHECK(kvengine::create_session() == 1);
    // a context of 40 tokens: 25 of the prompt kept beside 15 new ones
    CHECK(kvengine::generate_beams(1, random_tokens(300, 4), 4, 15, b) == 15 && kvengine::pos(1) == 25);
    // the session goes on where its prompt ended
    int n = 0;
    CHECK(kvengine::generate_session(1, random_tokens(20, 4), 3, 0.f, [&](int, const std::string&) { return ++n > 0; }) == 3 && n == 3);
}

int main() {
    setvbuf(stdout, nullptr, _IOLBF, 0);
    int ndev = 0;
    if (hipGetDeviceCount(&ndev) != hipSuccess || ndev < 1) {
        fprintf(stderr, "no HIP device\n");
        return 2;
    }
    run(0, 70, 1, 3);
    run(0, 200, 5, 4);
    run(2, 33, 4, 5);
    run(1, 64, 8, 1);
    run(2, 250, 3, 9);  // past a snapshot boundary
    test_refusals_and_room();
    kvengine::shutdown();
    printf("%d of %d checks passed\n", g_checks - g_failed, g_checks);
    return g_failed ? 1 : 0;
}
