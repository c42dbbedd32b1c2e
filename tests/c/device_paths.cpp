// The host code of the paths that need a device, on tests/c/hip_stand_in.cpp, under AddressSanitizer and UndefinedBehaviorSanitizer: models
// loaded and closed many times; prompts in portions, recorded steps of single tokens, trees of drafted tokens, accepted paths kept, forks
// and the copies of shared pages, logits judged on the device; and what is left where a copy fails.  Kernels do not run: results are of no
// interest here.
//
//   device_paths ATTENTION_DIR STATEFUL_DIR
#include <cstdio>
#include <cstdlib>
#include <random>
#include <string>
#include <vector>

#include "celeg_amd.h"

extern "C" long hip_stand_in_launches();
extern "C" void hip_stand_in_fail_copy(long after);
extern "C" size_t hip_stand_in_memory();

static int failures = 0;
#define EXPECT(cond) do { if (!(cond)) { std::fprintf(stderr, "line %d: %s\n  last error: %s\n", __LINE__, #cond, celeg_last_error()); ++failures; } } while (0)

struct Loaded {
    celeg_model* model = nullptr;
    int vocab = 0, room = 0;
    explicit Loaded(const char* folder, int pages, const char* dtype = "float32") {
        celeg_engine_options o;
        celeg_engine_options_init(&o, sizeof o);
        o.dtype = dtype;
        o.max_active_requests = 4;
        o.max_batched_tokens = 64;
        o.page_tokens = 8;
        o.logical_kv_pages = pages;
        o.context = 128;
        EXPECT(celeg_model_create(folder, &o, &model) == CELEG_OK && model);
        const std::string text = celeg_model_describe(model);
        vocab = std::atoi(text.c_str() + text.find("\"logit_width\":") + 14);
    }
    ~Loaded() { celeg_model_destroy(model); }
    int open() { int32_t s = -1; EXPECT(celeg_model_open_slot(model, &s) == CELEG_OK); return s; }
    bool prepare(int slot, int start, int n) {
        int32_t ok = 0;
        return celeg_model_prepare(model, slot, start, n, &ok) == CELEG_OK && ok;
    }
    std::vector<int32_t> tokens(int n, std::mt19937& rng) {
        std::vector<int32_t> t;
        for (int i = 0; i < n; ++i) t.push_back(static_cast<int32_t>(rng() % 40));
        return t;
    }
    celeg_status step(int slot, int start, const std::vector<int32_t>& t, const std::vector<int32_t>& parents = {}) {
        const int32_t s = slot, at = start, n = static_cast<int32_t>(t.size()), wants = 1, want = n - 1;
        std::vector<float> logits(static_cast<size_t>(vocab));
        return celeg_model_step_tree(model, 1, &s, &at, &n, t.data(), parents.empty() ? nullptr : parents.data(), &wants, &want, logits.data(),
                                     logits.size());
    }
    void close(int slot) { EXPECT(celeg_model_close_slot(model, slot) == CELEG_OK); }
    void check() { EXPECT(celeg_model_check_cache(model) == CELEG_OK); }
};

static const std::vector<int32_t> TREE{-1, 0, 0, 1, 1, 2, -1, 6, 3, 8, 8};

// requests that are fed, decode, draft, keep, fork and are judged, in turn
static void requests(const char* folder, bool trees, unsigned seed, const char* dtype) {
    Loaded m(folder, 60, dtype);
    std::mt19937 rng(seed);
    std::vector<int> slots, length;
    for (int i = 0; i < 2; ++i) {
        slots.push_back(m.open());
        length.push_back(0);
        for (int n : {23, 9, 23}) {
            EXPECT(m.prepare(slots.back(), length.back(), n));
            EXPECT(m.step(slots.back(), length.back(), m.tokens(n, rng)) == CELEG_OK);
            length.back() += n;
        }
    }
    for (int turn = 0; turn < 12; ++turn) {
        const size_t i = rng() % slots.size();
        const int slot = slots[i];
        switch (turn % 4) {
            case 0: {                                    // a fork, which writes first or second
                int32_t other = -1;
                EXPECT(celeg_model_fork_slot(m.model, slot, length[i], &other) == CELEG_OK);
                if (!trees) EXPECT(celeg_model_fork_slot(m.model, slot, length[i] - 1, &other) != CELEG_OK);
                if (other >= 0) {
                    slots.push_back(other);
                    length.push_back(length[i]);
                }
                break;
            }
            case 1: {                                    // a tree and its accepted path, or a portion
                const int n = static_cast<int>(TREE.size());
                EXPECT(m.prepare(slot, length[i], n));
                EXPECT(m.step(slot, length[i], m.tokens(n, rng), trees ? TREE : std::vector<int32_t>()) == CELEG_OK);
                const int32_t kept[] = {length[i], length[i] + 1, length[i] + 3, length[i] + 8};
                const celeg_status s = celeg_model_keep(m.model, slot, length[i], kept, 4);
                EXPECT((s == CELEG_OK) == trees);
                length[i] += trees ? 4 : n;
                break;
            }
            case 2: {                                    // logits judged on the device
                const std::vector<int32_t> t = m.tokens(5, rng), targets = m.tokens(10, rng);
                const int32_t s = slot, at = length[i], n = 5, wants = 5, want[] = {0, 1, 2, 3, 4};
                std::vector<float> p(10), entropy(5), best(15);
                std::vector<int32_t> ranks(10), ids(15);
                EXPECT(m.prepare(slot, length[i], 5));
                EXPECT(celeg_model_step_logprobs(m.model, 1, &s, &at, &n, t.data(), nullptr, &wants, want, targets.data(), 2, 3, p.data(), ranks.data(),
                                                 entropy.data(), ids.data(), best.data()) == CELEG_OK);
                length[i] += 5;
                break;
            }
            default:                                     // single tokens: a recorded step
                for (int k = 0; k < 3; ++k) {
                    EXPECT(m.prepare(slot, length[i], 1));
                    EXPECT(m.step(slot, length[i]++, m.tokens(1, rng)) == CELEG_OK);
                }
        }
        m.check();
    }
    for (int slot : slots) {
        m.close(slot);
        m.check();
    }
}

// a copy that fails inside prepare() of a shared page, and inside keep(): nothing is lost, and the next call does what this one did not
static void failing_copies(const char* folder) {
    for (long after = 1; after <= 6; ++after) {
        Loaded m(folder, 12);
        std::mt19937 rng(7);
        const int a = m.open();
        EXPECT(m.prepare(a, 0, 20));
        EXPECT(m.step(a, 0, m.tokens(20, rng)) == CELEG_OK);
        int32_t b = -1;
        EXPECT(celeg_model_fork_slot(m.model, a, 20, &b) == CELEG_OK && b >= 0);
        hip_stand_in_fail_copy(after);
        (void)m.prepare(b, 20, 11);
        hip_stand_in_fail_copy(0);
        m.check();
        EXPECT(m.prepare(b, 20, 11));
        m.check();
        EXPECT(m.step(b, 20, m.tokens(11, rng), TREE) == CELEG_OK);
        EXPECT(celeg_model_fork_slot(m.model, b, 31, &b) == CELEG_OK && b >= 0);
        const int32_t kept[] = {20, 21, 23, 28};
        hip_stand_in_fail_copy(after);
        const celeg_status first = celeg_model_keep(m.model, b, 20, kept, 4);
        hip_stand_in_fail_copy(0);
        m.check();
        const long launched = hip_stand_in_launches();
        if (first != CELEG_OK) EXPECT(celeg_model_keep(m.model, b, 20, kept, 4) == CELEG_OK);
        // (the second copy is that of the block table's new entries: they come again, and then the move)
        if (after == 2) EXPECT(first != CELEG_OK && hip_stand_in_launches() == launched + 2);
        m.check();
        EXPECT(m.prepare(b, 24, 1));
        EXPECT(m.step(b, 24, m.tokens(1, rng)) == CELEG_OK);
        m.check();
    }
}

// lists of any length are launched (the stand-in ends the program at a launch that no GPU takes); kernels do not run, so nothing is read
static void long_lists() {
    void* const memory = reinterpret_cast<void*>(size_t(1) << 40);
    int32_t* const list = static_cast<int32_t*>(memory);
    celeg_paged_cache cache{sizeof(celeg_paged_cache), memory, memory, list, 1, 100, 2, 256, 16, 32, 32, 1, 8};
    EXPECT(celeg_copy_pages(&cache, list, list, 2147483647, nullptr) == CELEG_OK);
    EXPECT(celeg_move_tokens(&cache, 2147483646, list, list, list, list, 2147483647, list, nullptr) == CELEG_OK);
    for (int64_t vocab : {1, 1500, 8193, 100003, 1 << 24})
        for (int64_t rows : {1ll << 20, 1ll << 24, (1ll << 31) - 1}) {
            celeg_token_logprobs_args a{sizeof(celeg_token_logprobs_args), memory, rows, vocab, vocab, 0, 1, 1, list, static_cast<float*>(memory), list,
                                        static_cast<float*>(memory), list, static_cast<float*>(memory)};
            size_t bytes = 0;
            if (celeg_token_logprobs_workspace(&a, &bytes) != CELEG_OK) continue;      // (too many logits for a call)
            EXPECT(celeg_token_logprobs(&a, memory, bytes, nullptr) == CELEG_OK);
        }
    for (int32_t kv_heads : {1, 8, 256, 60000}) {
        cache.kv_heads = kv_heads;
        cache.n_layers = 1;
        for (int32_t nodes : {1, 40, 256}) {
            celeg_tree_attention_args a{sizeof(celeg_tree_attention_args), memory, kv_heads * 32ll, memory, 9, kv_heads, 65535 / nodes, 0, list, list, list,
                                        list, 1.f, 0, nodes, 100};
            size_t bytes = 0;
            EXPECT(celeg_tree_attention_workspace(&a, &cache, &bytes) == CELEG_OK);
            EXPECT(celeg_tree_attention(&a, &cache, memory, bytes, nullptr) == CELEG_OK);
        }
    }
}

int main(int argc, char** argv) {
    if (argc != 3) return 2;
    requests(argv[1], true, 0, "float32");
    const size_t memory = hip_stand_in_memory();
    for (unsigned i = 1; i <= 12; ++i) requests(argv[1 + i % 2], i % 2 == 0, i, i % 4 < 2 ? "float32" : "bfloat16");
    failing_copies(argv[1]);
    long_lists();
    EXPECT(hip_stand_in_memory() == memory);             // closed models leave nothing
    EXPECT(hip_stand_in_launches() > 1000);
    std::printf("failures: %d\n", failures);
    return failures != 0;
}
