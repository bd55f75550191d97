// The C++ mirror's 8-bit cache (include/fusor_hip.hpp) on a GPU, on numbers that the codes hold exactly.
#include <cmath>
#include <cstdio>
#include <vector>

#include "fusor_hip.hpp"

using namespace fusor_hip;

static int failures = 0;
#define EXPECT(cond, ...)                              \
    do {                                               \
        if (!(cond)) {                                 \
            failures++;                                \
            printf("%s:%d: ", __FILE__, __LINE__);     \
            printf(__VA_ARGS__);                       \
            printf("\n");                              \
        }                                              \
    } while (0)

static std::vector<float> host(const Tensor<4> &t) {
    std::vector<float> v(t.numel());
    t.to_host(v.data());
    return v;
}

// keys all equal, values (127 = the largest first, whole numbers behind): the output is the mean of the values that a row sees
static void test_steps(const Device &d, Q8Format format, uint32_t block) {
    const uint32_t H = 4, Hkv = 2, D = 64, limit = 64;
    Q8KvCache cache(d, 2, limit, format, block);
    const float top = format == Q8Format::INT8 ? 127.0f : 448.0f;
    uint32_t at = 0;
    for (uint32_t n : {5u, 1u, 1u, 20u, 1u}) {
        const uint32_t ks[4] = {1, Hkv, n, D}, qs[4] = {1, H, n, D};
        std::vector<float> k((size_t)Hkv * n * D, 1.0f), v(k.size()), q((size_t)H * n * D, 0.5f);
        for (uint32_t h = 0; h < Hkv; h++)
            for (uint32_t r = 0; r < n; r++)
                for (uint32_t e = 0; e < D; e++) v[(h * n + r) * D + e] = e == 0 ? top : (float)((at + r + e) % 8);
        auto tk = Tensor<4>::from_slice(d, DType::F32, ks, k.data()), tv = Tensor<4>::from_slice(d, DType::F32, ks, v.data());
        auto tq = Tensor<4>::from_slice(d, DType::F32, qs, q.data());
        auto all = cache.append(tk, tv);
        EXPECT(cache.current_seq_len() == at + n && all.first.shape()[2] == at + n, "length %llu", (unsigned long long)cache.current_seq_len());
        auto back = host(all.second.dequantize());
        for (uint32_t r = 0; r < at + n; r++) EXPECT(back[r * D + 3] == (float)((r + 3) % 8), "row %u reads back as %f", r, back[r * D + 3]);
        const fhip_analytic_mask causal{1, 1, (int64_t)at, 0};
        auto out = host(flash_attention(tq, all.first, all.second, 0.125f, std::nullopt, &causal));
        for (uint32_t h = 0; h < H; h++)
            for (uint32_t r = 0; r < n; r++) {
                double want = 0;
                for (uint32_t j = 0; j <= at + r; j++) want += (j + 9) % 8;
                want /= at + r + 1;
                const float got = out[(h * n + r) * D + 9];
                EXPECT(std::fabs(got - want) < 1e-5, "head %u row %u: %f, want %f", h, at + r, got, want);
            }
        at += n;
    }
    cache.reset();
    EXPECT(cache.current_seq_len() == 0, "reset");
}

static void test_refusals(const Device &d) {
    bool threw = false;
    try {
        Q8KvCache cache(d, 2, 16, Q8Format::INT8, 5);
    } catch (const Panic &) {
        threw = true;
    }
    EXPECT(threw, "blocks of 5 tokens are refused");
}

int main() {
    try {
        Device d(0);
        for (uint32_t block : {1u, 16u}) {
            test_steps(d, Q8Format::INT8, block);
            test_steps(d, Q8Format::E4M3, block);
        }
        test_refusals(d);
    } catch (const std::exception &e) {
        printf("exception: %s\n", e.what());
        return 2;
    }
    printf("%s (%d failures)\n", failures ? "FAILED" : "ok", failures);
    return failures ? 1 : 0;
}
