// The C++ mirror's attention over a context in two parts (include/fusor_hip.hpp) on a GPU: keys are all alike, so a row's result is the mean of the
// values that it sees.
#include <cmath>
#include <cstdio>
#include <cstring>
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

// a small number, exact in `dtype`, as its bits there; and back
static uint32_t bits_of(DType dtype, float x) {
    uint32_t u;
    memcpy(&u, &x, 4);
    if (dtype == DType::F32) return u;
    if (dtype == DType::BF16) return u >> 16;
    return x == 0.0f ? 0 : ((u >> 13) & 0x3ff) | (((u >> 23) - 127 + 15) << 10);
}
static float number_of(DType dtype, uint32_t bits) {
    const uint32_t u = dtype == DType::F32 ? bits : dtype == DType::BF16 ? bits << 16 : bits == 0 ? 0 : (bits & 0x3ff) << 13 | ((bits >> 10) + 127 - 15) << 23;
    float x;
    memcpy(&x, &u, 4);
    return x;
}
static Tensor<4> upload(const Device &d, DType dtype, const uint32_t (&shape)[4], const std::vector<float> &v) {
    std::vector<uint16_t> two;
    for (float x : v) {
        const uint32_t u = bits_of(dtype, x);
        two.push_back((uint16_t)u);
        if (dtype == DType::F32) two.push_back((uint16_t)(u >> 16));
    }
    return Tensor<4>::from_slice(d, dtype, shape, two.data());
}
static std::vector<float> download(const Tensor<4> &t) {
    const bool f32 = t.dtype() == DType::F32;
    std::vector<uint16_t> two(t.numel() * (f32 ? 2 : 1));
    t.to_host(two.data());
    std::vector<float> v;
    for (size_t i = 0; i < t.numel(); i++) v.push_back(number_of(t.dtype(), f32 ? two[2 * i] | (uint32_t)two[2 * i + 1] << 16 : two[i]));
    return v;
}

static Tensor<4> alike(const Device &d, DType dtype, uint32_t b, uint32_t h, uint32_t n, uint32_t dim, float x) {
    const uint32_t shape[4] = {b, h, n, dim};
    return upload(d, dtype, shape, std::vector<float>((size_t)b * h * n * dim, x));
}
// values that tell batch, head, row and dim: whole numbers, exact in every type
static float value(uint32_t b, uint32_t h, uint32_t row, uint32_t dim) { return (float)((5 * b + 3 * h + row + dim) % 8); }

static Tensor<4> values(const Device &d, DType dtype, uint32_t b, uint32_t h, uint32_t n, uint32_t dim, uint32_t from) {
    const uint32_t shape[4] = {b, h, n, dim};
    std::vector<float> v;
    for (uint32_t i = 0; i < b; i++)
        for (uint32_t j = 0; j < h; j++)
            for (uint32_t r = 0; r < n; r++)
                for (uint32_t e = 0; e < dim; e++) v.push_back(value(i, j, from + r, e));
    return upload(d, dtype, shape, v);
}

// rows of the batch behind a prefix of `rows` keys (0: none), each at the end of its cache
static void test_rows(const Device &d, DType dtype, uint32_t n, uint32_t rows, int64_t window, int64_t sinks) {
    const uint32_t B = 2, H = 4, Hkv = 2, own = 90, D = 64;
    const auto q = alike(d, dtype, B, H, n, D, 0.5f), k = alike(d, dtype, B, Hkv, own, D, 1.0f), v = values(d, dtype, B, Hkv, own, D, rows);
    const auto pk = alike(d, dtype, 1, Hkv, rows, D, 1.0f), pv = values(d, dtype, 1, Hkv, rows, D, 0);
    Context context;
    if (rows) context.prefix_k = &pk, context.prefix_v = &pv;
    context.q_pos_offset = rows + own - n, context.window = window, context.sinks = sinks;
    const auto got = download(flash_attention_context(q, k, v, 0.125f, context));
    // a 16-bit result is off by half a step of its type, of weights that add up to one: 2^-8 of 7 at most and as much again for the weights' rounding
    const double off = dtype == DType::F32 ? 1e-5 : 2 * 7.0 / 256;
    for (uint32_t b = 0; b < B; b++)
        for (uint32_t h = 0; h < H; h++)
            for (uint32_t r = 0; r < n; r++) {
                const int64_t at = context.q_pos_offset + r;
                double want = 0;
                int count = 0;
                for (int64_t j = 0; j < rows + own && j <= at; j++)
                    if (window == 0 || j + window > at || j < sinks) want += value(j < rows ? 0 : b, h / 2, (uint32_t)j, 9), count++;
                want /= count;
                const float x = got[((size_t)(b * H + h) * n + r) * D + 9];
                EXPECT(std::fabs(x - want) < off, "sequence %u head %u row %u: %f, want %f", b, h, r, x, want);
            }
}

template <typename F>
static void refused(const char *what, F call) {
    bool threw = false;
    try {
        call();
    } catch (const Panic &) {
        threw = true;
    }
    EXPECT(threw, "%s is refused", what);
}

int main() {
    try {
        Device d(0);
        for (DType dtype : {DType::F32, DType::F16, DType::BF16})
            for (uint32_t n : {1u, 3u, 40u}) {
                test_rows(d, dtype, n, 0, 30, 4);
                test_rows(d, dtype, n, 300, 0, 0);
                test_rows(d, dtype, n, 300, 100, 7);
            }
        const auto q = alike(d, DType::F32, 1, 4, 1, 64, 1.0f), k = alike(d, DType::F32, 1, 2, 9, 64, 1.0f), p = alike(d, DType::F32, 1, 2, 5, 64, 1.0f),
                   half = alike(d, DType::F16, 1, 2, 5, 64, 1.0f), two = alike(d, DType::F32, 2, 2, 5, 64, 1.0f);
        auto with = [&](const Tensor<4> *a, const Tensor<4> *b, int64_t sinks) {
            Context context;
            context.prefix_k = a, context.prefix_v = b, context.sinks = sinks;
            flash_attention_context(q, k, k, 1.0f, context);
        };
        refused("a prefix without values", [&] { with(&p, nullptr, 0); });
        refused("a prefix of another type", [&] { with(&half, &half, 0); });
        refused("a prefix for each sequence", [&] { with(&two, &two, 0); });
        refused("a negative number of first tokens", [&] { with(&p, &p, -1); });
    } catch (const std::exception &e) {
        printf("exception: %s\n", e.what());
        return 2;
    }
    printf("%s (%d failures)\n", failures ? "FAILED" : "ok", failures);
    return failures ? 1 : 0;
}
