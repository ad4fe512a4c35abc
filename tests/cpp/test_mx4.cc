// test_mx4.cc -- C++ client of the 4-bit microscaled matrices of include/RandBLAS.hh (host and device
// arrays). Every number is a small integer or an E2M1 value under a power of two, so results are exact.
// Built and run by tests/test_gpu_mx4.py; prints "ALL PASSED" on success.
#include <RandBLAS.hh>
#include <hip/hip_runtime_api.h>

#include <cmath>
#include <cstdio>
#include <cstring>
#include <vector>

using blas::Layout;
using blas::Op;
using RandBLAS::ext::MX4Matrix;
using RandBLAS::ext::bf16;
using RandBLAS::ext::f16;
using RandBLAS::ext::mx4_dequantize;
using RandBLAS::ext::mx4_quantize;
using RandBLAS::ext::mxmm;

static int g_fail = 0;
#define CHECK(c)                                                       \
    do {                                                               \
        if (!(c)) {                                                    \
            std::printf("FAILED %s:%d: %s\n", __FILE__, __LINE__, #c); \
            g_fail++;                                                  \
        }                                                              \
    } while (0)

// values that a block of scale 1 holds exactly (with a 4 or a 6 in each block)
static std::vector<float> exact(int64_t rows, int64_t cols, unsigned key) {
    static const float grid[16] = {0, .5f, 1, 1.5f, 2, 3, 4, 6, 0, -.5f, -1, -1.5f, -2, -3, -4, -6};
    std::vector<float> a(rows * cols);
    unsigned x = key * 2654435761u + 1;
    for (int64_t i = 0; i < rows * cols; ++i) {
        x = x * 1664525u + 1013904223u;
        a[i] = i % cols % 32 == 0 ? 6.f : grid[x >> 28];
    }
    return a;
}

template <typename T> static T make(float v);
template <> float make<float>(float v) { return v; }
template <> double make<double>(float v) { return v; }
template <> bf16 make<bf16>(float v) {
    uint32_t u;
    std::memcpy(&u, &v, 4);
    return bf16{(uint16_t)(u >> 16)};
}
static float value(float v) { return v; }
static float value(double v) { return (float)v; }
static float value(bf16 v) {
    const uint32_t u = (uint32_t)v.bits << 16;
    float f;
    std::memcpy(&f, &u, 4);
    return f;
}

template <typename T> static void there_and_back() {
    const int64_t rows = 21, cols = 70;
    const std::vector<float> a = exact(rows, cols, 3);
    std::vector<T> A(rows * cols), B(cols * rows), W(5 * 38);
    for (size_t i = 0; i < A.size(); ++i) A[i] = make<T>(a[i]);
    MX4Matrix Q(rows, cols);
    mx4_quantize(Layout::RowMajor, Op::NoTrans, rows, cols, A.data(), cols, Q);
    CHECK(Q.scales[0] == 127 && Q.ld_codes == 48 && Q.ld_scales == 3);
    mx4_dequantize(Layout::ColMajor, Op::NoTrans, rows, cols, Q, 0, 0, B.data(), rows);
    mx4_dequantize(Layout::RowMajor, Op::NoTrans, 5, 38, Q, 2, 32, W.data(), 38);
    bool same = true;
    for (int64_t i = 0; i < rows; ++i)
        for (int64_t j = 0; j < cols; ++j) same = same && value(B[i + j * rows]) == a[i * cols + j];
    for (int64_t i = 0; i < 5; ++i)
        for (int64_t j = 0; j < 38; ++j) same = same && value(W[i * 38 + j]) == a[(i + 2) * cols + j + 32];
    CHECK(same);
}

template <typename T> static void products() {
    const int64_t m = 18, n = 25, k = 70;
    const std::vector<float> a = exact(m, k, 5), b = exact(n, k, 6);
    std::vector<T> A(m * k), B(n * k), C(m * n);
    for (size_t i = 0; i < A.size(); ++i) A[i] = make<T>(std::trunc(a[i] / 3));
    for (size_t i = 0; i < B.size(); ++i) B[i] = make<T>(std::trunc(b[i] / 3));
    MX4Matrix QA(m, k), QB(n, k);
    mx4_quantize(Layout::RowMajor, Op::NoTrans, m, k, a.data(), k, QA);
    mx4_quantize(Layout::RowMajor, Op::NoTrans, n, k, b.data(), k, QB);
    for (int which = 0; which < 3; ++which) {
        const float beta = which == 1 ? 2.f : 0.f;
        for (T &c : C) c = make<T>(1.f);
        if (which == 0) mxmm(Layout::RowMajor, Op::NoTrans, Op::Trans, m, n, k, 1.f, A.data(), k, QB, 0, 0, beta, C.data(), n);
        else if (which == 1) mxmm(Layout::RowMajor, Op::NoTrans, Op::Trans, m, n, k, 1.f, QA, 0, 0, B.data(), k, beta, C.data(), n);
        else mxmm(Layout::RowMajor, Op::NoTrans, Op::Trans, m, n, k, 1.f, QA, 0, 0, QB, 0, 0, beta, C.data(), n);
        bool same = true;
        for (int64_t i = 0; i < m; ++i)
            for (int64_t j = 0; j < n; ++j) {
                float sum = beta;
                for (int64_t q = 0; q < k; ++q)
                    sum += (which == 0 ? value(A[i * k + q]) : a[i * k + q]) * (which == 1 ? value(B[j * k + q]) : b[j * k + q]);
                const float got = value(C[i * n + j]);   // sums are exact; a 16-bit result is rounded once
                same = same && std::fabs(got - sum) <= (sizeof(T) == 2 ? std::ldexp(std::fabs(sum), -8) : 0.f);
            }
        CHECK(same);
    }
}

static void stochastic_words_continue() {
    const int64_t rows = 6, cols = 40;
    const std::vector<float> a = exact(rows, cols, 9);
    MX4Matrix Q(rows, cols), P(rows, cols);
    RandBLAS::RNGState<> s(7);
    const RandBLAS::RNGState<> next = mx4_quantize(Layout::RowMajor, Op::NoTrans, rows, cols, a.data(), cols, Q, s);
    CHECK(next.counter.v[0] == (uint32_t)(rows * 10) && next.counter.v[1] == 0 && next.key.v[0] == 7);
    mx4_quantize(Layout::RowMajor, Op::NoTrans, rows, cols, a.data(), cols, P);
    CHECK(std::memcmp(Q.codes, P.codes, rows * Q.ld_codes) == 0);   // exact numbers do not move
}

static void device_arrays() {
    const int64_t rows = 9, cols = 64;
    const std::vector<float> a = exact(rows, cols, 2);
    uint8_t *codes, *scales;
    float *A;
    CHECK(hipMalloc(&codes, rows * 32) == hipSuccess && hipMalloc(&scales, rows * 2) == hipSuccess &&
          hipMalloc(&A, rows * cols * 4) == hipSuccess);
    CHECK(hipMemcpy(A, a.data(), rows * cols * 4, hipMemcpyHostToDevice) == hipSuccess);
    MX4Matrix Q(rows, cols, codes, 32, scales, 2);
    mx4_quantize(Layout::RowMajor, Op::NoTrans, rows, cols, A, cols, Q);
    std::vector<float> back(rows * cols);
    mx4_dequantize(Layout::RowMajor, Op::NoTrans, rows, cols, Q, 0, 0, back.data(), cols);
    CHECK(back == a);
    CHECK(hipFree(codes) == hipSuccess && hipFree(scales) == hipSuccess && hipFree(A) == hipSuccess);
}

static void refusals() {
    MX4Matrix Q(4, 40);
    std::vector<float> a(160);
    auto throws = [](auto f) {
        try {
            f();
        } catch (const RandBLAS::exceptions::Error &) {
            return true;
        }
        return false;
    };
    CHECK(throws([&] { mx4_quantize(Layout::RowMajor, Op::NoTrans, 4, 39, a.data(), 40, Q); }));
    CHECK(throws([&] { mx4_dequantize(Layout::RowMajor, Op::NoTrans, 4, 8, Q, 0, 16, a.data(), 40); }));
    CHECK(throws([&] { mxmm(Layout::RowMajor, Op::NoTrans, Op::NoTrans, 4, 4, 40, 1.f, Q, 0, 0, Q, 0, 0, 0.f, a.data(), 4); }));
    MX4Matrix moved(std::move(Q));
    CHECK(moved.own_memory && !Q.own_memory);
}

int main() {
    try {
        there_and_back<float>();
        there_and_back<double>();
        there_and_back<bf16>();
        products<float>();
        products<bf16>();
        stochastic_words_continue();
        device_arrays();
        refusals();
    } catch (const std::exception &e) {
        std::printf("FAILED: %s\n", e.what());
        return 1;
    }
    std::printf(g_fail ? "%d FAILED\n" : "ALL PASSED\n", g_fail);
    return g_fail != 0;
}
