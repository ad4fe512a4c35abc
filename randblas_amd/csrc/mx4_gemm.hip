// mx4_gemm.hip -- products with 4-bit microscaled matrices (gfx950).
#include "common.hpp"
#include "mx4.hpp"

namespace rbh {
namespace {

template <int TYPE> struct Elem;
template <> struct Elem<MX4_F32> { typedef float mem; };
template <> struct Elem<MX4_F16> { typedef _Float16 mem; };
template <> struct Elem<MX4_BF16> { typedef __bf16 mem; };

__device__ __forceinline__ float scale_f32(uint32_t s) {
    return __builtin_bit_cast(float, s == 255 ? 0x7FC00000u : s == 0 ? 0x00400000u : s << 23);
}
__device__ __forceinline__ float value(const Mx4View &Q, int64_t r, int64_t c) {
    const uint32_t byte = Q.codes[r * Q.ldq + (c >> 1)], code = (c & 1) ? byte >> 4 : byte & 15u;
    const uint32_t m = code & 7u;
    // 0, 0.5, 1, 1.5, 2, 3, 4, 6 in halves, 4 bits each
    const float v = 0.5f * (float)((0xC8643210u >> (4 * m)) & 15u);
    return (code & 8u ? -v : v) * scale_f32(Q.scales[r * Q.lds + (c >> 5)]);
}

// One 64 x 64 tile of C a workgroup, 4 x 4 entries a thread, both factors decoded to 32 bits in LDS, one
// block of 32 at a time; a block's sum is formed apart and added to the total.
template <int TYPE, bool BOTH>
__global__ __launch_bounds__(256) void product_plain_kernel(Mx4Product p) {
    typedef typename Elem<TYPE>::mem T;
    __shared__ float xs[32][65], ys[32][65];
    const int64_t i0 = (int64_t)blockIdx.x * 64, j0 = (int64_t)blockIdx.y * 64;
    const int ti = threadIdx.x & 15, tj = threadIdx.x >> 4;
    float acc[4][4] = {};
    const T *x = (const T *)p.X.ptr;
    for (int64_t k0 = 0; k0 < p.K; k0 += 32) {
        for (int t = threadIdx.x; t < 64 * 32; t += 256) {
            const int o = t & 63, kk = t >> 6;
            const int64_t i = i0 + o, j = j0 + o, k = k0 + kk;
            float xv = 0.f, yv = 0.f;
            if (i < p.M && k < p.K) {
                if constexpr (BOTH) xv = value(p.XQ, i, k);
                else xv = (float)x[i * p.X.sr + k * p.X.sc];
            }
            if (j < p.N && k < p.K) yv = p.yt ? value(p.Y, k, j) : value(p.Y, j, k);
            xs[kk][o] = xv;
            ys[kk][o] = yv;
        }
        __syncthreads();
        float part[4][4] = {};
        for (int kk = 0; kk < 32; ++kk)
            for (int a = 0; a < 4; ++a)
                for (int b = 0; b < 4; ++b) part[a][b] += xs[kk][ti + 16 * a] * ys[kk][tj + 16 * b];
        for (int a = 0; a < 4; ++a)
            for (int b = 0; b < 4; ++b) acc[a][b] += part[a][b];
        __syncthreads();
    }
    T *C = (T *)p.C;
    for (int a = 0; a < 4; ++a)
        for (int b = 0; b < 4; ++b) {
            const int64_t i = i0 + ti + 16 * a, j = j0 + tj + 16 * b;
            if (i >= p.M || j >= p.N) continue;
            T &c = C[i * p.ci + j * p.cj];
            float v = p.alpha * acc[a][b];
            if (p.beta != 0.f) v += p.beta * (float)c;
            c = (T)v;
        }
}

// C = beta C (beta = 0: zeros, whatever C holds)
template <int TYPE> __global__ __launch_bounds__(256) void scale_kernel(Mx4Product p, int64_t inner, int64_t outer, int64_t ld) {
    typedef typename Elem<TYPE>::mem T;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= inner) return;
    for (int64_t j = blockIdx.y; j < outer; j += gridDim.y) {
        T &c = ((T *)p.C)[j * ld + i];
        c = p.beta == 0.f ? (T)0.f : (T)(p.beta * (float)c);
    }
}

template <int TYPE> hipError_t product_t(const Mx4Product &p, void *work, hipStream_t s) {
    if (p.K <= 0 || p.alpha == 0.f) {
        const int64_t inner = p.ci == 1 ? p.M : p.N, outer = p.ci == 1 ? p.N : p.M;
        hipLaunchKernelGGL((scale_kernel<TYPE>), dim3((unsigned)((inner + 255) / 256), (unsigned)(outer < 65535 ? outer : 65535)),
                           dim3(256), 0, s, p, inner, outer, p.ci == 1 ? p.cj : p.ci);
        return hipGetLastError();
    }
    const dim3 grid((unsigned)((p.M + 63) / 64), (unsigned)((p.N + 63) / 64));
    if (p.both) hipLaunchKernelGGL((product_plain_kernel<TYPE, true>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((product_plain_kernel<TYPE, false>), grid, dim3(256), 0, s, p);
    return hipGetLastError();
}

}  // namespace

size_t mx4_product_work(const Mx4Product &p) { return 0; }

hipError_t launch_mx4_product(const Mx4Product &p, void *work, hipStream_t s) {
    if (p.M <= 0 || p.N <= 0) return hipSuccess;
    switch (p.type) {
        case MX4_F32: return product_t<MX4_F32>(p, work, s);
        case MX4_F16: return product_t<MX4_F16>(p, work, s);
        default: return product_t<MX4_BF16>(p, work, s);
    }
}

}  // namespace rbh
