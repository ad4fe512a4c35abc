// mx4.hip -- quantisation to 4-bit microscaled matrices and its inverse (gfx950).
//
// Quantisation of a block x[0..31]: top = max |x|, e = floor(log2 top) - 2 clamped to [-127, 125] (the
// largest power of two of the block on the largest one of E2M1, MX v1.0 section 6.3), scale byte e + 127.
//   nearest:    code = x 2^-e rounded to the nearest E2M1 value, ties to even, above 6 to 6.
//   stochastic: e is one more where top > 6 * 2^e, so that nothing is cut to 6; with low <= v < high the
//               E2M1 neighbours of v = |x| 2^-e, code is high iff w < floor((v - low) / (high - low) 2^32),
//               w the element's 32 random bits. The mean over w is x 2^-e up to 2^-32 of a step.
// x 2^-e is exact (a power of two; what underflows is far below half a step), so codes and scales do not
// depend on the kernel. A block that holds an infinity or a NaN gets the NaN scale and zero codes.
//
// Both kernels move each byte once and are bound by HBM. Two forms, by which direction is contiguous:
//   rows: blocks lie along memory. Four lanes share a block (8 elements each, 16-64 bytes of load and
//         4 bytes of codes a lane, both contiguous over the wave); the block's maximum crosses the four
//         lanes in two quad permutes. Accesses are as wide where a row starts at an odd multiple of an element
//         (4096 x 5731 bf16 back to elements: single elements stored, four a lane, 35 us, this 24 us).
//   cols: blocks lie across memory. A lane owns a row's block: 32 loads, each contiguous over the 64
//         lanes, the maximum in registers, 16 bytes of codes a lane.
// Quantising and dequantising, two launches: 8192 x 16384 f32 192 us (5.96 TB/s; a copy through the caches runs at
// 4.9), 8192 x 8192 bf16 56 us, stochastic 90 us (bound by the generator's integer multiplications), 1024 x 16384 f32
// across memory 29 us.
#include "common.hpp"
#include "mx4.hpp"

namespace rbh {
namespace {

constexpr int MXT = 256;

template <int TYPE> struct Elem;
template <> struct Elem<MX4_F64> { typedef double mem; typedef double val; };
template <> struct Elem<MX4_F32> { typedef float mem; typedef float val; };
template <> struct Elem<MX4_F16> { typedef _Float16 mem; typedef float val; };
template <> struct Elem<MX4_BF16> { typedef __bf16 mem; typedef float val; };

__device__ __forceinline__ uint32_t bits(float x) { return __builtin_bit_cast(uint32_t, x); }
__device__ __forceinline__ uint64_t bits(double x) { return __builtin_bit_cast(uint64_t, x); }
__device__ __forceinline__ uint32_t abs_bits(float x) { return bits(x) & 0x7FFFFFFFu; }
__device__ __forceinline__ uint64_t abs_bits(double x) { return bits(x) & 0x7FFFFFFFFFFFFFFFull; }

// the maximum over the 4 lanes of a quad (quad_perm [1,0,3,2], then [2,3,0,1])
template <int CTRL> __device__ __forceinline__ uint32_t quad(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, true);
}
template <int CTRL> __device__ __forceinline__ uint64_t quad(uint64_t v) {
    return ((uint64_t)quad<CTRL>((uint32_t)(v >> 32)) << 32) | quad<CTRL>((uint32_t)v);
}
template <typename B> __device__ __forceinline__ B quad_max(B v) {
    B o = quad<0xB1>(v);
    v = o > v ? o : v;
    o = quad<0x4E>(v);
    return o > v ? o : v;
}

// the block's exponent e (127 + e is the scale byte) from the bits of its largest magnitude; 128 = NaN.
// Numbers below 2^-125 all have e = -127, so subnormals need no normalisation.
template <bool SR> __device__ __forceinline__ int block_exp(uint32_t top) {
    const int E = (int)(top >> 23);
    if (E == 255) return 128;
    const int e = E - 129 + (SR && (top & 0x7FFFFFu) > 0x400000u ? 1 : 0);
    return e < -127 ? -127 : e > 125 ? 125 : e;
}
template <bool SR> __device__ __forceinline__ int block_exp(uint64_t top) {
    const int E = (int)(top >> 52);
    if (E == 2047) return 128;
    const int e = E - 1025 + (SR && (top & 0xFFFFFFFFFFFFFull) > 0x8000000000000ull ? 1 : 0);
    return e < -127 ? -127 : e > 125 ? 125 : e;
}
// 2^-e
__device__ __forceinline__ float inv_scale(int e, float) { return __builtin_bit_cast(float, (uint32_t)(127 - e) << 23); }
__device__ __forceinline__ double inv_scale(int e, double) { return __builtin_bit_cast(double, (uint64_t)(1023 - e) << 52); }

// v = x 2^-e as a float that rounds to the same E2M1 value: a double keeps what it loses below the last
// bit as a set last bit (so no second rounding meets a tie that was none)
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(double v) {
    const float f = __double2float_rz(v);
    return (double)f == v ? f : __builtin_bit_cast(float, bits(f) | 1u);
}

// |v| <= 6 on its E2M1 neighbours by the random word w; the result is an E2M1 value
template <typename V> __device__ __forceinline__ float stochastic(V v, uint32_t w) {
    V a = v < 0 ? -v : v;
    a = a > (V)6 ? (V)6 : a;
    const V per = a < (V)2 ? (V)2 : a < (V)4 ? (V)1 : (V)0.5, step = a < (V)2 ? (V)0.5 : a < (V)4 ? (V)1 : (V)2;
    const V t = a * per, low = __builtin_floor(t);
    const uint32_t part = (uint32_t)((t - low) * (V)4294967296.0);
    const float r = (float)((low + (V)(w < part ? 1 : 0)) * step);
    return __builtin_copysignf(r, (float)v);
}

// 8 codes of v[0..7] (E2M1 nearest even, above 6 to 6), v[0] in the low 4 bits
__device__ __forceinline__ uint32_t codes8(const float *v) {
    uint32_t o = 0;
    o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[0], v[1], 1.0f, 0);
    o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[2], v[3], 1.0f, 1);
    o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[4], v[5], 1.0f, 2);
    o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[6], v[7], 1.0f, 3);
    return o;
}

// 8 elements of row r from column c of a block with exponent e
template <bool SR, typename V>
__device__ __forceinline__ uint32_t encode8(const V *x, int e, const Mx4Random &rnd, int64_t r, int64_t c) {
    if (e == 128) return 0;
    const V inv = inv_scale(e, (V)0);
    float v[8];
    if constexpr (SR) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t ctr[4];
            rb::ctr_add(rnd.ctr, (uint64_t)r * rnd.quads + (uint64_t)(c >> 2) + (uint64_t)h, ctr);
            const rb::u32x4 w = rnd.rng == rb::RNG_PHILOX ? rb::philox4x32_uk(ctr[0], ctr[1], ctr[2], ctr[3], rnd.key[0], rnd.key[1])
                                                          : rb::cbrng(rnd.rng, ctr, rnd.key);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 * h + i] = stochastic(x[4 * h + i] * inv, w.v[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f32(x[i] * inv);
    }
    return codes8(v);
}

// n / d for 32-bit n, d >= 1 (Granlund and Montgomery, 1994: a rounded-up reciprocal of 33 bits)
struct FastDiv {
    uint32_t mul, shift, d;
};
FastDiv fast_div(uint32_t d) {
    uint32_t l = 0;
    while (l < 32 && ((uint64_t)1 << l) < d) ++l;
    const uint64_t m = ((((uint64_t)1 << l) - d) << 32) / d + 1;
    return {(uint32_t)m, l, d};
}
__device__ __forceinline__ uint32_t operator/(uint32_t n, const FastDiv &f) {
    const uint32_t t = __umulhi(f.mul, n);
    return f.d == 1 ? n : (((n - t) >> 1) + t) >> (f.shift - 1);
}

template <int TYPE, bool SR, bool NT>
__global__ __launch_bounds__(MXT) void quantize_rows_kernel(const typename Elem<TYPE>::mem *__restrict__ A, int64_t ld,
                                                             Mx4View Q, FastDiv nb, uint32_t units, int64_t row0,
                                                             Mx4Random rnd) {
    typedef typename Elem<TYPE>::mem M;
    typedef typename Elem<TYPE>::val V;
    typedef M any8_t __attribute__((ext_vector_type(8), aligned(sizeof(M))));   // one or a few wide loads wherever it is
    const uint32_t u = blockIdx.x * (uint32_t)MXT + threadIdx.x;
    const bool live = u < units;   // whole quads only: 4 units a block
    const uint32_t ub = (live ? u : 0u) >> 2, q = u & 3u;
    const uint32_t rr = ub / nb, b = ub - rr * nb.d;
    const int64_t r = row0 + rr, c = (int64_t)b * MX4_BLOCK + 8 * q;
    const M *p = A + r * ld + c;
    V x[8];
    if (c + 8 <= Q.cols) {
        const any8_t m = NT ? __builtin_nontemporal_load((const any8_t *)p) : *(const any8_t *)p;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (V)m[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = c + i < Q.cols ? (V)p[i] : (V)0;
    }
    auto top = abs_bits(x[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) top = abs_bits(x[i]) > top ? abs_bits(x[i]) : top;
    const int e = block_exp<SR>(quad_max(top));
    if (!live) return;
    const uint32_t o = encode8<SR>(x, e, rnd, r, c);
    *reinterpret_cast<uint32_t *>(Q.codes + r * Q.ldq + (int64_t)b * 16 + 4 * q) = o;
    if (q == 0) Q.scales[r * Q.lds + b] = (uint8_t)(e + 127);
}

template <int TYPE, bool SR, bool NT>
__global__ __launch_bounds__(MXT) void quantize_cols_kernel(const typename Elem<TYPE>::mem *__restrict__ A, int64_t ld,
                                                             Mx4View Q, int64_t nb, Mx4Random rnd) {
    typedef typename Elem<TYPE>::val V;
    const int64_t r = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
    if (r >= Q.rows) return;
    for (int64_t b = (int64_t)blockIdx.y * (MXT / 64) + (threadIdx.x >> 6); b < nb; b += (int64_t)gridDim.y * (MXT / 64)) {
        const int64_t c0 = b * MX4_BLOCK;
        const auto *p = A + r + c0 * ld;
        V x[MX4_BLOCK];
        if (c0 + MX4_BLOCK <= Q.cols) {
#pragma unroll
            for (int i = 0; i < MX4_BLOCK; ++i) x[i] = (V)(NT ? __builtin_nontemporal_load(p + i * ld) : p[i * ld]);
        } else {
#pragma unroll
            for (int i = 0; i < MX4_BLOCK; ++i) x[i] = c0 + i < Q.cols ? (V)p[i * ld] : (V)0;
        }
        auto top = abs_bits(x[0]);
#pragma unroll
        for (int i = 1; i < MX4_BLOCK; ++i) top = abs_bits(x[i]) > top ? abs_bits(x[i]) : top;
        const int e = block_exp<SR>(top);
        uint4 o;
        o.x = encode8<SR>(x, e, rnd, r, c0);
        o.y = encode8<SR>(x + 8, e, rnd, r, c0 + 8);
        o.z = encode8<SR>(x + 16, e, rnd, r, c0 + 16);
        o.w = encode8<SR>(x + 24, e, rnd, r, c0 + 24);
        *reinterpret_cast<uint4 *>(Q.codes + r * Q.ldq + b * 16) = o;
        Q.scales[r * Q.lds + b] = (uint8_t)(e + 127);
    }
}

// 2^(s - 127), NaN for s = 255; the smallest is a subnormal float
__device__ __forceinline__ float scale_f32(uint32_t s) {
    return __builtin_bit_cast(float, s == 255 ? 0x7FC00000u : s == 0 ? 0x00400000u : s << 23);
}

// the 8 values of a word of codes. A product with the scale is exact in 32 bits (and in the 16 of bf16,
// whose exponents are the same); above 2^128 it is infinite there and in 16-bit results.
template <int TYPE> __device__ __forceinline__ void decode8(uint32_t w, float scale, typename Elem<TYPE>::mem *o) {
    typedef typename Elem<TYPE>::mem M;
    typedef float v2_t __attribute__((ext_vector_type(2)));
    v2_t v[4];
    v[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0);
    v[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
    v[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2);
    v[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = v[i >> 1][i & 1];
        if constexpr (TYPE == MX4_F64) o[i] = (double)x * (double)scale;
        // the sign apart: a product rounded to f16 becomes x * scale + 0 in one instruction, which turns -0 to 0
        else if constexpr (TYPE == MX4_F16) o[i] = (M)__builtin_copysignf(x * scale, x);
        else o[i] = (M)(x * scale);
    }
}

template <int TYPE>
__global__ __launch_bounds__(MXT) void dequantize_rows_kernel(Mx4View Q, typename Elem<TYPE>::mem *__restrict__ A,
                                                               int64_t ld, FastDiv nb, uint32_t units, int64_t row0) {
    typedef typename Elem<TYPE>::mem M;
    constexpr int E = 16 / sizeof(M), UB = MX4_BLOCK / E;   // elements a lane, lanes a block: 16 bytes a lane, side by side
    typedef M any_t __attribute__((ext_vector_type(E), aligned(sizeof(M))));
    const uint32_t u = blockIdx.x * (uint32_t)MXT + threadIdx.x;
    if (u >= units) return;
    const uint32_t ub = u / UB, q = u % UB;
    const uint32_t rr = ub / nb, b = ub - rr * nb.d;
    const int64_t r = row0 + rr, c = (int64_t)b * MX4_BLOCK + E * q;
    if (c >= Q.cols) return;
    const uint8_t *from = Q.codes + r * Q.ldq + (int64_t)b * 16 + E / 2 * q;
    const uint32_t w = E == 8 ? *reinterpret_cast<const uint32_t *>(from) : E == 4 ? *reinterpret_cast<const uint16_t *>(from) : *from;
    M o[8];
    decode8<TYPE>(w, scale_f32(Q.scales[r * Q.lds + b]), o);
    M *p = A + r * ld + c;
    if (c + E <= Q.cols) {
        any_t m;
#pragma unroll
        for (int i = 0; i < E; ++i) m[i] = o[i];
        // the caches keep what is read (8192 x 16384 f32 and back 211 us, without 255; no reader of the result measured)
        __builtin_nontemporal_store(m, (any_t *)p);
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (c + i < Q.cols) p[i] = o[i];
    }
}

template <int TYPE, bool NT>
__global__ __launch_bounds__(MXT) void dequantize_cols_kernel(Mx4View Q, typename Elem<TYPE>::mem *__restrict__ A,
                                                               int64_t ld, int64_t nb) {
    typedef typename Elem<TYPE>::mem M;
    const int64_t r = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
    if (r >= Q.rows) return;
    for (int64_t b = (int64_t)blockIdx.y * (MXT / 64) + (threadIdx.x >> 6); b < nb; b += (int64_t)gridDim.y * (MXT / 64)) {
        const uint4 w = *reinterpret_cast<const uint4 *>(Q.codes + r * Q.ldq + b * 16);
        const float scale = scale_f32(Q.scales[r * Q.lds + b]);
        const int64_t c0 = b * MX4_BLOCK;
        M o[MX4_BLOCK];
        decode8<TYPE>(w.x, scale, o);
        decode8<TYPE>(w.y, scale, o + 8);
        decode8<TYPE>(w.z, scale, o + 16);
        decode8<TYPE>(w.w, scale, o + 24);
        M *p = A + r + c0 * ld;
#pragma unroll
        for (int i = 0; i < MX4_BLOCK; ++i)
            if (c0 + i < Q.cols) {
                if constexpr (NT) __builtin_nontemporal_store(o[i], p + i * ld);
                else p[i * ld] = o[i];
            }
    }
}

// Launches over rows or row blocks: f(row0, rows) is called for chunks whose unit count stays below 2^31
template <typename F> hipError_t row_chunks(int64_t rows, int64_t units_a_row, F f) {
    const int64_t most = ((int64_t)1 << 31) / units_a_row;
    for (int64_t r = 0; r < rows; r += most) {
        const hipError_t e = f(r, rows - r < most ? rows - r : most);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

dim3 cols_grid(int64_t rows, int64_t nb) {
    const int64_t y = (nb + MXT / 64 - 1) / (MXT / 64);
    return dim3((unsigned)((rows + 63) / 64), (unsigned)(y < 65535 ? y : 65535));
}

template <int TYPE, bool SR>
hipError_t quantize_t(const Mx4Dense &A, const Mx4View &Q, const Mx4Random &rnd, hipStream_t s) {
    typedef typename Elem<TYPE>::mem M;
    const M *a = (const M *)A.ptr;
    const int64_t nb = mx4_blocks(Q.cols);
    // What the last-level cache (256 MB) cannot hold passes it by: 8192 x 16384 f32 225 and 250 us with the way back,
    // 4096 x 8192 f64 across memory 104 and 121, but 3412 x 5730 f32, which it can hold, 36 and 32
    const bool past = Q.rows * Q.cols * (int64_t)sizeof(M) >= ((int64_t)1 << 28);
    if (A.sc == 1) {
        return row_chunks(Q.rows, nb * 4, [&](int64_t r0, int64_t rows) {
            const uint32_t units = (uint32_t)(rows * nb * 4);
            auto go = [&](auto kernel) {
                hipLaunchKernelGGL(kernel, dim3((units + MXT - 1) / MXT), dim3(MXT), 0, s, a, A.sr, Q, fast_div((uint32_t)nb), units, r0, rnd);
            };
            past ? go(quantize_rows_kernel<TYPE, SR, true>) : go(quantize_rows_kernel<TYPE, SR, false>);
            return hipGetLastError();
        });
    }
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, cols_grid(Q.rows, nb), dim3(MXT), 0, s, a, A.sc, Q, nb, rnd); };
    past ? go(quantize_cols_kernel<TYPE, SR, true>) : go(quantize_cols_kernel<TYPE, SR, false>);
    return hipGetLastError();
}

template <int TYPE> hipError_t dequantize_t(const Mx4View &Q, const Mx4Dense &A, hipStream_t s) {
    typedef typename Elem<TYPE>::mem M;
    M *a = (M *)const_cast<void *>(A.ptr);
    const int64_t nb = mx4_blocks(Q.cols);
    if (A.sc == 1) {
        constexpr int a_block = MX4_BLOCK * sizeof(M) / 16;
        return row_chunks(Q.rows, nb * a_block, [&](int64_t r0, int64_t rows) {
            const uint32_t units = (uint32_t)(rows * nb * a_block);
            hipLaunchKernelGGL((dequantize_rows_kernel<TYPE>), dim3((units + MXT - 1) / MXT), dim3(MXT), 0, s, Q, a, A.sr,
                               fast_div((uint32_t)nb), units, r0);
            return hipGetLastError();
        });
    }
    // Past the caches only where a wave writes whole lines: 16384 x 16384 f32 547 and 572 us with the way there, 4097 x
    // 8191 bf16 82 and 61
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, cols_grid(Q.rows, nb), dim3(MXT), 0, s, Q, a, A.sc, nb); };
    (uintptr_t)a % 128 == 0 && A.sc * (int64_t)sizeof(M) % 128 == 0 ? go(dequantize_cols_kernel<TYPE, true>) : go(dequantize_cols_kernel<TYPE, false>);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_mx4_quantize(const Mx4Dense &A, const Mx4View &Q, const Mx4Random *rnd, hipStream_t s) {
    if (Q.rows <= 0 || Q.cols <= 0) return hipSuccess;
    const Mx4Random r = rnd ? *rnd : Mx4Random{};
    switch (A.type) {
        case MX4_F64: return rnd ? quantize_t<MX4_F64, true>(A, Q, r, s) : quantize_t<MX4_F64, false>(A, Q, r, s);
        case MX4_F32: return rnd ? quantize_t<MX4_F32, true>(A, Q, r, s) : quantize_t<MX4_F32, false>(A, Q, r, s);
        case MX4_F16: return rnd ? quantize_t<MX4_F16, true>(A, Q, r, s) : quantize_t<MX4_F16, false>(A, Q, r, s);
        default: return rnd ? quantize_t<MX4_BF16, true>(A, Q, r, s) : quantize_t<MX4_BF16, false>(A, Q, r, s);
    }
}

hipError_t launch_mx4_dequantize(const Mx4View &Q, const Mx4Dense &A, hipStream_t s) {
    if (Q.rows <= 0 || Q.cols <= 0) return hipSuccess;
    switch (A.type) {
        case MX4_F64: return dequantize_t<MX4_F64>(Q, A, s);
        case MX4_F32: return dequantize_t<MX4_F32>(Q, A, s);
        case MX4_F16: return dequantize_t<MX4_F16>(Q, A, s);
        default: return dequantize_t<MX4_BF16>(Q, A, s);
    }
}

}  // namespace rbh
