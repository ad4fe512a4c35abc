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
template <int TYPE>
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
            if (i < p.M && k < p.K) xv = (float)x[i * p.X.sr + k * p.X.sc];
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

// ---------------------------------------------------------------------------------------------
// Two 4-bit factors on the scaled matrix instruction
// ---------------------------------------------------------------------------------------------
typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

// D += A B^T over 128 columns: lane l holds row l & 15 of a factor, the block l >> 4 of its 4 blocks (32
// codes, 16 bytes) and that block's scale in the low byte of a word; D: column l & 15 (B's row), rows
// 4 (l >> 4) .. + 3 (A's rows).
__device__ __forceinline__ v4f mfma_mx4(v4i a, v4i b, v4f c, int sa, int sb) {
    const v8i wa = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1);
    const v8i wb = __builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1);
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, wb, c, 4, 4, 0, sa, 0, sb);
}

// out[o * ld + p] = alpha * sum + beta * out[o * ld + p]
struct Out {
    void *ptr;
    int64_t ld;
    int64_t np, no;
    float alpha, beta;
    bool vec;   // four consecutive p at a multiple of four are one aligned access
};
template <typename T> __device__ __forceinline__ void store4(const Out &o, int64_t p, int64_t q, v4f v) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    if (q >= o.no || p >= o.np) return;
    T *c = (T *)o.ptr + q * o.ld + p;
    if (o.vec && p + 4 <= o.np) {
        t4 r;
        if (o.beta != 0.f) {
            const t4 old = *(const t4 *)c;
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = (T)(o.alpha * v[i] + o.beta * (float)old[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = (T)(o.alpha * v[i]);
        }
        *(t4 *)c = r;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (p + i < o.np) c[i] = (T)(o.beta != 0.f ? o.alpha * v[i] + o.beta * (float)c[i] : o.alpha * v[i]);
    }
}

// A range of memory for loads straight to LDS (16 bytes a lane, lane after lane from `lds`, which is the
// same for the wave). An offset at or past the range's end reads zeros; `soffset` is added to the address
// and does not count for that.
typedef __amdgpu_buffer_rsrc_t Buffer;
constexpr uint32_t OUTSIDE = 0x7FFFFFF0u;
__device__ __forceinline__ Buffer buffer(const void *p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, (int)bytes, 0x00020000);
}
__device__ __forceinline__ void load_lds16(Buffer b, void *lds, uint32_t voffset, uint32_t soffset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (__attribute__((address_space(3))) void *)lds, 16, (int)voffset,
                                             (int)soffset, 0, 0);
}

__device__ __forceinline__ void load_lds4(Buffer b, void *lds, uint32_t voffset, uint32_t soffset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (__attribute__((address_space(3))) void *)lds, 4, (int)voffset,
                                             (int)soffset, 0, 0);
}
// Every wave's loads to LDS have arrived and every wave has read what they will overwrite. The wait has to
// be written out: __syncthreads does not wait for loads that go to LDS.
__device__ __forceinline__ void arrive() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// Tile t of a workgroup: workgroups go to the 8 XCDs in turn, so XCD x takes a run of consecutive tiles,
// and the runs go down groups of 8 tiles of o before the next p, so the tiles that one XCD works on
// together share rows of both factors in its L2.
__device__ __forceinline__ void tile_of(uint32_t bid, uint32_t tp, uint32_t to, uint32_t &ip, uint32_t &io) {
    const uint32_t n = tp * to, q = n / 8, r = n % 8, x = bid % 8, y = bid / 8;
    const uint32_t t = x * q + (x < r ? x : r) + y;
    const uint32_t group = t / (8 * tp), g0 = group * 8;
    const uint32_t h = to - g0 < 8 ? to - g0 : 8, in = t - group * 8 * tp;
    io = g0 + in % h;
    ip = in / h;
}

// BP x BO entries of the result a workgroup, WP x WO a wave; 256 columns (8 blocks) of both factors a step,
// loaded straight to LDS, double-buffered. A row of a step is 128 bytes of codes; its 16-byte blocks are
// kept at place block ^ (row / 2 & 7), which spreads the 16 rows that a matrix operand reads at once over
// all banks (the lane that fills a place loads the block that belongs there). A row's 8 scale bytes lie
// behind the codes.
template <typename T, int BP, int BO, int WP, int WO>
__global__ __launch_bounds__((BP / WP) * (BO / WO) * 64, 2) void both_tile_kernel(Mx4View P, Mx4View O, int nb, Out out) {
    constexpr int NW = (BP / WP) * (BO / WO), NT = NW * 64;
    constexpr int FP = WP / 16, FO = WO / 16;
    constexpr int ROWS = BP + BO;                       // rows staged, P's first
    constexpr int LP = BP * 8 / NT, LO = BO * 8 / NT;   // 16-byte loads a thread
    static_assert(BP * 8 % NT == 0 && BO * 8 % NT == 0 && NT / 8 % 16 == 0, "whole loads, one block for all rows of a thread");
    constexpr int SL = ROWS * 2 / NT;                   // 4-byte loads of scales a thread
    static_assert(ROWS * 2 % NT == 0 && BP % 32 == 0, "whole loads of one factor");
    __shared__ __attribute__((aligned(16))) uint8_t lds0[ROWS * 136], lds1[ROWS * 136];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    uint32_t ip, io;
    tile_of(blockIdx.x, (uint32_t)((P.rows + BP - 1) / BP), (uint32_t)((O.rows + BO - 1) / BO), ip, io);
    const int64_t p0 = (int64_t)ip * BP, o0 = (int64_t)io * BO;
    const int wp = wave % (BP / WP), wo = wave / (BP / WP);
    // rows beyond the last one lie outside the ranges and read as zeros
    const int np = (int)(P.rows - p0 < BP ? P.rows - p0 : BP), no = (int)(O.rows - o0 < BO ? O.rows - o0 : BO);
    const Buffer pb = buffer(P.codes + p0 * P.ldq, (uint32_t)((np - 1) * P.ldq + nb * 16));
    const Buffer ob = buffer(O.codes + o0 * O.ldq, (uint32_t)((no - 1) * O.ldq + nb * 16));
    const Buffer ps = buffer(P.scales + p0 * P.lds, (uint32_t)((np - 1) * P.lds + (nb + 3) / 4 * 4));
    const Buffer os = buffer(O.scales + o0 * O.lds, (uint32_t)((no - 1) * O.lds + (nb + 3) / 4 * 4));
    const int block = (tid & 7) ^ ((tid >> 4) & 7);
    const uint32_t vp = (uint32_t)((tid >> 3) * P.ldq) + block * 16, vo = (uint32_t)((tid >> 3) * O.ldq) + block * 16;
    const uint32_t rp = (uint32_t)P.ldq * (NT / 8), ro = (uint32_t)O.ldq * (NT / 8);
    // blocks b0 .. b0 + 7 of every row; those past the last are zero
    auto load = [&](int b0, uint8_t *lds) {
        const bool in = b0 + block < nb;
#pragma unroll
        for (int i = 0; i < LP; ++i) load_lds16(pb, lds + (i * NT + wave * 64) * 16, in ? vp + i * rp : OUTSIDE, b0 * 16);
#pragma unroll
        for (int i = 0; i < LO; ++i)
            load_lds16(ob, lds + BP * 128 + (i * NT + wave * 64) * 16, in ? vo + i * ro : OUTSIDE, b0 * 16);
#pragma unroll
        for (int i = 0; i < SL; ++i) {   // a wave's 32 rows are of one factor
            const int w = i * NW + wave, row = w * 32 + (lane >> 1), half = lane & 1;
            uint8_t *to = lds + ROWS * 128 + w * 256;
            const bool in = b0 + 4 * half < nb;
            if (w * 32 < BP) load_lds4(ps, to, in ? (uint32_t)(row * P.lds) + 4 * half : OUTSIDE, b0);
            else load_lds4(os, to, in ? (uint32_t)((row - BP) * O.lds) + 4 * half : OUTSIDE, b0);
        }
    };

    v4f acc[FP][FO];
#pragma unroll
    for (int a = 0; a < FP; ++a)
#pragma unroll
        for (int b = 0; b < FO; ++b) acc[a][b] = v4f{0.f, 0.f, 0.f, 0.f};

    // LDS places of this lane: one address a factor and half step, everything else an immediate
    int at[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) at[h] = ((h * 4 + g) ^ ((r16 >> 1) & 7)) * 16 + r16 * 128;
    const int pa = wp * WP * 128, pb_ = (BP + wo * WO) * 128;
    const int psc = ROWS * 128 + (wp * WP + r16) * 8, osc = ROWS * 128 + (BP + wo * WO + r16) * 8;
    auto compute = [&](int b0, const uint8_t *lds) {
        const uint8_t *ssa = lds + psc, *ssb = lds + osc;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint8_t *ca = lds + (pa + at[h]), *cb = lds + (pb_ + at[h]);
            v4i a[FP], b[FO];
            uint32_t sa[FP], sb[FO];
            const uint32_t width = b0 + h * 4 + g < nb ? 8 : 0;   // scales past the last block, whatever is there, as 0
#pragma unroll
            for (int f = 0; f < FO; ++f) {
                b[f] = *(const v4i *)(cb + f * 16 * 128);
                sb[f] = __builtin_amdgcn_ubfe(*(const uint32_t *)(ssb + f * 16 * 8 + h * 4), 8 * g, width);
            }
#pragma unroll
            for (int f = 0; f < FP; ++f) {
                a[f] = *(const v4i *)(ca + f * 16 * 128);
                sa[f] = __builtin_amdgcn_ubfe(*(const uint32_t *)(ssa + f * 16 * 8 + h * 4), 8 * g, width);
            }
#pragma unroll
            for (int fa = 0; fa < FP; ++fa)
#pragma unroll
                for (int fb = 0; fb < FO; ++fb) acc[fa][fb] = mfma_mx4(a[fa], b[fb], acc[fa][fb], (int)sa[fa], (int)sb[fb]);
        }
    };
    // two steps a round, so that each works on its own array and its loads are seen to go to the other
    load(0, lds0);
    arrive();
    int b0 = 0;
    for (; b0 + 8 < nb; b0 += 16) {
        load(b0 + 8, lds1);
        __builtin_amdgcn_sched_barrier(0);   // the loads leave before the products, not behind them
        compute(b0, lds0);
        arrive();
        load(b0 + 16, lds0);   // past the last block: nothing but zeros, unread or added
        __builtin_amdgcn_sched_barrier(0);
        compute(b0 + 8, lds1);
        arrive();
    }
    if (b0 < nb) compute(b0, lds0);
#pragma unroll
    for (int b = 0; b < FO; ++b)
#pragma unroll
        for (int a = 0; a < FP; ++a)
            store4<T>(out, p0 + wp * WP + a * 16 + 4 * g, o0 + wo * WO + b * 16 + r16, acc[a][b]);
}

template <typename T, int BP, int BO, int WP, int WO>
hipError_t launch_both_tile(const Mx4View &P, const Mx4View &O, const Out &out, hipStream_t s) {
    const int nb = (int)mx4_blocks(P.cols);
    const int64_t tiles = ((P.rows + BP - 1) / BP) * ((O.rows + BO - 1) / BO);
    constexpr int NT = (BP / WP) * (BO / WO) * 64;
    hipLaunchKernelGGL((both_tile_kernel<T, BP, BO, WP, WO>), dim3((unsigned)tiles), dim3(NT), 0, s, P, O, nb, out);
    return hipGetLastError();
}

// Scales whose rows do not start at multiples of 4 bytes are copied to rows that do.
bool aligned_scales(const Mx4View &v) { return (uintptr_t)v.scales % 4 == 0 && v.lds % 4 == 0; }
size_t scales_work(const Mx4View &v) {
    return aligned_scales(v) ? 0 : (size_t)((v.rows * ((mx4_blocks(v.cols) + 3) / 4 * 4) + 255) / 256 * 256);
}
__global__ __launch_bounds__(256) void copy_scales_kernel(const uint8_t *src, int64_t lds, int64_t rows, int nb, int nb4, uint8_t *dst) {
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b >= nb) return;
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) dst[r * nb4 + b] = src[r * lds + b];
}
hipError_t align_scales(Mx4View &v, uint8_t *&work, hipStream_t s) {
    if (aligned_scales(v)) return hipSuccess;
    const int nb = (int)mx4_blocks(v.cols), nb4 = (nb + 3) / 4 * 4;
    const dim3 grid((unsigned)((nb + 255) / 256), (unsigned)(v.rows < 65535 ? v.rows : 65535));
    hipLaunchKernelGGL(copy_scales_kernel, grid, dim3(256), 0, s, v.scales, v.lds, v.rows, nb, nb4, work);
    const size_t bytes = scales_work(v);
    v.scales = work;
    v.lds = nb4;
    work += bytes;
    return hipGetLastError();
}

template <int TYPE> hipError_t both_t(const Mx4Product &q, uint8_t *work, hipStream_t s) {
    Mx4Product p = q;
    hipError_t e = align_scales(p.XQ, work, s);
    if (e == hipSuccess) e = align_scales(p.Y, work, s);
    if (e != hipSuccess) return e;
    typedef typename Elem<TYPE>::mem T;
    // the factor whose rows are the contiguous index of C gives the operand whose 4 entries a lane holds
    const bool xp = p.ci == 1;
    const Mx4View &P = xp ? p.XQ : p.Y, &O = xp ? p.Y : p.XQ;
    const int64_t ld = xp ? p.cj : p.ci;
    const Out out{p.C, ld, P.rows, O.rows, p.alpha, p.beta, (uintptr_t)p.C % (4 * sizeof(T)) == 0 && ld % 4 == 0};
    auto tiles = [&](int64_t b) { return ((P.rows + b - 1) / b) * ((O.rows + b - 1) / b); };
    if (tiles(256) >= 256) return launch_both_tile<T, 256, 256, 128, 64>(P, O, out, s);
    return launch_both_tile<T, 128, 128, 64, 64>(P, O, out, s);
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
    if (p.both) return both_t<TYPE>(p, (uint8_t *)work, s);
    const dim3 grid((unsigned)((p.M + 63) / 64), (unsigned)((p.N + 63) / 64));
    hipLaunchKernelGGL((product_plain_kernel<TYPE>), grid, dim3(256), 0, s, p);
    return hipGetLastError();
}

}  // namespace

size_t mx4_product_work(const Mx4Product &p) {
    if (p.K <= 0 || p.alpha == 0.f) return 0;
    return p.both ? scales_work(p.XQ) + scales_work(p.Y) : 0;
}

hipError_t launch_mx4_product(const Mx4Product &p, void *work, hipStream_t s) {
    if (p.M <= 0 || p.N <= 0) return hipSuccess;
    switch (p.type) {
        case MX4_F32: return product_t<MX4_F32>(p, work, s);
        case MX4_F16: return product_t<MX4_F16>(p, work, s);
        default: return product_t<MX4_BF16>(p, work, s);
    }
}

}  // namespace rbh
