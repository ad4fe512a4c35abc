// mx4_gemm.hip -- products with 4-bit microscaled matrices (gfx950).
#include <type_traits>
#include <utility>

#include "common.hpp"
#include "mx4.hpp"

namespace rbh {
namespace {

template <int TYPE> struct Elem;
template <> struct Elem<MX4_F32> { typedef float mem; };
template <> struct Elem<MX4_F16> { typedef _Float16 mem; };
template <> struct Elem<MX4_BF16> { typedef __bf16 mem; };

// ---------------------------------------------------------------------------------------------
// Two 4-bit factors on the scaled matrix instruction
// ---------------------------------------------------------------------------------------------
typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

// D += A B^T over 128 columns: lane l holds row l & 15 of a factor, the block l >> 4 of its 4 blocks (32
// codes, 16 bytes) and that block's scale in the low byte of a word; D: column l & 15 (B's row), rows
// 4 (l >> 4) .. + 3 (A's rows).
__device__ __forceinline__ v4f mfma_mx4(v4i a, v4i b, v4f c, int sa, int sb) {
    const v8i wa = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1);
    const v8i wb = __builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1);
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, wb, c, 4, 4, 0, sa, 0, sb);
}

// the same in 32 x 32: lane l holds row l & 31 and the block l >> 5 of 2; D: column l & 31, rows 8 i + 4 (l >> 5)
// .. + 3 in entries 4 i .. + 3. Fed from registers by 2 waves a SIMD the 16 x 16 instruction reaches 5.46
// PFLOP/s on random codes, this one 6.51 (power is the bound: on zeros 9.63)
typedef float v16f __attribute__((ext_vector_type(16)));
template <int OA, int OB> __device__ __forceinline__ v16f mfma_mx4_32(v4i a, v4i b, v16f c, int sa, int sb) {
    const v8i wa = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1);
    const v8i wb = __builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1);
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wa, wb, c, 4, 4, OA, sa, OB, sb);
}

template <typename F, int... I> __device__ __forceinline__ void static_for_(F &&f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F> __device__ __forceinline__ void static_for(F &&f) { static_for_(f, std::make_integer_sequence<int, N>{}); }

// out[o * ld + p] = alpha * sum + beta * out[o * ld + p]. Four consecutive p are one access at any multiple of
// an element (3635 x 4651 f32 onto itself, single elements: 114 us, this 71).
struct Out {
    void *ptr;
    int64_t ld;
    int64_t np, no;
    float alpha, beta;
};
template <typename T> struct Four {
    typedef T t4 __attribute__((ext_vector_type(4)));
    T *c;
    int n;   // how many there are
    t4 old;
    __device__ __forceinline__ void load(const Out &o, T *at, int count) {
        c = at;
        n = count;
        if (o.beta == 0.f) return;
        if (n == 4) {
            __builtin_memcpy(&old, c, sizeof old);
        } else {
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (i < n) old[i] = c[i];
        }
    }
    // NT: past the caches, for results that fill them (8192 x 8192 x 1024 f32 82 us, 87 without; 4096 x 8192 x 512
    // bf16 42 and 45; f32 from planes, which lie there too, 109 and 103). Measured on products in a row, whose results
    // nobody reads; a reader of a result that would have stayed in the caches is not measured
    template <bool NT> __device__ __forceinline__ void store(const Out &o, v4f v) {
        t4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = (T)(o.beta != 0.f ? o.alpha * v[i] + o.beta * (float)old[i] : o.alpha * v[i]);
        if (n == 4) {
            typedef T any4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
            if constexpr (NT) __builtin_nontemporal_store((any4)r, (any4 *)c);
            else *(any4 *)c = (any4)r;
        } else {
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (i < n) c[i] = r[i];
        }
    }
};

// A range of memory for loads straight to LDS (16 bytes a lane, lane after lane from `lds`, which is the
// same for the wave). An offset at or past the range's end reads zeros; `soffset` is added to the address
// and does not count for that.
typedef __amdgpu_buffer_rsrc_t Buffer;
constexpr uint32_t OUTSIDE = 0x7FFFFFF0u;
__device__ __forceinline__ Buffer buffer(const void *p, uint32_t bytes) {
    // the same for the wave, which the compiler is told, or it loops over the lanes' descriptors
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000);
}
__device__ __forceinline__ void load_lds16(Buffer b, void *lds, uint32_t voffset, uint32_t soffset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (__attribute__((address_space(3))) void *)lds, 16, (int)voffset,
                                             (int)soffset, 0, 0);
}

__device__ __forceinline__ void load_lds4(Buffer b, void *lds, uint32_t voffset, uint32_t soffset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (__attribute__((address_space(3))) void *)lds, 4, (int)voffset,
                                             (int)soffset, 0, 0);
}
__device__ __forceinline__ v4u load16(Buffer b, uint32_t voffset, uint32_t soffset) {
    return __builtin_amdgcn_raw_buffer_load_b128(b, (int)voffset, (int)soffset, 0);
}
__device__ __forceinline__ v2u load8(Buffer b, uint32_t voffset, uint32_t soffset) {
    return __builtin_amdgcn_raw_buffer_load_b64(b, (int)voffset, (int)soffset, 0);
}
__device__ __forceinline__ uint32_t load4(Buffer b, uint32_t voffset, uint32_t soffset) {
    return __builtin_amdgcn_raw_buffer_load_b32(b, (int)voffset, (int)soffset, 0);
}
// All but this wave's last N loads have arrived. The compiler does not count loads to LDS for the reads of
// it, so their waits are written out; it leaves no load on the other side of one.
template <int N> __device__ __forceinline__ void wait_loads() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
    __builtin_amdgcn_sched_barrier(0);
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

// Scales as the tile kernel reads them: for 8 blocks of columns and 128 rows 1024 bytes, the scale of block k and
// row 32 f + r at byte 128 k + 4 r + f. A word then serves a lane's 4 operands, and a step's scales of a tile
// are contiguous; from their own rows, 8 bytes each, they cost more than all codes (8192^3 without the
// products: 162 us for the codes alone, 290 us with scales by rows). Zeros stand for what is not there.
constexpr int PACK_BLOCKS = 64;   // of columns a workgroup
struct PackJob {
    const uint8_t *src;
    int64_t lds, rows;
    uint32_t *dst;
};
int64_t pack_groups(const Mx4View &v) { return (v.rows + 127) / 128; }
size_t packed_scales(const Mx4View &v) { return (size_t)(pack_groups(v) * ((mx4_blocks(v.cols) + 7) / 8) * 1024); }

__global__ __launch_bounds__(256) void pack_scales_kernel(PackJob a, PackJob b, unsigned groups_a, int nb, int steps) {
    constexpr int PITCH = 132;   // bytes a block, so that those of a row are on different banks
    __shared__ __attribute__((aligned(16))) uint8_t packed[PACK_BLOCKS * PITCH];
    const PackJob &j = blockIdx.x < groups_a ? a : b;
    const int64_t group = blockIdx.x < groups_a ? blockIdx.x : blockIdx.x - groups_a, groups = (j.rows + 127) / 128;
    const int b0 = blockIdx.y * PACK_BLOCKS;
    const int w = threadIdx.x & 15, k0 = b0 + 4 * w;   // 16 threads a row, 4 scales each
    const bool words = (uintptr_t)j.src % 4 == 0 && j.lds % 4 == 0;
    const int64_t row0 = group * 128;
    uint32_t v[8];
    if (words) {   // all loads at once
        const int64_t left = j.rows - row0 < 128 ? j.rows - row0 : 128;
        const Buffer sb = buffer(j.src + row0 * j.lds, (uint32_t)((left - 1) * j.lds + (nb + 3) / 4 * 4));
        const uint32_t keep = nb - k0 >= 4 ? ~0u : nb > k0 ? (1u << (8 * (nb - k0))) - 1 : 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = load4(sb, k0 < nb ? (uint32_t)((i * 16 + (threadIdx.x >> 4)) * j.lds) + k0 : OUTSIDE, 0) & keep;
    } else {
        for (int i = 0; i < 8; ++i) {
            const int64_t row = row0 + i * 16 + (threadIdx.x >> 4);
            v[i] = 0;
            for (int q = 0; q < 4; ++q)
                if (row < j.rows && k0 + q < nb) v[i] |= (uint32_t)j.src[row * j.lds + k0 + q] << (8 * q);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = i * 16 + (threadIdx.x >> 4);
#pragma unroll
        for (int q = 0; q < 4; ++q) packed[(4 * w + q) * PITCH + (r & 31) * 4 + (r >> 5)] = (uint8_t)(v[i] >> (8 * q));
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PACK_BLOCKS * 32 / 256; ++i) {
        const int word = i * 256 + threadIdx.x, step = b0 / 8 + word / 256;   // 256 words a step
        if (step < steps) j.dst[((int64_t)step * groups + group) * 256 + (word & 255)] =
            ((const uint32_t *)packed)[word / 32 * (PITCH / 4) + word % 32];
    }
}

// this slice's partial sums as a result: [slice][no][np]
__device__ __forceinline__ Out partial_of(const Out &o, float *partial) {
    return Out{partial + (int64_t)blockIdx.y * o.np * o.no, o.np, o.np, o.no, 1.f, 0.f};
}

// A wave's WP x RO part of a result, RO rows of p after each other in LDS, to memory in whole lines: operands
// hold 4 consecutive entries of many rows, and stores of those are 16 bytes to a line. `pitch` words a row. What
// is there already is read some rows ahead of the stores.
template <typename T, int WP, int RO, int STEP, bool NT>
__device__ __forceinline__ void store_rows(const Out &o, const float *from, int pitch, int64_t p0, int64_t q0, int lane) {
    constexpr int L = WP / 4, R = 64 / L, N = RO / R, U = N < 16 ? N : 16;   // lanes a row, rows at once
    static_assert(WP % 4 == 0 && 64 % L == 0 && RO % R == 0 && N % U == 0, "whole rows");
    const int p = lane % L * 4, row = lane / L;
    const int have = (int)(o.no - q0 < RO * STEP ? o.no - q0 : RO * STEP);   // rows of the result from q0
    const int count = p0 + p >= o.np ? 0 : o.np - p0 - p < 4 ? (int)(o.np - p0 - p) : 4;
    T *c = (T *)o.ptr + (q0 + row * STEP) * o.ld + p0 + p;
    from += row * pitch + p;
#pragma unroll
    for (int r = 0; r < RO; r += U * R) {
        Four<T> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u].load(o, c + (r + u * R) * STEP * o.ld, (r + u * R + row) * STEP < have ? count : 0);
#pragma unroll
        for (int u = 0; u < U; ++u) x[u].template store<NT>(o, *(const v4f *)(from + (r + u * R) * pitch));
    }
}

// BP x BO entries of the result a workgroup, WP x WO a wave; 256 columns (8 blocks) of both factors a step,
// loaded straight to LDS, double-buffered. A row of a step is 128 bytes of codes, a whole line; its 16-byte
// blocks are kept at place block ^ (row / 2 & 7), which spreads the 16 rows that an access takes at once over
// all banks (the lane that fills a place loads the block that belongs there). The packed scales lie behind
// the codes.
// Bound by the power of the products (fed from registers alone 6.5 PFLOP/s): 8192^3 bf16 259 - 271 us on three cards with the
// scales' pass, 4.06 - 4.24 PFLOP/s. Short contractions are bound by the results' way to memory: 4096 x 4096 x 1024 f32 24 us, 2.9 TB/s.
template <typename T, int BP, int BO, int WP, int WO>
__global__ __launch_bounds__((BP / WP) * (BO / WO) * 64, 2) void both_tile_kernel(Mx4View P, Mx4View O, const uint8_t *ps, const uint8_t *os,
                                                                                  int nb, int steps_z, Out out, float *partial) {
    constexpr int NW = (BP / WP) * (BO / WO), NT = NW * 64;
    constexpr int FP = WP / 32, FO = WO / 32;
    constexpr int ROWS = BP + BO;                       // rows staged, P's first
    constexpr int LP = BP * 8 / NT, LO = BO * 8 / NT;   // 16-byte loads a thread
    static_assert(BP * 8 % NT == 0 && BO * 8 % NT == 0 && NT / 8 % 16 == 0, "whole loads, one block for all rows of a thread");
    constexpr int SL = ROWS / 128;                      // waves that load scales, 128 rows each
    static_assert(BP % 128 == 0 && BO % 128 == 0 && SL <= NW && 128 % WO == 0 && 128 % WP == 0, "scales by 128 rows");
    constexpr int STAGE = ROWS * 136, PITCH = WP + 4;
    constexpr int LDS = 2 * STAGE > NW * 32 * PITCH * 4 ? 2 * STAGE : NW * 32 * PITCH * 4;
    static_assert(LDS <= 160 * 1024, "LDS");
    __shared__ __attribute__((aligned(16))) uint8_t lds[LDS];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r32 = lane & 31, g = lane >> 5;
    uint32_t ip, io;
    tile_of(blockIdx.x, (uint32_t)((P.rows + BP - 1) / BP), (uint32_t)((O.rows + BO - 1) / BO), ip, io);
    const int64_t p0 = (int64_t)ip * BP, o0 = (int64_t)io * BO;
    const int wp = wave % (BP / WP), wo = wave / (BP / WP);
    // rows beyond the last one lie outside the ranges and read as zeros
    const int np = (int)(P.rows - p0 < BP ? P.rows - p0 : BP), no = (int)(O.rows - o0 < BO ? O.rows - o0 : BO);
    const Buffer pb = buffer(P.codes + p0 * P.ldq, (uint32_t)((np - 1) * P.ldq + nb * 16));
    const Buffer ob = buffer(O.codes + o0 * O.ldq, (uint32_t)((no - 1) * O.ldq + nb * 16));
    const int block = (tid & 7) ^ ((tid >> 4) & 7), steps = (nb + 7) / 8;
    const int t0 = blockIdx.y * steps_z, t1 = t0 + steps_z < steps ? t0 + steps_z : steps;   // this slice's
    const uint32_t vp = (uint32_t)((tid >> 3) * P.ldq) + block * 16, vo = (uint32_t)((tid >> 3) * O.ldq) + block * 16;
    const uint32_t rp = (uint32_t)P.ldq * (NT / 8), ro = (uint32_t)O.ldq * (NT / 8);
    // scales of this wave's 128 rows (of the first SL waves)
    const bool sp = wave * 128 < BP;
    const int64_t sg = ((sp ? P.rows : O.rows) + 127) / 128, s0 = sp ? p0 / 128 + wave : o0 / 128 + wave - BP / 128;
    const bool have = wave < SL && s0 < sg;
    const uint8_t *sbase = (sp ? ps : os) + (have ? s0 : 0) * 1024;
    // blocks 8 t .. 8 t + 7 of every row; those past the last are zero. Half h of the loads
    auto load = [&](int t, uint8_t *to, int h) {
        const bool in = t * 8 + block < nb;
        if (h == 0 && wave < SL) {
            const bool all = have && t < steps;
            load_lds16(buffer(sbase + (all ? t : 0) * sg * 1024, all ? 1024u : 0u), to + ROWS * 128 + wave * 1024, lane * 16, 0);
        }
#pragma unroll
        for (int i = h * LP / 2; i < (h + 1) * LP / 2; ++i) load_lds16(pb, to + (i * NT + wave * 64) * 16, in ? vp + i * rp : OUTSIDE, t * 128);
#pragma unroll
        for (int i = h * LO / 2; i < (h + 1) * LO / 2; ++i) load_lds16(ob, to + BP * 128 + (i * NT + wave * 64) * 16, in ? vo + i * ro : OUTSIDE, t * 128);
    };

    v16f acc[FP][FO];
#pragma unroll
    for (int a = 0; a < FP; ++a)
#pragma unroll
        for (int b = 0; b < FO; ++b) acc[a][b] = v16f{};

    // LDS places of this lane: one address a factor and quarter step, everything else an immediate
    int at[4];
#pragma unroll
    for (int h = 0; h < 4; ++h) at[h] = ((h * 2 + g) ^ ((r32 >> 1) & 7)) * 16 + r32 * 128;
    const int pa = wp * WP * 128, oa = (BP + wo * WO) * 128;
    const int psc = ROWS * 128 + (wp * WP) / 128 * 1024 + g * 128 + r32 * 4, pbit = wp * WP % 128 / 32 * 8;
    const int osc = ROWS * 128 + (BP + wo * WO) / 128 * 1024 + g * 128 + r32 * 4, obit = wo * WO % 128 / 32 * 8;
    struct Operands {
        v4i a[FP], b[FO];
        uint32_t sa, sb;
    };
    auto read = [&](const uint8_t *from, int h, Operands &x) {
        const uint8_t *ca = from + (pa + at[h]), *cb = from + (oa + at[h]);
        x.sa = *(const uint32_t *)(from + psc + h * 256) >> pbit;
        x.sb = *(const uint32_t *)(from + osc + h * 256) >> obit;
#pragma unroll
        for (int f = 0; f < FO; ++f) x.b[f] = *(const v4i *)(cb + f * 32 * 128);
#pragma unroll
        for (int f = 0; f < FP; ++f) x.a[f] = *(const v4i *)(ca + f * 32 * 128);
    };
    auto multiply = [&](const Operands &x) {
        static_for<FP>([&](auto fa) {
            static_for<FO>([&](auto fb) {
                constexpr int A = decltype(fa)::value, B = decltype(fb)::value;
                acc[A][B] = mfma_mx4_32<A, B>(x.a[A], x.b[B], acc[A][B], (int)x.sa, (int)x.sb);
            });
        });
    };
    load(t0, lds, 0);
    load(t0, lds, 1);
    arrive();
    int now = 0;
    for (int t = t0; t < t1; ++t) {
        // A quarter's products run beside the reads for the next one. The next step's loads go before the first
        // two: all at the start would keep the waves from their products until the last is issued, spread
        // over all four the last ones come late (8192^3: 301 and 298 us, this 278)
        Operands x[2];
        read(lds + now, 0, x[0]);
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            if (h < 2) load(t + 1, lds + STAGE - now, h);   // past the last step nothing but zeros
            if (h < 3) read(lds + now, h + 1, x[(h + 1) & 1]);
            __builtin_amdgcn_sched_barrier(0);
            multiply(x[h & 1]);
            __builtin_amdgcn_sched_barrier(0);
        }
        arrive();
        now = STAGE - now;
    }
    float *rows = (float *)lds + wave * 32 * PITCH;   // this wave's
#pragma unroll
    for (int b = 0; b < FO; ++b) {
#pragma unroll
        for (int a = 0; a < FP; ++a)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *(v4f *)(rows + r32 * PITCH + a * 32 + 8 * i + 4 * g) =
                    v4f{acc[a][b][4 * i], acc[a][b][4 * i + 1], acc[a][b][4 * i + 2], acc[a][b][4 * i + 3]};
        __builtin_amdgcn_wave_barrier();
        if (partial) store_rows<float, WP, 32, 1, false>(partial_of(out, partial), rows, PITCH, p0 + wp * WP, o0 + wo * WO + b * 32, lane);
        else store_rows<T, WP, 32, 1, true>(out, rows, PITCH, p0 + wp * WP, o0 + wo * WO + b * 32, lane);
        __builtin_amdgcn_wave_barrier();
    }
}

template <typename T, int BP, int BO, int WP, int WO>
hipError_t launch_both_tile(const Mx4View &P, const Mx4View &O, uint8_t *work, int slices, int steps_z, const Out &out, float *partial, hipStream_t s) {
    const int nb = (int)mx4_blocks(P.cols), steps = (nb + 7) / 8;
    uint8_t *ps = work, *os = work + packed_scales(P);
    const unsigned gp = (unsigned)pack_groups(P), go = (unsigned)pack_groups(O);
    hipLaunchKernelGGL(pack_scales_kernel, dim3(gp + go, (unsigned)((nb + PACK_BLOCKS - 1) / PACK_BLOCKS)), dim3(256), 0, s,
                       PackJob{P.scales, P.lds, P.rows, (uint32_t *)ps}, PackJob{O.scales, O.lds, O.rows, (uint32_t *)os}, gp, nb, steps);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int64_t tiles = ((P.rows + BP - 1) / BP) * ((O.rows + BO - 1) / BO);
    constexpr int NT = (BP / WP) * (BO / WO) * 64;
    hipLaunchKernelGGL((both_tile_kernel<T, BP, BO, WP, WO>), dim3((unsigned)tiles, (unsigned)slices), dim3(NT), 0, s, P, O, ps, os, nb, steps_z,
                       out, partial);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------------------------
// One dense and one 4-bit factor on the bf16 matrix instruction
// ---------------------------------------------------------------------------------------------
// A product of E2M1 and a power of two is a bf16 number, so the 4-bit factor enters exactly. The dense one
// enters as a sum of bf16 planes with all its bits: bf16 is one plane, f16 two (11 bits), f32 three (24
// bits, cut off from the top 8 at a time: each remainder is exact, and 3 bf16 products at 2.5 PFLOP/s are
// 5 times the f32 instruction's rate). The smallest bf16 is 2^-133, and what a f32 under 2^-110 has below that is
// left out. Sums are f32.
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

__device__ __forceinline__ v4f mfma_bf16(v4u a, v4u b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}
// 8 codes as bf16 times the scale, a float of which the exponent counts (0: 2^-127, 255: NaN)
__device__ __forceinline__ v4u decode_bf16(uint32_t w, float scale) {
    v4u r;
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
    return r;
}

// the same for the 4 of a half word
__device__ __forceinline__ v2u decode_bf16_4(uint32_t w, float scale) {
    v2u r;
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
    return r;
}

template <typename T> struct Planes { static constexpr int N = 1; };
template <> struct Planes<_Float16> { static constexpr int N = 2; };
template <> struct Planes<float> { static constexpr int N = 3; };

// x as a sum of bf16 numbers (their bits), without its bits below 2^-133; an infinity or a NaN is the first one alone
template <int PL> __device__ __forceinline__ void split(float x, uint32_t *b) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const bool finite = (u & 0x7F800000u) != 0x7F800000u;
    b[0] = u >> 16;
    if (!finite && (u & 0x7FFFFFu)) b[0] |= 0x40u;   // a NaN stays one without its low bits
    float r = x - __builtin_bit_cast(float, u & 0xFFFF0000u);
#pragma unroll
    for (int i = 1; i < PL; ++i) {
        const uint32_t v = __builtin_bit_cast(uint32_t, r);
        b[i] = finite ? v >> 16 : 0u;
        r = r - __builtin_bit_cast(float, v & 0xFFFF0000u);
    }
}
__device__ __forceinline__ uint32_t bf16_bits(__bf16 x) { return __builtin_bit_cast(unsigned short, x); }

// 8 elements of a row as 16 bytes of each plane
template <typename T> __device__ __forceinline__ void to_planes(const T (&v)[8], v4u (&w)[Planes<T>::N]) {
    constexpr int PL = Planes<T>::N;
    uint32_t b[8][PL];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (PL == 1) b[i][0] = bf16_bits(v[i]);
        else split<PL>((float)v[i], b[i]);
    }
#pragma unroll
    for (int q = 0; q < PL; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) w[q][i] = b[2 * i][q] | b[2 * i + 1][q] << 16;
}
// The planes of a dense factor in a workspace: plane i of element (r, c) at out[(i * rows + r) * ld + c], ld a
// multiple of 64, zeros behind the last column. One thread makes 8 columns of a row. Bound by HBM: 1001 x 8192 f32
// 13.5 us, 6.1 TB/s (with loads of single elements 20).
template <typename T>
__global__ __launch_bounds__(256) void planes_kernel(const T *__restrict__ x, int64_t stride, int64_t rows, int64_t cols,
                                                     int64_t ld, uint16_t *__restrict__ out) {
    constexpr int PL = Planes<T>::N;
    const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
    if (c >= ld) return;
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
        T v[8];
        if (c + 8 <= cols) {
            typedef T any8 __attribute__((ext_vector_type(8), aligned(sizeof(T))));
            const any8 m = *(const any8 *)(x + r * stride + c);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = m[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? x[r * stride + c + i] : (T)0.f;
        }
        v4u w[PL];
        to_planes(v, w);
#pragma unroll
        for (int q = 0; q < PL; ++q) *(v4u *)(out + ((int64_t)q * rows + r) * ld + c) = w[q];
    }
}
// The same for contiguous columns: 64 rows x 64 columns a workgroup, lanes along the rows, turned in LDS so that lines of
// 128 bytes are written whole (2400 x 7680 f32 31 us, 5.9 TB/s; pieces of 16 bytes to a row 65).
template <typename T>
__global__ __launch_bounds__(256) void planes_cols_kernel(const T *__restrict__ x, int64_t stride, int64_t rows, int64_t cols,
                                                          int64_t ld, uint16_t *__restrict__ out) {
    constexpr int PL = Planes<T>::N;
    __shared__ v4u tile[PL * 64 * 8];   // row's piece p at place p ^ row
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t r0 = (int64_t)blockIdx.x * 64, r = r0 + lane;
    for (int64_t c0 = (int64_t)blockIdx.y * 64; c0 < ld; c0 += (int64_t)gridDim.y * 64) {
        T v[2][8];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int64_t c = c0 + (wave + 4 * h) * 8 + i;
                v[h][i] = r < rows && c < cols ? x[c * stride + r] : (T)0.f;
            }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            v4u w[PL];
            to_planes(v[h], w);
#pragma unroll
            for (int q = 0; q < PL; ++q) tile[(q * 64 + lane) * 8 + ((wave + 4 * h) ^ (lane & 7))] = w[q];
        }
        __syncthreads();
        const int piece = threadIdx.x & 7;
#pragma unroll
        for (int q = 0; q < PL; ++q)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = (threadIdx.x >> 3) + 32 * h;
                if (r0 + row < rows) *(v4u *)(out + ((int64_t)q * rows + r0 + row) * ld + c0 + piece * 8) = tile[(q * 64 + row) * 8 + (piece ^ (row & 7))];
            }
        __syncthreads();
    }
}

// A dense factor as the product kernels read it: bf16 planes, rows of `chunks` 16-byte pieces, ld elements apart
struct Dense16 {
    const uint16_t *ptr;
    int64_t rows, ld, plane;
    int chunks;
};

// 4-bit values of 2^128 or more are infinities, as in other products of 32 bits. Where the dense factor is several planes,
// most numbers' lower ones are 0, and 0 times an infinity makes a NaN of a sum that is infinite. Every sum that this
// touches is a NaN, so the kernels look for one among their complete sums, then for scales under which infinities can
// be, and form those sums once more: with 0 for the infinite values of every plane but the first, which is 0 only with
// the number. That reads its operands from memory as they are needed: with an infinity in every sum 512 x 4096 x 4096 f32
// takes 690 us instead of 68, 16 x 4096 x 4096 81 and 17, with NaNs from elsewhere 63 and 17. Without a NaN the look
// at the sums is all that is added (-1 to 1.7 % over 36 sizes).
//
// Operands' places: a lane's row (yt: column) of the 4-bit factor is q, of the dense one d.
//
// The factors come from the kernel's arguments, which are read again for it: kept in scalar registers beside the loop
// they push others' loads behind it (some kernels 1 us longer).
struct Factors {   // how the arguments of every kernel that has planes begin
    Dense16 D;
    Mx4View Y;
};
static_assert(sizeof(Dense16) % alignof(Mx4View) == 0, "arguments lie as the members do");
__device__ __forceinline__ const Factors &factors_again() {
    auto p = __builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const Factors *)(const void *)p;
}
__device__ __forceinline__ v4u finite_or_0(v4u q) {
    v4u r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r[i] = (q[i] & 0x7F80u) == 0x7F80u ? q[i] & 0xFFFF0000u : q[i];
        r[i] = (q[i] & 0x7F800000u) == 0x7F800000u ? r[i] & 0xFFFFu : r[i];
    }
    return r;
}
// sum += q d over k0 <= k < k1, k0 a multiple of 32
template <bool YT, bool QFIRST, int PL>
__device__ __forceinline__ v4f add_finite(v4f sum, const Factors &x, int64_t q, int64_t d, int64_t k0, int64_t k1, int g) {
    const Mx4View &Y = x.Y;
    const Dense16 &D = x.D;
#pragma unroll 1
    for (int64_t k = k0; k < k1; k += 32) {   // lane group g: elements k + 8 g .. + 7
        v4u w{};
        if constexpr (YT) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int64_t row = k + 8 * g + j;
                const bool in = row < k1 && q < Y.cols;
                const uint8_t *const code = Y.codes + (in ? row * Y.ldq + q / 2 : 0), *const scale = Y.scales + (in ? row * Y.lds + q / 32 : 0);
                const uint32_t v = decode_bf16_4((uint32_t)*code >> (q % 2 * 4), __builtin_bit_cast(float, (uint32_t)*scale << 23))[0];
                w[j / 2] |= (in ? v & 0xFFFFu : 0u) << (j % 2 * 16);
            }
        } else if (q < Y.rows && k < Y.cols) {
            const uint32_t scale = Y.scales[q * Y.lds + k / 32];
            w = decode_bf16(*(const uint32_t *)(Y.codes + q * Y.ldq + k / 2 + 4 * g), __builtin_bit_cast(float, scale << 23));
        }
        const int64_t piece = k / 8 + g;
#pragma unroll
        for (int p = 0; p < PL; ++p) {
            const v4u v = d < D.rows && piece < D.chunks ? *(const v4u *)(D.ptr + p * D.plane + d * D.ld + piece * 8) : v4u{};
            const v4u wp = p ? finite_or_0(w) : w;
            sum = QFIRST ? mfma_bf16(wp, v, sum) : mfma_bf16(v, wp, sum);
        }
    }
    return sum;
}
// Whether a scale of 2^126 or 2^127 is among those of `count` rows (columns) of the 4-bit factor from q0, k0 <= k < k1 of
// the contraction; q0 (across) or k0 is a multiple of 128, scales are read by words of 4
template <bool YT> __device__ __forceinline__ bool infinities(const Mx4View &Y, int64_t q0, int count, int64_t k0, int64_t k1, int lane) {
    uint32_t found = 0;
    const int64_t q1 = q0 + count, rows = YT ? k1 : q1 < Y.rows ? q1 : Y.rows, cols = YT ? (q1 < Y.cols ? q1 : Y.cols) : k1;
    auto has_0 = [](uint32_t w) { return (w - 0x01010101u) & ~w & 0x80808080u; };   // not 0 if a byte is
    for (int64_t r = (YT ? k0 : q0) + lane; r < rows; r += 64)
#pragma unroll 8
        for (int64_t b = (YT ? q0 : k0) / 32; b < mx4_blocks(cols); b += 4) {
            const uint32_t w = *(const uint32_t *)(Y.scales + r * Y.lds + b);
            found |= has_0(w ^ 0xFDFDFDFDu) | has_0(w ^ 0xFEFEFEFEu);
        }
    return __any(found != 0);
}
__device__ __forceinline__ bool any_nan(v4f x, bool counts) {
    const float sum = (x[0] + x[1]) + (x[2] + x[3]);   // a NaN if one of them is
    return __builtin_expect(__any(sum != sum && counts), 0);
}
// A wave's operands of a tile: those of the 4-bit factor are qf apart, a lane's row (column) of one is ql times r16
template <bool YT, bool QFIRST, int PL, int FQ, int FD>
__device__ __forceinline__ void mend_tile(v4f (&acc)[FQ][FD], int64_t q0, int qf, int ql, int64_t d0, int64_t k0,
                                          int64_t k1, int lane) {
    v4f total = acc[0][0];
#pragma unroll
    for (int i = 1; i < FQ * FD; ++i) total += acc[i / FD][i % FD];
    if (!any_nan(total, true)) return;
    const Factors &x = factors_again();
    // blocks across: the words that the wave's two blocks are in
    if (!infinities<YT>(x.Y, YT ? q0 & -128 : q0, YT ? 128 : FQ * 16, k0, k1, lane)) return;
#pragma unroll 1
    for (int i = 0; i < FQ * FD; ++i) {
        v4f old = acc[0][0];
#pragma unroll
        for (int j = 1; j < FQ * FD; ++j) old = i == j ? acc[j / FD][j % FD] : old;
        if (!any_nan(old, true)) continue;
        const v4f sum = add_finite<YT, QFIRST, PL>(v4f{}, x, q0 + i / FD * qf + (lane & 15) * ql, d0 + i % FD * 16 + (lane & 15), k0, k1, lane >> 4);
#pragma unroll
        for (int j = 0; j < FQ * FD; ++j) acc[j / FD][j % FD] = i == j ? sum : acc[j / FD][j % FD];
    }
}

// A wave's part of the result to memory by way of LDS (16 rows of the second index at a time, `rows` this wave's
// place), q0 and d0 its first entry. Entry i of a lane's 4 is row 4 g + i of the first operand; with YT the 4-bit
// index of row r of operand f is 4 r + f.
template <typename T, bool YT, bool QFIRST, int FQ, int FD>
__device__ __forceinline__ void store_wave(const v4f (&acc)[FQ][FD], float *rows, const Out &out, float *partial, int64_t q0, int64_t d0, int lane) {
    constexpr int W1 = (QFIRST ? FQ : FD) * 16, PITCH = W1 + 4, STEP = YT && !QFIRST ? 4 : 1;
    static_assert(!YT || FQ == 4, "4 columns a lane");
    const int r16 = lane & 15, g = lane >> 4;
    const int64_t n1 = QFIRST ? q0 : d0;
    auto out_rows = [&](int64_t n2) {
        __builtin_amdgcn_wave_barrier();
        if (partial) store_rows<float, W1, 16, STEP, false>(partial_of(out, partial), rows, PITCH, n1, n2, lane);
        else store_rows<T, W1, 16, STEP, sizeof(T) == 2>(out, rows, PITCH, n1, n2, lane);
        __builtin_amdgcn_wave_barrier();
    };
    if constexpr (QFIRST) {
#pragma unroll
        for (int fd = 0; fd < FD; ++fd) {
            float *to = rows + r16 * PITCH;
            if constexpr (YT) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *(v4f *)(to + (4 * g + i) * 4) = v4f{acc[0][fd][i], acc[1][fd][i], acc[2][fd][i], acc[3][fd][i]};
            } else {
#pragma unroll
                for (int fq = 0; fq < FQ; ++fq) *(v4f *)(to + fq * 16 + 4 * g) = acc[fq][fd];
            }
            out_rows(d0 + fd * 16);
        }
    } else {
#pragma unroll
        for (int fq = 0; fq < FQ; ++fq) {
#pragma unroll
            for (int fd = 0; fd < FD; ++fd) *(v4f *)(rows + r16 * PITCH + fd * 16 + 4 * g) = acc[fq][fd];
            out_rows(q0 + (YT ? fq : fq * 16));
        }
    }
}
// LDS that the tile kernels' results pass through
constexpr int store_bytes(int waves, int wq, int wd, bool qfirst) { return waves * 16 * ((qfirst ? wq : wd) + 4) * 4; }

// acc += q d over 32 elements of the contraction, every plane
template <bool QFIRST, int FQ, int FD, int PL>
__device__ __forceinline__ void multiply_bf16(v4f (&acc)[FQ][FD], const v4u (&q)[FQ], const v4u (&d)[PL][FD]) {
#pragma unroll
    for (int fq = 0; fq < FQ; ++fq)
#pragma unroll
        for (int p = 0; p < PL; ++p)
#pragma unroll
            for (int fd = 0; fd < FD; ++fd)
                acc[fq][fd] = QFIRST ? mfma_bf16(q[fq], d[p][fd], acc[fq][fd]) : mfma_bf16(d[p][fd], q[fq], acc[fq][fd]);
}

// The dense factor's side of a tile: BD rows, 64 elements of the contraction a step, straight to LDS as rows of
// 128 bytes, a plane after the other. Where 16-byte pieces of a row are kept: the lanes that a read takes at once are rows
// 0 - 3 and 12 - 15 of one lane group and rows 4 - 11 of the next one, whose pieces differ in bit 1. XOR with row / 2
// puts the one on the other's banks, XOR with a map of it that sends 12 to 2 does not (bank conflicts 8.6 million and
// 0.1 million). The latter is faster with blocks along the contraction (4096 x 8192 x 4096, calls in a row: 231 and 240 us)
// and slower with blocks across (SPREAD off; 2048 x 4096 x 8192: 137 and 132).
template <int PL, int BD, int NT, bool SPREAD> struct DenseTile {
    static constexpr int LD = BD * 8 / NT, BYTES = PL * BD * 128, LOADS = PL * LD;
    static_assert(BD * 8 % NT == 0 && NT / 8 % 16 == 0, "whole loads of the dense rows");
    Buffer db[PL];
    uint32_t vd, rd;
    int piece, chunks, wave;
    static __device__ __forceinline__ int place(int piece, int row) {
        return SPREAD ? piece ^ (row >> 1 & 1) ^ (row & 4) ^ (row & 8 ? 6 : 0) : piece ^ (row >> 1 & 7);
    }
    __device__ __forceinline__ DenseTile(const Dense16 &D, int64_t d0, int tid, int w) : chunks(D.chunks), wave(w) {
        const int nd = (int)(D.rows - d0 < BD ? D.rows - d0 : BD);
#pragma unroll
        for (int i = 0; i < PL; ++i) db[i] = buffer(D.ptr + i * D.plane + d0 * D.ld, (uint32_t)((nd - 1) * D.ld * 2 + D.chunks * 16));
        piece = place(tid & 7, tid >> 3);
        vd = (uint32_t)((tid >> 3) * D.ld * 2) + piece * 16;
        rd = (uint32_t)(D.ld * 2) * (NT / 8);
    }
    // half h of the loads, or all of them
    __device__ __forceinline__ void load(int step, uint8_t *to, int h = 2) const {
        static_assert(LD % 2 == 0, "halves");
        const bool in = step * 8 + piece < chunks;   // past the last step zeros
#pragma unroll
        for (int p = 0; p < PL; ++p)
#pragma unroll
            for (int i = h == 1 ? LD / 2 : 0; i < (h == 0 ? LD / 2 : LD); ++i)
                load_lds16(db[p], to + (p * BD * 8 + i * NT + wave * 64) * 16, in ? vd + i * rd : OUTSIDE, step * 128);
    }
    // operands of instruction t of a step, for 16 FD rows from `row`
    template <int FD> static __device__ __forceinline__ void read(const uint8_t *from, int row, int t, int lane, v4u (&d)[PL][FD]) {
        const int r16 = lane & 15, g = lane >> 4;
        const uint8_t *dp = from + row * 128 + r16 * 128 + place(g * 2 + t, r16) * 16;
#pragma unroll
        for (int p = 0; p < PL; ++p)
#pragma unroll
            for (int f = 0; f < FD; ++f) d[p][f] = *(const v4u *)(dp + (p * BD + f * 16) * 128);
    }
};

// BQ rows of a 4-bit factor whose blocks lie along the contraction x BD rows of the dense one a workgroup, WQ x
// WD a wave; 64 elements of the contraction a step, loaded straight to LDS, double-buffered.
//
// A step's two matrix instructions take their 32 elements from all over the 64: lane group g holds
// elements 16 g + 8 t .. + 7 of both factors for instruction t, so a lane's 16 codes lie in one word pair
// and under one scale. Codes come SS steps at once, 256 elements, so that rows are whole lines of 128 bytes (128
// where LDS is short), the next ones a part of the rows a step; 16-byte blocks at place
// block ^ (row / 2), the rows' scales behind them.
//
// 256 x 256 tiles are bound by the products and their power: 4096 x 8192 x 4096 bf16 197 - 206 us on several cards, 1.33 -
// 1.39 PFLOP/s (a large bf16 product by the library: 1.35); 4096 x 1001 x 8192 f32, three planes, 165 - 173 us with
// their pass, 1.17 - 1.22.
template <typename T, int PL, int BQ, int BD, int WQ, int WD, bool QFIRST>
__global__ __launch_bounds__((BQ / WQ) * (BD / WD) * 64, 2) void mixed_tile_kernel(Dense16 D, Mx4View Y, int64_t K, int steps_z,
                                                                                   Out out, float *partial) {
    constexpr int NW = (BQ / WQ) * (BD / WD), NT = NW * 64;
    constexpr int FQ = WQ / 16, FD = WD / 16;
    typedef DenseTile<PL, BD, NT, true> Dense;
    constexpr int CW = BQ / 32;   // waves that load codes, one load a thread
    static_assert(CW <= NW, "waves that load codes");
    constexpr int STAGE = Dense::BYTES;
    // codes and scales of SS steps at a time
    constexpr int SS = 2 * (STAGE + BQ * 136) > 160 * 1024 ? 2 : 4, NP = 2 * SS, SUPER = BQ * 34 * SS;
    constexpr int RING = 2 * (STAGE + SUPER), STORE = store_bytes(NW, WQ, WD, QFIRST), LDS = RING > STORE ? RING : STORE;
    static_assert(LDS <= 160 * 1024, "LDS");
    __shared__ __attribute__((aligned(16))) uint8_t lds[LDS];
    uint8_t *const lds0 = lds, *const lds1 = lds + STAGE, *const supers = lds + 2 * STAGE;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    uint32_t iq, id;
    tile_of(blockIdx.x, (uint32_t)((Y.rows + BQ - 1) / BQ), (uint32_t)((D.rows + BD - 1) / BD), iq, id);
    const int64_t q0 = (int64_t)iq * BQ, d0 = (int64_t)id * BD;
    const int wq = wave % (BQ / WQ), wd = wave / (BQ / WQ);
    const int mq = (int)(Y.rows - q0 < BQ ? Y.rows - q0 : BQ);
    const int steps = (int)((K + 63) / 64), s0 = blockIdx.y * steps_z, s1 = s0 + steps_z < steps ? s0 + steps_z : steps;

    const Dense dense(D, d0, tid, wave);
    const int nb = (int)mx4_blocks(Y.cols);
    const Buffer qb = buffer(Y.codes + q0 * Y.ldq, (uint32_t)((mq - 1) * Y.ldq + nb * 16));
    const Buffer sb = buffer(Y.scales + q0 * Y.lds, (uint32_t)((mq - 1) * Y.lds + (nb + 3) / 4 * 4));
    const int qpart = (tid % NP) ^ ((tid >> 4) % NP);
    const uint32_t vq = (uint32_t)((tid / NP) * Y.ldq) + qpart * 16;
    const uint32_t vs = (uint32_t)((tid / (SS / 2)) * Y.lds) + tid % (SS / 2) * 4;
    // part c (of the rows) of codes and scales u
    auto load_super = [&](int u, int c) {
        uint8_t *to = supers + (u & 1) * SUPER;
        if (wave < CW)
            load_lds16(qb, to + (c * CW + wave) * 1024, u * NP + qpart < nb ? vq + (uint32_t)(c * (BQ / SS) * Y.ldq) : OUTSIDE, u * NP * 16);
        if (wave < BQ / 128)
            load_lds4(sb, to + BQ * 32 * SS + (c * (BQ / 2) + wave * 64) * 4,
                      u * NP + tid % (SS / 2) * 4 < nb ? vs + (uint32_t)(c * (BQ / SS) * Y.lds) : OUTSIDE, u * NP);
    };

    v4f acc[FQ][FD];
#pragma unroll
    for (int a = 0; a < FQ; ++a)
#pragma unroll
        for (int b = 0; b < FD; ++b) acc[a][b] = v4f{0.f, 0.f, 0.f, 0.f};

    auto compute = [&](int step, const uint8_t *from) {
        v2u raw[FQ];
        float scale[FQ];
        const int c = step % SS;
        const uint8_t *super = supers + (step / SS & 1) * SUPER;
        const uint8_t *cq = super + ((wq * WQ + r16) * 32 * SS + (((c * 2 + (g >> 1)) ^ ((r16 * NP >> 4) % NP)) * 16) + (g & 1) * 8);
        const uint8_t *sq = super + (BQ * 32 * SS + (wq * WQ + r16) * 2 * SS + (c >> 1) * 4);
        const int bit = (c & 1) * 16 + (g >> 1) * 8;
        const uint32_t width = step * 2 + (g >> 1) < nb ? 8 : 0;   // past the last block, whatever is there, as 0
#pragma unroll
        for (int f = 0; f < FQ; ++f) {
            raw[f] = *(const v2u *)(cq + f * 16 * 32 * SS);
            scale[f] = __builtin_bit_cast(float, __builtin_amdgcn_ubfe(*(const uint32_t *)(sq + f * 16 * 2 * SS), bit, width) << 23);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            v4u d[PL][FD], q[FQ];
            Dense::read(from, wd * WD, t, lane, d);
#pragma unroll
            for (int f = 0; f < FQ; ++f) q[f] = decode_bf16(raw[f][t], scale[f]);
            multiply_bf16<QFIRST>(acc, q, d);
        }
    };
#pragma unroll
    for (int c = 0; c < SS; ++c) load_super(s0 / SS, c);   // slices start at multiples of 4 steps
    dense.load(s0, lds0);
    arrive();
    int st = s0;
    for (; st + 1 < s1; st += 2) {
        load_super(st / SS + 1, st % SS);
        dense.load(st + 1, lds1);
        __builtin_amdgcn_sched_barrier(0);
        compute(st, lds0);
        arrive();
        load_super((st + 1) / SS + 1, (st + 1) % SS);
        dense.load(st + 2, lds0);
        __builtin_amdgcn_sched_barrier(0);
        compute(st + 1, lds1);
        arrive();
    }
    if (st < s1) compute(st, lds0);
    if constexpr (PL > 1)
        mend_tile<false, QFIRST, PL>(acc, q0 + wq * WQ, 16, 1, d0 + wd * WD, s0 * 64, s1 * 64 < K ? s1 * 64 : K, lane);
    __syncthreads();
    store_wave<T, false, QFIRST>(acc, (float *)lds + wave * (STORE / NW / 4), out, partial, q0 + wq * WQ, d0 + wd * WD, lane);
}

// The same with blocks across the contraction: BQ columns of the 4-bit factor, 64 of them a wave. A lane takes half
// a word (4 columns 4 c .. + 3) of 8 rows, decodes it under the 8 rows' scales and exchanges halves of words
// between rows; its 4 operands are then columns 4 c + f, and the operand f of the wave is columns f, f + 4, .. --
// an order of the result's rows or columns that the stores undo.
//
// The 32 elements of a lane's operands cost 40 instructions in every wave that decodes them (16 conversions, 16 permutations,
// 8 scales), about as long as their products take, so the two have to run at the same time: a wave decodes the next
// instruction's operands among the present one's products, also across steps. For that the codes are one step further ahead than the dense rows, which are two
// steps ahead (one where LDS is short), and the wait of a step leaves its own loads on their way.
// Scales go to LDS through registers, a block's after each other; the decoding instruction looks at a float's exponent
// only, so a shift of the word brings a scale there.
// 2048 x 4096 x 8192 bf16 (256 x 128 tiles) 120 - 129 us on several cards, 1.07 - 1.15 PFLOP/s, without the operands ahead and with
// 8 bytes' scales by two reads 146 beside 122; bound by the decoding beside the products and the reads from LDS.
template <typename T, int PL, int BQ, int BD, int WD, bool QFIRST>
__global__ __launch_bounds__((BQ / 64) * (BD / WD) * 64, 2) void mixed_tile_yt_kernel(Dense16 D, Mx4View Y, int64_t K, int steps_z,
                                                                                      Out out, float *partial) {
    constexpr int NW = (BQ / 64) * (BD / WD), NT = NW * 64, FQ = 4, FD = WD / 16;
    typedef DenseTile<PL, BD, NT, false> Dense;
    constexpr int PR = BQ / 32, CW = BQ / 32, WR = BQ / 128;   // 16-byte pieces a row; waves that load codes, scales
    static_assert(CW <= NW, "waves that load codes");
    constexpr int PITCH = BQ == 256 ? 1056 : 1088, ROW = BQ / 2;   // 64 lanes' codes; lane groups on different banks
    constexpr int CODES = CW * PITCH + PR * 64;
    constexpr int STAGE = Dense::BYTES + CODES, DS = 3 * STAGE <= 160 * 1024 ? 3 : 2;   // steps held
    constexpr int RING = DS * STAGE, STORE = store_bytes(NW, 64, WD, QFIRST), LDS = RING > STORE ? RING : STORE;
    static_assert(LDS <= 160 * 1024, "LDS");
    __shared__ __attribute__((aligned(16))) uint8_t lds[LDS];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    uint32_t iq, id;
    tile_of(blockIdx.x, (uint32_t)((Y.cols + BQ - 1) / BQ), (uint32_t)((D.rows + BD - 1) / BD), iq, id);
    const int64_t q0 = (int64_t)iq * BQ, d0 = (int64_t)id * BD;
    const int wq = wave % (BQ / 64), wd = wave / (BQ / 64);
    const int steps = (int)((K + 63) / 64), s0 = blockIdx.y * steps_z, s1 = s0 + steps_z < steps ? s0 + steps_z : steps;

    const Dense dense(D, d0, tid, wave);
    const int nb = (int)mx4_blocks(Y.cols - q0 < BQ ? Y.cols - q0 : BQ);   // blocks of a row here
    const int qpart = lane % PR;
    const uint32_t vq = qpart < nb ? (uint32_t)((wave * (64 / PR) + lane / PR) * Y.ldq) + qpart * 16 : OUTSIDE;
    const uint32_t vs = wave * 4 < nb ? (uint32_t)(lane * Y.lds) + wave * 4 : OUTSIDE;
    uint32_t sreg = 0;   // a row's scales of 4 blocks on their way to LDS
    // behind the last block 0, whatever is there: sums that are not stored are to be no NaN for that
    const uint32_t keep = nb - wave * 4 >= 4 ? ~0u : nb > wave * 4 ? (1u << (8 * (nb - wave * 4))) - 1 : 0u;
    auto put_scales = [&](uint8_t *to) {
        if constexpr (PL > 1) sreg &= keep;
#pragma unroll
        for (int i = 0; i < 4; ++i) to[Dense::BYTES + CW * PITCH + (wave * 4 + i) * 64 + lane] = (uint8_t)(sreg >> (8 * i));
    };
    // where the next step to be loaded begins, and how many rows are left there; past the last an empty range
    // reads zeros
    const uint32_t ldq = __builtin_amdgcn_readfirstlane((int)Y.ldq), ldk = __builtin_amdgcn_readfirstlane((int)Y.lds);
    const uint32_t code_bytes = nb * 16, scale_bytes = (nb + 3) / 4 * 4;   // of a row
    const uint8_t *cp = Y.codes + q0 / 2 + (int64_t)s0 * 64 * Y.ldq, *kp = Y.scales + q0 / 32 + (int64_t)s0 * 64 * Y.lds;
    int left = (int)K - s0 * 64;
    auto load_codes = [&](uint8_t *to) {
        const uint32_t rows = left < 64 ? left : 64;
        if (wave < WR) sreg = load4(buffer(kp, left > 0 ? (rows - 1) * ldk + scale_bytes : 0u), vs, 0);
        if (CW == NW || wave < CW)
            load_lds16(buffer(cp, left > 0 ? (rows - 1) * ldq + code_bytes : 0u), to + Dense::BYTES + wave * PITCH, vq, 0);
        cp += (uint64_t)ldq * 64;
        kp += (uint64_t)ldk * 64;
        left -= 64;
    };
    // The next step's loads have arrived, those of DS - 2 steps behind it may be on their way, but for the scales. The
    // barrier alone: __syncthreads would wait for all of them; what was read from LDS is in use already.
    auto next = [&](uint8_t *scales_to) {
        if (wave < WR) {
            wait_loads<DS == 2 ? 0 : Dense::LOADS + 1>();
            put_scales(scales_to);
        } else if (DS == 2) wait_loads<0>();
        else if (CW == NW || wave < CW) wait_loads<Dense::LOADS + 1>();
        else wait_loads<Dense::LOADS>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };

    v4f acc[FQ][FD];
#pragma unroll
    for (int a = 0; a < FQ; ++a)
#pragma unroll
        for (int b = 0; b < FD; ++b) acc[a][b] = v4f{0.f, 0.f, 0.f, 0.f};

    struct Raw {
        uint32_t c[8];
        v2u s;
    };
    auto read_codes = [&](const uint8_t *from, int t, Raw &x) {
        const uint8_t *cq = from + (Dense::BYTES + (BQ == 256 ? (g * 2 + t) * PITCH : g * PITCH + t * 8 * ROW) + wq * 32 + r16 * 2);
        x.s = *(const v2u *)(from + (Dense::BYTES + CW * PITCH + (wq * 2 + (r16 >> 3)) * 64 + 16 * g + 8 * t));
#pragma unroll
        for (int j = 0; j < 8; ++j) x.c[j] = *(const uint16_t *)(cq + j * ROW);
    };
    // byte i of a word to a float's exponent
    auto exponent = [](uint32_t w, int i) { return __builtin_bit_cast(float, i < 3 ? w << (23 - 8 * i) : w >> 1); };
    auto decode = [&](const Raw &x, v4u (&q)[FQ]) {
        v2u row[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            row[j] = decode_bf16_4(x.c[j], exponent(x.s[j >> 2], j & 3));
#pragma unroll
        for (int f = 0; f < FQ; ++f)
#pragma unroll
            for (int j = 0; j < 4; ++j)   // rows 2 j, 2 j + 1 of column f
                q[f][j] = __builtin_amdgcn_perm(row[2 * j + 1][f >> 1], row[2 * j][f >> 1], (f & 1) ? 0x07060302u : 0x05040100u);
    };
    struct Operands {
        v4u q[FQ], d[PL][FD];
    };
    // the products of `now`; among them the next operands (of instruction t) are read and decoded, and half of a
    // step's dense rows is sent for
    auto half = [&](const Operands &now, Operands &next, const uint8_t *from, int t, int step, uint8_t *to) {
        Raw x;
        read_codes(from, t, x);
        Dense::read(from, wd * WD, t, lane, next.d);
        dense.load(step, to, t);
        multiply_bf16<QFIRST>(acc, now.q, now.d);
        decode(x, next.q);
        constexpr int M = FQ * FD * PL, V = 40, L = Dense::LOADS / 2;   // matrix instructions, others, loads
        __builtin_amdgcn_sched_group_barrier(0x100, PL * FD + 9, 0);
#pragma unroll
        for (int i = 0; i < M; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
            if (i >= 3) __builtin_amdgcn_sched_group_barrier(0x2, (V + M - 4) / (M - 3), 0);
            if (i % (M / L) == M / L - 1) __builtin_amdgcn_sched_group_barrier(0x20, 1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int f = 0; f < FQ; ++f) asm volatile("" : "+v"(next.q[f]));   // here, and not behind the step's barrier
    };
#pragma unroll
    for (int i = 0; i < DS; ++i) {
        load_codes(lds + i * STAGE);
        if (wave < WR) put_scales(lds + i * STAGE);
        if (i < DS - 1) dense.load(s0 + i, lds + i * STAGE);
        else dense.load(s0 + i, lds + i * STAGE, 0);   // the other half goes with the first products
    }
    arrive();
    Operands a, b;
    {
        Raw x;
        read_codes(lds, 0, x);
        Dense::read(lds, wd * WD, 0, lane, a.d);
        decode(x, a.q);
    }
    // A step's first operands are read during the step before, its second ones during its own first half; then all
    // waves are done with its place, and the step DS further on goes there.
    int at = 0, last = (DS - 1) * STAGE;   // places of this step and of the one before
    for (int st = s0; st < s1; ++st) {
        half(a, b, lds + at, 1, st + DS - 1, lds + last);
        next(lds + last);
        load_codes(lds + at);
        __builtin_amdgcn_sched_barrier(0);
        last = at;
        at = at == (DS - 1) * STAGE ? 0 : at + STAGE;
        half(b, a, lds + at, 0, st + DS, lds + last);
    }
    if constexpr (PL > 1)
        mend_tile<true, QFIRST, PL>(acc, q0 + wq * 64, 1, 4, d0 + wd * WD, s0 * 64, s1 * 64 < K ? s1 * 64 : K, lane);
    arrive();   // nothing is on its way to LDS any more
    store_wave<T, true, QFIRST>(acc, (float *)lds + wave * (STORE / NW / 4), out, partial, q0 + wq * 64, d0 + wd * WD, lane);
}

// Few dense rows (at most 16 DF): a workgroup takes NQ columns of the result over one slice of the
// contraction, its 8 waves take the slice's units in turn, and each wave streams its codes from memory
// straight to registers, so nothing but the codes' bytes bounds it: every load of a unit is issued before the
// one before it is used, and no barrier stands between them. The waves' sums are added in LDS, in order.
//   blocks along the contraction: unit of 256 elements; lane (r, g) holds blocks 2 g and 2 g + 1 of row r
//   blocks across it (YT): unit of 32 rows and 256 columns; lane (c, g) holds columns 16 c .. + 15 of rows
//     8 g .. + 7 (128 bytes of a row, whole lines, are read by 16 lanes together)
// entry (q, d) of the result at ptr[q * sq + d * sd]; partial sums where `partial` is set
struct RowsOut {
    void *ptr;
    int64_t sq, sd, nq, nd;
    float alpha, beta;
    float *partial;
};
template <typename T> __device__ __forceinline__ void put1(const RowsOut &o, int64_t q, int64_t d, float v) {
    if (q >= o.nq || d >= o.nd) return;
    if (o.partial) {
        o.partial[(int64_t)blockIdx.y * o.nq * o.nd + q * o.sq + d * o.sd] = v;
    } else {
        T *c = (T *)o.ptr + q * o.sq + d * o.sd;
        *c = (T)(o.beta != 0.f ? o.alpha * v + o.beta * (float)*c : o.alpha * v);
    }
}

constexpr int ROWS_WAVES = 8;
// with dense rows in LDS: as many waves as it holds buffers for
__host__ __device__ constexpr int dense_waves(int planes) { return planes <= 2 ? 8 : 4; }

// adds the W waves' N operands and hands each sum to f(operand, lane, value)
template <int W, int N, typename F> __device__ __forceinline__ void add_waves(const v4f *acc, v4f *lds, int lane, int wave, F &&f) {
    constexpr int C = N < W ? N : W;
    static_assert(N % C == 0, "whole rounds");
#pragma unroll
    for (int r = 0; r < N; r += C) {
        if (r) __syncthreads();
#pragma unroll
        for (int i = 0; i < C; ++i) lds[(wave * C + i) * 64 + lane] = acc[r + i];
        __syncthreads();
        if (wave < C) {
            v4f sum = lds[wave * 64 + lane];
#pragma unroll
            for (int w = 1; w < W; ++w) sum += lds[(w * C + wave) * 64 + lane];
            f(r + wave, lane, sum);
        }
    }
}

// 16 NF rows of a 4-bit factor from row0 in one unit of 128 H columns: lane (r, g) holds the H blocks H g ..
// of row r of each 16 and the word that their scales are in. What lies behind the last block or row reads
// as zeros.
template <int NF, int H> struct RowCodes {
    v4u c[NF][H];
    uint32_t s[NF];
};
template <int NF, int H> struct RowReader {
    Buffer cb, sb;
    uint32_t co[NF], so[NF];
    int nb, g;
    __device__ __forceinline__ RowReader(const Mx4View &V, int64_t row0, int r16, int group) : nb((int)mx4_blocks(V.cols)), g(group) {
        const int64_t left = V.rows - row0 < NF * 16 ? V.rows - row0 : NF * 16;
        cb = buffer(V.codes + row0 * V.ldq, (uint32_t)((left - 1) * V.ldq + nb * 16));
        sb = buffer(V.scales + row0 * V.lds, (uint32_t)((left - 1) * V.lds + (nb + 3) / 4 * 4));
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            co[f] = (uint32_t)((f * 16 + r16) * V.ldq) + 16 * H * g;
            so[f] = (uint32_t)((f * 16 + r16) * V.lds) + (H * g / 4) * 4;
        }
    }
    __device__ __forceinline__ int block(int u, int h) const { return (u * 4 + g) * H + h; }
    __device__ __forceinline__ void load(int u, RowCodes<NF, H> &x) const {
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int f = 0; f < NF; ++f) x.c[f][h] = load16(cb, block(u, h) < nb ? co[f] + 16 * h : OUTSIDE, u * 64 * H);
#pragma unroll
        for (int f = 0; f < NF; ++f) x.s[f] = load4(sb, block(u, 0) < nb ? so[f] : OUTSIDE, u * 4 * H);
    }
    // the scale of this lane's block h of unit u; past the last block 0, whatever is there
    __device__ __forceinline__ uint32_t scale(int u, int h, uint32_t word) const {
        return __builtin_amdgcn_ubfe(word, 8 * ((g * H + h) & 3), block(u, h) < nb ? 8 : 0);
    }
};

// The dense rows of a unit go through LDS, each wave's own: a matrix operand wants 16 rows at once, 16 bytes
// of each, which as loads from memory would be 64 lines for one operand; straight to LDS a load takes whole
// lines, and only the rows that there are. A half unit (every other block, 128 elements, 256 bytes a row)
// is a buffer; its piece p of row r is kept at place p ^ r.
// RG: loads of 4 dense rows each.
// 1 x 16384 x 4096 bf16 10 us, 3.6 TB/s of codes and scales (a read runs at 3.7); 16 x 4096 x 16384 14.4 us, 2.5 TB/s,
// 2.5 us of it the addition of the slices.
template <typename T, int NF, int RG>
__global__ __launch_bounds__(dense_waves(Planes<T>::N * (RG > 4 ? 2 : 1)) * 64, dense_waves(Planes<T>::N * (RG > 4 ? 2 : 1)) / 4) void mixed_rows_kernel(Dense16 D, Mx4View Y, RowsOut out) {
    constexpr int PL = Planes<T>::N, DF = RG > 4 ? 2 : 1;
    constexpr int BUF = PL * DF * 16 * 256;             // bytes of a wave's half unit
    constexpr int W = dense_waves(PL * DF), C = NF * DF < W ? NF * DF : W;
    static_assert(2 * W * BUF <= 160 * 1024, "LDS");
    __shared__ __attribute__((aligned(16))) uint8_t half0[W * BUF < W * C * 1024 ? W * C * 1024 : W * BUF];
    __shared__ __attribute__((aligned(16))) uint8_t half1[W * BUF];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, g = lane >> 4;
    const int64_t q0 = (int64_t)blockIdx.x * (NF * 16);
    const RowReader<NF, 2> q(Y, q0, r16, g);
    const int units = (q.nb + 7) / 8, stride = W * gridDim.y;
    v4f acc[NF * DF];
#pragma unroll
    for (int i = 0; i < NF * DF; ++i) acc[i] = v4f{0.f, 0.f, 0.f, 0.f};
    const int64_t d0 = (int64_t)blockIdx.z * (16 * DF), rows = D.rows - d0 < 16 * DF ? D.rows - d0 : 16 * DF;
    Buffer db[PL];
#pragma unroll
    for (int i = 0; i < PL; ++i) db[i] = buffer(D.ptr + i * D.plane + d0 * D.ld, (uint32_t)((rows - 1) * D.ld * 2 + D.chunks * 16));
    // one load: 4 rows, lane l places l & 15 of row l / 16 of them; rows that are not there are zeros
    auto load_dense = [&](int hu, uint8_t *lds) {       // half unit hu
#pragma unroll
        for (int i = 0; i < RG; ++i) {                  // further rows' places hold anything: their results are not stored
            const int row = i * 4 + g, kept = r16 ^ (row & 15);   // piece of the half: 4 of each 8 of the unit
            const int piece = (hu >> 1) * 32 + (kept >> 2) * 8 + (hu & 1) * 4 + (kept & 3);
            const uint32_t where = piece < D.chunks ? (uint32_t)(row * D.ld * 2) + (uint32_t)piece * 16 : OUTSIDE;
#pragma unroll
            for (int p = 0; p < PL; ++p) load_lds16(db[p], lds + wave * BUF + (p * DF * 16 + i * 4) * 256, where, 0);
        }
    };
    auto compute = [&](int u, int h, const RowCodes<NF, 2> &x, const uint8_t *lds) {
        float scale[NF];
#pragma unroll
        for (int f = 0; f < NF; ++f) scale[f] = __builtin_bit_cast(float, q.scale(u, h, x.s[f]) << 23);
        const uint8_t *row = lds + wave * BUF + r16 * 256;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            v4u d[DF][PL];
#pragma unroll
            for (int e = 0; e < DF; ++e)
#pragma unroll
                for (int p = 0; p < PL; ++p) d[e][p] = *(const v4u *)(row + (p * DF + e) * 16 * 256 + ((g * 4 + t) ^ r16) * 16);
#pragma unroll
            for (int f = 0; f < NF; ++f) {
                const v4u w = decode_bf16(x.c[f][h][t], scale[f]);
#pragma unroll
                for (int e = 0; e < DF; ++e)
#pragma unroll
                    for (int p = 0; p < PL; ++p) acc[f * DF + e] = mfma_bf16(w, d[e][p], acc[f * DF + e]);
            }
        }
    };
    // Loads arrive in their order, and a use waits until no more are on their way than were issued behind
    // those it needs: LD of dense rows for a half, LC of codes and scales for a unit. The fences keep every
    // load on its side of a wait. A unit past the last is zeros.
    constexpr int LD = RG * PL, LC = 3 * NF;
    RowCodes<NF, 2> a, b;
    int u = blockIdx.y * W + wave;
    q.load(u, a);
    load_dense(2 * u, half0);
    load_dense(2 * u + 1, half1);
    auto unit = [&](const RowCodes<NF, 2> &now, RowCodes<NF, 2> &next) {
        q.load(u + stride, next);
        wait_loads<LD + LC>();                          // of half 1 and of the next codes
        compute(u, 0, now, half0);
        __builtin_amdgcn_sched_barrier(0);
        load_dense(2 * (u + stride), half0);
        wait_loads<LC + LD>();                          // of the next codes and of the next half 0
        compute(u, 1, now, half1);
        __builtin_amdgcn_sched_barrier(0);
        load_dense(2 * (u + stride) + 1, half1);
        u += stride;
    };
    while (u < units) {
        unit(a, b);
        unit(b, a);
    }
    arrive();   // nothing is on its way to LDS any more
    add_waves<W, NF * DF>(acc, (v4f *)half0, lane, wave, [&](int i, int l, v4f v) {
        if constexpr (PL > 1)
            if (any_nan(v, i % DF * 16 + (l & 15) < rows))
                if (const Factors &x = factors_again(); infinities<false>(x.Y, q0 + i / DF * 16, 16, 0, x.Y.cols, l)) {
                    v = v4f{};
                    for (int64_t k = blockIdx.y * W * 256; k < x.Y.cols; k += stride * 256)
                        v = add_finite<false, true, PL>(v, x, q0 + i / DF * 16 + (l & 15), d0 + i % DF * 16 + (l & 15), k,
                                                        k + W * 256 < x.Y.cols ? k + W * 256 : x.Y.cols, l >> 4);
                }
#pragma unroll
        for (int j = 0; j < 4; ++j) put1<T>(out, q0 + (i / DF) * 16 + 4 * (l >> 4) + j, d0 + (i % DF) * 16 + (l & 15), v[j]);
    });
}

// The same for two 4-bit factors, 16 NF x 16 DF entries of the result a workgroup: products too small for
// the tiles, where the time of a call is the way of its loads.
// 77 x 1000 x 2080 f16 runs in 6 us, less than a call takes on the host; 256 x 4096 x 2048 bf16 15 us.
template <typename T, int NF, int DF>
__global__ __launch_bounds__(ROWS_WAVES * 64, 2) void both_rows_kernel(Mx4View Q, Mx4View D, RowsOut out) {
    constexpr int H = NF * DF >= 8 ? 1 : 2;   // what two units in flight leave of the registers
    __shared__ v4f sums[ROWS_WAVES * (NF * DF < 8 ? NF * DF : 8) * 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, g = lane >> 4;
    const int64_t q0 = (int64_t)blockIdx.x * (NF * 16), d0 = (int64_t)blockIdx.z * (DF * 16);
    const RowReader<NF, H> q(Q, q0, r16, g);
    const RowReader<DF, H> d(D, d0, r16, g);
    const int units = (q.nb + 4 * H - 1) / (4 * H), stride = ROWS_WAVES * gridDim.y;
    v4f acc[NF * DF];
#pragma unroll
    for (int i = 0; i < NF * DF; ++i) acc[i] = v4f{0.f, 0.f, 0.f, 0.f};
    auto compute = [&](int u, const RowCodes<NF, H> &x, const RowCodes<DF, H> &y) {
#pragma unroll
        for (int h = 0; h < H; ++h) {
            uint32_t sy[DF];
#pragma unroll
            for (int e = 0; e < DF; ++e) sy[e] = d.scale(u, h, y.s[e]);
#pragma unroll
            for (int f = 0; f < NF; ++f) {
                const uint32_t sx = q.scale(u, h, x.s[f]);
#pragma unroll
                for (int e = 0; e < DF; ++e)
                    acc[f * DF + e] = mfma_mx4(__builtin_bit_cast(v4i, x.c[f][h]), __builtin_bit_cast(v4i, y.c[e][h]), acc[f * DF + e],
                                               (int)sx, (int)sy[e]);
            }
        }
    };
    RowCodes<NF, H> qa, qb;
    RowCodes<DF, H> da, db;
    int u = blockIdx.y * ROWS_WAVES + wave;
    q.load(u, qa);
    d.load(u, da);
    for (; u < units; u += 2 * stride) {
        q.load(u + stride, qb);
        d.load(u + stride, db);
        compute(u, qa, da);
        __builtin_amdgcn_sched_barrier(0);   // not three units at once
        q.load(u + 2 * stride, qa);
        d.load(u + 2 * stride, da);
        compute(u + stride, qb, db);
    }
    add_waves<ROWS_WAVES, NF * DF>(acc, sums, lane, wave, [&](int i, int l, v4f v) {
#pragma unroll
        for (int j = 0; j < 4; ++j) put1<T>(out, q0 + (i / DF) * 16 + 4 * (l >> 4) + j, d0 + (i % DF) * 16 + (l & 15), v[j]);
    });
}

// Few dense rows and blocks across the contraction: codes, scales and dense rows from memory to registers, two units on
// their way. 16 x 8192 x 8192 bf16 19.5 us: this kernel 15.7, 2.3 TB/s, and the sum of 8 slices 3.8. Bound by the way of its
// loads: a wave has 4 units and two of them on their way. Vector instructions (2 an element, counted) are a quarter of
// the kernel's time, matrix instructions a sixteenth, and waves wait for 43 % of theirs.
template <typename T, int DF>
__global__ __launch_bounds__(ROWS_WAVES * 64, 2) void mixed_rows_yt_kernel(Dense16 D, Mx4View Y, int K, RowsOut out) {
    constexpr int PL = Planes<T>::N;
    __shared__ v4f sums[ROWS_WAVES * 8 * 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, g = lane >> 4;
    const int64_t q0 = (int64_t)blockIdx.x * 256;
    const int nb = (int)(mx4_blocks(Y.cols) - q0 / 32), tile_nb = nb < 8 ? nb : 8;   // blocks of a row from this workgroup's first
    const int units = (K + 31) / 32, stride = ROWS_WAVES * gridDim.y;
    // a wave's scales of a unit, by block and row, as upper halves of floats: 8 blocks x 32 rows (in the place
    // of its sums, which come after the last unit)
    uint16_t *scales = (uint16_t *)&sums[wave * 8 * 64];
    const int64_t d0 = (int64_t)blockIdx.z * (16 * DF), rows = D.rows - d0 < 16 * DF ? D.rows - d0 : 16 * DF;
    Buffer db[PL];
#pragma unroll
    for (int i = 0; i < PL; ++i) db[i] = buffer(D.ptr + i * D.plane + d0 * D.ld, (uint32_t)((rows - 1) * D.ld * 2 + D.chunks * 16));
    auto dense = [&](int piece, v4u (&d)[DF][PL]) {
#pragma unroll
        for (int e = 0; e < DF; ++e)
#pragma unroll
            for (int i = 0; i < PL; ++i)
                d[e][i] = load16(db[i], piece < D.chunks ? (uint32_t)((e * 16 + r16) * D.ld * 2) + (uint32_t)piece * 16 : OUTSIDE, 0);
    };
    struct Codes {
        v2u c[8];
        uint32_t s;
        v4u d[DF][PL];
    };
    // behind the last block 0, whatever is there: sums that are not stored are to be no NaN for that
    const int mine = tile_nb - (lane & 1) * 4;
    const uint32_t keep = mine >= 4 ? ~0u : mine > 0 ? (1u << (8 * mine)) - 1 : 0u;
    auto load = [&](int u, Codes &x) {
        const int left = K - u * 32 < 32 ? K - u * 32 : 32;
        const int64_t k0 = left > 0 ? (int64_t)u * 32 : 0;   // past the last unit the ranges are empty
        const Buffer cb = buffer(Y.codes + q0 / 2 + k0 * Y.ldq, left > 0 ? (uint32_t)((left - 1) * Y.ldq + tile_nb * 16) : 0u);
        const Buffer sb = buffer(Y.scales + q0 / 32 + k0 * Y.lds, left > 0 ? (uint32_t)((left - 1) * Y.lds + (tile_nb + 3) / 4 * 4) : 0u);
#pragma unroll
        for (int j = 0; j < 8; ++j) x.c[j] = load8(cb, (r16 >> 1) < nb ? (uint32_t)((8 * g + j) * Y.ldq) + 8 * r16 : OUTSIDE, 0);
        // lane: row lane / 2, 4 blocks
        const int b = (lane & 1) * 4;
        x.s = load4(sb, b < nb ? (uint32_t)((lane >> 1) * Y.lds) + b : OUTSIDE, 0);
        if constexpr (PL > 1) x.s &= keep;
        dense(u * 4 + g, x.d);
    };
    v4f acc[16 * DF];
#pragma unroll
    for (int i = 0; i < 16 * DF; ++i) acc[i] = v4f{0.f, 0.f, 0.f, 0.f};
    auto compute = [&](const Codes &x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) scales[((lane & 1) * 4 + i) * 32 + (lane >> 1)] = (uint16_t)(((x.s >> (8 * i)) & 255u) << 7);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        v4u sc8;
        __builtin_memcpy(&sc8, __builtin_assume_aligned(&scales[(r16 >> 1) * 32 + g * 8], 16), sizeof sc8);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int w = 0; w < 2; ++w) {   // 8 columns a word
            v4u row[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t half = (j & 1) ? sc8[j >> 1] & 0xFFFF0000u : sc8[j >> 1] << 16;
                row[j] = decode_bf16(x.c[j][w], __builtin_bit_cast(float, half));
            }
#pragma unroll
            for (int f = 0; f < 8; ++f) {
                v4u q;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    q[j] = __builtin_amdgcn_perm(row[2 * j + 1][f >> 1], row[2 * j][f >> 1], (f & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
                for (int e = 0; e < DF; ++e)
#pragma unroll
                    for (int i = 0; i < PL; ++i) acc[(w * 8 + f) * DF + e] = mfma_bf16(q, x.d[e][i], acc[(w * 8 + f) * DF + e]);
            }
        }
    };
    // a unit past the last is zeros
    Codes a, b;
    int u = blockIdx.y * ROWS_WAVES + wave;
    load(u, a);
    for (; u < units; u += 2 * stride) {
        load(u + stride, b);
        compute(a);
        __builtin_amdgcn_sched_barrier(0);   // not three units at once
        load(u + 2 * stride, a);
        compute(b);
        __builtin_amdgcn_sched_barrier(0);
    }
    // whether f is true for one of the parts of the contraction that the workgroup's waves took together
    auto in_parts = [&](auto f) {
        bool any = false;
        for (int64_t k = blockIdx.y * ROWS_WAVES * 32; k < K; k += stride * 32) any |= f(k, k + ROWS_WAVES * 32 < K ? k + ROWS_WAVES * 32 : K);
        return any;
    };
    add_waves<ROWS_WAVES, 16 * DF>(acc, sums, lane, wave, [&](int i, int l, v4f v) {
        if constexpr (PL > 1)
            if (any_nan(v, i % DF * 16 + (l & 15) < rows)) {
                const Factors &x = factors_again();
                if (in_parts([&](int64_t k, int64_t end) { return infinities<true>(x.Y, q0, 256, k, end, l); })) {
                    v = v4f{};
                    in_parts([&](int64_t k, int64_t end) {
                        v = add_finite<true, true, PL>(v, x, q0 + (l & 15) * 16 + i / DF, d0 + i % DF * 16 + (l & 15), k, end, l >> 4);
                        return false;
                    });
                }
            }
#pragma unroll
        for (int j = 0; j < 4; ++j) put1<T>(out, q0 + (4 * (l >> 4) + j) * 16 + i / DF, d0 + (i % DF) * 16 + (l & 15), v[j]);
    });
}

// C = alpha * (the sum of the slices' partial sums, in their order) + beta * C
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(const float *__restrict__ partial, int slices, Out out) {
    const int64_t n4 = (out.np + 3) / 4, plane = out.np * out.no;
    for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < n4 * out.no; t += (int64_t)gridDim.x * 256) {
        const int64_t q = t / n4, p = (t - q * n4) * 4;
        const float *x = partial + q * out.np + p;
        Four<T> c;
        c.load(out, (T *)out.ptr + q * out.ld + p, out.np - p < 4 ? (int)(out.np - p) : 4);
        v4f sum{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int z = 0; z < slices; ++z) {
            v4f v;
            if (c.n == 4) {
                __builtin_memcpy(&v, x + z * plane, sizeof v);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = x[z * plane + (i < c.n ? i : 0)];
            }
            sum += v;
        }
        c.template store<false>(out, sum);
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

constexpr size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// A window that ends inside a block of a wider matrix holds that block's further codes, which the products
// would take with the other factor's: they are zeros in a copy.
__global__ __launch_bounds__(256) void trim_codes_kernel(const uint8_t *src, int64_t ldq, int64_t rows, int nb, int tail, uint8_t *dst) {
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b >= nb) return;
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
        v4u c = *(const v4u *)(src + r * ldq + b * 16);
        if (b == nb - 1)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int have = tail - 8 * i;   // columns of this word
                c[i] = have >= 8 ? c[i] : have > 0 ? c[i] & ((1u << (4 * have)) - 1) : 0u;
            }
        *(v4u *)(dst + ((int64_t)r * nb + b) * 16) = c;
    }
}
size_t trim_work(const Mx4View &v) { return v.cut ? round256((size_t)v.rows * mx4_blocks(v.cols) * 16) : 0; }
hipError_t trim_codes(Mx4View &v, uint8_t *&work, hipStream_t s) {
    if (!v.cut) return hipSuccess;
    const int nb = (int)mx4_blocks(v.cols);
    const dim3 grid((unsigned)((nb + 255) / 256), (unsigned)(v.rows < 65535 ? v.rows : 65535));
    hipLaunchKernelGGL(trim_codes_kernel, grid, dim3(256), 0, s, v.codes, v.ldq, v.rows, nb, (int)(v.cols - (nb - 1) * 32), work);
    const size_t bytes = trim_work(v);
    v.codes = work;
    v.ldq = nb * 16;
    v.cut = false;
    work += bytes;
    return hipGetLastError();
}

// One factor that ends in zeros is enough for two 4-bit ones, the smaller one. A dense factor ends in zeros too, but
// 0 times a 4-bit value of 2^128 or more would be a NaN. Across the contraction nothing has to be cut.
Mx4Product cut_once(const Mx4Product &q) {
    Mx4Product p = q;
    if (p.yt) p.Y.cut = false;
    if (p.both) {
        const bool cut = p.XQ.cut && p.Y.cut;
        p.XQ.cut = cut && p.M < p.N;
        p.Y.cut = cut && p.M >= p.N;
    }
    return p;
}

template <typename T> hipError_t launch_join(const float *partial, int slices, const Out &out, hipStream_t s) {
    const int64_t n = ((out.np + 3) / 4 * out.no + 255) / 256;
    hipLaunchKernelGGL((join_kernel<T>), dim3((unsigned)(n < 65536 ? n : 65536)), dim3(256), 0, s, partial, slices, out);
    return hipGetLastError();
}

// How a product of two 4-bit factors runs: tile 256 or 128, or 0 and the kernel for small ones
struct BothPlan {
    int tile, nf, df;
    int slices, steps_z;   // of the contraction; steps of the tile kernel in each
    size_t partials, scales;
};
BothPlan both_plan(const Mx4Product &p) {
    BothPlan m{};
    auto tiles = [&](int64_t b) { return ((p.M + b - 1) / b) * ((p.N + b - 1) / b); };
    m.slices = 1;
    const int64_t small = p.M < p.N ? p.M : p.N, large = p.M < p.N ? p.N : p.M;
    auto groups = [&] { return ((large + 16 * m.nf - 1) / (16 * m.nf)) * ((small + 16 * m.df - 1) / (16 * m.df)); };
    m.df = small <= 16 ? 1 : small <= 32 ? 2 : 4;
    m.nf = 4;
    // One workgroup a compute unit for the kernel for small products, whose workgroups read both factors
    // from the L2 (2048 x 2048 x 2048, 1024 workgroups: 44 us, tiles of 128: 19 us; 256 x 4096 x 2048, 256 of
    // them: 14 and 17 us, at 8192 columns 34 and 23 us). Of the tiles the ones whose last round leaves less of the
    // card idle: one of 256 a compute
    // unit takes 28 for a step where two of 128 take 15 (4096 x 4096 x 4096: 46 and 53 us; 2048 x 4096 x 4096: 47 and
    // 31; 4096 x 4864 x 4096, a second round for 48 of 304: 70 and 64). The contraction is cut to 256 workgroups
    // (2048 x 2048 x 8192 f32: 36 us, to 512 41 us; 4096 x 4096 x 4096 uncut 47 us, in two 87 us).
    if ((small > 32 && groups() > 256) || (small > 64 && p.K > 4096)) m.tile = (tiles(256) + 255) / 256 * 28 < (tiles(128) + 511) / 512 * 15 ? 256 : 128;
    if (m.tile) {
        const int64_t steps = (p.K + 255) / 256, t = tiles(m.tile);
        int64_t z = 1;
        while (t * z * 2 <= 256 && steps / (z * 2) >= 8) z *= 2;
        m.steps_z = (int)((steps + z - 1) / z);
        m.slices = (int)((steps + m.steps_z - 1) / m.steps_z);
        m.scales = packed_scales(p.XQ) + packed_scales(p.Y);
    } else {
        while (groups() < 256 && m.nf > 1) {
            m.nf /= 2;
            if (m.df > 2) m.df = 2;
            if (m.df == 2 && m.nf == 1) { m.nf = 2; break; }
        }
        const int64_t units = (p.K + 255) / 256;
        while (groups() * m.slices < 256 && units / (m.slices * 2) >= 2 * ROWS_WAVES) m.slices *= 2;
        m.scales = scales_work(p.XQ) + scales_work(p.Y);
    }
    m.scales = round256(m.scales);
    if (m.slices > 1) m.partials = round256((size_t)m.slices * p.M * p.N * 4);
    return m;
}

template <int TYPE> hipError_t both_t(const Mx4Product &q, uint8_t *work, hipStream_t s) {
    typedef typename Elem<TYPE>::mem T;
    const BothPlan m = both_plan(q);
    Mx4Product p = q;
    const bool xp = p.ci == 1;   // X's index is the contiguous one of C
    const int64_t ld = xp ? p.cj : p.ci;
    const Out out{p.C, ld, xp ? p.M : p.N, xp ? p.N : p.M, p.alpha, p.beta};
    if (m.tile) {
        // the factor whose rows are the contiguous index gives the operand whose 4 entries a lane holds
        const Mx4View &P = xp ? p.XQ : p.Y, &O = xp ? p.Y : p.XQ;
        float *partial = m.slices > 1 ? (float *)(work + m.scales) : nullptr;
        const hipError_t e = m.tile == 256 ? launch_both_tile<T, 256, 256, 128, 64>(P, O, work, m.slices, m.steps_z, out, partial, s)
                                           : launch_both_tile<T, 128, 128, 64, 64>(P, O, work, m.slices, m.steps_z, out, partial, s);
        return e == hipSuccess && partial ? launch_join<T>(partial, m.slices, out, s) : e;
    }
    hipError_t e = align_scales(p.XQ, work, s);
    if (e == hipSuccess) e = align_scales(p.Y, work, s);
    if (e != hipSuccess) return e;
    const bool xq = p.M >= p.N;   // the larger factor
    const Mx4View &Q = xq ? p.XQ : p.Y, &D = xq ? p.Y : p.XQ;
    float *partial = m.slices > 1 ? (float *)work : nullptr;
    RowsOut o{p.C, xq ? p.ci : p.cj, xq ? p.cj : p.ci, Q.rows, D.rows, p.alpha, p.beta, partial};
    if (partial) o.sq = xq == xp ? 1 : D.rows, o.sd = xq == xp ? Q.rows : 1;
    const dim3 grid((unsigned)((Q.rows + 16 * m.nf - 1) / (16 * m.nf)), (unsigned)m.slices, (unsigned)((D.rows + 16 * m.df - 1) / (16 * m.df)));
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(ROWS_WAVES * 64), 0, s, Q, D, o); };
    if (m.df == 4) go(both_rows_kernel<T, 4, 4>);
    else if (m.df == 2 && m.nf == 4) go(both_rows_kernel<T, 4, 2>);
    else if (m.df == 2) go(both_rows_kernel<T, 2, 2>);
    else if (m.nf == 4) go(both_rows_kernel<T, 4, 1>);
    else if (m.nf == 2) go(both_rows_kernel<T, 2, 1>);
    else go(both_rows_kernel<T, 1, 1>);
    e = hipGetLastError();
    return e == hipSuccess && partial ? launch_join<T>(partial, m.slices, out, s) : e;
}

// How a mixed product runs
struct MixedPlan {
    int rows;            // dense rows / 16 of the kernel for few rows, 0 for the tiles
    bool direct;         // the dense factor is read as it is
    int64_t ld;          // of its planes otherwise
    int bq, bd;          // tile
    int slices, steps_z; // of the contraction, and steps of 64 in each
    size_t planes, partials, scales;   // workspace bytes
};

MixedPlan mixed_plan(const Mx4Product &p) {
    MixedPlan m{};
    const int pl = p.type == MX4_F32 ? 3 : p.type == MX4_F16 ? 2 : 1;
    // 16-byte pieces of 8 elements, whole ones only, rows within reach of a 32-bit offset
    m.direct = p.type == MX4_BF16 && p.X.sc == 1 && (uintptr_t)p.X.ptr % 16 == 0 && p.X.sr % 8 == 0 && p.K % 8 == 0 &&
               p.X.sr <= (1 << 21);
    m.scales = scales_work(p.Y);
    m.ld = (p.K + 63) / 64 * 64;
    if (!m.direct) m.planes = round256((size_t)pl * p.M * m.ld * 2);
    // The kernel for few rows, 16 or 32 of them (3 planes of 32: more than LDS, or with blocks across the
    // registers, hold) and 16 to 64 columns (256) a workgroup. Columns: as many as leave a workgroup for every compute
    // unit, since the sum of slices is a launch of its own (16 x 8192 x 8192 bf16 in a graph, 32 columns 13.8 us, 64 and
    // slices 16.3; 16 x 4096 x 4096, 16 columns 6.9 and 11.6). But each workgroup reads its dense rows whole: where those
    // are 512 KB, enough columns that their codes are more (16 x 4096 x 16384, 64 columns 15.4 us, 16 17.0). Measured at 128,
    // 256 and 512 KB only: where between the last two the sides meet is not known. The contraction is cut until
    // there are 256 workgroups. More rows too where that makes
    // no more than a workgroup for each compute unit (64 x 8192 x 4096 bf16 16.5 us, in tiles 20.6; 88 x 59 x 812
    // f32 14.5 and 27.8), except for one or two planes with blocks across more than 128 columns (64 x 4096 x 4096 25.0 and
    // 19.9; but 426 x 28 x 12096 15.9 and 17.8).
    const int df = p.M <= 16 || pl == 3 ? 1 : 2;
    const int64_t dgroups = (p.M + 16 * df - 1) / (16 * df), rows = p.M < 16 * df ? p.M : 16 * df;
    const int64_t widest = p.yt ? 256 : 64;
    if (p.M <= 16 * df || ((!p.yt || pl == 3 || p.N <= 128) && (p.N + widest - 1) / widest * dgroups <= 256)) {
        m.rows = df;
        m.bq = (int)widest;
        if (!p.yt)
            for (m.bq = 16; m.bq < 64 && ((rows * pl * 2 * p.K >= 512 << 10 && m.bq < 4 * pl * rows) || p.N * dgroups >= 512 * m.bq);) m.bq *= 2;
        const int64_t groups = (p.N + m.bq - 1) / m.bq * dgroups, units = p.yt ? (p.K + 31) / 32 : (p.K + 255) / 256;
        m.slices = 1;
        while (groups * m.slices < 256 && units / (m.slices * 2) >= (p.yt ? 2 * ROWS_WAVES : dense_waves(pl * m.rows))) m.slices *= 2;
        if (m.slices > 1) m.partials = round256((size_t)m.slices * p.M * p.N * 4);
        return m;
    }
    const int64_t nq = p.N, nd = p.M;
    auto tiles = [&](int64_t q, int64_t d) { return ((nq + q - 1) / q) * ((nd + d - 1) / d); };
    m.bq = 256;
    m.bd = 128;
    if (pl == 1 && tiles(256, 256) >= 256) m.bd = 256;
    else if (tiles(256, 128) < 256) m.bq = 128;
    const int64_t steps = (p.K + 63) / 64, t = tiles(m.bq, m.bd);
    // one plane: two tiles of 128 x 128 fit a compute unit (533 x 4231 x 5056: cut to 512 workgroups 51.5 us, to 256 59.0)
    int64_t z = 1;
    while (t * z * 2 <= (pl == 1 && m.bq == 128 ? 512 : 256) && steps / (z * 2) >= 8) z *= 2;
    // few tiles: shorter slices (300 x 300 x 1000 f16 16.9 us, without 19.8; with 128 workgroups no longer, 512 x 512 x 2048
    // bf16 15.8 and 15.3)
    while (t * z * 2 <= 64 && steps / (z * 2) >= 4) z *= 2;
    m.steps_z = (int)((steps + z - 1) / z + 3) / 4 * 4;   // codes come by 4 steps
    m.slices = (int)((steps + m.steps_z - 1) / m.steps_z);
    if (m.slices > 1) m.partials = round256((size_t)m.slices * p.M * p.N * 4);
    return m;
}

template <typename T, bool YT, int BQ, int BD, int WD>
hipError_t launch_mixed_tile(const Dense16 &D, const Mx4View &Y, int64_t K, const MixedPlan &m, const Out &out, float *partial,
                             bool qfirst, hipStream_t s) {
    constexpr int PL = Planes<T>::N, WQ = 64;
    const int64_t nq = YT ? Y.cols : Y.rows;
    const dim3 grid((unsigned)(((nq + BQ - 1) / BQ) * ((D.rows + BD - 1) / BD)), (unsigned)m.slices), block((BQ / WQ) * (BD / WD) * 64);
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, s, D, Y, K, m.steps_z, out, partial); };
    if constexpr (YT) qfirst ? go(mixed_tile_yt_kernel<T, PL, BQ, BD, WD, true>) : go(mixed_tile_yt_kernel<T, PL, BQ, BD, WD, false>);
    else qfirst ? go(mixed_tile_kernel<T, PL, BQ, BD, WQ, WD, true>) : go(mixed_tile_kernel<T, PL, BQ, BD, WQ, WD, false>);
    return hipGetLastError();
}

template <typename T> hipError_t launch_mixed_rows(const Dense16 &D, const Mx4Product &p, const MixedPlan &m, const Out &final, bool qfirst, float *partial, hipStream_t s) {
    RowsOut out{p.C, p.cj, p.ci, p.N, p.M, p.alpha, p.beta, partial};
    if (partial) out.sq = qfirst ? 1 : p.M, out.sd = qfirst ? p.N : 1;
    const dim3 grid((unsigned)((p.N + m.bq - 1) / m.bq), (unsigned)m.slices, (unsigned)((p.M + 16 * m.rows - 1) / (16 * m.rows))), block((p.yt ? ROWS_WAVES : dense_waves(Planes<T>::N * m.rows)) * 64);
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, s, D, p.Y, out); };
    if (p.yt) {
        if (m.rows == 1) hipLaunchKernelGGL((mixed_rows_yt_kernel<T, 1>), grid, block, 0, s, D, p.Y, (int)p.K, out);
        else if constexpr (Planes<T>::N < 3) hipLaunchKernelGGL((mixed_rows_yt_kernel<T, 2>), grid, block, 0, s, D, p.Y, (int)p.K, out);
    } else if (p.M <= 4) {
        if (m.bq == 64) go(mixed_rows_kernel<T, 4, 1>);
        else if (m.bq == 32) go(mixed_rows_kernel<T, 2, 1>);
        else go(mixed_rows_kernel<T, 1, 1>);
    } else if (m.rows == 1) {
        if (m.bq == 64) go(mixed_rows_kernel<T, 4, 4>);
        else if (m.bq == 32) go(mixed_rows_kernel<T, 2, 4>);
        else go(mixed_rows_kernel<T, 1, 4>);
    } else if constexpr (Planes<T>::N < 3) {
        if (m.bq == 16) go(mixed_rows_kernel<T, 1, 8>);
        else if (m.bq == 32) go(mixed_rows_kernel<T, 2, 8>);
        else go(mixed_rows_kernel<T, 4, 8>);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess && partial ? launch_join<T>(partial, m.slices, final, s) : e;
}

template <int TYPE> hipError_t mixed_t(const Mx4Product &q, uint8_t *work, hipStream_t s) {
    typedef typename Elem<TYPE>::mem T;
    const MixedPlan m = mixed_plan(q);
    Mx4Product p = q;
    const bool qfirst = p.cj == 1;   // the 4-bit factor's index is the contiguous one of C
    const int64_t ld = qfirst ? p.ci : p.cj;
    const Out out{p.C, ld, qfirst ? p.N : p.M, qfirst ? p.M : p.N, p.alpha, p.beta};
    hipError_t e = align_scales(p.Y, work, s);
    if (e != hipSuccess) return e;
    Dense16 D{(const uint16_t *)p.X.ptr, p.M, p.X.sr, 0, (int)(p.K / 8)};
    if (!m.direct) {
        uint16_t *planes = (uint16_t *)work;
        work += m.planes;
        const T *x = (const T *)p.X.ptr;
        const int64_t n8 = m.ld / 8;
        if (p.X.sc == 1)
            hipLaunchKernelGGL((planes_kernel<T>), dim3((unsigned)((n8 + 255) / 256), (unsigned)(p.M < 65535 ? p.M : 65535)),
                               dim3(256), 0, s, x, p.X.sr, p.M, p.K, m.ld, planes);
        else
            hipLaunchKernelGGL((planes_cols_kernel<T>), dim3((unsigned)((p.M + 63) / 64), (unsigned)(n8 / 8 < 65535 ? n8 / 8 : 65535)), dim3(256), 0, s, x,
                               p.X.sc, p.M, p.K, m.ld, planes);
        e = hipGetLastError();
        if (e != hipSuccess) return e;
        D = Dense16{planes, p.M, m.ld, p.M * m.ld, (int)n8};
    }
    float *partial = m.slices > 1 ? (float *)work : nullptr;
    if (m.rows) return launch_mixed_rows<T>(D, p, m, out, qfirst, partial, s);
    auto go = [&](auto yt) -> hipError_t {
        constexpr bool YT = decltype(yt)::value;
        if constexpr (Planes<T>::N == 1)
            if (m.bd == 256) return launch_mixed_tile<T, YT, 256, 256, 128>(D, p.Y, p.K, m, out, partial, qfirst, s);
        if (m.bq == 256) return launch_mixed_tile<T, YT, 256, 128, 64>(D, p.Y, p.K, m, out, partial, qfirst, s);
        return launch_mixed_tile<T, YT, 128, 128, Planes<T>::N == 1 ? 64 : 32>(D, p.Y, p.K, m, out, partial, qfirst, s);
    };
    e = p.yt ? go(std::true_type{}) : go(std::false_type{});
    if (e != hipSuccess || !partial) return e;
    return launch_join<T>(partial, m.slices, out, s);
}

template <int TYPE> hipError_t product_t(const Mx4Product &p, void *work, hipStream_t s) {
    if (p.K <= 0 || p.alpha == 0.f) {
        const int64_t inner = p.ci == 1 ? p.M : p.N, outer = p.ci == 1 ? p.N : p.M;
        hipLaunchKernelGGL((scale_kernel<TYPE>), dim3((unsigned)((inner + 255) / 256), (unsigned)(outer < 65535 ? outer : 65535)),
                           dim3(256), 0, s, p, inner, outer, p.ci == 1 ? p.cj : p.ci);
        return hipGetLastError();
    }
    Mx4Product c = cut_once(p);
    uint8_t *w = (uint8_t *)work;
    hipError_t e = trim_codes(c.XQ, w, s);
    if (e == hipSuccess) e = trim_codes(c.Y, w, s);
    if (e != hipSuccess) return e;
    return c.both ? both_t<TYPE>(c, w, s) : mixed_t<TYPE>(c, w, s);
}

}  // namespace

size_t mx4_product_work(const Mx4Product &q) {
    if (q.K <= 0 || q.alpha == 0.f) return 0;
    const Mx4Product p = cut_once(q);
    const size_t cut = trim_work(p.XQ) + trim_work(p.Y);
    if (p.both) {
        const BothPlan b = both_plan(p);
        return cut + b.scales + b.partials;
    }
    const MixedPlan m = mixed_plan(p);
    return cut + m.scales + m.planes + m.partials;
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
