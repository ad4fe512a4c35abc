// mx4.hpp -- 4-bit microscaled (MX) matrices: quantisation, its inverse and products.
//
// Format: Open Compute Project Microscaling Formats (MX) v1.0, MXFP4. An element is E2M1 (sign, 2
// exponent bits, 1 mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6); 32 consecutive elements of a row share
// a scale 2^(s - 127) stored as the byte s (E8M0, 255 = NaN). Two elements a byte, the even column in
// the low half; a row is 16 bytes a block, the last block padded with zero codes.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace rbh {

enum Mx4Type : int { MX4_F64 = 0, MX4_F32 = 1, MX4_F16 = 2, MX4_BF16 = 3 };
inline int mx4_size(int type) { return type == MX4_F64 ? 8 : type == MX4_F32 ? 4 : 2; }

constexpr int MX4_BLOCK = 32;
__host__ __device__ inline int64_t mx4_blocks(int64_t cols) { return (cols + MX4_BLOCK - 1) / MX4_BLOCK; }

// rows x cols window of a 4-bit matrix that starts at a block; ldq / lds: bytes between rows; cut: it ends
// inside a block whose further codes belong to the matrix
struct Mx4View {
    uint8_t *codes, *scales;
    int64_t ldq, lds;
    int64_t rows, cols;
    bool cut;
};

// A dense matrix seen as element (r, c) = ptr[r * sr + c * sc]; sr or sc is 1
struct Mx4Dense {
    const void *ptr;
    int64_t sr, sc;
    int type;
};

// The random words of stochastic rounding: element (r, c) reads word c & 3 of the generator at
// ctr + r * quads + (c >> 2), quads = ceil(cols / 4) -- fill_dense's map of a row-major parent
struct Mx4Random {
    uint32_t ctr[4], key[4];
    int rng;
    uint64_t quads;
};

hipError_t launch_mx4_quantize(const Mx4Dense &A, const Mx4View &Q, const Mx4Random *rnd, hipStream_t s);
hipError_t launch_mx4_dequantize(const Mx4View &Q, const Mx4Dense &A, hipStream_t s);

// C(i, j) = alpha * sum_k X(i, k) Y(j, k) + beta * C(i, j), 0 <= i < M, 0 <= j < N, C(i, j) =
// C[i * ci + j * cj]. Y is a 4-bit matrix, N x K (yt = 0) or K x N (yt = 1). X is a dense matrix
// (M x K, sr and sc are its strides) or, with `both`, a 4-bit matrix M x K.
struct Mx4Product {
    int64_t M, N, K;
    bool both;
    Mx4Dense X;
    Mx4View XQ, Y;
    int yt;
    void *C;
    int64_t ci, cj;
    int type;            // of C, and of a dense X
    float alpha, beta;
};
// bytes of workspace launch_mx4_product needs for p (0: none)
size_t mx4_product_work(const Mx4Product &p);
hipError_t launch_mx4_product(const Mx4Product &p, void *work, hipStream_t s);

}  // namespace rbh
