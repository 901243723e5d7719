// What the Newton-Schulz paths share: orthogonalize.cu (arguments, small matrices, packing)
// and orthogonalize_tc.cu (products on the tensor cores).
#pragma once

#include "operators.cuh"

namespace mtc {
namespace ortho {

// One matrix as its short side m by its long side n (a tall one is taken transposed).
struct Matrix {
    const float *src;
    float *dst;
    int64_t rs, cs, out_rs, out_cs;  // strides of the short and of the long side
    int m, n;
    // Of the tensor-core path.  Packed operands lie in the workspace in blocks of 128 rows by 64
    // columns, hi and lo next to each other, 16 KB each; every block is the image of itself in
    // shared memory (a row 128 bytes, its 16-byte chunks permuted as the 128-byte swizzle does).
    // Positions are counted in rows of 128 bytes.
    int x_blocks, s_blocks;  // blocks of 64 columns of X (n) and of X X^T (m)
    int x[2], s, b;          // X before and after a step, S = X X^T, and B = b S + c S S
    int s_diagonal, b_diagonal;  // float32; s and b hold zeros there
    int part, parts;         // partial sums of squares
};

struct Step {
    float a, b, c;
    int x, s, b_exp;  // exponents of the scales of X before the step, of X X^T and of the polynomial
    int x_after;
};

// Packed columns are padded to whole tiles; a matrix of up to 128 rows has tiles of 128.
inline int tile_of(int m) { return m <= 128 ? 128 : 256; }
inline int64_t pad_to(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// All products of all steps over `count` matrices, packed at x[0] of each.
int products(const Matrix *matrices, int count, const Step *steps, int n_steps, char *workspace, size_t bytes, cudaStream_t stream);

constexpr int kMostMatrices = 128;  // of a launch: they travel in its parameters

template <int N>
struct Table {
    int count;
    int first[N + 1];  // unit of the launch's work that a matrix begins with
    Matrix matrix[N];
};

// The matrix that unit u belongs to.
template <int N>
__host__ __device__ __forceinline__ int find_matrix(const Table<N> &t, int u) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (t.first[mid] <= u) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

#ifdef __CUDACC__
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }

// Byte of the 16-byte chunk of hi that holds column c (a multiple of 8) of row r; lo lies 16384 on.
__device__ __forceinline__ int64_t chunk_at(int position, int blocks, int r, int c) {
    const int64_t block = static_cast<int64_t>(r / 128) * blocks + c / 64;
    return (static_cast<int64_t>(position) + block * 256 + r % 128) * 128 + (((c / 8) ^ r) & 7) * 16;
}
#endif

}  // namespace ortho
}  // namespace mtc
