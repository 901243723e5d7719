// What the Newton-Schulz paths share: orthogonalize.cu (arguments, small matrices, packing)
// and orthogonalize_tc.cu (products on the tensor cores).
#pragma once

#include <cmath>

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

constexpr int kMostSteps = 32;

// What the elements are multiplied by: zeros stay zeros whatever eps is, and one element that is
// not finite makes all of them NaN.
__host__ __device__ inline double inverse_norm(double squares, float eps) {
    if (squares == 0.0) return 0.0;
    const double norm = sqrt(squares);
    return isfinite(norm) ? 1.0 / (norm + static_cast<double>(eps)) : nan("");
}

// That and a scale as a float32 in [1, 2) and a power of two in two parts, which neither the
// largest nor the smallest norms take out of float32.
struct Factor {
    float f, two0, two1;
    __host__ __device__ Factor(double inverse, int scale) {
        int e = 0;
        f = 2.0f * static_cast<float>(frexp(inverse, &e));
        e += scale - 1;
        two0 = exp2f(static_cast<float>(e / 2));
        two1 = exp2f(static_cast<float>(e - e / 2));
    }
    __host__ __device__ float operator()(float v) const { return v * two0 * f * two1; }
};

// All steps over matrices of up to 128 x 128, a CTA each (one launch for each kMostMatrices).
int whole_matrices(const Matrix *matrices, int count, const Step *steps, int n_steps, float eps, cudaStream_t stream);

constexpr int kMostMatrices = 128;  // of a launch: they travel in its parameters

template <int N>
struct Table {
    int count;
    int first[N + 1];  // unit of the launch's work that a matrix begins with
    Matrix matrix[N];
};

// Calls f with a table of the matrices at hand: a small one where they are few.
template <class F>
int with_table(const Matrix *m, int count, F &&f) {
    auto fill = [&](auto &t) {
        std::memset(&t, 0, sizeof(t));
        t.count = count;
        for (int i = 0; i < count; ++i) t.matrix[i] = m[i];
        return f(t);
    };
    if (count <= 8) {
        Table<8> t;
        return fill(t);
    }
    Table<kMostMatrices> t;
    return fill(t);
}

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
