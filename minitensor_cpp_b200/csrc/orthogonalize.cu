// Updates of weight matrices made orthogonal by Newton-Schulz products:
//
//   X = T / (|T|_F + eps),  and in every step  S = X X^T,  B = b S + c S^2,  X <- a X + B X
//
// on the shorter side of T.  Each singular value x of X goes to p(x) = a x + b x^3 + c x^5, so it
// stays in [0, s], s = 1 at first and then the maximum of |p| over [0, s].  The host follows s;
// the elements of X, S and B are below it and its polynomials, which gives the packed operands
// of the tensor cores fixed scales: nothing is looked at while the products run.
//
// Small matrices are worked on by a CTA each, in shared memory: in float32 (k_small), or on the
// tensor cores where both sides are 128 or less and the products are enough.  All others are
// packed into pairs of 16-bit floats once and then stay so, from one product's epilogue to the
// next one's operands (orthogonalize_tc.cu).
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstring>
#include <exception>
#include <vector>

#include "orthogonalize.cuh"

namespace mtc {
namespace ortho {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ double block_sum(double v) {
    __shared__ double part[kThreads / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    __syncthreads();
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) v += part[i];
    return v;
}

// ---------------------------------------------------------- small matrices --

struct SmallSteps {
    int n;
    float eps;
    float a[kMostSteps], b[kMostSteps], c[kMostSteps];
};

// Shared memory of a small matrix: X twice and two squares, rows in whole float4 and 4 floats
// apart from a multiple of the banks.
__host__ __device__ inline int small_pitch(int cols) { return (cols + 3) / 4 * 4 + 4; }
inline size_t small_bytes(int m, int n) {
    const size_t rows = (m + 3) / 4 * 4;
    return 4 * rows * 2 * (static_cast<size_t>(small_pitch(n)) + small_pitch(m));
}

// to[i][j] = p old[i][j] + q sum_k x[i][k] y[j][k]; a thread has rows i, i + R, ... and columns
// j, j + R, ... (R a fourth of the rows), so that neighbours read neighbouring rows.
__device__ __forceinline__ void small_by_rows(const float *x, int pitch, int K, int R, const float *old, float *to,
                                              int to_pitch, float p, float q) {
    for (int t = threadIdx.x; t < R * R; t += kThreads) {
        const int ti = t / R, tj = t % R;
        float acc[4][4] = {};
        for (int k = 0; k < K; k += 4) {
            float4 u[4], v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                u[i] = *reinterpret_cast<const float4 *>(x + (ti + R * i) * pitch + k);
                v[i] = *reinterpret_cast<const float4 *>(x + (tj + R * i) * pitch + k);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    acc[i][j] = fmaf(u[i].x, v[j].x, acc[i][j]);
                    acc[i][j] = fmaf(u[i].y, v[j].y, acc[i][j]);
                    acc[i][j] = fmaf(u[i].z, v[j].z, acc[i][j]);
                    acc[i][j] = fmaf(u[i].w, v[j].w, acc[i][j]);
                }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int at = (ti + R * i) * to_pitch + tj + R * j;
                to[at] = old != nullptr ? fmaf(p, old[at], q * acc[i][j]) : q * acc[i][j];
            }
    }
}

// to[i][j] = a x[i][j] + sum_k s[i][k] x[k][j]; a thread has rows i, i + R, ... and four columns.
__device__ __forceinline__ void small_apply(const float *s, int s_pitch, const float *x, int pitch, int m, int R, int C,
                                            float *to, float a) {
    for (int t = threadIdx.x; t < R * C; t += kThreads) {
        const int ti = t / C, tj = t % C;
        float acc[4][4] = {};
        for (int k = 0; k < m; k += 4) {
            float4 u[4], v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                u[i] = *reinterpret_cast<const float4 *>(s + (ti + R * i) * s_pitch + k);
                v[i] = *reinterpret_cast<const float4 *>(x + (k + i) * pitch + 4 * tj);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    acc[i][0] = fmaf(w[q], v[q].x, acc[i][0]);
                    acc[i][1] = fmaf(w[q], v[q].y, acc[i][1]);
                    acc[i][2] = fmaf(w[q], v[q].z, acc[i][2]);
                    acc[i][3] = fmaf(w[q], v[q].w, acc[i][3]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = (ti + R * i) * pitch + 4 * tj;
            const float4 o = *reinterpret_cast<const float4 *>(x + at);
            *reinterpret_cast<float4 *>(to + at) = make_float4(fmaf(a, o.x, acc[i][0]), fmaf(a, o.y, acc[i][1]),
                                                               fmaf(a, o.z, acc[i][2]), fmaf(a, o.w, acc[i][3]));
        }
    }
}

template <int N>
__global__ void __launch_bounds__(kThreads) k_small(const __grid_constant__ Table<N> table, const SmallSteps steps) {
    extern __shared__ __align__(16) float smem[];
    const Matrix &mt = table.matrix[blockIdx.x];
    const int m = mt.m, n = mt.n, rows = (m + 3) / 4 * 4, pitch = small_pitch(n), s_pitch = small_pitch(m);
    float *x = smem, *y = x + rows * pitch, *s = y + rows * pitch, *b = s + rows * s_pitch;
    // rows and columns up to whole fours are zeros, and stay so
    const bool along = mt.cs == 1 || mt.rs != 1;
    double squares = 0.0;
    const int total = rows * pitch;
    for (int i = threadIdx.x; i < total; i += kThreads) {
        const int r = along ? i / pitch : i % rows, c = along ? i % pitch : i / rows;
        const float v = r < m && c < n ? mt.src[r * mt.rs + c * mt.cs] : 0.0f;
        x[r * pitch + c] = v;
        squares += static_cast<double>(v) * v;
    }
    const double inverse = inverse_norm(block_sum(squares), steps.eps);
    for (int i = threadIdx.x; i < total; i += kThreads) x[i] = static_cast<float>(x[i] * inverse);
    __syncthreads();
    const int R = rows / 4, C = (n + 3) / 4;
    for (int k = 0; k < steps.n; ++k) {
        small_by_rows(x, pitch, n, R, nullptr, s, s_pitch, 0.0f, 1.0f);
        __syncthreads();
        small_by_rows(s, s_pitch, m, R, s, b, s_pitch, steps.b[k], steps.c[k]);
        __syncthreads();
        small_apply(b, s_pitch, x, pitch, m, R, C, y, steps.a[k]);
        __syncthreads();
        float *const t = x;
        x = y;
        y = t;
    }
    const bool out_along = mt.out_cs == 1 || mt.out_rs != 1;
    for (int i = threadIdx.x; i < m * n; i += kThreads) {
        const int r = out_along ? i / n : i % m, c = out_along ? i % n : i / m;
        mt.dst[r * mt.out_rs + c * mt.out_cs] = x[r * pitch + c];
    }
}

// ----------------------------------------------------------------- packing --

// A unit is 32 rows of a block of 64 columns, eight elements a thread: read along the axis whose
// elements lie next to each other.
constexpr int kUnitRows = 32;

struct Unit {
    int r0, c0;
};

template <class F>
__device__ __forceinline__ void read_unit(const Matrix &mt, Unit at, F &&take) {
    const bool along = mt.cs == 1 || mt.rs != 1;
    const int r0 = along ? threadIdx.x / 64 : threadIdx.x % kUnitRows, c0 = along ? threadIdx.x % 64 : threadIdx.x / kUnitRows;
    const int dr = along ? kThreads / 64 : 0, dc = along ? 0 : kThreads / kUnitRows;
    const float *src = mt.src + (at.r0 + r0) * mt.rs + (at.c0 + c0) * mt.cs;
    const int64_t step = dr * mt.rs + dc * mt.cs;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const bool in = at.r0 + r0 + i * dr < mt.m && at.c0 + c0 + i * dc < mt.n;
        v[i] = in ? src[i * step] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) take(r0 + i * dr, c0 + i * dc, v[i]);
}

template <int N>
__global__ void __launch_bounds__(kThreads) k_squares(const __grid_constant__ Table<N> table, double *partials) {
    const int k = find_matrix(table, blockIdx.x);
    const Matrix &mt = table.matrix[k];
    const int cols = (mt.n + 63) / 64;
    const int64_t units = static_cast<int64_t>((mt.m + kUnitRows - 1) / kUnitRows) * cols;
    double acc = 0.0;
    for (int64_t i = static_cast<int>(blockIdx.x) - table.first[k]; i < units; i += mt.parts) {
        const Unit at{static_cast<int>(i / cols) * kUnitRows, static_cast<int>(i % cols) * 64};
        read_unit(mt, at, [&](int, int, float v) { acc += static_cast<double>(v) * v; });
    }
    acc = block_sum(acc);
    if (threadIdx.x == 0) partials[mt.part + static_cast<int>(blockIdx.x) - table.first[k]] = acc;
}

// Units of the padded matrix.
template <int N>
__global__ void __launch_bounds__(kThreads) k_pack_matrices(const __grid_constant__ Table<N> table, const double *partials,
                                                            float eps, int scale, char *workspace) {
    __shared__ float tile[kUnitRows * 65];
    wait_for_previous();
    const int k = find_matrix(table, blockIdx.x);
    const Matrix &mt = table.matrix[k];
    double squares = 0.0;
    for (int i = threadIdx.x; i < mt.parts; i += kThreads) squares += partials[mt.part + i];
    const Factor factor(inverse_norm(block_sum(squares), eps), scale);
    const int u = static_cast<int>(blockIdx.x) - table.first[k];
    const Unit at{u / mt.x_blocks * kUnitRows, u % mt.x_blocks * 64};
    read_unit(mt, at, [&](int r, int c, float v) { tile[r * 65 + c] = factor(v); });
    __syncthreads();
    const int r = threadIdx.x / 8, c = threadIdx.x % 8 * 8;  // a row's eight chunks side by side
    __half2 hi[4], lo[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float v0 = tile[r * 65 + c + 2 * j], v1 = tile[r * 65 + c + 2 * j + 1];
        hi[j] = __floats2half2_rn(v0, v1);
        const float2 f = __half22float2(hi[j]);
        lo[j] = __floats2half2_rn((v0 - f.x) * 2048.0f, (v1 - f.y) * 2048.0f);
    }
    char *to = workspace + chunk_at(mt.x[0], mt.x_blocks, at.r0 + r, at.c0 + c);
    *reinterpret_cast<uint4 *>(to) = *reinterpret_cast<const uint4 *>(hi);
    *reinterpret_cast<uint4 *>(to + 16384) = *reinterpret_cast<const uint4 *>(lo);
}

// ------------------------------------------------------------------- host --

// The maximum of |a x + b x^3 + c x^5| over [0, s].
double largest_value(double a, double b, double c, double s) {
    auto p = [&](double x) { return std::fabs(x * (a + x * x * (b + x * x * c))); };
    double most = p(s);
    auto at = [&](double y) {  // a root of the derivative in y = x^2
        if (y > 0.0 && y < s * s) most = std::max(most, p(std::sqrt(y)));
    };
    // 5 c y^2 + 3 b y + a = 0, without a difference of what may be nearly equal
    const double d = 9.0 * b * b - 20.0 * a * c;
    if (d >= 0.0) {
        const double q = -0.5 * (3.0 * b + std::copysign(std::sqrt(d), b));
        if (c != 0.0) at(q / (5.0 * c));
        if (q != 0.0) at(a / q);
    }
    return most;
}

// And of |b t + c t^2| over [0, s^2].
double largest_factor(double b, double c, double s) {
    const double t = s * s;
    double most = std::fabs(t * (b + c * t));
    if (c != 0.0) {
        const double y = -b / (2.0 * c);
        if (y > 0.0 && y < t) most = std::max(most, std::fabs(y * (b + c * y)));
    }
    return most;
}

// Scales bring what is bounded by `most` to 2^14: float16 ends at 2^16, and roundings may pass
// the bound a little.
int scale_for(double most) {
    if (most < 0x1p-60) return 74;
    int e;
    std::frexp(most, &e);  // most <= 2^e
    return 14 - e;
}

int follow_steps(const float *coefficients, int32_t n, std::vector<Step> &steps) {
    double s = 1.0;
    for (int k = 0; k < n; ++k) {
        const float *q = coefficients + 3 * k;
        Step t;
        t.a = q[0];
        t.b = q[1];
        t.c = q[2];
        const double factor = largest_factor(t.b, t.c, s), next = largest_value(t.a, t.b, t.c, s);
        if (!(factor <= 0x1p40 && next <= 0x1p20))
            return fail(MTC_ERR_INVALID_ARGUMENT, "step %d: with these coefficients singular values grow to %g", k, next);
        t.x = scale_for(s);
        t.s = scale_for(s * s);
        t.b_exp = scale_for(factor);
        t.x_after = scale_for(next);
        s = next;
        steps.push_back(t);
    }
    return MTC_OK;
}

void add_matrices(const mtc_desc &in, const mtc_desc &out, std::vector<Matrix> &all) {
    if (numel_of(in) == 0) return;
    const int r = in.rank;
    Matrix one;
    std::memset(&one, 0, sizeof(one));
    const int64_t rows = in.shape[r - 2], cols = in.shape[r - 1];
    const int shorter = rows <= cols ? r - 2 : r - 1, longer = rows <= cols ? r - 1 : r - 2;
    one.m = static_cast<int>(in.shape[shorter]);
    one.n = static_cast<int>(in.shape[longer]);
    one.rs = in.strides[shorter];
    one.cs = in.strides[longer];
    one.out_rs = out.strides[shorter];
    one.out_cs = out.strides[longer];
    int64_t count = 1;
    for (int i = 0; i < r - 2; ++i) count *= in.shape[i];
    for (int64_t k = 0; k < count; ++k) {
        int64_t at = k, from = 0, to = 0;
        for (int i = r - 3; i >= 0; --i) {
            from += at % in.shape[i] * in.strides[i];
            to += at % in.shape[i] * out.strides[i];
            at /= in.shape[i];
        }
        one.src = float_at(&in) + from;
        one.dst = float_at(&out) + to;
        all.push_back(one);
    }
}

// A CTA's matrix in float32: in shared memory, and of few products.  Up to 128 columns the other way
// is a CTA with the tensor cores (48 x 48: 38 us here, 47 there; 64 x 64: 50 and 48.5), beyond 17
// launches (64 x 100: 160 us there, and in proportion to its products some 70 here).
bool is_small(const Matrix &mt) {
    const int64_t m = mt.m, n = mt.n;
    return 2 * m * m * n + m * m * m <= (n <= 128 ? 3 * 60 * 60 * 60 : 9 * 64 * 64 * 64) &&
           small_bytes(mt.m, mt.n) <= 200 * 1024;
}

bool is_whole(const Matrix &mt) { return mt.n <= 128; }

int run_small(const std::vector<Matrix> &all, const std::vector<Step> &steps, float eps, cudaStream_t stream) {
    SmallSteps s;
    std::memset(&s, 0, sizeof(s));
    s.n = static_cast<int>(steps.size());
    s.eps = eps;
    for (int k = 0; k < s.n; ++k) {
        s.a[k] = steps[k].a;
        s.b[k] = steps[k].b;
        s.c[k] = steps[k].c;
    }
    for (size_t at = 0; at < all.size(); at += kMostMatrices) {
        const int count = static_cast<int>(std::min<size_t>(kMostMatrices, all.size() - at));
        size_t bytes = 0;
        for (int i = 0; i < count; ++i) bytes = std::max(bytes, small_bytes(all[at + i].m, all[at + i].n));
        MTC_TRY(with_table(all.data() + at, count, [&](const auto &t) {
            constexpr int N = sizeof(t.matrix) / sizeof(t.matrix[0]);
            MTC_CUDA_TRY(cudaFuncSetAttribute(k_small<N>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
            k_small<N><<<count, kThreads, bytes, stream>>>(t, s);
            return check_launch("orthogonalize (small)");
        }));
    }
    return MTC_OK;
}

size_t packed_bytes(const Matrix &m) {
    const int64_t tile = tile_of(m.m), rows = pad_to(m.m, tile);
    return static_cast<size_t>(4 * (2 * rows * pad_to(m.n, tile) + 2 * rows * rows + 2 * rows));
}

constexpr size_t kGroupBytes = size_t{4} << 30;  // of packed operands at a time

int run_group(Matrix *m, int count, const std::vector<Step> &steps, float eps, cudaStream_t stream) {
    size_t bytes = 0;
    int64_t blocks = 0;
    for (int i = 0; i < count; ++i) {
        bytes += packed_bytes(m[i]);
        blocks += pad_to(m[i].m, kUnitRows) / kUnitRows * (pad_to(m[i].n, 64) / 64);
    }
    // positions are counted in 32 bits
    if (bytes / 128 > INT_MAX) return fail(MTC_ERR_UNSUPPORTED, "a matrix of %d x %d is too large", m[0].m, m[0].n);
    const int64_t ctas = static_cast<int64_t>(sm_count(current_device())) * 8;
    int parts = 0, position = 0;
    for (int i = 0; i < count; ++i) {
        Matrix &x = m[i];
        const int64_t tile = tile_of(x.m), rows = pad_to(x.m, tile), cols = pad_to(x.n, tile);
        const int64_t mine = pad_to(x.m, kUnitRows) / kUnitRows * (pad_to(x.n, 64) / 64);
        const int64_t share = std::max<int64_t>(1, ctas * mine / blocks);
        x.x_blocks = static_cast<int>(cols / 64);
        x.s_blocks = static_cast<int>(rows / 64);
        const int of_x = static_cast<int>(rows / 128 * x.x_blocks * 256), of_s = static_cast<int>(rows / 128 * x.s_blocks * 256);
        x.x[0] = position;
        x.x[1] = x.x[0] + of_x;
        x.s = x.x[1] + of_x;
        x.b = x.s + of_s;
        x.s_diagonal = x.b + of_s;
        x.b_diagonal = x.s_diagonal + static_cast<int>(rows / 32);
        position = x.b_diagonal + static_cast<int>(rows / 32);
        x.part = parts;
        x.parts = static_cast<int>(std::min<int64_t>(std::min<int64_t>(mine, share), 1024));
        parts += x.parts;
    }
    Workspace ws;
    const int allocated = ws.allocate(bytes + 1024 + padded(parts * sizeof(double)), stream);
    if (allocated == MTC_ERR_RUNTIME && count > 1) {  // no memory for that: in smaller groups
        MTC_TRY(run_group(m, count / 2, steps, eps, stream));
        MTC_TRY(run_group(m + count / 2, count - count / 2, steps, eps, stream));
        clear_error();
        return MTC_OK;
    }
    MTC_TRY(allocated);
    double *partials = ws.take<double>(parts * sizeof(double));
    char *packed = ws.take<char>(bytes + 1024);
    packed += -reinterpret_cast<uintptr_t>(packed) & 1023;  // a block is where the swizzle has it
    MTC_TRY(with_table(m, count, [&](auto &t) {
        constexpr int N = sizeof(t.matrix) / sizeof(t.matrix[0]);
        for (int i = 0; i < count; ++i) t.first[i + 1] = t.first[i] + m[i].parts;
        k_squares<N><<<parts, kThreads, 0, stream>>>(t, partials);
        MTC_TRY(check_launch("orthogonalize (norms)"));
        int64_t units = 0;
        for (int i = 0; i < count; ++i) {
            units += pad_to(m[i].m, tile_of(m[i].m)) / kUnitRows * m[i].x_blocks;
            if (units > INT_MAX) return fail(MTC_ERR_UNSUPPORTED, "a matrix of %d x %d is too large", m[0].m, m[0].n);
            t.first[i + 1] = static_cast<int>(units);
        }
        return launch_dependent("orthogonalize (packing)", k_pack_matrices<N>, static_cast<unsigned>(units), kThreads, 0,
                                stream, t, partials, eps, steps[0].x, packed);
    }));
    return products(m, count, steps.data(), static_cast<int>(steps.size()), packed, bytes, stream);
}

int check_lists(const mtc_desc *tensors, int32_t n, const mtc_desc *outs) {
    if (n < 0 || (n > 0 && (tensors == nullptr || outs == nullptr)))
        return fail(MTC_ERR_INVALID_ARGUMENT, "bad tensor list");
    for (int i = 0; i < n; ++i) {
        MTC_TRY(need_float(&tensors[i], "tensor"));
        MTC_TRY(need_float(&outs[i], "output"));
        const int r = tensors[i].rank;
        if (r < 2) return fail(MTC_ERR_INVALID_ARGUMENT, "tensor %d is no matrix", i);
        bool same = r == outs[i].rank;
        for (int d = 0; same && d < r; ++d) same = tensors[i].shape[d] == outs[i].shape[d];
        if (!same) return fail(MTC_ERR_INVALID_ARGUMENT, "output %d differs in shape from its tensor", i);
        MTC_TRY(need_distinct(&outs[i], "output"));
        if (numel_of(tensors[i]) > 0 && (tensors[i].shape[r - 1] > (1 << 30) || tensors[i].shape[r - 2] > (1 << 30)))
            return fail(MTC_ERR_UNSUPPORTED, "tensor %d is too large", i);
    }
    return need_apart(outs, n);
}

int run(const mtc_desc *tensors, int32_t n, const float *coefficients, int32_t n_steps, float eps, const mtc_desc *outs,
        cudaStream_t stream) {
    MTC_TRY(check_lists(tensors, n, outs));
    std::vector<Step> steps;
    MTC_TRY(follow_steps(coefficients, n_steps, steps));
    std::vector<Matrix> all, small, whole, low, large;  // low: one row of tiles, of 128
    for (int i = 0; i < n; ++i) add_matrices(tensors[i], outs[i], all);
    for (const Matrix &m : all) (is_small(m) ? small : is_whole(m) ? whole : tile_of(m.m) == 128 ? low : large).push_back(m);
    for (std::vector<Matrix> *list : {&large, &low}) {
        for (size_t at = 0; at < list->size();) {
            size_t end = at, bytes = 0;
            while (end < list->size() && end - at < kMostMatrices &&
                   (end == at || bytes + packed_bytes((*list)[end]) <= kGroupBytes))
                bytes += packed_bytes((*list)[end++]);
            MTC_TRY(run_group(list->data() + at, static_cast<int>(end - at), steps, eps, stream));
            at = end;
        }
    }
    if (!whole.empty()) {  // small ones along with them, on other SMs, not after them
        for (size_t i = 0; i < small.size();) {
            if (!is_whole(small[i])) {
                ++i;
                continue;
            }
            whole.push_back(small[i]);
            small.erase(small.begin() + static_cast<std::ptrdiff_t>(i));
        }
        MTC_TRY(whole_matrices(whole.data(), static_cast<int>(whole.size()), steps.data(), static_cast<int>(steps.size()), eps, stream));
    }
    return small.empty() ? MTC_OK : run_small(small, steps, eps, stream);
}

}  // namespace
}  // namespace ortho
}  // namespace mtc

using namespace mtc;

extern "C" int mtc_orthogonalize(const mtc_desc *tensors, int32_t n, const float *coefficients, int32_t steps, float eps,
                                 const mtc_desc *outs, void *stream) {
    clear_error();
    if (steps < 1 || steps > ortho::kMostSteps || coefficients == nullptr)
        return fail(MTC_ERR_INVALID_ARGUMENT, "%d steps; 1 to %d are possible", steps, ortho::kMostSteps);
    if (!(eps >= 0.0f && eps < INFINITY)) return fail(MTC_ERR_INVALID_ARGUMENT, "eps %g is not a number >= 0", eps);
    try {
        return ortho::run(tensors, n, coefficients, steps, eps, outs, static_cast<cudaStream_t>(stream));
    } catch (const std::exception &e) {
        return fail(MTC_ERR_RUNTIME, "orthogonalize: %s", e.what());
    }
}
