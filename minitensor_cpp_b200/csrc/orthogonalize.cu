// Updates of weight matrices made orthogonal by Newton-Schulz products:
//
//   X = T / (|T|_F + eps),  and in every step  S = X X^T,  B = b S + c S^2,  X <- a X + B X
//
// on the shorter side of T.  Each singular value x of X goes to p(x) = a x + b x^3 + c x^5, so it
// stays in [0, s], s = 1 at first and then the maximum of |p| over [0, s].  The host follows s;
// the elements of X, S and B are below it and its polynomials, which gives the packed operands
// of the tensor cores fixed scales: nothing is looked at while the products run.
//
// Matrices of few rows are worked on in shared memory, in float32 (k_slabs), others of up to 128 x
// 128 by a CTA each that has them there on the tensor cores.  All others are
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

template <int THREADS>
__device__ __forceinline__ double block_sum(double v) {
    __shared__ double part[THREADS / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    __syncthreads();
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) v += part[i];
    return v;
}

// ------------------------------------------------- matrices of few rows --
//
// Up to 64 rows, in float32: the CTAs of a cluster (or one) have equal parts of the columns in
// shared memory for all steps.  Each adds up the products of its own columns, S is the sum of
// the CTAs' in their order, everything of m x m is worked out by all of them, and B X needs no
// other columns than its own, so X is replaced where it lies.  S and B are symmetric: tiles of 4 x 4
// on and above the diagonal are worked out, and where that leaves threads, they share K.
// Bound by shared memory (of B X a warp reads 20 lines of 128 bytes for 64 multiply-adds) and, where
// there is little to do, by the syncs: five steps of 3 x 64 take 15 us, of 48 x 48 39 (packed for the
// tensor cores of one CTA 46), of 60 x 2000 113 (in 17 launches, as tiles of 128 rows, 182), 64 of
// 10 x 8192 152 (1410).  256 threads that work out all of S took 64 us for 48 x 48, and where each
// CTA of eight added up all parts itself, 376 for 60 x 2000.

struct SlabSteps {
    int n;
    float eps;
    float a[kMostSteps], b[kMostSteps], c[kMostSteps];
};

constexpr int kSlabRows = 64, kMostCluster = 8, kSlabThreads = 512;
constexpr int kJoin = 17 * kSlabThreads;  // floats in which the threads' parts of S are added up

// Rows of an odd number of float4, so that eight neighbours' lie in different banks.
__host__ __device__ inline int slab_pitch(int cols) { return ((cols + 3) / 4 | 1) * 4; }
__host__ __device__ inline int slab_columns(int n, int ctas) { return ((n + ctas - 1) / ctas + 3) / 4 * 4; }
inline size_t slab_bytes(int m, int n, int ctas) {
    const size_t rows = (m + 3) / 4 * 4;
    return 4 * (rows * (static_cast<size_t>(slab_pitch(slab_columns(n, ctas))) + 3 * slab_pitch(m)) + kJoin);
}
constexpr size_t kMostSlab = 224 * 1024;

__device__ __forceinline__ uint32_t of_cta(const void *p, int rank) {
    uint32_t out;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                 : "=r"(out) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(rank));
    return out;
}

__device__ __forceinline__ void all_ctas() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// acc += x[row + R i][k..] . x[col + R j][k..] over k = first, first + step, ... below K; rows and
// columns R apart, so that neighbours read neighbouring rows.
__device__ __forceinline__ void slab_products(const float *x, int pitch, int row, int col, int R, int first, int step, int K,
                                              float (&acc)[4][4]) {
#pragma unroll 2
    for (int k = first; k < K; k += step) {
        float4 u[4], v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u[i] = *reinterpret_cast<const float4 *>(x + (row + R * i) * pitch + k);
            v[i] = *reinterpret_cast<const float4 *>(x + (col + R * i) * pitch + k);
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
}

__device__ __forceinline__ void write_both(float *s, int pitch, int r, int c, float v) {
    s[r * pitch + c] = v;
    s[c * pitch + r] = v;
}

template <int N>
__global__ void __launch_bounds__(kSlabThreads) k_slabs(const __grid_constant__ Table<N> table, const SlabSteps steps) {
    extern __shared__ __align__(16) float smem[];
    __shared__ double squares_of;
    uint32_t size_u, rank_u;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(size_u));
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank_u));
    const int size = static_cast<int>(size_u), rank = static_cast<int>(rank_u), thread = threadIdx.x;
    const Matrix &mt = table.matrix[blockIdx.x / size_u];
    const int m = mt.m, rows = (m + 3) / 4 * 4, R = rows / 4;
    const int per = slab_columns(mt.n, size), c0 = rank * per, L = max(min(mt.n - c0, per), 0);
    const int pitch = slab_pitch(per), s_pitch = slab_pitch(m), square = rows * s_pitch, total = rows * pitch;
    float *const x = smem, *const s = x + total, *const b = s + square, *const parts = b + square, *const join = parts + square;
    // rows and columns up to whole fours are zeros, and stay so
    const bool along = mt.cs == 1 || mt.rs != 1;
    double squares = 0.0;
    for (int first = thread; first < total; first += 4 * kSlabThreads) {
        float v[4];
        int to[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = first + u * kSlabThreads;
            const int r = along ? i / pitch : i % rows, c = along ? i % pitch : i / rows;
            to[u] = r * pitch + c;
            v[u] = r < m && c < L ? mt.src[r * mt.rs + (c0 + c) * mt.cs] : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (first + u * kSlabThreads < total) {
                x[to[u]] = v[u];
                squares += static_cast<double>(v[u]) * v[u];
            }
    }
    squares = block_sum<kSlabThreads>(squares);
    if (size > 1) {
        if (thread == 0) squares_of = squares;
        all_ctas();
        squares = 0.0;
        for (int c = 0; c < size; ++c) {
            double v;
            asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(of_cta(&squares_of, c)) : "memory");
            squares += v;
        }
    }
    const Factor factor(inverse_norm(squares, steps.eps), 0);
    for (int i = thread; i < total; i += kSlabThreads) x[i] = factor(x[i]);
    __syncthreads();
    // the tiles of S on and above the diagonal, each of `groups` threads that share its K (and have some: with
    // all 512 3 x 64 took 25 us)
    const int tiles = R * (R + 1) / 2, groups = min(kSlabThreads / tiles, per / 4), group = thread / tiles, tile = thread % tiles;
    const int sums = max(groups / 16, 1);  // of an element of S, by as many threads
    float *const halfway = join + 16 * kSlabThreads;
    int row = 0, col = tile;
    while (col >= R - row) col -= R - row++;
    col += row;
    const int wide = kSlabThreads / R, ti = thread / wide;  // columns' fours of a pass of B X
    for (int k = 0; k < steps.n; ++k) {
        float *const mine = size > 1 ? parts : s;
        if (group < groups) {
            float acc[4][4] = {};
            slab_products(x, pitch, row, col, R, 4 * group, 4 * groups, L, acc);
#pragma unroll
            for (int e = 0; e < 16; ++e) join[(group * 16 + e) * tiles + tile] = acc[e / 4][e % 4];
        }
        __syncthreads();
        if (group / 16 < sums && group < groups)
            for (int e = group % 16; e < 16; e += min(groups, 16)) {
                float sum = 0.0f;
                for (int g = group / 16; g < groups; g += sums) sum += join[(g * 16 + e) * tiles + tile];
                if (sums > 1) halfway[(group / 16 * 16 + e) * tiles + tile] = sum;
                else write_both(mine, s_pitch, row + R * (e / 4), col + R * (e % 4), sum);
            }
        if (sums > 1) {
            __syncthreads();
            if (group < 16) {
                float sum = 0.0f;
                for (int p = 0; p < sums; ++p) sum += halfway[(p * 16 + group) * tiles + tile];
                write_both(mine, s_pitch, row + R * (group / 4), col + R * (group % 4), sum);
            }
        }
        if (size > 1) {
            all_ctas();  // also: all are through with the last S
            for (int o = 4 * (rank + size * thread); o < square; o += 4 * size * kSlabThreads) {
                float4 v[kMostCluster];
#pragma unroll
                for (int c = 0; c < kMostCluster; ++c)
                    if (c < size)
                        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                     : "=f"(v[c].x), "=f"(v[c].y), "=f"(v[c].z), "=f"(v[c].w) : "r"(of_cta(parts + o, c)) : "memory");
                float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int c = 0; c < kMostCluster; ++c)
                    if (c < size) sum = make_float4(sum.x + v[c].x, sum.y + v[c].y, sum.z + v[c].z, sum.w + v[c].w);
#pragma unroll
                for (int c = 0; c < kMostCluster; ++c)
                    if (c < size)
                        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};"
                                     :: "r"(of_cta(s + o, c)), "f"(sum.x), "f"(sum.y), "f"(sum.z), "f"(sum.w) : "memory");
            }
            all_ctas();
        } else {
            __syncthreads();
        }
        if (group == 0) {
            float acc[4][4] = {};
            slab_products(s, s_pitch, row, col, R, 0, 4, m, acc);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int r = row + R * (e / 4), c = col + R * (e % 4);
                const float v = fmaf(steps.b[k], s[r * s_pitch + c], steps.c[k] * acc[e / 4][e % 4]);
                write_both(b, s_pitch, r, c, v);
            }
        }
        __syncthreads();
        for (int first = 0; 4 * first < L; first += wide) {
            const int tj = first + thread % wide;
            const bool here = ti < R && 4 * tj < L;
            float acc[4][4] = {};
            if (here) {
#pragma unroll 2
                for (int q = 0; q < m; q += 4) {
                    float4 u[4], v[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        u[i] = *reinterpret_cast<const float4 *>(b + (ti + R * i) * s_pitch + q);
                        v[i] = *reinterpret_cast<const float4 *>(x + (q + i) * pitch + 4 * tj);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
                        for (int h = 0; h < 4; ++h) {
                            acc[i][0] = fmaf(w[h], v[h].x, acc[i][0]);
                            acc[i][1] = fmaf(w[h], v[h].y, acc[i][1]);
                            acc[i][2] = fmaf(w[h], v[h].z, acc[i][2]);
                            acc[i][3] = fmaf(w[h], v[h].w, acc[i][3]);
                        }
                    }
                }
            }
            __syncthreads();  // these columns have been read
            if (here) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float4 *const at = reinterpret_cast<float4 *>(x + (ti + R * i) * pitch + 4 * tj);
                    const float4 o = *at;
                    *at = make_float4(fmaf(steps.a[k], o.x, acc[i][0]), fmaf(steps.a[k], o.y, acc[i][1]),
                                      fmaf(steps.a[k], o.z, acc[i][2]), fmaf(steps.a[k], o.w, acc[i][3]));
                }
            }
        }
        __syncthreads();
    }
    const bool out_along = mt.out_cs == 1 || mt.out_rs != 1;
    for (int i = thread; i < m * L; i += kSlabThreads) {
        const int r = out_along ? i / L : i % m, c = out_along ? i % L : i / m;
        mt.dst[r * mt.out_rs + (c0 + c) * mt.out_cs] = x[r * pitch + c];
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
    acc = block_sum<kThreads>(acc);
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
    const Factor factor(inverse_norm(block_sum<kThreads>(squares), eps), scale);
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
        // (scales end at 2^74, where what is smaller would lose digits of its pairs)
        if ((next > 0.0 && next < 0x1p-60) || (s > 0.0 && s < 0x1p-30 && (t.b != 0.0f || t.c != 0.0f)))
            return fail(MTC_ERR_INVALID_ARGUMENT, "step %d: with these coefficients all singular values fall to %g", k,
                        next < s ? next : s);
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

// The fewest CTAs whose shared memory takes the matrix's columns, or 0.
int slab_ctas(const Matrix &mt) {
    for (int c = 1; c <= kMostCluster; c *= 2)
        if (slab_bytes(mt.m, mt.n, c) <= kMostSlab) return c;
    return 0;
}

// Of few rows: worked on in float32.  Up to 128 columns the other way is a CTA with the tensor cores
// (56 x 56: 46.6 us here, 47.6 there; 60 x 60 50 and 47.6; 44 x 128 45.6 and 51.7), beyond 17 launches,
// whose time goes with the columns alone, as rows are padded to 128 (five steps of 64 matrices of
// 48 x 6000 951 and 1116, 64 x 2000 408 and 469, but 52 x 4000 818 and 800, 64 x 2600 797 and 590).
bool is_small(const Matrix &mt) {
    const int64_t m = mt.m, n = mt.n;
    if (m > kSlabRows || slab_ctas(mt) == 0) return false;
    return n <= 128 ? 2 * m * m * n + m * m * m <= 3 * 58 * 58 * 58 : m <= 48 || m * m * n <= 1 << 23;
}

bool is_whole(const Matrix &mt) { return mt.n <= 128; }

// CTAs that run at once: a cluster lies in one part of the GPU, and what is left over of each stays
// empty (64 x 2048 on clusters of eight: 15 of them 134 us, 16 of them 255; on four 208 both).
int64_t room() { return sm_count(current_device()) * 5 / 6; }

// On `ctas` CTAs each, as all of them need, or more while SMs are left over and that pays for the
// clusters' barriers: 32 columns and 25000 products of B X for each (1 x 8192 on one CTA 58 us, on
// four 37, on eight 33; 64 x 200 on two 74, on four 68; but 16 x 128 on one 25, on two 27).
int run_slabs(const std::vector<Matrix> &all, int ctas, const std::vector<Step> &steps, float eps, cudaStream_t stream) {
    SlabSteps s;
    std::memset(&s, 0, sizeof(s));
    s.n = static_cast<int>(steps.size());
    s.eps = eps;
    for (int k = 0; k < s.n; ++k) {
        s.a[k] = steps[k].a;
        s.b[k] = steps[k].b;
        s.c[k] = steps[k].c;
    }
    int64_t most = 0, columns = 0;  // products of a matrix's B X
    for (const Matrix &m : all) {
        const int64_t rows = (m.m + 3) / 4 * 4;
        most = std::max(most, rows * rows * m.n);
        columns = std::max<int64_t>(columns, m.n);
    }
    const int64_t matrices = static_cast<int64_t>(all.size());
    while (ctas < kMostCluster && 2 * ctas * matrices <= room() && most / ctas > 25000 && columns / ctas >= 64) ctas *= 2;
    for (size_t at = 0; at < all.size(); at += kMostMatrices) {
        const int count = static_cast<int>(std::min<size_t>(kMostMatrices, all.size() - at));
        size_t bytes = 0;
        for (int i = 0; i < count; ++i) bytes = std::max(bytes, slab_bytes(all[at + i].m, all[at + i].n, ctas));
        MTC_TRY(with_table(all.data() + at, count, [&](const auto &t) {
            constexpr int N = sizeof(t.matrix) / sizeof(t.matrix[0]);
            MTC_CUDA_TRY(cudaFuncSetAttribute(k_slabs<N>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSlab));
            cudaLaunchAttribute attr;
            std::memset(&attr, 0, sizeof(attr));
            attr.id = cudaLaunchAttributeClusterDimension;
            attr.val.clusterDim.x = static_cast<unsigned>(ctas);
            attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
            cudaLaunchConfig_t config;
            std::memset(&config, 0, sizeof(config));
            config.gridDim = static_cast<unsigned>(count * ctas);
            config.blockDim = kSlabThreads;
            config.dynamicSmemBytes = bytes;
            config.stream = stream;
            config.attrs = &attr;
            config.numAttrs = 1;
            MTC_CUDA_TRY(cudaLaunchKernelEx(&config, k_slabs<N>, t, s));
            return check_launch("orthogonalize (few rows)");
        }));
    }
    return MTC_OK;
}

int run_small(const std::vector<Matrix> &all, const std::vector<Step> &steps, float eps, cudaStream_t stream) {
    int most = 1;
    for (const Matrix &m : all) most = std::max(most, slab_ctas(m));
    if (static_cast<int64_t>(all.size()) * most <= room()) return run_slabs(all, most, steps, eps, stream);  // one launch
    for (int ctas = 1; ctas <= kMostCluster; ctas *= 2) {
        std::vector<Matrix> some;
        for (const Matrix &m : all)
            if (slab_ctas(m) == ctas) some.push_back(m);
        if (!some.empty()) MTC_TRY(run_slabs(some, ctas, steps, eps, stream));
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
        const auto rest = std::stable_partition(small.begin(), small.end(), [](const Matrix &m) { return !is_whole(m); });
        whole.insert(whole.end(), rest, small.end());
        small.erase(rest, small.end());
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
