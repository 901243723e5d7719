// Linear cross entropy of few rows, or over few classes: up to 16 of either.
//
// The few (rows of x, or rows of W) stay in shared memory and registers, the many (W, or x)
// stream past them: once for the logits and once more, next to the writing of their own
// gradient, for the gradients.  Bound by that streaming: one row against a 32000 x 1024 layer
// reads 131 MB in 27 us (4.9 TB/s), against 131072 x 4096 2.1 GB in 324 us (6.6 TB/s).
// Float32 products on the FMA units: with 16 of the few 16 FMAs for 4 bytes, which take about
// twice as long as the bytes.
//
// k_few_logits: a warp takes four of the many at a time, 128 columns a step and the next step
// under way, against all of the few; one lane for each of the 4 R logits.  Of few rows a lane
// keeps the softmax of its logits, joined over the CTAs afterwards; over few classes a row's
// logits are all in one warp, which writes the loss and g at once.
// k_few_grad: a CTA takes 128 (64) columns and a part of the many; the columns of the few and
// of their gradient stay in registers, the gradient of the many is written as it goes: 4 rows
// against 131072 x 2048 take 566 us for the loss and all gradients, where reading W twice and
// writing dW takes 492 us at the rate of a copy; 16 rows 1267 us, bound by the FMAs.  (The tensor
// path takes 1267 us for 17 rows, which is where the limit of 16 comes from.)
#include <cfloat>
#include <climits>
#include <cstring>

#include "linear_ce.cuh"

namespace mtc {
namespace {

constexpr int kFewThreads = 256;
constexpr int kFewShared = 160 * 1024;

// One of the two operands with its gradient.
struct Side {
    const float *p;
    int64_t rs, cs, rows;
    float *grad;  // null: not wanted
    int64_t g_rs, g_cs;
};

struct FewArgs {
    Side few, many;
    int vec, grad_vec;   // float4 access to the many, to their gradient
    int d_pad;           // a row of the few in shared memory, a multiple of 128
    float *z;            // few rows: the logits [N][V]; null: not wanted
    float *g;            // [many][R]
    Softmax *parts;      // [CTAs][R]
    int n_parts;
    float *z_target;     // [R]
    float *few_parts;    // [splits][few][D + 1], the last column the bias gradient over few classes
    int splits;
    unsigned long long *err;
};

// Sums over the warp of COUNT values a lane at once (COUNT a power of two up to 32): each
// step halves the list, a lane keeping the half its number has the bit for, so that lane l
// ends with the sum of value l % COUNT after COUNT - 1 shuffles and not 5 COUNT.
template <int COUNT>
__device__ __forceinline__ float warp_sums(const float *a) {
    const int lane = threadIdx.x % 32;
    float v[COUNT];
#pragma unroll
    for (int i = 0; i < COUNT; ++i) v[i] = a[i];
    int o = 1;
#pragma unroll
    for (int left = COUNT / 2; left > 0; left /= 2, o *= 2) {
#pragma unroll
        for (int i = 0; i < left; ++i) {
            const bool odd = (lane & o) != 0;
            const float keep = odd ? v[2 * i + 1] : v[2 * i], give = odd ? v[2 * i] : v[2 * i + 1];
            v[i] = keep + __shfl_xor_sync(0xFFFFFFFFu, give, o);
        }
    }
    for (; o < 32; o *= 2) v[0] += __shfl_xor_sync(0xFFFFFFFFu, v[0], o);
    return v[0];
}

// One step of a warp: 128 columns of four of the many.  Without VEC a lane's four columns are
// 32 apart, so that a load is contiguous where they are.
template <bool VEC>
__device__ __forceinline__ void load_step(const Side &m, int64_t D, int64_t v0, int64_t c0, float4 (&x)[4]) {
    const int lane = threadIdx.x % 32;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float *row = m.p + (v0 + j < m.rows ? v0 + j : m.rows - 1) * m.rs;
        x[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (VEC) {
            const int64_t c = c0 + lane * 4;
            if (c < D) x[j] = __ldcs(reinterpret_cast<const float4 *>(row + c));
        } else {
            const int64_t c = c0 + lane;
            if (c < D) x[j].x = __ldcs(row + c * m.cs);
            if (c + 32 < D) x[j].y = __ldcs(row + (c + 32) * m.cs);
            if (c + 64 < D) x[j].z = __ldcs(row + (c + 64) * m.cs);
            if (c + 96 < D) x[j].w = __ldcs(row + (c + 96) * m.cs);
        }
    }
}

// CTAs an SM holds, by registers: with one or two rows the loads in flight decide, and those
// come from warps.
constexpr int few_resident(int R) { return R <= 2 ? 4 : R <= 4 ? 3 : 2; }

template <int R, bool VEC, bool CLASSES>
__global__ void __launch_bounds__(kFewThreads, few_resident(R)) k_few_logits(const LinearCe p, const FewArgs a) {
    extern __shared__ __align__(16) float xs[];  // the few: [R][d_pad]
    __shared__ int target[R];
    __shared__ Softmax warps[kFewThreads / 32][R];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int64_t many = a.many.rows;
    const int64_t step = static_cast<int64_t>(gridDim.x) * (kFewThreads / 32) * 4;
    int64_t v0 = (static_cast<int64_t>(blockIdx.x) * (kFewThreads / 32) + warp) * 4, c0 = 0;
    float4 w[4], next[4];
    if (v0 < many) load_step<VEC>(a.many, p.D, v0, c0, w);  // under way while the few arrive
    if (!CLASSES && threadIdx.x < R)
        target[threadIdx.x] = threadIdx.x < p.N ? row_target(p, threadIdx.x, a.err, blockIdx.x == 0) : -1;
    for (int n = 0; n < R; ++n)
        for (int d = threadIdx.x; d < a.d_pad; d += kFewThreads)
            xs[n * a.d_pad + d] = n < a.few.rows && d < p.D ? a.few.p[n * a.few.rs + d * a.few.cs] : 0.0f;
    __syncthreads();
    if (!CLASSES) {
        for (int n = 0; n < R; ++n)
            if (target[n] < 0)
                for (int d = threadIdx.x; d < a.d_pad; d += kFewThreads) xs[n * a.d_pad + d] = 0.0f;
        __syncthreads();
    }
    constexpr int kMine = (4 * R + 31) / 32;  // logits of a lane: i = lane + 32 k is few i / 4 and many i % 4
    Softmax mine[kMine];
#pragma unroll
    for (int k = 0; k < kMine; ++k) mine[k] = no_logits();
    float acc[4 * R];
#pragma unroll
    for (int i = 0; i < 4 * R; ++i) acc[i] = 0.0f;
    while (v0 < many) {
        int64_t v1 = v0, c1 = c0 + 128;
        if (c1 >= p.D) {
            c1 = 0;
            v1 += step;
        }
        if (v1 < many) load_step<VEC>(a.many, p.D, v1, c1, next);
        if (c0 < p.D) {
#pragma unroll
            for (int n = 0; n < R; ++n) {
                const float *row = xs + n * a.d_pad + c0;
                float4 y;
                if (VEC) y = *reinterpret_cast<const float4 *>(row + lane * 4);
                else y = make_float4(row[lane], row[lane + 32], row[lane + 64], row[lane + 96]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float &c = acc[4 * n + j];
                    c = fmaf(w[j].x, y.x, c);
                    c = fmaf(w[j].y, y.y, c);
                    c = fmaf(w[j].z, y.z, c);
                    c = fmaf(w[j].w, y.w, c);
                }
            }
        }
        if (v1 != v0) {
            float z[kMine];
#pragma unroll
            for (int k = 0; k < kMine; ++k) z[k] = warp_sums<(4 * R < 32 ? 4 * R : 32)>(acc + 32 * k);
            if (CLASSES) {
                const int64_t n = v0 + lane % 4;  // the lanes of a row: its classes, lane / 4 apart
                const bool in = n < many && (R >= 8 || lane < 4 * R);
                const int t = n < many ? row_target(p, n, a.err, lane < 4) : -1;
                Softmax s = no_logits();
                float zt = -INFINITY;
#pragma unroll
                for (int k = 0; k < kMine; ++k) {
                    const int v = lane / 4 + 8 * k;
                    if (!in || v >= p.V) continue;
                    if (p.bias != nullptr) z[k] += __ldg(p.bias + v * p.b_s);
                    s = merge(s, one_logit(z[k]));
                    if (v == t) zt = z[k];
                }
                s = merge_lanes(s, 4, 32);
#pragma unroll
                for (int o = 4; o < 32; o *= 2) {  // the one lane that has the target's (which may be NaN)
                    const float other = __shfl_xor_sync(0xFFFFFFFFu, zt, o);
                    if (zt == -INFINITY) zt = other;
                }
                const LogSum l = s.log_sum();
                if (lane < 4 && n < many) {
                    if (p.loss != nullptr) p.loss[n * p.loss_s] = t < 0 ? 0.0f : l.loss(zt);
                    if (p.lse != nullptr) p.lse[n * p.lse_s] = t < 0 ? 0.0f : l.lse();
                }
                if (a.g != nullptr && in) {
                    const float d = t < 0 ? 0.0f : p.dloss[n * p.dl_s];
#pragma unroll
                    for (int k = 0; k < kMine; ++k) {
                        const int v = lane / 4 + 8 * k;
                        if (v < R) a.g[n * R + v] = t < 0 || v >= p.V ? 0.0f : softmax_grad(l.of(z[k]), d, v == t);
                    }
                }
            } else {
#pragma unroll
                for (int k = 0; k < kMine; ++k) {
                    const int i = lane + 32 * k, n = i / 4;
                    const int64_t v = v0 + i % 4;
                    if (n >= R || n >= p.N || v >= p.V) continue;
                    if (p.bias != nullptr) z[k] += __ldg(p.bias + v * p.b_s);
                    if (a.z != nullptr) a.z[n * p.V + v] = z[k];
                    if (v == target[n]) a.z_target[n] = z[k];
                    mine[k] = merge(mine[k], one_logit(z[k]));
                }
            }
#pragma unroll
            for (int i = 0; i < 4 * R; ++i) acc[i] = 0.0f;
        }
        v0 = v1;
        c0 = c1;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = next[j];
    }
    if constexpr (!CLASSES) {
#pragma unroll
        for (int k = 0; k < kMine; ++k) {
            const Softmax s = merge_lanes(mine[k], 1, 4);
            const int i = lane + 32 * k;
            if (i % 4 == 0 && i / 4 < R) warps[warp][i / 4] = s;
        }
        __syncthreads();
        if (threadIdx.x < R) {
            Softmax s = warps[0][threadIdx.x];
            for (int w = 1; w < kFewThreads / 32; ++w) s = merge(s, warps[w][threadIdx.x]);
            a.parts[blockIdx.x * R + threadIdx.x] = s;
        }
    }
}

// lse of row n from the CTAs' parts; every lane of the warp gets it.
__device__ __forceinline__ LogSum few_lse(const FewArgs &a, int R, int n) {
    Softmax s = no_logits();
    const Softmax *parts = a.parts + n;
#pragma unroll 8
    for (int i = threadIdx.x % 32; i < a.n_parts; i += 32) s = merge(s, parts[i * R]);
    return merge_lanes(s, 1, 32).log_sum();
}

__device__ __forceinline__ void store_loss(const LinearCe &p, const FewArgs &a, int n, int target, LogSum l) {
    if (p.loss != nullptr) p.loss[n * p.loss_s] = target < 0 ? 0.0f : l.loss(a.z_target[n]);
    if (p.lse != nullptr) p.lse[n * p.lse_s] = target < 0 ? 0.0f : l.lse();
}

__global__ void __launch_bounds__(32 * kFewRows) k_few_loss(const LinearCe p, const FewArgs a, int R) {
    wait_for_previous();
    const int n = threadIdx.x / 32;
    if (n >= p.N) return;
    const LogSum l = few_lse(a, R, n);
    if (threadIdx.x % 32 == 0) store_loss(p, a, n, row_target(p, n, a.err, false), l);
}

// With eight rows or more the exponentials are worth a pass of their own: z [N][V] -> g [V][R],
// instead of once for each slab of columns in k_few_grad.  The loss and the bias gradient with it.
constexpr bool g_before(int R, bool classes) { return classes || R >= 8; }

template <int R>
__global__ void __launch_bounds__(kFewThreads) k_few_g(const LinearCe p, const FewArgs a) {
    wait_for_previous();
    __shared__ LogSum lse[R];
    __shared__ float dloss[R];
    __shared__ int target[R];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    for (int n = warp; n < R; n += kFewThreads / 32) {
        const int t = n < p.N ? row_target(p, n, a.err, false) : -1;
        const LogSum l = n < p.N ? few_lse(a, R, n) : LogSum{0.0f, 0.0f};
        if (lane == 0) {
            lse[n] = l;
            target[n] = t;
            dloss[n] = t >= 0 ? p.dloss[n * p.dl_s] : 0.0f;
            if (n < p.N && blockIdx.x == 0) store_loss(p, a, n, t, l);
        }
    }
    __syncthreads();
    for (int64_t v = static_cast<int64_t>(blockIdx.x) * kFewThreads + threadIdx.x; v < p.V;
         v += static_cast<int64_t>(gridDim.x) * kFewThreads) {
        float g[R], sum = 0.0f;
#pragma unroll
        for (int n = 0; n < R; ++n) g[n] = n < p.N ? a.z[n * p.V + v] : 0.0f;
#pragma unroll
        for (int n = 0; n < R; ++n) {
            g[n] = target[n] >= 0 ? softmax_grad(lse[n].of(g[n]), dloss[n], v == target[n]) : 0.0f;
            sum += g[n];
        }
        if (p.db != nullptr) p.db[v * p.db_s] = sum;
#pragma unroll
        for (int n = 0; n < R; ++n) a.g[v * R + n] = g[n];
    }
}

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }

// C columns a lane, 32 C a CTA.  Two columns a multiply-add (FFMA2); g lies in shared memory
// twice over, as its operand wants it.
template <int R, int C, bool CLASSES>
__global__ void __launch_bounds__(kFewThreads, R <= 2 ? 3 : 2) k_few_grad(const LinearCe p, const FewArgs a) {
    wait_for_previous();
    __shared__ LogSum lse[R];
    __shared__ float dloss[R];
    __shared__ int target[R];
    __shared__ __align__(16) float sums[kFewThreads / 32][32 * C];
    __shared__ __align__(16) float2 gs[kFewThreads / 32][32][R + 2];  // of a warp's 32 of the many; a lane's row off the banks of the next
    __shared__ bool live[kFewThreads / 32][32];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    constexpr bool kBefore = g_before(R, CLASSES);
    if (!CLASSES) {
        for (int n = warp; n < R; n += kFewThreads / 32) {
            const int t = n < p.N ? row_target(p, n, a.err, false) : -1;
            const LogSum l = !kBefore && n < p.N ? few_lse(a, R, n) : LogSum{0.0f, 0.0f};
            if (lane == 0) {
                lse[n] = l;
                target[n] = t;
                dloss[n] = t >= 0 ? p.dloss[n * p.dl_s] : 0.0f;
                if (!kBefore && n < p.N && blockIdx.x == 0 && blockIdx.y == 0) store_loss(p, a, n, t, l);
            }
        }
        __syncthreads();
    }
    const Side &m = a.many;
    const int64_t c0 = (static_cast<int64_t>(blockIdx.x) * 32 + lane) * C;
    const int cols = static_cast<int>(p.D - c0 < 0 ? 0 : p.D - c0 < C ? p.D - c0 : C);
    const bool few_grad = a.few_parts != nullptr;
    float2 x[R][C / 2], dx[R][C / 2];
    float db[R];
#pragma unroll
    for (int n = 0; n < R; ++n) {
        db[n] = 0.0f;
        const float *row = a.few.p + n * a.few.rs + c0 * a.few.cs;
        const bool has = n < a.few.rows && (CLASSES || target[n] >= 0);
#pragma unroll
        for (int c = 0; c < C / 2; ++c) {
            dx[n][c] = make_float2(0.0f, 0.0f);
            x[n][c].x = has && 2 * c < cols ? row[2 * c * a.few.cs] : 0.0f;
            x[n][c].y = has && 2 * c + 1 < cols ? row[(2 * c + 1) * a.few.cs] : 0.0f;
        }
    }
    const int64_t step = static_cast<int64_t>(gridDim.y) * (kFewThreads / 32) * 32;
    for (int64_t v0 = (static_cast<int64_t>(blockIdx.y) * (kFewThreads / 32) + warp) * 32; v0 < m.rows; v0 += step) {
        const int64_t v = v0 + lane;
        float sum = 0.0f;
        bool any = !CLASSES;  // a row without a loss may hold anything
        __syncwarp();
#pragma unroll
        for (int n = 0; n < R; ++n) {
            float g = 0.0f;
            if (kBefore) {
                if (v < m.rows) g = a.g[v * R + n];
                any |= g != 0.0f;
                if (CLASSES) db[n] += g;
            } else {
                if (n < p.N && v < p.V && target[n] >= 0) g = softmax_grad(lse[n].of(a.z[n * p.V + v]), dloss[n], v == target[n]);
                sum += g;
            }
            gs[warp][lane][n] = make_float2(g, g);
        }
        if (CLASSES) live[warp][lane] = any;
        __syncwarp();
        if (!kBefore && p.db != nullptr && blockIdx.x == 0 && v < p.V) p.db[v * p.db_s] = sum;
        const int count = static_cast<int>(m.rows - v0 < 32 ? m.rows - v0 : 32);
        constexpr int U = R <= 4 ? 8 : 4;
        for (int j0 = 0; j0 < count; j0 += U) {
            float2 w[U][C / 2];
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int c = 0; c < C / 2; ++c) w[u][c] = make_float2(0.0f, 0.0f);
                if (!few_grad || j0 + u >= count || (CLASSES && !live[warp][j0 + u])) continue;
                const float *src = m.p + (v0 + j0 + u) * m.rs + c0 * m.cs;
                if (a.vec) {
                    if (cols <= 0) continue;
                    if (C == 4) {
                        const float4 y = __ldcs(reinterpret_cast<const float4 *>(src));
                        w[u][C / 2 - 1] = make_float2(y.z, y.w);
                        w[u][0] = make_float2(y.x, y.y);
                    } else {
                        w[u][0] = __ldcs(reinterpret_cast<const float2 *>(src));
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < C / 2; ++c) {
                        if (2 * c < cols) w[u][c].x = __ldcs(src + 2 * c * m.cs);
                        if (2 * c + 1 < cols) w[u][c].y = __ldcs(src + (2 * c + 1) * m.cs);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (j0 + u >= count) break;
                float2 dm[C / 2];
#pragma unroll
                for (int c = 0; c < C / 2; ++c) dm[c] = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int n = 0; n < R; ++n) {
                    const float2 gn = gs[warp][j0 + u][n];
#pragma unroll
                    for (int c = 0; c < C / 2; ++c) {
                        dx[n][c] = fma2(gn, w[u][c], dx[n][c]);
                        dm[c] = fma2(gn, x[n][c], dm[c]);
                    }
                }
                if (m.grad == nullptr) continue;
                if (CLASSES && !live[warp][j0 + u]) {  // W may hold infinities; the row has no loss
#pragma unroll
                    for (int c = 0; c < C / 2; ++c) dm[c] = make_float2(0.0f, 0.0f);
                }
                float *to = m.grad + (v0 + j0 + u) * m.g_rs + c0 * m.g_cs;
                if (a.grad_vec) {
                    if (cols <= 0) continue;
                    if (C == 4) *reinterpret_cast<float4 *>(to) = make_float4(dm[0].x, dm[0].y, dm[C / 2 - 1].x, dm[C / 2 - 1].y);
                    else *reinterpret_cast<float2 *>(to) = dm[0];
                } else {
#pragma unroll
                    for (int c = 0; c < C / 2; ++c) {
                        if (2 * c < cols) to[2 * c * m.g_cs] = dm[c].x;
                        if (2 * c + 1 < cols) to[(2 * c + 1) * m.g_cs] = dm[c].y;
                    }
                }
            }
        }
    }
    if (!few_grad) return;
#pragma unroll
    for (int n = 0; n < R; ++n) {
        if (n >= a.few.rows) break;
        __syncthreads();
#pragma unroll
        for (int c = 0; c < C / 2; ++c) *reinterpret_cast<float2 *>(&sums[warp][lane * C + 2 * c]) = dx[n][c];
        __syncthreads();
        float *part = a.few_parts + (blockIdx.y * a.few.rows + n) * (p.D + 1);
        if (static_cast<int>(threadIdx.x) < 32 * C) {
            const int64_t d = static_cast<int64_t>(blockIdx.x) * 32 * C + threadIdx.x;
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < kFewThreads / 32; ++w) s += sums[w][threadIdx.x];
            if (d < p.D) part[d] = s;
        }
        if (CLASSES && blockIdx.x == 0) {
            float s = db[n];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
            __syncthreads();
            if (lane == 0) sums[warp][0] = s;
            __syncthreads();
            if (threadIdx.x == 0) {
                for (int w = 1; w < kFewThreads / 32; ++w) s += sums[w][0];
                part[p.D] = s;
            }
        }
    }
}

// The gradient of the few: eight warps take the parts of 32 elements in turn.
template <bool CLASSES>
__global__ void __launch_bounds__(256) k_few_join(const LinearCe p, const FewArgs a) {
    wait_for_previous();
    __shared__ float sums[8][32];
    const int64_t width = p.D + 1, total = a.few.rows * width;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.x % 32;
    const int64_t n = i / width, d = i - n * width;
    float sum = 0.0f;
    if (i < total && (CLASSES || d < p.D)) {
#pragma unroll 8
        for (int s = threadIdx.x / 32; s < a.splits; s += 8) sum += a.few_parts[s * total + i];
    }
    sums[threadIdx.x / 32][threadIdx.x % 32] = sum;
    __syncthreads();
    if (threadIdx.x >= 32 || i >= total) return;
    for (int w = 1; w < 8; ++w) sum += sums[w][threadIdx.x];
    if (d == p.D) {
        if (CLASSES && p.db != nullptr) p.db[n * p.db_s] = sum;
        return;
    }
    if (a.few.grad == nullptr) return;
    if (!CLASSES && row_target(p, n, a.err, false) < 0) sum = 0.0f;
    a.few.grad[n * a.few.g_rs + d * a.few.g_cs] = sum;
}

template <int R, bool CLASSES>
int few_path(const LinearCe &p, FewArgs a, cudaStream_t stream) {
    const int sms = sm_count(current_device());
    const bool grads = p.dloss != nullptr && (p.dx != nullptr || p.dw != nullptr || p.db != nullptr);
    const Side &m = a.many;
    a.vec = aligned16(m.p) && m.cs == 1 && m.rs % 4 == 0 && p.D % 4 == 0;
    a.grad_vec = aligned16(m.grad) && m.g_cs == 1 && m.g_rs % 4 == 0 && p.D % 4 == 0;
    a.d_pad = static_cast<int>((p.D + 127) / 128 * 128);
    const size_t shared = static_cast<size_t>(R) * a.d_pad * 4;
    const int64_t wanted = (m.rows + 31) / 32;  // CTAs of 8 warps, four of the many each
    const int64_t most_ctas = static_cast<int64_t>(sms) * (shared > 72 * 1024 ? 1 : shared > 48 * 1024 ? 2 : few_resident(R));
    a.n_parts = static_cast<int>(wanted < most_ctas ? wanted : most_ctas);  // every SM as many: a CTA loads the few once
    constexpr int C = R <= 8 ? 4 : 2;  // columns a lane of k_few_grad: 2 R C values in registers
    const int64_t slabs = p.D > 0 ? (p.D + 32 * C - 1) / (32 * C) : 1;
    // two full waves of CTAs, two of which fill an SM
    const int64_t splits = static_cast<int64_t>(sms) * 4 / slabs > 0 ? static_cast<int64_t>(sms) * 4 / slabs : 1;
    const int64_t most = (m.rows + 255) / 256;  // 8 warps of 32
    a.splits = static_cast<int>(splits < most ? splits : most);
    const bool few_grad = grads && (a.few.grad != nullptr || (CLASSES && p.db != nullptr));
    const size_t parts = padded(static_cast<size_t>(a.n_parts) * R * sizeof(Softmax));
    const size_t zs = grads && !CLASSES ? padded(static_cast<size_t>(m.rows) * p.N * 4) : 0;
    const size_t gs = grads && g_before(R, CLASSES) ? padded(static_cast<size_t>(m.rows) * R * 4) : 0;
    const size_t fs = few_grad ? padded(static_cast<size_t>(a.splits) * a.few.rows * (p.D + 1) * 4) : 0;
    MTC_TRY(device_error_word(&a.err));
    Workspace ws;
    if (!CLASSES || grads) {
        MTC_TRY(ws.allocate(256 + parts + zs + gs + fs, stream));
        a.z_target = ws.take<float>(256);
        a.parts = ws.take<Softmax>(parts);
        float *z = ws.take<float>(zs);
        float *g = ws.take<float>(gs);
        float *f = ws.take<float>(fs);
        a.z = zs > 0 ? z : nullptr;
        a.g = gs > 0 ? g : nullptr;
        a.few_parts = few_grad ? f : nullptr;
    }
    if (a.vec) {
        MTC_CUDA_TRY(cudaFuncSetAttribute(k_few_logits<R, true, CLASSES>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewShared));
        k_few_logits<R, true, CLASSES><<<a.n_parts, kFewThreads, shared, stream>>>(p, a);
    } else {
        MTC_CUDA_TRY(cudaFuncSetAttribute(k_few_logits<R, false, CLASSES>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewShared));
        k_few_logits<R, false, CLASSES><<<a.n_parts, kFewThreads, shared, stream>>>(p, a);
    }
    MTC_TRY(check_launch("linear cross entropy (few)"));
    if (!grads) {
        if (CLASSES) return MTC_OK;
        return launch_dependent("linear cross entropy (loss)", k_few_loss, 1, static_cast<unsigned>(32 * p.N), 0, stream,
                                p, a, R);
    }
    if constexpr (!CLASSES && g_before(R, CLASSES)) {
        const int64_t ctas = (p.V + kFewThreads - 1) / kFewThreads;
        MTC_TRY(launch_dependent("linear cross entropy (few, gradient of the logits)", k_few_g<R>,
                                 static_cast<unsigned>(ctas < sms * 4 ? ctas : sms * 4), kFewThreads, 0, stream, p, a));
    }
    const dim3 grid(static_cast<unsigned>(slabs), static_cast<unsigned>(a.splits));
    MTC_TRY((launch_dependent("linear cross entropy (few, gradients)", k_few_grad<R, C, CLASSES>, grid, kFewThreads, 0,
                              stream, p, a)));
    if (!few_grad) return MTC_OK;
    return launch_dependent("linear cross entropy (few, join)", k_few_join<CLASSES>,
                            static_cast<unsigned>((a.few.rows * (p.D + 1) + 31) / 32), 256, 0, stream, p, a);
}

template <bool CLASSES>
int few_by_count(const LinearCe &p, const FewArgs &a, cudaStream_t stream) {
    if (a.few.rows == 1) return few_path<1, CLASSES>(p, a, stream);
    if (a.few.rows == 2) return few_path<2, CLASSES>(p, a, stream);
    if (a.few.rows <= 4) return few_path<4, CLASSES>(p, a, stream);
    if (a.few.rows <= 8) return few_path<8, CLASSES>(p, a, stream);
    return few_path<16, CLASSES>(p, a, stream);
}

// Up to 16 rows of D columns, in the next power of two, fit in shared memory.
bool fits(int64_t rows, int64_t D) {
    int64_t r = 1;
    while (r < rows) r *= 2;
    return rows <= kFewRows && r * ((D + 127) / 128 * 512) <= kFewShared;
}

}  // namespace

bool few_rows(const LinearCe &p) { return fits(p.N, p.D); }
bool few_classes(const LinearCe &p) { return fits(p.V, p.D); }

int linear_ce_few(const LinearCe &p, bool classes, cudaStream_t stream) {
    FewArgs a;
    std::memset(&a, 0, sizeof(a));
    const bool grads = p.dloss != nullptr;
    const Side x{p.x, p.x_rs, p.x_cs, p.N, grads ? p.dx : nullptr, p.dx_rs, p.dx_cs};
    const Side w{p.w, p.w_rs, p.w_cs, p.V, grads ? p.dw : nullptr, p.dw_rs, p.dw_cs};
    a.few = classes ? w : x;
    a.many = classes ? x : w;
    return classes ? few_by_count<true>(p, a, stream) : few_by_count<false>(p, a, stream);
}

}  // namespace mtc
