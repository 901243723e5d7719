// Softmax cross entropy of a linear layer over a large vocabulary, and its gradient.
//
//   z = x W^T + b            lse_n = log sum_v exp z_nv          loss_n = lse_n - z_{n,t_n}
//   g_nv = dloss_n (exp(z_nv - lse_n) - [v = t_n])
//   dx = g W                 dW = g^T x                          db_v = sum_n g_nv
//
// Three paths.  Few rows (up to 16) read W once in float32, whatever its size; small
// problems take a warp a row; the others run on the tensor cores (linear_ce_tc.cu), over
// the rows that have a loss: k_live_rows lists them in order, and only the device knows how
// many there are.
#include <cooperative_groups.h>

#include <cfloat>
#include <climits>
#include <cstring>

#include "linear_ce.cuh"

namespace mtc {
namespace {

constexpr int kListThreads = 1024, kListRows = 4, kListCtas = 16;

__device__ __forceinline__ int block_exclusive(int v, int *warp_sums, int &total) {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xFFFFFFFFu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    const int w = warp_sums[lane];
    total = __reduce_add_sync(0xFFFFFFFFu, w);
    return __reduce_add_sync(0xFFFFFFFFu, lane < warp ? w : 0) + x - v;
}

// The rows with a loss, in order, and from the end of the list backwards those without;
// zero loss and lse of the latter.  One cluster: each CTA counts its part of the rows, the
// counts before it tell where its rows go.
__global__ void __launch_bounds__(kListThreads) k_live_rows(const LinearCe p, const LiveRows live,
                                                            unsigned long long *err) {
    __shared__ int warp_sums[32];
    __shared__ int counted;
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const int me = static_cast<int>(cluster.block_rank()), ctas = static_cast<int>(cluster.num_blocks());
    constexpr int kTile = kListThreads * kListRows;
    const int64_t tiles = (p.N + kTile - 1) / kTile;
    const int64_t begin = tiles * me / ctas * kTile, end_tile = tiles * (me + 1) / ctas * kTile;
    const int64_t end = end_tile < p.N ? end_tile : p.N;
    int64_t t[kListRows];
    auto load = [&](int64_t n0, bool report) {  // targets of the tile at n0; how many have a loss
#pragma unroll
        for (int u = 0; u < kListRows; ++u) {
            const int64_t n = n0 + static_cast<int64_t>(threadIdx.x) * kListRows + u;
            t[u] = n < end ? p.targets[n * p.t_s] : p.ignore;
        }
        int mine = 0;
#pragma unroll
        for (int u = 0; u < kListRows; ++u) {
            if (t[u] == p.ignore) {
                t[u] = -1;
            } else if (t[u] < 0 || t[u] >= p.V) {
                if (report) report_index(err, t[u]);
                t[u] = -1;
            }
            mine += t[u] >= 0;
        }
        return mine;
    };
    int mine = 0;
    for (int64_t n0 = begin; n0 < end; n0 += kTile) mine += load(n0, true);
    int count;
    (void)block_exclusive(mine, warp_sums, count);
    if (threadIdx.x == 0) counted = count;
    cluster.sync();
    int first = 0, all = 0;
    for (int r = 0; r < ctas; ++r) {
        const int c = *cluster.map_shared_rank(&counted, r);
        if (r < me) first += c;
        all += c;
    }
    int64_t dead = p.N - 1 - (begin - first);  // where the next row without a loss goes
    for (int64_t n0 = begin; n0 < end; n0 += kTile) {
        const int has = load(n0, false);
        int total;
        int at = block_exclusive(has, warp_sums, total);
        const int64_t n1 = n0 + static_cast<int64_t>(threadIdx.x) * kListRows;
        int64_t none = dead - (static_cast<int64_t>(threadIdx.x) * kListRows - at);
        at += first;
#pragma unroll
        for (int u = 0; u < kListRows; ++u) {
            const int64_t n = n1 + u;
            if (n >= end) break;
            if (t[u] >= 0) {
                live.row[at] = static_cast<int>(n);
                live.target[at] = static_cast<int>(t[u]);
                if (p.dloss != nullptr) live.dloss[at] = p.dloss[n * p.dl_s];
                ++at;
            } else {
                live.row[none--] = static_cast<int>(n);
                if (p.loss != nullptr) p.loss[n * p.loss_s] = 0.0f;
                if (p.lse != nullptr) p.lse[n * p.lse_s] = 0.0f;
            }
        }
        first += total;
        dead -= kTile - total;
    }
    if (me == 0 && threadIdx.x == 0) {
        live.count[0] = all;
        live.count[1] = live.count[2] = live.count[3] = 0;
    }
    cluster.sync();  // nobody leaves while its count is read
}

// ------------------------------------------------------------ shared pieces --

// A row's target, or -1 for a row without a loss; reports one outside the vocabulary.
__device__ __forceinline__ int row_target(const LinearCe &p, int64_t n, unsigned long long *err, bool report) {
    const int64_t t = p.targets[n * p.t_s];
    if (t == p.ignore) return -1;
    if (t < 0 || t >= p.V) {
        if (report) report_index(err, t);
        return -1;
    }
    return static_cast<int>(t);
}

// Running maximum and sum of exponentials relative to it.  Infinite maxima count from 0,
// so that a row of +inf or -inf has its limit and not exp(inf - inf).
struct Softmax {
    float top, sum;
};

__device__ __forceinline__ float softmax_base(float top) { return isinf(top) ? 0.0f : top; }

__device__ __forceinline__ Softmax merge(Softmax a, Softmax b) {
    Softmax r;
    r.top = fmaxf(a.top, b.top);
    const float base = softmax_base(r.top);
    r.sum = (a.sum != 0.0f ? a.sum * expf(softmax_base(a.top) - base) : 0.0f) +
            (b.sum != 0.0f ? b.sum * expf(softmax_base(b.top) - base) : 0.0f);
    return r;
}

__device__ __forceinline__ Softmax merge_lanes(Softmax s, int from, int to) {
    for (int o = from; o < to; o <<= 1) {
        Softmax other;
        other.top = __shfl_xor_sync(0xFFFFFFFFu, s.top, o);
        other.sum = __shfl_xor_sync(0xFFFFFFFFu, s.sum, o);
        s = merge(s, other);
    }
    return s;
}

__device__ __forceinline__ float softmax_grad(float z, float lse, float d, bool hot) {
    const float x = z - lse;
    return d * (hot ? expm1f(x) : expf(x));
}

// ----------------------------------------------------------------- few rows --
// Up to 16 rows: bound by reading W, once for the loss (131 MB of a 32000 x 1024 layer at
// ## us) and once more, next to the writing of dW, for the gradients.  Float32 products on
// the FMA units: at 16 rows 16 FMAs for 4 bytes of W, still less than its reading takes.
//
// k_few_logits: a warp takes four rows of W at a time, 128 columns a step, against all rows
// of x in shared memory; one lane for each of its 4 N logits keeps their softmax.
// k_few_grad: a CTA takes 128 (64) columns and a part of the vocabulary; x's columns and the
// sums of dx stay in registers, g comes from the logits by one exponential a class and lane.

constexpr int kFewRows = 16;
constexpr int kFewThreads = 256;
constexpr int kFewShared = 160 * 1024;

struct FewArgs {
    int vec;             // float4 loads of W
    int d_pad;           // x's row in shared memory, a multiple of 128
    float *z;            // [N][V], null: not wanted
    Softmax *parts;      // [CTAs][R]
    int n_parts;
    float *z_target;     // [R]
    float *dx_parts;     // [splits][N][D]
    int splits;
    int dw_vec;
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

// One step of a warp: 128 S columns of four rows of W.  Without VEC a lane's four columns
// are 32 apart, so that a load is contiguous where W is.
template <int S, bool VEC>
__device__ __forceinline__ void load_step(const LinearCe &p, int64_t v0, int64_t c0, float4 (&x)[S][4]) {
    const int lane = threadIdx.x % 32;
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float *w = p.w + (v0 + j < p.V ? v0 + j : p.V - 1) * p.w_rs;
            x[s][j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (VEC) {
                const int64_t c = c0 + s * 128 + lane * 4;
                if (c < p.D) x[s][j] = __ldcs(reinterpret_cast<const float4 *>(w + c));
            } else {
                const int64_t c = c0 + s * 128 + lane;
                if (c < p.D) x[s][j].x = __ldcs(w + c * p.w_cs);
                if (c + 32 < p.D) x[s][j].y = __ldcs(w + (c + 32) * p.w_cs);
                if (c + 64 < p.D) x[s][j].z = __ldcs(w + (c + 64) * p.w_cs);
                if (c + 96 < p.D) x[s][j].w = __ldcs(w + (c + 96) * p.w_cs);
            }
        }
}

// CTAs an SM holds, by registers: with one or two rows the loads in flight decide, and those
// come from warps.
constexpr int few_resident(int R) { return R <= 2 ? 4 : R <= 4 ? 3 : 2; }

template <int R, bool VEC>
__global__ void __launch_bounds__(kFewThreads, few_resident(R)) k_few_logits(const LinearCe p, const FewArgs a) {
    extern __shared__ __align__(16) float xs[];  // [R][d_pad]
    __shared__ int target[R];
    __shared__ Softmax warps[kFewThreads / 32][R];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    constexpr int S = 1;
    const int64_t step = static_cast<int64_t>(gridDim.x) * (kFewThreads / 32) * 4;
    int64_t v0 = (static_cast<int64_t>(blockIdx.x) * (kFewThreads / 32) + warp) * 4, c0 = 0;
    float4 w[S][4], next[S][4];
    if (v0 < p.V) load_step<S, VEC>(p, v0, c0, w);  // under way while x arrives
    if (threadIdx.x < R) target[threadIdx.x] = threadIdx.x < p.N ? row_target(p, threadIdx.x, a.err, blockIdx.x == 0) : -1;
    for (int n = 0; n < R; ++n)
        for (int d = threadIdx.x; d < a.d_pad; d += kFewThreads)
            xs[n * a.d_pad + d] = n < p.N && d < p.D ? p.x[n * p.x_rs + d * p.x_cs] : 0.0f;
    __syncthreads();
    for (int n = 0; n < R; ++n)
        if (target[n] < 0)
            for (int d = threadIdx.x; d < a.d_pad; d += kFewThreads) xs[n * a.d_pad + d] = 0.0f;
    __syncthreads();
    constexpr int kMine = (4 * R + 31) / 32;  // logits of a lane: i = lane + 32 k is row i / 4 and class i % 4
    Softmax mine[kMine];
#pragma unroll
    for (int k = 0; k < kMine; ++k) mine[k] = Softmax{-INFINITY, 0.0f};
    float acc[4 * R];
#pragma unroll
    for (int i = 0; i < 4 * R; ++i) acc[i] = 0.0f;
    while (v0 < p.V) {
        int64_t v1 = v0, c1 = c0 + 128 * S;
        if (c1 >= p.D) {
            c1 = 0;
            v1 += step;
        }
        if (v1 < p.V) load_step<S, VEC>(p, v1, c1, next);
#pragma unroll
        for (int s = 0; s < S; ++s) {
            if (c0 + s * 128 >= p.D) break;
#pragma unroll
            for (int n = 0; n < R; ++n) {
                const float *row = xs + n * a.d_pad + c0 + s * 128;
                float4 y;
                if (VEC) y = *reinterpret_cast<const float4 *>(row + lane * 4);
                else y = make_float4(row[lane], row[lane + 32], row[lane + 64], row[lane + 96]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float &c = acc[4 * n + j];
                    c = fmaf(w[s][j].x, y.x, c);
                    c = fmaf(w[s][j].y, y.y, c);
                    c = fmaf(w[s][j].z, y.z, c);
                    c = fmaf(w[s][j].w, y.w, c);
                }
            }
        }
        if (v1 != v0) {
#pragma unroll
            for (int k = 0; k < kMine; ++k) {
                float x = warp_sums<(4 * R < 32 ? 4 * R : 32)>(acc + 32 * k);
                const int i = lane + 32 * k, n = i / 4;
                const int64_t v = v0 + i % 4;
                if (n >= R || n >= p.N || v >= p.V) continue;
                if (p.bias != nullptr) x += __ldg(p.bias + v * p.b_s);
                if (a.z != nullptr) a.z[n * p.V + v] = x;
                if (v == target[n]) a.z_target[n] = x;
                mine[k] = merge(mine[k], Softmax{x, isnan(x) ? x : isinf(x) ? (x > 0.0f ? x : 0.0f) : 1.0f});
            }
#pragma unroll
            for (int i = 0; i < 4 * R; ++i) acc[i] = 0.0f;
        }
        v0 = v1;
        c0 = c1;
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int j = 0; j < 4; ++j) w[s][j] = next[s][j];
    }
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

// lse of row n from the CTAs' parts; every lane of the warp gets it.
__device__ __forceinline__ float few_lse(const FewArgs &a, int R, int n) {
    Softmax s{-INFINITY, 0.0f};
    const Softmax *parts = a.parts + n;
#pragma unroll 8
    for (int i = threadIdx.x % 32; i < a.n_parts; i += 32) s.top = fmaxf(s.top, parts[i * R].top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s.top = fmaxf(s.top, __shfl_xor_sync(0xFFFFFFFFu, s.top, o));
    const float base = softmax_base(s.top);
#pragma unroll 8
    for (int i = threadIdx.x % 32; i < a.n_parts; i += 32) {
        const Softmax x = parts[i * R];
        if (x.sum != 0.0f) s.sum += x.sum * expf(softmax_base(x.top) - base);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s.sum += __shfl_xor_sync(0xFFFFFFFFu, s.sum, o);
    return softmax_base(s.top) + logf(s.sum);
}

__device__ __forceinline__ void store_loss(const LinearCe &p, const FewArgs &a, int n, int target, float lse) {
    if (p.loss != nullptr) p.loss[n * p.loss_s] = target < 0 ? 0.0f : lse - a.z_target[n];
    if (p.lse != nullptr) p.lse[n * p.lse_s] = target < 0 ? 0.0f : lse;
}

__global__ void __launch_bounds__(32 * kFewRows) k_few_loss(const LinearCe p, const FewArgs a, int R) {
    const int n = threadIdx.x / 32;
    if (n >= p.N) return;
    const float lse = few_lse(a, R, n);
    if (threadIdx.x % 32 == 0) store_loss(p, a, n, row_target(p, n, a.err, false), lse);
}

// C columns a lane, 32 C a CTA.
template <int R, int C>
__global__ void __launch_bounds__(kFewThreads) k_few_grad(const LinearCe p, const FewArgs a) {
    __shared__ float lse[R], dloss[R];
    __shared__ int target[R];
    __shared__ float sums[kFewThreads / 32][32 * C];
    __shared__ __align__(16) float gs[kFewThreads / 32][32][R];  // a warp's 32 classes
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    for (int n = warp; n < R; n += kFewThreads / 32) {
        const int t = n < p.N ? row_target(p, n, a.err, false) : -1;
        const float l = n < p.N ? few_lse(a, R, n) : 0.0f;
        if (lane == 0) {
            lse[n] = l;
            target[n] = t;
            dloss[n] = t >= 0 ? p.dloss[n * p.dl_s] : 0.0f;
            if (n < p.N && blockIdx.x == 0 && blockIdx.y == 0) store_loss(p, a, n, t, l);
        }
    }
    __syncthreads();
    const int64_t c0 = (static_cast<int64_t>(blockIdx.x) * 32 + lane) * C;
    const int cols = static_cast<int>(p.D - c0 < 0 ? 0 : p.D - c0 < C ? p.D - c0 : C);
    float x[R][C], dx[R][C];
#pragma unroll
    for (int n = 0; n < R; ++n)
#pragma unroll
        for (int c = 0; c < C; ++c) {
            dx[n][c] = 0.0f;
            x[n][c] = n < p.N && c < cols && target[n] >= 0 ? p.x[n * p.x_rs + (c0 + c) * p.x_cs] : 0.0f;
        }
    const int64_t step = static_cast<int64_t>(gridDim.y) * (kFewThreads / 32) * 32;
    for (int64_t v0 = (static_cast<int64_t>(blockIdx.y) * (kFewThreads / 32) + warp) * 32; v0 < p.V; v0 += step) {
        const int64_t v = v0 + lane;
        float db = 0.0f;
        __syncwarp();
#pragma unroll
        for (int n = 0; n < R; ++n) {
            float g = 0.0f;
            if (n < p.N && v < p.V && target[n] >= 0) g = softmax_grad(a.z[n * p.V + v], lse[n], dloss[n], v == target[n]);
            gs[warp][lane][n] = g;
            db += g;
        }
        __syncwarp();
        if (p.db != nullptr && blockIdx.x == 0 && v < p.V) p.db[v * p.db_s] = db;
        const int count = static_cast<int>(p.V - v0 < 32 ? p.V - v0 : 32);
        constexpr int U = 8;
        for (int j0 = 0; j0 < count; j0 += U) {
            float w[U][C];
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int c = 0; c < C; ++c) w[u][c] = 0.0f;
                if (p.dx == nullptr || j0 + u >= count) continue;
                const float *src = p.w + (v0 + j0 + u) * p.w_rs + c0 * p.w_cs;
                if (a.vec) {
                    if (cols <= 0) continue;
                    if (C == 4) {
                        const float4 y = __ldcs(reinterpret_cast<const float4 *>(src));
                        w[u][C - 1] = y.w;
                        w[u][2 % C] = y.z;
                        w[u][1] = y.y;
                        w[u][0] = y.x;
                    } else {
                        const float2 y = __ldcs(reinterpret_cast<const float2 *>(src));
                        w[u][0] = y.x;
                        w[u][1] = y.y;
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < C; ++c)
                        if (c < cols) w[u][c] = __ldcs(src + c * p.w_cs);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (j0 + u >= count) break;
                float dw[C];
#pragma unroll
                for (int c = 0; c < C; ++c) dw[c] = 0.0f;
#pragma unroll
                for (int n = 0; n < R; ++n) {
                    const float gn = gs[warp][j0 + u][n];
#pragma unroll
                    for (int c = 0; c < C; ++c) {
                        dx[n][c] = fmaf(gn, w[u][c], dx[n][c]);
                        dw[c] = fmaf(gn, x[n][c], dw[c]);
                    }
                }
                if (p.dw == nullptr) continue;
                float *to = p.dw + (v0 + j0 + u) * p.dw_rs + c0 * p.dw_cs;
                if (a.dw_vec) {
                    if (cols <= 0) continue;
                    if (C == 4) *reinterpret_cast<float4 *>(to) = make_float4(dw[0], dw[1], dw[2 % C], dw[3 % C]);
                    else *reinterpret_cast<float2 *>(to) = make_float2(dw[0], dw[1]);
                } else {
#pragma unroll
                    for (int c = 0; c < C; ++c)
                        if (c < cols) to[c * p.dw_cs] = dw[c];
                }
            }
        }
    }
    if (p.dx == nullptr) return;
#pragma unroll
    for (int n = 0; n < R; ++n) {
        if (n >= p.N) break;
        __syncthreads();
#pragma unroll
        for (int c = 0; c < C; ++c) sums[warp][lane * C + c] = dx[n][c];
        __syncthreads();
        if (static_cast<int>(threadIdx.x) >= 32 * C) continue;
        const int64_t d = static_cast<int64_t>(blockIdx.x) * 32 * C + threadIdx.x;
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < kFewThreads / 32; ++w) s += sums[w][threadIdx.x];
        if (d < p.D) a.dx_parts[(blockIdx.y * p.N + n) * p.D + d] = s;
    }
}

// Eight warps take the parts of 32 elements in turn.
__global__ void __launch_bounds__(256) k_few_dx(const LinearCe p, const FewArgs a) {
    __shared__ float sums[8][32];
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.x % 32;
    const int64_t n = i / p.D;
    float sum = 0.0f;
    if (i < p.N * p.D) {
#pragma unroll 8
        for (int s = threadIdx.x / 32; s < a.splits; s += 8) sum += a.dx_parts[s * p.N * p.D + i];
    }
    sums[threadIdx.x / 32][threadIdx.x % 32] = sum;
    __syncthreads();
    if (threadIdx.x >= 32 || i >= p.N * p.D) return;
    for (int w = 1; w < 8; ++w) sum += sums[w][threadIdx.x];
    if (row_target(p, n, a.err, false) < 0) sum = 0.0f;
    p.dx[n * p.dx_rs + (i - n * p.D) * p.dx_cs] = sum;
}

template <int R>
int few_path(const LinearCe &p, cudaStream_t stream) {
    const int sms = sm_count(current_device());
    const bool grads = p.dloss != nullptr && (p.dx != nullptr || p.dw != nullptr || p.db != nullptr);
    FewArgs a;
    std::memset(&a, 0, sizeof(a));
    a.vec = aligned16(p.w) && p.w_cs == 1 && p.w_rs % 4 == 0 && p.D % 4 == 0;
    a.dw_vec = aligned16(p.dw) && p.dw_cs == 1 && p.dw_rs % 4 == 0 && p.D % 4 == 0;
    a.d_pad = static_cast<int>((p.D + 127) / 128 * 128);
    const size_t shared = static_cast<size_t>(R) * a.d_pad * 4;
    const int64_t wanted = (p.V + 31) / 32;  // CTAs of 8 warps, 4 classes each
    const int64_t most_ctas = static_cast<int64_t>(sms) * (shared > 72 * 1024 ? 1 : shared > 48 * 1024 ? 2 : few_resident(R));
    const int64_t rounds = (wanted + most_ctas - 1) / most_ctas;  // even ones: a CTA loads x once
    a.n_parts = static_cast<int>((wanted + rounds - 1) / rounds);
    constexpr int C = R <= 8 ? 4 : 2;  // columns a lane of k_few_grad: 2 R C values in registers
    const int64_t slabs = p.D > 0 ? (p.D + 32 * C - 1) / (32 * C) : 1;
    const int64_t splits = (static_cast<int64_t>(sms) * 4 + slabs - 1) / slabs;
    const int64_t most = (p.V + 255) / 256;  // 8 warps of 32 classes
    a.splits = static_cast<int>(splits < most ? splits : most);
    const size_t parts = padded(static_cast<size_t>(a.n_parts) * R * sizeof(Softmax));
    const size_t zs = grads ? padded(static_cast<size_t>(p.N) * p.V * 4) : 0;
    const size_t dxs = grads && p.dx != nullptr ? padded(static_cast<size_t>(a.splits) * p.N * p.D * 4) : 0;
    Workspace ws;
    MTC_TRY(ws.allocate(256 + parts + zs + dxs, stream));
    a.z_target = ws.take<float>(256);
    a.parts = ws.take<Softmax>(parts);
    float *z = ws.take<float>(zs);
    a.dx_parts = ws.take<float>(dxs);
    a.z = grads ? z : nullptr;
    MTC_TRY(device_error_word(&a.err));
    if (a.vec) {
        MTC_CUDA_TRY(cudaFuncSetAttribute(k_few_logits<R, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewShared));
        k_few_logits<R, true><<<a.n_parts, kFewThreads, shared, stream>>>(p, a);
    } else {
        MTC_CUDA_TRY(cudaFuncSetAttribute(k_few_logits<R, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewShared));
        k_few_logits<R, false><<<a.n_parts, kFewThreads, shared, stream>>>(p, a);
    }
    MTC_TRY(check_launch("linear cross entropy (few rows)"));
    if (!grads) {
        k_few_loss<<<1, static_cast<unsigned>(32 * p.N), 0, stream>>>(p, a, R);
        return check_launch("linear cross entropy (loss)");
    }
    k_few_grad<R, C><<<dim3(static_cast<unsigned>(slabs), static_cast<unsigned>(a.splits)), kFewThreads, 0, stream>>>(p, a);
    MTC_TRY(check_launch("linear cross entropy (few rows' gradients)"));
    if (p.dx == nullptr || p.D == 0) return MTC_OK;
    k_few_dx<<<static_cast<unsigned>((p.N * p.D + 31) / 32), 256, 0, stream>>>(p, a);
    return check_launch("linear cross entropy (input gradient)");
}

// ------------------------------------------------------------- small problems --
// Up to 256 classes and 2^22 products: bound by latency, so two launches.  k_small_rows: a
// warp a row, its lanes over the classes (and over the columns where the classes are few),
// loss, g and the row of dx.  k_small_weights: a thread an element of dW (or of db), 32 rows
// a CTA; the last CTA of an element's to finish adds the parts in the order of the rows.

constexpr int kSmallClasses = 256;
constexpr int kSmallRows = 32;

struct SmallArgs {
    float *g;               // [N][V], null: no gradients
    float *parts;           // [splits][V D + V]
    unsigned int *arrived;  // [CTAs of one split]
    unsigned int n_arrived;
    int classes_log2;       // lanes over classes
    unsigned long long *err;
};

__global__ void __launch_bounds__(256) k_small_rows(const LinearCe p, const SmallArgs a) {
    if (a.g != nullptr)
        for (unsigned int i = blockIdx.x * 256 + threadIdx.x; i < a.n_arrived; i += gridDim.x * 256) a.arrived[i] = 0;
    const int lane = threadIdx.x % 32;
    const int64_t n = static_cast<int64_t>(blockIdx.x) * 8 + threadIdx.x / 32;
    if (n >= p.N) return;
    const int t = row_target(p, n, a.err, lane == 0);
    if (t < 0) {
        if (lane == 0) {
            if (p.loss != nullptr) p.loss[n * p.loss_s] = 0.0f;
            if (p.lse != nullptr) p.lse[n * p.lse_s] = 0.0f;
        }
        if (a.g == nullptr) return;
        for (int64_t v = lane; v < p.V; v += 32) a.g[n * p.V + v] = 0.0f;
        if (p.dx != nullptr)
            for (int64_t d = lane; d < p.D; d += 32) p.dx[n * p.dx_rs + d * p.dx_cs] = 0.0f;
        return;
    }
    const int C = 1 << a.classes_log2, L = 32 / C;  // L lanes share a class
    const int sub = lane % L;
    const float *x = p.x + n * p.x_rs;
    constexpr int kMost = kSmallClasses / 32;
    float z[kMost];
    Softmax s{-INFINITY, 0.0f};
    float zt = 0.0f;
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
        z[i] = 0.0f;
        if (i * C >= p.V) continue;
        const int v = i * C + lane / L;
        const float *w = p.w + (v < p.V ? v : 0) * p.w_rs;
        float sum = 0.0f;
        int64_t d = sub;
        for (; d + 15 * L < p.D; d += 16 * L) {
            float xv[16], wv[16];
#pragma unroll
            for (int u = 0; u < 16; ++u) {
                xv[u] = __ldg(x + (d + u * L) * p.x_cs);
                wv[u] = __ldg(w + (d + u * L) * p.w_cs);
            }
#pragma unroll
            for (int u = 0; u < 16; ++u) sum = fmaf(xv[u], wv[u], sum);
        }
        for (; d < p.D; d += L) sum = fmaf(__ldg(x + d * p.x_cs), __ldg(w + d * p.w_cs), sum);
        for (int o = 1; o < L; o <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        if (v >= p.V) {
            z[i] = -INFINITY;
            continue;
        }
        if (p.bias != nullptr) sum += __ldg(p.bias + v * p.b_s);
        z[i] = sum;
        if (v == t) zt = sum;
        if (sub == 0) s = merge(s, Softmax{sum, isnan(sum) ? sum : isinf(sum) ? (sum > 0.0f ? sum : 0.0f) : 1.0f});
    }
    s = merge_lanes(s, 1, 32);
    const float lse = softmax_base(s.top) + logf(s.sum);
    zt = __shfl_sync(0xFFFFFFFFu, zt, t % C * L);
    if (lane == 0) {
        if (p.loss != nullptr) p.loss[n * p.loss_s] = lse - zt;
        if (p.lse != nullptr) p.lse[n * p.lse_s] = lse;
    }
    if (a.g == nullptr) return;
    const float dl = p.dloss[n * p.dl_s];
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
        const int v = i * C + lane / L;
        if (i * C >= p.V || v >= p.V) {
            z[i] = 0.0f;
            continue;
        }
        z[i] = softmax_grad(z[i], lse, dl, v == t);
        if (sub == 0) a.g[n * p.V + v] = z[i];
    }
    if (p.dx == nullptr) return;
    for (int64_t d0 = 0; d0 < p.D; d0 += 128) {
        float dx[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < kMost; ++i) {
            if (i * C >= p.V) break;
            const int classes = static_cast<int>(p.V - i * C < C ? p.V - i * C : C);
#pragma unroll 4
            for (int c = 0; c < classes; ++c) {
                const float g = __shfl_sync(0xFFFFFFFFu, z[i], c * L);
                const float *w = p.w + static_cast<int64_t>(i * C + c) * p.w_rs;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int64_t d = d0 + u * 32 + lane;
                    if (d < p.D) dx[u] = fmaf(g, __ldg(w + d * p.w_cs), dx[u]);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t d = d0 + u * 32 + lane;
            if (d < p.D) p.dx[n * p.dx_rs + d * p.dx_cs] = dx[u];
        }
    }
}

__global__ void __launch_bounds__(256) k_small_weights(const LinearCe p, const SmallArgs a) {
    const int64_t weights = p.V * p.D, total = weights + p.V;
    const int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int64_t v = e < weights ? e / p.D : e - weights, d = e - v * p.D;
    float sum = 0.0f;
    if (e < total) {
        const int64_t r0 = static_cast<int64_t>(blockIdx.y) * kSmallRows;
        const int rows = static_cast<int>(p.N - r0 < kSmallRows ? p.N - r0 : kSmallRows);
        const float *g = a.g + r0 * p.V + v, *x = p.x + r0 * p.x_rs + d * p.x_cs;
        for (int j0 = 0; j0 < rows; j0 += 16) {
            float gv[16], xv[16];
#pragma unroll
            for (int u = 0; u < 16; ++u) {
                gv[u] = j0 + u < rows ? g[(j0 + u) * p.V] : 0.0f;
                xv[u] = e >= weights || j0 + u >= rows ? 1.0f : __ldg(x + (j0 + u) * p.x_rs);
            }
#pragma unroll
            for (int u = 0; u < 16; ++u)
                if (gv[u] != 0.0f) sum = fmaf(gv[u], xv[u], sum);  // a row without a loss may hold anything
        }
    }
    if (gridDim.y > 1) {
        __shared__ bool last;
        if (e < total) a.parts[blockIdx.y * total + e] = sum;
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) last = atomicAdd(&a.arrived[blockIdx.x], 1u) == gridDim.y - 1;
        __syncthreads();
        if (!last) return;
        __threadfence();
        if (e >= total) return;
        sum = 0.0f;
#pragma unroll 8
        for (unsigned int s = 0; s < gridDim.y; ++s) sum += __ldcg(a.parts + s * total + e);
    }
    if (e < weights) {
        if (p.dw != nullptr) p.dw[v * p.dw_rs + d * p.dw_cs] = sum;
    } else if (e < total && p.db != nullptr) {
        p.db[v * p.db_s] = sum;
    }
}

int small_path(const LinearCe &p, cudaStream_t stream) {
    const bool grads = p.dloss != nullptr && (p.dx != nullptr || p.dw != nullptr || p.db != nullptr);
    SmallArgs a;
    std::memset(&a, 0, sizeof(a));
    while (a.classes_log2 < 5 && (1 << a.classes_log2) < p.V) ++a.classes_log2;
    const int64_t total = p.V * p.D + p.V;
    const int64_t splits = (p.N + kSmallRows - 1) / kSmallRows;
    a.n_arrived = static_cast<unsigned int>((total + 255) / 256);
    MTC_TRY(device_error_word(&a.err));
    Workspace ws;
    if (grads) {
        const size_t gs = padded(static_cast<size_t>(p.N) * p.V * 4);
        const size_t parts = splits > 1 ? padded(static_cast<size_t>(splits) * total * 4) : 0;
        const size_t arrived = padded(static_cast<size_t>(a.n_arrived) * 4);
        MTC_TRY(ws.allocate(gs + parts + arrived, stream));
        a.g = ws.take<float>(gs);
        a.parts = ws.take<float>(parts);
        a.arrived = ws.take<unsigned int>(arrived);
    }
    k_small_rows<<<static_cast<unsigned>((p.N + 7) / 8), 256, 0, stream>>>(p, a);
    MTC_TRY(check_launch("linear cross entropy (small)"));
    if (!grads || (p.dw == nullptr && p.db == nullptr)) return MTC_OK;
    k_small_weights<<<dim3(a.n_arrived, static_cast<unsigned>(splits)), 256, 0, stream>>>(p, a);
    return check_launch("linear cross entropy (small, weight gradient)");
}

// ------------------------------------------------------------------- host --

int need_vector(const mtc_desc *d, const char *name, int64_t extent, bool written, float *&p, int64_t &stride) {
    p = nullptr;
    stride = 0;
    if (d == nullptr) return MTC_OK;
    MTC_TRY(need_float(d, name));
    if (d->rank != 1 || d->shape[0] != extent)
        return fail(MTC_ERR_INVALID_ARGUMENT, "%s: shape [%lld] expected", name, static_cast<long long>(extent));
    if (written) MTC_TRY(need_distinct(d, name));
    p = float_at(d);
    stride = d->strides[0];
    return MTC_OK;
}

int need_matrix(const mtc_desc *d, const char *name, int64_t rows, int64_t cols, bool written, float *&p, int64_t &rs,
                int64_t &cs) {
    p = nullptr;
    rs = cs = 0;
    if (d == nullptr) return MTC_OK;
    MTC_TRY(need_float(d, name));
    if (d->rank != 2 || d->shape[0] != rows || d->shape[1] != cols)
        return fail(MTC_ERR_INVALID_ARGUMENT, "%s: shape [%lld, %lld] expected", name, static_cast<long long>(rows),
                    static_cast<long long>(cols));
    if (written) MTC_TRY(need_distinct(d, name));
    p = float_at(d);
    rs = d->strides[0];
    cs = d->strides[1];
    return MTC_OK;
}

int zero_view(const mtc_desc *d, cudaStream_t stream) {
    if (d == nullptr) return MTC_OK;
    const float zero = 0.0f;
    return mtc_fill(d, &zero, stream);
}

int run_linear_ce(const mtc_desc *x, const mtc_desc *weight, const mtc_desc *bias, const mtc_desc *targets,
                  int64_t ignore, const mtc_desc *dloss, const mtc_desc *loss, const mtc_desc *lse, const mtc_desc *dx,
                  const mtc_desc *dw, const mtc_desc *db, bool grads, cudaStream_t stream) {
    LinearCe p;
    std::memset(&p, 0, sizeof(p));
    MTC_TRY(need_float(x, "x"));
    MTC_TRY(need_float(weight, "weight"));
    MTC_TRY(need_int(targets, "targets"));
    if (x->rank != 2 || weight->rank != 2) return fail(MTC_ERR_INVALID_ARGUMENT, "x and weight must be matrices");
    if (x->shape[1] != weight->shape[1])
        return fail(MTC_ERR_INVALID_ARGUMENT, "x has %lld columns, weight %lld", static_cast<long long>(x->shape[1]),
                    static_cast<long long>(weight->shape[1]));
    p.N = x->shape[0];
    p.V = weight->shape[0];
    p.D = x->shape[1];
    if (targets->rank != 1 || targets->shape[0] != p.N)
        return fail(MTC_ERR_INVALID_ARGUMENT, "targets: shape [%lld] expected", static_cast<long long>(p.N));
    if (p.N > INT32_MAX || p.V > INT32_MAX || p.D > INT32_MAX)
        return fail(MTC_ERR_UNSUPPORTED, "linear cross entropy: an extent exceeds 2^31 - 1");
    p.x = float_at(x);
    p.x_rs = x->strides[0];
    p.x_cs = x->strides[1];
    p.w = float_at(weight);
    p.w_rs = weight->strides[0];
    p.w_cs = weight->strides[1];
    p.targets = static_cast<const int64_t *>(targets->data) + targets->offset;
    p.t_s = targets->strides[0];
    p.ignore = ignore;
    float *b = nullptr, *dl = nullptr;
    MTC_TRY(need_vector(bias, "bias", p.V, false, b, p.b_s));
    MTC_TRY(need_vector(loss, "loss", p.N, true, p.loss, p.loss_s));
    MTC_TRY(need_vector(lse, "lse", p.N, true, p.lse, p.lse_s));
    if (grads) {
        if (dloss == nullptr) return fail(MTC_ERR_INVALID_ARGUMENT, "dloss: null descriptor");
        MTC_TRY(need_vector(dloss, "dloss", p.N, false, dl, p.dl_s));
        MTC_TRY(need_matrix(dx, "dx", p.N, p.D, true, p.dx, p.dx_rs, p.dx_cs));
        MTC_TRY(need_matrix(dw, "dweight", p.V, p.D, true, p.dw, p.dw_rs, p.dw_cs));
        MTC_TRY(need_vector(db, "dbias", p.V, true, p.db, p.db_s));
    } else if (loss == nullptr) {
        return fail(MTC_ERR_INVALID_ARGUMENT, "loss: null descriptor");
    }
    p.bias = b;
    p.dloss = dl;
    if (p.N > 0 && p.V == 0) return fail(MTC_ERR_INVALID_ARGUMENT, "cross entropy over no classes");
    if (p.N == 0) {  // sums over no rows
        MTC_TRY(zero_view(dw, stream));
        return zero_view(db, stream);
    }
    if (p.V <= kSmallClasses && p.N < (int64_t{1} << 21) && p.N * p.V < (int64_t{1} << 22) / (p.D + 1))
        return small_path(p, stream);
    if (p.N <= kFewRows) {
        const int64_t row = (p.D + 127) / 128 * 512;
        if (p.N == 1 && row <= kFewShared) return few_path<1>(p, stream);
        if (p.N <= 2 && 2 * row <= kFewShared) return few_path<2>(p, stream);
        if (p.N <= 4 && 4 * row <= kFewShared) return few_path<4>(p, stream);
        if (p.N <= 8 && 8 * row <= kFewShared) return few_path<8>(p, stream);
        if (16 * row <= kFewShared) return few_path<16>(p, stream);
    }
    return linear_ce_tensor(p, stream);
}

}  // namespace

int list_live_rows(const LinearCe &p, const LiveRows &live, cudaStream_t stream) {
    unsigned long long *err = nullptr;
    MTC_TRY(device_error_word(&err));
    const int64_t tiles = (p.N + kListThreads * kListRows - 1) / (kListThreads * kListRows);
    unsigned int ctas = 1;
    while (ctas < kListCtas && ctas < tiles) ctas *= 2;
    MTC_CUDA_TRY(cudaFuncSetAttribute(k_live_rows, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchConfig_t config;
    std::memset(&config, 0, sizeof(config));
    config.gridDim = dim3(ctas);
    config.blockDim = dim3(kListThreads);
    config.stream = stream;
    cudaLaunchAttribute attr;
    std::memset(&attr, 0, sizeof(attr));
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = ctas;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    config.attrs = &attr;
    config.numAttrs = 1;
    MTC_CUDA_TRY(cudaLaunchKernelEx(&config, k_live_rows, p, live, err));
    return check_launch("linear cross entropy (rows)");
}

}  // namespace mtc

using namespace mtc;

extern "C" {

int mtc_linear_cross_entropy(const mtc_desc *x, const mtc_desc *weight, const mtc_desc *bias, const mtc_desc *targets,
                             int64_t ignore_target, const mtc_desc *loss, const mtc_desc *lse, void *stream) {
    clear_error();
    return run_linear_ce(x, weight, bias, targets, ignore_target, nullptr, loss, lse, nullptr, nullptr, nullptr, false,
                         static_cast<cudaStream_t>(stream));
}

int mtc_linear_cross_entropy_grad(const mtc_desc *x, const mtc_desc *weight, const mtc_desc *bias,
                                  const mtc_desc *targets, int64_t ignore_target, const mtc_desc *dloss,
                                  const mtc_desc *loss, const mtc_desc *lse, const mtc_desc *dx,
                                  const mtc_desc *dweight, const mtc_desc *dbias, void *stream) {
    clear_error();
    return run_linear_ce(x, weight, bias, targets, ignore_target, dloss, loss, lse, dx, dweight, dbias, true,
                         static_cast<cudaStream_t>(stream));
}

}  // extern "C"
