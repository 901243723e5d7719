// Softmax cross entropy of a linear layer over a large vocabulary, and its gradient.
//
//   z = x W^T + b            lse_n = log sum_v exp z_nv          loss_n = lse_n - z_{n,t_n}
//   g_nv = dloss_n (exp(z_nv - lse_n) - [v = t_n])
//   dx = g W                 dW = g^T x                          db_v = sum_n g_nv
//
// Rows without a loss are left out before any product: one CTA lists the others
// in order (k_live_rows), and everything below runs over that list, whose length
// only the device knows.
#include <cfloat>
#include <climits>
#include <cstring>

#include "linear_ce.cuh"

namespace mtc {
namespace {

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
    int before = 0;
    total = 0;
    for (int w = 0; w < static_cast<int>(blockDim.x / 32); ++w) {
        if (w < warp) before += warp_sums[w];
        total += warp_sums[w];
    }
    return before + x - v;
}

// The rows with a loss, in order; zero loss, lse and dx count for the others.
__global__ void __launch_bounds__(1024) k_live_rows(const LinearCe p, const LiveRows live, unsigned long long *err) {
    __shared__ int warp_sums[32];
    constexpr int U = 4;
    int first = 0;
    for (int64_t n0 = 0; n0 < p.N; n0 += 1024 * U) {
        int64_t t[U];
        bool has[U];
        int mine = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t n = n0 + static_cast<int64_t>(threadIdx.x) * U + u;
            has[u] = false;
            t[u] = 0;
            if (n >= p.N) continue;
            t[u] = p.targets[n * p.t_s];
            has[u] = t[u] != p.ignore;
            if (has[u] && (t[u] < 0 || t[u] >= p.V)) {
                report_index(err, t[u]);
                has[u] = false;
            }
            mine += has[u];
            if (!has[u]) {
                if (p.loss != nullptr) p.loss[n * p.loss_s] = 0.0f;
                if (p.lse != nullptr) p.lse[n * p.lse_s] = 0.0f;
            }
        }
        int total;
        int at = first + block_exclusive(mine, warp_sums, total);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!has[u]) continue;
            const int64_t n = n0 + static_cast<int64_t>(threadIdx.x) * U + u;
            live.row[at] = static_cast<int>(n);
            live.target[at] = static_cast<int>(t[u]);
            if (p.dloss != nullptr) live.dloss[at] = p.dloss[n * p.dl_s];
            ++at;
        }
        first += total;
    }
    if (threadIdx.x == 0) {
        live.count[0] = first;
        live.count[1] = live.count[2] = live.count[3] = 0;
    }
}

// dx rows without a loss.
__global__ void __launch_bounds__(256) k_zero_dx(const LinearCe p) {
    for (int64_t n = blockIdx.x; n < p.N; n += gridDim.x) {
        const int64_t t = p.targets[n * p.t_s];
        if (t != p.ignore && t >= 0 && t < p.V) continue;
        for (int64_t d = threadIdx.x; d < p.D; d += 256) p.dx[n * p.dx_rs + d * p.dx_cs] = 0.0f;
    }
}

// ------------------------------------------------------------- small problems --
// Float32 products on the FMA units, 64 x 64 tiles of the result.

struct Mat {
    const float *p;
    int64_t rs, cs;
    const int *map;  // rows of the operand by way of this list; null: as they are
};

struct SimtArgs {
    Mat a, b;  // C[m, n] = sum_k a(m, k) b(k, n)
    float *c;
    int64_t c_rs, c_cs;
    const int *c_map;
    const float *bias;  // added to column n
    int64_t bias_s;
    int64_t M, N, K;
    const int *live;  // rows with a loss: bounds M (live_dim 0) or K (live_dim 1), first..first + extent
    int live_dim;
    int64_t first;
    int64_t k_split;  // K of one blockIdx.z; partial results [z][M][N] in c with several
};

__global__ void __launch_bounds__(256) k_simt_product(const SimtArgs g) {
    constexpr int T = 64, KT = 16;
    __shared__ float as[KT][T + 1], bs[KT][T + 1];
    int64_t M = g.M, K = g.K;
    if (g.live_dim == 0) M = live_extent(g.live, g.first, M);
    else K = live_extent(g.live, g.first, K);
    const int64_t m0 = static_cast<int64_t>(blockIdx.x) * T, n0 = static_cast<int64_t>(blockIdx.y) * T;
    if (m0 >= M) return;
    const int64_t k_begin = static_cast<int64_t>(blockIdx.z) * g.k_split;
    const int64_t k_end = k_begin + g.k_split < K ? k_begin + g.k_split : K;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const bool a_by_k = g.a.cs == 1, b_by_k = g.b.rs == 1;
    float acc[4][4] = {};
    for (int64_t k0 = k_begin; k0 < k_end; k0 += KT) {
#pragma unroll
        for (int j = 0; j < T * KT / 256; ++j) {
            const int e = j * 256 + threadIdx.x;
            const int am = a_by_k ? e / KT : e % T, ak = a_by_k ? e % KT : e / T;
            float v = 0.0f;
            if (m0 + am < M && k0 + ak < k_end) {
                const int64_t m = g.a.map != nullptr ? g.a.map[g.first + m0 + am] : m0 + am;
                v = g.a.p[m * g.a.rs + (k0 + ak) * g.a.cs];
            }
            as[ak][am] = v;
            const int bn = b_by_k ? e / KT : e % T, bk = b_by_k ? e % KT : e / T;
            v = 0.0f;
            if (n0 + bn < g.N && k0 + bk < k_end) {
                const int64_t k = g.b.map != nullptr ? g.b.map[g.first + k0 + bk] : k0 + bk;
                v = g.b.p[k * g.b.rs + (n0 + bn) * g.b.cs];
            }
            bs[bk][bn] = v;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < KT; ++k) {
            float a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = as[k][ty + 16 * i];
                b[i] = bs[k][tx + 16 * i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
        }
        __syncthreads();
    }
    float *c = g.c;
    if (gridDim.z > 1) c += static_cast<int64_t>(blockIdx.z) * g.M * g.N;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t m = m0 + ty + 16 * i;
        if (m >= M) continue;
        const int64_t row = g.c_map != nullptr ? g.c_map[g.first + m] : m;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t n = n0 + tx + 16 * j;
            if (n >= g.N) continue;
            float v = acc[i][j];
            if (g.bias != nullptr) v += g.bias[n * g.bias_s];
            if (gridDim.z > 1) c[m * g.N + n] = v;
            else c[row * g.c_rs + n * g.c_cs] = v;
        }
    }
}

// Sums the K splits in order into C, adding to it where `add`.
__global__ void __launch_bounds__(256) k_simt_join(const float *parts, int splits, int64_t M, int64_t N, float *c,
                                                   int64_t c_rs, int64_t c_cs, int add) {
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < M * N;
         i += static_cast<int64_t>(gridDim.x) * 256) {
        float sum = 0.0f;
        for (int s = 0; s < splits; ++s) sum += parts[s * M * N + i];
        float *to = c + (i / N) * c_rs + (i % N) * c_cs;
        *to = add ? *to + sum : sum;
    }
}

__device__ __forceinline__ float block_reduce(float v, bool take_max) {
    __shared__ float part[32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float y = __shfl_xor_sync(0xFFFFFFFFu, v, o);
        v = take_max ? fmaxf(v, y) : v + y;
    }
    __syncthreads();
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = v;
    __syncthreads();
    const int warps = blockDim.x / 32;
    v = static_cast<int>(threadIdx.x % 32) < warps ? part[threadIdx.x % 32] : take_max ? -INFINITY : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float y = __shfl_xor_sync(0xFFFFFFFFu, v, o);
        v = take_max ? fmaxf(v, y) : v + y;
    }
    return v;
}

// One CTA a row of logits: lse and loss, then g in the place of z.
__global__ void __launch_bounds__(256) k_softmax_rows(const LinearCe p, const LiveRows live, int64_t first, int64_t rows,
                                                      float *z) {
    const int64_t r = blockIdx.x;
    if (r >= live_extent(live.count, first, rows)) return;
    float *zr = z + r * p.V;
    float top = -INFINITY;
    bool nan = false;
    for (int64_t v = threadIdx.x; v < p.V; v += 256) {
        const float x = zr[v];
        top = fmaxf(top, x);
        nan |= isnan(x);
    }
    nan = __syncthreads_or(nan);
    top = block_reduce(top, true);
    if (nan) top = NAN;
    float sum = 0.0f;
    const float base = isinf(top) ? 0.0f : top;  // exp(inf - inf) would make a NaN of a row that has a limit
    for (int64_t v = threadIdx.x; v < p.V; v += 256) sum += expf(zr[v] - base);
    sum = block_reduce(sum, false);
    const float lse = base + logf(sum);
    const int t = live.target[first + r];
    const int64_t n = live.row[first + r];
    if (threadIdx.x == 0) {
        if (p.lse != nullptr) p.lse[n * p.lse_s] = lse;
        if (p.loss != nullptr) p.loss[n * p.loss_s] = lse - zr[t];
    }
    if (p.dloss == nullptr) return;
    __syncthreads();
    const float d = live.dloss[first + r];
    for (int64_t v = threadIdx.x; v < p.V; v += 256) {
        const float x = zr[v] - lse;
        zr[v] = d * (v == t ? expm1f(x) : expf(x));
    }
}

constexpr int64_t kSplitRows = 256;

int simt_product(SimtArgs &g, cudaStream_t stream, int splits) {
    const dim3 grid(static_cast<unsigned>((g.M + 63) / 64), static_cast<unsigned>((g.N + 63) / 64),
                    static_cast<unsigned>(splits));
    if ((g.N + 63) / 64 > 65535 || splits > 65535) return fail(MTC_ERR_UNSUPPORTED, "linear cross entropy: too many columns");
    k_simt_product<<<grid, 256, 0, stream>>>(g);
    return check_launch("linear cross entropy (product)");
}

// Column sums of g over the chunk's rows: a product with a row of ones.
__global__ void __launch_bounds__(256) k_column_sums(const float *g, int64_t V, const int *live, int64_t first,
                                                     int64_t rows, float *db, int64_t db_s, int add) {
    const int64_t v = static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.x % 32;
    const int64_t n = live_extent(live, first, rows);
    __shared__ float part[8][32];
    float sum = 0.0f;
    if (v < V)
        for (int64_t r = threadIdx.x / 32; r < n; r += 8) sum += g[r * V + v];
    part[threadIdx.x / 32][threadIdx.x % 32] = sum;
    __syncthreads();
    if (threadIdx.x >= 32 || v >= V) return;
    sum = 0.0f;
    for (int w = 0; w < 8; ++w) sum += part[w][threadIdx.x];
    db[v * db_s] = add ? db[v * db_s] + sum : sum;
}

int simt_path(const LinearCe &p, cudaStream_t stream) {
    int64_t chunk = (int64_t{1} << 28) / (p.V * 4);
    if (chunk < 64) chunk = 64;
    if (chunk > p.N) chunk = p.N;
    const int splits = static_cast<int>((chunk + kSplitRows - 1) / kSplitRows);
    const size_t list = padded(static_cast<size_t>(p.N) * 4);
    const size_t zs = padded(static_cast<size_t>(chunk) * p.V * 4);
    const size_t parts = p.dw != nullptr && splits > 1 ? padded(static_cast<size_t>(splits) * p.V * p.D * 4) : 0;
    Workspace ws;
    MTC_TRY(ws.allocate(256 + 3 * list + zs + parts, stream));
    LiveRows live;
    live.count = ws.take<int>(256);
    live.row = ws.take<int>(list);
    live.target = ws.take<int>(list);
    live.dloss = ws.take<float>(list);
    float *z = ws.take<float>(zs);
    float *part = ws.take<float>(parts);
    MTC_TRY(list_live_rows(p, live, stream));
    for (int64_t first = 0; first < p.N; first += chunk) {
        const int64_t rows = p.N - first < chunk ? p.N - first : chunk;
        SimtArgs g;
        std::memset(&g, 0, sizeof(g));
        g.a = Mat{p.x, p.x_rs, p.x_cs, live.row};
        g.b = Mat{p.w, p.w_cs, p.w_rs, nullptr};
        g.c = z;
        g.c_rs = p.V;
        g.c_cs = 1;
        g.bias = p.bias;
        g.bias_s = p.b_s;
        g.M = rows;
        g.N = p.V;
        g.K = g.k_split = p.D;
        g.live = live.count;
        g.first = first;
        MTC_TRY(simt_product(g, stream, 1));
        k_softmax_rows<<<static_cast<unsigned>(rows), 256, 0, stream>>>(p, live, first, rows, z);
        MTC_TRY(check_launch("linear cross entropy (softmax)"));
        if (p.dx != nullptr && p.D > 0) {
            std::memset(&g, 0, sizeof(g));
            g.a = Mat{z, p.V, 1, nullptr};
            g.b = Mat{p.w, p.w_rs, p.w_cs, nullptr};
            g.c = p.dx;
            g.c_rs = p.dx_rs;
            g.c_cs = p.dx_cs;
            g.c_map = live.row;
            g.M = rows;
            g.N = p.D;
            g.K = g.k_split = p.V;
            g.live = live.count;
            g.first = first;
            MTC_TRY(simt_product(g, stream, 1));
        }
        if (p.dw != nullptr && p.D > 0) {
            std::memset(&g, 0, sizeof(g));
            g.a = Mat{z, 1, p.V, nullptr};
            g.b = Mat{p.x, p.x_rs, p.x_cs, live.row};
            g.c = part;
            g.M = p.V;
            g.N = p.D;
            g.K = rows;
            g.live = live.count;
            g.live_dim = 1;
            g.first = first;
            const int s = static_cast<int>((rows + kSplitRows - 1) / kSplitRows);
            g.k_split = kSplitRows;
            if (s == 1 && first == 0) {
                g.c = p.dw;
                g.c_rs = p.dw_rs;
                g.c_cs = p.dw_cs;
                MTC_TRY(simt_product(g, stream, 1));
            } else {
                g.c_rs = p.D;
                g.c_cs = 1;
                MTC_TRY(simt_product(g, stream, s));
                const int64_t blocks = (p.V * p.D + 255) / 256;
                k_simt_join<<<static_cast<unsigned>(blocks < 4096 ? blocks : 4096), 256, 0, stream>>>(
                    part, s, p.V, p.D, p.dw, p.dw_rs, p.dw_cs, first > 0);
                MTC_TRY(check_launch("linear cross entropy (weight gradient)"));
            }
        }
        if (p.db != nullptr) {
            k_column_sums<<<static_cast<unsigned>((p.V + 31) / 32), 256, 0, stream>>>(z, p.V, live.count, first, rows,
                                                                                     p.db, p.db_s, first > 0);
            MTC_TRY(check_launch("linear cross entropy (bias gradient)"));
        }
    }
    return MTC_OK;
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
    // Small problems stay on the FMA units.
    if (p.N * p.V < (int64_t{1} << 22) / (p.D + 1)) return simt_path(p, stream);
    return linear_ce_tensor(p, stream);
}

}  // namespace

int list_live_rows(const LinearCe &p, const LiveRows &live, cudaStream_t stream) {
    unsigned long long *err = nullptr;
    MTC_TRY(device_error_word(&err));
    k_live_rows<<<1, 1024, 0, stream>>>(p, live, err);
    MTC_TRY(check_launch("linear cross entropy (rows)"));
    if (p.dx == nullptr || p.D == 0) return MTC_OK;
    k_zero_dx<<<static_cast<unsigned>(p.N < 1184 ? p.N : 1184), 256, 0, stream>>>(p);
    return check_launch("linear cross entropy (zero rows)");
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
