// Softmax cross entropy of a linear layer over a large vocabulary, and its gradient.
//
//   z = x W^T + b            lse_n = log sum_v exp z_nv          loss_n = lse_n - z_{n,t_n}
//   g_nv = dloss_n (exp(z_nv - lse_n) - [v = t_n])
//   dx = g W                 dW = g^T x                          db_v = sum_n g_nv
//
// Small problems take a warp a row (here), few rows or few classes stream the other operand
// past them (linear_ce_few.cu), and the rest runs on the tensor cores (linear_ce_tc.cu) over
// the rows that have a loss: k_live_rows lists them in order (8 us for 1031 rows, 13 us for
// 65536), and only the device knows how many there are.
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
        for (int i = 1; i < kLiveKnown; ++i) live.count[i] = 0;
    }
    cluster.sync();  // nobody leaves while its count is read
}

// ------------------------------------------------------------- small problems --
// Up to 256 classes, 4096 products a row and 2^22 in all: bound by latency, so two launches.
// k_small_rows: a warp a row, its lanes over the classes (and over the columns where the classes
// are few), loss, g and the row of dx.  A warp's time goes with the products of a row: 300 rows
// take 21 us for 1280 and 38 for 5120 for the loss and its gradients, where the tensor cores take
// 51 and 57, but 32 rows 111 us for 20480, where they take 59; 8 rows 21 us for 1280 and 33 for
// 5120, where the path of few rows takes 26 and 27, so that those leave at 2048.
// k_small_weights: a thread an element of dW (or of db), 32 rows a CTA; the last CTA of an
// element's to finish adds the parts in the order of the rows.
// 300 rows of 64 columns, 3 classes: 26 us a call with its checks, most of it the host's.

constexpr int kSmallClasses = 256;
constexpr int64_t kSmallRow = 4096, kSmallFewRow = 2048;  // products of a row
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
    // the logits in float64, which a latency-bound kernel has time for: of a few rows, each
    // rounding of one shows in the gradients
    double z[kMost], zt = 0.0, top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
        z[i] = 0.0;
        if (i * C >= p.V) continue;
        const int v = i * C + lane / L;
        const float *w = p.w + (v < p.V ? v : 0) * p.w_rs;
        double sum = 0.0;
        int64_t d = sub;
        for (; d + 15 * L < p.D; d += 16 * L) {
            float xv[16], wv[16];
#pragma unroll
            for (int u = 0; u < 16; ++u) {
                xv[u] = __ldg(x + (d + u * L) * p.x_cs);
                wv[u] = __ldg(w + (d + u * L) * p.w_cs);
            }
#pragma unroll
            for (int u = 0; u < 16; ++u) sum = fma(static_cast<double>(xv[u]), static_cast<double>(wv[u]), sum);
        }
        for (; d < p.D; d += L)
            sum = fma(static_cast<double>(__ldg(x + d * p.x_cs)), static_cast<double>(__ldg(w + d * p.w_cs)), sum);
        for (int o = 1; o < L; o <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        if (v >= p.V) {
            z[i] = -INFINITY;
            continue;
        }
        if (p.bias != nullptr) sum += __ldg(p.bias + v * p.b_s);
        z[i] = sum;
        if (v == t) zt = sum;
        top = fmax(top, sum);
    }
    for (int o = 1; o < 32; o <<= 1) top = fmax(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    const double base = isinf(top) ? 0.0 : top;
    double rest = 0.0;  // the others' exponentials, as in Softmax
    int same = 0;
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
        if (i * C >= p.V || sub != 0) continue;
        if (z[i] == top) ++same;
        else rest += expf(static_cast<float>(z[i] - base));
    }
    for (int o = 1; o < 32; o <<= 1) rest += __shfl_xor_sync(0xFFFFFFFFu, rest, o);
    rest += static_cast<double>(static_cast<int>(__reduce_add_sync(0xFFFFFFFFu, same)) - 1);
    const float beyond = static_cast<float>(!isinf(top) ? log1p(rest) : isnan(rest) ? rest : top);  // lse = base + beyond
    zt = __shfl_sync(0xFFFFFFFFu, zt, t % C * L);
    if (lane == 0) {
        if (p.loss != nullptr) p.loss[n * p.loss_s] = static_cast<float>(base - zt) + beyond;
        if (p.lse != nullptr) p.lse[n * p.lse_s] = static_cast<float>(base + beyond);
    }
    if (a.g == nullptr) return;
    float g[kMost];
    const float dl = p.dloss[n * p.dl_s];
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
        const int v = i * C + lane / L;
        if (i * C >= p.V || v >= p.V) {
            g[i] = 0.0f;
            continue;
        }
        g[i] = softmax_grad(static_cast<float>(z[i] - base) - beyond, dl, v == t);
        if (sub == 0) a.g[n * p.V + v] = g[i];
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
                const float gc = __shfl_sync(0xFFFFFFFFu, g[i], c * L);
                const float *w = p.w + static_cast<int64_t>(i * C + c) * p.w_rs;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int64_t d = d0 + u * 32 + lane;
                    if (d < p.D) dx[u] = fmaf(gc, __ldg(w + d * p.w_cs), dx[u]);
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
    wait_for_previous();
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
    return launch_dependent("linear cross entropy (small, weight gradient)", k_small_weights, dim3(a.n_arrived, static_cast<unsigned>(splits)), 256, 0, stream, p, a);
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
    const bool few = few_rows(p) || few_classes(p);
    if (p.V <= kSmallClasses && p.V * p.D <= (few ? kSmallFewRow : kSmallRow) && p.N < (int64_t{1} << 20) &&
        p.N * p.V < (int64_t{1} << 22) / (p.D + 1))
        return small_path(p, stream);
    if (few_rows(p)) return linear_ce_few(p, false, stream);
    if (few_classes(p)) return linear_ce_few(p, true, stream);
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
