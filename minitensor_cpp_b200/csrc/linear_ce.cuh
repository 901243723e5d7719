// The linear cross entropy as its float32 path (linear_ce.cu) and its tensor-core
// path (linear_ce_tc.cu) see it.
#pragma once

#include "operators.cuh"

namespace mtc {

struct LinearCe {
    int64_t N, V, D;
    const float *x;
    int64_t x_rs, x_cs;
    const float *w;
    int64_t w_rs, w_cs;
    const float *bias;  // null: none
    int64_t b_s;
    const int64_t *targets;
    int64_t t_s;
    int64_t ignore;
    const float *dloss;  // null: no gradients
    int64_t dl_s;
    float *loss, *lse;  // null: not wanted
    int64_t loss_s, lse_s;
    float *dx, *dw, *db;  // null: not wanted
    int64_t dx_rs, dx_cs, dw_rs, dw_cs, db_s;
};

// What the device knows about the rows that have a loss.
constexpr int kLiveKnown = 10;
struct LiveRows {
    int *count;      // [1], and behind it what the tensor-core path learns of the magnitudes, zeroed with it
    int *row;        // [N] the row of x; behind them, from the end backwards, the rows without a loss
    int *target;     // [N]
    float *dloss;    // [N]
};

// Lists the rows with a loss; writes the zero loss and lse of the others.
int list_live_rows(const LinearCe &p, const LiveRows &live, cudaStream_t stream);

// Tensor-core path (any sizes).
int linear_ce_tensor(const LinearCe &p, cudaStream_t stream);

// Up to kFewRows rows, or up to as many classes: float32 products that read W, or x, once for
// the loss and once more for the gradients (linear_ce_few.cu).  Whether one of the two holds
// and its rows fit in shared memory.
constexpr int kFewRows = 16;
bool few_rows(const LinearCe &p);
bool few_classes(const LinearCe &p);
int linear_ce_few(const LinearCe &p, bool classes, cudaStream_t stream);

#ifdef __CUDACC__
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

// lse in two parts: base + log rounds to the base's places, (z - base) - log does not.
struct LogSum {
    float base, log;
    __device__ __forceinline__ float lse() const { return base + log; }
    __device__ __forceinline__ float of(float z) const { return (z - base) - log; }  // log of the class's probability
    __device__ __forceinline__ float loss(float z) const { return log - (z - base); }
};

// Running maximum, and the sum of the others' exponentials relative to it: 1 + rest is the sum of
// all.  Of a row that is sure of its class the rest is little, and is the gradient; next to the 1 it
// would lose its digits.  (300 rows, 100 classes, the target's logit 16 above the others: with the
// 1 in float32 sums the target's gradient is off by 6e-3 of itself.)  No logits: -inf and -1.
struct Softmax {
    float top;
    double rest;
    // Infinite maxima count from 0, so that a row of +inf or -inf has its limit and not exp(inf - inf).
    __device__ __forceinline__ LogSum log_sum() const {
        if (isinf(top)) return LogSum{0.0f, isnan(rest) ? static_cast<float>(rest) : top};
        return LogSum{top, static_cast<float>(log1p(rest))};
    }
};

__device__ __forceinline__ Softmax no_logits() { return Softmax{-INFINITY, -1.0}; }

__device__ __forceinline__ Softmax one_logit(float z) {
    return Softmax{isnan(z) ? -INFINITY : z, isnan(z) ? z : z == -INFINITY ? -1.0 : 0.0};
}

__device__ __forceinline__ Softmax merge(Softmax a, Softmax b) {
    if (b.top > a.top) {
        const Softmax c = a;
        a = b;
        b = c;
    }
    // equal infinities: a factor of 1, so that -inf adds 1 - 1 and NaN stays
    a.rest += (1.0 + b.rest) * (a.top == b.top ? 1.0f : expf(b.top - a.top));
    return a;
}

__device__ __forceinline__ Softmax merge_lanes(Softmax s, int from, int to) {
    for (int o = from; o < to; o <<= 1) {
        Softmax other;
        other.top = __shfl_xor_sync(0xFFFFFFFFu, s.top, o);
        other.rest = __shfl_xor_sync(0xFFFFFFFFu, s.rest, o);
        s = merge(s, other);
    }
    return s;
}

__device__ __forceinline__ float softmax_grad(float log_p, float d, bool hot) {
    return d * (hot ? expm1f(log_p) : expf(log_p));
}

// How many of `extent` rows from `first` on have a loss.
__device__ __forceinline__ int64_t live_extent(const int *live, int64_t first, int64_t extent) {
    const int64_t left = *live - first;
    return left < 0 ? 0 : left < extent ? left : extent;
}
#endif

}  // namespace mtc
