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
struct LiveRows {
    int *count;      // [1], and behind it the largest finite |x|, |weight| and |dloss| as bits [3], zeroed with it
    int *row;        // [N] the row of x; behind them, from the end backwards, the rows without a loss
    int *target;     // [N]
    float *dloss;    // [N]
};

// Lists the rows with a loss; writes the zero loss and lse of the others.
int list_live_rows(const LinearCe &p, const LiveRows &live, cudaStream_t stream);

// Tensor-core path (any sizes).
int linear_ce_tensor(const LinearCe &p, cudaStream_t stream);

#ifdef __CUDACC__
// How many of `extent` rows from `first` on have a loss.
__device__ __forceinline__ int64_t live_extent(const int *live, int64_t first, int64_t extent) {
    const int64_t left = *live - first;
    return left < 0 ? 0 : left < extent ? left : extent;
}
#endif

}  // namespace mtc
