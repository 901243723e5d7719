// Global gradient norm over many tensors, and clipping to it.
//
//   norm = sqrt(sum_k sum_i t_k[i]^2),  out_k[i] = t_k[i] * (norm > max ? max / norm : 1)
//
// Both passes are bound by HBM: the norm reads 4 bytes an element, the scaling
// reads 4 and writes 4 (50 million elements: 34.5 us, 5.8 TB/s, and 63.4 us, 5.5 TB/s at a
// cold cache; 150.8 million: 291 us for both, 95 % of a copy's rate).  Squares are summed in float64 (no overflow below
// 1e154, and at 64 DFMA a clock and SM far from the bound), per thread, then
// per CTA in a fixed tree, then over the CTAs in index order, so the same
// tensors give the same bits.  No third launch joins the CTAs' sums: every CTA
// of the scaling adds the up to 1184 partial sums of a launch itself, in the
// same order.  Of many launches (views with gaps) there are too many for that,
// and one CTA adds them first.
//
// All tensors that are dense in memory go through one launch per pass: their
// addresses and sizes travel in the kernel's parameters (28 bytes each, up to
// 1024 in the 32 KB of a launch), cut into pieces of 8192 elements that the CTAs
// take in turn.  Views with gaps take a launch of their own.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstring>
#include <exception>
#include <vector>

#include "operators.cuh"

namespace mtc {
namespace {

constexpr int kPiece = 8192;   // elements: 256 threads x 8 float4
constexpr int kThreads = 256;

template <int N>
struct DenseTable {
    int count;
    int pieces;
    int in_place;  // every dst is its src
    int first_piece[N];
    const float *src[N];
    float *dst[N];
    long long n[N];
};

struct StridedTensor {
    long long numel;
    int rank;
    long long shape[MTC_MAX_RANK];
    long long src_stride[MTC_MAX_RANK], dst_stride[MTC_MAX_RANK];
    const float *src;
    float *dst;
};

__device__ __forceinline__ double block_sum(double v) {
    __shared__ double part[32];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    __syncthreads();
    if (lane == 0) part[warp] = v;
    __syncthreads();
    const int warps = blockDim.x / 32;
    v = lane < warps ? part[lane] : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

// Sum of the CTAs' partial sums; every thread of every CTA gets the same value.
__device__ __forceinline__ double sum_partials(const double *partials, int n) {
    double v = 0.0;
#pragma unroll 8
    for (int i = threadIdx.x; i < n; i += blockDim.x) v += partials[i];
    return block_sum(v);
}

__device__ __forceinline__ float clip_factor(double norm, float max_norm) {
    if (isnan(norm)) return __int_as_float(0x7FC00000);
    return norm > static_cast<double>(max_norm) ? static_cast<float>(static_cast<double>(max_norm) / norm) : 1.0f;
}

// The tensor that piece p belongs to, and the elements [begin, end) of it.  The
// first piece of a tensor also takes the up to three elements before its first
// 16-byte boundary, so that every later piece starts on one.
template <int N>
__device__ __forceinline__ int find_piece(const DenseTable<N> &t, int p, long long &begin, long long &end, int &head) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (t.first_piece[mid] <= p) lo = mid;
        else hi = mid - 1;
    }
    const long long k = p - t.first_piece[lo];
    head = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(t.src[lo]) & 15)) / 4) & 3;
    begin = k == 0 ? 0 : head + k * kPiece;
    end = head + (k + 1) * kPiece;
    if (end > t.n[lo]) end = t.n[lo];
    return lo;
}

__device__ __forceinline__ double square(float x) { return static_cast<double>(x) * static_cast<double>(x); }

template <int N>
__global__ void __launch_bounds__(kThreads) k_square_sum(const __grid_constant__ DenseTable<N> t, double *partials) {
    double acc0 = 0.0, acc1 = 0.0;
    for (int p = blockIdx.x; p < t.pieces; p += gridDim.x) {
        long long begin, end;
        int head;
        const int k = find_piece(t, p, begin, end, head);
        const float *src = t.src[k];
        long long at = begin;
        if (begin == 0 && head > 0) {
            at = head < end ? head : end;
            if (threadIdx.x < at) acc0 += square(src[threadIdx.x]);
        }
        const float4 *v4 = reinterpret_cast<const float4 *>(src + at);
        const int n4 = static_cast<int>((end - at) / 4);
        if (n4 == kPiece / 4) {
            float4 v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = v4[threadIdx.x + u * kThreads];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                acc0 += square(v[u].x);
                acc1 += square(v[u].y);
                acc0 += square(v[u].z);
                acc1 += square(v[u].w);
            }
        } else {
            for (int i = threadIdx.x; i < n4; i += kThreads) {
                const float4 v = v4[i];
                acc0 += square(v.x);
                acc1 += square(v.y);
                acc0 += square(v.z);
                acc1 += square(v.w);
            }
            for (long long i = at + 4ll * n4 + threadIdx.x; i < end; i += kThreads) acc1 += square(src[i]);
        }
    }
    const double sum = block_sum(acc0 + acc1);
    if (threadIdx.x == 0) partials[blockIdx.x] = sum;
}

// Pieces in descending order: the end of the last pass is what L2 still holds.
template <int N>
__global__ void __launch_bounds__(kThreads) k_scale(const __grid_constant__ DenseTable<N> t, const double *partials,
                                                    int n_partials, float max_norm, float *norm_out) {
    wait_for_previous();
    const double norm = sqrt(sum_partials(partials, n_partials));
    const float c = clip_factor(norm, max_norm);
    if (norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = static_cast<float>(norm);
    if (c == 1.0f && t.in_place) return;
    for (int p = t.pieces - 1 - static_cast<int>(blockIdx.x); p >= 0; p -= gridDim.x) {
        long long begin, end;
        int head;
        const int k = find_piece(t, p, begin, end, head);
        const float *src = t.src[k];
        float *dst = t.dst[k];
        long long at = begin;
        if (begin == 0 && head > 0) {
            at = head < end ? head : end;
            if (threadIdx.x < at) dst[threadIdx.x] = src[threadIdx.x] * c;
        }
        int n4 = 0;
        if ((reinterpret_cast<uintptr_t>(dst + at) & 15) == 0) {
            n4 = static_cast<int>((end - at) / 4);
            const float4 *v4 = reinterpret_cast<const float4 *>(src + at);
            float4 *o4 = reinterpret_cast<float4 *>(dst + at);
            if (n4 == kPiece / 4) {
                float4 v[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) v[u] = v4[threadIdx.x + u * kThreads];
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    o4[threadIdx.x + u * kThreads] = make_float4(v[u].x * c, v[u].y * c, v[u].z * c, v[u].w * c);
            } else {
                for (int i = threadIdx.x; i < n4; i += kThreads) {
                    const float4 v = v4[i];
                    o4[i] = make_float4(v.x * c, v.y * c, v.z * c, v.w * c);
                }
            }
        }
#pragma unroll 8
        for (long long i = at + 4ll * n4 + threadIdx.x; i < end; i += kThreads) dst[i] = src[i] * c;
    }
}

__device__ __forceinline__ void strided_offsets(const StridedTensor &t, long long i, long long &s, long long &d) {
    s = d = 0;
    for (int a = t.rank - 1; a >= 0; --a) {
        const long long q = i / t.shape[a], c = i - q * t.shape[a];
        s += c * t.src_stride[a];
        d += c * t.dst_stride[a];
        i = q;
    }
}

__global__ void __launch_bounds__(kThreads) k_square_sum_strided(const StridedTensor t, double *partials) {
    double acc = 0.0;
    for (long long i = blockIdx.x * static_cast<long long>(kThreads) + threadIdx.x; i < t.numel;
         i += static_cast<long long>(gridDim.x) * kThreads) {
        long long s, d;
        strided_offsets(t, i, s, d);
        acc += square(t.src[s]);
    }
    const double sum = block_sum(acc);
    if (threadIdx.x == 0) partials[blockIdx.x] = sum;
}

__global__ void __launch_bounds__(kThreads) k_scale_strided(const StridedTensor t, const double *partials,
                                                            int n_partials, float max_norm) {
    wait_for_previous();
    const float c = clip_factor(sqrt(sum_partials(partials, n_partials)), max_norm);
    for (long long i = blockIdx.x * static_cast<long long>(kThreads) + threadIdx.x; i < t.numel;
         i += static_cast<long long>(gridDim.x) * kThreads) {
        long long s, d;
        strided_offsets(t, i, s, d);
        t.dst[d] = t.src[s] * c;
    }
}

__global__ void __launch_bounds__(kThreads) k_write_norm(const double *partials, int n_partials, float *norm) {
    const double sum = sum_partials(partials, n_partials);
    if (threadIdx.x == 0) *norm = static_cast<float>(sqrt(sum));
}

// One partial sum in the place behind all others, in their stead.
__global__ void __launch_bounds__(kThreads) k_total(double *partials, int n_partials) {
    wait_for_previous();
    const double sum = sum_partials(partials, n_partials);
    if (threadIdx.x == 0) partials[n_partials] = sum;
}

// ------------------------------------------------------------------- host --

// Partial sums that every CTA of the scaling adds itself: those of three launches at most.  Each
// CTA of each launch reads them, which is quadratic in the number of views with gaps (of 1000 x 1022
// each: 4 take 91 us so and 82 with their sum taken first, 100 18.0 and 2.3 ms).
constexpr int kOwnPartials = 4096;

struct Dense {
    const float *src;
    float *dst;
    long long n;
};

struct Plan {
    std::vector<Dense> dense;
    std::vector<StridedTensor> strided;
    long long dense_total = 0;
};

// Axes by falling stride of the source: the order of the elements does not
// matter here, so a permuted dense tensor is a flat one too.
void sort_axes(IterSpace &s) {
    for (int i = 1; i < s.rank; ++i)
        for (int j = i; j > 0 && s.stride[0][j - 1] < s.stride[0][j]; --j) {
            std::swap(s.shape[j - 1], s.shape[j]);
            for (int k = 0; k < s.nops; ++k) std::swap(s.stride[k][j - 1], s.stride[k][j]);
        }
}

int plan_tensor(const mtc_desc &in, const mtc_desc &out, Plan &plan) {
    IterSpace s;
    s.rank = in.rank;
    s.nops = 2;
    for (int i = 0; i < in.rank; ++i) {
        s.shape[i] = in.shape[i];
        s.stride[0][i] = in.strides[i];
        s.stride[1][i] = out.strides[i];
    }
    if (numel_of(in) == 0) return MTC_OK;
    for (int i = 0; i < s.rank; ++i)
        if (s.shape[i] == 1) s.stride[0][i] = s.stride[1][i] = 0;  // last in the order, then dropped
    sort_axes(s);
    simplify(s);
    const float *src = float_at(&in);
    float *dst = float_at(&out);
    if (s.rank == 1 && (s.numel == 1 || (s.stride[0][0] == 1 && s.stride[1][0] == 1))) {
        plan.dense.push_back(Dense{src, dst, s.numel});
        plan.dense_total += s.numel;
        return MTC_OK;
    }
    StridedTensor t;
    std::memset(&t, 0, sizeof(t));
    t.numel = s.numel;
    t.rank = s.rank;
    for (int i = 0; i < s.rank; ++i) {
        t.shape[i] = s.shape[i];
        t.src_stride[i] = s.stride[0][i];
        t.dst_stride[i] = s.stride[1][i];
    }
    t.src = src;
    t.dst = dst;
    plan.strided.push_back(t);
    return MTC_OK;
}

constexpr int kSmallTable = 64, kLargeTable = 1024;

int pieces_of(const Dense &d) {
    const long long head = static_cast<long long>((16 - (reinterpret_cast<uintptr_t>(d.src) & 15)) / 4) & 3;
    const long long body = d.n > head ? d.n - head : 0;
    const long long p = (body + kPiece - 1) / kPiece;
    return static_cast<int>(p > 0 ? p : 1);
}

template <int N>
void fill_table(DenseTable<N> &t, const Dense *d, int count) {
    t.count = count;
    t.in_place = 1;
    int p = 0;
    for (int i = 0; i < count; ++i) {
        t.first_piece[i] = p;
        t.src[i] = d[i].src;
        t.dst[i] = d[i].dst;
        t.n[i] = d[i].n;
        t.in_place &= d[i].src == d[i].dst;
        p += pieces_of(d[i]);
    }
    t.pieces = p;
}

struct Launcher {
    const Plan &plan;
    cudaStream_t stream;
    int sms;
    double *partials = nullptr;
    int n_partials = 0;

    int grid(long long pieces) const {
        const long long most = static_cast<long long>(sms) * 8;  // eight CTAs of 256 threads fill an SM
        return static_cast<int>(pieces < most ? pieces : most);
    }

    template <int N, class F>
    int each_table(F &&launch) const {
        for (size_t at = 0; at < plan.dense.size(); at += N) {
            DenseTable<N> t;
            fill_table(t, plan.dense.data() + at, static_cast<int>(std::min<size_t>(N, plan.dense.size() - at)));
            MTC_TRY(launch(t));
        }
        return MTC_OK;
    }

    template <class F>
    int tables(F &&launch) const {
        return plan.dense.size() <= kSmallTable ? each_table<kSmallTable>(launch) : each_table<kLargeTable>(launch);
    }

    int count_partials() {
        long long n = 0;
        MTC_TRY(tables([&](const auto &t) {
            n += grid(t.pieces);
            return MTC_OK;
        }));
        for (const StridedTensor &t : plan.strided) n += grid((t.numel + kThreads - 1) / kThreads);
        if (n > INT_MAX) return fail(MTC_ERR_UNSUPPORTED, "too many tensors");
        n_partials = static_cast<int>(n);
        return MTC_OK;
    }

    int sum_squares() {
        double *to = partials;
        MTC_TRY(tables([&](const auto &t) {
            const int g = grid(t.pieces);
            k_square_sum<<<g, kThreads, 0, stream>>>(t, to);
            to += g;
            return check_launch("sum of squares");
        }));
        for (const StridedTensor &t : plan.strided) {
            const int g = grid((t.numel + kThreads - 1) / kThreads);
            k_square_sum_strided<<<g, kThreads, 0, stream>>>(t, to);
            to += g;
            MTC_TRY(check_launch("sum of squares (strided)"));
        }
        return MTC_OK;
    }

    int scale(float max_norm, float *norm) {
        if (n_partials > kOwnPartials) {
            MTC_TRY(launch_dependent("global norm (total)", k_total, 1, kThreads, 0, stream, partials, n_partials));
            partials += n_partials;
            n_partials = 1;
        }
        float *write = norm;  // by the first launch alone
        MTC_TRY(tables([&](const auto &t) {
            constexpr int N = sizeof(t.n) / sizeof(t.n[0]);
            float *once = write;
            write = nullptr;
            return launch_dependent("gradient clipping", k_scale<N>, grid(t.pieces), kThreads, 0, stream, t, partials,
                                    n_partials, max_norm, once);
        }));
        for (const StridedTensor &t : plan.strided) {
            MTC_TRY(launch_dependent("gradient clipping (strided)", k_scale_strided,
                                     grid((t.numel + kThreads - 1) / kThreads), kThreads, 0, stream, t, partials,
                                     n_partials, max_norm));
        }
        if (write != nullptr) return write_norm(write);
        return MTC_OK;
    }

    int write_norm(float *norm) {
        k_write_norm<<<1, kThreads, 0, stream>>>(partials, n_partials, norm);
        return check_launch("global norm");
    }
};

int check_lists(const mtc_desc *tensors, int32_t n, const mtc_desc *outs, const mtc_desc *norm) {
    if (n < 0 || (n > 0 && (tensors == nullptr || outs == nullptr)))
        return fail(MTC_ERR_INVALID_ARGUMENT, "bad tensor list");
    for (int i = 0; i < n; ++i) {
        MTC_TRY(need_float(&tensors[i], "tensor"));
        MTC_TRY(need_float(&outs[i], "output"));
        bool same = tensors[i].rank == outs[i].rank;
        for (int d = 0; same && d < tensors[i].rank; ++d) same = tensors[i].shape[d] == outs[i].shape[d];
        if (!same) return fail(MTC_ERR_INVALID_ARGUMENT, "output %d differs in shape from its tensor", i);
        if (numel_of(tensors[i]) > static_cast<int64_t>(kPiece) * (int64_t{1} << 29))
            return fail(MTC_ERR_UNSUPPORTED, "tensor %d has too many elements", i);
    }
    if (norm != nullptr) {
        MTC_TRY(need_float(norm, "norm"));
        if (numel_of(*norm) != 1) return fail(MTC_ERR_INVALID_ARGUMENT, "norm has %lld elements instead of one",
                                              static_cast<long long>(numel_of(*norm)));
    }
    return MTC_OK;
}

int run_norm(const mtc_desc *tensors, int32_t n, bool clip, float max_norm, const mtc_desc *outs, const mtc_desc *norm,
             cudaStream_t stream) {
    MTC_TRY(check_lists(tensors, n, outs, norm));
    if (clip) {
        for (int i = 0; i < n; ++i) MTC_TRY(need_distinct(&outs[i], "output"));
        MTC_TRY(need_apart(outs, n));
    }
    Plan plan;
    for (int i = 0; i < n; ++i) MTC_TRY(plan_tensor(tensors[i], outs[i], plan));
    // pieces are counted in 32 bits, the first and the last of a tensor apart
    if (plan.dense_total / kPiece + 2ll * n > (int64_t{1} << 30))
        return fail(MTC_ERR_UNSUPPORTED, "the tensors have too many elements");
    float *norm_ptr = norm != nullptr ? float_at(norm) : nullptr;
    Launcher l{plan, stream, sm_count(current_device())};
    MTC_TRY(l.count_partials());
    if (l.n_partials == 0 && norm_ptr == nullptr) return MTC_OK;
    Workspace ws;
    MTC_TRY(ws.allocate(padded(static_cast<size_t>(l.n_partials + 1) * sizeof(double)), stream));
    l.partials = ws.take<double>(static_cast<size_t>(l.n_partials + 1) * sizeof(double));
    MTC_TRY(l.sum_squares());
    return clip ? l.scale(max_norm, norm_ptr) : l.write_norm(norm_ptr);
}

}  // namespace
}  // namespace mtc

using namespace mtc;

extern "C" {

int mtc_global_norm(const mtc_desc *tensors, int32_t n, const mtc_desc *norm, void *stream) {
    clear_error();
    if (norm == nullptr) return fail(MTC_ERR_INVALID_ARGUMENT, "norm: null descriptor");
    try {
        return run_norm(tensors, n, false, 0.0f, tensors, norm, static_cast<cudaStream_t>(stream));
    } catch (const std::exception &e) {
        return fail(MTC_ERR_RUNTIME, "global norm: %s", e.what());
    }
}

int mtc_clip_global_norm(const mtc_desc *tensors, int32_t n, float max_norm, const mtc_desc *outs,
                         const mtc_desc *norm, void *stream) {
    clear_error();
    if (!(max_norm >= 0.0f)) return fail(MTC_ERR_INVALID_ARGUMENT, "max_norm %g is not a number >= 0", max_norm);
    try {
        return run_norm(tensors, n, true, max_norm, outs, norm, static_cast<cudaStream_t>(stream));
    } catch (const std::exception &e) {
        return fail(MTC_ERR_RUNTIME, "gradient clipping: %s", e.what());
    }
}

}  // extern "C"
