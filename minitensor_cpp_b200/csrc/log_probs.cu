// Log probabilities of given tokens with the entropy and the likeliest alternatives of each
// distribution, and the logits' gradient of any loss of the first two.
//
//   z = scale x,  M = max x,  d_v = scale (x_v - M),  S = sum_v exp d_v
//   log p_v = d_v - log S,  lse = scale M + log S
//   H = -sum_v p_v log p_v = log S + E,  E = -(sum_v d_v exp d_v) / S >= 0
//   dx_v = scale (dlp ([v = t] - p_v) - dH p_v (d_v + E))          (log p_v + H = d_v + E)
//
// S is kept as n + r, the number of elements that equal M and the sum of the others, so that
// log S = log1p(n - 1 + r), 1 - p_t and E of a row that is sure of its token keep the digits of
// what is left.  The gradient takes its statistics from the row anew instead of from the
// caller: a log-sum-exp rounded to float32 would cost them.
//
// Bound by HBM: 4 bytes an element, and for the gradient 8.  Up to 1024 classes a warp holds
// a row in its registers.  Beyond, a CTA streams it once: a thread keeps the maximum of what it
// has seen and sums relative to it, rescaled where a batch raises the maximum.  The gradient
// reads the row a second time, last elements first, out of L2.
//
// The k likeliest (k <= 32) need no second pass over the row.  Of 32 groups of threads each has
// a maximum, and the k-th largest of these is a bound that k threads' maxima reach; the k-th
// largest of those threads' maxima, told apart by their index where they are equal, is the
// next; exactly k threads reach that one, and only what these have read is looked at again.
// What is found is ranked by counting.  Elements that crowd in a few threads overflow the
// list and cost k passes over the row instead.
#include <climits>
#include <cmath>
#include <cstring>
#include <exception>

#include "operators.cuh"

namespace mtc {
namespace {

constexpr int kMostTop = 32;
constexpr int kWarpVocab = 1024;

enum Operand { kLogits, kTokens, kLogProbs, kLse, kEntropy, kTopLogProbs, kTopTokens, kDLogProbs, kDEntropy, kDLogits, kOperands };

struct RowArgs {
    int64_t rows;
    int vocab;
    int rank;  // of the leading axes, joined where they can be
    int64_t shape[MTC_MAX_RANK];
    int64_t stride[kOperands][MTC_MAX_RANK];
    const float *logits;
    int64_t cs;  // of the vocabulary's axis
    const long long *tokens;
    long long ignore;
    float scale, scale2;  // the second for 2^x: scale / ln 2
    float *log_probs, *lse, *entropy;
    int top;
    float *top_log_probs;
    long long *top_tokens;
    int64_t top_log_probs_s, top_tokens_s;
    const float *dlog_probs, *dentropy;
    float *dlogits;
    int64_t dcs;
    unsigned long long *err;
};

__device__ __forceinline__ int64_t at(const RowArgs &a, Operand o, int64_t row) {
    if (a.rank == 1) return row * a.stride[o][0];
    int64_t off = 0;
    for (int i = a.rank - 1; i >= 0; --i) {
        const int64_t q = row / a.shape[i];
        off += (row - q * a.shape[i]) * a.stride[o][i];
        row = q;
    }
    return off;
}

// -------------------------------------------------------------- statistics --

constexpr float kFloor = -200.0f;  // exponents below it are zeros of float32, of base 2 and of base e

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// Floats as whole numbers that order as they do: NaN the largest, -0 as 0.
__device__ __forceinline__ int ordered(float x) {
    if (isnan(x)) return INT_MAX;
    const int b = __float_as_int(x + 0.0f);
    return b < 0 ? b ^ INT_MAX : b;
}
constexpr int kNothing = INT_MIN;  // below all of them

__device__ __forceinline__ float from_ordered(int o) { return __int_as_float(o < 0 ? o ^ INT_MAX : o); }

// With the index, the lower the larger: no two are equal.
__device__ __forceinline__ unsigned long long key_of(int o, int index) {
    return (static_cast<unsigned long long>(static_cast<unsigned int>(o) ^ 0x80000000u) << 32) |
           (0xFFFFFFFFu - static_cast<unsigned int>(index));
}
__device__ __forceinline__ int key_index(unsigned long long k) { return static_cast<int>(0xFFFFFFFFu - static_cast<unsigned int>(k)); }
__device__ __forceinline__ float key_value(unsigned long long k) {
    return from_ordered(static_cast<int>(static_cast<unsigned int>(k >> 32) ^ 0x80000000u));
}

// Of what has been seen: the largest x, how many equal it, and of the others the sums of
// 2^u and u 2^u with u = scale2 (x - m).  -inf counts as nothing; bad: NaN or +inf.
struct Stats {
    float m = -INFINITY, n = 0.0f, r = 0.0f, e = 0.0f;
    bool bad = false;

    __device__ __forceinline__ void rise(float to, float scale2) {
        const float by = fmaxf((m - to) * scale2, kFloor), f = exp2_fast(by), all = n + r;
        r = all * f;
        e = (e + by * all) * f;
        n = 0.0f;
        m = to;
    }

    template <int N>
    __device__ __forceinline__ void add(const float (&x)[N], float largest, float scale2) {
        if (!(largest < INFINITY)) {
            bad = true;
            return;
        }
        if (largest == -INFINITY) return;
        if (largest > m) rise(largest, scale2);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float u = fmaxf((x[i] - m) * scale2, kFloor), y = exp2_fast(u);
            if (x[i] == m) {
                n += 1.0f;
            } else {
                r += y;
                e = fmaf(y, u, e);
            }
        }
    }

    // Of a warp's lanes together, the same in all.
    __device__ __forceinline__ void join_warp(float scale2) {
        bad = __any_sync(0xFFFFFFFFu, bad);
        const float top = from_ordered(__reduce_max_sync(0xFFFFFFFFu, ordered(m)));
        if (top > m) rise(top, scale2);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            n += __shfl_xor_sync(0xFFFFFFFFu, n, o);
            r += __shfl_xor_sync(0xFFFFFFFFu, r, o);
            e += __shfl_xor_sync(0xFFFFFFFFu, e, o);
        }
    }
};

// What the outputs need of a row.
struct Row {
    float m, total, log_total, spread, others;  // M, S, log S, E, S - 1
    bool bad, empty;

    __device__ __forceinline__ Row(const Stats &s) {
        constexpr float ln2 = 0.69314718055994531f;
        m = s.m;
        others = s.n - 1.0f + s.r;
        total = s.n + s.r;
        log_total = log1pf(others);
        spread = -ln2 * s.e / total;
        bad = s.bad;
        empty = s.n == 0.0f;
    }
    __device__ __forceinline__ float log_prob(float x, float scale) const {
        if (bad) return __int_as_float(0x7FC00000);
        if (empty) return -INFINITY;
        return (x - m) * scale - log_total;
    }
};

__device__ __forceinline__ void write_row(const RowArgs &a, int64_t row, const Row &s, float x_token) {
    const float nan = __int_as_float(0x7FC00000);
    if (a.log_probs != nullptr) a.log_probs[at(a, kLogProbs, row)] = s.log_prob(x_token, a.scale);
    if (a.lse != nullptr) a.lse[at(a, kLse, row)] = s.bad ? nan : s.empty ? -INFINITY : fmaf(s.m, a.scale, s.log_total);
    if (a.entropy != nullptr) a.entropy[at(a, kEntropy, row)] = s.bad ? nan : s.empty ? 0.0f : s.log_total + s.spread;
}

__device__ __forceinline__ void write_top(const RowArgs &a, int64_t row, const Row &s, int rank, unsigned long long key) {
    if (a.top_log_probs != nullptr)
        a.top_log_probs[at(a, kTopLogProbs, row) + rank * a.top_log_probs_s] = s.log_prob(key_value(key), a.scale);
    if (a.top_tokens != nullptr) a.top_tokens[at(a, kTopTokens, row) + rank * a.top_tokens_s] = key_index(key);
}

// A row that is not scored; by the threads of a warp or a CTA.
__device__ __forceinline__ void write_skipped(const RowArgs &a, int64_t row, int thread, int threads) {
    if (a.dlogits != nullptr) {
        float *to = a.dlogits + at(a, kDLogits, row);
        for (int v = thread; v < a.vocab; v += threads) to[v * a.dcs] = 0.0f;
        return;
    }
    if (thread == 0) {
        if (a.log_probs != nullptr) a.log_probs[at(a, kLogProbs, row)] = 0.0f;
        if (a.lse != nullptr) a.lse[at(a, kLse, row)] = 0.0f;
        if (a.entropy != nullptr) a.entropy[at(a, kEntropy, row)] = 0.0f;
    }
    for (int k = thread; k < a.top; k += threads) {
        if (a.top_log_probs != nullptr) a.top_log_probs[at(a, kTopLogProbs, row) + k * a.top_log_probs_s] = 0.0f;
        if (a.top_tokens != nullptr) a.top_tokens[at(a, kTopTokens, row) + k * a.top_tokens_s] = -1;
    }
}

// The row's token, or -1 without tokens; false: the row is not scored.
__device__ __forceinline__ bool token_of(const RowArgs &a, int64_t row, bool report, int &token) {
    token = -1;
    if (a.tokens == nullptr) return true;
    const long long t = a.tokens[at(a, kTokens, row)];
    if (t == a.ignore) return false;
    if (t < 0 || t >= a.vocab) {
        if (report) report_index(a.err, t);
        return false;
    }
    token = static_cast<int>(t);
    return true;
}

// One element of the gradient.
struct Slope {
    Row s;
    float by_prob, by_entropy, scale, inverse;
    int token;

    __device__ __forceinline__ Slope(const RowArgs &a, int64_t row, const Row &stats, int t) : s(stats), token(t) {
        scale = a.scale;
        by_prob = a.dlog_probs != nullptr ? a.dlog_probs[at(a, kDLogProbs, row)] * scale : 0.0f;
        by_entropy = a.dentropy != nullptr ? a.dentropy[at(a, kDEntropy, row)] * scale : 0.0f;
        inverse = 1.0f / s.total;
    }
    __device__ __forceinline__ float operator()(float x, int v) const {
        if (s.bad) return __int_as_float(0x7FC00000);
        if (s.empty) return 0.0f;
        const float d = fmaxf((x - s.m) * scale, kFloor);
        const float p = expf(d) * inverse;
        const float by_own = by_entropy * (d + s.spread);
        if (v == token) return by_prob * (x == s.m ? s.others * inverse : 1.0f - p) - p * by_own;
        return -p * (by_prob + by_own);
    }
};

// ------------------------------------------------------------ a warp a row --

__device__ __forceinline__ int sorted_falling(int v) {
    const int lane = threadIdx.x % 32;
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int o = size / 2; o > 0; o >>= 1) {
            const int w = __shfl_xor_sync(0xFFFFFFFFu, v, o);
            const bool larger = ((lane & o) == 0) == ((lane & size) == 0);
            v = larger ? max(v, w) : min(v, w);
        }
    return v;
}

__device__ __forceinline__ unsigned long long warp_max(unsigned long long k) {
    const unsigned int hi = __reduce_max_sync(0xFFFFFFFFu, static_cast<unsigned int>(k >> 32));
    const unsigned int lo =
        __reduce_max_sync(0xFFFFFFFFu, static_cast<unsigned int>(k >> 32) == hi ? static_cast<unsigned int>(k) : 0u);
    return (static_cast<unsigned long long>(hi) << 32) | lo;
}

constexpr int kWarpList = 64;

// R elements a lane, the 32 lanes side by side.
template <int R, bool GRAD>
__global__ void __launch_bounds__(256) k_warp_rows(const RowArgs a) {
    __shared__ unsigned long long lists[8][kWarpList];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + warp; row < a.rows; row += static_cast<int64_t>(gridDim.x) * 8) {
        int token;
        if (!token_of(a, row, lane == 0, token)) {
            write_skipped(a, row, lane, 32);
            continue;
        }
        const float *src = a.logits + at(a, kLogits, row);
        float x[R];
#pragma unroll
        for (int j = 0; j < R; ++j) x[j] = lane + 32 * j < a.vocab ? src[(lane + 32 * j) * a.cs] : -INFINITY;
        float largest = x[0];
#pragma unroll
        for (int j = 1; j < R; ++j) largest = max_nan(largest, x[j]);
        const int mine = lane < a.vocab ? ordered(largest) : kNothing;
        const float top = from_ordered(__reduce_max_sync(0xFFFFFFFFu, mine));
        Stats st;
        st.add(x, top, a.scale2);
        if (!st.bad) {
            st.m = top;
            st.join_warp(a.scale2);
        }
        const Row s(st);
        if (GRAD) {
            const Slope slope(a, row, s, token);
            float *to = a.dlogits + at(a, kDLogits, row);
#pragma unroll
            for (int j = 0; j < R; ++j)
                if (lane + 32 * j < a.vocab) to[(lane + 32 * j) * a.dcs] = slope(x[j], lane + 32 * j);
            continue;
        }
        if (lane == 0) write_row(a, row, s, token >= 0 ? src[token * a.cs] : 0.0f);
        if (a.top == 0) continue;
        // the k-th largest of the lanes' maxima: k elements reach it
        const int bound = __shfl_sync(0xFFFFFFFFu, sorted_falling(mine), a.top - 1);
        unsigned long long *list = lists[warp];
        int found = 0;
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const int o = lane + 32 * j < a.vocab ? ordered(x[j]) : kNothing;
            const bool hit = o >= bound && o != kNothing;
            const unsigned int hits = __ballot_sync(0xFFFFFFFFu, hit);
            if (hits == 0) continue;
            const int to = found + __popc(hits & ((1u << lane) - 1));
            if (hit && to < kWarpList) list[to] = key_of(o, lane + 32 * j);
            found += __popc(hits);
        }
        __syncwarp();
        if (found <= kWarpList) {
            for (int i = lane; i < found; i += 32) {
                const unsigned long long k = list[i];
                int rank = 0;
                for (int j = 0; j < found; ++j) rank += list[j] > k;
                if (rank < a.top) write_top(a, row, s, rank, k);
            }
            __syncwarp();
            continue;
        }
        unsigned long long last = ~0ull;  // equal elements: one after another
        for (int rank = 0; rank < a.top; ++rank) {
            unsigned long long best = 0;
#pragma unroll
            for (int j = 0; j < R; ++j) {
                const unsigned long long k = lane + 32 * j < a.vocab ? key_of(ordered(x[j]), lane + 32 * j) : 0;
                if (k < last && k > best) best = k;
            }
            last = warp_max(best);
            if (lane == 0) write_top(a, row, s, rank, last);
        }
    }
}

// ------------------------------------------------------------- a CTA a row --

constexpr int kBatch = 8;      // vectors of four that a thread has in flight
constexpr int kList = 512;

// A row in vectors of four that start on 16-byte boundaries, and up to three elements before
// and behind them.  With gaps between the elements, a vector is four loads.
template <bool VEC>
struct Source {
    const float *p;
    int64_t cs;
    int vocab, head, vecs, tail;

    __device__ __forceinline__ Source(const RowArgs &a, int64_t row) {
        p = a.logits + at(a, kLogits, row);
        cs = a.cs;
        vocab = a.vocab;
        head = VEC ? static_cast<int>((16 - (reinterpret_cast<uintptr_t>(p) & 15)) / 4) & 3 : 0;
        vecs = (vocab - head) / 4;
        tail = vocab - head - 4 * vecs;
    }
    __device__ __forceinline__ float4 vec(int j) const {
        if (VEC) return *reinterpret_cast<const float4 *>(p + head + 4 * j);
        const float *q = p + 4 * j * cs;
        return make_float4(q[0], q[cs], q[2 * cs], q[3 * cs]);
    }
    __device__ __forceinline__ float one(int v) const { return p[v * (VEC ? 1 : cs)]; }
    __device__ __forceinline__ int tail_at() const { return head + 4 * vecs; }
};

template <int T>
__device__ __forceinline__ void join_block(Stats &s, float scale2, float4 *parts) {
    static_assert(T >= 64 && T <= 1024, "warps");
    constexpr int W = T / 32;
    s.join_warp(scale2);
    if (threadIdx.x % 32 == 0) parts[threadIdx.x / 32] = make_float4(s.bad ? INFINITY : s.m, s.n, s.r, s.e);
    __syncthreads();
    const int lane = threadIdx.x % 32;
    Stats all;
    if (lane < W) {
        const float4 p = parts[lane];
        all.m = p.x;
        all.n = p.y;
        all.r = p.z;
        all.e = p.w;
        all.bad = p.x == INFINITY;
        if (all.bad) all.m = -INFINITY;
    }
    all.join_warp(scale2);
    s = all;
}

struct TopShared {
    int group[32];
    int found, listed;
    unsigned long long bound;
    unsigned long long maxima[1024];
    unsigned long long list[kList];
    unsigned long long warps[32];
};

// The k likeliest, see above.  `best` is this thread's largest element, first seen in batch
// `where` (kHead, kTail: before and behind the vectors).
constexpr int kHead = -1, kTail = -2;

template <int T, bool VEC>
__device__ __forceinline__ void find_top(const RowArgs &a, int64_t row, const Source<VEC> &src, const Row &s, int best,
                                         int where, TopShared &sh) {
    constexpr int G = T / 32;
    const int thread = threadIdx.x, lane = thread % 32;
    int m = best;
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    if (thread % G == 0) sh.group[thread / G] = m;
    if (thread == 0) sh.found = sh.listed = 0;
    __syncthreads();
    const int first = __shfl_sync(0xFFFFFFFFu, sorted_falling(sh.group[lane]), a.top - 1);
    unsigned long long mine = 0;
    if (best >= first) {
        int index = where == kHead ? thread : src.tail_at() + thread;
        if (where >= 0) {
            for (int u = kBatch - 1; u >= 0; --u) {
                const int j = thread + T * (where * kBatch + u);
                if (j >= src.vecs) continue;
                const float4 v = src.vec(j);
                const int i = src.head + 4 * j;
                if (ordered(v.w) == best) index = i + 3;
                if (ordered(v.z) == best) index = i + 2;
                if (ordered(v.y) == best) index = i + 1;
                if (ordered(v.x) == best) index = i;
            }
        }
        mine = key_of(best, index);
        sh.maxima[atomicAdd(&sh.found, 1)] = mine;
    }
    __syncthreads();
    const int found = sh.found;
    if (thread < found) {
        const unsigned long long k = sh.maxima[thread];
        int rank = 0;
        for (int j = 0; j < found; ++j) rank += sh.maxima[j] > k;
        if (rank == a.top - 1) sh.bound = k;
    }
    __syncthreads();
    const unsigned long long bound = sh.bound;
    auto look = [&](float x, int index) {
        const unsigned long long k = key_of(ordered(x), index);
        if (k < bound) return;
        const int to = atomicAdd(&sh.listed, 1);
        if (to < kList) sh.list[to] = k;
    };
    for (unsigned int of = __ballot_sync(0xFFFFFFFFu, mine >= bound); of != 0; of &= of - 1) {
        const int other = thread - lane + __ffs(of) - 1;
        for (int j = other + T * lane; j < src.vecs; j += T * 32) {
            const float4 v = src.vec(j);
            const int i = src.head + 4 * j;
            look(v.x, i);
            look(v.y, i + 1);
            look(v.z, i + 2);
            look(v.w, i + 3);
        }
        if (lane == 0 && other < src.head) look(src.one(other), other);
        if (lane == 1 && other < src.tail) look(src.one(src.tail_at() + other), src.tail_at() + other);
    }
    __syncthreads();
    const int listed = sh.listed;
    if (listed <= kList) {
        for (int i = thread; i < listed; i += T) {
            const unsigned long long k = sh.list[i];
            int rank = 0;
            for (int j = 0; j < listed; ++j) rank += sh.list[j] > k;
            if (rank < a.top) write_top(a, row, s, rank, k);
        }
        return;
    }
    unsigned long long last = ~0ull;
    for (int rank = 0; rank < a.top; ++rank) {
        unsigned long long most = 0;
        for (int v = thread; v < src.vocab; v += T) {
            const unsigned long long k = key_of(ordered(src.one(v)), v);
            if (k < last && k > most) most = k;
        }
        most = warp_max(most);
        __syncthreads();
        if (lane == 0) sh.warps[thread / 32] = most;
        __syncthreads();
        last = warp_max(lane < T / 32 ? sh.warps[lane] : 0);
        if (thread == 0) write_top(a, row, s, rank, last);
    }
}

template <int T, bool VEC, bool GRAD>
__global__ void __launch_bounds__(T) k_cta_rows(const RowArgs a) {
    __shared__ float4 parts[32];
    __shared__ TopShared sh;
    const int thread = threadIdx.x;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        int token;
        if (!token_of(a, row, thread == 0, token)) {
            write_skipped(a, row, thread, T);
            continue;
        }
        const Source<VEC> src(a, row);
        const float x_token = !GRAD && token >= 0 ? src.one(token) : 0.0f;
        Stats st;
        int best = kNothing, where = 0;
        auto keep = [&](float largest, int at) {
            if (GRAD) return;
            const int o = ordered(largest);
            if (o > best) {
                best = o;
                where = at;
            }
        };
        if (thread < src.head) {
            const float x[1] = {src.one(thread)};
            keep(x[0], kHead);
            st.add(x, x[0], a.scale2);
        }
        const int batches = (src.vecs + T * kBatch - 1) / (T * kBatch);
        for (int b = 0; b < batches; ++b) {
            float x[4 * kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int j = thread + T * (b * kBatch + u);
                const float4 v = j < src.vecs ? src.vec(j) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                x[4 * u] = v.x;
                x[4 * u + 1] = v.y;
                x[4 * u + 2] = v.z;
                x[4 * u + 3] = v.w;
            }
            float largest = x[0];
#pragma unroll
            for (int i = 1; i < 4 * kBatch; ++i) largest = max_nan(largest, x[i]);
            if (thread + T * b * kBatch < src.vecs) keep(largest, b);
            st.add(x, largest, a.scale2);
        }
        if (thread < src.tail) {
            const float x[1] = {src.one(src.tail_at() + thread)};
            keep(x[0], kTail);
            st.add(x, x[0], a.scale2);
        }
        join_block<T>(st, a.scale2, parts);
        const Row s(st);
        if (GRAD) {
            const Slope slope(a, row, s, token);
            float *to = a.dlogits + at(a, kDLogits, row);
            const bool whole = VEC && a.dcs == 1 && ((reinterpret_cast<uintptr_t>(to) ^ reinterpret_cast<uintptr_t>(src.p)) & 15) == 0;
            for (int b = batches - 1; b >= 0; --b) {
#pragma unroll
                for (int u = 0; u < kBatch; ++u) {
                    const int j = thread + T * (b * kBatch + u);
                    if (j >= src.vecs) continue;
                    const float4 v = src.vec(j);
                    const int i = src.head + 4 * j;
                    const float4 g = make_float4(slope(v.x, i), slope(v.y, i + 1), slope(v.z, i + 2), slope(v.w, i + 3));
                    if (whole) {
                        *reinterpret_cast<float4 *>(to + i) = g;
                    } else {
                        to[i * a.dcs] = g.x;
                        to[(i + 1) * a.dcs] = g.y;
                        to[(i + 2) * a.dcs] = g.z;
                        to[(i + 3) * a.dcs] = g.w;
                    }
                }
            }
            if (thread < src.head) to[thread * a.dcs] = slope(src.one(thread), thread);
            if (thread < src.tail) {
                const int i = src.tail_at() + thread;
                to[i * a.dcs] = slope(src.one(i), i);
            }
        } else {
            if (thread == 0) write_row(a, row, s, x_token);
            if (a.top > 0) find_top<T, VEC>(a, row, src, s, best, where, sh);
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------- host --

template <int R, bool GRAD>
int launch_warps(const RowArgs &a, cudaStream_t stream) {
    const int64_t ctas = (a.rows + 7) / 8, most = static_cast<int64_t>(sm_count(current_device())) * 64;
    k_warp_rows<R, GRAD><<<static_cast<unsigned>(ctas < most ? ctas : most), 256, 0, stream>>>(a);
    return check_launch("log probabilities (warps)");
}

template <int T, bool GRAD>
int launch_ctas(const RowArgs &a, cudaStream_t stream) {
    const unsigned grid = static_cast<unsigned>(a.rows < INT_MAX ? a.rows : INT_MAX);
    if (a.cs == 1) k_cta_rows<T, true, GRAD><<<grid, T, 0, stream>>>(a);
    else k_cta_rows<T, false, GRAD><<<grid, T, 0, stream>>>(a);
    return check_launch("log probabilities");
}

template <bool GRAD>
int launch(const RowArgs &a, cudaStream_t stream) {
    if (a.vocab <= 32) return launch_warps<1, GRAD>(a, stream);
    if (a.vocab <= 128) return launch_warps<4, GRAD>(a, stream);
    if (a.vocab <= 512) return launch_warps<16, GRAD>(a, stream);
    if (a.vocab <= kWarpVocab) return launch_warps<32, GRAD>(a, stream);
    if (a.vocab <= 8192) return launch_ctas<256, GRAD>(a, stream);
    return launch_ctas<512, GRAD>(a, stream);
}

// One operand over the leading axes of the logits; `extra` axes follow them.
int need_leading(const mtc_desc *d, const mtc_desc *logits, int extra, const char *name) {
    const int lead = logits->rank - 1;
    bool same = d->rank == lead + extra;
    for (int i = 0; same && i < lead; ++i) same = d->shape[i] == logits->shape[i];
    if (!same) return fail(MTC_ERR_INVALID_ARGUMENT, "%s: its leading axes differ from the logits'", name);
    return MTC_OK;
}

struct RowOperands {
    const mtc_desc *d[kOperands] = {};
};

int fill_args(const RowOperands &o, float scale, int64_t ignore, RowArgs &a) {
    static const char *const names[kOperands] = {"logits",  "tokens",     "log_probs",  "lse",      "entropy",
                                                 "top_log_probs", "top_tokens", "dlog_probs", "dentropy", "dlogits"};
    const mtc_desc *logits = o.d[kLogits];
    MTC_TRY(need_float(logits, names[kLogits]));
    if (logits->rank < 1) return fail(MTC_ERR_INVALID_ARGUMENT, "logits need an axis of classes");
    const int lead = logits->rank - 1;
    const int64_t vocab = logits->shape[lead];
    for (int k = 1; k < kOperands; ++k) {
        if (o.d[k] == nullptr) continue;
        MTC_TRY(k == kTokens || k == kTopTokens ? need_int(o.d[k], names[k]) : need_float(o.d[k], names[k]));
        MTC_TRY(need_leading(o.d[k], logits, k == kTopLogProbs || k == kTopTokens || k == kDLogits, names[k]));
        if (k != kTokens && k != kDLogProbs && k != kDEntropy) MTC_TRY(need_distinct(o.d[k], names[k]));
    }
    if (!(scale > 0.0f && scale <= 0x1p100f))
        return fail(MTC_ERR_INVALID_ARGUMENT, "scale %g is not in (0, 2^100]", scale);
    if (vocab == 0) return fail(MTC_ERR_INVALID_ARGUMENT, "logits over no classes");
    if (vocab > INT_MAX / 2) return fail(MTC_ERR_UNSUPPORTED, "%lld classes", static_cast<long long>(vocab));
    std::memset(&a, 0, sizeof(a));
    int64_t top = 0;
    for (const Operand k : {kTopLogProbs, kTopTokens}) {
        if (o.d[k] == nullptr) continue;
        const int64_t n = o.d[k]->shape[lead];
        if (top != 0 && n != top) return fail(MTC_ERR_INVALID_ARGUMENT, "top_log_probs and top_tokens differ in length");
        if (n < 1 || n > kMostTop || n > vocab)
            return fail(MTC_ERR_INVALID_ARGUMENT, "%lld alternatives of %lld classes; 1 to %d are possible",
                        static_cast<long long>(n), static_cast<long long>(vocab), kMostTop);
        top = n;
    }
    IterSpace s;
    s.rank = lead;
    s.nops = kOperands;
    for (int i = 0; i < lead; ++i) {
        s.shape[i] = logits->shape[i];
        s.numel *= logits->shape[i];
        for (int k = 0; k < kOperands; ++k) s.stride[k][i] = o.d[k] != nullptr ? o.d[k]->strides[i] : 0;
    }
    for (int k = 0; k < kOperands; ++k) s.offset[k] = 0;
    a.rows = s.numel;
    a.vocab = static_cast<int>(vocab);
    if (a.rows == 0) return MTC_OK;
    simplify(s);
    a.rank = s.rank;
    for (int i = 0; i < s.rank; ++i) {
        a.shape[i] = s.shape[i];
        for (int k = 0; k < kOperands; ++k) a.stride[k][i] = s.stride[k][i];
    }
    auto f = [&](Operand k) { return o.d[k] != nullptr ? float_at(o.d[k]) : nullptr; };
    auto w = [&](Operand k) { return o.d[k] != nullptr ? static_cast<long long *>(o.d[k]->data) + o.d[k]->offset : nullptr; };
    auto last = [&](Operand k) { return o.d[k] == nullptr ? 0 : o.d[k]->shape[lead] == 1 ? 1 : o.d[k]->strides[lead]; };
    a.logits = f(kLogits);
    a.cs = last(kLogits);
    a.tokens = w(kTokens);
    a.ignore = ignore;
    a.scale = scale;
    a.scale2 = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634);
    a.log_probs = f(kLogProbs);
    a.lse = f(kLse);
    a.entropy = f(kEntropy);
    a.top = static_cast<int>(top);
    a.top_log_probs = f(kTopLogProbs);
    a.top_log_probs_s = last(kTopLogProbs);
    a.top_tokens = w(kTopTokens);
    a.top_tokens_s = last(kTopTokens);
    a.dlog_probs = f(kDLogProbs);
    a.dentropy = f(kDEntropy);
    a.dlogits = f(kDLogits);
    a.dcs = last(kDLogits);
    return MTC_OK;
}

}  // namespace
}  // namespace mtc

using namespace mtc;

extern "C" {

int mtc_token_log_probs(const mtc_desc *logits, const mtc_desc *tokens, float scale, int64_t ignore_token,
                        const mtc_desc *log_probs, const mtc_desc *lse, const mtc_desc *entropy,
                        const mtc_desc *top_log_probs, const mtc_desc *top_tokens, void *stream) {
    clear_error();
    RowOperands o;
    o.d[kLogits] = logits;
    o.d[kTokens] = tokens;
    o.d[kLogProbs] = log_probs;
    o.d[kLse] = lse;
    o.d[kEntropy] = entropy;
    o.d[kTopLogProbs] = top_log_probs;
    o.d[kTopTokens] = top_tokens;
    RowArgs a;
    MTC_TRY(fill_args(o, scale, ignore_token, a));
    if (log_probs != nullptr && tokens == nullptr) return fail(MTC_ERR_INVALID_ARGUMENT, "log_probs without tokens");
    if (a.rows == 0) return MTC_OK;
    MTC_TRY(device_error_word(&a.err));
    return launch<false>(a, static_cast<cudaStream_t>(stream));
}

int mtc_token_log_probs_grad(const mtc_desc *logits, const mtc_desc *tokens, float scale, int64_t ignore_token,
                             const mtc_desc *dlog_probs, const mtc_desc *dentropy, const mtc_desc *dlogits, void *stream) {
    clear_error();
    if (dlogits == nullptr) return fail(MTC_ERR_INVALID_ARGUMENT, "dlogits: null descriptor");
    RowOperands o;
    o.d[kLogits] = logits;
    o.d[kTokens] = tokens;
    o.d[kDLogProbs] = dlog_probs;
    o.d[kDEntropy] = dentropy;
    o.d[kDLogits] = dlogits;
    RowArgs a;
    MTC_TRY(fill_args(o, scale, ignore_token, a));
    if (dlogits->shape[dlogits->rank - 1] != a.vocab)
        return fail(MTC_ERR_INVALID_ARGUMENT, "dlogits differ from the logits in shape");
    if (dlog_probs == nullptr && dentropy == nullptr)
        return fail(MTC_ERR_INVALID_ARGUMENT, "neither dlog_probs nor dentropy is given");
    if (dlog_probs != nullptr && tokens == nullptr) return fail(MTC_ERR_INVALID_ARGUMENT, "dlog_probs without tokens");
    if (a.rows == 0) return MTC_OK;
    MTC_TRY(device_error_word(&a.err));
    return launch<true>(a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
