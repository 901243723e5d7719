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
// what is left (of 129 to 512 classes only where the others come to less than 1/8: see
// k_warp_rows).  The gradient takes its statistics from the row anew instead of from the
// caller: a log-sum-exp rounded to float32 would cost them.
//
// Bound by HBM: 4 bytes an element, and for the gradient 8.  Up to 1024 classes (2048 without
// gradient) a warp holds a row in its registers.  Beyond, a CTA streams it once: a thread keeps
// the maximum of what it has seen and sums relative to it, rescaled where a batch raises the
// maximum.  The gradient reads the row a second time, last elements first, out of L2.  (A cluster a
// row, a thread's elements in registers, was slower: 2^28 logits of 131072 classes 478 us at best
// against 459, of 16000 420 against 379, of 50003 538 against 441: its CTAs wait for one another.)
//
// The k likeliest (k <= 32) need no second pass over the row.  Of 32 groups of threads each has
// a maximum, and the k-th largest of these is a bound that k elements reach; of the others few
// do.  Only what the threads whose maximum reaches it have read is looked at again, and what is
// found is ranked by counting.  Where too many elements are equal for the list, the k-th largest
// of those threads' maxima, told apart by their index, is the next bound; exactly k threads reach
// that one.  Elements that crowd in a few threads overflow the list again and cost k passes over
// the row.
#include <climits>
#include <cmath>
#include <cstring>
#include <exception>
#include <type_traits>

#include "operators.cuh"

namespace mtc {
namespace {

constexpr int kMostTop = 32;
constexpr int kWarps = 8;  // of a CTA that takes a row a warp

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

constexpr float kLn2 = 0.69314718055994531f;
constexpr float kFloor = -200.0f;  // exponents of 2 below it are zeros of float32
// (In sums, what is below 2^-126 of the largest term is one too: exp2_fast flushes it.)

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float exp2_full(float x) {  // with subnormal results
    float y;
    asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float y;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

template <int N>
__device__ __forceinline__ float largest_of(const float (&x)[N]) {
    float y = x[0];
#pragma unroll
    for (int i = 1; i + 1 < N; i += 2) y = max_nan(y, x[i], x[i + 1]);
    return N % 2 == 0 && N > 1 ? max_nan(y, x[N - 1]) : y;
}

// Floats as whole numbers that order as they do: NaN the largest, -0 as 0.
__device__ __forceinline__ int ordered(float x) {
    if (isnan(x)) return INT_MAX;
    const int b = __float_as_int(x + 0.0f);
    return b < 0 ? b ^ INT_MAX : b;
}
constexpr int kNothing = INT_MIN;  // below all of them

__device__ __forceinline__ float from_ordered(int o) { return __int_as_float(o < 0 ? o ^ INT_MAX : o); }

// With the index, the lower the larger: no two are equal, and none is 0 or ~0.
__device__ __forceinline__ unsigned long long key_of(int o, int index) {
    return (static_cast<unsigned long long>(static_cast<unsigned int>(o) ^ 0x80000000u) << 32) |
           static_cast<unsigned int>(INT_MAX - index);
}
__device__ __forceinline__ int key_index(unsigned long long k) { return INT_MAX - static_cast<int>(k); }
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

    // The same where m is at hand already, two elements an instruction where that is possible.
    template <int N>
    __device__ __forceinline__ void add_below(const float (&x)[N], float scale2) {
        if constexpr (N == 1) {
            add(x, m, scale2);
        } else {
            float n1 = 0.0f, r1 = 0.0f;
            float2 es = make_float2(e, 0.0f);
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                float2 u = __fmul2_rn(__fadd2_rn(make_float2(x[i], x[i + 1]), make_float2(-m, -m)), make_float2(scale2, scale2));
                u = make_float2(fmaxf(u.x, kFloor), fmaxf(u.y, kFloor));
                const float2 y = make_float2(exp2_fast(u.x), exp2_fast(u.y));
                if (x[i] == m) n += 1.0f;
                else r += y.x;
                if (x[i + 1] == m) n1 += 1.0f;
                else r1 += y.y;
                es = __ffma2_rn(y, u, es);
            }
            n += n1;
            r += r1;
            e = es.x + es.y;
        }
    }

    // Without a look for m: the sum of all elements from FIRST on, by halves, so that a 1 among
    // them is rounded log2 N times at the most, and theirs of u 2^u.
    template <int FIRST, int COUNT, int N>
    __device__ __forceinline__ float sum_all(const float (&x)[N], float scale2, float (&es)[2]) const {
        if constexpr (COUNT == 1) {
            const float u = fmaxf((x[FIRST] - m) * scale2, kFloor), y = exp2_fast(u);
            es[FIRST % 2] = fmaf(y, u, es[FIRST % 2]);
            return y;
        } else {
            const float half = sum_all<FIRST, COUNT / 2>(x, scale2, es);
            return half + sum_all<FIRST + COUNT / 2, COUNT - COUNT / 2>(x, scale2, es);
        }
    }

    // Of a warp's lanes together, the same in all.
    __device__ __forceinline__ void join_warp(float scale2) {
        bad = __any_sync(0xFFFFFFFFu, bad);
        const float top = from_ordered(__reduce_max_sync(0xFFFFFFFFu, ordered(m)));
        if (top > m) rise(top, scale2);
        sum_warp();
    }
    __device__ __forceinline__ void sum_warp() {
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
        m = s.m;
        others = s.n - 1.0f + s.r;
        total = s.n + s.r;
        log_total = log1pf(others);
        spread = -kLn2 * s.e / total;
        bad = s.bad;
        empty = s.n == 0.0f;
    }
    __device__ __forceinline__ float log_prob(float x, float scale) const {
        if (bad) return __int_as_float(0x7FC00000);
        if (empty) return -INFINITY;
        return fmaf(0.5f, x, -0.5f * m) * (2.0f * scale) - log_total;  // (x - m may be beyond float32)
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

// The row's token as it is: loaded a row ahead, so that nothing waits for it.
__device__ __forceinline__ long long token_at(const RowArgs &a, int64_t row) {
    return a.tokens != nullptr && row < a.rows ? a.tokens[at(a, kTokens, row)] : 0;
}

// Its index, or -1 without tokens; false: the row is not scored.
__device__ __forceinline__ bool token_of(const RowArgs &a, long long t, bool report, int &token) {
    token = -1;
    if (a.tokens == nullptr) return true;
    if (t == a.ignore) return false;
    if (t < 0 || t >= a.vocab) {
        if (report) report_index(a.err, t);
        return false;
    }
    token = static_cast<int>(t);
    return true;
}

// The gradient of a row: -p (by_entropy u + shift) with d = u ln 2 and shift = by_prob + own, and
// of the token's element apart: the entropy's part of it by `own`, which a rounded shift does
// not give back where it is little next to by_prob.
struct Slope {
    float m, scale2, by_entropy, shift, inverse, by_prob, own, others;
    bool whole;  // else every element is `fill`
    float fill;

    __device__ __forceinline__ Slope(const RowArgs &a, int64_t row, const Row &s) {
        m = s.m;
        asm volatile("" : "+f"(m));  // or the sums' exponents are kept for it, in memory
        scale2 = a.scale2;
        by_prob = a.dlog_probs != nullptr ? a.dlog_probs[at(a, kDLogProbs, row)] * a.scale : 0.0f;
        by_entropy = a.dentropy != nullptr ? a.dentropy[at(a, kDEntropy, row)] * a.scale : 0.0f;
        own = by_entropy * s.spread;
        shift = fmaf(by_entropy, s.spread, by_prob);
        by_entropy *= kLn2;
        inverse = 1.0f / s.total;
        others = s.others;
        whole = !s.bad && !s.empty;
        fill = s.bad ? __int_as_float(0x7FC00000) : 0.0f;
    }
    __device__ __forceinline__ float operator()(float x) const {
        const float u = fmaxf((x - m) * scale2, kFloor);
        return -(exp2_full(u) * inverse) * fmaf(by_entropy, u, shift);
    }
    __device__ __forceinline__ float of_token(float x) const {
        const float u = fmaxf((x - m) * scale2, kFloor), p = exp2_full(u) * inverse;
        return by_prob * (x == m ? others * inverse : 1.0f - p) - p * fmaf(by_entropy, u, own);
    }
};

// ------------------------------------------------------------ a warp a row --

// The k-th largest of the lanes' values.
__device__ __forceinline__ int kth_of_warp(int v, int k) {
    const int lane = threadIdx.x % 32;
    if (k <= 8) {  // the largest taken away one by one: fewer instructions than to sort
        int top = v;
        for (int i = 0; i < k; ++i) {
            top = __reduce_max_sync(0xFFFFFFFFu, v);
            const unsigned int at = __ballot_sync(0xFFFFFFFFu, v == top);
            if (lane == __ffs(at) - 1) v = kNothing;
        }
        return top;
    }
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int o = size / 2; o > 0; o >>= 1) {
            const int w = __shfl_xor_sync(0xFFFFFFFFu, v, o);
            const bool larger = ((lane & o) == 0) == ((lane & size) == 0);
            v = larger ? max(v, w) : min(v, w);
        }
    return __shfl_sync(0xFFFFFFFFu, v, k - 1);
}

__device__ __forceinline__ unsigned long long warp_max(unsigned long long k) {
    const unsigned int hi = __reduce_max_sync(0xFFFFFFFFu, static_cast<unsigned int>(k >> 32));
    const unsigned int lo =
        __reduce_max_sync(0xFFFFFFFFu, static_cast<unsigned int>(k >> 32) == hi ? static_cast<unsigned int>(k) : 0u);
    return (static_cast<unsigned long long>(hi) << 32) | lo;
}

constexpr int kWarpList = 64;

// R elements a lane: the 32 lanes side by side, or in vectors of four, 32 vectors side by side.
// Which of the two goes by the number of classes (next to each other), so that a row's sums, and
// with them its bits, do not depend on what the other rows lie on: kFours are vectors that some or
// all rows cannot load as such.  (2^28 logits of 1000 classes, rows 1002 apart, 220 us, all off 16
// bytes 237, their gradients 507 and 501; with the lanes side by side 218 and 217, 583 and 587.)
enum Lanes { kApart, kUnit, kFours, kVectors };

template <int R, Lanes LANES, bool GRAD>
__global__ void __launch_bounds__(32 * kWarps, R >= 64 ? 2 : R >= 32 ? 3 : 4) k_warp_rows(const RowArgs a) {
    __shared__ unsigned long long lists[kWarps][kWarpList];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kWarps;
    int64_t row = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
    long long next = token_at(a, row);
    for (; row < a.rows; row += step) {
        const long long given = next;
        next = token_at(a, row + step);
        int token;
        if (!token_of(a, given, lane == 0, token)) {
            write_skipped(a, row, lane, 32);
            continue;
        }
        const float *src = a.logits + at(a, kLogits, row);
        const int64_t cs = LANES != kApart ? 1 : a.cs;
        constexpr bool FOURS = LANES >= kFours;
        auto index = [&](int j) { return FOURS ? 4 * (lane + 32 * (j / 4)) + j % 4 : lane + 32 * j; };
        float x[R];
        if (LANES == kVectors || (LANES == kFours && reinterpret_cast<uintptr_t>(src) % 16 == 0)) {
#pragma unroll
            for (int j = 0; j < R; j += 4) {
                float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                if (index(j) < a.vocab) v = *reinterpret_cast<const float4 *>(src + index(j));
                x[j] = v.x;
                x[j + 1 < R ? j + 1 : j] = v.y;
                x[j + 2 < R ? j + 2 : j] = v.z;
                x[j + 3 < R ? j + 3 : j] = v.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < R; ++j) x[j] = index(j) < a.vocab ? src[index(j) * cs] : -INFINITY;
        }
        const float largest = largest_of(x);
        const int mine = index(0) < a.vocab ? ordered(largest) : kNothing;
        const int most = __reduce_max_sync(0xFFFFFFFFu, mine);
        const float top = from_ordered(most);
        Stats st;
        if (!(top < INFINITY)) {
            st.bad = true;
        } else if (top > -INFINITY) {
            st.m = top;
            if constexpr (R != 16) {
                st.add_below(x, a.scale2);
                st.sum_warp();
            } else {
                // Without a look at each element for the largest (2^28 logits of 200 classes 625 us, with it 680;
                // of 500 268 and 294; but of 1000 236 and 205, of 2000 227 and 187): a lane that has it takes its 1
                // out again before the lanes' sums are added.  Until then it costs the others up to log2 R = 4
                // roundings of a sum above 1, which is 36 2^-24 of them where they are 1/8 of it.  Where they are
                // less, they are added without it (rows sure of their class: 778 us of 200, 322 of 500).
                float es[2] = {};
                st.r = st.sum_all<0, R>(x, a.scale2, es);
                st.e = es[0] + es[1];
                if (lane == __ffs(__ballot_sync(0xFFFFFFFFu, mine == most)) - 1) st.r -= 1.0f;
                st.n = lane == 0 ? 1.0f : 0.0f;
                st.sum_warp();
                if (st.r < 0.125f) {
                    st = Stats();
                    st.m = top;
                    st.add_below(x, a.scale2);
                    st.sum_warp();
                }
            }
        }
        const Row s(st);
        if (GRAD) {
            const Slope slope(a, row, s);
            float *to = a.dlogits + at(a, kDLogits, row);
            auto of = [&](int j) { return !slope.whole ? slope.fill : index(j) == token ? slope.of_token(x[j]) : slope(x[j]); };
            if (FOURS && a.dcs == 1 && reinterpret_cast<uintptr_t>(to) % 16 == 0) {
#pragma unroll
                for (int j = 0; j < R; j += 4)
                    if (index(j) < a.vocab)
                        __stcs(reinterpret_cast<float4 *>(to + index(j)), make_float4(of(j), of(j + 1 < R ? j + 1 : j),
                                                                                      of(j + 2 < R ? j + 2 : j), of(j + 3 < R ? j + 3 : j)));
            } else {
#pragma unroll
                for (int j = 0; j < R; ++j)
                    if (index(j) < a.vocab) to[index(j) * a.dcs] = of(j);
            }
            continue;
        }
        if (lane == 0) write_row(a, row, s, token >= 0 ? src[token * a.cs] : 0.0f);
        if (a.top == 0) continue;
        // the k-th largest of the lanes' maxima: k elements reach it
        const float bound = from_ordered(kth_of_warp(mine, a.top));
        using Hits = typename std::conditional<(R > 32), unsigned long long, unsigned int>::type;
        unsigned long long *list = lists[warp];
        Hits hits = 0;
#pragma unroll
        for (int j = 0; j < R; ++j) hits |= static_cast<Hits>(x[j] >= bound ? 1 : 0) << j;
        if (index(R - 1) >= a.vocab) {  // (what is no element)
            const int n = FOURS ? 4 * ((a.vocab / 4 - lane + 31) / 32) : (a.vocab - lane + 31) / 32;
            hits &= (static_cast<Hits>(1) << n) - 1;
        }
        int found = __reduce_add_sync(0xFFFFFFFFu, R > 32 ? __popcll(hits) : __popc(hits));
        if (found < a.top || s.bad) found = kWarpList + 1;  // NaN, or fewer lanes than k have an element
        if (found <= kWarpList) {
            int base = 0;
            for (;; hits &= hits - 1) {
                const unsigned int any = __ballot_sync(0xFFFFFFFFu, hits != 0);
                if (any == 0) break;
                if (hits != 0) {
                    const int v = index((R > 32 ? __ffsll(hits) : __ffs(hits)) - 1);
                    list[base + __popc(any & ((1u << lane) - 1))] = key_of(ordered(src[v * cs]), v);
                }
                base += __popc(any);
            }
            __syncwarp();
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
                const unsigned long long k = index(j) < a.vocab ? key_of(ordered(x[j]), index(j)) : 0;
                if (k < last && k > best) best = k;
            }
            last = warp_max(best);
            if (lane == 0) write_top(a, row, s, rank, last);
        }
    }
}

// ------------------------------------------------------------- a CTA a row --

constexpr int kBatch = 8;      // vectors of four that a thread has in flight
constexpr int kAgain = 2;      // and the second time (one: 131072 classes 501 us, two 458, four 447; 50003: 480, 462, 480)
constexpr int kList = 512;
constexpr int kThreadsOfSm = 1024;  // 64 registers each

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

// A thread's vectors of a batch: j, j + step, ...
template <bool VEC>
__device__ __forceinline__ void read_batch(const Source<VEC> &src, int j, int step, float (&x)[4 * kBatch]) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
        const float4 v = j + step * u < src.vecs ? src.vec(j + step * u) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        x[4 * u] = v.x;
        x[4 * u + 1] = v.y;
        x[4 * u + 2] = v.z;
        x[4 * u + 3] = v.w;
    }
}

template <int T>
__device__ __forceinline__ void join_block(Stats &s, float scale2, float4 *parts) {
    static_assert(T >= 32 && T <= 1024, "warps");
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

template <int T>
struct TopShared {
    int group[32];
    int found, listed;
    unsigned long long bound;
    unsigned long long maxima[T];
    unsigned long long list[kList];
    unsigned long long warps[32];
};

// The k likeliest, see above.  `best` is this thread's largest element, first seen in batch
// `where` (kHead, kTail: before and behind the vectors).
constexpr int kHead = -1, kTail = -2;

template <int T, bool VEC>
__device__ __forceinline__ void find_top(const RowArgs &a, int64_t row, const Source<VEC> &src, const Row &s, int best,
                                         int where, TopShared<T> &sh) {
    constexpr int G = T / 32;
    const int thread = threadIdx.x, lane = thread % 32;
    int m = best;
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    if (thread % G == 0) sh.group[thread / G] = m;
    if (thread == 0) sh.found = sh.listed = 0;
    __syncthreads();
    const int first = kth_of_warp(sh.group[lane], a.top);
    // What the threads that reach it have read, and is as large: some 2 k elements, unless many
    // are equal or crowd.
    const bool reaches = best >= first;
    auto scan = [&](bool mine, auto &&look) {
        for (unsigned int of = __ballot_sync(0xFFFFFFFFu, mine); of != 0;) {
            int of_thread[2];  // (T: none)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                of_thread[q] = of != 0 ? thread - lane + __ffs(of) - 1 : T;
                of &= of - 1;
            }
            for (int at = T * lane; at < src.vecs; at += T * 32) {
                float4 v[2];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    v[q] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                    if (of_thread[q] < T && at + of_thread[q] < src.vecs) v[q] = src.vec(at + of_thread[q]);
                }
#pragma unroll
                for (int q = 0; q < 2; ++q)
                    if (of_thread[q] < T && at + of_thread[q] < src.vecs) look(v[q], src.head + 4 * (at + of_thread[q]), 4);
            }
            if (lane < 2) {
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const int v = lane == 0 ? of_thread[q] : src.tail_at() + of_thread[q];
                    if (of_thread[q] < (lane == 0 ? src.head : src.tail)) look(make_float4(src.one(v), 0.0f, 0.0f, 0.0f), v, 1);
                }
            }
        }
    };
    auto list = [&](unsigned long long k) {
        const int to = atomicAdd(&sh.listed, 1);
        if (to < kList) sh.list[to] = k;
    };
    auto rank_list = [&](int n) {
        for (int i = thread; i < n; i += T) {
            const unsigned long long k = sh.list[i];
            int rank = 0;
#pragma unroll 4
            for (int j = 0; j < n; ++j) rank += sh.list[j] > k;
            if (rank < a.top) write_top(a, row, s, rank, k);
        }
    };
    const float least = from_ordered(first);
    if (!s.bad && least > -INFINITY) {
        scan(reaches, [&](const float4 &v, int i, int n) {
            const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (k < n && x[k] >= least && sh.listed < kList) list(key_of(ordered(x[k]), i + k));
        });
        __syncthreads();
        if (sh.listed < kList) {
            rank_list(sh.listed);
            return;
        }
        __syncthreads();
        if (thread == 0) sh.listed = 0;
    }
    unsigned long long mine = 0;
    if (reaches) {
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
    scan(mine >= bound, [&](const float4 &v, int i, int n) {
        const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const unsigned long long key = key_of(ordered(x[k]), i + k);
            if (k < n && key >= bound) list(key);
        }
    });
    __syncthreads();
    if (sh.listed <= kList) {
        rank_list(sh.listed);
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
__global__ void __launch_bounds__(T, kThreadsOfSm / T) k_cta_rows(const RowArgs a) {
    __shared__ float4 parts[32];
    __shared__ TopShared<T> sh;
    const int thread = threadIdx.x;
    long long next = token_at(a, blockIdx.x);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const long long given = next;
        next = token_at(a, row + gridDim.x);
        int token;
        if (!token_of(a, given, thread == 0, token)) {
            write_skipped(a, row, thread, T);
            continue;
        }
        const Source<VEC> src(a, row);
        const float x_token = token >= 0 ? src.one(token) : 0.0f;
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
            read_batch(src, thread + T * kBatch * b, T, x);
            const float largest = largest_of(x);
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
        if (!GRAD) {
            if (thread == 0) write_row(a, row, s, x_token);
            if (a.top > 0) find_top<T, VEC>(a, row, src, s, best, where, sh);
            __syncthreads();
            continue;
        }
        const Slope slope(a, row, s);
        float *to = a.dlogits + at(a, kDLogits, row);
        if (!slope.whole) {
            for (int v = thread; v < a.vocab; v += T) to[v * a.dcs] = slope.fill;
            __syncthreads();
            continue;
        }
        const bool whole = VEC && a.dcs == 1 && ((reinterpret_cast<uintptr_t>(to) ^ reinterpret_cast<uintptr_t>(src.p)) & 15) == 0;
        for (int b = batches * (kBatch / kAgain) - 1; b >= 0; --b) {
            float4 x[kAgain];
#pragma unroll
            for (int u = 0; u < kAgain; ++u) {
                const int j = thread + T * (b * kAgain + u);
                x[u] = src.vec(j < src.vecs ? j : src.vecs - 1);
            }
#pragma unroll
            for (int u = 0; u < kAgain; ++u) {
                const int j = thread + T * (b * kAgain + u);
                if (j >= src.vecs) continue;
                const int i = src.head + 4 * j;
                const float4 g = make_float4(slope(x[u].x), slope(x[u].y), slope(x[u].z), slope(x[u].w));
                if (whole) {
                    __stcs(reinterpret_cast<float4 *>(to + i), g);
                } else {
                    to[i * a.dcs] = g.x;
                    to[(i + 1) * a.dcs] = g.y;
                    to[(i + 2) * a.dcs] = g.z;
                    to[(i + 3) * a.dcs] = g.w;
                }
            }
        }
        if (thread < src.head) to[thread * a.dcs] = slope(src.one(thread));
        if (thread < src.tail) {
            const int i = src.tail_at() + thread;
            to[i * a.dcs] = slope(src.one(i));
        }
        if (token >= 0) {  // by the thread that has just written it
            const int j = token - src.head;
            const int owner = j < 0 ? token : token >= src.tail_at() ? token - src.tail_at() : j / 4 % T;
            if (thread == owner) to[token * a.dcs] = slope.of_token(x_token);
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------- host --

template <int R, bool GRAD>
int launch_warps(const RowArgs &a, cudaStream_t stream) {
    const int64_t ctas = (a.rows + kWarps - 1) / (kWarps), most = static_cast<int64_t>(sm_count(current_device())) * 64;
    const unsigned grid = static_cast<unsigned>(ctas < most ? ctas : most);
    // (by the logits alone: the same logits give the same bits, wherever the gradient goes)
    const bool fours = R >= 4 && a.cs == 1 && a.vocab % 4 == 0;
    bool alike = true;  // in alignment
    for (int i = 0; i < a.rank; ++i) alike = alike && a.stride[kLogits][i] % 4 == 0;
    if (fours && alike && aligned16(a.logits)) k_warp_rows<R, R >= 4 ? kVectors : kUnit, GRAD><<<grid, 32 * kWarps, 0, stream>>>(a);
    else if (fours) k_warp_rows<R, R >= 4 ? kFours : kUnit, GRAD><<<grid, 32 * kWarps, 0, stream>>>(a);
    else if (a.cs == 1) k_warp_rows<R, kUnit, GRAD><<<grid, 32 * kWarps, 0, stream>>>(a);
    else k_warp_rows<R, kApart, GRAD><<<grid, 32 * kWarps, 0, stream>>>(a);
    return check_launch("log probabilities (warps)");
}

template <int T, bool GRAD>
int launch_ctas(const RowArgs &a, cudaStream_t stream) {
    const int64_t most = static_cast<int64_t>(sm_count(current_device())) * (kThreadsOfSm / T) * 8;
    const unsigned grid = static_cast<unsigned>(std::min(a.rows, most));
    if (a.cs == 1) k_cta_rows<T, true, GRAD><<<grid, T, 0, stream>>>(a);
    else k_cta_rows<T, false, GRAD><<<grid, T, 0, stream>>>(a);
    return check_launch("log probabilities");
}

// The number of threads goes by the classes alone, so that a row's results are the same to the
// bit whatever other rows the call has.  (For few rows more would be a little faster: of 32000
// classes one row with 20 alternatives takes 12.4 us by 512 threads and 15.4 by 256.)
// Times of 2^28 logits, without alternatives, with 5 and with 20:
//   1500 classes  64 elements a lane 226, 363, 466 us;  a CTA of 32 238, 432, 811
//   3000          CTAs of 32 211, 297, 525;  of 64 223, 367, 617
//   8000          of 64 162, 205, 310;  of 128 177, 250, 377
//   16000         of 128 164, 193, 261;  of 256 183, 242, 326
//   32000         of 256 164, 189, 236;  of 128 164, 193, 279;  of 512 193, 247, 305
//   131072        of 512 162, 183, 213;  of 256 168, 193, 273
int launch_forward(const RowArgs &a, cudaStream_t stream) {
    if (a.vocab <= 32) return launch_warps<1, false>(a, stream);
    if (a.vocab <= 128) return launch_warps<4, false>(a, stream);
    if (a.vocab <= 512) return launch_warps<16, false>(a, stream);
    if (a.vocab <= 1024) return launch_warps<32, false>(a, stream);
    if (a.vocab <= 2048) return launch_warps<64, false>(a, stream);
    if (a.vocab <= 4000) return launch_ctas<32, false>(a, stream);
    if (a.vocab <= 12000) return launch_ctas<64, false>(a, stream);
    if (a.vocab <= 24000) return launch_ctas<128, false>(a, stream);
    if (a.vocab <= 100000) return launch_ctas<256, false>(a, stream);
    return launch_ctas<512, false>(a, stream);
}

// Some 64 elements a thread, two batches, so that the rows at work are few enough for L2 (126 MB,
// half of which is another die's) when they are read again.  2^28 logits:
//   1500 classes  CTAs of 32 410 us;  64 elements a lane of a warp 561
//   4000          of 64 371;  of 32 418
//   8000          of 128 371;  of 64 412, of 256 439
//   16000         of 256 379;  of 128 420, of 512 453
//   24000         of 256 398;  of 512 447
//   32000         of 512 392;  of 256 418
//   50003         of 512 441;  of 1024 463
//   65536         of 1024 414;  of 512 426
//   131072        of 1024 459;  of 512 483
int launch_gradient(const RowArgs &a, cudaStream_t stream) {
    if (a.vocab <= 32) return launch_warps<1, true>(a, stream);
    if (a.vocab <= 128) return launch_warps<4, true>(a, stream);
    if (a.vocab <= 512) return launch_warps<16, true>(a, stream);
    if (a.vocab <= 1024) return launch_warps<32, true>(a, stream);
    if (a.vocab <= 3500) return launch_ctas<32, true>(a, stream);
    if (a.vocab <= 6000) return launch_ctas<64, true>(a, stream);
    if (a.vocab <= 12000) return launch_ctas<128, true>(a, stream);
    if (a.vocab <= 24000) return launch_ctas<256, true>(a, stream);
    if (a.vocab <= 56000) return launch_ctas<512, true>(a, stream);
    return launch_ctas<1024, true>(a, stream);
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
    // (below it, differences beyond float32 would be more than nothing in the sums)
    if (!(scale >= 0x1p-100f && scale <= 0x1p100f))
        return fail(MTC_ERR_INVALID_ARGUMENT, "scale %g is not in [2^-100, 2^100]", scale);
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
    return launch_forward(a, static_cast<cudaStream_t>(stream));
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
    return launch_gradient(a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
