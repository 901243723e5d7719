// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   out[i, :] = scale * table[tok_i, :]            dtable[v, :] = scale * sum_{i: tok_i = v} dout[i, :]
//
// The lookup reads each row once and writes 4 D bytes a position: bound by HBM
// for many positions (4099 of 4096 columns in 20.6 us, where 100 MB take 15.4 us; 16384 of
// 2048 in 35.6 us), by the launch for few.
//
// The gradient reads every dout row once and writes every table row once.
// Atomics would add the rows of a frequent token one after the other at one
// address, in an order that changes from run to run; a walk by token leaves a
// token of a natural text (a few own thousands of positions, most own none) to
// one CTA.  So the positions are sorted by token (stable, so ascending within a
// token), and the sorted list is cut into pieces of 32 positions, whatever the
// tokens: one CTA adds a piece's runs in registers, writes the rows whose run
// lies inside the piece, and leaves the run that came in from the piece before
// and the one that goes on into the next as partial rows.  The last piece of a run
// to finish adds its partial rows, in the order of the pieces: which sums are formed
// depends on the tokens alone.  Rows without a position are cleared by further CTAs
// of the same launch, 32 rows a bit mask.  16384 positions into 32000 x 1024 take 55 us: 15.5
// for the sort, the sums at 5.2 TB/s, the launches; 65536 into 131072 x 2048 266 us, 29.5 for the
// sort and the sums at 6.4 TB/s.
#include <cooperative_groups.h>

#include <climits>
#include <cstring>

#include "operators.cuh"

namespace mtc {
namespace {

constexpr int kThreads = 256;

// The positions: a token view of any rank next to rows of a float view.
struct Positions {
    long long n;
    int rank;  // after folding; 1 in most calls
    long long shape[MTC_MAX_RANK];
    long long tok_stride[MTC_MAX_RANK], row_stride[MTC_MAX_RANK];
    const long long *tokens;
};

__device__ __forceinline__ long long token_at(const Positions &p, long long i, long long &row) {
    if (p.rank == 1) {
        row = i * p.row_stride[0];
        return p.tokens[i * p.tok_stride[0]];
    }
    long long t = 0;
    row = 0;
    for (int a = p.rank - 1; a >= 0; --a) {
        const long long q = i / p.shape[a], c = i - q * p.shape[a];
        t += c * p.tok_stride[a];
        row += c * p.row_stride[a];
        i = q;
    }
    return p.tokens[t];
}

struct LookupArgs {
    Positions pos;
    int lanes_log2;      // lanes that share a segment of a row
    unsigned int segments;  // of a row, each kLookupLoads vectors a lane
    long long groups;    // positions x segments
    long long vectors;   // of a row
    const float *table;
    float *out;
    long long table_rs, table_cs, out_cs;
    long long vocab;
    long long padding;
    float scale;
    unsigned long long *err;
};

constexpr int kLookupLoads = 4;

// 2^lanes_log2 lanes take a segment of a row, one token for all of their four loads, and
// fetch the token of their next segment before they wait for the row of this one.
template <int VEC>
__global__ void __launch_bounds__(kThreads) k_embedding(const LookupArgs a) {
    constexpr int U = kLookupLoads;
    const int lanes = 1 << a.lanes_log2;
    const unsigned int thread = blockIdx.x * kThreads + threadIdx.x;
    const int lane = static_cast<int>(thread) & (lanes - 1);
    const long long stride = static_cast<long long>(gridDim.x) * kThreads >> a.lanes_log2;
    long long g = thread >> a.lanes_log2;
    if (g >= a.groups) return;
    long long i = a.segments == 1 ? g : g / a.segments;
    long long row;
    long long t = token_at(a.pos, i, row);
    while (true) {
        const long long c0 = (g - i * a.segments) * (lanes * U) + lane;
        float *dst = a.out + row + c0 * VEC * a.out_cs;
        const bool zero = t == a.padding, valid = t >= 0 && t < a.vocab;
        if (!zero && !valid && c0 == 0) report_index(a.err, t);
        const float *src = a.table + (valid ? t : 0) * a.table_rs + c0 * VEC * a.table_cs;
        float4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            v[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (!valid || zero || c0 + u * lanes >= a.vectors) continue;
            if (VEC == 4) v[u] = __ldg(reinterpret_cast<const float4 *>(src) + u * lanes);
            else v[u].x = __ldg(src + u * lanes * a.table_cs);
        }
        const long long next = g + stride;
        if (next < a.groups) {
            i = a.segments == 1 ? next : next / a.segments;
            t = token_at(a.pos, i, row);
        }
        if (valid || zero) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (c0 + u * lanes >= a.vectors) continue;
                if (VEC == 4)
                    __stcs(reinterpret_cast<float4 *>(dst) + u * lanes,
                           make_float4(v[u].x * a.scale, v[u].y * a.scale, v[u].z * a.scale, v[u].w * a.scale));
                else
                    dst[u * lanes * a.out_cs] = v[u].x * a.scale;
            }
        }
        if (next >= a.groups) return;
        g = next;
    }
}

// ---------------------------------------------------------------- the sort --
// Least-significant-digit radix sort of (token, position), stable.  A key of a
// position without a gradient is V, the largest.  A warp owns consecutive keys
// and ranks them 32 at a time by ballots, so equal digits keep their order;
// a key goes behind the smaller digits, the equal ones of the warps and CTAs
// before, and its rank.
//
// Up to 2048 positions are ranked instead (k_sort_rank).  Up to 65536 are sorted by one
// cluster of up to 16 CTAs in one launch, the keys in shared memory, counts read and keys
// sent over distributed shared memory.
// More positions take two launches a pass (three with many tiles).

constexpr int kTile = 4096;
constexpr int kMaxBins = 1024;
constexpr int kClusterTiles = 16;  // CTAs of the largest cluster
constexpr int kClusterBins = 512;
constexpr int kClusterThreads = 1024;

struct SortArgs {
    Positions pos;
    long long vocab, padding;
    unsigned int n;
    int shift, bits, passes;
    int tiles;
    int last;                     // this launch writes the sorted list
    const uint2 *in;        // (token, position); null: read the tokens
    uint2 *out;
    unsigned int *counts;   // [tiles][bins]
    unsigned int *before;   // [tiles][bins] sums over the tiles before, and [bins] totals behind them; null: few tiles
    unsigned int *present;  // a bit for each table row that has a position; null: not wanted
    unsigned int *arrived;  // counters of the sums, to be zeroed
    unsigned int n_arrived;
    unsigned long long *err;
};

// Keys of N indices of a thread, the loads all in flight at once.
template <int N, class Index>
__device__ __forceinline__ void load_keys(const SortArgs &a, unsigned int (&key)[N], unsigned int (&at)[N], Index index,
                                          bool report) {
    if (a.in != nullptr) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint2 x = index(j) < a.n ? a.in[index(j)] : make_uint2(0, 0);
            key[j] = x.x;
            at[j] = x.y;
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) at[j] = index(j);
    long long t[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        long long row;
        t[j] = index(j) < a.n ? token_at(a.pos, index(j), row) : 0;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
        key[j] = static_cast<unsigned int>(t[j]);
        if (t[j] == a.padding) {
            key[j] = static_cast<unsigned int>(a.vocab);
        } else if (t[j] < 0 || t[j] >= a.vocab) {
            if (report) report_index(a.err, t[j]);
            key[j] = static_cast<unsigned int>(a.vocab);
        }
    }
}

// What the sort's launches and the sums count in, zeroed by the first of them.
__device__ __forceinline__ void clear_flags(const SortArgs &a, unsigned int thread, unsigned int threads) {
    if (a.present != nullptr)
        for (long long i = thread; i < (a.vocab + 31) / 32; i += threads) a.present[i] = 0;
    for (unsigned int i = thread; i < a.n_arrived; i += threads) a.arrived[i] = 0;
}

// Sets the bits of N keys' rows; a frequent token's word is read before it is written
// to, so that its thousands of positions do not queue at one address.
template <int N, class Live>
__device__ __forceinline__ void mark_present(const SortArgs &a, const unsigned int (&key)[N], Live live) {
    if (a.present == nullptr) return;
    unsigned int word[N];
#pragma unroll
    for (int j = 0; j < N; ++j) word[j] = live(j) && key[j] < a.vocab ? __ldcg(a.present + key[j] / 32) : 0xFFFFFFFFu;
#pragma unroll
    for (int j = 0; j < N; ++j)
        if (!(word[j] >> (key[j] % 32) & 1)) atomicOr(&a.present[key[j] / 32], 1u << (key[j] % 32));
}

// Exclusive sum over the CTA of one value a thread.
__device__ __forceinline__ unsigned int block_exclusive(unsigned int v, unsigned int *warp_sums) {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    unsigned int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned int y = __shfl_up_sync(0xFFFFFFFFu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    const unsigned int mine = lane < warp ? warp_sums[lane] : 0;
    return __reduce_add_sync(0xFFFFFFFFu, mine) + x - v;
}

// Ranks of a warp's keys among the equal digits of its keys before: seen[d] counts them.
// The lanes with an equal digit come from one ballot a bit.
template <int N, class Live>
__device__ __forceinline__ void rank_keys(const unsigned int (&key)[N], unsigned short (&rank)[N], Live live, int shift,
                                          int bits, unsigned short *seen) {
    const int lane = threadIdx.x % 32;
    unsigned int same[N];
#pragma unroll
    for (int j = 0; j < N; ++j) same[j] = __ballot_sync(0xFFFFFFFFu, live(j));
    for (int b = 0; b < bits; ++b) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const bool one = (key[j] >> (shift + b)) & 1;
            const unsigned int ones = __ballot_sync(0xFFFFFFFFu, one);
            same[j] &= one ? ones : ~ones;
        }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const unsigned int d = (key[j] >> shift) & ((1u << bits) - 1);
        rank[j] = 0;
        if (live(j)) rank[j] = seen[d] + __popc(same[j] & ((1u << lane) - 1));
        __syncwarp();
        if (live(j) && (same[j] >> lane) == 1u) seen[d] = rank[j] + 1;  // the last of the equal lanes
        __syncwarp();
    }
}

struct ClusterSort {
    uint2 key[kTile];  // (token, position)
    unsigned short seen[kClusterThreads / 32][kClusterBins];
    unsigned int count[kClusterBins], place[kClusterBins];
    unsigned int warp_sums[32];
};

// N keys a thread, 1024 N a CTA: a scatter costs a clock a key of its SM's, so the keys
// are spread over as many CTAs as a cluster has.
template <int N>
__global__ void __launch_bounds__(kClusterThreads, 1) k_sort_cluster(const SortArgs a) {
    extern __shared__ __align__(16) unsigned char raw[];
    ClusterSort &s = *reinterpret_cast<ClusterSort *>(raw);
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const unsigned int me = cluster.block_rank(), ctas = cluster.num_blocks();
    constexpr int kKeys = kClusterThreads * N;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int bins = 1 << a.bits;
    const unsigned int first = me * kKeys + warp * (32 * N) + lane;
    auto index = [&](int j) { return first + j * 32; };
    auto live = [&](int j) { return index(j) < a.n; };
    clear_flags(a, me * kClusterThreads + threadIdx.x, ctas * kClusterThreads);
    unsigned int key[N], at[N];
    load_keys<N>(a, key, at, index, true);
    for (int pass = 0; pass < a.passes; ++pass) {
        const int shift = pass * a.bits;
        if (pass > 0) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const uint2 x = s.key[warp * (32 * N) + j * 32 + lane];
                key[j] = x.x;
                at[j] = x.y;
            }
        }
        for (int i = threadIdx.x; i < static_cast<int>(sizeof(s.seen) / 4); i += kClusterThreads)
            reinterpret_cast<unsigned int *>(s.seen)[i] = 0;
        __syncthreads();
        unsigned short rank[N];
        rank_keys<N>(key, rank, live, shift, a.bits, s.seen[warp]);
        __syncthreads();
        if (static_cast<int>(threadIdx.x) < bins) {
            unsigned short c[kClusterThreads / 32];
#pragma unroll
            for (int w = 0; w < kClusterThreads / 32; ++w) c[w] = s.seen[w][threadIdx.x];
            unsigned int sum = 0;
#pragma unroll
            for (int w = 0; w < kClusterThreads / 32; ++w) {
                s.seen[w][threadIdx.x] = static_cast<unsigned short>(sum);
                sum += c[w];
            }
            s.count[threadIdx.x] = sum;
        }
        cluster.sync();  // every CTA's counts, and its reading of the keys it had
        unsigned int total = 0, before = 0;
        if (static_cast<int>(threadIdx.x) < bins) {
            unsigned int c[kClusterTiles];
#pragma unroll
            for (unsigned int r = 0; r < kClusterTiles; ++r)
                c[r] = r < ctas ? cluster.map_shared_rank(s.count, r)[threadIdx.x] : 0;
#pragma unroll
            for (unsigned int r = 0; r < kClusterTiles; ++r) {
                if (r < me) before += c[r];
                total += c[r];
            }
        }
        const unsigned int base = block_exclusive(total, s.warp_sums);
        if (static_cast<int>(threadIdx.x) < bins) s.place[threadIdx.x] = base + before;
        __syncthreads();
        const bool last = pass == a.passes - 1;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (!live(j)) continue;
            const unsigned int d = (key[j] >> shift) & (bins - 1);
            const unsigned int to = s.place[d] + s.seen[warp][d] + rank[j];
            if (last) a.out[to] = make_uint2(key[j], at[j]);
            else cluster.map_shared_rank(s.key, to / kKeys)[to % kKeys] = make_uint2(key[j], at[j]);
        }
        if (last) mark_present<N>(a, key, live);
        cluster.sync();  // the keys have arrived, and nobody reads the counts any more
    }
}

// Up to 2048 positions: a position's place is the number of keys below its own, and of equal ones
// before it, which a CTA counts for 64 of them, 16 lanes each; every CTA reads all tokens, none
// waits for another.  The bits of the table's rows come from the same keys, a part of the rows a CTA.
// (The whole gradient, 131072 rows of 64 columns: 512 positions 21.0 us by the cluster, 16.8 so; 2048
// 23.0 and 20.9; 4096 25.1 and 28.2, the comparisons growing with the square.)
constexpr int kRankPositions = 2048, kRankThreads = 1024, kRankOf = kRankThreads / 16;

__global__ void __launch_bounds__(kRankThreads) k_sort_rank(const SortArgs a) {
    __shared__ unsigned int key[kRankPositions];
    __shared__ unsigned int bits[kRankThreads];
    for (unsigned int i = blockIdx.x * kRankThreads + threadIdx.x; i < a.n_arrived; i += gridDim.x * kRankThreads)
        a.arrived[i] = 0;
    constexpr int kMine = kRankPositions / kRankThreads;
    unsigned int mine[kMine], at[kMine];
    auto index = [&](int j) { return threadIdx.x + j * kRankThreads; };
    load_keys<kMine>(a, mine, at, index, blockIdx.x == 0);
#pragma unroll
    for (int j = 0; j < kMine; ++j)
        if (index(j) < a.n) key[index(j)] = mine[j];
    __syncthreads();
    const unsigned int p = blockIdx.x * kRankOf + threadIdx.x / 16;
    const unsigned int k = p < a.n ? key[p] : 0;
    unsigned int place = 0;
#pragma unroll 8
    for (unsigned int j = threadIdx.x % 16; j < a.n; j += 16) {
        const unsigned int x = key[j];
        place += x < k || (x == k && j < p);
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) place += __shfl_xor_sync(0xFFFFFFFFu, place, o);
    if (threadIdx.x % 16 == 0 && p < a.n) a.out[place] = make_uint2(k, p);
    if (a.present == nullptr) return;
    const unsigned int words = static_cast<unsigned int>((a.vocab + 31) / 32);
    const unsigned int share = (words + gridDim.x - 1) / gridDim.x;
    const unsigned int begin = blockIdx.x * share, end = begin + share < words ? begin + share : words;
    for (unsigned int w0 = begin; w0 < end; w0 += kRankThreads) {
        bits[threadIdx.x] = 0;
        __syncthreads();
        for (unsigned int j = threadIdx.x; j < a.n; j += kRankThreads) {
            const unsigned int w = key[j] / 32 - w0;  // below w0: beyond the array
            if (w < kRankThreads && key[j] < a.vocab) atomicOr(&bits[w], 1u << (key[j] % 32));
        }
        __syncthreads();
        if (w0 + threadIdx.x < end) a.present[w0 + threadIdx.x] = bits[threadIdx.x];
    }
}

constexpr int kTileKeys = kTile / kThreads;

__global__ void __launch_bounds__(kThreads) k_digit_count(const SortArgs a) {
    __shared__ unsigned int count[kMaxBins];
    const int bins = 1 << a.bits;
    for (int b = threadIdx.x; b < bins; b += kThreads) count[b] = 0;
    if (a.in == nullptr) clear_flags(a, blockIdx.x * kThreads + threadIdx.x, gridDim.x * kThreads);
    __syncthreads();
    const unsigned int first = blockIdx.x * kTile + threadIdx.x;
    unsigned int key[kTileKeys], at[kTileKeys];
    auto index = [&](int j) { return first + j * kThreads; };
    load_keys<kTileKeys>(a, key, at, index, true);
#pragma unroll
    for (int j = 0; j < kTileKeys; ++j)
        if (index(j) < a.n) atomicAdd(&count[(key[j] >> a.shift) & (bins - 1)], 1u);
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += kThreads) a.counts[blockIdx.x * bins + b] = count[b];
}

// Sums over the tiles before each tile, one thread a digit.
__global__ void __launch_bounds__(kThreads) k_digit_scan(const SortArgs a) {
    const int bins = 1 << a.bits;
    const int b = blockIdx.x * kThreads + threadIdx.x;
    if (b >= bins) return;
    unsigned int sum = 0;
    int t = 0;
    for (; t + 8 <= a.tiles; t += 8) {
        unsigned int c[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) c[u] = a.counts[static_cast<long long>(t + u) * bins + b];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            a.before[static_cast<long long>(t + u) * bins + b] = sum;
            sum += c[u];
        }
    }
    for (; t < a.tiles; ++t) {
        a.before[static_cast<long long>(t) * bins + b] = sum;
        sum += a.counts[static_cast<long long>(t) * bins + b];
    }
    a.before[static_cast<long long>(a.tiles) * bins + b] = sum;
}

__global__ void __launch_bounds__(kThreads) k_digit_place(const SortArgs a) {
    __shared__ unsigned int place[kMaxBins];      // where the tile's keys of a digit begin
    __shared__ unsigned short seen[8][kMaxBins];  // keys of a digit each warp has ranked so far
    __shared__ unsigned int warp_sums[8];
    const int bins = 1 << a.bits;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    for (int b = threadIdx.x; b < 8 * kMaxBins / 2; b += kThreads) reinterpret_cast<unsigned int *>(seen)[b] = 0;
    const unsigned int first = blockIdx.x * kTile + warp * (kTile / 8) + lane;
    auto index = [&](int j) { return first + j * 32; };
    auto live = [&](int j) { return index(j) < a.n; };
    unsigned int key[kTileKeys], at[kTileKeys];
    unsigned short rank[kTileKeys];
    load_keys<kTileKeys>(a, key, at, index, false);
    const int per_thread = (bins + kThreads - 1) / kThreads;
    unsigned int total[kMaxBins / kThreads], before[kMaxBins / kThreads], sum = 0;
#pragma unroll
    for (int j = 0; j < kMaxBins / kThreads; ++j) {
        total[j] = before[j] = 0;
        const int b = threadIdx.x * per_thread + j;
        if (j >= per_thread || b >= bins) continue;
        if (a.before != nullptr) {
            before[j] = a.before[static_cast<long long>(blockIdx.x) * bins + b];
            total[j] = a.before[static_cast<long long>(a.tiles) * bins + b];
        } else {
#pragma unroll 8
            for (int t = 0; t < a.tiles; ++t) {
                const unsigned int c = a.counts[t * bins + b];
                if (t < static_cast<int>(blockIdx.x)) before[j] += c;
                total[j] += c;
            }
        }
        sum += total[j];
    }
    unsigned int begin = block_exclusive(sum, warp_sums);
#pragma unroll
    for (int j = 0; j < kMaxBins / kThreads; ++j) {
        const int b = threadIdx.x * per_thread + j;
        if (j < per_thread && b < bins) place[b] = begin + before[j];
        begin += total[j];
    }
    __syncthreads();
    rank_keys<kTileKeys>(key, rank, live, a.shift, a.bits, seen[warp]);
    __syncthreads();
    // counts of the warps before: seen becomes each warp's first rank
    for (int b = threadIdx.x; b < bins; b += kThreads) {
        unsigned int s = 0;
#pragma unroll
        for (int w = 0; w < 8; ++w) {
            const unsigned int c = seen[w][b];
            seen[w][b] = static_cast<unsigned short>(s);
            s += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kTileKeys; ++j) {
        if (!live(j)) continue;
        const unsigned int d = (key[j] >> a.shift) & (bins - 1);
        a.out[place[d] + seen[warp][d] + rank[j]] = make_uint2(key[j], at[j]);
    }
    if (a.last) mark_present<kTileKeys>(a, key, live);
}

// ---------------------------------------------------------------- the sums --

constexpr int kRun = 32;      // sorted positions of a piece
constexpr int kZeroRows = 32;  // table rows a CTA checks for having no position

struct SumArgs {
    Positions pos;
    const uint2 *list;       // (token, position), sorted
    const unsigned int *present;
    unsigned int n;
    unsigned int pieces;
    unsigned int slabs;      // column slabs of kThreads * VEC
    unsigned int zero_units; // units behind the sums that clear rows without a position
    const float *dout;
    float *dtable;
    long long dout_cs, table_rs, table_cs;
    long long vocab, dim;
    float *partial;          // [pieces][2][dim]: the run that came in, the run that goes on
    unsigned int *arrived;   // [pieces][slabs] partial rows written of the run that begins in the piece
    float scale;
    int accumulate;
    int flat;                // rows to be cleared lie back to back and are cleared as one array
};

// A thread's columns of a row: VEC neighbouring ones moved at once, or, SPREAD, four that
// lie a CTA's width apart, for rows whose width, strides or address allow no vectors.
template <int VEC, bool SPREAD>
struct Columns {
    float v[VEC];
};

template <int VEC, bool SPREAD>
struct Place {
    using Values = Columns<VEC, SPREAD>;
    long long col;
    int count;  // columns that the row has; 0: none

    __device__ __forceinline__ Place(unsigned int slab, long long dim) {
        const long long first = static_cast<long long>(slab) * blockDim.x * VEC;
        if (SPREAD) {
            col = first + threadIdx.x;
            const long long left = dim - col + blockDim.x - 1;
            count = left <= 0 ? 0 : left / blockDim.x < VEC ? static_cast<int>(left / blockDim.x) : VEC;
        } else {
            col = first + static_cast<long long>(threadIdx.x) * VEC;
            count = col < dim ? VEC : 0;
        }
    }
    __device__ __forceinline__ Values zero() const {
        Values r;
#pragma unroll
        for (int j = 0; j < VEC; ++j) r.v[j] = 0.0f;
        return r;
    }
    template <bool SHARED = false>  // SHARED: another CTA has written it, past this SM's L1
    __device__ __forceinline__ Values load(const float *row, long long cs) const {
        Values r = zero();
        const float *p = row + col * cs;
        if (SPREAD) {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (j < count) r.v[j] = SHARED ? __ldcg(p + j * static_cast<long long>(blockDim.x) * cs)
                                               : p[j * static_cast<long long>(blockDim.x) * cs];
        } else if (count > 0) {
            if (VEC == 4) {
                const float4 *q = reinterpret_cast<const float4 *>(p);
                const float4 x = SHARED ? __ldcg(q) : *q;
                r.v[3 % VEC] = x.w;
                r.v[2 % VEC] = x.z;
                r.v[1] = x.y;
                r.v[0] = x.x;
            } else {
                const float2 *q = reinterpret_cast<const float2 *>(p);
                const float2 x = SHARED ? __ldcg(q) : *q;
                r.v[1] = x.y;
                r.v[0] = x.x;
            }
        }
        return r;
    }
    __device__ __forceinline__ void store(float *row, long long cs, const Values &r) const {
        float *p = row + col * cs;
        if (SPREAD) {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (j < count) p[j * static_cast<long long>(blockDim.x) * cs] = r.v[j];
        } else if (count > 0) {
            if (VEC == 4) *reinterpret_cast<float4 *>(p) = make_float4(r.v[0], r.v[1], r.v[2 % VEC], r.v[3 % VEC]);
            else *reinterpret_cast<float2 *>(p) = make_float2(r.v[0], r.v[1]);
        }
    }
    // scale * sum into a row of the table
    __device__ __forceinline__ void finish(const SumArgs &a, unsigned int k, Values r) const {
        float *row = a.dtable + k * a.table_rs;
#pragma unroll
        for (int j = 0; j < VEC; ++j) r.v[j] *= a.scale;
        if (a.accumulate) add(r, load(row, a.table_cs));
        store(row, a.table_cs, r);
    }
    static __device__ __forceinline__ void add(Values &a, const Values &b) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) a.v[j] += b.v[j];
    }
};

// Clears those of the table's rows v0 .. v0 + 31 that `has` has no bit for: this CTA's slab of
// their columns, or, of rows back to back at an odd or a small width, its share of the whole in
// 16-byte pieces.
template <class P>
__device__ __forceinline__ void clear_rows(const SumArgs &a, long long v0, unsigned int has, unsigned int slab) {
    const int rows = static_cast<int>(a.vocab - v0 < kZeroRows ? a.vocab - v0 : kZeroRows);
    if (a.flat) {
        float *base = a.dtable + v0 * a.table_rs;
        const unsigned int total = static_cast<unsigned int>(rows * a.dim), dim = static_cast<unsigned int>(a.dim);
        const unsigned int head = static_cast<unsigned int>((16 - (reinterpret_cast<uintptr_t>(base) & 15)) / 4) & 3;
        auto clear = [&](unsigned int e) {
            if (e < total && !(has >> (e / dim) & 1)) base[e] = 0.0f;
        };
        if (slab == 0 && threadIdx.x < head) clear(threadIdx.x);
        for (unsigned int e = head + 4 * (slab * blockDim.x + threadIdx.x); e < total; e += 4 * a.slabs * blockDim.x) {
            const unsigned int r0 = e / dim, r1 = (e + 3) / dim;
            if (e + 3 < total && !(has >> r0 & 1) && !(has >> r1 & 1) && r1 <= r0 + 1) {
                *reinterpret_cast<float4 *>(base + e) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            } else {
                for (int j = 0; j < 4; ++j) clear(e + j);
            }
        }
        return;
    }
    const P at(slab, a.dim);
    float *to = a.dtable + v0 * a.table_rs;
#pragma unroll 8
    for (int r = 0; r < kZeroRows; ++r)
        if (r < rows && !(has >> r & 1)) at.store(to + r * a.table_rs, a.table_cs, at.zero());
}

// Called by every piece that holds a part of a run of several pieces, once its partial
// row is written: the last of them adds the partial rows, in the order of the pieces,
// eight loads ahead.  `k`: the run's key; `on`: it goes on behind this piece.  One warp
// finds the run's first piece, another its last, 32 pieces a step.
template <class P>
__device__ __forceinline__ void join_run(const SumArgs &a, unsigned int k, unsigned int unit, bool on, const P &at) {
    __shared__ unsigned int range[2];
    __shared__ bool last_here;
    __threadfence();
    __syncthreads();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (warp == 0) {  // the piece is the first if its first key, or the one before it, is another
        for (unsigned int p0 = unit;; p0 -= 32) {
            const bool valid = p0 >= static_cast<unsigned int>(lane);
            const unsigned int p = valid ? p0 - lane : 0;
            const bool begins = p == 0 || a.list[p * kRun].x != k || a.list[p * kRun - 1].x != k;
            const unsigned int found = __ballot_sync(0xFFFFFFFFu, valid && begins);
            if (found != 0) {
                if (lane == 0) range[0] = p0 - (__ffs(found) - 1);
                break;
            }
        }
    } else if (warp == 1) {  // the last piece whose first key is still k
        unsigned int end = unit;
        for (unsigned int p0 = unit + 1; on; p0 += 32) {
            const unsigned int p = p0 + lane;
            const unsigned int found = __ballot_sync(0xFFFFFFFFu, p >= a.pieces || a.list[p * kRun].x != k);
            end = found != 0 ? p0 + __ffs(found) - 2 : p0 + 31;
            if (found != 0) break;
        }
        if (lane == 0) range[1] = end;
    }
    __syncthreads();
    const unsigned int begin = range[0];
    const unsigned int end = range[1];
    const unsigned int slab = blockIdx.x % a.slabs;
    if (threadIdx.x == 0) {
        last_here = atomicAdd(&a.arrived[begin * a.slabs + slab], 1u) == end - begin;
    }
    __syncthreads();
    if (!last_here) return;
    __threadfence();
    typename P::Values sum = at.zero();
    for (unsigned int p0 = begin; p0 <= end; p0 += 8) {
        typename P::Values x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (p0 + u <= end)
                x[u] = at.template load<true>(a.partial + (2ll * (p0 + u) + (p0 + u == begin)) * a.dim, 1);
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (p0 + u <= end) P::add(sum, x[u]);
    }
    at.finish(a, k, sum);
}

template <class P>
__global__ void __launch_bounds__(kThreads) k_token_sums(const SumArgs a) {
    wait_for_previous();
    const unsigned int unit = blockIdx.x / a.slabs;
    if (unit >= a.pieces) {
        // rows without a position
        const unsigned int group = unit - a.pieces;
        clear_rows<P>(a, static_cast<long long>(group) * kZeroRows, a.n > 0 ? a.present[group] : 0,
                        blockIdx.x - unit * a.slabs);
        return;
    }
    __shared__ unsigned int key[kRun + 2];   // with the neighbours' last and first
    __shared__ long long row[kRun];
    const unsigned int first = unit * kRun;
    const int count = static_cast<int>(a.n - first < kRun ? a.n - first : kRun);
    if (threadIdx.x < kRun + 2) {
        const long long i = static_cast<long long>(first) + threadIdx.x - 1;
        key[threadIdx.x] = i >= 0 && i < a.n ? a.list[i].x : 0xFFFFFFFFu;
    }
    if (threadIdx.x < count) {
        long long r;
        (void)token_at(a.pos, a.list[first + threadIdx.x].y, r);
        row[threadIdx.x] = r;
    }
    __syncthreads();
    const P at(blockIdx.x - unit * a.slabs, a.dim);
    typename P::Values sum = at.zero();
    // positions without a gradient are the last: their keys are V
    const bool comes_in = key[0] == key[1] && key[1] < a.vocab;
    const bool goes_on = key[count + 1] == key[count] && key[count] < a.vocab;
    bool head = comes_in;
    for (int i0 = 0; i0 < count && key[1 + i0] < a.vocab; i0 += 8) {
        typename P::Values x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (i0 + u < count && key[1 + i0 + u] < a.vocab) x[u] = at.load(a.dout + row[i0 + u], a.dout_cs);
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int i = i0 + u;
            if (i >= count || key[1 + i] >= a.vocab) break;
            const unsigned int k = key[1 + i];
            P::add(sum, x[u]);
            const bool on = key[2 + i] == k;
            if (on && i + 1 < count) continue;
            if (head) at.store(a.partial + (2ll * unit) * a.dim, 1, sum);
            else if (on) at.store(a.partial + (2ll * unit + 1) * a.dim, 1, sum);
            else at.finish(a, k, sum);
            head = false;
            sum = at.zero();
        }
    }
    const bool one_run = key[1] == key[count];  // (of a piece that goes on as it came in, the whole is the head)
    if (comes_in) join_run(a, key[1], unit, one_run && goes_on, at);
    if (goes_on && !(comes_in && one_run)) join_run(a, key[count], unit, true, at);
}

// Up to 256 positions need no sort: every CTA reads all tokens, the one of a token's first
// position adds the rows of all its positions, and the CTAs of the table's rows see which of
// them have none.  One launch instead of two.
constexpr int kFewPositions = kThreads;

template <class P>
__global__ void __launch_bounds__(kThreads) k_token_few(const SumArgs a, long long padding, unsigned long long *err) {
    __shared__ unsigned int key[kFewPositions];
    __shared__ long long row[kFewPositions];
    __shared__ unsigned short list[kFewPositions];
    __shared__ int before[kThreads / 32 + 1];
    __shared__ unsigned int has;
    const unsigned int unit = blockIdx.x / a.slabs;
    const unsigned int i = threadIdx.x;
    key[i] = 0xFFFFFFFFu;
    if (i == 0) has = 0;
    if (i < a.n) {
        long long r;
        const long long t = token_at(a.pos, i, r);
        if (t != padding && t >= 0 && t < a.vocab) key[i] = static_cast<unsigned int>(t);
        else if (t != padding && blockIdx.x == 0) report_index(err, t);
        row[i] = r;
    }
    __syncthreads();
    if (unit >= a.n) {
        const long long v0 = static_cast<long long>(unit - a.n) * kZeroRows;
        if (key[i] >= v0 && key[i] < v0 + kZeroRows) atomicOr(&has, 1u << (key[i] - v0));
        __syncthreads();
        clear_rows<P>(a, v0, has, blockIdx.x - unit * a.slabs);
        return;
    }
    const unsigned int k = key[unit];
    if (k == 0xFFFFFFFFu) return;
    if (__syncthreads_or(i < unit && key[i] == k)) return;
    const unsigned int same = __ballot_sync(0xFFFFFFFFu, key[i] == k);
    if (i % 32 == 0) before[i / 32 + 1] = __popc(same);
    if (i == 0) before[0] = 0;
    __syncthreads();
    int first = 0, count = 0;
#pragma unroll
    for (int w = 1; w <= kThreads / 32; ++w) {
        if (w <= static_cast<int>(i / 32)) first += before[w];
        count += before[w];
    }
    if (key[i] == k) list[first + __popc(same & ((1u << (i % 32)) - 1))] = static_cast<unsigned short>(i);
    __syncthreads();
    const P at(blockIdx.x - unit * a.slabs, a.dim);
    typename P::Values sum = at.zero();
    for (int i0 = 0; i0 < count; i0 += 8) {
        typename P::Values x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (i0 + u < count) x[u] = at.load(a.dout + row[list[i0 + u]], a.dout_cs);
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (i0 + u < count) P::add(sum, x[u]);
    }
    at.finish(a, k, sum);
}

using Vectors4 = Place<4, false>;
using Vectors2 = Place<2, false>;
using Spread4 = Place<4, true>;

// ------------------------------------------------------------------- host --

// Checks tokens against rows [tokens.shape + [D]] and a table [V, D], and folds
// the positions' axes.
int positions(const mtc_desc &table, const mtc_desc &tokens, const mtc_desc &rows, Positions &p) {
    if (table.rank != 2) return fail(MTC_ERR_INVALID_ARGUMENT, "the embedding table has rank %d instead of 2", table.rank);
    if (rows.rank != tokens.rank + 1)
        return fail(MTC_ERR_INVALID_ARGUMENT, "embedding rows have rank %d instead of %d", rows.rank, tokens.rank + 1);
    for (int i = 0; i < tokens.rank; ++i)
        if (rows.shape[i] != tokens.shape[i])
            return fail(MTC_ERR_INVALID_ARGUMENT, "embedding rows and tokens differ in extent %d", i);
    if (rows.shape[tokens.rank] != table.shape[1])
        return fail(MTC_ERR_INVALID_ARGUMENT, "embedding rows have %lld columns, the table %lld",
                    static_cast<long long>(rows.shape[tokens.rank]), static_cast<long long>(table.shape[1]));
    if (table.shape[0] >= (int64_t{1} << 32) - 1)
        return fail(MTC_ERR_UNSUPPORTED, "the embedding table has too many rows");
    IterSpace s;
    s.rank = tokens.rank;
    s.nops = 2;
    for (int i = 0; i < tokens.rank; ++i) {
        s.shape[i] = tokens.shape[i];
        s.stride[0][i] = tokens.strides[i];
        s.stride[1][i] = rows.strides[i];
    }
    simplify(s);
    std::memset(&p, 0, sizeof(p));
    p.n = s.numel;
    p.rank = s.rank;
    for (int i = 0; i < s.rank; ++i) {
        p.shape[i] = s.shape[i];
        p.tok_stride[i] = s.stride[0][i];
        p.row_stride[i] = s.stride[1][i];
    }
    p.tokens = static_cast<const long long *>(tokens.data) + tokens.offset;
    return MTC_OK;
}

// Whether the columns of a row can be moved `vec` at a time: contiguous, a
// multiple of it, every row on a boundary of it.
bool vector_rows(int vec, const float *base, int64_t dim, int64_t col_stride, const long long *row_strides,
                 int n_strides) {
    bool ok = reinterpret_cast<uintptr_t>(base) % (4 * vec) == 0 && dim % vec == 0 && col_stride == 1;
    for (int i = 0; i < n_strides && ok; ++i) ok = row_strides[i] % vec == 0;
    return ok;
}

int run_embedding(const mtc_desc *table, const mtc_desc *tokens, float scale, int64_t padding, const mtc_desc *out,
                  cudaStream_t stream) {
    MTC_TRY(need_float(table, "table"));
    MTC_TRY(need_int(tokens, "tokens"));
    MTC_TRY(need_float(out, "output"));
    LookupArgs a;
    std::memset(&a, 0, sizeof(a));
    MTC_TRY(positions(*table, *tokens, *out, a.pos));
    MTC_TRY(need_distinct(out, "output"));
    const int64_t dim = table->shape[1];
    if (a.pos.n == 0 || dim == 0) return MTC_OK;
    a.table = float_at(table);
    a.out = float_at(out);
    a.table_rs = table->strides[0];
    a.table_cs = table->strides[1];
    a.out_cs = out->strides[out->rank - 1];
    a.vocab = table->shape[0];
    a.padding = padding;
    a.scale = scale;
    MTC_TRY(device_error_word(&a.err));
    const long long table_rs = a.table_rs;
    const bool vec = vector_rows(4, a.table, dim, a.table_cs, &table_rs, 1) &&
                     vector_rows(4, a.out, dim, a.out_cs, a.pos.row_stride, a.pos.rank);
    a.vectors = vec ? dim / 4 : dim;
    while (a.lanes_log2 < 5 && (int64_t{kLookupLoads} << a.lanes_log2) < a.vectors) ++a.lanes_log2;
    const int64_t segment = int64_t{kLookupLoads} << a.lanes_log2;
    if (a.vectors / segment >= UINT32_MAX) return fail(MTC_ERR_UNSUPPORTED, "embedding rows are too wide");
    a.segments = static_cast<unsigned int>((a.vectors + segment - 1) / segment);
    a.groups = a.pos.n * a.segments;
    const int64_t ctas = ((a.groups << a.lanes_log2) + kThreads - 1) / kThreads;
    const int64_t most = static_cast<int64_t>(sm_count(current_device())) * 8;
    const unsigned int grid = static_cast<unsigned int>(ctas < most ? ctas : most);
    if (vec) k_embedding<4><<<grid, kThreads, 0, stream>>>(a);
    else k_embedding<1><<<grid, kThreads, 0, stream>>>(a);
    return check_launch("embedding");
}

constexpr int kFewTiles = 32;      // tiles whose counts every CTA adds itself (one launch less)

int digit_bits(int64_t vocab, int most, int &passes) {
    int bits = 1;
    while ((int64_t{1} << bits) <= vocab) ++bits;  // keys 0..vocab
    passes = (bits + most - 1) / most;
    return (bits + passes - 1) / passes;
}

template <int N>
int sort_in_cluster(SortArgs a, cudaStream_t stream) {
    a.bits = digit_bits(a.vocab, 9, a.passes);
    const unsigned int keys = kClusterThreads * N;
    unsigned int ctas = 1;
    while (ctas * keys < a.n) ctas *= 2;
    MTC_CUDA_TRY(cudaFuncSetAttribute(k_sort_cluster<N>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(ClusterSort)));
    MTC_CUDA_TRY(cudaFuncSetAttribute(k_sort_cluster<N>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchConfig_t config;
    std::memset(&config, 0, sizeof(config));
    config.gridDim = dim3(ctas);
    config.blockDim = dim3(kClusterThreads);
    config.dynamicSmemBytes = sizeof(ClusterSort);
    config.stream = stream;
    cudaLaunchAttribute attr;
    std::memset(&attr, 0, sizeof(attr));
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = ctas;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    config.attrs = &attr;
    config.numAttrs = 1;
    MTC_CUDA_TRY(cudaLaunchKernelEx(&config, k_sort_cluster<N>, a));
    return check_launch("token sort");
}

// Sorts the positions by token; `sums.list` becomes one of the two `buffers` of n.
int sort_positions(SumArgs &sums, int64_t padding, uint2 *buffers, unsigned int *counts, unsigned int *before,
                   unsigned int *present, cudaStream_t stream) {
    SortArgs a;
    std::memset(&a, 0, sizeof(a));
    a.pos = sums.pos;
    a.vocab = sums.vocab;
    a.padding = padding;
    a.n = sums.n;
    a.tiles = static_cast<int>((sums.pos.n + kTile - 1) / kTile);
    a.present = present;
    a.arrived = sums.arrived;
    a.n_arrived = sums.pieces * sums.slabs;
    MTC_TRY(device_error_word(&a.err));
    a.out = buffers;
    sums.list = a.out;
    if (a.n <= kRankPositions && a.vocab < (int64_t{1} << 24)) {
        k_sort_rank<<<(a.n + kRankOf - 1) / kRankOf, kRankThreads, 0, stream>>>(a);
        return check_launch("token sort (ranks)");
    }
    if (a.n <= kClusterThreads * kClusterTiles) return sort_in_cluster<1>(a, stream);
    if (a.n <= kClusterThreads * kClusterTiles * 2) return sort_in_cluster<2>(a, stream);
    if (a.n <= kClusterThreads * kClusterTiles * 4) return sort_in_cluster<4>(a, stream);
    a.counts = counts;
    a.before = a.tiles > kFewTiles ? before : nullptr;
    a.bits = digit_bits(a.vocab, 10, a.passes);
    for (int p = 0; p < a.passes; ++p) {
        a.shift = p * a.bits;
        a.last = p == a.passes - 1;
        a.out = buffers + (p % 2) * static_cast<int64_t>(a.n);
        k_digit_count<<<a.tiles, kThreads, 0, stream>>>(a);
        MTC_TRY(check_launch("token sort (count)"));
        if (a.before != nullptr) {
            k_digit_scan<<<((1 << a.bits) + kThreads - 1) / kThreads, kThreads, 0, stream>>>(a);
            MTC_TRY(check_launch("token sort (scan)"));
        }
        k_digit_place<<<a.tiles, kThreads, 0, stream>>>(a);
        MTC_TRY(check_launch("token sort (place)"));
        a.in = a.out;
    }
    sums.list = a.in;
    return MTC_OK;
}

int run_embedding_grad(const mtc_desc *dout, const mtc_desc *tokens, float scale, int64_t padding, int accumulate,
                       const mtc_desc *dtable, cudaStream_t stream) {
    MTC_TRY(need_float(dout, "dout"));
    MTC_TRY(need_int(tokens, "tokens"));
    MTC_TRY(need_float(dtable, "dtable"));
    SumArgs a;
    std::memset(&a, 0, sizeof(a));
    MTC_TRY(positions(*dtable, *tokens, *dout, a.pos));
    MTC_TRY(need_distinct(dtable, "dtable"));
    a.vocab = dtable->shape[0];
    a.dim = dtable->shape[1];
    if (a.vocab == 0 || a.dim == 0) return MTC_OK;
    if (a.pos.n > INT32_MAX) return fail(MTC_ERR_UNSUPPORTED, "more than 2^31 - 1 positions");
    a.n = static_cast<unsigned int>(a.pos.n);
    a.pieces = (a.n + kRun - 1) / kRun;
    a.dout = float_at(dout);
    a.dtable = float_at(dtable);
    a.dout_cs = dout->strides[dout->rank - 1];
    a.table_rs = dtable->strides[0];
    a.table_cs = dtable->strides[1];
    a.scale = scale;
    a.accumulate = accumulate != 0;
    const long long table_rs = a.table_rs;
    auto fits = [&](int v) {
        return vector_rows(v, a.dtable, a.dim, a.table_cs, &table_rs, 1) &&
               (a.n == 0 || vector_rows(v, a.dout, a.dim, a.dout_cs, a.pos.row_stride, a.pos.rank));
    };
    const int vec = fits(4) ? 4 : fits(2) ? 2 : 1;
    // narrow rows take smaller CTAs (of two warps at least), so that their threads have columns
    const bool few = a.n > 0 && a.n <= kFewPositions;
    const int columns = vec == 2 ? 2 : 4;  // of a thread
    const int64_t lanes = ((a.dim + columns - 1) / columns + 31) / 32 * 32;
    const int threads = few || lanes > kThreads ? kThreads : lanes < 64 ? 64 : static_cast<int>(lanes);
    const int64_t slab = static_cast<int64_t>(threads) * columns;
    a.slabs = static_cast<unsigned int>((a.dim + slab - 1) / slab);
    // 131072 rows of 64 columns, one position: 31 us by rows of 16 threads, 11 us flat; of 512
    // columns both 41.  Among many rows that have positions, flat costs up to a quarter more.
    a.flat = (vec < 4 || (few && a.dim < 512)) && a.table_cs == 1 && a.table_rs == a.dim && a.dim < (int64_t{1} << 26);
    const int64_t zero_units = accumulate ? 0 : (a.vocab + kZeroRows - 1) / kZeroRows;
    if ((zero_units + a.pieces + kFewPositions) * static_cast<int64_t>(a.slabs) > INT32_MAX)
        return fail(MTC_ERR_UNSUPPORTED, "the embedding gradient is too large for one launch");
    a.zero_units = static_cast<unsigned int>(zero_units);
    if (a.pieces + a.zero_units == 0) return MTC_OK;
    if (few) {
        unsigned long long *err = nullptr;
        MTC_TRY(device_error_word(&err));
        const unsigned int ctas = (a.n + a.zero_units) * a.slabs;
        if (vec == 4) k_token_few<Vectors4><<<ctas, kThreads, 0, stream>>>(a, padding, err);
        else if (vec == 2) k_token_few<Vectors2><<<ctas, kThreads, 0, stream>>>(a, padding, err);
        else k_token_few<Spread4><<<ctas, kThreads, 0, stream>>>(a, padding, err);
        return check_launch("embedding gradient (few positions)");
    }
    const size_t list = padded(2 * static_cast<size_t>(a.n) * sizeof(uint2));
    const size_t tiles = (static_cast<size_t>(a.n) + kTile - 1) / kTile;
    const size_t counts = padded(tiles * kMaxBins * sizeof(unsigned int));
    const size_t before = padded((tiles + 1) * kMaxBins * sizeof(unsigned int));
    const size_t partial = padded(static_cast<size_t>(a.pieces) * 2 * a.dim * sizeof(float));
    const size_t present = padded(static_cast<size_t>((a.vocab + 31) / 32) * sizeof(unsigned int));
    Workspace ws;
    const size_t arrived = padded(static_cast<size_t>(a.pieces) * a.slabs * sizeof(unsigned int));
    if (a.n > 0) {
        MTC_TRY(ws.allocate(list + counts + before + partial + arrived + present, stream));
        uint2 *buffers = ws.take<uint2>(list);
        unsigned int *c = ws.take<unsigned int>(counts);
        unsigned int *b = ws.take<unsigned int>(before);
        a.partial = ws.take<float>(partial);
        a.arrived = ws.take<unsigned int>(arrived);
        unsigned int *rows = accumulate ? nullptr : ws.take<unsigned int>(present);
        a.present = rows;
        MTC_TRY(sort_positions(a, padding, buffers, c, b, rows, stream));
    }
    const unsigned int grid = (a.pieces + a.zero_units) * a.slabs;
    auto sums = vec == 4 ? k_token_sums<Vectors4> : vec == 2 ? k_token_sums<Vectors2> : k_token_sums<Spread4>;
    if (a.n > 0) return launch_dependent("embedding gradient (sums)", sums, grid, threads, 0, stream, a);
    sums<<<grid, threads, 0, stream>>>(a);  // nothing but rows to clear: the call's first launch
    return check_launch("embedding gradient (sums)");
}

}  // namespace
}  // namespace mtc

using namespace mtc;

extern "C" {

int mtc_embedding(const mtc_desc *table, const mtc_desc *tokens, float scale, int64_t padding_token,
                  const mtc_desc *out, void *stream) {
    clear_error();
    return run_embedding(table, tokens, scale, padding_token, out, static_cast<cudaStream_t>(stream));
}

int mtc_embedding_grad(const mtc_desc *dout, const mtc_desc *tokens, float scale, int64_t padding_token,
                       int32_t accumulate, const mtc_desc *dtable, void *stream) {
    clear_error();
    return run_embedding_grad(dout, tokens, scale, padding_token, accumulate, dtable,
                              static_cast<cudaStream_t>(stream));
}

}  // extern "C"
