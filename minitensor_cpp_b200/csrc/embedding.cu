// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   out[i, :] = scale * table[tok_i, :]            dtable[v, :] = scale * sum_{i: tok_i = v} dout[i, :]
//
// The lookup reads each row once and writes 4 D bytes a position: bound by HBM
// for many positions, by the launch for few.  Threads walk the flat space of
// (position, four columns), four loads in flight each, so rows of any width
// keep the CTA full and neighbouring threads stay on neighbouring addresses.
//
// The gradient reads every dout row once and writes every table row once.
// Atomics would add the rows of a frequent token one after the other at one
// address, in an order that changes from run to run; a walk by token leaves a
// token of a natural text (a few own thousands of positions, most own none) to
// one CTA.  So the positions are sorted by token (stable, so ascending within a
// token), and the sorted list is cut into pieces of 32 positions, whatever the
// tokens: one CTA adds a piece's runs in registers, writes the rows whose run
// lies inside the piece, and leaves the run that came in from the piece before
// and the one that goes on into the next as partial rows.  A second kernel joins
// those.  Which sums are formed depends on the tokens alone.
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
    long long first;      // position of the launch's first row
    unsigned int total;   // vectors of the launch
    FastDiv per_row;      // vectors a row
    const float *table;
    float *out;
    long long table_rs, table_cs, out_cs;
    long long vocab;
    long long padding;
    float scale;
    unsigned long long *err;
};

template <int VEC>
__global__ void __launch_bounds__(kThreads) k_embedding(const LookupArgs a) {
    constexpr int U = 4;
    const unsigned int base = blockIdx.x * (kThreads * U) + threadIdx.x;
    float4 v[U];
    float *dst[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const unsigned int q = base + u * kThreads;
        dst[u] = nullptr;
        v[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (q >= a.total) continue;
        const unsigned int r = fastdiv(q, a.per_row);
        const long long c = q - r * a.per_row.d;
        long long row;
        const long long t = token_at(a.pos, a.first + r, row);
        if (t == a.padding) {
            dst[u] = a.out + row + c * VEC * a.out_cs;
            continue;
        }
        if (t < 0 || t >= a.vocab) {
            if (c == 0) report_index(a.err, t);
            continue;
        }
        dst[u] = a.out + row + c * VEC * a.out_cs;
        const float *src = a.table + t * a.table_rs + c * VEC * a.table_cs;
        if (VEC == 4) v[u] = __ldg(reinterpret_cast<const float4 *>(src));
        else v[u].x = __ldg(src);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (dst[u] == nullptr) continue;
        if (VEC == 4)
            *reinterpret_cast<float4 *>(dst[u]) =
                make_float4(v[u].x * a.scale, v[u].y * a.scale, v[u].z * a.scale, v[u].w * a.scale);
        else
            *dst[u] = v[u].x * a.scale;
    }
}

// ---------------------------------------------------------------- the sort --
// Least-significant-digit radix sort of (token, position), stable.  A tile is
// 4096 keys of one CTA; a key of a position without a gradient is V, the
// largest.  Each pass: count the digits of every tile, then place every tile
// after the sum of the counts before it.  Eight warps own 512 consecutive keys
// of the tile each and rank them 32 at a time with match_any, so equal digits
// keep their order.

constexpr int kTile = 4096;
constexpr int kWarpKeys = 512;  // kTile / 8 warps
constexpr int kMaxBins = 1024;

struct SortArgs {
    Positions pos;
    long long vocab, padding;
    unsigned int n;
    int shift, bits;
    int tiles;
    const unsigned int *keys_in;  // null: read the tokens
    const unsigned int *at_in;
    unsigned int *keys_out, *at_out;
    unsigned int *counts;  // [tiles][bins]
    unsigned int *before;  // [tiles][bins] sums over the tiles before, and [bins] totals behind them; null: few tiles
    unsigned long long *err;
};

__device__ __forceinline__ unsigned int key_of(const SortArgs &a, unsigned int i, bool report) {
    if (a.keys_in != nullptr) return a.keys_in[i];
    long long row;
    const long long t = token_at(a.pos, i, row);
    if (t == a.padding) return static_cast<unsigned int>(a.vocab);
    if (t < 0 || t >= a.vocab) {
        if (report) report_index(a.err, t);
        return static_cast<unsigned int>(a.vocab);
    }
    return static_cast<unsigned int>(t);
}

__global__ void __launch_bounds__(kThreads) k_digit_count(const SortArgs a) {
    __shared__ unsigned int count[kMaxBins];
    const int bins = 1 << a.bits;
    for (int b = threadIdx.x; b < bins; b += kThreads) count[b] = 0;
    __syncthreads();
    const unsigned int first = blockIdx.x * kTile;
#pragma unroll 4
    for (int j = 0; j < kTile / kThreads; ++j) {
        const unsigned int i = first + j * kThreads + threadIdx.x;
        if (i < a.n) atomicAdd(&count[(key_of(a, i, true) >> a.shift) & (bins - 1)], 1u);
    }
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
        for (int u = 0; u < 8; ++u) c[u] = a.counts[(t + u) * bins + b];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            a.before[(t + u) * bins + b] = sum;
            sum += c[u];
        }
    }
    for (; t < a.tiles; ++t) {
        a.before[t * bins + b] = sum;
        sum += a.counts[t * bins + b];
    }
    a.before[a.tiles * bins + b] = sum;
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
    unsigned int before = 0;
    for (int w = 0; w < warp; ++w) before += warp_sums[w];
    return before + x - v;
}

__global__ void __launch_bounds__(kThreads) k_digit_place(const SortArgs a) {
    __shared__ unsigned int place[kMaxBins];           // where the tile's keys of a digit begin
    __shared__ unsigned short seen[8][kMaxBins];       // keys of a digit each warp has ranked so far
    __shared__ unsigned int warp_sums[8];
    const int bins = 1 << a.bits;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    for (int b = threadIdx.x; b < 8 * kMaxBins / 2; b += kThreads) reinterpret_cast<unsigned int *>(seen)[b] = 0;
    const int per_thread = (bins + kThreads - 1) / kThreads;
    unsigned int total[kMaxBins / kThreads], before[kMaxBins / kThreads], sum = 0;
#pragma unroll
    for (int j = 0; j < kMaxBins / kThreads; ++j) {
        total[j] = before[j] = 0;
        const int b = threadIdx.x * per_thread + j;
        if (j >= per_thread || b >= bins) continue;
        if (a.before != nullptr) {
            before[j] = a.before[blockIdx.x * bins + b];
            total[j] = a.before[a.tiles * bins + b];
        } else {
            for (int t = 0; t < a.tiles; ++t) {
                const unsigned int c = a.counts[t * bins + b];
                if (t < static_cast<int>(blockIdx.x)) before[j] += c;
                total[j] += c;
            }
        }
        sum += total[j];
    }
    unsigned int at = block_exclusive(sum, warp_sums);
#pragma unroll
    for (int j = 0; j < kMaxBins / kThreads; ++j) {
        const int b = threadIdx.x * per_thread + j;
        if (j < per_thread && b < bins) place[b] = at + before[j];
        at += total[j];
    }
    __syncthreads();
    // ranks within the warp's 512 keys
    const unsigned int first = blockIdx.x * kTile + warp * kWarpKeys;
    unsigned int key[kWarpKeys / 32];
    unsigned short rank[kWarpKeys / 32];
#pragma unroll
    for (int j = 0; j < kWarpKeys / 32; ++j) {
        const unsigned int i = first + j * 32 + lane;
        key[j] = i < a.n ? key_of(a, i, false) : 0u;
    }
#pragma unroll
    for (int j = 0; j < kWarpKeys / 32; ++j) {
        const bool live = first + j * 32 + lane < a.n;
        const unsigned int d = (key[j] >> a.shift) & (bins - 1);
        const unsigned int same = __match_any_sync(0xFFFFFFFFu, live ? d : 0xFFFFFFFFu);
        rank[j] = 0;
        if (live) rank[j] = seen[warp][d] + __popc(same & ((1u << lane) - 1));
        __syncwarp();
        if (live && (same >> lane) == 1u) seen[warp][d] = rank[j] + 1;  // the last of the equal lanes
        __syncwarp();
    }
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
    for (int j = 0; j < kWarpKeys / 32; ++j) {
        const unsigned int i = first + j * 32 + lane;
        if (i >= a.n) continue;
        const unsigned int d = (key[j] >> a.shift) & (bins - 1);
        const unsigned int to = place[d] + seen[warp][d] + rank[j];
        a.keys_out[to] = key[j];
        a.at_out[to] = a.at_in != nullptr ? a.at_in[i] : i;
    }
}

// ---------------------------------------------------------------- the sums --

constexpr int kRun = 32;      // sorted positions of a piece
constexpr int kZeroRows = 8;  // table rows a CTA checks for having no position

struct SumArgs {
    Positions pos;
    const unsigned int *keys, *at;
    unsigned int n;
    unsigned int pieces;
    unsigned int slabs;      // column slabs of kThreads * VEC
    unsigned int zero_units; // units behind the sums that clear rows without a position
    const float *dout;
    float *dtable;
    long long dout_cs, table_rs, table_cs;
    long long vocab, dim;
    float *partial;          // [pieces][2][dim]: the run that came in, the run that goes on
    float scale;
    int accumulate;
};

template <int VEC>
struct Row {
    float v[VEC];
};

template <int VEC>
__device__ __forceinline__ Row<VEC> load_row(const float *p) {
    Row<VEC> r;
    if (VEC == 4) {
        const float4 x = *reinterpret_cast<const float4 *>(p);
        r.v[3 % VEC] = x.w;
        r.v[2 % VEC] = x.z;
        r.v[1 % VEC] = x.y;
        r.v[0] = x.x;
    } else {
        r.v[0] = *p;
    }
    return r;
}

template <int VEC>
__device__ __forceinline__ void store_row(float *p, const Row<VEC> &r) {
    if (VEC == 4) *reinterpret_cast<float4 *>(p) = make_float4(r.v[0], r.v[1 % VEC], r.v[2 % VEC], r.v[3 % VEC]);
    else *p = r.v[0];
}

template <int VEC>
__device__ __forceinline__ void finish_row(const SumArgs &a, float *p, Row<VEC> r) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) r.v[j] *= a.scale;
    if (a.accumulate) {
        const Row<VEC> old = load_row<VEC>(p);
#pragma unroll
        for (int j = 0; j < VEC; ++j) r.v[j] += old.v[j];
    }
    store_row<VEC>(p, r);
}

__device__ __forceinline__ unsigned int lower_bound(const unsigned int *keys, unsigned int n, unsigned int v) {
    unsigned int lo = 0, hi = n;
    while (lo < hi) {
        const unsigned int mid = (lo + hi) / 2;
        if (keys[mid] < v) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

template <int VEC>
__global__ void __launch_bounds__(kThreads) k_token_sums(const SumArgs a) {
    const unsigned int unit = blockIdx.x / a.slabs;
    const long long col = (static_cast<long long>(blockIdx.x - unit * a.slabs) * kThreads + threadIdx.x) * VEC;
    if (unit >= a.pieces) {
        // rows without a position
        __shared__ unsigned char empty[kZeroRows];
        const long long v0 = static_cast<long long>(unit - a.pieces) * kZeroRows;
        if (threadIdx.x < kZeroRows) {
            const long long v = v0 + threadIdx.x;
            bool none = v < a.vocab;
            if (none) {
                const unsigned int at = lower_bound(a.keys, a.n, static_cast<unsigned int>(v));
                none = at >= a.n || a.keys[at] != static_cast<unsigned int>(v);
            }
            empty[threadIdx.x] = none;
        }
        __syncthreads();
        if (col >= a.dim) return;
        Row<VEC> zero;
#pragma unroll
        for (int j = 0; j < VEC; ++j) zero.v[j] = 0.0f;
#pragma unroll
        for (int r = 0; r < kZeroRows; ++r)
            if (empty[r]) store_row<VEC>(a.dtable + (v0 + r) * a.table_rs + col * a.table_cs, zero);
        return;
    }
    __shared__ unsigned int key[kRun + 2];   // with the neighbours' last and first
    __shared__ long long row[kRun];
    const unsigned int first = unit * kRun;
    const int count = static_cast<int>(a.n - first < kRun ? a.n - first : kRun);
    if (threadIdx.x < kRun + 2) {
        const long long i = static_cast<long long>(first) + threadIdx.x - 1;
        key[threadIdx.x] = i >= 0 && i < a.n ? a.keys[i] : 0xFFFFFFFFu;
    }
    if (threadIdx.x < count) {
        long long r;
        (void)token_at(a.pos, a.at[first + threadIdx.x], r);
        row[threadIdx.x] = r;
    }
    __syncthreads();
    if (col >= a.dim) return;
    const float *src = a.dout + col * a.dout_cs;
    Row<VEC> sum;
#pragma unroll
    for (int j = 0; j < VEC; ++j) sum.v[j] = 0.0f;
    bool came_in = key[0] == key[1];
    for (int i0 = 0; i0 < count; i0 += 8) {
        Row<VEC> x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (i0 + u < count && key[1 + i0 + u] < a.vocab) x[u] = load_row<VEC>(src + row[i0 + u]);
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int i = i0 + u;
            if (i >= count) break;
            const unsigned int k = key[1 + i];
            if (k >= a.vocab) return;  // positions without a gradient are the last
#pragma unroll
            for (int j = 0; j < VEC; ++j) sum.v[j] += x[u].v[j];
            const bool goes_on = key[2 + i] == k;
            if (goes_on && i + 1 < count) continue;
            if (came_in) {
                store_row<VEC>(a.partial + (2ll * unit) * a.dim + col, sum);
            } else if (goes_on) {
                store_row<VEC>(a.partial + (2ll * unit + 1) * a.dim + col, sum);
            } else {
                finish_row<VEC>(a, a.dtable + k * a.table_rs + col * a.table_cs, sum);
            }
            came_in = false;
#pragma unroll
            for (int j = 0; j < VEC; ++j) sum.v[j] = 0.0f;
        }
    }
}

// Joins the runs that cross pieces: the piece in which a run begins adds the
// partial rows of the pieces after it, eight loads ahead.
template <int VEC>
__global__ void __launch_bounds__(kThreads) k_token_join(const SumArgs a) {
    const unsigned int unit = blockIdx.x / a.slabs;
    const long long col = (static_cast<long long>(blockIdx.x - unit * a.slabs) * kThreads + threadIdx.x) * VEC;
    const unsigned int last = (unit + 1) * kRun - 1;  // the piece's last position; there is a piece after it
    const unsigned int k = a.keys[last];
    if (k >= a.vocab || a.keys[last + 1] != k) return;
    const unsigned int first = unit * kRun;
    if (first > 0 && a.keys[first] == k && a.keys[first - 1] == k) return;  // began before
    unsigned int end = unit + 1;  // the last piece that the run reaches
    {
        unsigned int lo = unit + 1, hi = a.pieces - 1;
        while (lo < hi) {  // its first key is still k
            const unsigned int mid = (lo + hi + 1) / 2;
            if (a.keys[mid * kRun] == k) lo = mid;
            else hi = mid - 1;
        }
        end = lo;
    }
    if (col >= a.dim) return;
    Row<VEC> sum = load_row<VEC>(a.partial + (2ll * unit + 1) * a.dim + col);
    for (unsigned int p0 = unit + 1; p0 <= end; p0 += 8) {
        Row<VEC> x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (p0 + u <= end) x[u] = load_row<VEC>(a.partial + (2ll * (p0 + u)) * a.dim + col);
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (p0 + u <= end) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) sum.v[j] += x[u].v[j];
            }
    }
    finish_row<VEC>(a, a.dtable + k * a.table_rs + col * a.table_cs, sum);
}

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

// Whether the columns of a row can be moved four at a time: contiguous, a
// multiple of four, every row on a 16-byte boundary.
bool vector_rows(const float *base, int64_t dim, int64_t col_stride, const long long *row_strides, int n_strides) {
    bool ok = aligned16(base) && dim % 4 == 0 && col_stride == 1;
    for (int i = 0; i < n_strides && ok; ++i) ok = row_strides[i] % 4 == 0;
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
    const bool vec = vector_rows(a.table, dim, a.table_cs, &table_rs, 1) &&
                     vector_rows(a.out, dim, a.out_cs, a.pos.row_stride, a.pos.rank);
    const int64_t per_row = vec ? dim / 4 : dim;
    if (per_row >= (int64_t{1} << 31)) return fail(MTC_ERR_UNSUPPORTED, "embedding rows are too wide");
    a.per_row = make_fastdiv(static_cast<uint32_t>(per_row));
    const int64_t rows_a_launch = (int64_t{1} << 31) / per_row;
    for (a.first = 0; a.first < a.pos.n; a.first += rows_a_launch) {
        const int64_t rows = a.pos.n - a.first < rows_a_launch ? a.pos.n - a.first : rows_a_launch;
        a.total = static_cast<unsigned int>(rows * per_row);
        const unsigned int grid = static_cast<unsigned int>((static_cast<int64_t>(a.total) + kThreads * 4 - 1) / (kThreads * 4));
        if (vec) k_embedding<4><<<grid, kThreads, 0, stream>>>(a);
        else k_embedding<1><<<grid, kThreads, 0, stream>>>(a);
        MTC_TRY(check_launch("embedding"));
    }
    return MTC_OK;
}

// The positions in token order: keys and positions in two buffers of n each.
struct Sorted {
    const unsigned int *keys;
    const unsigned int *at;
};

constexpr int kFewTiles = 32;  // tiles whose counts every CTA adds itself (one launch less)

int digit_bits(int64_t vocab, int &passes) {
    int bits = 1;
    while ((int64_t{1} << bits) <= vocab) ++bits;  // keys 0..vocab
    passes = (bits + 9) / 10;
    return (bits + passes - 1) / passes;
}

int sort_positions(const Positions &pos, int64_t vocab, int64_t padding, unsigned int *buffers, unsigned int *counts,
                   unsigned int *before, cudaStream_t stream, Sorted &sorted) {
    SortArgs a;
    std::memset(&a, 0, sizeof(a));
    a.pos = pos;
    a.vocab = vocab;
    a.padding = padding;
    a.n = static_cast<unsigned int>(pos.n);
    a.tiles = static_cast<int>((pos.n + kTile - 1) / kTile);
    a.counts = counts;
    a.before = a.tiles > kFewTiles ? before : nullptr;
    MTC_TRY(device_error_word(&a.err));
    int passes;
    a.bits = digit_bits(vocab, passes);
    unsigned int *from = nullptr, *to = buffers;
    for (int p = 0; p < passes; ++p) {
        a.shift = p * a.bits;
        a.keys_in = from;
        a.at_in = from != nullptr ? from + pos.n : nullptr;
        a.keys_out = to;
        a.at_out = to + pos.n;
        k_digit_count<<<a.tiles, kThreads, 0, stream>>>(a);
        MTC_TRY(check_launch("token sort (count)"));
        if (a.before != nullptr) {
            k_digit_scan<<<((1 << a.bits) + kThreads - 1) / kThreads, kThreads, 0, stream>>>(a);
            MTC_TRY(check_launch("token sort (scan)"));
        }
        k_digit_place<<<a.tiles, kThreads, 0, stream>>>(a);
        MTC_TRY(check_launch("token sort (place)"));
        unsigned int *next = from != nullptr ? from : buffers + 2 * pos.n;
        from = to;
        to = next;
    }
    sorted.keys = from;
    sorted.at = from + pos.n;
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
    const bool vec = vector_rows(a.dtable, a.dim, a.table_cs, &table_rs, 1) &&
                     (a.n == 0 || vector_rows(a.dout, a.dim, a.dout_cs, a.pos.row_stride, a.pos.rank));
    const int64_t slab = kThreads * (vec ? 4 : 1);
    a.slabs = static_cast<unsigned int>((a.dim + slab - 1) / slab);
    const int64_t zero_units = accumulate ? 0 : (a.vocab + kZeroRows - 1) / kZeroRows;
    if ((zero_units + a.pieces) * static_cast<int64_t>(a.slabs) > INT32_MAX)
        return fail(MTC_ERR_UNSUPPORTED, "the embedding gradient is too large for one launch");
    a.zero_units = static_cast<unsigned int>(zero_units);
    if (a.pieces + a.zero_units == 0) return MTC_OK;
    const size_t list = padded(4 * static_cast<size_t>(a.n) * sizeof(unsigned int));
    const size_t tiles = (static_cast<size_t>(a.n) + kTile - 1) / kTile;
    const size_t counts = padded(tiles * kMaxBins * sizeof(unsigned int));
    const size_t before = padded((tiles + 1) * kMaxBins * sizeof(unsigned int));
    const size_t partial = padded(static_cast<size_t>(a.pieces) * 2 * a.dim * sizeof(float));
    Workspace ws;
    if (a.n > 0) {
        MTC_TRY(ws.allocate(list + counts + before + partial, stream));
        unsigned int *buffers = ws.take<unsigned int>(list);
        unsigned int *c = ws.take<unsigned int>(counts);
        unsigned int *b = ws.take<unsigned int>(before);
        a.partial = ws.take<float>(partial);
        Sorted sorted;
        MTC_TRY(sort_positions(a.pos, a.vocab, padding, buffers, c, b, stream, sorted));
        a.keys = sorted.keys;
        a.at = sorted.at;
    }
    const unsigned int grid = (a.pieces + a.zero_units) * a.slabs;
    if (vec) k_token_sums<4><<<grid, kThreads, 0, stream>>>(a);
    else k_token_sums<1><<<grid, kThreads, 0, stream>>>(a);
    MTC_TRY(check_launch("embedding gradient (sums)"));
    if (a.pieces < 2) return MTC_OK;
    const unsigned int joins = (a.pieces - 1) * a.slabs;
    if (vec) k_token_join<4><<<joins, kThreads, 0, stream>>>(a);
    else k_token_join<1><<<joins, kThreads, 0, stream>>>(a);
    return check_launch("embedding gradient (join)");
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
