// Linear cross entropy on the tensor cores, with float32 accuracy.
//
// A float32 operand becomes a pair of 16-bit floats.  Scaled by a power of two that
// brings the largest finite magnitude of its tensor to [2^8, 2^15), x is kept as
//   hi = f16(x),  lo = f16((x - hi) * 2^11),   x = hi + lo * 2^-11 within 2^-22 |x| or 2^-36
// (f16 ends at 2^-24, so an unscaled lo would end there; scaled, lo reaches 2^-35).  That
// holds a row or a column to 2^-24 of its largest element where that is 2^-12 at least, scaled.
// Of x and weight each row and each column is looked at while they are packed, and where one
// is not held so, beside others 2^20 times as large, the products of the call are float32
// products of the operands as they are (k_plain_products).  The logits' gradient, whose rows
// and classes do differ so much, has a scale a row (dx) or a class (dweight).
// The scale comes from a sample of the rows with 2^6 to spare, so that the packing reads
// the tensor once; it finds the largest magnitude on its way, and where that does not fit
// after all, a second packing with its own scale follows (k_pack<true>, which otherwise
// returns at once).  Against a pass of its own for the maximum: 64 rows, 131072 columns
// of length 2048: 839 -> 684 us for the loss; 16384 rows, 32000 columns of length 1024:
// 2636 -> 2585 us; within the noise where the products take most of the time.  Up to 1184
// rows of either tensor are all in the sample, which then is the largest magnitude.
// A product is three MMAs, hi.lo + lo.hi first and then hi.hi:
//   a.b = hi.hi + 2^-11 (hi.lo + lo.hi)          (lo.lo is below 2^-22)
// with the 2^-11 applied by the MMA itself (scale-input-d) when hi.hi is added.  f16
// MMAs run at twice the rate of the TF32 ones that a split in TF32 would need.
//
// The tensor core truncates its accumulator at every addition, which over a long K
// costs a part in 2^24 each time, always towards zero.  So 256 values of K stay in
// tensor memory at most: the epilogue warps read each piece of 256 and add it, rounded
// to nearest, to sums in registers, while the next piece runs in the other half of
// tensor memory.  A piece is the cross terms of its four blocks of 64, then the hi.hi of
// all four.  (Pieces of 64 were 20 % slower than of 128: a piece's hand-over, from the MMAs'
// commit by way of the epilogues of both CTAs to the next MMA, takes some 1500 clocks and the
// reading 1900, which two pieces of 1536 clocks do not cover.  Pieces of 256 gain another 5 %:
// the reads of tensor memory share it with the MMAs, and under the power limit their energy
// is taken from the MMAs' clock.)
//
// All three products read the same packed operands, [row][64 columns][hi, lo], K-major
// or MN-major by the matrix descriptors alone:
//   logits   z  = x' w'^T   A = x' K-major,  B = w' K-major      softmax statistics in the epilogue,
//                                                                split along D when the tiles are few
//   dx       dx = g' w'     A = g' K-major,  B = w' MN-major     split along V when the tiles are few
//   dweight  dw = g'^T x'   A = g' MN-major, B = x' MN-major     added up over the pieces of the rows
// The logits of one piece of the rows are written once, as float32; k_softmax_grad
// turns them into g', 256 bytes of z into 128 of hi and 128 of lo, on one scale a row for dx and
// on one a class and 256 rows for dweight.
//
// A pair of CTAs works on a 256 x 256 tile (tcgen05.mma.cta_group::2): each stages its
// own 128 rows of A and 128 columns of B, 64 KB for 1536 clocks of MMAs.  The lo halves
// are free after a piece's cross terms, the hi halves only at its end, so each has a ring
// of its own: five stages of hi, two of lo, 32 KB each.  Warp 0 loads (TMA), warp 1 of the
// leader issues, warps 4..11 are the epilogue: two warps for each quarter of the tensor
// memory's lanes, 128 columns each, with 208 registers a thread (128 sums, 64 of a load in
// flight) that the first four warps give up.  A lane holds a row and stores it itself, a
// 32-byte sector at a time: the 32 KB of shared memory that would make whole lines of it are
// worth more as a stage.  Results whose rows allow no such stores go by way of a padded
// workspace.
// Bound by the MMAs and, in long calls, by the power limit: 4096 x 32000 x 2048 takes 1183 us
// for the logits (1265 with a bias) and 1131 and 1153 us for dx and dweight, 454 to 475 TFLOP/s
// of products (three times that of MMAs) with the tensor pipe active in 75, 84 and 82 % of the time.
// Every wait is bounded; on expiry the device error word is set and the roles leave.
#include <cuda_fp16.h>

#include <climits>
#include <cstring>

#include "linear_ce.cuh"
#include "tcgen05.cuh"

namespace mtc {
namespace {

constexpr int kBlock = 64;                       // columns of a packed block: 64 hi, 64 lo, 256 bytes
constexpr int kTileRows = 256, kTileCols = 256;  // of a CTA pair
constexpr int kOperandBytes = 16384;             // 128 rows (or columns) x 64 of K, hi or lo
constexpr int kStageBytes = 2 * kOperandBytes;   // A and B
constexpr int kHiStages = 5, kLoStages = 2;
constexpr int kStages = kHiStages + kLoStages;
constexpr int kPieceBlocks = 4;                  // blocks of K that are summed in tensor memory
constexpr int kSmemBytes = kStages * kStageBytes + 1024 + 256;
constexpr int kCtaThreads = 384;
constexpr int kEpilogueRegs = 208, kOtherRegs = 88;
static_assert(kSmemBytes <= 227 * 1024, "shared memory per CTA");
static_assert(256 * kEpilogueRegs + 128 * kOtherRegs <= kCtaThreads * 168, "registers of the launch (168 a thread)");
constexpr uint32_t kTmemCols = 512;

// ---------------------------------------------------------------- packing --

// Largest finite magnitude of a tensor -> the exponent of its scale.
__device__ __forceinline__ int scale_exponent(int amax_bits) {
    const float amax = __int_as_float(amax_bits);
    if (amax == 0.0f) return 0;
    int e;
    frexpf(amax, &e);  // amax = m 2^e, 1/2 <= m < 1
    const int s = 15 - e;
    return s < 126 ? s : 126;
}

// (the exponents of the scales lie in [-119, 126])
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }

// Four neighbouring columns of a packed block: hi, and lo 64 columns on.
__device__ __forceinline__ void store_pairs(__half *to, float x0, float x1, float x2, float x3) {
    const __half2 h0 = __floats2half2_rn(x0, x1), h1 = __floats2half2_rn(x2, x3);
    const float2 f0 = __half22float2(h0), f1 = __half22float2(h1);
    const __half2 l0 = __floats2half2_rn((x0 - f0.x) * 2048.0f, (x1 - f0.y) * 2048.0f);
    const __half2 l1 = __floats2half2_rn((x2 - f1.x) * 2048.0f, (x3 - f1.y) * 2048.0f);
    *reinterpret_cast<uint2 *>(to) =
        make_uint2(*reinterpret_cast<const uint32_t *>(&h0), *reinterpret_cast<const uint32_t *>(&h1));
    *reinterpret_cast<uint2 *>(to + kBlock) =
        make_uint2(*reinterpret_cast<const uint32_t *>(&l0), *reinterpret_cast<const uint32_t *>(&l1));
}

// What the device knows of the scales of x and weight, behind the count of the live rows.
// kWide: the pairs would not hold x and weight; kRepacked: the second packing counts.
enum Known { kLargest = 1, kSampled = 3, kExponent = 5, kWide = 7, kRepacked = 8 };
static_assert(kRepacked + 2 == kLiveKnown, "zeroed with the count");

// Whether the pairs hold a tensor.  With a scaled x off by 2^-36 at most, a row or a column is
// held to 2^-24 of its largest element, as float32 would round that one, where an element of it
// reaches 2^-12.  Beside the largest of the tensor, scaled to 2^8 at least, such a row may be
// smaller by 2^20.  A byte each says whether the row (column) has an element that large and
// whether it has any at all that is finite and not zero: one that has but the latter makes the
// products go by float32 (plain_sums).
constexpr float kHeld = 0x1p-12f;
struct Held {
    unsigned char *row_ok, *row_some, *col_ok, *col_some;
    int64_t rows16, cols16;  // their lengths in 16 bytes
};

struct PackSource {
    const float *p;
    int64_t rs, cs;
    int64_t rows, cols;
    const int *map;   // rows by way of the list of live rows; null: as they are
    const int *live;  // their count; null: all
    int vec;          // float4 loads
    __half *to;       // [rows_out][blocks][2][64]
    int64_t rows_out; // with zero rows behind the live ones, up to a multiple of 64
    int which;        // 0: x, 1: weight
    Held held[2];     // by the first packing, and by the second
};

struct PackArgs {
    PackSource s[2];
    int64_t first_of_second;  // blocks of the grid before the second tensor
    int *known;               // the live rows' count and what follows it
    uint4 *flags;             // all of Held's bytes, to be zeroed
    int64_t flags16;
    int headroom;             // powers of two above the sample; 0: it is the whole
    float *dx;                // its rows without a loss become zero; null: not wanted
    int64_t dx_rs, dx_cs;
    int dx_vec;
};

__device__ __forceinline__ void keep_max(float v, int *to) {
    int bits = __float_as_int(v);
    bits = __reduce_max_sync(0xFFFFFFFFu, bits);  // magnitudes order as their bits
    __shared__ int part[8];
    __syncthreads();
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = bits;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 8; ++i) bits = max(bits, part[i]);
        if (bits > 0) atomicMax(to, bits);
    }
}

__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a <= 3.402823466e38f ? a : 0.0f;
}

__device__ __forceinline__ int64_t source_rows(const PackSource &s) {
    return s.live != nullptr ? (*s.live < s.rows ? *s.live : s.rows) : s.rows;
}

__device__ __forceinline__ const float *source_row(const PackSource &s, int64_t r) {
    return s.p + (s.map != nullptr ? s.map[r] : r) * s.rs;
}

// The scale of the first packing: the sampled maximum to [2^8, 2^9).
__device__ __forceinline__ int first_exponent(const PackArgs &a, int which) {
    const int sampled = a.known[kSampled + which];
    return sampled == 0 ? 0 : scale_exponent(sampled) - a.headroom;
}

// And the one that counts: the same, unless the largest magnitude needs a smaller one (or
// the sample was all zeros).
__device__ __forceinline__ int last_exponent(const PackArgs &a, int which) {
    const int exact = scale_exponent(a.known[kLargest + which]);
    if (a.known[kSampled + which] == 0) return exact;
    const int first = first_exponent(a, which);
    return first < exact ? first : exact;
}

// Largest finite magnitudes of x (rows with a loss) and weight over a sample of the rows, one
// a warp; the zero rows of dx, and Held's zeroes.  7 to 30 us for 1184 rows of 1024 to 8192 columns,
// a warp's latency.
__global__ void __launch_bounds__(256) k_sample(const PackArgs a) {
    wait_for_previous();
    const bool second = blockIdx.x >= a.first_of_second;
    const PackSource &s = a.s[second];
    const int64_t block = second ? blockIdx.x - a.first_of_second : blockIdx.x;
    const int64_t blocks = second ? gridDim.x - a.first_of_second : a.first_of_second;
    const int lane = threadIdx.x % 32;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < a.flags16; i += gridDim.x * 256)
        a.flags[i] = make_uint4(0, 0, 0, 0);
    float m0 = 0.0f, m1 = 0.0f;
    const int64_t rows = source_rows(s);
    const int64_t warp_at = block * 8 + threadIdx.x / 32, warps = blocks * 8;
    if (warp_at < rows) {
        const float *src = source_row(s, rows > warps ? warp_at * rows / warps : warp_at);
        if (s.vec) {
            const float4 *v4 = reinterpret_cast<const float4 *>(src);
            const int n4 = static_cast<int>(s.cols / 4);
            int c = lane;
            for (; c + 96 < n4; c += 128) {
                float4 v[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) v[u] = __ldg(v4 + c + 32 * u);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    m0 = fmaxf(m0, fmaxf(finite_abs(v[u].x), finite_abs(v[u].y)));
                    m1 = fmaxf(m1, fmaxf(finite_abs(v[u].z), finite_abs(v[u].w)));
                }
            }
            for (; c < n4; c += 32) {
                const float4 v = __ldg(v4 + c);
                m0 = fmaxf(m0, fmaxf(finite_abs(v.x), finite_abs(v.y)));
                m1 = fmaxf(m1, fmaxf(finite_abs(v.z), finite_abs(v.w)));
            }
        } else {
            int64_t c = lane;
            for (; c + 480 < s.cols; c += 512) {
                float v[16];
#pragma unroll
                for (int u = 0; u < 16; ++u) v[u] = __ldg(src + (c + 32 * u) * s.cs);
#pragma unroll
                for (int u = 0; u < 16; u += 2) {
                    m0 = fmaxf(m0, finite_abs(v[u]));
                    m1 = fmaxf(m1, finite_abs(v[u + 1]));
                }
            }
            float v[16];
#pragma unroll
            for (int u = 0; u < 16; ++u) v[u] = c + 32 * u < s.cols ? __ldg(src + (c + 32 * u) * s.cs) : 0.0f;
#pragma unroll
            for (int u = 0; u < 16; ++u) m0 = fmaxf(m0, finite_abs(v[u]));
        }
    }
    keep_max(fmaxf(m0, m1), a.known + kSampled + s.which);
    if (a.dx != nullptr) {
        const PackSource &x = a.s[0];
        const int64_t dead = x.rows - source_rows(x);
        const int64_t warp = static_cast<int64_t>(blockIdx.x) * 8 + threadIdx.x / 32;
        for (int64_t i = warp; i < dead; i += static_cast<int64_t>(gridDim.x) * 8) {
            float *to = a.dx + x.map[x.rows - 1 - i] * a.dx_rs;
            if (a.dx_vec) {
                for (int64_t c = lane; c < x.cols / 4; c += 32) reinterpret_cast<float4 *>(to)[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            } else {
                for (int64_t c = lane; c < x.cols; c += 32) to[c * a.dx_cs] = 0.0f;
            }
        }
    }
}

// Sets the bytes of four columns with these largest elements.  Nothing is read: a read of bytes
// that others are setting waits for them (2928 rows of 174: 9 us more).
__device__ __forceinline__ void mark_columns(const Held &h, int64_t c, float4 largest, float enough) {
    const float x[4] = {largest.x, largest.y, largest.z, largest.w};
    if (x[0] >= enough && x[1] >= enough && x[2] >= enough && x[3] >= enough) {
        *reinterpret_cast<unsigned int *>(h.col_ok + c) = 0x01010101u;
        return;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (x[k] > 0.0f) (x[k] >= enough ? h.col_ok : h.col_some)[c + k] = 1;
}

// Each half-warp packs one block of 64 columns of four rows in every so many: a lane four columns.
// AGAIN: only the tensors whose scale was wrong; and the exponents are written down.  Bound by
// HBM, 8 bytes an element: 36096 rows of 2048 in 96 us (6.2 TB/s).
template <bool AGAIN>
__global__ void __launch_bounds__(256) k_pack(const PackArgs a) {
    wait_for_previous();
    if ((AGAIN || a.headroom == 0) && blockIdx.x == 0 && threadIdx.x < 2)
        a.known[kExponent + threadIdx.x] = AGAIN ? last_exponent(a, threadIdx.x) : first_exponent(a, threadIdx.x);
    const bool second = blockIdx.x >= a.first_of_second;
    const PackSource &s = a.s[second];
    const int block = static_cast<int>(second ? blockIdx.x - a.first_of_second : blockIdx.x);
    const int grid = static_cast<int>(second ? gridDim.x - a.first_of_second : a.first_of_second);
    const int64_t blocks = (s.cols + kBlock - 1) / kBlock;
    const int64_t rows = source_rows(s);
    const int64_t rows_out = s.live != nullptr && (rows + 63) / 64 * 64 < s.rows_out ? (rows + 63) / 64 * 64 : s.rows_out;
    const int e = AGAIN ? last_exponent(a, s.which) : first_exponent(a, s.which);
    if (AGAIN && (e == first_exponent(a, s.which) || a.known[kLargest + s.which] == 0)) {
        return;
    }
    if (AGAIN && block == 0 && threadIdx.x == 0) a.known[kRepacked + s.which] = 1;
    const Held &held = s.held[AGAIN];
    const float f = power_of_two(e), enough = kHeld * power_of_two(-e);  // of an element as it is
    const int lane = threadIdx.x % 16;
    const unsigned int mates = 0xFFFFu << (threadIdx.x & 16);
    float largest = 0.0f;
    constexpr int U = 4;
    const int halves = grid * 16;
    const int abreast = blocks < halves ? static_cast<int>(blocks) : halves;  // half-warps along a row
    const int step = abreast > 0 ? halves / abreast : 0;                      // rows at a time
    const int half = block * 16 + threadIdx.x / 16;
    const int at = abreast > 0 ? half % abreast : 0, r_first = abreast > 0 ? half / abreast : 0;
    for (int64_t b0 = 0; b0 < blocks; b0 += abreast) {
        const int64_t b = b0 + at, c = b * kBlock + lane * 4;
        const bool mine = b < blocks && r_first < step, reads = mine && c < s.cols;
        float col[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int64_t r0 = 0; r0 < rows_out; r0 += static_cast<int64_t>(step) * U) {
            float4 v[U];
            unsigned int rows_ok = 0;  // a byte a row, of the half-warp's
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t r = r0 + r_first * U + u;
                v[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (!reads || r >= rows) continue;
                const float *src = source_row(s, r);
                if (s.vec) {
                    v[u] = __ldg(reinterpret_cast<const float4 *>(src + c));
                } else {
                    v[u].x = __ldg(src + c * s.cs);
                    if (c + 1 < s.cols) v[u].y = __ldg(src + (c + 1) * s.cs);
                    if (c + 2 < s.cols) v[u].z = __ldg(src + (c + 2) * s.cs);
                    if (c + 3 < s.cols) v[u].w = __ldg(src + (c + 3) * s.cs);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t r = r0 + r_first * U + u;
                float4 m = v[u];  // its magnitudes: a maximum passes NaN over, and infinities are taken out
                float top = fmaxf(fmaxf(fabsf(m.x), fabsf(m.y)), fmaxf(fabsf(m.z), fabsf(m.w)));
                if (isinf(top)) {
                    m = make_float4(finite_abs(m.x), finite_abs(m.y), finite_abs(m.z), finite_abs(m.w));
                    top = fmaxf(fmaxf(m.x, m.y), fmaxf(m.z, m.w));
                }
                col[0] = fmaxf(col[0], fabsf(m.x));
                col[1] = fmaxf(col[1], fabsf(m.y));
                col[2] = fmaxf(col[2], fabsf(m.z));
                col[3] = fmaxf(col[3], fabsf(m.w));
                const unsigned int ok = __ballot_sync(0xFFFFFFFFu, top >= enough) & mates;
                const unsigned int some = __ballot_sync(0xFFFFFFFFu, top > 0.0f) & mates;
                rows_ok |= (ok != 0 ? 1u : 0u) << (8 * u);
                if (!mine || r >= rows_out) continue;
                if (lane == 0 && some != 0 && ok == 0) held.row_some[r] = 1;
                store_pairs(s.to + (r * blocks + b) * 2 * kBlock + lane * 4, v[u].x * f, v[u].y * f, v[u].z * f,
                            v[u].w * f);
            }
            // (bytes that are not set stay as another half-warp may have set them)
            const int64_t r = r0 + r_first * U;
            if (lane == 0 && rows_ok == 0x01010101u) {
                *reinterpret_cast<unsigned int *>(held.row_ok + r) = rows_ok;
            } else if (lane == 0) {
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (rows_ok >> (8 * u) & 1) held.row_ok[r + u] = 1;
            }
        }
        largest = fmaxf(largest, fmaxf(fmaxf(col[0], col[1]), fmaxf(col[2], col[3])));
        // of half-warps of this CTA that have the same columns the first speaks for all
        __shared__ float4 columns[16][16];
        const int group = threadIdx.x / 16;
        float4 all = make_float4(col[0], col[1], col[2], col[3]);
        if (abreast < 16) {
            columns[group][lane] = mine ? all : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            __syncthreads();
            for (int o = group + abreast; group < abreast && o < 16; o += abreast) {
                const float4 x = columns[o][lane];
                all = make_float4(fmaxf(all.x, x.x), fmaxf(all.y, x.y), fmaxf(all.z, x.z), fmaxf(all.w, x.w));
            }
        }
        if (mine && group < abreast) mark_columns(held, c, all, enough);
    }
    if (!AGAIN && a.headroom != 0) keep_max(largest, a.known + kLargest + s.which);
}

// ---------------------------------------------------------------- products --

enum class Out { Logits, Sum };

// An operand as float32, wherever it lies: element k of row r at map[r] rs + map[k] ks.
struct Plain {
    const float *p;
    int64_t rs, ks;
    const int *rows, *ks_map;  // null: as they are
};

struct TileArgs {
    int64_t M, N, K;  // M or K: of the piece, of which the first live ones count
    const int *live;
    int64_t first;
    bool live_k;      // the live rows bound K instead of M
    int tiles_n;
    int group;        // row tiles that share a sweep of the columns
    int splits;       // of K
    // Exponents of the operands' scales: one for a packed tensor, and of g' one a row as the rows
    // of dx, or one a class and piece of K as the rows of dweight.
    const int *exp_a, *exp_b;
    int64_t exp_pitch;  // [pieces][exp_pitch]
    int *wide;          // set: float32 products of the operands themselves
    bool judges;        // whether that is so is found out in this launch, next to the products
    Held held[2][2];    // by x and weight, and by the packing
    const int *repacked;  // [2]
    Plain a, b;
    unsigned long long *err;
    // Logits
    float *z;         // [M][z_pitch], null: statistics alone
    int64_t z_pitch;
    const float *bias;
    int64_t bias_s;
    const int *target;
    float *part_max, *part_rest;  // [M][2 tiles_n], see Softmax
    float *z_target;              // [M]
    // Sum
    float *out;       // rows of 32-byte sectors
    int64_t out_rs;
    const int *out_map;
    int add;
    float *parts;     // the splits' partial results [splits][M][parts_pitch]; null: straight to out
    int64_t parts_pitch;
};

__device__ __forceinline__ void tma_load_operand(void *dst, const CUtensorMap *map, uint32_t leader_bar, int row, int block,
                                                 int lo) {
    asm volatile(
        "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(leader_bar), "r"(0), "r"(row), "r"(block), "r"(lo)
        : "memory");
}

// Shared-memory matrix descriptor, 128-byte swizzle, version 1 (bit 46).  K-major: rows
// of 128 bytes, eight rows 1024 bytes.  MN-major: 64 columns a row of 128 bytes, eight
// rows of K 1024 bytes, the next 64 columns 8192 bytes on (64 rows of K).
template <bool MN>
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
    return ((addr & 0x3FFFFull) >> 4) | ((MN ? 8192ull >> 4 : 1ull) << 16) | ((1024ull >> 4) << 32) | (1ull << 46) |
           (2ull << 61);
}

// D = F32, A = B = F16, M = 256 (two CTAs), N = 256.
template <bool A_MN, bool B_MN>
__device__ __forceinline__ constexpr uint32_t instr_desc() {
    return (1u << 4) | (A_MN ? 1u << 15 : 0u) | (B_MN ? 1u << 16 : 0u) | (uint32_t(kTileCols >> 3) << 17) |
           (uint32_t(kTileRows >> 4) << 24);
}

__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// D = A B + D 2^-11
__device__ __forceinline__ void mma_pair_scaled(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p, 11;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(1)
        : "memory");
}

struct Extent {
    int64_t tiles_m, tiles, units;
    int kblocks, per_split;
    int64_t M, K;
};

__device__ __forceinline__ Extent extent_of(const TileArgs &a) {
    Extent e;
    int64_t K = a.K;
    e.M = a.M;
    if (a.live != nullptr) {
        if (a.live_k) K = live_extent(a.live, a.first, K);
        else e.M = live_extent(a.live, a.first, e.M);
    }
    e.K = K;
    e.kblocks = static_cast<int>((K + kBlock - 1) / kBlock);
    e.tiles_m = (e.M + kTileRows - 1) / kTileRows;
    e.tiles = e.tiles_m * a.tiles_n;
    e.units = e.tiles * a.splits;
    if (a.live_k && K == 0 && a.first > 0) e.units = 0;  // nothing left to add
    e.per_split = (e.kblocks + a.splits - 1) / a.splits;
    if (a.live_k) e.per_split = (e.per_split + kPieceBlocks - 1) / kPieceBlocks * kPieceBlocks;  // the pieces of g'
    return e;
}

// Unit u: split u / tiles (the tiles of a split run next to one another and share
// their panels in L2), and its tile in groups of row tiles.
__device__ __forceinline__ void unit_of(const TileArgs &a, const Extent &e, int64_t u, int &tm, int &tn, int &split,
                                        int &kb0, int &kb1) {
    split = static_cast<int>(u / e.tiles);
    const int64_t t = u - split * e.tiles;
    const int64_t span = static_cast<int64_t>(a.group) * a.tiles_n;
    const int64_t g = t / span;
    const int64_t first_m = g * a.group;
    const int64_t size = e.tiles_m - first_m < a.group ? e.tiles_m - first_m : a.group;
    const int64_t in_group = t - g * span;
    tm = static_cast<int>(first_m + in_group % size);
    tn = static_cast<int>(in_group / size);
    kb0 = split * e.per_split;
    kb1 = kb0 + e.per_split < e.kblocks ? kb0 + e.per_split : e.kblocks;
    if (kb1 < kb0) kb1 = kb0;
}

__device__ __forceinline__ void tmem_ld64(uint32_t taddr, uint32_t (&r)[64]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
        "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
        "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
          "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
          "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
          "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
          "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void store8(float *to, const float *v) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "f"(v[0]), "f"(v[1]), "f"(v[2]),
                 "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                 : "memory");
}

__device__ __forceinline__ void load8(const float *from, float (&v)[8]) {
    asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                 : "l"(from)
                 : "memory");
}

// The first n of a lane's 128 columns to its row, whole sectors.
__device__ __forceinline__ void store_row(float *to, float (&acc)[128], int n, bool add) {
#pragma unroll
    for (int j = 0; j < 128; j += 8) {
        if (j >= n) break;
        if (add) {
            float old[8];
            load8(to + j, old);
#pragma unroll
            for (int k = 0; k < 8; ++k) acc[j + k] += old[k];
        }
        store8(to + j, acc + j);
    }
}

// x 2^e in place; e beyond float32's exponents takes a second factor.
__device__ __forceinline__ void rescale(float (&acc)[128], float f0, float f1) {
#pragma unroll
    for (int j = 0; j < 128; ++j) acc[j] *= f0;
    if (f1 != 1.0f) {
#pragma unroll
        for (int j = 0; j < 128; ++j) acc[j] *= f1;
    }
}

// The logits' epilogue: this lane's row, 128 columns from col0 on.  What most tiles do
// not need (a ragged end, a bias, the target) is kept out of the loops of the others.
__device__ __forceinline__ void store_logits(const TileArgs &a, int64_t M, float (&acc)[128], int64_t row, int64_t col0,
                                             int part, float f0, float f1) {
    if (col0 >= a.N) return;
    const int n = static_cast<int>(a.N - col0 < 128 ? a.N - col0 : 128);
    const bool live = row < M;
    rescale(acc, f0, f1);
    if (a.bias != nullptr) {
#pragma unroll
        for (int j = 0; j < 128; ++j)
            if (j < n) acc[j] += __ldg(a.bias + (col0 + j) * a.bias_s);
    }
    if (n < 128) {
#pragma unroll
        for (int j = 0; j < 128; ++j)
            if (j >= n) acc[j] = -INFINITY;
    }
    const int target = live ? a.target[a.first + row] - static_cast<int>(col0) : -1;
    if (target >= 0 && target < n) {
        float zt = 0.0f;
#pragma unroll
        for (int j = 0; j < 128; ++j)
            if (j == target) zt = acc[j];
        a.z_target[row] = zt;
    }
    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < 128; ++j) top[j % 4] = fmaxf(top[j % 4], acc[j]);
    top[0] = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
    // exp by the hardware's 2^x (2^-22): its error and the product's weigh little in a sum
    // whose largest terms have arguments near zero
    const float base = isinf(top[0]) ? 0.0f : top[0];
    float sum[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < 128; ++j) sum[j % 8] += __expf(acc[j] - base);
    auto total = [&] { return ((sum[0] + sum[1]) + (sum[2] + sum[3])) + ((sum[4] + sum[5]) + (sum[6] + sum[7])); };
    float rest = total() - 1.0f;
    // The 1 costs the others of its eighth digits where they are little next to it: then these are
    // summed again, without the one logit that is the largest.  (Every tile waits for the slowest of
    // its 16 warps.  3000 x 32000 x 1024, logits of deviation 2, which leaves 1 of 1700 rows of 128 so:
    // 501 us for the logits; 534 from 1/8 on and with all eighths summed again; 485 not at all.)
    if (rest < 0.0625f && !isinf(top[0])) {
        float again = base;
        asm volatile("" : "+f"(again));  // or the first sum's exponentials are kept, in memory
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            bool here = false;
#pragma unroll
            for (int j = k; j < 128; j += 8) here |= acc[j] == again;
            if (!here) continue;
            sum[k] = 0.0f;
#pragma unroll
            for (int j = k; j < 128; j += 8)
                if (acc[j] != again) sum[k] += __expf(acc[j] - again);
        }
        rest = total();
    }
    if (live) {
        a.part_max[row * 2 * a.tiles_n + part] = top[0];
        a.part_rest[row * 2 * a.tiles_n + part] = rest;
    }
    // rows are padded to 64 columns: the last sector of a ragged end may reach behind V
    if (a.z != nullptr && live) store_row(a.z + row * a.z_pitch + col0, acc, n, false);
}

__device__ __forceinline__ void store_sum(const TileArgs &a, int64_t M, float (&acc)[128], int64_t row, int64_t col0,
                                          int split, float f0, float f1) {
    if (row >= M || col0 >= a.N) return;
    const int n = static_cast<int>(a.N - col0 < 128 ? a.N - col0 : 128);
    rescale(acc, f0, f1);
    if (a.parts != nullptr) store_row(a.parts + (split * a.M + row) * a.parts_pitch + col0, acc, n, false);
    else store_row(a.out + (a.out_map != nullptr ? a.out_map[a.first + row] : row) * a.out_rs + col0, acc, n, a.add);
}

// Looks the bytes over, 16 at a time, a share of them a thread.
__device__ __forceinline__ void judge(const Held &h, int64_t at, int64_t step, int *wide) {
    bool bad = false;
    auto look = [&](const unsigned char *ok, const unsigned char *some, int64_t n) {
        for (int64_t i = at; i < n; i += step) {
            const uint4 o = __ldcg(reinterpret_cast<const uint4 *>(ok) + i), m = __ldcg(reinterpret_cast<const uint4 *>(some) + i);
            bad |= ((m.x & ~o.x) | (m.y & ~o.y) | (m.z & ~o.z) | (m.w & ~o.w)) != 0;
        }
    };
    look(h.row_ok, h.row_some, h.rows16);
    look(h.col_ok, h.col_some, h.cols16);
    if (bad) atomicOr(wide, 1);
}

template <bool A_MN, bool B_MN, Out MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kCtaThreads, 1)
    k_pair_product(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                   const TileArgs args) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    // the same aligned offset in both CTAs (same dynamic size, same static layout)
    unsigned char *smem =
        reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + kStages * kStageBytes);  // leader's: both CTAs' bytes
    uint64_t *empty = full + kStages;    // each CTA's: the stage's MMAs are done (hi stages first, then lo)
    uint64_t *acc_full = empty + kStages;  // [2] each CTA's: a piece is in tensor memory
    uint64_t *acc_empty = acc_full + 2;    // [2] leader's: both epilogues have read it
    uint64_t *drain = acc_empty + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t rank = cluster_rank();
    const bool leader = rank == 0;
    const int64_t cluster = blockIdx.x / 2, clusters = gridDim.x / 2;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], 16);  // 8 epilogue warps x 2 CTAs
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(kTmemCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // the peer's barriers are initialised before any remote arrive
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    wait_for_previous();
    Extent e = extent_of(args);
    if (!args.judges && *args.wide != 0) e.units = 0;  // k_plain_products'

    if (warp >= 4) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpilogueRegs));
        const int quadrant = warp % 4, half = (warp - 4) / 4;
        const uint32_t release[2] = {peer_addr(&acc_empty[0], 0), peer_addr(&acc_empty[1], 0)};
        const int exp_b = *args.exp_b;
        int64_t piece = 0;
        bool ok = true;
        for (int64_t u = cluster; u < e.units && ok; u += clusters) {
            int tm, tn, split, kb0, kb1;
            unit_of(args, e, u, tm, tn, split, kb0, kb1);
            const int64_t row = static_cast<int64_t>(tm) * kTileRows + rank * 128 + quadrant * 32 + lane;
            float acc[128];
#pragma unroll
            for (int j = 0; j < 128; ++j) acc[j] = 0.0f;
            for (int kb = kb0; kb < kb1; kb += kPieceBlocks, ++piece) {
                const int b = static_cast<int>(piece & 1);
                float unscale = 1.0f;  // of a class's row in this piece
                if (A_MN && row < e.M)
                    unscale = power_of_two(-args.exp_a[static_cast<int64_t>(kb / kPieceBlocks) * args.exp_pitch + row]);
                if (!mbar_wait(&acc_full[b], static_cast<uint32_t>(piece >> 1) & 1u, abort_flag)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t at = tmem_base + (static_cast<uint32_t>(quadrant * 32) << 16) +
                                    static_cast<uint32_t>(b * kTileCols + half * 128);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t v[64];
                    tmem_ld64(at + static_cast<uint32_t>(c * 64), v);
#pragma unroll
                    for (int j = 0; j < 64; ++j)
                        acc[c * 64 + j] = A_MN ? fmaf(__uint_as_float(v[j]), unscale, acc[c * 64 + j])
                                               : acc[c * 64 + j] + __uint_as_float(v[j]);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_remote(release[b]);
            }
            if (!ok) break;
            const int scale = -exp_b - (A_MN ? 0 : B_MN ? args.exp_a[row < e.M ? row : 0] : *args.exp_a);
            const int most = scale < -126 ? -126 : scale > 126 ? 126 : scale;
            const float f0 = power_of_two(most), f1 = power_of_two(scale - most);
            const int64_t col0 = static_cast<int64_t>(tn) * kTileCols + half * 128;
            if (MODE == Out::Logits) store_logits(args, e.M, acc, row, col0, tn * 2 + half, f0, f1);
            else store_sum(args, e.M, acc, row, col0, split, f0, f1);
            __syncwarp();
        }
        if (!ok) atomicCAS(args.err, 0ull, static_cast<unsigned long long>(MTC_ERR_RUNTIME));
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == 0) {
            if (lane == 0) {
                int64_t it = 0;
                bool ok = true;
                for (int64_t u = cluster; u < e.units && ok; u += clusters) {
                    int tm, tn, split, kb0, kb1;
                    unit_of(args, e, u, tm, tn, split, kb0, kb1);
                    const int a0 = tm * kTileRows + static_cast<int>(rank) * 128;
                    const int b0 = tn * kTileCols + static_cast<int>(rank) * 128;
                    for (int kb = kb0; kb < kb1 && ok; ++kb, ++it) {
                        for (int lo = 0; lo < 2; ++lo) {
                            const int depth = lo ? kLoStages : kHiStages;
                            const int s = (lo ? kHiStages : 0) + static_cast<int>(it % depth);
                            if (!mbar_wait(&empty[s], (static_cast<uint32_t>(it / depth) & 1u) ^ 1u, abort_flag)) {
                                ok = false;
                                break;
                            }
                            unsigned char *st = smem + s * kStageBytes;
                            if (leader) mbar_expect_tx(&full[s], 2 * kStageBytes);
                            const uint32_t fb = peer_addr(&full[s], 0);
                            tma_load_operand(st, &map_a, fb, A_MN ? kb * kBlock : a0, A_MN ? a0 / kBlock : kb, lo);
                            tma_load_operand(st + kOperandBytes, &map_b, fb, B_MN ? kb * kBlock : b0,
                                             B_MN ? b0 / kBlock : kb, lo);
                        }
                    }
                }
                if (!ok) atomicCAS(args.err, 0ull, static_cast<unsigned long long>(MTC_ERR_RUNTIME));
                if (leader) {  // every stage issued by the pair has landed before the cluster exits
                    for (int lo = 0; lo < 2; ++lo) {
                        const int depth = lo ? kLoStages : kHiStages;
                        for (int64_t d = it > depth ? it - depth : 0; d < it; ++d) {
                            uint64_t *bar = &full[(lo ? kHiStages : 0) + d % depth];
                            const uint32_t round = static_cast<uint32_t>(d / depth);
                            for (long long i = 0; i < kWaitLimit && !mbar_try_wait(bar, round & 1u); ++i) {
                            }
                        }
                    }
                }
            }
        } else if (warp >= 2) {
            if (!A_MN && !B_MN && args.judges) {
                const int64_t at = static_cast<int64_t>(blockIdx.x) * 64 + threadIdx.x - 64, step = static_cast<int64_t>(gridDim.x) * 64;
#pragma unroll 1
                for (int which = 0; which < 2; ++which)
                    judge(args.repacked[which] ? args.held[which][1] : args.held[which][0], at, step, args.wide);
            }
        } else if (warp == 1) {
            if (lane == 0 && leader) {
                constexpr uint32_t idesc = instr_desc<A_MN, B_MN>();
                constexpr uint64_t a_step = (A_MN ? 2048 : 32) >> 4, b_step = (B_MN ? 2048 : 32) >> 4;  // 16 of K
                int64_t it = 0, piece = 0;
                bool ok = true;
                for (int64_t u = cluster; u < e.units && ok; u += clusters) {
                    int tm, tn, split, kb0, kb1;
                    unit_of(args, e, u, tm, tn, split, kb0, kb1);
                    for (int kb = kb0; kb < kb1 && ok; kb += kPieceBlocks, ++piece) {
                        const int n = kb1 - kb < kPieceBlocks ? kb1 - kb : kPieceBlocks;
                        const int b = static_cast<int>(piece & 1);
                        if (!mbar_wait(&acc_empty[b], (static_cast<uint32_t>(piece >> 1) & 1u) ^ 1u, abort_flag)) {
                            ok = false;
                            break;
                        }
                        const uint32_t d = tmem_base + static_cast<uint32_t>(b * kTileCols);
                        for (int j = 0; j < n; ++j) {
                            const int sh = static_cast<int>((it + j) % kHiStages);
                            const int sl = kHiStages + static_cast<int>((it + j) % kLoStages);
                            if (!mbar_wait(&full[sh], static_cast<uint32_t>((it + j) / kHiStages) & 1u, abort_flag) ||
                                !mbar_wait(&full[sl], static_cast<uint32_t>((it + j) / kLoStages) & 1u, abort_flag)) {
                                ok = false;
                                break;
                            }
                            tc_fence_after();
                            const uint32_t hi = smem_u32(smem + sh * kStageBytes), lo = smem_u32(smem + sl * kStageBytes);
                            const uint64_t ah = operand_desc<A_MN>(hi), bh = operand_desc<B_MN>(hi + kOperandBytes);
                            const uint64_t al = operand_desc<A_MN>(lo), bl = operand_desc<B_MN>(lo + kOperandBytes);
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                mma_pair(d, ah + k * a_step, bl + k * b_step, idesc, j > 0 || k > 0);
                                mma_pair(d, al + k * a_step, bh + k * b_step, idesc, 1);
                            }
                            umma_commit_both(&empty[sl]);
                        }
                        if (!ok) break;
                        for (int j = 0; j < n; ++j) {
                            const int sh = static_cast<int>((it + j) % kHiStages);
                            const uint32_t hi = smem_u32(smem + sh * kStageBytes);
                            const uint64_t ah = operand_desc<A_MN>(hi), bh = operand_desc<B_MN>(hi + kOperandBytes);
                            if (j == 0) mma_pair_scaled(d, ah, bh, idesc);
                            else mma_pair(d, ah, bh, idesc, 1);
#pragma unroll
                            for (int k = 1; k < 4; ++k) mma_pair(d, ah + k * a_step, bh + k * b_step, idesc, 1);
                            umma_commit_both(&empty[sh]);
                        }
                        umma_commit_both(&acc_full[b]);
                        it += n;
                    }
                }
                if (!ok) atomicCAS(args.err, 0ull, static_cast<unsigned long long>(MTC_ERR_RUNTIME));
                umma_commit_pair_local(drain);  // all MMAs of the pair are done before either CTA frees tensor memory
                for (long long i = 0; i < kWaitLimit && !mbar_try_wait(drain, 0u); ++i) {
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // the leader's MMAs into this CTA's tensor memory have drained
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols));
    }
}

// The products in float32, on the FMA units, for operands whose rows or columns are of so unlike
// size that pairs on one scale lose the small ones: k_plain_products follows the logits' launch and
// the two gradients', and returns at once where the pairs hold (2 us; as a part of the same kernel
// it took 5 % of the tensor cores' time away).  The tiles, splits and results are the same.  The
// first four warps stage 16 columns of K at a time in one of two buffers while eight work on the
// other, 8 x 16 sums a thread, and make of them a row of 128 a lane by way of shared memory.  Bound by the FMAs and the
// waits of two warps a scheduler: 4096 x 32000 x 1024 in 11.9 ms for the loss and 34.7 with dx and
// dweight, 23 TFLOP/s, where pairs take 0.62 and 2.1 ms.
constexpr int kPlainK = 16, kPlainPitchA = 132, kPlainPitchB = 260;
constexpr int kPlainBuffer = kPlainK * (kPlainPitchA + kPlainPitchB);  // floats
constexpr int kPlainSmem = (2 * kPlainBuffer + 128 * kPlainPitchB) * 4;  // two buffers and the sums of a CTA
static_assert(kPlainSmem <= 227 * 1024, "shared memory per CTA");

__device__ __forceinline__ void plain_barrier() { asm volatile("bar.sync 1, 384;" ::: "memory"); }

struct PlainRange {
    int64_t begin, end;  // of K
    __device__ __forceinline__ PlainRange(const Extent &e, int kb0, int kb1) {
        begin = static_cast<int64_t>(kb0) * kBlock;
        end = static_cast<int64_t>(kb1) * kBlock < e.K ? static_cast<int64_t>(kb1) * kBlock : e.K;
    }
};

// ROWS rows of 16 columns of an operand; zeros beyond its ends.  128 threads, next to one another
// where the operand's elements are.
template <int ROWS>
__device__ __forceinline__ void stage_plain(const Plain &o, int64_t row0, int64_t rows, int64_t k0, int64_t k1, float *to,
                                            int pitch) {
    const bool along_k = o.ks == 1 || o.rs != 1;
    const int thread = threadIdx.x;
#pragma unroll 8
    for (int i = 0; i < ROWS / 8; ++i) {
        const int r = along_k ? thread / kPlainK + 8 * i : thread + 128 * (i % (ROWS / 128));
        const int k = along_k ? thread % kPlainK : i / (ROWS / 128);
        const int64_t row = row0 + r, col = k0 + k;
        const float *from = o.p;
        int bytes = 0;  // none: a zero
        if (row < rows && col < k1) {
            from += (o.rows != nullptr ? o.rows[row] : row) * o.rs + (o.ks_map != nullptr ? o.ks_map[col] : col) * o.ks;
            bytes = 4;
        }
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(to + k * pitch + r)), "l"(from), "r"(bytes)
                     : "memory");
    }
}

// `turn` counts the buffers filled (emptied) so far.  A buffer is filled again after the barrier
// behind which the other one is read, so after it has been read.
__device__ __forceinline__ void plain_stages(const TileArgs &a, const Extent &e, float *smem, int tm, int tn, int rank,
                                             PlainRange k, int &turn) {
    for (int64_t k0 = k.begin; k0 < k.end; k0 += kPlainK, ++turn) {
        float *as = smem + (turn & 1) * kPlainBuffer;
        stage_plain<128>(a.a, static_cast<int64_t>(tm) * kTileRows + rank * 128, e.M, k0, k.end, as, kPlainPitchA);
        stage_plain<256>(a.b, static_cast<int64_t>(tn) * kTileCols, a.N, k0, k.end, as + kPlainK * kPlainPitchA, kPlainPitchB);
        cp_async_wait_all();
        plain_barrier();
    }
}

__device__ __forceinline__ void plain_sums(float *smem, PlainRange k, int &turn, float (&acc)[128]) {
#pragma unroll
    for (int j = 0; j < 128; ++j) acc[j] = 0.0f;
    if (k.begin >= k.end) return;
    const int thread = threadIdx.x - 128, ty = thread / 16, tx = thread % 16;
    float2 two[8][8];  // rows, pairs of columns: two of a multiply-add (FFMA2)
#pragma unroll
    for (int r = 0; r < 8; ++r)
#pragma unroll
        for (int q = 0; q < 8; ++q) two[r][q] = make_float2(0.0f, 0.0f);
    for (int64_t k0 = k.begin; k0 < k.end; k0 += kPlainK, ++turn) {
        plain_barrier();
        const float *as = smem + (turn & 1) * kPlainBuffer + ty * 8;
        const float *bs = smem + (turn & 1) * kPlainBuffer + kPlainK * kPlainPitchA + tx * 4;
#pragma unroll 2
        for (int i = 0; i < kPlainK; ++i) {
            const float4 x0 = *reinterpret_cast<const float4 *>(as + i * kPlainPitchA);
            const float4 x1 = *reinterpret_cast<const float4 *>(as + i * kPlainPitchA + 4);
            const float x[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
            float4 y[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) y[q] = *reinterpret_cast<const float4 *>(bs + i * kPlainPitchB + 64 * q);
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                const float2 xx = make_float2(x[r], x[r]);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    two[r][2 * q] = __ffma2_rn(xx, make_float2(y[q].x, y[q].y), two[r][2 * q]);
                    two[r][2 * q + 1] = __ffma2_rn(xx, make_float2(y[q].z, y[q].w), two[r][2 * q + 1]);
                }
            }
        }
    }
    float *sums = smem + 2 * kPlainBuffer;
#pragma unroll
    for (int r = 0; r < 8; ++r)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *reinterpret_cast<float4 *>(sums + (ty * 8 + r) * kPlainPitchB + tx * 4 + 64 * q) =
                make_float4(two[r][2 * q].x, two[r][2 * q].y, two[r][2 * q + 1].x, two[r][2 * q + 1].y);
    asm volatile("bar.sync 2, 256;" ::: "memory");  // the eight warps alone
    const float *mine = sums + (thread % 128) * kPlainPitchB + thread / 128 * 128;
#pragma unroll
    for (int j = 0; j < 128; j += 4) {
        const float4 v = *reinterpret_cast<const float4 *>(mine + j);
        acc[j] = v.x;
        acc[j + 1] = v.y;
        acc[j + 2] = v.z;
        acc[j + 3] = v.w;
    }
}

template <Out MODE>
__device__ __forceinline__ void plain_product(const TileArgs &args, float *smem, int &turn) {
    const Extent e = extent_of(args);
    const int warp = threadIdx.x / 32, half = (warp - 4) / 4, rank = blockIdx.x % 2;
    for (int64_t u = blockIdx.x / 2; u < e.units; u += gridDim.x / 2) {
        int tm, tn, split, kb0, kb1;
        unit_of(args, e, u, tm, tn, split, kb0, kb1);
        if (warp < 4) {
            plain_stages(args, e, smem, tm, tn, rank, PlainRange(e, kb0, kb1), turn);
            continue;
        }
        float acc[128];
        plain_sums(smem, PlainRange(e, kb0, kb1), turn, acc);
        const int64_t row = static_cast<int64_t>(tm) * kTileRows + rank * 128 + warp % 4 * 32 + threadIdx.x % 32;
        const int64_t col0 = static_cast<int64_t>(tn) * kTileCols + half * 128;
        if (MODE == Out::Logits) store_logits(args, e.M, acc, row, col0, tn * 2 + half, 1.0f, 1.0f);
        else store_sum(args, e.M, acc, row, col0, split, 1.0f, 1.0f);
    }
}

template <Out MODE>
__global__ void __launch_bounds__(kCtaThreads, 1) k_plain_products(const __grid_constant__ TileArgs args0,
                                                                   const __grid_constant__ TileArgs args1, int n) {
    extern __shared__ __align__(16) float plain_smem[];
    wait_for_previous();
    if (*args0.wide == 0) return;
    int turn = 0;
#pragma unroll 1
    for (int i = 0; i < n; ++i) plain_product<MODE>(i == 0 ? args0 : args1, plain_smem, turn);
}

// The splits' partial results in order, into the rows of the result, whatever their layout.
// Bound by HBM, 4 bytes an element and split and 4 more.
__global__ void __launch_bounds__(256) k_join_splits(const TileArgs a, int64_t out_cs, int vec) {
    wait_for_previous();
    int64_t M = a.M;
    if (a.live != nullptr && !a.live_k) M = live_extent(a.live, a.first, M);
    if (a.live_k && a.first > 0 && live_extent(a.live, a.first, a.K) == 0) return;
    const int64_t plane = a.M * a.parts_pitch;
    if (vec) {
        const int64_t per_row = a.N / 4;
        for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < M * per_row;
             i += static_cast<int64_t>(gridDim.x) * 256) {
            const int64_t r = i / per_row, c = (i - r * per_row) * 4;
            const float *src = a.parts + r * a.parts_pitch + c;
            float4 sum = *reinterpret_cast<const float4 *>(src);
            for (int s = 1; s < a.splits; ++s) {
                const float4 v = *reinterpret_cast<const float4 *>(src + s * plane);
                sum.x += v.x;
                sum.y += v.y;
                sum.z += v.z;
                sum.w += v.w;
            }
            float4 *to = reinterpret_cast<float4 *>(
                a.out + (a.out_map != nullptr ? a.out_map[a.first + r] : r) * a.out_rs + c);
            if (a.add) {
                const float4 o = *to;
                sum.x += o.x;
                sum.y += o.y;
                sum.z += o.z;
                sum.w += o.w;
            }
            *to = sum;
        }
        return;
    }
    // a warp a row, eight columns of a lane in flight
    const int lane = threadIdx.x % 32;
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * 8 + threadIdx.x / 32; r < M;
         r += static_cast<int64_t>(gridDim.x) * 8) {
        const float *src = a.parts + r * a.parts_pitch;
        float *to = a.out + (a.out_map != nullptr ? a.out_map[a.first + r] : r) * a.out_rs;
        for (int64_t c0 = lane; c0 < a.N; c0 += 256) {
            float sum[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) sum[u] = c0 + 32 * u < a.N ? src[c0 + 32 * u] : 0.0f;
            for (int s = 1; s < a.splits; ++s)
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    if (c0 + 32 * u < a.N) sum[u] += src[s * plane + c0 + 32 * u];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                if (c0 + 32 * u >= a.N) break;
                float *p = to + (c0 + 32 * u) * out_cs;
                *p = a.add ? *p + sum[u] : sum[u];
            }
        }
    }
}

// The logits of few tiles, split along the columns of x: their partial sums added in order, and
// what store_logits does with them.  A warp takes 128 classes of a row.
__global__ void __launch_bounds__(256) k_join_logits(const TileArgs a) {
    wait_for_previous();
    const int lane = threadIdx.x % 32;
    const int64_t M = live_extent(a.live, a.first, a.M), chunks = (a.N + 127) / 128, plane = a.M * a.parts_pitch;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 8 + threadIdx.x / 32; i < M * chunks;
         i += static_cast<int64_t>(gridDim.x) * 8) {
        const int64_t r = i / chunks, k = i - r * chunks, c = k * 128 + lane * 4;
        float z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (c < a.parts_pitch) {
            const float *src = a.parts + r * a.parts_pitch + c;
#pragma unroll 4
            for (int s = 0; s < a.splits; ++s) {
                const float4 v = *reinterpret_cast<const float4 *>(src + s * plane);
                z[0] += v.x;
                z[1] += v.y;
                z[2] += v.z;
                z[3] += v.w;
            }
        }
        const int64_t target = a.target[a.first + r];
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (c + j >= a.N) {
                z[j] = -INFINITY;
                continue;
            }
            if (a.bias != nullptr) z[j] += __ldg(a.bias + (c + j) * a.bias_s);
            if (c + j == target) a.z_target[r] = z[j];
            top = fmaxf(top, z[j]);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        const float base = isinf(top) ? 0.0f : top;
        float sum = 0.0f;
        int same = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (z[j] == top) ++same;
            else sum += expf(z[j] - base);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        same = __reduce_add_sync(0xFFFFFFFFu, same);
        if (lane == 0) {
            a.part_max[r * 2 * a.tiles_n + k] = top;
            a.part_rest[r * 2 * a.tiles_n + k] = top == -INFINITY && !isnan(sum) ? -1.0f : sum + static_cast<float>(same - 1);
        }
        if (a.z != nullptr && c < a.z_pitch)
            *reinterpret_cast<float4 *>(a.z + r * a.z_pitch + c) = make_float4(z[0], z[1], z[2], z[3]);
    }
}

// ----------------------------------------------------------------- softmax --

struct RowArgs {
    int64_t first, rows;  // of the live rows
    const int *live;
    int parts, part_pitch;  // of a row
    const float *part_max, *part_rest, *z_target;
    const int *row;       // of x
    LogSum *lse_live;     // [rows]
    const float *dloss;   // null: no gradients
    int *row_exp;         // [rows] exponent of the scale of g' as the rows of dx
    float *loss, *lse;
    int64_t loss_s, lse_s;
};

// One warp a row: the statistics of its tiles make lse and the loss (8 bytes for 128 logits:
// 7 us for 4096 x 32000).
__global__ void __launch_bounds__(256) k_row_loss(const RowArgs a) {
    wait_for_previous();
    const int64_t r = static_cast<int64_t>(blockIdx.x) * 8 + threadIdx.x / 32;
    const int lane = threadIdx.x % 32;
    if (r >= live_extent(a.live, a.first, a.rows)) return;
    const float *m = a.part_max + r * a.part_pitch, *s = a.part_rest + r * a.part_pitch;
    Softmax all = no_logits();
    for (int j = lane; j < a.parts; j += 32) all = merge(all, Softmax{m[j], s[j]});
    all = merge_lanes(all, 1, 32);
    if (lane != 0) return;
    const LogSum l = all.log_sum();
    a.lse_live[r] = l;
    // the largest |g| of a row is that of its target, to which all others add up
    if (a.dloss != nullptr)
        a.row_exp[r] = scale_exponent(__float_as_int(finite_abs(a.dloss[a.first + r] * expm1f(l.of(a.z_target[r])))));
    const int64_t n = a.row[a.first + r];
    if (a.lse != nullptr) a.lse[n * a.lse_s] = l.lse();
    if (a.loss != nullptr) a.loss[n * a.loss_s] = l.loss(a.z_target[r]);
}

struct GradArgs {
    int64_t first;
    const int *live;
    int64_t rows;
    int64_t V;
    float *z;            // [rows][pitch], becomes g' as the rows of dx (of dweight, where there is no dx)
    int64_t pitch;
    const LogSum *lse_live;
    const int *target;
    const float *dloss;
    const int *row_exp;  // [rows] exponents of the scales of g' as the rows of dx; null: not wanted
    int *class_exp;      // [row blocks][pitch] of g' as the rows of dweight; null: not wanted
    __half *by_class;    // [rows][pitch][2], that g'
    float *column_parts; // [row blocks][pitch] column sums of g; null: not wanted
    const int *wide;     // set: z becomes g, as float32, for both
};

constexpr int kGradRows = kPieceBlocks * kBlock;  // rows of a CTA: a piece of dweight's K
constexpr int kGradThreads = 512, kGradWarps = kGradThreads / 32;

// z -> g'.  The two products want g on scales of their own, or the small ones among its entries
// lose their digits next to the large ones: dx takes each row to its largest entry (rows whose
// dloss is small, rows sure of their class), dweight each class to its largest in a piece of K
// (classes that are improbable everywhere).  So g goes out twice, once in the place of z.
// A CTA takes 64 columns of 256 rows, a thread four columns of 8 of the rows, in registers;
// everything is read before anything is written.  Bound by HBM, 12 bytes a logit: 4096 x 32000
// in 252 us (6.2 TB/s).
__global__ void __launch_bounds__(kGradThreads, 2) k_softmax_grad(const GradArgs a) {
    wait_for_previous();
    struct Row {
        LogSum lse;
        float d;
        int target;
    };
    __shared__ __align__(16) Row rows[kGradRows];
    __shared__ float row_scale[kGradRows];
    __shared__ __align__(16) float sums[kGradWarps][kBlock], tops[kGradWarps][kBlock], class_scale[kBlock];
    const int64_t live = live_extent(a.live, a.first, a.rows), packed = (live + 63) / 64 * 64;
    const int64_t r0 = static_cast<int64_t>(blockIdx.y) * kGradRows;
    if (r0 >= packed) return;
    constexpr int kGroups = kGradThreads / 16, kMine = kGradRows / kGroups;
    const int group = threadIdx.x / 16, warp = threadIdx.x / 32, quad = threadIdx.x % 16;
    const int64_t c0 = static_cast<int64_t>(blockIdx.x) * kBlock, c = c0 + quad * 4;
    float *z = a.z + (r0 + group) * a.pitch + c;
    const int64_t stride = kGroups * a.pitch;  // from a row of this thread's to the next
    const int mine = static_cast<int>(live - r0 - group);  // rows from its first on, row j of them kGroups j
    float g[kMine][4];
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
        const float4 v = j * kGroups < mine ? __ldcs(reinterpret_cast<const float4 *>(z + j * stride))
                                            : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        g[j][0] = v.x;
        g[j][1] = v.y;
        g[j][2] = v.z;
        g[j][3] = v.w;
    }
    if (threadIdx.x < kGradRows) {  // rows without a loss get a g of zero
        const int64_t r = r0 + threadIdx.x;
        const bool has = r < live;
        rows[threadIdx.x] = Row{has ? a.lse_live[r] : LogSum{0.0f, 0.0f}, has ? a.dloss[a.first + r] : 0.0f,
                                has ? a.target[a.first + r] : -1};
        row_scale[threadIdx.x] = has && a.row_exp != nullptr ? power_of_two(a.row_exp[r]) : 1.0f;
    }
    if (c0 + kBlock > a.V) {  // behind the last class
#pragma unroll
        for (int j = 0; j < kMine; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (c + k >= a.V) g[j][k] = -INFINITY;
    }
    __syncthreads();
    float column[4] = {0.0f, 0.0f, 0.0f, 0.0f}, top[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
        const Row row = rows[j * kGroups + group];
        const unsigned int hot = row.target - static_cast<int>(c);
        float at_hot = 0.0f;
        if (hot < 4) at_hot = row.d * expm1f(row.lse.of(hot == 0 ? g[j][0] : hot == 1 ? g[j][1] : hot == 2 ? g[j][2] : g[j][3]));
#pragma unroll
        for (int k = 0; k < 4; ++k) g[j][k] = row.d * expf(row.lse.of(g[j][k]));
        if (hot < 4) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (hot == k) g[j][k] = at_hot;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            column[k] += g[j][k];
            top[k] = fmaxf(top[k], fabsf(g[j][k]));
        }
    }
    if (a.column_parts != nullptr || a.class_exp != nullptr) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            column[k] += __shfl_xor_sync(0xFFFFFFFFu, column[k], 16);
            top[k] = fmaxf(top[k], __shfl_xor_sync(0xFFFFFFFFu, top[k], 16));
        }
        if (threadIdx.x % 32 < 16) {
            *reinterpret_cast<float4 *>(&sums[warp][quad * 4]) = make_float4(column[0], column[1], column[2], column[3]);
            *reinterpret_cast<float4 *>(&tops[warp][quad * 4]) = make_float4(top[0], top[1], top[2], top[3]);
        }
        __syncthreads();
        if (threadIdx.x < kBlock) {  // a class each
            float sum = 0.0f, largest = 0.0f;
#pragma unroll
            for (int w = 0; w < kGradWarps; ++w) {
                sum += sums[w][threadIdx.x];
                largest = fmaxf(largest, tops[w][threadIdx.x]);
            }
            // (of a class with an infinite entry the others do not matter)
            const int e = scale_exponent(__float_as_int(fminf(largest, 3.402823466e38f)));
            const int64_t at = blockIdx.y * a.pitch + c0 + threadIdx.x;
            class_scale[threadIdx.x] = power_of_two(e);
            if (a.column_parts != nullptr) a.column_parts[at] = sum;
            if (a.class_exp != nullptr) a.class_exp[at] = e;
        }
        __syncthreads();
    }
    if (*a.wide != 0) {
#pragma unroll
        for (int j = 0; j < kMine; ++j)
            if (j * kGroups < mine) *reinterpret_cast<float4 *>(z + j * stride) = make_float4(g[j][0], g[j][1], g[j][2], g[j][3]);
        return;
    }
    const int packs = static_cast<int>(packed - r0 - group);
    const int64_t at = 2 * ((r0 + group) * a.pitch + c0) + quad * 4;
    if (a.row_exp != nullptr) {
        __half *to = reinterpret_cast<__half *>(a.z) + at;
#pragma unroll
        for (int j = 0; j < kMine; ++j) {
            const float f = row_scale[j * kGroups + group];
            if (j * kGroups < packs) store_pairs(to + 2 * j * stride, g[j][0] * f, g[j][1] * f, g[j][2] * f, g[j][3] * f);
        }
    }
    if (a.class_exp != nullptr) {
        const float4 f = *reinterpret_cast<const float4 *>(&class_scale[quad * 4]);
        __half *to = a.by_class + at;
#pragma unroll
        for (int j = 0; j < kMine; ++j)
            if (j * kGroups < packs)
                store_pairs(to + 2 * j * stride, g[j][0] * f.x, g[j][1] * f.y, g[j][2] * f.z, g[j][3] * f.w);
    }
}

// A CTA takes 32 columns; its warps, up to 32, take the row blocks in turn (4 bytes for 256 rows
// of a column: 4 us for 4096 x 32000).
__global__ void __launch_bounds__(1024) k_bias_grad(const GradArgs a, float *db, int64_t db_s, int add) {
    wait_for_previous();
    __shared__ float sums[32][32];
    const int warps = blockDim.x / 32;
    const int64_t v = static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.x % 32;
    const int blocks = static_cast<int>((live_extent(a.live, a.first, a.rows) + kGradRows - 1) / kGradRows);
    float sum = 0.0f;
    if (v < a.V) {
#pragma unroll 8
        for (int b = threadIdx.x / 32; b < blocks; b += warps) sum += a.column_parts[b * a.pitch + v];
    }
    sums[threadIdx.x / 32][threadIdx.x % 32] = sum;
    __syncthreads();
    if (threadIdx.x >= 32 || v >= a.V) return;
    for (int w = 1; w < warps; ++w) sum += sums[w][threadIdx.x];
    db[v * db_s] = add ? db[v * db_s] + sum : sum;
}

// ------------------------------------------------------------------- host --

// Tensor map of a packed operand: (64 columns, rows, blocks, hi / lo).
int operand_map(CUtensorMap &map, const __half *base, int64_t rows, int64_t blocks, int64_t pitch_blocks, bool mn) {
    EncodeTiled enc = tensor_map_encoder();
    if (enc == nullptr) return fail(MTC_ERR_RUNTIME, "cuTensorMapEncodeTiled is unavailable");
    const cuuint64_t dims[4] = {kBlock, static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(blocks), 2};
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(pitch_blocks) * 256, 256, 128};
    const cuuint32_t box[4] = {kBlock, mn ? 64u : 128u, mn ? 2u : 1u, 1};
    const cuuint32_t elem[4] = {1, 1, 1, 1};
    const CUresult r = enc(&map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<__half *>(base), dims, strides, box, elem,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(MTC_ERR_RUNTIME, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
    return MTC_OK;
}

template <bool A_MN, bool B_MN, Out MODE>
int launch_product(const CUtensorMap &a, const CUtensorMap &b, const TileArgs &args, int sms, cudaStream_t stream) {
    MTC_CUDA_TRY(cudaFuncSetAttribute(k_pair_product<A_MN, B_MN, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      kSmemBytes));
    const int64_t units = (args.M + kTileRows - 1) / kTileRows * args.tiles_n * args.splits;
    const int64_t pairs = units < sms / 2 ? units : sms / 2;
    return launch_dependent("linear cross entropy (tensor-core product)", k_pair_product<A_MN, B_MN, MODE>,
                            static_cast<unsigned>(2 * pairs), kCtaThreads, kSmemBytes, stream, a, b, args);
}

// The float32 products in their stead, of one or of both gradients.
template <Out MODE>
int launch_plain(const TileArgs *args, int n, int sms, cudaStream_t stream) {
    MTC_CUDA_TRY(cudaFuncSetAttribute(k_plain_products<MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPlainSmem));
    return launch_dependent("linear cross entropy (float32 products)", k_plain_products<MODE>,
                            static_cast<unsigned>(sms / 2 * 2), kCtaThreads, kPlainSmem, stream, args[0], args[n - 1], n);
}

// Splits of K so that the tiles of a product fill the pairs of SMs: the fewest whose
// last wave is nearly full, each at least 512 of K, or 256 (a piece) where half of the GPU
// would idle: there the partial results are small (17 x 1000 x 4096: 78 -> 68 us for the loss
// and its gradients, against 249 -> 287 us for 4096 x 2500 x 1024).
int choose_splits(int64_t tiles, int64_t K, int64_t pairs, size_t bytes) {
    int best = 1;
    double best_cost = 1e30;
    const int64_t least = 2 * tiles <= pairs ? 256 : 512;
    for (int s = 1; s <= 16; ++s) {
        if (s > 1 && (K / s < least || bytes * s > (size_t{1} << 30))) break;
        const double waves = static_cast<double>((tiles * s + pairs - 1) / pairs);
        const double cost = waves / s * (1.0 + 0.01 * (s - 1));
        if (cost < best_cost * 0.98) {
            best_cost = cost;
            best = s;
        }
    }
    return best;
}

// Whether rows can be stored a 32-byte sector a time.
bool sector_rows(const float *p, int64_t rs, int64_t cs, int64_t cols) {
    return reinterpret_cast<uintptr_t>(p) % 32 == 0 && cs == 1 && rs % 8 == 0 && cols % 8 == 0;
}

bool vector_source(const float *p, int64_t rs, int64_t cs, int64_t cols) {
    return aligned16(p) && cs == 1 && rs % 4 == 0 && cols % 4 == 0;
}

// `most_rows`: of a piece, a multiple of 256.
int in_pieces(const LinearCe &p, cudaStream_t stream, int64_t most_rows) {
    const int sms = sm_count(current_device());
    const int64_t pairs = sms / 2;
    const bool grads = p.dloss != nullptr && ((p.D > 0 && (p.dx != nullptr || p.dw != nullptr)) || p.db != nullptr);
    const int64_t d_blocks = (p.D + kBlock - 1) / kBlock, v_blocks = (p.V + kBlock - 1) / kBlock;
    const int64_t pitch = v_blocks * kBlock;
    const int tiles_v = static_cast<int>((p.V + kTileCols - 1) / kTileCols);
    const int tiles_d = static_cast<int>((p.D + kTileCols - 1) / kTileCols);
    // rows at a time: the logits of a piece, and the second g' of both products, fill at most
    // 4 GiB (a piece more reads and writes dweight once more); without gradients only their
    // statistics are kept, 8 bytes for 128 logits
    const int64_t rows_all = (p.N + 255) / 256 * 256;
    const bool two = p.dx != nullptr && p.dw != nullptr && p.D > 0;
    const int64_t row_bytes = grads ? pitch * (two ? 8 : 4) : static_cast<int64_t>(tiles_v) * 16;
    int64_t piece = (int64_t{4} << 30) / row_bytes / 256 * 256;
    if (piece < 256) piece = 256;
    if (piece > most_rows) piece = most_rows;
    const int64_t pieces = (rows_all + piece - 1) / piece;
    piece = ((rows_all + pieces - 1) / pieces + 255) / 256 * 256;
    if (rows_all * d_blocks > (int64_t{1} << 40) || pitch > INT32_MAX)
        return fail(MTC_ERR_UNSUPPORTED, "linear cross entropy: too large");

    const int splits_dx = choose_splits(piece / 256 * tiles_d, p.V, pairs, static_cast<size_t>(piece) * p.D * 4);
    const int splits_dw = choose_splits(static_cast<int64_t>(tiles_v) * tiles_d, piece, pairs,
                                        static_cast<size_t>(p.V) * p.D * 4);
    // A tile of logits takes 13 ns a column of x, however few there are of them: split where they
    // leave half of the GPU idle.  (60 rows, 200 classes of length 4096: 90 -> 38 us for the loss.)
    const int64_t tiles_z = piece / 256 * tiles_v;
    const int splits_z = 2 * tiles_z <= pairs ? choose_splits(tiles_z, p.D, pairs, static_cast<size_t>(piece) * pitch * 4) : 1;
    const size_t list = padded(static_cast<size_t>(p.N) * 4);
    const size_t x_bytes = padded(static_cast<size_t>(rows_all) * d_blocks * 256);
    const size_t w_bytes = padded(static_cast<size_t>(p.V) * d_blocks * 256);
    const size_t stat = padded(static_cast<size_t>(piece) * 2 * tiles_v * 4);
    const size_t row_stat = padded(static_cast<size_t>(piece) * 4);
    const size_t z_bytes = grads ? padded(static_cast<size_t>(piece) * pitch * 4) : 0;
    const size_t by_class_bytes = grads && two ? z_bytes : 0;
    const size_t col_bytes = padded(static_cast<size_t>(piece / kGradRows) * pitch * 4);
    const size_t db_bytes = grads && p.db != nullptr ? col_bytes : 0;
    const size_t exp_bytes = grads && p.dw != nullptr ? col_bytes : 0;
    const int64_t parts_pitch = (p.D + 7) / 8 * 8;
    const bool parts_dx = splits_dx > 1 || !sector_rows(p.dx, p.dx_rs, p.dx_cs, p.D);
    const bool parts_dw = splits_dw > 1 || !sector_rows(p.dw, p.dw_rs, p.dw_cs, p.D);
    const size_t split_dx = p.dx != nullptr && parts_dx ? static_cast<size_t>(splits_dx) * piece * parts_pitch * 4 : 0;
    const size_t split_dw = p.dw != nullptr && parts_dw ? static_cast<size_t>(splits_dw) * p.V * parts_pitch * 4 : 0;
    const size_t split_z = splits_z > 1 ? static_cast<size_t>(splits_z) * piece * pitch * 4 : 0;
    const size_t split_grad = !grads ? 0 : padded(split_dx) + padded(split_dw);
    const size_t split_bytes = padded(split_z) > split_grad ? padded(split_z) : split_grad;
    // a byte a row and one a column of either tensor, four times: see Held
    const int64_t d_pad = d_blocks * kBlock;
    const size_t held_x = padded(static_cast<size_t>(rows_all)), held_w = padded(static_cast<size_t>(p.V));
    const size_t held_d = padded(static_cast<size_t>(d_pad)), held = 4 * (held_x + held_w + 2 * held_d);
    Workspace ws;
    const int allocated = ws.allocate(256 + held + 3 * list + x_bytes + w_bytes + 2 * stat + 4 * row_stat + z_bytes +
                                          by_class_bytes + db_bytes + exp_bytes + split_bytes,
                                      stream);
    if (allocated == MTC_ERR_RUNTIME && piece > 256) {  // no memory for that: in smaller pieces
        MTC_TRY(in_pieces(p, stream, piece / 2 / 256 * 256));
        clear_error();
        return MTC_OK;
    }
    MTC_TRY(allocated);
    LiveRows live;
    live.count = ws.take<int>(256);
    live.row = ws.take<int>(list);
    live.target = ws.take<int>(list);
    live.dloss = ws.take<float>(list);
    unsigned char *flags = ws.take<unsigned char>(held);
    __half *xp = ws.take<__half>(x_bytes);
    __half *wp = ws.take<__half>(w_bytes);
    float *part_max = ws.take<float>(stat);
    float *part_rest = ws.take<float>(stat);
    float *z_target = ws.take<float>(row_stat);
    LogSum *lse_live = ws.take<LogSum>(2 * row_stat);
    int *row_exp = ws.take<int>(row_stat);
    float *z = ws.take<float>(z_bytes);
    __half *by_class = two ? ws.take<__half>(by_class_bytes) : reinterpret_cast<__half *>(z);
    float *columns = ws.take<float>(db_bytes);
    int *class_exp = ws.take<int>(exp_bytes);
    float *split_ws = ws.take<float>(split_bytes);
    unsigned long long *err = nullptr;
    MTC_TRY(device_error_word(&err));
    MTC_TRY(list_live_rows(p, live, stream));

    PackArgs k;
    std::memset(&k, 0, sizeof(k));
    k.s[0] = PackSource{p.x, p.x_rs, p.x_cs, p.N, p.D, live.row, live.count, vector_source(p.x, p.x_rs, p.x_cs, p.D),
                        xp, rows_all, 0, {}};
    k.s[1] = PackSource{p.w, p.w_rs, p.w_cs, p.V, p.D, nullptr, nullptr, vector_source(p.w, p.w_rs, p.w_cs, p.D),
                        wp, p.V, 1, {}};
    k.flags = reinterpret_cast<uint4 *>(flags);
    k.flags16 = static_cast<int64_t>(held / 16);
    for (PackSource &s : k.s) {
        const size_t rows = s.which == 0 ? held_x : held_w;
        for (Held &h : s.held) {
            h = Held{flags, flags + rows, flags + 2 * rows, flags + 2 * rows + held_d, static_cast<int64_t>(rows / 16),
                     static_cast<int64_t>(held_d / 16)};
            flags += 2 * (rows + held_d);
        }
    }
    if (p.dx != nullptr && p.D > 0) k.dx = p.dx;
    k.dx_rs = p.dx_rs;
    k.dx_cs = p.dx_cs;
    k.dx_vec = vector_source(p.dx, p.dx_rs, p.dx_cs, p.D);
    k.known = live.count;
    // CTAs in proportion to the tensors' rows, four to an SM in all
    const int64_t most = static_cast<int64_t>(sms) * 4;
    const int64_t share = most * p.N / (p.N + p.V);
    k.first_of_second = share < 1 ? 1 : share > most - 1 ? most - 1 : share;
    const unsigned ctas = static_cast<unsigned>(most);
    {
        PackArgs few = k;  // half of the CTAs, a quarter for each
        few.first_of_second = sms;
        MTC_TRY(launch_dependent("linear cross entropy (sample)", k_sample, static_cast<unsigned>(2 * sms), 256, 0, stream, few));
    }
    const int64_t sample = 8 * sms;
    k.headroom = p.N <= sample && p.V <= sample ? 0 : 6;
    MTC_TRY(launch_dependent("linear cross entropy (packing)", k_pack<false>, ctas, 256, 0, stream, k));
    if (k.headroom != 0)
        MTC_TRY(launch_dependent("linear cross entropy (packing again)", k_pack<true>, ctas, 256, 0, stream, k));

    CUtensorMap x_k, w_k, w_mn, x_mn, g_k, g_mn;
    const int64_t map_blocks = d_blocks > 0 ? d_blocks : 1;
    for (int64_t first = 0; first < p.N; first += piece) {
        const int64_t rows = p.N - first < piece ? p.N - first : piece;
        const int64_t rows_up = (rows + 63) / 64 * 64;
        const __half *xc = xp + first * d_blocks * 2 * kBlock;
        MTC_TRY(operand_map(x_k, xc, rows_up, map_blocks, map_blocks, false));
        MTC_TRY(operand_map(w_k, wp, p.V, map_blocks, map_blocks, false));
        TileArgs t;
        std::memset(&t, 0, sizeof(t));
        t.M = rows;
        t.N = p.V;
        t.K = p.D;
        t.live = live.count;
        t.first = first;
        t.tiles_n = tiles_v;
        t.group = 16;
        t.splits = splits_z;
        t.exp_a = live.count + kExponent;
        t.exp_b = live.count + kExponent + 1;
        t.wide = live.count + kWide;
        t.judges = first == 0;
        std::memcpy(t.held[0], k.s[0].held, sizeof(t.held[0]));
        std::memcpy(t.held[1], k.s[1].held, sizeof(t.held[1]));
        t.repacked = live.count + kRepacked;
        t.a = Plain{p.x, p.x_rs, p.x_cs, live.row + first, nullptr};
        t.b = Plain{p.w, p.w_rs, p.w_cs, nullptr, nullptr};
        t.err = err;
        t.z = grads ? z : nullptr;
        t.z_pitch = pitch;
        t.bias = p.bias;
        t.bias_s = p.b_s;
        t.target = live.target;
        t.part_max = part_max;
        t.part_rest = part_rest;
        t.z_target = z_target;
        if (splits_z > 1) {
            t.parts = split_ws;
            t.parts_pitch = pitch;
            MTC_TRY((launch_product<false, false, Out::Sum>(x_k, w_k, t, sms, stream)));
            MTC_TRY(launch_plain<Out::Sum>(&t, 1, sms, stream));
            const int64_t ctas = (rows * ((p.V + 127) / 128) + 7) / 8;
            MTC_TRY(launch_dependent("linear cross entropy (logits)", k_join_logits,
                                     static_cast<unsigned>(ctas < sms * 8 ? ctas : sms * 8), 256, 0, stream, t));
        } else {
            MTC_TRY((launch_product<false, false, Out::Logits>(x_k, w_k, t, sms, stream)));
            MTC_TRY(launch_plain<Out::Logits>(&t, 1, sms, stream));
        }
        // (a last tile of 128 columns or less has no second half)
        const RowArgs ra{first, rows, live.count, static_cast<int>((p.V + 127) / 128), 2 * tiles_v, part_max, part_rest,
                         z_target, live.row, lse_live, grads ? live.dloss : nullptr, row_exp, p.loss, p.lse, p.loss_s, p.lse_s};
        MTC_TRY((launch_dependent("linear cross entropy (loss)", k_row_loss, static_cast<unsigned>((rows + 7) / 8), 256, 0, stream, ra)));
        if (!grads) continue;
        const bool dx = p.dx != nullptr && p.D > 0, dw = p.dw != nullptr && p.D > 0;
        const GradArgs ga{first, live.count, rows_up, p.V, z, pitch, lse_live, live.target, live.dloss,
                          dx ? row_exp : nullptr, dw ? class_exp : nullptr, by_class, p.db != nullptr ? columns : nullptr,
                          live.count + kWide};
        const dim3 grid(static_cast<unsigned>(v_blocks), static_cast<unsigned>((rows_up + kGradRows - 1) / kGradRows));
        MTC_TRY((launch_dependent("linear cross entropy (gradient of the logits)", k_softmax_grad, grid, kGradThreads, 0, stream, ga)));
        if (p.db != nullptr) {
            MTC_TRY((launch_dependent("linear cross entropy (bias gradient)", k_bias_grad, static_cast<unsigned>((p.V + 31) / 32), piece > 16 * kGradRows ? 1024 : 256, 0, stream, ga, p.db, p.db_s, first > 0)));
        }
        TileArgs of[2];
        int n = 0;
        if (dx) {
            TileArgs &t = of[n++];
            MTC_TRY(operand_map(g_k, reinterpret_cast<const __half *>(z), rows_up, v_blocks, v_blocks, false));
            MTC_TRY(operand_map(w_mn, wp, p.V, d_blocks, d_blocks, true));
            std::memset(&t, 0, sizeof(t));
            t.M = rows;
            t.N = p.D;
            t.K = p.V;
            t.live = live.count;
            t.first = first;
            t.tiles_n = tiles_d;
            t.group = 16;
            t.splits = splits_dx;
            t.exp_a = row_exp;
            t.exp_b = live.count + kExponent + 1;
            t.wide = live.count + kWide;
            t.a = Plain{z, pitch, 1, nullptr, nullptr};
            t.b = Plain{p.w, p.w_cs, p.w_rs, nullptr, nullptr};
            t.err = err;
            t.out = p.dx;
            t.out_rs = p.dx_rs;
            t.out_map = live.row;
            t.parts = parts_dx ? split_ws : nullptr;
            t.parts_pitch = parts_pitch;
            MTC_TRY((launch_product<false, true, Out::Sum>(g_k, w_mn, t, sms, stream)));
        }
        if (dw) {
            TileArgs &t = of[n++];
            MTC_TRY(operand_map(g_mn, by_class, rows_up, v_blocks, v_blocks, true));
            MTC_TRY(operand_map(x_mn, xc, rows_up, d_blocks, d_blocks, true));
            std::memset(&t, 0, sizeof(t));
            t.M = p.V;
            t.N = p.D;
            t.K = rows;
            t.live = live.count;
            t.live_k = true;
            t.first = first;
            t.tiles_n = tiles_d;
            t.group = 16;
            t.splits = splits_dw;
            t.exp_a = class_exp;
            t.exp_pitch = pitch;
            t.exp_b = live.count + kExponent;
            t.wide = live.count + kWide;
            t.a = Plain{z, 1, pitch, nullptr, nullptr};
            t.b = Plain{p.x, p.x_cs, p.x_rs, nullptr, live.row + first};
            t.err = err;
            t.out = p.dw;
            t.out_rs = p.dw_rs;
            t.add = first > 0;
            t.parts = parts_dw ? split_ws + padded(split_dx) / sizeof(float) : nullptr;
            t.parts_pitch = parts_pitch;
            MTC_TRY((launch_product<true, true, Out::Sum>(g_mn, x_mn, t, sms, stream)));
        }
        if (n == 0) continue;
        MTC_TRY(launch_plain<Out::Sum>(of, n, sms, stream));
        if (dx && parts_dx)
            MTC_TRY(launch_dependent("linear cross entropy (input gradient)", k_join_splits, static_cast<unsigned>(sms * 8),
                                     256, 0, stream, of[0], p.dx_cs, vector_source(p.dx, p.dx_rs, p.dx_cs, p.D)));
        if (dw && parts_dw)
            MTC_TRY(launch_dependent("linear cross entropy (weight gradient)", k_join_splits, static_cast<unsigned>(sms * 8),
                                     256, 0, stream, of[n - 1], p.dw_cs, vector_source(p.dw, p.dw_rs, p.dw_cs, p.D)));
    }
    return MTC_OK;
}

}  // namespace

int linear_ce_tensor(const LinearCe &p, cudaStream_t stream) {
    return in_pieces(p, stream, int64_t{1} << 21);  // k_softmax_grad's grid
}

}  // namespace mtc
