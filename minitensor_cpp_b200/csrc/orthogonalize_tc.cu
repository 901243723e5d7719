// The products of the Newton-Schulz steps on the tensor cores, with float32 accuracy.
//
// An operand is a pair of 16-bit floats, scaled by a power of two that is known beforehand (see
// orthogonalize.cu) so that what may occur lies below 2^14:
//   hi = f16(x),  lo = f16((x - hi) 2^11),   x = hi + lo 2^-11 within 2^-22 |x| or 2^-36
// and a product three MMAs, hi.lo + lo.hi first and then hi.hi, the 2^-11 applied by the MMA
// itself (scale-input-d) when hi.hi is added.  The tensor core truncates its accumulator at every
// addition, so 256 values of K stay in tensor memory at most; the epilogue warps add each such
// piece, rounded to nearest, to sums in registers.  What truncation takes is not noise: pieces of
// 256 lost 4 (products of both signs) to 13 (of one sign) 2^-24 of themselves, 64 2 to 3, so a
// piece counts as 1 + 2^-23 for each 64.  (S S X of 1024 x 4096: 1.9e-6 off, with it 1.4e-7.)
//
// Nor is it noise that small products lose when they are added to a large one, which the
// diagonals of S and B make of every sum as X nears orthogonality (1024 x 4096 after five steps:
// 5.5e-6 off, with the diagonals apart 7.4e-7, in float32 3.4e-6).  So S = D + R and B = E + Q with the diagonals D and E apart, in float32, and
// zeros in their place:
//   S S = D^2 + D R + R D + R R,   B X = E X + Q X
// whose first terms are the epilogues'.
//
// Three products a step, all from packed operands to packed operands:
//   D + R = X X^T             operands X and X, both K-major
//   E + Q = b S + c S S       operands R and R (symmetric), both K-major; R is read again as it is
//   X = (a + E) X + Q X       operands Q, K-major, and X, MN-major
// R and Q are symmetric, so only tiles on and above the diagonal are computed, and their
// epilogue writes a tile and its mirror image.
//
// A CTA works on a tile of 128 x 128, a pair of CTAs (tcgen05.mma.cta_group::2) on one of 256 x
// 256; either way a CTA stages 128 rows of A and 128 columns of B, 64 KB for 64 of K.  A pair has
// rings of five stages of hi (free at the end of a piece) and two of lo (free after its cross
// terms), 32 KB each.  A single CTA keeps the cross terms in columns of their own of the tensor
// memory, which its smaller tiles leave, and has one ring of six: its blocks take half the time,
// and two stages of lo would not cover a load.  Warp 0 loads (TMA: the workspace is one tensor of rows of 128 bytes), warp 1 issues,
// warps 4..11 are the epilogue, two for each quarter of the tensor memory's lanes.
// ptxas assigns the 168 registers of the launch to all warps, also to the epilogue's, which have 208:
// single tiles' X spills 62 words, pairs' X 26 and their symmetric products 51.
// Every wait is bounded; on expiry the device error word is set and the roles leave.
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstring>

#include "orthogonalize.cuh"
#include "tcgen05.cuh"

namespace mtc {
namespace ortho {
namespace {

constexpr int kBlock = 64;
constexpr int kHalfBytes = 8192;                 // 64 rows of 128 bytes: a TMA box
constexpr int kOperandBytes = 2 * kHalfBytes;
constexpr int kStageBytes = 2 * kOperandBytes;   // A and B, hi or lo
constexpr int kHiStages = 5, kLoStages = 2, kStages = kHiStages + kLoStages;  // of a pair
constexpr int kRing = 6;                         // of a single CTA; the epilogue warps have the seventh
constexpr int kPieceBlocks = 4;                  // blocks of K that are summed in tensor memory
constexpr int kSmemBytes = kStages * kStageBytes + 1024 + 256;
constexpr int kCtaThreads = 384;
constexpr float kCutOff = 0x1p-23f;              // what a sum loses a block, see above
constexpr int kEpilogueRegs = 208, kOtherRegs = 88;
static_assert(kSmemBytes <= 227 * 1024, "shared memory per CTA");
static_assert(256 * kEpilogueRegs + 128 * kOtherRegs <= kCtaThreads * 168, "registers of the launch (168 a thread)");
constexpr int kSumPitch = 132;                   // of a CTA's sums in shared memory, which the stages have left
static_assert(128 * kSumPitch * 4 <= kRing * kStageBytes, "sums");
static_assert(kRing % 2 == 0, "hi and lo in turn");
static_assert(8 * 4096 <= kStageBytes, "the epilogue warps' rows");

enum Product { kSymmetric, kApply };

template <int N>
struct Args {
    Table<N> table;
    int units;
    int from;           // kSymmetric: S from X (0), or B from S (1); kApply: from X 0 or 1
    int last;           // kApply: to the outputs
    float q;            // of the sums of products
    float p, r;         // kSymmetric: R times p + r (D_i + D_j); kApply: X times p (r + E_i)
    float b, c, unit;   // of the diagonals: D = unit sums, E = b D + c D^2 + unit sums
    char *workspace;
    unsigned long long *err;
};

__device__ __forceinline__ void load_rows(void *dst, const char *src, uint64_t *bar, int bytes) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}

__device__ __forceinline__ void load_half_pair(void *dst, const CUtensorMap *map, uint32_t leader_bar, int row) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%3, %4}], [%2];"
        ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(leader_bar), "r"(0), "r"(row)
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

// D = F32, A = B = F16, tiles of 128 x 128 or 256 x 256.
template <bool PAIR, bool B_MN>
__device__ __forceinline__ constexpr uint32_t instr_desc() {
    constexpr uint32_t tile = PAIR ? 256 : 128;
    return (1u << 4) | (B_MN ? 1u << 16 : 0u) | ((tile >> 3) << 17) | ((tile >> 4) << 24);
}

template <bool PAIR>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
}

// D = A B + D 2^-11
template <bool PAIR>
__device__ __forceinline__ void mma_scaled(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
    if (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p, 11;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(1)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p, 11;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(1)
            : "memory");
}

// Arrives on the barrier (of both CTAs of a pair) when the MMAs issued so far are done.
template <bool PAIR>
__device__ __forceinline__ void commit(uint64_t *bar) {
    if (PAIR) {
        umma_commit_both(bar);
    } else {
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                     : "memory");
    }
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

// Two blocks of 32 columns, waited for once.
__device__ __forceinline__ void tmem_ld32_two(uint32_t from_v, uint32_t from_w, float (&v)[32], float (&w)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%64];\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
        "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%65];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
          "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
          "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
          "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31]),
          "=f"(w[0]), "=f"(w[1]), "=f"(w[2]), "=f"(w[3]), "=f"(w[4]), "=f"(w[5]), "=f"(w[6]), "=f"(w[7]),
          "=f"(w[8]), "=f"(w[9]), "=f"(w[10]), "=f"(w[11]), "=f"(w[12]), "=f"(w[13]), "=f"(w[14]), "=f"(w[15]),
          "=f"(w[16]), "=f"(w[17]), "=f"(w[18]), "=f"(w[19]), "=f"(w[20]), "=f"(w[21]), "=f"(w[22]), "=f"(w[23]),
          "=f"(w[24]), "=f"(w[25]), "=f"(w[26]), "=f"(w[27]), "=f"(w[28]), "=f"(w[29]), "=f"(w[30]), "=f"(w[31])
        : "r"(from_v), "r"(from_w)
        : "memory");
}

// The loader and the issuer run their loops with all lanes of their warps and values that the
// compiler can tell are the same in all, so that these stay in uniform registers, which the
// instructions that one lane of them issues want; a lone lane's loop moves each of them there
// first, and a block of 128 x 128 x 64 took twice the time of its MMAs.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}

__device__ __forceinline__ bool wait_all(uint64_t *bar, uint32_t parity, volatile int *abort_flag) {
    return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, abort_flag));
}

// Where a block's hi or lo is staged, and the parity of its barriers, from block to block.  (Kept:
// a division for each costs a lone thread more than the MMAs of a block.)
template <bool PAIR>
struct Stages {
    int at[2] = {0, PAIR ? kHiStages : 1};
    uint32_t parity[2] = {0, 0};

    __device__ __forceinline__ void next() {
#pragma unroll
        for (int lo = 0; lo < 2; ++lo) {
            at[lo] += PAIR ? 1 : 2;
            const int end = !PAIR ? kRing : lo ? kStages : kHiStages;
            if (at[lo] < end) continue;
            at[lo] = PAIR && lo ? kHiStages : lo;
            parity[lo] ^= 1;
        }
    }
};

// A unit of work: a tile of one matrix.
struct Unit {
    int matrix, tm, tn;
};

constexpr int kBand = 8;  // row tiles that share a sweep of the columns: their panels meet in L2

__host__ __device__ inline int symmetric_tiles(int tiles) { return tiles * (tiles + 1) / 2; }

// Tile t of those on and above the diagonal of T x T: bands of kBand rows, each column by column.
__device__ __forceinline__ void symmetric_tile(int t, int T, int &tm, int &tn) {
    int first = 0;
    for (;;) {
        const int rows = T - first < kBand ? T - first : kBand;
        const int corner = symmetric_tiles(rows), all = corner + (T - first - rows) * rows;
        if (t < all) {
            if (t < corner) {
                int c = 0;
                while (symmetric_tiles(c + 1) <= t) ++c;
                tm = first + t - symmetric_tiles(c);
                tn = first + c;
            } else {
                tm = first + (t - corner) % rows;
                tn = first + rows + (t - corner) / rows;
            }
            return;
        }
        t -= all;
        first += rows;
    }
}

__device__ __forceinline__ void band_tile(int t, int tiles_m, int tiles_n, int &tm, int &tn) {
    const int band = t / (kBand * tiles_n), first = band * kBand;
    const int rows = tiles_m - first < kBand ? tiles_m - first : kBand;
    t -= first * tiles_n;
    tm = first + t % rows;
    tn = t / rows;
}

template <Product PRODUCT, int N>
__device__ __forceinline__ Unit unit_of(const Args<N> &a, int u, int tile) {
    Unit r;
    r.matrix = find_matrix(a.table, u);
    const Matrix &mt = a.table.matrix[r.matrix];
    const int t = u - a.table.first[r.matrix];
    const int tiles_m = (mt.m + tile - 1) / tile;
    if (PRODUCT == kSymmetric) symmetric_tile(t, tiles_m, r.tm, r.tn);
    else band_tile(t, tiles_m, (mt.n + tile - 1) / tile, r.tm, r.tn);
    return r;
}

// Eight neighbouring columns of a row as pairs, an element's hi in the low half of a word and its
// lo in the high half.
__device__ __forceinline__ void to_pairs(const float (&v)[8], uint32_t (&w)[8]) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const __half2 h = __floats2half2_rn(v[j], v[j + 1]);
        const float2 f = __half22float2(h);
        const __half2 l = __floats2half2_rn((v[j] - f.x) * 2048.0f, (v[j + 1] - f.y) * 2048.0f);
        const uint32_t hb = *reinterpret_cast<const uint32_t *>(&h), lb = *reinterpret_cast<const uint32_t *>(&l);
        w[j] = __byte_perm(hb, lb, 0x5410);
        w[j + 1] = __byte_perm(hb, lb, 0x7632);
    }
}

__device__ __forceinline__ void from_pairs(const uint4 &h, const uint4 &l, float (&v)[8]) {
    const uint32_t hw[4] = {h.x, h.y, h.z, h.w}, lw[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&hw[j]));
        const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&lw[j]));
        v[2 * j] = fmaf(b.x, 0x1p-11f, a.x);
        v[2 * j + 1] = fmaf(b.y, 0x1p-11f, a.y);
    }
}

__device__ __forceinline__ void split_pairs(const uint32_t (&w)[8], uint4 &h, uint4 &l) {
    h.x = __byte_perm(w[0], w[1], 0x5410);
    h.y = __byte_perm(w[2], w[3], 0x5410);
    h.z = __byte_perm(w[4], w[5], 0x5410);
    h.w = __byte_perm(w[6], w[7], 0x5410);
    l.x = __byte_perm(w[0], w[1], 0x7632);
    l.y = __byte_perm(w[2], w[3], 0x7632);
    l.z = __byte_perm(w[4], w[5], 0x7632);
    l.w = __byte_perm(w[6], w[7], 0x7632);
}

// Two chunks of a row that share a sector; in odd rows the swizzle has them the other way round.
template <int N>
__device__ __forceinline__ void load_sector(const char *from, int swapped, uint4 (&v)[N]) {
    uint4 a, b;
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
                 : "l"(from)
                 : "memory");
    v[0] = swapped ? b : a;
    v[N - 1] = swapped ? a : b;
}

template <int N>
__device__ __forceinline__ void store_sector(char *to, int swapped, const uint4 (&v)[N]) {
    const uint4 a = swapped ? v[N - 1] : v[0], b = swapped ? v[0] : v[N - 1];
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(to), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
                 : "memory");
}

// What is left of `chunks` chunks of eight columns, from `col` (of whole chunks) on, of a warp's 32
// neighbouring rows, once their sums are there.  What they are added to is asked for early: kAhead
// chunks at a time.
template <bool PAIR, Product PRODUCT, int N>
struct Finish {
    // A pair takes two chunks at a time: the 32 bytes of a sector, which the swizzle keeps together.
    static constexpr int kStep = PAIR ? 2 : 1, kAhead = PAIR ? 0 : 4, kHeld = PAIR ? 4 : 2;
    const Args<N> &a;
    const Matrix &mt;
    int row, col, chunks;
    bool with_old, mirror;
    const char *old;
    char *to, *image;
    float factor;           // kSymmetric: D of the row; kApply: p (r + E of the row)
    float held[kHeld];      // kSymmetric: D of the columns, 32 a register
    uint4 hi[PAIR ? 1 : kAhead][kStep], lo[PAIR ? 1 : kAhead][kStep];

    __device__ __forceinline__ Finish(const Args<N> &args, const Matrix &m, int r, int c, int n, bool image_too)
        : a(args), mt(m), row(r), col(c), chunks(n), mirror(image_too) {
        const int lane = threadIdx.x % 32;
        with_old = PRODUCT == kApply || a.from == 1;
        const int blocks = PRODUCT == kApply ? mt.x_blocks : mt.s_blocks;
        const int64_t at = static_cast<int64_t>(row / 128 * blocks + col / 64) * 256 + row % 128;
        const int from = PRODUCT == kApply ? mt.x[a.from] : mt.s;
        const int into = PRODUCT == kApply ? mt.x[a.from ^ 1] : a.from == 0 ? mt.s : mt.b;
        old = a.workspace + (from + at) * 128;
        to = a.workspace + (into + at) * 128;
        if (PRODUCT == kSymmetric)
            image = a.workspace + (into + static_cast<int64_t>(col / 128 * blocks + row / 64) * 256 + col % 128) * 128;
        if (!with_old) return;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) ask(i * kStep, i);
        const float *d = reinterpret_cast<const float *>(a.workspace + static_cast<int64_t>(mt.s_diagonal) * 128);
        if (PRODUCT == kSymmetric) {
            factor = d[row];
#pragma unroll
            for (int i = 0; i < kHeld; ++i) {  // (within the padded diagonal)
                const int at_col = col + 32 * i + lane;
                held[i] = at_col < mt.s_blocks * 64 ? d[at_col] : 0.0f;
            }
        } else {
            factor = a.p * (a.r + reinterpret_cast<const float *>(a.workspace + static_cast<int64_t>(mt.b_diagonal) * 128)[row]);
        }
    }

    __device__ __forceinline__ int offset(int c) const {  // of chunk c in this row
        const int k = col / 8 % 8 + c;
        return k / 8 * 2 * kOperandBytes + ((k ^ row) & 7) * 16;
    }

    __device__ __forceinline__ void ask(int c, int slot) {
        if (c >= chunks) return;
        if (PAIR) {
            load_sector(old + (offset(c) & ~31), row & 1, hi[slot]);
            load_sector(old + (offset(c) & ~31) + kOperandBytes, row & 1, lo[slot]);
        } else {
            hi[slot][0] = *reinterpret_cast<const uint4 *>(old + offset(c));
            lo[slot][0] = *reinterpret_cast<const uint4 *>(old + offset(c) + kOperandBytes);
        }
    }

    // Sums and old values of chunk c to what comes of them.
    __device__ __forceinline__ void combine(int c, const float (&x)[8], float (&v)[8]) {
        if (PRODUCT == kApply) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = fmaf(factor, x[j], a.q * v[j]);
            return;
        }
        const int first = col + 8 * c;
        const bool own = row >= first && row < first + 8;
        float on = 0.0f;
        if (own) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (row == first + j) on = v[j] * a.unit;
        }
        if (!with_old) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] *= a.q;
        } else {
            float d = held[0];
#pragma unroll
            for (int i = 1; i < kHeld; ++i)
                if (c / 4 == i) d = held[i];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float dj = __shfl_sync(0xFFFFFFFFu, d, c % 4 * 8 + j);
                v[j] = fmaf(fmaf(a.r, factor + dj, a.p), x[j], a.q * v[j]);
            }
        }
        if (own) {
            const int diagonal = a.from == 0 ? mt.s_diagonal : mt.b_diagonal;
            reinterpret_cast<float *>(a.workspace + static_cast<int64_t>(diagonal) * 128)[row] =
                with_old ? fmaf(fmaf(a.c, factor, a.b), factor, on) : on;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (row == first + j) v[j] = 0.0f;
        }
    }

    // Rows become columns: of two neighbouring lanes and columns each lane gets two neighbours of
    // one row of the image.
    __device__ __forceinline__ void store_image(int c, const uint32_t (&w)[8]) {
        const int odd = row & 1;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const uint32_t other = __shfl_xor_sync(0xFFFFFFFFu, odd ? w[j] : w[j + 1], 1);
            const uint32_t left = odd ? other : w[j], right = odd ? w[j + 1] : other;
            const int r = 8 * c + j + odd;  // from the image's first row on, a multiple of 8 in its block
            char *at = image + r * 128 + (((row / 8) ^ r) & 7) * 16 + (row & 6) * 2;
            *reinterpret_cast<uint32_t *>(at) = __byte_perm(left, right, 0x5410);
            *reinterpret_cast<uint32_t *>(at + kOperandBytes) = __byte_perm(left, right, 0x7632);
        }
    }

    __device__ __forceinline__ void operator()(int c, float (&v)[kStep][8]) {
        uint4 h[kStep], l[kStep];
        if (with_old) {
            if (kAhead == 0) ask(c, 0);
#pragma unroll
            for (int i = 0; i < kStep; ++i) {
                h[i] = hi[0][i];
                l[i] = lo[0][i];
            }
#pragma unroll
            for (int i = 0; i + 1 < kAhead; ++i)
#pragma unroll
                for (int k = 0; k < kStep; ++k) {
                    hi[i][k] = hi[i + 1][k];
                    lo[i][k] = lo[i + 1][k];
                }
            if (kAhead > 0) ask(c + kAhead * kStep, kAhead > 0 ? kAhead - 1 : 0);
        }
#pragma unroll
        for (int i = 0; i < kStep; ++i) {
            float x[8];
            if (with_old) from_pairs(h[i], l[i], x);
            combine(c + i, x, v[i]);
        }
        if (PRODUCT == kApply && a.last) {
#pragma unroll
            for (int i = 0; i < kStep; ++i) store_output(col + 8 * (c + i), v[i]);
            return;
        }
#pragma unroll
        for (int i = 0; i < kStep; ++i) {
            uint32_t w[8];
            to_pairs(v[i], w);
            split_pairs(w, h[i], l[i]);
            if (PRODUCT == kSymmetric && mirror) store_image(c + i, w);
        }
        if (PAIR) {
            store_sector(to + (offset(c) & ~31), row & 1, h);
            store_sector(to + (offset(c) & ~31) + kOperandBytes, row & 1, l);
        } else {
            *reinterpret_cast<uint4 *>(to + offset(c)) = h[0];
            *reinterpret_cast<uint4 *>(to + offset(c) + kOperandBytes) = l[0];
        }
    }

    __device__ __forceinline__ void store_output(int first, const float (&v)[8]) const {
        if (row >= mt.m || first >= mt.n) return;
        float *out = mt.dst + row * mt.out_rs + first * mt.out_cs;
        if (mt.out_cs == 1 && first + 8 <= mt.n && (reinterpret_cast<uintptr_t>(out) & 15) == 0) {
            reinterpret_cast<float4 *>(out)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4 *>(out)[1] = make_float4(v[4], v[5], v[6], v[7]);
            return;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (first + j < mt.n) out[j * mt.out_cs] = v[j];
    }
};

// The warp's buffer is free: the copies out of it that lane 0 has begun have read it.
__device__ __forceinline__ void rows_are_read() {
    if (threadIdx.x % 32 == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
}

// A warp's 32 rows of a block of 64 columns, which are 4 KB in a row of the workspace, hi or lo, by
// way of its 4 KB of shared memory: a lane reads and writes chunks of one row, but 16 bytes of each
// of 32 rows at a time are 32 times the work of 512 bytes for the load and store units (a tile of
// 128 x 128 read and written so took 5.1 us, which is most of a small product).
__device__ __forceinline__ void rows_to_lanes(const char *from, char *buffer, uint4 (&v)[8]) {
    const int lane = threadIdx.x % 32;
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = *reinterpret_cast<const uint4 *>(from + k * 512 + lane * 16);
    rows_are_read();
#pragma unroll
    for (int k = 0; k < 8; ++k) *reinterpret_cast<uint4 *>(buffer + k * 512 + lane * 16) = v[k];
    __syncwarp();
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = *reinterpret_cast<const uint4 *>(buffer + lane * 128 + ((k ^ lane) & 7) * 16);
}

__device__ __forceinline__ void lanes_to_rows(const uint4 (&v)[8], char *buffer, char *to) {
    const int lane = threadIdx.x % 32;
    rows_are_read();
#pragma unroll
    for (int k = 0; k < 8; ++k) *reinterpret_cast<uint4 *>(buffer + lane * 128 + ((k ^ lane) & 7) * 16) = v[k];
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) {
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], 4096;" ::"l"(to), "r"(smem_u32(buffer)) : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
}

// The same for 32 of the outputs' columns, next to one another.
__device__ __forceinline__ void lanes_to_output(const float *v, char *buffer, const Matrix &mt, int row0, int col) {
    const int lane = threadIdx.x % 32;
    rows_are_read();
#pragma unroll
    for (int k = 0; k < 8; ++k)
        *reinterpret_cast<float4 *>(buffer + lane * 128 + ((k ^ lane) & 7) * 16) =
            make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
    __syncwarp();
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const int r = 4 * k + lane / 8, c = col + lane % 8 * 4;
        const float4 x = *reinterpret_cast<const float4 *>(buffer + r * 128 + ((lane ^ r) & 7) * 16);
        if (row0 + r >= mt.m) continue;
        float *out = mt.dst + (row0 + r) * mt.out_rs + c;
        if (c + 4 <= mt.n && (reinterpret_cast<uintptr_t>(out) & 15) == 0) {
            *reinterpret_cast<float4 *>(out) = x;
        } else {
            if (c < mt.n) out[0] = x.x;
            if (c + 1 < mt.n) out[1] = x.y;
            if (c + 2 < mt.n) out[2] = x.z;
            if (c + 3 < mt.n) out[3] = x.w;
        }
    }
}

// Without PAIR, the CTAs of a cluster share the K of one tile, a cluster a tile, and add their sums
// by way of their shared memory, each an equal share of the columns, in the order of the CTAs.
template <bool PAIR, Product PRODUCT, int N>
__global__ void __launch_bounds__(kCtaThreads, 1)
    k_step_product(const __grid_constant__ CUtensorMap map, const __grid_constant__ Args<N> args) {
    constexpr bool B_MN = PRODUCT == kApply;
    constexpr int kTile = PAIR ? 256 : 128, kColumns = kTile / 2;  // of an epilogue thread
    constexpr uint32_t kTmemCols = 512;
    constexpr int kSums = PAIR ? kTile : 2 * kTile;  // columns of a piece in tensor memory
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    // the same aligned offset in all CTAs of a cluster (same dynamic size, same static layout)
    unsigned char *smem =
        reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + kStages * kStageBytes);  // a pair's leader's: both CTAs' bytes
    uint64_t *empty = full + kStages;      // each CTA's: the stage's MMAs are done (hi stages first, then lo)
    uint64_t *acc_full = empty + kStages;  // [2] each CTA's: a piece is in tensor memory
    uint64_t *acc_empty = acc_full + 2;    // [2] a pair's leader's: the epilogues have read it
    uint64_t *drain = acc_empty + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = __shfl_sync(0xFFFFFFFFu, static_cast<int>(threadIdx.x / 32), 0), lane = threadIdx.x % 32;
    uint32_t cluster_size;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(cluster_size));
    const int rank = static_cast<int>(cluster_rank());
    const int group = static_cast<int>(blockIdx.x / cluster_size), groups = static_cast<int>(gridDim.x / cluster_size);
    const int splits = PAIR ? 1 : static_cast<int>(cluster_size), split = PAIR ? 0 : rank;
    const int pair_rank = PAIR ? rank : 0;
    const bool leader = pair_rank == 0;

    // The first unit, which the parameters' way from memory makes the longest part of a launch's
    // beginning, while the barriers and the tensor memory are set up.
    const Unit first_unit = unit_of<PRODUCT>(args, group < args.units ? group : 0, kTile);
    if (PAIR && threadIdx.x == 96) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map)) : "memory");
    if (threadIdx.x == 64) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], PAIR ? 16 : 8);  // the epilogue warps
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                         "r"(kTmemCols));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                         "r"(kTmemCols));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        }
    }
    tc_fence_before();
    __syncthreads();
    if (cluster_size > 1) cluster_sync_all();  // the peers' barriers are initialised before any remote arrive
    tc_fence_after();
    const uint32_t tmem_base = __shfl_sync(0xFFFFFFFFu, *tmem_slot, 0);
    wait_for_previous();

    // K blocks of a unit that are this CTA's
    auto k_range = [&](const Matrix &mt, int &kb0, int &kb1) {
        const int K = PRODUCT == kSymmetric && args.from == 0 ? mt.n : mt.m, blocks = (K + kBlock - 1) / kBlock;
        const int each = (blocks + splits - 1) / splits;
        kb0 = min(split * each, blocks);
        kb1 = min(kb0 + each, blocks);
    };

    if (warp >= 4) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpilogueRegs));
        const int quadrant = warp % 4, half = (warp - 4) / 4;
        const uint32_t release[2] = {peer_addr(&acc_empty[0], PAIR ? 0 : rank), peer_addr(&acc_empty[1], PAIR ? 0 : rank)};
        uint32_t piece = 0;
        bool ok = true;
        for (int u = group; u < args.units && ok; u += groups) {
            const Unit unit = u == group ? first_unit : unit_of<PRODUCT>(args, u, kTile);
            const Matrix &mt = args.table.matrix[unit.matrix];
            int kb0, kb1;
            k_range(mt, kb0, kb1);
            const int row0 = quadrant * 32 + lane;
            const bool whole_unit = PAIR || splits == 1;
            // (of a shared tile the sums alone are worked out here)
            Finish<PAIR, PRODUCT, N> finish(args, mt, unit.tm * kTile + pair_rank * 128 + row0,
                                            unit.tn * kTile + half * kColumns, PAIR ? kColumns / 8 : 0,
                                            PRODUCT == kSymmetric && unit.tm != unit.tn);
            char *const buffer = reinterpret_cast<char *>(smem) + kRing * kStageBytes + (warp - 4) * 4096;
            const int64_t lane_rows = lane * 128;  // from the warp's first row on
            uint4 old_hi[8], old_lo[8];
            if (!PAIR && whole_unit && finish.with_old) {
                rows_to_lanes(finish.old - lane_rows, buffer, old_hi);
                rows_to_lanes(finish.old - lane_rows + kOperandBytes, buffer, old_lo);
            }
            float acc[kColumns];
#pragma unroll
            for (int j = 0; j < kColumns; ++j) acc[j] = 0.0f;
            for (int kb = kb0; kb < kb1; kb += kPieceBlocks, ++piece) {
                const int b = static_cast<int>(piece & 1);
                if (!mbar_wait(&acc_full[b], (piece >> 1) & 1u, abort_flag)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const float whole = 1.0f + (kb1 - kb < kPieceBlocks ? kb1 - kb : kPieceBlocks) * kCutOff;
                const uint32_t at = tmem_base + (static_cast<uint32_t>(quadrant * 32) << 16) +
                                    static_cast<uint32_t>(b * kSums + half * kColumns);
                if (PAIR) {
#pragma unroll
                    for (int c = 0; c < kColumns / 64; ++c) {
                        uint32_t v[64];
                        tmem_ld64(at + static_cast<uint32_t>(c * 64), v);
#pragma unroll
                        for (int j = 0; j < 64; ++j) acc[c * 64 + j] = fmaf(__uint_as_float(v[j]), whole, acc[c * 64 + j]);
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < kColumns / 32; ++c) {
                        float v[32], w[32];
                        tmem_ld32_two(at + static_cast<uint32_t>(c * 32), at + static_cast<uint32_t>(kTile + c * 32), v, w);
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            acc[c * 32 + j] = fmaf(v[j], whole, fmaf(w[j], 0x1p-11f, acc[c * 32 + j]));
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_remote(release[b]);
            }
            if (!whole_unit) {
                // All MMAs of this CTA are done (and with them its loads): the stages hold the sums now.
                float *sums = reinterpret_cast<float *>(smem) + row0 * kSumPitch + half * kColumns;
#pragma unroll
                for (int j = 0; j < kColumns; j += 4)
                    *reinterpret_cast<float4 *>(sums + j) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
                // An equal share of the columns for each CTA, and of that for each half of the warps.
                const int share = 64 / splits, col0 = rank * 2 * share + half * share;
                Finish<PAIR, PRODUCT, N> finish_share(args, mt, unit.tm * kTile + row0, unit.tn * kTile + col0, share / 8,
                                                      PRODUCT == kSymmetric && unit.tm != unit.tn);
                cluster_sync_all();
                const float *mine = reinterpret_cast<const float *>(smem) + row0 * kSumPitch + col0;
#pragma unroll 1
                for (int c = 0; c < share / 8; ++c) {
                    float v[Finish<PAIR, PRODUCT, N>::kStep][8] = {};
#pragma unroll 4
                    for (int s = 0; s < splits; ++s) {
                        const uint32_t from = peer_addr(mine + 8 * c, static_cast<uint32_t>(s));
                        float x[8];
                        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                     : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]) : "r"(from) : "memory");
                        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                     : "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7]) : "r"(from + 16) : "memory");
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[0][i] += x[i];
                    }
                    finish_share(c, v);
                }
                break;  // one unit a cluster
            }
            if (!ok) break;
            if (!PAIR) {
                const bool floats = PRODUCT == kApply && args.last != 0;
                uint4 out_hi[8], out_lo[8];
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    float x[8], v[8];
                    if (finish.with_old) from_pairs(old_hi[c], old_lo[c], x);
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = acc[8 * c + i];
                    finish.combine(c, x, v);
#pragma unroll
                    for (int i = 0; i < 8; ++i) acc[8 * c + i] = v[i];
                    if (floats) continue;
                    uint32_t w[8];
                    to_pairs(v, w);
                    split_pairs(w, out_hi[c], out_lo[c]);
                    if (PRODUCT == kSymmetric && finish.mirror) finish.store_image(c, w);
                }
                if (!floats) {
                    lanes_to_rows(out_hi, buffer, finish.to - lane_rows);
                    lanes_to_rows(out_lo, buffer, finish.to - lane_rows + kOperandBytes);
                } else if (mt.out_cs == 1) {
                    lanes_to_output(acc, buffer, mt, finish.row - lane, finish.col);
                    lanes_to_output(acc + 32, buffer, mt, finish.row - lane, finish.col + 32);
                } else if (finish.row < mt.m) {
                    float *out = mt.dst + finish.row * mt.out_rs + finish.col * mt.out_cs;
#pragma unroll
                    for (int j = 0; j < 64; ++j)
                        if (finish.col + j < mt.n) out[j * mt.out_cs] = acc[j];
                }
                __syncwarp();
                continue;
            }
            // A rolled loop, the sums moved up by sixteen each time.
#pragma unroll 1
            for (int c = 0; c < kColumns / 8; c += 2) {
                float v[Finish<PAIR, PRODUCT, N>::kStep][8];
#pragma unroll
                for (int k = 0; k < Finish<PAIR, PRODUCT, N>::kStep; ++k)
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[k][i] = acc[8 * k + i];
#pragma unroll
                for (int i = 0; i + 16 < kColumns; ++i) acc[i] = acc[i + 16];
                finish(c, v);
            }
            __syncwarp();
        }
        if (!ok) atomicCAS(args.err, 0ull, static_cast<unsigned long long>(MTC_ERR_RUNTIME));
        if (!PAIR && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");  // written, before the next launch
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == 0) {
            const bool elected = elect_one();
            Stages<PAIR> stages;
            int64_t it = 0;
            bool ok = true;
            for (int u = group; u < args.units && ok; u += groups) {
                const Unit unit = u == group ? first_unit : unit_of<PRODUCT>(args, u, kTile);
                const Matrix &mt = args.table.matrix[unit.matrix];
                int kb0, kb1;
                k_range(mt, kb0, kb1);
                const int ta = unit.tm * (kTile / 128) + pair_rank, tb = unit.tn * (kTile / 128) + pair_rank;
                const bool of_x = PRODUCT == kSymmetric && args.from == 0;
                const int a_at = PRODUCT == kApply ? mt.b : of_x ? mt.x[args.last] : mt.s;
                const int a_blocks = of_x ? mt.x_blocks : mt.s_blocks;
                const int b_at = PRODUCT == kApply ? mt.x[args.from] : a_at;
                const int b_blocks = PRODUCT == kApply ? mt.x_blocks : a_blocks;
                for (int kb = kb0; kb < kb1 && ok; ++kb, ++it, stages.next()) {
#pragma unroll
                    for (int lo = 0; lo < 2; ++lo) {
                        const int s = stages.at[lo];
                        if (!wait_all(&empty[s], stages.parity[lo] ^ 1u, abort_flag)) {
                            ok = false;
                            break;
                        }
                        unsigned char *st = smem + s * kStageBytes;
                        if (!elected) continue;
                        if (leader) mbar_expect_tx(&full[s], (PAIR ? 2 : 1) * kStageBytes);
                        const uint32_t fb = peer_addr(&full[s], 0);
                        const int a_row = a_at + ((ta * a_blocks + kb) * 2 + lo) * 128;
                        const int b_row = B_MN ? b_at + ((kb / 2 * b_blocks + tb * 2) * 2 + lo) * 128 + kb % 2 * 64
                                               : b_at + ((tb * b_blocks + kb) * 2 + lo) * 128;
                        constexpr int b_step = B_MN ? 256 : 64;  // to the second half
                        if (PAIR) {
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                load_half_pair(st + h * kHalfBytes, &map, fb, a_row + h * 64);
                                load_half_pair(st + kOperandBytes + h * kHalfBytes, &map, fb, b_row + h * b_step);
                            }
                        } else {
                            const char *a_src = args.workspace + static_cast<int64_t>(a_row) * 128;
                            const char *b_src = args.workspace + static_cast<int64_t>(b_row) * 128;
                            load_rows(st, a_src, &full[s], kOperandBytes);
                            if (B_MN) {
                                load_rows(st + kOperandBytes, b_src, &full[s], kHalfBytes);
                                load_rows(st + kOperandBytes + kHalfBytes, b_src + b_step * 128, &full[s], kHalfBytes);
                            } else {
                                load_rows(st + kOperandBytes, b_src, &full[s], kOperandBytes);
                            }
                        }
                    }
                }
                if (!PAIR && splits > 1) break;
            }
            if (!ok && elected) atomicCAS(args.err, 0ull, static_cast<unsigned long long>(MTC_ERR_RUNTIME));
            if (leader && elected) {  // every stage issued has landed before the cluster exits
                // (the last filling of each: of those that were filled, the one before the next)
                for (int64_t d = it > kHiStages ? it - kHiStages : 0; d < it; ++d)
                    for (int lo = 0; lo < 2; ++lo) {
                        const int64_t depth = !PAIR ? kRing : lo ? kLoStages : kHiStages, n = PAIR ? d : 2 * d + lo;
                        if (n + depth < (PAIR ? it : 2 * it)) continue;  // filled again since
                        const int s = static_cast<int>(n % depth) + (PAIR && lo ? kHiStages : 0);
                        for (long long i = 0; i < kWaitLimit && !mbar_try_wait(&full[s], static_cast<uint32_t>(n / depth) & 1u); ++i) {
                        }
                    }
            }
        } else if (warp == 1) {
            if (leader) {
                const bool elected = elect_one();
                constexpr uint32_t idesc = instr_desc<PAIR, B_MN>();
                constexpr uint64_t a_step = 32 >> 4, b_step = (B_MN ? 2048 : 32) >> 4;  // 16 of K
                Stages<PAIR> stages;  // of the next block
                uint32_t piece = 0;
                bool ok = true;
                for (int u = group; u < args.units && ok; u += groups) {
                    const Unit unit = u == group ? first_unit : unit_of<PRODUCT>(args, u, kTile);
                    int kb0, kb1;
                    k_range(args.table.matrix[unit.matrix], kb0, kb1);
                    for (int kb = kb0; kb < kb1 && ok; kb += kPieceBlocks, ++piece) {
                        const int n = kb1 - kb < kPieceBlocks ? kb1 - kb : kPieceBlocks;
                        const int b = static_cast<int>(piece & 1);
                        if (!wait_all(&acc_empty[b], ((piece >> 1) & 1u) ^ 1u, abort_flag)) {
                            ok = false;
                            break;
                        }
                        const uint32_t d = tmem_base + static_cast<uint32_t>(b * kSums);
                        const uint32_t cross = PAIR ? d : d + kTile;
                        int hi_stage = stages.at[0];
                        for (int j = 0; j < n; ++j, stages.next()) {
                            const int sh = stages.at[0], sl = stages.at[1];
                            if (!wait_all(&full[sh], stages.parity[0], abort_flag) ||
                                !wait_all(&full[sl], stages.parity[1], abort_flag)) {
                                ok = false;
                                break;
                            }
                            tc_fence_after();
                            if (!elected) continue;
                            const uint32_t hi = smem_u32(smem + sh * kStageBytes), lo = smem_u32(smem + sl * kStageBytes);
                            const uint64_t ah = operand_desc<false>(hi), bh = operand_desc<B_MN>(hi + kOperandBytes);
                            const uint64_t al = operand_desc<false>(lo), bl = operand_desc<B_MN>(lo + kOperandBytes);
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                mma<PAIR>(cross, ah + k * a_step, bl + k * b_step, idesc, j > 0 || k > 0);
                                if (!PAIR) mma<PAIR>(d, ah + k * a_step, bh + k * b_step, idesc, j > 0 || k > 0);
                                mma<PAIR>(cross, al + k * a_step, bh + k * b_step, idesc, 1);
                            }
                            commit<PAIR>(&empty[sl]);
                            if (!PAIR) commit<PAIR>(&empty[sh]);
                        }
                        if (!ok) break;
                        for (int j = 0; PAIR && j < n; ++j) {
                            const int sh = hi_stage;
                            hi_stage = hi_stage + 1 < kHiStages ? hi_stage + 1 : 0;
                            if (!elected) continue;
                            const uint32_t hi = smem_u32(smem + sh * kStageBytes);
                            const uint64_t ah = operand_desc<false>(hi), bh = operand_desc<B_MN>(hi + kOperandBytes);
                            if (j == 0) mma_scaled<PAIR>(d, ah, bh, idesc);
                            else mma<PAIR>(d, ah, bh, idesc, 1);
#pragma unroll
                            for (int k = 1; k < 4; ++k) mma<PAIR>(d, ah + k * a_step, bh + k * b_step, idesc, 1);
                            commit<PAIR>(&empty[sh]);
                        }
                        if (elected) commit<PAIR>(&acc_full[b]);
                    }
                    if (!PAIR && splits > 1) break;
                }
                if (!ok && elected) atomicCAS(args.err, 0ull, static_cast<unsigned long long>(MTC_ERR_RUNTIME));
                // all MMAs are done before a CTA frees its tensor memory
                if (elected) {
                    if (PAIR) umma_commit_pair_local(drain);
                    else commit<false>(drain);
                }
                for (long long i = 0; i < kWaitLimit && !mbar_try_wait(drain, 0u); ++i) {
                }
            }
        }
        __syncwarp();
        if (!PAIR && splits > 1) cluster_sync_all();  // with the epilogue warps: the sums are in shared memory
    }

    tc_fence_before();
    __syncthreads();
    if (cluster_size > 1) cluster_sync_all();  // a pair's MMAs have drained; the sums of a shared tile have been read
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        if (PAIR)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols));
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols));
    }
}

// What a step's epilogues multiply by.
struct Scales {
    float gram, d_unit;                // S = X X^T: of the sums of products, and of those that give D
    float square, p, r, b, c, e_unit;  // B from S
    float apply, own, a;               // X
};

// In 64 bits until a coefficient is in: a power of two of its own may leave float32, and 0 times
// it is 0.
Scales scales_of(const Step &s, bool last) {
    auto two = [](int e) { return std::ldexp(1.0, e); };
    const int to = last ? 0 : s.x_after;
    Scales f;
    f.gram = static_cast<float>(two(s.s - 2 * s.x));
    f.d_unit = static_cast<float>(two(-2 * s.x));
    f.square = static_cast<float>(s.c * two(s.b_exp - 2 * s.s));
    f.p = static_cast<float>(s.b * two(s.b_exp - s.s));
    f.r = static_cast<float>(s.c * two(s.b_exp - s.s));
    f.b = s.b;
    f.c = s.c;
    f.e_unit = static_cast<float>(s.c * two(-2 * s.s));
    f.apply = static_cast<float>(two(to - s.b_exp - s.x));
    f.own = static_cast<float>(two(to - s.x));
    f.a = s.a;
    return f;
}

// --------------------------------------------------- matrices of one tile --
//
// Up to 128 x 128: a CTA has X, R and Q in shared memory as blocks' images, 64 KB each, and goes
// through all products of all steps: the MMAs of one, then its sums out of tensor memory, worked
// out and written to the next one's operand by all threads.  Bound by that chain's latency, 3 to
// 4.5 us a product: five steps of 64 x 64 in 48 us, of 128 x 128 in 69 (by launches of their own,
// 145), 64 of these in 78 (164).

constexpr int kWholeThreads = 256, kImage = 4 * kOperandBytes;  // two blocks, hi and lo
constexpr int kTilePitch = 129;                                 // of X as float32, in the place of R and Q
constexpr int kWholeBytes = 3 * kImage + 1024 + 2 * 128 * 4 + 64;
static_assert(kWholeBytes <= 227 * 1024 && 128 * kTilePitch * 4 <= 2 * kImage, "shared memory");

struct WholeSteps {
    int n, scale;  // (exponent of X's scale at first)
    float eps;
    Scales step[kMostSteps];
};

__device__ __forceinline__ double whole_sum(double v, double *part) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int i = 0; i < kWholeThreads / 32; ++i) v += part[i];
    return v;
}

template <int N>
__global__ void __launch_bounds__(kWholeThreads, 1)
    k_whole(const __grid_constant__ Table<N> table, const __grid_constant__ WholeSteps steps, unsigned long long *err) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ double part[kWholeThreads / 32];
    char *const x = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    char *const r = x + kImage, *const q = r + kImage;
    float *const d = reinterpret_cast<float *>(q + kImage), *const e = d + 128;
    uint64_t *const bar = reinterpret_cast<uint64_t *>(e + 128);
    uint32_t *const tmem_slot = reinterpret_cast<uint32_t *>(bar + 1);
    volatile int *const abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = __shfl_sync(0xFFFFFFFFu, static_cast<int>(threadIdx.x / 32), 0), lane = threadIdx.x % 32;
    const Matrix &mt = table.matrix[blockIdx.x];
    if (threadIdx.x == 64) {
        mbar_init(bar, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 256;" ::"r"(smem_u32(tmem_slot)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    // X as it is, and its norm
    float *const tile = reinterpret_cast<float *>(r);
    const bool along = mt.cs == 1 || mt.rs != 1;
    double squares = 0.0;
#pragma unroll 8
    for (int i = threadIdx.x; i < 128 * 128; i += kWholeThreads) {
        const int row = along ? i / 128 : i % 128, col = along ? i % 128 : i / 128;
        const float v = row < mt.m && col < mt.n ? mt.src[row * mt.rs + col * mt.cs] : 0.0f;
        squares += static_cast<double>(v) * v;
        tile[row * kTilePitch + col] = v;
    }
    tc_fence_before();
    const Factor factor(inverse_norm(whole_sum(squares, part), steps.eps), steps.scale);
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *tmem_slot, 0);
    // a thread's row and the first of its 64 columns, which are one block
    const int row = warp % 4 * 32 + lane, col0 = warp / 4 * 64;
    const int at = warp / 4 * 2 * kOperandBytes + row * 128;
    auto chunk = [&](char *image, int c) { return image + at + ((c ^ row) & 7) * 16; };
    auto put = [&](char *image, int c, const float (&v)[8]) {
        uint32_t w[8];
        uint4 h, l;
        to_pairs(v, w);
        split_pairs(w, h, l);
        *reinterpret_cast<uint4 *>(chunk(image, c)) = h;
        *reinterpret_cast<uint4 *>(chunk(image, c) + kOperandBytes) = l;
    };
    auto get = [&](char *image, int c, float (&v)[8]) {
        from_pairs(*reinterpret_cast<const uint4 *>(chunk(image, c)),
                   *reinterpret_cast<const uint4 *>(chunk(image, c) + kOperandBytes), v);
    };
#pragma unroll 2
    for (int c = 0; c < 8; ++c) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = factor(tile[row * kTilePitch + col0 + 8 * c + j]);
        put(x, c, v);
    }
    uint32_t phase = 0;
    float acc[64];
    // The sums of a product over `blocks` blocks of K, A K-major and B either way.  Warps without a
    // row or a column of the result leave it be; of R and Q, whose columns are K after that, rows
    // count up to a whole block.
    auto product = [&](char *a, char *b, bool mn, int blocks, bool here) {
        tc_fence_before();
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();  // the operands are written, and the last sums read
        if (warp == 0 && elect_one()) {
            tc_fence_after();
            const uint32_t idesc = mn ? instr_desc<false, true>() : instr_desc<false, false>();
            for (int k = 0; k < 4 * blocks; ++k) {
                const uint32_t block = static_cast<uint32_t>(k / 4 * 2 * kOperandBytes + k % 4 * 32);
                const uint64_t ah = operand_desc<false>(smem_u32(a) + block);
                const uint64_t al = operand_desc<false>(smem_u32(a) + block + kOperandBytes);
                // of 16 rows of X, the next 64 columns a block on
                const uint64_t far = static_cast<uint64_t>((2 * kOperandBytes - 8192) >> 4) << 16;
                const uint64_t bh = mn ? operand_desc<true>(smem_u32(b) + k * 2048) + far
                                       : operand_desc<false>(smem_u32(b) + block);
                const uint64_t bl = mn ? operand_desc<true>(smem_u32(b) + k * 2048 + kOperandBytes) + far
                                       : operand_desc<false>(smem_u32(b) + block + kOperandBytes);
                mma<false>(tmem + 128, ah, bl, idesc, k > 0);
                mma<false>(tmem, ah, bh, idesc, k > 0);
                mma<false>(tmem + 128, al, bh, idesc, 1);
            }
            commit<false>(bar);
        }
        __syncwarp();
        const bool ok = mbar_wait(bar, phase, abort_flag);
        phase ^= 1;
        tc_fence_after();
        if (!here) return ok;
        const float whole = 1.0f + blocks * kCutOff;
        const uint32_t from = tmem + (static_cast<uint32_t>(warp % 4 * 32) << 16) + static_cast<uint32_t>(col0);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            float v[32], w[32];
            tmem_ld32_two(from + c * 32, from + 128 + c * 32, v, w);
#pragma unroll
            for (int j = 0; j < 32; ++j) acc[c * 32 + j] = fmaf(v[j], whole, w[j] * 0x1p-11f);
        }
        return ok;
    };
    const int m_blocks = (mt.m + kBlock - 1) / kBlock, n_blocks = (mt.n + kBlock - 1) / kBlock;
    const bool of_s = warp % 4 * 32 < m_blocks * kBlock && col0 < mt.m, of_x = warp % 4 * 32 < mt.m && col0 < mt.n;
    bool ok = true;
    for (int k = 0; k < steps.n; ++k) {
        const Scales s = steps.step[k];  // (a copy: read where they are used, 2 us of 50 more)
        ok = product(x, x, false, n_blocks, of_s) && ok;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            if (!of_s) break;
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = acc[8 * c + j] * s.gram;
                if (row == col0 + 8 * c + j) {
                    d[row] = acc[8 * c + j] * s.d_unit;
                    v[j] = 0.0f;
                }
            }
            put(r, c, v);
        }
        ok = product(r, r, false, m_blocks, of_s) && ok;
        const float di = d[row];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            if (!of_s) break;
            float v[8], old[8];
            get(r, c, old);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int col = col0 + 8 * c + j;
                v[j] = fmaf(fmaf(s.r, di + d[col], s.p), old[j], s.square * acc[8 * c + j]);
                if (row == col) {
                    e[row] = fmaf(fmaf(s.c, di, s.b), di, s.e_unit * acc[8 * c + j]);
                    v[j] = 0.0f;
                }
            }
            put(q, c, v);
        }
        ok = product(q, x, true, m_blocks, of_x) && ok;
        const bool last = k == steps.n - 1;
        const float own = s.own * (s.a + e[row]);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            if (!of_x) break;
            float v[8], old[8];
            get(x, c, old);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = fmaf(own, old[j], s.apply * acc[8 * c + j]);
                if (last) tile[row * kTilePitch + col0 + 8 * c + j] = v[j];
            }
            if (!last) put(x, c, v);
        }
        if (!__syncthreads_and(ok)) break;
    }
    if (!ok && lane == 0) atomicCAS(err, 0ull, static_cast<unsigned long long>(MTC_ERR_RUNTIME));
    const bool out_along = mt.out_cs == 1 || mt.out_rs != 1;
    for (int i = threadIdx.x; i < mt.m * mt.n; i += kWholeThreads) {
        const int row = out_along ? i / mt.n : i % mt.m, col = out_along ? i % mt.n : i / mt.m;
        mt.dst[row * mt.out_rs + col * mt.out_cs] = tile[row * kTilePitch + col];
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 256;" ::"r"(tmem));
    }
}

// ------------------------------------------------------------------- host --

// The workspace as rows of 128 bytes, in boxes of 64.
int workspace_map(CUtensorMap &map, char *workspace, size_t bytes) {
    EncodeTiled enc = tensor_map_encoder();
    if (enc == nullptr) return fail(MTC_ERR_RUNTIME, "cuTensorMapEncodeTiled is unavailable");
    const cuuint64_t dims[2] = {64, bytes / 128};
    const cuuint64_t strides[1] = {128};
    const cuuint32_t box[2] = {64, 64}, elem[2] = {1, 1};
    const CUresult r = enc(&map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, workspace, dims, strides, box, elem,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(MTC_ERR_RUNTIME, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
    return MTC_OK;
}

template <bool PAIR, Product PRODUCT, int N>
int launch(const CUtensorMap &map, const Args<N> &args, int cluster, int ctas, cudaStream_t stream) {
    auto *kernel = k_step_product<PAIR, PRODUCT, N>;
    MTC_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
    cudaLaunchAttribute attr[2];
    std::memset(attr, 0, sizeof(attr));
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t config;
    std::memset(&config, 0, sizeof(config));
    config.gridDim = static_cast<unsigned>(ctas);
    config.blockDim = kCtaThreads;
    config.dynamicSmemBytes = kSmemBytes;
    config.stream = stream;
    config.attrs = attr;
    config.numAttrs = 2;
    MTC_CUDA_TRY(cudaLaunchKernelEx(&config, kernel, map, args));
    return check_launch("orthogonalize (product)");
}

// Units of a product in tiles of `tile`, written to the table.
template <int N>
int64_t count_units(Table<N> &t, Product product, int tile) {
    int64_t units = 0;
    t.first[0] = 0;
    for (int i = 0; i < t.count; ++i) {
        const int64_t m = (t.matrix[i].m + tile - 1) / tile, n = (t.matrix[i].n + tile - 1) / tile;
        units += product == kSymmetric ? m * (m + 1) / 2 : m * n;
        t.first[i + 1] = static_cast<int>(units < INT_MAX ? units : INT_MAX);
    }
    return units;
}

int blocks_of(const Matrix &m, bool of_x) { return ((of_x ? m.n : m.m) + kBlock - 1) / kBlock; }

struct Shape {
    bool pairs;
    int cluster, ctas;
};

// Microseconds of a launch whose units, those of most blocks first, go to `at_once` of them in
// turn: `begin` and `end` of the launch, and for a unit of n blocks `block` times n / splits, or
// the epilogue where that is longer.
template <int N>
double estimate(const Table<N> &t, bool of_x, int64_t units, int at_once, int splits, double begin, double block,
                double epilogue, double end) {
    double sum = begin + end;
    int64_t u = 0;
    for (int k = 0; k < 64 && u < units; ++k, u += at_once) {
        const int n = (blocks_of(t.matrix[find_matrix(t, static_cast<int>(u))], of_x) + splits - 1) / splits;
        sum += block * n > epilogue ? block * n : epilogue;
    }
    return u < units ? sum * static_cast<double>(units) / static_cast<double>(u) : sum;
}

// Pairs on tiles of 256, single CTAs on tiles of 128, or these in clusters that share K: whatever
// takes the shortest, by what the parts of a launch were seen to take (timers in the kernel).  A
// block of 64 of K takes a pair 0.83 us, all pairs together 1.05 (L2 gives some 9 TB/s), a single
// CTA 0.67 (what an SM takes in) and all together 1.05, for a quarter of the products.  A launch
// begins and ends for 9.5 us on single tiles, 16 to 28 on pairs' (the epilogue of a symmetric
// product writes its image too), 14 to 19 on shared ones, which are launched anew for each that
// an SM takes.  (2048 x 2048, B X: 64 pairs 49 us, 256 single tiles 62; 1024 x 1024, X X^T: 36
// clusters of 2 19 us, of 4 34, 10 pairs 30; 512 x 512: 10 single tiles 15, clusters of 8 20.)
template <int N>
int choose_shape(Args<N> &args, Product product, bool of_x, Shape &shape) {
    Table<N> &t = args.table;
    std::stable_sort(t.matrix, t.matrix + t.count,
                     [&](const Matrix &a, const Matrix &b) { return blocks_of(a, of_x) > blocks_of(b, of_x); });
    const int sms = sm_count(current_device());
    double best = 1e30;
    bool pairs = true;
    for (int i = 0; i < t.count; ++i) pairs = pairs && tile_of(t.matrix[i].m) == 256;
    if (pairs) {
        const int64_t units = count_units(t, product, 256);
        if (units < INT_MAX) {
            const int at_once = static_cast<int>(units < sms / 2 ? units : sms / 2);
            best = estimate(t, of_x, units, at_once, 1, 6.0, at_once * 3 < sms ? 0.83 : 1.05, 10.0, product == kSymmetric ? 22.0 : 10.0);
            shape = Shape{true, 2, 2 * at_once};
        }
    }
    const int64_t units = count_units(t, product, 128);
    if (units >= INT_MAX && !(best < 1e30)) return fail(MTC_ERR_UNSUPPORTED, "orthogonalize: too many tiles");
    // clusters that an SM's whole shared memory a CTA leaves room for, of 148 SMs
    const int room[4] = {sms, sms / 2, sms * 33 / 148, sms * 15 / 148};
    for (int i = 0, splits = 1; units < INT_MAX && i < 4; ++i, splits *= 2) {
        if (splits > 1 && units * splits > INT_MAX / 2) break;
        const int at_once = static_cast<int>(units < room[i] ? units : room[i]);
        if (at_once < 1) break;
        const double block = at_once * splits * 2 <= sms ? 0.67 : 1.05;
        const double shared[4] = {0.0, 14.0, 15.0, 19.0};
        const double time = splits == 1 ? estimate(t, of_x, units, at_once, 1, 4.5, block, 4.0, 5.0)
                                        : estimate(t, of_x, units, at_once, splits, 0.0, block, 0.0, 0.0) +
                                              shared[i] * static_cast<double>((units + at_once - 1) / at_once);
        if (time >= best) continue;
        best = time;
        shape = Shape{false, splits, static_cast<int>(splits > 1 ? units * splits : at_once)};
    }
    args.units = static_cast<int>(count_units(t, product, shape.pairs ? 256 : 128));
    return MTC_OK;
}

template <Product PRODUCT, int N>
int launch_product(const CUtensorMap &map, const Args<N> &args, const Shape &shape, cudaStream_t stream) {
    return shape.pairs ? launch<true, PRODUCT, N>(map, args, shape.cluster, shape.ctas, stream)
                       : launch<false, PRODUCT, N>(map, args, shape.cluster, shape.ctas, stream);
}

template <int N>
int run_products(const Matrix *matrices, int count, const Step *steps, int n, char *workspace, size_t bytes,
                 cudaStream_t stream) {
    CUtensorMap map;
    MTC_TRY(workspace_map(map, workspace, bytes));
    Args<N> gram;
    std::memset(&gram, 0, sizeof(gram));
    gram.table.count = count;
    for (int i = 0; i < count; ++i) gram.table.matrix[i] = matrices[i];
    gram.workspace = workspace;
    MTC_TRY(device_error_word(&gram.err));
    Args<N> square = gram, apply = gram;
    Shape gram_shape, square_shape, apply_shape;
    MTC_TRY(choose_shape(gram, kSymmetric, true, gram_shape));
    MTC_TRY(choose_shape(square, kSymmetric, false, square_shape));
    MTC_TRY(choose_shape(apply, kApply, false, apply_shape));
    for (int k = 0; k < n; ++k) {
        const Scales f = scales_of(steps[k], k == n - 1);
        gram.from = 0;
        gram.last = k % 2;  // (which X it is)
        gram.q = f.gram;
        gram.unit = f.d_unit;
        MTC_TRY((launch_product<kSymmetric, N>(map, gram, gram_shape, stream)));
        square.from = 1;
        square.q = f.square;
        square.p = f.p;
        square.r = f.r;
        square.b = f.b;
        square.c = f.c;
        square.unit = f.e_unit;
        MTC_TRY((launch_product<kSymmetric, N>(map, square, square_shape, stream)));
        apply.from = k % 2;
        apply.last = k == n - 1;
        apply.q = f.apply;
        apply.p = f.own;
        apply.r = f.a;
        MTC_TRY((launch_product<kApply, N>(map, apply, apply_shape, stream)));
    }
    return MTC_OK;
}

}  // namespace

int products(const Matrix *matrices, int count, const Step *steps, int n_steps, char *workspace, size_t bytes, cudaStream_t stream) {
    return count <= 8 ? run_products<8>(matrices, count, steps, n_steps, workspace, bytes, stream)
                      : run_products<kMostMatrices>(matrices, count, steps, n_steps, workspace, bytes, stream);
}

int whole_matrices(const Matrix *matrices, int count, const Step *steps, int n_steps, float eps, cudaStream_t stream) {
    WholeSteps w;
    std::memset(&w, 0, sizeof(w));
    w.n = n_steps;
    w.scale = steps[0].x;
    w.eps = eps;
    for (int k = 0; k < n_steps; ++k) w.step[k] = scales_of(steps[k], k == n_steps - 1);
    unsigned long long *err = nullptr;
    MTC_TRY(device_error_word(&err));
    for (int at = 0; at < count; at += kMostMatrices) {
        const int n = count - at < kMostMatrices ? count - at : kMostMatrices;
        MTC_TRY(with_table(matrices + at, n, [&](const auto &t) {
            constexpr int N = sizeof(t.matrix) / sizeof(t.matrix[0]);
            MTC_CUDA_TRY(cudaFuncSetAttribute(k_whole<N>, cudaFuncAttributeMaxDynamicSharedMemorySize, kWholeBytes));
            k_whole<N><<<n, kWholeThreads, kWholeBytes, stream>>>(t, w, err);
            return check_launch("orthogonalize (one tile)");
        }));
    }
    return MTC_OK;
}

}  // namespace ortho
}  // namespace mtc
