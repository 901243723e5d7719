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
// 256; either way a CTA stages 128 rows of A and 128 columns of B, 64 KB for 64 of K: rings of
// five stages of hi (free at the end of a piece) and two of lo (free after its cross terms), 32
// KB each.  Warp 0 loads (TMA: the workspace is one tensor of rows of 128 bytes), warp 1 issues,
// warps 4..11 are the epilogue, two for each quarter of the tensor memory's lanes.
// Every wait is bounded; on expiry the device error word is set and the roles leave.
#include <cuda_fp16.h>

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
constexpr int kHiStages = 5, kLoStages = 2, kStages = kHiStages + kLoStages;
constexpr int kPieceBlocks = 4;                  // blocks of K that are summed in tensor memory
constexpr int kSmemBytes = kStages * kStageBytes + 1024 + 256;
constexpr int kCtaThreads = 384;
constexpr float kCutOff = 0x1p-23f;              // what a sum loses a block, see above
constexpr int kEpilogueRegs = 208, kOtherRegs = 88;
static_assert(kSmemBytes <= 227 * 1024, "shared memory per CTA");
static_assert(256 * kEpilogueRegs + 128 * kOtherRegs <= kCtaThreads * 168, "registers of the launch (168 a thread)");
constexpr int kSumPitch = 132;                   // of a CTA's sums in shared memory, which the stages have left
static_assert(128 * kSumPitch * 4 <= kStages * kStageBytes, "sums");

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

__device__ __forceinline__ void load_half(void *dst, const CUtensorMap *map, uint64_t *bar, int row) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(0), "r"(row)
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

__device__ __forceinline__ void load_pairs(const char *from, float (&v)[8]) {
    const uint4 h = *reinterpret_cast<const uint4 *>(from), l = *reinterpret_cast<const uint4 *>(from + kOperandBytes);
    const uint32_t hw[4] = {h.x, h.y, h.z, h.w}, lw[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&hw[j]));
        const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&lw[j]));
        v[2 * j] = fmaf(b.x, 0x1p-11f, a.x);
        v[2 * j + 1] = fmaf(b.y, 0x1p-11f, a.y);
    }
}

__device__ __forceinline__ void store_pairs(char *to, const uint32_t (&w)[8]) {
    uint4 h, l;
    h.x = __byte_perm(w[0], w[1], 0x5410);
    h.y = __byte_perm(w[2], w[3], 0x5410);
    h.z = __byte_perm(w[4], w[5], 0x5410);
    h.w = __byte_perm(w[6], w[7], 0x5410);
    l.x = __byte_perm(w[0], w[1], 0x7632);
    l.y = __byte_perm(w[2], w[3], 0x7632);
    l.z = __byte_perm(w[4], w[5], 0x7632);
    l.w = __byte_perm(w[6], w[7], 0x7632);
    *reinterpret_cast<uint4 *>(to) = h;
    *reinterpret_cast<uint4 *>(to + kOperandBytes) = l;
}

// Eight columns, from `col` on, of a warp's 32 neighbouring rows: this lane's sums of products.
template <Product PRODUCT, int N>
__device__ __forceinline__ void finish(const Args<N> &a, const Matrix &mt, int row, int col, bool mirror, float (&v)[8]) {
    float *const d = reinterpret_cast<float *>(a.workspace + static_cast<int64_t>(mt.s_diagonal) * 128);
    float *const e = reinterpret_cast<float *>(a.workspace + static_cast<int64_t>(mt.b_diagonal) * 128);
    if (PRODUCT == kSymmetric) {
        float on = 0.0f;
        const bool own = row >= col && row < col + 8;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (row == col + j) on = v[j] * a.unit;
        if (a.from == 0) {
            if (own) d[row] = on;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] *= a.q;
        } else {
            float old[8];
            load_pairs(a.workspace + chunk_at(mt.s, mt.s_blocks, row, col), old);
            const float4 d0 = *reinterpret_cast<const float4 *>(d + col), d1 = *reinterpret_cast<const float4 *>(d + col + 4);
            const float dj[8] = {d0.x, d0.y, d0.z, d0.w, d1.x, d1.y, d1.z, d1.w}, di = d[row];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = fmaf(fmaf(a.r, di + dj[j], a.p), old[j], a.q * v[j]);
            if (own) e[row] = fmaf(fmaf(a.c, di, a.b), di, on);
        }
        if (own) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (row == col + j) v[j] = 0.0f;
        }
        uint32_t w[8];
        to_pairs(v, w);
        const int to = a.from == 0 ? mt.s : mt.b;
        store_pairs(a.workspace + chunk_at(to, mt.s_blocks, row, col), w);
        if (!mirror) return;
        // Rows become columns: of two neighbouring lanes and columns each lane gets two neighbours
        // of one row of the image.
        const int odd = row & 1;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const uint32_t other = __shfl_xor_sync(0xFFFFFFFFu, odd ? w[j] : w[j + 1], 1);
            const uint32_t left = odd ? other : w[j], right = odd ? w[j + 1] : other;
            char *at = a.workspace + chunk_at(to, mt.s_blocks, col + j + odd, row & ~7) + (row & 6) * 2;
            *reinterpret_cast<uint32_t *>(at) = __byte_perm(left, right, 0x5410);
            *reinterpret_cast<uint32_t *>(at + kOperandBytes) = __byte_perm(left, right, 0x7632);
        }
        return;
    }
    float old[8];
    load_pairs(a.workspace + chunk_at(mt.x[a.from], mt.x_blocks, row, col), old);
    const float factor = a.p * (a.r + e[row]);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = fmaf(factor, old[j], a.q * v[j]);
    if (!a.last) {
        uint32_t w[8];
        to_pairs(v, w);
        store_pairs(a.workspace + chunk_at(mt.x[a.from ^ 1], mt.x_blocks, row, col), w);
        return;
    }
    if (row >= mt.m || col >= mt.n) return;
    float *to = mt.dst + row * mt.out_rs + col * mt.out_cs;
    if (mt.out_cs == 1 && col + 8 <= mt.n && (reinterpret_cast<uintptr_t>(to) & 15) == 0) {
        reinterpret_cast<float4 *>(to)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4 *>(to)[1] = make_float4(v[4], v[5], v[6], v[7]);
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (col + j < mt.n) to[j * mt.out_cs] = v[j];
}

// Without PAIR, the CTAs of a cluster share the K of one tile and add their sums by way of their
// shared memory, each an equal share of the columns, in the order of the CTAs.
template <bool PAIR, Product PRODUCT, int N>
__global__ void __launch_bounds__(kCtaThreads, 1)
    k_step_product(const __grid_constant__ CUtensorMap map, const __grid_constant__ Args<N> args) {
    constexpr bool B_MN = PRODUCT == kApply;
    constexpr int kTile = PAIR ? 256 : 128, kColumns = kTile / 2;  // of an epilogue thread
    constexpr uint32_t kTmemCols = 2 * kTile;
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

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    uint32_t cluster_size;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(cluster_size));
    const int rank = static_cast<int>(cluster_rank());
    const int group = static_cast<int>(blockIdx.x / cluster_size), groups = static_cast<int>(gridDim.x / cluster_size);
    const int splits = PAIR ? 1 : static_cast<int>(cluster_size), split = PAIR ? 0 : rank;
    const int pair_rank = PAIR ? rank : 0;
    const bool leader = pair_rank == 0;

    if (threadIdx.x == 0) {
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
    const uint32_t tmem_base = *tmem_slot;
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
        int64_t piece = 0;
        bool ok = true;
        for (int u = group; u < args.units && ok; u += groups) {
            const Unit unit = unit_of<PRODUCT>(args, u, kTile);
            const Matrix &mt = args.table.matrix[unit.matrix];
            int kb0, kb1;
            k_range(mt, kb0, kb1);
            float acc[kColumns];
#pragma unroll
            for (int j = 0; j < kColumns; ++j) acc[j] = 0.0f;
            for (int kb = kb0; kb < kb1; kb += kPieceBlocks, ++piece) {
                const int b = static_cast<int>(piece & 1);
                if (!mbar_wait(&acc_full[b], static_cast<uint32_t>(piece >> 1) & 1u, abort_flag)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const float whole = 1.0f + (kb1 - kb < kPieceBlocks ? kb1 - kb : kPieceBlocks) * kCutOff;
                const uint32_t at = tmem_base + (static_cast<uint32_t>(quadrant * 32) << 16) +
                                    static_cast<uint32_t>(b * kTile + half * kColumns);
#pragma unroll
                for (int c = 0; c < kColumns / 64; ++c) {
                    uint32_t v[64];
                    tmem_ld64(at + static_cast<uint32_t>(c * 64), v);
#pragma unroll
                    for (int j = 0; j < 64; ++j) acc[c * 64 + j] = fmaf(__uint_as_float(v[j]), whole, acc[c * 64 + j]);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_remote(release[b]);
            }
            const int row0 = quadrant * 32 + lane;
            if (!PAIR && splits > 1) {
                // All MMAs of this CTA are done (and with them its loads): the stages hold the sums now.
                float *sums = reinterpret_cast<float *>(smem) + row0 * kSumPitch + half * kColumns;
#pragma unroll
                for (int j = 0; j < kColumns; j += 4)
                    *reinterpret_cast<float4 *>(sums + j) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
                break;  // one unit a cluster
            }
            if (!ok) break;
            const int row = unit.tm * kTile + pair_rank * 128 + row0, col = unit.tn * kTile + half * kColumns;
            const bool mirror = PRODUCT == kSymmetric && unit.tm != unit.tn;
#pragma unroll
            for (int j = 0; j < kColumns; j += 8) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = acc[j + i];
                finish<PRODUCT>(args, mt, row, col + j, mirror, v);
            }
            __syncwarp();
        }
        if (!ok) atomicCAS(args.err, 0ull, static_cast<unsigned long long>(MTC_ERR_RUNTIME));
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == 0) {
            if (lane == 0) {
                int64_t it = 0;
                bool ok = true;
                for (int u = group; u < args.units && ok; u += groups) {
                    const Unit unit = unit_of<PRODUCT>(args, u, kTile);
                    const Matrix &mt = args.table.matrix[unit.matrix];
                    int kb0, kb1;
                    k_range(mt, kb0, kb1);
                    const int ta = unit.tm * (kTile / 128) + pair_rank, tb = unit.tn * (kTile / 128) + pair_rank;
                    const bool of_x = PRODUCT == kSymmetric && args.from == 0;
                    const int a_at = PRODUCT == kApply ? mt.b : of_x ? mt.x[args.last] : mt.s;
                    const int a_blocks = of_x ? mt.x_blocks : mt.s_blocks;
                    const int b_at = PRODUCT == kApply ? mt.x[args.from] : a_at;
                    const int b_blocks = PRODUCT == kApply ? mt.x_blocks : a_blocks;
                    for (int kb = kb0; kb < kb1 && ok; ++kb, ++it) {
                        for (int lo = 0; lo < 2; ++lo) {
                            const int depth = lo ? kLoStages : kHiStages;
                            const int s = (lo ? kHiStages : 0) + static_cast<int>(it % depth);
                            if (!mbar_wait(&empty[s], (static_cast<uint32_t>(it / depth) & 1u) ^ 1u, abort_flag)) {
                                ok = false;
                                break;
                            }
                            unsigned char *st = smem + s * kStageBytes;
                            if (leader) mbar_expect_tx(&full[s], (PAIR ? 2 : 1) * kStageBytes);
                            const uint32_t fb = peer_addr(&full[s], 0);
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const int a_row = a_at + ((ta * a_blocks + kb) * 2 + lo) * 128 + h * 64;
                                const int b_row = B_MN ? b_at + ((kb / 2 * b_blocks + tb * 2 + h) * 2 + lo) * 128 + kb % 2 * 64
                                                       : b_at + ((tb * b_blocks + kb) * 2 + lo) * 128 + h * 64;
                                if (PAIR) {
                                    load_half_pair(st + h * kHalfBytes, &map, fb, a_row);
                                    load_half_pair(st + kOperandBytes + h * kHalfBytes, &map, fb, b_row);
                                } else {
                                    load_half(st + h * kHalfBytes, &map, &full[s], a_row);
                                    load_half(st + kOperandBytes + h * kHalfBytes, &map, &full[s], b_row);
                                }
                            }
                        }
                    }
                    if (!PAIR && splits > 1) break;
                }
                if (!ok) atomicCAS(args.err, 0ull, static_cast<unsigned long long>(MTC_ERR_RUNTIME));
                if (leader) {  // every stage issued has landed before the cluster exits
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
        } else if (warp == 1) {
            if (lane == 0 && leader) {
                constexpr uint32_t idesc = instr_desc<PAIR, B_MN>();
                constexpr uint64_t a_step = 32 >> 4, b_step = (B_MN ? 2048 : 32) >> 4;  // 16 of K
                int64_t it = 0, piece = 0;
                bool ok = true;
                for (int u = group; u < args.units && ok; u += groups) {
                    const Unit unit = unit_of<PRODUCT>(args, u, kTile);
                    int kb0, kb1;
                    k_range(args.table.matrix[unit.matrix], kb0, kb1);
                    for (int kb = kb0; kb < kb1 && ok; kb += kPieceBlocks, ++piece) {
                        const int n = kb1 - kb < kPieceBlocks ? kb1 - kb : kPieceBlocks;
                        const int b = static_cast<int>(piece & 1);
                        if (!mbar_wait(&acc_empty[b], (static_cast<uint32_t>(piece >> 1) & 1u) ^ 1u, abort_flag)) {
                            ok = false;
                            break;
                        }
                        const uint32_t d = tmem_base + static_cast<uint32_t>(b * kTile);
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
                            const uint64_t ah = operand_desc<false>(hi), bh = operand_desc<B_MN>(hi + kOperandBytes);
                            const uint64_t al = operand_desc<false>(lo), bl = operand_desc<B_MN>(lo + kOperandBytes);
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                mma<PAIR>(d, ah + k * a_step, bl + k * b_step, idesc, j > 0 || k > 0);
                                mma<PAIR>(d, al + k * a_step, bh + k * b_step, idesc, 1);
                            }
                            commit<PAIR>(&empty[sl]);
                        }
                        if (!ok) break;
                        for (int j = 0; j < n; ++j) {
                            const int sh = static_cast<int>((it + j) % kHiStages);
                            const uint32_t hi = smem_u32(smem + sh * kStageBytes);
                            const uint64_t ah = operand_desc<false>(hi), bh = operand_desc<B_MN>(hi + kOperandBytes);
                            if (j == 0) mma_scaled<PAIR>(d, ah, bh, idesc);
                            else mma<PAIR>(d, ah, bh, idesc, 1);
#pragma unroll
                            for (int k = 1; k < 4; ++k) mma<PAIR>(d, ah + k * a_step, bh + k * b_step, idesc, 1);
                            commit<PAIR>(&empty[sh]);
                        }
                        commit<PAIR>(&acc_full[b]);
                        it += n;
                    }
                    if (!PAIR && splits > 1) break;
                }
                if (!ok) atomicCAS(args.err, 0ull, static_cast<unsigned long long>(MTC_ERR_RUNTIME));
                // all MMAs are done before a CTA frees its tensor memory
                if (PAIR) umma_commit_pair_local(drain);
                else commit<false>(drain);
                for (long long i = 0; i < kWaitLimit && !mbar_try_wait(drain, 0u); ++i) {
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (cluster_size > 1) cluster_sync_all();  // the leader's MMAs have drained; all sums are in shared memory
    if (!PAIR && splits > 1) {
        if (warp >= 4 && group < args.units) {
            const Unit unit = unit_of<PRODUCT>(args, group, kTile);
            const Matrix &mt = args.table.matrix[unit.matrix];
            const int quadrant = warp % 4, half = (warp - 4) / 4, share = 64 / splits;
            const int row0 = quadrant * 32 + lane, col0 = rank * 2 * share + half * share;
            const bool mirror = PRODUCT == kSymmetric && unit.tm != unit.tn;
            const float *mine = reinterpret_cast<const float *>(smem) + row0 * kSumPitch + col0;
            for (int j = 0; j < share; j += 8) {
                float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
                for (int s = 0; s < splits; ++s) {
                    const uint32_t from = peer_addr(mine + j, static_cast<uint32_t>(s));
                    float x[8];
                    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                 : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]) : "r"(from) : "memory");
                    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                 : "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7]) : "r"(from + 16) : "memory");
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] += x[i];
                }
                finish<PRODUCT>(args, mt, unit.tm * kTile + row0, unit.tn * kTile + col0 + j, mirror, v);
            }
        }
        cluster_sync_all();  // the sums have been read
    }
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        if (PAIR)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols));
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols));
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

template <Product PRODUCT, int N>
int launch_product(const CUtensorMap &map, Args<N> &args, cudaStream_t stream) {
    const int sms = sm_count(current_device());
    bool pairs = true;
    int64_t blocks = INT_MAX;  // of K, of the matrix with the fewest
    for (int i = 0; i < args.table.count; ++i) {
        const Matrix &m = args.table.matrix[i];
        const int64_t k = ((PRODUCT == kSymmetric && args.from == 0 ? m.n : m.m) + kBlock - 1) / kBlock;
        pairs = pairs && tile_of(m.m) == 256;
        blocks = k < blocks ? k : blocks;
    }
    if (pairs) {
        const int64_t units = count_units(args.table, PRODUCT, 256);
        if (units >= sms / 2) {
            if (units >= INT_MAX) return fail(MTC_ERR_UNSUPPORTED, "orthogonalize: too many tiles");
            args.units = static_cast<int>(units);
            return launch<true, PRODUCT, N>(map, args, 2, sms / 2 * 2, stream);
        }
    }
    const int64_t units = count_units(args.table, PRODUCT, 128);
    if (units >= INT_MAX) return fail(MTC_ERR_UNSUPPORTED, "orthogonalize: too many tiles");
    args.units = static_cast<int>(units);
    int splits = 1;
    while (splits < 8 && units * splits * 2 <= sms && blocks >= splits * 4) splits *= 2;
    const int64_t ctas = splits > 1 ? units * splits : units < sms ? units : sms;
    return launch<false, PRODUCT, N>(map, args, splits, static_cast<int>(ctas), stream);
}

template <int N>
int all_steps(Args<N> &args, const CUtensorMap &map, const Step *steps, int n, cudaStream_t stream) {
    auto two = [](int e) { return std::ldexp(1.0, e); };
    for (int k = 0; k < n; ++k) {
        const Step &s = steps[k];
        args.from = 0;
        args.last = k % 2;  // (which X it is)
        args.q = static_cast<float>(two(s.s - 2 * s.x));
        args.unit = static_cast<float>(two(-2 * s.x));
        MTC_TRY((launch_product<kSymmetric, N>(map, args, stream)));
        args.from = 1;
        args.q = static_cast<float>(s.c * two(s.b_exp - 2 * s.s));
        args.p = static_cast<float>(s.b * two(s.b_exp - s.s));
        args.r = static_cast<float>(s.c * two(s.b_exp - s.s));
        args.b = s.b;
        args.c = s.c;
        args.unit = static_cast<float>(s.c * two(-2 * s.s));
        MTC_TRY((launch_product<kSymmetric, N>(map, args, stream)));
        const int to = k == n - 1 ? 0 : s.x_after;
        args.from = k % 2;
        args.last = k == n - 1;
        args.q = static_cast<float>(two(to - s.b_exp - s.x));
        args.p = static_cast<float>(two(to - s.x));
        args.r = s.a;
        MTC_TRY((launch_product<kApply, N>(map, args, stream)));
    }
    return MTC_OK;
}

template <int N>
int run_products(const Matrix *matrices, int count, const Step *steps, int n, char *workspace, size_t bytes,
                 cudaStream_t stream) {
    CUtensorMap map;
    MTC_TRY(workspace_map(map, workspace, bytes));
    Args<N> args;
    std::memset(&args, 0, sizeof(args));
    args.table.count = count;
    for (int i = 0; i < count; ++i) args.table.matrix[i] = matrices[i];
    args.workspace = workspace;
    MTC_TRY(device_error_word(&args.err));
    return all_steps(args, map, steps, n, stream);
}

}  // namespace

int products(const Matrix *matrices, int count, const Step *steps, int n_steps, char *workspace, size_t bytes, cudaStream_t stream) {
    return count <= 8 ? run_products<8>(matrices, count, steps, n_steps, workspace, bytes, stream)
                      : run_products<kMostMatrices>(matrices, count, steps, n_steps, workspace, bytes, stream);
}

}  // namespace ortho
}  // namespace mtc
