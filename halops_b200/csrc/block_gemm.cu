// FP8 products whose operands carry a float32 scale per block of 128 along K:
//
//   out[m, n] = sum over blocks b of sfa[m, b] * sfb[n / 128 or n, b] * sum over k in b of a[m, k] * w[n, k]
//
// dense, or with the rows of `a` in runs of one expert each.  The tensor cores' block scales are powers of two per 32 values,
// so a float32 scale cannot ride along with the MMA: the products of one block of 128 are summed in tensor memory (four MMAs,
// K = 32 each), and the sums then leave for registers, where they are scaled and added up in float32.
//
// Per CTA (one per SM, persistent over output tiles of 128 x BN, BN = 64, 128, 192 or 256):
//   8 warps (BN = 192: 12)  promotion: tcgen05.ld of a block's sums, accumulators += scale * sums (two columns an instruction); after the
//               last block the accumulators are rounded once and stored.  A thread has one row and a half (a third) of the tile's columns.
//   1 warp      TMA producer: A and B tiles (128-byte swizzle) into a ring of stages
//   1 warp      brings the scales of four blocks at a time into shared memory, multiplied where a row has one factor per block (loaded by the
//               threads that use them, a float of a row each, they took a sixth of the time: 8192 x 8192 x 8192 625 us, 537 without)
//   1 or 2 warps  issue the MMAs of a step (BN > 128: one block; else two, one each) into the next of 2 sets of buffers in tensor memory
//
// What bounds it.  A k-tile of 256 columns takes 850 to 870 cycles, 512 of them MMAs (ncu: the tensor pipe busy for 52 % of 4096 x 7168 x 2048, L2
// and the way from it for a third, issue slots for 39 %).  Without the promotion's products it takes 640 to 670; the rest is the round of
// the promotion (287 cycles of loads and 260 of products, one after the other in warps that wait together).  Large problems run
// at the power cap besides: 8192 x 8192 x 8192 takes 545 to 605 us at 1.38 GHz and 990 W (the MXFP8 kernel 432 at 1.17), 458 in a burst of a few
// milliseconds.  Measured and left:
// 16 promotion warps on 256 columns (registers spill; 595 us against 540), double-buffered loads (648), half of B's bytes, as a CTA pair
// would load (518, without what a pair's remote signals would add).
//
// Every mbarrier wait is bounded, as in the other GEMM kernels: a role that waits longer than kTimeoutNs records a code in the
// status word, raises the CTA's abort flag and all roles leave through the common teardown.

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"
#include "gemm_common.cuh"
#include "ptx.cuh"

namespace hq {
namespace {

constexpr int kTileM = 128;
constexpr int kBlockK = 128;  // values, and bytes, of a k-tile row
constexpr int kMaxExperts = 1024;
constexpr int kSmemBudget = 232448;
constexpr int kGroupK = 4;      // k-tiles whose scales are brought together
constexpr int kScaleSlots = 2;  // such groups in shared memory

struct BlockBars {
    uint64_t full[8];
    uint64_t empty[8];
    uint64_t acc_full[2];
    uint64_t acc_empty[2];
    uint64_t sf_full[kScaleSlots];
    uint64_t sf_empty[kScaleSlots];
    uint32_t tmem_base;
    uint32_t abort;
};

template <int BN, bool kRowScales>
struct BlockCfg {
    static constexpr int kParts = BN == 192 ? 3 : 2;  // groups of four warps that share a tile's columns
    static constexpr int kPromoWarps = 4 * kParts;
    static constexpr int kLoadWarp = kPromoWarps, kScaleWarp = kPromoWarps + 1, kMmaWarp = kPromoWarps + 2;  // and kMmaWarp + 1
    // k-tiles of a step, which share a stage and a set of buffers: what a step's waits and signals cost (400 to 500 cycles from role to
    // role) is more than a narrow tile's k-tile has to do, 16 x 4096 x 7168 on 64 columns takes 11.8 us in steps of two and 13.1 of one,
    // 8192 x 8192 x 8192 on 128 columns 579 and 615
    static constexpr int kStep = BN > 128 ? 1 : 2;
    static constexpr int kABytes = kTileM * kBlockK;  // per k-tile
    static constexpr int kBBytes = BN * kBlockK;
    static constexpr int kStageBytes = kStep * (kABytes + kBBytes);
    static constexpr int kBarBytes = 512;
    static constexpr int kTableBytes = (kMaxExperts + 8) * 8;                // grouped: row tiles before, first row of, each expert
    static constexpr int kWeightBlocks = kRowScales ? 1 : (BN + 127) / 128;  // blocks of 128 weight rows that a tile spans
    // a k-tile's scales: per row of the tile one for each of its blocks of weights (the product of both), or (kRowScales) the rows' and then the columns'
    static constexpr int kScales = kRowScales ? kTileM + BN : kTileM * kWeightBlocks;
    static constexpr int kScaleBytes = kScaleSlots * kGroupK * kScales * 4;
    // a warp's finished 32 x 32 values on their way to a TMA store; all of a 256-wide tile's at a time
    static constexpr int kEpiSlots = kRowScales ? 0 : BN == 256 ? 4 : BN == 192 ? 2 : 1;
    static constexpr int kEpiBytes = kPromoWarps * kEpiSlots * 2048;
    static constexpr int kExtra = kBarBytes + kTableBytes + kScaleBytes + kEpiBytes + 1024;
    static constexpr int kFit = (kSmemBudget - kExtra) / kStageBytes;
    static constexpr int kStages = kFit;
    static constexpr int kSmemBytes = kStages * kStageBytes + kExtra;
    static constexpr int kBufs = 2;  // of kStep accumulators each
    static constexpr int kTmemCols = BN == 192 ? 512 : kBufs * kStep * BN;  // (a power of two)
    static constexpr int kCols = BN / kParts;  // columns of a promotion warp
    static constexpr int kLd = BN == 64 || BN == 192 ? 32 : 16;  // of which one load brings
    static constexpr int kThreads = (kPromoWarps + 4) * 32;
    // BN = 256: 128 accumulators a thread; the third warpgroup gives registers to the other two (168 * 384 = 208 * 256 + 88 * 128)
    static constexpr bool kRegSplit = BN == 256;
    static_assert(sizeof(BlockBars) <= kBarBytes && kStages >= 3 && kStages <= 8 && kTmemCols <= 512, "budgets");
    static_assert(BN > 128 || kTileM * (BN + 4) * 4 <= kStages * kStageBytes, "split-K partial sums fit into the ring");
    static_assert(kRowScales || kCols / 32 % kEpiSlots == 0, "a tile's pieces go round the slots as a whole");
};

struct BlockArgs {
    const float* sfa;
    const float* sfb;
    void* out;
    const int* offsets;  // grouped: first row of each expert, and the end of the last
    int64_t ldo;
    int m, n, k_tiles, tiles_m, tiles_n;
    int n_blocks;   // scales of the second operand per expert along N (rows of sfb)
    int experts;
    int box_rows;   // rows of `a` per copy
    int out_type;   // HQ_DTYPE_*
    int out_align;  // 32, 16, 4 or 2: bytes that every row of the output starts on
    int staged;     // 16-bit output that TMA can store
    int split;      // CTAs of a cluster that share a tile's k-tiles
    int wide_scales;  // both operands' scales are on 16 bytes
    int pdl;
};

struct BlockTile {
    int row0, valid, n0, expert;
};

// The sequence of a CTA's tiles; every role walks it for itself.
template <int BN, bool kGrouped>
struct BlockWalk {
    const BlockArgs& p;
    const int* const tiles_before;  // grouped, in shared memory: [experts + 1]
    const int* const first_row;
    int tile;
    const int step, total;
    __device__ __forceinline__ BlockWalk(const BlockArgs& args, const int* tables, int first, int step_)
        : p(args), tiles_before(tables), first_row(tables + kMaxExperts + 8), tile(first), step(step_),
          total(kGrouped ? tables[args.experts] * args.tiles_n : args.tiles_m * args.tiles_n) {}
    __device__ __forceinline__ bool next(BlockTile& t) {
        if (tile >= total) return false;
        if constexpr (kGrouped) {
            // the expert whose tiles hold this one
            int lo = 0, hi = p.experts;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (tiles_before[mid] * p.tiles_n <= tile) lo = mid; else hi = mid;
            }
            // within an expert down the rows first: the CTAs that run at the same time share the weight's tiles
            const int row_tiles = tiles_before[lo + 1] - tiles_before[lo];
            const int r = tile - tiles_before[lo] * p.tiles_n;
            const int n_tile = r / row_tiles;
            t.expert = lo;
            t.row0 = first_row[lo] + (r - n_tile * row_tiles) * kTileM;
            t.valid = min(kTileM, first_row[lo + 1] - t.row0);
            t.n0 = n_tile * BN;
        } else {
            // groups of 8 row tiles, then across the columns: one wave of CTAs shares a small set of tiles in L2
            constexpr int kGroup = 8;
            const int per = kGroup * p.tiles_n;
            const int g = tile / per, first_m = g * kGroup;
            const int gsz = min(kGroup, p.tiles_m - first_m);
            const int r = tile - g * per;
            const int n_tile = r / gsz;
            t.expert = 0;
            t.row0 = (first_m + r - n_tile * gsz) * kTileM;
            t.valid = min(kTileM, p.m - t.row0);
            t.n0 = n_tile * BN;
        }
        tile += step;
        return true;
    }
};

// d (+)= a . b^T, K = 32 e4m3 values, float32 sums in tensor memory.
__device__ __forceinline__ void mma_e4m3(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
        "}" ::"r"(d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// 32 lanes x 32 or 16 columns; the values are there behind load_wait on the same registers.
__device__ __forceinline__ void load_columns(uint32_t taddr, uint32_t (&r)[32]) { ptx::tc_load_32x32(taddr, r); }
__device__ __forceinline__ void load_columns(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void load_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                   "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                   "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void load_wait(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}

// 16 lanes x 32 columns as fragments of 8 x 8: register 4 g + 2 h + i is row lane / 4 + 8 h, column 8 g + 2 (lane % 4) + i.
__device__ __forceinline__ void load_fragments(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}

// Scales, which the preceding kernel may still write before pdl_wait: volatile, so that they stay behind it.  (As plain loads, among which
// the compiler keeps the order of the stores to shared memory, the widest tile spilled.)
__device__ __forceinline__ float load_scale(const float* p) {
    float v;
    asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ float4 load_scales(const float* p) {
    float4 v;
    asm volatile("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
    return v;
}

// (a, b) += (x, y) * s as one packed instruction.  It needs the issue slots of two scalar ones, but not their operand reads: 128 columns
// of 8 warps, loads included, take 292 cycles with it and 421 with fmaf.
__device__ __forceinline__ void add_scaled2(float& a, float& b, uint32_t x, uint32_t y, float s) {
    asm("{\n\t"
        ".reg .b64 v, f, c;\n\t"
        "mov.b64 v, {%2, %3};\n\t"
        "mov.b64 f, {%4, %4};\n\t"
        "mov.b64 c, {%0, %1};\n\t"
        "fma.rn.f32x2 c, v, f, c;\n\t"
        "mov.b64 {%0, %1}, c;\n\t"
        "}"
        : "+f"(a), "+f"(b)
        : "r"(x), "r"(y), "f"(s));
}
// (x, y) *= (s, t)
__device__ __forceinline__ void scale2(uint32_t& x, uint32_t& y, float s, float t) {
    asm("{\n\t"
        ".reg .b64 v, f;\n\t"
        "mov.b64 v, {%0, %1};\n\t"
        "mov.b64 f, {%2, %3};\n\t"
        "mul.rn.f32x2 v, v, f;\n\t"
        "mov.b64 {%0, %1}, v;\n\t"
        "}"
        : "+r"(x), "+r"(y)
        : "f"(s), "f"(t));
}

__device__ __forceinline__ uint32_t pack16(float lo, float hi, int type) {
    uint32_t r;
    if (type == HQ_DTYPE_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        memcpy(&r, &h, 4);
    } else {
        const __half2 h = __floats2half2_rn(lo, hi);
        memcpy(&r, &h, 4);
    }
    return r;
}

__device__ __forceinline__ void store_32_bytes(void* p, const uint32_t (&w)[8], int align) {
    if (align >= 32) {
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                     "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                     : "memory");
    } else {
        reinterpret_cast<uint4*>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
        reinterpret_cast<uint4*>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
}

// kN neighbouring values of a row from column `col` on, `left` of which exist.
template <int kN>
__device__ __forceinline__ void store_values(const float (&f)[kN], void* out, int64_t at, int left, int type, int align) {
    if (type == HQ_DTYPE_FP32) {
        float* const o = static_cast<float*>(out) + at;
        if (left >= kN && align >= 16) {
            if constexpr (kN >= 8) {
#pragma unroll
                for (int i = 0; i < kN; i += 8) {
                    uint32_t w[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(f[i + j]);
                    store_32_bytes(o + i, w, align);
                }
            } else {
#pragma unroll
                for (int i = 0; i < kN; i += 2) *reinterpret_cast<float2*>(o + i) = make_float2(f[i], f[i + 1]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                if (i < left) o[i] = f[i];
            }
        }
        return;
    }
    uint32_t w[kN / 2];
#pragma unroll
    for (int i = 0; i < kN / 2; ++i) w[i] = pack16(f[2 * i], f[2 * i + 1], type);
    uint16_t* const o = static_cast<uint16_t*>(out) + at;
    if (left >= kN && align >= 16) {
        if constexpr (kN == 16) {
            store_32_bytes(o, w, align);
        } else if constexpr (kN == 4) {
            *reinterpret_cast<uint2*>(o) = make_uint2(w[0], w[1]);
        } else {
            *reinterpret_cast<uint32_t*>(o) = w[0];
        }
    } else {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            if (i < left) o[i] = uint16_t(w[i / 2] >> (i % 2 * 16));
        }
    }
}

// ---------------------------------------------------------------------------- MMA issuers
//
// One for each k-tile of a step.  Every k-tile has a buffer of its own, so nothing has to be kept in order between them.  (Two that took
// turns at the steps would skip phases of the stages' barriers, and a wait for the next but one is over before it began.)
//
// kEach: an issuer's k-tile u is a constant and every instruction elected for itself, which keeps its operands warp-uniform (the same mask
// elects the same lane each time, so a commit follows the MMAs of its own thread).  It is for tiles of up to 128 columns with scales of
// blocks, where the round between the roles counts most: 4736 x 768 x 4096 on 64 columns 22.7 -> 21.1 us, 4736 x 1024 x 4096 on 128 23.3 ->
// 22.9, 1 x 7168 x 2048 5.8 -> 5.3.  Wide tiles and scales of rows have one copy of the loop and one election a step: 7168 x 2048 x 4096
// 73.4 us against 74.8, 1024 x 2048 x 256 with scales of rows 7.0 against 7.2.  (A half of 256 columns for each of two issuers, with
// buffers and signals of its own: no faster.)
template <int BN, bool kRowScales, bool kGrouped, bool kEach>
__device__ __forceinline__ void issue_mmas(const BlockArgs& p, const int* tables, int first, int step, int k_begin, int k_end, BlockBars* bars,
                                           volatile uint32_t* abort, uint32_t a_base, uint32_t b_base, uint32_t tmem, uint32_t u) {
    using C = BlockCfg<BN, kRowScales>;
    // float32 sums, e4m3 operands, both K-major; N >> 3, M >> 4
    constexpr uint32_t idesc = (1u << 4) | (uint32_t(BN >> 3) << 17) | (uint32_t(kTileM >> 4) << 24);
    // (addresses are in the descriptors' low bits, in units of 16 bytes; K = 32 bytes is a step of 2 inside of the swizzle atom)
    const uint64_t adesc0 = ptx::smem_desc(a_base + u * C::kABytes, 16, 1024, 2);
    const uint64_t bdesc0 = ptx::smem_desc(b_base + u * C::kBBytes, 16, 1024, 2);
    uint32_t it = 0;
    bool ok = true;
    BlockWalk<BN, kGrouped> walk(p, tables, first, step);
    BlockTile t;
    while (ok && walk.next(t)) {
        for (int kt = k_begin; kt < k_end; kt += C::kStep, ++it) {
            const uint32_t s = it % C::kStages, buf = it % C::kBufs;
            ok = wait_bars<C::kRegSplit>(ptx::smem_u32(&bars->full[s]), (it / C::kStages) & 1u, true, ptx::smem_u32(&bars->acc_empty[buf]),
                                         ((it / C::kBufs) & 1u) ^ 1u, abort, kStatusMma);
            if (!ok) break;
            ptx::tc_fence_after();
            const uint64_t adesc = adesc0 + s * (C::kStep * C::kABytes >> 4), bdesc = bdesc0 + s * (C::kStep * C::kBBytes >> 4);
            const uint32_t d = tmem + (buf * C::kStep + u) * BN;
            if constexpr (kEach) {
                if (ptx::elect_one()) mma_e4m3(d, adesc, bdesc, idesc, 0u);
                if (ptx::elect_one()) mma_e4m3(d, adesc + 2, bdesc + 2, idesc, 1u);
                if (ptx::elect_one()) mma_e4m3(d, adesc + 4, bdesc + 4, idesc, 1u);
                if (ptx::elect_one()) mma_e4m3(d, adesc + 6, bdesc + 6, idesc, 1u);
                if (ptx::elect_one()) ptx::tc_commit(ptx::smem_u32(&bars->acc_full[buf]));
                if (ptx::elect_one()) ptx::tc_commit(ptx::smem_u32(&bars->empty[s]));
            } else if (ptx::elect_one()) {
                mma_e4m3(d, adesc, bdesc, idesc, 0u);
                mma_e4m3(d, adesc + 2, bdesc + 2, idesc, 1u);
                mma_e4m3(d, adesc + 4, bdesc + 4, idesc, 1u);
                mma_e4m3(d, adesc + 6, bdesc + 6, idesc, 1u);
                ptx::tc_commit(ptx::smem_u32(&bars->acc_full[buf]));
                ptx::tc_commit(ptx::smem_u32(&bars->empty[s]));
            }
        }
    }
}

// kAnyRows: output rows on no 16 bytes.  (An instantiation of its own: as a branch it cost the 256-wide tile registers, 8192 x 8192 x 8192
// 580 -> 615 us.)
template <int BN, bool kRowScales, bool kGrouped, bool kSplit, bool kAnyRows>
__global__ void __launch_bounds__((BlockCfg<BN, kRowScales>::kThreads), 1)
block_gemm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const __grid_constant__ CUtensorMap tm_d,
                  const __grid_constant__ BlockArgs p) {
    using C = BlockCfg<BN, kRowScales>;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t a_base = ptx::smem_u32(smem);
    const uint32_t b_base = a_base + C::kStages * C::kStep * C::kABytes;
    constexpr int kBarOffset = C::kStages * C::kStageBytes + C::kEpiBytes;
    BlockBars* const bars = reinterpret_cast<BlockBars*>(smem + kBarOffset);
    int* const tables = reinterpret_cast<int*>(smem + kBarOffset + C::kBarBytes);
    float* const scales = reinterpret_cast<float*>(smem + kBarOffset + C::kBarBytes + C::kTableBytes);
    const uint32_t epi_base = a_base + C::kStages * C::kStageBytes;
    volatile uint32_t* const abort = &bars->abort;
    const int warp = warp_index();
    const int lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            ptx::mbar_init(ptx::smem_u32(&bars->full[s]), 1);
            ptx::mbar_init(ptx::smem_u32(&bars->empty[s]), C::kStep);  // one commit per k-tile
        }
        for (int s = 0; s < C::kBufs; ++s) {
            ptx::mbar_init(ptx::smem_u32(&bars->acc_full[s]), C::kStep);
            ptx::mbar_init(ptx::smem_u32(&bars->acc_empty[s]), C::kPromoWarps);
        }
        for (int s = 0; s < kScaleSlots; ++s) {
            ptx::mbar_init(ptx::smem_u32(&bars->sf_full[s]), 1);
            ptx::mbar_init(ptx::smem_u32(&bars->sf_empty[s]), C::kPromoWarps);
        }
        bars->abort = 0;
        ptx::fence_mbar_init();
        ptx::prefetch_tmap(&tm_a);
        ptx::prefetch_tmap(&tm_b);
        if (p.staged != 0) ptx::prefetch_tmap(&tm_d);
    }
    if (warp == C::kMmaWarp) {
        ptx::tmem_alloc<1>(ptx::smem_u32(&bars->tmem_base), C::kTmemCols);
        ptx::tmem_relinquish<1>();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = bars->tmem_base;

    // A dense problem of few rows is bound by the weight's way from HBM: its first k-tiles are asked for into L2 while the preceding kernel
    // finishes (a hint, so it may have been that kernel that wrote the weight).
    if constexpr (!kGrouped) {
        if (warp == C::kLoadWarp && p.pdl != 0 && p.tiles_m == 1) {
            const int share = kSplit ? int(blockIdx.x) % p.split : 0, parts = kSplit ? p.split : 1;
            const int n0 = (kSplit ? int(blockIdx.x) / parts : int(blockIdx.x)) * BN;
            const int from = int(int64_t(p.k_tiles) * share / parts), to = int(int64_t(p.k_tiles) * (share + 1) / parts);
            for (int kt = from; kt < min(to, from + 16); ++kt) {
                if (ptx::elect_one()) ptx::tma_prefetch_2d(&tm_b, kt * kBlockK, n0);
            }
        }
    }
    // nothing below may run before the preceding kernel's writes are visible (so no load below is one of constant data)
    ptx::pdl_wait();
    if constexpr (kGrouped) {
        if (warp == 0) {
            // row tiles before each expert; offsets that go back or point outside are clamped, so that no row is touched that is not there
            int before = 0, last = 0;
            int* const first_row = tables + kMaxExperts + 8;
            for (int e0 = 0; e0 <= p.experts; e0 += 32) {
                const int e = e0 + lane;
                int start = e <= p.experts ? min(max(p.offsets[e], 0), p.m) : 0;
#pragma unroll
                for (int d = 1; d < 32; d *= 2) {
                    const int v = __shfl_up_sync(0xffffffffu, start, d);
                    if (lane >= d) start = max(start, v);
                }
                start = max(start, last);
                int prev = __shfl_up_sync(0xffffffffu, start, 1);
                if (lane == 0) prev = last;
                // tiles of expert e - 1
                int sum = e >= 1 && e <= p.experts ? (start - prev + kTileM - 1) / kTileM : 0;
#pragma unroll
                for (int d = 1; d < 32; d *= 2) {
                    const int v = __shfl_up_sync(0xffffffffu, sum, d);
                    if (lane >= d) sum += v;
                }
                if (e <= p.experts) {
                    first_row[e] = start;
                    tables[e] = before + sum;
                }
                before += __shfl_sync(0xffffffffu, sum, 31);
                last = __shfl_sync(0xffffffffu, start, 31);
            }
        }
        __syncthreads();
    }
    const int rank = kSplit ? int(blockIdx.x) % p.split : 0;
    const int first = kSplit ? int(blockIdx.x) / p.split : int(blockIdx.x);
    const int step = kSplit ? int(gridDim.x) / p.split : int(gridDim.x);
    // (whole steps per CTA of a cluster; a step that sticks out beyond K reads zeros there and has zeros for scales)
    const int steps = (p.k_tiles + C::kStep - 1) / C::kStep;
    const int k_begin = kSplit ? int(int64_t(steps) * rank / p.split) * C::kStep : 0;
    const int k_end = kSplit ? min(int(int64_t(steps) * (rank + 1) / p.split) * C::kStep, p.k_tiles) : p.k_tiles;

    if (warp >= C::kPromoWarps) {
        if constexpr (C::kRegSplit) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == C::kLoadWarp) {
            // ------------------------------------------------------------ TMA producer
            uint32_t it = 0;
            bool ok = true;
            BlockWalk<BN, kGrouped> walk(p, tables, first, step);
            BlockTile t;
            while (ok && walk.next(t)) {
                const int boxes = (t.valid + p.box_rows - 1) / p.box_rows;
                const int b_row = t.expert * p.n + t.n0;
                const uint32_t bytes = C::kStep * uint32_t(boxes * p.box_rows * kBlockK + C::kBBytes);
                for (int kt = k_begin; kt < k_end; kt += C::kStep, ++it) {
                    const uint32_t s = it % C::kStages;
                    ok = wait_bar<C::kRegSplit>(ptx::smem_u32(&bars->empty[s]), ((it / C::kStages) & 1u) ^ 1u, abort, kStatusProducer);
                    if (!ok) break;
                    const uint32_t full = ptx::smem_u32(&bars->full[s]);
                    const uint32_t a_to = a_base + s * (C::kStep * C::kABytes), b_to = b_base + s * (C::kStep * C::kBBytes);
                    if (ptx::elect_one()) {
                        ptx::mbar_arrive_expect_tx(full, bytes);
#pragma unroll
                        for (int u = 0; u < C::kStep; ++u) {
                            ptx::tma_load_2d(b_to + u * C::kBBytes, &tm_b, (kt + u) * kBlockK, b_row, full);
                            ptx::tma_load_2d(a_to + u * C::kABytes, &tm_a, (kt + u) * kBlockK, t.row0, full);
                        }
                    }
                    for (int b = 1; b < boxes; ++b) {
                        const int skip = b * p.box_rows;
                        if (ptx::elect_one()) {
#pragma unroll
                            for (int u = 0; u < C::kStep; ++u) {
                                ptx::tma_load_2d(a_to + u * C::kABytes + skip * kBlockK, &tm_a, (kt + u) * kBlockK, t.row0 + skip, full);
                            }
                        }
                    }
                }
            }
            ptx::pdl_launch_dependents();
            // the releases of the last stages arrive in this CTA's shared memory: it is not left before they have
            for (uint32_t d = it > uint32_t(C::kStages) ? it - C::kStages : 0u; ok && d < it; ++d) {
                ok = wait_bar<C::kRegSplit>(ptx::smem_u32(&bars->empty[d % C::kStages]), (d / C::kStages) & 1u, abort, kStatusProducer);
            }
        } else if (warp >= C::kMmaWarp && warp < C::kMmaWarp + C::kStep) {
            constexpr bool kEach = C::kStep == 2 && !kRowScales;
            if (kEach && warp == C::kMmaWarp) {
                issue_mmas<BN, kRowScales, kGrouped, kEach>(p, tables, first, step, k_begin, k_end, bars, abort, a_base, b_base, tmem, 0u);
            } else {
                const uint32_t u = kEach ? 1u : warp - C::kMmaWarp;
                issue_mmas<BN, kRowScales, kGrouped, kEach>(p, tables, first, step, k_begin, k_end, bars, abort, a_base, b_base, tmem, u);
            }
        } else if (warp == C::kScaleWarp) {
            // ------------------------------------------------------------ scales
            // A group's are in registers before its slot is free.  A lane has every 32nd row; four neighbouring k-tiles are one load where
            // they lie on 16 bytes.
            constexpr int kRowsA = kTileM / 32, kRowsB = kRowScales ? BN / 32 : 1;
            const bool wide = p.k_tiles % 4 == 0 && p.wide_scales != 0;
            const auto load4 = [&](const float* q, int k0, float (&v)[kGroupK]) {
                if (wide && k0 % 4 == 0 && k0 + kGroupK <= k_end) {
                    const float4 f = load_scales(q + k0);
                    v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
                } else {
#pragma unroll
                    for (int i = 0; i < kGroupK; ++i) v[i] = k0 + i < k_end ? load_scale(q + k0 + i) : 0.0f;
                }
            };
            uint32_t group = 0;
            bool ok = true;
            BlockWalk<BN, kGrouped> walk(p, tables, first, step);
            BlockTile t;
            while (ok && walk.next(t)) {
                const float* const pa = p.sfa + int64_t(t.row0) * p.k_tiles;
                const int n_block = t.n0 / 128;
                for (int k0 = k_begin; k0 < k_end; k0 += kGroupK, ++group) {
                    float a[kRowsA][kGroupK], b[kRowScales ? kRowsB : C::kWeightBlocks][kGroupK];
#pragma unroll
                    for (int j = 0; j < kRowsA; ++j) load4(pa + int64_t(min(j * 32 + lane, t.valid - 1)) * p.k_tiles, k0, a[j]);
                    if constexpr (kRowScales) {
#pragma unroll
                        for (int j = 0; j < kRowsB; ++j) load4(p.sfb + int64_t(min(t.n0 + j * 32 + lane, p.n - 1)) * p.k_tiles, k0, b[j]);
                    } else {
#pragma unroll
                        for (int j = 0; j < C::kWeightBlocks; ++j) {
                            load4(p.sfb + (int64_t(t.expert) * p.n_blocks + min(n_block + j, p.n_blocks - 1)) * p.k_tiles, k0, b[j]);
                        }
                    }
                    const uint32_t slot = group % kScaleSlots;
                    ok = wait_bar<C::kRegSplit>(ptx::smem_u32(&bars->sf_empty[slot]), ((group / kScaleSlots) & 1u) ^ 1u, abort, kStatusProducer);
                    if (!ok) break;
                    float* const to = scales + slot * (kGroupK * C::kScales) + lane;
#pragma unroll
                    for (int i = 0; i < kGroupK; ++i) {
#pragma unroll
                        for (int j = 0; j < kRowsA; ++j) {
                            if constexpr (kRowScales) {
                                to[i * C::kScales + j * 32] = a[j][i];
                            } else {
#pragma unroll
                                for (int h = 0; h < C::kWeightBlocks; ++h) to[i * C::kScales + h * kTileM + j * 32] = a[j][i] * b[h][i];
                            }
                        }
                        if constexpr (kRowScales) {
#pragma unroll
                            for (int j = 0; j < kRowsB; ++j) to[i * C::kScales + kTileM + j * 32] = b[j][i];
                        }
                    }
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&bars->sf_full[slot]));
                }
            }
        }
    } else {
        // ------------------------------------------------------------ promotion and epilogue
        if constexpr (C::kRegSplit) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int quarter = warp & 3, part = warp >> 2;  // lanes of tensor memory, columns
        const int row = quarter * 32 + lane;
        const uint32_t taddr = tmem + (uint32_t(quarter * 32) << 16) + part * C::kCols;
        uint32_t it = 0, group = 0;
        bool ok = true;
        BlockWalk<BN, kGrouped> walk(p, tables, first, step);
        BlockTile t;
        while (ok && walk.next(t)) {
            float acc[C::kCols];
#pragma unroll
            for (int i = 0; i < C::kCols; ++i) acc[i] = 0.0f;
            const bool row_ok = row < t.valid;
            const bool busy = quarter * 32 < t.valid;  // warp-uniform
            for (int k0 = k_begin; ok && k0 < k_end; k0 += kGroupK, ++group) {
                const uint32_t slot = group % kScaleSlots;
                ok = wait_bar<C::kRegSplit>(ptx::smem_u32(&bars->sf_full[slot]), (group / kScaleSlots) & 1u, abort, kStatusEpilogue);
                if (!ok) break;
                const float* const from = scales + slot * (kGroupK * C::kScales);
#pragma unroll
                for (int i = 0; i < kGroupK; i += C::kStep) {
                    if (k0 + i >= k_end) break;
                    const uint32_t buf = it % C::kBufs;
                    float s[C::kStep][kRowScales ? 4 : 1];
#pragma unroll
                    for (int u = 0; u < C::kStep; ++u) {
                        if constexpr (kRowScales) {
#pragma unroll
                            for (int q = 0; q < 4; ++q) s[u][q] = from[(i + u) * C::kScales + quarter * 32 + q * 8 + lane / 4];
                        } else {
                            s[u][0] = from[(i + u) * C::kScales + (C::kWeightBlocks == 2 ? (t.n0 % 128 + part * C::kCols) / 128 * kTileM : 0) + row];
                        }
                    }
                    ok = wait_bar<C::kRegSplit>(ptx::smem_u32(&bars->acc_full[buf]), (it / C::kBufs) & 1u, abort, kStatusEpilogue);
                    if (!ok) break;
                    if (busy) {
                        ptx::tc_fence_after();
                        const auto drained = [&] {
                            ptx::tc_fence_before();
                            __syncwarp();
                            if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&bars->acc_empty[buf]));
                        };
                        if constexpr (kRowScales) {
                            // fragments: a thread has 4 rows and 2 of 8 columns, so that it reads a quarter of the columns' scales (with a row and
                            // all columns, the shared-memory reads of 128 x 128 scales a k-tile took longer than its products)
#pragma unroll
                            for (int c = 0; c < C::kCols; c += 32) {
#pragma unroll
                                for (int u = 0; u < C::kStep; ++u) {
                                    uint32_t r[2][16];
                                    load_fragments(taddr + (buf * C::kStep + u) * BN + c, r[0]);
                                    load_fragments(taddr + (16u << 16) + (buf * C::kStep + u) * BN + c, r[1]);
                                    const float* const col = from + (i + u) * C::kScales + kTileM + part * C::kCols + c + lane % 4 * 2;
                                    float2 w[4];
#pragma unroll
                                    for (int g = 0; g < 4; ++g) w[g] = *reinterpret_cast<const float2*>(col + g * 8);
                                    load_wait(r[0]);
                                    load_wait(r[1]);
                                    if (c + 32 == C::kCols && u + 1 == C::kStep) drained();
#pragma unroll
                                    for (int g = 0; g < 4; ++g) {
#pragma unroll
                                        for (int q = 0; q < 4; ++q) {
                                            uint32_t &x = r[q / 2][g * 4 + q % 2 * 2], &y = r[q / 2][g * 4 + q % 2 * 2 + 1];
                                            float* const to = acc + c + (g * 4 + q) * 2;
                                            scale2(x, y, w[g].x, w[g].y);
                                            add_scaled2(to[0], to[1], x, y, s[u][q]);
                                        }
                                    }
                                }
                            }
                        } else {
                            constexpr int kLd = C::kLd;
#pragma unroll
                            for (int c = 0; c < C::kCols; c += kLd) {
                                uint32_t r[C::kStep][kLd];
#pragma unroll
                                for (int u = 0; u < C::kStep; ++u) load_columns(taddr + (buf * C::kStep + u) * BN + c, r[u]);
#pragma unroll
                                for (int u = 0; u < C::kStep; ++u) load_wait(r[u]);
                                if (c + kLd == C::kCols) drained();
#pragma unroll
                                for (int u = 0; u < C::kStep; ++u) {
#pragma unroll
                                    for (int j = 0; j < kLd; j += 2) add_scaled2(acc[c + j], acc[c + j + 1], r[u][j], r[u][j + 1], s[u][0]);
                                }
                            }
                        }
                    } else if (lane == 0) {
                        ptx::mbar_arrive(ptx::smem_u32(&bars->acc_empty[buf]));
                    }
                    ++it;
                }
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&bars->sf_empty[slot]));
            }
            if (!ok) break;
            if constexpr (kSplit) {
                // this CTA's sums into its own ring, which nothing uses any more (the last MMAs are done); lines of BN + 4 values
                // keep the lanes' 16-byte stores apart
                if (busy) {
                    float* const line = reinterpret_cast<float*>(smem) + row * (BN + 4) + part * C::kCols;
#pragma unroll
                    for (int c = 0; c < C::kCols; c += 4) {
                        *reinterpret_cast<float4*>(line + c) = make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
                    }
                }
            } else if constexpr (kRowScales) {
#pragma unroll
                for (int c = 0; c < C::kCols; c += 8) {
                    const int col = t.n0 + part * C::kCols + c + lane % 4 * 2;
                    if (col >= p.n) continue;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int r = quarter * 32 + q * 8 + lane / 4;
                        if (r < t.valid) {
                            const float f[2] = {acc[(c / 8 * 4 + q) * 2], acc[(c / 8 * 4 + q) * 2 + 1]};
                            store_values<2>(f, p.out, int64_t(t.row0 + r) * p.ldo + col, p.n - col, p.out_type, p.out_align);
                        }
                    }
                }
            } else if constexpr (kAnyRows) {
                // Rows on no 16 bytes: 64 bytes of 32 rows at a time through the warp's slot, from where neighbouring lanes store neighbouring
                // words.  8 loads before their stores: 8192 x 8190 x 2048 220 -> 187 us, 2631 x 2505 x 1872 29.2 -> 24.4 (with TMA stores,
                // 2631 x 2504 x 1872 takes 22.3).  (Each thread its row's values one by one: twice the time of 5776 x 4740 x 5024, 167.)
                if (busy) {
                    const uint32_t slot = epi_base + warp * (C::kEpiSlots * 2048);
                    const bool f32 = p.out_type == HQ_DTYPE_FP32;
                    const int rows = min(32, t.valid - quarter * 32);
                    const int64_t row0 = t.row0 + quarter * 32;
                    // lanes of `bytes` each have one row's 64
                    const int bytes = f32 || p.out_align >= 4 ? 4 : 2, lanes = 64 / bytes, size = f32 ? 4 : 2, per = 32 / lanes;
                    const int at = lane % lanes * bytes, first = at / size, mine = lane / lanes;
                    const auto store_rows = [&](int col) {
                        __syncwarp();
                        const int left = p.n - col - first;
                        char* to = static_cast<char*>(p.out) + ((row0 + mine) * p.ldo + col + first) * size;
                        const int64_t next = int64_t(per) * p.ldo * size;
                        for (int r0 = mine; r0 < rows; r0 += 8 * per) {
                            uint32_t w[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const int r = r0 + i * per;  // (below 32)
                                const uint32_t from = slot + r * 64 + (((at >> 4) ^ ((r >> 1) & 3)) << 4) + (at & 12);
                                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[i]) : "r"(from) : "memory");
                                if (at & 2) w[i] >>= 16;
                            }
#pragma unroll
                            for (int i = 0; i < 8; ++i, to += next) {
                                if (r0 + i * per >= rows || left <= 0) continue;
                                if (bytes == 4 && (f32 || left > 1)) {
                                    *reinterpret_cast<uint32_t*>(to) = w[i];
                                } else {
                                    *reinterpret_cast<uint16_t*>(to) = uint16_t(w[i]);
                                }
                            }
                        }
                        __syncwarp();
                    };
#pragma unroll
                    for (int c = 0; c < C::kCols; c += 32) {
                        const int col = t.n0 + part * C::kCols + c;
                        if (col >= p.n) break;
                        if (f32) {
#pragma unroll
                            for (int h = 0; h < 32; h += 16) {
                                if (col + h >= p.n) break;
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    const float* const f = acc + c + h + j * 4;
                                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(slot + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)),
                                                 "r"(__float_as_uint(f[0])), "r"(__float_as_uint(f[1])), "r"(__float_as_uint(f[2])),
                                                 "r"(__float_as_uint(f[3])) : "memory");
                                }
                                store_rows(col + h);
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const float* const f = acc + c + j * 8;
                                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(slot + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)),
                                             "r"(pack16(f[0], f[1], p.out_type)), "r"(pack16(f[2], f[3], p.out_type)),
                                             "r"(pack16(f[4], f[5], p.out_type)), "r"(pack16(f[6], f[7], p.out_type)) : "memory");
                            }
                            store_rows(col);
                        }
                    }
                }
            } else if (p.staged != 0 && (kGrouped ? quarter * 32 + 32 <= t.valid : busy)) {
                // 32 x 32 values at a time (rows and columns that are not there are dropped by the store; a run's last rows go the other way).
                // 16-byte piece j of row r is at piece j ^ (r >> 1 & 3), the 64-byte swizzle of the tensor map.
                const uint32_t slots = epi_base + warp * (C::kEpiSlots * 2048);
#pragma unroll
                for (int c = 0; c < C::kCols; c += 32) {
                    const int col = t.n0 + part * C::kCols + c;
                    if (col >= p.n) {
                        // A group without a store: every tile commits one for each of its pieces, so that a slot's last store is always
                        // kEpiSlots groups back, also on the tile behind one that sticks out beyond N.
                        if (lane == 0) ptx::bulk_commit();
                        continue;
                    }
                    const uint32_t slot = slots + c / 32 % C::kEpiSlots * 2048;
                    // the store that last read this slot (of this tile, or the one before) is done with it
                    if (lane == 0) ptx::bulk_wait_read<C::kEpiSlots - 1>();
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t w[4];
#pragma unroll
                        for (int l = 0; l < 4; ++l) w[l] = pack16(acc[c + j * 8 + 2 * l], acc[c + j * 8 + 2 * l + 1], p.out_type);
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(slot + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)), "r"(w[0]),
                                     "r"(w[1]), "r"(w[2]), "r"(w[3])
                                     : "memory");
                    }
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        ptx::tma_store_2d(&tm_d, slot, col, t.row0 + quarter * 32);
                        ptx::bulk_commit();
                    }
                }
            } else if (row_ok) {
                const int col = t.n0 + part * C::kCols;
                const int64_t at = int64_t(t.row0 + row) * p.ldo + col;
#pragma unroll
                for (int c = 0; c < C::kCols / 16; ++c) {
                    if (col + c * 16 >= p.n) break;
                    float f[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) f[j] = acc[c * 16 + j];
                    store_values<16>(f, p.out, at + c * 16, p.n - col - c * 16, p.out_type, p.out_align);
                }
            }
        }
    }

    if (!kSplit && !kRowScales && warp < C::kPromoWarps && lane == 0) ptx::bulk_wait<0>();
    __syncwarp();

    if constexpr (kSplit) {
        // One tile per cluster: every CTA adds up its share of the tile over the CTAs, in their order.
        __syncwarp();
        ptx::cluster_sync();
        if (warp < C::kPromoWarps) {
            BlockWalk<BN, kGrouped> walk(p, tables, first, step);
            BlockTile t;
            if (walk.next(t)) {
                constexpr int kVecs = BN / 4;
                const int total = t.valid * kVecs;
                const int end = int(int64_t(total) * (rank + 1) / p.split);
                for (int i = int(int64_t(total) * rank / p.split) + threadIdx.x; i < end; i += C::kPromoWarps * 32) {
                    const int r = i / kVecs, c = (i - r * kVecs) * 4;
                    const uint32_t addr = a_base + (r * (BN + 4) + c) * 4;
                    float f[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    for (int s = 0; s < p.split; ++s) {
                        float v[4];
                        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                     : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3])
                                     : "r"(ptx::mapa_cluster(addr, s))
                                     : "memory");
#pragma unroll
                        for (int j = 0; j < 4; ++j) f[j] += v[j];
                    }
                    if (t.n0 + c < p.n) {
                        store_values<4>(f, p.out, int64_t(t.row0 + r) * p.ldo + t.n0 + c, p.n - t.n0 - c, p.out_type, p.out_align);
                    }
                }
            }
        }
        __syncwarp();
    }
    if (*abort != 0u) {
        // bounded grace period for copies and MMAs in flight before the memory they target is released
        for (int i = 0; i < 64; ++i) __nanosleep(1000);
    }
    ptx::tc_fence_before();
    __syncthreads();
    // no CTA leaves while another reads its sums
    if constexpr (kSplit) ptx::cluster_sync();
    if (warp == C::kMmaWarp) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc<1>(tmem, C::kTmemCols);
    }
}

// ---------------------------------------------------------------------------- host

struct BlockProblem {
    const void* a;
    const void* b;
    int64_t rows_a, n, k, experts;
    bool row_scales, grouped;
    BlockArgs args;
    int sms;
    cudaStream_t stream;
};

template <int BN, bool kRowScales, bool kGrouped, bool kSplit, bool kAnyRows = false>
int launch_block_gemm(const BlockProblem& g, char* err, size_t errlen) {
    using C = BlockCfg<BN, kRowScales>;
    static SmemOptIn opt_in;
    const auto kernel = block_gemm_kernel<BN, kRowScales, kGrouped, kSplit, kAnyRows>;
    HQ_CUDA_TRY(opt_in.ensure(kernel, C::kSmemBytes));
    BlockArgs p = g.args;
    p.tiles_m = int((g.rows_a + kTileM - 1) / kTileM);
    p.tiles_n = int((g.n + BN - 1) / BN);
    CUtensorMap tm_a, tm_b, tm_d;
    if (!make_tmap_2d(&tm_a, CU_TENSOR_MAP_DATA_TYPE_UINT8, g.a, uint64_t(g.k), uint64_t(g.rows_a), uint64_t(g.k), kBlockK,
                      uint32_t(p.box_rows), CU_TENSOR_MAP_SWIZZLE_128B) ||
        !make_tmap_2d(&tm_b, CU_TENSOR_MAP_DATA_TYPE_UINT8, g.b, uint64_t(g.k), uint64_t(g.n * g.experts), uint64_t(g.k), kBlockK, BN,
                      CU_TENSOR_MAP_SWIZZLE_128B)) {
        return fail(err, errlen, HQ_ERR_CUDA, "cuTensorMapEncodeTiled failed for the GEMM operands");
    }
    // 16-bit results in whole pieces of 16 bytes leave through TMA (it stores a piece that the tensor ends in as a whole); others from
    // registers, and another map stands in
    p.staged = !kSplit && !kRowScales && p.out_type != HQ_DTYPE_FP32 && p.out_align >= 16 && g.n % 8 == 0 &&
               make_tmap_2d(&tm_d, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p.out, uint64_t(g.n), uint64_t(g.rows_a), uint64_t(p.ldo) * 2, 32, 32,
                            CU_TENSOR_MAP_SWIZZLE_64B);
    if (p.staged == 0) tm_d = tm_a;
    // grouped: a run may add a tile to those that its rows fill
    const int64_t row_tiles = kGrouped ? std::min<int64_t>(g.rows_a, g.rows_a / kTileM + g.experts) : p.tiles_m;
    const int64_t tiles = row_tiles * p.tiles_n;
    if (!kSplit) p.split = 1;
    const int64_t grid = kSplit ? tiles * p.split : std::min<int64_t>(tiles, g.sms);
    HQ_CUDA_TRY(launch(kernel, dim3(unsigned(grid)), dim3(C::kThreads), size_t(C::kSmemBytes), g.stream, p.pdl != 0,
                       kSplit ? unsigned(p.split) : 1u, tm_a, tm_b, tm_d, p));
    return HQ_OK;
}

// The tile, and the CTAs that share one.
struct BlockChoice {
    int bn, split;
};

// The least time by figures of the four tiles, GEMM alone.  A k-tile takes `alone` microseconds with few CTAs running and `full` with all
// (then the CTAs share L2 and power); `tile` is what a tile's end costs, and a launch is 3.  Measured for 64, 128, 192, 256 columns:
//   8 tiles, K from 4096 to 16384                0.139  0.187  0.311  0.396 a k-tile
//   8192 x 8192 x 8192 in a burst                0.179  0.270  0.400  0.511 a k-tile; 640, 484, 486, 458 us
//   the same at the power cap                    -      0.336  0.492  0.638 a k-tile; -, 602, 598, 572 us
//   9472 rows by 2 and by 20 widths, K = 256     0.47   0.71   0.79   1.32 a tile beside its k-tiles
// The table stands between the burst and the cap.  Of 20 shapes from 16 x 4096 x 7168 to 8192 x 8192 x 8192, each on all four widths, the chosen one
// was the fastest on 18 and within 3.5 % on the others (4736 x 768 x 4096: 22.3, 21.2, 17.4, 21.0 us; 2048 x 1024 x 2048: 9.2, 7.4, 9.8, 11.1;
// 1000 x 4104 x 4112: 48.4, 34.7, 42.0, 27.4).  Scales per row on both sides have dearer k-tiles than the table's: 128 columns are chosen and
// right for 7168 x 2048 x 4096 (109 us, 124 on 64), but 64 are faster where K is short (1024 x 2048 x 256 5.6 us, 7.1 chosen).
// With a CTA's share of K in `split` CTAs of a cluster: 2.2 more for its barriers and the exchange (16 x 4096 x 7168 on 128 columns 13.1 us whole,
// 9.8 in two, 8.4 in four; 8 x 1024 x 4096 8.5 whole, 5.5 in eight; 1 x 7168 x 2048 5.9 whole, 6.4 in two).
BlockChoice choose(const BlockProblem& g) {
    struct Cost {
        int bn;
        double alone, full, tile;
    };
    constexpr Cost kCosts[] = {{128, 0.20, 0.30, 1.0}, {64, 0.157, 0.21, 0.7}, {192, 0.30, 0.42, 1.2}, {256, 0.42, 0.53, 1.6}};  // (in order of preference where the floor decides)
    const int k_tiles = g.args.k_tiles;
    const int64_t runs = std::min(g.experts, g.rows_a);  // with rows
    const int64_t mean = (g.rows_a + runs - 1) / runs;
    const int64_t row_tiles = runs * ((mean + kTileM - 1) / kTileM);  // (of runs of the same length)
    // the operands and the result pass HBM once at best
    const double floor_us = (double(g.rows_a) * g.k + double(runs) * g.n * g.k + 2.0 * g.rows_a * g.n) / 6.0e6 + 4.0;
    BlockChoice best = {128, 1};
    double least = 1e30;
    for (const Cost& c : kCosts) {
        if (g.row_scales && c.bn > 128) continue;
        const int64_t tiles = row_tiles * ((g.n + c.bn - 1) / c.bn);
        for (int split = 1; split <= 8; split *= 2) {
            // (clusters of 8 do not fill every group of SMs)
            if (split > 1 && (g.grouped || g.row_scales || c.bn > 128 || tiles * split > (split == 8 ? g.sms * 6 / 7 : g.sms) || k_tiles < 4 * split)) break;
            const int64_t ctas = tiles * split, waves = (ctas + g.sms - 1) / g.sms;
            const double busy = double(std::min<int64_t>(ctas, g.sms)) / g.sms;
            const double step = c.alone + (c.full - c.alone) * busy;
            const double t = std::max(floor_us, 3.0 + (split > 1 ? 2.2 : 0.0) + double(waves) * (step * ((k_tiles + split - 1) / split) + c.tile));
            if (t < least) least = t, best = {c.bn, split};
        }
    }
    return best;
}

template <int BN, bool kRowScales>
int launch_kind(const BlockProblem& g, char* err, size_t errlen) {
    if constexpr (kRowScales) {
        return launch_block_gemm<BN, true, false, false>(g, err, errlen);
    } else {
        const bool any = g.args.out_align < 16;
        if (g.grouped) return any ? launch_block_gemm<BN, false, true, false, true>(g, err, errlen) : launch_block_gemm<BN, false, true, false>(g, err, errlen);
        if constexpr (BN <= 128) {
            if (g.args.split > 1) return launch_block_gemm<BN, false, false, true>(g, err, errlen);
        }
        return any ? launch_block_gemm<BN, false, false, false, true>(g, err, errlen) : launch_block_gemm<BN, false, false, false>(g, err, errlen);
    }
}

int block_gemm(const void* a, const void* b, const float* sfa, const float* sfb, const int32_t* offsets, void* out, int out_type, int64_t m,
               int64_t n, int64_t k, int64_t experts, int row_scales, bool grouped, int64_t ldo, int sm_count, int use_pdl, int device,
               void* stream, char* err, size_t errlen) {
    if (out_type != HQ_DTYPE_BF16 && out_type != HQ_DTYPE_FP16 && out_type != HQ_DTYPE_FP32) {
        return fail(err, errlen, HQ_ERR_INVALID, "output dtype must be bfloat16, float16 or float32");
    }
    if (m < 0 || n < 0 || experts < 0 || m > INT32_MAX - 128 || n > INT32_MAX - 256) {
        return fail(err, errlen, HQ_ERR_INVALID, "at most 2^31 - 256 rows and columns, got M=%lld, N=%lld", static_cast<long long>(m),
                    static_cast<long long>(n));
    }
    if (k < 16 || k % 16 != 0 || k > (int64_t(1) << 30)) {
        return fail(err, errlen, HQ_ERR_INVALID, "K must be a positive multiple of 16, got K=%lld", static_cast<long long>(k));
    }
    if (experts > kMaxExperts || experts * n > INT32_MAX - 256) {
        return fail(err, errlen, HQ_ERR_INVALID, "at most %d experts and 2^31 - 256 weight rows, got %lld of %lld", kMaxExperts,
                    static_cast<long long>(experts), static_cast<long long>(n));
    }
    if (((m + 127) / 128 + experts) * ((n + 63) / 64) > INT32_MAX / 8) {
        return fail(err, errlen, HQ_ERR_INVALID, "the output has too many tiles, got M=%lld, N=%lld", static_cast<long long>(m),
                    static_cast<long long>(n));
    }
    if (m == 0 || n == 0 || experts == 0) return HQ_OK;
    if (a == nullptr || b == nullptr || sfa == nullptr || sfb == nullptr || out == nullptr || (grouped && offsets == nullptr)) {
        return fail(err, errlen, HQ_ERR_INVALID, "null pointer argument");
    }
    if (!aligned(a, 16) || !aligned(b, 16)) return fail(err, errlen, HQ_ERR_INVALID, "input and weight must be 16-byte aligned");
    const int size = out_type == HQ_DTYPE_FP32 ? 4 : 2;
    if (ldo < n || !aligned(sfa, 4) || !aligned(sfb, 4) || !aligned(out, size_t(size))) {
        return fail(err, errlen, HQ_ERR_INVALID, "output rows must hold N values, got a row stride of %lld", static_cast<long long>(ldo));
    }
    const DeviceGuard guard(device);
    if (!guard.ok()) return fail(err, errlen, HQ_ERR_CUDA, "cannot select CUDA device %d", device);
    const int sms = hq_sm_count(device);
    if (sms <= 0) return fail(err, errlen, HQ_ERR_CUDA, "cannot read the SM count of CUDA device %d", device);
    BlockProblem g = {};
    g.a = a, g.b = b, g.rows_a = m, g.n = n, g.k = k, g.experts = experts, g.row_scales = row_scales != 0, g.grouped = grouped;
    g.sms = sm_count > 0 ? std::min(sm_count, sms) : sms;
    g.stream = static_cast<cudaStream_t>(stream);
    BlockArgs& p = g.args;
    p.sfa = sfa, p.sfb = sfb, p.out = out, p.offsets = offsets, p.ldo = ldo;
    p.m = int(m), p.n = int(n), p.k_tiles = int((k + kBlockK - 1) / kBlockK);
    p.n_blocks = int((n + 127) / 128), p.experts = int(experts), p.out_type = out_type, p.pdl = use_pdl != 0;
    p.wide_scales = aligned(sfa, 16) && aligned(sfb, 16);
    const int64_t row_bytes = ldo * size;
    const auto starts = [&](int a) { return aligned(out, size_t(a)) && row_bytes % a == 0; };
    p.out_align = starts(32) ? 32 : starts(16) ? 16 : starts(4) ? 4 : 2;
    // Rows of `a` per copy: all of a tile's, or about those of a run, so that short runs do not read their neighbours' rows.
    const int64_t mean = grouped ? (m + std::min(experts, m) - 1) / std::min(experts, m) : m;
    p.box_rows = 8;
    while (p.box_rows < kTileM && p.box_rows < mean) p.box_rows *= 2;
    const BlockChoice c = choose(g);
    p.split = c.split;
    if (g.row_scales) return c.bn == 128 ? launch_kind<128, true>(g, err, errlen) : launch_kind<64, true>(g, err, errlen);
    return c.bn == 256   ? launch_kind<256, false>(g, err, errlen)
           : c.bn == 192 ? launch_kind<192, false>(g, err, errlen)
           : c.bn == 128 ? launch_kind<128, false>(g, err, errlen)
                         : launch_kind<64, false>(g, err, errlen);
}

}  // namespace

// Reads and clears this file's status word; the stream has been synchronised.
cudaError_t take_block_gemm_status(uint32_t* status) {
    uint32_t host[4] = {0, 0, 0, 0};
    cudaError_t e = cudaMemcpyFromSymbol(host, g_status, sizeof(host));
    if (e == cudaSuccess && host[0] != 0) {
        const uint32_t zero[4] = {0, 0, 0, 0};
        e = cudaMemcpyToSymbol(g_status, zero, sizeof(zero));
    }
    *status = host[0];
    return e;
}

}  // namespace hq

extern "C" int hq_describe_block_tile(int64_t m, int64_t n, int64_t k, int64_t num_experts, int row_scales, int sm_count, int device, char* buf,
                                      size_t buflen) {
    if (m < 1 || n < 1 || k < 16 || k % 16 != 0 || num_experts < 0 || num_experts > hq::kMaxExperts || m > INT32_MAX - 128 ||
        n > INT32_MAX - 256 || k > (int64_t(1) << 30) || (num_experts > 0 && row_scales != 0)) {
        return hq::fail(buf, buflen, HQ_ERR_INVALID, "No block-128 tile for M=%lld, N=%lld, K=%lld, %lld experts", static_cast<long long>(m),
                        static_cast<long long>(n), static_cast<long long>(k), static_cast<long long>(num_experts));
    }
    const int sms = sm_count > 0 ? sm_count : hq_sm_count(device);
    hq::BlockProblem g = {};
    g.rows_a = m, g.n = n, g.k = k, g.experts = std::max<int64_t>(num_experts, 1), g.grouped = num_experts > 0, g.row_scales = row_scales != 0;
    g.sms = sms > 0 ? sms : 148;
    g.args.k_tiles = int((k + hq::kBlockK - 1) / hq::kBlockK);
    const hq::BlockChoice c = hq::choose(g);
    if (buf != nullptr && buflen > 0) {
        snprintf(buf, buflen, "[gemm] mode=%s kind=block128%s m=%lld n=%lld k=%lld sm=%d -> %dx%d/%d split=%d", g.grouped ? "experts" : "dense",
                 g.row_scales ? "-rows" : "", static_cast<long long>(m), static_cast<long long>(n), static_cast<long long>(k), g.sms, hq::kTileM,
                 c.bn, hq::kBlockK, c.split);
    }
    return HQ_OK;
}

extern "C" int hq_block_gemm(const void* a, const void* b, const float* sfa, const float* sfb, void* out, int out_dtype, int64_t m, int64_t n,
                             int64_t k, int row_scales, int64_t ldo, int sm_count, int use_pdl, int device, void* stream, char* err,
                             size_t errlen) {
    return hq::block_gemm(a, b, sfa, sfb, nullptr, out, out_dtype, m, n, k, 1, row_scales, false, ldo, sm_count, use_pdl, device, stream, err,
                          errlen);
}

extern "C" int hq_group_block_gemm(const void* a, const void* b, const float* sfa, const float* sfb, const int32_t* offsets, void* out,
                                   int out_dtype, int64_t num_experts, int64_t m, int64_t n, int64_t k, int64_t ldo, int sm_count, int use_pdl,
                                   int device, void* stream, char* err, size_t errlen) {
    return hq::block_gemm(a, b, sfa, sfb, offsets, out, out_dtype, m, n, k, num_experts, 0, true, ldo, sm_count, use_pdl, device, stream, err,
                          errlen);
}
