// What the GEMM kernels share: the device status word, bounded barrier waits, tensor maps and the opt-in to large
// shared memory.  Everything here is per source file: each has a status word of its own, and hq_device_status reads them all.
#pragma once

#include <mutex>

#include "common.cuh"
#include "ptx.cuh"

namespace hq {
namespace {

constexpr uint64_t kTimeoutNs = 2000000000ull;    // bound of every device-side wait

// device status word: non-zero when a kernel gave up on a bounded wait
__device__ uint32_t g_status[4];

enum : uint32_t {
    kStatusProducer = 0x01,
    kStatusMma = 0x02,
    kStatusEpilogue = 0x04,
};
// Bounded mbarrier wait of one lane.  Returns false when the CTA is aborting.  kCluster: the barrier is one
// that CTAs of the cluster arrive on with release semantics; the wait acquires what they wrote into
// this CTA's shared memory before arriving.  A function of its own: the roles come here only when a first
// try_wait, which holds a converged warp until the phase ends (woken 84 cycles after the arrival, also after
// 6000 cycles), has returned without it, and the polling code is not in their loops.  (InPlace: inline after all, for the split-K
// kernel, which took 170 cycles a k-tile longer with the calls in its loops: 125 x 704 x 8064 10.8 us, 13.7 with them.  Inline in every
// kernel: SituQuant 300 x 5120 x 2048 7.5 -> 8.6 us, NVFP4 2048 x 8192 x 2048 20.7 -> 26.0, W4A8 12 slots of 256 x 3072 x 2048
// 18.7 -> 25.5.)
enum class InPlace {};
template <bool kCluster = false>
__device__ __forceinline__ bool wait_bar_lane(InPlace, uint32_t bar, uint32_t parity, volatile uint32_t* abort, uint32_t code,
                                              uint64_t limit_ns = kTimeoutNs) {
    const auto done = [&] { return kCluster ? ptx::mbar_try_wait_cluster(bar, parity) : ptx::mbar_try_wait(bar, parity); };
    if (done()) return true;
    const uint64_t t0 = ptx::globaltimer_ns();
    uint32_t spins = 0;
    while (!done()) {
        if ((++spins & 31u) == 0u) {
            if (*abort != 0u) return false;
            if (ptx::globaltimer_ns() - t0 > limit_ns) {
                *abort = 1u;
                atomicOr(&g_status[0], code);
                return false;
            }
        }
    }
    return true;
}
template <bool kCluster = false>
__device__ __noinline__ bool wait_bar_lane(uint32_t bar, uint32_t parity, volatile uint32_t* abort, uint32_t code,
                                           uint64_t limit_ns = kTimeoutNs) {
    return wait_bar_lane<kCluster>(InPlace{}, bar, parity, abort, code, limit_ns);
}

// The wait of a role: called by all lanes of a warp, with one result for all of them.  Lanes poll for
// themselves, so when a wait runs out while its barrier completes after all, some of them see the one and
// some the other; leaving the role's loop on that would send a part of the warp into
// .sync.aligned instructions, __syncwarp and elections that count on all 32 lanes.
// The first try and its vote are straight-line code (a completed barrier: 58 cycles); with the polling loop inline, lane by
// lane, a wait on a completed barrier took a role 125: 512 x 1536 x 4096 8.8 -> 8.5 us, 1024 x 1536 x 8192 26.0 -> 24.9 (both on
// the 128 x 64 tile), NVFP4 512 x 4096 x 8192 12.9 -> 12.7, GEMM alone.
template <bool kInPlace = false>
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, volatile uint32_t* abort, uint32_t code) {
    if (__all_sync(0xffffffffu, ptx::mbar_try_wait(bar, parity) ? 1 : 0) != 0) return true;
    const bool mine = kInPlace ? wait_bar_lane(InPlace{}, bar, parity, abort, code) : wait_bar_lane(bar, parity, abort, code);
    return __all_sync(0xffffffffu, mine ? 1 : 0) != 0;
}
// Two waits with one vote (the second only if `both`): a vote between a barrier and the work behind it is on the
// critical path of a k-step.
template <bool kInPlace = false>
__device__ __forceinline__ bool wait_bars(uint32_t bar, uint32_t parity, bool both, uint32_t bar2, uint32_t parity2,
                                          volatile uint32_t* abort, uint32_t code) {
    bool mine = ptx::mbar_try_wait(bar, parity);
    if (both) mine = ptx::mbar_try_wait(bar2, parity2) && mine;
    if (__all_sync(0xffffffffu, mine ? 1 : 0) != 0) return true;
    if constexpr (kInPlace) {
        mine = wait_bar_lane(InPlace{}, bar, parity, abort, code) && (!both || wait_bar_lane(InPlace{}, bar2, parity2, abort, code));
    } else {
        mine = wait_bar_lane(bar, parity, abort, code) && (!both || wait_bar_lane(bar2, parity2, abort, code));
    }
    return __all_sync(0xffffffffu, mine ? 1 : 0) != 0;
}
template <bool kInPlace = false>
__device__ __forceinline__ bool wait_bar_cluster(uint32_t bar, uint32_t parity, volatile uint32_t* abort, uint32_t code) {
    if (__all_sync(0xffffffffu, ptx::mbar_try_wait_cluster(bar, parity) ? 1 : 0) != 0) return true;
    const bool mine = kInPlace ? wait_bar_lane<true>(InPlace{}, bar, parity, abort, code) : wait_bar_lane<true>(bar, parity, abort, code);
    return __all_sync(0xffffffffu, mine ? 1 : 0) != 0;
}

// The warp's index in its CTA, known to be warp-uniform.
__device__ __forceinline__ int warp_index() { return __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0); }

// ---------------------------------------------------------------------------- host

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled_fn() {
    static EncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess) {
            p = nullptr;
        }
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    return fn;
}

// rank-2 row-major tensor map: `inner` elements per row, `rows` rows, `pitch` bytes between rows
bool make_tmap_2d(CUtensorMap* map, CUtensorMapDataType dtype, const void* base, uint64_t inner,
                  uint64_t rows, uint64_t pitch, uint32_t box_inner, uint32_t box_rows,
                  CUtensorMapSwizzle swizzle) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (fn == nullptr) return false;
    const cuuint64_t dims[2] = {inner, rows};
    const cuuint64_t strides[1] = {pitch};
    const cuuint32_t box[2] = {box_inner, box_rows};
    const cuuint32_t estr[2] = {1, 1};
    return fn(map, dtype, 2, const_cast<void*>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Per-device, once: the opt-in to more than 48 KB of dynamic shared memory for one kernel.
// A failed attempt is not remembered, so the next call tries (and reports) again.
struct SmemOptIn {
    std::mutex mu;
    bool done[64] = {};
    template <typename Kernel>
    cudaError_t ensure(Kernel kernel, int bytes, int* dev_out = nullptr) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        if (dev_out != nullptr) *dev_out = dev;
        std::lock_guard<std::mutex> lock(mu);
        if (dev >= 0 && dev < 64 && done[dev]) return cudaSuccess;
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess && dev >= 0 && dev < 64) done[dev] = true;
        return e;
    }
};
}  // namespace
}  // namespace hq
