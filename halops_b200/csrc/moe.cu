// Tokens in the order of the experts that a router gave them, and back.
//
// A pair p = token * topk + slot has an expert ids[p]; one outside of [0, experts) is dropped (it belongs to another device).
// The pairs of an expert keep their order and become a run of rows that starts on a multiple of `align`:
//   offsets[e]     first row of expert e's run; offsets[experts] is the end of the last
//   rows[p]        the pair's row, -1 for a dropped one
//   pairs[r]       the row's pair, -1 for a row that pads a run or lies behind the last
//   expert_ids[r]  the run that row r is in, experts - 1 behind the last run
//
// The sort is one launch; what moves tokens is bound by HBM: every token is read once and written once per expert,
// or the other way round.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "common.cuh"

namespace hq {
namespace {

// No kernel pointer here is __restrict__ or read through __ldg: what it points to changes, in the preceding kernel, while this one
// waits for it, and a load of constant data may be moved to before the wait.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// ---------------------------------------------------------------------------- sort
//
// A stable counting sort by one cluster of 1, 8 or 16 CTAs.  Every warp has a stretch of the pairs: it counts their experts into a
// line of its own in shared memory, the lines are summed over the warps of the CTA and, through distributed shared memory, over the
// CTAs before this one, and then the warp goes over its stretch again, 32 pairs at a time: a pair's row is its expert's
// start plus the pairs of that expert before it, counted in the warp's line and, among the 32, by a match of the lanes.  All
// counts are whole numbers, so the order in which warps run changes nothing.

constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxExperts = 1024;
constexpr int64_t kMaxSortPairs = (int64_t(1) << 31) - 8192;  // the kernel's steps past the last pair, and a run's padding, stay below 2^31

template <typename Id>
__device__ __forceinline__ int expert_of(const Id* ids, int p, int pairs_n, int experts) {
    if (p >= pairs_n) return -1;
    const Id id = ids[p];
    return id >= 0 && id < Id(experts) ? int(id) : -1;
}

template <typename Id>
__global__ void __launch_bounds__(kSortThreads) moe_sort_kernel(const Id* ids, int pairs_n, int experts, int align, int n_rows,
                                                                int ctas, int* rows, int* pairs,
                                                                int* offsets, int* expert_ids) {
    extern __shared__ int smem[];
    int* const lines = smem;                             // [warp][expert]
    int* const total = lines + kSortWarps * experts;     // this CTA's pairs per expert, read by the cluster
    int* const count = total + experts;                  // all pairs per expert
    int* const base = count + experts;                   // row of this CTA's first pair of the expert
    int* const start = base + experts;                   // first row of the expert's run, and the end of the last
    __shared__ int warp_sums[kSortWarps];
    grid_wait();
    grid_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cta = blockIdx.x;
    // warps with pairs: few pairs make few lines to zero and to sum over
    const int used = min(kSortWarps, max(1, (pairs_n + 32 * ctas - 1) / (32 * ctas)));
    for (int i = tid; i < used * experts; i += kSortThreads) lines[i] = 0;
    __syncthreads();

    const int stretch = (pairs_n + ctas * used - 1) / (ctas * used);
    const int64_t first = warp < used ? int64_t(cta * used + warp) * stretch : pairs_n;
    const int begin = int(min(first, int64_t(pairs_n))), end = int(min(first + stretch, int64_t(pairs_n)));
    int* const line = lines + warp * experts;
    // the first pairs' experts stay in registers for the second pass, and are all asked for before the first is counted
    constexpr int kHeld = 8;
    int held[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) held[i] = expert_of(ids, begin + i * 32 + lane, end, experts);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        if (held[i] >= 0) atomicAdd(line + held[i], 1);
    }
    for (int p = begin + kHeld * 32 + lane; p < end; p += 32) {
        const int e = expert_of(ids, p, end, experts);
        if (e >= 0) atomicAdd(line + e, 1);
    }
    __syncthreads();
    // a thread per expert (experts <= threads): exclusive sums over the lines, eight of which are read at a time
    if (tid < experts) {
        int sum = 0;
        for (int w0 = 0; w0 < used; w0 += 8) {
            int c[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) c[j] = w0 + j < used ? lines[(w0 + j) * experts + tid] : 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (w0 + j < used) lines[(w0 + j) * experts + tid] = sum;
                sum += c[j];
            }
        }
        total[tid] = sum;
    }
    int all = 0, before = 0;
    if (ctas > 1) {
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (tid < experts) {
            const uint32_t addr = static_cast<uint32_t>(__cvta_generic_to_shared(total + tid));
            for (int c = 0; c < ctas; ++c) {
                uint32_t remote, v;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(c));
                asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(remote) : "memory");
                if (c < cta) before += int(v);
                all += int(v);
            }
        }
        // no CTA leaves while another reads its counts: the other half of this barrier is at the end
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    } else if (tid < experts) {
        all = total[tid];
    }
    // exclusive sums of the padded counts over the experts
    const int padded = tid < experts ? (all + align - 1) / align * align : 0;
    int sum = padded;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int v = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += v;
    }
    if (lane == 31) warp_sums[warp] = sum;
    __syncthreads();
    if (warp == 0) {
        int v = warp_sums[lane];
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int u = __shfl_up_sync(0xffffffffu, v, d);
            if (lane >= d) v += u;
        }
        warp_sums[lane] = v;
    }
    __syncthreads();
    const int run = sum - padded + (warp > 0 ? warp_sums[warp - 1] : 0);
    if (tid < experts) {
        count[tid] = all;
        start[tid] = run;
        if (tid == experts - 1) start[experts] = run + padded;
        base[tid] = run + before;
        if (cta == 0) {
            offsets[tid] = run;
            if (tid == experts - 1) offsets[experts] = run + padded;
        }
    }
    __syncthreads();

    const auto place = [&](int p0, int e) {
        const int p = p0 + lane;
        const uint32_t same = __match_any_sync(0xffffffffu, e);
        int at = -1;
        int seen = 0;
        if (e >= 0) seen = line[e], at = base[e] + seen + __popc(same & ((1u << lane) - 1u));
        __syncwarp();
        if (e >= 0 && lane == 31 - __clz(same)) line[e] = seen + __popc(same);
        __syncwarp();
        if (p < end) rows[p] = at;
        if (at >= 0 && at < n_rows) pairs[at] = p;
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        if (begin + i * 32 < end) place(begin + i * 32, held[i]);
    }
    for (int p0 = begin + kHeld * 32; p0 < end; p0 += 32) place(p0, expert_of(ids, p0 + lane, end, experts));
    // The rows' experts (the last whose run starts at or before a row: empty runs start where the next does), and the rows without a
    // pair: where there are more rows than threads, four neighbouring ones a thread, of which only the first is searched for.
    int top = 1;
    while (top * 2 < experts) top *= 2;
    const int per = n_rows > ctas * kSortThreads ? 4 : 1;
    for (int64_t r0 = per * int64_t(cta * kSortThreads + tid); r0 < n_rows; r0 += per * ctas * kSortThreads) {
        int e = 0;
        for (int d = top; d > 0; d /= 2) {
            if (e + d < experts && start[e + d] <= r0) e += d;
        }
        for (int i = 0; i < per && r0 + i < n_rows; ++i) {
            const int r = int(r0) + i;
            while (e + 1 < experts && start[e + 1] <= r) ++e;
            expert_ids[r] = e;
            if (r - start[e] >= count[e]) pairs[r] = -1;
        }
    }
    __syncwarp();
    if (ctas > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The rows that pad expert e's run: [*first, *end), behind the rows with pairs.  kPadCtas CTAs share them (one wrote 64 rows of 16 KB in 20 us).
constexpr int kPadCtas = 16;
__device__ __forceinline__ void padding_of(const int* pairs, const int* offsets, int n_rows, int e, int* first, int* end) {
    int lo = max(offsets[e], 0);
    const int hi = min(offsets[e + 1], n_rows);
    *end = hi;
    for (int n = hi - lo; n > 0;) {  // the first row without a pair
        const int half = n / 2;
        if (pairs[lo + half] >= 0) lo += half + 1, n -= half + 1; else n = half;
    }
    *first = lo;
}

// ---------------------------------------------------------------------------- tokens to rows
//
// A CTA reads a piece of one token and writes it to each of the token's rows; the CTAs behind the tokens zero the rows that
// pad the experts' runs.  Unit: the widest word that the rows' starts and length allow.

constexpr int kMoveThreads = 256;

template <typename Unit, int kPer>
__global__ void __launch_bounds__(kMoveThreads) moe_permute_kernel(const Unit* x, int64_t ld, int tokens, int units, int topk,
                                                                   const int* rows, const int* pairs,
                                                                   const int* offsets, int n_rows, Unit* out) {
    grid_wait();
    grid_launch_dependents();
    const int c = blockIdx.y * (kMoveThreads * kPer) + threadIdx.x;
    if (int(blockIdx.x) >= tokens) {
        const int pad = int(blockIdx.x) - tokens;
        int first, end;
        padding_of(pairs, offsets, n_rows, pad / kPadCtas, &first, &end);
        for (int r = first + pad % kPadCtas; r < end; r += kPadCtas) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                if (c + i * kMoveThreads < units) out[int64_t(r) * units + c + i * kMoveThreads] = Unit{};
            }
        }
        return;
    }
    const int64_t token = blockIdx.x;
    Unit v[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        if (c + i * kMoveThreads < units) v[i] = x[token * ld + c + i * kMoveThreads];
    }
    for (int j0 = 0; j0 < topk; j0 += 8) {
        int r[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = j0 + j < topk ? rows[token * topk + j0 + j] : -1;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (r[j] < 0 || r[j] >= n_rows) continue;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                if (c + i * kMoveThreads < units) out[int64_t(r[j]) * units + c + i * kMoveThreads] = v[i];
            }
        }
    }
}

// ---------------------------------------------------------------------------- rows to tokens
//
// y[t] = sum over the token's slots, in their order and in float32, of weight * z[row]; rounded once.

template <typename T>
struct Floats;  // a piece of kN values in one load
template <>
struct Floats<__nv_bfloat16> {
    static constexpr int kN = 8;
    using Vec = uint4;
    static __device__ __forceinline__ void get(const uint4& v, float (&f)[8]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ uint4 put(const float (&f)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            memcpy(&w[i], &h, 4);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <>
struct Floats<__half> {
    static constexpr int kN = 8;
    using Vec = uint4;
    static __device__ __forceinline__ void get(const uint4& v, float (&f)[8]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            __half2 h;
            memcpy(&h, &w[i], 4);
            const float2 p = __half22float2(h);
            f[2 * i] = p.x;
            f[2 * i + 1] = p.y;
        }
    }
    static __device__ __forceinline__ uint4 put(const float (&f)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
            memcpy(&w[i], &h, 4);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <>
struct Floats<float> {
    static constexpr int kN = 4;
    using Vec = float4;
    static __device__ __forceinline__ void get(const float4& v, float (&f)[4]) { f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w; }
    static __device__ __forceinline__ float4 put(const float (&f)[4]) { return make_float4(f[0], f[1], f[2], f[3]); }
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// A piece of a row in one load: 16 bytes where all rows start on 16, pairs of 16-bit values where they start on 4, else single values.
template <typename T, int kBytes>
struct Piece;
template <typename T>
struct Piece<T, 16> {
    static constexpr int kN = Floats<T>::kN;
    using Vec = typename Floats<T>::Vec;
    Vec v;
    __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const Vec*>(p); }
    // a row that is read once: not kept in L1 (moe_unpermute of 4096 tokens of 4096, 4 of 16: 33.5 -> 27.5 us)
    __device__ __forceinline__ void load_once(const T* p) {
        uint4 u;
        asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(p));
        memcpy(&v, &u, 16);
    }
    __device__ __forceinline__ void get(float (&f)[kN]) const { Floats<T>::get(v, f); }
    static __device__ __forceinline__ void store(T* p, const float (&f)[kN]) { *reinterpret_cast<Vec*>(p) = Floats<T>::put(f); }
};
template <typename T>
struct Piece<T, 4> {
    static constexpr int kN = 4 / int(sizeof(T));
    uint32_t v;
    __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint32_t*>(p); }
    __device__ __forceinline__ void load_once(const T* p) { load(p); }
    __device__ __forceinline__ void get(float (&f)[kN]) const {
        T one[kN];
        memcpy(one, &v, 4);
#pragma unroll
        for (int i = 0; i < kN; ++i) f[i] = to_float(one[i]);
    }
    static __device__ __forceinline__ void store(T* p, const float (&f)[kN]) {
        T one[kN];
#pragma unroll
        for (int i = 0; i < kN; ++i) one[i] = from_float<T>(f[i]);
        uint32_t w;
        memcpy(&w, one, 4);
        *reinterpret_cast<uint32_t*>(p) = w;
    }
};
template <typename T>
struct Piece<T, 2> {
    static constexpr int kN = 1;
    T one;
    __device__ __forceinline__ void load(const T* p) { one = p[0]; }
    __device__ __forceinline__ void load_once(const T* p) { load(p); }
    __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = to_float(one); }
    static __device__ __forceinline__ void store(T* p, const float (&f)[1]) { p[0] = from_float<T>(f[0]); }
};

template <typename T, int kBytes, int kPer>
__global__ void __launch_bounds__(kMoveThreads) moe_unpermute_kernel(const T* z, int64_t ld, int tokens, int h, int topk,
                                                                     const int* rows, int n_rows,
                                                                     const float* weights, T* y) {
    using P = Piece<T, kBytes>;
    constexpr int kSlots = 4;  // rows loaded before the first is added
    grid_wait();
    grid_launch_dependents();
    const int64_t token = blockIdx.x;
    constexpr int kStep = kMoveThreads * P::kN;
    const int c = blockIdx.y * (kStep * kPer) + threadIdx.x * P::kN;
    if (c >= h) return;
    float sum[kPer][P::kN];
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
#pragma unroll
        for (int i = 0; i < P::kN; ++i) sum[q][i] = 0.0f;
    }
    for (int j0 = 0; j0 < topk; j0 += kSlots) {
        P piece[kSlots][kPer];
        float w[kSlots];
        bool here[kSlots];
#pragma unroll
        for (int j = 0; j < kSlots; ++j) {
            int r = -1;
            if (j0 + j < topk) r = rows[token * topk + j0 + j];
            here[j] = r >= 0 && r < n_rows;
            w[j] = 1.0f;
            if (here[j]) {
#pragma unroll
                for (int q = 0; q < kPer; ++q) {
                    if (c + q * kStep < h) piece[j][q].load_once(z + int64_t(r) * ld + c + q * kStep);
                }
                if (weights != nullptr) w[j] = weights[token * topk + j0 + j];
            }
        }
#pragma unroll
        for (int j = 0; j < kSlots; ++j) {
            if (!here[j]) continue;
#pragma unroll
            for (int q = 0; q < kPer; ++q) {
                if (c + q * kStep >= h) continue;
                float f[P::kN];
                piece[j][q].get(f);
#pragma unroll
                for (int i = 0; i < P::kN; ++i) sum[q][i] = fmaf(w[j], f[i], sum[q][i]);
            }
        }
    }
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
        if (c + q * kStep < h) P::store(y + token * h + c + q * kStep, sum[q]);
    }
}

// The gradients of the above: gz[row] = weight * gy[token], gw[pair] = <gy[token], z[row]>.  A group of kGroup threads has one pair
// (a warp; a whole CTA where there are few pairs), with kAhead pieces of both rows in flight per thread; the pairs of a token are
// neighbours, so that its gradient comes from HBM once.  The CTAs behind the pairs zero the rows that pad the runs.
template <typename T, int kBytes, int kGroup>
__global__ void __launch_bounds__(kMoveThreads) moe_unpermute_backward_kernel(
    const T* gy, int64_t ld_g, const T* z, int64_t ld_z, int pairs_n, int pair_ctas, int h, int topk,
    const int* rows, const int* pairs, const int* offsets, int n_rows,
    const float* weights, T* gz, float* gw) {
    using P = Piece<T, kBytes>;
    constexpr int kAhead = kBytes == 16 ? 4 : 8, kStep = kGroup * P::kN;
    __shared__ float parts[kMoveThreads / 32];
    grid_wait();
    grid_launch_dependents();
    if (int(blockIdx.x) >= pair_ctas) {
        const int pad = int(blockIdx.x) - pair_ctas;
        float zero[P::kN];
#pragma unroll
        for (int i = 0; i < P::kN; ++i) zero[i] = 0.0f;
        int first, end;
        padding_of(pairs, offsets, n_rows, pad / kPadCtas, &first, &end);
        for (int r = first + pad % kPadCtas; r < end; r += kPadCtas) {
            for (int c = threadIdx.x * P::kN; c < h; c += kMoveThreads * P::kN) P::store(gz + int64_t(r) * h + c, zero);
        }
        return;
    }
    const int64_t pair = int64_t(blockIdx.x) * (kMoveThreads / kGroup) + threadIdx.x / kGroup;
    if (pair >= pairs_n) return;  // (whole groups)
    const int r = rows[pair];
    const bool here = r >= 0 && r < n_rows;
    // eight sums a thread: one alone would be a chain of h / 32 additions, each of which can lose half a unit of it
    constexpr int kSums = 8;
    static_assert(kAhead * P::kN % kSums == 0, "a round of pieces goes round the sums as a whole");
    float sums[kSums] = {};
    if (here) {
        const T* const g = gy + pair / topk * ld_g;
        const T* const s = z + int64_t(r) * ld_z;
        T* const to = gz + int64_t(r) * h;
        const float w = weights != nullptr ? weights[pair] : 1.0f;
        for (int c0 = (threadIdx.x % kGroup) * P::kN; c0 < h; c0 += kAhead * kStep) {
            P a[kAhead], b[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                if (c0 + i * kStep < h) {
                    a[i].load(g + c0 + i * kStep);
                    if (gw != nullptr) b[i].load(s + c0 + i * kStep);
                }
            }
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                if (c0 + i * kStep >= h) continue;
                float f[P::kN], o[P::kN];
                a[i].get(f);
                if (gw != nullptr) {
                    float u[P::kN];
                    b[i].get(u);
#pragma unroll
                    for (int j = 0; j < P::kN; ++j) sums[(i * P::kN + j) % kSums] = fmaf(f[j], u[j], sums[(i * P::kN + j) % kSums]);
                }
#pragma unroll
                for (int j = 0; j < P::kN; ++j) o[j] = w * f[j];
                P::store(to + c0 + i * kStep, o);
            }
        }
    }
    if (gw != nullptr) {
        float dot = ((sums[0] + sums[1]) + (sums[2] + sums[3])) + ((sums[4] + sums[5]) + (sums[6] + sums[7]));
#pragma unroll
        for (int d = 16; d > 0; d /= 2) dot += __shfl_xor_sync(0xffffffffu, dot, d);
        if constexpr (kGroup > 32) {
            if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = dot;
            __syncthreads();
            dot = 0.0f;
#pragma unroll
            for (int i = 0; i < kMoveThreads / 32; ++i) dot += parts[i];
        }
        if (threadIdx.x % kGroup == 0) gw[pair] = dot;
    }
}

struct SortOptIn {
    std::mutex mu;
    int done[64] = {};
    int fits[64] = {}, fails[64] = {};  // shared memory a CTA with which a cluster of 16 is known to find room, and not to
};

// Whether the device, or the part of it that this process has, holds a cluster of 16 CTAs with `bytes` of shared memory each.
template <typename Id>
cudaError_t cluster16_fits(SortOptIn& opt, int dev, int bytes, bool* fits) {
    if (dev >= 0 && dev < 64 && bytes <= opt.fits[dev]) return *fits = true, cudaSuccess;
    if (dev >= 0 && dev < 64 && opt.fails[dev] != 0 && bytes >= opt.fails[dev]) return *fits = false, cudaSuccess;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(16);
    cfg.blockDim = dim3(kSortThreads);
    cfg.dynamicSmemBytes = size_t(bytes);
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 16, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    const cudaError_t e = cudaOccupancyMaxActiveClusters(&clusters, moe_sort_kernel<Id>, &cfg);
    if (e != cudaSuccess) return e;
    *fits = clusters > 0;
    if (dev >= 0 && dev < 64) (*fits ? opt.fits : opt.fails)[dev] = bytes;
    return cudaSuccess;
}

template <typename Id>
cudaError_t launch_sort(const void* ids, int pairs_n, int experts, int align, int n_rows, bool pdl, int* rows, int* pairs, int* offsets,
                        int* expert_ids, cudaStream_t stream) {
    static SortOptIn opt;
    // One CTA goes over 128 pairs a warp in 4 steps; from there on 8 CTAs repay the two barriers of their cluster, and 16 (which a kernel
    // has to opt in to, and for which there has to be room) where there are thousands of pairs for each: 65536 pairs 15.2 -> 11.8 us, 32768 9.6 -> 8.5.
    int ctas = pairs_n > 16384 ? 16 : pairs_n > 4096 || n_rows > 16384 ? 8 : 1;
    const auto need = [](int e) { return int(sizeof(int)) * (kSortWarps * e + 4 * e + 1); };
    const int bytes = need(experts);
    if (bytes > 40 * 1024 || ctas > 8) {
        int dev = 0;
        const cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        const std::lock_guard<std::mutex> lock(opt.mu);
        if (dev < 0 || dev >= 64 || opt.done[dev] == 0) {
            cudaError_t f = cudaFuncSetAttribute(moe_sort_kernel<Id>, cudaFuncAttributeMaxDynamicSharedMemorySize, need(kMaxExperts));
            if (f == cudaSuccess) f = cudaFuncSetAttribute(moe_sort_kernel<Id>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (f != cudaSuccess) return f;
            if (dev >= 0 && dev < 64) opt.done[dev] = 1;
        }
        if (ctas > 8) {
            bool fits = false;
            const cudaError_t f = cluster16_fits<Id>(opt, dev, bytes, &fits);
            if (f != cudaSuccess) return f;
            if (!fits) ctas = 8;
        }
    }
    return launch(moe_sort_kernel<Id>, dim3(ctas), dim3(kSortThreads), size_t(bytes), stream, pdl, unsigned(ctas), static_cast<const Id*>(ids),
                  pairs_n, experts, align, n_rows, ctas, rows, pairs, offsets, expert_ids);
}

template <typename Unit>
cudaError_t launch_permute(const void* x, int64_t ld_bytes, int64_t tokens, int64_t row_bytes, int topk, const int* rows, const int* pairs,
                           const int* offsets, int64_t pad_ctas, int n_rows, void* out, bool pdl, cudaStream_t stream) {
    constexpr int kPer = sizeof(Unit) == 16 ? 2 : sizeof(Unit) == 4 ? 4 : 8;
    const int units = int(row_bytes / int64_t(sizeof(Unit)));
    const dim3 grid(unsigned(tokens + pad_ctas), unsigned((units + kMoveThreads * kPer - 1) / (kMoveThreads * kPer)));
    return launch(moe_permute_kernel<Unit, kPer>, grid, dim3(kMoveThreads), 0, stream, pdl, 1, static_cast<const Unit*>(x),
                  ld_bytes / int64_t(sizeof(Unit)), int(tokens), units, topk, rows, pairs, offsets, n_rows, static_cast<Unit*>(out));
}

// What the calls on tokens and rows have in common.
int check_moe(int64_t tokens, int64_t topk, int64_t n_rows, int64_t experts, char* err, size_t errlen) {
    if (tokens < 0 || topk < 0 || n_rows < 0 || experts < 0 || tokens > INT32_MAX || topk > INT32_MAX || n_rows > INT32_MAX ||
        tokens * topk > INT32_MAX || experts > kMaxExperts || tokens * std::max<int64_t>(topk, 1) + experts * kPadCtas > INT32_MAX) {
        return fail(err, errlen, HQ_ERR_INVALID, "at most 2^31 - 1 pairs and rows and %d experts, got %lld tokens of %lld, %lld rows, %lld experts",
                    kMaxExperts, static_cast<long long>(tokens), static_cast<long long>(topk), static_cast<long long>(n_rows),
                    static_cast<long long>(experts));
    }
    return HQ_OK;
}

int element_size(int dtype) { return dtype == HQ_DTYPE_FP32 ? 4 : dtype == HQ_DTYPE_BF16 || dtype == HQ_DTYPE_FP16 ? 2 : 0; }

}  // namespace
}  // namespace hq

extern "C" int hq_moe_sort(const void* ids, int ids_bytes, int64_t tokens, int64_t topk, int64_t num_experts, int64_t align, int64_t n_rows,
                           int use_pdl, int32_t* rows, int32_t* pairs, int32_t* offsets, int32_t* expert_ids, int device, void* stream,
                           char* err, size_t errlen) {
    using hq::fail;
    if (ids_bytes != 4 && ids_bytes != 8) return fail(err, errlen, HQ_ERR_INVALID, "topk_ids must be int32 or int64");
    if (num_experts < 1) return fail(err, errlen, HQ_ERR_INVALID, "num_experts must be at least 1, got %lld", static_cast<long long>(num_experts));
    const int rc = hq::check_moe(tokens, topk, n_rows, num_experts, err, errlen);
    if (rc != HQ_OK) return rc;
    if (align < 1 || align > 4096) return fail(err, errlen, HQ_ERR_INVALID, "align must be in [1, 4096], got %lld", static_cast<long long>(align));
    const int64_t n = tokens * topk;
    if (n > hq::kMaxSortPairs) return fail(err, errlen, HQ_ERR_INVALID, "at most 2^31 - 8192 pairs, got %lld", static_cast<long long>(n));
    // any ids have to fit: what pads the runs of as many experts as there can be
    const int64_t need = (n + (n < num_experts ? n : num_experts) * (align - 1)) / align * align;
    if (n_rows < need) {
        return fail(err, errlen, HQ_ERR_INVALID, "%lld rows are needed for %lld pairs, %lld experts and runs on multiples of %lld, got %lld",
                    static_cast<long long>(need), static_cast<long long>(n), static_cast<long long>(num_experts), static_cast<long long>(align),
                    static_cast<long long>(n_rows));
    }
    if (offsets == nullptr || (n > 0 && (ids == nullptr || rows == nullptr)) || (n_rows > 0 && (pairs == nullptr || expert_ids == nullptr))) {
        return fail(err, errlen, HQ_ERR_INVALID, "null pointer argument");
    }
    const hq::DeviceGuard guard(device);
    if (!guard.ok()) return fail(err, errlen, HQ_ERR_CUDA, "cannot select CUDA device %d", device);
    const auto s = static_cast<cudaStream_t>(stream);
    HQ_CUDA_TRY(ids_bytes == 8 ? hq::launch_sort<int64_t>(ids, int(n), int(num_experts), int(align), int(n_rows), use_pdl != 0, rows, pairs,
                                                          offsets, expert_ids, s)
                               : hq::launch_sort<int32_t>(ids, int(n), int(num_experts), int(align), int(n_rows), use_pdl != 0, rows, pairs,
                                                          offsets, expert_ids, s));
    return HQ_OK;
}

extern "C" int hq_moe_permute(const void* input, int64_t ld_bytes, int64_t tokens, int64_t row_bytes, int64_t topk, const int32_t* rows,
                              const int32_t* pairs, const int32_t* offsets, int64_t num_experts, int64_t n_rows, int padded, int use_pdl,
                              void* output, int device, void* stream, char* err, size_t errlen) {
    using hq::fail;
    const int rc = hq::check_moe(tokens, topk, n_rows, num_experts, err, errlen);
    if (rc != HQ_OK) return rc;
    if (row_bytes < 0 || row_bytes > (int64_t(1) << 24)) return fail(err, errlen, HQ_ERR_INVALID, "rows of at most 16 MiB");
    if (tokens == 0 || topk == 0 || row_bytes == 0) return HQ_OK;  // no pairs, no runs
    if (input == nullptr || rows == nullptr || pairs == nullptr || offsets == nullptr || output == nullptr) {
        return fail(err, errlen, HQ_ERR_INVALID, "null pointer argument");
    }
    const hq::DeviceGuard guard(device);
    if (!guard.ok()) return fail(err, errlen, HQ_ERR_CUDA, "cannot select CUDA device %d", device);
    const auto s = static_cast<cudaStream_t>(stream);
    const auto fits = [&](size_t a) {
        return hq::aligned(input, a) && hq::aligned(output, a) && ld_bytes % int64_t(a) == 0 && row_bytes % int64_t(a) == 0;
    };
    const auto go = [&](auto unit) {
        return hq::launch_permute<decltype(unit)>(input, ld_bytes, tokens, row_bytes, int(topk), rows, pairs, offsets,
                                                  padded != 0 ? num_experts * hq::kPadCtas : 0, int(n_rows), output, use_pdl != 0, s);
    };
    HQ_CUDA_TRY(fits(16) ? go(uint4{}) : fits(4) ? go(uint32_t{}) : fits(2) ? go(uint16_t{}) : go(uint8_t{}));
    return HQ_OK;
}

extern "C" int hq_moe_unpermute(const void* input, int64_t ld_elems, int dtype, int64_t n_rows, int64_t h, int64_t tokens, int64_t topk,
                                const int32_t* rows, const float* weights, int use_pdl, void* output, int device, void* stream, char* err,
                                size_t errlen) {
    using hq::fail;
    const int rc = hq::check_moe(tokens, topk, n_rows, 0, err, errlen);
    if (rc != HQ_OK) return rc;
    const int size = hq::element_size(dtype);
    if (size == 0) return fail(err, errlen, HQ_ERR_INVALID, "input dtype must be bfloat16, float16 or float32");
    if (h < 0 || h > (int64_t(1) << 22)) return fail(err, errlen, HQ_ERR_INVALID, "hidden size must be at most 2^22");
    if (tokens == 0 || h == 0) return HQ_OK;
    if (output == nullptr || (topk > 0 && rows == nullptr) || (n_rows > 0 && input == nullptr)) {
        return fail(err, errlen, HQ_ERR_INVALID, "null pointer argument");
    }
    const hq::DeviceGuard guard(device);
    if (!guard.ok()) return fail(err, errlen, HQ_ERR_CUDA, "cannot select CUDA device %d", device);
    const auto fits = [&](int a) { return hq::aligned(input, a) && hq::aligned(output, a) && ld_elems * size % a == 0 && h * size % a == 0; };
    const int bytes = fits(16) ? 16 : fits(4) ? 4 : 2;
    // several pieces a thread where rows fill them and there are tokens for all SMs: more bytes in flight per CTA
    const int64_t one = hq::kMoveThreads * int64_t(std::max(1, bytes / size));
    const int pieces = bytes == 16 ? 2 : 4;
    const bool many = h >= pieces * one && tokens >= 1024;
    const int64_t per = many ? pieces * one : one;
    const dim3 grid(unsigned(tokens), unsigned((h + per - 1) / per));
    const auto go = [&](auto kernel, auto* z) {
        using T = std::remove_const_t<std::remove_pointer_t<decltype(z)>>;
        return hq::launch(kernel, grid, dim3(hq::kMoveThreads), 0, static_cast<cudaStream_t>(stream), use_pdl != 0, 1, z, ld_elems, int(tokens),
                          int(h), int(topk), rows, int(n_rows), weights, static_cast<T*>(output));
    };
    const auto typed = [&](auto* z) {
        using T = std::remove_const_t<std::remove_pointer_t<decltype(z)>>;
        if (bytes == 16) return many ? go(hq::moe_unpermute_kernel<T, 16, 2>, z) : go(hq::moe_unpermute_kernel<T, 16, 1>, z);
        if constexpr (sizeof(T) == 2) {
            if (bytes == 2) return many ? go(hq::moe_unpermute_kernel<T, 2, 4>, z) : go(hq::moe_unpermute_kernel<T, 2, 1>, z);
        }
        return many ? go(hq::moe_unpermute_kernel<T, 4, 4>, z) : go(hq::moe_unpermute_kernel<T, 4, 1>, z);
    };
    HQ_CUDA_TRY(dtype == HQ_DTYPE_BF16   ? typed(static_cast<const __nv_bfloat16*>(input))
                : dtype == HQ_DTYPE_FP16 ? typed(static_cast<const __half*>(input))
                                         : typed(static_cast<const float*>(input)));
    return HQ_OK;
}

extern "C" int hq_moe_unpermute_backward(const void* grad_output, int64_t ld_grad, const void* input, int64_t ld_input, int dtype, int64_t n_rows,
                                         int64_t h, int64_t tokens, int64_t topk, const int32_t* rows, const int32_t* pairs,
                                         const int32_t* offsets, int64_t num_experts, int padded, const float* weights, int use_pdl,
                                         void* grad_input, float* grad_weights, int device, void* stream, char* err, size_t errlen) {
    using hq::fail;
    const int rc = hq::check_moe(tokens, topk, n_rows, num_experts, err, errlen);
    if (rc != HQ_OK) return rc;
    const int size = hq::element_size(dtype);
    if (size == 0) return fail(err, errlen, HQ_ERR_INVALID, "input dtype must be bfloat16, float16 or float32");
    if (h < 0 || h > (int64_t(1) << 22)) return fail(err, errlen, HQ_ERR_INVALID, "hidden size must be at most 2^22");
    if (tokens == 0 || topk == 0) return HQ_OK;
    if ((h > 0 && (grad_output == nullptr || grad_input == nullptr || (grad_weights != nullptr && input == nullptr))) || rows == nullptr ||
        pairs == nullptr || offsets == nullptr) {
        return fail(err, errlen, HQ_ERR_INVALID, "null pointer argument");
    }
    const hq::DeviceGuard guard(device);
    if (!guard.ok()) return fail(err, errlen, HQ_ERR_CUDA, "cannot select CUDA device %d", device);
    const auto fits = [&](int a) {
        return hq::aligned(grad_output, a) && hq::aligned(grad_input, a) && hq::aligned(input, a) && ld_grad * size % a == 0 &&
               ld_input * size % a == 0 && h * size % a == 0;
    };
    const int bytes = fits(16) ? 16 : fits(4) ? 4 : 2;
    // a warp per pair once they fill the SMs (two CTAs of 8 warps each), else a CTA
    const int sms = hq_sm_count(device);
    if (sms <= 0) return fail(err, errlen, HQ_ERR_CUDA, "cannot read the SM count of CUDA device %d", device);
    const int64_t n = tokens * topk;
    const bool warps = n >= int64_t(sms) * 16;
    const int64_t pair_ctas = warps ? (n + hq::kMoveThreads / 32 - 1) / (hq::kMoveThreads / 32) : n;
    const dim3 grid(unsigned(pair_ctas + (padded != 0 ? num_experts * hq::kPadCtas : 0)));
    const auto go = [&](auto kernel, auto* g) {
        using T = std::remove_const_t<std::remove_pointer_t<decltype(g)>>;
        return hq::launch(kernel, grid, dim3(hq::kMoveThreads), 0, static_cast<cudaStream_t>(stream), use_pdl != 0, 1, g, ld_grad,
                          static_cast<const T*>(input), ld_input, int(n), int(pair_ctas), int(h), int(topk), rows, pairs, offsets, int(n_rows), weights,
                          static_cast<T*>(grad_input), grad_weights);
    };
    const auto typed = [&](auto* g) {
        using T = std::remove_const_t<std::remove_pointer_t<decltype(g)>>;
        constexpr int kAll = hq::kMoveThreads;
        if (bytes == 16) return warps ? go(hq::moe_unpermute_backward_kernel<T, 16, 32>, g) : go(hq::moe_unpermute_backward_kernel<T, 16, kAll>, g);
        if constexpr (sizeof(T) == 2) {
            if (bytes == 2) return warps ? go(hq::moe_unpermute_backward_kernel<T, 2, 32>, g) : go(hq::moe_unpermute_backward_kernel<T, 2, kAll>, g);
        }
        return warps ? go(hq::moe_unpermute_backward_kernel<T, 4, 32>, g) : go(hq::moe_unpermute_backward_kernel<T, 4, kAll>, g);
    };
    HQ_CUDA_TRY(dtype == HQ_DTYPE_BF16   ? typed(static_cast<const __nv_bfloat16*>(grad_output))
                : dtype == HQ_DTYPE_FP16 ? typed(static_cast<const __half*>(grad_output))
                                         : typed(static_cast<const float*>(grad_output)));
    return HQ_OK;
}
