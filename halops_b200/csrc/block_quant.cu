// Quantisers to e4m3 codes with a float32 scale per block of 128 (block_quant.cuh has the rule): rows in blocks of
// 1 x 128, also of SwiGLU and of gathered tokens, and tiles of 128 x 128, for weights and for transposed operands.
//
// All are bound by HBM: a value is 2 bytes read and 1 byte (plus 1/32 for rows) written.

#include "block_quant.cuh"

namespace hq {
namespace {

constexpr int kRowThreads = 256;

// (Not ld.global.nc, which is for data that nothing writes while the kernel runs: see block_quant.cuh.)
__device__ __forceinline__ uint4 load_stream(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// ---------------------------------------------------------------------------- rows
//
// A lane holds 16 neighbouring values, 8 lanes a block; a warp has kVec pieces of 512 values of one row, all
// loaded before the first is worked on.  (With 8 values a lane and 8-byte stores of codes 8192 x 8192 took 39.3 us, so 33.3.)

// Maximum over the 8 lanes that hold a block.
__device__ __forceinline__ uint32_t max8(uint32_t m) {
#pragma unroll
    for (int d = 1; d < 8; d *= 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
    return m;
}

template <typename T, int kVec>
__global__ void __launch_bounds__(kRowThreads) block_quant_rows_kernel(const T* x, int64_t ld, int64_t m, int k, int segs,
                                                                       uint8_t* q, float* sf) {
    grid_wait();
    grid_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int64_t task = int64_t(blockIdx.x) * (kRowThreads / 32) + (threadIdx.x >> 5);
    const int64_t row = task / segs;
    if (row >= m) return;
    const int col = int(task - row * segs) * (kVec * 512) + lane * 16;
    const int kb = (k + kQBlock - 1) / kQBlock;
    const T* const src = x + row * ld + col;
    uint4 v[kVec][2];
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
        v[i][0] = v[i][1] = make_uint4(0, 0, 0, 0);
        if (col + i * 512 < k) v[i][0] = load_stream(src + i * 512), v[i][1] = load_stream(src + i * 512 + 8);
    }
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
        const int c = col + i * 512;
        const BlockScale s = block_scale(magnitude_f32<T>(max8(max(amax16(v[i][0]), amax16(v[i][1])))), true);
        if (c < k) {
            const uint2 lo = codes8<T>(v[i][0], s), hi = codes8<T>(v[i][1], s);
            *reinterpret_cast<uint4*>(q + row * k + c) = make_uint4(lo.x, lo.y, hi.x, hi.y);
            if ((lane & 7) == 0) sf[row * kb + c / kQBlock] = s.scale;
        }
    }
}

// ---------------------------------------------------------------------------- SwiGLU
//
// h = gate * sigmoid(gate) * up in float32, quantised from there; gate is the first half of a row, up the second.
// Rows from *row_limit on (behind the last expert's run) are left alone.

// exp(-a) for a >= 0: 2^t for the rounded t = -a log2(e), corrected by the rest of t, which a second fma gives exactly, so that the error does
// not grow with a (ex2's 2^-22 and two roundings).  Zero from 87.3 on, below which it would be subnormal.
__device__ __forceinline__ float exp_minus(float a) {
    constexpr float kLog2e = 1.44269504f, kLog2eRest = 1.92596299e-8f, kLn2 = 0.693147181f;
    a = fminf(a, 128.0f);  // (of an infinity the rest would be NaN)
    const float t = a * -kLog2e;
    float p;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(t));
    const float rest = fmaf(a, -kLog2eRest, fmaf(a, -kLog2e, -t));
    return fmaf(p, rest * kLn2, p);
}

// gate * sigmoid(gate) from e = exp(-|gate|): nothing overflows, and the divisor is in [1, 2].
// 16384 x 2 x 2048 takes 33.1 us, with expf and a correctly rounded quotient 42.2, with uncorrected exponentials (3e-6 off at -60, zero below -87.3) 30.2.
__device__ __forceinline__ float silu(float gate) {
    const float e = exp_minus(fabsf(gate));
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return (gate < 0.0f ? gate * e : gate) * r;
}

// Gates below -87: silu leaves the range of normal numbers, while its product with a large `up` may not.  (1 + e is 1 there.)
constexpr float kFarGate = -87.0f;
template <typename T>
constexpr uint32_t kFarBits = 0xc2aeu;  // kFarGate as T: all lower gates, and negative NaNs, have larger bits
template <>
constexpr uint32_t kFarBits<__half> = 0xd570u;
template <bool kFar>
__device__ __forceinline__ float gated(float gate, float up) {
    if (kFar && gate < kFarGate) {
        const float half = exp_minus(-0.5f * gate);
        return (gate * half) * (up * half);
    }
    return silu(gate) * up;
}
template <typename T, bool kFar>
__device__ __forceinline__ void gated16(const uint4 (&gate)[2], const uint4 (&up)[2], float2 (&h)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t gw[4] = {gate[i].x, gate[i].y, gate[i].z, gate[i].w}, uw[4] = {up[i].x, up[i].y, up[i].z, up[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 g = two_floats<T>(gw[j]), u = two_floats<T>(uw[j]);
            h[i * 4 + j] = make_float2(gated<kFar>(g.x, u.x), gated<kFar>(g.y, u.y));
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) swiglu_block_quant_kernel(const T* x, int64_t ld, int64_t m, int k, int segs,
                                                                         const int* row_limit, uint8_t* q,
                                                                         float* sf) {
    grid_wait();
    grid_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int64_t task = int64_t(blockIdx.x) * (kRowThreads / 32) + (threadIdx.x >> 5);
    const int64_t row = task / segs;
    if (row >= m || (row_limit != nullptr && row >= *row_limit)) return;
    const int c = int(task - row * segs) * 512 + lane * 16;
    const int kb = (k + kQBlock - 1) / kQBlock;
    const T* const src = x + row * ld + c;
    uint4 gate[2], up[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        gate[i] = up[i] = make_uint4(0, 0, 0, 0);
        if (c < k) gate[i] = load_stream(src + i * 8), up[i] = load_stream(src + k + i * 8);
    }
    float2 h[8];
    uint32_t amax = 0;
    const uint32_t low = __vmaxu2(__vmaxu2(__vmaxu2(gate[0].x, gate[0].y), __vmaxu2(gate[0].z, gate[0].w)),
                                  __vmaxu2(__vmaxu2(gate[1].x, gate[1].y), __vmaxu2(gate[1].z, gate[1].w)));
    if (max(low & 0xffffu, low >> 16) <= kFarBits<T>) {
        gated16<T, false>(gate, up, h);
    } else {  // (both forms of every value: rare, and as a second pass over the values it cost registers, 16384 x 2 x 2048 39 us)
        gated16<T, true>(gate, up, h);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = max(amax, max(__float_as_uint(h[j].x) & 0x7fffffffu, __float_as_uint(h[j].y) & 0x7fffffffu));
    const BlockScale s = block_scale(max8(amax), false);
    if (c < k) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = code2(h[2 * j], s) | code2(h[2 * j + 1], s) << 16;
        *reinterpret_cast<uint4*>(q + row * k + c) = make_uint4(w[0], w[1], w[2], w[3]);
        if ((lane & 7) == 0) sf[row * kb + c / kQBlock] = s.scale;
    }
}

// ---------------------------------------------------------------------------- gathered tokens
//
// A CTA reads and quantises 4096 values of one token, 16 a thread, once and writes them to each of the token's rows.  The blocks
// behind the tokens write the rows that pad the experts' runs as the codes of zeros.

constexpr int kPadCtas = 16;  // CTAs that share the padding of a run

template <typename T>
__global__ void __launch_bounds__(kRowThreads) permute_block_quant_kernel(const T* x, int64_t ld, int tokens, int k, int topk,
                                                                          const int* rows, const int* pairs,
                                                                          const int* offsets, int n_rows,
                                                                          uint8_t* q, float* sf) {
    grid_wait();
    grid_launch_dependents();
    const int kb = (k + kQBlock - 1) / kQBlock;
    const int c = blockIdx.y * (kRowThreads * 16) + threadIdx.x * 16;
    if (int(blockIdx.x) >= tokens) {
        const int pad = int(blockIdx.x) - tokens, e = pad / kPadCtas;
        const BlockScale s = block_scale(0, true);
        // the first row without a pair, by halving
        int first = max(offsets[e], 0);
        const int end = min(offsets[e + 1], n_rows);
        for (int n = end - first; n > 0;) {
            const int half = n / 2;
            if (pairs[first + half] >= 0) first += half + 1, n -= half + 1; else n = half;
        }
        for (int r = first + pad % kPadCtas; r < end; r += kPadCtas) {
            if (c < k) {
                *reinterpret_cast<uint4*>(q + int64_t(r) * k + c) = make_uint4(0, 0, 0, 0);
                if ((threadIdx.x & 7) == 0) sf[int64_t(r) * kb + c / kQBlock] = s.scale;
            }
        }
        return;
    }
    const int64_t token = blockIdx.x;
    uint4 v = make_uint4(0, 0, 0, 0), w = v;
    if (c < k) v = load_stream(x + token * ld + c), w = load_stream(x + token * ld + c + 8);
    const BlockScale s = block_scale(magnitude_f32<T>(max8(max(amax16(v), amax16(w)))), true);
    const uint2 lo = codes8<T>(v, s), hi = codes8<T>(w, s);
    if (c >= k) return;
    for (int j0 = 0; j0 < topk; j0 += 8) {
        int r[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = j0 + j < topk ? rows[token * topk + j0 + j] : -1;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (r[j] < 0 || r[j] >= n_rows) continue;
            *reinterpret_cast<uint4*>(q + int64_t(r[j]) * k + c) = make_uint4(lo.x, lo.y, hi.x, hi.y);
            if ((threadIdx.x & 7) == 0) sf[int64_t(r[j]) * kb + c / kQBlock] = s.scale;
        }
    }
}

// ---------------------------------------------------------------------------- tiles of 128 x 128
//
// kSquare: one scale per tile, else one per column of 128 rows (the rows of the transposed matrix).  A thread holds 8 x 8
// values: 16 threads side by side read 256 bytes of a row, a thread's rows follow one another, so that the transposed codes
// of a column are 8 bytes of one thread.  They pass through shared memory in pieces of 8 bytes, whose place in a line of 128
// bytes is XORed with the line's thread column: neither side has bank conflicts.

template <typename T, bool kSquare, bool kTranspose>
__global__ void __launch_bounds__(256) block_quant_tile_kernel(const T* x, int64_t ld, int64_t batch_stride, int64_t m, int k,
                                                               int64_t m_out, uint8_t* q, float* sf) {
    __shared__ uint32_t amax_s[8][64];
    __shared__ float2 factors[kSquare ? 1 : 128];  // of each column: 448 / amax, and whether its block is finite
    __shared__ __align__(16) uint8_t tile[kTranspose ? 128 * 128 : 16];
    grid_wait();
    grid_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int cg = tid & 15, rg = tid >> 4;  // 8 columns from cg * 8, 8 rows from rg * 8
    const int64_t row0 = int64_t(blockIdx.x) * kQBlock;
    const int col0 = blockIdx.y * kQBlock, col = col0 + cg * 8;
    const int kb = (k + kQBlock - 1) / kQBlock;
    const int64_t mb = (m + kQBlock - 1) / kQBlock;
    const T* const src = x + int64_t(blockIdx.z) * batch_stride + (row0 + rg * 8) * ld + col;
    uint4 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] = make_uint4(0, 0, 0, 0);
        if (row0 + rg * 8 + i < m && col < k) v[i] = load_stream(src + i * ld);
    }
    BlockScale s[kSquare ? 1 : 8];
    if constexpr (kSquare) {
        uint32_t a = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) a = max(a, amax16(v[i]));
        a = __reduce_max_sync(0xffffffffu, a);
        if (lane == 0) amax_s[0][warp] = a;
        __syncthreads();
        a = 0;
#pragma unroll
        for (int w = 0; w < 8; ++w) a = max(a, amax_s[0][w]);
        s[0] = block_scale(magnitude_f32<T>(a), true);
        if (tid == 0) {
            sf[int64_t(blockIdx.z) * mb * kb + (kTranspose ? int64_t(blockIdx.y) * mb + blockIdx.x : int64_t(blockIdx.x) * kb + blockIdx.y)] =
                s[0].scale;
        }
    } else {
        // two columns a word: the maxima of 8 rows, of the warp's other 8 rows, of the 8 warps
        uint32_t a[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            a[0] = __vmaxu2(a[0], v[i].x & 0x7fff7fffu);
            a[1] = __vmaxu2(a[1], v[i].y & 0x7fff7fffu);
            a[2] = __vmaxu2(a[2], v[i].z & 0x7fff7fffu);
            a[3] = __vmaxu2(a[3], v[i].w & 0x7fff7fffu);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            a[j] = __vmaxu2(a[j], __shfl_xor_sync(0xffffffffu, a[j], 16));
            if (lane < 16) amax_s[warp][cg * 4 + j] = a[j];
        }
        __syncthreads();
        // a thread per column: the divisions are made once for its 16 readers
        if (tid < 128) {
            uint32_t b = 0;
#pragma unroll
            for (int w = 0; w < 8; ++w) b = __vmaxu2(b, amax_s[w][tid / 2]);
            const BlockScale one = block_scale(magnitude_f32<T>(tid % 2 == 0 ? b & 0xffffu : b >> 16), true);
            factors[tid] = make_float2(one.inverse, __uint_as_float(one.add));
            if (col0 + tid < k) sf[int64_t(col0 + tid) * mb + blockIdx.x] = one.scale;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float2 f = factors[cg * 8 + j];
            s[j].inverse = f.x;
            s[j].add = __float_as_uint(f.y);
            s[j].mask = s[j].add != 0 ? ~7u : ~0u;
        }
    }
    if constexpr (!kTranspose) {
        uint8_t* const out = q + (int64_t(blockIdx.z) * m + row0 + rg * 8) * k + col;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (row0 + rg * 8 + i < m && col < k) *reinterpret_cast<uint2*>(out + int64_t(i) * k) = codes8<T>(v[i], s[0]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            // columns j and j + 1: the same word of every row
            uint32_t lo[2] = {0, 0}, hi[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t w = j == 0 ? v[i].x : j == 2 ? v[i].y : j == 4 ? v[i].z : v[i].w;
                const float2 f = two_floats<T>(w);
                const BlockScale &s0 = s[kSquare ? 0 : j], &s1 = s[kSquare ? 0 : j + 1];
                const float a = __uint_as_float((__float_as_uint(f.x * s0.inverse) + s0.add) & s0.mask);
                const float b = __uint_as_float((__float_as_uint(f.y * s1.inverse) + s1.add) & s1.mask);
                const uint32_t c = e4m3x2(a, b);
                lo[i / 4] |= (c & 0xffu) << (i % 4 * 8);
                hi[i / 4] |= (c >> 8) << (i % 4 * 8);
            }
            uint8_t* const line = tile + (cg * 8 + j) * 128 + (rg ^ cg) * 8;
            *reinterpret_cast<uint2*>(line) = make_uint2(lo[0], lo[1]);
            *reinterpret_cast<uint2*>(line + 128) = make_uint2(hi[0], hi[1]);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = i * 16 + rg;  // column of the tile = row of the transposed matrix
            const uint2 w = *reinterpret_cast<const uint2*>(tile + c * 128 + (cg ^ (c / 8)) * 8);
            if (col0 + c < k && row0 + cg * 8 < m_out) {
                *reinterpret_cast<uint2*>(q + (int64_t(blockIdx.z) * k + col0 + c) * m_out + row0 + cg * 8) = w;
            }
        }
    }
}

bool quant_operand(const void* input, int64_t ld, int64_t k) {
    return ld >= k && ld % 8 == 0 && aligned(input, 16);
}

template <typename T>
cudaError_t launch_block_quant(const void* input, int64_t ld, int64_t batch_stride, int64_t batches, int64_t m, int k, bool square,
                               bool transpose, bool pdl, void* q, void* sf, cudaStream_t stream) {
    const T* const x = static_cast<const T*>(input);
    uint8_t* const oq = static_cast<uint8_t*>(q);
    float* const os = static_cast<float*>(sf);
    if (!square && !transpose) {
        // Few rows: a piece of 512 values per warp, for more warps; else 2, for more bytes in flight per warp.
        const bool few = m * k < (int64_t(1) << 20);
        const int segs = (k + (few ? 511 : 1023)) / (few ? 512 : 1024);
        const dim3 grid(unsigned((m * segs + kRowThreads / 32 - 1) / (kRowThreads / 32)));
        return few ? launch(block_quant_rows_kernel<T, 1>, grid, dim3(kRowThreads), 0, stream, pdl, 1, x, ld, m, k, segs, oq, os)
                   : launch(block_quant_rows_kernel<T, 2>, grid, dim3(kRowThreads), 0, stream, pdl, 1, x, ld, m, k, segs, oq, os);
    }
    const int64_t m_out = (m + 15) / 16 * 16;
    const dim3 grid(unsigned((m + kQBlock - 1) / kQBlock), unsigned((k + kQBlock - 1) / kQBlock), unsigned(batches));
    const auto go = [&](auto kernel) { return launch(kernel, grid, dim3(256), 0, stream, pdl, 1, x, ld, batch_stride, m, k, m_out, oq, os); };
    if (square && transpose) return go(block_quant_tile_kernel<T, true, true>);
    if (square) return go(block_quant_tile_kernel<T, true, false>);
    return go(block_quant_tile_kernel<T, false, true>);
}

}  // namespace
}  // namespace hq

extern "C" int hq_block_quant(const void* input, int64_t ld_elems, int64_t batch_stride, int in_dtype, int64_t batches, int64_t m, int64_t k,
                              int block_rows, int transpose, int use_pdl, void* out_q, void* out_sf, int device, void* stream, char* err,
                              size_t errlen) {
    using hq::fail;
    if (in_dtype != HQ_DTYPE_BF16 && in_dtype != HQ_DTYPE_FP16) {
        return fail(err, errlen, HQ_ERR_INVALID, "input dtype must be bfloat16 or float16");
    }
    if (block_rows != 1 && block_rows != 128) {
        return fail(err, errlen, HQ_ERR_INVALID, "block must be (1, 128) or (128, 128)");
    }
    if (batches < 0 || m < 0 || k < 0 || k > (int64_t(1) << 22) || m > (int64_t(1) << 31) || batches > 65535) {
        return fail(err, errlen, HQ_ERR_INVALID, "input is too large: at most 65535 matrices of 2^31 x 2^22");
    }
    if (k % 16 != 0) {
        return fail(err, errlen, HQ_ERR_INVALID, "k must be divisible by 16, got k=%lld", static_cast<long long>(k));
    }
    if (batches == 0 || m == 0 || k == 0) return HQ_OK;
    if (batches > 1 && block_rows == 1) {
        return fail(err, errlen, HQ_ERR_INVALID, "blocks of (1, 128) are taken of a matrix, blocks of (128, 128) of several");
    }
    if (input == nullptr || out_q == nullptr || out_sf == nullptr) return fail(err, errlen, HQ_ERR_INVALID, "null pointer argument");
    if (!hq::quant_operand(input, ld_elems, k) || batch_stride % 8 != 0) {
        return fail(err, errlen, HQ_ERR_INVALID, "input rows must be contiguous and 16-byte aligned");
    }
    if (!hq::aligned(out_q, 16) || !hq::aligned(out_sf, 4)) {
        return fail(err, errlen, HQ_ERR_INVALID, "output_quant must be 16-byte aligned");
    }
    if (block_rows == 1 && transpose == 0 && m * ((k + 255) / 256) > (int64_t(1) << 33)) {
        return fail(err, errlen, HQ_ERR_INVALID, "m is too large for one launch");
    }
    const hq::DeviceGuard guard(device);
    if (!guard.ok()) return fail(err, errlen, HQ_ERR_CUDA, "cannot select CUDA device %d", device);
    const auto s = static_cast<cudaStream_t>(stream);
    const bool square = block_rows == 128;
    HQ_CUDA_TRY(in_dtype == HQ_DTYPE_BF16
                    ? hq::launch_block_quant<__nv_bfloat16>(input, ld_elems, batch_stride, batches, m, int(k), square, transpose != 0,
                                                            use_pdl != 0, out_q, out_sf, s)
                    : hq::launch_block_quant<__half>(input, ld_elems, batch_stride, batches, m, int(k), square, transpose != 0,
                                                     use_pdl != 0, out_q, out_sf, s));
    return HQ_OK;
}

extern "C" int hq_swiglu_block_quant(const void* input, int64_t ld_elems, int in_dtype, int64_t m, int64_t k, const int32_t* row_limit,
                                     int use_pdl, void* out_q, void* out_sf, int device, void* stream, char* err, size_t errlen) {
    using hq::fail;
    if (in_dtype != HQ_DTYPE_BF16 && in_dtype != HQ_DTYPE_FP16) {
        return fail(err, errlen, HQ_ERR_INVALID, "input dtype must be bfloat16 or float16");
    }
    if (m < 0 || k < 0 || k > (int64_t(1) << 22) || m * ((k + 511) / 512) > (int64_t(1) << 33)) {
        return fail(err, errlen, HQ_ERR_INVALID, "input is too large for one launch");
    }
    if (k % 16 != 0) {
        return fail(err, errlen, HQ_ERR_INVALID, "half of the columns must be divisible by 16, got %lld", static_cast<long long>(k));
    }
    if (m == 0 || k == 0) return HQ_OK;
    if (input == nullptr || out_q == nullptr || out_sf == nullptr) return fail(err, errlen, HQ_ERR_INVALID, "null pointer argument");
    if (!hq::quant_operand(input, ld_elems, 2 * k)) {
        return fail(err, errlen, HQ_ERR_INVALID, "input rows must be contiguous and 16-byte aligned");
    }
    if (!hq::aligned(out_q, 16) || !hq::aligned(out_sf, 4)) {
        return fail(err, errlen, HQ_ERR_INVALID, "output_quant must be 16-byte aligned");
    }
    const hq::DeviceGuard guard(device);
    if (!guard.ok()) return fail(err, errlen, HQ_ERR_CUDA, "cannot select CUDA device %d", device);
    const int segs = int((k + 511) / 512);
    const dim3 grid(unsigned((m * segs + hq::kRowThreads / 32 - 1) / (hq::kRowThreads / 32)));
    const auto go = [&](auto kernel, auto* x) {
        return hq::launch(kernel, grid, dim3(hq::kRowThreads), 0, static_cast<cudaStream_t>(stream), use_pdl != 0, 1, x, ld_elems, m, int(k),
                          segs, row_limit, static_cast<uint8_t*>(out_q), static_cast<float*>(out_sf));
    };
    HQ_CUDA_TRY(in_dtype == HQ_DTYPE_BF16 ? go(hq::swiglu_block_quant_kernel<__nv_bfloat16>, static_cast<const __nv_bfloat16*>(input))
                                          : go(hq::swiglu_block_quant_kernel<__half>, static_cast<const __half*>(input)));
    return HQ_OK;
}

extern "C" int hq_moe_permute_block_quant(const void* input, int64_t ld_elems, int in_dtype, int64_t tokens, int64_t k, int64_t topk,
                                          const int32_t* rows, const int32_t* pairs, const int32_t* offsets, int64_t num_experts,
                                          int64_t n_rows, int padded, int use_pdl, void* out_q, void* out_sf, int device, void* stream,
                                          char* err, size_t errlen) {
    using hq::fail;
    if (in_dtype != HQ_DTYPE_BF16 && in_dtype != HQ_DTYPE_FP16) {
        return fail(err, errlen, HQ_ERR_INVALID, "input dtype must be bfloat16 or float16");
    }
    if (tokens < 0 || topk < 0 || num_experts < 0 || n_rows < 0 || tokens * topk > INT32_MAX || n_rows > INT32_MAX || num_experts > 65535 ||
        tokens + num_experts * hq::kPadCtas > INT32_MAX) {
        return fail(err, errlen, HQ_ERR_INVALID, "too many tokens, rows or experts");
    }
    if (k < 0 || k > (int64_t(1) << 22) || k % 16 != 0) {
        return fail(err, errlen, HQ_ERR_INVALID, "hidden size must be divisible by 16 and at most 2^22, got %lld", static_cast<long long>(k));
    }
    if (tokens == 0 || topk == 0 || k == 0) return HQ_OK;  // no pairs, no runs
    if (input == nullptr || rows == nullptr || pairs == nullptr || offsets == nullptr || out_q == nullptr || out_sf == nullptr) {
        return fail(err, errlen, HQ_ERR_INVALID, "null pointer argument");
    }
    if (!hq::quant_operand(input, ld_elems, k)) {
        return fail(err, errlen, HQ_ERR_INVALID, "input rows must be contiguous and 16-byte aligned");
    }
    if (!hq::aligned(out_q, 16) || !hq::aligned(out_sf, 4)) {
        return fail(err, errlen, HQ_ERR_INVALID, "output_quant must be 16-byte aligned");
    }
    const hq::DeviceGuard guard(device);
    if (!guard.ok()) return fail(err, errlen, HQ_ERR_CUDA, "cannot select CUDA device %d", device);
    const dim3 grid(unsigned(tokens + (padded != 0 ? num_experts * hq::kPadCtas : 0)), unsigned((k + hq::kRowThreads * 16 - 1) / (hq::kRowThreads * 16)));
    const auto go = [&](auto kernel, auto* x) {
        return hq::launch(kernel, grid, dim3(hq::kRowThreads), 0, static_cast<cudaStream_t>(stream), use_pdl != 0, 1, x, ld_elems,
                          int(tokens), int(k), int(topk), rows, pairs, offsets, int(n_rows), static_cast<uint8_t*>(out_q),
                          static_cast<float*>(out_sf));
    };
    HQ_CUDA_TRY(in_dtype == HQ_DTYPE_BF16 ? go(hq::permute_block_quant_kernel<__nv_bfloat16>, static_cast<const __nv_bfloat16*>(input))
                                          : go(hq::permute_block_quant_kernel<__half>, static_cast<const __half*>(input)));
    return HQ_OK;
}
