// Row-wise kernels of the 8-bit linear layer: quantization to e4m3 with power-of-two block scales, the RMS norm
// that writes its output in that form, and the norm's backward pass.
//
// The 8-bit form.  A block is 128 neighbouring values of a row, or a tile of 128 x 128.  Its scale is the
// smallest 2^e with max|v| <= 448 * 2^e (448 is e4m3's largest value), held as the e8m0 byte e + 127; the
// values are v * 2^-e, rounded once to nearest even.  v * 2^-e is exact in fp32 (or far below e4m3's smallest
// step), so that rounding is the only one, and q * 2^e is exact in bf16 again: what reads the 8-bit form later
// loses nothing more.  A block of zeros has scale 1; one that holds an infinity or a NaN has the NaN scale
// (255) and NaN values, so that it shows.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "ptx.cuh"

namespace vk {

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }

// Eight neighbouring elements as they lie in memory.
template <typename T>
struct alignas(16) Vec8 {
    T v[8];
};

// n elements (the rest become zeros).  VEC: n is at least 8 or at most 0, and the address is 16-byte aligned; then the
// load is one predicated instruction, and several stay in flight together.
template <bool VEC, typename T>
__device__ __forceinline__ Vec8<T> load8(const T* src, int n)
{
    Vec8<T> r;
    if constexpr (VEC) {
        const uint4* s = reinterpret_cast<const uint4*>(src);
        uint4* d = reinterpret_cast<uint4*>(&r);
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(r) / 16); ++i) d[i] = n > 0 ? s[i] : make_uint4(0, 0, 0, 0);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.v[i] = i < n ? src[i] : from_f32<T>(0.f);
    }
    return r;
}

template <bool VEC, typename T>
__device__ __forceinline__ void store8(T* dst, const Vec8<T>& r, int n)
{
    if constexpr (VEC) {
        if (n <= 0) return;
        const uint4* s = reinterpret_cast<const uint4*>(&r);
        uint4* d = reinterpret_cast<uint4*>(dst);
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(r) / 16); ++i) d[i] = s[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) dst[i] = r.v[i];
    }
}

// |v| as an integer that orders like the number, NaN above infinity above every finite value.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The e8m0 byte of a block whose largest |v| has these bits.  With |v| = 1.f * 2^x: 448 = 1.75 * 2^8, so e is
// x - 8 when 1.f <= 1.75 and x - 7 otherwise.
__device__ __forceinline__ uint32_t block_scale(uint32_t top)
{
    if (top >= 0x7f800000u) return 255u;
    if (top == 0u) return 127u;
    const int e = static_cast<int>(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    return static_cast<uint32_t>(max(e, 0));
}

// 2^-e of a scale byte (NaN for the NaN scale): the scales above have e <= 120, so 2^-e is a normal number.
__device__ __forceinline__ float inverse_scale(uint32_t s)
{
    return s == 255u ? __uint_as_float(0x7fffffffu) : __uint_as_float((254u - s) << 23);
}

__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d)
{
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}

// Eight values of a block with this scale as e4m3 bytes; n of them are written.  VEC as above, and 8-byte alignment.
template <bool VEC>
__device__ __forceinline__ void store_q8(uint8_t* dst, const float (&f)[8], uint32_t s, int n)
{
    const float inv = inverse_scale(s);
    uint2 w;
    w.x = pack_e4m3(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
    w.y = pack_e4m3(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv);
    if constexpr (VEC) {
        if (n > 0) *reinterpret_cast<uint2*>(dst) = w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) dst[i] = static_cast<uint8_t>((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
    }
}

__device__ __forceinline__ uint32_t top_of(const float (&f)[8])
{
    uint32_t t = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) t = max(t, abs_bits(f[i]));
    return t;
}

// The largest value over the 16 lanes that share a block of 128.
__device__ __forceinline__ uint32_t top_of_16_lanes(uint32_t t)
{
#pragma unroll
    for (int d = 8; d >= 1; d >>= 1) t = max(t, __shfl_xor_sync(0xffffffffu, t, d));
    return t;
}

// ------------------------------------------------------------------------------------------
// Quantization
// ------------------------------------------------------------------------------------------
struct QuantParams {
    const void* x;
    uint8_t* q;
    uint8_t* scale;
    long long rows, ldx, ldq, lds;
    int cols, blocks;  // blocks of 128 in a row
};

// Blocks of 128 of one row: 16 lanes hold one block, 8 values each; UNROLL blocks at a time, so that as many loads are in
// flight, and on over the whole matrix.
template <typename T, bool VEC, int UNROLL>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantParams p)
{
    const int sub = threadIdx.x & 15;
    const long long step = static_cast<long long>(gridDim.x) * 16;
    const long long first = static_cast<long long>(blockIdx.x) * 16 + (threadIdx.x >> 4);
    const long long total = p.rows * p.blocks;
    const long long drow = step / p.blocks;
    const int dblk = static_cast<int>(step % p.blocks);
    long long row = first / p.blocks;
    int blk = static_cast<int>(first % p.blocks);
    const T* x = static_cast<const T*>(p.x);
    // a warp's two halves leave the loop together: the shuffles below need every lane
    for (long long at = first & ~1ll; at < total; at += step * UNROLL) {
        Vec8<T> v[UNROLL];
        long long rows[UNROLL];
        int blks[UNROLL];
#pragma unroll
        for (int j = 0; j < UNROLL; ++j) {
            rows[j] = row;
            blks[j] = blk;
            const int c = blk * 128 + sub * 8;
            const int n = row < p.rows ? p.cols - c : 0;
            v[j] = load8<VEC>(x + (n > 0 ? row * p.ldx + c : 0), n);
            row += drow;
            blk += dblk;
            if (blk >= p.blocks) {
                blk -= p.blocks;
                ++row;
            }
        }
#pragma unroll
        for (int j = 0; j < UNROLL; ++j) {
            const int c = blks[j] * 128 + sub * 8;
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = to_f32(v[j].v[i]);
            const uint32_t s = block_scale(top_of_16_lanes(top_of(f)));
            if (rows[j] >= p.rows) continue;
            store_q8<VEC>(p.q + rows[j] * p.ldq + c, f, s, p.cols - c);
            if (sub == 0) p.scale[rows[j] * p.lds + blks[j]] = static_cast<uint8_t>(s);
        }
    }
}

// One 128 x 128 tile per CTA, held in registers between its maximum and its rounding: 16 lanes per row, 16 rows at a time.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quantize_tiles_kernel(const QuantParams p)
{
    __shared__ uint32_t tops[8];
    const long long tr = blockIdx.x / p.blocks;
    const int blk = static_cast<int>(blockIdx.x % p.blocks);
    const int c = blk * 128 + (threadIdx.x & 15) * 8;
    const long long row0 = tr * 128 + (threadIdx.x >> 4);
    const T* x = static_cast<const T*>(p.x);
    Vec8<T> v[8];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const long long row = row0 + 16 * j;
        const int n = row < p.rows ? p.cols - c : 0;
        v[j] = load8<VEC>(x + (n > 0 ? row * p.ldx + c : 0), n);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, abs_bits(to_f32(v[j].v[i])));
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) top = max(top, tops[w]);
    const uint32_t s = block_scale(top);
    if (threadIdx.x == 0) p.scale[tr * p.lds + blk] = static_cast<uint8_t>(s);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const long long row = row0 + 16 * j;
        if (row >= p.rows) break;
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = to_f32(v[j].v[i]);
        store_q8<VEC>(p.q + row * p.ldq + c, f, s, p.cols - c);
    }
}

// ------------------------------------------------------------------------------------------
// RMS norm
// ------------------------------------------------------------------------------------------
// Sum over the CTA's threads, the same on all of them.  `slots` alternates between calls (one barrier each).
__device__ __forceinline__ float cta_sum(float v, float* slots)
{
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.f;
    for (int w = 0; w < static_cast<int>(blockDim.x) / 32; ++w) t += slots[w];
    return t;
}

struct NormParams {
    const void* x;
    const void* residual;  // may be null: h = x and nothing is written for it
    const void* weight;
    uint8_t* q;
    uint8_t* scale;
    void* h;               // where x + residual goes (null without a residual)
    float* rstd;
    long long ldx, ldr, ldq, lds, ldh;
    int cols;
    float eps;
};

// One row per CTA; thread t holds the vectors of 8 at t, t + blockDim.x, ... (NV of them; NV = 0: any number, read again
// from h for the second pass).  blockDim.x is a multiple of 32, so the 16 lanes of an aligned group hold one block.
// VEC: rows and weight are aligned for 16-byte accesses (q: 8) and cols is a multiple of 8.
template <typename T, int NV, bool VEC>
__global__ void __launch_bounds__(NV == 0 ? 512 : 256) rmsnorm_fp8_kernel(const NormParams p)
{
    __shared__ float slots[16];
    constexpr int kHeld = NV > 0 ? NV : 1;
    const int threads = blockDim.x;
    const long long row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    const T* r = p.residual ? static_cast<const T*>(p.residual) + row * p.ldr : nullptr;
    const T* w = static_cast<const T*>(p.weight);
    T* h = p.residual ? static_cast<T*>(p.h) + row * p.ldh : nullptr;
    const int nv = NV > 0 ? NV : ((p.cols + 127) / 128 * 16 + threads - 1) / threads;

    Vec8<T> held[kHeld], res[kHeld], gain[kHeld];
    float sq = 0.f;
    auto load = [&](int j, int slot) {
        const int c = (threadIdx.x + j * threads) * 8;
        const int n = p.cols - c, o = n > 0 ? c : 0;
        held[slot] = load8<VEC>(x + o, n);
        if (r != nullptr) res[slot] = load8<VEC>(r + o, n);
    };
    auto first_pass = [&](int j, int slot) {
        const int c = (threadIdx.x + j * threads) * 8;
        Vec8<T>& a = held[slot];
        if (r != nullptr) {
#pragma unroll
            for (int i = 0; i < 8; ++i) a.v[i] = from_f32<T>(to_f32(a.v[i]) + to_f32(res[slot].v[i]));
            store8<VEC>(h + c, a, p.cols - c);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float f = to_f32(a.v[i]);
            sq = fmaf(f, f, sq);
        }
    };
    auto load_gain = [&](int j, int slot) {
        const int c = (threadIdx.x + j * threads) * 8;
        gain[slot] = load8<VEC>(w + (c < p.cols ? c : 0), p.cols - c);
    };
    auto second_pass = [&](int j, int slot, float rstd) {
        const int c = (threadIdx.x + j * threads) * 8;
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = to_f32(held[slot].v[i]) * rstd * to_f32(gain[slot].v[i]);
        const uint32_t s = block_scale(top_of_16_lanes(top_of(f)));
        if (c < p.cols) {
            store_q8<VEC>(p.q + row * p.ldq + c, f, s, p.cols - c);
            if ((threadIdx.x & 15) == 0) p.scale[row * p.lds + c / 128] = static_cast<uint8_t>(s);
        }
    };
    if constexpr (NV > 0) {
#pragma unroll
        for (int j = 0; j < NV; ++j) load(j, j);
#pragma unroll
        for (int j = 0; j < NV; ++j) load_gain(j, j);
#pragma unroll
        for (int j = 0; j < NV; ++j) first_pass(j, j);
    } else {
        for (int j = 0; j < nv; ++j) {
            load(j, 0);
            first_pass(j, 0);
        }
    }
    const float total = cta_sum(sq, slots);
    const float rstd = 1.0f / sqrtf(total / static_cast<float>(p.cols) + p.eps);
    if (threadIdx.x == 0) p.rstd[row] = rstd;
    if constexpr (NV > 0) {
#pragma unroll
        for (int j = 0; j < NV; ++j) second_pass(j, j, rstd);
    } else {
        const T* src = r != nullptr ? h : x;  // this thread's own writes
        for (int j = 0; j < nv; ++j) {
            const int c = (threadIdx.x + j * threads) * 8;
            held[0] = load8<VEC>(src + (c < p.cols ? c : 0), p.cols - c);
            load_gain(j, 0);
            second_pass(j, 0, rstd);
        }
    }
}

struct NormBackParams {
    const void* dy;
    const void* h;
    const void* weight;
    const float* rstd;
    const void* dres;  // may be null
    void* dx;
    float* part;       // [gridDim.x][cols] fp32: each CTA's share of dweight
    long long rows, lddy, ldh, lddres, lddx;
    int cols;
    int stages;        // rows in flight (rmsnorm_fp8_backward_kernel)
    unsigned long long timeout_ns;
};

// dx = rstd * (g - xhat * mean(g * xhat)) + dres with g = dy * weight, xhat = h * rstd; dweight = sum over rows of
// dy * xhat.  CTAs walk over the rows.  Here, any alignment and any number of columns: a thread adds its columns' share
// of dweight in its CTA's row of `part` (each element belongs to one thread), and reads a row twice.
template <typename T>
__global__ void __launch_bounds__(512) rmsnorm_fp8_backward_any_kernel(const NormBackParams p)
{
    __shared__ float slots[2][16];
    const T* w = static_cast<const T*>(p.weight);
    float* part = p.part + static_cast<long long>(blockIdx.x) * p.cols;
    for (int c = threadIdx.x; c < p.cols; c += blockDim.x) part[c] = 0.f;
    int turn = 0;
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        const T* dy = static_cast<const T*>(p.dy) + row * p.lddy;
        const T* h = static_cast<const T*>(p.h) + row * p.ldh;
        const T* dres = p.dres ? static_cast<const T*>(p.dres) + row * p.lddres : nullptr;
        T* dx = static_cast<T*>(p.dx) + row * p.lddx;
        const float rstd = p.rstd[row];
        float dot = 0.f;
        for (int c = threadIdx.x; c < p.cols; c += blockDim.x) dot = fmaf(to_f32(dy[c]) * to_f32(w[c]), to_f32(h[c]) * rstd, dot);
        const float mean = cta_sum(dot, slots[turn]) / static_cast<float>(p.cols);
        for (int c = threadIdx.x; c < p.cols; c += blockDim.x) {
            const float dyf = to_f32(dy[c]), xhat = to_f32(h[c]) * rstd;
            float t = rstd * (dyf * to_f32(w[c]) - xhat * mean);
            if (dres != nullptr) t += to_f32(dres[c]);
            dx[c] = from_f32<T>(t);
            part[c] = fmaf(dyf, xhat, part[c]);
        }
    }
}

// The same for aligned rows of at most 512 * 8 * NV columns, a multiple of 8.  One CTA per SM; rows arrive ahead in
// shared memory (one bulk copy per tensor and row, p.stages rows deep), so that memory stays busy through the two passes
// and the barrier of each row; dweight's share stays in registers.
template <typename T, int NV>
__global__ void __launch_bounds__(512, 1) rmsnorm_fp8_backward_kernel(const NormBackParams p)
{
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float slots[2][16];
    __shared__ __align__(8) uint64_t bars[8];
    const int threads = blockDim.x;
    const uint32_t row_bytes = static_cast<uint32_t>(p.cols) * 2, pitch = (row_bytes + 127u) & ~127u;
    const int tensors = p.dres ? 3 : 2;
    auto issue = [&](long long row, int stage) {
        const uint32_t bar = smem_u32(&bars[stage]), dst = smem_u32(smem) + static_cast<uint32_t>(stage) * 3 * pitch;
        mbar_arrive_expect_tx(bar, row_bytes * tensors);
        bulk_load(dst, static_cast<const T*>(p.dy) + row * p.lddy, row_bytes, bar);
        bulk_load(dst + pitch, static_cast<const T*>(p.h) + row * p.ldh, row_bytes, bar);
        if (p.dres) bulk_load(dst + 2 * pitch, static_cast<const T*>(p.dres) + row * p.lddres, row_bytes, bar);
    };
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) mbar_init(smem_u32(&bars[s]), 1);
        fence_mbar_init();
        fence_proxy_async_smem();
        for (int s = 0; s < p.stages; ++s)
            if (blockIdx.x + static_cast<long long>(s) * gridDim.x < p.rows) issue(blockIdx.x + static_cast<long long>(s) * gridDim.x, s);
    }
    const T* w = static_cast<const T*>(p.weight);
    Vec8<T> gain[NV];
    float acc[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (threadIdx.x + j * threads) * 8;
        gain[j] = load8<true>(w + (c < p.cols ? c : 0), p.cols - c);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[j][i] = 0.f;
    }
    __syncthreads();
    int stage = 0, turn = 0;
    uint32_t phase = 0;
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        const float rstd = p.rstd[row];
        if (!mbar_wait(smem_u32(&bars[stage]), phase, p.timeout_ns, kErrWaitProducer, stage)) break;
        const uint8_t* base = smem + static_cast<size_t>(stage) * 3 * pitch;
        Vec8<T> a[NV], b[NV], d[NV];
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (threadIdx.x + j * threads) * 8;
            const int n = p.cols - c, o = n > 0 ? c * 2 : 0;
            a[j] = load8<true>(reinterpret_cast<const T*>(base + o), n);
            b[j] = load8<true>(reinterpret_cast<const T*>(base + pitch + o), n);
            if (p.dres) d[j] = load8<true>(reinterpret_cast<const T*>(base + 2 * pitch + o), n);
        }
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                dot = fmaf(to_f32(a[j].v[i]) * to_f32(gain[j].v[i]), to_f32(b[j].v[i]) * rstd, dot);
        fence_proxy_async_smem();  // this thread has read its part of the stage
        const float mean = cta_sum(dot, slots[turn]) / static_cast<float>(p.cols);
        const long long ahead = row + static_cast<long long>(p.stages) * gridDim.x;
        if (threadIdx.x == 0 && ahead < p.rows) issue(ahead, stage);
        T* dx = static_cast<T*>(p.dx) + row * p.lddx;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (threadIdx.x + j * threads) * 8;
            Vec8<T> o;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float dyf = to_f32(a[j].v[i]), xhat = to_f32(b[j].v[i]) * rstd;
                float t = rstd * (dyf * to_f32(gain[j].v[i]) - xhat * mean);
                if (p.dres) t += to_f32(d[j].v[i]);
                o.v[i] = from_f32<T>(t);
                acc[j][i] = fmaf(dyf, xhat, acc[j][i]);
            }
            store8<true>(dx + c, o, p.cols - c);
        }
        if (++stage == p.stages) {
            stage = 0;
            phase ^= 1u;
        }
    }
    float* part = p.part + static_cast<long long>(blockIdx.x) * p.cols;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (threadIdx.x + j * threads) * 8;
        if (c >= p.cols) continue;
#pragma unroll
        for (int i = 0; i < 8; i += 4)
            *reinterpret_cast<float4*>(part + c + i) = make_float4(acc[j][i], acc[j][i + 1], acc[j][i + 2], acc[j][i + 3]);
    }
}

// dweight[c] = sum of the `parts` rows of part, in row order: 32 columns x 8 groups of rows per CTA.
__global__ void __launch_bounds__(256) norm_weight_grad_kernel(const float* part, int parts, int cols, float* dweight)
{
    __shared__ float sums[8][33];
    const int lane = threadIdx.x & 31, group = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;
    float t = 0.f;
    if (c < cols)
        for (int r = group; r < parts; r += 8) t += part[static_cast<long long>(r) * cols + c];
    sums[group][lane] = t;
    __syncthreads();
    if (group == 0 && c < cols) {
#pragma unroll
        for (int g = 1; g < 8; ++g) t += sums[g][lane];
        dweight[c] = t;
    }
}

}  // namespace vk
