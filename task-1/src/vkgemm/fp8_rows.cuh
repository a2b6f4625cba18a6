// Row-wise kernels of the 8-bit linear layer: quantization to e4m3 with power-of-two block scales, the RMS norm
// that writes its output in that form, and the norm's backward pass.
//
// The 8-bit form.  A block is 128 neighbouring values of a row, or a tile of 128 x 128.  Its scale is the
// smallest 2^e with max|v| <= 448 * 2^e (448 is e4m3's largest value), held as the e8m0 byte e + 127; the
// values are v * 2^-e, rounded once to nearest even.  v * 2^-e is exact in fp32 (or far below e4m3's smallest
// step), so that rounding is the only one, and q * 2^e is exact in bf16 again from e = -124 on and below 2^128 (a block's
// largest value of 248 * 2^120 or more is rounded to that): what reads the 8-bit form later loses nothing more.  A block of
// zeros has scale 1; one that holds an infinity or a NaN has the NaN scale (255) and NaN values, so that it shows.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <type_traits>

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

// Elements i and i + 1 (i even) of a vector in fp32, and back, rounded to nearest.  16-bit elements are taken out of the
// 32-bit registers that hold them two by two.  (One by one, rmsnorm_fp8_kernel took 57 registers for 32 and issued 21
// instructions for an element: 8192 x 4096 bf16 31 us, against 22.9.)
__device__ __forceinline__ float2 two(const Vec8<float>& v, int i) { return make_float2(v.v[i], v.v[i + 1]); }
__device__ __forceinline__ float2 two(const Vec8<__half>& v, int i) { return __half22float2(reinterpret_cast<const __half2*>(v.v)[i / 2]); }
__device__ __forceinline__ float2 two(const Vec8<__nv_bfloat16>& v, int i)
{
    const uint32_t w = reinterpret_cast<const uint32_t*>(v.v)[i / 2];
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ void put_two(Vec8<__half>& v, int i, float2 f) { reinterpret_cast<__half2*>(v.v)[i / 2] = __float22half2_rn(f); }
__device__ __forceinline__ void put_two(Vec8<__nv_bfloat16>& v, int i, float2 f)
{
    reinterpret_cast<__nv_bfloat162*>(v.v)[i / 2] = __float22bfloat162_rn(f);
}

// a + b, each sum rounded once to its type.
template <typename T>
__device__ __forceinline__ Vec8<T> sum8(const Vec8<T>& a, const Vec8<T>& b)
{
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    Vec8<T> r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        reinterpret_cast<T2*>(r.v)[i] = __hadd2_rn(reinterpret_cast<const T2*>(a.v)[i], reinterpret_cast<const T2*>(b.v)[i]);
    return r;
}

// Elements c .. c + 7 of a row that begins at `row` and has `cols` (those it does not have become zeros).
// VEC: rows are 16-byte aligned and cols a multiple of 8; the load is one predicated instruction, and several stay in
// flight together.  Otherwise the two aligned 16-byte units around the elements are loaded and shifted where both lie
// in the row, and single elements at its ends (4001 x 3333 bf16: norm 36 us, against 56 with single elements
// everywhere).
template <bool VEC, typename T>
__device__ __forceinline__ Vec8<T> load8(const T* row, int c, int cols)
{
    Vec8<T> r;
    uint4* d = reinterpret_cast<uint4*>(&r);
    const int n = cols - c;
    const T* src = row + (n > 0 ? c : 0);
    if constexpr (VEC) {
        const uint4* s = reinterpret_cast<const uint4*>(src);
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(r) / 16); ++i) d[i] = n > 0 ? s[i] : make_uint4(0, 0, 0, 0);
        return r;
    }
    const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(src)) & 15u;
    if (sizeof(T) == 2 && ((off == 0 && n >= 8) || (c >= 8 && n >= 16))) {
        const uint4* s = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(src) - off);
        const uint4 lo = s[0], hi = off ? s[1] : make_uint4(0, 0, 0, 0);
        uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        if (off & 8u) {
#pragma unroll
            for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
        }
        if (off & 4u) {
#pragma unroll
            for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
        }
        const uint32_t bits = (off & 2u) * 8;
        *d = make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits),
                        __funnelshift_r(w[3], w[4], bits));
        return r;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = i < n ? src[i] : from_f32<T>(0.f);
    return r;
}

// The same elements back.
template <bool VEC, typename T>
__device__ __forceinline__ void store8(T* row, int c, int cols, const Vec8<T>& r)
{
    const int n = cols - c;
    if (n <= 0) return;
    T* dst = row + c;
    if constexpr (VEC) {
        const uint4* s = reinterpret_cast<const uint4*>(&r);
        uint4* d = reinterpret_cast<uint4*>(dst);
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(r) / 16); ++i) d[i] = s[i];
        return;
    }
    if (sizeof(T) == 2 && n >= 8) {  // as 32-bit pairs, with a single element at both ends when the row begins between two
        const uint4 v = *reinterpret_cast<const uint4*>(&r);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        if ((reinterpret_cast<uintptr_t>(dst) & 2u) == 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) reinterpret_cast<uint32_t*>(dst)[i] = w[i];
        } else {
            dst[0] = r.v[0];
#pragma unroll
            for (int i = 0; i < 3; ++i) *reinterpret_cast<uint32_t*>(dst + 1 + 2 * i) = __funnelshift_r(w[i], w[i + 1], 16);
            dst[7] = r.v[7];
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) dst[i] = r.v[i];
}

// |v| as an integer that orders like the number, NaN above infinity above every finite value.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The e8m0 byte of a block whose largest |v| has these bits.  With |v| = 1.f * 2^x: 448 = 1.75 * 2^8, so e is
// x - 8 when 1.f <= 1.75 and x - 7 otherwise.
__device__ __forceinline__ uint32_t block_scale(uint32_t top)
{
    if (top >= 0x7f800000u) return 255u;
    if (top == 0u) return 127u;
    return static_cast<uint32_t>(max(static_cast<int>((top + 0x1fffffu) >> 23) - 8, 0));  // a fraction above .75 carries
}

// 2^-e of a scale byte (NaN for the NaN scale): the scales above have e <= 120, so 2^-e is a normal number.
__device__ __forceinline__ float inverse_scale(uint32_t s)
{
    return s == 255u ? __uint_as_float(0x7fffffffu) : __uint_as_float((254u - s) << 23);
}

__device__ __forceinline__ uint32_t pack_e4m3(float2 a, float2 b)
{
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}

// Eight values of a block with this scale as e4m3 bytes; n of them are written.  VEC: 8 or none, and 8-byte aligned.
template <bool VEC>
__device__ __forceinline__ void store_q8(uint8_t* dst, const float (&f)[8], uint32_t s, int n)
{
    const float inv = inverse_scale(s);
    uint2 w;
    w.x = pack_e4m3(__fmul2_rn(make_float2(f[0], f[1]), make_float2(inv, inv)), __fmul2_rn(make_float2(f[2], f[3]), make_float2(inv, inv)));
    w.y = pack_e4m3(__fmul2_rn(make_float2(f[4], f[5]), make_float2(inv, inv)), __fmul2_rn(make_float2(f[6], f[7]), make_float2(inv, inv)));
    if (VEC ? n > 0 : n >= 8 && (reinterpret_cast<uintptr_t>(dst) & 7u) == 0) {
        *reinterpret_cast<uint2*>(dst) = w;
    } else if (!VEC) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) dst[i] = static_cast<uint8_t>((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
    }
}

__device__ __forceinline__ uint32_t top_of(const float (&f)[8])
{
    float t = f[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) asm("max.NaN.xorsign.abs.f32 %0, %0, %1;" : "+f"(t) : "f"(f[i]));
    return abs_bits(t);
}

// The same of eight stored values.  16-bit ones are compared two at a time, as integers that order like the numbers.
__device__ __forceinline__ uint32_t top_of(const Vec8<float>& v) { return top_of(v.v); }

template <typename T>
__device__ __forceinline__ uint32_t top_of(const Vec8<T>& v)
{
    const uint4 w = *reinterpret_cast<const uint4*>(&v);
    constexpr uint32_t kAbs = 0x7fff7fffu;
    const uint32_t t = __vmaxu2(__vmaxu2(w.x & kAbs, w.y & kAbs), __vmaxu2(w.z & kAbs, w.w & kAbs));
    const uint16_t top = static_cast<uint16_t>(max(t & 0xffffu, t >> 16));
    return abs_bits(to_f32(*reinterpret_cast<const T*>(&top)));
}

// The largest value over the 16 lanes that share a block of 128.
__device__ __forceinline__ uint32_t top_of_16_lanes(uint32_t t)
{
#pragma unroll
    for (int d = 8; d >= 1; d >>= 1) t = max(t, __shfl_xor_sync(0xffffffffu, t, d));
    return t;
}

// Scales of N (2 or 4) blocks of a row from block `blk`, of which the row has `blocks`; one store where it can be.
template <int N>
__device__ __forceinline__ void put_scales(uint8_t* row, int blk, int blocks, uint32_t scales)
{
    uint8_t* out = row + blk;
    if (blk + N <= blocks && (reinterpret_cast<uintptr_t>(out) & (N - 1)) == 0) {
        if constexpr (N == 4)
            *reinterpret_cast<uint32_t*>(out) = scales;
        else
            *reinterpret_cast<uint16_t*>(out) = static_cast<uint16_t>(scales);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (blk + j < blocks) out[j] = static_cast<uint8_t>(scales >> (8 * j));
    }
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

// Rows: 16 lanes hold one block, 8 values each, and have four neighbouring blocks of a row, so that four loads are in
// flight and the four scales leave in one store.  16 such quads to a CTA.  Bound by memory: 8192 x 8192 bf16 31.5 us, 6.4 TB/s
// (blocks one by one, a grid apart: 45 us); 8192 x 4096 fp32 26.6 us, 6.3 TB/s.  Rows at any alignment: 4001 x 3333 15.3 us, 2.6 TB/s.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantParams p)
{
    const int sub = threadIdx.x & 15;
    const int quads = (p.blocks + 3) / 4;
    const long long item = static_cast<long long>(blockIdx.x) * 16;
    const unsigned in = static_cast<unsigned>(item % quads) + (threadIdx.x >> 4);
    const long long row = item / quads + in / quads;
    const int blk = static_cast<int>(in % quads) * 4;
    const int c = blk * 128 + sub * 8;
    const int cols = row < p.rows ? p.cols : 0, left = cols - c;
    const T* x = static_cast<const T*>(p.x) + (left > 0 ? row * p.ldx : 0);
    Vec8<T> v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = load8<VEC>(x, c + 128 * j, cols);
    uint32_t scales = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t s = block_scale(top_of_16_lanes(top_of(v[j])));
        scales |= s << (8 * j);
        if (left <= 128 * j) continue;
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const float2 t = two(v[j], i);
            f[i] = t.x;
            f[i + 1] = t.y;
        }
        store_q8<VEC>(p.q + row * p.ldq + c + 128 * j, f, s, left - 128 * j);
    }
    if (sub == 0 && left > 0) put_scales<4>(p.scale + row * p.lds, blk, p.blocks, scales);
}

// One 128 x 128 tile per CTA, held in registers between its maximum and its rounding: 16 lanes per row, 16 rows at a time.
// Bound by memory: 16384 x 4096 bf16 31 us, 6.5 TB/s; 8192 x 4096 fp32 30.2 us, 5.6 TB/s.  Rows at any alignment: 4001 x 3333 16.0 us.
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
        const bool in = row < p.rows;
        v[j] = load8<VEC>(x + (in ? row * p.ldx : 0), c, in ? p.cols : 0);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, top_of(v[j]));
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
        for (int i = 0; i < 8; i += 2) {
            const float2 t = two(v[j], i);
            f[i] = t.x;
            f[i + 1] = t.y;
        }
        store_q8<VEC>(p.q + row * p.ldq + c, f, s, p.cols - c);
    }
}

// ------------------------------------------------------------------------------------------
// RMS norm
// ------------------------------------------------------------------------------------------
// Sum over the CTA's threads (16 warps at most), the same on all of them.
// `slots` alternates between calls (one barrier each).
__device__ __forceinline__ float cta_sum(float v, float* slots)
{
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
    __syncthreads();
    const int from = threadIdx.x & 15;
    v = from < static_cast<int>(blockDim.x) / 32 ? slots[from] : 0.f;
#pragma unroll
    for (int d = 8; d >= 1; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
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
    float eps, inv_cols;  // 1 / cols
};

// The second pass over a row: a warp's 2 NV neighbouring blocks of y in 8 bits.
template <typename T, int NV, bool VEC>
__device__ __forceinline__ void norm_row_out(const NormParams& p, long long row, int first, const Vec8<T> (&held)[NV], const Vec8<T> (&gain)[NV], float rstd)
{
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t scales[(NV + 1) / 2] = {};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (first + j * 32) * 8;
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const float2 y = __fmul2_rn(__fmul2_rn(two(held[j], i), make_float2(rstd, rstd)), two(gain[j], i));
            f[i] = y.x;
            f[i + 1] = y.y;
        }
        const uint32_t s = block_scale(top_of_16_lanes(top_of(f)));
        store_q8<VEC>(p.q + row * p.ldq + c, f, s, p.cols - c);
        scales[j / 2] |= (s | __shfl_down_sync(0xffffffffu, s, 16) << 8) << (16 * (j & 1));
    }
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < (NV + 1) / 2; ++i)
            put_scales<NV == 1 ? 2 : 4>(p.scale + row * p.lds, warp * 2 * NV + 4 * i, (p.cols + 127) / 128, scales[i]);
    }
}

// One row per CTA, held in registers between its two passes; a warp has 32 NV neighbouring vectors of 8, 2 NV blocks, and
// stores their scales at once (a byte at a time costs memory more than the row's values do).  VEC: rows and weight are
// aligned for 16-byte accesses (q: 8) and cols is a multiple of 8.  Bound by memory: 4001 x 5120 fp16 with a residual
// 20.9 us, 6.9 TB/s (part of it from L2); 8192 x 8192 bf16 70.3 us, 6.7 TB/s; without a residual by the instructions of
// the second pass, which fewer bytes hide (issue slots 69 % busy with 89 % of the warps there, 18.4 instructions for an
// element): 8192 x 4096 22.5 us, 4.5 TB/s; 4096 x 12288 39.6 us, 3.8 TB/s.  Rows at any alignment hold 57 registers for 32, so
// that 41 % of the warps are there and wait for memory: 4001 x 3333 35.8 us, 2.6 TB/s.  (CTAs that walk over rows, which arrive
// ahead in shared memory by bulk copies: 24.3, 85.6 and 26.0 us.)
template <typename T, int NV, bool VEC>
__global__ void __launch_bounds__(NV == 1 ? 256 : 512) rmsnorm_fp8_kernel(const NormParams p)
{
    __shared__ float slots[16];
    const int first = (threadIdx.x >> 5) * 32 * NV + (threadIdx.x & 31);
    const long long row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    const T* r = static_cast<const T*>(p.residual) + row * p.ldr;
    const T* w = static_cast<const T*>(p.weight);
    Vec8<T> held[NV], res[NV], gain[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (first + j * 32) * 8;
        held[j] = load8<VEC>(x, c, p.cols);
        if (p.residual != nullptr) res[j] = load8<VEC>(r, c, p.cols);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) gain[j] = load8<VEC>(w, (first + j * 32) * 8, p.cols);
    float2 sq = make_float2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (first + j * 32) * 8;
        if (p.residual != nullptr) {
            held[j] = sum8(held[j], res[j]);
            store8<VEC>(static_cast<T*>(p.h) + row * p.ldh, c, p.cols, held[j]);
        }
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const float2 f = two(held[j], i);
            sq = __ffma2_rn(f, f, sq);
        }
    }
    const float total = cta_sum(sq.x + sq.y, slots);
    const float rstd = rsqrtf(fmaf(total, p.inv_cols, p.eps));
    if (threadIdx.x == 0) p.rstd[row] = rstd;
    norm_row_out<T, NV, VEC>(p, row, first, held, gain, rstd);
}

// The same for any number of columns: h (or x) is read again for the second pass, from L2 (2000 x 16384 with a residual
// 45.4 us, 5.1 TB/s; held in registers 37.0).
template <typename T, bool VEC>
__global__ void __launch_bounds__(512) rmsnorm_fp8_long_kernel(const NormParams p)
{
    __shared__ float slots[16];
    const long long row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    const T* r = static_cast<const T*>(p.residual) + row * p.ldr;
    const T* w = static_cast<const T*>(p.weight);
    T* h = static_cast<T*>(p.h) + row * p.ldh;
    const int nv = ((p.cols + 127) / 128 * 16 + 511) / 512;
    float sq = 0.f;
    for (int j = 0; j < nv; ++j) {
        const int c = (threadIdx.x + j * 512) * 8;
        Vec8<T> a = load8<VEC>(x, c, p.cols);
        if (p.residual != nullptr) {
            const Vec8<T> b = load8<VEC>(r, c, p.cols);
#pragma unroll
            for (int i = 0; i < 8; ++i) a.v[i] = from_f32<T>(to_f32(a.v[i]) + to_f32(b.v[i]));
            store8<VEC>(h, c, p.cols, a);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float f = to_f32(a.v[i]);
            sq = fmaf(f, f, sq);
        }
    }
    const float total = cta_sum(sq, slots);
    const float rstd = rsqrtf(fmaf(total, p.inv_cols, p.eps));
    if (threadIdx.x == 0) p.rstd[row] = rstd;
    const T* src = p.residual != nullptr ? h : x;  // this thread's own writes
    for (int j = 0; j < nv; ++j) {
        const int c = (threadIdx.x + j * 512) * 8, n = p.cols - c;
        const Vec8<T> a = load8<VEC>(src, c, p.cols), gain = load8<VEC>(w, c, p.cols);
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = to_f32(a.v[i]) * rstd * to_f32(gain.v[i]);
        const uint32_t s = block_scale(top_of_16_lanes(top_of(f)));
        if (n > 0) {
            store_q8<VEC>(p.q + row * p.ldq + c, f, s, n);
            if ((threadIdx.x & 15) == 0) p.scale[row * p.lds + c / 128] = static_cast<uint8_t>(s);
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
    float inv_cols;    // 1 / cols
    int stages;        // rows in flight (rmsnorm_fp8_backward_kernel)
    unsigned long long timeout_ns;
};

// dx = rstd * (g - xhat * mean(g * xhat)) + dres with g = dy * weight, xhat = h * rstd; dweight = sum over rows of
// dy * xhat.  CTAs walk over the rows.  Here, any number of columns: a thread adds its columns' share
// of dweight in its CTA's row of `part` (each element belongs to one thread), and reads a row twice, one 16-bit element at a time.
// Far from memory's rate: 4096 x 12288 bf16 with dres 799 us, 0.5 TB/s; 2000 x 16384 531.  It runs for rows over 8192 wide only.
template <typename T>
__global__ void __launch_bounds__(512) rmsnorm_fp8_backward_any_kernel(const NormBackParams p)
{
    __shared__ float slots[2][16];
    const T* w = static_cast<const T*>(p.weight);
    float* part = p.part + static_cast<long long>(blockIdx.x) * p.cols;
    // (unsigned: a thread's last column and blockDim.x add up to more than an int where cols is near its end)
    const unsigned cols = static_cast<unsigned>(p.cols);
    for (unsigned c = threadIdx.x; c < cols; c += blockDim.x) part[c] = 0.f;
    int turn = 0;
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        const T* dy = static_cast<const T*>(p.dy) + row * p.lddy;
        const T* h = static_cast<const T*>(p.h) + row * p.ldh;
        const T* dres = p.dres ? static_cast<const T*>(p.dres) + row * p.lddres : nullptr;
        T* dx = static_cast<T*>(p.dx) + row * p.lddx;
        const float rstd = p.rstd[row];
        float dot = 0.f;
        for (unsigned c = threadIdx.x; c < cols; c += blockDim.x) dot = fmaf(to_f32(dy[c]) * to_f32(w[c]), to_f32(h[c]) * rstd, dot);
        const float mean = cta_sum(dot, slots[turn]) * p.inv_cols;
        for (unsigned c = threadIdx.x; c < cols; c += blockDim.x) {
            const float dyf = to_f32(dy[c]), xhat = to_f32(h[c]) * rstd;
            float t = rstd * (dyf * to_f32(w[c]) - xhat * mean);
            if (dres != nullptr) t += to_f32(dres[c]);
            dx[c] = from_f32<T>(t);
            part[c] = fmaf(dyf, xhat, part[c]);
        }
    }
}

// The same for rows of at most 512 * 8 * NV columns; dweight's share stays in registers.  VEC (16-byte aligned rows, a
// multiple of 8 columns): rows arrive ahead in shared memory, one bulk copy per tensor and row, p.stages rows deep, so
// that memory stays busy through the two passes and the barrier of each row: 8192 x 8192 bf16 with dres 85.8 us, 6.3 TB/s.
// Narrower rows wait more at their barrier for each byte: 4096 x 4096 27.7 us, 4.9 TB/s; 8000 x 1000 18.7 us, 3.4 TB/s, 15 of them
// here (issue slots 41 % busy, a warp's waits about even between the barrier and memory) and the rest in the sum of 1184 partial rows.
// Otherwise from memory as they are needed (4001 x 3333: 61 us).
template <typename T, int NV, bool VEC>
__global__ void __launch_bounds__(512, NV == 1 ? 2 : 1) rmsnorm_fp8_backward_kernel(const NormBackParams p)
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
    if (VEC && threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) mbar_init(smem_u32(&bars[s]), 1);
        fence_mbar_init();
        fence_proxy_async_smem();
        for (int s = 0; s < p.stages; ++s)
            if (blockIdx.x + static_cast<long long>(s) * gridDim.x < p.rows) issue(blockIdx.x + static_cast<long long>(s) * gridDim.x, s);
    }
    const T* w = static_cast<const T*>(p.weight);
    Vec8<T> gain[NV];
    float2 acc[NV][4];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (threadIdx.x + j * threads) * 8;
        gain[j] = load8<VEC>(w, c, p.cols);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] = make_float2(0.f, 0.f);
    }
    __syncthreads();
    int stage = 0, before = p.stages - 1, turn = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        const float rstd = p.rstd[row];
        // A thread whose wait gives up goes on with whatever lies there: the others may not have, and count on it at the barrier.
        if (VEC && ok) ok = mbar_wait(smem_u32(&bars[stage]), phase, p.timeout_ns, kErrWaitProducer, stage);
        const uint8_t* base = smem + static_cast<size_t>(stage) * 3 * pitch;
        const T* dy = VEC ? reinterpret_cast<const T*>(base) : static_cast<const T*>(p.dy) + row * p.lddy;
        const T* h = VEC ? reinterpret_cast<const T*>(base + pitch) : static_cast<const T*>(p.h) + row * p.ldh;
        const T* dres = VEC ? reinterpret_cast<const T*>(base + 2 * pitch) : static_cast<const T*>(p.dres) + row * p.lddres;
        Vec8<T> a[NV], b[NV], d[NV];
        float2 dot = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (threadIdx.x + j * threads) * 8;
            a[j] = load8<VEC>(dy, c, p.cols);
            b[j] = load8<VEC>(h, c, p.cols);
            if (!VEC && p.dres) d[j] = load8<VEC>(dres, c, p.cols);
#pragma unroll
            for (int i = 0; i < 8; i += 2) dot = __ffma2_rn(__fmul2_rn(two(a[j], i), two(gain[j], i)), __fmul2_rn(two(b[j], i), make_float2(rstd, rstd)), dot);
        }
        const float mean = cta_sum(dot.x + dot.y, slots[turn]) * p.inv_cols;
        // Behind this barrier no thread reads the row before any more: its stage is free.
        const long long ahead = row + static_cast<long long>(p.stages - 1) * gridDim.x;
        if (VEC && threadIdx.x == 0 && ok && row != blockIdx.x && ahead < p.rows) issue(ahead, before);
        T* dx = static_cast<T*>(p.dx) + row * p.lddx;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (threadIdx.x + j * threads) * 8;
            if (VEC && p.dres) d[j] = load8<VEC>(dres, c, p.cols);
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const float2 dyf = two(a[j], i), xhat = __fmul2_rn(two(b[j], i), make_float2(rstd, rstd));
                const float2 g = __ffma2_rn(xhat, make_float2(-mean, -mean), __fmul2_rn(dyf, two(gain[j], i)));
                const float2 rest = p.dres ? two(d[j], i) : make_float2(0.f, 0.f);
                put_two(d[j], i, __ffma2_rn(make_float2(rstd, rstd), g, rest));
                acc[j][i / 2] = __ffma2_rn(dyf, xhat, acc[j][i / 2]);
            }
            store8<VEC>(dx, c, p.cols, d[j]);
        }
        if (VEC) fence_proxy_async_smem();  // read before the stage is written again
        before = stage;
        if (++stage == p.stages) {
            stage = 0;
            phase ^= 1u;
        }
    }
    if (VEC && threadIdx.x == 0 && !ok) settle();
    float* part = p.part + static_cast<long long>(blockIdx.x) * p.cols;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (threadIdx.x + j * threads) * 8;
        if (c >= p.cols) continue;
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < 8; i += 4)
                *reinterpret_cast<float4*>(part + c + i) = make_float4(acc[j][i / 2].x, acc[j][i / 2].y, acc[j][i / 2 + 1].x, acc[j][i / 2 + 1].y);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < p.cols) part[c + i] = i & 1 ? acc[j][i / 2].y : acc[j][i / 2].x;
        }
    }
}

// dweight[c] = sum of the `parts` rows of part: 32 columns x 32 groups of rows per CTA.
__global__ void __launch_bounds__(1024) norm_weight_grad_kernel(const float* part, int parts, int cols, float* dweight)
{
    __shared__ float sums[32][33];
    const int lane = threadIdx.x & 31, group = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;
    float t = 0.f;
    if (c < cols) {
#pragma unroll 4
        for (int r = group; r < parts; r += 32) t += part[static_cast<long long>(r) * cols + c];
    }
    sums[group][lane] = t;
    __syncthreads();
    t = sums[lane][group];  // column `group` of this CTA
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
    if (lane == 0 && blockIdx.x * 32 + group < cols) dweight[blockIdx.x * 32 + group] = t;
}

}  // namespace vk
