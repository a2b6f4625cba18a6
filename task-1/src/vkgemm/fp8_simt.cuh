// CUDA-core products of 8-bit operands: any strides, alignment and layout (what the tensor-core kernels' TMA
// loads cannot describe), fp32 accumulation in the order of the contraction.  Bound by the CUDA cores; a fallback that
// is not tuned further.
#pragma once

#include <type_traits>

#include "fp8_rows.cuh"

namespace vk {

__device__ __forceinline__ float e4m3_to_f32(uint8_t v)
{
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(v, __NV_E4M3)));
}

__device__ __forceinline__ float e8m0_to_f32(uint8_t s)
{
    // 2^(s - 127); 2^-127 is a subnormal number
    return s == 255u ? __uint_as_float(0x7fffffffu) : s == 0u ? __uint_as_float(0x400000u) : __uint_as_float(static_cast<uint32_t>(s) << 23);
}

// Element (i, t) of an 8-bit operand: i the output's index, t the contraction's.  Strides in elements of q and of
// scale; shifts say how many neighbours share a scale (7 = 128, 0 = one).
struct F8Operand {
    const uint8_t* q;
    const uint8_t* scale;
    long long qi, qt, si, st;
    int shift_i, shift_t;
    __device__ __forceinline__ float at(long long i, long long t) const
    {
        return e4m3_to_f32(q[i * qi + t * qt]) * e8m0_to_f32(scale[(i >> shift_i) * si + (t >> shift_t) * st]);
    }
};

// The same with each value rounded to the type of the operand it meets: exact in bf16 (see fp8_rows.cuh), within
// fp16's finite range.
template <typename T>
struct F8OperandAs {
    F8Operand f;
    __device__ __forceinline__ float at(long long i, long long t) const
    {
        float v = f.at(i, t);
        if constexpr (std::is_same_v<T, __half>)
            v = v > 65504.f ? 65504.f : v < -65504.f ? -65504.f : v;  // keeps NaN
        return to_f32(from_f32<T>(v));
    }
};

// The same for a 16-bit operand.
template <typename T>
struct HalfOperand {
    const T* p;
    long long pi, pt;
    __device__ __forceinline__ float at(long long i, long long t) const { return to_f32(p[i * pi + t * pt]); }
};

struct F8Output {
    void* c;
    long long ld;
    int kind;        // vk_dtype
    int accumulate;  // C += the product
};

__device__ __forceinline__ void put_output(const F8Output& o, long long row, long long col, float v)
{
    const long long at = row * o.ld + col;
    if (o.kind == 0) {
        __half* c = static_cast<__half*>(o.c) + at;
        *c = from_f32<__half>(o.accumulate ? v + to_f32(*c) : v);
    } else if (o.kind == 2) {
        __nv_bfloat16* c = static_cast<__nv_bfloat16*>(o.c) + at;
        *c = from_f32<__nv_bfloat16>(o.accumulate ? v + to_f32(*c) : v);
    } else {
        float* c = static_cast<float*>(o.c) + at;
        *c = o.accumulate ? v + *c : v;
    }
}

// C[i][j] = sum over t of a(i, t) * b(j, t): 64 x 64 tile, 256 threads of 4 x 4 outputs, 16 steps of t at a time.  A grid has
// at most 65535 rows of CTAs, so a CTA walks over tile rows.
template <typename LA, typename LB>
__global__ void __launch_bounds__(256) fp8_simt_kernel(const LA a, const LB b, const F8Output out, long long M, long long N, long long K)
{
    __shared__ float sa[16][65], sb[16][65];
    const long long j0 = static_cast<long long>(blockIdx.x) * 64;
    const int ti = threadIdx.x >> 4, tj = threadIdx.x & 15;
    for (long long i0 = static_cast<long long>(blockIdx.y) * 64; i0 < M; i0 += static_cast<long long>(gridDim.y) * 64) {
        float acc[4][4] = {};
        for (long long t0 = 0; t0 < K; t0 += 16) {
#pragma unroll
            for (int e = threadIdx.x; e < 1024; e += 256) {
                const int t = e & 15, i = e >> 4;
                sa[t][i] = (i0 + i < M && t0 + t < K) ? a.at(i0 + i, t0 + t) : 0.f;
                sb[t][i] = (j0 + i < N && t0 + t < K) ? b.at(j0 + i, t0 + t) : 0.f;
            }
            __syncthreads();
#pragma unroll
            for (int t = 0; t < 16; ++t)
#pragma unroll
                for (int y = 0; y < 4; ++y)
#pragma unroll
                    for (int x = 0; x < 4; ++x) acc[y][x] = fmaf(sa[t][ti + 16 * y], sb[t][tj + 16 * x], acc[y][x]);
            __syncthreads();
        }
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const long long i = i0 + ti + 16 * y, j = j0 + tj + 16 * x;
                if (i < M && j < N) put_output(out, i, j, acc[y][x]);
            }
    }
}

}  // namespace vk
