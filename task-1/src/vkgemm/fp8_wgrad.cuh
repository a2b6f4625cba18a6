// dW = dY^T * X on the tensor cores of sm_100a: dY in 16 bits, X as the forward pass kept it, e4m3 with a power-of-two
// scale for each token and 128 columns.
//
// X's scale changes along the sum (the tokens), so neither the tensor core's block scales nor the epilogue can apply
// it, and one MMA takes both operands in the same type.  Four warps therefore turn each stage of X into dY's type on
// its way from TMA to the MMAs, inside shared memory: q * 2^e is exact in bf16, and the product is that of the 16-bit
// kernel.  X costs half the bytes of a 16-bit checkpoint in memory and on the way into the SM.
//
// Roles (448 threads per CTA, pairs of CTAs on one 256 x 256 tile, 64 tokens a stage):
//   warp 0      TMA loads: dY (128 of the tile's rows, M-major) and X's bytes (this CTA's 128 columns).
//   warp 1      tensor memory, and in the pair's leader the MMAs (one lane).
//   warps 2..5  epilogue: tensor memory -> registers -> swizzled staging -> TMA stores.
//   warps 6..13 X's bytes -> 16-bit values in the 128-byte swizzled layout of an N-major operand; four warps to a stage.
//
// A tile's tokens can be split over the pairs of a larger cluster (p.slices): each pair sums its share, leaves it in its
// own shared memory, and adds its part of the columns from all of them in slice order.
#pragma once

#include "fp8_gemm.cuh"

namespace vk {

struct WgradParams {
    int M, N, K;  // rows and columns of dW, tokens
    int tiles_m, tiles_n, num_st;
    int raster_group;
    int slices;   // pairs of CTAs per cluster, each with its share of the tokens
    const uint8_t* scale;
    long long lds;
    void* C;
    long long ldc;
    int c_tma, c_vec, accumulate;
    unsigned long long timeout_ns;
};

constexpr int kWgStages = 5;
constexpr int kWgBK = 64;
constexpr int kWgABytes = 128 * kWgBK * 2;
constexpr int kWgRawBytes = 128 * kWgBK;
constexpr int kWgBBytes = 128 * kWgBK * 2;
constexpr int kWgStageBytes = kWgABytes + kWgRawBytes + kWgBBytes;
constexpr int kWgBars = 4 * kWgStages + 4;
constexpr int kWgSmemBytes = 1024 + kWgStages * kWgStageBytes + 4 * kF8EpiWarpBytes + kWgBars * 8 + 16;
constexpr int kWgGroups = 2;  // of four conversion warps, taking turns at the stages
constexpr int kWgThreads = 192 + 128 * kWgGroups;
static_assert(kWgSmemBytes <= 232448, "shared memory per CTA");
static_assert(kWgStages * kWgStageBytes >= 128 * 256 * 4, "a slice's partial sums fit the stages");

template <typename T>
__device__ __forceinline__ uint32_t scaled_pair(uint32_t two, float scale)
{
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two), __NV_E4M3);
    const float2 f = __half22float2(__half2(h));
    if constexpr (std::is_same_v<T, __half>) {
        // within fp16's finite numbers, NaN kept
        const __half2 most = __float2half2_rn(65504.f);
        const __half2 v = __hmax2_nan(__hmin2_nan(__floats2half2_rn(f.x * scale, f.y * scale), most), __hneg2(most));
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __nv_bfloat162 v = __floats2bfloat162_rn(f.x * scale, f.y * scale);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}

__device__ __forceinline__ float e8m0_scale(uint32_t s)
{
    return s == 255u ? __uint_as_float(0x7fffffffu) : s == 0u ? __uint_as_float(0x400000u) : __uint_as_float(s << 23);
}

// f += C of this lane's row.
template <int OUT>
__device__ __forceinline__ void add_box(const BoxOut& o, int c_vec, int row, int col, float (&f)[32])
{
    using T = std::conditional_t<OUT == 0, __half, std::conditional_t<OUT == 1, float, __nv_bfloat16>>;
    if (row >= o.M) return;
    const T* c = static_cast<const T*>(o.C) + static_cast<long long>(row) * o.ldc + col;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const Vec8<T> v = load8(c + (col + 8 * j < o.N ? 8 * j : 0), o.N - col - 8 * j, c_vec);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[8 * j + i] += to_f32(v.v[i]);
    }
}

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr)
{
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

// T: dY's type; OUT: vk_dtype of dW.
template <typename T, int OUT>
__global__ void __launch_bounds__(kWgThreads, 1)
    wgrad_fp8_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                     const __grid_constant__ CUtensorMap tmap_c, const WgradParams p)
{
#if defined(__CUDA_ARCH__) && (__CUDA_ARCH__ >= 1000)
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sA = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sB = sA + kWgStages * kWgABytes;
    uint8_t* sX = sB + kWgStages * kWgBBytes;
    uint8_t* epi = sX + kWgStages * kWgRawBytes;
    uint64_t* bars = reinterpret_cast<uint64_t*>(epi + 4 * kF8EpiWarpBytes);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kWgBars);

    const uint32_t bar0 = smem_u32(bars);
    auto full_bar = [&](int s) { return bar0 + 8u * s; };
    auto empty_bar = [&](int s) { return bar0 + 8u * (kWgStages + s); };
    auto x_bar = [&](int s) { return bar0 + 8u * (2 * kWgStages + s); };
    auto ready_bar = [&](int s) { return bar0 + 8u * (3 * kWgStages + s); };
    auto tfull_bar = [&](int a) { return bar0 + 8u * (4 * kWgStages + a); };
    auto tempty_bar = [&](int a) { return bar0 + 8u * (4 * kWgStages + 2 + a); };

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const uint32_t lead = rank & ~1u;        // the pair's leader
    const int half = static_cast<int>(rank & 1u);
    const int slice = static_cast<int>(rank >> 1);
    const int cluster_id = blockIdx.x / (2 * p.slices);
    const int num_clusters = gridDim.x / (2 * p.slices);
    const int tiles = p.tiles_m * p.tiles_n;
    const int st0 = static_cast<int>(static_cast<long long>(p.num_st) * slice / p.slices);
    const int st1 = static_cast<int>(static_cast<long long>(p.num_st) * (slice + 1) / p.slices);

    if (warp == 0 && lane == 0) {
        prefetch_tmap(&tmap_a);
        prefetch_tmap(&tmap_b);
        if (p.c_tma) prefetch_tmap(&tmap_c);
        for (int s = 0; s < kWgStages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
            mbar_init(x_bar(s), 1);
            mbar_init(ready_bar(s), 8);  // the conversion warps of both CTAs
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(tfull_bar(a), 1);
            mbar_init(tempty_bar(a), 8);  // the epilogue warps of both CTAs
        }
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc<2>(smem_u32(tmem_slot), 512);
        tmem_relinquish<2>();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int t = cluster_id; ok && t < tiles; t += num_clusters) {
                int tm, tn;
                f8_tile_coords(t, p.tiles_m, p.tiles_n, p.raster_group, tm, tn);
                const int m0 = tm * 256 + half * 128;
                const int n0 = tn * 256 + half * 128;
                for (int st = st0; st < st1; ++st) {
                    if (!mbar_wait(empty_bar(stage), phase ^ 1u, p.timeout_ns, kErrWaitProducer, stage)) {
                        ok = false;
                        break;
                    }
                    const int k0 = st * kWgBK;
                    mbar_arrive_expect_tx(x_bar(stage), kWgRawBytes);
                    tma_load_2d(smem_u32(sX + stage * kWgRawBytes), &tmap_b, x_bar(stage), n0, k0);
                    if (half == 0) mbar_arrive_expect_tx(full_bar(stage), 2 * kWgABytes);
                    const uint32_t bar = mapa_shared(full_bar(stage), lead);
                    const uint32_t a_dst = smem_u32(sA + stage * kWgABytes);
                    tma_load_2d_pair(a_dst, &tmap_a, bar, m0, k0);
                    tma_load_2d_pair(a_dst + 64 * kWgBK * 2, &tmap_a, bar, m0 + 64, k0);
                    if (++stage == kWgStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            for (int i = 0; ok && i < kWgStages; ++i) {
                if (!mbar_wait(empty_bar(stage), phase ^ 1u, p.timeout_ns, kErrWaitTail, stage)) break;
                if (++stage == kWgStages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
    } else if (warp == 1) {
        if (half == 0 && lane == 0) {
            constexpr uint32_t kType = std::is_same_v<T, __half> ? 0u : 1u;
            // D fp32, A and B of T, A M-major, B N-major
            constexpr uint32_t kIdesc = idesc_f16(256, 256, true, true) | (1u << 15) | (kType << 7) | (kType << 10);
            int stage = 0, it = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int t = cluster_id; ok && t < tiles; t += num_clusters, ++it) {
                const int acc = it & 1;
                if (!mbar_wait(tempty_bar(acc), (static_cast<uint32_t>(it >> 1) & 1u) ^ 1u, p.timeout_ns, kErrWaitMma, 100 + acc)) break;
                tc_fence_after();
                const uint32_t d = tmem + static_cast<uint32_t>(acc * 256);
                for (int st = st0; st < st1; ++st) {
                    if (!mbar_wait(full_bar(stage), phase, p.timeout_ns, kErrWaitMma, stage) ||
                        !mbar_wait(ready_bar(stage), phase, p.timeout_ns, kErrWaitMma, 200 + stage)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a_addr = smem_u32(sA + stage * kWgABytes), b_addr = smem_u32(sB + stage * kWgBBytes);
                    const int kk_end = min(kWgBK / 16, (p.K - st * kWgBK + 15) / 16);
#pragma unroll
                    for (int kk = 0; kk < kWgBK / 16; ++kk) {
                        if (kk >= kk_end) break;
                        umma_f16<2>(d, smem_desc_sw128(a_addr + kk * 16 * 128, kWgBK * 128, 1024),
                                    smem_desc_sw128(b_addr + kk * 16 * 128, kWgBK * 128, 1024), kIdesc, (st != st0 || kk != 0) ? 1u : 0u);
                    }
                    umma_commit<2>(mapa_shared(empty_bar(stage), lead));
                    umma_commit<2>(mapa_shared(empty_bar(stage), lead | 1u));
                    if (++stage == kWgStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                umma_commit<2>(mapa_shared(tfull_bar(acc), lead));
                umma_commit<2>(mapa_shared(tfull_bar(acc), lead | 1u));
            }
        }
    } else if (warp >= 6) {
        // Lanes 8g .. 8g+7 hold the 16-byte chunks c of two rows, 0..3 of one and 4..7 of the next: the reads cover all
        // banks once, and so do the writes (chunks 2(c%4), 2(c%4)+1 of 64-column atom c/4, xor row % 8).
        const int w = warp & 3, group = (warp - 6) >> 2, c = lane & 7, g = (lane >> 3) ^ (c >> 2);
        int stage = 0, count = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int t = cluster_id; ok && t < tiles; t += num_clusters) {
            int tm, tn;
            f8_tile_coords(t, p.tiles_m, p.tiles_n, p.raster_group, tm, tn);
            const int blk = tn * 2 + half;
            const bool in = blk * 128 < p.N;
            auto scale_of = [&](int st) {
                const int row = st * kWgBK + w * 16 + (lane & 15);
                return in && row < p.K ? static_cast<uint32_t>(p.scale[row * p.lds + blk]) : 127u;
            };
            // this group's stages of the tile
            const int first = st0 + (group - count % kWgGroups + kWgGroups) % kWgGroups;
            uint32_t next = scale_of(first), after = scale_of(first + kWgGroups);
            for (int st = st0; st < st1; ++st, ++count) {
                if (count % kWgGroups == group) {
                    const float mine = e8m0_scale(next);
                    if (!mbar_wait(x_bar(stage), phase, p.timeout_ns, kErrWaitMma, 300 + stage)) {
                        ok = false;
                        break;
                    }
                    const uint8_t* src = sX + stage * kWgRawBytes;
                    uint8_t* dst = sB + stage * kWgBBytes + (c >> 2) * (kWgBK * 128);
                    uint4 v[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const uint4*>(src + (w * 16 + 4 * i + g) * 128 + c * 16);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int row = w * 16 + 4 * i + g;
                        const float s = __shfl_sync(0xffffffffu, mine, 4 * i + g);
                        const uint4 lo = make_uint4(scaled_pair<T>(v[i].x & 0xffffu, s), scaled_pair<T>(v[i].x >> 16, s),
                                                    scaled_pair<T>(v[i].y & 0xffffu, s), scaled_pair<T>(v[i].y >> 16, s));
                        const uint4 hi = make_uint4(scaled_pair<T>(v[i].z & 0xffffu, s), scaled_pair<T>(v[i].z >> 16, s),
                                                    scaled_pair<T>(v[i].w & 0xffffu, s), scaled_pair<T>(v[i].w >> 16, s));
                        uint4* out = reinterpret_cast<uint4*>(dst + row * 128);
                        const int chunk = (c & 3) * 2;
                        out[chunk ^ (row & 7)] = lo;
                        out[(chunk + 1) ^ (row & 7)] = hi;
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_pair(mapa_shared(ready_bar(stage), lead));
                    next = after;
                    after = scale_of(st + 2 * kWgGroups);
                }
                if (++stage == kWgStages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            ok = __all_sync(0xffffffffu, ok);
        }
    }

    const int q = warp & 3;  // the lane quarter an epilogue warp may read
    const bool epilogue = warp >= 2 && warp < 6;
    const BoxOut out{&tmap_c, p.C, p.ldc, p.M, p.N, p.c_tma};
    uint8_t* stg = epi + q * kF8EpiWarpBytes;
    uint32_t turn = 0;
    if (epilogue) {
        int it = 0;
        for (int t = cluster_id; t < tiles; t += num_clusters, ++it) {
            const int acc = it & 1;
            if (!mbar_wait(tfull_bar(acc), static_cast<uint32_t>(it >> 1) & 1u, p.timeout_ns, kErrWaitEpilogue, acc)) break;
            tc_fence_after();
            int tm, tn;
            f8_tile_coords(t, p.tiles_m, p.tiles_n, p.raster_group, tm, tn);
            const int row0 = tm * 256 + half * 128 + q * 32;
            const uint32_t base = tmem + static_cast<uint32_t>(acc * 256) + (static_cast<uint32_t>(q * 32) << 16);
#pragma unroll 1
            for (int c = 0; c < 256; c += 32) {
                uint32_t r[32];
                tmem_ld_32x32b_x32(base + static_cast<uint32_t>(c), r);
                tmem_ld_wait();
                float f[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(r[i]);
                if (p.slices > 1) {
                    // this slice's sums, four columns of 128 rows at a time; the MMAs have read every stage
                    float4* part = reinterpret_cast<float4*>(sA) + (c / 4) * 128 + q * 32 + lane;
#pragma unroll
                    for (int j = 0; j < 8; ++j) part[j * 128] = make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]);
                    continue;
                }
                const int col = tn * 256 + c;
                if (col >= p.N) continue;
                if (p.accumulate) add_box<OUT>(out, p.c_vec, row0 + lane, col, f);
                store_box<OUT>(out, stg, row0, lane, col, f, turn);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_pair(mapa_shared(tempty_bar(acc), lead));
        }
    }
    if (p.slices > 1) {
        __syncthreads();
        cluster_sync_all();
        if (epilogue) {
            int tm, tn;
            f8_tile_coords(cluster_id, p.tiles_m, p.tiles_n, p.raster_group, tm, tn);
            const int row0 = tm * 256 + half * 128 + q * 32;
#pragma unroll 1
            for (int ch = 8 * slice / p.slices; ch < 8 * (slice + 1) / p.slices; ++ch) {
                const int col = tn * 256 + ch * 32;
                if (col >= p.N) break;
                const uint32_t at = smem_u32(sA) + static_cast<uint32_t>((ch * 8 * 128 + q * 32 + lane) * 16);
                float f[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) f[i] = 0.f;
#pragma unroll 1
                for (int s = 0; s < p.slices; ++s) {
                    const uint32_t from = mapa_shared(at, static_cast<uint32_t>(2 * s + half));
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float4 v = ld_cluster_f4(from + static_cast<uint32_t>(j * 128 * 16));
                        f[4 * j] += v.x;
                        f[4 * j + 1] += v.y;
                        f[4 * j + 2] += v.z;
                        f[4 * j + 3] += v.w;
                    }
                }
                if (p.accumulate) add_box<OUT>(out, p.c_vec, row0 + lane, col, f);
                store_box<OUT>(out, stg, row0, lane, col, f, turn);
            }
        }
    }
    if (epilogue && p.c_tma && lane == 0) bulk_wait_group_all();

    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc<2>(tmem, 512);
    }
#endif
}

}  // namespace vk
