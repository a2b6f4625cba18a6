// dW = dY^T * X on the tensor cores of sm_100a: dY in 16 bits, X as the forward pass kept it, e4m3 with a power-of-two
// scale for each token and 128 columns.
//
// X's scale changes along the sum (the tokens), so neither the tensor core's block scales nor the epilogue can apply
// it, and one MMA takes both operands in the same type.  Four warps therefore turn each stage of X into dY's type on
// its way from TMA to the MMAs, inside shared memory: q * 2^e is exact in bf16, and the product is that of the 16-bit
// kernel.  X costs half the bytes of a 16-bit checkpoint in memory and on the way into the SM.
//
// Roles (480 threads per CTA, pairs of CTAs on one 256 x 256 tile):
//   warp 0      TMA loads of dY: 128 of the tile's rows, M-major, 128 tokens a stage.
//   warp 1      tensor memory, and in the pair's leader the MMAs (one lane).
//   warps 2..5  epilogue: tensor memory -> registers -> swizzled staging -> TMA stores.
//   warps 6..13 X's bytes -> 16-bit values in the 128-byte swizzled layout of an N-major operand; four warps to a block.
//   warp 14     TMA loads of X's bytes: this CTA's 128 columns, 64 tokens a block.
// A block of X's bytes is free again once it is converted and waits for none of dY's longer way; a stage of dY and X's
// values is free once it is multiplied.  Tiles are handed out as in fp8_gemm.cuh.
#pragma once

#include "fp8_gemm.cuh"

namespace vk {

struct WgradParams {
    int M, N, K;  // rows and columns of dW, tokens
    TileWork work;
    const uint8_t* scale;
    long long lds;
    void* C;
    long long ldc;
    int c_tma, accumulate;
    unsigned long long timeout_ns;
};

constexpr int kWgStages = 3, kWgBK = 128;  // dY and X's values, tokens of a stage
constexpr int kWgXStages = 3, kWgXK = 64;  // X's bytes, tokens of a block
constexpr int kWgABytes = 128 * kWgBK * 2;
constexpr int kWgBBytes = 128 * kWgBK * 2;
constexpr int kWgRawBytes = 128 * kWgXK;
constexpr int kWgEpiWarpBytes = 2048;
constexpr int kWgBars = 3 * kWgStages + 2 * kWgXStages + 4;
constexpr int kWgSmemBytes =
    1024 + kWgStages * (kWgABytes + kWgBBytes) + kWgXStages * kWgRawBytes + 4 * kWgEpiWarpBytes + kWgBars * 8 + 16;
constexpr int kWgThreads = 192 + 256 + 32;
static_assert(kWgSmemBytes <= 232448, "shared memory per CTA");
static_assert(kWgStages * (kWgABytes + kWgBBytes) >= 128 * 256 * 4, "a shared tile's sums fit the stages");

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
    uint8_t* epi = sB + kWgStages * kWgBBytes;
    uint8_t* sX = epi + 4 * kWgEpiWarpBytes;
    uint64_t* bars = reinterpret_cast<uint64_t*>(sX + kWgXStages * kWgRawBytes);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kWgBars);

    const uint32_t bar0 = smem_u32(bars);
    auto full_bar = [&](int s) { return bar0 + 8u * s; };                           // dY loaded
    auto ready_bar = [&](int s) { return bar0 + 8u * (kWgStages + s); };            // X's values written
    auto empty_bar = [&](int s) { return bar0 + 8u * (2 * kWgStages + s); };
    auto x_full = [&](int s) { return bar0 + 8u * (3 * kWgStages + s); };
    auto x_empty = [&](int s) { return bar0 + 8u * (3 * kWgStages + kWgXStages + s); };
    auto tfull_bar = [&](int a) { return bar0 + 8u * (3 * kWgStages + 2 * kWgXStages + a); };
    auto tempty_bar = [&](int a) { return bar0 + 8u * (3 * kWgStages + 2 * kWgXStages + 2 + a); };

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const uint32_t lead = rank & ~1u;  // the pair's leader
    const int half = static_cast<int>(rank & 1u), part = static_cast<int>(rank >> 1);
    const int cluster_id = blockIdx.x / (2 * p.work.pairs);
    const int num_clusters = gridDim.x / (2 * p.work.pairs);
    const int units = work_units(p.work);

    if (warp == 0 && lane == 0) {
        prefetch_tmap(&tmap_a);
        prefetch_tmap(&tmap_b);
        if (p.c_tma) prefetch_tmap(&tmap_c);
        for (int s = 0; s < kWgStages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(ready_bar(s), 16);  // the conversion warps of both CTAs
            mbar_init(empty_bar(s), 1);
        }
        for (int s = 0; s < kWgXStages; ++s) {
            mbar_init(x_full(s), 1);
            mbar_init(x_empty(s), 4);     // the block's four conversion warps
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
            Ring r(kWgStages);
            bool ok = true;
            for (int u = cluster_id; ok && u < units; u += num_clusters) {
                const Work w = work_unit(p.work, u, part);
                const int m0 = w.tm * 256 + half * 128;
                for (int st = w.st0; st < w.st1; ++st, r.next()) {
                    if (!mbar_wait(empty_bar(r.at), r.phase ^ 1u, p.timeout_ns, kErrWaitProducer, r.at)) {
                        ok = false;
                        break;
                    }
                    if (half == 0) mbar_arrive_expect_tx(full_bar(r.at), 2 * kWgABytes);
                    const uint32_t bar = mapa_shared(full_bar(r.at), lead);
                    const uint32_t dst = smem_u32(sA + r.at * kWgABytes);
                    tma_load_2d_pair(dst, &tmap_a, bar, m0, st * kWgBK);
                    tma_load_2d_pair(dst + 64 * kWgBK * 2, &tmap_a, bar, m0 + 64, st * kWgBK);
                }
            }
            // the MMAs' signals to this CTA's barriers have all arrived before the CTA may exit
            for (int i = 0; ok && i < kWgStages; ++i, r.next())
                ok = mbar_wait(empty_bar(r.at), r.phase ^ 1u, p.timeout_ns, kErrWaitTail, r.at);
        }
    } else if (warp == 14) {
        if (lane == 0) {
            Ring r(kWgXStages);
            bool ok = true;
            for (int u = cluster_id; ok && u < units; u += num_clusters) {
                const Work w = work_unit(p.work, u, part);
                for (int blk = 2 * w.st0; blk < 2 * w.st1; ++blk, r.next()) {
                    if (!mbar_wait(x_empty(r.at), r.phase ^ 1u, p.timeout_ns, kErrWaitProducer, 300 + r.at)) {
                        ok = false;
                        break;
                    }
                    mbar_arrive_expect_tx(x_full(r.at), kWgRawBytes);
                    tma_load_2d(smem_u32(sX + r.at * kWgRawBytes), &tmap_b, x_full(r.at), w.tn * 256 + half * 128, blk * kWgXK);
                }
            }
        }
    } else if (warp == 1) {
        if (half == 0 && lane == 0) {
            constexpr uint32_t kType = std::is_same_v<T, __half> ? 0u : 1u;
            // D fp32, A and B of T, A M-major, B N-major
            constexpr uint32_t kIdesc = idesc_f16(256, 256, true, true) | (1u << 15) | (kType << 7) | (kType << 10);
            Ring r(kWgStages);
            int it = 0;
            bool ok = true;
            for (int u = cluster_id; ok && u < units; u += num_clusters, ++it) {
                const Work w = work_unit(p.work, u, part);
                const int acc = it & 1;
                if (!mbar_wait(tempty_bar(acc), (static_cast<uint32_t>(it >> 1) & 1u) ^ 1u, p.timeout_ns, kErrWaitMma, 100 + acc)) break;
                tc_fence_after();
                const uint32_t d = tmem + static_cast<uint32_t>(acc * 256);
                for (int st = w.st0; st < w.st1; ++st, r.next()) {
                    if (!mbar_wait(full_bar(r.at), r.phase, p.timeout_ns, kErrWaitMma, r.at) ||
                        !mbar_wait(ready_bar(r.at), r.phase, p.timeout_ns, kErrWaitMma, 200 + r.at)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a_addr = smem_u32(sA + r.at * kWgABytes), b_addr = smem_u32(sB + r.at * kWgBBytes);
                    const int kk_end = min(kWgBK / 16, (p.K - st * kWgBK + 15) / 16);
#pragma unroll
                    for (int kk = 0; kk < kWgBK / 16; ++kk) {
                        if (kk >= kk_end) break;
                        umma_f16<2>(d, smem_desc_sw128(a_addr + kk * 16 * 128, kWgBK * 128, 1024),
                                    smem_desc_sw128(b_addr + kk * 16 * 128, kWgBK * 128, 1024), kIdesc, (st != w.st0 || kk != 0) ? 1u : 0u);
                    }
                    umma_commit<2>(mapa_shared(empty_bar(r.at), lead));
                    umma_commit<2>(mapa_shared(empty_bar(r.at), lead | 1u));
                }
                if (!ok) break;
                umma_commit<2>(mapa_shared(tfull_bar(acc), lead));
                umma_commit<2>(mapa_shared(tfull_bar(acc), lead | 1u));
            }
        }
    } else if (warp >= 6) {
        // Four warps take the even blocks of 64 tokens, four the odd ones; a warp has 16 tokens.  Lanes 8g .. 8g+7 hold the
        // 16-byte chunks c of two rows, 0..3 of one and 4..7 of the next: the reads cover all banks once, and so do the
        // writes (chunks 2(c%4), 2(c%4)+1 of 64-column atom c/4, xor row % 8).
        const int w4 = warp & 3, group = (warp - 6) >> 2, c = lane & 7, g = (lane >> 3) ^ (c >> 2);
        Ring rx(kWgXStages), r(kWgStages);
        if (group) rx.next();
        bool ok = true;
        for (int u = cluster_id; ok && u < units; u += num_clusters) {
            const Work w = work_unit(p.work, u, part);
            const int col_blk = w.tn * 2 + half;
            const bool in = col_blk * 128 < p.N;
            auto scale_of = [&](int st) {
                const int row = st * kWgBK + group * kWgXK + w4 * 16 + (lane & 15);
                return in && row < p.K ? static_cast<uint32_t>(p.scale[row * p.lds + col_blk]) : 127u;
            };
            uint32_t next = scale_of(w.st0), after = scale_of(w.st0 + 1);  // two stages ahead of their use
            for (int st = w.st0; st < w.st1; ++st, r.next(), rx.next(), rx.next()) {
                const float mine = e8m0_scale(next);
                if (!mbar_wait(x_full(rx.at), rx.phase, p.timeout_ns, kErrWaitMma, 300 + rx.at)) {
                    ok = false;
                    break;
                }
                const uint8_t* src = sX + rx.at * kWgRawBytes;
                uint4 v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const uint4*>(src + (w4 * 16 + 4 * i + g) * 128 + c * 16);
                __syncwarp();
                if (lane == 0) mbar_arrive(x_empty(rx.at));
                if (!mbar_wait(empty_bar(r.at), r.phase ^ 1u, p.timeout_ns, kErrWaitMma, 400 + r.at)) {
                    ok = false;
                    break;
                }
                uint8_t* dst = sB + r.at * kWgBBytes + (c >> 2) * (kWgBK * 128) + group * (kWgXK * 128);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = w4 * 16 + 4 * i + g;
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
                if (lane == 0) mbar_arrive_pair(mapa_shared(ready_bar(r.at), lead));
                next = after;
                after = scale_of(st + 2);
            }
            ok = __all_sync(0xffffffffu, ok);
        }
    }

    const bool epilogue = warp >= 2 && warp < 6;
    const int q = warp & 3;  // the lane quarter an epilogue warp may read
    const BoxOut out{&tmap_c, p.C, p.ldc, p.M, p.N, p.c_tma, p.accumulate};
    uint8_t* stg = epi + q * kWgEpiWarpBytes;
    float4* sums = reinterpret_cast<float4*>(sA);  // of a shared tile: its stages have all been read by then
    uint32_t turn = 0;
    if (epilogue) {
        int it = 0;
        for (int u = cluster_id; u < units; u += num_clusters, ++it) {
            const Work w = work_unit(p.work, u, part);
            const int acc = it & 1;
            if (!mbar_wait(tfull_bar(acc), static_cast<uint32_t>(it >> 1) & 1u, p.timeout_ns, kErrWaitEpilogue, acc)) break;
            tc_fence_after();
            finish_unit<OUT, 1>(p.work, w, out, stg, p.work.pairs > 1 ? sums : nullptr, tmem + static_cast<uint32_t>(acc * 256), 0, half, q, lane,
                                turn, p.timeout_ns, [] {});
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_pair(mapa_shared(tempty_bar(acc), lead));
        }
    }
    if (p.work.pairs > 1) {
        __syncthreads();
        cluster_sync_all();
        if (epilogue) finish_shared<OUT, 1>(p.work, work_unit(p.work, cluster_id, part), out, stg, sums, part, half, q, lane, turn);
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
