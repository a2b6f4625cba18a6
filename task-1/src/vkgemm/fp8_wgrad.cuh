// dW = dY^T * X on the tensor cores of sm_100a: dY in 16 bits, X as the forward pass kept it, e4m3 with a power-of-two
// scale for each token and 128 columns.
//
// X's scale changes along the sum (the tokens), so neither the tensor core's block scales nor the epilogue can apply
// it, and one MMA takes both operands in the same type.  Four warps therefore turn each stage of X into dY's type on
// its way to the MMAs: q * 2^e is exact in bf16 (see fp8_rows.cuh), and the product is that of the 16-bit kernel.  X costs half
// the bytes of a 16-bit checkpoint in memory and on the way into the SM.  Bound by the conversion: at 8192 x 4096 x 4096 the
// tensor pipe is active for 70 % of the time, in fp16, which takes two multiplies, a conversion, a minimum and a maximum for a pair
// of values where bf16 takes a conversion and a multiply, for 61 %.  bf16 214 to 219 us, 1.27 PFLOP/s; fp16 236; bf16 into fp32 222,
// added to an fp32 dW 234 (4000 x 1000 x 3333, whose rows take no TMA stores: 44 and 82, C being read a row to a lane).
//
// Roles (576 threads per CTA, pairs of CTAs on one 256 x 256 tile, 128 tokens a stage):
//   warp 0      TMA loads of dY: 128 of the tile's rows, M-major.
//   warp 1      tensor memory, and in the pair's leader the MMAs.
//   warps 2..5  epilogue: tensor memory -> registers -> swizzled staging -> TMA stores.
//   warps 6..17 X's bytes, from global memory through registers -> 16-bit values in the 128-byte swizzled layout of an
//               N-major operand.  Each four warps have one of the ring's three stages: a stage's way (load, wait, convert,
//               make visible, signal) is longer than its MMAs, and three overlap (8192 x 4096 x 4096: two groups 252 us,
//               three 219 when that was tried).
// X's bytes took a ring of TMA loads in shared memory first: its waits, and the fence before a block can be written
// again, cost as much as the conversion (290 us).
// Tiles are handed out as in fp8_gemm.cuh.
#pragma once

#include "fp8_gemm.cuh"

namespace vk {

struct WgradParams {
    int M, N, K;  // rows and columns of dW, tokens
    TileWork work;
    const uint8_t* X;
    const uint8_t* scale;
    long long ldx, lds;
    void* C;
    long long ldc;
    int c_tma, c_width, accumulate;
    unsigned long long timeout_ns;
};

constexpr int kWgStages = 3, kWgBK = 128;
constexpr int kWgABytes = 128 * kWgBK * 2;
constexpr int kWgBBytes = 128 * kWgBK * 2;
constexpr int kWgBars = 2 * kWgStages + 4;
constexpr int kWgSmemBytes = 1024 + kWgStages * (kWgABytes + kWgBBytes) + 4 * kF8EpiWarpBytes + kWgBars * 8 + 16;
constexpr int kWgThreads = 192 + 128 * kWgStages;
static_assert(kWgSmemBytes <= 232448, "shared memory per CTA");
static_assert(kWgStages * (kWgABytes + kWgBBytes) >= 128 * 256 * 4 + 16 * kF8EpiWarpBytes, "a shared tile's sums and staging fit the stages");

// The first n (below 16) bytes at src, and zeros.
__device__ __noinline__ uint4 first_bytes(const uint8_t* src, int n)
{
    uint64_t lo = 0, hi = 0;
    for (int b = 0; b < n; ++b) (b < 8 ? lo : hi) |= static_cast<uint64_t>(src[b]) << (8 * (b & 7));
    return make_uint4(static_cast<uint32_t>(lo), static_cast<uint32_t>(lo >> 32), static_cast<uint32_t>(hi), static_cast<uint32_t>(hi >> 32));
}

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
        // a power of two: exact, but for bf16's smallest step and beyond its largest number
        const __nv_bfloat162 v = __hmul2(__floats2bfloat162_rn(f.x, f.y), __float2bfloat162_rn(scale));
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
    wgrad_fp8_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_c, const WgradParams p)
{
#if defined(__CUDA_ARCH__) && (__CUDA_ARCH__ >= 1000)
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sA = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sB = sA + kWgStages * kWgABytes;
    uint8_t* epi = sB + kWgStages * kWgBBytes;
    uint64_t* bars = reinterpret_cast<uint64_t*>(epi + 4 * kF8EpiWarpBytes);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kWgBars);
    volatile uint32_t* gave_up = tmem_slot + 1;  // a wait of this CTA has

    const uint32_t bar0 = smem_u32(bars);
    auto full_bar = [&](int s) { return bar0 + 8u * s; };
    auto empty_bar = [&](int s) { return bar0 + 8u * (kWgStages + s); };
    auto tfull_bar = [&](int a) { return bar0 + 8u * (2 * kWgStages + a); };
    auto tempty_bar = [&](int a) { return bar0 + 8u * (2 * kWgStages + 2 + a); };

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = blockIdx.x % (2 * p.work.pairs);  // in the cluster
    const uint32_t lead = rank & ~1u;                       // the pair's leader
    const int half = static_cast<int>(rank & 1u), part = static_cast<int>(rank >> 1);
    const int cluster_id = blockIdx.x / (2 * p.work.pairs);
    const int num_clusters = gridDim.x / (2 * p.work.pairs);
    const int units = work_units(p.work);

    if (warp == 0 && lane == 0) {
        prefetch_tmap(&tmap_a);
        if (p.c_tma) prefetch_tmap(&tmap_c);
        for (int s = 0; s < kWgStages; ++s) {
            mbar_init(full_bar(s), 9);  // dY's bytes, and the stage's four conversion warps of both CTAs
            mbar_init(empty_bar(s), 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(tfull_bar(a), 1);
            mbar_init(tempty_bar(a), 8);  // the epilogue warps of both CTAs
        }
        fence_mbar_init();
        *gave_up = 0;
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
            if (!ok) *gave_up = 1;
        }
    } else if (warp == 1) {
        if (half == 0) {  // the whole warp, one lane issuing: see gemm_fp8_kernel
            constexpr uint32_t kType = std::is_same_v<T, __half> ? 0u : 1u;
            // D fp32, A and B of T, A M-major, B N-major
            constexpr uint32_t kIdesc = idesc_f16(256, 256, true, true) | (1u << 15) | (kType << 7) | (kType << 10);
            constexpr uint32_t kIdescHalf = idesc_f16(256, 128, true, true) | (1u << 15) | (kType << 7) | (kType << 10);
            const bool one = elect_one();
            const uint32_t base = __shfl_sync(0xffffffffu, tmem, 0);
            const uint64_t a_desc = smem_desc_sw128(smem_u32(sA), kWgBK * 128, 1024);
            const uint64_t b_desc = smem_desc_sw128(smem_u32(sB), kWgBK * 128, 1024);
            Ring r(kWgStages);
            int it = 0;
            bool ok = true;
            for (int u = cluster_id; ok && u < units; u += num_clusters, ++it) {
                const Work w = work_unit(p.work, u, part);
                const int acc = it & 1;
                ok = mbar_wait_pair_warp(tempty_bar(acc), (static_cast<uint32_t>(it >> 1) & 1u) ^ 1u, p.timeout_ns, kErrWaitMma, 100 + acc);
                if (!ok) break;
                const uint32_t d = base + static_cast<uint32_t>(acc * 256);
                const uint32_t idesc = w.cols == 256 ? kIdesc : kIdescHalf;
                for (int st = w.st0; st < w.st1; ++st, r.next()) {
                    ok = mbar_wait_pair_warp(full_bar(r.at), r.phase, p.timeout_ns, kErrWaitMma, r.at);
                    if (!ok) break;
                    tc_fence_after();
                    if (one) {
                        const uint64_t a = a_desc + static_cast<uint32_t>(r.at) * (kWgABytes >> 4);
                        const uint64_t b = b_desc + static_cast<uint32_t>(r.at) * (kWgBBytes >> 4);
                        const int kk_end = min(kWgBK / 16, (p.K - st * kWgBK + 15) / 16);
                        auto mma = [&](int kk) {
                            umma_f16<2>(d, a + (kk * 16 * 128 >> 4), b + (kk * 16 * 128 >> 4), idesc, (st != w.st0 || kk != 0) ? 1u : 0u);
                        };
                        if (kk_end == kWgBK / 16) {
#pragma unroll
                            for (int kk = 0; kk < kWgBK / 16; ++kk) mma(kk);
                        } else {
                            for (int kk = 0; kk < kk_end; ++kk) mma(kk);
                        }
                        umma_commit_pair(empty_bar(r.at), lead);
                        if (st + 1 == w.st1) umma_commit_pair(tfull_bar(acc), lead);
                    }
                    __syncwarp();
                }
            }
            if (!ok) *gave_up = 1;
        }
    } else if (warp >= 6) {
        // A warp has 32 tokens of its stages.  Whole tiles: lanes 8g .. 8g+7 hold the 16-byte chunks c of two rows, 0..3 of
        // one and 4..7 of the next, so that the writes (chunks 2(c%4), 2(c%4)+1 of 64-column atom c/4, xor row % 8) cover all
        // banks once.  Halved ones: chunks 0..3 of two rows, which do too.
        const int w4 = warp & 3, group = (warp - 6) >> 2;
        // the group's stages, one after the other: always the same place in the ring
        int u = cluster_id, st = 0;
        uint32_t phase = 0;
        Work w = {};
        auto open = [&] {
            if (u < units) {
                w = work_unit(p.work, u, part);
                st = w.st0;
            }
        };
        auto step = [&](int n) {
            for (; n > 0 && u < units; --n) {
                if (++st < w.st1) continue;
                u += num_clusters;
                open();
            }
        };
        uint4 v[8];
        uint32_t scale = 127;
        auto fetch = [&] {
            const bool whole = w.cols == 256;
            const int col0 = w.n0 + half * (w.cols / 2), t0 = st * kWgBK + w4 * 32;
            const int c = whole ? lane & 7 : lane & 3, g = whole ? (lane >> 3) ^ (c >> 2) : lane >> 2;
            const int n = p.N - col0 - c * 16;  // bytes of this chunk that exist
            const uint8_t* src = p.X + static_cast<long long>(t0 + g) * p.ldx + col0 + c * 16;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int row = (whole ? 4 : 8) * i;
                v[i] = make_uint4(0, 0, 0, 0);
                if (n > 0 && (whole || i < 4) && t0 + g + row < p.K) {
                    // a row's last chunk reads into the row's padding, which every row but the last is sure to have
                    if (n >= 16 || t0 + g + row + 1 < p.K)
                        v[i] = *reinterpret_cast<const uint4*>(src + row * p.ldx);
                    else
                        v[i] = first_bytes(src + row * p.ldx, n);
                }
            }
            const int blk = w.n0 / 128 + (whole ? half : 0);
            scale = t0 + lane < p.K && blk * 128 < p.N ? p.scale[(t0 + lane) * p.lds + blk] : 127u;
        };
        auto convert = [&](auto whole_tag, uint8_t* dst) {
            constexpr bool kWhole = decltype(whole_tag)::value;
            const int c = kWhole ? lane & 7 : lane & 3, g = kWhole ? (lane >> 3) ^ (c >> 2) : lane >> 2;
            const float mine = e8m0_scale(scale);
#pragma unroll
            for (int i = 0; i < (kWhole ? 8 : 4); ++i) {
                const int t = (kWhole ? 4 : 8) * i + g;  // of this warp's tokens
                const float s = __shfl_sync(0xffffffffu, mine, t);
                const uint4 lo = make_uint4(scaled_pair<T>(v[i].x & 0xffffu, s), scaled_pair<T>(v[i].x >> 16, s),
                                            scaled_pair<T>(v[i].y & 0xffffu, s), scaled_pair<T>(v[i].y >> 16, s));
                const uint4 hi = make_uint4(scaled_pair<T>(v[i].z & 0xffffu, s), scaled_pair<T>(v[i].z >> 16, s),
                                            scaled_pair<T>(v[i].w & 0xffffu, s), scaled_pair<T>(v[i].w >> 16, s));
                uint4* out = reinterpret_cast<uint4*>(dst + (c >> 2) * (kWgBK * 128) + (w4 * 32 + t) * 128);
                const int chunk = (c & 3) * 2;
                out[chunk ^ (t & 7)] = lo;
                out[(chunk + 1) ^ (t & 7)] = hi;
            }
        };
        open();
        step(group);
        uint8_t* dst = sB + group * kWgBBytes;
        if (u < units) fetch();
        while (u < units) {
            if (!mbar_wait_warp(empty_bar(group), phase ^ 1u, p.timeout_ns, kErrWaitMma, 400 + group)) {
                *gave_up = 1;
                break;
            }
            if (w.cols == 256)
                convert(std::true_type{}, dst);
            else
                convert(std::false_type{}, dst);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive_pair(mapa_shared(full_bar(group), lead));
            phase ^= 1u;
            step(kWgStages);
            if (u < units) fetch();  // behind the fence, which would wait for the loads
        }
    }

    const bool epilogue = warp >= 2 && warp < 6;
    const int q = warp & 3;  // the lane quarter an epilogue warp may read
    const BoxOut out{&tmap_c, p.C, p.ldc, p.M, p.N, p.c_tma, p.accumulate, p.c_width};
    uint8_t* stg = epi + q * kF8EpiWarpBytes;
    float4* sums = reinterpret_cast<float4*>(sA);  // of a shared tile: its stages have all been read by then
    uint32_t turn = 0;
    if (epilogue) {
        int it = 0;
        for (int u = cluster_id; u < units; u += num_clusters, ++it) {
            const Work w = work_unit(p.work, u, part);
            const int acc = it & 1;
            if (!mbar_wait_warp(tfull_bar(acc), static_cast<uint32_t>(it >> 1) & 1u, sum_timeout_ns(p.timeout_ns, w.st1 - w.st0), kErrWaitEpilogue, acc)) {
                *gave_up = 1;
                break;
            }
            tc_fence_after();
            finish_unit<OUT>(w, out, stg, p.work.pairs > 1 ? sums : nullptr, tmem + static_cast<uint32_t>(acc * 256), 0, half, q, lane, turn, [] {});
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_pair(mapa_shared(tempty_bar(acc), lead));
        }
    }
    if (p.work.pairs > 1) {
        __syncthreads();
        cluster_sync_all();
        finish_shared<OUT>(p.work, work_unit(p.work, cluster_id, part), out, sA + 128 * 256 * 4, sums, part, half, warp, kWgThreads / 32, lane);
    }
    if (epilogue && p.c_tma && lane == 0) bulk_wait_group_all();

    tc_fence_before();
    __syncthreads();
    if (warp == 1 && *gave_up != 0) settle();
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc<2>(tmem, 512);
    }
#endif
}

}  // namespace vk
