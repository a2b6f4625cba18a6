// C = A * B^T of 8-bit operands with at most 128 rows of A (single tokens of a few sequences): bound by B's bytes.
//
// The roles of the operands are swapped: 128 rows of B are the MMA's M, the few rows of A its N (16 to 128), so that no
// tensor work is spent on rows that do not exist and B streams through the whole GPU.  A tile of 128 rows of B is shared
// by a cluster of up to 8 CTAs, each with its part of k; they add their sums through shared memory, in the order of k.  A CTA
// has as many loads in flight as its shared memory holds (200 KB), which for common sizes is all it will ever load.  1 x 16384 x
// 4096 15 us, 4.5 TB/s; 64 x 8192 x 8192 17.2 us, 4.0 TB/s (DRAM 43 % busy: 128 CTAs on 148 SMs, and about 3 us of setup, first trip
// to memory and join); 8 x 4096 x 4096 7.6 us, with B in L2 from the call before 6.3.  k is shared up to n = 9472, where 2
// CTAs to a tile can all run at once: 8 x 11008 x 4096 takes 12.5 us on 86 of 148 SMs, 8 x 28672 x 4096 26.0.
//
// Roles (224 threads): warp 0 TMA loads, warp 1 tensor memory and MMAs, warps 2..5 epilogue, warp 6 scales (as in
// fp8_gemm.cuh).
#pragma once

#include "fp8_gemm.cuh"

namespace vk {

struct ThinParams {
    int M, N, K;
    int slices;  // CTAs per tile
    ScaleSource sa, sb;
    void* C;
    long long ldc;
    unsigned long long timeout_ns;
};

constexpr int kThinThreads = 224;
constexpr int kThinSfSlots = 4;
constexpr int kThinSfBytes = 1024;  // B's unit, A's unit

template <int NPAD>
struct ThinCfg {
    static constexpr int kStageBytes = 128 * 128 + NPAD * 128;
    static constexpr int kStages = 204800 / kStageBytes;
    static constexpr int kSfCol = NPAD < 64 ? 64 : NPAD;  // tensor memory: sums, then two sets of scales
    static constexpr int kTmemCols = 2 * kSfCol;
    static constexpr int kBars = 2 * kStages + 2 * kThinSfSlots + 1;
    static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kThinSfSlots * kThinSfBytes + kBars * 8 + 16;
    static_assert(kSmemBytes <= 232448, "shared memory per CTA");
};

__device__ __forceinline__ void umma_mxf8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void tmem_copy_scales(uint32_t taddr, uint64_t desc)
{
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

template <int NPAD, int OUT>
__global__ void __launch_bounds__(kThinThreads, 1)
    gemm_fp8_thin_kernel(const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ CUtensorMap tmap_a, const ThinParams p)
{
#if defined(__CUDA_ARCH__) && (__CUDA_ARCH__ >= 1000)
    using Cfg = ThinCfg<NPAD>;
    constexpr int kStages = Cfg::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sSf = stages + kStages * Cfg::kStageBytes;
    uint64_t* bars = reinterpret_cast<uint64_t*>(sSf + kThinSfSlots * kThinSfBytes);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Cfg::kBars);
    volatile uint32_t* gave_up = tmem_slot + 1;  // a wait of this CTA has
    const uint32_t bar0 = smem_u32(bars);
    auto full_bar = [&](int s) { return bar0 + 8u * s; };
    auto empty_bar = [&](int s) { return bar0 + 8u * (kStages + s); };
    auto sf_full_bar = [&](int s) { return bar0 + 8u * (2 * kStages + s); };
    auto sf_empty_bar = [&](int s) { return bar0 + 8u * (2 * kStages + kThinSfSlots + s); };
    const uint32_t done_bar = bar0 + 8u * (2 * kStages + 2 * kThinSfSlots);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int slice = blockIdx.x % p.slices;
    const int n0 = blockIdx.x / p.slices * 128;
    const int num_kb = (p.K + 127) / 128;
    const int kb0 = static_cast<int>(static_cast<long long>(num_kb) * slice / p.slices);
    const int kb1 = static_cast<int>(static_cast<long long>(num_kb) * (slice + 1) / p.slices);

    if (warp == 0 && lane == 0) {
        prefetch_tmap(&tmap_b);
        prefetch_tmap(&tmap_a);
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (int s = 0; s < kThinSfSlots; ++s) {
            mbar_init(sf_full_bar(s), 1);
            mbar_init(sf_empty_bar(s), 1);
        }
        mbar_init(done_bar, 1);
        fence_mbar_init();
        *gave_up = 0;
    }
    if (warp == 1) {
        tmem_alloc<1>(smem_u32(tmem_slot), Cfg::kTmemCols);
        tmem_relinquish<1>();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    bool ok = true;

    if (warp == 0) {
        if (lane == 0) {
            Ring r(kStages);
            for (int kb = kb0; kb < kb1; ++kb, r.next()) {
                if (!mbar_wait(empty_bar(r.at), r.phase ^ 1u, p.timeout_ns, kErrWaitProducer, r.at)) {
                    *gave_up = 1;
                    break;
                }
                mbar_arrive_expect_tx(full_bar(r.at), Cfg::kStageBytes);
                const uint32_t dst = smem_u32(stages + r.at * Cfg::kStageBytes);
                tma_load_2d(dst, &tmap_b, full_bar(r.at), kb * 128, n0);
                tma_load_2d(dst + 128 * 128, &tmap_a, full_bar(r.at), kb * 128, 0);
            }
        }
    } else if (warp == 1) {
        constexpr uint32_t kIdesc = idesc_mxf8(128, NPAD, false);
        const bool one = elect_one();
        const uint32_t base = __shfl_sync(0xffffffffu, tmem, 0);
        const uint64_t desc = smem_desc_sw128(smem_u32(stages), 16, 1024);
        const uint64_t sf_desc = smem_desc_rows16(smem_u32(sSf));
        Ring r(kStages), sf(kThinSfSlots);
        uint32_t set = 0;
        for (int kb = kb0; kb < kb1; ++kb, r.next()) {
            const int in = (kb - kb0) & 3;  // of a set of scales
            if ((in == 0 && !mbar_wait_warp(sf_full_bar(sf.at), sf.phase, p.timeout_ns, kErrWaitMma, 200 + sf.at)) ||
                !mbar_wait_warp(full_bar(r.at), r.phase, p.timeout_ns, kErrWaitMma, r.at)) {
                *gave_up = 1;
                break;
            }
            tc_fence_after();
            const uint32_t sfa = base + Cfg::kSfCol + set * 16, sfb = sfa + 8;
            const bool last = in == 3 || kb + 1 == kb1;
            if (one) {
                if (in == 0) {
                    const uint64_t src = sf_desc + static_cast<uint32_t>(sf.at) * (kThinSfBytes >> 4);
                    tmem_copy_scales(sfa, src);
                    tmem_copy_scales(sfb, src + (512 >> 4));
                }
                const uint64_t a = desc + static_cast<uint32_t>(r.at) * (Cfg::kStageBytes >> 4), b = a + (128 * 128 >> 4);
                const uint32_t idesc = kIdesc | (static_cast<uint32_t>(in) << 4) | (static_cast<uint32_t>(in) << 29);
                const int kk_end = min(4, (p.K - kb * 128 + 31) / 32);
                auto mma = [&](int kk) { umma_mxf8(base, a + (kk * 32 >> 4), b + (kk * 32 >> 4), idesc, sfa, sfb, kb != kb0 || kk != 0); };
                if (kk_end == 4) {
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) mma(kk);
                } else {
                    for (int kk = 0; kk < kk_end; ++kk) mma(kk);
                }
                umma_commit<1>(empty_bar(r.at));
                if (last) umma_commit<1>(sf_empty_bar(sf.at));
                if (kb + 1 == kb1) umma_commit<1>(done_bar);
            }
            __syncwarp();
            if (last) {
                set ^= 1u;
                sf.next();
            }
        }
    } else if (warp == 6) {
        Ring sf(kThinSfSlots);
        for (int kb = kb0; kb < kb1; kb += 4, sf.next()) {
            constexpr int kWords = (NPAD + 31) / 32;
            uint32_t b[4], a[kWords];
            ScaleWords<4> of_b;
            ScaleWords<kWords> of_a;
            of_b.load(p.sb, n0 + lane, 32, kb);
            of_a.load(p.sa, lane, 32, kb);
            of_b.use(b, num_kb - kb);
            of_a.use(a, num_kb - kb);
            if (!mbar_wait_warp(sf_empty_bar(sf.at), sf.phase ^ 1u, p.timeout_ns, kErrWaitProducer, 200 + sf.at)) {
                *gave_up = 1;
                break;
            }
            uint4* dst = reinterpret_cast<uint4*>(sSf + sf.at * kThinSfBytes) + lane;
            dst[0] = make_uint4(b[0], b[1], b[2], b[3]);
            dst[32] = make_uint4(a[0], a[kWords > 1 ? 1 : 0], a[kWords > 2 ? 2 : 0], a[kWords > 2 ? 3 : 0]);  // (of rows that the MMA does not have: any)
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(sf_full_bar(sf.at));
        }
    } else {
        ok = mbar_wait_warp(done_bar, 0, sum_timeout_ns(p.timeout_ns, kb1 - kb0), kErrWaitEpilogue, 0);
        if (!ok) *gave_up = 1;
        tc_fence_after();
    }

    // Epilogue thread t has row n0 + t of B in tensor memory lane t: column j is row j of A.
    using T = std::conditional_t<OUT == 0, __half, std::conditional_t<OUT == 1, float, __nv_bfloat16>>;
    const bool epilogue = warp >= 2 && warp < 6;
    const int t = (warp & 3) * 32 + lane;
    T* c = static_cast<T*>(p.C) + n0 + t;
    float4* sums = reinterpret_cast<float4*>(stages);  // [NPAD / 4][128]; the loads and MMAs of this CTA are over
    if (epilogue) {
#pragma unroll
        for (int j0 = 0; j0 < NPAD; j0 += 32) {
            float f[32];
            tmem_chunk(tmem + static_cast<uint32_t>(j0) + (static_cast<uint32_t>((warp & 3) * 32) << 16), f);
#pragma unroll
            for (int j = 0; j < (NPAD < 32 ? NPAD : 32); j += 4) {
                if (p.slices > 1) {
                    sums[(j0 + j) / 4 * 128 + t] = make_float4(f[j], f[j + 1], f[j + 2], f[j + 3]);
                    continue;
                }
#pragma unroll
                for (int i = j; i < j + 4; ++i)
                    if (j0 + i < p.M && n0 + t < p.N && ok) c[(j0 + i) * p.ldc] = from_f32<T>(f[i]);
            }
        }
        tc_fence_before();
    }
    if (p.slices > 1) {
        __syncthreads();
        cluster_sync_all();
        // by all warps: four rows of A and 32 of B at a time, all slices' sums on their way together
        for (int i = warp; ; i += kThinThreads / 32) {
            const int g = slice + (i >> 2) * p.slices, n = (i & 3) * 32 + lane;
            if (g * 4 >= p.M) break;
            const uint32_t at = smem_u32(sums + g * 128 + n);
            float4 v[8];
#pragma unroll
            for (int s = 0; s < 8; ++s)
                if (s < p.slices) v[s] = ld_cluster_f4(mapa_shared(at, static_cast<uint32_t>(s)));
            float4 f = v[0];
#pragma unroll
            for (int s = 1; s < 8; ++s) {
                if (s >= p.slices) break;
                f.x += v[s].x;
                f.y += v[s].y;
                f.z += v[s].z;
                f.w += v[s].w;
            }
            const float row[4] = {f.x, f.y, f.z, f.w};
            T* to = static_cast<T*>(p.C) + n0 + n;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (g * 4 + j < p.M && n0 + n < p.N) to[(g * 4 + j) * p.ldc] = from_f32<T>(row[j]);
        }
        cluster_sync_all();
    }
    __syncthreads();
    if (warp == 1 && *gave_up != 0) settle();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc<1>(tmem, Cfg::kTmemCols);
    }
#endif
}

}  // namespace vk
