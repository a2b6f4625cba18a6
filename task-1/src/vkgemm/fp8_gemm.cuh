// C = A * op(B) of 8-bit operands with a power-of-two scale for each block of 128, on the tensor cores of sm_100a.
//
// The block scales are applied by the tensor core itself: tcgen05.mma kind::mxf8f6f4 takes a scale byte for each row of
// A and of B and each 32 steps of k from tensor memory, and the four instructions of a 128-deep k-block are given the
// same byte (the instruction descriptor says which of a 32-bit word's four it is).  Sums are fp32 in tensor memory from
// the first k-block to the last, so the epilogue only rounds.  A scale held in fp32 would instead have to be applied to
// every 128-deep partial product by the CUDA cores: a read of the whole accumulator per k-block.
//
// Roles (224 threads per CTA, one CTA per SM, pairs of CTAs on one 256 x 256 tile, persistent over tiles):
//   warp 0      TMA loads: 256-deep stages of A (128 rows) and B (this CTA's 128 of the tile's 256 columns), 64 KB each.
//   warp 1      tensor memory, and in the pair's leader the MMAs (one lane).
//   warps 2..5  epilogue: tensor memory -> registers -> swizzled staging -> TMA stores.
//   warp 6      scales: global bytes -> the 512-byte units that tcgen05.cp copies to tensor memory.
//
// Tensor memory: two 256-column accumulators would fill all 512 columns, and the scales need some too.  So the second
// accumulator begins at column 224: the two share 32 columns, which the epilogue reads first; the next tile's MMAs start
// once it has.  Columns 480..511 hold two sets of scales (4 columns for A's 128 rows, 8 for B's 256), each for 512 of k.
//
// Scales in shared memory and tensor memory: row r's word (4 k-blocks) of a unit of 128 rows sits at byte
// (r % 32) * 16 + (r / 32) * 4; tcgen05.cp.32x128b.warpx4 makes that lane r % 32, column r / 32, in all four lane quarters.
#pragma once

#include "fp8_rows.cuh"
#include "ptx.cuh"

namespace vk {

// The scales of one operand: the word of four k-blocks for an output index (a row of A, a row or column of B).
struct ScaleSource {
    const uint8_t* p;
    long long si, st;  // strides per output index (or tile of 128) and per k-block
    int count;         // output indexes
    int tile;          // a scale for 128 output indexes
    int words;         // four k-blocks from a multiple of four are an aligned 32-bit word

    // k-blocks kb..kb+3 of output index i; what does not exist is 1
    __device__ __forceinline__ uint32_t word(int i, int kb, int num_kb) const
    {
        if (i >= count) return 0x7f7f7f7fu;
        const uint8_t* s = p + static_cast<long long>(tile ? i >> 7 : i) * si;
        if (words && (kb & 3) == 0 && kb + 4 <= num_kb) return *reinterpret_cast<const uint32_t*>(s + kb);
        uint32_t w = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b)
            w |= (kb + b < num_kb ? static_cast<uint32_t>(s[static_cast<long long>(kb + b) * st]) : 127u) << (8 * b);
        return w;
    }
};

struct F8GemmParams {
    int M, N, K;
    int tiles_m, tiles_n, num_st;  // 256-deep stages
    int raster_group;
    ScaleSource sa, sb;
    int b_k;                       // B stored n x k
    void* C;
    long long ldc;
    int c_tma;                     // C can take TMA stores
    unsigned long long timeout_ns;
};

constexpr int kF8Stages = 3;
constexpr int kF8ABytes = 128 * 256;
constexpr int kF8BBytes = 128 * 256;
constexpr int kF8StageBytes = kF8ABytes + kF8BBytes;
constexpr int kF8SfSlots = 3;
constexpr int kF8SfBytes = 512 + 1024;  // a slot: A's unit, B's two
constexpr int kF8EpiWarpBytes = 4096;   // two 32 x 32 boxes of 16-bit results, or one of fp32
constexpr int kF8Bars = 2 * kF8Stages + 3 + 2 * kF8SfSlots;
constexpr int kF8SmemBytes =
    1024 + kF8Stages * kF8StageBytes + 4 * kF8EpiWarpBytes + kF8SfSlots * kF8SfBytes + kF8Bars * 8 + 16;
constexpr int kF8Threads = 224;
constexpr int kF8Acc1 = 224;  // first column of the second accumulator
constexpr int kF8SfCol = 480;
static_assert(kF8SmemBytes <= 232448, "shared memory per CTA");

// D (+)= (A * scale_a) * (B * scale_b), e4m3, K = 32.
__device__ __forceinline__ void umma_mxf8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

// 32 rows of 16 bytes of each CTA's shared memory -> 4 columns of its tensor memory, in all four lane quarters.
__device__ __forceinline__ void tmem_copy_scales_pair(uint32_t taddr, uint64_t desc)
{
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// Unswizzled shared-memory descriptor of 8-row groups 128 bytes apart (rows of 16 bytes).
__device__ __forceinline__ uint64_t smem_desc_rows16(uint32_t addr)
{
    return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(128 >> 4) << 16) |
           (static_cast<uint64_t>(128 >> 4) << 32) | (1ull << 46);
}

// Instruction descriptor for kind::mxf8f6f4, e4m3 A and B, e8m0 scales:
//   [4,6) B's scale byte, [7,10) A format (0 = e4m3), [10,13) B format, [16] B major (1 = N-major), [17,23) N >> 3,
//   [23] scale format (1 = e8m0), [27,29) M >> 7, [29,31) A's scale byte.
__host__ __device__ constexpr uint32_t idesc_mxf8(int M, int N, bool b_n_major)
{
    return (static_cast<uint32_t>(b_n_major ? 1 : 0) << 16) | (static_cast<uint32_t>(N >> 3) << 17) | (1u << 23) |
           (static_cast<uint32_t>(M >> 7) << 27);
}

__device__ __forceinline__ void f8_tile_coords(int t, int tiles_m, int tiles_n, int group, int& tm, int& tn)
{
    const int per_group = group * tiles_n;
    const int g = t / per_group;
    const int first_m = g * group;
    const int gsz = min(tiles_m - first_m, group);
    const int r = t - g * per_group;
    tm = first_m + r % gsz;
    tn = r / gsz;
}

template <int OUT>
__device__ __forceinline__ uint32_t pack16(float lo, float hi)
{
    if constexpr (OUT == 0) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}

// Where an epilogue warp's 32 x 32 boxes go.  OUT: vk_dtype of C.
struct BoxOut {
    const CUtensorMap* map;  // boxes of 32 x 32, 64-byte (16-bit) or 128-byte (fp32) swizzle
    void* C;
    long long ldc;
    int M, N;
    int c_tma;
};

// This lane's row (row0 + lane), columns col .. col + 31.  `turn` counts the boxes of this warp.
template <int OUT>
__device__ __forceinline__ void store_box(const BoxOut& o, uint8_t* stg, int row0, int lane, int col, const float (&f)[32], uint32_t& turn)
{
    if (o.c_tma) {
        if constexpr (OUT == 1) {
            if (lane == 0) bulk_wait_group_read<0>();
            __syncwarp();
            uint4* row = reinterpret_cast<uint4*>(stg + lane * 128);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                row[j ^ (lane & 7)] = make_uint4(__float_as_uint(f[4 * j]), __float_as_uint(f[4 * j + 1]),
                                                 __float_as_uint(f[4 * j + 2]), __float_as_uint(f[4 * j + 3]));
        } else {
            stg += (turn & 1u) * 2048;
            if (lane == 0) bulk_wait_group_read<1>();
            __syncwarp();
            uint4* row = reinterpret_cast<uint4*>(stg + lane * 64);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                row[j ^ ((lane >> 1) & 3)] =
                    make_uint4(pack16<OUT>(f[8 * j], f[8 * j + 1]), pack16<OUT>(f[8 * j + 2], f[8 * j + 3]),
                               pack16<OUT>(f[8 * j + 4], f[8 * j + 5]), pack16<OUT>(f[8 * j + 6], f[8 * j + 7]));
        }
        ++turn;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && row0 < o.M) {
            tma_store_2d(o.map, smem_u32(stg), col, row0);
            bulk_commit_group();
        }
        return;
    }
    const int row = row0 + lane;
    if (row >= o.M) return;
    using T = std::conditional_t<OUT == 0, __half, std::conditional_t<OUT == 1, float, __nv_bfloat16>>;
    T* c = static_cast<T*>(o.C) + static_cast<long long>(row) * o.ldc + col;
#pragma unroll
    for (int i = 0; i < 32; ++i)
        if (col + i < o.N) c[i] = from_f32<T>(f[i]);
}

template <int OUT>
__global__ void __launch_bounds__(kF8Threads, 1)
    gemm_fp8_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                    const __grid_constant__ CUtensorMap tmap_c, const F8GemmParams p)
{
#if defined(__CUDA_ARCH__) && (__CUDA_ARCH__ >= 1000)
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sA = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sB = sA + kF8Stages * kF8ABytes;
    uint8_t* epi = sB + kF8Stages * kF8BBytes;
    uint8_t* sSf = epi + 4 * kF8EpiWarpBytes;
    uint64_t* bars = reinterpret_cast<uint64_t*>(sSf + kF8SfSlots * kF8SfBytes);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kF8Bars);

    const uint32_t bar0 = smem_u32(bars);
    auto full_bar = [&](int s) { return bar0 + 8u * s; };
    auto empty_bar = [&](int s) { return bar0 + 8u * (kF8Stages + s); };
    auto tfull_bar = [&](int a) { return bar0 + 8u * (2 * kF8Stages + a); };
    const uint32_t tempty_bar = bar0 + 8u * (2 * kF8Stages + 2);
    auto sf_full_bar = [&](int s) { return bar0 + 8u * (2 * kF8Stages + 3 + s); };
    auto sf_empty_bar = [&](int s) { return bar0 + 8u * (2 * kF8Stages + 3 + kF8SfSlots + s); };

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int cluster_id = blockIdx.x / 2;
    const int num_clusters = gridDim.x / 2;
    const int tiles = p.tiles_m * p.tiles_n;

    if (warp == 0 && lane == 0) {
        prefetch_tmap(&tmap_a);
        prefetch_tmap(&tmap_b);
        if (p.c_tma) prefetch_tmap(&tmap_c);
        for (int s = 0; s < kF8Stages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        mbar_init(tfull_bar(0), 1);
        mbar_init(tfull_bar(1), 1);
        mbar_init(tempty_bar, 8);  // the epilogue warps of both CTAs
        for (int s = 0; s < kF8SfSlots; ++s) {
            mbar_init(sf_full_bar(s), 2);  // both CTAs' scales
            mbar_init(sf_empty_bar(s), 1);
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
                const int m0 = tm * 256 + static_cast<int>(rank) * 128;
                const int n0 = tn * 256 + static_cast<int>(rank) * 128;
                for (int st = 0; st < p.num_st; ++st) {
                    if (!mbar_wait(empty_bar(stage), phase ^ 1u, p.timeout_ns, kErrWaitProducer, stage)) {
                        ok = false;
                        break;
                    }
                    if (rank == 0) mbar_arrive_expect_tx(full_bar(stage), 2 * kF8StageBytes);
                    const uint32_t bar = mapa_shared(full_bar(stage), 0);
                    const uint32_t a_dst = smem_u32(sA + stage * kF8ABytes), b_dst = smem_u32(sB + stage * kF8BBytes);
                    const int k0 = st * 256;
                    tma_load_2d_pair(a_dst, &tmap_a, bar, k0, m0);
                    tma_load_2d_pair(a_dst + 128 * 128, &tmap_a, bar, k0 + 128, m0);
                    if (p.b_k) {
                        tma_load_2d_pair(b_dst, &tmap_b, bar, k0, n0);
                        tma_load_2d_pair(b_dst + 128 * 128, &tmap_b, bar, k0 + 128, n0);
                    } else {
                        tma_load_2d_pair(b_dst, &tmap_b, bar, n0, k0);
                    }
                    if (++stage == kF8Stages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            // every stage this CTA filled is released by the MMAs before the CTA may exit
            for (int i = 0; ok && i < kF8Stages; ++i) {
                if (!mbar_wait(empty_bar(stage), phase ^ 1u, p.timeout_ns, kErrWaitTail, stage)) break;
                if (++stage == kF8Stages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
    } else if (warp == 1) {
        auto mma_loop = [&](auto b_k_tag) {
            constexpr bool B_K = decltype(b_k_tag)::value;
            constexpr uint32_t kIdesc = idesc_mxf8(256, 256, !B_K);
            int stage = 0, slot = 0, it = 0;
            uint32_t phase = 0, sf_phase = 0, set = 0;
            for (int t = cluster_id; t < tiles; t += num_clusters, ++it) {
                // the tile before has left the columns the two accumulators share (and, before that, this one's)
                if (!mbar_wait(tempty_bar, static_cast<uint32_t>(it & 1) ^ 1u, p.timeout_ns, kErrWaitMma, 100)) return;
                tc_fence_after();
                const uint32_t d = tmem + ((it & 1) ? kF8Acc1 : 0);
                for (int st = 0; st < p.num_st; ++st) {
                    if (!mbar_wait(full_bar(stage), phase, p.timeout_ns, kErrWaitMma, stage)) return;
                    const uint32_t sfa = tmem + kF8SfCol + set * 16, sfb = sfa + 4;
                    if ((st & 1) == 0) {
                        if (!mbar_wait(sf_full_bar(slot), sf_phase, p.timeout_ns, kErrWaitMma, 200 + slot)) return;
                        tc_fence_after();
                        const uint32_t src = smem_u32(sSf + slot * kF8SfBytes);
                        tmem_copy_scales_pair(sfa, smem_desc_rows16(src));
                        tmem_copy_scales_pair(sfb, smem_desc_rows16(src + 512));
                        tmem_copy_scales_pair(sfb + 4, smem_desc_rows16(src + 1024));
                    }
                    tc_fence_after();
                    const uint32_t a_addr = smem_u32(sA + stage * kF8ABytes), b_addr = smem_u32(sB + stage * kF8BBytes);
                    const int kk_end = min(8, (p.K - st * 256 + 31) / 32);
                    const uint32_t id0 = static_cast<uint32_t>(st & 1) * 2;  // scale bytes of this stage's two k-blocks
                    const uint32_t idesc = kIdesc | (id0 << 4) | (id0 << 29);
#pragma unroll
                    for (int kk = 0; kk < 8; ++kk) {
                        if (kk >= kk_end) break;
                        const uint64_t a = smem_desc_sw128(a_addr + (kk >> 2) * (128 * 128) + (kk & 3) * 32, 16, 1024);
                        const uint64_t b = B_K ? smem_desc_sw128(b_addr + (kk >> 2) * (128 * 128) + (kk & 3) * 32, 16, 1024)
                                               : smem_desc_sw128(b_addr + kk * 32 * 128, 256 * 128, 1024);
                        umma_mxf8_pair(d, a, b, idesc + (kk >> 2) * ((1u << 4) | (1u << 29)), sfa, sfb, (st | kk) != 0);
                    }
                    umma_commit<2>(empty_bar(stage));
                    umma_commit<2>(mapa_shared(empty_bar(stage), 1));
                    if (++stage == kF8Stages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                    if ((st & 1) || st + 1 == p.num_st) {
                        umma_commit<2>(sf_empty_bar(slot));
                        umma_commit<2>(mapa_shared(sf_empty_bar(slot), 1));
                        set ^= 1u;
                        if (++slot == kF8SfSlots) {
                            slot = 0;
                            sf_phase ^= 1u;
                        }
                    }
                }
                umma_commit<2>(tfull_bar(it & 1));
                umma_commit<2>(mapa_shared(tfull_bar(it & 1), 1));
            }
        };
        if (rank == 0 && lane == 0) {
            if (p.b_k)
                mma_loop(std::true_type{});
            else
                mma_loop(std::false_type{});
        }
    } else if (warp == 6) {
        int slot = 0;
        uint32_t phase = 0;
        const int num_kb = (p.K + 127) / 128;
        bool ok = true;
        for (int t = cluster_id; ok && t < tiles; t += num_clusters) {
            int tm, tn;
            f8_tile_coords(t, p.tiles_m, p.tiles_n, p.raster_group, tm, tn);
            const int m0 = tm * 256 + static_cast<int>(rank) * 128 + lane, n0 = tn * 256 + lane;
            for (int kb = 0; kb < num_kb; kb += 4) {
                uint4 a, b0, b1;
                a.x = p.sa.word(m0, kb, num_kb);
                a.y = p.sa.word(m0 + 32, kb, num_kb);
                a.z = p.sa.word(m0 + 64, kb, num_kb);
                a.w = p.sa.word(m0 + 96, kb, num_kb);
                b0.x = p.sb.word(n0, kb, num_kb);
                b0.y = p.sb.word(n0 + 32, kb, num_kb);
                b0.z = p.sb.word(n0 + 64, kb, num_kb);
                b0.w = p.sb.word(n0 + 96, kb, num_kb);
                b1.x = p.sb.word(n0 + 128, kb, num_kb);
                b1.y = p.sb.word(n0 + 160, kb, num_kb);
                b1.z = p.sb.word(n0 + 192, kb, num_kb);
                b1.w = p.sb.word(n0 + 224, kb, num_kb);
                if (!mbar_wait(sf_empty_bar(slot), phase ^ 1u, p.timeout_ns, kErrWaitProducer, 200 + slot)) {
                    ok = false;
                    break;
                }
                uint4* dst = reinterpret_cast<uint4*>(sSf + slot * kF8SfBytes) + lane;
                dst[0] = a;
                dst[32] = b0;
                dst[64] = b1;
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive_pair(mapa_shared(sf_full_bar(slot), 0));
                if (++slot == kF8SfSlots) {
                    slot = 0;
                    phase ^= 1u;
                }
            }
            ok = __all_sync(0xffffffffu, ok);
        }
        // the MMAs' signals to this CTA's barriers have all arrived before the CTA may exit
        for (int i = 0; ok && i < kF8SfSlots; ++i) {
            if (!mbar_wait(sf_empty_bar(slot), phase ^ 1u, p.timeout_ns, kErrWaitTail, 200 + slot)) break;
            if (++slot == kF8SfSlots) {
                slot = 0;
                phase ^= 1u;
            }
        }
    } else {
        const int q = warp & 3;  // the lane quarter this warp may read
        const BoxOut out{&tmap_c, p.C, p.ldc, p.M, p.N, p.c_tma};
        uint8_t* stg = epi + q * kF8EpiWarpBytes;
        uint32_t turn = 0;
        int it = 0;
        for (int t = cluster_id; t < tiles; t += num_clusters, ++it) {
            const int acc = it & 1;
            if (!mbar_wait(tfull_bar(acc), static_cast<uint32_t>(it >> 1) & 1u, p.timeout_ns, kErrWaitEpilogue, acc)) break;
            tc_fence_after();
            int tm, tn;
            f8_tile_coords(t, p.tiles_m, p.tiles_n, p.raster_group, tm, tn);
            const int row0 = tm * 256 + static_cast<int>(rank) * 128 + q * 32;
            const uint32_t base = tmem + (acc ? kF8Acc1 : 0) + (static_cast<uint32_t>(q * 32) << 16);
#pragma unroll 1
            for (int j = 0; j < 8; ++j) {
                // the shared columns first: the last 32 of accumulator 0, the first 32 of accumulator 1
                const int c = (acc ? j : (j + 7) & 7) * 32;
                uint32_t r[32];
                tmem_ld_32x32b_x32(base + static_cast<uint32_t>(c), r);
                tmem_ld_wait();
                if (j == 0) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_pair(mapa_shared(tempty_bar, 0));
                }
                const int col = tn * 256 + c;
                if (col >= p.N) continue;
                float f[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(r[i]);
                store_box<OUT>(out, stg, row0, lane, col, f, turn);
            }
            tc_fence_before();
        }
        if (p.c_tma && lane == 0) bulk_wait_group_all();
    }

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
