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
//   warp 1      tensor memory, and in the pair's leader the MMAs.
//   warps 2..5  epilogue: tensor memory -> registers -> swizzled staging -> TMA stores.
//   warp 6      scales: global bytes -> the 512-byte units that tcgen05.cp copies to tensor memory.
//
// Tensor memory: two 256-column accumulators would fill all 512 columns, and the scales need some too.  So the second
// accumulator begins at column 224: the two share 32 columns, which the epilogue reads first; the next tile's MMAs start
// once it has.  Columns 480..511 hold two sets of scales (4 columns for A's 128 rows, 8 for B's 256), each for 512 of k.
//
// Bound by the MMAs: at 8192 x 8192 x 8192, bf16 out, the tensor pipe is active for 93 % of the time (519 thousand cycles for 14
// waves of 32 stages, 1160 a stage with all that is around them; its eight 256 x 256 x 32 instructions are rated at 1024).  373 to
// 388 us, 2.8 to 2.9 PFLOP/s, until the power limit lowers the clock (455 us at 1.07 GHz); 4096 x 4096 x 4096 52.4 to 53.3 us, B stored
// k x n 55.0.  512 x 4096 x 4096, 64 half tiles of 16 stages, 13.3 to 14.2 us: the pipe is active for a third of the time.  Half
// tiles read as much of A for half the work, 0.48 us a stage instead of 0.3.
//
// How tiles are handed out (TileWork): pairs walk over whole tiles; when the last wave would leave half of them or more
// without one, its tiles are cut into column halves.  (Cutting them along k, with the partial sums joined through
// global memory, was built and measured first: writing the sums took 5 us and adding them 10, which held up the next
// tile by more than the shorter wave gave.)  When there are fewer tiles than pairs, a cluster of 2 to 4 pairs shares one
// tile: each pair sums its share of k, leaves it in its own shared memory, and adds its part of the columns from all.
//
// Scales in shared memory and tensor memory: row r's word (4 k-blocks) of a unit of 128 rows sits at byte
// (r % 32) * 16 + (r / 32) * 4; tcgen05.cp.32x128b.warpx4 makes that lane r % 32, column r / 32, in all four lane quarters.
#pragma once

#include "fp8_rows.cuh"
#include "ptx.cuh"

namespace vk {

// Four scales that are st apart, one by one; those from `left` on are 1.
__device__ __noinline__ uint32_t scale_bytes(const uint8_t* at, long long st, int left)
{
    uint32_t w = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) w |= (b < left ? static_cast<uint32_t>(at[b * st]) : 127u) << (8 * b);
    return w;
}

// A word of scales of which only the first `left` k-blocks exist.
__device__ __forceinline__ uint32_t scale_word(uint32_t w, int left)
{
    return left >= 4 ? w : (w & ~(0xffffffffu << (8 * left))) | (0x7f7f7f7fu << (8 * left));
}

// The scales of one operand, as words of four k-blocks for each output index (a row of A, a row or column of B).  (40 bytes:
// with 48, the kernel for few rows of A is compiled to a slower join, 128 x 4096 x 4096 11.6 us for 9.5.)
struct ScaleSource {
    const uint8_t* p;
    const uint8_t* end;  // behind the last scale
    long long si, st;    // strides per output index (or tile of 128) and per k-block
    int count;           // output indexes
    unsigned tile : 1;     // a scale for 128 output indexes
    unsigned aligned : 1;  // four k-blocks from a multiple of four are an aligned 32-bit word

    __device__ __forceinline__ const uint8_t* at(int i, int kb) const
    {
        return i < count ? p + static_cast<long long>(tile ? i >> 7 : i) * si + static_cast<long long>(kb) * st : nullptr;
    }
};

// The words of k-blocks kb..kb+3 of N output indexes, k-blocks being neighbours: out of the one or two aligned words around
// them, as rows of scales may begin anywhere (k = 11008 has 86 blocks: 4096 x 4096 x 11008 byte by byte 230 us, against 135).
// What would reach beyond the first or the last scale is left to the bytes.  Apart: the loads, and their use, so that those
// of both operands are in flight together.  Used by whole warps.
template <int N>
struct ScaleWords {
    const uint8_t* from[N];  // what is left to the bytes
    uint32_t lo[N], hi[N], bits[N];
    bool todo;

    __device__ __forceinline__ void load(const ScaleSource& s, int i0, int step, int kb)
    {
        todo = false;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint8_t* at = s.at(i0 + step * j, kb);
            const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(at)) & 3u;
            const uint8_t* w = at - off;
            const bool in = w >= s.p && w + (off ? 8 : 4) <= s.end;  // (not of nullptr)
            lo[j] = in ? *reinterpret_cast<const uint32_t*>(w) : 0x7f7f7f7fu;
            hi[j] = in && off ? *reinterpret_cast<const uint32_t*>(w + 4) : 0x7f7f7f7fu;
            bits[j] = off * 8;
            from[j] = in ? nullptr : at;
            todo |= from[j] != nullptr;
        }
    }
    // left: the k-blocks that exist
    __device__ __forceinline__ void use(uint32_t (&out)[N], int left)
    {
        const bool any = __any_sync(0xffffffffu, todo);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            out[j] = scale_word(__funnelshift_r(lo[j], hi[j], bits[j]), left);
            if (any && from[j] != nullptr) out[j] = scale_bytes(from[j], 1, left);
        }
    }
};

// The same, whole: words of k-blocks kb..kb+3 of output indexes i0 + step * j (step 32 or 128).
template <int N>
__device__ __forceinline__ void fetch_words(uint32_t (&out)[N], const ScaleSource& s, int i0, int step, int kb, int left)
{
    if (s.aligned && left >= 4) {  // one load for each (4000 x 5120 x 3000, scales by rows: with two 54.7 us, against 51.5)
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint8_t* at = s.at(i0 + step * j, kb);
            out[j] = at != nullptr ? *reinterpret_cast<const uint32_t*>(at) : 0x7f7f7f7fu;
        }
    } else if (s.st == 1) {
        ScaleWords<N> w;
        w.load(s, i0, step, kb);
        w.use(out, left);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint8_t* at = s.at(i0 + step * j, kb);
            out[j] = at != nullptr ? scale_bytes(at, s.st, left) : 0x7f7f7f7fu;
        }
    }
}

// Output indexes 32 apart from i0, which is less than 32 above a multiple of 128: four of them share a tile's scale.
template <int N>
__device__ __forceinline__ void fetch_words(uint32_t (&out)[N], const ScaleSource& s, int i0, int kb, int left)
{
    if (s.tile) {
        uint32_t w[N / 4];
        fetch_words(w, s, i0, 128, kb, left);
#pragma unroll
        for (int j = 0; j < N; ++j) out[j] = w[j / 4];
    } else {
        fetch_words(out, s, i0, 32, kb, left);
    }
}

// How the 256 x 256 tiles of an output are shared out over clusters.
struct TileWork {
    int tiles_m, tiles_n, raster_group;
    int n;       // columns of the output
    int stages;  // k-stages of a tile
    int grain;   // stages that a share of k begins at multiples of
    int pairs;   // pairs of CTAs that share each tile through their cluster's shared memory (1: none)
    int halved;  // the last `halved` tiles are two units of 128 columns each
};

// A pair's next piece of work: stages [st0, st1) of `cols` columns from column n0 of tile row tm.
struct Work {
    int tm, n0, cols, st0, st1;
};

__host__ __device__ __forceinline__ int work_units(const TileWork& w) { return w.tiles_m * w.tiles_n + w.halved; }

// Unit u; `part`: which of w.pairs this pair is.
__device__ __forceinline__ Work work_unit(const TileWork& w, int u, int part)
{
    Work r;
    const int whole = w.tiles_m * w.tiles_n - w.halved;
    const int t = u < whole ? u : whole + (u - whole) / 2;
    const int grains = (w.stages + w.grain - 1) / w.grain;
    r.st0 = 0;
    r.st1 = w.stages;
    if (w.pairs > 1) {
        r.st0 = grains * part / w.pairs * w.grain;
        r.st1 = min(w.stages, grains * (part + 1) / w.pairs * w.grain);
    }
    const int per_group = w.raster_group * w.tiles_n;
    const int g = t / per_group;
    const int first_m = g * w.raster_group;
    const int rows = w.tiles_m - first_m < w.raster_group ? w.tiles_m - first_m : w.raster_group;
    const int in = t - g * per_group;
    r.tm = first_m + in % rows;
    r.n0 = in / rows * 256 + (u < whole ? 0 : (u - whole) % 2 * 128);
    r.cols = u < whole && w.n - r.n0 > 128 ? 256 : 128;  // a ragged last column needs no more
    return r;
}

struct F8GemmParams {
    int M, N, K;
    TileWork work;
    ScaleSource sa, sb;
    int b_k;                       // B stored n x k
    void* C;
    long long ldc;
    int c_tma, c_width;            // see BoxOut
    unsigned long long timeout_ns;
};

constexpr int kF8Stages = 3;
constexpr int kF8ABytes = 128 * 256;
constexpr int kF8BBytes = 128 * 256;
constexpr int kF8StageBytes = kF8ABytes + kF8BBytes;
constexpr int kF8SfSlots = 3;
constexpr int kF8SfBytes = 512 + 1024;  // a slot: A's unit, B's two
constexpr int kF8EpiWarpBytes = 4096;   // two boxes of 32 rows x 64 bytes, or one with rows 80 bytes apart
constexpr int kF8Bars = 2 * kF8Stages + 3 + 2 * kF8SfSlots;
constexpr int kF8SmemBytes =
    1024 + kF8Stages * kF8StageBytes + 4 * kF8EpiWarpBytes + kF8SfSlots * kF8SfBytes + kF8Bars * 8 + 16;
constexpr int kF8Threads = 224;
constexpr int kF8Acc1 = 224;  // first column of the second accumulator
constexpr int kF8SfCol = 480;
static_assert(kF8SmemBytes <= 232448, "shared memory per CTA");
static_assert(kF8Stages * kF8StageBytes >= 128 * 256 * 4 + 16 * kF8EpiWarpBytes, "a shared tile's sums and staging fit the stages");

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

// Where an epilogue warp's results go.  OUT: vk_dtype of C.
struct BoxOut {
    const CUtensorMap* map;  // boxes of 32 rows x 64 bytes, 64-byte swizzle
    void* C;
    long long ldc;
    int M, N;
    int c_tma;               // C can take TMA stores (and 16-byte accesses)
    int accumulate;          // C += the results
    int width;               // bytes that divide C's address and the distance of its rows (1, 2, 4 or 8 without TMA stores)
};

// Results of one row that leave together: 64 bytes.
struct Packed {
    uint4 w[4];
};

// A C that cannot take TMA stores: a warp's 32 rows go through the staging buffer, 80 bytes apart, to runs of 64 bytes
// per row from column col, in the widest stores W that C's alignment allows.  (Each lane its own row: 4001 x 3333 x 2999
// bf16 167 us, against 47.)  Not inlined: its registers would be taken from the kernels' other roles.
template <typename T, typename W>
__device__ __noinline__ void put_rows(T* C, long long ldc, int rows, int cols, uint8_t* stg, int lane, Packed p)
{
    constexpr int kLanes = 64 / sizeof(W), kRows = 32 / kLanes, kCount = sizeof(W) / sizeof(T);
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(stg + lane * 80 + j * 16) = p.w[j];
    __syncwarp();
    const int at = lane % kLanes, first = at * kCount, count = min(kCount, cols - first);
    const int left = rows - lane / kLanes;
    const uint8_t* from = stg + lane / kLanes * 80 + at * sizeof(W);
    T* to = C + lane / kLanes * ldc + first;
#pragma unroll
    for (int r0 = 0; r0 < 32; r0 += 8 * kRows) {
        W v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (r0 + i * kRows < 32) v[i] = *reinterpret_cast<const W*>(from + (r0 + i * kRows) * 80);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = r0 + i * kRows;
            if (r >= 32 || r >= left) continue;
            if (count == kCount) {
                *reinterpret_cast<W*>(to + r * ldc) = v[i];
            } else {
                for (int e = 0; e < count; ++e) to[r * ldc + e] = reinterpret_cast<const T*>(from + r * 80)[e];
            }
        }
    }
}

// Results col .. col + 31 of this lane's row (row0 + lane).  Two boxes of staging take turns; `turn` counts them.
template <int OUT>
__device__ __forceinline__ void store_box(const BoxOut& o, uint8_t* stg, int row0, int lane, int col, float (&f)[32], uint32_t& turn)
{
    using T = std::conditional_t<OUT == 0, __half, std::conditional_t<OUT == 1, float, __nv_bfloat16>>;
    constexpr int kCols = 64 / sizeof(T);  // of a box
    const int row = row0 + lane;
    if (o.accumulate && row < o.M) {
        const T* c = static_cast<const T*>(o.C) + static_cast<long long>(row) * o.ldc + col;
        if (o.c_tma && col + 32 <= o.N) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const Vec8<T> v = load8<true>(c, 8 * j, 32);
#pragma unroll
                for (int i = 0; i < 8; ++i) f[8 * j + i] += to_f32(v.v[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (col + i < o.N) f[i] += to_f32(c[i]);
        }
    }
#pragma unroll
    for (int h = 0; h < 32 / kCols; ++h) {
        if (col + h * kCols >= o.N) break;
        Packed p;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (OUT == 1) {
                const float* g = f + 16 * h + 4 * j;
                p.w[j] = make_uint4(__float_as_uint(g[0]), __float_as_uint(g[1]), __float_as_uint(g[2]), __float_as_uint(g[3]));
            } else {
                p.w[j] = make_uint4(pack16<OUT>(f[8 * j], f[8 * j + 1]), pack16<OUT>(f[8 * j + 2], f[8 * j + 3]),
                                    pack16<OUT>(f[8 * j + 4], f[8 * j + 5]), pack16<OUT>(f[8 * j + 6], f[8 * j + 7]));
            }
        }
        if (o.c_tma) {
            uint8_t* box = stg + (turn & 1u) * 2048;
            if (lane == 0) bulk_wait_group_read<1>();
            __syncwarp();
            uint4* to = reinterpret_cast<uint4*>(box + lane * 64);
#pragma unroll
            for (int j = 0; j < 4; ++j) to[j ^ ((lane >> 1) & 3)] = p.w[j];  // the 64-byte swizzle
            ++turn;
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && row0 < o.M) {
                tma_store_2d(o.map, smem_u32(box), col + h * kCols, row0);
                bulk_commit_group();
            }
            continue;
        }
        const int first = col + h * kCols;
        T* c = static_cast<T*>(o.C) + static_cast<long long>(row0) * o.ldc + first;
        if (sizeof(T) == 2 && o.width <= 2)
            put_rows<T, std::conditional_t<sizeof(T) == 2, uint16_t, uint32_t>>(c, o.ldc, o.M - row0, o.N - first, stg, lane, p);
        else if (o.width <= 4)
            put_rows<T, uint32_t>(c, o.ldc, o.M - row0, o.N - first, stg, lane, p);
        else
            put_rows<T, uint2>(c, o.ldc, o.M - row0, o.N - first, stg, lane, p);
    }
}

__device__ __forceinline__ void tmem_chunk(uint32_t addr, float (&f)[32])
{
    uint32_t r[32];
    tmem_ld_32x32b_x32(addr, r);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr)
{
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

// An epilogue warp's way with one unit's accumulator, from column acc of its lane quarter, in chunks of 32 columns
// beginning with chunk `first`; `early()` is called once that one has been read.  sums: where a pair that shares its
// tile leaves what it has (null otherwise).
template <int OUT, typename Early>
__device__ __forceinline__ void finish_unit(const Work& u, const BoxOut& out, uint8_t* stg, float4* sums, uint32_t acc, int first, int half,
                                            int q, int lane, uint32_t& turn, const Early& early)
{
    const int row0 = u.tm * 256 + half * 128 + q * 32;
    const uint32_t base = acc + (static_cast<uint32_t>(q * 32) << 16);
    const int chunks = u.cols / 32;
#pragma unroll 1
    for (int j = 0; j < chunks; ++j) {
        const int ch = (j + first) & (chunks - 1);
        float f[32];
        tmem_chunk(base + static_cast<uint32_t>(ch * 32), f);
        if (j == 0) early();
        const int col = u.n0 + ch * 32;
        if (sums != nullptr) {
            float4* to = sums + ch * 8 * 128 + q * 32 + lane;
#pragma unroll
            for (int i = 0; i < 8; ++i) to[i * 128] = make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
        } else if (col < out.N) {
            store_box<OUT>(out, stg, row0, lane, col, f, turn);
        }
    }
}

// The columns of a shared tile that fall to pair `part`, added from all pairs' shared memory: boxes of 32 x 32, by every
// warp of the CTA.  stg: staging of the first 16 warps, behind the sums.
template <int OUT>
__device__ __forceinline__ void finish_shared(const TileWork& w, const Work& u, const BoxOut& out, uint8_t* stg, const float4* sums,
                                              int part, int half, int warp, int warps, int lane)
{
    if (warp >= 16) return;
    const int first = 8 * part / w.pairs, chunks = 8 * (part + 1) / w.pairs - first;
    stg += warp * kF8EpiWarpBytes;
    uint32_t turn = 0;
#pragma unroll 1
    for (int i = warp; i < 4 * chunks; i += min(warps, 16)) {
        const int ch = first + (i >> 2), q = i & 3, col = u.n0 + ch * 32;
        if (col >= out.N) break;
        const uint32_t at = smem_u32(sums + ch * 8 * 128 + q * 32 + lane);
        float f[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) f[j] = 0.f;
#pragma unroll 1
        for (int s = 0; s < w.pairs; ++s) {
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
        store_box<OUT>(out, stg, u.tm * 256 + half * 128 + q * 32, lane, col, f, turn);
    }
    if (out.c_tma && lane == 0) bulk_wait_group_all();
}

// A place in a ring of stages and the parity of its barriers.
struct Ring {
    int at = 0, size;
    uint32_t phase = 0;
    __device__ __forceinline__ explicit Ring(int n) : size(n) {}
    __device__ __forceinline__ void next()
    {
        if (++at == size) {
            at = 0;
            phase ^= 1u;
        }
    }
};

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
    volatile uint32_t* gave_up = tmem_slot + 1;  // a wait of this CTA has

    const uint32_t bar0 = smem_u32(bars);
    auto full_bar = [&](int s) { return bar0 + 8u * s; };
    auto empty_bar = [&](int s) { return bar0 + 8u * (kF8Stages + s); };
    auto tfull_bar = [&](int a) { return bar0 + 8u * (2 * kF8Stages + a); };
    const uint32_t tempty_bar = bar0 + 8u * (2 * kF8Stages + 2);
    auto sf_full_bar = [&](int s) { return bar0 + 8u * (2 * kF8Stages + 3 + s); };
    auto sf_empty_bar = [&](int s) { return bar0 + 8u * (2 * kF8Stages + 3 + kF8SfSlots + s); };

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
            Ring r(kF8Stages);
            bool ok = true;
            for (int u = cluster_id; ok && u < units; u += num_clusters) {
                const Work w = work_unit(p.work, u, part);
                const int m0 = w.tm * 256 + half * 128, n0 = w.n0 + half * (w.cols / 2);
                const int b_boxes = w.cols / 128;  // of 64 rows of a B stored n x k
                const uint32_t bytes = kF8ABytes + (p.b_k ? w.cols / 2 * 256 : kF8BBytes);
                for (int st = w.st0; st < w.st1; ++st, r.next()) {
                    if (!mbar_wait(empty_bar(r.at), r.phase ^ 1u, p.timeout_ns, kErrWaitProducer, r.at)) {
                        ok = false;
                        break;
                    }
                    if (half == 0) mbar_arrive_expect_tx(full_bar(r.at), 2 * bytes);
                    const uint32_t bar = mapa_shared(full_bar(r.at), lead);
                    const uint32_t a_dst = smem_u32(sA + r.at * kF8ABytes), b_dst = smem_u32(sB + r.at * kF8BBytes);
                    const int k0 = st * 256;
                    tma_load_2d_pair(a_dst, &tmap_a, bar, k0, m0);
                    tma_load_2d_pair(a_dst + 128 * 128, &tmap_a, bar, k0 + 128, m0);
                    if (p.b_k) {
                        for (int i = 0; i < b_boxes; ++i) {
                            tma_load_2d_pair(b_dst + i * 64 * 128, &tmap_b, bar, k0, n0 + 64 * i);
                            tma_load_2d_pair(b_dst + (128 + i * 64) * 128, &tmap_b, bar, k0 + 128, n0 + 64 * i);
                        }
                    } else {
                        // 128 columns whatever their number in use: the width of a swizzled row
                        tma_load_2d_pair(b_dst, &tmap_b, bar, n0, k0);
                    }
                }
            }
            // the MMAs' signals to this CTA's barriers have all arrived before the CTA may exit
            for (int i = 0; ok && i < kF8Stages; ++i, r.next())
                ok = mbar_wait(empty_bar(r.at), r.phase ^ 1u, p.timeout_ns, kErrWaitTail, r.at);
            if (!ok) *gave_up = 1;
        }
    } else if (warp == 1) {
        // The whole warp walks through the loop and one lane issues: what the instructions take is then the same in every
        // lane and stays in uniform registers.  With one lane in the loop, issuing the eight MMAs of a stage took longer
        // than running them (the step that changed it, among others, took 8192 x 8192 x 8192 from 512 to 474 us in a loop).
        auto mma_loop = [&](auto b_k_tag) {
            constexpr bool B_K = decltype(b_k_tag)::value;
            constexpr uint32_t kIdesc = idesc_mxf8(256, 256, !B_K), kIdescHalf = idesc_mxf8(256, 128, !B_K);
            const bool one = elect_one();
            const uint32_t base = __shfl_sync(0xffffffffu, tmem, 0);
            const uint64_t a_desc = smem_desc_sw128(smem_u32(sA), 16, 1024);
            const uint64_t b_desc = B_K ? smem_desc_sw128(smem_u32(sB), 16, 1024) : smem_desc_sw128(smem_u32(sB), 256 * 128, 1024);
            const uint64_t sf_desc = smem_desc_rows16(smem_u32(sSf));
            Ring r(kF8Stages), sf(kF8SfSlots);
            int it = 0;
            uint32_t set = 0;
            bool ok = true;
            for (int u = cluster_id; ok && u < units; u += num_clusters, ++it) {
                const Work w = work_unit(p.work, u, part);
                // the unit before has left the columns the two accumulators share (and, before that, this one's)
                ok = mbar_wait_pair_warp(tempty_bar, static_cast<uint32_t>(it & 1) ^ 1u, p.timeout_ns, kErrWaitMma, 100);
                const uint32_t d = base + ((it & 1) ? kF8Acc1 : 0);
                for (int st = w.st0; ok && st < w.st1; ++st) {
                    const uint32_t sfa = base + kF8SfCol + set * 16, sfb = sfa + 4;
                    if ((st & 1) == 0) ok = mbar_wait_pair_warp(sf_full_bar(sf.at), sf.phase, p.timeout_ns, kErrWaitMma, 200 + sf.at);
                    ok = ok && mbar_wait_pair_warp(full_bar(r.at), r.phase, p.timeout_ns, kErrWaitMma, r.at);
                    if (!ok) break;
                    tc_fence_after();
                    const bool last = (st & 1) || st + 1 == w.st1;  // of its set of scales
                    if (one) {
                        if ((st & 1) == 0) {
                            const uint64_t src = sf_desc + static_cast<uint32_t>(sf.at) * (kF8SfBytes >> 4);
                            tmem_copy_scales_pair(sfa, src);
                            tmem_copy_scales_pair(sfb, src + (512 >> 4));
                            tmem_copy_scales_pair(sfb + 4, src + (1024 >> 4));
                        }
                        const uint64_t a = a_desc + static_cast<uint32_t>(r.at) * (kF8ABytes >> 4);
                        const uint64_t b = b_desc + static_cast<uint32_t>(r.at) * (kF8BBytes >> 4);
                        const int kk_end = min(8, (p.K - st * 256 + 31) / 32);
                        const uint32_t id0 = static_cast<uint32_t>(st & 1) * 2;  // scale bytes of this stage's two k-blocks
                        const uint32_t idesc = (w.cols == 256 ? kIdesc : kIdescHalf) | (id0 << 4) | (id0 << 29);
                        auto mma = [&](int kk) {
                            umma_mxf8_pair(d, a + (((kk >> 2) * (128 * 128) + (kk & 3) * 32) >> 4),
                                           b + ((B_K ? (kk >> 2) * (128 * 128) + (kk & 3) * 32 : kk * 32 * 128) >> 4),
                                           idesc + (kk >> 2) * ((1u << 4) | (1u << 29)), sfa, sfb, st != w.st0 || kk != 0);
                        };
                        if (kk_end == 8) {
#pragma unroll
                            for (int kk = 0; kk < 8; ++kk) mma(kk);
                        } else {
                            for (int kk = 0; kk < kk_end; ++kk) mma(kk);
                        }
                        umma_commit_pair(empty_bar(r.at), lead);
                        if (last) umma_commit_pair(sf_empty_bar(sf.at), lead);
                        if (st + 1 == w.st1) umma_commit_pair(tfull_bar(it & 1), lead);
                    }
                    __syncwarp();
                    r.next();
                    if (last) {
                        set ^= 1u;
                        sf.next();
                    }
                }
            }
            if (!ok) *gave_up = 1;
        };
        if (half == 0) {
            if (p.b_k)
                mma_loop(std::true_type{});
            else
                mma_loop(std::false_type{});
        }
    } else if (warp == 6) {
        Ring sf(kF8SfSlots);
        const int num_kb = (p.K + 127) / 128;
        bool ok = true;
        for (int u = cluster_id; ok && u < units; u += num_clusters) {
            const Work w = work_unit(p.work, u, part);
            const int m0 = w.tm * 256 + half * 128 + lane, n0 = w.n0 + lane;
            for (int kb = w.st0 * 2; kb < min(num_kb, w.st1 * 2); kb += 4, sf.next()) {
                uint32_t a[4], b[8];
                fetch_words(a, p.sa, m0, kb, num_kb - kb);
                fetch_words(b, p.sb, n0, kb, num_kb - kb);
                ok = mbar_wait_warp(sf_empty_bar(sf.at), sf.phase ^ 1u, p.timeout_ns, kErrWaitProducer, 200 + sf.at);
                if (!ok) break;
                uint4* dst = reinterpret_cast<uint4*>(sSf + sf.at * kF8SfBytes) + lane;
                dst[0] = make_uint4(a[0], a[1], a[2], a[3]);
                dst[32] = make_uint4(b[0], b[1], b[2], b[3]);
                dst[64] = make_uint4(b[4], b[5], b[6], b[7]);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive_pair(mapa_shared(sf_full_bar(sf.at), lead));
            }
        }
        // as above
        for (int i = 0; ok && i < kF8SfSlots; ++i, sf.next())
            ok = mbar_wait_warp(sf_empty_bar(sf.at), sf.phase ^ 1u, p.timeout_ns, kErrWaitTail, 200 + sf.at);
        if (!ok) *gave_up = 1;
    }

    const bool epilogue = warp >= 2 && warp < 6;
    const int q = warp & 3;  // the lane quarter an epilogue warp may read
    const BoxOut out{&tmap_c, p.C, p.ldc, p.M, p.N, p.c_tma, 0, p.c_width};
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
            // the shared columns first: the last 32 of accumulator 0, the first 32 of accumulator 1
            finish_unit<OUT>(w, out, stg, p.work.pairs > 1 ? sums : nullptr, tmem + (acc ? kF8Acc1 : 0), acc ? 0 : 7, half, q, lane, turn, [&] {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_pair(mapa_shared(tempty_bar, lead));
            });
            tc_fence_before();
        }
    }
    if (p.work.pairs > 1) {
        __syncthreads();
        cluster_sync_all();
        finish_shared<OUT>(p.work, work_unit(p.work, cluster_id, part), out, sA + 128 * 256 * 4, sums, part, half, warp, kF8Threads / 32, lane);
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
