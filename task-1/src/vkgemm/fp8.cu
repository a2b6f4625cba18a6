// C ABI of the 8-bit linear layer (include/vkgemm.h, "8-bit operands"): argument checks, kernel choice, launches.
// No call here allocates, synchronises or keeps anything between calls but kernel attributes and how many clusters fit, so all
// of them can be captured into CUDA graphs.
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstring>
#include <type_traits>

#include "vkgemm.h"
#include "fp8_gemm.cuh"
#include "fp8_rows.cuh"
#include "fp8_simt.cuh"
#include "fp8_thin.cuh"
#include "fp8_wgrad.cuh"
#include "vk_internal.h"

using namespace vk;

#define F8_CUDA_TRY(expr)                                                                             \
    do {                                                                                              \
        cudaError_t _e = (expr);                                                                      \
        if (_e != cudaSuccess) return set_error(VK_ERR_CUDA, "%s: %s", #expr, cudaGetErrorString(_e)); \
    } while (0)

namespace {

constexpr int64_t kMaxDim = (1LL << 31) - 256;

size_t bytes_of(int dtype) { return dtype == VK_DTYPE_F32 ? 4 : 2; }

bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

int use_device()
{
    int dev = 0;
    return current_device(&dev, nullptr);
}

int bad_size(const char* name, const char* what, int64_t v)
{
    return set_error(v < 0 ? VK_ERR_INVALID_ARGUMENT : VK_ERR_UNSUPPORTED, "%s: %s = %lld is out of range", name, what,
                     (long long)v);
}

// A leading dimension of 0 stands for the row's length.  That of a single row means nothing, so it becomes one that
// alignment cannot fail on.
int ld_of(const char* name, const char* what, int64_t given, int64_t row, int64_t rows, long long* out)
{
    *out = given ? given : row;
    if (given < 0 || *out < row)
        return set_error(VK_ERR_INVALID_ARGUMENT, "%s: %s = %lld is smaller than the row length %lld", name, what,
                         (long long)given, (long long)row);
    if (*out > (1LL << 40)) return set_error(VK_ERR_UNSUPPORTED, "%s: %s = %lld is too large", name, what, (long long)given);
    if (rows <= 1) *out = (*out + 15) / 16 * 16;
    return VK_OK;
}

// Addresses that an element of the type cannot have.
int element_aligned(const char* name, const char* what, const void* p, size_t esize)
{
    if (aligned(p, esize)) return VK_OK;
    return set_error(VK_ERR_ALIGNMENT, "%s: %s is not aligned to its elements of %zu bytes", name, what, esize);
}

// An output in an input's place whose rows would lie elsewhere.
int in_place(const char* name, const char* what, const void* out, long long ldo, const void* in, long long ldi, int64_t rows)
{
    if (out == nullptr || out != in || ldo == ldi || rows <= 1) return VK_OK;
    return set_error(VK_ERR_INVALID_ARGUMENT, "%s: %s in place needs the same leading dimension (%lld, not %lld)", name, what, ldi, ldo);
}

bool rows_at(const void* p, long long ld, size_t esize, size_t to)
{
    return aligned(p, to) && (static_cast<unsigned long long>(ld) * esize) % to == 0;
}

template <typename F>
int for_type(int dtype, const F& f)
{
    if (dtype == VK_DTYPE_F16) return f(__half());
    if (dtype == VK_DTYPE_BF16) return f(__nv_bfloat16());
    return f(float());
}

int launched()
{
    F8_CUDA_TRY(cudaGetLastError());
    return VK_OK;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encoder()
{
    static const EncodeTiledFn fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<EncodeTiledFn>(f);
    }();
    return fn;
}

// Map of a row-major matrix of 1-, 2- or 4-byte elements (bits are only moved): box_cols x box_rows boxes, zeros outside.
int make_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, long long ld, int esize, uint32_t box_cols,
             uint32_t box_rows, CUtensorMapSwizzle swizzle)
{
    const EncodeTiledFn encode = encoder();
    if (encode == nullptr) return set_error(VK_ERR_CUDA, "cuTensorMapEncodeTiled not available from the driver");
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * esize};
    const cuuint32_t box[2] = {box_cols, box_rows}, steps[2] = {1, 1};
    const CUtensorMapDataType type = esize == 1   ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                     : esize == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16
                                                  : CU_TENSOR_MAP_DATA_TYPE_UINT32;
    const CUresult r = encode(map, type, 2, const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return set_error(VK_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d) rows=%lld cols=%lld ld=%lld", (int)r,
                         (long long)rows, (long long)cols, ld);
    return VK_OK;
}

bool tma_ok(const void* p, long long ld, int esize) { return rows_at(p, ld, esize, 16) && ld * esize < (1LL << 40); }

int make_out_map(CUtensorMap* map, void* c, int64_t m, int64_t n, long long ldc, int dtype, int* c_tma, int* c_width)
{
    const int esize = static_cast<int>(bytes_of(dtype));
    *c_width = 16;
    while (*c_width > 1 && !rows_at(c, ldc, esize, *c_width)) *c_width /= 2;
    memset(map, 0, sizeof(*map));
    *c_tma = tma_ok(c, ldc, esize);
    if (!*c_tma) return VK_OK;
    return make_map(map, c, m, n, ldc, esize, 64 / esize, 32, CU_TENSOR_MAP_SWIZZLE_64B);
}

// Clusters of 2, 4, 6 and 8 CTAs of each kernel that fit on each device (0: not asked yet; the kernel's shared-memory
// attribute is set by then.  Kernels without clusters: 1 once that is set).
constexpr int kKernels = 32, kDevices = 64;
std::atomic<int> g_clusters[kKernels][kDevices][4];

template <typename Kernel>
int prepare_kernel(Kernel fn, int id, int smem, int threads, int clusters[4])
{
    int dev = 0;
    F8_CUDA_TRY(cudaGetDevice(&dev));
    std::atomic<int>* known = g_clusters[id][dev];
    if (known[0].load(std::memory_order_acquire) == 0) {
        F8_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        int sms = 0;
        F8_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
        for (int pairs = 4; pairs >= 1; --pairs) {
            cudaLaunchConfig_t cfg = {};
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = 2 * pairs;
            attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
            cfg.gridDim = dim3(2 * pairs * sms);
            cfg.blockDim = dim3(threads);
            cfg.dynamicSmemBytes = smem;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            int n = 0;
            F8_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, fn, &cfg));
            if (n <= 0 && pairs == 1) return set_error(VK_ERR_CUDA, "kernel cannot be resident (%d bytes of shared memory)", smem);
            known[pairs - 1].store(n, std::memory_order_release);
        }
    }
    for (int i = 0; i < 4; ++i) clusters[i] = known[i].load(std::memory_order_acquire);
    return VK_OK;
}

// For a kernel without clusters: its shared memory.
template <typename Kernel>
int prepare_smem(Kernel fn, int id, int smem)
{
    int dev = 0;
    F8_CUDA_TRY(cudaGetDevice(&dev));
    std::atomic<int>& known = g_clusters[id][dev][0];
    if (known.load(std::memory_order_acquire) != 0) return VK_OK;
    F8_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    known.store(1, std::memory_order_release);
    return VK_OK;
}

// Shares the tiles out.  Fewer tiles than clusters of several pairs: as many pairs to a tile as can all run at once, where
// that saves each of them kShareSaves stages: the join takes as long as 15 or so (512 x 4096 x 4096, two pairs, 8 stages
// saved: 16.1 us, unshared 13.6; k = 8192, 16 saved: 21.7 and 22.3; k = 16384: 33.4 and 38.9.  Weight gradients of
// 1000 x 1000, three pairs: 2048 tokens, 10 saved: 18.1 and 15.5; 3500, 18 saved: 20.8 and 22.0; 5000: 24.9 and 28.9).
// Otherwise the tiles of a last wave that at most half of the pairs would have are halved (4000 x 5120 x 3000 51.2 us,
// with whole tiles 52.8; weight gradient 8192 x 4096 x 4096 211 and 217).
constexpr int kShareSaves = 16;
int plan_work(TileWork& w, const int clusters[4])
{
    const long long tiles = static_cast<long long>(w.tiles_m) * w.tiles_n;
    const int grains = (w.stages + w.grain - 1) / w.grain;
    w.raster_group = 8;
    w.pairs = 1;
    w.halved = 0;
    for (int s = 4; s >= 2; --s)
        if (tiles <= clusters[s - 1] && w.stages - (grains + s - 1) / s * w.grain >= kShareSaves) {
            w.pairs = s;
            return static_cast<int>(tiles);
        }
    const long long rest = tiles % clusters[0];
    if (2 * rest <= clusters[0]) w.halved = static_cast<int>(rest);
    const int units = work_units(w);
    return units < clusters[0] ? units : clusters[0];
}

template <typename Kernel, typename... Args>
int launch_clusters(Kernel fn, int clusters, int cluster, int threads, int smem, cudaStream_t stream, const Args&... args)
{
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(clusters * cluster);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    F8_CUDA_TRY(cudaLaunchKernelEx(&cfg, fn, args...));
    return VK_OK;
}

}  // namespace

namespace vk {
void release_fp8_state()
{
    for (auto& kernel : g_clusters)
        for (auto& device : kernel) device[0].store(0, std::memory_order_release);
}

cudaError_t fp8_error_word(unsigned long long* word, bool clear)
{
    cudaError_t e = cudaMemcpyFromSymbol(word, g_device_error, sizeof(*word));
    const unsigned long long zero = 0;
    if (e == cudaSuccess && clear && *word != 0) e = cudaMemcpyToSymbol(g_device_error, &zero, sizeof(zero));
    return e;
}
}  // namespace vk

// ------------------------------------------------------------------------------------------
// Quantization
// ------------------------------------------------------------------------------------------
extern "C" int vk_quantize_fp8(const vk_quantize_fp8_args* a)
{
    static const char* const name = "vk_quantize_fp8";
    if (a == nullptr) return set_error(VK_ERR_INVALID_ARGUMENT, "%s: args is NULL", name);
    if (a->rows < 0 || a->rows > kMaxDim) return bad_size(name, "rows", a->rows);
    if (a->cols < 0 || a->cols > kMaxDim) return bad_size(name, "cols", a->cols);
    if (a->dtype != VK_DTYPE_F16 && a->dtype != VK_DTYPE_BF16 && a->dtype != VK_DTYPE_F32)
        return set_error(VK_ERR_INVALID_ARGUMENT, "%s: unknown dtype %d", name, a->dtype);
    if (a->scaling != VK_FP8_ROW && a->scaling != VK_FP8_TILE)
        return set_error(VK_ERR_INVALID_ARGUMENT, "%s: unknown scaling %d", name, a->scaling);
    QuantParams p;
    const int64_t blocks = (a->cols + 127) / 128;
    int rc = ld_of(name, "ldx", a->ldx, a->cols, a->rows, &p.ldx);
    if (rc == VK_OK) rc = ld_of(name, "ldq", a->ldq, a->cols, a->rows, &p.ldq);
    if (rc == VK_OK) rc = ld_of(name, "ld_scale", a->ld_scale, blocks, 2, &p.lds);
    if (rc != VK_OK) return rc;
    if (a->rows == 0 || a->cols == 0) return VK_OK;
    if (a->X == nullptr || a->Q == nullptr || a->scale == nullptr)
        return set_error(VK_ERR_INVALID_ARGUMENT, "%s: X, Q or scale is NULL", name);
    rc = element_aligned(name, "X", a->X, bytes_of(a->dtype));
    if (rc == VK_OK) rc = use_device();
    if (rc != VK_OK) return rc;
    p.x = a->X;
    p.q = static_cast<uint8_t*>(a->Q);
    p.scale = static_cast<uint8_t*>(a->scale);
    p.rows = a->rows;
    p.cols = static_cast<int>(a->cols);
    p.blocks = static_cast<int>(blocks);
    const bool vec = rows_at(a->X, p.ldx, bytes_of(a->dtype), 16) && rows_at(a->Q, p.ldq, 1, 8) && a->cols % 8 == 0;
    const cudaStream_t stream = static_cast<cudaStream_t>(a->stream);
    if (a->scaling == VK_FP8_TILE) {
        const int64_t tiles = (a->rows + 127) / 128 * blocks;
        if (tiles > kMaxDim) return set_error(VK_ERR_UNSUPPORTED, "%s: too many tiles", name);
        const unsigned grid = static_cast<unsigned>(tiles);
        return for_type(a->dtype, [&](auto t) {
            if (vec)
                quantize_tiles_kernel<decltype(t), true><<<grid, 256, 0, stream>>>(p);
            else
                quantize_tiles_kernel<decltype(t), false><<<grid, 256, 0, stream>>>(p);
            return launched();
        });
    }
    const int64_t ctas = (a->rows * ((blocks + 3) / 4) + 15) / 16;
    if (ctas > kMaxDim) return set_error(VK_ERR_UNSUPPORTED, "%s: too many blocks", name);
    const unsigned grid = static_cast<unsigned>(ctas);
    return for_type(a->dtype, [&](auto t) {
        if (vec)
            quantize_rows_kernel<decltype(t), true><<<grid, 256, 0, stream>>>(p);
        else
            quantize_rows_kernel<decltype(t), false><<<grid, 256, 0, stream>>>(p);
        return launched();
    });
}

// ------------------------------------------------------------------------------------------
// RMS norm
// ------------------------------------------------------------------------------------------
// Vectors of 8 columns to a thread.  Two from 65 vectors on: half the warps to add up and to launch (8000 x 1000 bf16 with a
// residual 8.8 us, with one 10.2; 8192 x 1600 14.9 and 16.6; at 200 columns, one 6.1 us and two 6.3).  Four only where two
// would not do: 4001 x 5120 21.5 us for 20.9, unaligned rows of 3333 49 us for 36, for their registers.
template <typename T, bool VEC>
static int launch_norm(const NormParams& p, int64_t rows, cudaStream_t stream)
{
    const unsigned grid = static_cast<unsigned>(rows);
    const int vectors = (p.cols + 127) / 128 * 16;  // of 8 columns, whole blocks
    if (vectors > 2048) {
        rmsnorm_fp8_long_kernel<T, VEC><<<grid, 512, 0, stream>>>(p);
        return launched();
    }
    const int nv = vectors > 1024 ? 4 : vectors > 64 ? 2 : 1;
    const int threads = ((vectors + nv - 1) / nv + 31) / 32 * 32;
    if (nv == 1)
        rmsnorm_fp8_kernel<T, 1, VEC><<<grid, threads, 0, stream>>>(p);
    else if (nv == 2)
        rmsnorm_fp8_kernel<T, 2, VEC><<<grid, threads, 0, stream>>>(p);
    else
        rmsnorm_fp8_kernel<T, 4, VEC><<<grid, threads, 0, stream>>>(p);
    return launched();
}

extern "C" int vk_rmsnorm_fp8(const vk_rmsnorm_fp8_args* a)
{
    static const char* const name = "vk_rmsnorm_fp8";
    if (a == nullptr) return set_error(VK_ERR_INVALID_ARGUMENT, "%s: args is NULL", name);
    if (a->rows < 0 || a->rows > kMaxDim) return bad_size(name, "rows", a->rows);
    if (a->cols < 1 || a->cols > kMaxDim) return set_error(VK_ERR_INVALID_ARGUMENT, "%s: cols = %lld is out of range", name, (long long)a->cols);
    if (a->dtype != VK_DTYPE_F16 && a->dtype != VK_DTYPE_BF16)
        return set_error(VK_ERR_INVALID_ARGUMENT, "%s: dtype must be VK_DTYPE_F16 or VK_DTYPE_BF16", name);
    if (!(a->eps >= 0.f)) return set_error(VK_ERR_INVALID_ARGUMENT, "%s: eps must be >= 0", name);
    NormParams p;
    const int64_t blocks = (a->cols + 127) / 128;
    int rc = ld_of(name, "ldx", a->ldx, a->cols, a->rows, &p.ldx);
    if (rc == VK_OK) rc = ld_of(name, "ld_residual", a->ld_residual, a->cols, a->rows, &p.ldr);
    if (rc == VK_OK) rc = ld_of(name, "ldq", a->ldq, a->cols, a->rows, &p.ldq);
    if (rc == VK_OK) rc = ld_of(name, "ld_scale", a->ld_scale, blocks, 2, &p.lds);
    if (rc == VK_OK) rc = ld_of(name, "ldh", a->ldh, a->cols, a->rows, &p.ldh);
    if (rc != VK_OK) return rc;
    if (a->rows == 0) return VK_OK;
    if (a->X == nullptr || a->weight == nullptr || a->Q == nullptr || a->scale == nullptr || a->rstd == nullptr)
        return set_error(VK_ERR_INVALID_ARGUMENT, "%s: X, weight, Q, scale or rstd is NULL", name);
    if ((a->residual == nullptr) != (a->H == nullptr))
        return set_error(VK_ERR_INVALID_ARGUMENT, "%s: H is given with a residual and only then", name);
    rc = element_aligned(name, "X", a->X, 2);
    if (rc == VK_OK) rc = element_aligned(name, "residual", a->residual, 2);
    if (rc == VK_OK) rc = element_aligned(name, "weight", a->weight, 2);
    if (rc == VK_OK) rc = element_aligned(name, "H", a->H, 2);
    if (rc == VK_OK) rc = element_aligned(name, "rstd", a->rstd, 4);
    if (rc == VK_OK) rc = in_place(name, "H", a->H, p.ldh, a->X, p.ldx, a->rows);
    if (rc == VK_OK) rc = in_place(name, "H", a->H, p.ldh, a->residual, p.ldr, a->rows);
    if (rc == VK_OK) rc = use_device();
    if (rc != VK_OK) return rc;
    p.x = a->X;
    p.residual = a->residual;
    p.weight = a->weight;
    p.q = static_cast<uint8_t*>(a->Q);
    p.scale = static_cast<uint8_t*>(a->scale);
    p.h = a->H;
    p.rstd = a->rstd;
    p.cols = static_cast<int>(a->cols);
    p.eps = a->eps;
    p.inv_cols = 1.0f / static_cast<float>(a->cols);
    const bool vec = rows_at(a->X, p.ldx, 2, 16) && (a->residual == nullptr || (rows_at(a->residual, p.ldr, 2, 16) && rows_at(a->H, p.ldh, 2, 16))) &&
                     aligned(a->weight, 16) && rows_at(a->Q, p.ldq, 1, 8) && a->cols % 8 == 0;
    const cudaStream_t stream = static_cast<cudaStream_t>(a->stream);
    return for_type(a->dtype, [&](auto t) {
        using T = std::conditional_t<std::is_same_v<decltype(t), __half>, __half, __nv_bfloat16>;
        return vec ? launch_norm<T, true>(p, a->rows, stream) : launch_norm<T, false>(p, a->rows, stream);
    });
}

// How the backward pass is laid out: threads of a CTA with nv vectors of 8 columns each (nv = 0: the kernel for any number
// of columns), and CTAs, each with a row of fp32 partial sums in the workspace.  Narrow rows need several CTAs on an SM
// to keep memory busy (8000 x 1000: 18.6 us, with one on each 46.9); where rows are few, a CTA has two (777 x 1000: 6.4 us, with four
// 7.2).
struct NormBackPlan {
    int nv, threads, per_sm;
    int64_t parts;
};

static NormBackPlan norm_backward_plan(int64_t rows, int64_t cols)
{
    NormBackPlan plan;
    plan.nv = cols <= 512 * 8 ? 1 : cols <= 512 * 16 ? 2 : 0;
    plan.threads = plan.nv ? static_cast<int>(((cols + 7) / 8 + plan.nv - 1) / plan.nv + 31) / 32 * 32 : 512;
    plan.per_sm = plan.nv != 1 ? 1 : plan.threads <= 128 ? 8 : plan.threads <= 256 ? 4 : 2;
    const int64_t most = 148 * plan.per_sm, wanted = (rows + 1) / 2;
    plan.parts = wanted < 148 ? (rows < 148 ? rows : 148) : wanted < most ? wanted : most;
    return plan;
}

extern "C" int vk_rmsnorm_fp8_workspace(int64_t rows, int64_t cols, size_t* bytes)
{
    static const char* const name = "vk_rmsnorm_fp8_workspace";
    if (bytes == nullptr) return set_error(VK_ERR_INVALID_ARGUMENT, "%s: bytes is NULL", name);
    if (rows < 0 || rows > kMaxDim) return bad_size(name, "rows", rows);
    if (cols < 1 || cols > kMaxDim) return set_error(VK_ERR_INVALID_ARGUMENT, "%s: cols = %lld is out of range", name, (long long)cols);
    *bytes = static_cast<size_t>(norm_backward_plan(rows, cols).parts) * static_cast<size_t>(cols) * sizeof(float);
    return VK_OK;
}

// Shared memory per SM that the rows in flight may take.
constexpr int kNormBackBytes = 208 * 1024;

template <typename T, int NV, bool VEC>
static int launch_norm_backward(NormBackParams p, int id, const NormBackPlan& plan, cudaStream_t stream)
{
    if (!VEC) {
        rmsnorm_fp8_backward_kernel<T, NV, VEC><<<static_cast<unsigned>(plan.parts), plan.threads, 0, stream>>>(p);
        return launched();
    }
    const int pitch = (p.cols * 2 + 127) / 128 * 128;
    const int rc = prepare_smem(rmsnorm_fp8_backward_kernel<T, NV, VEC>, id, kNormBackBytes / (NV == 1 ? 2 : 1));
    if (rc != VK_OK) return rc;
    p.stages = kNormBackBytes / plan.per_sm / (3 * pitch);
    if (p.stages > 8) p.stages = 8;
    rmsnorm_fp8_backward_kernel<T, NV, VEC><<<static_cast<unsigned>(plan.parts), plan.threads, p.stages * 3 * pitch, stream>>>(p);
    return launched();
}

extern "C" int vk_rmsnorm_fp8_backward(const vk_rmsnorm_fp8_backward_args* a)
{
    static const char* const name = "vk_rmsnorm_fp8_backward";
    if (a == nullptr) return set_error(VK_ERR_INVALID_ARGUMENT, "%s: args is NULL", name);
    size_t need = 0;
    NormBackParams p;
    if (a->rows < 0 || a->rows > kMaxDim) return bad_size(name, "rows", a->rows);
    if (a->cols < 1 || a->cols > kMaxDim) return set_error(VK_ERR_INVALID_ARGUMENT, "%s: cols = %lld is out of range", name, (long long)a->cols);
    if (a->dtype != VK_DTYPE_F16 && a->dtype != VK_DTYPE_BF16)
        return set_error(VK_ERR_INVALID_ARGUMENT, "%s: dtype must be VK_DTYPE_F16 or VK_DTYPE_BF16", name);
    int rc = ld_of(name, "lddy", a->lddy, a->cols, a->rows, &p.lddy);
    if (rc == VK_OK) rc = ld_of(name, "ldh", a->ldh, a->cols, a->rows, &p.ldh);
    if (rc == VK_OK) rc = ld_of(name, "ld_dres", a->ld_dres, a->cols, a->rows, &p.lddres);
    if (rc == VK_OK) rc = ld_of(name, "lddx", a->lddx, a->cols, a->rows, &p.lddx);
    if (rc == VK_OK) rc = vk_rmsnorm_fp8_workspace(a->rows, a->cols, &need);
    if (rc != VK_OK) return rc;
    if (a->dweight == nullptr) return set_error(VK_ERR_INVALID_ARGUMENT, "%s: dweight is NULL", name);
    if (a->rows > 0 && (a->dY == nullptr || a->H == nullptr || a->weight == nullptr || a->rstd == nullptr || a->dX == nullptr))
        return set_error(VK_ERR_INVALID_ARGUMENT, "%s: dY, H, weight, rstd or dX is NULL", name);
    if (a->rows > 0 && (a->workspace == nullptr || a->workspace_bytes < need || !aligned(a->workspace, 16)))
        return set_error(VK_ERR_INVALID_ARGUMENT, "%s: needs a workspace of %zu bytes, 16-byte aligned (vk_rmsnorm_fp8_workspace)", name, need);
    rc = element_aligned(name, "dweight", a->dweight, 4);
    if (rc == VK_OK) rc = element_aligned(name, "dY", a->dY, 2);
    if (rc == VK_OK) rc = element_aligned(name, "H", a->H, 2);
    if (rc == VK_OK) rc = element_aligned(name, "weight", a->weight, 2);
    if (rc == VK_OK) rc = element_aligned(name, "rstd", a->rstd, 4);
    if (rc == VK_OK) rc = element_aligned(name, "dres", a->dres, 2);
    if (rc == VK_OK) rc = element_aligned(name, "dX", a->dX, 2);
    if (rc == VK_OK) rc = in_place(name, "dX", a->dX, p.lddx, a->dY, p.lddy, a->rows);
    if (rc == VK_OK) rc = in_place(name, "dX", a->dX, p.lddx, a->dres, p.lddres, a->rows);
    if (rc == VK_OK) rc = use_device();
    if (rc != VK_OK) return rc;
    const cudaStream_t stream = static_cast<cudaStream_t>(a->stream);
    const NormBackPlan plan = norm_backward_plan(a->rows, a->cols);
    p.dy = a->dY;
    p.h = a->H;
    p.weight = a->weight;
    p.rstd = a->rstd;
    p.dres = a->dres;
    p.dx = a->dX;
    p.part = static_cast<float*>(a->workspace);
    p.rows = a->rows;
    p.cols = static_cast<int>(a->cols);
    p.stages = 0;
    p.inv_cols = 1.0f / static_cast<float>(a->cols);
    p.timeout_ns = wait_timeout_ns();
    const bool vec = rows_at(a->dY, p.lddy, 2, 16) && rows_at(a->H, p.ldh, 2, 16) && aligned(a->weight, 16) &&
                     (a->dres == nullptr || rows_at(a->dres, p.lddres, 2, 16)) && rows_at(a->dX, p.lddx, 2, 16) && a->cols % 8 == 0;
    if (a->rows > 0) {
        rc = for_type(a->dtype, [&](auto t) {
            using T = std::conditional_t<std::is_same_v<decltype(t), __half>, __half, __nv_bfloat16>;
            constexpr int kId = 9 + (std::is_same_v<T, __half> ? 0 : 2);
            if (plan.nv == 1)
                return vec ? launch_norm_backward<T, 1, true>(p, kId, plan, stream) : launch_norm_backward<T, 1, false>(p, 0, plan, stream);
            if (plan.nv == 2)
                return vec ? launch_norm_backward<T, 2, true>(p, kId + 1, plan, stream) : launch_norm_backward<T, 2, false>(p, 0, plan, stream);
            rmsnorm_fp8_backward_any_kernel<T><<<static_cast<unsigned>(plan.parts), 512, 0, stream>>>(p);
            return launched();
        });
        if (rc != VK_OK) return rc;
    }
    norm_weight_grad_kernel<<<static_cast<unsigned>((a->cols + 31) / 32), 1024, 0, stream>>>(
        p.part, static_cast<int>(plan.parts), p.cols, a->dweight);
    return launched();
}

// ------------------------------------------------------------------------------------------
// Products
// ------------------------------------------------------------------------------------------
template <typename LA, typename LB>
static int launch_simt(const LA& la, const LB& lb, const F8Output& out, int64_t m, int64_t n, int64_t k, cudaStream_t stream)
{
    const int64_t rows = (m + 63) / 64;  // of tiles
    const dim3 grid(static_cast<unsigned>((n + 63) / 64), static_cast<unsigned>(rows < 65535 ? rows : 65535));
    fp8_simt_kernel<<<grid, 256, 0, stream>>>(la, lb, out, m, n, k);
    return launched();
}

template <int OUT>
static int launch_gemm(F8GemmParams p, const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, cudaStream_t stream)
{
    int fit[4];
    const int rc = prepare_kernel(gemm_fp8_kernel<OUT>, OUT, kF8SmemBytes, kF8Threads, fit);
    if (rc != VK_OK) return rc;
    const int clusters = plan_work(p.work, fit);
    return launch_clusters(gemm_fp8_kernel<OUT>, clusters, 2 * p.work.pairs, kF8Threads, kF8SmemBytes, stream, ta, tb, tc, p);
}

template <int NPAD, int OUT>
static int launch_thin(ThinParams p, const CUtensorMap& tb, const CUtensorMap& ta, cudaStream_t stream)
{
    using Cfg = ThinCfg<NPAD>;
    constexpr int kId = 16 + 3 * (NPAD == 16 ? 0 : NPAD == 32 ? 1 : NPAD == 64 ? 2 : 3) + OUT;
    int fit[4];
    const int rc = prepare_kernel(gemm_fp8_thin_kernel<NPAD, OUT>, kId, Cfg::kSmemBytes, kThinThreads, fit);
    if (rc != VK_OK) return rc;
    // as many CTAs to a tile as can all run at once, with two k-blocks each at least
    const int tiles = static_cast<int>((static_cast<int64_t>(p.N) + 127) / 128), num_kb = (p.K + 127) / 128;
    p.slices = 1;
    for (int i = 3; i >= 0 && p.slices == 1; --i)
        if (tiles <= fit[i] && num_kb >= 4 * (i + 1)) p.slices = 2 * (i + 1);
    return launch_clusters(gemm_fp8_thin_kernel<NPAD, OUT>, tiles, p.slices, kThinThreads, Cfg::kSmemBytes, stream, tb, ta, p);
}

// Scales as the tensor-core kernels read them: strides per output index (or tile) and per k-block.
static ScaleSource scales(const void* p, long long ld, int64_t count, int scaling, bool along_row, int num_kb)
{
    ScaleSource s;
    s.p = static_cast<const uint8_t*>(p);
    s.si = along_row ? ld : 1;
    s.st = along_row ? 1 : ld;
    s.count = static_cast<int>(count);
    s.tile = scaling == VK_FP8_TILE;
    s.aligned = along_row && rows_at(p, ld, 1, 4);
    s.end = s.p + ((scaling == VK_FP8_TILE ? (count + 127) / 128 : count) - 1) * s.si + (num_kb - 1) * s.st + 1;
    return s;
}

extern "C" int vk_gemm_fp8(const vk_gemm_fp8_args* a)
{
    static const char* const name = "vk_gemm_fp8";
    if (a == nullptr) return set_error(VK_ERR_INVALID_ARGUMENT, "%s: args is NULL", name);
    if (a->m < 0 || a->m > kMaxDim) return bad_size(name, "m", a->m);
    if (a->n < 0 || a->n > kMaxDim) return bad_size(name, "n", a->n);
    if (a->k < 0 || a->k > kMaxDim) return bad_size(name, "k", a->k);
    if (a->dtype != VK_DTYPE_F16 && a->dtype != VK_DTYPE_BF16 && a->dtype != VK_DTYPE_F32)
        return set_error(VK_ERR_INVALID_ARGUMENT, "%s: unknown dtype %d", name, a->dtype);
    if (a->trans_b != 0 && a->trans_b != 1) return set_error(VK_ERR_INVALID_ARGUMENT, "%s: trans_b must be 0 or 1", name);
    if ((a->a_scaling != VK_FP8_ROW && a->a_scaling != VK_FP8_TILE) || (a->b_scaling != VK_FP8_ROW && a->b_scaling != VK_FP8_TILE))
        return set_error(VK_ERR_INVALID_ARGUMENT, "%s: unknown scaling", name);
    if (!a->trans_b && a->b_scaling != VK_FP8_TILE)
        return set_error(VK_ERR_UNSUPPORTED, "%s: a B that is stored k x n needs tile scales (a row's blocks run along n, not along the sum)", name);
    const int64_t kb = (a->k + 127) / 128;
    const int64_t b_row = a->trans_b ? a->k : a->n;
    long long lda, ldb, ldc, ldas, ldbs;
    int rc = ld_of(name, "lda", a->lda, a->k, a->m, &lda);
    if (rc == VK_OK) rc = ld_of(name, "ldb", a->ldb, b_row, a->trans_b ? a->n : a->k, &ldb);
    if (rc == VK_OK) rc = ld_of(name, "ldc", a->ldc, a->n, a->m, &ldc);
    if (rc == VK_OK) rc = ld_of(name, "ld_a_scale", a->ld_a_scale, kb, 2, &ldas);
    if (rc == VK_OK) rc = ld_of(name, "ld_b_scale", a->ld_b_scale, (b_row + 127) / 128, 2, &ldbs);
    if (rc != VK_OK) return rc;
    if (a->m == 0 || a->n == 0) return VK_OK;
    if (a->C == nullptr) return set_error(VK_ERR_INVALID_ARGUMENT, "%s: C is NULL", name);
    if (a->k > 0 && (a->A == nullptr || a->B == nullptr || a->a_scale == nullptr || a->b_scale == nullptr))
        return set_error(VK_ERR_INVALID_ARGUMENT, "%s: A, B, a_scale or b_scale is NULL", name);
    rc = element_aligned(name, "C", a->C, bytes_of(a->dtype));
    if (rc == VK_OK) rc = use_device();
    if (rc != VK_OK) return rc;
    const cudaStream_t stream = static_cast<cudaStream_t>(a->stream);
    if (a->k > 0 && tma_ok(a->A, lda, 1) && tma_ok(a->B, ldb, 1)) {
        const int num_kb = static_cast<int>(kb);
        // Up to 128 rows of A, B is the MMA's M: 128 x 4096 x 4096 9.6 us, as pairs of CTAs 15.4; 100 x 1000 x 1000 8.4 and 7.9;
        // 128 x 16384 x 4096 20.0 and 19.8.  (With B stored k x n there is no such kernel.)
        if (a->trans_b && a->m <= 128) {
            ThinParams p;
            p.M = static_cast<int>(a->m);
            p.N = static_cast<int>(a->n);
            p.K = static_cast<int>(a->k);
            p.sa = scales(a->a_scale, ldas, a->m, a->a_scaling, true, num_kb);
            p.sb = scales(a->b_scale, ldbs, a->n, a->b_scaling, true, num_kb);
            p.C = a->C;
            p.ldc = ldc;
            p.timeout_ns = wait_timeout_ns();
            const int npad = a->m <= 16 ? 16 : a->m <= 32 ? 32 : a->m <= 64 ? 64 : 128;
            CUtensorMap tb, ta;
            rc = make_map(&tb, a->B, a->n, a->k, ldb, 1, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B);
            if (rc == VK_OK) rc = make_map(&ta, a->A, a->m, a->k, lda, 1, 128, npad, CU_TENSOR_MAP_SWIZZLE_128B);
            if (rc != VK_OK) return rc;
            auto launch = [&](auto out) {
                constexpr int kOut = decltype(out)::value;
                return npad == 16   ? launch_thin<16, kOut>(p, tb, ta, stream)
                       : npad == 32 ? launch_thin<32, kOut>(p, tb, ta, stream)
                       : npad == 64 ? launch_thin<64, kOut>(p, tb, ta, stream)
                                    : launch_thin<128, kOut>(p, tb, ta, stream);
            };
            return a->dtype == VK_DTYPE_F16   ? launch(std::integral_constant<int, VK_DTYPE_F16>())
                   : a->dtype == VK_DTYPE_F32 ? launch(std::integral_constant<int, VK_DTYPE_F32>())
                                              : launch(std::integral_constant<int, VK_DTYPE_BF16>());
        }
        const int64_t tiles = (a->m + 255) / 256 * ((a->n + 255) / 256);
        if (tiles > kMaxDim) return set_error(VK_ERR_UNSUPPORTED, "%s: too many tiles", name);
        F8GemmParams p;
        p.M = static_cast<int>(a->m);
        p.N = static_cast<int>(a->n);
        p.K = static_cast<int>(a->k);
        p.work.tiles_m = static_cast<int>((a->m + 255) / 256);
        p.work.tiles_n = static_cast<int>((a->n + 255) / 256);
        p.work.n = p.N;
        p.work.stages = static_cast<int>((a->k + 255) / 256);
        p.work.grain = 2;  // a slice begins with a whole set of scales
        p.sa = scales(a->a_scale, ldas, a->m, a->a_scaling, true, num_kb);
        p.sb = scales(a->b_scale, ldbs, a->n, a->b_scaling, a->trans_b, num_kb);
        p.b_k = a->trans_b;
        p.C = a->C;
        p.ldc = ldc;
        p.timeout_ns = wait_timeout_ns();
        CUtensorMap ta, tb, tc;
        rc = make_map(&ta, a->A, a->m, a->k, lda, 1, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B);
        if (rc == VK_OK)
            rc = a->trans_b ? make_map(&tb, a->B, a->n, a->k, ldb, 1, 128, 64, CU_TENSOR_MAP_SWIZZLE_128B)
                            : make_map(&tb, a->B, a->k, a->n, ldb, 1, 128, 256, CU_TENSOR_MAP_SWIZZLE_128B);
        if (rc == VK_OK) rc = make_out_map(&tc, a->C, a->m, a->n, ldc, a->dtype, &p.c_tma, &p.c_width);
        if (rc != VK_OK) return rc;
        return a->dtype == VK_DTYPE_F16   ? launch_gemm<VK_DTYPE_F16>(p, ta, tb, tc, stream)
               : a->dtype == VK_DTYPE_F32 ? launch_gemm<VK_DTYPE_F32>(p, ta, tb, tc, stream)
                                          : launch_gemm<VK_DTYPE_BF16>(p, ta, tb, tc, stream);
    }
    const int tile_a = a->a_scaling == VK_FP8_TILE ? 7 : 0, tile_b = a->b_scaling == VK_FP8_TILE ? 7 : 0;
    const F8Operand fa{static_cast<const uint8_t*>(a->A), static_cast<const uint8_t*>(a->a_scale), lda, 1, ldas, 1, tile_a, 7};
    F8Operand fb{static_cast<const uint8_t*>(a->B), static_cast<const uint8_t*>(a->b_scale), ldb, 1, ldbs, 1, tile_b, 7};
    if (!a->trans_b) {
        fb.qi = 1;
        fb.qt = ldb;
        fb.si = 1;
        fb.st = ldbs;
    }
    const F8Output out{a->C, ldc, a->dtype, 0};
    return launch_simt(fa, fb, out, a->m, a->n, a->k, stream);
}

template <typename T, int OUT>
static int launch_wgrad(WgradParams p, const CUtensorMap& ta, const CUtensorMap& tc, cudaStream_t stream)
{
    constexpr int kId = 3 + 3 * (std::is_same_v<T, __half> ? 0 : 1) + OUT;
    int fit[4];
    const int rc = prepare_kernel(wgrad_fp8_kernel<T, OUT>, kId, kWgSmemBytes, kWgThreads, fit);
    if (rc != VK_OK) return rc;
    const int clusters = plan_work(p.work, fit);
    return launch_clusters(wgrad_fp8_kernel<T, OUT>, clusters, 2 * p.work.pairs, kWgThreads, kWgSmemBytes, stream, ta, tc, p);
}

extern "C" int vk_wgrad_fp8(const vk_wgrad_fp8_args* a)
{
    static const char* const name = "vk_wgrad_fp8";
    if (a == nullptr) return set_error(VK_ERR_INVALID_ARGUMENT, "%s: args is NULL", name);
    if (a->tokens < 0 || a->tokens > kMaxDim) return bad_size(name, "tokens", a->tokens);
    if (a->n < 0 || a->n > kMaxDim) return bad_size(name, "n", a->n);
    if (a->k < 0 || a->k > kMaxDim) return bad_size(name, "k", a->k);
    if (a->dtype != VK_DTYPE_F16 && a->dtype != VK_DTYPE_BF16)
        return set_error(VK_ERR_INVALID_ARGUMENT, "%s: dtype must be VK_DTYPE_F16 or VK_DTYPE_BF16", name);
    if (a->out_dtype != VK_DTYPE_F16 && a->out_dtype != VK_DTYPE_BF16 && a->out_dtype != VK_DTYPE_F32)
        return set_error(VK_ERR_INVALID_ARGUMENT, "%s: unknown out_dtype %d", name, a->out_dtype);
    if (a->accumulate != 0 && a->accumulate != 1) return set_error(VK_ERR_INVALID_ARGUMENT, "%s: accumulate must be 0 or 1", name);
    long long lddy, ldx, ldxs, lddw;
    int rc = ld_of(name, "lddy", a->lddy, a->n, a->tokens, &lddy);
    if (rc == VK_OK) rc = ld_of(name, "ldx", a->ldx, a->k, a->tokens, &ldx);
    if (rc == VK_OK) rc = ld_of(name, "ld_x_scale", a->ld_x_scale, (a->k + 127) / 128, 2, &ldxs);
    if (rc == VK_OK) rc = ld_of(name, "lddw", a->lddw, a->k, a->n, &lddw);
    if (rc != VK_OK) return rc;
    if (a->n == 0 || a->k == 0) return VK_OK;
    if (a->dW == nullptr) return set_error(VK_ERR_INVALID_ARGUMENT, "%s: dW is NULL", name);
    if (a->tokens > 0 && (a->dY == nullptr || a->X == nullptr || a->x_scale == nullptr))
        return set_error(VK_ERR_INVALID_ARGUMENT, "%s: dY, X or x_scale is NULL", name);
    rc = element_aligned(name, "dY", a->dY, 2);
    if (rc == VK_OK) rc = element_aligned(name, "dW", a->dW, bytes_of(a->out_dtype));
    if (rc == VK_OK) rc = use_device();
    if (rc != VK_OK) return rc;
    const cudaStream_t stream = static_cast<cudaStream_t>(a->stream);
    if (a->tokens > 0 && tma_ok(a->dY, lddy, 2) && tma_ok(a->X, ldx, 1)) {
        const int64_t tiles = (a->n + 255) / 256 * ((a->k + 255) / 256);
        if (tiles > kMaxDim) return set_error(VK_ERR_UNSUPPORTED, "%s: too many tiles", name);
        WgradParams p;
        p.M = static_cast<int>(a->n);
        p.N = static_cast<int>(a->k);
        p.K = static_cast<int>(a->tokens);
        p.work.tiles_m = static_cast<int>((a->n + 255) / 256);
        p.work.tiles_n = static_cast<int>((a->k + 255) / 256);
        p.work.n = p.N;
        p.work.stages = static_cast<int>((a->tokens + kWgBK - 1) / kWgBK);
        p.work.grain = 1;
        p.X = static_cast<const uint8_t*>(a->X);
        p.ldx = ldx;
        p.scale = static_cast<const uint8_t*>(a->x_scale);
        p.lds = ldxs;
        p.C = a->dW;
        p.ldc = lddw;
        p.accumulate = a->accumulate;
        p.timeout_ns = wait_timeout_ns();
        CUtensorMap ta, tc;
        rc = make_map(&ta, a->dY, a->tokens, a->n, lddy, 2, 64, kWgBK, CU_TENSOR_MAP_SWIZZLE_128B);
        if (rc == VK_OK) rc = make_out_map(&tc, a->dW, a->n, a->k, lddw, a->out_dtype, &p.c_tma, &p.c_width);
        if (rc != VK_OK) return rc;
        return for_type(a->dtype, [&](auto t) {
            using T = std::conditional_t<std::is_same_v<decltype(t), __half>, __half, __nv_bfloat16>;
            return a->out_dtype == VK_DTYPE_F16   ? launch_wgrad<T, VK_DTYPE_F16>(p, ta, tc, stream)
                   : a->out_dtype == VK_DTYPE_F32 ? launch_wgrad<T, VK_DTYPE_F32>(p, ta, tc, stream)
                                                  : launch_wgrad<T, VK_DTYPE_BF16>(p, ta, tc, stream);
        });
    }
    const F8Operand fx{static_cast<const uint8_t*>(a->X), static_cast<const uint8_t*>(a->x_scale), 1, ldx, 1, ldxs, 7, 0};
    const F8Output out{a->dW, lddw, a->out_dtype, a->accumulate};
    if (a->dtype == VK_DTYPE_F16) {
        const HalfOperand<__half> fy{static_cast<const __half*>(a->dY), 1, lddy};
        return launch_simt(fy, F8OperandAs<__half>{fx}, out, a->n, a->k, a->tokens, stream);
    }
    const HalfOperand<__nv_bfloat16> fy{static_cast<const __nv_bfloat16*>(a->dY), 1, lddy};
    return launch_simt(fy, F8OperandAs<__nv_bfloat16>{fx}, out, a->n, a->k, a->tokens, stream);
}
