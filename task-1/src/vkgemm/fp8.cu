// C ABI of the 8-bit linear layer (include/vkgemm.h, "8-bit operands"): argument checks, kernel choice, launches.
// No call here allocates, keeps anything between calls but tensor maps and kernel attributes, or synchronises, so all
// of them can be captured into CUDA graphs.
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstring>

#include "vkgemm.h"
#include "fp8_rows.cuh"
#include "fp8_simt.cuh"
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

// A leading dimension of 0 stands for the row's length.
int ld_of(const char* name, const char* what, int64_t given, int64_t row, long long* out)
{
    *out = given ? given : row;
    if (given < 0 || *out < row)
        return set_error(VK_ERR_INVALID_ARGUMENT, "%s: %s = %lld is smaller than the row length %lld", name, what,
                         (long long)given, (long long)row);
    if (*out > (1LL << 40)) return set_error(VK_ERR_UNSUPPORTED, "%s: %s = %lld is too large", name, what, (long long)given);
    return VK_OK;
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

}  // namespace

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
    int rc = ld_of(name, "ldx", a->ldx, a->cols, &p.ldx);
    if (rc == VK_OK) rc = ld_of(name, "ldq", a->ldq, a->cols, &p.ldq);
    if (rc == VK_OK) rc = ld_of(name, "ld_scale", a->ld_scale, blocks, &p.lds);
    if (rc != VK_OK) return rc;
    if (a->rows == 0 || a->cols == 0) return VK_OK;
    if (a->X == nullptr || a->Q == nullptr || a->scale == nullptr)
        return set_error(VK_ERR_INVALID_ARGUMENT, "%s: X, Q or scale is NULL", name);
    rc = use_device();
    if (rc != VK_OK) return rc;
    p.x = a->X;
    p.q = static_cast<uint8_t*>(a->Q);
    p.scale = static_cast<uint8_t*>(a->scale);
    p.rows = a->rows;
    p.cols = static_cast<int>(a->cols);
    p.blocks = static_cast<int>(blocks);
    p.vec_x = rows_at(a->X, p.ldx, bytes_of(a->dtype), 16);
    p.vec_q = rows_at(a->Q, p.ldq, 1, 8);
    const cudaStream_t stream = static_cast<cudaStream_t>(a->stream);
    if (a->scaling == VK_FP8_TILE) {
        const int64_t tiles = (a->rows + 127) / 128 * blocks;
        if (tiles > kMaxDim) return set_error(VK_ERR_UNSUPPORTED, "%s: too many tiles", name);
        return for_type(a->dtype, [&](auto t) {
            quantize_tiles_kernel<decltype(t)><<<static_cast<unsigned>(tiles), 256, 0, stream>>>(p);
            return launched();
        });
    }
    const int64_t need = (a->rows * blocks + 15) / 16, most = 148 * 32;
    return for_type(a->dtype, [&](auto t) {
        quantize_rows_kernel<decltype(t)><<<static_cast<unsigned>(need < most ? need : most), 256, 0, stream>>>(p);
        return launched();
    });
}

// ------------------------------------------------------------------------------------------
// RMS norm
// ------------------------------------------------------------------------------------------
template <typename T>
static int launch_norm(const NormParams& p, int64_t rows, cudaStream_t stream)
{
    const unsigned grid = static_cast<unsigned>(rows);
    if (p.cols <= 1024)
        rmsnorm_fp8_kernel<T, 128, 1><<<grid, 128, 0, stream>>>(p);
    else if (p.cols <= 2048)
        rmsnorm_fp8_kernel<T, 256, 1><<<grid, 256, 0, stream>>>(p);
    else if (p.cols <= 4096)
        rmsnorm_fp8_kernel<T, 256, 2><<<grid, 256, 0, stream>>>(p);
    else if (p.cols <= 8192)
        rmsnorm_fp8_kernel<T, 512, 2><<<grid, 512, 0, stream>>>(p);
    else
        rmsnorm_fp8_kernel<T, 512, 0><<<grid, 512, 0, stream>>>(p);
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
    int rc = ld_of(name, "ldx", a->ldx, a->cols, &p.ldx);
    if (rc == VK_OK) rc = ld_of(name, "ld_residual", a->ld_residual, a->cols, &p.ldr);
    if (rc == VK_OK) rc = ld_of(name, "ldq", a->ldq, a->cols, &p.ldq);
    if (rc == VK_OK) rc = ld_of(name, "ld_scale", a->ld_scale, blocks, &p.lds);
    if (rc == VK_OK) rc = ld_of(name, "ldh", a->ldh, a->cols, &p.ldh);
    if (rc != VK_OK) return rc;
    if (a->rows == 0) return VK_OK;
    if (a->X == nullptr || a->weight == nullptr || a->Q == nullptr || a->scale == nullptr || a->rstd == nullptr)
        return set_error(VK_ERR_INVALID_ARGUMENT, "%s: X, weight, Q, scale or rstd is NULL", name);
    if ((a->residual == nullptr) != (a->H == nullptr))
        return set_error(VK_ERR_INVALID_ARGUMENT, "%s: H is given with a residual and only then", name);
    rc = use_device();
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
    p.vec_x = rows_at(a->X, p.ldx, 2, 16);
    p.vec_r = rows_at(a->residual, p.ldr, 2, 16);
    p.vec_w = aligned(a->weight, 16);
    p.vec_q = rows_at(a->Q, p.ldq, 1, 8);
    p.vec_h = rows_at(a->H, p.ldh, 2, 16);
    const cudaStream_t stream = static_cast<cudaStream_t>(a->stream);
    return a->dtype == VK_DTYPE_F16 ? launch_norm<__half>(p, a->rows, stream) : launch_norm<__nv_bfloat16>(p, a->rows, stream);
}

// CTAs of the backward pass, each with a row of fp32 partial sums in the workspace: two per SM of B200.
static int64_t norm_backward_parts(int64_t rows) { return rows < 296 ? rows : 296; }

extern "C" int vk_rmsnorm_fp8_workspace(int64_t rows, int64_t cols, size_t* bytes)
{
    static const char* const name = "vk_rmsnorm_fp8_workspace";
    if (bytes == nullptr) return set_error(VK_ERR_INVALID_ARGUMENT, "%s: bytes is NULL", name);
    if (rows < 0 || rows > kMaxDim) return bad_size(name, "rows", rows);
    if (cols < 1 || cols > kMaxDim) return set_error(VK_ERR_INVALID_ARGUMENT, "%s: cols = %lld is out of range", name, (long long)cols);
    *bytes = static_cast<size_t>(norm_backward_parts(rows)) * static_cast<size_t>(cols) * sizeof(float);
    return VK_OK;
}

template <typename T>
static int launch_norm_backward(const NormBackParams& p, unsigned grid, cudaStream_t stream)
{
    if (p.cols <= 1024)
        rmsnorm_fp8_backward_kernel<T, 128, 1><<<grid, 128, 0, stream>>>(p);
    else if (p.cols <= 2048)
        rmsnorm_fp8_backward_kernel<T, 256, 1><<<grid, 256, 0, stream>>>(p);
    else if (p.cols <= 4096)
        rmsnorm_fp8_backward_kernel<T, 512, 1><<<grid, 512, 0, stream>>>(p);
    else if (p.cols <= 8192)
        rmsnorm_fp8_backward_kernel<T, 512, 2><<<grid, 512, 0, stream>>>(p);
    else
        rmsnorm_fp8_backward_kernel<T, 512, 0><<<grid, 512, 0, stream>>>(p);
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
    int rc = ld_of(name, "lddy", a->lddy, a->cols, &p.lddy);
    if (rc == VK_OK) rc = ld_of(name, "ldh", a->ldh, a->cols, &p.ldh);
    if (rc == VK_OK) rc = ld_of(name, "ld_dres", a->ld_dres, a->cols, &p.lddres);
    if (rc == VK_OK) rc = ld_of(name, "lddx", a->lddx, a->cols, &p.lddx);
    if (rc == VK_OK) rc = vk_rmsnorm_fp8_workspace(a->rows, a->cols, &need);
    if (rc != VK_OK) return rc;
    if (a->dweight == nullptr) return set_error(VK_ERR_INVALID_ARGUMENT, "%s: dweight is NULL", name);
    if (a->rows > 0 && (a->dY == nullptr || a->H == nullptr || a->weight == nullptr || a->rstd == nullptr || a->dX == nullptr))
        return set_error(VK_ERR_INVALID_ARGUMENT, "%s: dY, H, weight, rstd or dX is NULL", name);
    if (a->rows > 0 && (a->workspace == nullptr || a->workspace_bytes < need || !aligned(a->workspace, 16)))
        return set_error(VK_ERR_INVALID_ARGUMENT, "%s: needs a workspace of %zu bytes, 16-byte aligned (vk_rmsnorm_fp8_workspace)", name, need);
    rc = use_device();
    if (rc != VK_OK) return rc;
    const cudaStream_t stream = static_cast<cudaStream_t>(a->stream);
    const int64_t parts = norm_backward_parts(a->rows);
    p.dy = a->dY;
    p.h = a->H;
    p.weight = a->weight;
    p.rstd = a->rstd;
    p.dres = a->dres;
    p.dx = a->dX;
    p.part = static_cast<float*>(a->workspace);
    p.rows = a->rows;
    p.cols = static_cast<int>(a->cols);
    p.vec_dy = rows_at(a->dY, p.lddy, 2, 16);
    p.vec_h = rows_at(a->H, p.ldh, 2, 16);
    p.vec_w = aligned(a->weight, 16);
    p.vec_dres = rows_at(a->dres, p.lddres, 2, 16);
    p.vec_dx = rows_at(a->dX, p.lddx, 2, 16);
    if (a->rows > 0) {
        rc = a->dtype == VK_DTYPE_F16 ? launch_norm_backward<__half>(p, static_cast<unsigned>(parts), stream)
                                      : launch_norm_backward<__nv_bfloat16>(p, static_cast<unsigned>(parts), stream);
        if (rc != VK_OK) return rc;
    }
    norm_weight_grad_kernel<<<static_cast<unsigned>((a->cols + 31) / 32), 256, 0, stream>>>(
        p.part, static_cast<int>(parts), p.cols, a->dweight);
    return launched();
}

// ------------------------------------------------------------------------------------------
// Products
// ------------------------------------------------------------------------------------------
template <typename LA, typename LB>
static int launch_simt(const LA& la, const LB& lb, const F8Output& out, int64_t m, int64_t n, int64_t k, cudaStream_t stream)
{
    const dim3 grid(static_cast<unsigned>((n + 63) / 64), static_cast<unsigned>((m + 63) / 64));
    if (grid.y > 65535u) return set_error(VK_ERR_UNSUPPORTED, "m too large for the CUDA-core kernel");
    fp8_simt_kernel<<<grid, 256, 0, stream>>>(la, lb, out, m, n, k);
    return launched();
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
    int rc = ld_of(name, "lda", a->lda, a->k, &lda);
    if (rc == VK_OK) rc = ld_of(name, "ldb", a->ldb, b_row, &ldb);
    if (rc == VK_OK) rc = ld_of(name, "ldc", a->ldc, a->n, &ldc);
    if (rc == VK_OK) rc = ld_of(name, "ld_a_scale", a->ld_a_scale, kb, &ldas);
    if (rc == VK_OK) rc = ld_of(name, "ld_b_scale", a->ld_b_scale, (b_row + 127) / 128, &ldbs);
    if (rc != VK_OK) return rc;
    if (a->m == 0 || a->n == 0) return VK_OK;
    if (a->C == nullptr) return set_error(VK_ERR_INVALID_ARGUMENT, "%s: C is NULL", name);
    if (a->k > 0 && (a->A == nullptr || a->B == nullptr || a->a_scale == nullptr || a->b_scale == nullptr))
        return set_error(VK_ERR_INVALID_ARGUMENT, "%s: A, B, a_scale or b_scale is NULL", name);
    rc = use_device();
    if (rc != VK_OK) return rc;
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
    return launch_simt(fa, fb, out, a->m, a->n, a->k, static_cast<cudaStream_t>(a->stream));
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
    int rc = ld_of(name, "lddy", a->lddy, a->n, &lddy);
    if (rc == VK_OK) rc = ld_of(name, "ldx", a->ldx, a->k, &ldx);
    if (rc == VK_OK) rc = ld_of(name, "ld_x_scale", a->ld_x_scale, (a->k + 127) / 128, &ldxs);
    if (rc == VK_OK) rc = ld_of(name, "lddw", a->lddw, a->k, &lddw);
    if (rc != VK_OK) return rc;
    if (a->n == 0 || a->k == 0) return VK_OK;
    if (a->dW == nullptr) return set_error(VK_ERR_INVALID_ARGUMENT, "%s: dW is NULL", name);
    if (a->tokens > 0 && (a->dY == nullptr || a->X == nullptr || a->x_scale == nullptr))
        return set_error(VK_ERR_INVALID_ARGUMENT, "%s: dY, X or x_scale is NULL", name);
    rc = use_device();
    if (rc != VK_OK) return rc;
    const cudaStream_t stream = static_cast<cudaStream_t>(a->stream);
    const F8Operand fx{static_cast<const uint8_t*>(a->X), static_cast<const uint8_t*>(a->x_scale), 1, ldx, 1, ldxs, 7, 0};
    const F8Output out{a->dW, lddw, a->out_dtype, a->accumulate};
    if (a->dtype == VK_DTYPE_F16) {
        const HalfOperand<__half> fy{static_cast<const __half*>(a->dY), 1, lddy};
        return launch_simt(fy, F8OperandAs<__half>{fx}, out, a->n, a->k, a->tokens, stream);
    }
    const HalfOperand<__nv_bfloat16> fy{static_cast<const __nv_bfloat16*>(a->dY), 1, lddy};
    return launch_simt(fy, F8OperandAs<__nv_bfloat16>{fx}, out, a->n, a->k, a->tokens, stream);
}
