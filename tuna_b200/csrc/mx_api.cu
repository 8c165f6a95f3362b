// C ABI of the microscaled 4-bit operators: argument checks, workspace layout, dispatch.
#include <algorithm>
#include "launchers.h"
#include "mx_format.cuh"

namespace tuna {

static bool aligned_to(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
static bool is_number_type(int t) { return t == TUNA_FP16 || t == TUNA_BF16 || t == TUNA_FP32; }
static int type_bytes(int t) { return t == TUNA_FP32 ? 4 : 2; }

// Sizes in 32 bits leave room for being rounded up to whole tiles; the quantizers' grids have the chunks, by fours, in y.
static bool too_long(int rows, int k) { return rows > 0x7fffffff - 1023 || k > 65535 * 4 * kMxChunk; }

// rows x k elements, `batch` of them: what the kernels number in 64 bits, but grids in 32
static int check_matrix(int rows, int k, int batch)
{
    if (rows < 1 || k < 1 || batch < 1 || k % kMxBlock) return TUNA_ERR_BAD_SHAPE;
    if (too_long(rows, k) || (double)rows * k * batch > (double)(1ll << 41) || (double)rows * batch > (double)(1ll << 31)) return TUNA_ERR_TOO_LARGE;
    return TUNA_OK;
}

// The workspace holds the codes and scales of tokens that a launch before the product quantizes.
struct MxWorkspace {
    size_t scales, total;
};
static MxWorkspace mx_workspace(int m, int n, int k, int experts, int x_type, bool grouped, int sm_count)
{
    MxWorkspace w = {0, 0};
    if (!mx_gemm_takes(m, n, k, experts, x_type, grouped, sm_count)) {
        w.scales = (size_t)div_up(k, kMxChunk) * n * kMxChunkBytes;
        w.total = w.scales + (size_t)div_up(k, kMxScaleCols) * n * 4;
    }
    return w;
}

static int mx_product(const void *x, int x_type, const void *xs, const void *q, const void *s, const void *offsets, void *o, int o_type, int m, int n, int k,
                      int experts, void *workspace, size_t workspace_bytes, void *stream)
{
    const bool packed = x_type == TUNA_MXFP4;
    if (!x || !q || !s || !o || (packed && !xs)) return TUNA_ERR_NULL_POINTER;
    if (m < 1 || m % 8 || n < 1 || k < 1 || k % kMxBlock || experts < 1) return TUNA_ERR_BAD_SHAPE;
    if ((!packed && x_type != TUNA_FP16 && x_type != TUNA_BF16) || !is_number_type(o_type)) return TUNA_ERR_BAD_CONFIG;
    if (too_long(m, k) || too_long(n, k) || experts > TUNA_MX_MAX_EXPERTS || (double)experts * m * k > (double)(1ll << 41) || (double)n * k > (double)(1ll << 41)) return TUNA_ERR_TOO_LARGE;
    if (!aligned_to(x, 16) || !aligned_to(q, 16) || !aligned_to(s, 16) || !aligned_to(o, 16) || !aligned_to(xs, 4) || !aligned_to(offsets, 4) || !aligned_to(workspace, 16))
        return TUNA_ERR_MISALIGNED;
    const int sms = device_sm_count();
    const MxWorkspace w = mx_workspace(m, n, k, experts, x_type, offsets != nullptr, sms);
    if (w.total > 0 && (!workspace || workspace_bytes < w.total)) return TUNA_ERR_WORKSPACE;
    MxGemmArgs a;
    a.x = x; a.xs = xs; a.q = q; a.s = s; a.offsets = offsets; a.o = o;
    a.m = m; a.n = n; a.k = k; a.experts = experts; a.x_type = x_type; a.o_type = o_type;
    a.stream = (cudaStream_t)stream; a.sm_count = sms;
    a.numbers = nullptr;
    if (w.total > 0) {
        a.numbers = x;
        a.x = workspace;
        a.xs = (uint8_t *)workspace + w.scales;
    }
    return launch_mx_gemm(a);
}

}  // namespace tuna

using namespace tuna;

extern "C" int tuna_mx_quantize(const void *x, int x_type, long long row_stride, void *q, void *s, int rows, int k, int batch, void *stream)
{
    if (!x || !q || !s) return TUNA_ERR_NULL_POINTER;
    const int st = check_matrix(rows, k, batch);
    if (st != TUNA_OK) return st;
    if (!is_number_type(x_type)) return TUNA_ERR_BAD_CONFIG;
    if (row_stride < k || row_stride > 1ll << 40) return TUNA_ERR_BAD_SHAPE;
    if (!aligned_to(x, 16) || (row_stride * type_bytes(x_type)) % 16 || !aligned_to(q, 16) || !aligned_to(s, 16)) return TUNA_ERR_MISALIGNED;
    return launch_mx_quantize(x, x_type, row_stride, q, s, rows, k, batch, (cudaStream_t)stream) == cudaSuccess ? TUNA_OK : TUNA_ERR_LAUNCH;
}

extern "C" int tuna_mx_dequant(const void *q, const void *s, void *o, int o_type, int rows, int k, int batch, void *stream)
{
    if (!q || !s || !o) return TUNA_ERR_NULL_POINTER;
    const int st = check_matrix(rows, k, batch);
    if (st != TUNA_OK) return st;
    if (!is_number_type(o_type)) return TUNA_ERR_BAD_CONFIG;
    if (!aligned_to(q, 16) || !aligned_to(s, 4) || !aligned_to(o, 16)) return TUNA_ERR_MISALIGNED;
    return launch_mx_dequant(q, s, o, o_type, rows, k, batch, (cudaStream_t)stream) == cudaSuccess ? TUNA_OK : TUNA_ERR_LAUNCH;
}

extern "C" int tuna_mx_matmul(const void *x, int x_type, const void *xs, const void *q, const void *s, void *o, int o_type, int m, int n, int k, void *workspace,
                              size_t workspace_bytes, void *stream)
{
    return mx_product(x, x_type, xs, q, s, nullptr, o, o_type, m, n, k, 1, workspace, workspace_bytes, stream);
}

extern "C" int tuna_mx_matmul_grouped(const void *x, int x_type, const void *xs, const void *q, const void *s, const void *offsets, void *o, int o_type, int m, int n,
                                      int k, int experts, void *workspace, size_t workspace_bytes, void *stream)
{
    if (n == 0) return TUNA_OK;
    if (!offsets) return TUNA_ERR_NULL_POINTER;
    return mx_product(x, x_type, xs, q, s, offsets, o, o_type, m, n, k, experts, workspace, workspace_bytes, stream);
}

extern "C" size_t tuna_mx_workspace_bytes(int m, int n, int k, int experts, int x_type)
{
    if (m < 1 || m % 8 || n < 1 || k < 1 || k % kMxBlock || experts < 0 || experts > TUNA_MX_MAX_EXPERTS || too_long(m, k) || too_long(n, k)) return 0;
    return mx_workspace(m, n, k, std::max(1, experts), x_type, experts > 0, device_sm_count()).total;
}
