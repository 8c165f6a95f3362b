// C ABI of the 8-bit block-scaled operators: argument checks, workspace layout, dispatch.
#include "fp8_format.cuh"
#include "launchers.h"

namespace tuna {

static bool aligned_to(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
static bool is_number_type(int t) { return t == TUNA_FP16 || t == TUNA_BF16 || t == TUNA_FP32; }
static bool is_16bit(int t) { return t == TUNA_FP16 || t == TUNA_BF16; }

constexpr int kFp8MaxWidth = 1 << 23;  // grids have tiles of 128 columns in y

// Sizes in 32 bits leave room for being rounded up to whole tiles, and a matrix's elements for sums in 64.
static bool too_large(int rows, int k) { return rows > 0x7fffffff - 1023 || k > kFp8MaxWidth || (double)rows * k > (double)(1ll << 41); }

static size_t round_up(size_t v) { return (v + 255) / 256 * 256; }
static size_t word_bytes(int along, int across) { return (size_t)div_up(along, kFp8Word) * across * 4; }  // scales of blocks along one dimension

// Codes and scales of an operand in the workspace, from `at` on; `at` moves behind them.
static Fp8Codes place(void *workspace, size_t &at, size_t codes, size_t scales)
{
    Fp8Codes c = {(uint8_t *)workspace + at, (uint8_t *)workspace + at + round_up(codes)};
    at += round_up(codes) + round_up(scales);
    return c;
}
static size_t room(size_t codes, size_t scales) { return round_up(codes) + round_up(scales); }

static size_t product_workspace(bool gated, int m, int n, int k, int x_type, int sms)
{
    return fp8_gemm_takes(gated, m, n, k, x_type, sms) ? 0 : room((size_t)n * k, word_bytes(k, n));
}
static size_t backward_workspace(bool with_dx, bool with_dw, int m, int n, int k, int x_type)
{
    size_t bytes = 0;
    if (with_dx) bytes += room((size_t)n * m, word_bytes(m, n));
    if (with_dw) bytes += room((size_t)n * m, word_bytes(n, m)) + (x_type == TUNA_FP8 ? 0 : room((size_t)n * k, word_bytes(n, k)));
    return bytes;
}

static int check_sizes(int m, int n, int k)
{
    if (m < 1 || m % 16 || n < 1 || k < 1 || k % 16) return TUNA_ERR_BAD_SHAPE;
    if (too_large(m, k) || too_large(n, k) || too_large(n, m)) return TUNA_ERR_TOO_LARGE;
    return TUNA_OK;
}

static int product(bool gated, const void *x, int x_type, const void *xs, const void *q, const void *s, void *o, int o_type, void *z, int m, int n, int k, int activation,
                   void *workspace, size_t workspace_bytes, void *stream)
{
    const bool packed = x_type == TUNA_FP8;
    if (!x || !q || !s || !o || (packed && !xs)) return TUNA_ERR_NULL_POINTER;
    const int st = check_sizes(m, n, k);
    if (st != TUNA_OK) return st;
    if ((!packed && !is_16bit(x_type)) || !is_number_type(o_type) || (activation != TUNA_SILU && activation != TUNA_GELU) || (z && !is_16bit(o_type))) return TUNA_ERR_BAD_CONFIG;
    if (!aligned_to(x, 16) || !aligned_to(q, 16) || !aligned_to(o, 16) || !aligned_to(z, 16) || (packed && !aligned_to(xs, 4)) || !aligned_to(workspace, 16)) return TUNA_ERR_MISALIGNED;
    const int sms = device_sm_count();
    const size_t need = product_workspace(gated, m, n, k, x_type, sms);
    if (need > 0 && (!workspace || workspace_bytes < need)) return TUNA_ERR_WORKSPACE;
    Fp8ProductArgs a;
    a.w = {const_cast<void *>(q), const_cast<void *>(s)};
    a.x = {const_cast<void *>(x), const_cast<void *>(xs)};
    a.numbers = nullptr;
    if (!packed) {
        size_t at = 0;
        a.x = need > 0 ? place(workspace, at, (size_t)n * k, word_bytes(k, n)) : Fp8Codes{nullptr, nullptr};
        a.numbers = x;
    }
    a.o = o; a.z = z; a.m = m; a.n = n; a.k = k; a.x_type = x_type; a.o_type = o_type; a.gated = gated; a.gelu = activation == TUNA_GELU;
    a.stream = (cudaStream_t)stream; a.sm_count = sms;
    return launch_fp8_product(a);
}

// z: of a gated block, dy is dh then
static int backward(const void *dy, const void *z, int dy_type, const void *x, int x_type, const void *xs, const void *q, const void *s, void *dx, int dx_type, void *dw, int dw_type,
                    int m, int n, int k, int activation, void *workspace, size_t workspace_bytes, cudaStream_t stream)
{
    const bool packed = x_type == TUNA_FP8;
    if (!dy || (!dx && !dw) || (dx && (!q || !s)) || (dw && (!x || (packed && !xs)))) return TUNA_ERR_NULL_POINTER;
    const int st = check_sizes(m, n, k);
    if (st != TUNA_OK) return st;
    if (!is_16bit(dy_type) || (dx && !is_number_type(dx_type)) || (dw && (!is_number_type(dw_type) || (!packed && !is_16bit(x_type)))) ||
        (activation != TUNA_SILU && activation != TUNA_GELU))
        return TUNA_ERR_BAD_CONFIG;
    if (!aligned_to(dy, 16) || !aligned_to(z, 16) || !aligned_to(workspace, 16) || (dx && (!aligned_to(dx, 16) || !aligned_to(q, 16))) ||
        (dw && (!aligned_to(dw, 16) || !aligned_to(x, 16) || (packed && !aligned_to(xs, 4)))))
        return TUNA_ERR_MISALIGNED;
    const size_t need = backward_workspace(dx, dw, m, n, k, x_type);
    if (need > 0 && (!workspace || workspace_bytes < need)) return TUNA_ERR_WORKSPACE;
    size_t at = 0;
    Fp8Codes by_row = {nullptr, nullptr}, by_column = {nullptr, nullptr}, xt = {const_cast<void *>(x), const_cast<void *>(xs)};
    if (dx) by_row = place(workspace, at, (size_t)n * m, word_bytes(m, n));
    if (dw) by_column = place(workspace, at, (size_t)n * m, word_bytes(n, m));
    Fp8BackwardArgs a;
    Fp8GradientArgs &g = a.operands;
    g.dy = dy; g.z = z; g.x = x; g.type = dy_type; g.x_type = x_type; g.gelu = activation == TUNA_GELU; g.rows = n; g.cols = m; g.x_cols = k;
    g.by_row = by_row; g.by_column = by_column; g.x_to = {nullptr, nullptr}; g.stream = stream; g.sm_count = device_sm_count();
    if (dw && !packed) g.x_to = xt = place(workspace, at, (size_t)n * k, word_bytes(n, k));
    a.w = {const_cast<void *>(q), const_cast<void *>(s)};
    a.x = xt;
    a.dx = dx; a.dw = dw; a.dx_type = dx_type; a.dw_type = dw_type;
    return launch_fp8_backward(a);
}

}  // namespace tuna

using namespace tuna;

extern "C" int tuna_fp8_quantize(const void *x, int x_type, long long row_stride, int blocks, void *q, void *s, void *q2, void *s2, int rows, int k, void *stream)
{
    if (!x || !q || !s || (blocks == TUNA_FP8_BOTH && (!q2 || !s2))) return TUNA_ERR_NULL_POINTER;
    if (rows < 1 || k < 1 || k % 16 || row_stride < k || row_stride > 1ll << 40) return TUNA_ERR_BAD_SHAPE;
    if (too_large(rows, k)) return TUNA_ERR_TOO_LARGE;
    if (!is_number_type(x_type) || blocks < TUNA_FP8_ROW || blocks > TUNA_FP8_SQUARE) return TUNA_ERR_BAD_CONFIG;
    if (!aligned_to(x, 16) || (row_stride * (x_type == TUNA_FP32 ? 4 : 2)) % 16 || !aligned_to(q, 16) || !aligned_to(q2, 16)) return TUNA_ERR_MISALIGNED;
    if (blocks != TUNA_FP8_SQUARE && (!aligned_to(s, 4) || !aligned_to(s2, 4))) return TUNA_ERR_MISALIGNED;
    const cudaError_t e = blocks == TUNA_FP8_ROW ? launch_fp8_quantize_rows(x, x_type, row_stride, q, s, rows, k, false, (cudaStream_t)stream)
                                                 : launch_fp8_quantize_tiles(x, x_type, row_stride, blocks, {q, s}, {q2, s2}, rows, k, (cudaStream_t)stream);
    return e == cudaSuccess ? TUNA_OK : TUNA_ERR_LAUNCH;
}

extern "C" int tuna_fp8_dequant(const void *q, const void *s, int blocks, void *o, int o_type, int rows, int k, void *stream)
{
    if (!q || !s || !o) return TUNA_ERR_NULL_POINTER;
    if (rows < 1 || k < 1 || k % 16) return TUNA_ERR_BAD_SHAPE;
    if (too_large(rows, k)) return TUNA_ERR_TOO_LARGE;
    if (!is_number_type(o_type) || (blocks != TUNA_FP8_ROW && blocks != TUNA_FP8_COLUMN && blocks != TUNA_FP8_SQUARE)) return TUNA_ERR_BAD_CONFIG;
    if (!aligned_to(q, 16) || !aligned_to(o, 16)) return TUNA_ERR_MISALIGNED;
    return launch_fp8_dequant(q, s, blocks, o, o_type, rows, k, (cudaStream_t)stream) == cudaSuccess ? TUNA_OK : TUNA_ERR_LAUNCH;
}

extern "C" int tuna_fp8_matmul(const void *x, int x_type, const void *xs, const void *q, const void *s, void *o, int o_type, int m, int n, int k, void *workspace,
                               size_t workspace_bytes, void *stream)
{
    return product(false, x, x_type, xs, q, s, o, o_type, nullptr, m, n, k, TUNA_SILU, workspace, workspace_bytes, stream);
}

extern "C" int tuna_fp8_gated(const void *x, int x_type, const void *xs, const void *q, const void *s, void *h, int h_type, void *z, int f, int n, int k, int activation,
                              void *workspace, size_t workspace_bytes, void *stream)
{
    if (f < 1 || f % 16) return TUNA_ERR_BAD_SHAPE;
    if (f > kFp8MaxWidth / 2) return TUNA_ERR_TOO_LARGE;
    return product(true, x, x_type, xs, q, s, h, h_type, z, 2 * f, n, k, activation, workspace, workspace_bytes, stream);
}

extern "C" int tuna_fp8_matmul_backward(const void *dy, int dy_type, const void *x, int x_type, const void *xs, const void *q, const void *s, void *dx, int dx_type, void *dw,
                                        int dw_type, int m, int n, int k, void *workspace, size_t workspace_bytes, void *stream)
{
    return backward(dy, nullptr, dy_type, x, x_type, xs, q, s, dx, dx_type, dw, dw_type, m, n, k, TUNA_SILU, workspace, workspace_bytes, (cudaStream_t)stream);
}

extern "C" int tuna_fp8_gated_backward(const void *dh, const void *z, int type, const void *x, int x_type, const void *xs, const void *q, const void *s, void *dx, int dx_type,
                                       void *dw, int dw_type, int f, int n, int k, int activation, void *workspace, size_t workspace_bytes, void *stream)
{
    if (!z) return TUNA_ERR_NULL_POINTER;
    if (f < 1 || f % 16) return TUNA_ERR_BAD_SHAPE;
    if (f > kFp8MaxWidth / 2) return TUNA_ERR_TOO_LARGE;
    return backward(dh, z, type, x, x_type, xs, q, s, dx, dx_type, dw, dw_type, 2 * f, n, k, activation, workspace, workspace_bytes, (cudaStream_t)stream);
}

extern "C" size_t tuna_fp8_workspace_bytes(int call, int m, int n, int k, int x_type)
{
    if (check_sizes(m, n, k) != TUNA_OK || call < TUNA_FP8_MATMUL || call > TUNA_FP8_BACKWARD) return 0;
    if (call == TUNA_FP8_BACKWARD) return backward_workspace(true, true, m, n, k, x_type);
    return product_workspace(call == TUNA_FP8_GATED, m, n, k, x_type, device_sm_count());
}
