// Microscaled 4-bit quantizer and its inverse (format and layout: mx_format.cuh).
//
// A warp takes a few rows of one 256-column chunk: a lane eight columns of each, so a block of 32 is four lanes and its largest
// magnitude takes two shuffles.  A row's 128 bytes of codes are one warp store and neighbouring rows' one run of memory; the rows'
// scale words are gathered into one lane each.  Numbers stay as they were loaded until they are needed and maxima of 16-bit
// types are taken in pairs: with fp32 copies of eight rows 57344x8192 took 369 us, waiting for loads with 40 % of the warps that fit, so 191.
//
// HBM bounds both: 57344x8192 in fp16 191 us and 195 back, 6.2 and 6.1 TB/s, where a copy reaches 6.55; 5000x8224 in fp32 28 us (6.6 TB/s)
// and 34 back (5.4 TB/s, seven eighths of it stores).
#include <algorithm>
#include "launchers.h"
#include "mx_format.cuh"

namespace tuna {

constexpr int kMxqWarps = 4;

// The warps of a CTA take neighbouring chunks, 1 << log_c of them, of as many row groups as that leaves; grid (row groups, chunks).
struct MxqPlace {
    int c, matrix, row0;
    bool any;
};
template <int ROWS>
__device__ __forceinline__ MxqPlace mxq_place(int rows, int chunks, int batch, int log_c)
{
    const int warp = threadIdx.x >> 5, groups = div_up(rows, ROWS);
    MxqPlace l;
    l.c = (int)(blockIdx.y << log_c) + (warp & ((1 << log_c) - 1));
    const long long g = ((long long)blockIdx.x << (2 - log_c)) + (warp >> log_c);
    l.matrix = batch == 1 ? 0 : (int)(g / groups);
    const int group = (int)(g - (long long)l.matrix * groups);
    l.row0 = group * ROWS;
    l.any = l.c < chunks && l.matrix < batch && group < groups;
    return l;
}

template <typename T, int ROWS>
__global__ void __launch_bounds__(kMxqWarps * 32)
mx_quantize_kernel(const T *__restrict__ x, long long row_stride, uint8_t *__restrict__ q, uint32_t *__restrict__ s, int rows, int k, int chunks, int batch,
                   int log_c, MxChained chained)
{
    // Part of a product, which may start (and read its weights, not this kernel's) while this one runs.
    if (chained == kMxChained) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (chained) asm volatile("griddepcontrol.wait;" ::: "memory");
    if (chained == kMxChainedAfter) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 31;
    const MxqPlace l = mxq_place<ROWS>(rows, chunks, batch, log_c);
    if (!l.any) return;
    const int col = l.c * kMxChunk + lane * 8;
    const T *src = x + ((long long)l.matrix * rows + l.row0) * row_stride + col;
    uint8_t *dst = q + (((long long)l.matrix * chunks + l.c) * rows + l.row0) * kMxChunkBytes + lane * 4;

    Mx8<T> v[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        if (col < k && l.row0 + r < rows) v[r].load(src + r * row_stride);
        else v[r].zero();
    }
    uint32_t mine = 0;  // the scale of row lane % ROWS
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const uint32_t e = mx_scale(v[r].largest());
        const float inverse = mx_inverse(e);
        float f[8];
        v[r].values(f);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] *= inverse;
        const uint32_t codes = e == 255u ? 0u : mx_encode8(f);
        if (l.row0 + r < rows) *reinterpret_cast<uint32_t *>(dst + (size_t)r * kMxChunkBytes) = codes;
        if (r == 0 || (lane & 3) == r) mine = e;
    }
    // a block's four lanes have the scales of one row each; the word of a row is what four neighbouring blocks have of it
    mine <<= 8 * ((lane >> 2) & 3);
    mine |= __shfl_xor_sync(0xffffffffu, mine, 4);
    mine |= __shfl_xor_sync(0xffffffffu, mine, 8);
    const int r = lane & 15, words = div_up(k, kMxScaleCols), word = 2 * l.c + (lane >> 4);
    if (r < ROWS && l.row0 + r < rows && word < words) s[((long long)l.matrix * words + word) * rows + l.row0 + r] = mine;
}

__device__ __forceinline__ void mx_store8(__half *p, const float (&v)[8])
{
    *reinterpret_cast<uint4 *>(p) = make_uint4(pack_half2(v[0], v[1]), pack_half2(v[2], v[3]), pack_half2(v[4], v[5]), pack_half2(v[6], v[7]));
}
__device__ __forceinline__ void mx_store8(__nv_bfloat16 *p, const float (&v)[8])
{
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
    *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// o = code * scale in fp32 (exact: three significant bits, exponents of fp32's range), rounded once to T.  Results of two bytes: a
// lane has eight columns side by side, 16 bytes; of four: four columns of each half of the chunk, 16 bytes each.
template <typename T, int ROWS>
__global__ void __launch_bounds__(kMxqWarps * 32)
mx_dequant_kernel(const uint8_t *__restrict__ q, const uint32_t *__restrict__ s, T *__restrict__ o, int rows, int k, int chunks, int batch, int log_c)
{
    constexpr bool kWide = sizeof(T) == 4;
    const int lane = threadIdx.x & 31;
    const MxqPlace l = mxq_place<ROWS>(rows, chunks, batch, log_c);
    if (!l.any) return;
    const int words = div_up(k, kMxScaleCols);
    const int col = l.c * kMxChunk + lane * (kWide ? 4 : 8);
    const uint8_t *src = q + (((long long)l.matrix * chunks + l.c) * rows + l.row0) * kMxChunkBytes;
    T *dst = o + ((long long)l.matrix * rows + l.row0) * k + col;

    const int wr = lane & 15, word = 2 * l.c + (lane >> 4);
    uint32_t codes[ROWS], scales = 0;
    if (wr < ROWS && l.row0 + wr < rows && word < words) scales = __ldg(s + ((long long)l.matrix * words + word) * rows + l.row0 + wr);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        codes[r] = 0;
        if (l.row0 + r < rows) {
            if (kWide) {
                const uint16_t *p = reinterpret_cast<const uint16_t *>(src + (size_t)r * kMxChunkBytes) + lane;
                codes[r] = (uint32_t)__ldg(p) | ((uint32_t)__ldg(p + 32) << 16);
            } else {
                codes[r] = __ldg(reinterpret_cast<const uint32_t *>(src + (size_t)r * kMxChunkBytes) + lane);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        float scale[2];  // of the first and the last four columns
        if (kWide) {
            scale[0] = mx_scale_value((__shfl_sync(0xffffffffu, scales, r) >> (8 * (lane >> 3))) & 255u);
            scale[1] = mx_scale_value((__shfl_sync(0xffffffffu, scales, 16 | r) >> (8 * (lane >> 3))) & 255u);
        } else {
            scale[0] = scale[1] = mx_scale_value((__shfl_sync(0xffffffffu, scales, (lane & 16) | r) >> (8 * ((lane >> 2) & 3))) & 255u);
        }
        uint32_t h[4];
        mx_decode8(codes[r], h);
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[i]));
            v[2 * i] = f.x * scale[i >> 1];
            v[2 * i + 1] = f.y * scale[i >> 1];
        }
        if (l.row0 + r >= rows) continue;
        T *p = dst + (size_t)r * k;
        if constexpr (kWide) {
            if (col < k) *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
            if (col + 128 < k) *reinterpret_cast<float4 *>(p + 128) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            if (col < k) mx_store8(p, v);
        }
    }
}

// Row groups and chunks of a launch: a CTA's four warps side by side along the columns as far as there are chunks.
template <typename Kernel>
static cudaError_t mxq_launch(int rows, int k, int batch, int rows_per_warp, Kernel kernel)
{
    const int chunks = div_up(k, kMxChunk), log_c = chunks >= 4 ? 2 : chunks >= 2 ? 1 : 0;
    const long long groups = (long long)batch * div_up(rows, rows_per_warp);
    return kernel(dim3((unsigned)div_up_ll(groups, 4 >> log_c), (unsigned)div_up(chunks, 1 << log_c)), chunks, log_c);
}

// Rows of a warp: many where bandwidth counts (57344x8192 in fp16: quantizing 2 rows 227 us, 4 191, 8 188, but of 1999x14336 in bf16 15.3, 13.1,
// 15.1; back 2 rows 202, 4 193, 8 195 and 15.0, 14.0, 13.6), two where the launch is short (4096 columns in bf16, us, quantizing 2 / 4 and
// back 2 / 8: 1 row 1.28 / 1.54 and 1.28 / 1.79, 64 1.79 / 2.05 and 1.54 / 2.18, 512 2.56 / 2.97 and 2.69 / 3.08, 1024 3.72 / 3.84 and 4.10 / 3.86).
static bool mxq_short(int rows, int k, int batch) { return (long long)rows * batch * div_up(k, kMxChunk) <= 8192; }

template <typename T, int ROWS>
static cudaError_t quantize_as(const void *x, long long row_stride, void *q, void *s, int rows, int k, int batch, MxChained chained, cudaStream_t stream)
{
    return mxq_launch(rows, k, batch, ROWS, [&](dim3 grid, int chunks, int log_c) {
        cudaLaunchConfig_t lc = {};
        lc.gridDim = grid;
        lc.blockDim = dim3(kMxqWarps * 32);
        lc.stream = stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        lc.attrs = attr;
        lc.numAttrs = chained ? 1 : 0;
        return cudaLaunchKernelEx(&lc, mx_quantize_kernel<T, ROWS>, (const T *)x, row_stride, (uint8_t *)q, (uint32_t *)s, rows, k, chunks, batch, log_c, chained);
    });
}

template <typename T>
static cudaError_t quantize_any(const void *x, long long row_stride, void *q, void *s, int rows, int k, int batch, MxChained chained, cudaStream_t stream)
{
    return mxq_short(rows, k, batch) ? quantize_as<T, 2>(x, row_stride, q, s, rows, k, batch, chained, stream)
                                     : quantize_as<T, 4>(x, row_stride, q, s, rows, k, batch, chained, stream);
}

cudaError_t launch_mx_quantize(const void *x, int type, long long row_stride, void *q, void *s, int rows, int k, int batch, cudaStream_t stream, MxChained chained)
{
    switch (type) {
        case TUNA_FP16: return quantize_any<__half>(x, row_stride, q, s, rows, k, batch, chained, stream);
        case TUNA_BF16: return quantize_any<__nv_bfloat16>(x, row_stride, q, s, rows, k, batch, chained, stream);
        default: return quantize_any<float>(x, row_stride, q, s, rows, k, batch, chained, stream);
    }
}

template <typename T, int ROWS>
static cudaError_t dequant_as(const void *q, const void *s, void *o, int rows, int k, int batch, cudaStream_t stream)
{
    return mxq_launch(rows, k, batch, ROWS, [&](dim3 grid, int chunks, int log_c) {
        mx_dequant_kernel<T, ROWS><<<grid, kMxqWarps * 32, 0, stream>>>((const uint8_t *)q, (const uint32_t *)s, (T *)o, rows, k, chunks, batch, log_c);
        return cudaGetLastError();
    });
}

template <typename T>
static cudaError_t dequant_any(const void *q, const void *s, void *o, int rows, int k, int batch, cudaStream_t stream)
{
    return mxq_short(rows, k, batch) ? dequant_as<T, 2>(q, s, o, rows, k, batch, stream) : dequant_as<T, 8>(q, s, o, rows, k, batch, stream);
}

cudaError_t launch_mx_dequant(const void *q, const void *s, void *o, int type, int rows, int k, int batch, cudaStream_t stream)
{
    switch (type) {
        case TUNA_FP16: return dequant_any<__half>(q, s, o, rows, k, batch, stream);
        case TUNA_BF16: return dequant_any<__nv_bfloat16>(q, s, o, rows, k, batch, stream);
        default: return dequant_any<float>(q, s, o, rows, k, batch, stream);
    }
}

}  // namespace tuna
