// Microscaled 4-bit quantizer and its inverse (format and layout: mx_format.cuh).
//
// A warp takes eight rows of one 256-column chunk: a lane eight columns of each, so a block of 32 is four lanes and its largest
// magnitude takes two shuffles.  A row's 128 bytes of codes are one warp store, eight rows' 1 KB of one run of memory; the rows'
// scale words are gathered into one lane each and leave as two runs of 32 bytes.
#include <algorithm>
#include "launchers.h"
#include "mx_format.cuh"

namespace tuna {

constexpr int kMxqWarps = 4;

template <typename T, int ROWS>
__global__ void __launch_bounds__(kMxqWarps * 32)
mx_quantize_kernel(const T *__restrict__ x, long long row_stride, uint8_t *__restrict__ q, uint32_t *__restrict__ s, int rows, int k, int chunks,
                   long long items)
{
    const int lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * kMxqWarps + (threadIdx.x >> 5);
    if (item >= items) return;
    const int words = div_up(k, kMxScaleCols);
    const int groups = div_up(rows, ROWS);
    const int c = (int)(item % chunks);
    const long long g = item / chunks;
    const int matrix = (int)(g / groups), row0 = (int)(g - (long long)matrix * groups) * ROWS;
    const int col = c * kMxChunk + lane * 8;
    const T *src = x + ((long long)matrix * rows + row0) * row_stride + col;
    uint8_t *dst = q + (((long long)matrix * chunks + c) * rows + row0) * kMxChunkBytes + lane * 4;

    float v[ROWS][8];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        if (col < k && row0 + r < rows) {
            mx_load8(src + r * row_stride, v[r]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[r][i] = 0.f;
        }
    }
    uint32_t mine = 0;  // the word of scales of row (lane % 16), columns 128 (lane / 16) .. + 127 of the chunk
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        uint32_t largest = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) largest = max(largest, __float_as_uint(v[r][i]) & 0x7fffffffu);
        largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
        largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
        const uint32_t e = mx_scale(largest);
        const float inverse = mx_inverse(e);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[r][i] *= inverse;
        const uint32_t codes = e == 255u ? 0u : mx_encode8(v[r]);
        if (row0 + r < rows) *reinterpret_cast<uint32_t *>(dst + (size_t)r * kMxChunkBytes) = codes;
        uint32_t w = e << (8 * ((lane >> 2) & 3));
        w |= __shfl_xor_sync(0xffffffffu, w, 4);
        w |= __shfl_xor_sync(0xffffffffu, w, 8);
        if ((lane & 15) == r) mine = w;
    }
    const int r = lane & 15, word = 2 * c + (lane >> 4);
    if (r < ROWS && row0 + r < rows && word < words) s[((long long)matrix * words + word) * rows + row0 + r] = mine;
}

template <typename T>
__device__ __forceinline__ void mx_store8(T *p, const float (&v)[8]);
template <>
__device__ __forceinline__ void mx_store8<__half>(__half *p, const float (&v)[8])
{
    *reinterpret_cast<uint4 *>(p) = make_uint4(pack_half2(v[0], v[1]), pack_half2(v[2], v[3]), pack_half2(v[4], v[5]), pack_half2(v[6], v[7]));
}
template <>
__device__ __forceinline__ void mx_store8<__nv_bfloat16>(__nv_bfloat16 *p, const float (&v)[8])
{
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
    *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
template <>
__device__ __forceinline__ void mx_store8<float>(float *p, const float (&v)[8])
{
    reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// o = code * scale in fp32 (exact: three significant bits, exponents of fp32's range), rounded once to T.
template <typename T, int ROWS>
__global__ void __launch_bounds__(kMxqWarps * 32)
mx_dequant_kernel(const uint8_t *__restrict__ q, const uint32_t *__restrict__ s, T *__restrict__ o, int rows, int k, int chunks, long long items)
{
    const int lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * kMxqWarps + (threadIdx.x >> 5);
    if (item >= items) return;
    const int words = div_up(k, kMxScaleCols);
    const int groups = div_up(rows, ROWS);
    const int c = (int)(item % chunks);
    const long long g = item / chunks;
    const int matrix = (int)(g / groups), row0 = (int)(g - (long long)matrix * groups) * ROWS;
    const int col = c * kMxChunk + lane * 8;
    const uint8_t *src = q + (((long long)matrix * chunks + c) * rows + row0) * kMxChunkBytes + lane * 4;

    const int wr = lane & 15, word = 2 * c + (lane >> 4);
    uint32_t codes[ROWS], scales = 0;
    if (wr < ROWS && row0 + wr < rows && word < words) scales = __ldg(s + ((long long)matrix * words + word) * rows + row0 + wr);
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
        codes[r] = row0 + r < rows ? __ldg(reinterpret_cast<const uint32_t *>(src + (size_t)r * kMxChunkBytes)) : 0u;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const uint32_t e = (__shfl_sync(0xffffffffu, scales, (lane & 16) | r) >> (8 * ((lane >> 2) & 3))) & 255u;
        const float scale = mx_scale_value(e);
        uint32_t h[4];
        mx_decode8(codes[r], h);
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[i]));
            v[2 * i] = f.x * scale;
            v[2 * i + 1] = f.y * scale;
        }
        if (col < k && row0 + r < rows) mx_store8<T>(o + ((long long)matrix * rows + row0 + r) * k + col, v);
    }
}

static long long mx_items(int rows, int k, int batch, int rows_per_warp) { return (long long)batch * div_up(rows, rows_per_warp) * div_up(k, kMxChunk); }

template <typename T>
static cudaError_t quantize_as(const void *x, long long row_stride, void *q, void *s, int rows, int k, int batch, cudaStream_t stream)
{
    const int chunks = div_up(k, kMxChunk);
    const long long items = mx_items(rows, k, batch, 8);
    mx_quantize_kernel<T, 8><<<(unsigned)div_up_ll(items, kMxqWarps), kMxqWarps * 32, 0, stream>>>((const T *)x, row_stride, (uint8_t *)q, (uint32_t *)s,
                                                                                                  rows, k, chunks, items);
    return cudaGetLastError();
}

cudaError_t launch_mx_quantize(const void *x, int type, long long row_stride, void *q, void *s, int rows, int k, int batch, cudaStream_t stream)
{
    switch (type) {
        case TUNA_FP16: return quantize_as<__half>(x, row_stride, q, s, rows, k, batch, stream);
        case TUNA_BF16: return quantize_as<__nv_bfloat16>(x, row_stride, q, s, rows, k, batch, stream);
        default: return quantize_as<float>(x, row_stride, q, s, rows, k, batch, stream);
    }
}

template <typename T>
static cudaError_t dequant_as(const void *q, const void *s, void *o, int rows, int k, int batch, cudaStream_t stream)
{
    const int chunks = div_up(k, kMxChunk);
    const long long items = mx_items(rows, k, batch, 8);
    mx_dequant_kernel<T, 8><<<(unsigned)div_up_ll(items, kMxqWarps), kMxqWarps * 32, 0, stream>>>((const uint8_t *)q, (const uint32_t *)s, (T *)o, rows, k,
                                                                                                 chunks, items);
    return cudaGetLastError();
}

cudaError_t launch_mx_dequant(const void *q, const void *s, void *o, int type, int rows, int k, int batch, cudaStream_t stream)
{
    switch (type) {
        case TUNA_FP16: return dequant_as<__half>(q, s, o, rows, k, batch, stream);
        case TUNA_BF16: return dequant_as<__nv_bfloat16>(q, s, o, rows, k, batch, stream);
        default: return dequant_as<float>(q, s, o, rows, k, batch, stream);
    }
}

}  // namespace tuna
