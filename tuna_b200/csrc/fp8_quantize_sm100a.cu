// Quantizers of the 8-bit block-scaled format (fp8_format.cuh), their inverse, and the quantizer of a gated block's gradients.
#include <algorithm>
#include "launchers.h"
#include "fp8_format.cuh"

namespace tuna {

// ---- blocks of a row

constexpr int kFp8qWarps = 4;
constexpr int kFp8Chunk = 256;  // columns of a warp: eight of a lane, sixteen lanes a block

// A warp takes ROWS rows of 256 columns; grid (row groups, chunks by fours).
template <typename T, int ROWS>
__global__ void __launch_bounds__(kFp8qWarps * 32)
fp8_quantize_rows_kernel(const T *x, long long row_stride, uint8_t *q, uint8_t *s, int rows, int k, int log_c, bool chained)
{
    // Part of a product, which may start (and read its weights, not this kernel's) while this one runs.
    if (chained) {
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
        asm volatile("griddepcontrol.wait;" ::: "memory");
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, blocks = div_up(k, kFp8Block);
    const int c = (int)(blockIdx.y << log_c) + (warp & ((1 << log_c) - 1));
    const long long row0 = (((long long)blockIdx.x << (2 - log_c)) + (warp >> log_c)) * ROWS;
    if (c * kFp8Chunk >= k || row0 >= rows) return;
    const int col = c * kFp8Chunk + lane * 8;
    Mx8<T> v[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        if (col < k && row0 + r < rows) v[r].load(x + (row0 + r) * row_stride + col);
        else v[r].zero();
    }
    uint32_t mine = 0;  // the scale of row lane % 16
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        uint32_t m = v[r].largest();  // of four lanes
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 4));
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 8));
        const uint32_t e = fp8_scale(m);
        const float inverse = fp8_inverse(e);
        float f[8];
        v[r].values(f);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] *= inverse;
        uint2 codes = make_uint2(fp8_encode4(f[0], f[1], f[2], f[3]), fp8_encode4(f[4], f[5], f[6], f[7]));
        if (e == 255u) codes = make_uint2(0, 0);
        if (col < k && row0 + r < rows) *reinterpret_cast<uint2 *>(q + (row0 + r) * k + col) = codes;
        if ((lane & 15) == r) mine = e;
    }
    const long long row = row0 + (lane & 15);
    const int b = 2 * c + (lane >> 4);
    if ((lane & 15) >= ROWS || row >= rows || b >= blocks) return;
    uint8_t *at = s + ((long long)(b >> 2) * rows + row) * 4 + (b & 3);
    *at = (uint8_t)mine;
    if (b + 1 == blocks)
        for (int i = 1; i < 4 - (b & 3); ++i) at[i] = 0;  // blocks that the last word does not have
}

template <typename T, int ROWS>
static cudaError_t quantize_rows_as(const void *x, long long row_stride, void *q, void *s, int rows, int k, bool chained, cudaStream_t stream)
{
    const int chunks = div_up(k, kFp8Chunk), log_c = chunks >= 4 ? 2 : chunks >= 2 ? 1 : 0;
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)div_up(div_up(rows, ROWS), 4 >> log_c), (unsigned)div_up(chunks, 1 << log_c));
    lc.blockDim = dim3(kFp8qWarps * 32);
    lc.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = attr;
    lc.numAttrs = chained ? 1 : 0;
    return cudaLaunchKernelEx(&lc, fp8_quantize_rows_kernel<T, ROWS>, (const T *)x, row_stride, (uint8_t *)q, (uint8_t *)s, rows, k, log_c, chained);
}

template <typename T>
static cudaError_t quantize_rows(const void *x, long long row_stride, void *q, void *s, int rows, int k, bool chained, cudaStream_t stream)
{
    return (long long)rows * div_up(k, kFp8Chunk) <= 8192 ? quantize_rows_as<T, 2>(x, row_stride, q, s, rows, k, chained, stream)
                                                          : quantize_rows_as<T, 4>(x, row_stride, q, s, rows, k, chained, stream);
}

cudaError_t launch_fp8_quantize_rows(const void *x, int type, long long row_stride, void *q, void *s, int rows, int k, bool chained, cudaStream_t stream)
{
    switch (type) {
        case TUNA_FP16: return quantize_rows<__half>(x, row_stride, q, s, rows, k, chained, stream);
        case TUNA_BF16: return quantize_rows<__nv_bfloat16>(x, row_stride, q, s, rows, k, chained, stream);
        default: return quantize_rows<float>(x, row_stride, q, s, rows, k, chained, stream);
    }
}

// ---- tiles of 128 x 128: blocks of a column, of a row and a column, square ones

// A warp has 16 rows of the tile, a lane eight of them (every second) and eight columns: 16 lanes are a row's block.  All of a lane's numbers are loaded before
// the first is used.
constexpr int kFp8TileWarps = 8;
constexpr int kFp8TileRows = kFp8Block / kFp8TileWarps;
constexpr int kFp8LaneRows = kFp8TileRows / 2;

__device__ __forceinline__ uint32_t fp8_magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }  // compare as the numbers do, NaN above infinity

// Rows' maxima over the 16 lanes that have them: in every step a lane keeps half of the rows and sends the other half, so that in the end lanes 2 r and 2 r + 1 have
// that of row r.  30 instructions for eight rows, where every lane taking part in every row's would be 64, and one scale a lane to work out instead of eight.
template <typename V, typename Max>
__device__ __forceinline__ V fp8_rows_max(V (&v)[kFp8LaneRows], int lane, Max largest)
{
#pragma unroll
    for (int half = kFp8LaneRows / 2; half >= 1; half >>= 1) {
        const int d = 2 * half;
        const bool upper = lane & d;
#pragma unroll
        for (int r = 0; r < half; ++r) {
            const V keep = upper ? v[r + half] : v[r], give = upper ? v[r] : v[r + half];
            v[r] = largest(keep, __shfl_xor_sync(0xffffffffu, give, d));
        }
    }
    return largest(v[0], __shfl_xor_sync(0xffffffffu, v[0], 1));
}

// A lane's numbers as they were loaded, the bits (fp32) of their largest magnitudes, and their values.
template <typename T>
struct Fp8Raw {  // 16 bits: maxima in pairs
    Mx8<T> v[kFp8LaneRows];
    using Pair = decltype(v[0].pair(0));
    __device__ __forceinline__ static Pair with(Pair a, Pair b) { return __hmax2_nan(a, __habs2(b)); }
    __device__ __forceinline__ static float2 widen(__half2 p) { return __half22float2(p); }
    __device__ __forceinline__ static float2 widen(__nv_bfloat162 p) { return __bfloat1622float2(p); }
    __device__ __forceinline__ uint32_t row_max(int lane) const  // of row (lane / 2) % 8 of the lane's
    {
        Pair m[kFp8LaneRows];
#pragma unroll
        for (int r = 0; r < kFp8LaneRows; ++r) m[r] = with(with(__habs2(v[r].pair(0)), v[r].pair(1)), __hmax2_nan(__habs2(v[r].pair(2)), __habs2(v[r].pair(3))));
        const float2 f = widen(fp8_rows_max(m, lane, [](Pair a, Pair b) { return __hmax2_nan(a, b); }));
        return max(fp8_magnitude(f.x), fp8_magnitude(f.y));
    }
    __device__ __forceinline__ void col_max(uint32_t (&m)[8]) const  // of the warp's 16 rows
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            Pair p = __habs2(v[0].pair(i));
#pragma unroll
            for (int r = 1; r < kFp8LaneRows; ++r) p = with(p, v[r].pair(i));
            p = __hmax2_nan(p, __shfl_xor_sync(0xffffffffu, p, 16));
            const float2 f = widen(p);
            m[2 * i] = fp8_magnitude(f.x);
            m[2 * i + 1] = fp8_magnitude(f.y);
        }
    }
    __device__ __forceinline__ uint32_t lane_max() const
    {
        Pair m = __habs2(v[0].pair(0));
#pragma unroll
        for (int r = 0; r < kFp8LaneRows; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) m = with(m, v[r].pair(i));
        const float2 f = widen(m);
        return max(fp8_magnitude(f.x), fp8_magnitude(f.y));
    }
    __device__ __forceinline__ void values(int r, float (&f)[8]) const { v[r].values(f); }
};
struct Fp8RawFloat {
    float v[kFp8LaneRows][8];
    __device__ __forceinline__ uint32_t row_max(int lane) const
    {
        uint32_t m[kFp8LaneRows];
#pragma unroll
        for (int r = 0; r < kFp8LaneRows; ++r) {
            m[r] = fp8_magnitude(v[r][0]);
#pragma unroll
            for (int i = 1; i < 8; ++i) m[r] = max(m[r], fp8_magnitude(v[r][i]));
        }
        return fp8_rows_max(m, lane, [](uint32_t a, uint32_t b) { return max(a, b); });
    }
    __device__ __forceinline__ void col_max(uint32_t (&m)[8]) const
    {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            m[i] = 0;
#pragma unroll
            for (int r = 0; r < kFp8LaneRows; ++r) m[i] = max(m[i], fp8_magnitude(v[r][i]));
            m[i] = max(m[i], __shfl_xor_sync(0xffffffffu, m[i], 16));
        }
    }
    __device__ __forceinline__ uint32_t lane_max() const
    {
        uint32_t m = 0;
#pragma unroll
        for (int r = 0; r < kFp8LaneRows; ++r)
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, fp8_magnitude(v[r][i]));
        return m;
    }
    __device__ __forceinline__ void values(int r, float (&f)[8]) const
    {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = v[r][i];
    }
};
template <> struct Fp8Raw<float> : Fp8RawFloat {};

// Where a tile's numbers come from: rows row0, row0 + 2 .. of columns col .. col + 7.
template <typename T>
struct Fp8Plain {
    const T *x;
    long long row_stride;
    using Raw = Fp8Raw<T>;
    __device__ __forceinline__ void load(Raw &to, long long row0, int col, int rows, int cols) const
    {
#pragma unroll
        for (int r = 0; r < kFp8LaneRows; ++r) {
            const bool in = col < cols && row0 + 2 * r < rows;
            const T *at = x + (row0 + 2 * r) * row_stride + col;
            if constexpr (sizeof(T) == 2) {
                if (in) to.v[r].load(at);
                else to.v[r].zero();
            } else {
                Mx8<float> v;
                if (in) v.load(at);
                else v.zero();
                v.values(to.v[r]);
            }
        }
    }
};
// Columns 0 .. f - 1: the gradient of a gated block's gate, dh u act'(g); f .. 2f - 1: of the other projection, dh act(g).  z = [g | u].
template <typename T, bool GELU>
struct Fp8Gated {
    const T *z, *dh;
    int f;
    using Raw = Fp8RawFloat;
    __device__ __forceinline__ void load(Raw &to, long long row0, int col, int rows, int cols) const
    {
        constexpr int kBatch = 4;  // rows in flight
        const bool gate = col < f;
        const int at = gate ? col : col - f;  // f is a multiple of 16: eight columns are of one kind
#pragma unroll
        for (int r0 = 0; r0 < kFp8LaneRows; r0 += kBatch) {
            Mx8<T> g[kBatch], u[kBatch], d[kBatch];
#pragma unroll
            for (int r = 0; r < kBatch; ++r) {
                const long long row = row0 + 2 * (r0 + r);
                const bool in = col < cols && row < rows;
                const T *zr = z + row * 2 * f + at;
                if (in) {
                    g[r].load(zr);
                    d[r].load(dh + row * f + at);
                } else {
                    g[r].zero();
                    d[r].zero();
                }
                if (in && gate) u[r].load(zr + f);
                else u[r].zero();
            }
#pragma unroll
            for (int r = 0; r < kBatch; ++r) {
                float gv[8], uv[8], dv[8];
                g[r].values(gv);
                u[r].values(uv);
                d[r].values(dv);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float sigma = fp8_gate<GELU>(gv[i]);
                    to.v[r0 + r][i] = gate ? dv[i] * uv[i] * fp8_gate_slope<GELU>(gv[i], sigma) : dv[i] * (gv[i] * sigma);
                }
            }
        }
    }
};

template <int WAYS, typename Source>  // WAYS: 1 << kFp8Row | 1 << kFp8Column, one of them, or 1 << kFp8Square
__global__ void __launch_bounds__(32 * kFp8TileWarps, sizeof(typename Source::Raw) > 128 ? 2 : WAYS & (WAYS - 1) ? 3 : 4)
fp8_quantize_tile_kernel(const Source src, uint8_t *q, uint8_t *s, uint8_t *q2, uint8_t *s2, int rows, int cols, bool two_halves, bool chained)
{
    constexpr bool kRows = WAYS & (1 << kFp8Row), kCols = WAYS & (1 << kFp8Column), kSquare = WAYS & (1 << kFp8Square);
    __shared__ uint4 s_max[kFp8TileWarps][32];  // of a warp's rows, column by column
    __shared__ __align__(16) float s_inverse[kFp8Block];
    __shared__ uint32_t s_square[kFp8TileWarps];
    __shared__ int s_none;  // a column's block is NaN
    if (chained) {
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
        asm volatile("griddepcontrol.wait;" ::: "memory");
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int col_tiles = gridDim.x, row_tiles = div_up(rows, kFp8Block);
    // Halves of the columns that read the same: tile t of the one and of the other follow one another, so that L2 has it.
    const int ct = !two_halves ? blockIdx.x : (blockIdx.x & 1) ? (col_tiles + 1) / 2 + (blockIdx.x >> 1) : blockIdx.x >> 1;
    const int col = ct * kFp8Block + (lane & 15) * 8;
    const size_t step = 2 * (size_t)cols;
    for (int rt = blockIdx.y; rt < row_tiles; rt += gridDim.y) {
        const long long row0 = (long long)rt * kFp8Block + warp * kFp8TileRows + (lane >> 4);
        typename Source::Raw raw;
        src.load(raw, row0, col, rows, cols);
        const int have = col < cols ? (int)min((long long)rows - row0, 2ll * kFp8LaneRows) : 0;  // of the rows from row0 on
        // Codes of row r; MASKED: zeros where a bit of `none` says so.  Two ways and no test in the common one: with it square blocks of 28672x4096 in bf16 took 73 us, so 55.
        auto write = [&](auto masked, uint8_t *to, int r, const float (&inverse)[8], uint32_t none) {
            float f[8];
            raw.values(r, f);
            uint2 w = make_uint2(fp8_encode4(f[0] * inverse[0], f[1] * inverse[1], f[2] * inverse[2], f[3] * inverse[3]),
                                 fp8_encode4(f[4] * inverse[4], f[5] * inverse[5], f[6] * inverse[6], f[7] * inverse[7]));
            if constexpr (decltype(masked)::value)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (none >> i & 1) (i < 4 ? w.x : w.y) &= ~(0xffu << (8 * (i & 3)));
            if (2 * r < have) *reinterpret_cast<uint2 *>(to + r * step) = w;
        };
        if constexpr (kRows) {
            const uint32_t e = fp8_scale(raw.row_max(lane));  // of the lane's row (lane / 2) % 8
            const float mine = fp8_inverse(e);
            uint8_t *to = q + (size_t)row0 * cols + col;
            auto rows_of = [&](auto masked) {
#pragma unroll
                for (int r = 0; r < kFp8LaneRows; ++r) {
                    const float i = __shfl_sync(0xffffffffu, mine, (lane & 16) + 2 * r);
                    const uint32_t none = decltype(masked)::value && __shfl_sync(0xffffffffu, e, (lane & 16) + 2 * r) == 255u ? 255u : 0u;
                    write(masked, to, r, {i, i, i, i, i, i, i, i}, none);
                }
            };
            if (__any_sync(0xffffffffu, e == 255u)) rows_of(Int<1>());
            else rows_of(Int<0>());
            const long long row = row0 + 2 * ((lane >> 1) & 7);
            if ((lane & 1) == 0 && row < rows) {
                uint8_t *at = s + ((long long)(ct >> 2) * rows + row) * 4 + (ct & 3);
                *at = (uint8_t)e;
                if (ct + 1 == col_tiles)
                    for (int i = 1; i < 4 - (ct & 3); ++i) at[i] = 0;
            }
        }
        if constexpr (kCols || kSquare) {
            if (rt != (int)blockIdx.y) __syncthreads();  // what was there before has been read
            uint8_t *to = (kRows ? q2 : q) + (size_t)row0 * cols + col, *words = kRows ? s2 : s;
            float inverse[8];
            uint32_t none = 0;
            if constexpr (kSquare) {
                uint32_t m = raw.lane_max();
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
                if (lane == 0) s_square[warp] = m;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < kFp8TileWarps; ++w) m = max(m, s_square[w]);
                const uint32_t e = fp8_scale(m);
#pragma unroll
                for (int i = 0; i < 8; ++i) inverse[i] = fp8_inverse(e);
                none = e == 255u ? 255u : 0u;
                if (threadIdx.x == 0) words[(long long)rt * col_tiles + ct] = (uint8_t)e;
            } else {
                uint32_t m[8];
                raw.col_max(m);
                if (lane < 16) {
                    s_max[warp][2 * lane] = make_uint4(m[0], m[1], m[2], m[3]);
                    s_max[warp][2 * lane + 1] = make_uint4(m[4], m[5], m[6], m[7]);
                }
                if (threadIdx.x == 0) s_none = 0;
                __syncthreads();
                if (threadIdx.x < kFp8Block) {  // one column each
                    uint32_t e = 0;
#pragma unroll
                    for (int w = 0; w < kFp8TileWarps; ++w) e = max(e, reinterpret_cast<const uint32_t *>(s_max[w])[threadIdx.x]);
                    e = fp8_scale(e);
                    s_inverse[threadIdx.x] = e == 255u ? 0.0f : fp8_inverse(e);
                    if (e == 255u) s_none = 1;
                    const int at_col = ct * kFp8Block + threadIdx.x;
                    if (at_col < cols) {
                        uint8_t *at = words + ((long long)(rt >> 2) * cols + at_col) * 4 + (rt & 3);
                        *at = (uint8_t)e;
                        if (rt + 1 == row_tiles)
                            for (int j = 1; j < 4 - (rt & 3); ++j) at[j] = 0;
                    }
                }
                __syncthreads();
                *reinterpret_cast<float4 *>(inverse) = *reinterpret_cast<const float4 *>(s_inverse + 8 * (lane & 15));
                *reinterpret_cast<float4 *>(inverse + 4) = *reinterpret_cast<const float4 *>(s_inverse + 8 * (lane & 15) + 4);
                if (s_none)
#pragma unroll
                    for (int i = 0; i < 8; ++i) none |= inverse[i] == 0.0f ? 1u << i : 0u;
            }
            auto rows_of = [&](auto masked) {
#pragma unroll
                for (int r = 0; r < kFp8LaneRows; ++r) write(masked, to, r, inverse, none);
            };
            if (__any_sync(0xffffffffu, none != 0u)) rows_of(Int<1>());
            else rows_of(Int<0>());
        }
    }
}

template <int WAYS, typename Source>
static cudaError_t tile_launch(const Source &src, const Fp8Codes &to, const Fp8Codes &to2, int rows, int cols, bool two_halves, bool chained, cudaStream_t stream)
{
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)div_up(cols, kFp8Block), (unsigned)std::min(div_up(rows, kFp8Block), 65535));
    lc.blockDim = dim3(32 * kFp8TileWarps);
    lc.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = attr;
    lc.numAttrs = chained ? 1 : 0;
    return cudaLaunchKernelEx(&lc, fp8_quantize_tile_kernel<WAYS, Source>, src, (uint8_t *)to.q, (uint8_t *)to.s, (uint8_t *)to2.q, (uint8_t *)to2.s, rows, cols, two_halves, chained);
}

template <typename Source>
static cudaError_t tile_ways(const Source &src, int blocks, const Fp8Codes &to, const Fp8Codes &to2, int rows, int cols, bool two_halves, bool chained, cudaStream_t stream)
{
    switch (blocks) {
        case kFp8Column: return tile_launch<1 << kFp8Column>(src, to, to2, rows, cols, two_halves, chained, stream);
        case kFp8Square: return tile_launch<1 << kFp8Square>(src, to, to2, rows, cols, two_halves, chained, stream);
        default: return tile_launch<1 << kFp8Row | 1 << kFp8Column>(src, to, to2, rows, cols, two_halves, chained, stream);
    }
}

cudaError_t launch_fp8_quantize_tiles(const void *x, int type, long long row_stride, int blocks, const Fp8Codes &to, const Fp8Codes &to2, int rows, int k, bool chained,
                                      cudaStream_t stream)
{
    switch (type) {
        case TUNA_FP16: return tile_ways(Fp8Plain<__half>{(const __half *)x, row_stride}, blocks, to, to2, rows, k, false, chained, stream);
        case TUNA_BF16: return tile_ways(Fp8Plain<__nv_bfloat16>{(const __nv_bfloat16 *)x, row_stride}, blocks, to, to2, rows, k, false, chained, stream);
        default: return tile_ways(Fp8Plain<float>{(const float *)x, row_stride}, blocks, to, to2, rows, k, false, chained, stream);
    }
}

template <typename Source>
static cudaError_t gated_ways(const Source &src, const Fp8Codes &by_row, const Fp8Codes &by_column, int rows, int f, cudaStream_t stream)
{
    if (by_row.q && by_column.q) return tile_launch<1 << kFp8Row | 1 << kFp8Column>(src, by_row, by_column, rows, 2 * f, true, true, stream);
    if (by_row.q) return tile_launch<1 << kFp8Row>(src, by_row, by_row, rows, 2 * f, true, true, stream);
    return tile_launch<1 << kFp8Column>(src, by_column, by_column, rows, 2 * f, true, true, stream);
}

cudaError_t launch_fp8_gated_gradient(const void *z, const void *dh, int type, int gelu, const Fp8Codes &by_row, const Fp8Codes &by_column, int rows, int f, cudaStream_t stream)
{
    if (type == TUNA_FP16) {
        if (gelu) return gated_ways(Fp8Gated<__half, true>{(const __half *)z, (const __half *)dh, f}, by_row, by_column, rows, f, stream);
        return gated_ways(Fp8Gated<__half, false>{(const __half *)z, (const __half *)dh, f}, by_row, by_column, rows, f, stream);
    }
    if (gelu) return gated_ways(Fp8Gated<__nv_bfloat16, true>{(const __nv_bfloat16 *)z, (const __nv_bfloat16 *)dh, f}, by_row, by_column, rows, f, stream);
    return gated_ways(Fp8Gated<__nv_bfloat16, false>{(const __nv_bfloat16 *)z, (const __nv_bfloat16 *)dh, f}, by_row, by_column, rows, f, stream);
}

// ---- the inverse

__device__ __forceinline__ void fp8_store(float *p, const float (&v)[4]) { *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]); }
template <typename T>
__device__ __forceinline__ void fp8_store(T *p, const float (&v)[8])
{
    *reinterpret_cast<uint4 *>(p) = make_uint4(mx_pack2<T>(v[0], v[1]), mx_pack2<T>(v[2], v[3]), mx_pack2<T>(v[4], v[5]), mx_pack2<T>(v[6], v[7]));
}

// o = code * scale in fp32 (exact: four significant bits; below fp32's range it rounds), rounded once to T.  A thread has 16 bytes of the result, COLS columns, of ROWS rows;
// grid (columns, rows).
template <typename T, int BLOCKS, int ROWS>
__global__ void __launch_bounds__(128)
fp8_dequant_kernel(const uint8_t *q, const uint8_t *s, T *o, int rows, int k)
{
    constexpr int COLS = 16 / sizeof(T);
    const int col = (blockIdx.x * 128 + threadIdx.x) * COLS;
    if (col >= k) return;
    for (long long row0 = (long long)blockIdx.y * ROWS; row0 < rows; row0 += (long long)gridDim.y * ROWS) {
        uint32_t codes[ROWS][COLS / 4];
        const int have = (int)min((long long)rows - row0, (long long)ROWS);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const uint8_t *at = q + (row0 + min(r, have - 1)) * k + col;
            if constexpr (COLS == 4) {
                codes[r][0] = __ldcg(reinterpret_cast<const uint32_t *>(at));
            } else {
                const uint2 w = __ldcg(reinterpret_cast<const uint2 *>(at));
                codes[r][0] = w.x;
                codes[r][1] = w.y;
            }
        }
        uint32_t byte[BLOCKS == kFp8Column ? COLS : BLOCKS == kFp8Row ? ROWS : 1];  // ROWS divides 128: the rows are of one block
        if constexpr (BLOCKS == kFp8Column) {
#pragma unroll
            for (int i = 0; i < COLS; ++i) byte[i] = __ldcg(s + ((row0 >> 9) * k + col + i) * 4 + ((row0 >> 7) & 3));
        } else if constexpr (BLOCKS == kFp8Row) {
#pragma unroll
            for (int r = 0; r < ROWS; ++r) byte[r] = __ldcg(s + ((long long)(col >> 9) * rows + row0 + min(r, have - 1)) * 4 + ((col >> 7) & 3));
        } else {
            byte[0] = s[(row0 >> 7) * div_up(k, kFp8Block) + (col >> 7)];  // by way of L1: few bytes, which everybody reads
        }
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            if (r >= have) break;
            float v[COLS];
#pragma unroll
            for (int i = 0; i < COLS; i += 4) {
                uint32_t h[2];
                fp8_decode4(codes[r][i / 4], h);
                const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&h[0])), b = __half22float2(*reinterpret_cast<const __half2 *>(&h[1]));
                const float n[4] = {a.x, a.y, b.x, b.y};
#pragma unroll
                for (int j = 0; j < 4; ++j) v[i + j] = n[j] * mx_scale_value(byte[BLOCKS == kFp8Column ? i + j : BLOCKS == kFp8Row ? r : 0]);
            }
            fp8_store(o + (row0 + r) * k + col, v);
        }
    }
}

template <typename T, int BLOCKS, int ROWS>
static cudaError_t dequant_rows(const void *q, const void *s, void *o, int rows, int k, cudaStream_t stream)
{
    const dim3 grid((unsigned)div_up(k, 16 / (int)sizeof(T) * 128), (unsigned)std::min(div_up(rows, ROWS), 65535));
    fp8_dequant_kernel<T, BLOCKS, ROWS><<<grid, 128, 0, stream>>>((const uint8_t *)q, (const uint8_t *)s, (T *)o, rows, k);
    return cudaGetLastError();
}

template <typename T, int BLOCKS>
static cudaError_t dequant_as(const void *q, const void *s, void *o, int rows, int k, cudaStream_t stream)
{
    return (long long)rows * k <= 1 << 20 ? dequant_rows<T, BLOCKS, 2>(q, s, o, rows, k, stream) : dequant_rows<T, BLOCKS, 8>(q, s, o, rows, k, stream);
}

template <typename T>
static cudaError_t dequant_any(const void *q, const void *s, int blocks, void *o, int rows, int k, cudaStream_t stream)
{
    switch (blocks) {
        case kFp8Row: return dequant_as<T, kFp8Row>(q, s, o, rows, k, stream);
        case kFp8Column: return dequant_as<T, kFp8Column>(q, s, o, rows, k, stream);
        default: return dequant_as<T, kFp8Square>(q, s, o, rows, k, stream);
    }
}

cudaError_t launch_fp8_dequant(const void *q, const void *s, int blocks, void *o, int type, int rows, int k, cudaStream_t stream)
{
    switch (type) {
        case TUNA_FP16: return dequant_any<__half>(q, s, blocks, o, rows, k, stream);
        case TUNA_BF16: return dequant_any<__nv_bfloat16>(q, s, blocks, o, rows, k, stream);
        default: return dequant_any<float>(q, s, blocks, o, rows, k, stream);
    }
}

}  // namespace tuna
