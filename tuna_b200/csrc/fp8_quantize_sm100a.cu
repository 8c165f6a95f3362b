// Quantizers of the 8-bit block-scaled format (fp8_format.cuh), their inverse, and the quantizer of a gated block's gradients.
//
// A block's scale is a power of two, so dividing by it is exact and the only rounding is that of the code.  A block by row is 16 lanes of a warp, one by column or a square one
// a tile of 128 x 128 that a CTA holds in registers: its numbers are read once, whatever is made of them.  Nothing is transposed: blocks by column are codes in the
// same place, with other scales.
//
// HBM bounds them (6.55 TB/s is the measured copy rate): 28672x4096 in fp32, square 88 us = 6.7 TB/s, by row 92, back 89; in bf16 square 58 and back 56 = 6.3, by row 59; 2048x28672 in
// bf16 by row and by column at once 45 us = 5.2 TB/s, where half of the issue slots are busy and a tile's loads, maxima and stores follow one another.  A gated block's
// gradients, 14336 features of 2048 tokens both ways, 79 us for 290 MB (GELU 88): the issue slots (62 % busy).
#include <algorithm>
#include <mutex>
#include "launchers.h"
#include "fp8_format.cuh"
#include "sm100_ptx.cuh"

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

// A lane has eight pieces of a row, eight columns each; 16 lanes are a row's block.  PARTS 1: a warp has 16 rows of a tile, a CTA of eight warps a tile.  PARTS 2: a warp
// has eight rows of two tiles, a CTA of sixteen warps both: the two projections of a gated block, whose numbers have a factor in common.  All of a lane's numbers are
// loaded before the first is used.
constexpr int kFp8Pieces = 8;
template <int PARTS>
struct Fp8Tile {
    static constexpr int kWarps = 8 * PARTS, kRows = kFp8Block / kWarps, kLaneRows = kRows / 2;
    // Piece i: part i / kLaneRows, row 2 (i % kLaneRows) from the lane's first
};

__device__ __forceinline__ uint32_t fp8_magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }  // compare as the numbers do, NaN above infinity

// Pieces' maxima over the 16 lanes that have the rest of their rows: in every step a lane keeps half of the pieces and sends the other half, so that in the end lanes 2 i
// and 2 i + 1 have that of piece i.  30 instructions for eight rows, where every lane taking part in every row's would be 64, and one scale a lane to work out instead of eight.
template <typename V, typename Max>
__device__ __forceinline__ V fp8_rows_max(V (&v)[kFp8Pieces], int lane, Max largest)
{
#pragma unroll
    for (int half = kFp8Pieces / 2; half >= 1; half >>= 1) {
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
    Mx8<T> v[kFp8Pieces];
    using Pair = decltype(v[0].pair(0));
    __device__ __forceinline__ static Pair with(Pair a, Pair b) { return __hmax2_nan(a, __habs2(b)); }
    __device__ __forceinline__ static float2 widen(__half2 p) { return __half22float2(p); }
    __device__ __forceinline__ static float2 widen(__nv_bfloat162 p) { return __bfloat1622float2(p); }
    __device__ __forceinline__ uint32_t row_max(int lane) const  // of piece (lane / 2) % 8
    {
        Pair m[kFp8Pieces];
#pragma unroll
        for (int r = 0; r < kFp8Pieces; ++r) m[r] = with(with(__habs2(v[r].pair(0)), v[r].pair(1)), __hmax2_nan(__habs2(v[r].pair(2)), __habs2(v[r].pair(3))));
        const float2 f = widen(fp8_rows_max(m, lane, [](Pair a, Pair b) { return __hmax2_nan(a, b); }));
        return max(fp8_magnitude(f.x), fp8_magnitude(f.y));
    }
    template <int FIRST, int COUNT>
    __device__ __forceinline__ void col_max(uint32_t (&m)[8]) const  // of the warp's rows of these pieces
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            Pair p = __habs2(v[FIRST].pair(i));
#pragma unroll
            for (int r = 1; r < COUNT; ++r) p = with(p, v[FIRST + r].pair(i));
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
        for (int r = 0; r < kFp8Pieces; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) m = with(m, v[r].pair(i));
        const float2 f = widen(m);
        return max(fp8_magnitude(f.x), fp8_magnitude(f.y));
    }
    __device__ __forceinline__ void values(int r, float (&f)[8]) const { v[r].values(f); }
};
struct Fp8RawFloat {
    float v[kFp8Pieces][8];
    __device__ __forceinline__ uint32_t row_max(int lane) const
    {
        uint32_t m[kFp8Pieces];
#pragma unroll
        for (int r = 0; r < kFp8Pieces; ++r) {
            m[r] = fp8_magnitude(v[r][0]);
#pragma unroll
            for (int i = 1; i < 8; ++i) m[r] = max(m[r], fp8_magnitude(v[r][i]));
        }
        return fp8_rows_max(m, lane, [](uint32_t a, uint32_t b) { return max(a, b); });
    }
    template <int FIRST, int COUNT>
    __device__ __forceinline__ void col_max(uint32_t (&m)[8]) const
    {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            m[i] = 0;
#pragma unroll
            for (int r = 0; r < COUNT; ++r) m[i] = max(m[i], fp8_magnitude(v[FIRST + r][i]));
            m[i] = max(m[i], __shfl_xor_sync(0xffffffffu, m[i], 16));
        }
    }
    __device__ __forceinline__ uint32_t lane_max() const
    {
        uint32_t m = 0;
#pragma unroll
        for (int r = 0; r < kFp8Pieces; ++r)
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

// Where a tile's numbers come from: rows row0, row0 + 2 .. of columns col .. col + 7 and, of a second part, the columns kPartCols() further on.
template <typename T, int PARTS>
struct Fp8Plain {
    const T *x;
    long long row_stride;
    using Raw = Fp8Raw<T>;
    static constexpr int kParts = PARTS;
    __device__ __forceinline__ int part_cols() const { return kFp8Block; }
    __device__ __forceinline__ int column_tile(int at, int) const { return PARTS * at; }
    __device__ __forceinline__ void load(Raw &to, long long row0, int col, int rows, int cols) const
    {
        constexpr int kLaneRows = Fp8Tile<PARTS>::kLaneRows;
#pragma unroll
        for (int i = 0; i < kFp8Pieces; ++i) {
            const long long row = row0 + 2 * (i % kLaneRows);
            const int at_col = col + i / kLaneRows * kFp8Block;
            const bool in = at_col < cols && row < rows;
            const T *at = x + row * row_stride + at_col;
            if constexpr (sizeof(T) == 2) {
                if (in) to.v[i].load(at);
                else to.v[i].zero();
            } else {
                Mx8<float> v;
                if (in) v.load(at);
                else v.zero();
                v.values(to.v[i]);
            }
        }
    }
};
// Eight columns of a gated block's gradients: of the gate, dh u act'(g), and of the other projection, dh act(g); or of one of them.
template <typename T, bool GELU>
__device__ __forceinline__ void fp8_gated_row(const Mx8<T> &g, const Mx8<T> &u, const Mx8<T> &d, float minus_zero, float (&of_gate)[8], float (&of_other)[8])
{
    float gv[8], uv[8], dv[8];
    g.values(gv);
    u.values(uv);
    d.values(dv);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const Fp8Two gate(gv[i], gv[i + 1]), dh(dv[i], dv[i + 1]);
        Fp8Two sigma, derivative;
        fp8_gate_and_slope<GELU>(gate, minus_zero, sigma, derivative);
        const float2 a = (dh * Fp8Two(uv[i], uv[i + 1]) * derivative).both(), b = (dh * gate * sigma).both();
        of_gate[i] = a.x, of_gate[i + 1] = a.y;
        of_other[i] = b.x, of_other[i + 1] = b.y;
    }
}
template <typename T, bool GELU>
__device__ __forceinline__ void fp8_gated_row(const Mx8<T> &g, const Mx8<T> &u, const Mx8<T> &d, float minus_zero, bool gate, float (&to)[8])
{
    float of_other[8];
    fp8_gated_row<T, GELU>(g, u, d, minus_zero, to, of_other);
    if (!gate)
#pragma unroll
        for (int i = 0; i < 8; ++i) to[i] = of_other[i];
}

// Columns 0 .. f - 1: the gradient of a gated block's gate, dh u act'(g); f .. 2f - 1: of the other projection, dh act(g).  z = [g | u].  What bounds it is the
// activation's arithmetic: where blocks end between the projections two parts share it, otherwise a tile is of either.
template <typename T, bool GELU, int PARTS>
struct Fp8Gated {
    const T *z, *dh;
    int f;
    float minus_zero = -0.0f;
    using Raw = Fp8RawFloat;
    static constexpr int kParts = PARTS;
    __device__ __forceinline__ int part_cols() const { return f; }
    // PARTS 1: tile t of the one and of the other projection, which read the same, follow one another, so that L2 has it
    __device__ __forceinline__ int column_tile(int at, int tiles) const { return PARTS == 2 ? at : (at & 1) ? (tiles + 1) / 2 + (at >> 1) : at >> 1; }
    __device__ __forceinline__ void load(Raw &to, long long row0, int col, int rows, int cols) const
    {
        constexpr int kLaneRows = Fp8Tile<PARTS>::kLaneRows, kBatch = PARTS == 2 ? 2 : 4;  // rows in flight
        const bool gate = col < f;
        const int at = gate ? col : col - f;  // f is a multiple of 16: eight columns are of one kind
#pragma unroll
        for (int r0 = 0; r0 < kLaneRows; r0 += kBatch) {
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
                if (in && (PARTS == 2 || gate)) u[r].load(zr + f);
                else u[r].zero();
            }
#pragma unroll
            for (int r = 0; r < kBatch; ++r) {
                if constexpr (PARTS == 2) fp8_gated_row<T, GELU>(g[r], u[r], d[r], minus_zero, to.v[r0 + r], to.v[kLaneRows + r0 + r]);
                else fp8_gated_row<T, GELU>(g[r], u[r], d[r], minus_zero, gate, to.v[r0 + r]);
            }
        }
    }
};

template <int PARTS>
struct Fp8TileShared {
    uint4 max[8 * PARTS][PARTS][32];  // of a warp's rows, column by column
    float inverse[PARTS][kFp8Block];
    uint32_t square[8 * PARTS];
    int none;  // a column's block is NaN
};

// The tile of columns kFp8Block ct .. and rows kFp8Block rt ..; `again`: `shared` was in use for another one.
template <int WAYS, typename Source>  // WAYS: 1 << kFp8Row | 1 << kFp8Column, one of them, or 1 << kFp8Square
__device__ __forceinline__ void fp8_quantize_tile(Source &src, uint8_t *q, uint8_t *s, uint8_t *q2, uint8_t *s2, int rows, int cols, int ct, int rt, bool again,
                                                  Fp8TileShared<Source::kParts> &shared)
{
    constexpr bool kRows = WAYS & (1 << kFp8Row), kCols = WAYS & (1 << kFp8Column), kSquare = WAYS & (1 << kFp8Square);
    constexpr int kParts = Source::kParts, kWarps = Fp8Tile<kParts>::kWarps, kLaneRows = Fp8Tile<kParts>::kLaneRows;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row_tiles = div_up(rows, kFp8Block), col_blocks = div_up(cols, kFp8Block);
    const int col = ct * kFp8Block + (lane & 15) * 8, part_cols = src.part_cols();
    const size_t step = 2 * (size_t)cols;
    {
        const long long row0 = (long long)rt * kFp8Block + warp * Fp8Tile<kParts>::kRows + (lane >> 4);
        typename Source::Raw raw;
        src.load(raw, row0, col, rows, cols);
        const int have = (int)min((long long)rows - row0, 2ll * kLaneRows);  // of the rows from row0 on
        // Codes of piece i; MASKED: zeros where a bit of `none` says so.  Two ways and no test in the common one: with it square blocks of 28672x4096 in bf16 took 73 us, so 55.
        auto write = [&](auto masked, uint8_t *to, int i, const float (&inverse)[8], uint32_t none) {
            float f[8];
            raw.values(i, f);
            uint2 w = make_uint2(fp8_encode4(f[0] * inverse[0], f[1] * inverse[1], f[2] * inverse[2], f[3] * inverse[3]),
                                 fp8_encode4(f[4] * inverse[4], f[5] * inverse[5], f[6] * inverse[6], f[7] * inverse[7]));
            if constexpr (decltype(masked)::value)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (none >> j & 1) (j < 4 ? w.x : w.y) &= ~(0xffu << (8 * (j & 3)));
            const int part = i / kLaneRows, r = i % kLaneRows;
            if (2 * r < have && col + part * part_cols < cols) *reinterpret_cast<uint2 *>(to + r * step + part * (size_t)part_cols) = w;
        };
        if constexpr (kRows) {
            const uint32_t e = fp8_scale(raw.row_max(lane));  // of piece (lane / 2) % 8
            const float mine = fp8_inverse(e);
            uint8_t *to = q + (size_t)row0 * cols + col;
            auto pieces = [&](auto masked) {
#pragma unroll
                for (int i = 0; i < kFp8Pieces; ++i) {
                    const float v = __shfl_sync(0xffffffffu, mine, (lane & 16) + 2 * i);
                    const uint32_t none = decltype(masked)::value && __shfl_sync(0xffffffffu, e, (lane & 16) + 2 * i) == 255u ? 255u : 0u;
                    write(masked, to, i, {v, v, v, v, v, v, v, v}, none);
                }
            };
            if (__any_sync(0xffffffffu, e == 255u)) pieces(Int<1>());
            else pieces(Int<0>());
            const int piece = (lane >> 1) & 7, block = ct + piece / kLaneRows * (part_cols / kFp8Block);
            const long long row = row0 + 2 * (piece % kLaneRows);
            if ((lane & 1) == 0 && row < rows && block < col_blocks) {
                uint8_t *at = s + ((long long)(block >> 2) * rows + row) * 4 + (block & 3);
                *at = (uint8_t)e;
                if (block + 1 == col_blocks)
                    for (int i = 1; i < 4 - (block & 3); ++i) at[i] = 0;
            }
        }
        if constexpr (kCols || kSquare) {
            if (again) __syncthreads();  // what was there before has been read
            uint8_t *to = (kRows ? q2 : q) + (size_t)row0 * cols + col, *words = kRows ? s2 : s;
            float inverse[kParts][8];
            uint32_t none[kParts] = {};
            if constexpr (kSquare) {
                static_assert(kParts == 1, "a tile is a block");
                uint32_t m = raw.lane_max();
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
                if (lane == 0) shared.square[warp] = m;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < kWarps; ++w) m = max(m, shared.square[w]);
                const uint32_t e = fp8_scale(m);
#pragma unroll
                for (int i = 0; i < 8; ++i) inverse[0][i] = fp8_inverse(e);
                none[0] = e == 255u ? 255u : 0u;
                if (threadIdx.x == 0) words[(long long)rt * col_blocks + ct] = (uint8_t)e;
            } else {
                auto maxima = [&](auto part) {
                    constexpr int kPart = decltype(part)::value;
                    uint32_t m[8];
                    raw.template col_max<kPart * kLaneRows, kLaneRows>(m);
                    if (lane < 16) {
                        shared.max[warp][kPart][2 * lane] = make_uint4(m[0], m[1], m[2], m[3]);
                        shared.max[warp][kPart][2 * lane + 1] = make_uint4(m[4], m[5], m[6], m[7]);
                    }
                };
                maxima(Int<0>());
                if constexpr (kParts == 2) maxima(Int<1>());
                if (threadIdx.x == 0) shared.none = 0;
                __syncthreads();
                if (threadIdx.x < kParts * kFp8Block) {  // one column each
                    const int part = threadIdx.x / kFp8Block, c = threadIdx.x % kFp8Block;
                    uint32_t e = 0;
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) e = max(e, reinterpret_cast<const uint32_t *>(shared.max[w][part])[c]);
                    e = fp8_scale(e);
                    shared.inverse[part][c] = e == 255u ? 0.0f : fp8_inverse(e);
                    if (e == 255u) shared.none = 1;
                    const long long at_col = (long long)ct * kFp8Block + (long long)part * part_cols + c;
                    if (at_col < cols) {
                        uint8_t *at = words + ((long long)(rt >> 2) * cols + at_col) * 4 + (rt & 3);
                        *at = (uint8_t)e;
                        if (rt + 1 == row_tiles)
                            for (int j = 1; j < 4 - (rt & 3); ++j) at[j] = 0;
                    }
                }
                __syncthreads();
#pragma unroll
                for (int part = 0; part < kParts; ++part) {
                    const float4 *from = reinterpret_cast<const float4 *>(shared.inverse[part] + 8 * (lane & 15));
                    *reinterpret_cast<float4 *>(inverse[part]) = from[0];
                    *reinterpret_cast<float4 *>(inverse[part] + 4) = from[1];
                }
                if (shared.none)
#pragma unroll
                    for (int part = 0; part < kParts; ++part)
#pragma unroll
                        for (int i = 0; i < 8; ++i) none[part] |= inverse[part][i] == 0.0f ? 1u << i : 0u;
            }
            auto pieces = [&](auto masked) {
#pragma unroll
                for (int i = 0; i < kFp8Pieces; ++i) write(masked, to, i, inverse[i / kLaneRows], none[i / kLaneRows]);
            };
            if (__any_sync(0xffffffffu, (none[0] | none[kParts - 1]) != 0u)) pieces(Int<1>());
            else pieces(Int<0>());
        }
    }
}

// One column of tiles, number `at` of `tiles`.
template <int WAYS, typename Source>
__device__ __forceinline__ void fp8_quantize_tiles(Source src, uint8_t *q, uint8_t *s, uint8_t *q2, uint8_t *s2, int rows, int cols, int at, int tiles, Fp8TileShared<Source::kParts> &shared)
{
    const int ct = src.column_tile(at, tiles);
    for (int rt = blockIdx.y; rt < div_up(rows, kFp8Block); rt += gridDim.y) fp8_quantize_tile<WAYS>(src, q, s, q2, s2, rows, cols, ct, rt, rt != (int)blockIdx.y, shared);
}

template <typename Source>
__host__ __device__ constexpr int fp8_tile_ctas(int ways)  // of an SM: what registers there are for
{
    return (sizeof(typename Source::Raw) > 128 ? 2 : ways & (ways - 1) ? 3 : 4) / Source::kParts;
}

template <int WAYS, typename Source>
__global__ void __launch_bounds__(256 * Source::kParts, fp8_tile_ctas<Source>(WAYS))
fp8_quantize_tile_kernel(const Source src, uint8_t *q, uint8_t *s, uint8_t *q2, uint8_t *s2, int rows, int cols, bool chained)
{
    __shared__ __align__(16) Fp8TileShared<Source::kParts> shared;
    if (chained) {
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
        asm volatile("griddepcontrol.wait;" ::: "memory");
    }
    fp8_quantize_tiles<WAYS>(src, q, s, q2, s2, rows, cols, blockIdx.x, gridDim.x, shared);
}

// The same, and the columns of a second matrix of as many rows, its blocks by column: what a weight's gradient multiplies, in one launch (gradients of 1552x1040 at 301 tokens
// 22.7 -> 21.3 us).
template <int WAYS, typename Source, typename T>
__global__ void __launch_bounds__(256 * Source::kParts, fp8_tile_ctas<Source>(WAYS))
fp8_quantize_two_kernel(const Source src, uint8_t *q, uint8_t *s, uint8_t *q2, uint8_t *s2, int rows, int cols, int tiles, const Fp8Plain<T, Source::kParts> x, uint8_t *xq, uint8_t *xs,
                        int x_cols)
{
    __shared__ __align__(16) Fp8TileShared<Source::kParts> shared;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if ((int)blockIdx.x < tiles) fp8_quantize_tiles<WAYS>(src, q, s, q2, s2, rows, cols, blockIdx.x, tiles, shared);
    else fp8_quantize_tiles<1 << kFp8Column>(x, xq, xs, xq, xs, rows, x_cols, blockIdx.x - tiles, gridDim.x - tiles, shared);
}

// ---- a gated block's gradients, streamed

// The same numbers as Fp8Gated's of two parts, for many tiles: one CTA an SM walks through them, and TMA has the next tile's three boxes of 32 KB under way while one is worked
// on.  Loaded by the lanes themselves, one tile a CTA, 14336 features of 2048 tokens took 115 us where this took 66 (the activation by
// fast approximations in both), most of it waiting: 512 threads of 128 registers leave no room for another
// CTA that would work meanwhile.
constexpr int kFp8BoxBytes = kFp8Block * kFp8Block * 2, kFp8StreamBytes = 2 * 3 * kFp8BoxBytes;

template <typename T, bool GELU>
struct Fp8GatedStaged {
    int f, col_tiles, tiles, stride, next;  // the tile that is copied next, and how far apart the CTA's are
    uint32_t box, bar;                      // of the tile that is loaded
    float minus_zero;
    const CUtensorMap *z, *dh;
    using Raw = Fp8RawFloat;
    static constexpr int kParts = 2;
    __device__ __forceinline__ int part_cols() const { return f; }
    __device__ __forceinline__ void copy()  // into the boxes at `box`
    {
        if (next >= tiles || threadIdx.x) return;
        const int rt = next / col_tiles, c = (next - rt * col_tiles) * kFp8Block;
        mbar_expect_tx(bar, 3 * kFp8BoxBytes);
        tma_load_2d(box, z, c, rt * kFp8Block, bar);
        tma_load_2d(box + kFp8BoxBytes, z, f + c, rt * kFp8Block, bar);
        tma_load_2d(box + 2 * kFp8BoxBytes, dh, c, rt * kFp8Block, bar);
    }
    __device__ __forceinline__ void load(Raw &to, long long, int, int, int)
    {
        constexpr int kLaneRows = Fp8Tile<2>::kLaneRows;
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        auto piece = [](uint32_t at) {
            Mx8<T> v;
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.r.x), "=r"(v.r.y), "=r"(v.r.z), "=r"(v.r.w) : "r"(at) : "memory");
            return v;
        };
#pragma unroll
        for (int r = 0; r < kLaneRows; ++r) {
            const uint32_t at = box + (uint32_t)(warp * Fp8Tile<2>::kRows + 2 * r + (lane >> 4)) * (2 * kFp8Block) + (uint32_t)(lane & 15) * 16u;
            fp8_gated_row<T, GELU>(piece(at), piece(at + kFp8BoxBytes), piece(at + 2 * kFp8BoxBytes), minus_zero, to.v[r], to.v[kLaneRows + r]);
        }
        __syncthreads();  // everybody has read the boxes
        copy();
        next += stride;
    }
};

template <typename T, bool GELU, int WAYS>
__global__ void __launch_bounds__(512, 1)
fp8_gated_stream_kernel(const __grid_constant__ CUtensorMap tmap_z, const __grid_constant__ CUtensorMap tmap_dh, uint8_t *q, uint8_t *s, uint8_t *q2, uint8_t *s2, int rows, int f,
                        float minus_zero, DeviceStatus *status)
{
    extern __shared__ __align__(128) uint8_t boxes[];
    __shared__ __align__(16) Fp8TileShared<2> shared;
    __shared__ __align__(8) uint64_t bars[2];
    __shared__ int s_abort;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        s_abort = 0;
        mbar_init(smem_u32(&bars[0]), 1);
        mbar_init(smem_u32(&bars[1]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        prefetch_map(&tmap_z);
        prefetch_map(&tmap_dh);
    }
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    Fp8GatedStaged<T, GELU> src;
    src.f = f;
    src.minus_zero = minus_zero;
    src.col_tiles = f / kFp8Block;
    src.tiles = src.col_tiles * div_up(rows, kFp8Block);
    src.stride = gridDim.x;
    src.next = blockIdx.x;
    src.z = &tmap_z;
    src.dh = &tmap_dh;
    auto turn = [&](int b) {
        src.box = smem_u32(boxes) + (uint32_t)(b * 3 * kFp8BoxBytes);
        src.bar = smem_u32(&bars[b]);
    };
    for (int b = 0; b < 2; ++b) {
        turn(b);
        src.copy();
        src.next += src.stride;
    }
    int turns = 0;
    for (int t = blockIdx.x; t < src.tiles; t += gridDim.x, ++turns) {
        turn(turns & 1);
        const bool ok = mbar_wait(src.bar, (uint32_t)(turns >> 1) & 1u, &s_abort, status, 320);
        if (__syncthreads_or(!ok)) {  // given up: no copy may land in what is no longer this CTA's
            if (threadIdx.x == 0)
                for (int i = 0; i < 2; ++i)
                    for (const long long t0 = clock64(); !mbar_try_wait(smem_u32(&bars[(turns + i) & 1]), (uint32_t)((turns + i) >> 1) & 1u) && t + i * (int)gridDim.x < src.tiles && clock64() - t0 < kWaitCycles;) {}
            return;
        }
        const int rt = t / src.col_tiles;
        fp8_quantize_tile<WAYS>(src, q, s, q2, s2, rows, 2 * f, t - rt * src.col_tiles, rt, turns > 0, shared);
    }
}

// What a launch quantizes beside its own matrix: nothing where q is null.
struct Fp8Second {
    const void *x;
    Fp8Codes to;
    int cols;
};

static cudaLaunchConfig_t tile_config(int tiles, int rows, int threads, bool chained, cudaLaunchAttribute &attr, cudaStream_t stream)
{
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)tiles, (unsigned)std::min(div_up(rows, kFp8Block), 65535));
    lc.blockDim = dim3((unsigned)threads);
    lc.stream = stream;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = &attr;
    lc.numAttrs = chained ? 1 : 0;
    return lc;
}

template <int WAYS, typename Source>
static cudaError_t tile_launch(const Source &src, int tiles, const Fp8Codes &to, const Fp8Codes &to2, int rows, int cols, bool chained, cudaStream_t stream)
{
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t lc = tile_config(tiles, rows, 256 * Source::kParts, chained, attr, stream);
    return cudaLaunchKernelEx(&lc, fp8_quantize_tile_kernel<WAYS, Source>, src, (uint8_t *)to.q, (uint8_t *)to.s, (uint8_t *)to2.q, (uint8_t *)to2.s, rows, cols, chained);
}

// Part of a gradient's call: by row, by column, or both, and x by column.
template <int WAYS, typename Source, typename T>
static cudaError_t gradient_launch(const Source &src, int tiles, const Fp8Codes &to, const Fp8Codes &to2, int rows, int cols, const Fp8Second &x, cudaStream_t stream)
{
    if (!x.to.q) return tile_launch<WAYS>(src, tiles, to, to2, rows, cols, true, stream);
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t lc = tile_config(tiles + div_up(x.cols, Source::kParts * kFp8Block), rows, 256 * Source::kParts, true, attr, stream);
    return cudaLaunchKernelEx(&lc, fp8_quantize_two_kernel<WAYS, Source, T>, src, (uint8_t *)to.q, (uint8_t *)to.s, (uint8_t *)to2.q, (uint8_t *)to2.s, rows, cols, tiles,
                              Fp8Plain<T, Source::kParts>{(const T *)x.x, x.cols}, (uint8_t *)x.to.q, (uint8_t *)x.to.s, x.cols);
}
template <typename T, typename Source>
static cudaError_t gradient_ways(const Source &src, int tiles, const Fp8Codes &by_row, const Fp8Codes &by_column, int rows, int cols, const Fp8Second &x, cudaStream_t stream)
{
    if (by_row.q && by_column.q) return gradient_launch<1 << kFp8Row | 1 << kFp8Column, Source, T>(src, tiles, by_row, by_column, rows, cols, x, stream);
    if (by_row.q) return gradient_launch<1 << kFp8Row, Source, T>(src, tiles, by_row, by_row, rows, cols, Fp8Second{nullptr, {nullptr, nullptr}, 0}, stream);
    return gradient_launch<1 << kFp8Column, Source, T>(src, tiles, by_column, by_column, rows, cols, x, stream);
}

template <typename T>
static cudaError_t tile_ways(const Fp8Plain<T, 1> &src, int blocks, const Fp8Codes &to, const Fp8Codes &to2, int rows, int cols, cudaStream_t stream)
{
    const int tiles = div_up(cols, kFp8Block);
    switch (blocks) {
        case kFp8Column: return tile_launch<1 << kFp8Column>(src, tiles, to, to2, rows, cols, false, stream);
        case kFp8Square: return tile_launch<1 << kFp8Square>(src, tiles, to, to2, rows, cols, false, stream);
        default: return tile_launch<1 << kFp8Row | 1 << kFp8Column>(src, tiles, to, to2, rows, cols, false, stream);
    }
}

cudaError_t launch_fp8_quantize_tiles(const void *x, int type, long long row_stride, int blocks, const Fp8Codes &to, const Fp8Codes &to2, int rows, int k, cudaStream_t stream)
{
    switch (type) {
        case TUNA_FP16: return tile_ways(Fp8Plain<__half, 1>{(const __half *)x, row_stride}, blocks, to, to2, rows, k, stream);
        case TUNA_BF16: return tile_ways(Fp8Plain<__nv_bfloat16, 1>{(const __nv_bfloat16 *)x, row_stride}, blocks, to, to2, rows, k, stream);
        default: return tile_ways(Fp8Plain<float, 1>{(const float *)x, row_stride}, blocks, to, to2, rows, k, stream);
    }
}

template <typename T>
static cudaError_t second_alone(const Fp8Second &x, int rows, cudaStream_t stream)
{
    return tile_launch<1 << kFp8Column>(Fp8Plain<T, 1>{(const T *)x.x, x.cols}, div_up(x.cols, kFp8Block), x.to, x.to, rows, x.cols, true, stream);
}

template <typename T, bool GELU, int WAYS>
static cudaError_t stream_launch(const Fp8GradientArgs &a, const Fp8Codes &to, const Fp8Codes &to2)
{
    static bool attr_set[64] = {false};
    static std::mutex mu;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || dev < 0 || dev >= 64) return e != cudaSuccess ? e : cudaErrorInvalidDevice;
    {
        std::lock_guard<std::mutex> lock(mu);
        if (!attr_set[dev]) {
            e = cudaFuncSetAttribute(fp8_gated_stream_kernel<T, GELU, WAYS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFp8StreamBytes);
            if (e != cudaSuccess) return e;
            attr_set[dev] = true;
        }
    }
    const int f = a.cols / 2;
    CUtensorMap z, dh;
    const CUtensorMapDataType type = sizeof(T) == 2 && a.type == TUNA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    DeviceStatus *status = device_status_word();
    if (!status || !make_tensor_map_2d(&z, type, a.z, (uint64_t)a.cols, (uint64_t)a.rows, (uint64_t)a.cols * 2, kFp8Block, kFp8Block, CU_TENSOR_MAP_SWIZZLE_NONE) ||
        !make_tensor_map_2d(&dh, type, a.dy, (uint64_t)f, (uint64_t)a.rows, (uint64_t)f * 2, kFp8Block, kFp8Block, CU_TENSOR_MAP_SWIZZLE_NONE))
        return cudaErrorUnknown;
    cudaLaunchAttribute attr;
    cudaLaunchConfig_t lc = tile_config(a.sm_count, 1, 512, true, attr, a.stream);
    lc.dynamicSmemBytes = kFp8StreamBytes;
    return cudaLaunchKernelEx(&lc, fp8_gated_stream_kernel<T, GELU, WAYS>, z, dh, (uint8_t *)to.q, (uint8_t *)to.s, (uint8_t *)to2.q, (uint8_t *)to2.s, a.rows, f, -0.0f, status);
}

template <typename T, bool GELU>
static cudaError_t gated_gradient(const Fp8GradientArgs &a, const Fp8Second &x)
{
    const int f = a.cols / 2;
    const long long tiles = (long long)(f / kFp8Block) * div_up(a.rows, kFp8Block);
    if (f % kFp8Block == 0 && tiles >= 2 * a.sm_count && tiles < 1 << 30) {
        if (x.to.q) {
            const cudaError_t e = second_alone<T>(x, a.rows, a.stream);
            if (e != cudaSuccess) return e;
        }
        if (a.by_row.q && a.by_column.q) return stream_launch<T, GELU, 1 << kFp8Row | 1 << kFp8Column>(a, a.by_row, a.by_column);
        if (a.by_row.q) return stream_launch<T, GELU, 1 << kFp8Row>(a, a.by_row, a.by_row);
        return stream_launch<T, GELU, 1 << kFp8Column>(a, a.by_column, a.by_column);
    }
    if (f % kFp8Block == 0)
        return gradient_ways<T>(Fp8Gated<T, GELU, 2>{(const T *)a.z, (const T *)a.dy, f}, f / kFp8Block, a.by_row, a.by_column, a.rows, a.cols, x, a.stream);
    return gradient_ways<T>(Fp8Gated<T, GELU, 1>{(const T *)a.z, (const T *)a.dy, f}, div_up(a.cols, kFp8Block), a.by_row, a.by_column, a.rows, a.cols, x, a.stream);
}

template <typename T>
static cudaError_t gradient_of(const Fp8GradientArgs &a, const Fp8Second &x)
{
    if (a.z) return a.gelu ? gated_gradient<T, true>(a, x) : gated_gradient<T, false>(a, x);
    if (!a.by_column.q) return launch_fp8_quantize_rows(a.dy, a.type, a.cols, a.by_row.q, a.by_row.s, a.rows, a.cols, true, a.stream);
    return gradient_ways<T>(Fp8Plain<T, 1>{(const T *)a.dy, a.cols}, div_up(a.cols, kFp8Block), a.by_row, a.by_column, a.rows, a.cols, x, a.stream);
}

cudaError_t launch_fp8_gradient(const Fp8GradientArgs &a)
{
    // x in the same launch where it is of dy's type
    const Fp8Second x = {a.x, a.x_to, a.x_cols}, none = {nullptr, {nullptr, nullptr}, 0};
    const bool together = x.to.q && a.x_type == a.type && a.by_column.q;
    if (x.to.q && !together) {
        const cudaError_t e = a.x_type == TUNA_FP16 ? second_alone<__half>(x, a.rows, a.stream) : second_alone<__nv_bfloat16>(x, a.rows, a.stream);
        if (e != cudaSuccess) return e;
    }
    return a.type == TUNA_FP16 ? gradient_of<__half>(a, together ? x : none) : gradient_of<__nv_bfloat16>(a, together ? x : none);
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
