// Products of microscaled 4-bit matrices (format and layout: mx_format.cuh) on the 5th-generation tensor cores of sm_100a:
// o[t][r] = sum over k of x[t][k] * w[r][k], one matrix or one per expert, the tokens of an expert being a range of rows
// that the device knows.
//
// The tensor cores multiply e2m1 codes and apply both blocks' scales themselves (tcgen05.mma kind::mxf4, scale_vec::2X), so
// there is nothing to dequantize: per 256 columns a tile's codes are copied to shared memory and its scales written to tensor
// memory, and four MMAs of 64 columns add to fp32 accumulators.  Weights are operand A (128 rows), tokens operand B (N
// columns): few tokens cost few columns.
//
// Persistent CTAs, or pairs of CTAs (cta_group::2: 256 weight rows, every CTA stages its own 128 and half of the tokens), of 12 warps:
//   warp 0     MMA issue (one elected lane; in a pair the first CTA's)
//   warp 1     TMA producer of the weights' codes and scales
//   warp 2     TMA producer of the tokens' codes and, in wide tiles, their scales.  A tile starts at any token, a copy at a multiple
//              of four words: the scales' copies start up to three words early, and the readers skip those
//   warp 3     tensor-memory allocation; scales of the tokens in tiles of up to 16 tokens, as 4-byte copies (cp.async).  In wide
//              tiles this warp would set the pace (0.30 us per 256 columns of a 256-token tile before any other work), in narrow
//              ones the small TMA copies would (4096x4096 at 1 token 7.3 us, so 4.5)
//   warps 4-7  epilogue: tensor memory -> registers -> output type -> memory, of more than 16 tokens by way of shared memory,
//              where rows become contiguous.  Up to 128 tokens leave tensor memory before the first goes to memory
//   warps 8-11 scales, one warp per lane quarter: a word of scales is four blocks (128 columns) of one row or token, and the MMAs want that of
//              row r at lane r % 32, column r / 32, in every quarter.  So each warp reads all words of a stage from shared memory and
//              writes them to its quarter (tcgen05.st).  Copies by the tensor pipe (tcgen05.cp) take its time: 57344x8192 at 4096
//              tokens 923 us with them, 756 without.
// RESIDENT: a few tokens in 16 bits are quantized by the CTA itself before its first MMA, all of K, and stay in shared memory: no
// launch before this one.
//
// Work split.  Tiles are numbered expert by expert and handed out in turn; no sum is cut, so nothing is added up outside of a
// tile.  Up to 16 tokens one matrix is cut into row tiles of equal height, a multiple of 8 up to 128, a whole number of them for
// every CTA: the MMAs compute 128 rows whatever the height, which costs nothing where the weights' bytes are the bound.  Where
// a tile has at most 64 (32) of the 128 rows, two (four) chunks of K lie side by side in it ("folded"): the MMA's rows are
// those of the tile for each chunk in turn, its columns the tokens for each chunk, and the epilogue adds up the blocks where the
// two belong together (4096x4096 at 1 token 6.6 us unfolded, 4.5 folded).  More tokens, and experts, go in tiles of 256 rows
// on pairs, of as many tokens as an estimate (mx_pair_tokens) says.
//
// Every wait is bounded, as in the other pipeline kernels.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <mutex>
#include "launchers.h"
#include "mx_format.cuh"
#include "sm100_ptx.cuh"
#include "tcgen05.cuh"

namespace tuna {

constexpr int kMxWarps = 12;
constexpr int kMxEpilogueWarp0 = 4;
constexpr int kMxScaleWarp0 = 8;
constexpr int kMxMaxStages = 12;
constexpr int kMxStageTokens = 128;     // tokens of the output staging buffer
constexpr int kMxDirectTokens = 16;     // tiles of up to so many tokens are stored from registers
constexpr int kMxSlackBytes = 1024;     // of shared memory at the end: scales of columns that a tile does not have are read from behind its own
constexpr uint32_t kMxFoldBytes = kMxDirectTokens * kBlockRows * 4;  // where the parts of a folded tile are added up
// Up to here the weights of one matrix count as constants and are copied ahead of the dependency wait; above, they follow ordinary stream order as in
// tuna_matmul: a kernel before this one that has let its dependents start may still be writing them.  Graph replay, us, ahead / after: codes, 512x512
// at 100 tokens 3.2 / 3.5, 4096x4096 at 65 6.4 / 7.6, 6144x4096 at 256 8.6 / 9.0, 10240x8192 at 777 and 8192x8192 at 4096 the same;
// below the line 28672x4096 at 43 13.6 / 14.9.  Copies into L2 ahead of the wait, which would be in order, do not help (4096x4096 at 65
// 7.6, 11000x4128 at 70 8.9 -> 10.0).
constexpr int kMxAheadTokens = 64;
constexpr int kMxResidentRows = 4;      // loads in flight of a quantizing warp
constexpr uint32_t kMxScaleBytes = 2 * kBlockRows * 4;  // of the weights' scales in a stage
constexpr int kMxSmemMax = 225 * 1024;   // dynamic shared memory of a CTA alone on its SM (1 KB is the kernel's static part, 1 KB the system's)
constexpr int kMxSmemHalf = 111 * 1024;  // of one that leaves room for another

struct MxParams {
    const uint32_t *xs;   // words of the tokens' scales [words][n]
    const int *offsets;   // first token of each expert, and the end; nullptr: one matrix, all tokens
    void *o;
    DeviceStatus *status;
    int m, n, k;
    int experts;
    int tile_tok;   // N
    int chunks;     // ceil(k / 256)
    int units;      // stages of a tile: ceil(chunks / fold)
    int fold_log;   // log2(fold): chunks side by side in a stage
    int words;      // ceil(k / 128)
    int row_tiles;
    int w_bytes;    // of the weights in a stage
    int x_rows;     // tokens in a stage of a CTA
    int xs_pitch;   // bytes between the copies of a stage's token scales
    int xs_bytes;   // of all of them
    int xs_skew;    // words from where tmap_xs starts, which is a multiple of 16 bytes, to p.xs
    int flex;       // row tiles of equal height: tile t has the groups of 8 rows t * groups / row_tiles up to the next tile's
    int groups;     // m / 8
    int x_bf16;     // RESIDENT: type of the tokens
    const void *x;  // RESIDENT: the tokens [n][k]
    int last_steps; // MMAs of the last chunk: 64 columns each
    int stages;
    int nd;         // accumulators that are free of one another
    int d_cols;     // tensor-memory columns of an accumulator: tokens of a tile times fold
    int d_step;     // where the second one starts; nd = 1: 0, or where it overlaps the first
    int sf_col;     // where the scales start
    int ahead;      // what says which weights are wanted is there before the dependency wait, and they are read from then on
};

// The tiles of a worker in order, and where each lies.
struct MxTiles {
    int next_tile, step, tiles, units, row_tiles, tile_tok;
    const int *first_tile, *begin, *count;  // per expert (shared memory)
    int e, rt, tok0, valid;  // the tile: its expert, its rows' number, its first token and how many there are
    __device__ void init(const MxParams &p, int worker, int workers, const int *tables)
    {
        next_tile = worker;
        step = workers;
        units = p.units;
        row_tiles = p.row_tiles;
        tile_tok = p.tile_tok;
        begin = tables;
        count = tables + p.experts;
        first_tile = tables + 2 * p.experts;
        tiles = first_tile[p.experts];
        e = 0;
    }
    __device__ bool next()
    {
        if (next_tile >= tiles) return false;
        while (next_tile >= first_tile[e + 1]) ++e;  // tiles come in increasing order, and the last expert's end is their number
        const int local = next_tile - first_tile[e], tok_tiles = div_up(count[e], tile_tok);
        rt = local / tok_tiles;
        const int tt = local - rt * tok_tiles, width = (div_up(count[e], tok_tiles) + 15) & ~15;  // tiles of equal width, as many as the widest need
        tok0 = begin[e] + tt * width;
        valid = min(width, count[e] - tt * width);
        next_tile += step;
        return true;
    }
    __device__ int total_units() const { return next_tile < tiles ? ((tiles - 1 - next_tile) / step + 1) * units : 0; }
};

__device__ __forceinline__ void tma_load_1d(uint32_t dst, const CUtensorMap *map, int c0, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.1d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2}], [%3];" ::"r"(dst), "l"(map), "r"(c0), "r"(bar) : "memory");
}

// The same as tma_load_3d, the lines it brings to L2 being kept there by `policy`.
__device__ __forceinline__ void tma_load_3d_policy(uint32_t dst, const CUtensorMap *map, int c0, int c1, int c2, uint32_t bar, uint64_t policy)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3, %4}], [%5], %6;" ::"r"(dst), "l"(map),
                 "r"(c0), "r"(c1), "r"(c2), "r"(bar), "l"(policy)
                 : "memory");
}

// One lane's words to eight columns of this warp's lanes.
__device__ __forceinline__ void tc_st_x8(uint32_t taddr, const uint32_t (&v)[8])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
                 "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

// D[tmem] (+)= (A * scale A) (B * scale B), 64 columns of e2m1 with a scale per 32
template <int CG>
__device__ __forceinline__ void tc_mma_mx(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate)
{
    if (CG == 1)
        asm volatile(
            "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
            " tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}"
            ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
            " tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}"
            ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
}

// Instruction descriptor, kind::mxf4: A and B e2m1 (1 at bits 7-9 and 10-11), both K-major, N >> 3 at bits 17-22, e8m0 scales
// (bit 23), M >> 7 at bits 27-28, which half of a scale word A and B use (0 or 2) at bits 29-30 and 4-5.
template <int CG>
__host__ __device__ constexpr uint32_t mx_idesc(int cols, int half)
{
    return (1u << 7) | (1u << 10) | ((uint32_t)(cols >> 3) << 17) | (1u << 23) | ((uint32_t)CG << 27) | ((uint32_t)(2 * half) << 29) | ((uint32_t)(2 * half) << 4);
}

// Words of a half (128 columns) of the tokens' scales that a lane holds, for so many columns of an accumulator.
__host__ __device__ constexpr int mx_token_words(int cols) { return cols <= 64 ? 2 : cols <= 128 ? 4 : 8; }
// Tensor-memory columns of a stage's scales: four per half for the weights, four per half and 128 tokens.
__host__ __device__ constexpr uint32_t mx_scale_cols(int token_words) { return token_words == 8 ? 24 : 16; }

// First row of row block b (a CTA's share of a tile).
__device__ __forceinline__ int mx_row(const MxParams &p, int b) { return p.flex ? 8 * (int)((long long)b * p.groups / p.row_tiles) : b * kBlockRows; }

// Four bytes of global memory, or zeros; the barrier counts the thread's copies in when they have landed.
__device__ __forceinline__ void cp_async_word(uint32_t dst, const uint32_t *src, bool have)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(have ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) { asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory"); }

// Quantizes the tokens' numbers, all of K: warp `w` of `warps` takes every warps-th (chunk, token).  Codes as TMA would have put
// them (128-byte swizzle), scale words [stage][half][token of a chunk of the stage].
template <typename T, int R>  // R: loads in flight
__device__ __forceinline__ void mx_quantize_resident(const MxParams &p, int w, int warps, int lane, uint32_t codes_at, uint32_t words_at)
{
    const int items = (p.units << p.fold_log) * p.n;  // chunks behind the last one are zeros
    for (int i0 = w; i0 < items; i0 += R * warps) {
        Mx8<T> v[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int i = i0 + r * warps, c = i / p.n, t = i - c * p.n, col = c * kMxChunk + lane * 8;
            if (i < items && col < p.k) v[r].load(static_cast<const T *>(p.x) + (size_t)t * p.k + col);
            else v[r].zero();
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int i = i0 + r * warps, c = i / p.n, t = i - c * p.n;
            if (i >= items) break;
            uint32_t e = mx_scale(v[r].largest());
            const float inverse = mx_inverse(e);
            float f[8];
            v[r].values(f);
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] *= inverse;
            const uint32_t codes = e == 255u ? 0u : mx_encode8(f);
            // 16-byte piece lane / 4 of the token's 128 bytes, XORed with the token's number mod 8
            asm volatile("st.shared.u32 [%0], %1;" ::"r"(codes_at + ((uint32_t)c * p.x_rows + (uint32_t)t) * kMxChunkBytes + ((((uint32_t)lane >> 2) ^ ((uint32_t)t & 7u)) << 4) + ((uint32_t)lane & 3u) * 4u),
                         "r"(codes)
                         : "memory");
            const int unit = c >> p.fold_log, at = (c - (unit << p.fold_log)) * p.x_rows + t;
            e <<= 8 * ((lane >> 2) & 3);  // four neighbouring blocks make a word
            e |= __shfl_xor_sync(0xffffffffu, e, 4);
            e |= __shfl_xor_sync(0xffffffffu, e, 8);
            if ((lane & 15) == 0) asm volatile("st.shared.u32 [%0], %1;" ::"r"(words_at + (uint32_t)unit * 512u + (uint32_t)(lane >> 4) * 256u + (uint32_t)at * 4u), "r"(e) : "memory");
        }
    }
}

// CG: CTAs of a worker (1 or 2).  NW: mx_token_words.  RESIDENT: the tokens are numbers in 16 bits and quantized here.
// Tiles of up to 16 tokens of one matrix (NW 2) leave room for a second CTA on the SM: that of the next launch, which copies its first
// weights meanwhile.
template <int CG, int NW, bool RESIDENT, typename OT>
__global__ void __launch_bounds__(32 * kMxWarps, NW == 2 ? 2 : 1)
mx_gemm_kernel(const __grid_constant__ MxParams p, const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_w2,
               const __grid_constant__ CUtensorMap tmap_ws, const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_xs)
{
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[3 * kMxMaxStages + 4];
    __shared__ uint32_t s_tmem_base;
    __shared__ int s_abort;

    constexpr uint32_t kTmemCols = NW == 2 ? 256 : 512;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int rank = CG == 1 ? 0 : (int)cluster_ctarank();
    const int worker = blockIdx.x / CG, workers = gridDim.x / CG;
    const int N = p.tile_tok, S = p.stages;
    // [stages of weights][of tokens][of the weights' scales][of the tokens' scales][staging buffer][tables]; the MMAs read 128
    // rows, in low tiles past their stage's end.  RESIDENT: of tokens, all of a tile's stages.
    const int x_stages = RESIDENT ? p.units : S;
    const uint32_t base = smem_u32(smem), w_bytes = (uint32_t)p.w_bytes, x_bytes = (uint32_t)(p.x_rows << p.fold_log) * kMxChunkBytes;
    const uint32_t x_ring = base + (uint32_t)S * w_bytes, ws_ring = x_ring + (uint32_t)x_stages * x_bytes, xs_ring = ws_ring + (uint32_t)S * kMxScaleBytes;
    const uint32_t staging = xs_ring + (uint32_t)(x_stages * p.xs_bytes);
    constexpr uint32_t kTokPitch = kBlockRows * (uint32_t)sizeof(OT) + (sizeof(OT) == 2 ? 16 : 0);  // 16-bit results: 16 bytes more, so that a column of 8 tokens meets all banks
    constexpr uint32_t kStagingBytes = kMxStageTokens * kTokPitch;
    int *tables = reinterpret_cast<int *>(smem + (staging - base) + (p.fold_log ? kMxFoldBytes : N > kMxDirectTokens ? kStagingBytes : 0));

    // landed: a stage's copies; full: its scales are written as well; empty: its MMAs are done
    const uint32_t landed = smem_u32(&bars[0]), full = landed + 8 * kMxMaxStages, empty = full + 8 * kMxMaxStages, d_full = empty + 8 * kMxMaxStages, d_empty = d_full + 16;
    volatile int *abort_flag = &s_abort;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (warp == 1) {
        auto count = [&](int i) {
            if (i < kMxMaxStages) return RESIDENT ? 1 : NW == 2 ? 34 : 2;  // landed: weights, tokens, the lanes that copy their scales
            if (i < 2 * kMxMaxStages) return 4 * CG;            // full: the scale warps of each CTA
            return i < 3 * kMxMaxStages + 2 ? 1 : 4 * CG;       // empty, d_full: a commit; d_empty: the epilogue warps of each CTA
        };
        for (int i = lane; i < 3 * kMxMaxStages + 4; i += 32) mbar_init(landed + 8 * i, count(i));
        if (lane == 0) s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (elect_one_sync()) {
            prefetch_map(&tmap_w);
            prefetch_map(&tmap_ws);
            if (!RESIDENT) prefetch_map(&tmap_x);
            if (NW > 2) prefetch_map(&tmap_xs);
        }
    }
    if (warp == 3) {
        if (CG == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem_base)), "r"(kTmemCols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem_base)), "r"(kTmemCols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        }
    }
    auto depend = [] { asm volatile("griddepcontrol.wait;" ::: "memory"); };
    if (warp == 0) {  // the experts' tiles: first token, tokens, tiles before
        if (p.offsets && !p.ahead) depend();
        int before = 0, reached = 0;
        for (int e0 = 0; e0 < p.experts; e0 += 32) {
            const int e = e0 + lane;
            int begin = 0, cnt = p.n;
            if (p.offsets) {  // whatever they are: inside the tokens, and none below one before it
                auto largest = [&](int v) {
#pragma unroll
                    for (int d = 1; d < 32; d <<= 1) v = max(v, __shfl_up_sync(0xffffffffu, v, d));
                    return max(v, reached);
                };
                begin = largest(min(max(__ldcg(p.offsets + min(e, p.experts)), 0), p.n));
                const int end = max(begin, min(max(__ldcg(p.offsets + min(e + 1, p.experts)), 0), p.n));
                cnt = end - begin;
                reached = __shfl_sync(0xffffffffu, end, 31);
            }
            if (e >= p.experts) cnt = 0;
            const int mine = div_up(cnt, N) * p.row_tiles;
            int sum = mine;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, sum, d);
                if (lane >= d) sum += v;
            }
            if (e < p.experts) {
                tables[e] = begin;
                tables[p.experts + e] = cnt;
                tables[2 * p.experts + e] = before + sum - mine;
            }
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (lane == 0) tables[3 * p.experts] = before;
    }
    tc_fence_before();
    __syncthreads();
    if (CG == 2) cluster_sync_all();  // the other CTA's barriers are there
    tc_fence_after();
    const uint32_t tmem = s_tmem_base;
    const uint32_t sf_col = (uint32_t)p.sf_col;
    const int fold = 1 << p.fold_log, part = kBlockRows >> p.fold_log;  // rows of a part
    constexpr int kScaleCols = (int)mx_scale_cols(NW), kTokenCols = NW < 4 ? 4 : NW;  // of a stage, and of a half of its tokens
    MxTiles tile;
    tile.init(p, worker, workers, tables);
    const int total = tile.total_units();
    auto tile_cols = [&] { return (tile.valid + 8 * CG - 1) & -(8 * CG); };  // tokens that the tile's MMAs cover

    if (RESIDENT && warp != 1) {  // the weights are on their way meanwhile
        depend();
        const int w = warp == 0 ? 0 : warp - 1;
        auto quantize = [&](auto type) {
            using T = decltype(type);
            if ((p.units << p.fold_log) * p.n <= 2 * (kMxWarps - 1)) mx_quantize_resident<T, 2>(p, w, kMxWarps - 1, lane, x_ring, xs_ring);
            else mx_quantize_resident<T, kMxResidentRows>(p, w, kMxWarps - 1, lane, x_ring, xs_ring);
        };
        if (p.x_bf16) quantize(__nv_bfloat16());
        else quantize(__half());
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the MMAs read the codes
        asm volatile("bar.sync 2, %0;" ::"n"(32 * (kMxWarps - 1)) : "memory");
    }
    // Whoever makes a bounded wait that ends only after the kernels before this one waits for those first.
    if (warp == 0) {
        if (CG == 1 || rank == 0) {
            depend();
            Ring ru, rd;
            bool ok = true;
            int second = 0;  // which accumulator
            // -------------------------------------------------------------- MMA issue
            constexpr uint64_t sw128 = ((uint64_t)((1024u >> 4) | (1u << 14) | (2u << 29))) << 32;  // 8-row groups 1024 bytes apart, version 1, 128-byte swizzle
            while (ok && tile.next()) {
                const uint32_t idesc = mx_idesc<CG>(p.fold_log ? p.d_cols : tile_cols(), 0);
                constexpr uint32_t kHalf = mx_idesc<CG>(0, 1) ^ mx_idesc<CG>(0, 0);
                ok = mbar_wait_warp(d_empty + 8 * rd.idx, rd.phase ^ 1, abort_flag, p.status, 203);
                const uint32_t d = tmem + (uint32_t)(second * p.d_step);
                second ^= 1;
                for (int c = 0; ok && c < p.units; ++c) {
                    ok = mbar_wait_warp(full + 8 * ru.idx, ru.phase, abort_flag, p.status, 204);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one_sync()) {
                        const uint64_t a = sw128 | (uint64_t)(((base + (uint32_t)ru.idx * w_bytes) & 0x3FFFFu) >> 4);
                        const uint64_t b = sw128 | (uint64_t)(((x_ring + (uint32_t)(RESIDENT ? c : ru.idx) * x_bytes) & 0x3FFFFu) >> 4);
                        const uint32_t sfa = tmem + sf_col + (uint32_t)(ru.idx * kScaleCols), sfb = sfa + 8;
                        const int steps = c + 1 == p.units && !p.fold_log ? p.last_steps : 4;
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            if (kk < steps)
                                tc_mma_mx<CG>(d, a + 2 * kk, b + 2 * kk, (kk & 1) ? idesc ^ kHalf : idesc, sfa + 4 * (kk >> 1), sfb + kTokenCols * (kk >> 1),
                                              c == 0 && kk == 0 ? 0u : 1u);
                        if (CG == 1) {
                            tc_commit(empty + 8 * ru.idx);
                            if (c + 1 == p.units) tc_commit(d_full + 8 * rd.idx);
                        } else {
                            tc_commit_pair(empty + 8 * ru.idx);
                            if (c + 1 == p.units) tc_commit_pair(d_full + 8 * rd.idx);
                        }
                    }
                    __syncwarp();
                    ru.advance(S);
                }
                rd.advance(p.nd);
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------------ weights
        Ring ru;
        bool ok = true;
        int issued = 0;
        // The weights of tiles of up to 128 tokens leave L2 first.  A program that goes through a few times what L2 holds, again and again, then
        // finds a part of it there the next time, where the oldest lines leaving first would have replaced all (us, first / as other lines, of 0.3 GB of
        // matrices in turn: 28672x4096 at 16 tokens 12.5 / 13.4, 57344x8192 at 43 42.0 / 45.3, eight 28672x4096 of 32 67.3 / 71.0; of 0.6 GB
        // 28672x4096 at 16 12.5 / 13.4, 57344x8192 at 43 42.5 / 43.9; 3 GB the same).  Where several tiles of tokens want the same weights, they mostly want them at
        // once: 512x4096 at 4096 tokens (32 tiles) 9.2 / 9.1, 512x16384 at 1000 17.5 / 17.3, 4096x14336 at 500 20.6 / 20.6, eight 14336x4096 of
        // 800, 600 of them one expert's, 63.4 / 64.2, eight 4096x14336 of 710, 500 one's, 56.3 / 58.4; asking, tile by tile, for the number of
        // token tiles gives 9.4, 17.5, 21.0, 63.5, 59.0.  In wider tiles it costs (57344x8192 at 4096 tokens 753 -> 761).
        uint64_t first_out;
        if constexpr (NW < 8) asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(first_out));
        if (!p.ahead) depend();
        while (ok && tile.next()) {
            const int block = CG * tile.rt + rank, row = mx_row(p, block), rows = mx_row(p, block + 1) - row;
            const CUtensorMap *map = !p.flex || rows == 8 * div_up(p.groups, p.row_tiles) ? &tmap_w : &tmap_w2;  // boxes of the taller and of the lower tiles
            for (int c = 0; c < p.units; ++c, ru.advance(S)) {
                if (issued++ == S) depend();
                ok = mbar_wait_warp(empty + 8 * ru.idx, ru.phase ^ 1, abort_flag, p.status, 200);
                if (!ok) break;
                if (elect_one_sync()) {
                    const uint32_t bar = landed + 8 * ru.idx;
                    mbar_expect_tx(bar, (uint32_t)(rows << p.fold_log) * kMxChunkBytes + kMxScaleBytes);
                    for (int f = 0; f < fold; ++f) {  // chunks behind the last one read as zeros
                        const int chunk = (c << p.fold_log) + f;
                        const uint32_t to = base + (uint32_t)ru.idx * w_bytes + (uint32_t)(f * part) * kMxChunkBytes;
                        if constexpr (NW < 8) tma_load_3d_policy(to, map, 0, row, tile.e * p.chunks + chunk, bar, first_out);
                        else tma_load_3d(to, map, 0, row, tile.e * p.chunks + chunk, bar);
                        tma_load_2d(ws_ring + (uint32_t)ru.idx * kMxScaleBytes + (uint32_t)(f * part) * 8u, &tmap_ws, row, tile.e * p.words + 2 * chunk, bar);
                    }
                }
                __syncwarp();
            }
        }
        // The MMAs' commits have arrived at every stage in use before the CTA leaves.
        depend();
        if (total < S) ru = Ring();
        for (int i = min(S, total); ok && i > 0; --i, ru.advance(S)) ok = mbar_wait_warp(empty + 8 * ru.idx, total < S ? 0u : ru.phase ^ 1, abort_flag, p.status, 210);
    } else if (warp == 2 && !RESIDENT) {
        // ------------------------------------------------------------------ tokens' codes
        Ring ru;
        bool ok = true;
        constexpr int kPieces = NW == 8 ? 2 : 1;  // 128 words each
        const uint32_t xs_copy = (uint32_t)(min(N, 128) + 4) * 4u;
        depend();
        while (ok && tile.next()) {
            const int tok = tile.tok0 + rank * (tile_cols() / CG);
            for (int c = 0; c < p.units; ++c, ru.advance(S)) {
                ok = mbar_wait_warp(empty + 8 * ru.idx, ru.phase ^ 1, abort_flag, p.status, 211);
                if (!ok) break;
                if (elect_one_sync()) {
                    const uint32_t bar = landed + 8 * ru.idx;
                    mbar_expect_tx(bar, x_bytes + (NW > 2 ? 2 * kPieces * xs_copy : 0u));
                    tma_load_3d(x_ring + (uint32_t)ru.idx * x_bytes, &tmap_x, 0, tok, c << p.fold_log, bar);
                    if constexpr (NW > 2) {
#pragma unroll
                        for (int h = 0; h < 2; ++h)  // a word behind the last one reads as zeros
#pragma unroll
                            for (int j = 0; j < kPieces; ++j)
                                tma_load_1d(xs_ring + (uint32_t)(ru.idx * p.xs_bytes + (kPieces * h + j) * p.xs_pitch), &tmap_xs,
                                            (int)((((unsigned)(2 * c + h) * (unsigned)p.n + (unsigned)(tile.tok0 + p.xs_skew)) & ~3u) + 128u * j), bar);
                    }
                }
                __syncwarp();
            }
        }
    } else if (warp == 3 && !RESIDENT && NW == 2) {
        // ------------------------------------------------------------------ tokens' scales in narrow tiles
        Ring ru;
        bool ok = true;
        depend();
        while (ok && tile.next()) {
            for (int c = 0; c < p.units; ++c, ru.advance(S)) {
                ok = mbar_wait_warp(empty + 8 * ru.idx, ru.phase ^ 1, abort_flag, p.status, 201);
                if (!ok) break;
                const uint32_t to = xs_ring + (uint32_t)(ru.idx * p.xs_bytes) + 4u * lane;
#pragma unroll
                for (int j = 0; j < NW; ++j) {  // token t of the stage's chunk f: zeros behind the last word, where the codes are zeros too
                    const int f = p.fold_log ? (32 * j + lane) / p.x_rows : 0, t = 32 * j + lane - f * p.x_rows;
                    if (f >= fold || t >= tile.valid) continue;  // whatever lies there scales columns that nobody reads
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int word = 2 * ((c << p.fold_log) + f) + h;
                        cp_async_word(to + 128u * (NW * h + j), p.xs + (size_t)min(word, p.words - 1) * p.n + tile.tok0 + t, word < p.words);
                    }
                }
                cp_async_arrive(landed + 8 * ru.idx);
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp >= kMxScaleWarp0) {
        // ------------------------------------------------------------------ scales to tensor memory
        const int quarter = warp - kMxScaleWarp0;
        const uint32_t lanes = tmem + ((uint32_t)(32 * quarter) << 16) + sf_col;
        const uint32_t leader_full = CG == 1 ? full : map_to_rank(full, 0);
        Ring ru;
        bool ok = true;
        if (!RESIDENT) depend();
        while (ok && tile.next()) {
            for (int c = 0; c < p.units; ++c, ru.advance(S)) {
                // a stage's copies have landed, so its MMAs of the round before are done, and its scales may be overwritten
                ok = mbar_wait_warp(landed + 8 * ru.idx, ru.phase, abort_flag, p.status, 212);
                if (!ok) break;
                tc_fence_after();
                const uint32_t to = lanes + (uint32_t)(ru.idx * kScaleCols), x_at = xs_ring + (uint32_t)((RESIDENT ? c : ru.idx) * p.xs_bytes);
                // One store if it fits: what a store takes from the MMAs is hardly a matter of its size (57344x8192 at 4096 tokens, 721 us without any:
                // with 8 columns 75 more, with 16 83, with 32 102, with 8 and 16 apart 138; but 32 columns a stage leave room for four
                // stages of 256 tokens instead of five, 770 us against 735).
                uint32_t v[kScaleCols];
#pragma unroll
                for (int i = 0; i < 8; ++i) {  // weights, half i / 4: MMA row 32 (i % 4) + lane is row `of` of part f
                    const int row = 32 * (i & 3) + lane, f = row >> (7 - p.fold_log), of = row & (part - 1);
                    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[i]) : "r"(ws_ring + (uint32_t)ru.idx * kMxScaleBytes + (uint32_t)((2 * f + (i >> 2)) * part + of) * 4u));
                }
#pragma unroll
                for (int i = 8; i < (int)kScaleCols; ++i) v[i] = 0;
#pragma unroll
                for (int h = 0; h < 2; ++h) {  // tokens: column 32 j + lane, half h
                    const uint32_t skip = NW == 2 ? 0u : (((unsigned)(2 * c + h) * (unsigned)p.n + (unsigned)(tile.tok0 + p.xs_skew)) & 3u) * 4u;
#pragma unroll
                    for (int j = 0; j < NW; ++j) {
                        const uint32_t at = NW == 2 ? (uint32_t)(NW * h + j) * 128u : (uint32_t)((NW == 8 ? 2 * h + (j >> 2) : h) * p.xs_pitch) + (uint32_t)(j & 3) * 128u + skip;
                        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[8 + kTokenCols * h + j]) : "r"(x_at + at + 4u * lane));
                    }
                }
                if constexpr (NW == 8) {
                    uint32_t w[8], x[16];
#pragma unroll
                    for (int i = 0; i < 8; ++i) w[i] = v[i];
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[i] = v[8 + i];
                    tc_st_x8(to, w);
                    tc_st_x16(to + 8, x);
                } else {
                    tc_st_x16(to, v);
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (CG == 1) mbar_arrive(full + 8 * ru.idx);
                    else mbar_arrive_cluster(leader_full + 8 * ru.idx);
                }
            }
        }
    } else if (warp >= kMxEpilogueWarp0) {
        // ------------------------------------------------------------------ epilogue
        const int quarter = warp & 3, thread = threadIdx.x - 32 * kMxEpilogueWarp0;
        const uint32_t tmem_q = tmem + ((uint32_t)(32 * quarter) << 16);
        OT *o = static_cast<OT *>(p.o);
        Ring rd;
        depend();
        int row0 = 0, rows = 0;
        // The staging buffer's tokens, which are the tile's from t0 on, to memory: 16 bytes a thread and step.
        auto copy_out = [&](int t0) {
            constexpr int kPieces = kBlockRows * (int)sizeof(OT) / 16, kStep = 128 / kPieces;
            const int piece = thread % kPieces, end = min(kMxStageTokens, tile.valid - t0);
            if (piece * (16 / (int)sizeof(OT)) >= rows) return;
            uint8_t *to = reinterpret_cast<uint8_t *>(o + (size_t)(tile.tok0 + t0) * p.m + row0) + 16 * piece;
#pragma unroll 8
            for (int t = thread / kPieces; t < end; t += kStep) {
                uint4 v;
                asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(staging + (uint32_t)t * kTokPitch + 16u * piece));
                *reinterpret_cast<uint4 *>(to + (size_t)t * p.m * sizeof(OT)) = v;
            }
        };
        // 32 tokens of the accumulator at `d`, columns from t on.
        auto fill_from = [&](uint32_t d, int t, uint32_t at) {
            if constexpr (sizeof(OT) == 2) {
                // Fragments of 8 rows x 8 tokens, packed, are written transposed (stmatrix): 16 bytes = 8 rows of one token.
                uint32_t lo[16], hi[16];
                tc_ld_16x256b_x4(d + t, lo);
                tc_ld_16x256b_x4(d + (16u << 16) + t, hi);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                const uint32_t to = at + (uint32_t)(lane & 7) * kTokPitch + (uint32_t)(4 * quarter + (lane >> 3)) * 16u;
                auto pack = [](uint32_t a, uint32_t b) { return mx_pack2<OT>(__uint_as_float(a), __uint_as_float(b)); };
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    stmatrix_x4_trans(to + 8u * i * kTokPitch, pack(lo[4 * i], lo[4 * i + 1]), pack(lo[4 * i + 2], lo[4 * i + 3]), pack(hi[4 * i], hi[4 * i + 1]), pack(hi[4 * i + 2], hi[4 * i + 3]));
            } else {
#pragma unroll
                for (int h = 0; h < 32; h += 16) {
                    float v[16];
                    tc_ld_x16(d + t + h, v);
#pragma unroll
                    for (int i = 0; i < 16; ++i) asm volatile("st.shared.f32 [%0], %1;" ::"r"(at + (uint32_t)(h + i) * kTokPitch + (uint32_t)thread * 4u), "f"(v[i]) : "memory");
                }
            }
        };
        const uint32_t leader_d_empty = CG == 1 ? d_empty : map_to_rank(d_empty, 0);
        auto drained = [&] {  // the accumulator may be overwritten
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (CG == 1) mbar_arrive(d_empty + 8 * rd.idx);
                else mbar_arrive_cluster(leader_d_empty + 8 * rd.idx);
            }
        };
        int second = 0;
        for (; tile.next(); second ^= 1) {
            const bool ok = mbar_wait_warp(d_full + 8 * rd.idx, rd.phase, abort_flag, p.status, 206);
            if (bar_any(1, 128, !ok)) break;  // the four warps go on together or not at all
            tc_fence_after();
            const uint32_t d = tmem_q + (uint32_t)(second * p.d_step);
            row0 = mx_row(p, CG * tile.rt + rank);
            rows = min(mx_row(p, CG * tile.rt + rank + 1), p.m) - row0;
            if (p.fold_log) {
                // Part f's sums of row i are lane part * f + i, columns x_rows * f ..: added up in the order of the parts.
                const int f = thread >> (7 - p.fold_log);
                float *sums = reinterpret_cast<float *>(smem + (staging - base));
                float v[16];
                tc_ld_x16(d + f * p.x_rows, v);
#pragma unroll
                for (int t = 0; t < 16; ++t)
                    if (t < tile.valid) sums[t * kBlockRows + thread] = v[t];
                drained();
                asm volatile("bar.sync 1, 128;" ::: "memory");
                const int i = thread & (part - 1);
                for (int t = f; t < tile.valid && i < rows; t += fold) {
                    float sum = sums[t * kBlockRows + i];
                    for (int g = 1; g < fold; ++g) sum += sums[t * kBlockRows + g * part + i];
                    o[(size_t)(tile.tok0 + t) * p.m + row0 + i] = mx_convert<OT>(sum);
                }
                asm volatile("bar.sync 1, 128;" ::: "memory");  // they have been read
            } else if (N <= kMxDirectTokens) {
                float v[16];
                tc_ld_x16(d, v);
                drained();
                OT *to = o + (size_t)tile.tok0 * p.m + row0 + thread;
                if (thread < rows) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (i < tile.valid) to[(size_t)i * p.m] = mx_convert<OT>(v[i]);
                }
            } else {
                // Of two accumulators that overlap, the columns they share first: then the other one may be written.
                const bool shared = p.nd == 1 && p.d_step;
                const int turn = shared && second == 0 ? p.d_step : 0;
                for (int b = 0; b < N; b += kMxStageTokens) {
                    const int t0 = b + turn < N ? b + turn : b + turn - N;
                    asm volatile("bar.sync 1, 128;" ::: "memory");  // what was staged before has been copied
#pragma unroll
                    for (int h = 0; h < kMxStageTokens; h += 32)
                        if (t0 + h < tile.valid) fill_from(d, t0 + h, staging + (uint32_t)h * kTokPitch);
                    if (shared ? b == 0 : b + kMxStageTokens >= N) drained();
                    asm volatile("bar.sync 1, 128;" ::: "memory");
                    copy_out(t0);
                }
            }
            rd.advance(p.nd);
        }
    }

    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (CG == 2) cluster_sync_all();
    if (warp == 3) {
        tc_fence_after();
        if (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
    }
}

// ------------------------------------------------------------------ host side

struct MxPlan {
    int cg, tile_tok, words, stages, nd, d_cols, d_step, sf_col;
    bool resident;
    int flex, fold_log, row_tiles, w_bytes, x_rows, xs_copy, xs_pitch, xs_bytes;
    int workers;
    size_t smem;
};

// Microseconds that tiles of 256 rows and `cols` tokens take on `pairs` pairs, beside what a launch costs: rounds of tiles, each with its
// steps of 256 columns (the tensor pipe's four MMAs, which take hardly less for few tokens; wide tiles at the rate of the copies
// to shared memory as well) and what of a wide tile's epilogue nothing hides; what all tiles copy, from L2; the weights,
// from HBM.  Fitted to 1250 launches (graph replay; 11 matrices from 512x16384 to 57344x8192, 17 to 4096 tokens, every width): what it
// chooses takes 1.6 % longer than the fastest width in the mean, 20 % at worst (2048x2048 at 17 tokens). All of them read weights ahead of
// the dependency wait, as those above 64 tokens no longer do; that adds up to 1.2 us to a launch in a chain and was not fitted again.
static double mx_pair_us(int m, int n, int k, int cols, int pairs)
{
    const int row_tiles = div_up(m, 2 * kBlockRows), chunks = div_up(k, kMxChunk);
    const double tiles = (double)row_tiles * div_up(n, cols);
    const double rounds = std::ceil(tiles / pairs);
    const int width = div_up(div_up(n, div_up(n, cols)), 16) * 16;  // tiles are of equal width
    const double step = cols <= 128 ? 0.183 + 0.00013 * width : 0.036 + 0.00118 * width;
    const double work = rounds * (std::max(0.0, 0.0086 * width - 0.5) + chunks * step);
    const double copies = tiles * (2 * kBlockRows + cols) * chunks * 136.0 / 21.7e6, weights = (double)m * k * (17.0 / 32) / 8.1e6;
    return std::sqrt(work * work + copies * copies + weights * weights);
}

static int mx_pair_tokens(int m, int n, int k, int pairs)
{
    static const int widths[] = {256, 192, 176, 160, 128, 112, 96, 80, 64, 48, 32, 16, 0};
    int best = 0;
    double best_us = 0;
    for (int i = 0; widths[i]; ++i) {
        const int cols = widths[i];
        if (div_up(n, div_up(n, cols)) <= widths[i + 1]) continue;  // the next narrower one holds the same tiles
        const double us = mx_pair_us(m, n, k, cols, pairs);
        if (!best || us < best_us) best = cols, best_us = us;
    }
    return best;
}

// Tokens of a tile of experts: their numbers are on the device, so it goes by the mean.  Narrow enough that an expert of the mean
// size fills a good part of a tile, wide enough that popular ones do not read their weights often (us, 64 / 128 / 176 / 256: eight experts
// 28672x4096 of 4 in the mean 70 / - / - / -, eight 4096x14336 of 37 51 / 43 / 45 / 47 and of 187 101 / 72 / 68 / 72, sixteen 4096x4096 of
// 250 73 / 55 / 51 / 52, eight 14336x4096 of 100 68 / 57 / 60 / 57, 64 2048x1024 of 2 13.5 / - / - / -).
static int mx_expert_tokens(int mean) { return mean <= 24 ? 64 : mean <= 110 ? 128 : 176; }

static MxPlan mx_plan(int m, int n, int k, int experts, int x_type, int o_type, bool grouped, int sm_count)
{
    MxPlan l = {};
    const int chunks = div_up(k, kMxChunk);
    l.cg = grouped || n > kMxDirectTokens ? 2 : 1;
    l.workers = sm_count / l.cg;
    if (l.cg == 1) {
        l.flex = 1;
        l.tile_tok = kMxDirectTokens;
        l.row_tiles = (int)std::min<long long>(m / 8, div_up_ll(m, (long long)kBlockRows * sm_count) * sm_count);
        const int height = 8 * div_up(m / 8, l.row_tiles);
        l.fold_log = height <= 32 ? 2 : height <= 64 ? 1 : 0;
        l.w_bytes = (l.fold_log ? kBlockRows : height) * kMxChunkBytes;
    } else {
        // Rows in tiles of 256, also where that leaves the last round of tiles short: lower ones that fill it copy more tokens per row
        // (us, 256 / lower: 28672x4096 at 43 tokens 14.0 / 15.0, 4096x14336 at 256 17.0 / 20.1, 57344x8192 at 43 43.1 / 42.7).
        l.tile_tok = grouped ? mx_expert_tokens(div_up(n, experts)) : mx_pair_tokens(m, n, k, l.workers);
        l.row_tiles = div_up(m, 2 * kBlockRows);
        l.w_bytes = kBlockRows * kMxChunkBytes;
    }
    const int fold = 1 << l.fold_log;
    l.x_rows = l.fold_log ? div_up(n, 8) * 8 : l.tile_tok / l.cg;
    l.d_cols = l.fold_log ? l.x_rows * fold : l.tile_tok;
    const int words = l.words = l.cg == 1 ? 2 : std::max(4, mx_token_words(l.d_cols));  // the kernels that there are: launch_mx_as
    const size_t room = words == 2 ? kMxSmemHalf : kMxSmemMax;
    const size_t pitch = kBlockRows * (o_type == TUNA_FP32 ? 4 : 2) + (o_type == TUNA_FP32 ? 0 : 16);
    size_t fixed = (l.fold_log ? kMxFoldBytes : l.tile_tok > kMxDirectTokens ? kMxStageTokens * pitch : 0) + (3 * (size_t)experts + 1) * 4 + kMxSlackBytes;
    const size_t w_stage = (size_t)l.w_bytes + kMxScaleBytes;
    l.xs_copy = std::min(l.tile_tok, 128) + 4;  // words
    l.xs_pitch = div_up(l.xs_copy * 4, 128) * 128;
    l.xs_bytes = words == 2 ? 512 : 2 * (words == 8 ? 2 : 1) * l.xs_pitch;
    size_t x_stage = (size_t)l.x_rows * fold * kMxChunkBytes + l.xs_bytes;
    // Tokens that the CTAs quantize themselves: one round of the quantizing warps, and shared memory left for stages enough.  (bf16, us, so / a
    // quantizing launch before it: 4096x4096 at 1 token 4.4 / 5.5, at 2 4.6 / 5.5, with eight loads in flight at 4 5.7 / 5.7; 28672x4096 at 1 13.1 /
    // 13.5.)
    const int rows8 = div_up(n, 8) * 8, units = div_up(chunks, fold);
    const size_t resident = (size_t)units * (rows8 * fold * kMxChunkBytes + l.xs_bytes);
    l.resident = l.cg == 1 && x_type != TUNA_MXFP4 && n * units * fold <= kMxResidentRows * (kMxWarps - 1) && resident + 4 * w_stage + fixed <= room;
    if (l.resident) {
        l.x_rows = rows8;
        fixed += resident;
        x_stage = 0;
    }
    l.stages = (int)std::min<size_t>(kMxMaxStages, (room - fixed) / (w_stage + x_stage));
    const int tmem_cols = words == 2 ? 256 : 512, scale_cols = (int)mx_scale_cols(words);
    l.nd = 2 * l.d_cols + std::min(l.stages, 4) * scale_cols <= tmem_cols ? 2 : 1;
    // two accumulators that share the columns in the middle, where two whole ones do not fit
    if (l.nd == 2) l.d_step = l.d_cols;
    else if (l.d_cols == 2 * kMxStageTokens) l.d_step = kMxStageTokens;
    l.sf_col = l.d_cols + l.d_step;
    l.stages = std::min(l.stages, (tmem_cols - l.sf_col) / scale_cols);
    // the last stage's MMAs read 128 rows
    l.smem = std::max((size_t)l.stages * (w_stage + x_stage) + fixed, (size_t)(l.stages - 1) * l.w_bytes + kBlockRows * kMxChunkBytes);
    return l;
}

bool mx_gemm_takes(int m, int n, int k, int experts, int x_type, bool grouped, int sm_count)
{
    if (x_type == TUNA_MXFP4) return true;
    return !grouped && n <= kMxDirectTokens && mx_plan(m, n, k, experts, x_type, TUNA_FP16, grouped, sm_count).resident;
}

struct MxMaps {
    CUtensorMap w, w2, ws, x, xs;
};

template <int CG, int NW, bool RESIDENT, typename OT>
static int launch_mx(const MxParams &p, const MxMaps &maps, int ctas, size_t smem, cudaStream_t stream)
{
    static bool attr_set[64] = {false};
    static std::mutex mu;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return TUNA_ERR_NO_DEVICE;
    {
        std::lock_guard<std::mutex> lock(mu);
        if (!attr_set[dev]) {
            if (cudaFuncSetAttribute(mx_gemm_kernel<CG, NW, RESIDENT, OT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMxSmemMax) != cudaSuccess) return TUNA_ERR_NO_DEVICE;
            attr_set[dev] = true;
        }
    }
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)ctas);
    lc.blockDim = dim3(32 * kMxWarps);
    lc.dynamicSmemBytes = smem;
    lc.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = CG;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    lc.attrs = attr;
    lc.numAttrs = CG == 1 ? 1 : 2;
    return cudaLaunchKernelEx(&lc, mx_gemm_kernel<CG, NW, RESIDENT, OT>, p, maps.w, maps.w2, maps.ws, maps.x, maps.xs) == cudaSuccess ? TUNA_OK : TUNA_ERR_LAUNCH;
}

template <typename OT>
static int launch_mx_as(const MxPlan &l, const MxParams &p, const MxMaps &maps, int ctas, cudaStream_t stream)
{
    if (l.cg == 1) return l.resident ? launch_mx<1, 2, true, OT>(p, maps, ctas, l.smem, stream) : launch_mx<1, 2, false, OT>(p, maps, ctas, l.smem, stream);
    return l.words == 4 ? launch_mx<2, 4, false, OT>(p, maps, ctas, l.smem, stream) : launch_mx<2, 8, false, OT>(p, maps, ctas, l.smem, stream);
}

int launch_mx_gemm(const MxGemmArgs &a)
{
    const MxPlan l = mx_plan(a.m, a.n, a.k, a.experts, a.numbers ? TUNA_MXFP4 : a.x_type, a.o_type, a.offsets != nullptr, a.sm_count);
    MxParams p;
    std::memset(&p, 0, sizeof(p));
    p.xs = (const uint32_t *)a.xs; p.x = a.x; p.offsets = (const int *)a.offsets; p.o = a.o;
    p.m = a.m; p.n = a.n; p.k = a.k; p.experts = a.experts;
    p.x_bf16 = a.x_type == TUNA_BF16;
    p.tile_tok = l.tile_tok;
    p.chunks = div_up(a.k, kMxChunk);
    p.words = div_up(a.k, kMxScaleCols);
    p.last_steps = div_up(a.k - (p.chunks - 1) * kMxChunk, 64);
    p.units = div_up(p.chunks, 1 << l.fold_log); p.fold_log = l.fold_log;
    p.row_tiles = l.row_tiles; p.w_bytes = l.w_bytes; p.flex = l.flex; p.groups = a.m / 8;
    p.x_rows = l.x_rows; p.xs_pitch = l.xs_pitch; p.xs_bytes = l.xs_bytes;
    p.stages = l.stages; p.nd = l.nd; p.d_cols = l.d_cols; p.d_step = l.d_step; p.sf_col = l.sf_col;
    // Experts: after a quantizing launch, which lets this one start when the kernels that may have written the offsets and weights are done.
    p.ahead = a.offsets ? a.numbers != nullptr : a.n <= kMxAheadTokens;
    p.status = device_status_word();
    if (!p.status) return TUNA_ERR_NO_DEVICE;
    // the kernel numbers tiles, a worker's stages, and words of scales in 32 bits
    const long long tiles = ((long long)div_up(a.n, l.tile_tok) + a.experts - 1) * p.row_tiles;  // at most
    if (tiles >= 1ll << 30 || (tiles / l.workers + 2) * p.chunks >= 1ll << 30 || (long long)a.experts * p.words >= 1ll << 30 ||
        (long long)(p.words + 8) * a.n >= 1ll << 31)
        return TUNA_ERR_TOO_LARGE;

    MxMaps maps;
    auto tiles_of = [](CUtensorMap *map, const void *at, uint64_t rows, uint64_t chunks, uint32_t box_rows, uint32_t box_chunks) {  // [chunks][rows][128 bytes]
        return make_tensor_map_3d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, at, kMxChunkBytes, rows, chunks, kMxChunkBytes, rows * kMxChunkBytes, kMxChunkBytes, box_rows, box_chunks,
                                  CU_TENSOR_MAP_SWIZZLE_128B);
    };
    if (!tiles_of(&maps.w, a.q, (uint64_t)a.m, (uint64_t)a.experts * p.chunks, l.flex ? 8u * (uint32_t)div_up(p.groups, p.row_tiles) : kBlockRows, 1)) return TUNA_ERR_NO_DEVICE;
    maps.w2 = maps.x = maps.xs = maps.w;
    if (l.flex && p.groups % p.row_tiles && !tiles_of(&maps.w2, a.q, (uint64_t)a.m, (uint64_t)p.chunks, 8u * (uint32_t)(p.groups / p.row_tiles), 1)) return TUNA_ERR_NO_DEVICE;
    if (!make_tensor_map_2d(&maps.ws, CU_TENSOR_MAP_DATA_TYPE_UINT32, a.s, (uint64_t)a.m, (uint64_t)a.experts * p.words, (uint64_t)a.m * 4, (uint32_t)kBlockRows >> l.fold_log, 2, CU_TENSOR_MAP_SWIZZLE_NONE))
        return TUNA_ERR_NO_DEVICE;
    if (!l.resident && !tiles_of(&maps.x, a.x, (uint64_t)a.n, (uint64_t)p.chunks, (uint32_t)l.x_rows, 1u << l.fold_log)) return TUNA_ERR_NO_DEVICE;
    if (l.words > 2) {
        p.xs_skew = (int)((reinterpret_cast<uintptr_t>(a.xs) & 15) / 4);
        const uint64_t dim = (uint64_t)p.words * a.n + p.xs_skew;
        const uint32_t box = (uint32_t)l.xs_copy;
        if (!make_tensor_map_nd(&maps.xs, CU_TENSOR_MAP_DATA_TYPE_UINT32, (const uint32_t *)a.xs - p.xs_skew, 1, &dim, nullptr, &box, CU_TENSOR_MAP_SWIZZLE_NONE)) return TUNA_ERR_NO_DEVICE;
    }
    if (a.numbers && launch_mx_quantize(a.numbers, a.x_type, a.k, const_cast<void *>(a.x), const_cast<void *>(a.xs), a.n, a.k, 1, a.stream, a.offsets ? kMxChainedAfter : kMxChained) != cudaSuccess)
        return TUNA_ERR_LAUNCH;
    const int ctas = l.workers * l.cg;
    switch (a.o_type) {
        case TUNA_FP16: return launch_mx_as<__half>(l, p, maps, ctas, a.stream);
        case TUNA_BF16: return launch_mx_as<__nv_bfloat16>(l, p, maps, ctas, a.stream);
        default: return launch_mx_as<float>(l, p, maps, ctas, a.stream);
    }
}

}  // namespace tuna
