// Products of microscaled 4-bit matrices (format and layout: mx_format.cuh) on the 5th-generation tensor cores of sm_100a:
// o[t][r] = sum over k of x[t][k] * w[r][k], one matrix or one per expert, the tokens of an expert being a range of rows
// that the device knows.
//
// The tensor cores multiply e2m1 codes and apply both blocks' scales themselves (tcgen05.mma kind::mxf4, scale_vec::2X), so
// there is nothing to dequantize: per 256 columns a tile's codes and scales are copied to shared memory, the scales go on
// to tensor memory (tcgen05.cp), and four MMAs of 64 columns add to fp32 accumulators.  Weights are operand A (128 rows),
// tokens operand B (N columns): few tokens cost few columns.
//
// Persistent CTAs of 8 warps:
//   warp 0     MMA issue (one elected lane): the stage's scales to tensor memory, then its MMAs
//   warp 1     TMA producer: codes and scales of the weights, codes of the tokens
//   warp 2     scales of the tokens.  Tiles start at any token, so these words are 4-byte copies (cp.async) that put each
//              one where tcgen05.cp wants it: row t at lane t % 32, word t / 32
//   warp 3     tensor-memory allocation
//   warps 4-7  epilogue: tensor memory -> registers -> output type -> shared memory -> one bulk copy per token
//
// A tile's weight rows are permuted so that its scales need no such copies: 128 consecutive words in shared memory are, to
// tcgen05.cp, lane i's words 4i .. 4i+3, the scales of MMA rows i, 32 + i, 64 + i and 96 + i.  MMA row 32 j + i therefore
// is weight row 4 i + j (the copy's box walks rows 0, 4, .., 124, 1, 5, ..), and so are the accumulator's lanes.
//
// Work split.  Tiles are numbered expert by expert.  Whole waves go out one tile per CTA; what is left over (everything, if
// there are fewer tiles than CTAs) is cut evenly along K.  A cut tile is finished by the CTA that arrives last, which
// adds the fp32 partial sums in K order: the result does not depend on the order of arrival.
//
// Every wait is bounded, as in the other pipeline kernels.
#include <algorithm>
#include <cstring>
#include <mutex>
#include "launchers.h"
#include "mx_format.cuh"
#include "sm100_ptx.cuh"
#include "tcgen05.cuh"

namespace tuna {

constexpr int kMxWarps = 8;
constexpr int kMxEpilogueWarp0 = 4;
constexpr int kMxMaxStages = 10;
constexpr int kMxScaleDepth = 3;       // stages of token scales in flight; fewer than there are stages
constexpr int kMxStageTokens = 32;     // tokens of an output staging buffer
constexpr int kMxTmemCols = 512;
constexpr uint32_t kMxWeightBytes = kBlockRows * kMxChunkBytes;
constexpr uint32_t kMxAtomBytes = 512;  // scales of 128 rows x 128 columns
constexpr int kMxSmemMax = 227 * 1024 - 2048;  // dynamic part: 1 KB alignment, 1 KB static

struct MxParams {
    const uint32_t *xs;   // words of the tokens' scales [words][tokens]
    const int *offsets;   // first token of each expert, and the end; nullptr: one matrix, all tokens
    void *o;
    float *partials;
    unsigned int *counters;
    DeviceStatus *status;
    int m, n, k;
    int experts;
    int tile_tok;   // N
    int chunks;     // ceil(k / 256)
    int words;      // ceil(k / 128)
    int row_tiles;  // ceil(m / 128)
    int last_steps; // MMAs of the last chunk: 64 columns each
    int stages;
    int nd;         // accumulator buffers
    int ahead;      // weights are taken from before the dependency wait
};

// How the launch's tiles are handed out: tiles 0 .. sk_tiles - 1 cut along K over workers 0 .. sk_workers - 1 in ranges of
// sk_q units (the first sk_r one more), the others whole.
struct MxSplit {
    int tiles, sk_tiles, sk_workers, sk_q, sk_r;
};

__device__ __forceinline__ MxSplit mx_split(int tiles, int chunks, int workers)
{
    MxSplit s = {tiles, 0, 0, 1, 0};
    const int rest = tiles % workers;
    if (rest == 0) return s;
    const int ctas = min(workers, rest * chunks / 2);  // two chunks at least
    if (ctas <= rest) return s;
    s.sk_tiles = rest;
    s.sk_workers = ctas;
    s.sk_q = rest * chunks / ctas;
    s.sk_r = rest * chunks % ctas;
    return s;
}

// The segments of a worker in order, and where each lies.
struct MxSegs {
    int u, u_end, dp, dp_step, tiles, chunks, row_tiles, tile_tok;
    const int *first_tile, *begin, *count;  // per expert (shared memory)
    int e;
    int tile, c0, c1;     // the segment
    int rt, tok0, valid;  // its rows' tile, its first token and how many there are
    __device__ void init(const MxParams &p, const MxSplit &s, int worker, int workers, const int *tables)
    {
        u = worker * s.sk_q + min(worker, s.sk_r);
        u_end = u + (worker < s.sk_workers ? s.sk_q + (worker < s.sk_r ? 1 : 0) : 0);
        if (s.sk_tiles == 0) u = u_end = 0;
        dp = s.sk_tiles + worker;
        dp_step = workers;
        tiles = s.tiles;
        chunks = p.chunks;
        row_tiles = p.row_tiles;
        tile_tok = p.tile_tok;
        begin = tables;
        count = tables + p.experts;
        first_tile = tables + 2 * p.experts;
        e = 0;
    }
    __device__ bool more() const { return u < u_end || dp < tiles; }
    __device__ bool next()
    {
        if (u < u_end) {
            tile = u / chunks;
            c0 = u - tile * chunks;
            c1 = min(chunks, c0 + (u_end - u));
            u += c1 - c0;
        } else if (dp < tiles) {
            tile = dp;
            c0 = 0;
            c1 = chunks;
            dp += dp_step;
        } else {
            return false;
        }
        while (tile >= first_tile[e + 1]) ++e;  // tiles come in increasing order, and the last expert's end is their number
        const int local = tile - first_tile[e], tok_tiles = div_up(count[e], tile_tok);
        rt = local / tok_tiles;
        const int tt = local - rt * tok_tiles;
        tok0 = begin[e] + tt * tile_tok;
        valid = min(tile_tok, count[e] - tt * tile_tok);
        return true;
    }
    __device__ int total_units() const { return (u_end - u) + (dp < tiles ? ((tiles - 1 - dp) / dp_step + 1) * chunks : 0); }
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, int c0, int c1, int c2, int c3, uint32_t bar)
{
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
        ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
        : "memory");
}

// Four bytes, or zeros where `have` is false.
__device__ __forceinline__ void cp_async_word(uint32_t dst, const uint32_t *src, bool have)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(have ? 4 : 0) : "memory");
}

// 32 rows of 16 bytes -> 4 columns of 32 lanes, the same in all four lane quarters.
__device__ __forceinline__ void tc_copy_scales(uint32_t taddr, uint64_t desc)
{
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// D[tmem] (+)= (A * scale A) (B * scale B), 64 columns of e2m1 with a scale per 32
__device__ __forceinline__ void tc_mma_mx(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate)
{
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

// Instruction descriptor, kind::mxf4: A and B e2m1 (1 at bits 7-9 and 10-11), both K-major, N >> 3 at bits 17-22, e8m0 scales
// (bit 23), M >> 7 at bits 27-28, which half of a scale word A and B use (0 or 2) at bits 29-30 and 4-5.
__host__ __device__ constexpr uint32_t mx_idesc(int cols, int half)
{
    return (1u << 7) | (1u << 10) | ((uint32_t)(cols >> 3) << 17) | (1u << 23) | (1u << 27) | ((uint32_t)(2 * half) << 29) | ((uint32_t)(2 * half) << 4);
}

template <typename T>
__device__ __forceinline__ T mx_convert(float v);
template <> __device__ __forceinline__ __half mx_convert<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 mx_convert<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ float mx_convert<float>(float v) { return v; }

__device__ __forceinline__ void mx_store_shared(uint32_t a, __half v) { asm volatile("st.shared.u16 [%0], %1;" ::"r"(a), "h"(__half_as_ushort(v)) : "memory"); }
__device__ __forceinline__ void mx_store_shared(uint32_t a, __nv_bfloat16 v) { asm volatile("st.shared.u16 [%0], %1;" ::"r"(a), "h"(__bfloat16_as_ushort(v)) : "memory"); }
__device__ __forceinline__ void mx_store_shared(uint32_t a, float v) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory"); }

__host__ __device__ constexpr uint32_t mx_scale_atoms(int tile_tok) { return (uint32_t)((tile_tok + 127) / 128); }
__host__ __device__ constexpr uint32_t mx_stage_bytes(int tile_tok)
{
    return kMxWeightBytes + (uint32_t)tile_tok * kMxChunkBytes + 2 * kMxAtomBytes + 2 * mx_scale_atoms(tile_tok) * kMxAtomBytes;
}
// Tensor-memory columns of a stage's scales: two atoms of four columns for the weights, as many per 128 tokens.
__host__ __device__ constexpr uint32_t mx_scale_cols(int tile_tok) { return 8 + 8 * mx_scale_atoms(tile_tok); }

template <typename OT>
__global__ void __launch_bounds__(32 * kMxWarps, 1)
mx_gemm_kernel(const __grid_constant__ MxParams p, const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_ws,
               const __grid_constant__ CUtensorMap tmap_x)
{
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[2 * kMxMaxStages + 4];
    __shared__ uint32_t s_tmem_base;
    __shared__ int s_abort, s_last;
    __shared__ MxSplit s_split;

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int N = p.tile_tok, S = p.stages;
    const uint32_t base = (smem_u32(smem) + 1023u) & ~1023u;
    const uint32_t stage_bytes = mx_stage_bytes(N);
    const uint32_t x_off = kMxWeightBytes, ws_off = x_off + (uint32_t)N * kMxChunkBytes, xs_off = ws_off + 2 * kMxAtomBytes;
    const uint32_t staging = base + (uint32_t)S * stage_bytes;
    constexpr uint32_t kTokBytes = kBlockRows * (uint32_t)sizeof(OT);
    constexpr uint32_t kStagingBytes = kMxStageTokens * kTokBytes;
    int *tables = reinterpret_cast<int *>(smem + (base - smem_u32(smem)) + (size_t)S * stage_bytes + 2 * kStagingBytes);

    const uint32_t full = smem_u32(&bars[0]), empty = full + 8 * kMxMaxStages, d_full = empty + 8 * kMxMaxStages, d_empty = d_full + 16;
    volatile int *abort_flag = &s_abort;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (warp == 1) {
        auto count = [](int i) { return i < kMxMaxStages ? 2 : i < 2 * kMxMaxStages + 2 ? 1 : 4; };  // full: the copies and the scales; d_empty: four warps
        for (int i = lane; i < 2 * kMxMaxStages + 4; i += 32) mbar_init(full + 8 * i, count(i));
        if (lane == 0) s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (elect_one_sync()) {
            prefetch_map(&tmap_w);
            prefetch_map(&tmap_ws);
            prefetch_map(&tmap_x);
        }
    }
    if (warp == 3) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem_base)), "r"(kMxTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    auto depend = [] { asm volatile("griddepcontrol.wait;" ::: "memory"); };
    if (warp == 0) {  // the experts' tiles: first token, tokens, tiles before
        if (p.offsets) depend();
        int before = 0;
        for (int e0 = 0; e0 < p.experts; e0 += 32) {
            const int e = e0 + lane;
            int begin = 0, cnt = 0;
            if (e < p.experts) {
                if (p.offsets) {  // whatever they are, inside the tokens
                    begin = min(max(__ldcg(p.offsets + e), 0), p.n);
                    cnt = max(min(max(__ldcg(p.offsets + e + 1), 0), p.n) - begin, 0);
                } else {
                    cnt = p.n;
                }
            }
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
        if (lane == 0) {
            tables[3 * p.experts] = before;
            s_split = mx_split(before, p.chunks, gridDim.x);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem_base;
    const uint32_t sf_col = (uint32_t)(p.nd * N), sf_cols = mx_scale_cols(N);
    MxSegs segs;
    segs.init(p, s_split, blockIdx.x, gridDim.x, tables);
    const int total = segs.total_units();

    if (warp == 0) {
        // ------------------------------------------------------------------ MMA issue
        constexpr uint64_t sw128 = ((uint64_t)((1024u >> 4) | (1u << 14) | (2u << 29))) << 32;  // 8-row groups 1024 bytes apart, version 1, 128-byte swizzle
        constexpr uint64_t plain = ((uint64_t)((128u >> 4) | (1u << 14))) << 32;                // 8-row groups of 16 bytes a row, 128 bytes apart, no swizzle
        Ring ru, rd;
        bool ok = true;
        while (ok && segs.next()) {
            const int cols = (segs.valid + 15) & ~15;
            ok = mbar_wait_warp(d_empty + 8 * rd.idx, rd.phase ^ 1, abort_flag, p.status, 203);
            const uint32_t d = tmem + (uint32_t)(rd.idx * N);
            for (int c = segs.c0; ok && c < segs.c1; ++c) {
                ok = mbar_wait_warp(full + 8 * ru.idx, ru.phase, abort_flag, p.status, 204);
                if (!ok) break;
                tc_fence_after();
                if (elect_one_sync()) {
                    const uint32_t at = base + (uint32_t)ru.idx * stage_bytes;
                    const uint32_t sfa = tmem + sf_col + (uint32_t)ru.idx * sf_cols, sfb = sfa + 8, atoms = mx_scale_atoms(N);
                    auto desc = [](uint64_t kind, uint32_t addr) { return kind | (uint64_t)((addr & 0x3FFFFu) >> 4); };
                    for (uint32_t h = 0; h < 2; ++h) {
                        tc_copy_scales(sfa + 4 * h, desc(plain, at + ws_off + h * kMxAtomBytes));
                        for (uint32_t a = 0; a < atoms; ++a)
                            tc_copy_scales(sfb + 4 * (h * atoms + a), desc(plain, at + xs_off + (h * atoms + a) * kMxAtomBytes));
                    }
                    const int steps = c + 1 == p.chunks ? p.last_steps : 4;
                    for (int kk = 0; kk < steps; ++kk)
                        tc_mma_mx(d, desc(sw128, at + 32 * kk), desc(sw128, at + x_off + 32 * kk), mx_idesc(cols, kk & 1), sfa + 4 * (kk >> 1),
                                  sfb + 4 * atoms * (kk >> 1), c == segs.c0 && kk == 0 ? 0u : 1u);
                    tc_commit(empty + 8 * ru.idx);
                    if (c + 1 == segs.c1) tc_commit(d_full + 8 * rd.idx);
                }
                __syncwarp();
                ru.advance(S);
            }
            rd.advance(p.nd);
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------------ weights and tokens' codes
        Ring ru;
        bool ok = true;
        depend();
        while (ok && segs.next()) {
            for (int c = segs.c0; c < segs.c1; ++c, ru.advance(S)) {
                ok = mbar_wait_warp(empty + 8 * ru.idx, ru.phase ^ 1, abort_flag, p.status, 200);
                if (!ok) break;
                if (elect_one_sync()) {
                    const uint32_t at = base + (uint32_t)ru.idx * stage_bytes, bar = full + 8 * ru.idx;
                    mbar_expect_tx(bar, kMxWeightBytes + (uint32_t)N * kMxChunkBytes + 2 * kMxAtomBytes);
                    tma_load_4d(at, &tmap_w, 0, segs.rt * (kBlockRows / 4), 0, segs.e * p.chunks + c, bar);
                    tma_load_2d(at + ws_off, &tmap_ws, segs.rt * kBlockRows, segs.e * p.words + 2 * c, bar);
                    tma_load_3d(at + x_off, &tmap_x, 0, segs.tok0, c, bar);
                }
                __syncwarp();
            }
        }
        // The MMAs' commits have arrived at every stage in use before the CTA leaves.
        if (total < S) ru = Ring();
        for (int i = min(S, total); ok && i > 0; --i, ru.advance(S)) ok = mbar_wait_warp(empty + 8 * ru.idx, total < S ? 0u : ru.phase ^ 1, abort_flag, p.status, 210);
    } else if (warp == 2) {
        // ------------------------------------------------------------------ tokens' scales
        Ring ru, ra;
        int flying = 0;
        bool ok = true;
        auto arrive = [&] {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // what cp.async wrote is read by tcgen05.cp
            __syncwarp();
            if (lane == 0) mbar_arrive(full + 8 * ra.idx);
            ra.advance(S);
        };
        depend();
        while (ok && segs.next()) {
            const int rows = min(N, p.n - segs.tok0);
            for (int c = segs.c0; c < segs.c1; ++c, ru.advance(S)) {
                ok = mbar_wait_warp(empty + 8 * ru.idx, ru.phase ^ 1, abort_flag, p.status, 201);
                if (!ok) break;
                const uint32_t at = base + (uint32_t)ru.idx * stage_bytes + xs_off, half = mx_scale_atoms(N) * kMxAtomBytes;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int word = min(2 * c + h, p.words - 1);  // behind the last word of an odd number of them nothing is multiplied
                    const uint32_t *src = p.xs + (size_t)word * p.n + segs.tok0;
                    for (int t = lane; t < N; t += 32)
                        cp_async_word(at + h * half + (uint32_t)(t >> 7) * kMxAtomBytes + (uint32_t)((t & 31) * 16 + ((t >> 5) & 3) * 4), src + min(t, rows - 1), t < rows);
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
                if (++flying > kMxScaleDepth) {
                    asm volatile("cp.async.wait_group %0;" ::"n"(kMxScaleDepth) : "memory");
                    arrive();
                    --flying;
                }
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        for (; flying > 0; --flying) arrive();
    } else if (warp >= kMxEpilogueWarp0) {
        // ------------------------------------------------------------------ epilogue
        const int quarter = warp & 3, thread = threadIdx.x - 32 * kMxEpilogueWarp0;
        const int row = 4 * lane + quarter;  // of the tile: see the head of the file
        const uint32_t tmem_q = tmem + ((uint32_t)(32 * quarter) << 16);
        const size_t slot_floats = (size_t)kBlockRows * N;
        OT *o = static_cast<OT *>(p.o);
        Ring rd;
        uint32_t buf = 0;
        depend();
        // Rows of `valid` tokens, 16 at a time from `get`, through the staging buffers to memory.
        auto store_tile = [&](auto get) {
            const uint32_t bytes = (uint32_t)min(kBlockRows, p.m - segs.rt * kBlockRows) * (uint32_t)sizeof(OT);
            for (int t0 = 0; t0 < segs.valid; t0 += kMxStageTokens, buf ^= 1) {
                const uint32_t to = staging + buf * kStagingBytes;
                if (lane < 8) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");  // the buffer's previous tokens have left it
                asm volatile("bar.sync 1, 128;" ::: "memory");
#pragma unroll
                for (int h = 0; h < kMxStageTokens; h += 16) {
                    if (t0 + h >= segs.valid) break;
                    float v[16];
                    get(t0 + h, v);
#pragma unroll
                    for (int i = 0; i < 16; ++i) mx_store_shared(to + (uint32_t)(h + i) * kTokBytes + (uint32_t)row * (uint32_t)sizeof(OT), mx_convert<OT>(v[i]));
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                asm volatile("bar.sync 1, 128;" ::: "memory");
                if (lane < 8) {
                    const int t = 8 * quarter + lane;
                    if (t0 + t < segs.valid)
                        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(o + (size_t)(segs.tok0 + t0 + t) * p.m + segs.rt * kBlockRows),
                                     "r"(to + (uint32_t)t * kTokBytes), "r"(bytes)
                                     : "memory");
                    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                }
            }
        };
        while (segs.next()) {
            const bool ok = mbar_wait_warp(d_full + 8 * rd.idx, rd.phase, abort_flag, p.status, 206);
            if (bar_any(1, 128, !ok)) break;  // the four warps go on together or not at all
            tc_fence_after();
            const uint32_t d = tmem_q + (uint32_t)(rd.idx * N);
            if (segs.c0 == 0 && segs.c1 == p.chunks) {
                store_tile([&](int t, float (&v)[16]) { tc_ld_x16(d + t, v); });
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(d_empty + 8 * rd.idx);
            } else {
                // [4-token group][128 lanes] float4: a warp store is 512 contiguous bytes
                float4 *dst = reinterpret_cast<float4 *>(p.partials + (size_t)(2 * blockIdx.x + (segs.c0 == 0 ? 1 : 0)) * slot_floats) + 32 * quarter + lane;
                for (int t0 = 0; t0 < segs.valid; t0 += 16) {
                    float v[16];
                    tc_ld_x16(d + t0, v);
#pragma unroll
                    for (int i = 0; i < 4; ++i) dst[(size_t)(t0 / 4 + i) * kBlockRows] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(d_empty + 8 * rd.idx);
                auto worker_of = [&](int unit) {
                    const int big = s_split.sk_r * (s_split.sk_q + 1);
                    return unit < big ? unit / (s_split.sk_q + 1) : s_split.sk_r + (unit - big) / s_split.sk_q;
                };
                const int first = worker_of(segs.tile * p.chunks), nseg = worker_of((segs.tile + 1) * p.chunks - 1) - first + 1;
                asm volatile("bar.sync 1, 128;" ::: "memory");
                if (thread == 0) {
                    unsigned int old;
                    // releases the four warps' partials (ordered before it by the barrier) and acquires the others'
                    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(old) : "l"(p.counters + segs.tile) : "memory");
                    s_last = old == (unsigned)nseg - 1;
                    if (s_last) p.counters[segs.tile] = 0;  // left clean for the next call
                }
                asm volatile("bar.sync 1, 128;" ::: "memory");
                if (s_last) {
                    store_tile([&](int t, float (&v)[16]) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] = 0.f;
                        for (int s = 0; s < nseg; ++s) {
                            const float4 *src = reinterpret_cast<const float4 *>(p.partials + (size_t)(2 * (first + s) + (s == 0 ? 1 : 0)) * slot_floats) + (size_t)(t / 4) * kBlockRows + 32 * quarter + lane;
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float4 w = __ldcg(src + i * kBlockRows);
                                v[4 * i] += w.x; v[4 * i + 1] += w.y; v[4 * i + 2] += w.z; v[4 * i + 3] += w.w;
                            }
                        }
                    });
                }
                asm volatile("bar.sync 1, 128;" ::: "memory");  // s_last has been read
            }
            rd.advance(p.nd);
        }
        if (lane < 8) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }

    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 3) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kMxTmemCols) : "memory");
    }
}

// ------------------------------------------------------------------ host side

struct MxPlan {
    int tile_tok, stages, nd;
    size_t smem;
};

static MxPlan mx_plan(int n, int experts, int o_type)
{
    MxPlan l;
    const int each = div_up(n, experts);
    l.tile_tok = each <= 16 ? 16 : each <= 32 ? 32 : each <= 64 ? 64 : 128;
    const size_t tail = 2 * (size_t)kMxStageTokens * kBlockRows * (o_type == TUNA_FP32 ? 4 : 2) + (3 * (size_t)experts + 1) * 4;
    const size_t room = kMxSmemMax - tail;
    l.stages = (int)std::min<size_t>(kMxMaxStages, room / mx_stage_bytes(l.tile_tok));
    l.nd = 2;
    l.smem = (size_t)l.stages * mx_stage_bytes(l.tile_tok) + tail + 1024;
    return l;
}

size_t mx_gemm_workspace_bytes(int m, int n, int k, int experts, int sm_count)
{
    (void)m; (void)k;
    const MxPlan l = mx_plan(n, experts, TUNA_FP32);
    return kMxCounterBytes + 2 * (size_t)sm_count * kBlockRows * l.tile_tok * 4;
}

template <typename OT>
static int launch_mx(const MxParams &p, const CUtensorMap &mw, const CUtensorMap &ms, const CUtensorMap &mx, int ctas, size_t smem, cudaStream_t stream)
{
    static bool attr_set[64] = {false};
    static std::mutex mu;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return TUNA_ERR_NO_DEVICE;
    {
        std::lock_guard<std::mutex> lock(mu);
        if (!attr_set[dev]) {
            if (cudaFuncSetAttribute(mx_gemm_kernel<OT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMxSmemMax + 1024) != cudaSuccess) return TUNA_ERR_NO_DEVICE;
            attr_set[dev] = true;
        }
    }
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)ctas);
    lc.blockDim = dim3(32 * kMxWarps);
    lc.dynamicSmemBytes = smem;
    lc.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = attr;
    lc.numAttrs = 1;
    return cudaLaunchKernelEx(&lc, mx_gemm_kernel<OT>, p, mw, ms, mx) == cudaSuccess ? TUNA_OK : TUNA_ERR_LAUNCH;
}

int launch_mx_gemm(const MxGemmArgs &a)
{
    const MxPlan l = mx_plan(a.n, a.experts, a.o_type);
    MxParams p;
    std::memset(&p, 0, sizeof(p));
    p.xs = (const uint32_t *)a.xs; p.offsets = (const int *)a.offsets; p.o = a.o;
    p.m = a.m; p.n = a.n; p.k = a.k; p.experts = a.experts;
    p.tile_tok = l.tile_tok;
    p.chunks = div_up(a.k, kMxChunk);
    p.words = div_up(a.k, kMxScaleCols);
    p.row_tiles = div_up(a.m, kBlockRows);
    p.last_steps = div_up(a.k - (p.chunks - 1) * kMxChunk, 64);
    p.stages = l.stages;
    p.nd = l.nd;
    p.counters = (unsigned int *)a.workspace;
    p.partials = (float *)((uint8_t *)a.workspace + kMxCounterBytes);
    p.status = device_status_word();
    if (!p.status) return TUNA_ERR_NO_DEVICE;
    const long long tiles = ((long long)div_up(a.n, l.tile_tok) + a.experts - 1) * p.row_tiles;  // at most
    if (tiles >= 1ll << 30 || (tiles / a.sm_count + 2) * p.chunks >= 1ll << 30 || (long long)a.sm_count * p.chunks >= 1ll << 30 || (long long)a.experts * p.words >= 1ll << 30) return TUNA_ERR_TOO_LARGE;

    CUtensorMap mw, ms, mx;
    {
        const uint64_t dims[4] = {kMxChunkBytes, (uint64_t)a.m / 4, 4, (uint64_t)a.experts * p.chunks};
        const uint64_t strides[3] = {4 * kMxChunkBytes, kMxChunkBytes, (uint64_t)a.m * kMxChunkBytes};
        const uint32_t box[4] = {kMxChunkBytes, kBlockRows / 4, 4, 1};
        if (!make_tensor_map_nd(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.q, 4, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return TUNA_ERR_NO_DEVICE;
    }
    if (!make_tensor_map_2d(&ms, CU_TENSOR_MAP_DATA_TYPE_UINT32, a.s, (uint64_t)a.m, (uint64_t)a.experts * p.words, (uint64_t)a.m * 4, kBlockRows, 2, CU_TENSOR_MAP_SWIZZLE_NONE))
        return TUNA_ERR_NO_DEVICE;
    if (!make_tensor_map_3d(&mx, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.x, kMxChunkBytes, (uint64_t)a.n, (uint64_t)p.chunks, kMxChunkBytes, (uint64_t)a.n * kMxChunkBytes,
                            kMxChunkBytes, (uint32_t)l.tile_tok, 1, CU_TENSOR_MAP_SWIZZLE_128B))
        return TUNA_ERR_NO_DEVICE;
    const int ctas = a.sm_count;
    switch (a.o_type) {
        case TUNA_FP16: return launch_mx<__half>(p, mw, ms, mx, ctas, l.smem, a.stream);
        case TUNA_BF16: return launch_mx<__nv_bfloat16>(p, mw, ms, mx, ctas, l.smem, a.stream);
        default: return launch_mx<float>(p, mw, ms, mx, ctas, l.smem, a.stream);
    }
}

}  // namespace tuna
