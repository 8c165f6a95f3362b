// Products of 8-bit block-scaled matrices (format: fp8_format.cuh) on the 5th-generation tensor cores of sm_100a, one kernel in four forms:
//
//   product  o[t][r]  = sum over c of x[t][c] w[r][c]                     x by row, w square
//   gated    h[t][i]  = act(g) u, g and u the same sums for rows i and f + i of w; z = [g | u] on wish
//   dx       dx[t][c] = sum over r of dy[t][r] w[r][c]                    dy by row, w square: the same codes and scales, read across
//   dw       dw[r][c] = sum over t of dy[t][r] x[t][c]                    both by column: the blocks lie along the tokens
//
// (x, w and so on are the blocks' codes times their scales.)  The tensor cores apply the scales themselves (tcgen05.mma kind::mxf8f6f4, scale_vec::1X), so per
// 128 of what is summed over a tile's codes are copied to shared memory as they lie in memory and four MMAs of 32 add to fp32
// accumulators; the scales of four such blocks are one 32-bit word a row, written to tensor memory once for sixteen MMAs.
//
// What a lane of tensor memory has is what lies side by side in the output: operand A are its columns (weights' rows, or their columns in dx, x's in
// dw), B its rows.  Where an operand's summed dimension is not the one that lies side by side in memory (w in dx, both in dw) it is
// taken "MN-major": 128 bytes of a staged row are 128 rows of the operand, and nothing is ever transposed in memory.
//
// gated: a tile's rows are, by a four-dimensional tensor map, eight of the gate and the eight of the other projection that belong to them in turn.  So
// the fragments that a thread takes out of tensor memory (lanes i and i + 8) hold both factors, and the product is made in its registers.
//
// Persistent CTAs (12 warps), or pairs of CTAs (cta_group::2, 16 warps: 256 rows of A, every CTA stages its own 128 and half of B):
//   warp 0     MMA issue (one elected lane; in a pair the first CTA's)
//   warp 1, 2  TMA producers of A and of B
//   warp 3     tensor-memory allocation; in a pair, tells the first CTA that a stage has landed
//   warps 4-7  epilogue: tensor memory -> registers -> output type -> shared memory, where rows become contiguous -> memory; in a pair 12-15 too
//   warps 8-11 scales, one warp per lane quarter: global memory -> registers, two groups of four units ahead -> tensor memory, the word of row r at lane r % 32,
//              column r / 32, in every quarter
// RESIDENT: a few tokens in 16 bits are quantized by the CTA itself before its first MMA, all of K, and stay in shared memory.
//
// Work split.  No sum is cut.  Up to 16 tokens weights of few rows are cut into row tiles of equal height, a whole number of them for every CTA: the MMAs compute 128
// rows whatever the height, which costs nothing where the weights' bytes are the bound.  Where a tile has at most 64 (32) of the
// 128 rows, two (four) blocks of K lie side by side in it ("folded"): the MMA's rows are those of the tile for each block in turn, its columns the tokens
// for each block, and the epilogue adds up what belongs together.  Everything else goes in tiles of 256 rows on pairs, of as many columns as an estimate says.
//
// What bounds it (graph replay, weights of 0.4 GB in turn; 6.55 TB/s is the measured copy rate, 3.39 PFLOP/s twice the measured bf16 burst, 2.79 twice the sustained rate):
//   weights' bytes    57344x8192 at 1 token 74 us = 6.3 TB/s, 28672x4096 21.5 = 5.5 (17.9 of bytes and what is left of a launch's chain of 4 us)
//   a launch's chain  4096x4096 at 1 token 6.1 us: end of the kernel before, the tokens' copy and scales, the last stages, epilogue
//   steps in a row    4096x14336 at 43 tokens 22 us: 16 tiles on 74 pairs, each 112 units of 0.17 us one after another
//   tensor pipe       28672x4096 at 2048 tokens 175 us = 2.75 PFLOP/s (gated 170 to 185), active for 77 to 80 % of the time, at the power cap; dx of the same the same
//   stores            dw of the same, 235 MB of results in bf16, 205 us without them and 235 with them
// Sums of parts.  The accumulators are fp32, and what an addition has below their last bit is cut off, so a long sum in one of them ends up nearer to zero: 2.5e-6 off for 28672 columns, 2.1e-7 for
// 4096 (2-norm against 64 bits, 64 tokens, random numbers; sums in fp32 that round are 1e-7 and 0.6e-7 off).  Where that can be seen - results in 32 bits, and z, which in 16 bits decides on which side
// of a border a gradient's code falls - the tensor cores add up at most 1024 columns (2048 in tiles of more than 128 columns, whose epilogue two parts have to cover: gated 4096x2048 at 2048 tokens with z
// 47 us in parts of 1536, 41 in parts of 2048), and the epilogue the parts, to nearest, in its registers: 1.2e-7 and 0.7e-7.  It costs what reading an accumulator does: 28672x4096 at 43
// tokens in 32 bits 23.1 -> 23.4 us, 4096x14336 at 43 (14 parts) 22.6 -> 23.8, 6144x4096 with gradients in 32 bits at 4096 204 -> 208.  Results in 16 bits are a hundredth of a rounding off without.
// Every wait is bounded, as in the other pipeline kernels.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <mutex>
#include "launchers.h"
#include "fp8_format.cuh"
#include "fp8_scales.h"
#include "sm100_ptx.cuh"
#include "tcgen05.cuh"

namespace tuna {

enum Fp8Form { kFp8Product, kFp8GatedProduct, kFp8Dx, kFp8Dw };

// Warps of a CTA: pairs have eight for the epilogue, two groups of four that take turns on 32 columns.  With four, gated tiles waited for them (14336x4096 at 2048 tokens 206 -> 185
// us, with z 233 -> 200).
__host__ __device__ constexpr int fp8_warps(int cg) { return cg == 1 ? 12 : 16; }
constexpr int kFp8EpilogueWarp0 = 4;
constexpr int kFp8ScaleWarp0 = 8;
// Registers of a thread where the parts of a wide tile's sums are added up: the epilogue's hold the sums, 128 of theirs, and the four groups of four warps share what the CTA was launched with.
constexpr int kFp8LaunchRegs = 128, kFp8IssueRegs = 40, kFp8ScaleRegs = 72, kFp8EpilogueRegs = 200;
static_assert(kFp8IssueRegs + kFp8ScaleRegs + 2 * kFp8EpilogueRegs <= 4 * kFp8LaunchRegs, "a group would wait for registers that nobody gives back");
constexpr int kFp8MaxStages = 12;
constexpr int kFp8Deep = 2;               // units of a stage: what a wait, a commit and the turn of the issuing warp cost is paid once for eight MMAs (one unit: 4096x14336 at 43 tokens 28 us, so 22)
constexpr int kFp8SingleCols = 16;        // tokens up to which single CTAs may take the tiles
constexpr int kFp8StageCols = 32;         // columns of a group's output staging buffer
constexpr int kFp8NarrowCols = 128;      // tiles whose sums every warp has registers for
constexpr int kFp8WideSlices = 4, kFp8NarrowSlices = 2;  // staging buffers of columns that an epilogue group has of a tile at most: of 240 columns, and of 128
constexpr int kFp8AheadTokens = 64;       // up to here weights count as constants and are copied ahead of the dependency wait, as in mx_gemm_sm100a.cu
constexpr int kFp8ResidentLoads = 4;      // loads in flight of a quantizing warp
constexpr int kFp8PartSteps = 4, kFp8WidePartSteps = 8;  // stages of a part of a sum at most, and of wide tiles: 1024 columns (folded: for each block of a unit), 2048
constexpr int kFp8SfCols = 16;            // tensor-memory columns of a group's scales: A's words at 0 to 3, B's at 8 to 15
constexpr uint32_t kFp8SumBytes = kFp8SingleCols * kBlockRows * 4;  // where the parts of a folded tile, or a gated one's projections, meet
constexpr int kFp8SmemMax = 225 * 1024;   // dynamic shared memory of a CTA alone on its SM (1 KB is the kernel's static part, 1 KB the system's)
constexpr int kFp8SmemHalf = 111 * 1024;  // of one that leaves room for another

struct Fp8Params {
    const uint8_t *as;  // scales of A
    const uint8_t *bs;  // of B
    void *o, *z;
    DeviceStatus *status;
    int rows;        // of A; gated: 2f
    int cols;        // of B
    int red;         // what is summed over
    int blocks;      // ceil(red / 128)
    int units;       // of a tile: ceil(blocks / fold), four MMAs each
    int fold_log;    // log2(fold): blocks side by side in a unit
    int steps;       // stages of a tile: ceil(units / kFp8Deep)
    int part_steps;  // stages of a part of the sum: the tensor cores add these up, the epilogue the parts
    int parts;       // ceil(steps / part_steps)
    int tile_cols;   // N
    int width;       // columns of a tile, all but the last
    int row_tiles, col_tiles;
    int rows_inner;  // tiles follow one another along the rows
    int a_bytes;     // of a unit of A
    int b_rows;      // rows of B in a unit of a CTA (MN-major: 128)
    int stages;
    int d_cols;      // tensor-memory columns of each of the two accumulators: columns of a tile times fold
    int ahead;       // A is there before the dependency wait
    int beside;      // dx and dw of one call: dw is launched right behind dx
    int x_bf16;      // RESIDENT: type of the tokens
    const void *x;   // RESIDENT: the tokens [cols][red]
    int stagger;     // row tiles start their sums at different groups
    int gelu;
    int z_offset;    // gated: where z is staged
};

struct Fp8Tiles {
    int next_tile, step, rt, col0, valid;
    __device__ void init(int worker, int workers) { next_tile = worker; step = workers; }
    __device__ bool next(const Fp8Params &p)
    {
        if (next_tile >= p.row_tiles * p.col_tiles) return false;
        const int inner = p.rows_inner ? p.row_tiles : p.col_tiles, outer_at = next_tile / inner, inner_at = next_tile - outer_at * inner;
        rt = p.rows_inner ? inner_at : outer_at;
        col0 = (p.rows_inner ? outer_at : inner_at) * p.width;
        valid = min(p.width, p.cols - col0);
        next_tile += step;
        return true;
    }
    // Units come in groups of four (one word of scales); a tile starts with this one and goes round.
    __device__ int first_group(const Fp8Params &p, int groups) const { return p.stagger ? rt % groups : 0; }
    __device__ int total(const Fp8Params &p) const { const int n = p.row_tiles * p.col_tiles; return next_tile < n ? (n - 1 - next_tile) / step + 1 : 0; }
};

// The stages of a tile in order: `c` is a stage's first unit, and it has those before `end`.
struct Fp8Stages {
    int c, units;
    __device__ Fp8Stages(const Fp8Params &p, int first_group) : c(4 * first_group), units(p.units) {}
    __device__ int end() const { return min(c + kFp8Deep, units); }
    __device__ void advance()
    {
        c += kFp8Deep;
        if (c >= units) c = 0;
    }
};

// D[tmem] (+)= (A * scale A) (B * scale B), 32 columns of e4m3 with one scale
template <int CG>
__device__ __forceinline__ void tc_mma_fp8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate)
{
    if (CG == 1)
        asm volatile(
            "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
            " tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}"
            ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
            " tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}"
            ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
}

// Instruction descriptor, kind::mxf8f6f4: A and B e4m3 (0 at bits 7-9 and 10-12), A and B MN-major at bits 15 and 16, N >> 3 at bits 17-22, e8m0 scales
// (bit 23), M >> 7 at bits 27-28, which byte of a scale word A and B use at bits 29-30 and 4-5.
template <int CG>
__host__ __device__ constexpr uint32_t fp8_idesc(int cols, bool a_mn, bool b_mn)
{
    return ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(cols >> 3) << 17) | (1u << 23) | ((uint32_t)CG << 27);
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, int c0, int c1, int c2, int c3, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst), "l"(map), "r"(c0), "r"(c1),
                 "r"(c2), "r"(c3), "r"(bar)
                 : "memory");
}

// First row of row block b (a CTA's share of a tile).  Single CTAs: blocks of equal height, a multiple of four rows.  Gated: twice the first feature.
template <int CG>
__device__ __forceinline__ int fp8_row(const Fp8Params &p, int b) { return CG == 1 ? 4 * (int)((long long)b * (p.rows / 4) / p.row_tiles) : b * kBlockRows; }

// Quantizes the tokens' numbers, all of K: warp `w` of `warps` takes every warps-th (two blocks, token).  Codes by 16 bytes, [block][piece of 16 columns][token]: the MMAs
// read eight tokens from there, of which those behind the last are the next pieces' and give columns that nobody reads, so that a token takes no more room than its
// codes.  Scale bytes in words [group of four units][64 columns: token of a block of the unit].
template <typename T>
__device__ __forceinline__ void fp8_quantize_resident(const Fp8Params &p, int w, int warps, int lane, uint32_t codes_at, uint32_t words_at)
{
    const int items = ((p.units << p.fold_log) + 1) / 2 * p.cols, limit = p.units << p.fold_log;  // blocks behind the last one are zeros
    for (int i0 = w; i0 < items; i0 += kFp8ResidentLoads * warps) {
        Mx8<T> v[kFp8ResidentLoads];
#pragma unroll
        for (int r = 0; r < kFp8ResidentLoads; ++r) {
            const int i = i0 + r * warps, c = i / p.cols, t = i - c * p.cols, col = c * 256 + lane * 8;
            if (i < items && col < p.red) v[r].load(static_cast<const T *>(p.x) + (size_t)t * p.red + col);
            else v[r].zero();
        }
#pragma unroll
        for (int r = 0; r < kFp8ResidentLoads; ++r) {
            const int i = i0 + r * warps, c = i / p.cols, t = i - c * p.cols, b = 2 * c + (lane >> 4);
            if (i >= items) break;
            uint32_t m = v[r].largest();
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 4));
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 8));
            const uint32_t e = fp8_scale(m);
            const float inverse = fp8_inverse(e);
            float f[8];
            v[r].values(f);
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] *= inverse;
            uint32_t lo = fp8_encode4(f[0], f[1], f[2], f[3]), hi = fp8_encode4(f[4], f[5], f[6], f[7]);
            if (e == 255u) lo = hi = 0;
            if (b >= limit) continue;
            asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(codes_at + ((uint32_t)(8 * b + ((lane >> 1) & 7)) * (uint32_t)p.cols + (uint32_t)t) * 16u + ((uint32_t)lane & 1u) * 8u),
                         "r"(lo), "r"(hi)
                         : "memory");
            const int unit = b >> p.fold_log, at = (b - (unit << p.fold_log)) * p.b_rows + t;
            if ((lane & 15) == 0) asm volatile("st.shared.u8 [%0], %1;" ::"r"(words_at + (uint32_t)(unit >> 2) * 256u + (uint32_t)at * 4u + ((uint32_t)unit & 3u)), "r"(e) : "memory");
        }
    }
}

// activation(g) u of two numbers of the output's type
template <typename OT>
__device__ __forceinline__ float2 fp8_activation(float g0, float u0, float g1, float u1, int gelu)
{
    constexpr bool kExact = sizeof(OT) == 4;
    const float2 s = (gelu ? fp8_gate<true, kExact>(g0, g1) : fp8_gate<false, kExact>(g0, g1)).both();
    return make_float2(g0 * s.x * u0, g1 * s.y * u1);
}

// CG: CTAs of a worker (1 or 2).  SLICES: 0 where sums have one part; otherwise the slices of a tile's columns whose parts an epilogue group adds up.  Single CTAs leave room for a second one on the SM: that of the next launch, which copies its first weights meanwhile.
template <int CG, int FORM, bool RESIDENT, int SLICES, typename OT>
__device__ __forceinline__ void fp8_gemm(const Fp8Params &p, const CUtensorMap &tmap_a, const CUtensorMap &tmap_a2, const CUtensorMap &tmap_b, int worker, int workers)
{
    extern __shared__ __align__(1024) uint8_t smem[];
    // landed, full, empty: of the stages; d_full, d_empty, sf_full, sf_empty: two each
    __shared__ __align__(8) uint64_t bars[3 * kFp8MaxStages + 8];
    __shared__ uint32_t s_tmem_base;
    __shared__ int s_abort;

    constexpr bool kParts = SLICES > 0, kShares = SLICES > kFp8NarrowSlices;
    constexpr bool kGated = FORM == kFp8GatedProduct, kAcrossA = FORM >= kFp8Dx, kAcrossB = FORM == kFp8Dw;
    constexpr uint32_t kTmemCols = CG == 1 ? 256 : 512, kSfCol = kTmemCols - 2 * kFp8SfCols;  // two accumulators below
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int rank = CG == 1 ? 0 : (int)cluster_ctarank();
    const int S = p.stages;
    // [stages of A][of B][words of the resident tokens' scales][staging buffer]; the MMAs read 128 rows of A, in low tiles past their stage's end.
    // RESIDENT: of B, all of a tile's stages.
    const int b_units = RESIDENT ? p.units : S * kFp8Deep, groups = (p.units + 3) >> 2;
    const uint32_t base = smem_u32(smem), a_bytes = (uint32_t)p.a_bytes, b_bytes = (uint32_t)((RESIDENT ? p.cols : p.b_rows) << p.fold_log) * 128u;  // of a unit
    const uint32_t b_ring = base + (uint32_t)(S * kFp8Deep) * a_bytes, words_at = b_ring + (uint32_t)b_units * b_bytes, staging = words_at + (RESIDENT ? 256u * (uint32_t)groups : 0u);

    const uint32_t landed = smem_u32(&bars[0]), full = CG == 1 ? landed : landed + 8 * kFp8MaxStages, empty = landed + 16 * kFp8MaxStages;
    const uint32_t d_full = empty + 8 * kFp8MaxStages, d_empty = d_full + 16, sf_full = d_empty + 16, sf_empty = sf_full + 16;
    volatile int *abort_flag = &s_abort;

    if (FORM != kFp8Dx || !p.beside) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (warp == 1) {
        auto count = [&](int i) {
            if (i < kFp8MaxStages) return RESIDENT ? 1 : 2;       // landed: the producers
            if (i < 2 * kFp8MaxStages) return 2;                  // full: both CTAs of the pair
            if (i < 3 * kFp8MaxStages + 2) return 1;              // empty, d_full: a commit
            if (i < 3 * kFp8MaxStages + 4) return CG == 1 ? 4 : 16;  // d_empty: the epilogue warps of each CTA
            if (i < 3 * kFp8MaxStages + 6) return 4 * CG;         // sf_full: the scale warps of each CTA
            return 1;                                             // sf_empty: a commit
        };
        for (int i = lane; i < 3 * kFp8MaxStages + 8; i += 32) mbar_init(landed + 8 * i, count(i));
        if (lane == 0) s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (elect_one_sync()) {
            prefetch_map(&tmap_a);
            if (!RESIDENT) prefetch_map(&tmap_b);
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
    // dw beside dx started when the kernels before dx were done (below), and reads nothing of dx's.  It waits for dx only in the end, for those who wait for it.
    auto depend = [&] {
        if (FORM != kFp8Dw || !p.beside) asm volatile("griddepcontrol.wait;" ::: "memory");
    };
    tc_fence_before();
    __syncthreads();
    if (CG == 2) cluster_sync_all();  // the other CTA's barriers are there
    tc_fence_after();
    if (FORM == kFp8Dx && p.beside) {  // what dw reads is there as well
        depend();
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    }
    const uint32_t tmem = s_tmem_base;
    const int fold = 1 << p.fold_log, part = kBlockRows >> p.fold_log;  // rows of a part
    Fp8Tiles tile;
    tile.init(worker, workers);
    const int tiles = tile.total(p), total = tiles * p.steps;
    auto mma_cols = [&] {  // that the tile's MMAs cover; a half's first column is a multiple of 16 where it is a coordinate of bytes
        constexpr int kUnit = kAcrossB ? 32 : 8 * CG;
        return (tile.valid + kUnit - 1) & -kUnit;
    };

    if (RESIDENT && warp != 1) {  // the weights are on their way meanwhile
        depend();
        const int w = warp == 0 ? 0 : warp - 1;
        if (p.x_bf16) fp8_quantize_resident<__nv_bfloat16>(p, w, fp8_warps(CG) - 1, lane, b_ring, words_at);
        else fp8_quantize_resident<__half>(p, w, fp8_warps(CG) - 1, lane, b_ring, words_at);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the MMAs read the codes
        asm volatile("bar.sync 2, %0;" ::"n"(32 * (fp8_warps(CG) - 1)) : "memory");
    }
    // Whoever makes a bounded wait that ends only after the kernels before this one waits for those first.
    auto issue = [&] {
        if (CG == 1 || rank == 0) {
            depend();
            Ring ru, rd, rs;
            bool ok = true;
            // -------------------------------------------------------------- MMA issue
            // Rows, or along the sum for what is read across, by eights 1024 bytes apart, version 1, 128-byte swizzle.  Read across, an MMA's 32 are 32
            // staged rows of 128 bytes, otherwise 32 of a row's 128 bytes.
            constexpr uint64_t sw128 = ((uint64_t)((1024u >> 4) | (1u << 14) | (2u << 29))) << 32;
            constexpr uint64_t kStepA = (kAcrossA ? 32 * 128 : 32) >> 4;
            // Resident tokens: not swizzled, pieces of 16 columns 16 bytes a token apart, the eight rows of the next block a block's bytes.
            const uint64_t kStepB = RESIDENT ? 2 * (uint64_t)p.cols : (kAcrossB ? 32 * 128 : 32) >> 4;
            const uint64_t b_form = RESIDENT ? ((uint64_t)p.cols << 16) | ((uint64_t)(8u * (uint32_t)p.cols | (1u << 14)) << 32) : sw128;
            while (ok && tile.next(p)) {
                const uint32_t idesc = fp8_idesc<CG>(p.fold_log ? p.d_cols : mma_cols(), kAcrossA, kAcrossB);
                uint32_t d = 0;
                auto next_accumulator = [&] {
                    ok = mbar_wait_warp<!kShares>(d_empty + 8 * rd.idx, rd.phase ^ 1, abort_flag, p.status, 303);
                    d = tmem + (uint32_t)(rd.idx * p.d_cols);
                };
                if (!kParts) next_accumulator();
                Fp8Stages st(p, tile.first_group(p, groups));
                for (int i = 0, of_part = 0; ok && i < p.steps; ++i, st.advance()) {
                    if (kParts && of_part == 0) next_accumulator();
                    if (ok && (st.c & 3) == 0) ok = mbar_wait_warp<!kShares>(sf_full + 8 * rs.idx, rs.phase, abort_flag, p.status, 304);
                    ok = ok && mbar_wait_warp<!kShares>(full + 8 * ru.idx, ru.phase, abort_flag, p.status, 305);
                    if (!ok) break;
                    tc_fence_after();
                    const int end = st.end();
                    const bool last = i + 1 == p.steps || (kParts && of_part + 1 == p.part_steps), group_ends = end == p.units || (end & 3) == 0;
                    if (elect_one_sync()) {
                        const uint32_t sfa = tmem + kSfCol + (uint32_t)(rs.idx * kFp8SfCols), sfb = sfa + 8;
                        const uint64_t a = sw128 | (uint64_t)(((base + (uint32_t)(ru.idx * kFp8Deep) * a_bytes) & 0x3FFFFu) >> 4);
                        const uint64_t b = b_form | (uint64_t)(((b_ring + (uint32_t)(RESIDENT ? st.c : ru.idx * kFp8Deep) * b_bytes) & 0x3FFFFu) >> 4);
                        const uint32_t id = idesc | ((uint32_t)(st.c & 3) << 29) | ((uint32_t)(st.c & 3) << 4);
                        // what lies behind the last block's columns is zeros, and multiplied like the rest
#pragma unroll
                        for (int u = 0; u < kFp8Deep; ++u)
                            if (u == 0 || st.c + u < end)
#pragma unroll
                                for (int kk = 0; kk < 4; ++kk)
                                    tc_mma_fp8<CG>(d, a + u * (a_bytes >> 4) + kStepA * kk, b + u * (b_bytes >> 4) + kStepB * kk, id + u * ((1u << 29) | (1u << 4)), sfa, sfb,
                                                   (kParts ? of_part : i) == 0 && u == 0 && kk == 0 ? 0u : 1u);
                        if (CG == 1) {
                            tc_commit(empty + 8 * ru.idx);
                            if (group_ends) tc_commit(sf_empty + 8 * rs.idx);
                            if (last) tc_commit(d_full + 8 * rd.idx);
                        } else {
                            tc_commit_pair(empty + 8 * ru.idx);
                            if (group_ends) tc_commit_pair(sf_empty + 8 * rs.idx);
                            if (last) tc_commit_pair(d_full + 8 * rd.idx);
                        }
                    }
                    __syncwarp();
                    ru.advance(S);
                    if (group_ends) rs.advance(2);
                    ++of_part;
                    if (kParts && last) {
                        rd.advance(2);
                        of_part = 0;
                    }
                }
                if (!kParts) rd.advance(2);
            }
        }
    };
    auto copy_a = [&] {
        // ------------------------------------------------------------------ A
        Ring ru;
        bool ok = true;
        int issued = 0;
        if (!p.ahead) depend();
        while (ok && tile.next(p)) {
            const int block = CG * tile.rt + rank, row = fp8_row<CG>(p, block), rows = CG == 1 ? fp8_row<CG>(p, block + 1) - row : kBlockRows;
            const CUtensorMap *map = CG == 2 || rows == 4 * div_up(p.rows / 4, p.row_tiles) ? &tmap_a : &tmap_a2;  // boxes of the taller and of the lower tiles
            Fp8Stages st(p, tile.first_group(p, groups));
            for (int i = 0; i < p.steps; ++i, st.advance(), ru.advance(S)) {
                if (issued++ == S) depend();
                ok = mbar_wait_warp<!kShares>(empty + 8 * ru.idx, ru.phase ^ 1, abort_flag, p.status, 300);
                if (!ok) break;
                if (elect_one_sync()) {
                    const uint32_t bar = landed + 8 * ru.idx;
                    const int end = st.end();
                    mbar_expect_tx(bar, (uint32_t)((end - st.c) * (rows << p.fold_log)) * 128u);
                    for (int c = st.c; c < end; ++c) {
                        const uint32_t unit = base + (uint32_t)(ru.idx * kFp8Deep + c - st.c) * a_bytes;
                        for (int f = 0; f < fold; ++f) {  // what lies behind the last block reads as zeros
                            const int at = ((c << p.fold_log) + f) * kFp8Block;
                            const uint32_t to = unit + (uint32_t)(f * part) * 128u;
                            if constexpr (kGated && CG == 1) tma_load_3d(to, map, at, row >> 1, 0, bar);
                            else if constexpr (kGated) tma_load_4d(to, map, at, 0, 0, row >> 4, bar);
                            else if constexpr (kAcrossA) tma_load_2d(to, map, row, at, bar);
                            else tma_load_2d(to, map, at, row, bar);
                        }
                    }
                }
                __syncwarp();
            }
        }
        // The MMAs' commits have arrived at every stage in use before the CTA leaves.
        depend();
        if (total < S) ru = Ring();
        for (int i = min(S, total); ok && i > 0; --i, ru.advance(S)) ok = mbar_wait_warp<!kShares>(empty + 8 * ru.idx, total < S ? 0u : ru.phase ^ 1, abort_flag, p.status, 310);
    };
    auto copy_b = [&] {
        // ------------------------------------------------------------------ B
        Ring ru;
        bool ok = true;
        depend();
        while (ok && tile.next(p)) {
            const int col = tile.col0 + rank * (mma_cols() / CG);
            Fp8Stages st(p, tile.first_group(p, groups));
            for (int i = 0; i < p.steps; ++i, st.advance(), ru.advance(S)) {
                ok = mbar_wait_warp<!kShares>(empty + 8 * ru.idx, ru.phase ^ 1, abort_flag, p.status, 301);
                if (!ok) break;
                if (elect_one_sync()) {
                    const uint32_t bar = landed + 8 * ru.idx;
                    const int end = st.end();
                    mbar_expect_tx(bar, (uint32_t)(end - st.c) * b_bytes);
                    for (int c = st.c; c < end; ++c) {
                        const uint32_t unit = b_ring + (uint32_t)(ru.idx * kFp8Deep + c - st.c) * b_bytes;
                        for (int f = 0; f < fold; ++f) {
                            const int at = ((c << p.fold_log) + f) * kFp8Block;
                            const uint32_t to = unit + (uint32_t)(f * p.b_rows) * 128u;
                            if constexpr (kAcrossB) tma_load_2d(to, &tmap_b, col, at, bar);
                            else tma_load_2d(to, &tmap_b, at, col, bar);
                        }
                    }
                }
                __syncwarp();
            }
        }
    };
    auto landed_here = [&] {
        // ------------------------------------------------------------------ a stage has landed
        const uint32_t leader_full = map_to_rank(full, 0);
        Ring ru;
        depend();
        for (int i = 0; i < total; ++i, ru.advance(S)) {
            if (!mbar_wait_warp<!kShares>(landed + 8 * ru.idx, ru.phase, abort_flag, p.status, 302)) break;
            if (lane == 0) mbar_arrive_cluster(leader_full + 8 * ru.idx);
        }
    };
    auto scales = [&] {
        // ------------------------------------------------------------------ scales to tensor memory
        const int quarter = warp - kFp8ScaleWarp0;
        const uint32_t lanes = tmem + ((uint32_t)(32 * quarter) << 16) + kSfCol;
        const uint32_t leader_full = CG == 1 ? sf_full : map_to_rank(sf_full, 0);
        // Some groups ahead are on their way, as loaded: A's words (dw) or, spread over the lanes, its bytes; B's words, those of a folded tile spread over the lanes too.  They
        // are put together when their turn comes.  One group ahead the loads' latency, 1.5 us while the weights stream, was what single CTAs took for four stages (gated
        // 14336x4096 at 1 token 28.1 us).
        constexpr bool kWordsA = FORM == kFp8Dw;
        constexpr int kAhead = 2;
        struct Group {
            int g, row0, features, col0, valid;  // its number, its tile's rows and columns
            uint32_t a[kWordsA ? 4 : 2], b[CG == 1 ? 2 : 8];
        } ring[kAhead];
        // Square scales: a tile's rows are of one block or two, gated of as many for each projection.  A group has 4 * fold bytes of each, which lie side by side: byte
        // `pos` of slot `slot` is lane (slot * 4 * fold + pos) % 32's.  (A byte for every row, loaded by all lanes, made one line of L2 what all SMs waited for:
        // 8192x8192 at 4096 tokens 205 -> 290 us.)
        const int fold_log = CG == 1 ? p.fold_log : 0;
        bool more = tile.next(p);
        int g = more ? tile.first_group(p, groups) : 0, left = groups;
        auto take = [&](Group &r) {  // the next group
            r.g = g;
            r.row0 = fp8_row<CG>(p, CG * tile.rt + rank);
            r.features = CG == 1 && kGated ? (fp8_row<CG>(p, tile.rt + 1) - r.row0) >> 1 : 8;
            r.col0 = tile.col0;
            r.valid = tile.valid;
            if (++g == groups) g = 0;
            if (--left == 0) {
                left = groups;
                more = tile.next(p);
                if (more) g = tile.first_group(p, groups);
            }
        };
        // Group r.g of the tile: stages 4 r.g .. 4 r.g + 3.  What lies behind the last block or column is any of them: nothing is multiplied with it.
        auto fetch_a = [&](Group &r) {
            if constexpr (kWordsA) {
#pragma unroll
                for (int i = 0; i < 4; ++i) r.a[i] = __ldcg(reinterpret_cast<const uint32_t *>(p.as) + (size_t)r.g * p.rows + min(r.row0 + 32 * i + lane, p.rows - 1));
            } else {
#pragma unroll
                for (int i = 0; i < (CG == 1 ? 2 : 1); ++i) {
                    const int idx = 32 * i + lane, slot = idx >> (2 + fold_log), kb = (4 * r.g << fold_log) + (idx & ((4 << fold_log) - 1));
                    if (slot < (FORM == kFp8Dx ? 1 : kGated ? 4 : 2)) r.a[i] = __ldcg(p.as + fp8_square_scale(FORM == kFp8Dx, kGated, r.row0, slot, kb, p.rows, p.blocks));
                }
            }
        };
        auto fetch_b = [&](Group &r) {
            if constexpr (RESIDENT) {
            } else if (CG == 1 && fold_log) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {  // word w, of `fold` that a group has of a token, of token t: at w * b_rows + t, of 64 at most
                    const int idx = 32 * i + lane, w = idx / p.b_rows, t = min(idx - w * p.b_rows, r.valid - 1), at = min((r.g << fold_log) + w, (p.blocks + 3) / 4 - 1);
                    r.b[i] = __ldcg(reinterpret_cast<const uint32_t *>(p.bs) + (size_t)at * p.cols + r.col0 + t);
                }
            } else {
#pragma unroll
                for (int j = 0; j < (CG == 1 ? 2 : 8); ++j)
                    if (32 * j < r.valid) r.b[j] = __ldcg(reinterpret_cast<const uint32_t *>(p.bs) + (size_t)r.g * p.cols + r.col0 + min(32 * j + lane, r.valid - 1));
            }
        };
        // The last unit's blocks behind the last one are multiplied, zeros that they are: their scales must be numbers, whatever the last words have there.
        uint32_t there[2] = {~0u, ~0u};
        if (CG == 1 && !RESIDENT && fold_log)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int blocks = p.blocks - (4 * (groups - 1) << fold_log) - (32 * j + lane) / p.b_rows, bytes = (blocks + fold - 1) >> fold_log;  // of a column's word
                there[j] = bytes >= 4 ? ~0u : (1u << (8 * max(bytes, 0))) - 1u;
            }
        // MMA column 32 j + lane is column t of block f of a unit
        auto word_b = [&](const Group &r, int j) {
            if constexpr (RESIDENT) {
                uint32_t w;
                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(words_at + 256u * (uint32_t)r.g + 128u * j + 4u * lane));
                return w;
            } else if (CG == 1 && fold_log) {
                const int at = 32 * j + lane, f = at / p.b_rows, t = at - f * p.b_rows;
                uint32_t w = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int block = (i << fold_log) + f, idx = (block >> 2) * p.b_rows + t;  // of the group
                    const uint32_t w0 = __shfl_sync(0xffffffffu, r.b[0], idx & 31), w1 = __shfl_sync(0xffffffffu, r.b[1], idx & 31);
                    w |= (((idx < 32 ? w0 : w1) >> (8 * (block & 3))) & 255u) << (8 * i);
                }
                return r.g + 1 == groups ? w & there[j] : w;
            } else {
                return r.b[j];
            }
        };
        // MMA row 32 i + lane is row `of` of part f
        auto word_a = [&](const Group &r, int i) {
            if constexpr (kWordsA) {
                return r.a[i];
            } else {
                const int m = 32 * i + lane, f = m >> (7 - fold_log), of = m & ((kBlockRows >> fold_log) - 1);
                int slot = 0;
                if constexpr (kGated) {
                    // pairs: eight rows of either projection in turn; single CTAs: one's, then the other's
                    const bool up = CG == 1 ? of >= r.features : (of & 8) != 0;
                    const int base = up ? p.rows / 2 : 0, first = r.row0 >> 1, at = CG == 1 ? (up ? of - r.features : of) : ((of >> 4) << 3) + (of & 7);
                    slot = (up ? 2 : 0) + (base + min(first + at, p.rows / 2 - 1)) / kFp8Block - (base + first) / kFp8Block;
                } else if (FORM == kFp8Product) {
                    slot = min(r.row0 + of, p.rows - 1) / kFp8Block - r.row0 / kFp8Block;
                }
                uint32_t w = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int idx = (slot << (2 + fold_log)) + (j << fold_log) + f;
                    uint32_t b = __shfl_sync(0xffffffffu, r.a[0], idx & 31);
                    if (CG == 1) {
                        const uint32_t b2 = __shfl_sync(0xffffffffu, r.a[1], idx & 31);
                        if (idx >= 32) b = b2;
                    }
                    w |= b << (8 * j);
                }
                return w;
            }
        };
        const int total_groups = tiles * groups;
        int taken = 0, written = 0;
        Ring rs;
        bool ok = true;
        if (!p.ahead) depend();
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            for (uint32_t &w : ring[k].a) w = 0;
            for (uint32_t &w : ring[k].b) w = 0;
            if (taken < total_groups) {
                take(ring[k]);
                fetch_a(ring[k]);
                ++taken;
            }
        }
        depend();
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (k < taken) fetch_b(ring[k]);
        while (ok && written < total_groups) {
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                if (!ok || written >= total_groups) break;
                Group &r = ring[k];
                uint32_t v[kFp8SfCols];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = word_a(r, i), v[4 + i] = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) v[8 + i] = CG == 2 || i < 2 ? word_b(r, CG == 2 ? i : i & 1) : 0u;
                if (taken < total_groups) {
                    take(r);
                    fetch_a(r);
                    fetch_b(r);
                    ++taken;
                }
                ok = mbar_wait_warp<!kShares>(sf_empty + 8 * rs.idx, rs.phase ^ 1, abort_flag, p.status, 306);
                if (!ok) break;
                tc_fence_after();
                tc_st_x16(lanes + (uint32_t)(rs.idx * kFp8SfCols), v);
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (CG == 1) mbar_arrive(sf_full + 8 * rs.idx);
                    else mbar_arrive_cluster(leader_full + 8 * rs.idx);
                }
                rs.advance(2);
                ++written;
            }
        }
        // the commits for the last two groups have arrived before the CTA leaves
        if (total_groups == 1) rs = Ring();
        for (int i = min(2, total_groups); ok && i > 0; --i, rs.advance(2)) ok = mbar_wait_warp<!kShares>(sf_empty + 8 * rs.idx, total_groups == 1 ? 0u : rs.phase ^ 1, abort_flag, p.status, 311);
    };
    auto epilogue = [&] {
        // ------------------------------------------------------------------ epilogue
        const int quarter = warp & 3, thread = threadIdx.x & 127, half = warp / (kFp8ScaleWarp0 + 4);  // which group
        const uint32_t tmem_q = tmem + ((uint32_t)(32 * quarter) << 16);
        OT *o = static_cast<OT *>(p.o), *z = static_cast<OT *>(p.z);
        const int out = kGated ? p.rows / 2 : p.rows;  // numbers of a row of the output
        constexpr int kTileOut = kGated ? kBlockRows / 2 : kBlockRows;
        constexpr uint32_t kPitch = kTileOut * (uint32_t)sizeof(OT) + (sizeof(OT) == 2 || kGated ? 16 : 0);  // 16 bytes more, so that a column of 8 rows meets all banks
        constexpr uint32_t kPitchZ = kBlockRows * 2 + 16;
        const uint32_t out_staging = staging + (uint32_t)(half * kFp8StageCols) * kPitch, z_staging = staging + (uint32_t)p.z_offset + (uint32_t)(half * kFp8StageCols) * kPitchZ;
        auto meet = [&] { asm volatile("bar.sync %0, 128;" ::"r"(1 + 2 * half) : "memory"); };  // the group's four warps
        Ring rd;
        depend();
        int row0 = 0, rows = 0;
        const uint32_t leader_d_empty = CG == 1 ? d_empty : map_to_rank(d_empty, 0);
        auto drained = [&] {  // the accumulator may be overwritten
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (CG == 1) mbar_arrive(d_empty + 8 * rd.idx);
                else mbar_arrive_cluster(leader_d_empty + 8 * rd.idx);
            }
        };
        // The group's staging buffer, which has 32 columns of the tile from t0 on, to memory: 16 bytes a thread and step.
        auto copy_out = [&](int t0) {
            constexpr int kPieces = kTileOut * (int)sizeof(OT) / 16, kStep = 128 / kPieces;
            const int piece = thread % kPieces, have = min(kFp8StageCols, tile.valid - t0);
            if (piece * (16 / (int)sizeof(OT)) < (kGated ? rows / 2 : rows)) {
                uint8_t *to = reinterpret_cast<uint8_t *>(o + (size_t)(tile.col0 + t0) * out + (kGated ? row0 / 2 : row0)) + 16 * piece;
#pragma unroll
                for (int t = thread / kPieces; t < kFp8StageCols; t += kStep) {
                    uint4 v;
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(out_staging + (uint32_t)t * kPitch + 16u * piece));
                    if (t < have) *reinterpret_cast<uint4 *>(to + (size_t)t * out * sizeof(OT)) = v;
                }
            }
            if constexpr (kGated && sizeof(OT) == 2) {
                if (z) {
                    const int which = (thread >> 3) & 1, group = thread & 7;  // of the projections, and eight features of it
                    if (group < rows / 16) {
                        OT *to = z + (size_t)(tile.col0 + t0) * p.rows + (size_t)which * out + row0 / 2 + 8 * group;
#pragma unroll
                        for (int t = thread >> 4; t < kFp8StageCols; t += 8) {
                            uint4 v;
                            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                                         : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                                         : "r"(z_staging + (uint32_t)t * kPitchZ + 16u * (2 * group + which)));
                            if (t < have) *reinterpret_cast<uint4 *>(to + (size_t)t * p.rows) = v;
                        }
                    }
                }
            }
        };
        // 32 columns of the accumulator at `d`, from t on.  16 bits and gated: lo, then hi halves of the lanes in fragments of 8 x 8; otherwise a lane a thread.
        constexpr bool kFragments = kGated || sizeof(OT) == 2;
        auto load = [&](uint32_t d, int t, auto &&take) {
            if constexpr (kFragments) {
                uint32_t lo[16], hi[16];
                tc_ld_16x256b_x4(d + t, lo);
                tc_ld_16x256b_x4(d + (16u << 16) + t, hi);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int i = 0; i < 16; ++i) take(i, __uint_as_float(lo[i])), take(16 + i, __uint_as_float(hi[i]));
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float r[16];
                    tc_ld_x16(d + t + 16 * h, r);
#pragma unroll
                    for (int i = 0; i < 16; ++i) take(16 * h + i, r[i]);
                }
            }
        };
        // 32 columns' sums to the group's staging buffer.
        auto fill_from = [&](const float (&v)[32]) {
            const uint32_t to = out_staging;
            if constexpr (kFragments) {
                auto lo = [&](int i) { return v[i]; };
                auto hi = [&](int i) { return v[16 + i]; };
                // Fragments of 8 rows x 8 columns, packed, are written transposed (stmatrix): 16 bytes = 8 rows of one column.
                auto rows_of_8 = [&](uint32_t at_, uint32_t pitch) {
                    if constexpr (sizeof(OT) == 2) {
                        const uint32_t dst = at_ + (uint32_t)(lane & 7) * pitch + (uint32_t)(4 * quarter + (lane >> 3)) * 16u;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            stmatrix_x4_trans(dst + 8u * i * pitch, mx_pack2<OT>(lo(4 * i), lo(4 * i + 1)), mx_pack2<OT>(lo(4 * i + 2), lo(4 * i + 3)), mx_pack2<OT>(hi(4 * i), hi(4 * i + 1)),
                                              mx_pack2<OT>(hi(4 * i + 2), hi(4 * i + 3)));
                    }
                };
                if constexpr (!kGated) {
                    rows_of_8(to, kPitch);
                } else {
                    if (z) rows_of_8(z_staging, kPitchZ);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {  // lanes i and i + 8 of a half: gate and other projection of one feature, two columns
                        const float2 l = fp8_activation<OT>(lo(4 * i), lo(4 * i + 2), lo(4 * i + 1), lo(4 * i + 3), p.gelu);
                        const float2 h = fp8_activation<OT>(hi(4 * i), hi(4 * i + 2), hi(4 * i + 1), hi(4 * i + 3), p.gelu);
                        if constexpr (sizeof(OT) == 2) {
                            stmatrix_x2_trans(to + (uint32_t)(8 * i + (lane & 7)) * kPitch + (uint32_t)(2 * quarter + ((lane >> 3) & 1)) * 16u, mx_pack2<OT>(l.x, l.y), mx_pack2<OT>(h.x, h.y));
                        } else {
                            const uint32_t dst = to + (uint32_t)(8 * i + 2 * (lane & 3)) * kPitch + (uint32_t)(16 * quarter + (lane >> 2)) * 4u;
                            asm volatile("st.shared.f32 [%0], %1;" ::"r"(dst), "f"(l.x) : "memory");
                            asm volatile("st.shared.f32 [%0], %1;" ::"r"(dst + kPitch), "f"(l.y) : "memory");
                            asm volatile("st.shared.f32 [%0], %1;" ::"r"(dst + 32u), "f"(h.x) : "memory");
                            asm volatile("st.shared.f32 [%0], %1;" ::"r"(dst + kPitch + 32u), "f"(h.y) : "memory");
                        }
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) asm volatile("st.shared.f32 [%0], %1;" ::"r"(to + (uint32_t)i * kPitch + (uint32_t)thread * 4u), "f"(v[i]) : "memory");
            }
        };
        auto next_part = [&] {  // the group's four warps go on together or not at all
            const bool ok = mbar_wait_warp<!kShares>(d_full + 8 * rd.idx, rd.phase, abort_flag, p.status, 307);
            if (bar_any(1 + 2 * half, 128, !ok)) return false;
            tc_fence_after();
            return true;
        };
        // The parts of a tile's sum in order: `take` what the accumulator at `d` has.
        auto each_part = [&](auto &&take) {
            for (int i = 0; i < p.parts; ++i, rd.advance(2)) {
                if (!next_part()) return false;
                take(tmem_q + (uint32_t)(rd.idx * p.d_cols));
                drained();
            }
            return true;
        };
        while (tile.next(p)) {
            row0 = fp8_row<CG>(p, CG * tile.rt + rank);
            rows = max(0, min(CG == 1 ? fp8_row<CG>(p, tile.rt + 1) : row0 + kBlockRows, p.rows) - row0);
            if constexpr (CG == 1) {
                const int f = thread >> (7 - p.fold_log), features = rows >> 1;
                float *sums = reinterpret_cast<float *>(smem + (staging - base));
                float v[kFp8SingleCols];
                if constexpr (kParts) {
#pragma unroll
                    for (int c = 0; c < kFp8SingleCols; ++c) v[c] = -0.0f;  // as below
                    if (!each_part([&](uint32_t d) {
                            float w[kFp8SingleCols];
                            tc_ld_x16(d + f * p.b_rows, w);
#pragma unroll
                            for (int c = 0; c < kFp8SingleCols; ++c) v[c] += w[c];
                        }))
                        break;
                } else {
                    if (!next_part()) break;
                    tc_ld_x16(tmem_q + (uint32_t)(rd.idx * p.d_cols) + f * p.b_rows, v);
                    drained();
                    rd.advance(2);
                }
                if (!kGated && p.fold_log == 0) {
                    OT *to = o + row0 + thread;
                    if (thread < rows) {
#pragma unroll
                        for (int i = 0; i < kFp8SingleCols; ++i)
                            if (i < tile.valid) to[(size_t)i * out] = mx_convert<OT>(v[i]);
                    }
                } else {
                    // Part f's sums of row i are lane part * f + i, columns b_rows * f ..: added up in the order of the parts.
#pragma unroll
                    for (int t = 0; t < kFp8SingleCols; ++t)
                        if (t < tile.valid) sums[t * kBlockRows + thread] = v[t];
                    meet();
                    auto sum = [&](int t, int i) {
                        float s = sums[t * kBlockRows + i];
                        for (int g = 1; g < fold; ++g) s += sums[t * kBlockRows + g * part + i];
                        return s;
                    };
                    if constexpr (kGated) {
                        const int i = thread & 63;
                        for (int t = thread >> 6; t < tile.valid && i < features; t += 2) {
                            const float g = sum(t, i), u = sum(t, features + i);
                            o[(size_t)t * out + row0 / 2 + i] = mx_convert<OT>(fp8_activation<OT>(g, u, g, u, p.gelu).x);
                            if (z) {
                                OT *to = z + (size_t)t * p.rows + row0 / 2 + i;
                                to[0] = mx_convert<OT>(g);
                                to[out] = mx_convert<OT>(u);
                            }
                        }
                    } else {
                        const int i = thread & (part - 1);
                        for (int t = f; t < tile.valid && i < rows; t += fold) o[(size_t)t * out + row0 + i] = mx_convert<OT>(sum(t, i));
                    }
                    meet();  // they have been read
                }
            } else if constexpr (!kParts) {
                if (!next_part()) break;
                const uint32_t d = tmem_q + (uint32_t)(rd.idx * p.d_cols);
                for (int t0 = half * kFp8StageCols; t0 < p.tile_cols; t0 += 2 * kFp8StageCols) {
                    meet();  // what was staged before has been copied
                    if (t0 < tile.valid) {
                        float v[kFp8StageCols];
                        load(d, t0, [&](int c, float w) { v[c] = w; });
                        fill_from(v);
                    }
                    if (t0 + 2 * kFp8StageCols >= p.tile_cols) drained();
                    meet();
                    copy_out(t0);
                }
                if (half * kFp8StageCols >= p.tile_cols) drained();
                rd.advance(2);
            } else {
                float v[SLICES][kFp8StageCols];  // columns 32 half + 64 j on
#pragma unroll
                for (int j = 0; j < SLICES; ++j)
#pragma unroll
                    for (int c = 0; c < kFp8StageCols; ++c) v[j][c] = -0.0f;  // any number that is added to it stays as it is
                if (!each_part([&](uint32_t d) {
#pragma unroll
                        for (int j = 0; j < SLICES; ++j)
                            if ((half + 2 * j) * kFp8StageCols < tile.valid) load(d, (half + 2 * j) * kFp8StageCols, [&](int c, float w) { v[j][c] += w; });
                    }))
                    break;
                // One copy of what follows, whose first run by a CTA waits for its instructions: the sums move down instead of being indexed (unrolled, gated 14336x4096 at 43 tokens
                // 34 us, so 30).
#pragma unroll 1
                for (int t0 = half * kFp8StageCols; t0 < tile.valid; t0 += 2 * kFp8StageCols) {
                    meet();  // what was staged before has been copied
                    fill_from(v[0]);
#pragma unroll
                    for (int j = 0; j + 1 < SLICES; ++j)
#pragma unroll
                        for (int c = 0; c < kFp8StageCols; ++c) v[j][c] = v[j + 1][c];
                    meet();
                    copy_out(t0);
                }
            }
        }
    };
    if constexpr (kShares) {  // four groups of four warps: each takes its share of the registers
        if (warp < kFp8EpilogueWarp0) {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFp8IssueRegs));
            if (warp == 0) issue();
            else if (warp == 1) copy_a();
            else if (warp == 2) copy_b();
            else landed_here();
        } else if (warp >= kFp8ScaleWarp0 && warp < kFp8ScaleWarp0 + 4) {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFp8ScaleRegs));
            scales();
        } else {
            asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kFp8EpilogueRegs));
            epilogue();
        }
    } else {  // one choice after the other: nested as above a launch of few tokens takes 0.5 us longer
        if (warp == 0) issue();
        else if (warp == 1) copy_a();
        else if (warp == 2 && !RESIDENT) copy_b();
        else if (warp == 3 && CG == 2) landed_here();
        else if (warp >= kFp8ScaleWarp0 && warp < kFp8ScaleWarp0 + 4) scales();
        else if (warp >= kFp8EpilogueWarp0) epilogue();
    }

    __syncwarp();
    if (FORM == kFp8Dw && p.beside) asm volatile("griddepcontrol.wait;" ::: "memory");
    tc_fence_before();
    __syncthreads();
    if (CG == 2) cluster_sync_all();
    if (warp == 3) {
        tc_fence_after();
        if (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
    }
}

template <int CG, int FORM, bool RESIDENT, int SLICES, typename OT>
__global__ void __launch_bounds__(32 * fp8_warps(CG), CG == 1 ? 2 : 1)
fp8_gemm_kernel(const __grid_constant__ Fp8Params p, const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_a2, const __grid_constant__ CUtensorMap tmap_b)
{
    fp8_gemm<CG, FORM, RESIDENT, SLICES, OT>(p, tmap_a, tmap_a2, tmap_b, blockIdx.x / CG, gridDim.x / CG);
}

// dx and dw in one launch, the first `dx_pairs` pairs and the others: where neither fills the device.
template <int SLICES, typename XT, typename WT>
__global__ void __launch_bounds__(32 * fp8_warps(2), 1)
fp8_gradients_kernel(const __grid_constant__ Fp8Params dx, const __grid_constant__ CUtensorMap dx_a, const __grid_constant__ CUtensorMap dx_b, const __grid_constant__ Fp8Params dw,
                     const __grid_constant__ CUtensorMap dw_a, const __grid_constant__ CUtensorMap dw_b, int dx_pairs)
{
    const int pair = blockIdx.x / 2, pairs = gridDim.x / 2;
    if (pair < dx_pairs) fp8_gemm<2, kFp8Dx, false, sizeof(XT) == 4 ? SLICES : 0, XT>(dx, dx_a, dx_a, dx_b, pair, dx_pairs);
    else fp8_gemm<2, kFp8Dw, false, sizeof(WT) == 4 ? SLICES : 0, WT>(dw, dw_a, dw_a, dw_b, pair - dx_pairs, pairs - dx_pairs);
}

// ------------------------------------------------------------------ host side

struct Fp8Plan {
    int cg, tile_cols, width, col_tiles, stages, d_cols;
    bool resident;
    int fold_log, row_tiles, a_bytes, b_rows, z_offset;
    int workers;
    size_t smem;
};

// Microseconds that tiles of 256 rows and `cols` columns take on `pairs` pairs, beside what a launch costs: rounds of tiles, each with its steps of 128 (the
// tensor pipe's four MMAs, which take hardly less for few columns) and what of a wide tile's epilogue nothing hides; what all tiles copy, from L2; A, from HBM.  Compared with 2400
// launches (16 matrices from 512x4096 to 57344x8192, plain and gated, 1 to 4096 tokens, every width): what it chooses takes 1.4 % longer than the fastest width in the mean,
// 18 % at worst (2720x784, gated, at 2000 tokens); constants fitted to these launches choose no better.
static double fp8_pair_us(int rows, int n, int red, int cols, int pairs)
{
    const int row_tiles = div_up(rows, 2 * kBlockRows), blocks = div_up(red, kFp8Block);
    const double tiles = (double)row_tiles * div_up(n, cols);
    const double rounds = std::ceil(tiles / pairs);
    const int width = div_up(div_up(n, div_up(n, cols)), 16) * 16;  // tiles are of equal width
    const double step = cols <= 128 ? 0.183 + 0.00013 * width : 0.036 + 0.00118 * width;
    const double work = rounds * (std::max(0.0, 0.0086 * width - 0.5) + blocks * step);
    const double copies = tiles * (2 * kBlockRows + cols) * blocks * 128.0 / 21.7e6, weights = (double)rows * red / 6.5e6;
    return std::sqrt(work * work + copies * copies + weights * weights);
}

static int fp8_pair_cols(int rows, int n, int red, int form, int pairs)
{
    // Two accumulators and two buffers of scales fill tensor memory with 240.  Of dw multiples of 32: what a CTA stages starts at a multiple of 16 columns
    static const int widths[] = {240, 224, 208, 192, 176, 160, 144, 128, 112, 96, 80, 64, 48, 32, 16, 0};
    const int unit = form == kFp8Dw ? 32 : 16;
    int best = 0;
    double best_us = 0;
    for (int i = 0; widths[i]; ++i) {
        const int cols = widths[i];
        int narrower = 0;
        for (int j = i + 1; widths[j] && !narrower; ++j)
            if (widths[j] % unit == 0) narrower = widths[j];
        if (cols % unit || div_up(n, div_up(n, cols)) <= narrower) continue;  // the next narrower one holds the same tiles
        const double us = fp8_pair_us(rows, n, red, cols, pairs);
        if (!best || us < best_us) best = cols, best_us = us;
    }
    return best;
}

// Shared memory: `fixed` bytes, and as many stages as `room` has place for.
static void fp8_stages(Fp8Plan &l, size_t room, size_t fixed, size_t b_unit)
{
    const size_t unit = l.a_bytes + b_unit;
    l.stages = (int)std::min<size_t>(kFp8MaxStages, (room - fixed) / (kFp8Deep * unit));
    // the last unit's MMAs read 128 rows
    l.smem = std::max((size_t)(l.stages * kFp8Deep) * unit + fixed, (size_t)(l.stages * kFp8Deep - 1) * l.a_bytes + kBlockRows * 128);
}

static Fp8Plan fp8_plan_single(bool gated, int rows, int n, int red, int x_type, int sm_count)
{
    Fp8Plan l = {};
    const int blocks = div_up(red, kFp8Block);
    l.cg = 1;
    l.workers = sm_count;
    l.tile_cols = l.width = l.b_rows = div_up(n, 8) * 8;
    l.col_tiles = 1;
    l.row_tiles = (int)std::min<long long>(rows / 4, div_up_ll(rows, (long long)kBlockRows * sm_count) * sm_count);
    const int height = 4 * div_up(rows / 4, l.row_tiles);
    l.fold_log = height <= 32 ? 2 : height <= 64 ? 1 : 0;
    l.a_bytes = (l.fold_log ? kBlockRows : div_up(height, 8) * 8) * 128;
    const int fold = 1 << l.fold_log, units = div_up(blocks, fold);
    l.d_cols = l.b_rows * fold;
    const size_t fixed = l.fold_log || gated ? kFp8SumBytes : 0;
    // Tokens that the CTAs quantize themselves: one round of the quantizing warps, and shared memory left for stages enough.
    const size_t resident = (size_t)units * fold * n * 128 + 256 * (size_t)div_up(units, 4);
    l.resident = x_type != TUNA_FP8 && n <= 8 && (long long)div_up(units * fold, 2) * n <= kFp8ResidentLoads * (fp8_warps(1) - 1) && resident + 4 * (size_t)l.a_bytes + fixed <= kFp8SmemHalf;
    if (l.resident) fp8_stages(l, kFp8SmemHalf, fixed + resident, 0);
    else fp8_stages(l, kFp8SmemHalf, fixed, (size_t)l.b_rows * fold * 128);
    return l;
}

static Fp8Plan fp8_plan_pairs(int form, int rows, int n, int red, int o_type, bool with_z, int sm_count)
{
    Fp8Plan l = {};
    const bool gated = form == kFp8GatedProduct;
    const int o_bytes = o_type == TUNA_FP32 ? 4 : 2, unit = form == kFp8Dw ? 32 : 16;
    l.cg = 2;
    l.workers = sm_count / 2;
    l.tile_cols = l.d_cols = fp8_pair_cols(rows, n, red, form, l.workers);
    l.width = div_up(div_up(n, div_up(n, l.tile_cols)), unit) * unit;
    l.col_tiles = div_up(n, l.width);
    l.row_tiles = div_up(rows, 2 * kBlockRows);
    // Rows in tiles of 256, also where that leaves the last round of tiles short: tiles of equal height that fill it are no faster (us, 256 / equal: 28672x4096 at 43 tokens
    // 21.7 / 22.3, 11024x4112 at 43 13.5 / 13.3, 57344x8192 at 64 78.9 / 77.4, 4096x14336 at 64 22.5 / 25.4).
    l.a_bytes = kBlockRows * 128;
    l.b_rows = form == kFp8Dw ? kBlockRows : l.tile_cols / 2;
    const size_t pitch = gated ? 64 * o_bytes + 16 : kBlockRows * o_bytes + (o_bytes == 2 ? 16 : 0);
    size_t fixed = 2 * kFp8StageCols * pitch;
    l.z_offset = (int)fixed;
    if (with_z) fixed += 2 * kFp8StageCols * (kBlockRows * 2 + 16);
    fp8_stages(l, kFp8SmemMax, fixed, (size_t)l.b_rows * 128);
    return l;
}

// rows x red of A, n columns.  x_type: TUNA_FP8, or what B is before it is quantized.
static Fp8Plan fp8_plan(int form, int rows, int n, int red, int x_type, int o_type, bool with_z, int sm_count)
{
    // Single CTAs take what they quantize themselves, and few rows of long sums, which their tiles of any height share evenly and fold (us, single / pairs, codes: 4096x4096
    // at 16 tokens 7.1 / 8.5, 4096x14336 at 1 14.5 / 21.5, 10240x8192 at 1 16.8 / 18.1; 1024x1024 at 8 4.5 / 4.0, 28672x4096 at 16 22.1 / 20.5).
    if (form <= kFp8GatedProduct && n <= kFp8SingleCols) {
        const Fp8Plan l = fp8_plan_single(form == kFp8GatedProduct, rows, n, red, x_type, sm_count);
        if (l.resident || (rows <= sm_count * kBlockRows && red >= 2048)) return l;
    }
    return fp8_plan_pairs(form, rows, n, red, o_type, with_z, sm_count);
}

bool fp8_gemm_takes(bool gated, int rows, int n, int red, int x_type, int sm_count)
{
    if (x_type == TUNA_FP8) return true;
    return fp8_plan(gated ? kFp8GatedProduct : kFp8Product, rows, n, red, x_type, TUNA_FP16, false, sm_count).resident;
}

struct Fp8Maps {
    CUtensorMap a, a2, b;
};

// Launches a kernel on `ctas` CTAs, CG of a cluster.
template <int CG, typename... Params, typename... Args>
static int launch_fp8_kernel(void (*kernel)(Params...), int ctas, size_t smem, cudaStream_t stream, const Args &...args)
{
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)ctas);
    lc.blockDim = dim3(32 * fp8_warps(CG));
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
    return cudaLaunchKernelEx(&lc, kernel, args...) == cudaSuccess ? TUNA_OK : TUNA_ERR_LAUNCH;
}

// Once a device: the kernel may have as much shared memory as it asks for, and, if its warps share their registers out, was built to be launched with what they share (with
// fewer, those who ask for more would wait for good).
struct Fp8Allowed {
    bool set[64] = {false};
    std::mutex mu;
    int allow(const void *kernel, bool shares)
    {
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return TUNA_ERR_NO_DEVICE;
        std::lock_guard<std::mutex> lock(mu);
        if (set[dev]) return TUNA_OK;
        cudaFuncAttributes has;
        if (cudaFuncGetAttributes(&has, kernel) != cudaSuccess || (shares && has.numRegs < kFp8LaunchRegs)) return TUNA_ERR_NO_DEVICE;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kFp8SmemMax) != cudaSuccess) return TUNA_ERR_NO_DEVICE;
        set[dev] = true;
        return TUNA_OK;
    }
};

template <int CG, int FORM, bool RESIDENT, int SLICES, typename OT>
static int launch_fp8(const Fp8Params &p, const Fp8Maps &maps, int ctas, size_t smem, cudaStream_t stream)
{
    static Fp8Allowed allowed;
    const int st = allowed.allow((const void *)fp8_gemm_kernel<CG, FORM, RESIDENT, SLICES, OT>, SLICES > kFp8NarrowSlices);
    return st != TUNA_OK ? st : launch_fp8_kernel<CG>(fp8_gemm_kernel<CG, FORM, RESIDENT, SLICES, OT>, ctas, smem, stream, p, maps.a, maps.a2, maps.b);
}

// A launch: plan, parameters and tensor maps.
struct Fp8Launch {
    int form, o_type;
    Fp8Plan l;
    Fp8Params p;
    Fp8Maps maps;
    int pairs() const { return (int)std::min<long long>((long long)l.row_tiles * l.col_tiles, l.workers); }  // or single CTAs
};

template <int SLICES, typename OT>
static int launch_fp8_pairs(const Fp8Launch &a, cudaStream_t stream)
{
    const int ctas = 2 * a.pairs();
    if (a.form == kFp8GatedProduct) return launch_fp8<2, kFp8GatedProduct, false, SLICES, OT>(a.p, a.maps, ctas, a.l.smem, stream);
    constexpr int kSlices = sizeof(OT) == 4 ? SLICES : 0;
    switch (a.form) {
        case kFp8Product: return launch_fp8<2, kFp8Product, false, kSlices, OT>(a.p, a.maps, ctas, a.l.smem, stream);
        case kFp8Dx: return launch_fp8<2, kFp8Dx, false, kSlices, OT>(a.p, a.maps, ctas, a.l.smem, stream);
        default: return launch_fp8<2, kFp8Dw, false, kSlices, OT>(a.p, a.maps, ctas, a.l.smem, stream);
    }
}

template <int SLICES, typename OT>
static int launch_fp8_singles(const Fp8Launch &a, cudaStream_t stream)
{
    const int ctas = a.pairs();
    if (a.form == kFp8GatedProduct)
        return a.l.resident ? launch_fp8<1, kFp8GatedProduct, true, SLICES, OT>(a.p, a.maps, ctas, a.l.smem, stream) : launch_fp8<1, kFp8GatedProduct, false, SLICES, OT>(a.p, a.maps, ctas, a.l.smem, stream);
    constexpr int kSlices = sizeof(OT) == 4 ? SLICES : 0;
    return a.l.resident ? launch_fp8<1, kFp8Product, true, kSlices, OT>(a.p, a.maps, ctas, a.l.smem, stream) : launch_fp8<1, kFp8Product, false, kSlices, OT>(a.p, a.maps, ctas, a.l.smem, stream);
}

template <typename OT>
static int launch_fp8_as(const Fp8Launch &a, cudaStream_t stream)
{
    const Fp8Plan &l = a.l;
    if (l.cg == 1) return a.p.parts == 1 ? launch_fp8_singles<0, OT>(a, stream) : launch_fp8_singles<1, OT>(a, stream);
    if (a.p.parts == 1) return launch_fp8_pairs<0, OT>(a, stream);
    return l.tile_cols <= kFp8NarrowCols ? launch_fp8_pairs<kFp8NarrowSlices, OT>(a, stream) : launch_fp8_pairs<kFp8WideSlices, OT>(a, stream);
}

static int launch_fp8_any(const Fp8Launch &a, cudaStream_t stream)
{
    switch (a.o_type) {
        case TUNA_FP16: return launch_fp8_as<__half>(a, stream);
        case TUNA_BF16: return launch_fp8_as<__nv_bfloat16>(a, stream);
        default: return launch_fp8_as<float>(a, stream);
    }
}

// x_type: of tokens that the product takes as they are, otherwise TUNA_FP8
static int prepare_fp8(Fp8Launch &out, int form, const Fp8Codes &a, int rows, const Fp8Codes &b, int cols, int red, const void *numbers, int x_type, void *o, int o_type, void *z, int gelu,
                       int sm_count)
{
    const Fp8Plan l = fp8_plan(form, rows, cols, red, numbers && !b.q ? x_type : TUNA_FP8, o_type, z != nullptr, sm_count);
    Fp8Params &p = out.p;
    std::memset(&p, 0, sizeof(p));
    p.as = (const uint8_t *)a.s; p.bs = (const uint8_t *)b.s; p.o = o; p.z = z; p.x = numbers;
    p.rows = rows; p.cols = cols; p.red = red;
    p.blocks = div_up(red, kFp8Block);
    p.fold_log = l.fold_log; p.units = div_up(p.blocks, 1 << l.fold_log); p.steps = div_up(p.units, kFp8Deep);
    p.parts = o_type == TUNA_FP32 || z ? div_up(p.steps, l.tile_cols <= kFp8NarrowCols ? kFp8PartSteps : kFp8WidePartSteps) : 1;
    p.part_steps = div_up(p.steps, p.parts); p.parts = div_up(p.steps, p.part_steps);
    p.tile_cols = l.tile_cols; p.width = l.width; p.row_tiles = l.row_tiles; p.col_tiles = l.col_tiles;
    p.rows_inner = l.row_tiles < l.col_tiles;
    p.a_bytes = l.a_bytes; p.b_rows = l.b_rows; p.stages = l.stages; p.d_cols = l.d_cols;
    p.ahead = form <= kFp8GatedProduct && cols <= kFp8AheadTokens;
    p.stagger = form <= kFp8GatedProduct && !l.fold_log;
    p.x_bf16 = x_type == TUNA_BF16; p.gelu = gelu; p.z_offset = l.z_offset;
    p.status = device_status_word();
    if (!p.status) return TUNA_ERR_NO_DEVICE;
    // the kernel numbers tiles and a worker's stages in 32 bits
    const long long tiles = (long long)p.row_tiles * p.col_tiles;
    if (tiles >= 1ll << 30 || (tiles / l.workers + 2) * p.units >= 1ll << 30) return TUNA_ERR_TOO_LARGE;

    Fp8Maps &maps = out.maps;
    auto matrix = [](CUtensorMap *map, const void *at, int inner, int outer, int box_outer) {  // row by row; boxes of 128 columns
        return make_tensor_map_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, at, (uint64_t)inner, (uint64_t)outer, (uint64_t)inner, kFp8Block, (uint32_t)box_outer, CU_TENSOR_MAP_SWIZZLE_128B);
    };
    auto weights = [&](CUtensorMap *map, int height) {
        if (form == kFp8Product) return matrix(map, a.q, red, rows, height);
        if (form != kFp8GatedProduct) return matrix(map, a.q, rows, red, kFp8Block);
        const uint64_t k = (uint64_t)red, f = (uint64_t)rows / 2;
        if (l.cg == 1)  // [gate or other][features][k]
            return make_tensor_map_3d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.q, k, f, 2, k, f * k, kFp8Block, (uint32_t)height / 2, 2, CU_TENSOR_MAP_SWIZZLE_128B);
        // [features by eight][gate or other][eight][k]
        const uint64_t dims[4] = {k, 8, 2, f / 8}, strides[3] = {k, f * k, 8 * k};
        const uint32_t box[4] = {kFp8Block, 8, 2, (uint32_t)height / 16};
        return make_tensor_map_nd(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.q, 4, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    };
    if (!weights(&maps.a, l.cg == 1 ? 4 * div_up(rows / 4, l.row_tiles) : kBlockRows)) return TUNA_ERR_NO_DEVICE;
    maps.a2 = maps.b = maps.a;
    if (l.cg == 1 && rows / 4 % l.row_tiles && !weights(&maps.a2, 4 * (rows / 4 / l.row_tiles))) return TUNA_ERR_NO_DEVICE;
    if (!l.resident && !(form == kFp8Dw ? matrix(&maps.b, b.q, cols, red, kFp8Block) : matrix(&maps.b, b.q, red, cols, l.b_rows))) return TUNA_ERR_NO_DEVICE;
    out.form = form;
    out.o_type = o_type;
    out.l = l;
    return TUNA_OK;
}

int launch_fp8_product(const Fp8ProductArgs &a)
{
    Fp8Launch launch;
    const int st = prepare_fp8(launch, a.gated ? kFp8GatedProduct : kFp8Product, a.w, a.m, a.x, a.n, a.k, a.numbers, a.x_type, a.o, a.o_type, a.z, a.gelu, a.sm_count);
    if (st != TUNA_OK) return st;
    if (a.numbers && a.x.q && launch_fp8_quantize_rows(a.numbers, a.x_type, a.k, a.x.q, a.x.s, a.n, a.k, true, a.stream) != cudaSuccess) return TUNA_ERR_LAUNCH;
    return launch_fp8_any(launch, a.stream);
}

template <int SLICES, typename XT, typename WT>
static int launch_fp8_both_of(const Fp8Launch &dx, const Fp8Launch &dw, cudaStream_t stream)
{
    static Fp8Allowed allowed;
    const int st = allowed.allow((const void *)fp8_gradients_kernel<SLICES, XT, WT>, SLICES > kFp8NarrowSlices), dx_pairs = dx.pairs();
    return st != TUNA_OK ? st : launch_fp8_kernel<2>(fp8_gradients_kernel<SLICES, XT, WT>, 2 * (dx_pairs + dw.pairs()), std::max(dx.l.smem, dw.l.smem), stream, dx.p, dx.maps.a, dx.maps.b, dw.p,
                                                     dw.maps.a, dw.maps.b, dx_pairs);
}
template <typename XT, typename WT>
static int launch_fp8_both(const Fp8Launch &dx, const Fp8Launch &dw, cudaStream_t stream)
{
    if constexpr (sizeof(XT) == 4 || sizeof(WT) == 4)
        if (dx.p.parts > 1 || dw.p.parts > 1)
            return std::max(dx.l.tile_cols, dw.l.tile_cols) <= kFp8NarrowCols ? launch_fp8_both_of<kFp8NarrowSlices, XT, WT>(dx, dw, stream) : launch_fp8_both_of<kFp8WideSlices, XT, WT>(dx, dw, stream);
    return launch_fp8_both_of<0, XT, WT>(dx, dw, stream);
}
template <typename XT>
static int launch_fp8_both_as(const Fp8Launch &dx, const Fp8Launch &dw, cudaStream_t stream)
{
    switch (dw.o_type) {
        case TUNA_FP16: return launch_fp8_both<XT, __half>(dx, dw, stream);
        case TUNA_BF16: return launch_fp8_both<XT, __nv_bfloat16>(dx, dw, stream);
        default: return launch_fp8_both<XT, float>(dx, dw, stream);
    }
}

int launch_fp8_backward(const Fp8BackwardArgs &a)
{
    const Fp8GradientArgs &g = a.operands;
    const int m = g.cols, n = g.rows, k = g.x_cols;
    Fp8Launch dx, dw;
    auto plan = [&](int sms) {
        int st = a.dx ? prepare_fp8(dx, kFp8Dx, a.w, k, g.by_row, n, m, nullptr, TUNA_FP8, a.dx, a.dx_type, nullptr, 0, sms) : TUNA_OK;
        if (st == TUNA_OK && a.dw) st = prepare_fp8(dw, kFp8Dw, a.x, k, g.by_column, m, n, nullptr, TUNA_FP8, a.dw, a.dw_type, nullptr, 0, sms);
        return st;
    };
    int st = plan(g.sm_count);
    if (st != TUNA_OK) return st;
    // Up to 2^35 products side by side in one launch, half of the pairs each; above, dw behind dx, and beside it where that leaves pairs idle (us, one launch / two:
    // 1552x1040 at 301 tokens 14.7 / 19.5, 2048x2048 at 256 17.2 / 22.9, at 1024 23.5 / 27.6, 6144x4096 at 300 41.4 / 40.7, at 1024 61.2 / 64.5, at 4096 195 / 190, 28672x4096 at 2048
    // 547 / 450 to 490).
    const bool together = a.dx && a.dw && (double)m * n * k <= (double)(1ll << 35);
    if (together && (st = plan(g.sm_count / 2)) != TUNA_OK) return st;
    if (launch_fp8_gradient(g) != cudaSuccess) return TUNA_ERR_LAUNCH;
    if (!a.dx || !a.dw) return launch_fp8_any(a.dx ? dx : dw, g.stream);
    if (together) {
        switch (a.dx_type) {
            case TUNA_FP16: return launch_fp8_both_as<__half>(dx, dw, g.stream);
            case TUNA_BF16: return launch_fp8_both_as<__nv_bfloat16>(dx, dw, g.stream);
            default: return launch_fp8_both_as<float>(dx, dw, g.stream);
        }
    }
    dx.p.beside = dw.p.beside = 1;
    st = launch_fp8_any(dx, g.stream);
    return st != TUNA_OK ? st : launch_fp8_any(dw, g.stream);
}

}  // namespace tuna
