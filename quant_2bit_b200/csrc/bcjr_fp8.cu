// 8-bit floating point (e4m3) linear layers with one fp32 scale for each
// block of 128: the two quantizers and the product.
//
//   rows    segment (t, j) = x[t, 128 j .. 128 j + 127]
//   blocks  block (i, j)   = w[128 i .. 128 i + 127, 128 j .. 128 j + 127]
//   amax = max(max |x|, 2^-100),  scale = amax (1/448),  q = e4m3(x (448 (1/amax)))
//
// with fp32 products and reciprocals rounded to nearest, so that the same
// elementary operations give the same bits anywhere.  448 is the largest e4m3
// value; q is off by at most half a step, 2^-4 relative above the subnormals;
// 2^-100 keeps the reciprocal finite for blocks of zeros.
//
//   forward  out[t, n] = sum_j xs[t, j] ws[n / 128, j] sum_{k in j} xq[t, k] wq[n, k]
//   dgrad    out[t, k] = sum_i gs[t, i] ws[i, k / 128] sum_{n in i} gq[t, n] wq[n, k]
//
// The inner sums run on the tensor cores into fp32 accumulators, one for each
// block of 128; the outer sum is fp32 in registers (kernel: bcjr_mm.cuh).
#include "../../include/bcjr_b200.h"
#include "bcjr_kernels.h"
#include "bcjr_mm.cuh"

namespace bcjr {
namespace mm {
namespace {

constexpr int kQThreads = 256, kUnroll = 4, kQRows = kQThreads / 16;

// 16 lanes per segment, 8 elements per lane (the width is a multiple of 16).
// 8192 x 2048 bf16 (50 MB) 12.6 us = 4.0 TB/s of 6.5, one row 2 us a launch.
// Bound by issue and latency: the issue slots are 54 % busy, memory 41 %.
// A block has 16 rows and kUnroll neighbouring segments of each, all loaded
// before the first is used; the scales of a column of segments, side by side
// when they are stored block by block, leave together.
template <typename T>
__global__ void __launch_bounds__(kQThreads)
quantize_rows(const T *__restrict__ x, long ld, long rows, int k, uint8_t *__restrict__ q,
              float *__restrict__ scale, long s_row, long s_blk) {
    let_next_start();              // the product's set-up may overlap (it waits for this kernel's end)
    const int sub = threadIdx.x & 15, blk0 = blockIdx.y * kUnroll;
    const long row = long(blockIdx.x) * kQRows + (threadIdx.x >> 4);
    const bool live = row < rows;
    float v[kUnroll][8];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int c = (blk0 + u) * 128 + sub * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[u][i] = 0.f;
        if (live && c < k) load8(x + row * ld + c, v[u]);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        float m = amax8(v[u]);
#pragma unroll
        for (int d = 8; d; d >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
        m = block_amax(m);
        const int c = (blk0 + u) * 128 + sub * 8;
        if (live && c < k) *reinterpret_cast<uint2 *>(q + row * k + c) = to_e4m3(v[u], block_inv(m));
        if (live && sub == 0 && c < k) scale[row * s_row + (blk0 + u) * s_blk] = block_scale(m);
    }
}

// One block of 128 x 128 per thread block, held in registers between its
// maximum and its rounding: read once.  2048 x 8192 fp32 (84 MB) 14.3 us = 5.9
// TB/s, bound by memory; in bf16 (50 MB) 13.3 us = 3.8 TB/s, bound by latency:
// the same number of elements in flight are half the bytes.
template <typename T>
__global__ void __launch_bounds__(kQThreads)
quantize_blocks(const T *__restrict__ w, int n, int k, uint8_t *__restrict__ q,
                float *__restrict__ scale) {
    __shared__ float part[kQThreads / 32];
    const int kb = (k + 127) / 128, nb = (n + 127) / 128;
    const long id = blockIdx.x, e = id / (long(nb) * kb);
    const int in = int(id - e * nb * kb), bi = in / kb, bj = in - bi * kb;
    const int c = bj * 128 + (threadIdx.x & 15) * 8, r0 = bi * 128 + (threadIdx.x >> 4);
    const long base = e * n * long(k);
    float v[8][8], m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
        if (r0 + 16 * i < n && c < k) load8(w + base + (r0 + 16 * i) * long(k) + c, v[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max_nan(m, amax8(v[i]));
#pragma unroll
    for (int d = 16; d; d >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kQThreads / 32; ++i) m = max_nan(m, part[i]);
    m = block_amax(m);
    const float inv = block_inv(m);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (r0 + 16 * i < n && c < k)
            *reinterpret_cast<uint2 *>(q + base + (r0 + 16 * i) * long(k) + c) = to_e4m3(v[i], inv);
    if (threadIdx.x == 0) scale[id] = block_scale(m);
}

template <typename T>
cudaError_t run_rows(const void *x, long ld, long rows, int k, void *q, float *scale, long s_row,
                     long s_blk, cudaStream_t st) {
    const dim3 grid(unsigned((rows + kQRows - 1) / kQRows), unsigned(((k + 127) / 128 + kUnroll - 1) / kUnroll));
    quantize_rows<T><<<grid, kQThreads, 0, st>>>(
        static_cast<const T *>(x), ld, rows, k, static_cast<uint8_t *>(q), scale, s_row, s_blk);
    return cudaGetLastError();
}

template <typename T>
cudaError_t run_blocks(const void *w, long blocks, int n, int k, void *q, float *scale, cudaStream_t st) {
    quantize_blocks<T><<<unsigned(blocks), kQThreads, 0, st>>>(static_cast<const T *>(w), n, k,
                                                               static_cast<uint8_t *>(q), scale);
    return cudaGetLastError();
}

// ---------------------------------------------------------------------------
// The product with more than a few rows to a group.
//
// Every k block of 128 is scaled on its own, so the tensor core's sums leave
// TMEM once for each of them, and that traffic and the fp32 additions, not the
// products, bound the kernel.  Here the rows of x lie on the lanes and the
// features on the columns (the other way round from mm_kernel): a thread has
// one row, a half of the epilogue one block of 128 features, and the two
// scales become one factor per thread and block, against one for each column.
// Each half has accumulator buffers and an issuing warp of its own, so that
// they run out of step: one half's sums run under the other's products.
//
// 8192 x 8192 x 2048: 127 us = 2.2 PFLOP/s (one accumulator chain with a column's
// factor for each sum: 234 us); 64 experts, 32768 rows, 2048 x 1024: 94 us.  The
// tensor pipe is busy 54 %, the issue slots 46 %: each k block's hand-over
// (barrier, TMEM loads, 128 fp32 sums a thread, barrier) bounds it.  Two blocks
// to a tile of 256 rows measured the same on one large matrix and 8 % slower
// on 64 experts (more rows of a tile lie behind a group's end); sixteen epilogue
// warps of 64 sums a thread 10 % slower; scales through shared memory 14 % slower
// than from registers.
constexpr int kRowTile = 128, kFeatTile = 256, kRowStages = 3;
constexpr int kStoreBytes = 32 * 128;             // 32 rows of 64 features, as a box of the output's map
constexpr uint32_t kBlockBytes = 128 * kRowBytes;
// Registers: 3 warpgroups x 168 at launch; the two of the epilogue hold 128
// sums a thread and take over most of the third one's share.
constexpr int kLaunchRegs = 168, kFewRegs = 56, kManyRegs = 224;
static_assert(kFewRegs + 2 * kManyRegs == 3 * kLaunchRegs, "");

struct RowsCtl {
    unsigned char stage[kEpiWarps][2][kStoreBytes];      // first: on 1024 bytes
    unsigned long long full[kRowStages], empty[kRowStages];
    unsigned long long tfull[2][2], tempty[2][2], done[2];     // [half][buffer]
    uint32_t tmem;
    int fail;
    Groups groups;
};
constexpr size_t kRowsBytes = 1024 + size_t(kRowStages) * 3 * kBlockBytes + sizeof(RowsCtl);
static_assert(kRowsBytes <= 232448, "shared memory of one block");

struct RowTile {
    int group, row0, rows, feat0;
};

// Feature tiles of a row tile follow one another: they share the rows, and the
// weights of a layer stay in L2.
struct RowWalk {
    const Groups &g;
    const Params &p;
    int feat_tiles, total, tile, group;
    __device__ RowWalk(const Groups &g_, const Params &p_) : g(g_), p(p_) {
        feat_tiles = (p.lanes + kFeatTile - 1) / kFeatTile;
        total = g.first[p.E] * feat_tiles;
        tile = blockIdx.x;
        group = 0;
    }
    __device__ bool next(RowTile &t) {
        if (tile >= total) return false;
        while (tile >= g.first[group + 1] * feat_tiles) ++group;
        const int in = tile - g.first[group] * feat_tiles, r = in / feat_tiles;
        t.group = group;
        t.row0 = g.off[group] + r * kRowTile;
        t.rows = min(kRowTile, g.off[group + 1] - t.row0);
        t.feat0 = (in - r * feat_tiles) * kFeatTile;
        tile += gridDim.x;
        return true;
    }
};

template <typename OUT, int WHICH>
__global__ void __launch_bounds__(kThreads, 1)
fp8_rows_kernel(const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap tx,
                const __grid_constant__ CUtensorMap ty, const __grid_constant__ Params p) {
    constexpr bool W_MN = WHICH == kDgrad;
    constexpr int BK = kRowBytes, SLICES = 4;
    constexpr uint32_t W_STEP = W_MN ? BK / SLICES * kRowBytes : 32;

    extern __shared__ unsigned char raw[];
    unsigned char *buf = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    RowsCtl &ctl = *reinterpret_cast<RowsCtl *>(buf + size_t(kRowStages) * 3 * kBlockBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int *fail = &ctl.fail;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kRowStages; ++i) {
            bar_init(smem_u32(&ctl.full[i]), 1);
            bar_init(smem_u32(&ctl.empty[i]), 2);
        }
        for (int i = 0; i < 4; ++i) {
            bar_init(smem_u32(&ctl.tfull[i >> 1][i & 1]), 1);
            bar_init(smem_u32(&ctl.tempty[i >> 1][i & 1]), kEpiWarps / 2);
        }
        bar_init(smem_u32(&ctl.done[0]), 1);
        bar_init(smem_u32(&ctl.done[1]), 1);
        ctl.fail = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (blockIdx.x == 0 && p.status) *p.status = 0;   // a failure is a second away
    }
    if (threadIdx.x == 32) {
        prefetch_map(&tw);
        prefetch_map(&tx);
        prefetch_map(&ty);
    }
    if (warp == kMmaWarp) tmem_alloc(smem_u32(&ctl.tmem), 512);
    read_groups<kThreads>(ctl.groups, p);
    __syncthreads();
    if (warp == kTmaWarp) scan_groups<kRowTile>(ctl.groups, p, lane);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctl.tmem;
    const int nkb = (p.depth + BK - 1) / BK;
    RowWalk walk(ctl.groups, p);
    RowTile t;

    // (a warpgroup sets its registers in one place, and the two sides meet only
    // at the end: where branches meet, the compiler holds the code to the
    // smaller share)
    if (warp >= kEpiWarps) {
        regs_down<kFewRegs>();
        if (warp == kTmaWarp) {
            if (elect_one()) {
                uint32_t it = 0, ahead = 0;
                bool ok = true;
                auto load_w = [&](const RowTile &t, int kb, uint32_t s) {
                    const uint32_t bar = smem_u32(&ctl.full[s]), w = smem_u32(buf + s * 3 * kBlockBytes) + kBlockBytes;
                    const bool two = t.feat0 + 128 < p.lanes;
                    bar_expect(bar, (two ? 3 : 2) * kBlockBytes);
                    for (int h = 0; h < (two ? 2 : 1); ++h) {
                        if constexpr (W_MN) tma3(w + h * kBlockBytes, &tw, t.feat0 + h * 128, kb * BK, t.group, bar);
                        else tma3(w + h * kBlockBytes, &tw, kb * BK, t.feat0 + h * 128, t.group, bar);
                    }
                };
                const bool drop = p.drop && blockIdx.x == 0;      // test option: the first load is withheld
                if (p.dependent) {
                    // the weights do not come from the kernel before this one
                    RowWalk first = walk;
                    if (first.next(t))
                        for (; ahead < kRowStages && int(ahead) < nkb; ++ahead)
                            if (!drop || ahead) load_w(t, ahead, ahead);
                    wait_for_previous();
                }
                while (ok && walk.next(t)) {
                    for (int kb = 0; kb < nkb; ++kb, ++it) {
                        const uint32_t s = it % kRowStages;
                        if (it >= ahead) {
                            if (!bar_wait(smem_u32(&ctl.empty[s]), ((it / kRowStages) & 1) ^ 1, fail, p.status)) {
                                ok = false;
                                break;
                            }
                            if (!drop || it) load_w(t, kb, s);
                        }
                        if (drop && it == 0) continue;
                        tma2(smem_u32(buf + s * 3 * kBlockBytes), &tx, kb * BK, t.row0, smem_u32(&ctl.full[s]));
                    }
                }
                if (!ok) {
                    // copies in flight land before the block ends
                    volatile int never = 0;
                    for (uint32_t i = it > kRowStages ? it - kRowStages : 0; i < it; ++i)
                        if (!(drop && i == 0))
                            bar_wait(smem_u32(&ctl.full[i % kRowStages]), (i / kRowStages) & 1, &never, nullptr);
                }
            }
        } else if (warp <= kMmaWarp + 1) {
            // one issuing thread for each half of the features
            if (elect_one()) {
                const int half = warp - kMmaWarp;
                uint32_t it = 0, acc = 0;
                bool ok = true;
                while (ok && walk.next(t)) {
                    const int n = min(128, p.lanes - t.feat0 - half * 128);
                    const uint32_t idesc = instr_desc<kE4M3, false, W_MN>(n > 0 ? n : 16);
                    for (int kb = 0; kb < nkb; ++kb, ++it) {
                        const uint32_t s = it % kRowStages;
                        if (n > 0)
                            ok = bar_wait(smem_u32(&ctl.tempty[half][acc & 1]), ((acc >> 1) & 1) ^ 1, fail, p.status);
                        if (ok) ok = bar_wait(smem_u32(&ctl.full[s]), (it / kRowStages) & 1, fail, p.status);
                        if (!ok) break;
                        if (n > 0) {
                            tc_fence_after();
                            const uint32_t x = smem_u32(buf + s * 3 * kBlockBytes);
                            const uint64_t dx = operand_desc(x, 0), dw = operand_desc(x + (1 + half) * kBlockBytes, 0);
                            const uint32_t d = tmem + (half * 2 + (acc & 1)) * 128;
#pragma unroll
                            for (int j = 0; j < SLICES; ++j)
                                mma<kE4M3>(d, dx + ((j * 32) >> 4), dw + ((j * W_STEP) >> 4), idesc, j > 0 ? 1u : 0u);
                            mma_commit(smem_u32(&ctl.tfull[half][acc++ & 1]));
                            mma_commit(smem_u32(&ctl.empty[s]));
                        } else {
                            bar_arrive(smem_u32(&ctl.empty[s]));
                        }
                    }
                }
                // every matrix instruction has ended before the block frees its TMEM
                mma_commit(smem_u32(&ctl.done[half]));
                volatile int never = 0;
                bar_wait(smem_u32(&ctl.done[half]), 0, &never, nullptr);
            }
        }
    } else {
        regs_up<kManyRegs>();
        const int quad = warp & 3, half = warp >> 2;
        const uint32_t lanes_at = static_cast<uint32_t>(quad * 32) << 16;
        unsigned char *stage = ctl.stage[warp][0];
        uint32_t acc = 0;
        bool ok = true;
        if (p.dependent) wait_for_previous();
        bool more = walk.next(t);
        // scales of this thread's row and of the half's weight block, two k
        // blocks ahead; those of the next tile are on their way while this one
        // is stored
        const float *xs = p.xs, *ws = p.ws;
        long xs_step = 0, ws_step = 0;
        float x0 = 0.f, x1 = 0.f, w0 = 0.f, w1 = 0.f;
        auto begin = [&] {
            const int r = quad * 32 + lane, f = t.feat0 + half * 128;
            const bool real = r < t.rows && f < p.lanes;
            xs = p.xs + (real ? (t.row0 + r) * p.xs_row : 0);
            ws = p.ws + (real ? t.group * p.ws_group + (f >> 7) * p.ws_lane : 0);
            xs_step = real ? p.xs_blk : 0;
            ws_step = real ? p.ws_blk : 0;
            x0 = *xs;
            w0 = *ws;
            if (nkb > 1) {
                x1 = *(xs += xs_step);
                w1 = *(ws += ws_step);
            }
        };
        if (more) begin();
        while (more) {
            const int feats = min(128, p.lanes - t.feat0 - half * 128);
            const RowTile now = t;
            if (feats > 0) {
                float sum[4][32];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 32; ++j) sum[i][j] = 0.f;
                // one k block: its sums times f, the product of its two scales
                auto add_block = [&](float f) {
                    if (ok) ok = warp_wait(smem_u32(&ctl.tfull[half][acc & 1]), (acc >> 1) & 1, fail, p.status);
                    if (!ok) return;
                    tc_fence_after();
                    const uint32_t at = tmem + lanes_at + (half * 2 + (acc & 1)) * 128;
                    const float2 ff = make_float2(f, f);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        float v[16];
                        tmem_ld_row(v, at + i * 16);
                        tmem_wait_row(v);
                        if (i == 7) {
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) bar_arrive_tmem(smem_u32(&ctl.tempty[half][acc & 1]));
                        }
#pragma unroll
                        for (int j = 0; j < 16; j += 2) {
                            float *s = &sum[i >> 1][(i & 1) * 16 + j];
                            const float2 r = __ffma2_rn(make_float2(v[j], v[j + 1]), ff, make_float2(s[0], s[1]));
                            s[0] = r.x;
                            s[1] = r.y;
                        }
                    }
                };
                // (two at a time, so that a scale stays in its register from its
                // load to its use: a move in between waited for the load)
                for (int kb = 0; kb < nkb; kb += 2) {
                    const float f0 = x0 * w0;
                    if (kb + 2 < nkb) {
                        x0 = *(xs += xs_step);
                        w0 = *(ws += ws_step);
                    }
                    add_block(f0);
                    ++acc;
                    if (kb + 1 == nkb) break;
                    const float f1 = x1 * w1;
                    if (kb + 3 < nkb) {
                        x1 = *(xs += xs_step);
                        w1 = *(ws += ws_step);
                    }
                    add_block(f1);
                    ++acc;
                }
                more = walk.next(t);
                if (more) begin();
                // Each thread's row into shared memory, laid out as two boxes of
                // the output's map: a warp's 32 rows leave in two asynchronous
                // stores under the next tile's sums.  (All blocks store at about
                // the same time: vector stores held the epilogue up for 5600
                // clocks a tile, one bulk copy per row for 1500 to issue.)
                const int live = min(32, now.rows - quad * 32);       // rows that the group has
                const int row0 = now.row0 + quad * 32, feat0 = now.feat0 + half * 128;
                bulk_wait_read();
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float *v = &sum[i >> 2][(i & 3) * 8];
                    if (!ok) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = __int_as_float(0x7fffffff);
                    }
                    *reinterpret_cast<uint4 *>(stage + (i >> 3) * kStoreBytes + lane * 128 + ((i ^ lane) & 7) * 16) =
                        make_uint4(pack<OUT>(v[0], v[1]), pack<OUT>(v[2], v[3]), pack<OUT>(v[4], v[5]), pack<OUT>(v[6], v[7]));
                }
                if (live == 32) {
                    fence_async();
                    __syncwarp();
                    if (elect_one()) {
                        tma_store2(&ty, feat0, row0, smem_u32(stage));
                        if (feats > 64) tma_store2(&ty, feat0 + 64, row0, smem_u32(stage + kStoreBytes));
                        bulk_commit();
                    }
                } else {
                    // a group ends here: the rows behind it are another's
                    __syncwarp();
                    for (int i = lane; i < live * 16; i += 32) {
                        const int r = i >> 4, c = i & 15;
                        if (c * 8 < feats)
                            *reinterpret_cast<uint4 *>(static_cast<OUT *>(p.out) + (row0 + r) * p.ldo + feat0 + c * 8) =
                                *reinterpret_cast<const uint4 *>(stage + (c >> 3) * kStoreBytes + r * 128 + ((c ^ r) & 7) * 16);
                    }
                }
            } else {
                more = walk.next(t);
                if (more) begin();
            }
        }
        bulk_wait_all();
        zero_other_rows<OUT>(ctl.groups, p);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kMmaWarp) tmem_free(tmem, 512);
}

template <typename OUT, int WHICH>
cudaError_t launch_many(const Call &c) {
    using U = unsigned long long;
    CUtensorMap tw, tx, ty;
    int dev = 0;
    const int sms = grid_sms(&dev);
    if (sms <= 0) return cudaErrorInvalidDevice;
    const U wd[3] = {U(c.a_inner), U(c.a_rows), U(c.p.E)}, wst[2] = {U(c.a_inner), U(c.a_inner) * U(c.a_rows)};
    const U xd[2] = {U(c.b_inner), U(c.p.T)}, xst[1] = {U(c.ld_b)};
    const unsigned wb[3] = {128, 128, 1}, xb[2] = {128, unsigned(kRowTile)};
    if (!make_map(&tw, kE4M3, 3, c.a, wd, wst, wb) || !make_map(&tx, kE4M3, 2, c.b, xd, xst, xb)) return cudaErrorInvalidValue;
    const U yd[2] = {U(c.p.lanes), U(c.p.T)}, yst[1] = {U(c.p.ldo) * sizeof(OUT)};
    const unsigned yb[2] = {64, 32};
    if (!make_map(&ty, c.out_kind, 2, c.p.out, yd, yst, yb)) return cudaErrorInvalidValue;
    const auto k = &fp8_rows_kernel<OUT, WHICH>;
    static std::atomic<bool> ready[kMaxDevices];
    const cudaError_t e = set_up(k, kRowsBytes, kLaunchRegs, ready[dev]);
    if (e != cudaSuccess) return e;
    const long tiles = max_col_tiles<kRowTile>(c) * ((c.p.lanes + kFeatTile - 1) / kFeatTile);
    return launch_on(k, tiles < sms ? tiles : sms, kThreads, 1, kRowsBytes, c, tw, tx, ty, c.p);
}

template <typename OUT>
cudaError_t run_mm(const Call &c) {
    if (few_rows(c)) return c.which == kForward ? launch_few<kE4M3, OUT, kForward>(c) : launch_few<kE4M3, OUT, kDgrad>(c);
    return c.which == kForward ? launch_many<OUT, kForward>(c) : launch_many<OUT, kDgrad>(c);
}

template <typename OUT>
cudaError_t run_raw(const Call &c) {
    return c.which == kForward ? launch_few<kE4M3, OUT, kForward, true>(c) : launch_few<kE4M3, OUT, kDgrad, true>(c);
}

bool aligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
bool float_type(int d) { return d == BCJR_BF16 || d == BCJR_F16 || d == BCJR_F32; }
int status_of(cudaError_t e) {
    return e == cudaSuccess ? BCJR_OK : e == cudaErrorInvalidDevice ? BCJR_ERR_DEVICE : BCJR_ERR_LAUNCH;
}

}  // namespace
}  // namespace mm
}  // namespace bcjr

using namespace bcjr::mm;

extern "C" {

int bcjr_fp8_quantize_rows(const void *x, long ld, long rows, int k, int dtype, void *q,
                           float *scale, long scale_row, long scale_block, bcjr_stream_t stream) {
    if (rows < 0 || rows > kMaxRows || k < 16 || k % 16 || k > (1 << 24) || ld < k || scale_row < 0 ||
        scale_block < 0)
        return BCJR_ERR_BAD_SHAPE;
    if (!float_type(dtype)) return BCJR_ERR_UNSUPPORTED;
    if (rows == 0) return BCJR_OK;
    if (!x || !q || !scale) return BCJR_ERR_NULL_POINTER;
    if (!aligned(x, 16) || ld % (dtype == BCJR_F32 ? 4 : 8) || !aligned(q, 8) || !aligned(scale, 4))
        return BCJR_ERR_ALIGNMENT;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    switch (dtype) {
        case BCJR_BF16: return status_of(run_rows<__nv_bfloat16>(x, ld, rows, k, q, scale, scale_row, scale_block, st));
        case BCJR_F16: return status_of(run_rows<__half>(x, ld, rows, k, q, scale, scale_row, scale_block, st));
        default: return status_of(run_rows<float>(x, ld, rows, k, q, scale, scale_row, scale_block, st));
    }
}

int bcjr_fp8_quantize_blocks(const void *w, int E, int N, int K, int dtype, void *q, float *scale,
                             bcjr_stream_t stream) {
    if (E < 0 || N < 1 || N > (1 << 24) || K < 16 || K % 16 || K > (1 << 24)) return BCJR_ERR_BAD_SHAPE;
    if (!float_type(dtype)) return BCJR_ERR_UNSUPPORTED;
    const long blocks = long(E) * ((N + 127) / 128) * ((K + 127) / 128);
    if (blocks > 0x7fffffffL) return BCJR_ERR_BAD_SHAPE;
    if (E == 0) return BCJR_OK;
    if (!w || !q || !scale) return BCJR_ERR_NULL_POINTER;
    if (!aligned(w, 16) || !aligned(q, 8) || !aligned(scale, 4)) return BCJR_ERR_ALIGNMENT;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    switch (dtype) {
        case BCJR_BF16: return status_of(run_blocks<__nv_bfloat16>(w, blocks, N, K, q, scale, st));
        case BCJR_F16: return status_of(run_blocks<__half>(w, blocks, N, K, q, scale, st));
        default: return status_of(run_blocks<float>(w, blocks, N, K, q, scale, st));
    }
}

// How the rows of a product come: quantized; quantized by the kernel launched
// just before; in 16 bits, for the product to quantize.
enum { kReady = 0, kFollows = 1, kRaw = 2 };
static int check_mm(const void *rows, long ld_rows, const float *rows_scale, long scale_row,
                    long scale_block, const void *w, const float *w_scale, const void *offsets,
                    int offsets_bytes, long T, int E, int N, int K, int transpose_w, const void *out,
                    int out_dtype, const int *status, int come) {
    if (T < 0 || T > kMaxRows || E < 1 || E > kMaxGroups || N < 16 || K < 16 || N % 16 || K % 16 ||
        N > (1 << 24) || K > (1 << 24))
        return BCJR_ERR_BAD_SHAPE;
    if (out_dtype != BCJR_BF16 && out_dtype != BCJR_F16) return BCJR_ERR_UNSUPPORTED;
    if (offsets ? (offsets_bytes != 4 && offsets_bytes != 8) : E != 1) return BCJR_ERR_BAD_SHAPE;
    if (T == 0) return BCJR_OK;
    if (!rows || (!rows_scale && come != kRaw) || !w || !w_scale || !out) return BCJR_ERR_NULL_POINTER;
    const int depth = transpose_w ? N : K;
    if (ld_rows < depth || ld_rows > (1L << 32) || scale_row < 0 || scale_block < 0) return BCJR_ERR_BAD_SHAPE;
    if (!aligned(rows, 16) || ld_rows % (come == kRaw ? 8 : 16) || !aligned(w, 16) || !aligned(out, 16) || !aligned(status, 4) ||
        !aligned(rows_scale, 4) || !aligned(w_scale, 4) || (offsets && !aligned(offsets, size_t(offsets_bytes))))
        return BCJR_ERR_ALIGNMENT;
    return BCJR_OK;
}

static int fp8_mm(const void *rows, long ld_rows, const float *rows_scale, long scale_row,
                  long scale_block, const void *w, const float *w_scale, const void *offsets,
                  int offsets_bytes, long T, int E, int N, int K, int transpose_w, void *out,
                  int out_dtype, int *status, bcjr_stream_t stream, int come) {
    const int st = check_mm(rows, ld_rows, rows_scale, scale_row, scale_block, w, w_scale, offsets, offsets_bytes,
                            T, E, N, K, transpose_w, out, out_dtype, status, come);
    if (st || T == 0) return st;
    const int depth = transpose_w ? N : K, lanes = transpose_w ? K : N;
    const long kb = (K + 127) / 128, nb = (N + 127) / 128;
    Call c = {};
    c.kind = kE4M3;
    c.which = transpose_w ? kDgrad : kForward;
    c.a = w;
    c.a_rows = N;
    c.a_inner = K;
    if (come == kRaw) {
        c.p.raw = rows;
        c.p.ld_raw = ld_rows;
    } else {
        c.b = rows;
        c.ld_b = ld_rows;
        c.b_inner = depth;
    }
    c.stream = reinterpret_cast<cudaStream_t>(stream);
    c.p.offsets = offsets;
    c.p.offsets64 = offsets_bytes == 8;
    c.p.T = int(T);
    c.p.E = E;
    c.p.lanes = lanes;
    c.p.depth = depth;
    c.p.out = out;
    c.p.ldo = lanes;
    c.p.xs = rows_scale;
    c.p.xs_row = scale_row;
    c.p.xs_blk = scale_block;
    c.p.ws = w_scale;
    c.p.ws_group = nb * kb;
    c.p.ws_lane = transpose_w ? 1 : kb;
    c.p.ws_blk = transpose_w ? kb : 1;
    c.p.status = status;
    c.p.drop = bcjr::test_option(bcjr::kOptDropSends);
    c.p.dependent = come == kFollows;
    c.out_kind = out_dtype == BCJR_BF16 ? kBF16 : kF16;
    if (come == kRaw) return status_of(out_dtype == BCJR_BF16 ? run_raw<__nv_bfloat16>(c) : run_raw<__half>(c));
    return status_of(out_dtype == BCJR_BF16 ? run_mm<__nv_bfloat16>(c) : run_mm<__half>(c));
}

int bcjr_fp8_mm(const void *rows, long ld_rows, const float *rows_scale, long scale_row,
                long scale_block, const void *w, const float *w_scale, const void *offsets,
                int offsets_bytes, long T, int E, int N, int K, int transpose_w, void *out,
                int out_dtype, int *status, bcjr_stream_t stream) {
    return fp8_mm(rows, ld_rows, rows_scale, scale_row, scale_block, w, w_scale, offsets, offsets_bytes, T, E,
                  N, K, transpose_w, out, out_dtype, status, stream, kReady);
}

// The quantized rows first, then their scales, block by block, so that a tile
// reads those of its rows side by side.
size_t bcjr_fp8_linear_workspace_bytes(long T, int depth) {
    if (T < 0 || T > kMaxRows || depth < 16 || depth % 16 || depth > (1 << 24)) return 0;
    if (T <= kRawRows) return 16;
    return size_t(T) * depth + size_t(T) * ((depth + 127) / 128) * 4 + 16;
}

// Up to kRawRows rows one kernel quantizes and multiplies (one row, 8192 x 2048:
// 12.7 us a call with its host time, 17.5 as two kernels; 9.5 and 10.4 on the
// GPU).  With more the product is launched to overlap the end of the quantizer:
// its set-up and its first weight loads run before it waits for the quantized
// rows.  The quantizer itself is an ordinary launch, so everything before it has
// ended.
int bcjr_fp8_linear(const void *x, long ld, int dtype, const void *w, const float *w_scale,
                    const void *offsets, int offsets_bytes, long T, int E, int N, int K,
                    int transpose_w, void *out, void *ws, size_t ws_bytes, int *status,
                    bcjr_stream_t stream) {
    if (dtype != BCJR_BF16 && dtype != BCJR_F16) return BCJR_ERR_UNSUPPORTED;
    const int depth = transpose_w ? N : K;
    const size_t need = bcjr_fp8_linear_workspace_bytes(T, depth);
    if (!need) return BCJR_ERR_BAD_SHAPE;
    if (T <= kRawRows)
        return fp8_mm(x, ld, nullptr, 0, 0, w, w_scale, offsets, offsets_bytes, T, E, N, K, transpose_w, out,
                      dtype, status, stream, kRaw);
    if (!ws || ws_bytes < need) return BCJR_ERR_WORKSPACE;
    if (!aligned(ws, 16)) return BCJR_ERR_ALIGNMENT;
    float *scale = reinterpret_cast<float *>(static_cast<char *>(ws) + size_t(T) * depth);
    // nothing is launched for a call that the product will refuse
    int st = check_mm(ws, depth, scale, 1, T, w, w_scale, offsets, offsets_bytes, T, E, N, K, transpose_w, out,
                      dtype, status, kFollows);
    if (st) return st;
    st = bcjr_fp8_quantize_rows(x, ld, T, depth, dtype, ws, scale, 1, T, stream);
    if (st) return st;
    return fp8_mm(ws, depth, scale, 1, T, w, w_scale, offsets, offsets_bytes, T, E, N, K, transpose_w, out,
                  dtype, status, stream, kFollows);
}

}  // extern "C"
