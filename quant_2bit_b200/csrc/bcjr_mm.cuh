// Tensor-core matrix products for the linear layers around the quantizers
// (bcjr_grouped.cu: 16-bit types, bcjr_fp8.cu: e4m3 with block scales).
//
// One persistent kernel serves three products over row groups (experts) e
// with rows [off_e, off_{e+1}) of the row matrices:
//
//   forward  out[t, n]    = sum_k X[t, k]  W[e, n, k]     t in group e
//   dgrad    out[t, k]    = sum_n dY[t, n] W[e, n, k]
//   wgrad    out[e, n, k] = sum_{t in e} dY[t, n] X[t, k]
//
// All three put the features of the output's innermost axis on the 128 lanes
// of the accumulator and the other axis of the output on its columns:
//
//   D[lane, col] = sum_c A[lane, c] B[col, c]
//     forward  A = W[e] (K-major)     B = X  (K-major)    lane = n, col = t
//     dgrad    A = W[e]^T (MN-major)  B = dY (K-major)    lane = k, col = t
//     wgrad    A = X^T (MN-major)     B = dY^T (MN-major) lane = k, col = n
//
// so that the ragged token count is the N of the matrix instruction, which is
// any multiple of 16 up to 256 and is chosen per tile: one token and 256
// tokens run the same code, and a group of 300 rows costs 304 columns, not
// 3 x 128.
//
// Warp roles: one TMA producer, one issuer of matrix instructions, eight warps
// that empty the accumulators, two that fetch scales (e4m3) or zero the ragged
// ends (wgrad); accumulators and operand stages are rings between them, and
// the blocks are persistent, so loads, products and stores of neighbouring
// tiles overlap.
//
// Measured on a B200 (cold L2; 1.62 PFLOP/s is cuBLAS bf16 at the same size):
//   8192 x 8192 x 2048 bf16  forward 168 us = 1.64 PFLOP/s, gradients 180 us
//     each = 1.53; the tensor pipe is busy 86 and 78 % of the time: bound by it.
//   64 experts, 32768 rows, 1024 x 2048 bf16  113 us forward, 113 and 135 us:
//     ragged tiles, 0.47 GB of memory traffic a product (4.2 TB/s).  Back to
//     back for seconds 152, 153 and 167 us: power (1000 W at 1.18 GHz).
//   64 experts, 488 rows, 2048 x 1024 fp16  48 us = 5.6 TB/s of weights: bound
//     by memory.
//   8 rows by 8 of 64 experts, 1024 x 2048  14 us (34 MB): launch, set-up and
//     the first loads' latency are half of it.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "bcjr_e4m3.cuh"
#include "bcjr_kernels.h"
#include "bcjr_tiles.cuh"

#include <atomic>
#include <cstdint>

namespace bcjr {
namespace mm {

enum { kBF16 = 0, kF16 = 1, kE4M3 = 2 };          // element type of A and B
enum { kForward = 0, kDgrad = 1, kWgrad = 2 };    // which product
// Blocks to a tile: one; several that share its contraction (few rows); two
// that share its products (many rows).
enum { kAlone = 0, kSplit = 1, kPair = 2 };

constexpr int kLanes = 128;                       // M of the matrix instruction
constexpr int kRowBytes = 128;                    // one swizzled shared-memory row
constexpr int kEpiWarps = 8;
constexpr int kTmaWarp = 8, kMmaWarp = 9, kScaleWarp = 10;   // scales: two warps
constexpr int kThreads = 384;
constexpr int kChunk = 32;                        // columns that a half of the epilogue stores at once
constexpr int kPitch = kLanes * 2 + 16;           // bytes of a staged output row: 16-byte pieces of
                                                  // 8 rows fall into different banks
constexpr int kMaxGroups = 1024;
constexpr int kRawRows = 32;                      // rows that the e4m3 product quantizes itself
constexpr int kMaxSplit = 4;                      // blocks of a cluster that share a tile (eight: 37 rows x 2048 x
                                                  // 8192 in e4m3 16 -> 25 us, 64 rows x 2048 x 2048 14 -> 23)
constexpr int kBoxRows = 64;                      // rows of one TMA box
constexpr long long kWaitLimitClocks = 2000000000ll;   // about 1 s

struct Params {
    const void *offsets;      // E + 1 group bounds, or NULL: one group of all rows
    int offsets64;            // offsets are int64 (else int32)
    int T, E;                 // rows, groups
    int lanes, cols;          // extent of the lane axis; of the column axis (wgrad)
    int depth;                // extent of the contraction (forward, dgrad)
    void *out;
    long ldo;                 // elements between output rows (columns of D)
    long out_group;           // elements between groups of the output (wgrad)
    const void *raw;          // e4m3, quantized here: the rows, of the output's type,
    long ld_raw;              // and the elements between them
    const float *xs;          // e4m3: row scales, element (row, block) at row xs_row + block xs_blk
    long xs_row, xs_blk;
    const float *ws;          // e4m3: weight scales, (group, lane block, contraction block)
    long ws_group, ws_lane, ws_blk;
    int *status;
    int keep_status;          // a later kernel of one call: the word is not reset
    int drop;                 // test option: the first load of block 0 is withheld
    int dependent;            // launched to overlap the kernel that writes the row matrix
};

// ---------------------------------------------------------------------------
// PTX wrappers.

__device__ __forceinline__ uint32_t smem_u32(const void *p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
// True for one lane of a converged warp.  (Tensor-core and TMA instructions
// take their operands from uniform registers; under a branch that this
// instruction made the compiler knows that one lane runs them, under
// `lane == 0` it does not, and four matrix instructions took 770 clocks.)
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(one));
    return one != 0;
}
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// For accumulators that have been read (after tcgen05.fence::before_thread_sync,
// which orders the TMEM loads): nothing else has to be visible.
__device__ __forceinline__ void bar_arrive_tmem(uint32_t bar) {
    asm volatile("mbarrier.arrive.relaxed.cta.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;"
        " selp.u32 %0, 1, 0, p; }"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
// The same for a barrier that other blocks of the cluster arrive on.
__device__ __forceinline__ bool bar_try_cluster(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{ .reg .pred p; mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;"
        " selp.u32 %0, 1, 0, p; }"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
// Bounded wait (about 1 s).  False when it gave up or another warp of the
// block did; the block then finishes with NaN outputs and the status word
// says BCJR_ERR_TIMEOUT.
// `stages` of products, at well under 4096 clocks each, are waited for.
template <bool CLUSTER = false>
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int *fail,
                                         int *status, int stages = 0) {
    auto test = [&] { return CLUSTER ? bar_try_cluster(bar, parity) : bar_try(bar, parity); };
    if (test()) return true;
    const long long t0 = clock64();
    while (true) {
        for (int i = 0; i < 32; ++i)
            if (test()) return true;
        if (*fail) return false;
        if (clock64() - t0 > kWaitLimitClocks + 4096ll * stages) {
            *fail = 1;
            if (status) atomicExch(status, 8 /* BCJR_ERR_TIMEOUT */);
            return false;
        }
    }
}
// The same for a whole warp: every lane gets the same answer.  (All lanes
// test the barrier; one lane that tests and hands its answer around measured
// 5 % slower.)
template <bool CLUSTER = false>
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int *fail,
                                          int *status, int stages = 0) {
    return __all_sync(0xffffffffu, bar_wait<CLUSTER>(bar, parity, fail, status, stages));
}
__device__ __forceinline__ void tma2(uint32_t dst, const CUtensorMap *map, int x, int y,
                                     uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma3(uint32_t dst, const CUtensorMap *map, int x, int y, int z,
                                     uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
template <int KIND>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                    uint32_t accumulate) {
    if constexpr (KIND == kE4M3)
        asm volatile(
            "{ .reg .pred p; setp.ne.b32 p, %4, 0;"
            " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p; }"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{ .reg .pred p; setp.ne.b32 p, %4, 0;"
            " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
}
// The barrier gets one arrival when every matrix instruction issued so far by
// this thread has completed.
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];"
                 ::"r"(bar)
                 : "memory");
}
__device__ __forceinline__ void tmem_alloc(uint32_t dst, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(dst), "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols)
                 : "memory");
}
__device__ __forceinline__ void tc_fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// 16 lanes and 32 columns: v[4 j + i] of thread t is lane t / 4 + 8 (i / 2),
// column 8 j + 2 (t % 4) + i % 2.
__device__ __forceinline__ void tmem_ld(float (&v)[16], uint32_t addr) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
// The loaded registers may be used after this: it passes them through.
__device__ __forceinline__ void tmem_wait(float (&a)[16], float (&b)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(a[0]), "+f"(a[1]), "+f"(a[2]), "+f"(a[3]), "+f"(a[4]), "+f"(a[5]),
                   "+f"(a[6]), "+f"(a[7]), "+f"(a[8]), "+f"(a[9]), "+f"(a[10]), "+f"(a[11]),
                   "+f"(a[12]), "+f"(a[13]), "+f"(a[14]), "+f"(a[15])
                 :
                 : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) asm volatile("" : "+f"(b[i]));
}
// One lane and 16 columns per thread.
__device__ __forceinline__ void tmem_ld_row(float (&v)[16], uint32_t addr) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_wait_row(float (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) asm volatile("" : "+f"(v[i]));
}
// Four 8 x 8 blocks of 16-bit values, transposed on the way: thread t gives
// row t / 4, columns 2 (t % 4).. of each; the address of thread 8 m + c
// receives column c of block m.
__device__ __forceinline__ void st_transposed(uint32_t addr, uint32_t a, uint32_t b, uint32_t c,
                                              uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};"
                 ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d)
                 : "memory");
}
// Asynchronous store of a box of a tiled map, in a bulk group of this thread;
// what lies outside the map is not written.
__device__ __forceinline__ void tma_store2(const CUtensorMap *map, int x, int y, uint32_t src) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];"
                 ::"l"(map), "r"(x), "r"(y), "r"(src)
                 : "memory");
}
__device__ __forceinline__ void bulk_commit() {
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// This thread's stores have read their source; have been written.
__device__ __forceinline__ void bulk_wait_read() {
    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}
__device__ __forceinline__ void bulk_wait_all() {
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}
// Programmatic dependent launch: the next kernel of the stream may start; the
// one before has ended and its writes are visible.
__device__ __forceinline__ void let_next_start() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void wait_for_previous() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap *m) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
}
// 4 bytes global -> shared, or zero.
__device__ __forceinline__ void copy4(uint32_t dst, const float *src, bool real) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;"
                 ::"r"(dst), "l"(src), "r"(real ? 4 : 0)
                 : "memory");
}
// One arrival of this thread on `bar` when its copies so far have landed.
__device__ __forceinline__ void copy_arrive(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
// Pairs of blocks whose tensor cores work on one tile (cta_group::2): rank 0
// issues the matrix instructions, each block holds half of either operand and
// the sums of its half of the lanes.  A load of either block completes on a
// barrier of rank 0 (its address in the cluster is given); a commit arrives on
// the same barrier of both.
// (Relaxed: the thread has written nothing that others read, and a release at
// cluster scope for every stage took longer than the stage's products.)
__device__ __forceinline__ void pair_expect(uint32_t bar0, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.relaxed.cluster.shared::cluster.b64 _, [%0], %1;"
                 ::"r"(bar0), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void pair_tma2(uint32_t dst, const CUtensorMap *map, int x, int y,
                                          uint32_t bar0) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar0)
        : "memory");
}
__device__ __forceinline__ void pair_tma3(uint32_t dst, const CUtensorMap *map, int x, int y, int z,
                                          uint32_t bar0) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar0)
        : "memory");
}
// (16-bit types only: e4m3 has no pairs.)
__device__ __forceinline__ void pair_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                         uint32_t accumulate) {
    asm volatile(
        "{ .reg .pred p; setp.ne.b32 p, %4, 0;"
        " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p; }"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void pair_commit(uint32_t bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
        ::"r"(bar), "h"(static_cast<uint16_t>(3))
        : "memory");
}
template <bool PAIR> __device__ __forceinline__ void commit(uint32_t bar) {
    if constexpr (PAIR) pair_commit(bar);
    else mma_commit(bar);
}
__device__ __forceinline__ void pair_tmem_alloc(uint32_t dst, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(dst), "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void pair_tmem_free(uint32_t addr, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols)
                 : "memory");
}
// Thread block clusters: own rank, size, id; the address of `addr` in rank r.
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t in_rank(uint32_t addr, uint32_t r) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(r));
    return a;
}
__device__ __forceinline__ void bar_arrive_in(uint32_t bar, uint32_t r) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_rank(bar, r))
                 : "memory");
}
// For accumulators of the other block's products that have been read, as
// bar_arrive_tmem above.  (A release would wait for the output's stores as well:
// 64 experts of 512 rows forward 113 -> 115 us, weights' gradient 135 -> 147.)
__device__ __forceinline__ void bar_arrive_relaxed_in(uint32_t bar, uint32_t r) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_rank(bar, r))
                 : "memory");
}
__device__ __forceinline__ float2 load2_in(uint32_t addr, uint32_t r) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(in_rank(addr, r)));
    return v;
}
__device__ __forceinline__ void fence_async() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
// Registers of this warpgroup from here on.
template <int N> __device__ __forceinline__ void regs_down() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N> __device__ __forceinline__ void regs_up() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
// The 128 threads of one half of the epilogue.
__device__ __forceinline__ void half_sync(int half) {
    asm volatile("bar.sync %0, 128;" ::"r"(half + 1) : "memory");
}

// Shared-memory operand descriptor, 128-byte swizzle.  K-major: rows of the
// M or N axis are 128-byte shared-memory rows, 8-row groups 1024 bytes apart.
// MN-major: 128 bytes of the M or N axis are contiguous, one such row per
// step of the contraction, 8-step groups 1024 bytes apart, and the next 128
// bytes of the M or N axis `mn_stride` bytes further.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, uint32_t mn_stride) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((addr & 0x3ffff) >> 4);
    d |= static_cast<uint64_t>((mn_stride & 0x3ffff) >> 4) << 16;
    d |= static_cast<uint64_t>(1024 >> 4) << 32;
    d |= 1ull << 46;
    d |= 2ull << 61;
    return d;
}

template <int KIND, bool A_MN, bool B_MN, int M = kLanes>
__device__ __forceinline__ uint32_t instr_desc(int n) {
    const uint32_t fmt = KIND == kBF16 ? 1u : 0u;   // f16 0, bf16 1; e4m3 0
    return (1u << 4) | (fmt << 7) | (fmt << 10) | (A_MN ? 1u << 15 : 0u) |
           (B_MN ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
           (static_cast<uint32_t>(M >> 4) << 24);
}

// ---------------------------------------------------------------------------
// Groups and tiles.

// Group bounds as the kernel uses them: within [0, T] and not decreasing,
// whatever the caller's memory holds, so no access can leave the matrices.
// first[e] is the number of column tiles before group e (forward, dgrad).
struct Groups {
    int off[kMaxGroups + 1];
    int first[kMaxGroups + 1];
};

// Two steps: the whole block reads the bounds, then (after a block barrier)
// one warp makes them monotone and counts tiles.
template <int THREADS>
__device__ __forceinline__ void read_groups(Groups &g, const Params &p) {
    for (int e = threadIdx.x; e <= p.E; e += THREADS) {
        long long v;
        if (!p.offsets) v = e == 0 ? 0 : p.T;
        else if (p.offsets64) v = static_cast<const long long *>(p.offsets)[e];
        else v = static_cast<const int *>(p.offsets)[e];
        g.off[e] = v < 0 ? 0 : v > p.T ? p.T : static_cast<int>(v);
    }
}
// Every lane has a run of neighbouring bounds, so one pass over the warp joins
// them (lane by lane, a layer of 64 experts took three).
template <int COLS>
__device__ __forceinline__ void scan_groups(Groups &g, const Params &p, int lane) {
    const int run = (p.E + 32) / 32, lo = lane * run, hi = min(lo + run, p.E + 1);
    int top = 0;
    for (int e = lo; e < hi; ++e) top = max(top, g.off[e]);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, top, d);
        if (lane >= d) top = max(top, u);
    }
    int before = __shfl_up_sync(0xffffffffu, top, 1);     // the largest bound of the lanes before
    if (lane == 0) before = 0;
    int o = before, tiles = 0;
    for (int e = lo; e < hi; ++e) {
        const int next = max(o, g.off[e]);
        // tiles of group e - 1, which ends at this bound
        if (e > 0) tiles += col_tiles<COLS>(next - o);
        g.off[e] = o = next;
        g.first[e] = tiles;
    }
    int sum = tiles;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += u;
    }
    for (int e = lo; e < hi; ++e) g.first[e] += sum - tiles;
}

struct Tile {
    int group;
    int lane_tile;
    int col0;       // first output row (forward, dgrad: row of X; wgrad: n)
    int valid;      // columns to write
    int ncols;      // columns computed, a multiple of 16 (of 32 by a pair)
    int k0;         // first contraction index (wgrad: row of X)
    int depth;      // contraction length from k0 on
    int nkb;        // its stages (0: the output is zero)
};

// The tiles of a block, one after the other; every warp walks the same list.
// kSplit: the blocks of a cluster share each tile, every one with its part of
// the contraction.  kPair: two blocks have the halves of 256 lanes.
template <int WHICH, int COLS, int BK, int MODE>
struct Walk {
    static constexpr bool SPLIT = MODE == kSplit;
    static constexpr int LANES = MODE == kPair ? 2 * kLanes : kLanes;
    static constexpr int STEP = MODE == kPair ? 32 : 16;     // of the columns' number
    const Groups &g;
    const Params &p;
    int lane_tiles, total, tile, step, group, part, parts;
    __device__ Walk(const Groups &g_, const Params &p_) : g(g_), p(p_) {
        parts = SPLIT ? cluster_size() : 1;
        part = SPLIT ? cluster_rank() : 0;
        const int blocks = MODE == kPair ? 2 : parts;
        step = gridDim.x / blocks;
        lane_tiles = (p.lanes + LANES - 1) / LANES;
        total = WHICH == kWgrad ? p.E * lane_tiles * col_tiles<COLS>(p.cols)
                                : g.first[p.E] * lane_tiles;
        tile = blockIdx.x / blocks;
        group = 0;
    }
    // Column and lane tile of a group's tile `in`: bands of 2048 lanes, column
    // by column within a band.  The blocks at work then share a part of either
    // operand that L2 holds.  (Lane tile by lane tile, the gradients of 8192 x
    // 8192 x 2048 read 578 MB from memory for 200 MB of operands.)
    __device__ int place(int in, int ct, int &lane_tile) const {
        constexpr int BAND = 2048 / LANES;
        const int band = in / (BAND * ct), at = in - band * BAND * ct;
        const int height = min(BAND, lane_tiles - band * BAND), c = at / height;
        lane_tile = band * BAND + at - c * height;
        return c;
    }
    __device__ bool next(Tile &t) {
        if (tile >= total) return false;
        if constexpr (WHICH == kWgrad) {
            const int ct = col_tiles<COLS>(p.cols), per = lane_tiles * ct;
            t.group = tile / per;
            const int in = tile - t.group * per;
            t.col0 = place(in, ct, t.lane_tile) * COLS;
            t.valid = min(COLS, p.cols - t.col0);
            t.ncols = (t.valid + STEP - 1) & ~(STEP - 1);
            t.k0 = g.off[t.group];
            t.depth = g.off[t.group + 1] - t.k0;
            t.nkb = (t.depth + BK - 1) / BK;
        } else {
            while (tile >= g.first[group + 1] * lane_tiles) ++group;
            const int in = tile - g.first[group] * lane_tiles;
            const int ct = g.first[group + 1] - g.first[group];
            t.group = group;
            const int c = place(in, ct, t.lane_tile);
            const int rows = g.off[group + 1] - g.off[group];
            const int share = tile_share(rows, ct, STEP);
            t.col0 = g.off[group] + c * share;
            t.valid = min(share, g.off[group + 1] - t.col0);
            t.ncols = (t.valid + STEP - 1) & ~(STEP - 1);
            const int nkb = (p.depth + BK - 1) / BK;
            const int kb0 = SPLIT ? nkb * part / parts : 0;
            t.nkb = (SPLIT ? nkb * (part + 1) / parts : nkb) - kb0;
            t.k0 = kb0 * BK;
            t.depth = p.depth - t.k0;
        }
        tile += step;
        return true;
    }
};

template <typename T> __device__ __forceinline__ uint32_t pack(float a, float b);
template <> __device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <> __device__ __forceinline__ uint32_t pack<__half>(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}

// Rows of no group (before the first, behind the last) are zero: all threads
// of all epilogues.
template <typename OUT>
__device__ __forceinline__ void zero_other_rows(const Groups &g, const Params &p) {
    const int lo = g.off[0], hi = g.off[p.E];
    const long rows = static_cast<long>(lo) + (p.T - hi);
    for (long r = blockIdx.x; r < rows; r += gridDim.x) {
        uint4 *o = reinterpret_cast<uint4 *>(static_cast<OUT *>(p.out) + (r < lo ? r : r - lo + hi) * p.ldo);
        for (int f = threadIdx.x; f < p.lanes / 8; f += kEpiWarps * 32) o[f] = make_uint4(0, 0, 0, 0);
    }
}

constexpr int kScaleStages = 8;
constexpr int kPartPitch = kLanes + 4;            // floats: no bank conflicts either way


template <int KIND, int COLS, int STAGES, int MODE>
struct Smem {
    static constexpr bool SPLIT = MODE == kSplit;
    static constexpr int kA = kLanes * kRowBytes;
    static constexpr int kB = COLS * kRowBytes / (MODE == kPair ? 2 : 1);
    static constexpr int kStage = kA + kB;
    static constexpr int kScales = KIND == kE4M3 ? kScaleStages : 1;
    // accumulator buffers.  16-bit types use one for a tile, e4m3 one for a k
    // block: eight of them, so that the tensor core runs ahead of the epilogue
    // (one token, 8192 x 2048: 740 clocks a block with two, 630 with eight).
    static constexpr int kAcc = KIND == kE4M3 ? 8 : 2;
    struct Ctl {
        unsigned long long full[STAGES], empty[STAGES], zeroed[STAGES], ragged[STAGES], tfull[kAcc], tempty[kAcc], done;
        unsigned long long sfull[kScaleStages], sempty[kScaleStages];
        uint32_t tmem;
        int fail;
        alignas(16) float xs[kScales][COLS];      // e4m3: scales of the tile's rows, and
        float ws[kScales];                        // of its weight block, one slot per k block
        alignas(16) unsigned char stage[2][SPLIT ? 16 : kChunk * kPitch];
        unsigned long long pfull;                 // a split tile's sums: written by all blocks;
        alignas(16) float part[SPLIT ? COLS : 1][kPartPitch];     // this block's
        Groups groups;
    };
    static constexpr size_t bytes() { return 1024 + size_t(STAGES) * kStage + sizeof(Ctl); }
};

// 32 columns of the tile from one half of the epilogue: v[h] holds lanes
// 16 h.. of this warp's 32.  Packed and transposed into rows of 128 features
// in shared memory, and from there to the rows that the output has, 256
// contiguous bytes for half a warp.  (One bulk copy for each row in place of
// the vector stores took 22 clocks a row: 268 MB of weight gradients left at
// 3.2 TB/s.)
template <typename OUT>
__device__ __forceinline__ void store_chunk(const float (&v)[2][16], unsigned char *stage, int half,
                                            int quad, int lane, OUT *out, long ldo, int c0,
                                            int valid, int features) {
    half_sync(half);               // the last chunk has been read
    const uint32_t base = smem_u32(stage) + (lane & 7) * kPitch + quad * 64 + (lane >> 3) * 16;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        st_transposed(base + j * 8 * kPitch, pack<OUT>(v[0][4 * j], v[0][4 * j + 1]),
                      pack<OUT>(v[0][4 * j + 2], v[0][4 * j + 3]),
                      pack<OUT>(v[1][4 * j], v[1][4 * j + 1]),
                      pack<OUT>(v[1][4 * j + 2], v[1][4 * j + 3]));
    half_sync(half);
    const int piece = lane & 15;
    if (piece * 8 < features) {
#pragma unroll
        for (int i = 0; i < kChunk / 8; ++i) {
            const int c = i * 8 + quad * 2 + (lane >> 4);
            if (c0 + c < valid)
                *reinterpret_cast<uint4 *>(out + static_cast<long>(c0 + c) * ldo + piece * 8) =
                    *reinterpret_cast<const uint4 *>(stage + c * kPitch + piece * 16);
        }
    }
}

// A tile whose contraction is split over the blocks of a cluster: every block
// leaves its fp32 sums in its shared memory, and block r adds those of all
// blocks, in the order of their ranks, for features r * 128 / size .. and
// writes them.  (A cluster has one tile: the launch gives every tile a cluster
// of its own, and nobody overwrites the sums.)  A block that failed leaves NaN.
template <typename OUT>
__device__ __forceinline__ bool add_parts(const float (&v)[2][16], float (*part)[kPartPitch],
                                          uint32_t pfull, int half, int quad, int lane,
                                          OUT *out, long ldo, int valid,
                                          int features, bool ok, volatile int *fail, int *status) {
    const uint32_t size = cluster_size(), rank = cluster_rank();
    const int f0 = quad * 32 + (lane >> 2), c0 = half * kChunk + 2 * (lane & 3);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (c0 + 8 * j + (q & 1) < valid)
                    part[c0 + 8 * j + (q & 1)][f0 + 16 * h + 8 * (q >> 1)] =
                        ok ? v[h][4 * j + q] : __int_as_float(0x7fffffff);
    __syncwarp();
    if (lane < size) bar_arrive_in(pfull, lane);
    if (ok) ok = warp_wait<true>(pfull, 0, fail, status);
    const int per = kLanes / 2 / size;              // feature pairs of this block
    for (int i = threadIdx.x; i < valid * per; i += kEpiWarps * 32) {
        const int c = i / per, f = (rank * per + i - c * per) * 2;
        if (f >= features) continue;
        const uint32_t at = smem_u32(&part[c][f]);
        float2 w[kMaxSplit];                        // all on their way before the first is added
#pragma unroll
        for (uint32_t r = 0; r < kMaxSplit; ++r)
            if (r < size) w[r] = load2_in(at, r);
        float2 s = w[0];
#pragma unroll
        for (uint32_t r = 1; r < kMaxSplit; ++r)
            if (r < size) {
                s.x += w[r].x;
                s.y += w[r].y;
            }
        if (!ok) s.x = s.y = __int_as_float(0x7fffffff);
        *reinterpret_cast<uint32_t *>(out + c * ldo + f) = pack<OUT>(s.x, s.y);
    }
    return ok;
}

// KIND: element type; OUT: output type; WHICH: product; COLS: columns of a
// tile; STAGES: depth of the shared-memory ring; MODE: blocks to a tile; RAW: the
// rows are 16-bit and the kernel quantizes them (e4m3, at most kRawRows).
template <int KIND, typename OUT, int WHICH, int COLS, int STAGES, int MODE, bool RAW>
__global__ void __launch_bounds__(kThreads, 1)
mm_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb,
          const __grid_constant__ Params p) {
    constexpr bool SPLIT = MODE == kSplit, PAIR = MODE == kPair;
    constexpr bool A_MN = WHICH != kForward, B_MN = WHICH == kWgrad;
    constexpr int ESIZE = KIND == kE4M3 ? 1 : 2;
    constexpr int BK = kRowBytes / ESIZE;             // contraction per stage
    constexpr int MNB = kRowBytes / ESIZE;            // M or N elements of one MN-major row
    constexpr int SLICES = 4;                         // matrix instructions per stage
    constexpr int KSLICE = BK / SLICES;
    // bytes from one slice to the next
    constexpr uint32_t A_STEP = A_MN ? KSLICE * kRowBytes : 32;
    constexpr uint32_t B_STEP = B_MN ? KSLICE * kRowBytes : 32;
    constexpr uint32_t MN_BLOCK = BK * kRowBytes;     // an MN-major block of BK rows
    using S = Smem<KIND, COLS, STAGES, MODE>;
    constexpr uint32_t ACC = S::kAcc, TMEM_COLS = ACC * COLS;
    static_assert(TMEM_COLS <= 512 && (TMEM_COLS & (TMEM_COLS - 1)) == 0 && TMEM_COLS >= 32, "");
    static_assert(KIND != kE4M3 || (WHICH != kWgrad && COLS == 64), "e4m3: few rows, forward and dgrad");
    static_assert(BK % kBoxRows == 0 && COLS % 32 == 0, "");
    static_assert(!PAIR || KIND != kE4M3, "pairs: 16-bit types");
    static_assert(!RAW || KIND == kE4M3, "");

    extern __shared__ unsigned char raw[];
    unsigned char *buf = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    typename S::Ctl &ctl = *reinterpret_cast<typename S::Ctl *>(buf + size_t(STAGES) * S::kStage);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? cluster_rank() : 0;
    volatile int *fail = &ctl.fail;

    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) {
            // full: the loads, and with RAW the warp that quantizes.  A pair's
            // rank 0 is told by both blocks: by their loads, or by the warps that
            // zero the end of a group (which the loads tell first, on `ragged`).
            bar_init(smem_u32(&ctl.full[i]), RAW || PAIR ? 2 : 1);
            bar_init(smem_u32(&ctl.empty[i]), B_MN && !PAIR ? 2 : 1);
            bar_init(smem_u32(&ctl.zeroed[i]), 1);
            bar_init(smem_u32(&ctl.ragged[i]), 1);
        }
        for (int i = 0; i < ACC; ++i) {
            bar_init(smem_u32(&ctl.tfull[i]), 1);
            bar_init(smem_u32(&ctl.tempty[i]), PAIR ? 2 * kEpiWarps : kEpiWarps);
        }
        bar_init(smem_u32(&ctl.done), 1);
        if constexpr (SPLIT) bar_init(smem_u32(&ctl.pfull), kEpiWarps * cluster_size());
        for (int i = 0; i < kScaleStages; ++i) {
            bar_init(smem_u32(&ctl.sfull[i]), RAW ? 1 : 64);
            bar_init(smem_u32(&ctl.sempty[i]), kEpiWarps);
        }
        ctl.fail = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (blockIdx.x == 0 && p.status && !p.keep_status) *p.status = 0;   // a failure is a second away
    }
    if (threadIdx.x == 32) {
        prefetch_map(&ta);
        prefetch_map(&tb);
    }
    if (warp == kMmaWarp) {
        if constexpr (PAIR) pair_tmem_alloc(smem_u32(&ctl.tmem), TMEM_COLS);
        else tmem_alloc(smem_u32(&ctl.tmem), TMEM_COLS);
    }
    read_groups<kThreads>(ctl.groups, p);
    __syncthreads();
    if (warp == kTmaWarp) scan_groups<COLS>(ctl.groups, p, lane);
    tc_fence_before();
    if constexpr (MODE != kAlone) cluster_sync();
    else __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctl.tmem;
    Walk<WHICH, COLS, BK, MODE> walk(ctl.groups, p);
    Tile t;

    if (warp >= kEpiWarps) {
        if (warp == kTmaWarp) {
            // TMA producer
            if (elect_one()) {
                uint32_t it = 0, ahead = 0;
                bool ok = true;
                // This block's part of the lanes and of the columns, and the
                // barrier that its loads complete on.
                auto lanes_at = [&](const Tile &t) { return t.lane_tile * walk.LANES + int(rank) * kLanes; };
                auto cols = [&](const Tile &t) { return PAIR ? t.ncols / 2 : t.ncols; };
                auto full = [&](uint32_t s) {
                    const uint32_t bar = smem_u32(&ctl.full[s]);
                    return PAIR ? in_rank(bar, 0) : bar;
                };
                // Arms the stage's barrier for both operands and loads the one
                // that has the output's lanes.
                auto load_a = [&](const Tile &t, int kb, uint32_t s) {
                    const uint32_t bar = full(s), a = smem_u32(buf + s * S::kStage);
                    const int boxes = (cols(t) + (B_MN ? MNB : kBoxRows) - 1) / (B_MN ? MNB : kBoxRows);
                    const int kc = t.k0 + kb * BK;
                    const uint32_t bytes = S::kA + (RAW ? 0 : boxes * (B_MN ? MN_BLOCK : kBoxRows * kRowBytes));
                    if constexpr (PAIR) pair_expect(bar, bytes);
                    else bar_expect(bar, bytes);
                    if constexpr (WHICH == kForward) {
                        if constexpr (PAIR) pair_tma3(a, &ta, kc, lanes_at(t), t.group, bar);
                        else tma3(a, &ta, kc, lanes_at(t), t.group, bar);
                    } else {
#pragma unroll
                        for (int j = 0; j < kLanes / MNB; ++j) {
                            const int x = lanes_at(t) + j * MNB;
                            if constexpr (PAIR && B_MN) pair_tma2(a + j * MN_BLOCK, &ta, x, kc, bar);
                            else if constexpr (B_MN) tma2(a + j * MN_BLOCK, &ta, x, kc, bar);
                            else if constexpr (PAIR) pair_tma3(a + j * MN_BLOCK, &ta, x, kc, t.group, bar);
                            else tma3(a + j * MN_BLOCK, &ta, x, kc, t.group, bar);
                        }
                    }
                };
                // The end of a group in a pair's weights' gradient: both operands,
                // complete on a barrier of this block, for the warp that zeroes.
                // `own` has a bit for every stage whose last load was such an
                // end, `turn` the phase of its next one.
                uint32_t own = 0, turn = 0;
                auto load_end = [&](const Tile &t, int kb, uint32_t s) {
                    const uint32_t bar = smem_u32(&ctl.ragged[s]), a = smem_u32(buf + s * S::kStage);
                    const int kc = t.k0 + kb * BK, n = cols(t), c = t.col0 + int(rank) * n;
                    bar_expect(bar, S::kA + (n + MNB - 1) / MNB * MN_BLOCK);
                    for (int j = 0; j < kLanes / MNB; ++j) tma2(a + j * MN_BLOCK, &ta, lanes_at(t) + j * MNB, kc, bar);
                    for (int j = 0; j * MNB < n; ++j) tma2(a + S::kA + j * MN_BLOCK, &tb, c + j * MNB, kc, bar);
                    own |= 1u << s;
                    turn ^= 1u << s;
                };
                const bool drop = p.drop && blockIdx.x == 0;      // test option: the first load is withheld
                if (p.dependent) {
                    // the weights do not come from the kernel before this one
                    Walk<WHICH, COLS, BK, MODE> first = walk;
                    if (first.next(t))
                        for (; ahead < STAGES && ahead < t.nkb; ++ahead)
                            if (!drop || ahead) load_a(t, ahead, ahead);
                    wait_for_previous();
                }
                while (ok && walk.next(t)) {
                    for (int kb = 0; kb < t.nkb; ++kb, ++it) {
                        const uint32_t s = it % STAGES;
                        if (it >= ahead) {
                            if (!bar_wait(smem_u32(&ctl.empty[s]), ((it / STAGES) & 1) ^ 1, fail, p.status)) {
                                ok = false;
                                break;
                            }
                            if (PAIR && B_MN && t.depth - kb * BK < BK) {
                                if (!drop || it) load_end(t, kb, s);
                                continue;
                            }
                            own &= ~(1u << s);
                            if (!drop || it) load_a(t, kb, s);
                        }
                        if (RAW || (drop && it == 0)) continue;
                        const uint32_t bar = full(s), b = smem_u32(buf + s * S::kStage) + S::kA;
                        const int kc = t.k0 + kb * BK, n = cols(t), c = t.col0 + int(rank) * n;
                        if constexpr (B_MN) {
                            for (int j = 0; j * MNB < n; ++j) {
                                if constexpr (PAIR) pair_tma2(b + j * MN_BLOCK, &tb, c + j * MNB, kc, bar);
                                else tma2(b + j * MN_BLOCK, &tb, c + j * MNB, kc, bar);
                            }
                        } else {
                            for (int j = 0; j * kBoxRows < n; ++j) {
                                if constexpr (PAIR) pair_tma2(b + j * kBoxRows * kRowBytes, &tb, kc, c + j * kBoxRows, bar);
                                else tma2(b + j * kBoxRows * kRowBytes, &tb, kc, c + j * kBoxRows, bar);
                            }
                        }
                    }
                }
                if (!ok) {
                    // copies in flight land before the block (the pair) ends:
                    // rank 0 knows of the loads that complete on its barriers
                    volatile int never = 0;
                    for (uint32_t i = it > STAGES ? it - STAGES : 0; i < it; ++i) {
                        const uint32_t s = i % STAGES;
                        if (drop && i == 0) continue;
                        if (own >> s & 1) bar_wait(smem_u32(&ctl.ragged[s]), (turn >> s & 1) ^ 1, &never, nullptr);
                        else if (rank == 0) bar_wait<PAIR>(smem_u32(&ctl.full[s]), (i / STAGES) & 1, &never, nullptr);
                    }
                }
            }
        } else if (warp == kMmaWarp && rank == 0) {
            // MMA issuer: one thread runs the whole loop (a warp that elected a
            // thread and met again for every stage took 220 clocks more for it)
            if (elect_one()) {
                uint32_t it = 0, acc = 0;
                bool ok = true;
                while (ok && walk.next(t)) {
                    if (t.nkb == 0) continue;
                    const uint32_t idesc = instr_desc<KIND, A_MN, B_MN, decltype(walk)::LANES>(t.ncols);
                    for (int kb = 0; kb < t.nkb; ++kb, ++it) {
                        const uint32_t s = it % STAGES;
                        // e4m3: every stage has an accumulator buffer of its own
                        // (scaled and added in fp32 registers); otherwise every tile
                        if (KIND == kE4M3 || kb == 0)
                            ok = bar_wait<PAIR>(smem_u32(&ctl.tempty[acc % ACC]), ((acc / ACC) & 1) ^ 1, fail, p.status);
                        if (ok)
                            ok = bar_wait<PAIR>(smem_u32(B_MN && !PAIR && t.depth - kb * BK < BK ? &ctl.zeroed[s] : &ctl.full[s]),
                                                (it / STAGES) & 1, fail, p.status);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t a = smem_u32(buf + s * S::kStage);
                        const uint64_t da = operand_desc(a, MN_BLOCK), db = operand_desc(a + S::kA, MN_BLOCK);
                        const uint32_t d = tmem + (acc % ACC) * COLS;
#pragma unroll
                        for (int j = 0; j < SLICES; ++j) {
                            const uint64_t aj = da + ((j * A_STEP) >> 4), bj = db + ((j * B_STEP) >> 4);
                            const uint32_t add = (KIND == kE4M3 ? j > 0 : (kb | j) > 0) ? 1u : 0u;
                            if constexpr (PAIR) pair_mma(d, aj, bj, idesc, add);
                            else mma<KIND>(d, aj, bj, idesc, add);
                        }
                        if (KIND == kE4M3 || kb == t.nkb - 1) commit<PAIR>(smem_u32(&ctl.tfull[acc++ % ACC]));
                        commit<PAIR>(smem_u32(&ctl.empty[s]));
                    }
                }
                // every matrix instruction has ended before the block frees its TMEM
                commit<PAIR>(smem_u32(&ctl.done));
                volatile int never = 0;
                bar_wait(smem_u32(&ctl.done), 0, &never, nullptr);
            }
        } else if constexpr (WHICH == kWgrad) {
            // The rows of a group's last stage that belong to the next group (or
            // lie behind the last one) do not count, whatever they hold: one
            // warp makes them zero in both factors before they are multiplied.
            auto zero_end = [&](uint32_t s, int rows, int n) {
                unsigned char *a = buf + s * S::kStage;
                const int cells = (BK - rows) * (kRowBytes / 16);
                const int blocks = kLanes / MNB + (n + MNB - 1) / MNB;
                for (int j = 0; j < blocks; ++j) {
                    uint4 *z = reinterpret_cast<uint4 *>(a + j * MN_BLOCK + rows * kRowBytes);
                    for (int i = lane; i < cells; i += 32) z[i] = make_uint4(0, 0, 0, 0);
                }
                fence_async();
                __syncwarp();
            };
            uint32_t it = 0;
            bool ok = warp == kScaleWarp;
            if constexpr (PAIR) {
                // Both blocks' warps tell rank 0 of a group's last stage, with a
                // release: the zeros and the loads that the warp saw are there.
                // All other stages' loads complete on rank 0's barrier by
                // themselves: a warp that handed those on as well would need
                // such a release for every stage (a relaxed arrival orders no
                // load before rank 0's products), which takes longer than the
                // stage's products.  A wait may last as long as the tiles since
                // the last one, with 32 stages' time for each one's stores.
                uint32_t turn = 0;                  // phase of each stage's `ragged`
                int passed = 0;
                while (ok && walk.next(t)) {
                    it += t.nkb;
                    passed += t.nkb + 32;
                    const int rows = t.depth - (t.nkb - 1) * BK;
                    if (t.nkb == 0 || rows == BK) continue;
                    const uint32_t s = (it - 1) % STAGES;
                    ok = warp_wait(smem_u32(&ctl.ragged[s]), turn >> s & 1, fail, p.status, passed);
                    if (!ok) break;
                    turn ^= 1u << s;
                    passed = 0;
                    zero_end(s, rows, t.ncols / 2);
                    if (lane == 0) bar_arrive_in(smem_u32(&ctl.full[s]), 0);
                }
            } else {
                // It follows every stage, and a stage is loaded again only after
                // it, so that nobody mistakes a barrier's phase.
                while (ok && walk.next(t)) {
                    for (int kb = 0; kb < t.nkb; ++kb, ++it) {
                        const uint32_t s = it % STAGES;
                        ok = warp_wait(smem_u32(&ctl.full[s]), (it / STAGES) & 1, fail, p.status);
                        if (!ok) break;
                        const int rows = t.depth - kb * BK;
                        if (rows < BK) zero_end(s, rows, t.ncols);
                        if (lane == 0) {
                            bar_arrive(smem_u32(&ctl.zeroed[s]));
                            bar_arrive(smem_u32(&ctl.empty[s]));
                        }
                    }
                }
            }
        } else if constexpr (RAW) {
            // The rows of a k block, quantized into the stage by one of two warps
            // in turn: half a warp per row, 8 elements a lane, loaded two k blocks
            // ahead.  Every block does its own (a few KB of rows for 16 KB of
            // weights a stage); a kernel of their own would cost a launch and its
            // workspace.
            constexpr int PASSES = kRawRows / 2;
            const int odd = warp - kScaleWarp, sub = lane & 15, first = lane >> 4;
            uint32_t it0 = 0;                       // stages of the tiles before
            bool ok = true;
            while (ok && walk.next(t)) {
                const float *ws = p.ws + t.group * p.ws_group + t.lane_tile * p.ws_lane + t.k0 / BK * p.ws_blk;
                const OUT *x = static_cast<const OUT *>(p.raw) + (t.col0 + first) * p.ld_raw + t.k0 + sub * 8;
                uint4 v[PASSES];
                float w = 0.f;
                auto fetch = [&](int kb) {
                    if (kb >= t.nkb) return;
                    w = ws[kb * p.ws_blk];
#pragma unroll
                    for (int i = 0; i < PASSES; ++i) {
                        if (i * 2 >= t.valid) break;
                        v[i] = make_uint4(0, 0, 0, 0);
                        if (i * 2 + first < t.valid && kb * BK + sub * 8 < t.depth)
                            v[i] = __ldg(reinterpret_cast<const uint4 *>(x + i * 2 * p.ld_raw + kb * BK));
                    }
                };
                int kb = (odd ^ it0) & 1;           // the warp of an even (odd) count of stages
                fetch(kb);
                for (; kb < t.nkb; kb += 2) {
                    const uint32_t it = it0 + kb, s = it % STAGES, z = it % kScaleStages;
                    ok = warp_wait(smem_u32(&ctl.empty[s]), ((it / STAGES) & 1) ^ 1, fail, p.status) &&
                         warp_wait(smem_u32(&ctl.sempty[z]), ((it / kScaleStages) & 1) ^ 1, fail, p.status);
                    if (!ok) break;
                    unsigned char *b = buf + s * S::kStage + S::kA;
#pragma unroll
                    for (int i = 0; i < PASSES; ++i) {
                        if (i * 2 >= t.valid) break;
                        float f[8];
                        unpack8<OUT>(v[i], f);
                        float m = amax8(f);
#pragma unroll
                        for (int d = 8; d; d >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
                        m = block_amax(m);
                        const int r = i * 2 + first;
                        if (r < t.valid) {
                            // 16-byte pieces of a row change places by the row (128-byte swizzle)
                            *reinterpret_cast<uint2 *>(b + r * kRowBytes + (((sub >> 1) ^ r) & 7) * 16 + (sub & 1) * 8) =
                                to_e4m3(f, block_inv(m));
                            if (sub == 0) ctl.xs[z][r] = block_scale(m);
                        }
                    }
                    if (lane == 0) ctl.ws[z] = w;
                    fence_async();
                    __syncwarp();
                    if (lane == 0) {
                        bar_arrive(smem_u32(&ctl.full[s]));
                        bar_arrive(smem_u32(&ctl.sfull[z]));
                    }
                    fetch(kb + 2);
                }
                it0 += t.nkb;
            }
        } else if constexpr (KIND == kE4M3) {
            // Scales of the rows and of the weight block, one slot for each k
            // block, fetched up to kScaleStages blocks ahead by two warps
            // (alternate chunks of 32 columns).  Addresses and bounds are set
            // up once for a tile: with one warp that formed them for each
            // block, fetching scales took three times as long as the products.
            constexpr int N = COLS / (2 * 32);
            const int odd = warp - kScaleWarp;
            if (p.dependent) wait_for_previous();
            uint32_t it = 0;
            bool ok = true;
            while (ok && walk.next(t)) {
                const int nkb = t.nkb;
                const long kb0 = t.k0 / BK;
                const float *ws = p.ws + t.group * p.ws_group + t.lane_tile * p.ws_lane + kb0 * p.ws_blk;
                const float *xs[N];
                bool real[N];
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int c = (2 * i + odd) * 32 + lane;
                    real[i] = c < t.valid;
                    xs[i] = real[i] ? p.xs + (t.col0 + c) * p.xs_row + kb0 * p.xs_blk : p.xs;
                }
                for (int kb = 0; kb < nkb; ++kb, ++it) {
                    const uint32_t s = it % kScaleStages;
                    ok = warp_wait(smem_u32(&ctl.sempty[s]), ((it / kScaleStages) & 1) ^ 1, fail, p.status);
                    if (!ok) break;
                    const uint32_t dst = smem_u32(&ctl.xs[s][odd * 32 + lane]);
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if ((2 * i + odd) * 32 < t.ncols) {
                            copy4(dst + i * 256, xs[i], real[i]);
                            if (real[i]) xs[i] += p.xs_blk;
                        }
                    if (lane == 0 && odd == 0) copy4(smem_u32(&ctl.ws[s]), ws, true);
                    ws += p.ws_blk;
                    copy_arrive(smem_u32(&ctl.sfull[s]));
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        }
    } else {
        // epilogue: warp w has lanes 32 (w % 4).., column chunks w / 4, w / 4 + 2, ...
        static_assert(COLS == 2 * kChunk || (KIND != kE4M3 && !SPLIT && COLS % (2 * kChunk) == 0), "");
        const int quad = warp & 3, half = warp >> 2;
        const uint32_t lanes_at = static_cast<uint32_t>(quad * 32) << 16;
        unsigned char *stage = ctl.stage[half];
        uint32_t acc = 0;
        bool ok = true;
        while (walk.next(t)) {
            const int nkb = t.nkb;
            const int lane0 = t.lane_tile * walk.LANES + int(rank) * kLanes;
            const int features = min(kLanes, p.lanes - lane0);
            OUT *out = static_cast<OUT *>(p.out) + (WHICH == kWgrad ? t.group * p.out_group : 0) +
                       static_cast<long>(t.col0) * p.ldo + lane0;
            if constexpr (KIND == kE4M3) {
                float sum[2][16];
#pragma unroll
                for (int j = 0; j < 32; ++j) sum[j >> 4][j & 15] = 0.f;
                const int c0 = half * kChunk;
                for (int kb = 0; kb < nkb; ++kb, ++acc) {
                    const uint32_t s = acc % kScaleStages;
                    if (ok) ok = warp_wait(smem_u32(&ctl.sfull[s]), (acc / kScaleStages) & 1, fail, p.status);
                    if (ok) ok = warp_wait(smem_u32(&ctl.tfull[acc % ACC]), (acc / ACC) & 1, fail, p.status);
                    if (!ok) continue;
                    tc_fence_after();
                    if (c0 < t.ncols) {
                        float v[2][16];
                        const uint32_t at = tmem + lanes_at + (acc % ACC) * COLS + c0;
                        tmem_ld(v[0], at);
                        tmem_ld(v[1], at + (16u << 16));
                        tmem_wait(v[0], v[1]);
                        const float ws = ctl.ws[s];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            float2 f = *reinterpret_cast<const float2 *>(&ctl.xs[s][c0 + 8 * j + 2 * (lane & 3)]);
                            f = __fmul2_rn(f, make_float2(ws, ws));
#pragma unroll
                            for (int h = 0; h < 2; ++h)
#pragma unroll
                                for (int k = 4 * j; k < 4 * j + 4; k += 2) {
                                    const float2 r = __ffma2_rn(make_float2(v[h][k], v[h][k + 1]), f,
                                                                make_float2(sum[h][k], sum[h][k + 1]));
                                    sum[h][k] = r.x;
                                    sum[h][k + 1] = r.y;
                                }
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        bar_arrive_tmem(smem_u32(&ctl.tempty[acc % ACC]));
                        bar_arrive(smem_u32(&ctl.sempty[s]));
                    }
                }
                if (!ok) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) sum[j >> 4][j & 15] = __int_as_float(0x7fffffff);
                }
                if constexpr (SPLIT)
                    ok = add_parts<OUT>(sum, ctl.part, smem_u32(&ctl.pfull), half, quad, lane, out, p.ldo, t.valid,
                                        features, ok, fail, p.status);
                else if (c0 < t.valid)
                    store_chunk<OUT>(sum, stage, half, quad, lane, out, p.ldo, c0, t.valid, features);
            } else {
                if (nkb && ok) ok = warp_wait(smem_u32(&ctl.tfull[acc % ACC]), (acc / ACC) & 1, fail, p.status, nkb);
                tc_fence_after();
                const uint32_t at = tmem + lanes_at + (acc % ACC) * COLS;
                float v[2][16];
                for (int c0 = half * kChunk; c0 < (SPLIT ? COLS : t.valid); c0 += 2 * kChunk) {
                    if (nkb && ok) {
                        tmem_ld(v[0], at + c0);
                        tmem_ld(v[1], at + c0 + (16u << 16));
                        tmem_wait(v[0], v[1]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j >> 4][j & 15] = ok ? 0.f : __int_as_float(0x7fffffff);
                    }
                    if constexpr (!SPLIT)
                        store_chunk<OUT>(v, stage, half, quad, lane, out, p.ldo, c0, t.valid, features);
                }
                if (nkb) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if constexpr (PAIR) bar_arrive_relaxed_in(smem_u32(&ctl.tempty[acc % ACC]), 0);
                        else bar_arrive_tmem(smem_u32(&ctl.tempty[acc % ACC]));
                    }
                    ++acc;
                }
                if constexpr (SPLIT)
                    ok = add_parts<OUT>(v, ctl.part, smem_u32(&ctl.pfull), half, quad, lane, out, p.ldo, t.valid,
                                        features, ok, fail, p.status);
            }
        }
        if constexpr (WHICH != kWgrad) zero_other_rows<OUT>(ctl.groups, p);
    }
    __syncwarp();
    tc_fence_before();
    if constexpr (PAIR) {
        // Rank 1 stays until the last arrival from rank 0 is here: when all of its
        // own work is done that is a few products away, however long the launch
        // has run.  (After a failure rank 0 may still be in a wait of its own.)
        __syncthreads();
        if (rank == 1 && threadIdx.x == 0) {
            volatile int never = 0;
            bar_wait<true>(smem_u32(&ctl.done), 0, &never, nullptr, int(2 * kWaitLimitClocks / 4096));
        }
        __syncwarp();
    }
    if constexpr (MODE != kAlone) cluster_sync();   // nobody reads this block's sums, or its operands, any more
    else __syncthreads();
    tc_fence_after();
    if (warp == kMmaWarp) {
        if constexpr (PAIR) pair_tmem_free(tmem, TMEM_COLS);
        else tmem_free(tmem, TMEM_COLS);
    }
}

// ---------------------------------------------------------------------------
// Host side (bcjr_mm.cu).

// A tiled map of a matrix of `rank` axes (innermost first), `strides` in
// bytes from the second axis on, 128-byte swizzle, zeros outside.
bool make_map(CUtensorMap *m, int kind, int rank, const void *base, const unsigned long long *dims,
              const unsigned long long *strides, const unsigned *box);
// SMs of the current device for a persistent grid (less the reserved ones);
// 0 when the device is not sm_100.  Makes the device's context current.
constexpr int kMaxDevices = 64;
int grid_sms(int *device);

struct Call {
    int kind, which;          // element type, product
    int out_kind;             // e4m3: output type
    const void *a, *b;        // weights (wgrad: X) and row matrix (wgrad: dY)
    long ld_a, ld_b;          // elements between rows of wgrad's X; of the row matrix
    long a_rows, a_inner;     // weight rows (N) and row length (K); wgrad: K in a_inner
    long b_inner;             // row length of the row matrix
    int split;                // blocks that share a tile
    cudaStream_t stream;
    Params p;
};


// Both operand maps of a call.
template <int KIND, int WHICH>
bool make_maps(const Call &c, CUtensorMap &ta, CUtensorMap &tb, bool raw) {
    constexpr unsigned es = KIND == kE4M3 ? 1 : 2, inner = kRowBytes / es;
    using U = unsigned long long;
    if (WHICH == kWgrad) {
        const U dims[2] = {U(c.a_inner), U(c.p.T)}, st[1] = {U(c.ld_a) * es};
        const unsigned box[2] = {inner, inner};
        if (!make_map(&ta, KIND, 2, c.a, dims, st, box)) return false;
    } else {
        const U dims[3] = {U(c.a_inner), U(c.a_rows), U(c.p.E)};
        const U st[2] = {U(c.a_inner) * es, U(c.a_inner) * U(c.a_rows) * es};
        const unsigned box[3] = {inner, WHICH == kForward ? unsigned(kLanes) : inner, 1};
        if (!make_map(&ta, KIND, 3, c.a, dims, st, box)) return false;
    }
    if (raw) {                 // the kernel loads the rows itself
        tb = ta;
        return true;
    }
    const U dims[2] = {U(c.b_inner), U(c.p.T)}, st[1] = {U(c.ld_b) * es};
    const unsigned box[2] = {inner, WHICH == kWgrad ? inner : unsigned(kBoxRows)};
    return make_map(&tb, KIND, 2, c.b, dims, st, box);
}

template <int COLS> long max_col_tiles(const Call &c) { return max_col_tiles<COLS>(c.p.T, c.p.E); }

template <typename... A>
cudaError_t launch_on(void (*k)(A...), long blocks, int threads, int cluster, size_t bytes,
                      const Call &c, const A &...args) {
    if (blocks > 0x7fffffffL) return cudaErrorInvalidValue;
    cudaLaunchAttribute a[2];
    cudaLaunchConfig_t cfg = {};
    if (c.p.dependent) {
        a[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        a[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        a[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        a[cfg.numAttrs].val.clusterDim.x = unsigned(cluster);
        a[cfg.numAttrs].val.clusterDim.y = a[cfg.numAttrs].val.clusterDim.z = 1;
        ++cfg.numAttrs;
    }
    cfg.gridDim = dim3(unsigned(blocks));
    cfg.blockDim = dim3(unsigned(threads));
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = c.stream;
    cfg.attrs = a;
    return cudaLaunchKernelEx(&cfg, k, args...);
}

// A kernel's settings on the current device, once: its shared memory, and for
// one that splits registers that it was compiled for the expected number (a
// split of more registers than a block is launched with would wait for good).
template <typename K>
cudaError_t set_up(K k, size_t bytes, int regs, std::atomic<bool> &ready) {
    if (ready.load(std::memory_order_acquire)) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
    if (e != cudaSuccess) return e;
    cudaFuncAttributes f;
    if (regs && (cudaFuncGetAttributes(&f, k) != cudaSuccess || f.numRegs != regs)) return cudaErrorInvalidConfiguration;
    ready.store(true, std::memory_order_release);
    return cudaSuccess;
}

template <int KIND, typename OUT, int WHICH, int COLS, int STAGES, int MODE, bool RAW = false>
cudaError_t launch(const Call &c) {
    CUtensorMap ta, tb;
    int dev = 0;
    const int sms = grid_sms(&dev);
    if (sms <= 0) return cudaErrorInvalidDevice;
    if (!make_maps<KIND, WHICH>(c, ta, tb, RAW)) return cudaErrorInvalidValue;
    const auto k = &mm_kernel<KIND, OUT, WHICH, COLS, STAGES, MODE, RAW>;
    constexpr size_t bytes = Smem<KIND, COLS, STAGES, MODE>::bytes();
    static_assert(bytes <= 232448, "shared memory of one block");
    static std::atomic<bool> ready[kMaxDevices];
    const cudaError_t e = set_up(k, bytes, 0, ready[dev]);
    if (e != cudaSuccess) return e;
    // no more blocks than there can be tiles
    const long col_tiles = WHICH == kWgrad ? long(c.p.E) * ((c.p.cols + COLS - 1) / COLS) : max_col_tiles<COLS>(c);
    constexpr long lanes = MODE == kPair ? 2 * kLanes : kLanes;
    const long tiles = (c.p.lanes + lanes - 1) / lanes * col_tiles;
    constexpr bool SPLIT = MODE == kSplit;
    if (MODE == kPair) {
        const long pairs = sms / 2 > 0 ? sms / 2 : 1;
        return launch_on(k, 2 * (tiles < pairs ? tiles : pairs), kThreads, 2, bytes, c, ta, tb, c.p);
    }
    return launch_on(k, SPLIT ? tiles * c.split : tiles < sms ? tiles : sms, kThreads, SPLIT ? c.split : 1, bytes, c, ta, tb, c.p);
}

// Two ways for forward and dgrad: few rows to a tile (64 columns, eight stages
// of 16 KB of weights each; with few tiles up to four blocks of a cluster share
// one's contraction), or many (256 columns, or the e4m3 kernel's 128 rows by
// 256 features).  Estimated by the stages that a block works through one after
// the other: a stage of the small tile costs about 0.6 of a large one's, in
// e4m3 about 0.5.  Measured, small against large tiles:
//   1 group,   8 x 2048 x 8192    16-bit 18 | 39 us   e4m3 16 | 37 us
//   1 group, 192 x 2048 x 8192    16-bit 29 | 43      e4m3 23 | 37
//   1 group, 192 x 8192 x 2048    16-bit 25 | 21      e4m3 21 | 18
//   64 groups of about 32, 1024 x 2048   16-bit 49 | 55   e4m3 35 | 35
//   64 groups of about 96, 1024 x 2048   16-bit 72 | 55   e4m3 53 | 43
inline int k_blocks(const Call &c) {
    return (c.p.depth * (c.kind == kE4M3 ? 1 : 2) + kRowBytes - 1) / kRowBytes;
}
inline long few_tiles(const Call &c) { return (c.p.lanes + kLanes - 1L) / kLanes * max_col_tiles<64>(c); }
inline int few_split(const Call &c, int sms) {
    const long tiles = few_tiles(c);
    const int nkb = k_blocks(c);
    int split = 1;
    while (split < kMaxSplit && tiles * split * 2 <= sms && nkb >= split * 2 * 2) split *= 2;
    return split;
}
// Many features: pairs of blocks.  (64 experts, 32768 rows, 1024 and 2048
// features: 113 us forward, 113 and 135 us gradients in pairs, 125, 125 and 157
// us alone.  4 experts, 3000 rows, 1040 features: the same.  96 experts, 3079
// rows, 272 features, weights' gradient: 27 us in pairs, 20 alone: 272 lanes are
// two tiles of 256 but three of 128.)  64 experts, 32768 rows, lanes x the other
// feature axis, us alone | in pairs:
//                      512 x 2048  640 x 1024  768 x 2048  896 x 1024  1040 x 1024  1408 x 1024
//   forward             78 |  70    53 |  53   102 |  90    66 |  66     78 |  76     96 |  88
//   weights' gradient   88 |  84    59 |  76   131 | 121    78 |  76     91 |  94    115 | 117
// Pairs gain where the lanes fill tiles of 256; where they do not, the weights'
// gradient loses a quarter below 1024 lanes and a few per cent from there on.
inline bool in_pairs(const Call &c) {
    const int forced = test_option(kOptLinearTiles);
    return c.kind != kE4M3 && (forced ? forced == 3 : c.p.lanes >= 1024);
}
inline bool few_rows(const Call &c) {
    if (const int forced = test_option(kOptLinearTiles)) return forced == 1;
    int dev = 0;
    const long sms = grid_sms(&dev);
    if (sms <= 0) return true;
    auto waves = [](long tiles, long slots) { return (tiles + slots - 1) / slots; };
    const long nkb = k_blocks(c), split = few_split(c, int(sms));
    const long few = waves(few_tiles(c) * split, sms) * ((nkb + split - 1) / split);
    if (c.kind == kE4M3) return few <= 2 * waves((c.p.lanes + 255L) / 256 * max_col_tiles<128>(c), sms) * nkb;
    const long lanes = in_pairs(c) ? 2 * kLanes : kLanes, slots = in_pairs(c) ? (sms > 1 ? sms / 2 : 1) : sms;
    return 3 * few < 5 * waves((c.p.lanes + lanes - 1) / lanes * max_col_tiles<256>(c), slots) * nkb;
}
template <int KIND, typename OUT, int WHICH, bool RAW = false>
cudaError_t launch_few(Call c) {
    int dev = 0;
    c.split = few_split(c, grid_sms(&dev));
    if (c.split == 1) return launch<KIND, OUT, WHICH, 64, 8, kAlone, RAW>(c);
    return launch<KIND, OUT, WHICH, 64, 6, kSplit, RAW>(c);
}

}  // namespace mm
}  // namespace bcjr
