// Products grouped by expert with ragged sizes, bf16 and fp16 (the kernel and
// its mathematics: bcjr_mm.cuh).  C entry points bcjr_grouped_mm (forward and
// the gradient of the rows) and bcjr_grouped_wgrad (gradient of the weights).
#include "../../include/bcjr_b200.h"
#include "bcjr_kernels.h"
#include "bcjr_mm.cuh"

namespace bcjr {
namespace mm {
namespace {

template <int KIND, typename T>
cudaError_t run(const Call &c) {
    if (c.which == kWgrad) return launch<KIND, T, kWgrad, 256, 4, false>(c);
    if (c.p.T <= 64) return c.which == kForward ? launch_few<KIND, T, kForward>(c) : launch_few<KIND, T, kDgrad>(c);
    return c.which == kForward ? launch<KIND, T, kForward, 256, 4, false>(c) : launch<KIND, T, kDgrad, 256, 4, false>(c);
}

bool aligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

int check(const void *offsets, int offsets_bytes, long T, int E, int N, int K, int dtype) {
    if (T < 0 || T > 0x7fffff00L || E < 1 || E > kMaxGroups || N < 16 || K < 16 || N % 16 || K % 16 ||
        N > (1 << 24) || K > (1 << 24))
        return BCJR_ERR_BAD_SHAPE;
    if (dtype != BCJR_BF16 && dtype != BCJR_F16) return BCJR_ERR_UNSUPPORTED;
    if (offsets ? (offsets_bytes != 4 && offsets_bytes != 8) : E != 1) return BCJR_ERR_BAD_SHAPE;
    if (offsets && !aligned(offsets, size_t(offsets_bytes))) return BCJR_ERR_ALIGNMENT;
    return BCJR_OK;
}

}  // namespace
}  // namespace mm
}  // namespace bcjr

using namespace bcjr::mm;

extern "C" {

int bcjr_grouped_mm(const void *rows, long ld_rows, const void *w, const void *offsets,
                    int offsets_bytes, long T, int E, int N, int K, int dtype, int transpose_w,
                    void *out, int *status, bcjr_stream_t stream) {
    const int st = check(offsets, offsets_bytes, T, E, N, K, dtype);
    if (st) return st;
    if (T == 0) return BCJR_OK;
    if (!rows || !w || !out) return BCJR_ERR_NULL_POINTER;
    const int depth = transpose_w ? N : K, lanes = transpose_w ? K : N;
    if (ld_rows < depth || ld_rows > (1L << 32)) return BCJR_ERR_BAD_SHAPE;
    if (!aligned(rows, 16) || ld_rows % 8 || !aligned(w, 16) || !aligned(out, 16) || !aligned(status, 4))
        return BCJR_ERR_ALIGNMENT;
    Call c = {};
    c.kind = dtype == BCJR_BF16 ? kBF16 : kF16;
    c.which = transpose_w ? kDgrad : kForward;
    c.a = w;
    c.a_rows = N;
    c.a_inner = K;
    c.b = rows;
    c.ld_b = ld_rows;
    c.b_inner = depth;
    c.stream = reinterpret_cast<cudaStream_t>(stream);
    c.p.offsets = offsets;
    c.p.offsets64 = offsets_bytes == 8;
    c.p.T = int(T);
    c.p.E = E;
    c.p.lanes = lanes;
    c.p.depth = depth;
    c.p.out = out;
    c.p.ldo = lanes;
    c.p.status = status;
    c.p.drop = bcjr::test_option(bcjr::kOptDropSends);
    const cudaError_t e = c.kind == kBF16 ? run<kBF16, __nv_bfloat16>(c) : run<kF16, __half>(c);
    return e == cudaSuccess ? BCJR_OK : e == cudaErrorInvalidDevice ? BCJR_ERR_DEVICE : BCJR_ERR_LAUNCH;
}

int bcjr_grouped_wgrad(const void *dy, long ld_dy, const void *x, long ld_x, const void *offsets,
                       int offsets_bytes, long T, int E, int N, int K, int dtype, void *dw,
                       int *status, bcjr_stream_t stream) {
    const int st = check(offsets, offsets_bytes, T, E, N, K, dtype);
    if (st) return st;
    if (!dw || (T > 0 && (!dy || !x))) return BCJR_ERR_NULL_POINTER;
    if (T > 0 && (ld_dy < N || ld_x < K || ld_dy > (1L << 32) || ld_x > (1L << 32)))
        return BCJR_ERR_BAD_SHAPE;
    if (!aligned(dw, 16) || !aligned(status, 4)) return BCJR_ERR_ALIGNMENT;
    if (T > 0 && (!aligned(dy, 16) || !aligned(x, 16) || ld_dy % 8 || ld_x % 8)) return BCJR_ERR_ALIGNMENT;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (T == 0)
        return cudaMemsetAsync(dw, 0, size_t(E) * N * K * 2, s) == cudaSuccess ? BCJR_OK : BCJR_ERR_LAUNCH;
    Call c = {};
    c.kind = dtype == BCJR_BF16 ? kBF16 : kF16;
    c.which = kWgrad;
    c.a = x;
    c.ld_a = ld_x;
    c.a_inner = K;
    c.b = dy;
    c.ld_b = ld_dy;
    c.b_inner = N;
    c.stream = s;
    c.p.offsets = offsets;
    c.p.offsets64 = offsets_bytes == 8;
    c.p.T = int(T);
    c.p.E = E;
    c.p.lanes = K;
    c.p.cols = N;
    c.p.out = dw;
    c.p.ldo = K;
    c.p.out_group = long(N) * K;
    c.p.status = status;
    c.p.drop = bcjr::test_option(bcjr::kOptDropSends);
    const cudaError_t e = c.kind == kBF16 ? run<kBF16, __nv_bfloat16>(c) : run<kF16, __half>(c);
    return e == cudaSuccess ? BCJR_OK : e == cudaErrorInvalidDevice ? BCJR_ERR_DEVICE : BCJR_ERR_LAUNCH;
}

}  // extern "C"
