// Products grouped by expert with ragged sizes, bf16 and fp16 (the kernel and
// its mathematics: bcjr_mm.cuh).  C entry points bcjr_grouped_mm and
// bcjr_grouped_backward (gradients of the rows and of the weights).
#include "../../include/bcjr_b200.h"
#include "bcjr_kernels.h"
#include "bcjr_mm.cuh"

namespace bcjr {
namespace mm {
namespace {

template <int KIND, typename T, int WHICH>
cudaError_t launch_many(const Call &c) {
    if (in_pairs(c)) return launch<KIND, T, WHICH, 256, 6, kPair>(c);
    return launch<KIND, T, WHICH, 256, 4, kAlone>(c);
}

template <int KIND, typename T>
cudaError_t launch_which(const Call &c) {
    if (c.which == kWgrad) return launch_many<KIND, T, kWgrad>(c);
    if (few_rows(c)) return c.which == kForward ? launch_few<KIND, T, kForward>(c) : launch_few<KIND, T, kDgrad>(c);
    return c.which == kForward ? launch_many<KIND, T, kForward>(c) : launch_many<KIND, T, kDgrad>(c);
}

bool aligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

int check(const void *offsets, int offsets_bytes, long T, int E, int N, int K, int dtype) {
    if (T < 0 || T > kMaxRows || E < 1 || E > kMaxGroups || N < 16 || K < 16 || N % 16 || K % 16 ||
        N > (1 << 24) || K > (1 << 24))
        return BCJR_ERR_BAD_SHAPE;
    if (dtype != BCJR_BF16 && dtype != BCJR_F16) return BCJR_ERR_UNSUPPORTED;
    if (offsets ? (offsets_bytes != 4 && offsets_bytes != 8) : E != 1) return BCJR_ERR_BAD_SHAPE;
    if (offsets && !aligned(offsets, size_t(offsets_bytes))) return BCJR_ERR_ALIGNMENT;
    return BCJR_OK;
}

Call call(const void *offsets, int offsets_bytes, long T, int E, int dtype, int *status,
          bcjr_stream_t stream) {
    Call c = {};
    c.kind = dtype == BCJR_BF16 ? kBF16 : kF16;
    c.stream = reinterpret_cast<cudaStream_t>(stream);
    c.p.offsets = offsets;
    c.p.offsets64 = offsets_bytes == 8;
    c.p.T = int(T);
    c.p.E = E;
    c.p.status = status;
    c.p.drop = test_option(kOptDropSends);
    return c;
}

int run(const Call &c) {
    const cudaError_t e = c.kind == kBF16 ? launch_which<kBF16, __nv_bfloat16>(c) : launch_which<kF16, __half>(c);
    return e == cudaSuccess ? BCJR_OK : e == cudaErrorInvalidDevice ? BCJR_ERR_DEVICE : BCJR_ERR_LAUNCH;
}

}  // namespace
}  // namespace mm
}  // namespace bcjr

using namespace bcjr::mm;

extern "C" {

int bcjr_grouped_mm(const void *x, long ld_x, const void *w, const void *offsets,
                    int offsets_bytes, long T, int E, int N, int K, int dtype, void *y,
                    int *status, bcjr_stream_t stream) {
    const int st = check(offsets, offsets_bytes, T, E, N, K, dtype);
    if (st) return st;
    if (T == 0) return BCJR_OK;
    if (!x || !w || !y) return BCJR_ERR_NULL_POINTER;
    if (ld_x < K || ld_x > (1L << 32)) return BCJR_ERR_BAD_SHAPE;
    if (!aligned(x, 16) || ld_x % 8 || !aligned(w, 16) || !aligned(y, 16) || !aligned(status, 4))
        return BCJR_ERR_ALIGNMENT;
    Call c = call(offsets, offsets_bytes, T, E, dtype, status, stream);
    c.which = kForward;
    c.a = w;
    c.a_rows = N;
    c.a_inner = K;
    c.b = x;
    c.ld_b = ld_x;
    c.b_inner = c.p.depth = K;
    c.p.out = y;
    c.p.ldo = c.p.lanes = N;
    return run(c);
}

int bcjr_grouped_backward(const void *dy, long ld_dy, const void *x, long ld_x, const void *w,
                          const void *offsets, int offsets_bytes, long T, int E, int N, int K,
                          int dtype, void *dx, void *dw, int *status, bcjr_stream_t stream) {
    int st = check(offsets, offsets_bytes, T, E, N, K, dtype);
    if (st) return st;
    if (T == 0) {
        cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
        if (dw && cudaMemsetAsync(dw, 0, size_t(E) * N * K * 2, s) != cudaSuccess) return BCJR_ERR_LAUNCH;
        return BCJR_OK;
    }
    if (!dy || (dx && !w) || (dw && !x)) return BCJR_ERR_NULL_POINTER;
    if (ld_dy < N || ld_dy > (1L << 32) || (dw && (ld_x < K || ld_x > (1L << 32)))) return BCJR_ERR_BAD_SHAPE;
    if (!aligned(dy, 16) || ld_dy % 8 || !aligned(dx, 16) || !aligned(dw, 16) || !aligned(status, 4) ||
        (dx && !aligned(w, 16)) || (dw && (!aligned(x, 16) || ld_x % 8)))
        return BCJR_ERR_ALIGNMENT;
    Call c = call(offsets, offsets_bytes, T, E, dtype, status, stream);
    c.b = dy;
    c.ld_b = ld_dy;
    c.b_inner = N;
    c.a_inner = K;
    c.p.ldo = c.p.lanes = K;
    if (dx) {
        c.which = kDgrad;
        c.a = w;
        c.a_rows = N;
        c.p.depth = N;
        c.p.out = dx;
        if ((st = run(c))) return st;
    }
    if (dw) {
        c.which = kWgrad;
        c.a = x;
        c.ld_a = ld_x;
        c.p.cols = N;
        c.p.out = dw;
        c.p.out_group = long(N) * K;
        c.p.keep_status = dx != nullptr;       // a failure of the first kernel stays
        if ((st = run(c))) return st;
    }
    return BCJR_OK;
}

}  // extern "C"
