"""GPU tests of the linear layers beyond test_gpu_linear.py (whose plain products
and tolerances they use): hand-overs inside pairs of blocks, results of a whole
training step, what is kept and refused, and failures of shared tiles."""
import pytest
import torch

from test_linear import difference_holds
from test_gpu_linear import (_check_grouped, _close, _counts_to_offsets, _expand, _grouped64, _inputs,
                             _quantize_plain, _wgrad64)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counts,N,K", [
    ([64, 1, 128, 63, 0, 65, 192, 7, 640, 64, 64, 2] * 4, 528, 1040),     # six tiles to a pair of blocks
    ([64] * 30, 272, 1024),                                               # no stage ends inside a group
    ([3] * 60, 1040, 272),                                                # every stage does
    ([1000, 24, 0, 999], 32, 16),
])
def test_full_and_ragged_stages_of_paired_blocks(cuda_ok, counts, N, K, dtype):
    """Contractions over the rows of a group whose last stage is full, ragged or
    the only one, in every order, so that each stage of the ring is both; the
    results do not change from run to run."""
    from quant_2bit_b200 import _lib, grouped_linear
    x, w, dy = _inputs(sum(counts), len(counts), N, K, dtype, seed=N)
    offsets = _counts_to_offsets(counts)
    with _lib.test_option(_lib.OPT_LINEAR_TILES, 3):
        _check_grouped(x, w, dy, offsets)
        w.requires_grad_()
        first = None
        for _ in range(20):
            dw, = torch.autograd.grad(grouped_linear(x, w, offsets), w, dy)
            first = dw if first is None else first
            assert torch.equal(dw, first)


def test_training_step_of_a_layer_repeats_itself(cuda_ok):
    """64 experts, 32768 rows, 1024 x 2048: forward and both gradients within
    their bounds of the 64-bit products, and the same bits every time."""
    from quant_2bit_b200 import grouped_linear
    E, T, N, K = 64, 32768, 1024, 2048
    g = torch.Generator(device="cuda").manual_seed(4)
    counts = torch.bincount(torch.multinomial(torch.rand(E, generator=g, device="cuda"), T, True,
                                              generator=g), minlength=E).tolist()
    offsets = _counts_to_offsets(counts)
    x, w, dy = _inputs(T, E, N, K, torch.bfloat16)
    x.requires_grad_()
    w.requires_grad_()
    first = None
    for _ in range(10):
        y = grouped_linear(x, w, offsets)
        out = [y.detach(), *torch.autograd.grad(y, (x, w), dy)]
        first = first or out
        assert all(torch.equal(a, b) for a, b in zip(first, out))
    y, dx, dw = first
    ref, mag = _grouped64(x.detach(), w.detach(), offsets)
    _close(y, ref, mag, K, "y")
    ref, mag = _grouped64(dy, w.detach().transpose(1, 2), offsets)
    _close(dx, ref, mag, N, "dx")
    ref, mag = _wgrad64(dy, x.detach(), offsets, E)
    _close(dw, ref, mag, max(counts), "dw")


def test_a_product_longer_than_a_wait_may_last(cuda_ok):
    """A weights' gradient in pairs of blocks that runs for about two seconds:
    limits count from each wait's start and grow with the work waited for.
    (393216 rows of whole numbers up to 2 serve as both factors, so that all
    sums are exact in fp32; 64 x 64 of the 65536 x 65536 are checked.)"""
    import ctypes
    from quant_2bit_b200 import _lib
    T, N = 393216, 65536
    lib = _lib.load()
    x = torch.empty(T, N, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(8)
    for rows in x.split(32768):
        rows.random_(0, 5, generator=g).sub_(2)
    dw = torch.zeros(N, N, dtype=torch.bfloat16, device="cuda")
    status = torch.full((1,), 77, dtype=torch.int32, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.bcjr_grouped_backward(x.data_ptr(), N, x.data_ptr(), N, None, None, 0, T, 1, N, N, 0, None,
                                     dw.data_ptr(), status.data_ptr(), stream) == 0
    assert lib.bcjr_ws_status(ctypes.c_void_p(status.data_ptr()), stream) == 0
    exact = x[:, 1000:1064].double().t() @ x[:, -64:].double()
    assert float(exact.abs().max()) < 2 ** 24 and torch.equal(dw[1000:1064, -64:], exact.to(torch.bfloat16))


def test_forward_mode_derivatives_are_refused(cuda_ok):
    from torch.autograd import forward_ad
    from quant_2bit_b200 import fp8_linear, fp8_quantize_weight, grouped_linear
    x, w, _ = _inputs(20, 2, 32, 64, torch.bfloat16)
    offsets = _counts_to_offsets([5, 15])
    q, s = fp8_quantize_weight(w[0])
    want = grouped_linear(x, w, offsets), fp8_linear(x, q, s)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for f, args in ((grouped_linear, (dual, w, offsets)), (fp8_linear, (dual, q, s)),
                        (grouped_linear, (x, forward_ad.make_dual(w, torch.ones_like(w)), offsets))):
            with pytest.raises(NotImplementedError):
                f(*args)
        assert torch.equal(grouped_linear(x, w, offsets), want[0]) and torch.equal(fp8_linear(x, q, s), want[1])


@pytest.mark.parametrize("frozen", ["x", "weight"])
def test_gradient_of_one_operand_keeps_the_other_only(cuda_ok, frozen):
    """With one operand frozen its gradient's partner is not kept: it may be
    changed in place before the backward pass, and its memory is not held."""
    from quant_2bit_b200 import grouped_linear
    counts = [70, 0, 31]
    offsets = _counts_to_offsets(counts)
    x, w, dy = _inputs(101, 3, 64, 112, torch.bfloat16)
    x0, w0 = x.clone(), w.clone()
    leaf = w if frozen == "x" else x
    leaf.requires_grad_()
    y = grouped_linear(x, w, offsets)
    with torch.no_grad():
        leaf.zero_()                     # read by neither gradient
    grad, = torch.autograd.grad(y, leaf, dy)
    ref, mag = _wgrad64(dy, x0, offsets, 3) if frozen == "x" else _grouped64(dy, w0.transpose(1, 2), offsets)
    _close(grad, ref, mag, 70 if frozen == "x" else 64, "gradient")


@pytest.mark.parametrize("tiles", [1, 2, 3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients_against_differences_along_the_gradient(cuda_ok, dtype, tiles):
    """<dy, f(d)> = <gradient, d> with d the 64-bit gradient, where both sides are
    a sum of squares (a displacement of its own leaves a sum of signed terms, in
    which the tolerance hides a missing gradient)."""
    from quant_2bit_b200 import _lib, grouped_linear
    counts = [70, 0, 31, 200]
    offsets = _counts_to_offsets(counts)
    x, w, dy = _inputs(301, 4, 96, 112, dtype, seed=5)
    dx64, dx_mag = _grouped64(dy, w.transpose(1, 2), offsets)
    dw64, dw_mag = _wgrad64(dy, x, offsets, 4)
    d_x, d_w = dx64.to(dtype), dw64.to(dtype)
    leaves = x.clone().requires_grad_(), w.clone().requires_grad_()
    with _lib.test_option(_lib.OPT_LINEAR_TILES, tiles):
        dx, dw = torch.autograd.grad(grouped_linear(*leaves, offsets), leaves, dy)
        f_x, f_w = grouped_linear(d_x, w, offsets), grouped_linear(x, d_w, offsets)
    assert difference_holds(dy, f_x, _grouped64(d_x, w, offsets)[1], 112, dx, dx_mag, 96, d_x)
    assert difference_holds(dy, f_w, _grouped64(x, d_w, offsets)[1], 112, dw, dw_mag, 200, d_w)


def test_a_wait_that_runs_out_in_shared_and_long_tiles(cuda_ok):
    """The first load of block 0 withheld where blocks of a cluster share a
    tile's contraction, where the 8-bit product overlaps its quantizer in small
    tiles, and where a contraction is longer than the ring of stages: the call
    reports it, the first tile's outputs are NaN, the next call is clean."""
    import ctypes
    from quant_2bit_b200 import _lib, fp8_quantize_weight
    lib = _lib.load()
    stream = torch.cuda.current_stream().cuda_stream
    status = torch.full((1,), 77, dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(torch.bfloat16)

    x, w = rand(1000, 4096), rand(272, 4096)
    q, s = fp8_quantize_weight(w)
    out = torch.zeros(1000, 272, dtype=torch.bfloat16, device="cuda")
    narrow, dw = rand(1000, 272), torch.zeros(272, 4096, dtype=torch.bfloat16, device="cuda")
    ws = torch.empty(lib.bcjr_fp8_linear_workspace_bytes(1000, 4096), dtype=torch.uint8, device="cuda")

    def forward(rows, K):
        return lambda: lib.bcjr_grouped_mm(x.data_ptr(), 4096, w.data_ptr(), None, 0, rows, 1, 272, K, 0,
                                           out.data_ptr(), status.data_ptr(), stream)

    def fp8(rows, K):
        return lambda: lib.bcjr_fp8_linear(x.data_ptr(), 4096, 0, q.data_ptr(), s.data_ptr(), None, 0, rows, 1,
                                           272, K, 0, out.data_ptr(), ws.data_ptr(), ws.numel(),
                                           status.data_ptr(), stream)

    def weights():
        return lib.bcjr_grouped_backward(narrow.data_ptr(), 272, x.data_ptr(), 4096, None, None, 0, 1000, 1, 272,
                                         4096, 0, None, dw.data_ptr(), status.data_ptr(), stream)

    # (tiles, call, the outputs of block 0's tile)
    for tiles, call, hit in ((1, forward(20, 1040), out[:20, :128]), (1, forward(20, 4096), out[:20, :128]),
                             (1, fp8(20, 1040), out[:20, :128]), (1, fp8(20, 4096), out[:20, :128]),
                             (1, fp8(40, 1040), out[:40, :128]), (1, fp8(40, 4096), out[:40, :128]),
                             (2, forward(200, 4096), out[:200, :128]), (3, forward(200, 4096), out[:200, :256]),
                             (2, fp8(128, 4096), out[:128, :256]), (2, weights, dw[:256, :128]),
                             (3, weights, dw[:256, :256])):
        with _lib.test_option(_lib.OPT_LINEAR_TILES, tiles):
            with _lib.test_option(_lib.OPT_TEST_DROP_SENDS, 1):
                assert call() == 0
                assert lib.bcjr_ws_status(ctypes.c_void_p(status.data_ptr()), stream) == _lib.BCJR_ERR_TIMEOUT
            assert hit.isnan().all()
            assert call() == 0
            assert lib.bcjr_ws_status(ctypes.c_void_p(status.data_ptr()), stream) == 0
            assert torch.isfinite(hit).all()


def test_8_bit_layers_beyond_32_bits(cuda_ok):
    """Rows, outputs, codes and weights of more than 2^31 elements."""
    from quant_2bit_b200 import _lib, fp8_linear, fp8_matmul, fp8_quantize_rows, fp8_quantize_weight
    g = torch.Generator(device="cuda").manual_seed(3)
    T, N, K = 2_150_000, 16, 1008
    x = torch.empty(T, K, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    assert x.numel() > 2 ** 31
    q, s = fp8_quantize_weight(torch.randn(N, K, generator=g, device="cuda"))
    w64 = _expand(q, s, 128)
    xq, xs = fp8_quantize_rows(x)
    y = fp8_matmul(xq, xs, q, s)
    ends = (slice(0, 300), slice(T - 300, T))
    for rows in ends:
        a, b = _quantize_plain(x[rows], 1)
        assert torch.equal(xq[rows].view(torch.uint8), a.contiguous().view(torch.uint8)) and torch.equal(xs[rows], b)
        a = _expand(a, b, 1)
        _close(y[rows], a @ w64.t(), a.abs() @ w64.abs().t(), K, "y", extra=4)
    del xq, xs
    assert torch.equal(fp8_linear(x, q, s), y)
    # the gradient: T x 1008 out
    x.requires_grad_()
    dy = torch.randn(T, N, generator=g, device="cuda").to(torch.bfloat16)
    dx, = torch.autograd.grad(fp8_linear(x, q, s), x, dy)
    for rows in ends:
        a = _expand(*_quantize_plain(dy[rows], 1), 1)
        _close(dx[rows], a @ w64, a.abs() @ w64.abs(), N, "dx", extra=4)
    del x, y, dx

    E, N, K = 1024, 2064, 1024
    w = torch.zeros(E, N, K, dtype=torch.bfloat16, device="cuda")
    w[-2:] = torch.randn(2, N, K, generator=g, device="cuda")
    q, s = fp8_quantize_weight(w)
    assert q.numel() > 2 ** 31
    for e in (E - 2, E - 1):
        a, b = _quantize_plain(w[e], 128)
        assert torch.equal(q[e].view(torch.uint8), a.contiguous().view(torch.uint8)) and torch.equal(s[e], b)
    del w
    w64 = torch.stack([_expand(q[e], s[e], 128) for e in (E - 2, E - 1)])
    for T, tiles in ((30, 0), (40, 1), (300, 2)):
        x, dy = (torch.randn(T, n, generator=g, device="cuda").to(torch.bfloat16) for n in (K, N))
        offsets = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
        offsets[-2], offsets[-1] = 17, T
        x.requires_grad_()
        with _lib.test_option(_lib.OPT_LINEAR_TILES, tiles):
            y = fp8_linear(x, q, s, offsets)
            dx, = torch.autograd.grad(y, x, dy)
        two = torch.tensor([0, 17, T])
        for got, rows, weight, depth in ((y.detach(), x.detach(), w64, K), (dx, dy, w64.transpose(1, 2), N)):
            ref, mag = _grouped64(_expand(*_quantize_plain(rows, 1), 1), weight, two)
            _close(got, ref, mag, depth, "fp8", extra=4)
