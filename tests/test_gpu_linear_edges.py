"""GPU tests of the linear layers beyond test_gpu_linear.py (whose plain products
and tolerances they use): hand-overs inside pairs of blocks, results of a whole
training step, what is kept and refused, and failures of shared tiles."""
import pytest
import torch

from test_gpu_linear import _check_grouped, _close, _counts_to_offsets, _grouped64, _inputs, _wgrad64

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
