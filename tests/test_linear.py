"""CPU tests of the linear layers' entry points: what the C ABI refuses before
any device work, and that CPU tensors raise (there is no CPU path)."""
import pytest
import torch
from torch.autograd import forward_ad

from quant_2bit_b200 import _lib

OK, SHAPE, UNSUPPORTED, NULL, ALIGN = 0, 1, 2, 3, 4
P = 1 << 20                       # stands for a device pointer: refused calls never use it


@pytest.fixture(scope="module")
def lib():
    from quant_2bit_b200 import build
    build.build()
    return _lib.load()


def _mm(lib, x=P, ld=64, w=P, off=P, off_size=4, T=8, E=2, N=32, K=64, dtype=0, y=P, status=P):
    return lib.bcjr_grouped_mm(x, ld, w, off, off_size, T, E, N, K, dtype, y, status, None)


def _backward(lib, dy=P, ld_dy=32, x=P, ld_x=64, w=P, off=P, off_size=4, T=8, E=2, N=32, K=64, dtype=0,
              dx=P, dw=P, status=P):
    return lib.bcjr_grouped_backward(dy, ld_dy, x, ld_x, w, off, off_size, T, E, N, K, dtype, dx, dw,
                                     status, None)


def _fp8(lib, rows=P, ld=64, xs=P, s_row=1, s_blk=8, w=P, ws=P, off=P, off_size=4, T=8, E=2, N=32,
         K=64, tr=0, out=P, dtype=0, status=P):
    return lib.bcjr_fp8_mm(rows, ld, xs, s_row, s_blk, w, ws, off, off_size, T, E, N, K, tr, out,
                           dtype, status, None)


@pytest.mark.parametrize("call", [_mm, _backward, _fp8])
def test_products_refuse_bad_sizes(lib, call):
    for bad in (dict(T=-1), dict(T=1 << 31), dict(E=0), dict(E=1025), dict(N=0), dict(N=24),
                dict(K=8), dict(K=72), dict(off_size=2), dict(off=None), dict(N=1 << 25)):
        assert call(lib, **bad) == SHAPE, bad
    assert call(lib, dtype=2) == UNSUPPORTED
    assert call(lib, dtype=-1) == UNSUPPORTED


def test_products_refuse_bad_pointers_and_strides(lib):
    assert _mm(lib, T=0, x=None, y=None, status=None) == OK              # nothing to do
    assert _backward(lib, T=0, dy=None, x=None, dw=None) == OK
    assert _fp8(lib, T=0, rows=None, xs=None, out=None, status=None) == OK
    for call, names in ((_mm, ("x", "w", "y")), (_backward, ("dy", "x", "w")),
                        (_fp8, ("rows", "xs", "w", "ws", "out"))):
        for n in names:
            assert call(lib, **{n: None}) == NULL, n
    assert _mm(lib, ld=56) == SHAPE
    assert _mm(lib, ld=68) == ALIGN
    assert _mm(lib, x=P + 8) == ALIGN
    assert _mm(lib, w=P + 2) == ALIGN
    assert _mm(lib, y=P + 8) == ALIGN
    assert _mm(lib, off=P + 4, off_size=8) == ALIGN
    assert _backward(lib, ld_dy=16) == SHAPE
    assert _backward(lib, ld_x=48) == SHAPE
    assert _backward(lib, ld_x=68) == ALIGN
    assert _backward(lib, dx=P + 8) == _backward(lib, dw=P + 8) == ALIGN
    assert _backward(lib, w=P + 8) == ALIGN
    assert _fp8(lib, ld=72) == ALIGN
    assert _fp8(lib, s_row=-1) == SHAPE
    assert _fp8(lib, xs=P + 2) == ALIGN


def test_fp8_linear_refuses(lib):
    def call(x=P, ld=64, dtype=0, w=P, s=P, T=40, N=32, K=64, tr=0, out=P, ws=P, size=1 << 20):
        return lib.bcjr_fp8_linear(x, ld, dtype, w, s, P, 4, T, 2, N, K, tr, out, ws, size, None, None)

    need = lib.bcjr_fp8_linear_workspace_bytes(40, 64)
    assert need >= 40 * 64 + 40 * 4 and lib.bcjr_fp8_linear_workspace_bytes(8, 40) == 0
    assert call(size=need - 1) == call(ws=None) == 5
    assert call(dtype=2) == UNSUPPORTED
    assert call(K=40) == call(T=-1) == call(ld=32) == SHAPE
    assert call(x=P + 8) == call(ws=P + 8) == ALIGN
    assert call(x=None) == NULL
    assert call(T=0, x=None, ws=None) == OK
    # few rows: no workspace, the other checks as before
    assert call(T=8, ws=None, size=0, dtype=2) == UNSUPPORTED
    assert call(T=8, ws=None, size=0, x=P + 8) == call(T=8, ws=None, ld=68) == ALIGN
    assert call(T=8, ws=None, w=None) == call(T=8, ws=None, x=None) == NULL
    assert call(T=8, ws=None, ld=32) == SHAPE


def test_workspace_formula(lib):
    """The binding sizes the workspace by the library's formula."""
    from quant_2bit_b200 import linear
    assert lib.bcjr_fp8_linear_workspace_bytes(linear._RAW_ROWS, 144) == 16      # not used
    for T, C in ((linear._RAW_ROWS + 1, 16), (64, 144), (4097, 2048)):
        assert lib.bcjr_fp8_linear_workspace_bytes(T, C) == T * (C + 4 * linear._blocks(C)) + 16


def test_quantizers_refuse(lib):
    def rows(x=P, ld=64, n=8, k=64, dtype=0, q=P, s=P, s_row=1, s_blk=8):
        return lib.bcjr_fp8_quantize_rows(x, ld, n, k, dtype, q, s, s_row, s_blk, None)

    def blocks(w=P, E=1, N=8, K=64, dtype=0, q=P, s=P):
        return lib.bcjr_fp8_quantize_blocks(w, E, N, K, dtype, q, s, None)

    for bad in (dict(n=-1), dict(k=24), dict(k=0), dict(ld=48), dict(s_row=-1)):
        assert rows(**bad) == SHAPE, bad
    for bad in (dict(E=-1), dict(N=0), dict(K=24), dict(E=1 << 20, N=1 << 20)):
        assert blocks(**bad) == SHAPE, bad
    assert rows(dtype=3) == blocks(dtype=3) == UNSUPPORTED
    assert rows(n=0, x=None) == blocks(E=0, w=None) == OK
    assert rows(q=None) == blocks(s=None) == NULL
    assert rows(x=P + 8) == rows(ld=68) == blocks(q=P + 4) == ALIGN


def test_cpu_tensors_raise():
    import quant_2bit_b200 as q
    x, w = torch.zeros(4, 32, dtype=torch.bfloat16), torch.zeros(2, 16, 32, dtype=torch.bfloat16)
    off = torch.tensor([0, 1, 4])
    f8 = torch.zeros(16, 32).to(torch.float8_e4m3fn)
    for f, args in ((q.grouped_linear, (x, w, off)), (q.fp8_quantize_rows, (x,)),
                    (q.fp8_quantize_weight, (w,)), (q.fp8_linear, (x, f8, torch.ones(1, 1))),
                    (q.fp8_matmul, (f8, torch.ones(16, 1), f8, torch.ones(1, 1)))):
        with pytest.raises(RuntimeError, match="CUDA"):
            f(*args)


@pytest.fixture
def stubbed(monkeypatch):
    """The Python layer alone: CPU tensors pass and no C call is made."""
    from quant_2bit_b200 import build, linear
    build.build()
    calls = []
    monkeypatch.setattr(linear, "_need_cuda", lambda *a: -1)
    monkeypatch.setattr(linear, "_call", lambda fn, *a: calls.append(fn.__name__))
    return calls


def _operands():
    x, w = torch.zeros(4, 32, dtype=torch.bfloat16), torch.zeros(2, 16, 32, dtype=torch.bfloat16)
    return x, w, torch.tensor([0, 1, 4]), torch.zeros(16, 32).to(torch.float8_e4m3fn), torch.ones(1, 1)


@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_derivatives_are_refused(stubbed, grad_mode):
    """A dual tensor does not require a gradient; its tangent must not be lost."""
    import quant_2bit_b200 as q
    x, w, off, f8, s = _operands()
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for f, args in ((q.grouped_linear, (dual(x), w, off)), (q.grouped_linear, (x, dual(w), off)),
                        (q.fp8_linear, (dual(x), f8, s)), (q.fp8_linear, (dual(x.view(2, 2, 32)), f8, s)),
                        (q.fp8_linear, (x, f8, dual(s)))):
            with pytest.raises(NotImplementedError):
                f(*args)
        assert q.grouped_linear(x, w, off).shape == (4, 16)          # nothing to lose
        assert q.fp8_linear(x, f8, s).shape == (4, 16)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda a: q.grouped_linear(a, w, off), (x,), (x,))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda a: q.grouped_linear(a, w, off))(x.view(2, 2, 32))


def test_fp8_matmul_refuses_derivatives(stubbed):
    """It has none: what would need one is refused, not dropped."""
    import quant_2bit_b200 as q
    x, _, _, f8, s = _operands()
    xq, xs = x.to(torch.float8_e4m3fn), torch.ones(4, 1)
    for args in ((xq, xs.clone().requires_grad_(), f8, s), (xq.clone().requires_grad_(), xs, f8, s),
                 (xq, xs, f8, s.clone().requires_grad_())):
        with pytest.raises(AssertionError):
            q.fp8_matmul(*args)
    with forward_ad.dual_level(), torch.no_grad():
        for args in ((xq, forward_ad.make_dual(xs, xs.clone()), f8, s),
                     (xq, xs, f8, forward_ad.make_dual(s, s.clone()))):
            with pytest.raises(AssertionError):
                q.fp8_matmul(*args)
        assert q.fp8_matmul(xq, xs, f8, s).shape == (4, 16)
    with torch.no_grad():
        assert q.fp8_matmul(xq, xs.clone().requires_grad_(), f8, s).shape == (4, 16)
    assert stubbed == ["bcjr_fp8_mm"] * 2


def test_only_what_the_backward_pass_reads_is_kept(stubbed):
    """The rows' gradient reads the weight only, the weight's the rows only:
    the other operand is not held, and may be changed in place."""
    import quant_2bit_b200 as q
    x, w, off, _, _ = _operands()
    for need_x, need_w in ((True, False), (False, True), (True, True)):
        x, w = x.detach().clone().requires_grad_(need_x), w.detach().clone().requires_grad_(need_w)
        kept = []

        def pack(t):
            kept.append(t)
            return t

        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            y = q.grouped_linear(x, w, off)
        assert [any(t.data_ptr() == k.data_ptr() for k in kept) for t in (x, w)] == [need_w, need_x]
        if not (need_x and need_w):
            (w if need_w else x).detach().zero_()      # the one that has the gradient: not read by it
        grads = torch.autograd.grad(y, [t for t in (x, w) if t.requires_grad], torch.zeros_like(y))
        assert [g.shape for g in grads] == [t.shape for t in (x, w) if t.requires_grad]
    assert stubbed == ["bcjr_grouped_mm", "bcjr_grouped_backward"] * 3


def test_rows_further_apart_than_the_library_takes_are_copied():
    from quant_2bit_b200 import linear
    near = torch.empty(2, 1 << 32, device="meta", dtype=torch.bfloat16)[:, :32]
    far = torch.empty(2, (1 << 32) + 8, device="meta", dtype=torch.bfloat16)[:, :32]
    assert linear._rows(near)[1] == 1 << 32
    rows, step = linear._rows(far)
    assert step == 32 and rows.is_contiguous()


# A gradient against differences: the product f is linear in each operand, so
# <dy, f(d)> = <gradient, d> for every displacement d.  Along the gradient itself
# (64 bits, rounded to the type) both sides are a sum of squares, and what the
# roundings can move them by is about 1 % of it in bf16: every f and every
# gradient is off by half a step, eps / 2 of its size, and by 2^-23 of the
# products' magnitudes for each of its `depth` products.


def difference_holds(dy, f, f_mag, f_depth, grad, grad_mag, grad_depth, d):
    lhs, rhs = dy.double() * f.double(), grad.double() * d.double()
    half = torch.finfo(f.dtype).eps / 2
    tol = half * float(lhs.abs().sum() + rhs.abs().sum()) * (1 + 2 * half)
    tol += 2.0 ** -23 * float((dy.double().abs() * f_mag * f_depth).sum() + (d.double().abs() * grad_mag * grad_depth).sum())
    return abs(float(lhs.sum() - rhs.sum())) <= tol


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_the_difference_check_tells_wrong_gradients(dtype):
    """The check that the GPU test uses: right gradients pass; a zero, negated,
    halved, doubled or partly missing one does not, for several inputs."""
    for seed in range(20):
        g = torch.Generator().manual_seed(seed)
        x, w, dy = torch.randn(301, 112, generator=g), torch.randn(96, 112, generator=g) / 112 ** 0.5, torch.randn(301, 96, generator=g)
        x, w, dy = (t.to(dtype).double() for t in (x, w, dy))
        for grad64, mag, depth, product, product_depth in (
                (dy @ w, dy.abs() @ w.abs(), 96, lambda d: d @ w.t(), 112),
                (dy.t() @ x, dy.abs().t() @ x.abs(), 301, lambda d: x @ d.t(), 112)):
            d = grad64.to(dtype)
            f_mag = d.double().abs() @ w.abs().t() if depth == 96 else x.abs() @ d.double().abs().t()
            f, grad = product(d.double()).to(dtype), grad64.to(dtype)
            missing = grad.clone()
            missing[-len(grad) // 5:] = 0
            assert difference_holds(dy, f, f_mag, product_depth, grad, mag, depth, d)
            for wrong in (torch.zeros_like(grad), -grad, grad / 2, grad * 2, missing):
                assert not difference_holds(dy, f, f_mag, product_depth, wrong, mag, depth, d)


def test_fp8_linear_refuses_before_its_quantizer_runs(lib):
    """What only the product can refuse is refused first too: the workspace of a
    refused call is not written (without a GPU a launch would be the error)."""
    def call(x=P, ld=64, w=P, s=P, off=P, off_size=4, T=40, E=2, N=32, K=64, out=P, status=None):
        return lib.bcjr_fp8_linear(x, ld, 0, w, s, off, off_size, T, E, N, K, 0, out, P, 1 << 20, status, None)

    for bad in (dict(w=None), dict(s=None), dict(out=None)):
        assert call(**bad) == NULL, bad
    for bad in (dict(N=24), dict(N=1 << 25), dict(E=0), dict(E=1025), dict(off=None), dict(off_size=2)):
        assert call(**bad) == SHAPE, bad
    for bad in (dict(w=P + 8), dict(out=P + 8), dict(s=P + 2), dict(off=P + 4, off_size=8), dict(status=P + 2)):
        assert call(**bad) == ALIGN, bad
