"""GPU tests of the linear layers (quant_2bit_b200/linear.py): products grouped
by expert and e4m3 products with block scales, forward and gradients, against
plain products in 64 bits.

Tolerances.  Every result is one sum of `depth` products in fp32, rounded once
to its type: at most half a step, eps / 2 relative, for the rounding, and
depth * 2^-23 of the sum of the products' magnitudes for the sum (2^-23 a
term, twice the half step of a rounded addition: a tensor core may cut instead
of rounding).  e4m3 products add the rounding of the product of the two scales
and of its multiplication: 4 * 2^-23 more.  The products themselves are exact
(bf16, fp16 and e4m3 mantissas fit fp32)."""
import ctypes

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

EPS32 = 2.0 ** -23
F8 = torch.float8_e4m3fn


def _counts_to_offsets(counts, head=0, dtype=torch.int32):
    off = np.concatenate([[0], np.cumsum(counts)]) + head
    return torch.tensor(off, dtype=dtype, device="cuda")


def _close(got, ref, mag, depth, what, extra=0):
    """|got - ref| <= eps/2 |ref| + (depth + extra) 2^-23 mag, plus half the
    type's smallest step (fp16 results can be subnormal)."""
    eps, tiny = torch.finfo(got.dtype).eps, torch.finfo(got.dtype).smallest_normal
    err = (got.double() - ref).abs()
    tol = eps / 2 * ref.abs() * (1 + eps) + (depth + extra) * EPS32 * mag + eps * tiny / 2
    bad = ~(err <= tol)
    assert not bool(bad.any()), (what, int(bad.sum()), float((err - tol).max()))


def _grouped64(x, w, offsets):
    """(y, magnitudes) of the grouped product in 64 bits; zero outside the groups."""
    y = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(y)
    off = offsets.tolist()
    for e in range(w.shape[0]):
        a, b = off[e], off[e + 1]
        y[a:b] = x[a:b].double() @ w[e].double().t()
        mag[a:b] = x[a:b].double().abs() @ w[e].double().abs().t()
    return y, mag


def _wgrad64(dy, x, offsets, E):
    dw = torch.zeros(E, dy.shape[1], x.shape[1], dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(dw)
    off = offsets.tolist()
    for e in range(E):
        a, b = off[e], off[e + 1]
        dw[e] = dy[a:b].double().t() @ x[a:b].double()
        mag[e] = dy[a:b].double().abs().t() @ x[a:b].double().abs()
    return dw, mag


def _inputs(T, E, N, K, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, K, generator=g, device="cuda").to(dtype)
    w = (torch.randn(E, N, K, generator=g, device="cuda") / K ** 0.5).to(dtype)
    dy = torch.randn(T, N, generator=g, device="cuda").to(dtype)
    return x, w, dy


def _check_grouped(x, w, dy, offsets):
    from quant_2bit_b200 import grouped_linear
    x = x.detach().requires_grad_()
    w = w.detach().requires_grad_()
    y = grouped_linear(x, w, offsets)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    E, N, K = w.shape
    ref, mag = _grouped64(x.detach(), w.detach(), offsets)
    _close(y.detach(), ref, mag, K, "y")
    ref, mag = _grouped64(dy, w.detach().transpose(1, 2), offsets)
    _close(dx, ref, mag, N, "dx")
    ref, mag = _wgrad64(dy, x.detach(), offsets, E)
    _close(dw, ref, mag, max(1, int((offsets[1:] - offsets[:-1]).max())), "dw")
    assert y.dtype == dx.dtype == dw.dtype == x.dtype


GROUPS = [
    ([1], 16, 16),
    ([1, 0, 0, 1], 48, 144),
    ([0, 16, 17, 15], 128, 128),
    ([5, 0, 58, 1], 272, 80),                      # 64 rows: the last T of the small tiles
    ([65], 16, 528),
    ([63, 64, 65, 1], 144, 64),
    ([255, 256, 257, 0, 1], 256, 272),
    ([0, 0, 300, 0, 513, 2], 400, 48),
    ([0, 0, 0], 64, 64),
    ([3, 0, 5], 144, 1040),                        # few tiles, long contraction: clusters share
    ([1], 1040, 2064),                             # tiles (forward and rows' gradient)
    ([33], 16, 8208),
    ([0, 64, 0], 528, 512),
    ([7, 33, 0, 64, 12, 1] * 40, 144, 272),        # several tiles and short groups for each block
    ([90, 0, 3, 1, 20, 0, 0, 0, 2], 80, 208),      # more than 64 rows, few to a group
    ([100, 0, 37, 301], 1040, 1168),               # many features: pairs of blocks
    ([300, 5], 2064, 1024),
    ([3, 1, 4, 1, 5, 9, 2, 6, 5, 3, 5, 8, 9, 7, 9, 3] * 5, 32, 96),   # 80 groups
]


# tiles: 0 as the library chooses, 1 few rows, 2 many rows, 3 many rows in pairs of blocks
@pytest.mark.parametrize("tiles", [0, 1, 2, 3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counts,N,K", GROUPS)
def test_grouped_forward_and_gradients(cuda_ok, counts, N, K, dtype, tiles):
    from quant_2bit_b200 import _lib
    T = sum(counts)
    x, w, dy = _inputs(T, len(counts), N, K, dtype, seed=T)
    with _lib.test_option(_lib.OPT_LINEAR_TILES, tiles):
        _check_grouped(x, w, dy, _counts_to_offsets(counts))


def test_many_rows_and_features(cuda_ok):
    """Sizes for which the library takes the large tiles by itself."""
    for counts, N, K, dtype in (([3000, 0, 1501, 77], 1040, 1024, torch.bfloat16),
                                ([2500, 2500], 528, 400, torch.float16)):
        x, w, dy = _inputs(sum(counts), len(counts), N, K, dtype)
        _check_grouped(x, w, dy, _counts_to_offsets(counts))
    x, q, s, w64, dy = _fp8_operands(5000, 0, 1040, 656, torch.bfloat16)
    _check_fp8(x, q, s, w64, dy, None)


@pytest.mark.parametrize("tiles", [1, 2, 3])
@pytest.mark.parametrize("off_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("head,tail", [(7, 0), (0, 9), (70, 130)])
def test_rows_of_no_group_are_zero_and_do_not_count(cuda_ok, head, tail, off_dtype, tiles):
    """Rows before the first and behind the last group: zero output and zero
    gradient, whatever they hold."""
    counts = [33, 0, 70, 5]
    T = head + sum(counts) + tail
    x, w, dy = _inputs(T, 4, 64, 96, torch.bfloat16)
    offsets = _counts_to_offsets(counts, head, off_dtype)
    for t in (x, dy):
        t[:head] = float("nan")
        t[T - tail:] = float("inf")
    from quant_2bit_b200 import _lib
    with _lib.test_option(_lib.OPT_LINEAR_TILES, tiles):
        _check_grouped(x, w, dy, offsets)


@pytest.mark.parametrize("tiles", [1, 2, 3])
def test_non_finite_rows_stay_in_their_group(cuda_ok, tiles):
    """A NaN or infinity in one group's rows reaches that group only, in every
    direction (tiles end inside the next group's rows)."""
    from quant_2bit_b200 import _lib, grouped_linear
    counts = [40, 24, 100, 30]
    x, w, dy = _inputs(194, 4, 48, 80, torch.bfloat16)
    offsets = _counts_to_offsets(counts)
    x[64:164] = float("nan")
    dy[64:164] = float("inf")
    x.requires_grad_()
    w.requires_grad_()
    with _lib.test_option(_lib.OPT_LINEAR_TILES, tiles):
        y = grouped_linear(x, w, offsets)
        dx, dw = torch.autograd.grad(y, (x, w), dy)
    clean = torch.ones(194, dtype=torch.bool, device="cuda")
    clean[64:164] = False
    for t in (y.detach(), dx):
        assert torch.isfinite(t[clean]).all() and not torch.isfinite(t[~clean]).any()
    assert torch.isfinite(dw[[0, 1, 3]]).all() and not torch.isfinite(dw[2]).any()
    x2, dy2 = x.detach().clone(), dy.clone()
    x2[64:164] = 0
    dy2[64:164] = 0
    ref, mag = _wgrad64(dy2, x2, offsets, 4)
    _close(dw[[0, 1, 3]], ref[[0, 1, 3]], mag[[0, 1, 3]], 64, "dw")


def test_strided_transposed_and_misaligned_operands(cuda_ok):
    counts = [20, 3, 50]
    N, K = 64, 48
    offsets = _counts_to_offsets(counts)
    x, w, dy = _inputs(73, 3, N, K, torch.float16)
    wide = torch.full((73, K + 40), float("nan"), dtype=torch.float16, device="cuda")
    wide[:, 8:8 + K] = x
    odd = torch.full((73, K + 3), float("nan"), dtype=torch.float16, device="cuda")
    odd[:, 1:1 + K] = x
    views = [wide[:, 8:8 + K], odd[:, 1:1 + K], x.t().contiguous().t(),
             torch.cat([x.new_zeros(1), x.reshape(-1)])[1:].view(73, K)]
    for v in views:
        _check_grouped(v, w.transpose(1, 2).contiguous().transpose(1, 2), dy, offsets)
    _check_grouped(x, torch.cat([w.new_zeros(3), w.reshape(-1)])[3:].view_as(w),
                   dy[:, :1].expand(73, N), offsets)
    _check_grouped(x, w[:1].expand(3, N, K), dy[:1].expand(73, N), offsets)


def test_gradient_of_a_sum_and_of_one_leaf_only(cuda_ok):
    from quant_2bit_b200 import grouped_linear
    offsets = _counts_to_offsets([9, 30])
    x, w, _ = _inputs(39, 2, 32, 64, torch.bfloat16)
    ones = torch.ones(39, 32, dtype=torch.bfloat16, device="cuda")
    x.requires_grad_()
    grouped_linear(x, w, offsets).sum().backward()
    ref, mag = _grouped64(ones, w.transpose(1, 2), offsets)
    _close(x.grad, ref, mag, 32, "dx")
    w.requires_grad_()
    grouped_linear(x.detach(), w, offsets).sum().backward()
    ref, mag = _wgrad64(ones, x.detach(), offsets, 2)
    _close(w.grad, ref, mag, 30, "dw")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients_against_differences(cuda_ok, dtype):
    """The product is linear in each operand, so a difference quotient is the
    product at the displacement: <dy, f(d)> = <gradient, d>, in 64 bits from
    outputs that are each rounded once (half a step of every term)."""
    from quant_2bit_b200 import grouped_linear
    offsets = _counts_to_offsets([70, 0, 31, 200])
    x, w, dy = _inputs(301, 4, 96, 112, dtype, seed=5)
    d_x, d_w, _ = _inputs(301, 4, 96, 112, dtype, seed=6)
    x.requires_grad_()
    w.requires_grad_()
    dx, dw = torch.autograd.grad(grouped_linear(x, w, offsets), (x, w), dy)
    half = torch.finfo(dtype).eps / 2 + 301 * EPS32 * 50
    for grad, d, f in ((dx, d_x, grouped_linear(d_x, w.detach(), offsets)),
                       (dw, d_w, grouped_linear(x.detach(), d_w, offsets))):
        lhs, rhs = (dy.double() * f.double()), (grad.double() * d.double())
        assert abs(float(lhs.sum() - rhs.sum())) <= half * float(lhs.abs().sum() + rhs.abs().sum())


def test_offsets_outside_the_rows_are_clamped(cuda_ok):
    """Bounds beyond [0, T] are clamped and a decreasing one counts as its
    predecessor: no access leaves the matrices."""
    from quant_2bit_b200 import grouped_linear
    x, w, dy = _inputs(50, 4, 32, 32, torch.bfloat16)
    bad = torch.tensor([-5, 20, 10, 1 << 40, 7], dtype=torch.int64, device="cuda")
    good = torch.tensor([0, 20, 20, 50, 50], dtype=torch.int64, device="cuda")
    for a in (x, w):
        a.requires_grad_()
    got, want = [], []
    for off, to in ((bad, got), (good, want)):
        y = grouped_linear(x, w, off)
        to += [y.detach(), *torch.autograd.grad(y, (x, w), dy)]
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_results_do_not_change_from_run_to_run(cuda_ok):
    from quant_2bit_b200 import fp8_linear, fp8_quantize_weight, grouped_linear
    counts = [0, 700, 3, 41, 256]
    offsets = _counts_to_offsets(counts)
    x, w, dy = _inputs(1000, 5, 272, 336, torch.bfloat16)
    q, s = fp8_quantize_weight(w)
    x.requires_grad_()
    w.requires_grad_()
    first = None
    for _ in range(5):
        y = grouped_linear(x, w, offsets)
        z = fp8_linear(x, q, s, offsets)
        out = [y.detach(), *torch.autograd.grad(y, (x, w), dy), z.detach(),
               *torch.autograd.grad(z, x, dy)]
        first = first or out
        assert all(torch.equal(a, b) for a, b in zip(first, out))


def test_captured_and_replayed_with_other_rows_and_groups(cuda_ok):
    """Forward and backward of both layers in one CUDA graph; replays follow
    what the buffers hold then, the group bounds included."""
    from quant_2bit_b200 import fp8_linear, fp8_quantize_weight, grouped_linear
    T, E, N, K = 150, 4, 64, 80
    x, w, dy = _inputs(T, E, N, K, torch.bfloat16)
    q, s = fp8_quantize_weight(w)
    offsets = _counts_to_offsets([50, 0, 100, 0])
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()

    def step():
        y = grouped_linear(xs, ws, offsets)
        z = fp8_linear(xs, q, s, offsets)
        return [y.detach(), *torch.autograd.grad(y, (xs, ws), dy), z.detach(),
                *torch.autograd.grad(z, xs, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for counts, seed in (([1, 2, 3, 144], 1), ([0, 0, 0, 20], 2), ([40, 40, 40, 30], 3)):
        x2, _, dy2 = _inputs(T, E, N, K, torch.bfloat16, seed)
        with torch.no_grad():
            xs.copy_(x2)
        dy.copy_(dy2)
        offsets.copy_(_counts_to_offsets(counts))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_two_graphs_in_turn_and_other_streams(cuda_ok):
    """Two captured graphs of the 8-bit layer (quantizer, workspace, dependent
    launch) replayed in turn, back to back, each keep their own results."""
    from quant_2bit_b200 import fp8_linear, fp8_quantize_weight
    ops = []
    for seed, (T, N, K) in enumerate(((40, 528, 1040), (700, 272, 400))):
        x, w, _ = _inputs(T, 1, N, K, torch.bfloat16, seed)
        q, s = fp8_quantize_weight(w[0])
        want = fp8_linear(x, q, s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = fp8_linear(x, q, s)
        ops.append((graph, out, want, (x, q, s)))
    for _ in range(20):
        for graph, out, _, _ in ops:
            graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for _, out, want, _ in ops)
    side = torch.cuda.Stream()
    for _ in range(20):
        ops[0][0].replay()
        with torch.cuda.stream(side):
            ops[1][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for _, out, want, _ in ops)


def test_other_streams_side_by_side(cuda_ok):
    from quant_2bit_b200 import grouped_linear
    x, w, _ = _inputs(600, 3, 256, 512, torch.bfloat16)
    offsets = _counts_to_offsets([100, 450, 50])
    want = grouped_linear(x, w, offsets)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            outs.append(grouped_linear(x, w, offsets))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_offsets_beyond_32_bits(cuda_ok):
    """Outputs and weights of more than 2^31 elements (2^32 bytes)."""
    from quant_2bit_b200 import grouped_linear
    T, N, K = 2_150_000, 1008, 16
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(T, K, generator=g, device="cuda").to(torch.bfloat16)
    w = torch.randn(2, N, K, generator=g, device="cuda").to(torch.bfloat16)
    offsets = torch.tensor([0, T - 300, T], device="cuda")
    y = grouped_linear(x, w, offsets)
    assert y.numel() > 2 ** 31
    for e, rows in ((0, slice(T - 700, T - 300)), (1, slice(T - 300, T)), (0, slice(0, 300))):
        ref = x[rows].double() @ w[e].double().t()
        _close(y[rows], ref, x[rows].double().abs() @ w[e].double().abs().t(), K, "y")
    del y
    E, N, K = 1024, 2064, 1024
    w = torch.empty(E, N, K, dtype=torch.bfloat16, device="cuda")
    w[-2:] = torch.randn(2, N, K, generator=g, device="cuda")
    assert w.numel() > 2 ** 31
    x = torch.randn(40, K, generator=g, device="cuda").to(torch.bfloat16).requires_grad_()
    offsets = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    offsets[-2], offsets[-1] = 17, 40
    dy = torch.randn(40, N, generator=g, device="cuda").to(torch.bfloat16)
    w.requires_grad_()
    y = grouped_linear(x, w, offsets)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    for e, rows in ((E - 2, slice(0, 17)), (E - 1, slice(17, 40))):
        a, b, d = x.detach()[rows].double(), w.detach()[e].double(), dy[rows].double()
        _close(y.detach()[rows], a @ b.t(), a.abs() @ b.abs().t(), K, "y")
        _close(dx[rows], d @ b, d.abs() @ b.abs(), N, "dx")
        _close(dw[e], d.t() @ a, d.abs().t() @ a.abs(), 23, "dw")
    assert not dw[:E - 2].any()


def test_grouped_refusals(cuda_ok):
    from quant_2bit_b200 import grouped_linear
    x, w, _ = _inputs(10, 2, 32, 48, torch.bfloat16)
    off = _counts_to_offsets([4, 6])
    for args in ((x.float(), w.float(), off), (x, w.half(), off), (x, w, off.float())):
        with pytest.raises(ValueError):
            grouped_linear(*args)
    for args in ((x, w, off[:2]), (x, w[:, :, :32].contiguous(), off), (x[:, :40], w[:, :, :40], off),
                 (x, w[:, :8], off), (x[0], w, off), (x, w[0], off),
                 (x, w.new_zeros(1025, 32, 48), torch.zeros(1026, dtype=torch.int32, device="cuda"))):
        with pytest.raises(AssertionError):
            grouped_linear(*args)
    for args in ((x.cpu(), w, off), (x, w.cpu(), off), (x, w, off.cpu())):
        with pytest.raises(RuntimeError, match="CUDA"):
            grouped_linear(*args)
    x.requires_grad_()
    g = torch.autograd.grad(grouped_linear(x, w, off).float().sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        g.sum().backward()          # no second derivative


# --------------------------------------------------------------------------
# e4m3


def _quantize_plain(x, rows_of_block):
    """The quantizers' definition with elementary fp32 operations."""
    n, k = x.shape
    xp = torch.nn.functional.pad(x.float(), (0, -k % 128, 0, -n % rows_of_block))
    b = xp.view(xp.shape[0] // rows_of_block, rows_of_block, xp.shape[1] // 128, 128)
    amax = b.abs().amax(3).amax(1).clamp(min=2.0 ** -100)
    inv = torch.full_like(amax, 448.0) * torch.reciprocal(amax)
    scale = amax * torch.full_like(amax, float(np.float32(1) / np.float32(448)))
    q = (b * inv[:, None, :, None]).to(F8).view(xp.shape)[:n, :k]
    return q, scale


def _expand(q, scale, rows_of_block):
    s = scale.double().repeat_interleave(128, 1)[:, :q.shape[1]]
    return q.double() * s.repeat_interleave(rows_of_block, 0)[:q.shape[0]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,k", [(1, 16), (3, 128), (130, 144), (257, 2048), (64, 272), (1000, 80)])
def test_quantizers_follow_their_definition_bit_for_bit(cuda_ok, n, k, dtype):
    from quant_2bit_b200 import fp8_quantize_rows, fp8_quantize_weight
    g = torch.Generator(device="cuda").manual_seed(n + k)
    x = (torch.randn(n, k, generator=g, device="cuda") *
         torch.exp(3 * torch.randn(n, 1, generator=g, device="cuda"))).to(dtype)
    x[0, :16] = 0
    for f, rows in ((fp8_quantize_rows, 1), (fp8_quantize_weight, 128)):
        q, s = f(x)
        qr, sr = _quantize_plain(x, rows)
        assert q.shape == x.shape and q.dtype == F8 and torch.equal(s, sr)
        assert torch.equal(q.view(torch.uint8), qr.contiguous().view(torch.uint8))
        # half a step: 2^-4 relative, 2^-10 of the scale among the subnormals
        err = (_expand(q, s, rows) - x.double()).abs()
        sx = _expand(torch.ones_like(q, dtype=torch.float64), s, rows)
        assert bool((err <= (2.0 ** -4 * x.double().abs()).maximum(2.0 ** -10 * sx) * (1 + 2.0 ** -20)).all())


def test_quantizers_at_the_edges(cuda_ok):
    """Zero blocks, the type's extremes, NaN and infinity, empty inputs, leading
    axes, strides, and the blocks of several weights."""
    from quant_2bit_b200 import fp8_quantize_rows, fp8_quantize_weight
    q, s = fp8_quantize_rows(torch.zeros(2, 256, device="cuda"))
    assert not q.float().any() and bool((s == 2.0 ** -100 * float(np.float32(1) / np.float32(448))).all())
    x = torch.ones(4, 256, device="cuda")
    x[0, 3], x[1, 130] = float("nan"), float("-inf")
    x[2, 5], x[3, 7] = torch.finfo(torch.float32).max, 1e-40
    q, s = fp8_quantize_rows(x)
    qf = q.float()
    assert qf[0, :128].isnan().all() and s[0, 0].isnan() and (qf[0, 128:] == 448).all()
    assert s[1, 1].isinf() and qf[1, 130].isnan() and not qf[1, 131:].any() and (qf[1, :128] == 448).all()
    assert qf[2, 5] == 448 and qf[3, 7] == 0
    for f in (fp8_quantize_rows, fp8_quantize_weight):
        qr, sr = _quantize_plain(x[2:], 1 if f is fp8_quantize_rows else 128)
        q, s = f(x[2:])
        assert torch.equal(q.float(), qr.float()) and torch.equal(s, sr)
    assert fp8_quantize_rows(torch.zeros(0, 32, device="cuda"))[1].shape == (0, 1)
    x = torch.randn(3, 5, 272, device="cuda").to(torch.bfloat16)
    q, s = fp8_quantize_rows(x)
    assert q.shape == x.shape and s.shape == (3, 5, 3)
    assert torch.equal(q[1].float(), fp8_quantize_rows(x[1])[0].float())
    wide = torch.randn(9, 400, device="cuda")
    for v in (wide[:, 4:148], wide[:, 1:145], wide.t().contiguous().t()[:, :144]):
        assert torch.equal(fp8_quantize_rows(v)[0].float(), fp8_quantize_rows(v.clone())[0].float())
    w = torch.randn(3, 200, 144, device="cuda")
    q, s = fp8_quantize_weight(w)
    assert s.shape == (3, 2, 2)
    for e in range(3):
        qe, se = fp8_quantize_weight(w[e])
        assert torch.equal(q[e].float(), qe.float()) and torch.equal(s[e], se)


def _fp8_operands(T, E, N, K, dtype, seed=0):
    from quant_2bit_b200 import fp8_quantize_weight
    x, w, dy = _inputs(T, max(E, 1), N, K, dtype, seed)
    x[:, ::37] *= 12
    q, s = fp8_quantize_weight(w if E else w[0])
    w64 = torch.stack([_expand(a, b, 128) for a, b in zip(q.view(-1, N, K), s.view(-1, *s.shape[-2:]))])
    return x, q, s, w64, dy


def _check_fp8(x, q, s, w64, dy, offsets):
    from quant_2bit_b200 import fp8_linear
    x = x.detach().requires_grad_()
    y = fp8_linear(x, q, s, offsets)
    dx = torch.autograd.grad(y, x, dy)[0]
    bounds = torch.tensor([0, x.shape[0]]) if offsets is None else offsets
    N, K = q.shape[-2:]
    for got, rows, w, depth in ((y.detach(), x.detach(), w64, K), (dx, dy, w64.transpose(1, 2), N)):
        rows64 = _expand(*_quantize_plain(rows, 1), 1)
        ref, mag = _grouped64(rows64, w, bounds)
        _close(got, ref, mag, depth, "y" if depth == K else "dx", extra=4)
    assert y.dtype == dx.dtype == x.dtype


@pytest.mark.parametrize("tiles", [0, 1, 2])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,N,K", [(1, 16, 16), (1, 128, 256), (17, 144, 272), (64, 2000, 400),
                                   (65, 48, 128), (300, 272, 1040), (513, 128, 144), (37, 48, 4240), (1, 2064, 528),
                                   (64, 144, 1280), (200, 656, 304), (129, 16, 16), (2, 1040, 2064),
                                   (31, 272, 4112), (32, 4112, 144), (33, 144, 4112)])
def test_fp8_linear_forward_and_gradient(cuda_ok, T, N, K, dtype, tiles):
    from quant_2bit_b200 import _lib
    x, q, s, w64, dy = _fp8_operands(T, 0, N, K, dtype, seed=T)
    with _lib.test_option(_lib.OPT_LINEAR_TILES, tiles):
        _check_fp8(x, q, s, w64, dy, None)


@pytest.mark.parametrize("tiles", [0, 1, 2])
@pytest.mark.parametrize("counts,N,K", [([3, 0, 1, 12], 144, 272), ([130, 0, 300, 70], 272, 144),
                                        ([0, 0], 128, 128), ([257, 1], 128, 384),
                                        ([9, 0, 1], 144, 2064), ([1, 5, 0, 20], 400, 272), ([0, 26], 2064, 656),
                                        ([90, 0, 3, 1, 20, 0, 0, 0, 2], 208, 272)])
def test_fp8_linear_by_expert(cuda_ok, counts, N, K, tiles):
    T = sum(counts) + 6
    x, q, s, w64, dy = _fp8_operands(T, len(counts), N, K, torch.bfloat16, seed=T)
    x[:2] = float("nan")
    x[T - 4:] = float("inf")
    dy[:2] = float("inf")
    offsets = _counts_to_offsets(counts, head=2, dtype=torch.int64)
    inside = slice(2, T - 4)
    from quant_2bit_b200 import _lib, fp8_linear
    xg = x.detach().requires_grad_()
    with _lib.test_option(_lib.OPT_LINEAR_TILES, tiles):
        y = fp8_linear(xg, q, s, offsets)
        dx = torch.autograd.grad(y, xg, dy)[0]
    assert not y[:2].any() and not y[T - 4:].any() and not dx[:2].any() and not dx[T - 4:].any()
    for got, rows, w, depth in ((y.detach(), x, w64, K), (dx, dy, w64.transpose(1, 2), N)):
        rows64 = _expand(*_quantize_plain(rows[inside].contiguous(), 1), 1)
        ref, mag = _grouped64(rows64, w, offsets - 2)
        _close(got[inside], ref, mag, depth, "fp8", extra=4)


def test_fp8_matmul_takes_any_scales(cuda_ok):
    """Scales that no quantizer made: signs, wide ranges, strided row scales."""
    from quant_2bit_b200 import fp8_matmul
    T, N, K = 90, 160, 400
    g = torch.Generator(device="cuda").manual_seed(3)
    xq = (8 * torch.randn(T, K, generator=g, device="cuda")).to(F8)
    q = (8 * torch.randn(N, K, generator=g, device="cuda")).to(F8)
    xs = torch.randn(T, 4, generator=g, device="cuda") * torch.tensor([1e-3, 1.0, 0.0, 10.0], device="cuda")
    ws = torch.randn(2, 4, generator=g, device="cuda")
    a, b = _expand(xq, xs, 1), _expand(q, ws, 128)
    for s in (xs, xs.t().contiguous().t(), xs[:, :1].expand(T, 4)):
        a = _expand(xq, s, 1)
        for dt in (torch.bfloat16, torch.float16):
            _close(fp8_matmul(xq, s, q, ws, out_dtype=dt), a @ b.t(), a.abs() @ b.abs().t(), K, "y", extra=4)
    for t in (1, 17):          # few quantized rows (the layer quantizes those itself)
        _close(fp8_matmul(xq[:t], xs[:t], q, ws), _expand(xq[:t], xs[:t], 1) @ b.t(),
               _expand(xq[:t], xs[:t], 1).abs() @ b.abs().t(), K, "y", extra=4)
    wide = torch.zeros(T, K + 48, dtype=torch.uint8, device="cuda").view(F8)
    wide[:, 16:16 + K] = xq
    assert torch.equal(fp8_matmul(wide[:, 16:16 + K], xs, q, ws), fp8_matmul(xq, xs, q, ws))
    assert torch.equal(fp8_matmul(wide[:, 16:16 + K], xs[:1].expand(T, 4), q, ws),
                       fp8_matmul(xq, xs[:1].repeat(T, 1), q, ws))


def test_few_and_many_rows_of_the_fp8_layer_agree(cuda_ok):
    """Up to 32 rows one kernel quantizes and multiplies, above two do: the same
    codes, scales and (in 64 columns) sums, also for strided rows, extreme and
    non-finite values."""
    from quant_2bit_b200 import _lib, fp8_linear, fp8_matmul, fp8_quantize_rows, fp8_quantize_weight
    g = torch.Generator(device="cuda").manual_seed(9)
    for T, N, K in ((1, 144, 272), (13, 528, 2064), (32, 16, 144)):
        wide = torch.randn(T, K + 24, generator=g, device="cuda").to(torch.bfloat16)
        x = wide[:, 8:8 + K]
        x[0, :16] = 0
        x[T // 2, 3] = 3e38
        if T > 2:
            x[1], x[2, 5] = 1e-40, float("inf")
            x[T - 1, K - 1] = float("nan")
        q, s = fp8_quantize_weight(torch.randn(N, K, generator=g, device="cuda"))
        with _lib.test_option(_lib.OPT_LINEAR_TILES, 1):
            want = fp8_matmul(*fp8_quantize_rows(x), q, s)
        got = fp8_linear(x, q, s)
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


def test_fp8_leading_axes_and_empty(cuda_ok):
    from quant_2bit_b200 import fp8_linear
    x, q, s, w64, dy = _fp8_operands(24, 0, 48, 144, torch.bfloat16)
    want = fp8_linear(x, q, s)
    assert torch.equal(fp8_linear(x.view(2, 3, 4, 144), q, s).view(24, 48), want)
    assert torch.equal(fp8_linear(x[5], q, s), want[5])
    x0 = x[:0].requires_grad_()
    y0 = fp8_linear(x0, q, s)
    assert y0.shape == (0, 48) and torch.autograd.grad(y0.sum(), x0)[0].shape == (0, 144)


def test_fp8_refusals(cuda_ok):
    from quant_2bit_b200 import fp8_linear, fp8_matmul, fp8_quantize_rows, fp8_quantize_weight
    x, q, s, _, _ = _fp8_operands(10, 0, 48, 144, torch.bfloat16)
    off = torch.tensor([0, 10], device="cuda")
    for f, a in ((fp8_linear, (x.float(), q, s)), (fp8_linear, (x, q.float(), s)),
                 (fp8_linear, (x, q, s.double())), (fp8_quantize_rows, (q,)),
                 (fp8_quantize_weight, (q,)), (fp8_matmul, (x, s, q, s)),
                 (fp8_matmul, (*fp8_quantize_rows(x), q, s, None, torch.float32))):
        with pytest.raises(ValueError):
            f(*a)
    for f, a in ((fp8_linear, (x[:, :128], q, s)), (fp8_linear, (x, q, s[:, :1])),
                 (fp8_linear, (x, q, s, off)), (fp8_linear, (x, q[None], s[None])),
                 (fp8_linear, (x[None], q[None], s[None], off)),
                 (fp8_linear, (x, q, s.clone().requires_grad_())),
                 (fp8_quantize_rows, (x[:, :24],)), (fp8_quantize_weight, (x[:, :24],)),
                 (fp8_quantize_weight, (x[0],))):
        with pytest.raises(AssertionError):
            f(*a)
    with pytest.raises(RuntimeError, match="CUDA"):
        fp8_quantize_rows(x.cpu())


# --------------------------------------------------------------------------
# together, and failures


def test_quantized_experts_train_through_the_grouped_product(cuda_ok):
    """The MoE layer path: experts quantized together, their product by groups,
    a frozen e4m3 projection behind it, and gradients back to the latent
    weights, against the same steps expert by expert."""
    from quant_2bit_b200 import fp8_linear, fp8_quantize_weight
    from quant_2bit_b200 import quant
    E, N, K = 3, 32, 64
    g = torch.Generator(device="cuda").manual_seed(2)
    cb = torch.randn(256, 1, generator=g, device="cuda")
    weights = [torch.randn(N, K, generator=g, device="cuda").requires_grad_() for _ in range(E)]
    sl = [torch.tensor(quant.make_sign_vector(N, e), device="cuda") for e in range(E)]
    sr = [torch.tensor(quant.make_sign_vector(K, 9 + e), device="cuda") for e in range(E)]
    x = torch.randn(50, K, generator=g, device="cuda").to(torch.bfloat16).requires_grad_()
    frozen = fp8_quantize_weight(torch.randn(48, N, generator=g, device="cuda"))
    dy = torch.randn(50, 48, generator=g, device="cuda").to(torch.bfloat16)
    offsets = _counts_to_offsets([20, 0, 30])
    h = quant.bcjr_experts_linear(x, offsets, weights, sl, sr, cb, 0.5)
    y = fp8_linear(h, *frozen)
    grads = torch.autograd.grad(y, [x, *weights], dy)
    assert y.shape == (50, 48)

    wq = [quant.bcjr_quantize_weight(w, a, b, cb, 0.5) for w, a, b in zip(weights, sl, sr)]
    w16 = torch.stack([w.detach() for w in wq]).to(torch.bfloat16)
    ref, mag = _grouped64(x.detach(), w16, offsets)
    _close(h.detach(), ref, mag, K, "h")
    dh = torch.autograd.grad(y := fp8_linear(hh := h.detach().requires_grad_(), *frozen), hh, dy)[0]
    ref, mag = _grouped64(dh, w16.transpose(1, 2), offsets)
    _close(grads[0], ref, mag, N, "dx")
    dw, _ = _wgrad64(dh, x.detach(), offsets, E)
    # the cast's gradient is the bf16 weight gradient; from there on the same fp32 kernels
    want = torch.autograd.grad(wq, weights, [d.to(torch.bfloat16).float() for d in dw])
    for a, b in zip(grads[1:], want):
        # half a bf16 step of dw either way, through a linear map: compare in norm
        assert float((a - b).norm()) <= 2.0 ** -8 * float(b.norm()) + 1e-12
    assert not grads[2].any()


def test_a_wait_that_runs_out_is_reported(cuda_ok):
    """With the first load of block 0 withheld, the kernel gives up after its
    limit, its outputs are NaN and the status word says so."""
    from quant_2bit_b200 import _lib
    lib = _lib.load()
    x, w, dy = _inputs(20, 1, 32, 64, torch.bfloat16)
    status = torch.full((1,), 77, dtype=torch.int32, device="cuda")
    y = torch.zeros(20, 32, dtype=torch.bfloat16, device="cuda")
    dw = torch.zeros(1, 32, 64, dtype=torch.bfloat16, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream

    dx = torch.zeros(20, 64, dtype=torch.bfloat16, device="cuda")

    def forward():
        return lib.bcjr_grouped_mm(x.data_ptr(), 64, w.data_ptr(), None, 0, 20, 1, 32, 64, 0,
                                   y.data_ptr(), status.data_ptr(), stream)

    def backward(rows, weights):
        return lib.bcjr_grouped_backward(dy.data_ptr(), 32, x.data_ptr(), 64, w.data_ptr(), None, 0, 20,
                                         1, 32, 64, 0, dx.data_ptr() if rows else None,
                                         dw.data_ptr() if weights else None, status.data_ptr(), stream)

    from quant_2bit_b200 import fp8_quantize_weight
    q, s = fp8_quantize_weight(torch.randn(32, 64, device="cuda"))
    x8 = torch.randn(70, 64, device="cuda").to(torch.bfloat16)
    y8 = torch.zeros(70, 32, dtype=torch.bfloat16, device="cuda")
    ws = torch.empty(lib.bcjr_fp8_linear_workspace_bytes(70, 64), dtype=torch.uint8, device="cuda")

    def fp8(rows):
        return lib.bcjr_fp8_linear(x8.data_ptr(), 64, 0, q.data_ptr(), s.data_ptr(), None, 0, rows, 1,
                                   32, 64, 0, y8.data_ptr(), ws.data_ptr(), ws.numel(),
                                   status.data_ptr(), stream)

    # pairs of blocks: the first tile of 256 features (x's rows serve as dy's too)
    wide = torch.zeros(100, 1024, dtype=torch.bfloat16, device="cuda")
    w_wide = torch.randn(1024, 64, device="cuda").to(torch.bfloat16)
    x_wide = torch.randn(100, 1024, device="cuda").to(torch.bfloat16)
    narrow = torch.randn(100, 64, device="cuda").to(torch.bfloat16)
    dw_wide = torch.zeros(64, 1024, dtype=torch.bfloat16, device="cuda")

    def forward_pair():
        return lib.bcjr_grouped_mm(narrow.data_ptr(), 64, w_wide.data_ptr(), None, 0, 100, 1, 1024, 64, 0,
                                   wide.data_ptr(), status.data_ptr(), stream)

    def weights_pair():
        return lib.bcjr_grouped_backward(narrow.data_ptr(), 64, x_wide.data_ptr(), 1024, None, None, 0, 100,
                                         1, 64, 1024, 0, None, dw_wide.data_ptr(), status.data_ptr(), stream)

    def forced(tiles, call):
        def run():
            with _lib.test_option(_lib.OPT_LINEAR_TILES, tiles):
                return call()
        return run

    for call, out in ((forced(3, forward_pair), wide[:, :256]), (weights_pair, dw_wide[:, :256]),
                      (forced(2, forward), y), (forced(2, lambda: fp8(70)), y8),
                      (forward, y), (lambda: backward(1, 0), dx), (lambda: backward(0, 1), dw),
                      (lambda: backward(1, 1), dw), (lambda: fp8(20), y8[:20])):
        with _lib.test_option(_lib.OPT_TEST_DROP_SENDS, 1):
            assert call() == 0
            assert lib.bcjr_ws_status(ctypes.c_void_p(status.data_ptr()), stream) == _lib.BCJR_ERR_TIMEOUT
        assert out.isnan().all()
        assert call() == 0
        assert lib.bcjr_ws_status(ctypes.c_void_p(status.data_ptr()), stream) == 0
        assert torch.isfinite(out).all()
