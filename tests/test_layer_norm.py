"""Layer norm with trained weight and bias (graspo_b200/ops/layer_norm.py) against
the definition in 64 bits, element by element, and its gradients against differences.

Tolerances, with u = 2^-24 for fp32 arithmetic and the storage type's rounding
(bf16 2^-8, fp16 2^-11, fp32 2^-24).  A row's sums are chains of at most
``k = 64 + H / 1024`` additions, so the mean is off by k u mean|x| and the
variance relatively by k u (a shift of the mean enters it squared).  The
normalised value n carries rstd times the mean's error and (k + 8) u of itself;
y, dx and the column sums follow from n by the formulas below, with a column's
chain of ``64 + rows / 100`` additions."""

import pytest
import torch

U = 2.0 ** -24
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 1e-38, torch.float16: 2.0 ** -25, torch.float32: 1e-38}


def _case(rows, H, dtype, param=None, seed=0, device="cuda"):
    g = torch.Generator().manual_seed(seed + rows + H)
    x = torch.randn(rows, H, generator=g) * (0.2 + torch.rand(rows, 1, generator=g)) + torch.randn(rows, 1, generator=g)
    w, b = 1 + 0.2 * torch.randn(H, generator=g), 0.3 * torch.randn(H, generator=g)
    dy = torch.randn(rows, H, generator=g)
    param = param or dtype
    return x.to(device, dtype), w.to(device, param), b.to(device, param), dy.to(device, dtype)


def _oracle(x, w, b, dy, eps):
    dt, pt = x.dtype, w.dtype
    rows, H = x.shape
    x, w, b, dy = (t.double() for t in (x, w, b, dy))
    k = 64 + H / 1024
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    rstd = 1 / torch.sqrt(c.square().mean(-1, keepdim=True) + eps)
    n = c * rstd
    a = dy * w
    ma, man = a.mean(-1, keepdim=True), (a * n).mean(-1, keepdim=True)
    y, dx = n * w + b, rstd * (a - ma - n * man)
    dw, db = (dy * n).sum(0), dy.sum(0)
    en = rstd * k * U * x.abs().mean(-1, keepdim=True) + n.abs() * (k + 8) * U + 2 * U * rstd * x.abs()
    ey = w.abs() * en + 2 * U * ((n * w).abs() + b.abs())
    eman = (a.abs() * en).mean(-1, keepdim=True) + k * U * (a * n).abs().mean(-1, keepdim=True)
    size = a.abs() + a.abs().mean(-1, keepdim=True) + (n * man).abs()
    edx = rstd * (k * U * a.abs().mean(-1, keepdim=True) + en * man.abs() + n.abs() * eman + (k + 12) * U * size)
    chain = (64 + rows / 100) * U
    edw = (dy.abs() * en).sum(0) + chain * (dy * n).abs().sum(0)
    edb = chain * dy.abs().sum(0)
    stored = lambda v, e, t: e + ROUND[t] * (v.abs() + e) + TINY[t]  # noqa: E731
    return (y, dx, dw, db), (stored(y, ey, dt), stored(dx, edx, dt), stored(dw, edw, pt), stored(db, edb, pt))


def _within(got, want, bound, what):
    assert got.shape == want.shape
    off = (got.double() - want).abs() - bound
    assert bool((off <= 0).all()), f"{what}: {int((off > 0).sum())} values outside, worst by {float(off.max()):.3g}"


SHAPES = [(1, 1), (1, 8), (3, 7), (5, 64), (256, 1152), (33, 160), (1000, 136), (7, 1280), (9, 1288), (17, 1001),
          (40, 4097), (3, 8192), (2, 16384), (5, 16400), (2, 40000), (2500, 72), (65, 515)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,H", SHAPES)
def test_forward_backward_against_64_bits(rows, H, dtype):
    from graspo_b200.ops.layer_norm import layer_norm_backward, layer_norm_forward

    x, w, b, dy = _case(rows, H, dtype)
    y, mean, rstd = layer_norm_forward(x, w, b, 1e-6)
    got = (y, *layer_norm_backward(dy, x, w, mean, rstd))
    want, bound = _oracle(x, w, b, dy, 1e-6)
    for name, g, v, e in zip(("y", "dx", "dw", "db"), got, want, bound):
        _within(g, v, e, name)
    again = layer_norm_backward(dy, x, w, mean, rstd)
    assert all(torch.equal(p, q) for p, q in zip(got[1:], again)), "two calls differ"


@pytest.mark.gpu
def test_many_rows():
    from graspo_b200.ops.layer_norm import layer_norm_backward, layer_norm_forward

    x, w, b, dy = _case(30011, 264, torch.bfloat16)
    y, mean, rstd = layer_norm_forward(x, w, b, 1e-6)
    want, bound = _oracle(x, w, b, dy, 1e-6)
    for name, g, v, e in zip(("y", "dx", "dw", "db"), (y, *layer_norm_backward(dy, x, w, mean, rstd)), want, bound):
        _within(g, v, e, name)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,H,dtype", [(4736, 512, torch.bfloat16), (4741, 1152, torch.bfloat16),
                                          (9999, 2048, torch.float16), (4801, 1024, torch.float32),
                                          (20001, 640, torch.float32), (15000, 1160, torch.bfloat16)])
def test_rows_through_the_shared_memory_ring(rows, H, dtype):
    from graspo_b200.ops._ext import check_errors
    from graspo_b200.ops.layer_norm import layer_norm_backward, layer_norm_forward

    x, w, b, dy = _case(rows, H, dtype)
    y, mean, rstd = layer_norm_forward(x, w, b, 1e-6)
    want, bound = _oracle(x, w, b, dy, 1e-6)
    got = (y, *layer_norm_backward(dy, x, w, mean, rstd))
    for name, g, v, e in zip(("y", "dx", "dw", "db"), got, want, bound):
        _within(g, v, e, name)
    gap = torch.zeros(rows, H + 16, device="cuda", dtype=dtype)      # rows with a gap
    gap[:, :H] = x
    again = layer_norm_backward(dy, gap[:, :H], w, mean, rstd)
    assert all(torch.equal(p, q) for p, q in zip(got[1:], again))
    check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_fp32_parameters_and_autograd(dtype):
    from graspo_b200.ops.layer_norm import layer_norm

    x, w, b, dy = _case(50, 192, dtype, param=torch.float32)
    leaves = [t.clone().requires_grad_(True) for t in (x.view(5, 10, 192), w, b)]
    y = layer_norm(*leaves, 1e-5)
    y.backward(dy.view(5, 10, 192))
    want, bound = _oracle(x, w, b, dy, 1e-5)
    got = (y.detach().view(50, 192), leaves[0].grad.view(50, 192), leaves[1].grad, leaves[2].grad)
    assert leaves[1].grad.dtype == leaves[2].grad.dtype == torch.float32
    for name, g, v, e in zip(("y", "dx", "dw", "db"), got, want, bound):
        _within(g, v, e, name)


@pytest.mark.gpu
def test_no_bias_and_mixed_parameter_types():
    from graspo_b200.ops.layer_norm import layer_norm

    x, w, b, dy = _case(20, 80, torch.bfloat16)
    leaves = [t.clone().requires_grad_(True) for t in (x, w)]
    y = layer_norm(*leaves)
    y.backward(dy)
    want, bound = _oracle(x, w, torch.zeros_like(b), dy, 1e-6)
    for name, g, v, e in zip(("y", "dx", "dw"), (y.detach(), leaves[0].grad, leaves[1].grad), want, bound):
        _within(g, v, e, name)
    b32 = b.float().requires_grad_(True)
    layer_norm(x, w, b32).backward(dy)
    assert b32.grad.dtype == torch.float32
    _within(b32.grad, want[3], bound[3], "db")


@pytest.mark.gpu
def test_strides_offsets_expanded_gradient_and_stream():
    from graspo_b200.ops.layer_norm import layer_norm_backward, layer_norm_forward

    x, w, b, dy = _case(30, 96, torch.bfloat16)
    y, mean, rstd = layer_norm_forward(x, w, b)
    want = layer_norm_backward(dy, x, w, mean, rstd)
    gap = torch.zeros(30, 104, device="cuda", dtype=x.dtype)
    gap[:, :96] = x
    odd = torch.zeros(30, 99, device="cuda", dtype=x.dtype)
    odd[:, 1:97] = x
    # rows off a 16-byte boundary are walked value by value: the sums are taken in another order
    (_, dxw, dww, dbw), bound = _oracle(x, w, b, dy, 1e-6)
    for view, exact in ((gap[:, :96], True), (odd[:, 1:97], False), (x.T.contiguous().T, True)):
        y2, m2, r2 = layer_norm_forward(view, w, b)
        got = layer_norm_backward(dy, view, w, m2, r2)
        if exact:
            assert torch.equal(y, y2) and all(torch.equal(p, q) for p, q in zip(want, got))
        for g, v, e in zip(got, (dxw, dww, dbw), bound[1:]):
            _within(g, v, e, "gradient")
    one = torch.ones(1, 1, device="cuda", dtype=x.dtype).expand(30, 96)     # sum().backward()'s gradient
    got, full = layer_norm_backward(one, x, w, mean, rstd), layer_norm_backward(one.contiguous(), x, w, mean, rstd)
    assert all(torch.equal(p, q) for p, q in zip(got, full))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer_norm_backward(dy, x, w, *layer_norm_forward(x, w, b)[1:])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(want, got))


@pytest.mark.gpu
def test_offset_rows_keep_their_variance():
    """Values around 1000 with a spread of 1e-2: E[x^2] - mean^2 would lose the variance in fp32."""
    from graspo_b200.ops.layer_norm import layer_norm_forward

    g = torch.Generator().manual_seed(0)
    x = (1000 + 0.01 * torch.randn(6, 512, generator=g)).cuda()
    w, b = torch.ones(512, device="cuda"), torch.zeros(512, device="cuda")
    y, _, _ = layer_norm_forward(x, w, b, 1e-12)
    want, bound = _oracle(x, w, b, torch.zeros_like(x), 1e-12)
    _within(y, want[0], bound[0], "y")
    flat, _, _ = layer_norm_forward(torch.full_like(x, 3.5), w, b, 1e-6)
    assert not flat.any()


@pytest.mark.gpu
def test_non_finite_rows_stay_in_their_rows():
    from graspo_b200.ops.layer_norm import layer_norm_forward

    x, w, b, _ = _case(12, 256, torch.bfloat16)
    clean, _, _ = layer_norm_forward(x, w, b)
    x[3, 5], x[7, 0] = float("nan"), float("inf")
    y, _, _ = layer_norm_forward(x, w, b)
    keep = [i for i in range(12) if i not in (3, 7)]
    assert y[[3, 7]].isnan().all() and torch.equal(y[keep], clean[keep])


@pytest.mark.gpu
def test_no_rows():
    from graspo_b200.ops.layer_norm import layer_norm_backward, layer_norm_forward

    for H in (64, 1288, 40000):
        x, w, b, dy = _case(0, H, torch.bfloat16)
        y, mean, rstd = layer_norm_forward(x, w, b)
        dx, dw, db = layer_norm_backward(dy, x, w, mean, rstd)
        assert y.shape == dx.shape == (0, H) and not dw.any() and not db.any()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_gradients_against_differences(device):
    from graspo_b200.ops.layer_norm import layer_norm

    x, w, b, dy = _case(6, 40, torch.float32, device=device)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    layer_norm(*leaves, 1e-6).backward(dy)
    g = torch.Generator().manual_seed(5)
    _, bound = _oracle(x, w, b, dy, 1e-6)
    for leaf, base, e in zip(leaves, (x, w, b), bound[1:]):
        u = torch.randn(base.shape, generator=g).to(device).double()
        h = 1e-6

        def total(sign):
            p = [t.double() + (sign * h * u if t is base else 0) for t in (x, w, b)]
            c = p[0] - p[0].mean(-1, keepdim=True)
            n = c / torch.sqrt(c.square().mean(-1, keepdim=True) + 1e-6)
            return float(((n * p[1] + p[2]) * dy.double()).sum())

        along = (total(1) - total(-1)) / (2 * h)
        # the difference itself: h^2 times a third derivative of some 10^3, and 64-bit rounding over h
        assert abs(float((leaf.grad.double() * u).sum()) - along) <= float((e * u.abs()).sum()) + 1e-7


def test_cpu_form_matches_64_bits():
    from graspo_b200.ops.layer_norm import layer_norm_backward, layer_norm_forward

    for dtype in (torch.bfloat16, torch.float32):
        x, w, b, dy = _case(9, 100, dtype, device="cpu")
        y, mean, rstd = layer_norm_forward(x, w, b, 1e-6)
        want, bound = _oracle(x, w, b, dy, 1e-6)
        for name, g, v, e in zip(("y", "dx", "dw", "db"), (y, *layer_norm_backward(dy, x, w, mean, rstd)), want, bound):
            _within(g, v, e, name)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_refusals(device):
    from graspo_b200.ops.layer_norm import layer_norm, layer_norm_backward, layer_norm_forward

    x, w, b, dy = _case(4, 16, torch.float32, device=device)
    y, mean, rstd = layer_norm_forward(x, w, b)
    for bad in [lambda: layer_norm(x, w[:8], b), lambda: layer_norm(x, w, b[:8]),
                lambda: layer_norm(x.double(), w.double(), b.double()), lambda: layer_norm(x, w.bfloat16(), b),
                lambda: layer_norm(x[:, :0], w[:0], b[:0]),
                lambda: layer_norm_backward(dy[:3], x, w, mean, rstd),
                lambda: layer_norm_backward(dy.bfloat16(), x, w, mean, rstd),
                lambda: layer_norm_backward(dy, x, w, mean[:2], rstd)]:
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_second_derivatives_are_refused(device):
    """Also where the upstream gradient is a constant, and where a larger loss holds the term."""
    from graspo_b200.ops.layer_norm import layer_norm

    x, w, b, dy = _case(4, 16, torch.float32, device=device)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(*leaves)
    plain = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    grads = torch.autograd.grad(y, leaves, dy, create_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(plain, grads))
    for g in grads:
        for leaf in leaves[:2]:
            with pytest.raises(RuntimeError, match="second derivative"):
                torch.autograd.grad(y.sum() + g.square().sum(), leaf, retain_graph=True)
    y.square().sum().backward()
    assert all(t.grad is not None for t in leaves)


@pytest.mark.gpu
def test_waits_that_give_up_end_the_call():
    """With an error already recorded a wait may give up: the call ends, the error is raised, the next call is right."""
    from graspo_b200.ops._ext import KernelTimeout, check_errors, err_word
    from graspo_b200.ops.layer_norm import layer_norm_backward, layer_norm_forward

    x, w, b, dy = _case(20000, 1152, torch.bfloat16)
    _, mean, rstd = layer_norm_forward(x, w, b)
    want = layer_norm_backward(dy, x, w, mean, rstd)
    check_errors()
    for _ in range(3):
        err_word(x.device)[0] = 1
        layer_norm_backward(dy, x, w, mean, rstd)
        with pytest.raises(KernelTimeout):
            check_errors()
        got = layer_norm_backward(dy, x, w, mean, rstd)
        check_errors()
        assert all(torch.equal(p, q) for p, q in zip(want, got))


@pytest.mark.gpu
def test_rows_too_long_for_the_column_sums_are_refused():
    """Twice the row's length is an int in the backward: the last lengths below 2^30 are refused up front."""
    from graspo_b200.ops.layer_norm import layer_norm_backward, layer_norm_forward

    H = (1 << 30) - 15
    one = torch.ones(1, 1, device="cuda", dtype=torch.bfloat16).expand(1, H)
    with pytest.raises(ValueError):
        layer_norm_forward(one, one[0], None)
    with pytest.raises(ValueError):
        layer_norm_backward(one, one, one[0], torch.zeros(1, device="cuda"), torch.ones(1, device="cuda"))
