"""Cross entropy over a vocabulary projection (graspo_b200/ops/cross_entropy.py):
losses and both gradients against the definition in 64 bits, element by element.

Tolerances.  With bf16 operands every product is exact in fp32.  The tensor cores
add 16 products per step, so a logit is off by at most
``delta = (H / 16 + 16) * 2^-22 * max sum_k |h_k W_k|`` (one rounding or
truncation of a partial sum per step).  The loss is the difference of two such
values plus a log-sum-exp of fp32 exponentials (relative error below 2^-18).
An entry of the softmax gradient d carries the logit's and the log-sum-exp's
error (relative 3 delta + 2^-17) and one rounding to bf16 (8 significant bits:
2^-8); dh and dW sum entries with those errors and are rounded to bf16 once more.
"""

import contextlib
import math

import pytest
import torch

IGNORE = -100


def _case(T, H, V, valid, seed=0, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(T, H, generator=g).to(torch.bfloat16)
    w = (torch.randn(V, H, generator=g) * (2.0 / math.sqrt(H))).to(torch.bfloat16)
    t = torch.randint(0, V, (T,), generator=g)
    t[torch.rand(T, generator=g) >= valid] = IGNORE
    up = torch.randn(T, generator=g)
    return h.to(device), w.to(device), t.to(device), up.to(device)


def _oracle(h, w, t, scale, ignore=IGNORE):
    """(loss per token, dh, dw) and the elementwise error bounds, in 64 bits."""
    live = t != ignore
    hd, wd = torch.where(live[:, None], h.double(), 0.0), w.double()
    logits = hd @ wd.T
    lse = torch.logsumexp(logits, -1)
    at = torch.where(live, t, 0)[:, None]
    loss = torch.where(live, lse - logits.gather(1, at)[:, 0], 0.0)
    p = torch.exp(logits - lse[:, None])
    hot = torch.zeros_like(p).scatter_(1, at, 1.0)
    s = torch.where(live, scale.double(), 0.0)[:, None]
    d, size = (p - hot) * s, (p + hot) * s.abs()
    H = h.shape[1]
    delta = (H / 16 + 16) * 2.0 ** -22 * float((hd.abs() @ wd.abs().T).max())
    rel = (2.0 ** -8 + 3 * delta + 2.0 ** -17) * (1 + 2.0 ** -8)
    dh, dw = d @ wd, d.T @ hd
    return loss, dh, dw, {
        "loss": 2 * delta + 2.0 ** -18 * (1 + loss.abs()),
        "dh": rel * (size @ wd.abs()) + 2.0 ** -8 * dh.abs() + 1e-30,
        "dw": rel * (size.T @ hd.abs()) + 2.0 ** -8 * dw.abs() + 1e-30,
    }


def _within(got, want, bound, what):
    assert got.shape == want.shape
    off = (got.double() - want).abs() - bound
    assert bool((off <= 0).all()), f"{what}: {int((off > 0).sum())} values outside, worst by {float(off.max()):.3g}"


SHAPES = [
    # tokens, hidden, vocabulary, share of trained tokens, piece
    (1, 64, 256, 1.0, 0),
    (1, 8, 1, 1.0, 0),              # one column: loss 0, gradient 0
    (2, 1, 3, 1.0, 0),              # one hidden value
    (61, 512, 4096, 0.8, 0),
    (127, 72, 300, 1.0, 256),
    (128, 64, 256, 1.0, 0),
    (129, 200, 1000, 0.5, 256),
    (333, 1001, 777, 0.6, 256),     # odd rows
    (300, 136, 2055, 0.1, 512),
    (1030, 264, 513, 0.97, 0),
    (64, 512, 30001, 1.0, 0),       # the contraction over the vocabulary is split
    (64, 512, 30001, 1.0, 8192),
    (40, 64, 64, 0.0, 0),           # no trained token
]


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,V,valid,piece", SHAPES)
def test_grads_against_64_bits(T, H, V, valid, piece):
    from graspo_b200.ops._ext import check_errors
    from graspo_b200.ops.cross_entropy import linear_cross_entropy_grads

    h, w, t, up = _case(T, H, V, valid, seed=T)
    loss, dh, dw = linear_cross_entropy_grads(h, w, t, grad=up, reduction="none", piece=piece)
    check_errors()
    want, wh, ww, bound = _oracle(h, w, t, up)
    assert loss.dtype == torch.float32 and dh.dtype == dw.dtype == torch.bfloat16
    _within(loss, want, bound["loss"], "loss")
    _within(dh, wh, bound["dh"], "dh")
    _within(dw, ww, bound["dw"], "dw")
    assert torch.equal(loss[t == IGNORE], torch.zeros_like(loss[t == IGNORE]))
    assert not dh[t == IGNORE].any()
    again = linear_cross_entropy_grads(h, w, t, grad=up, reduction="none", piece=piece)
    assert all(torch.equal(a, b) for a, b in zip((loss, dh, dw), again)), "two calls differ"


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_autograd_reductions_and_batch_shape(reduction):
    from graspo_b200.ops.cross_entropy import linear_cross_entropy

    h, w, t, up = _case(6 * 35, 128, 515, 0.7, seed=3)
    hl, wl = h.view(6, 35, 128).clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = linear_cross_entropy(hl, wl, t.view(6, 35), reduction=reduction)
    n = int((t != IGNORE).sum())
    if reduction == "none":
        assert loss.shape == (6, 35)
        (loss * up.view(6, 35)).sum().backward()
        scale = up
    else:
        (loss * 1.75).backward()
        scale = torch.full_like(up, 1.75 / (n if reduction == "mean" else 1))
    want, wh, ww, bound = _oracle(h, w, t, scale)
    if reduction == "none":
        _within(loss.detach().view(-1), want, bound["loss"], "loss")
    else:
        k = 1 / n if reduction == "mean" else 1
        assert abs(float(loss.detach()) - float(want.sum()) * k) <= (float(bound["loss"].sum()) * k
                                                                    + 2.0 ** -23 * float(want.sum()) * k)
    _within(hl.grad.view(-1, 128), wh, bound["dh"], "dh")
    _within(wl.grad, ww, bound["dw"], "dw")


@pytest.mark.gpu
def test_gradient_against_differences():
    """<dh, u> and <dW, u> against central differences of the 64-bit loss along u."""
    from graspo_b200.ops.cross_entropy import linear_cross_entropy_grads

    h, w, t, up = _case(50, 96, 700, 0.8, seed=9)
    _, dh, dw = linear_cross_entropy_grads(h, w, t, grad=up, reduction="none")
    _, _, _, bound = _oracle(h, w, t, up)
    g = torch.Generator().manual_seed(1)
    u, q = torch.randn(h.shape, generator=g).cuda().double(), torch.randn(w.shape, generator=g).cuda().double()

    def total(a, b):
        live = t != IGNORE
        logp = torch.log_softmax(a[live] @ b.T, -1)
        return float((-logp.gather(1, t[live][:, None])[:, 0] * up[live].double()).sum())

    e = 1e-5  # the next term of the difference is of the order e^2 times a third derivative of some 10^4
    hd, wd = h.double(), w.double()
    along_h = (total(hd + e * u, wd) - total(hd - e * u, wd)) / (2 * e)
    along_w = (total(hd, wd + e * q) - total(hd, wd - e * q)) / (2 * e)
    assert abs(float((dh.double() * u).sum()) - along_h) <= float((bound["dh"] * u.abs()).sum()) + 1e-4
    assert abs(float((dw.double() * q).sum()) - along_w) <= float((bound["dw"] * q.abs()).sum()) + 1e-4


@pytest.mark.gpu
def test_ignored_rows_may_hold_anything():
    from graspo_b200.ops.cross_entropy import linear_cross_entropy_grads

    h, w, t, up = _case(200, 128, 600, 0.5, seed=4)
    clean = linear_cross_entropy_grads(h, w, t, grad=up, reduction="none")
    dead = t == IGNORE
    h2, up2 = h.clone(), up.clone()
    h2[dead] = float("nan")
    h2[dead.nonzero()[0]] = float("inf")
    up2[dead] = float("nan")
    dirty = linear_cross_entropy_grads(h2, w, t, grad=up2, reduction="none")
    assert all(torch.equal(a, b) for a, b in zip(clean, dirty))


@pytest.mark.gpu
def test_other_ignore_index_and_int32_targets():
    from graspo_b200.ops.cross_entropy import linear_cross_entropy_grads

    h, w, t, up = _case(90, 64, 300, 1.0, seed=5)
    t[::3] = 7
    loss, dh, dw = linear_cross_entropy_grads(h, w, t.int(), grad=up, reduction="none", ignore_index=7)
    want, wh, ww, bound = _oracle(h, w, t, up, ignore=7)
    _within(loss, want, bound["loss"], "loss")
    _within(dh, wh, bound["dh"], "dh")
    _within(dw, ww, bound["dw"], "dw")


@pytest.mark.gpu
def test_target_outside_the_vocabulary():
    from graspo_b200.ops._ext import KernelDataError, check_errors
    from graspo_b200.ops.cross_entropy import linear_cross_entropy_grads

    h, w, t, up = _case(70, 64, 300, 1.0, seed=6)
    bad = t.clone()
    bad[3], bad[40] = 300, -1
    loss, dh, dw = linear_cross_entropy_grads(h, w, bad, grad=up, reduction="none")
    with pytest.raises(KernelDataError):
        check_errors()
    check_errors()                                  # reported once
    assert loss.isnan().nonzero()[:, 0].tolist() == [3, 40]
    t[3] = t[40] = IGNORE
    want, wh, ww, bound = _oracle(h, w, t, up)
    ok = t != IGNORE
    _within(loss[ok], want[ok], bound["loss"][ok], "loss")
    _within(dh, wh, bound["dh"], "dh")
    _within(dw, ww, bound["dw"], "dw")


@pytest.mark.gpu
def test_strides_offsets_and_another_stream():
    from graspo_b200.ops.cross_entropy import linear_cross_entropy_grads

    h, w, t, up = _case(100, 96, 520, 0.8, seed=7)
    want = linear_cross_entropy_grads(h, w, t, grad=up, reduction="none")
    wide = torch.randn(100, 200, device="cuda").to(torch.bfloat16)
    wide[:, 3:99] = h                               # rows that start off a 16-byte boundary
    pad = torch.randn(520, 104, device="cuda").to(torch.bfloat16)
    pad[:, :96] = w                                 # rows with a gap
    off = torch.empty(520 * 96 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(520, 96)
    off.copy_(w)
    for hh in (wide[:, 3:99], h.T.contiguous().T):
        for ww in (pad[:, :96], off, w.T.contiguous().T):
            got = linear_cross_entropy_grads(hh, ww, t, grad=up, reduction="none")
            assert all(torch.equal(a, b) for a, b in zip(want, got))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = linear_cross_entropy_grads(h, w, t, grad=up, reduction="none")
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.gpu
def test_large_logits_do_not_overflow():
    from graspo_b200.ops.cross_entropy import linear_cross_entropy_grads

    h, w, t, up = _case(64, 64, 512, 1.0, seed=8)
    h = (h.float() * 60).to(torch.bfloat16)         # logits of some hundreds
    loss, dh, dw = linear_cross_entropy_grads(h, w, t, grad=up, reduction="none")
    want, wh, ww, bound = _oracle(h, w, t, up)
    _within(loss, want, bound["loss"], "loss")
    _within(dh, wh, bound["dh"], "dh")
    _within(dw, ww, bound["dw"], "dw")


@pytest.mark.gpu
def test_frozen_projection_and_no_trained_token():
    from graspo_b200.ops.cross_entropy import linear_cross_entropy, linear_cross_entropy_grads

    h, w, t, _ = _case(30, 64, 256, 1.0)
    loss, dh, dw = linear_cross_entropy_grads(h, w, t, weight_grad=False)
    full = linear_cross_entropy_grads(h, w, t)
    assert dw is None and torch.equal(loss, full[0]) and torch.equal(dh, full[1])
    hl = h.clone().requires_grad_(True)
    out = linear_cross_entropy(hl, w, torch.full_like(t, IGNORE))
    out.backward()
    assert float(out.detach()) == 0.0 and not hl.grad.any()
    empty = linear_cross_entropy_grads(h[:0], w, t[:0])
    assert float(empty[0]) == 0.0 and empty[1].shape == (0, 64) and not empty[2].any()


def test_cpu_form_matches_64_bits():
    from graspo_b200.ops.cross_entropy import linear_cross_entropy, linear_cross_entropy_grads

    h, w, t, up = _case(37, 24, 50, 0.6, device="cpu")
    h, w = h.float(), w.float()
    loss, dh, dw = linear_cross_entropy_grads(h, w, t, grad=up, reduction="none")
    want, wh, ww, _ = _oracle(h, w, t, up)
    for a, b in ((loss, want), (dh, wh), (dw, ww)):      # fp32 sums of at most 50 terms of order 10
        assert (a.double() - b).abs().max() < 50 * 2.0 ** -23 * 10
    hl = h.clone().requires_grad_(True)
    linear_cross_entropy(hl, w, torch.full_like(t, IGNORE)).backward()
    assert not hl.grad.any()
    with pytest.raises(IndexError):
        linear_cross_entropy(h, w, torch.full_like(t, 50))


def test_host_logic_on_emulated_kernels():
    """Row compaction, upstream weights and reductions around the kernels, emulated on the CPU."""
    from graspo_b200.ops.cross_entropy import _LinearCrossEntropy
    from graspo_b200.ops.emulate import use_emulation

    h, w, t, up = _case(150, 40, 333, 0.5, seed=2, device="cpu")
    n = int((t != IGNORE).sum())
    for reduction, scale in (("none", up), ("sum", torch.full_like(up, 0.5)), ("mean", torch.full_like(up, 0.5 / n))):
        with use_emulation():
            hl, wl = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
            loss = _LinearCrossEntropy.apply(hl, wl, t, IGNORE, reduction, 256)
            (loss * (up if reduction == "none" else 0.5)).sum().backward()
        want, wh, ww, bound = _oracle(h, w, t, scale)
        if reduction == "none":
            _within(loss.detach(), want, bound["loss"], "loss")
        _within(hl.grad, wh, bound["dh"], "dh")
        _within(wl.grad, ww, bound["dw"], "dw")


def test_refusals():
    from graspo_b200.ops.cross_entropy import linear_cross_entropy, linear_cross_entropy_grads

    h, w, t = torch.randn(4, 8), torch.randn(10, 8), torch.zeros(4, dtype=torch.long)
    for args, kw in [
        ((h, w, t), {"reduction": "max"}),
        ((h, w[:, :7], t), {}),
        ((h, w[:0], t), {}),
        ((h, w, t[:3]), {}),
        ((h, w, t.float()), {}),
        ((h, w[0], t), {}),
        ((h, w, t), {"piece": 100}),
    ]:
        with pytest.raises(ValueError):
            linear_cross_entropy(*args, **kw)
    with pytest.raises(ValueError):
        linear_cross_entropy_grads(h, w, t, grad=torch.ones(4))
    with pytest.raises(ValueError):
        linear_cross_entropy_grads(h, w, t, grad=torch.ones(3), reduction="none")


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    from graspo_b200.ops.cross_entropy import linear_cross_entropy, linear_cross_entropy_grads

    h, w, t, _ = _case(8, 64, 256, 1.0)
    with pytest.raises(ValueError):
        linear_cross_entropy(h.float(), w.float(), t)
    with pytest.raises(ValueError):
        linear_cross_entropy(h, w, t.cpu())
    with pytest.raises(ValueError):
        linear_cross_entropy_grads(h, w, t, piece=100)


def _confident(T, H, V, offset, device):
    """Tokens whose target leads by 6 to 20 (losses of 1e-1 down to 1e-6), all logits shifted by `offset`."""
    g = torch.Generator().manual_seed(H + offset)
    u = torch.randn(H, generator=g)
    u /= u.norm()
    w = torch.randn(V, H, generator=g) * (2.0 / math.sqrt(H))
    w += (2.0 - w @ u)[:, None] * u                          # every row has the same part along u
    t = torch.randint(0, V, (T,), generator=g)
    lead = torch.linspace(1.5, 5.0, T)[:, None] * (w[t] - 2.0 * u)
    h = lead + (offset / 2.0) * u
    return h.to(device, torch.bfloat16), w.to(device, torch.bfloat16), t.to(device)


def _confident_oracle(h, w, t):
    """Logits' error delta as above, and loss, others' share R of each target's and 64-bit logits.  The loss is
    log(1 + R) with R = sum exp(l_v - l_y) over the others: two logits' errors and the exponentials' (2^-16 with the
    roundings of the exponent, at most 32 here) are errors relative to the loss itself."""
    logits = h.double() @ w.double().T
    at = t[:, None]
    lead = logits - logits.gather(1, at)
    share = torch.exp(lead.scatter(1, at, -torch.inf))
    delta = (h.shape[1] / 16 + 16) * 2.0 ** -22 * float((h.double().abs() @ w.double().abs().T).max())
    return torch.log1p(share.sum(-1)), share, delta


CONFIDENT = [(96, 4096, 515, 0), (96, 4096, 515, 300), (130, 64, 777, 40), (50, 1000, 300, -100)]


@pytest.mark.parametrize("T,H,V,offset", CONFIDENT)
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_losses_of_confident_tokens(T, H, V, offset, device):
    from graspo_b200.ops.cross_entropy import _LinearCrossEntropy
    from graspo_b200.ops.emulate import use_emulation

    h, w, t = _confident(T, H, V, offset, device)
    want, _, delta = _confident_oracle(h, w, t)
    assert float(want.min()) < 1e-5 and float(want.max()) > 1e-2
    with use_emulation() if device == "cpu" else contextlib.nullcontext():
        loss = _LinearCrossEntropy.apply(h, w, t, IGNORE, "none", 0)
    _within(loss, want, want * (math.expm1(2 * delta) + 2.0 ** -16), "loss")


@pytest.mark.gpu
def test_infinite_logits():
    """As log_softmax has it: an infinite logit leaves no loss (NaN) unless it is the target's and -inf (inf)."""
    from graspo_b200.ops.cross_entropy import linear_cross_entropy

    w = torch.zeros(300, 64, device="cuda", dtype=torch.bfloat16)
    w[:, 1] = torch.linspace(-1, 1, 300)
    h = torch.ones(5, 64, device="cuda", dtype=torch.bfloat16)
    t = torch.tensor([7, 299, 0, 150, 7], device="cuda")
    for value, want in ((math.inf, [math.nan] * 5), (-math.inf, [math.inf, None, None, None, math.inf]),
                        (math.nan, [math.nan] * 5)):
        bad = w.clone()
        bad[7, 0] = value
        loss = linear_cross_entropy(h, bad, t, reduction="none")
        logits = h.double() @ bad.double().T
        ref = -torch.log_softmax(logits, -1).gather(1, t[:, None])[:, 0]
        assert torch.equal(loss.isnan(), ref.isnan()) and torch.equal(loss.isinf(), ref.isinf())
        for got, r, v in zip(loss.tolist(), ref.tolist(), want):
            assert v is None and abs(got - r) < 1e-5 or v is not None and (got == v or got != got and v != v)


@pytest.mark.parametrize("T,H,V,offset", CONFIDENT)
@pytest.mark.parametrize("reduction", ["none", "mean"])
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_gradients_of_confident_tokens(T, H, V, offset, reduction, device):
    """The target's entry of d is -(1 - p), whose error is relative to 1 - p and not to 1: every entry of dh and
    dW within the logits' error and the rounding of d (2^-8) of sums over |p - hot|."""
    from graspo_b200.ops.cross_entropy import _LinearCrossEntropy
    from graspo_b200.ops.emulate import use_emulation

    h, w, t = _confident(T, H, V, offset, device)
    up = torch.randn(T, generator=torch.Generator().manual_seed(1)).to(device)
    _, share, delta = _confident_oracle(h, w, t)
    rest = share.sum(-1, keepdim=True)
    d = (share / (1 + rest)).scatter(1, t[:, None], -rest / (1 + rest))
    d = d * (up.double()[:, None] if reduction == "none" else 1 / T)
    hl, wl = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    with use_emulation() if device == "cpu" else contextlib.nullcontext():
        loss = _LinearCrossEntropy.apply(hl, wl, t, IGNORE, reduction, 0)
        loss.backward(up if reduction == "none" else None)
    rel = (2.0 ** -8 + 4 * delta + 2.0 ** -16) * (1 + 2.0 ** -8)
    wh, ww = d @ w.double(), d.T @ h.double()
    _within(hl.grad, wh, rel * (d.abs() @ w.double().abs()) + 2.0 ** -8 * wh.abs() + 1e-30, "dh")
    _within(wl.grad, ww, rel * (d.T.abs() @ h.double().abs()) + 2.0 ** -8 * ww.abs() + 1e-30, "dw")


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("frozen", [False, True])
def test_second_derivatives_are_refused(device, frozen):
    """Also where the upstream gradient is a constant, and where a larger loss holds the term."""
    from graspo_b200.ops.cross_entropy import _kernel_loss
    from graspo_b200.ops.emulate import use_emulation

    h, w, t, _ = _case(20, 64, 256, 1.0, device=device)
    hl, wl = h.clone().requires_grad_(True), w.clone().requires_grad_(not frozen)
    leaves = (hl,) if frozen else (hl, wl)
    with use_emulation() if device == "cpu" else contextlib.nullcontext():
        loss = _kernel_loss(hl, wl, t, IGNORE, "mean", 0)
        plain = torch.autograd.grad(loss, leaves, retain_graph=True)
        grads = torch.autograd.grad(loss, leaves, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(plain, grads))
        for second in grads:
            for leaf in leaves:
                with pytest.raises(RuntimeError, match="second derivative"):
                    torch.autograd.grad(loss + second.float().square().sum(), leaf, retain_graph=True)
        (loss + hl.float().sum()).backward()                 # nothing of a second order in it
    assert hl.grad is not None


def test_second_derivatives_of_the_cpu_form():
    """The CPU form is PyTorch's own operations: differentiable twice."""
    from graspo_b200.ops.cross_entropy import linear_cross_entropy

    h, w, t, _ = _case(9, 6, 11, 0.7, device="cpu")
    both = []
    for form in (lambda a, b: linear_cross_entropy(a, b, t),
                 lambda a, b: torch.nn.functional.cross_entropy(a @ b.T, t, ignore_index=IGNORE)):
        a, b = h.float().requires_grad_(True), w.float().requires_grad_(True)
        da, db = torch.autograd.grad(form(a, b), (a, b), create_graph=True)
        both.append(torch.autograd.grad(da.square().sum() + db.square().sum(), (a, b)))
    for x, y in zip(*both):                                  # fp32 sums of at most 11 terms of order 1
        assert (x - y).abs().max() < 64 * 2.0 ** -23


@pytest.mark.gpu
def test_waits_that_give_up_end_the_call():
    """With an error already recorded a wait may give up: the call ends, the error is raised, the next call is right."""
    from graspo_b200.ops._ext import KernelTimeout, check_errors, err_word
    from graspo_b200.ops.cross_entropy import linear_cross_entropy_grads

    h, w, t, up = _case(700, 520, 9000, 0.8, seed=13)
    want = linear_cross_entropy_grads(h, w, t, grad=up, reduction="none", piece=2048)
    check_errors()
    for _ in range(3):
        err_word(h.device)[0] = 1
        linear_cross_entropy_grads(h, w, t, grad=up, reduction="none", piece=2048)
        with pytest.raises(KernelTimeout):
            check_errors()
        got = linear_cross_entropy_grads(h, w, t, grad=up, reduction="none", piece=2048)
        check_errors()
        assert all(torch.equal(p, q) for p, q in zip(want, got))


@pytest.mark.gpu
def test_backward_leaves_the_saved_state_alone():
    """Two backward passes of one graph, on two streams too, each have their own weights."""
    from graspo_b200.ops.cross_entropy import linear_cross_entropy

    h, w, t, up = _case(300, 128, 999, 0.8, seed=12)
    hl, wl = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    for reduction, first, second in (("none", up, 3 * up.flip(0)), ("mean", torch.tensor(0.3, device="cuda"),
                                                                     torch.tensor(-7.0, device="cuda"))):
        loss = linear_cross_entropy(hl, wl, t, reduction=reduction)
        saved = [s.clone() for s in loss.grad_fn.saved_tensors]
        one = torch.autograd.grad(loss, (hl, wl), first, retain_graph=True)
        two = torch.autograd.grad(loss, (hl, wl), second, retain_graph=True)
        # bits: rows that no token filled hold anything, NaN among it
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8))
                   for a, b in zip(saved, loss.grad_fn.saved_tensors))
        again = torch.autograd.grad(loss, (hl, wl), first)
        assert all(torch.equal(a, b) for a, b in zip(one, again))
        assert not torch.equal(one[0], two[0])


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_calls_in_a_row_do_not_mix(reduction):
    """Small calls start their kernels early: many of them back to back, each with its own unit and number of tokens,
    give what each gives by itself."""
    from graspo_b200.ops.cross_entropy import linear_cross_entropy_grads

    cases = []
    for i in range(4):
        h, w, t, up = _case(61 + 40 * i, 512, 4096, 0.9 - 0.2 * i, seed=20 + i)
        cases.append((h, w, t, up * 10.0 ** (3 * i - 4) if reduction == "none" else up[0].abs() * 10.0 ** (3 * i - 4)))
    want = []
    for h, w, t, g in cases:
        want.append(linear_cross_entropy_grads(h, w, t, grad=g, reduction=reduction))
        torch.cuda.synchronize()
    got = [linear_cross_entropy_grads(h, w, t, grad=g, reduction=reduction)
           for _ in range(60) for h, w, t, g in cases]
    for i, out in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(out, want[i % 4]))


# Rules on sizes choose segments, launches, slices and pieces; each row reaches one that SHAPES does not.
LARGE = [
    # tokens, hidden, vocabulary, share of trained tokens
    (40, 1025, 300, 1.0),           # a second segment of one K-block
    (61, 2056, 515, 0.8),           # three segments
    (70, 4096, 600, 1.0),           # four segments
    (700, 136, 12000, 1.0),         # 282 tiles: a CTA takes several
    (600, 2048, 4100, 1.0),         # kernels launched one after the other
    (2432, 2048, 4100, 1.0),        # 152 tiles of dh, in two slices
    (8200, 72, 16500, 0.9),         # two pieces of the vocabulary by default
]


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,V,valid", LARGE)
def test_larger_shapes_against_64_bits(T, H, V, valid):
    from graspo_b200.ops._ext import check_errors
    from graspo_b200.ops.cross_entropy import linear_cross_entropy_grads

    h, w, t, up = _case(T, H, V, valid, seed=T)
    loss, dh, dw = linear_cross_entropy_grads(h, w, t, grad=up, reduction="none")
    check_errors()
    want, wh, ww, bound = _oracle(h, w, t, up)
    _within(loss, want, bound["loss"], "loss")
    _within(dh, wh, bound["dh"], "dh")
    _within(dw, ww, bound["dw"], "dw")
    again = linear_cross_entropy_grads(h, w, t, grad=up, reduction="none")
    assert all(torch.equal(a, b) for a, b in zip((loss, dh, dw), again)), "two calls differ"


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,V,valid,piece", [(61, 512, 4096, 0.8, 0), (333, 1001, 777, 0.6, 256),
                                               (600, 2048, 4100, 0.7, 0), (1, 8, 1, 1.0, 0)])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("upstream", [None, -1.75])
def test_reduced_loss_and_gradients_in_one_call(T, H, V, valid, piece, reduction, upstream):
    from graspo_b200.ops.cross_entropy import linear_cross_entropy_grads

    h, w, t, _ = _case(T, H, V, valid, seed=T + 1)
    grad = None if upstream is None else torch.tensor(upstream, device="cuda")
    loss, dh, dw = linear_cross_entropy_grads(h, w, t, grad=grad, reduction=reduction, piece=piece)
    k = 1 / int((t != IGNORE).sum()) if reduction == "mean" else 1.0
    want, wh, ww, bound = _oracle(h, w, t, torch.full((T,), (upstream or 1.0) * k, device="cuda", dtype=torch.float64))
    assert loss.shape == () and loss.dtype == torch.float32
    assert abs(float(loss) - float(want.sum()) * k) <= (float(bound["loss"].sum()) * k
                                                        + 2.0 ** -23 * float(want.sum()) * k)
    _within(dh, wh, bound["dh"], "dh")
    _within(dw, ww, bound["dw"], "dw")


@pytest.mark.gpu
@pytest.mark.parametrize("H,piece,copies,pieces", [(64, 0, 0, 1), (64, 256, 0, 4), (1001, 0, 1, 1), (1001, 512, 1, 2)])
def test_every_launch_is_counted(H, piece, copies, pieces):
    from graspo_b200.ops._ext import launches
    from graspo_b200.ops.cross_entropy import linear_cross_entropy, linear_cross_entropy_grads

    h, w, t, up = _case(600, H, 1000, 0.8, seed=14)

    def counted(call):
        before = launches.count
        out = call()
        return launches.count - before, out

    # compaction, (a copy of W's odd rows), product, row sums; per piece of the vocabulary the products; the rows of
    # dh; two for the sums that dW's rows lack
    forward = 3 + copies
    assert counted(lambda: linear_cross_entropy_grads(h, w, t, piece=piece))[0] == forward + 3 * pieces + 3
    assert counted(lambda: linear_cross_entropy_grads(h, w, t, piece=piece, weight_grad=False))[0] == forward + 2 * pieces + 1
    assert counted(lambda: linear_cross_entropy_grads(h, w, t, grad=up, reduction="none", piece=piece))[0] == (
        forward + 1 + 3 * pieces + 3)
    hl, wl = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    n, loss = counted(lambda: linear_cross_entropy(hl, wl, t, piece=piece))
    assert n == forward + 1                                   # and the total
    assert counted(loss.backward)[0] == 1 + copies + 3 * pieces + 3


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,V,common", [(300, 264, 20011, 0.0), (61, 512, 4096, 0.0), (777, 1001, 5000, 0.4), (1, 72, 900, 0.0),
                                          (2500, 136, 3000, 0.0), (700, 2056, 30000, 0.1)])
def test_weights_per_token_are_not_rounded(T, H, V, common):
    """The target's entry r (p - 1) carries no rounding to bf16: dh and dW are off by the rounding of the result (2^-8),
    the errors of logits and exponentials, and the rounding of the other entries, which are sums over p.  In the norm
    that is the error of rounding the exact result, where p is spread over the vocabulary (its square is below a tenth
    of 1)."""
    from graspo_b200.ops.cross_entropy import linear_cross_entropy_grads

    h, w, t, up = _case(T, H, V, 1.0, seed=T + V)
    t[torch.rand(T, generator=torch.Generator().manual_seed(3)).cuda() < common] = 17       # one frequent target
    _, dh, dw = linear_cross_entropy_grads(h, w, t, grad=up, reduction="none")
    _, wh, ww, _ = _oracle(h, w, t, up)
    hd, wd, s = h.double(), w.double(), up.double().abs()[:, None]
    p = torch.softmax(hd @ wd.T, -1)
    delta = (H / 16 + 16) * 2.0 ** -22 * float((hd.abs() @ wd.abs().T).max())
    hot = torch.zeros_like(p).scatter_(1, t[:, None], 1.0)
    rel = (2.0 ** -8 + 3 * delta + 2.0 ** -17) * (1 + 2.0 ** -8)
    exact = 4 * delta + 2.0 ** -15
    err = (p * (1 - hot) * rel + hot * exact) * s
    _within(dh, wh, err @ wd.abs() + 2.0 ** -8 * wh.abs() * (1 + 2.0 ** -8) + 1e-30, "dh")
    _within(dw, ww, err.T @ hd.abs() + 2.0 ** -8 * ww.abs() * (1 + 2.0 ** -8) + 1e-30, "dw")
    if T > 1:
        for got, want in ((dh, wh), (dw, ww)):
            best = (want.to(torch.bfloat16).double() - want).norm()
            assert float((got.double() - want).norm()) <= 1.12 * float(best)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [40, 300, 2300])
@pytest.mark.parametrize("frozen", [None, "h", "w"])
def test_autograd_gives_what_one_call_gives(T, frozen):
    """The tokens by target are ranked, or sorted, for dW only; both forms have the same kernels."""
    from graspo_b200.ops._ext import check_errors
    from graspo_b200.ops.cross_entropy import linear_cross_entropy, linear_cross_entropy_grads

    h, w, t, up = _case(T, 136, 900, 0.8, seed=T + 2)
    want = linear_cross_entropy_grads(h, w, t, grad=up, reduction="none", weight_grad=frozen != "w")
    hl, wl = h.clone().requires_grad_(frozen != "h"), w.clone().requires_grad_(frozen != "w")
    loss = linear_cross_entropy(hl, wl, t, reduction="none")
    loss.backward(up)
    assert torch.equal(loss.detach(), want[0])
    assert hl.grad is None if frozen == "h" else torch.equal(hl.grad, want[1])
    assert wl.grad is None if frozen == "w" else torch.equal(wl.grad, want[2])
    check_errors()
