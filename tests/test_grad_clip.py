"""Global gradient norm and clipping over many tensors (graspo_b200/ops/grad_clip.py)
against 64 bits.

Tolerances, with u = 2^-24: a thread adds at most 20 fp32 squares before its sum
goes to 64 bits, so the norm is relatively within 24 u; the coefficient carries
that and three roundings (28 u), a scaled value one more and the rounding of its
storage type."""

import math

import pytest
import torch

U = 2.0 ** -24
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 1e-38, torch.float16: 2.0 ** -25, torch.float32: 1e-38}
GPU = pytest.param("cuda", marks=pytest.mark.gpu)


def _grads(sizes, dtypes, device, seed=0, flat=False):
    g = torch.Generator().manual_seed(seed)
    if flat:                                       # views of one buffer, at any alignment
        buf = torch.randn(sum(sizes), generator=g).to(device, dtypes[0])
        return list(buf.split(sizes))
    return [torch.randn(n, generator=g).to(device, dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]


def _norm64(grads):
    return math.sqrt(sum(float(g.double().square().sum()) for g in grads))


def _check_scaled(before, after, coef):
    for b, a in zip(before, after):
        want = b.double() * coef
        bound = 30 * U * want.abs() + ROUND[a.dtype] * want.abs() * (1 + 30 * U) + TINY[a.dtype]
        assert a.shape == b.shape and bool(((a.double() - want).abs() <= bound).all())


F32, BF, HF = torch.float32, torch.bfloat16, torch.float16
LISTS = [
    ([1], [F32], False),
    ([5, 0, 17, 1, 4096], [F32, BF, HF], False),
    ([3, 8, 13, 16384, 16385, 7, 40001], [F32], True),
    ([9, 2, 33, 16383, 50000, 1], [BF], True),
    ([100003, 11, 65536], [HF], True),
    ([1 + (i * 37) % 200 for i in range(2000)], [F32, BF], False),        # several launches
    ([65, 3] * 33, [BF], True),                                          # just past the small table
    ([3000001, 700000], [BF, F32], False),
]


@pytest.mark.parametrize("device", ["cpu", GPU])
@pytest.mark.parametrize("sizes,dtypes,flat", LISTS)
def test_norm_and_clipping_against_64_bits(sizes, dtypes, flat, device):
    from graspo_b200.ops.grad_clip import clip_grad_norm_, grad_norm

    grads = _grads(sizes, dtypes, device, flat=flat)
    before = [g.clone() for g in grads]
    want = _norm64(grads)
    assert abs(float(grad_norm(grads)) - want) <= 24 * U * want
    # above the limit nothing changes
    assert abs(float(clip_grad_norm_(grads, 2 * want)) - want) <= 24 * U * want
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    limit = want / 3
    coef = limit / (want + 1e-6)
    for dtype in (F32, BF):
        out = [torch.full_like(g, 7, dtype=dtype) for g in grads]
        norm = clip_grad_norm_(grads, limit, out=out)
        assert norm.shape == () and norm.dtype == F32 and abs(float(norm) - want) <= 24 * U * want
        assert all(torch.equal(a, b) for a, b in zip(grads, before))
        _check_scaled(before, out, coef)
    clip_grad_norm_(grads, limit)
    _check_scaled(before, grads, coef)


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_out_below_the_limit_is_a_copy(device):
    from graspo_b200.ops.grad_clip import clip_grad_norm_

    grads = _grads([50, 129, 20000], [BF], device)
    out = [torch.zeros_like(g, dtype=F32) for g in grads]
    clip_grad_norm_(grads, 1e6, out=out)
    assert all(torch.equal(o, g.float()) for o, g in zip(out, grads))
    clip_grad_norm_(grads, 0.0, out=out)                # 0: no clipping
    assert all(torch.equal(o, g.float()) for o, g in zip(out, grads))


@pytest.mark.gpu
def test_misaligned_outputs():
    """Inputs and outputs that never reach a 16-byte boundary together."""
    from graspo_b200.ops.grad_clip import clip_grad_norm_

    g = torch.Generator().manual_seed(3)
    for off_in in range(0, 9):
        for off_out in (0, 1, 3, 6):
            src = torch.randn(5000 + off_in, generator=g).cuda().to(BF)[off_in:]
            dst = torch.full((5000 + off_out + 8,), 9.0, device="cuda")
            view = dst[off_out : off_out + 5000]
            norm = clip_grad_norm_([src], 1.0, out=[view])
            _check_scaled([src], [view], 1.0 / (_norm64([src]) + 1e-6))
            assert (dst[:off_out] == 9).all() and (dst[off_out + 5000 :] == 9).all() and float(norm) > 1


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_empty_and_zero(device):
    from graspo_b200.ops.grad_clip import clip_grad_norm_, grad_norm

    z = [torch.zeros(10, device=device), torch.zeros(0, device=device)]
    assert float(grad_norm(z)) == 0.0 and float(clip_grad_norm_(z, 1.0)) == 0.0 and not z[0].any()
    assert float(grad_norm([])) == 0.0 and float(clip_grad_norm_([], 1.0)) == 0.0
    assert float(clip_grad_norm_([z[1]], 1.0)) == 0.0
    assert float(grad_norm(torch.full((4,), 3.0, device=device))) == 6.0


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_non_finite_norms(device):
    from graspo_b200.ops.grad_clip import clip_grad_norm_

    a = [torch.ones(100, device=device), torch.ones(50, device=device)]
    a[1][7] = float("nan")
    assert math.isnan(float(clip_grad_norm_(a, 1.0))) and all(t.isnan().all() for t in a)
    b = [torch.ones(100, device=device), torch.ones(50, device=device)]
    b[0][3] = float("inf")
    assert math.isinf(float(clip_grad_norm_(b, 1.0)))
    assert b[0].isnan().nonzero()[:, 0].tolist() == [3] and not b[1].any()


@pytest.mark.gpu
def test_same_bits_in_every_call_and_on_another_stream():
    from graspo_b200.ops.grad_clip import grad_norm

    grads = _grads([100001, 77, 300000] * 20, [F32, BF], "cuda")
    first = grad_norm(grads)
    for _ in range(5):
        assert torch.equal(first, grad_norm(grads))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = grad_norm(grads)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, other)


@pytest.mark.gpu
def test_more_than_31_bits_of_values():
    from graspo_b200.ops.grad_clip import clip_grad_norm_

    n = (1 << 31) + 5
    g = torch.zeros(n, device="cuda", dtype=BF)
    g[-1], g[0], g[n // 2] = 3.0, 4.0, 12.0
    norm = clip_grad_norm_([g], 6.5)
    assert float(norm) == 13.0
    assert float(g[-1]) == 1.5 and float(g[0]) == 2.0 and float(g[n // 2]) == 6.0


@pytest.mark.parametrize("device", ["cpu", GPU])
def test_refusals(device):
    from graspo_b200.ops.grad_clip import clip_grad_norm_, grad_norm

    g = [torch.ones(4, 6, device=device), torch.ones(3, device=device)]
    for bad in [lambda: clip_grad_norm_(g, -1.0), lambda: clip_grad_norm_(g, float("nan")),
                lambda: clip_grad_norm_(g, 1.0, out=g[:1]),
                lambda: clip_grad_norm_(g, 1.0, out=[g[0], torch.ones(4, device=device)]),
                lambda: grad_norm([g[0].T]), lambda: grad_norm([g[1].long()]),
                lambda: grad_norm([g[1].double()])]:
        with pytest.raises(ValueError):
            bad()
    if device == "cuda":
        with pytest.raises(ValueError):
            grad_norm([g[0], torch.ones(3)])


# far from 1: squares past the ends of fp32's range, and one value far above the others
SCALES = [(F32, 1e25), (BF, 1e25), (F32, 1e-25), (BF, 1e-25), (F32, 1e-21), (BF, 1e-21), (F32, 1e-38)]


@pytest.mark.parametrize("device", ["cpu", GPU])
@pytest.mark.parametrize("dtype,scale", SCALES)
def test_norms_of_very_large_and_small_gradients(dtype, scale, device):
    from graspo_b200.ops.grad_clip import clip_grad_norm_, grad_norm

    for sizes, flat in (([1], False), ([5, 12291, 70001, 3, 1000003], True), ([4096, 17], False)):
        grads = [(g.float() * scale).to(dtype) for g in _grads(sizes, [F32], device, flat=flat)]
        want = _norm64(grads)
        assert want > 0
        small = 2.0 ** -149                        # a norm below fp32's normal range is stored with fewer bits
        assert abs(float(grad_norm(grads)) - want) <= 24 * U * want + small
        if scale > 1:
            out = [torch.empty_like(g, dtype=F32) for g in grads]
            clip_grad_norm_(grads, want / 3, out=out)
            _check_scaled(grads, out, 1 / 3)
        else:
            before = [g.clone() for g in grads]
            clip_grad_norm_(grads, 1.0)            # below the limit
            assert all(torch.equal(a, b) for a, b in zip(grads, before))


@pytest.mark.parametrize("device", ["cpu", GPU])
@pytest.mark.parametrize("big,at", [(3e19, 0), (3e19, 5000), (-2e30, 12345), (1e-30, 7)])
def test_one_value_far_from_the_others(big, at, device):
    """One large value among ordinary ones; a tiny one among zeros."""
    from graspo_b200.ops.grad_clip import clip_grad_norm_, grad_norm

    (g,) = _grads([20011], [F32], device)
    if abs(big) < 1:
        g.zero_()
    g[at] = big
    want = _norm64([g])
    assert abs(float(grad_norm([g])) - want) <= 24 * U * want
    if abs(big) > 1:
        out = torch.empty_like(g)
        clip_grad_norm_([g], want / 4, out=[out])
        _check_scaled([g], [out], 0.25)
