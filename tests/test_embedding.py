"""Scaled embedding lookup and the gradient of its table (graspo_b200/ops/embedding.py)
against 64 bits.

Tolerances, with u = 2^-24: the lookup rounds one product to fp32 and to the
storage type; a table row's gradient is a chain of at most ``64 + 32 + n / 32``
fp32 additions for n tokens, a product with the scale and one rounding to the
storage type (with an existing gradient, one more addition)."""

import pytest
import torch

U = 2.0 ** -24
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 1e-38, torch.float16: 2.0 ** -25, torch.float32: 1e-38}


def _case(T, V, H, dtype, heavy=0.0, seed=0, device="cuda"):
    g = torch.Generator().manual_seed(seed + T)
    ids = torch.randint(0, V, (T,), generator=g)
    ids[torch.rand(T, generator=g) < heavy] = V // 2
    table = torch.randn(V, H, generator=g)
    dy = torch.randn(T, H, generator=g)
    return ids.to(device), table.to(device, dtype), dy.to(device, dtype)


def _grad_oracle(dy, ids, V, scale, padding=None, base=None, out_dtype=None):
    keep = ids != (-1 if padding is None else padding)
    d, i = dy.double()[keep], ids[keep]
    want = torch.zeros(V, dy.shape[1], dtype=torch.float64, device=dy.device).index_add_(0, i, d) * scale
    size = torch.zeros_like(want).index_add_(0, i, d.abs()) * abs(scale)
    n = torch.bincount(i, minlength=V)[:, None]
    err = (64 + 32 + n / 32) * U * size
    if base is not None:
        want = want + base.double()
        err = err + U * want.abs()
    t = out_dtype or dy.dtype
    return want, err + ROUND[t] * (want.abs() + err) + TINY[t]


def _within(got, want, bound, what):
    assert got.shape == want.shape
    off = (got.double() - want).abs() - bound
    assert bool((off <= 0).all()), f"{what}: {int((off > 0).sum())} values outside, worst by {float(off.max()):.3g}"


SHAPES = [
    # tokens, table rows, hidden, share of one repeated id
    (1, 1, 1, 0.0),
    (1, 50, 8, 0.0),
    (31, 7, 64, 0.0),
    (32, 5, 72, 1.0),               # one whole group
    (33, 300, 513, 0.5),
    (64, 4096, 512, 0.0),
    (2047, 100, 40, 0.3),
    (2048, 3000, 40, 0.9),
    (2049, 3000, 33, 0.9),          # a second sorted chunk of one key
    (9000, 17, 24, 0.0),            # long runs everywhere
    (12345, 20011, 136, 0.4),
    (4097, 260, 2056, 0.2),         # more than one block of columns
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,V,H,heavy", SHAPES)
def test_lookup_and_gradient_against_64_bits(T, V, H, heavy, dtype):
    from graspo_b200.ops._ext import check_errors
    from graspo_b200.ops.embedding import embedding, embedding_grad

    ids, table, dy = _case(T, V, H, dtype, heavy)
    y = embedding(ids, table, scale=0.7)
    want = table[ids].double() * 0.7
    # 0.7 itself is rounded to fp32 on its way to the kernel
    _within(y, want, 2 * U * want.abs() + ROUND[dtype] * want.abs() * (1 + 2 * U) + TINY[dtype], "y")
    got = embedding_grad(dy, ids, V, scale=0.7)
    _within(got, *_grad_oracle(dy, ids, V, 0.7), "gradient")
    assert torch.equal(got, embedding_grad(dy, ids, V, scale=0.7)), "two calls differ"
    check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,out_dtype", [(torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16),
                                             (torch.float32, torch.float32), (torch.float32, torch.bfloat16),
                                             (torch.float16, torch.float32)])
@pytest.mark.parametrize("T,V,H,heavy", [(1, 3, 8, 0.0), (700, 900, 96, 0.3), (5000, 777, 131, 0.5), (40, 9, 2056, 0.9)])
def test_adding_to_an_existing_gradient(T, V, H, heavy, dtype, out_dtype):
    from graspo_b200.ops.embedding import embedding_grad

    ids, _, dy = _case(T, V, H, dtype, heavy)
    base = torch.randn(V, H, generator=torch.Generator().manual_seed(1)).cuda().to(out_dtype)
    out = base.clone()
    assert embedding_grad(dy, ids, V, scale=2.0, out=out) is out
    _within(out, *_grad_oracle(dy, ids, V, 2.0, base=base, out_dtype=out_dtype), "gradient")
    untouched = torch.ones(V, dtype=torch.bool, device="cuda")
    untouched[ids] = False
    assert torch.equal(out[untouched], base[untouched])


@pytest.mark.gpu
@pytest.mark.parametrize("into", [False, True])
def test_padding_row_gets_no_gradient(into):
    from graspo_b200.ops.embedding import embedding, embedding_grad

    ids, table, dy = _case(3000, 500, 64, torch.bfloat16, 0.4)
    pad = 250
    dy[ids == pad] = float("nan")                       # what padding positions hold is not read
    out = torch.ones(500, 64, device="cuda") if into else None
    got = embedding_grad(dy, ids, 500, padding_idx=pad, out=out)
    base = torch.ones(500, 64, device="cuda") if into else None
    want = _grad_oracle(dy, ids, 500, 1.0, padding=pad, base=base, out_dtype=got.dtype)
    _within(got, *want, "gradient")
    assert torch.equal(embedding(ids, table, padding_idx=pad), table[ids])
    only = torch.full((70,), pad, device="cuda")
    assert not embedding_grad(dy[:70], only, 500, padding_idx=pad).any()


@pytest.mark.gpu
def test_autograd_shapes_and_linearity():
    """The lookup is linear in the table: <dE, Q> is <dy, s Q[ids]> for every Q."""
    from graspo_b200.ops.embedding import embedding

    ids, table, dy = _case(6 * 50, 80, 48, torch.float32)
    leaf = table.clone().requires_grad_(True)
    y = embedding(ids.view(6, 50).int(), leaf, scale=1.5)
    assert y.shape == (6, 50, 48)
    y.backward(dy.view(6, 50, 48))
    q = torch.randn(80, 48, generator=torch.Generator().manual_seed(2)).cuda().double()
    along = float((dy.double() * 1.5 * q[ids]).sum())
    _, bound = _grad_oracle(dy, ids, 80, 1.5)
    assert abs(float((leaf.grad.double() * q).sum()) - along) <= float((bound * q.abs()).sum())
    assert embedding(ids[:0], leaf).shape == (0, 48)


@pytest.mark.gpu
def test_ids_outside_the_table():
    from graspo_b200.ops._ext import KernelDataError, check_errors
    from graspo_b200.ops.embedding import embedding, embedding_grad

    ids, table, dy = _case(400, 90, 64, torch.bfloat16)
    bad = ids.clone()
    bad[5], bad[77], bad[399] = 90, -1, 1 << 40
    y = embedding(bad, table)
    with pytest.raises(KernelDataError):
        check_errors()
    assert y.isnan().all(-1).nonzero()[:, 0].tolist() == [5, 77, 399]
    got = embedding_grad(dy, bad, 90)
    with pytest.raises(KernelDataError):
        check_errors()
    keep = (bad >= 0) & (bad < 90)
    _within(got, *_grad_oracle(dy[keep], ids[keep], 90, 1.0), "gradient")


@pytest.mark.gpu
def test_strides_offsets_and_another_stream():
    from graspo_b200.ops.embedding import embedding, embedding_grad

    ids, table, dy = _case(500, 60, 64, torch.bfloat16)
    y, want = embedding(ids, table), embedding_grad(dy, ids, 60)
    wide = torch.zeros(60, 72, device="cuda", dtype=table.dtype)
    wide[:, 3:67] = table
    wdy = torch.zeros(500, 80, device="cuda", dtype=dy.dtype)
    wdy[:, 1:65] = dy
    assert torch.equal(embedding(ids, wide[:, 3:67]), y)
    for view in (wdy[:, 1:65], dy.T.contiguous().T):
        assert torch.equal(embedding_grad(view, ids, 60), want)
    assert torch.equal(embedding(torch.stack([ids, ids], 1)[:, 0], table), y)
    one = torch.ones(1, 1, device="cuda", dtype=dy.dtype).expand(500, 64)
    assert torch.equal(embedding_grad(one, ids, 60), embedding_grad(one.contiguous(), ids, 60))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = embedding_grad(dy, ids, 60)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    off = torch.zeros(60 * 64 + 1, device="cuda", dtype=torch.float32)[1:].view(60, 64)
    embedding_grad(dy, ids, 60, out=off)
    _within(off, *_grad_oracle(dy, ids, 60, 1.0, out_dtype=torch.float32), "gradient")


@pytest.mark.gpu
def test_no_tokens():
    from graspo_b200.ops.embedding import embedding, embedding_grad

    _, table, dy = _case(4, 30, 16, torch.bfloat16)
    none = torch.empty(0, dtype=torch.long, device="cuda")
    assert embedding(none, table).shape == (0, 16)
    assert not embedding_grad(dy[:0], none, 30).any()
    out = torch.ones(30, 16, device="cuda")
    assert torch.equal(embedding_grad(dy[:0], none, 30, out=out), torch.ones(30, 16, device="cuda"))


@pytest.mark.gpu
def test_rows_past_31_bits():
    """A table of more than 2^31 values: its last rows are reached."""
    from graspo_b200.ops.embedding import embedding, embedding_grad

    V, H = 300001, 8192
    table = torch.empty(V, H, device="cuda", dtype=torch.bfloat16)
    table[-1] = 3.0
    table[1] = 2.0
    ids = torch.tensor([V - 1, 1, V - 1], device="cuda")
    y = embedding(ids, table, scale=0.5)
    assert (y[0] == 1.5).all() and (y[1] == 1.0).all()
    out = torch.zeros(V, H, device="cuda", dtype=torch.bfloat16)
    embedding_grad(torch.ones_like(y), ids, V, out=out)
    assert (out[-1] == 2).all() and (out[1] == 1).all() and not out[2:-1].any()
    dense = embedding_grad(torch.ones_like(y), ids, V)
    assert torch.equal(dense, out)


@pytest.mark.parametrize("padding", [None, 3])
def test_cpu_form_matches_64_bits(padding):
    from graspo_b200.ops.embedding import embedding, embedding_grad

    ids, table, dy = _case(80, 20, 12, torch.bfloat16, 0.3, device="cpu")
    _within(embedding_grad(dy, ids, 20, scale=0.5, padding_idx=padding),
            *_grad_oracle(dy, ids, 20, 0.5, padding=padding), "gradient")
    leaf = table.clone().requires_grad_(True)
    embedding(ids.view(8, 10), leaf, scale=0.5, padding_idx=padding).backward(dy.view(8, 10, 12))
    _within(leaf.grad, *_grad_oracle(dy, ids, 20, 0.5, padding=padding), "gradient")
    with pytest.raises(IndexError):
        embedding(torch.tensor([20]), table)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_refusals(device):
    from graspo_b200.ops.embedding import embedding, embedding_grad

    ids, table, dy = _case(6, 10, 8, torch.float32, device=device)
    for bad in [lambda: embedding(ids.float(), table), lambda: embedding(ids, table[0]),
                lambda: embedding(ids, table.double()), lambda: embedding(ids, table, padding_idx=10),
                lambda: embedding(ids, table[:0]), lambda: embedding_grad(dy[:5], ids, 10),
                lambda: embedding_grad(dy.double(), ids, 10), lambda: embedding_grad(dy, ids, 0),
                lambda: embedding_grad(dy, ids, 10, out=torch.zeros(9, 8, device=device)),
                lambda: embedding_grad(dy, ids, 10, out=torch.zeros(8, 10, device=device).T),
                lambda: embedding_grad(dy, ids, 10, padding_idx=-1)]:
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_second_derivatives_are_refused(device):
    from graspo_b200.ops.embedding import embedding

    ids, table, dy = _case(6, 10, 8, torch.float32, device=device)
    leaf, up = table.clone().requires_grad_(True), dy.clone().requires_grad_(True)
    (grad,) = torch.autograd.grad(embedding(ids, leaf), leaf, up, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(up.sum() + grad.square().sum(), up, retain_graph=True)
    # with a constant upstream gradient the table's does not depend on anything
    (grad,) = torch.autograd.grad(embedding(ids, leaf), leaf, dy, create_graph=True)
    assert not grad.requires_grad
