"""Training-block operators on the GPU against their float64 definitions: sizes, types and
layouts where they can go wrong, gradients against formulas and differences, refusals."""

import pytest
import torch

import block_refs as R
from flashcart_b200 import ops

pytestmark = pytest.mark.gpu

F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16
UNIT = {F32: 2.0 ** -24, F64: 2.0 ** -53, BF16: 2.0 ** -24}   # of the sums
STORE = {F32: 2.0 ** -24, F64: 2.0 ** -53, BF16: 2.0 ** -8}   # of one stored value


def _randn(gen, *shape, dtype=F32):
    return torch.randn(*shape, generator=gen, dtype=F64).to("cuda", dtype)


# ------------------------------------------------------------------------------ embedding

# rows around the one-block sort's limit, one / two / three digit passes, single and long
# runs, odd widths, rows of one element
EMBED = [(1, 1, 1), (5, 2, 3), (192, 2, 64), (8192, 4, 16), (8193, 4, 16), (3000, 255, 33), (3000, 256, 20),
         (20000, 300, 130), (5000, 70000, 8), (20000, 70000, 8), (100003, 1, 12), (50001, 3, 257), (4097, 5000, 2944)]


@pytest.mark.parametrize("dtype", [F32, F64, BF16])
@pytest.mark.parametrize("rows,types,dim", EMBED)
def test_embedding_and_gradient(cuda_device, dtype, rows, types, dim):
    gen = torch.Generator().manual_seed(rows * 7 + dim)
    table = _randn(gen, types, dim, dtype=dtype)
    # a skewed draw: half of the rows on one type, the rest spread
    idx = torch.randint(0, types, (rows,), generator=gen)
    idx[torch.rand(rows, generator=gen) < 0.5] = types // 2
    idx = idx.cuda()
    grad = _randn(gen, rows, dim, dtype=dtype)
    t = table.clone().requires_grad_(True)
    y = ops.embedding(t, idx, 1.75, 1.0)
    want = R.embedding(table, idx, 1.75, 1.0)
    err = (y.detach().cpu().double() - want).abs()
    assert (err <= 2 * UNIT[dtype] * (1 + (want - 1).abs()) * 1.5 + STORE[dtype] * want.abs() * 1.01).all()
    (gt,) = torch.autograd.grad(y, t, grad)
    want, mag, count = R.embedding_grad(grad, idx, types, 1.75)
    bound = (count[:, None] + 2) * UNIT[dtype] * mag + STORE[dtype] * want.abs() * 1.01
    assert ((gt.cpu().double() - want).abs() <= bound).all()
    again = torch.autograd.grad(ops.embedding(t, idx, 1.75, 1.0), t, grad)[0]
    assert torch.equal(gt, again)  # equal inputs, equal bits
    ops.check_device_status()


def test_embedding_empty_rows_and_shapes(cuda_device):
    t = torch.randn(3, 4, device="cuda", requires_grad=True)
    y = ops.embedding(t, torch.zeros(0, dtype=torch.int64, device="cuda"))
    assert y.shape == (0, 4)
    (g,) = torch.autograd.grad(y, t, torch.zeros(0, 4, device="cuda"))
    assert torch.equal(g, torch.zeros(3, 4, device="cuda"))
    idx = torch.tensor([[0, 2], [1, 1]], device="cuda", dtype=torch.int32)
    y = ops.embedding(t, idx)
    assert torch.equal(y, t[idx.long()])
    wide = torch.randn(3, 8, device="cuda")[:, ::2]  # a strided table
    assert torch.equal(ops.embedding(wide, idx), wide[idx.long()])


@pytest.mark.parametrize("dim", [6, 8])
def test_embedding_misaligned_tensors(cuda_device, dim):
    store = torch.randn(1 + 50 * dim, device="cuda")
    table = store[1:].view(50, dim)  # 4 bytes off the vector boundary
    idx = torch.randint(0, 50, (333,), device="cuda")
    assert torch.equal(ops.embedding(table, idx), table[idx])
    grad = torch.randn(1 + 333 * dim, device="cuda")[1:].view(333, dim)
    got = torch.ops.flashcart.embedding_bwd(grad, idx, 50, 1.0)
    want, mag, count = R.embedding_grad(grad, idx, 50, 1.0)
    assert ((got.cpu().double() - want).abs() <= (count[:, None] + 3) * 2.0 ** -24 * mag).all()


def test_embedding_bad_index(cuda_device):
    ops.check_device_status()
    t = torch.ones(3, 4, device="cuda", requires_grad=True)
    idx = torch.tensor([0, 3, -1, 2], device="cuda")
    y = ops.embedding(t, idx, 1.0, 0.5)
    assert y[:, 0].tolist() == [1.5, 0.0, 0.0, 1.5]
    (g,) = torch.autograd.grad(y, t, torch.ones_like(y))
    assert g[:, 0].tolist() == [1.0, 0.0, 1.0]
    with pytest.raises(RuntimeError, match="outside"):
        ops.check_device_status()


@pytest.mark.parametrize("dtype", [F32, F64, BF16])
@pytest.mark.parametrize("dim", [1, 2, 3, 4, 5, 7, 8, 9, 15, 31, 33, 63])
def test_embedding_vectors_across_rows(cuda_device, dtype, dim):
    # rows that are no whole vectors, a wrong index on either side of a row's end
    ops.check_device_status()
    t = _randn(torch.Generator().manual_seed(dim), 6, dim, dtype=dtype)
    for rows in (1, 2, 259):
        idx = torch.randint(0, 6, (rows,), device="cuda")
        want = t[idx]
        assert torch.equal(ops.embedding(t, idx), want)
        idx[::5] = 6
        idx[-1:] = -2
        want = torch.where(((idx >= 0) & (idx < 6))[:, None], want, torch.zeros_like(want))
        assert torch.equal(ops.embedding(t, idx), want)
        with pytest.raises(RuntimeError, match="outside"):
            ops.check_device_status()


def test_embedding_differences_and_second_derivative(cuda_device):
    t = torch.randn(5, 3, dtype=F64, device="cuda", requires_grad=True)
    idx = torch.tensor([0, 4, 4, 1, 4, 0], device="cuda")
    f = lambda w: ops.embedding(w, idx, 0.7, 1.0)
    assert torch.autograd.gradcheck(f, (t,))
    assert torch.autograd.gradgradcheck(lambda w: f(w) ** 2, (t,))


def test_embedding_more_than_2_to_31_elements(cuda_device):
    rows, dim = 2 ** 22 + 3, 520
    idx = torch.arange(rows, device="cuda") % 7
    table = torch.randn(7, dim, device="cuda").to(BF16)
    y = ops.embedding(table, idx)
    at = torch.tensor([0, 1, 2 ** 21, 2 ** 22, rows - 2, rows - 1], device="cuda")
    assert torch.equal(y[at], table[idx[at]])
    del y
    g = torch.zeros(rows, dim, dtype=BF16, device="cuda")
    g[at] = 1.0
    got = torch.ops.flashcart.embedding_bwd(g, idx, 7, 1.0).float()
    assert torch.equal(got[:, 0].cpu(), torch.bincount(idx[at], minlength=7).float().cpu())
    assert (got == got[:, :1]).all()


def test_embedding_refusals(cuda_device):
    t, idx = torch.randn(3, 4, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="float32, float64 and bfloat16"):
        ops.embedding(t.half(), idx)
    with pytest.raises(ValueError, match="int64 or int32"):
        ops.embedding(t, idx.float())
    with pytest.raises(ValueError, match="n_types"):
        ops.embedding(t[0], idx)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.embedding(t, idx.cpu())
    with pytest.raises(ValueError, match="grad_out"):
        torch.ops.flashcart.embedding_bwd(t, idx, 3, 1.0)


# ------------------------------------------------------------------------------ dropout


@pytest.mark.parametrize("dtype", [F32, F64, BF16])
@pytest.mark.parametrize("n,l_max,c", [(1, 0, 1), (7, 0, 8), (33, 0, 7), (65, 0, 4), (5, 1, 3), (9, 2, 64), (3, 3, 12),
                                       (2, 3, 129), (700, 0, 20)])
def test_dropout_mask_and_gradient(cuda_device, dtype, n, l_max, c):
    gen = torch.Generator().manual_seed(n + c)
    p = 0.3
    x = _randn(gen, n, (l_max + 1) ** 2 * c, dtype=dtype).requires_grad_(True)
    rng = torch.tensor([2 ** 40 + 17, 5], device="cuda")
    y = ops.irreps_dropout(x, rng, p, l_max)
    keep = R.dropout_keep(n, l_max, c, 2 ** 40 + 17, 5, p)
    want = torch.where(keep, x.detach().cpu().double() / (1 - p), torch.zeros((), dtype=F64))
    # two roundings (the factor, the product) and the storage's
    assert ((y.detach().cpu().double() - want).abs() <= (2.02 * UNIT[dtype] + STORE[dtype]) * want.abs()).all()
    g = _randn(gen, *x.shape, dtype=dtype)
    (gx,) = torch.autograd.grad(y, x, g)
    want = torch.where(keep, g.cpu().double() / (1 - p), torch.zeros((), dtype=F64))
    assert ((gx.cpu().double() - want).abs() <= (2.02 * UNIT[dtype] + STORE[dtype]) * want.abs()).all()


def test_dropout_edges(cuda_device):
    rng = torch.tensor([1, 2], device="cuda")
    x = torch.randn(10, 4 * 6, device="cuda")
    assert torch.equal(ops.irreps_dropout(x, rng, 0.0, 1), x)
    assert torch.equal(ops.irreps_dropout(x, rng, 1.0, 1), torch.zeros_like(x))
    bad = torch.full_like(x, float("nan"))
    assert torch.equal(ops.irreps_dropout(bad, rng, 1.0, 1), torch.zeros_like(x))
    assert ops.irreps_dropout(x[:0], rng, 0.5, 1).shape == (0, 24)
    part = torch.randn(10, 48, device="cuda")[:, ::2]  # strided rows
    assert torch.equal(ops.irreps_dropout(part, rng, 0.5, 1), ops.irreps_dropout(part.contiguous(), rng, 0.5, 1))
    off = torch.randn(241, device="cuda")[1:].view(10, 24)  # misaligned rows
    assert torch.equal(ops.irreps_dropout(off, rng, 0.5, 1), ops.irreps_dropout(off.clone(), rng, 0.5, 1))


def test_dropout_rates_and_independence(cuda_device):
    n, c, p = 4096, 256, 0.2
    x = torch.ones(n, c, device="cuda")
    a = ops.irreps_dropout(x, torch.tensor([3, 0], device="cuda"), p) > 0
    b = ops.irreps_dropout(x, torch.tensor([3, 1], device="cuda"), p) > 0
    # 2^20 draws: the standard deviation of a rate is at most 0.5 / 1024; six of them
    assert abs(a.double().mean().item() - 0.8) < 6 * 0.5 / 1024
    assert abs((a & b).double().mean().item() - 0.64) < 6 * 0.5 / 1024


def test_dropout_more_than_2_to_31_elements(cuda_device):
    n, c = 2 ** 21 + 1, 1028
    x = torch.ones(n, c, dtype=BF16, device="cuda")
    rng = torch.tensor([9, 9], device="cuda")
    y = ops.irreps_dropout(x, rng, 0.5)
    quads = c // 4
    for row in (0, 2 ** 20, n - 1):
        words = [w for q in (0, quads - 1) for w in R.philox(row * quads + q, 9, 9)]
        got = torch.cat([y[row, :4], y[row, -4:]]).float().tolist()
        assert got == [2.0 if w >= 2 ** 31 else 0.0 for w in words]


def test_dropout_differences(cuda_device):
    rng = torch.tensor([4, 4], device="cuda")
    x = torch.randn(3, 9 * 5, dtype=F64, device="cuda", requires_grad=True)
    f = lambda t: ops.irreps_dropout(t, rng, 0.4, 2)
    assert torch.autograd.gradcheck(f, (x,))
    assert torch.autograd.gradgradcheck(lambda t: f(t) ** 2, (x,))


def test_dropout_refusals(cuda_device):
    x, rng = torch.randn(4, 36, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError, match=r"\[0, 1\]"):
            ops.irreps_dropout(x, rng, p)
    with pytest.raises(ValueError, match="rng"):
        ops.irreps_dropout(x, rng.float(), 0.5)
    with pytest.raises(ValueError, match="rng"):
        ops.irreps_dropout(x, rng[:1], 0.5)
    with pytest.raises(NotImplementedError, match="l_max"):
        ops.irreps_dropout(x, rng, 0.5, 4)
    with pytest.raises(ValueError, match="features"):
        ops.irreps_dropout(x[:, :35], rng, 0.5, 2)
    with pytest.raises(ValueError, match="float32, float64 and bfloat16"):
        ops.irreps_dropout(x.half(), rng, 0.5)


# ------------------------------------------------------------------------------ gated block


def _rel(got, want):
    d = (got.double() - want).norm().item()
    return d / max(want.norm().item(), 1e-300)


def _gated_tol(dtype, k, rows):
    """Relative 2-norm error. float64: rounding of sums. float32: three terms of 2^-22 per
    product (the rounded low parts and the dropped low x low), 48 truncating accumulations per
    unit of 128 products, one float32 addition per unit of the reduction. bfloat16: the same
    (one term) and one rounding to 8 bits."""
    if dtype == F64:
        return 2.0 ** -53 * (16 + 2 * k + rows)
    acc = 3 * 2.0 ** -22 + 48 * 2.0 ** -24 + (k + rows) / 128 * 2.0 ** -24
    return acc + (2.0 ** -8 if dtype == BF16 else 0.0)


# one row, odd and tiny channels, widths around the 32- and 128-wide tiles, rows around the
# 128-row tile, hidden width unlike the input's, more than one tile of channels
GATED = [(1, 0, 1, 1), (3, 0, 5, 7), (130, 0, 33, 70), (128, 0, 128, 128), (257, 0, 200, 72), (300, 0, 96, 200),
         (1, 1, 4, 4), (127, 1, 36, 20), (129, 2, 64, 64), (40, 2, 31, 66), (97, 3, 128, 128), (200, 3, 8, 136),
         (33, 3, 132, 40), (2000, 1, 64, 32), (5000, 0, 16, 16)]


@pytest.mark.parametrize("act,bias", [("silu", True), ("sigmoid", False)])
@pytest.mark.parametrize("dtype", [F32, F64, BF16])
@pytest.mark.parametrize("n,l_max,c,h", GATED)
def test_gated_and_gradients(cuda_device, dtype, n, l_max, c, h, act, bias):
    x, wv, wg, b, sc, g = R.gated_inputs(n, l_max, c, h, bias, dtype, "cuda", seed=n + c)
    ins = [x, wg, *([b] if bias else []), *wv]
    for t in ins:
        t.requires_grad_(True)
    y = ops.gated_feed_forward(x, wv, wg, b, sc, l_max, act)
    got = torch.autograd.grad(y, ins, g)
    want_y, want = R.gated_grads(x, wv, wg, b, sc, l_max, act, g)
    want = [t for t in want if t is not None]
    assert y.dtype == dtype and all(t.dtype == dtype for t in got)
    assert _rel(y.detach(), want_y) <= _gated_tol(dtype, c, 0)
    assert _rel(got[0], want[0]) <= _gated_tol(dtype, (l_max + 2) * h, 0)
    for a, w in zip(got[1:], want[1:]):
        assert _rel(a, w) <= _gated_tol(dtype, c, n * (2 * l_max + 1))
    with torch.no_grad():
        assert torch.equal(ops.gated_feed_forward(x, wv, wg, b, sc, l_max, act), y)
    again = torch.autograd.grad(ops.gated_feed_forward(x, wv, wg, b, sc, l_max, act), ins, g)
    assert all(torch.equal(p, q) for p, q in zip(got, again))
    ops.check_device_status()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gated_water_box_size(cuda_device, dtype):
    n, l_max, c, h = 27648, 3, 128, 128
    x, wv, wg, b, sc, g = R.gated_inputs(n, l_max, c, h, True, dtype, "cuda", seed=5)
    ins = [x, wg, b, *wv]
    for t in ins:
        t.requires_grad_(True)
    y = ops.gated_feed_forward(x, wv, wg, b, sc, l_max, "sigmoid")
    got = torch.autograd.grad(y, ins, g)
    want_y, want = R.gated_grads(x, wv, wg, b, sc, l_max, "sigmoid", g)
    assert _rel(y.detach(), want_y) <= _gated_tol(dtype, c, 0)
    assert _rel(got[0], want[0]) <= _gated_tol(dtype, 5 * h, 0)
    for a, w in zip(got[1:], want[1:]):
        assert _rel(a, w) <= _gated_tol(dtype, c, 7 * n)


@pytest.mark.parametrize("dtype,n,l_max,c,h", [(F32, 27648, 3, 128, 128), (BF16, 27648, 3, 128, 128),
                                               (F32, 9001, 2, 200, 136), (BF16, 100003, 0, 96, 200),
                                               (F32, 13869, 3, 48, 88), (F32, 27648, 2, 96, 96),
                                               (F32, 27648, 3, 24, 32), (F32, 27648, 1, 160, 224),
                                               (BF16, 20001, 2, 40, 72), (BF16, 9001, 1, 300, 136)])
def test_gated_large_passes_repeat_their_bits(cuda_device, dtype, n, l_max, c, h):
    # one ring stage refilled while a few of its values are still being read shows in one product of
    # 10^5: about one pass of three at these sizes, so a hundred passes show it. Odd numbers of slabs
    # (88, 96, 24 channels): weights used before they are there
    x, wv, wg, _, scales, g = R.gated_inputs(n, l_max, c, h, False, dtype, "cuda", seed=3)
    for t in (x, wg, *wv):
        t.requires_grad_(True)
    want = None
    for _ in range(100):
        y = ops.gated_feed_forward(x, wv, wg, None, scales, l_max, "silu")
        got = [y.detach(), *torch.autograd.grad(y, [x, wg, *wv], g)]
        want = want or got
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gated_more_than_2_to_31_elements(cuda_device, dtype):
    # 1,100 times the same 1,000 rows: every copy has the first one's results, and the weights'
    # gradients are 1,100 times its own
    n, reps, l_max, c = 1000, 1100, 3, 128
    x, wv, wg, b, sc, g = R.gated_inputs(n, l_max, c, c, True, dtype, "cuda", seed=7)
    ins = [wg, b, *wv]
    for t in ins:
        t.requires_grad_(True)

    def both(x, g):
        x = x.requires_grad_(True)
        y = ops.gated_feed_forward(x, wv, wg, b, sc, l_max, "silu")
        return y.detach(), *torch.autograd.grad(y, [x, *ins], g)

    want_y, want_x, *_ = both(x.clone(), g)
    _, exact = R.gated_grads(x, wv, wg, b, sc, l_max, "silu", g)
    y, gx, *got = both(x.repeat(reps, 1), g.repeat(reps, 1))
    assert y.numel() > 2 ** 31
    assert bool((y.view(reps, n, -1) == want_y).all()) and bool((gx.view(reps, n, -1) == want_x).all())
    for a, w in zip(got, exact[1:]):
        assert _rel(a, reps * w) <= _gated_tol(dtype, c, 7 * n * reps)


def test_gated_subsets_of_gradients(cuda_device):
    x, wv, wg, b, sc, g = R.gated_inputs(300, 2, 64, 64, True, F32, "cuda")
    every = [x, wg, b, *wv]
    for t in every:
        t.requires_grad_(True)
    full = torch.autograd.grad(ops.gated_feed_forward(x, wv, wg, b, sc, 2, "silu"), every, g)
    for only in range(len(every)):
        for k, t in enumerate(every):
            t.requires_grad_(k == only)
        (got,) = torch.autograd.grad(ops.gated_feed_forward(x, wv, wg, b, sc, 2, "silu"), [every[only]], g)
        assert torch.equal(got, full[only])


def test_gated_zero_rows(cuda_device):
    x, wv, wg, b, sc, g = R.gated_inputs(0, 1, 8, 8, True, F32, "cuda")
    ins = [x, wg, b, *wv]
    for t in ins:
        t.requires_grad_(True)
    y = ops.gated_feed_forward(x, wv, wg, b, sc, 1, "silu")
    got = torch.autograd.grad(y, ins, g)
    assert y.shape == (0, 32) and all((t == 0).all() for t in got)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gated_layouts(cuda_device, dtype):
    """Strided rows, misaligned tensors and another stream give the contiguous result."""
    x, wv, wg, b, sc, g = R.gated_inputs(150, 1, 32, 32, True, dtype, "cuda")
    want = ops.gated_feed_forward(x, wv, wg, b, sc, 1, "silu")
    wide = torch.empty(150, 2 * x.shape[1], dtype=dtype, device="cuda")
    wide[:, ::2] = x
    assert torch.equal(ops.gated_feed_forward(wide[:, ::2], wv, wg, b, sc, 1, "silu"), want)
    off = torch.empty(x.numel() + 1, dtype=dtype, device="cuda")[1:].view_as(x)
    off.copy_(x)
    woff = torch.empty(wg.numel() + 1, dtype=dtype, device="cuda")[1:].view_as(wg)
    woff.copy_(wg)
    ins, outs = [off, woff, b, *wv], []
    for rows, gate in ((x, wg), (off, woff)):
        leaves = [t.detach().requires_grad_(True) for t in (rows, gate, b, *wv)]
        y = ops.gated_feed_forward(leaves[0], leaves[3:], leaves[1], leaves[2], sc, 1, "silu")
        outs.append([y.detach(), *torch.autograd.grad(y, leaves, g)])
    for p, q in zip(*outs):
        assert _rel(p, q.double()) <= _gated_tol(dtype, 3 * 32, 450)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = ops.gated_feed_forward(x, wv, wg, b, sc, 1, "silu")
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, want)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf"), 1e30])
def test_gated_rows_do_not_reach_each_other(cuda_device, dtype, value):
    x, wv, wg, b, sc, g = R.gated_inputs(200, 1, 64, 64, True, dtype, "cuda")
    clean = ops.gated_feed_forward(x, wv, wg, b, sc, 1, "silu")
    x2 = x.clone()
    x2[77, 3] = value
    x2[131, 64 + 5] = value
    y = ops.gated_feed_forward(x2, wv, wg, b, sc, 1, "silu")
    keep = torch.ones(200, dtype=torch.bool, device="cuda")
    keep[[77, 131]] = False
    assert torch.equal(y[keep], clean[keep])
    assert torch.equal(y[131, :64], clean[131, :64])  # its scalars do not see the bad component


def test_gated_saturated_gates(cuda_device):
    """Pre-activations far beyond the exponential's range: gates of 0 and 1, no NaN."""
    n, c = 64, 8
    x = torch.ones(n, c, device="cuda", requires_grad=True)
    w = torch.eye(c, device="cuda").requires_grad_(True)
    b = torch.tensor([-1e4, -200.0, -90.0, -30.0, 30.0, 90.0, 200.0, 1e4], device="cuda")
    sc = torch.tensor([1.0, 1.0, 1.0], device="cuda")
    for act in ("sigmoid", "silu"):
        y = ops.gated_feed_forward(x, [w], w, b, sc, 0, act)
        z = 1.0 + b.double()
        s = torch.sigmoid(z)
        want = s if act == "sigmoid" else z * s
        assert ((y.detach().double() - want).abs() <= 1e-6 * want.abs() + 1e-30).all()
        gx, gw = torch.autograd.grad(y, [x, w], torch.ones_like(y))
        assert torch.isfinite(gx).all() and torch.isfinite(gw).all()


@pytest.mark.parametrize("l_max,act", [(0, "silu"), (1, "sigmoid"), (2, "silu")])
def test_gated_differences_and_second_derivative(cuda_device, l_max, act):
    x, wv, wg, b, sc, _ = R.gated_inputs(3, l_max, 3, 2, True, F64, "cuda")
    ins = [x, wg, b, *wv]
    for t in ins:
        t.requires_grad_(True)
    f = lambda x, wg, b, *wv: ops.gated_feed_forward(x, list(wv), wg, b, sc, l_max, act)
    assert torch.autograd.gradcheck(f, ins)
    assert torch.autograd.gradgradcheck(f, ins)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gated_second_derivative_close_to_float64(cuda_device, dtype):
    """A force-like loss: the gradient of a function of the input gradient."""
    x, wv, wg, b, sc, g = R.gated_inputs(50, 1, 16, 16, True, dtype, "cuda")

    def second(x, wv, wg, b, sc, f):
        ins = [x, wg, b, *wv]
        gx = torch.autograd.grad(f(x, wv, wg, b, sc), x, g.to(x.dtype), create_graph=True)[0]
        return torch.autograd.grad((gx.double() ** 2).sum(), ins, allow_unused=True)

    leaf = lambda t, dt: t.detach().to(dt).requires_grad_(True)
    pick = lambda dt: (leaf(x, dt), [leaf(w, dt) for w in wv], leaf(wg, dt), leaf(b, dt))
    got = second(*pick(dtype), sc, lambda *a: ops.gated_feed_forward(*a, 1, "silu"))
    want = second(*pick(F64), sc.double(), lambda *a: R.gated(*a, 1, "silu"))
    for p, q in zip(got, want):
        assert _rel(p, q) <= (5e-5 if dtype == F32 else 0.03)


def test_gated_registered_operator(cuda_device):
    x, wv, wg, b, sc, g = R.gated_inputs(60, 1, 8, 12, True, F32, "cuda")
    ins = [x, wg, b, *wv]
    for t in ins:
        t.requires_grad_(True)
    a = ops.gated_feed_forward(x, wv, wg, b, sc, 1, "sigmoid")
    o = torch.ops.flashcart.gated_ff_fwd(x, wv, wg, b, sc, 1, "sigmoid")
    assert torch.equal(a, o)
    for p, q in zip(torch.autograd.grad(a, ins, g), torch.autograd.grad(o, ins, g)):
        assert torch.equal(p, q)


def test_gated_refusals(cuda_device):
    x, wv, wg, b, sc, _ = R.gated_inputs(4, 1, 8, 4, True, F32, "cuda")
    call = lambda x=x, wv=wv, wg=wg, b=b, sc=sc, l_max=1, act="silu": ops.gated_feed_forward(x, wv, wg, b, sc, l_max,
                                                                                             act)
    call()
    for error, match, kw in [
            (ValueError, "activation", dict(act="relu")), (NotImplementedError, "l_max", dict(l_max=4)),
            (ValueError, "value weights expected", dict(wv=wv[:1])), (ValueError, "hidden, in", dict(wv=[wv[0], wv[1].T])),
            (ValueError, "gate_weight", dict(wg=wg[:4])), (ValueError, "gate_bias", dict(b=b[:4])),
            (RuntimeError, "last dimension", dict(x=x[:, :31])), (ValueError, "type of x", dict(wg=wg.double())),
            (ValueError, "scales", dict(sc=sc[:3])), (ValueError, "scales", dict(sc=sc.double())),
            (RuntimeError, "CUDA", dict(wg=wg.cpu())),
            (ValueError, "float32, float64 and bfloat16", dict(x=x.half()))]:
        with pytest.raises(error, match=match):
            call(**kw)
