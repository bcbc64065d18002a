"""Training-block operators on the GPU where a rule of their launches ends: empty tables, the
largest rows and widths, several host threads, sizes whose races or rounding small ones hide."""

import ctypes
import threading

import pytest
import torch

import block_refs as R
from flashcart_b200 import _native as N
from flashcart_b200 import ops
from flashcart_b200.nn.blocks import IrrepsDropout

pytestmark = pytest.mark.gpu

F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16


@pytest.mark.parametrize("dtype", [F32, F64, BF16])
@pytest.mark.parametrize("dim", [3, 5, 8, 63, 64])
def test_embedding_in_an_empty_table(cuda_device, dtype, dim):
    """No row to read: zeros, the status bit, and a gradient without rows."""
    ops.check_device_status()
    table = torch.empty(0, dim, dtype=dtype, device="cuda", requires_grad=True)
    for rows in (1, 259):
        idx = torch.arange(rows, device="cuda") - 1
        y = ops.embedding(table, idx, 2.0, 1.0)
        assert torch.equal(y, torch.zeros(rows, dim, dtype=dtype, device="cuda"))
        (g,) = torch.autograd.grad(y, table, torch.ones_like(y))
        assert g.shape == (0, dim)
        with pytest.raises(RuntimeError, match="outside"):
            ops.check_device_status()
    assert ops.embedding(table, idx[:0]).shape == (0, dim)
    ops.check_device_status()


def _leaves(*ts):
    return [None if t is None else t.detach().clone().requires_grad_(True) for t in ts]


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("use", ["twice", "value and gate", "two ranks"])
def test_gated_weights_in_two_places(cuda_device, graph, use):
    """A weight used by two calls of which one feeds the other, and one tensor as two of a call's
    weights: every gradient is the definition's, whether or not the backward builds a graph."""
    l_max = 1 if use == "two ranks" else 0
    x, wv, wg, b, sc, g = R.gated_inputs(7, l_max, 6, 6, True, F64, "cuda", seed=1)

    def run(f):
        xs, w0, w1, gate, bias = _leaves(x, wv[0], wv[-1], wg, b)
        ws = [w0, w0] if use == "two ranks" else [w0]
        gate = w0 if use == "value and gate" else gate
        y = f(xs, ws, gate, bias, sc, l_max, "silu")
        if use == "twice":
            y = f(y, ws, gate, bias, sc, l_max, "silu")
        ins = [xs, w0, bias] + ([] if use == "value and gate" else [gate])
        return [t.detach() for t in torch.autograd.grad(y, ins, g, create_graph=graph)]

    for got, want in zip(run(ops.gated_feed_forward), run(R.gated)):
        # sums of some dozen terms, twice over
        assert ((got - want).norm() / want.norm()).item() <= 2.0 ** -53 * 512


@pytest.mark.parametrize("graph", [False, True])
def test_gated_gradient_hooks_run_once(cuda_device, graph):
    """A hook that scales a gradient scales it once, and none runs for what is not asked for."""
    x, wv, wg, b, sc, g = R.gated_inputs(5, 1, 4, 4, True, F64, "cuda", seed=2)

    def run(f, hooks):
        xs, w0, w1, gate, bias = _leaves(x, *wv, wg, b)
        seen = []
        if hooks:
            for name, t, k in (("x", xs, 10.0), ("w", w0, 3.0), ("gate", gate, 7.0)):
                t.register_hook(lambda v, name=name, k=k: seen.append(name) or k * v)
        y = f(xs, [w0, w1], gate, bias, sc, 1, "sigmoid")
        return torch.autograd.grad(y, [xs, w0, gate, bias], g, create_graph=graph), seen

    (gx, gw, gg, gb), seen = run(ops.gated_feed_forward, True)
    assert sorted(seen) == ["gate", "w", "x"]
    plain, _ = run(ops.gated_feed_forward, False)
    for got, want, k in zip((gx, gw, gg, gb), plain, (10.0, 3.0, 7.0, 1.0)):
        assert torch.equal(got, k * want)
    xs, w0, w1, gate, bias = _leaves(x, *wv, wg, b)
    w0.register_hook(lambda v: pytest.fail("the weight's gradient was not asked for"))
    torch.autograd.grad(ops.gated_feed_forward(xs, [w0, w1], gate, bias, sc, 1, "sigmoid"), xs, g, create_graph=graph)


def test_forward_mode(cuda_device):
    """Tangents of the linear operators (also where nothing needs a gradient); the gated block,
    which has none, says so."""
    fw = torch.autograd.forward_ad
    gen = torch.Generator().manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=F64).cuda()
    idx = torch.tensor([0, 4, 4, 1], device="cuda")
    rng = torch.tensor([4, 4], device="cuda")
    table, t_table, x, t_x = r(5, 3), r(5, 3), r(3, 9 * 5), r(3, 9 * 5)
    for grad in (False, True):
        with fw.dual_level():
            dual = lambda t, v: fw.make_dual(t.clone().requires_grad_(grad), v)
            y = fw.unpack_dual(ops.embedding(dual(table, t_table), idx, 0.7, 1.0))
            assert torch.equal(y.primal.detach(), ops.embedding(table, idx, 0.7, 1.0))
            assert torch.equal(y.tangent, ops.embedding(t_table, idx, 0.7))
            y = fw.unpack_dual(ops.irreps_dropout(dual(x, t_x), rng, 0.4, 2))
            assert torch.equal(y.tangent, ops.irreps_dropout(t_x, rng, 0.4, 2))
            gx, wv, wg, b, sc, _ = R.gated_inputs(3, 1, 4, 4, True, F64, "cuda")
            with pytest.raises(NotImplementedError, match="forward-mode"):
                ops.gated_feed_forward(dual(gx, gx), wv, wg, b, sc, 1, "silu")
            ops.gated_feed_forward(gx, wv, wg, b, sc, 1, "silu")  # nothing to carry: as ever
    t = table.clone().requires_grad_(True)
    assert torch.autograd.gradcheck(lambda w: ops.embedding(w, idx, 0.7, 1.0), (t,), check_forward_ad=True)
    assert torch.autograd.gradgradcheck(lambda w: ops.embedding(w, idx, 0.7, 1.0) ** 2, (t,), check_fwd_over_rev=True)
    t = x.clone().requires_grad_(True)
    assert torch.autograd.gradcheck(lambda v: ops.irreps_dropout(v, rng, 0.4, 2), (t,), check_forward_ad=True)


def test_calls_are_recorded(cuda_device):
    """Traced programs hold the operators, not what a call past the dispatcher leaves behind."""
    from torch.fx.experimental.proxy_tensor import make_fx

    x, wv, wg, b, sc, _ = R.gated_inputs(6, 0, 8, 8, True, F32, "cuda")
    rng = torch.tensor([1, 2], device="cuda")
    idx = torch.arange(6, device="cuda") % 3

    def f(x, w, table):
        y = ops.gated_feed_forward(x + ops.embedding(table, idx), [w], wg, b, sc, 0, "silu")
        return ops.irreps_dropout(y, rng, 0.5)

    table = torch.randn(3, 8, device="cuda")
    other = (x * 2, wv[0] - 1, table + 1)
    for traced in (make_fx(f)(x, wv[0], table), torch.jit.trace(f, (x, wv[0], table), check_trace=False)):
        assert torch.equal(traced(*other), f(*other))


@pytest.mark.parametrize("l_max,act,bias", [(0, "silu", False), (1, "sigmoid", True)])
def test_registered_gated_operator_twice(cuda_device, l_max, act, bias):
    """The registered operator's second derivative: differences, and the entry point's."""
    x, wv, wg, b, sc, g = R.gated_inputs(3, l_max, 3, 2, bias, F64, "cuda")
    ins = [t.requires_grad_(True) for t in (x, wg, *([b] if bias else []), *wv)]
    n = 3 if bias else 2
    f = lambda op: lambda x, wg, *rest: op(x, list(rest[n - 2:]), wg, rest[0] if bias else None, sc, l_max, act)
    registered = f(torch.ops.flashcart.gated_ff_fwd)
    assert torch.autograd.gradgradcheck(registered, ins)
    second = []
    for call in (registered, f(ops.gated_feed_forward)):
        (gx,) = torch.autograd.grad(call(*ins), x, g, create_graph=True)
        second.append(torch.autograd.grad(gx.square().sum(), ins))
    for a, c in zip(*second):
        assert ((a - c).norm() / c.norm()).item() <= 1e-13  # some hundred roundings of 2^-53


@pytest.mark.parametrize("reentrant", [False, True])
def test_dropout_under_checkpointing(cuda_device, reentrant):
    """A recomputed forward has the mask that the loss had; a layer with a stream of its own,
    which cannot know it, refuses."""
    from torch.utils.checkpoint import checkpoint

    layer = IrrepsDropout(0.5, l_max=1).train()
    x = torch.randn(200, 4 * 8, device="cuda", requires_grad=True)
    for _ in range(2):  # the second call's recomputation is not the first's mask
        y = checkpoint(lambda t: layer(t) * 1.0, x, use_reentrant=reentrant)
        want = y.detach() / x.detach()
        x.grad = None
        y.sum().backward()
        assert torch.allclose(x.grad, want, rtol=1e-6, atol=0)
        assert set(want.round().unique().tolist()) == {0.0, 2.0}
    own = IrrepsDropout(0.5, l_max=1, seed=3).cuda().train()
    y = checkpoint(lambda t: own(t) * 1.0, x, use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match="leave the seed out"):
        y.sum().backward()


def test_dropout_follows_torch_generator(cuda_device):
    layer = IrrepsDropout(0.5).train()
    x = torch.ones(100, 16, device="cuda")
    torch.manual_seed(1)
    a, state, b = layer(x), torch.cuda.get_rng_state(), layer(x)
    assert not torch.equal(a, b)
    torch.cuda.set_rng_state(state)
    assert torch.equal(layer(x), b)
    torch.manual_seed(1)
    assert torch.equal(layer(x), a)
    torch.manual_seed(2)
    assert not torch.equal(layer(x), a)
    assert not list(layer.state_dict()) and IrrepsDropout(0.5).cuda().eval()(x) is x
    # a captured step draws on with every replay
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(x)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        y = layer(x)
    graph.replay()
    first = y.clone()
    graph.replay()
    assert not torch.equal(first, y)


def test_embedding_gradients_from_several_threads(cuda_device):
    """Host threads whose calls need different shared memory of the one-block sort."""
    errors = []

    def work(rows):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                idx = torch.arange(rows, device="cuda") % 5
                grad = torch.ones(rows, 4, device="cuda")
                want = torch.bincount(idx, minlength=5).float()[:, None].expand(5, 4)
                for _ in range(300):
                    got = torch.ops.flashcart.embedding_bwd(grad, idx, 5, 1.0)
                assert torch.equal(got, want)
        except Exception as e:  # told to the main thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(rows,)) for rows in (8192, 7, 8000, 64, 6000, 900)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


@pytest.mark.parametrize("dtype", [F32, F64])
def test_embedding_of_the_widest_rows(cuda_device, dtype):
    """2^22 features, over several chunks of sorted rows: the joining kernel's column tiles exceed
    what a launch takes in 64 bits."""
    rows, dim = 264, 2 ** 22  # (chunks are up to 256 rows)
    idx = torch.arange(rows, device="cuda") % 2
    grad = torch.ones(rows, dim, dtype=dtype, device="cuda")
    grad[:, -1] = 2.0
    got = torch.ops.flashcart.embedding_bwd(grad, idx, 2, 1.0)
    assert bool((got[:, :-1] == rows // 2).all()) and bool((got[:, -1] == rows).all())


def test_gated_float64_of_the_widest_gates(cuda_device):
    """2^20 hidden channels in four ranks: the gates' column tiles exceed what a launch takes."""
    x, wv, wg, b, sc, g = R.gated_inputs(2, 3, 1, 2 ** 20, False, F64, "cuda")
    x.requires_grad_(True)
    y = ops.gated_feed_forward(x, wv, wg, None, sc, 3, "silu")
    (gx,) = torch.autograd.grad(y, x, g)
    want_y, (want_x, *_) = R.gated_grads(x, wv, wg, None, sc, 3, "silu", g)
    # one product a value; sums of 5 x 2^20 terms whose roundings do not add up in one direction
    assert ((y.detach() - want_y).norm() / want_y.norm()).item() <= 2.0 ** -53 * 32
    assert ((gx - want_x).norm() / want_x.norm()).item() <= 2.0 ** -53 * 5 * 2 ** 20


@pytest.mark.parametrize("dtype,code", [(F32, N.FC_F32), (BF16, N.FC_BF16)])
def test_gated_workspace_holds_what_a_call_needs(cuda_device, dtype, code):
    """Nothing of the size of x for a forward, and dv and dz for a backward; what padded copies
    there are, rows that need them have."""
    n, l_max, c = 27648, 3, 128
    size = torch.empty(0, dtype=dtype).element_size()
    query = lambda c, h, back: N.lib().fc_gated_ff_workspace_bytes(
        ctypes.byref(N.GatedFfDesc(l_max, c, h, N.FC_GATE_SILU, code)), n, back)
    assert query(c, c, 0) <= 8 * 2 ** 20
    # (both in float, or two bfloat16 parts) and the partial weight gradients
    assert query(c, c, 1) <= n * (16 + 4) * c * 4 + 64 * 2 ** 20
    odd = n * 16 * 33 * size
    assert query(33, c, 0) >= odd and query(c, 33, 0) >= odd
    assert query(33, c, 1) >= n * 20 * c * 4 + 2 * odd and query(c, 33, 1) >= n * 20 * 33 * 4 + odd


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("c,h", [(32, 32), (33, 32), (32, 33), (7, 9)])
def test_gated_misaligned_rows(cuda_device, dtype, c, h):
    """Rows whose memory begins off a 16-byte boundary, with and without whole vectors."""
    x, wv, wg, b, sc, g = R.gated_inputs(150, 1, c, h, True, dtype, "cuda")
    off = lambda t: torch.empty(t.numel() + 1, dtype=dtype, device="cuda")[1:].view_as(t).copy_(t)
    got = []
    for rows, grad in ((x, g), (off(x), off(g))):
        ins = [t.detach().requires_grad_(True) for t in (rows, wg, b, *wv)]
        y = ops.gated_feed_forward(ins[0], ins[3:], ins[1], ins[2], sc, 1, "silu")
        got.append([y.detach(), *torch.autograd.grad(y, ins, grad)])
    assert all(torch.equal(p, q) for p, q in zip(*got))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("c", [8, 136, 264])
@pytest.mark.parametrize("act", ["sigmoid", "silu"])
def test_gated_gates_at_the_ends_of_the_type(cuda_device, dtype, c, act):
    """Pre-activations up to the type's largest value: gates of 0 and 1, finite gradients."""
    x = torch.ones(4, c, dtype=dtype, device="cuda", requires_grad=True)
    w = (torch.eye(c, device="cuda") / 4).to(dtype).requires_grad_(True)
    b = torch.tensor([-3.3e38, -2.5e38, -2.3e38, -1e38, 1e38, 2.3e38, 2.5e38, 3.3e38], device="cuda").to(dtype)
    bias = b.repeat(c // 8)
    sc = torch.ones(3, device="cuda")
    y = ops.gated_feed_forward(x, [w], w, bias, sc, 0, act)
    z = (bias.double() + 0.25).float().double()
    want = torch.where(z > 0, torch.ones_like(z) if act == "sigmoid" else z, torch.zeros_like(z)) / 4
    # the product, the sum with the bias and the gate are one rounding each, then the storage's
    assert ((y.double() - want).abs() <= (4 * 2.0 ** -24 + (2.0 ** -8 if dtype == BF16 else 0)) * want).all()
    gx, gw = torch.autograd.grad(y, [x, w], torch.full_like(y, 2.0 ** -20))
    assert torch.isfinite(gx).all() and torch.isfinite(gw).all()


@pytest.mark.parametrize("l_max", [0, 1])
@pytest.mark.parametrize("c", [320, 1024, 4096, 16384])
def test_gated_error_of_long_reductions(cuda_device, c, l_max):
    """float32 results from long rows. Two chained products (z and v, then the gradient's), each
    with three terms of 2^-22 (the parts' rounding, the left-out low x low) and 48 truncating
    accumulations in a unit of the reduction; the units' additions are rounded, so they grow the
    error by the square root of their number at most: 2^-24 times 16 for 256 units."""
    x, wv, wg, b, sc, g = R.gated_inputs(64, l_max, c, 40, True, F32, "cuda", seed=c)
    ins = [t.requires_grad_(True) for t in (x, wg, b, *wv)]
    y = ops.gated_feed_forward(x, wv, wg, b, sc, l_max, "silu")
    want_y, want = R.gated_grads(x, wv, wg, b, sc, l_max, "silu", g)
    bound = 2 * (3 * 2.0 ** -22 + 48 * 2.0 ** -24 + 16 * 2.0 ** -24)
    for got, ref in zip((y.detach(), *torch.autograd.grad(y, ins, g)), (want_y, *want)):
        assert ((got.double() - ref).norm() / ref.norm()).item() <= bound


def test_kernel_timer_counts_launches(cuda_device):
    """What the timer counts for a call is what the GPU ran, whatever the sizes."""
    from torch.profiler import ProfilerActivity, profile

    own = ("embed_", "sort_", "dropout_kernel", "gated_", "wgrad_", "prep_kernel", "repitch_kernel")

    def count(f):
        timer = ops.KernelTimer()
        torch.cuda.synchronize()
        with profile(activities=[ProfilerActivity.CUDA]) as prof:
            ops.set_kernel_timer(timer)
            try:
                f()
            finally:
                ops.set_kernel_timer(None)
            torch.cuda.synchronize()
        seen = [e for e in prof.events() if e.device_type == torch.autograd.DeviceType.CUDA
                and any(name in e.name for name in own)]
        return timer.launches, len(seen)

    def embed(rows, types, dim):
        idx = torch.arange(rows, device="cuda") % types
        grad = torch.ones(rows, dim, device="cuda")
        return lambda: torch.ops.flashcart.embedding_bwd(grad, idx, types, 1.0)

    def gated(n, l_max, c, h, dtype, only_x=False):
        x, wv, wg, b, sc, g = R.gated_inputs(n, l_max, c, h, True, dtype, "cuda")
        ins = [t.requires_grad_(True) for t in ((x,) if only_x else (x, wg, b, *wv))]
        return lambda: torch.autograd.grad(ops.gated_feed_forward(x, wv, wg, b, sc, l_max, "silu"), ins, g)

    x, rng = torch.ones(50, 64, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    calls = [lambda: ops.irreps_dropout(x, rng, 0.5), lambda: ops.embedding(x, rng), embed(10, 2, 8), embed(9000, 3, 8),
             embed(200_000, 300, 64), embed(200_000, 70_000, 4), embed(200_000, 3, 4), gated(40, 1, 32, 32, F32),
             gated(40, 1, 33, 31, F32), gated(40, 0, 200, 40, F32, True), gated(40, 1, 32, 32, BF16),
             gated(40, 0, 300, 33, BF16), gated(40, 1, 5, 7, F64)]
    for f in calls:
        f()
    counts = [count(f) for f in calls]
    if not any(seen for _, seen in counts):
        pytest.skip("the profiler records no kernels here")
    assert all(a == b and a > 0 for a, b in counts), counts


@pytest.mark.parametrize("dtype,n,l_max,c,h", [(F32, 27648, 3, 128, 128), (BF16, 27648, 3, 128, 128),
                                               (F32, 9001, 2, 200, 136), (BF16, 100003, 0, 96, 200),
                                               (F32, 13869, 3, 48, 88), (F32, 27648, 2, 96, 96),
                                               (F32, 27648, 3, 24, 32), (F32, 27648, 1, 160, 224),
                                               (F32, 9001, 1, 320, 352), (BF16, 20001, 2, 40, 72),
                                               (BF16, 9001, 1, 300, 136), (BF16, 20001, 1, 72, 264)])
def test_gated_large_passes_are_right(cuda_device, dtype, n, l_max, c, h):
    """The first passes at sizes whose kernels have every role busy, against 64 bits: weights or rows
    used before they are there, or after they have gone, show here (odd and even numbers of slabs,
    resident and streamed weights). Errors as in test_gated_error_of_long_reductions; bfloat16
    results add one rounding to 8 bits, and what is handed between the backward's halves in two
    bfloat16 parts (2^-17)."""
    x, wv, wg, _, scales, g = R.gated_inputs(n, l_max, c, h, False, dtype, "cuda", seed=3)
    ins = [t.requires_grad_(True) for t in (x, wg, *wv)]
    want_y, want = R.gated_grads(x, wv, wg, None, scales, l_max, "silu", g)
    want = [want_y, *(t for t in want if t is not None)]
    bound = 2 * (3 * 2.0 ** -22 + 48 * 2.0 ** -24 + 16 * 2.0 ** -24) + (2.0 ** -8 + 2.0 ** -17 if dtype == BF16 else 0.0)
    for _ in range(3):
        y = ops.gated_feed_forward(x, wv, wg, None, scales, l_max, "silu")
        for got, ref in zip((y.detach(), *torch.autograd.grad(y, ins, g)), want):
            assert ((got.double() - ref).norm() / ref.norm()).item() <= bound
            # and no single row off: a few wrong values hide in a norm over 10^8
            worst = (got.double() - ref).abs().amax() / ref.abs().amax()
            assert worst.item() <= 16 * bound


def test_gated_force_step_is_captured(cuda_device):
    """A step with a second derivative in a CUDA graph: the replay's gradients are the eager ones."""
    x, wv, wg, b, sc, g = R.gated_inputs(40, 2, 16, 24, True, F32, "cuda", seed=8)
    ins = [t.requires_grad_(True) for t in (x, wg, b, *wv)]

    def step():
        y = ops.gated_feed_forward(x, wv, wg, b, sc, 2, "silu")
        (gx,) = torch.autograd.grad(y, x, g, create_graph=True)
        return torch.autograd.grad(gx.square().sum(), ins)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for t in got:
        t.zero_()
    graph.replay()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
