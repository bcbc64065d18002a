"""The training blocks inside the potential: same parameters and results as the layers they
stand for, differentiable twice, dropout that commutes with rotations."""

import copy

import pytest
import torch
import torch.nn as nn

from flashcart_b200.model.flashcart import FlashCartPotential
from flashcart_b200.nn.blocks import GatedFeedForward, IrrepsDropout, ScaledEmbedding, use_training_blocks
from flashcart_b200.nn.layers import EquivariantGatedLayer
from flashcart_b200.training import batch_graph, energy_force_loss, synthetic_molecules

ARCH = dict(elements=["H", "C", "N", "O"], r_max=4.0, n_hidden_feats=16, l_max_hidden_feats=2, l_max_edge_attrs=2,
            n_radial=6, n_interactions=2, correlation=2, layer_norm=True, nonlinearity=True, avg_neighbors=12.0,
            element_agnostic_interaction=False, element_agnostic_product=False, n_element_interaction_features=8)


def _model(**kw):
    torch.manual_seed(0)
    model = FlashCartPotential(**dict(ARCH, **kw))
    with torch.no_grad():  # the zero-initialised parts must not hide the blocks
        for layer in model.nonlinearities:
            for w in layer.output_linear.weight:
                w.normal_()
        for product in model.products:
            for w in product.path_weights:
                if w.element_dependent:
                    w.delta.weight.normal_(0, 0.1)
    return model


def test_blocks_keep_parameters_and_names():
    stock = _model()
    keys = {k: v.clone() for k, v in stock.state_dict().items()}
    params = {id(p) for p in stock.parameters()}
    state = torch.random.get_rng_state()
    blocks = use_training_blocks(stock, dropout=0.1)
    assert torch.equal(torch.random.get_rng_state(), state)
    got = blocks.state_dict()
    assert list(got) == list(keys) and all(torch.equal(got[k], keys[k]) for k in keys)
    assert {id(p) for p in blocks.parameters()} == params
    assert isinstance(blocks.embedding, ScaledEmbedding)
    assert all(isinstance(m, GatedFeedForward) for m in blocks.nonlinearities)
    ids = lambda it: [id(p) for p in it]
    again = _model()
    named = dict(again.named_parameters())
    want = [n for n, p in named.items() if id(p) in set(ids(again.non_muon_parameters()))]
    have = [n for n, p in blocks.named_parameters() if id(p) in set(ids(blocks.non_muon_parameters()))]
    assert want == have


def test_block_refusals():
    with pytest.raises(ValueError, match=r"\[0, 1\]"):
        IrrepsDropout(1.5)
    with pytest.raises(ValueError, match="positive"):
        ScaledEmbedding(0, 4)
    with pytest.raises(ValueError, match="weight must be"):
        ScaledEmbedding(3, 4, weight=nn.Parameter(torch.zeros(4, 3)))
    with pytest.raises(ValueError, match="gate_activation"):
        GatedFeedForward(1, 8, gate_activation="relu")
    x = torch.ones(3, 4)
    d = IrrepsDropout(0.5).eval()
    assert d(x) is x


def _graph(dtype):
    return batch_graph(synthetic_molecules(3, rank=1), ARCH["r_max"], torch.device("cuda"), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tol", [(torch.float64, 1e-10), (torch.float32, 2e-4)])
@pytest.mark.parametrize("agnostic", [False, True])
def test_blocks_give_the_stock_model(cuda_device, dtype, tol, agnostic):
    """Energies, forces and every parameter gradient of the energy + force loss (which runs the
    operators' second derivatives). float64: rounding; float32: 1e-4-level noise of forces that
    two evaluation orders of this model show."""
    stock = _model(element_agnostic_interaction=agnostic, element_agnostic_product=agnostic).to("cuda", dtype)
    blocks = use_training_blocks(copy.deepcopy(stock))
    graph = _graph(dtype)
    gen = torch.Generator().manual_seed(3)
    e = torch.randn(3, generator=gen, dtype=torch.float64).to("cuda", dtype)
    f = torch.randn(graph["positions"].shape, generator=gen, dtype=torch.float64).to("cuda", dtype)
    grads = []
    for model in (stock, blocks):
        model.zero_grad(set_to_none=True)
        loss, out = energy_force_loss(model, graph, e, f)
        loss.backward()
        grads.append((out, {n: p.grad for n, p in model.named_parameters()}))
    (o0, g0), (o1, g1) = grads
    for k in ("energy", "forces"):
        scale = o0[k].abs().max().item()
        assert (o0[k] - o1[k]).abs().max().item() <= tol * scale
    for n, g in g0.items():
        assert (g is None) == (g1[n] is None), n
        if g is not None:
            assert (g - g1[n]).abs().max().item() <= 10 * tol * max(g.abs().max().item(), 1e-6), n
    # evaluation without a second derivative (fused first-order operators elsewhere in the model)
    a = stock.predict(graph, compute_forces=True)
    b = blocks.predict(graph, compute_forces=True)
    assert (a["forces"] - b["forces"]).abs().max().item() <= tol * a["forces"].abs().max().item()


@pytest.mark.gpu
def test_blocks_train_with_first_derivatives_only(cuda_device):
    """Energy-only training: the fused backward with weight gradients against the stock layers."""
    stock = _model().to("cuda", torch.float64)
    blocks = use_training_blocks(copy.deepcopy(stock))
    graph = _graph(torch.float64)
    got = []
    for model in (stock, blocks):
        model(graph).square().sum().backward()
        got.append({n: p.grad for n, p in model.named_parameters()})
    for n, g in got[0].items():
        if g is not None:
            assert (g - got[1][n]).abs().max().item() <= 1e-9 * max(g.abs().max().item(), 1e-6), n


@pytest.mark.gpu
def test_dropout_in_the_model(cuda_device):
    model = use_training_blocks(_model().to("cuda", torch.float64), dropout=0.3, seed=11)
    graph = _graph(torch.float64)
    plain = model.eval()(graph)
    assert torch.equal(plain, model(graph))
    model.train()
    rewind = lambda: [m.rng[1].zero_() for m in model.modules() if isinstance(m, IrrepsDropout)]
    a = model(graph)
    assert all(int(m.rng[1]) == 1 for m in model.modules() if isinstance(m, IrrepsDropout))
    b = model(graph)
    assert not torch.allclose(a, plain) and not torch.allclose(a, b)
    rewind()
    assert torch.equal(model(graph), a)  # the stream decides, nothing else
    # whole irreps are dropped: energies do not change when the molecules turn
    gen = torch.Generator().manual_seed(1)
    turn = torch.linalg.qr(torch.randn(3, 3, generator=gen, dtype=torch.float64))[0].cuda()
    rewind()
    turned = model(dict(graph, positions=graph["positions"] @ turn))
    assert (turned - a).abs().max().item() <= 1e-9 * a.abs().max().item()
    # and the forces are the energy's gradient under the same masks
    rewind()
    forces = model.predict(graph, compute_forces=True)["forces"]
    step, k = 1e-5, (7, 1)
    energies = []
    for s in (step, -step):
        pos = graph["positions"].clone()
        pos[k] += s
        rewind()
        energies.append(model(dict(graph, positions=pos)).sum().item())
    slope = (energies[0] - energies[1]) / (2 * step)
    # central difference: error about step^2 times the third derivative, far below this bound
    assert abs(slope + forces[k].item()) <= 1e-5 * max(1.0, forces.abs().max().item())


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "sigmoid"])
def test_gated_layer_in_its_types(cuda_device, act):
    """bfloat16 rows against the stock layer in float32 (the output map has no bfloat16
    gradient, so forward only)."""
    torch.manual_seed(2)
    stock = EquivariantGatedLayer(2, 32, 48, gate_activation=act).cuda()
    with torch.no_grad():
        for w in stock.output_linear.weight:
            w.normal_()
    block = GatedFeedForward.from_layer(stock)
    x = torch.randn(50, 9 * 32, device="cuda")
    with torch.no_grad():
        want = stock(x)
        assert ((block(x) - want).norm() / want.norm()).item() <= 2e-6
        low = block(x.bfloat16()).float()
        # roundings to 8 bits of x, the weights, the hidden rows, the map and the sum
        assert ((low - want).norm() / want.norm()).item() <= 6 * 2.0 ** -8
