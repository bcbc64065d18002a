"""Training blocks as modules, without a GPU: what they keep of the layers they stand for, and
what they refuse."""

import copy
import ctypes

import pytest
import torch
import torch.nn as nn

from abi_calls import p
from flashcart_b200 import _native as N
from flashcart_b200 import build_ext
from flashcart_b200.model.flashcart import FlashCartPotential
from flashcart_b200.nn.blocks import IrrepsDropout, ScaledEmbedding, use_training_blocks

ARCH = dict(elements=["H", "C"], r_max=4.0, n_hidden_feats=8, l_max_hidden_feats=1, l_max_edge_attrs=1, n_radial=4,
            n_interactions=3, correlation=2, layer_norm=True, nonlinearity=True, avg_neighbors=12.0,
            element_agnostic_interaction=False, element_agnostic_product=False, n_element_interaction_features=4)


def test_dropout_streams_of_layers_and_seeds():
    """No layer of one seed shares its stream with another layer, of this seed or of another."""
    stock = FlashCartPotential(**ARCH)
    keys = []
    for seed in (0, 1, 2, 3, -1, 10 ** 6, 2 ** 63 - 1):
        model = use_training_blocks(copy.deepcopy(stock), dropout=0.1, seed=seed)
        layers = [m for m in model.modules() if isinstance(m, IrrepsDropout)]
        assert len(layers) > 1
        keys += [int(m.rng[0]) for m in layers]
    assert len(set(keys)) == len(keys)


@pytest.mark.parametrize("options", [dict(padding_idx=0), dict(max_norm=1.0), dict(scale_grad_by_freq=True),
                                     dict(sparse=True)])
def test_embeddings_with_options_are_not_replaced(options):
    emb = nn.Embedding(2, 8, **options)
    with pytest.raises(ValueError, match="plain embeddings"):
        ScaledEmbedding.from_embedding(emb)
    model = FlashCartPotential(**ARCH)
    model.embedding, model.interactions[0].emb_j = emb, nn.Embedding(2, 4, **options)
    blocks = use_training_blocks(model)
    assert blocks.embedding is emb and type(blocks.interactions[0].emb_j) is nn.Embedding
    assert type(blocks.interactions[0].emb_i) is ScaledEmbedding
    plain = nn.Embedding(2, 8)
    assert ScaledEmbedding.from_embedding(plain).weight is plain.weight


def test_gated_rows_in_place_have_to_be_aligned(emu_lib):
    t, keep = torch.zeros(64), torch.zeros(64)
    off = ctypes.c_void_p(keep.data_ptr() + 4)
    ws = torch.zeros(2 ** 16, dtype=torch.uint8)
    one = (ctypes.c_void_p * 1)(t.data_ptr())

    def call(c, h, x=p(t), y=p(t), gy=p(t), gx=p(t), n=1):
        d = ctypes.byref(N.GatedFfDesc(0, c, h, N.FC_GATE_SILU, N.FC_F32))
        return (emu_lib.fc_gated_ff_fwd(d, x, one, p(t), None, p(t), n, p(ws), y, None, None),
                emu_lib.fc_gated_ff_bwd(d, gy, x, one, p(t), None, p(t), n, p(ws), gx, None, None, None, None, None))

    ok, no = N.FC_OK, N.FC_ERR_INVALID
    assert call(4, 4) == (ok, ok)
    assert call(4, 4, x=off) == (no, no) and b"x must be 16-byte aligned" in emu_lib.fc_last_error()
    assert call(4, 4, y=off) == (no, ok) and call(4, 4, gy=off) == (ok, no) and call(4, 4, gx=off) == (ok, no)
    assert call(4, 4, x=off, y=off, gy=off, gx=off, n=0) == (ok, ok)
    assert call(3, 3, x=off, y=off, gy=off, gx=off) == (ok, ok)


def test_build_checks_shared_registers():
    line = ("ptxas info    : Compiling entry function '{}' for 'sm_100a'\n"
            "ptxas info    : Function properties for {}\n    0 bytes stack frame\n"
            "ptxas info    : Used {} registers, used 2 barriers\n")
    tc, other = "_ZN2fc3gtc15gated_tc_kernelILi0EfEEvNS0_4MapsENS0_4ArgsE", "_ZN2fc3gtc11prep_kernelIfEEvNS0_8PrepArgsE"
    assert build_ext.check_registers(line.format(tc, tc, 96) + line.format(other, other, 40)) == 1
    assert build_ext.check_registers("") == 0
    for used in (88, 104):
        with pytest.raises(RuntimeError, match=f"uses {used} registers"):
            build_ext.check_registers(line.format(other, other, 96) + line.format(tc, tc, used))
    # every kernel of the table is one of the sources'
    text = "".join(open(f).read() for f in build_ext.sources() if "gated_ff" in f)
    assert all(f" {name}(" in text for name in build_ext.SHARED_REGISTERS)
