"""Training-block operators without a GPU: the host-emulated kernels through the C ABI against
the float64 definitions, and the refusals of the C ABI and of the Python entry points."""

import ctypes

import pytest
import torch

import block_refs as R
from abi_calls import p
from flashcart_b200 import _native as N
from flashcart_b200 import ops

CODES = {torch.float32: N.FC_F32, torch.float64: N.FC_F64, torch.bfloat16: N.FC_BF16}
# largest relative difference of one value: the storage rounding (half a unit in the last
# place) plus a few roundings of the arithmetic
ONE = {torch.float32: 2.0 ** -22, torch.float64: 2.0 ** -51, torch.bfloat16: 2.0 ** -8 + 2.0 ** -22}
UNIT = {torch.float32: 2.0 ** -24, torch.float64: 2.0 ** -53, torch.bfloat16: 2.0 ** -24}
STORE = {torch.float32: 2.0 ** -24, torch.float64: 2.0 ** -53, torch.bfloat16: 2.0 ** -8}


def _ptrs(ts):
    return (ctypes.c_void_p * len(ts))(*[None if t is None else t.data_ptr() for t in ts])


@pytest.mark.parametrize("dtype", list(CODES))
@pytest.mark.parametrize("rows,types,dim", [(1, 1, 1), (7, 3, 5), (40, 6, 16), (33, 300, 9), (0, 4, 3)])
def test_embedding_emulated(emu_lib, dtype, rows, types, dim):
    g = torch.Generator().manual_seed(rows + dim)
    table = torch.randn(types, dim, generator=g, dtype=torch.float64).to(dtype)
    idx = torch.randint(0, types, (rows,), generator=g)
    out, status = torch.empty(rows, dim, dtype=dtype), torch.zeros(1, dtype=torch.int32)
    rc = emu_lib.fc_embedding_fwd(p(table), types, dim, CODES[dtype], p(idx), rows, 1.5, 1.0, p(out), p(status), None)
    assert rc == 0 and status.item() == 0
    ref = R.embedding(table, idx, 1.5, 1.0)
    mag = 1.0 + (ref - 1.0).abs()
    assert ((out.double() - ref).abs() <= ONE[dtype] * mag).all()
    grad = torch.randn(rows, dim, generator=g, dtype=torch.float64).to(dtype)
    gt = torch.full((types, dim), float("nan"), dtype=dtype)
    ws = torch.empty(emu_lib.fc_embedding_bwd_workspace_bytes(rows, types, dim, CODES[dtype]) + 16, dtype=torch.uint8)
    rc = emu_lib.fc_embedding_bwd(p(grad), p(idx), rows, types, dim, CODES[dtype], 1.5, p(ws), p(gt), p(status), None)
    assert rc == 0
    want, mag, count = R.embedding_grad(grad, idx, types, 1.5)
    bound = (count[:, None] + 2) * UNIT[dtype] * mag + STORE[dtype] * want.abs() * 1.01
    assert ((gt.double() - want).abs() <= bound).all()


def test_embedding_bad_index_is_flagged(emu_lib):
    table, idx = torch.ones(3, 4), torch.tensor([0, 3, -1, 2])
    out, status = torch.empty(4, 4), torch.zeros(1, dtype=torch.int32)
    emu_lib.fc_embedding_fwd(p(table), 3, 4, N.FC_F32, p(idx), 4, 1.0, 0.5, p(out), p(status), None)
    assert status.item() == N.FC_DEV_BAD_INDEX
    assert out[:, 0].tolist() == [1.5, 0.0, 0.0, 1.5]


@pytest.mark.parametrize("dtype", list(CODES))
@pytest.mark.parametrize("n,l_max,c,prob", [(5, 0, 6, 0.3), (3, 2, 4, 0.5), (4, 3, 7, 0.1), (2, 1, 1, 0.0),
                                            (2, 1, 5, 1.0), (0, 2, 4, 0.5)])
def test_dropout_emulated(emu_lib, dtype, n, l_max, c, prob):
    gen = torch.Generator().manual_seed(c)
    x = torch.randn(n, (l_max + 1) ** 2 * c, generator=gen, dtype=torch.float64).to(dtype)
    rng = torch.tensor([-5, 7], dtype=torch.int64)
    y = torch.empty_like(x)
    rc = emu_lib.fc_irreps_dropout(l_max, c, CODES[dtype], p(x), p(rng), prob, n, p(y), None)
    assert rc == 0
    keep = R.dropout_keep(n, l_max, c, -5 & (2 ** 64 - 1), 7, prob)
    want = torch.where(keep, x.double() / (1 - prob) if prob < 1 else x.double(), torch.zeros(()).double())
    assert ((y.double() - want).abs() <= ONE[dtype] * want.abs()).all()


@pytest.mark.parametrize("dtype", list(CODES))
@pytest.mark.parametrize("n,l_max,c,h,act,bias", [(1, 0, 1, 1, "silu", False), (5, 0, 6, 9, "sigmoid", True),
                                                  (7, 1, 5, 4, "silu", True), (4, 2, 3, 8, "sigmoid", False),
                                                  (6, 3, 4, 4, "silu", True), (0, 1, 4, 4, "silu", True)])
def test_gated_emulated(emu_lib, dtype, n, l_max, c, h, act, bias):
    x, wv, wg, b, sc, g = R.gated_inputs(n, l_max, c, h, bias, dtype, "cpu", seed=n)
    d = N.GatedFfDesc(l_max, c, h, {"silu": 0, "sigmoid": 1}[act], CODES[dtype])
    ws = lambda back: torch.empty(emu_lib.fc_gated_ff_workspace_bytes(ctypes.byref(d), n, back) + 16,
                                  dtype=torch.uint8)
    y, w0, w1 = torch.empty_like(g), ws(0), ws(1)
    rc = emu_lib.fc_gated_ff_fwd(ctypes.byref(d), p(x), _ptrs(wv), p(wg), p(b), p(sc), n, p(w0), p(y), None, None)
    assert rc == 0, emu_lib.fc_last_error()
    outs = [torch.full_like(t, float("nan")) for t in (x, wg, *([b] if bias else []), *wv)]
    gx, gwg = outs[0], outs[1]
    gb = outs[2] if bias else None
    gwv = outs[3 if bias else 2:]
    rc = emu_lib.fc_gated_ff_bwd(ctypes.byref(d), p(g), p(x), _ptrs(wv), p(wg), p(b), p(sc), n, p(w1), p(gx),
                                 _ptrs(gwv), p(gwg), p(gb), None, None)
    assert rc == 0
    want_y, want = R.gated_grads(x, wv, wg, b, sc, l_max, act, g)
    # sums of at most 3 (c + h) n terms in the arithmetic type, then the storage rounding
    rel = STORE[dtype] + UNIT[dtype] * (16 + 3 * (c + h + n * (2 * l_max + 1)))
    for got, ref in [(y, want_y), (gx, want[0]), (gwg, want[1]), *([(gb, want[2])] if bias else []),
                     *zip(gwv, want[3:])]:
        scale = max(ref.abs().max().item(), 1e-30) if ref.numel() else 0.0
        assert got.numel() == 0 or (got.double() - ref).abs().max().item() <= 4 * rel * scale


def test_abi_refusals(emu_lib):
    t = torch.zeros(4, 4)
    idx = torch.zeros(4, dtype=torch.int64)
    ws = torch.zeros(4096, dtype=torch.uint8)
    f = emu_lib
    assert f.fc_embedding_fwd(p(t), 4, 4, 9, p(idx), 4, 1.0, 0.0, p(t), None, None) == N.FC_ERR_INVALID
    assert f.fc_embedding_fwd(p(t), 4, -1, 0, p(idx), 4, 1.0, 0.0, p(t), None, None) == N.FC_ERR_INVALID
    assert f.fc_embedding_fwd(p(t), 4, 4, 0, None, 4, 1.0, 0.0, p(t), None, None) == N.FC_ERR_INVALID
    assert f.fc_embedding_fwd(p(t), 4, 4, 0, None, 0, 1.0, 0.0, None, None, None) == N.FC_OK
    assert f.fc_embedding_bwd_workspace_bytes(2 ** 31, 4, 4, 0) == N.FC_ERR_CAPACITY
    assert f.fc_embedding_bwd(p(t), p(idx), 4, 4, 4, 0, 1.0, None, p(t), None, None) == N.FC_ERR_INVALID
    assert f.fc_embedding_bwd(p(t), p(idx), 4, 4, 4, 0, 1.0, ctypes.c_void_p(ws.data_ptr() + 8), p(t), None,
                              None) == N.FC_ERR_INVALID
    rng = torch.zeros(2, dtype=torch.int64)
    assert f.fc_irreps_dropout(4, 1, 0, p(t), p(rng), 0.1, 1, p(t), None) == N.FC_ERR_UNSUPPORTED
    for prob in (-0.1, 1.1, float("nan")):
        assert f.fc_irreps_dropout(0, 4, 0, p(t), p(rng), prob, 4, p(t), None) == N.FC_ERR_INVALID
    assert f.fc_irreps_dropout(0, 4, 0, p(t), None, 0.1, 4, p(t), None) == N.FC_ERR_INVALID
    good = N.GatedFfDesc(0, 4, 4, 0, 0)
    call = lambda d, n=4, w=ws, wv=(t,): f.fc_gated_ff_fwd(ctypes.byref(d) if d else None, p(t), _ptrs(wv), p(t), None,
                                                           p(t), n, p(w) if w is not None else None, p(t), None, None)
    assert call(None) == N.FC_ERR_INVALID
    assert call(N.GatedFfDesc(4, 4, 4, 0, 0)) == N.FC_ERR_UNSUPPORTED
    assert call(N.GatedFfDesc(0, 0, 4, 0, 0)) == N.FC_ERR_INVALID
    assert call(N.GatedFfDesc(0, 4, 4, 7, 0)) == N.FC_ERR_INVALID
    assert call(N.GatedFfDesc(0, 4, 4, 0, 5)) == N.FC_ERR_INVALID
    assert call(good, n=-1) == N.FC_ERR_INVALID
    assert call(good, n=2 ** 40) == N.FC_ERR_CAPACITY
    assert call(good, w=None) == N.FC_ERR_INVALID
    assert call(good, wv=(None,)) == N.FC_ERR_INVALID
    assert b"fc_gated_ff_fwd" in f.fc_last_error()


def test_entry_points_refuse_cpu_tensors():
    x, w = torch.zeros(2, 4), torch.zeros(4, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.embedding(w, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.irreps_dropout(x, torch.zeros(2, dtype=torch.int64), 0.5)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.gated_feed_forward(x, [w], w, None, torch.zeros(3), 0, "silu")
