"""Definitions of the training-block operators in float64 (numpy / torch on the CPU), used by
the CPU tests (host-emulated kernels) and the GPU tests."""

import numpy as np
import torch


def embedding(table, index, scale, offset):
    return offset + scale * table.double().cpu()[index.cpu().long()]


def embedding_grad(grad, index, n_types, scale):
    """(sum, sum of magnitudes, rows per type), the last two for error bounds."""
    g, idx = grad.double().cpu().reshape(-1, grad.shape[-1]), index.cpu().long().reshape(-1)
    out = torch.zeros(n_types, g.shape[1], dtype=torch.float64)
    mag = torch.zeros_like(out)
    out.index_add_(0, idx, g * scale)
    mag.index_add_(0, idx, (g * scale).abs())
    return out, mag, torch.bincount(idx, minlength=n_types)


def philox(block, offset, seed):
    """Four 32-bit words per 64-bit block index (Philox 4x32, ten rounds), as Python integers."""
    c = [block & 0xFFFFFFFF, block >> 32, offset & 0xFFFFFFFF, (offset >> 32) & 0xFFFFFFFF]
    k = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for _ in range(10):
        p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & 0xFFFFFFFF, (p0 >> 32) ^ c[3] ^ k[1], p0 & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def dropout_keep(n, l_max, channels, seed, offset, p):
    """Boolean (n, (l_max+1)^2 * channels): what is kept."""
    ranks, quads = l_max + 1, (channels + 3) // 4
    words = np.array([philox(b, offset, seed) for b in range(n * ranks * quads)], dtype=np.uint64).reshape(-1, 4)
    keep = (words >= np.uint64(int(p * 2 ** 32))).reshape(n, ranks, quads * 4)[:, :, :channels]
    keep = np.repeat(keep, [2 * l + 1 for l in range(ranks)], axis=1)
    return torch.from_numpy(np.ascontiguousarray(keep)).reshape(n, ranks * ranks * channels)


def gated(x, wv, wg, bias, scales, l_max, act):
    """The gated feed-forward block, rank by rank; differentiable float64 on x's device."""
    n, ranks, (h, c) = x.shape[0], l_max + 1, wv[0].shape
    z = scales[ranks] * (x[:, :c] @ wg.T)
    if bias is not None:
        z = z + bias
    s = torch.sigmoid(z)
    a = scales[ranks + 1] * (s if act == "sigmoid" else z * s)
    parts = []
    for l in range(ranks):
        xl = x[:, l * l * c:(l + 1) ** 2 * c].reshape(n, 2 * l + 1, c)
        v = scales[l] * (xl @ wv[l].T)
        parts.append((v * a[:, None, l * h:(l + 1) * h]).reshape(n, (2 * l + 1) * h))
    return torch.cat(parts, 1)


def gated_grads(x, wv, wg, bias, scales, l_max, act, g):
    """(y, [gx, gwg, gbias or None, *gwv]) of :func:`gated` in float64."""
    leaf = lambda t: None if t is None else t.detach().double().requires_grad_(True)
    xs, ws, gw, bs = leaf(x), [leaf(w) for w in wv], leaf(wg), leaf(bias)
    y = gated(xs, ws, gw, bs, scales.double(), l_max, act)
    ins = [xs, gw, *([bs] if bs is not None else []), *ws]
    got = list(torch.autograd.grad(y, ins, g.double()))
    if bs is None:
        got.insert(2, None)
    return y.detach(), got


def gated_inputs(n, l_max, c, h, bias, dtype, device, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64).to(device=device, dtype=dtype)
    ranks = l_max + 1
    acc = torch.float64 if dtype == torch.float64 else torch.float32
    scales = torch.tensor([c ** -0.5 * (1 + 0.1 * l) for l in range(ranks)] + [0.9 * c ** -0.5, 1.7], dtype=acc,
                          device=device)
    return (r(n, ranks * ranks * c), [r(h, c) for _ in range(ranks)], r(ranks * h, c),
            r(ranks * h) * 0.5 if bias else None, scales, r(n, ranks * ranks * h))
