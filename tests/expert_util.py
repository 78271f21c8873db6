"""Plain definitions in 64 bits, on the CPU, of the operators of a layer's feed-forward half with experts, and the tensors their
tests use."""
import numpy as np
import torch

from decode_util import BF16_HALF, F32_EPS

FORMATS = ("bf16", "fp8", "int4", "int4zp")
STEP = {"bf16": 8, "fp8": 16, "int4": 128, "int4zp": 128}      # what K is a multiple of


def make_experts(fmt, E, N, K, seed=0, bias=False):
    """(operands of ops.experts_*, bias or None) on the CPU."""
    g = torch.Generator().manual_seed(seed)
    b = torch.randn(E, N, generator=g).bfloat16() if bias else None
    if fmt == "bf16":
        return (torch.randn(E, N, K, generator=g).mul_(K ** -0.5).bfloat16(),), b
    if fmt == "fp8":
        W = torch.randn(E, N, K, generator=g).mul_(60.0).clamp_(-448, 448).to(torch.float8_e4m3fn)
        return (W, torch.rand(E, N, generator=g).add_(0.5).mul_(0.02 * K ** -0.5)), b
    W = torch.randint(0, 256, (E, N, K // 2), dtype=torch.uint8, generator=g)
    s = torch.rand(E, N, K // 128, generator=g).add_(0.1).mul_(0.3 * K ** -0.5)
    if fmt == "int4":
        return (W, s.half()), b
    z = torch.randint(0, 256, (E, N, (K // 128 + 1) // 2), dtype=torch.uint8, generator=g)
    return (W, s.bfloat16(), z), b


def weights64(fmt, W, e):
    """(what expert e's matrix stands for, and |q| + |zero| times the scale: the terms that its sums have), 64 bits [N, K]."""
    if fmt == "bf16":
        w = W[0][e].double()
        return w, w.abs()
    if fmt == "fp8":
        w = W[0][e].float().double() * W[1][e].double()[:, None]
        return w, w.abs()
    q = torch.stack([W[0][e] & 15, W[0][e] >> 4], -1).flatten(1).double()
    G = q.shape[1] // 128
    z = torch.full((q.shape[0], G), 8.0, dtype=torch.float64)
    if fmt == "int4zp":
        z = torch.stack([W[2][e] & 15, W[2][e] >> 4], -1).flatten(1)[:, :G].double()
    z = z.repeat_interleave(128, 1)
    s = W[1][e].double().repeat_interleave(128, 1)
    return (q - z) * s, (q + z) * s.abs()


def order64(ids, E):
    """(order, offsets) of ids [M, k]: a stable sort."""
    flat = ids.flatten().long()
    key = torch.where((flat >= 0) & (flat < E), flat, torch.full_like(flat, E))
    at = np.argsort(key.numpy(), kind="stable")
    offsets = np.searchsorted(np.sort(key.numpy()), np.arange(E + 1))
    return torch.from_numpy(at).int(), torch.from_numpy(offsets).int()


def experts64(fmt, W, x, order, offsets, bias=None, gated=False):
    """(out, bound) [pairs, N or N / 2], 64 bits.

    Bound. A sum of K products in fp32 is off by (K + 8) 2^-24 of its terms' absolute sum T (the products of bf16 values are
    exact; INT4 sums hold q x and zero x apart, and one factor more), bias and scale by two roundings more. silu(g) has a slope
    below 1.1; its exponential is off by (|g| + 2) 2^-23. Then one rounding to bf16."""
    R, N, K = order.numel(), W[0].shape[1], x.shape[1]
    k = R // x.shape[0]
    half = N // 2
    out = torch.zeros(R, half if gated else N, dtype=torch.float64)
    bound = torch.zeros_like(out)
    for e in range(W[0].shape[0]):
        p = order[int(offsets[e]):int(offsets[e + 1])].long()
        if len(p) == 0:
            continue
        w, a = weights64(fmt, W, e)
        rows = x[p // k].double()
        y, t = rows @ w.t(), (rows.abs() @ a.t()) * ((K + 8) * F32_EPS)
        if bias is not None:
            y = y + bias[e].double()
        t = t + 3 * F32_EPS * y.abs() + (F32_EPS * bias[e].double().abs() if bias is not None else 0.0)
        if gated:
            g, v, tg, tv = y[:, :half], y[:, half:], t[:, :half], t[:, half:]
            s = g / (1.0 + torch.exp(-g))
            t = 1.1 * tg * (v.abs() + tv) + s.abs() * tv + ((g.abs() + 2) * 2.0 ** -23 + 4 * F32_EPS) * (s * v).abs()
            y = s * v
        out[p] = y
        bound[p] = t * 1.01 + BF16_HALF * (y.abs() + t) + 2.0 ** -133
    return out, bound


def norm64(x, residual, norm, post_norm=None, gate=None, weights=None, scale=1.0, eps=1e-6, plus_one=False):
    """(out, r, bound of out, bound of r before the roundings to the outputs' types), 64 bits.

    Bound. The sum over P pairs is off by (P + 1) 2^-24 of its terms' absolute sum S. A mean of D squares is summed by at most 32
    values a thread, 6 steps of a wave and 16 waves: with root, division and factors its norm's factor is off by 64 2^-24, and
    by the relative error, in the 2-norm, of what is normed. Every further product or sum adds 2^-24 of its terms."""
    one = 1.0 if plus_one else 0.0
    y = x.double()
    size = y.abs()
    P = 0
    if weights is not None:
        w = weights.double()[:, :, None]
        y = torch.where(w != 0, w * y, torch.zeros((), dtype=torch.float64))
        P, size, y = x.shape[1], y.abs().sum(1), y.sum(1)
    err = (P + 1) * F32_EPS * size if P else torch.zeros_like(y)

    def rms(v, e, w):
        length = v.square().sum(-1, keepdim=True).sqrt()
        by = (v.square().mean(-1, keepdim=True) + eps).rsqrt()
        rel = 64 * F32_EPS + e.square().sum(-1, keepdim=True).sqrt() / length.clamp(min=1e-300)
        f = one + w.double()
        return v * by * f, (v.abs() * rel + e) * by * f.abs() + 3 * F32_EPS * v.abs() * by * f.abs()

    if post_norm is not None:
        y, err = rms(y, err, post_norm)
    f = torch.as_tensor(float(np.float32(scale)), dtype=torch.float64)
    if gate is not None:
        f = f * gate.double()
    y, err = f * y, f.abs() * err + 2 * F32_EPS * (f * y).abs()
    if residual is not None:
        y = residual.double() + y
    err = err + F32_EPS * y.abs()
    h, err_h = rms(y, err, norm)
    return h, y, err_h, err


def route64(logits, k, bias=None, scoring="softmax", renormalize=True, scale=1.0):
    """(ids, weights) in 64 bits, one token at a time."""
    M, E = logits.shape
    ids, weights = torch.full((M, k), -1, dtype=torch.int32), torch.zeros(M, k, dtype=torch.float64)
    for m in range(M):
        v = logits[m].double().numpy()
        b = np.zeros(E) if bias is None else bias.double().numpy()
        open_ = (v > -np.inf) & (b > -np.inf)
        with np.errstate(all="ignore"):
            score = 1.0 / (1.0 + np.exp(-v))
        key = score + b if scoring == "sigmoid" else v
        chosen = sorted(np.nonzero(open_)[0], key=lambda e: (-key[e], e))[:k]
        if not chosen:
            continue
        if scoring == "softmax":
            with np.errstate(all="ignore"):
                score = np.where(open_, np.exp(v - v[chosen[0]]), 0.0)
                score = score / score.sum()
        w = score[chosen]
        if renormalize:
            w = w / w.sum() if w.sum() > 0 else w * 0.0
        ids[m, :len(chosen)] = torch.tensor([int(e) for e in chosen], dtype=torch.int32)
        weights[m, :len(chosen)] = torch.from_numpy(w * float(np.float32(scale)))
    return ids, weights
