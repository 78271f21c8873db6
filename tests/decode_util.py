"""Plain definitions in 64 bits, on the CPU, of the operators between and beside a decode step's projections, and the
tensors their tests use."""
import math

import torch

F32_EPS = 2.0 ** -24
BF16_HALF = 2.0 ** -8        # largest relative error of one rounding to bf16


def codes(cache):
    """A cache's values in 64 bits (e4m3 codes: the values they stand for, before the head's factor)."""
    c = cache.detach().cpu()
    return c.view(torch.uint8).view(torch.float8_e4m3fn).float().double() if c.element_size() == 1 else c.double()


def bits(t):
    """A tensor's bit patterns in its own memory order, as integers."""
    t = t.detach().cpu()
    return t.view(torch.uint8) if t.element_size() == 1 else t.view(torch.int16)


def make_cache(pages, kv_heads, page_size, dim, fp8, layout, gen, fill=None):
    """[pages, kv_heads, page_size, dim] on the CPU; "hpd" contiguous, "phd" [pages, page_size, heads, dim] in memory, "gap"
    rows 48 values apart more than they need (16-byte multiples)."""
    if layout == "gap":
        c = torch.empty(pages, kv_heads, page_size, dim + 48)[..., :dim]
    elif layout == "phd":
        c = torch.empty(pages, page_size, kv_heads, dim).transpose(1, 2)
    else:
        c = torch.empty(pages, kv_heads, page_size, dim)
    vals = torch.randn(c.shape, generator=gen) if fill is None else torch.full(c.shape, fill)
    dtype = torch.float8_e4m3fn if fp8 else torch.bfloat16
    out = torch.empty_strided(c.shape, c.stride(), dtype=torch.uint8 if fp8 else dtype)
    out.copy_((vals * (16.0 if fp8 else 1.0)).to(dtype).view(out.dtype))
    return out.view(dtype)


def on(t, device):
    """The tensor on a device with its strides kept (gaps too)."""
    if t is None:
        return None
    out = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=device)
    raw = torch.uint8 if t.element_size() == 1 else t.dtype
    out.view(raw).copy_(t.view(raw))
    return out


def rope64(qkv, positions, cos_sin, heads, kv_heads, dim, q_norm=None, k_norm=None, eps=1e-6, pairs=False):
    """(q, k, v) [M, heads, dim] in 64 bits."""
    M, rot = qkv.shape[0], cos_sin.shape[1]
    x = qkv.double().view(M, heads + 2 * kv_heads, dim)
    q, k, v = x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
    cs = cos_sin.double()[positions]
    c, s = cs[:, None, :rot // 2], cs[:, None, rot // 2:]

    def turn(h, w):
        if w is not None:
            h = h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
        h = h.clone()
        i = torch.arange(rot // 2)
        lo, hi = (2 * i, 2 * i + 1) if pairs else (i, i + rot // 2)
        a, b = h[..., lo], h[..., hi]
        h[..., lo], h[..., hi] = a * c - b * s, b * c + a * s
        return h

    return turn(q, q_norm), turn(k, k_norm), v


def attention64(q, k_cache, v_cache, table, lens, scale=None, window=0, k_scale=None, v_scale=None):
    """In 64 bits on the CPU, one token at a time over exactly the positions it sees: out [B, T, heads, dim], lse [B, T,
    heads], and for error bounds sum of weight * |v| (like out) and the largest sum of |q_i k_i| * |scale| (like lse).
    k_cache and v_cache [pages, kv_heads, page_size, dim]."""
    B, T, Hq, D = q.shape
    pages, H, P, _ = k_cache.shape
    scale = D ** -0.5 if scale is None else scale
    out, size = torch.zeros(2, B, T, Hq, D, dtype=torch.float64)
    lse, terms = torch.full((B, T, Hq), -math.inf, dtype=torch.float64), torch.zeros(B, T, Hq, dtype=torch.float64)
    G = Hq // H
    for b in range(B):
        n = max(0, min(int(lens[b]), table.shape[1] * P))
        at = torch.arange(n)
        page = table[b].long()[at // P]
        for t in range(T):
            end = n - (T - 1 - t)
            see = (at < end) & (page >= 0) & (page < pages)
            if window:
                see &= at >= end - window
            if not see.any():
                continue
            pg, off = page[see], at[see] % P
            k = codes(k_cache[pg, :, off]) * (1.0 if k_scale is None else k_scale.double()[None, :, None])
            v = codes(v_cache[pg, :, off]) * (1.0 if v_scale is None else v_scale.double()[None, :, None])
            k, v, x = k.transpose(0, 1), v.transpose(0, 1), q[b, t].double().view(H, G, D)
            a = torch.matmul(x, k.transpose(1, 2)) * scale
            w = torch.softmax(a, -1)
            lse[b, t] = torch.logsumexp(a, -1).view(Hq)
            out[b, t] = torch.matmul(w, v).view(Hq, D)
            size[b, t] = torch.matmul(w, v.abs()).view(Hq, D)
            terms[b, t] = (torch.matmul(x.abs(), k.abs().transpose(1, 2)).amax(-1) * abs(scale)).view(Hq)
    return out, lse, size, terms


def lora64(y, x, A, B, ids, scaling, splits):
    """y + the rows' adapters in 64 bits, on the CPU. ids outside [0, adapters) add nothing."""
    out, R = y.double().clone(), B.shape[2]
    for m, a in enumerate(ids.tolist()):
        if not 0 <= a < A.shape[0]:
            continue
        h = A[a].double() @ x[m].double()
        s = 1.0 if scaling is None else float(scaling[a])
        at = 0
        for j, n in enumerate(splits):
            out[m, at:at + n] += s * (B[a, at:at + n].double() @ h[j * R:(j + 1) * R])
            at += n
    return out
