"""The operators of a decoder layer's feed-forward half with experts, as measured work: residual and norms, routing, the experts'
products.

A case is a dict of plain values:
  op "norm"     ops.add_norm: `M` tokens of `D` values. x is the last block's output, or with `pairs` > 0 the outputs of a token's
                `pairs` experts, summed by their weights. `post` adds a norm of that, `gate` a factor per channel ("channel") or per
                token and channel ("row"). `res` is the residual's type. `plus_one`: norm weights are kept less 1.
  op "route"    ops.route_experts: `k` of `E` experts for each of `M` tokens, of `logits` type. `scoring` softmax or sigmoid (the
                latter with a bias on the choice). `skip` tokens are padding of a captured batch: all their experts are masked.
                `masked` experts are masked for all tokens.
  op "experts"  ops.experts_*: the products of `M` tokens with the `k` of `E` experts [N, K] that each chose, weights in `fmt`.
                `gated` joins the rows' halves to silu(gate) * up. `own_rows`: every pair of token and expert has a row of x of
                its own (the down projection); else a token's pairs share its row. `skip` tokens chose none.
                `skew` says how unevenly the experts are chosen (the standard deviation of the logarithm of their odds).

How many tokens each expert has follows from the case alone; the seed decides which expert that is, and every value.
"""
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False     # False: plain torch operations in 32 bits; True: the framework's operators

_PKG = str(Path(__file__).resolve().parent.parent / "paia-project_amd")


def _ops():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from paia_gemv import ops
    return ops


def _norm(name, M, D, **more):
    return {"name": name, "op": "norm", "M": M, "D": D, "pairs": 0, "post": False, "gate": "", "res": "bf16",
            "scale": 1.0, "plus_one": False, **more}


def _route(name, M, E, k, **more):
    return {"name": name, "op": "route", "M": M, "E": E, "k": k, "logits": "bf16", "scoring": "softmax", "renormalize": True,
            "scale": 1.0, "skip": 0, "masked": 0, **more}


def _experts(name, M, E, k, N, K, fmt, **more):
    return {"name": name, "op": "experts", "M": M, "E": E, "k": k, "N": N, "K": K, "fmt": fmt, "gated": False,
            "own_rows": False, "bias": False, "skip": 0, "skew": 0.7, **more}


def listed():
    return [
        # one token's residual and norm ahead of a projection: the call made twice a layer and token, where latency counts
        _norm("norm_m1_d4096", 1, 4096),
        # a decode batch behind eight experts a token: weighted sum, norm behind the block, gate, residual kept in 32 bits
        _norm("norm_m13_pairs8_post_gate_d3584", 13, 3584, pairs=8, post=True, gate="channel", res="fp32", plus_one=True),
        # a prompt's tokens behind two experts each
        _norm("norm_prompt_m8001_pairs2_d4096", 8001, 4096, pairs=2),
        # one token's choice among fine-grained experts
        _route("route_m1_e64_k8", 1, 64, 8),
        # a decode batch with three rows of padding, scores by sigmoid with a bias that balances the load, odd number of experts
        _route("route_m61_e160_k6_sigmoid", 61, 160, 6, logits="fp32", scoring="sigmoid", scale=2.5, skip=3),
        # a prompt's choices among many experts, a few of them switched off
        _route("route_prompt_m8001_e256_k8", 8001, 256, 8, masked=5, renormalize=False),
        # one token, eight small experts: the smallest products
        _experts("experts_m1_e64_fp8_gate_up", 1, 64, 8, 2048, 2048, "fp8", gated=True),
        # one token, two large experts in four bits
        _experts("experts_m1_e8_int4_gate_up", 1, 8, 2, 28672, 4096, "int4", gated=True),
        # sixteen tokens (two of them padding) through the down projections of large experts
        _experts("experts_m16_e8_fp8_down", 16, 8, 2, 4096, 14336, "fp8", own_rows=True, skip=2),
        # a large decode batch over many small experts with a bias, sizes that divide nothing
        _experts("experts_m200_e60_int4zp_odd", 200, 60, 4, 1003, 3584, "int4zp", bias=True, own_rows=True),
        # a short prompt over many experts, a few dozen tokens each
        _experts("experts_m509_e64_bf16_gate_up", 509, 64, 4, 2816, 2048, "bf16", gated=True),
        # a prompt through large experts: the largest products
        _experts("experts_prompt_m4001_e8_fp8_gate_up", 4001, 8, 2, 28672, 4096, "fp8", gated=True),
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "route", "experts", "experts", "experts"])
    if op == "norm":
        M, D, pairs = _log_between(rng, 1, 8192), max(8, _log_between(rng, 64, 18944) // 8 * 8), rng.choice([0, 0, 2, 4, 8])
        while M * D * (pairs + 4) > 8001 * 4096 * 6:
            M //= 2
        case = _norm("", M, D, pairs=pairs, post=rng.random() < 0.4, gate=rng.choice(["", "", "channel", "row"]),
                     res=rng.choice(["bf16", "bf16", "fp32", "none"]), scale=rng.choice([1.0, 1.0, 0.22]),
                     plus_one=rng.random() < 0.3)
    elif op == "route":
        M, E = _log_between(rng, 1, 8001), rng.choice([8, 16, 60, 64, 100, 128, 160, 256])
        scoring = rng.choice(["softmax", "softmax", "sigmoid"])
        case = _route("", M, E, rng.choice([1, 2, 4, 6, 8]), logits=rng.choice(["bf16", "fp32"]), scoring=scoring,
                      renormalize=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]), skip=rng.choice([0, 0, M // 5]),
                      masked=rng.choice([0, 0, 3]))
    else:
        E, k = rng.choice([(8, 2), (16, 1), (16, 4), (60, 4), (64, 8), (64, 6), (128, 8), (7, 3), (32, 4)])
        fmt = rng.choice(["bf16", "fp8", "fp8", "int4", "int4zp"])
        step = {"bf16": 8, "fp8": 16, "int4": 128, "int4zp": 128}[fmt]
        K = max(step, _log_between(rng, 256, 14336) // step * step)
        N = _log_between(rng, 64, 28672)
        gated = rng.random() < 0.5
        N += N % 2 if gated else 0
        while E * N * K > 8 * 28672 * 4096:
            N = max(2, N // 4 * 2)
        M = _log_between(rng, 1, 4001)
        while M * k * N * K > 8002 * 28672 * 4096 or M * k * N > 8002 * 28672:
            M = max(1, M // 2)
        case = _experts("", M, E, k, N, K, fmt, gated=gated, own_rows=rng.random() < 0.5,
                        bias=fmt != "int4" and rng.random() < 0.3, skip=rng.choice([0, 0, M // 5]),
                        skew=rng.choice([0.0, 0.7, 1.5]))
    del case["name"]
    return case


def _choices(case):
    """[M, k] different experts of each token, drawn by the case's sizes alone; -1 in the tokens that chose none."""
    M, E, k = case["M"], case["E"], case["k"]
    rng = np.random.default_rng([M, E, k])
    odds = rng.normal(size=E) * case["skew"]
    ids = np.argsort(-(odds + rng.gumbel(size=(M, E))), axis=1)[:, :k]
    ids[M - case["skip"]:] = -1
    return ids


def _bf16(*shape, gen):
    return torch.randn(*shape, dtype=torch.bfloat16, device="cuda", generator=gen)


def _prepare_norm(case, gen):
    M, D, P = case["M"], case["D"], case["pairs"]
    off = 1.0 if case["plus_one"] else 0.0
    s = {"x": _bf16(*((M, P, D) if P else (M, D)), gen=gen), "weights": None, "residual": None, "post": None, "gate": None}
    if P:
        s["weights"] = torch.softmax(torch.randn(M, P, device="cuda", generator=gen), dim=1)
    if case["res"] != "none":
        s["residual"] = _bf16(M, D, gen=gen).mul_(4.0).to(torch.float32 if case["res"] == "fp32" else torch.bfloat16)
    s["norm"] = _bf16(D, gen=gen).mul_(0.2).add_(1.0 - off)
    if case["post"]:
        s["post"] = _bf16(D, gen=gen).mul_(0.2).add_(1.0 - off)
    if case["gate"]:
        s["gate"] = _bf16(*((M, D) if case["gate"] == "row" else (D,)), gen=gen).mul_(0.3)
    return s


def _prepare_route(case, gen):
    M, E = case["M"], case["E"]
    dtype = torch.float32 if case["logits"] == "fp32" else torch.bfloat16
    logits = torch.randn(M, E, device="cuda", generator=gen).mul_(1.5).to(dtype)
    perm = torch.randperm(M, device="cuda", generator=gen)
    logits[perm[:case["skip"]]] = -math.inf
    logits[:, torch.randperm(E, device="cuda", generator=gen)[:case["masked"]]] = -math.inf
    s = {"logits": logits, "bias": None}
    if case["scoring"] == "sigmoid":
        s["bias"] = torch.randn(E, device="cuda", generator=gen).mul_(0.05)
    return s


def _prepare_experts(case, gen):
    M, E, k, N, K, fmt = (case[n] for n in ("M", "E", "k", "N", "K", "fmt"))
    label = torch.randperm(E, device="cuda", generator=gen)
    ids = torch.from_numpy(_choices(case)).cuda()
    ids = torch.where(ids >= 0, label[ids.clamp(min=0)], -1)[torch.randperm(M, device="cuda", generator=gen)].flatten()
    key = torch.where(ids >= 0, ids, E)
    s = {"order": torch.sort(key, stable=True).indices.int(),
         "offsets": torch.searchsorted(torch.sort(key).values, torch.arange(E + 1, device="cuda")).int()}
    counts = np.zeros(E + 1, dtype=int)
    base = _choices(case).ravel()
    counts[label.cpu().numpy()] = np.bincount(base[base >= 0], minlength=E)[:E]
    s["counts"] = counts[:E].tolist()          # known on the host as a program that keeps its ids there has them; plain form only
    s["x"] = _bf16(M * k if case["own_rows"] else M, K, gen=gen)
    if fmt == "bf16":
        s["W"] = (_bf16(E, N, K, gen=gen).mul_(K ** -0.5),)
    elif fmt == "fp8":
        W = _bf16(E, N, K, gen=gen).mul_(100.0).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn)
        s["W"] = (W, torch.rand(E, N, device="cuda", generator=gen).mul_(0.01 * K ** -0.5).add_(0.005 * K ** -0.5))
    else:
        W = torch.randint(0, 256, (E, N, K // 2), dtype=torch.uint8, device="cuda", generator=gen)
        scales = torch.rand(E, N, K // 128, device="cuda", generator=gen).mul_(0.3).add_(0.05).mul_(K ** -0.5)
        if fmt == "int4":
            s["W"] = (W, scales.half())
        else:
            zeros = torch.randint(0, 256, (E, N, (K // 128 + 1) // 2), dtype=torch.uint8, device="cuda", generator=gen)
            s["W"] = (W, scales.bfloat16(), zeros)
    s["bias"] = _bf16(E, N, gen=gen).mul_(0.2) if case["bias"] else None
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    make = {"norm": _prepare_norm, "route": _prepare_route, "experts": _prepare_experts}[case["op"]]
    return {"case": case, **make(case, gen)}


# ---- plain forms --------------------------------------------------------------------------------------------------------

def _rms(x, w, plus_one):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * (w.float() + 1.0 if plus_one else w.float())


def _plain_norm(s, case):
    y = s["x"].float()
    if case["pairs"]:
        y = (y * s["weights"][:, :, None]).sum(1)
    if case["post"]:
        y = _rms(y, s["post"], case["plus_one"])
    if case["gate"]:
        y = y * s["gate"].float()
    r = y * case["scale"]
    if s["residual"] is not None:
        r = r + s["residual"].float()
    return (_rms(r, s["norm"], case["plus_one"]).to(torch.bfloat16),
            r.to(torch.float32 if case["res"] == "fp32" else torch.bfloat16))


def _plain_route(s, case):
    M, E, k = case["M"], case["E"], case["k"]
    logits = s["logits"].double()               # 64 bits: neighbouring scores decide the choice
    held = (logits > -math.inf).logical_and_(logits == logits)
    if case["scoring"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-logits))
        key = score + s["bias"].double()
    else:
        key = logits
        score = torch.exp(logits - torch.where(held, logits, -math.inf).amax(1, keepdim=True).clamp(min=-1e300))
        score = torch.where(held, score, 0.0)
        score = score / score.sum(1, keepdim=True).clamp(min=1e-300)
    key = torch.where(held, key, -math.inf)
    ids = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :k]
    there = held.gather(1, ids)
    weights = torch.where(there, score.gather(1, ids), 0.0)
    if case["renormalize"]:
        weights = weights / weights.sum(1, keepdim=True).clamp(min=1e-300)
    ids = torch.where(there, ids, -1)
    flat = torch.where(ids >= 0, ids, E).flatten()
    ordered = torch.sort(flat, stable=True)
    offsets = (ordered.values[None, :] < torch.arange(E + 1, device="cuda")[:, None]).sum(1)
    return ids.int(), (weights * case["scale"]).float(), ordered.indices.int(), offsets.int()


def _nibbles(q):
    return torch.stack([q & 15, q >> 4], dim=-1).flatten(-2)


def _expert_weights(W, fmt, e):
    """Expert e's matrix [N, K]."""
    if fmt == "bf16":
        return W[0][e].float()
    if fmt == "fp8":
        return W[0][e].float() * W[1][e][:, None]
    q = _nibbles(W[0][e]).float().unflatten(1, (-1, 128))
    zero = 8.0 if fmt == "int4" else _nibbles(W[2][e])[:, :q.shape[1], None].float()
    return ((q - zero) * W[1][e].float()[:, :, None]).flatten(1)


def _plain_experts(s, case):
    N, R = case["N"], case["M"] * case["k"]
    half = N // 2
    out = torch.zeros(R, half if case["gated"] else N, dtype=torch.bfloat16, device="cuda")
    at = 0
    for e, n in enumerate(s["counts"]):
        if n == 0:
            continue
        pair = s["order"][at:at + n].long()
        x = s["x"][pair if case["own_rows"] else pair // case["k"]].float()
        y = torch.matmul(x, _expert_weights(s["W"], case["fmt"], e).t())
        if case["bias"]:
            y = y + s["bias"][e].float()
        if case["gated"]:
            g = y[:, :half]
            y = g / (1.0 + torch.exp(-g)) * y[:, half:]
        out[pair] = y.to(torch.bfloat16)
        at += n
    return out


def run(state):
    s, case = state, state["case"]
    if case["op"] == "norm":
        if own:
            return _ops().add_norm(s["x"], s["residual"], s["norm"], post_norm=s["post"], gate=s["gate"],
                                   weights=s["weights"], scale=case["scale"], eps=1e-6, plus_one=case["plus_one"])
        return _plain_norm(s, case)
    if case["op"] == "route":
        if own:
            return _ops().route_experts(s["logits"], case["k"], bias=s["bias"], scoring=case["scoring"],
                                        renormalize=case["renormalize"], scale=case["scale"])
        return _plain_route(s, case)
    if own:
        o, fmt = _ops(), case["fmt"]
        if fmt == "int4":
            return o.experts_int4(*s["W"], s["x"], s["order"], s["offsets"], gated=case["gated"])
        call = {"bf16": o.experts_bf16, "fp8": o.experts_fp8, "int4zp": o.experts_int4_zp}[fmt]
        return call(*s["W"], s["x"], s["order"], s["offsets"], bias=s["bias"], gated=case["gated"])
    return _plain_experts(s, case)


def work(case):
    M = case["M"]
    if case["op"] == "norm":
        D, P = case["D"], case["pairs"]
        res = {"bf16": 4.0, "fp32": 8.0, "none": 2.0}[case["res"]]
        rows = M * D * (2.0 * max(1, P) + res + 2.0 + (2.0 if case["gate"] == "row" else 0.0)) + 4.0 * M * P
        return {"bytes": rows + D * (2.0 + 2.0 * case["post"] + 2.0 * (case["gate"] == "channel")),
                "flops": M * D * (2.0 * P + 5.0 + 4.0 * case["post"] + 1.0 * bool(case["gate"]))}
    if case["op"] == "route":
        E, k = case["E"], case["k"]
        e = 4.0 if case["logits"] == "fp32" else 2.0
        return {"bytes": M * (E * e + 12.0 * k) + 4.0 * (E + 1) + (4.0 * E if case["scoring"] == "sigmoid" else 0.0),
                "flops": M * (4.0 * E + 4.0 * k)}
    E, k, N, K = (case[n] for n in ("E", "k", "N", "K"))
    ids = _choices(case).ravel()
    ids = ids[ids >= 0]
    used, R = len(set(ids.tolist())), M * k
    row = {"bf16": 2.0 * K, "fp8": K + 4.0, "int4": K / 2 + 2.0 * (K // 128),
           "int4zp": K / 2 + 2.0 * (K // 128) + (K // 128 + 1) // 2}[case["fmt"]] + 2.0 * case["bias"]
    rows = len(ids) if case["own_rows"] else M - case["skip"]
    return {"bytes": used * N * row + 2.0 * rows * K + 2.0 * R * (N // 2 if case["gated"] else N) + 4.0 * (R + E + 1),
            "flops": 2.0 * len(ids) * N * K}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------

def _exact_norm(s, case):
    D, one = case["D"], 1.0 if case["plus_one"] else 0.0
    x = s["x"].double()
    if case["pairs"]:
        x = torch.stack([w @ rows for w, rows in zip(s["weights"].double(), x)])
    if s["post"] is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + 1e-6) * (one + s["post"].double())
    if s["gate"] is not None:
        x = s["gate"].double() * x
    r = case["scale"] * x
    if s["residual"] is not None:
        r = s["residual"].double() + r
    return r / torch.sqrt((r * r).sum(-1, keepdim=True) / D + 1e-6) * (one + s["norm"].double()), r


def _exact_route(s, case):
    """An expert's rank is the number of experts that come before it."""
    M, E, k = case["M"], case["E"], case["k"]
    ids, weights = [], []
    index = torch.arange(E, device="cuda")
    for logits in s["logits"].double().split(512):
        open_ = torch.isfinite(logits)
        if case["scoring"] == "sigmoid":
            score = torch.sigmoid(logits)
            key = score + s["bias"].double()
        else:
            score, key = torch.nan_to_num(torch.softmax(logits, dim=1)), logits
        score = torch.where(open_, score, 0.0)
        a, b = key[:, :, None], key[:, None, :]
        ahead = (b > a) | ((b == a) & (index[None, :] < index[:, None]))
        rank = (ahead & open_[:, None, :]).sum(2)
        for j in range(k):
            here = (rank == j) & open_
            ids.append(torch.where(here.any(1), (here * index).sum(1), -1))
            weights.append((here * score).sum(1))
        w = torch.stack(weights[-k:], 1)
        ids[-k:], weights[-k:] = [torch.stack(ids[-k:], 1)], [
            case["scale"] * (torch.nan_to_num(w / w.sum(1, keepdim=True)) if case["renormalize"] else w)]
    ids = torch.cat(ids)
    flat, order, offsets = ids.flatten(), [], [0]
    for e in range(E):
        order.append((flat == e).nonzero()[:, 0])
        offsets.append(offsets[-1] + len(order[-1]))
    order.append((flat < 0).nonzero()[:, 0])
    return (ids.int(), torch.cat(weights), torch.cat(order).int(),
            torch.tensor(offsets, dtype=torch.int32, device="cuda"))


def _weights64(W, case, e):
    """What the codes of expert e stand for."""
    if case["fmt"] in ("bf16", "fp8"):
        full = W[0][e].float().double()
        return full if case["fmt"] == "bf16" else full.mul_(W[1][e].double().view(-1, 1))
    full = torch.empty(case["N"], case["K"], dtype=torch.float64, device="cuda")
    full[:, 0::2], full[:, 1::2] = W[0][e] % 16, W[0][e] // 16
    for g in range(case["K"] // 128):
        z = 8 if case["fmt"] == "int4" else ((W[2][e][:, g // 2] >> (4 * (g % 2))) & 15).double()[:, None]
        full[:, 128 * g:128 * g + 128] = (full[:, 128 * g:128 * g + 128] - z) * W[1][e][:, g:g + 1].double()
    return full


def _exact_experts(s, case):
    R, N = case["M"] * case["k"], case["N"]
    out = torch.zeros(R, N // 2 if case["gated"] else N, dtype=torch.float64, device="cuda")
    bounds = s["offsets"].tolist()
    for e in range(case["E"]):
        pair = s["order"][bounds[e]:bounds[e + 1]].long()
        if len(pair) == 0:
            continue
        rows = pair if case["own_rows"] else torch.div(pair, case["k"], rounding_mode="floor")
        y = (_weights64(s["W"], case, e) @ s["x"][rows].double().t()).t()
        if s["bias"] is not None:
            y = y + s["bias"][e].double()
        if case["gated"]:
            y = y[:, :N // 2] * torch.sigmoid(y[:, :N // 2]) * y[:, N // 2:]
        out[pair] = y
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "route": _exact_route, "experts": _exact_experts}[case["op"]](s, case)
