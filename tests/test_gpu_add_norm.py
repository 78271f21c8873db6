"""ops.add_norm and GemvLib.add_norm against the definition in 64 bits; tolerances as expert_util.norm64 derives them."""
import pytest
import torch

from decode_util import BF16_HALF, F32_EPS, bits
from expert_util import norm64
from gpu_util import note
from paia_gemv import load_lib, ops

pytestmark = pytest.mark.gpu


def operands(M, D, pairs=0, post=False, gate="", residual="bf16", seed=0):
    g = torch.Generator().manual_seed(seed + M * 7919 + D)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    o = {"x": r(*((M, pairs, D) if pairs else (M, D))).bfloat16(), "norm": (r(D) * 0.2 + 1).bfloat16(),
         "residual": None if residual == "none" else (r(M, D) * 3).to(torch.float32 if residual == "fp32" else torch.bfloat16),
         "post_norm": (r(D) * 0.2 + 1).bfloat16() if post else None, "weights": None, "gate": None}
    if pairs:
        o["weights"] = torch.softmax(r(M, pairs), 1)
        o["weights"][::3, 0] = 0.0
    if gate:
        o["gate"] = r(*((M, D) if gate == "row" else (D,))).bfloat16()
    return o


def to(o, dev):
    return {k: None if v is None else v.to(dev) for k, v in o.items()}


def check(o, got, **more):
    h, r, eh, er = norm64(**o, **more)
    out, res = (t.cpu().double() for t in got)
    half = F32_EPS if got[1].dtype == torch.float32 else BF16_HALF
    for got_, want, err, step in ((out, h, eh, BF16_HALF), (res, r, er, half)):
        held = want == want                          # 0 / 0 where a row of zeros is normed without eps
        assert torch.equal(got_ == got_, held)
        worst = ((got_ - want).abs() - (err + step * (want.abs() + err)))[held].max() if held.any() else 0
        assert worst <= 0, f"beyond the bound by {worst:.3e}"
    assert got[0].dtype == torch.bfloat16


@pytest.mark.parametrize("D", [8, 64, 520, 1000, 3584, 4096, 8200, 16384, 18944, 32768])
@pytest.mark.parametrize("M", [1, 3, 300])
def test_sizes(cuda, M, D):
    for pairs, post, gate, residual in ((0, False, "", "bf16"), (3, True, "row", "fp32"), (8, False, "channel", "none")):
        if M * D * max(1, pairs) > 6e6:
            continue
        note(f"add_norm M={M} D={D} pairs={pairs} post={post} gate={gate!r} residual={residual}")
        o = operands(M, D, pairs, post, gate, residual)
        check(o, ops.add_norm(**to(o, cuda)))


@pytest.mark.parametrize("pairs", [0, 1, 2, 5, 8, 13])
@pytest.mark.parametrize("residual", ["bf16", "fp32", "none"])
def test_options(cuda, pairs, residual):
    for post in (False, True):
        for gate in ("", "channel", "row"):
            for plus_one, scale, eps in ((False, 1.0, 1e-6), (True, 0.22, 1e-5), (False, -3.0, 0.0)):
                o = operands(5, 264, pairs, post, gate, residual, seed=pairs)
                more = dict(plus_one=plus_one, scale=scale, eps=eps)
                note(f"add_norm pairs={pairs} {residual} {post} {gate!r} {more}")
                check(o, ops.add_norm(**to(o, cuda), **more), **more)


def test_a_weight_of_zero_hides_its_row(cuda):
    """NaN and infinities in pairs of weight 0 reach nothing; in others they reach their row alone."""
    o = operands(4, 128, 6)
    o["weights"][1, :] = 0.0
    clean = {**o, "x": o["x"].clone()}
    o["x"][0, 0], o["x"][1], o["x"][3, 0, 5] = float("nan"), float("inf"), float("-inf")
    o["weights"][0, 0] = o["weights"][3, 0] = 0.0
    clean["weights"] = o["weights"]
    note("add_norm weights of 0")
    got, want = ops.add_norm(**to(o, cuda)), ops.add_norm(**to(clean, cuda))
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(got, want))
    check(clean, got)
    o["x"][2, 1, 7] = float("nan")
    got = ops.add_norm(**to(o, cuda))
    assert got[0][2].isnan().all() and got[1][2, 7].isnan() and got[0][[0, 1, 3]].isfinite().all()


def test_zero_rows(cuda):
    """A row of zeros stays zero (eps holds the quotient), without eps it is 0 / 0."""
    o = operands(2, 64, residual="none")
    o["x"][0] = 0.0
    note("add_norm zero rows")
    assert (ops.add_norm(**to(o, cuda))[0][0] == 0).all()
    got = ops.add_norm(**to(o, cuda), eps=0.0)[0]
    assert got[0].isnan().all() and got[1].isfinite().all()


@pytest.mark.parametrize("pairs", [0, 3])
def test_strided_and_in_place(cuda, pairs):
    """Rows of wider tensors; the residual updated in place; out in x's place."""
    o = operands(6, 136, pairs, True, "row", "bf16")
    want = ops.add_norm(**to(o, cuda))
    d = to(o, cuda)

    def wide(t):
        w = torch.full((*t.shape[:-1], t.shape[-1] + 24), float("nan"), dtype=t.dtype, device=cuda)
        w[..., 8:8 + t.shape[-1]] = t
        return w, w[..., 8:8 + t.shape[-1]]

    note(f"add_norm strided pairs={pairs}")
    (xw, d["x"]), (rw, d["residual"]), (_, d["gate"]), (ow, out) = wide(d["x"]), wide(d["residual"]), wide(d["gate"]), wide(want[0])
    got = ops.add_norm(**d, out=out, residual_out=d["residual"])
    assert got[0] is out and torch.equal(bits(out.contiguous()), bits(want[0]))
    assert torch.equal(bits(d["residual"].contiguous()), bits(want[1]))
    for w in (ow, rw):
        assert w[:, :8].isnan().all() and w[:, 144:].isnan().all()
    if not pairs:
        d = to(o, cuda)
        ops.add_norm(**d, out=d["x"], residual_out=d["residual"])
        assert torch.equal(bits(d["x"]), bits(want[0])) and torch.equal(bits(d["residual"]), bits(want[1]))
        part = ops.add_norm(**to(o, cuda), out=torch.empty_like(want[0]))
        assert torch.equal(bits(part[1]), bits(want[1]))


def test_many_rows_and_far_offsets(cuda):
    """More rows than a launch has blocks (2^21), and rows beyond 2^32 bytes."""
    note("add_norm many rows")
    M, D = (1 << 21) + 3, 8
    x = torch.randn(M, D, device=cuda).bfloat16()
    norm = torch.ones(D, device=cuda).bfloat16()
    out, r = ops.add_norm(x, None, norm)
    assert torch.equal(r, x)
    tail = ops.add_norm(x[-5:].clone(), None, norm)[0]
    assert torch.equal(out[-5:], tail) and torch.equal(out[:5], ops.add_norm(x[:5].clone(), None, norm)[0])
    note("add_norm far rows")
    M, D = 70000, 32768
    x = torch.zeros(M, D, dtype=torch.bfloat16, device=cuda)
    x[-2:] = torch.randn(2, D, device=cuda).bfloat16()
    out, r = ops.add_norm(x, None, torch.ones(D, device=cuda).bfloat16())
    want = ops.add_norm(x[-2:].clone(), None, torch.ones(D, device=cuda).bfloat16())
    assert torch.equal(out[-2:], want[0]) and torch.equal(r[-2:], want[1]) and not out[:-2].any()


def test_graph_and_another_stream(cuda):
    o = operands(3, 512, 2, True, "channel", "fp32")
    d = to(o, cuda)
    want = ops.add_norm(**d)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.add_norm(**d)
    for i in range(3):
        d["x"].copy_(o["x"] * (i + 1))
        torch.cuda.synchronize()
        note(f"add_norm replay {i}")
        graph.replay()
        torch.cuda.synchronize()
        eager = ops.add_norm(**d)
        assert all(torch.equal(bits(a), bits(b)) for a, b in zip(got, eager))
    d["x"].copy_(o["x"])
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        lib, out, r = load_lib(), torch.empty_like(want[0]), torch.empty_like(want[1])
        lib.add_norm(d["x"].data_ptr(), d["residual"].data_ptr(), d["norm"].data_ptr(), out.data_ptr(), r.data_ptr(), 3, 512,
                     weights_ptr=d["weights"].data_ptr(), pairs=2, post_norm_ptr=d["post_norm"].data_ptr(),
                     gate_ptr=d["gate"].data_ptr(), residual_fp32=True)
    st.synchronize()
    assert torch.equal(bits(out), bits(want[0])) and torch.equal(r, want[1])


def test_refusals(cuda):
    o = to(operands(4, 64, 2, True, "row"), cuda)

    def refused(match, **change):
        with pytest.raises(RuntimeError, match=match):
            ops.add_norm(**{**o, **change})

    refused("x must be", x=o["x"].float())
    refused("x must be", x=o["x"].transpose(1, 2))
    refused("weights go with", weights=None)
    refused("weights go with", x=o["x"][:, 0])
    refused("weights must be", weights=o["weights"].double())
    refused("weights must be", weights=o["weights"][:3])
    refused("residual must be", residual=o["residual"].half())
    refused("residual must be", residual=o["residual"][:3])
    refused("residual must be on", residual=o["residual"].cpu())
    refused("gate must be", gate=o["gate"][:, :8])
    refused("gate must be", gate=o["gate"].float())
    refused("norm must be", norm=o["norm"][:8])
    refused("post_norm must be", post_norm=o["post_norm"].float())
    refused("out must be", out=torch.empty(4, 63, dtype=torch.bfloat16, device=cuda))
    refused("residual_out must be", residual_out=torch.empty(4, 64, device=cuda))
    refused("-2", eps=-1.0)
    refused("-2", residual=torch.empty(4, 68, dtype=torch.bfloat16, device=cuda)[:, 1:65])
    with pytest.raises(RuntimeError, match="-2"):
        e = torch.empty(2, 12, dtype=torch.bfloat16, device=cuda)
        ops.add_norm(e, None, e[0])
    assert ops.add_norm(o["x"][:0], o["residual"][:0], o["norm"], weights=o["weights"][:0])[0].shape == (0, 64)
