"""Dimensions of size 1 have no stride that counts: the operators take such tensors whatever stride they carry (a transposed column,
a cache of one page or one head cut out of something else) and give the bits of the plain layout."""
import pytest
import torch

from decode_util import bits, on
from gpu_util import note
from paia_gemv import ops
import test_gpu_attention
import test_gpu_lora
import test_gpu_rope

pytestmark = pytest.mark.gpu


def odd(t, dims):
    """The same tensor with stride 1 in dimensions of size 1 (the kernels' strides are multiples of 8 elements)."""
    assert all(t.shape[d] == 1 for d in dims)
    s = list(t.stride())
    for d in dims:
        s[d] = 1
    r = t.as_strided(t.shape, s)
    assert r.data_ptr() == t.data_ptr() and r.stride() == tuple(s)
    return r


def test_rope_append(cuda):
    note("unit dims rope")
    o = test_gpu_rope.operands(1, 8, 1, 128, 128, False, "hpd", 16, True, pages=1)
    want = test_gpu_rope.call(o, cuda, 8)
    d = {k: on(v, cuda) for k, v in o.items()}
    k, v = (odd(d[n], (0, 1)) for n in ("k_cache", "v_cache"))
    q = ops.rope_append(odd(d["qkv"], (0,)), d["positions"], d["cos_sin"], k, v, d["slots"], 8, q_norm=d["q_norm"],
                        k_norm=d["k_norm"])
    assert torch.equal(bits(q), bits(want[0])) and torch.equal(bits(k), bits(want[1])) and torch.equal(bits(v), bits(want[2]))


def test_paged_attention(cuda):
    note("unit dims attention")
    o = test_gpu_attention.operands([1], 1, 1, 1, 128, False, "hpd", 1)
    for n in ("k_cache", "v_cache"):
        o[n] = o[n][:1].contiguous()
    o["table"] = torch.zeros(1, 1, dtype=torch.int32)
    want = test_gpu_attention.call(o, cuda)
    d = {k: on(v, cuda) for k, v in o.items()}
    out, lse = ops.paged_attention(odd(d["q"], (0, 1, 2)), odd(d["k_cache"], (0, 1, 2)), odd(d["v_cache"], (0, 1, 2)),
                                   odd(d["table"], (0, 1)), d["lens"], return_lse=True)
    assert torch.equal(bits(out), bits(want[0])) and torch.equal(lse, want[1])
    q = d["q"].view(-1, 1).t()[:, None]                # [1, 1, 128] of a column
    assert torch.equal(bits(ops.paged_attention(q, d["k_cache"], d["v_cache"], d["table"], d["lens"])).view(-1),
                       bits(want[0]).view(-1))


@pytest.mark.parametrize("rank", [8, 40])
def test_lora_add(cuda, rank):
    note(f"unit dims lora rank={rank}")
    o = test_gpu_lora.operands(1, 256, [96], rank, 2, ids=[1])
    want = test_gpu_lora.call(o, cuda, None)
    d = {k: v.to(cuda) for k, v in o.items()}
    x, y = (d[n].view(-1, 1).t() for n in ("x", "y"))
    assert x.stride(0) == 1 and y.stride(0) == 1
    out = torch.empty(96, 1, dtype=torch.bfloat16, device=cuda).t()
    ops.lora_add(y, x, d["A"], d["B"], d["ids"], scaling=d["scaling"], out=out)
    assert torch.equal(bits(out), bits(want))
    ops.lora_add(odd(d["y"], (0,)), odd(d["x"], (0,)), d["A"], d["B"], d["ids"], scaling=d["scaling"], out=out)
    assert torch.equal(bits(out), bits(want))
