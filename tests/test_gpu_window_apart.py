"""Gradients of sinks whose further queries have a launch of their own (SinkChunks::apart: long
calls), against the closed forms in 64 bits: whole dK, dV, dK2 and dV2 of the first and the last
key/value head, and the sinks' rows alone, the sum of parts that two kernels write.

Tolerances: those of test_gpu_window.py (check), fixed before the first run. A sink's row sums up to
2500 queries' terms, each rounded to the inputs' type once on its own (u relatively; fp16 below
2^-14 by 2^-25, 3 % of a term's size of 1e-6 where a typical one, P = 1 / window, is 1e-3), so
roundings still add up in squares, as the terms themselves do: the same 4 u. In fp32 the running sum of
n such terms adds 2^-24 sqrt(n / 2) = 2.1e-6 of the result to a score's 4e-6, three times in a chain:
1.8e-5, within 2e-5.
"""

from __future__ import annotations

import pytest
import torch

import window_reference as ref
from helpers import default_scale, make_inputs
from test_gpu_window import case_id, check

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32

# (batch, n_q, n_k, heads, kv_heads, head_dim, dtype, alignment, window, sinks)
CASES = [
    (2, 2500, 2500, 24, 24, 64, BF16, "top_left", 1000, 4),
    (1, 2000, 2600, 64, 16, 64, FP16, "bottom_right", 800, 70),  # sinks in three key blocks
    (2, 2300, 2000, 32, 8, 64, BF16, "bottom_right", 1200, 35),  # the first queries see nothing
    (1, 2500, 2500, 48, 12, 128, BF16, "top_left", 1000, 33),
    (3, 1700, 1500, 32, 8, 128, FP16, "top_left", 700, 1),       # the last windows end behind the keys
    (2, 2200, 2200, 32, 16, 64, FP32, "top_left", 900, 40),
]


@pytest.mark.parametrize("case", CASES, ids=case_id)
def test_gradients(case, cuda_device):
    from flash_hog import _hip

    B, nq, nk, H, Hk, D, dtype, alignment, window, sinks = case
    print("[case] apart", case_id(case), flush=True)
    scale, group = default_scale(D), H // Hk
    code = 2 if alignment == "bottom_right" else 1
    x = make_inputs(B, nq, nk, H, D, dtype, seed=5, kv_heads=Hk)
    mask = ref.visible(nq, nk, alignment, window, sinks)
    g = {n: t.to(cuda_device) for n, t in x.items()}
    o, lse = _hip.attention_fwd(g["q"], g["k"], g["v"], code, scale, window, sinks)
    args = (g["q"], g["k"], g["v"], o, g["do"])
    first = _hip.attention_bwd(*args, lse, code, scale, window, sinks)[:3]
    second = _hip.attention_bwdbwd(*args, g["ddq"], g["ddk"], g["ddv"], lse, code, scale, window=window, sinks=sinks)
    again = _hip.attention_bwdbwd(*args, g["ddq"], g["ddk"], g["ddv"], lse, code, scale, window=window, sinks=sinks)
    assert all(torch.equal(a, b) for a, b in zip(second, again))
    o, lse = o.cpu(), lse.cpu()
    for b, hk in ((0, 0), (B - 1, Hk - 1)):
        heads = {n: slice(hk, hk + 1) if n in ("k", "v", "ddk", "ddv") else slice(hk * group, (hk + 1) * group) for n in x}
        one = {n: t[b:b + 1, :, heads[n]] for n, t in x.items()}
        o1, lse1 = o[b:b + 1, :, heads["q"]], lse[b:b + 1, heads["q"]]
        want = ref.backward(one["q"], one["k"], one["v"], o1, one["do"], lse1, mask, scale)[:3]
        want2 = ref.double_backward(one["q"], one["k"], one["v"], o1, one["do"], one["ddq"], one["ddk"], one["ddv"], lse1,
                                    mask, scale)
        for got, r, n in zip((*first, *second), (*want, *want2), ("dq", "dk", "dv", "dq2", "dk2", "dv2", "ddo")):
            a = got[b:b + 1, :, heads["k" if n[:2] in ("dk", "dv") else "q"]]
            check(a, r, dtype, f"{n} of head {hk}")
            if n[:2] in ("dk", "dv"):
                check(a[:, :sinks], r[:, :sinks], dtype, f"{n} of head {hk}, sinks")
                check(a[:, sinks:], r[:, sinks:], dtype, f"{n} of head {hk}, others")
