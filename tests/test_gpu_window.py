"""Windowed attention with sinks: forward, first backward and double backward against the
closed forms in 64 bits, through the C ABI's wrappers and through dot_product_attention.

Tolerances, fixed before the first run. u = eps / 2 is a rounding's relative size.
- 2-byte types, 2-norm of the error over the output's: the result carries its own rounding
  (u), those of the probabilities and score gradients that enter its last products (u each)
  and, in the backwards, of the O that D is formed from: at most 4 u, as independent
  roundings add up in squares and P (dP - D) at most doubles one. The largest single error
  over the largest entry: twice that, for a row whose terms all round one way.
- fp32: scores of magnitude up to 6 are sums of up to 128 products, off by about
  sqrt(128) 6 2^-24 = 4e-6, which the exponential hands on relatively; the second derivative
  chains three such sums: 2e-5, and twice that for a single entry.
Outputs that are zero in exact arithmetic (the gradients of queries that see one key) are
measured against a floor: DEGENERATE_FLOOR, and 0.1 for fp32, whose tolerance is so much
tighter: there dP - D cancels two sums of D <= 128 products of N(0, 1) numbers. Partial sums
stay below 3 sqrt(64) = 24 at head dim 64, so an addition rounds by at most 24 2^-24 / 2 and
64 of them by about sqrt(64) as much, 6e-6; the two sums 8e-6, times scale (1/8) and an entry
of K (up to 4): 4e-6, which is twice the tolerance of 2e-5 on a scale of 0.1.
"""

from __future__ import annotations

import pytest
import torch

import window_reference as ref
from helpers import DEGENERATE_FLOOR, default_scale, make_inputs

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def tolerance(dtype):
    return 2e-5 if dtype == FP32 else 4 * torch.finfo(dtype).eps / 2


def check(got, want, dtype, what):
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), f"{what}: not finite"
    tol = tolerance(dtype)
    floor = 0.1 if dtype == FP32 else DEGENERATE_FLOOR
    norm = max(want.norm().item(), floor * want.numel() ** 0.5)
    err = (got - want).norm().item() / norm
    big = (got - want).abs().max().item() / max(want.abs().max().item(), floor)
    assert err <= tol, f"{what}: 2-norm error {err:.2e} > {tol:.2e}"
    assert big <= 2 * tol, f"{what}: largest error {big:.2e} > {2 * tol:.2e}"


# (batch, n_q, n_k, heads, kv_heads, head_dim, dtype, alignment, window, sinks)
CASES = [
    (1, 1, 1, 1, 1, 64, BF16, "top_left", 1, 0),
    (1, 70, 70, 2, 2, 64, BF16, "top_left", 1, 0),         # every query sees itself alone
    (1, 70, 70, 2, 1, 64, FP16, "top_left", 1, 1),
    (2, 200, 200, 2, 2, 64, BF16, "top_left", 33, 0),
    (1, 333, 333, 4, 2, 64, BF16, "top_left", 64, 4),
    (1, 257, 257, 2, 1, 64, FP16, "top_left", 100, 31),
    (1, 1300, 1300, 1, 1, 64, BF16, "top_left", 40, 4),    # sinks' queries in three chunks
    (1, 1300, 1300, 2, 1, 64, FP16, "top_left", 17, 70),   # sinks in two key blocks
    (1, 900, 900, 1, 1, 64, BF16, "top_left", 32, 300),    # more sinks than window
    (1, 130, 60, 2, 2, 64, BF16, "top_left", 20, 0),       # queries behind the last window see nothing
    (1, 300, 60, 2, 2, 64, BF16, "top_left", 20, 3),       # ... or sinks only
    (1, 300, 60, 1, 1, 64, BF16, "top_left", 20, 1),       # ... or one sink
    (1, 150, 90, 2, 2, 64, BF16, "bottom_right", 16, 2),   # the first queries see nothing
    (1, 90, 300, 2, 2, 64, BF16, "bottom_right", 50, 5),
    (1, 1, 300, 2, 2, 64, BF16, "bottom_right", 50, 5),    # one query of a long context
    (1, 5, 1000, 2, 1, 64, FP16, "bottom_right", 700, 1),
    (1, 300, 300, 2, 1, 128, BF16, "top_left", 65, 4),
    (2, 190, 190, 4, 2, 128, FP16, "top_left", 40, 0),
    (1, 700, 700, 1, 1, 128, BF16, "top_left", 30, 2),
    (1, 100, 260, 2, 2, 128, BF16, "bottom_right", 70, 40),
    (1, 200, 200, 2, 1, 256, BF16, "top_left", 65, 4),
    (1, 650, 650, 1, 1, 256, FP16, "top_left", 48, 33),
    (1, 90, 40, 1, 1, 256, BF16, "top_left", 20, 0),
    (1, 300, 300, 2, 1, 64, FP32, "top_left", 65, 4),
    (1, 700, 700, 1, 1, 64, FP32, "top_left", 30, 40),
    (1, 130, 60, 1, 1, 64, FP32, "top_left", 20, 1),
    (1, 70, 150, 2, 2, 64, FP32, "bottom_right", 1, 0),
    (1, 200, 200, 2, 1, 128, FP32, "top_left", 50, 4),
    (1, 100, 230, 2, 2, 128, FP32, "bottom_right", 64, 0),
]


def case_id(c):
    B, nq, nk, H, Hk, D, dt, al, w, s = c
    return f"b{B}_q{nq}_k{nk}_h{H}_{Hk}_d{D}_{str(dt)[6:]}_{al}_w{w}_s{s}"


def run_case(c, device, scale=None, seed=3):
    from flash_hog import _hip

    B, nq, nk, H, Hk, D, dtype, alignment, window, sinks = c
    print("[case]", case_id(c), scale, flush=True)
    scale = default_scale(D) if scale is None else scale
    code = 2 if alignment == "bottom_right" else 1
    x = make_inputs(B, nq, nk, H, D, dtype, seed=seed, kv_heads=Hk)
    mask = ref.visible(nq, nk, alignment, window, sinks)
    g = {n: t.to(device) for n, t in x.items()}

    o, lse = _hip.attention_fwd(g["q"], g["k"], g["v"], code, scale, window, sinks)
    o_ref, lse_ref = ref.forward(x["q"], x["k"], x["v"], mask, scale)
    check(o, o_ref, dtype, "o")
    empty = ~mask.any(-1)
    assert torch.isposinf(lse[:, :, empty]).all() and (o[:, empty] == 0).all()
    # a logsumexp carries its scores' error: the operands are exact, so fp32's in every type
    torch.testing.assert_close(lse.cpu()[:, :, ~empty], lse_ref[:, :, ~empty].float(), rtol=1e-5, atol=2e-5)

    # the backwards from the same residuals, the forward's rounded exact ones
    o_in, lse_in = o_ref.to(dtype), lse_ref.float()
    args = [g[n] for n in ("q", "k", "v")] + [o_in.to(device), g["do"]]
    got = _hip.attention_bwd(*args, lse_in.to(device), code, scale, window, sinks)
    want = ref.backward(x["q"], x["k"], x["v"], o_in, x["do"], lse_in, mask, scale)
    for a, r, n in zip(got[:3], want[:3], ("dq", "dk", "dv")):
        check(a, r, dtype, n)
    torch.testing.assert_close(got[3].cpu().double(), want[3], rtol=1e-5, atol=1e-4)

    got = _hip.attention_bwdbwd(*args, g["ddq"], g["ddk"], g["ddv"], lse_in.to(device), code, scale, window=window,
                                sinks=sinks)
    want = ref.double_backward(x["q"], x["k"], x["v"], o_in, x["do"], x["ddq"], x["ddk"], x["ddv"], lse_in, mask, scale)
    for a, r, n in zip(got, want, ("dq2", "dk2", "dv2", "ddo")):
        check(a, r, dtype, n)


@pytest.mark.parametrize("case", CASES, ids=case_id)
def test_kernels(case, cuda_device):
    run_case(case, cuda_device)


@pytest.mark.parametrize("scale", [-0.11, 0.3, 0.125])
@pytest.mark.parametrize("case", [CASES[4], CASES[12], CASES[16], CASES[20], CASES[23]], ids=case_id)
def test_other_scales(case, scale, cuda_device):
    run_case(case, cuda_device, scale=scale, seed=11)


@pytest.mark.parametrize("variant", ["compiled", "pair"])
@pytest.mark.parametrize("case", [c for c in CASES if c[6] != FP32 and c[5] <= 128][1::2], ids=case_id)
def test_kernel_variants(case, variant, cuda_device, monkeypatch):
    """The kernels with one wave and with two per 32 rows, whichever the sizes would choose."""
    for name in ("FLASH_HOG_FWD", "FLASH_HOG_BWD", "FLASH_HOG_BWDQ", "FLASH_HOG_STAGE2"):
        monkeypatch.setenv(name, variant)
    run_case(case, cuda_device, seed=17)


@pytest.mark.parametrize("variant", ["few", "other"])
@pytest.mark.parametrize("case", [c for c in CASES if c[5] * (4 if c[6] == FP32 else 2) <= 256], ids=case_id)
def test_few_rows_kernels(case, variant, cuda_device, monkeypatch):
    """The kernels with one 32-row block a workgroup, and the others (any other name), at every case."""
    for name in ("FLASH_HOG_FWD", "FLASH_HOG_BWD", "FLASH_HOG_BWDQ", "FLASH_HOG_STAGE2"):
        monkeypatch.setenv(name, variant)
    run_case(case, cuda_device, seed=23)
