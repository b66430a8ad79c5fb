"""Which windowed calls give the sinks' further queries a launch of their own, and where a window is
none: the rules behind test_gpu_window_apart.py and dot_product_attention."""

from __future__ import annotations

import torch

from flash_hog.torch.attention import _effective_window
from test_gpu_window_apart import CASES
from test_window_paged_rules import rules, sink_chunks  # noqa: F401 (a fixture)
from window_reference import visible


def test_cases_go_apart(rules):  # noqa: F811
    """Every case of test_gpu_window_apart.py has its chunks apart, several of them, and all kernel
    instances of that launch are reached."""
    for B, nq, nk, H, Hk, D, dtype, alignment, window, sinks in CASES:
        coff = nk - nq if alignment == "bottom_right" else 0
        apart, step, count = sink_chunks(rules, nq, nk, coff, window, sinks, D * dtype.itemsize, B * H, B * Hk)
        assert apart and count >= 2, (B, nq, nk, H, D)
    assert {(c[5], c[6]) for c in CASES} == {(64, torch.bfloat16), (64, torch.float16), (128, torch.bfloat16),
                                             (128, torch.float16), (64, torch.float32)}
    assert any(c[9] > 64 for c in CASES) and any(c[9] < 32 for c in CASES)


def test_effective_window_is_none_exactly_where_it_hides_nothing():
    for n_q in (1, 5, 12):
        for n_k in (1, 4, 12):
            for alignment in ("top_left", "bottom_right"):
                for window in (1, 3, 8, 11, 12, 13, 50):
                    for sinks in (0, 1, 3, 12, 40):
                        same = torch.equal(visible(n_q, n_k, alignment, window, sinks),
                                           visible(n_q, n_k, alignment, 0, 0))
                        got = _effective_window(n_q, n_k, alignment, window, sinks)
                        assert (got == (0, 0)) == same, (n_q, n_k, alignment, window, sinks)
