"""Windowed attention through dot_product_attention: both derivatives against the closed forms and
against differences, broadcast and strided inputs, graphs, streams, repeats, long sequences.

Tolerances: the front-end's parity bar (helpers.TOL on the largest error over the largest
entry) where outputs of one kernel feed the next. Differences, fp32: a gradient's 2-norm error is at
most 2e-5 of its norm (test_gpu_window.py), its product with a direction d off by at most that
times |g| |d|; central differences in 64 bits with a step of 1e-3 add the third derivative's
1e-6 / 6, relative to terms of the same size: 4e-5 |g| |d| together.
"""

from __future__ import annotations

import pytest
import torch

import window_reference as ref
from helpers import DEGENERATE_FLOOR, TOL, default_scale, make_inputs, rel_err

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
NAMES = ("q", "k", "v", "do")


def bwd_bwd(x, is_causal=True, **kw):
    """out, (dq, dk, dv), (dq2, dk2, dv2, ddo) by autograd."""
    import flash_hog

    leaves = [x[n].detach().requires_grad_(True) for n in NAMES]
    out = flash_hog.dot_product_attention(*leaves[:3], is_causal=is_causal, **kw)
    g = torch.autograd.grad(out, leaves[:3], leaves[3], create_graph=True)
    h = torch.autograd.grad(g, leaves, (x["ddq"], x["ddk"], x["ddv"]))
    return [out.detach(), *(t.detach() for t in g), *h]


def reference(x, mask, scale):
    c = {n: t.double().cpu() for n, t in x.items()}
    o, lse = ref.forward(c["q"], c["k"], c["v"], mask, scale)
    g = ref.backward(c["q"], c["k"], c["v"], o, c["do"], lse, mask, scale)[:3]
    h = ref.double_backward(c["q"], c["k"], c["v"], o, c["do"], c["ddq"], c["ddk"], c["ddv"], lse, mask, scale)
    return [o, *g, *h]


def compare(got, want, dtype, what):
    for a, r, n in zip(got, want, ("o", "dq", "dk", "dv", "dq2", "dk2", "dv2", "ddo")):
        err = rel_err(a, r, DEGENERATE_FLOOR)
        assert err < TOL[dtype], f"{what} {n}: {err:.2e}"


# (batch, n_q, n_k, heads, kv_heads, head_dim, dtype, alignment, window, sinks)
CASES = [
    (2, 192, 192, 4, 2, 64, BF16, "top_left", 50, 3),
    (1, 100, 230, 4, 4, 64, FP16, "bottom_right", 33, 0),
    (1, 230, 100, 2, 1, 64, BF16, "bottom_right", 20, 2),
    (1, 60, 130, 2, 2, 64, BF16, "top_left", 16, 1),  # keys behind the last query
    (1, 300, 300, 2, 2, 80, BF16, "top_left", 40, 5),
    (1, 150, 150, 2, 1, 40, FP32, "top_left", 31, 2),
    (1, 150, 150, 2, 1, 200, FP16, "top_left", 31, 2),
    (1, 150, 150, 2, 1, 96, FP32, "top_left", 64, 0),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[1]}x{c[2]}_d{c[5]}_{str(c[6])[6:]}_{c[7]}_w{c[8]}_s{c[9]}")
def test_derivatives(case, cuda_device):
    B, nq, nk, H, Hk, D, dtype, alignment, window, sinks = case
    print("[case] frontend", case, flush=True)
    x = make_inputs(B, nq, nk, H, D, dtype, seed=2, kv_heads=Hk)
    got = bwd_bwd({n: t.to(cuda_device) for n, t in x.items()}, causal_alignment=alignment, window=window, sinks=sinks)
    compare(got, reference(x, ref.visible(nq, nk, alignment, window, sinks), default_scale(D)), dtype, case)


def test_random_cases(cuda_device):
    """Sizes, windows and sinks drawn at random."""
    gen = torch.Generator().manual_seed(99)
    draw = lambda *options: options[int(torch.randint(len(options), (1,), generator=gen))]
    number = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=gen))
    for i in range(40):
        Hk = draw(1, 2, 3)
        case = (number(1, 3), number(1, 400), number(1, 400), Hk * draw(1, 2, 5), Hk, draw(64, 64, 128, 256),
                draw(BF16, FP16, FP32), draw("top_left", "bottom_right"), number(1, 300), draw(0, 0, 1, 4, number(1, 200)))
        B, nq, nk, H, Hk, D, dtype, alignment, window, sinks = case
        if dtype == FP32 and D == 256:
            continue
        print("[case] random", i, case, flush=True)
        x = make_inputs(B, nq, nk, H, D, dtype, seed=200 + i, kv_heads=Hk)
        got = bwd_bwd({n: t.to(cuda_device) for n, t in x.items()}, causal_alignment=alignment, window=window,
                      sinks=sinks)
        compare(got, reference(x, ref.visible(nq, nk, alignment, window, sinks), default_scale(D)), dtype, case)


def test_differences(cuda_device):
    """Gradients and second derivatives along directions, against central differences of the 64-bit
    forward and backward."""
    print("[case] differences", flush=True)
    nq = nk = 90
    window, sinks, scale, step = 20, 3, default_scale(64), 1e-3
    x = make_inputs(1, nq, nk, 2, 64, FP32, seed=31, kv_heads=1)
    c = {n: t.double() for n, t in x.items()}
    mask = ref.visible(nq, nk, "top_left", window, sinks)
    got = bwd_bwd({n: t.to(cuda_device) for n, t in x.items()}, window=window, sinks=sinks)
    _, dq, dk, dv, dq2, dk2, dv2, ddo = (t.double().cpu() for t in got)
    tangents = make_inputs(1, nq, nk, 2, 64, FP32, seed=77, kv_heads=1)

    def loss(y):
        return (ref.forward(y["q"], y["k"], y["v"], mask, scale)[0] * y["do"]).sum()

    def grad_loss(y):  # <gradient, (ddq, ddk, ddv)>
        o, lse = ref.forward(y["q"], y["k"], y["v"], mask, scale)
        g = ref.backward(y["q"], y["k"], y["v"], o, y["do"], lse, mask, scale)[:3]
        return sum((a * y[n]).sum() for a, n in zip(g, ("ddq", "ddk", "ddv")))

    for f, grads in ((loss, {"q": dq, "k": dk, "v": dv}), (grad_loss, {"q": dq2, "k": dk2, "v": dv2, "do": ddo})):
        for name, g in grads.items():
            d = tangents[name].double()
            d = d / d.norm()
            ends = [f({**c, name: c[name] + s * step * d}) for s in (1, -1)]
            want = (ends[0] - ends[1]) / (2 * step)
            assert abs((g * d).sum() - want) <= 4e-5 * g.norm(), (f.__name__, name)


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "f32"])
def test_window_that_hides_nothing_is_causal(dtype, cuda_device):
    print("[case] wide windows", dtype, flush=True)
    x = {n: t.to(cuda_device) for n, t in make_inputs(2, 130, 200, 4, 64, dtype, seed=5, kv_heads=2).items()}
    for alignment, window, sinks in (("bottom_right", 200, 0), ("bottom_right", 10**12, 10**12), ("top_left", 130, 3),
                                     ("bottom_right", 150, 50), ("top_left", 1, 200)):
        want = bwd_bwd(x, causal_alignment=alignment)
        got = bwd_bwd(x, causal_alignment=alignment, window=window, sinks=sinks)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), (alignment, window, sinks)


PATHS = [CASES[0], CASES[2], CASES[4], (1, 900, 900, 2, 1, 128, FP16, "top_left", 32, 40)]


@pytest.mark.parametrize("case", PATHS, ids=lambda c: f"{c[1]}x{c[2]}_d{c[5]}")
def test_all_paths_give_the_same_bits(case, cuda_device, monkeypatch):
    """The C++ autograd Functions, the Python ones, and those over the Python wrappers."""
    from flash_hog import _hip
    from flash_hog.torch import attention as att

    B, nq, nk, H, Hk, D, dtype, alignment, window, sinks = case
    print("[case] paths", case, flush=True)
    x = {n: t.to(cuda_device) for n, t in make_inputs(B, nq, nk, H, D, dtype, seed=12, kv_heads=Hk).items()}
    kw = dict(causal_alignment=alignment, window=window, sinks=sinks)
    want = bwd_bwd(x, **kw)
    monkeypatch.setattr(att, "_native_path", lambda *t: None)
    assert all(torch.equal(a, b) for a, b in zip(bwd_bwd(x, **kw), want))
    monkeypatch.setattr(_hip, "torch_ext", lambda: None)
    assert all(torch.equal(a, b) for a, b in zip(bwd_bwd(x, **kw), want))


def test_strided_and_broadcast_inputs(cuda_device):
    """Heads-first storage, a slice, a step, keys broadcast over the batch and heads: the same
    values as from contiguous copies, and gradients summed over what was broadcast."""
    import flash_hog

    print("[case] strides", flush=True)
    kw = dict(is_causal=True, window=17, sinks=2)
    x = make_inputs(2, 80, 80, 4, 64, BF16, seed=6, kv_heads=2)
    q = torch.randn(2, 4, 160, 64, device=cuda_device).to(BF16)[:, :, ::2].transpose(1, 2)  # (2, 80, 4, 64)
    k = x["k"][:1].to(cuda_device)
    v = x["v"][:, :, :1].to(cuda_device)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    assert not leaves[0].is_contiguous()
    args = [leaves[0], leaves[1].expand(2, -1, -1, -1), leaves[2].expand(-1, -1, 2, -1)]
    out = flash_hog.dot_product_attention(*args, **kw)
    cot = x["do"].to(cuda_device).transpose(1, 2).contiguous().transpose(1, 2)
    g = torch.autograd.grad(out, leaves, cot)
    full = [t.detach().contiguous().requires_grad_(True) for t in args]
    out2 = flash_hog.dot_product_attention(*full, **kw)
    g2 = torch.autograd.grad(out2, full, cot.contiguous())
    assert torch.equal(out, out2) and torch.equal(g[0], g2[0])
    # (the sum of two bf16 values, rounded once by torch)
    assert torch.equal(g[1], g2[1].sum(0, keepdim=True)) and torch.equal(g[2], g2[2].sum(2, keepdim=True))
    unbatched = flash_hog.dot_product_attention(*(t[0].detach() for t in full), **kw)
    with torch.no_grad():
        assert torch.equal(unbatched, flash_hog.dot_product_attention(*(t[:1] for t in full), **kw)[0])


def test_vmap_and_compile(cuda_device):
    import flash_hog

    print("[case] vmap, compile", flush=True)
    x = {n: t.to(cuda_device) for n, t in make_inputs(3, 70, 70, 4, 64, BF16, seed=8, kv_heads=2).items()}

    def attn(q, k, v):
        return flash_hog.dot_product_attention(q, k, v, is_causal=True, window=20, sinks=2)

    want = attn(x["q"], x["k"], x["v"])
    assert torch.equal(torch.func.vmap(attn)(x["q"], x["k"], x["v"]), want)
    loss = lambda q, k, v, do: (attn(q, k, v) * do).sum()
    got = torch.func.vmap(torch.func.grad(loss, argnums=(0, 1, 2)))(x["q"], x["k"], x["v"], x["do"])
    leaves = [x[n].detach().requires_grad_(True) for n in "qkv"]
    grads = torch.autograd.grad(attn(*leaves), leaves, x["do"])
    assert all(torch.equal(a, b) for a, b in zip(got, grads))
    compiled = torch.compile(attn, backend="aot_eager", fullgraph=True)
    assert torch.equal(compiled(x["q"], x["k"], x["v"]), want)
    out = compiled(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, x["do"]), grads))


# many queries behind each sink: several parts to join, in one launch and apart
REPEATED = [(1, 3000, 3000, 4, 2, 64, BF16, "top_left", 64, 5), (2, 4001, 4001, 16, 4, 128, FP16, "top_left", 512, 4),
            (1, 700, 700, 2, 1, 64, FP32, "top_left", 40, 33)]


@pytest.mark.parametrize("case", REPEATED, ids=lambda c: f"b{c[0]}_n{c[1]}_d{c[5]}_{str(c[6])[6:]}")
def test_repeats_and_streams(case, cuda_device):
    """Repeated calls, and two at once on streams of their own, give the same bits."""
    B, nq, nk, H, Hk, D, dtype, alignment, window, sinks = case
    print("[case] repeats", case, flush=True)
    xs = [{n: t.to(cuda_device) for n, t in make_inputs(B, nq, nk, H, D, dtype, seed=s, kv_heads=Hk).items()}
          for s in (1, 40)]
    kw = dict(causal_alignment=alignment, window=window, sinks=sinks)
    want = [bwd_bwd(x, **kw) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(3):
        got = []
        for x, stream in zip(xs, streams):
            with torch.cuda.stream(stream):
                got.append(bwd_bwd(x, **kw))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(s, t) for s, t in zip(a, b))


@pytest.mark.parametrize("shape", [(1, 500, 500, 4, 2, 64, "top_left"), (2, 200, 320, 4, 4, 64, "bottom_right"),
                                   (1, 3000, 3000, 2, 2, 128, "top_left")], ids=["n500", "ragged", "n3000"])
def test_graph_replays_match_eager(shape, cuda_device):
    """The whole double backward, sinks' workspace and join included, captured once and replayed
    with other values and eager calls between."""
    B, nq, nk, H, Hk, D, alignment = shape
    print("[case] graph", shape, flush=True)
    kw = dict(causal_alignment=alignment, window=40, sinks=5)
    draw = lambda seed: {n: t.to(cuda_device) for n, t in make_inputs(B, nq, nk, H, D, BF16, seed=seed, kv_heads=Hk).items()}
    static = draw(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            bwd_bwd(static, **kw)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs of the same call: workspaces of their own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, bwd_bwd(static, **kw)))
    torch.cuda.synchronize()
    for replay in range(4):
        new = draw(100 + replay)
        for n in static:
            static[n].copy_(new[n])
        eager = bwd_bwd(new, **kw)
        torch.cuda.synchronize()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, outputs in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outputs, eager)), replay


def test_long_sequence_beyond_32_bit_offsets(cuda_device):
    """Tensors of more than 2^31 elements and 2^32 bytes: the last queries give the bits of a short
    call on the keys that they see."""
    from flash_hog import _hip

    n, heads, d, window = (1 << 18) + 70, 64, 128, 48
    print("[case] long", n, flush=True)
    tail = 512  # the last queries, whose windows lie in the last tail + 64 keys
    q, k, v, do, ddq, ddk, ddv = (torch.zeros((1, n, heads, d), dtype=BF16, device=cuda_device) for _ in range(7))
    gen = torch.Generator(device=cuda_device).manual_seed(1)
    xs = (q, k, v, do, ddq, ddk, ddv)
    assert q.numel() > 1 << 31
    for t in xs:
        t[:, -(tail + 64):].normal_(generator=gen)
    short = [t[:, -(tail + 64):].clone() for t in xs]
    scale = d ** -0.5
    o, lse = _hip.attention_fwd(q, k, v, 1, scale, window)
    o_s, lse_s = _hip.attention_fwd(*short[:3], 1, scale, window)
    def same(a, b, dim=1):
        a, b = a.narrow(dim, a.shape[dim] - 256, 256), b.narrow(dim, b.shape[dim] - 256, 256)
        torch.testing.assert_close(a.double(), b.double(), rtol=0, atol=2 * TOL[BF16] * b.double().abs().max().item())
    same(o, o_s)
    same(lse, lse_s, 2)
    g = _hip.attention_bwd(q, k, v, o, do, lse, 1, scale, window)
    g_s = _hip.attention_bwd(*short[:3], o_s, short[3], lse_s, 1, scale, window)
    for a, b in zip(g[:3], g_s[:3]):
        same(a, b)
    del g
    h = _hip.attention_bwdbwd(q, k, v, o, do, ddq, ddk, ddv, lse, 1, scale, window=window)
    h_s = _hip.attention_bwdbwd(*short[:3], o_s, *short[3:], lse_s, 1, scale, window=window)
    for a, b in zip(h, h_s):
        same(a, b)
