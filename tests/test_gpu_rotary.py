"""qk_norm_rotary and its derivatives against 64 bits (rotary_reference.py).

Tolerances. A stored value is off by half a step of its type, and by fp32's arithmetic before that. A row's
sums have at most 16 fused steps in a lane and 4 between lanes, a reciprocal root, and an angle that is
off by 2^-24 of a half turn plus two steps of sine and cosine; a result takes up to four such factors: 128
roundings of 2^-24 relative to the magnitudes that the formula adds (scales) hold all of it. A
weight's gradient adds rows one after the other: as many roundings more as there are rows, of the sum
of their magnitudes.
"""

from __future__ import annotations

import pytest
import torch

import rotary_reference as ref

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
STEPS = 128 * 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def near(got, want, scale, what):
    got = got.detach()
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    bound = half_step(got.dtype) * want.abs() + (1 + half_step(got.dtype)) * STEPS * scale + tiny
    error = (got.double().cpu() - want).abs()
    assert torch.isfinite(got).all(), what
    assert (error <= bound).all(), f"{what}: {float((error / bound).max()):.2f} times the bound"


def frequencies(rotated, device="cpu"):
    return (10000.0 ** (-torch.arange(0, rotated, 2, dtype=torch.float64) / rotated)).float().to(device) if rotated else None


def check(q, k, wq, wk, positions, freq, interleaved, eps, call, seed=0):
    """Forward, gradients and their derivatives of call(q, k, wq, wk) -> (q_out, k_out) against the oracle;
    q (T, N, H) after flattening; positions (T,) for it."""
    gen = torch.Generator().manual_seed(seed + 77)
    rand = lambda t: torch.randn(t.shape, generator=gen).to(t.dtype).to(t.device)
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (q, k, wq, wk)]
    cot = [rand(q).requires_grad_(), rand(k).requires_grad_()]
    out = call(*leaves)
    assert all(o.is_contiguous() and o.dtype == q.dtype for o in out)
    given = [t for t in leaves if t is not None]
    grads = torch.autograd.grad(out, given, cot, create_graph=True)
    tangents = [rand(t) for t in given]
    wanted = [*given, *cot] if eps is not None else cot
    second = torch.autograd.grad(grads, wanted, tangents)
    grads, tangents, second = list(grads), list(tangents), list(second)
    take = lambda values, present: [values.pop(0) if p else None for p in present]
    present = [True, True, wq is not None, wk is not None]
    grads, tangents = take(grads, present), take(tangents, present)
    second = take(second, [*(p and eps is not None for p in present), True, True])
    for i, n in enumerate("qk"):
        x, w = (q, k)[i], (wq, wk)[i]
        flat = lambda t: t.detach().flatten(0, -3).cpu() if t.ndim == 4 else t.detach().cpu()
        args = (flat(x), None if w is None else w.detach().cpu(), positions, None if freq is None else freq.cpu(),
                interleaved, eps, flat(cot[i]), flat(tangents[i]), tangents[2 + i])
        want = ref.derivatives(*args)
        scale = ref.scales(args[0], args[1], eps, args[6], args[7], None if w is None else tangents[2 + i])
        near(flat(out[i]), want["y"], scale["y"], n + " out")
        near(flat(grads[i]), want["dx"], scale["dx"], n + " gradient")
        near(flat(second[4 + i]), want["ddy"], scale["ddy"], n + " cotangent's")
        if eps is not None:
            near(flat(second[i]), want["dx2"], scale["dx2"], n + " second")
        if w is not None:
            rows = args[0].shape[0] * args[0].shape[1]
            for got, key in ((grads[2 + i], "dw"), (second[2 + i], "dw2")):
                near(got, want[key], (1 + rows / 128) * scale[key].sum(), f"{n} weight {key}")


# head_dim, rotated, interleaved, norm, weights
SHAPES = [(64, 64, False, True, True), (64, 32, True, True, True), (128, 128, False, True, True),
          (128, 128, True, True, True), (128, 96, False, True, True), (128, 48, False, True, True),
          (256, 256, False, True, True), (256, 64, True, True, True),
          (80, 80, False, True, True), (96, 32, False, True, True), (64, 0, False, True, True),
          (64, 64, False, False, False), (128, 64, True, False, False), (80, 20, False, False, False),
          (64, 64, False, True, False), (1, 0, False, True, True), (2, 2, False, True, True), (7, 6, True, True, True),
          (33, 10, False, True, True), (255, 254, True, True, True)]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_rows(shape, dtype, cuda_device):
    import flash_hog

    H, R, interleaved, norm, weights = shape
    print("[case] rows", shape, dtype, flush=True)
    gen = torch.Generator().manual_seed(H + R)
    T, N, Nk = 13, 6, 2
    make = lambda *s: (torch.randn(s, generator=gen) * torch.exp(torch.randn((*s[:-1], 1), generator=gen))).to(dtype).to(cuda_device)
    q, k = make(2, T, N, H), make(2, T, Nk, H)
    wq, wk = ((1 + 0.3 * torch.randn(H, generator=gen)).to(dtype).to(cuda_device) if weights else None for _ in range(2))
    freq, eps = frequencies(R, cuda_device), 1e-6 if norm else None
    check(q, k, wq, wk, torch.arange(T).repeat(2), freq, interleaved, eps,
          lambda *x: flash_hog.qk_norm_rotary(*x[:2], frequencies=freq, query_weight=x[2], key_weight=x[3], eps=eps,
                                              interleaved=interleaved))


# (batch, tokens): one token, tiles of 1, 4 and 16 tokens and their rests, more tiles than workgroups
@pytest.mark.parametrize("batch,tokens", [(1, 1), (3, 1), (1, 341), (2, 600), (1, 4099), (1, 16400), (3, 11111)])
def test_sizes(batch, tokens, cuda_device):
    import flash_hog

    print("[case] sizes", batch, tokens, flush=True)
    gen = torch.Generator().manual_seed(tokens)
    q, k = (torch.randn((batch, tokens, n, 64), generator=gen).to(BF16).to(cuda_device) for n in (3, 1))
    wq, wk = (torch.randn(64, generator=gen).to(cuda_device) for _ in range(2))  # fp32 beside bf16 rows
    freq = frequencies(64, cuda_device)
    check(q, k, wq, wk, torch.arange(tokens).repeat(batch), freq, False, 1e-5,
          lambda *x: flash_hog.qk_norm_rotary(*x[:2], frequencies=freq, query_weight=x[2], key_weight=x[3], eps=1e-5))


@pytest.mark.parametrize("kind", ["fused", "heads_first", "offset", "expanded", "columns"])
def test_layouts(kind, cuda_device):
    """Rows anywhere: views of a joint projection, heads before tokens, addresses of 2 bytes' alignment, one row
    for all tokens, columns at a stride."""
    import flash_hog

    print("[case] layout", kind, flush=True)
    B, T, N, Nk, H = 2, 37, 4, 2, 64
    gen = torch.Generator().manual_seed(3)
    rand = lambda *s: torch.randn(s, generator=gen).to(BF16).to(cuda_device)
    if kind == "fused":
        x = rand(B, T, N + 2 * Nk, H)
        q, k = x[:, :, :N], x[:, :, N:N + Nk]
    elif kind == "heads_first":
        q, k = rand(B, N, T, H).transpose(1, 2), rand(B, Nk, T, H).transpose(1, 2)
    elif kind == "offset":
        q, k = rand(B * T * N * H + 1)[1:].view(B, T, N, H), rand(B, T, Nk, H + 2)[..., 1:H + 1]
    elif kind == "expanded":
        q, k = rand(1, 1, N, H).expand(B, T, N, H), rand(B, T, 1, H).expand(B, T, Nk, H)
    else:
        q, k = rand(B, T, N, 2 * H)[..., ::2], rand(B, T, H, Nk).transpose(2, 3)
    wq, wk = rand(2 * H)[::2], rand(H + 1)[1:]
    freq = frequencies(64, cuda_device)
    call = lambda *x: flash_hog.qk_norm_rotary(*x[:2], frequencies=freq, query_weight=x[2], key_weight=x[3])
    check(q, k, wq, wk, torch.arange(T).repeat(B), freq, False, 1e-6, call)
    # a cotangent that is one number for all
    q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
    a = torch.autograd.grad(sum(o.float().sum() for o in call(q, k, wq, wk)), (q, k))
    out = call(q, k, wq, wk)
    b = torch.autograd.grad(out, (q, k), [torch.ones_like(o) for o in out])
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
@pytest.mark.parametrize("rows", [1, 3])
def test_positions(kind, rows, cuda_device):
    """Far, negative and repeated positions, for all sequences or for each."""
    import flash_hog

    print("[case] positions", kind, rows, flush=True)
    gen = torch.Generator().manual_seed(rows)
    T = 50
    most = 2 ** 31 - 1 if kind == torch.int32 else 2 ** 40
    positions = torch.randint(-1000, 200000, (rows, T), generator=gen).to(kind)
    positions[0, :4] = torch.tensor([most, -most, 0, 1 << 20], dtype=kind)
    q, k = (torch.randn((3, T, n, 64), generator=gen).to(cuda_device) for n in (2, 1))
    freq = frequencies(64, cuda_device)
    given = (positions if rows > 1 else positions[0]).to(cuda_device)
    out = flash_hog.qk_norm_rotary(q, k, given, frequencies=freq, eps=None)
    # An angle of A radians is a product of 64 bits, A 2^-53, reduced by another: A 2^-52 beside what STEPS holds.
    for x, y in zip((q, k), out):
        at = positions.expand(3, T).reshape(-1)
        want = ref.rotate(x.double().cpu().flatten(0, 1), at, freq.cpu(), False)
        scale = 2 * x.abs().amax(-1, keepdim=True).double().cpu().flatten(0, 1)
        near(y.flatten(0, 1), want, scale * (1 + at.abs()[:, None, None] * 2.0 ** -52 / STEPS), "rotation")


def test_cache_positions(cuda_device):
    """Positions from lengths and offsets: single tokens, chunks of unequal length, empty ones, rows before the
    first sequence and behind the last."""
    import flash_hog

    print("[case] cache positions", flush=True)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda_device)
    gen = torch.Generator().manual_seed(0)
    freq = frequencies(64, cuda_device)

    def run(total, positions, lengths, offsets):
        q, k = (torch.randn((total, n, 64), generator=gen).to(BF16).to(cuda_device) for n in (4, 2))
        got = flash_hog.qk_norm_rotary(q, k, frequencies=freq, lengths=lengths, query_offsets=offsets)
        want = flash_hog.qk_norm_rotary(q, k, torch.tensor(positions, device=cuda_device), frequencies=freq)
        assert all(torch.equal(a, b) for a, b in zip(got, want))

    run(3, [4, 99999, -1], i32(5, 100000, 0), None)
    run(1, [0], i32(1), None)
    run(8, [7, 8, 9, 0, 1, 100, 0, 0], i32(10, 5, 2, 101), i32(0, 3, 3, 5, 6))
    run(6, [0, 2, 3, 0, 0, 0], i32(4, 8), i32(1, 3, 3))


def test_no_rows(cuda_device):
    """No tokens: empty results, and weights' gradients of zero."""
    import flash_hog

    q, k = (torch.zeros((2, 0, n, 64), device=cuda_device, requires_grad=True) for n in (4, 2))
    wq, wk = (torch.ones(64, device=cuda_device, requires_grad=True) for _ in range(2))
    out = flash_hog.qk_norm_rotary(q, k, frequencies=frequencies(64, cuda_device), query_weight=wq, key_weight=wk)
    grads = torch.autograd.grad(out, (q, k, wq, wk), [torch.zeros_like(o) for o in out], create_graph=True)
    assert grads[0].shape == q.shape and torch.equal(grads[2], torch.zeros_like(wq))
    second = torch.autograd.grad(grads, (q, k, wq, wk), [torch.ones_like(g) for g in grads])
    assert torch.equal(second[3], torch.zeros_like(wk))


def test_special_rows(cuda_device):
    """Rows of zeros have finite derivatives; a NaN or an infinity stays in its row, and reaches the weights' gradients only."""
    import flash_hog

    print("[case] special rows", flush=True)
    gen = torch.Generator().manual_seed(0)
    q, k = (torch.randn((1, 9, n, 64), generator=gen).to(cuda_device) for n in (2, 1))
    freq = frequencies(64, cuda_device)
    q[0, 2] = 0
    clean = flash_hog.qk_norm_rotary(q, k, frequencies=freq)
    assert torch.equal(clean[0][0, 2], torch.zeros_like(q[0, 2]))
    q[0, 3, 0, 5], q[0, 4, 1, 6] = float("nan"), float("inf")
    leaf = q.clone().requires_grad_()
    out = flash_hog.qk_norm_rotary(leaf, k, frequencies=freq)
    grad, = torch.autograd.grad(out, leaf, [torch.ones_like(o) for o in out])
    bad = torch.zeros(9, 2, dtype=torch.bool, device=cuda_device)
    bad[3, 0] = bad[4, 1] = True
    assert torch.equal(out[0][0][~bad], clean[0][0][~bad]) and torch.isfinite(grad[0][~bad]).all()
    assert torch.isnan(out[0][0][3, 0]).all()


def test_differences(cuda_device):
    """The gradient against central differences of the kernel's own forward, step h = 2^-6: they leave
    h^2 / 6 of a third derivative of about one, and 2^-24 / h of the forward's rounding for each of the 2000
    values that are summed, with random signs."""
    import flash_hog

    gen = torch.Generator().manual_seed(1)
    q, k = (torch.randn((1, 8, n, 64), generator=gen).to(cuda_device) for n in (3, 1))
    w = [torch.rand(64, generator=gen).to(cuda_device) + 0.5 for _ in range(2)]
    freq = frequencies(32, cuda_device)
    cot = [torch.randn(t.shape, generator=gen).to(cuda_device) for t in (q, k)]

    def value(*x):
        out = flash_hog.qk_norm_rotary(*x[:2], frequencies=freq, query_weight=x[2], key_weight=x[3])
        return sum((o.double() * c.double()).sum() for o, c in zip(out, cot))

    leaves = [t.requires_grad_() for t in (q, k, *w)]
    grads = torch.autograd.grad(value(*leaves), leaves, create_graph=True)
    tangents = [torch.randn(t.shape, generator=gen).to(cuda_device) for t in leaves]
    slope = sum((g.double() * t.double()).sum() for g, t in zip(grads, tangents))
    second = torch.autograd.grad(grads, leaves, tangents)
    h = 2.0 ** -6
    moved = lambda s: [(t + s * h * d).detach().requires_grad_() for t, d in zip(leaves, tangents)]
    with torch.no_grad():
        difference = (value(*moved(1)) - value(*moved(-1))) / (2 * h)
    spread = float(sum((t.double() ** 2).sum() for t in tangents)) ** 0.5
    assert abs(float(difference - slope)) <= (h * h + 2000 ** 0.5 * 2.0 ** -24 / h) * spread * 4
    ahead, behind = (torch.autograd.grad(value(*x), x) for x in (moved(1), moved(-1)))
    for s, a, b in zip(second, ahead, behind):
        d = (a.double() - b.double()) / (2 * h)
        assert float((s.double() - d).norm()) <= (h * h * 4 + 2.0 ** -22 / h) * (float(d.norm()) + spread)


def test_repeats_and_graphs(cuda_device):
    """Repeated calls give the same bits, and so do replays of a captured training step, with other work between."""
    import flash_hog

    print("[case] graphs", flush=True)
    gen = torch.Generator().manual_seed(1)
    q, k = (torch.randn((2, 2100, n, 128), generator=gen).to(BF16).to(cuda_device) for n in (4, 2))
    w = [torch.rand(128, generator=gen).to(BF16).to(cuda_device) for _ in range(2)]
    freq = frequencies(128, cuda_device)
    cot = [torch.randn(t.shape, generator=gen).to(BF16).to(cuda_device) for t in (q, k)]
    tangents = [torch.randn(t.shape, generator=gen).to(BF16).to(cuda_device) for t in (q, k, *w)]

    def step(*x):
        leaves = [t.detach().requires_grad_() for t in x]
        out = flash_hog.qk_norm_rotary(*leaves[:2], frequencies=freq, query_weight=leaves[2], key_weight=leaves[3])
        grads = torch.autograd.grad(out, leaves, cot, create_graph=True)
        return [t.detach() for t in (*out, *grads, *torch.autograd.grad(grads, leaves, tangents))]

    want = step(q, k, *w)
    assert all(torch.equal(a, b) for a, b in zip(want, step(q, k, *w)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert all(torch.equal(a, b) for a, b in zip(want, step(q, k, *w)))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(q, k, *w)
    for i in range(3):
        q.copy_(torch.randn(q.shape, generator=gen).to(BF16))
        graph.replay()
        torch.cuda.synchronize()
        want = step(q, k, *w)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), f"replay {i}"


def test_through_attention(cuda_device):
    """A Hessian-vector product through norms, rotation and attention, as a model has them, against 64 bits."""
    import flash_hog
    from oracle import autodiff  # noqa: F401  (the oracle package is importable)

    print("[case] through attention", flush=True)
    gen = torch.Generator().manual_seed(2)
    B, T, N, Nk, H = 1, 65, 4, 2, 64
    x = [torch.randn(s, generator=gen).to(cuda_device) for s in ((B, T, N, H), (B, T, Nk, H), (B, T, Nk, H), (H,), (H,))]
    freq = frequencies(64, cuda_device)
    cot = torch.randn((B, T, N, H), generator=gen).to(cuda_device)
    tangents = [torch.randn(t.shape, generator=gen).to(cuda_device) for t in x]

    def attend(q, k, v):
        k, v = (t.repeat_interleave(N // Nk, 2) for t in (k, v))
        s = torch.einsum("btnh,bsnh->bnts", q, k) * H ** -0.5
        s = s.masked_fill(torch.arange(T)[:, None] < torch.arange(T), float("-inf"))
        return torch.einsum("bnts,bsnh->btnh", torch.softmax(s, -1), v)

    def products(leaves, call, cot, tangents):
        grads = torch.autograd.grad(call(*leaves), leaves, cot, create_graph=True)
        return [*(g.detach() for g in grads), *torch.autograd.grad(grads, leaves, tangents)]

    def ours(q, k, v, wq, wk):
        q, k = flash_hog.qk_norm_rotary(q, k, frequencies=freq, query_weight=wq, key_weight=wk)
        return flash_hog.dot_product_attention(q, k, v, is_causal=True)

    def plain(q, k, v, wq, wk):
        q, k = (ref.apply(t[0], w, torch.arange(T), freq.cpu(), False, 1e-6)[None] for t, w in ((q, wq), (k, wk)))
        return attend(q, k, v)

    got = products([t.requires_grad_() for t in x], ours, cot, tangents)
    double = lambda ts: [t.detach().double().cpu() for t in ts]
    want = products([t.requires_grad_() for t in double(x)], plain, double([cot])[0], double(tangents))
    for a, b in zip(got, want):  # (fp32 attention's own bound in test_gpu_parity.py is 2e-5 of the largest value)
        assert float((a.double().cpu() - b).abs().max()) <= 4e-5 * float(b.abs().max())


@pytest.mark.parametrize("extension", [True, False])
@pytest.mark.parametrize("norm", [True, False])
def test_parts_of_a_graph(norm, extension, cuda_device, monkeypatch):
    """One result used, one leaf asked for, one gradient differentiated: as with zeros in the other places."""
    import flash_hog
    from flash_hog import _hip

    if not extension:
        monkeypatch.setattr(_hip, "torch_ext", lambda: None)
    gen = torch.Generator().manual_seed(3)
    rand = lambda *shape: torch.randn(shape, generator=gen).to(cuda_device)
    q, k, wq, wk = rand(2, 9, 4, 64), rand(2, 9, 2, 64), rand(64), rand(64)
    cq, ck, freq = rand(2, 9, 4, 64), rand(2, 9, 2, 64), frequencies(64, cuda_device)
    leaves = [t.requires_grad_() for t in ((q, k, wq, wk) if norm else (q, k))]
    weights = dict(query_weight=wq, key_weight=wk) if norm else dict(eps=None)
    call = lambda q=q, k=k: flash_hog.qk_norm_rotary(q, k, frequencies=freq, **weights)
    full = torch.autograd.grad(call(), leaves, (cq, torch.zeros_like(ck)))
    part = torch.autograd.grad(call()[0], leaves, cq, allow_unused=True)
    for a, b in zip(full, part):
        assert torch.equal(a, b) if b is not None else not a.any()
    both = torch.autograd.grad(call(), leaves, (cq, ck))
    for leaf, want in zip(leaves, both):
        assert torch.equal(torch.autograd.grad(call(), leaf, (cq, ck))[0], want)
    # q alone needs a gradient; k is a leaf that needs none
    assert torch.equal(torch.autograd.grad(call(k=k.detach()), q, (cq, ck))[0], both[0])
    for i, leaf in enumerate(leaves):
        c = [cq.clone().requires_grad_(), ck.clone().requires_grad_()]
        wanted = (*leaves, *c) if norm else c
        tangent = rand(*leaf.shape)
        grads = torch.autograd.grad(call(), leaves, c, create_graph=True)
        one = torch.autograd.grad(grads[i], wanted, tangent, allow_unused=True, retain_graph=True)
        zeros = [tangent if j == i else torch.zeros_like(g) for j, g in enumerate(grads)]
        for a, b in zip(torch.autograd.grad(grads, wanted, zeros), one):
            assert torch.equal(a, b) if b is not None else not a.any()


def test_transforms(cuda_device):
    """torch.func.grad, vmap (also of weights), and jvp, which is refused."""
    import flash_hog

    print("[case] transforms", flush=True)
    gen = torch.Generator().manual_seed(4)
    q, k = (torch.randn((3, 2, 9, n, 64), generator=gen).to(cuda_device) for n in (2, 1))
    wq, wk = (torch.rand((3, 64), generator=gen).to(cuda_device) for _ in range(2))
    freq = frequencies(64, cuda_device)

    def loss(q, k, wq, wk):
        a, b = flash_hog.qk_norm_rotary(q, k, frequencies=freq, query_weight=wq, key_weight=wk)
        return (a ** 2).sum() + (b ** 3).sum()

    def product(q, k, wq, wk):
        grads = torch.func.grad(loss, argnums=(0, 1, 2, 3))(q, k, wq, wk)
        return sum((g * g.detach()).sum() for g in grads)

    second = torch.func.grad(product, argnums=(0, 2))
    got = torch.func.vmap(second)(q, k, wq, wk)
    for i in range(3):
        leaves = [t[i].detach().requires_grad_() for t in (q, k, wq, wk)]
        grads = torch.autograd.grad(loss(*leaves), leaves, create_graph=True)
        want = torch.autograd.grad(sum((g * g.detach()).sum() for g in grads), (leaves[0], leaves[2]))
        for a, b in zip(got, want):
            assert torch.equal(a[i], b)
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(lambda t: loss(t, k[0], wq[0], wk[0]), (q[0],), (q[0],))
    with torch.autograd.forward_ad.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        loss(torch.autograd.forward_ad.make_dual(q[0], q[0]), k[0], wq[0], wk[0])


def test_compile(cuda_device):
    import flash_hog

    print("[case] compile", flush=True)
    gen = torch.Generator().manual_seed(5)
    q, k = (torch.randn((2, 9, n, 64), generator=gen).to(cuda_device).requires_grad_() for n in (2, 1))
    w = torch.rand(64, generator=gen).to(cuda_device).requires_grad_()
    freq = frequencies(64, cuda_device)

    def loss(q, k, w):
        a, b = flash_hog.qk_norm_rotary(q, k, frequencies=freq, query_weight=w, key_weight=w)
        return (a * b.sum(2, keepdim=True)).sum()

    want = torch.autograd.grad(loss(q, k, w), (q, k, w))
    got = torch.autograd.grad(torch.compile(loss, backend="aot_eager")(q, k, w), (q, k, w))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("extension", [True, False])
def test_third_derivative_raises(extension, cuda_device, monkeypatch):
    import flash_hog
    from flash_hog import _hip

    if not extension:
        monkeypatch.setattr(_hip, "torch_ext", lambda: None)

    q, k = (torch.randn((1, 5, n, 64), device=cuda_device, requires_grad=True) for n in (2, 1))
    out = flash_hog.qk_norm_rotary(q, k)
    first = torch.autograd.grad(sum((o ** 2).sum() for o in out), (q, k), create_graph=True)
    second = torch.autograd.grad(sum((g ** 2).sum() for g in first), (q, k), create_graph=True)
    with pytest.raises(RuntimeError):
        sum((s ** 2).sum() for s in second).backward()


def test_python_wrappers_agree(cuda_device, monkeypatch):
    """The calls through ctypes give the bits of those through the extension, if it is there."""
    import flash_hog
    from flash_hog import _hip

    gen = torch.Generator().manual_seed(6)
    q, k = (torch.randn((1, 77, n, 128), generator=gen).to(FP16).to(cuda_device) for n in (4, 2))
    w = torch.rand(128, generator=gen).to(FP16).to(cuda_device)
    freq = frequencies(64, cuda_device)

    def run():
        leaves = [t.detach().requires_grad_() for t in (q, k, w)]
        out = flash_hog.qk_norm_rotary(*leaves[:2], frequencies=freq, query_weight=leaves[2], interleaved=True)
        grads = torch.autograd.grad(out, leaves, [torch.ones_like(o) for o in out], create_graph=True)
        return [*out, *grads, *torch.autograd.grad(grads, leaves, [torch.ones_like(g) for g in grads])]

    assert _hip.torch_ext() is not None
    a = run()
    monkeypatch.setattr(_hip, "torch_ext", lambda: None)
    assert all(torch.equal(x, y) for x, y in zip(a, run()))


@pytest.mark.parametrize("extension", [True, False])
def test_refusals(extension, cuda_device, monkeypatch):
    """Both front doors say the same."""
    import flash_hog
    from flash_hog import _hip

    if not extension:
        monkeypatch.setattr(_hip, "torch_ext", lambda: None)
    q, k = (torch.zeros((2, 5, n, 64), dtype=BF16, device=cuda_device) for n in (4, 2))
    w, freq = torch.ones(64, dtype=BF16, device=cuda_device), frequencies(64, cuda_device)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=cuda_device)
    call = flash_hog.qk_norm_rotary
    for bad, match in ((lambda: call(q, k[:1]), "of the same tokens and head_dim"), (lambda: call(q, k[..., :32]), "of the same tokens"),
                       (lambda: call(q, k.float()), "key has dtype"), (lambda: call(q, k.cpu()), "must be on a GPU device"),
                       (lambda: call(q.double(), k.double()), "unsupported dtype"),
                       (lambda: call(q, k, query_weight=w[:32]), "query_weight has shape"),
                       (lambda: call(q, k, query_weight=w, key_weight=w.float()), "key_weight has dtype"),
                       (lambda: call(q, k, query_weight=w.half()), "weights must be of"),
                       (lambda: call(q, k, query_weight=w, eps=None), "weights need norms"),
                       (lambda: call(q, k, frequencies=freq.double()), "frequencies must be"),
                       (lambda: call(q, k, frequencies=torch.cat([freq, freq])), "frequencies must be"),
                       (lambda: call(q, k, i32(5).float()), "positions has dtype"), (lambda: call(q, k, i32(2, 4)), "positions has shape"),
                       (lambda: call(q, k, i32(1, 5)), "positions has shape"), (lambda: call(q[0], k[0], i32(5), lengths=i32(5)), "exclude each other"),
                       (lambda: call(q[0], k[0], lengths=i32(4)), "lengths has shape"),
                       (lambda: call(q[0], k[0], lengths=i32(4), query_offsets=i32(4)), "query_offsets has shape"),
                       (lambda: call(q[0], k[0], query_offsets=i32(4)), "query_offsets needs lengths"),
                       (lambda: call(q[0], k[0], lengths=i32(5).long()), "lengths has dtype"),
                       (lambda: call(q, k, lengths=i32(10)), "packed tokens")):
        with pytest.raises(ValueError, match=match):
            bad()
    for bad, match in ((lambda: call(q, k, eps=-1.0), "eps must be finite"),
                       (lambda: call(torch.zeros((1, 1, 1, 300), device=cuda_device), torch.zeros((1, 1, 1, 300), device=cuda_device)),
                        "head_dim must be 1 to 256")):
        with pytest.raises(_hip.FlashHogError, match=match):
            bad()


def test_in_place_changes_are_noticed(cuda_device):
    """A row or a position that changed after the forward makes its backward raise."""
    import flash_hog

    for which in range(3):
        q, k = (torch.randn((1, 5, n, 64), device=cuda_device) for n in (2, 1))
        w, positions = torch.ones(64, device=cuda_device, requires_grad=True), torch.arange(5, device=cuda_device)
        out = flash_hog.qk_norm_rotary(q, k, positions, frequencies=frequencies(64, cuda_device), query_weight=w)
        (q, k, positions)[which].add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out[0].sum().backward()


@pytest.mark.parametrize("eps", [1e-6, None])
def test_vmap_of_nothing(eps, cuda_device):
    """No elements: empty results of the elements' shapes, of the derivatives as well."""
    import flash_hog

    print("[case] vmap of nothing", flush=True)
    q, k = (torch.zeros((5, 0, 3, n, 64), device=cuda_device) for n in (4, 2))
    freq = frequencies(64, cuda_device)
    call = lambda a, b: flash_hog.qk_norm_rotary(a, b, frequencies=freq, eps=eps)
    out = torch.func.vmap(call, in_dims=1)(q, k)
    assert out[0].shape == (0, 5, 3, 4, 64) and out[1].shape == (0, 5, 3, 2, 64)
    squares = lambda x, y: (x ** 2).sum() + (y ** 2).sum()  # (0 + a batch of no numbers is an error of torch's own)
    loss = lambda a, b: squares(*call(a, b))
    second = torch.func.grad(lambda a, b: squares(*torch.func.grad(loss, (0, 1))(a, b)), (0, 1))
    for run in (torch.func.grad(loss, (0, 1)), second):
        grads = torch.func.vmap(run, in_dims=(1, 1))(q, k)
        assert grads[0].shape == (0, 5, 3, 4, 64) and grads[1].shape == (0, 5, 3, 2, 64)
