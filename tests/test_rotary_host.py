"""qk_norm_rotary without a GPU: what the C ABI and the front-end refuse, shapes on meta tensors, and
the oracle's derivatives against differences."""

from __future__ import annotations

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import flash_hog
import rotary_reference as ref
from flash_hog import _hip

BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def lib():
    return _hip.lib()


def shape(**kwargs):
    s = _hip.Rotary(batch=2, tokens=5, heads=4, kv_heads=2, head_dim=64, rotated=64, dtype=2, weight_dtype=2,
                    interleaved=0, norm=1, eps=1e-6, frequencies=16)
    s.q_stride[:] = [5 * 4 * 64, 4 * 64, 64]
    s.k_stride[:] = [5 * 2 * 64, 2 * 64, 64]
    for name, value in kwargs.items():
        setattr(s, name, value)
    return s


CALLS = {"fhog_qk_norm_rotary_fwd": 6, "fhog_qk_norm_rotary_bwd": 11, "fhog_qk_norm_rotary_bwdbwd": 17}
REFUSALS = [
    (dict(batch=-1), 1, "sizes must not be negative"),
    (dict(heads=0), 1, "sizes must be >= 1"),
    (dict(dtype=3, weight_dtype=3), 2, "dtype must be bf16, fp16 or fp32"),
    (dict(weight_dtype=1), 2, "weights must be of dtype"),
    (dict(head_dim=0, rotated=0), 2, "head_dim must be 1 to 256"),
    (dict(head_dim=257), 2, "head_dim must be 1 to 256"),
    (dict(rotated=66), 1, "rotated must be even, 0 to head_dim"),
    (dict(rotated=31), 1, "rotated must be even"),
    (dict(rotated=-2), 1, "rotated must be even"),
    (dict(eps=-1.0), 1, "eps must be finite and >= 0"),
    (dict(eps=float("nan")), 1, "eps must be finite"),
    (dict(eps=float("inf")), 1, "eps must be finite"),
    (dict(frequencies=None), 1, "frequencies is null"),
    (dict(positions=16, position_bytes=2, position_rows=1), 1, "elements of 4 or 8 bytes"),
    (dict(positions=12, position_bytes=8, position_rows=1), 1, "aligned elements"),
    (dict(positions=16, position_bytes=4, position_rows=3), 1, "1 or batch rows"),
    (dict(positions=16, position_bytes=4, position_rows=1, lengths=16), 1, "exclude each other"),
    (dict(lengths=16, sequences=5), 1, "packed tokens have batch 1"),
    (dict(batch=1, lengths=16, sequences=4), 1, "without query_offsets there is one row a sequence"),
    (dict(batch=1, lengths=16, query_offsets=16, sequences=0), 1, "rows without a sequence"),
    (dict(query_offsets=16), 1, "query_offsets needs lengths"),
    (dict(batch=1 << 20, tokens=1 << 20), 1, "problem too large"),
    (dict(heads=1 << 24), 1, "problem too large"),
]


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("kwargs,status,needle", REFUSALS)
def test_refusals(lib, name, kwargs, status, needle):
    assert getattr(lib, name)(None, ctypes.byref(shape(**kwargs)), *[16] * CALLS[name]) == status
    message = lib.fhog_last_error().decode()
    assert needle in message and message.startswith(name)


def test_pointers_are_checked(lib):
    s = ctypes.byref(shape())
    assert lib.fhog_qk_norm_rotary_fwd(None, None, *[16] * 6) == 1
    assert lib.fhog_qk_norm_rotary_fwd(None, s, None, *[16] * 5) == 1 and b"q is null" in lib.fhog_last_error()
    assert lib.fhog_qk_norm_rotary_fwd(None, s, 16, 16, 15, 16, 16, 16) == 1 and b"a weight is not aligned" in lib.fhog_last_error()
    assert lib.fhog_qk_norm_rotary_fwd(None, s, *[16] * 4, 16, 3) == 1 and b"k_out is null or not" in lib.fhog_last_error()
    assert lib.fhog_qk_norm_rotary_bwd(None, s, *[16] * 8, None, 16, 16) == 1 and b"or the reverse" in lib.fhog_last_error()
    assert lib.fhog_qk_norm_rotary_bwd(None, s, *[16] * 10, None) == 1 and b"workspace is null" in lib.fhog_last_error()
    assert lib.fhog_qk_norm_rotary_bwdbwd(None, s, *[16] * 8, None, *[16] * 8) == 1 and b"or the reverse" in lib.fhog_last_error()
    plain = ctypes.byref(shape(norm=0))
    assert lib.fhog_qk_norm_rotary_fwd(None, plain, *[16] * 6) == 1 and b"weights need norms" in lib.fhog_last_error()
    assert lib.fhog_qk_norm_rotary_bwdbwd(None, plain, *[16] * 17) == 2 and b"linear" in lib.fhog_last_error()


def test_no_tokens_launch_nothing(lib):
    assert lib.fhog_qk_norm_rotary_fwd(None, ctypes.byref(shape(tokens=0)), None, None, None, None, None, None) == 0
    assert lib.fhog_qk_norm_rotary_workspace_bytes(ctypes.byref(shape(norm=0))) == 0
    assert lib.fhog_qk_norm_rotary_workspace_bytes(ctypes.byref(shape(head_dim=300))) == 0


def cpu(*s, dtype=BF16):
    return torch.zeros(*s, dtype=dtype)


def test_front_end_refuses():
    q, k = cpu(2, 5, 4, 64), cpu(2, 5, 2, 64)
    with pytest.raises(ValueError, match="must be on a GPU device"):
        flash_hog.qk_norm_rotary(q, k)
    with pytest.raises(ValueError, match=r"expected \(B, T, N, H\)"):
        flash_hog.qk_norm_rotary(q, k[0])
    with pytest.raises(ValueError, match=r"expected \(B, T, N, H\)"):
        flash_hog.qk_norm_rotary(q[0, 0], k[0, 0])
    with pytest.raises(ValueError, match="packed tokens"):
        flash_hog.qk_norm_rotary(q, k, lengths=torch.ones(2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="no derivative in frequencies"):
        flash_hog.qk_norm_rotary(q, k, frequencies=torch.ones(32, requires_grad=True))


@pytest.mark.parametrize("device", ["cuda", "cpu"])
def test_fake_tensors(device):
    with FakeTensorMode():
        q, k = (torch.zeros(2, 5, n, 64, dtype=BF16, device=device, requires_grad=True) for n in (4, 2))
        w = torch.ones(64, dtype=BF16, device=device, requires_grad=True)
        out = flash_hog.qk_norm_rotary(q, k, query_weight=w)
        assert [t.shape for t in out] == [q.shape, k.shape] and all(t.dtype == BF16 and t.device == q.device for t in out)
        if device == "cuda":
            return  # (autograd asks a real device about its streams)
        grads = torch.autograd.grad(out, (q, k, w), [torch.ones_like(o) for o in out], create_graph=True)
        second = torch.autograd.grad(grads, (q, k, w), [torch.ones_like(g) for g in grads])
        for x in (grads, second):
            assert [t.shape for t in x[:2]] == [q.shape, k.shape] and all(t.dtype == BF16 for t in x)
        assert grads[2].shape == second[2].shape == w.shape


@pytest.mark.parametrize("interleaved", [False, True])
def test_oracle_by_differences(interleaved):
    """The oracle's first derivative against differences of it, in 64 bits: h^2 and 2^-53 / h."""
    gen = torch.Generator().manual_seed(0)
    x, w, dy, u = (torch.randn(s, generator=gen, dtype=torch.float64) for s in ((5, 2, 16), (16,), (5, 2, 16), (5, 2, 16)))
    positions, freq = torch.arange(5), torch.tensor([1.0, 0.1, 0.01])
    got = ref.derivatives(x, w, positions, freq, interleaved, 1e-6, dy, u, torch.ones(16))
    h = 1e-5
    value = lambda t: (ref.apply(t, w, positions, freq, interleaved, 1e-6) * dy).sum()
    assert abs(float((value(x + h * u) - value(x - h * u)) / (2 * h) - (got["dx"] * u).sum())) < 1e-6
    assert torch.allclose(ref.rotate(ref.rotate(x, positions, freq, interleaved), -positions, freq, interleaved), x)
