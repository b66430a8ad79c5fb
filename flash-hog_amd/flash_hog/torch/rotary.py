"""Norms of queries and keys for each head, with the position rotation in the same pass.

qk_norm_rotary stands before both kinds of attention: dot_product_attention, whose second
derivatives it shares (a Hessian-vector product through norms, rotation and attention runs in HIP
kernels throughout), and the paged cache's, whose lengths can give it the positions. No counterpart
in the reference.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from flash_hog import _hip

Tensor = torch.Tensor


# The three kernel calls as operators, for traces and transforms. Gradients of absent weights are
# tensors of no elements there, as an operator's results cannot be None.

def _given(t, like):
    return like.new_empty(0) if t is None else t


@torch.library.custom_op("flash_hog::qk_norm_rotary", mutates_args=())
def qk_norm_rotary_op(q: Tensor, k: Tensor, wq: Tensor | None, wk: Tensor | None, frequencies: Tensor | None,
                      positions: Tensor | None, lengths: Tensor | None, query_offsets: Tensor | None,
                      interleaved: bool, eps: float | None) -> tuple[Tensor, Tensor]:
    return _hip.qk_norm_rotary_fwd(q, k, wq, wk, frequencies, positions, lengths, query_offsets, interleaved, eps)


@torch.library.custom_op("flash_hog::qk_norm_rotary_bwd", mutates_args=())
def qk_norm_rotary_bwd_op(q: Tensor, k: Tensor, wq: Tensor | None, wk: Tensor | None, gq: Tensor, gk: Tensor,
                          frequencies: Tensor | None, positions: Tensor | None, lengths: Tensor | None,
                          query_offsets: Tensor | None, interleaved: bool,
                          eps: float | None) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    dq, dk, dwq, dwk = _hip.qk_norm_rotary_bwd(q, k, wq, wk, gq, gk, frequencies, positions, lengths, query_offsets,
                                               interleaved, eps)
    return dq, dk, _given(dwq, q), _given(dwk, k)


@torch.library.custom_op("flash_hog::qk_norm_rotary_bwdbwd", mutates_args=())
def qk_norm_rotary_bwdbwd_op(q: Tensor, k: Tensor, wq: Tensor | None, wk: Tensor | None, gq: Tensor, gk: Tensor,
                             uq: Tensor, uk: Tensor, zq: Tensor, zk: Tensor, frequencies: Tensor | None,
                             positions: Tensor | None, lengths: Tensor | None, query_offsets: Tensor | None,
                             interleaved: bool,
                             eps: float | None) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    dq2, dk2, dwq2, dwk2, dgq, dgk = _hip.qk_norm_rotary_bwdbwd(q, k, wq, wk, gq, gk, uq, uk, zq, zk, frequencies,
                                                                positions, lengths, query_offsets, interleaved, eps)
    return dq2, dk2, _given(dwq2, q), _given(dwk2, k), dgq, dgk


def _like(*tensors):
    return tuple(torch.empty_like(t, memory_format=torch.contiguous_format) for t in tensors)


def _like_weights(q, k, wq, wk):
    return tuple(x.new_empty(0) if w is None else torch.empty_like(w) for w, x in ((wq, q), (wk, k)))


@qk_norm_rotary_op.register_fake
def _(q, k, wq, wk, frequencies, positions, lengths, query_offsets, interleaved, eps):
    return _like(q, k)


@qk_norm_rotary_bwd_op.register_fake
def _(q, k, wq, wk, gq, gk, frequencies, positions, lengths, query_offsets, interleaved, eps):
    return (*_like(q, k), *_like_weights(q, k, wq, wk))


@qk_norm_rotary_bwdbwd_op.register_fake
def _(q, k, wq, wk, gq, gk, uq, uk, zq, zk, frequencies, positions, lengths, query_offsets, interleaved, eps):
    return (*_like(q, k), *_like_weights(q, k, wq, wk), *_like(gq, gk))


def _one_by_one(op):
    """vmap rule: a call for each element (weights' gradients are sums over a call's rows, so elements
    cannot share one)."""

    def rule(info, in_dims, *args):
        if info.batch_size == 0:  # (a call on zeros for the results' shapes)
            one = op(*(a if d is None else a.new_zeros(a.shape[:d] + a.shape[d + 1:]) for a, d in zip(args, in_dims)))
            outs = tuple(x.new_empty((0, *x.shape)) for x in one)
        else:
            each = [op(*(a if d is None else a.select(d, i) for a, d in zip(args, in_dims))) for i in range(info.batch_size)]
            outs = tuple(torch.stack(x) for x in zip(*each))
        return outs, (0,) * len(outs)

    op.register_vmap(rule)


for _op in (qk_norm_rotary_op, qk_norm_rotary_bwd_op, qk_norm_rotary_bwdbwd_op):
    _one_by_one(_op)


def _plain(*tensors) -> bool:
    """Whether a call goes straight to the C ABI: no trace, no transform, every tensor with memory of its own."""
    return (not torch._C._are_functorch_transforms_active() and not torch.compiler.is_compiling()
            and all(t is None or type(t) in (Tensor, torch.nn.Parameter) for t in tensors))


def _fwd(q, k, wq, wk, where, interleaved, eps):
    call = _hip.qk_norm_rotary_fwd if _plain(q, k, wq, wk, *where) else qk_norm_rotary_op
    return tuple(call(q, k, wq, wk, *where, interleaved, eps))


# As in flash_hog.torch.attention: Functions in the setup_context form, which torch.func transforms
# compose with, and in the ctx-first form for eager calls without the torch extension, which has the same
# two in C++ (csrc/fhog_torch.cpp, RotaryFn and RotaryBwdFn). `where`: frequencies, positions, lengths,
# query_offsets.

class _QKNormRotary(torch.autograd.Function):
    generate_vmap_rule = True

    @staticmethod
    def forward(q, k, wq, wk, frequencies, positions, lengths, query_offsets, interleaved, eps):
        return _fwd(q, k, wq, wk, (frequencies, positions, lengths, query_offsets), interleaved, eps)

    @staticmethod
    def setup_context(ctx, inputs, output):
        q, k, wq, wk, frequencies, positions, lengths, query_offsets, interleaved, eps = inputs
        where = frequencies, positions, lengths, query_offsets
        if eps is None:  # the rotation's derivative needs no rows
            ctx.save_for_backward(*where)
        else:
            ctx.save_for_backward(*where, q, k, wq, wk)
        ctx.interleaved, ctx.eps = interleaved, eps

    @staticmethod
    def backward(ctx, gq, gk):
        where, rest = ctx.saved_tensors[:4], ctx.saved_tensors[4:]
        # (without norms the cotangents stand in for the rows, of which only the shapes matter)
        q, k, wq, wk = rest if rest else (gq.detach(), gk.detach(), None, None)
        fn = _QKNormRotaryBwd if torch._C._are_functorch_transforms_active() else _QKNormRotaryBwdEager
        dq, dk, dwq, dwk = fn.apply(q, k, wq, wk, gq, gk, *where, ctx.interleaved, ctx.eps)
        return (dq, dk, None if wq is None else dwq, None if wk is None else dwk) + (None,) * 6


class _QKNormRotaryBwd(torch.autograd.Function):
    generate_vmap_rule = True

    @staticmethod
    def forward(q, k, wq, wk, gq, gk, frequencies, positions, lengths, query_offsets, interleaved, eps):
        where = frequencies, positions, lengths, query_offsets
        if _plain(q, k, wq, wk, gq, gk, *where):
            dq, dk, dwq, dwk = _hip.qk_norm_rotary_bwd(q, k, wq, wk, gq, gk, *where, interleaved, eps)
            return dq, dk, _given(dwq, q), _given(dwk, k)
        return tuple(qk_norm_rotary_bwd_op(q, k, wq, wk, gq, gk, *where, interleaved, eps))

    @staticmethod
    def setup_context(ctx, inputs, output):
        q, k, wq, wk, gq, gk, frequencies, positions, lengths, query_offsets, interleaved, eps = inputs
        where = frequencies, positions, lengths, query_offsets
        if eps is None:
            ctx.save_for_backward(*where)
        else:
            ctx.save_for_backward(*where, q, k, wq, wk, gq, gk)
        ctx.interleaved, ctx.eps = interleaved, eps

    @staticmethod
    @once_differentiable
    def backward(ctx, uq, uk, zq, zk):
        where, rest = ctx.saved_tensors[:4], ctx.saved_tensors[4:]
        if ctx.eps is None:
            dgq, dgk = _fwd(uq, uk, None, None, where, ctx.interleaved, None)
            return (None,) * 4 + (dgq, dgk) + (None,) * 6
        wq, wk = rest[2:4]
        if _plain(uq, uk, zq, zk, *rest, *where):
            dq2, dk2, dwq2, dwk2, dgq, dgk = _hip.qk_norm_rotary_bwdbwd(*rest, uq, uk, zq, zk, *where, ctx.interleaved,
                                                                        ctx.eps)
        else:
            dq2, dk2, dwq2, dwk2, dgq, dgk = qk_norm_rotary_bwdbwd_op(*rest, uq, uk, zq, zk, *where, ctx.interleaved,
                                                                      ctx.eps)
        return (dq2, dk2, None if wq is None else dwq2, None if wk is None else dwk2, dgq, dgk) + (None,) * 6


class _QKNormRotaryEager(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *args):
        output = _QKNormRotary.forward(*args)
        _QKNormRotary.setup_context(ctx, args, output)
        return output

    backward = _QKNormRotary.backward


class _QKNormRotaryBwdEager(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *args):
        output = _QKNormRotaryBwd.forward(*args)
        _QKNormRotaryBwd.setup_context(ctx, args, output)
        return output

    backward = _QKNormRotaryBwd.backward


def qk_norm_rotary(query, key, positions=None, *, frequencies=None, query_weight=None, key_weight=None,
                   eps: float | None = 1e-6, interleaved: bool = False, lengths=None, query_offsets=None):
    """Queries (B, T, N, H) and keys (B, T, N_kv, H) of the same tokens, or unbatched (T, N, H) and
    (T, N_kv, H), normalised head by head and rotated; returns both, contiguous, in their dtype.

    A row x of H values is divided by its root mean square, sqrt(mean(x ** 2) + eps), and multiplied by
    its weight (H,), of the rows' dtype or float32 (both alike; None: ones). eps=None leaves norms out.

    Then the pairs of its first R columns turn by position * frequencies[i], with frequencies
    (R / 2,) float32, for instance 10000.0 ** (-arange(0, R, 2) / R): columns i and i + R / 2, or 2 i and
    2 i + 1 if interleaved. Angles are formed in 64 bits, so far positions lose nothing. Columns from
    R on stay as they are; frequencies=None leaves rotation out.

    positions: (T,) or (B, T) of int32 or int64; None: 0 to T - 1. Or, for packed tokens (T, N, H), a paged
    cache's lengths and query_offsets (flash_hog.torch.paged; the new tokens' last positions; rows of
    no sequence are at position 0). They are read on the device only.

    Any H from 1 to 256, bfloat16, float16 or float32; sums are fp32. Rows may lie anywhere, as views of a
    joint projection do. They are read in wide loads where H and R are multiples of 8 and all rows begin at multiples
    of four elements' size; else element by element, which takes 1.3 to 2 times as long.
    Differentiable twice in query, key and the weights. Weights' gradients are summed in a fixed order.
    torch.func.vmap makes a call for each element.
    """
    if query.ndim not in (3, 4) or key.ndim != query.ndim:
        raise ValueError(f"expected (B, T, N, H) or (T, N, H) tensors, got {tuple(query.shape)} and {tuple(key.shape)}")
    if frequencies is not None and frequencies.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("qk_norm_rotary has no derivative in frequencies")
    if lengths is not None and query.ndim != 3:
        raise ValueError(f"lengths go with packed tokens (T, N, H), got {tuple(query.shape)}")
    if eps is not None:
        eps = float(eps)
    tensors = (query, key, query_weight, key_weight, frequencies, positions, lengths, query_offsets)
    if _plain(*tensors) and forward_ad._current_level < 0:
        ext = _hip.torch_ext()
        if ext is not None:  # the Functions above in C++
            return ext.qk_norm_rotary(*tensors, bool(interleaved), eps)
    unbatched = query.ndim == 3
    if unbatched:
        query, key = query.unsqueeze(0), key.unsqueeze(0)
    args = (query, key, query_weight, key_weight, frequencies, positions, lengths, query_offsets, bool(interleaved), eps)
    if torch._C._are_functorch_transforms_active() or torch.compiler.is_compiling():
        q, k = _QKNormRotary.apply(*args)
    elif forward_ad._current_level >= 0 or (torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in args[:4])):
        q, k = _QKNormRotaryEager.apply(*args)
    else:
        q, k = _fwd(*args[:4], args[4:8], *args[8:])
    return (q[0], k[0]) if unbatched else (q, k)
