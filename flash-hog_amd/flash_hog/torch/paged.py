"""Attention over a paged key/value cache: serving what dot_product_attention trains.

  paged_cache_write   the keys and values of new tokens into their sequences' pages,
                      quantised to e4m3 on the way where the cache holds that
  paged_attention     the new tokens' attention over the cached keys of their sequences:
                      one token each (decoding) or chunks of unequal length (prompts), with the
                      window and sinks of dot_product_attention
  paged_cache_read    cached sequences back as dense tensors, as dot_product_attention takes them

No counterpart in the reference, which trains only. All three enqueue their kernels on the
current stream of the tensors' device, read no length back to the host, and can be captured in
a HIP graph; workspaces come from torch's allocator, a new one for each call.

A cache is two contiguous tensors (pages, kv_heads, page_size, head_dim), of the queries' dtype
(bfloat16 or float16) or float8_e4m3fn; the page size is a power of two from 16 on, the head dim
64, 128 or 256. An e4m3 cache has key_scale and value_scale, (pages, kv_heads, page_size) of
float8_e8m0fnu (or its bytes, uint8): a row of the cache stands for its e4m3 values times its
scale, a power of two.

page_table (batch, pages per sequence) int32: token s of sequence b is row s % page_size of page
page_table[b, s // page_size]. lengths (batch,) int32: the tokens that a sequence holds, its new
ones included. query_offsets (batch + 1,) int32: the new tokens of all sequences are packed,
sequence b's are rows query_offsets[b] to query_offsets[b + 1] and take its last positions, in
order; None: each sequence has one.

The index tensors are read on the device only, so mistakes in them cannot raise: an attended
page outside the cache, or a length beyond its table, gives NaN in rows of its sequence, those
that depend on it at least (paged_cache_write leaves such a token out), and no access leaves its
tensor. Entries and cache
slots that no visible token needs may hold anything, NaN included. Among the keys of one 32-key
tile, though, a NaN or infinity in a value that one token sees also reaches the rows beside it.

The functions have no derivative: tensors that require a gradient (in grad mode) or carry a tangent are
refused, and so are ones that torch.func.vmap maps over. What they write to gets a new autograd version.

For speed: how a sequence's keys are split over workgroups follows from the table's width, since no
length is read back, and how rows are tiled from the average number of new tokens. So give short chunks
a table not much wider than they need (64 tokens of 8192 take three times as long with one 32 times as wide;
single tokens hardly lose), and give prompts and single tokens on long contexts a call each (a prompt
of 2048 and a token of 32768, 32 heads over 8 of 128: 69 and 38 us, in one call 888).
"""

from __future__ import annotations

import operator

import torch
from torch.autograd import forward_ad

from flash_hog import _hip
from flash_hog.torch._hip_gpu import _default_scale

Tensor = torch.Tensor


_PLAIN = Tensor.__torch_dispatch__


def _checked(name, index, *tensors) -> bool:
    """Refuses tensors that carry a derivative or that vmap maps over. Returns whether the call goes
    through its operator, because it is traced or because some tensor has no memory of its own to
    point at (fake tensors, the wrappers of torch.func transforms); plain ones go straight to the C ABI.
    index: the tensors that find tokens, which carry no derivative."""
    through = torch.compiler.is_compiling()
    grad = torch.is_grad_enabled()
    for t in tensors:
        if t is None:
            continue
        if grad and t.requires_grad:
            raise RuntimeError(f"{name} has no derivative: call it under torch.no_grad() (training attends through "
                               "flash_hog.dot_product_attention)")
        if type(t) is not Tensor and getattr(type(t), "__torch_dispatch__", _PLAIN) is not _PLAIN:
            through = True
    # A forward-mode dual tensor does not require a gradient, in grad mode or out of it.
    if forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled():
        if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
            raise RuntimeError(f"{name} has no derivative, in forward mode either: call it on tensors without a tangent")
    if torch._C._are_functorch_transforms_active():
        ours = [t for t in (*tensors, *index) if isinstance(t, Tensor)]
        if any(map(torch._C._functorch.is_batchedtensor, ours)):
            raise RuntimeError(f"{name} has no batching rule, so torch.func.vmap cannot map it: its sequences are a batch "
                               "already")
        through = through or any(map(torch._C._functorch.is_functorch_wrapped_tensor, ours))
    return through


@torch.library.custom_op("flash_hog::paged_attention", mutates_args=())
def paged_attention_op(query: Tensor, key_cache: Tensor, value_cache: Tensor, page_table: Tensor, lengths: Tensor,
                       query_offsets: Tensor | None, key_scale: Tensor | None, value_scale: Tensor | None, window: int,
                       sinks: int, scale: float) -> Tensor:
    return _hip.paged_attention(query, key_cache, value_cache, page_table, lengths, query_offsets, key_scale,
                                value_scale, window, sinks, scale)


@paged_attention_op.register_fake
def _(query, key_cache, value_cache, page_table, lengths, query_offsets, key_scale, value_scale, window, sinks, scale):
    return torch.empty_like(query, memory_format=torch.contiguous_format)


@torch.library.custom_op("flash_hog::paged_cache_write",
                         mutates_args=("key_cache", "value_cache", "key_scale", "value_scale"))
def paged_cache_write_op(key: Tensor, value: Tensor, key_cache: Tensor, value_cache: Tensor, page_table: Tensor,
                         lengths: Tensor, query_offsets: Tensor | None, key_scale: Tensor | None,
                         value_scale: Tensor | None) -> None:
    _hip.paged_cache_write(key, value, key_cache, value_cache, page_table, lengths, query_offsets, key_scale,
                           value_scale)


@torch.library.custom_op("flash_hog::paged_cache_read", mutates_args=())
def paged_cache_read_op(key_cache: Tensor, value_cache: Tensor, page_table: Tensor, lengths: Tensor, max_length: int,
                        dtype: torch.dtype, key_scale: Tensor | None,
                        value_scale: Tensor | None) -> tuple[Tensor, Tensor]:
    return _hip.paged_cache_read(key_cache, value_cache, page_table, lengths, max_length, dtype, key_scale, value_scale)


@paged_cache_read_op.register_fake
def _(key_cache, value_cache, page_table, lengths, max_length, dtype, key_scale, value_scale):
    shape = (page_table.shape[0], max_length, key_cache.shape[1], key_cache.shape[3])
    return key_cache.new_empty(shape, dtype=dtype), key_cache.new_empty(shape, dtype=dtype)


def paged_attention(query, key_cache, value_cache, page_table, lengths, query_offsets=None, *, key_scale=None,
                    value_scale=None, window: int | None = None, sinks: int = 0, scale: float | None = None, out=None):
    """Attention of the packed new tokens query (T, N, H) over the cached keys and values of
    their sequences; returns (T, N, H). The new tokens' own keys are read from the cache too:
    paged_cache_write goes first.

    A token at position p of its sequence sees its keys s <= p; with a window those with
    s > p - window, and the first `sinks` ones besides. One that sees none (a sequence of length
    zero) gives zeros. Query heads share key/value heads as in dot_product_attention; scale
    defaults to H ** -0.5.

    out: a contiguous tensor for the result; its rows of no sequence (from query_offsets[batch]
    on, a padded batch) are left as they were. Without it they are zero. It may be query itself, and
    overlaps neither query otherwise nor the caches.
    """
    through = _checked("paged_attention", (page_table, lengths, query_offsets), query, key_cache, value_cache, key_scale,
                       value_scale, out)
    if window is None:
        if sinks != 0:
            raise ValueError(f"sinks needs a window, got sinks={sinks}")
        window = 0
    else:
        window, sinks = operator.index(window), operator.index(sinks)
        if window < 1 or sinks < 0:
            raise ValueError(f"window must be >= 1 and sinks >= 0, got {window} and {sinks}")
    scale = _default_scale(query, scale)
    args = (query, key_cache, value_cache, page_table, lengths, query_offsets, key_scale, value_scale, window, sinks,
            scale)
    if through:
        if out is None:
            return paged_attention_op(*args)
        raise ValueError("out is not supported under torch.compile, transforms or fake tensors")
    return _hip.paged_attention(*args, out=out)


def paged_cache_write(key, value, key_cache, value_cache, page_table, lengths, query_offsets=None, *, key_scale=None,
                      value_scale=None) -> None:
    """Writes key and value (T, N_kv, H) of the packed new tokens to their places in the cache, in
    place. An e4m3 cache gets each row quantised: its scale is the smallest power of two (at least
    2 ** -126) with which the row's largest finite magnitude stays within 448, its values round
    to nearest even, and infinities become NaN; a value within 1/32 of the type's largest may
    round beyond it, and then reads as infinite. Rows of no sequence and tokens at
    positions below zero (a sequence of length zero) are not written. No two tokens may name the
    same place: pages that sequences share are read-only. key and value may lie in the cache too, but not
    where this call writes."""
    through = _checked("paged_cache_write", (page_table, lengths, query_offsets), key, value, key_cache, value_cache,
                       key_scale, value_scale)
    call = paged_cache_write_op if through else _hip.paged_cache_write
    call(key, value, key_cache, value_cache, page_table, lengths, query_offsets, key_scale, value_scale)


def paged_cache_read(key_cache, value_cache, page_table, lengths, *, max_length: int | None = None, dtype=None,
                     key_scale=None, value_scale=None):
    """The first max_length tokens (default: what the table can hold) of the sequences as dense
    keys and values (batch, max_length, N_kv, H), zeros behind a sequence's length. dtype is the
    cache's, or for an e4m3 cache bfloat16 (default) or float16, to which its values are rounded."""
    through = _checked("paged_cache_read", (page_table, lengths), key_cache, value_cache, key_scale, value_scale)
    if dtype is None:
        dtype = torch.bfloat16 if key_cache.dtype == torch.float8_e4m3fn else key_cache.dtype
    if max_length is None:
        if page_table.ndim != 2 or key_cache.ndim != 4:
            raise ValueError("expected a (batch, pages) page_table and a (pages, kv_heads, page_size, head_dim) cache, "
                             f"got {tuple(page_table.shape)} and {tuple(key_cache.shape)}")
        max_length = page_table.shape[1] * key_cache.shape[2]
    call = paged_cache_read_op if through else _hip.paged_cache_read
    return call(key_cache, value_cache, page_table, lengths, max_length, dtype, key_scale, value_scale)
