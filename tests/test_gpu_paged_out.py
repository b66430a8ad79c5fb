"""What the paged cache's functions write to may not share memory with what finds tokens in the cache, nor with its
scales: kernels would read what others have written."""

from __future__ import annotations

import pytest
import torch

from test_gpu_blocks import BF16, make

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[False, True], ids=["extension", "python"])
def flash_hog(request, monkeypatch):
    import flash_hog
    from flash_hog import _hip

    if request.param:
        monkeypatch.setattr(_hip, "torch_ext", lambda: None)
    return flash_hog


@pytest.mark.parametrize("name", ["page_table", "lengths", "query_offsets", "key_scale", "value_scale"])
def test_out_apart_from_what_is_read(name, flash_hog, cuda_device):
    print("[case] out", name, flush=True)
    cache, counts, q, moved, where = make((4, 2, 64, BF16, True, 16, [40, 30], [3, 2]), cuda_device)
    q, kv = q.to(cuda_device), (moved["key_cache"], moved["value_cache"])
    chosen = torch.zeros((q.shape[0], 2, 2), dtype=torch.int32, device=cuda_device)
    args = {**where, "key_scale": moved["key_scale"], "value_scale": moved["value_scale"]}
    means = torch.zeros((kv[0].shape[0], 2, 64), device=cuda_device)
    calls = {"out": (lambda a, out: flash_hog.paged_attention(q, *kv, **a, out=out), q),
             "out ": (lambda a, out: flash_hog.paged_block_attention(q, chosen, *kv, **a, out=out), q)}
    if name != "value_scale":
        scale = lambda a: {k: t for k, t in a.items() if k != "value_scale"}
        calls["key_means"] = (lambda a, out: flash_hog.paged_key_means(kv[0], out, **scale(a)), means)
    for what, (call, like) in calls.items():
        # the tensor's bytes right behind the output's, and then 16 before their end
        bytes_of = args[name].view(torch.uint8).flatten()
        room = torch.zeros(like.nbytes + bytes_of.numel() + 64, dtype=torch.uint8, device=cuda_device)
        for at, fits in ((like.nbytes, True), (like.nbytes - 16, False)):
            out = room[:like.nbytes].view(like.dtype).view(like.shape)
            shared = room[at:at + bytes_of.numel()].view(args[name].dtype).view(args[name].shape)
            shared.view(torch.uint8).flatten().copy_(bytes_of)
            if fits:
                call({**args, name: shared}, out)
            else:
                with pytest.raises(ValueError, match=f"{what.strip()} overlaps {name}"):
                    call({**args, name: shared}, out)
