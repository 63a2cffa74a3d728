"""Calls on a cache from streams that do not wait for each other (every torch side stream is a non-blocking one), with work
still queued on the stream that a call uses inside."""
import numpy as np
import pytest

import rows_oracle as ro
from common import device_view

pytestmark = pytest.mark.gpu

FP8 = 1
QUEUED = 100_000_000        # clock cycles of a waiting kernel: some 50 ms


def new_cache(pa, pages=8, hkv=2, slots=4, per_slot=4, dtype=FP8):
    return pa.PagedKVCache(pa.PagedKVCache.Config(pages, 16, hkv, 128, slots, per_slot, pa.KVDtype(dtype)))


def block_scales(c, torch, pages=8, hkv=2):
    return device_view(c.block_scales(), pages * hkv * 8, torch).view(torch.float32).view(pages, hkv, 2).cpu()


def test_block_scales_are_zeroed_before_the_first_append(torch_cuda, pa):
    torch = torch_cuda
    side = torch.cuda.Stream()
    x = torch.ones(16, 2, 128, dtype=torch.float16, device="cuda")
    rows = pa.qkv_params(None, x, x)
    c = new_cache(pa)
    slot = c.admit()
    pa.kernel_status()                              # the status word exists
    torch.cuda.synchronize()
    torch.cuda._sleep(QUEUED)
    c.set_block_scales()
    assert c.append_qkv([slot], [16], rows, None, None, side.cuda_stream)
    torch.cuda.synchronize()
    s = block_scales(c, torch)
    assert (s[c.block_table(slot)[0]] == 2.0 ** -8).all() and (s == 0).sum() == s.numel() - 4
