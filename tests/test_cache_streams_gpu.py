"""Calls on a cache from streams that do not wait for each other (every torch side stream is a non-blocking one), with work
still queued on the stream that a call uses inside; lengths that do not fit."""
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


def test_a_new_cache_is_zeroed_before_the_first_append(torch_cuda, pa):
    """Pools, block table and lengths; the device-side plan reads the last two."""
    torch = torch_cuda
    hkv, hq = 2, 4
    side = torch.cuda.Stream()
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(40, hkv, 128, device="cuda", generator=g).half() for _ in range(2))
    q = torch.randn(1, hq, 128, device="cuda", generator=g).half()
    out = torch.zeros_like(q)
    rows = pa.qkv_params(None, k, v)
    pa.kernel_status()
    torch.cuda.synchronize()
    torch.cuda._sleep(QUEUED)
    c = new_cache(pa, dtype=0)
    slots = [c.admit() for _ in range(2)]
    assert c.append_qkv(slots[1:], [40], rows, None, None, side.cuda_stream)
    torch.cuda.synchronize()
    assert device_view(c.params().seq_lens, 16, torch).view(torch.int32).tolist() == [0, 40, 0, 0]
    pool = device_view(c.params().k_cache, 8 * hkv * 16 * 128 * 2, torch).view(torch.float16).view(8, hkv, 16, 128)
    pages = c.block_table(1)
    assert torch.equal(pool[torch.from_numpy(pages[:2].astype(np.int64)).cuda()].transpose(1, 2).reshape(32, hkv, 128), k[:32])
    assert not pool[int(pages[2]), :, 8:].any()
    c.plan([1], hq)
    c.run(q, out)
    assert pa.kernel_status() == 0
    want, tol = ro.attention(q[0].double().cpu().numpy(), k.double().cpu().numpy(), v.double().cpu().numpy(), 1 / np.sqrt(np.float32(128)))
    assert (np.abs(out[0].double().cpu().numpy() - want) <= tol).all()


@pytest.mark.parametrize("batched", [False, True])
def test_a_released_slot_is_zeroed_before_its_next_append(batched, torch_cuda, pa):
    """release() zeroes the slot's device length, which the device-side plan reads, on the default stream."""
    torch = torch_cuda
    hkv, hq = 2, 4
    side = torch.cuda.Stream()
    g = torch.Generator(device="cuda").manual_seed(2)
    k, v = (torch.randn(40, hkv, 128, device="cuda", generator=g).half() for _ in range(2))
    q = torch.randn(1, hq, 128, device="cuda", generator=g).half()
    out = torch.zeros_like(q)
    c = new_cache(pa, dtype=0)
    assert c.admit() == 0 and c.append(0, v, k, 17)
    torch.cuda.synchronize()
    torch.cuda._sleep(QUEUED)
    c.release(0)
    assert c.admit() == 0
    if batched:
        assert c.append_batch([0], [k], [v], [40], side.cuda_stream)
    else:
        assert c.append(0, k, v, 40, side.cuda_stream)
    c.plan_device(1, hq, stream=side.cuda_stream)
    c.run(q, out, side.cuda_stream)
    torch.cuda.synchronize()
    assert pa.kernel_status() == 0
    assert device_view(c.params().seq_lens, 16, torch).view(torch.int32).tolist() == [40, 0, 0, 0]
    want, tol = ro.attention(q[0].double().cpu().numpy(), k.double().cpu().numpy(), v.double().cpu().numpy(), 1 / np.sqrt(np.float32(128)))
    assert (np.abs(out[0].double().cpu().numpy() - want) <= tol).all()


def test_a_device_plan_sees_a_released_slot_as_empty(torch_cuda, pa):
    torch = torch_cuda
    side = torch.cuda.Stream()
    x = torch.ones(40, 2, 128, dtype=torch.float16, device="cuda")
    q, out = torch.ones(2, 4, 128, dtype=torch.float16, device="cuda"), torch.full((2, 4, 128), 7.0, dtype=torch.float16, device="cuda")
    c = new_cache(pa, dtype=0)
    assert [c.admit(), c.admit()] == [0, 1] and c.append(0, x, x, 40) and c.append(1, x, x, 20)
    torch.cuda.synchronize()
    torch.cuda._sleep(QUEUED)
    c.release(0)
    c.plan_device(2, 4, stream=side.cuda_stream)
    c.run(q, out, side.cuda_stream)
    torch.cuda.synchronize()
    assert pa.kernel_status() == 0
    assert (out[0] == 7).all() and (out[1] == 1).all()          # a row of length 0 is left as it was


@pytest.mark.parametrize("blocks", [False, True])
def test_single_and_batched_appends_on_two_streams(blocks, torch_cuda, pa):
    """append_qkv and append_batch on one stream, kept busy, and append on another, for the same slots: lengths, tables, bytes and
    scales as from the same calls with waits in between."""
    torch = torch_cuda
    hkv, pages = 2, 24
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    rng = np.random.default_rng(3)
    # magnitudes that grow: with block scales every call re-encodes what the one before it left in the block
    x = torch.from_numpy(rng.standard_normal((12, 2, 5, hkv, 128)) * 2.0 ** np.arange(12)[:, None, None, None, None]).half().cuda()
    results = []
    for wait in (True, False):
        c = new_cache(pa, pages=pages, slots=2, per_slot=12)
        if blocks:
            c.set_block_scales()
        slots = [c.admit(), c.admit()]
        torch.cuda.synchronize()

        def then():
            if wait:
                torch.cuda.synchronize()
        for i in range(12):
            rows = x[i].reshape(10, hkv, 128)
            if not wait:
                with torch.cuda.stream(a):
                    torch.cuda._sleep(QUEUED // 20)
            if i % 3:
                assert c.append_qkv(slots, [5, 5], pa.qkv_params(None, rows, rows), None, None, a.cuda_stream)
            else:
                assert c.append_batch(slots, [x[i, 0], x[i, 1]], [x[i, 1], x[i, 0]], [5, 4], a.cuda_stream)
            then()
            assert c.append(slots[i % 2], x[i, 0], x[i, 1], 3, b.cuda_stream)
            then()
        torch.cuda.synchronize()
        assert pa.kernel_status() == 0
        p, bytes_ = c.params(), pages * hkv * 16 * 128
        state = [device_view(ptr, n, torch).clone() for ptr, n in ((p.k_cache, bytes_), (p.v_cache, bytes_), (p.seq_lens, 8), (p.block_table, 2 * 12 * 4))]
        if blocks:
            state.append(device_view(c.block_scales(), pages * hkv * 8, torch).clone())
        results.append(state)
        assert state[2].view(torch.int32).tolist() == [c.seq_len(s) for s in slots] == [78, 74]
        c.close()
    assert all(torch.equal(s, t) for s, t in zip(*results))


@pytest.mark.parametrize("dtype, blocks", [(0, False), (1, False), (1, True)])
def test_a_length_past_31_bits_is_refused(dtype, blocks, torch_cuda, pa):
    """Nothing may be launched for it: a sum that wraps would pass the check against max_pages_per_slot."""
    torch = torch_cuda
    x = torch.ones(3, 2, 128, dtype=torch.float16, device="cuda")
    c = new_cache(pa, dtype=dtype)
    if blocks:
        c.set_block_scales()
    slot = c.admit()
    assert c.append(slot, x, x, 3)
    for n in (2 ** 31 - 1, 2 ** 31 - 3, 2 ** 31 - 16, 4 * 16 - 2):
        with pytest.raises(pa.LengthError):
            c.append(slot, x, x, n)
        with pytest.raises(pa.LengthError):
            c.append_batch([slot], [x], [x], [n])
    assert c.seq_len(slot) == 3 and c.free_pages() == 7


def test_a_device_plan_is_captured_behind_a_release(torch_cuda, pa):
    """The capture neither fails on the wait for the release's zero nor leaves it out of the replays' past."""
    torch = torch_cuda
    side = torch.cuda.Stream()
    x = torch.ones(40, 2, 128, dtype=torch.float16, device="cuda")
    q, out = torch.ones(2, 4, 128, dtype=torch.float16, device="cuda"), torch.zeros(2, 4, 128, dtype=torch.float16, device="cuda")
    c = new_cache(pa, dtype=0)
    assert [c.admit(), c.admit()] == [0, 1] and c.append(0, x, x, 40) and c.append(1, x, x, 20)
    c.plan_device(2, 4, stream=side.cuda_stream)
    c.run(q, out, side.cuda_stream)                              # first use: buffers are sized
    torch.cuda.synchronize()
    c.release(0)
    torch.cuda.synchronize()
    out.fill_(7)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        c.plan_device(2, 4, stream=side.cuda_stream)
        c.run(q, out, side.cuda_stream)
    g.replay()
    torch.cuda.synchronize()
    assert (out[0] == 7).all() and (out[1] == 1).all()
    assert c.admit() == 0 and c.append_batch([0], [x], [x], [33], side.cuda_stream)
    torch.cuda.synchronize()
    g.replay()
    torch.cuda.synchronize()
    assert pa.kernel_status() == 0 and (out == 1).all()
