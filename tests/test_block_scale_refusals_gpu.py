"""A block-scaled cache in the decodes that cannot read it: refused, nothing launched, and usable afterwards."""
import pytest

pytestmark = pytest.mark.gpu

FP8 = 1


def test_gathered_static_and_plain_decode_refuse_it(torch_cuda, pa):
    from paged_attention_b200.sharding import GatherGroup
    torch = torch_cuda
    c = pa.PagedKVCache(pa.PagedKVCache.Config(8, 16, 2, 128, 2, 4, pa.KVDtype.FP8_E4M3))
    c.set_block_scales()
    x = torch.ones(40, 2, 128, dtype=torch.float16, device="cuda")
    slot = c.admit()
    assert c.append(slot, x, x, 40)
    q, out = torch.ones(1, 4, 128, dtype=torch.float16, device="cuda"), torch.full((1, 4, 128), 7.0, dtype=torch.float16, device="cuda")
    plan, dp = pa.make_plan(FP8, [40], 4, 2, 128), pa.DevicePlan()
    dp.upload(plan, 2, 128)
    p = c.params()
    p.q, p.out, p.batch, p.num_q_heads = q.data_ptr(), out.data_ptr(), 1, 4
    dp.bind(p)
    g = GatherGroup(out.numel() * 2)
    for call in (lambda: pa.paged_decode(FP8, p, 0, 8), lambda: pa.paged_decode_static(FP8, p, plan, 0, 8),
                 lambda: g.decode(FP8, p, 4, num_pages=8), lambda: g.decode(FP8, p, 4, num_pages=8, sync=True)):
        with pytest.raises(pa.InvalidArgument, match="block-scaled"):
            call()
    assert g.epoch == 0
    torch.cuda.synchronize()
    assert (out == 7).all()
    pa.paged_decode(FP8, p, 0, 8, d_block_scales=c.block_scales())
    assert pa.kernel_status() == 0 and (out == 1).all()
    p.k_scale = p.v_scale = 2.0 ** -8               # every block of these rows has this scale
    g.decode(FP8, p, 4, num_pages=8, sync=True)
    torch.cuda.synchronize()
    from common import device_view
    assert g.epoch == 1 and (device_view(g.buffer_ptr(), out.numel() * 2, torch).view(torch.float16) == 1).all()
    g.close()
