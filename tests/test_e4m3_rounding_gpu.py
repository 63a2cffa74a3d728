"""The two appends of plain rows into an e4m3 cache leave the same bytes, those of value * (1 / scale) in fp32, also where that lies
on or next to a border between two e4m3 values."""
import numpy as np
import pytest

from test_block_scales_gpu import encode

pytestmark = pytest.mark.gpu

FP8 = 1


def on_borders(rng, heads):
    """fp16 rows [heads, 128] of few magnitudes, and a scale per head that puts them within a few steps of fp32 of a tie."""
    v = rng.uniform(1, 2, heads).astype(np.float16)
    tie = 1 + (2 * rng.integers(0, 8, heads) + 1) / 16
    s = (v / tie).astype(np.float32)
    s = (s.view(np.int32) + rng.integers(-2, 3, heads, dtype=np.int32)).view(np.float32)
    rows = v[:, None] * 2.0 ** rng.integers(-5, 6, (heads, 128)) * rng.choice([-1, 1], (heads, 128))
    return rows.astype(np.float16), s


@pytest.mark.parametrize("kind", ["head", "tensor"])
@pytest.mark.parametrize("seed", range(4))
def test_bytes_of_plain_rows(kind, seed, torch_cuda, pa):
    torch = torch_cuda
    rng = np.random.default_rng(seed)
    hkv = 2000
    (k, ks), (v, vs) = on_borders(rng, hkv), on_borders(rng, hkv)
    kw = dict(d_k_scales=torch.from_numpy(ks).cuda(), d_v_scales=torch.from_numpy(vs).cuda())
    if kind == "tensor":
        ks[:], vs[:] = ks[0], vs[0]
        kw = dict(k_scale=float(ks[0]), v_scale=float(vs[0]))
    x = [torch.from_numpy(r[None]).cuda() for r in (k, v)]
    pools = [torch.zeros(1, hkv, 16, 128, dtype=torch.uint8, device="cuda") for _ in range(4)]
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    t = pa.append_target(pools[0], pools[1], table, torch.tensor([3], dtype=torch.int32, device="cuda"), **kw)
    pa.append_qkv(FP8, pa.qkv_params(None, *x), None, t, None)
    pa.append_tokens(FP8, *x, pools[2], pools[3], table, 3, 1, hkv, 128, 16, **kw)
    assert pa.kernel_status() == 0
    for rows, s, mine, other in ((k, ks, pools[0], pools[2]), (v, vs, pools[1], pools[3])):
        want = encode(rows.astype(np.float32) * (np.float32(1) / s)[:, None])
        assert np.array_equal(other.cpu().numpy()[0, :, 3], want)
        assert np.array_equal(mine.cpu().numpy()[0, :, 3], want)
        assert torch.equal(mine, other)
