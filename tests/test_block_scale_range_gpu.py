"""Decode over a block-scaled cache whose V scales differ by large factors: in the dims an outlier does not touch, the other
tokens carry the result, and the outlier's scale must take no bits from them.  Element by element against 64 bits
on the stored bytes, with the bound of an equal-scale decode (every weight rounded once to fp16)."""
import numpy as np
import pytest

import rows_oracle as ro
from test_block_scales_gpu import FP8, bind, pools, random_cache, want_decode
from test_qkv_rows_gpu import paged

pytestmark = pytest.mark.gpu


def outlier_rows(rng, lens, hq, hkv, at, power, share, one_sign):
    """q, and k, v per sequence: token `at` has one V element 2^power times the size of all others and `share` of the
    attention of every head."""
    group = hq // hkv
    top = min(2.0 ** 15, 2.0 ** power)
    q = np.repeat(rng.standard_normal((len(lens), hkv, 1, 128)), group, 2)
    q = (q + 0.05 * rng.standard_normal(q.shape)).reshape(len(lens), hq, 128).astype(np.float16)
    ks, vs = [], []
    for b, n in enumerate(lens):
        k = rng.standard_normal((n, hkv, 128)) * 0.3
        v = (0.9 + 0.02 * rng.standard_normal(k.shape) if one_sign else rng.standard_normal(k.shape)) * top / 2.0 ** power
        i = at % n
        for h in range(hkv):
            lead = q[b, h * group].astype(np.float64)
            s = k[:, h] @ lead / np.sqrt(128)
            s[i] = -np.inf
            want = np.log(np.exp(s - s.max()).sum()) + s.max() + np.log(share / (1 - share)) if n > 1 else 0.0
            k[i, h] = lead * want * np.sqrt(128) / (lead @ lead)
            v[i, h, 7 + h] = top
        ks.append(k)
        vs.append(v)
    return q, ks, vs


def check(torch, pa, q, kc, vc, scales, table, lens, ps, ctas):
    hq, (pages, hkv) = q.shape[1], kc.shape[:2]
    want, tol = want_decode(q, (kc.cpu().numpy(), vc.cpu().numpy()), scales.cpu().numpy(), table, lens, ps)
    dq, d_table = torch.from_numpy(q).cuda(), torch.from_numpy(table).cuda()
    d_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    mode = pa.head_fused()
    try:
        for fused, device_plan in ((0, False), (2, False), (2, True)):
            pa.set_head_fused(fused)
            out = torch.full_like(dq, float("nan"))
            p, dp = bind(torch, pa, dq, out, kc, vc, d_table, d_lens, lens, hq, hkv, ps, ctas, device_plan)
            pa.paged_decode(FP8, p, 0, pages, d_block_scales=scales)
            assert pa.kernel_status() == 0
            err = np.abs(out.double().cpu().numpy() - want)
            assert (err <= tol).all(), (fused, device_plan, (err / tol).max())
    finally:
        pa.set_head_fused(mode)


@pytest.mark.parametrize("power, share", [(4, 0.5), (7, 0.5), (10, 0.5), (12, 0.1), (12, 0.5), (14, 0.9), (18, 0.5), (28, 0.5),
                                          # an outlier that counts although it has next to no share
                                          (18, 2.0 ** -17), (28, 2.0 ** -27), (28, 2.0 ** -35)])
@pytest.mark.parametrize("one_sign", [False, True])
@pytest.mark.parametrize("ps, hq, hkv, lens, at, ctas", [
    (16, 32, 8, [4096, 40, 1], 5, 0), (64, 8, 8, [1500, 700], 900, 3), (16, 8, 1, [2000], 1999, 1), (24, 16, 8, [500, 77], 12, 2), (8, 4, 4, [333], 100, 0),
    (4, 8, 8, [200, 31], 17, 1), (2, 8, 2, [150], 3, 0), (5, 16, 8, [130, 64], 33, 0)])
def test_an_outlier_takes_no_bits(ps, hq, hkv, lens, at, ctas, power, share, one_sign, torch_cuda, pa):
    """The cache is filled by the append, which gives the outlier's block its large scale."""
    torch = torch_cuda
    rng = np.random.default_rng(power * 100 + ps)
    table, pages = paged(rng, lens, ps)
    q, ks, vs = outlier_rows(rng, lens, hq, hkv, at, power, share, one_sign)
    kc, vc, scales = pools(torch, pages, hkv, ps)
    rows = [torch.from_numpy(np.concatenate(x)).half().cuda() for x in (ks, vs)]
    begin = torch.from_numpy(np.cumsum([0] + lens).astype(np.int32)).cuda()
    t = pa.append_target(kc, vc, torch.from_numpy(table).cuda(), torch.zeros(len(lens), dtype=torch.int32, device="cuda"), begin, d_block_scales=scales)
    pa.append_qkv(FP8, pa.qkv_params(None, *rows), None, t, None)
    check(torch, pa, q, kc, vc, scales, table, lens, ps, ctas)


@pytest.mark.parametrize("power_of_two", [True, False])
@pytest.mark.parametrize("ps, hq, hkv, lens, ctas", [(16, 32, 8, [1, 17, 1000], 0), (24, 16, 8, [333, 5], 1), (4, 8, 2, [250], 0), (1, 8, 8, [77, 32], 0), (6, 64, 8, [99], 3)])
def test_scales_all_over_the_range(ps, hq, hkv, lens, ctas, power_of_two, torch_cuda, pa):
    """V scales anywhere in what the append writes, 2^-32 .. 2^8, neighbours included, and scales of the caller's own that are
    no powers of two; in half of the dims only the blocks of small scales have bytes."""
    torch = torch_cuda
    rng = np.random.default_rng(ps * 3 + power_of_two)
    table, pages, bytes_, scales = random_cache(rng, lens, hkv, ps, 1)
    e = rng.uniform(-32, 8, scales.shape[:3])
    scales[..., 1] = 2.0 ** np.floor(e) if power_of_two else 2.0 ** e
    if not power_of_two:
        scales[..., 0] *= rng.uniform(0.5, 2, scales.shape[:3])
    token_scale = np.repeat(scales[..., 1], ro.block_tokens(ps), axis=2)
    bytes_[1][..., :64][token_scale > 2.0 ** -12] = 0
    q = rng.standard_normal((len(lens), hq, 128)).astype(np.float16)
    check(torch, pa, q, *(torch.from_numpy(x).cuda() for x in (*bytes_, scales)), table, lens, ps, ctas)


@pytest.mark.parametrize("ps, hq, hkv, lens, ctas", [(16, 32, 8, [100, 700, 16], 0), (8, 8, 4, [77, 300], 3), (3, 16, 8, [40, 2], 0)])
def test_scale_zero_and_scales_far_outside_the_appends_range(ps, hq, hkv, lens, ctas, torch_cuda, pa):
    """Blocks of scale 0 count as zeros whatever their bytes; blocks of huge scales whose V bytes are zeros take no bits either; V
    scales that fp16 outputs cannot show."""
    torch = torch_cuda
    rng = np.random.default_rng(ps)
    table, pages, bytes_, scales = random_cache(rng, lens, hkv, ps, 1)
    kind = rng.integers(0, 5, scales.shape[:3])
    scales[kind == 0] = 0
    scales[..., 1][kind == 1] = 2.0 ** rng.uniform(20, 125, (kind == 1).sum())
    scales[..., 1][kind == 2] = 2.0 ** rng.uniform(-120, -33, (kind == 2).sum())
    bytes_[1][np.repeat(kind, ro.block_tokens(ps), axis=2) == 1] = 0
    q = rng.standard_normal((len(lens), hq, 128)).astype(np.float16)
    check(torch, pa, q, *(torch.from_numpy(x).cuda() for x in (*bytes_, scales)), table, lens, ps, ctas)
