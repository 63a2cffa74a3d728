"""The CTA shape of the e4m3 decode that a tuning build may set (PD_B200_NVCC_FLAGS): tiles of 256 tokens, which with pages of
four tokens and less have more boxes than the producer warp has lanes."""
import os
import subprocess
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))


def check():
    import torch
    import paged_attention_b200 as pa
    from test_block_scales_gpu import FP8, bind, random_cache, want_decode
    torch.cuda.set_device(0)
    pa.set_adaptive_cut(False)
    assert pa.tile_tokens(pa.KVDtype.FP8_E4M3, 128, 2) == 256
    rng = np.random.default_rng(1)
    lens, hq, hkv = [700, 256, 1, 333], 8, 4
    for ps in (16, 8, 4, 2, 1, 3, 12):
        table, pages, bytes_, scales = random_cache(rng, lens, hkv, ps, 1)
        q = rng.standard_normal((len(lens), hq, 128)).astype(np.float16)
        dq, d_lens, d_table = torch.from_numpy(q).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), torch.from_numpy(table).cuda()
        kc, vc = (torch.from_numpy(b).cuda() for b in bytes_)
        for blocks in (True, False):
            want, tol = want_decode(q, bytes_, scales if blocks else np.full_like(scales, 2.0 ** -7), table, lens, ps)
            out = torch.full_like(dq, float("nan"))
            p, dp = bind(torch, pa, dq, out, kc, vc, d_table, d_lens, lens, hq, hkv, ps)
            if blocks:
                pa.paged_decode(FP8, p, 0, pages, d_block_scales=torch.from_numpy(scales).cuda())
            else:
                p.k_scale = p.v_scale = 2.0 ** -7
                pa.paged_decode(FP8, p, 0, pages)
            assert pa.kernel_status() == 0
            err = np.abs(out.double().cpu().numpy() - want)
            assert (err <= tol).all(), (ps, blocks, (err / tol).max())


def test_tiles_of_more_boxes_than_lanes(tmp_path, monkeypatch, torch_cuda):
    from paged_attention_b200 import build
    lib = str(tmp_path / "libpd_b200.so")
    monkeypatch.setenv("PD_B200_NVCC_FLAGS", os.environ.get("PD_B200_NVCC_FLAGS", "") + " -DPD_B200_FP8_SHAPE=8221")
    build.build(out=lib)
    code = f"import sys; sys.path[:0] = [{os.path.dirname(HERE)!r}, {HERE!r}]; import test_tuned_shape_gpu; test_tuned_shape_gpu.check()"
    subprocess.run([sys.executable, "-c", code], env=dict(os.environ, PD_B200_LIB=lib), check=True, timeout=300)
