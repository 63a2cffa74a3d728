"""Refusals and host logic of the row operators, without a GPU."""
import ctypes as C

import numpy as np
import pytest

import rows_oracle as ro


def rows(pa, **kw):
    x = pa.QKVParams()
    x.q, x.k, x.v = 1 << 20, 2 << 20, 3 << 20
    x.num_tokens, x.num_q_heads, x.num_kv_heads, x.head_dim, x.eps = 5, 8, 2, 128, 1e-6
    for k, v in kw.items():
        setattr(x, k, v)
    return x


def target(pa, **kw):
    t = pa.AppendTarget()
    t.k_cache, t.v_cache, t.block_table, t.start_pos = 4 << 20, 5 << 20, 6 << 20, 7 << 20
    t.k_scale = t.v_scale = 1.0
    t.block_table_stride, t.num_slots, t.batch, t.num_pages, t.page_size = 4, 5, 5, 20, 16
    for k, v in kw.items():
        setattr(t, k, v)
    return t


@pytest.mark.parametrize("args", [
    dict(inv_freq=[1.0] * 7), dict(inv_freq=[1.0] * 4), dict(inv_freq=[1.0] * 72), dict(inv_freq=[]),
    dict(inv_freq=[1.0] * 63 + [np.inf]), dict(inv_freq=[1.0] * 63 + [np.nan]), dict(inv_freq=[1e7] * 64),
    dict(inv_freq=[1.0] * 64, axes=[0] * 63 + [4]), dict(inv_freq=[1.0] * 64, axes=[-1] * 64),
    dict(inv_freq=[1.0] * 64, axes=[0] * 32), dict(inv_freq=[1.0] * 64, scale=np.nan), dict(inv_freq=np.ones((2, 32)))])
def test_rope_refusals(args, pa):
    with pytest.raises(pa.InvalidArgument):
        pa.Rope(**args)


def test_rope_accepts(pa):
    for r in range(16, 129, 16):
        pa.Rope.with_base(500000.0, r, interleaved=True, axes=[i % 4 for i in range(r // 2)], scale=0.5)
    pa.Rope([-1.0, 0.0, 6.283185307179586, 1e6, 0.5, 0.25, 0.125, 3.0])


@pytest.mark.parametrize("bad, match", [
    (dict(act_dtype=2), "dtype"), (dict(head_dim=64), "head_dim"), (dict(num_tokens=-1), "count"), (dict(num_q_heads=-1), "count"),
    (dict(q=None), "q is null"), (dict(k=None), "k is null"), (dict(q=(1 << 20) + 8), "aligned"), (dict(q_stride=8 * 128 + 4), "multiples"),
    (dict(q_stride=7 * 128), "at least"), (dict(k_stride=-256), "at least"), (dict(q_norm=8), "aligned"),
    (dict(q_norm=16, eps=-1.0), "eps"), (dict(k_norm=16, eps=float("nan")), "eps"), (dict(positions=None), "positions"), (dict(positions=(1 << 16) + 2), "aligned"),
    (dict(num_axes=1, axes3=True), "axes"), (dict(num_axes=3, positions_stride=4, axes3=True), "positions_stride")])
def test_qk_norm_rope_refusals(bad, match, pa):
    bad = dict(dict(positions=1 << 16, num_axes=1, positions_stride=5), **bad)
    rope = pa.Rope.with_base(axes=[i % 3 for i in range(64)] if bad.pop("axes3", False) else None)
    with pytest.raises(pa.InvalidArgument, match=match):
        pa.qk_norm_rope(rows(pa, **bad), rope, 8 << 20, 9 << 20)


def test_qk_norm_rope_output_refusals(pa):
    x = rows(pa, q_stride=12 * 128)
    for q_out, k_out in ((None, 9 << 20), (8 << 20, None), ((8 << 20) + 4, 9 << 20), (x.q, 9 << 20)):   # the last: in place, other stride
        with pytest.raises(pa.InvalidArgument):
            pa.qk_norm_rope(x, None, q_out, k_out)
    pa.qk_norm_rope(rows(pa, num_tokens=0), None, None, None)                       # nothing to do
    pa.qk_norm_rope(rows(pa, num_q_heads=0, num_kv_heads=0), None, None, None)


@pytest.mark.parametrize("bad, match", [
    (dict(page_size=0), "positive"), (dict(num_pages=0), "positive"), (dict(num_slots=0), "positive"), (dict(block_table_stride=0), "positive"),
    (dict(batch=-1), "positive"), (dict(k_cache=None), "null"), (dict(block_table=None), "null"), (dict(start_pos=None), "null"),
    (dict(v_cache=(5 << 20) + 8), "aligned"), (dict(k_scale=0.0), "scales"), (dict(v_scale=float("nan")), "scales"),
    (dict(block_table=(6 << 20) + 1), "aligned"), (dict(token_begin=(6 << 20) + 2), "aligned"), (dict(d_v_scales=6), "aligned"),
    (dict(d_block_scales=1 << 16, d_k_scales=1 << 16), "exclude"), (dict(d_block_scales=(1 << 16) + 4), "aligned")])
def test_append_qkv_refusals(bad, match, pa):
    with pytest.raises(pa.InvalidArgument, match=match):
        pa.append_qkv(pa.KVDtype.FP8_E4M3, rows(pa), None, target(pa, **bad), 8 << 20)


def test_append_qkv_more_refusals(pa):
    with pytest.raises(pa.InvalidArgument, match="only an fp8"):
        pa.append_qkv(pa.KVDtype.FP16, rows(pa), None, target(pa, d_block_scales=1 << 16), 8 << 20)
    for x, out in ((rows(pa, v=None), 8 << 20), (rows(pa), None), (rows(pa, num_kv_heads=0), 8 << 20), (rows(pa), (8 << 20) + 2)):
        with pytest.raises(pa.InvalidArgument):
            pa.append_qkv(pa.KVDtype.FP16, x, None, target(pa), out)
    with pytest.raises(pa.InvalidArgument, match="dtype"):
        pa.append_qkv(7, rows(pa), None, target(pa), 8 << 20)
    pa.append_qkv(pa.KVDtype.FP16, rows(pa, num_tokens=0), None, target(pa), None)   # nothing to do
    pa.append_qkv(pa.KVDtype.FP16, rows(pa), None, target(pa, batch=0), 8 << 20)


def test_block_scaled_decode_refusals(pa):
    p = pa.DecodeParams()
    p.num_q_heads, p.num_kv_heads, p.head_dim, p.page_size = 8, 8, 128, 16
    for dtype, pages, scales in ((pa.KVDtype.FP16, 4, 1 << 16), (pa.KVDtype.FP8_E4M3, 0, 1 << 16), (pa.KVDtype.FP8_E4M3, 4, (1 << 16) + 4)):
        with pytest.raises(pa.InvalidArgument):
            pa.paged_decode(dtype, p, 0, pages, d_block_scales=scales)
    with pytest.raises(pa.InvalidArgument, match="exclude"):
        pa.paged_decode(pa.KVDtype.FP8_E4M3, p, 0, 4, d_k_scales=16, d_block_scales=1 << 16)


def test_scale_block_tokens(pa):
    for ps in list(range(1, 130)) + [256, 1000]:
        b = pa.scale_block_tokens(ps)
        assert b == ro.block_tokens(ps) and ps % b == 0 and 1 <= b <= 16
    assert pa.scale_block_tokens(0) == 0


def test_builders_check_their_tensors(pa):
    torch = pytest.importorskip("torch")
    h = lambda *s, dtype=torch.float16: torch.zeros(*s, dtype=dtype)   # noqa: E731
    for kw in (dict(q=h(3, 4, 64), k=h(3, 2, 64)), dict(q=h(2, 4, 128), k=h(3, 2, 128)), dict(q=h(3, 4, 128, dtype=torch.bfloat16), k=h(3, 2, 128)),
               dict(q=None, k=h(3, 2, 128, dtype=torch.float32)), dict(q=None, k=h(3, 2, 256)[:, :, ::2]), dict(q=None, k=h(3, 4, 128)[:, ::2]),
               dict(q=None, k=h(3, 2, 128), v=h(3, 1, 128)), dict(q=None, k=h(3, 2, 128), k_norm=h(128, dtype=torch.float32)),
               dict(q=None, k=h(3, 2, 128), positions=torch.zeros(3)), dict(q=None, k=h(3, 2, 128), positions=torch.zeros(2, dtype=torch.int32)),
               dict(q=None, k=h(1, 2, 128).expand(3, 2, 128)), dict(q=h(3, 4, 128), k=h(3, 1, 128).expand(3, 2, 128)),
               dict(q=None, k=h(3, 2, 128), positions=torch.zeros(1, 3, dtype=torch.int32).expand(2, 3)),
               dict(q=None, k=h(3, 2, 128))):                                   # the last: not on a GPU
        with pytest.raises(pa.InvalidArgument):
            pa.qkv_params(**kw)


def test_struct_layouts(pa):
    assert C.sizeof(pa.QKVParams) == 3 * 8 + 3 * 8 + 3 * 8 + 8 + 6 * 4 + 4 + 4 and C.sizeof(pa.AppendTarget) == 9 * 8 + 2 * 4 + 5 * 4 + 4


def test_oracle_e4m3_table():
    torch = pytest.importorskip("torch")
    want = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    got = ro.decode_e4m3(np.arange(256))
    assert np.array_equal(got, want, equal_nan=True)
    assert ro.need_scale(448.0) == 1.0 and ro.need_scale(448.0000001) == 2.0 and ro.need_scale(0.0) == 2.0 ** -32 and ro.need_scale(1e30) == 256.0


def test_oracle_e4m3_rounding():
    torch = pytest.importorskip("torch")
    x = np.concatenate([np.linspace(0, 0.05, 2001), np.linspace(0, 447, 4001), (ro.e4m3_values()[1:] + ro.e4m3_values()[:-1]) / 2])
    x = x.astype(np.float32).astype(np.float64)
    assert np.array_equal(ro.round_e4m3(x), torch.from_numpy(x).to(torch.float32).to(torch.float8_e4m3fn).double().numpy())


def test_outputs_are_checked(pa):
    torch = pytest.importorskip("torch")
    x = rows(pa, num_tokens=3, num_q_heads=2, positions=1 << 16, num_axes=1)
    x._dtype = torch.float16
    h = lambda *s, dtype=torch.float16: torch.zeros(*s, dtype=dtype)   # noqa: E731
    k = 9 << 20
    for q in (h(3, 2, 64), h(2, 2, 128), h(3, 2, 128, dtype=torch.bfloat16), h(1, 2, 128).expand(3, 2, 128), h(3, 1, 128).expand(3, 2, 128),
              h(3, 4, 128)[:, ::2], h(3, 2, 256)[:, :, ::2]):
        with pytest.raises(pa.InvalidArgument):
            pa.qk_norm_rope(x, None, q, k)
    for q in (h(3, 2, 64), h(4, 2, 128), h(3, 2, 128, dtype=torch.bfloat16), h(3, 4, 128)[:, :2]):
        with pytest.raises(pa.InvalidArgument):
            pa.append_qkv(pa.KVDtype.FP16, x, None, target(pa), q)
