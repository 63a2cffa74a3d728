"""The block-scaled e4m3 cache: appends (blocks begun by one call and continued by others, scales that grow) and decode,
against 64-bit forms."""
import numpy as np
import pytest

import rows_oracle as ro
from common import device_view
from test_qkv_rows_gpu import Rows, assert_rows, paged, STEP

pytestmark = pytest.mark.gpu

FP8 = 1


def pools(torch, pages, hkv, ps):
    b = ro.block_tokens(ps)
    kc, vc = (torch.full((pages, hkv, ps, 128), 0x11, dtype=torch.uint8, device="cuda") for _ in range(2))
    return kc, vc, torch.zeros(pages, hkv, ps // b, 2, device="cuda")


def check_pools(kc, vc, scales, models, written):
    """Scales equal; every written value within its bound; every other byte as it was."""
    s = scales.cpu().numpy().astype(np.float64)
    for which, (pool, m) in enumerate(zip((kc, vc), models)):
        assert np.array_equal(s[..., which], m.scale), "scales differ"
        raw = pool.cpu().numpy()
        per_token = np.repeat(m.scale, m.b, axis=2)[..., None]
        err = np.abs(ro.decode_e4m3(raw) * per_token - np.clip(m.x, -448 * per_token, 448 * per_token))
        live = written[:, None, :, None] & np.ones_like(err, bool)
        assert (err[live] <= m.off[live]).all(), (err[live] / m.off[live]).max()
        assert (ro.decode_e4m3(raw) == m.slack[..., None])[~live].all()


def append_calls(torch, pa, ps, hkv, act, calls):
    """One append per entry of `calls` (new tokens of each sequence), then everything the pools and scales hold."""
    rng = np.random.default_rng(ps * 31 + hkv)
    total = np.sum(calls, 0)
    table, pages = paged(rng, total, ps)
    kc, vc, scales = pools(torch, pages, hkv, ps)
    models = [ro.BlockPool(pages, hkv, ps) for _ in range(2)]
    written = np.zeros((pages, ps), bool)
    past = np.zeros(len(total), int)
    d_table = torch.from_numpy(table).cuda()
    for call, new in enumerate(calls):
        tokens = sum(new)
        place = np.concatenate([np.arange(p, p + n) for n, p in zip(new, past)] + [np.zeros(2, int)])
        w = Rows(torch, pa, tokens + 2, 4, hkv, act=act, norm=call % 2 == 0, r=(128, 64)[call % 3 == 1], interleaved=call % 2 == 1, seed=call)
        grow = torch.tensor(2.0 ** rng.integers(-6, 7, (w.tokens, hkv, 1)), device="cuda").to(w.dt)     # magnitudes that jump from token to token
        w.v.mul_(grow)
        if call % 2:
            w.k.mul_(grow.flip(0))
        one_each = all(n == 1 for n in new)
        begin = torch.from_numpy(np.cumsum([0] + list(new)).astype(np.int32)).cuda()
        t = pa.append_target(kc, vc, d_table, torch.from_numpy(past.astype(np.int32)).cuda(), None if one_each else begin, d_block_scales=scales)
        q_out = torch.full((w.tokens, 4, 128), 9.0, dtype=torch.float16, device="cuda")
        pa.append_qkv(FP8, w.params(), w.rope, t, q_out)
        assert pa.kernel_status() == 0
        q, sq = w.want(w.q, w.wq, place)
        assert_rows(q_out[:tokens], q[:tokens], sq[:tokens], *STEP["fp16"])
        assert (q_out[tokens:] == 9).all()
        k, size = w.want(w.k, w.wk, place)
        v = w.v.double().cpu().numpy()
        at = 0
        for b, n in enumerate(new):
            models[0].append(table[b], past[b], k[at:at + n], ro.rows_bound(k, size, 0, 0)[at:at + n])
            models[1].append(table[b], past[b], v[at:at + n], np.zeros_like(v[at:at + n]))
            for p in range(past[b], past[b] + n):
                written[table[b, p // ps], p % ps] = True
            at += n
        past = past + np.asarray(new)
    check_pools(kc, vc, scales, models, written)


@pytest.mark.parametrize("ps, hkv, act, calls", [
    # calls: lists of (new tokens per sequence), one append each
    (16, 8, "fp16", [[1, 1, 1]] * 20), (16, 8, "bf16", [[5, 40, 0], [1, 7, 3], [33, 1, 64]]), (16, 2, "fp16", [[100, 3, 17]]),
    (64, 1, "bf16", [[10, 64, 70], [60, 1, 1], [300, 0, 2]]), (24, 3, "fp16", [[5, 9, 30], [4, 40, 1]]), (1, 2, "fp16", [[3, 1, 0], [1, 1, 1]]),
    (5, 2, "bf16", [[3, 6, 11], [9, 1, 1]]), (8, 4, "fp16", [[2, 3, 4]] * 5), (6, 5, "fp16", [[7, 1, 2], [2, 2, 2]]), (256, 8, "bf16", [[700, 15, 250], [3, 300, 9]]),
    (16, 16, "fp16", [[0, 2, 0], [0, 0, 1], [16, 15, 14]])])
def test_append_blocks(ps, hkv, act, calls, torch_cuda, pa):
    append_calls(torch_cuda, pa, ps, hkv, act, calls)


@pytest.mark.parametrize("seed", range(16))
def test_append_blocks_random(seed, torch_cuda, pa):
    rng = np.random.default_rng(900 + seed)
    ps = int(rng.choice([1, 2, 4, 7, 8, 12, 16, 16, 16, 20, 32, 48, 128]))
    batch, top = int(rng.integers(1, 40)), int(rng.choice([1, 2, 10, 17, 90]))
    calls = [rng.integers(0 if top > 1 else 1, top + 1, batch).tolist() for _ in range(int(rng.integers(1, 6)))]
    calls.append([1] * batch)
    append_calls(torch_cuda, pa, ps, int(rng.integers(1, 10)), str(rng.choice(["fp16", "bf16"])), calls)


def test_a_reused_page_forgets_its_scale(torch_cuda, pa):
    """A block whose first token is new takes the new tokens' scale, whatever was there; appending the same rows again
    leaves the same bytes."""
    torch = torch_cuda
    kc, vc, scales = pools(torch, 2, 2, 16)
    scales.fill_(2.0 ** 7)
    w = Rows(torch, pa, 18, 2, 2, norm=False)
    t = pa.append_target(kc, vc, torch.tensor([[1, 0]], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"),
                         torch.tensor([0, 18], dtype=torch.int32, device="cuda"), d_block_scales=scales)
    q_out = torch.zeros(18, 2, 128, dtype=torch.float16, device="cuda")
    pa.append_qkv(FP8, w.params(), w.rope, t, q_out)
    assert (scales < 1).all()
    first = [x.clone() for x in (kc, vc, scales)]
    pa.append_qkv(FP8, w.params(), w.rope, t, q_out)
    assert all(torch.equal(x, y) for x, y in zip(first, (kc, vc, scales)))


def test_extreme_values(torch_cuda, pa):
    """Zeros, the largest and smallest numbers, infinities (saturate) and NaN (stay NaN, do not move the scale)."""
    torch = torch_cuda
    kc, vc, scales = pools(torch, 8, 1, 16)
    v = torch.zeros(128, 1, 128, dtype=torch.bfloat16, device="cuda")
    v[16:32] = 3.0e38
    v[32:48] = 1e-30
    v[48:64, 0, 5] = float("inf")
    v[64:80] = 1.0
    v[70, 0, 9] = float("nan")
    v[80:96] = 448.0
    v[96:112] = -450.0
    v[112:128] = 2.0 ** -24 * 448
    x = pa.qkv_params(None, v, v)
    t = pa.append_target(kc, vc, torch.arange(8, dtype=torch.int32, device="cuda")[None].contiguous(), torch.zeros(1, dtype=torch.int32, device="cuda"),
                         torch.tensor([0, 128], dtype=torch.int32, device="cuda"), d_block_scales=scales)
    pa.append_qkv(FP8, x, None, t, None)
    assert scales[:, 0, 0, 1].tolist() == [2.0 ** -32, 256.0, 2.0 ** -32, 256.0, 2.0 ** -8, 1.0, 2.0, 2.0 ** -24]
    assert torch.equal(scales[..., 0], scales[..., 1]) and torch.equal(kc, vc)
    val = ro.decode_e4m3(vc.cpu().numpy())
    assert (val[0] == 0).all() and (val[1] == 448).all() and (val[2] == 0).all()
    assert (val[3, 0, :, 5] == 448).all() and (val[3, 0, :, 6] == 0).all()
    assert np.isnan(val[4, 0, 6, 9]) and np.isnan(val[4]).sum() == 1 and val[4, 0, 0, 0] == 256.0
    assert (val[5] == 448).all() and (val[6] == -224).all() and (val[7] == 448).all()


def random_cache(rng, lens, hkv, ps, spread):
    """Bytes and scales of a filled cache; V scales differ by up to 2^(2 spread) between blocks."""
    table, pages = paged(rng, lens, ps)
    b = ro.block_tokens(ps)
    raw = rng.standard_normal((2, pages, hkv, ps, 128)) * 90
    bytes_ = encode(raw)
    scales = np.empty((pages, hkv, ps // b, 2), np.float32)
    scales[..., 0] = 2.0 ** rng.integers(-8, -5, scales.shape[:3])
    scales[..., 1] = 2.0 ** rng.integers(-7 - spread, -6 + spread, scales.shape[:3])
    return table, pages, bytes_, scales


def encode(x):
    import torch
    return torch.from_numpy(np.clip(x, -448, 448)).float().to(torch.float8_e4m3fn).view(torch.uint8).numpy()


def want_decode(q, bytes_, scales, table, lens, ps):
    k, v = (ro.decode_e4m3(b) * np.repeat(scales[..., i].astype(np.float64), ro.block_tokens(ps), axis=2)[..., None] for i, b in enumerate(bytes_))
    outs, tols = [], []
    for i, n in enumerate(lens):
        t = np.arange(n)
        page, off = table[i, t // ps], t % ps
        o, tol = ro.attention(q[i].astype(np.float64), k[page, :, off], v[page, :, off], 1 / np.sqrt(np.float32(128)))
        outs.append(o)
        tols.append(tol)
    return np.array(outs), np.array(tols)


def bind(torch, pa, dq, out, kc, vc, d_table, d_lens, lens, hq, hkv, ps, ctas=0, device_plan=False):
    dp = pa.DevicePlan()
    if device_plan:
        dp.build(FP8, d_lens, len(lens), hq, hkv, 128, ctas)
    else:
        dp.upload(pa.make_plan(FP8, lens, hq, hkv, 128, ctas), hq // hkv, 128)
    p = pa.DecodeParams()
    p.q, p.out, p.k_cache, p.v_cache = dq.data_ptr(), out.data_ptr(), kc.data_ptr(), vc.data_ptr()
    p.block_table, p.seq_lens, p.block_table_stride = d_table.data_ptr(), d_lens.data_ptr(), d_table.shape[1]
    p.batch, p.num_q_heads, p.num_kv_heads, p.head_dim, p.page_size = len(lens), hq, hkv, 128, ps
    p.sm_scale = 1.0 / float(np.sqrt(np.float32(128)))
    p.k_scale = p.v_scale = float("nan")            # not used
    dp.bind(p)
    return p, dp


DECODES = [
    # page, hq, hkv, lens, ctas, spread of V scales
    (16, 32, 8, [1, 2, 15, 16, 17, 31, 33, 127, 128, 129, 500], 0, 1), (16, 8, 8, [1000, 3], 37, 1), (16, 8, 1, [700, 1, 40], 0, 6),
    (16, 64, 8, [300, 77], 5, 1), (32, 16, 8, [1, 64, 999], 0, 3), (64, 4, 4, [65, 400], 11, 1), (128, 8, 2, [129, 1], 0, 1), (256, 32, 8, [500, 3, 256], 0, 1),
    (8, 32, 8, [9, 100, 333], 0, 2), (24, 16, 8, [25, 130, 1], 0, 1), (1, 8, 8, [5, 77, 1], 0, 1), (1, 16, 2, [3, 40], 0, 1), (2, 16, 8, [33, 2], 0, 1), (3, 8, 1, [50, 7], 0, 1),
    (5, 64, 8, [61, 130], 0, 2), (4, 8, 4, [129, 5], 0, 1), (100, 16, 16, [101, 350], 0, 1), (16, 32, 4, [9000], 0, 1), (48, 2, 2, [1500], 200, 8)]


@pytest.mark.parametrize("case", DECODES, ids=lambda c: "ps%d-%dx%d-%s-c%d-s%d" % (c[0], c[1], c[2], "_".join(map(str, c[3])), c[4], c[5]))
def test_decode_block_scaled(case, torch_cuda, pa):
    torch = torch_cuda
    ps, hq, hkv, lens, ctas, spread = case
    rng = np.random.default_rng(hq * 7 + ps)
    table, pages, bytes_, scales = random_cache(rng, lens, hkv, ps, spread)
    q = rng.standard_normal((len(lens), hq, 128)).astype(np.float16)
    want, tol = want_decode(q, bytes_, scales, table, lens, ps)
    # what no token of a sequence covers must not matter: NaN bytes, scales that are NaN, zero, negative
    used = np.zeros((pages, ps), bool)
    for i, n in enumerate(lens):
        t = np.arange(n)
        used[table[i, t // ps], t % ps] = True
    for b in bytes_:
        b.transpose(0, 2, 1, 3)[~used] = 0x7f
    dead = ~used.reshape(pages, -1, ro.block_tokens(ps)).any(-1)
    scales.transpose(0, 2, 1, 3)[dead] = rng.choice(np.array([np.nan, 0, -1, np.inf], np.float32), (int(dead.sum()), hkv, 2))
    kc, vc = (torch.from_numpy(b).cuda() for b in bytes_)
    d_scales, d_table = torch.from_numpy(scales).cuda(), torch.from_numpy(table).cuda()
    dq, d_lens = torch.from_numpy(q).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")
    mode = pa.head_fused()
    try:
        for fused, device_plan in ((0, False), (2, False), (2, True)):
            pa.set_head_fused(fused)
            out = torch.full_like(dq, float("nan"))
            p, dp = bind(torch, pa, dq, out, kc, vc, d_table, d_lens, lens, hq, hkv, ps, ctas, device_plan)
            pa.paged_decode(FP8, p, 0, pages, d_block_scales=d_scales)
            assert pa.kernel_status() == 0
            err = np.abs(out.double().cpu().numpy() - want)
            assert (err <= tol).all(), (fused, device_plan, (err / tol).max())
    finally:
        pa.set_head_fused(mode)


def test_equal_scales_are_the_per_tensor_decode(torch_cuda, pa):
    """One power-of-two scale everywhere: the same numbers as k_scale / v_scale, up to the outputs' rounding."""
    torch = torch_cuda
    rng = np.random.default_rng(5)
    lens = [300, 1, 4000, 129]
    table, pages, bytes_, scales = random_cache(rng, lens, 8, 16, 1)
    kc, vc = (torch.from_numpy(b).cuda() for b in bytes_)
    dq = torch.from_numpy(rng.standard_normal((4, 32, 128)).astype(np.float16)).cuda()
    d_lens, d_table = torch.tensor(lens, dtype=torch.int32, device="cuda"), torch.from_numpy(table).cuda()
    out, ref = torch.empty_like(dq), torch.empty_like(dq)
    p, dp = bind(torch, pa, dq, out, kc, vc, d_table, d_lens, lens, 32, 8, 16)
    pa.paged_decode(FP8, p, 0, pages, d_block_scales=torch.full((pages, 8, 1, 2), 2.0 ** -7, device="cuda"))
    p.out, p.k_scale, p.v_scale = ref.data_ptr(), 2.0 ** -7, 2.0 ** -7
    pa.paged_decode(FP8, p, 0, pages)
    # the same sums in fp32 with different roundings of the exponent, then one rounding each to fp16
    assert ((out - ref).abs() <= 2.0 ** -10 * ref.abs() + 2.0 ** -12).all()


def test_pages_outside_the_pool_read_as_zeros(torch_cuda, pa):
    """As with per-tensor scales: K and V of such a page are zeros, and its scales are not read."""
    torch = torch_cuda
    rng = np.random.default_rng(6)
    table, pages, bytes_, scales = random_cache(rng, [48], 8, 16, 1)
    q = rng.standard_normal((1, 32, 128)).astype(np.float16)
    bad = table[0, 1]
    zeroed = [b.copy() for b in bytes_]
    for b in zeroed:
        b[bad] = 0
    want, tol = want_decode(q, zeroed, scales, table, [48], 16)
    table[0, 1] = pages + 5
    kc, vc = (torch.from_numpy(b).cuda() for b in bytes_)
    dq, out = torch.from_numpy(q).cuda(), torch.empty(1, 32, 128, dtype=torch.float16, device="cuda")
    d_lens, d_table = torch.tensor([48], dtype=torch.int32, device="cuda"), torch.from_numpy(table).cuda()
    p, dp = bind(torch, pa, dq, out, kc, vc, d_table, d_lens, [48], 32, 8, 16)
    pa.paged_decode(FP8, p, 0, pages, d_block_scales=torch.from_numpy(scales).cuda())
    assert pa.kernel_status() == 0
    assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()


@pytest.mark.parametrize("blocks", [False, True])
def test_a_served_batch(blocks, torch_cuda, pa):
    """Prompts, then decode steps, through the cache object: append_qkv, plan, run; append and append_batch mixed in;
    a released slot's pages are used again.  Outputs against attention over what the appends were given."""
    torch = torch_cuda
    hq, hkv, ps = 32, 8, 16
    cfg = pa.PagedKVCache.Config(num_pages=60, page_size=ps, num_kv_heads=hkv, head_dim=128, max_slots=4, max_pages_per_slot=30,
                                 dtype=pa.KVDtype.FP8_E4M3 if blocks else pa.KVDtype.FP16)
    cache = pa.PagedKVCache(cfg)
    cache.shuffle_free_pages(3)
    assert cache.block_scales() is None
    if blocks:
        cache.set_block_scales()
        assert cache.block_scales()
    history = {}                                    # slot -> ([k], [v]) in float64

    def remember(slot, k, v):
        history.setdefault(slot, ([], []))
        history[slot][0].append(k)
        history[slot][1].append(v)

    def rows(slots, ns, seed):
        place = np.concatenate([np.arange(cache.seq_len(s), cache.seq_len(s) + n) for s, n in zip(slots, ns)])
        w = Rows(torch, pa, int(sum(ns)), hq, hkv, act="bf16" if seed % 2 else "fp16", seed=seed)
        q_out = torch.empty(w.tokens, hq, 128, dtype=torch.float16, device="cuda")
        assert cache.append_qkv(slots, ns, w.params(), w.rope, q_out)
        q, sq = w.want(w.q, w.wq, place)
        assert_rows(q_out, q, sq, *STEP["fp16"])
        k, v = w.want(w.k, w.wk, place)[0], w.v.double().cpu().numpy()
        at = 0
        for s, n in zip(slots, ns):
            remember(s, k[at:at + n], v[at:at + n])
            at += n
        return q_out

    def step(slots, seed):
        q = rows(slots, [1] * len(slots), seed)
        out = torch.full_like(q, float("nan"))
        cache.plan(slots, hq)
        cache.run(q, out)
        assert pa.kernel_status() == 0
        prm, b = cache.params(), ro.block_tokens(ps)
        shape, width = (cfg.num_pages, hkv, ps, 128), 1 if blocks else 2
        stored = [device_view(ptr, int(np.prod(shape)) * width, torch).cpu().numpy() for ptr in (prm.k_cache, prm.v_cache)]
        stored = [ro.decode_e4m3(x).reshape(shape) if blocks else x.view(np.float16).astype(np.float64).reshape(shape) for x in stored]
        if blocks:
            sc = device_view(cache.block_scales(), cfg.num_pages * hkv * 8, torch).cpu().numpy().view(np.float32).reshape(cfg.num_pages, hkv, 1, 2)
            stored = [x * sc[..., i, None] for i, x in enumerate(stored)]
        for i, s in enumerate(slots):
            at = np.arange(cache.seq_len(s))
            page = cache.block_table(s)[at // ps]
            k, v = (x[page, :, at % ps] for x in stored)
            for got, want in zip((k, v), history[s]):
                want = np.concatenate(want)
                # one rounding of the cache's type, in e4m3 relative to the block's largest value below its normal range
                # (2^-10 of the scale, which is below max / 224), re-encoded at most a few times
                bound = 1.1 * np.abs(want) * 2.0 ** -4 + np.abs(want).max() * 2.0 ** -15 if blocks else np.abs(want) * 2.0 ** -10 + 1e-5
                assert len(want) == len(got) and (np.abs(got - want) <= bound).all()
            want, tol = ro.attention(q[i].double().cpu().numpy(), k, v, 1 / np.sqrt(np.float32(128)))
            assert (np.abs(out[i].double().cpu().numpy() - want) <= tol).all()
        return out

    slots = [cache.admit() for _ in range(3)]
    rows(slots, [37, 1, 100], 1)
    for i in range(18):
        step(slots, 2 + i)
    # plain appends of rows that somebody else rotated
    k, v = (torch.randn(6, hkv, 128, device="cuda").half() for _ in range(2))
    assert cache.append(slots[1], k, v, 6)
    remember(slots[1], k.double().cpu().numpy(), v.double().cpu().numpy())
    assert cache.append_batch(slots[:2], [k, v], [v, k], [3, 5])
    remember(slots[0], k[:3].double().cpu().numpy(), v[:3].double().cpu().numpy())
    remember(slots[1], v[:5].double().cpu().numpy(), k[:5].double().cpu().numpy())
    step(slots, 40)
    cache.release(slots[2])
    history.pop(slots[2])
    slots[2] = cache.admit()
    rows([slots[2]], [90], 41)
    step([slots[2], slots[0]], 42)
    # all or nothing
    free, lens = cache.free_pages(), [cache.seq_len(s) for s in slots]
    w = Rows(torch, pa, 480 + 470, hq, hkv, seed=50)
    q_out = torch.empty(w.tokens, hq, 128, dtype=torch.float16, device="cuda")
    fits = [480 - lens[0], w.tokens - (480 - lens[0])]
    with pytest.raises(pa.LengthError):
        cache.append_qkv(slots[:2], fits, w.params(), w.rope, q_out)
    few = Rows(torch, pa, 4, hq, hkv, seed=52)
    for args in (([slots[0], slots[0]], [2, 2]), ([3], [4]), ([slots[0]], [1]), ([], []), ([slots[0]], [-4]), ([slots[0], 9], [4, 0])):
        with pytest.raises(pa.InvalidArgument):
            cache.append_qkv(*args, few.params(), few.rope, q_out[:4])
    for out in (q_out, q_out[:3], None):
        with pytest.raises(pa.InvalidArgument):
            cache.append_qkv([slots[0]], [4], few.params(), few.rope, out)
    w = Rows(torch, pa, 1200, hq, hkv, seed=51)
    q_out = torch.empty(w.tokens, hq, 128, dtype=torch.float16, device="cuda")
    room = [480 - n for n in lens]
    assert not cache.append_qkv(slots, [room[0], room[1], 1200 - room[0] - room[1]], w.params(), w.rope, q_out)
    assert cache.free_pages() == free and [cache.seq_len(s) for s in slots] == lens
    step(slots, 43)
    cache.close()


def test_cache_scale_modes_exclude_each_other(torch_cuda, pa):
    torch = torch_cuda
    def cache(dtype):
        return pa.PagedKVCache(pa.PagedKVCache.Config(4, 16, 2, 128, 2, 2, dtype))
    c = cache(pa.KVDtype.FP16)
    with pytest.raises(pa.InvalidArgument):
        c.set_block_scales()
    c = cache(pa.KVDtype.FP8_E4M3)
    c.set_head_scales([1.0, 2.0], [1.0, 2.0])
    with pytest.raises(pa.InvalidArgument):
        c.set_block_scales()
    c.set_head_scales(None, None)
    c.set_block_scales()
    c.set_block_scales()                            # again: nothing to do
    with pytest.raises(pa.InvalidArgument):
        c.set_head_scales([1.0, 2.0], [1.0, 2.0])
    slot = c.admit()
    x = torch.ones(3, 2, 128, dtype=torch.float16, device="cuda")
    with pytest.raises(pa.InvalidArgument):
        c.append(slot, x.data_ptr() + 2, x, 1)
    assert c.seq_len(slot) == 0 and c.free_pages() == 4
    assert c.append(slot, x, x, 3)
    with pytest.raises(pa.InvalidArgument):
        c.set_block_scales(False)
    assert torch.equal(device_view(c.block_scales(), 4, torch).view(torch.float32).cpu(), torch.tensor([2.0 ** -8]))
    c.release(slot)
    c.set_block_scales(False)
    assert c.block_scales() is None


def test_decoder_binding(torch_cuda, pa):
    """The tensor binding takes the scales too, and checks them."""
    from paged_attention_b200.torch_decode import Decoder
    torch = torch_cuda
    rng = np.random.default_rng(9)
    lens = [70, 1, 333]
    table, pages, bytes_, scales = random_cache(rng, lens, 4, 32, 2)
    q = rng.standard_normal((3, 16, 128)).astype(np.float16)
    want, tol = want_decode(q, bytes_, scales, table, lens, 32)
    kc, vc = (torch.from_numpy(b).cuda() for b in bytes_)
    d_scales, d_lens = torch.from_numpy(scales).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")
    dec = Decoder(16, 4, 128, 32, True)
    dec.plan(torch.tensor(lens, dtype=torch.int32))
    args = (torch.from_numpy(q).cuda(), kc, vc, torch.from_numpy(table).cuda(), d_lens)
    out = dec.run(*args, block_scales=d_scales)
    assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()
    for bad in (d_scales[:1], d_scales.half(), d_scales.transpose(1, 2), d_scales.cpu()):
        with pytest.raises(TypeError):
            dec.run(*args, block_scales=bad)


def test_decode_replayed_in_a_graph_on_another_stream(torch_cuda, pa):
    """Append and decode captured together and replayed as the sequences grow: lengths, positions and the plan are read on
    the device."""
    torch = torch_cuda
    hq, hkv, ps, batch, steps = 8, 8, 16, 5, 40
    pages = batch * 4
    kc, vc, scales = pools(torch, pages, hkv, ps)
    table = torch.randperm(pages, device="cuda").to(torch.int32).view(batch, 4).contiguous()
    start = torch.tensor([0, 3, 15, 16, 9], dtype=torch.int32, device="cuda")
    # the tokens before: one ragged append
    first = Rows(torch, pa, int(start.sum()), hq, hkv, seed=1)
    begin = torch.zeros(batch + 1, dtype=torch.int32, device="cuda")
    begin[1:] = torch.cumsum(start, 0)
    pa.append_qkv(FP8, first.params(), first.rope, pa.append_target(kc, vc, table, torch.zeros_like(start), begin, d_block_scales=scales),
                  torch.empty(first.tokens, hq, 128, dtype=torch.float16, device="cuda"))
    w = Rows(torch, pa, batch, hq, hkv, seed=2)
    x, q = w.params(), torch.empty(batch, hq, 128, dtype=torch.float16, device="cuda")
    out, lens = torch.empty_like(q), torch.empty_like(start)
    target = pa.append_target(kc, vc, table, start, d_block_scales=scales)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()

    def step(p, dp):
        pa.append_qkv(FP8, x, w.rope, target, q, s.cuda_stream)
        torch.add(start, 1, out=lens)
        dp.build(FP8, lens, batch, hq, hkv, 128, 0, None, s.cuda_stream)
        dp.bind(p)
        pa.paged_decode(FP8, p, s.cuda_stream, pages, d_block_scales=scales)
        start.copy_(lens)

    with torch.cuda.stream(s):
        p, dp = bind(torch, pa, q, out, kc, vc, table, lens, [1] * batch, hq, hkv, ps)
        step(p, dp)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            step(p, dp)
    for i in range(steps):
        w.k.mul_(1.07)          # in place: the captured rows grow, and scales with them
        w.v.mul_(1.07)
        g.replay()
        if i % 13 == 0 or i == steps - 1:
            torch.cuda.synchronize()
            assert pa.kernel_status() == 0
            want, tol = want_decode(q.cpu().numpy(), (kc.cpu().numpy(), vc.cpu().numpy()), scales.cpu().numpy(), table.cpu().numpy(),
                                    lens.tolist(), ps)
            assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()
    assert lens.tolist() == [n + 1 + steps for n in [0, 3, 15, 16, 9]]


@pytest.mark.parametrize("hkv", [1, 3, 5])
def test_many_short_sequences_of_plain_rows(hkv, torch_cuda, pa):
    """Blocks of nine and more rows, several to a window of rows, neither normed nor rotated: pairs of warps meet over every
    (head, K or V) of one block after the other.  V scales are exact here, so every byte is determined."""
    torch = torch_cuda
    new = [9, 16, 12, 10, 9, 9, 15, 11] * 40
    g = torch.Generator(device="cuda").manual_seed(hkv)
    tokens = sum(new)
    k, v = (torch.randn(tokens, hkv, 128, generator=g, device="cuda").mul_(torch.exp2(torch.randint(-6, 7, (tokens, hkv, 1), generator=g, device="cuda"))).half()
            for _ in range(2))
    kc, vc, scales = pools(torch, len(new), hkv, 16)
    table = torch.randperm(len(new), generator=g, device="cuda").to(torch.int32)[:, None].contiguous()
    begin = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device="cuda")
    t = pa.append_target(kc, vc, table, torch.zeros(len(new), dtype=torch.int32, device="cuda"), begin, d_block_scales=scales)
    for _ in range(5):
        pa.append_qkv(FP8, pa.qkv_params(None, k, v), None, t, None)
    assert pa.kernel_status() == 0
    page, at = table[:, 0].tolist(), 0
    got_s = scales.cpu().numpy()
    for which, (pool, x) in enumerate(((kc, k), (vc, v))):
        raw, x64, at = pool.cpu().numpy(), x.double().cpu().numpy(), 0
        for p, n in zip(page, new):
            for h in range(hkv):
                s = ro.need_scale(np.abs(x64[at:at + n, h]).max())
                assert got_s[p, h, 0, which] == s
                assert np.array_equal(raw[p, h, :n], encode(x64[at:at + n, h] / s))
            at += n


def test_params_of_a_block_scaled_cache_do_not_fit_another_decode(torch_cuda, pa):
    torch = torch_cuda
    c = pa.PagedKVCache(pa.PagedKVCache.Config(4, 16, 8, 128, 2, 2, pa.KVDtype.FP8_E4M3))
    assert c.params().k_scale == 1.0
    c.set_block_scales()
    assert np.isnan(c.params().k_scale) and np.isnan(c.params().v_scale)


@pytest.mark.parametrize("blocks", [False, True])
def test_batches_on_alternating_streams(blocks, torch_cuda, pa):
    """Appends to one cache from two streams in turn, nothing waited for: each batch's lists are its own."""
    torch = torch_cuda
    hkv, slots, steps = 2, 24, 30
    c = pa.PagedKVCache(pa.PagedKVCache.Config(slots * 4, 16, hkv, 128, slots, 4, pa.KVDtype.FP8_E4M3 if blocks else pa.KVDtype.FP16))
    if blocks:
        c.set_block_scales()
    ids = [c.admit() for _ in range(slots)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    # token i of a slot is 2^(i % 5) everywhere: exact in every type and under every block's scale
    inputs = []
    for i in range(steps):
        x = torch.full((slots, hkv, 128), float(2 ** (i % 5)), dtype=torch.float16, device="cuda")
        inputs.append((x, pa.qkv_params(None, x, x)))
    torch.cuda.synchronize()
    for i, (x, p) in enumerate(inputs):
        order = ids if i % 3 else ids[::-1]
        assert c.append_qkv(order, [1] * slots, p, None, None, streams[i % 2].cuda_stream)
    torch.cuda.synchronize()
    assert pa.kernel_status() == 0
    prm = c.params()
    raw = device_view(prm.k_cache, slots * 4 * hkv * 16 * 128 * (1 if blocks else 2), torch).cpu().numpy()
    val = ro.decode_e4m3(raw) if blocks else raw.view(np.float16).astype(np.float64)
    val = val.reshape(slots * 4, hkv, 16, 128)
    if blocks:
        sc = device_view(c.block_scales(), slots * 4 * hkv * 8, torch).cpu().numpy().view(np.float32).reshape(slots * 4, hkv, 1, 2)
        val = val * sc[..., 0, None]
    want = 2.0 ** (np.arange(steps) % 5)
    for s in ids:
        at = np.arange(steps)
        got = val[c.block_table(s)[at // 16], :, at % 16]
        assert np.array_equal(got, np.broadcast_to(want[:, None, None], got.shape))


def test_calls_right_behind_one_another(torch_cuda, pa):
    """Each call reads what the one before it wrote - rows rotated in place, a block's scale and bytes, positions - with nothing
    in between; the same sequence with waits in between must leave the same bits."""
    torch = torch_cuda
    hq, hkv, batch, steps = 4, 2, 96, 48
    rng = np.random.default_rng(3)
    rows = torch.from_numpy(rng.standard_normal((steps, batch, hq + 2 * hkv, 128)) * 2.0 ** rng.integers(-5, 6, (steps, batch, 1, 1))).half().cuda()
    w = torch.rand(128, device="cuda").add_(0.5).half()
    rope = pa.Rope.with_base()
    results = []
    for wait in (True, False):
        x = rows.clone()
        kc, vc, scales = pools(torch, batch * 3, hkv, 16)
        table = torch.arange(batch * 3, dtype=torch.int32, device="cuda").view(batch, 3)
        starts = torch.arange(steps, dtype=torch.int32, device="cuda")[:, None].expand(steps, batch).contiguous()
        q = torch.zeros(steps, batch, hq, 128, dtype=torch.float16, device="cuda")
        calls = []
        for i in range(steps):
            r = x[i]
            first = pa.qkv_params(r[:, :hq], r[:, hq:hq + hkv], r[:, hq + hkv:], q_norm=w, k_norm=w, positions=starts[i])
            plain = pa.qkv_params(r[:, :hq], r[:, hq:hq + hkv], r[:, hq + hkv:])
            calls.append((first, plain, r, pa.append_target(kc, vc, table, starts[i], d_block_scales=scales)))
        torch.cuda.synchronize()
        for i, (first, plain, r, target) in enumerate(calls):
            pa.qk_norm_rope(first, rope, r[:, :hq], r[:, hq:hq + hkv])
            if wait:
                torch.cuda.synchronize()
            pa.append_qkv(FP8, plain, None, target, q[i])
            if wait:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        results.append((x, kc, vc, scales, q))
    assert pa.kernel_status() == 0
    for a, b in zip(*results):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_a_pool_past_32_bits(torch_cuda, pa):
    """Appends to and decode from the far end of pools of more than 2^32 bytes."""
    torch = torch_cuda
    hq, hkv, ps, pages, n = 16, 8, 16, 280000, 100           # 280000 * 8 * 16 * 128 = 4.6 GB
    kc, vc = (torch.zeros(pages, hkv, ps, 128, dtype=torch.uint8, device="cuda") for _ in range(2))
    scales = torch.zeros(pages, hkv, 1, 2, device="cuda")
    ids = [pages - 1 - 3 * i for i in range(7)]
    table = torch.tensor([ids], dtype=torch.int32, device="cuda")
    w = Rows(torch, pa, n, hq, hkv, seed=4)
    q = torch.zeros(n, hq, 128, dtype=torch.float16, device="cuda")
    start, begin = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.tensor([0, n], dtype=torch.int32, device="cuda")
    pa.append_qkv(FP8, w.params(), w.rope, pa.append_target(kc, vc, table, start, begin, d_block_scales=scales), q)
    dq, lens = q[-1:].contiguous(), torch.tensor([n], dtype=torch.int32, device="cuda")
    out = torch.zeros_like(dq)
    p, dp = bind(torch, pa, dq, out, kc, vc, table, lens, [n], hq, hkv, ps)
    pa.paged_decode(FP8, p, 0, pages, d_block_scales=scales)
    assert pa.kernel_status() == 0
    near = [x[torch.tensor(ids, device="cuda")].cpu().numpy() for x in (kc, vc, scales)]
    want, tol = want_decode(dq.cpu().numpy(), near[:2], near[2], np.arange(7, dtype=np.int32)[None], [n], ps)
    assert (np.abs(out.double().cpu().numpy() - want) <= tol).all() and np.abs(want).max() > 0.1
    k = w.want(w.k, w.wk, np.arange(n))[0]
    got = (ro.decode_e4m3(near[0]) * near[2][..., 0, None])[np.arange(n) // ps, :, np.arange(n) % ps]
    assert (np.abs(got - k) <= 1.1 * np.abs(k) * 2.0 ** -4 + np.abs(k).max() * 2.0 ** -15).all()


def test_schedule_of_few_long_rows(torch_cuda, pa):
    """16 rows cut in about ten pieces each: head-fused over a block-scaled cache, (row, kv head) otherwise; both right."""
    torch = torch_cuda
    rng = np.random.default_rng(12)
    lens = [2400 + 7 * i for i in range(16)]
    c = pa.PagedKVCache(pa.PagedKVCache.Config(16 * 160, 16, 8, 128, 16, 160, pa.KVDtype.FP8_E4M3))
    c.set_block_scales()
    ids = [c.admit() for _ in lens]
    tokens = sum(lens)
    k, v = (torch.randn(tokens, 8, 128, device="cuda").half() for _ in range(2))
    assert c.append_qkv(ids, lens, pa.qkv_params(None, k, v), None, None)
    q = torch.from_numpy(rng.standard_normal((16, 16, 128)).astype(np.float16)).cuda()
    outs = []
    mode = pa.head_fused()
    try:
        for m, schedule in ((1, "head-fused rows"), (0, "caller's plan")):
            pa.set_head_fused(m)
            c.plan(ids, 16)
            d = c.describe_launch()
            assert d["schedule"] == schedule
            out = torch.full_like(q, float("nan"))
            c.run(q, out)
            assert pa.kernel_status() == 0
            outs.append(out)
    finally:
        pa.set_head_fused(mode)
    p = c.params()
    raw = [device_view(ptr, 16 * 160 * 8 * 16 * 128, torch).cpu().numpy().reshape(16 * 160, 8, 16, 128) for ptr in (p.k_cache, p.v_cache)]
    sc = device_view(c.block_scales(), 16 * 160 * 8 * 8, torch).cpu().numpy().view(np.float32).reshape(16 * 160, 8, 1, 2)
    for row in (0, 7, 15):
        table = np.zeros((1, 160), np.int32)
        t = c.block_table(row)
        table[0, :len(t)] = t
        want, tol = want_decode(q[row:row + 1].cpu().numpy(), raw, sc, table, lens[row:row + 1], 16)
        for out in outs:
            assert (np.abs(out[row].double().cpu().numpy() - want[0]) <= tol[0]).all()
    # a per-tensor cache keeps its schedule
    pa.set_head_fused(1)
    plan = pa.make_plan(FP8, lens, 16, 8, 128)
    dp = pa.DevicePlan()
    dp.upload(plan, 2, 128)
    prm = pa.DecodeParams()
    prm.batch, prm.num_q_heads, prm.num_kv_heads, prm.head_dim, prm.page_size = 16, 16, 8, 128, 16
    dp.bind(prm)
    assert pa.describe_launch(FP8, prm)["schedule"] == "caller's plan"
    pa.set_head_fused(mode)
