"""Norm + rotation of q / k rows, and the same on the way into the paged cache, against 64-bit forms element by element."""
import numpy as np
import pytest

import rows_oracle as ro

pytestmark = pytest.mark.gpu

FP16, FP8 = 0, 1
# half a step relative to the value, and half of the smallest number, of the row types
STEP = {"fp16": (2.0 ** -10, 2.0 ** -25), "bf16": (2.0 ** -7, 0.0)}


def freqs(r, base=500000.0):
    return base ** (-np.arange(0, r, 2) / r)


def axes_of(r, axes):
    return [i * axes // (r // 2) for i in range(r // 2)]


class Rows:
    """Random rows as slices of one packed projection (or dense), with the 64-bit results."""

    def __init__(self, torch, pa, tokens, hq, hkv, act="fp16", norm=True, r=128, interleaved=False, axes=1, positions=None,
                 packed=True, seed=0, scale=1.0, eps=1e-6):
        g = torch.Generator(device="cuda").manual_seed(seed)
        dt = {"fp16": torch.float16, "bf16": torch.bfloat16}[act]
        self.pa, self.act, self.dt, self.hq, self.hkv, self.tokens = pa, act, dt, hq, hkv, tokens
        x = torch.randn(tokens, hq + 2 * hkv, 128, generator=g, device="cuda").mul_(torch.rand(1, hq + 2 * hkv, 1, generator=g, device="cuda") * 4 + 0.05).to(dt)
        self.q, self.k, self.v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
        if not packed:
            self.q, self.k, self.v = self.q.contiguous(), self.k.contiguous(), self.v.contiguous()
        self.wq, self.wk = ((torch.rand(128, generator=g, device="cuda") * 2 + 0.1).to(dt) for _ in range(2)) if norm else (None, None)
        self.eps, self.r, self.interleaved, self.scale = eps, r, interleaved, scale
        self.axes = axes_of(r, axes) if r else None
        self.rope = pa.Rope(freqs(r), interleaved=interleaved, axes=self.axes, scale=scale) if r else None
        self.positions = positions

    def params(self):
        import torch
        p = None if self.positions is None else torch.from_numpy(np.ascontiguousarray(self.positions, np.int32)).cuda()
        return self.pa.qkv_params(self.q if self.hq else None, self.k, self.v, self.wq if self.hq else None, self.wk, self.eps, p)

    def want(self, x, w, positions):
        x = x.double().cpu().numpy()
        y = ro.norm(x, None if w is None else w.double().cpu().numpy(), self.eps)
        if not self.r:
            return y, np.abs(y)
        return ro.rotate(y, np.atleast_2d(positions), freqs(self.r), self.axes, self.interleaved, self.scale)


def assert_rows(got, y, size, step, tiny):
    got = got.double().cpu().numpy()
    bound = ro.rows_bound(y, size, step, tiny)
    worst = np.abs(got - y) / np.maximum(bound, 1e-300)
    assert worst.size == 0 or worst.max() <= 1.0, f"off by {worst.max():.3g} of the bound at {np.unravel_index(worst.argmax(), worst.shape)}"


CASES = [dict(tokens=t, hq=hq, hkv=hkv, act=a, norm=n, r=r, interleaved=i, axes=x, packed=p) for t, hq, hkv, a, n, r, i, x, p in [
    (1, 1, 1, "fp16", True, 128, False, 1, False), (1, 32, 8, "bf16", True, 128, True, 1, True), (2, 5, 3, "fp16", False, 128, False, 1, True),
    (7, 8, 1, "bf16", False, 64, False, 3, True), (33, 28, 4, "fp16", True, 96, True, 2, True), (129, 64, 8, "bf16", True, 16, False, 4, False),
    (64, 32, 8, "fp16", True, 48, False, 1, True), (1000, 3, 2, "fp16", True, 128, False, 3, True), (2500, 32, 8, "bf16", True, 128, False, 1, True),
    (4099, 1, 1, "fp16", False, 80, True, 1, False), (17, 0, 5, "bf16", True, 128, False, 1, True), (40, 9, 2, "fp16", True, 0, False, 1, True),
    (5, 300, 1, "fp16", True, 112, False, 2, True)]]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v) for v in c.values()))
@pytest.mark.parametrize("in_place", [False, True])
def test_norm_rope(case, in_place, torch_cuda, pa):
    torch = torch_cuda
    rng = np.random.default_rng(case["tokens"])
    pos = rng.integers(-1000, 200000, (case["axes"], case["tokens"]))
    pos[:, 0] = 2 ** 31 - 1 if case["tokens"] % 2 else -2 ** 31
    w = Rows(torch, pa, positions=pos if case["r"] else None, **case)
    q, sq = w.want(w.q, w.wq, pos)
    k, sk = w.want(w.k, w.wk, pos)
    before = w.v.clone()
    q_out = w.q if in_place else torch.full((w.tokens, w.hq, 128), 7.0, dtype=w.dt, device="cuda")
    k_out = w.k if in_place else torch.full((w.tokens, w.hkv, 128), 7.0, dtype=w.dt, device="cuda")
    pa.qk_norm_rope(w.params(), w.rope, q_out if w.hq else None, k_out, torch.cuda.current_stream().cuda_stream)
    assert_rows(q_out, q, sq, *STEP[w.act])
    assert_rows(k_out, k, sk, *STEP[w.act])
    assert torch.equal(w.v, before)


def test_norm_rope_strided_output_and_scale(torch_cuda, pa):
    torch = torch_cuda
    pos = np.arange(50)[None] * 977
    w = Rows(torch, pa, 50, 8, 2, positions=pos, scale=1.3, norm=False)
    room = torch.full((50, 12, 128), 3.0, dtype=w.dt, device="cuda")
    pa.qk_norm_rope(w.params(), w.rope, room[:, :8], room[:, 9:11])
    assert_rows(room[:, :8], *w.want(w.q, None, pos), *STEP["fp16"])
    assert_rows(room[:, 9:11], *w.want(w.k, None, pos), *STEP["fp16"])
    assert (room[:, 8] == 3).all() and (room[:, 11] == 3).all()


def test_values_outside_the_rotation_stay(torch_cuda, pa):
    """Infinities and NaN touch their own pair and nothing else; dims behind rotary_dim are copied bit for bit."""
    torch = torch_cuda
    for interleaved in (False, True):
        w = Rows(torch, pa, 3, 1, 1, norm=False, r=64, interleaved=interleaved, positions=np.array([[5, 6, 7]]), packed=False)
        w.k[0, 0, 100], w.k[1, 0, 3], w.k[2, 0, 127] = float("inf"), float("nan"), float("nan")
        out = torch.zeros_like(w.k)
        pa.qk_norm_rope(w.params(), w.rope, torch.zeros_like(w.q), out)
        assert torch.equal(out[..., 64:].view(torch.int16)[:2], w.k[..., 64:].view(torch.int16)[:2])
        bad = torch.isnan(out)
        pair = [3, 2] if interleaved else [3, 35]
        assert bad.sum() == 3 and bad[1, 0, pair].all() and bad[2, 0, 127]
        assert torch.isinf(out).sum() == 1


def paged(rng, lens, ps, spare=3):
    need = [(n + ps - 1) // ps for n in lens]
    perm = rng.permutation(sum(need) + spare).astype(np.int32)
    table = np.full((len(lens), max(max(need), 1) + 1), -7, np.int32)    # entries nobody may follow
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, sum(need) + spare


APPENDS = [
    # cache, scales, act, page, hq, hkv, norm, r, interleaved, new tokens, tokens before
    ("fp16", None, "fp16", 16, 32, 8, False, 128, False, [1] * 9, [0, 1, 15, 16, 17, 31, 300, 5, 64]),
    ("fp16", None, "bf16", 1, 2, 2, True, 128, True, [3, 1, 8], [0, 5, 2]),
    ("fp16", None, "fp16", 24, 8, 1, True, 64, False, [100, 0, 7, 0, 1], [3, 9, 23, 0, 24]),
    ("fp16", None, "bf16", 256, 16, 4, True, 128, False, [700, 33], [0, 255]),
    ("e4m3", "tensor", "fp16", 16, 4, 4, True, 128, False, [5, 40, 1], [0, 3, 16]),
    ("e4m3", "head", "bf16", 7, 32, 8, True, 96, False, [21, 1, 2], [6, 7, 0]),
    ("e4m3", "head", "fp16", 64, 0, 3, False, 0, False, [130], [1]),
    ("fp16", None, "fp16", 16, 8, 8, True, 128, False, [1] * 70, list(range(70))),
    ("fp16", None, "fp16", 16, 1, 1, False, 128, False, [n % 3 for n in range(1200)], [0] * 1200),
]


@pytest.mark.parametrize("case", APPENDS, ids=lambda c: "-".join(str(x) for x in c[:9]) + "x%d" % len(c[9]))
def test_append(case, torch_cuda, pa):
    torch = torch_cuda
    cache, kind, act, ps, hq, hkv, norm, r, inter, new, past = case
    rng = np.random.default_rng(ps)
    table, pages = paged(rng, [a + b for a, b in zip(new, past)], ps)
    tokens, pad = sum(new), 5                               # rows behind the last sequence
    place = np.concatenate([np.arange(p, p + n) for n, p in zip(new, past)] + [np.zeros(pad, int)])
    w = Rows(torch, pa, tokens + pad, hq, hkv, act=act, norm=norm, r=r, interleaved=inter)
    dt = torch.float16 if cache == "fp16" else torch.uint8
    fill = torch.randint(0, 100, (pages, hkv, ps, 128), device="cuda")
    kc, vc = fill.to(dt), (fill + 1).to(dt)
    k0, v0 = kc.clone(), vc.clone()
    q_out = torch.full((tokens + pad, hq, 128), 9.0, dtype=torch.float16, device="cuda")
    ks = vs = None
    kw = {}
    if kind == "head":
        ks, vs = (rng.uniform(0.01, 0.2, hkv).astype(np.float32) for _ in range(2))
        kw = dict(d_k_scales=torch.from_numpy(ks).cuda(), d_v_scales=torch.from_numpy(vs).cuda())
    elif kind == "tensor":
        kw = dict(k_scale=0.05, v_scale=0.02)
        ks, vs = np.full(hkv, 0.05, np.float32), np.full(hkv, 0.02, np.float32)
    begin = torch.from_numpy(np.cumsum([0] + new).astype(np.int32)).cuda()
    one_each = all(n == 1 for n in new)
    t = pa.append_target(kc, vc, torch.from_numpy(table).cuda(), torch.tensor(past, dtype=torch.int32, device="cuda"),
                         token_begin=None if one_each else begin, **kw)
    pa.append_qkv(FP16 if cache == "fp16" else FP8, w.params(), w.rope, t, q_out if hq else None, torch.cuda.current_stream().cuda_stream)
    assert pa.kernel_status() == 0
    q, sq = w.want(w.q, w.wq, place)
    assert_rows(q_out[:tokens], q[:tokens], sq[:tokens], *STEP["fp16"])
    assert (q_out[tokens:] == 9).all()
    seq = np.repeat(np.arange(len(new)), new)
    page, off = table[seq, place[:tokens] // ps], place[:tokens] % ps
    for pool, pool0, (y, size), s in ((kc, k0, w.want(w.k, w.wk, place), ks), (vc, v0, (w.v.double().cpu().numpy(),) * 2, vs)):
        got = pool.cpu().numpy()
        y, size = y[:tokens], np.abs(size[:tokens])
        if cache == "fp16":
            bound = ro.rows_bound(y, size, *STEP["fp16"])
            value = got.astype(np.float64)
        else:
            s = s.astype(np.float64)[:, None]
            bound = ro.e4m3_bound(y, s) + 1.07 * ro.rows_bound(y, size, 0, 0)   # a step of e4m3 is 1/16: the bound's slope
            value = ro.decode_e4m3(got) * s[None, :, :, None].reshape(1, hkv, 1, 1)
            y = np.clip(y, -448 * s, 448 * s)
        err = np.abs(value[page, :, off] - y)
        assert (err <= bound).all(), (err / bound).max()
        untouched = np.ones(pool.shape[:1] + pool.shape[2:3], bool)
        untouched[page, off] = False
        assert (got.transpose(0, 2, 1, 3)[untouched] == pool0.cpu().numpy().transpose(0, 2, 1, 3)[untouched]).all()


def test_plain_rows_into_an_fp16_cache_are_copied_bit_for_bit(torch_cuda, pa):
    """Without norm and rotation the append is append_tokens'."""
    torch = torch_cuda
    w = Rows(torch, pa, 50, 0, 4, norm=False, r=0, packed=False)
    w.k[3, 1, 5], w.v[4, 2, 6] = float("inf"), float("-inf")
    table = torch.arange(4, dtype=torch.int32, device="cuda")[None].flip(1).contiguous()
    pools = [torch.zeros(4, 4, 16, 128, dtype=torch.float16, device="cuda") for _ in range(4)]
    t = pa.append_target(pools[0], pools[1], table, torch.tensor([5], dtype=torch.int32, device="cuda"),
                         token_begin=torch.tensor([0, 50], dtype=torch.int32, device="cuda"))
    pa.append_qkv(FP16, w.params(), None, t, None)
    pa.append_tokens(FP16, w.k, w.v, pools[2], pools[3], table[0], 5, 50, 4, 128, 16)
    assert torch.equal(pools[0].view(torch.int16), pools[2].view(torch.int16))
    assert torch.equal(pools[1].view(torch.int16), pools[3].view(torch.int16))


@pytest.mark.parametrize("blocks", [False, True])
def test_skipped_and_misplaced_sequences(blocks, torch_cuda, pa):
    """Negative slots and rows before the first sequence are skipped silently; a page outside the pool, a position behind the
    table, a negative position and a slot behind the table's rows are skipped and reported.  Nothing else changes."""
    torch = torch_cuda
    new, past = [2, 3, 1, 4, 2, 1, 2], [0, 14, 5, 30, -1, 2, 3]
    slots = [0, -1, 2, 1, 3, 9, 4]                  # 9: no such row
    table = torch.tensor([[0, 1], [2, 3], [99, 4], [5, 6], [-2, 7]], dtype=torch.int32, device="cuda")
    w = Rows(torch, pa, 2 + sum(new), 2, 2, norm=True)
    begin = torch.from_numpy((2 + np.cumsum([0] + new)).astype(np.int32)).cuda()     # two rows before the first sequence
    dt = torch.uint8 if blocks else torch.float16
    kc, vc = (torch.zeros(8, 2, 16, 128, dtype=dt, device="cuda") for _ in range(2))
    scales = torch.zeros(8, 2, 1, 2, device="cuda") if blocks else None
    q_out = torch.full((w.tokens, 2, 128), 9.0, dtype=torch.float16, device="cuda")
    t = pa.append_target(kc, vc, table, torch.tensor(past, dtype=torch.int32, device="cuda"), begin,
                         torch.tensor(slots, dtype=torch.int32, device="cuda"), d_block_scales=scales)
    pa.append_qkv(FP8 if blocks else FP16, w.params(), w.rope, t, q_out)
    import paged_attention_b200._lib as lib
    with pytest.raises(lib.KernelTimeout, match="no place"):
        pa.kernel_status()
    assert pa.kernel_status() == 0                  # reading it clears it
    assert (q_out[:2] == 9).all() and (q_out[4:7] == 9).all() and (q_out[2:4] != 9).any() and not (q_out[7:] == 9).all(-1).any()
    wrote = {(0, 0), (0, 1), (3, 14), (3, 15), (5, 0)}      # sequence 0; the half of sequence 3 inside the table; -1, 0 -> 0
    for pool in (kc, vc):
        hit = (pool.view(torch.uint8) != 0).any(-1).any(1).cpu().numpy()
        assert set(zip(*np.nonzero(hit))) == wrote


def test_streams_graphs_and_two_calls_at_once(torch_cuda, pa):
    """A captured append replays on whatever its device arrays say then; two appends on two streams do not meet."""
    torch = torch_cuda
    ps, hkv = 16, 2
    a, b = (Rows(torch, pa, 4, 2, hkv, seed=s) for s in (1, 2))
    out = []
    for w in (a, b):
        pools = [torch.zeros(8, hkv, ps, 128, dtype=torch.float16, device="cuda") for _ in range(2)]
        table = torch.tensor([[3, 1, 0, 2], [4, 5, 6, 7], [0, 0, 0, 0], [0, 0, 0, 0]], dtype=torch.int32, device="cuda")
        start = torch.tensor([0, 0], dtype=torch.int32, device="cuda")
        begin = torch.tensor([0, 3, 4], dtype=torch.int32, device="cuda")
        q_out = torch.zeros(4, 2, 128, dtype=torch.float16, device="cuda")
        out.append((w, pools, table, start, begin, q_out, pa.append_target(*pools, table, start, begin)))
    pa.kernel_status()                              # the status word exists before the capture
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    graphs = []
    for s, (w, pools, table, start, begin, q_out, t) in zip((s1, s2), out):
        x = w.params()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            pa.append_qkv(FP16, x, w.rope, t, q_out, s.cuda_stream)
        graphs.append((g, x))
    for first, moved in ((0, [0, 3, 4]), (17, [0, 1, 4]), (40, [0, 0, 2])):
        for _, pools, table, start, begin, q_out, t in out:
            start.fill_(first)
            begin.copy_(torch.tensor(moved, dtype=torch.int32))
            q_out.fill_(9)
        torch.cuda.synchronize()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert pa.kernel_status() == 0
        for w, pools, table, start, begin, q_out, t in out:
            seq = np.repeat([0, 1], np.diff(moved))
            n = len(seq)
            place = first + np.concatenate([np.arange(m) for m in np.diff(moved)])
            where = np.append(place, [0] * (4 - n)).astype(int)
            assert_rows(q_out[:n], *(y[:n] for y in w.want(w.q, w.wq, where)), *STEP["fp16"])
            assert (q_out[n:] == 9).all()
            tab = table.cpu().numpy()
            k, size = (y[:n] for y in w.want(w.k, w.wk, where))
            got = pools[0].double().cpu().numpy()[tab[seq, place // ps], :, place % ps]
            assert (np.abs(got - k) <= ro.rows_bound(k, size, *STEP["fp16"])).all()
            assert torch.equal(pools[1][torch.from_numpy(tab[seq, place // ps]).long().cuda(), :, torch.from_numpy(place % ps).long().cuda()], w.v[:n])


def test_offsets_past_32_bits(torch_cuda, pa):
    """A pool of more than 2^32 bytes and rows of more than 2^31 elements into it."""
    torch = torch_cuda
    hkv, ps, pages = 8, 16, 140000                  # 140000 * 8 * 16 * 128 * 2 = 4.6 GB
    kc, vc = (torch.zeros(pages, hkv, ps, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    w = Rows(torch, pa, 33, 8, hkv)
    table = torch.tensor([[139999, 0, 139998]], dtype=torch.int32, device="cuda")
    t = pa.append_target(kc, vc, table, torch.tensor([7], dtype=torch.int32, device="cuda"), torch.tensor([0, 33], dtype=torch.int32, device="cuda"))
    pa.append_qkv(FP16, w.params(), w.rope, t, torch.empty(33, 8, 128, dtype=torch.float16, device="cuda"))
    place = np.arange(7, 40)
    got = torch.cat([kc[139999, :, 7:], kc[0], kc[139998, :, :8]], 1).transpose(0, 1)
    k, size = w.want(w.k, w.wk, place)
    assert_rows(got, k, size, *STEP["fp16"])
    assert torch.equal(torch.cat([vc[139999, :, 7:], vc[0], vc[139998, :, :8]], 1).transpose(0, 1), w.v)
    assert not kc[1:139998].any()


def test_tensors_of_another_device_are_refused(torch_cuda, pa):
    torch = torch_cuda
    w = Rows(torch, pa, 2, 2, 2, positions=np.arange(2)[None])
    x = w.params()
    x._device = 5                                   # as a tensor on cuda:5 would say
    with pytest.raises(pa.InvalidArgument, match="current device"):
        pa.qk_norm_rope(x, w.rope, torch.zeros_like(w.q), torch.zeros_like(w.k))


@pytest.mark.parametrize("blocks", [False, True])
@pytest.mark.parametrize("axes, r, interleaved", [(1, 128, False), (3, 128, False), (4, 96, True), (2, 16, False)])
def test_append_with_positions_of_its_own(blocks, axes, r, interleaved, torch_cuda, pa):
    """Rotation positions that are not the places in the cache (offsets, several axes, negative and far ones)."""
    torch = torch_cuda
    new, past, ps, hkv = [20, 1, 7, 16], [5, 0, 31, 16], 16, 3
    rng = np.random.default_rng(axes)
    table, pages = paged(rng, [a + b for a, b in zip(new, past)], ps)
    tokens = sum(new)
    pos = rng.integers(-10 ** 6, 10 ** 9, (axes, tokens))
    w = Rows(torch, pa, tokens, 6, hkv, act="bf16", r=r, interleaved=interleaved, axes=axes, positions=pos)
    kc, vc = (torch.zeros(pages, hkv, ps, 128, dtype=torch.uint8 if blocks else torch.float16, device="cuda") for _ in range(2))
    scales = torch.zeros(pages, hkv, 1, 2, device="cuda") if blocks else None
    q_out = torch.zeros(tokens, 6, 128, dtype=torch.float16, device="cuda")
    t = pa.append_target(kc, vc, torch.from_numpy(table).cuda(), torch.tensor(past, dtype=torch.int32, device="cuda"),
                         torch.from_numpy(np.cumsum([0] + new).astype(np.int32)).cuda(), d_block_scales=scales)
    pa.append_qkv(FP8 if blocks else FP16, w.params(), w.rope, t, q_out)
    assert pa.kernel_status() == 0
    assert_rows(q_out, *w.want(w.q, w.wq, pos), *STEP["fp16"])
    k, size = w.want(w.k, w.wk, pos)
    seq = np.repeat(np.arange(4), new)
    place = np.concatenate([np.arange(o, o + n) for n, o in zip(new, past)])
    page, off = table[seq, place // ps], place % ps
    if blocks:
        s = scales.cpu().numpy().astype(np.float64)[page, :, 0, 0][..., None]
        got, bound = ro.decode_e4m3(kc.cpu().numpy())[page, :, off] * s, ro.e4m3_bound(k, s) + 1.07 * ro.rows_bound(k, size, 0, 0)
    else:
        got, bound = kc.double().cpu().numpy()[page, :, off], ro.rows_bound(k, size, *STEP["fp16"])
    assert (np.abs(got - k) <= bound).all()


def test_forty_thousand_sequences(torch_cuda, pa):
    """The search for a row's sequence over several levels, with empty sequences between."""
    torch = torch_cuda
    rng = np.random.default_rng(1)
    batch = 40000
    new = rng.integers(0, 2, batch)
    new[-1] = 1
    new[:100] = 0
    past = rng.integers(0, 12, batch)
    tokens = int(new.sum())
    w = Rows(torch, pa, tokens + 3, 1, 1, norm=False)
    kc, vc = (torch.zeros(batch, 1, 16, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    table = torch.randperm(batch, device="cuda").to(torch.int32)[:, None].contiguous()
    q_out = torch.full((tokens + 3, 1, 128), 9.0, dtype=torch.float16, device="cuda")
    t = pa.append_target(kc, vc, table, torch.from_numpy(past.astype(np.int32)).cuda(),
                         torch.from_numpy(np.cumsum(np.append(0, new)).astype(np.int32)).cuda())
    pa.append_qkv(FP16, w.params(), w.rope, t, q_out)
    assert pa.kernel_status() == 0
    seq = np.repeat(np.arange(batch), new)
    place = past[seq]
    pages = table[:, 0].cpu().numpy()[seq]
    k, size = w.want(w.k, None, np.append(place, [0, 0, 0]))
    got = kc.double().cpu().numpy()[pages, :, place]
    assert (np.abs(got - k[:tokens]) <= ro.rows_bound(k, size, *STEP["fp16"])[:tokens]).all()
    assert torch.equal(vc[torch.from_numpy(pages).long().cuda(), :, torch.from_numpy(place).cuda()], w.v[:tokens])
    assert (vc != 0).any(-1).sum() == tokens and (q_out[tokens:] == 9).all()


def test_empty_calls_and_one_kind_of_heads(torch_cuda, pa):
    """No tokens, no sequences, no q heads, no k heads: nothing happens where there is nothing to do."""
    torch = torch_cuda
    e = torch.empty(0, 4, 128, dtype=torch.float16, device="cuda")
    pa.qk_norm_rope(pa.qkv_params(e, e[:, :2]), None, e.clone(), e[:, :2].clone())
    kc, vc = (torch.zeros(2, 2, 16, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    pa.append_qkv(FP16, pa.qkv_params(e, e[:, :2], e[:, :2]), None, pa.append_target(kc, vc, table, torch.zeros(1, dtype=torch.int32, device="cuda")), e.clone())
    x = torch.ones(3, 2, 128, dtype=torch.float16, device="cuda")
    pa.append_qkv(FP16, pa.qkv_params(None, x, x), None, pa.append_target(kc, vc, table, none), None)
    assert not kc.any()
    q, out = torch.randn(3, 5, 128, device="cuda").half(), torch.zeros(3, 5, 128, dtype=torch.float16, device="cuda")
    pa.qk_norm_rope(pa.qkv_params(q, x[:, :0]), None, out, None)
    assert torch.equal(out, q)
    # per-head scales for K beside a per-tensor scale for V
    k8, v8 = (torch.zeros(2, 2, 16, 128, dtype=torch.uint8, device="cuda") for _ in range(2))
    t = pa.append_target(k8, v8, table, torch.tensor([2], dtype=torch.int32, device="cuda"), torch.tensor([0, 3], dtype=torch.int32, device="cuda"),
                         v_scale=0.25, d_k_scales=torch.tensor([1.0, 2.0], device="cuda"))
    pa.append_qkv(FP8, pa.qkv_params(None, x, x), None, t, None)
    k, v = (ro.decode_e4m3(p.cpu().numpy())[0, :, 2:5] for p in (k8, v8))
    assert (k[0] == 1).all() and (k[1] == 0.5).all() and (v == 4).all()
