"""Workloads of the operators around the paged decode: per-head norm + position rotation of queries and keys
(`norm_rope`), the same on the way into the paged cache (`append`, with fp16, per-head e4m3 and block-scaled e4m3
pools), and decode attention over the block-scaled e4m3 cache (`decode`).

`run` computes an operator in its plain form (elementary torch operations, 32 bits, 64 where a rounding border or a
far angle needs them) or, with `own` true, through the framework's entry points.  Head dimension 128 throughout, as
everywhere in the framework.
"""
import math
import random

import torch

own = False

D = 128
E4M3_MAX = 448.0
EPS = 1e-6
MIN_SCALE_EXP, MAX_SCALE_EXP = -32, 8     # block scales are powers of two in this range
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---- cases -----------------------------------------------------------------------------------------------------

def listed():
    return [
        # one token of one sequence: what a call costs when nothing hides it
        dict(name="norm_rope_1", op="norm_rope", tokens=1, hq=32, hkv=8, act="fp16", norm=True, rotary=128,
             interleaved=False, axes=1, far=131071),
        # a prompt chunk out of a packed bf16 projection (rows of q|k|v), norm of q and k, neox rotation
        dict(name="norm_rope_8192", op="norm_rope", tokens=8192, hq=32, hkv=8, act="bf16", norm=True, rotary=128,
             interleaved=False, axes=1, far=4096),
        # image and video tokens: three position axes, odd count, half of each head rotated in adjacent pairs, no norm
        dict(name="norm_rope_axes_20001", op="norm_rope", tokens=20001, hq=64, hkv=8, act="fp16", norm=False, rotary=64,
             interleaved=True, axes=3, far=1000000),
        # a decode step of 64 sequences into the fp16 cache (the batch of the headline layer)
        dict(name="append_step_64", op="append", cache="fp16", act="fp16", batch=64, new_min=1, new_max=1, past_max=1000,
             page=16, hq=32, hkv=8, norm=False, rotary=128, interleaved=False, axes=1),
        # chunked prefill of a ragged batch with norm, e4m3 cache with one scale per kv head
        dict(name="append_chunks_e4m3", op="append", cache="e4m3", act="bf16", batch=24, new_min=1, new_max=1100,
             past_max=700, page=16, hq=32, hkv=8, norm=True, rotary=128, interleaved=False, axes=1),
        # whole prompts of a 64-query-head layer into the fp16 cache
        dict(name="append_prompts_fp16", op="append", cache="fp16", act="bf16", batch=8, new_min=2500, new_max=5500,
             past_max=0, page=64, hq=64, hkv=8, norm=True, rotary=128, interleaved=False, axes=1),
        # a decode step of 128 sequences into block-scaled pages: partly filled blocks whose scale may grow
        dict(name="append_step_128_blocks", op="append", cache="blocks", act="fp16", batch=128, new_min=1, new_max=1,
             past_max=500, page=16, hq=32, hkv=8, norm=True, rotary=128, interleaved=False, axes=1),
        # ragged prompt chunks that start and end inside blocks, with three position axes
        dict(name="append_chunks_blocks", op="append", cache="blocks", act="bf16", batch=13, new_min=3, new_max=2200,
             past_max=300, page=32, hq=32, hkv=8, norm=True, rotary=128, interleaved=False, axes=3),
        # four short sequences, down to one token: the smallest decode call
        dict(name="decode_4_short", op="decode", batch=4, len_min=1, len_max=300, page=16, hq=32, hkv=8),
        # the 128 x 4096 layer of the framework's fp8 benchmark, with block scales
        dict(name="decode_128x4096", op="decode", batch=128, len_min=4096, len_max=4096, page=16, hq=32, hkv=8),
        # a ragged batch of 256 on a layer of 64 query heads
        dict(name="decode_256_ragged", op="decode", batch=256, len_min=1, len_max=8192, page=16, hq=64, hkv=8),
        # one very long sequence of a layer of four kv heads, wide pages: the split over the whole grid and its merge
        dict(name="decode_1x200001", op="decode", batch=1, len_min=200001, len_max=200001, page=64, hq=32, hkv=4),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_rope", "append", "append", "decode", "decode"])
    if op == "norm_rope":
        hkv = rng.choice([1, 2, 4, 8])
        return dict(op=op, tokens=_log_int(rng, 1, 16000), hq=hkv * rng.choice([1, 2, 4, 8]), hkv=hkv,
                    act=rng.choice(["fp16", "bf16"]), norm=rng.random() < 0.6, rotary=rng.choice([32, 64, 96, 128, 128, 128]),
                    interleaved=rng.random() < 0.3, axes=rng.choice([1, 1, 3]), far=_log_int(rng, 1, 1000000))
    hkv = rng.choice([1, 2, 4, 8, 8])
    hq = hkv * rng.choice([1, 2, 4, 8])
    page = rng.choice([8, 16, 16, 16, 24, 32, 64])
    if op == "append":
        if rng.random() < 0.4:
            new_min = new_max = 1
            batch = _log_int(rng, 1, 256)
        else:
            new_min, new_max, batch = 1, _log_int(rng, 2, 3000), rng.randint(1, 8)
        return dict(op=op, cache=rng.choice(["fp16", "e4m3", "blocks", "blocks"]), act=rng.choice(["fp16", "bf16"]), batch=batch,
                    new_min=new_min, new_max=new_max, past_max=rng.randint(0, 400), page=page, hq=hq, hkv=hkv,
                    norm=rng.random() < 0.6, rotary=rng.choice([64, 128, 128]), interleaved=rng.random() < 0.3,
                    axes=rng.choice([1, 1, 3]))
    batch = _log_int(rng, 1, 128)
    top = _log_int(rng, 1, max(2, min(100000, 500000 // batch)))
    return dict(op=op, batch=batch, len_min=rng.choice([1, top]), len_max=top, page=page, hq=hq, hkv=hkv)


def _rng(case):
    """Lengths belong to the case, not to the seed: work() counts them too."""
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _new_and_past(case):
    r = _rng(case)
    new = [r.randint(case["new_min"], case["new_max"]) for _ in range(case["batch"])]
    past = [r.randint(0, case["past_max"]) for _ in range(case["batch"])]
    return new, past


def _lens(case):
    r = _rng(case)
    return [r.randint(case["len_min"], case["len_max"]) for _ in range(case["batch"])]


def _block(page):
    """Tokens that share a scale: the largest power of two that divides the page, at most 16."""
    return min(16, page & -page)


def work(case):
    hq, hkv = case["hq"], case["hkv"]
    if case["op"] == "norm_rope":
        n = case["tokens"] * (hq + hkv) * D
        return {"bytes": 4 * n + 4 * case["tokens"] * case["axes"], "flops": 8 * n}
    if case["op"] == "append":
        new, past = _new_and_past(case)
        t, cached = sum(new), 2 if case["cache"] == "fp16" else 1
        n = 2 * t * (hq + 2 * hkv) * D + 2 * t * hq * D + t * 2 * hkv * D * cached
        if case["cache"] == "blocks":
            b = _block(case["page"])
            n += sum((o + m + b - 1) // b - o // b for m, o in zip(new, past)) * 8 * hkv
        return {"bytes": n, "flops": 8 * t * (hq + hkv) * D}
    lens, b = _lens(case), _block(case["page"])
    blocks = sum((n + b - 1) // b for n in lens)
    return {"bytes": sum(lens) * 2 * hkv * D + blocks * 8 * hkv + 4 * case["batch"] * hq * D, "flops": 4 * sum(lens) * hq * D}


# ---- inputs ----------------------------------------------------------------------------------------------------

def _inv_freq(rotary):
    return [500000.0 ** (-2.0 * i / rotary) for i in range(rotary // 2)]


def _axis_of(rotary, axes):
    """Frequencies in contiguous sections: a quarter for the first axis, three eighths for each of the others."""
    n = rotary // 2
    return [0 if axes == 1 or i < n // 4 else 1 if i < n * 5 // 8 else 2 for i in range(n)]


def _positions(case, tokens, g):
    """[axes, tokens]: text counts on; with three axes, patches of a grid that moves on in time."""
    t = torch.arange(tokens, device="cuda")
    start = int(torch.randint(0, 1000, (1,), generator=g, device="cuda"))
    first = case.get("far", 0) + start
    if case["axes"] == 1:
        return (first + t).to(torch.int32).unsqueeze(0).contiguous()
    return torch.stack([first + t // 667, t // 29 % 23, t % 29]).to(torch.int32).contiguous()


def _paged(case, lens, g, spare=3):
    """A scattered block table for sequences of `lens` tokens: (table [batch, pages], pages of the pool)."""
    page = case["page"]
    need = [(n + page - 1) // page for n in lens]
    pool = sum(need) + spare
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), max(need), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pool


def _pool(shape, cache, g):
    """A pool with earlier tokens in it."""
    x = torch.empty(shape, dtype=torch.float16, device="cuda").normal_(generator=g)
    return x if cache == "fp16" else (x * 100).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def _power_of_two(exp):
    """2^exp in 32 bits for a tensor of whole numbers, by its bits."""
    return (exp.to(torch.int32) + 127 << 23).view(torch.float32)


def _block_scales(pool, hkv, blocks, g):
    """[page, kv head, block, K|V]: powers of two, as the append leaves them."""
    return _power_of_two(torch.randint(-8, -5, (pool, hkv, blocks, 2), generator=g, device="cuda"))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    hq, hkv = case["hq"], case["hkv"]
    s = {"case": case}
    if case["op"] == "decode":
        lens, page = _lens(case), case["page"]
        s["table"], pool = _paged(case, lens, g)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["k_pool"], s["v_pool"] = (_pool((pool, hkv, page, D), "blocks", g) for _ in range(2))
        s["scales"] = _block_scales(pool, hkv, page // _block(page), g)
        s["q"] = torch.empty(case["batch"], hq, D, dtype=torch.float16, device="cuda").normal_(generator=g)
        s["out"] = torch.zeros_like(s["q"])
        if own:
            _own_decode(s, lens)
        return s
    act = TYPES[case["act"]]
    new, past = _new_and_past(case) if case["op"] == "append" else ([case["tokens"]], [0])
    tokens = sum(new)
    qkv = torch.empty(tokens, hq + 2 * hkv, D, dtype=act, device="cuda").normal_(generator=g)
    qkv[:, hq:hq + hkv] *= torch.empty(hkv, 1, device="cuda").uniform_(0.3, 3, generator=g).to(act)   # heads differ in size
    s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    s["q_norm"] = s["k_norm"] = None
    if case["norm"]:
        s["q_norm"], s["k_norm"] = (torch.empty(D, device="cuda").uniform_(0.5, 2, generator=g).to(act) for _ in range(2))
    s["inv_freq"], s["axis"] = _inv_freq(case["rotary"]), _axis_of(case["rotary"], case["axes"])
    s["inv_freq_dev"] = torch.tensor(s["inv_freq"], dtype=torch.float64, device="cuda")
    s["axis_dev"] = torch.tensor(s["axis"], device="cuda")
    if case["op"] == "norm_rope":
        s["positions"] = _positions(case, tokens, g)
        s["q_out"] = torch.zeros(tokens, hq, D, dtype=act, device="cuda")
        s["k_out"] = torch.zeros(tokens, hkv, D, dtype=act, device="cuda")
    else:
        page = case["page"]
        s["table"], pool = _paged(case, [o + n for o, n in zip(past, new)], g)
        s["start"] = torch.tensor(past, dtype=torch.int32, device="cuda")
        s["token_begin"] = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda")
        s["positions"] = _positions(case, tokens, g) if case["axes"] > 1 else None   # None: the place in the cache
        s["k_pool"], s["v_pool"] = (_pool((pool, hkv, page, D), case["cache"], g) for _ in range(2))
        s["scales"] = None
        if case["cache"] == "blocks":
            s["scales"] = _block_scales(pool, hkv, page // _block(page), g)
        elif case["cache"] == "e4m3":
            s["scales"] = torch.empty(2, hkv, device="cuda").uniform_(0.01, 0.04, generator=g)   # K, V per kv head
        s["q_out"] = torch.zeros(tokens, hq, D, dtype=torch.float16, device="cuda")
    if own:
        _own_rows(s)
    return s


# ---- the framework's calls -------------------------------------------------------------------------------------

def _own_rows(s):
    """The filled argument structs over the program's buffers, kept as pd_params is for a decode."""
    import paged_attention_b200 as pa
    case = s["case"]
    s["rope"] = pa.Rope(s["inv_freq"], interleaved=case["interleaved"], axes=s["axis"])
    s["x"] = pa.qkv_params(s["q"], s["k"], s["v"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS, positions=s["positions"])
    if case["op"] == "append":
        k_scales = v_scales = blocks = None
        if case["cache"] == "e4m3":
            k_scales, v_scales = s["scales"][0], s["scales"][1]
        elif case["cache"] == "blocks":
            blocks = s["scales"]
        s["target"] = pa.append_target(s["k_pool"], s["v_pool"], s["table"], s["start"], token_begin=s["token_begin"],
                                       d_k_scales=k_scales, d_v_scales=v_scales, d_block_scales=blocks)
        s["dtype"] = pa.KVDtype.FP16 if case["cache"] == "fp16" else pa.KVDtype.FP8_E4M3


def _own_decode(s, lens):
    """The plan of the step and the bound params, made once per step and used by every layer."""
    import paged_attention_b200 as pa
    case = s["case"]
    plan = pa.make_plan(pa.KVDtype.FP8_E4M3, lens, case["hq"], case["hkv"], D)
    s["plan"] = pa.DevicePlan()
    s["plan"].upload(plan, case["hq"] // case["hkv"], D, torch.cuda.current_stream().cuda_stream)
    p = pa.DecodeParams()
    p.q, p.out = s["q"].data_ptr(), s["out"].data_ptr()
    p.k_cache, p.v_cache = s["k_pool"].data_ptr(), s["v_pool"].data_ptr()
    p.block_table, p.seq_lens, p.block_table_stride = s["table"].data_ptr(), s["lens"].data_ptr(), s["table"].shape[1]
    p.batch, p.num_q_heads, p.num_kv_heads, p.head_dim, p.page_size = case["batch"], case["hq"], case["hkv"], D, case["page"]
    p.sm_scale = 1.0 / math.sqrt(D)
    s["plan"].bind(p)
    s["params"] = p


def _run_own(s):
    import paged_attention_b200 as pa
    stream = torch.cuda.current_stream().cuda_stream
    op = s["case"]["op"]
    if op == "norm_rope":
        pa.qk_norm_rope(s["x"], s["rope"], s["q_out"], s["k_out"], stream=stream)
        return {"q": s["q_out"], "k": s["k_out"]}
    if op == "append":
        pa.append_qkv(s["dtype"], s["x"], s["rope"], s["target"], s["q_out"], stream=stream)
        return _append_outputs(s, s["q_out"])
    pa.paged_decode(pa.KVDtype.FP8_E4M3, s["params"], stream, s["k_pool"].shape[0], d_block_scales=s["scales"])
    return {"out": s["out"]}


# ---- plain forms -----------------------------------------------------------------------------------------------

def _rotated(s, x, weight, positions, ft):
    """Norm (where there is a weight) and rotation of [tokens, heads, D], in the type `ft`, unrounded."""
    case = s["case"]
    x = x.to(ft)
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.to(ft)
    angle = positions[s["axis_dev"]].t().double() * s["inv_freq_dev"]           # [tokens, R/2]
    cos, sin = (f(angle).to(ft).unsqueeze(1) for f in (torch.cos, torch.sin))
    r = case["rotary"]
    if case["interleaved"]:
        lo, hi = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack((lo * cos - hi * sin, hi * cos + lo * sin), -1).flatten(-2)
    else:
        lo, hi = x[..., :r // 2], x[..., r // 2:r]
        y = torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), -1)
    return torch.cat((y, x[..., r:]), -1)


def _to_e4m3(x):
    return x.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float32).to(torch.float8_e4m3fn)


def _append_outputs(s, q):
    out = {"q": q, "k_pool": s["k_pool"], "v_pool": s["v_pool"]}
    if s["case"]["cache"] == "blocks":
        out["scales"] = s["scales"]
    return out


def _append_blocks(s, pool, which, x, seq, place):
    """Tokens x [tokens, hkv, D] into the block-scaled e4m3 pool; scales[..., which] are its scales."""
    case, scales = s["case"], s["scales"]
    page, b = case["page"], _block(case["page"])
    row = s["table"][seq, place // page].long()
    off = place % page
    start = s["start"].long()
    # one line per block that receives tokens: numbered by its sequence and its block within the sequence
    per_seq = s["table"].shape[1] * (page // b)
    line = seq * per_seq + place // b
    amax = torch.zeros(s["table"].shape[0] * per_seq, case["hkv"], dtype=x.dtype, device="cuda")
    amax.index_reduce_(0, line, x.abs().amax(-1), "amax")
    frac, exp = torch.frexp(amax / E4M3_MAX)                                   # amax / max = frac * 2^exp, frac in [0.5, 1)
    exp = torch.where(frac == 0.5, exp - 1, exp).clamp(MIN_SCALE_EXP, MAX_SCALE_EXP)
    exp = torch.where(amax > 0, exp, MIN_SCALE_EXP)
    need = _power_of_two(exp).to(x.dtype)
    # blocks that were begun earlier keep at least their scale, and their tokens move to the new one
    # (every sequence has new tokens here, so the block its tokens start in is its own)
    begun = torch.arange(case["batch"], device="cuda")
    has = start % b != 0
    first_row = s["table"][begun, start // page].long()
    first_blk = start % page // b
    old = scales[first_row, :, first_blk, which].to(x.dtype)                   # [batch, hkv]
    first_line = begun * per_seq + start // b
    need[first_line] = torch.where(has[:, None], torch.maximum(need[first_line], old), need[first_line])
    ratio = torch.where(has[:, None], old / need[first_line], torch.ones_like(old))
    slot = first_blk[:, None] * b + torch.arange(b, device="cuda")             # [batch, b] token slots of those blocks
    kept = pool[first_row[:, None], :, slot].to(x.dtype)                       # [batch, b, hkv, D]
    moved = _to_e4m3(kept * ratio[:, None, :, None])
    pool[first_row[:, None], :, slot] = moved
    pool[row, :, off] = _to_e4m3(x / need[line][..., None])
    scales[row, :, off // b, which] = need[line].to(scales.dtype)


def _run_append(s):
    case = s["case"]
    tokens = s["q"].shape[0]
    i = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(s["token_begin"].long(), i, right=True) - 1
    place = s["start"].long()[seq] + i - s["token_begin"].long()[seq]
    positions = s["positions"] if s["positions"] is not None else place.unsqueeze(0)
    ft = torch.float64 if case["cache"] == "blocks" else torch.float32
    q = _rotated(s, s["q"], s["q_norm"], positions, torch.float32).to(torch.float16)
    k, v = _rotated(s, s["k"], s["k_norm"], positions, ft), s["v"].to(ft)
    page = case["page"]
    row, off = s["table"][seq, place // page].long(), place % page
    if case["cache"] == "fp16":
        s["k_pool"][row, :, off] = k.to(torch.float16)
        s["v_pool"][row, :, off] = v.to(torch.float16)
    elif case["cache"] == "e4m3":
        s["k_pool"][row, :, off] = _to_e4m3(k / s["scales"][0][:, None])
        s["v_pool"][row, :, off] = _to_e4m3(v / s["scales"][1][:, None])
    else:
        _append_blocks(s, s["k_pool"], 0, k, seq, place)
        _append_blocks(s, s["v_pool"], 1, v, seq, place)
    return _append_outputs(s, q)


def _run_decode(s):
    case = s["case"]
    batch, hq, hkv, page = case["batch"], case["hq"], case["hkv"], case["page"]
    rows = s["table"].long()
    b = _block(page)

    def gathered(pool, which):
        """[batch, hkv, tokens, D] in 32 bits, dequantised."""
        scale = s["scales"][rows, :, :, which].repeat_interleave(b, -1)        # [batch, pages, hkv, page]
        x = pool[rows].float() * scale[..., None]
        return x.transpose(1, 2).reshape(batch, hkv, -1, D)

    q = s["q"].float().view(batch, hkv, hq // hkv, D)
    score = q @ gathered(s["k_pool"], 0).transpose(-1, -2) / math.sqrt(D)      # [batch, hkv, group, tokens]
    dead = torch.arange(score.shape[-1], device="cuda") >= s["lens"][:, None, None, None]
    score = score.masked_fill(dead, -math.inf)
    p = (score - score.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    return {"out": (p @ gathered(s["v_pool"], 1)).reshape(batch, hq, D).to(torch.float16)}


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "norm_rope":
        act = TYPES[state["case"]["act"]]
        return {n: _rotated(state, state[n], state[n + "_norm"], state["positions"], torch.float32).to(act) for n in ("q", "k")}
    return _run_append(state) if op == "append" else _run_decode(state)


# ---- from the definition, in 64 bits ---------------------------------------------------------------------------

def _exact_rows(case, s, x, weight, pos):
    """Rotation as a product of complex numbers.  pos: [axes, tokens] float64."""
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * weight.double()
    r = case["rotary"]
    turn = torch.stack([pos[a] * f for f, a in zip(s["inv_freq"], s["axis"])], -1)
    unit = torch.polar(torch.ones_like(turn), turn)[:, None]
    y = x.clone()
    if case["interleaved"]:
        z = torch.view_as_complex(x[..., :r].reshape(*x.shape[:-1], r // 2, 2).contiguous()) * unit
        y[..., :r] = torch.view_as_real(z).reshape(*x.shape[:-1], r)
    else:
        z = torch.complex(x[..., :r // 2].contiguous(), x[..., r // 2:r].contiguous()) * unit
        y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
    return y


def _exact_append(case, s):
    """Sequence by sequence; e4m3 pools as the unrounded multiples of their scales."""
    new, past = _new_and_past(case)
    page, hkv = case["page"], case["hkv"]
    b = _block(page)
    pools = [s["k_pool"].double(), s["v_pool"].double()]
    scales = s["scales"].double() if s["scales"] is not None else None
    place = torch.cat([torch.arange(o, o + n, device="cuda") for n, o in zip(new, past)])
    pos = s["positions"].double() if s["positions"] is not None else place.double()[None]
    q = _exact_rows(case, s, s["q"], s["q_norm"], pos)
    rows = [_exact_rows(case, s, s["k"], s["k_norm"], pos), s["v"].double()]
    at = 0
    for i, (n, o) in enumerate(zip(new, past)):
        where = torch.arange(o, o + n, device="cuda")
        pages, offs = s["table"][i, where // page].long(), where % page
        for which in range(2):
            x = rows[which][at:at + n]
            if case["cache"] == "e4m3":
                x = (x / scales[which][:, None]).clamp(-E4M3_MAX, E4M3_MAX)
            elif case["cache"] == "blocks":
                lo = o // b
                blocks = (o + n - 1) // b - lo + 1
                padded = torch.zeros(blocks * b, hkv, D, dtype=torch.float64, device="cuda")
                padded[o - lo * b:o - lo * b + n] = x
                top = padded.view(blocks, b, hkv, D).abs().amax((1, 3))         # [blocks, hkv]
                # the smallest power of two that brings the block's largest value to at most 448
                want = torch.full_like(top, 2.0 ** MIN_SCALE_EXP)
                for e in range(MIN_SCALE_EXP, MAX_SCALE_EXP):
                    want = torch.where(top > 448.0 * 2.0 ** e, torch.full_like(top, 2.0 ** (e + 1)), want)
                if o % b:
                    page0, blk0 = int(s["table"][i, o // page]), o % page // b
                    was = scales[page0, :, blk0, which].clone()
                    want[0] = torch.maximum(want[0], was)
                    pools[which][page0, :, blk0 * b:blk0 * b + b] *= (was / want[0])[:, None, None]
                mine = want[where // b - lo]                                    # [n, hkv]
                x = (x / mine[..., None]).clamp(-E4M3_MAX, E4M3_MAX)
                scales[pages, :, offs // b, which] = mine
            pools[which][pages, :, offs] = x
        at += n
    out = {"q": q, "k_pool": pools[0], "v_pool": pools[1]}
    if case["cache"] == "blocks":
        out["scales"] = scales
    return out


def _exact_decode(case, s):
    hq, hkv, page = case["hq"], case["hkv"], case["page"]
    b = _block(page)
    out = torch.empty(case["batch"], hq, D, dtype=torch.float64, device="cuda")
    for i, n in enumerate(_lens(case)):
        t = torch.arange(n, device="cuda")
        pages, offs = s["table"][i, t // page].long(), t % page
        k = s["k_pool"].view(torch.uint8)[pages, :, offs].view(torch.float8_e4m3fn).double()
        v = s["v_pool"].view(torch.uint8)[pages, :, offs].view(torch.float8_e4m3fn).double()
        k *= s["scales"][pages, :, offs // b, 0].double()[..., None]            # [n, hkv, D]
        v *= s["scales"][pages, :, offs // b, 1].double()[..., None]
        q = s["q"][i].double().view(hkv, hq // hkv, D)
        w = torch.softmax(torch.einsum("hgd,nhd->hgn", q, k) * D ** -0.5, -1)
        out[i] = torch.einsum("hgn,nhd->hgd", w, v).reshape(hq, D)
    return {"out": out}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm_rope":
        pos = s["positions"].double()
        return {n: _exact_rows(case, s, s[n], s[n + "_norm"], pos) for n in ("q", "k")}
    return _exact_append(case, s) if case["op"] == "append" else _exact_decode(case, s)
