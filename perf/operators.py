"""The operators around the paged latent cache that serve many users at once, as timed cases.

  rows    new rows enter a cache that holds E4M3 values, and are read back: quantised as they are
          written (groups of 64 latent values with a power-of-two scale, the rope dims stay bf16)
  attend  absorbed attention of new query tokens over such a cache: decode and verify blocks
  prefix  absorbed attention of a batch whose sequences share a long prefix (one set of pages, a
          system prompt or a document) and go on with rows of their own; bf16 or E4M3 cache

Shapes are the framework's two forms: "baseline" rows of 576 = 512 latent + 64 rope values, "v4" rows of
512 with the rope dims at their tail, a sink logit per head and the inverse rotation of the output tail.
64 heads.  Where `own` is false `run` computes in plain torch operations in 32 bits.
"""
import math
import random

import torch

own = False

HEADS, ROPE, D_V, PAGE, GROUP = 64, 64, 512, 64, 64
MAX_STEP = 512  # rows of a chunk in which `prepare` fills a cache


def _case(name, op, preset="baseline", cache="e4m3", batch=1, q=(1, 1), ctx=(1, 1), prefix=0):
    """q: new tokens per sequence; ctx: rows cached before them (behind the prefix, if there is one)."""
    return {"name": name, "op": op, "preset": preset, "cache": cache, "batch": batch, "q_lo": q[0], "q_hi": q[1],
            "ctx_lo": ctx[0], "ctx_hi": ctx[1], "prefix": prefix}


def listed():
    return [
        # a decode step of 64 users: one new row each, somewhere in a page
        _case("rows_64x1", "rows", batch=64, ctx=(1000, 5000)),
        # chunks of five prompts of uneven length
        _case("rows_v4_5", "rows", preset="v4", batch=5, q=(130, 900), ctx=(0, 300)),
        # a long prompt in one chunk
        _case("rows_1x8191", "rows", q=(8191, 8191), ctx=(0, 0)),
        # one chat at its start
        _case("attend_1x300", "attend", ctx=(300, 300)),
        # one very long document
        _case("attend_1x131072", "attend", ctx=(131072, 131072)),
        # the batched-decode workload of the benchmark: 64 users, 1024 to 8192 cached rows
        _case("attend_64", "attend", batch=64, ctx=(1024, 8192)),
        # many users with short contexts, the live engine's form
        _case("attend_v4_192", "attend", preset="v4", batch=192, ctx=(250, 2000)),
        # speculative verify: 16 causal rows of each of 8 sequences over 16384 cached rows
        _case("attend_8x16x16384", "attend", batch=8, q=(16, 16), ctx=(16384, 16384)),
        # eight users of one assistant whose instructions take 4000 rows
        _case("prefix_8x4000", "prefix", cache="bf16", batch=8, ctx=(1, 250), prefix=4000),
        # 200 short questions on one page of text, the live engine's form
        _case("prefix_v4_200x1500", "prefix", preset="v4", cache="bf16", batch=200, ctx=(10, 120), prefix=1500),
        # 64 users over one document
        _case("prefix_64x16384", "prefix", batch=64, ctx=(20, 700), prefix=16384),
        # 24 users over a book that the L2 cache does not hold
        _case("prefix_24x130000", "prefix", cache="bf16", batch=24, ctx=(20, 700), prefix=130000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rows", "attend", "attend", "prefix", "prefix"])
    preset = rng.choice(["baseline", "v4"])
    if op == "rows":
        batch = _log(rng, 1, 256)
        hi = _log(rng, 1, max(1, 8191 // batch))
        lo = rng.randint(max(1, hi // 4), hi)
        c0 = rng.choice([0, _log(rng, 1, 5000)])
        c = _case("", op, preset=preset, batch=batch, q=(lo, hi), ctx=(c0 // 2, c0))
    elif op == "attend":
        if rng.random() < 0.6:
            batch = _log(rng, 1, 256)
            hi = _log(rng, 1, min(131072 if preset == "baseline" else 8192, 280000 // batch))
            c = _case("", op, preset=preset, batch=batch, ctx=(rng.randint(max(1, hi // 8), hi), hi))
        else:
            batch = _log(rng, 1, 16)
            q = (rng.randint(1, 16),) * 2 if rng.random() < 0.6 else (1, rng.randint(2, 40))
            hi = _log(rng, 1, min(8192, 1800000 // (batch * q[1])))
            c = _case("", op, preset=preset, batch=batch, q=q, ctx=(rng.randint(max(1, hi // 2), hi), hi))
    else:
        batch = _log(rng, 2, 256)
        prefix = _log(rng, 60, min(120000 if preset == "baseline" else 8192, 2500000 // batch))
        hi = rng.randint(1, 700)
        c = _case("", op, preset=preset, cache=rng.choice(["bf16", "e4m3"]), batch=batch, ctx=(rng.randint(1, hi), hi),
                  prefix=prefix)
    del c["name"]
    return c


def _spread(lo, hi, n, phase):
    """n whole numbers spread over [lo, hi], not in order."""
    if n == 1:
        return [hi]
    return [lo + int((hi - lo) * ((phase + i * 0.6180339887498949) % 1.0)) for i in range(n)]


def _sizes(case):
    """(new tokens, rows cached in front of them) of every sequence; the prefix is not counted."""
    return (_spread(case["q_lo"], case["q_hi"], case["batch"], 0.5),
            _spread(case["ctx_lo"], case["ctx_hi"], case["batch"], 0.0))


def _dims(case):
    """(row width, quantised values of a row, scale of the scores)"""
    return (576, 512, 192.0 ** -0.5) if case["preset"] == "baseline" else (512, 448, 512.0 ** -0.5)


# ---- inputs ------------------------------------------------------------------------------------------


def _rows(gen, n, row, n8):
    """Cache rows as a layer's norm leaves them: channels of their own size, here and there one that stands out."""
    channel = torch.randn(row, generator=gen, device="cuda").mul_(0.5).exp_()
    channel[torch.randint(0, n8, (8,), generator=gen, device="cuda")] *= 8.0
    return torch.randn(n, row, generator=gen, device="cuda").mul_(channel).to(torch.bfloat16)


def _pow2(k):
    """2^k in 32 bits, from its bits (a pow() on the device need not end on the very value)."""
    return ((k.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantize(rows, n8):
    """bf16 rows -> E4M3 values (in 32 bits), the exponents of their groups' scales, the rope dims."""
    x = rows[:, :n8].float().reshape(rows.shape[0], n8 // GROUP, GROUP)
    m, e = torch.frexp(x.abs().amax(-1, keepdim=True))
    k = torch.clamp(e - 9 + (m > 0.875), -100, 120)  # the least k with |x| <= 448 * 2^k; 448 = 0.875 * 2^9
    y = x * _pow2(-k)
    step = torch.clamp(torch.frexp(y).exponent - 1, min=-6) - 3  # three bits behind the leading one, or 2^-9
    y = torch.round(y * _pow2(-step)) * _pow2(step)
    return y, k, rows[:, n8:]


def _dequantize(y, k, rope):
    return torch.cat([(y.float() * _pow2(k)).reshape(y.shape[0], y.shape[1] * GROUP), rope.float()], 1)


def _fill(ctx, seq, pos, rows):
    for i in range(0, rows.shape[0], MAX_STEP):
        part = rows[i:i + MAX_STEP]
        ctx.plan([(seq, pos + i, part.shape[0])])
        ctx.cache_append_device(0, part.data_ptr())


def _context(case, st):
    """The handle that a serving process keeps: a context with the sequences' rows in its cache and the step's plan."""
    from fastar_b200 import mla
    v4 = case["preset"] == "v4"
    ends = [c + q for c, q in zip(st["ctx"], st["q"])]
    shared = case["prefix"] // PAGE
    pages = sum((case["prefix"] + e + PAGE - 1) // PAGE - shared + 1 for e in ends) + shared + 2
    cfg = mla.make_config(mla.PRESET_FASTAR_V4 if v4 else mla.PRESET_BASELINE, hidden=64, q_lora=64, o_lora=64,
                          n_pages=pages, max_seqs=case["batch"] + 1, max_tokens=max(sum(st["q"]), MAX_STEP))
    ctx = mla.MlaContext(cfg)
    if case["cache"] == "e4m3":
        ctx.set_cache_format(mla.CACHE_E4M3)
    if v4 and case["op"] != "rows":
        import numpy as np
        w = {name: np.zeros(shape, np.uint16) for name, shape in mla.weight_shapes(cfg).items()}
        w["attn_sinks"] = st["sinks"].cpu().numpy()
        ctx.set_layer_weights(0, w)
    if case["prefix"]:
        base = ctx.seq_alloc()
        _fill(ctx, base, 0, st["prefix_rows"])
        seqs = [ctx.seq_fork(base, case["prefix"]) for _ in ends]
    else:
        seqs = [ctx.seq_alloc() for _ in ends]
    # the sequences grow side by side: their pages are interleaved
    grow = [b for b, e in enumerate(ends) for _ in range(0, e, PAGE)]
    random.Random(st["seed"]).shuffle(grow)
    have = [0] * len(ends)
    for b in grow:
        have[b] = min(have[b] + PAGE, ends[b])
        ctx.seq_reserve(seqs[b], case["prefix"] + have[b])
    st["seqs"], st["handle"] = seqs, ctx
    if case["op"] == "rows":
        st["ranges"] = mla.seq_steps([(s, c, q) for s, c, q in zip(seqs, st["ctx"], st["q"])])
        ctx.plan(st["ranges"])
    else:
        at = 0
        for s, e in zip(seqs, ends):
            _fill(ctx, s, case["prefix"], st["rows"][at:at + e])
            at += e
        ctx.plan([(s, case["prefix"] + c, q) for s, c, q in zip(seqs, st["ctx"], st["q"])], causal=True)
    ctx.sync()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    row, n8, scale = _dims(case)
    q, ctx = _sizes(case)
    T = sum(q)
    st = {"case": case, "seed": seed, "q": q, "ctx": ctx, "scale": scale}
    if case["op"] == "rows":
        st["rows"] = _rows(gen, T, row, n8)
        st["out"] = torch.zeros_like(st["rows"])
    else:
        st["prefix_rows"] = _rows(gen, case["prefix"], row, n8)
        st["rows"] = _rows(gen, sum(ctx) + T, row, n8)
        st["q_eff"] = torch.randn(T * HEADS, row, generator=gen, device="cuda").to(torch.bfloat16)
        st["out"] = torch.zeros(T * HEADS, D_V, dtype=torch.bfloat16, device="cuda")
        st["sinks"] = torch.randn(HEADS, generator=gen, device="cuda") if case["preset"] == "v4" else None
        st["where"] = _where(case, q, ctx)
    if own:
        _context(case, st)
    elif case["cache"] == "e4m3" and case["op"] != "rows":
        # the cache as it is held: a byte per latent value
        for name in ("prefix_rows", "rows"):
            y, k, rope = _quantize(st[name], n8)
            st[name] = (y.to(torch.float8_e4m3fn), k, rope)
    torch.cuda.synchronize()
    return st


def _where(case, q, ctx):
    """Index tables: the rows of every sequence, and of every token what it sees of them.  Sequences are padded to the longest one's
    rows and tokens; what is padded points at row 0 or token 0 and is masked or dropped."""
    ends = torch.tensor([c + n for c, n in zip(ctx, q)], device="cuda")
    n_q, n_c = torch.tensor(q, device="cuda"), torch.tensor(ctx, device="cuda")
    first = torch.cumsum(ends, 0) - ends
    i = torch.arange(int(ends.max()), device="cuda")
    t = torch.arange(max(q), device="cuda")
    tok0 = torch.cumsum(n_q, 0) - n_q
    inside = t[None] < n_q[:, None]
    return {"row": torch.where(i[None] < ends[:, None], first[:, None] + i[None], 0),
            "tok": torch.where(inside, tok0[:, None] + t[None], 0),
            "sees": i[None, None] <= (n_c[:, None] + t[None])[:, :, None],  # causal: rows up to the token's own
            "inside": inside,
            "pos": (case["prefix"] + n_c[:, None] + t[None])[inside]}


# ---- one pass ----------------------------------------------------------------------------------------


def run(st):
    case = st["case"]
    if own:
        ctx = st["handle"]
        if case["op"] == "rows":
            ctx.cache_append_device(0, st["rows"].data_ptr())
            ctx.cache_read_device(0, st["ranges"], st["out"].data_ptr())
        else:
            ctx.attention_device(0, st["q_eff"].data_ptr(), st["out"].data_ptr())
        return st["out"]
    row, n8, scale = _dims(case)
    if case["op"] == "rows":
        return _dequantize(*_quantize(st["rows"], n8)).to(torch.bfloat16)
    prefix, rows = (_dequantize(*st[n]) if case["cache"] == "e4m3" else st[n].float() for n in ("prefix_rows", "rows"))
    w = st["where"]
    B, G = w["tok"].shape
    q = st["q_eff"].float().reshape(-1, HEADS, row)[w["tok"]]  # [sequence, token, head, row]
    k = rows[w["row"]]  # [sequence, cached row, row]
    s = torch.matmul(q.reshape(B, G * HEADS, row), k.transpose(1, 2)).reshape(B, G, HEADS, -1) * scale
    s = torch.where(w["sees"][:, :, None], s, -math.inf)
    top = s.amax(-1, keepdim=True)
    if case["prefix"]:
        s0 = torch.matmul(q, prefix.T) * scale  # the whole batch against the one prefix
        top = torch.maximum(top, s0.amax(-1, keepdim=True))
    sinks = st["sinks"]
    if sinks is not None:
        top = torch.maximum(top, sinks[:, None])
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(B, G * HEADS, -1), k[:, :, :D_V]).reshape(B, G, HEADS, D_V)
    if case["prefix"]:
        p0 = torch.exp(s0 - top)
        total = total + p0.sum(-1, keepdim=True)
        o = o + torch.matmul(p0, prefix[:, :D_V])
    if sinks is not None:
        total = total + torch.exp(sinks[:, None] - top)
    o = (o / total)[w["inside"]]  # [token, head, value]
    if case["preset"] == "v4":  # the output's tail back by the angle of the token's position
        j = torch.arange(ROPE // 2, device=o.device, dtype=torch.float64)
        angle = w["pos"].double()[:, None, None] * 10000.0 ** (-2.0 * j / ROPE)
        c, sn = torch.cos(angle).float(), torch.sin(angle).float()
        x0, x1 = o[..., D_V - ROPE::2], o[..., D_V - ROPE + 1::2]
        tail = torch.stack([x0 * c + x1 * sn, x1 * c - x0 * sn], -1).flatten(-2)
        o = torch.cat([o[..., :D_V - ROPE], tail], -1)
    return o.reshape(-1, D_V).to(torch.bfloat16)


def work(case):
    """Every row, query and output once; an E4M3 row is a byte per latent value, one per group, and its rope dims."""
    row, n8, _ = _dims(case)
    q, ctx = _sizes(case)
    T = sum(q)
    held = n8 + n8 // GROUP + 2 * ROPE if case["cache"] == "e4m3" else 2 * row
    if case["op"] == "rows":
        return {"bytes": T * (2 * row + held + held + 2 * row), "flops": 4 * T * n8}
    pairs = sum(n * (case["prefix"] + c) + n * (n + 1) // 2 for n, c in zip(q, ctx))
    return {"bytes": (case["prefix"] + sum(ctx) + T) * held + 2 * T * HEADS * (row + D_V),
            "flops": 2 * HEADS * (row + D_V) * pairs}


# ---- the same in 64 bits, from the definitions --------------------------------------------------------


def _e4m3_grid():
    """The non-negative E4M3 values: eight subnormal steps of 2^-9, then 1.000 to 1.111 times 2^-6 .. 2^8, without the last."""
    low = [m * 2.0 ** -9 for m in range(8)]
    return low + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1]


def _held(rows, n8):
    """What an E4M3 cache holds of these rows, in 64 bits: the nearest grid value of every latent value, ties to the even one."""
    grid = torch.tensor(_e4m3_grid(), dtype=torch.float64, device=rows.device)
    x = rows.double()
    out = x.clone()
    for g in range(0, n8, GROUP):
        part = x[:, g:g + GROUP]
        most = part.abs().max(1, keepdim=True).values
        k = torch.clamp(torch.ceil(torch.log2(torch.clamp(most, min=1e-300) / 448.0)), -100, 120)
        scale = ((k.long() + 1023) << 52).view(torch.float64)
        scale = torch.where(most > 448.0 * scale, scale * 2, scale)  # log2 may end on the wrong side of a whole number
        scale = torch.where(most <= 224.0 * scale, torch.clamp(scale / 2, min=2.0 ** -100), scale)
        a = part.abs() / scale
        hi = torch.clamp(torch.searchsorted(grid, a.contiguous()), max=len(grid) - 1)
        lo = torch.clamp(hi - 1, min=0)
        up, down = grid[hi] - a, a - grid[lo]
        near = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), grid[hi], grid[lo])
        out[:, g:g + GROUP] = torch.copysign(near, part) * scale
    return out


def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare({**case, "cache": "bf16"}, seed)  # the rows as they were made, unquantised
    finally:
        own = was
    row, n8, scale = _dims(case)
    if case["op"] == "rows":
        return _held(st["rows"], n8)
    hold = (lambda r: _held(r, n8)) if case["cache"] == "e4m3" else (lambda r: r.double())
    prefix, rows = hold(st["prefix_rows"]), hold(st["rows"])
    out = torch.zeros(sum(st["q"]), HEADS, D_V, dtype=torch.float64, device="cuda")
    at = tok = 0
    for n, c in zip(st["q"], st["ctx"]):
        seen = torch.cat([prefix, rows[at:at + c + n]])
        at += c + n
        for i in range(n):
            keys = seen[:case["prefix"] + c + i + 1]
            logits = (st["q_eff"][(tok + i) * HEADS:(tok + i + 1) * HEADS].double() @ keys.T) * scale
            if st["sinks"] is not None:
                logits = torch.cat([logits, st["sinks"].double()[:, None]], 1)
            weight = torch.softmax(logits, 1)[:, :keys.shape[0]]
            o = weight @ keys[:, :D_V]
            if case["preset"] == "v4":
                pos = case["prefix"] + c + i
                turn = torch.polar(torch.ones(ROPE // 2, dtype=torch.float64, device="cuda"),
                                   -pos * 10000.0 ** (-torch.arange(0, ROPE, 2, dtype=torch.float64, device="cuda") / ROPE))
                tail = torch.view_as_complex(o[:, D_V - ROPE:].reshape(HEADS, ROPE // 2, 2).contiguous()) * turn
                o[:, D_V - ROPE:] = torch.view_as_real(tail).reshape(HEADS, ROPE)
            out[tok + i] = o
        tok += n
    return out.reshape(-1, D_V)
