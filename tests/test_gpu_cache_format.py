"""The E4M3 cache: rows quantised as they are written (every entry point that writes rows), read back, and the
attention over them.  Quantised values are compared bit for bit with the definition in plain numpy; the attention with
softmax(scale * q K^T) V in 64 bits over the values that the cache stands for, and with the bf16 cache that holds
those values."""
import math

import numpy as np
import pytest

from fastar_b200 import mla, synth

pytestmark = pytest.mark.gpu

bits, f32 = synth.to_bf16_bits, synth.from_bf16_bits


def grid():
    low = [m * 2.0 ** -9 for m in range(8)]
    return np.array(low + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1])


def held(rows, n8):
    """The definition, in 64 bits: bf16 values [n, row] -> the values an E4M3 cache holds."""
    x = np.asarray(rows, np.float64)
    out = x.copy()
    g = grid()
    top = 1.875 * 2.0 ** 127
    for c in range(0, n8, 64):
        part = x[:, c:min(c + 64, n8)]
        for r in range(x.shape[0]):
            v = part[r]
            if np.isnan(v).any():
                out[r, c:c + v.size] = np.nan
                continue
            v = np.clip(v, -top, top)
            a = np.abs(v).max()
            k = -100
            while k < 120 and a > 448.0 * 2.0 ** k:
                k += 1
            y = np.abs(v) / 2.0 ** k
            hi = np.minimum(np.searchsorted(g, y), len(g) - 1)
            lo = np.maximum(hi - 1, 0)
            up, down = g[hi] - y, y - g[lo]
            q = np.where((up < down) | ((up == down) & (hi % 2 == 0)), g[hi], g[lo])
            out[r, c:c + v.size] = np.copysign(q, v) * 2.0 ** k
    return out


def same_values(got_bits, want):
    got = f32(got_bits).astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    bad = np.argwhere(ok & (got != want))
    assert bad.size == 0, (bad[:4], [(got[tuple(b)], want[tuple(b)]) for b in bad[:4]])


def awkward_rows(rng, n, row):
    """Rows of every kind of value: ordinary, of one sign, zeros, ties between two codes, tiny, subnormal, huge."""
    x = rng.standard_normal((n, row)).astype(np.float32) * np.exp(rng.standard_normal(row)).astype(np.float32)
    with np.errstate(over="ignore", under="ignore"):
        for r in range(n):
            kind = r % 12
            if kind == 1:
                x[r] = 0.0
            elif kind == 2:
                x[r] = rng.integers(-480, 480, row)          # ties at 8-bit integers
            elif kind == 3:
                x[r] *= 2.0 ** -120
            elif kind == 4:
                x[r] *= np.float32(2.0 ** 100)
            elif kind == 5:
                x[r, ::3] *= 2.0 ** -16                     # far below the group's largest: E4M3 subnormals and zeros
            elif kind == 6:
                x[r] = 448.0 * 2.0 ** rng.integers(-3, 4)   # exactly the largest value of a scale
            elif kind == 7:
                x[r] = np.float32(450.0)                    # just above it
            elif kind == 8:
                x[r, :64] = 2.0 ** -130                     # bf16 subnormals
            elif kind == 9:
                x[r, 5] = 1.99 * 2.0 ** 127
            elif kind == 10:
                x[r, 70] = -1e5                             # one value far above 57344, scale 2^8
            elif kind == 11:
                x[r] = -np.abs(x[r])
    return bits(x)


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


def dev(torch, a):
    return torch.from_numpy(np.ascontiguousarray(a).view(np.int16)).cuda()


def host(t):
    return t.cpu().numpy().view(np.uint16)


def make(preset=mla.PRESET_BASELINE, e4m3=True, **kw):
    kw = {**dict(hidden=64, q_lora=64, o_lora=64, n_pages=64, max_seqs=8, max_tokens=64), **kw}
    cfg = mla.make_config(preset, **kw)
    ctx = mla.MlaContext(cfg)
    if e4m3:
        ctx.set_cache_format(mla.CACHE_E4M3)
    return ctx


def n8_of(ctx):
    return ctx.dims["row"] - ctx.cfg.qk_rope


SHAPES = [
    dict(preset=mla.PRESET_BASELINE),
    dict(preset=mla.PRESET_FASTAR_V4),
    # narrow rows, pages of 32: 64 latent values and a rope part of 16; a last group of 48 values in the V4 form
    dict(preset=mla.PRESET_BASELINE, kv_lora=64, qk_rope=16, n_heads=3, page_tokens=32, n_pages=100),
    dict(preset=mla.PRESET_FASTAR_V4, kv_lora=128, qk_rope=16, n_heads=8, o_groups=8, page_tokens=24, n_pages=100),
]


@pytest.mark.parametrize("shape", SHAPES)
def test_rows_written_and_read_back(torch, shape):
    """Device append and read-back, host write and read: the same values, whatever page boundary is crossed."""
    rng = np.random.default_rng(3)
    with make(n_layers=2, max_tokens=200, **shape) as ctx:
        row, n8 = ctx.dims["row"], n8_of(ctx)
        pt = ctx.cfg.page_tokens
        assert ctx.cache_page_bytes() < pt * row * 2
        lens = [1, pt + 1, 131]
        seqs = [ctx.seq_alloc() for _ in lens]
        rows = awkward_rows(rng, sum(lens), row)
        want = held(f32(rows), n8)
        d_rows = dev(torch, rows)
        ctx.plan([(s, 3, n) for s, n in zip(seqs, lens)])  # from row 3 on
        ctx.cache_append_device(1, d_rows.data_ptr())
        d_out = dev(torch, np.full((sum(lens) + 1, row), 0x7777, np.uint16))
        ctx.cache_read_device(1, [(s, 3, n) for s, n in zip(seqs, lens)], d_out.data_ptr())
        ctx.sync()
        got = host(d_out)
        same_values(got[:-1], want)
        assert (got[-1] == 0x7777).all()  # behind the last row: left as it was
        # the other layer, and the rows in front, hold nothing
        for s in seqs:
            assert not ctx.cache_read(0, s, 0, ctx.seq_len(s)).any()
            assert not ctx.cache_read(1, s, 0, 3).any()
        # host read, a part of a sequence, the same sequence twice
        at = lens[0] + lens[1]
        assert np.array_equal(ctx.cache_read(1, seqs[2], 3 + 20, 100), got[at + 20:at + 120])
        ctx.cache_read_device(1, [(seqs[2], 23, 2), (seqs[0], 3, 0), (seqs[2], 23, 2)], d_out.data_ptr())
        ctx.sync()
        got2 = host(d_out)
        assert np.array_equal(got2[:2], got[at + 20:at + 22]) and np.array_equal(got2[2:4], got2[:2])
        # host write into the other layer
        ctx.cache_write(0, seqs[2], 3, rows[at:at + 131])
        assert np.array_equal(ctx.cache_read(0, seqs[2], 3, 131), got[at:at + 131])
        # what is read back can be written again without a change
        ctx.cache_write(0, seqs[2], 3, got[at:at + 131])
        back = ctx.cache_read(0, seqs[2], 3, 131)
        finite = np.isfinite(want[at:at + 131])
        assert np.array_equal(back[finite], got[at:at + 131][finite])


def test_more_pages_than_a_kernel_argument_holds(torch):
    """A read-back and a host write over 300 pages: staged runs, more than one turn."""
    rng = np.random.default_rng(4)
    with make(n_pages=330, max_seqs=2, max_tokens=8) as ctx:
        s, t = ctx.seq_alloc(), ctx.seq_alloc()
        for n in range(64, 64 * 301, 64):  # interleave the pages of two sequences
            ctx.seq_reserve(s, n)
            if n % 640 == 0:
                ctx.seq_reserve(t, n // 10)
        n = 64 * 300 - 5
        rows = bits(rng.standard_normal((n, 576)).astype(np.float32))
        ctx.cache_write(0, s, 0, rows)
        want = held(f32(rows[:200]), 512)
        out = torch.zeros(n, 576, dtype=torch.int16, device="cuda")
        for _ in range(2):
            ctx.cache_read_device(0, [(s, 0, n)], out.data_ptr())
        ctx.sync()
        got = host(out)
        assert np.array_equal(got, ctx.cache_read(0, s, 0, n))
        same_values(got[:200], want)
        # rounding: half a step of three bits
        x = f32(rows)[:, :512].astype(np.float64)
        # (half of 2^-3 at the value, or of the smallest step 2^-9 of a group whose largest value is over 224 steps of 2^k)
        top = np.abs(x.reshape(n, 8, 64)).max(2).repeat(64, 1)
        assert (np.abs(f32(got)[:, :512] - x) <= np.maximum(np.abs(x) / 16, top / 224 * 2.0 ** -10)).all()
        assert np.array_equal(got[:, 512:], rows[:, 512:])


def test_nan_stays_in_its_group(torch):
    with make() as ctx:
        s = ctx.seq_alloc()
        x = np.random.default_rng(5).standard_normal((4, 576)).astype(np.float32)
        x[1, 100] = np.nan
        x[2, 0] = np.inf
        x[2, 1] = -np.inf
        x[3, 570] = np.nan
        rows = bits(x)
        ctx.cache_write(0, s, 0, rows)
        got = f32(ctx.cache_read(0, s, 0, 4))
        assert np.isnan(got[1, 64:128]).all() and np.isfinite(got[1, :64]).all() and np.isfinite(got[1, 128:]).all()
        assert got[2, 0] == 1.875 * 2.0 ** 127 and got[2, 1] == -1.875 * 2.0 ** 127
        assert np.isnan(got[3, 570]) and np.isfinite(got[3, :570]).all()


def test_truncate_zeroes_and_reset_clears(torch):
    with make(n_layers=2) as ctx:
        s = ctx.seq_alloc()
        rows = bits(np.random.default_rng(6).standard_normal((150, 576)).astype(np.float32))
        ctx.cache_write(0, s, 0, rows)
        ctx.cache_write(1, s, 0, rows)
        kept = ctx.cache_read(1, s, 0, 70)
        ctx.seq_truncate(s, 70)
        ctx.seq_reserve(s, 192)
        assert np.array_equal(ctx.cache_read(1, s, 0, 70), kept)
        assert not ctx.cache_read(1, s, 70, 122).any() and not ctx.cache_read(0, s, 70, 122).any()
        assert ctx.pool_read(0).shape == (64, ctx.cache_page_bytes())
        ctx.reset()
        assert not ctx.pool_read(0).any() and not ctx.pool_read(1).any()


def plain_attention(q, keys, d_v, scale, sink=None):
    """64-bit softmax(scale * q K^T) V; q [H, d], keys [n, d]."""
    logits = q @ keys.T * scale
    top = logits.max(1) if keys.shape[0] else np.full(q.shape[0], -np.inf)
    if sink is not None:
        top = np.maximum(top, sink)
    w = np.exp(logits - top[:, None])
    den = w.sum(1) + (np.exp(sink - top) if sink is not None else 0.0)
    return w @ keys[:, :d_v] / den[:, None], np.abs(w) @ np.abs(keys[:, :d_v]) / den[:, None]


def unrotate(o, pos, rope, theta=10000.0):
    o = o.copy()
    ang = pos * theta ** (-2.0 * np.arange(rope // 2) / rope)
    x0, x1 = o[:, -rope::2].copy(), o[:, -rope + 1::2].copy()
    o[:, -rope::2] = x0 * np.cos(ang) + x1 * np.sin(ang)
    o[:, -rope + 1::2] = x1 * np.cos(ang) - x0 * np.sin(ang)
    return o


def check_attention(got_bits, q, keys_of, d_v, scale, sinks, pos, rope, v4):
    """Each weight and each output are rounded to bf16 once (2^-9 of the value each); the V4 form rounds the output before
    the inverse rotation too; sums are 32-bit (2^-16 covers the longest here).  The bound per element: 2^-8 of
    sum_j p_j |v_j| for the weights (half a step and the differences of exp2 in 32 bits), plus 2^-8 (V4: 2^-7) of the output."""
    got = f32(got_bits).astype(np.float64)
    for t, keys in enumerate(keys_of):
        H = got.shape[1]
        if keys.shape[0] == 0:
            assert not got[t].any()
            continue
        o, a = plain_attention(q[t], keys, d_v, scale, sinks)
        tol = 2.0 ** -8 * a + 2.0 ** -8 * np.abs(o)
        if v4:
            o = unrotate(o, pos[t], rope)
            tol = 2.0 ** -8 * a + 2.0 ** -7 * np.abs(o)
            pair = tol[:, -rope:].reshape(H, rope // 2, 2).sum(2).repeat(2, 1)  # a rotated value has errors of both
            tol[:, -rope:] = pair + 2.0 ** -12 * np.abs(pair)
            tol += 2.0 ** -11 * np.abs(o).max()  # 32-bit angles at positions up to some thousand
        err = np.abs(got[t] - o)
        assert (err <= tol + 1e-30).all(), (t, float((err / (tol + 1e-30)).max()))


ATTEND = [
    # (preset, batch of (cached rows, new tokens), causal)
    (mla.PRESET_BASELINE, [(0, 1)], False),
    (mla.PRESET_BASELINE, [(62, 1), (63, 1), (64, 1), (1, 1)], False),
    (mla.PRESET_BASELINE, [(1000, 1), (5, 1), (129, 1)], False),
    (mla.PRESET_BASELINE, [(300, 7), (300, 7)], True),
    (mla.PRESET_BASELINE, [(0, 40), (70, 3), (0, 1)], True),
    (mla.PRESET_BASELINE, [(6000, 1)], False),
    (mla.PRESET_FASTAR_V4, [(0, 1)], False),
    (mla.PRESET_FASTAR_V4, [(62, 1), (63, 1), (64, 1), (1, 1)], False),
    (mla.PRESET_FASTAR_V4, [(1000, 5), (40, 5)], True),
    (mla.PRESET_FASTAR_V4, [(2500, 1), (128, 1)], False),
]


@pytest.mark.parametrize("impl", [mla.IMPL_TENSOR, mla.IMPL_SIMT])
@pytest.mark.parametrize("preset,batch,causal", ATTEND)
def test_attention_over_quantised_rows(torch, preset, batch, causal, impl):
    rng = np.random.default_rng(7)
    v4 = preset == mla.PRESET_FASTAR_V4
    T = sum(q for _, q in batch)
    kw = dict(n_pages=160, max_tokens=64, attn_impl=impl)
    with make(preset, **kw) as ctx, make(preset, e4m3=False, **kw) as plain:
        row, n8 = ctx.dims["row"], n8_of(ctx)
        sinks = rng.standard_normal(64).astype(np.float32) if v4 else None
        w = {n: np.zeros(sh, np.uint16) for n, sh in mla.weight_shapes(ctx.cfg).items()}
        w["attn_sinks"] = sinks
        ctx.set_layer_weights(0, w)
        plain.set_layer_weights(0, w)
        q = bits(rng.standard_normal((T * 64, row)).astype(np.float32))
        steps, keys_of, pos = [], [], []
        for L, n in batch:
            rows = bits(rng.standard_normal((L + n, row)).astype(np.float32) * 1.3)
            s, p = ctx.seq_alloc(), plain.seq_alloc()
            ctx.cache_write(0, s, 0, rows)
            values = ctx.cache_read(0, s, 0, L + n)
            plain.cache_write(0, p, 0, values)
            assert s == p
            steps.append((s, L, n))
            for i in range(n):
                keys_of.append(f32(values[:L + i + 1 if causal else L + n]).astype(np.float64))
                pos.append(L + i)
        d_q = dev(torch, q)
        out = []
        for c in (ctx, plain):
            c.plan(steps, causal=causal)
            d_o = dev(torch, np.full((T * 64 + 64, 512), 0x7777, np.uint16))
            c.attention_device(0, d_q.data_ptr(), d_o.data_ptr())
            c.sync()
            o = host(d_o)
            assert (o[T * 64:] == 0x7777).all()
            out.append(o[:T * 64])
            assert np.array_equal(c.attention_only(0, q), out[-1])  # the host-buffer form
        # the same values in the same order of operations (the two formats cut and order their work alike): same bits
        assert np.array_equal(out[0], out[1])
        scale = mla.default_scale(ctx.cfg)
        check_attention(out[0].reshape(T, 64, 512), f32(q).astype(np.float64).reshape(T, 64, row), keys_of, 512, scale, sinks, pos,
                        64, v4)


@pytest.mark.parametrize("factor", [2.0 ** -40, 2.0 ** 20, 0.0, math.nan])
@pytest.mark.parametrize("preset", [mla.PRESET_BASELINE, mla.PRESET_FASTAR_V4])
def test_scales_of_every_size(torch, preset, factor):
    """Groups whose scale is no fp16 number, groups of zeros and of NaN among ordinary ones: what a bf16 cache of the
    same values gives, bit for bit."""
    rng = np.random.default_rng(13)
    with make(preset, n_pages=40) as ctx, make(preset, e4m3=False, n_pages=40) as plain:
        row = ctx.dims["row"]
        w = {n: np.zeros(sh, np.uint16) for n, sh in mla.weight_shapes(ctx.cfg).items()}
        w["attn_sinks"] = np.zeros(64, np.float32)
        x = rng.standard_normal((400, row)).astype(np.float32) * np.float32(2.0 ** -12)
        x[130, 64:128] *= np.float32(factor)   # one group of one row of the third page
        x[300:320, :448] *= np.float32(factor)
        q = bits(rng.standard_normal((2 * 64, row)).astype(np.float32))
        outs = []
        for c in (ctx, plain):
            c.set_layer_weights(0, w)
            s, t = c.seq_alloc(), c.seq_alloc()
            c.cache_write(0, s, 0, bits(x) if c is ctx else values)
            c.cache_write(0, t, 0, bits(x[:130]))
            values = c.cache_read(0, s, 0, 400)
            if c is plain:
                c.cache_write(0, t, 0, ctx.cache_read(0, t, 0, 130))
            c.plan([(s, 400, 1, -1, 0), (t, 130, 1, -1, 0)])
            o = dev(torch, np.zeros((2 * 64, 512), np.uint16))
            c.attention_device(0, dev(torch, q).data_ptr(), o.data_ptr())
            c.sync()
            outs.append(f32(host(o)))
        assert np.array_equal(outs[0], outs[1], equal_nan=True)
        assert np.isfinite(outs[0][64:]).all() and np.isnan(outs[0][:64]).any() == math.isnan(factor)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -3.3e38])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("preset", [mla.PRESET_BASELINE, mla.PRESET_FASTAR_V4])
@pytest.mark.parametrize("n_seq,rows,new,window", [(1, 293, 7, 0), (2, 60, 5, 0), (3, 300, 1, 64), (4, 2000, 16, 0), (4, 2000, 16, 100)])
def test_what_masked_rows_hold(torch, preset, e4m3, bad, n_seq, rows, new, window):
    """Rows that a token does not see hold NaN, infinities or huge values, in the latent or the rope dims: the bits of its
    output are those with ordinary rows in their place.  (Rows of later tokens; rows in front of the window.)"""
    rng = np.random.default_rng(17)
    n = rows + new
    with make(preset, e4m3=e4m3, n_pages=40 * n_seq) as ctx:
        row = ctx.dims["row"]
        w = {k: np.zeros(sh, np.uint16) for k, sh in mla.weight_shapes(ctx.cfg).items()}
        w["attn_sinks"] = np.zeros(64, np.float32)
        ctx.set_layer_weights(0, w)
        x = rng.standard_normal((n_seq, n, row)).astype(np.float32)
        q = dev(torch, bits(rng.standard_normal((n_seq * new * 64, row)).astype(np.float32)))
        o = dev(torch, np.zeros((n_seq * new * 64, 512), np.uint16))
        seqs = [ctx.seq_alloc() for _ in range(n_seq)]
        first = new // 2  # tokens from here on see bad rows of later tokens
        outs = []
        for spoiled in (False, True):
            y = x.copy()
            if spoiled:
                for b in range(n_seq):
                    if new > 1:
                        y[b, rows + first, 5 + b] = bad
                        y[b, n - 1, 400] = -bad
                        y[b, n - 2, row - 3] = bad
                    if window:
                        y[b, rows - window - 8, 77] = bad
                        y[b, rows - window - 20] = bad
                        y[b, rows - window - 30, row - 1] = bad
            for s, r in zip(seqs, y):
                ctx.cache_write(0, s, 0, bits(r))
            ctx.plan([(s, rows, new, -1, 1, window) for s in seqs], causal=True)
            ctx.attention_device(0, q.data_ptr(), o.data_ptr())
            ctx.sync()
            outs.append(host(o).reshape(n_seq, new, 64, 512))
        sees_none = first if new > 1 else 1
        assert np.isfinite(f32(outs[0])).all()
        assert np.array_equal(outs[0][:, :sees_none], outs[1][:, :sees_none])
        if new > 1 and not math.isfinite(bad) and not (e4m3 and math.isinf(bad)):
            assert np.isnan(f32(outs[1][:, first:])).any((2, 3)).all()  # who sees the row has it


def test_attention_without_rows(torch):
    """Tokens that see nothing get zeros, also beside tokens that see something."""
    with make() as ctx:
        a, b = ctx.seq_alloc(), ctx.seq_alloc()
        ctx.cache_write(0, b, 0, bits(np.ones((3, 576), np.float32)))
        q = dev(torch, bits(np.ones((2 * 64, 576), np.float32)))
        o = dev(torch, np.full((2 * 64, 512), 0x7777, np.uint16))
        ctx.plan([(a, 0, 1, -1, 0), (b, 3, 1, -1, 0)])
        ctx.attention_device(0, q.data_ptr(), o.data_ptr())
        ctx.sync()
        got = f32(host(o))
        assert not got[:64].any() and np.allclose(got[64:], 1.0, rtol=2.0 ** -7)


def test_window(torch):
    rng = np.random.default_rng(8)
    with make(n_pages=40) as ctx:
        s = ctx.seq_alloc()
        ctx.cache_write(0, s, 0, bits(rng.standard_normal((1000, 576)).astype(np.float32)))
        values = f32(ctx.cache_read(0, s, 0, 1000)).astype(np.float64)
        q = bits(rng.standard_normal((64, 576)).astype(np.float32))
        d_q, d_o = dev(torch, q), dev(torch, np.zeros((64, 512), np.uint16))
        for w in (1, 63, 200):
            ctx.plan([(s, 1000, 1, -1, 0, w)])
            ctx.attention_device(0, d_q.data_ptr(), d_o.data_ptr())
            ctx.sync()
            check_attention(host(d_o).reshape(1, 64, 512), f32(q).astype(np.float64)[None], [values[1000 - w:]], 512,
                            mla.default_scale(ctx.cfg), None, [0], 64, False)


def test_window_over_a_prompt(torch):
    """Many rows with a sliding window: pages are expanded, from the first one that some token sees."""
    rng = np.random.default_rng(14)
    with make(n_pages=20, max_tokens=400) as ctx:
        s, t = ctx.seq_alloc(), ctx.seq_alloc()
        values = []
        for q, n in ((s, 400), (t, 150)):
            ctx.cache_write(0, q, 0, bits(rng.standard_normal((n, 576)).astype(np.float32)))
            values.append(f32(ctx.cache_read(0, q, 0, n)).astype(np.float64))
        steps = [(s, 150, 250, -1, 1, 70), (t, 0, 150, -1, 1, 33)]
        q = bits(rng.standard_normal((400 * 64, 576)).astype(np.float32))
        d_q, d_o = dev(torch, q), dev(torch, np.zeros((400 * 64, 512), np.uint16))
        ctx.plan(steps, causal=True)
        ctx.attention_device(0, d_q.data_ptr(), d_o.data_ptr())
        ctx.sync()
        keys = [v[max(0, p + i + 1 - w):p + i + 1] for v, (_, p, n, _, _, w) in zip(values, steps) for i in range(n)]
        check_attention(host(d_o).reshape(400, 64, 512), f32(q).astype(np.float64).reshape(400, 64, 576), keys, 512,
                        mla.default_scale(ctx.cfg), None, [0] * 400, 64, False)


@pytest.mark.parametrize("preset", [mla.PRESET_BASELINE, mla.PRESET_FASTAR_V4])
def test_layer_calls(torch, preset):
    """Layer calls over an E4M3 cache: the rows they append are the quantised STAGE_KV rows, and a bf16 context
    that holds those rows gives the same attention for the next call's queries."""
    rng = np.random.default_rng(9)
    kw = dict(hidden=256, q_lora=128, o_lora=128, n_pages=40, max_tokens=80)
    with make(preset, **kw) as ctx, make(preset, e4m3=False, **kw) as plain:
        w = synth.weights_to_bits(synth.layer_weights_f32(ctx.cfg, 0, 0))
        for c in (ctx, plain):
            c.set_layer_weights(0, w)
        n8 = n8_of(ctx)
        seqs = [ctx.seq_alloc(), ctx.seq_alloc()]
        assert [plain.seq_alloc(), plain.seq_alloc()] == seqs
        pos = [0, 0]
        for q_lens, causal in (((50, 20), True), ((1, 1), False), ((5, 5), True), ((1, 1), False)):
            h = bits(rng.standard_normal((sum(q_lens), 256)).astype(np.float32))
            ctx.forward(0, h, seqs, pos, list(q_lens), causal=causal)
            kv = ctx.get_stage(mla.STAGE_KV)
            q_eff, o_lat = ctx.get_stage(mla.STAGE_QEFF), ctx.get_stage(mla.STAGE_OLAT)
            at = 0
            for s, p, n in zip(seqs, pos, q_lens):
                values = ctx.cache_read(0, s, p, n)
                same_values(values, held(f32(kv[at:at + n]), n8))
                plain.cache_write(0, s, p, values)
                at += n
            plain.plan([(s, p, n) for s, p, n in zip(seqs, pos, q_lens)], causal=causal)
            assert np.array_equal(plain.attention_only(0, q_eff), o_lat)
            pos = [p + n for p, n in zip(pos, q_lens)]
        # append_rows: the KV side alone
        h = bits(rng.standard_normal((2, 256)).astype(np.float32))
        ctx.append_rows(0, h, [seqs[0]], [pos[0]], [2])
        assert ctx.seq_len(seqs[0]) == pos[0] + 2


def test_compressed_layers(torch):
    """A ratio-4 and a ratio-128 layer over an E4M3 cache: the compressed rows are those of a bf16 context bit for bit (they are
    E4M3 values already), and the attention over raw and compressed rows is what the bf16 context gives when it
    holds the quantised raw rows."""
    rng = np.random.default_rng(15)
    kw = dict(hidden=256, q_lora=128, o_lora=128, n_layers=2, n_pages=60, max_seqs=2, max_tokens=160)
    with make(mla.PRESET_FASTAR_V4, e4m3=False, **kw) as ctx, make(mla.PRESET_FASTAR_V4, e4m3=False, **kw) as plain:
        for c in (ctx, plain):
            wr = np.random.default_rng(16)
            for lid, ratio in enumerate((4, 128)):
                c.set_layer_weights(lid, synth.weights_to_bits(synth.layer_weights_f32(c.cfg, lid, 0)))
                c.set_layer_rope(lid, True)
                width = 1024 if ratio == 4 else 512
                m = [bits(wr.standard_normal((width, 256)).astype(np.float32) * 0.1) for _ in range(2)]
                c.set_layer_compressor(lid, ratio, *m, wr.standard_normal((ratio, width)).astype(np.float32),
                                       bits((1 + 0.1 * wr.standard_normal(512)).astype(np.float32)))
        ctx.set_cache_format(mla.CACHE_E4M3)
        seqs = [ctx.seq_alloc(), ctx.seq_alloc()]
        assert [plain.seq_alloc(), plain.seq_alloc()] == seqs
        pos = [0, 0]
        for q_lens, causal in (((150, 10), True), ((130, 20), True), ((1, 1), False), ((6, 6), True)):
            h = bits(rng.standard_normal((sum(q_lens), 256)).astype(np.float32))
            for lid in range(2):
                ctx.forward(lid, h, seqs, pos, list(q_lens), causal=causal)
                q_eff, o_lat = ctx.get_stage(mla.STAGE_QEFF), ctx.get_stage(mla.STAGE_OLAT)
                plain.forward(lid, h, seqs, pos, list(q_lens), causal=causal)
                for s, p, n in zip(seqs, pos, q_lens):
                    a, b = ctx.cmp_read(lid, s), plain.cmp_read(lid, s)
                    assert a.shape == ((p + n) // (4, 128)[lid], 512) and np.array_equal(a, b)
                    plain.cache_write(lid, s, p, ctx.cache_read(lid, s, p, n))
                plain.plan([(s, p, n) for s, p, n in zip(seqs, pos, q_lens)], causal=causal)
                assert np.array_equal(plain.attention_only(lid, q_eff), o_lat)
            pos = [p + n for p, n in zip(pos, q_lens)]
        ctx.seq_truncate(seqs[0], 0)
        ctx.forward(0, h[:6], [seqs[0]], [0], [6], causal=True)
        assert ctx.cmp_read(0, seqs[0]).shape == (1, 512)


def test_split_over_two_slices(torch):
    """Partials of two contexts, each with a slice of the rows, merged: what one context with all rows gives."""
    rng = np.random.default_rng(10)
    kw = dict(hidden=256, q_lora=128, n_pages=40, max_tokens=4)
    with make(**kw) as one, make(**kw) as a, make(**kw) as b:
        w = synth.weights_to_bits(synth.layer_weights_f32(one.cfg, 0, 0))
        rows = bits(rng.standard_normal((500, 576)).astype(np.float32))
        h = dev(torch, bits(rng.standard_normal((1, 256)).astype(np.float32)))
        for c in (one, a, b):
            c.set_layer_weights(0, w)
            c.seq_alloc()
        one.cache_write(0, 0, 0, rows)
        a.cache_write(0, 0, 0, rows[:256])
        b.cache_write(0, 0, 0, rows[256:])
        one.plan([(0, 500, 1)])
        a.plan([(0, 256, 1, 500, 0)])
        b.plan([(0, 244, 1, 500, 1)])
        out1, out2 = torch.zeros(1, 256, dtype=torch.int16, device="cuda"), torch.zeros(1, 256, dtype=torch.int16, device="cuda")
        one.run_device(0, h.data_ptr(), out1.data_ptr())
        parts = torch.zeros(2, 64, 514, device="cuda")
        a.run_partial_device(0, h.data_ptr(), parts[0].data_ptr())
        b.run_partial_device(0, h.data_ptr(), parts[1].data_ptr())
        b.sync()
        a.run_merge_device(0, parts.data_ptr(), 2, out2.data_ptr())
        for c in (one, a, b):
            c.sync()
        x, y = f32(host(out1)), f32(host(out2))
        # both round weights, latent outputs and the projections' results to bf16: a few steps of the largest value apart
        assert np.abs(x - y).max() <= 8 * 2.0 ** -8 * np.abs(x).max()


def test_other_stream_and_graph(torch):
    """On a stream of the caller's; captured into a graph and replayed with new queries and rows in the same buffers."""
    rng = np.random.default_rng(11)
    with make(n_pages=40) as ctx:
        st = torch.cuda.Stream()
        ctx.set_stream(st.cuda_stream)
        s = ctx.seq_alloc()
        ctx.cache_write(0, s, 0, bits(rng.standard_normal((700, 576)).astype(np.float32)))
        ctx.plan([(s, 700, 1)])
        q, rows = dev(torch, np.zeros((64, 576), np.uint16)), dev(torch, np.zeros((1, 576), np.uint16))
        o, back = dev(torch, np.zeros((64, 512), np.uint16)), dev(torch, np.zeros((3, 576), np.uint16))

        def step():
            ctx.cache_append_device(0, rows.data_ptr())
            ctx.attention_device(0, q.data_ptr(), o.data_ptr())
            ctx.cache_read_device(0, [(s, 698, 3)], back.data_ptr())
        torch.cuda.synchronize()
        step()  # attributes are set outside the capture
        ctx.sync()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            step()
        for _ in range(3):
            qn = bits(rng.standard_normal((64, 576)).astype(np.float32))
            rn = bits(rng.standard_normal((1, 576)).astype(np.float32))
            with torch.cuda.stream(st):
                q.copy_(dev(torch, qn))
                rows.copy_(dev(torch, rn))
                st.synchronize()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            values = ctx.cache_read(0, s, 0, 701)
            same_values(values[700:], held(f32(rn), 512))
            assert np.array_equal(host(back), values[698:])
            check_attention(host(o).reshape(1, 64, 512), f32(qn).astype(np.float64)[None], [f32(values).astype(np.float64)], 512,
                            mla.default_scale(ctx.cfg), None, [700], 64, False)


def test_repeats_are_bit_equal(torch):
    rng = np.random.default_rng(12)
    with make(n_pages=400, max_seqs=8) as ctx:
        steps = []
        for n in (4000, 1, 777, 6400):
            s = ctx.seq_alloc()
            ctx.cache_write(0, s, 0, bits(rng.standard_normal((n, 576)).astype(np.float32)))
            steps.append((s, n, 1, -1, 0))
        q = dev(torch, bits(rng.standard_normal((4 * 64, 576)).astype(np.float32)))
        ctx.plan(steps)
        outs = []
        for _ in range(20):
            o = torch.zeros(4 * 64, 512, dtype=torch.int16, device="cuda")
            ctx.attention_device(0, q.data_ptr(), o.data_ptr())
            ctx.sync()
            outs.append(host(o))
        assert all(np.array_equal(o, outs[0]) for o in outs)


def refused(code, fn, *a):
    with pytest.raises(mla.MlaError) as e:
        fn(*a)
    assert e.value.code == code, str(e.value)


def test_refusals(torch):
    buf = torch.zeros(64 * 576 + 8, dtype=torch.int16, device="cuda")
    p = buf.data_ptr()
    with make(e4m3=False) as ctx:
        refused(mla.ERR_ARG, ctx.set_cache_format, 2)
        refused(mla.ERR_STATE, ctx.cache_append_device, 0, p)      # no plan
        refused(mla.ERR_STATE, ctx.attention_device, 0, p, p)
        s = ctx.seq_alloc()
        ctx.seq_reserve(s, 5)
        refused(mla.ERR_STATE, ctx.set_cache_format, mla.CACHE_E4M3)  # rows are held
        ctx.set_cache_format(mla.CACHE_BF16)                        # (what it is already)
        ctx.seq_truncate(s, 0)
        ctx.set_cache_format(mla.CACHE_E4M3)
        assert ctx.seq_alloc() != s  # sequences stay
        ctx.plan([(s, 0, 1)])
        for bad in (0, p + 2):
            refused(mla.ERR_ARG, ctx.cache_append_device, 0, bad)
            refused(mla.ERR_ARG, ctx.attention_device, 0, bad, p)
            refused(mla.ERR_ARG, ctx.attention_device, 0, p, bad)
            refused(mla.ERR_ARG, ctx.cache_read_device, 0, [(s, 0, 1)], bad)
        refused(mla.ERR_ARG, ctx.cache_append_device, 1, p)
        refused(mla.ERR_ARG, ctx.attention_device, -1, p, p)
        refused(mla.ERR_ARG, ctx.cache_read_device, 1, [(s, 0, 1)], p)
        for r in ((s, 0, 2), (s, 1, 1), (s, -1, 1), (s, 0, -1), (7, 0, 0), (-1, 0, 0), (s, 2 ** 31 - 1, 2 ** 31 - 1)):
            refused(mla.ERR_ARG, ctx.cache_read_device, 0, [r], p)
        ctx.cache_read_device(0, [], 0)
        ctx.cache_read_device(0, [(s, 1, 0)], 0)
        refused(mla.ERR_STATE, ctx.row_offset, s, 0)
        ctx.sync()
    with make(mla.PRESET_FASTAR_V4) as ctx:
        s = ctx.seq_alloc()
        ctx.plan([(s, 0, 1)])
        refused(mla.ERR_STATE, ctx.attention_device, 0, p, p)  # no weights: no sink logits
    with make(mla.PRESET_FASTAR_V4, e4m3=False, kv_lora=64, qk_rope=12, n_heads=8) as ctx:  # 52 latent values
        refused(mla.ERR_ARG, ctx.set_cache_format, mla.CACHE_E4M3)
