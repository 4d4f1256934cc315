"""Forked sequences: pages shared and copied on write, and attention of batches over a shared prefix."""
import numpy as np
import pytest

from fastar_b200 import mla, synth
from tests.test_gpu_cache_format import (bits, check_attention, dev, f32, host, make, refused)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


def rows_of(rng, n, row=576):
    return bits(rng.standard_normal((n, row)).astype(np.float32))


FORMATS = [False, True]


@pytest.mark.parametrize("e4m3", FORMATS)
def test_forks_are_sequences_of_their_own(torch, e4m3):
    rng = np.random.default_rng(0)
    with make(e4m3=e4m3, n_layers=2, n_pages=40, max_seqs=6) as ctx:
        a = ctx.seq_alloc()
        base = rows_of(rng, 200)
        for lid in range(2):
            ctx.cache_write(lid, a, 0, base[::1 if lid else -1])
        held = [ctx.cache_read(lid, a, 0, 200) for lid in range(2)]
        free = ctx.free_pages()
        b = ctx.seq_fork(a, 150)      # two whole pages shared, 22 rows copied
        c = ctx.seq_fork(a, 128)      # whole pages only
        d = ctx.seq_fork(b, 0)
        assert ctx.free_pages() == free - 1
        assert [ctx.seq_len(s) for s in (a, b, c, d)] == [200, 150, 128, 0]
        assert list(ctx.block_table(b)[:2]) == list(ctx.block_table(a)[:2]) == list(ctx.block_table(c))
        assert ctx.block_table(b)[2] != ctx.block_table(a)[2]
        for lid in range(2):
            assert np.array_equal(ctx.cache_read(lid, b, 0, 150), held[lid][:150])
        # behind the copied rows there is nothing
        ctx.seq_reserve(b, 192)
        assert not ctx.cache_read(0, b, 150, 42).any()
        ctx.seq_truncate(b, 150)
        # appends of one are not seen by the other
        more = rows_of(rng, 30)
        ctx.cache_write(0, b, 150, more)
        ctx.cache_write(0, c, 128, more[:5])
        assert np.array_equal(ctx.cache_read(0, a, 0, 200), held[0])
        # a write into a shared page: a copy of that page alone
        free = ctx.free_pages()
        ctx.cache_write(1, c, 70, more[:1])
        assert ctx.free_pages() == free - 1
        assert ctx.block_table(c)[1] != ctx.block_table(a)[1] and ctx.block_table(c)[0] == ctx.block_table(a)[0]
        got = ctx.cache_read(1, c, 0, 128)
        assert np.array_equal(np.delete(got, 70, 0), np.delete(held[1][:128], 70, 0)) and not np.array_equal(got[70], held[1][70])
        assert np.array_equal(ctx.cache_read(0, c, 0, 128), held[0][:128])
        for s in (a, b):
            assert np.array_equal(ctx.cache_read(1, s, 0, 128), held[1][:128])
        # a plan that appends over shared rows (a step taken back and done again)
        ctx.plan([(b, 127, 2)])
        assert ctx.block_table(b)[1] != ctx.block_table(a)[1]
        assert np.array_equal(ctx.cache_read(0, b, 64, 64), held[0][64:128])
        # truncation into a shared page: the others keep their rows
        e = ctx.seq_fork(a, 192)
        ctx.seq_truncate(e, 100)
        assert np.array_equal(ctx.cache_read(0, e, 0, 100), held[0][:100])
        ctx.seq_reserve(e, 128)
        assert not ctx.cache_read(0, e, 100, 28).any()
        assert np.array_equal(ctx.cache_read(0, a, 0, 200), held[0])
        # pages go back with their last holder, zeroed
        ctx.seq_free(a)
        assert np.array_equal(ctx.cache_read(0, e, 0, 64), held[0][:64])
        for s in (b, c, d, e):
            ctx.seq_free(s)
        assert ctx.free_pages() == 40
        assert not ctx.pool_read(0).any() and not ctx.pool_read(1).any()


def test_page_accounting_against_a_count(torch):
    """Random forks, appends, truncations and frees: pages in use are the distinct pages of the tables, lengths and
    rows are what a plain copy of every sequence says."""
    rng = np.random.default_rng(1)
    with make(e4m3=False, kv_lora=64, qk_rope=16, n_heads=2, page_tokens=8, n_pages=60, max_seqs=9) as ctx:
        row, live, tag = ctx.dims["row"], {}, 0
        for it in range(400):
            op = rng.integers(0, 6)
            try:
                if op == 0 and len(live) < 9:
                    live[ctx.seq_alloc()] = np.zeros((0, row), np.uint16)
                elif op == 1 and live and len(live) < 9:
                    s = int(rng.choice(list(live)))
                    n = int(rng.integers(0, len(live[s]) + 1))
                    live[ctx.seq_fork(s, n)] = live[s][:n].copy()
                elif op in (2, 3) and live:
                    s = int(rng.choice(list(live)))
                    pos, n = int(rng.integers(max(0, len(live[s]) - 20), len(live[s]) + 1)), int(rng.integers(1, 30))
                    tag += 1
                    r = np.full((n, row), tag % 30000, np.uint16)
                    old = live[s]
                    try:
                        ctx.cache_write(0, s, pos, r)
                    except mla.MlaError:
                        # (the length may have grown by then: rows without a value)
                        grown = np.zeros((ctx.seq_len(s), row), np.uint16)
                        grown[:len(old)] = old
                        live[s] = grown
                        raise
                    new = np.zeros((max(len(old), pos + n), row), np.uint16)
                    new[:len(old)] = old
                    new[pos:pos + n] = r
                    live[s] = new
                elif op == 4 and live:
                    s = int(rng.choice(list(live)))
                    n = int(rng.integers(0, len(live[s]) + 1))
                    ctx.seq_truncate(s, n)
                    live[s] = live[s][:n]
                elif op == 5 and live:
                    s = int(rng.choice(list(live)))
                    ctx.seq_free(s)
                    del live[s]
            except mla.MlaError as e:
                assert e.code == mla.ERR_PAGES, str(e)
            used = set()
            for s, r in live.items():
                assert ctx.seq_len(s) == len(r)
                t = [int(x) for x in ctx.block_table(s)]
                assert len(t) == (len(r) + 7) // 8
                used |= set(t)
                if len(r):
                    assert np.array_equal(ctx.cache_read(0, s, 0, len(r)), r)
            assert ctx.free_pages() == 60 - len(used)


def run_batch(torch, ctx, steps, q, T, causal):
    ctx.plan(steps, causal=causal)
    o = dev(torch, np.full((T * 64 + 64, 512), 0x7777, np.uint16))
    ctx.attention_device(0, dev(torch, q).data_ptr(), o.data_ptr())
    ctx.sync()
    got = host(o)
    assert (got[T * 64:] == 0x7777).all()
    return got[:T * 64].reshape(T, 64, 512)


BATCHES = [
    # prefix, (rows of their own, new tokens) per fork, sequences beside them, causal
    (64, [(0, 1), (1, 1)], [], False),
    (1000, [(0, 1), (3, 1), (70, 1), (64, 1), (200, 1)], [], False),
    (1000, [(5, 1)] * 30, [300, 1], False),
    (640, [(10, 5), (0, 5), (100, 5)], [], True),
    (640, [(10, 1), (0, 7), (100, 3)], [50], True),
    (130, [(9, 1)] * 70, [], False),
]


@pytest.mark.parametrize("e4m3", FORMATS)
@pytest.mark.parametrize("preset", [mla.PRESET_BASELINE, mla.PRESET_FASTAR_V4])
@pytest.mark.parametrize("prefix,forks,others,causal", BATCHES)
def test_attention_over_a_shared_prefix(torch, prefix, forks, others, causal, preset, e4m3):
    rng = np.random.default_rng(2)
    v4 = preset == mla.PRESET_FASTAR_V4
    with make(preset, e4m3=e4m3, n_pages=300, max_seqs=80, max_tokens=128) as ctx:
        row = ctx.dims["row"]
        sinks = rng.standard_normal(64).astype(np.float32) if v4 else None
        w = {n: np.zeros(sh, np.uint16) for n, sh in mla.weight_shapes(ctx.cfg).items()}
        w["attn_sinks"] = sinks
        ctx.set_layer_weights(0, w)
        base = ctx.seq_alloc()
        ctx.cache_write(0, base, 0, rows_of(rng, prefix + 10, row))
        steps, keys_of, pos = [], [], []
        seqs = [ctx.seq_fork(base, prefix) for _ in forks]
        todo = [(s, prefix, c, n) for s, (c, n) in zip(seqs, forks)]
        for n in others:
            todo.insert(1, (ctx.seq_alloc(), 0, n, 1))
        for s, p, c, n in todo:
            ctx.cache_write(0, s, p, rows_of(rng, c + n, row))
            values = f32(ctx.cache_read(0, s, 0, p + c + n)).astype(np.float64)
            steps.append((s, p + c, n))
            for i in range(n):
                keys_of.append(values[:p + c + (i + 1 if causal else n)])
                pos.append(p + c + i)
        T = len(pos)
        q = bits(rng.standard_normal((T * 64, row)).astype(np.float32))
        for on in (True, False):
            ctx.set_shared_prefix(on)
            got = run_batch(torch, ctx, steps, q, T, causal)
            check_attention(got, f32(q).astype(np.float64).reshape(T, 64, row), keys_of, 512, mla.default_scale(ctx.cfg), sinks,
                            pos, 64, v4)


@pytest.mark.parametrize("e4m3,n_tok", [(False, 3), (False, 9), (True, 9), (True, 12)])
def test_prefix_that_l2_does_not_hold(torch, e4m3, n_tok):
    """The epochs: a prefix of over 64 MiB, two forks of a second prefix, a sequence by itself and one that sees nothing."""
    rng = np.random.default_rng(3)
    prefix = 120000 if e4m3 else 62000
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    with make(e4m3=e4m3, n_pages=prefix // 64 + 100, max_seqs=n_tok + 8, max_tokens=512) as ctx:
        assert prefix // 64 * ctx.cache_page_bytes() > 64 << 20
        base = ctx.seq_alloc()
        x = torch.randn(prefix, 576, generator=g, device="cuda").to(torch.bfloat16)
        for i in range(0, prefix, 512):
            ctx.plan([(base, i, min(512, prefix - i))])
            ctx.cache_append_device(0, x[i:i + 512].data_ptr())
        forks = [ctx.seq_fork(base, prefix) for _ in range(n_tok)]
        second = ctx.seq_alloc()
        ctx.cache_write(0, second, 0, rows_of(rng, 320))
        seqs = forks + [ctx.seq_fork(second, 320), ctx.seq_fork(second, 300), ctx.seq_alloc(), ctx.seq_alloc()]
        steps = []
        for i, s in enumerate(seqs[:-1]):
            n = ctx.seq_len(s)
            ctx.cache_write(0, s, n, rows_of(rng, 1 + 37 * (i % 3)))
            steps.append((s, ctx.seq_len(s), 1, -1, 0))
        steps.append((seqs[-1], 0, 1, -1, 0))
        T = len(steps)
        q = bits(rng.standard_normal((T * 64, 576)).astype(np.float32))
        shared = run_batch(torch, ctx, steps, q, T, False)
        again = run_batch(torch, ctx, steps, q, T, False)
        assert np.array_equal(shared, again)
        info = ctx.plan_info()
        ctx.set_shared_prefix(False)
        alone = run_batch(torch, ctx, steps, q, T, False)
        assert info["kv_rows"] == ctx.plan_info()["kv_rows"]
        # (three users are not worth epochs, which leave more partials)
        assert (info["n_partials"] > ctx.plan_info()["n_partials"]) == (n_tok >= 8)
        assert not shared[-1].any()
        qd = torch.from_numpy(q.view(np.int16)).cuda().view(torch.bfloat16).double().reshape(T, 64, 576)
        for t, (s, n, *_) in enumerate(steps[:-1]):
            buf = torch.zeros(n, 576, dtype=torch.bfloat16, device="cuda")
            ctx.cache_read_device(0, [(s, 0, n)], buf.data_ptr())
            ctx.sync()
            keys = buf.double()
            p = torch.softmax(qd[t] @ keys.T * 192.0 ** -0.5, 1)
            o, a = p @ keys[:, :512], p @ keys[:, :512].abs()
            # as in check_attention: the weights' rounding to bf16, and the output's
            tol = 2.0 ** -8 * a + 2.0 ** -8 * o.abs()
            for got in (shared[t], alone[t]):
                err = (torch.from_numpy(f32(got).astype(np.float64)).cuda() - o).abs()
                assert bool((err <= tol).all()), (t, float((err / tol).max()))


@pytest.mark.parametrize("e4m3", FORMATS)
def test_a_run_of_them_together(torch, e4m3):
    """A server's life: a prompt goes through two layers, is forked for three users, who decode, verify a block, take it
    back, and leave; every layer output equals that of users who hold the prompt each for themselves."""
    rng = np.random.default_rng(5)
    kw = dict(e4m3=e4m3, hidden=256, q_lora=128, n_layers=2, n_pages=80, max_seqs=5, max_tokens=160)
    with make(**kw) as ctx, make(**kw) as ref:
        for lid in range(2):
            w = synth.weights_to_bits(synth.layer_weights_f32(ctx.cfg, lid, 0))
            ctx.set_layer_weights(lid, w)
            ref.set_layer_weights(lid, w)
        ctx.set_shared_prefix(True)
        prompt = rows_of(rng, 150, 256)
        base = ctx.seq_alloc()
        for lid in range(2):
            ctx.forward(lid, prompt, [base], [0], [150], causal=True)
        users = [ctx.seq_fork(base, 150) for _ in range(3)]
        ctx.seq_free(base)
        own = [ref.seq_alloc() for _ in range(3)]
        for u in own:
            for lid in range(2):
                ref.forward(lid, prompt, [u], [0], [150], causal=True)

        def both(h, pos, q, causal):
            for lid in range(2):
                x, y = ctx.forward(lid, h, users, pos, q, causal=causal), ref.forward(lid, h, own, pos, q, causal=causal)
                a, b = f32(x), f32(y)
                # the same rows; parts may be added in another order (a step of the weights' and of every later rounding)
                assert np.abs(a - b).max() <= 8 * 2.0 ** -8 * np.abs(b).max()
                for u, v, p, n in zip(users, own, pos, q):
                    assert np.array_equal(ctx.cache_read(lid, u, 0, p + n), ref.cache_read(lid, v, 0, p + n))
        pos = [150] * 3
        for _ in range(2):
            both(rows_of(rng, 3, 256), pos, [1] * 3, False)
            pos = [p + 1 for p in pos]
        both(rows_of(rng, 15, 256), pos, [5] * 3, True)
        for c, seqs in ((ctx, users), (ref, own)):
            for s, keep in zip(seqs, (152, 140, 154)):  # the second user goes back into the prompt
                c.seq_truncate(s, keep)
        pos = [152, 140, 154]
        both(rows_of(rng, 12, 256), pos, [4, 1, 7], True)
        for u in users:
            ctx.seq_free(u)
        assert ctx.free_pages() == 80


def test_more_table_entries_than_pages(torch):
    """64 forks name 60 shared pages each: more than the pool has.  A graph captured before gives the same until then."""
    rng = np.random.default_rng(6)
    with make(e4m3=False, n_pages=100, max_seqs=70, max_tokens=64) as ctx:
        st = torch.cuda.Stream()
        ctx.set_stream(st.cuda_stream)
        a = ctx.seq_alloc()
        ctx.cache_write(0, a, 0, rows_of(rng, 64 * 60))
        q = dev(torch, rows_of(rng, 64))
        o = dev(torch, np.zeros((64, 512), np.uint16))
        steps = [(a, 64 * 60, 1, -1, 0)]
        ctx.plan(steps)
        ctx.attention_device(0, q.data_ptr(), o.data_ptr())
        ctx.sync()
        want = host(o)
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=st):
            ctx.attention_device(0, q.data_ptr(), o.data_ptr())
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(host(o), want)
        forks = [ctx.seq_fork(a, 64 * 60) for _ in range(64)]  # 65 tables of 60 pages: more than the pool has
        q2 = dev(torch, rows_of(rng, 64 * 64))
        o2 = dev(torch, np.zeros((64 * 64, 512), np.uint16))
        ctx.plan([(s, 64 * 60, 1, -1, 0) for s in forks])
        ctx.attention_device(0, q2.data_ptr(), o2.data_ptr())
        ctx.sync()
        q2h = host(q2).reshape(64, 64, 576)
        k = f32(ctx.cache_read(0, a, 0, 64 * 60)).astype(np.float64)
        check_attention(host(o2).reshape(64, 64, 512), f32(q2h).astype(np.float64), [k] * 64, 512, mla.default_scale(ctx.cfg), None,
                        [0] * 64, 64, False)


def test_no_page_copies_in_a_capture(torch):
    """A fork, a write or a truncation that would copy a page is refused while the stream is captured, and works behind it."""
    rng = np.random.default_rng(7)
    with make(e4m3=False, n_pages=12, max_seqs=3) as ctx:
        st = torch.cuda.Stream()
        ctx.set_stream(st.cuda_stream)
        s = ctx.seq_alloc()
        rows = rows_of(rng, 150)
        ctx.cache_write(0, s, 0, rows)
        t = ctx.seq_fork(s, 128)
        free = ctx.free_pages()
        ctx.sync()
        buf = dev(torch, np.zeros((128, 576), np.uint16))
        ctx.cache_read_device(0, [(t, 0, 128)], buf.data_ptr())  # attributes are set outside the capture
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            refused(mla.ERR_STATE, ctx.seq_fork, s, 150)
            refused(mla.ERR_STATE, ctx.seq_truncate, t, 100)
            ctx.cache_read_device(0, [(t, 0, 128)], buf.data_ptr())
        assert ctx.free_pages() == free and ctx.seq_len(t) == 128
        buf.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(host(buf), rows[:128])
        u = ctx.seq_fork(s, 150)
        ctx.seq_truncate(t, 100)
        assert np.array_equal(ctx.cache_read(0, u, 0, 150), rows) and np.array_equal(ctx.cache_read(0, t, 0, 100), rows[:100])


def test_refusals(torch):
    with make(e4m3=False, n_pages=3, max_seqs=3) as ctx:
        s = ctx.seq_alloc()
        ctx.seq_reserve(s, 130)
        refused(mla.ERR_ARG, ctx.seq_fork, s, 131)
        refused(mla.ERR_ARG, ctx.seq_fork, s, -1)
        refused(mla.ERR_ARG, ctx.seq_fork, 2, 0)
        refused(mla.ERR_PAGES, ctx.seq_fork, s, 130)   # the last page needs a copy
        t = ctx.seq_fork(s, 128)                       # this does not
        refused(mla.ERR_PAGES, ctx.cache_write, 0, t, 5, np.zeros((1, 576), np.uint16))
        refused(mla.ERR_PAGES, ctx.plan, [(t, 5, 1)])
        refused(mla.ERR_PAGES, ctx.seq_truncate, t, 100)
        assert ctx.seq_len(t) == 128 and list(ctx.block_table(t)) == list(ctx.block_table(s)[:2])
        ctx.seq_truncate(t, 64)                        # whole pages: no copy
        ctx.seq_fork(s, 0)
        refused(mla.ERR_CAPACITY, ctx.seq_fork, s, 0)
    with make(mla.PRESET_FASTAR_V4, e4m3=False) as ctx:
        z = lambda *sh: np.zeros(sh, np.uint16)  # noqa: E731
        ctx.set_layer_compressor(0, 4, z(1024, 64), z(1024, 64), np.zeros((4, 1024), np.float32), z(512))
        refused(mla.ERR_STATE, ctx.seq_fork, ctx.seq_alloc(), 0)


@pytest.mark.parametrize("preset", [mla.PRESET_BASELINE, mla.PRESET_FASTAR_V4])
def test_engine_with_forks_and_a_quantised_cache(preset):
    """FSTEngine: one prompt in an E4M3 cache, two chats forked from it, a batched decode step over all three: the bits
    that the same steps give through the context."""
    import ctypes as C
    from tests.test_gpu_engine import load, weights_for
    rng = np.random.default_rng(7)
    L = load()
    p16, pi = C.POINTER(C.c_uint16), C.POINTER(C.c_int)
    L.fst_engine_fork_sequence.argtypes = [C.c_void_p, C.c_int, C.c_int]
    L.fst_engine_set_cache_format.argtypes = [C.c_void_p, C.c_int]
    L.fst_engine_process_mla_batch.argtypes = [C.c_void_p, C.c_int, p16, pi, pi, pi, C.c_int, C.c_int]
    L.fst_engine_current_sequence.argtypes = [C.c_void_p]
    e = L.fst_engine_create(preset, 1, 256, 3, 80, 0, mla.IMPL_AUTO, mla.IMPL_AUTO)
    assert e, L.fst_engine_last_error()
    w, _ = weights_for(preset)
    for name, a in w.items():
        if name == "attn_sinks":
            a = np.ascontiguousarray(a, np.float32)
            assert L.fst_engine_set_sinks(e, 0, a.ctypes.data_as(C.POINTER(C.c_float)), a.size) == 0
        else:
            a = np.ascontiguousarray(a, np.uint16)
            assert L.fst_engine_set_weight(e, 0, name.encode(), a.ctypes.data_as(p16), a.size) == 0
    assert L.fst_engine_preload(e) == 0, L.fst_engine_last_error()
    assert L.fst_engine_set_cache_format(e, mla.CACHE_E4M3) == 0, L.fst_engine_last_error()
    prompt, h = rows_of(rng, 75, 4096), rows_of(rng, 3, 4096)
    got = prompt.copy()
    assert L.fst_engine_process_mla(e, 0, got.ctypes.data_as(p16), 75) == 0, L.fst_engine_last_error()
    s0 = L.fst_engine_current_sequence(e)
    seqs = [s0, L.fst_engine_fork_sequence(e, s0, 75), L.fst_engine_fork_sequence(e, s0, 64)]
    assert L.fst_engine_fork_sequence(e, s0, 76) == -1
    arr = [np.array(x, np.int32) for x in (seqs, [75, 75, 64], [1, 1, 1])]
    step = h.copy()
    assert L.fst_engine_process_mla_batch(e, 0, step.ctypes.data_as(p16), *(a.ctypes.data_as(pi) for a in arr), 3, 0) == 0
    assert L.fst_engine_set_cache_format(e, mla.CACHE_BF16) == -1  # rows are held
    L.fst_engine_destroy(e)
    with mla.MlaContext(mla.make_config(preset, n_pages=64, max_seqs=3, max_tokens=80)) as ctx:
        ctx.set_cache_format(mla.CACHE_E4M3)
        ctx.set_layer_weights(0, w)
        a = ctx.seq_alloc()
        assert np.array_equal(ctx.forward(0, prompt, [a], [0], [75], causal=True), got)
        f = [a, ctx.seq_fork(a, 75), ctx.seq_fork(a, 64)]
        assert np.array_equal(ctx.forward(0, h, f, [75, 75, 64], [1, 1, 1]), step)


def check_on_device(torch, ctx, steps, q, got, causal, sinks=None):
    """check_attention in 64 bits on the device, for long contexts; the rows are read back from the cache."""
    row = ctx.dims["row"]
    v4 = ctx.cfg.preset == mla.PRESET_FASTAR_V4
    qd = torch.from_numpy(q.view(np.int16)).cuda().view(torch.bfloat16).double().reshape(-1, 64, row)
    gd = torch.from_numpy(f32(got).astype(np.float64)).cuda()
    scale = mla.default_scale(ctx.cfg)
    t = 0
    for s, pos0, n, *more in steps:
        own = not more or len(more) < 2 or more[1]
        total = pos0 + (n if own else 0)
        buf = torch.zeros(max(total, 1), row, dtype=torch.bfloat16, device="cuda")
        ctx.cache_read_device(0, [(s, 0, total)], buf.data_ptr())
        ctx.sync()
        keys = buf.double()
        for i in range(n):
            k = keys[:(pos0 + i + 1 if causal else total)]
            logits = qd[t] @ k.T * scale
            if sinks is not None:
                logits = torch.cat([logits, torch.from_numpy(sinks).cuda().double()[:, None]], 1)
            p = torch.softmax(logits, 1)[:, :k.shape[0]]
            o, a = p @ k[:, :512], p @ k[:, :512].abs()
            tol = 2.0 ** -8 * a + 2.0 ** -8 * o.abs()
            if v4:
                tol = 2.0 ** -8 * a + 2.0 ** -7 * o.abs()
                ang = (pos0 + i) * 10000.0 ** (-torch.arange(0, 64, 2, device="cuda", dtype=torch.float64) / 64)
                x0, x1 = o[:, 448::2].clone(), o[:, 449::2].clone()
                o[:, 448::2], o[:, 449::2] = x0 * ang.cos() + x1 * ang.sin(), x1 * ang.cos() - x0 * ang.sin()
                pair = tol[:, 448:].reshape(64, 32, 2).sum(2).repeat_interleave(2, 1)
                tol[:, 448:] = pair * (1 + 2.0 ** -12)
                tol += 2.0 ** -11 * o.abs().max()
            err = (gd[t] - o).abs()
            assert bool((err <= tol).all()), (t, float((err / tol).max()))
            t += 1


def fill(torch, ctx, seq, n, gen, row, pos=0):
    x = torch.randn(n, row, generator=gen, device="cuda").to(torch.bfloat16)
    for i in range(0, n, 512):
        ctx.plan([(seq, pos + i, min(512, n - i))])
        ctx.cache_append_device(0, x[i:i + 512].data_ptr())
    ctx.sync()


LONG = [
    # (prefix, users, rows of their own up to, new tokens, other sequences)
    (6400, 30, 1, 1, 0),        # the shared pages are all but a row of it
    (6400, 31, 200, 1, 2),      # an odd number of users, others beside them
    (6401, 24, 70, 1, 0),       # a prefix that ends inside a page
    (3000, 20, 90, 3, 1),       # blocks of new tokens on a shared prefix
    (20000, 8, 300, 1, 0),
    (700, 148, 400, 1, 0),      # a lane for every SM; own rows longer than the prefix for some
    (130, 74, 130, 1, 0),
    (5000, 2, 900, 1, 0),
]


@pytest.mark.parametrize("e4m3", FORMATS)
@pytest.mark.parametrize("preset", [mla.PRESET_BASELINE, mla.PRESET_FASTAR_V4])
@pytest.mark.parametrize("prefix,users,own,q_len,others", LONG)
def test_long_shared_prefix(torch, prefix, users, own, q_len, others, preset, e4m3):
    rng = np.random.default_rng(8)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(9)
    v4 = preset == mla.PRESET_FASTAR_V4
    with make(preset, e4m3=e4m3, n_pages=prefix // 64 + (users + others + 2) * 8, max_seqs=users + others + 1, max_tokens=512) as ctx:
        row = ctx.dims["row"]
        sinks = rng.standard_normal(64).astype(np.float32) if v4 else None
        w = {n: np.zeros(sh, np.uint16) for n, sh in mla.weight_shapes(ctx.cfg).items()}
        w["attn_sinks"] = sinks
        ctx.set_layer_weights(0, w)
        base = ctx.seq_alloc()
        fill(torch, ctx, base, prefix, gen, row)
        seqs = [ctx.seq_fork(base, prefix) for _ in range(users)]
        steps = []
        for i, s in enumerate(seqs):
            n = 1 + (i * 37) % own
            fill(torch, ctx, s, n - 1 + q_len, gen, row, prefix)
            steps.append((s, prefix + n - 1, q_len))
        for i in range(others):
            s = ctx.seq_alloc()
            fill(torch, ctx, s, 100 + 37 * i + 1, gen, row)
            steps.insert(3 * i, (s, 100 + 37 * i, 1))
        T = sum(s[2] for s in steps)
        q = bits(rng.standard_normal((T * 64, row)).astype(np.float32) * (3.0 if v4 else 1.0))
        got = run_batch(torch, ctx, steps, q, T, True)
        check_on_device(torch, ctx, steps, q, got, True, sinks)
        for _ in range(3):
            assert np.array_equal(run_batch(torch, ctx, steps, q, T, True), got)


@pytest.mark.parametrize("prefix,users", [(64, 2400), (130, 1301), (200, 900)])
def test_many_users_of_a_page_or_two(torch, prefix, users):
    """Segments of one, two and three tiles, many to a block; more users than thread blocks."""
    rng = np.random.default_rng(13)
    with make(e4m3=False, n_pages=users + 10, max_seqs=users + 1, max_tokens=users) as ctx:
        base = ctx.seq_alloc()
        ctx.cache_write(0, base, 0, rows_of(rng, prefix))
        seqs = [ctx.seq_fork(base, prefix) for _ in range(users)]
        steps = [(s, prefix, 1, -1, 0) for s in seqs]
        q = bits(rng.standard_normal((users * 64, 576)).astype(np.float32))
        launches = ctx.launch_count()
        got = run_batch(torch, ctx, steps, q, users, False)
        k = torch.from_numpy(f32(ctx.cache_read(0, base, 0, prefix)).astype(np.float64)).cuda()
        qd = torch.from_numpy(q.view(np.int16)).cuda().view(torch.bfloat16).double()
        p = torch.softmax(qd @ k.T * 192.0 ** -0.5, 1)
        o, a = p @ k[:, :512], p @ k[:, :512].abs()
        err = (torch.from_numpy(f32(got).astype(np.float64)).cuda().reshape(-1, 512) - o).abs()
        assert bool((err <= 2.0 ** -8 * a + 2.0 ** -8 * o.abs()).all())
        assert np.array_equal(run_batch(torch, ctx, steps, q, users, False), got)
        assert ctx.launch_count() > launches


@pytest.mark.parametrize("n_seq,ctx_len,q_len", [(4, 6000, 16), (3, 9000, 11), (2, 4000, 40)])
def test_verify_blocks_over_expanded_pages(torch, n_seq, ctx_len, q_len):
    """Blocks of new tokens over an E4M3 cache, whose pages are expanded to bf16 for them."""
    rng = np.random.default_rng(10)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(11)
    with make(n_pages=n_seq * (ctx_len // 64 + 3), max_seqs=n_seq, max_tokens=512) as ctx:
        steps = []
        for i in range(n_seq):
            s = ctx.seq_alloc()
            n = ctx_len - 61 * i
            fill(torch, ctx, s, n + q_len, gen, 576)
            steps.append((s, n, q_len))
        T = n_seq * q_len
        q = bits(rng.standard_normal((T * 64, 576)).astype(np.float32))
        for causal in (True, False):
            got = run_batch(torch, ctx, steps, q, T, causal)
            check_on_device(torch, ctx, steps, q, got, causal)


def test_sharp_softmax(torch):
    """Scores that grow along the prefix: the running maximum moves in almost every tile, for each token at its own places."""
    rng = np.random.default_rng(12)
    with make(e4m3=False, n_pages=400, max_seqs=20, max_tokens=512) as ctx:
        base = ctx.seq_alloc()
        n = 64 * 160
        x = rng.standard_normal((n, 576)).astype(np.float32) * 0.05
        x[:, 0] = np.linspace(0, 40, n)
        x[:, 1] = np.linspace(40, 0, n)
        x[:, 570] = 30 * np.sin(np.linspace(0, 60, n))
        ctx.cache_write(0, base, 0, bits(x))
        seqs = [ctx.seq_fork(base, n) for _ in range(16)]
        steps = [(s, n, 1, -1, 0) for s in seqs]
        q = np.zeros((16, 64, 576), np.float32)
        q[:, :, 0] = rng.uniform(0, 60, (16, 64))
        q[:, :, 1] = rng.uniform(0, 60, (16, 64))
        q[:, :, 570] = rng.uniform(-40, 40, (16, 64))
        q = bits(q.reshape(16 * 64, 576))
        got = run_batch(torch, ctx, steps, q, 16, False)
        check_on_device(torch, ctx, steps, q, got, False)
