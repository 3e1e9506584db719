"""The paged cache on the GPU (slm_paged.h): append, single tokens and runs of
rows against the operators written out in 64 bits (paged_testlib)."""
import ctypes
import math

import numpy as np
import pytest

from paged_testlib import BF16, SENTINEL, U, Batch, check_attention, to_bf16
from slm_testlib import assert_bitwise, load_product

P = load_product()
pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def log(msg):
    print(msg, flush=True)


# ---- single tokens ----

# lengths around a page, a tile and several chunks, an empty sequence among them
LENS = [1, 0, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 300, 1000]

HEADS = [  # heads, kv_heads, hd: every head_dim, kv_mul 1 to 16
    (4, 4, 16), (8, 2, 32), (6, 6, 48), (9, 3, 64), (8, 8, 96), (8, 2, 128), (4, 4, 256),
    (10, 2, 32), (7, 1, 64), (16, 2, 128), (32, 2, 16), (4, 2, 256), (6, 2, 96), (12, 2, 48),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,hd", HEADS)
def test_decode_every_head_layout(heads, kv_heads, hd, dtype):
    b = Batch(heads, kv_heads, hd, 16, [(m, 1) for m in LENS], dtype, seed=1, decode=True)
    with b.upload(torch, layers=3, layer=1) as d:
        rel = check_attention(d.host(d.attend()), b)
    log(f"{heads}/{kv_heads} heads of {hd}, {dtype}: {rel:.2e}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (7, 3), (64, 4), (100, 17), (5000, 9)])
def test_decode_pages_windows_sinks(page, window, sinks, dtype):
    b = Batch(8, 2, 64, page, [(m, 1) for m in LENS], dtype, seed=2, decode=True)
    with b.upload(torch) as d:
        check_attention(d.host(d.attend(window, sinks)), b, window, sinks)


@pytest.mark.parametrize("hd,heads,kv_heads,dtype", [(128, 8, 2, "bf16"), (64, 3, 1, "f32"),
                                                     (256, 4, 1, "bf16")])
@pytest.mark.parametrize("length", [1, 4097, 20011])
def test_decode_one_long_sequence(hd, heads, kv_heads, dtype, length):
    b = Batch(heads, kv_heads, hd, 64, [(length, 1)], dtype, seed=3, decode=True)
    with b.upload(torch) as d:
        check_attention(d.host(d.attend()), b)
        out = torch.full_like(d.out, SENTINEL)
        check_attention(d.host(d.attend(1000, 5, out)), b, 1000, 5)


def test_decode_many_sequences():
    # more rows than a wave has lanes, and than one plan stretch
    rng = np.random.default_rng(4)
    b = Batch(4, 2, 32, 16, [(int(m), 1) for m in rng.integers(0, 90, 200)], "bf16", seed=4,
              decode=True)
    with b.upload(torch) as d:
        first = d.host(d.attend()).copy()
        check_attention(first, b)
        assert_bitwise(d.host(d.attend()), first, "the same call again")


# ---- runs of rows ----

RUNS = [(0, 0), (1, 1), (16, 16), (5, 0), (40, 7), (17, 17), (130, 1), (200, 65), (90, 90),
        (3, 2), (33, 16)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,hd", HEADS)
def test_runs_every_head_layout(heads, kv_heads, hd, dtype):
    b = Batch(heads, kv_heads, hd, 16, RUNS, dtype, seed=5, tail=3)
    with b.upload(torch, layers=2, layer=1) as d:
        rel = check_attention(d.host(d.attend()), b)
    log(f"{heads}/{kv_heads} heads of {hd}, {dtype}: {rel:.2e}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (7, 3), (64, 4), (100, 17), (5000, 9)])
def test_runs_pages_windows_sinks(page, window, sinks, dtype):
    b = Batch(8, 2, 128, page, RUNS, dtype, seed=6)
    with b.upload(torch) as d:
        check_attention(d.host(d.attend(window, sinks)), b, window, sinks)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd,heads,kv_heads", [(128, 8, 2), (64, 6, 2)])
@pytest.mark.parametrize("seqs", [[(700, 700)], [(1500, 300), (64, 64), (900, 1)]])
def test_runs_long(hd, heads, kv_heads, dtype, seqs):
    b = Batch(heads, kv_heads, hd, 32, seqs, dtype, seed=7)
    with b.upload(torch) as d:
        check_attention(d.host(d.attend()), b)
        out = torch.full_like(d.out, SENTINEL)
        check_attention(d.host(d.attend(200, 4, out)), b, 200, 4)


def test_more_rows_than_the_sequence_holds():
    # rows in front of position 0 are empty: zeros
    b = Batch(4, 2, 64, 16, [(3, 8), (20, 4), (0, 5)], "f32", seed=8)
    with b.upload(torch) as d:
        got = d.host(d.attend())
        assert np.all(got[:5] == 0) and np.all(got[12:] == 0)
        check_attention(got, b)


# ---- values that are not finite, in places that a row does not see ----

@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_hidden_rows_may_hold_anything(dtype, value):
    # rows behind a row's position and outside its window, in pages and tiles
    # that it does read
    b = Batch(8, 2, 64, 16, [(120, 40), (50, 50)], dtype, seed=9)
    clean = Batch(8, 2, 64, 16, [(120, 40), (50, 50)], dtype, seed=9)
    window, sinks = 20, 2
    hit = {0: [110, 118, 10], 1: [3, 30, 45]}
    for i, ts in hit.items():
        for t in ts:
            b.pool[b.table[i, t // 16], :, :, t % 16] = value
    with b.upload(torch) as d:
        got = d.host(d.attend(window, sinks))
    want, tol = clean.attend64(window, sinks)
    seen_any = 0
    for r, i, p in b.positions():
        sees = any(t <= p and (t > p - window or t < sinks) for t in hit[i])
        if sees:
            seen_any += 1
            continue
        assert np.all(np.abs(got[r] - want[r]) <= tol[r]), (r, i, p)
    assert 0 < seen_any < b.n


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_visible_nan_or_infinite_v_shows_in_its_dimension(dtype):
    b = Batch(4, 2, 64, 16, [(70, 1), (33, 1)], dtype, seed=10, decode=True)
    b.pool[b.table[0, 2], 1, 0, 5, 7] = math.nan
    b.pool[b.table[1, 1], 1, 1, 3, 9] = math.inf
    with b.upload(torch) as d:
        got = d.host(d.attend()).reshape(2, 4, 64)
    assert np.isnan(got[0, :2, 7]).all() and np.isinf(got[1, 2:, 9]).all()
    got[0, :2, 7] = got[1, 2:, 9] = 0
    assert np.isfinite(got).all()


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("q_scale,k_scale", [(1e-30, 1e30), (1e18, 1e-18), (1e-20, 1.0)])
def test_values_of_any_size(q_scale, k_scale, dtype, decode):
    b = Batch(4, 2, 64, 16, [(70, 1 if decode else 30), (33, 1 if decode else 33)], dtype,
              seed=11, decode=decode, q_scale=q_scale, k_scale=k_scale)
    with b.upload(torch) as d:
        check_attention(d.host(d.attend()), b)


# ---- bad metadata ----

@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_bad_pages_and_lengths_give_nan_rows(dtype, decode):
    rows = 1 if decode else 20
    b = Batch(8, 2, 64, 16, [(70, rows)] * 6, dtype, seed=12, decode=decode)
    b.table[1, 2] = b.pages  # behind the pool
    b.table[2, 0] = -1
    want, tol = Batch(8, 2, 64, 16, [(70, rows)] * 6, dtype, seed=12, decode=decode).attend64()
    with b.upload(torch) as d:
        lens = b.lens.copy()
        lens[3], lens[4] = -5, b.max_len + 1
        d.lens.copy_(torch.from_numpy(lens))
        torch.cuda.synchronize()
        got = d.host(d.attend()).reshape(6, rows, -1)
    want, tol = want.reshape(got.shape), tol.reshape(got.shape)
    for i in range(6):
        if i in (0, 5):
            assert np.all(np.abs(got[i] - want[i]) <= tol[i])
        else:
            assert np.isnan(got[i]).all(), i


def test_row_starts_that_make_no_sense_stay_inside():
    b = Batch(4, 2, 64, 16, [(40, 10), (30, 10), (20, 10)], "bf16", seed=13, tail=2)
    with b.upload(torch) as d:
        for bad in ([0, 20, 10, 30], [-100, 5, 1 << 30, 30], [0, 0, 0, 1 << 30],
                    [30, 20, 10, 0], [5, 5, 5, 5]):
            d.row_start.copy_(torch.tensor(bad, dtype=torch.int32))
            d.out.fill_(SENTINEL)
            torch.cuda.synchronize()
            d.attend()
            d.append()
            d.ctx.sync()
        d.row_start.copy_(torch.from_numpy(b.row_start))


# ---- append ----

def append64(b, tables, q_norm, k_norm, eps):
    """(q_out, pool) of an append in 64 bits, with the context's own tables."""
    cos, sin = (t.astype(np.float64) for t in tables)
    out = np.full((b.n, b.dim), SENTINEL, np.float64)
    pool = b.pool.astype(np.float64)

    def turn(x, w, p):
        x = x.astype(np.float64).reshape(-1, b.hd)
        if w is not None:
            x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
        y = np.empty_like(x)
        y[:, 0::2] = x[:, 0::2] * cos[p] - x[:, 1::2] * sin[p]
        y[:, 1::2] = x[:, 0::2] * sin[p] + x[:, 1::2] * cos[p]
        return y

    for r, i, p in b.positions():
        if p < 0:
            continue
        out[r] = turn(b.q[r], q_norm, p).reshape(-1)
        page = b.table[i, p // b.page]
        pool[page, 0, :, p % b.page] = turn(b.k[r], k_norm, p)
        pool[page, 1, :, p % b.page] = b.v[r].reshape(b.kv_heads, b.hd)
    return out, pool


def check_append(got_q, got_pool, b, tables, q_norm=None, k_norm=None, eps=1e-5):
    """A norm's sum of hd squares is off by (hd + 2) u at most, so its root by
    half of that, the division, root and two products by 4 u; a rotated value is
    the sum of two products, off by 3 u of their magnitudes; together (hd / 2 +
    8) u of |x| |cos| + |y| |sin| <= sqrt(2) times the pair's length.  A bf16
    value is off by another half step."""
    want_q, want_pool = append64(b, tables, q_norm, k_norm, eps)
    pair = lambda x: np.repeat(np.hypot(x[..., 0::2], x[..., 1::2]), 2, -1)  # noqa: E731
    tq = (b.hd / 2 + 8) * U * math.sqrt(2) * pair(want_q)
    assert np.all(np.abs(got_q - want_q) <= tq), "q"
    hit = want_pool != b.pool.astype(np.float64)
    hit &= ~(np.isnan(want_pool) & np.isnan(b.pool))
    same = got_pool[~hit]
    assert np.array_equal(same, b.pool[~hit], equal_nan=True), "a row that is not the call's"
    tk = (b.hd / 2 + 8) * U * math.sqrt(2) * pair(want_pool)
    tk[:, 1] = 0.0  # V is stored as it is
    if b.dtype == "bf16":
        tk += BF16 * (np.abs(want_pool) + tk)
    assert np.all(np.abs(got_pool[hit] - want_pool[hit]) <= tk[hit]), "cache"


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("norms", ["", "q", "k", "qk"])
@pytest.mark.parametrize("heads,kv_heads,hd", HEADS[:7] + [(7, 1, 64)])
def test_append_every_head_dim(heads, kv_heads, hd, norms, dtype):
    b = Batch(heads, kv_heads, hd, 16, RUNS + [(3, 8)], dtype, seed=20, tail=2)
    w = {c: (1 + 0.1 * b.rng.standard_normal(hd)).astype(np.float32) if c in norms else None
         for c in "qk"}
    with b.upload(torch, layers=2, layer=1) as d:
        wd = {c: torch.from_numpy(w[c]).cuda() if w[c] is not None else None for c in "qk"}
        torch.cuda.synchronize()
        got = d.host(d.append(wd["q"], wd["k"]))
        pool = d.host(d.pool)
        check_append(got, pool, b, d.ctx.rope_tables(), w["q"], w["k"])
        assert d.all_layers[0].isnan().all().item(), "another layer was written"


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_append_single_tokens(page, dtype):
    b = Batch(8, 2, 128, page, [(m, 1) for m in LENS], dtype, seed=21, decode=True)
    with b.upload(torch) as d:
        got = d.host(d.append())
        check_append(got, d.host(d.pool), b, d.ctx.rope_tables())


def test_append_gives_the_arenas_bits():
    # f32 without norms: the rows that slm_kv_append_dev and slm_rope_apply_dev give
    b = Batch(9, 3, 64, 16, [(40, 40)], "f32", seed=22)
    with b.upload(torch) as d:
        q = d.host(d.append())
        d.ctx.kv_append_dev(0, 0, 40, d.k.data_ptr(), d.v.data_ptr())
        d.ctx.rope_apply_dev(d.q.data_ptr(), 40, b.dim, 0)
        assert_bitwise(q, d.host(d.q), "q")
        pool = d.host(d.pool)
        for which in (0, 1):
            rows = np.moveaxis(pool[b.table[0, :3], which], 1, 2).reshape(-1, b.kvd)[:40]
            assert_bitwise(rows, d.ctx.kv_read(0, which, 0, 40), "K V"[2 * which])


def test_append_in_place_and_without_q():
    b = Batch(4, 2, 64, 16, [(20, 5), (9, 9)], "bf16", seed=23, tail=1)
    with b.upload(torch) as d:
        want = d.host(d.append()).copy()
        pool = d.host(d.pool).copy()
        d.pool.copy_(torch.from_numpy(b.pool))
        torch.cuda.synchronize()
        d.append(with_q=False)
        assert np.array_equal(d.host(d.pool), pool, equal_nan=True)
        q0 = d.host(d.q).copy()
        got = d.host(d.append(q_out=d.q))
        assert_bitwise(got[:b.rows], want[:b.rows], "in place")
        assert_bitwise(got[b.rows:], q0[b.rows:], "rows of no sequence")


def test_append_bad_metadata():
    b = Batch(4, 2, 64, 16, [(40, 4)] * 4, "f32", seed=24)
    b.table[1, 2] = b.pages + 3  # the new rows' page
    with b.upload(torch) as d:
        lens = b.lens.copy()
        lens[2], lens[3] = -1, b.max_len + 7
        d.lens.copy_(torch.from_numpy(lens))
        torch.cuda.synchronize()
        got = d.host(d.append())
        pool = d.host(d.pool)
    assert np.isfinite(got[:8]).all() and np.isnan(got[8:]).all()
    changed = ~((pool == b.pool) | (np.isnan(pool) & np.isnan(b.pool)))
    assert set(np.argwhere(changed)[:, 0]) == {b.table[0, 2]}


# ---- as they are used together ----

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_conversations_grow_as_the_arena_does(dtype):
    """Three conversations in one paged cache, prompts first and then tokens
    one at a time, against each of them alone in an arena.  With f32 pages the
    two differ by the order of sums only, twice the bound of attend64; bf16
    pages are checked against attend64 itself."""
    heads, kv_heads, hd, msl, theta = 9, 3, 64, 96, 1e5
    dim, kvd = heads * hd, kv_heads * hd
    rng = np.random.default_rng(25)
    prompts, steps = [17, 40, 1], 9
    data = [[(rng.standard_normal((n + steps, w)) * s).astype(np.float32)
             for w, s in ((dim, 1.0), (kvd, 1.0), (kvd, 0.5))] for n in prompts]
    b = Batch(heads, kv_heads, hd, 16, [(n + steps, n) for n in prompts], dtype, seed=25)
    b.pool[:] = np.nan
    with b.upload(torch, theta=theta, msl=msl) as d:
        d.cache_rows = None
        up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        arenas = [P.AttentionContext(dim, heads, kv_heads, msl, 1, theta) for _ in prompts]
        for step in range(steps + 1):
            rows = [slice(0, n) if step == 0 else slice(n + step - 1, n + step) for n in prompts]
            lens = np.array([r.stop for r in rows], np.int32)
            counts = [r.stop - r.start for r in rows]
            q, k, v = (np.concatenate([c[j][r] for c, r in zip(data, rows)]) for j in range(3))
            b.lens, b.q, b.n = lens, q, len(q)
            b.rows, b.row_start = b.n, np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
            d.q, d.k, d.v = up(q), up(k), up(v)
            d.out = torch.empty((b.n, dim), device="cuda")
            d.lens.copy_(up(lens))
            d.row_start.copy_(up(b.row_start))
            bt = P.PagedBatch(3, d.table.data_ptr(), b.stride, d.lens.data_ptr(), msl
                              if msl <= b.stride * 16 else b.max_len,
                              d.row_start.data_ptr() if step == 0 else 0, b.n)
            d.batch = bt
            torch.cuda.synchronize()
            d.append(q_out=d.q)
            got = d.host(d.attend())
            b.q, b.pool = d.host(d.q), d.host(d.pool)
            want, tol = b.attend64()
            assert np.all(np.abs(got - want) <= tol), step
            if dtype == "f32":
                for i, (c, r) in enumerate(zip(data, rows)):
                    ref = arenas[i].prefill(0, r.start, *(x[r] for x in c))
                    at = slice(b.row_start[i], b.row_start[i + 1])
                    assert np.all(np.abs(got[at] - ref) <= 2 * tol[at]), (step, i)
        for a in arenas:
            a.close()


@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 2)])
def test_graph_replays_follow_the_lengths(window, sinks):
    """A captured step of append and attention, replayed while the lengths and
    rows on the device move on; every replay against the same calls made
    eagerly on another cache."""
    b = Batch(8, 2, 64, 16, [(60, 1), (33, 1), (0, 1), (5, 1)], "bf16", seed=26, decode=True)
    rng = np.random.default_rng(27)
    with b.upload(torch, msl=80) as d, b.upload(torch, ctx=d.ctx) as e:
        d.batch.c.max_len = e.batch.c.max_len = min(80, b.stride * 16)
        q_rot = [torch.empty_like(d.q), torch.empty_like(d.q)]
        torch.cuda.synchronize()
        d.append(q_out=q_rot[0])  # sizes nothing: the calls allocate nothing
        d.ctx.sync()
        d.pool.copy_(torch.from_numpy(b.pool))
        torch.cuda.synchronize()
        d.ctx.capture_begin()
        d.append(q_out=q_rot[0])
        d.ctx.paged_attend_dev(d.cache, 0, d.batch, q_rot[0].data_ptr(), d.out.data_ptr(), window,
                               sinks)
        graph = d.ctx.capture_end()
        with graph:
            for step in range(4):
                lens = torch.tensor([60 + step, 33 + step, 0, 5 + step], dtype=torch.int32)
                for x in (d, e):
                    x.lens.copy_(lens)
                    x.out.fill_(SENTINEL)
                for name in "qkv":
                    new = torch.from_numpy(rng.standard_normal(
                        getattr(d, name).shape).astype(np.float32))
                    getattr(d, name).copy_(new)
                    getattr(e, name).copy_(new)
                torch.cuda.synchronize()
                d.ctx.graph_launch(graph)
                e.append(q_out=q_rot[1])
                e.ctx.paged_attend_dev(e.cache, 0, e.batch, q_rot[1].data_ptr(),
                                       e.out.data_ptr(), window, sinks)
                assert_bitwise(d.host(d.out), d.host(e.out), f"replay {step}")
                assert np.array_equal(d.host(d.pool), d.host(e.pool), equal_nan=True)
                assert np.all(d.host(d.out)[2] == 0)


def test_on_another_stream():
    b = Batch(8, 2, 128, 32, [(500, 1), (90, 1)], "bf16", seed=28, decode=True)
    with b.upload(torch) as d:
        s = torch.cuda.Stream()
        d.ctx.set_stream(s.cuda_stream)
        q = d.q.clone()
        d.q.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            d.q.copy_(q)  # on the stream, ahead of the call
        got = d.host(d.attend())
        check_attention(got, b)
        d.ctx.set_stream(None)


def test_a_shared_prefix_may_be_read_by_both():
    b = Batch(4, 2, 64, 16, [(40, 1), (40, 1)], "f32", seed=29, decode=True)
    b.table[1, :2] = b.table[0, :2]  # the first two pages are common
    with b.upload(torch) as d:
        check_attention(d.host(d.attend()), b)


# ---- refusals ----

def test_refusals():
    b = Batch(4, 2, 64, 16, [(40, 4), (20, 2)], "f32", seed=30)
    with b.upload(torch, max_seqs=2) as d:
        ctx, cache = d.ctx, d.cache

        def code(fn):
            with pytest.raises(P.SlmAttnError) as ei:
                fn()
            return ei.value.code

        def batch(**kw):
            bt = P.PagedBatch(2, d.table.data_ptr(), b.stride, d.lens.data_ptr(), b.max_len,
                              d.row_start.data_ptr(), b.n)
            for k, v in kw.items():
                setattr(bt.c, k, v)
            return bt

        q, k, v, o = (t.data_ptr() for t in (d.q, d.k, d.v, d.out))
        calls = [lambda bt, layer=0: ctx.paged_attend_dev(cache, layer, bt, q, o),
                 lambda bt, layer=0: ctx.paged_append_dev(cache, layer, bt, q, k, v, o)]
        for call in calls:
            assert code(lambda: call(batch(), 1)) == P.ERR_LAYER
            assert code(lambda: call(batch(), -1)) == P.ERR_LAYER
            for kw in (dict(n_seqs=-1), dict(n_rows=-1), dict(n_seqs=3), dict(max_len=0),
                       dict(max_len=41), dict(table_stride=0), dict(table_stride=2),
                       dict(row_start=None)):
                assert code(lambda: call(batch(**kw))) == P.ERR_BATCH, kw
            for kw in (dict(page_table=None), dict(lens=None),
                       dict(lens=d.lens.data_ptr() + 2)):
                assert code(lambda: call(batch(**kw))) == P.ERR_ARG, kw
            call(batch(n_seqs=0))
            call(batch(n_rows=0))
        at, ap = ctx.paged_attend_dev, ctx.paged_append_dev
        bt = batch()
        assert code(lambda: at(cache, 0, bt, q, o, -1, 0)) == P.ERR_ARG
        assert code(lambda: at(cache, 0, bt, q, o, 8, -1)) == P.ERR_ARG
        assert code(lambda: at(cache, 0, bt, None, o)) == P.ERR_ARG
        assert code(lambda: at(cache, 0, bt, q, o + 4)) == P.ERR_ARG
        assert code(lambda: at(cache, 0, bt, q, q)) == P.ERR_ALIAS
        assert code(lambda: at(cache, 0, bt, q, q + 16)) == P.ERR_ALIAS
        assert code(lambda: at(cache, 0, bt, q, cache.device_ptr())) == P.ERR_ALIAS
        assert code(lambda: ap(cache, 0, bt, q, k, v, 0)) == P.ERR_ARG
        assert code(lambda: ap(cache, 0, bt, q, None, v, o)) == P.ERR_ARG
        assert code(lambda: ap(cache, 0, bt, q, k, v + 4, o)) == P.ERR_ARG
        assert code(lambda: ap(cache, 0, bt, q, k, v, o, q_norm=k + 8)) == P.ERR_ARG
        assert code(lambda: ap(cache, 0, bt, q, k, v, o, q_norm=k, norm_eps=-1.0)) == P.ERR_ARG
        assert code(lambda: ap(cache, 0, bt, q, k, v, q + 16)) == P.ERR_ALIAS
        assert code(lambda: ap(cache, 0, bt, q, k, v, k)) == P.ERR_ALIAS
        assert code(lambda: ap(cache, 0, bt, q, cache.device_ptr(), v, o)) == P.ERR_ALIAS
        assert code(lambda: ap(cache, 0, bt, q, k, v, d.lens.data_ptr() & ~15)) == P.ERR_ALIAS
        with P.AttentionContext(b.dim, b.heads, b.kv_heads, 64, 1) as other:
            assert code(lambda: other.paged_attend_dev(cache, 0, bt, q, o)) == P.ERR_ARG
        ctx.capture_begin()
        assert code(lambda: P.PagedCache(ctx, 1, 4)) == P.ERR_CAPTURE
        ctx.capture_end().close()
        for kw in (dict(num_layers=0), dict(num_pages=0), dict(page_size=8), dict(page_size=48),
                   dict(page_size=512), dict(max_seqs=0), dict(max_seqs=65537),
                   dict(num_layers=1 << 20, num_pages=1 << 30)):
            args = dict(num_layers=1, num_pages=4, page_size=16, max_seqs=4) | kw
            assert code(lambda: P.PagedCache(ctx, **args)) == P.ERR_CONFIG, kw
        with pytest.raises(ValueError):
            P.PagedCache(ctx, 1, 4, dtype="f16")
        assert cache.offset(0, 1, 1, 1, 3) == ((1 * 2 + 1) * 2 + 1) * 16 * 64 + 3 * 64
        bad = ctypes.c_size_t(-1).value
        for a in ((1, 0, 0, 0, 0), (0, b.pages, 0, 0, 0), (0, 0, 2, 0, 0), (0, 0, 0, 2, 0),
                  (0, 0, 0, 0, 16)):
            assert cache.offset(*a) == bad
