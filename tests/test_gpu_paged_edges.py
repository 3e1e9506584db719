"""The paged cache on the GPU at its edges: many sequences, rows split over
workgroups, values at the ends of their types, windows that hide nothing, pools
of more than 2^32 values, and the workspace that a cache's calls share."""
import math

import numpy as np
import pytest

from paged_testlib import SENTINEL, Batch, check_attention, to_bf16
from slm_testlib import assert_bitwise, load_product

P = load_product()
pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

INT_MAX = 0x7FFFFFFF


# ---- many sequences ----

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,hd", [(4, 2, 64), (8, 1, 128), (6, 6, 48)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3)])
def test_runs_of_more_sequences_than_a_wave_has_lanes(heads, kv_heads, hd, dtype, window, sinks):
    rng = np.random.default_rng(40)
    seqs = [(int(m), int(min(m, r))) for m, r in zip(rng.integers(0, 120, 150),
                                                     rng.integers(0, 70, 150))]
    b = Batch(heads, kv_heads, hd, 16, seqs, dtype, seed=40, tail=5)
    with b.upload(torch) as d:
        first = d.host(d.attend(window, sinks)).copy()
        check_attention(first, b, window, sinks)
        assert_bitwise(d.host(d.attend(window, sinks)), first, "the same call again")


@pytest.mark.parametrize("decode", [True, False])
def test_thousands_of_short_sequences(decode):
    rng = np.random.default_rng(41)
    b = Batch(4, 2, 16, 16, [(int(m), 1) for m in rng.integers(0, 4, 3000)], "bf16", seed=41,
              decode=decode)
    with b.upload(torch) as d:
        check_attention(d.host(d.attend()), b)


# ---- rows split over workgroups ----

SPLIT = [(128, 8, 2, [(3000, 20)]), (64, 6, 2, [(2500, 33), (2500, 1), (0, 0), (700, 5)]),
         (48, 6, 6, [(1800, 40)]), (256, 4, 1, [(1500, 9), (900, 3)]), (96, 4, 2, [(2100, 50)]),
         (16, 4, 4, [(5000, 7)]), (32, 8, 2, [(4100, 64)])]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd,heads,kv_heads,seqs", SPLIT)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1500, 70)])
def test_few_rows_behind_many(hd, heads, kv_heads, seqs, dtype, window, sinks):
    b = Batch(heads, kv_heads, hd, 16, seqs, dtype, seed=42, tail=2)
    with b.upload(torch) as d:
        first = d.host(d.attend(window, sinks)).copy()
        check_attention(first, b, window, sinks)
        assert_bitwise(d.host(d.attend(window, sinks)), first, "the same call again")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd,heads,kv_heads", [(128, 8, 2), (64, 3, 3), (256, 4, 1)])
def test_bad_page_in_one_part_of_a_split_row(hd, heads, kv_heads, dtype):
    seqs = [(3000, 6), (3000, 6)]
    b = Batch(heads, kv_heads, hd, 32, seqs, dtype, seed=43)
    clean = Batch(heads, kv_heads, hd, 32, seqs, dtype, seed=43)
    b.table[1, 40] = b.pages
    want, tol = clean.attend64()
    with b.upload(torch) as d:
        got = d.host(d.attend())
        assert np.all(np.abs(got[:6] - want[:6]) <= tol[:6])
        assert np.isnan(got[6:]).all()
        # a window that the page lies in front of
        out = torch.full_like(d.out, SENTINEL)
        want, tol = clean.attend64(900, 9)
        got = d.host(d.attend(900, 9, out))
        assert np.all(np.abs(got - want) <= tol)


# ---- values at the ends of their types ----

def scaled(b, which, factor):
    b.pool[:, which] *= np.float32(factor)
    if b.dtype == "bf16":
        b.pool = to_bf16(b.pool)
    return b


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("seqs", [[(70, 30), (33, 33)], [(2900, 12)]])
@pytest.mark.parametrize("k_scale,v_scale,q_scale", [
    (1.0, 2.0 ** 70, 1.0),  # V that bf16 planes must not be multiplied with
    (2.0 ** 80, 1.0, 2.0 ** -80), (2.0 ** -60, 2.0 ** -60, 2.0 ** 60),
    (2.0 ** -86, 1.0, 2.0 ** 86), (1.0, 2.0 ** -100, 1.0)])
def test_large_and_small_values(k_scale, v_scale, q_scale, seqs, dtype):
    b = Batch(8, 2, 64, 16, seqs, dtype, seed=44, q_scale=q_scale)
    scaled(scaled(b, 0, k_scale), 1, v_scale)
    with b.upload(torch) as d:
        check_attention(d.host(d.attend()), b)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,hd", [(8, 2, 64), (8, 2, 128), (6, 2, 96), (8, 2, 32)])
@pytest.mark.parametrize("k_scale,v_scale,q_scale", [
    (1.0, 2.0 ** 70, 1.0), (2.0 ** 80, 1.0, 2.0 ** -80), (2.0 ** -86, 1.0, 2.0 ** 86),
    (1.0, 2.0 ** -100, 1.0)])
def test_large_and_small_values_of_single_tokens(heads, kv_heads, hd, k_scale, v_scale, q_scale,
                                                 dtype):
    b = Batch(heads, kv_heads, hd, 16, [(m, 1) for m in (1, 70, 0, 130, 2900)], dtype, seed=55,
              decode=True, q_scale=q_scale)
    scaled(scaled(b, 0, k_scale), 1, v_scale)
    with b.upload(torch) as d:
        check_attention(d.host(d.attend()), b)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [32, 64, 96, 128])
def test_nan_and_infinity_stay_in_their_head_and_dimension(hd, dtype):
    # the last key of a row and one amid a tile; NaN in one row's query
    b = Batch(8, 2, hd, 16, [(70, 1), (33, 1), (45, 1)], dtype, seed=56, decode=True)
    want, tol = b.attend64()
    want, tol = want.reshape(3, 8, hd), tol.reshape(3, 8, hd)
    b.pool[b.table[0, 4], 1, 0, 5, 7] = math.nan
    b.pool[b.table[1, 1], 1, 1, 3, 9] = -math.inf
    b.q[2, 3 * hd + 1] = math.nan
    with b.upload(torch) as d:
        got = d.host(d.attend()).reshape(3, 8, hd)
    assert np.isnan(got[0, :4, 7]).all() and (got[1, 4:, 9] == -math.inf).all()
    assert np.isnan(got[2, 3]).all()
    for r, h, c in ((0, slice(0, 4), 7), (1, slice(4, 8), 9), (2, 3, slice(None))):
        got[r, h, c] = want[r, h, c]
    assert np.all(np.abs(got - want) <= tol)


def test_small_f32_keys():
    b = Batch(8, 2, 64, 16, [(70, 30), (2900, 12)], "f32", seed=45, q_scale=2.0 ** 110)
    scaled(b, 0, 2.0 ** -110)
    with b.upload(torch) as d:
        check_attention(d.host(d.attend()), b)


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_equal_scores_of_any_size_weigh_the_same(dtype, decode):
    # the largest keys there are, and q of one sign: every key has the same
    # score, about 2^111, and an output is the mean of V
    b = Batch(4, 2, 256, 16, [(300, 1 if decode else 40), (77, 1 if decode else 77)], dtype,
              seed=46, decode=decode)
    b.pool[:, 0] = to_bf16(np.float32(3.3e38))
    b.q[:] = 2.0 ** -20
    with b.upload(torch) as d:
        got = d.host(d.attend())
    for r, i, p in b.positions():
        _, v = b.keys(i)
        want = np.repeat(v[:p + 1].mean(0), 2, axis=0).reshape(-1)
        mean_abs = np.repeat(np.abs(v[:p + 1]).mean(0), 2, axis=0).reshape(-1)
        assert np.all(np.abs(got[r] - want) <= (p + 17) * 2.0 ** -24 * mean_abs), (r, p)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("decode", [True, False])
def test_zero_keys_and_huge_queries(dtype, decode):
    b = Batch(4, 2, 64, 16, [(90, 1 if decode else 20)], dtype, seed=47, decode=decode,
              q_scale=3e37)
    b.pool[:, 0] = 0.0
    with b.upload(torch) as d:
        check_attention(d.host(d.attend()), b)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_nan_query_row_stays_alone(dtype):
    b = Batch(8, 2, 128, 16, [(70, 40)], dtype, seed=48)
    want, tol = b.attend64()
    b.q[7, 130] = math.nan  # head 1
    with b.upload(torch) as d:
        got = d.host(d.attend())
    assert np.isnan(got[7, 128:256]).all()
    got[7, 128:256] = want[7, 128:256]
    assert np.all(np.abs(got - want) <= tol)


# ---- windows ----

@pytest.mark.parametrize("decode", [True, False])
def test_windows_that_hide_nothing(decode):
    b = Batch(8, 2, 64, 16, [(130, 1 if decode else 60), (3, 1 if decode else 9)], "bf16", seed=49,
              decode=decode)
    with b.upload(torch) as d:
        full = d.host(d.attend()).copy()
        check_attention(full, b)
        for window, sinks in ((INT_MAX, INT_MAX), (INT_MAX, 0), (1, INT_MAX), (130, 0), (100, 30),
                              (0, 50)):
            out = torch.full_like(d.out, SENTINEL)
            assert_bitwise(d.host(d.attend(window, sinks, out)), full, f"{window} {sinks}")
        out = torch.full_like(d.out, SENTINEL)
        check_attention(d.host(d.attend(99, 30, out)), b, 99, 30)


# ---- memory ----

@pytest.mark.parametrize("decode", [True, False])
def test_a_pool_of_more_than_32_bits_of_values(decode):
    # pages of 2^19 values; the sequences lie in the last of 8400
    b = Batch(8, 8, 128, 256, [(700, 1 if decode else 40), (300, 1 if decode else 9)], "bf16",
              seed=50, decode=decode)
    pages = 8400
    with P.AttentionContext(b.dim, 8, 8, b.max_len, 1) as ctx:
        cache = P.PagedCache(ctx, 1, pages, 256, "bf16", 2)
        first = cache.offset(0, pages - b.pages, 0, 0, 0)
        assert first > 1 << 32

        class Tail:
            __cuda_array_interface__ = {"shape": b.pool.shape, "typestr": "<i2", "version": 3,
                                        "data": (cache.device_ptr() + 2 * first, False)}

        tail = torch.as_tensor(Tail(), device="cuda").view(torch.bfloat16)
        tail.copy_(torch.from_numpy(b.pool))
        table = np.where((b.table >= 0) & (b.table < b.pages), b.table + pages - b.pages, b.table)
        up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        table, lens, start = up(table.astype(np.int32)), up(b.lens), up(b.row_start)
        q, k, v = up(b.q), up(b.k), up(b.v)
        out = torch.full((b.n, b.dim), SENTINEL, device="cuda")
        batch = P.PagedBatch(2, table.data_ptr(), b.stride, lens.data_ptr(), b.max_len,
                             0 if decode else start.data_ptr(), b.n)
        torch.cuda.synchronize()
        ctx.paged_attend_dev(cache, 0, batch, q.data_ptr(), out.data_ptr())
        ctx.sync()
        check_attention(out.cpu().numpy(), b)
        ctx.paged_append_dev(cache, 0, batch, 0, k.data_ptr(), v.data_ptr(), 0)
        ctx.sync()
        got = tail.float().cpu().numpy()
        for r, i, p in b.positions():
            row = got[b.table[i, p // 256], 1, :, p % 256].reshape(-1)
            assert np.array_equal(row, to_bf16(b.v[r])), (r, p)
        cache.close()


def test_a_page_may_stand_twice_in_a_table():
    for decode in (True, False):
        b = Batch(4, 2, 64, 16, [(90, 1 if decode else 30)], "bf16", seed=51, decode=decode)
        b.table[0, 3] = b.table[0, 1]
        with b.upload(torch) as d:
            check_attention(d.host(d.attend()), b)


def test_two_graphs_share_a_workspace():
    """A split decode and a split run of rows, captured apart and replayed in
    turns, with eager calls and waits between; each replay against the first
    eager result."""
    one = Batch(8, 2, 128, 16, [(5000, 1), (900, 1)], "bf16", seed=52, decode=True)
    run = Batch(8, 2, 128, 16, [(3000, 10)], "bf16", seed=53)
    with one.upload(torch) as d, run.upload(torch, ctx=d.ctx) as e:
        # the run's batch over its own cache, and once more over the decode's workspace
        want = [d.host(d.attend()).copy(), d.host(e.attend()).copy()]
        check_attention(want[0], one)
        check_attention(want[1], run)
        outs = [torch.full_like(x.out, SENTINEL) for x in (d, d, e)]
        q2 = torch.from_numpy(one.q[::-1].copy()).cuda()
        torch.cuda.synchronize()
        eager2 = torch.full_like(d.out, SENTINEL)
        d.ctx.paged_attend_dev(d.cache, 0, d.batch, q2.data_ptr(), eager2.data_ptr())
        want2 = d.host(eager2).copy()
        graphs = []
        for call in (lambda: d.attend(out=outs[0]),
                     lambda: d.ctx.paged_attend_dev(d.cache, 0, d.batch, q2.data_ptr(),
                                                    outs[1].data_ptr()),
                     lambda: e.attend(out=outs[2])):
            d.ctx.capture_begin()
            call()
            graphs.append(d.ctx.capture_end())
        for step in range(4):
            for o in outs:
                o.fill_(SENTINEL)
            torch.cuda.synchronize()
            order = [0, 1, 2] if step % 2 else [2, 1, 0]
            for g in order:
                d.ctx.graph_launch(graphs[g])
            assert_bitwise(d.host(outs[0]), want[0], f"decode, replay {step}")
            assert_bitwise(d.host(outs[1]), want2, f"the other decode, replay {step}")
            assert_bitwise(d.host(outs[2]), want[1], f"run, replay {step}")
            assert_bitwise(d.host(d.attend()), want[0], f"eager, {step}")
        for g in graphs:
            g.close()


def test_two_contexts_at_once():
    """Split calls of two contexts, each on its stream, without waits between."""
    bs = [Batch(8, 2, 128, 16, [(6000, 1), (4000, 1)], "bf16", seed=54 + i, decode=True)
          for i in range(2)]
    with bs[0].upload(torch) as d, bs[1].upload(torch) as e:
        outs = [[torch.full_like(x.out, SENTINEL) for _ in range(6)] for x in (d, e)]
        torch.cuda.synchronize()
        for i in range(6):
            d.attend(out=outs[0][i])
            e.attend(out=outs[1][i])
        d.ctx.sync()
        e.ctx.sync()
        for x, b, os in ((d, bs[0], outs[0]), (e, bs[1], outs[1])):
            first = os[0].cpu().numpy()
            check_attention(first, b)
            for o in os[1:]:
                assert_bitwise(o.cpu().numpy(), first, "a call among others")


@pytest.mark.parametrize("decode", [True, False])
def test_nothing_but_empty_sequences(decode):
    b = Batch(4, 2, 64, 16, [(0, 1 if decode else 3)] * 5, "f32", seed=60, decode=decode)
    with b.upload(torch) as d:
        got = d.host(d.attend())
        assert np.all(got == 0)
        d.out.fill_(SENTINEL)
        torch.cuda.synchronize()
        assert np.all(d.host(d.append()) == SENTINEL)
        assert d.pool.isnan().all().item()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd,heads,kv_heads", [(64, 6, 2), (128, 8, 2), (48, 4, 4)])
def test_rows_in_front_of_the_first_sequence(hd, heads, kv_heads, dtype):
    # row_start[0] = 3: rows 0 to 2 belong to no sequence, nor do the last two
    b = Batch(heads, kv_heads, hd, 16, [(40, 7), (90, 33), (9, 9)], dtype, seed=61, tail=5)
    want, tol = b.attend64(20, 3)
    q = np.concatenate([b.q[b.rows:b.rows + 3], b.q[:b.rows], b.q[b.rows + 3:]])
    with b.upload(torch) as d:
        d.q.copy_(torch.from_numpy(q))
        d.row_start += 3
        torch.cuda.synchronize()
        got = d.host(d.attend(20, 3))
        assert np.all(got[:3] == SENTINEL) and np.all(got[b.rows + 3:] == SENTINEL)
        assert np.all(np.abs(got[3:b.rows + 3] - want[:b.rows]) <= tol[:b.rows])
        d.out.fill_(SENTINEL)
        torch.cuda.synchronize()
        out = d.host(d.append())
        assert np.all(out[:3] == SENTINEL) and np.all(out[b.rows + 3:] == SENTINEL)
        assert not np.any(out[3:b.rows + 3] == SENTINEL)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("window,sinks", [(0, 0), (30, 2), (9000, 1)])
def test_a_bound_far_above_the_lengths(decode, dtype, window, sinks):
    seqs = [(m, 1 if decode else r) for m, r in ((5, 5), (0, 2), (130, 40), (17, 1), (64, 64))]
    b = Batch(8, 2, 128, 16, seqs, dtype, seed=62, decode=decode, stride_extra=2000)
    b.max_len = 30000
    with b.upload(torch) as d:
        check_attention(d.host(d.attend(window, sinks)), b, window, sinks)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_windows_of_rows_in_front_of_the_sequence(dtype):
    # more rows than positions, with a window: the rows in front are zeros
    b = Batch(8, 2, 128, 16, [(20, 50), (200, 230), (1, 40)], dtype, seed=63)
    with b.upload(torch) as d:
        got = d.host(d.attend(6, 2))
        for r, _, p in b.positions():
            assert p >= 0 or np.all(got[r] == 0)
        check_attention(got, b, 6, 2)
