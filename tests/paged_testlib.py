"""What the tests of the paged cache share: batches with poisoned memory around
them, and the operators written out in 64 bits, one row after another.

Everything that a call must not use holds NaN (the pool outside the sequences'
own rows) or an id far outside the pool (table entries behind a sequence's last
page), so that a use shows."""
from __future__ import annotations

import math

import numpy as np

from slm_testlib import load_product

P = load_product()
U = 2.0 ** -24  # half a step of f32, relative
BF16 = 2.0 ** -8  # half a step of bf16, relative: eps / 2
SENTINEL = 777.0  # in outputs that a call leaves alone
JUNK = (-1, -7, 1 << 30, 0x7FFFFFFF)


def to_bf16(x):
    """f32 values rounded to bf16, ties to even."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint32) << 16
    out = r.astype(np.uint32).view(np.float32)
    return np.where(np.isnan(x), np.float32(np.nan), out)


class Batch:
    """seqs: [(len, new rows)].  The pool's rows of every sequence hold K from
    N(0, k_scale) and V from N(0, 0.5); `tail` rows of q belong to no sequence."""

    def __init__(self, heads, kv_heads, hd, page, seqs, dtype="f32", seed=0, decode=False,
                 tail=0, k_scale=1.0, q_scale=1.0, spare=3, stride_extra=1):
        self.heads, self.kv_heads, self.hd, self.page = heads, kv_heads, hd, page
        self.dtype, self.decode = dtype, decode
        self.seqs = list(seqs)
        rng = self.rng = np.random.default_rng([seed, heads, hd, page, len(self.seqs)])
        self.lens = np.array([m for m, _ in self.seqs], np.int32)
        counts = [1] * len(self.seqs) if decode else [r for _, r in self.seqs]
        self.row_start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.rows = int(self.row_start[-1])
        self.n = self.rows + (0 if decode else tail)
        self.max_len = max(1, int(self.lens.max(initial=0)))
        need = [-(-int(m) // page) for m in self.lens]
        self.stride = max(1, max(need, default=1)) + stride_extra
        self.pages = sum(need) + spare
        order = rng.permutation(self.pages).astype(np.int32)
        self.table = rng.choice(np.array(JUNK, np.int32), (len(self.seqs), self.stride))
        at = 0
        for i, k in enumerate(need):
            self.table[i, :k] = order[at:at + k]
            at += k
        self.pool = np.full((self.pages, 2, kv_heads, page, hd), np.nan, np.float32)
        for i, m in enumerate(self.lens):
            for t in range(0, int(m), page):
                w = min(page, int(m) - t)
                pg = self.table[i, t // page]
                self.pool[pg, 0, :, :w] = rng.standard_normal((kv_heads, w, hd)) * k_scale
                self.pool[pg, 1, :, :w] = rng.standard_normal((kv_heads, w, hd)) * 0.5
        if dtype == "bf16":
            self.pool = to_bf16(self.pool)
        self.dim, self.kvd = heads * hd, kv_heads * hd
        self.q = (rng.standard_normal((self.n, self.dim)) * q_scale).astype(np.float32)
        self.k = rng.standard_normal((self.n, self.kvd)).astype(np.float32)
        self.v = (rng.standard_normal((self.n, self.kvd)) * 0.5).astype(np.float32)

    def positions(self):
        """(row, sequence, position) of every row of a sequence."""
        for i, m in enumerate(self.lens):
            for r in range(self.row_start[i], self.row_start[i + 1]):
                yield r, i, int(m) - (int(self.row_start[i + 1]) - r)

    def keys(self, i, pool=None):
        """K and V of sequence i's rows, [len][kv_heads][hd] in 64 bits."""
        pool = self.pool if pool is None else pool
        m = int(self.lens[i])
        pages = self.table[i, :-(-m // self.page)]
        kv = pool[pages].astype(np.float64)
        k, v = (np.moveaxis(kv[:, w], 1, 2).reshape(-1, self.kv_heads, self.hd)[:m]
                for w in (0, 1))
        return k, v

    def attend64(self, window=0, sinks=0, bounds=True):
        """out [n][dim] (SENTINEL in rows of no sequence), and for each value a
        bound of its rounding in f32: with s = sum q k / sqrt(hd) computed to
        within d = 4 hd u sum |q k| / sqrt(hd) (each of the hd products of the
        split or f32 operands and each sum rounds by u; at most 3 hd sums), the
        exponent's argument to within 4 u (|s| + |max|) more, and the exponential
        and the sums over m keys by (m + 16) u, an output is off by at most
        (2 d + (m + 16) u) sum p |v|."""
        out = np.full((self.n, self.dim), SENTINEL, np.float64)
        tol = np.zeros((self.n, self.dim))
        mul = self.heads // self.kv_heads
        kv = {}
        for r, i, p in self.positions():
            if p < 0:
                out[r] = 0.0
                continue
            if i not in kv:
                kv[i] = self.keys(i)
            k, v = kv[i]
            t = np.arange(p + 1)
            seen = t if not window else t[(t > p - window) | (t < sinks)]
            kk, vv = k[seen], v[seen]
            q = self.q[r].astype(np.float64).reshape(self.kv_heads, mul, self.hd)
            sc = np.einsum("gmd,tgd->gmt", q, kk) / math.sqrt(self.hd)
            mx = sc.max(-1, keepdims=True)
            e = np.exp(sc - mx)
            w = e / e.sum(-1, keepdims=True)
            out[r] = np.einsum("gmt,tgd->gmd", w, vv).reshape(-1)
            if bounds:
                big = np.einsum("gmd,tgd->gmt", np.abs(q), np.abs(kk)) / math.sqrt(self.hd)
                d = (4 * self.hd * U * big + 4 * U * (np.abs(sc) + np.abs(mx))).max(-1)
                pv = np.einsum("gmt,tgd->gmd", w, np.abs(vv))
                tol[r] = ((2 * d + (len(seen) + 16) * U)[..., None] * pv).reshape(-1)
        return out, tol

    # ---- the device's side ----

    def upload(self, torch, ctx=None, theta=1e4, layers=1, layer=0, max_seqs=None, msl=None):
        """A Device of this batch; the other layers of the pool hold NaN."""
        return Device(self, torch, ctx, theta, layers, layer, max_seqs, msl)


class _Pool:
    def __init__(self, cache, shape, dtype):
        self.cache = cache
        self.__cuda_array_interface__ = {"shape": tuple(shape),
                                         "typestr": "<f4" if dtype == "f32" else "<i2",
                                         "data": (cache.device_ptr(), False), "version": 3}


class Device:
    def __init__(self, b, torch, ctx, theta, layers, layer, max_seqs, msl):
        self.b, self.torch, self.layer = b, torch, layer
        self.ctx = ctx or P.AttentionContext(b.dim, b.heads, b.kv_heads, msl or b.max_len, 1,
                                             theta)
        self.cache = P.PagedCache(self.ctx, layers, b.pages, b.page, b.dtype,
                                  max_seqs or max(1, len(b.seqs)))
        view = torch.as_tensor(_Pool(self.cache, (layers,) + b.pool.shape, b.dtype),
                               device="cuda")
        self.all_layers = view if b.dtype == "f32" else view.view(torch.bfloat16)
        self.all_layers.fill_(float("nan"))
        self.pool = self.all_layers[layer]
        self.pool.copy_(torch.from_numpy(b.pool))
        up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        self.table, self.lens, self.row_start = up(b.table), up(b.lens), up(b.row_start)
        self.q, self.k, self.v = up(b.q), up(b.k), up(b.v)
        self.out = torch.full((b.n, b.dim), SENTINEL, device="cuda")
        self.batch = P.PagedBatch(len(b.seqs), self.table.data_ptr(), b.stride,
                                  self.lens.data_ptr(), b.max_len,
                                  0 if b.decode else self.row_start.data_ptr(), b.n)
        torch.cuda.synchronize()

    def attend(self, window=0, sinks=0, out=None):
        out = self.out if out is None else out
        self.ctx.paged_attend_dev(self.cache, self.layer, self.batch, self.q.data_ptr(),
                                  out.data_ptr(), window, sinks)
        return out

    def append(self, q_norm=None, k_norm=None, eps=1e-5, q_out=None, with_q=True):
        q_out = self.out if q_out is None else q_out
        self.ctx.paged_append_dev(self.cache, self.layer, self.batch,
                                  self.q.data_ptr() if with_q else 0, self.k.data_ptr(),
                                  self.v.data_ptr(), q_out.data_ptr() if with_q else 0,
                                  q_norm.data_ptr() if q_norm is not None else 0,
                                  k_norm.data_ptr() if k_norm is not None else 0, eps)
        return q_out

    def host(self, t):
        self.ctx.sync()
        return t.float().cpu().numpy()

    def close(self):
        self.torch.cuda.synchronize()
        self.pool = self.all_layers = None
        self.ctx.close()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()


# Norm-wise bound of an attention output's error: the rounding errors of a
# score are independent, u sqrt(3 hd) |q||k| / sqrt(3 hd) of them remain, about
# 4 u for the scores of these tests (a few nats), and twice that in an output;
# 32 u leaves room for unlucky draws, and is below the 2^-18 that an operand
# split in two bf16 values instead of three would leave.
NORMWISE = 32 * U


def check_attention(got, b, window=0, sinks=0):
    want, tol = b.attend64(window, sinks)
    assert got.shape == want.shape
    rest = np.ones(b.n, bool)
    rest[:b.rows] = False
    assert np.all(got[rest] == SENTINEL), "rows of no sequence were written"
    g, w, t = got[:b.rows].astype(np.float64), want[:b.rows], tol[:b.rows]
    assert np.all(np.isfinite(g)), f"{int((~np.isfinite(g)).sum())} values are not finite"
    bad = np.abs(g - w) > t
    assert not bad.any(), (
        f"{int(bad.sum())} of {bad.size} values out of bounds, first at {np.argwhere(bad)[0]}, "
        f"largest error {np.abs(g - w).max():.3e}")
    norm = np.linalg.norm(w)
    rel = np.linalg.norm(g - w) / norm if norm else 0.0
    assert rel <= NORMWISE, f"norm-wise error {rel:.3e}"
    return rel
