"""Index arithmetic of the paged cache (csrc/paged_index.h), compiled for the
host: rows, visible keys and addresses against plain restatements, and every
index inside its array whatever the batch's arrays hold."""
import subprocess

import numpy as np
import pytest

from slm_testlib import load_product

P = load_product()

PROBE = r"""
#include <stdio.h>
#include <stdlib.h>
#include <vector>
#include "paged_index.h"
static long rd() { long x; if (scanf("%ld", &x) != 1) exit(3); return x; }
static void check(bool ok, const char* what) { if (!ok) { printf("%s\n", what); exit(1); } }
int main(void) {
    long cases = rd();
    while (cases--) {
        slm::PagedView b{};
        b.n_seqs = rd(), b.n_rows = rd(), b.max_len = rd(), b.stride = rd();
        b.num_pages = rd(), b.ps_shift = rd(), b.kv_heads = rd();
        const int hd = rd(), window = rd(), sinks = rd();
        // arrays of the exact size, so that an access behind them shows under ASan
        std::vector<int32_t> table((size_t)b.n_seqs * b.stride), lens(b.n_seqs), start(b.n_seqs + 1);
        for (auto& x : table) x = rd();
        for (auto& x : lens) x = rd();
        for (auto& x : start) x = rd();
        b.table = table.data(), b.lens = lens.data(), b.row_start = start.data();
        const size_t values = ((size_t)b.num_pages * 2 * b.kv_heads << b.ps_shift) * hd;
        for (int row = 0; row < b.n_rows; ++row) {
            const slm::PagedRow r = slm::paged_row(b, row);
            printf("%d %d %d", r.seq, r.pos, (int)r.bad);
            check(r.seq >= -1 && r.seq < b.n_seqs, "seq");
            check(r.pos < b.max_len, "pos");
            const slm::Visible vis(r.pos, window, sinks);
            check(vis.count >= 0 && vis.count <= b.max_len, "count");
            long sum = 0;
            for (int u = 0; u < vis.count; ++u) {
                const int t = vis.row(u);
                check(t >= 0 && t <= r.pos, "row");
                check(u == 0 || t > vis.row(u - 1), "rows ascend");
                const size_t e = (size_t)r.seq * b.stride + (t >> b.ps_shift);
                check(e < table.size(), "table");
                const int page = table[e];
                if (!slm::paged_page_ok(b, page)) continue;
                const size_t at = slm::paged_at(b, page, 1, b.kv_heads - 1,
                                                t & ((1 << b.ps_shift) - 1), hd);
                check(at + hd <= values, "values");
                sum += t + 1;
            }
            printf(" %d %ld\n", vis.count, sum);
        }
    }
    return 0;
}
"""


@pytest.fixture(scope="module")
def probe(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged")
    src = d / "probe.cpp"
    src.write_text(PROBE)
    exe = d / "probe"
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-Wall", "-Werror", "-fsanitize=address",
                    f"-I{P.PKG_DIR / 'csrc'}", str(src), "-o", str(exe)], check=True)

    def run(cases):
        words = [len(cases)]
        for c in cases:
            words += c["head"] + c["table"] + c["lens"] + c["start"]
        r = subprocess.run([str(exe)], input=" ".join(map(str, words)), capture_output=True,
                           text=True)
        assert r.returncode == 0, (r.stdout[-200:], r.stderr[-2000:])
        return [[int(x) for x in ln.split()] for ln in r.stdout.splitlines()]

    return run


def case(rng, sane):
    n_seqs, page_shift = int(rng.integers(1, 9)), int(rng.integers(4, 7))
    stride, pages = int(rng.integers(1, 5)), int(rng.integers(1, 9))
    max_len = int(rng.integers(1, (stride << page_shift) + 1))
    counts = rng.integers(0, 6, n_seqs)
    start = np.concatenate([[0], np.cumsum(counts)])
    n_rows = max(1, int(start[-1]) + int(rng.integers(0, 3)))
    lens = rng.integers(0, max_len + 1, n_seqs)
    table = rng.integers(0, pages, n_seqs * stride)
    if not sane:
        wild = np.array([-1, -2**31, 2**31 - 1, 1 << 30, max_len + 1, n_rows + 1, pages])
        for a in (lens, table, start):
            hit = rng.random(len(a)) < 0.5
            a[hit] = rng.choice(wild, hit.sum())
    window = int(rng.choice([0, 0, 1, 5, 20, 2**31 - 1]))
    sinks = int(rng.choice([0, 1, 7, 2**31 - 1]))
    return {"head": [n_seqs, n_rows, max_len, stride, pages, page_shift, 3, 16, window, sinks],
            "table": table.tolist(), "lens": lens.tolist(), "start": start.tolist(),
            "n_rows": n_rows, "window": window, "sinks": sinks}


def test_rows_and_visible_keys(probe):
    rng = np.random.default_rng(1)
    cases = [case(rng, True) for _ in range(200)]
    got = iter(probe(cases))
    for c in cases:
        for row in range(c["n_rows"]):
            seq, pos = -1, -1
            for i, m in enumerate(c["lens"]):
                if c["start"][i] <= row < c["start"][i + 1]:
                    seq, pos = i, m - (c["start"][i + 1] - row)
            seen = [t for t in range(pos + 1)
                    if not c["window"] or t > pos - c["window"] or t < c["sinks"]]
            assert next(got) == [seq, pos, 0, len(seen), sum(seen) + len(seen)]


def test_nonsense_stays_inside(probe):
    rng = np.random.default_rng(2)
    cases = [case(rng, False) for _ in range(400)]
    assert len(probe(cases)) == sum(c["n_rows"] for c in cases)
