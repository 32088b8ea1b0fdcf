"""The line of work of the paged attention (csrc/qd_paged_line.h) with the terms that shared beginnings and pages of 8
bits bring: blocks that other rows of work cover (jb), a fixed cost of few-row units (few_cost), and layouts all of
whose units are of tiles (tpf = 0), compiled for the host, against the same counts in Python's whole numbers."""

import ctypes
import os
import random
import subprocess

import pytest

from conftest import PKG_ROOT

DRIVER = r"""
#include "qd_paged_line.h"
using namespace qd;
static PgShape shape(int nq, int nkv, int few_cost, int no_few) {
  PgShape s = pg_shape(nq, nkv);
  s.few_cost = few_cost;
  if (no_few) s.tpf = 0;
  return s;
}
// rows of work as five numbers each: first token row, tokens, first position, keys, blocks before the first
static PgReq work(const PgShape& s, const int* w) {
  PgReq r;
  r.row0 = w[0]; r.n = w[1]; r.pos0 = w[2]; r.kv = w[3]; r.jb = w[4];
  r.pairs = (r.n + 2 * s.tpt - 1) / (2 * s.tpt);
  return r;
}
extern "C" {
void places(int nq, int nkv, int few_cost, int no_few, int n, const int* w, long long* out) {
  const PgShape s = shape(nq, nkv, few_cost, no_few);
  for (int i = 0; i < n; ++i) out[i] = nkv * pg_sum_cost(s, work(s, w + 5 * i));
}
// where place `at` of the i-th is: pair, head, place of the unit
void place(int nq, int nkv, int few_cost, int no_few, const int* w, long long at, int* out) {
  const PgShape s = shape(nq, nkv, few_cost, no_few);
  const PgPlace p = pg_place(s, work(s, w), at, false);
  out[0] = p.k; out[1] = p.h; out[2] = p.o;
}
}
"""


@pytest.fixture(scope="module")
def line(tmp_path_factory):
    d = tmp_path_factory.mktemp("terms")
    src, so = d / "terms.cpp", d / "libterms.so"
    src.write_text(DRIVER)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=undefined", "-static-libubsan",
                    "-shared", "-fPIC", "-I", os.path.join(PKG_ROOT, "csrc"), str(src), "-o", str(so)], check=True)
    return ctypes.CDLL(str(so))


def _units(nq, nkv, few_cost, no_few, n, pos0, kv, jb):
    """Places of each pair of tiles, by the definition."""
    group = nq // nkv
    tpt, tpf = 128 // group, 0 if no_few else 16 // group
    costs = []
    for t in range(0, n, 2 * tpt):
        tok, keys = n - t, min(kv, pos0 + min(n, t + 2 * tpt))
        blocks = max(-(-keys // 128) - jb, 1)
        costs.append((5 if tok > tpt else 4 if tok > tpf else 2) * blocks + (8 if tok > tpf else few_cost))
    return costs


def _check(line, rng, nq, nkv, few_cost, no_few, rows):
    flat = (ctypes.c_int * (5 * len(rows)))(*(x for r in rows for x in r))
    got = (ctypes.c_longlong * len(rows))()
    line.places(nq, nkv, few_cost, no_few, len(rows), flat, got)
    for i, (_, n, pos0, kv, jb) in enumerate(rows):
        costs = _units(nq, nkv, few_cost, no_few, n, pos0, kv, jb)
        assert got[i] == nkv * sum(costs), (nq, nkv, rows[i], got[i], nkv * sum(costs))
        if not costs:
            continue
        out, one = (ctypes.c_int * 3)(), (ctypes.c_int * 5)(*rows[i])
        for at in {0, got[i] - 1, rng.randrange(got[i]), rng.randrange(got[i])}:
            line.place(nq, nkv, few_cost, no_few, one, ctypes.c_longlong(at), out)
            k, h, o = out
            assert 0 <= h < nkv and 0 <= o < costs[k] and nkv * sum(costs[:k]) + h * costs[k] + o == at, (rows[i], at, list(out))


LAYOUTS = [1, 2, 3, 4, 7, 16, 17, 33, 71, 128]


def test_rows_of_work_over_a_requests_own_keys(line):
    """A request's own keys begin `jb` blocks on, all of which are before its first new token."""
    rng = random.Random(8)
    for _ in range(1500):
        nkv = rng.choice([1, 2, 3, 8])
        rows = []
        for _ in range(rng.randint(1, 6)):
            n, pos0 = rng.choice([0, 1, 1, 2, 5, rng.randint(1, 700)]), rng.randint(0, 6000)
            kv = pos0 + n if rng.random() < 0.8 else rng.randint(0, pos0 + n)  # (cut to its table row)
            rows.append((0, n, pos0, kv, rng.choice([0, pos0 // 128, rng.randint(0, pos0 // 128)])))
        _check(line, rng, nkv * rng.choice(LAYOUTS), nkv, rng.choice([0, 3]), 0, rows)


def test_rows_of_work_over_common_keys(line):
    """A group's tokens over its common blocks: every token sees all of them, so no sum grows with the pairs."""
    rng = random.Random(9)
    for _ in range(1500):
        nkv = rng.choice([1, 2, 3, 8])
        rows = []
        for _ in range(rng.randint(1, 6)):
            blocks = rng.randint(1, 300)
            rows.append((rng.randint(0, 99), rng.choice([2, 3, 16, rng.randint(2, 900)]), blocks * 128 - 1, blocks * 128, 0))
        _check(line, rng, nkv * rng.choice(LAYOUTS), nkv, 3, 0, rows)


def test_units_of_tiles_alone(line):
    rng = random.Random(10)
    for _ in range(1500):
        nkv = rng.choice([1, 2, 3, 8])
        rows = []
        for _ in range(rng.randint(1, 6)):
            n, before = rng.choice([0, 1, 2, 17, rng.randint(1, 700)]), rng.randint(-3, 6000)
            rows.append((0, n, before, rng.choice([before + n, max(before + n - 200, 0)]) if before >= 0 else max(before + n, 0), 0))
        _check(line, rng, nkv * rng.choice(LAYOUTS), nkv, 0, 1, rows)


@pytest.mark.parametrize("group", [4, 71])
def test_rows_of_work_past_32_bits(line, group):
    rng = random.Random(11)
    rows = [(0, 470_000, 1_000_000, 1_470_000, 7000), (0, 900_000, 0, 900_000, 0), (0, 30_000, 0x7fffff00 - 30_000 - 1, 0x7fffff00 - 30_000, 0),
            (0, 1, 0x7ffffe00, 0x7ffffe01, 0x7ffffe00 // 128)]
    _check(line, rng, 8 * group, 8, 3, 0, rows)
    _check(line, rng, 8 * group, 8, 0, 1, rows)
