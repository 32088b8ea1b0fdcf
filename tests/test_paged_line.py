"""The line of work of the paged attention (csrc/qd_paged_line.h), compiled for the host: the sums of places, the
place that each CTA starts from and the owners of places, against the same counts in Python's whole numbers, up to
calls that would take the GPU seconds to minutes."""

import ctypes
import os
import random
import subprocess

import pytest

from conftest import PKG_ROOT

DRIVER = r"""
#include "qd_paged_line.h"
using namespace qd;
extern "C" {
// places of every request
void places(int nq, int nkv, int n, const int* cu, const int* kv, int tokens, int room, long long* out) {
  const PgShape s = pg_shape(nq, nkv);
  for (int i = 0; i < n; ++i) out[i] = nkv * pg_sum_cost(s, pg_make_request(s, cu[i], cu[i + 1], kv[i], tokens, room));
}
// CTA c's places, and where the first of them is in request r: request, pair, head, place of the unit
int start(int nq, int nkv, int n, const int* cu, const int* kv, int tokens, int room, long long total, int grid,
          int least, int c, long long* from, long long* to, int* at) {
  const PgShape s = pg_shape(nq, nkv);
  const PgLine line = pg_line(total, grid, least);
  if (c >= line.ctas) return 0;
  *from = line.begin(c);
  *to = line.begin(c + 1);
  int64_t before = 0;
  for (int i = 0; i < n; ++i) {
    const PgReq r = pg_make_request(s, cu[i], cu[i + 1], kv[i], tokens, room);
    const int64_t mine = nkv * pg_sum_cost(s, r);
    if (*from >= before && *from < before + mine) {
      const PgPlace p = pg_place(s, r, *from - before, false);
      at[0] = i; at[1] = p.k; at[2] = p.h; at[3] = p.o;
      return 1;
    }
    before += mine;
  }
  return -1;
}
int owner(long long total, int grid, int least, long long at) { return pg_line(total, grid, least).owner(at); }
}
"""
ROOM = 0x7fffff00


@pytest.fixture(scope="module")
def line(tmp_path_factory):
    d = tmp_path_factory.mktemp("line")
    src, so = d / "line.cpp", d / "libline.so"
    src.write_text(DRIVER)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=undefined", "-static-libubsan",
                    "-shared", "-fPIC", "-I", os.path.join(PKG_ROOT, "csrc"), str(src), "-o", str(so)], check=True)
    return ctypes.CDLL(str(so))


def _unit_costs(nq, nkv, n, kv, room):
    """(pairs, cost of each) of a request in runs of equal costs: [(count, cost)], by the definition."""
    group = nq // nkv
    tpt, tpf = 128 // group, 16 // group
    runs = []
    for t in range(0, n, 2 * tpt):
        tok, keys = n - t, min(kv, room, kv - n + min(n, t + 2 * tpt))
        blocks = max(-(-keys // 128), 1)
        runs.append((5 if tok > tpt else 4 if tok > tpf else 2) * blocks + (8 if tok > tpf else 0))
    return runs


def _ints(v):
    return (ctypes.c_int * len(v))(*v)


def _check(line, nq, nkv, spec, room=ROOM, grid=148, least=12):
    cu, kv = [0], [k for _, k in spec]
    for n, _ in spec:
        cu.append(cu[-1] + n)
    costs = [_unit_costs(nq, nkv, n, k, room) for n, k in spec]
    want = [nkv * sum(c) for c in costs]
    got = (ctypes.c_longlong * len(spec))()
    args = (nq, nkv, len(spec), _ints(cu), _ints(kv), cu[-1], room)
    line.places(*args, got)
    assert list(got) == want, (spec[:4], list(got)[:4], want[:4])
    total = sum(want)
    a, b, at = ctypes.c_longlong(), ctypes.c_longlong(), (ctypes.c_int * 4)()
    last, ctas = 0, max(total // least, min(total, 1))
    for c in range(grid):
        found = line.start(*args, ctypes.c_longlong(total), grid, least, c, ctypes.byref(a), ctypes.byref(b), at)
        if c >= ctas:
            assert found == 0
            continue
        assert found == 1 and a.value == last and b.value > a.value, (c, found, a.value, b.value)
        last = b.value
        i, k, h, o = at
        place = sum(want[:i]) + nkv * sum(costs[i][:k]) + h * costs[i][k] + o
        assert 0 <= h < nkv and 0 <= o < costs[i][k] and place == a.value, (c, list(at))
        for x in (a.value, (a.value + b.value) // 2, b.value - 1):
            assert line.owner(ctypes.c_longlong(total), grid, least, ctypes.c_longlong(x)) == c
    assert last == total
    return total


def test_lines_of_ordinary_calls(line):
    rng = random.Random(3)
    for _ in range(60):
        nkv = rng.choice([1, 2, 3, 8])
        nq = nkv * rng.choice([1, 2, 3, 4, 7, 16, 17, 71, 128])
        spec = []
        for _ in range(rng.randint(1, 40)):
            n = rng.choice([0, 1, 1, 1, rng.randint(1, 300)])
            spec.append((n, max(0, n + rng.choice([0, -3, rng.randint(0, 2000)]))))
        _check(line, nq, nkv, spec, room=rng.choice([ROOM, 1024]), grid=rng.choice([1, 5, 148]), least=rng.choice([2, 12]))


@pytest.mark.parametrize("nq,nkv,spec", [
    (32, 8, [(938_000, 938_000)]), (32, 8, [(469_000, 469_000)] * 4), (32, 8, [(240_000, 240_000)] * 16),
    (71, 1, [(470_000, 470_000)]), (128, 8, [(470_000, 470_000)]), (64, 8, [(3, 90), (700_000, 700_000), (1, 5)]),
    (32, 8, [(200_000, 2_000_000_000), (1, 7)]), (32, 8, [(1, 0x7fffffff), (40, 0x7fffffff)]), (8, 8, [(1_000_000, 3_000_000), (5, 5)])])
def test_lines_past_32_bits(line, nq, nkv, spec):
    """Counts that pass 2^31 in a request or over all of them, and lengths at the end of 32 bits."""
    assert _check(line, nq, nkv, spec) > 2 ** 27
