"""CPU: how the attention over cache pages deals out its work (ttb_paged_rules.cuh), compiled for the host: every unit of every tile in one place of the line."""
import ctypes
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "turbotransformers_b200", "csrc")


class Split(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("block_heads", "blocks", "head_blocks", "tile_tokens", "unit_shift", "causal", "half", "pair_shift")]


class Place(ctypes.Structure):
    _fields_ = [("tile", ctypes.c_int64), ("block", ctypes.c_int), ("units", ctypes.c_int64), ("first", ctypes.c_int64)]


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged")
    src, so = d / "rules.cpp", d / "rules.so"
    src.write_text('#include "ttb_paged_rules.cuh"\nusing namespace ttb::paged;\nextern "C" {\n'
                   'int64_t floor_sum_(int64_t n, int64_t m, int64_t a, int64_t b) { return floor_sum(n, m, a, b); }\n'
                   'void split_(int heads, int kv, int rows, int parts, int unit, int causal, int pair, Split* s) { *s = split_of(heads, kv, rows, parts, unit, causal, pair); }\n'
                   'int64_t units_of_sequence_(const Split* s, int64_t past, int64_t n) { return units_of_sequence(*s, past, n); }\n'
                   'int64_t units_of_tile_(const Split* s, int64_t past, int64_t n, int64_t t) { return units_of_tile(*s, past, n, t); }\n'
                   'void place_(const Split* s, int64_t past, int64_t n, int64_t x, Place* p) { *p = place_of(*s, past, n, x); }\n'
                   'int ctas_(int64_t u, int c, int least) { return ctas_of(u, c, least); }\n'
                   'int64_t first_(int64_t u, int n, int c) { return first_unit(u, n, c); }\n}\n')
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, str(src), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    i64 = ctypes.c_int64
    lib.floor_sum_.restype, lib.floor_sum_.argtypes = i64, [i64] * 4
    lib.split_.argtypes = [ctypes.c_int] * 7 + [ctypes.POINTER(Split)]
    lib.units_of_sequence_.restype, lib.units_of_sequence_.argtypes = i64, [ctypes.POINTER(Split), i64, i64]
    lib.units_of_tile_.restype, lib.units_of_tile_.argtypes = i64, [ctypes.POINTER(Split), i64, i64, i64]
    lib.place_.argtypes = [ctypes.POINTER(Split), i64, i64, i64, ctypes.POINTER(Place)]
    lib.ctas_.argtypes = [i64, ctypes.c_int, ctypes.c_int]
    lib.first_.restype, lib.first_.argtypes = i64, [i64, ctypes.c_int, ctypes.c_int]
    return lib


def test_lattice_points_under_a_line(rules):
    rng = random.Random(0)
    for _ in range(2000):
        n, m, a, b = rng.randint(0, 40), rng.choice([1, 2, 3, 64, 128]), rng.randint(0, 300), rng.randint(0, 5000)
        assert rules.floor_sum_(n, m, a, b) == sum((a * i + b) // m for i in range(n))
    assert rules.floor_sum_(1 << 22, 128, 64, 1 << 30) == sum((64 * i + (1 << 30)) // 128 for i in range(1 << 22))


@pytest.mark.parametrize("rows,parts", [(16, 1), (128, 2), (128, 1)])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (12, 12), (32, 8), (7, 1), (40, 2), (20, 1), (300, 1), (64, 1)])
def test_a_tile_holds_whole_tokens_and_every_head_once(rules, heads, kv_heads, rows, parts):
    s = Split()
    rules.split_(heads, kv_heads, rows, parts, 128, 1, 0, s)
    group = heads // kv_heads
    assert s.tile_tokens >= 1 and s.tile_tokens % parts == 0 and s.tile_tokens // parts * s.block_heads <= rows
    taken = [(b // s.head_blocks, h) for b in range(s.blocks) for h in range(b % s.head_blocks * s.block_heads, min(group, (b % s.head_blocks + 1) * s.block_heads))]
    assert sorted(taken) == [(k, h) for k in range(kv_heads) for h in range(group)]
    assert all(b % s.head_blocks * s.block_heads < group for b in range(s.blocks))


@pytest.mark.parametrize("pair", [0, 1])
@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("heads,kv_heads,rows,parts,unit", [(12, 12, 16, 1, 128), (32, 8, 16, 1, 128), (7, 1, 128, 2, 128), (6, 2, 128, 2, 64), (40, 1, 16, 1, 128)])
def test_every_unit_has_its_place(rules, heads, kv_heads, rows, parts, unit, causal, pair):
    s, p, rng = Split(), Place(), random.Random(heads * rows + causal)
    rules.split_(heads, kv_heads, rows, parts, unit, causal, pair, s)
    for past, n in [(0, 0), (0, 1), (unit - 1, 1), (unit, 1), (0, unit + 1), (1000, 3)] + [(rng.randint(0, 700), rng.randint(1, 400)) for _ in range(12)]:
        tiles = -(-n // s.tile_tokens)
        line = []
        for t in range(tiles):
            keys = past + (min(n, (t + 1) * s.tile_tokens) if causal else n)
            units = -(-keys // unit)
            if parts == 2 and n - t * s.tile_tokens <= s.tile_tokens // 2:  # one set's rows: both sets take its units in turn
                units = -(-units // (1 + pair))
            assert rules.units_of_tile_(s, past, n, t) == units
            line += [(t, b, units, u) for b in range(s.blocks) for u in range(units)]
        assert rules.units_of_sequence_(s, past, n) == len(line)
        for x in range(len(line)) if len(line) < 400 else [0, 1, len(line) - 1] + [rng.randrange(len(line)) for _ in range(300)]:
            rules.place_(s, past, n, x, p)
            assert (p.tile, p.block, p.units, p.first) == line[x]


def test_stretches_cover_the_line(rules):
    for units in (0, 1, 5, 147, 148, 149, 1000, 1 << 40):
        for grid in (1, 2, 148, 160):
            n = rules.ctas_(units, grid, 1)
            assert n <= grid and (n > 0) == (units > 0) and n <= units
            edges = [rules.first_(units, n, c) for c in range(n + 1)] if n else [0]
            assert edges[0] == 0 and edges[-1] == units and all(a < b for a, b in zip(edges, edges[1:]))


class Sequences(ctypes.Structure):
    _fields_ = [("table", ctypes.c_void_p), ("table_stride", ctypes.c_longlong), ("cu", ctypes.c_void_p), ("past", ctypes.c_void_p)] + \
               [(n, ctypes.c_int) for n in ("B", "tokens", "pages", "page_shift", "cap")] + [("status", ctypes.c_void_p)]


@pytest.fixture(scope="module")
def views(tmp_path_factory):
    d = tmp_path_factory.mktemp("views")
    src, so = d / "views.cpp", d / "views.so"
    src.write_text('#include "ttb_paged_rules.cuh"\nusing namespace ttb::paged;\nextern "C" {\n'
                   'int sequence_(const Sequences* s, int b, int* out) { bool bad; const Sequence q = sequence_of(*s, b, &bad);'
                   ' out[0] = q.tok0; out[1] = q.n; out[2] = q.past; return bad; }\n'
                   'int page_(const Sequences* s, int b, int at, int* page) { bool bad; *page = page_of(*s, b, at, &bad); return bad; }\n}\n')
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, str(src), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    lib.sequence_.argtypes = [ctypes.POINTER(Sequences), ctypes.c_int, ctypes.c_void_p]
    lib.page_.argtypes = [ctypes.POINTER(Sequences), ctypes.c_int, ctypes.c_int, ctypes.c_void_p]
    return lib


def test_what_does_not_fit_a_call_is_cut_and_reported(views):
    """Offsets outside the rows, negative lengths, more tokens than the table lists, pages outside the pool: nothing that is used is outside."""
    top, low = 2**31 - 1, -2**31
    cases = [((0, 3), 5, (0, 3, 5), 0), ((3, 3), 5, (3, 0, 5), 0), ((0, 10), 54, (0, 10, 54), 0), ((0, 10), 55, (0, 10, 55), 1), ((0, 11), 5, (0, 0, 5), 1),
             ((-1, 3), 5, (0, 0, 5), 1), ((4, 3), 5, (0, 0, 5), 1), ((0, 3), -1, (0, 3, 0), 1), ((0, 3), top, (0, 3, 64), 1), ((0, 3), low, (0, 3, 0), 1),
             ((low, top), 0, (0, 0, 0), 1), ((top, low), 64, (0, 0, 64), 1)]
    for (cu0, cu1), past, want, bad in cases:
        cu, pa, out = (ctypes.c_int * 2)(cu0, cu1), (ctypes.c_int * 1)(past), (ctypes.c_int * 3)()
        s = Sequences(None, 4, ctypes.addressof(cu), ctypes.addressof(pa), 1, 10, 7, 4, 64, None)
        assert views.sequence_(s, 0, out) == bad and tuple(out) == want
    table, page = (ctypes.c_int * 4)(6, -1, 7, top), ctypes.c_int()
    s = Sequences(ctypes.addressof(table), 4, None, None, 1, 10, 7, 4, 64, None)
    assert [views.page_(s, 0, at, ctypes.byref(page)) for at in (0, 15, 16, 32, 63)] == [0, 0, 1, 1, 1]
