"""Every address of the kernels of 4-bit products and of the router's losses, checked on the CPU as in test_emulated.py:
buffers of exactly their sizes, group sizes around the edges of every row tile, every tiling, offsets of any values."""
import random
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from tests import emu
from tests.test_emulated import ENV, SIZES, pytestmark, run  # noqa: F401

TILES = {"rule": -1, "few rows": -2, "256": 0, "128": 1, "64": 2}


@pytest.fixture(scope="module")
def programs(tmp_path_factory):
    to = {name: tmp_path_factory.mktemp(name) / "build" for name in ("mx", "router")}
    with ThreadPoolExecutor(2) as pool:
        return dict(zip(to, pool.map(emu.build, to.values(), to)))


def text(*values):
    return " ".join(map(str, values))


@pytest.mark.parametrize("tiles", TILES)
def test_grouped_products(tiles, programs):
    r = random.Random(tiles)
    lines = []
    for i, sizes in enumerate(SIZES):
        for four in (0, 1):
            K, N = r.choice(((160, 328), (96, 520), (288, 8), (544, 136), (32, 264), (1056, 40)))
            lines.append(text("linear", f"grouped{i}{four}", four, int(not four or i % 2), i % 5, i % 2, i // 2 % 2, 1, TILES[tiles], K, N,
                              r.choice((0, 5, 70)), *sizes))
    run(programs["mx"], lines)


def test_dense_products(programs):
    lines = []
    for i, (M, K, N) in enumerate([(1, 256, 48), (17, 64, 520), (64, 160, 24), (65, 96, 264), (385, 288, 136), (700, 32, 1032),
                                   (1153, 544, 8), (3, 32, 8), (500, 32, 8), (15, 1568, 8)]):
        for four in (0, 1):
            lines += [text("linear", f"dense{i}{four}t{t}", four, int(not four or t % 2), i % 5, i % 2, t % 2, 0, t, K, N, 0, M)
                      for t in (-2, -1, 0, 1, 2)]
    run(programs["mx"], lines)


def test_drawn_products(programs):
    r = random.Random(6)
    edges = [0, 0, 1, 2, 31, 33] + [b + d for b in range(64, 577, 64) for d in (-1, 0, 1)]
    widths = [8, 16, 24, 40, 72, 120, 128, 136, 200, 256, 264, 392, 520]
    lines = []
    for i in range(80):
        four, grouped, few = int(r.random() < 0.5), int(r.random() < 0.8), r.random() < 0.4
        sizes = [r.randint(0, 20) if few else r.choice(edges) for _ in range(r.choice((1, 2, 3, 5, 70)) if few else r.choice((1, 2, 3, 4)))]
        sizes = sizes if grouped else sizes[:1]
        sizes[0] += not sum(sizes)
        lines.append(text("linear", f"drawn{i}", four, int(not four or r.random() < 0.5), r.randrange(5), r.randint(0, 1), r.randint(0, 1),
                          grouped, r.choice((-1, -1, -2, 0, 1, 2)), 32 * r.choice((1, 2, 3, 5, 8, 15, 16, 17, 33)), r.choice(widths),
                          r.choice((0, 1, 5, 64, 300)) if grouped else 0, *sizes))
    run(programs["mx"], lines)


def test_ranges_of_experts_and_offsets_that_are_none(programs):
    r = random.Random(10)
    lines = []
    for i in range(40):
        M, E = r.choice((7, 40, 300, 600)), r.choice((1, 2, 5, 40, 130))
        top = r.choice((M, M, M // 2, 3 * M, 2 ** 31 - 1))
        offsets = [r.randint(-5 if i % 3 else 0, top) for _ in range(E + 1)]
        if i % 2:
            offsets = sorted(min(max(o, 0), M) for o in offsets)
        lines.append(text("linear", f"?offsets{i}", i // 2 % 2, 1, i % 5, 1, i % 3 % 2, 1, r.choice((-1, -2, 0, 1, 2)),
                          r.choice((32, 160)), r.choice((40, 264)), M, *offsets))
    run(programs["mx"], lines)


def test_quantisation(programs):
    run(programs["mx"], [text("quant", f"q{d}{n}", d, n) for d in (0, 1) for n in (1, 2, 3, 15, 16, 17, 63, 64, 65, 1000)])


def test_router(programs):
    lines = []
    for i, E in enumerate((1, 3, 4, 12, 16, 17, 20, 32, 33, 64, 68, 96, 100, 128, 160, 164, 256, 257, 260, 512, 516, 700, 1000, 1023, 1024)):
        T = (1, 7, 40, 130)[i % 4]
        lines.append(text(f"one{i}", i % 2, 4 + 4 * (i // 2 % 2), i // 3 % 2, T, E, (1, 2, 7, 16)[i % 4], 0))
        lines.append(text(f"seq{i}", 1 - i % 2, 4, i % 2, T, E, 3, (1, 2, 9, 50)[i // 2 % 4]))
    lines += [text("none", 0, 4, 0, 0, 8, 2, 0), text("none2", 0, 4, 0, 0, 8, 2, 3), text("many", 1, 4, 1, 900, 16, 2, 400),
              text("long", 0, 8, 0, 9000, 8, 1, 3), text("gaps", 0, 4, 1, 300, 64, 4, 4, 17, 17, 90, 90, 255)]
    r = random.Random(3)
    for i in range(24):
        T, S = r.choice((5, 60, 300)), r.choice((1, 3, 20))
        offsets = [r.randint(-9, r.choice((T, 3 * T, 2 ** 31 - 1))) for _ in range(S + 1)]
        lines.append(text(f"offsets{i}", i % 2, 4, i // 2 % 2, T, r.choice((12, 33, 64)), 2, S, *offsets))
    run(programs["router"], lines)


@pytest.mark.parametrize("program,line", [("mx", "linear !short 0 1 0 0 0 1 0 160 328 0 130 257"), ("mx", "linear !s 1 1 0 0 0 1 1 160 328 0 130 257"),
                                          ("mx", "linear /scale 1 1 0 0 0 1 -2 544 328 0 13 25"), ("mx", "linear /scale 0 1 0 0 0 1 2 160 328 0 65 64"),
                                          ("router", "!short 0 4 0 65 33 2 0")])
def test_an_access_outside_a_buffer_is_seen(program, line, programs):
    r = subprocess.run([programs[program]], input=line + "\n", env=ENV, capture_output=True, text=True, timeout=300)
    assert r.returncode != 0 and ("out of bounds" in r.stdout or "AddressSanitizer" in r.stderr), (r.stdout[-500:], r.stderr[-500:])
