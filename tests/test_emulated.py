"""Every address of the operators' kernels, and of the GEMM core's under them, checked on the CPU: the C
entries run on an emulated device (tests/emu) under AddressSanitizer, with buffers of exactly their sizes.
Group sizes lie around the edges of every row tile, for every tiling, whether the launch rule would take it
for that shape or not."""
import os
import random
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from tests import emu

ENV = dict(os.environ, ASAN_OPTIONS="detect_leaks=0:detect_stack_use_after_return=0")
TILES = {"rule": -1, "256": 0, "384": 1, "128": 2, "64": 3, "256 group by group": 4}

pytestmark = pytest.mark.skipif(not os.path.exists(emu.CLANG), reason="needs ROCm's clang++")


@pytest.fixture(scope="module")
def programs(tmp_path_factory):
    to = {name: tmp_path_factory.mktemp(name) / "build" for name in ("linear", "rows")}
    with ThreadPoolExecutor(2) as pool:
        return dict(zip(to, pool.map(emu.build, to.values(), to)))


def run(program, lines):
    """Runs the calls over four processes."""
    def part(i):
        mine = lines[i::4]
        r = subprocess.run([program], input="\n".join(mine) + "\n", env=ENV, capture_output=True, text=True, timeout=600)
        assert r.returncode == 0 and r.stdout.count("ok ") == len(mine), (r.stdout[-800:], r.stderr[-3000:])
    with ThreadPoolExecutor(4) as pool:
        list(pool.map(part, range(4)))


# row counts at the edges of 64- to 384-row tiles and of their tails, in a few groups with and without rows
SIZES = ([0, 1, 64, 65, 0], [319, 320, 321, 0], [383, 384, 385], [256, 257, 576, 577], [705, 640, 513, 3], [63, 127, 129, 193],
         [2, 0, 0, 1], [1153])


@pytest.mark.parametrize("tiles", TILES)
def test_grouped_products(tiles, programs):
    r = random.Random(tiles)
    lines = []
    for i, sizes in enumerate(SIZES):
        K, N = r.choice(((136, 328), (24, 520), (264, 8), (200, 136), (8, 264)))
        lines.append(f"grouped{i} {int(tiles != 'rule' or i % 2)} {i % 5} {i % 2} {i % 3 % 2} 1 {TILES[tiles]} {K} {N} "
                     f"{r.choice((0, 5, 70))} " + " ".join(map(str, sizes)))
    run(programs["linear"], lines)


def test_dense_products(programs):
    lines = []
    for i, (M, K, N) in enumerate([(1, 256, 48), (17, 64, 520), (64, 136, 24), (65, 136, 264), (385, 264, 136), (700, 8, 1032),
                                   (1153, 200, 8)]):
        for dtype in (0, 1):
            lines.append(f"dense{i} {dtype} {i % 5} 1 {i % 2} 0 -1 {K} {N} 0 {M}")
        lines += [f"dense{i}t{t} 1 {i % 5} 0 {i % 2} 0 {t} {K} {N} 0 {M}" for t in range(4)]
    run(programs["linear"], lines)


def test_drawn_products(programs):
    r = random.Random(5)
    edges = [0, 0, 1, 2, 31, 33] + [b + d for b in range(64, 833, 64) for d in (-1, 0, 1)]
    widths = [8, 16, 24, 40, 64, 72, 120, 128, 136, 200, 248, 256, 264, 320, 384, 392, 520]
    lines = []
    for i in range(160):
        dtype, grouped = int(r.random() < 0.8), int(r.random() < 0.8)
        few = r.random() < 0.3
        sizes = [r.randint(0, 20) if few else r.choice(edges) for _ in range(r.choice((1, 2, 3, 5, 8, 12)) if grouped else 1)]
        sizes[0] += not sum(sizes)
        lines.append(f"drawn{i} {dtype} {r.randrange(5)} {r.randint(0, 1)} {r.randint(0, 1)} {grouped} "
                     f"{r.choice((-1, -1, 0, 1, 2, 3, 4)) if dtype else -1} {r.choice(widths)} {r.choice(widths)} "
                     f"{r.choice((0, 1, 5, 64, 300)) if grouped else 0} " + " ".join(map(str, sizes)))
    run(programs["linear"], lines)


def test_ranges_of_experts_and_offsets_that_are_none(programs):
    # a range of a longer array, whose other rows are no group's; and offsets of any values, which may leave rows
    # undefined but no buffer
    r = random.Random(9)
    lines = []
    for i in range(40):
        M, E = r.choice((7, 40, 300, 600)), r.choice((1, 2, 5, 40, 130))
        top = r.choice((M, M, M // 2, 3 * M, 2 ** 31 - 1))
        offsets = [r.randint(-5 if i % 3 else 0, top) for _ in range(E + 1)]
        if i % 2:
            offsets = sorted(min(max(o, 0), M) for o in offsets)
        lines.append(f"?offsets{i} {i % 4 > 0:d} {i % 5} 1 {i % 2} 1 {r.choice((-1, -1, 0, 1, 2, 3, 4)) if i % 4 else -1} "
                     f"{r.choice((24, 136))} {r.choice((40, 264))} {M} " + " ".join(map(str, offsets)))
    run(programs["linear"], lines)


def test_sorting_rows_and_norms(programs):
    lines = ["sort a 4 1 1 1 0", "sort b 8 300 5 33 4", "sort c 4 5000 6 64 9", "sort d 4 40 16 1024 3", "sort e 8 0 2 3 0",
             "rows f 0 33 3 12 520 5", "rows g 1 64 8 16 4096 0", "rows h 1 7 16 8 64 2", "rows i 1 5 2 7 1032 0",
             "rows s 0 40 3 8 64 -1", "rows t 1 40 8 8 520 -2", "rows u 1 9 16 8 1032 -3",
             "norm j 1 1 8 0 1 1 0", "norm k 0 33 520 1 1 1 1", "norm l 1 66 2048 2 1 0 0", "norm m 1 9 7168 3 0 1 0",
             "norm n 0 5 8200 1 1 1 0", "norm o 1 3 16392 1 1 1 0", "norm p 0 300 1032 0 0 1 0", "norm q 0 130 64 2 0 0 1",
             "norm r 1 70 520 3 1 1 0"]
    run(programs["rows"], lines)


def test_an_access_outside_a_buffer_is_seen(programs):
    r = subprocess.run([programs["linear"]], input="!short 1 0 0 0 1 2 136 328 0 130 257\n", env=ENV, capture_output=True,
                       text=True, timeout=300)
    assert r.returncode != 0 and "out of bounds" in r.stdout, r.stdout[-500:]
