"""The waits of the direct-to-LDS pipelines on the emulated device: a direct load stays in flight until its wave waits for
it, and what it writes is touched by no thread before, neither by a main loop's reads nor by the epilogue that reuses the
LDS. Row counts and depths around one, two and more k-tiles of every tiling."""
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from tests import emu
from tests.test_emulated import ENV, pytestmark, run  # noqa: F401


@pytest.fixture(scope="module")
def programs(tmp_path_factory):
    to = {name: tmp_path_factory.mktemp(name + "_waits") / "build" for name in ("mx", "linear")}
    with ThreadPoolExecutor(2) as pool:
        return dict(zip(to, pool.map(lambda t, name: emu.build(t, name, waits=True), to.values(), to)))


# bf16 rows have k-tiles of 64, 4-bit rows of 256; the loops are two to four k-tiles deep
@pytest.mark.parametrize("tiles", (0, 1, 2))
@pytest.mark.parametrize("four", (0, 1))
def test_products_over_four_bits(four, tiles, programs):
    lines = []
    for i, (M, K, N) in enumerate([(257, 32, 264), (130, 96, 136), (65, 160, 72), (200, 544, 264), (300, 1056, 136)]):
        lines.append(f"linear dense{i} {four} 1 {i % 3} 1 {i % 2} 0 {tiles} {K} {N} 0 {M}")
    lines.append(f"linear grouped {four} 1 1 1 1 1 {tiles} 544 264 5 0 1 63 130 200 257")
    run(programs["mx"], lines)


@pytest.mark.parametrize("dtype", (0, 1))
def test_products(dtype, programs):
    lines = [f"dense{i}t{t} {dtype} {i % 5} 1 {i % 2} 0 {t} {K} {N} 0 {M}"
             for i, (M, K, N) in enumerate([(200, 40, 264), (300, 136, 136), (400, 328, 264)]) for t in ((0, 1, 2, 3) if dtype else (-1,))]
    lines.append(f"grouped {dtype} 1 1 1 1 -1 136 264 5 0 1 63 130 257 385")
    run(programs["linear"], lines)


def test_a_read_of_what_is_in_flight_is_seen(tmp_path):
    # the oracle's own check: a program that waits for one load too few
    src = tmp_path / "short.cpp"
    src.write_text("""
#include "hip/hip_runtime.h"
void kernel(const char* from, int left, float* out) {
  __shared__ float tile[2][256];
  const emu::Rsrc r{from, 2048};
  emu::load_lds(r, tile[0], 16, 16 * emu::lane(), 0);
  emu::load_lds(r, tile[1], 16, 16 * emu::lane(), 1024);
  emu::wait_direct(left);
  emu::barrier();
  out[threadIdx.x] = tile[1][255 - threadIdx.x];
}
int main(int, char** v) {
  static char from[2048];
  static float out[64];
  const int left = atoi(v[1]);
  hipLaunchKernelGGL(kernel, dim3(1), dim3(64), 0, nullptr, from, left, out);
  puts("ok");
}
""")
    exe = tmp_path / "short"
    subprocess.run([emu.CLANG, *emu.FLAGS, "-DEMU_WAITS", "-I", emu.HERE, str(src), emu.HERE + "/emu.cpp", "-o", str(exe), "-lm"],
                   check=True)
    for left, good in ((0, True), (1, False)):
        r = subprocess.run([str(exe), str(left)], env=ENV, capture_output=True, text=True, timeout=60)
        assert (r.returncode == 0) == good and ("AddressSanitizer" in r.stderr) == (not good), (r.stdout, r.stderr[-500:])
