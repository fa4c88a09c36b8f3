"""Builds the library's kernels for the emulated device of this folder (a CPU program under
AddressSanitizer), from copies of the sources in which only this is changed: waits and barriers in inline asm go,
dynamic LDS comes from the emulator, names have internal linkage (the sanitizer leaves static arrays of
others alone, and LDS arrays become such), and a caller may name the row tiles (and fewer blocks fill
what belongs to no expert)."""
import os
import re
import shutil
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(os.path.dirname(HERE))
CLANG = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "clang++")
FLAGS = ["-x", "c++", "-std=c++17", "-O1", "-g1", "-w", "-fno-strict-aliasing", "-Xarch_host", "-fsanitize=address"]


def replaced(text, old, new):
    assert old in text, old
    return text.replace(old, new)


def sources(to):
    """The csrc folder and the header, with the changes."""
    src = os.path.join(to, "oxidizr_amd", "csrc")
    os.makedirs(src)
    os.makedirs(os.path.join(to, "include"))
    shutil.copy(os.path.join(ROOT, "include", "moe_hip.h"), os.path.join(to, "include"))
    for name in os.listdir(os.path.join(ROOT, "oxidizr_amd", "csrc")):
        if not name.endswith((".hpp", ".hip")):
            continue
        text = open(os.path.join(ROOT, "oxidizr_amd", "csrc", name)).read()
        text = re.sub(r"asm volatile\([^;]*\);", ";", text)
        text = re.sub(r"extern __shared__ int (\w+)\[\];", r"int* \1 = (int*)emu::dynamic_lds();", text)
        text = text.replace("namespace moe {", "namespace moe { namespace {").replace("}  // namespace moe", "} }")
        if name == "ops_api.hip":
            text = replaced(text, "RowTiles pick_tiles(bool grouped, int E, int64_t M, int N) {",
                            "RowTiles pick_tiles(bool grouped, int E, int64_t M, int N) {\n"
                            "  if (emu::tiles >= 0 && sizeof(D) == 2) return (RowTiles)(emu::tiles & 3);")
            # the blocks past the first share a loop: three of them take the place of 128
            text = replaced(text, "constexpr int kPrepBlocks = 1 + 128;", "constexpr int kPrepBlocks = 1 + 3;")
            text = replaced(text, "bool linear_skinny(int64_t M, int K, int N, int E, bool grouped) {",
                            "bool linear_skinny(int64_t M, int K, int N, int E, bool grouped) {\n"
                            "  if (emu::tiles >= 0) return false;")
            text = replaced(text, "p.tiles = big <= tall ? RowTiles::kBig : RowTiles::kTall;",
                            "if (emu::tiles < 0) p.tiles = big <= tall ? RowTiles::kBig : RowTiles::kTall;")
            text = replaced(text, "(big && M >= 2 * (int64_t)C::BM * E)",
                            "(big && (emu::tiles < 0 ? M >= 2 * (int64_t)C::BM * E : emu::tiles == 0))")
        with open(os.path.join(src, name), "w") as f:
            f.write(text)


def build(to, program):
    """The path of `program`.cpp, built in the folder `to`."""
    to = str(to)
    sources(to)
    objs = []
    procs = []
    for name in ("emu.cpp", program + ".cpp"):
        objs.append(os.path.join(to, name + ".o"))
        cmd = [CLANG, *FLAGS, "-I", HERE, "-I", to, "-c", os.path.join(HERE, name), "-o", objs[-1]]
        procs.append((cmd, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    for cmd, p in procs:
        out = p.communicate()[0]
        assert p.returncode == 0, " ".join(cmd) + "\n" + out[:6000]
    exe = os.path.join(to, program)
    subprocess.run([CLANG, "-Xarch_host", "-fsanitize=address", *objs, "-o", exe, "-lm"], check=True)
    return exe
