// The entries of 4-bit numbers and of the products over them on the emulated device.  Each input line is one call:
//   quant name dtype blocks
//   linear name four dtype act bias res grouped tiles K N tail sizes...   (a name with ! has weights 16 bytes of codes short,
//   one with / weights a scale short; one with ? gives num_rows in place of the tail and the offsets themselves, of any values)
// tiles: -1 the rule's, -2 the stream of few rows, 0 / 1 / 2 256-, 128- and 64-row tiles.  Buffers are of exactly their
// sizes, scales at an odd address.  Checked: every access; that tiles store each output of a group's rows once, and that
// every output is written.
#include <unistd.h>
#include <cstdarg>
#include <iostream>
#include <sstream>
#include <string>
#include <vector>

namespace emu { int tiles = -1; }
#include "oxidizr_amd/csrc/mx_api.hip"

namespace emu {
void count_stores(const void* base, size_t bytes);
const std::vector<uint8_t>& stores_of(const void* base);
void forget_counts();
}
namespace moe { namespace {
moe_status fail(moe_status st, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vprintf(fmt, ap);
  va_end(ap);
  printf("\n");
  return st;
}
} }

namespace {
std::string name;
void expect(bool ok, const char* what) {
  if (ok) return;
  printf("%s: %s\n", name.c_str(), what);
  fflush(stdout);
  _exit(4);
}
struct Buffer {
  char* base = nullptr;
  char* p = nullptr;
  size_t n;
  // off: the address is that far behind an aligned one
  explicit Buffer(size_t bytes, int fill = 0, int off = 0) : n(bytes) {
    if (!n) return;
    if (posix_memalign((void**)&base, 256, n + off)) abort();
    p = base + off;
    memset(p, fill, n);
  }
  Buffer(const Buffer&) = delete;
  ~Buffer() { free(base); }
  bool written(size_t step = 16) const {  // no `step` bytes of the fill 0x5a left
    for (size_t i = 0; i + step <= n; i += step) {
      bool left = true;
      for (size_t j = 0; j < step; ++j) left &= p[i + j] == 0x5a;
      if (left) return false;
    }
    return true;
  }
};
void once(const Buffer& out, size_t row_bytes, int64_t first, int64_t last, const char* what) {
  const auto& c = emu::stores_of(out.p);
  for (size_t i = 0; i < c.size(); ++i) {
    const int64_t row = (int64_t)(i * 16 / row_bytes);
    if (c[i] != (row >= first && row < last ? 1 : 0)) {
      printf("row %lld of %s stored %d times\n", (long long)row, what, c[i]);
      expect(false, what);
    }
  }
}
}  // namespace

int main() {
  std::string line, kind;
  while (std::getline(std::cin, line)) {
    std::istringstream in(line);
    if (!(in >> kind >> name)) continue;
    if (kind == "quant") {
      int dtype;
      int64_t blocks;
      in >> dtype >> blocks;
      const size_t b = dtype == MOE_DTYPE_F32 ? 4 : 2;
      Buffer x(blocks * 32 * b, 1), codes(blocks * 16, 0x5a), scales(blocks, 0x5a, 3), y(blocks * 32 * b, 0x5a);
      expect(moe_mx_quantize(0, nullptr, dtype, blocks, x.p, (uint8_t*)codes.p, (uint8_t*)scales.p) == MOE_OK, "quantize");
      expect(codes.written(4) && scales.written(1), "an output was not written");
      expect(moe_mx_dequantize(0, nullptr, dtype, blocks, (uint8_t*)codes.p, (uint8_t*)scales.p, y.p) == MOE_OK, "dequantize");
      expect(y.written(), "y was not written");
    } else {
      int four, dtype, act, bias, res, grouped, K, N;
      int64_t tail;
      in >> four >> dtype >> act >> bias >> res >> grouped >> emu::tiles >> K >> N >> tail;
      const bool given = name[0] == '?';
      std::vector<int> offsets;
      if (!given) offsets.push_back(0);
      for (int n; in >> n;) offsets.push_back(given ? n : offsets.back() + n);
      const int E = grouped ? (int)offsets.size() - 1 : 1;
      const int64_t rows = offsets.back(), M = given ? tail : rows + tail, first = grouped ? offsets[0] : 0;
      const bool valid = !given || (std::is_sorted(offsets.begin(), offsets.end()) && offsets[0] >= 0 && offsets.back() <= M);
      const size_t b = dtype == MOE_DTYPE_F32 ? 4 : 2;
      Buffer off(offsets.size() * 4), x(four ? M * K / 2 : M * K * 2), xs(four ? M * K / 32 : 0, 0, 1),
          w((size_t)E * N * K / 2 - (name[0] == '!' ? 16 : 0)), ws((size_t)E * N * K / 32 - (name[0] == '/' ? 1 : 0), 0, 5),
          bs(bias ? (size_t)E * N * b : 0), r(res ? M * N * b : 0), y(M * N * b, 0x5a), pre(M * N * b, 0x5a);
      memcpy(off.p, offsets.data(), off.n);
      const int* o = grouped ? (const int*)off.p : nullptr;
      const bool stream = mx_skinny(four, M, K, N, E, grouped);
      emu::count_stores(y.p, y.n);
      expect(moe_mx_linear_forward(0, nullptr, four, dtype, M, K, N, E, o, x.p, (uint8_t*)xs.p, (uint8_t*)w.p,
                                   (uint8_t*)ws.p, bs.p, r.p, act, y.p, pre.p) == MOE_OK, "forward");
      if (!stream && valid) once(y, N * b, first, grouped ? rows : M, "y");
      expect(!valid || (y.written() && pre.written()), "an output was not written");
      emu::forget_counts();
      if (!four) {
        Buffer scratch(moe_mx_linear_workspace_bytes(M, K, N, E, grouped, act)), dy(M * N * 2), dx(M * K * 2, 0x5a),
            db((size_t)E * N * 2, 0x5a);
        emu::count_stores(dx.p, dx.n);
        expect(moe_mx_linear_backward(0, nullptr, M, K, N, E, o, dy.p, (uint8_t*)w.p, (uint8_t*)ws.p, pre.p, act, dx.p, db.p,
                                      scratch.p) == MOE_OK, "backward");
        if (valid) once(dx, K * 2, first, grouped ? rows : M, "dx");
        expect(!valid || (dx.written() && db.written()), "a gradient was not written");
        emu::forget_counts();
      }
    }
    printf("ok %s\n", name.c_str());
    fflush(stdout);
  }
}
