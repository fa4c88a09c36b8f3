// expert_linear's C entries on the emulated device.  Each input line is one call:
//   name dtype act bias res grouped tiles K N tail sizes...   (a name with ! has a weight 16 bytes short;
//   one with ? gives num_rows in place of the tail and the offsets themselves, of any values)
// dtype 0 fp32, 1 bf16; tiles: -1 the rule's, 0 256-row, 1 384-row, 2 128-row, 3 64-row, 4 256-row group by
// group (none of 0 to 4 runs few rows as a stream).  Forward and backward run with buffers of exactly
// their sizes.  Checked: every access; the tables of a grouped call against their definition; that
// tiles store each output of a group's rows once, and that every output is written.
#include <unistd.h>
#include <cstdarg>
#include <iostream>
#include <sstream>
#include <string>
#include <vector>

namespace emu { int tiles = -1; }
#include "oxidizr_amd/csrc/ops_api.hip"

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
struct Buffer {
  char* p;
  size_t n;
  explicit Buffer(size_t bytes, int fill = 0) : p(nullptr), n(bytes) {
    if (!n) return;
    if (posix_memalign((void**)&p, 256, n)) abort();
    memset(p, fill, n);
  }
  ~Buffer() { free(p); }
  bool written(size_t from = 0) const {  // no 16 bytes of the fill 0x5a left
    for (size_t i = from; i + 16 <= n; i += 16) {
      bool left = true;
      for (int j = 0; j < 16; ++j) left &= p[i + j] == 0x5a;
      if (left) return false;
    }
    return true;
  }
};
void expect(bool ok, const std::string& name, const char* what) {
  if (ok) return;
  printf("%s: %s\n", name.c_str(), what);
  fflush(stdout);
  _exit(4);
}
// Tiles' stores: once in a group's rows, none elsewhere.
void once(const std::string& name, const Buffer& out, size_t row_bytes, int64_t first, int64_t last, const char* what) {
  const auto& c = emu::stores_of(out.p);
  for (size_t i = 0; i < c.size(); ++i) {
    const int64_t row = (int64_t)(i * 16 / row_bytes);
    if (c[i] != (row >= first && row < last ? 1 : 0)) {
      printf("row %lld of %s stored %d times\n", (long long)row, what, c[i]);
      expect(false, name, what);
    }
  }
}
}  // namespace

int main() {
  std::string line;
  while (std::getline(std::cin, line)) {
    std::istringstream in(line);
    std::string name;
    int dtype, act, bias, res, grouped, K, N;
    int64_t tail;
    if (!(in >> name >> dtype >> act >> bias >> res >> grouped >> emu::tiles >> K >> N >> tail)) continue;
    const bool given = name[0] == '?';
    std::vector<int> offsets;
    if (!given) offsets.push_back(0);
    for (int n; in >> n;) offsets.push_back(given ? n : offsets.back() + n);
    const int E = grouped ? (int)offsets.size() - 1 : 1;
    const int64_t rows = offsets.back(), M = given ? tail : rows + tail, first = grouped ? offsets[0] : 0;
    // whether the offsets ascend within 0 .. M: only then is it defined which rows are a group's
    const bool valid = !given || (std::is_sorted(offsets.begin(), offsets.end()) && offsets[0] >= 0 && offsets.back() <= M);
    const size_t b = dtype == MOE_DTYPE_F32 ? 4 : 2;
    Buffer off(offsets.size() * 4), x(M * K * b), w((size_t)E * N * K * b - (name[0] == '!' ? 16 : 0)), bs(bias ? (size_t)E * N * b : 0),
        r(res ? M * N * b : 0), y(M * N * b, 0x5a), pre(M * N * b, 0x5a);
    memcpy(off.p, offsets.data(), off.n);
    const int* o = grouped ? (const int*)off.p : nullptr;
    const bool stream = emu::tiles < 0 && (dtype ? linear_skinny<bf16_t>(M, K, N, E, grouped) : linear_skinny<float>(M, K, N, E, grouped));
    {
      Buffer ws(moe_linear_workspace_bytes(dtype, M, K, N, E, grouped, act, 0));
      emu::count_stores(y.p, y.n);
      expect(moe_linear_forward(0, nullptr, dtype, M, K, N, E, o, x.p, w.p, bs.p, r.p, act, y.p, pre.p, ws.p) == MOE_OK,
             name, "forward");
      if (!stream && valid) once(name, y, N * b, first, grouped ? rows : M, "y");
      if (grouped && !stream && valid) {
        const LinearWs L = linear_ws(dtype, M, K, N, E, true, act, false);
        std::vector<int> want(kNumTilePrefixes * (E + 1), 0);
        for (int s = 0; s < kNumTilePrefixes; ++s)
          for (int e = 0; e < E; ++e) {
            const int bm = kPrefixBM[s], c = offsets[e + 1] - offsets[e], rest = c % bm;
            const bool merged = c > bm && rest > 0 && rest <= tall_rows_for(bm), own = rest > 0 && !merged;
            want[s * (E + 1) + e + 1] = want[s * (E + 1) + e] +
                (kPrefixKind[s] == 0 ? c / bm + own : kPrefixKind[s] == 1 ? c / bm + (rest > bm / 2) : own && rest <= bm / 2);
          }
        expect(!memcmp(ws.p + L.offs, offsets.data(), off.n), name, "offsets");
        expect(!memcmp(ws.p + L.prefixes, want.data(), want.size() * 4), name, "prefixes");
      }
      expect(!valid || (y.written() && pre.written()), name, "an output was not written");
      emu::forget_counts();
    }
    if (M * std::max(K, N) * (int64_t)b < kMaxExtentBytes) {
      Buffer ws(moe_linear_workspace_bytes(dtype, M, K, N, E, grouped, act, 1)), dy(M * N * b), dx(M * K * b, 0x5a),
          dw((size_t)E * N * K * b, 0x5a), db((size_t)E * N * b, 0x5a);
      emu::count_stores(dx.p, dx.n);
      expect(moe_linear_backward(0, nullptr, dtype, M, K, N, E, o, dy.p, x.p, w.p, pre.p, act, dx.p, dw.p, db.p, ws.p) ==
                 MOE_OK, name, "backward");
      if (M && valid) once(name, dx, K * b, first, grouped ? rows : M, "dx");
      expect(!valid || (dx.written() && dw.written() && db.written()), name, "a gradient was not written");
      emu::forget_counts();
    }
    printf("ok %s\n", name.c_str());
    fflush(stdout);
  }
}
