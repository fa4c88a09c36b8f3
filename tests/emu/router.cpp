// The entries of the router's losses on the emulated device.  Each input line is one call:
//   name dtype index_bytes score T E k sequences offsets...   (sequences 0: none; - 1 offsets of any values follow, 0 .. T where
//   none do; a name with ! has logits four bytes short)
// Buffers are of exactly their sizes.  Checked: every access, that every output is written, and (ascending offsets) the counts.
#include <unistd.h>
#include <cstdarg>
#include <iostream>
#include <sstream>
#include <string>
#include <vector>

namespace emu { int tiles = -1; }
#include "oxidizr_amd/csrc/router_api.hip"

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
  char* p = nullptr;
  size_t n;
  explicit Buffer(size_t bytes, int fill = 0) : n(bytes) {
    if (!n) return;
    if (posix_memalign((void**)&p, 256, n)) abort();
    memset(p, fill, n);
  }
  Buffer(const Buffer&) = delete;
  ~Buffer() { free(p); }
  bool written(size_t step = 4) const {
    for (size_t i = 0; i + step <= n; i += step) {
      bool left = true;
      for (size_t j = 0; j < step; ++j) left &= p[i + j] == 0x5a;
      if (left) return false;
    }
    return true;
  }
};
}  // namespace

int main() {
  std::string line;
  while (std::getline(std::cin, line)) {
    std::istringstream in(line);
    int dtype, bytes, score, E, k, S;
    int64_t T;
    if (!(in >> name >> dtype >> bytes >> score >> T >> E >> k >> S)) continue;
    std::vector<int> offsets;
    for (int n; in >> n;) offsets.push_back(n);
    const bool seqs = S > 0;
    if (seqs && offsets.empty())
      for (int i = 0; i <= S; ++i) offsets.push_back((int)(T * i / S));
    if (!seqs) S = 1;
    bool valid = true;
    for (size_t i = 0; i < offsets.size(); ++i)
      valid &= offsets[i] >= (i ? offsets[i - 1] : 0) && offsets[i] <= T;
    const size_t b = dtype == MOE_DTYPE_F32 ? 4 : 2;
    Buffer logits(T * E * b - (name[0] == '!' ? 4 : 0)), idx(T * k * bytes), off(offsets.size() * 4), balance(S * 4, 0x5a),
        z(S * 4, 0x5a), counts(S * E * 4, 0x5a), slope(S * E * 4, 0x5a), inv(S * 4, 0x5a),
        d((T * E * b + 15) / 16 * 16, 0x5a), up(S * 4);
    if (off.n) memcpy(off.p, offsets.data(), off.n);
    std::vector<int> want(S * E, 0);
    uint32_t h = 7;
    for (int64_t i = 0; i < T * k; ++i) {
      h = h * 1664525u + 1013904223u;
      int64_t e = (h >> 8) % (E + 2) - 1;  // -1 and E: no expert
      if (bytes == 8) ((int64_t*)idx.p)[i] = e;
      else ((int32_t*)idx.p)[i] = (int)e;
      for (int s = 0; s < S && e >= 0 && e < E; ++s)
        if (!seqs || (i / k >= offsets[s] && i / k < offsets[s + 1])) ++want[s * E + e];
    }
    Buffer ws(moe_router_losses_workspace_bytes(T, E, S), 0x11);
    const int* o = seqs ? (const int*)off.p : nullptr;
    expect(moe_router_losses(0, nullptr, dtype, T, E, k, bytes, logits.p, idx.p, score, 0.5f, 1.0f, 1.0f, o, S, (float*)balance.p,
                             (float*)z.p, (int*)counts.p, (float*)slope.p, (float*)inv.p, ws.p) == MOE_OK, "forward");
    expect(balance.written() && z.written() && counts.written() && slope.written() && inv.written(), "an output was not written");
    if (valid) expect(!memcmp(counts.p, want.data(), counts.n), "counts");
    expect(moe_router_losses_backward(0, nullptr, dtype, T, E, k, bytes, logits.p, idx.p, score, 0.5f, o, S, (float*)slope.p,
                                      (float*)inv.p, (float*)up.p, (float*)up.p, d.p) == MOE_OK, "backward");
    d.n = T * E * b;
    expect(d.written(b), "d_logits was not written");
    printf("ok %s\n", name.c_str());
    fflush(stdout);
  }
}
