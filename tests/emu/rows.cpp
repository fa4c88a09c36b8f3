// The sort, row and norm entries on the emulated device.  Each input line is one call:
//   sort name index_bytes T k E pad            (against a stable sort; pad: every pad-th index has no expert)
//   rows name dtype T k E H pad                (permute, unpermute with and without weights, their gradients;
//                                               pad < 0: over an order that no sort made)
//   norm name dtype T H gate post next given   (forward and backward; given: from h_out)
// Buffers are of exactly their sizes: every access is checked, and that every output is written.
#include <unistd.h>
#include <cstdarg>
#include <iostream>
#include <sstream>
#include <string>
#include <vector>

namespace emu { int tiles = -1; }
#include "oxidizr_amd/csrc/ops_api.hip"

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
  void written(const char* what) const {
    for (size_t i = 0; i + 4 <= n; i += 4)
      if (!memcmp(p + i, "\x5a\x5a\x5a\x5a", 4)) expect(false, what);
  }
};
struct Out : Buffer {
  explicit Out(size_t bytes) : Buffer(bytes, 0x5a) {}
};

// counts, offsets, perm, inv of T k indices
struct Order {
  Buffer counts, offsets, perm, inv;
  Order(int64_t T, int k, int E, int bytes, int pad)
      : counts(E * 4, 0x5a), offsets((E + 1) * 4, 0x5a), perm(T * k * 4, 0x5a), inv(T * k * 4, 0x5a) {
    const int64_t n = T * k;
    Buffer idx(n * bytes), ws(moe_sort_workspace_bytes(T, k, E));
    std::vector<int> key(n);
    uint32_t h = 1;
    for (int64_t i = 0; i < n; ++i) {
      h = h * 1664525u + 1013904223u;
      int64_t e = (h >> 8) % E;
      if (pad && (h >> 4) % pad == 0) e = h & 1 ? -1 - (int)(h % 7) : E + (int)(h % 9);
      key[i] = e < 0 || e >= E ? E : (int)e;
      if (bytes == 8) ((int64_t*)idx.p)[i] = e;
      else ((int32_t*)idx.p)[i] = (int)e;
    }
    expect(moe_sort_tokens(0, nullptr, T, k, E, bytes, idx.p, (int*)counts.p, (int*)offsets.p, (int*)perm.p, (int*)inv.p,
                           ws.p) == MOE_OK, "sort");
    std::vector<int> start(E + 2, 0);
    for (int e : key) ++start[e + 1];
    for (int e = 0; e < E; ++e) expect(((int*)counts.p)[e] == start[e + 1], "counts");
    for (int e = 0; e <= E; ++e) start[e + 1] += start[e];
    for (int e = 0; e <= E; ++e) expect(((int*)offsets.p)[e] == start[e], "offsets");
    for (int64_t i = 0; i < n; ++i) {
      const int at = start[key[i]]++;
      expect(((int*)inv.p)[i] == at && ((int*)perm.p)[at] == i, "order");
    }
  }
};
}  // namespace

int main() {
  std::string line, kind;
  while (std::getline(std::cin, line)) {
    std::istringstream in(line);
    if (!(in >> kind >> name)) continue;
    if (kind == "sort") {
      int bytes, k, E, pad;
      int64_t T;
      in >> bytes >> T >> k >> E >> pad;
      Order(T, k, E, bytes, pad);
    } else if (kind == "rows") {
      int dtype, k, E, H, pad;
      int64_t T;
      in >> dtype >> T >> k >> E >> H >> pad;
      const size_t b = dtype == MOE_DTYPE_F32 ? 4 : 2;
      Order o(T, k, E, 4, std::max(pad, 0));
      int* inv = (int*)o.inv.p;
      if (pad < 0) {
        const int any[] = {-1, INT_MAX, INT_MIN, (int)(T * k), (int)(T * k) - 1, 1000000007};
        for (int64_t i = 0; i < T * k; i += 3) inv[i] = any[i / 3 % 6];
        ((int*)o.offsets.p)[E] = pad == -1 ? INT_MAX : pad == -2 ? -7 : (int)(T * k) + 1;
      }
      const int* kept = (int*)o.offsets.p + E;
      Buffer x(T * H * b), y(T * k * H * b), w(T * k * 4);
      Out xp(y.n), out(x.n), plain(x.n), dy(y.n), dy2(y.n), dw(w.n);
      expect(moe_permute(0, nullptr, dtype, T, k, H, inv, kept, x.p, xp.p) == MOE_OK, "permute");
      expect(moe_unpermute(0, nullptr, dtype, T, k, H, inv, kept, y.p, (float*)w.p, out.p) == MOE_OK, "unpermute");
      expect(moe_unpermute(0, nullptr, dtype, T, k, H, inv, kept, y.p, nullptr, plain.p) == MOE_OK, "unpermute");
      expect(moe_unpermute_backward(0, nullptr, dtype, T, k, H, inv, kept, x.p, y.p, (float*)w.p, dy.p, (float*)dw.p) ==
                 MOE_OK, "backward");
      expect(moe_unpermute_backward(0, nullptr, dtype, T, k, H, inv, kept, x.p, nullptr, nullptr, dy2.p, nullptr) ==
                 MOE_OK, "backward");
      if (pad >= 0) xp.written("x_perm"), dy.written("d_y"), dy2.written("d_y");
      out.written("out"), plain.written("out");
      dw.written("d_weights");
    } else {
      int dtype, H, gate, post, next, given;
      int64_t T;
      in >> dtype >> T >> H >> gate >> post >> next >> given;
      const size_t b = dtype == MOE_DTYPE_F32 ? 4 : 2, n = T * H * b, g = gate == 0 ? 0 : gate == 1 ? H * b : gate == 2 ? T * b : n;
      Buffer h(n), y(n), w2(post ? H * b : 0), gt((g + 15) / 16 * 16), w3(next ? H * b : 0), dn(next ? n : 0), dh_out(n);
      Out hn(n), nn(next ? n : 0), r2(post ? T * 4 : 0), r3(next ? T * 4 : 0), dh(n), dy(n), dw2(w2.n), dg(gt.n), dw3(w3.n);
      Buffer ws(moe_residual_norm_workspace_bytes(T, H));
      expect(moe_residual_norm(0, nullptr, dtype, T, H, h.p, y.p, w2.p, gt.p, gate, w3.p, 0.5f, 1e-6f, hn.p, nn.p,
                               (float*)r2.p, (float*)r3.p) == MOE_OK, "norm");
      hn.written("h_out"), nn.written("n_out"), r2.written("rstd"), r3.written("rstd");
      auto* backward = given ? moe_residual_norm_backward : moe_residual_norm_backward_from_input;
      expect(backward(0, nullptr, dtype, T, H, dh_out.p, dn.p, given ? hn.p : h.p, y.p, w2.p, gt.p, gate, w3.p, 0.5f,
                      (float*)r2.p, (float*)r3.p, dh.p, dy.p, dw2.p, dg.p, dw3.p, ws.p) == MOE_OK, "norm backward");
      dh.written("d_h"), dy.written("d_y"), dw2.written("d_post"), dw3.written("d_next");
      if (gate != 2) dg.written("d_gate");  // a token gate's buffer is rounded up
      if (next && !post && !gate) {  // the same entry without y
        Out n2(n), d2(n), dw(w3.n);
        expect(moe_residual_norm(0, nullptr, dtype, T, H, h.p, nullptr, nullptr, nullptr, 0, w3.p, 1.0f, 1e-6f, nullptr,
                                 n2.p, nullptr, (float*)r3.p) == MOE_OK, "rms norm");
        expect(backward(0, nullptr, dtype, T, H, nullptr, dn.p, h.p, nullptr, nullptr, nullptr, 0, w3.p, 1.0f, nullptr,
                        (float*)r3.p, d2.p, nullptr, nullptr, nullptr, dw.p, ws.p) == MOE_OK, "rms norm backward");
        n2.written("n"), d2.written("d"), dw.written("dw");
      }
    }
    printf("ok %s\n", name.c_str());
    fflush(stdout);
  }
}
