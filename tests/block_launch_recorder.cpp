// launch_recorder.cpp's stand-ins for HIP, for the norms around a block and the
// output layer's cross entropy.  Calls are read from the standard input, a line
// each:
//   FAIL OP NUMBER...
#include <iostream>
#include <sstream>

#define main token_main
#include "launch_recorder.cpp"
#undef main

extern "C" {
int hipo_block_norms(const void*, const void*, int, const void*, const void*, const void*,
                     const void*, const void*, void*, void*, float*, int64_t, int64_t, int64_t,
                     float, float, float, int, void*);
size_t hipo_block_norms_bwd_workspace_bytes(int64_t, int64_t);
int hipo_block_norms_bwd(const void*, const void*, const void*, const void*, const float*, int,
                         const void*, const void*, const void*, const void*, const void*, void*,
                         void*, void*, void*, void*, void*, void*, int64_t, int64_t, int64_t,
                         float, float, int, void*, size_t, void*);
size_t hipo_linear_cross_entropy_workspace_bytes(const void*, int, int64_t, int64_t, int64_t,
                                                 int64_t);
int hipo_linear_cross_entropy(const void*, const void*, int, const void*, int, float*, float*,
                              int64_t, int64_t, int64_t, int64_t, int64_t, float, int64_t, void*,
                              size_t, void*);
size_t hipo_linear_cross_entropy_bwd_workspace_bytes(const void*, int, int64_t, int64_t, int64_t,
                                                     int64_t);
int hipo_linear_cross_entropy_bwd(const float*, const void*, const void*, int, const void*, int,
                                  const float*, const float*, void*, void*, int64_t, int64_t,
                                  int64_t, int64_t, int64_t, float, int64_t, void*, size_t,
                                  void*);
decltype(hipo_linear_cross_entropy_bwd_workspace_bytes)
    hipo_linear_cross_entropy_bwd_two_parts_workspace_bytes;
decltype(hipo_linear_cross_entropy_bwd) hipo_linear_cross_entropy_bwd_two_parts;
}

namespace {
int call(const std::string& op, const std::vector<int64_t>& n) {
  void* const p = reinterpret_cast<void*>(uintptr_t{1} << 12);
  float* const f = static_cast<float*>(p);
  if (op == "block_norms" && n.size() == 5) {  // rows cols gate_rows elem_size layer
    return hipo_block_norms(p, p, static_cast<int>(n[3]), p, nullptr, p, nullptr,
                            n[2] ? p : nullptr, p, p, f, n[0], n[1], n[2], 1.0f, 0.0f, 1e-6f,
                            static_cast<int>(n[4]), nullptr);
  }
  if (op == "block_norms_bwd" && n.size() == 5) {
    return hipo_block_norms_bwd(p, p, p, p, f, static_cast<int>(n[3]), p, nullptr, p, nullptr,
                                n[2] ? p : nullptr, p, p, n[2] ? p : nullptr, p, nullptr, p,
                                nullptr, n[0], n[1], n[2], 1.0f, 0.0f, static_cast<int>(n[4]), p,
                                hipo_block_norms_bwd_workspace_bytes(n[0], n[1]), nullptr);
  }
  if (n.size() != 4) return 2;  // rows width vocab elem_size
  const int e = static_cast<int>(n[3]);
  if (op == "linear_cross_entropy") {
    return hipo_linear_cross_entropy(
        p, p, e, p, 8, f, f, n[0], n[1], n[2], n[1], n[1], 1.0f, -100, p,
        hipo_linear_cross_entropy_workspace_bytes(p, e, n[0], n[1], n[2], n[1]), nullptr);
  }
  if (op == "linear_cross_entropy_bwd") {
    return hipo_linear_cross_entropy_bwd(
        f, p, p, e, p, 8, f, nullptr, p, p, n[0], n[1], n[2], n[1], n[1], 1.0f, -100, p,
        hipo_linear_cross_entropy_bwd_workspace_bytes(p, e, n[0], n[1], n[2], n[1]), nullptr);
  }
  if (op == "linear_cross_entropy_bwd_two_parts") {
    return hipo_linear_cross_entropy_bwd_two_parts(
        f, p, p, e, p, 8, f, nullptr, p, p, n[0], n[1], n[2], n[1], n[1], 1.0f, -100, p,
        hipo_linear_cross_entropy_bwd_two_parts_workspace_bytes(p, e, n[0], n[1], n[2], n[1]),
        nullptr);
  }
  return 2;
}
}  // namespace

int main() {
  std::string line;
  while (std::getline(std::cin, line)) {
    std::istringstream in(line);
    std::string op;
    std::vector<int64_t> n;
    in >> fail_at >> op;
    for (int64_t v; in >> v;) n.push_back(v);
    launches = 0;
    const int rc = call(op, n);
    std::printf("rc %d\n", rc);
  }
  return 0;
}
