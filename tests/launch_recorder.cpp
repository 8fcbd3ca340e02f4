// Calls one of the token operators with pointers that nothing reads and prints
// the launches it makes: the HIP functions that the library calls are the ones
// below, so nothing reaches a GPU.
//   launch_recorder FAIL OP NUMBER...
// The FAIL-th launch (from 0; -1: none) returns an error.  A line per launch:
//   kernel grid.x grid.y grid.z block.x block.y block.z
// and at the end "rc" with what the call returned.
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <string>
#include <vector>

struct Dim {
  uint32_t x, y, z;
};

namespace {
std::map<const void*, std::string>& names() {
  static std::map<const void*, std::string> m;
  return m;
}
Dim grid, block;
int launches = 0, fail_at = -1, error = 0;
constexpr int kInvalidConfiguration = 9;
}  // namespace

extern "C" {
void** __hipRegisterFatBinary(const void*) {
  static void* handle;
  return &handle;
}
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterFunction(void**, const void* host, char*, const char* name, unsigned, void*,
                           void*, Dim*, Dim*, int*) {
  names()[host] = name;
}
void __hipRegisterVar(void**, void*, char*, char*, int, size_t, int, int) {}
int __hipPushCallConfiguration(Dim g, Dim b, size_t, void*) {
  grid = g;
  block = b;
  return 0;
}
int __hipPopCallConfiguration(Dim* g, Dim* b, size_t* shared, void** stream) {
  *g = grid;
  *b = block;
  *shared = 0;
  *stream = nullptr;
  return 0;
}
int hipLaunchKernel(const void* host, Dim g, Dim b, void**, size_t, void*) {
  const int rc = launches++ == fail_at ? kInvalidConfiguration : 0;
  if (rc != 0) error = rc;
  std::printf("%s %u %u %u %u %u %u\n", names()[host].c_str(), g.x, g.y, g.z, b.x, b.y, b.z);
  return rc;
}
int hipGetLastError() {
  const int was = error;
  error = 0;
  return was;
}
const char* hipGetErrorString(int) { return "planted"; }

int hipo_token_logprobs(const void*, int, const void*, int, float*, float*, float*, float*,
                        int64_t*, int64_t, int64_t, int64_t, float, int64_t, int64_t, void*,
                        size_t, void*);
int hipo_token_logprobs_bwd(const float*, const void*, int, const void*, int, const float*,
                            const float*, const float*, const float*, void*, int64_t, int64_t,
                            int64_t, int64_t, float, int64_t, void*);
int hipo_embedding(const void*, int, const void*, int, void*, int64_t, int64_t, int64_t, int64_t,
                   float, void*);
int hipo_embedding_bwd(const void*, int, const void*, int, void*, int, int64_t, int64_t, int64_t,
                       float, int64_t, int, void*, size_t, void*);
const char* hipo_last_error(void);
}

int main(int argc, char** argv) {
  if (argc < 3) return 2;
  fail_at = std::atoi(argv[1]);
  const std::string op = argv[2];
  std::vector<int64_t> n;
  for (int i = 3; i < argc; ++i) n.push_back(std::strtoll(argv[i], nullptr, 10));
  char* p = reinterpret_cast<char*>(uintptr_t{1} << 30);
  float* f = reinterpret_cast<float*>(p);
  char* q = p + (int64_t{1} << 46);
  const size_t any = SIZE_MAX;
  int rc;
  if (op == "token_logprobs" && n.size() == 4) {  // rows vocab elem top
    rc = hipo_token_logprobs(p, static_cast<int>(n[2]), p, 8, f, f, f, f,
                             reinterpret_cast<int64_t*>(p), n[0], n[1], n[1], 1.0f, -100, n[3], q,
                             any, nullptr);
  } else if (op == "token_logprobs_bwd" && n.size() == 3) {  // rows vocab elem
    rc = hipo_token_logprobs_bwd(f, p, static_cast<int>(n[2]), p, 8, f, f, f, f, q, n[0], n[1],
                                 n[1], n[1], 1.0f, -100, nullptr);
  } else if (op == "embedding" && n.size() == 4) {  // count width vocab elem
    rc = hipo_embedding(p, static_cast<int>(n[3]), p, 8, q, n[0], n[1], n[2], n[1], 1.0f, nullptr);
  } else if (op == "embedding_bwd" && n.size() == 6) {  // count width vocab elem out accumulate
    rc = hipo_embedding_bwd(p, static_cast<int>(n[3]), p, 8, q, static_cast<int>(n[4]), n[0], n[1],
                            n[2], 1.0f, -1, static_cast<int>(n[5]), q, any, nullptr);
  } else {
    return 2;
  }
  std::printf("rc %d %s\n", rc, hipo_last_error());
  return 0;
}
