// The tensor-core matrix products after an expired wait. The kernels are compiled into
// this program with no tries for the wait for a stage's operands, so that every CTA's
// MMA thread gives up before its first instruction (the other waits keep their limit,
// and few enough stages are filled that none of them has to wait for a freed one).
// The context's flag has to be up, and no result, nor a residual that is its own
// output, may have been touched.
#define CFHE_STAGE_TRIES 0
#include "../../cheddar-fhe_b200/csrc/gemm_tc.cu"

#include <stdio.h>

namespace cfhe {
static std::string message;
void set_error(const std::string &m) { message = m; }
const std::string &get_error() { return message; }
std::atomic<unsigned long long> g_kernel_launches{0};
}  // namespace cfhe
using namespace cfhe;

static void check(cudaError_t e) {
  if (e != cudaSuccess) {
    printf("FAIL: %s\n", cudaGetErrorString(e));
    exit(1);
  }
}
static uint32_t *device_words(size_t n, int byte) {
  void *p = nullptr;
  check(cudaMalloc(&p, n * sizeof(uint32_t)));
  check(cudaMemset(p, byte, n * sizeof(uint32_t)));
  return static_cast<uint32_t *>(p);
}
static uint32_t *const *device_table(uint32_t *polys, int count) {
  std::vector<uint32_t *> t;
  for (int i = 0; i < count; i++) t.push_back(polys + (size_t)i * kN);
  void *p = nullptr;
  check(cudaMalloc(&p, count * sizeof(void *)));
  check(cudaMemcpy(p, t.data(), count * sizeof(void *), cudaMemcpyHostToDevice));
  return static_cast<uint32_t *const *>(p);
}

int main() {
  const int n_in = 16, n_out = 8;  // one K step; at most four tiles for a CTA that stays
  Context c;
  check(cudaStreamCreate(&c.stream));
  c.NP = 1;
  c.q = {1073872897u};
  uint32_t inv = 1;
  for (int i = 0; i < 5; i++) inv *= 2u - c.q[0] * inv;
  c.nqinv = {0u - inv};
  check(cudaMalloc(&c.d_error_flag, sizeof(int)));
  const int gidx[1] = {0};
  const size_t scratch = gemm_scratch_bytes(n_in);
  uint32_t *const x = device_words((size_t)2 * n_in * kN, 1), *const y = device_words((size_t)2 * n_out * kN, 0x5a);
  uint32_t *const xp = device_words(kMaxGroup * scratch / 4, 0);
  uint32_t *const w = device_words(gemm_packed_weight_bytes(n_in, n_out) / 4, 1);
  uint32_t *const *const xt = device_table(x, 2 * n_in), *const *const yt = device_table(y, 2 * n_out);

  for (int call = 0; call < 2; call++) {
    check(cudaMemset(c.d_error_flag, 0, sizeof(int)));
    check(cudaDeviceSynchronize());
    int r;
    if (call == 0) {
      uint8_t *const buffers[2] = {reinterpret_cast<uint8_t *>(xp), nullptr};
      r = launch_ctpt_gemm(c, yt, xt, reinterpret_cast<uint8_t *>(w), buffers, n_in, n_out, gidx, 1);
    } else {
      ProjectCall p = {};
      for (int poly = 0; poly < 2; poly++) {
        p.x[poly] = xt + poly * n_in;
        p.y[poly] = yt + poly * n_out;
        p.res[poly] = yt + poly * n_out;
      }
      p.packed = reinterpret_cast<uint8_t *>(w);
      p.scratch = reinterpret_cast<uint8_t *>(xp);
      p.n_in = n_in;
      p.n_out = n_out;
      p.n_limbs = 1;
      p.gidx = gidx;
      r = launch_ctpt_project(c, p);
    }
    if (r) {
      printf("FAIL: %s\n", message.c_str());
      return 1;
    }
    check(cudaStreamSynchronize(c.stream));
    int flag = 0;
    check(cudaMemcpy(&flag, c.d_error_flag, sizeof(int), cudaMemcpyDeviceToHost));
    std::vector<uint32_t> got((size_t)2 * n_out * kN);
    check(cudaMemcpy(got.data(), y, got.size() * sizeof(uint32_t), cudaMemcpyDeviceToHost));
    size_t touched = 0;
    for (uint32_t v : got) touched += v != 0x5a5a5a5au;
    printf("%s: flag %d, %zu words stored\n", call ? "projection" : "product", flag, touched);
    if (flag != 1 || touched) {
      printf("FAIL\n");
      return 1;
    }
  }
  printf("PASS\n");
  return 0;
}
