// Host tables (operand pointers, constants) brought to the device inside the
// parameters of small kernels: no copy from pageable memory, which would make
// the host wait for the stream, and nothing of the caller's is read after the
// call returns, so that a call can also be captured into a graph.
#include <string.h>

#include "context.h"
#include "kernels.h"

namespace cfhe {
namespace {

constexpr int kUploadWords = 7936;  // 31 KB of the 32 764 bytes that kernel parameters may take
struct UploadArgs {
  uint32_t *dst;
  int n;
  uint32_t w[kUploadWords];
};

__global__ void __launch_bounds__(256) upload_kernel(const __grid_constant__ UploadArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  for (int i = blockIdx.x * 256 + threadIdx.x; i < a.n; i += gridDim.x * 256) a.dst[i] = a.w[i];
}

}  // namespace

int launch_upload(const Context &c, void *dst, const void *src, size_t words) {
  UploadArgs a;
  for (size_t at = 0; at < words; at += kUploadWords) {
    a.dst = static_cast<uint32_t *>(dst) + at;
    a.n = (int)(words - at < (size_t)kUploadWords ? words - at : (size_t)kUploadWords);
    memcpy(a.w, static_cast<const uint32_t *>(src) + at, (size_t)a.n * sizeof(uint32_t));
    CFHE_CUDA(launch_kernel(c.use_pdl, upload_kernel, dim3((a.n + 1023) / 1024), dim3(256), 0, c.stream, a));
  }
  return 0;
}

}  // namespace cfhe
