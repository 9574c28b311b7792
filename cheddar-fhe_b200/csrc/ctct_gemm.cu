// Matrix product of ciphertexts, three-part results:
//   D[i][j] = w[i][j] (*) sum_t L[i][t] (x) R[t][j],
// (x) the tensor product (b b', b a' + a b', a a') and w an optional weight per
// result, a plaintext polynomial or one constant per limb: the scores and the
// weighted values of (decayed linear) attention over encrypted tokens. Words as
// from cfhe_tensor_accum followed by a plaintext or constant product.
#include "context.h"
#include "kernels.h"
#include "modmath.cuh"

namespace cfhe {
namespace {

constexpr int kCcThreads = 256;

// One result per block row: every operand word comes from memory (or L2) once
// per result that it enters.
__global__ void __launch_bounds__(kCcThreads) ctct_kernel(const __grid_constant__ CtctArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int l = blockIdx.z, o = blockIdx.y, i = o / a.n, j = o % a.n;
  const size_t at = (size_t)l * kN + blockIdx.x * kCcThreads + threadIdx.x;
  const uint32_t q = a.q[l], nq = a.nqinv[l];
  const uint64_t q32 = (uint64_t)q << 32;
  const int mk = a.m * a.k, kn = a.k * a.n, mn = a.m * a.n;
  const uint32_t *const *lb = a.table + i * a.k, *const *la = lb + mk;
  const uint32_t *const *rb = a.table + 2 * mk + j, *const *ra = rb + kn;
  const uint32_t *const *out = a.table + 2 * (mk + kn) + o;
  uint64_t s0 = 0, s1 = 0, s2 = 0;
  for (int t = 0; t < a.k; t++) {
    const uint32_t xb = lb[t][at], xa = la[t][at], yb = rb[t * a.n][at], ya = ra[t * a.n][at];
    mac_fold(s0, xb, yb, q32);
    mac_fold(s1, xb, ya, q32);
    mac_fold(s1, xa, yb, q32);
    mac_fold(s2, xa, ya, q32);
  }
  uint32_t d[3] = {mont_reduce(s0, q, nq), mont_reduce(s1, q, nq), mont_reduce(s2, q, nq)};
  if (a.weights || a.consts) {
    const uint32_t w = a.weights ? out[3 * mn][at] : a.consts[(size_t)o * a.n_limbs + l];
    for (int p = 0; p < 3; p++) d[p] = mont_mul(d[p], w, q, nq);
  }
  for (int p = 0; p < 3; p++) const_cast<uint32_t *>(out[p * mn])[at] = d[p];
}

}  // namespace

int launch_ctct_gemm(const Context &ctx, const CtctArgs &args) {
  const dim3 grid(kN / kCcThreads, args.m * args.n, args.n_limbs), block(kCcThreads);
  CFHE_CUDA(launch_kernel(ctx.use_pdl, ctct_kernel, grid, block, 0, ctx.stream, args));
  CFHE_CUDA(cudaGetLastError());
  return 0;
}

}  // namespace cfhe
