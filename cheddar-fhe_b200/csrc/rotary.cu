// Rotary positions on ciphertexts: every pair of features (u, v) of a token is
// turned by the angle of the token's position on the pair's axis,
//   u' = c u - s v,   v' = s u + c v,
// c and s either plaintext polynomials (each slot holds its token's cosine) or,
// where every slot stands at the same position, one constant per limb. The
// words are those of two plaintext products and a sum or difference per
// polynomial; how many axes there are and which pair follows which is in the
// angles.
//
// Bound by memory: per pair, row and word 16 bytes move against eight
// multiplications. A thread keeps its four words of c and s and walks the rows
// (heads, queries and keys, both polynomials), so the plaintexts are read once
// for all of them.
#include "context.h"
#include "kernels.h"
#include "modmath.cuh"

namespace cfhe {
namespace {

constexpr int kRotThreads = 256;

template <int SLOTS, int WORDS>
struct RotaryArgs {
  static constexpr int kSlots = SLOTS;  // pairs times rows of one launch
  static constexpr int kWords = WORDS;  // pairs times limbs of one launch (constants)
  int n_rows, n_pairs, n_limbs;
  uint32_t q[kMaxLimbs], nqinv[kMaxLimbs];
  RotarySlot slot[SLOTS];
  union {
    struct {
      const uint32_t *cos, *sin;
    } pt[WORDS];
    struct {
      uint32_t cos, sin;
    } word[WORDS];
  };
};

__device__ __forceinline__ uint32_t turn(uint32_t a, uint32_t x, uint32_t b, uint32_t y, uint32_t q, uint32_t nq) {
  return mont_reduce((uint64_t)a * x + (uint64_t)b * y, q, nq);  // at most 2 q^2 < q 2^32
}
__device__ __forceinline__ uint4 turn4(uint4 a, uint4 x, uint4 b, uint4 y, uint32_t q, uint32_t nq) {
  return make_uint4(turn(a.x, x.x, b.x, y.x, q, nq), turn(a.y, x.y, b.y, y.y, q, nq),
                    turn(a.z, x.z, b.z, y.z, q, nq), turn(a.w, x.w, b.w, y.w, q, nq));
}

template <bool CONST, typename Args>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const __grid_constant__ Args a) {
  pdl_launch_dependents();
  pdl_wait();
  const int l = blockIdx.y, i = blockIdx.z;
  const size_t at = (size_t)l * (kN / 4) + blockIdx.x * kRotThreads + threadIdx.x;
  const uint32_t q = a.q[l], nq = a.nqinv[l];
  uint4 c, s;
  if constexpr (CONST) {
    const uint32_t wc = a.word[i * a.n_limbs + l].cos, ws = a.word[i * a.n_limbs + l].sin;
    c = make_uint4(wc, wc, wc, wc);
    s = make_uint4(ws, ws, ws, ws);
  } else {
    c = reinterpret_cast<const uint4 *>(a.pt[i].cos)[at];
    s = reinterpret_cast<const uint4 *>(a.pt[i].sin)[at];
  }
  const uint4 ms = make_uint4(q - s.x, q - s.y, q - s.z, q - s.w);  // in (0, q]
#pragma unroll 2
  for (int r = 0; r < a.n_rows; r++) {
    const RotarySlot &o = a.slot[r * a.n_pairs + i];
    const uint4 u = reinterpret_cast<const uint4 *>(o.u)[at], v = reinterpret_cast<const uint4 *>(o.v)[at];
    reinterpret_cast<uint4 *>(o.yu)[at] = turn4(c, u, ms, v, q, nq);
    reinterpret_cast<uint4 *>(o.yv)[at] = turn4(s, u, c, v, q, nq);
  }
}

// Launches pairs [i0, i1) of rows [r0, r1)
template <typename Args>
int launch_part(const Context &ctx, const RotaryCall &call, int i0, int i1, int r0, int r1) {
  Args a;
  a.n_rows = r1 - r0;
  a.n_pairs = i1 - i0;
  a.n_limbs = call.n_limbs;
  for (int l = 0; l < call.n_limbs; l++) {
    a.q[l] = ctx.q[call.gidx[l]];
    a.nqinv[l] = ctx.nqinv[call.gidx[l]];
  }
  for (int r = r0; r < r1; r++)
    for (int i = i0; i < i1; i++)
      a.slot[(r - r0) * a.n_pairs + i - i0] = call.slots[(size_t)r * call.n_pairs + i];
  const dim3 grid(kN / 4 / kRotThreads, call.n_limbs, a.n_pairs), block(kRotThreads);
  if (call.cos_c) {
    for (int i = i0; i < i1; i++)
      for (int l = 0; l < call.n_limbs; l++) {
        const size_t from = (size_t)i * call.n_limbs + l;
        a.word[(i - i0) * call.n_limbs + l] = {call.cos_c[from] % a.q[l], call.sin_c[from] % a.q[l]};
      }
    CFHE_CUDA(launch_kernel(ctx.use_pdl, rotary_kernel<true, Args>, grid, block, 0, ctx.stream, a));
  } else {
    for (int i = i0; i < i1; i++) a.pt[i - i0] = {call.cos[i], call.sin[i]};
    CFHE_CUDA(launch_kernel(ctx.use_pdl, rotary_kernel<false, Args>, grid, block, 0, ctx.stream, a));
  }
  return 0;
}

}  // namespace

int launch_rotary(const Context &ctx, const RotaryCall &call) {
  // Operand tables travel as kernel parameters: 512 pairs x rows and as many
  // constants or plaintext pointers a launch
  using Args = RotaryArgs<512, 512>;
  const int per_pair = call.cos_c ? call.n_limbs : 1;
  const int pairs = min(call.n_pairs, Args::kWords / per_pair);
  for (int i0 = 0; i0 < call.n_pairs; i0 += pairs) {
    const int i1 = min(call.n_pairs, i0 + pairs), rows = Args::kSlots / (i1 - i0);
    for (int r0 = 0; r0 < call.n_rows; r0 += rows)
      if (int r = launch_part<Args>(ctx, call, i0, i1, r0, min(call.n_rows, r0 + rows))) return r;
  }
  CFHE_CUDA(cudaGetLastError());
  return 0;
}

}  // namespace cfhe
