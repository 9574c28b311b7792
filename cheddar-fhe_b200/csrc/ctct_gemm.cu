// Matrix product of ciphertexts, three-part results:
//   D[i][j] = w[i][j] (*) sum_t L[i][t] (x) R[t][j],
// (x) the tensor product (b b', b a' + a b', a a') and w an optional weight per
// result, a plaintext polynomial or one constant per limb: the scores and the
// weighted values of (decayed linear) attention over encrypted tokens. Words as
// from cfhe_tensor_accum followed by a plaintext or constant product.
//
// For every word position this is an m x k by k x n matrix product over Z_q, a
// small one with other operands at each position. Result by result each operand
// word would be read once per result that it enters; here a block owns a tile of
// results on C positions and every word is read once per tile. (The product of the
// transposes is taken where m > n: the tensor product commutes, so m <= n below.)
// Sixteen warps share the operand rows (C words of a polynomial) in a ring of
// shared-memory stages. The stages of a block's tiles form one pipeline: copies
// run ahead of the products over tile ends, and the pointers ahead of the copies.
//
// C is 64 or more: every row is another page, and an SM gets to a page that it did
// not visit shortly before about every eight clocks, so rows of 64 and 128 bytes come
// at 2.5 and 4.5 TB/s at most, of 256 bytes at 6.4 to 7.0 (8.9 from L2).
//
// m <= 2: bound by reading R, whose words enter one or two results, where there are
// terms enough: 0.73 to 0.83 of the copy rate for one row and 60 terms or more, 0.65
// for 2 x 64 x 64. Where a block has few stages, by the latency of the first and of the
// stores: 0.45 for 2 x 9 x 13, 0.35 for 1 x 5 x 9.
//
// m >= 3: bound by the multipliers. A 32 x 32 + 64-bit multiply-add is three instructions
// here, and 64-bit sums of products have to be folded; so a sum T of products is kept twice, as
// its low 32 bits (32-bit multiply-adds) and as a double (rounded), one instruction
// each:  T mod q = T - q round(T / q), which only needs the low bits of T and a T / q
// that is off by less than a quarter. Three products a term: b a' + a b' comes from the
// product of the sums. The two kinds of multiply-add hold each other up. 24 of each for
// four warps, operands in registers: the 32-bit ones take 270 clocks, the double ones
// 387 (221 to 283 if no operand were subnormal, as those of tiny() are), both 712 (644
// to 661), more than one after the other; 592 with operands from shared memory, which
// is 3.8 of the 5.4 ms of 8 x 64 x 16 on 14 limbs. No pipe is full meanwhile and the
// stall is in dispatch; what causes it is not known. With 64-bit sums it took 6.6 ms,
// with four products a term and each result's weight fetched on its own 6.0; bytes on the tensor cores
// (tcgen05.mma wants 64 rows, a position has 2 n; mma.sync with operands split into byte
// planes, whose seven 32-bit sums a result only fit tensor memory and leave a tile of
// 4 x 8) 6.1; copies of whole rows that the warps wait for one by one, so that they may
// be stages apart, 6.6.
#include <math.h>

#include "context.h"
#include "kernels.h"
#include "modmath.cuh"

namespace cfhe {
namespace {

// n / d for n below 2^31
struct Divisor {
  uint32_t d, mul, shift;
  void set(uint32_t by) {
    d = by;
    shift = 31;
    while ((1ull << (shift - 31)) < by) shift++;
    mul = (uint32_t)(((1ull << shift) + by - 1) / by);
  }
  __device__ __forceinline__ int quotient(int n) const { return (int)((uint64_t)(uint32_t)n * mul >> shift); }
};

struct CtctPlan {
  Divisor m_tiles, tiles;  // tiles along m, in all
  int items;               // tiles x groups of positions x limbs
};

__device__ __forceinline__ uint32_t cc_smem(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

// Tile and first position of an item
struct Where {
  int i0, j0, l, position;
};
template <typename T>
__device__ __forceinline__ Where where(const CtctPlan &p, int item) {
  constexpr int kChunks = kN / T::C;
  const int rest = p.tiles.quotient(item), tile = item - rest * (int)p.tiles.d;
  const int tj = p.m_tiles.quotient(tile), ti = tile - tj * (int)p.m_tiles.d;
  return {ti * T::kBm, tj * T::kBn, rest / kChunks, rest % kChunks * T::C};
}

// The asynchronous copies of a block. T: kBm x kBn results of a tile, C positions,
// kTerms terms and kStages stages of the ring (kStage words each), kRowsT rows of a
// term, those of R before kRowsR; entry(r, part): column or row of the tile and part
// of row r; kWarps warps.
template <typename T>
struct Feed {
  static constexpr int kThreads = 32 * T::kWarps;
  static constexpr int kRows = T::kTerms * T::kRowsT, kPieces = T::C / 4;  // 16-byte pieces of a row
  static constexpr int kCopies = (kRows * kPieces + kThreads - 1) / kThreads;
  static constexpr int kPointers = (kRows + kThreads - 1) / kThreads;
  const CtctArgs &a;
  const CtctPlan &p;
  uint32_t *const ring;
  const uint32_t **const pointers;  // of the rows of 2 kStages stages, a ring of its own
  const int tid, n_stages;
  // pointers
  int p_item, p_s = 0, p_slot = 0;
  const uint32_t *const *p_at[kPointers];  // null: no such row
  // copies
  int c_item, c_s = 0, c_slot = 0, c_pslot = 0;
  size_t c_at = 0;

  __device__ __forceinline__ Feed(const CtctArgs &args, const CtctPlan &plan, uint32_t *smem)
      : a(args), p(plan), ring(smem), pointers(reinterpret_cast<const uint32_t **>(smem + T::kStages * T::kStage)),
        tid(threadIdx.x), n_stages((args.k + T::kTerms - 1) / T::kTerms), p_item(blockIdx.x), c_item(blockIdx.x) {}

  // The pointers of one stage out of the tables, kStages stages before it is copied;
  // a row that does not exist, or is past the last term, gets a null.
  __device__ __forceinline__ void point() {
#pragma unroll
    for (int x = 0; x < kPointers; x++) {
      const int row = tid + x * kThreads, t = row / T::kRowsT, r = row % T::kRowsT;
      if (kRows % kThreads && row >= kRows) break;
      const bool right = r < T::kRowsR;
      const int width = right ? a.n : a.m;
      if (p_s == 0) {
        const Where w = where<T>(p, p_item);
        int part;
        const int e = T::entry(r, part) + (right ? w.j0 : w.i0);
        const CtctPair *const tab = (right ? a.right : a.left) + (size_t)t * width + e;
        p_at[x] = p_item < p.items && e < width ? reinterpret_cast<const uint32_t *const *>(tab) + part : nullptr;
      }
      const bool there = p_at[x] && p_s * T::kTerms + t < a.k;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(cc_smem(pointers + p_slot * kRows + row)),
                   "l"(there ? (const void *)p_at[x] : (const void *)a.right), "r"(there ? 8 : 0)
                   : "memory");
      if (p_at[x]) p_at[x] += 2 * T::kTerms * width;
    }
    if (++p_s == n_stages) {
      p_s = 0;
      p_item += gridDim.x;
    }
    p_slot = p_slot + 1 == 2 * T::kStages ? 0 : p_slot + 1;
  }
  // One stage on its way. Nothing is copied where there is no row or term: what the
  // ring holds there is not used.
  __device__ __forceinline__ void copy() {
    if (c_s == 0) {
      const Where w = where<T>(p, c_item);
      c_at = (size_t)w.l * kN + w.position + tid % kPieces * 4;
    }
    if (c_item < p.items) {
      const uint32_t stage = cc_smem(ring + c_slot * T::kStage + tid % kPieces * 4);
      const uint32_t *const *const from = pointers + c_pslot * kRows + tid / kPieces;
#pragma unroll
      for (int x = 0; x < kCopies; x++) {
        const int row = tid / kPieces + x * (kThreads / kPieces);
        if (kRows * kPieces % kThreads && row >= kRows) break;
        const uint32_t *const src = from[x * (kThreads / kPieces)];
        if (src)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(stage + 4 * row * T::C), "l"(src + c_at)
                       : "memory");
      }
    }
    if (++c_s == n_stages) {
      c_s = 0;
      c_item += gridDim.x;
    }
    c_slot = c_slot + 1 == T::kStages ? 0 : c_slot + 1;
    c_pslot = c_pslot + 1 == 2 * T::kStages ? 0 : c_pslot + 1;
  }
  __device__ __forceinline__ void step() {
    copy();
    point();
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  __device__ __forceinline__ void start() {  // pointers of kStages stages, copies of one less
    for (int s = 0; s < T::kStages; s++) point();
    asm volatile("cp.async.commit_group;\n\tcp.async.wait_all;" ::: "memory");
    __syncthreads();
    for (int s = 0; s + 1 < T::kStages; s++) step();
  }
  __device__ __forceinline__ void arrived() {  // the oldest step, for every thread
    asm volatile("cp.async.wait_group %0;" ::"n"(T::kStages - 2) : "memory");
    __syncthreads();
  }
};

// A 32-bit integer as the double that is the integer times 2^-1074
__device__ __forceinline__ double tiny(uint32_t v) { return __hiloint2double(0, (int)v); }

// A sum of products of residues: its low 32 bits, and 2^-1074 times the sum, rounded.
// Up to kSumTerms terms of two products, or of one of sums of two residues: the sum is
// below 1024 q^2, its roundings together (512 of sums below 512 q^2, 256 of sums below
// 1024 q^2) less than 2^18 q^2 2^-53, that is 2^-4 of a quotient by q, and the product
// with inv and the rounding of inv less than 2^-11.
constexpr int kSumTerms = 256;
struct Sum {
  uint32_t lo;
  double f;
  __device__ __forceinline__ void add(uint32_t a, uint32_t b, double b_f) {
    lo += a * b;
    f = fma(tiny(a), b_f, f);
  }
  // the sum mod q. inv: 2^1000 / q; adding 1.5 2^52 in the scale of the product leaves
  // the rounded quotient in the low bits
  __device__ __forceinline__ uint32_t mod(uint32_t q, double inv) const {
    const double magic = __hiloint2double((1023 + 52 - 74) << 20 | 0x80000, 0);  // 1.5 * 2^(52 - 74)
    const uint32_t r = lo - (uint32_t)__double2loint(fma(f, inv, magic)) * q;  // in (-q, q)
    return min(r, r + q);
  }
};

// Thread tiles of MT x NT results; WM warps along m, POSITIONS / 32 groups of
// positions, the other warps along n; stages of TERMS terms
template <int MT, int NT, int WM, int POSITIONS, int TERMS>
struct SumsTile {
  static constexpr int kWarps = 16, C = POSITIONS, kGroups = C / 32, kWn = kWarps / (kGroups * WM);
  static constexpr int kBm = MT * WM, kBn = NT * kWn, kTerms = TERMS;
  static constexpr int kRowsR = 2 * kBn, kRowsT = kRowsR + 2 * kBm, kStage = kTerms * kRowsT * C;
  static constexpr int kFit = 220 * 1024 / (kStage * 4 + 2 * kTerms * kRowsT * 8);
  static constexpr int kStages = kFit < 8 ? kFit : 8;
  static constexpr int kBytes = kStages * (kStage * 4 + 2 * kTerms * kRowsT * 8);
  static __device__ __forceinline__ int entry(int r, int &part) {
    part = r & 1;
    return (r < kRowsR ? r : r - kRowsR) >> 1;
  }
};
template <int MT, int NT, int WM, int POSITIONS, int TERMS>
__global__ void __launch_bounds__(512, 1) ctct_sums_kernel(const __grid_constant__ CtctArgs a,
                                                           const __grid_constant__ CtctPlan p) {
  using T = SumsTile<MT, NT, WM, POSITIONS, TERMS>;
  constexpr bool kThree = MT > 2;  // three products a term
  extern __shared__ __align__(16) uint32_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  pdl_wait();
  Feed<T> feed(a, p, smem);
  feed.start();
  const int group = warp % T::kGroups, wj = warp / T::kGroups % T::kWn, wi = warp / (T::kGroups * T::kWn);
  const int my_r = 2 * wj * NT * T::C + 32 * group + lane, my_l = (T::kRowsR + 2 * wi * MT) * T::C + 32 * group + lane;
  int slot = 0;
  for (int item = blockIdx.x; item < p.items; item += gridDim.x) {
    const Where w = where<T>(p, item);
    const int i0 = w.i0 + wi * MT, j0 = w.j0 + wj * NT;
    const uint32_t q = a.q[w.l], nq = a.nqinv[w.l];
    const double inv = a.inv[w.l];
    Sum s0[MT][NT], s1[MT][NT], s2[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
      for (int j = 0; j < NT; j++) s0[i][j] = s1[i][j] = s2[i][j] = {0u, 0.0};
    for (int s = 0; s < feed.n_stages; s++) {
      feed.arrived();  // and all have left the stage before
      feed.step();
      const uint32_t *const stage = smem + slot * T::kStage;
      slot = slot + 1 == T::kStages ? 0 : slot + 1;
      if (i0 >= a.m || j0 >= a.n) continue;
#pragma unroll
      for (int u = 0; u < T::kTerms; u++) {
        if (u > 0 && s * T::kTerms + u >= a.k) break;
        const uint32_t *const lp = stage + my_l + u * T::kRowsT * T::C, *const rp = stage + my_r + u * T::kRowsT * T::C;
        uint32_t lb[MT], la[MT], ls[MT];
#pragma unroll
        for (int i = 0; i < MT; i++) {
          lb[i] = lp[2 * i * T::C];
          la[i] = lp[(2 * i + 1) * T::C];
          ls[i] = lb[i] + la[i];
        }
#pragma unroll
        for (int j = 0; j < NT; j++) {
          const uint32_t rb = rp[2 * j * T::C], ra = rp[(2 * j + 1) * T::C], rs = rb + ra;
          const double rb_f = rb, ra_f = ra, rs_f = rb_f + ra_f;
#pragma unroll
          for (int i = 0; i < MT; i++) {
            s0[i][j].add(lb[i], rb, rb_f);
            if (kThree) {
              s1[i][j].add(ls[i], rs, rs_f);
            } else {
              s1[i][j].add(lb[i], ra, ra_f);
              s1[i][j].add(la[i], rb, rb_f);
            }
            s2[i][j].add(la[i], ra, ra_f);
          }
        }
      }
      if ((s + 1) * TERMS % kSumTerms == 0) {
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
          for (int j = 0; j < NT; j++)
            for (Sum *x : {&s0[i][j], &s1[i][j], &s2[i][j]}) {
              const uint32_t r = x->mod(q, inv);
              *x = {r, tiny(r)};
            }
      }
    }
    // The weights are on their way before the first is waited for, the pointers of a
    // result before the one before it is stored.
    const size_t at = (size_t)w.l * kN + w.position + 32 * group + lane;
    if (i0 >= a.m || j0 >= a.n) continue;
    const size_t o0 = (size_t)i0 * a.n + j0;
    auto there = [&](int i, int j) { return i0 + i < a.m && j0 + j < a.n; };
    uint32_t v[MT][NT];
    const uint32_t *weight[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
      for (int j = 0; j < NT; j++) weight[i][j] = there(i, j) ? a.out[o0 + i * a.n + j].weight : nullptr;
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
      for (int j = 0; j < NT; j++)
        v[i][j] = weight[i][j]                 ? weight[i][j][at]
                  : a.consts && there(i, j) ? a.consts[(o0 + i * a.n + j) * a.n_limbs + w.l]
                                            : 0;
    CtctOut next = a.out[o0];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
      for (int j = 0; j < NT; j++) {
        const CtctOut to = next;
        const int ni = j + 1 < NT ? i : i + 1, nj = j + 1 < NT ? j + 1 : 0;
        if (ni < MT && there(ni, nj)) next = a.out[o0 + ni * a.n + nj];
        const uint32_t t0 = s0[i][j].mod(q, inv), t2 = s2[i][j].mod(q, inv);
        uint32_t t1 = s1[i][j].mod(q, inv);
        if (kThree) {
          t1 -= t0;
          t1 = min(t1, t1 + q);
          t1 -= t2;
          t1 = min(t1, t1 + q);
        }
        uint32_t d0 = mont_reduce(t0, q, nq), d1 = mont_reduce(t1, q, nq), d2 = mont_reduce(t2, q, nq);
        if (to.weight || a.consts) {
          d0 = mont_mul(d0, v[i][j], q, nq);
          d1 = mont_mul(d1, v[i][j], q, nq);
          d2 = mont_mul(d2, v[i][j], q, nq);
        }
        if (there(i, j)) {
          to.d0[at] = d0;
          to.d1[at] = d1;
          to.d2[at] = d2;
        }
      }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// ---- launches
template <typename T, typename Kernel>
int launch_tiles(const Context &ctx, const CtctArgs &a, Kernel kernel, PerDeviceOnce &once) {
  if (int r = once.run(ctx.device, [&] {
        CFHE_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, T::kBytes));
        return 0;
      }))
    return r;
  CtctPlan p;
  p.m_tiles.set((a.m + T::kBm - 1) / T::kBm);
  p.tiles.set(p.m_tiles.d * ((a.n + T::kBn - 1) / T::kBn));
  p.items = p.tiles.d * (kN / T::C) * a.n_limbs;
  CFHE_CUDA(launch_kernel(ctx.use_pdl, kernel, dim3(min(p.items, ctx.num_sms)), dim3(32 * T::kWarps), T::kBytes,
                          ctx.stream, a, p));
  return 0;
}

template <int MT, int NT, int WM, int POSITIONS, int TERMS>
int launch_sums(const Context &ctx, const CtctArgs &a) {
  using T = SumsTile<MT, NT, WM, POSITIONS, TERMS>;
  static_assert(T::kStages >= 3, "copies ahead of the products");
  static PerDeviceOnce once;
  return launch_tiles<T>(ctx, a, ctct_sums_kernel<MT, NT, WM, POSITIONS, TERMS>, once);
}

}  // namespace

// args.m <= args.n. Tiles of 8 columns (4 where there are no more, so that no warp is
// without results) and as many positions as the warps then have room for: longer rows
// and no columns without results are worth more than reading L once per 8 columns
// instead of once per 32. Rows of 1 KB and 8 columns against 256 bytes and 32, on 7
// limbs: 1 x 60 x 64 1910 -> 1924 us, 1 x 16 x 17 244 -> 199, 2 x 64 x 33 2688 -> 1610;
// 4 x 16 x 64 (512 bytes against 256, 16 columns) 1379 -> 1397, 3 x 16 x 17 689 -> 447;
// 4 columns against 8: 2 x 5 x 3 47 -> 39, 4 x 64 x 4 406 -> 338. With m >= 5 L is half of the
// rows: 8 x 64 x 8 947 us, with 512 bytes and 4 columns 1150.
int launch_ctct_gemm(const Context &ctx, const CtctArgs &args) {
  CtctArgs a = args;
  for (int l = 0; l < a.n_limbs; l++) a.inv[l] = ldexp(1.0 / a.q[l], 1000);
  const bool narrow = a.n <= 4;
  int r;
  if (a.m == 1)
    r = narrow ? launch_sums<1, 2, 1, 256, 4>(ctx, a) : launch_sums<1, 4, 1, 256, 2>(ctx, a);
  else if (a.m == 2)
    r = narrow ? launch_sums<2, 2, 1, 256, 4>(ctx, a) : launch_sums<2, 4, 1, 256, 2>(ctx, a);
  else if (a.m <= 4)
    r = narrow ? launch_sums<4, 2, 1, 256, 2>(ctx, a) : launch_sums<4, 2, 1, 128, 4>(ctx, a);
  else
    r = launch_sums<4, 2, 2, 64, 8>(ctx, a);
  if (r) return r;
  CFHE_CUDA(cudaGetLastError());
  return 0;
}

}  // namespace cfhe
