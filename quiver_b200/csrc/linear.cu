// Linear adapters: y = act(x W^T + bias) + residual, and its gradients
//   dz = dy * act'(z),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz     (z = x W^T + bias).
//
// The three products run in one tensor-core kernel, product_kernel: D[m][n] = sum_k A[m][k] B[n][k]
// with either operand stored along k or across it, so that no operand is transposed in memory.
// 16-bit operands are multiplied as they are. Float32 operands are split into 16-bit planes whose
// sum they are, and the product is the sum of the plane products that reach float32's last bit:
// * x W^T: every row is scaled by a power of two that brings its largest element below 2^15, then
//   split into two float16 (11 + 11 bits and the sign of the remainder: off by at most 2^-23 of the
//   element, or 2^-39 of the row's largest where that is more), three products; the product of the
//   two low planes, at most 2^-22 of a term, is left out. The scales come off each result exactly.
//   The sums run along the rows, so a row's scale is a result's. Rows whose elements differ too
//   widely for that (split_rows_kernel) take the next form, with another scale (lifted).
// * dz W and dz^T x, whose sums run across the rows: three bfloat16 planes (8 + 8 + 8 bits, the
//   element itself down to the planes' last bit, 2^-133), six products; what is left out is at most
//   2^-24 of a term. Smallest products first: a sum next to float32's end is not passed on the way.
// Batches of a few rows (single queries) take a kernel that reads the weights once with plain
// loads.
#include <algorithm>
#include <mutex>

#include "embed.cuh"
#include "linear.cuh"
#include "tc_common.cuh"

namespace qv {
namespace {

using dev::Pack;

// ---- packing: operands TMA cannot read in place, and float32 as three bfloat16 planes ------------

// Infinities in the parts of float32 values: the last part holds it and the first has 1 with its sign.
// The last part of one operand meets only the first of the other, which is zero only where the value
// is (bfloat16: tiny values round away from zero; float16: or is below 2^-39 of its row's largest): so
// every infinite term comes out once, with its sign, or as NaN against a zero, and nothing else of the
// sum is infinite.

// x as a sum of three bfloat16: each is the rounded remainder of the ones before, and the last
// remainder has at most 8 bits left, so that the sum is x itself. The largest finite values round
// to infinity in the first plane and are cut there instead; NaN stays in the first.
__device__ __forceinline__ void split3(float x, __nv_bfloat16 (&p)[3]) {
  p[0] = __float2bfloat16_rn(x);
  p[1] = p[2] = __float2bfloat16_rn(0.0f);
  if ((__float_as_uint(x) & 0x7f800000u) == 0x7f800000u) {
    if (x == x) {
      p[0] = __float2bfloat16_rn(copysignf(1.0f, x));
      p[2] = __float2bfloat16_rn(x);
    }
    return;
  }
  if (__hisinf(p[0])) p[0] = __float2bfloat16_rz(x);
  if (x != 0.0f && __bfloat162float(p[0]) == 0.0f)
    p[0] = __float2bfloat16_rn(copysignf(0x1p-133f, x));
  const float r = x - __bfloat162float(p[0]);
  p[1] = __float2bfloat16_rn(r);
  p[2] = __float2bfloat16_rn(r - __bfloat162float(p[1]));
}

// The element type the tensor core multiplies for values of type T, and its planes.
template <class T>
struct Operand {
  using type = T;
  static constexpr int kPlanes = 1;
};
template <>
struct Operand<float> {
  using type = __nv_bfloat16;
  static constexpr int kPlanes = 3;
};

// Writes kV consecutive values as an operand at dst[at], planes `plane` elements apart.
template <class T, int kV>
__device__ __forceinline__ void put_operand(const float (&x)[kV],
                                            typename Operand<T>::type* __restrict__ dst,
                                            int64_t plane, int64_t at) {
  if constexpr (sizeof(T) == 4) {
    Pack<__nv_bfloat16, kV> y[3];
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      __nv_bfloat16 p[3];
      split3(x[j], p);
#pragma unroll
      for (int i = 0; i < 3; ++i) y[i].v[j] = p[i];
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) dev::store_pack<__nv_bfloat16, kV>(dst + i * plane + at, y[i]);
  } else {
    Pack<T, kV> y;
#pragma unroll
    for (int j = 0; j < kV; ++j) y.v[j] = dev::from_f32<T>(x[j]);
    dev::store_pack<T, kV>(dst + at, y);
  }
}

// One matrix to pack: rows x cols values, written with rows of ld (a multiple of 8) elements.
struct PackJob {
  const void* src;
  void* dst;
  int64_t rows, cols, stride, ld;
  int* exponents;  // scaled rows: each row's scale was 2^-exponent
};

// A row's exponent as three bfloat16 planes, from its exponent as two float16 planes. The planes end
// at 2^-133, bfloat16's last bit, so that elements below 2^-110 would lose bits: rows whose largest
// is below 2^-20 are brought up to that, which keeps every product with another row in range.
__device__ __forceinline__ int lifted(int exponent) { return min(0, exponent + 34); }

// float32 rows scaled and split into two float16 planes, or (kPlanes) lifted and split into three
// bfloat16 ones; one warp per row, which keeps up to 32 * kSplitHeld pieces of it in registers and
// reads what is more a second time.
//
// The planes hold an element to 2^-23 of itself or 2^-39 of the row's largest, X. The second part
// adds up to 2^-39 (X sum|w| + W sum|x|) <= 2^-38 k X W to a result, which is nothing beside
// S = sum |x||w| unless the large elements of x meet small ones of w. So the rows tell which share
// of their elements lies within 2^-6 of their largest, in 256ths: where the least shares p of x and
// q of w have p + q >= 1 + 1/8, at least k / 8 terms of every result have both factors there,
// S >= 2^-15 k X W, and the addition is at most 2^-23 S. Otherwise the call's product takes three
// bfloat16 planes (choose_planes_kernel). Vectors of normally distributed elements have shares of
// 0.9 and more, half of them zero (ReLU) about 0.45. Rows of zeros and rows that hold infinity or
// NaN (whose results are none but these) tell 256. Three blocks an SM: counting
// took the kernel to 126 registers and from 12.6 to 15.8 us for 10,000 + 768 rows of 768; held to 80
// it takes 13.0.
constexpr int kSplitHeld = 8, kSplitBlocks = 148 * 8;
constexpr uint32_t kShareOne = 256, kSharesNeeded = kShareOne + kShareOne / 8;
template <int kV, bool kPlanes>
__global__ void __launch_bounds__(256, 3)
    split_rows_kernel(const PackJob j0, const PackJob j1, uint32_t* __restrict__ shares) {
  dev::allow_next();
  const PackJob& j = blockIdx.y == 0 ? j0 : j1;
  const int lane = threadIdx.x & 31;
  uint32_t least = kShareOne;
  const int64_t plane = j.rows * j.ld;
  const int64_t warps = gridDim.x * 8ll;
  for (int64_t r = blockIdx.x * 8ll + (threadIdx.x >> 5); r < j.rows; r += warps) {
    const float* src = static_cast<const float*>(j.src) + r * j.stride;
    __half* dst = static_cast<__half*>(j.dst) + r * j.ld;
    Pack<float, kV> held[kSplitHeld];
    uint32_t top = 0;  // bits of the largest magnitude (which order like the magnitudes)
    auto see = [&](const Pack<float, kV>& x) {
#pragma unroll
      for (int v = 0; v < kV; ++v) top = max(top, __float_as_uint(x.v[v]) & 0x7fffffffu);
    };
    const int64_t last = j.cols - kV;  // pieces past the row's end read its last: no branches
#pragma unroll
    for (int h = 0; h < kSplitHeld; ++h)
      held[h] = dev::load_pack<float, kV>(src + min(static_cast<int64_t>((h * 32 + lane) * kV), last));
#pragma unroll
    for (int h = 0; h < kSplitHeld; ++h) see(held[h]);
    constexpr int64_t kHeld = kSplitHeld * 32 * kV;
#pragma unroll 4
    for (int64_t c = kHeld + lane * kV; c < j.cols; c += 32 * kV)
      see(dev::load_pack<float, kV>(src + c));
    top = __reduce_max_sync(dev::kFull, top);
    const bool odd = top >= 0x7f800000u;  // infinity or NaN among them: the largest of the others
    if (odd) {
      top = 0;
#pragma unroll 1
      for (int64_t c = lane; c < j.cols; c += 32) {
        const uint32_t bits = __float_as_uint(src[c]) & 0x7fffffffu;
        top = max(top, bits < 0x7f800000u ? bits : 0u);
      }
      top = __reduce_max_sync(dev::kFull, top);
    }
    const int shift = top == 0 ? 0 : min(14 + 127 - static_cast<int>(top >> 23), 126);
    const int exponent = kPlanes ? lifted(-shift) : -shift;
    const float scale = __uint_as_float(static_cast<uint32_t>(127 - exponent) << 23);
    if (lane == 0) j.exponents[r] = exponent;
    const float from = __uint_as_float(top) * scale * 0x1p-6f;
    uint32_t large = 0;
    auto split = [&](const Pack<float, kV>& x, int64_t c) {
      if constexpr (kPlanes) {
        float y[kV];
#pragma unroll
        for (int v = 0; v < kV; ++v) y[v] = x.v[v] * scale;
        put_operand<float, kV>(y, static_cast<__nv_bfloat16*>(j.dst), plane, r * j.ld + c);
      } else {
        Pack<__half, kV> hi, lo;
#pragma unroll
        for (int v = 0; v < kV; ++v) {
          const float y = x.v[v] * scale;
          large += fabsf(y) >= from;
          hi.v[v] = __float2half_rn(y);
          lo.v[v] = __float2half_rn(y - __half2float(hi.v[v]));
        }
        dev::store_pack<__half, kV>(dst + c, hi);
        dev::store_pack<__half, kV>(dst + plane + c, lo);
      }
    };
#pragma unroll
    for (int h = 0; h < kSplitHeld; ++h) {
      const int64_t c = (h * 32ll + lane) * kV;
      if (c < j.cols) split(held[h], c);
    }
#pragma unroll 4
    for (int64_t c = kHeld + lane * kV; c < j.cols; c += 32 * kV)
      split(dev::load_pack<float, kV>(src + c), c);
    if (!kPlanes && odd) {  // infinities once more, in their own form
      __syncwarp();
#pragma unroll 1
      for (int64_t c = lane; c < j.cols; c += 32) {
        if ((__float_as_uint(src[c]) & 0x7fffffffu) != 0x7f800000u) continue;
        dst[c] = __float2half_rn(copysignf(1.0f, src[c]));
        dst[plane + c] = __float2half_rn(src[c]);
      }
    }
    const uint32_t count = __reduce_add_sync(dev::kFull, large);
    if (top != 0 && !odd)
      least = min(least, count * kShareOne / static_cast<uint32_t>(j.cols));
  }
  if constexpr (kPlanes) {
    dev::wait_previous();
    return;
  }
  __shared__ uint32_t s_least[8];
  if (lane == 0) s_least[threadIdx.x >> 5] = least;
  __syncthreads();
  if (threadIdx.x < 8) {
    least = __reduce_min_sync(0xffu, s_least[threadIdx.x]);
    if (threadIdx.x == 0) shares[blockIdx.y * gridDim.x + blockIdx.x] = least;
  }
  dev::wait_previous();
}

// Up to two matrices in one launch (blockIdx.y). Bound by memory: every thread moves kV values of
// kPackRows rows at a time.
constexpr int kPackRows = 4;
// kLift: rows whose scale for the float16 planes was 2^-exponent are lifted by 2^-lifted(exponent).
template <class T, int kV, bool kLift>
__device__ __forceinline__ void pack_rows(const PackJob& j) {
  using O = typename Operand<T>::type;
  const T* src = static_cast<const T*>(j.src);
  O* dst = static_cast<O*>(j.dst);
  const uint32_t per_row = static_cast<uint32_t>((j.cols + kV - 1) / kV);
  const int64_t plane = j.rows * j.ld;
  const int64_t groups = (j.rows + kPackRows - 1) / kPackRows;
  const int64_t total = groups * per_row;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const int64_t r0 = i / per_row * kPackRows;
    const int64_t c = (i - i / per_row * per_row) * kV;
    Pack<T, kV> x[kPackRows];
#pragma unroll
    for (int u = 0; u < kPackRows; ++u)
      x[u] = dev::load_pack<T, kV>(src + min(r0 + u, j.rows - 1) * j.stride + c);
#pragma unroll
    for (int u = 0; u < kPackRows; ++u) {
      if (r0 + u >= j.rows) break;
      float f[kV];
#pragma unroll
      for (int v = 0; v < kV; ++v) f[v] = dev::to_f32<T>(x[u].v[v]);
      if constexpr (kLift) {
        const float scale = __int_as_float((127 - lifted(j.exponents[r0 + u])) << 23);
#pragma unroll
        for (int v = 0; v < kV; ++v) f[v] *= scale;
      }
      put_operand<T, kV>(f, dst, plane, (r0 + u) * j.ld + c);
    }
  }
}
template <class T, int kV>
__global__ void __launch_bounds__(256) pack_kernel(const PackJob j0, const PackJob j1) {
  dev::allow_next();
  pack_rows<T, kV, false>(blockIdx.y == 0 ? j0 : j1);
  // Chained after the dz kernel, whose results are not used here: its end is this kernel's.
  dev::wait_previous();
}

// Whether the two operands that split_rows_kernel made (in `blocks` blocks each) serve every
// result; where they do not, three bfloat16 planes of each in their place.
template <int kV>
__global__ void __launch_bounds__(256)
    choose_planes_kernel(const PackJob j0, const PackJob j1, const uint32_t* shares,
                         uint32_t blocks, int* wide) {
  dev::allow_next();
  dev::wait_previous();
  __shared__ uint32_t s_least[2][8];
  uint32_t a = kShareOne, b = kShareOne;
  for (uint32_t i = threadIdx.x; i < blocks; i += 256) {
    a = min(a, shares[i]);
    b = min(b, shares[blocks + i]);
  }
  a = __reduce_min_sync(dev::kFull, a);
  b = __reduce_min_sync(dev::kFull, b);
  if ((threadIdx.x & 31) == 0) {
    s_least[0][threadIdx.x >> 5] = a;
    s_least[1][threadIdx.x >> 5] = b;
  }
  __syncthreads();
  for (int w = 0; w < 8; ++w) {
    a = min(a, s_least[0][w]);
    b = min(b, s_least[1][w]);
  }
  const bool planes = a + b < kSharesNeeded;
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *wide = planes;
  if (planes) pack_rows<float, kV, true>(blockIdx.y == 0 ? j0 : j1);
}

// ---- the product kernel -----------------------------------------------------------------------------
// Warp-specialized and persistent: one thread feeds 128-byte-swizzled tiles of A and B through a
// ring of shared-memory stages with TMA, one thread issues the MMAs into one of two accumulators
// in tensor memory, and sixteen warps finish the other accumulator's elements meanwhile.
//
// The tensor core's float32 sums are cut, not rounded, several times in 16 terms: over k terms of one
// sign the result falls short by about k * 6.4e-9 of itself (2.6e-5 measured at k = 4096), and
// sums of random signs lose a fifth of that. So no sum stays there for more than `chunk` blocks of
// 64 terms: the epilogue warps then add it to one in their registers, rounding, while the next
// chunk's MMAs fill the other accumulator. Float32 products take chunks of 2 blocks (8e-7); 16-bit
// operands chunks of 128 for 16-bit results (5e-5, a fortieth of bfloat16's half step and a tenth of
// float16's), of 8 for float32 results (3.4e-6; chunks of 2 took 544 us for 32,768 x 1024 x 4096
// where one of 16 takes 247).
//
// Large products run in CTA pairs (tcgen05 cta_group::2): 256 x 256 tiles, each CTA loading its
// 128 rows of A and half of B. A CTA by itself would have to load 384 rows of operands for
// 128 x 256 results, 96 bytes per SM and cycle at full MMA rate; the pair loads 64.

constexpr int kBM = 128, kBK = 64;  // rows of A per CTA, k per stage
constexpr int kEpilogueWarps = 16;
constexpr int kProductThreads = 64 + 32 * kEpilogueWarps;  // producer, MMA, epilogue
constexpr int kPieceBytes = 4096;  // an epilogue warp's piece of the result: 32 rows x 128 bytes

template <int kBN, bool kPair>
struct Tile {
  static constexpr int kM = kPair ? 2 * kBM : kBM;           // rows of a tile
  static constexpr int kBRows = kPair ? kBN / 2 : kBN;       // rows of B loaded by one CTA
  static constexpr int kABytes = kBM * kBK * 2;
  static constexpr int kBBytes = kBRows * kBK * 2;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = kStageBytes >= 32768 ? 4 : 5;  // 6 measured no faster
  static constexpr size_t kSmem = static_cast<size_t>(kStages) * kStageBytes +
                                  kEpilogueWarps * kPieceBytes + 1024 + 512;
};

// Plane pairs of a product, smallest terms first: of three planes, of two, of one.
__constant__ int8_t kPairA[10] = {2, 0, 1, 1, 0, 0, 1, 0, 0, 0};
__constant__ int8_t kPairB[10] = {0, 2, 1, 0, 1, 0, 0, 1, 0, 0};
__device__ __forceinline__ int first_pair(int pairs) { return pairs == 6 ? 0 : (pairs == 3 ? 6 : 9); }
// v * 2^e for -252 <= e <= 252: in two steps, neither of which overflows or underflows before the
// result does.
__device__ __forceinline__ float times_pow2(float v, int e) {
  const int h = e >> 1;
  return v * __int_as_float((127 + h) << 23) * __int_as_float((127 + e - h) << 23);
}

struct ProductArgs {
  int64_t m, n;
  int pairs;              // plane pairs: 1, or 3 or 6 for float32
  const int* exp_a;       // scaled rows of A and B: their exponents, or nullptr
  const int* exp_b;
  int k_blocks;           // 64-wide blocks of k
  int tiles_m, tiles_n, splits, blocks_per_split;
  int chunk;              // blocks of k whose sum stays in tensor memory
  uint32_t idesc;
  uint32_t a_mn, b_mn;    // operand stored across k (MN-major)
  Epilogue ep;
  float* partial;         // splits > 1: [split][m][n] float32 sums, joined afterwards
};
// Up to two products of one launch (a layer's dx and dW), their tiles one list of work units.
struct ProductGroup {
  ProductArgs p[2];
  int units[2];
  // One float32 product whose operands are either scaled or three planes (maps.a[1], maps.b[1]):
  // the word that says so, and the instruction descriptor of the planes; or nullptr.
  const int* wide;
  uint32_t wide_idesc;
  long long wait_cycles;
  uint64_t drain_ns;
};
struct ProductMaps {
  CUtensorMap a[2], b[2], out[2], residual[2];
};

// A unit of work: product q, split, then tile row / column, columns fastest (a wave's CTAs share rows
// of A and all of B in L2), and the split's blocks of k.
struct Unit {
  int q, split, tm, tn, b0, b1;
};
__device__ __forceinline__ Unit unit_of(const ProductGroup& g, int u) {
  Unit w;
  w.q = u >= g.units[0];
  u -= w.q ? g.units[0] : 0;
  const ProductArgs& a = g.p[w.q];
  const int per = a.tiles_m * a.tiles_n;
  w.split = u / per;
  const int t = u - w.split * per;
  w.tm = t / a.tiles_n;
  w.tn = t - w.tm * a.tiles_n;
  w.b0 = w.split * a.blocks_per_split;
  w.b1 = min(a.k_blocks, w.b0 + a.blocks_per_split);
  return w;
}

// TMA loads; in a pair the bytes are counted on the leader's barrier (a shared::cluster address).
template <bool kPair>
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y,
                                            int z, uint32_t bar) {
  if constexpr (kPair)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, "
        "{%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
// One lane of a converged warp, the same each time.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}\n"
      : "=r"(p));
  return p != 0;
}
// 128-byte swizzled operand tiles. Along k: 64-element rows, 8-row groups 1024 bytes apart.
// Across k: [64 k][64 m-or-n] blocks of 8 KB (the leading offset), 8-k groups 1024 bytes apart.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, uint32_t across) {
  return (static_cast<uint64_t>(addr >> 4) & 0x3FFFull) |
         (static_cast<uint64_t>(across ? 8192 >> 4 : 1) << 16) | (64ull << 32) | (1ull << 46) |
         (2ull << 61);
}
template <bool kPair>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t acc) {
  if constexpr (kPair)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int x, int y, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(src)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// 16 columns of this warp's 32 TMEM lanes.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]),
        "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]),
        "=f"(r[14]), "=f"(r[15])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const float (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15, %16};" ::"r"(taddr),
      "f"(r[0]), "f"(r[1]), "f"(r[2]), "f"(r[3]), "f"(r[4]), "f"(r[5]), "f"(r[6]), "f"(r[7]),
      "f"(r[8]), "f"(r[9]), "f"(r[10]), "f"(r[11]), "f"(r[12]), "f"(r[13]), "f"(r[14]), "f"(r[15])
      : "memory");
}

// One epilogue warp's piece of a tile: 32 rows (one a lane) x kCols columns of results of type Out,
// out of tensor memory into shared memory in the tensor map's swizzle. exp_b: the columns'
// exponents (exp_a: this lane's row's) where operands were scaled, or nullptr. residual: the piece
// holds it, in type Out. preact: this lane's row, or nullptr. kFast: the activation for 16-bit
// results.
template <class T, class Out, int kCols, int kAct, bool kFast>
__device__ __forceinline__ void finish_piece(uint32_t taddr, const float* bias, const int* exp_b,
                                             int exp_a, T* preact, bool preact_wide,
                                             bool residual, unsigned char* piece, int lane) {
  constexpr uint32_t kRow = kCols * sizeof(Out);
  constexpr uint32_t kSwizzle = kRow == 128 ? 7 : (kRow == 64 ? 3 : 1);
  constexpr int kPer = 16 / static_cast<int>(sizeof(Out));  // elements of 16 bytes
  const uint32_t row = tc::smem_u32(piece) + lane * kRow;
  const uint32_t swizzle = ((lane * kRow >> 7) & kSwizzle) << 4;
#pragma unroll(sizeof(T) == 2 ? kCols / 16 : 1)
  for (int i = 0; i < kCols; i += 16) {
    float v[16];
    tmem_ld16(taddr + i, v);
    if constexpr (sizeof(T) == 4) {
      if (exp_b != nullptr) {
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = times_pow2(v[j], exp_a + exp_b[i + j]);
      }
    }
    if (bias != nullptr) {
#pragma unroll
      for (int j = 0; j < 16; j += 4) {
        const float4 b = *reinterpret_cast<const float4*>(bias + i + j);
        const float2 lo = add2(make_float2(v[j], v[j + 1]), make_float2(b.x, b.y));
        const float2 hi = add2(make_float2(v[j + 2], v[j + 3]), make_float2(b.z, b.w));
        v[j] = lo.x;
        v[j + 1] = lo.y;
        v[j + 2] = hi.x;
        v[j + 3] = hi.y;
      }
    }
    if (preact != nullptr) put16<T>(preact + i, v, 16, preact_wide ? 32 : 16);
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
      const float2 y = activate2<kFast>(kAct, make_float2(v[j], v[j + 1]));
      v[j] = y.x;
      v[j + 1] = y.y;
    }
#pragma unroll
    for (int k = 0; k < 16 / kPer; ++k) {
      const uint32_t at = row + ((i * static_cast<uint32_t>(sizeof(Out)) + k * 16) ^ swizzle);
      if (residual) {
        Pack<Out, kPer> r;
        uint4& q = reinterpret_cast<uint4&>(r);
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w)
                     : "r"(at));
#pragma unroll
        for (int j = 0; j < kPer; ++j) v[kPer * k + j] += dev::to_f32<Out>(r.v[j]);
      }
      Pack<Out, kPer> y;
#pragma unroll
      for (int j = 0; j < kPer; ++j) y.v[j] = dev::from_f32<Out>(v[kPer * k + j]);
      const uint4& q = reinterpret_cast<const uint4&>(y);
      asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(q.x), "r"(q.y),
                   "r"(q.z), "r"(q.w));
    }
  }
}

// NaN over a piece (this lane's row of it), where the pipeline gave up.
template <class Out, int kCols>
__device__ __noinline__ void poison_piece(unsigned char* piece, int lane) {
  Out* row = reinterpret_cast<Out*>(piece) + lane * kCols;
  for (int c = 0; c < kCols; ++c) row[c] = dev::from_f32<Out>(__uint_as_float(0x7fc00000u));
}

// The preactivations of a piece's columns where they can neither be stored whole nor through the
// piece: each lane its row.
template <class T>
__device__ __forceinline__ void store_preact(uint32_t taddr, bool ok, const float* bias,
                                             const int* exp_b, int exp_a, T* first,
                                             int64_t stride, int rows, int cols, int lane) {
  for (int i = 0; i < cols; i += 16) {
    float v[16];
    tmem_ld16(taddr + i, v);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      if (sizeof(T) == 4 && exp_b != nullptr) v[j] = times_pow2(v[j], exp_a + exp_b[i + j]);
      if (bias != nullptr) v[j] += bias[i + j];
      if (!ok) v[j] = __uint_as_float(0x7fc00000u);
    }
    if (lane < rows) put16<T>(first + lane * stride + i, v, min(16, cols - i), 2);
  }
}

// Stores a piece of kCols float32 columns to rows of any alignment: lanes along a row, so that a row's
// columns are written together; residual (at the piece's first element, or nullptr) is added first.
template <class T, class Out, int kCols>
__device__ __forceinline__ void store_piece(const unsigned char* piece, Out* out, int64_t stride,
                                            const T* residual, int64_t residual_stride, int rows,
                                            int cols, int lane) {
  constexpr uint32_t kRow = kCols * 4;
  constexpr uint32_t kSwizzle = kRow == 128 ? 7 : 3;
  constexpr int kPerStep = 32 / kCols;  // rows at a time
  constexpr int kBatch = 8;             // steps whose residuals are in flight together
  const int c = lane % kCols;
  const bool in = c < cols;
#pragma unroll 1
  for (int b = 0; b < 32; b += kBatch * kPerStep) {
    T res[kBatch];
    if (residual != nullptr) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int r = min(b + u * kPerStep + lane / kCols, rows - 1);
        res[u] = residual[r * residual_stride + min(c, cols - 1)];
      }
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int r = b + u * kPerStep + lane / kCols;
      const uint32_t off = r * kRow + c * 4;
      float v = *reinterpret_cast<const float*>(piece + (off ^ (((off >> 7) & kSwizzle) << 4)));
      if (residual != nullptr) v += dev::to_f32<T>(res[u]);
      if (in && r < rows) out[r * stride + c] = dev::from_f32<Out>(v);
    }
  }
}

// T: the operands' type, Out: the results' (T or float32).
template <class T, class Out, int kBN, bool kPair, bool kChunked>
__global__ void __launch_bounds__(kProductThreads, 1)
    product_kernel(const __grid_constant__ ProductMaps maps,
                   const __grid_constant__ ProductGroup g) {
  using S = Tile<kBN, kPair>;
  constexpr bool kOutF32 = sizeof(Out) == 4;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* tiles = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* pieces = tiles + S::kStages * S::kStageBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(pieces + kEpilogueWarps * kPieceBytes);
  // full[stage], empty[stage], acc_full[2], acc_empty[2], drain, residual[epilogue warp]. In a pair the leader's full and
  // acc_empty barriers stand for both CTAs; empty and acc_full are signalled in each.
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  // Each epilogue warp's columns of the bias, two tiles' worth.
  __shared__ __align__(16) float s_bias[kEpilogueWarps][2][kBN / 4];
  __shared__ int s_exp[kEpilogueWarps][2][sizeof(T) == 4 ? kBN / 4 : 1];  // and of exp_b
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = kPair ? tc::cluster_ctarank() : 0;
  const bool leader = rank == 0;
  auto bar = [&](int i) { return tc::smem_u32(bars + i); };
  auto lbar = [&](int i) { return kPair ? tc::mapa_shared(bar(i), 0) : bar(i); };
  dev::allow_next();
  constexpr int FULL = 0, EMPTY = S::kStages, ACC_FULL = 2 * S::kStages, ACC_EMPTY = ACC_FULL + 2,
                DRAIN = ACC_EMPTY + 2, RESIDUAL = DRAIN + 1;
  static_assert((RESIDUAL + kEpilogueWarps) * 8 <= 512, "the barriers fit behind the pieces");
  const int units = g.units[0] + g.units[1];
  const int worker = kPair ? static_cast<int>(blockIdx.x >> 1) : static_cast<int>(blockIdx.x);
  const int workers = kPair ? static_cast<int>(gridDim.x >> 1) : static_cast<int>(gridDim.x);
  auto unit = [&](int u) { return unit_of(g, u); };

  // Ahead of the set-up's barrier: the first unit's parameters and tensor maps are on their way
  // while tensor memory is allocated.
  const Unit first = unit(worker < units ? worker : 0);
  if (warp == 0 && elect_one()) {
    prefetch_map(&maps.a[first.q]);
    prefetch_map(&maps.b[first.q]);
  }
  constexpr int kBars = RESIDUAL + kEpilogueWarps;
  static_assert(kBars <= 32, "one barrier a lane");
  if (threadIdx.x < kBars) {
    if (threadIdx.x == 0) s_abort = 0;
    const bool acc_empty = threadIdx.x == ACC_EMPTY || threadIdx.x == ACC_EMPTY + 1;
    tc::mbar_init(bar(threadIdx.x), acc_empty ? (kPair ? 2 : 1) * kEpilogueWarps : 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if constexpr (kPair) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                       tc::smem_u32(&s_tmem)),
                   "r"(2 * kBN));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                       tc::smem_u32(&s_tmem)),
                   "r"(2 * kBN));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if constexpr (kPair) tc::cluster_sync();  // both CTAs' barriers exist before either uses them
  tc::tc_fence_after();
  dev::wait_previous();  // what packed the operands
  const uint32_t tmem = s_tmem;
  bool in_planes = false;  // a vote, so that what depends on it stays uniform
  if constexpr (sizeof(T) == 4)
    in_planes = g.wide != nullptr &&
                __any_sync(dev::kFull, *static_cast<const volatile int*>(g.wide) != 0);
  volatile int* abort_flag = &s_abort;
  // Bounded wait of a whole warp; false on timeout or abort, after which the CTA's remaining results
  // are NaN.
  auto wait = [&](uint32_t b, uint32_t parity) {
    auto test = [&] {
      return kPair ? tc::mbar_test_cluster(b, parity) : tc::mbar_test(b, parity);
    };
    auto sleep_test = [&] {
      return kPair ? tc::mbar_sleep_test_cluster(b, parity) : tc::mbar_sleep_test(b, parity);
    };
    // Every exit is the warp's vote: warp-wide instructions follow each wait.
    if (__all_sync(dev::kFull, test())) return true;
    const long long t0 = clock64();
    for (;;) {
      if (__all_sync(dev::kFull, sleep_test())) return true;
      if (__any_sync(dev::kFull, *abort_flag != 0 || clock64() - t0 > g.wait_cycles)) {
        *abort_flag = 1;
        return false;
      }
    }
  };
  // The producer and MMA loops run warp-uniformly and elect a lane for the copies and MMAs alone:
  // their addresses and descriptors then stay in uniform registers, which those instructions take.
  // With a single lane in the whole loop, operands moved there one by one, a block of k took
  // 620 cycles to issue where its MMAs take 512.
  const uint32_t tiles_at = tc::smem_u32(tiles), full_at = lbar(FULL), empty_at = bar(EMPTY);
  if (warp == 0) {
    int s = 0;
    uint32_t phase = 1;
    bool ok = true;
    auto produce = [&](auto a_mn, auto b_mn, const Unit& w, int q) {
      const ProductArgs& a = g.p[q];
      const int form = in_planes ? 1 : q;
      const int pairs = in_planes ? 6 : a.pairs;
      const CUtensorMap* map_a = &maps.a[form];
      const CUtensorMap* map_b = &maps.b[form];
      const int row_a = w.tm * S::kM + static_cast<int>(rank) * kBM;
      const int row_b = w.tn * kBN + static_cast<int>(rank) * S::kBRows;
      for (int pass = 0, c0 = w.b0; c0 < w.b1 && ok;) {  // pairs of planes within chunks of k
        const int pa = kPairA[first_pair(pairs) + pass], pb = kPairB[first_pair(pairs) + pass];
        const int c1 = min(w.b1, c0 + a.chunk);
        for (int k0 = c0 * kBK; k0 < c1 * kBK; k0 += kBK) {
          if (!wait(empty_at + s * 8, phase)) {
            ok = false;
            break;
          }
          if (elect_one()) {
            const uint32_t full = full_at + s * 8;
            const uint32_t da = tiles_at + s * S::kStageBytes, db = da + S::kABytes;
            if (leader) tc::mbar_expect_tx(bar(FULL) + s * 8, (kPair ? 2 : 1) * S::kStageBytes);
            if constexpr (decltype(a_mn)::value) {
#pragma unroll
              for (int c = 0; c < kBM / 64; ++c)
                tma_load_3d<kPair>(da + c * 8192, map_a, row_a + c * 64, k0, pa, full);
            } else {
              tma_load_3d<kPair>(da, map_a, k0, row_a, pa, full);
            }
            if constexpr (decltype(b_mn)::value) {
#pragma unroll
              for (int c = 0; c < S::kBRows / 64; ++c)
                tma_load_3d<kPair>(db + c * 8192, map_b, row_b + c * 64, k0, pb, full);
            } else {
              tma_load_3d<kPair>(db, map_b, k0, row_b, pb, full);
            }
          }
          s = s + 1 == S::kStages ? 0 : s + 1;
          phase ^= s == 0;
        }
        pass = pass + 1 == pairs ? 0 : pass + 1;
        c0 = pass == 0 ? c1 : c0;
      }
    };
    for (int u = worker; u < units && ok; u += workers) {
      const Unit w = u == worker ? first : unit(u);
      const int q = w.q;
      // The three forms of a layer's products: x W^T, dz W, dz^T x.
      if (g.p[q].a_mn)
        produce(std::true_type{}, std::true_type{}, w, q);
      else if (g.p[q].b_mn)
        produce(std::false_type{}, std::true_type{}, w, q);
      else
        produce(std::false_type{}, std::false_type{}, w, q);
    }
  } else if (warp == 1) {
    if (leader) {  // in a pair the leader issues for both CTAs
      int t = 0, s = 0;
      uint32_t phase = 0;
      bool ok = true;
      auto commit = [&](uint32_t at) {  // signals a barrier (of both CTAs) after the MMAs so far
        if constexpr (kPair)
          tc::umma_commit_pair_mc(at, 0x3);
        else
          tc::umma_commit(at);
      };
      for (int u = worker; u < units && ok; u += workers) {
        const Unit w = u == worker ? first : unit(u);
        const ProductArgs& a = g.p[w.q];
        const uint32_t idesc = in_planes ? g.wide_idesc : a.idesc;
        const uint32_t a_step = a.a_mn ? 2048 >> 4 : 32 >> 4, b_step = a.b_mn ? 2048 >> 4 : 32 >> 4;
        const uint64_t ad0 = operand_desc(tiles_at, a.a_mn);
        const uint64_t bd0 = operand_desc(tiles_at + S::kABytes, a.b_mn);
        const int pairs = in_planes ? 6 : a.pairs, chunk = a.chunk;
        for (int c0 = w.b0; c0 < w.b1 && ok; c0 += chunk, ++t) {
          const int slot = t & 1;
          if (!wait(bar(ACC_EMPTY + slot), ((t >> 1) & 1) ^ 1)) {
            ok = false;
            break;
          }
          tc::tc_fence_after();
          const uint32_t d = tmem + slot * kBN;
          const int blocks = min(chunk, w.b1 - c0) * pairs;
          for (int i = 0; i < blocks; ++i) {
            if (!wait(bar(FULL) + s * 8, phase)) {
              ok = false;
              break;
            }
            tc::tc_fence_after();
            if (elect_one()) {
              const uint64_t ad = ad0 + static_cast<uint32_t>(s * (S::kStageBytes >> 4));
              const uint64_t bd = bd0 + static_cast<uint32_t>(s * (S::kStageBytes >> 4));
#pragma unroll
              for (int q = 0; q < kBK / 16; ++q)
                mma_f16<kPair>(d, ad + q * a_step, bd + q * b_step, idesc, (i | q) != 0);
              commit(empty_at + s * 8);
              if (i == blocks - 1) commit(bar(ACC_FULL + slot));
            }
            __syncwarp();
            s = s + 1 == S::kStages ? 0 : s + 1;
            phase ^= s == 0;
          }
        }
      }
      if (*abort_flag) {  // wait (bounded) for the MMAs in flight before their memory goes
        if (elect_one()) {
          if constexpr (kPair)
            tc::umma_commit_pair_mc(bar(DRAIN), 0x1);
          else
            tc::umma_commit(bar(DRAIN));
        }
        __syncwarp();
        const uint64_t t0 = tc::gtimer();
        while (!tc::mbar_test(bar(DRAIN), 0) && tc::gtimer() - t0 < g.drain_ns) {
        }
      }
    }
  } else {
    // Each warp finishes a quarter of the tile's rows and of its columns: a row per lane, 16
    // columns at a time. Results (and residuals) that TMA can address go through a piece of 32
    // rows x up to 128 bytes in shared memory, in the tensor map's swizzle, so that memory sees
    // whole lines and the residual is on its way while the tile is still being multiplied; the
    // others are stored from registers.
    const int quarter = warp & 3;            // TMEM lanes this warp may read
    const int ew = warp - 2;
    const int group = ew >> 2;               // which quarter of the columns it takes
    constexpr int kCols = kBN / 4;
    unsigned char* piece = pieces + ew * kPieceBytes;
    const uint32_t res_bar = bar(RESIDUAL + ew);
    uint32_t res_phase = 0;
    // Waits for the piece's residual; given up, its copy must still land before the piece goes.
    auto wait_residual = [&](uint32_t b, uint32_t& phase) {
      const bool ok = wait(b, phase);
      if (!ok) {
        const uint64_t t0 = tc::gtimer();
        while (!tc::mbar_test(b, phase) && tc::gtimer() - t0 < g.drain_ns) {
        }
      }
      phase ^= 1;
      __syncwarp();
      return ok;
    };
    auto release = [&](int slot) {  // the accumulator may be overwritten
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (kPair)
          tc::mbar_arrive_cluster(lbar(ACC_EMPTY + slot));
        else
          tc::mbar_arrive(bar(ACC_EMPTY + slot));
      }
    };
    // Once a wait has failed, this warp neither waits nor arrives any more, and all its remaining
    // results are NaN: a barrier that nobody advances would satisfy the wait after next with the
    // phase before, and arrivals out of turn would stand in for the other CTA's.
    bool alive = true;
    int t = 0, parity = 0;  // chunks read so far; of units
    for (int u = worker; u < units; u += workers, parity ^= 1) {
      const Unit w = u == worker ? first : unit(u);
      const ProductArgs& a = g.p[w.q];
      int slot = 0;  // accumulator of the unit's last chunk, where its sums end up
      const int64_t col0 = static_cast<int64_t>(w.tn) * kBN + group * kCols;
      const int64_t row0 = static_cast<int64_t>(w.tm) * S::kM + rank * kBM + quarter * 32;
      const int64_t row = row0 + lane;
      float* bias = s_bias[ew][parity];
      if (a.ep.bias != nullptr) {  // loaded ahead of the wait
        for (int j = lane; j < kCols; j += 32)
          bias[j] = col0 + j < a.n
                        ? dev::to_f32<T>(static_cast<const T*>(a.ep.bias)[col0 + j]) : 0.0f;
      }
      int* exp_b = s_exp[ew][parity];
      int exp_a = 0;
      if constexpr (sizeof(T) == 4) {
        if (a.exp_a != nullptr) {
          auto form = [&](int e) { return in_planes ? lifted(e) : e; };
          exp_a = row < a.m ? form(a.exp_a[row]) : 0;
          for (int j = lane; j < kCols; j += 32)
            exp_b[j] = col0 + j < a.n ? form(a.exp_b[col0 + j]) : 0;
        }
      }
      const bool res_tiles = a.splits == 1 && a.ep.residual_tiles;
      const bool in_tiles =
          a.splits == 1 && a.ep.out_tiles && (a.ep.residual == nullptr || res_tiles);
      // The piece's columns: 128 bytes at most, of the result or, where that is not stored as a
      // tile, of float32.
      constexpr int kWide = kCols < 32 ? kCols : 32;
      const int per_piece = in_tiles && !kOutF32 ? kCols : kWide;
#pragma unroll 1
      for (int c = 0; c < kCols; c += per_piece) {
        const int64_t col = col0 + c;
        const bool any = col < a.n && row0 < a.m;
        const bool load = any && res_tiles && alive;
        if (any) {
          if (lane == 0) {
            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // the piece is free
            if (load) {
              tc::mbar_expect_tx(res_bar, 32 * per_piece * sizeof(Out));
              tc::tma_load_2d(tc::smem_u32(piece), &maps.residual[w.q], static_cast<int>(col),
                              static_cast<int>(row0), res_bar);
            }
          }
          __syncwarp();
        }
        if (c == 0 && alive) {
          alive = wait(bar(ACC_FULL + (t & 1)), (t >> 1) & 1);
          tc::tc_fence_after();
          slot = t & 1;
          ++t;
          if (kChunked && alive && w.b1 - w.b0 > a.chunk) {
            // Chunks before the last, added up in registers.
            const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
            float sum[kCols];
#pragma unroll
            for (int i = 0; i < kCols; i += 16)
              tmem_ld16(tmem + slot * kBN + group * kCols + i + lanes, *reinterpret_cast<float(*)[16]>(sum + i));
            for (int c0 = w.b0 + a.chunk; c0 < w.b1; c0 += a.chunk, ++t) {
              release(slot);
              slot = t & 1;
              alive = wait(bar(ACC_FULL + slot), (t >> 1) & 1);
              if (!alive) break;
              tc::tc_fence_after();
#pragma unroll
              for (int i = 0; i < kCols; i += 16) {
                float v[16];
                tmem_ld16(tmem + slot * kBN + group * kCols + i + lanes, v);
#pragma unroll
                for (int j = 0; j < 16; j += 2) {
                  const float2 y = add2(make_float2(sum[i + j], sum[i + j + 1]),
                                        make_float2(v[j], v[j + 1]));
                  sum[i + j] = y.x;
                  sum[i + j + 1] = y.y;
                }
              }
            }
#pragma unroll
            for (int i = 0; i < kCols; i += 16)
              tmem_st16(tmem + slot * kBN + group * kCols + i + lanes, *reinterpret_cast<float(*)[16]>(sum + i));
            tc::tmem_wait_st();
          }
        }
        if (!any) continue;
        // The parameters in registers and the activation chosen once per piece. (Reading them per
        // 16 columns made a 128 x 256 tile's epilogue take 10,500 cycles, more than the MMAs of
        // k = 1024.)
        if (load) alive = wait_residual(res_bar, res_phase) && alive;
        const uint32_t taddr = tmem + slot * kBN + group * kCols + c +
                               (static_cast<uint32_t>(quarter * 32) << 16);
        const float* b = a.splits == 1 && a.ep.bias != nullptr ? bias + c : nullptr;
        const int* e = sizeof(T) == 4 && a.exp_a != nullptr ? exp_b + c : nullptr;
        auto by_act = [&](int act, auto&& finish) {
          switch (act) {
            case QV_ACT_RELU: finish(std::integral_constant<int, QV_ACT_RELU>{}); break;
            case QV_ACT_GELU: finish(std::integral_constant<int, QV_ACT_GELU>{}); break;
            case QV_ACT_GELU_TANH: finish(std::integral_constant<int, QV_ACT_GELU_TANH>{}); break;
            case QV_ACT_SILU: finish(std::integral_constant<int, QV_ACT_SILU>{}); break;
            default: finish(std::integral_constant<int, QV_ACT_NONE>{}); break;
          }
        };
        auto finish_f32 = [&](int act, T* preact, bool wide, bool residual) {
          by_act(act, [&](auto k) {
            finish_piece<T, float, kWide, decltype(k)::value, !kOutF32>(
                taddr, b, e, exp_a, preact, wide, residual, piece, lane);
          });
          if (!alive) poison_piece<float, kWide>(piece, lane);
          __syncwarp();
        };
        const int rows = static_cast<int>(min(static_cast<int64_t>(32), a.m - row0));
        const int cols = static_cast<int>(min(static_cast<int64_t>(per_piece), a.n - col));
        // Preactivations: whole aligned pieces straight from the registers, others by a pass of
        // their own.
        T* preact = nullptr;
        bool wide = false;
        if (a.splits == 1 && a.ep.preact != nullptr) {
          T* first = static_cast<T*>(a.ep.preact) + row0 * a.ep.preact_stride + col;
          if (alive && in_tiles && cols == per_piece && a.ep.preact_align >= 16) {
            preact = row < a.m ? first + lane * a.ep.preact_stride : nullptr;
            wide = a.ep.preact_align >= 32;
          } else if (!res_tiles && per_piece == kWide) {
            finish_f32(QV_ACT_NONE, nullptr, false, false);
            store_piece<T, T, kWide>(piece, first, a.ep.preact_stride, nullptr, 0, rows, cols, lane);
            __syncwarp();
          } else {  // the piece holds the residual, or more columns than float32 has room for
            store_preact<T>(taddr, alive, b, e, exp_a, first, a.ep.preact_stride, rows, cols, lane);
          }
        }
        if (in_tiles) {
          if constexpr (kOutF32) {
            finish_f32(a.ep.act, preact, wide, res_tiles);
          } else {
            by_act(a.ep.act, [&](auto k) {
              finish_piece<T, T, kCols, decltype(k)::value, true>(
                  taddr, b, e, exp_a, preact, wide, res_tiles, piece, lane);
            });
            if (!alive) poison_piece<T, kCols>(piece, lane);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0)
            tma_store_2d(&maps.out[w.q], static_cast<int>(col), static_cast<int>(row0),
                         tc::smem_u32(piece));
          continue;
        }
        // Rows that TMA cannot address, a residual that it cannot, or a split's sums.
        finish_f32(a.splits > 1 ? QV_ACT_NONE : a.ep.act, preact, wide, false);
        if (a.splits > 1) {
          store_piece<T, float, kWide>(
              piece, a.partial + (static_cast<int64_t>(w.split) * a.m + row0) * a.n + col, a.n,
              nullptr, 0, rows, cols, lane);
        } else {
          auto store = [&](auto type) {
            using R = decltype(type);
            const R* residual = a.ep.residual != nullptr
                                    ? static_cast<const R*>(a.ep.residual) +
                                          row0 * a.ep.residual_stride + col
                                    : nullptr;
            store_piece<R, Out, kWide>(
                piece, static_cast<Out*>(a.ep.out) + row0 * a.ep.out_stride + col, a.ep.out_stride,
                residual, a.ep.residual_stride, rows, cols, lane);
          };
          if (kOutF32 && a.ep.residual_f32)
            store(float{});
          else
            store(T{});
        }
        __syncwarp();
      }
      if (alive) release(slot);
    }
    // The pieces stay until the last stores have read them.
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  }
  tc::tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    // Whoever gave up, copies that the producer issued may still be in flight (it may itself be
    // done long before), and they must land before the CTA leaves. They may be counted on barriers
    // that this CTA cannot poll (a pair's leader's): wait out the bound, far longer than any copy.
    // Without the flag every copy was multiplied, or no result would have come.
    const uint64_t t0 = tc::gtimer();
    while (tc::gtimer() - t0 < g.drain_ns) {
    }
    __syncthreads();
  }
  // A CTA of a pair stays until the other is done with its barriers, tiles and accumulators.
  if constexpr (kPair) tc::cluster_sync();
  if (warp == 1) {
    tc::tc_fence_after();
    if constexpr (kPair)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                   "r"(2 * kBN));
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                   "r"(2 * kBN));
  }
}

// What is left after a launch of products, by block row: the splits of each one's k joined in their
// order and their elements finished, kV neighbours a thread, and the bias gradient from its row
// ranges' sums.
struct SplitJob {
  const float* partial;
  int splits;  // 0: nothing to join
  int64_t m, n;
  Epilogue ep;
};
struct SumsJob {
  const float* sums;  // nullptr: none
  int blocks;
  int64_t n;
  void* db;
};
struct JoinJobs {
  SplitJob split[2];
  SumsJob sums;
};
template <class T, class Out, int kV>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ JoinJobs jobs) {
  dev::wait_previous();
  if (blockIdx.y < 2) {
    const SplitJob& j = jobs.split[blockIdx.y];
    if (j.splits == 0) return;
    const int64_t size = j.m * j.n;
    const int splits = j.splits;
    const float* partial = j.partial;
    const uint32_t per_row = static_cast<uint32_t>(j.n / kV);
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < size / kV; i += gridDim.x * 256ll) {
      float s[kV];
#pragma unroll
      for (int v = 0; v < kV; ++v) s[v] = 0.0f;
#pragma unroll 8
      for (int k = 0; k < splits; ++k) {
        const Pack<float, kV> x = dev::load_pack<float, kV>(partial + k * size + i * kV);
#pragma unroll
        for (int v = 0; v < kV; ++v) s[v] += x.v[v];
      }
      const int64_t row = i >> 32 ? i / per_row : static_cast<uint32_t>(i) / per_row;
      const int64_t col = (i - row * per_row) * kV;
#pragma unroll
      for (int v = 0; v < kV; ++v) finish1<T, sizeof(Out) == 2>(j.ep, row, col + v, s[v]);
    }
    return;
  }
  // 32 columns at a time: each warp a run of row ranges, then the warps in order.
  const SumsJob& j = jobs.sums;
  __shared__ float part[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = (j.blocks + 7) / 8;
  const int b1 = min(j.blocks, (warp + 1) * per);
  for (int64_t c0 = blockIdx.x * 32ll; c0 < j.n; c0 += gridDim.x * 32ll) {
    const int64_t col = c0 + lane;
    float s = 0.0f;
    if (col < j.n) {
#pragma unroll 8
      for (int b = warp * per; b < b1; ++b) s += j.sums[b * j.n + col];
    }
    part[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && col < j.n) {
      float t = 0.0f;
#pragma unroll
      for (int w = 0; w < 8; ++w) t += part[w][lane];
      static_cast<T*>(j.db)[col] = dev::from_f32<T>(t);
    }
    __syncthreads();
  }
}

// ---- few rows: every weight read once with plain loads -------------------------------------------

// One warp per kCols output columns and kRows rows of x: lanes stride over k, float32 sums two terms
// at a time, and every piece of x is unpacked once for the warp's columns. One row is bound by
// reading the weights (4096 x 4096 bfloat16: 5.3 us); with eight the arithmetic costs more (18 us
// with two columns a warp, 20 with one), and narrow layers have too few warps for two columns each
// (8 rows of 768 x 768: 4.3 us against 5.3).
template <class T, int kRows, int kCols, int kV>
__global__ void __launch_bounds__(128)
    few_rows_kernel(const T* __restrict__ x, int64_t x_stride, const T* __restrict__ w,
                    int64_t w_stride, int m, int64_t n, int64_t k, Epilogue ep) {
  const int lane = threadIdx.x & 31;
  const int64_t col = ((blockIdx.x * 128ll + threadIdx.x) >> 5) * kCols;
  if (col >= n) return;
  const int64_t row0 = static_cast<int64_t>(blockIdx.y) * kRows;
  x += row0 * x_stride;
  m -= static_cast<int>(row0);
  float2 acc[kRows][kCols];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
#pragma unroll
    for (int q = 0; q < kCols; ++q) acc[r][q] = both(0.0f);
  }
#pragma unroll(kRows* kCols >= 16 ? 1 : 4)
  for (int64_t c = lane * kV; c < k; c += 32 * kV) {
    // Columns and rows past the last read it again: loads without a branch, all in flight.
    Pack<T, kV> a[kCols];
#pragma unroll
    for (int q = 0; q < kCols; ++q)
      a[q] = dev::load_pack<T, kV>(w + min(col + q, n - 1) * w_stride + c);
    Pack<T, kV> b[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r)
      b[r] = dev::load_pack<T, kV>(x + min(r, m - 1) * x_stride + c);
    if constexpr (kV == 1) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
#pragma unroll
        for (int q = 0; q < kCols; ++q)
          acc[r][q].x = fmaf(dev::to_f32<T>(a[q].v[0]), dev::to_f32<T>(b[r].v[0]), acc[r][q].x);
      }
    } else {
#pragma unroll
      for (int j = 0; j < kV; j += 2) {
        float2 wf[kCols];
#pragma unroll
        for (int q = 0; q < kCols; ++q)
          wf[q] = make_float2(dev::to_f32<T>(a[q].v[j]), dev::to_f32<T>(a[q].v[j + (kV > 1)]));
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const float2 xf =
              make_float2(dev::to_f32<T>(b[r].v[j]), dev::to_f32<T>(b[r].v[j + (kV > 1)]));
#pragma unroll
          for (int q = 0; q < kCols; ++q) acc[r][q] = fma2(wf[q], xf, acc[r][q]);
        }
      }
    }
  }
#pragma unroll
  for (int q = 0; q < kCols; ++q) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      float s = acc[r][q].x + acc[r][q].y;
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(dev::kFull, s, d);
      if (r < m && lane == r && col + q < n) {
        if (sizeof(T) == 2 && !ep.out_f32)
          finish1<T, true>(ep, row0 + r, col + q, s);
        else
          finish1<T, false>(ep, row0 + r, col + q, s);
      }
    }
  }
}

// ---- dz and the bias gradient ----------------------------------------------------------------------

// dz = dy * act'(z), rounded to the operand type (float32: three planes), and float32 column sums
// of the unrounded dz; dy is of type G (T, or float32 as it comes from a float32 result) over this block's rows. A block takes 32 pieces' columns and a range of rows:
// warp w walks rows w, w + 8, .. of it, and the warps' sums are added in order at the end, so the
// sums have a fixed order. Bound by memory: dy and z read, dz written.
constexpr int kDzWarps = 8, kDzRows = 4;  // rows in flight per warp
constexpr int dz_pieces(size_t piece_bytes) {  // 2-byte pieces: four a lane
  return piece_bytes == 2 ? 4 : 1;
}

template <class T, class G, int kV, bool kStore, int kAct>
__global__ void __launch_bounds__(32 * kDzWarps)
    dz_kernel(const G* __restrict__ dy, int64_t dy_stride, const T* __restrict__ z,
              int64_t z_stride, int64_t m, int64_t n, int64_t rows_per_block,
              typename Operand<T>::type* __restrict__ dz, int64_t ld, float* __restrict__ sums) {
  dev::allow_next();
  constexpr int kC = dz_pieces(sizeof(T) * kV);  // pieces of a row per lane
  constexpr int kCols = 32 * kV * kC;
  __shared__ float part[kDzWarps][kCols];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t col0 = static_cast<int64_t>(blockIdx.y) * kCols;
  const int64_t r1 = min(m, (blockIdx.x + 1) * rows_per_block);
  int64_t col[kC];
  bool on[kC];
  float s[kC][kV];
#pragma unroll
  for (int q = 0; q < kC; ++q) {
    col[q] = col0 + (q * 32 + lane) * kV;
    on[q] = col[q] < n;
    if (!on[q]) col[q] = col0;  // pieces past the last column read the first: no branches
#pragma unroll
    for (int j = 0; j < kV; ++j) s[q][j] = 0.0f;
  }
  for (int64_t r = blockIdx.x * rows_per_block + warp; r < r1; r += kDzWarps * kDzRows) {
    Pack<G, kV> g[kDzRows][kC];
    Pack<T, kV> x[kDzRows][kC];
#pragma unroll
    for (int u = 0; u < kDzRows; ++u) {
      const int64_t row = min(r + u * kDzWarps, r1 - 1);  // past the range its last row again
#pragma unroll
      for (int q = 0; q < kC; ++q) {
        g[u][q] = dev::load_pack<G, kV>(dy + row * dy_stride + col[q]);
        if (kAct != QV_ACT_NONE) x[u][q] = dev::load_pack<T, kV>(z + row * z_stride + col[q]);
      }
    }
#pragma unroll
    for (int u = 0; u < kDzRows; ++u) {
      const int64_t row = r + u * kDzWarps;
      if (row >= r1) break;
#pragma unroll
      for (int q = 0; q < kC; ++q) {
        float d[kV];
#pragma unroll
        for (int j = 0; j < kV; ++j) d[j] = dev::to_f32<G>(g[u][q].v[j]);
        if constexpr (kAct != QV_ACT_NONE) {
#pragma unroll
          for (int j = 0; j < kV; j += 2) {
            const bool two = j + 1 < kV;
            const float2 f = act_grad2<sizeof(T) == 2>(
                kAct, make_float2(dev::to_f32<T>(x[u][q].v[j]),
                                  dev::to_f32<T>(x[u][q].v[two ? j + 1 : j])));
            // rounded before the sum in every variant, so that dbias does not depend on which runs
            d[j] = __fmul_rn(d[j], f.x);
            if (two) d[two ? j + 1 : j] = __fmul_rn(d[two ? j + 1 : j], f.y);
          }
        }
#pragma unroll
        for (int j = 0; j < kV; ++j) s[q][j] += d[j];
        if (kStore && on[q]) put_operand<T, kV>(d, dz, m * ld, row * ld + col[q]);
      }
    }
  }
  if (sums == nullptr) return;
#pragma unroll
  for (int q = 0; q < kC; ++q) {
#pragma unroll
    for (int j = 0; j < kV; ++j) part[warp][(q * 32 + lane) * kV + j] = s[q][j];
  }
  __syncthreads();
  for (int c = threadIdx.x; c < kCols; c += 32 * kDzWarps) {
    if (col0 + c >= n) continue;
    float t = 0.0f;
#pragma unroll
    for (int w = 0; w < kDzWarps; ++w) t += part[w][c];
    sums[blockIdx.x * n + col0 + c] = t;
  }
}

// ---- host side ----------------------------------------------------------------------------------------

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                              const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static EncodeFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeFn>(p);
  });
  if (fn == nullptr) fail(QV_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  return fn;
}

// A stored operand: `outer` rows of `inner` elements, ld apart, `planes` copies plane_stride apart.
struct Stored {
  const int* exponents = nullptr;  // of scaled rows
  const void* p = nullptr;
  int64_t inner = 0, outer = 0, ld = 0;
  int planes = 1;
  bool bf16 = true;
};

CUtensorMap operand_map(const Stored& s, uint32_t box_outer) {
  CUtensorMap m;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(s.inner), static_cast<cuuint64_t>(s.outer),
                              static_cast<cuuint64_t>(s.planes)};
  // A single row may have any stride; the map wants one that holds it.
  const int64_t ld = s.outer > 1 ? s.ld : (s.inner + 7) / 8 * 8;
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld * 2),
                                 static_cast<cuuint64_t>(ld * s.outer * 2)};
  const cuuint32_t box[3] = {64, box_outer, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = encode_fn()(
      &m, s.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
      const_cast<void*>(s.p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) fail(QV_ERR_CUDA, "cuTensorMapEncodeTiled failed: " + std::to_string(r));
  return m;
}

// One product of a launch: D[m][n] = sum_k A B, finished by `ep`. a_mn / b_mn: the operand is
// stored with m (n) inner.
struct Product {
  int64_t m, n, k;
  bool a_mn, b_mn;
  Stored a, b;
  Epilogue ep;
  const int* wide = nullptr;  // scaled operands that may be three planes instead: which they are
};
// Scaled rows where choose_planes_kernel has replaced them.
Stored as_planes(Stored s) {
  s.planes = 3;
  s.bf16 = true;
  return s;
}
// A result or residual of the epilogue's pieces: 32 rows x 128 bytes at most.
CUtensorMap piece_map(const void* p, int64_t rows, int64_t cols, int64_t stride, uint32_t dtype,
                      int tile_cols) {
  CUtensorMap m;
  const int64_t elem = dtype == QV_DTYPE_F32 ? 4 : 2;
  const int64_t per_piece = std::min<int64_t>(tile_cols, 128 / elem);
  const int64_t ld = rows > 1 ? stride : (cols + 7) / 8 * 8;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld * elem)};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(per_piece), 32};
  const cuuint32_t estr[2] = {1, 1};
  const int64_t bytes = per_piece * elem;
  const CUresult r = encode_fn()(
      &m,
      dtype == QV_DTYPE_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
      : dtype == QV_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                              : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
      2, const_cast<void*>(p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
      bytes == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
      : bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                    : CU_TENSOR_MAP_SWIZZLE_32B,
      CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) fail(QV_ERR_CUDA, "cuTensorMapEncodeTiled failed: " + std::to_string(r));
  return m;
}

struct ProductPlan {
  int bn = 128;
  bool pair = false;
  int splits[2] = {1, 1}, blocks_per_split[2] = {1, 1}, k_blocks[2] = {1, 1};
  size_t partial_bytes[2] = {0, 0};
  double cycles = 0;
};

// Tiles and splits of k with the least estimated time. In cycles: a 64-wide block of k takes the
// larger of the MMAs and the copies into shared memory, a tile's results about 10 cycles a column
// (hidden behind the next tile's blocks when there is one), and the splits are written, read and
// joined in a launch of their own. Splits of a product are chosen with the tile width alone.
ProductPlan plan_products(const Product* p, int count, int pairs, int sms) {
  ProductPlan best;
  double best_t = 1e300;
  for (int bn : {64, 128, 256}) {
    ProductPlan plan;
    plan.bn = bn;
    plan.pair = bn == 256;
    const int workers = plan.pair ? sms / 2 : sms;
    const double per_block = bn == 256 ? 540 : (bn == 128 ? 400 : 280);
    double work = 0, longest = 0, joins = 0, waves_t = 0;
    for (int q = 0; q < count; ++q) {
      const int64_t m = p[q].m, n = p[q].n;
      const int64_t kb = std::max<int64_t>(1, static_cast<int64_t>(ceil_div(p[q].k, kBK)));
      const double tiles =
          static_cast<double>(ceil_div(m, plan.pair ? 2 * kBM : kBM)) * ceil_div(n, bn);
      double best_q = 1e300, unit_q = 0, units_q = 0, join_q = 0;
      for (int s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
        if (s > 1 && (s > kb || tiles * s > 2.0 * workers)) break;
        const int64_t per = static_cast<int64_t>(ceil_div(kb, s));
        const int64_t used = static_cast<int64_t>(ceil_div(kb, per));
        const double unit = std::max(static_cast<double>(per) * pairs * per_block, 10.0 * bn);
        const double join = used > 1 ? 4000 + 8.0 * m * n * used / 3000.0 : 0.0;
        const double t = std::ceil(tiles * used / workers) * unit + join;
        if (t < best_q) {
          best_q = t;
          unit_q = unit;
          units_q = tiles * used;
          join_q = join;
          plan.splits[q] = static_cast<int>(used);
          plan.blocks_per_split[q] = static_cast<int>(per);
          plan.k_blocks[q] = static_cast<int>(kb);
        }
      }
      work += unit_q * units_q / workers;
      longest = std::max(longest, unit_q);
      joins = std::max(joins, join_q);
      waves_t = std::ceil(units_q / workers) * unit_q;
      plan.partial_bytes[q] =
          plan.splits[q] > 1 ? (static_cast<size_t>(plan.splits[q]) * m * n * 4 + 255) / 256 * 256
                             : 0;
    }
    const double t =
        (count == 1 ? waves_t : std::max(longest, work + 0.5 * longest)) + joins + 10.0 * bn;
    if (t < best_t) {
      best_t = t;
      best = plan;
      best.cycles = t;
    }
  }
  return best;
}

template <class T, class Out, int kBN, bool kPair, bool kChunked>
void launch_products(const Product* p, int count, const ProductGroup& g, bool chained, int sms,
                     cudaStream_t st) {
  using S = Tile<kBN, kPair>;
  ProductMaps maps;
  for (int q = 0; q < count; ++q) {
    maps.a[q] = operand_map(p[q].a, p[q].a_mn ? kBK : kBM);
    maps.b[q] = operand_map(p[q].b, p[q].b_mn ? kBK : S::kBRows);
    const Epilogue& ep = p[q].ep;
    const uint32_t type = std::is_same_v<T, float>    ? QV_DTYPE_F32
                          : std::is_same_v<T, __half> ? QV_DTYPE_F16
                                                      : QV_DTYPE_BF16;
    if (g.p[q].splits == 1 && ep.out_tiles)
      maps.out[q] = piece_map(ep.out, p[q].m, p[q].n, ep.out_stride,
                              ep.out_f32 ? QV_DTYPE_F32 : type, kBN / 4);
    if (g.p[q].splits == 1 && ep.residual_tiles)
      maps.residual[q] =
          piece_map(ep.residual, p[q].m, p[q].n, ep.residual_stride,
                    ep.residual_f32 ? QV_DTYPE_F32 : type, kBN / 4);
  }
  if (p[0].wide != nullptr) {  // along k, by itself
    maps.a[1] = operand_map(as_planes(p[0].a), kBM);
    maps.b[1] = operand_map(as_planes(p[0].b), S::kBRows);
  }
  static std::once_flag once[16];
  int device = 0;
  QV_CUDA(cudaGetDevice(&device));
  std::call_once(once[device & 15], [&] {
    QV_CUDA(cudaFuncSetAttribute(product_kernel<T, Out, kBN, kPair, kChunked>,
                                 cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(S::kSmem)));
  });
  const int units = g.units[0] + g.units[1];
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(kPair ? 2 * std::min(units, sms / 2)
                                                 : std::min(units, sms)));
  cfg.blockDim = dim3(kProductThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = chained ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = kPair ? 2 : 1;
  cudaLaunchKernelEx(&cfg, product_kernel<T, Out, kBN, kPair, kChunked>, maps, g);  // reported by check_launch
  check_launch("product_kernel");
}

// Runs the products and what joins them (with the bias gradient's sums); chained: after another
// launch of the same call. partial: the plan's
// partial bytes, product by product.
template <class T>
void run_products(const Product* p, int count, const ProductPlan& plan, unsigned char* partial,
                  const SumsJob& sums, bool chained, int sms, cudaStream_t st) {
  ProductGroup g{};
  JoinJobs jobs{};
  jobs.sums = sums;
  size_t items = 0;
  for (int q = 0; q < count; ++q) {
    ProductArgs& a = g.p[q];
    a.m = p[q].m;
    a.n = p[q].n;
    a.pairs = p[q].a.planes == 3 ? 6 : (p[q].a.planes == 2 ? 3 : 1);
    a.exp_a = p[q].a.exponents;
    a.exp_b = p[q].b.exponents;
    a.k_blocks = plan.k_blocks[q];
    a.tiles_m = static_cast<int>(ceil_div(a.m, plan.pair ? 2 * kBM : kBM));
    a.tiles_n = static_cast<int>(ceil_div(a.n, plan.bn));
    a.splits = plan.splits[q];
    a.blocks_per_split = plan.blocks_per_split[q];
    a.chunk = a.pairs > 1 ? 2 : (p[q].ep.out_f32 ? 8 : 128);
    auto idesc = [&](bool bf16) {
      const uint32_t fmt = bf16 ? 1 : 0;
      return (1u << 4) | (fmt << 7) | (fmt << 10) | (static_cast<uint32_t>(p[q].a_mn) << 15) |
             (static_cast<uint32_t>(p[q].b_mn) << 16) |
             (static_cast<uint32_t>(plan.bn >> 3) << 17) |
             (static_cast<uint32_t>((plan.pair ? 2 * kBM : kBM) >> 4) << 24);
    };
    a.idesc = idesc(p[q].a.bf16);
    if (p[q].wide != nullptr) {
      g.wide = p[q].wide;
      g.wide_idesc = idesc(true);
    }
    a.a_mn = p[q].a_mn;
    a.b_mn = p[q].b_mn;
    a.ep = p[q].ep;
    a.partial = reinterpret_cast<float*>(partial);
    partial += plan.partial_bytes[q];
    g.units[q] = a.tiles_m * a.tiles_n * a.splits;
    if (a.splits > 1) {
      jobs.split[q] = SplitJob{a.partial, a.splits, a.m, a.n, a.ep};
      items = std::max(items, static_cast<size_t>(a.m) * a.n);
    }
  }
  g.wait_cycles = tc::wait_limit_cycles();
  g.drain_ns = tc::drain_limit_ns();
  if (count > 0) {
    auto launch = [&](auto out, auto chunked) {
      using Out = decltype(out);
      constexpr bool kChunked = decltype(chunked)::value;
      if (plan.pair)
        launch_products<T, Out, 256, true, kChunked>(p, count, g, chained, sms, st);
      else if (plan.bn == 128)
        launch_products<T, Out, 128, false, kChunked>(p, count, g, chained, sms, st);
      else
        launch_products<T, Out, 64, false, kChunked>(p, count, g, chained, sms, st);
    };
    // Sums of one chunk (16-bit operands and results with k up to 8192) leave the adding out of the
    // kernel, whose registers cost 4 % there. Float32 results of 16-bit operands have kernels of
    // their own: with both results in one, linear layers of 16-bit results took 14 % longer.
    bool chunked = std::is_same_v<T, float>;
    for (int q = 0; q < count; ++q) chunked |= plan.blocks_per_split[q] > g.p[q].chunk;
    if constexpr (std::is_same_v<T, float>)
      launch(float{}, std::true_type{});
    else if (p[0].ep.out_f32)  // a forward product, by itself
      launch(float{}, std::true_type{});
    else if (chunked)
      launch(T{}, std::true_type{});
    else
      launch(T{}, std::false_type{});
  }
  if (sums.sums != nullptr) items = std::max(items, static_cast<size_t>(sums.n) * 8);
  if (items > 0) {
    bool four = true;
    for (int q = 0; q < count; ++q) four &= plan.splits[q] == 1 || p[q].n % 4 == 0;
    const size_t threads = four ? ceil_div(items, 4) : items;
    const bool f32 = count > 0 && p[0].ep.out_f32;
    auto* join = f32 ? (four ? join_kernel<T, float, 4> : join_kernel<T, float, 1>)
                     : (four ? join_kernel<T, T, 4> : join_kernel<T, T, 1>);
    launch_chained(join,
                   dim3(static_cast<unsigned>(std::min<size_t>(ceil_div(threads, 256), 148 * 8)),
                        sums.sums != nullptr ? 3 : 2),
                   256, 0, st, jobs);
    check_launch("join_kernel");
  }
}

// Whether TMA can read 16-bit rows in place: 16-byte aligned rows.
bool in_place(uint32_t dtype, const void* p, size_t rows, size_t stride) {
  return dtype != QV_DTYPE_F32 && reinterpret_cast<uintptr_t>(p) % 16 == 0 &&
         (rows <= 1 || (stride * 2) % 16 == 0);
}
size_t packed_ld(size_t cols) { return (cols + 7) / 8 * 8; }
size_t packed_bytes(uint32_t dtype, size_t rows, size_t cols) {
  return (rows * packed_ld(cols) * 2 * (dtype == QV_DTYPE_F32 ? 3 : 1) + 255) / 256 * 256;
}
// A scaled float32 operand: two float16 planes, or three bfloat16 ones in their place, and the rows'
// exponents; behind both operands the rows' shares and the word that says which it is.
size_t scaled_bytes(size_t rows, size_t cols) {
  return packed_bytes(QV_DTYPE_F32, rows, cols) + (rows * 4 + 255) / 256 * 256;
}
constexpr size_t kSharesBytes = (2 * kSplitBlocks * 4 + 255) / 256 * 256, kChoiceBytes = kSharesBytes + 256;

// The operands of one call that have to be packed first, collected and packed in one launch.
template <class T>
class Packer {
 public:
  // scaled: rows with exponents, for products whose sums run along the rows; float32 ones as two
  // float16 planes where those do, or (planes) three bfloat16 ones at once.
  Packer(uint32_t dtype, bool scaled, bool planes, unsigned char* ws)
      : dtype_(dtype), scaled_(scaled && sizeof(T) == 4), planes_(planes), ws_(ws) {}
  Stored rows(const void* src, size_t rows, size_t cols, size_t stride) {
    Stored s;
    s.inner = static_cast<int64_t>(cols);
    s.outer = static_cast<int64_t>(rows);
    s.bf16 = !std::is_same_v<T, __half>;
    if (in_place(dtype_, src, rows, stride)) {
      s.p = src;
      s.ld = static_cast<int64_t>(stride);
      return s;
    }
    s.p = ws_;
    s.ld = static_cast<int64_t>(packed_ld(cols));
    const bool halves = scaled_ && !planes_;
    s.planes = halves ? 2 : Operand<T>::kPlanes;
    s.bf16 = s.bf16 && !halves;
    int* exponents = nullptr;
    if (scaled_)
      exponents = reinterpret_cast<int*>(ws_ + scaled_bytes(rows, cols) -
                                         (rows * 4 + 255) / 256 * 256);
    s.exponents = exponents;
    jobs_[count_++] =
        PackJob{src, ws_, s.outer, s.inner, static_cast<int64_t>(stride), s.ld, exponents};
    const size_t e = sizeof(T);
    align_ = std::min(align_, common_align({reinterpret_cast<uintptr_t>(src),
                                            rows > 1 ? stride * e : 0, cols * e}));
    ws_ += scaled_ ? scaled_bytes(rows, cols) : packed_bytes(dtype_, rows, cols);
    return s;
  }
  int count() const { return count_; }
  // Packs what was collected (chained: after another launch of the same call); returns the
  // workspace behind it.
  unsigned char* run(bool chained, cudaStream_t st) {
    if (count_ == 0) return ws_;
    if (align_ >= 16)
      launch<16 / sizeof(T)>(chained, st);
    else if (align_ == 8)
      launch<8 / sizeof(T)>(chained, st);
    else
      launch<1>(chained, st);
    count_ = 0;
    return ws_;
  }
  // Of a scaled call, after run(): which planes its operands are.
  const int* wide() const { return wide_; }

 private:
  template <int kV>
  void launch(bool chained, cudaStream_t st) {
    if constexpr (sizeof(T) == 4) {
      if (scaled_) {
        // Both operands are float32, so both are here.
        const size_t rows = static_cast<size_t>(std::max(jobs_[0].rows, jobs_[1].rows));
        const unsigned blocks =
            static_cast<unsigned>(std::min<size_t>(ceil_div(rows, 8), kSplitBlocks));
        if (planes_) {
          split_rows_kernel<kV, true><<<dim3(blocks, 2), 256, 0, st>>>(jobs_[0], jobs_[1], nullptr);
          check_launch("split_rows_kernel");
          return;
        }
        uint32_t* shares = reinterpret_cast<uint32_t*>(ws_);
        int* wide = reinterpret_cast<int*>(ws_ + kSharesBytes);
        ws_ += kChoiceBytes;
        wide_ = wide;
        split_rows_kernel<kV, false><<<dim3(blocks, 2), 256, 0, st>>>(jobs_[0], jobs_[1], shares);
        check_launch("split_rows_kernel");
        // Two blocks an SM in all: it rarely packs.
        launch_chained(choose_planes_kernel<kV>, dim3(std::min(blocks, 148u), 2), 256, 0, st,
                       jobs_[0], jobs_[1], static_cast<const uint32_t*>(shares), blocks, wide);
        check_launch("choose_planes_kernel");
        return;
      }
    }
    size_t most = 0;
    for (int i = 0; i < count_; ++i)
      most = std::max(most, ceil_div(jobs_[i].rows, kPackRows) * ceil_div(jobs_[i].cols, kV));
    const unsigned blocks = static_cast<unsigned>(std::min<size_t>(ceil_div(most, 256), 148 * 8));
    if (chained)
      launch_chained(pack_kernel<T, kV>, dim3(blocks, count_), 256, 0, st, jobs_[0],
                     jobs_[count_ - 1]);
    else
      pack_kernel<T, kV><<<dim3(blocks, count_), 256, 0, st>>>(jobs_[0], jobs_[count_ - 1]);
    check_launch("pack_kernel");
  }
  uint32_t dtype_;
  bool scaled_, planes_;
  unsigned char* ws_;
  PackJob jobs_[2];
  int count_ = 0, align_ = 16;
  const int* wide_ = nullptr;
};

constexpr size_t kWideFew = 2048;  // output columns from which a warp takes two
// Whether the batch takes the few-rows kernel, by the estimated times in us for W million weights.
// Measured, 4096 x 4096: 16-bit 4 rows 10.8, 8 rows 18, the tensor cores 12 to 14; float32 8 rows
// 17, the tensor cores (which split all the weights first) 61. 768 x 768: 8 rows 4.3 and 5.5, the
// tensor cores 7 and 12.
bool few_rows(uint32_t dtype, size_t m, size_t n, size_t k) {
  const double w = static_cast<double>(n) * k * 1e-6;
  const double groups = static_cast<double>(ceil_div(m, 8));  // each reads the weights again
  const double few = w * (0.25 + 0.104 * std::min<size_t>(m, 8)) * (1 + 2.2 * (groups - 1));
  return m <= 256 && few < (dtype == QV_DTYPE_F32 ? 12.0 + 2.9 * w : 7.0 + 0.35 * w);
}
constexpr size_t kMaxDim = 65536;
constexpr size_t kMaxLinearRows = (size_t{1} << 31) - 256;

template <class F>
void by_type(uint32_t dtype, F&& f) {
  if (dtype == QV_DTYPE_F32)
    f(float{});
  else if (dtype == QV_DTYPE_F16)
    f(__half{});
  else
    f(__nv_bfloat16{});
}

void check_matrix(const char* what, uint32_t dtype, const void* p, size_t rows, size_t cols,
                  size_t stride) {
  QV_REQUIRE(p != nullptr || rows == 0, std::string("null ") + what);
  QV_REQUIRE(reinterpret_cast<uintptr_t>(p) % dtype_size(dtype) == 0,
             std::string(what) + " is not aligned to its element type");
  QV_REQUIRE(stride >= cols || rows <= 1, std::string(what) + ": row stride below its columns");
  QV_REQUIRE(stride < (size_t{1} << 36), std::string(what) + ": row stride too large");
}

uint32_t out_dtype(const qv_linear& l) {
  return l.out_dtype & ~static_cast<uint32_t>(QV_RESIDUAL_F32);
}
bool residual_f32(const qv_linear& l) {
  return l.dtype == QV_DTYPE_F32 || (l.out_dtype & QV_RESIDUAL_F32) != 0;
}

void check_linear(const qv_linear& l) {
  check_dtype(l.dtype);
  QV_REQUIRE(l.activation <= QV_ACT_SILU, "unknown activation");
  QV_REQUIRE(l.k >= 1 && l.k <= kMaxDim && l.n >= 1 && l.n <= kMaxDim,
             "dimensions must be between 1 and 65536");
  QV_REQUIRE(l.m <= kMaxLinearRows, "too many rows");
  QV_REQUIRE(out_dtype(l) == l.dtype || out_dtype(l) == QV_DTYPE_F32,
             "results have the inputs' type or float32");
  QV_REQUIRE((l.out_dtype & QV_RESIDUAL_F32) == 0 || out_dtype(l) == QV_DTYPE_F32,
             "a float32 residual goes with float32 results");
  if (l.m == 0) return;
  check_matrix("x", l.dtype, l.x, l.m, l.k, l.x_stride);
  check_matrix("weight", l.dtype, l.weight, l.n, l.k, l.weight_stride);
  check_matrix("out", out_dtype(l), l.out, l.m, l.n, l.out_stride);
  if (l.bias != nullptr) check_matrix("bias", l.dtype, l.bias, 1, l.n, l.n);
  if (l.residual != nullptr) {
    // Stride 0 adds one row to every row of the result.
    check_matrix("residual", residual_f32(l) ? QV_DTYPE_F32 : l.dtype, l.residual, l.residual_stride == 0 ? 1 : l.m, l.n,
                 l.residual_stride);
  }
  if (l.preact != nullptr) check_matrix("preact", l.dtype, l.preact, l.m, l.n, l.preact_stride);
}

Epilogue epilogue_of(const qv_linear& l) {
  Epilogue e{};
  e.act = static_cast<int>(l.activation);
  e.bias = l.bias;
  e.residual = l.residual;
  e.residual_stride = static_cast<int64_t>(l.residual_stride);
  e.out = l.out;
  e.out_stride = static_cast<int64_t>(l.out_stride);
  e.out_f32 = out_dtype(l) == QV_DTYPE_F32;
  e.residual_f32 = residual_f32(l);
  e.preact = l.preact;
  e.preact_stride = static_cast<int64_t>(l.preact_stride);
  e.set_aligns(dtype_size(l.dtype));
  return e;
}

struct LinearPlan {
  bool few = false;
  bool planes = false;  // float32: three bfloat16 planes whatever the elements
  ProductPlan product;
  size_t bytes = 0;
};
LinearPlan linear_plan(const qv_linear& l, int sms) {
  LinearPlan p;
  p.few = few_rows(l.dtype, l.m, l.n, l.k);
  if (p.few || l.m == 0) return p;
  Product d{};
  d.m = static_cast<int64_t>(l.m);
  d.n = static_cast<int64_t>(l.n);
  d.k = static_cast<int64_t>(l.k);
  p.product = plan_products(&d, 1, l.dtype == QV_DTYPE_F32 ? 3 : 1, sms);
  if (l.dtype == QV_DTYPE_F32) {
    // Scaled operands need one launch more (choose_planes_kernel, 2.5 us of the GPU and as much of the
    // host), three planes twice the MMAs. Scaled and as planes, us on the GPU and a pass: 4097 x 100 x
    // 100 14.0 and 13.9, 21.8 and 19.0; 1000 x 768 x 768 19.5 and 26.5, 22.1 and 28.8.
    const ProductPlan six = plan_products(&d, 1, 6, sms);
    p.planes = six.cycles <= p.product.cycles + 5000;
    if (p.planes) p.product = six;
  }
  auto packed = [&](const void* src, size_t rows, size_t stride) -> size_t {
    if (in_place(l.dtype, src, rows, stride)) return 0;
    return l.dtype == QV_DTYPE_F32 ? scaled_bytes(rows, l.k) : packed_bytes(l.dtype, rows, l.k);
  };
  p.bytes += packed(l.x, l.m, l.x_stride) + packed(l.weight, l.n, l.weight_stride);
  if (l.dtype == QV_DTYPE_F32 && !p.planes) p.bytes += kChoiceBytes;
  p.bytes += p.product.partial_bytes[0];
  return p;
}

template <class T, int kRows, int kCols>
void launch_few(const qv_linear& l, const Epilogue& ep, cudaStream_t st) {
  const size_t e = sizeof(T);
  const int align = common_align({reinterpret_cast<uintptr_t>(l.x),
                                  reinterpret_cast<uintptr_t>(l.weight),
                                  l.m > 1 ? l.x_stride * e : 0, l.n > 1 ? l.weight_stride * e : 0,
                                  l.k * e});
  const dim3 blocks(static_cast<unsigned>(ceil_div(l.n, 4 * kCols)),
                    static_cast<unsigned>(ceil_div(l.m, kRows)));
  auto go = [&](auto v) {
    constexpr int kV = decltype(v)::value;
    few_rows_kernel<T, kRows, kCols, kV><<<blocks, 128, 0, st>>>(
        static_cast<const T*>(l.x), static_cast<int64_t>(l.x_stride),
        static_cast<const T*>(l.weight), static_cast<int64_t>(l.weight_stride),
        static_cast<int>(l.m), static_cast<int64_t>(l.n), static_cast<int64_t>(l.k), ep);
  };
  if (align == 16)
    go(std::integral_constant<int, 16 / sizeof(T)>{});
  else if (align == 8)
    go(std::integral_constant<int, 8 / sizeof(T)>{});
  else
    go(std::integral_constant<int, 1>{});
  check_launch("few_rows_kernel");
}
template <class T>
void launch_few(const qv_linear& l, const Epilogue& ep, cudaStream_t st) {
  const bool wide = l.n >= kWideFew;
  if (l.m == 1)
    launch_few<T, 1, 1>(l, ep, st);
  else if (l.m == 2)
    wide ? launch_few<T, 2, 2>(l, ep, st) : launch_few<T, 2, 1>(l, ep, st);
  else if (l.m <= 4)
    wide ? launch_few<T, 4, 2>(l, ep, st) : launch_few<T, 4, 1>(l, ep, st);
  else
    wide ? launch_few<T, 8, 2>(l, ep, st) : launch_few<T, 8, 1>(l, ep, st);
}

}  // namespace

size_t linear_workspace(const qv_linear& l, int sms) {
  check_linear(l);
  return linear_plan(l, sms).bytes;
}

void linear_forward(const qv_linear& l, void* workspace, size_t workspace_bytes, int sms,
                    cudaStream_t st) {
  check_linear(l);
  if (l.m == 0) return;
  const LinearPlan p = linear_plan(l, sms);
  QV_REQUIRE(p.bytes == 0 || (workspace != nullptr && workspace_bytes >= p.bytes),
             "workspace too small: qv_linear_workspace tells the size");
  QV_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 256 == 0 || p.bytes == 0,
             "workspace must be 256-byte aligned");
  const Epilogue ep = epilogue_of(l);
  by_type(l.dtype, [&](auto t) {
    using T = decltype(t);
    if (p.few) {
      launch_few<T>(l, ep, st);
      return;
    }
    Packer<T> pack(l.dtype, true, p.planes, static_cast<unsigned char*>(workspace));
    Product d{};
    d.m = static_cast<int64_t>(l.m);
    d.n = static_cast<int64_t>(l.n);
    d.k = static_cast<int64_t>(l.k);
    d.a = pack.rows(l.x, l.m, l.k, l.x_stride);
    d.b = pack.rows(l.weight, l.n, l.k, l.weight_stride);
    d.ep = ep;
    const bool packed = pack.count() > 0;
    unsigned char* partial = pack.run(false, st);
    d.wide = pack.wide();
    run_products<T>(&d, 1, p.product, partial, SumsJob{}, packed, sms, st);
  });
}

// ---- gradients -------------------------------------------------------------------------------------

namespace {

// The type of everything but the gradient, and whether that is float32.
uint32_t grad_dtype(const qv_linear_grad& g) { return g.dtype & ~static_cast<uint32_t>(QV_GRAD_F32); }
bool grad_f32(const qv_linear_grad& g) {
  return (g.dtype & QV_GRAD_F32) != 0 || g.dtype == QV_DTYPE_F32;
}

void check_linear_grad(const qv_linear_grad& g) {
  const uint32_t dtype = grad_dtype(g);
  check_dtype(dtype);
  QV_REQUIRE(g.activation <= QV_ACT_SILU, "unknown activation");
  QV_REQUIRE(g.k >= 1 && g.k <= kMaxDim && g.n >= 1 && g.n <= kMaxDim,
             "dimensions must be between 1 and 65536");
  QV_REQUIRE(g.m <= kMaxLinearRows, "too many rows");
  if (g.dweight != nullptr)
    check_matrix("dweight", dtype, g.dweight, g.n, g.k, g.dweight_stride);
  if (g.dbias != nullptr) check_matrix("dbias", dtype, g.dbias, 1, g.n, g.n);
  if (g.m == 0) return;
  check_matrix("grad", grad_f32(g) ? QV_DTYPE_F32 : dtype, g.grad, g.m, g.n, g.grad_stride);
  if (g.activation != QV_ACT_NONE)
    check_matrix("preact", dtype, g.preact, g.m, g.n, g.preact_stride);
  if (g.dx != nullptr) {
    check_matrix("weight", dtype, g.weight, g.n, g.k, g.weight_stride);
    check_matrix("dx", dtype, g.dx, g.m, g.k, g.dx_stride);
  }
  if (g.dweight != nullptr) check_matrix("x", dtype, g.x, g.m, g.k, g.x_stride);
}

struct GradLayout {
  bool wide_dz = false;       // 16-byte pieces of the gradient, and as many preactivations
  bool store_dz = false;      // dz is not the caller's gradient itself
  size_t row_blocks = 0;      // row ranges of the column sums
  int64_t rows_per_block = 0;
  Product products[2];        // dx and dweight, those that are asked for
  int count = 0;
  ProductPlan plan;
  size_t off_dz = 0, off_sums = 0, off_packed = 0, off_partial = 0, bytes = 0;
};
GradLayout grad_layout(const qv_linear_grad& g, int sms) {
  GradLayout L;
  if (g.m == 0) return L;
  const uint32_t dtype = grad_dtype(g);
  const int pairs = dtype == QV_DTYPE_F32 ? 6 : 1;
  const bool products = g.dx != nullptr || g.dweight != nullptr;
  L.store_dz = products && (g.activation != QV_ACT_NONE || (grad_f32(g) && dtype != QV_DTYPE_F32) ||
                            !in_place(dtype, g.grad, g.m, g.grad_stride));
  const size_t e = dtype_size(dtype), ge = grad_f32(g) ? 4 : e;
  L.wide_dz = common_align({reinterpret_cast<uintptr_t>(g.grad), g.m > 1 ? g.grad_stride * ge : 0,
                            g.n * ge}) == 16 &&
              common_align({reinterpret_cast<uintptr_t>(g.preact),
                            g.m > 1 ? g.preact_stride * e : 0}) >= static_cast<int>(16 / ge * e);
  // About eight blocks an SM, each with at least one round of its warps.
  const size_t col_blocks = ceil_div(g.n, L.wide_dz ? 32 * 16 / ge : 32 * dz_pieces(e));
  L.row_blocks = std::min<size_t>(ceil_div(g.m, kDzWarps * kDzRows),
                                  std::max<size_t>(1, sms * 8 / col_blocks));
  L.rows_per_block = static_cast<int64_t>(ceil_div(g.m, L.row_blocks));
  L.row_blocks = ceil_div(g.m, L.rows_per_block);
  size_t o = 0;
  auto take = [&](size_t bytes) {
    const size_t at = o;
    o += (bytes + 255) / 256 * 256;
    return at;
  };
  L.off_dz = take(L.store_dz ? packed_bytes(dtype, g.m, g.n) : 0);
  L.off_sums = take(g.dbias != nullptr ? L.row_blocks * g.n * sizeof(float) : 0);
  L.off_packed = o;
  // dweight first: its units are the longest where there are many rows.
  if (g.dweight != nullptr) {
    Product& d = L.products[L.count++];
    d = Product{};
    d.m = static_cast<int64_t>(g.n);
    d.n = static_cast<int64_t>(g.k);
    d.k = static_cast<int64_t>(g.m);
    d.a_mn = d.b_mn = true;
    if (!in_place(dtype, g.x, g.m, g.x_stride)) take(packed_bytes(dtype, g.m, g.k));
  }
  if (g.dx != nullptr) {
    Product& d = L.products[L.count++];
    d = Product{};
    d.m = static_cast<int64_t>(g.m);
    d.n = static_cast<int64_t>(g.k);
    d.k = static_cast<int64_t>(g.n);
    d.b_mn = true;
    if (!in_place(dtype, g.weight, g.n, g.weight_stride)) take(packed_bytes(dtype, g.n, g.k));
  }
  if (L.count > 0) L.plan = plan_products(L.products, L.count, pairs, sms);
  L.off_partial = take(L.plan.partial_bytes[0] + L.plan.partial_bytes[1]);
  L.bytes = o;
  return L;
}

}  // namespace

size_t linear_grad_workspace(const qv_linear_grad& g, int sms) {
  check_linear_grad(g);
  return grad_layout(g, sms).bytes;
}

void linear_grad(const qv_linear_grad& g, void* workspace, size_t workspace_bytes, int sms,
                 cudaStream_t st) {
  check_linear_grad(g);
  const uint32_t dtype = grad_dtype(g);
  const size_t e = dtype_size(dtype);
  if (g.m == 0) {  // no rows: the sums over them are zero
    if (g.dweight != nullptr)
      QV_CUDA(cudaMemset2DAsync(g.dweight, std::max(g.dweight_stride, g.k) * e, 0, g.k * e, g.n,
                                st));
    if (g.dbias != nullptr) QV_CUDA(cudaMemsetAsync(g.dbias, 0, g.n * e, st));
    return;
  }
  GradLayout L = grad_layout(g, sms);
  QV_REQUIRE(L.bytes == 0 || (workspace != nullptr && workspace_bytes >= L.bytes),
             "workspace too small: qv_linear_grad_workspace tells the size");
  QV_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 256 == 0 || L.bytes == 0,
             "workspace must be 256-byte aligned");
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  by_type(dtype, [&](auto t) {
    using T = decltype(t);
    using O = typename Operand<T>::type;
    const int64_t m = g.m, n = g.n;
    float* sums = g.dbias != nullptr ? reinterpret_cast<float*>(ws + L.off_sums) : nullptr;
    Stored dz;
    dz.inner = n;
    dz.outer = m;
    dz.bf16 = dtype != QV_DTYPE_F16;
    if (L.store_dz || sums != nullptr) {
      O* store = reinterpret_cast<O*>(ws + L.off_dz);
      const int64_t ld = static_cast<int64_t>(packed_ld(g.n));
      auto launch = [&](auto type, auto v, auto act) {
        using G = decltype(type);
        constexpr int kV = decltype(v)::value;
        constexpr int kAct = decltype(act)::value;
        const dim3 grid(static_cast<unsigned>(L.row_blocks),
                        static_cast<unsigned>(ceil_div(g.n, 32 * kV * dz_pieces(sizeof(T) * kV))));
        auto* kernel = L.store_dz ? dz_kernel<T, G, kV, true, kAct> : dz_kernel<T, G, kV, false, kAct>;
        kernel<<<grid, 32 * kDzWarps, 0, st>>>(
            static_cast<const G*>(g.grad), g.grad_stride, static_cast<const T*>(g.preact),
            g.preact_stride, m, n, L.rows_per_block, store, ld, sums);
      };
      auto go = [&](auto wide, auto act) {
        auto by_grad = [&](auto type) {
          constexpr int kV = decltype(wide)::value ? 16 / static_cast<int>(sizeof(type)) : 1;
          launch(type, std::integral_constant<int, kV>{}, act);
        };
        if (grad_f32(g))
          by_grad(float{});
        else
          by_grad(T{});
      };
      auto by_act = [&](auto v) {
        switch (g.activation) {
          case QV_ACT_RELU: go(v, std::integral_constant<int, QV_ACT_RELU>{}); break;
          case QV_ACT_GELU: go(v, std::integral_constant<int, QV_ACT_GELU>{}); break;
          case QV_ACT_GELU_TANH: go(v, std::integral_constant<int, QV_ACT_GELU_TANH>{}); break;
          case QV_ACT_SILU: go(v, std::integral_constant<int, QV_ACT_SILU>{}); break;
          default: go(v, std::integral_constant<int, QV_ACT_NONE>{}); break;
        }
      };
      if (L.wide_dz)
        by_act(std::true_type{});
      else
        by_act(std::false_type{});
      check_launch("dz_kernel");
    }
    if (L.store_dz) {
      dz.p = ws + L.off_dz;
      dz.ld = static_cast<int64_t>(packed_ld(g.n));
      dz.planes = std::is_same_v<T, float> ? 3 : 1;
    } else {
      dz.p = g.grad;
      dz.ld = static_cast<int64_t>(g.grad_stride);
    }
    Packer<T> pack(dtype, false, false, ws + L.off_packed);
    auto result = [&](void* p, size_t stride) {
      Epilogue ep{};
      ep.out = p;
      ep.out_stride = static_cast<int64_t>(stride);
      ep.out_f32 = dtype == QV_DTYPE_F32;
      ep.set_aligns(e);
      return ep;
    };
    int q = 0;
    if (g.dweight != nullptr) {
      Product& d = L.products[q++];
      d.a = dz;
      d.b = pack.rows(g.x, g.m, g.k, g.x_stride);
      d.ep = result(g.dweight, g.dweight_stride);
    }
    if (g.dx != nullptr) {
      Product& d = L.products[q++];
      d.a = dz;
      d.b = pack.rows(g.weight, g.n, g.k, g.weight_stride);
      d.ep = result(g.dx, g.dx_stride);
    }
    const bool first = L.store_dz || sums != nullptr;  // the dz kernel ran
    const bool chained = first || pack.count() > 0;
    pack.run(first, st);
    SumsJob sj{};
    if (sums != nullptr) sj = SumsJob{sums, static_cast<int>(L.row_blocks), n, g.dbias};
    run_products<T>(L.products, L.count, L.plan, ws + L.off_partial, sj, chained, sms, st);
  });
}

}  // namespace qv

extern "C" {

qv_status qv_linear_workspace(int device, const qv_linear* args, size_t* bytes) {
  return qv::guarded([&] {
    QV_REQUIRE(args != nullptr && bytes != nullptr, "null argument");
    *bytes = qv::linear_workspace(*args, qv::sm_count(device));
  });
}

qv_status qv_linear_device(int device, const qv_linear* args, void* workspace,
                           size_t workspace_bytes, void* stream) {
  return qv::guarded([&] {
    QV_REQUIRE(args != nullptr, "null argument");
    qv::DeviceScope scope(device);
    qv::linear_forward(*args, workspace, workspace_bytes, qv::sm_count(device),
                       static_cast<cudaStream_t>(stream));
  });
}

qv_status qv_linear_grad_workspace(int device, const qv_linear_grad* args, size_t* bytes) {
  return qv::guarded([&] {
    QV_REQUIRE(args != nullptr && bytes != nullptr, "null argument");
    *bytes = qv::linear_grad_workspace(*args, qv::sm_count(device));
  });
}

qv_status qv_linear_grad_device(int device, const qv_linear_grad* args, void* workspace,
                                size_t workspace_bytes, void* stream) {
  return qv::guarded([&] {
    QV_REQUIRE(args != nullptr, "null argument");
    qv::DeviceScope scope(device);
    qv::linear_grad(*args, workspace, workspace_bytes, qv::sm_count(device),
                    static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
