// Embedding tables: rows by id with a scale, and the table's gradient from sorted ids.
//
//   lookup: out[i] = scale * table[ids[i]]           (one rounding, from float32)
//   grad:   grad[r] = scale * sum_{i: ids[i] = r} up[i]   (float32 sums, i ascending)
//
// Both move bytes and compute next to nothing: n rows read and n written, and n rows read and
// all rows of the table written.
#include "embed.cuh"

namespace qv {
namespace {

using dev::Pack;

template <class Id>
__device__ __forceinline__ int64_t load_id(const void* ids, size_t i) {
  return static_cast<int64_t>(static_cast<const Id*>(ids)[i]);
}

// ---- lookup ------------------------------------------------------------------------------------
// The output as one run of n * nv pieces of kV elements: every thread takes kUnroll pieces, so
// short rows leave no lanes idle and each thread has several loads in flight.
constexpr int kLookupThreads = 256, kLookupUnroll = 4;

template <class T, class Id, int kV>
__global__ void __launch_bounds__(kLookupThreads)
    lookup_kernel(const T* __restrict__ table, int64_t rows, int64_t table_stride,
                  const void* __restrict__ ids, size_t n, uint32_t nv, float scale,
                  T* __restrict__ out, int64_t out_stride) {
  constexpr uint32_t kTile = kLookupThreads * kLookupUnroll;
  const uint64_t first = static_cast<uint64_t>(blockIdx.x) * kTile;
  const uint64_t i0 = first / nv;
  const uint32_t v0 = static_cast<uint32_t>(first - i0 * nv);
  Pack<T, kV> x[kLookupUnroll];
  uint64_t row[kLookupUnroll];
  uint32_t col[kLookupUnroll];
  int state[kLookupUnroll];  // 0: past the end, 1: a row, 2: zeros (id < 0), 3: NaN (id >= rows)
#pragma unroll
  for (int u = 0; u < kLookupUnroll; ++u) {
    const uint32_t p = v0 + u * kLookupThreads + threadIdx.x;
    const uint32_t q = p / nv;
    row[u] = i0 + q;
    col[u] = (p - q * nv) * kV;
    state[u] = 0;
    if (row[u] >= n) continue;
    const int64_t id = load_id<Id>(ids, row[u]);
    state[u] = id < 0 ? 2 : id >= rows ? 3 : 1;
    if (state[u] == 1) x[u] = dev::load_pack<T, kV>(table + id * table_stride + col[u]);
  }
#pragma unroll
  for (int u = 0; u < kLookupUnroll; ++u) {
    if (state[u] == 0) continue;
    Pack<T, kV> y;
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      const float f = state[u] == 1 ? dev::to_f32<T>(x[u].v[j]) * scale
                                    : (state[u] == 2 ? 0.0f : __int_as_float(0x7fc00000));
      y.v[j] = dev::from_f32<T>(f);
    }
    dev::store_pack<T, kV>(out + static_cast<int64_t>(row[u]) * out_stride + col[u], y);
  }
}

template <class T, class Id, int kV>
void launch_lookup(const void* table, size_t rows, size_t dim, size_t table_stride,
                   const void* ids, size_t n, float scale, void* out, size_t out_stride,
                   cudaStream_t st) {
  const uint32_t nv = static_cast<uint32_t>(dim / kV);
  const size_t blocks = ceil_div(n * nv, kLookupThreads * kLookupUnroll);
  lookup_kernel<T, Id, kV><<<static_cast<unsigned>(blocks), kLookupThreads, 0, st>>>(
      static_cast<const T*>(table), static_cast<int64_t>(rows),
      static_cast<int64_t>(table_stride), ids, n, nv, scale, static_cast<T*>(out),
      static_cast<int64_t>(out_stride));
  check_launch("lookup_kernel");
}

// ---- gradient: sorting ids -----------------------------------------------------------------------
// Stable least-significant-digit radix sort of (id, position) pairs; ids that take no gradient
// (negative or past the table) become `rows` and end up last. Each pass: per-tile digit counts,
// a prefix over tiles per digit, and a scatter that ranks a tile's entries in input order.
constexpr int kSortThreads = 256, kSortItems = 8;
constexpr int kSortTile = kSortThreads * kSortItems;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxDigitBits = 11;

__device__ __forceinline__ uint32_t clip_id(int64_t id, uint32_t rows) {
  return id < 0 || id >= static_cast<int64_t>(rows) ? rows : static_cast<uint32_t>(id);
}

// Key of entry i: from the caller's ids in the first pass, from sorted keys afterwards.
template <class Id, bool kFirst>
__device__ __forceinline__ uint32_t sort_key(const void* src, size_t i, uint32_t rows) {
  return kFirst ? clip_id(load_id<Id>(src, i), rows) : static_cast<const uint32_t*>(src)[i];
}

template <class Id, bool kFirst>
__global__ void __launch_bounds__(kSortThreads)
    digit_count_kernel(const void* __restrict__ src, uint32_t n, uint32_t rows, int shift,
                       int bits, uint32_t tiles, uint32_t* __restrict__ counts) {
  extern __shared__ uint32_t hist[];
  const int bins = 1 << bits;
  for (int b = threadIdx.x; b < bins; b += kSortThreads) hist[b] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const uint32_t i = blockIdx.x * kSortTile + j * kSortThreads + threadIdx.x;
    if (i < n) atomicAdd(&hist[(sort_key<Id, kFirst>(src, i, rows) >> shift) & (bins - 1)], 1u);
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += kSortThreads)
    counts[static_cast<size_t>(b) * tiles + blockIdx.x] = hist[b];
}

// One warp per digit: its tiles' counts become the entries of that digit in earlier tiles;
// totals[digit] their sum.
__global__ void digit_scan_kernel(uint32_t* __restrict__ counts, int bins, uint32_t tiles,
                                  uint32_t* __restrict__ totals) {
  const int b = (blockIdx.x * blockDim.x + threadIdx.x) >> 5, lane = threadIdx.x & 31;
  if (b >= bins) return;
  uint32_t* c = counts + static_cast<size_t>(b) * tiles;
  uint32_t sum = 0;
  for (uint32_t t0 = 0; t0 < tiles; t0 += 32) {
    const uint32_t t = t0 + lane;
    const uint32_t v = t < tiles ? c[t] : 0;
    uint32_t s = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t o = __shfl_up_sync(dev::kFull, s, d);
      if (lane >= d) s += o;
    }
    if (t < tiles) c[t] = sum + s - v;
    sum += __shfl_sync(dev::kFull, s, 31);
  }
  if (lane == 0) totals[b] = sum;
}

template <class Id, bool kFirst>
__global__ void __launch_bounds__(kSortThreads)
    digit_scatter_kernel(const void* __restrict__ src, const uint32_t* __restrict__ src_pos,
                         uint32_t n, uint32_t rows, int shift, int bits, uint32_t tiles,
                         const uint32_t* __restrict__ counts,
                         const uint32_t* __restrict__ totals, uint32_t* __restrict__ keys,
                         uint32_t* __restrict__ pos) {
  extern __shared__ uint32_t smem[];
  const int bins = 1 << bits;
  uint32_t* base = smem;                                             // bins: first slot of a digit
  uint16_t* wcount = reinterpret_cast<uint16_t*>(smem + bins);       // kSortWarps x bins
  __shared__ uint32_t wsum[kSortWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int b = threadIdx.x; b < kSortWarps * bins; b += kSortThreads) wcount[b] = 0;
  // Exclusive prefix of the digits' totals: each thread sums a run of digits.
  const int per = (bins + kSortThreads - 1) / kSortThreads;
  uint32_t mine = 0;
  for (int j = 0; j < per; ++j) {
    const int b = threadIdx.x * per + j;
    if (b < bins) mine += totals[b];
  }
  uint32_t s = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t o = __shfl_up_sync(dev::kFull, s, d);
    if (lane >= d) s += o;
  }
  if (lane == 31) wsum[warp] = s;
  __syncthreads();
  uint32_t run = s - mine;
  for (int w = 0; w < warp; ++w) run += wsum[w];
  for (int j = 0; j < per; ++j) {
    const int b = threadIdx.x * per + j;
    if (b < bins) {
      base[b] = run + counts[static_cast<size_t>(b) * tiles + blockIdx.x];
      run += totals[b];
    }
  }
  // Each warp ranks its own run of 32 * kSortItems entries in order.
  uint32_t key[kSortItems], p[kSortItems];
  uint32_t rank[kSortItems];
  uint16_t* wc = wcount + warp * bins;
  const uint32_t first = blockIdx.x * kSortTile + warp * (32 * kSortItems);
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const uint32_t i = first + j * 32 + lane;
    key[j] = i < n ? sort_key<Id, kFirst>(src, i, rows) : 0u;
    p[j] = kFirst ? i : (i < n ? src_pos[i] : 0u);
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const uint32_t i = first + j * 32 + lane;
    // Entries past the end match only each other (a value no digit has).
    const uint32_t digit = i < n ? (key[j] >> shift) & (bins - 1) : 0xffffffffu;
    const uint32_t same = __match_any_sync(dev::kFull, digit);
    const uint32_t before = __popc(same & ((1u << lane) - 1));
    rank[j] = i < n ? wc[digit] + before : 0u;
    __syncwarp();
    if (i < n && before == 0) wc[digit] = static_cast<uint16_t>(wc[digit] + __popc(same));
    __syncwarp();
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += kSortThreads) {
    uint32_t acc = 0;
    for (int w = 0; w < kSortWarps; ++w) {
      const uint32_t c = wcount[w * bins + b];
      wcount[w * bins + b] = static_cast<uint16_t>(acc);
      acc += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const uint32_t i = first + j * 32 + lane;
    if (i >= n) continue;
    const uint32_t digit = (key[j] >> shift) & (bins - 1);
    const uint32_t o = base[digit] + wc[digit] + rank[j];
    keys[o] = key[j];
    pos[o] = p[j];
  }
}

// ---- gradient: segmented sums ---------------------------------------------------------------------
// The sorted entries and the table's rows are one sequence: each row's entries, then its row end.
// Entry e stands at place key[e] + e of it. Equal runs of that sequence go to the units (warps),
// so a token that fills a tenth of the batch is shared out and empty rows cost what they write.
// A row that begins in one unit and ends in another is joined afterwards from the units' partial
// sums, in order: tail[u] is what unit u summed of a row it did not end, head[u] what it summed
// of the row it ended that began before it.

// Number of entries among the first d places of the sequence: the first e with key[e] + e >= d,
// found by a warp in 32-way steps.
__device__ __forceinline__ uint32_t entries_before(const uint32_t* __restrict__ keys, uint32_t n,
                                                   uint64_t d, int lane) {
  uint32_t lo = 0, hi = n;  // the answer is in [lo, hi]
  while (lo < hi) {
    const uint32_t len = hi - lo;
    const uint32_t step = (len + 31) / 32;
    const uint32_t e = lo + lane * step;
    const bool in = e < hi && static_cast<uint64_t>(keys[e]) + e < d;
    const uint32_t m = __ballot_sync(dev::kFull, in);
    if (m == 0) return lo;
    const uint32_t last = lo + (31 - __clz(m)) * step;  // the last probe that is before d
    lo = last + 1;
    hi = min(hi, last + step);
  }
  return lo;
}

constexpr int kSumThreads = 256;
constexpr int kSumBatch = 8;  // rows in flight per lane

template <class T, int kV>
__global__ void __launch_bounds__(kSumThreads)
    segment_sum_kernel(const T* __restrict__ up, int64_t up_stride,
                       const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos,
                       uint32_t n, uint32_t rows, uint32_t dim, uint32_t run, uint32_t units,
                       float scale, T* __restrict__ grad, int64_t grad_stride,
                       float* __restrict__ head, float* __restrict__ tail) {
  const int lane = threadIdx.x & 31;
  const uint32_t unit = (blockIdx.x * kSumThreads + threadIdx.x) >> 5;
  if (unit >= units) return;
  const uint32_t c = (blockIdx.y * 32 + lane) * kV;
  const bool on = c < dim;
  const uint64_t total = static_cast<uint64_t>(rows) + n;
  const uint64_t d0 = static_cast<uint64_t>(unit) * run;
  const uint64_t d1 = d0 + run < total ? d0 + run : total;
  const uint32_t e0 = entries_before(keys, n, d0, lane);
  const uint32_t e1 = entries_before(keys, n, d1, lane);
  uint32_t r = static_cast<uint32_t>(d0 - e0);
  const uint32_t r1 = static_cast<uint32_t>(d1 - e1);
  bool began_before = e0 > 0 && keys[e0 - 1] == r;  // row r has entries in an earlier unit
  float acc[kV];
#pragma unroll
  for (int j = 0; j < kV; ++j) acc[j] = 0.0f;
  bool open = false;
  auto finish_row = [&]() {
    if (on) {
      if (began_before) {
#pragma unroll
        for (int j = 0; j < kV; ++j) head[static_cast<size_t>(unit) * dim + c + j] = acc[j];
      } else {
        Pack<T, kV> y;
#pragma unroll
        for (int j = 0; j < kV; ++j) y.v[j] = dev::from_f32<T>(acc[j] * scale);
        dev::store_pack<T, kV>(grad + static_cast<int64_t>(r) * grad_stride + c, y);
      }
    }
#pragma unroll
    for (int j = 0; j < kV; ++j) acc[j] = 0.0f;
    began_before = false;
    open = false;
    ++r;
  };
  for (uint32_t e = e0; e < e1; e += 32) {
    const uint32_t mine = e + lane;
    const uint32_t my_key = mine < e1 ? keys[mine] : rows;
    const uint32_t my_pos = mine < e1 ? pos[mine] : 0u;
    const int count = static_cast<int>(min(32u, e1 - e));
    for (int b = 0; b < count; b += kSumBatch) {
      Pack<T, kV> x[kSumBatch];
#pragma unroll
      for (int j = 0; j < kSumBatch; ++j) {
        const uint32_t p = __shfl_sync(dev::kFull, my_pos, (b + j) & 31);
        if (on && b + j < count) x[j] = dev::load_pack<T, kV>(up + static_cast<int64_t>(p) * up_stride + c);
      }
#pragma unroll
      for (int j = 0; j < kSumBatch; ++j) {
        if (b + j >= count) break;
        const uint32_t k = __shfl_sync(dev::kFull, my_key, b + j);
        while (r < k) finish_row();
        if (on) {
#pragma unroll
          for (int v = 0; v < kV; ++v) acc[v] += dev::to_f32<T>(x[j].v[v]);
        }
        open = true;
      }
    }
  }
  while (r < r1) finish_row();
  if (open && on) {
#pragma unroll
    for (int j = 0; j < kV; ++j) tail[static_cast<size_t>(unit) * dim + c + j] = acc[j];
  }
}

// Unit u's first row, when it began in an earlier unit and ends in u: the tails of the units from
// the one it began in up to u - 1, in order, and head[u]. One warp per unit and 32 columns.
template <class T>
__global__ void __launch_bounds__(kSumThreads)
    join_rows_kernel(const uint32_t* __restrict__ keys, uint32_t n, uint32_t rows, uint32_t dim,
                     uint32_t run, uint32_t units, float scale, T* __restrict__ grad,
                     int64_t grad_stride, const float* __restrict__ head,
                     const float* __restrict__ tail) {
  const int lane = threadIdx.x & 31;
  const uint32_t unit = (blockIdx.x * kSumThreads + threadIdx.x) >> 5;
  if (unit == 0 || unit >= units) return;
  const uint64_t total = static_cast<uint64_t>(rows) + n;
  const uint64_t d0 = static_cast<uint64_t>(unit) * run;
  const uint64_t d1 = d0 + run < total ? d0 + run : total;
  const uint32_t e0 = entries_before(keys, n, d0, lane);
  const uint32_t r = static_cast<uint32_t>(d0 - e0);
  if (e0 == 0 || r >= rows || keys[e0 - 1] != r) return;
  // The row ends here iff its row end, after its last entry, is one of this unit's places.
  const uint32_t e1 = entries_before(keys, n, d1, lane);
  if (static_cast<uint32_t>(d1 - e1) <= r) return;
  uint32_t first = 0, hi = e0 - 1;  // the row's first entry: keys[first] == r
  while (first < hi) {
    const uint32_t mid = (first + hi) / 2;
    if (keys[mid] < r) first = mid + 1; else hi = mid;
  }
  const uint32_t u0 = static_cast<uint32_t>((static_cast<uint64_t>(r) + first) / run);
  for (uint32_t c = blockIdx.y * 32 + lane; c < dim; c += gridDim.y * 32) {
    float s = 0.0f;
    for (uint32_t u = u0; u < unit; ++u) s += tail[static_cast<size_t>(u) * dim + c];
    s += head[static_cast<size_t>(unit) * dim + c];
    grad[static_cast<int64_t>(r) * grad_stride + c] = dev::from_f32<T>(s * scale);
  }
}

struct GradPlan {
  int passes, bits;         // radix passes and digit width
  uint32_t tiles;           // sort tiles
  uint32_t run, units;      // places per unit, units
  size_t off_keys[2], off_pos[2], off_counts, off_totals, off_head, off_tail, bytes;
};

GradPlan grad_plan(size_t n, size_t rows, size_t dim) {
  GradPlan p{};
  int bits = 1;
  while ((size_t{1} << bits) <= rows) ++bits;  // keys 0 .. rows
  p.passes = static_cast<int>(ceil_div(bits, kMaxDigitBits));
  p.bits = static_cast<int>(ceil_div(bits, p.passes));
  p.tiles = static_cast<uint32_t>(ceil_div(n, kSortTile));
  p.run = static_cast<uint32_t>(std::max<size_t>(32, ceil_div(n + rows, 148 * 64)));
  p.units = static_cast<uint32_t>(ceil_div(n + rows, p.run));
  size_t o = 0;
  auto take = [&](size_t bytes) {
    const size_t at = o;
    o += (bytes + 255) / 256 * 256;
    return at;
  };
  for (int i = 0; i < 2; ++i) {
    p.off_keys[i] = take(n * 4);
    p.off_pos[i] = take(n * 4);
  }
  p.off_counts = take((size_t{1} << p.bits) * p.tiles * 4);
  p.off_totals = take((size_t{1} << p.bits) * 4);
  p.off_head = take(p.units * dim * 4);
  p.off_tail = take(p.units * dim * 4);
  p.bytes = o;
  return p;
}

template <class Id>
int sort_ids(const GradPlan& p, const void* ids, uint32_t n, uint32_t rows, unsigned char* ws,
             cudaStream_t st) {
  uint32_t* counts = reinterpret_cast<uint32_t*>(ws + p.off_counts);
  uint32_t* totals = reinterpret_cast<uint32_t*>(ws + p.off_totals);
  const int bins = 1 << p.bits;
  const size_t smem = bins * 4 + static_cast<size_t>(kSortWarps) * bins * 2;
  for (int k = 0; k < p.passes; ++k) {
    uint32_t* ok = reinterpret_cast<uint32_t*>(ws + p.off_keys[k & 1]);
    uint32_t* op = reinterpret_cast<uint32_t*>(ws + p.off_pos[k & 1]);
    const uint32_t* ik = reinterpret_cast<uint32_t*>(ws + p.off_keys[(k & 1) ^ 1]);
    const uint32_t* ip = reinterpret_cast<uint32_t*>(ws + p.off_pos[(k & 1) ^ 1]);
    const int shift = k * p.bits;
    if (k == 0)
      digit_count_kernel<Id, true><<<p.tiles, kSortThreads, bins * 4, st>>>(
          ids, n, rows, shift, p.bits, p.tiles, counts);
    else
      digit_count_kernel<Id, false><<<p.tiles, kSortThreads, bins * 4, st>>>(
          ik, n, rows, shift, p.bits, p.tiles, counts);
    check_launch("digit_count_kernel");
    digit_scan_kernel<<<static_cast<unsigned>(ceil_div(bins, 8)), 256, 0, st>>>(counts, bins,
                                                                               p.tiles, totals);
    check_launch("digit_scan_kernel");
    if (k == 0)
      digit_scatter_kernel<Id, true><<<p.tiles, kSortThreads, smem, st>>>(
          ids, nullptr, n, rows, shift, p.bits, p.tiles, counts, totals, ok, op);
    else
      digit_scatter_kernel<Id, false><<<p.tiles, kSortThreads, smem, st>>>(
          ik, ip, n, rows, shift, p.bits, p.tiles, counts, totals, ok, op);
    check_launch("digit_scatter_kernel");
  }
  return (p.passes - 1) & 1;
}

template <class T, int kV>
void launch_sums(const GradPlan& p, int which, const void* up, size_t up_stride, uint32_t n,
                 uint32_t rows, uint32_t dim, float scale, void* grad, size_t grad_stride,
                 unsigned char* ws, cudaStream_t st) {
  const uint32_t* keys = reinterpret_cast<uint32_t*>(ws + p.off_keys[which]);
  const uint32_t* pos = reinterpret_cast<uint32_t*>(ws + p.off_pos[which]);
  float* head = reinterpret_cast<float*>(ws + p.off_head);
  float* tail = reinterpret_cast<float*>(ws + p.off_tail);
  const unsigned blocks = static_cast<unsigned>(ceil_div(p.units, kSumThreads / 32));
  segment_sum_kernel<T, kV>
      <<<dim3(blocks, static_cast<unsigned>(ceil_div(dim, 32 * kV))), kSumThreads, 0, st>>>(
          static_cast<const T*>(up), static_cast<int64_t>(up_stride), keys, pos, n, rows, dim,
          p.run, p.units, scale, static_cast<T*>(grad), static_cast<int64_t>(grad_stride), head,
          tail);
  check_launch("segment_sum_kernel");
  join_rows_kernel<T>
      <<<dim3(blocks, static_cast<unsigned>(std::min<size_t>(ceil_div(dim, 32), 65535))),
         kSumThreads, 0, st>>>(keys, n, rows, dim, p.run, p.units, scale, static_cast<T*>(grad),
                               static_cast<int64_t>(grad_stride), head, tail);
  check_launch("join_rows_kernel");
}

// ---- argument checks and dispatch -----------------------------------------------------------------

constexpr size_t kMaxEmbedDim = 65536;               // as the indexes' dimension limit
constexpr size_t kMaxRows = (size_t{1} << 31) - 2;   // row numbers are 32-bit inside the sort

void check_ids(uint32_t id_type, const void* ids, size_t n) {
  QV_REQUIRE(id_type == QV_ID_I32 || id_type == QV_ID_I64, "unknown id type");
  QV_REQUIRE(ids != nullptr || n == 0, "null ids");
  const size_t size = id_type == QV_ID_I32 ? 4 : 8;
  QV_REQUIRE(reinterpret_cast<uintptr_t>(ids) % size == 0, "ids are not aligned to their size");
}

void check_rows(const char* what, uint32_t dtype, const void* p, size_t count, size_t dim,
                size_t stride) {
  QV_REQUIRE(p != nullptr || count == 0, std::string("null ") + what);
  QV_REQUIRE(reinterpret_cast<uintptr_t>(p) % dtype_size(dtype) == 0,
             std::string(what) + " is not aligned to its element type");
  QV_REQUIRE(stride >= dim || count <= 1, std::string(what) + ": row stride below the dimension");
  QV_REQUIRE(stride < (size_t{1} << 40), std::string(what) + ": row stride too large");
}

template <class F>
void by_pack(int elem, int align, F&& f) {
  // 16-byte pieces where every address allows it, else the widest that is aligned.
  switch (std::max(elem, align) / elem) {
    case 8: f(std::integral_constant<int, 8>{}); break;
    case 4: f(std::integral_constant<int, 4>{}); break;
    case 2: f(std::integral_constant<int, 2>{}); break;
    default: f(std::integral_constant<int, 1>{}); break;
  }
}

template <class F>
void by_dtype(uint32_t dtype, F&& f) {
  if (dtype == QV_DTYPE_F32)
    f(float{});
  else if (dtype == QV_DTYPE_F16)
    f(__half{});
  else
    f(__nv_bfloat16{});
}

}  // namespace

void embedding_lookup(uint32_t dtype, const void* table, size_t rows, size_t dim,
                      size_t table_stride, uint32_t id_type, const void* ids, size_t n,
                      float scale, void* out, size_t out_stride, cudaStream_t st) {
  check_dtype(dtype);
  check_ids(id_type, ids, n);
  QV_REQUIRE(dim >= 1 && dim <= kMaxEmbedDim, "dimension must be between 1 and 65536");
  QV_REQUIRE(n < (size_t{1} << 40) / dim, "n * dim is too large");
  check_rows("table", dtype, table, rows, dim, table_stride);
  check_rows("out", dtype, out, n, dim, out_stride);
  if (n == 0) return;
  const size_t e = dtype_size(dtype);
  const int align =
      common_align({reinterpret_cast<uintptr_t>(table), reinterpret_cast<uintptr_t>(out),
                    table_stride * e, out_stride * e, dim * e});
  by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    by_pack(sizeof(T), align, [&](auto v) {
      constexpr int kV = decltype(v)::value;
      if constexpr (kV * sizeof(T) <= 16) {
        if (id_type == QV_ID_I32)
          launch_lookup<T, int32_t, kV>(table, rows, dim, table_stride, ids, n, scale, out,
                                        out_stride, st);
        else
          launch_lookup<T, int64_t, kV>(table, rows, dim, table_stride, ids, n, scale, out,
                                        out_stride, st);
      }
    });
  });
}

namespace {
void check_grad_sizes(size_t n, size_t rows, size_t dim) {
  QV_REQUIRE(dim >= 1 && dim <= kMaxEmbedDim, "dimension must be between 1 and 65536");
  QV_REQUIRE(rows <= kMaxRows && n <= kMaxRows, "more than 2^31 - 2 rows");
}
}  // namespace

size_t embedding_grad_workspace(size_t n, size_t rows, size_t dim) {
  check_grad_sizes(n, rows, dim);
  return n == 0 || rows == 0 ? 0 : grad_plan(n, rows, dim).bytes;
}

void embedding_grad(uint32_t dtype, const void* up, size_t up_stride, uint32_t id_type,
                    const void* ids, size_t n, size_t rows, size_t dim, float scale, void* grad,
                    size_t grad_stride, void* workspace, size_t workspace_bytes,
                    cudaStream_t st) {
  check_dtype(dtype);
  check_ids(id_type, ids, n);
  check_grad_sizes(n, rows, dim);
  check_rows("upstream", dtype, up, n, dim, up_stride);
  check_rows("grad", dtype, grad, rows, dim, grad_stride);
  if (rows == 0) return;
  const size_t e = dtype_size(dtype);
  if (n == 0) {
    QV_CUDA(cudaMemset2DAsync(grad, std::max(grad_stride, dim) * e, 0, dim * e, rows, st));
    return;
  }
  const GradPlan p = grad_plan(n, rows, dim);
  QV_REQUIRE(workspace != nullptr && workspace_bytes >= p.bytes,
             "workspace too small: qv_embedding_grad_workspace tells the size");
  QV_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "workspace must be 16-byte aligned");
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  const uint32_t n32 = static_cast<uint32_t>(n), rows32 = static_cast<uint32_t>(rows);
  const int which = id_type == QV_ID_I32 ? sort_ids<int32_t>(p, ids, n32, rows32, ws, st)
                                         : sort_ids<int64_t>(p, ids, n32, rows32, ws, st);
  const int align =
      common_align({reinterpret_cast<uintptr_t>(up), reinterpret_cast<uintptr_t>(grad),
                    up_stride * e, grad_stride * e, dim * e});
  by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    by_pack(sizeof(T), align, [&](auto v) {
      constexpr int kV = decltype(v)::value;
      if constexpr (kV * sizeof(T) <= 16)
        launch_sums<T, kV>(p, which, up, up_stride, n32, rows32, static_cast<uint32_t>(dim),
                           scale, grad, grad_stride, ws, st);
    });
  });
}

}  // namespace qv

extern "C" {

qv_status qv_embedding_lookup_device(int device, uint32_t dtype, const void* table, size_t rows,
                                     size_t dim, size_t table_stride, uint32_t id_type,
                                     const void* ids, size_t n, float scale, void* out,
                                     size_t out_stride, void* stream) {
  return qv::guarded([&] {
    qv::DeviceScope scope(device);
    qv::embedding_lookup(dtype, table, rows, dim, table_stride, id_type, ids, n, scale, out,
                         out_stride, static_cast<cudaStream_t>(stream));
  });
}

qv_status qv_embedding_grad_workspace(size_t n, size_t rows, size_t dim, size_t* bytes) {
  return qv::guarded([&] {
    QV_REQUIRE(bytes != nullptr, "null argument");
    *bytes = qv::embedding_grad_workspace(n, rows, dim);
  });
}

qv_status qv_embedding_grad_device(int device, uint32_t dtype, const void* upstream,
                                   size_t upstream_stride, uint32_t id_type, const void* ids,
                                   size_t n, size_t rows, size_t dim, float scale, void* grad,
                                   size_t grad_stride, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  return qv::guarded([&] {
    qv::DeviceScope scope(device);
    qv::embedding_grad(dtype, upstream, upstream_stride, id_type, ids, n, rows, dim, scale, grad,
                       grad_stride, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
