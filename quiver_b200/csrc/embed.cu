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
// kG lanes share a row and move kV elements at a time, with two to eight pieces in flight per lane
// where the row has more than kG of them, else a piece of each of four rows. Written past the L2's older lines
// (streaming stores), so that the results do not push out table rows other ids will read.
// 131,072 rows of 1024 bfloat16 by a power law of ids: 57 us, 5.9 TB/s of the bytes that have to
// move (64 us with a branch around each load, which then wait for one another; 104 us with one
// thread per piece of the result and a division to find its row).
constexpr int kLookupThreads = 256;

template <class T, int kV>
__device__ __forceinline__ Pack<T, kV> scaled(const Pack<T, kV>& x, float scale) {
  Pack<T, kV> y;
#pragma unroll
  for (int j = 0; j < kV; ++j) y.v[j] = dev::from_f32<T>(dev::to_f32<T>(x.v[j]) * scale);
  return y;
}
template <class T, int kV>
__device__ __forceinline__ Pack<T, kV> filled(float f) {
  Pack<T, kV> y;
#pragma unroll
  for (int j = 0; j < kV; ++j) y.v[j] = dev::from_f32<T>(f);
  return y;
}

template <class T, class Id, int kV, int kG, int kPieces>
__global__ void __launch_bounds__(kLookupThreads)
    lookup_kernel(const T* __restrict__ table, int64_t rows, int64_t table_stride,
                  const Id* __restrict__ ids, int64_t n, int nv, float scale,
                  T* __restrict__ out, int64_t out_stride) {
  constexpr bool kLong = kPieces > 0;  // rows of more than kG pieces, kPieces in flight
  constexpr int kRows = kLong ? 1 : 4;
  constexpr int kGroups = kLookupThreads / kG;
  const int lane = threadIdx.x % kG;
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / kG) * kRows;
  if (first >= n) return;
  const T* src[kRows];
  bool held[kRows];
  float fill[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const int64_t id = first + u < n ? static_cast<int64_t>(ids[first + u]) : -1;
    held[u] = id >= 0 && id < rows;
    src[u] = table + (held[u] ? id : 0) * table_stride;
    fill[u] = id < 0 ? 0.0f : __int_as_float(0x7fc00000);
  }
  T* dst = out + first * out_stride;
  if constexpr (kLong) {
    if (!held[0]) {
      for (int v = lane; v < nv; v += kG) dev::stream_pack<T, kV>(dst + v * kV, filled<T, kV>(fill[0]));
      return;
    }
    for (int v = lane; v < nv; v += kPieces * kG) {
      Pack<T, kV> x[kPieces];
#pragma unroll
      for (int u = 0; u < kPieces; ++u)  // past the row's end its last piece: no branches
        x[u] = dev::load_pack<T, kV>(src[0] + min(v + u * kG, nv - 1) * kV);
#pragma unroll
      for (int u = 0; u < kPieces; ++u)
        if (v + u * kG < nv)
          dev::stream_pack<T, kV>(dst + (v + u * kG) * kV, scaled<T, kV>(x[u], scale));
    }
  } else {
    if (lane >= nv) return;
    Pack<T, kV> x[kRows];
    if (rows > 0) {  // ids without a row read the first: no branches
#pragma unroll
      for (int u = 0; u < kRows; ++u) x[u] = dev::load_pack<T, kV>(src[u] + lane * kV);
    }
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      if (first + u >= n) break;
      dev::stream_pack<T, kV>(dst + u * out_stride + lane * kV,
                              held[u] ? scaled<T, kV>(x[u], scale) : filled<T, kV>(fill[u]));
    }
  }
}

template <class T, class Id, int kV>
void launch_lookup(const void* table, size_t rows, size_t dim, size_t table_stride,
                   const void* ids, size_t n, float scale, void* out, size_t out_stride,
                   cudaStream_t st) {
  const int nv = static_cast<int>(dim / kV);
  auto go = [&](auto g, auto pieces) {
    constexpr int kG = decltype(g)::value;
    constexpr int kPieces = decltype(pieces)::value;
    const size_t per_block = kLookupThreads / kG * (kPieces > 0 ? 1 : 4);
    lookup_kernel<T, Id, kV, kG, kPieces>
        <<<static_cast<unsigned>(ceil_div(n, per_block)), kLookupThreads, 0, st>>>(
            static_cast<const T*>(table), static_cast<int64_t>(rows),
            static_cast<int64_t>(table_stride), static_cast<const Id*>(ids),
            static_cast<int64_t>(n), nv, scale, static_cast<T*>(out),
            static_cast<int64_t>(out_stride));
  };
  using Short = std::integral_constant<int, 0>;
  if (nv <= 4)
    go(std::integral_constant<int, 4>{}, Short{});
  else if (nv <= 8)
    go(std::integral_constant<int, 8>{}, Short{});
  else if (nv <= 16)
    go(std::integral_constant<int, 16>{}, Short{});
  else if (nv <= 32)
    go(std::integral_constant<int, 32>{}, Short{});
  else if (nv <= 64)
    go(std::integral_constant<int, 32>{}, std::integral_constant<int, 2>{});
  else if (nv <= 128 || kV * sizeof(T) > 8)
    go(std::integral_constant<int, 32>{}, std::integral_constant<int, 4>{});
  else  // long rows of narrow pieces
    go(std::integral_constant<int, 32>{}, std::integral_constant<int, 8>{});
  check_launch("lookup_kernel");
}

// ---- gradient: zeros ---------------------------------------------------------------------------
// Most rows of a large table get no gradient, and their zeros are most of the bytes. They are
// written while the ids are sorted: sorting is a chain of short launches that leaves the memory
// idle, so each of its launches carries extra blocks that clear a share of the result. Rows that do
// get a gradient are written once more afterwards. The launches are chained: the clearing of one
// begins while the one before still runs, and only its sorting blocks wait for that one's end.
// 131,072 rows of 1024 bfloat16: the sort alone takes 20 us, clearing 268 MB 42 us (6.4 TB/s), both
// together 50 us.
struct Clear {
  unsigned char* p;
  int64_t rows, row_bytes, stride;  // bytes
  int align;                        // of every row
  uint32_t parts;                   // launches that share the work
};

template <class V>
__device__ __forceinline__ void clear_rows(const Clear& c, int64_t r0, int64_t r1, int64_t block,
                                           int64_t blocks) {
  const int64_t per_row = c.row_bytes / static_cast<int64_t>(sizeof(V));
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int64_t r = r0 + block * warps + warp; r < r1; r += blocks * warps) {
    V* row = reinterpret_cast<V*>(c.p + r * c.stride);
    for (int64_t i = lane; i < per_row; i += 32) row[i] = V{};
  }
}

// Share `part` of the clearing, by block `block` of `blocks`. A result without gaps is cleared by
// bulk copies of zeros out of shared memory, a few at a time per block: ordinary stores at the
// memory's full rate fill the SMs' load / store queues, and any number of bulk copies the memory's,
// and the sorting blocks' few loads then wait behind them (the sort of 50,001 ids took 116 us
// beside ordinary stores instead of 34).
__device__ __forceinline__ void clear_part(const Clear& c, uint32_t part, uint32_t block,
                                           uint32_t blocks) {
  if (c.stride == c.row_bytes) {
    constexpr int64_t kPiece = 8192;
    __shared__ __align__(128) uint4 zeros[kPiece / 16];
    for (uint32_t i = threadIdx.x; i < kPiece / 16; i += blockDim.x) zeros[i] = uint4{};
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    // Whole 16-byte units; what is left at the two ends (2-byte elements) by the first block.
    const int64_t bytes = c.rows * c.row_bytes;
    const int64_t lead = min(bytes, static_cast<int64_t>(-reinterpret_cast<intptr_t>(c.p) & 15));
    const int64_t units = (bytes - lead) / 16;
    unsigned char* body = c.p + lead;
    if (part == 0 && block == 0) {
      for (int64_t i = threadIdx.x * 2; i < lead; i += blockDim.x * 2)
        *reinterpret_cast<uint16_t*>(c.p + i) = 0;
      for (int64_t i = units * 16 + threadIdx.x * 2; i < bytes - lead; i += blockDim.x * 2)
        *reinterpret_cast<uint16_t*>(body + i) = 0;
    }
    if (threadIdx.x != 0) return;
    const int64_t u0 = units * part / c.parts, u1 = units * (part + 1) / c.parts;
    const int64_t per = (u1 - u0 + blocks - 1) / blocks;
    const int64_t begin = (u0 + per * block) * 16, end = min(u1, u0 + per * (block + 1)) * 16;
    // The next launch starts its share when half of this one is written: none of the launches'
    // ramps leave the memory idle, and no more than two shares are under way at a time.
    bool told = false;
    for (int64_t at = begin; at < end; at += kPiece) {
      if (!told && at - begin >= (end - begin) / 2) {
        dev::allow_next();
        told = true;
      }
      const uint32_t bytes = static_cast<uint32_t>(min(kPiece, end - at));
      asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(body + at),
                   "r"(static_cast<uint32_t>(__cvta_generic_to_shared(zeros))), "r"(bytes)
                   : "memory");
      asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group 3;" ::: "memory");
    }
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    return;
  }
  const int64_t r0 = c.rows * part / c.parts, r1 = c.rows * (part + 1) / c.parts;
  switch (c.align) {
    case 16: clear_rows<uint4>(c, r0, r1, block, blocks); break;
    case 8: clear_rows<uint2>(c, r0, r1, block, blocks); break;
    case 4: clear_rows<uint32_t>(c, r0, r1, block, blocks); break;
    default: clear_rows<uint16_t>(c, r0, r1, block, blocks); break;
  }
}

// ---- gradient: sorting ids -----------------------------------------------------------------------
// Stable least-significant-digit radix sort of (id, position) pairs; ids that take no gradient
// (negative or past the table) become `rows` and end up last. Each pass: per-tile digit counts,
// a prefix over tiles per digit, and a scatter that ranks a tile's entries in input order.
constexpr int kSortThreads = 256, kSortItems = 4;
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
    digit_count_kernel(const void* src, uint32_t n, uint32_t rows, int shift,
                       int bits, uint32_t tiles, uint32_t* counts, const Clear clear,
                       uint32_t part) {
  if (blockIdx.x >= tiles) {
    clear_part(clear, part, blockIdx.x - tiles, gridDim.x - tiles);
    return;
  }
  dev::allow_next();
  dev::wait_previous();
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
__global__ void __launch_bounds__(kSortThreads)
    digit_scan_kernel(uint32_t* counts, int bins, uint32_t tiles,
                      uint32_t* totals, uint32_t blocks, const Clear clear,
                      uint32_t part) {
  if (blockIdx.x >= blocks) {
    clear_part(clear, part, blockIdx.x - blocks, gridDim.x - blocks);
    return;
  }
  dev::allow_next();
  dev::wait_previous();
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
    digit_scatter_kernel(const void* src, const uint32_t* src_pos, uint32_t n, uint32_t rows,
                         int shift, int bits, uint32_t tiles, const uint32_t* counts,
                         const uint32_t* totals, uint32_t* keys, uint32_t* pos,
                         const Clear clear, uint32_t part) {
  if (blockIdx.x >= tiles) {
    clear_part(clear, part, blockIdx.x - tiles, gridDim.x - tiles);
    return;
  }
  dev::allow_next();
  dev::wait_previous();
  extern __shared__ uint32_t smem[];
  const int bins = 1 << bits;
  uint32_t* base = smem;                                             // bins: first slot of a digit
  uint16_t* wcount = reinterpret_cast<uint16_t*>(smem + bins);       // kSortWarps x bins
  __shared__ uint32_t wsum[kSortWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
  // Exclusive prefix of the digits' totals: each thread takes a run of up to kPer digits.
  constexpr int kPer = (1 << kMaxDigitBits) / kSortThreads;
  const int per = (bins + kSortThreads - 1) / kSortThreads;
  uint32_t sum[kPer], ahead[kPer];
  uint32_t mine = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int b = threadIdx.x * per + j;
    const bool in = j < per && b < bins;
    sum[j] = in ? totals[b] : 0;
    ahead[j] = in ? counts[static_cast<size_t>(b) * tiles + blockIdx.x] : 0;
    mine += sum[j];
  }
  for (int b = threadIdx.x; b < kSortWarps * bins / 4; b += kSortThreads)
    reinterpret_cast<uint2*>(wcount)[b] = uint2{};
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
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int b = threadIdx.x * per + j;
    if (j < per && b < bins) {
      base[b] = run + ahead[j];
      run += sum[j];
    }
  }
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
#pragma unroll
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

// The same sort of up to 8 * 1024 entries by one block in one launch: between passes the entries
// stay in shared memory. (A cluster of eight blocks doing this for 131,072 entries, exchanging them
// through each other's shared memory, took 88 us; the launches above take about 20.)
constexpr int kBlockSortThreads = 1024, kBlockDigitBits = 8;
constexpr int kBlockSortWarps = kBlockSortThreads / 32;
constexpr int kBlockSortMost = 8 * kBlockSortThreads;

template <class Id, int kItems>
__global__ void __launch_bounds__(kBlockSortThreads)
    block_sort_kernel(const void* __restrict__ ids, uint32_t n, uint32_t rows, int key_bits,
                      uint32_t* __restrict__ keys, uint32_t* __restrict__ pos, const Clear clear) {
  if (blockIdx.x > 0) {
    clear_part(clear, 0, blockIdx.x - 1, gridDim.x - 1);
    return;
  }
  dev::allow_next();
  constexpr int kBins = 1 << kBlockDigitBits;
  extern __shared__ uint32_t smem[];
  uint32_t* skey = smem;                                   // kItems * threads
  uint16_t* spos = reinterpret_cast<uint16_t*>(skey + kItems * kBlockSortThreads);
  uint16_t* wcount = spos + kItems * kBlockSortThreads;    // kBlockSortWarps x kBins
  __shared__ uint32_t total[kBins], wsum[kBins / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t first = warp * 32 * kItems + lane;
  uint16_t* wc = wcount + warp * kBins;
  uint32_t key[kItems], p[kItems], rank[kItems];
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    p[j] = first + j * 32;
    // Entries past the end carry the largest key and stay last (the sort is stable).
    key[j] = p[j] < n ? clip_id(load_id<Id>(ids, p[j]), rows) : 0xffffffffu;
  }
  for (int shift = 0; shift < key_bits; shift += kBlockDigitBits) {
    for (int b = lane; b < kBins / 2; b += 32) reinterpret_cast<uint32_t*>(wc)[b] = 0;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      const uint32_t digit = (key[j] >> shift) & (kBins - 1);
      const uint32_t same = __match_any_sync(dev::kFull, digit);
      const uint32_t before = __popc(same & ((1u << lane) - 1));
      rank[j] = wc[digit] + before;
      __syncwarp();
      if (before == 0) wc[digit] = static_cast<uint16_t>(wc[digit] + __popc(same));
      __syncwarp();
    }
    __syncthreads();
    // Prefix over warps per digit (one thread a digit), then over digits.
    if (threadIdx.x < kBins) {
      uint32_t acc = 0;
#pragma unroll
      for (int w = 0; w < kBlockSortWarps; ++w) {
        const uint32_t c = wcount[w * kBins + threadIdx.x];
        wcount[w * kBins + threadIdx.x] = static_cast<uint16_t>(acc);
        acc += c;
      }
      uint32_t s = acc;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const uint32_t o = __shfl_up_sync(dev::kFull, s, d);
        if (lane >= d) s += o;
      }
      if (lane == 31) wsum[warp] = s;
      total[threadIdx.x] = s - acc;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      const uint32_t digit = (key[j] >> shift) & (kBins - 1);
      uint32_t o = total[digit] + wc[digit] + rank[j];
      for (uint32_t w = 0; w < digit >> 5; ++w) o += wsum[w];
      skey[o] = key[j];
      spos[o] = static_cast<uint16_t>(p[j]);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      key[j] = skey[first + j * 32];
      p[j] = spos[first + j * 32];
    }
  }
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    if (first + j * 32 >= n) continue;
    keys[first + j * 32] = key[j];
    pos[first + j * 32] = p[j];
  }
}

// ---- gradient: segmented sums ---------------------------------------------------------------------
// Equal runs of the sorted entries go to the warps, so a token that fills a tenth of the batch is
// shared out. What a warp summed of a row that it did not end is its tail, what it summed of a row
// that it ended but that began before it is its head; rows that span warps are joined in order, in
// the block where they end in it, else by join_rows_kernel from the blocks' tails and heads.
// Bound by memory: upstream rows are read once, the rows they sum to written once. Four rows in
// flight per lane and five blocks an SM took 64 us for 131,072 x 1024 bfloat16 entries (325 MB,
// 5.1 TB/s, while the cleared zeros still leave the L2), eight rows and three blocks 68 us.
constexpr int kSumWarps = 8, kSumThreads = 32 * kSumWarps;
constexpr int kSumBatch = 4;  // rows in flight per lane
constexpr int kMaxRun = 32;   // entries per warp
constexpr uint32_t kNoRow = 0xffffffffu;

template <class T, int kV, int kC>
__global__ void __launch_bounds__(kSumThreads, 5)
    segment_sum_kernel(const T* __restrict__ up, int64_t up_stride,
                       const uint32_t* keys, const uint32_t* pos, uint32_t n, uint32_t rows,
                       uint32_t dim, uint32_t run, uint32_t col_tiles, float scale,
                       T* __restrict__ grad, int64_t grad_stride, float* head, float* tail, uint32_t* head_row,
                       uint32_t* tail_row) {
  dev::allow_next();
  dev::wait_previous();
  // The column tiles of the same entries are neighbours: they read the same rows at a time.
  const uint32_t block = blockIdx.x / col_tiles, col_tile = blockIdx.x - block * col_tiles;
  constexpr uint32_t kCols = 32 * kV * kC;
  __shared__ __align__(16) float s_head[kSumWarps][kCols];
  __shared__ __align__(16) float s_tail[kSumWarps][kCols];
  // Keys of the block's entries with the one before and the one after; kNoRow outside.
  __shared__ uint32_t s_keys[kSumWarps * kMaxRun + 2], s_pos[kSumWarps * kMaxRun];
  __shared__ uint32_t s_tail_row[kSumWarps];
  const uint32_t* s_key = s_keys + 1;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t b0 = block * run * kSumWarps;
  const uint32_t count = min(n - b0, run * kSumWarps);
  for (uint32_t i = threadIdx.x; i < count + 2; i += kSumThreads) {
    const uint32_t e = b0 + i - 1;  // wraps to 2^32 - 1 ahead of the first entry
    s_keys[i] = e < n ? keys[e] : kNoRow;
    if (i < count) s_pos[i] = pos[b0 + i];
  }
  __syncthreads();
  const uint32_t col0 = col_tile * kCols;
  // This lane's columns: kC pieces of kV. Pieces past the last column read the first.
  uint32_t c[kC];
  bool on[kC];
#pragma unroll
  for (int q = 0; q < kC; ++q) {
    c[q] = col0 + (q * 32 + lane) * kV;
    on[q] = c[q] < dim;
    if (!on[q]) c[q] = col0;
  }
  const uint32_t e0 = min(count, warp * run), e1 = min(count, e0 + run);
  const int before = static_cast<int>(e0) - 1;
  const uint32_t r0 = e0 < e1 ? s_key[e0] : kNoRow;
  const uint32_t before_key = s_key[-1];
  const bool began_before = e0 < e1 && r0 < rows && s_key[before] == r0;
  // The last row of this warp's entries, when it goes on in a later warp.
  const uint32_t last = e0 < e1 ? s_key[e1 - 1] : kNoRow;
  const bool has_tail = e0 < e1 && last < rows && s_key[e1] == last;
  if (lane == 0) s_tail_row[warp] = has_tail ? last : kNoRow;
  const bool ends_first = began_before && !(has_tail && last == r0);
  float acc[kC][kV];
  auto clear_acc = [&]() {
#pragma unroll
    for (int q = 0; q < kC; ++q) {
#pragma unroll
      for (int j = 0; j < kV; ++j) acc[q][j] = 0.0f;
    }
  };
  auto keep = [&](float* to) {
#pragma unroll
    for (int q = 0; q < kC; ++q) {
#pragma unroll
      for (int j = 0; j < kV; ++j) to[(q * 32 + lane) * kV + j] = acc[q][j];
    }
  };
  clear_acc();
  bool is_head = began_before;
  uint32_t r = r0;
  auto finish_row = [&]() {
    if (is_head) {
      keep(s_head[warp]);
    } else if (r < rows) {
#pragma unroll
      for (int q = 0; q < kC; ++q) {
        if (!on[q]) continue;
        Pack<T, kV> y;
#pragma unroll
        for (int j = 0; j < kV; ++j) y.v[j] = dev::from_f32<T>(acc[q][j] * scale);
        dev::stream_pack<T, kV>(grad + static_cast<int64_t>(r) * grad_stride + c[q], y);
      }
    }
    clear_acc();
    is_head = false;
  };
  for (uint32_t e = e0; e < e1; e += kSumBatch) {
    if (s_key[e] >= rows) break;  // ids that take no gradient, all at the end
    Pack<T, kV> x[kSumBatch][kC];
#pragma unroll
    for (int j = 0; j < kSumBatch; ++j) {  // past the run its last row again: no branches
      const T* src = up + s_pos[min(e + j, e1 - 1)] * up_stride;
#pragma unroll
      for (int q = 0; q < kC; ++q) x[j][q] = dev::load_once<T, kV>(src + c[q]);
    }
#pragma unroll
    for (int j = 0; j < kSumBatch; ++j) {
      if (e + j >= e1) break;
      const uint32_t k = s_key[e + j];
      if (k != r) {
        finish_row();
        r = k;
      }
#pragma unroll
      for (int q = 0; q < kC; ++q) {
#pragma unroll
        for (int v = 0; v < kV; ++v) acc[q][v] += dev::to_f32<T>(x[j][q].v[v]);
      }
    }
  }
  if (has_tail) {
    keep(s_tail[warp]);
  } else if (e0 < e1) {
    finish_row();
  }
  __syncthreads();
  // A row that began in an earlier warp and ended in this one: that run of tails, then the head.
  if (ends_first) {
    int v = warp;
    while (v > 0 && s_tail_row[v - 1] == r0) --v;
    const bool beyond = v == 0 && before_key == r0;  // it began in an earlier block
#pragma unroll 1
    for (uint32_t j = lane; j < kCols && col0 + j < dim; j += 32) {
      float s = 0.0f;
      for (int u = v; u < warp; ++u) s += s_tail[u][j];
      s += s_head[warp][j];
      if (beyond)
        head[static_cast<size_t>(block) * dim + col0 + j] = s;
      else
        grad[static_cast<int64_t>(r0) * grad_stride + col0 + j] = dev::from_f32<T>(s * scale);
    }
  }
  if (warp == 0) {
    // The row that came open into this block, if it ends in it.
    const bool ends = before_key < rows && s_key[0] == before_key && s_key[count] != before_key;
    if (lane == 0 && col_tile == 0) head_row[block] = ends ? before_key : kNoRow;
    // The row left open at the end of the block.
    const int lw = static_cast<int>((count - 1) / run);  // the last warp with entries
    const uint32_t open_row = s_tail_row[lw];
    if (lane == 0 && col_tile == 0) tail_row[block] = open_row;
    if (open_row != kNoRow) {
      int v = lw;
      while (v > 0 && s_tail_row[v - 1] == open_row) --v;
#pragma unroll 1
      for (uint32_t j = lane; j < kCols && col0 + j < dim; j += 32) {
        float s = 0.0f;
        for (int u = v; u <= lw; ++u) s += s_tail[u][j];
        tail[static_cast<size_t>(block) * dim + col0 + j] = s;
      }
    }
  }
}

// Block b's first row, where it began in an earlier block and ends in b: the tails of the blocks
// from the one it began in up to b - 1, in order, and b's head.
template <class T, int kV>
__global__ void __launch_bounds__(kSumThreads)
    join_rows_kernel(uint32_t dim, float scale, T* __restrict__ grad, int64_t grad_stride,
                     const float* head, const float* tail, const uint32_t* head_row,
                     const uint32_t* tail_row) {
  dev::wait_previous();
  const uint32_t r = head_row[blockIdx.x];
  if (r == kNoRow) return;
  uint32_t began = blockIdx.x;  // every warp looks back over 32 blocks at a time
  for (bool more = true; more;) {
    const uint32_t back = began - 1 - (threadIdx.x & 31);  // past block 0 it wraps
    const uint32_t open = __ballot_sync(dev::kFull, back < blockIdx.x && tail_row[back] == r);
    const int run = __ffs(~open) - 1;  // -1: all 32
    began -= run < 0 ? 32 : run;
    more = run < 0;
  }
  for (uint32_t c = (blockIdx.y * kSumThreads + threadIdx.x) * kV; c < dim;
       c += gridDim.y * kSumThreads * kV) {
    const Pack<float, kV> last =
        dev::load_pack<float, kV>(head + static_cast<size_t>(blockIdx.x) * dim + c);
    float s[kV];
#pragma unroll
    for (int j = 0; j < kV; ++j) s[j] = 0.0f;
#pragma unroll 16
    for (uint32_t u = began; u < blockIdx.x; ++u) {
      const Pack<float, kV> x =
          dev::load_pack<float, kV>(tail + static_cast<size_t>(u) * dim + c);
#pragma unroll
      for (int j = 0; j < kV; ++j) s[j] += x.v[j];
    }
    Pack<T, kV> y;
#pragma unroll
    for (int j = 0; j < kV; ++j) y.v[j] = dev::from_f32<T>((s[j] + last.v[j]) * scale);
    dev::store_pack<T, kV>(grad + static_cast<int64_t>(r) * grad_stride + c, y);
  }
}

struct GradPlan {
  bool one_block;              // sorted by one block
  int key_bits, passes, bits;  // width of a key, radix passes and digit width
  uint32_t tiles;              // sort tiles
  uint32_t run, blocks;        // entries per warp, blocks of the sums
  size_t off_keys[2], off_pos[2], off_counts, off_totals, off_head, off_tail, off_row, off_open, bytes;
};

GradPlan grad_plan(size_t n, size_t rows, size_t dim) {
  GradPlan p{};
  p.key_bits = 1;
  while ((size_t{1} << p.key_bits) <= rows) ++p.key_bits;  // keys 0 .. rows
  p.one_block = n <= kBlockSortMost;
  p.passes = p.one_block ? 1 : static_cast<int>(ceil_div(p.key_bits, kMaxDigitBits));
  p.bits = static_cast<int>(ceil_div(p.key_bits, p.passes));
  p.tiles = static_cast<uint32_t>(ceil_div(n, kSortTile));
  // Short runs while they are what fills the GPU, long ones once there are warps enough.
  p.run = n <= 148 * 64 * 8 ? 8 : kMaxRun;
  p.blocks = static_cast<uint32_t>(ceil_div(n, p.run * kSumWarps));
  size_t o = 0;
  auto take = [&](size_t bytes) {
    const size_t at = o;
    o += (bytes + 255) / 256 * 256;
    return at;
  };
  for (int i = 0; i < (p.one_block ? 1 : 2); ++i) {
    p.off_keys[i] = take(n * 4);
    p.off_pos[i] = take(n * 4);
  }
  if (!p.one_block) {
    p.off_counts = take((size_t{1} << p.bits) * p.tiles * 4);
    p.off_totals = take((size_t{1} << p.bits) * 4);
  }
  p.off_head = take(p.blocks * dim * 4);
  p.off_tail = take(p.blocks * dim * 4);
  p.off_row = take(p.blocks * 4);
  p.off_open = take(p.blocks * 4);
  p.bytes = o;
  return p;
}

// Extra blocks that clear a share of the result: at least 32 KB each, six to an SM at most.
uint32_t clear_blocks(const Clear& c) {
  const size_t bytes = static_cast<size_t>(c.rows) * c.row_bytes / c.parts;
  return static_cast<uint32_t>(
      std::max<size_t>(1, std::min<size_t>(ceil_div(bytes, 32768), 148 * 6)));
}

template <class Id, int kItems>
void launch_block_sort(const GradPlan& p, const void* ids, uint32_t n, uint32_t rows,
                       const Clear& clear, unsigned char* ws, cudaStream_t st) {
  constexpr size_t smem =
      kItems * kBlockSortThreads * 6 + kBlockSortWarps * (size_t{2} << kBlockDigitBits);
  QV_CUDA(cudaFuncSetAttribute(block_sort_kernel<Id, kItems>,
                               cudaFuncAttributeMaxDynamicSharedMemorySize,
                               static_cast<int>(smem)));
  block_sort_kernel<Id, kItems>
      <<<1 + clear_blocks(clear), kBlockSortThreads, smem, st>>>(
          ids, n, rows, p.key_bits, reinterpret_cast<uint32_t*>(ws + p.off_keys[0]),
          reinterpret_cast<uint32_t*>(ws + p.off_pos[0]), clear);
  check_launch("block_sort_kernel");
}

// Sorts the ids and clears the result; returns which key / position buffers hold the order.
template <class Id>
int sort_ids(const GradPlan& p, const void* ids, uint32_t n, uint32_t rows, Clear clear,
             unsigned char* ws, cudaStream_t st) {
  if (p.one_block) {
    clear.parts = 1;
    if (n <= kBlockSortThreads)
      launch_block_sort<Id, 1>(p, ids, n, rows, clear, ws, st);
    else if (n <= 4 * kBlockSortThreads)
      launch_block_sort<Id, 4>(p, ids, n, rows, clear, ws, st);
    else
      launch_block_sort<Id, 8>(p, ids, n, rows, clear, ws, st);
    return 0;
  }
  clear.parts = static_cast<uint32_t>(3 * p.passes);
  const uint32_t extra = clear_blocks(clear);
  uint32_t* counts = reinterpret_cast<uint32_t*>(ws + p.off_counts);
  uint32_t* totals = reinterpret_cast<uint32_t*>(ws + p.off_totals);
  const int bins = 1 << p.bits;
  const uint32_t scan_blocks = static_cast<uint32_t>(ceil_div(bins, kSortWarps));
  const size_t smem = bins * 4 + static_cast<size_t>(kSortWarps) * bins * 2;
  uint32_t part = 0;
  for (int k = 0; k < p.passes; ++k) {
    uint32_t* ok = reinterpret_cast<uint32_t*>(ws + p.off_keys[k & 1]);
    uint32_t* op = reinterpret_cast<uint32_t*>(ws + p.off_pos[k & 1]);
    const uint32_t* ik = reinterpret_cast<uint32_t*>(ws + p.off_keys[(k & 1) ^ 1]);
    const uint32_t* ip = reinterpret_cast<uint32_t*>(ws + p.off_pos[(k & 1) ^ 1]);
    const int shift = k * p.bits;
    if (k == 0)  // not chained: the caller's work before it may still use the result's memory
      digit_count_kernel<Id, true><<<p.tiles + extra, kSortThreads, bins * 4, st>>>(
          ids, n, rows, shift, p.bits, p.tiles, counts, clear, part++);
    else
      launch_chained(digit_count_kernel<Id, false>, p.tiles + extra, kSortThreads, bins * 4, st, ik,
                     n, rows, shift, p.bits, p.tiles, counts, clear, part++);
    check_launch("digit_count_kernel");
    launch_chained(digit_scan_kernel, scan_blocks + extra, kSortThreads, 0, st, counts, bins,
                   p.tiles, totals, scan_blocks, clear, part++);
    check_launch("digit_scan_kernel");
    auto* scatter = k == 0 ? digit_scatter_kernel<Id, true> : digit_scatter_kernel<Id, false>;
    // The widest digits' need whatever this call's is: the limit is the kernel's, and another
    // thread's call may set it between this line and the launch.
    QV_CUDA(cudaFuncSetAttribute(scatter, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (4 + 2 * kSortWarps) << kMaxDigitBits));
    launch_chained(scatter, p.tiles + extra, kSortThreads, smem, st, k == 0 ? ids : ik,
                   k == 0 ? nullptr : ip, n, rows, shift, p.bits, p.tiles, counts, totals, ok, op,
                   clear, part++);
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
  uint32_t* head_row = reinterpret_cast<uint32_t*>(ws + p.off_row);
  uint32_t* tail_row = reinterpret_cast<uint32_t*>(ws + p.off_open);
  constexpr int kC = kV * sizeof(T) < 8 ? 4 : 1;  // narrow pieces: four a lane
  const size_t col_tiles = ceil_div(dim, 32 * kV * kC);
  QV_REQUIRE(p.blocks * col_tiles < (size_t{1} << 31), "n * dim is too large");
  launch_chained(segment_sum_kernel<T, kV, kC>,
                 static_cast<unsigned>(p.blocks * col_tiles), kSumThreads, 0, st,
                 static_cast<const T*>(up), static_cast<int64_t>(up_stride), keys, pos, n, rows,
                 dim, p.run, static_cast<uint32_t>(col_tiles), scale, static_cast<T*>(grad), static_cast<int64_t>(grad_stride), head,
                 tail, head_row, tail_row);
  check_launch("segment_sum_kernel");
  if (p.blocks == 1) return;
  constexpr int kJoin = kV >= 4 ? 4 : 1;  // 16-byte pieces of the partial sums
  launch_chained(join_rows_kernel<T, kJoin>,
                 dim3(p.blocks, static_cast<unsigned>(ceil_div(dim, kSumThreads * kJoin))),
                 kSumThreads, 0, st, dim, scale, static_cast<T*>(grad), static_cast<int64_t>(grad_stride),
                 static_cast<const float*>(head), static_cast<const float*>(tail),
                 static_cast<const uint32_t*>(head_row), static_cast<const uint32_t*>(tail_row));
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
  QV_REQUIRE(n < (size_t{1} << 31), "more than 2^31 - 1 ids");
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
  const int align =
      common_align({reinterpret_cast<uintptr_t>(up), reinterpret_cast<uintptr_t>(grad),
                    n > 1 ? up_stride * e : 0, rows > 1 ? grad_stride * e : 0, dim * e});
  Clear clear{};
  clear.p = static_cast<unsigned char*>(grad);
  clear.rows = static_cast<int64_t>(rows);
  clear.row_bytes = static_cast<int64_t>(dim * e);
  clear.stride = static_cast<int64_t>(rows > 1 ? grad_stride * e : dim * e);
  clear.align = common_align({reinterpret_cast<uintptr_t>(grad),
                              static_cast<uint64_t>(clear.stride), dim * e});
  const int which = id_type == QV_ID_I32 ? sort_ids<int32_t>(p, ids, n32, rows32, clear, ws, st)
                                         : sort_ids<int64_t>(p, ids, n32, rows32, clear, ws, st);
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
