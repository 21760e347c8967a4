// Embedding rows and their gradient.
//
// Lookup: out[t] = round(scale * table[i_t]).  A copy with a product: bound by the bytes of the rows, each read where the
// index says and written in order.
//
// Gradient: out[v] = round(scale * sum over t with i_t = v of grad[t]), every row of the table written.  The tokens are
// sorted by index (a stable radix sort of (index, token) pairs), then summed in the sorted order, fp32, without atomics on
// floats: the same inputs give the same bits.  The sum is split evenly over the sorted tokens, not over the rows, so one
// row that all tokens name costs no more than many short ones: a worker takes `share` consecutive sorted tokens, writes the
// rows that begin and end inside its share, and leaves the pieces of the others to be joined, first in its block, then
// (join kernel) between blocks, always in the order of the tokens.  Rows that no token names are filled with zeros by further
// blocks of the same launch.
//
// Three ways to sort, by the number of tokens: up to 2048, every block that sums sorts all of them itself (one launch for
// the whole gradient where one block can sum them); up to 65536, a cluster of eight blocks sorts in its shared memory; above, tiles of
// 2048 tokens are counted, scanned and scattered digit by digit.
#include <cooperative_groups.h>

#include <algorithm>

#include "gnr_internal.cuh"
#include "gnr_types.cuh"

namespace {

constexpr int kThreads = 256;

// ---- lookup --------------------------------------------------------------------------------------------------------

// rows of a thread: 1.5M rows of 48 fp32 take 59, 49, 57, 63, 86 us with 1, 2, 3, 4, 8 of them, 20000 of 771 fp16 60, 43, 37, 39, 45
__host__ __device__ constexpr int lookup_depth(int piece_bytes) { return piece_bytes == 32 ? 2 : 3; }

// A piece is N neighbouring values; `per_row` of them make a row.  `lanes` threads of a block cover (part `blockIdx.x % n_cols` of) a row,
// `group` rows stand side by side in a block, and every thread has its piece of kDeep rows, `group` apart, in flight at once.  Bound by HBM:
// 1.5M rows of 48 fp32 49 us = 6.1 TB/s, 32768 of 2048 bf16 from a table of 131072 43 us = 5.6 TB/s.
template <typename T, typename I, int N>
__global__ void __launch_bounds__(kThreads)
embedding_lookup_kernel(const T* __restrict__ table, int64_t rows, int64_t table_stride, const I* __restrict__ index, int64_t n, uint32_t per_row,
                        uint32_t lanes, uint32_t n_cols, uint32_t group, float scale, T* __restrict__ out, int64_t out_stride) {
  constexpr int kDeep = lookup_depth(sizeof(T) * N);
  const uint32_t mine = threadIdx.x / lanes, piece = blockIdx.x % n_cols * lanes + threadIdx.x % lanes;
  if (mine >= group || piece >= per_row) return;
  const int64_t c = (int64_t)piece * N, first = (int64_t)(blockIdx.x / n_cols) * (group * kDeep) + mine;
  int64_t row[kDeep];
  Raw<T, N> x[kDeep];
#pragma unroll
  for (int k = 0; k < kDeep; ++k) row[k] = first + k * group < n ? (int64_t)index[first + k * group] : -1;
#pragma unroll
  for (int k = 0; k < kDeep; ++k) {
    const T* from = table + (row[k] >= 0 && row[k] < rows ? row[k] : 0) * table_stride + c;  // a row of the table in any case
    if constexpr (sizeof(T) * N == 32) load32(x[k], from);
    else x[k].load(from);
  }
#pragma unroll
  for (int k = 0; k < kDeep; ++k) {
    if (first + k * group >= n) break;
    T* to = out + (first + k * group) * out_stride + c;
    Pack<T, N> y;
    if (row[k] >= 0 && row[k] < rows) {
#pragma unroll
      for (int j = 0; j < N; ++j) y.v[j] = from_float<T>(x[k].get(j) * scale);
    } else {  // a masked place gives zeros, an index past the table NaN
      const T fill = from_float<T>(row[k] < 0 ? 0.0f : __int_as_float(0x7fc00000));
#pragma unroll
      for (int j = 0; j < N; ++j) y.v[j] = fill;
    }
    if constexpr (sizeof(T) * N == 32) store32(to, y);
    else *reinterpret_cast<Pack<T, N>*>(to) = y;
  }
}

// ---- sort ----------------------------------------------------------------------------------------------------------

constexpr int kMaxBits = 9;  // bits of a digit
constexpr int kMaxRadix = 1 << kMaxBits;
constexpr uint32_t kNoKey = 0xffffffffu;

// Tokens to sort: their indices as the caller gave them, 32 or 64 bits wide.
struct Tokens {
  const void* index;
  int wide;
  int64_t n, rows, padding;
  // a token's key: its row, or `rows` for what the gradient leaves out (masked, past the table, the padding row)
  __device__ __forceinline__ uint32_t key_of(int64_t i) const { return i < 0 || i >= rows || i == padding ? (uint32_t)rows : (uint32_t)i; }
  __device__ __forceinline__ uint32_t key(int64_t t) const {
    return key_of(wide ? static_cast<const int64_t*>(index)[t] : static_cast<const int32_t*>(index)[t]);
  }
  // keys of several tokens (0 for those past the last), all loads in flight at once
  template <int Items, typename At> __device__ __forceinline__ void keys(At at, uint32_t (&key)[Items]) const {
    if (wide) {
      int64_t i[Items];
#pragma unroll
      for (int j = 0; j < Items; ++j) i[j] = at(j) < n ? static_cast<const int64_t*>(index)[at(j)] : 0;
#pragma unroll
      for (int j = 0; j < Items; ++j) key[j] = key_of(i[j]);
    } else {
      int32_t i[Items];
#pragma unroll
      for (int j = 0; j < Items; ++j) i[j] = at(j) < n ? static_cast<const int32_t*>(index)[at(j)] : 0;
#pragma unroll
      for (int j = 0; j < Items; ++j) key[j] = key_of(i[j]);
    }
  }
};

template <int Warps> struct Counts {
  uint16_t of_warp[Warps][kMaxRadix];  // tokens of a digit in a warp's share, then in the shares before it
  uint32_t base[kMaxRadix];
  uint32_t scan[32];
};

// place of a thread's j-th token in its block's tile: every warp has a run of neighbours
template <int Items> __device__ __forceinline__ int tile_place(int j) {
  return (threadIdx.x >> 5) * (32 * Items) + j * 32 + (threadIdx.x & 31);
}

// lanes whose digit is this lane's.  The more digits a warp holds, the longer it takes; for runs of one code, what samples of rays bring, the
// gradient of 1.5M tokens of 4 values takes 60 us, with one vote per bit instead 79.
__device__ __forceinline__ uint32_t digit_peers(uint32_t digit, bool there) { return __match_any_sync(0xffffffffu, there ? digit : kNoKey); }

// Ranks of a tile's tokens among the tokens of the same digit, in the tile's order (the first `n` places hold one).  Afterwards
// of_warp[w][d] holds the tokens of digit d in the warps before w, and sums[k] those of digit threadIdx.x + k * threads in the tile.
template <int Warps, int Items>
__device__ __forceinline__ void rank_tile(Counts<Warps>& s, const uint32_t (&key)[Items], int shift, int bits, int n, uint32_t (&rank)[Items],
                                          uint32_t (&sums)[(kMaxRadix + Warps * 32 - 1) / (Warps * 32)]) {
  constexpr int kAll = Warps * 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t radix = 1u << bits;
  for (uint32_t i = lane; i < radix; i += 32) s.of_warp[warp][i] = 0;
  __syncwarp();
#pragma unroll
  for (int j = 0; j < Items; ++j) {
    const uint32_t digit = key[j] >> shift & (radix - 1);
    const bool there = tile_place<Items>(j) < n;
    const uint32_t peers = digit_peers(digit, there), before = peers & ((1u << lane) - 1u);
    const uint32_t upto = there ? s.of_warp[warp][digit] : 0u;
    rank[j] = upto + __popc(before);
    __syncwarp();
    if (there && before == 0) s.of_warp[warp][digit] = (uint16_t)(upto + __popc(peers));
    __syncwarp();
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < (kMaxRadix + kAll - 1) / kAll; ++k) {
    const uint32_t d = threadIdx.x + k * kAll;
    sums[k] = 0;
    if (d < radix)
#pragma unroll 8
      for (int w = 0; w < Warps; ++w) {
        const uint32_t c = s.of_warp[w][d];
        s.of_warp[w][d] = (uint16_t)sums[k];
        sums[k] += c;
      }
  }
}

// exclusive sum over the block's threads
template <int Warps> __device__ __forceinline__ uint32_t block_exclusive(uint32_t* scan, uint32_t x) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t sum = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += y;
  }
  if (lane == 31) scan[warp] = sum;
  __syncthreads();
  uint32_t before = 0;
#pragma unroll
  for (int w = 0; w < Warps; ++w) before += w < warp ? scan[w] : 0u;
  __syncthreads();
  return before + sum - x;
}

// base[d]: tokens of smaller digits
template <int Warps>
__device__ __forceinline__ void digit_bases(Counts<Warps>& s, const uint32_t (&sums)[(kMaxRadix + Warps * 32 - 1) / (Warps * 32)], int bits) {
  constexpr int kAll = Warps * 32;
  uint32_t carry = 0;
#pragma unroll
  for (int k = 0; k < (kMaxRadix + kAll - 1) / kAll; ++k) {
    const uint32_t d = threadIdx.x + k * kAll, at = block_exclusive<Warps>(s.scan, sums[k]);
    if (d < (1u << bits)) s.base[d] = carry + at;
    if (k + 1 < (kMaxRadix + kAll - 1) / kAll) {  // the next digits lie behind all of these
      if (threadIdx.x == kAll - 1) s.scan[31] = at + sums[k];
      __syncthreads();
      carry += s.scan[31];
      __syncthreads();
    }
  }
  __syncthreads();
}

// Sorts up to Warps * 32 * Items tokens in the block; the result in shared memory, `keys` and `places` (token numbers).
template <int Warps, int Items, typename Place>
__device__ __forceinline__ void sort_block(Counts<Warps>& s, const Tokens& tokens, int passes, int bits, uint32_t* keys, Place* places) {
  const int n = (int)tokens.n, warp = threadIdx.x >> 5;
  uint32_t key[Items], place[Items], rank[Items], sums[(kMaxRadix + Warps * 32 - 1) / (Warps * 32)];
  tokens.keys([](int j) { return (int64_t)tile_place<Items>(j); }, key);
#pragma unroll
  for (int j = 0; j < Items; ++j) place[j] = tile_place<Items>(j);
  for (int pass = 0; pass < passes; ++pass) {
    rank_tile<Warps, Items>(s, key, pass * bits, bits, n, rank, sums);
    digit_bases<Warps>(s, sums, bits);
#pragma unroll
    for (int j = 0; j < Items; ++j)
      if (tile_place<Items>(j) < n) {
        const uint32_t digit = key[j] >> (pass * bits) & ((1u << bits) - 1u);
        const uint32_t at = s.base[digit] + s.of_warp[warp][digit] + rank[j];
        keys[at] = key[j];
        places[at] = (Place)place[j];
      }
    __syncthreads();
    if (pass + 1 < passes) {
#pragma unroll
      for (int j = 0; j < Items; ++j) {
        const int i = tile_place<Items>(j);
        if (i < n) {
          key[j] = keys[i];
          place[j] = places[i];
        }
      }
      __syncthreads();
    }
  }
}

// A cluster of eight blocks sorts up to 65536 tokens in their shared memory: every block ranks its eighth, reads the others' digit
// counts, and puts each token where it belongs, in whichever block that is.
constexpr int kCluster = 8;
constexpr int kClusterWarps = 32;
constexpr int kClusterItems = 8;  // at most
constexpr int kClusterSort = kCluster * kClusterWarps * 32 * kClusterItems;

template <int Items> struct ClusterShared {
  Counts<kClusterWarps> counts;
  uint32_t totals[kMaxRadix];
  uint32_t keys[2][kClusterWarps * 32 * Items], places[2][kClusterWarps * 32 * Items];
};

template <int Items>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kClusterWarps * 32, 1)
embedding_sort_cluster_kernel(Tokens tokens, int passes, int bits, uint32_t* __restrict__ out_keys, uint32_t* __restrict__ out_places) {
  extern __shared__ __align__(16) unsigned char smem[];
  ClusterShared<Items>& s = *reinterpret_cast<ClusterShared<Items>*>(smem);
  constexpr int kMine = kClusterWarps * 32 * Items;
  const cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  const int me = (int)cluster.block_rank(), warp = threadIdx.x >> 5;
  const int64_t tile0 = (int64_t)me * kMine;
  const int n = (int)max((int64_t)0, min((int64_t)kMine, tokens.n - tile0));
  uint32_t key[Items], place[Items], rank[Items], sums[1];
  tokens.keys([&](int j) { return tile0 + tile_place<Items>(j); }, key);
#pragma unroll
  for (int j = 0; j < Items; ++j) place[j] = (uint32_t)(tile0 + tile_place<Items>(j));
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * bits;
    rank_tile<kClusterWarps, Items>(s.counts, key, shift, bits, n, rank, sums);
    if (threadIdx.x < (1u << bits)) s.totals[threadIdx.x] = sums[0];
    cluster.sync();
    uint32_t before = 0, all = 0;
    if (threadIdx.x < (1u << bits)) {
#pragma unroll
      for (int c = 0; c < kCluster; ++c) {
        const uint32_t there = cluster.map_shared_rank(s.totals, c)[threadIdx.x];
        if (c < me) before += there;
        all += there;
      }
    }
    const uint32_t base = block_exclusive<kClusterWarps>(s.counts.scan, all);
    if (threadIdx.x < (1u << bits)) s.counts.base[threadIdx.x] = base + before;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < Items; ++j)
      if (tile_place<Items>(j) < n) {
        const uint32_t digit = key[j] >> shift & ((1u << bits) - 1u);
        const uint32_t at = s.counts.base[digit] + s.counts.of_warp[warp][digit] + rank[j];
        cluster.map_shared_rank(s.keys[pass & 1], at / kMine)[at % kMine] = key[j];
        cluster.map_shared_rank(s.places[pass & 1], at / kMine)[at % kMine] = place[j];
      }
    cluster.sync();
    if (pass + 1 < passes) {
#pragma unroll
      for (int j = 0; j < Items; ++j) {
        const int i = tile_place<Items>(j);
        key[j] = i < n ? s.keys[pass & 1][i] : 0u;
        place[j] = i < n ? s.places[pass & 1][i] : 0u;
      }
    }
  }
  for (int i = threadIdx.x; i < n; i += kClusterWarps * 32) {
    out_keys[tile0 + i] = s.keys[(passes - 1) & 1][i];
    out_places[tile0 + i] = s.places[(passes - 1) & 1][i];
  }
}

constexpr int kTileWarps = 16;
constexpr int kItems = 4;
constexpr int kTile = kTileWarps * 32 * kItems;  // tokens of a tile

// keys of a tile; `sorted` null: from the indices
__device__ __forceinline__ void tile_keys(const Tokens& tokens, const uint32_t* sorted, int64_t tile0, uint32_t (&key)[kItems]) {
  if (sorted) {
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      const int64_t i = tile0 + tile_place<kItems>(j);
      key[j] = i < tokens.n ? sorted[i] : 0u;
    }
  } else {
    tokens.keys([&](int j) { return tile0 + tile_place<kItems>(j); }, key);
  }
}

// tokens of every digit in every tile: counts[digit][tile].  `keys` null: the first pass, which reads the indices.
__global__ void __launch_bounds__(kTileWarps * 32)
embedding_count_kernel(Tokens tokens, const uint32_t* __restrict__ keys, int shift, int bits, uint32_t* __restrict__ counts, int n_tiles) {
  __shared__ uint32_t s_count[kMaxRadix];
  const uint32_t radix = 1u << bits;
  for (uint32_t d = threadIdx.x; d < radix; d += kTileWarps * 32) s_count[d] = 0;
  griddep_wait();
  const int64_t tile0 = (int64_t)blockIdx.x * kTile;
  uint32_t key[kItems];
  tile_keys(tokens, keys, tile0, key);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    // one addition for every run of equal digits in the warp
    const uint32_t digit = tile0 + tile_place<kItems>(j) < tokens.n ? key[j] >> shift & (radix - 1) : kNoKey;
    const int lane = threadIdx.x & 31;
    const bool head = __shfl_up_sync(0xffffffffu, digit, 1) != digit || lane == 0;
    const uint32_t behind = __ballot_sync(0xffffffffu, head) >> lane >> 1;  // heads of later runs
    if (head && digit != kNoKey) atomicAdd(&s_count[digit], behind ? (uint32_t)__ffs(behind) : 32u - lane);
  }
  __syncthreads();
  for (uint32_t d = threadIdx.x; d < radix; d += kTileWarps * 32) counts[(int64_t)d * n_tiles + blockIdx.x] = s_count[d];
}

// One block per digit: its counts become the tokens of that digit in the tiles before, and totals[digit] their sum.
__global__ void __launch_bounds__(kThreads) embedding_scan_kernel(uint32_t* __restrict__ counts, int n_tiles, uint32_t* __restrict__ totals) {
  __shared__ uint32_t s_scan[kThreads / 32], s_sum;
  griddep_wait();
  uint32_t* row = counts + (int64_t)blockIdx.x * n_tiles;
  uint32_t carry = 0;
  for (int first = 0; first < n_tiles; first += kThreads) {
    const int i = first + threadIdx.x;
    const uint32_t x = i < n_tiles ? row[i] : 0u;
    const uint32_t before = block_exclusive<kThreads / 32>(s_scan, x);
    if (i < n_tiles) row[i] = carry + before;
    if (threadIdx.x == kThreads - 1) s_sum = before + x;
    __syncthreads();
    carry += s_sum;
    __syncthreads();
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

__global__ void __launch_bounds__(kTileWarps * 32)
embedding_scatter_kernel(Tokens tokens, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ places, int shift, int bits,
                         const uint32_t* __restrict__ counts, const uint32_t* __restrict__ totals, int n_tiles, uint32_t* __restrict__ out_keys,
                         uint32_t* __restrict__ out_places) {
  __shared__ Counts<kTileWarps> s;
  griddep_wait();
  const uint32_t radix = 1u << bits;
  const int64_t tile0 = (int64_t)blockIdx.x * kTile;
  const int n = (int)min((int64_t)kTile, tokens.n - tile0);
  const uint32_t total = threadIdx.x < radix ? totals[threadIdx.x] : 0u;
  const uint32_t here = threadIdx.x < radix ? counts[(int64_t)threadIdx.x * n_tiles + blockIdx.x] : 0u;
  uint32_t key[kItems], place[kItems], rank[kItems], sums[1];
  tile_keys(tokens, keys, tile0, key);
#pragma unroll
  for (int j = 0; j < kItems; ++j) place[j] = (uint32_t)(tile0 + tile_place<kItems>(j));
  if (keys) {
#pragma unroll
    for (int j = 0; j < kItems; ++j) place[j] = place[j] < tokens.n ? places[place[j]] : 0u;
  }
  rank_tile<kTileWarps, kItems>(s, key, shift, bits, n, rank, sums);
  const uint32_t base = block_exclusive<kTileWarps>(s.scan, total);
  if (threadIdx.x < radix) s.base[threadIdx.x] = base + here;
  __syncthreads();
  const int warp = threadIdx.x >> 5;
#pragma unroll
  for (int j = 0; j < kItems; ++j)
    if (tile_place<kItems>(j) < n) {
      const uint32_t digit = key[j] >> shift & (radix - 1);
      const uint32_t at = s.base[digit] + s.of_warp[warp][digit] + rank[j];
      out_keys[at] = key[j];
      out_places[at] = place[j];
    }
}

// ---- sums ----------------------------------------------------------------------------------------------------------

constexpr int kSpan = 2048;               // sorted tokens of a block, at most
constexpr int kLocal = kThreads * 8;      // tokens that every block sorts itself
constexpr int kFillRows = 1024;           // rows of a block that fills, at most

struct SumArgs {
  Tokens tokens;
  int passes, bits;
  const uint32_t* keys;    // sorted (unless the blocks sort themselves); entries of key `rows` are left out
  const uint32_t* places;
  const void* grad;
  int64_t grad_stride;
  void* out;
  int64_t out_stride;
  int dim, lanes, n_cols;  // lanes: pieces of a row that a block's worker takes, n_cols such parts make a row
  int hop;                 // pieces of a row
  int workers;             // workers of a block
  int share;               // sorted tokens of a worker
  int64_t n_blocks;        // blocks along the tokens
  // Pieces [n_blocks][2][piece_stride] of the rows that blocks share: the sum of a block's tokens of the row that an earlier block began
  // (its key in keys_of[2 * block], else `rows`), and of the row that goes on in a later block and began in this one.
  float* pieces;
  uint32_t* keys_of;
  int64_t piece_stride;
  float scale;
  int fill_rows;           // rows of a block that fills rows without a token with zeros, 0: there are none
};

// A piece of a row, as it is loaded and written: N neighbours from c on (Whole), or, where their alignment forbids that, the values at
// c, c + hop, c + 2 hop ... that lie in the row, so that neighbouring threads have neighbouring values.
template <typename T, int N, bool Whole> struct Piece {
  std::conditional_t<Whole, Raw<T, N>, T[N]> x;
  __device__ __forceinline__ void load(const SumArgs& a, const T* row, int64_t c) {
    if constexpr (Whole) {
      x.load(row + c);
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) x[k] = c + k * a.hop < a.dim ? row[c + k * a.hop] : from_float<T>(0.0f);
    }
  }
  __device__ __forceinline__ float get(int k) const {
    if constexpr (Whole) return x.get(k);
    else return to_float(x[k]);
  }
};

// row = scale * sum, added to what was there (`old`) with Add
template <typename T, int N, bool Whole, bool Add>
__device__ __forceinline__ void write_row(const SumArgs& a, uint32_t row, int64_t c, const float (&sum)[N], const Piece<T, N, Whole>& old) {
  T* at = static_cast<T*>(a.out) + (int64_t)row * a.out_stride + c;
  T y[N];
#pragma unroll
  for (int k = 0; k < N; ++k) y[k] = from_float<T>(Add ? fmaf(sum[k], a.scale, old.get(k)) : sum[k] * a.scale);
  if constexpr (Whole) {
    Pack<T, N> z;
#pragma unroll
    for (int k = 0; k < N; ++k) z.v[k] = y[k];
    *reinterpret_cast<Pack<T, N>*>(at) = z;
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (c + k * a.hop < a.dim) at[k * a.hop] = y[k];
  }
}
template <typename T> __device__ __forceinline__ T* row_at(const SumArgs& a, uint32_t row) { return static_cast<T*>(a.out) + (int64_t)row * a.out_stride; }
template <typename T, int N, bool Whole, bool Add>
__device__ __forceinline__ void write_row(const SumArgs& a, uint32_t row, int64_t c, const float (&sum)[N]) {
  Piece<T, N, Whole> old;
  if (Add) old.load(a, row_at<T>(a, row), c);
  write_row<T, N, Whole, Add>(a, row, c, sum, old);
}

// where the pieces of rows that blocks share are kept: N values of a thread side by side
__device__ __forceinline__ float* piece_at(const SumArgs& a, int64_t block, int which, int64_t at) {
  return a.pieces + (block * 2 + which) * a.piece_stride + at;
}

// Which of the answers 0 .. n a search by 32 probes at once finds; `below(lo, hi, step)` counts those of the places lo + step - 1,
// lo + 2 step - 1, ... lo + 32 step - 1 that lie before `hi` and before the answer.  hi - lo + 1 answers are left, the probes part them
// into 33 runs of `step`: 33 step has to reach all of them, or the last would be cut off.
template <typename Below> __device__ __forceinline__ int64_t probed_bound(int64_t n, Below below) {
  int64_t lo = 0, hi = n;
  while (lo < hi) {
    const int64_t step = (hi - lo) / 33 + 1;
    lo += below(lo, hi, step) * step;
    hi = lo + step - 1 < hi ? lo + step - 1 : hi;
  }
  return lo;
}

// first position of the sorted keys that is not below `key`, found by a warp
__device__ __forceinline__ int64_t warp_lower_bound(const uint32_t* keys, int64_t n, uint32_t key) {
  return probed_bound(n, [&](int64_t lo, int64_t hi, int64_t step) {
    const int64_t at = lo + ((threadIdx.x & 31) + 1) * step - 1;
    return __popc(__ballot_sync(0xffffffffu, at < hi && keys[at] < key));
  });
}

// zeros in those rows from `first` on that no token names
template <typename TO, bool Local> __device__ __forceinline__ void fill_rows(const SumArgs& a, int64_t first, uint32_t* named, int64_t* range) {
  const int64_t last = min(first + a.fill_rows, a.tokens.rows);
  for (int i = threadIdx.x; i < kFillRows / 32; i += kThreads) named[i] = 0;
  if (!Local && threadIdx.x < 64) {
    const int64_t at = warp_lower_bound(a.keys, a.tokens.n, (uint32_t)(threadIdx.x < 32 ? first : last));
    range[threadIdx.x >> 5] = at;
  }
  __syncthreads();
  const int64_t lo = Local ? 0 : range[0], hi = Local ? a.tokens.n : range[1];
  if (Local || hi - lo <= 4096) {  // few tokens: all of them, the first of a row marking it
    for (int64_t i = lo + threadIdx.x; i < hi; i += kThreads) {
      const uint32_t key = Local ? a.tokens.key(i) : a.keys[i];
      if (key >= first && key < last && (Local || i == lo || a.keys[i - 1] != key)) atomicOr(&named[(key - first) >> 5], 1u << ((key - first) & 31));
    }
  } else {  // many: a search for every row
    for (int r = threadIdx.x; r < last - first; r += kThreads) {
      const uint32_t key = (uint32_t)(first + r);
      int64_t from = lo, to = hi;
      while (from < to) {
        const int64_t mid = (from + to) >> 1;
        if (a.keys[mid] < key) from = mid + 1;
        else to = mid;
      }
      if (from < hi && a.keys[from] == key) atomicOr(&named[r >> 5], 1u << (r & 31));
    }
  }
  __syncthreads();
  TO* out = static_cast<TO*>(a.out) + first * a.out_stride;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  constexpr int kWide = 16 / sizeof(TO);
  if (a.out_stride == a.dim && a.dim % kWide == 0 && (uintptr_t)a.out % 16 == 0) {
    const uint32_t per_row = a.dim / kWide, all = (uint32_t)(last - first) * per_row;
    for (uint32_t i = threadIdx.x; i < all; i += kThreads) {
      const uint32_t r = i / per_row;
      if (!(named[r >> 5] >> (r & 31) & 1u)) reinterpret_cast<uint4*>(out)[i] = zero;
    }
  } else {  // a warp to a row: single values up to a 16-byte boundary, 16 bytes at a time, single values
    for (int r = threadIdx.x >> 5; r < last - first; r += kThreads / 32) {
      if (named[r >> 5] >> (r & 31) & 1u) continue;
      TO* row = out + (int64_t)r * a.out_stride;
      const int lane = threadIdx.x & 31;
      const int head = min(a.dim, (int)((16 - (uintptr_t)row % 16) % 16 / sizeof(TO))), body = (a.dim - head) / kWide;
      if (lane < head) row[lane] = from_float<TO>(0.0f);
      for (int i = lane; i < body; i += 32) reinterpret_cast<uint4*>(row + head)[i] = zero;
      const int tail = head + body * kWide + lane;
      if (tail < a.dim) row[tail] = from_float<TO>(0.0f);
    }
  }
}

template <int N> struct SumShared {
  union {
    Counts<kThreads / 32> sort;
    struct {
      float head[kThreads][N], tail[kThreads][N];
    };
  };
  int through[kThreads];      // the whole share is one row that began before it and goes on behind it
  uint32_t key[kSpan + 2];    // of the tokens before, of and behind the block
  uint32_t token[kSpan];
  int valid;                  // tokens of the block that are summed
  uint32_t named[kFillRows / 32];
  int64_t range[2];
};

// Bound by the latency of rows fetched from anywhere, eight of them in flight a thread: 1.5M rows of 48 fp32 55 us, 5.2 TB/s (four in flight 63, 16 65 us); with
// Add two, beside the rows that they are added to (16384 tokens of 2048 bf16 into fp32 rows 53 us, 5.7 TB/s).
// Local: every block sorts all tokens itself.  (The sort's registers would cost the other form its fourth block on an SM: 1.5M samples 104
// against 93 us.  Of single fp32 values, sums of rows 3 wide say, 20 bytes a thread spill: 1.5M samples into 65,536 rays 77 us with the sort.)
template <typename TI, typename TO, int N, bool Whole, bool Add, bool Local>
__global__ void __launch_bounds__(kThreads) embedding_sum_kernel(SumArgs a) {
  __shared__ SumShared<N> s;
  constexpr int kBatch = Add ? (Whole ? 2 : 4) : 8;  // rows in flight
  griddep_wait();
  const int64_t sum_blocks = a.n_blocks * a.n_cols;
  if (blockIdx.x >= sum_blocks) {
    fill_rows<TO, Local>(a, ((int64_t)blockIdx.x - sum_blocks) * a.fill_rows, s.named, s.range);
    return;
  }
  const int64_t block = blockIdx.x / a.n_cols, block0 = block * a.workers * a.share;
  const int count = (int)min((int64_t)a.workers * a.share, a.tokens.n - block0);
  const uint32_t none = (uint32_t)a.tokens.rows;
  if (threadIdx.x == 0) s.valid = 0;
  int off = 0;  // of the block's first token in s.token, and in s.key of the token before it
  if constexpr (Local) {
    off = (int)block0;
    if (a.tokens.n <= kLocal / 2) sort_block<kThreads / 32, 4>(s.sort, a.tokens, a.passes, a.bits, s.key + 1, s.token);
    else sort_block<kThreads / 32, 8>(s.sort, a.tokens, a.passes, a.bits, s.key + 1, s.token);
    if (threadIdx.x == 0) s.key[0] = s.key[a.tokens.n + 1] = kNoKey;
  } else {
    for (int i = threadIdx.x; i < count; i += kThreads) {
      s.key[i + 1] = a.keys[block0 + i];
      s.token[i] = a.places[block0 + i];
    }
    if (threadIdx.x == 0) s.key[0] = block0 > 0 ? a.keys[block0 - 1] : kNoKey;
    if (threadIdx.x == 1) s.key[count + 1] = block0 + count < a.tokens.n ? a.keys[block0 + count] : kNoKey;
  }
  __syncthreads();
  const uint32_t* keys = s.key + off + 1;  // keys[-1]: before the block
  const uint32_t* tokens = s.token + off;
  for (int i = threadIdx.x; i < count; i += kThreads)  // tokens that are left out lie behind all others
    if (keys[i] != none && (i + 1 == count || keys[i + 1] == none)) s.valid = i + 1;
  __syncthreads();
  const int worker = threadIdx.x / a.lanes;
  const int piece = (int)(blockIdx.x % a.n_cols) * a.lanes + (int)threadIdx.x % a.lanes;
  const bool on = worker < a.workers && piece < a.hop;
  const int64_t c = Whole ? (int64_t)piece * N : piece;
  const int begin = worker * a.share, end = min(begin + a.share, s.valid);
  const TI* grad = static_cast<const TI*>(a.grad);
  bool through = false, tail = false;
  if (on && begin < end) {
    bool first = keys[begin - 1] == keys[begin];  // the row that began before the share
    float acc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = 0.0f;
    for (int i = begin; i < end; i += kBatch) {
      Piece<TI, N, Whole> x[kBatch];
      Piece<TO, N, Whole> old[Add ? kBatch : 1];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) x[b].load(a, grad + (int64_t)tokens[min(i + b, end - 1)] * a.grad_stride, c);
      if constexpr (Add) {
#pragma unroll
        for (int b = 0; b < kBatch; ++b)
          if (i + b < end && keys[i + b + 1] != keys[i + b]) old[b].load(a, row_at<TO>(a, keys[i + b]), c);
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        if (i + b >= end) break;
        const uint32_t key = keys[i + b];
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] += x[b].get(k);
        if (keys[i + b + 1] != key) {  // the row ends
          if (first) {
#pragma unroll
            for (int k = 0; k < N; ++k) s.head[threadIdx.x][k] = acc[k];
          } else {
            write_row<TO, N, Whole, Add>(a, key, c, acc, old[Add ? b : 0]);
          }
          first = false;
#pragma unroll
          for (int k = 0; k < N; ++k) acc[k] = 0.0f;
        }
      }
    }
    if (keys[end] == keys[end - 1]) {  // the last row goes on
      through = first;
      tail = !first;
#pragma unroll
      for (int k = 0; k < N; ++k) (first ? s.head : s.tail)[threadIdx.x][k] = acc[k];
    }
  }
  s.through[threadIdx.x] = through;
  __syncthreads();
  const bool from_before = keys[0] != none && keys[-1] == keys[0];
  if (threadIdx.x == 0 && blockIdx.x % a.n_cols == 0 && a.n_blocks > 1) {
    const uint32_t last = keys[count - 1];
    a.keys_of[2 * block] = from_before ? keys[0] : none;
    a.keys_of[2 * block + 1] = last != none && keys[count] == last && !(from_before && keys[0] == last) ? last : none;
  }
  if (!on) return;
  // A row that goes on behind a worker's share is joined by the worker it begins with; the one that came from the block
  // before by the first.
  for (int kind = 0; kind < 2; ++kind) {
    if (kind == 0 ? worker != 0 || !from_before : !tail) continue;
    float acc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = (kind == 0 ? s.head : s.tail)[threadIdx.x][k];
    bool open = kind == 0 ? through : true;
    for (int w = worker + 1; open && w < a.workers; ++w) {
      const int t = w * a.lanes + (int)threadIdx.x % a.lanes;
      if (w * a.share >= count) break;  // it goes on in the next block
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] += s.head[t][k];
      open = s.through[t];
    }
    if (kind == 1 && !open) {
      write_row<TO, N, Whole, Add>(a, keys[end - 1], c, acc);
    } else {
      float* at = piece_at(a, block, kind, (int64_t)piece * N);
#pragma unroll
      for (int k = 0; k < N; ++k) at[k] = acc[k];
    }
  }
}

// Rows that several blocks share: the block that one begins in adds the others' pieces, its workers equal shares of them.
template <typename TO, int N, bool Whole, bool Add> __global__ void __launch_bounds__(kThreads) embedding_join_kernel(SumArgs a) {
  __shared__ float s_sum[kThreads][N];
  griddep_wait();
  const int64_t block = blockIdx.x / a.n_cols;
  const uint32_t key = a.keys_of[2 * block + 1];
  if (key == (uint32_t)a.tokens.rows) return;
  int64_t count = 0;  // blocks behind this one that go on with the row
  for (bool more = true; more;) {
    const int64_t b = block + 1 + count + threadIdx.x;
    const int found = __syncthreads_count(b < a.n_blocks && a.keys_of[2 * b] == key);
    count += found;
    more = found == kThreads;
  }
  const int worker = threadIdx.x / a.lanes;
  const int piece = (int)(blockIdx.x % a.n_cols) * a.lanes + (int)threadIdx.x % a.lanes;
  const bool on = worker < a.workers && piece < a.hop;
  const int64_t c = Whole ? (int64_t)piece * N : piece;
  const int64_t each = (count + a.workers - 1) / a.workers;
  const int64_t from = block + 1 + min(worker * each, count), to = block + 1 + min((worker + 1) * each, count);
  float acc[N];
#pragma unroll
  for (int k = 0; k < N; ++k) acc[k] = on && worker == 0 ? piece_at(a, block, 1, (int64_t)piece * N)[k] : 0.0f;
  if (on) {
#pragma unroll 8
    for (int64_t b = from; b < to; ++b) {
      const float* at = piece_at(a, b, 0, (int64_t)piece * N);
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] += at[k];
    }
  }
#pragma unroll
  for (int k = 0; k < N; ++k) s_sum[threadIdx.x][k] = acc[k];
  __syncthreads();
  if (!on || worker != 0) return;
  for (int w = 1; w < a.workers && w * each < count; ++w)
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] += s_sum[w * a.lanes + threadIdx.x][k];
  write_row<TO, N, Whole, Add>(a, key, c, acc);
}

// ---- plan ----------------------------------------------------------------------------------------------------------

size_t align256(size_t v) { return (v + 255) / 256 * 256; }

// Everything that the sizes decide.
struct GradPlan {
  int hop, lanes, n_cols, workers, share;
  int64_t n_blocks, piece_stride;
  int passes, bits, n_tiles;
  size_t keys[2], places[2], counts, totals, pieces, keys_of, total;
};

GradPlan grad_plan(int64_t n, int64_t rows, int dim, int n_values) {
  GradPlan p{};
  const int per_row = (dim + n_values - 1) / n_values;
  p.hop = per_row;
  p.n_cols = (per_row + kThreads - 1) / kThreads;
  p.lanes = (per_row + p.n_cols - 1) / p.n_cols;
  p.workers = kThreads / p.lanes;
  // as many tokens to a worker as let two waves of half-full SMs cover them; one block where that is not far off
  const int64_t wave = (int64_t)GNR_SM_COUNT_FALLBACK * 2048;
  int64_t share = std::max<int64_t>(16, (n * p.lanes * p.n_cols + wave - 1) / wave);
  if (n <= (int64_t)p.workers * 32) share = std::max<int64_t>(1, (n + p.workers - 1) / p.workers);
  p.share = (int)std::min<int64_t>((share + 7) / 8 * 8, std::max(8, kSpan / p.workers / 8 * 8));
  const int64_t span = (int64_t)p.share * p.workers;
  p.n_blocks = (n + span - 1) / span;
  p.piece_stride = (int64_t)per_row * n_values;
  int key_bits = 1;
  while (((uint64_t)rows >> key_bits) != 0) ++key_bits;
  p.passes = (key_bits + kMaxBits - 1) / kMaxBits;
  p.bits = (key_bits + p.passes - 1) / p.passes;
  p.n_tiles = (int)((n + kTile - 1) / kTile);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += align256(bytes);
    return here;
  };
  if (n > kLocal)
    for (int k = 0; k < (n > kClusterSort ? 2 : 1); ++k) {
      p.keys[k] = take((size_t)n * 4);
      p.places[k] = take((size_t)n * 4);
    }
  if (n > kClusterSort) {
    p.counts = take((size_t)p.n_tiles * kMaxRadix * 4);
    p.totals = take(kMaxRadix * 4);
  }
  if (p.n_blocks > 1) {
    p.pieces = take((size_t)p.n_blocks * 2 * p.piece_stride * 4);
    p.keys_of = take((size_t)p.n_blocks * 2 * 4);
  }
  p.total = at;
  return p;
}

int check_rows(const char* what, int type, int64_t rows, int dim, int index_bits, int64_t n) {
  if (gnr_type_size(type) == 0) {
    gnr_set_error("%s: unknown element type %d", what, type);
    return -1;
  }
  if (index_bits != 32 && index_bits != 64) {
    gnr_set_error("%s: indices of %d bits (32 or 64)", what, index_bits);
    return -1;
  }
  if (rows < 1 || rows > 0x7ffffffe || dim < 1 || n < 0 || n > 0x7fffffff) {
    gnr_set_error("%s: %lld rows of %d values and %lld indices (at least one row and one value, at most 2^31 - 2 rows and 2^31 - 1 indices)",
                  what, (long long)rows, dim, (long long)n);
    return -1;
  }
  return 0;
}

bool aligned(const void* p, int64_t stride, int size, int to) { return (uintptr_t)p % to == 0 && (stride * size) % to == 0; }

}  // namespace

extern "C" int gnr_embedding_lookup(const void* table, int type, int64_t rows, int dim, int64_t table_stride, const void* indices,
                                    int index_bits, int64_t n, float scale, void* out, int64_t out_stride, void* stream) {
  if (int rc = check_rows("gnr_embedding_lookup", type, rows, dim, index_bits, n)) return rc;
  if (n == 0) return 0;
  if (!table || !indices || !out || table_stride < dim || out_stride < dim) {
    gnr_set_error("gnr_embedding_lookup: null pointer, or rows closer than %d values", dim);
    return -1;
  }
  const cudaStream_t st = (cudaStream_t)stream;
  const int size = gnr_type_size(type);
  // pieces of 32 bytes, 16 or one value
  auto fits = [&](int to) { return (int64_t)dim * size % to == 0 && aligned(table, table_stride, size, to) && aligned(out, out_stride, size, to); };
  const int piece = fits(32) ? 32 / size : fits(16) ? 16 / size : 1;
  const int64_t deep = lookup_depth(piece * size);
  const uint32_t per_row = (uint32_t)(dim / piece), n_cols = (per_row + kThreads - 1) / kThreads, lanes = (per_row + n_cols - 1) / n_cols;
  const uint32_t group = (uint32_t)std::min<int64_t>(kThreads / lanes, std::max<int64_t>(1, (n + deep - 1) / deep));
  const uint32_t threads = (group * lanes + 31) / 32 * 32;
  const int64_t blocks = (n + group * deep - 1) / (group * deep) * n_cols;
  if (blocks > 0x7fffffff) {
    gnr_set_error("gnr_embedding_lookup: %lld values are too many for one call", (long long)(n * dim));
    return -1;
  }
  return gnr_with_type(type, [&](auto t) {
    using T = decltype(t);
    constexpr int N = 16 / sizeof(T);
    auto go = [&](auto* index) {
      using I = std::remove_const_t<std::remove_pointer_t<decltype(index)>>;
      auto* kernel = piece == 2 * N ? embedding_lookup_kernel<T, I, 2 * N> : piece == N ? embedding_lookup_kernel<T, I, N> : embedding_lookup_kernel<T, I, 1>;
      kernel<<<(unsigned)blocks, threads, 0, st>>>((const T*)table, rows, table_stride, index, n, per_row, lanes, n_cols, group, scale, (T*)out, out_stride);
    };
    if (index_bits == 64) go((const int64_t*)indices);
    else go((const int32_t*)indices);
    GNR_CUDA_OK(cudaGetLastError());
    return 0;
  });
}

extern "C" int gnr_embedding_grad_workspace_bytes(int64_t n, int64_t rows, int dim, size_t* bytes_h) {
  if (int rc = check_rows("gnr_embedding_grad_workspace_bytes", GNR_FP32, rows, dim, 64, n)) return rc;
  if (!bytes_h) {
    gnr_set_error("gnr_embedding_grad_workspace_bytes: null pointer");
    return -1;
  }
  size_t most = 0;  // of the layouts that the alignments may choose
  for (int n_values : {4, 8}) most = std::max(most, grad_plan(n, rows, dim, n_values).total);
  *bytes_h = most;
  return 0;
}

extern "C" int gnr_embedding_grad(const void* grad, int grad_type, int dim, int64_t grad_stride, const void* indices, int index_bits, int64_t n,
                                  int64_t rows, int64_t padding_row, float scale, int accumulate, void* out, int out_type, int64_t out_stride,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_rows("gnr_embedding_grad", grad_type, rows, dim, index_bits, n)) return rc;
  if (gnr_type_size(out_type) == 0 || !out || out_stride < dim || (n > 0 && (!grad || !indices || grad_stride < dim))) {
    gnr_set_error("gnr_embedding_grad: null pointer, unknown type, or rows closer than %d values", dim);
    return -1;
  }
  const cudaStream_t st = (cudaStream_t)stream;
  const int wide = 16 / gnr_type_size(grad_type), out_wide = std::min(16, wide * gnr_type_size(out_type));
  const bool vec = dim % wide == 0 && aligned(grad, grad_stride, gnr_type_size(grad_type), 16) &&
                   aligned(out, out_stride, gnr_type_size(out_type), out_wide);
  const GradPlan p = grad_plan(n, rows, dim, vec ? wide : 4);
  if (p.total > 0 && (!workspace || p.total > workspace_bytes || (uintptr_t)workspace % 16 != 0)) {
    gnr_set_error("gnr_embedding_grad: workspace of %zu bytes, %zu are needed on a 16-byte boundary", workspace_bytes, p.total);
    return -1;
  }
  // blocks that fill: three to an SM, with 16 KB to write at least and kFillRows rows at most
  const int64_t fill = accumulate ? 0 : std::min<int64_t>(kFillRows, std::max<int64_t>((rows + 3 * GNR_SM_COUNT_FALLBACK - 1) / (3 * GNR_SM_COUNT_FALLBACK),
                                                                                16384 / ((int64_t)dim * gnr_type_size(out_type)) + 1));
  const int64_t blocks = p.n_blocks * p.n_cols + (accumulate ? 0 : (rows + fill - 1) / fill);
  if (blocks > 0x7fffffff) {
    gnr_set_error("gnr_embedding_grad: %lld tokens of %d values are too many for one call", (long long)n, dim);
    return -1;
  }
  if (blocks == 0) return 0;
  char* ws = (char*)workspace;
  auto u32 = [&](size_t at) { return (uint32_t*)(ws + at); };
  const Tokens tokens{indices, index_bits == 64, n, rows, padding_row};
  int cur = 0;
  const bool local = n <= kLocal;
  if (!local && n <= kClusterSort) {
    constexpr int kEach = kClusterSort / kClusterItems;
    auto go = [&](auto items) {
      constexpr int Items = decltype(items)::value;
      GNR_CUDA_OK(cudaFuncSetAttribute(embedding_sort_cluster_kernel<Items>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(ClusterShared<Items>)));
      embedding_sort_cluster_kernel<Items><<<kCluster, kClusterWarps * 32, sizeof(ClusterShared<Items>), st>>>(tokens, p.passes, p.bits, u32(p.keys[0]),
                                                                                                            u32(p.places[0]));
      GNR_CUDA_OK(cudaGetLastError());
      return 0;
    };
    if (int rc = n <= kEach       ? go(std::integral_constant<int, 1>())
                 : n <= 2 * kEach ? go(std::integral_constant<int, 2>())
                 : n <= 4 * kEach ? go(std::integral_constant<int, 4>())
                                  : go(std::integral_constant<int, 8>()))
      return rc;
  } else if (!local) {
    for (int pass = 0; pass < p.passes; ++pass) {
      const uint32_t* keys = pass == 0 ? nullptr : u32(p.keys[cur]);
      const int shift = pass * p.bits, to = pass == 0 ? 0 : cur ^ 1;
      GNR_CUDA_OK((cudaError_t)gnr_launch(embedding_count_kernel, p.n_tiles, kTileWarps * 32, 0, st, pass > 0, tokens, keys, shift, p.bits,
                                          u32(p.counts), p.n_tiles));
      GNR_CUDA_OK((cudaError_t)gnr_launch(embedding_scan_kernel, 1u << p.bits, kThreads, 0, st, true, u32(p.counts), p.n_tiles, u32(p.totals)));
      GNR_CUDA_OK((cudaError_t)gnr_launch(embedding_scatter_kernel, p.n_tiles, kTileWarps * 32, 0, st, true, tokens, keys, u32(p.places[cur]), shift,
                                          p.bits, u32(p.counts), u32(p.totals), p.n_tiles, u32(p.keys[to]), u32(p.places[to])));
      cur = to;
    }
  }
  SumArgs a{};
  a.tokens = tokens;
  a.passes = p.passes;
  a.bits = p.bits;
  a.keys = u32(p.keys[cur]);
  a.places = u32(p.places[cur]);
  a.grad = grad;
  a.grad_stride = grad_stride;
  a.out = out;
  a.out_stride = out_stride;
  a.dim = dim;
  a.hop = p.hop;
  a.lanes = p.lanes;
  a.n_cols = p.n_cols;
  a.workers = p.workers;
  a.share = p.share;
  a.n_blocks = p.n_blocks;
  a.pieces = (float*)(ws + p.pieces);
  a.keys_of = u32(p.keys_of);
  a.piece_stride = p.piece_stride;
  a.scale = scale;
  a.fill_rows = (int)fill;
  return gnr_with_type(grad_type, [&](auto ti) {
    return gnr_with_type(out_type, [&](auto to) {
      using TI = decltype(ti);
      using TO = decltype(to);
      constexpr int N = 16 / sizeof(TI);
      auto pick = [&](auto is_local) {
        constexpr bool L = decltype(is_local)::value;
        return vec ? accumulate ? embedding_sum_kernel<TI, TO, N, true, true, L> : embedding_sum_kernel<TI, TO, N, true, false, L>
                   : accumulate ? embedding_sum_kernel<TI, TO, 4, false, true, L> : embedding_sum_kernel<TI, TO, 4, false, false, L>;
      };
      auto* sum = local ? pick(std::true_type()) : pick(std::false_type());
      auto* join = vec ? accumulate ? embedding_join_kernel<TO, N, true, true> : embedding_join_kernel<TO, N, true, false>
                       : accumulate ? embedding_join_kernel<TO, 4, false, true> : embedding_join_kernel<TO, 4, false, false>;
      GNR_CUDA_OK((cudaError_t)gnr_launch(sum, (unsigned)blocks, kThreads, 0, st, !local, a));
      if (p.n_blocks > 1) GNR_CUDA_OK((cudaError_t)gnr_launch(join, (unsigned)(p.n_blocks * p.n_cols), kThreads, 0, st, true, a));
      return 0;
    });
  });
}
