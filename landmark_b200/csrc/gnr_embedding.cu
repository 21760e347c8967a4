// Embedding rows and their gradient.
//
// Lookup: out[t] = round(scale * table[i_t]).  A copy with a product: bound by the bytes of the rows, each read where the
// index says and written in order.
//
// Gradient: out[v] = round(scale * sum over t with i_t = v of grad[t]), every row of the table written.  The tokens are
// sorted by index (a stable radix sort of (index, token) pairs), then summed in the sorted order, fp32, without atomics on
// floats: the same inputs give the same bits.  The sum is split evenly over the sorted tokens, not over the rows, so one
// row that all tokens name costs no more than many short ones: a worker takes `L` consecutive sorted tokens, writes the rows
// that begin and end inside its share, and leaves the pieces of the others to be joined, first in its block, then
// (join kernel) between blocks, always in the order of the tokens.
#include <algorithm>

#include "gnr_internal.cuh"
#include "gnr_types.cuh"

namespace {

constexpr int kThreads = 256;

// ---- lookup --------------------------------------------------------------------------------------------------------

// One thread per N values of the output; `per_row` such pieces make a row.
template <typename T, typename I, int N>
__global__ void __launch_bounds__(kThreads)
embedding_lookup_kernel(const T* __restrict__ table, int64_t rows, int64_t table_stride, const I* __restrict__ index, int64_t n_pieces,
                        uint32_t per_row, float scale, T* __restrict__ out, int64_t out_stride) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= n_pieces) return;
  const int64_t t = i / per_row;
  const int64_t c = (i - t * per_row) * N;
  const int64_t row = (int64_t)index[t];
  Pack<T, N> x;
  if (row >= 0 && row < rows) {
    x = *reinterpret_cast<const Pack<T, N>*>(table + row * table_stride + c);
#pragma unroll
    for (int k = 0; k < N; ++k) x.v[k] = from_float<T>(to_float(x.v[k]) * scale);
  } else {  // a masked place gives zeros, an index past the table NaN
    const T fill = from_float<T>(row < 0 ? 0.0f : __int_as_float(0x7fc00000));
#pragma unroll
    for (int k = 0; k < N; ++k) x.v[k] = fill;
  }
  *reinterpret_cast<Pack<T, N>*>(out + t * out_stride + c) = x;
}

// ---- sort ----------------------------------------------------------------------------------------------------------

constexpr int kSortThreads = 512;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kItems = 8;                      // tokens of a thread
constexpr int kTile = kSortThreads * kItems;   // tokens of a block
constexpr int kMaxBits = 9;                    // bits of a digit
constexpr int kMaxRadix = 1 << kMaxBits;

struct SortShared {
  uint16_t warp_count[kSortWarps][kMaxRadix];  // tokens of a digit in a warp's share, then before it in the block
  uint32_t base[kMaxRadix];
  uint32_t scan[kSortWarps];
};

// A token's key: its row, or `rows` for what the gradient leaves out (masked, past the table, the padding row).
template <typename I> __device__ __forceinline__ uint32_t token_key(I index, int64_t rows, int64_t padding) {
  const int64_t i = (int64_t)index;
  return i < 0 || i >= rows || i == padding ? (uint32_t)rows : (uint32_t)i;
}

// place of a thread's j-th token in its block's tile: every warp has a run of neighbours
__device__ __forceinline__ int tile_place(int j) { return (threadIdx.x >> 5) * (32 * kItems) + j * 32 + (threadIdx.x & 31); }

// Ranks of a tile's tokens among the tokens of the same digit, in the tile's order.  digit < 0: no token.
// Afterwards warp_count[w][d] holds the tokens of digit d in the warps before w, and the return value of thread d < radix is
// the number of them in the tile.
__device__ __forceinline__ uint32_t rank_tile(SortShared& s, const int (&digit)[kItems], uint32_t (&rank)[kItems], int radix) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kSortWarps * kMaxRadix / 2; i += kSortThreads) reinterpret_cast<uint32_t*>(s.warp_count)[i] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const uint32_t peers = __match_any_sync(0xffffffffu, digit[j]);
    const uint32_t before = peers & ((1u << lane) - 1u);
    rank[j] = digit[j] < 0 ? 0u : s.warp_count[warp][digit[j]] + __popc(before);
    __syncwarp();
    if (digit[j] >= 0 && before == 0) s.warp_count[warp][digit[j]] += (uint16_t)__popc(peers);
    __syncwarp();
  }
  __syncthreads();
  uint32_t sum = 0;
  if (threadIdx.x < radix)
    for (int w = 0; w < kSortWarps; ++w) {
      const uint32_t c = s.warp_count[w][threadIdx.x];
      s.warp_count[w][threadIdx.x] = (uint16_t)sum;
      sum += c;
    }
  __syncthreads();
  return sum;
}

// exclusive sum over the block's threads
__device__ __forceinline__ uint32_t block_exclusive(SortShared& s, uint32_t x) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t sum = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += y;
  }
  if (lane == 31) s.scan[warp] = sum;
  __syncthreads();
  uint32_t before = 0;
  for (int w = 0; w < warp; ++w) before += s.scan[w];
  __syncthreads();
  return before + sum - x;
}

// Every pass of the sort in one block, for at most kTile tokens.
template <typename I>
__global__ void __launch_bounds__(kSortThreads)
embedding_sort_block_kernel(const I* __restrict__ index, int n, int64_t rows, int64_t padding, int passes, int bits,
                            uint32_t* __restrict__ keys, uint32_t* __restrict__ tokens) {
  extern __shared__ __align__(16) unsigned char smem[];
  SortShared& s = *reinterpret_cast<SortShared*>(smem);
  uint32_t* s_key = reinterpret_cast<uint32_t*>(smem + sizeof(SortShared));
  uint32_t* s_token = s_key + kTile;
  uint32_t key[kItems], token[kItems], rank[kItems];
  int digit[kItems];
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const int i = tile_place(j);
    token[j] = i;
    key[j] = i < n ? token_key(index[i], rows, padding) : 0xffffffffu;
  }
  const int radix = 1 << bits;
  for (int pass = 0; pass < passes; ++pass) {
#pragma unroll
    for (int j = 0; j < kItems; ++j) digit[j] = tile_place(j) < n ? (int)((key[j] >> (pass * bits)) & (radix - 1)) : -1;
    const uint32_t count = rank_tile(s, digit, rank, radix);
    const uint32_t base = block_exclusive(s, count);
    if (threadIdx.x < radix) s.base[threadIdx.x] = base;
    __syncthreads();
    const int warp = threadIdx.x >> 5;
#pragma unroll
    for (int j = 0; j < kItems; ++j)
      if (digit[j] >= 0) {
        const uint32_t at = s.base[digit[j]] + s.warp_count[warp][digit[j]] + rank[j];
        s_key[at] = key[j];
        s_token[at] = token[j];
      }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      const int i = tile_place(j);
      if (i < n) {
        key[j] = s_key[i];
        token[j] = s_token[i];
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const int i = tile_place(j);
    if (i < n) {
      keys[i] = key[j];
      tokens[i] = token[j];
    }
  }
}

// tokens of every digit in every tile: counts[digit][tile].  `index`: the first pass reads the indices themselves.
template <typename I>
__global__ void __launch_bounds__(kSortThreads)
embedding_count_kernel(const I* __restrict__ index, const uint32_t* __restrict__ keys, int64_t n, int64_t rows, int64_t padding, int shift,
                       int bits, uint32_t* __restrict__ counts, int n_tiles) {
  __shared__ uint32_t s_count[kMaxRadix];
  const int radix = 1 << bits;
  griddep_wait();
  for (int d = threadIdx.x; d < radix; d += kSortThreads) s_count[d] = 0;
  __syncthreads();
  const int64_t tile0 = (int64_t)blockIdx.x * kTile;
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const int64_t i = tile0 + tile_place(j);
    int d = -1;
    if (i < n) d = (int)(((index ? token_key(index[i], rows, padding) : keys[i]) >> shift) & (radix - 1));
    const uint32_t peers = __match_any_sync(0xffffffffu, d);
    if (d >= 0 && (peers & ((1u << (threadIdx.x & 31)) - 1u)) == 0) atomicAdd(&s_count[d], __popc(peers));
  }
  __syncthreads();
  for (int d = threadIdx.x; d < radix; d += kSortThreads) counts[(int64_t)d * n_tiles + blockIdx.x] = s_count[d];
}

// One block per digit: its counts become the tokens of that digit in the tiles before, and totals[digit] their sum.
__global__ void __launch_bounds__(kThreads) embedding_scan_kernel(uint32_t* __restrict__ counts, int n_tiles, uint32_t* __restrict__ totals) {
  __shared__ uint32_t s_sum[kThreads / 32];
  griddep_wait();
  uint32_t* row = counts + (int64_t)blockIdx.x * n_tiles;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t carry = 0;
  for (int first = 0; first < n_tiles; first += kThreads) {
    const int i = first + threadIdx.x;
    const uint32_t x = i < n_tiles ? row[i] : 0u;
    uint32_t sum = x;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += y;
    }
    if (lane == 31) s_sum[warp] = sum;
    __syncthreads();
    uint32_t before = 0, all = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) before += s_sum[w];
      all += s_sum[w];
    }
    if (i < n_tiles) row[i] = carry + before + sum - x;
    carry += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

template <typename I>
__global__ void __launch_bounds__(kSortThreads)
embedding_scatter_kernel(const I* __restrict__ index, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ tokens, int64_t n,
                         int64_t rows, int64_t padding, int shift, int bits, const uint32_t* __restrict__ counts,
                         const uint32_t* __restrict__ totals, int n_tiles, uint32_t* __restrict__ out_keys,
                         uint32_t* __restrict__ out_tokens) {
  __shared__ SortShared s;
  griddep_wait();
  const int radix = 1 << bits;
  const int64_t tile0 = (int64_t)blockIdx.x * kTile;
  uint32_t key[kItems], token[kItems], rank[kItems];
  int digit[kItems];
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const int64_t i = tile0 + tile_place(j);
    digit[j] = -1;
    if (i < n) {
      key[j] = index ? token_key(index[i], rows, padding) : keys[i];
      token[j] = index ? (uint32_t)i : tokens[i];
      digit[j] = (int)((key[j] >> shift) & (radix - 1));
    }
  }
  rank_tile(s, digit, rank, radix);
  const uint32_t base = block_exclusive(s, threadIdx.x < radix ? totals[threadIdx.x] : 0u);
  if (threadIdx.x < radix) s.base[threadIdx.x] = base + counts[(int64_t)threadIdx.x * n_tiles + blockIdx.x];
  __syncthreads();
  const int warp = threadIdx.x >> 5;
#pragma unroll
  for (int j = 0; j < kItems; ++j)
    if (digit[j] >= 0) {
      const uint32_t at = s.base[digit[j]] + s.warp_count[warp][digit[j]] + rank[j];
      out_keys[at] = key[j];
      out_tokens[at] = token[j];
    }
}

// ---- sums ----------------------------------------------------------------------------------------------------------

struct SumArgs {
  const void* grad;
  int64_t grad_stride;
  void* out;
  int64_t out_stride;
  const uint32_t* keys;    // sorted; entries of key `rows` are left out
  const uint32_t* tokens;
  int64_t n, rows;
  int dim, lanes, n_cols;  // lanes: pieces of a row that a block's worker takes, n_cols such parts make a row
  int workers;             // workers of a block
  int share;               // sorted tokens of a worker
  int64_t n_blocks;        // blocks along the tokens
  float* pieces;           // [n_blocks][2][padded dim]: the sum that a block's first row had before its first token's share ...
  int64_t piece_stride;    // ... (the row began in an earlier block), and that of a row that ends in a later one
  float scale;
  int accumulate;
  int64_t fill_rows;       // rows of a block that writes the rows without a token, 0: none does
};

template <typename TO, int N> __device__ __forceinline__ void write_row(const SumArgs& a, uint32_t row, int64_t c, const float (&x)[N]) {
  Pack<TO, N>* at = reinterpret_cast<Pack<TO, N>*>(static_cast<TO*>(a.out) + (int64_t)row * a.out_stride + c);
  Pack<TO, N> y;
  if (a.accumulate) {
    const Pack<TO, N> old = *at;
#pragma unroll
    for (int k = 0; k < N; ++k) y.v[k] = from_float<TO>(fmaf(x[k], a.scale, to_float(old.v[k])));
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) y.v[k] = from_float<TO>(x[k] * a.scale);
  }
  *at = y;
}

template <int N> __device__ __forceinline__ float* piece_at(const SumArgs& a, int64_t block, int which, int64_t c) {
  return a.pieces + (block * 2 + which) * a.piece_stride + c;
}

// first position of the sorted keys that is not below `key`
__device__ __forceinline__ int64_t lower_bound(const uint32_t* keys, int64_t n, uint32_t key) {
  int64_t lo = 0, hi = n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (keys[mid] < key) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

// zeros in the rows that no token names
template <typename TO, int N> __device__ __forceinline__ void fill_rows(const SumArgs& a, int64_t first) {
  __shared__ uint32_t s_named[kThreads / 32];
  const int64_t last = min(first + a.fill_rows, a.rows);
  if (threadIdx.x < kThreads / 32) s_named[threadIdx.x] = 0;
  __syncthreads();
  if (threadIdx.x < last - first) {
    const uint32_t row = (uint32_t)(first + threadIdx.x);
    const int64_t at = lower_bound(a.keys, a.n, row);
    if (at < a.n && a.keys[at] == row) atomicOr(&s_named[threadIdx.x >> 5], 1u << (threadIdx.x & 31));
  }
  __syncthreads();
  const int per_row = a.dim / N;
  Pack<TO, N> zero;
#pragma unroll
  for (int k = 0; k < N; ++k) zero.v[k] = from_float<TO>(0.0f);
  for (int64_t row = first; row < last; ++row) {
    const int r = (int)(row - first);
    if (s_named[r >> 5] >> (r & 31) & 1u) continue;
    for (int c = threadIdx.x; c < per_row; c += kThreads)
      *reinterpret_cast<Pack<TO, N>*>(static_cast<TO*>(a.out) + row * a.out_stride + (int64_t)c * N) = zero;
  }
}

constexpr int kBatch = 8;  // rows in flight per worker

template <typename TI, typename TO, int N> __global__ void __launch_bounds__(kThreads) embedding_sum_kernel(SumArgs a) {
  __shared__ float s_head[kThreads][N], s_tail[kThreads][N];
  __shared__ uint32_t s_tail_key[kThreads];  // key of the row that goes on behind a worker's share, or `rows`
  __shared__ int s_through[kThreads];        // the whole share is one row that began before it and goes on behind it
  griddep_wait();
  const int64_t sum_blocks = a.n_blocks * a.n_cols;
  if (blockIdx.x >= sum_blocks) {
    fill_rows<TO, N>(a, ((int64_t)blockIdx.x - sum_blocks) * a.fill_rows);
    return;
  }
  const int64_t block = blockIdx.x / a.n_cols;
  const int worker = threadIdx.x / a.lanes;
  const int piece = (int)(blockIdx.x % a.n_cols) * a.lanes + (int)threadIdx.x % a.lanes;
  const bool on = worker < a.workers && piece * N < a.dim;
  const int64_t c = (int64_t)piece * N;
  const uint32_t none = (uint32_t)a.rows;
  const int64_t begin = (block * a.workers + worker) * a.share, end = min(begin + a.share, a.n);
  const TI* grad = static_cast<const TI*>(a.grad) + c;
  uint32_t tail_key = none, head_key = none;
  bool through = false;
  if (on && begin < end) {
    uint32_t cur = a.keys[begin];
    bool first = begin > 0 && a.keys[begin - 1] == cur;  // this row began before the share
    if (first) head_key = cur;
    float acc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = 0.0f;
    for (int64_t i = begin; i < end; i += kBatch) {
      uint32_t key[kBatch];
      Pack<TI, N> x[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        key[b] = i + b < end ? a.keys[i + b] : none;
        if (key[b] != none) x[b] = *reinterpret_cast<const Pack<TI, N>*>(grad + (int64_t)a.tokens[i + b] * a.grad_stride);
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        if (i + b >= end) break;
        if (key[b] != cur) {
          if (first) {
#pragma unroll
            for (int k = 0; k < N; ++k) s_head[threadIdx.x][k] = acc[k];
          } else if (cur != none) {
            write_row<TO, N>(a, cur, c, acc);
          }
          first = false;
          cur = key[b];
#pragma unroll
          for (int k = 0; k < N; ++k) acc[k] = 0.0f;
        }
        if (cur != none) {
#pragma unroll
          for (int k = 0; k < N; ++k) acc[k] += to_float(x[b].v[k]);
        }
      }
    }
    const bool goes_on = cur != none && end < a.n && a.keys[end] == cur;
    if (first) {
#pragma unroll
      for (int k = 0; k < N; ++k) s_head[threadIdx.x][k] = acc[k];
      through = goes_on;
    } else if (goes_on) {
#pragma unroll
      for (int k = 0; k < N; ++k) s_tail[threadIdx.x][k] = acc[k];
      tail_key = cur;
    } else if (cur != none) {
      write_row<TO, N>(a, cur, c, acc);
    }
  }
  s_tail_key[threadIdx.x] = tail_key;
  s_through[threadIdx.x] = through;
  __syncthreads();
  if (!on) return;
  // A row that goes on behind a worker's share is joined by the worker it begins with; the one that came from the block
  // before by the first.
  const bool from_before = worker == 0 && head_key != none;
  for (int kind = 0; kind < 2; ++kind) {
    if (kind == 0 ? !from_before : tail_key == none) continue;
    float acc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = kind == 0 ? s_head[threadIdx.x][k] : s_tail[threadIdx.x][k];
    bool open = kind == 0 ? through : true;
    for (int w = worker + 1; open && w < a.workers; ++w) {
      const int t = w * a.lanes + (int)threadIdx.x % a.lanes;
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] += s_head[t][k];
      open = s_through[t];
    }
    if (kind == 1 && !open) {
      write_row<TO, N>(a, tail_key, c, acc);
    } else {
      float* at = piece_at<N>(a, block, kind, c);
#pragma unroll
      for (int k = 0; k < N; ++k) at[k] = acc[k];
    }
  }
}

// Rows that several blocks share: the block that one begins in adds the others' pieces, its workers equal shares of them.
template <typename TO, int N> __global__ void __launch_bounds__(kThreads) embedding_join_kernel(SumArgs a) {
  __shared__ float s_sum[kThreads][N];
  griddep_wait();
  const int64_t block = blockIdx.x / a.n_cols;
  const int64_t span = (int64_t)a.workers * a.share;
  const int64_t begin = block * span, end = begin + span;
  if (end >= a.n) return;
  const uint32_t key = a.keys[end];
  if (key == (uint32_t)a.rows || a.keys[end - 1] != key) return;
  if (begin > 0 && a.keys[begin - 1] == key) return;  // it began before this block
  // blocks whose first token is of this row: [block + 1, last)
  int64_t lo = block + 1, hi = a.n_blocks;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (a.keys[mid * span] == key) lo = mid + 1;
    else hi = mid;
  }
  const int64_t count = lo - (block + 1);
  const int worker = threadIdx.x / a.lanes;
  const int piece = (int)(blockIdx.x % a.n_cols) * a.lanes + (int)threadIdx.x % a.lanes;
  const bool on = worker < a.workers && piece * N < a.dim;
  const int64_t c = (int64_t)piece * N;
  const int64_t each = (count + a.workers - 1) / a.workers;
  const int64_t first = block + 1 + min(worker * each, count), last = block + 1 + min((worker + 1) * each, count);
  float acc[N];
#pragma unroll
  for (int k = 0; k < N; ++k) acc[k] = on && worker == 0 ? piece_at<N>(a, block, 1, c)[k] : 0.0f;
  if (on) {
#pragma unroll 8
    for (int64_t b = first; b < last; ++b) {
      const float* at = piece_at<N>(a, b, 0, c);
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
  write_row<TO, N>(a, key, c, acc);
}

// ---- plan ----------------------------------------------------------------------------------------------------------

size_t align256(size_t v) { return (v + 255) / 256 * 256; }

// Everything that the sizes decide.
struct GradPlan {
  int n_values;            // values of a piece
  int lanes, n_cols, workers, share;
  int64_t n_blocks, piece_stride;
  int passes, bits, n_tiles;
  size_t keys[2], tokens[2], counts, totals, pieces, total;
};

GradPlan grad_plan(int64_t n, int64_t rows, int dim, int n_values) {
  GradPlan p{};
  p.n_values = n_values;
  const int per_row = (dim + n_values - 1) / n_values;
  p.lanes = std::min(per_row, kThreads);
  p.n_cols = (per_row + p.lanes - 1) / p.lanes;
  p.workers = kThreads / p.lanes;
  // as many tokens to a worker as let the threads of one wave of full SMs cover them, at least two batches
  const int64_t wave = (int64_t)GNR_SM_COUNT_FALLBACK * 2048;
  const int64_t share = (n * p.lanes * p.n_cols + wave - 1) / wave;
  p.share = (int)std::max<int64_t>(2 * kBatch, (share + kBatch - 1) / kBatch * kBatch);
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
  for (int k = 0; k < 2; ++k) {
    p.keys[k] = take((size_t)n * 4);
    p.tokens[k] = take((size_t)n * 4);
  }
  p.counts = take((size_t)p.n_tiles * kMaxRadix * 4);
  p.totals = take(kMaxRadix * 4);
  p.pieces = take((size_t)p.n_blocks * 2 * p.piece_stride * 4);
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
  const int size = gnr_type_size(type), wide = 16 / size;
  const bool vec = dim % wide == 0 && aligned(table, table_stride, size, 16) && aligned(out, out_stride, size, 16);
  const int per_row = vec ? dim / wide : dim;
  const int64_t pieces = n * per_row, blocks = (pieces + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffff) {
    gnr_set_error("gnr_embedding_lookup: %lld values are too many for one call", (long long)(n * dim));
    return -1;
  }
  return gnr_with_type(type, [&](auto t) {
    using T = decltype(t);
    constexpr int N = 16 / sizeof(T);
    auto go = [&](auto* index) {
      using I = std::remove_pointer_t<decltype(index)>;
      if (vec)
        embedding_lookup_kernel<T, I, N><<<(unsigned)blocks, kThreads, 0, st>>>((const T*)table, rows, table_stride, index, pieces, per_row,
                                                                              scale, (T*)out, out_stride);
      else
        embedding_lookup_kernel<T, I, 1><<<(unsigned)blocks, kThreads, 0, st>>>((const T*)table, rows, table_stride, index, pieces, per_row,
                                                                              scale, (T*)out, out_stride);
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
  for (int n_values : {1, 4, 8}) most = std::max(most, grad_plan(n, rows, dim, n_values).total);
  *bytes_h = most;
  return 0;
}

extern "C" int gnr_embedding_grad(const void* grad, int grad_type, int dim, int64_t grad_stride, const void* indices, int index_bits, int64_t n,
                                  int64_t rows, int64_t padding_row, float scale, int accumulate, void* out, int out_type, int64_t out_stride,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_rows("gnr_embedding_grad", grad_type, rows, dim, index_bits, n)) return rc;
  if (gnr_type_size(out_type) == 0 || !out || out_stride < dim || (n > 0 && (!grad || !indices || !workspace || grad_stride < dim))) {
    gnr_set_error("gnr_embedding_grad: null pointer, unknown type, or rows closer than %d values", dim);
    return -1;
  }
  const cudaStream_t st = (cudaStream_t)stream;
  const int wide = 16 / gnr_type_size(grad_type), out_wide = std::min(16, wide * gnr_type_size(out_type));
  const bool vec = dim % wide == 0 && aligned(grad, grad_stride, gnr_type_size(grad_type), 16) &&
                   aligned(out, out_stride, gnr_type_size(out_type), out_wide);
  const GradPlan p = grad_plan(n, rows, dim, vec ? wide : 1);
  if (n > 0 && (p.total > workspace_bytes || (uintptr_t)workspace % 16 != 0)) {
    gnr_set_error("gnr_embedding_grad: workspace of %zu bytes, %zu are needed on a 16-byte boundary", workspace_bytes, p.total);
    return -1;
  }
  char* ws = (char*)workspace;
  auto u32 = [&](size_t at) { return (uint32_t*)(ws + at); };
  int cur = 0;
  auto sort = [&](auto* index) {
    using I = std::remove_const_t<std::remove_pointer_t<decltype(index)>>;
    if (n <= kTile) {
      const size_t smem = sizeof(SortShared) + 2 * kTile * 4;
      GNR_CUDA_OK(cudaFuncSetAttribute(embedding_sort_block_kernel<I>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
      embedding_sort_block_kernel<I><<<1, kSortThreads, smem, st>>>(index, (int)n, rows, padding_row, p.passes, p.bits, u32(p.keys[0]),
                                                                    u32(p.tokens[0]));
      GNR_CUDA_OK(cudaGetLastError());
      return 0;
    }
    for (int pass = 0; pass < p.passes; ++pass) {
      const I* source = pass == 0 ? index : nullptr;
      const int shift = pass * p.bits, to = pass == 0 ? 0 : cur ^ 1;
      GNR_CUDA_OK((cudaError_t)gnr_launch(embedding_count_kernel<I>, p.n_tiles, kSortThreads, 0, st, pass > 0, source, u32(p.keys[cur]), n, rows,
                                          padding_row, shift, p.bits, u32(p.counts), p.n_tiles));
      GNR_CUDA_OK((cudaError_t)gnr_launch(embedding_scan_kernel, 1u << p.bits, kThreads, 0, st, true, u32(p.counts), p.n_tiles, u32(p.totals)));
      GNR_CUDA_OK((cudaError_t)gnr_launch(embedding_scatter_kernel<I>, p.n_tiles, kSortThreads, 0, st, true, source, u32(p.keys[cur]),
                                          u32(p.tokens[cur]), n, rows, padding_row, shift, p.bits, u32(p.counts), u32(p.totals), p.n_tiles,
                                          u32(p.keys[to]), u32(p.tokens[to])));
      cur = to;
    }
    return 0;
  };
  if (n > 0)
    if (int rc = index_bits == 64 ? sort((const int64_t*)indices) : sort((const int32_t*)indices)) return rc;
  SumArgs a{};
  a.grad = grad;
  a.grad_stride = grad_stride;
  a.out = out;
  a.out_stride = out_stride;
  a.keys = u32(p.keys[cur]);
  a.tokens = u32(p.tokens[cur]);
  a.n = n;
  a.rows = rows;
  a.dim = dim;
  a.lanes = p.lanes;
  a.n_cols = p.n_cols;
  a.workers = p.workers;
  a.share = p.share;
  a.n_blocks = p.n_blocks;
  a.pieces = (float*)(ws + p.pieces);
  a.piece_stride = p.piece_stride;
  a.scale = scale;
  a.accumulate = accumulate != 0;
  // a block of the fill writes some 32 KB
  a.fill_rows = accumulate ? 0 : std::max<int64_t>(1, std::min<int64_t>(kThreads, 32768 / ((int64_t)dim * gnr_type_size(out_type))));
  const int64_t fill_blocks = accumulate ? 0 : (rows + a.fill_rows - 1) / a.fill_rows;
  const int64_t blocks = p.n_blocks * p.n_cols + fill_blocks;
  if (blocks > 0x7fffffff) {
    gnr_set_error("gnr_embedding_grad: %lld tokens of %d values are too many for one call", (long long)n, dim);
    return -1;
  }
  if (blocks == 0) return 0;
  return gnr_with_type(grad_type, [&](auto ti) {
    return gnr_with_type(out_type, [&](auto to) {
      using TI = decltype(ti);
      using TO = decltype(to);
      constexpr int N = 16 / sizeof(TI);
      GNR_CUDA_OK((cudaError_t)(vec ? gnr_launch(embedding_sum_kernel<TI, TO, N>, (unsigned)blocks, kThreads, 0, st, n > 0, a)
                                    : gnr_launch(embedding_sum_kernel<TI, TO, 1>, (unsigned)blocks, kThreads, 0, st, n > 0, a)));
      if (p.n_blocks > 1)
        GNR_CUDA_OK((cudaError_t)(vec ? gnr_launch(embedding_join_kernel<TO, N>, (unsigned)(p.n_blocks * p.n_cols), kThreads, 0, st, true, a)
                                      : gnr_launch(embedding_join_kernel<TO, 1>, (unsigned)(p.n_blocks * p.n_cols), kThreads, 0, st, true, a)));
      return 0;
    });
  });
}
