// Token embedding: rows of a table, scaled, and the table's gradient by sorted tokens.
//
//   forward   x[t] = round(scale * table[id[t]])
//   gradient  d_table[i] = scale * sum over the tokens t with id[t] = i, in order of t, of dy[t]; zero rows elsewhere
//
// The lookup is bound by memory: 69 us for 16384 tokens out of a 49152 x 4096 fp32 table to bf16 (5.2 TB/s of the 363 MB
// that have to move, 0.80 of a plain copy).
// The gradient is bound by its dense result: every row is written once, 805 MB for 49152 x 4096 in fp32, of which 16384
// tokens touch a quarter. So nothing is cleared beforehand and nothing is accumulated in memory: the tokens are sorted by id
// (stable radix sort, a few us), every row knows its run of tokens and one kernel writes zeros, single rows and sums.
// Sums are taken in token order in fp32 by the thread that owns the column: no atomics, repeated calls are bit-identical.
// A run of more than 32 tokens (frequent tokens of a text) would keep one block busy, so runs are cut at multiples of 32
// in the sorted order; the pieces of long runs are summed first, by as many blocks, and then added in order.
#include "common.cuh"

namespace ct {
namespace {

constexpr int kRadixBits = 8, kRadix = 1 << kRadixBits;
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32;
// Up to 1024 tokens are sorted by one block in shared memory, up to 32768 by a cluster of eight blocks in one launch (for
// calls of this size launches count: 12 thousand tokens on a narrow table take 32 us, 45 with two launches per digit), more
// by as many blocks as it takes, two launches per digit.
constexpr int kOneBlockItems = kSortThreads;
constexpr int kCluster = 8, kClusterItems = 4 * kCluster * kSortThreads;
constexpr int kManySteps = 4, kManyItems = kManySteps * kSortThreads;
constexpr int kPiece = 32;                             // sorted tokens per piece of a long run
constexpr int kBadToken = 9;                           // device error code

// ---- forward ---------------------------------------------------------------------------
template <typename T> struct alignas(16) Vec { T v[16 / sizeof(T)]; };

// 8 columns per thread: one or two 16-byte loads, one store of 16 or 32 bytes (which has to be aligned to its size).
template <typename T> __device__ __forceinline__ void load8(float (&x)[8], const T* p) {
  constexpr int N = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 8 / N; ++i) {
    const Vec<T> w = reinterpret_cast<const Vec<T>*>(p)[i];
#pragma unroll
    for (int e = 0; e < N; ++e) x[N * i + e] = to_float<T>(w.v[e]);
  }
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {      // one 32-byte store
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]),
               "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
               : "memory");
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  constexpr int N = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 8 / N; ++i) {
    Vec<T> w;
#pragma unroll
    for (int e = 0; e < N; ++e) w.v[e] = from_float<T>(x[N * i + e]);
    reinterpret_cast<Vec<T>*>(p)[i] = w;
  }
}

template <typename W, typename T, bool VECTOR>
__global__ void __launch_bounds__(256) embedding_forward_kernel(const int64_t* ids, const W* table, T* out, int64_t tokens,
                                                                int64_t rows, int64_t width, float scale, int* error_flag) {
  const int64_t per_row = VECTOR ? width / 8 : width, total = tokens * per_row;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += step) {
    const int64_t token = i / per_row, column = (i - token * per_row) * (VECTOR ? 8 : 1);
    const int64_t id = ids[token];
    const bool known = id >= 0 && id < rows;
    if (!known && column == 0) atomicCAS(error_flag, 0, kBadToken);
    if constexpr (VECTOR) {
      float x[8] = {};
      if (known) load8<W>(x, table + id * width + column);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= scale;
      store8(out + token * width + column, x);
    } else {
      out[token * width + column] = from_float<T>(known ? to_float<W>(table[id * width + column]) * scale : 0.0f);
    }
  }
}

// ---- stable radix sort of (key, position) --------------------------------------------------
// A block ranks its items by one digit: every warp owns a contiguous stretch and counts its digits in order, which gives each
// item its rank; the counts are summed over warps and digits, and every item goes to its place.
struct SortShared {
  int counts[kSortWarps][kRadix];
  int digit_base[kRadix];
};

// Lanes of the warp whose digit equals this lane's, among lanes with an item (digit >= 0). A vote per bit: the match
// instruction made the one-block sort of 16384 tokens take 81 us.
__device__ __forceinline__ uint32_t same_digit(int digit) {
  uint32_t peers = __ballot_sync(0xffffffffu, digit >= 0);
#pragma unroll
  for (int bit = 0; bit < kRadixBits; ++bit) {
    const uint32_t ones = __ballot_sync(0xffffffffu, (digit >> bit) & 1);
    peers &= (digit >> bit) & 1 ? ones : ~ones;
  }
  return peers;
}

// Counts the warp's digits; rank[k] = items of the same digit before item k in the warp's stretch.
template <int STEPS> __device__ __forceinline__ void count_digits(SortShared& s, const int (&digit)[STEPS], int (&rank)[STEPS]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = lane; i < kRadix; i += 32) s.counts[warp][i] = 0;
  __syncwarp();
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    const uint32_t peers = same_digit(digit[k]);
    rank[k] = digit[k] >= 0 ? s.counts[warp][digit[k]] + __popc(peers & ((1u << lane) - 1)) : 0;
    __syncwarp();
    if (digit[k] >= 0 && lane == __ffs(peers) - 1) s.counts[warp][digit[k]] += __popc(peers);
    __syncwarp();
  }
}

// Counts of the warps -> first place of each warp within each digit; returns (threads < kRadix) the digit's total.
__device__ __forceinline__ int sum_over_warps(SortShared& s) {
  int total = 0;
  __syncthreads();
  if (threadIdx.x < kRadix) {
    for (int w = 0; w < kSortWarps; ++w) {
      const int c = s.counts[w][threadIdx.x];
      s.counts[w][threadIdx.x] = total;
      total += c;
    }
  }
  return total;
}

// Exclusive sum over the digits of `value` (threads < kRadix); all threads of the block call it.
__device__ __forceinline__ void digit_sums(SortShared& s, int value) {
  const int lane = threadIdx.x & 31;
  __shared__ int warp_sum[kRadix / 32];
  int inclusive = value;
  if (threadIdx.x < kRadix) {
#pragma unroll
    for (int step = 1; step < 32; step <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, inclusive, step);
      if (lane >= step) inclusive += other;
    }
    if (lane == 31) warp_sum[threadIdx.x >> 5] = inclusive;
  }
  __syncthreads();
  if (threadIdx.x < kRadix) {
    int before = 0;
    for (int w = 0; w < static_cast<int>(threadIdx.x >> 5); ++w) before += warp_sum[w];
    s.digit_base[threadIdx.x] = before + inclusive - value;
  }
  __syncthreads();
}

template <int STEPS, typename Place>
__device__ __forceinline__ void hand_out(const SortShared& s, const int (&digit)[STEPS], const int (&rank)[STEPS], Place place) {
  const int warp = threadIdx.x >> 5;
#pragma unroll
  for (int k = 0; k < STEPS; ++k)
    if (digit[k] >= 0) place(k, s.digit_base[digit[k]] + s.counts[warp][digit[k]] + rank[k]);
}

// Tokens of the padding row and of ids outside the table get the key `rows`: behind every row's run.
__device__ __forceinline__ int key_of(int64_t id, int64_t rows, int64_t padding, int* error_flag) {
  if (id < 0 || id >= rows) {
    atomicCAS(error_flag, 0, kBadToken);
    return static_cast<int>(rows);
  }
  return id == padding ? static_cast<int>(rows) : static_cast<int>(id);
}

__device__ __forceinline__ int item_index(int k, int items_per_warp) {
  return (threadIdx.x >> 5) * items_per_warp + 32 * k + (threadIdx.x & 31);
}

__global__ void __launch_bounds__(kSortThreads) embedding_sort_one_block_kernel(const int64_t* ids, int tokens, int64_t rows, int64_t padding,
                                                                                int bits, int* keys, int* positions, int* error_flag) {
  grid_dependency_wait();
  constexpr int STEPS = 1;
  __shared__ int2 items[kOneBlockItems];                 // (key, position)
  __shared__ SortShared s;
  int2 mine[STEPS];
  int digit[STEPS], rank[STEPS];
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    const int at = item_index(k, 32 * STEPS);
    mine[k] = at < tokens ? make_int2(key_of(ids[at], rows, padding, error_flag), at) : make_int2(-1, 0);
  }
  for (int shift = 0; shift < bits; shift += kRadixBits) {
#pragma unroll
    for (int k = 0; k < STEPS; ++k) digit[k] = mine[k].x < 0 ? -1 : (mine[k].x >> shift) & (kRadix - 1);
    count_digits(s, digit, rank);
    const int total = sum_over_warps(s);
    digit_sums(s, total);
    hand_out(s, digit, rank, [&](int k, int at) { items[at] = mine[k]; });
    __syncthreads();
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
      const int at = item_index(k, 32 * STEPS);
      mine[k] = at < tokens ? items[at] : make_int2(-1, 0);
    }
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    const int at = item_index(k, 32 * STEPS);
    if (at < tokens) {
      keys[at] = mine[k].x;
      positions[at] = mine[k].y;
    }
  }
}

// The first pass takes its keys from the ids (src_keys null).
template <int STEPS>
__device__ __forceinline__ void load_items(int (&key)[STEPS], int (&position)[STEPS], const int64_t* ids, const int* src_keys,
                                           const int* src_positions, int64_t tokens, int64_t rows, int64_t padding, int* error_flag) {
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    const int64_t at = static_cast<int64_t>(blockIdx.x) * STEPS * kSortThreads + item_index(k, 32 * STEPS);
    key[k] = -1;
    position[k] = 0;
    if (at < tokens) {
      key[k] = src_keys ? src_keys[at] : key_of(ids[at], rows, padding, error_flag);
      position[k] = src_keys ? src_positions[at] : static_cast<int>(at);
    }
  }
}

template <int STEPS>
__global__ void __launch_bounds__(kSortThreads) embedding_sort_count_kernel(const int64_t* ids, const int* src_keys, int64_t tokens, int64_t rows,
                                                                            int64_t padding, int shift, int* histogram, int* error_flag) {
  grid_dependency_wait();
  __shared__ SortShared s;
  int key[STEPS], position[STEPS], digit[STEPS], rank[STEPS];
  load_items(key, position, ids, src_keys, src_keys, tokens, rows, padding, error_flag);
#pragma unroll
  for (int k = 0; k < STEPS; ++k) digit[k] = key[k] < 0 ? -1 : (key[k] >> shift) & (kRadix - 1);
  count_digits(s, digit, rank);
  const int total = sum_over_warps(s);
  if (threadIdx.x < kRadix) histogram[static_cast<int64_t>(blockIdx.x) * kRadix + threadIdx.x] = total;
}

// The blocks' histograms -> the first place of each digit's items of this block: the items of smaller digits in all blocks,
// and those of the digit in the blocks before. Every block sums the histograms for itself.
__device__ __forceinline__ void place_digits(SortShared& s, const int* histogram, int blocks, int block) {
  int total = 0, before = 0;
  if (threadIdx.x < kRadix)
    for (int b = 0; b < blocks; ++b) {
      const int n = histogram[static_cast<int64_t>(b) * kRadix + threadIdx.x];
      before += b < block ? n : 0;
      total += n;
    }
  digit_sums(s, total);
  if (threadIdx.x < kRadix) s.digit_base[threadIdx.x] += before;
  __syncthreads();
}

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The whole sort by one cluster: items and histograms go through memory, the passes are separated by cluster barriers.
template <int STEPS>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kSortThreads)
    embedding_sort_cluster_kernel(const int64_t* ids, int64_t tokens, int64_t rows, int64_t padding, int passes, int* keys, int* positions,
                                  int* other_keys, int* other_positions, int* histogram, int* error_flag) {
  grid_dependency_wait();
  __shared__ SortShared s;
  int key[STEPS], position[STEPS], digit[STEPS], rank[STEPS];
  load_items(key, position, ids, nullptr, nullptr, tokens, rows, padding, error_flag);
  for (int pass = 0; pass < passes; ++pass) {
    const bool to_first = (passes - 1 - pass) % 2 == 0;
    int* to_keys = to_first ? keys : other_keys;
    int* to_positions = to_first ? positions : other_positions;
#pragma unroll
    for (int k = 0; k < STEPS; ++k) digit[k] = key[k] < 0 ? -1 : (key[k] >> (pass * kRadixBits)) & (kRadix - 1);
    count_digits(s, digit, rank);
    const int total = sum_over_warps(s);
    if (threadIdx.x < kRadix) histogram[blockIdx.x * kRadix + threadIdx.x] = total;
    __threadfence();
    cluster_barrier();
    place_digits(s, histogram, kCluster, blockIdx.x);
    hand_out(s, digit, rank, [&](int k, int at) {
      to_keys[at] = key[k];
      to_positions[at] = position[k];
    });
    __threadfence();
    cluster_barrier();                  // also: nobody counts the next digit before all have read this one's histograms
    if (pass + 1 < passes) load_items(key, position, ids, to_keys, to_positions, tokens, rows, padding, error_flag);
  }
}

template <int STEPS>
__global__ void __launch_bounds__(kSortThreads) embedding_sort_scatter_kernel(const int64_t* ids, const int* src_keys, const int* src_positions,
                                                                              int64_t tokens, int64_t rows, int64_t padding, int shift,
                                                                              const int* histogram, int* keys, int* positions, int* error_flag) {
  grid_dependency_wait();
  __shared__ SortShared s;
  int key[STEPS], position[STEPS], digit[STEPS], rank[STEPS];
  load_items(key, position, ids, src_keys, src_positions, tokens, rows, padding, error_flag);
#pragma unroll
  for (int k = 0; k < STEPS; ++k) digit[k] = key[k] < 0 ? -1 : (key[k] >> shift) & (kRadix - 1);
  count_digits(s, digit, rank);
  sum_over_warps(s);
  place_digits(s, histogram, gridDim.x, blockIdx.x);
  hand_out(s, digit, rank, [&](int k, int at) {
    keys[at] = key[k];
    positions[at] = position[k];
  });
}

// ---- gradient -------------------------------------------------------------------------------
struct GradientArgs {
  const void* dy;
  int64_t ld;               // elements between the rows of dy
  void* out;
  const int* keys;          // sorted
  const int* positions;
  int* starts;              // [rows + 1]: first sorted token of every row
  float* pieces;            // [ceil(tokens / kPiece)][2][width]: sums of the pieces of long runs
  int64_t tokens, rows, width;
  float scale;
  int log_lanes;            // 2^log_lanes threads per row, up to 256: a block takes 256 / that rows (or pieces) side by side
  __host__ __device__ int lanes() const { return 1 << log_lanes; }
  __host__ __device__ int side_by_side() const { return 256 >> log_lanes; }
  __device__ int lane() const { return threadIdx.x & (lanes() - 1); }
  __device__ int line() const { return threadIdx.x >> log_lanes; }
};

__device__ __forceinline__ int lower_bound(const int* keys, int count, int key) {
  int low = 0;
  while (count > 0) {
    const int half = count / 2;
    if (keys[low + half] < key) {
      low += half + 1;
      count -= half + 1;
    } else {
      count = half;
    }
  }
  return low;
}

// One thread's columns: 8 (VECTOR) or 1.
template <typename T, bool VECTOR, int N = VECTOR ? 8 : 1>
__device__ __forceinline__ void load_columns(float (&x)[N], const T* p) {
  if constexpr (VECTOR) load8<T>(x, p);
  else x[0] = to_float<T>(*p);
}

// sum += dy[positions[i]] for i in [first, last), in order; eight rows in flight.
template <typename T, bool VECTOR, int N = VECTOR ? 8 : 1>
__device__ __forceinline__ void add_rows(float (&sum)[N], const GradientArgs& a, int first, int last, int64_t column) {
  const T* dy = static_cast<const T*>(a.dy) + column;
  int i = first;
  for (; i + 8 <= last; i += 8) {
    float x[8][N];
#pragma unroll
    for (int u = 0; u < 8; ++u) load_columns<T, VECTOR>(x[u], dy + a.positions[i + u] * a.ld);
#pragma unroll
    for (int u = 0; u < 8; ++u)
#pragma unroll
      for (int e = 0; e < N; ++e) sum[e] += x[u][e];
  }
  for (; i < last; ++i) {
    float x[N];
    load_columns<T, VECTOR>(x, dy + a.positions[i] * a.ld);
#pragma unroll
    for (int e = 0; e < N; ++e) sum[e] += x[e];
  }
}

// Blocks [0, start_blocks): the rows' first tokens by search. The others: pieces (256 / lanes each) x blocks of columns. A piece
// holds parts of at most two long runs: the one that reaches in from before or fills it, and the one that reaches out.
template <typename T, bool VECTOR>
__global__ void __launch_bounds__(256) embedding_runs_kernel(GradientArgs a, int start_blocks, int column_blocks) {
  grid_dependency_wait();
  constexpr int N = VECTOR ? 8 : 1;
  const int tokens = static_cast<int>(a.tokens);
  if (static_cast<int>(blockIdx.x) < start_blocks) {
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (row <= a.rows) a.starts[row] = lower_bound(a.keys, tokens, static_cast<int>(row));
    return;
  }
  const int block = blockIdx.x - start_blocks, piece = block / column_blocks * a.side_by_side() + a.line();
  const int64_t column = (static_cast<int64_t>(block % column_blocks) * a.lanes() + a.lane()) * N;
  const int begin = piece * kPiece, end = min(tokens, begin + kPiece);
  if (begin >= tokens) return;
  const int head = a.keys[begin], tail = a.keys[end - 1];
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const int key = which ? tail : head;
    if (key >= a.rows || (which && tail == head)) continue;
    // a run that neither reaches in nor reaches out is not a long one
    const bool reaches_in = !which && begin > 0 && a.keys[begin - 1] == key;
    const bool reaches_out = key == tail && end < tokens && a.keys[end] == key;
    if (!reaches_in && !reaches_out) continue;
    const int first = lower_bound(a.keys, tokens, key), last = lower_bound(a.keys, tokens, key + 1);
    if (last - first <= kPiece || column >= a.width) continue;
    float sum[N] = {};
    add_rows<T, VECTOR>(sum, a, max(first, begin), min(last, end), column);
    float* dst = a.pieces + (static_cast<int64_t>(piece) * 2 + which) * a.width + column;
#pragma unroll
    for (int e = 0; e < N; ++e) dst[e] = sum[e];
  }
}

// Every row of the table, every column: zeros, or the sum of the row's run. A block takes kRowsPerBlock rows so that the
// (dependent) load of where their runs start is paid once: 158 us instead of 204 with a row per block, 16384 tokens on
// 49152 x 4096 (940 MB: 143 us at the rate of a plain copy); the whole gradient takes 178 us, sort and runs included.
constexpr int kRowsPerBlock = 8;
template <typename T, typename W, bool VECTOR, bool WIDE>
__global__ void __launch_bounds__(256) embedding_gradient_kernel(GradientArgs a) {
  grid_dependency_wait();
  if constexpr (WIDE) a.log_lanes = 8;
  constexpr int N = VECTOR ? 8 : 1;
  const int64_t column = (static_cast<int64_t>(blockIdx.y) * a.lanes() + a.lane()) * N;
  if (column >= a.width) return;
  W* out = static_cast<W*>(a.out) + column;
  // rows a grid's width apart: frequent tokens tend to be neighbours and should not meet in one block
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * a.side_by_side() + a.line();
  const int64_t row_step = static_cast<int64_t>(gridDim.x) * a.side_by_side();
  int starts[kRowsPerBlock], ends[kRowsPerBlock];
#pragma unroll
  for (int r = 0; r < kRowsPerBlock; ++r) {
    const int64_t row = row0 + r * row_step;
    starts[r] = row < a.rows ? a.starts[row] : 0;
    ends[r] = row < a.rows ? a.starts[row + 1] : 0;
  }
#pragma unroll
  for (int r = 0; r < kRowsPerBlock; ++r) {
    const int first = starts[r], last = ends[r];
    const int64_t row = row0 + r * row_step;
    if (row >= a.rows) break;
    float sum[N] = {};
    if (last - first <= kPiece) {
      add_rows<T, VECTOR>(sum, a, first, last, column);
    } else {
#pragma unroll 4
      for (int piece = first / kPiece; piece * kPiece < last; ++piece) {
        // the run fills the piece's first place unless it begins inside the piece, behind another run
        const int which = first > piece * kPiece ? 1 : 0;
        const float* src = a.pieces + (static_cast<int64_t>(piece) * 2 + which) * a.width + column;
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] += src[e];
      }
    }
#pragma unroll
    for (int e = 0; e < N; ++e) sum[e] *= a.scale;
    if constexpr (VECTOR) store8(out + row * a.width, sum);
    else out[row * a.width] = from_float<W>(sum[0]);
  }
}

bool known(int dtype) { return dtype == CT_F32 || dtype == CT_BF16 || dtype == CT_F16; }
bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// fp32 results leave in 32-byte stores, 16-bit ones in 16-byte stores
bool stores_aligned(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % (8 * dtype_size(dtype)) == 0; }
int64_t padded(int64_t bytes) { return (bytes + 255) / 256 * 256; }
int64_t sort_blocks(int64_t tokens) { return tokens <= kClusterItems ? kCluster : (tokens + kManyItems - 1) / kManyItems; }
int64_t piece_count(int64_t tokens) { return (tokens + kPiece - 1) / kPiece; }

template <typename F> int by_type(int dtype, F f) {
  if (dtype == CT_F32) return f(float{});
  if (dtype == CT_BF16) return f(__nv_bfloat16{});
  return f(__half{});
}

int bits_of(int64_t value) {
  int bits = 1;
  while (value >> bits) ++bits;
  return bits;
}

// keys / positions end up in the first of the two pairs of buffers.
int sort_tokens(const int64_t* ids, int64_t tokens, int64_t rows, int64_t padding, int* keys, int* positions, int* other_keys,
                int* other_positions, int* histogram, int* error_flag, cudaStream_t stream) {
  const int bits = bits_of(rows), passes = (bits + kRadixBits - 1) / kRadixBits;
  if (tokens <= kOneBlockItems) {
    launch_dependent(embedding_sort_one_block_kernel, dim3(1), dim3(kSortThreads), 0, stream, ids, static_cast<int>(tokens), rows, padding, bits,
                     keys, positions, error_flag);
    count_launch(false);
    return check_launch("embedding_sort_one_block_kernel");
  }
  if (tokens <= kClusterItems) {
    const auto kernel = tokens <= kClusterItems / 4   ? embedding_sort_cluster_kernel<1>
                        : tokens <= kClusterItems / 2 ? embedding_sort_cluster_kernel<2>
                                                      : embedding_sort_cluster_kernel<4>;
    launch_dependent(kernel, dim3(kCluster), dim3(kSortThreads), 0, stream, ids, tokens, rows, padding, passes, keys, positions, other_keys,
                     other_positions, histogram, error_flag);
    count_launch(false);
    return check_launch("embedding_sort_cluster_kernel");
  }
  const unsigned blocks = static_cast<unsigned>(sort_blocks(tokens));
  const int* from_keys = nullptr;
  const int* from_positions = nullptr;
  for (int pass = 0; pass < passes; ++pass) {
    const bool last_is_first = (passes - 1 - pass) % 2 == 0;
    int* to_keys = last_is_first ? keys : other_keys;
    int* to_positions = last_is_first ? positions : other_positions;
    const int shift = pass * kRadixBits;
    const auto count = embedding_sort_count_kernel<kManySteps>;
    const auto scatter = embedding_sort_scatter_kernel<kManySteps>;
    launch_dependent(count, dim3(blocks), dim3(kSortThreads), 0, stream, ids, from_keys, tokens, rows, padding, shift, histogram, error_flag);
    launch_dependent(scatter, dim3(blocks), dim3(kSortThreads), 0, stream, ids, from_keys, from_positions, tokens, rows, padding, shift, histogram,
                     to_keys, to_positions, error_flag);
    for (int i = 0; i < 2; ++i) count_launch(false);
    from_keys = to_keys;
    from_positions = to_positions;
  }
  return check_launch("embedding_sort");
}

template <typename T, typename W, bool VECTOR> int gradient(GradientArgs a, cudaStream_t stream) {
  a.log_lanes = 0;
  while (a.log_lanes < 8 && a.lanes() * (VECTOR ? 8 : 1) < a.width) ++a.log_lanes;
  const int64_t per_block = a.lanes() * (VECTOR ? 8 : 1), side_by_side = a.side_by_side();
  const int64_t column_blocks = (a.width + per_block - 1) / per_block, start_blocks = (a.rows + 256) / 256;
  if (column_blocks > 65535) return fail(CT_ERR_UNSUPPORTED, "ct_embedding_gradient: width %lld", (long long)a.width);
  const int64_t blocks = start_blocks + (piece_count(a.tokens) + side_by_side - 1) / side_by_side * column_blocks;
  if (blocks > 0x7fffffff) return fail(CT_ERR_UNSUPPORTED, "ct_embedding_gradient: %lld tokens", (long long)a.tokens);
  launch_dependent(embedding_runs_kernel<T, VECTOR>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, a, static_cast<int>(start_blocks),
                   static_cast<int>(column_blocks));
  count_launch(false);
  const int rc = check_launch("embedding_runs_kernel");
  if (rc) return rc;
  const int64_t grid = (a.rows + kRowsPerBlock * side_by_side - 1) / (kRowsPerBlock * side_by_side);
  launch_dependent(a.log_lanes == 8 ? embedding_gradient_kernel<T, W, VECTOR, true> : embedding_gradient_kernel<T, W, VECTOR, false>,
                   dim3(static_cast<unsigned>(grid), static_cast<unsigned>(column_blocks)), dim3(256), 0, stream, a);
  count_launch(false);
  return check_launch("embedding_gradient_kernel");
}

}  // namespace
}  // namespace ct

using namespace ct;

extern "C" int ct_embedding_forward(const int64_t* ids, const void* table, void* out, int64_t tokens, int64_t rows, int64_t width,
                                    float scale, int table_dtype, int out_dtype, void* stream) {
  if (tokens < 0 || rows < 0 || width < 0) return fail(CT_ERR_ARG, "ct_embedding_forward: negative size");
  if (!known(table_dtype) || !known(out_dtype)) return fail(CT_ERR_ARG, "ct_embedding_forward: dtype");
  if (tokens == 0 || width == 0) return CT_OK;
  if (!ids || !out || (rows > 0 && !table)) return fail(CT_ERR_ARG, "ct_embedding_forward: null pointer");
  int* flag = device_error_flag();
  if (!flag) return fail(CT_ERR_CUDA, "cannot allocate the device error flag");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool vector = width % 8 == 0 && aligned(table) && stores_aligned(out, out_dtype);
  const int64_t work = (tokens * (vector ? width / 8 : width) + 255) / 256;
  const unsigned grid = static_cast<unsigned>(work < (1 << 30) ? work : 1 << 30);
  return by_type(table_dtype, [&](auto w) {
    return by_type(out_dtype, [&](auto t) {
      using W = decltype(w);
      using T = decltype(t);
      if (vector)
        embedding_forward_kernel<W, T, true><<<grid, 256, 0, s>>>(ids, static_cast<const W*>(table), static_cast<T*>(out), tokens, rows, width, scale, flag);
      else
        embedding_forward_kernel<W, T, false><<<grid, 256, 0, s>>>(ids, static_cast<const W*>(table), static_cast<T*>(out), tokens, rows, width, scale, flag);
      count_launch(false);
      return check_launch("embedding_forward_kernel");
    });
  });
}

extern "C" int64_t ct_embedding_gradient_workspace(int64_t tokens, int64_t rows, int64_t width) {
  if (tokens < 0 || rows < 0 || width < 0) return 0;
  const int64_t list = padded(tokens * 4);
  const bool many = tokens > kOneBlockItems;
  return (many ? 4 : 2) * list + (many ? padded(sort_blocks(tokens) * kRadix * 4) : 0) + padded((rows + 1) * 4) +
         padded(piece_count(tokens) * 2 * width * 4);
}

extern "C" int ct_embedding_gradient(const void* dy, int64_t ld, const int64_t* ids, void* d_table, int64_t tokens, int64_t rows, int64_t width,
                                     float scale, int64_t padding, int dy_dtype, int table_dtype, void* workspace, void* stream) {
  if (tokens < 0 || rows < 0 || width < 0 || ld < width) return fail(CT_ERR_ARG, "ct_embedding_gradient: sizes");
  if (!known(dy_dtype) || !known(table_dtype)) return fail(CT_ERR_ARG, "ct_embedding_gradient: dtype");
  if (rows == 0 || width == 0) return CT_OK;
  if (!d_table || !workspace || (tokens > 0 && (!dy || !ids))) return fail(CT_ERR_ARG, "ct_embedding_gradient: null pointer");
  if (tokens >= (int64_t(1) << 31) - 65536 || rows >= (int64_t(1) << 31) - 1024)
    return fail(CT_ERR_UNSUPPORTED, "ct_embedding_gradient: %lld tokens, %lld rows", (long long)tokens, (long long)rows);
  int* flag = device_error_flag();
  if (!flag) return fail(CT_ERR_CUDA, "cannot allocate the device error flag");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t list = padded(tokens * 4);
  const bool many = tokens > kOneBlockItems;
  char* at = static_cast<char*>(workspace);
  auto take = [&](int64_t bytes) {
    char* p = at;
    at += bytes;
    return p;
  };
  int* keys = reinterpret_cast<int*>(take(list));
  int* positions = reinterpret_cast<int*>(take(list));
  int* other_keys = reinterpret_cast<int*>(take(many ? list : 0));
  int* other_positions = reinterpret_cast<int*>(take(many ? list : 0));
  int* histogram = reinterpret_cast<int*>(take(many ? padded(sort_blocks(tokens) * kRadix * 4) : 0));
  GradientArgs a{dy, ld, d_table, keys, positions, nullptr, nullptr, tokens, rows, width, scale, 0};
  a.starts = reinterpret_cast<int*>(take(padded((rows + 1) * 4)));
  a.pieces = reinterpret_cast<float*>(at);
  if (tokens) {
    const int rc = sort_tokens(ids, tokens, rows, padding, keys, positions, other_keys, other_positions, histogram, flag, s);
    if (rc) return rc;
  }
  const bool vector = width % 8 == 0 && aligned(dy) && stores_aligned(d_table, table_dtype) && ld * dtype_size(dy_dtype) % 16 == 0;
  return by_type(dy_dtype, [&](auto t) {
    return by_type(table_dtype, [&](auto w) {
      using T = decltype(t);
      using W = decltype(w);
      return vector ? gradient<T, W, true>(a, s) : gradient<T, W, false>(a, s);
    });
  });
}
