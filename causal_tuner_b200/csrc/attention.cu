// Document attention, shape-generic kernels, and the C entry points.
//
// Token t of a document attends to the document's tokens up to itself:
//   S = scale * q k^T,  P = softmax over the allowed keys,  y = P v;
//   backward, P recomputed from q, k and the row's log-sum: delta = sum(dy * y), dv = P^T dy,
//   dS = P * (dy v^T - delta), dq = scale * dS k, dk = scale * dS^T q.
//
// These kernels take every dtype, stride and head_dim up to 128 on fp32 FMA units: 64 x 64 tiles of scores, a 4 x 4
// register tile per thread, operands in padded shared memory. They carry the fp32 decoder and operands that TMA cannot
// fetch; bf16 / fp16 operands go to attention_tc.cu. Sums have a fixed order: dk and dv of heads that share a key head
// are written per head in fp32 and added head by head. Probabilities and dS stay in fp32.
// Measured on the tiny fp32 decoder (2 x 512 tokens, 4 heads of 64 on one, documents of 32 to 256): forward 23 us, query
// gradients 30, key gradients 36, sum of heads 10, delta 2; bound by the latency of the few tiles of each block (a tile of
// 64 x 64 scores takes 6 us), the call by the host (170 us).
#include "attention.cuh"

namespace ct {
namespace {

constexpr int TILE = 64, THREADS = 256, PITCH_S = TILE + 4;
constexpr float kLog2e = 1.4426950408889634f;

// Four neighbouring elements as fp32 (p is aligned to four elements).
template <typename T> __device__ __forceinline__ float4 load4(const T* p) {
  struct alignas(4 * sizeof(T)) Four { T v[4]; };
  const Four f = *reinterpret_cast<const Four*>(p);
  return make_float4(to_float<T>(f.v[0]), to_float<T>(f.v[1]), to_float<T>(f.v[2]), to_float<T>(f.v[3]));
}

// Rows [row0, row0 + 64) of one head of one document into shared memory as fp32; rows at or past `length` and
// channels at or past `dim` are zeros, whatever memory holds there.
template <typename T, int HD>
__device__ __forceinline__ void load_tile(float* dst, const T* base, int64_t token_stride, int row0, int length, int dim) {
  if (dim % 4 == 0 && token_stride % 4 == 0 && reinterpret_cast<uintptr_t>(base) % (4 * sizeof(T)) == 0) {
#pragma unroll
    for (int i = threadIdx.x; i < TILE * HD / 4; i += THREADS) {
      const int r = i / (HD / 4), c = 4 * (i % (HD / 4));
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row0 + r < length && c < dim) v = load4<T>(base + (row0 + r) * token_stride + c);
      *reinterpret_cast<float4*>(dst + r * (HD + 4) + c) = v;
    }
    return;
  }
  for (int i = threadIdx.x; i < TILE * HD; i += THREADS) {
    const int r = i / HD, c = i % HD;
    float v = 0.0f;
    if (row0 + r < length && c < dim) v = to_float<T>(base[(row0 + r) * token_stride + c]);
    dst[r * (HD + 4) + c] = v;
  }
}

// A thread's 4 x 4 part of a 64 x 64 tile: rows 4 ty + i, columns tx + 16 j.
// acc[i][j] = sum over channels of a[4 ty + i] . b[tx + 16 j]
template <int HD>
__device__ __forceinline__ void tile_dot(float (&acc)[4][4], const float* a, const float* b, int ty, int tx) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
#pragma unroll 4
  for (int c = 0; c < HD; c += 4) {
    float4 x[4], y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const float4*>(a + (4 * ty + i) * (HD + 4) + c);
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const float4*>(b + (tx + 16 * j) * (HD + 4) + c);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        acc[i][j] += x[i].x * y[j].x + x[i].y * y[j].y + x[i].z * y[j].z + x[i].w * y[j].w;
  }
}

// acc[i][g] += sum over n of w(4 ty + i, n) * b[n][4 tx + 64 g ..]; w is read at w[row * PITCH_S + n], or with
// TRANSPOSED at w[n * PITCH_S + row].
template <int HD, bool TRANSPOSED>
__device__ __forceinline__ void tile_product(float4 (&acc)[4][HD / 64], const float* w, const float* b, int ty, int tx) {
#pragma unroll 2
  for (int n = 0; n < TILE; n += 4) {
    float x[4][4];                                    // [n][i]
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float4 v = *reinterpret_cast<const float4*>(TRANSPOSED ? w + (n + u) * PITCH_S + 4 * ty : w + (4 * ty + u) * PITCH_S + n);
      if constexpr (TRANSPOSED) {
        x[u][0] = v.x; x[u][1] = v.y; x[u][2] = v.z; x[u][3] = v.w;
      } else {
        x[0][u] = v.x; x[1][u] = v.y; x[2][u] = v.z; x[3][u] = v.w;
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int g = 0; g < HD / 64; ++g) {
        const float4 y = *reinterpret_cast<const float4*>(b + (n + u) * (HD + 4) + 4 * tx + 64 * g);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[i][g].x += x[u][i] * y.x; acc[i][g].y += x[u][i] * y.y; acc[i][g].z += x[u][i] * y.z; acc[i][g].w += x[u][i] * y.w;
        }
      }
  }
}

template <typename T, int HD>
__device__ __forceinline__ void store_rows(T* base, int64_t token_stride, const float4 (&acc)[4][HD / 64],
                                           const float (&factor)[4], int row0, int length, int dim, int ty, int tx) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = row0 + 4 * ty + i;
    if (row >= length) continue;
    T* dst = base + row * token_stride;
#pragma unroll
    for (int g = 0; g < HD / 64; ++g) {
      const float v[4] = {acc[i][g].x, acc[i][g].y, acc[i][g].z, acc[i][g].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = 4 * tx + 64 * g + e;
        if (c < dim) dst[c] = from_float<T>(v[e] * factor[i]);
      }
    }
  }
}

template <int HD> __device__ __forceinline__ void clear(float4 (&acc)[4][HD / 64]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int g = 0; g < HD / 64; ++g) acc[i][g] = make_float4(0.f, 0.f, 0.f, 0.f);
}

// A plan tile holds 128 tokens: two blocks of 64 rows each. Returns false for a block past the document's end.
__device__ __forceinline__ bool locate(const PlanRecord* tiles, int block, PlanRecord& r, int& row0) {
  r = tiles[block >> 1];
  row0 = r.a + TILE * (block & 1);
  return row0 < r.length;
}

template <typename T, int HD>
__global__ void __launch_bounds__(THREADS) attention_forward_kernel(const PlanRecord* tiles, AttentionArgs a) {
  extern __shared__ float smem[];
  float* qs = smem;
  float* ks = qs + TILE * (HD + 4);
  float* vs = ks + TILE * (HD + 4);
  float* ps = vs + TILE * (HD + 4);
  PlanRecord r;
  int row0;
  if (!locate(tiles, blockIdx.x, r, row0)) return;
  const int head = blockIdx.y, shared = head / (a.heads / a.kv_heads), dim = a.head_dim;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const int64_t start = r.start;
  const T* q = static_cast<const T*>(a.q.data) + start * a.q.token_stride + head * a.q.head_stride;
  const T* k = static_cast<const T*>(a.k.data) + start * a.k.token_stride + shared * a.k.head_stride;
  const T* v = static_cast<const T*>(a.v.data) + start * a.v.token_stride + shared * a.v.head_stride;
  load_tile<T, HD>(qs, q, a.q.token_stride, row0, r.length, dim);
  const float scale = a.scale * kLog2e;       // scores in units of log2
  float top[4], sum[4];
  float4 acc[4][HD / 64];
  clear<HD>(acc);
#pragma unroll
  for (int i = 0; i < 4; ++i) { top[i] = -INFINITY; sum[i] = 0.0f; }
  const int end = min(r.length, row0 + TILE);
  for (int key0 = 0; key0 < end; key0 += TILE) {
    __syncthreads();
    load_tile<T, HD>(ks, k, a.k.token_stride, key0, r.length, dim);
    load_tile<T, HD>(vs, v, a.v.token_stride, key0, r.length, dim);
    __syncthreads();
    float s[4][4];
    tile_dot<HD>(s, qs, ks, ty, tx);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = row0 + 4 * ty + i;
      float best = top[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = key0 + tx + 16 * j;
        s[i][j] = key <= row && key < r.length ? s[i][j] * scale : -INFINITY;
        best = fmaxf(best, s[i][j]);
      }
#pragma unroll
      for (int step = 8; step; step >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, step));
      // key 0 is allowed for every row, so `best` is a score from the first tile on
      const float factor = exp2f(top[i] - best);
      top[i] = best;
      float part = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = s[i][j] == -INFINITY ? 0.0f : exp2f(s[i][j] - best);
        part += p;
        ps[(4 * ty + i) * PITCH_S + tx + 16 * j] = p;
      }
#pragma unroll
      for (int step = 8; step; step >>= 1) part += __shfl_xor_sync(0xffffffffu, part, step);
      sum[i] = sum[i] * factor + part;
#pragma unroll
      for (int g = 0; g < HD / 64; ++g) {
        acc[i][g].x *= factor; acc[i][g].y *= factor; acc[i][g].z *= factor; acc[i][g].w *= factor;
      }
    }
    __syncthreads();
    tile_product<HD, false>(acc, ps, vs, ty, tx);
  }
  float factor[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    factor[i] = 1.0f / sum[i];
    const int row = row0 + 4 * ty + i;
    if (tx == 0 && row < r.length && a.lse) a.lse[(start + row) * a.heads + head] = top[i] + log2f(sum[i]);
  }
  T* out = static_cast<T*>(a.out) + (start * a.heads + head) * dim;
  store_rows<T, HD>(out, static_cast<int64_t>(a.heads) * dim, acc, factor, row0, r.length, dim, ty, tx);
}

// The probabilities of one 64 x 64 tile and dS = P * (dP - delta), from s = q k^T and dp = dy v^T. The document's first query
// sees one key, so that P = 1, y = v and its dS is 0 (as a product with 0: a NaN stays one), not two sums' rounding errors.
__device__ __forceinline__ void tile_slopes(float (&s)[4][4], float (&dp)[4][4], const float (&lse)[4], const float (&delta)[4],
                                            float scale, int row0, int key0, int length, int ty, int tx) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = row0 + 4 * ty + i;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int key = key0 + tx + 16 * j;
      const bool allowed = key <= row && row < length;
      s[i][j] = allowed ? exp2f(s[i][j] * scale - lse[i]) : 0.0f;
      dp[i][j] = allowed ? (row ? s[i][j] : 0.0f) * (dp[i][j] - delta[i]) : 0.0f;
    }
  }
}

template <typename T, int HD>
__global__ void __launch_bounds__(THREADS) attention_query_gradient_kernel(const PlanRecord* tiles, AttentionArgs a) {
  extern __shared__ float smem[];
  float* qs = smem;
  float* gs = qs + TILE * (HD + 4);
  float* ks = gs + TILE * (HD + 4);
  float* vs = ks + TILE * (HD + 4);
  float* ds = vs + TILE * (HD + 4);
  PlanRecord r;
  int row0;
  if (!locate(tiles, blockIdx.x, r, row0)) return;
  const int head = blockIdx.y, shared = head / (a.heads / a.kv_heads), dim = a.head_dim;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const int64_t start = r.start, row_stride = static_cast<int64_t>(a.heads) * dim;
  const T* k = static_cast<const T*>(a.k.data) + start * a.k.token_stride + shared * a.k.head_stride;
  const T* v = static_cast<const T*>(a.v.data) + start * a.v.token_stride + shared * a.v.head_stride;
  load_tile<T, HD>(qs, static_cast<const T*>(a.q.data) + start * a.q.token_stride + head * a.q.head_stride,
                   a.q.token_stride, row0, r.length, dim);
  load_tile<T, HD>(gs, static_cast<const T*>(a.dy) + start * row_stride + head * dim, row_stride, row0, r.length, dim);
  float lse[4], delta[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = row0 + 4 * ty + i;
    lse[i] = row < r.length ? a.lse[(start + row) * a.heads + head] : 0.0f;
    delta[i] = row < r.length ? a.delta[(start + row) * a.heads + head] : 0.0f;
  }
  float4 acc[4][HD / 64];
  clear<HD>(acc);
  const int end = min(r.length, row0 + TILE);
  for (int key0 = 0; key0 < end; key0 += TILE) {
    __syncthreads();
    load_tile<T, HD>(ks, k, a.k.token_stride, key0, r.length, dim);
    load_tile<T, HD>(vs, v, a.v.token_stride, key0, r.length, dim);
    __syncthreads();
    float s[4][4], dp[4][4];
    tile_dot<HD>(s, qs, ks, ty, tx);
    tile_dot<HD>(dp, gs, vs, ty, tx);
    tile_slopes(s, dp, lse, delta, a.scale * kLog2e, row0, key0, r.length, ty, tx);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) ds[(4 * ty + i) * PITCH_S + tx + 16 * j] = dp[i][j];
    __syncthreads();
    tile_product<HD, false>(acc, ds, ks, ty, tx);
  }
  const float factor[4] = {a.scale, a.scale, a.scale, a.scale};
  store_rows<T, HD>(static_cast<T*>(a.dq) + start * row_stride + head * dim, row_stride, acc, factor, row0, r.length, dim, ty, tx);
}

// One block per 64 keys and QUERY head. Where heads share a key head (PARTIAL) the block writes its share in fp32 to
// partials[0 = dk, 1 = dv][token][head][dim].
template <typename T, int HD, bool PARTIAL>
__global__ void __launch_bounds__(THREADS) attention_key_gradient_kernel(const PlanRecord* tiles, AttentionArgs a) {
  extern __shared__ float smem[];
  float* qs = smem;
  float* gs = qs + TILE * (HD + 4);
  float* ks = gs + TILE * (HD + 4);
  float* vs = ks + TILE * (HD + 4);
  float* ps = vs + TILE * (HD + 4);
  float* ds = ps + TILE * PITCH_S;
  PlanRecord r;
  int key0;
  if (!locate(tiles, blockIdx.x, r, key0)) return;
  const int head = blockIdx.y, shared = head / (a.heads / a.kv_heads), dim = a.head_dim;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const int64_t start = r.start, row_stride = static_cast<int64_t>(a.heads) * dim;
  const T* q = static_cast<const T*>(a.q.data) + start * a.q.token_stride + head * a.q.head_stride;
  const T* dy = static_cast<const T*>(a.dy) + start * row_stride + head * dim;
  load_tile<T, HD>(ks, static_cast<const T*>(a.k.data) + start * a.k.token_stride + shared * a.k.head_stride,
                   a.k.token_stride, key0, r.length, dim);
  load_tile<T, HD>(vs, static_cast<const T*>(a.v.data) + start * a.v.token_stride + shared * a.v.head_stride,
                   a.v.token_stride, key0, r.length, dim);
  float4 dk[4][HD / 64], dv[4][HD / 64];
  clear<HD>(dk);
  clear<HD>(dv);
  for (int row0 = key0; row0 < r.length; row0 += TILE) {
    __syncthreads();
    load_tile<T, HD>(qs, q, a.q.token_stride, row0, r.length, dim);
    load_tile<T, HD>(gs, dy, row_stride, row0, r.length, dim);
    float lse[4], delta[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = row0 + 4 * ty + i;
      lse[i] = row < r.length ? a.lse[(start + row) * a.heads + head] : 0.0f;
      delta[i] = row < r.length ? a.delta[(start + row) * a.heads + head] : 0.0f;
    }
    __syncthreads();
    float s[4][4], dp[4][4];
    tile_dot<HD>(s, qs, ks, ty, tx);
    tile_dot<HD>(dp, gs, vs, ty, tx);
    tile_slopes(s, dp, lse, delta, a.scale * kLog2e, row0, key0, r.length, ty, tx);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        ps[(4 * ty + i) * PITCH_S + tx + 16 * j] = s[i][j];
        ds[(4 * ty + i) * PITCH_S + tx + 16 * j] = dp[i][j];
      }
    __syncthreads();
    tile_product<HD, true>(dv, ps, gs, ty, tx);
    tile_product<HD, true>(dk, ds, qs, ty, tx);
  }
  const float key_factor[4] = {a.scale, a.scale, a.scale, a.scale}, value_factor[4] = {1.f, 1.f, 1.f, 1.f};
  if constexpr (PARTIAL) {
    float* base = a.partials + start * row_stride + head * dim;
    store_rows<float, HD>(base, row_stride, dk, key_factor, key0, r.length, dim, ty, tx);
    store_rows<float, HD>(base + a.tokens * row_stride, row_stride, dv, value_factor, key0, r.length, dim, ty, tx);
  } else {
    store_rows<T, HD>(static_cast<T*>(a.dk) + start * row_stride + head * dim, row_stride, dk, key_factor, key0, r.length, dim, ty, tx);
    store_rows<T, HD>(static_cast<T*>(a.dv) + start * row_stride + head * dim, row_stride, dv, value_factor, key0, r.length, dim, ty, tx);
  }
}

// dk / dv of 64 tokens of one key head: the group's partial rows added head by head.
template <typename T>
__global__ void attention_sum_heads_kernel(const PlanRecord* tiles, AttentionArgs a) {
  PlanRecord r;
  int row0;
  if (!locate(tiles, blockIdx.x, r, row0)) return;
  const int group = a.heads / a.kv_heads, dim = a.head_dim, shared = blockIdx.y;
  const int rows = min(TILE, r.length - row0);
  const int64_t row_stride = static_cast<int64_t>(a.heads) * dim;
  const float* src = a.partials + blockIdx.z * a.tokens * row_stride;
  T* dst = static_cast<T*>(blockIdx.z ? a.dv : a.dk);
  for (int i = threadIdx.x; i < rows * dim; i += blockDim.x) {
    const int64_t token = static_cast<int64_t>(r.start) + row0 + i / dim;
    const int c = i % dim;
    float sum = 0.0f;
    for (int h = 0; h < group; ++h) sum += src[token * row_stride + (static_cast<int64_t>(shared) * group + h) * dim + c];
    dst[(token * a.kv_heads + shared) * dim + c] = from_float<T>(sum);
  }
}

// delta[row] = sum over the channels of dy * y, rows = (token, head) of the contiguous matrices. A row is shared by LANES
// lanes with 16 bytes each (VECTOR: rows are whole numbers of 16-byte pieces), or by a warp, element by element.
template <typename T, bool VECTOR>
__global__ void __launch_bounds__(256) attention_delta_kernel(const T* dy, const T* y, float* delta, int64_t rows, int dim, int lanes) {
  // (inside the query-gradient kernel, by its two idle warps, this cost more than the 48 us of its own at 16384 x 32 rows:
  // 409 against 281 us for the packed 7B batch)
  constexpr int N = 16 / sizeof(T);
  const int64_t thread = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t row = thread / lanes;
  const int lane = static_cast<int>(thread % lanes);
  float sum = 0.0f;
  if (row < rows) {
    if constexpr (VECTOR) {
      if (lane * N < dim) {
        const uint4 a = *reinterpret_cast<const uint4*>(dy + row * dim + lane * N), b = *reinterpret_cast<const uint4*>(y + row * dim + lane * N);
        const T* x = reinterpret_cast<const T*>(&a);
        const T* z = reinterpret_cast<const T*>(&b);
#pragma unroll
        for (int i = 0; i < N; ++i) sum += to_float<T>(x[i]) * to_float<T>(z[i]);
      }
    } else {
      for (int c = lane; c < dim; c += lanes) sum += to_float<T>(dy[row * dim + c]) * to_float<T>(y[row * dim + c]);
    }
  }
  for (int step = lanes / 2; step; step >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, step);
  if (lane == 0 && row < rows) delta[row] = sum;
}

// Zeros for the tokens between documents: up to three matrices of `bytes[i]` per token, a multiple of 2.
struct GapTargets {
  void* data[3];
  int64_t bytes[3];
};
__global__ void attention_clear_gaps_kernel(const PlanRecord* gaps, GapTargets t) {
  const PlanRecord r = gaps[blockIdx.x];
  char* base = static_cast<char*>(t.data[blockIdx.y]) + r.start * t.bytes[blockIdx.y];
  const int64_t total = r.length * t.bytes[blockIdx.y];
  for (int64_t i = 2 * threadIdx.x; i < total; i += 2 * blockDim.x) *reinterpret_cast<uint16_t*>(base + i) = 0;
}

int clear_gaps(const AttentionArgs& a, const GapTargets& t, int targets, cudaStream_t stream) {
  if (!a.count[kPlanGaps]) return CT_OK;
  attention_clear_gaps_kernel<<<dim3(a.count[kPlanGaps], targets), 256, 0, stream>>>(section(a, kPlanGaps), t);
  count_launch(false);
  return check_launch("attention_clear_gaps_kernel");
}

template <auto Kernel, typename... Args>
int launch(const char* name, dim3 grid, int smem, cudaStream_t stream, Args... args) {
  static DynamicSmem allowed;
  const int rc = allowed.set(name, reinterpret_cast<const void*>(Kernel), smem);
  if (rc) return rc;
  Kernel<<<grid, THREADS, smem, stream>>>(args...);
  count_launch(false);
  return check_launch(name);
}

template <typename T, int HD> int simt_forward(const AttentionArgs& a, cudaStream_t stream) {
  const int smem = (3 * TILE * (HD + 4) + TILE * PITCH_S) * sizeof(float);
  return launch<attention_forward_kernel<T, HD>>("attention_forward_kernel", dim3(2 * a.count[kPlanTiles], a.heads), smem, stream, section(a, kPlanTiles), a);
}

template <typename T> int delta_pass(const AttentionArgs& a, cudaStream_t stream) {
  const int64_t rows = a.tokens * a.heads;
  const bool vector = a.head_dim * sizeof(T) % 16 == 0 && ((reinterpret_cast<uintptr_t>(a.dy) | reinterpret_cast<uintptr_t>(a.out)) & 15) == 0;
  int lanes = 32;
  while (vector && lanes > 1 && (lanes / 2) * 16 >= a.head_dim * static_cast<int>(sizeof(T))) lanes /= 2;
  const int64_t blocks = (rows * lanes + 255) / 256;
  if (blocks > 0x7fffffff) return fail(CT_ERR_UNSUPPORTED, "ct_attention_backward: %lld rows", (long long)rows);
  const T* dy = static_cast<const T*>(a.dy);
  const T* y = static_cast<const T*>(a.out);
  if (vector) attention_delta_kernel<T, true><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(dy, y, a.delta, rows, a.head_dim, lanes);
  else attention_delta_kernel<T, false><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(dy, y, a.delta, rows, a.head_dim, lanes);
  count_launch(false);
  return check_launch("attention_delta_kernel");
}

template <typename T, int HD> int simt_backward(const AttentionArgs& a, cudaStream_t stream) {
  const dim3 grid(2 * a.count[kPlanTiles], a.heads);
  const PlanRecord* tiles = section(a, kPlanTiles);
  const int query_smem = (4 * TILE * (HD + 4) + TILE * PITCH_S) * sizeof(float);
  const int key_smem = query_smem + TILE * PITCH_S * sizeof(float);
  int rc = launch<attention_query_gradient_kernel<T, HD>>("attention_query_gradient_kernel", grid, query_smem, stream, tiles, a);
  if (rc) return rc;
  if (a.heads == a.kv_heads)
    return launch<attention_key_gradient_kernel<T, HD, false>>("attention_key_gradient_kernel", grid, key_smem, stream, tiles, a);
  rc = launch<attention_key_gradient_kernel<T, HD, true>>("attention_key_gradient_kernel", grid, key_smem, stream, tiles, a);
  if (rc) return rc;
  return launch<attention_sum_heads_kernel<T>>("attention_sum_heads_kernel", dim3(grid.x, a.kv_heads, 2), 0, stream, tiles, a);
}

template <typename T> int simt_pass(const AttentionArgs& a, bool backward, cudaStream_t stream) {
  if (a.head_dim <= 64) return backward ? simt_backward<T, 64>(a, stream) : simt_forward<T, 64>(a, stream);
  return backward ? simt_backward<T, 128>(a, stream) : simt_forward<T, 128>(a, stream);
}

int simt(const AttentionArgs& a, bool backward, cudaStream_t stream) {
  if (a.dtype == CT_F32) return simt_pass<float>(a, backward, stream);
  if (a.dtype == CT_BF16) return simt_pass<__nv_bfloat16>(a, backward, stream);
  return simt_pass<__half>(a, backward, stream);
}

bool known(int dtype) { return dtype == CT_F32 || dtype == CT_BF16 || dtype == CT_F16; }

// Shared argument checks. Fills everything but the tensors.
int describe(AttentionArgs& a, const char* name, const int32_t* plan, const int64_t* sections, int64_t tokens, int heads,
             int kv_heads, int head_dim, float scale, int dtype) {
  if (tokens < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads || head_dim < 1)
    return fail(CT_ERR_ARG, "%s: sizes (tokens %lld, heads %d, kv_heads %d, head_dim %d)", name, (long long)tokens, heads, kv_heads, head_dim);
  if (!known(dtype)) return fail(CT_ERR_ARG, "%s: dtype", name);
  if (head_dim > 128) return fail(CT_ERR_UNSUPPORTED, "%s: head_dim %d is above 128", name, head_dim);
  if (heads > 65535 || kv_heads > 32767) return fail(CT_ERR_UNSUPPORTED, "%s: %d heads, %d key heads", name, heads, kv_heads);
  if (tokens >= (int64_t(1) << 31) - 256) return fail(CT_ERR_UNSUPPORTED, "%s: %lld tokens", name, (long long)tokens);
  if (!sections) return fail(CT_ERR_ARG, "%s: null sections", name);
  a = AttentionArgs{};
  int64_t used = 0;
  for (int s = 0; s < kPlanSections; ++s) {
    a.first[s] = sections[2 * s];
    a.count[s] = sections[2 * s + 1];
    if (a.first[s] < 0 || a.count[s] < 0 || a.count[s] > 0x3fffffff) return fail(CT_ERR_ARG, "%s: plan section %d", name, s);
    used += a.count[s];
  }
  if (used && !plan) return fail(CT_ERR_ARG, "%s: null plan", name);
  a.plan = reinterpret_cast<const PlanRecord*>(plan);
  a.tokens = tokens;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.head_dim = head_dim;
  a.scale = scale;
  a.dtype = dtype;
  return CT_OK;
}

// The path is the caller's, as ct_attention_path names it (the workspace depends on it).
int check_path(const AttentionArgs& a, const char* name, int path) {
  if (path != CT_PATH_SIMT && path != CT_PATH_TCGEN05) return fail(CT_ERR_ARG, "%s: path %d", name, path);
  if (path == CT_PATH_TCGEN05 && !attention_tc_supported(a))
    return fail(CT_ERR_UNSUPPORTED, "%s: the tensor-core path needs 16-bit types, 16-byte aligned rows, head_dim a multiple of 8 and a scale that is not tiny", name);
  return CT_OK;
}

constexpr int64_t kAlign = 256;
int64_t padded(int64_t bytes) { return (bytes + kAlign - 1) / kAlign * kAlign; }

}  // namespace
}  // namespace ct

using namespace ct;

extern "C" int ct_attention_tile_tokens(int heads, int kv_heads) {
  if (heads < 1 || kv_heads < 1 || heads % kv_heads) return fail(CT_ERR_ARG, "ct_attention_tile_tokens: heads");
  return 128 / packed_heads(heads, kv_heads);
}

extern "C" int ct_attention_forward(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token, int64_t k_head,
                                    const void* v, int64_t v_token, int64_t v_head, void* out, float* lse, const int32_t* plan,
                                    const int64_t* sections, int64_t tokens, int heads, int kv_heads, int head_dim, float scale,
                                    int dtype, int path, void* stream) {
  AttentionArgs a;
  int rc = describe(a, "ct_attention_forward", plan, sections, tokens, heads, kv_heads, head_dim, scale, dtype);
  if (rc || tokens == 0) return rc;
  if (!q || !k || !v || !out) return fail(CT_ERR_ARG, "ct_attention_forward: null pointer");
  a.q = {q, q_token, q_head};
  a.k = {k, k_token, k_head};
  a.v = {v, v_token, v_head};
  a.out = out;
  a.lse = lse;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (path == CT_PATH_AUTO) path = attention_tc_supported(a) ? CT_PATH_TCGEN05 : CT_PATH_SIMT;
  rc = check_path(a, "ct_attention_forward", path);
  if (rc) return rc;
  const int64_t row = static_cast<int64_t>(heads) * head_dim * dtype_size(dtype);
  rc = clear_gaps(a, GapTargets{{out, nullptr, nullptr}, {row, 0, 0}}, 1, s);
  if (rc || !a.count[kPlanTiles]) return rc;
  return path == CT_PATH_TCGEN05 ? attention_tc_forward(a, s) : simt(a, false, s);
}

extern "C" int ct_attention_path(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token, int64_t k_head,
                                 const void* v, int64_t v_token, int64_t v_head, int heads, int kv_heads, int head_dim, float scale, int dtype) {
  if (heads < 1 || kv_heads < 1 || heads % kv_heads || head_dim < 1 || !known(dtype)) return fail(CT_ERR_ARG, "ct_attention_path: sizes");
  AttentionArgs a{};
  a.q = {q, q_token, q_head};
  a.k = {k, k_token, k_head};
  a.v = {v, v_token, v_head};
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.head_dim = head_dim;
  a.scale = scale;
  a.dtype = dtype;
  return attention_tc_supported(a) ? CT_PATH_TCGEN05 : CT_PATH_SIMT;
}

extern "C" int64_t ct_attention_backward_workspace(int64_t tokens, int heads, int kv_heads, int head_dim, int64_t key_slots, int path) {
  if (tokens < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads || head_dim < 1 || key_slots < 0) return 0;
  const int64_t per_head = heads == kv_heads ? 0 : 2 * tokens * heads * head_dim * 4;
  return padded(tokens * heads * 4) + (path == CT_PATH_TCGEN05 ? attention_tc_workspace(key_slots, kv_heads, head_dim) : per_head);
}

extern "C" int ct_attention_backward(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token, int64_t k_head,
                                     const void* v, int64_t v_token, int64_t v_head, const void* out, const float* lse, const void* dy,
                                     void* dq, void* dk, void* dv, const int32_t* plan, const int64_t* sections, int64_t tokens,
                                     int heads, int kv_heads, int head_dim, float scale, int dtype, int path, void* workspace,
                                     void* stream) {
  AttentionArgs a;
  int rc = describe(a, "ct_attention_backward", plan, sections, tokens, heads, kv_heads, head_dim, scale, dtype);
  if (rc || tokens == 0) return rc;
  if (!q || !k || !v || !out || !lse || !dy || !dq || !dk || !dv || !workspace)
    return fail(CT_ERR_ARG, "ct_attention_backward: null pointer");
  a.q = {q, q_token, q_head};
  a.k = {k, k_token, k_head};
  a.v = {v, v_token, v_head};
  a.out = const_cast<void*>(out);
  a.lse = const_cast<float*>(lse);
  a.dy = dy;
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  a.delta = static_cast<float*>(workspace);
  a.partials = reinterpret_cast<float*>(static_cast<char*>(workspace) + padded(tokens * heads * 4));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  rc = check_path(a, "ct_attention_backward", path);
  if (rc) return rc;
  const int64_t row = static_cast<int64_t>(heads) * head_dim * dtype_size(dtype);
  const int64_t shared_row = static_cast<int64_t>(kv_heads) * head_dim * dtype_size(dtype);
  rc = clear_gaps(a, GapTargets{{dq, dk, dv}, {row, shared_row, shared_row}}, 3, s);
  if (rc || !a.count[kPlanTiles]) return rc;
  rc = dtype == CT_F32 ? delta_pass<float>(a, s) : dtype == CT_BF16 ? delta_pass<__nv_bfloat16>(a, s) : delta_pass<__half>(a, s);
  if (rc) return rc;
  return path == CT_PATH_TCGEN05 ? attention_tc_backward(a, s) : simt(a, true, s);
}
