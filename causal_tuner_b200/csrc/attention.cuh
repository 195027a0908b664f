// Document attention: the description of one call, shared by the shape-generic kernels (attention.cu) and the
// tensor-core kernels (attention_tc.cu).
#pragma once

#include <atomic>

#include "common.cuh"

namespace ct {

// The dynamic shared memory a kernel may use is raised once per device (a driver call of a microsecond otherwise).
struct DynamicSmem {
  std::atomic<uint64_t> done{0};
  int set(const char* name, const void* kernel, int bytes) {
    int device = 0;
    cudaError_t err = cudaGetDevice(&device);
    const uint64_t bit = 1ull << (device & 63);
    if (err == cudaSuccess && (done.load(std::memory_order_relaxed) & bit)) return CT_OK;
    if (err == cudaSuccess) err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (err != cudaSuccess) return fail(CT_ERR_CUDA, "%s: %s", name, cudaGetErrorString(err));
    done.fetch_or(bit, std::memory_order_relaxed);
    return CT_OK;
  }
};

// A plan record: one tile of one document. `start` is the document's first token in the flattened batch, `length`
// its token count, `a` and `b` depend on the section (include/ct_b200.h).
struct PlanRecord {
  int start, length, a, b;
};

enum PlanSection { kPlanForward, kPlanQuery, kPlanKeys, kPlanReduce, kPlanTiles, kPlanGaps, kPlanSections };

struct HeadsView {          // [tokens, heads, head_dim], innermost stride 1
  const void* data;
  int64_t token_stride, head_stride;
};

struct AttentionArgs {
  HeadsView q, k, v;
  void* out;                // [tokens, heads, head_dim] contiguous
  float* lse;               // [tokens, heads]: log2 of the sum over the row's keys of exp(scaled score)
  const void* dy;           // backward: [tokens, heads, head_dim] contiguous
  float* delta;             // backward: [tokens, heads] workspace, sum over the channels of dy * out
  void* dq;                 // contiguous, as out
  void* dk;                 // [tokens, kv_heads, head_dim] contiguous
  void* dv;
  float* partials;          // backward workspace behind delta
  const PlanRecord* plan;   // device
  int64_t first[kPlanSections], count[kPlanSections];
  int64_t tokens;
  int heads, kv_heads, head_dim;
  float scale;
  int dtype;
};

inline const PlanRecord* section(const AttentionArgs& a, PlanSection s) { return a.plan + a.first[s]; }

// Heads of one group that share a 128-row tile of the tensor-core kernels: the largest power of two (at most 128)
// that divides the group, so that a tile is 128 / packed tokens x packed heads.
__host__ __device__ inline int packed_heads(int heads, int kv_heads) {
  const int group = heads / kv_heads;
  int packed = 1;
  while (packed < 128 && group % (2 * packed) == 0) packed *= 2;
  return packed;
}

bool attention_tc_supported(const AttentionArgs& a);
int attention_tc_forward(const AttentionArgs& a, cudaStream_t stream);
int64_t attention_tc_workspace(int64_t key_slots, int kv_heads, int head_dim);
int attention_tc_backward(const AttentionArgs& a, cudaStream_t stream);

}  // namespace ct
