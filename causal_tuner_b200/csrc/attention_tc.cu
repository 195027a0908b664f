// Document attention on the Blackwell tensor cores (tcgen05 + TMEM + TMA), bf16 and fp16, head_dim a multiple of 8 up
// to 128.
//
// Rows of a tile. The query heads of a group read the same keys, so a 128-row tile holds 128 / P tokens x P heads (P =
// the largest power of two that divides the group, packed_heads): with 32 heads on one key head a tile is 4 tokens, a
// 64-token document fills 16 tiles instead of half-filling 32, and both 128-row stages of a CTA end on the same key
// tile. One TMA box {64 channels, P heads, 128 / P tokens} brings such a tile in the 128-byte swizzle the tensor core
// reads; K and V tiles are boxes of 128 keys, each serving as a K-major operand (scores) and as an MN-major one.
//
// head_dim below 64 or 128 is padded by the copies themselves (channels past the tensor are zeros).
// Rows of another document that a tile takes in: scores are dropped by the key limit of each row, and operand rows that
// would be MULTIPLIED by a zero probability are overwritten with zeros in shared memory, so that a NaN in foreign or
// padding rows cannot spread.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>

#include "attention.cuh"
#include "tcgen05.cuh"

namespace ct {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int KEYS = 128;                          // keys per tile
constexpr uint32_t BOX_BYTES = 128 * 128;          // 128 rows x 64 channels

template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ float exp2_approx(float x) {   // special-function unit, relative error about 2^-22
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 lanes per instruction: halves the issue slots of everything between the exponentials.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
// 2^x for x <= 128 on the FMA units, so that the special-function units (16 results per SM and cycle, which is what the
// tensor core's pace asks of them in full) can be relieved of a share. Range reduction by rounding to the nearest integer
// n (Cody and Waite), |x - n| <= 1/2, and a degree-5 polynomial fitted here for the smallest relative error of 2^f on
// [-1/2, 1/2] (7.5e-8; 2.1e-7 in fp32 arithmetic, the accuracy of ex2.approx). Below 2^-125 the result stays 2^-125.
__device__ __forceinline__ float2 exp2_fma(float2 x) {
  x.x = fmaxf(x.x, -125.0f);
  x.y = fmaxf(x.y, -125.0f);
  const float round = 12582912.0f;                  // 1.5 * 2^23: the sum's low mantissa bits are n
  const float2 t = add2(x, make_float2(round, round));
  const float2 f = add2(x, fma2(t, make_float2(-1.0f, -1.0f), make_float2(round, round)));
  float2 r = fma2(f, make_float2(1.3276472454890609e-3f, 1.3276472454890609e-3f), make_float2(9.675540961325169e-3f, 9.675540961325169e-3f));
  r = fma2(r, f, make_float2(0.05550713092088699f, 0.05550713092088699f));
  r = fma2(r, f, make_float2(0.24022120237350464f, 0.24022120237350464f));
  r = fma2(r, f, make_float2(0.6931469440460205f, 0.6931469440460205f));
  r = fma2(r, f, make_float2(1.0000001192092896f, 1.0000001192092896f));
  r.x = __int_as_float(__float_as_int(r.x) + (__float_as_int(t.x) << 23));
  r.y = __int_as_float(__float_as_int(r.y) + (__float_as_int(t.y) << 23));
  return r;
}
__device__ __forceinline__ float2 exp2_pair(float2 x, bool on_fma) {
  return on_fma ? exp2_fma(x) : make_float2(exp2_approx(x.x), exp2_approx(x.y));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Keeps the code behind a rare condition behind a branch (the compiler would rather compute it always and select).
__device__ __forceinline__ void rare() { asm volatile("" ::: "memory"); }

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// D += A . B with A in shared memory (K-major) or in TMEM (packed pairs along k), B in shared memory.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
  umma_bf16(d, a_lo, desc_high(1024), b_lo, b_hi, idesc, accumulate);
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}"
      ::"r"(d), "r"(a_tmem), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Instruction descriptor: fp32 accumulator, both operands T, A K-major, M = 128.
template <typename T> __device__ __forceinline__ constexpr uint32_t operand_desc(bool b_mn, int n) {
  constexpr uint32_t type = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (type << 7) | (type << 10) | (static_cast<uint32_t>(b_mn) << 16) | (static_cast<uint32_t>(n >> 3) << 17) | (8u << 24);
}

__device__ __forceinline__ bool elect_one() {
  uint32_t chosen;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(chosen));
  return chosen != 0;
}
// A value that all lanes hold, in a form that the compiler knows to be uniform.
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ PlanRecord uniform(PlanRecord r) { return {uniform(r.start), uniform(r.length), uniform(r.a), uniform(r.b)}; }

// MMAs of one thread execute in the order of issue; where an accumulator takes the place of an operand in TMEM (S over P,
// S over dS), nothing else orders the two.
// The MMA warp walks its loops as a whole - with uniform control flow descriptors stay in uniform registers, and a chain
// of MMAs costs few instructions each - and one elected lane issues. (With one lane in the loop an MMA took 110 cycles to issue.)
// scores: D[128, 128] = A[128, HD] . B[128, HD]^T, both tiles as 128-row boxes of 64 channels. Always all 128 columns: with
// both operands in shared memory an MMA is bound by reading them, and fewer columns take no less time.
template <typename T, int HD>
__device__ __forceinline__ void product_nt(uint32_t d, uint32_t a, uint32_t b) {
  constexpr uint32_t idesc = operand_desc<T>(false, 128);
  const uint32_t a_lo = desc_low(a, 16), b_lo = desc_low(b, 16);
  if (elect_one()) {
#pragma unroll
    for (int k = 0; k < HD / 16; ++k) {
      const uint32_t offset = ((k / 4) * BOX_BYTES + (k % 4) * 32) >> 4;
      mma_ss(d, a_lo + offset, b_lo + offset, desc_high(1024), idesc, k > 0);
    }
  }
}

// D[128, HD] += A (TMEM) . B, B a 128-row tile read along its rows (MN-major), k steps [FIRST, LAST) of 16 rows. Step k of A
// starts at column k / SPAN * STRIDE + k % SPAN * 8.
template <typename T, int HD, int SPAN, int STRIDE, int FIRST, int LAST>
__device__ __forceinline__ void product_tn(uint32_t d, uint32_t a, uint32_t b, bool accumulate) {
  constexpr uint32_t idesc = operand_desc<T>(true, HD);
  const uint32_t b_lo = desc_low(b, BOX_BYTES);
  if (elect_one()) {
#pragma unroll
    for (int k = FIRST; k < LAST; ++k)
      mma_ts(d, a + k / SPAN * STRIDE + k % SPAN * 8, b_lo + k * (2048 >> 4), desc_high(1024), idesc, accumulate || k > FIRST);
  }
}
__device__ __forceinline__ void commit(uint32_t bar) {
  if (elect_one()) umma_commit(bar);
}

__device__ __forceinline__ void tmem_store_16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_store_32(uint32_t taddr, const uint32_t* r) {
  tmem_store_16(taddr, r);
  tmem_store_16(taddr + 16, r + 16);
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_alloc(uint32_t slot) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(512) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t base) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(512) : "memory");
}

// Zeros over rows [from, to) of a tile of BOXES boxes, by `threads` threads of which this is number `thread`, made
// visible to the tensor core.
template <int BOXES>
__device__ __forceinline__ void clear_rows(uint32_t tile, int from, int to, int thread, int threads) {
  for (int i = thread; i < (to - from) * 8 * BOXES; i += threads) {
    const int row = from + i / (8 * BOXES), piece = i % (8 * BOXES);
    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(tile + (piece / 8) * BOX_BYTES + row * 128 + (piece % 8) * 16), "r"(0)
                 : "memory");
  }
  fence_async_shared();
}

struct AttentionParams {
  CUtensorMap q, k, v, dy;
  const PlanRecord* items;
  void* out;               // forward: y; backward: dq
  void* dk;
  void* dv;
  float* lse;
  float* delta;
  float* partials;
  int heads, kv_heads, dim;
  int packed, tile_tokens; // packed * tile_tokens = 128
  int head_blocks;         // 128-row blocks of heads: heads / packed
  int units;               // records x head blocks (key gradients: x key heads)
  float scale;
  int* error_flag;
};

// The waiting side of the barriers of one CTA. Bounded like mbar_wait (tcgen05.cuh), but the clock is read only after
// some tries: reading it costs a few hundred cycles, during which the tensor core runs dry.
struct Waiter {
  volatile int* abort_flag;
  int* error_flag;
  __device__ __forceinline__ bool operator()(uint32_t bar, uint32_t parity, int code) const {
    uint64_t start = 0;
    for (uint32_t tries = 1; !mbar_try_wait(bar, parity); ++tries) {
      if ((tries & 63u) == 0) {
        if (*abort_flag) return false;
        const uint64_t now = global_timer_ns();
        if (start == 0) start = now;
        if (now - start > kWaitLimitNs) {
          *abort_flag = 1;
          atomicCAS(error_flag, 0, code);
          return false;
        }
      }
    }
    return true;
  }
  // two barriers, by a whole warp: one round trip where both are complete
  __device__ __forceinline__ bool both(uint32_t a, uint32_t a_parity, uint32_t b, uint32_t b_parity, int code) const {
    const uint32_t first = mbar_try_wait(a, a_parity), second = mbar_try_wait(b, b_parity);
    if (__all_sync(0xffffffffu, first & second)) return true;
    return warp(a, a_parity, code) && warp(b, b_parity, code);
  }
  // by a whole warp, which stays together
  __device__ __forceinline__ bool warp(uint32_t bar, uint32_t parity, int code) const {
    return __all_sync(0xffffffffu, (*this)(bar, parity, code));
  }
};

// A CTA that gave up leaves copies in flight; it stays until they have landed (a bounded pause, no one waits on it).
__device__ __forceinline__ void settle(const volatile int* abort_flag) {
  if (!*abort_flag) return;
  const uint64_t start = global_timer_ns();
  while (global_timer_ns() - start < 1000000ull) __nanosleep(1000);
}

// The forward and the query-gradient kernel are persistent, one CTA per SM: copies and first products of a CTA's next unit run
// under the tail of the last one, which pays where documents are short (a CTA per tile spent 4 to 6 us on starting, the
// first copies and the end, as much as 500 keys of work). Units are sorted by falling work and dealt back and forth, so
// that the CTAs' sums come out even.
__device__ __forceinline__ int unit_of_round(int round) {
  const int ctas = gridDim.x, cta = blockIdx.x;
  return round * ctas + (round & 1 ? ctas - 1 - cta : cta);
}

// A CTA's walk over its units, `per_record` units to a record; the record after the current one is read ahead.
struct Walk {
  const PlanRecord* records;
  int units, per_record, round, unit;
  PlanRecord here, ahead;
  __device__ __forceinline__ PlanRecord read(int u) const { return records[min(u, units - 1) / per_record]; }
  __device__ __forceinline__ Walk(const PlanRecord* r, int n, int per) : records(r), units(n), per_record(per), round(0), unit(unit_of_round(0)) {
    here = uniform(read(unit));
    ahead = read(unit_of_round(1));
  }
  __device__ __forceinline__ bool valid() const { return unit < units; }
  __device__ __forceinline__ void next() {
    unit = unit_of_round(++round);
    here = uniform(ahead);
    ahead = read(unit_of_round(round + 1));
  }
};

// ---- forward -------------------------------------------------------------------------
// Two 128-row stages per CTA against one stream of key tiles; per stage and tile
//   tensor core   S = Q K^T (128 x 128), then O += P V with P as the TMEM operand over S's own columns
//   warpgroup     row maximum and exponentials of S (a thread owns a row), P back to TMEM
// so one stage's products run under the other's exponentials. O stays in TMEM; it is rescaled by the warpgroup only
// when a row's maximum has grown by more than 2^8 (P and the sums stay below 2^8 times their scaled size: no
// overflow in fp32 or fp16, and the final division cancels the factor).
// P is rounded to the operands' type for the second product (the sum that divides it is not); scores, maxima, sums and O
// are fp32; y is rounded once.
// Measured, 4 x 4096 tokens in one document per row, 32 heads of 128 on one key head, bf16: 486 us = 1131 TFLOP/s of the
// causal half (FlashAttention-2: 1427 us); packed documents of 64 to 4096 tokens: 214 us. What bounds it: the chain
// scores -> exponentials -> P V -> next scores of the two stages (a tile of both takes 3.6 thousand cycles, of which the
// tensor core works 2048 and the special-function units 2048), at the clock the power limit leaves (1.5 to 1.7 GHz).
template <int HD> struct ForwardShape {
  static constexpr int kBoxes = HD / 64;
  static constexpr uint32_t kTile = kBoxes * BOX_BYTES;
  static constexpr int kRing = 2;
  static constexpr int kSmem = (2 + 2 * kRing) * kTile + 1024 + 256;
};
// Three warpgroups: two own a stage each, the third holds the copy and the MMA warp (two of its warps idle). Launched
// with 168 registers a thread; the third hands down registers so that a thread can hold half a row of scores, its packed form and the unit's state:
// 2 x 200 + 104 = 3 x 168.
constexpr int kForwardThreads = 384;
template <int N> __device__ __forceinline__ void registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
constexpr uint32_t kOutColumn = 256;       // TMEM: S of the stages at 0 and 128, O at 256 and 384

// Two stages of queries and their positions among the document's keys: stage s holds the tokens from a + s * tile_tokens
// on and sees the keys [0, end[s]).
struct ForwardWalk : Walk {
  int tile_tokens, head_blocks, group, packed;
  int end0, end1, n0, n1, n, head0, shared;
  __device__ __forceinline__ ForwardWalk(const AttentionParams& p)
      : Walk(p.items, p.units, p.head_blocks), tile_tokens(p.tile_tokens), head_blocks(p.head_blocks), group(p.heads / p.kv_heads), packed(p.packed) {
    open();
  }
  __device__ __forceinline__ void open() {
    head0 = unit % head_blocks * packed;
    shared = head0 / group;
    const int first1 = here.a + tile_tokens;
    end0 = min(here.length, first1);
    end1 = first1 < here.length ? min(here.length, first1 + tile_tokens) : 0;
    n0 = (end0 + KEYS - 1) / KEYS;
    n1 = (end1 + KEYS - 1) / KEYS;
    n = max(n0, n1);
  }
  __device__ __forceinline__ void next_unit() {
    next();
    open();
  }
  __device__ __forceinline__ int count(int s) const { return s ? n1 : n0; }
  // whether the stage needs more than the first 64 keys of tile j
  __device__ __forceinline__ bool both_halves(int s, int j) const { return (s ? end1 : end0) > j * KEYS + 64; }
};

template <typename T, int HD>
__global__ void __launch_bounds__(kForwardThreads, 1) attention_forward_tc_kernel(const __grid_constant__ AttentionParams p) {
  using Shape = ForwardShape<HD>;
  constexpr int BOXES = Shape::kBoxes, RING = Shape::kRing;
  constexpr uint32_t TILE = Shape::kTile;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t q_tile = smem_u32(smem), k_ring = q_tile + 2 * TILE, v_ring = k_ring + RING * TILE;
  const uint32_t bars = v_ring + RING * TILE;
  auto q_full = [&](int s) { return bars + 8u * s; };
  auto q_empty = [&](int s) { return bars + 16u + 8u * s; };
  auto s_full = [&](int s) { return bars + 32u + 8u * s; };
  auto p_full = [&](int s, int h) { return bars + 48u + 16u * s + 8u * h; };
  auto half_done = [&](int s) { return bars + 80u + 8u * s; };
  auto o_full = [&](int s) { return bars + 96u + 8u * s; };
  auto k_full = [&](int r) { return bars + 112u + 8u * r; };
  auto k_empty = [&](int r) { return bars + 112u + 8u * (RING + r); };
  auto v_full = [&](int r) { return bars + 112u + 8u * (2 * RING + r); };
  auto v_empty = [&](int r) { return bars + 112u + 8u * (3 * RING + r); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + (2 + 2 * RING) * TILE + 112 + 32 * RING);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(q_full(s), 1);
      mbar_init(q_empty(s), 1);
      mbar_init(s_full(s), 1);
      for (int h = 0; h < 2; ++h) mbar_init(p_full(s, h), 4);
      mbar_init(half_done(s), 1);
      mbar_init(o_full(s), 1);
    }
    for (int r = 0; r < RING; ++r) {
      mbar_init(k_full(r), 1);
      mbar_init(k_empty(r), 1);
      mbar_init(v_full(r), 1);
      mbar_init(v_empty(r), 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_shared();
  }
  if (warp == 9) tmem_alloc(smem_u32(tmem_slot));
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);
  const Waiter wait{abort_flag, p.error_flag};
  // Tiles of keys are counted through all units (t, the first of the current unit): ring slots and phases go by it. A
  // stage's own phases go by the tiles (and units) that it takes part in.

  if (warp >= 8) {
    registers_down<104>();
    if (warp == 8) {
      bool alive = true;
      int t = 0, loads0 = 0, loads1 = 0;
      for (ForwardWalk w(p); w.valid() && alive; w.next_unit()) {
        auto load_q = [&](int s, int& loads) {
          if (!wait.warp(q_empty(s), (loads & 1) ^ 1, 6)) { alive = false; return; }
          ++loads;
          if (elect_one()) {
            mbar_expect_tx(q_full(s), TILE);
            for (int b = 0; b < BOXES; ++b)
              tma_load_3d(q_tile + s * TILE + b * BOX_BYTES, &p.q, q_full(s), 64 * b, w.head0, w.here.start + w.here.a + s * w.tile_tokens);
          }
        };
        load_q(0, loads0);
        for (int j = 0; j < w.n && alive; ++j, ++t) {
          const int r = t % RING;
          const uint32_t free_parity = ((t / RING) & 1) ^ 1;
          if (!wait.warp(k_empty(r), free_parity, 6)) { alive = false; break; }
          if (elect_one()) {
            mbar_expect_tx(k_full(r), TILE);
            for (int b = 0; b < BOXES; ++b)
              tma_load_3d(k_ring + r * TILE + b * BOX_BYTES, &p.k, k_full(r), 64 * b, w.shared, w.here.start + j * KEYS);
          }
          if (j == 0 && w.n1) load_q(1, loads1);
          if (!alive || !wait.warp(v_empty(r), free_parity, 6)) { alive = false; break; }
          if (elect_one()) {
            mbar_expect_tx(v_full(r), TILE);
            for (int b = 0; b < BOXES; ++b)
              tma_load_3d(v_ring + r * TILE + b * BOX_BYTES, &p.v, v_full(r), 64 * b, w.shared, w.here.start + j * KEYS);
          }
        }
      }
    } else if (warp == 9) {
      int tiles[2] = {0, 0}, halves[2] = {0, 0}, units[2] = {0, 0};          // per stage
      auto scores = [&](const ForwardWalk& w, int s, int j, int t) {
        product_nt<T, HD>(tmem + s * 128, q_tile + s * TILE, k_ring + (t % RING) * TILE);
        commit(s_full(s));
        if (j + 1 == w.count(s)) commit(q_empty(s));
      };
      ForwardWalk w(p);
      bool alive = wait.warp(q_full(0), 0, 7) && wait.warp(k_full(0), 0, 7);
      if (alive) {
        tcgen05_fence_after();
        scores(w, 0, 0, 0);
        ++units[0];
        if (w.n1) {
          alive = wait.warp(q_full(1), 0, 7);
          if (alive) scores(w, 1, 0, 0);
          ++units[1];
        }
        commit(k_empty(0));
      }
      for (int t0 = 0; w.valid() && alive;) {
        ForwardWalk following = w;
        following.next_unit();
        for (int j = 0; j < w.n && alive; ++j) {
          const int t = t0 + j, r = t % RING, next = (t + 1) % RING;
          const uint32_t next_parity = ((t + 1) / RING) & 1;
          // a wait costs this warp 150 cycles even where nothing is to wait for: those for the copies go with others
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const int count = w.count(s);
            if (j < count) {
              if (!(s == 0 || j >= w.n0 ? wait.both(v_full(r), (t / RING) & 1, p_full(s, 0), tiles[s] & 1, 7) : wait.warp(p_full(s, 0), tiles[s] & 1, 7))) { alive = false; break; }
              tcgen05_fence_after();
              product_tn<T, HD, 8, 64, 0, 4>(tmem + kOutColumn + s * 128, tmem + s * 128, v_ring + r * TILE, j > 0);
              commit(half_done(s));
              ++tiles[s];
              if (w.both_halves(s, j)) {
                if (!(s == 0 && j + 1 < w.n ? wait.both(k_full(next), next_parity, p_full(s, 1), halves[s] & 1, 7) : wait.warp(p_full(s, 1), halves[s] & 1, 7))) { alive = false; break; }
                ++halves[s];
                tcgen05_fence_after();
                product_tn<T, HD, 8, 64, 4, 8>(tmem + kOutColumn + s * 128, tmem + s * 128, v_ring + r * TILE, true);
              }
              if (j + 1 == count) commit(o_full(s));
            }
            if (s == 1) commit(v_empty(r));
            if (j + 1 < w.n) {
              if (s == 0 && !(j < count && w.both_halves(s, j)) && !wait.warp(k_full(next), next_parity, 7)) { alive = false; break; }
              if (j + 1 < count) scores(w, s, j + 1, t + 1);
              if (s == 1) commit(k_empty(next));
            } else if (following.valid()) {                        // the next unit's first scores
              if (following.count(s)) {
                if (!wait.warp(q_full(s), units[s] & 1, 7) || (s == 0 && !wait.warp(k_full(next), next_parity, 7))) { alive = false; break; }
                ++units[s];
                scores(following, s, 0, t + 1);
              }
              if (s == 1) commit(k_empty(next));
            }
          }
        }
        t0 += w.n;
        w = following;
      }
    }
  } else {
    registers_up<200>();
    const int s = warp >> 2, thread = threadIdx.x & 127;
    const float c = p.scale * kLog2e;
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;          // this warp's 32 TMEM lanes
    const uint32_t s_addr = tmem + lanes + s * 128, o_addr = tmem + lanes + kOutColumn + s * 128;
    // fp16: probabilities are kept 2^7 above their size (at most 2^15 with the late rescaling), so that small ones do not
    // fall among the subnormals; the sum carries the factor too
    constexpr float kLift = std::is_same<T, __half>::value ? 7.0f : 0.0f;
    float top = -INFINITY, sum = 0.0f;
    bool alive = true;
    const float2 c2 = make_float2(c, c);
    // A unit's output is stored behind the next unit's first exponentials: the last P V is complete by then.
    bool pending = false;
    int finished = 0;
    int64_t out_row = -1;
    float out_top = 0.0f, out_sum = 0.0f;
    auto store = [&]() {
      if (!wait.warp(o_full(s), finished & 1, 8)) return false;
      ++finished;
      pending = false;
      tcgen05_fence_after();
      const float factor = 1.0f / out_sum;
      T* dst = static_cast<T*>(p.out) + out_row * p.dim;
      if (out_row >= 0 && p.lse) p.lse[out_row] = out_top * c + log2f(out_sum) - kLift;
#pragma unroll 1
      for (int g = 0; g < HD / 32; ++g) {
        uint32_t o[32];
        tmem_load_32(o_addr + 32 * g, o);
        if (out_row >= 0) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint4 v;
            uint32_t* word = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              word[e] = pack2<T>(__uint_as_float(o[8 * i + 2 * e]) * factor, __uint_as_float(o[8 * i + 2 * e + 1]) * factor);
            if (32 * g + 8 * i < p.dim) *reinterpret_cast<uint4*>(dst + 32 * g + 8 * i) = v;
          }
        }
      }
      return true;
    };
    // These threads hold a row of scores each, so they walk the units with less state than ForwardWalk.
    auto read = [&](int round) { return p.items[min(unit_of_round(round), p.units - 1) / p.head_blocks]; };
    PlanRecord ahead = read(0);
    int t0 = 0, tiles = 0;
    for (int round = 0; unit_of_round(round) < p.units && alive; ++round) {
      const PlanRecord here = uniform(ahead);
      ahead = read(round + 1);
      const int first = here.a + s * p.tile_tokens;                // the stage's first token
      const int end = first < here.length ? min(here.length, first + p.tile_tokens) : 0, count = (end + KEYS - 1) / KEYS;
      const int token = first + thread / p.packed;
      const int last_key = min(token, here.length - 1);
      if (!count && pending && !store()) { alive = false; break; }       // idle in this unit: nothing to store behind
      for (int j = 0; j < count && alive; ++j, ++tiles) {
        const int cols = end > j * KEYS + 64 ? KEYS : 64, t = t0 + j;      // the halves this tile needs
        const bool partial = j * KEYS + cols - 1 > first;
        const int limit = last_key - j * KEYS;                   // columns above it are not this row's
        if (!wait.warp(s_full(s), tiles & 1, 8)) { alive = false; break; }
        tcgen05_fence_after();
        if (j * KEYS + cols > here.length) {
          // the tile runs past the document: rows of V behind its end must not meet the zero probabilities
          if (!wait.warp(v_full(t % RING), (t / RING) & 1, 8)) { alive = false; break; }
          clear_rows<BOXES>(v_ring + (t % RING) * TILE, here.length - j * KEYS, cols, thread, 128);
        }
        // Halves of 64 keys: the first half of P V runs under the exponentials of the second. The exponentials do not wait
        // for the half's maximum: they use the maximum so far, and the half is done again with the new one in the rare
        // case that a score is more than 2^8 above it.
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {                            // (rolled: the MMA warp shares the instruction cache)
          if (64 * h >= cols) break;
          uint32_t x[2][32];
#pragma unroll
          for (int g = 0; g < 2; ++g) tmem_load_32_issue(s_addr + 64 * h + 32 * g, x[g]);
#pragma unroll
          for (int g = 0; g < 2; ++g) tmem_load_wait(x[g]);
          if (partial) {
            rare();
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (64 * h + 32 * g + i > limit) x[g][i] = 0xff800000u;     // -infinity
          }
          if (j == 0 && h == 0) {                                // key 0 is every row's: a score, not -infinity
            rare();
            top = -INFINITY;
            sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 32; ++i) top = max3(top, __uint_as_float(x[0][i]), __uint_as_float(x[1][i]));
          }
          uint32_t packed[32];
          float2 part[2];
          while (true) {
            const float shift = kLift - top * c;
            const float2 shift2 = make_float2(shift, shift);
            float peak[4] = {top, top, top, top};
            part[0] = part[1] = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float2 raw = make_float2(__uint_as_float(x[i / 16][2 * (i % 16)]), __uint_as_float(x[i / 16][2 * (i % 16) + 1]));
              peak[i & 3] = max3(peak[i & 3], raw.x, raw.y);
              float2 e = fma2(raw, c2, shift2);
              e.x = exp2_approx(e.x);
              e.y = exp2_approx(e.y);
              part[i & 1] = add2(part[i & 1], e);
              packed[i] = pack2<T>(e.x, e.y);
            }
            const float best = fmaxf(fmaxf(peak[0], peak[1]), fmaxf(peak[2], peak[3]));
            if (!__any_sync(0xffffffffu, (best - top) * c > 8.0f)) break;
            rare();
            // O holds the products of all halves so far; the last one issued has to be complete
            const bool issued = h == 1 || j > 0;
            if (h == 1 && !wait.warp(half_done(s), tiles & 1, 8)) { alive = false; break; }
            tcgen05_fence_after();
            const float factor = exp2_approx((top - best) * c);
            top = best;
            sum *= factor;
            if (issued) {
#pragma unroll 1
              for (int g = 0; g < HD / 32; ++g) {
                uint32_t o[32];
                tmem_load_32(o_addr + 32 * g, o);
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
                tmem_store_32(o_addr + 32 * g, o);
              }
            }
          }
          if (!alive) break;
          part[0] = add2(part[0], part[1]);
          sum += part[0].x + part[0].y;
          tmem_store_32(s_addr + 32 * h, packed);
          tmem_store_wait();
          if (h == 0 && pending && !store()) { alive = false; break; }       // O is free for this unit's products
          tcgen05_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(p_full(s, h));
        }
      }
      if (alive && count) {
        pending = true;
        const int head = unit_of_round(round) % p.head_blocks * p.packed + thread % p.packed;
        out_row = token < here.length ? (static_cast<int64_t>(here.start) + token) * p.heads + head : int64_t(-1);
        out_top = top;
        out_sum = sum;
      }
      t0 += (min(here.length, here.a + 2 * p.tile_tokens) + KEYS - 1) / KEYS;      // the tiles of both stages
    }
    if (alive && pending) store();
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  settle(abort_flag);
  if (warp == 9) tmem_free(tmem);
}

// ---- backward ------------------------------------------------------------------------
// Two kernels that each recompute the probabilities, instead of one that would have to add query gradients from many key
// tiles into memory: 14 instead of 10 FLOP per pair and channel, but no atomics and no order that changes the sums.
// Measured, 4 x 4096 tokens, 32 heads of 128 on one key head, bf16: query gradients 653 us, key gradients 954 us, delta
// 48 us, sum of the pieces 16 us (1196 TFLOP/s of the products that run; FlashAttention-2 with atomics: 4.5 ms).
// dS is rounded to the operands' type for its two products, as P is for dv, and delta is formed in fp32 from the rounded
// y: in bf16 dq and dk come out 2.4e-3 to 2.5e-3 (relative norm) from the exact values, 1.7e-3 of it the rounding of the
// results themselves.
// A document's first query sees one key: P = 1 and y = v, so its dS is 0 and is set to 0 (times 0: a NaN stays one); as
// the difference of two sums it would be their rounding errors, and nothing but those for documents of one token.
//
// fp16 keeps 10 more bits of range for small probabilities: P is formed as 2^10 P (at most 1024) and the factor is
// taken out of dv at the end and out of dS where it is formed.
template <typename T> struct Lift {
  static constexpr float kBits = std::is_same<T, __half>::value ? 10.0f : 0.0f;
  static constexpr float kInverse = std::is_same<T, __half>::value ? 0x1p-10f : 1.0f;
};
constexpr int kBackwardThreads = 384;      // two elementwise warpgroups and one that holds the copy, MMA and statistics warps

// dP^T / dS and P: each warpgroup packs its own 64 columns over the first half of where they were.
constexpr int kHalfSpan = 4, kHalfStride = 64;

// dk and dv of one 128-key tile over a run of query tiles. Everything is transposed - a thread owns a KEY -, so that P^T
// and dS^T come out of TMEM in the layout in which they go back as A operands:
//   S^T = K Q^T, dP^T = V dY^T, dV += P^T dY, dK += dS^T Q
// The tensor core runs dV(i), S(i + 1), dK(i), dP(i + 1): the exponentials of tile i + 1 run under dK(i) and dP(i + 1),
// dS under dV and S. TMEM: S^T / P^T at 0, dP^T / dS^T at 128, dV at 256, dK at 384 - all of it.
// What bounds it: P(i) -> dV(i) -> S(i + 1) -> exponentials -> P(i + 1), 2.7 thousand cycles a tile against 2176 of tensor
// work. One CTA per piece: a persistent form was 7 % slower (its longer code and state in the loop cost more than the
// starts, as pieces are 16 query tiles or more).
template <int HD> struct KeyShape {
  static constexpr uint32_t kTile = HD / 64 * BOX_BYTES;
  static constexpr int kRing = 2;
  static constexpr uint32_t kStatTile = 128 * 32;                // 128 rows x 16 values
  static constexpr uint32_t kStats = 2 * kStatTile;              // log-sums, deltas
  static constexpr int kSmem = (2 + 2 * kRing) * kTile + kStatTile + kRing * kStats + 1024 + 256;
};

// The statistics of a query tile vary along the COLUMNS of the transposed score tile, so every thread would need all of
// them - 128 broadcast loads from shared memory per thread and tile, on the bandwidth the MMAs' operands need (1.3 of
// 3.6 thousand cycles per tile). Instead they are subtracted by the tensor core as one more k step of 16: rows of
// weights (the same for every key) times the value of each query split into parts of the operand type,
//   value = 8 * w0 * part0 + w1 * part1 + w2 * part2    (k = 0..7: part0, 8: part1, 9: part2, others 0)
// exact to 2^-24 for bf16, and for fp16 from 2^-29 up to 2^34.
template <typename T> struct Split {
  static constexpr float kWeight0 = std::is_same<T, __half>::value ? 32768.0f : 1.0f;
  static constexpr float kWeight1 = std::is_same<T, __half>::value ? 256.0f : 1.0f;
  static constexpr float kWeight2 = std::is_same<T, __half>::value ? 0.0625f : 1.0f;
};
// Row `row` of such a tile: K-major without swizzle, 8 x 16-byte blocks, the two k halves 2 KB apart.
__device__ __forceinline__ void store_stat_row(uint32_t tile, int row, uint32_t eight, uint32_t two) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(tile + row * 16), "r"(eight) : "memory");
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %2, %2};" ::"r"(tile + 2048 + row * 16), "r"(two), "r"(0) : "memory");
}
template <typename T> __device__ __forceinline__ void store_split(uint32_t tile, int row, float value) {
  const float part0 = round_to<T>(value * (0.125f / Split<T>::kWeight0));
  const float rest0 = value - part0 * (8.0f * Split<T>::kWeight0);
  const float part1 = round_to<T>(rest0 * (1.0f / Split<T>::kWeight1));
  const float rest1 = rest0 - part1 * Split<T>::kWeight1;
  store_stat_row(tile, row, pack2<T>(part0, part0), pack2<T>(part1, rest1 * (1.0f / Split<T>::kWeight2)));
}
template <typename T> __device__ __forceinline__ void subtract_stats(uint32_t d, uint32_t weights, uint32_t stats) {
  const uint32_t plain = desc_high(128) & ~(7u << 29);           // no swizzle, 8-row groups 128 bytes apart
  const uint32_t idesc = operand_desc<T>(false, 128), a_lo = desc_low(weights, 2048), b_lo = desc_low(stats, 2048);
  if (elect_one()) umma_bf16(d, a_lo, plain, b_lo, plain, idesc, 1);
}

template <typename T, int HD>
__global__ void __launch_bounds__(kBackwardThreads, 1) attention_key_gradient_tc_kernel(const __grid_constant__ AttentionParams p) {
  using Shape = KeyShape<HD>;
  constexpr int BOXES = HD / 64, RING = Shape::kRing;
  constexpr uint32_t TILE = Shape::kTile;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t k_tile = smem_u32(smem), v_tile = k_tile + TILE, q_ring = v_tile + TILE, g_ring = q_ring + RING * TILE;
  const uint32_t weights = g_ring + RING * TILE, stats = weights + Shape::kStatTile;      // per ring stage: log-sums, deltas
  const uint32_t bars = stats + RING * Shape::kStats;
  const uint32_t kv_full = bars, s_full = bars + 8, dp_full = bars + 16, p_ready = bars + 24, ds_ready = bars + 32, done = bars + 40;
  auto q_full = [&](int r) { return bars + 48u + 8u * r; };
  auto q_empty = [&](int r) { return bars + 48u + 8u * (RING + r); };
  auto g_full = [&](int r) { return bars + 48u + 8u * (2 * RING + r); };
  auto g_empty = [&](int r) { return bars + 48u + 8u * (3 * RING + r); };
  auto stat_full = [&](int r) { return bars + 48u + 8u * (4 * RING + r); };
  auto stat_empty = [&](int r) { return bars + 48u + 8u * (5 * RING + r); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + (2 + 2 * RING) * TILE + Shape::kStatTile + RING * Shape::kStats + 48 + 48 * RING);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(kv_full, 1);
    mbar_init(s_full, 1);
    mbar_init(dp_full, 1);
    mbar_init(p_ready, 8);
    mbar_init(ds_ready, 8);
    mbar_init(done, 1);
    for (int r = 0; r < RING; ++r) {
      mbar_init(q_full(r), 1);
      mbar_init(q_empty(r), 1);
      mbar_init(g_full(r), 1);
      mbar_init(g_empty(r), 1);
      mbar_init(stat_full(r), 1);
      mbar_init(stat_empty(r), 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_shared();
  }
  if (threadIdx.x < 128) {
    store_stat_row(weights, threadIdx.x, pack2<T>(Split<T>::kWeight0, Split<T>::kWeight0), pack2<T>(Split<T>::kWeight1, Split<T>::kWeight2));
    fence_async_shared();
  }
  if (warp == 9) tmem_alloc(smem_u32(tmem_slot));
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);
  const Waiter wait{abort_flag, p.error_flag};

  const PlanRecord item = uniform(p.items[2 * (blockIdx.x / p.kv_heads)]);
  const PlanRecord range = uniform(p.items[2 * (blockIdx.x / p.kv_heads) + 1]);
  const int shared = blockIdx.x % p.kv_heads, key0 = item.a, slot = item.b;
  const int first = range.start, count = range.length - range.start;          // query tiles of this piece
  const int per_block = (item.length - key0 + p.tile_tokens - 1) / p.tile_tokens;
  const int group0 = shared * (p.heads / p.kv_heads);
  // query tile i of the piece: its first token in the document and first head
  auto tile_token = [&](int i) { return key0 + ((first + i) % per_block) * p.tile_tokens; };
  auto tile_head = [&](int i) { return group0 + ((first + i) / per_block) * p.packed; };

  if (warp >= 8) {
    registers_down<104>();
    if (warp == 8) {
      if (lane == 0) {
        mbar_expect_tx(kv_full, 2 * TILE);
        for (int b = 0; b < BOXES; ++b) tma_load_3d(k_tile + b * BOX_BYTES, &p.k, kv_full, 64 * b, shared, item.start + key0);
        for (int b = 0; b < BOXES; ++b) tma_load_3d(v_tile + b * BOX_BYTES, &p.v, kv_full, 64 * b, shared, item.start + key0);
        for (int i = 0; i < count; ++i) {
          const int r = i % RING;
          const uint32_t free_parity = ((i / RING) & 1) ^ 1;
          const int token = item.start + tile_token(i), head = tile_head(i);
          if (!wait(q_empty(r), free_parity, 6)) break;
          mbar_expect_tx(q_full(r), TILE);
          for (int b = 0; b < BOXES; ++b) tma_load_3d(q_ring + r * TILE + b * BOX_BYTES, &p.q, q_full(r), 64 * b, head, token);
          if (!wait(g_empty(r), free_parity, 6)) break;
          mbar_expect_tx(g_full(r), TILE);
          for (int b = 0; b < BOXES; ++b) tma_load_3d(g_ring + r * TILE + b * BOX_BYTES, &p.dy, g_full(r), 64 * b, head, token);
        }
      }
      __syncwarp();
    } else if (warp == 9) {
      auto scores = [&](int r) {                                 // log2 P / c
        product_nt<T, HD>(tmem, k_tile, q_ring + r * TILE);
        subtract_stats<T>(tmem, weights, stats + r * Shape::kStats);
        commit(s_full);
      };
      auto slopes = [&](int r) {                                 // dP - delta
        product_nt<T, HD>(tmem + 128, v_tile, g_ring + r * TILE);
        subtract_stats<T>(tmem + 128, weights, stats + r * Shape::kStats + Shape::kStatTile);
        commit(dp_full);
      };
      bool alive = wait.warp(kv_full, 0, 7) && wait.warp(q_full(0), 0, 7) && wait.warp(stat_full(0), 0, 7);
      if (alive) {
        tcgen05_fence_after();
        scores(0);
        alive = wait.warp(g_full(0), 0, 7);
        if (alive) slopes(0);
      }
      for (int i = 0; i < count && alive; ++i) {
        const int r = i % RING, next = (i + 1) % RING;
        const uint32_t next_parity = ((i + 1) / RING) & 1;
        if (!wait.warp(p_ready, i & 1, 7)) break;
        tcgen05_fence_after();
        product_tn<T, HD, kHalfSpan, kHalfStride, 0, 8>(tmem + 256, tmem, g_ring + r * TILE, i > 0);
        commit(g_empty(r));
        if (i + 1 < count) {
          if (!wait.both(q_full(next), next_parity, stat_full(next), next_parity, 7)) break;
          scores(next);
        }
        if (!wait.warp(ds_ready, i & 1, 7)) break;
        tcgen05_fence_after();
        product_tn<T, HD, kHalfSpan, kHalfStride, 0, 8>(tmem + 384, tmem + 128, q_ring + r * TILE, i > 0);
        commit(q_empty(r));
        if (i + 1 < count) {
          if (!wait.warp(g_full(next), next_parity, 7)) break;
          slopes(next);
        } else {
          commit(done);
        }
      }
      __syncwarp();
    } else if (warp == 10) {
      const float per_score = -1.0f / (p.scale * kLog2e);
      for (int i = 0; i < count; ++i) {
        const int r = i % RING;
        const int token0 = tile_token(i), head0 = tile_head(i);
        float values[2][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = lane + 32 * e, token = token0 + row / p.packed;
          const int64_t at = (static_cast<int64_t>(item.start) + token) * p.heads + head0 + row % p.packed;
          const bool inside = token < item.length;
          values[0][e] = inside ? (p.lse[at] - Lift<T>::kBits) * per_score : 0.0f;
          values[1][e] = inside ? -p.delta[at] : 0.0f;
        }
        if (!wait.warp(stat_empty(r), ((i / RING) & 1) ^ 1, 6)) break;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          store_split<T>(stats + r * Shape::kStats, lane + 32 * e, values[0][e]);
          store_split<T>(stats + r * Shape::kStats + Shape::kStatTile, lane + 32 * e, values[1][e]);
        }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(stat_full(r));
      }
    }
  } else {
    registers_up<200>();
    const int half = warp >> 2, thread = threadIdx.x & 127;
    const int key = key0 + thread;
    const float c = p.scale * kLog2e;
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;
    const uint32_t s_addr = tmem + lanes + 64 * half, dp_addr = s_addr + 128;
    bool alive = true;
    int token0 = tile_token(0) - p.tile_tokens;
    for (int i = 0; i < count; ++i) {
      const int r = i % RING;
      token0 += p.tile_tokens;
      if (token0 >= item.length) token0 = key0;
      // this thread's columns [low, high) of the tile: queries at or after its key, inside the document
      const bool partial = token0 < key0 + 127 || token0 + p.tile_tokens > item.length;
      // (clamped to the tile, so that the products fit for documents of any length)
      const int low = max(key - token0, 0) * p.packed - 64 * half, high = min(item.length - token0, p.tile_tokens) * p.packed - 64 * half;
      if (!wait.warp(s_full, i & 1, 8)) { alive = false; break; }
      tcgen05_fence_after();
      float prob[64];
#pragma unroll
      for (int g = 0; g < 2; ++g) tmem_load_32_issue(s_addr + 32 * g, *reinterpret_cast<uint32_t(*)[32]>(&prob[32 * g]));
#pragma unroll
      for (int g = 0; g < 2; ++g) tmem_load_wait(*reinterpret_cast<uint32_t(*)[32]>(&prob[32 * g]));
      // a quarter on the FMA units: 944 us of 978 without at 4 x 4096 tokens, 32 heads; an eighth 956, a half 965 (the
      // forward and the query-gradient kernel are no faster with any share)
#pragma unroll
      for (int e = 0; e < 64; e += 2) {
        const float2 a = exp2_pair(mul2(make_float2(prob[e], prob[e + 1]), make_float2(c, c)), e % 16 < 4);
        prob[e] = a.x;
        prob[e + 1] = a.y;
      }
      if (partial) {
        rare();
#pragma unroll
        for (int e = 0; e < 64; ++e)
          if (e < low || e >= high) prob[e] = 0.0f;
      }
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        uint32_t packed[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) packed[e] = pack2<T>(prob[32 * g + 2 * e], prob[32 * g + 2 * e + 1]);
        tmem_store_16(s_addr + 16 * g, packed);
      }
      if (token0 + p.tile_tokens > item.length) {
        // rows of dY and Q behind the document's end must not meet the zeros of P and dS
        if (!wait.warp(g_full(r), (i / RING) & 1, 8)) { alive = false; break; }
        const int from = (item.length - token0) * p.packed;
        clear_rows<BOXES>(g_ring + r * TILE, from, 128, threadIdx.x, 256);
        clear_rows<BOXES>(q_ring + r * TILE, from, 128, threadIdx.x, 256);
      }
      tmem_store_wait();
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_ready);
      if (!wait.warp(dp_full, i & 1, 8)) { alive = false; break; }
      tcgen05_fence_after();
      if (threadIdx.x == 0) mbar_arrive(stat_empty(r));
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        uint32_t x[32], packed[16];
        tmem_load_32(dp_addr + 32 * g, x);
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          float2 slope = mul2(make_float2(prob[32 * g + e], prob[32 * g + e + 1]), make_float2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])));
          if constexpr (Lift<T>::kBits != 0.0f) slope = mul2(slope, make_float2(Lift<T>::kInverse, Lift<T>::kInverse));
          x[e] = __float_as_uint(slope.x);
          x[e + 1] = __float_as_uint(slope.y);
        }
        if (partial) {
          rare();
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (32 * g + e < low || 32 * g + e >= high) x[e] = 0u;
          if (token0 == 0 && key == 0) {                           // the document's first query
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (32 * g + e < p.packed - 64 * half) x[e] = __float_as_uint(__uint_as_float(x[e]) * 0.0f);
          }
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) packed[e] = pack2<T>(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1]));
        // chunk g goes over columns that chunk 0 has been read from
        tmem_store_16(dp_addr + 16 * g, packed);
      }
      tmem_store_wait();
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_ready);
    }
    if (alive && wait.warp(done, 0, 8)) {
      tcgen05_fence_after();
      const bool mine = key < item.length;
      const int64_t row = (static_cast<int64_t>(item.start) + key) * p.kv_heads + shared;
#pragma unroll 1
      for (int g = 0; g < HD / 32; ++g) {
        // half 0 takes dk, half 1 dv
        uint32_t o[32];
        tmem_load_32(tmem + lanes + (half ? 256 : 384) + 32 * g, o);
        const float factor = half ? Lift<T>::kInverse : p.scale;
        if (mine && slot < 0) {
          T* dst = static_cast<T*>(half ? p.dv : p.dk) + row * p.dim + 32 * g;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint4 v;
            uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
            for (int f = 0; f < 4; ++f)
              w[f] = pack2<T>(__uint_as_float(o[8 * e + 2 * f]) * factor, __uint_as_float(o[8 * e + 2 * f + 1]) * factor);
            if (32 * g + 8 * e < p.dim) *reinterpret_cast<uint4*>(dst + 8 * e) = v;
          }
        } else if (mine) {
          float* dst = p.partials + (((static_cast<int64_t>(slot) * p.kv_heads + shared) * 2 + half) * 128 + thread) * p.dim + 32 * g;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (32 * g + 4 * e < p.dim)
              *reinterpret_cast<float4*>(dst + 4 * e) =
                  make_float4(__uint_as_float(o[4 * e]) * factor, __uint_as_float(o[4 * e + 1]) * factor,
                              __uint_as_float(o[4 * e + 2]) * factor, __uint_as_float(o[4 * e + 3]) * factor);
        }
      }
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  settle(abort_flag);
  if (warp == 9) tmem_free(tmem);
}

// dk and dv of the key tiles that were cut into pieces: the pieces' shares added in order, four channels per thread.
template <typename T>
__global__ void __launch_bounds__(256) attention_sum_pieces_kernel(const __grid_constant__ AttentionParams p) {
  const PlanRecord r = p.items[blockIdx.x];            // (first token, rows, first slot, slots)
  const int shared = blockIdx.z / 2, which = blockIdx.z % 2, quads = p.dim / 4;
  const int i = blockIdx.y * 256 + threadIdx.x;
  if (i >= r.length * quads) return;
  const int64_t step = static_cast<int64_t>(p.kv_heads) * 2 * 128 * p.dim;
  const float* src = p.partials + ((static_cast<int64_t>(r.a) * p.kv_heads + shared) * 2 + which) * 128 * p.dim + 4 * i;
  float4 sum = *reinterpret_cast<const float4*>(src);
#pragma unroll 4
  for (int s = 1; s < r.b; ++s) {
    const float4 v = __ldcs(reinterpret_cast<const float4*>(src + s * step));
    sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
  }
  const int row = i / quads, at = 4 * (i % quads);
  *reinterpret_cast<uint2*>(static_cast<T*>(which ? p.dv : p.dk) + ((static_cast<int64_t>(r.start) + row) * p.kv_heads + shared) * p.dim + at) =
      make_uint2(pack2<T>(sum.x, sum.y), pack2<T>(sum.z, sum.w));
}

// dq of one 128-row tile over the document's keys: S = Q K^T, dP = dY V^T, dQ += dS K. A thread owns a row (two
// threads share it, 64 columns each). S has two buffers and dS goes back over its own S, so dP(j + 1) may start as soon
// as dP(j) has been read: the tensor core runs dP(j + 1), dQ(j), S(j + 2) under the exponentials of tile j + 1.
// TMEM: S at 0 and 128, dP at 256, dQ at 384. What bounds it: the issue of 24 MMAs, two commits and three waits a tile,
// 2.2 thousand cycles against 1536 of tensor work, and about as much work of the warpgroups.
template <int HD> struct QueryShape {
  static constexpr uint32_t kTile = HD / 64 * BOX_BYTES;
  static constexpr int kKeyRing = 3, kValueRing = 2;
  static constexpr int kSmem = (2 + kKeyRing + kValueRing) * kTile + 1024 + 256;
};

// A tile of queries and its position among the document's keys, as the MMA warp walks them.
struct QueryWalk : Walk {
  int tile_tokens, head_blocks, group, packed;
  int n, end, head0, shared, j;
  __device__ __forceinline__ QueryWalk(const AttentionParams& p)
      : Walk(p.items, p.units, p.head_blocks), tile_tokens(p.tile_tokens), head_blocks(p.head_blocks), group(p.heads / p.kv_heads), packed(p.packed) {
    open();
  }
  __device__ __forceinline__ void open() {
    head0 = unit % head_blocks * packed;
    shared = head0 / group;
    end = min(here.length, here.a + tile_tokens);                 // keys [0, end) are all the tile can see
    n = (end + KEYS - 1) / KEYS;
    j = 0;
  }
  __device__ __forceinline__ void next_unit() {
    next();
    open();
  }
  __device__ __forceinline__ void advance() {
    if (++j == n) next_unit();
  }
  __device__ __forceinline__ bool last() const { return j + 1 == n; }
  // whether the tile needs more than its first 64 keys
  __device__ __forceinline__ bool both_halves(int tile) const { return end > tile * KEYS + 64; }
};

template <typename T, int HD>
__global__ void __launch_bounds__(kBackwardThreads, 1) attention_query_gradient_tc_kernel(const __grid_constant__ AttentionParams p) {
  using Shape = QueryShape<HD>;
  constexpr int BOXES = HD / 64, KR = Shape::kKeyRing, VR = Shape::kValueRing;
  constexpr uint32_t TILE = Shape::kTile;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t q_tile = smem_u32(smem), g_tile = q_tile + TILE, k_ring = g_tile + TILE, v_ring = k_ring + KR * TILE;
  const uint32_t bars = v_ring + VR * TILE;
  const uint32_t q_full = bars, g_full = bars + 8, dp_full = bars + 16, ds_ready = bars + 24, done = bars + 32, q_empty = bars + 40, g_empty = bars + 48;
  auto s_full = [&](int b) { return bars + 56u + 8u * b; };
  auto k_full = [&](int r) { return bars + 72u + 8u * r; };
  auto v_full = [&](int r) { return bars + 72u + 8u * (KR + r); };
  auto v_empty = [&](int r) { return bars + 72u + 8u * (KR + VR + r); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + (2 + KR + VR) * TILE + 72 + 8 * (KR + 2 * VR));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(g_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(g_empty, 1);
    mbar_init(dp_full, 1);
    mbar_init(ds_ready, 8);
    mbar_init(done, 1);
    for (int b = 0; b < 2; ++b) mbar_init(s_full(b), 1);
    for (int r = 0; r < KR; ++r) mbar_init(k_full(r), 1);
    for (int r = 0; r < VR; ++r) {
      mbar_init(v_full(r), 1);
      mbar_init(v_empty(r), 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_shared();
  }
  if (warp == 9) tmem_alloc(smem_u32(tmem_slot));
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);
  const Waiter wait{abort_flag, p.error_flag};
  // Tiles of keys are counted through all units (t): ring slots, S buffers and barrier phases go by t; those that are
  // used once per unit go by the round.

  if (warp >= 8) {
    registers_down<104>();
    if (warp == 8) {
      bool alive = true;
      int t = 0;
      for (QueryWalk w(p); w.valid() && alive; w.next_unit()) {
        const int token = w.here.start + w.here.a;
        const uint32_t free_parity = (w.round & 1) ^ 1;
        if (!wait.warp(q_empty, free_parity, 6)) break;
        if (elect_one()) {
          mbar_expect_tx(q_full, TILE);
          for (int b = 0; b < BOXES; ++b) tma_load_3d(q_tile + b * BOX_BYTES, &p.q, q_full, 64 * b, w.head0, token);
        }
        for (int j = 0; j < w.n; ++j, ++t) {
          const int kr = t % KR, vr = t % VR, key = w.here.start + j * KEYS;
          // the slot's last tile, t - 3, was read by its dQ, and S(t - 1) was issued behind that (its next phase needs this
          // tile, so the phase waited for cannot be missed)
          if (t >= KR && !wait.warp(s_full((t - 1) & 1), ((t - 1) >> 1) & 1, 6)) { alive = false; break; }
          if (elect_one()) {
            mbar_expect_tx(k_full(kr), TILE);
            for (int b = 0; b < BOXES; ++b) tma_load_3d(k_ring + kr * TILE + b * BOX_BYTES, &p.k, k_full(kr), 64 * b, w.shared, key);
          }
          if (j == 0) {
            if (!wait.warp(g_empty, free_parity, 6)) { alive = false; break; }
            if (elect_one()) {
              mbar_expect_tx(g_full, TILE);
              for (int b = 0; b < BOXES; ++b) tma_load_3d(g_tile + b * BOX_BYTES, &p.dy, g_full, 64 * b, w.head0, token);
            }
          }
          if (!wait.warp(v_empty(vr), ((t / VR) & 1) ^ 1, 6)) { alive = false; break; }
          if (elect_one()) {
            mbar_expect_tx(v_full(vr), TILE);
            for (int b = 0; b < BOXES; ++b) tma_load_3d(v_ring + vr * TILE + b * BOX_BYTES, &p.v, v_full(vr), 64 * b, w.shared, key);
          }
        }
      }
    } else if (warp == 9) {
      bool alive = true;
      auto scores = [&](const QueryWalk& w, int t) {
        alive = (w.j > 0 || wait.warp(q_full, w.round & 1, 7)) && wait.warp(k_full(t % KR), (t / KR) & 1, 7);
        if (!alive) return;
        product_nt<T, HD>(tmem + (t & 1) * 128, q_tile, k_ring + (t % KR) * TILE);
        commit(s_full(t & 1));
        if (w.last()) commit(q_empty);
      };
      // a commit costs this warp 130 cycles: slots of the rings are released by who sees the products complete
      auto slopes = [&](const QueryWalk& w, int t) {
        if (w.j == 0 && !wait.warp(g_full, w.round & 1, 7)) alive = false;
        if (!alive) return;
        product_nt<T, HD>(tmem + 256, g_tile, v_ring + (t % VR) * TILE);
        commit(dp_full);
        if (w.last()) commit(g_empty);
      };
      QueryWalk cur(p), nxt = cur;
      nxt.advance();
      QueryWalk ahd = nxt;
      if (nxt.valid()) ahd.advance();
      scores(cur, 0);
      alive = alive && wait.warp(v_full(0), 0, 7);
      if (alive) slopes(cur, 0);
      if (alive && nxt.valid()) scores(nxt, 1);
      for (int t = 0; alive && cur.valid(); ++t) {
        if (!(nxt.valid() ? wait.both(v_full((t + 1) % VR), ((t + 1) / VR) & 1, ds_ready, t & 1, 7) : wait.warp(ds_ready, t & 1, 7))) break;
        tcgen05_fence_after();
        if (nxt.valid()) slopes(nxt, t + 1);
        if (!alive) break;
        product_tn<T, HD, kHalfSpan, kHalfStride, 0, 4>(tmem + 384, tmem + (t & 1) * 128, k_ring + (t % KR) * TILE, cur.j > 0);
        if (cur.both_halves(cur.j)) product_tn<T, HD, kHalfSpan, kHalfStride, 4, 8>(tmem + 384, tmem + (t & 1) * 128, k_ring + (t % KR) * TILE, true);
        if (cur.last()) commit(done);
        if (ahd.valid()) scores(ahd, t + 2);
        cur = nxt;
        nxt = ahd;
        if (ahd.valid()) ahd.advance();
      }
    }
  } else {
    registers_up<200>();
    const int half = warp >> 2, thread = threadIdx.x & 127;
    const float c = p.scale * kLog2e;
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;
    bool alive = true;
    int t = 0;
    // A unit's dq is stored while the next unit's first exponentials are done: `done` comes 800 cycles after the last dS.
    T* dst = nullptr;
    auto store = [&](int round) {
      if (!wait.warp(done, round & 1, 8)) return false;
      tcgen05_fence_after();
#pragma unroll 1
      for (int g = 0; g < HD / 64; ++g) {
        uint32_t o[32];
        tmem_load_32(tmem + lanes + 384 + half * (HD / 2) + 32 * g, o);
        if (dst) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint4 v;
            uint32_t* word = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
            for (int f = 0; f < 4; ++f)
              word[f] = pack2<T>(__uint_as_float(o[8 * e + 2 * f]) * p.scale, __uint_as_float(o[8 * e + 2 * f + 1]) * p.scale);
            if (half * (HD / 2) + 32 * g + 8 * e < p.dim) *reinterpret_cast<uint4*>(dst + 32 * g + 8 * e) = v;
          }
        }
      }
      return true;
    };
    auto row_of = [&](const QueryWalk& w) {
      const int token = w.here.a + thread / p.packed;
      return token < w.here.length ? (static_cast<int64_t>(w.here.start) + token) * p.heads + w.head0 + thread % p.packed : int64_t(-1);
    };
    // infinite for the document's first query, which leaves nothing of its dS
    auto log_sum = [&](const QueryWalk& w, int64_t row) {
      return row < 0 ? 0.0f : w.here.a + thread / p.packed == 0 ? __int_as_float(0x7f800000) : p.lse[row];
    };
    QueryWalk w(p);
    int64_t row = row_of(w);
    float lse = log_sum(w, row), delta = row >= 0 ? p.delta[row] : 0.0f;
    while (w.valid() && alive) {
      const int last_key = min(w.here.a + thread / p.packed, w.here.length - 1);
      QueryWalk following = w;                                     // its statistics are on their way meanwhile
      following.next_unit();
      const int64_t next_row = following.valid() ? row_of(following) : int64_t(-1);
      const float next_lse = log_sum(following, next_row), next_delta = next_row >= 0 ? p.delta[next_row] : 0.0f;
      for (int j = 0; j < w.n; ++j, ++t) {
        const int all_cols = w.both_halves(j) ? KEYS : 64;
        const bool idle = half && all_cols == 64;                  // nothing in this warpgroup's 64 columns
        const uint32_t s_addr = tmem + lanes + (t & 1) * 128 + 64 * half, dp_addr = tmem + lanes + 256 + 64 * half;
        const bool partial = j * KEYS + all_cols - 1 > w.here.a;
        const int limit = last_key - j * KEYS - 64 * half;         // columns above it are not this row's
        if (!wait.warp(s_full(t & 1), (t >> 1) & 1, 8)) { alive = false; break; }
        tcgen05_fence_after();
        float prob[64];
        if (!idle) {
#pragma unroll
          for (int g = 0; g < 2; ++g) tmem_load_32_issue(s_addr + 32 * g, *reinterpret_cast<uint32_t(*)[32]>(&prob[32 * g]));
#pragma unroll
          for (int g = 0; g < 2; ++g) tmem_load_wait(*reinterpret_cast<uint32_t(*)[32]>(&prob[32 * g]));
#pragma unroll
          for (int e = 0; e < 64; e += 2) {
            const float2 a = fma2(make_float2(prob[e], prob[e + 1]), make_float2(c, c), make_float2(-lse, -lse));
            prob[e] = exp2_approx(a.x);
            prob[e + 1] = exp2_approx(a.y);
          }
        }
        if (j == 0 && t > 0 && !store(w.round - 1)) { alive = false; break; }
        if (!wait.warp(dp_full, t & 1, 8)) { alive = false; break; }
        tcgen05_fence_after();
        if (threadIdx.x == 0) mbar_arrive(v_empty(t % VR));
        if (!idle) {
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            uint32_t x[32], packed[16];
            tmem_load_32(dp_addr + 32 * g, x);
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const float2 slope = mul2(make_float2(prob[32 * g + e], prob[32 * g + e + 1]),
                                        add2(make_float2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), make_float2(-delta, -delta)));
              x[e] = __float_as_uint(slope.x);
              x[e + 1] = __float_as_uint(slope.y);
            }
            if (partial) {
              rare();
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (32 * g + e > limit) x[e] = 0u;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) packed[e] = pack2<T>(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1]));
            tmem_store_16(s_addr + 16 * g, packed);
          }
        }
        if (j * KEYS + all_cols > w.here.length)                   // rows of K behind the document's end
          clear_rows<BOXES>(k_ring + (t % KR) * TILE, w.here.length - j * KEYS, all_cols, threadIdx.x, 256);
        tmem_store_wait();
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(ds_ready);
      }
      dst = row >= 0 ? static_cast<T*>(p.out) + row * p.dim + half * (HD / 2) : nullptr;
      w = following;
      row = next_row;
      lse = next_lse;
      delta = next_delta;
    }
    if (alive && t > 0) store(w.round - 1);
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  settle(abort_flag);
  if (warp == 9) tmem_free(tmem);
}

// ---- host side -------------------------------------------------------------------------
PFN_cuTensorMapEncodeTiled_v12000 encode_function() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult status;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &status) != cudaSuccess ||
        status != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  }();
  return fn;
}

// Boxes of 64 channels x `box_heads` heads x `box_tokens` tokens over [tokens, heads, dim].
int heads_map(CUtensorMap* map, const HeadsView& view, int64_t tokens, int heads, int dim, int box_heads, int box_tokens, int dtype) {
  auto fn = encode_function();
  if (!fn) return fail(CT_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(tokens)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(view.head_stride) * 2, static_cast<cuuint64_t>(view.token_stride) * 2};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_tokens)};
  cuuint32_t elem[3] = {1, 1, 1};
  auto encode = [&] {
    return fn(map, dtype == CT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(view.data),
              dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult rc = encode();
  int device = 0;
  // a host thread (autograd's, say) whose first CUDA call this is has no context bound yet
  if (rc == CUDA_ERROR_INVALID_CONTEXT && cudaGetDevice(&device) == cudaSuccess && cudaSetDevice(device) == cudaSuccess) rc = encode();
  if (rc != CUDA_SUCCESS) return fail(CT_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", (int)rc);
  return CT_OK;
}

bool view_ok(const HeadsView& v) {
  return (reinterpret_cast<uintptr_t>(v.data) & 15) == 0 && v.token_stride > 0 && v.head_stride > 0 && v.token_stride % 8 == 0 &&
         v.head_stride % 8 == 0 && v.token_stride < (int64_t(1) << 38) && v.head_stride < (int64_t(1) << 38);
}
bool address_ok(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int fill(AttentionParams& p, const AttentionArgs& a, PlanSection which) {
  p.items = section(a, which);
  p.out = a.out;
  p.lse = a.lse;
  p.delta = a.delta;
  p.partials = a.partials;
  p.heads = a.heads;
  p.kv_heads = a.kv_heads;
  p.dim = a.head_dim;
  p.packed = packed_heads(a.heads, a.kv_heads);
  p.tile_tokens = 128 / p.packed;
  p.head_blocks = a.heads / p.packed;
  p.scale = a.scale;
  p.error_flag = device_error_flag();
  if (!p.error_flag) return fail(CT_ERR_CUDA, "cannot allocate the device error flag");
  int rc = heads_map(&p.q, a.q, a.tokens, a.heads, a.head_dim, p.packed, p.tile_tokens, a.dtype);
  if (!rc) rc = heads_map(&p.k, a.k, a.tokens, a.kv_heads, a.head_dim, 1, KEYS, a.dtype);
  if (!rc) rc = heads_map(&p.v, a.v, a.tokens, a.kv_heads, a.head_dim, 1, KEYS, a.dtype);
  return rc;
}

int sm_count() {
  static std::atomic<int> counts[64];
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return 1;
  int n = counts[device & 63].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n < 1) n = 1;
    counts[device & 63].store(n, std::memory_order_relaxed);
  }
  return n;
}

// One persistent CTA per SM, or per unit where there are fewer.
template <auto Kernel, bool PERSISTENT>
int launch_tc(const char* name, AttentionParams& p, int64_t units, int threads, int smem, cudaStream_t stream) {
  if (units > 0x3fffffff) return fail(CT_ERR_UNSUPPORTED, "%s: %lld tiles", name, (long long)units);
  static DynamicSmem allowed;
  const int rc = allowed.set(name, reinterpret_cast<const void*>(Kernel), smem);
  if (rc) return rc;
  p.units = static_cast<int>(units);
  Kernel<<<PERSISTENT ? std::min(p.units, sm_count()) : p.units, threads, smem, stream>>>(p);
  count_launch(true);
  return check_launch(name);
}

template <typename T, int HD> int forward(const AttentionArgs& a, AttentionParams& p, cudaStream_t stream) {
  return launch_tc<attention_forward_tc_kernel<T, HD>, true>("attention_forward_tc_kernel", p, a.count[kPlanForward] * p.head_blocks,
                   kForwardThreads, ForwardShape<HD>::kSmem, stream);
}

template <typename T, int HD> int backward(const AttentionArgs& a, cudaStream_t stream) {
  AttentionParams p{};
  int rc = fill(p, a, kPlanQuery);
  const HeadsView dy{a.dy, static_cast<int64_t>(a.heads) * a.head_dim, a.head_dim};
  if (!rc) rc = heads_map(&p.dy, dy, a.tokens, a.heads, a.head_dim, p.packed, p.tile_tokens, a.dtype);
  if (rc) return rc;
  p.dk = a.dk;
  p.dv = a.dv;
  p.out = a.dq;
  rc = launch_tc<attention_query_gradient_tc_kernel<T, HD>, true>("attention_query_gradient_tc_kernel", p,
                 a.count[kPlanQuery] * p.head_blocks, kBackwardThreads, QueryShape<HD>::kSmem, stream);
  if (rc) return rc;
  p.items = section(a, kPlanKeys);
  rc = launch_tc<attention_key_gradient_tc_kernel<T, HD>, false>("attention_key_gradient_tc_kernel", p, a.count[kPlanKeys] * p.kv_heads,
                 kBackwardThreads, KeyShape<HD>::kSmem, stream);
  if (rc || !a.count[kPlanReduce]) return rc;
  p.items = section(a, kPlanReduce);
  const dim3 grid(a.count[kPlanReduce], (128 * a.head_dim / 4 + 255) / 256, 2 * a.kv_heads);
  attention_sum_pieces_kernel<T><<<grid, 256, 0, stream>>>(p);
  count_launch(false);
  return check_launch("attention_sum_pieces_kernel");
}

}  // namespace

// The forward pass takes row maxima of unscaled scores, so the scale has to be positive, and the backward pass divides the
// log-sums by it (Split), so it must not be tiny; other scales go to the shape-generic kernels.
bool scale_ok(const AttentionArgs& a) { return a.scale >= (a.dtype == CT_F16 ? 1e-6f : 1e-20f); }

bool attention_tc_supported(const AttentionArgs& a) {
  return scale_ok(a) && (a.dtype == CT_BF16 || a.dtype == CT_F16) && a.head_dim % 8 == 0 && a.head_dim <= 128 && view_ok(a.q) && view_ok(a.k) &&
         view_ok(a.v) && address_ok(a.out) && address_ok(a.dy) && address_ok(a.dq) && address_ok(a.dk) && address_ok(a.dv);
}

int attention_tc_forward(const AttentionArgs& a, cudaStream_t stream) {
  AttentionParams p{};
  const int rc = fill(p, a, kPlanForward);
  if (rc) return rc;
  if (a.dtype == CT_BF16) return a.head_dim <= 64 ? forward<__nv_bfloat16, 64>(a, p, stream) : forward<__nv_bfloat16, 128>(a, p, stream);
  return a.head_dim <= 64 ? forward<__half, 64>(a, p, stream) : forward<__half, 128>(a, p, stream);
}

int64_t attention_tc_workspace(int64_t key_slots, int kv_heads, int head_dim) { return key_slots * kv_heads * head_dim * 128 * 8; }

int attention_tc_backward(const AttentionArgs& a, cudaStream_t stream) {
  if (a.dtype == CT_BF16) return a.head_dim <= 64 ? backward<__nv_bfloat16, 64>(a, stream) : backward<__nv_bfloat16, 128>(a, stream);
  return a.head_dim <= 64 ? backward<__half, 64>(a, stream) : backward<__half, 128>(a, stream);
}

}  // namespace ct
