// Distillation from a teacher's top logits: the k largest logits of every row
// (with the row's log-sum-exp), and the distillation loss with its gradient.
// Rows are the tokens, columns the vocabulary; logits are bf16, fp16 or fp32,
// all arithmetic is fp32.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>
#include <torch/extension.h>

#include <cfloat>

#include "host_utils.h"
#include "ptx_attn.cuh"

namespace bdion {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTop = 1024;     // entries kept per row
constexpr int kMaxCand = 2048;    // candidates collected per row before ranking
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float as_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float as_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_f(float v) { return v; }

__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }

__device__ __forceinline__ void load8(const __half* p, float* v) {
  uint4 u = *reinterpret_cast<const uint4*>(p);
  const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(h[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void store8(__half* p, const float* v) {
  uint4 u;
  __half2* h = reinterpret_cast<__half2*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = u;
}
using bdion::load8;
using bdion::store8;

__device__ __forceinline__ float warp_sum(float v) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffff, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffff, v, o));
  return v;
}

// Block-wide sum / maximum; every thread gets the result. `buf` holds kWarps
// floats and may be used again once every thread has returned.
__device__ __forceinline__ float block_sum(float v, float* buf) {
  v = warp_sum(v);
  __syncthreads();
  if (threadIdx.x % 32 == 0) buf[threadIdx.x / 32] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) s += buf[i];
  return s;
}
__device__ __forceinline__ float block_max(float v, float* buf) {
  v = warp_max(v);
  __syncthreads();
  if (threadIdx.x % 32 == 0) buf[threadIdx.x / 32] = v;
  __syncthreads();
  float s = buf[0];
#pragma unroll
  for (int i = 1; i < kWarps; ++i) s = fmaxf(s, buf[i]);
  return s;
}

// A running sum of 2^(c * (x - m)) under its running maximum m. The maximum
// starts at the lowest finite float, so a row of -inf sums to 0 and no
// inf - inf arises.
struct RunningSum {
  float m = -FLT_MAX, s = 0.f;
  __device__ __forceinline__ void raise(float to, float c) {
    if (to > m) {
      s *= ex2((m - to) * c);
      m = to;
    }
  }
  __device__ __forceinline__ void add(float x, float c) {
    raise(x, c);
    s += ex2((x - m) * c);
  }
  // over the block: the common maximum and the sum under it
  __device__ __forceinline__ void join(float c, float* buf) {
    const float all = block_max(m, buf);
    s = block_sum(s * ex2((m - all) * c), buf);
    m = all;
  }
};

// Whole number whose order is the float's; -0 ranks as 0, a NaN above all.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// Elements before the first 8-element boundary of row `row` (all of them when
// the tensor's base is not aligned to 8 elements).
__device__ __forceinline__ int row_lead(int64_t row, int64_t ld, int V, bool vec) {
  return vec ? min(V, (int)((8 - (row * ld) % 8) % 8)) : V;
}

__device__ __forceinline__ float pair_max(uint32_t a, uint32_t b, uint32_t c, uint32_t d, __nv_bfloat16) {
  auto h = [](uint32_t x) { return *reinterpret_cast<const __nv_bfloat162*>(&x); };
  const float2 f = __bfloat1622float2(__hmax2(__hmax2(h(a), h(b)), __hmax2(h(c), h(d))));
  return fmaxf(f.x, f.y);
}
__device__ __forceinline__ float pair_max(uint32_t a, uint32_t b, uint32_t c, uint32_t d, __half) {
  auto h = [](uint32_t x) { return *reinterpret_cast<const __half2*>(&x); };
  const float2 f = __half22float2(__hmax2(__hmax2(h(a), h(b)), __hmax2(h(c), h(d))));
  return fmaxf(f.x, f.y);
}

// Eight elements as they lie in memory.
template <typename T>
struct Raw8 {
  uint4 u[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) u[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  }
  // the last use of these bytes: first to leave the caches
  __device__ __forceinline__ void load_last(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) u[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  }
  // eight elements at any alignment
  __device__ __forceinline__ void load_single(const T* p) {
#pragma unroll
    for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(u)[i] = p[i];
  }
  __device__ __forceinline__ float max() const {  // NaN are left out
    if constexpr (sizeof(T) == 2) {
      return pair_max(u[0].x, u[0].y, u[0].z, u[0].w, T{});
    } else {
      const float* v = reinterpret_cast<const float*>(u);
      return fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
    }
  }
  __device__ __forceinline__ void get(float* v) const { load8(reinterpret_cast<const T*>(u), v); }
};


// ------------------------------------------------------------ top logits
__device__ __forceinline__ float key_float(uint32_t key) {  // the float that order_key took (not for NaN)
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// Largest threshold that at least k of the keys reach (R per lane of one warp, or
// per thread of the block), bit by bit; stops early where exactly k do.
template <int R, bool BLOCK>
__device__ __forceinline__ uint32_t kth_key(const uint32_t (&key)[R], int k) {
  uint32_t thr = 0;
#pragma unroll 1
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t t = thr | (1u << bit);
    int cnt = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) cnt += BLOCK ? __syncthreads_count(key[i] >= t) : key[i] >= t;
    if (!BLOCK) cnt = __reduce_add_sync(0xffffffffu, cnt);
    if (cnt >= k) thr = t;
    if (cnt == k) break;
  }
  return thr;
}

// One block per row, in one pass over it and a sample. The sample (`ns` of the
// row's rounds of kThreads groups, spread evenly) gives the maximum of each of
// kThreads * G sets of columns; the k-th largest of those bounds the row's k-th
// largest logit from below. The pass then takes the log-sum-exp and collects
// the columns above that bound: a group's maximum decides for eight columns at
// once. The host takes ns so that about 256 come together. A candidate's rank
// is the number of larger ones (value, then the lower index), counted after a
// second bound has thinned them out. Rows with too many candidates (equal
// values; also checked: too few), and rows with a NaN or +inf, take the exact
// threshold over the whole row bit by bit and keep the lowest indices of the equal ones.
// 4096 x 128256 bf16, k = 64: 379 us, 2.8 TB/s (161 us at the copy rate); the same in
// fp32 behind a head's product 514 us; 1500 x 50009 fp32, k = 200: 140 us. Bound by
// instructions (70 % of the issue slots) and by the steps in which one warp searches for
// a bound while the row's others wait; three rows to an SM (two in fp32, whose groups
// take twice the registers) overlap these. Two full passes took 576 us, a sample of half
// the size (twice the candidates) 601 us where this took 534.
// Beyond 256 entries the sample is the whole row: k = 300 at 4096 x 128256 bf16 takes 563
// us. Where the candidates' buffer then overflows, most of all in small vocabularies, the
// rows take the exact way: 4096 x 4096 at k = 512 610 us, at k = 1024 1157 us, 4096 x
// 32768 at k = 1024 1506 us, against 504 us for 1024 x 128256 at k = 1024.
template <typename T, int G>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 3 : 2)
    top_logits_kernel(const T* __restrict__ logits, int64_t ld, int V, int k, bool vec, int ns, float inv_tau,
                      float c, float* __restrict__ values, int64_t* __restrict__ indices, float* __restrict__ lse) {
  __shared__ float red[kWarps];
  __shared__ uint32_t s_max[kThreads * G];
  __shared__ uint64_t s_cand[2][kMaxCand];
  // candidates, and those behind the second bound: a place of its own, so that no thread
  // clears the first count while another has yet to read it
  __shared__ int s_n, s_left;
  __shared__ uint32_t s_thr;
  const int64_t row = blockIdx.x;
  const T* x = logits + row * ld;
  const int tid = threadIdx.x;
  const int lead = vec ? row_lead(row, ld, V, true) : 0;
  const int n8 = (V - lead) / 8, tail0 = lead + n8 * 8, rounds = (n8 + kThreads - 1) / kThreads;
  // a row whose lead takes its last group may have a round less than the host counted; a
  // round that was sampled twice would put its columns into two of the sets
  ns = min(ns, max(rounds, 1));
  auto load = [&](int g, Raw8<T>& r) {
    if (vec)
      r.load(x + lead + g * 8);
    else
      r.load_single(x + g * 8);
  };
  // columns outside the groups, one per thread
  const int end_col = tid < 8 ? (tid < lead ? tid : -1) : (tid < 16 && tail0 + tid - 8 < V ? tail0 + tid - 8 : -1);
  const float end_z = end_col >= 0 ? as_f(x[end_col]) : -INFINITY;

  // the sample's bound
  float best[G];
#pragma unroll
  for (int i = 0; i < G; ++i) best[i] = -INFINITY;
  for (int j = 0; j < ns; j += 4) {
    Raw8<T> r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int g = (j + i) * rounds / ns * kThreads + tid;
      if (j + i < ns && g < n8) load(g, r[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int g = (j + i) * rounds / ns * kThreads + tid;
      if (j + i < ns && g < n8) best[i % G] = fmaxf(best[i % G], r[i].max());
    }
  }
#pragma unroll
  for (int i = 0; i < G; ++i) s_max[tid * G + i] = best[i] == -INFINITY ? 0u : order_key(best[i]);
  if (tid == 0) s_n = s_left = 0;
  __syncthreads();
  if (G == 1) {
    if (tid < 32) {
      uint32_t keys[kThreads / 32];
#pragma unroll
      for (int i = 0; i < kThreads / 32; ++i) keys[i] = s_max[i * 32 + tid];
      const uint32_t t = kth_key<kThreads / 32, false>(keys, k);
      if (tid == 0) s_thr = t;
    }
  } else {
    uint32_t keys[G];
#pragma unroll
    for (int i = 0; i < G; ++i) keys[i] = s_max[i * kThreads + tid];
    const uint32_t t = kth_key<G, true>(keys, k);
    if (tid == 0) s_thr = t;
  }
  __syncthreads();
  uint32_t thr = s_thr;
  const float thr_f = thr == 0 ? -INFINITY : key_float(thr);
  auto collect_one = [&](float v, int col) {
    const int at = atomicAdd(&s_n, 1);
    if (at < kMaxCand) s_cand[0][at] = ((uint64_t)order_key(v) << 32) | (uint32_t)~(uint32_t)col;
  };

  // the pass
  RunningSum sum;
  for (int j = 0; j < rounds; j += 4) {
    Raw8<T> r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int g = (j + i) * kThreads + tid;
      if (g < n8) load(g, r[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int g = (j + i) * kThreads + tid;
      if (g < n8) {
        float v[8];
        r[i].get(v);
        const float vm = r[i].max();
        sum.raise(vm, c);
        const f2 neg_m = make_f2(-sum.m, -sum.m), c2 = make_f2(c, c);
        f2 s2 = make_f2(0.f, 0.f);
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const f2 z = mul2(add2(make_f2(v[e], v[e + 1]), neg_m), c2);
          s2 = add2(s2, make_f2(ex2(lo_of(z)), ex2(hi_of(z))));
        }
        sum.s += lo_of(s2) + hi_of(s2);
        if (vm >= thr_f) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (v[e] >= thr_f) collect_one(v[e], lead + g * 8 + e);
        }
      }
    }
  }
  if (end_col >= 0) {
    sum.add(end_z, c);
    if (end_z >= thr_f) collect_one(end_z, end_col);
  }
  sum.join(c, red);  // its barriers also end the collection
  int n = s_n;
  int from = 0;
  const bool special = !(sum.s <= FLT_MAX) || !(sum.m <= FLT_MAX);  // a NaN or +inf somewhere
  // (m * c would overflow for a row that is masked throughout by the type's lowest value)
  if (!special && tid == 0) lse[row] = sum.m * inv_tau + logf(sum.s);
  if (n > kMaxCand || n < k || special) {
    auto for_all = [&](auto f) {
      for (int col = tid; col < V; col += kThreads) f(col, order_key(as_f(x[col])));
    };
    // exact threshold: the largest one that at least k logits reach
    thr = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t t = thr | (1u << bit);
      int cnt = 0;
      for_all([&](int, uint32_t key) { cnt += key >= t; });
      __syncthreads();
      if (tid == 0) s_n = 0;
      __syncthreads();
      cnt = __reduce_add_sync(0xffffffffu, cnt);
      if (tid % 32 == 0) atomicAdd(&s_n, cnt);
      __syncthreads();
      if (s_n >= k) thr = t;
    }
    __syncthreads();
    if (tid == 0) s_n = 0;
    __syncthreads();
    // those above it, fewer than k
    for_all([&](int col, uint32_t key) {
      if (key > thr) s_cand[0][atomicAdd(&s_n, 1)] = ((uint64_t)key << 32) | (uint32_t)~(uint32_t)col;
    });
    __syncthreads();
    // the equal ones in the order of their indices, as many as are wanted
    int have = s_n;
    __syncthreads();
    for (int c0 = 0; c0 < V && have < k; c0 += kThreads) {
      const int col = c0 + tid;
      const bool eq = col < V && order_key(as_f(x[col])) == thr;
      const uint32_t votes = __ballot_sync(0xffffffffu, eq);
      if (tid % 32 == 0) s_max[tid / 32] = __popc(votes);
      __syncthreads();
      int before = have, all = 0;
      for (int w = 0; w < kWarps; ++w) {
        if (w < tid / 32) before += s_max[w];
        all += s_max[w];
      }
      before += __popc(votes & ((1u << (tid % 32)) - 1u));
      if (eq && before < k) s_cand[0][before] = ((uint64_t)thr << 32) | (uint32_t)~(uint32_t)col;
      have += all;
      __syncthreads();
    }
    n = min(have, k);
  } else if (n > 2 * k && n > 128) {
    // a second bound, now over the candidates
    if (n <= kThreads) {
      if (tid < 32) {
        uint32_t keys[kThreads / 32];
#pragma unroll
        for (int i = 0; i < kThreads / 32; ++i)
          keys[i] = i * 32 + tid < n ? (uint32_t)(s_cand[0][i * 32 + tid] >> 32) : 0u;
        const uint32_t t = kth_key<kThreads / 32, false>(keys, k);
        if (tid == 0) s_thr = t;
      }
    } else {
      uint32_t keys[kMaxCand / kThreads];
#pragma unroll
      for (int i = 0; i < kMaxCand / kThreads; ++i)
        keys[i] = i * kThreads + tid < n ? (uint32_t)(s_cand[0][i * kThreads + tid] >> 32) : 0u;
      const uint32_t t = kth_key<kMaxCand / kThreads, true>(keys, k);
      if (tid == 0) s_thr = t;
    }
    __syncthreads();
    thr = s_thr;
    for (int i = tid; i < n; i += kThreads) {
      const uint64_t cand = s_cand[0][i];
      if ((uint32_t)(cand >> 32) >= thr) s_cand[1][atomicAdd(&s_left, 1)] = cand;
    }
    __syncthreads();
    n = s_left;
    from = 1;
  }
  for (int i = tid; i < n; i += kThreads) {
    const uint64_t mine = s_cand[from][i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += s_cand[from][j] > mine;
    if (rank < k) {
      const int col = (int)~(uint32_t)mine;
      values[row * k + rank] = as_f(x[col]);
      indices[row * k + rank] = col;
      // a NaN makes the sum one, +inf without a NaN makes it +inf
      if (special && rank == 0) lse[row] = (uint32_t)(mine >> 32) == 0xffffffffu ? NAN : as_f(x[col]);
    }
  }
}

// ------------------------------------------------------------ distillation loss
struct DistillArgs {
  const int64_t* labels;  // may be null
  const float* top_values;
  const void* top_indices;
  bool idx64;
  const float* top_lse;   // may be null: the teacher's entries alone are normalised
  float* row_loss;
  int64_t ld_in, ld_out;
  int V, k;
  bool vec;
  float inv_tau, alpha, tau, grad_scale;
};

// How the label's softmax (temperature 1) is taken beside the teacher's: not at
// all (the same, or no labels); as the square of the teacher's exponentials at
// temperature 2, 2^(x log2e) = (2^(x log2e / 2))^2; as their third or fourth power
// or by exponentials of its own.
enum HardMode { kHardNone, kHardSquare, kHardOther };

// One block per row, which it reads twice (the second time mostly from L2):
//   p_j   teacher's probability of entry j (of the whole vocabulary when its
//         log-sum-exp is given, p_rest = 1 - sum p; else of the k entries)
//   q     student's softmax(z / tau); q_rest its sum outside the entries
//   loss  (1 - alpha) CE(z, label) + alpha tau^2 [sum p_j log(p_j / q_j) + p_rest log(p_rest / q_rest)]
//   grad  grad_scale * dloss/dz, in the second pass
// The entries' columns are marked in a bitmap, so that the sum over the rest
// is taken directly (1 - sum q_j would cancel when the student is sure) and
// keeps a maximum of its own. 4096 x 128256 bf16 at temperature 2 with labels:
// 495 us, 4.2 TB/s of the bytes that have to move (322 us at the copy rate); 512 us in
// passes repeated for over a second (1822 MHz). fp32 logits: 2048 x 128256 with an fp32
// gradient 493 us at 1725 MHz, 4096 x 128256 with a bf16 one 907 us within linear
// distillation (1522 MHz). No unit is full (58 % of the issue slots and of DRAM): the
// two passes of a row with sums between them, two rows to an SM, leave latency. Holding
// a row in the registers of a cluster of four blocks, so that it is read once, took 714
// us at best: its blocks wait for one another's sums with nothing else to do.
template <typename T, typename TG, int MODE>
__global__ void __launch_bounds__(kThreads, 2)
    distill_kernel(const T* __restrict__ logits, TG* __restrict__ grad, const DistillArgs a) {
  constexpr bool both = MODE != kHardNone;
  constexpr int U = sizeof(T) == 2 ? 4 : 2;  // groups in flight per thread
  extern __shared__ uint32_t bitmap[];       // a byte per group of 8 columns; the row's ends behind them
  __shared__ float red[kWarps];
  __shared__ float s_p[kMaxTop], s_z[kMaxTop];
  __shared__ int s_i[kMaxTop];
  __shared__ int s_marked, s_twice;
  const int64_t row = blockIdx.x;
  const int V = a.V, tid = threadIdx.x;
  const T* x = logits + row * a.ld_in;
  TG* gx = grad + row * a.ld_out;
  const bool vec = a.vec;
  const int lead = vec ? row_lead(row, a.ld_in, V, true) : 0;
  const int n8 = (V - lead) / 8, tail0 = lead + n8 * 8;
  // columns outside the groups, one per thread
  const int end_col = tid < 8 ? (tid < lead ? tid : -1) : (tid < 16 && tail0 + tid - 8 < V ? tail0 + tid - 8 : -1);
  auto store = [&](int g, const float (&v)[8]) {
    TG* to = gx + lead + g * 8;
    if (vec) {
      store8(to, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) put(to + e, v[e]);
    }
  };
  const int64_t label = a.labels ? a.labels[row] : 0;
  if (label < 0 || label >= V) {  // takes no part
    const float zero[8] = {};
    if (tid == 0) a.row_loss[row] = 0.f;
    if (grad == nullptr) return;
    for (int g = tid; g < n8; g += kThreads) store(g, zero);
    if (end_col >= 0) put(gx + end_col, 0.f);
    return;
  }
  const bool hard = a.labels != nullptr && a.alpha != 1.f;
  const float c = a.inv_tau * kLog2e;
  const float end_z = end_col >= 0 ? as_f(x[end_col]) : -INFINITY;
  const float zy = hard ? as_f(x[label]) : 0.f;
  // bit of a column: groups in order, then the 16 places of the ends
  auto bit_of = [&](int col) {
    return col < lead ? n8 * 8 + col : col >= tail0 ? n8 * 8 + 8 + col - tail0 : col - lead;
  };
  auto is_marked = [&](int col) {
    const int bit = bit_of(col);
    return ((bitmap[bit >> 5] >> (bit & 31)) & 1u) != 0;
  };

  for (int i = tid; i < (n8 * 8 + 16 + 31) / 32; i += kThreads) bitmap[i] = 0;
  if (tid == 0) s_marked = s_twice = 0;
  __syncthreads();
  // the teacher's entries
  float tmax = -FLT_MAX;
  for (int j = tid; j < a.k; j += kThreads) {
    const int64_t i = a.idx64 ? static_cast<const int64_t*>(a.top_indices)[row * a.k + j]
                              : static_cast<const int*>(a.top_indices)[row * a.k + j];
    const bool in = i >= 0 && i < V;
    const float t = a.top_values[row * a.k + j];
    s_i[j] = in ? (int)i : -1;
    s_p[j] = in ? t : -INFINITY;
    if (in) {
      s_z[j] = as_f(x[i]);
      const int bit = bit_of((int)i);
      const uint32_t m = 1u << (bit & 31);
      if (atomicOr(&bitmap[bit >> 5], m) & m)
        s_twice = 1;
      else
        atomicAdd(&s_marked, 1);
      tmax = fmaxf(tmax, t);
    }
  }
  // log p = (t - tref) / tau - tlog of an entry t. Without a log-sum-exp tref is the
  // entries' maximum: the softmax does not know an offset that all of them have, and a
  // sum tref / tau + tlog would round the second term away where the first is large (at
  // the type's lowest value altogether).
  float tref = 0.f, tlog;
  if (a.top_lse != nullptr) {
    tlog = a.top_lse[row];
  } else {
    tref = block_max(tmax, red);
    float s = 0.f;
    for (int j = tid; j < a.k; j += kThreads)
      if (s_i[j] >= 0) s += ex2((s_p[j] - tref) * c);
    s = block_sum(s, red);
    tlog = logf(s);  // -inf without entries; s_p stays -inf there and gives p = 0 below
  }
  auto log_p = [&](float t) { return (t - tref) * a.inv_tau - tlog; };
  __syncthreads();

  // y = 2^(c (z - ref)) of the teacher's softmax -> the label's
  auto full_of = [&](float y, float z, float ref) {
    if (MODE == kHardSquare) return y * y;
    return a.tau == 3.f ? y * y * y : a.tau == 4.f ? (y * y) * (y * y) : ex2((z - ref) * kLog2e);
  };
  // columns in the set count as -inf in the first pass
  auto strike = [&](int g, float (&v)[8]) {
    const uint32_t marks = reinterpret_cast<const uint8_t*>(bitmap)[g];
    if (marks) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if ((marks >> e) & 1u) v[e] = -INFINITY;
    }
    return marks;
  };
  // the rest's maximum m, sum of 2^(c (z - m)), and that at temperature 1
  float m = -FLT_MAX, rest = 0.f, full = 0.f;
  auto raise = [&](float to) {
    if (to > m) {
      const float f = ex2((m - to) * c);
      rest *= f;
      if (both) full *= full_of(f, m, to);
      m = to;
    }
  };
  for (int j = tid; j < n8; j += U * kThreads) {
    Raw8<T> r[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (j + i * kThreads < n8) {
        if (vec)
          r[i].load(x + lead + (j + i * kThreads) * 8);
        else
          r[i].load_single(x + (j + i * kThreads) * 8);
      }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int g = j + i * kThreads;
      if (g >= n8) break;
      float v[8];
      r[i].get(v);
      if (strike(g, v)) {
        float vm = v[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) vm = fmaxf(vm, v[e]);
        raise(vm);
      } else {
        raise(r[i].max());
      }
      const f2 neg_m = make_f2(-m, -m), c2 = make_f2(c, c);
      f2 s2 = make_f2(0.f, 0.f), f2s = s2;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const f2 z = mul2(add2(make_f2(v[e], v[e + 1]), neg_m), c2);
        const f2 y = make_f2(ex2(lo_of(z)), ex2(hi_of(z)));
        s2 = add2(s2, y);
        if (MODE == kHardSquare) f2s = fma2(y, y, f2s);
        if (MODE == kHardOther) f2s = add2(f2s, make_f2(full_of(lo_of(y), v[e], m), full_of(hi_of(y), v[e + 1], m)));
      }
      rest += lo_of(s2) + hi_of(s2);
      if (both) full += lo_of(f2s) + hi_of(f2s);
    }
  }
  const bool end_rest = end_col >= 0 && !is_marked(end_col);
  if (end_rest) {
    raise(end_z);
    const float y = ex2((end_z - m) * c);
    rest += y;
    if (both) full += full_of(y, end_z, m);
  }
  const float rm = block_max(m, red);
  {
    const float f = ex2((m - rm) * c);
    rest = block_sum(rest * f, red);
    if (both) full = block_sum(full * full_of(f, m, rm), red);
  }

  // the set's own part of the student's sums
  const bool twice = s_twice != 0;
  auto first_of = [&](int j) {  // whether entry j is the first with its column
    if (twice)
      for (int i = 0; i < j; ++i)
        if (s_i[i] == s_i[j]) return false;
    return true;
  };
  float zmax = -FLT_MAX;
  for (int j = tid; j < a.k; j += kThreads)
    if (s_i[j] >= 0) zmax = fmaxf(zmax, s_z[j]);
  const float top = fmaxf(block_max(zmax, red), rm);
  float set = 0.f, setf = 0.f, psum = 0.f, cross = 0.f;  // the last: sum p (log p - (z - top) / tau)
  for (int j = tid; j < a.k; j += kThreads)
    if (s_i[j] >= 0) {
      const float lp = log_p(s_p[j]), p = s_p[j] == -INFINITY ? 0.f : ex2(lp * kLog2e);
      psum += p;
      if (p != 0.f) cross += p * (lp - (s_z[j] - top) * a.inv_tau);
      if (first_of(j)) {
        const float y = ex2((s_z[j] - top) * c);
        set += y;
        if (both) setf += full_of(y, s_z[j], top);
      }
    }
  set = block_sum(set, red);
  psum = block_sum(psum, red);
  cross = block_sum(cross, red);
  const float to_top = ex2((rm - top) * c);
  const float B = set + rest * to_top;
  float F = 0.f, to_top_full = 0.f;
  if (both) {
    to_top_full = ex2((rm - top) * kLog2e);
    F = block_sum(setf, red) + full * to_top_full;
  }
  const bool has_rest = a.top_lse != nullptr && s_marked < V;
  const float p_rest = has_rest ? fmaxf(1.f - psum, 0.f) : 0.f;
  const float q_set = set / B;
  if (tid == 0) {
    // all logits relative to the largest one: the loss does not know a common offset
    const float logB = logf(B);  // log of the sum of exp((z - top) / tau)
    float kl = psum != 0.f ? cross + psum * logB : 0.f;
    if (p_rest > 0.f) {
      // log(p_rest / q_rest); where the set holds little, from the set's two sums, whose
      // roundings are far smaller than those of two numbers near 1
      const float log_ratio = q_set < 0.5f && psum < 0.5f
                                  ? log1pf(-psum) - log1pf(-q_set)
                                  : logf(p_rest) - ((rm - top) * a.inv_tau + logf(rest) - logB);
      kl += p_rest * log_ratio;
    }
    a.row_loss[row] = (a.alpha > 0.f ? a.alpha * a.tau * a.tau * kl : 0.f) +
                      (hard ? (1.f - a.alpha) * ((both ? logf(F) : logB) + (top - zy)) : 0.f);
  }
  if (grad == nullptr) return;

  // gradient. In the set: w_hard softmax(z) + w_soft (mass q - p), mass = sum p + p_rest,
  // which is not 1 where the entries hold more than all (columns that come twice), or less
  // over the whole vocabulary. Outside: w_hard softmax(z) + w_soft q (1 - p_rest / q_rest)
  // if there is a rest, where 1 - p_rest / q_rest = (psum - q_set) / q_rest: at a high
  // temperature the set holds little on either side, and the difference of two numbers near
  // 1 would keep few bits
  const float w_soft = a.grad_scale * a.alpha * a.tau;
  const float mass = p_rest > 0.f ? 1.f : psum;
  const float w_hard = hard ? a.grad_scale * (1.f - a.alpha) : 0.f;
  const float inv_B = 1.f / B, inv_F = both ? 1.f / F : inv_B;
  // factors of 2^(c (z - rm)), the first of them the teacher's part alone, and of 2^(log2e (z - rm))
  float f_soft = 0.f, f_rest = 0.f, f_full = 0.f;
  if (rest > 0.f || rest != rest) {
    f_soft = w_soft * (p_rest > 0.f ? (psum - q_set) / rest : mass * to_top * inv_B);
    f_rest = f_soft + (both ? 0.f : w_hard * to_top * inv_B);
    f_full = both ? w_hard * to_top_full * inv_F : 0.f;
  }
  const f2 neg_m = make_f2(-rm, -rm), c2 = make_f2(c, c), fr2 = make_f2(f_rest, f_rest), ff2 = make_f2(f_full, f_full);
  for (int j = tid; j < n8; j += U * kThreads) {
    Raw8<T> r[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (j + i * kThreads < n8) {
        if (vec)
          r[i].load_last(x + lead + (j + i * kThreads) * 8);
        else
          r[i].load_single(x + (j + i * kThreads) * 8);
      }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int g = j + i * kThreads;
      if (g >= n8) break;
      float v[8];
      r[i].get(v);
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const f2 z = mul2(add2(make_f2(v[e], v[e + 1]), neg_m), c2);
        const f2 y = make_f2(ex2(lo_of(z)), ex2(hi_of(z)));
        f2 o;
        if (MODE == kHardNone)
          o = mul2(fr2, y);
        else if (MODE == kHardSquare)
          o = mul2(y, fma2(y, ff2, fr2));
        else
          o = fma2(ff2, make_f2(full_of(lo_of(y), v[e], rm), full_of(hi_of(y), v[e + 1], rm)), mul2(fr2, y));
        v[e] = lo_of(o);
        v[e + 1] = hi_of(o);
      }
      store(g, v);
    }
  }
  if (end_col >= 0) {
    const float y = ex2((end_z - rm) * c);
    put(gx + end_col, both ? f_rest * y + f_full * full_of(y, end_z, rm) : f_rest * y);
  }
  __syncthreads();
  // the set's columns and the label's
  auto soft_at = [&](float z) { return ex2((z - top) * c) * inv_B; };
  auto hard_at = [&](float z) { return both ? ex2((z - top) * kLog2e) * inv_F : soft_at(z); };
  for (int j = tid; j < a.k; j += kThreads) {
    const int i = s_i[j];
    if (i < 0 || !first_of(j)) continue;
    float p = 0.f;
    for (int e = j; e < (twice ? a.k : j + 1); ++e)
      if (s_i[e] == i && s_p[e] != -INFINITY) p += ex2(log_p(s_p[e]) * kLog2e);
    float g = w_soft * (mass * soft_at(s_z[j]) - p);
    if (hard) g += w_hard * (hard_at(s_z[j]) - (i == label ? 1.f : 0.f));
    put(gx + i, g);
  }
  if (hard && tid == 0 && !is_marked((int)label)) {
    put(gx + label, f_soft * ex2((zy - rm) * c) + w_hard * (hard_at(zy) - 1.f));
  }
}

// out = x * f[0], rounded once
template <typename TO>
__global__ void __launch_bounds__(256) scale_cast_kernel(const float* __restrict__ x, const float* __restrict__ f,
                                                         TO* __restrict__ out, int64_t n) {
  const float s = *f;
  const int64_t step = (int64_t)gridDim.x * 256;
  int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  for (; i < n / 8; i += step) {
    float v[8];
    load8(x + i * 8, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= s;
    store8(out + i * 8, v);
  }
  if (blockIdx.x == 0 && (int)threadIdx.x < n % 8) put(out + n / 8 * 8 + threadIdx.x, x[n / 8 * 8 + threadIdx.x] * s);
}

bool aligned8(const at::Tensor& t) {
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % (8 * t.element_size()) == 0;
}

void check_rows(const at::Tensor& t, const char* op) {
  TORCH_CHECK(t.is_cuda() && t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1),
              "dion_b200 ", op, ": logits [T, V] on a CUDA device with contiguous rows");
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf || t.scalar_type() == at::kFloat,
              "dion_b200 ", op, ": bf16, fp16 or fp32 logits");
  TORCH_CHECK(t.size(0) < (1ll << 28) && t.size(1) >= 1 && t.size(1) <= (1 << 20), "dion_b200 ", op,
              ": 1 <= V <= 2^20 and T < 2^28");
}

void check_out(const at::Tensor& t, const at::Tensor& like, at::ScalarType dtype, at::IntArrayRef shape,
               const char* what) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.scalar_type() == dtype && t.sizes() == shape &&
                  t.is_contiguous(),
              "dion_b200 ", what, ": a contiguous tensor of the stated shape and type on the logits' device");
}

template <typename F>
void by_type(at::ScalarType t, F f) {
  if (t == at::kBFloat16)
    f(__nv_bfloat16{});
  else if (t == at::kHalf)
    f(__half{});
  else
    f(float{});
}

}  // namespace

// values / indices [T, k]: the k largest logits of each row in falling order
// (equal ones by the lower index); lse [T]: log sum exp(logits / tau)
void top_logits(const at::Tensor& logits, at::Tensor& values, at::Tensor& indices, at::Tensor& lse, double tau) {
  check_rows(logits, "top_logits");
  const int64_t T = logits.size(0);
  const int V = (int)logits.size(1), k = (int)values.size(1);
  TORCH_CHECK(k >= 1 && k <= std::min(V, kMaxTop), "dion_b200 top_logits: 1 <= k <= min(V, 1024)");
  TORCH_CHECK(tau >= 1e-18 && tau <= 1e18, "dion_b200 top_logits: temperature > 0 (1e-18 to 1e18)");
  check_out(values, logits, at::kFloat, {T, k}, "top_logits values");
  check_out(indices, logits, at::kLong, {T, k}, "top_logits indices");
  check_out(lse, logits, at::kFloat, {T}, "top_logits lse");
  if (T == 0) return;
  c10::cuda::CUDAGuard guard(logits.device());
  auto s = at::cuda::getCurrentCUDAStream();
  by_type(logits.scalar_type(), [&](auto tag) {
    using E = decltype(tag);
    // rounds in the sample: about 256 columns reach its bound, or more than k where k is larger
    const int rounds = (V / 8 + kThreads - 1) / kThreads;
    const int ns = std::max(1, std::min(rounds, (rounds * k + 255) / 256));
    auto launch = [&](auto g) {
      top_logits_kernel<E, decltype(g)::value><<<(unsigned)T, kThreads, 0, s>>>(
          static_cast<const E*>(logits.data_ptr()), logits.stride(0), V, k, aligned8(logits), ns, (float)(1 / tau),
          (float)(kLog2e / tau), values.data_ptr<float>(), indices.data_ptr<int64_t>(), lse.data_ptr<float>());
    };
    // at least twice as many sets as entries, where the row has that many groups, keeps the
    // candidates near 1.4 k
    if (k <= kThreads / 2)
      launch(std::integral_constant<int, 1>{});
    else
      launch(std::integral_constant<int, 4>{});
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  note_launch();
}

// loss: the sum of the rows' losses; grad (optional): grad_scale * d loss / d logits
void distill_fwd_bwd(const at::Tensor& logits, const c10::optional<at::Tensor>& labels, const at::Tensor& top_values,
                     const at::Tensor& top_indices, const c10::optional<at::Tensor>& top_lse,
                     const c10::optional<at::Tensor>& grad, at::Tensor& loss, double tau, double alpha, double grad_scale) {
  check_rows(logits, "distill");
  const int64_t T = logits.size(0);
  const int V = (int)logits.size(1), k = (int)top_values.size(1);
  TORCH_CHECK(k >= 1 && k <= kMaxTop, "dion_b200 distill: 1 to 1024 teacher entries per row");
  TORCH_CHECK(tau >= 1e-18 && tau <= 1e18, "dion_b200 distill: temperature > 0 (1e-18 to 1e18)");
  check_out(top_values, logits, at::kFloat, {T, k}, "distill top_values");
  TORCH_CHECK(top_indices.scalar_type() == at::kLong || top_indices.scalar_type() == at::kInt,
              "dion_b200 distill: int32 or int64 top_indices");
  check_out(top_indices, logits, top_indices.scalar_type(), {T, k}, "distill top_indices");
  if (labels.has_value()) check_out(*labels, logits, at::kLong, {T}, "distill labels");
  if (top_lse.has_value()) check_out(*top_lse, logits, at::kFloat, {T}, "distill top_lse");
  const auto gtype = grad.has_value() ? grad->scalar_type() : logits.scalar_type();
  if (grad.has_value()) {
    TORCH_CHECK(gtype == logits.scalar_type() ||
                    (logits.scalar_type() == at::kFloat && (gtype == at::kBFloat16 || gtype == at::kHalf)),
                "dion_b200 distill: gradient in the logits' type, or bf16 or fp16 of fp32 logits");
    check_out(*grad, logits, gtype, {T, V}, "distill grad");
  }
  c10::cuda::CUDAGuard guard(logits.device());
  if (T == 0) {
    loss.zero_();
    return;
  }
  auto rows = at::empty({T}, logits.options().dtype(at::kFloat));
  DistillArgs a;
  a.labels = labels.has_value() ? labels->data_ptr<int64_t>() : nullptr;
  a.top_values = top_values.data_ptr<float>();
  a.top_indices = top_indices.data_ptr();
  a.idx64 = top_indices.scalar_type() == at::kLong;
  a.top_lse = top_lse.has_value() ? top_lse->data_ptr<float>() : nullptr;
  a.row_loss = rows.data_ptr<float>();
  a.ld_in = logits.stride(0);
  a.ld_out = V;
  a.V = V;
  a.k = k;
  // 8-element groups of the logits and of the gradient have to start together
  a.vec = aligned8(logits) && (!grad.has_value() || (aligned8(*grad) && (T == 1 || a.ld_in % 8 == a.ld_out % 8)));
  a.inv_tau = (float)(1.0 / tau);
  a.tau = (float)tau;
  a.alpha = (float)alpha;
  a.grad_scale = (float)grad_scale;
  const size_t smem = ((size_t)V + 16 + 31) / 32 * 4;
  auto s = at::cuda::getCurrentCUDAStream();
  by_type(logits.scalar_type(), [&](auto tag) {
    using E = decltype(tag);
    by_type(gtype, [&](auto gtag) {
      using G = decltype(gtag);
      if constexpr (std::is_same_v<E, G> || std::is_same_v<E, float>) {
        auto run = [&](auto mode) {
          auto kern = distill_kernel<E, G, decltype(mode)::value>;
          C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
          kern<<<(unsigned)T, kThreads, smem, s>>>(static_cast<const E*>(logits.data_ptr()),
                                                   grad.has_value() ? static_cast<G*>(grad->data_ptr()) : nullptr, a);
        };
        if (!a.labels || a.alpha == 1.f || a.tau == 1.f)
          run(std::integral_constant<int, kHardNone>{});
        else if (a.tau == 2.f)
          run(std::integral_constant<int, kHardSquare>{});
        else
          run(std::integral_constant<int, kHardOther>{});
      }
    });
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  note_launch();
  at::sum_out(loss, rows, 0);
}

// out (bf16, fp16 or fp32) = x (fp32) * f (one fp32 value on the device)
void scale_cast(const at::Tensor& x, const at::Tensor& f, at::Tensor& out) {
  TORCH_CHECK(x.is_cuda() && x.scalar_type() == at::kFloat && x.is_contiguous() && aligned8(x) && f.numel() == 1 &&
                  f.scalar_type() == at::kFloat && f.device() == x.device(),
              "dion_b200 scale_cast: contiguous fp32 x and one fp32 factor on one CUDA device");
  TORCH_CHECK(out.scalar_type() == at::kBFloat16 || out.scalar_type() == at::kHalf || out.scalar_type() == at::kFloat,
              "dion_b200 scale_cast: bf16, fp16 or fp32 out");
  check_out(out, x, out.scalar_type(), x.sizes(), "scale_cast out");
  TORCH_CHECK(aligned8(out), "dion_b200 scale_cast: out aligned to 8 elements");
  if (x.numel() == 0) return;
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t blocks = (x.numel() / 8 + 255) / 256;
  by_type(out.scalar_type(), [&](auto tag) {
    using E = decltype(tag);
    scale_cast_kernel<E><<<(unsigned)std::max<int64_t>(1, std::min<int64_t>(blocks, 148 * 16)), 256, 0,
                           at::cuda::getCurrentCUDAStream()>>>(x.data_ptr<float>(), f.data_ptr<float>(),
                                                               static_cast<E*>(out.data_ptr()), x.numel());
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  note_launch();
}

}  // namespace bdion
