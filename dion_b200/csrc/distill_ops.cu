// Distillation from a teacher's top logits: the k largest logits of every row
// (with the row's log-sum-exp), and the distillation loss with its gradient.
// Rows are the tokens, columns the vocabulary; logits are bf16, fp16 or fp32,
// all arithmetic is fp32.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <torch/extension.h>

#include <cfloat>
#include <map>
#include <mutex>
#include <tuple>

#include "host_utils.h"
#include "ptx_attn.cuh"

namespace bdion {

namespace {

constexpr int kThreads = 512;
constexpr int kRowThreads = 256;  // of the kernel that holds rows in registers
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTop = 1024;     // entries kept per row
constexpr int kMaxCand = 2048;    // candidates collected per row before ranking
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

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

// Calls f(column, values, count) over the row: 8 elements at a time where the
// row is 16-byte aligned, single ones at its ends (`lead` elements first), or
// everywhere when `vec` is false.
template <typename T, typename F>
__device__ __forceinline__ void for_row(const T* row, int V, int lead, F f) {
  for (int c = threadIdx.x; c < lead; c += kThreads) {
    float v[8] = {as_f(row[c])};
    f(c, v, std::integral_constant<int, 1>{});
  }
  const int n8 = (V - lead) / 8;
  for (int g = threadIdx.x; g < n8; g += kThreads) {
    float v[8];
    load8(row + lead + g * 8, v);
    f(lead + g * 8, v, std::integral_constant<int, 8>{});
  }
  for (int c = lead + n8 * 8 + threadIdx.x; c < V; c += kThreads) {
    float v[8] = {as_f(row[c])};
    f(c, v, std::integral_constant<int, 1>{});
  }
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
  __device__ __forceinline__ void get(f2 (&v)[4]) const {
    float x[8];
    get(x);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = make_f2(x[2 * i], x[2 * i + 1]);
  }
};


// ------------------------------------------------------------ top logits
__device__ __forceinline__ float key_float(uint32_t key) {  // the float that order_key took (not for NaN)
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// Largest threshold that at least k of the n keys reach, bit by bit (one warp);
// stops early where exactly k do. key(i) may be called for i < n only.
template <typename F>
__device__ __forceinline__ uint32_t kth_key(int n, int k, F key) {
  uint32_t thr = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t t = thr | (1u << bit);
    int cnt = 0;
    for (int i = threadIdx.x % 32; i < n; i += 32) cnt += key(i) >= t;
    cnt = __reduce_add_sync(0xffffffffu, cnt);
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
// once. The host takes ns so that about 512 come together. A candidate's rank
// is the number of larger ones (value, then the lower index), counted after a
// second bound has thinned them out. Rows with too many candidates (equal
// values), and rows with a NaN or +inf, take the exact threshold over the whole
// row bit by bit and keep the lowest indices of the equal ones.
template <typename T, int G>
__global__ void __launch_bounds__(kThreads) top_logits_kernel(const T* __restrict__ logits, int64_t ld, int V, int k,
                                                              bool vec, int ns, float c, float* __restrict__ values,
                                                              int64_t* __restrict__ indices,
                                                              float* __restrict__ lse) {
  __shared__ float red[kWarps];
  __shared__ uint32_t s_max[kThreads * G];
  __shared__ uint64_t s_cand[2][kMaxCand];
  __shared__ int s_n;
  __shared__ uint32_t s_thr;
  const int64_t row = blockIdx.x;
  const T* x = logits + row * ld;
  const int tid = threadIdx.x;
  const int lead = vec ? row_lead(row, ld, V, true) : 0;
  const int n8 = (V - lead) / 8, tail0 = lead + n8 * 8, rounds = (n8 + kThreads - 1) / kThreads;
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
  if (tid == 0) s_n = 0;
  __syncthreads();
  if (tid < 32) {
    const uint32_t t = kth_key(kThreads * G, k, [&](int i) { return s_max[i]; });
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
  if (!special && tid == 0) lse[row] = sum.m * c * kLn2 + logf(sum.s);
  if (n > kMaxCand || special) {
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
    if (tid < 32) {
      const uint32_t t = kth_key(n, k, [&](int i) { return (uint32_t)(s_cand[0][i] >> 32); });
      if (tid == 0) s_thr = t, s_n = 0;
    }
    __syncthreads();
    thr = s_thr;
    for (int i = tid; i < n; i += kThreads) {
      const uint64_t cand = s_cand[0][i];
      if ((uint32_t)(cand >> 32) >= thr) s_cand[1][atomicAdd(&s_n, 1)] = cand;
    }
    __syncthreads();
    n = s_n;
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
  int64_t T, ld_in, ld_out;
  int V, k;
  bool vec;
  float inv_tau, alpha, tau, grad_scale;
};

// One block per row:
//   p_j   teacher's probability of entry j (of the whole vocabulary when its
//         log-sum-exp is given, p_rest = 1 - sum p; else of the k entries)
//   q     student's softmax(z / tau); q_rest its sum outside the entries
//   loss  (1 - alpha) CE(z, label) + alpha tau^2 [sum p_j log(p_j / q_j) + p_rest log(p_rest / q_rest)]
//   grad  grad_scale * dloss/dz, in the pass that reads the row again
// The entries' columns are marked in a bitmap, so that the sum over the rest
// is taken directly (1 - sum q_j would cancel when the student is sure) and
// keeps a maximum of its own.
template <typename T, typename TG>
__global__ void __launch_bounds__(kThreads) distill_kernel(const T* __restrict__ logits, TG* __restrict__ grad,
                                                           const DistillArgs a) {
  extern __shared__ uint32_t bitmap[];
  __shared__ float red[kWarps];
  __shared__ float s_p[kMaxTop], s_z[kMaxTop];
  __shared__ int s_i[kMaxTop];
  __shared__ int s_marked, s_twice;
  const int64_t row = blockIdx.x;
  const int V = a.V, tid = threadIdx.x;
  const T* x = logits + row * a.ld_in;
  TG* gx = grad + row * a.ld_out;
  const int lead = row_lead(row, a.ld_in, V, a.vec);
  const int shift = (8 - lead % 8) % 8;  // bit of column c is c + shift: 8-element groups are whole bytes
  const int64_t label = a.labels ? a.labels[row] : 0;
  if (label < 0 || label >= V) {  // takes no part
    const float zero[8] = {};
    if (tid == 0) a.row_loss[row] = 0.f;
    if (grad == nullptr) return;
    for (int i = tid; i < lead; i += kThreads) put(gx + i, 0.f);
    const int n8 = (V - lead) / 8;
    for (int g = tid; g < n8; g += kThreads) store8(gx + lead + g * 8, zero);
    for (int c = lead + n8 * 8 + tid; c < V; c += kThreads) put(gx + c, 0.f);
    return;
  }
  const bool hard = a.labels != nullptr && a.alpha != 1.f;
  const bool both = hard && a.inv_tau != 1.f;  // the label's softmax differs from the teacher's
  const float c = a.inv_tau * kLog2e;

  for (int i = tid; i < (V + 7 + 31) / 32; i += kThreads) bitmap[i] = 0;
  if (tid == 0) s_marked = s_twice = 0;
  __syncthreads();
  // the teacher's entries
  float tmax = -FLT_MAX;
  for (int j = tid; j < a.k; j += kThreads) {
    const int64_t i = a.idx64 ? static_cast<const int64_t*>(a.top_indices)[row * a.k + j]
                              : static_cast<const int*>(a.top_indices)[row * a.k + j];
    const bool in = i >= 0 && i < V;
    const float t = a.top_values[row * a.k + j] * a.inv_tau;
    s_i[j] = in ? (int)i : -1;
    s_p[j] = in ? t : -INFINITY;
    if (in) {
      s_z[j] = as_f(x[i]);
      const uint32_t bit = (uint32_t)i + shift, m = 1u << (bit & 31);
      if (atomicOr(&bitmap[bit >> 5], m) & m)
        s_twice = 1;
      else
        atomicAdd(&s_marked, 1);
      tmax = fmaxf(tmax, t);
    }
  }
  float tlse;
  if (a.top_lse != nullptr) {
    tlse = a.top_lse[row];
  } else {
    tmax = block_max(tmax, red);
    float s = 0.f;
    for (int j = tid; j < a.k; j += kThreads)
      if (s_i[j] >= 0) s += ex2((s_p[j] - tmax) * kLog2e);
    s = block_sum(s, red);
    tlse = tmax + logf(s);  // -inf without entries; s_p stays -inf there and gives p = 0 below
  }
  __syncthreads();

  // the row: sums over the columns outside the set, and over all at temperature 1 where the label needs it
  RunningSum rest, full;
  for_row(x, V, lead, [&](int col, const float* v, auto n) {
    constexpr int N = decltype(n)::value;
    const uint32_t bit = (uint32_t)(col + shift);
    const uint32_t marks = (bitmap[bit >> 5] >> (bit & 31)) & ((1u << N) - 1u);
    float vm = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) vm = fmaxf(vm, v[i]);
    if (both) {
      full.raise(vm, kLog2e);
#pragma unroll
      for (int i = 0; i < N; ++i) full.s += ex2((v[i] - full.m) * kLog2e);
    }
    if (marks == 0) {
      rest.raise(vm, c);
#pragma unroll
      for (int i = 0; i < N; ++i) rest.s += ex2((v[i] - rest.m) * c);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (!((marks >> i) & 1u)) rest.add(v[i], c);
    }
  });
  rest.join(c, red);
  if (both) full.join(kLog2e, red);

  // the set's own part of the student's sum
  const bool twice = s_twice != 0;
  auto first_of = [&](int j) {  // whether entry j is the first with its index
    if (twice)
      for (int i = 0; i < j; ++i)
        if (s_i[i] == s_i[j]) return false;
    return true;
  };
  float zmax = -FLT_MAX;
  for (int j = tid; j < a.k; j += kThreads)
    if (s_i[j] >= 0) zmax = fmaxf(zmax, s_z[j]);
  const float m = fmaxf(block_max(zmax, red), rest.m);
  float set = 0.f, psum = 0.f;
  for (int j = tid; j < a.k; j += kThreads)
    if (s_i[j] >= 0) {
      if (first_of(j)) set += ex2((s_z[j] - m) * c);
      psum += s_p[j] == -INFINITY ? 0.f : ex2((s_p[j] - tlse) * kLog2e);
    }
  set = block_sum(set, red);
  psum = block_sum(psum, red);
  const float B = set + rest.s * ex2((rest.m - m) * c);
  const float logB = logf(B), logz = m * a.inv_tau + logB;  // log of the sum of exp(z / tau)
  const bool has_rest = a.top_lse != nullptr && s_marked < V;
  const float p_rest = has_rest ? fmaxf(1.f - psum, 0.f) : 0.f;

  float kl = 0.f;
  for (int j = tid; j < a.k; j += kThreads)
    if (s_i[j] >= 0 && s_p[j] != -INFINITY) {
      const float logp = s_p[j] - tlse, p = ex2(logp * kLog2e);
      if (p > 0.f) kl += p * (logp - (s_z[j] * a.inv_tau - logz));
      if (p != p) kl = p;
    }
  kl = block_sum(kl, red);
  if (p_rest > 0.f) kl += p_rest * (logf(p_rest) - (rest.m * a.inv_tau + logf(rest.s) - logz));
  const float zy = hard ? as_f(x[label]) : 0.f;
  const float log_full = !hard ? 0.f : both ? full.m + logf(full.s) : logz;
  if (tid == 0)
    a.row_loss[row] = (a.alpha > 0.f ? a.alpha * a.tau * a.tau * kl : 0.f) +
                      (hard ? (1.f - a.alpha) * (log_full - zy) : 0.f);

  if (grad == nullptr) return;
  // gradient. Outside the set: w_hard softmax(z) + w_soft (q - p_rest q / q_rest)
  const float w_soft = a.grad_scale * a.alpha * a.tau * (psum + p_rest == 0.f ? 0.f : 1.f);
  const float w_hard = hard ? a.grad_scale * (1.f - a.alpha) : 0.f;
  const float inv_B = 1.f / B;
  float f_rest = 0.f;  // factor of 2^(c (z - rest.m))
  if (rest.s > 0.f || rest.s != rest.s)
    f_rest = w_soft * (ex2((rest.m - m) * c) * inv_B - p_rest / rest.s) +
             (both ? 0.f : w_hard * ex2((rest.m - m) * c) * inv_B);
  const float f_full = both ? w_hard / full.s : 0.f;
  __syncthreads();
  for_row(x, V, lead, [&](int col, const float* v, auto n) {
    constexpr int N = decltype(n)::value;
    float g[8];
#pragma unroll
    for (int i = 0; i < N; ++i) g[i] = f_rest * ex2((v[i] - rest.m) * c);
    if (both) {
#pragma unroll
      for (int i = 0; i < N; ++i) g[i] += f_full * ex2((v[i] - full.m) * kLog2e);
    }
    if (N == 8)
      store8(gx + col, g);
    else
      put(gx + col, g[0]);
  });
  __syncthreads();
  // the set's columns and the label's
  auto at_label = [&](float z) { return both ? ex2((z - full.m) * kLog2e) / full.s : ex2((z - m) * c) * inv_B; };
  for (int j = tid; j < a.k; j += kThreads) {
    const int i = s_i[j];
    if (i < 0 || !first_of(j)) continue;
    float p = 0.f;
    for (int e = j; e < (twice ? a.k : j + 1); ++e)
      if (s_i[e] == i && s_p[e] != -INFINITY) p += ex2((s_p[e] - tlse) * kLog2e);
    float g = w_soft * (ex2((s_z[j] - m) * c) * inv_B - p);
    if (hard) g += w_hard * (at_label(s_z[j]) - (i == label ? 1.f : 0.f));
    put(gx + i, g);
  }
  if (hard && tid == 0) {
    const uint32_t bit = (uint32_t)label + shift;
    if (!((bitmap[bit >> 5] >> (bit & 31)) & 1u)) {
      const float q = ex2((zy - m) * c) * inv_B;
      const float r = rest.s > 0.f ? p_rest * ex2((zy - rest.m) * c) / rest.s : 0.f;
      put(gx + label, w_soft * (q - r) + w_hard * (at_label(zy) - 1.f));
    }
  }
}

// ------------------------------------------------------------ distillation loss, row held in registers
constexpr int kEnds = 16;          // elements before the first and after the last 8-element group
constexpr int kMaxCluster = 8;

// Sums (or maxima) of N <= kRowWarps values over a block of kRowThreads in two
// barriers; `buf` holds N * (kRowWarps + 1) floats, which the next call may use
// at once.
constexpr int kRowWarps = kRowThreads / 32;
template <int N, bool MAX>
__device__ __forceinline__ void block_all(float (&v)[N], float* buf) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = MAX ? warp_max(v[i]) : warp_sum(v[i]);
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) buf[N + i * kRowWarps + warp] = v[i];
  }
  __syncthreads();
  if (warp < N) {
    float x = lane < kRowWarps ? buf[N + warp * kRowWarps + lane] : (MAX ? -FLT_MAX : 0.f);
    x = MAX ? warp_max(x) : warp_sum(x);
    if (lane == 0) buf[warp] = x;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = buf[i];
}

// How the label's softmax (temperature 1) is taken beside the teacher's.
enum HardMode { kHardNone, kHardSquare, kHardOther };

// A cluster of `C` blocks holds one row in registers: each thread up to NV
// groups of 8 elements, so the row is read once. The blocks exchange eight
// partial results (one cluster barrier) and each writes its own part of the
// gradient. The entries belong to the block that holds their column. Clusters
// stay on their SMs and take rows in turn; the next row's elements are loaded
// into the registers that the gradient has just been computed from, its label
// and entries before that, so memory is busy through the row's reductions.
//
// Where the label's softmax differs from the teacher's, temperature 2 gives it
// as the square of the teacher's exponentials, 2^(x log2e) = (2^(x log2e / 2))^2
// (kHardSquare): at two exponentials per element and pass the SFU would take
// longer than memory. Temperatures 3 and 4 take powers likewise (kHardOther
// with `power`), others an exponential of their own.
template <typename T, typename TG, int NV, int MODE>
__global__ void __launch_bounds__(kRowThreads, 2)
    distill_row_kernel(const T* __restrict__ logits, TG* __restrict__ grad, const DistillArgs a, int C, int power) {
  namespace cg = cooperative_groups;
  constexpr bool both = MODE != kHardNone;
  __shared__ uint32_t s_marks[kRowThreads * NV / 4];  // one byte per group: which of its columns are in the set
  __shared__ uint32_t s_end_marks;
  __shared__ float red_max[2 * (kRowWarps + 1)], red_sum[6 * (kRowWarps + 1)];
  __shared__ float s_p[kMaxTop], s_z[kMaxTop];
  __shared__ int s_i[kMaxTop];
  __shared__ int s_marked, s_twice;
  enum { kM, kZ, kS, kF, kSet, kSetF, kCross, kCount, kParts };
  __shared__ float s_parts[2][kMaxCluster][kParts];  // two turns: a block may be one row ahead of another
  auto cluster = cg::this_cluster();
  const int rank = blockIdx.x % C;
  const int64_t stride = gridDim.x / C;
  const int V = a.V, tid = threadIdx.x;
  const bool hard = a.labels != nullptr && a.alpha != 1.f;
  const float c = a.inv_tau * kLog2e;

  // which columns this block holds of a row
  struct Part {
    int lead, g0, n, tail0;  // columns before the groups, first group, groups, columns behind all groups
  };
  auto part_of = [&](int64_t row) {
    Part p;
    p.lead = row_lead(row, a.ld_in, V, true);
    const int n8 = (V - p.lead) / 8, per = (n8 + C - 1) / C;
    p.g0 = min(n8, rank * per);
    p.n = min(n8, p.g0 + per) - p.g0;
    p.tail0 = p.lead + n8 * 8;
    return p;
  };
  auto owner_bit = [&](const Part& p, int col, uint32_t*& word) -> int {  // bit of this block's marks, -1 if another's
    if (col < p.lead || col >= p.tail0) {
      word = &s_end_marks;
      return rank == 0 ? (col < p.lead ? col : 8 + col - p.tail0) : -1;
    }
    const int g = (col - p.lead) / 8 - p.g0;
    if (g < 0 || g >= p.n) return -1;
    word = &s_marks[g / 4];
    return g % 4 * 8 + (col - p.lead) % 8;
  };
  auto label_of = [&](int64_t row) -> int {  // -1: takes no part
    if (row >= a.T) return -1;
    const int64_t y = a.labels ? a.labels[row] : 0;
    return y >= 0 && y < V ? (int)y : -1;
  };
  auto index_of = [&](int64_t row, int j) -> int {  // -1: unused entry
    const int64_t i = a.idx64 ? static_cast<const int64_t*>(a.top_indices)[row * a.k + j]
                              : static_cast<const int*>(a.top_indices)[row * a.k + j];
    return i >= 0 && i < V ? (int)i : -1;
  };
  auto clear_marks = [&] {
    for (int i = tid; i < kRowThreads * NV / 4; i += kRowThreads) s_marks[i] = 0;
    if (tid == 0) s_marked = s_twice = 0, s_end_marks = 0;
  };

  cluster.barrier_arrive();  // waited for before the first store into another block
  bool arrived = true;
  int turn = 0;
  int64_t row = blockIdx.x / C;
  int label = label_of(row);
  Raw8<T> raw[NV];
  if (label >= 0) {
    const Part p = part_of(row);
    const T* xg = logits + row * a.ld_in + p.lead + (int64_t)p.g0 * 8;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (i * kRowThreads + tid < p.n) raw[i].load(xg + (i * kRowThreads + tid) * 8);
  }
  int ahead_i = -1;       // this thread's first entry of the next row
  float ahead_t = 0.f;
  if (label >= 0 && tid < a.k) {
    ahead_i = index_of(row, tid);
    ahead_t = a.top_values[row * a.k + tid];
  }
  clear_marks();
  __syncthreads();

  for (; row < a.T; row += stride) {
  const Part mine_of = part_of(row);
  const int lead = mine_of.lead, g0 = mine_of.g0, n_mine = mine_of.n, tail0 = mine_of.tail0;
  const T* x = logits + row * a.ld_in;
  TG* gx = grad + row * a.ld_out;
  const int next_label = label_of(row + stride);
  const Part next = part_of(row + stride);
  const T* next_x = logits + (row + stride) * a.ld_in + next.lead + (int64_t)next.g0 * 8;
  // the next row's group i into the place of this row's
  auto load_next = [&](int i) {
    if (next_label >= 0 && i * kRowThreads + tid < next.n) raw[i].load(next_x + (i * kRowThreads + tid) * 8);
  };
  const int now_i = ahead_i;
  const float now_t = ahead_t;
  if (next_label >= 0 && tid < a.k) {
    ahead_i = index_of(row + stride, tid);
    ahead_t = a.top_values[(row + stride) * a.k + tid];
  }
  if (label < 0) {  // takes no part: the whole cluster alike
    const float zero[8] = {};
    if (tid == 0 && rank == 0) a.row_loss[row] = 0.f;
    if (grad != nullptr) {
      for (int g = tid; g < n_mine; g += kRowThreads) store8(gx + lead + (g0 + g) * 8, zero);
      if (rank == 0 && tid < lead) put(gx + tid, 0.f);
      if (rank == 0 && tail0 + tid < V) put(gx + tail0 + tid, 0.f);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) load_next(i);
    label = next_label;
    continue;
  }
  // ends of the row: columns [0, lead) and [tail0, V), one per thread of block 0
  int end_col = -1;
  if (rank == 0 && tid < 8 && tid < lead) end_col = tid;
  if (rank == 0 && tid >= 8 && tid < kEnds && tail0 + tid - 8 < V) end_col = tail0 + tid - 8;
  const float end_z = end_col >= 0 ? as_f(x[end_col]) : -INFINITY;
  const float zy = hard ? as_f(x[label]) : 0.f;

  float mx[2] = {-FLT_MAX, -FLT_MAX};  // outside the set, in it
  float tmax = -FLT_MAX;
  for (int j = tid; j < a.k; j += kRowThreads) {
    const int i = j == tid ? now_i : index_of(row, j);
    const float t = (j == tid ? now_t : a.top_values[row * a.k + j]) * a.inv_tau;
    int mine = -1;  // this block's column, or -1
    if (i >= 0) {
      uint32_t* word;
      const int bit = owner_bit(mine_of, i, word);
      if (bit >= 0) {
        mine = i;
        const float z = as_f(x[i]);
        s_z[j] = z;
        mx[1] = fmaxf(mx[1], z);
        if (atomicOr(word, 1u << bit) & (1u << bit))
          s_twice = 1;
        else
          atomicAdd(&s_marked, 1);
      }
      tmax = fmaxf(tmax, t);
    }
    s_i[j] = mine;
    s_p[j] = i >= 0 ? t : -INFINITY;
  }
  float tlse;
  if (a.top_lse != nullptr) {
    tlse = a.top_lse[row];
  } else {
    float tm[1] = {tmax}, ts[1] = {};
    block_all<1, true>(tm, red_max);
    for (int j = tid; j < a.k; j += kRowThreads) ts[0] += s_p[j] == -INFINITY ? 0.f : ex2((s_p[j] - tm[0]) * kLog2e);
    block_all<1, false>(ts, red_sum);
    tlse = tm[0] + logf(ts[0]);
  }
  __syncthreads();

  // maximum outside the set, then the sums under it; columns in the set count as -inf
  auto marks_of = [&](int i) -> uint32_t { return reinterpret_cast<const uint8_t*>(s_marks)[i * kRowThreads + tid]; };
  auto strike = [](float v, uint32_t marks, int e) { return (marks >> e) & 1u ? -INFINITY : v; };
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (i * kRowThreads + tid < n_mine) {
      const uint32_t marks = marks_of(i);
      if (marks == 0) {
        mx[0] = fmaxf(mx[0], raw[i].max());
      } else {
        float v[8];
        raw[i].get(v);
#pragma unroll
        for (int e = 0; e < 8; ++e) mx[0] = fmaxf(mx[0], strike(v[e], marks, e));
      }
    }
  const bool end_rest = end_col >= 0 && !((s_end_marks >> tid) & 1u);
  if (end_rest) mx[0] = fmaxf(mx[0], end_z);
  block_all<2, true>(mx, red_max);
  const float m = mx[0], zmax = mx[1];
  // y = 2^(c (z - ref)) of the teacher's softmax -> the label's
  auto full_of = [&](float y, float z, float ref) {
    if (MODE == kHardSquare) return y * y;
    return power == 3 ? y * y * y : power == 4 ? (y * y) * (y * y) : ex2((z - ref) * kLog2e);
  };
  float sum[6] = {};  // rest; rest at temperature 1; set; set at temperature 1; teacher's mass; sum p (log p - z / tau)
  {
    const f2 neg_m = make_f2(-m, -m), c2 = make_f2(c, c);
    f2 rest2 = make_f2(0.f, 0.f), full2 = rest2;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (i * kRowThreads + tid < n_mine) {
        f2 v[4];
        raw[i].get(v);
        const uint32_t marks = marks_of(i);
        if (marks) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            v[e] = make_f2(strike(lo_of(v[e]), marks, 2 * e), strike(hi_of(v[e]), marks, 2 * e + 1));
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const f2 z = mul2(add2(v[e], neg_m), c2);
          const f2 y = make_f2(ex2(lo_of(z)), ex2(hi_of(z)));
          rest2 = add2(rest2, y);
          if (MODE == kHardSquare) full2 = fma2(y, y, full2);
          if (MODE == kHardOther)
            full2 = add2(full2, make_f2(full_of(lo_of(y), lo_of(v[e]), m), full_of(hi_of(y), hi_of(v[e]), m)));
        }
      }
    sum[0] = lo_of(rest2) + hi_of(rest2);
    sum[1] = lo_of(full2) + hi_of(full2);
  }
  if (end_rest) {
    const float y = ex2((end_z - m) * c);
    sum[0] += y;
    if (both) sum[1] += full_of(y, end_z, m);
  }
  const bool twice = s_twice != 0;
  auto first_of = [&](int j) {
    if (twice)
      for (int i = 0; i < j; ++i)
        if (s_i[i] == s_i[j]) return false;
    return true;
  };
  for (int j = tid; j < a.k; j += kRowThreads) {
    const float logp = s_p[j] - tlse, p = s_p[j] == -INFINITY ? 0.f : ex2(logp * kLog2e);
    sum[4] += p;
    if (s_i[j] >= 0) {
      if (p != 0.f) sum[5] += p * (logp - s_z[j] * a.inv_tau);
      if (first_of(j)) {
        const float y = ex2((s_z[j] - zmax) * c);
        sum[2] += y;
        if (both) sum[3] += full_of(y, s_z[j], zmax);
      }
    }
  }
  block_all<6, false>(sum, red_sum);
  const float psum = sum[4];
  auto s_part = s_parts[turn];
  turn ^= 1;
  if (arrived) cluster.barrier_wait();
  arrived = false;
  if (tid < C * kParts) {
    const int to = tid / kParts, what = tid % kParts;
    const float mine[kParts] = {m, zmax, sum[0], sum[1], sum[2], sum[3], sum[5], (float)s_marked};
    float v = mine[0];
#pragma unroll
    for (int i = 1; i < kParts; ++i) v = what == i ? mine[i] : v;
    *cluster.map_shared_rank(&s_part[rank][what], to) = v;
  }
  cluster.sync();
  float rm = -FLT_MAX, zm = -FLT_MAX;  // over the row
  for (int r = 0; r < C; ++r) {
    rm = fmaxf(rm, s_part[r][kM]);
    zm = fmaxf(zm, s_part[r][kZ]);
  }
  const float top = fmaxf(rm, zm);
  float rest_s = 0.f, rest_f = 0.f, B = 0.f, F = 0.f, cross = 0.f, marked = 0.f;
  for (int r = 0; r < C; ++r) {
    const float* q = s_part[r];
    rest_s += q[kS] * ex2((q[kM] - rm) * c);
    B += q[kSet] * ex2((q[kZ] - top) * c);
    if (both) {
      rest_f += q[kF] * ex2((q[kM] - rm) * kLog2e);
      F += q[kSetF] * ex2((q[kZ] - top) * kLog2e);
    }
    cross += q[kCross];
    marked += q[kCount];
  }
  const float to_top = ex2((rm - top) * c);
  B += rest_s * to_top;
  if (both) F += rest_f * ex2((rm - top) * kLog2e);
  const float logz = top * a.inv_tau + logf(B);
  const bool has_rest = a.top_lse != nullptr && marked < (float)V;
  const float p_rest = has_rest ? fmaxf(1.f - psum, 0.f) : 0.f;
  if (rank == 0 && tid == 0) {
    float kl = psum != 0.f ? cross + psum * logz : 0.f;
    if (p_rest > 0.f) kl += p_rest * (logf(p_rest) - (rm * a.inv_tau + logf(rest_s) - logz));
    const float log_full = both ? top + logf(F) : logz;
    a.row_loss[row] = (a.alpha > 0.f ? a.alpha * a.tau * a.tau * kl : 0.f) +
                      (hard ? (1.f - a.alpha) * (log_full - zy) : 0.f);
  }
  if (grad == nullptr) {
#pragma unroll
    for (int i = 0; i < NV; ++i) load_next(i);
    __syncthreads();
    clear_marks();
    __syncthreads();
    label = next_label;
    continue;
  }

  const float w_soft = a.grad_scale * a.alpha * a.tau * (psum + p_rest == 0.f ? 0.f : 1.f);
  const float w_hard = hard ? a.grad_scale * (1.f - a.alpha) : 0.f;
  const float inv_B = 1.f / B, inv_F = both ? 1.f / F : inv_B;
  float f_rest = 0.f, f_full = 0.f;
  if (rest_s > 0.f || rest_s != rest_s) {
    f_rest = w_soft * (to_top * inv_B - p_rest / rest_s) + (both ? 0.f : w_hard * to_top * inv_B);
    f_full = both ? w_hard * ex2((rm - top) * kLog2e) * inv_F : 0.f;
  }
  {
    const f2 neg_m = make_f2(-rm, -rm), c2 = make_f2(c, c);
    const f2 fr2 = make_f2(f_rest, f_rest), ff2 = make_f2(f_full, f_full);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      f2 v[4];
      raw[i].get(v);
      load_next(i);
      if (i * kRowThreads + tid < n_mine) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const f2 z = mul2(add2(v[e], neg_m), c2);
          const f2 y = make_f2(ex2(lo_of(z)), ex2(hi_of(z)));
          if (MODE == kHardNone)
            v[e] = mul2(fr2, y);
          else if (MODE == kHardSquare)
            v[e] = mul2(y, fma2(y, ff2, fr2));
          else
            v[e] = fma2(ff2, make_f2(full_of(lo_of(y), lo_of(v[e]), rm), full_of(hi_of(y), hi_of(v[e]), rm)), mul2(fr2, y));
        }
        const float g[8] = {lo_of(v[0]), hi_of(v[0]), lo_of(v[1]), hi_of(v[1]),
                            lo_of(v[2]), hi_of(v[2]), lo_of(v[3]), hi_of(v[3])};
        store8(gx + lead + (g0 + i * kRowThreads + tid) * 8, g);
      }
    }
  }
  if (end_col >= 0) {
    const float y = ex2((end_z - rm) * c);
    put(gx + end_col, both ? f_rest * y + f_full * full_of(y, end_z, rm) : f_rest * y);
  }
  __syncthreads();
  auto soft_at = [&](float z) { return ex2((z - top) * c) * inv_B; };
  auto hard_at = [&](float z) { return both ? ex2((z - top) * kLog2e) * inv_F : soft_at(z); };
  for (int j = tid; j < a.k; j += kRowThreads) {
    const int i = s_i[j];
    if (i < 0 || !first_of(j)) continue;
    float p = 0.f;
    for (int e = j; e < (twice ? a.k : j + 1); ++e)
      if (s_i[e] == i && s_p[e] != -INFINITY) p += ex2((s_p[e] - tlse) * kLog2e);
    float g = w_soft * (soft_at(s_z[j]) - p);
    if (hard) g += w_hard * (hard_at(s_z[j]) - (i == label ? 1.f : 0.f));
    put(gx + i, g);
  }
  if (hard && tid == 0) {
    uint32_t* word;
    const int bit = owner_bit(mine_of, label, word);
    if (bit >= 0 && !((*word >> bit) & 1u)) {
      const float r = rest_s > 0.f ? p_rest * ex2((zy - rm) * c) / rest_s : 0.f;
      put(gx + label, w_soft * (soft_at(zy) - r) + w_hard * (hard_at(zy) - 1.f));
    }
  }
  __syncthreads();
  clear_marks();
  __syncthreads();
  label = next_label;
  }
  if (arrived) cluster.barrier_wait();
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

// Clusters of C blocks that the device holds at once (asked once per kernel, device and C).
template <typename K>
int resident_clusters(K kern, const cudaLaunchConfig_t& cfg, int device, int C) {
  static std::mutex lock;
  static std::map<std::tuple<K, int, int>, int> known;
  std::lock_guard<std::mutex> hold(lock);
  int& n = known[{kern, device, C}];
  if (n == 0) {
    C10_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&n, kern, &cfg));
    n = std::max(n, 1);
  }
  return n;
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
  TORCH_CHECK(tau > 0, "dion_b200 top_logits: temperature > 0");
  check_out(values, logits, at::kFloat, {T, k}, "top_logits values");
  check_out(indices, logits, at::kLong, {T, k}, "top_logits indices");
  check_out(lse, logits, at::kFloat, {T}, "top_logits lse");
  if (T == 0) return;
  c10::cuda::CUDAGuard guard(logits.device());
  auto s = at::cuda::getCurrentCUDAStream();
  by_type(logits.scalar_type(), [&](auto tag) {
    using E = decltype(tag);
    // rounds in the sample: about 512 columns reach its bound
    const int rounds = (V / 8 + kThreads - 1) / kThreads;
    const int ns = std::max(1, std::min(rounds, (rounds * k + 511) / 512));
    auto launch = [&](auto g) {
      top_logits_kernel<E, decltype(g)::value><<<(unsigned)T, kThreads, 0, s>>>(
          static_cast<const E*>(logits.data_ptr()), logits.stride(0), V, k, aligned8(logits), ns, (float)(kLog2e / tau),
          values.data_ptr<float>(), indices.data_ptr<int64_t>(), lse.data_ptr<float>());
    };
    // at least twice as many groups as entries keeps the candidates near 1.4 k
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
  TORCH_CHECK(tau > 0, "dion_b200 distill: temperature > 0");
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
  a.T = T;
  a.V = V;
  a.k = k;
  // 8-element groups of the logits and of the gradient have to start together
  a.vec = aligned8(logits) && (!grad.has_value() || (aligned8(*grad) && (T == 1 || a.ld_in % 8 == a.ld_out % 8)));
  a.inv_tau = (float)(1.0 / tau);
  a.tau = (float)tau;
  a.alpha = (float)alpha;
  a.grad_scale = (float)grad_scale;
  const size_t smem = ((size_t)V + 7 + 31) / 32 * 4;
  auto s = at::cuda::getCurrentCUDAStream();
  by_type(logits.scalar_type(), [&](auto tag) {
    using E = decltype(tag);
    by_type(gtype, [&](auto gtag) {
      using G = decltype(gtag);
      if constexpr (std::is_same_v<E, G> || std::is_same_v<E, float>) {
        // Rows of up to kMaxCluster blocks' registers are read once; longer ones, and
        // those whose logits and gradient are not aligned alike, twice.
        constexpr int kMost = sizeof(E) == 2 ? 16 : 8;  // 64 registers of logits per thread
        const int64_t groups = V / 8;
        if (a.vec && groups <= (int64_t)kMaxCluster * kRowThreads * kMost) {
          int C = 1;
          while (groups > (int64_t)C * kRowThreads * kMost) C *= 2;
          const int64_t per_thread = (groups + C * kRowThreads - 1) / (C * kRowThreads);
          const int power = tau == 3 || tau == 4 ? (int)tau : 0;
          auto run = [&](auto nv, auto mode) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3((unsigned)C);
            cfg.blockDim = dim3(kRowThreads);
            cfg.stream = s;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim = {(unsigned)C, 1u, 1u};
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            auto kern = distill_row_kernel<E, G, decltype(nv)::value, decltype(mode)::value>;
            cfg.gridDim.x = (unsigned)(C * std::min<int64_t>(T, resident_clusters(kern, cfg, logits.get_device(), C)));
            C10_CUDA_CHECK(cudaLaunchKernelEx(
                &cfg, kern,
                static_cast<const E*>(logits.data_ptr()),
                grad.has_value() ? static_cast<G*>(grad->data_ptr()) : nullptr, a, C, power));
          };
          auto by_mode = [&](auto nv) {
            if (!a.labels || a.alpha == 1.f || a.inv_tau == 1.f)
              run(nv, std::integral_constant<int, kHardNone>{});
            else if (tau == 2)
              run(nv, std::integral_constant<int, kHardSquare>{});
            else
              run(nv, std::integral_constant<int, kHardOther>{});
          };
          if (per_thread <= 1)
            by_mode(std::integral_constant<int, 1>{});
          else if (per_thread <= 4)
            by_mode(std::integral_constant<int, 4>{});
          else
            by_mode(std::integral_constant<int, kMost>{});
          return;
        }
        auto kern = distill_kernel<E, G>;
        C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        kern<<<(unsigned)T, kThreads, smem, s>>>(static_cast<const E*>(logits.data_ptr()),
                                                 grad.has_value() ? static_cast<G*>(grad->data_ptr()) : nullptr, a);
      }
    });
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  note_launch();
  at::sum_out(loss, rows, 0);
}

}  // namespace bdion
