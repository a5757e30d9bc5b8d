// Causal attention with a sliding window and a few first tokens that stay
// visible: query i sees key j where j <= i and (i - j < window or j < sinks).
//
//   S = Q K^T / sqrt(d), P = softmax over the visible keys, O = P V
//   delta_i = dO_i . O_i, dS = P o (dO V^T - delta)
//   dQ = dS K / sqrt(d), dK = dS^T Q / sqrt(d), dV = P^T dO
//
// dK and dV of a key head sum over the query heads that share it. The forward
// pass keeps each row's log-sum-exp; the backward pass recomputes P from it.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>
#include <torch/extension.h>
#include <torch/library.h>

#include "common.cuh"
#include "host_utils.h"

namespace bdion {

namespace {

struct WinArgs {
  int b, s, hq, hkv, d, window, sinks;
  float scale;
  // strides in elements over (batch, position, head); the head dim is contiguous
  int64_t q[3], k[3], v[3], g[3];
};

__device__ __forceinline__ float as_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float as_f(__half v) { return __half2float(v); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }

__device__ __forceinline__ float warp_sum(float v) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffff, v, o);
  return v;
}

template <typename T>
__device__ __forceinline__ void load_row(const T* p, int d, float (&x)[4]) {
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int c = r * 32 + threadIdx.x % 32;
    x[r] = c < d ? as_f(p[c]) : 0.f;
  }
}
__device__ __forceinline__ float dot(const float (&x)[4], const float (&y)[4]) {
  return warp_sum(x[0] * y[0] + x[1] * y[1] + x[2] * y[2] + x[3] * y[3]);
}

// Calls f(j) for every key that query i sees.
template <typename F>
__device__ __forceinline__ void for_keys(const WinArgs& a, int i, F f) {
  const int lo = max(0, i - a.window + 1);
  for (int j = 0; j < min(a.sinks, lo); ++j) f(j);
  for (int j = lo; j <= i; ++j) f(j);
}

// One warp per query: o and the row's log-sum-exp (natural logarithm).
template <typename T>
__global__ void __launch_bounds__(128) window_fwd_kernel(const T* q, const T* k, const T* v, T* o, float* lse,
                                                         const WinArgs a) {
  const int64_t w = (int64_t)blockIdx.x * 4 + threadIdx.x / 32;  // (b, i, h)
  if (w >= (int64_t)a.b * a.s * a.hq) return;
  const int h = w % a.hq, i = (w / a.hq) % a.s, b = w / a.hq / a.s, hk = h / (a.hq / a.hkv);
  float x[4], acc[4] = {}, m = -INFINITY, sum = 0.f;
  load_row(q + b * a.q[0] + i * a.q[1] + h * a.q[2], a.d, x);
  for_keys(a, i, [&](int j) {
    float y[4];
    load_row(k + b * a.k[0] + j * a.k[1] + hk * a.k[2], a.d, y);
    const float sc = dot(x, y) * a.scale, mn = fmaxf(m, sc), f = __expf(m - mn), p = __expf(sc - mn);
    load_row(v + b * a.v[0] + j * a.v[1] + hk * a.v[2], a.d, y);
    for (int r = 0; r < 4; ++r) acc[r] = acc[r] * f + p * y[r];
    sum = sum * f + p;
    m = mn;
  });
  for (int r = 0; r < 4; ++r) {
    const int c = r * 32 + threadIdx.x % 32;
    if (c < a.d) put(o + w * a.d + c, acc[r] / sum);
  }
  if (threadIdx.x % 32 == 0) lse[((int64_t)b * a.hq + h) * a.s + i] = m + logf(sum);
}

// One warp per query: dq and delta.
template <typename T>
__global__ void __launch_bounds__(128) window_dq_kernel(const T* q, const T* k, const T* v, const T* o, const T* g,
                                                        const float* lse, T* dq, float* delta, const WinArgs a) {
  const int64_t w = (int64_t)blockIdx.x * 4 + threadIdx.x / 32;
  if (w >= (int64_t)a.b * a.s * a.hq) return;
  const int h = w % a.hq, i = (w / a.hq) % a.s, b = w / a.hq / a.s, hk = h / (a.hq / a.hkv);
  const int64_t at = ((int64_t)b * a.hq + h) * a.s + i;
  float x[4], y[4], go[4], acc[4] = {};
  load_row(q + b * a.q[0] + i * a.q[1] + h * a.q[2], a.d, x);
  load_row(g + b * a.g[0] + i * a.g[1] + h * a.g[2], a.d, go);
  load_row(o + w * a.d, a.d, y);
  const float dl = dot(go, y), L = lse[at];
  if (threadIdx.x % 32 == 0) delta[at] = dl;
  for_keys(a, i, [&](int j) {
    load_row(v + b * a.v[0] + j * a.v[1] + hk * a.v[2], a.d, y);
    const float dp = dot(go, y);
    load_row(k + b * a.k[0] + j * a.k[1] + hk * a.k[2], a.d, y);
    const float ds = __expf(dot(x, y) * a.scale - L) * (dp - dl) * a.scale;
    for (int r = 0; r < 4; ++r) acc[r] += ds * y[r];
  });
  for (int r = 0; r < 4; ++r) {
    const int c = r * 32 + threadIdx.x % 32;
    if (c < a.d) put(dq + w * a.d + c, acc[r]);
  }
}

// One warp per key: dk and dv over the queries that see it and the heads of the group.
template <typename T>
__global__ void __launch_bounds__(128) window_dkv_kernel(const T* q, const T* k, const T* v, const T* g,
                                                         const float* lse, const float* delta, T* dk, T* dv,
                                                         const WinArgs a) {
  const int64_t w = (int64_t)blockIdx.x * 4 + threadIdx.x / 32;
  if (w >= (int64_t)a.b * a.s * a.hkv) return;
  const int hk = w % a.hkv, j = (w / a.hkv) % a.s, b = w / a.hkv / a.s, group = a.hq / a.hkv;
  float kx[4], vx[4], x[4], go[4], ak[4] = {}, av[4] = {};
  load_row(k + b * a.k[0] + j * a.k[1] + hk * a.k[2], a.d, kx);
  load_row(v + b * a.v[0] + j * a.v[1] + hk * a.v[2], a.d, vx);
  const int last = j < a.sinks ? a.s : (int)min((int64_t)a.s, (int64_t)j + a.window);
  for (int h = hk * group; h < (hk + 1) * group; ++h)
    for (int i = j; i < last; ++i) {
      const int64_t at = ((int64_t)b * a.hq + h) * a.s + i;
      load_row(q + b * a.q[0] + i * a.q[1] + h * a.q[2], a.d, x);
      load_row(g + b * a.g[0] + i * a.g[1] + h * a.g[2], a.d, go);
      const float p = __expf(dot(x, kx) * a.scale - lse[at]);
      const float ds = p * (dot(go, vx) - delta[at]) * a.scale;
      for (int r = 0; r < 4; ++r) {
        ak[r] += ds * x[r];
        av[r] += p * go[r];
      }
    }
  for (int r = 0; r < 4; ++r) {
    const int c = r * 32 + threadIdx.x % 32;
    if (c < a.d) {
      put(dk + w * a.d + c, ak[r]);
      put(dv + w * a.d + c, av[r]);
    }
  }
}

void check_heads(const at::Tensor& t, const at::Tensor& like, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.scalar_type() == like.scalar_type() && t.dim() == 4 &&
                  t.size(0) == like.size(0) && t.size(1) == like.size(1) && t.size(3) == like.size(3) &&
                  t.stride(3) == 1,
              "dion_b200 window_attention: ", what,
              " [b, s, heads, d] of q's type on q's device with a contiguous head dimension");
}

WinArgs make_args(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, int64_t window, int64_t sinks) {
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf,
              "dion_b200 window_attention: bf16 or fp16");
  check_heads(q, q, "q");
  check_heads(k, q, "k");
  check_heads(v, q, "v");
  TORCH_CHECK(k.size(2) == v.size(2) && k.size(2) >= 1 && q.size(2) % k.size(2) == 0,
              "dion_b200 window_attention: as many v as k heads, and a multiple of them for q");
  TORCH_CHECK(q.size(3) % 8 == 0 && q.size(3) >= 8 && q.size(3) <= 128,
              "dion_b200 window_attention: head dimension a multiple of 8, at most 128");
  TORCH_CHECK(window >= 1 && sinks >= 0, "dion_b200 window_attention: window >= 1 and sinks >= 0");
  TORCH_CHECK(q.size(1) < (1 << 30), "dion_b200 window_attention: fewer than 2^30 positions");
  WinArgs a;
  a.b = (int)q.size(0);
  a.s = (int)q.size(1);
  a.hq = (int)q.size(2);
  a.hkv = (int)k.size(2);
  a.d = (int)q.size(3);
  a.window = (int)std::min<int64_t>(window, a.s);
  a.sinks = (int)std::min<int64_t>(sinks, a.s);
  a.scale = 1.f / std::sqrt((float)a.d);
  for (int i = 0; i < 3; ++i) {
    a.q[i] = q.stride(i);
    a.k[i] = k.stride(i);
    a.v[i] = v.stride(i);
    a.g[i] = 0;
  }
  return a;
}

template <typename F>
void by_type(at::ScalarType t, F f) {
  if (t == at::kBFloat16)
    f(__nv_bfloat16{});
  else
    f(__half{});
}

unsigned warps_grid(int64_t rows) {
  TORCH_CHECK((rows + 3) / 4 < (1ll << 31), "dion_b200 window_attention: too many rows");
  return (unsigned)((rows + 3) / 4);
}

}  // namespace

// o [b, s, hq, d] and the rows' log-sum-exp [b, hq, s]
std::tuple<at::Tensor, at::Tensor> window_attention_fwd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                        int64_t window, int64_t sinks) {
  const WinArgs a = make_args(q, k, v, window, sinks);
  c10::cuda::CUDAGuard guard(q.device());
  auto o = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  auto lse = at::empty({a.b, a.hq, a.s}, q.options().dtype(at::kFloat));
  if (o.numel() == 0) return {o, lse};
  by_type(q.scalar_type(), [&](auto tag) {
    using E = decltype(tag);
    window_fwd_kernel<E><<<warps_grid((int64_t)a.b * a.s * a.hq), 128, 0, at::cuda::getCurrentCUDAStream()>>>(
        (const E*)q.data_ptr(), (const E*)k.data_ptr(), (const E*)v.data_ptr(), (E*)o.data_ptr(),
        lse.data_ptr<float>(), a);
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  note_launch();
  return {o, lse};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> window_attention_bwd(const at::Tensor& go, const at::Tensor& q,
                                                                    const at::Tensor& k, const at::Tensor& v,
                                                                    const at::Tensor& o, const at::Tensor& lse,
                                                                    int64_t window, int64_t sinks) {
  WinArgs a = make_args(q, k, v, window, sinks);
  check_heads(go, q, "the output's gradient");
  TORCH_CHECK(go.sizes() == q.sizes() && o.sizes() == q.sizes() && o.is_contiguous() && lse.is_contiguous() &&
                  lse.scalar_type() == at::kFloat && lse.numel() == (int64_t)a.b * a.hq * a.s,
              "dion_b200 window_attention: o and lse as the forward pass gave them");
  for (int i = 0; i < 3; ++i) a.g[i] = go.stride(i);
  c10::cuda::CUDAGuard guard(q.device());
  auto st = at::cuda::getCurrentCUDAStream();
  auto like = [](const at::Tensor& t) {
    return at::empty(t.sizes(), t.options().memory_format(at::MemoryFormat::Contiguous));
  };
  auto dq = like(q), dk = like(k), dv = like(v);
  if (q.numel() == 0) return {dq, dk.zero_(), dv.zero_()};
  auto delta = at::empty_like(lse);
  by_type(q.scalar_type(), [&](auto tag) {
    using E = decltype(tag);
    window_dq_kernel<E><<<warps_grid((int64_t)a.b * a.s * a.hq), 128, 0, st>>>(
        (const E*)q.data_ptr(), (const E*)k.data_ptr(), (const E*)v.data_ptr(), (const E*)o.data_ptr(),
        (const E*)go.data_ptr(), lse.data_ptr<float>(), (E*)dq.data_ptr(), delta.data_ptr<float>(), a);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    window_dkv_kernel<E><<<warps_grid((int64_t)a.b * a.s * a.hkv), 128, 0, st>>>(
        (const E*)q.data_ptr(), (const E*)k.data_ptr(), (const E*)v.data_ptr(), (const E*)go.data_ptr(),
        lse.data_ptr<float>(), delta.data_ptr<float>(), (E*)dk.data_ptr(), (E*)dv.data_ptr(), a);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  });
  note_launch(2);
  return {dq, dk, dv};
}

}  // namespace bdion

// A dispatcher op, so that selective activation checkpointing can name its
// output among those that it keeps.
TORCH_LIBRARY(dion_b200, m) {
  m.def("window_attention_fwd(Tensor q, Tensor k, Tensor v, int window, int sinks) -> (Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(dion_b200, CUDA, m) { m.impl("window_attention_fwd", &bdion::window_attention_fwd); }
