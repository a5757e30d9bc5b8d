// Causal attention with a sliding window and a few first tokens that stay
// visible: query i sees key j where j <= i and (i - j < window or j < sinks).
//
//   S = Q K^T / sqrt(d), P = softmax over the visible keys, O = P V
//   delta_i = dO_i . O_i, dS = P o (dO V^T - delta)
//   dQ = dS K / sqrt(d), dK = dS^T Q / sqrt(d), dV = P^T dO
//
// dK and dV of a key head sum over the query heads that share it. The forward
// pass keeps each row's log-sum-exp; the backward pass recomputes P from it. A
// row that sees one key has P = 1 and dS = 0, which both kernels write as such.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>
#include <torch/extension.h>
#include <torch/library.h>

#include "host_utils.h"
#include "tensor_map.h"
#include "window_tc.cuh"

namespace bdion {

namespace {

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
  a.s_pad = (a.s + kTile - 1) / kTile * kTile;
  a.scale = 1.f / std::sqrt((float)a.d);
  a.scale_log2 = a.scale * 1.4426950408889634f;
  a.status = status_device_ptr();
  a.limit_ns = wait_limit_ns();
  return a;
}

// [b, s, heads, d] as a 4-D map (d, s, heads, b): boxes of 64 elements (one
// swizzled 128-byte row) by `rows` positions of one head; elements beyond d
// and rows beyond s read as zero.
CUtensorMap head_map(const at::Tensor& t, int rows, const char* what) {
  CUtensorMap m;
  const cuuint64_t dims[4] = {(cuuint64_t)t.size(3), (cuuint64_t)t.size(1), (cuuint64_t)t.size(2),
                              (cuuint64_t)t.size(0)};
  cuuint64_t strides[3];
  const int axis[3] = {1, 2, 0};
  for (int i = 0; i < 3; ++i) {
    const int64_t st = t.size(axis[i]) > 1 ? t.stride(axis[i]) * 2 : 16;
    TORCH_CHECK(st > 0 && st % 16 == 0, "dion_b200 window_attention: ", what,
                ": strides that are positive multiples of 16 bytes");
    strides[i] = (cuuint64_t)st;
  }
  TORCH_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, "dion_b200 window_attention: ", what,
              ": a base aligned to 16 bytes");
  const cuuint32_t box[4] = {64u, (cuuint32_t)rows, 1u, 1u}, step[4] = {1u, 1u, 1u, 1u};
  const CUresult r =
      encode_fn()(&m, t.scalar_type() == at::kHalf ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                  4, t.data_ptr(), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "dion_b200 window_attention: cuTensorMapEncodeTiled failed with ", (int)r);
  return m;
}

// The tensor-map encoder wants a current context, which a thread that has made
// no runtime call yet (autograd's backward threads) lacks.
void bind_context(const at::Tensor& t) { C10_CUDA_CHECK(cudaSetDevice(t.get_device())); }

// Launches with the kernel's shared memory allowed on the current device.
template <typename K, typename... Args>
void launch(K kern, int64_t grid, int threads, int smem, cudaStream_t st, Args... args) {
  TORCH_CHECK(grid < (1ll << 31), "dion_b200 window_attention: too many tiles");
  C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  kern<<<(unsigned)grid, threads, smem, st>>>(args...);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  note_launch();
}

// f(element type, padded head dimension)
template <typename F>
void by_case(at::ScalarType t, int d, F f) {
  auto with = [&](auto tag) {
    if (d <= 64)
      f(tag, std::integral_constant<int, 64>{});
    else
      f(tag, std::integral_constant<int, 128>{});
  };
  if (t == at::kBFloat16)
    with(__nv_bfloat16{});
  else
    with(__half{});
}

// Parts of the dK / dV kernel. A tile is cut where the whole tiles would not
// give every SM two parts; a tile with first tokens where its steps would
// outlast the others'. A part has 4 steps at least: fewer cost more in its
// start and its sums' way through memory than they bring.
KeySplit split_keys(const WinArgs& a) {
  KeySplit p;
  const int64_t group = a.hq / a.hkv, sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  p.n_tiles = a.s_pad / kTile;
  p.n_first = std::min(p.n_tiles, (a.sinks + kTile - 1) / kTile);
  const int64_t heads = (int64_t)a.b * a.hkv, per_head = a.s_pad / kTile;
  const int64_t band = group * std::min<int64_t>(per_head, ((int64_t)kTile + a.window - 2) / kTile + 1);
  const int64_t first = group * per_head;
  auto cut = [](int64_t parts, int64_t steps) { return (int)std::max<int64_t>(1, std::min(parts, steps / 4)); };
  p.c_band = cut((2 * sms + heads * p.n_tiles - 1) / (heads * p.n_tiles), band);
  const int64_t total = heads * (p.n_first * first + (p.n_tiles - p.n_first) * band);
  const int64_t longest = std::max((band + p.c_band - 1) / p.c_band, total / (4 * sms));
  p.c_first = cut((first + longest - 1) / longest, first);
  return p;
}

}  // namespace

// o [b, s, hq, d]; with `backward` what its rounding left out, as another tensor of
// o's type (else an empty one); and minus the log2 of each row's sum of exponentials [b, hq,
// s rounded up to 128] (-inf behind the last position) for the backward pass
std::tuple<at::Tensor, at::Tensor, at::Tensor> window_attention_fwd(const at::Tensor& q, const at::Tensor& k,
                                                                    const at::Tensor& v, int64_t window,
                                                                    int64_t sinks, bool backward) {
  const WinArgs a = make_args(q, k, v, window, sinks);
  c10::cuda::CUDAGuard guard(q.device());
  bind_context(q);
  auto o = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  auto o_low = backward ? at::empty_like(o) : at::empty({0}, o.options());
  auto lse = at::empty({a.b, a.hq, a.s_pad}, q.options().dtype(at::kFloat));
  if (o.numel() == 0) return {o, o_low, lse};
  const CUtensorMap mq = head_map(q, kTile, "q"), mk = head_map(k, kHalfTile, "k"), mv = head_map(v, kHalfTile, "v");
  by_case(q.scalar_type(), a.d, [&](auto tag, auto dp) {
    using E = decltype(tag);
    constexpr int DP = decltype(dp)::value;
    launch(window_fwd_tc<E, DP>, (int64_t)a.b * a.hq * (a.s_pad / kTile), 192, FwdCfg<E, DP>::kSmemBytes,
           at::cuda::getCurrentCUDAStream(), mq, mk, mv, (E*)o.data_ptr(),
           backward ? (E*)o_low.data_ptr() : nullptr, lse.data_ptr<float>(), a);
  });
  return {o, o_low, lse};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> window_attention_bwd(const at::Tensor& go, const at::Tensor& q,
                                                                    const at::Tensor& k, const at::Tensor& v,
                                                                    const at::Tensor& o, const at::Tensor& o_low,
                                                                    const at::Tensor& lse, int64_t window,
                                                                    int64_t sinks) {
  const WinArgs a = make_args(q, k, v, window, sinks);
  check_heads(go, q, "the output's gradient");
  TORCH_CHECK(go.sizes() == q.sizes() && o.sizes() == q.sizes() && o.is_contiguous() && o.device() == q.device() &&
                  o.scalar_type() == q.scalar_type() && o_low.sizes() == q.sizes() && o_low.is_contiguous() &&
                  o_low.device() == q.device() && o_low.scalar_type() == q.scalar_type() && lse.is_contiguous() && lse.device() == q.device() &&
                  lse.scalar_type() == at::kFloat && lse.numel() == (int64_t)a.b * a.hq * a.s_pad,
              "dion_b200 window_attention: o, its remainder and lse as the forward pass gave them");
  c10::cuda::CUDAGuard guard(q.device());
  bind_context(q);
  auto st = at::cuda::getCurrentCUDAStream();
  auto like = [](const at::Tensor& t) {
    return at::empty(t.sizes(), t.options().memory_format(at::MemoryFormat::Contiguous));
  };
  auto dq = like(q), dk = like(k), dv = like(v);
  if (q.numel() == 0) return {dq, dk.zero_(), dv.zero_()};
  auto delta = at::empty_like(lse);
  const KeySplit split = split_keys(a);
  const CUtensorMap mq = head_map(q, kTile, "q"), mk = head_map(k, kTile, "k"), mv = head_map(v, kTile, "v"),
                    mg = head_map(go, kTile, "the output's gradient");
  by_case(q.scalar_type(), a.d, [&](auto tag, auto dp) {
    using E = decltype(tag);
    constexpr int DP = decltype(dp)::value;
    launch(window_dq_tc<E, DP>, (int64_t)a.b * a.hq * (a.s_pad / kTile), 576, DqCfg<E, DP>::kSmemBytes, st, mq, mk, mv,
           mg, (const E*)o.data_ptr(), (const E*)o_low.data_ptr(), (const E*)go.data_ptr(), go.stride(0), go.stride(1), go.stride(2),
           lse.data_ptr<float>(), delta.data_ptr<float>(), (E*)dq.data_ptr(), a);
    at::Tensor work;
    const int64_t slots = (int64_t)a.b * a.hkv * split.slots();
    if (slots > 0) work = at::empty({slots, 2, kTile, DP}, lse.options());
    launch(window_dkv_tc<E, DP>, (int64_t)a.b * a.hkv * split.parts(), 576, DkvCfg<E, DP>::kSmemBytes, st, mq, mk, mv,
           mg, lse.data_ptr<float>(), delta.data_ptr<float>(), (E*)dk.data_ptr(), (E*)dv.data_ptr(),
           slots > 0 ? work.data_ptr<float>() : nullptr, split, a);
    if (slots > 0) {
      const int tile0 = split.c_first > 1 ? 0 : split.n_first;
      const int tile1 = split.c_band > 1 ? split.n_tiles : split.n_first;
      launch(window_dkv_join<E, DP>, (int64_t)(tile1 - tile0) * a.b * a.hkv * 2 * (kTile / 16), 16 * DP / 8, 0, st,
             work.data_ptr<float>(), (E*)dk.data_ptr(), (E*)dv.data_ptr(), split, tile0, a);
    }
  });
  return {dq, dk, dv};
}

// The op alone records no gradient (ops/fused.py wraps both passes): a call that would
// drop one is an error.
std::tuple<at::Tensor, at::Tensor, at::Tensor> window_attention_fwd_checked(const at::Tensor& q, const at::Tensor& k,
                                                                            const at::Tensor& v, int64_t window,
                                                                            int64_t sinks, bool backward) {
  TORCH_CHECK(!at::GradMode::is_enabled() || !(q.requires_grad() || k.requires_grad() || v.requires_grad()),
              "dion_b200 window_attention_fwd: this op records no gradient; dion_b200.ops.fused.window_attention does");
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("dion_b200::window_attention_fwd", "")
                             .typed<decltype(window_attention_fwd)>();
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(q, k, v, window, sinks, backward);
}

}  // namespace bdion

// A dispatcher op, so that selective activation checkpointing can name its
// output among those that it keeps.
TORCH_LIBRARY(dion_b200, m) {
  m.def("window_attention_fwd(Tensor q, Tensor k, Tensor v, int window, int sinks, bool backward) -> (Tensor, "
        "Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(dion_b200, CUDA, m) { m.impl("window_attention_fwd", &bdion::window_attention_fwd); }
TORCH_LIBRARY_IMPL(dion_b200, Autograd, m) { m.impl("window_attention_fwd", &bdion::window_attention_fwd_checked); }
