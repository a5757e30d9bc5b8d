// Tensor-core kernels of the sliding-window attention (see window_attn.cu for
// the mathematics and the host side).
#pragma once
#include "ptx_attn.cuh"

namespace bdion {

struct WinArgs {
  int b, s, hq, hkv, d, window, sinks;
  int s_pad;        // positions rounded up to 128: row length of lse and delta
  float scale;      // 1 / sqrt(d)
  float scale_log2; // scale * log2(e)
  int* status;
  uint64_t limit_ns;
};

template <typename T>
struct AttnType;
template <>
struct AttnType<__nv_bfloat16> {
  static constexpr uint32_t kFmt = 1;
};
template <>
struct AttnType<__half> {
  static constexpr uint32_t kFmt = 0;
};

// The warps that issue products or hold rows run as a whole (see umma_ss; TMEM is
// read and written by whole warps), so they wait, and give up, as a whole.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort, uint64_t limit_ns) {
  return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort, limit_ns));
}

constexpr int kTile = 128;         // query rows of a CTA, and keys of a step
constexpr int kPanel = kTile * 128;  // bytes of 128 rows of one 128-byte swizzle row (64 elements)

// The key tiles that a tile of queries sees, in the order of their positions:
// those with first tokens that lie before the band, then the band's.
template <int NK>
struct KeyTiles {
  int n_first, band, n;
  __device__ __forceinline__ KeyTiles(const WinArgs& a, int q0) {
    band = max(0, q0 - a.window + 1) / NK;
    n_first = min((a.sinks + NK - 1) / NK, band);
    const int last = min(q0 + kTile, a.s) - 1;
    n = n_first + last / NK - band + 1;
  }
  __device__ __forceinline__ int k0(int t) const { return (t < n_first ? t : band + t - n_first) * NK; }
  // whether each of the 128 queries from q0 on sees each key of the tile at k0
  static __device__ __forceinline__ bool whole(const WinArgs& a, int q0, int k0) {
    return k0 + NK - 1 <= q0 && (q0 + kTile - 1 - k0 < a.window || k0 + NK <= a.sinks);
  }
};

// Query i sees one key: the first position always, every one with a window of one
// and no first tokens. P = 1 whatever the score there, so dS = 0 exactly, where
// dP - delta would be the difference of two fp32 sums of the same terms.
__device__ __forceinline__ bool all_see_one(const WinArgs& a) { return a.window == 1 && a.sinks == 0; }
__device__ __forceinline__ bool sees_one(const WinArgs& a, int i) { return i == 0 || all_see_one(a); }

// Which of 32 keys k0 .. k0 + 31 query i sees, as a bit mask.
__device__ __forceinline__ uint32_t seen_mask(const WinArgs& a, int i, int k0) {
  const int hi = i - k0;                       // last visible column
  const int lo = max(0, i - a.window + 1 - k0);  // first column of the band
  const int first = a.sinks - k0;              // columns before this one are first tokens
  uint32_t m = 0xffffffffu;
  if (lo > 0) m = lo >= 32 ? 0u : 0xffffffffu << lo;
  if (first > 0) m |= first >= 32 ? 0xffffffffu : (1u << first) - 1u;
  if (hi < 31) m &= hi < 0 ? 0u : 0xffffffffu >> (31 - hi);
  return m;
}

constexpr int kHalfTile = 64;               // keys (forward, dQ) or queries (dK, dV) of a step
constexpr int kHalfPanel = kHalfTile * 128;

template <typename T, int DP>
struct FwdCfg {
  static constexpr int kPanels = DP / 64;
  static constexpr int kRowBytes = kPanels * kPanel;       // Q
  static constexpr int kStepBytes = kPanels * kHalfPanel;  // K, V
  static constexpr int kStages = DP == 64 ? 3 : 2;
  static constexpr int kSmemBytes = kRowBytes + 2 * kStages * kStepBytes + 1024 + 256;
  static constexpr int kTmemCols = 256;
  static constexpr int kO = 256 - DP;  // columns: two buffers of S with P on it at 0 and 64, O at the end
};

// One CTA per (128 queries, head, sequence), steps of 64 keys; two CTAs share an
// SM. Warp 0 loads (TMA), warp 1 issues the products, warps 2-5 hold one query
// row per thread. S has two buffers, so the next step's scores are there when a
// row is done with this one's, and P V runs under the next step's exponentials.
//
// Measured in passes repeated for over a second (SM clock beside it; the power cap
// lowers it): 1 x 32763 positions, 8 heads of 128 on one key head, fp16, window 4096:
// 566 us, 0.92 PFLOP/s at 1507 MHz (485 us in a run too short for the cap); 1 x 8192,
// 32 heads of 128, window 2048, with o's remainder: 301 us at 1687 MHz (260); 2 x 4096,
// 32 heads of 64, window 1024: 134 us at 1882 MHz (127). Steps of 128 keys with one
// buffer of S: 309 us where these took 244, both without the remainder and in short
// runs. At 128 a product of 128 x 64 x 16 from shared memory takes about as long as one
// of 128 x 128 x 16, so S runs at half the tensor cores' rate; at 64 no unit is half
// busy, and the chain from TMEM load to TMEM store bounds it with the few warps (17 %)
// that two CTAs of four row warps are.
//
// A row's running maximum is the reference of its exponentials. It is moved
// only when a step exceeds it by more than 2^8, so O in TMEM is rarely rescaled;
// P <= 2^8 loses nothing in 16 bits (its rounding is relative) and the sum is
// kept in fp32 from the unrounded values.
template <typename T, int DP>
__global__ void __launch_bounds__(192, 2)
    window_fwd_tc(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                  const __grid_constant__ CUtensorMap tv, T* __restrict__ o, T* __restrict__ o_low,
                  float* __restrict__ neg_lse, const WinArgs a) {
  using Cfg = FwdCfg<T, DP>;
  constexpr int ST = Cfg::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + Cfg::kRowBytes;
  uint8_t* sV = sK + ST * Cfg::kStepBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + ST * Cfg::kStepBytes);
  uint64_t *q_full = bars, *k_full = bars + 1, *k_empty = bars + 4, *v_full = bars + 7, *v_empty = bars + 10,
           *s_full = bars + 13, *p_full = bars + 15, *o_done = bars + 17, *drain = bars + 19;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 20);
  volatile int* abort = reinterpret_cast<volatile int*>(bars + 21);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const int h = blockIdx.x % a.hq;
  const int n_q = a.s_pad / kTile;
  const int q0 = (blockIdx.x / a.hq) % n_q * kTile;
  const int b = blockIdx.x / a.hq / n_q;
  const int hk = h / (a.hq / a.hkv);
  const KeyTiles<kHalfTile> tiles(a, q0);

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < 3; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_done[i], 1);
    }
    mbar_init(drain, 1);
    *abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, Cfg::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint64_t limit = a.limit_ns;

  if (warp == 0) {
    if (lane == 0) {
      mbar_arrive_expect_tx(q_full, Cfg::kRowBytes);
      for (int p = 0; p < Cfg::kPanels; ++p) tma_load_4d(&tq, q_full, sQ + p * kPanel, p * 64, q0, h, b);
      int t = 0;
      bool ok = true;
      for (; t < tiles.n; ++t) {
        const int st = t % ST, k0 = tiles.k0(t);
        const uint32_t ph = (t / ST) & 1;
        if (!mbar_wait_bounded(&k_empty[st], ph ^ 1, abort, limit)) { ok = false; break; }
        mbar_arrive_expect_tx(&k_full[st], Cfg::kStepBytes);
        for (int p = 0; p < Cfg::kPanels; ++p)
          tma_load_4d(&tk, &k_full[st], sK + st * Cfg::kStepBytes + p * kHalfPanel, p * 64, k0, hk, b);
        if (!mbar_wait_bounded(&v_empty[st], ph ^ 1, abort, limit)) { ok = false; break; }
        mbar_arrive_expect_tx(&v_full[st], Cfg::kStepBytes);
        for (int p = 0; p < Cfg::kPanels; ++p)
          tma_load_4d(&tv, &v_full[st], sV + st * Cfg::kStepBytes + p * kHalfPanel, p * 64, k0, hk, b);
      }
      if (!ok) {
        report_status(a.status, kStatusWindowProducerTimeout);
        // copies in flight land before the shared memory is given up (bounded)
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(q_full, 0) && globaltimer_ns() - t0 < 100000000ull) {
        }
        for (int i = max(0, t - ST); i <= t; ++i) {
          while (!mbar_try_wait(&k_full[i % ST], (i / ST) & 1) && globaltimer_ns() - t0 < 100000000ull) {
          }
          while (!mbar_try_wait(&v_full[i % ST], (i / ST) & 1) && globaltimer_ns() - t0 < 100000000ull) {
          }
        }
      }
    }
  } else if (warp == 1) {
    const bool leader = elect_one();
    constexpr uint32_t kS = make_idesc(kTile, kHalfTile, false, false, AttnType<T>::kFmt);
    constexpr uint32_t kPV = make_idesc(kTile, DP, false, true, AttnType<T>::kFmt);
    const uint32_t q_base = smem_u32(sQ);
    bool ok = warp_wait(q_full, 0, abort, limit);
    auto scores = [&](int t) {
      const int st = t % ST, buf = t & 1;
      if (!warp_wait(&k_full[st], (t / ST) & 1, abort, limit)) return false;
      // the buffer's P of two steps ago has been read
      if (t >= 2 && !warp_wait(&o_done[buf], ((t >> 1) - 1) & 1, abort, limit)) return false;
      tc_fence_after();
      const uint32_t k_base = smem_u32(sK + st * Cfg::kStepBytes);
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        const uint32_t qo = (k / 4) * kPanel + (k % 4) * 32, ko = (k / 4) * kHalfPanel + (k % 4) * 32;
        umma_ss(leader, tmem + buf * 64, sdesc_low(q_base + qo, 16), sdesc_low(k_base + ko, 16), kS, k != 0);
      }
      umma_commit_by(leader, &k_empty[st]);
      umma_commit_by(leader, &s_full[buf]);
      return true;
    };
    if (ok) ok = scores(0);
    for (int t = 0; t < tiles.n && ok; ++t) {
      const int st = t % ST, buf = t & 1;
      if (t + 1 < tiles.n && !scores(t + 1)) { ok = false; break; }
      if (!warp_wait(&p_full[buf], (t >> 1) & 1, abort, limit)) { ok = false; break; }
      if (!warp_wait(&v_full[st], (t / ST) & 1, abort, limit)) { ok = false; break; }
      tc_fence_after();
      const uint32_t v_base = smem_u32(sV + st * Cfg::kStepBytes);
#pragma unroll
      for (int k = 0; k < kHalfTile / 16; ++k)
        umma_ts(leader, tmem + Cfg::kO, tmem + buf * 64 + k * 8, sdesc_low(v_base + k * 2048, kHalfPanel), kPV,
                (t | k) != 0);
      umma_commit_by(leader, &v_empty[st]);
      umma_commit_by(leader, &o_done[buf]);
    }
    if (!ok) {
      if (lane == 0) report_status(a.status, kStatusWindowMmaTimeout);
      umma_commit_by(leader, drain);
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(drain, 0) && globaltimer_ns() - t0 < 100000000ull) {
      }
    }
  } else {
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane, i = q0 + r;
    const uint32_t row = tmem + ((uint32_t)(quarter * 32) << 16);
    const float c = a.scale_log2;
    float m = -INFINITY, l = 0.f;  // reference of the exponentials (in score units), sum under it
    bool ok = true;
    for (int t = 0; t < tiles.n; ++t) {
      const int k0 = tiles.k0(t), buf = t & 1;
      if (!warp_wait(&s_full[buf], (t >> 1) & 1, abort, limit)) { ok = false; break; }
      tc_fence_after();
      uint32_t x[64], pk[32];
      auto load = [&] {
        tmem_ld_32x32b_x32(row + buf * 64, reinterpret_cast<uint32_t(&)[32]>(x[0]));
        tmem_ld_32x32b_x32(row + buf * 64 + 32, reinterpret_cast<uint32_t(&)[32]>(x[32]));
        tmem_wait_ld();
        if (!tiles.whole(a, q0, k0)) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t seen = seen_mask(a, i, k0 + j * 32);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!((seen >> e) & 1u)) x[j * 32 + e] = 0xff800000u;  // -inf
          }
        }
      };
      load();
      float mt[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int e = 0; e < 64; e += 2)
        mt[e / 2 % 4] = max3(mt[e / 2 % 4], __uint_as_float(x[e]), __uint_as_float(x[e + 1]));
      const float top = fmaxf(fmaxf(mt[0], mt[1]), fmaxf(mt[2], mt[3]));
      // move the reference where this step exceeds it by more than 8 powers of two
      float f = 1.f;
      if ((top - m) * c > 8.f) {  // also the first visible step (m = -inf); never while nothing is visible
        f = ex2((m - top) * c);
        m = top;
        l *= f;
      }
      const float mc = m == -INFINITY ? 0.f : m * c;
      const f2 c2 = make_f2(c, c), neg_mc = make_f2(-mc, -mc);
      f2 sum[2] = {};
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const f2 z = make_f2(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1]));
        const f2 p = ex2_pair(e, fma2(z, c2, neg_mc));
        sum[e % 2] = add2(sum[e % 2], p);
        pk[e] = pack2(p, T{});
      }
      sum[0] = add2(sum[0], sum[1]);
      l += lo_of(sum[0]) + hi_of(sum[0]);
      if (t > 0 && __any_sync(0xffffffffu, f != 1.f)) {
        // O is free once the step before is done
        if (!warp_wait(&o_done[buf ^ 1], ((t - 1) >> 1) & 1, abort, limit)) { ok = false; break; }
        tc_fence_after();
#pragma unroll
        for (int j = 0; j < DP / 32; ++j) {
          uint32_t y[32];
          tmem_ld_32x32b_x32(row + Cfg::kO + j * 32, y);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) y[e] = __float_as_uint(__uint_as_float(y[e]) * f);
          tmem_st_32x32b_x32(row + Cfg::kO + j * 32, y);
        }
      }
      tmem_st_32x32b_x32(row + buf * 64, pk);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[buf]);
    }
    // the last step's products stand for all before them
    if (ok) ok = warp_wait(&o_done[(tiles.n - 1) & 1], ((tiles.n - 1) >> 1) & 1, abort, limit);
    if (!ok) {
      if (lane == 0) report_status(a.status, kStatusWindowSoftmaxTimeout);
    } else {
      tc_fence_after();
      const bool real = i < a.s;
      neg_lse[((int64_t)b * a.hq + h) * a.s_pad + i] = real ? -(m * c + log2f(l)) : -INFINITY;
      const float inv = 1.f / l;
      const int64_t orow = (((int64_t)b * a.s + i) * a.hq + h) * a.d;
#pragma unroll
      for (int j = 0; j < DP / 32; ++j) {
        uint32_t y[32];
        tmem_ld_32x32b_x32(row + Cfg::kO + j * 32, y);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          if (real && j * 32 + e < a.d) {
            // o, and what its rounding left out: the backward pass takes delta = do . o from
            // both. Where one key has nearly all of a row, dP - delta is far smaller than
            // its terms, and the rounding of o alone made it off by as much as itself.
            uint4 u, v;
            uint32_t *hi = reinterpret_cast<uint32_t*>(&u), *lo = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              const float x0 = __uint_as_float(y[e + 2 * n]) * inv, x1 = __uint_as_float(y[e + 2 * n + 1]) * inv;
              hi[n] = pack2(x0, x1, T{});
              const T* r = reinterpret_cast<const T*>(&hi[n]);
              lo[n] = pack2(x0 - (float)r[0], x1 - (float)r[1], T{});
            }
            *reinterpret_cast<uint4*>(o + orow + j * 32 + e) = u;
            if (o_low != nullptr) *reinterpret_cast<uint4*>(o_low + orow + j * 32 + e) = v;
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, Cfg::kTmemCols);
}

// ------------------------------------------------------------ backward: dQ
// Column of the 16 elements that product k of a step reads. Each of the four
// threads of a row packs its 32 elements into the first 16 of the 32 columns
// that it has read itself, so none waits for another.
__device__ constexpr int part_col(int k) { return k / 2 * 32 + k % 2 * 8; }

template <typename T, int DP>
struct DqCfg {
  static constexpr int kPanels = DP / 64;
  static constexpr int kRowBytes = kPanels * kPanel;  // Q, dO; K, V of a step
  // K stays until its step's dQ, so the step after next needs a third place for it
  static constexpr int kStagesK = 3, kStagesV = 2;
  static constexpr int kSmemBytes = (2 + kStagesK + kStagesV) * kRowBytes + 1024 + 256 + kTile * 4;
  static constexpr int kTmemCols = 512;
  // columns: S at 0, two buffers of dP with dS on them, dQ
  static constexpr int kDP = 128, kDQ = 384;
};

// One CTA per (128 queries, head, sequence), one to an SM, steps of 128 keys: S
// and dP by the tensor cores, dS = P o (dP - delta) by four threads per query
// row (a quarter of the step's keys each), dQ += dS K with dS read from TMEM.
// The next step's S is computed as soon as the rows have read this one's, its dP
// goes into the other buffer, so the rows work from step to step without waiting
// for the sums. (Steps of 64 keys: a product of 128 x 64 x 16 takes as long from
// shared memory as one of 128 x 128 x 16; 492 us where this took 389 in short runs, 1 x
// 8192, 32 heads of 128, window 2048. At 64 both took about 182 us at 2 x 4096, 32
// heads, window 1024.) In passes repeated for over a second: 450 us at 1687 MHz and 197
// us at 1882 MHz. At 128 the tensor cores bound it, 24 products of 128 x 128 x 16 a step
// at some 80 cycles; at 64 the chain S, rows, dQ, with 28 % of the warps. delta is taken
// here from O and dO and kept, negated, for the dK / dV kernel (0 behind the last
// position).
template <typename T, int DP>
__global__ void __launch_bounds__(576, 1)
    window_dq_tc(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                 const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap tg,
                 const T* __restrict__ o, const T* __restrict__ o_low, const T* __restrict__ go, int64_t go_b, int64_t go_s, int64_t go_h,
                 const float* __restrict__ neg_lse, float* __restrict__ neg_delta, T* __restrict__ dq,
                 const WinArgs a) {
  using Cfg = DqCfg<T, DP>;
  constexpr int SK = Cfg::kStagesK, SV = Cfg::kStagesV;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sG = sQ + Cfg::kRowBytes;
  uint8_t* sK = sG + Cfg::kRowBytes;
  uint8_t* sV = sK + SK * Cfg::kRowBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + SV * Cfg::kRowBytes);
  uint64_t *q_full = bars, *k_full = bars + 1, *k_empty = bars + 4, *v_full = bars + 7, *v_empty = bars + 9,
           *s_full = bars + 11, *s_read = bars + 12, *dp_full = bars + 13, *ds_full = bars + 15, *dq_done = bars + 17,
           *all_done = bars + 19, *drain = bars + 20;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 21);
  volatile int* abort = reinterpret_cast<volatile int*>(bars + 22);
  float* s_delta = reinterpret_cast<float*>(bars + 24);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const int h = blockIdx.x % a.hq;
  const int n_q = a.s_pad / kTile;
  const int q0 = (blockIdx.x / a.hq) % n_q * kTile;
  const int b = blockIdx.x / a.hq / n_q;
  const int hk = h / (a.hq / a.hkv);
  const KeyTiles<kTile> tiles(a, q0);

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(s_full, 1);
    mbar_init(s_read, 16);
    for (int i = 0; i < SK; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&dp_full[i], 1);
      mbar_init(&ds_full[i], 16);
      mbar_init(&dq_done[i], 1);
    }
    mbar_init(all_done, 1);
    mbar_init(drain, 1);
    *abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, Cfg::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint64_t limit = a.limit_ns;

  if (warp == 0) {
    if (lane == 0) {
      mbar_arrive_expect_tx(q_full, 2 * Cfg::kRowBytes);
      for (int p = 0; p < Cfg::kPanels; ++p) {
        tma_load_4d(&tq, q_full, sQ + p * kPanel, p * 64, q0, h, b);
        tma_load_4d(&tg, q_full, sG + p * kPanel, p * 64, q0, h, b);
      }
      int t = 0;
      bool ok = true;
      for (; t < tiles.n; ++t) {
        const int sk = t % SK, sv = t % SV, k0 = tiles.k0(t);
        // K is free once dQ is done, V already after dP
        if (!mbar_wait_bounded(&k_empty[sk], ((t / SK) & 1) ^ 1, abort, limit)) { ok = false; break; }
        mbar_arrive_expect_tx(&k_full[sk], Cfg::kRowBytes);
        for (int p = 0; p < Cfg::kPanels; ++p)
          tma_load_4d(&tk, &k_full[sk], sK + sk * Cfg::kRowBytes + p * kPanel, p * 64, k0, hk, b);
        if (!mbar_wait_bounded(&v_empty[sv], ((t / SV) & 1) ^ 1, abort, limit)) { ok = false; break; }
        mbar_arrive_expect_tx(&v_full[sv], Cfg::kRowBytes);
        for (int p = 0; p < Cfg::kPanels; ++p)
          tma_load_4d(&tv, &v_full[sv], sV + sv * Cfg::kRowBytes + p * kPanel, p * 64, k0, hk, b);
      }
      if (!ok) {
        report_status(a.status, kStatusWindowProducerTimeout);
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(q_full, 0) && globaltimer_ns() - t0 < 100000000ull) {
        }
        for (int i = max(0, t - SK); i <= t; ++i) {
          while (!mbar_try_wait(&k_full[i % SK], (i / SK) & 1) && globaltimer_ns() - t0 < 100000000ull) {
          }
          while (!mbar_try_wait(&v_full[i % SV], (i / SV) & 1) && globaltimer_ns() - t0 < 100000000ull) {
          }
        }
      }
    }
  } else if (warp == 1) {
    const bool leader = elect_one();
    constexpr uint32_t kS = make_idesc(kTile, kTile, false, false, AttnType<T>::kFmt);
    constexpr uint32_t kD = make_idesc(kTile, DP, false, true, AttnType<T>::kFmt);
    const uint32_t q_base = smem_u32(sQ), g_base = smem_u32(sG);
    bool ok = warp_wait(q_full, 0, abort, limit);
    auto scores = [&](int t) {  // S of step t; the rows have read the step before it
      if (!warp_wait(&k_full[t % SK], (t / SK) & 1, abort, limit)) return false;
      if (t > 0 && !warp_wait(s_read, (t - 1) & 1, abort, limit)) return false;
      tc_fence_after();
      const uint32_t k_base = smem_u32(sK + t % SK * Cfg::kRowBytes);
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        const uint32_t off = (k / 4) * kPanel + (k % 4) * 32;
        umma_ss(leader, tmem, sdesc_low(q_base + off, 16), sdesc_low(k_base + off, 16), kS, k != 0);
      }
      umma_commit_by(leader, s_full);
      return true;
    };
    auto grads = [&](int t) {  // dP of step t; its buffer's dS of two steps ago has been read
      if (!warp_wait(&v_full[t % SV], (t / SV) & 1, abort, limit)) return false;
      if (t >= 2 && !warp_wait(&dq_done[t & 1], ((t >> 1) - 1) & 1, abort, limit)) return false;
      tc_fence_after();
      const uint32_t v_base = smem_u32(sV + t % SV * Cfg::kRowBytes);
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        const uint32_t off = (k / 4) * kPanel + (k % 4) * 32;
        umma_ss(leader, tmem + Cfg::kDP + (t & 1) * 128, sdesc_low(g_base + off, 16), sdesc_low(v_base + off, 16), kS,
                k != 0);
      }
      umma_commit_by(leader, &v_empty[t % SV]);
      umma_commit_by(leader, &dp_full[t & 1]);
      return true;
    };
    if (ok) ok = scores(0) && grads(0);
    for (int t = 0; t < tiles.n && ok; ++t) {
      if (t + 1 < tiles.n && !(scores(t + 1) && grads(t + 1))) { ok = false; break; }
      if (!warp_wait(&ds_full[t & 1], (t >> 1) & 1, abort, limit)) { ok = false; break; }
      tc_fence_after();
      const uint32_t k_base = smem_u32(sK + t % SK * Cfg::kRowBytes);
#pragma unroll
      for (int k = 0; k < kTile / 16; ++k)
        umma_ts(leader, tmem + Cfg::kDQ, tmem + Cfg::kDP + (t & 1) * 128 + part_col(k), sdesc_low(k_base + k * 2048, kPanel),
                kD, (t | k) != 0);
      umma_commit_by(leader, &k_empty[t % SK]);
      umma_commit_by(leader, &dq_done[t & 1]);
    }
    if (ok) {
      umma_commit_by(leader, all_done);
    } else {
      if (lane == 0) report_status(a.status, kStatusWindowMmaTimeout);
      umma_commit_by(leader, drain);
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(drain, 0) && globaltimer_ns() - t0 < 100000000ull) {
      }
    }
  } else {
    const int quarter = warp & 3, part = (warp - 2) / 4;
    const int r = quarter * 32 + lane, i = q0 + r;
    const uint32_t row = tmem + ((uint32_t)(quarter * 32) << 16);
    const int64_t at = ((int64_t)b * a.hq + h) * a.s_pad + q0;
    // a row that sees one key: P = 0 here, for its dS
    const float nl = sees_one(a, i) ? neg_lse[at + r] - INFINITY : neg_lse[at + r];
    const f2 c2 = make_f2(a.scale_log2, a.scale_log2), neg_l = make_f2(nl, nl);
    {
      // delta of 8 rows per warp, DP / 8 lanes to a row
      constexpr int kLanes = DP / 8, kRows = 32 / kLanes;
      const int col = lane % kLanes * 8;
      float v[8 / kRows];
#pragma unroll
      for (int n = 0; n < 8 / kRows; ++n) {
        const int rr = q0 + (warp - 2) * 8 + n * kRows + lane / kLanes;
        v[n] = 0.f;
        if (rr < a.s && col < a.d) {
          const int64_t at_o = (((int64_t)b * a.s + rr) * a.hq + h) * a.d + col;
          const uint4 ou = *reinterpret_cast<const uint4*>(o + at_o), lu = *reinterpret_cast<const uint4*>(o_low + at_o);
          const uint4 gu = *reinterpret_cast<const uint4*>(go + b * go_b + rr * go_s + h * go_h + col);
          const T *op = reinterpret_cast<const T*>(&ou), *lp = reinterpret_cast<const T*>(&lu),
                  *gp = reinterpret_cast<const T*>(&gu);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[n] += ((float)op[e] + (float)lp[e]) * (float)gp[e];
        }
      }
#pragma unroll
      for (int n = 0; n < 8 / kRows; ++n) {
#pragma unroll
        for (int m = kLanes / 2; m > 0; m >>= 1) v[n] += __shfl_xor_sync(0xffffffffu, v[n], m);
        const int rr = (warp - 2) * 8 + n * kRows + lane / kLanes;
        if (col == 0) {
          s_delta[rr] = -v[n];
          neg_delta[at + rr] = -v[n];
        }
      }
      asm volatile("bar.sync 1, 512;" ::: "memory");
    }
    const f2 neg_d = make_f2(s_delta[r], s_delta[r]);
    bool ok = true;
    for (int t = 0; t < tiles.n; ++t) {
      const int k0 = tiles.k0(t);
      if (!warp_wait(s_full, t & 1, abort, limit)) { ok = false; break; }
      tc_fence_after();
      uint32_t x[32];
      f2 p[16];
      tmem_ld_32x32b_x32(row + part * 32, x);
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_read);
      if (!tiles.whole(a, q0, k0)) {
        const uint32_t seen = seen_mask(a, i, k0 + part * 32);
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (!((seen >> e) & 1u)) x[e] = 0xff800000u;  // -inf
      }
#pragma unroll
      for (int e = 0; e < 16; ++e)
        p[e] = ex2_pair(e, fma2(make_f2(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])), c2, neg_l));
      if (!warp_wait(&dp_full[t & 1], (t >> 1) & 1, abort, limit)) { ok = false; break; }
      tc_fence_after();
      const uint32_t buf = row + Cfg::kDP + (t & 1) * 128 + part * 32;
      tmem_ld_32x32b_x32(buf, x);
      tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 16; ++e)
        x[e] = pack2(mul2(p[e], add2(make_f2(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])), neg_d)), T{});
      tmem_st_32x32b_x16(buf, x);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ds_full[t & 1]);
    }
    if (ok) ok = warp_wait(all_done, 0, abort, limit);
    if (!ok) {
      if (lane == 0) report_status(a.status, kStatusWindowSoftmaxTimeout);
    } else {
      tc_fence_after();
      T* out = dq + (((int64_t)b * a.s + i) * a.hq + h) * a.d;
      for (int j = part; j < DP / 32; j += 4) {
        uint32_t y[32];
        tmem_ld_32x32b_x32(row + Cfg::kDQ + j * 32, y);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          if (i < a.s && j * 32 + e < a.d) {
            uint4 u;
            uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
            for (int n = 0; n < 4; ++n)
              w[n] = pack2(__uint_as_float(y[e + 2 * n]) * a.scale, __uint_as_float(y[e + 2 * n + 1]) * a.scale, T{});
            *reinterpret_cast<uint4*>(out + j * 32 + e) = u;
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, Cfg::kTmemCols);
}

// ------------------------------------------------------------ backward: dK, dV
// How the key tiles' steps (a step: 128 queries of one head) are split over
// CTAs. The queries that see first tokens reach to the end of the sequence,
// those of every other tile only as far as the window: the tiles with first
// tokens are cut into `c_first` parts, the others into `c_band`. A part of a
// cut tile writes fp32 sums to its slot of the workspace, and a second kernel
// adds the slots in order.
struct KeySplit {
  int n_tiles, n_first;   // key tiles, and those that hold first tokens
  int c_first, c_band;
  __host__ __device__ __forceinline__ int parts() const { return n_first * c_first + (n_tiles - n_first) * c_band; }
  // parts of tile `tile`, and the number of the first of them
  __host__ __device__ __forceinline__ int of(int tile) const { return tile < n_first ? c_first : c_band; }
  __host__ __device__ __forceinline__ int first_part(int tile) const {
    return tile < n_first ? tile * c_first : n_first * c_first + (tile - n_first) * c_band;
  }
  // workspace slots: parts of cut tiles only
  __host__ __device__ __forceinline__ int slots() const {
    return (c_first > 1 ? n_first * c_first : 0) + (c_band > 1 ? (n_tiles - n_first) * c_band : 0);
  }
  __host__ __device__ __forceinline__ int slot(int tile) const {
    return tile < n_first ? tile * c_first : (c_first > 1 ? n_first * c_first : 0) + (tile - n_first) * c_band;
  }
};

template <typename T, int DP>
struct DkvCfg {
  static constexpr int kPanels = DP / 64;
  static constexpr int kRowBytes = kPanels * kPanel;  // K, V; Q, dO of a step
  static constexpr int kStages = DP == 64 ? 3 : 2;
  static constexpr int kStatBytes = kTile * 4;
  static constexpr int kSmemBytes = 2 * kRowBytes + kStages * (2 * kRowBytes + 2 * kStatBytes) + 1024 + 256;
  static constexpr int kTmemCols = 512;
  // columns: S^T at 0, buffers of dP^T (two where there is room) with P^T and dS^T on
  // them, dV, dK
  static constexpr int kBufs = DP == 64 ? 2 : 1;
  static constexpr int kDPT = 128, kDV = kDPT + kBufs * 128, kDK = kDV + DP;
};

// One CTA per (128 keys, key head, sequence, part), steps of 128 queries of one
// head. With the keys as rows, P^T and dS^T come out of TMEM in the place where
// dV += P^T dO and dK += dS^T Q want their A operand, so neither passes through
// shared memory. Four threads share a key row, a quarter of the step's queries
// each: a thread reads its 32 columns of dP^T and packs P^T and dS^T into them,
// so S^T is free for the next step as soon as it has been read. 2 x 4096, 32 heads of
// 64 on 8, window 1024, in short runs: 191 us (216 with P^T on S^T, 273 in steps of 64
// queries); 1 x 8192, 32 heads of 128 on 8, window 2048: 521 us (508, 540). In passes
// repeated for over a second: 201 us at 1882 MHz and 606 us at 1687 MHz. At 128 TMEM has
// room for one buffer of dP^T, and the chain dP^T -> rows -> dV, dK -> next dP^T bounds it.
template <typename T, int DP>
__global__ void __launch_bounds__(576, 1)
    window_dkv_tc(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                  const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap tg,
                  const float* __restrict__ neg_lse, const float* __restrict__ neg_delta, T* __restrict__ dk,
                  T* __restrict__ dv, float* __restrict__ work, const KeySplit split, const WinArgs a) {
  using Cfg = DkvCfg<T, DP>;
  constexpr int ST = Cfg::kStages, NB = Cfg::kBufs;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sK = smem;
  uint8_t* sV = sK + Cfg::kRowBytes;
  uint8_t* sQ = sV + Cfg::kRowBytes;
  uint8_t* sG = sQ + ST * Cfg::kRowBytes;
  float* sL = reinterpret_cast<float*>(sG + ST * Cfg::kRowBytes);
  float* sD = sL + ST * kTile;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sD + ST * kTile);
  uint64_t *k_full = bars, *q_full = bars + 1, *q_empty = bars + 4, *s_full = bars + 7, *s_read = bars + 8,
           *dp_full = bars + 9, *ds_full = bars + 11, *acc_done = bars + 13, *all_done = bars + 15, *drain = bars + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 18);
  volatile int* abort = reinterpret_cast<volatile int*>(bars + 19);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const int hk = blockIdx.x % a.hkv, group = a.hq / a.hkv;
  const int part = (blockIdx.x / a.hkv) % split.parts();
  const int b = blockIdx.x / a.hkv / split.parts();
  const int in_first = split.n_first * split.c_first;
  const int tile = part < in_first ? part / split.c_first : split.n_first + (part - in_first) / split.c_band;
  const int parts = split.of(tile), mine = part - split.first_part(tile);
  const int k0 = tile * kTile;
  // steps of the whole tile, and this part's
  const int q_first = k0 / kTile;
  const int last_key = min(k0 + kTile, a.s) - 1;
  const int q_last = (k0 < a.sinks ? a.s - 1 : (int)min((int64_t)a.s - 1, (int64_t)last_key + a.window - 1)) / kTile;
  const int nq = q_last - q_first + 1;
  const int64_t all = (int64_t)nq * group;
  const int lo = (int)(all * mine / parts), n = (int)(all * (mine + 1) / parts) - lo;

  if (threadIdx.x == 0) {
    mbar_init(k_full, 1);
    for (int i = 0; i < ST; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
    }
    mbar_init(s_full, 1);
    mbar_init(s_read, 16);
    for (int i = 0; i < NB; ++i) {
      mbar_init(&dp_full[i], 1);
      mbar_init(&ds_full[i], 16);
      mbar_init(&acc_done[i], 1);
    }
    mbar_init(all_done, 1);
    mbar_init(drain, 1);
    *abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, Cfg::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint64_t limit = a.limit_ns;

  if (warp == 0) {
    if (lane == 0 && n > 0) {
      mbar_arrive_expect_tx(k_full, 2 * Cfg::kRowBytes);
      for (int p = 0; p < Cfg::kPanels; ++p) {
        tma_load_4d(&tk, k_full, sK + p * kPanel, p * 64, k0, hk, b);
        tma_load_4d(&tv, k_full, sV + p * kPanel, p * 64, k0, hk, b);
      }
      bool ok = true;
      int t = 0;
      for (; t < n; ++t) {
        const int st = t % ST;
        const int h = hk * group + (lo + t) / nq, q0 = (q_first + (lo + t) % nq) * kTile;
        if (!mbar_wait_bounded(&q_empty[st], ((t / ST) & 1) ^ 1, abort, limit)) { ok = false; break; }
        mbar_arrive_expect_tx(&q_full[st], 2 * Cfg::kRowBytes + 2 * Cfg::kStatBytes);
        for (int p = 0; p < Cfg::kPanels; ++p) {
          tma_load_4d(&tq, &q_full[st], sQ + st * Cfg::kRowBytes + p * kPanel, p * 64, q0, h, b);
          tma_load_4d(&tg, &q_full[st], sG + st * Cfg::kRowBytes + p * kPanel, p * 64, q0, h, b);
        }
        const int64_t at = ((int64_t)b * a.hq + h) * a.s_pad + q0;
        bulk_load(sL + st * kTile, neg_lse + at, Cfg::kStatBytes, &q_full[st]);
        bulk_load(sD + st * kTile, neg_delta + at, Cfg::kStatBytes, &q_full[st]);
      }
      if (!ok) {
        report_status(a.status, kStatusWindowProducerTimeout);
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(k_full, 0) && globaltimer_ns() - t0 < 100000000ull) {
        }
        for (int i = max(0, t - ST); i < t; ++i)
          while (!mbar_try_wait(&q_full[i % ST], (i / ST) & 1) && globaltimer_ns() - t0 < 100000000ull) {
          }
      }
    }
  } else if (warp == 1) {
    if (n > 0) {
      const bool leader = elect_one();
      constexpr uint32_t kS = make_idesc(kTile, kTile, false, false, AttnType<T>::kFmt);
      constexpr uint32_t kD = make_idesc(kTile, DP, false, true, AttnType<T>::kFmt);
      const uint32_t k_base = smem_u32(sK), v_base = smem_u32(sV);
      bool ok = warp_wait(k_full, 0, abort, limit);
      auto scores = [&](int t) {  // S^T of step t; the rows have read the one before
        if (!warp_wait(&q_full[t % ST], (t / ST) & 1, abort, limit)) return false;
        if (t > 0 && !warp_wait(s_read, (t - 1) & 1, abort, limit)) return false;
        tc_fence_after();
        const uint32_t q_base = smem_u32(sQ + t % ST * Cfg::kRowBytes);
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          const uint32_t off = (k / 4) * kPanel + (k % 4) * 32;
          umma_ss(leader, tmem, sdesc_low(k_base + off, 16), sdesc_low(q_base + off, 16), kS, k != 0);
        }
        umma_commit_by(leader, s_full);
        return true;
      };
      auto grads = [&](int t) {  // dP^T of step t; P^T and dS^T in its buffer have been read
        if (!warp_wait(&q_full[t % ST], (t / ST) & 1, abort, limit)) return false;
        if (t >= NB && !warp_wait(&acc_done[t % NB], (t / NB - 1) & 1, abort, limit)) return false;
        tc_fence_after();
        const uint32_t g_base = smem_u32(sG + t % ST * Cfg::kRowBytes);
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          const uint32_t off = (k / 4) * kPanel + (k % 4) * 32;
          umma_ss(leader, tmem + Cfg::kDPT + t % NB * 128, sdesc_low(v_base + off, 16), sdesc_low(g_base + off, 16), kS,
                  k != 0);
        }
        umma_commit_by(leader, &dp_full[t % NB]);
        return true;
      };
      if (ok) ok = scores(0) && grads(0);
      for (int t = 0; t < n && ok; ++t) {
        const int st = t % ST;
        const uint32_t q_base = smem_u32(sQ + st * Cfg::kRowBytes), g_base = smem_u32(sG + st * Cfg::kRowBytes);
        const uint32_t pds = tmem + Cfg::kDPT + t % NB * 128;
        if (t + 1 < n && !scores(t + 1)) { ok = false; break; }
        if (NB == 2 && t + 1 < n && !grads(t + 1)) { ok = false; break; }
        if (!warp_wait(&ds_full[t % NB], (t / NB) & 1, abort, limit)) { ok = false; break; }
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < kTile / 16; ++k) {
          umma_ts(leader, tmem + Cfg::kDV, pds + part_col(k), sdesc_low(g_base + k * 2048, kPanel), kD, (t | k) != 0);
          umma_ts(leader, tmem + Cfg::kDK, pds + part_col(k) + 16, sdesc_low(q_base + k * 2048, kPanel), kD, (t | k) != 0);
        }
        umma_commit_by(leader, &q_empty[st]);
        umma_commit_by(leader, &acc_done[t % NB]);
        if (NB == 1 && t + 1 < n && !grads(t + 1)) { ok = false; break; }
      }
      if (ok) {
        umma_commit_by(leader, all_done);
      } else {
        if (lane == 0) report_status(a.status, kStatusWindowMmaTimeout);
        umma_commit_by(leader, drain);
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(drain, 0) && globaltimer_ns() - t0 < 100000000ull) {
        }
      }
    }
  } else {
    const int quarter = warp & 3, part = (warp - 2) / 4;
    const int r = quarter * 32 + lane, j = k0 + r;
    const uint32_t row = tmem + ((uint32_t)(quarter * 32) << 16);
    const f2 c2 = make_f2(a.scale_log2, a.scale_log2);
    bool ok = true;
    int qt = lo % nq, st = 0;  // this step's query tile (from q_first) and stage
    for (int t = 0; t < n; ++t) {
      const int q0 = (q_first + qt) * kTile;
      const uint32_t pds = row + Cfg::kDPT + t % NB * 128 + part * 32;
      // (the stage's copies as well: the rows read lse and delta from it)
      if (!warp_wait(&q_full[st], (t / ST) & 1, abort, limit)) { ok = false; break; }
      if (!warp_wait(s_full, t & 1, abort, limit)) { ok = false; break; }
      tc_fence_after();
      uint32_t x[32], y[32];
      f2 p[16];
      tmem_ld_32x32b_x32(row + part * 32, x);
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_read);
      // queries q0 + e that see key j: e in [j - q0, j + window - q0), without an end for first tokens
      if (!(q0 >= k0 + kTile - 1 && (q0 + kTile - 1 - k0 < a.window || k0 + kTile <= a.sinks))) {
        const int e0 = j - q0 - part * 32;
        const int e1 = j < a.sinks ? kTile : (int)min((int64_t)kTile, (int64_t)j + a.window - q0 - part * 32);
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (e < e0 || e >= e1) x[e] = 0xff800000u;  // -inf
      }
      const float *pl = sL + st * kTile + part * 32, *pd = sD + st * kTile + part * 32;
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const ulonglong2 L = *reinterpret_cast<const ulonglong2*>(pl + 2 * e);
        p[e] = ex2_pair(e, fma2(make_f2(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])), c2, L.x));
        p[e + 1] = ex2_pair(e + 1, fma2(make_f2(__uint_as_float(x[2 * e + 2]), __uint_as_float(x[2 * e + 3])), c2, L.y));
      }
      if (!warp_wait(&dp_full[t % NB], (t / NB) & 1, abort, limit)) { ok = false; break; }
      tc_fence_after();
      tmem_ld_32x32b_x32(pds, x);
      tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const ulonglong2 D = *reinterpret_cast<const ulonglong2*>(pd + 2 * e);
        const f2 g0 = make_f2(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1]));
        const f2 g1 = make_f2(__uint_as_float(x[2 * e + 2]), __uint_as_float(x[2 * e + 3]));
        y[e] = pack2(p[e], T{});
        y[e + 1] = pack2(p[e + 1], T{});
        // query 0's dS is 0 (see sees_one)
        const f2 p0 = e == 0 && q0 + part == 0 ? make_f2(0.f, hi_of(p[0])) : p[e];
        y[16 + e] = pack2(mul2(p0, add2(g0, D.x)), T{});
        y[16 + e + 1] = pack2(mul2(p[e + 1], add2(g1, D.y)), T{});
      }
      tmem_st_32x32b_x32(pds, y);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ds_full[t % NB]);
      qt = qt + 1 == nq ? 0 : qt + 1;
      st = st + 1 == ST ? 0 : st + 1;
    }
    if (ok && n > 0) ok = warp_wait(all_done, 0, abort, limit);
    if (!ok) {
      if (lane == 0) report_status(a.status, kStatusWindowSoftmaxTimeout);
    } else {
      tc_fence_after();
      // two of a row's threads store dV, two dK, half of the row each
      const uint32_t acc = row + (part < 2 ? Cfg::kDV : Cfg::kDK);
      const float f = part < 2 ? 1.f : all_see_one(a) ? 0.f : a.scale;
      T* out = (part < 2 ? dv : dk) + (((int64_t)b * a.s + j) * a.hkv + hk) * a.d;
      float* slot = nullptr;
      if (parts > 1)
        slot = work + ((((int64_t)b * a.hkv + hk) * split.slots() + split.slot(tile) + mine) * 2 + part / 2) * kTile * DP +
               (int64_t)r * DP;
#pragma unroll
      for (int j2 = part % 2 * (DP / 64); j2 < (part % 2 + 1) * (DP / 64); ++j2) {
        uint32_t y[32];
        if (n > 0) {
          tmem_ld_32x32b_x32(acc + j2 * 32, y);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) y[e] = 0u;
        }
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          float v[8];
#pragma unroll
          for (int n2 = 0; n2 < 8; ++n2) v[n2] = __uint_as_float(y[e + n2]) * f;
          if (slot != nullptr) {
            store8(slot + j2 * 32 + e, v);
          } else if (j < a.s && j2 * 32 + e < a.d) {
            uint4 u;
            uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
            for (int n2 = 0; n2 < 4; ++n2) w[n2] = pack2(v[2 * n2], v[2 * n2 + 1], T{});
            *reinterpret_cast<uint4*>(out + j2 * 32 + e) = u;
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, Cfg::kTmemCols);
}

// dK / dV of the cut tiles: the sum of their parts' slots, in order. One block
// per 16 rows of (tile, key head, sequence, dK or dV).
template <typename T, int DP>
__global__ void __launch_bounds__(16 * DP / 8)
    window_dkv_join(const float* __restrict__ work, T* __restrict__ dk, T* __restrict__ dv, const KeySplit split,
                    int tile0, const WinArgs a) {
  const int which = blockIdx.x % 2, r = blockIdx.x / 2 % (kTile / 16) * 16 + threadIdx.x / (DP / 8);
  const int rest = blockIdx.x / (2 * kTile / 16);
  const int hk = rest % a.hkv, b = rest / a.hkv % a.b, tile = tile0 + rest / a.hkv / a.b;
  const int col = threadIdx.x % (DP / 8) * 8, j = tile * kTile + r;
  if (j >= a.s || col >= a.d) return;
  const float* p = work + (((int64_t)b * a.hkv + hk) * split.slots() + split.slot(tile)) * 2 * kTile * DP +
                   (int64_t)which * kTile * DP + (int64_t)r * DP + col;
  float s[8] = {};
  for (int i = 0; i < split.of(tile); ++i) {
    float v[8];
    load8(p + (int64_t)i * 2 * kTile * DP, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] += v[e];
  }
  uint4 u;
  uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = pack2(s[2 * e], s[2 * e + 1], T{});
  *reinterpret_cast<uint4*>((which == 0 ? dv : dk) + (((int64_t)b * a.s + j) * a.hkv + hk) * a.d + col) = u;
}

}  // namespace bdion
