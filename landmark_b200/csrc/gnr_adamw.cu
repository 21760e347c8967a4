// One AdamW step over many tensors.
//
//   m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2,
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// in fp32 whatever the types of p and g; with a 32-bit copy ("master") of a 16-bit p, that copy is the parameter and p its
// rounded image.  Every value is read once and written once: bound by HBM.  The tensors' addresses travel as a kernel
// argument, so nothing about them is kept between calls and a captured graph needs no table in memory.
//
// States in 8 bits: blocks of 256 values of a tensor share two fp32 scales, m = s_m c and v = (s_v c)^2 with e4m3 codes c
// and s = (largest in the block) / 448.  The square root halves v's range in the exponent: an e4m3 code reaches 2^-17.8 of
// the largest one, v then 2^-35.6 of it.  Codes are rounded up or down at random, with the probability that keeps
// the mean of m and the mean of v: a step with b2 = 0.999 changes v by a thousandth of itself, a code is an eighth of v
// wide, so rounding to nearest would never move it.  The random bits are a hash of seed, step, tensor and place (16 for m,
// 16 for v).  A positive v is never rounded to 0, which would make its next step as large as |m| / eps.
// The arithmetic of the codes is in separately rounded operations (no fused multiply-add), so that the codes of equal
// inputs are equal wherever they are computed.
#include <cuda_fp8.h>
#include <math.h>
#include <string.h>

#include "gnr_internal.cuh"
#include "gnr_types.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kBlock = GNR_ADAMW_BLOCK;
constexpr int kChunk = 4096;  // values of a thread block: 16 blocks of codes
constexpr float kTop = 448.0f;

struct Tensor {
  void* p;
  const void* g;
  void* m;
  void* v;
  float* m_scale;
  float* v_scale;
  float* master;
  int64_t n;
  uint32_t first;  // thread blocks before this tensor's
  uint32_t seed;
};

struct Hyper {
  float b1, b1c, b2, b2c;  // betas and 1 - betas
  float keep;              // 1 - lr * weight decay
  float rate;              // lr / (1 - b1^t)
  float c2;                // sqrt(1 - b2^t)
  float eps;
};

template <int K> struct Table {
  Hyper h;
  int n;
  Tensor t[K];
};
constexpr int kSmall = 24, kLarge = 400;  // tensors of a launch: 2 and 32 KB of arguments
static_assert(sizeof(Table<kLarge>) <= 32764, "kernel arguments");

__host__ __device__ __forceinline__ uint32_t hash32(uint32_t i, uint32_t seed) {
  // multiplicative hashing: an odd number near 2^32 / golden ratio, then the fractional bits of the square roots of 2 and 3
  uint32_t x = i * 0x9E3779B9u + seed;
  x ^= x >> 16;
  x *= 0x6A09E667u;
  x ^= x >> 15;
  x *= 0xBB67AE85u;
  return x ^ (x >> 16);
}

// m and v after the gradient g
__device__ __forceinline__ void moments(const Hyper& h, float g, float& m, float& v) {
  m = __fadd_rn(__fmul_rn(h.b1, m), __fmul_rn(h.b1c, g));
  v = __fadd_rn(__fmul_rn(h.b2, v), __fmul_rn(__fmul_rn(h.b2c, g), g));
}

__device__ __forceinline__ float stepped(const Hyper& h, float x, float m, float root) {
  return x * h.keep - h.rate * (m / (root / h.c2 + h.eps));
}

// `count` (at most 4) neighbours from `at`, as one access where all four are there and `wide`
template <typename T> __device__ __forceinline__ void load4(const T* at, bool whole, int count, float (&x)[4]) {
  if (whole) {
    const Pack<T, 4> y = *reinterpret_cast<const Pack<T, 4>*>(at);
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = to_float(y.v[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = k < count ? to_float(at[k]) : 0.0f;
  }
}
template <typename T> __device__ __forceinline__ void store4(T* at, bool whole, int count, const float (&x)[4]) {
  if (whole) {
    Pack<T, 4> y;
#pragma unroll
    for (int k = 0; k < 4; ++k) y.v[k] = from_float<T>(x[k]);
    *reinterpret_cast<Pack<T, 4>*>(at) = y;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < count) at[k] = from_float<T>(x[k]);
  }
}

// the tensor that a thread block works on
template <int K> __device__ __forceinline__ const Tensor& find_tensor(const Table<K>& table) {
  int lo = 0, hi = table.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (table.t[mid].first <= blockIdx.x) lo = mid;
    else hi = mid - 1;
  }
  return table.t[lo];
}

template <typename P, typename G, bool Master> __device__ __forceinline__ bool all_wide(const Tensor& t, int state_align) {
  return (uintptr_t)t.p % (4 * sizeof(P)) == 0 && (uintptr_t)t.g % (4 * sizeof(G)) == 0 && (uintptr_t)t.m % state_align == 0 &&
         (uintptr_t)t.v % state_align == 0 && (!Master || (uintptr_t)t.master % 16 == 0);
}

template <typename P, typename G, bool Master, int K>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const __grid_constant__ Table<K> table) {
  const Hyper& h = table.h;
  const Tensor& t = find_tensor(table);
  const int64_t begin = (int64_t)(blockIdx.x - t.first) * kChunk;
  const bool wide = all_wide<P, G, Master>(t, 16);
  float* m_at = static_cast<float*>(t.m);
  float* v_at = static_cast<float*>(t.v);
  constexpr int kEach = kChunk / (kThreads * 4);
  float x[kEach][4], g[kEach][4], m[kEach][4], v[kEach][4];
#pragma unroll
  for (int r = 0; r < kEach; ++r) {
    const int64_t i = begin + (r * kThreads + threadIdx.x) * 4;
    const int count = (int)max((int64_t)0, min((int64_t)4, t.n - i));
    const bool whole = wide && count == 4;
    load4(static_cast<const G*>(t.g) + i, whole, count, g[r]);
    load4(m_at + i, whole, count, m[r]);
    load4(v_at + i, whole, count, v[r]);
    if constexpr (Master) load4(t.master + i, whole, count, x[r]);
    else load4(static_cast<const P*>(t.p) + i, whole, count, x[r]);
  }
#pragma unroll
  for (int r = 0; r < kEach; ++r) {
    const int64_t i = begin + (r * kThreads + threadIdx.x) * 4;
    const int count = (int)max((int64_t)0, min((int64_t)4, t.n - i));
    const bool whole = wide && count == 4;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      moments(h, g[r][k], m[r][k], v[r][k]);
      x[r][k] = stepped(h, x[r][k], m[r][k], sqrtf(v[r][k]));
    }
    store4(m_at + i, whole, count, m[r]);
    store4(v_at + i, whole, count, v[r]);
    if constexpr (Master) store4(t.master + i, whole, count, x[r]);
    store4(static_cast<P*>(t.p) + i, whole, count, x[r]);
  }
}

// ---- 8-bit states ----------------------------------------------------------------------------------------------------

using Fp8 = __nv_fp8_e4m3;

__device__ __forceinline__ void load_codes(const uint8_t* at, bool whole, int count, float (&x)[4]) {
  uint32_t bits = 0;
  if (whole) bits = *reinterpret_cast<const uint32_t*>(at);
  else
    for (int k = 0; k < count; ++k) bits |= (uint32_t)at[k] << (8 * k);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    Fp8 c;
    c.__x = (uint8_t)(bits >> (8 * k));
    x[k] = (float)c;
  }
}

__device__ __forceinline__ void store_codes(uint8_t* at, bool whole, int count, const float (&x)[4]) {
  uint32_t bits = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) bits |= (uint32_t)Fp8(x[k]).__x << (8 * k);  // exact: x is an e4m3 value or NaN
  if (whole) *reinterpret_cast<uint32_t*>(at) = bits;
  else
    for (int k = 0; k < count; ++k) at[k] = (uint8_t)(bits >> (8 * k));
}

__device__ __forceinline__ float finite_or_zero(float x) { return isfinite(x) ? x : 0.0f; }

// |x| * inv as one of its two neighbouring e4m3 values, unit in (0, 1) deciding which, with x's sign
template <bool Squared> __device__ __forceinline__ float code_of(float x, float inv, float unit) {
  if (!isfinite(x)) return __int_as_float(0x7fc00000);
  const float y = fminf(__fmul_rn(fabsf(x), inv), kTop);
  const int bits = __float_as_int(y);
  const float low = y < 0.015625f ? floorf(y * 512.0f) * 0.001953125f : __int_as_float(bits & ~0xfffff);
  const float step = fmaxf(__int_as_float(bits & 0x7f800000), 0.015625f) * 0.125f;
  float c;
  if (Squared) {
    const bool up = __fmul_rn(__fmul_rn(unit, __fadd_rn(2.0f * low, step)), step) < __fmul_rn(__fsub_rn(y, low), __fadd_rn(y, low));
    c = up ? low + step : low;
    if (y > 0.0f && c == 0.0f) c = 0.001953125f;
  } else {
    c = __fmul_rn(unit, step) < __fsub_rn(y, low) ? low + step : low;
  }
  return copysignf(c, x);
}

// largest of a warp's non-negative numbers
__device__ __forceinline__ float warp_top(float x) { return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(x))); }

// a warp takes one block of 256 values at a time, a lane the four at 4 * lane and the four 128 behind them
template <typename P, typename G, bool Master, int K>
__global__ void __launch_bounds__(kThreads) adamw_8bit_kernel(const __grid_constant__ Table<K> table) {
  const Hyper& h = table.h;
  const Tensor& t = find_tensor(table);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool wide = all_wide<P, G, Master>(t, 4);
  uint8_t* m_at = static_cast<uint8_t*>(t.m);
  uint8_t* v_at = static_cast<uint8_t*>(t.v);
  constexpr int kEach = kChunk / kBlock / (kThreads / 32);
  for (int r = 0; r < kEach; ++r) {
    const int64_t block = (int64_t)(blockIdx.x - t.first) * (kChunk / kBlock) + r * (kThreads / 32) + warp;
    if (block * kBlock >= t.n) return;
    const float m_scale = t.m_scale[block], v_scale = t.v_scale[block];
    float x[2][4], g[2][4], m[2][4], v[2][4];
    float m_top = 0.0f, v_top = 0.0f;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int64_t i = block * kBlock + s * 128 + lane * 4;
      const int count = (int)max((int64_t)0, min((int64_t)4, t.n - i));
      const bool whole = wide && count == 4;
      load4(static_cast<const G*>(t.g) + i, whole, count, g[s]);
      load_codes(m_at + i, whole, count, m[s]);
      load_codes(v_at + i, whole, count, v[s]);
      if constexpr (Master) load4(t.master + i, whole, count, x[s]);
      else load4(static_cast<const P*>(t.p) + i, whole, count, x[s]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float root = __fmul_rn(v[s][k], v_scale);
        m[s][k] = __fmul_rn(m[s][k], m_scale);
        v[s][k] = __fmul_rn(root, root);
        moments(h, g[s][k], m[s][k], v[s][k]);
        v[s][k] = __fsqrt_rn(v[s][k]);
        x[s][k] = stepped(h, x[s][k], m[s][k], v[s][k]);
        m_top = fmaxf(m_top, finite_or_zero(fabsf(m[s][k])));
        v_top = fmaxf(v_top, finite_or_zero(v[s][k]));
      }
    }
    m_top = warp_top(m_top);
    v_top = warp_top(v_top);
    if (m_top < 1e-30f) m_top = 0.0f;  // 448 / m_top has to be finite
    if (v_top < 1e-30f) v_top = 0.0f;
    const float m_inv = m_top > 0.0f ? __fmul_rn(__frcp_rn(m_top), kTop) : 0.0f, v_inv = v_top > 0.0f ? __fmul_rn(__frcp_rn(v_top), kTop) : 0.0f;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int64_t i = block * kBlock + s * 128 + lane * 4;
      const int count = (int)max((int64_t)0, min((int64_t)4, t.n - i));
      const bool whole = wide && count == 4;
      const uint32_t seed = t.seed + (uint32_t)(i >> 32) * 0xBB67AE85u;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t r32 = hash32((uint32_t)i + k, seed);
        m[s][k] = code_of<false>(m[s][k], m_inv, ((float)(r32 & 0xffffu) + 0.5f) * (1.0f / 65536.0f));
        v[s][k] = code_of<true>(v[s][k], v_inv, ((float)(r32 >> 16) + 0.5f) * (1.0f / 65536.0f));
      }
      store_codes(m_at + i, whole, count, m[s]);
      store_codes(v_at + i, whole, count, v[s]);
      if constexpr (Master) store4(t.master + i, whole, count, x[s]);
      store4(static_cast<P*>(t.p) + i, whole, count, x[s]);
    }
    if (lane == 0) {
      t.m_scale[block] = __fmul_rn(m_top, 1.0f / kTop);
      t.v_scale[block] = __fmul_rn(v_top, 1.0f / kTop);
    }
  }
}

template <int K> int launch_table(const Table<K>& table, uint32_t blocks, int p_type, int g_type, bool master, int bits, cudaStream_t st) {
  return gnr_with_type(p_type, [&](auto p) {
    return gnr_with_type(g_type, [&](auto g) {
      using P = decltype(p);
      using G = decltype(g);
      auto go = [&](auto has) {
        constexpr bool M = decltype(has)::value && sizeof(P) == 2;
        if (bits == 8) adamw_8bit_kernel<P, G, M, K><<<blocks, kThreads, 0, st>>>(table);
        else adamw_kernel<P, G, M, K><<<blocks, kThreads, 0, st>>>(table);
      };
      if (master) go(std::true_type());
      else go(std::false_type());
      GNR_CUDA_OK(cudaGetLastError());
      return 0;
    });
  });
}

template <int K>
int step_all(const GnrAdamwTensor* tensors, int n, const Hyper& h, int p_type, int g_type, bool master, int bits, uint32_t seed, cudaStream_t st) {
  Table<K> table;
  table.h = h;
  int k = 0;
  while (k < n) {
    uint64_t blocks = 0;
    table.n = 0;
    for (; k < n && table.n < K; ++k) {
      const GnrAdamwTensor& t = tensors[k];
      if (t.n == 0) continue;
      const uint64_t need = (uint64_t)(t.n + kChunk - 1) / kChunk;
      if (blocks + need > 0x7fffffff) break;
      table.t[table.n++] = {t.param, t.grad, t.exp_avg, t.exp_avg_sq, t.exp_avg_scale, t.exp_avg_sq_scale, t.master, t.n, (uint32_t)blocks,
                            hash32((uint32_t)t.number, seed)};
      blocks += need;
    }
    if (table.n > 0)
      if (int rc = launch_table(table, (uint32_t)blocks, p_type, g_type, master, bits, st)) return rc;
  }
  return 0;
}

}  // namespace

extern "C" int gnr_adamw_step(const GnrAdamwTensor* tensors_h, int n_tensors, int param_type, int grad_type, int state_bits, int64_t step,
                              double lr, double beta1, double beta2, double eps, double weight_decay, uint32_t seed, void* stream) {
  if (n_tensors < 0 || (n_tensors > 0 && !tensors_h) || gnr_type_size(param_type) == 0 || gnr_type_size(grad_type) == 0 ||
      (state_bits != 8 && state_bits != 32)) {
    gnr_set_error("gnr_adamw_step: null pointer, unknown element type, or states of %d bits (8 or 32)", state_bits);
    return -1;
  }
  if (step < 1 || !(lr >= 0.0) || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 1e-30) || !(weight_decay >= 0.0) ||
      !isfinite(lr) || !isfinite(eps) || !isfinite(weight_decay)) {
    gnr_set_error("gnr_adamw_step: step %lld (from 1), lr %g, betas %g %g ([0, 1)), eps %g (at least 1e-30), weight decay %g",
                  (long long)step, lr, beta1, beta2, eps, weight_decay);
    return -1;
  }
  const bool master = n_tensors > 0 && tensors_h[0].master != nullptr;
  if (master && param_type == GNR_FP32) {
    gnr_set_error("gnr_adamw_step: fp32 parameters have no 32-bit copy");
    return -1;
  }
  for (int k = 0; k < n_tensors; ++k) {
    const GnrAdamwTensor& t = tensors_h[k];
    if (t.n < 0 || t.n > ((int64_t)0x7fffffff * kChunk) ||
        (t.n > 0 && (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq || (state_bits == 8 && (!t.exp_avg_scale || !t.exp_avg_sq_scale)))) ||
        (t.master != nullptr) != master) {
      gnr_set_error("gnr_adamw_step: tensor %d of %lld values: null pointer, or some tensors have a 32-bit copy and others none", k, (long long)t.n);
      return -1;
    }
  }
  Hyper h;
  h.b1 = (float)beta1;
  h.b1c = (float)(1.0 - beta1);
  h.b2 = (float)beta2;
  h.b2c = (float)(1.0 - beta2);
  h.keep = (float)(1.0 - lr * weight_decay);
  h.rate = (float)(lr / (1.0 - pow(beta1, (double)step)));
  h.c2 = (float)sqrt(1.0 - pow(beta2, (double)step));
  h.eps = (float)eps;
  const uint32_t of_step = hash32((uint32_t)step, seed + (uint32_t)((uint64_t)step >> 32) * 0xBB67AE85u);
  const cudaStream_t st = (cudaStream_t)stream;
  return n_tensors <= kSmall ? step_all<kSmall>(tensors_h, n_tensors, h, param_type, grad_type, master, state_bits, of_step, st)
                             : step_all<kLarge>(tensors_h, n_tensors, h, param_type, grad_type, master, state_bits, of_step, st);
}
