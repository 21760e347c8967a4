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
// 16 for v).  A positive v is never rounded to 0, which would make its next step as large as |m| / eps: where its root is below the
// smallest code it becomes that code, which is the one place where the mean is not kept.
// The arithmetic of the codes is in separately rounded operations (no fused multiply-add), so that the codes of equal
// inputs are equal wherever they are computed with the same 448 / (largest in the block): here that quotient is the exact reciprocal's
// but for some blocks in a million (scale_up).
#include <cuda_fp8.h>
#include <math.h>
#include <string.h>

#include <algorithm>

#include "gnr_internal.cuh"
#include "gnr_types.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kBlock = GNR_ADAMW_BLOCK;
constexpr int kChunk = 4096;                       // values of a thread block
constexpr int kThreads8 = 256;                     // with 8-bit states
constexpr int kChunk8 = kThreads8 / 32 * kBlock;   // ... a block of codes for each warp
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
  uint32_t seed;
};

// A number twice, as the packed operations take it: from the kernel's arguments without a move.
struct alignas(8) Twice {
  float x, y;
};

struct Hyper {
  Twice b1, b1c, b2, b2c;  // betas and 1 - betas
  Twice keep;              // 1 - lr * weight decay
  Twice rate;              // -lr / (1 - b1^t)
  Twice c2_inv;            // 1 / sqrt(1 - b2^t)
  Twice eps;
  Twice minus_one, two, eighth;
};

// Rates and count of steps in device memory, for steps that are captured into a CUDA graph: every replay advances them.
struct Clock {
  Hyper h;
  uint32_t of_step;  // what the tensors' random bits begin with
  uint32_t seed;
  int64_t step;
  double lr, beta1, beta2, eps, decay;
  double power1, power2;  // betas to the power of step
};
static_assert(sizeof(Clock) <= GNR_ADAMW_CLOCK_BYTES, "clock");

template <int K> struct Table {
  Hyper h;
  int n;
  uint32_t first[K];  // thread blocks before each tensor's, apart from the rest so that the search stays in a few cache lines
  Tensor t[K];
};
constexpr int kSmall = 24, kLarge = 400;  // tensors of a launch: 2 and 31 KB of arguments
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

__host__ __device__ __forceinline__ Twice twice(double x) { return {(float)x, (float)x}; }

// The numbers of a step from its rates and the betas' powers.  Before the `first` step, where the powers are 1: no step, told by c2_inv = 0.
__host__ __device__ __forceinline__ Hyper hyper_of(double lr, double beta1, double beta2, double eps, double decay, double power1, double power2, bool first) {
  Hyper h;
  h.b1 = twice(beta1);
  h.b1c = twice(1.0 - beta1);
  h.b2 = twice(beta2);
  h.b2c = twice(1.0 - beta2);
  h.keep = twice(1.0 - lr * decay);
  h.rate = twice(first ? 0.0 : -lr / (1.0 - power1));
  h.c2_inv = twice(first ? 0.0 : 1.0 / sqrt(1.0 - power2));
  h.eps = twice(eps);
  h.minus_one = twice(-1.0);
  h.two = twice(2.0);
  h.eighth = twice(0.125);
  return h;
}

__host__ __device__ __forceinline__ uint32_t hash_of_step(int64_t step, uint32_t seed) {
  return hash32((uint32_t)step, seed + (uint32_t)((uint64_t)step >> 32) * 0xBB67AE85u);
}

// (a negative step: the clock's own count stays)
__global__ void adamw_set_clock_kernel(Clock* clock, Clock to) {
  if (to.step < 0) {
    to.step = clock->step;
    to.seed = clock->seed;
    to.of_step = clock->of_step;
    to.power1 = pow(to.beta1, (double)to.step);
    to.power2 = pow(to.beta2, (double)to.step);
    to.h = hyper_of(to.lr, to.beta1, to.beta2, to.eps, to.decay, to.power1, to.power2, to.step == 0);
  }
  *clock = to;
}

__global__ void adamw_advance_clock_kernel(Clock* clock) {
  Clock c = *clock;
  ++c.step;
  c.power1 *= c.beta1;
  c.power2 *= c.beta2;
  c.h = hyper_of(c.lr, c.beta1, c.beta2, c.eps, c.decay, c.power1, c.power2, false);
  c.of_step = hash_of_step(c.step, c.seed);
  *clock = c;
}

// A step's numbers: the kernel's arguments, or (Clocked) the clock's, brought to shared memory by all threads of the block.
template <bool Clocked, int K> __device__ __forceinline__ const Hyper& hyper_for(const Table<K>& table, const Clock* clock) {
  if constexpr (Clocked) {
    __shared__ Hyper s_h;
    constexpr int kWords = sizeof(Hyper) / 4;
    if (threadIdx.x < kWords) reinterpret_cast<uint32_t*>(&s_h)[threadIdx.x] = reinterpret_cast<const uint32_t*>(&clock->h)[threadIdx.x];
    __syncthreads();
    return s_h;
  } else {
    return table.h;
  }
}

// Two fp32 numbers in one operation of the packed fp32 instructions: each half rounded as the single operation rounds it.
struct Two {
  unsigned long long v;
};
__device__ __forceinline__ Two two(float x, float y) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ Two two(float x) { return two(x, x); }
__device__ __forceinline__ Two two(const Twice& x) {
  Two r;
  r.v = *reinterpret_cast<const unsigned long long*>(&x);
  return r;
}
__device__ __forceinline__ void split(Two a, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a.v)); }
__device__ __forceinline__ Two mul2(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two add2_up(Two a, Two b) {
  Two r;
  asm("add.rp.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two add2_zero(Two a, Two b) {
  Two r;
  asm("add.rz.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ Two sub2(const Hyper& h, Two a, Two b) { return fma2(b, two(h.minus_one), a); }

// m and v after the gradient g
__device__ __forceinline__ void moments(const Hyper& h, float g, float& m, float& v) {
  m = __fadd_rn(__fmul_rn(h.b1.x, m), __fmul_rn(h.b1c.x, g));
  v = __fadd_rn(__fmul_rn(h.b2.x, v), __fmul_rn(__fmul_rn(h.b2c.x, g), g));
}

// 1 / x of a normal number, within one unit of the last place
__device__ __forceinline__ float quick_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float stepped(const Hyper& h, float x, float m, float root) {
  return fmaf(h.rate.x, m * quick_rcp(fmaf(root, h.c2_inv.x, h.eps.x)), x * h.keep.x);
}

// Four values of a thread: the neighbours from i on, or (not Wide) those kThreads apart from i on that lie before `end`, 0 for the others.
template <bool Wide, typename T> __device__ __forceinline__ void load4(const T* at, int i, int end, float (&x)[4]) {
  if constexpr (Wide) {
    const Pack<T, 4> y = *reinterpret_cast<const Pack<T, 4>*>(at + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = to_float(y.v[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = i + k * kThreads < end ? to_float(at[i + k * kThreads]) : 0.0f;
  }
}
template <bool Wide, typename T> __device__ __forceinline__ void store4(T* at, int i, int end, const float (&x)[4]) {
  if constexpr (Wide) {
    Pack<T, 4> y;
#pragma unroll
    for (int k = 0; k < 4; ++k) y.v[k] = from_float<T>(x[k]);
    *reinterpret_cast<Pack<T, 4>*>(at + i) = y;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i + k * kThreads < end) at[i + k * kThreads] = from_float<T>(x[k]);
  }
}

// the tensor that a thread block works on
template <int K> __device__ __forceinline__ int find_tensor(const Table<K>& table) {
  int lo = 0, hi = table.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (table.first[mid] <= blockIdx.x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <typename P, typename G, bool Master> __device__ __forceinline__ bool all_wide(const Tensor& t, int state_align) {
  return (uintptr_t)t.p % (4 * sizeof(P)) == 0 && (uintptr_t)t.g % (4 * sizeof(G)) == 0 && (uintptr_t)t.m % state_align == 0 &&
         (uintptr_t)t.v % state_align == 0 && (!Master || (uintptr_t)t.master % 16 == 0);
}

// Bound by HBM: 16 values of every array in flight a thread; 335M fp32 values with gradients take 1355 us, 6.9 TB/s (with divisions for the two
// quotients 1517 us), 60M bf16 values with fp32 copies in 300 tensors 250 us, 6.7 TB/s.
template <typename P, typename G, bool Master, bool Clocked, int K>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const __grid_constant__ Table<K> table, const Clock* __restrict__ clock) {
  const Hyper& h = hyper_for<Clocked>(table, clock);
  if (Clocked && h.c2_inv.x == 0.0f) return;  // not advanced yet: no step
  const int number = find_tensor(table);
  const Tensor& t = table.t[number];
  const int64_t begin = (int64_t)(blockIdx.x - table.first[number]) * kChunk;
  constexpr int kEach = kChunk / (kThreads * 4);
  float x[kEach][4], g[kEach][4], m[kEach][4], v[kEach][4];
  const int left = (int)min((int64_t)kChunk, t.n - begin);
  const G* g_at = static_cast<const G*>(t.g) + begin;
  P* p_at = static_cast<P*>(t.p) + begin;
  float *m_at = static_cast<float*>(t.m) + begin, *v_at = static_cast<float*>(t.v) + begin, *master_at = Master ? t.master + begin : nullptr;
  // four neighbours to a thread and access, or single values, neighbours in neighbouring threads, where the alignment or the end forbids it
  auto all = [&](auto is_wide) {
    constexpr bool Wide = decltype(is_wide)::value;
#pragma unroll
    for (int r = 0; r < kEach; ++r) {
      const int i = Wide ? (r * kThreads + threadIdx.x) * 4 : r * kThreads * 4 + threadIdx.x;
      load4<Wide>(g_at, i, left, g[r]);
      load4<Wide>(m_at, i, left, m[r]);
      load4<Wide>(v_at, i, left, v[r]);
      if constexpr (Master) load4<Wide>(master_at, i, left, x[r]);
      else load4<Wide>(p_at, i, left, x[r]);
    }
#pragma unroll
    for (int r = 0; r < kEach; ++r) {
      const int i = Wide ? (r * kThreads + threadIdx.x) * 4 : r * kThreads * 4 + threadIdx.x;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        moments(h, g[r][k], m[r][k], v[r][k]);
        x[r][k] = stepped(h, x[r][k], m[r][k], sqrtf(v[r][k]));
      }
      store4<Wide>(m_at, i, left, m[r]);
      store4<Wide>(v_at, i, left, v[r]);
      if constexpr (Master) store4<Wide>(master_at, i, left, x[r]);
      store4<Wide>(p_at, i, left, x[r]);
    }
  };
  if (left == kChunk && all_wide<P, G, Master>(t, 16)) all(std::true_type());
  else all(std::false_type());
}

// ---- 8-bit states ----------------------------------------------------------------------------------------------------

constexpr uint32_t kNotFinite = 0x7f800000u;  // bits of |x| from here on: infinities and NaN
constexpr uint32_t kNanCode = 0x7f;

// four e4m3 codes as fp32, exactly
__device__ __forceinline__ void decode4(uint32_t codes, float (&x)[4]) {
#pragma unroll
  for (int k = 0; k < 4; k += 2) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes >> (8 * k)), __NV_E4M3);
    const float2 y = __half22float2(h);
    x[k] = y.x;
    x[k + 1] = y.y;
  }
}

template <typename T> __device__ __forceinline__ void store_some(T* at, bool whole, int count, const float (&x)[4]) {
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

// `count` (at most 4) neighbours as they lie in memory, zeros behind them
template <typename T> __device__ __forceinline__ Pack<T, 4> load_raw(const T* at, bool whole, int count) {
  if (whole) return *reinterpret_cast<const Pack<T, 4>*>(at);
  Pack<T, 4> y;
#pragma unroll
  for (int k = 0; k < 4; ++k) y.v[k] = k < count ? at[k] : from_float<T>(0.0f);
  return y;
}

__device__ __forceinline__ uint32_t load_codes(const uint8_t* at, bool whole, int count) {
  if (whole) return *reinterpret_cast<const uint32_t*>(at);
  uint32_t codes = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) if (k < count) codes |= (uint32_t)at[k] << (8 * k);
  return codes;
}

__device__ __forceinline__ void store_codes(uint8_t* at, bool whole, int count, uint32_t codes) {
  if (whole) *reinterpret_cast<uint32_t*>(at) = codes;
  else
#pragma unroll
    for (int k = 0; k < 4; ++k) if (k < count) at[k] = (uint8_t)(codes >> (8 * k));
}

// Codes by the bits of an fp32 number: its exponent and three mantissa bits, 960 = (127 - 7) << 3 lower, are the e4m3 code of a
// value from 2^-6 on.  Below, the codes are 2^-9 apart as in the binade above: 2^-6 is added (kShift) and 8 taken off.
constexpr float kShift = 0.015625f;

// the signs of four numbers as those of four codes
__device__ __forceinline__ uint32_t signs(const float (&m)[4]) {
  const uint32_t low = __byte_perm(__float_as_uint(m[0]), __float_as_uint(m[1]), 0x73), high = __byte_perm(__float_as_uint(m[2]), __float_as_uint(m[3]), 0x73);
  return __byte_perm(low, high, 0x5410) & 0x80808080u;
}

// |m| * inv rounded up where a uniform u = (r + 1/2) / 2^16 is below the part of it past the code below: adding 1 - u of a code, less
// one, to the bits carries into the code in just these cases (u has 17 bits, the part 20; rounded upwards where the shift cuts it).
__device__ __forceinline__ void codes_of_m(const float (&m)[2], Two inv, const uint32_t (&r32)[2], uint32_t (&code)[2]) {
  float y[2], shift[2], z[2];
  split(mul2(two(m[0], m[1]), inv), y[0], y[1]);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    y[k] = fminf(fabsf(y[k]), kTop);
    shift[k] = y[k] < kShift ? kShift : 0.0f;
  }
  split(add2_up(two(y[0], y[1]), two(shift[0], shift[1])), z[0], z[1]);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint32_t at = (__float_as_uint(z[k]) + ((~r32[k] & 0xffffu) << 4 | 7u)) >> 20;
    code[k] = at - (y[k] < kShift ? 968u : 960u);
  }
}

// root * inv rounded so that the mean of its square is kept: up where u < (y^2 - low^2) / ((low + step)^2 - low^2)
__device__ __forceinline__ void codes_of_root(const Hyper& h, const float (&root)[2], Two inv, const uint32_t (&r32)[2], uint32_t (&code)[2]) {
  float y[2], shift[2], z[2], a[2], b[2];
  split(mul2(two(root[0], root[1]), inv), y[0], y[1]);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    y[k] = fminf(y[k], kTop);
    shift[k] = y[k] < kShift ? kShift : 0.0f;
  }
  const Two yy = two(y[0], y[1]), shifts = two(shift[0], shift[1]);
  split(add2_zero(yy, shifts), z[0], z[1]);
  const uint32_t z0 = __float_as_uint(z[0]), z1 = __float_as_uint(z[1]);
  const Two low = sub2(h, two(__uint_as_float(z0 & ~0xfffffu), __uint_as_float(z1 & ~0xfffffu)), shifts);
  const Two step = mul2(two(__uint_as_float(z0 & 0x7f800000u), __uint_as_float(z1 & 0x7f800000u)), two(h.eighth));
  const Two u = add2(two(__uint_as_float(0x3f800040u | (r32[0] >> 16) << 7), __uint_as_float(0x3f800040u | (r32[1] >> 16) << 7)), two(h.minus_one));
  split(mul2(mul2(u, fma2(two(h.two), low, step)), step), a[0], a[1]);
  split(mul2(sub2(h, yy, low), add2(yy, low)), b[0], b[1]);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint32_t at = (__float_as_uint(z[k]) >> 20) - (y[k] < kShift ? 968u : 960u) + (a[k] < b[k] ? 1u : 0u);
    code[k] = max(at, min(__float_as_uint(root[k]), 1u));  // never 0 where the root is not
  }
}

// a lane's part of a block of 256 values as it lies in memory: the four values at 4 * lane and the four 128 behind them
template <typename X, typename G> struct Part {
  Pack<X, 4> x[2];
  Pack<G, 4> g[2];
  uint32_t m[2], v[2];
  float m_scale, v_scale;
};

// 448 / top, 0 for 0: the quick reciprocal and one Newton step (rounded like the exact one but for some in a million, where a value on the
// border of two codes may get the other one; the exact one in every case takes 335M values 976 instead of 969 us)
__device__ __forceinline__ float scale_up(float top) {
  if (top > 1e30f) return __fmul_rn(__frcp_rn(top), kTop);
  const float r = quick_rcp(top);
  return top > 0.0f ? __fmul_rn(__fmaf_rn(r, __fmaf_rn(-top, r, 1.0f), r), kTop) : 0.0f;
}

// A thread block's values of a tensor with 8-bit states; all places count from their beginning.
template <typename P, typename G, bool Master> struct Chunk8 {
  using X = std::conditional_t<Master, float, P>;
  P* p_at;
  const G* g_at;
  uint8_t *m_at, *v_at;
  float *ms_at, *vs_at, *master_at;
  int left;        // values there are
  uint32_t place;  // low half of the first one's place in the tensor
  uint32_t seed;

  // the part at `at` = 4 * lane past the beginning of a block
  template <bool Full> __device__ __forceinline__ Part<X, G> fetch(int at) const {
    Part<X, G> part;
    const X* x_at = Master ? reinterpret_cast<const X*>(master_at) : reinterpret_cast<const X*>(p_at);
    part.m_scale = ms_at[at / kBlock];
    part.v_scale = vs_at[at / kBlock];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int i = at + s * 128;
      const int count = Full ? 4 : min(4, max(0, left - i));
      part.g[s] = load_raw(g_at + i, Full, count);
      part.m[s] = load_codes(m_at + i, Full, count);
      part.v[s] = load_codes(v_at + i, Full, count);
      part.x[s] = load_raw(x_at + i, Full, count);
    }
    return part;
  }

  template <bool Full> __device__ __forceinline__ void step(const Hyper& h, const Part<X, G>& part, int at) const {
    float x[2][4], g[2][4], m[2][4], root[2][4];
    uint32_t m_bits = 0, v_bits = 0;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      decode4(part.m[s], m[s]);
      decode4(part.v[s], root[s]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        g[s][k] = to_float(part.g[s].v[k]);
        x[s][k] = to_float(part.x[s].v[k]);
      }
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int k = 0; k < 4; k += 2) {
        const Two gg = two(g[s][k], g[s][k + 1]), old = mul2(two(root[s][k], root[s][k + 1]), two(part.v_scale));
        // (the sums as single additions: a packed one behind packed products is compiled to a fused multiply-add)
        float old_m[2], new_m[2], old_v[2], new_v[2];
        split(mul2(two(h.b1), mul2(two(m[s][k], m[s][k + 1]), two(part.m_scale))), old_m[0], old_m[1]);
        split(mul2(two(h.b1c), gg), new_m[0], new_m[1]);
        split(mul2(two(h.b2), mul2(old, old)), old_v[0], old_v[1]);
        split(mul2(mul2(two(h.b2c), gg), gg), new_v[0], new_v[1]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          m[s][k + j] = __fadd_rn(old_m[j], new_m[j]);
          root[s][k + j] = __fsqrt_rn(__fadd_rn(old_v[j], new_v[j]));
        }
        float d0, d1;
        split(fma2(two(root[s][k], root[s][k + 1]), two(h.c2_inv), two(h.eps)), d0, d1);
        const Two q = mul2(two(m[s][k], m[s][k + 1]), two(quick_rcp(d0), quick_rcp(d1)));
        split(fma2(two(h.rate), q, mul2(two(x[s][k], x[s][k + 1]), two(h.keep))), x[s][k], x[s][k + 1]);
        m_bits = max(max(m_bits, __float_as_uint(m[s][k]) & 0x7fffffffu), __float_as_uint(m[s][k + 1]) & 0x7fffffffu);
        v_bits = max(max(v_bits, __float_as_uint(root[s][k])), __float_as_uint(root[s][k + 1]));
      }
      const int i = at + s * 128;
      const int count = Full ? 4 : min(4, max(0, left - i));
      if constexpr (Master) store_some(master_at + i, Full, count, x[s]);
      store_some(p_at + i, Full, count, x[s]);
    }
    m_bits = __reduce_max_sync(0xffffffffu, m_bits);  // non-negative numbers are ordered as their bits are
    v_bits = __reduce_max_sync(0xffffffffu, v_bits);
    const bool odd = max(m_bits, v_bits) >= kNotFinite;  // a value that is not finite: the others' scale leaves it out
    if (odd) {
      m_bits = v_bits = 0;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t a = __float_as_uint(m[s][k]) & 0x7fffffffu, b = __float_as_uint(root[s][k]) & 0x7fffffffu;
          m_bits = max(m_bits, a < kNotFinite ? a : 0u);
          v_bits = max(v_bits, b < kNotFinite ? b : 0u);
        }
      m_bits = __reduce_max_sync(0xffffffffu, m_bits);
      v_bits = __reduce_max_sync(0xffffffffu, v_bits);
    }
    float m_top = __uint_as_float(m_bits), v_top = __uint_as_float(v_bits);
    if (m_top < 1e-30f) m_top = 0.0f;  // 448 / m_top has to be finite
    if (v_top < 1e-30f) v_top = 0.0f;
    const float m_inv = scale_up(m_top), v_inv = scale_up(v_top);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int i = at + s * 128;
      const int count = Full ? 4 : min(4, max(0, left - i));
      uint32_t m_codes = 0, v_codes = 0;
#pragma unroll
      for (int k = 0; k < 4; k += 2) {
        const uint32_t r32[2] = {hash32(place + i + k, seed), hash32(place + i + k + 1, seed)};
        const float mk[2] = {m[s][k], m[s][k + 1]}, rk[2] = {root[s][k], root[s][k + 1]};
        uint32_t m_code[2], v_code[2];
        codes_of_m(mk, two(m_inv), r32, m_code);
        codes_of_root(h, rk, two(v_inv), r32, v_code);
        m_codes |= (m_code[0] | m_code[1] << 8) << (8 * k);
        v_codes |= (v_code[0] | v_code[1] << 8) << (8 * k);
      }
      m_codes |= signs(m[s]);
      if (odd) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if ((__float_as_uint(m[s][k]) & 0x7fffffffu) >= kNotFinite) m_codes = (m_codes & ~(0xffu << (8 * k))) | kNanCode << (8 * k);
          if ((__float_as_uint(root[s][k]) & 0x7fffffffu) >= kNotFinite) v_codes = (v_codes & ~(0xffu << (8 * k))) | kNanCode << (8 * k);
        }
      }
      store_codes(m_at + i, Full, count, m_codes);
      store_codes(v_at + i, Full, count, v_codes);
    }
    if ((threadIdx.x & 31) == 0) {
      ms_at[at / kBlock] = __fmul_rn(m_top, 1.0f / kTop);
      vs_at[at / kBlock] = __fmul_rn(v_top, 1.0f / kTop);
    }
  }
};

// A warp takes one block of 256 values.  Bound by its instructions, 89 a value with the packed fp32 ones counted for two (86 % of the issue
// slots), and by the power they draw: 335M fp32 values take 966 us at 1965 MHz, 5.6 TB/s, and 1040 to 1140 us in a long run, where the power
// cap holds the clock at 1.65 to 1.75 GHz.  Five thread blocks to an SM (48 registers, of which 24 to 36 bytes a thread spill) hide the
// loads better than a longer run of blocks with the next one's loads ahead of the work (1058 against 948 us on zeros), six spill more (1000).
// By a clock four (64 registers, 36 to 68 bytes spill): five would take those 335M values 1154 instead of 1206 us, but 9M unaligned bf16
// values with fp32 copies, the form of single accesses, 57 instead of 45.  A root by Newton's step from the quick reciprocal
// root, with a way out for its range, takes as long (954 us), in a pass of its own longer (1091).
template <typename P, typename G, bool Master, bool Clocked, int K>
__global__ void __launch_bounds__(kThreads8, Clocked ? 4 : 5) adamw_8bit_kernel(const __grid_constant__ Table<K> table, const Clock* __restrict__ clock) {
  const Hyper& h = hyper_for<Clocked>(table, clock);
  if (Clocked && h.c2_inv.x == 0.0f) return;  // not advanced yet: no step
  const int number = find_tensor(table);
  const Tensor& t = table.t[number];
  const int64_t first = (int64_t)(blockIdx.x - table.first[number]) * kChunk8;
  Chunk8<P, G, Master> c;
  c.p_at = static_cast<P*>(t.p) + first;
  c.g_at = static_cast<const G*>(t.g) + first;
  c.m_at = static_cast<uint8_t*>(t.m) + first;
  c.v_at = static_cast<uint8_t*>(t.v) + first;
  c.ms_at = t.m_scale + first / kBlock;
  c.vs_at = t.v_scale + first / kBlock;
  c.master_at = Master ? t.master + first : nullptr;
  c.left = (int)min((int64_t)kChunk8, t.n - first);
  c.place = (uint32_t)first;
  c.seed = (Clocked ? hash32(t.seed, clock->of_step) : t.seed) + (uint32_t)(first >> 32) * 0xBB67AE85u;
  const int lane = threadIdx.x & 31;
  const int at = (threadIdx.x >> 5) * kBlock;
  if (at >= c.left) return;
  if (all_wide<P, G, Master>(t, 4) && at + kBlock <= c.left) c.template step<true>(h, c.template fetch<true>(at + lane * 4), at + lane * 4);
  else c.template step<false>(h, c.template fetch<false>(at + lane * 4), at + lane * 4);
}

template <bool Clocked, int K>
int launch_table(const Table<K>& table, const Clock* clock, uint32_t blocks, int p_type, int g_type, bool master, int bits, cudaStream_t st) {
  return gnr_with_type(p_type, [&](auto p) {
    return gnr_with_type(g_type, [&](auto g) {
      using P = decltype(p);
      using G = decltype(g);
      auto go = [&](auto has) {
        constexpr bool M = decltype(has)::value && sizeof(P) == 2;
        if (bits == 8) adamw_8bit_kernel<P, G, M, Clocked, K><<<blocks, kThreads8, 0, st>>>(table, clock);
        else adamw_kernel<P, G, M, Clocked, K><<<blocks, kThreads, 0, st>>>(table, clock);
      };
      if (master) go(std::true_type());
      else go(std::false_type());
      GNR_CUDA_OK(cudaGetLastError());
      return 0;
    });
  });
}

// Whether the tensors have 32-bit copies: as the first one with values has (one without has no addresses).
bool has_master(const GnrAdamwTensor* tensors, int n) {
  for (int k = 0; k < n; ++k)
    if (tensors[k].n > 0) return tensors[k].master != nullptr;
  return false;
}

// (`clock`: null, or where the step's numbers are instead of in `h` and `seed`)
template <bool Clocked, int K>
int step_all(const GnrAdamwTensor* tensors, int n, const Hyper& h, const Clock* clock, int p_type, int g_type, int bits, uint32_t seed, cudaStream_t st) {
  const int chunk = bits == 8 ? kChunk8 : kChunk;
  Table<K> table;
  table.h = h;
  const bool master = has_master(tensors, n);
  int k = 0;
  while (k < n) {
    uint64_t blocks = 0;
    table.n = 0;
    for (; k < n && table.n < K; ++k) {
      const GnrAdamwTensor& t = tensors[k];
      if (t.n == 0) continue;
      const uint64_t need = (uint64_t)(t.n + chunk - 1) / chunk;
      if (blocks + need > 0x7fffffff) break;
      table.first[table.n] = (uint32_t)blocks;
      table.t[table.n++] = {t.param, t.grad, t.exp_avg, t.exp_avg_sq, t.exp_avg_scale, t.exp_avg_sq_scale, t.master, t.n,
                            Clocked ? (uint32_t)t.number : hash32((uint32_t)t.number, seed)};
      blocks += need;
    }
    if (table.n > 0)
      if (int rc = launch_table<Clocked>(table, clock, (uint32_t)blocks, p_type, g_type, master, bits, st)) return rc;
  }
  return 0;
}

int check_tensors(const char* what, const GnrAdamwTensor* tensors, int n, int param_type, int grad_type, int bits) {
  if (n < 0 || (n > 0 && !tensors) || gnr_type_size(param_type) == 0 || gnr_type_size(grad_type) == 0 || (bits != 8 && bits != 32)) {
    gnr_set_error("%s: null pointer, unknown element type, or states of %d bits (8 or 32)", what, bits);
    return -1;
  }
  const bool master = has_master(tensors, n);
  if (master && param_type == GNR_FP32) {
    gnr_set_error("%s: fp32 parameters have no 32-bit copy", what);
    return -1;
  }
  for (int k = 0; k < n; ++k) {
    const GnrAdamwTensor& t = tensors[k];
    if (t.n < 0 || t.n > (int64_t)0x7fffffff * (bits == 8 ? kChunk8 : kChunk) ||
        (t.n > 0 && (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq || (bits == 8 && (!t.exp_avg_scale || !t.exp_avg_sq_scale)))) ||
        (t.n > 0 && (t.master != nullptr) != master)) {
      gnr_set_error("%s: tensor %d of %lld values: null pointer, or some tensors have a 32-bit copy and others none", what, k, (long long)t.n);
      return -1;
    }
  }
  return 0;
}

int check_rates(const char* what, int64_t step, int64_t least, double lr, double beta1, double beta2, double eps, double weight_decay) {
  if (step < least || !(lr >= 0.0) || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 1e-30) || !(weight_decay >= 0.0) ||
      !isfinite(lr) || !isfinite(eps) || !isfinite(weight_decay)) {
    gnr_set_error("%s: step %lld (from %lld), lr %g, betas %g %g ([0, 1)), eps %g (at least 1e-30), weight decay %g", what, (long long)step, (long long)least,
                  lr, beta1, beta2, eps, weight_decay);
    return -1;
  }
  return 0;
}

int check_clock(const char* what, const void* clock) {
  if (clock && (uintptr_t)clock % 8 == 0) return 0;
  gnr_set_error("%s: the clock is %d bytes of device memory on an 8-byte boundary", what, GNR_ADAMW_CLOCK_BYTES);
  return -1;
}

}  // namespace

extern "C" int gnr_adamw_step(const GnrAdamwTensor* tensors_h, int n_tensors, int param_type, int grad_type, int state_bits, int64_t step,
                              double lr, double beta1, double beta2, double eps, double weight_decay, uint32_t seed, void* stream) {
  if (int rc = check_tensors("gnr_adamw_step", tensors_h, n_tensors, param_type, grad_type, state_bits)) return rc;
  if (int rc = check_rates("gnr_adamw_step", step, 1, lr, beta1, beta2, eps, weight_decay)) return rc;
  const Hyper h = hyper_of(lr, beta1, beta2, eps, weight_decay, pow(beta1, (double)step), pow(beta2, (double)step), false);
  const uint32_t of_step = hash_of_step(step, seed);
  const cudaStream_t st = (cudaStream_t)stream;
  return n_tensors <= kSmall ? step_all<false, kSmall>(tensors_h, n_tensors, h, nullptr, param_type, grad_type, state_bits, of_step, st)
                             : step_all<false, kLarge>(tensors_h, n_tensors, h, nullptr, param_type, grad_type, state_bits, of_step, st);
}

extern "C" int gnr_adamw_clock_set(void* clock, int64_t step, double lr, double beta1, double beta2, double eps, double weight_decay, uint32_t seed,
                                   void* stream) {
  if (int rc = check_clock("gnr_adamw_clock_set", clock)) return rc;
  if (int rc = check_rates("gnr_adamw_clock_set", step, -1, lr, beta1, beta2, eps, weight_decay)) return rc;
  Clock c{};
  c.power1 = pow(beta1, (double)std::max<int64_t>(step, 0));
  c.power2 = pow(beta2, (double)std::max<int64_t>(step, 0));
  c.h = hyper_of(lr, beta1, beta2, eps, weight_decay, c.power1, c.power2, step <= 0);
  c.of_step = hash_of_step(step, seed);
  c.seed = seed;
  c.step = step;
  c.lr = lr;
  c.beta1 = beta1;
  c.beta2 = beta2;
  c.eps = eps;
  c.decay = weight_decay;
  adamw_set_clock_kernel<<<1, 1, 0, (cudaStream_t)stream>>>((Clock*)clock, c);
  GNR_CUDA_OK(cudaGetLastError());
  return 0;
}

extern "C" int gnr_adamw_clock_advance(void* clock, void* stream) {
  if (int rc = check_clock("gnr_adamw_clock_advance", clock)) return rc;
  adamw_advance_clock_kernel<<<1, 1, 0, (cudaStream_t)stream>>>((Clock*)clock);
  GNR_CUDA_OK(cudaGetLastError());
  return 0;
}

extern "C" int gnr_adamw_step_clocked(const GnrAdamwTensor* tensors_h, int n_tensors, int param_type, int grad_type, int state_bits, const void* clock,
                                      void* stream) {
  if (int rc = check_tensors("gnr_adamw_step_clocked", tensors_h, n_tensors, param_type, grad_type, state_bits)) return rc;
  if (int rc = check_clock("gnr_adamw_step_clocked", clock)) return rc;
  return step_all<true, kLarge>(tensors_h, n_tensors, Hyper{}, (const Clock*)clock, param_type, grad_type, state_bits, 0, (cudaStream_t)stream);
}
