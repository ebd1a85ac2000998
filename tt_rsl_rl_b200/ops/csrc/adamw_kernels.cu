// AdamW over many tensors (see adamw_kernels.cuh). The tensors' pointers travel as kernel arguments, so nothing is
// uploaded or kept between calls and a captured step stays valid as long as its tensors do.
//
// Every operation is rounded on its own (no fused multiply-add), as the same expression written with tensor operations
// rounds it, and the norm is summed together with its rounding errors: the step does not depend on how tensors are split.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <vector>

#include "adamw_kernels.cuh"
#include "philox.cuh"
#include "sm100_primitives.cuh"

namespace rlb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// Kernel arguments hold at most 32,764 bytes: 400 tensors a launch; short lists travel in a small table. The prepare
// kernel's threads read `id` and nothing else: 64-byte entries read by 150 threads cost 20 us of constant-cache misses.
struct Entry {
  void *p, *g, *m, *v;
  float *m_scale, *v_scale;
  int16_t* low;
  int64_t n;
};

template <int K>
struct AdamTable {
  int count;
  uint32_t units;
  uint32_t run;               // consecutive units of a warp
  uint32_t first_unit[K + 1];  // units before each tensor; the last entry: all of them
  uint32_t vec[(K + 31) / 32];  // bit i: every pointer of tensor i allows 4-element accesses
  uint16_t id[K];
  Entry t[K];
  __device__ __forceinline__ bool wide(int i) const { return vec[i >> 5] >> (i & 31) & 1u; }
};

// Per tensor, from its step count: 1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t), the step itself.
struct AdamFactors {
  float decay, step_size, unbias;
  uint32_t step;
};

struct AdamConsts {
  double max_norm;
  // -0: the assembler fuses mul.rn.f32x2 and add.rn.f32x2 into one rounding (unlike their single forms), but not a product
  // that is a fused multiply-add with an addend it does not know
  float none;
  float beta1, beta1c, beta2, beta2c, eps;
  int maximize;
  uint32_t first_stream;
  uint64_t seed;
};

// Calls fn(tensor, first unit in the tensor, units) for a warp's units: runs of `run` consecutive units are dealt out over
// all warps in turn, and a run is cut where a tensor ends. The tensor of a run's first unit is searched, the following
// ones are found by stepping on.
template <int K, typename Fn>
__device__ __forceinline__ void walk_units(const AdamTable<K>& t, Fn&& fn) {
  const uint32_t stride = gridDim.x * kWarps * t.run;
  for (uint32_t at = (blockIdx.x * kWarps + (threadIdx.x >> 5)) * t.run; at < t.units; at += stride) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (t.first_unit[mid] <= at) lo = mid;
      else hi = mid - 1;
    }
    const uint32_t end = min(at + t.run, t.units);
    for (uint32_t unit = at; unit < end; ++lo) {  // an empty tensor ends where it begins
      const uint32_t first = t.first_unit[lo], stop = min(end, t.first_unit[lo + 1]);
      if (stop > unit) fn(lo, unit - first, stop - unit);
      unit = max(unit, stop);
    }
  }
}

__device__ __forceinline__ double block_sum64(double x, double* smem) {  // result in every thread; fixed order
  for (int o = 16; o >= 1; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = x;
  __syncthreads();
  double y = 0.0;
  for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) y += smem[i];
  return y;
}

// Advances the steps of the table's tensors and writes their factors (one block).
template <int K>
__device__ void prepare_factors(const AdamTable<K>& t, const AdamHyper& h, float* steps, AdamFactors* f) {
  double lr = h.lr;
  if (h.lr_device) lr = h.lr_f64 ? *static_cast<const double*>(h.lr_device) : *static_cast<const float*>(h.lr_device);
  for (int i = threadIdx.x; i < t.count; i += blockDim.x) {
    const float s = steps[t.id[i]] + 1.f;
    steps[t.id[i]] = s;
    f[i].decay = static_cast<float>(1.0 - lr * h.weight_decay);
    f[i].step_size = static_cast<float>(lr / (1.0 - pow(h.beta1, static_cast<double>(s))));
    f[i].unbias = static_cast<float>(1.0 / sqrt(1.0 - pow(h.beta2, static_cast<double>(s))));
    f[i].step = static_cast<uint32_t>(s);
  }
}

template <int K>
__global__ void __launch_bounds__(kThreads) adamw_prepare_kernel(const __grid_constant__ AdamTable<K> t,
                                                                 const AdamHyper h, float* steps, AdamFactors* f) {
  griddep_wait();  // launched with programmatic stream serialization (launch_pdl)
  griddep_launch_dependents();
  prepare_factors(t, h, steps, f);
}

// Four consecutive elements.
__device__ __forceinline__ void load4(const float* p, float (&x)[4]) {
  const float4 v = *reinterpret_cast<const float4*>(p);
  x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}
__device__ __forceinline__ void load4(const __nv_bfloat16* p, float (&x)[4]) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  x[0] = __uint_as_float(v.x << 16), x[1] = __uint_as_float(v.x & 0xffff0000u);
  x[2] = __uint_as_float(v.y << 16), x[3] = __uint_as_float(v.y & 0xffff0000u);
}

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// Two sums of squares side by side, each with its rounding errors: s + e is right to about 2^-40 (hundreds of terms each), so
// the norm in fp32 does not depend on the order of the sum, at fp32 speed: summing in fp64 took 648 us for 335 M bf16
// gradients, this 139 for one tensor, 152 for 194 (4.4 TB/s). D. E. Knuth, "The Art of Computer Programming", volume 2: with t = s + x and
// b = t - s, the error of t is (s - (t - b)) + (x - b), whichever of s and x is the larger (a gradient may outgrow all before
// it).
struct SquareSum {
  Pair s = Pair(0.f, 0.f), e = Pair(0.f, 0.f);
  template <bool kExact>  // kExact: x * x fits fp32 where it is in range (bf16 gradients)
  __device__ __forceinline__ void add(const Pair& x, const Pair& none) {
    const Pair minus(-1.f, -1.f), q = fma2(x, x, none);  // a product of its own (AdamConsts::none)
    if (!kExact) e = add2(e, fma2(x, x, mul2(q, minus)));
    const Pair t = add2(s, q), b = fma2(s, minus, t);
    e = add2(e, add2(fma2(fma2(b, minus, t), minus, s), fma2(b, minus, q)));
    s = t;
  }
  // s overflows (or holds a NaN): the errors are not numbers then, the sum is
  __device__ __forceinline__ double value() const {
    float big[2], small[2];
    s.split(big[0], big[1]);
    e.split(small[0], small[1]);
    const double sum = static_cast<double>(big[0]) + static_cast<double>(big[1]);
    return isfinite(sum) ? sum + (static_cast<double>(small[0]) + static_cast<double>(small[1])) : sum;
  }
};

// Squares leave fp32's range above 1.8e19 (infinite) and lose digits below 4e-16. A block whose sum overflows, or is so small
// that what its squares lost (2^-149 each) could show, sums its share again in fp64, whose range holds every square.
constexpr double kLeastSum = 8.271806125530277e-25;  // 2^-80

// Sum of the squares of every gradient, one partial per block; the last block also prepares the factors.
template <typename T, int K>
__global__ void __launch_bounds__(kThreads) adamw_norm_kernel(const __grid_constant__ AdamTable<K> t,
                                                              const AdamHyper h, float* steps, AdamFactors* f,
                                                              double* partial, float minus_zero) {
  griddep_wait();  // launched with programmatic stream serialization (launch_pdl)
  griddep_launch_dependents();
  __shared__ double smem[kWarps];
  if (blockIdx.x == gridDim.x - 1) prepare_factors(t, h, steps, f);
  const int lane = threadIdx.x & 31;
  constexpr bool kExact = sizeof(T) == 2;
  constexpr int kBatch = kExact ? 4 : 2;  // units in flight: eight 8-byte or four 16-byte loads a lane
  SquareSum sum[2];
  const Pair none(minus_zero, minus_zero);
  walk_units(t, [&](int ti, uint32_t first, uint32_t units) {
    const Entry& a = t.t[ti];
    const int64_t base = static_cast<int64_t>(first) * kAdamBlock;
    const T* g = static_cast<const T*>(a.g) + base;
    const int64_t left = min(a.n - base, static_cast<int64_t>(units) * kAdamBlock);
    int64_t at = 0;
    if (t.wide(ti)) {
      for (; at + kBatch * kAdamBlock <= left; at += kBatch * kAdamBlock) {
        float x[2 * kBatch][4];
#pragma unroll
        for (int j = 0; j < 2 * kBatch; ++j) load4(g + at + j * 128 + lane * 4, x[j]);
#pragma unroll
        for (int i = 0; i < 4 * kBatch; ++i) {
          sum[i & 1].template add<kExact>(Pair(x[i >> 1][2 * i & 2], x[i >> 1][2 * i & 2 | 1]), none);
        }
      }
      for (; at + 128 <= left; at += 128) {
        float x[4];
        load4(g + at + lane * 4, x);
#pragma unroll
        for (int i = 0; i < 2; ++i) sum[i].template add<kExact>(Pair(x[2 * i], x[2 * i + 1]), none);
      }
    }
    for (at += lane; at < left; at += 32) sum[0].template add<kExact>(Pair(load1(g + at), 0.f), none);
  });
  double total = sum[0].value() + sum[1].value();
  total = block_sum64(total, smem);
  if (!(total >= kLeastSum && isfinite(total))) {  // the same in every thread; gradients of zeros come here too
    total = 0.0;
    walk_units(t, [&](int ti, uint32_t first, uint32_t units) {
      const Entry& a = t.t[ti];
      const int64_t base = static_cast<int64_t>(first) * kAdamBlock;
      const T* g = static_cast<const T*>(a.g) + base;
      const int64_t left = min(a.n - base, static_cast<int64_t>(units) * kAdamBlock);
      for (int64_t at = lane; at < left; at += 32) {
        const double x = load1(g + at);
        total = fma(x, x, total);
      }
    });
    total = block_sum64(total, smem);
  }
  if (threadIdx.x == 0) partial[blockIdx.x] = total;
}

// ---- 8-bit codes ----------------------------------------------------------------------------------------------------
// An e4m3 number without sign is the upper 12 bits of the fp32 number 2^-120 times as large (subnormal ones included), so
// codes and values differ by a shift and a product that is exact. Codes are handled where they leave those bits, in bits
// 20 to 26, and four of them packed at the end.
constexpr float kUp = 1.329227995784916e36f, kDown = 7.52316384526264e-37f;  // 2^120, 2^-120
constexpr uint32_t kCode = 1u << 20;
// The code below or above y (0 <= y <= 448, or half a unit more by the scale's rounding): above with probability
// (y - below) / (above - below), which is what the 20 bits under the code say. Rounding the scaled y up leaves a fraction
// that is not zero above every fraction below it.
__device__ __forceinline__ uint32_t linear_code(float y, uint32_t rnd16) {
  return __float_as_uint(__fmul_ru(y, kDown)) + (0xffff7u - 16u * rnd16);
}
// The same with probability (y^2 - below^2) / (above^2 - below^2), for two numbers.
__device__ __forceinline__ void square_codes(const Pair& y, uint32_t rnd0, uint32_t rnd1, uint32_t (&code)[2]) {
  float x[2], a[2], b[2];
  y.split(x[0], x[1]);
  const uint32_t c0 = __float_as_uint(__fmul_rz(x[0], kDown)) & 0xfff00000u;
  const uint32_t c1 = __float_as_uint(__fmul_rz(x[1], kDown)) & 0xfff00000u;
  const Pair up(kUp, kUp), minus(-1.f, -1.f);
  const Pair lo = mul2(Pair(__uint_as_float(c0), __uint_as_float(c1)), up);
  const Pair hi = mul2(Pair(__uint_as_float(c0 + kCode), __uint_as_float(c1 + kCode)), up);
  const Pair u = add2(Pair(__uint_as_float(0x3f800040u | rnd0 << 7), __uint_as_float(0x3f800040u | rnd1 << 7)), minus);
  mul2(mul2(fma2(lo, minus, hi), add2(hi, lo)), u).split(a[0], a[1]);
  mul2(fma2(lo, minus, y), add2(y, lo)).split(b[0], b[1]);
  code[0] = a[0] < b[0] ? c0 + kCode : c0;
  code[1] = a[1] < b[1] ? c1 + kCode : c1;
}
// Bytes 3 of four words.
__device__ __forceinline__ uint32_t pack_top(const uint32_t (&x)[4]) {
  return __byte_perm(__byte_perm(x[0], x[1], 0x0073), __byte_perm(x[2], x[3], 0x0073), 0x5410);
}
__device__ __forceinline__ void unpack_codes(uint32_t c, float (&x)[4]) {  // signed values, exact
  const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(c & 0xffffu), __NV_E4M3);
  const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(c >> 16), __NV_E4M3);
  const float2 a = __half22float2(__half2(lo)), b = __half22float2(__half2(hi));
  x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}

__device__ __forceinline__ float max_nan(float a, float b) {  // a NaN wins
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// ---- roots and quotients, two at a time -----------------------------------------------------------------------------------
// P. Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor" (1990): Newton steps from an
// approximation, then one step with the exact remainder, whose result is rounded from a value within about 2^-21 of a step of
// the true one: the rounded one, but for one in a million that lies so near the middle of two numbers, where it may be the
// neighbour (none of 67 million pairs; below about 1e-30 more often: the remainder is subnormal). For 0 <= v < 1e30 and |a| < 1e18, 1e-20 <= d < 1e30: a
// quotient stays below 1e38 (an infinite one would leave a NaN as its remainder); the functions of CUDA check for more and
// take one number.
__device__ __forceinline__ Pair neg2(const Pair& a) { return mul2(a, Pair(-1.f, -1.f)); }

__device__ __forceinline__ void sqrt2(const float (&v)[2], float (&r)[2]) {
  float y[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {  // from the smallest number up: zero stays zero below
    asm("rsqrt.approx.f32 %0, %1;" : "=f"(y[i]) : "f"(fmaxf(v[i], __int_as_float(1))));
  }
  const Pair x(v[0], v[1]), y2(y[0], y[1]), half(0.5f, 0.5f);
  Pair g = mul2(x, y2), h = mul2(y2, half);
  const Pair e = fma2(neg2(h), g, half);
  g = fma2(g, e, g), h = fma2(h, e, h);
  fma2(fma2(neg2(g), g, x), h, g).split(r[0], r[1]);
}
__device__ __forceinline__ Pair div2(const Pair& a, const Pair& d) {
  float x[2], y[2];
  d.split(x[0], x[1]);
#pragma unroll
  for (int i = 0; i < 2; ++i) asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y[i]) : "f"(x[i]));
  const Pair nd = neg2(d);
  Pair y2(y[0], y[1]);
  y2 = fma2(y2, fma2(nd, y2, Pair(1.f, 1.f)), y2);
  const Pair q = mul2(a, y2);
  return fma2(fma2(nd, q, a), y2, q);
}

// ---- the step ---------------------------------------------------------------------------------------------------------
// Four elements of every tensor of a step, as they lie in memory.
template <typename T, bool kBits8>
struct Quad {
  float p[4], g[4], m[4], v[4];  // fp32 tensors
  uint32_t pb[2], lb[2], gb[2];  // bf16 weights, their lower bits, gradients
  uint32_t mc, vc;               // codes

  static constexpr bool kSplit = sizeof(T) == 2;

  __device__ __forceinline__ void load(const Entry& a, int64_t at) {
    if (kSplit) {
      const uint2 x = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.p) + at);
      const uint2 y = *reinterpret_cast<const uint2*>(a.low + at);
      const uint2 z = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.g) + at);
      pb[0] = x.x, pb[1] = x.y, lb[0] = y.x, lb[1] = y.y, gb[0] = z.x, gb[1] = z.y;
    } else {
      load4(static_cast<const float*>(a.p) + at, p);
      load4(static_cast<const float*>(a.g) + at, g);
    }
    if (kBits8) {
      mc = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.m) + at);
      vc = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.v) + at);
    } else {
      load4(static_cast<const float*>(a.m) + at, m);
      load4(static_cast<const float*>(a.v) + at, v);
    }
  }
  __device__ __forceinline__ void store(const Entry& a, int64_t at) const {
    if (kSplit) {
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.p) + at) = make_uint2(pb[0], pb[1]);
      *reinterpret_cast<uint2*>(a.low + at) = make_uint2(lb[0], lb[1]);
    } else {
      *reinterpret_cast<float4*>(static_cast<float*>(a.p) + at) = make_float4(p[0], p[1], p[2], p[3]);
    }
    if (kBits8) {
      *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.m) + at) = mc;
      *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.v) + at) = vc;
    } else {
      *reinterpret_cast<float4*>(static_cast<float*>(a.m) + at) = make_float4(m[0], m[1], m[2], m[3]);
      *reinterpret_cast<float4*>(static_cast<float*>(a.v) + at) = make_float4(v[0], v[1], v[2], v[3]);
    }
  }
  // The same for the `in` first elements, one by one; the others count as zeros.
  __device__ __forceinline__ void load_some(const Entry& a, int64_t at, int in) {
    pb[0] = pb[1] = lb[0] = lb[1] = gb[0] = gb[1] = mc = vc = 0u;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      p[e] = g[e] = m[e] = v[e] = 0.f;
      if (e >= in) continue;
      if (kSplit) {
        pb[e >> 1] |= static_cast<uint32_t>(static_cast<const uint16_t*>(a.p)[at + e]) << (16 * (e & 1));
        lb[e >> 1] |= static_cast<uint32_t>(static_cast<uint16_t>(a.low[at + e])) << (16 * (e & 1));
        gb[e >> 1] |= static_cast<uint32_t>(static_cast<const uint16_t*>(a.g)[at + e]) << (16 * (e & 1));
      } else {
        p[e] = static_cast<const float*>(a.p)[at + e];
        g[e] = static_cast<const float*>(a.g)[at + e];
      }
      if (kBits8) {
        mc |= static_cast<uint32_t>(static_cast<const uint8_t*>(a.m)[at + e]) << (8 * e);
        vc |= static_cast<uint32_t>(static_cast<const uint8_t*>(a.v)[at + e]) << (8 * e);
      } else {
        m[e] = static_cast<const float*>(a.m)[at + e];
        v[e] = static_cast<const float*>(a.v)[at + e];
      }
    }
  }
  __device__ __forceinline__ void store_some(const Entry& a, int64_t at, int in) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (e >= in) continue;
      if (kSplit) {
        static_cast<uint16_t*>(a.p)[at + e] = static_cast<uint16_t>(pb[e >> 1] >> (16 * (e & 1)));
        a.low[at + e] = static_cast<int16_t>(lb[e >> 1] >> (16 * (e & 1)));
      } else {
        static_cast<float*>(a.p)[at + e] = p[e];
      }
      if (kBits8) {
        static_cast<uint8_t*>(a.m)[at + e] = static_cast<uint8_t>(mc >> (8 * e));
        static_cast<uint8_t*>(a.v)[at + e] = static_cast<uint8_t>(vc >> (8 * e));
      } else {
        static_cast<float*>(a.m)[at + e] = m[e];
        static_cast<float*>(a.v)[at + e] = v[e];
      }
    }
  }

  // Memory's form to fp32 and back. Rounding a weight to bf16 by adding half a unit (halves up) leaves a remainder of 16
  // signed bits, which are the fp32 weight's lower 16 bits as they are.
  __device__ __forceinline__ void decode(float m_scale, float v_scale) {
    if (kSplit) {
      uint32_t odd = 0u;  // a sign that the lower bits have changed: they belong to another weight
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t b = e & 1 ? pb[e >> 1] & 0xffff0000u : pb[e >> 1] << 16;
        const uint32_t joined = __byte_perm(lb[e >> 1], pb[e >> 1], e & 1 ? 0x7632 : 0x5410);
        const uint32_t w = joined - ((joined & 0x8000u) << 1);
        odd |= w ^ b;
        p[e] = __uint_as_float(w);
        g[e] = __uint_as_float(e & 1 ? gb[e >> 1] & 0xffff0000u : gb[e >> 1] << 16);
      }
      if (static_cast<int32_t>(odd) < 0) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t b = e & 1 ? pb[e >> 1] & 0xffff0000u : pb[e >> 1] << 16;
          if (static_cast<int32_t>(__float_as_uint(p[e]) ^ b) < 0) p[e] = __uint_as_float(b);
        }
      }
    }
    if (kBits8) {
      unpack_codes(mc, m);
      unpack_codes(vc, v);
      const Pair ms(m_scale, m_scale), vs(v_scale, v_scale);
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        mul2(Pair(m[e], m[e + 1]), ms).split(m[e], m[e + 1]);
        const Pair r = mul2(Pair(v[e], v[e + 1]), vs);
        mul2(r, r).split(v[e], v[e + 1]);
      }
    }
  }
  __device__ __forceinline__ void encode_weights() {
    if (!kSplit) return;
    uint32_t b[4];
    float finite = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      finite = fmaf(p[e], 0.f, finite);
      b[e] = __float_as_uint(p[e]);
    }
    if (isnan(finite)) {  // a NaN's bits do not survive the carry: one that does
#pragma unroll
      for (int e = 0; e < 4; ++e) b[e] = isnan(p[e]) ? 0x7fc00000u : b[e];
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      pb[i] = __byte_perm(b[2 * i] + 0x8000u, b[2 * i + 1] + 0x8000u, 0x7632);
      lb[i] = __byte_perm(b[2 * i], b[2 * i + 1], 0x5410);
    }
  }
  // `v` holds the roots.
  __device__ __forceinline__ void encode_states(float m_inv, float v_inv, const Philox& rnd) {
    uint32_t x[4], y[4];
    const Pair mi(m_inv, m_inv), vi(v_inv, v_inv);
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      float z[2];
      uint32_t d[2];
      mul2(Pair(fabsf(m[e]), fabsf(m[e + 1])), mi).split(z[0], z[1]);
      square_codes(mul2(Pair(v[e], v[e + 1]), vi), rnd.c[e] >> 16, rnd.c[e + 1] >> 16, d);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // the stored m is right on average
        x[e + i] = (linear_code(z[i], rnd.c[e + i] & 0xffffu) << 4 & 0x7f000000u) |
                   (__float_as_uint(m[e + i]) & 0x80000000u);
        // v, not its root, is right on average; never down to zero, which would leave m / eps as the next step
        y[e + i] = (v_inv > 0.f && v[e + i] > 0.f ? max(d[i], kCode) : d[i]) << 4 & 0x7f000000u;
      }
    }
    mc = pack_top(x);
    vc = pack_top(y);
  }
};

// A warp takes units of 256 elements: lane l elements [4 l, 4 l + 4) and [128 + 4 l, ...), so every access of the warp is
// contiguous. The unit is also the block of a scale, whose maximum is a warp reduction. With 32-bit states the step is
// bound by memory; with 8-bit states by its instructions, about 110 an element (random numbers, both roundings, root and
// quotient): 335 M bf16 weights in 1,497 us, 2.1 times the bytes' time, with 70 % of the issue slots used. Codes taken and
// packed by shifts and products instead of conversions, and pairs, brought it there from 2,832.
template <typename T, bool kBits8, int K>
__global__ void __launch_bounds__(kThreads, 3) adamw_step_kernel(const __grid_constant__ AdamTable<K> t,
                                                              const AdamConsts c, const AdamFactors* factors,
                                                              const double* partial, int partials, float* norm_out) {
  griddep_wait();  // launched with programmatic stream serialization (launch_pdl)
  griddep_launch_dependents();
  __shared__ double smem[kWarps];
  float clip = 1.f;
  if (partials > 0) {
    double s = 0.0;
    for (int i = threadIdx.x; i < partials; i += kThreads) s += partial[i];
    const double norm = sqrt(block_sum64(s, smem));
    const double f = c.max_norm / (norm + 1e-6);
    clip = static_cast<float>(f > 1.0 ? 1.0 : f);  // a NaN norm stays NaN
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = static_cast<float>(norm);
  }
  if (c.maximize) clip = -clip;
  const int lane = threadIdx.x & 31;
  const Pair none(c.none, c.none), clip2(clip, clip), b1(c.beta1, c.beta1), b1c(c.beta1c, c.beta1c), b2(c.beta2, c.beta2),
      b2c(c.beta2c, c.beta2c);
  walk_units(t, [&](int ti, uint32_t first, uint32_t units) {
    const Entry a = t.t[ti];
    const AdamFactors f = factors[ti];
    const bool wide = t.wide(ti);
    for (uint32_t u = first; u < first + units; ++u) {
      const int64_t at = static_cast<int64_t>(u) * kAdamBlock + lane * 4;
      const int left = static_cast<int>(min(a.n - static_cast<int64_t>(u) * kAdamBlock, static_cast<int64_t>(kAdamBlock)));
      const bool whole = wide && left == kAdamBlock;
      Quad<T, kBits8> q[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (whole) q[j].load(a, at + j * 128);
        else q[j].load_some(a, at + j * 128, left - j * 128 - lane * 4);
      }
      const float ms = kBits8 ? a.m_scale[u] : 0.f, vs = kBits8 ? a.v_scale[u] : 0.f;
      float top[2] = {0.f, 0.f};  // of the moments: |m|, and for 8-bit states the root of v
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        q[j].decode(ms, vs);
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          float *m = q[j].m + e, *v = q[j].v + e;
          const Pair g = mul2(Pair(q[j].g[e], q[j].g[e + 1]), clip2);
          add2(fma2(Pair(m[0], m[1]), b1, none), fma2(g, b1c, none)).split(m[0], m[1]);
          add2(fma2(Pair(v[0], v[1]), b2, none), fma2(mul2(g, g), b2c, none)).split(v[0], v[1]);
          top[0] = max_nan(max_nan(top[0], fabsf(m[0])), fabsf(m[1]));
          top[1] = max_nan(max_nan(top[1], v[0]), v[1]);
        }
      }
      // the quick forms are for numbers: all lanes take the slow ones where one has to, and with a tiny eps
      const bool quick = __all_sync(0xffffffffu, top[0] < 1e18f && top[1] < 1e30f) && c.eps >= 1e-20f;
      const Pair unbias(f.unbias, f.unbias), eps(c.eps, c.eps), keep(f.decay, f.decay), rate(-f.step_size, -f.step_size);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const float m[2] = {q[j].m[e], q[j].m[e + 1]}, v[2] = {q[j].v[e], q[j].v[e + 1]};
          float r[2];
          Pair x;
          if (quick) {
            sqrt2(v, r);
            x = div2(Pair(m[0], m[1]), add2(fma2(Pair(r[0], r[1]), unbias, none), eps));
          } else {
            for (int i = 0; i < 2; ++i) r[i] = __fsqrt_rn(v[i]);
            x = Pair(__fdiv_rn(m[0], __fadd_rn(__fmul_rn(r[0], f.unbias), c.eps)),
                     __fdiv_rn(m[1], __fadd_rn(__fmul_rn(r[1], f.unbias), c.eps)));
            if (kBits8) {  // as the codes take it; a NaN stays one in its block's scale
              for (int i = 0; i < 2; ++i) r[i] = fminf(r[i], 3e38f);
            }
          }
          add2(fma2(Pair(q[j].p[e], q[j].p[e + 1]), keep, none), fma2(rate, x, none)).split(q[j].p[e], q[j].p[e + 1]);
          if (kBits8) q[j].v[e] = r[0], q[j].v[e + 1] = r[1];
        }
      }
      if (kBits8) {
        float m_top = top[0], r_top = __fsqrt_rn(top[1]);  // the root grows with its argument
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) {
          m_top = max_nan(m_top, __shfl_xor_sync(0xffffffffu, m_top, o));
          r_top = max_nan(r_top, __shfl_xor_sync(0xffffffffu, r_top, o));
        }
        // blocks below 1e-30 are held as zero, so the scale's inverse stays finite
        const bool m_on = !(m_top < 1e-30f), r_on = !(r_top < 1e-30f);
        const float mi = m_on ? __fmul_rn(__frcp_rn(m_top), 448.f) : 0.f;
        // a root beyond fp32 leaves an infinite scale: no code is zero or a NaN then, so that all of the block stay infinite
        const float ri = r_on ? fmaxf(__fmul_rn(__frcp_rn(r_top), 448.f), 1e-38f) : 0.f;
        if (lane == 0) {
          a.m_scale[u] = m_on ? __fmul_rn(m_top, 1.f / 448.f) : 0.f;
          a.v_scale[u] = r_on ? __fmul_rn(r_top, 1.f / 448.f) : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint64_t i4 = static_cast<uint64_t>(at + j * 128) >> 2;
          q[j].encode_states(mi, ri, philox10(static_cast<uint32_t>(i4), static_cast<uint32_t>(i4 >> 32),
                                              c.first_stream + t.id[ti], f.step, static_cast<uint32_t>(c.seed),
                                              static_cast<uint32_t>(c.seed >> 32)));
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        q[j].encode_weights();
        if (whole) q[j].store(a, at + j * 128);
        else q[j].store_some(a, at + j * 128, left - j * 128 - lane * 4);
      }
    }
  });
}

constexpr int kSmallTable = 40, kLargeTable = 400;
constexpr int kNormBlocks = 1184;
static_assert(sizeof(AdamTable<kLargeTable>) + 256 <= 32764, "kernel arguments");

int sm_count() {
  int dev = 0, n = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n;
}

template <int K>
void fill_table(AdamTable<K>& t, const AdamLaunch& a, int first) {
  t.count = std::min(K, a.count - first);
  t.units = 0;
  for (uint32_t& x : t.vec) x = 0;
  for (int i = 0; i < t.count; ++i) {
    const AdamTensor& x = a.tensors[first + i];
    t.t[i] = Entry{x.p, x.g, x.m, x.v, x.m_scale, x.v_scale, x.low, x.n};
    t.id[i] = static_cast<uint16_t>(x.id);
    t.first_unit[i] = t.units;
    t.units += static_cast<uint32_t>((x.n + kAdamBlock - 1) / kAdamBlock);
    const uintptr_t wide = a.bf16 ? 7u : 15u, state = a.bits8 ? 3u : 15u;
    const uintptr_t bad = ((reinterpret_cast<uintptr_t>(x.p) | reinterpret_cast<uintptr_t>(x.g) |
                            reinterpret_cast<uintptr_t>(x.low)) & wide) |
                          ((reinterpret_cast<uintptr_t>(x.m) | reinterpret_cast<uintptr_t>(x.v)) & state);
    if (bad == 0) t.vec[i >> 5] |= 1u << (i & 31);
  }
  t.first_unit[t.count] = t.units;
  // up to 8 units a run, while every warp of a full grid still has one
  t.run = std::min<uint32_t>(8, std::max<uint32_t>(1, t.units / (148 * 6 * kWarps)));
}

// Blocks whose warps all have a run.
unsigned blocks_of(uint32_t units, uint32_t run, unsigned most) {
  const uint32_t runs = (units + run - 1) / run;
  return std::min<unsigned>(most, std::max<unsigned>(1, (runs + kWarps - 1) / kWarps));
}

// What one step over several lists shares: the partial sums of the norm come from every list before the first is stepped.
struct Shared {
  AdamFactors* factors;
  double* partial;
  int partials;
  double max_norm;
  float* norm;
};

template <typename T, int K>
cudaError_t prepare(const AdamLaunch& a, AdamFactors* factors, Shared& sh, cudaStream_t stream) {
  AdamTable<K> t;
  for (int first = 0; first < a.count; first += K) {
    fill_table(t, a, first);
    cudaError_t e;
    if (sh.max_norm > 0.0) {
      const unsigned grid = blocks_of(t.units, t.run, kNormBlocks);
      e = launch_pdl(adamw_norm_kernel<T, K>, dim3(grid), dim3(kThreads), 0, stream, t, a.h, a.steps, factors + first,
                     sh.partial + sh.partials, -0.f);
      sh.partials += static_cast<int>(grid);
    } else {
      e = launch_pdl(adamw_prepare_kernel<K>, dim3(1), dim3(kThreads), 0, stream, t, a.h, a.steps, factors + first);
    }
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

template <typename T, bool kBits8, int K>
cudaError_t step(const AdamLaunch& a, const AdamFactors* factors, Shared& sh, cudaStream_t stream) {
  AdamConsts c{};
  c.beta1 = static_cast<float>(a.h.beta1), c.beta1c = static_cast<float>(1.0 - a.h.beta1);
  c.beta2 = static_cast<float>(a.h.beta2), c.beta2c = static_cast<float>(1.0 - a.h.beta2);
  c.none = -0.f, c.eps = static_cast<float>(a.h.eps), c.max_norm = sh.max_norm;
  c.maximize = a.h.maximize, c.seed = a.h.seed, c.first_stream = a.first_stream;
  AdamTable<K> t;
  for (int first = 0; first < a.count; first += K) {
    fill_table(t, a, first);
    const unsigned grid = blocks_of(t.units, t.run, static_cast<unsigned>(sm_count()) * 6);  // one at least: the norm
    const cudaError_t e = launch_pdl(adamw_step_kernel<T, kBits8, K>, dim3(grid), dim3(kThreads), 0, stream, t, c,
                                     factors + first, static_cast<const double*>(sh.partial), sh.partials, sh.norm);
    sh.norm = nullptr;  // written once
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

template <typename T>
cudaError_t step_typed(const AdamLaunch& a, const AdamFactors* f, Shared& sh, cudaStream_t stream) {
  if (a.count <= kSmallTable) {
    return a.bits8 ? step<T, true, kSmallTable>(a, f, sh, stream) : step<T, false, kSmallTable>(a, f, sh, stream);
  }
  return a.bits8 ? step<T, true, kLargeTable>(a, f, sh, stream) : step<T, false, kLargeTable>(a, f, sh, stream);
}

template <typename T>
cudaError_t prepare_typed(const AdamLaunch& a, AdamFactors* f, Shared& sh, cudaStream_t stream) {
  return a.count <= kSmallTable ? prepare<T, kSmallTable>(a, f, sh, stream) : prepare<T, kLargeTable>(a, f, sh, stream);
}

int64_t factor_count(const AdamLaunch* lists, int n) {
  int64_t count = 0;
  for (int i = 0; i < n; ++i) count += lists[i].count;
  return (count + 1) / 2 * 2;
}

}  // namespace

int64_t adamw_workspace_bytes(const AdamLaunch* lists, int n) {
  int64_t tables = 0;
  for (int i = 0; i < n; ++i) tables += (lists[i].count + kLargeTable - 1) / kLargeTable;
  return factor_count(lists, n) * static_cast<int64_t>(sizeof(AdamFactors)) +
         tables * kNormBlocks * static_cast<int64_t>(sizeof(double));
}

cudaError_t adamw_step(const AdamLaunch* lists, int n, double max_norm, void* workspace, float* norm,
                       cudaStream_t stream) {
  Shared sh{static_cast<AdamFactors*>(workspace), nullptr, 0, max_norm, norm};
  sh.partial = reinterpret_cast<double*>(sh.factors + factor_count(lists, n));
  AdamFactors* f = sh.factors;
  for (int i = 0; i < n; ++i) {
    const cudaError_t e = lists[i].bf16 ? prepare_typed<__nv_bfloat16>(lists[i], f, sh, stream)
                                        : prepare_typed<float>(lists[i], f, sh, stream);
    if (e != cudaSuccess) return e;
    f += lists[i].count;
  }
  f = sh.factors;
  for (int i = 0; i < n; ++i) {
    const cudaError_t e = lists[i].bf16 ? step_typed<__nv_bfloat16>(lists[i], f, sh, stream)
                                        : step_typed<float>(lists[i], f, sh, stream);
    if (e != cudaSuccess) return e;
    f += lists[i].count;
  }
  return cudaSuccess;
}

}  // namespace rlb
