// AdamW over many tensors (see adamw_kernels.cuh). The tensors' pointers travel as kernel arguments, so nothing is
// uploaded or kept between calls and a captured step stays valid as long as its tensors do.
//
// Every operation is rounded on its own (no fused multiply-add), as the same expression written with tensor operations
// rounds it, and the norm is summed in 64 bits in a fixed order: the step does not depend on how tensors are split.
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

// Kernel arguments hold at most 32,764 bytes: 400 tensors a launch; short lists travel in a small table.
template <int K>
struct AdamTable {
  int count;
  uint32_t units;
  AdamTensor t[K];
};

// Per tensor, from its step count: 1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t), the step itself.
struct AdamFactors {
  float decay, step_size, unbias;
  uint32_t step;
};

struct AdamConsts {
  double max_norm;
  float beta1, beta1c, beta2, beta2c, eps;
  int maximize;
  uint64_t seed;
};

template <int K>
__device__ __forceinline__ int find_tensor(const AdamTable<K>& t, uint32_t unit) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.t[mid].first_unit <= unit) lo = mid;
    else hi = mid - 1;
  }
  return lo;
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
    const float s = steps[t.t[i].id] + 1.f;
    steps[t.t[i].id] = s;
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

// Sum of the squares of every gradient, one partial per block; the last block also prepares the factors.
template <typename T, int K>
__global__ void __launch_bounds__(kThreads) adamw_norm_kernel(const __grid_constant__ AdamTable<K> t,
                                                              const AdamHyper h, float* steps, AdamFactors* f,
                                                              double* partial) {
  griddep_wait();  // launched with programmatic stream serialization (launch_pdl)
  griddep_launch_dependents();
  __shared__ double smem[kWarps];
  if (blockIdx.x == gridDim.x - 1) prepare_factors(t, h, steps, f);
  const int lane = threadIdx.x & 31;
  double sum = 0.0;
  for (uint32_t unit = blockIdx.x * kWarps + (threadIdx.x >> 5); unit < t.units; unit += gridDim.x * kWarps) {
    const AdamTensor& a = t.t[find_tensor(t, unit)];
    const int64_t base = static_cast<int64_t>(unit - a.first_unit) * kAdamBlock;
    const T* g = static_cast<const T*>(a.g) + base;
    const int64_t left = a.n - base;
    if (a.vec && left >= kAdamBlock) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float x[4];
        load4(g + j * 128 + lane * 4, x);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += static_cast<double>(x[e]) * static_cast<double>(x[e]);
      }
    } else {
      for (int64_t i = lane; i < left && i < kAdamBlock; i += 32) {
        const double x = static_cast<double>(load1(g + i));
        sum += x * x;
      }
    }
  }
  sum = block_sum64(sum, smem);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// ---- 8-bit codes ----------------------------------------------------------------------------------------------------
// Value of an e4m3 code without sign (exact).
__device__ __forceinline__ float e4m3_value(uint32_t code) {
  return code >= 8u ? __uint_as_float((code << 20) + (120u << 23)) : static_cast<float>(code) * 0.001953125f;
}
// Code of the largest e4m3 value at most y, 0 <= y <= 448.
__device__ __forceinline__ uint32_t e4m3_below(float y) {
  return y >= 0.015625f ? (__float_as_uint(y) - (120u << 23)) >> 20 : static_cast<uint32_t>(y * 512.f);
}

// The fp32 weight of a bf16 one and its lower bits. Lower bits that do not belong to the weight (it was written from
// outside) move it by at most half of its last place, but across zero or past infinity they would make a NaN of it.
__device__ __forceinline__ float join(float p, int32_t low) {
  const uint32_t b = __float_as_uint(p), w = b + static_cast<uint32_t>(low);
  const bool keep = static_cast<int32_t>(w ^ b) >= 0 && !(low > 0 && (b & 0x7fffffffu) == 0x7f800000u);
  return __uint_as_float(keep ? w : b);
}

__device__ __forceinline__ float abs_max_bits(float a, float b) {  // NaN wins: its bits exceed every number's
  return __uint_as_float(max(__float_as_uint(a) & 0x7fffffffu, __float_as_uint(b) & 0x7fffffffu));
}

__device__ __forceinline__ uint32_t load_codes(const void* p) { return *static_cast<const uint32_t*>(p); }

// ---- the step ---------------------------------------------------------------------------------------------------------
// A warp takes a unit of 256 elements: lane l elements [4 l, 4 l + 4) and [128 + 4 l, ...), so every access of the warp
// is contiguous. The unit is also the block of a scale, whose maximum is a warp reduction.
template <typename T, bool kBits8, int K>
__global__ void __launch_bounds__(kThreads) adamw_step_kernel(const __grid_constant__ AdamTable<K> t,
                                                              const AdamConsts c, const AdamFactors* factors,
                                                              const double* partial, int partials, float* norm_out) {
  griddep_wait();  // launched with programmatic stream serialization (launch_pdl)
  griddep_launch_dependents();
  constexpr bool kSplit = sizeof(T) == 2;  // bf16 weights with their lower bits
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
  for (uint32_t unit = blockIdx.x * kWarps + (threadIdx.x >> 5); unit < t.units; unit += gridDim.x * kWarps) {
    const int ti = find_tensor(t, unit);
    const AdamTensor& a = t.t[ti];
    const int64_t base = static_cast<int64_t>(unit - a.first_unit) * kAdamBlock;
    const int left = static_cast<int>(min(a.n - base, static_cast<int64_t>(kAdamBlock)));
    const bool vec = a.vec && left == kAdamBlock;
    T* P = static_cast<T*>(a.p) + base;
    const T* G = static_cast<const T*>(a.g) + base;
    float p[8], g[8], m[8], v[8];
    uint32_t mc[2], vc[2];
    const int64_t blk = base / kAdamBlock;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int o = j * 128 + lane * 4;
      float(&pj)[4] = *reinterpret_cast<float(*)[4]>(p + 4 * j);
      float(&gj)[4] = *reinterpret_cast<float(*)[4]>(g + 4 * j);
      float(&mj)[4] = *reinterpret_cast<float(*)[4]>(m + 4 * j);
      float(&vj)[4] = *reinterpret_cast<float(*)[4]>(v + 4 * j);
      if (vec) {
        load4(P + o, pj);
        load4(G + o, gj);
        if (kSplit) {
          const uint2 w = *reinterpret_cast<const uint2*>(a.low + base + o);
          pj[0] = join(pj[0], static_cast<int16_t>(w.x & 0xffffu));
          pj[1] = join(pj[1], (static_cast<int32_t>(w.x) >> 16));
          pj[2] = join(pj[2], static_cast<int16_t>(w.y & 0xffffu));
          pj[3] = join(pj[3], (static_cast<int32_t>(w.y) >> 16));
        }
        if (kBits8) {
          mc[j] = load_codes(static_cast<uint8_t*>(a.m) + base + o);
          vc[j] = load_codes(static_cast<uint8_t*>(a.v) + base + o);
        } else {
          load4(static_cast<float*>(a.m) + base + o, mj);
          load4(static_cast<float*>(a.v) + base + o, vj);
        }
      } else {
        mc[j] = vc[j] = 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool in = o + e < left;
          pj[e] = in ? load1(P + o + e) : 0.f;
          gj[e] = in ? load1(G + o + e) : 0.f;
          if (kSplit && in) pj[e] = join(pj[e], a.low[base + o + e]);
          if (kBits8) {
            if (in) {
              mc[j] |= static_cast<uint32_t>(static_cast<uint8_t*>(a.m)[base + o + e]) << (8 * e);
              vc[j] |= static_cast<uint32_t>(static_cast<uint8_t*>(a.v)[base + o + e]) << (8 * e);
            }
          } else {
            mj[e] = in ? static_cast<float*>(a.m)[base + o + e] : 0.f;
            vj[e] = in ? static_cast<float*>(a.v)[base + o + e] : 0.f;
          }
        }
      }
    }
    if (kBits8) {
      const float ms = a.m_scale[blk], vs = a.v_scale[blk];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t cm = mc[i >> 2] >> (8 * (i & 3)), cv = vc[i >> 2] >> (8 * (i & 3));
        const float mv = e4m3_value(cm & 0x7fu);
        m[i] = __fmul_rn(cm & 0x80u ? -mv : mv, ms);
        const float r = __fmul_rn(e4m3_value(cv & 0x7fu), vs);
        v[i] = __fmul_rn(r, r);
      }
    }
    const AdamFactors f = factors[ti];
    float m_top = 0.f, r_top = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float gi = __fmul_rn(g[i], clip);
      m[i] = __fadd_rn(__fmul_rn(m[i], c.beta1), __fmul_rn(gi, c.beta1c));
      v[i] = __fadd_rn(__fmul_rn(v[i], c.beta2), __fmul_rn(__fmul_rn(gi, gi), c.beta2c));
      const float r = __fsqrt_rn(v[i]);
      const float u = __fdiv_rn(m[i], __fadd_rn(__fmul_rn(r, f.unbias), c.eps));
      p[i] = __fsub_rn(__fmul_rn(p[i], f.decay), __fmul_rn(f.step_size, u));
      if (kBits8) {
        v[i] = r;
        m_top = abs_max_bits(m_top, m[i]);
        r_top = abs_max_bits(r_top, r);
      }
    }
    if (kBits8) {
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) {
        m_top = abs_max_bits(m_top, __shfl_xor_sync(0xffffffffu, m_top, o));
        r_top = abs_max_bits(r_top, __shfl_xor_sync(0xffffffffu, r_top, o));
      }
      // blocks below 1e-30 are held as zero, so the scale's inverse stays finite
      const bool m_on = !(m_top < 1e-30f), r_on = !(r_top < 1e-30f);
      const float mi = m_on ? __fmul_rn(__frcp_rn(m_top), 448.f) : 0.f;
      const float ri = r_on ? __fmul_rn(__frcp_rn(r_top), 448.f) : 0.f;
      if (lane == 0) {
        a.m_scale[blk] = m_on ? __fmul_rn(m_top, 1.f / 448.f) : 0.f;
        a.v_scale[blk] = r_on ? __fmul_rn(r_top, 1.f / 448.f) : 0.f;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint64_t idx4 = static_cast<uint64_t>(base + j * 128 + lane * 4) >> 2;
        const Philox rnd = philox10(static_cast<uint32_t>(idx4), static_cast<uint32_t>(idx4 >> 32), a.stream, f.step,
                                    static_cast<uint32_t>(c.seed), static_cast<uint32_t>(c.seed >> 32));
        mc[j] = vc[j] = 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = 4 * j + e;
          // m: up with probability (y - low) / (high - low), so the stored value is right on average
          float u = __fmul_rn(static_cast<float>(rnd.c[e] & 0xffffu) + 0.5f, 1.f / 65536.f);
          float y = fminf(__fmul_rn(fabsf(m[i]), mi), 448.f);
          uint32_t code = e4m3_below(y);
          float lo = e4m3_value(code), hi = e4m3_value(code + 1u);
          if (__fmul_rn(hi - lo, u) < y - lo) ++code;
          mc[j] |= (code | (m[i] < 0.f ? 0x80u : 0u)) << (8 * e);
          // sqrt(v): up with probability (y^2 - low^2) / (high^2 - low^2), so that v, not its root, is right on average;
          // never down to zero, which would leave m / eps as the next step
          u = __fmul_rn(static_cast<float>(rnd.c[e] >> 16) + 0.5f, 1.f / 65536.f);
          y = fminf(__fmul_rn(v[i], ri), 448.f);
          code = e4m3_below(y);
          lo = e4m3_value(code), hi = e4m3_value(code + 1u);
          if (__fmul_rn(__fmul_rn(hi - lo, hi + lo), u) < __fmul_rn(y - lo, y + lo)) ++code;
          if (r_on && v[i] > 0.f) code = max(code, 1u);
          vc[j] |= code << (8 * e);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int o = j * 128 + lane * 4;
      uint32_t hi[4];
      int32_t lo[4];
      if (kSplit) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // round to nearest, halves up: the remainder fits 16 signed bits
          const uint32_t b = __float_as_uint(p[4 * j + e]);
          const bool nan = (b & 0x7fffffffu) > 0x7f800000u;
          hi[e] = nan ? 0x7fc0u : (b + 0x8000u) >> 16;
          lo[e] = nan ? 0 : static_cast<int32_t>(b - (hi[e] << 16));
        }
      }
      if (vec) {
        if (kSplit) {
          *reinterpret_cast<uint2*>(P + o) = make_uint2(hi[0] | hi[1] << 16, hi[2] | hi[3] << 16);
          *reinterpret_cast<uint2*>(a.low + base + o) =
              make_uint2((lo[0] & 0xffffu) | static_cast<uint32_t>(lo[1]) << 16,
                         (lo[2] & 0xffffu) | static_cast<uint32_t>(lo[3]) << 16);
        } else {
          *reinterpret_cast<float4*>(P + o) = make_float4(p[4 * j], p[4 * j + 1], p[4 * j + 2], p[4 * j + 3]);
        }
        if (kBits8) {
          *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.m) + base + o) = mc[j];
          *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.v) + base + o) = vc[j];
        } else {
          *reinterpret_cast<float4*>(static_cast<float*>(a.m) + base + o) =
              make_float4(m[4 * j], m[4 * j + 1], m[4 * j + 2], m[4 * j + 3]);
          *reinterpret_cast<float4*>(static_cast<float*>(a.v) + base + o) =
              make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (o + e >= left) continue;
          if (kSplit) {
            reinterpret_cast<uint16_t*>(P)[o + e] = static_cast<uint16_t>(hi[e]);
            a.low[base + o + e] = static_cast<int16_t>(lo[e]);
          } else {
            reinterpret_cast<float*>(P)[o + e] = p[4 * j + e];
          }
          if (kBits8) {
            static_cast<uint8_t*>(a.m)[base + o + e] = static_cast<uint8_t>(mc[j] >> (8 * e));
            static_cast<uint8_t*>(a.v)[base + o + e] = static_cast<uint8_t>(vc[j] >> (8 * e));
          } else {
            static_cast<float*>(a.m)[base + o + e] = m[4 * j + e];
            static_cast<float*>(a.v)[base + o + e] = v[4 * j + e];
          }
        }
      }
    }
  }
}

constexpr int kSmallTable = 40, kLargeTable = 400;
constexpr int kNormBlocks = 592;
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
  for (int i = 0; i < t.count; ++i) {
    AdamTensor& x = t.t[i] = a.tensors[first + i];
    x.first_unit = t.units;
    t.units += static_cast<uint32_t>((x.n + kAdamBlock - 1) / kAdamBlock);
    const uintptr_t wide = a.bf16 ? 7u : 15u, state = a.bits8 ? 3u : 15u;
    const uintptr_t bad = ((reinterpret_cast<uintptr_t>(x.p) | reinterpret_cast<uintptr_t>(x.g) |
                            reinterpret_cast<uintptr_t>(x.low)) & wide) |
                          ((reinterpret_cast<uintptr_t>(x.m) | reinterpret_cast<uintptr_t>(x.v)) & state);
    x.vec = bad == 0;
  }
}

unsigned norm_blocks(uint32_t units) {
  return static_cast<unsigned>(std::min<uint32_t>(kNormBlocks, std::max<uint32_t>(1, (units + kWarps - 1) / kWarps)));
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
      const unsigned grid = norm_blocks(t.units);
      e = launch_pdl(adamw_norm_kernel<T, K>, dim3(grid), dim3(kThreads), 0, stream, t, a.h, a.steps, factors + first,
                     sh.partial + sh.partials);
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
  c.eps = static_cast<float>(a.h.eps), c.max_norm = sh.max_norm;
  c.maximize = a.h.maximize, c.seed = a.h.seed;
  AdamTable<K> t;
  for (int first = 0; first < a.count; first += K) {
    fill_table(t, a, first);
    const unsigned blocks = std::max<unsigned>(1, (t.units + kWarps - 1) / kWarps);  // an empty list writes the norm
    const unsigned grid = std::min<unsigned>(static_cast<unsigned>(sm_count()) * 6, blocks);
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
