// Kernels of the token-policy operators (see token_kernels.cuh for the formulas).
//
// Determinism: every sum over a row, a sequence or a batch has a fixed order; no atomics.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "sm100_primitives.cuh"
#include "token_kernels.cuh"

namespace rlb {
namespace {

namespace cg = cooperative_groups;

constexpr double kLog2e = 1.4426950408889634;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kFar = -1e30f;  // stands for the exponent of a column of probability zero in products that must stay finite

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static constexpr int kPerVec = 4;
  static __device__ __forceinline__ float get(float x) { return x; }
  static __device__ __forceinline__ float put(float x) { return x; }
  static __device__ __forceinline__ void unpack(const uint4& v, float* x) {
    x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* x) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
};
template <>
struct Elem<__nv_bfloat16> {
  static constexpr int kPerVec = 8;
  static __device__ __forceinline__ float get(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 put(float x) { return __float2bfloat16_rn(x); }
  static __device__ __forceinline__ void unpack(const uint4& v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* x) {
    return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                      pack_bf16x2(x[6], x[7]));
  }
};
template <>
struct Elem<__half> {
  static constexpr int kPerVec = 8;
  static __device__ __forceinline__ float get(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half put(float x) { return __float2half_rn(x); }
  static __device__ __forceinline__ void unpack(const uint4& v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ uint32_t two(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint4 pack(const float* x) {
    return make_uint4(two(x[0], x[1]), two(x[2], x[3]), two(x[4], x[5]), two(x[6], x[7]));
  }
};

template <typename T>
__device__ __forceinline__ T* row_ptr(const TokenRows& r, int64_t row) {
  const int64_t o = row / r.inner, i = row - o * r.inner;
  return static_cast<T*>(r.base) + o * r.stride_outer + i * r.stride_inner;
}

__device__ __forceinline__ float row_weight(const TokenIndex& t, int64_t row) {
  if (t.mask == nullptr) return 1.f;
  if (t.mask_kind == 1) return static_cast<const uint8_t*>(t.mask)[row] != 0 ? 1.f : 0.f;
  return static_cast<const float*>(t.mask)[row];
}

// The row's token, or -1 where the row does not count; `w` its weight.
__device__ __forceinline__ int64_t row_token(const TokenIndex& t, int64_t row, int64_t vocab, float& w) {
  const int64_t tok = t.tokens_i64 ? static_cast<const int64_t*>(t.tokens)[row]
                                   : static_cast<int64_t>(static_cast<const int32_t*>(t.tokens)[row]);
  w = row_weight(t, row);
  if (tok < 0 || tok >= vocab || w == 0.f) {
    w = 0.f;
    return -1;
  }
  return tok;
}

// ---- running softmax ------------------------------------------------------------------------------------------------
// m: maximum so far (starts at the lowest finite value, so rows and columns at that value or at -inf stay defined),
// s: sum of 2^((z - m) k), t: sum of 2^((z - m) k) (z - m) k (entropy only).
struct Soft {
  float m, s, t;
};

// log2(e) / T as a sum of two floats, the first rounded towards zero: with one float its rounding shifts every exponent
// the same way, an error of the log-sum that all rows share and that the sum over a sequence adds up (mean error of a
// log-probability over 2,000 rows of 65,536 columns: below 1e-8; with one float, and rescaling by ex2.approx, 9e-8).
struct Base {
  float hi, lo;  // both positive, so -inf stays -inf
  float inv_temp;
  __device__ __forceinline__ float operator()(float dz) const { return fmaf(dz, hi, dz * lo); }
  // Factor of sums whose maximum grows, dz = old - new: rare, so by the accurate function.
  __device__ __forceinline__ float fall(float dz) const { return expf(dz * inv_temp); }
};

template <bool kEnt>
__device__ __forceinline__ void soft_raise(Soft& a, float m, const Base& k) {
  const float c = k.fall(a.m - m);
  if (kEnt) a.t = c * fmaf(a.s, fmaxf(k(a.m - m), kFar), a.t);
  a.s *= c;
  a.m = m;
}

template <bool kEnt, int N>
__device__ __forceinline__ void soft_absorb(Soft& a, const float (&x)[N], const Base& k) {
  float top = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) top = fmaxf(top, x[i]);
  if (top > a.m) soft_raise<kEnt>(a, top, k);
  float s[2] = {0.f, 0.f}, t[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = k(x[i] - a.m), e = ex2(d);
    s[i & 1] += e;
    if (kEnt) t[i & 1] = fmaf(e, fmaxf(d, kFar), t[i & 1]);
  }
  a.s += s[0] + s[1];
  if (kEnt) a.t += t[0] + t[1];
}

template <bool kEnt>
__device__ __forceinline__ void soft_warp_reduce(Soft& a, const Base& k) {
  float m = a.m;
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  soft_raise<kEnt>(a, m, k);
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
    if (kEnt) a.t += __shfl_xor_sync(0xffffffffu, a.t, o);
  }
}

// ---- the policy objective of one row ----------------------------------------------------------------------------------
// Tie rules are torch's: the clamp passes its gradient on the closed interval, max() prefers the larger branch. NaN in
// any input reaches the terms and the coefficient.
__device__ __forceinline__ void policy_row(const PolicyTerms& q, int64_t row, float logp, float H, float w,
                                           float4& terms, float2& coef) {
  const float ratio = expf(logp - q.old_logp[row]);
  const float na = -q.adv[row];
  const float free = na * ratio;
  const float cut = na * fminf(fmaxf(ratio, q.clip_lo), q.clip_hi);
  const bool up = free > cut || isnan(free);
  const bool open = up || (ratio >= q.clip_lo && ratio <= q.clip_hi);
  float a = open ? free : 0.f;
  float kl = 0.f;
  if (q.ref_logp != nullptr) {
    const float d = q.ref_logp[row] - logp;
    float g;
    if (q.kl_kind == kKl1) {
      kl = -d, g = 1.f;
    } else if (q.kl_kind == kKl2) {
      kl = 0.5f * d * d, g = -d;
    } else {
      const float e = expm1f(d);
      kl = e - d, g = -e;
    }
    if (q.kl_coef != 0.f) a = fmaf(q.kl_coef, g, a);
  }
  terms = make_float4(w * (up ? free : cut), w * kl, w * H, cut > free ? w : 0.f);
  coef = make_float2(w * a, -q.entropy_coef * w);
}

// ---- row statistics ---------------------------------------------------------------------------------------------------
constexpr int kStatThreads = 256;
constexpr int kStatWarps = kStatThreads / 32;
constexpr int kMaxCluster = 8;

// One cluster of CTAs per row (one CTA where there are enough rows), each CTA a share of the row's 16-byte vectors; the
// shares' (m, s, t) meet in the first CTA's shared memory.
template <typename T, bool kEnt>
__global__ void __launch_bounds__(kStatThreads) token_stats_kernel(const TokenStatsArgs a, const PolicyTerms q,
                                                                   bool policy, const Base k) {
  griddep_wait();  // launched with programmatic stream serialization (launch_pdl)
  griddep_launch_dependents();
  constexpr int VN = Elem<T>::kPerVec;
  constexpr int kVecs = 16 / VN * 2;  // vectors in flight per thread: 32 elements
  __shared__ Soft s_warp[kStatWarps];
  __shared__ Soft s_cta[2][kMaxCluster];
  const cg::cluster_group cluster = cg::this_cluster();
  const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int parity = 0;
  for (int64_t row = blockIdx.x / ranks; row < a.rows; row += gridDim.x / ranks) {
    float w;
    const int64_t tok = row_token(a.idx, row, a.vocab, w);
    if (tok < 0) {
      if (rank == 0 && threadIdx.x == 0) {
        a.logp[row] = 0.f;
        if (kEnt && a.entropy) a.entropy[row] = 0.f;
        if (a.ml) a.ml[row] = make_float2(0.f, 0.f);
        if (policy) {
          a.terms[row] = make_float4(0.f, 0.f, 0.f, 0.f);
          a.coef[row] = make_float2(0.f, 0.f);
        }
      }
      continue;
    }
    const T* z = row_ptr<const T>(a.z, row);
    const int mis = static_cast<int>(reinterpret_cast<uintptr_t>(z) & 15u) / static_cast<int>(sizeof(T));
    const int64_t head = min(static_cast<int64_t>(mis ? VN - mis : 0), a.vocab);
    const int64_t nvec = (a.vocab - head) / VN;
    const int64_t tail = head + nvec * VN;
    const uint4* zv = reinterpret_cast<const uint4*>(z + head);
    Soft acc{-FLT_MAX, 0.f, 0.f};
    if (rank == 0 && warp == 0) {  // at most VN - 1 elements before and behind the vectors
      float x[2] = {-INFINITY, -INFINITY};
      if (lane < head) x[0] = Elem<T>::get(z[lane]);
      if (lane < a.vocab - tail) x[1] = Elem<T>::get(z[tail + lane]);
      soft_absorb<kEnt>(acc, x, k);
    }
    const int64_t step = static_cast<int64_t>(ranks) * kStatThreads;
    int64_t i = static_cast<int64_t>(rank) * kStatThreads + threadIdx.x;
    for (; i + (kVecs - 1) * step < nvec; i += kVecs * step) {
      uint4 v[kVecs];
#pragma unroll
      for (int j = 0; j < kVecs; ++j) v[j] = __ldg(zv + i + j * step);
      float x[kVecs * VN];
#pragma unroll
      for (int j = 0; j < kVecs; ++j) Elem<T>::unpack(v[j], x + j * VN);
      soft_absorb<kEnt>(acc, x, k);
    }
    for (; i < nvec; i += step) {
      float x[VN];
      Elem<T>::unpack(__ldg(zv + i), x);
      soft_absorb<kEnt>(acc, x, k);
    }
    soft_warp_reduce<kEnt>(acc, k);
    __syncthreads();  // the previous row's s_warp has been read
    if (lane == 0) s_warp[warp] = acc;
    __syncthreads();
    if (warp == 0) {
      acc = lane < kStatWarps ? s_warp[lane] : Soft{-FLT_MAX, 0.f, 0.f};
      soft_warp_reduce<kEnt>(acc, k);
    }
    if (ranks > 1) {
      if (threadIdx.x == 0) *cluster.map_shared_rank(&s_cta[parity][rank], 0) = acc;
      cluster.sync();
      if (rank == 0 && warp == 0) {
        acc = lane < ranks ? s_cta[parity][lane] : Soft{-FLT_MAX, 0.f, 0.f};
        soft_warp_reduce<kEnt>(acc, k);
      }
      parity ^= 1;
    }
    if (rank == 0 && threadIdx.x == 0) {
      const float lns = logf(acc.s);
      const float logp = static_cast<float>((Elem<T>::get(z[tok]) - acc.m) * a.inv_temp) - lns;
      const float H = kEnt ? lns - acc.t / acc.s * kLn2 : 0.f;
      a.logp[row] = logp;
      if (kEnt && a.entropy) a.entropy[row] = H;
      if (a.ml) a.ml[row] = make_float2(acc.m, log2f(acc.s));
      if (policy) {
        float4 terms;
        float2 coef;
        policy_row(q, row, logp, H, w, terms, coef);
        a.terms[row] = terms;
        a.coef[row] = coef;
      }
    }
  }
}

int sm_count() {
  int dev = 0, n = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n;
}

Base base_of(double inv_temp) {
  const double k = inv_temp * kLog2e;
  Base b;
  b.hi = static_cast<float>(k);
  if (static_cast<double>(b.hi) >= k) b.hi = std::nextafterf(b.hi, 0.f);
  b.lo = static_cast<float>(k - static_cast<double>(b.hi));
  b.inv_temp = static_cast<float>(inv_temp);
  return b;
}

template <typename T, bool kEnt>
cudaError_t launch_stats(const TokenStatsArgs& a, cudaStream_t stream) {
  const int sms = sm_count();
  // few rows: a row's vectors over up to 8 CTAs, while every thread keeps a vector and the CTAs stay within two an SM
  int ranks = 1;
  const int64_t nvec = a.vocab / Elem<T>::kPerVec;
  while (ranks < kMaxCluster && a.rows * ranks * 2 <= 2 * sms && nvec >= 2 * ranks * kStatThreads) ranks *= 2;
  const int64_t clusters = std::min<int64_t>(a.rows, static_cast<int64_t>(sms) * 64);
  PolicyTerms q{};
  if (a.policy) q = *a.policy;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(clusters * ranks));
  cfg.blockDim = dim3(kStatThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, token_stats_kernel<T, kEnt>, a, q, a.policy != nullptr, base_of(a.inv_temp));
}

// ---- gradient of the logits from the row statistics -----------------------------------------------------------------------
constexpr int kGradThreads = 256;
constexpr int kGradVecs = 8;  // vectors per thread

// dz_j = scale / T (a (delta_j - p_j) - b p_j (log p_j + H)); a block writes one row's segment of 16-byte vectors.
template <typename T, bool kEnt>
__global__ void __launch_bounds__(kGradThreads) token_grad_kernel(const TokenGradArgs a, int64_t segs) {
  griddep_wait();  // launched with programmatic stream serialization (launch_pdl)
  griddep_launch_dependents();
  constexpr int VN = Elem<T>::kPerVec;
  const int64_t row = a.rows - 1 - blockIdx.x / segs, seg = blockIdx.x % segs;
  T* out = row_ptr<T>(a.out, row);
  float w;
  const int64_t tok = row_token(a.idx, row, a.vocab, w);
  const int mis = static_cast<int>(reinterpret_cast<uintptr_t>(out) & 15u) / static_cast<int>(sizeof(T));
  const int64_t head = min(static_cast<int64_t>(mis ? VN - mis : 0), a.vocab);
  const int64_t nvec = (a.vocab - head) / VN, tail = head + nvec * VN;
  uint4* ov = reinterpret_cast<uint4*>(out + head);
  const int64_t v0 = seg * (kGradThreads * kGradVecs), v1 = min(nvec, v0 + kGradThreads * kGradVecs);
  float ca = 0.f, cb = 0.f;
  if (tok >= 0) {
    float f = static_cast<float>(a.scale * a.inv_temp);
    if (a.scale_a) f *= *a.scale_a;
    if (a.scale_b) f *= *a.scale_b;
    if (!a.weighted) f *= w;
    ca = a.a[row * a.a_stride] * f;
    if (kEnt) cb = a.b[row * a.b_stride] * f;
  }
  if (tok < 0 || (ca == 0.f && (!kEnt || cb == 0.f))) {  // nothing to read
    for (int64_t i = v0 + threadIdx.x; i < v1; i += kGradThreads) ov[i] = make_uint4(0u, 0u, 0u, 0u);
    if (seg == 0 && threadIdx.x < head) out[threadIdx.x] = Elem<T>::put(0.f);
    if (seg == 0 && threadIdx.x < a.vocab - tail) out[tail + threadIdx.x] = Elem<T>::put(0.f);
    return;
  }
  const T* z = row_ptr<const T>(a.z, row);
  const float2 ml = a.ml[row];
  const float k = static_cast<float>(a.inv_temp * kLog2e);
  const float H = kEnt ? a.entropy[row] : 0.f;
  const float c0 = -ca - cb * H, c1 = -cb * kLn2;
  auto grad = [&](float x, int64_t col) {
    const float lp = (x - ml.x) * k - ml.y;  // log2 p
    const float p = ex2(lp);
    float g = p * (kEnt ? fmaf(c1, fmaxf(lp, kFar), c0) : c0);
    return col == tok ? g + ca : g;
  };
  if (seg == 0 && threadIdx.x < head) out[threadIdx.x] = Elem<T>::put(grad(Elem<T>::get(z[threadIdx.x]), threadIdx.x));
  if (seg == 0 && threadIdx.x < a.vocab - tail) {
    const int64_t col = tail + threadIdx.x;
    out[col] = Elem<T>::put(grad(Elem<T>::get(z[col]), col));
  }
  const bool same = ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
  if (same) {
    const uint4* zv = reinterpret_cast<const uint4*>(z + head);
#pragma unroll
    for (int h = 0; h < kGradVecs; h += 4) {
      uint4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t i = v0 + (h + j) * kGradThreads + threadIdx.x;
        if (i < v1) v[j] = __ldg(zv + i);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t i = v0 + (h + j) * kGradThreads + threadIdx.x;
        if (i >= v1) continue;
        float x[VN];
        Elem<T>::unpack(v[j], x);
        const int64_t col = head + i * VN;
#pragma unroll
        for (int e = 0; e < VN; ++e) x[e] = grad(x[e], col + e);
        ov[i] = Elem<T>::pack(x);
      }
    }
  } else {  // rows of input and output start at different places within 16 bytes
    for (int64_t i = v0 + threadIdx.x; i < v1; i += kGradThreads) {
      const int64_t col = head + i * VN;
      float x[VN];
#pragma unroll
      for (int e = 0; e < VN; ++e) x[e] = grad(Elem<T>::get(z[col + e]), col + e);
      ov[i] = Elem<T>::pack(x);
    }
  }
}

template <typename T>
cudaError_t launch_grad(const TokenGradArgs& a, cudaStream_t stream) {
  constexpr int64_t per = static_cast<int64_t>(kGradThreads) * kGradVecs * Elem<T>::kPerVec;
  const int64_t segs = std::max<int64_t>(1, (a.vocab + per - 1) / per);
  const dim3 grid(static_cast<unsigned>(a.rows * segs));
  if (a.b) return launch_pdl(token_grad_kernel<T, true>, grid, dim3(kGradThreads), 0, stream, a, segs);
  return launch_pdl(token_grad_kernel<T, false>, grid, dim3(kGradThreads), 0, stream, a, segs);
}

// ---- sums over rows, sequences and pairs -----------------------------------------------------------------------------------
template <int N>
__device__ __forceinline__ void block_sum(double (&x)[N], double* smem) {  // result in every thread; fixed order
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    for (int o = 16; o >= 1; o >>= 1) x[n] += __shfl_xor_sync(0xffffffffu, x[n], o);
  }
  __syncthreads();
  if (lane == 0) {
#pragma unroll
    for (int n = 0; n < N; ++n) smem[warp * N + n] = x[n];
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    x[n] = 0.0;
    for (int i = 0; i < warps; ++i) x[n] += smem[i * N + n];
  }
}

constexpr int kFinishThreads = 512;
__global__ void __launch_bounds__(kFinishThreads) policy_finish_kernel(const PolicyFinishArgs a) {
  griddep_wait();  // launched with programmatic stream serialization (launch_pdl)
  griddep_launch_dependents();
  __shared__ double s_sum[kFinishThreads / 32 * 5];
  double x[5] = {0.0, 0.0, 0.0, 0.0, 0.0};
  for (int64_t r = threadIdx.x; r < a.rows; r += kFinishThreads) {
    const float4 t = a.terms[r];
    float w;
    row_token(a.idx, r, a.vocab, w);
    x[0] += t.x, x[1] += t.y, x[2] += t.z, x[3] += t.w, x[4] += w;
  }
  block_sum(x, s_sum);
  if (threadIdx.x == 0) {
    const double inv = x[4] != 0.0 ? 1.0 / x[4] : 0.0;  // no row counts: loss and gradients are zero
    const double f = a.mean ? inv : 1.0;
    a.out[0] = static_cast<float>(f * (x[0] + a.kl_coef * x[1] - a.entropy_coef * x[2]));
    for (int n = 0; n < 4; ++n) a.out[1 + n] = static_cast<float>(inv * x[n]);
    a.out[5] = static_cast<float>(f);
  }
}

__device__ __forceinline__ int64_t seq_start(const PreferenceArgs& a, int64_t s) {
  int64_t o = a.offsets == nullptr ? s * a.length
              : a.offsets_i64      ? static_cast<const int64_t*>(a.offsets)[s]
                                   : static_cast<int64_t>(static_cast<const int32_t*>(a.offsets)[s]);
  return min(max(o, static_cast<int64_t>(0)), a.rows);
}

// -log sigmoid(x)
__device__ __forceinline__ double softplus_neg(double x) { return log1p(exp(-fabs(x))) + fmax(-x, 0.0); }

constexpr int kPairThreads = 1024;
// One block: a warp per sequence sums its tokens' log-probabilities in 64 bits, then the pairs' losses, then every row's
// coefficient. Tens of thousands of rows are a few hundred kilobytes, so one block's time stays far below the logits'.
__global__ void __launch_bounds__(kPairThreads) preference_pairs_kernel(const PreferenceArgs a) {
  griddep_wait();  // launched with programmatic stream serialization (launch_pdl)
  griddep_launch_dependents();
  __shared__ double s_sum[kPairThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = kPairThreads / 32;
  for (int64_t r = threadIdx.x; r < a.rows; r += kPairThreads) a.coef[r] = 0.f;
  __syncthreads();
  double loss[1] = {0.0};
  const int64_t pairs = a.seqs / 2;
  for (int64_t p = warp; p < pairs; p += warps) {
    double sum[2], count[2], lp[2];
    for (int c = 0; c < 2; ++c) {
      const int64_t r0 = seq_start(a, 2 * p + c), r1 = seq_start(a, 2 * p + c + 1);
      sum[c] = 0.0, count[c] = 0.0;
      for (int64_t r = r0 + lane; r < r1; r += 32) {
        float w;
        if (row_token(a.idx, r, a.vocab, w) < 0) continue;
        sum[c] += static_cast<double>(w) * a.logp[r];
        count[c] += w;
      }
      for (int o = 16; o >= 1; o >>= 1) {
        sum[c] += __shfl_xor_sync(0xffffffffu, sum[c], o);
        count[c] += __shfl_xor_sync(0xffffffffu, count[c], o);
      }
      lp[c] = !a.average ? sum[c] : count[c] != 0.0 ? sum[c] / count[c] : 0.0;
    }
    double rew[2];
    for (int c = 0; c < 2; ++c) rew[c] = a.beta * (lp[c] - (a.ref ? static_cast<double>(a.ref[2 * p + c]) : 0.0));
    const double h = rew[0] - rew[1];
    double l, dh;  // loss of the pair and its derivative by h
    if (a.kind == kPrefSigmoid) {
      l = (1.0 - a.smoothing) * softplus_neg(h) + a.smoothing * softplus_neg(-h);
      dh = a.smoothing / (1.0 + exp(-h)) - (1.0 - a.smoothing) / (1.0 + exp(h));
    } else if (a.kind == kPrefHinge) {
      l = fmax(1.0 - h, 0.0);
      l = isnan(h) ? h : l;
      dh = h < 1.0 ? -1.0 : 0.0;
    } else {  // squared distance of the log-ratio difference h / beta from 1 / (2 beta)
      const double d = h / a.beta - 0.5 / a.beta;
      l = d * d;
      dh = 2.0 * d / a.beta;
    }
    if (lane == 0) loss[0] += l;
    const double g = dh * a.beta / static_cast<double>(pairs);
    for (int c = 0; c < 2; ++c) {
      if (lane == 0) {
        a.seq_logp[2 * p + c] = static_cast<float>(lp[c]);
        a.rewards[2 * p + c] = static_cast<float>(rew[c]);
      }
      double gc = c == 0 ? g : -g;
      if (a.average) gc = count[c] != 0.0 ? gc / count[c] : 0.0;
      const int64_t r0 = seq_start(a, 2 * p + c), r1 = seq_start(a, 2 * p + c + 1);
      for (int64_t r = r0 + lane; r < r1; r += 32) {
        float w;
        row_token(a.idx, r, a.vocab, w);
        a.coef[r] = static_cast<float>(gc * w);
      }
    }
  }
  block_sum(loss, s_sum);
  if (threadIdx.x == 0) a.loss[0] = pairs ? static_cast<float>(loss[0] / static_cast<double>(pairs)) : 0.f;
}

}  // namespace

cudaError_t token_stats(const TokenStatsArgs& a, cudaStream_t stream) {
  if (a.rows == 0) return cudaSuccess;
  const bool ent = a.entropy != nullptr;
  switch (a.dtype) {
    case kTokF32: return ent ? launch_stats<float, true>(a, stream) : launch_stats<float, false>(a, stream);
    case kTokBF16:
      return ent ? launch_stats<__nv_bfloat16, true>(a, stream) : launch_stats<__nv_bfloat16, false>(a, stream);
    default: return ent ? launch_stats<__half, true>(a, stream) : launch_stats<__half, false>(a, stream);
  }
}

cudaError_t token_grad(const TokenGradArgs& a, cudaStream_t stream) {
  if (a.rows == 0) return cudaSuccess;
  switch (a.dtype) {
    case kTokF32: return launch_grad<float>(a, stream);
    case kTokBF16: return launch_grad<__nv_bfloat16>(a, stream);
    default: return launch_grad<__half>(a, stream);
  }
}

cudaError_t policy_finish(const PolicyFinishArgs& a, cudaStream_t stream) {
  return launch_pdl(policy_finish_kernel, dim3(1), dim3(kFinishThreads), 0, stream, a);
}

cudaError_t preference_pairs(const PreferenceArgs& a, cudaStream_t stream) {
  return launch_pdl(preference_pairs_kernel, dim3(1), dim3(kPairThreads), 0, stream, a);
}

}  // namespace rlb
