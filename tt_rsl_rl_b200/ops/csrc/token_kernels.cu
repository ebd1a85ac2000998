// Kernels of the token-policy operators (see token_kernels.cuh for the formulas).
//
// Determinism: every sum over a row, a sequence or a batch has a fixed order; no atomics.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <mutex>
#include <vector>

#include "sm100_primitives.cuh"
#include "token_kernels.cuh"

namespace rlb {
namespace {

namespace cg = cooperative_groups;

constexpr double kLog2e = 1.4426950408889634;
constexpr float kLn2 = 0.6931471805599453f, kLn2Lack = -1.90465429995776e-9f;  // ln 2 as a sum
constexpr float kFar = -1e30f;  // exponent of a column of probability zero: its product with that zero stays a number

// One instruction, within 2^-22 of 2^x; results below 2^-126 are zero. What is summed over columns is no more exact than that;
// what is done once a row uses the accurate functions.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float at_least_far(float d) {  // a NaN stays one
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(d), "f"(kFar));
  return y;
}

__device__ __forceinline__ Pair ex2(const Pair& x) {
  float lo, hi;
  x.split(lo, hi);
  return Pair(ex2(lo), ex2(hi));
}

// In a row whose maximum is not far from zero (is_near) a column below this one counts as it: its probability is zero, and
// that zero's products stay numbers.
constexpr float kLow = -73786976294838206464.f;  // -2^66
__device__ __forceinline__ float at_least_low(float z) {  // a NaN stays one
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(z), "f"(kLow));
  return y;
}

// Loads of a row that is read twice: the first keeps it in L2, the second lets it go.
__device__ __forceinline__ uint4 load_hint(const uint4* p, uint64_t policy) {
  uint4 v;
  asm volatile("ld.global.nc.L2::cache_hint.v4.u32 {%0, %1, %2, %3}, [%4], %5;"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p), "l"(policy));
  return v;
}
template <bool kAgain>
__device__ __forceinline__ uint4 load_first(const uint4* p) {
  if (!kAgain) return __ldg(p);
  uint64_t policy;
  asm("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(policy));
  return load_hint(p, policy);
}
__device__ __forceinline__ uint4 load_last(const uint4* p) {
  uint64_t policy;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  return load_hint(p, policy);
}

template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static constexpr int kPerVec = 4;
  static constexpr uint32_t kNone = 0xff800000u;  // -inf
  static __device__ __forceinline__ float top(const uint4& v) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  static __device__ __forceinline__ void unpack_low(const uint4& v, float* x) {
    unpack(v, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = at_least_low(x[i]);
  }
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
  static constexpr uint32_t kNone = 0xff80ff80u;
  static __device__ __forceinline__ float top(const uint4& v) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ void unpack_low(uint4 v, float* x) {
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
    const __nv_bfloat162 low = __float2bfloat162_rn(kLow);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __hmax2_nan(h[i], low);
    unpack(v, x);
  }
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
  static constexpr uint32_t kNone = 0xfc00fc00u;
  static __device__ __forceinline__ float top(const uint4& v) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
    const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ void unpack_low(const uint4& v, float* x) {
    unpack(v, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = at_least_low(x[i]);
  }
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
  if (row < r.inner) return static_cast<T*>(r.base) + row * r.stride_inner;
  const uint32_t o = static_cast<uint32_t>(row) / static_cast<uint32_t>(r.inner);  // rows are below 2^31
  const uint32_t i = static_cast<uint32_t>(row) - o * static_cast<uint32_t>(r.inner);
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
// The exponent of a column is d = z hi + c, one fused multiply-add, with c = -m hi for the largest z so far: any c near
// -m hi serves as long as the sums and their use agree on it, and c's rounding is at most 1/2 while |m| hi < 2^24. Beyond
// that (logits of 1.2e7 at T = 1, of 12 at T = 1e-6; a row masked with -1e10 or the lowest value everywhere) the maximum is
// subtracted first, d = (z - m) hi: c would shift the exponents out of range there. `hi` is log2(e) / T rounded to a float;
// what it lacks (lo) shifts every exponent of a row the same way, an error that the sum over a sequence's rows would add up,
// so the end corrects for it: d ln s / dk = sum p z.
//
// m: maximum so far (starts at the lowest finite value, so rows and columns at that value or at -inf stay defined),
// s: sum of 2^d, t: sum of 2^d d.
struct Soft {
  float m, s, t;
};

struct Base {
  float hi, lo;         // log2(e) / T as a sum
  float inv, inv_lack;  // 1 / T as a sum
};

// Rounded on its own: a product that the compiler fuses into the sum behind it is another shift than the columns' one.
__device__ __forceinline__ float shift_of(float m, const Base& k) { return __fmul_rn(-m, k.hi); }
__device__ __forceinline__ bool is_near(float m, const Base& k) { return fabsf(shift_of(m, k)) < 16777216.f; }

// The exponent of the maximum itself: what the rounding of c shifts all of its row's exponents by (exact).
__device__ __forceinline__ float offset_of(float m, const Base& k) {
  return is_near(m, k) ? fmaf(m, k.hi, shift_of(m, k)) : 0.f;
}

// Rare, so by the accurate function: a chain of these with ex2.approx, which is low by 5e-8 on average, shows in sums.
__device__ __forceinline__ void soft_raise(Soft& a, float m, const Base& k) {
  float d = shift_of(m, k) - shift_of(a.m, k);
  if (__builtin_expect(!(is_near(m, k) && is_near(a.m, k)), 0)) {
    d = (a.m - m) * k.hi + (offset_of(m, k) - offset_of(a.m, k));
  }
  const float f = expf(d * kLn2);
  a.t = f * fmaf(a.s, fmaxf(d, kFar), a.t);
  a.s *= f;
  a.m = m;
}

constexpr int kChunk = 4;  // vectors of a step: 32 or 16 columns

template <typename T>
__device__ __forceinline__ void soft_absorb(Soft& a, const uint4* v, const Base& k) {
  constexpr int VN = Elem<T>::kPerVec;
  float top = Elem<T>::top(v[0]);
#pragma unroll
  for (int j = 1; j < kChunk; ++j) top = fmaxf(top, Elem<T>::top(v[j]));
  if (top > a.m) soft_raise(a, top, k);
  if (__builtin_expect(is_near(a.m, k), 1)) {
    const float c = shift_of(a.m, k);
    const Pair hi2(k.hi, k.hi), c2(c, c);
    Pair s[2] = {{0.f, 0.f}, {0.f, 0.f}}, t[2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
    for (int j = 0; j < kChunk; ++j) {
      float x[VN];
      Elem<T>::unpack_low(v[j], x);
#pragma unroll
      for (int i = 0; i < VN; i += 2) {
        const Pair d = fma2(Pair(x[i], x[i + 1]), hi2, c2), e = ex2(d);
        s[(i >> 1) & 1] = add2(s[(i >> 1) & 1], e);
        t[(i >> 1) & 1] = fma2(e, d, t[(i >> 1) & 1]);
      }
    }
    float s0, s1, t0, t1;
    add2(s[0], s[1]).split(s0, s1);
    add2(t[0], t[1]).split(t0, t1);
    a.s += s0 + s1;
    a.t += t0 + t1;
  } else {
    float s = 0.f, t = 0.f;
#pragma unroll
    for (int j = 0; j < kChunk; ++j) {
      float x[VN];
      Elem<T>::unpack(v[j], x);
#pragma unroll
      for (int i = 0; i < VN; ++i) {
        const float d = at_least_far((x[i] - a.m) * k.hi), e = ex2(d);
        s += e;
        t = fmaf(e, d, t);
      }
    }
    a.s += s;
    a.t += t;
  }
}
// One column.
__device__ __forceinline__ void soft_absorb_one(Soft& a, float x, const Base& k) {
  if (x > a.m) soft_raise(a, x, k);
  const float d = at_least_far(is_near(a.m, k) ? fmaf(x, k.hi, shift_of(a.m, k)) : (x - a.m) * k.hi), e = ex2(d);
  a.s += e;
  a.t = fmaf(e, d, a.t);
}

__device__ __forceinline__ void soft_warp_reduce(Soft& a, const Base& k) {
  float m = a.m;
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (m > a.m) soft_raise(a, m, k);
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
    a.t += __shfl_xor_sync(0xffffffffu, a.t, o);
  }
}

// What a row's sums say: ln sum_j e^((z_j - m) / T) = lns + rest, where lns is a multiple of ln 2 and the rest below one, so
// that a log-probability is rounded once. The rest has what the rounding of c and of hi has shifted (about 1e-6 for ordinary
// logits, at most 1/2).
struct RowSoft {
  float m, lns, rest;
  float mean;  // of z - m under p
  float entropy;
};
__device__ __forceinline__ RowSoft row_soft(const Soft& a, const Base& k) {
  RowSoft r;
  r.m = a.m;
  const float off = offset_of(a.m, k);
  const uint32_t bits = __float_as_uint(a.s);
  const bool normal = a.s > 1e-30f && a.s < 1e30f;
  const float e = normal ? static_cast<float>(static_cast<int>(bits >> 23) - 127) : 0.f;
  const float f = normal ? __uint_as_float((bits & 0x7fffffu) | 0x3f800000u) : a.s;
  r.lns = __fmul_rn(e, kLn2);
  const float td = a.t / a.s;
  r.mean = (td - off) / k.hi;
  const float rest = logf(f) + (fmaf(e, kLn2, -r.lns) + e * kLn2Lack);  // of the sums as they are
  r.rest = rest + kLn2 * fmaf(k.lo, r.mean, -off);
  r.entropy = r.lns + (rest - td * kLn2);
  return r;
}
__device__ __forceinline__ float row_logp(const RowSoft& r, float z, const Base& k) {
  const float d = z - r.m;
  const float x = isinf(d) ? d : fmaf(d, k.inv, d * k.inv_lack), y = x - r.lns;
  if (isinf(x)) return y - r.rest;  // -inf, or the type's lowest value over a T below one; NaN where the sums are
  const float back = y + r.lns;  // the rounding of y by the two-sum
  return y + (((x - back) + (back - y - r.lns)) - r.rest);
}
// What a gradient needs of a row: p_j = f 2^(z_j hi + c), f the rounding of c to a float; f < 0 marks a row whose maximum is
// far from zero: p_j = 2^((z_j - c) hi + 1 + f).
__device__ __forceinline__ float2 row_shift(const RowSoft& r, const Base& k) {
  constexpr float kE = 1.44269504f, kELack = 1.92596299e-8f;  // log2(e) as a sum
  const float l = __fmul_rn(r.lns, kE), l_lack = fmaf(r.lns, kE, -l) + r.lns * kELack + r.rest * kE;
  if (!is_near(r.m, k)) return make_float2(r.m, -1.f - (l + l_lack));
  const float p = __fmul_rn(r.m, k.hi), p_lack = fmaf(r.m, k.hi, -p);
  const float c = -(p + l), t = -c - p;  // c's own rounding by the two-sum
  const float lack = (p - (-c - t)) + (l - t) + p_lack + l_lack;
  // what hi lacks at the mean of z; the columns around it differ by less than a rounding
  return make_float2(c, exp2f(fmaf(k.lo, r.mean, -lack)));
}

// ---- the policy objective of one row ----------------------------------------------------------------------------------
// Tie rules are torch's: the clamp passes its gradient on the closed interval, max() prefers the larger branch. NaN in
// any input reaches the terms and the coefficient.
struct PolicyIn {  // of one row; loaded before the row's sums, whose time hides the latency
  float old_logp, adv, ref_logp;
  __device__ __forceinline__ PolicyIn(float old, float advantage, float ref)
      : old_logp(old), adv(advantage), ref_logp(ref) {}
  __device__ __forceinline__ PolicyIn(const PolicyTerms& q, int64_t row)
      : old_logp(q.old_logp[row]), adv(q.adv[row]), ref_logp(q.ref_logp ? q.ref_logp[row] : 0.f) {}
};
__device__ __forceinline__ void policy_row(const PolicyTerms& q, const PolicyIn& in, float logp, float H, float w,
                                           float4& terms, float2& coef) {
  const float ratio = expf(logp - in.old_logp);
  const float na = -in.adv;
  const float free = na * ratio;
  const float cut = na * fminf(fmaxf(ratio, q.clip_lo), q.clip_hi);
  const bool up = free > cut || isnan(free);
  const bool open = up || (ratio >= q.clip_lo && ratio <= q.clip_hi);
  float a = open ? free : 0.f;
  float kl = 0.f;
  if (q.ref_logp != nullptr) {
    const float d = in.ref_logp - logp;
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

// ---- a row per CTA or cluster -------------------------------------------------------------------------------------------
constexpr int kMostThreads = 256;
constexpr int kMostWarps = kMostThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kFlight = 4;  // 16-byte loads that a thread has in flight on the way to the gradient

// A row's columns: up to VN - 1 single ones, 16-byte vectors, up to VN - 1 single ones.
template <typename T>
struct RowView {
  const T* z;
  const uint4* zv;
  int head, nvec, tail;  // first column of the vectors, their number, first column behind them
  __device__ __forceinline__ RowView(const T* row, int64_t vocab) : z(row) {
    constexpr int VN = Elem<T>::kPerVec;
    const int mis = static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15u) / static_cast<int>(sizeof(T));
    head = static_cast<int>(min(static_cast<int64_t>(mis ? VN - mis : 0), vocab));
    nvec = static_cast<int>(vocab - head) / VN;
    tail = head + nvec * VN;
    zv = reinterpret_cast<const uint4*>(row + head);
  }
};

// The row's single columns, by the first warp of the first CTA.
template <typename T>
__device__ __forceinline__ void edge_share(Soft& acc, const T* z, int head, int tail, int64_t vocab, const Base& k) {
  const int lane = threadIdx.x & 31;
  if (lane < head) soft_absorb_one(acc, Elem<T>::get(z[lane]), k);
  if (lane < static_cast<int>(vocab) - tail) soft_absorb_one(acc, Elem<T>::get(z[tail + lane]), k);
}

// This thread's share of the row's sums. Eight loads are issued before the first is used: 128 KB in flight on a
// multiprocessor of 1,024 threads.
template <bool kAgain, typename T>
__device__ __forceinline__ Soft row_share(const RowView<T>& r, int64_t vocab, int rank, int ranks, const Base& k) {
  const int threads = blockDim.x, step = ranks * threads;
  const uint4 none = make_uint4(Elem<T>::kNone, Elem<T>::kNone, Elem<T>::kNone, Elem<T>::kNone);
  Soft acc{-FLT_MAX, 0.f, 0.f};
  for (int i = rank * threads + threadIdx.x; i < r.nvec; i += 2 * kChunk * step) {
    uint4 v[2 * kChunk];
#pragma unroll
    for (int j = 0; j < 2 * kChunk; ++j) v[j] = i + j * step < r.nvec ? load_first<kAgain>(r.zv + i + j * step) : none;
    soft_absorb<T>(acc, v, k);
    if (i + kChunk * step < r.nvec) soft_absorb<T>(acc, v + kChunk, k);
  }
  if (rank == 0 && threadIdx.x < 32) edge_share(acc, r.z, r.head, r.tail, vocab, k);
  return acc;
}

struct RowExchange {  // double-buffered: a row's buffers are free once the next row's barrier has been passed
  Soft warp[2][kMostWarps];
  Soft cta[2][kMaxCluster];
};

// Sums of the whole row, in warp 0 of every CTA of the cluster.
__device__ __forceinline__ Soft row_total(Soft acc, RowExchange& x, int parity, int rank, int ranks, const Base& k,
                                          const cg::cluster_group& cluster) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  soft_warp_reduce(acc, k);
  if (warps > 1) {
    if (lane == 0) x.warp[parity][warp] = acc;
    __syncthreads();
    if (warp == 0) {
      acc = lane < warps ? x.warp[parity][lane] : Soft{-FLT_MAX, 0.f, 0.f};
      soft_warp_reduce(acc, k);
    }
  }
  if (ranks > 1) {
    if (static_cast<int>(threadIdx.x) < ranks) *cluster.map_shared_rank(&x.cta[parity][rank], threadIdx.x) = acc;
    cluster.sync();
    if (warp == 0) {
      acc = lane < ranks ? x.cta[parity][lane] : Soft{-FLT_MAX, 0.f, 0.f};
      soft_warp_reduce(acc, k);
    }
  }
  return acc;
}

// dz_j = a (delta_j - p_j) - b p_j (log p_j + H) of four or eight columns, a and b divided by T.
struct RowGrad {
  float2 cf;  // row_shift
  float hi, a, c0, c1;
  RowGrad() = default;
  __device__ __forceinline__ RowGrad(const float2& shift, const Base& k, float a_, float b, float H)
      : cf(shift), hi(k.hi), a(a_) {
    const float f = cf.y > 0.f ? cf.y : 1.f;
    c0 = -f * (a_ + b * (H + logf(f)));
    c1 = -f * b * kLn2;
  }
  template <bool kEnt>
  __device__ __forceinline__ float operator()(float z) const {
    const float q = cf.y > 0.f ? fmaf(z, hi, cf.x) : (z - cf.x) * hi + 1.f + cf.y;
    return ex2(q) * (kEnt ? fmaf(c1, fmaxf(q, kFar), c0) : c0);
  }
  template <typename T, bool kEnt>
  __device__ __forceinline__ uint4 vec(const uint4& v, int col, int tok) const {
    constexpr int VN = Elem<T>::kPerVec;
    float x[VN];
    if (cf.y > 0.f) {
      if (kEnt) Elem<T>::unpack_low(v, x);
      else Elem<T>::unpack(v, x);
      const Pair hi2(hi, hi), cx(cf.x, cf.x), c02(c0, c0), c12(c1, c1);
#pragma unroll
      for (int e = 0; e < VN; e += 2) {
        const Pair q = fma2(Pair(x[e], x[e + 1]), hi2, cx);
        mul2(ex2(q), kEnt ? fma2(c12, q, c02) : c02).split(x[e], x[e + 1]);
      }
    } else {
      Elem<T>::unpack(v, x);
#pragma unroll
      for (int e = 0; e < VN; ++e) x[e] = this->template operator()<kEnt>(x[e]);
    }
    if (static_cast<unsigned>(tok - col) < static_cast<unsigned>(VN)) {
#pragma unroll
      for (int e = 0; e < VN; ++e) x[e] += col + e == tok ? a : 0.f;
    }
    return Elem<T>::pack(x);
  }
  template <typename T, bool kEnt>
  __device__ __forceinline__ T one(T z, int col, int tok) const {
    const float g = this->template operator()<kEnt>(Elem<T>::get(z));
    return Elem<T>::put(col == tok ? g + a : g);
  }
};

template <typename T>
__device__ __forceinline__ void zero_row(T* out, int64_t vocab, int rank, int ranks, int threads) {
  const RowView<T> r(out, vocab);
  uint4* ov = reinterpret_cast<uint4*>(out + r.head);
  for (int i = rank * threads + threadIdx.x; i < r.nvec; i += ranks * threads) __stcs(ov + i, make_uint4(0, 0, 0, 0));
  if (rank == 0 && static_cast<int>(threadIdx.x) < r.head) out[threadIdx.x] = Elem<T>::put(0.f);
  if (rank == 0 && static_cast<int>(threadIdx.x) < static_cast<int>(vocab) - r.tail) {
    out[r.tail + threadIdx.x] = Elem<T>::put(0.f);
  }
}

// ---- row statistics -----------------------------------------------------------------------------------------------------
// A CTA per row, or a cluster of them where rows are few: each CTA a share of the row's vectors, whose sums meet in every
// CTA's shared memory. Bound by memory for fp32 (737 MB in 116 us, 97 % of the copy rate); for bf16 by the instructions of
// a column too (7.9 of them, one the ex2 of the special-function unit): 268 MB in 60 us, 2.1 GB in 316 us (95 %).
template <typename T>
__global__ void __launch_bounds__(kMostThreads, 4) token_stats_kernel(const TokenStatsArgs a, const PolicyTerms q,
                                                                      bool policy, const Base k) {
  __shared__ RowExchange x;
  const cg::cluster_group cluster = cg::this_cluster();
  const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  if (ranks > 1) cluster.barrier_arrive();  // no CTA writes into another before that one has started
  griddep_wait();  // launched with programmatic stream serialization (launch_pdl)
  griddep_launch_dependents();
  if (ranks > 1) cluster.barrier_wait();
  int parity = 0;
  for (int64_t row = blockIdx.x / ranks; row < a.rows; row += gridDim.x / ranks) {
    float w;
    const int64_t tok = row_token(a.idx, row, a.vocab, w);
    if (tok < 0) {
      if (rank == 0 && threadIdx.x == 0) {
        a.logp[row] = 0.f;
        if (a.entropy) a.entropy[row] = 0.f;
        if (a.ml) a.ml[row] = make_float2(0.f, 0.f);
        if (policy) {
          a.terms[row] = make_float4(0.f, 0.f, 0.f, 0.f);
          a.coef[row] = make_float2(0.f, 0.f);
        }
      }
      continue;
    }
    const RowView<T> r(row_ptr<const T>(a.z, row), a.vocab);
    const float zt = Elem<T>::get(r.z[tok]);
    const Soft acc = row_total(row_share<false>(r, a.vocab, rank, ranks, k), x, parity, rank, ranks, k, cluster);
    parity ^= 1;
    if (rank == 0 && threadIdx.x == 0) {
      const RowSoft soft = row_soft(acc, k);
      const float logp = row_logp(soft, zt, k);
      a.logp[row] = logp;
      if (a.entropy) a.entropy[row] = soft.entropy;
      if (a.ml) a.ml[row] = row_shift(soft, k);
      if (policy) {
        float4 terms;
        float2 coef;
        policy_row(q, PolicyIn(q, row), logp, soft.entropy, w, terms, coef);
        a.terms[row] = terms;
        a.coef[row] = coef;
      }
    }
  }
}

// ---- policy loss and gradient in one pass -------------------------------------------------------------------------------
// Sums of a block in fixed order, in every thread. smem: N numbers per warp.
template <int N>
__device__ __forceinline__ void block_sum(double (&x)[N], double* smem) {
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
  if (threadIdx.x < N) {  // fp64 adds are slow: one thread for each sum
    double y = smem[threadIdx.x];
    for (int i = 1; i < warps; ++i) y += smem[i * N + threadIdx.x];
    smem[threadIdx.x] = y;
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) x[n] = smem[n];
}

// A CTA or cluster per row as above, which turns to the row a second time for its gradient as soon as its sums are known:
// the rows in work fit L2 (row_launch), and loads that say which read is the last keep them there. Measured at 8,192 rows
// of 131,072 bf16 columns (a tenth masked): 888 us, where statistics and gradient as two kernels take 316 + 663; memory
// traffic is 1.15 times one read and one write, so most second reads hit. What remains is the latency between the two
// halves of a row (warps wait for loads 5 of 14 cycles). The row held in shared memory behind bulk copies, its clusters of
// 8 exchanging sums, took 1,016 us: an exchange costs 2 us a row.
template <typename T, bool kEnt>
__global__ void __launch_bounds__(kMostThreads, 4) token_policy_kernel(const TokenStatsArgs a, const PolicyTerms q,
                                                                       const TokenRows grad, float scale,
                                                                       const float* scale_device, int mean,
                                                                       const double* weight_sum, const Base k) {
  constexpr int VN = Elem<T>::kPerVec;
  __shared__ RowExchange x;
  __shared__ double s_sum[kMostWarps];
  __shared__ RowGrad s_grad[2];
  const cg::cluster_group cluster = cg::this_cluster();
  const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  if (ranks > 1) cluster.barrier_arrive();  // no CTA writes into another before that one has started
  griddep_wait();  // launched with programmatic stream serialization (launch_pdl)
  griddep_launch_dependents();
  const int threads = blockDim.x;
  if (scale_device) scale *= *scale_device;
  if (mean) {
    double total[1] = {0.0};
    if (weight_sum != nullptr) {
      total[0] = *weight_sum;
    } else {  // few rows: every CTA sums the weights for itself, in the same order
      for (int64_t r = threadIdx.x; r < a.rows; r += threads) {
        float w;
        row_token(a.idx, r, a.vocab, w);
        total[0] += w;
      }
      block_sum(total, s_sum);
    }
    scale *= total[0] != 0.0 ? static_cast<float>(1.0 / total[0]) : 0.f;
  }
  const float factor = scale * k.inv;
  if (ranks > 1) cluster.barrier_wait();
  int parity = 0;
  for (int64_t row = blockIdx.x / ranks; row < a.rows; row += gridDim.x / ranks) {
    float w;
    const int tok = static_cast<int>(row_token(a.idx, row, a.vocab, w));
    T* out = row_ptr<T>(grad, row);
    if (tok < 0) {
      if (rank == 0 && threadIdx.x == 0) {
        a.logp[row] = 0.f;
        a.terms[row] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      zero_row(out, a.vocab, rank, ranks, threads);
      continue;
    }
    const RowView<T> r(row_ptr<const T>(a.z, row), a.vocab);
    const PolicyIn in(q, row);
    const float zt = Elem<T>::get(r.z[tok]);
    const Soft acc = row_total(row_share<true>(r, a.vocab, rank, ranks, k), x, parity, rank, ranks, k, cluster);
    if (threadIdx.x < 32) {
      const RowSoft soft = row_soft(acc, k);
      const float logp = row_logp(soft, zt, k);
      float4 terms;
      float2 coef;
      policy_row(q, in, logp, soft.entropy, w, terms, coef);
      if (threadIdx.x == 0) {
        s_grad[parity] = RowGrad(row_shift(soft, k), k, coef.x * factor, kEnt ? coef.y * factor : 0.f, soft.entropy);
        if (rank == 0) {
          a.logp[row] = logp;
          a.terms[row] = terms;
        }
      }
    }
    __syncthreads();
    const RowGrad g = s_grad[parity];
    parity ^= 1;
    if (g.a == 0.f && (!kEnt || g.c1 == 0.f)) {
      zero_row(out, a.vocab, rank, ranks, threads);
      continue;
    }
    uint4* ov = reinterpret_cast<uint4*>(out + r.head);
    const int step = ranks * threads;
    for (int i = rank * threads + threadIdx.x; i < r.nvec; i += kFlight * step) {
      uint4 v[kFlight];
#pragma unroll
      for (int j = 0; j < kFlight; ++j) {
        if (i + j * step < r.nvec) v[j] = load_last(r.zv + i + j * step);
      }
#pragma unroll
      for (int j = 0; j < kFlight; ++j) {
        const int n = i + j * step;
        if (n < r.nvec) __stcs(ov + n, g.template vec<T, kEnt>(v[j], r.head + n * VN, tok));
      }
    }
    if (rank == 0 && static_cast<int>(threadIdx.x) < r.head) {
      out[threadIdx.x] = g.template one<T, kEnt>(r.z[threadIdx.x], threadIdx.x, tok);
    }
    const int end = r.tail + static_cast<int>(threadIdx.x);
    if (rank == 0 && end < static_cast<int>(a.vocab)) out[end] = g.template one<T, kEnt>(r.z[end], end, tok);
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
  b.lo = static_cast<float>(k - b.hi);
  b.inv = static_cast<float>(inv_temp);
  b.inv_lack = static_cast<float>(inv_temp - b.inv);
  return b;
}

struct RowLaunch {
  int threads, ranks;
  int64_t clusters;
};

// A launch without clusters says nothing of them: with a cluster dimension of one the kernels above ran up to 2.4 times
// slower for short rows (65,536 rows of 1,024 columns: 168 us against 69).
cudaLaunchConfig_t row_config(const RowLaunch& l, cudaStream_t stream, cudaLaunchAttribute (&attr)[2]) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(l.clusters * l.ranks));
  cfg.blockDim = dim3(static_cast<unsigned>(l.threads));
  cfg.stream = stream;
  cfg.attrs = attr;
  if (l.ranks > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = static_cast<unsigned>(l.ranks);
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  if (pdl_enabled()) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  return cfg;
}

// Clusters of a kernel that fit the device at once (a cluster stays within a group of multiprocessors, so fewer than
// their number suggests; one cluster too many would be a second wave). Asked once per shape and device.
template <typename Kern>
cudaError_t resident_clusters(Kern kern, const RowLaunch& l, int* count) {
  struct Known {
    const void* kern;
    int device, ranks, threads, count;
  };
  static std::mutex lock;
  static std::vector<Known> known;
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const std::lock_guard<std::mutex> guard(lock);
  for (const Known& x : known) {
    if (x.kern == reinterpret_cast<const void*>(kern) && x.device == device && x.ranks == l.ranks && x.threads == l.threads) {
      *count = x.count;
      return cudaSuccess;
    }
  }
  if (l.ranks == 1) {
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(count, kern, l.threads, 0);
    *count *= sm_count();
  } else {
    cudaLaunchAttribute attr[2];
    RowLaunch one = l;
    one.clusters = 1;
    const cudaLaunchConfig_t cfg = row_config(one, nullptr, attr);
    e = cudaOccupancyMaxActiveClusters(count, kern, &cfg);
  }
  if (e != cudaSuccess) return e;
  *count = std::max(*count, 1);
  known.push_back({reinterpret_cast<const void*>(kern), device, l.ranks, l.threads, *count});
  return cudaSuccess;
}

template <typename... KArgs, typename... Args>
cudaError_t launch_rows(void (*kern)(KArgs...), const RowLaunch& l, cudaStream_t stream, Args&&... args) {
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = row_config(l, stream, attr);
  return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}

// Threads of a CTA: eight vectors each, 32 to 256 (four CTAs of 256 hide a row's end behind other rows: 4,094 rows of 50,001
// fp32 columns took 116 us, with 512 threads 126, with 1,024 201).
// CTAs of a row: where rows are few, as many as stay within one wave and leave a thread four vectors or more (fewer are
// not worth the exchange: 1,024 rows of 1,024 bf16 columns 3.4 us unsplit, 12.7 in clusters of 4; 4 rows of 131,072 take
// 4.5 us in clusters of 8). With `again` (the row is read a second time) as many as keep the rows of a wave within
// `kCached` bytes of the 126 MB of L2 (8,192 rows of 131,072 bf16 columns: 893 us at 110 MB, 891 at 80, 931 at 60, 1,111
// at 32, where clusters of 8 wait for each other).
constexpr int64_t kCached = 80 << 20;
RowLaunch row_launch(int64_t rows, int64_t vocab, int size, bool again) {
  const int64_t sms = sm_count(), nvec = vocab * size / 16;
  RowLaunch l;
  l.threads = static_cast<int>(std::min<int64_t>(kMostThreads, std::max<int64_t>(32, (nvec / 8 + 31) / 32 * 32)));
  const int64_t resident = std::min<int64_t>(1024 / l.threads, 32) * sms;
  l.ranks = 1;
  while (l.ranks < kMaxCluster && nvec >= 8 * l.ranks * l.threads) {
    const bool idle = rows * l.ranks * 2 <= resident;
    const bool large = again && std::min(rows, resident / l.ranks) * vocab * size > kCached;
    if (!idle && !large) break;
    l.ranks *= 2;
  }
  l.clusters = std::min(rows, 32 * resident / l.ranks);
  return l;
}

template <typename T>
cudaError_t launch_stats(const TokenStatsArgs& a, cudaStream_t stream) {
  PolicyTerms q{};
  if (a.policy) q = *a.policy;
  return launch_rows(token_stats_kernel<T>, row_launch(a.rows, a.vocab, sizeof(T), false), stream, a, q,
                     a.policy != nullptr, base_of(a.inv_temp));
}

constexpr int kFinishThreads = 1024;
__global__ void __launch_bounds__(kFinishThreads) policy_weights_kernel(const TokenIndex idx, int64_t rows, int64_t vocab,
                                                                        double* out) {
  griddep_wait();  // launched with programmatic stream serialization (launch_pdl)
  griddep_launch_dependents();
  __shared__ double s_sum[kFinishThreads / 32];
  double x[1] = {0.0};
#pragma unroll 4
  for (int64_t r = threadIdx.x; r < rows; r += kFinishThreads) {
    float w;
    row_token(idx, r, vocab, w);
    x[0] += w;
  }
  block_sum(x, s_sum);
  if (threadIdx.x == 0) *out = x[0];
}

// Up to this many rows every CTA sums the weights itself; beyond it one block does so first, for all (whole call, own sum
// against one block's: 1,024 rows of 16,384 columns 21.5 against 22.6 us; 4,096 of 1,024 25.3 against 20.1).
constexpr int64_t kOwnWeights = 1024;

template <typename T>
cudaError_t launch_policy(const TokenStatsArgs& a, const TokenRows& grad, float scale, const float* scale_device, int mean,
                          double* weight_sum, cudaStream_t stream) {
  const PolicyTerms q = *a.policy;
  const auto kern = q.entropy_coef != 0.f ? token_policy_kernel<T, true> : token_policy_kernel<T, false>;
  RowLaunch l = row_launch(a.rows, a.vocab, sizeof(T), true);
  int resident = 0;
  cudaError_t e = resident_clusters(kern, l, &resident);
  if (e != cudaSuccess) return e;
  l.clusters = std::min<int64_t>(a.rows, resident);
  if (!mean || a.rows <= kOwnWeights) weight_sum = nullptr;
  if (weight_sum != nullptr) {
    e = launch_pdl(policy_weights_kernel, dim3(1), dim3(kFinishThreads), 0, stream, a.idx, a.rows, a.vocab, weight_sum);
    if (e != cudaSuccess) return e;
  }
  return launch_rows(kern, l, stream, a, q, grad, scale, scale_device, mean, static_cast<const double*>(weight_sum),
                     base_of(a.inv_temp));
}

// ---- gradient of the logits from the row statistics -----------------------------------------------------------------------
constexpr int kGradThreads = 256;
constexpr int kGradVecs = 8;  // vectors per thread

// A block writes one row's segment of 16-byte vectors. Rows run backwards: the last ones that the statistics read are
// still in L2. Bound by memory: 268 MB read and written in 84 us (6.4 TB/s, 98 % of the copy rate).
template <typename T, bool kEnt>
__global__ void __launch_bounds__(kGradThreads) token_grad_kernel(const TokenGradArgs a, int segs, const Base k) {
  griddep_wait();  // launched with programmatic stream serialization (launch_pdl)
  griddep_launch_dependents();
  constexpr int VN = Elem<T>::kPerVec;
  const int64_t row = a.rows - 1 - blockIdx.x / segs;
  const int seg = static_cast<int>(blockIdx.x % segs);
  T* out = row_ptr<T>(a.out, row);
  float w;
  const int tok = static_cast<int>(row_token(a.idx, row, a.vocab, w));
  const RowView<T> o(out, a.vocab);
  uint4* ov = reinterpret_cast<uint4*>(out + o.head);
  const int v0 = seg * (kGradThreads * kGradVecs) + threadIdx.x, v1 = min(o.nvec, (seg + 1) * (kGradThreads * kGradVecs));
  const int end = o.tail + static_cast<int>(threadIdx.x);
  float ca = 0.f, cb = 0.f;
  if (tok >= 0) {
    float f = static_cast<float>(a.scale * a.inv_temp);
    if (a.scale_a) f *= *a.scale_a;
    if (a.scale_b) f *= *a.scale_b;
    ca = a.a[row * a.a_stride] * f;
    if (kEnt) cb = a.b[row * a.b_stride] * f;
  }
  if (tok < 0 || (ca == 0.f && (!kEnt || cb == 0.f))) {  // nothing to read
    for (int i = v0; i < v1; i += kGradThreads) __stcs(ov + i, make_uint4(0u, 0u, 0u, 0u));
    if (seg == 0 && static_cast<int>(threadIdx.x) < o.head) out[threadIdx.x] = Elem<T>::put(0.f);
    if (seg == 0 && end < static_cast<int>(a.vocab)) out[end] = Elem<T>::put(0.f);
    return;
  }
  const T* z = row_ptr<const T>(a.z, row);
  const RowGrad g(a.ml[row], k, ca, cb, kEnt ? a.entropy[row] : 0.f);
  if (seg == 0 && static_cast<int>(threadIdx.x) < o.head) {
    out[threadIdx.x] = g.template one<T, kEnt>(z[threadIdx.x], threadIdx.x, tok);
  }
  if (seg == 0 && end < static_cast<int>(a.vocab)) out[end] = g.template one<T, kEnt>(z[end], end, tok);
  const bool same = ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
  if (same) {
    const uint4* zv = reinterpret_cast<const uint4*>(z + o.head);
    uint4 v[kGradVecs];
#pragma unroll
    for (int j = 0; j < kGradVecs; ++j) {
      if (v0 + j * kGradThreads < v1) v[j] = __ldg(zv + v0 + j * kGradThreads);
    }
#pragma unroll
    for (int j = 0; j < kGradVecs; ++j) {
      const int i = v0 + j * kGradThreads;
      if (i < v1) __stcs(ov + i, g.template vec<T, kEnt>(v[j], o.head + i * VN, tok));
    }
  } else {  // rows of input and output start at different places within 16 bytes
    for (int i = v0; i < v1; i += kGradThreads) {
      const int col = o.head + i * VN;
      float x[VN];
#pragma unroll
      for (int e = 0; e < VN; ++e) x[e] = Elem<T>::get(z[col + e]);
      __stcs(ov + i, g.template vec<T, kEnt>(Elem<T>::pack(x), col, tok));
    }
  }
}

template <typename T>
cudaError_t launch_grad(const TokenGradArgs& a, cudaStream_t stream) {
  constexpr int64_t per = static_cast<int64_t>(kGradThreads) * kGradVecs * Elem<T>::kPerVec;
  const int64_t segs = std::max<int64_t>(1, (a.vocab + per - 1) / per);
  const dim3 grid(static_cast<unsigned>(a.rows * segs));
  const Base k = base_of(a.inv_temp);
  const int n = static_cast<int>(segs);
  if (a.b) return launch_pdl(token_grad_kernel<T, true>, grid, dim3(kGradThreads), 0, stream, a, n, k);
  return launch_pdl(token_grad_kernel<T, false>, grid, dim3(kGradThreads), 0, stream, a, n, k);
}

// ---- sums over rows, sequences and pairs -----------------------------------------------------------------------------------
__global__ void __launch_bounds__(kFinishThreads) policy_finish_kernel(const PolicyFinishArgs a) {
  griddep_wait();  // launched with programmatic stream serialization (launch_pdl)
  griddep_launch_dependents();
  __shared__ double s_sum[kFinishThreads / 32 * 5];
  double x[5] = {0.0, 0.0, 0.0, 0.0, 0.0};
  constexpr int kRows = 4;  // in flight per thread
  for (int64_t r0 = threadIdx.x; r0 < a.rows; r0 += kRows * kFinishThreads) {
    float4 t[kRows];
    float w[kRows];
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      const int64_t r = r0 + j * kFinishThreads;
      t[j] = make_float4(0.f, 0.f, 0.f, 0.f), w[j] = 0.f;
      if (r < a.rows) {
        t[j] = a.terms[r];
        row_token(a.idx, r, a.vocab, w[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < kRows; ++j) x[0] += t[j].x, x[1] += t[j].y, x[2] += t[j].z, x[3] += t[j].w, x[4] += w[j];
  }
  block_sum(x, s_sum);
  if (threadIdx.x == 0) {
    const double inv = x[4] != 0.0 ? 1.0 / x[4] : 0.0;  // no row counts: loss and gradients are zero
    const double f = a.mean ? inv : 1.0;
    const double kl = a.kl_coef != 0.f ? a.kl_coef * x[1] : 0.0;  // a divergence without a weight may be infinite
    a.loss[0] = static_cast<float>(f * (x[0] + kl - a.entropy_coef * x[2]));
    for (int n = 0; n < 4; ++n) a.out[n] = static_cast<float>(inv * x[n]);
    a.out[4] = static_cast<float>(f);
  }
}

__device__ __forceinline__ int64_t seq_start(const PreferenceArgs& a, int64_t s) {
  int64_t o = a.offsets == nullptr ? s * a.length
              : a.offsets_i64      ? static_cast<const int64_t*>(a.offsets)[s]
                                   : static_cast<int64_t>(static_cast<const int32_t*>(a.offsets)[s]);
  return min(max(o, static_cast<int64_t>(0)), a.rows);
}

// -log sigmoid(x)
__device__ __forceinline__ float softplus_neg(float x) { return log1pf(expf(-fabsf(x))) + fmaxf(-x, 0.f); }

constexpr int kPairThreads = 1024;
// One block, split into teams of threads: a team sums the log-probabilities of a pair's two sequences (in 64 bits, in a
// fixed order), its first thread works out the pair's loss, and the team writes the rows' coefficients. Tens of thousands
// of rows are a few hundred kilobytes, so one block's time stays far below the logits' (8,000 rows: 15 us beside 430).
__global__ void __launch_bounds__(kPairThreads) preference_pairs_kernel(const PreferenceArgs a) {
  griddep_wait();  // launched with programmatic stream serialization (launch_pdl)
  griddep_launch_dependents();
  __shared__ double s_part[kPairThreads / 32][4];
  __shared__ float s_coef[kPairThreads / 32][2];
  __shared__ double s_loss[kPairThreads / 32];
  // Offsets that decrease would give a row to two teams. They are not known to the host, so what they lead to is a NaN.
  int bad = 0;  // looked at where the first pair's sums meet, so that these loads hide behind the rows'
  if (a.offsets != nullptr) {
    for (int64_t s = threadIdx.x; s < a.seqs; s += kPairThreads) bad |= seq_start(a, s + 1) < seq_start(a, s);
  }
  for (int64_t r = threadIdx.x; r < a.rows; r += kPairThreads) a.coef[r] = 0.f;
  const int64_t pairs = a.seqs / 2;
  int teams = 1;
  while (teams < kPairThreads / 32 && teams < pairs) teams *= 2;
  const int size = kPairThreads / teams, team = threadIdx.x / size, t = threadIdx.x % size;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = size / 32;
  double loss = 0.0;
  for (int64_t base = 0; base < pairs; base += teams) {
    const int64_t p = base + team;
    int64_t at[3] = {0, 0, 0};
    double x[4] = {0.0, 0.0, 0.0, 0.0};  // sums and weights of the two sequences
    if (p < pairs) {
      for (int c = 0; c < 3; ++c) at[c] = seq_start(a, 2 * p + c);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        constexpr int kRows = 4;  // in flight per thread
        for (int64_t r0 = at[c] + t; r0 < at[c + 1]; r0 += kRows * size) {
          float logp[kRows], w[kRows];
#pragma unroll
          for (int j = 0; j < kRows; ++j) {
            const int64_t r = r0 + j * size;
            logp[j] = w[j] = 0.f;
            if (r < at[c + 1]) {
              logp[j] = a.logp[r];
              row_token(a.idx, r, a.vocab, w[j]);
            }
          }
#pragma unroll
          for (int j = 0; j < kRows; ++j) {
            if (w[j] == 0.f) continue;
            x[c] += static_cast<double>(w[j]) * logp[j];
            x[2 + c] += w[j];
          }
        }
      }
    }
    for (int n = 0; n < 4; ++n) {
      for (int o = 16; o >= 1; o >>= 1) x[n] += __shfl_xor_sync(0xffffffffu, x[n], o);
    }
    // the rows are cleared, the last pairs' partial sums and coefficients have been read
    if (__syncthreads_or(bad)) {
      const float none = nanf("");
      for (int64_t r = threadIdx.x; r < a.rows; r += kPairThreads) a.coef[r] = none;
      for (int64_t s = threadIdx.x; s < a.seqs; s += kPairThreads) a.seq_logp[s] = a.rewards[s] = none;
      if (threadIdx.x == 0) a.loss[0] = none;
      return;
    }
    if (lane == 0) {
      for (int n = 0; n < 4; ++n) s_part[warp][n] = x[n];
    }
    __syncthreads();
    if (t == 0 && p < pairs) {
      for (int n = 0; n < 4; ++n) {
        x[n] = 0.0;
        for (int i = 0; i < warps; ++i) x[n] += s_part[warp + i][n];
      }
      double lp[2], rew[2];
      for (int c = 0; c < 2; ++c) {
        lp[c] = !a.average ? x[c] : x[2 + c] != 0.0 ? x[c] / x[2 + c] : 0.0;
        rew[c] = a.beta * (lp[c] - (a.ref ? static_cast<double>(a.ref[2 * p + c]) : 0.0));
        a.seq_logp[2 * p + c] = static_cast<float>(lp[c]);
        a.rewards[c * pairs + p] = static_cast<float>(rew[c]);
      }
      const float h = static_cast<float>(rew[0] - rew[1]);
      float l, dh;  // loss of the pair and its derivative by h
      if (a.kind == kPrefSigmoid) {
        l = (1.f - a.smoothing) * softplus_neg(h);
        if (a.smoothing != 0.f) l += a.smoothing * softplus_neg(-h);  // infinite for an infinite h
        dh = a.smoothing / (1.f + expf(-h)) - (1.f - a.smoothing) / (1.f + expf(h));
      } else if (a.kind == kPrefHinge) {
        l = isnan(h) ? h : fmaxf(1.f - h, 0.f);
        dh = h < 1.f ? -1.f : 0.f;
      } else {  // squared distance of the log-ratio difference h / beta from 1 / (2 beta)
        const double d = (rew[0] - rew[1] - 0.5) / a.beta;
        l = static_cast<float>(d * d);
        dh = static_cast<float>(2.0 * d / a.beta);
      }
      loss += l;
      const double g = static_cast<double>(dh) * a.beta / static_cast<double>(pairs);
      for (int c = 0; c < 2; ++c) {
        const double gc = c == 0 ? g : -g;
        s_coef[team][c] = static_cast<float>(!a.average ? gc : x[2 + c] != 0.0 ? gc / x[2 + c] : 0.0);
      }
    }
    __syncthreads();
    if (p < pairs) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float coef = s_coef[team][c];
#pragma unroll 4
        for (int64_t r = at[c] + t; r < at[c + 1]; r += size) {
          float w;
          row_token(a.idx, r, a.vocab, w);
          a.coef[r] = coef * w;
        }
      }
    }
  }
  if (t == 0) s_loss[team] = loss;
  __syncthreads();
  if (threadIdx.x == 0) {
    loss = 0.0;
    for (int i = 0; i < teams; ++i) loss += s_loss[i];
    a.loss[0] = pairs ? static_cast<float>(loss / static_cast<double>(pairs)) : 0.f;
  }
}

}  // namespace

cudaError_t token_stats(const TokenStatsArgs& a, cudaStream_t stream) {
  if (a.rows == 0) return cudaSuccess;
  switch (a.dtype) {
    case kTokF32: return launch_stats<float>(a, stream);
    case kTokBF16: return launch_stats<__nv_bfloat16>(a, stream);
    default: return launch_stats<__half>(a, stream);
  }
}

cudaError_t token_policy(const TokenStatsArgs& a, const TokenRows& grad, float scale, const float* scale_device, int mean,
                         double* weight_sum, cudaStream_t stream) {
  if (a.rows == 0) return cudaSuccess;
  switch (a.dtype) {
    case kTokF32: return launch_policy<float>(a, grad, scale, scale_device, mean, weight_sum, stream);
    case kTokBF16: return launch_policy<__nv_bfloat16>(a, grad, scale, scale_device, mean, weight_sum, stream);
    default: return launch_policy<__half>(a, grad, scale, scale_device, mean, weight_sum, stream);
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
