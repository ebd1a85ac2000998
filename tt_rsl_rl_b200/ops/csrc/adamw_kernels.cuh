// AdamW step over many tensors in one launch, with fp32 states or 8-bit states.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps).
//
// Weights are fp32, or bf16 with the 16 bits of the fp32 weight below its bf16 rounding in a tensor of their own. 8-bit
// states hold e4m3 codes of m and of sqrt(v), one fp32 scale per 256 elements, rounded stochastically.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace rlb {

constexpr int kAdamBlock = 256;  // elements that share a scale

struct AdamTensor {
  void *p, *g;
  void *m, *v;              // fp32, or e4m3 codes with scales
  float *m_scale, *v_scale;
  int16_t* low;             // bf16 weights: the fp32 weight's lower bits
  int64_t n;
  uint32_t id;              // the tensor's place in `steps`, below 65,536
};

struct AdamHyper {
  double lr, beta1, beta2, eps, weight_decay;
  const void* lr_device;  // learning rate on the device instead of `lr`; null: none
  int lr_f64;             // its type: 1 fp64, 0 fp32
  int maximize;
  uint64_t seed;
};

struct AdamLaunch {
  const AdamTensor* tensors;  // host
  int count;
  int bf16, bits8;
  AdamHyper h;
  uint32_t first_stream;  // tensor `id` draws its random numbers from stream first_stream + id
  float* steps;        // [tensors of the plan] steps taken; advanced by one for the tensors of this launch
};
// One step of several lists of tensors. max_norm > 0: every gradient is scaled by min(1, max_norm / (norm + 1e-6)) with
// the norm over all lists, which norm[0] receives.
int64_t adamw_workspace_bytes(const AdamLaunch* lists, int n);
cudaError_t adamw_step(const AdamLaunch* lists, int n, double max_norm, void* workspace, float* norm,
                       cudaStream_t stream);

}  // namespace rlb
