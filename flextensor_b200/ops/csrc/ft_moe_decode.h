// A whole mixture-of-experts feed-forward for a few tokens (moe_decode_sm100.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace ft {

constexpr int kMoeDecMaxTokens = 64;
constexpr int kMoeDecMaxExperts = 128;
constexpr int kMoeDecMaxTopk = 8;

struct MoeDecodeProblem {
  int T = 0, D = 0, F = 0, E = 0, topk = 0;
  const __nv_bfloat16* x = nullptr;       // [T, D]
  long long ldx = 0;
  const __nv_bfloat16* router = nullptr;  // [E, D]
  long long ldr = 0;
  const __nv_bfloat16* w_gate_up[kMoeDecMaxExperts] = {};  // [2F, D] per expert, gate and up rows interleaved
  const __nv_bfloat16* w_down[kMoeDecMaxExperts] = {};     // [D, F] per expert
  long long ld_gate_up = 0, ld_down = 0;  // row strides (elements), the same for every expert
  const __nv_bfloat16* residual = nullptr;
  long long ldres = 0;
  __nv_bfloat16* out = nullptr;           // [T, D], may be the residual
  long long ldo = 0;
  int num_sms = 148;
  void* workspace = nullptr;              // moe_decode_workspace(p) bytes, 256-byte aligned
};
size_t moe_decode_workspace(const MoeDecodeProblem& p);
// Whether one tensor map serves all experts: their weights lie at equal distances that a map can hold (a
// multiple of 16 bytes below 2^40). Else each has a map of its own.
bool moe_decode_one_map(const __nv_bfloat16* const* w, int E);
// four kernels
cudaError_t moe_decode(const MoeDecodeProblem& p, cudaStream_t stream);
int moe_decode_device_error(bool reset);

}  // namespace ft
