// Key/value cache in 8 bits: writing tokens into it and decode attention over it (cache_q8_sm100.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <vector>

namespace ft {

enum CacheFormat : int { CACHE_INT8 = 0, CACHE_E4M3 = 1 };

// One side (keys or values) of a cache: codes [B, L, Hk, 128] (one byte each, last dim packed;
// byte strides) and scales [B, ceil(L / block), Hk] fp32 (element strides).
struct CacheSide {
  uint8_t* codes = nullptr;
  long long c_b = 0, c_tok = 0, c_h = 0;
  float* scale = nullptr;
  long long s_b = 0, s_blk = 0, s_h = 0;
};

struct CacheAppendProblem {
  int B = 0, S = 0, Hk = 0, L = 0, block = 64, format = CACHE_INT8;
  const __nv_bfloat16* x[2] = {};          // new keys / values [B, S, Hk, 128]
  long long x_b[2] = {}, x_tok[2] = {}, x_h[2] = {};  // element strides
  CacheSide side[2];                       // keys / values
  const int* pos = nullptr;                // [B] first position of the new tokens; null: pos_all
  int pos_all = 0;
  const int* n_new = nullptr;              // [B] tokens to take of the S; null: all
};
cudaError_t cache_append(const CacheAppendProblem& p, cudaStream_t stream);

struct CacheDecodeProblem {
  int B = 0, Sq = 1, Hq = 0, Hk = 0, L = 0, block = 64, format = CACHE_INT8;
  const __nv_bfloat16* q = nullptr;        // [B, Sq, Hq, 128]
  long long q_b = 0, q_tok = 0, q_h = 0;   // element strides
  __nv_bfloat16* o = nullptr;
  long long o_b = 0, o_tok = 0, o_h = 0;
  CacheSide side[2];
  const int* kv_len = nullptr;             // [B]; null: len_all
  int len_all = 0;
  int max_len = 0;                         // bound of the lengths: a longer one is cut to it
  int later = 0;                           // tokens of each sequence that follow the Sq queries'
  float scale = 1.f;
  int num_sms = 148;
  float* scratch = nullptr;                // cache_decode_scratch_floats(p) floats
};
size_t cache_decode_scratch_floats(const CacheDecodeProblem& p);
// The p.Sq queries of a call in launches whose scratch stays within `most` bytes (where one query's does): their
// numbers of queries, and the scratch that the largest takes. It does not grow with the queries alone: how many
// heads stand side by side depends on what divides their number.
struct CacheDecodePlan {
  std::vector<int> queries;
  size_t scratch_bytes = 0;
};
CacheDecodePlan cache_decode_plan(CacheDecodeProblem p, size_t most);
// two kernels; where no key may count (max_len 0), the second alone
cudaError_t cache_decode(const CacheDecodeProblem& p, cudaStream_t stream);
int cache_device_error(bool reset);

}  // namespace ft
