// Key/value cache in 8 bits with one scale per block of tokens and head: writing tokens into it
// and decode attention over it, head_dim 128, for sm_100a.
//
// Writing. A block's scale is the smallest power of two s with max|x| <= qmax * s (qmax 127 for
// int8, 448 for e4m3), so x / s is exact and a code depends on the value alone; a block that
// already holds tokens keeps the larger of its old scale and the new tokens', and its old codes
// are rounded again when the scale grew. The largest magnitude is found on the bf16 bit patterns
// (sign cleared, as 16-bit integers): NaN and infinity compare above every finite value, and a
// block that received one gets the scale NaN, which reaches every output that reads the block.
//
// Decode attention. Per cached token and KV head 256 code bytes are read once and each takes part
// in 2 * G * Sq multiply-adds, so the kernel is bound by HBM. The codes go to f16 in registers
// (exact for both formats) and the products run as warp-level m16n8k16 MMAs with the *keys* on the
// 16-row side and the query rows (heads of one KV group x query tokens) on the 8-column side:
//   S^T[key, row] = K q^T,   O^T[dim, row] += V^T P^T.
// Eight rows are one column tile, so a group of 8 heads wastes no MMA work. Which physical
// dimension or key a fragment slot stands for is free as long as both operands agree, so every
// lane takes its fragments from 16-byte pieces of the cache rows as they lie in memory:
//   K: lane (g, c) holds rows g and g + 8 of a 16-key tile, dims 32c .. 32c+31;
//   V: lane (g, c) holds rows 2c, 2c+1, 2c+8, 2c+9, dims 16g .. 16g+15; two rows' bytes are
//      interleaved with PRMT into the (key, key+1) pairs the MMA wants.
// P goes from the accumulator layout to the B operand with one 8x8 transpose per 8 keys.
//
// Work. All (sequence, KV head, row group) units form one sequence of 32-key tiles, divided into
// equal contiguous runs, one per warp (8 warps an SM), so ragged batches and few long sequences load
// every SM alike. A warp streams its run by itself through its own three 8 KB stages (TMA, 128-byte
// swizzle; the warp's own program order says when a stage is free, so there is no producer and no
// barrier between warps) and writes fp32 partial results at unit ends; a second kernel, launched
// so that its start overlaps the first one's end, merges the partials of each row in run order.
//
// Scales: a score is (q . codes) * ks, and the weight of a value's codes is p * vs. The running
// reference m is the maximum of score + log2(vs), so p * vs <= 1 whatever the scales are and f16
// holds it to 2^-11 of the largest weight; the sum l takes p itself in fp32. q is scaled by a power
// of two per row into f16 (exact but for elements below 2^-24 of the row's largest).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "ft_cache.h"
#include "ft_ops.h"
#include "sm100_common.cuh"

namespace ft {

FT_DEFINE_ERROR_READER(cache_device_error)

namespace {

constexpr int HD = 128;  // head dim

// ------------------------------------------------------------------------------------ writing
struct AppendArgs {
  int B, S, Hk, L, n_rel;
  const __nv_bfloat16* x[2];
  long long x_b[2], x_tok[2], x_h[2];
  CacheSide side[2];
  const int* pos;
  int pos_all;
  const int* n_new;
};

// smallest power of two s with a <= qmax * s, for a bf16 magnitude given by its bits
template <int FMT>
__device__ __forceinline__ float pow2_scale(uint32_t bits) {
  if (bits >= 0x7f80u) return __int_as_float(0x7fc00000);
  if (bits == 0u) return 0.f;
  // a = (1/2 + man/256) 2^e; qmax = 254/256 * 2^7 (int8), 224/256 * 2^9 (e4m3)
  const int man = bits & 0x7f, e = (int)(bits >> 7) - 126;
  const int k = FMT == CACHE_INT8 ? e - 7 + (man > 126) : e - 9 + (man > 96);
  return __int_as_float((max(k, -120) + 127) << 23);
}

template <int FMT>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  if (FMT == CACHE_INT8) {
    const int ia = min(127, max(-127, __float2int_rn(a))), ib = min(127, max(-127, __float2int_rn(b)));
    const int ic = min(127, max(-127, __float2int_rn(c))), id = min(127, max(-127, __float2int_rn(d)));
    return __byte_perm(__byte_perm(ia, ib, 0x0040), __byte_perm(ic, id, 0x0040), 0x5410);
  }
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

// four codes of a word rounded again under a scale grown by 1 / ratio
template <int FMT>
__device__ __forceinline__ uint32_t recode4(uint32_t w, float ratio) {
  float f[4];
  if (FMT == CACHE_INT8) {
#pragma unroll
    for (int i = 0; i < 4; i++) f[i] = (float)(int8_t)(w >> (8 * i));
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) f[i] = __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)(w >> (8 * i)), __NV_E4M3)));
  }
  return encode4<FMT>(f[0] * ratio, f[1] * ratio, f[2] * ratio, f[3] * ratio);
}

// One CTA per (sequence, block of tokens, KV head, keys or values); the block's new tokens are
// held in registers between the maximum and the rounding, so they are read once.
template <int BLOCK, int FMT>
__global__ void __launch_bounds__(BLOCK <= 64 ? 128 : 256) cache_append_kernel(AppendArgs a) {
  constexpr int THREADS = BLOCK <= 64 ? 128 : 256;
  constexpr int ROWS = THREADS / 16;  // token rows per pass: 16 lanes hold a row's 128 values
  constexpr int ITERS = BLOCK / ROWS;
  __shared__ uint32_t warp_max[THREADS / 32];
  long long id = blockIdx.x;
  const int h = (int)(id % a.Hk);
  id /= a.Hk;
  const int rel = (int)(id % a.n_rel);
  id /= a.n_rel;
  const int kv = (int)(id & 1), b = (int)(id >> 1);
  const int p = a.pos ? a.pos[b] : a.pos_all, n = a.n_new ? a.n_new[b] : a.S;
  if (p < 0 || n < 0 || n > a.S || p > a.L - n) {  // nothing of such a sequence is written
    if (threadIdx.x == 0) record_error(kErrBadArgs);
    return;
  }
  const int j = p / BLOCK + rel;
  const int t0 = max(p, j * BLOCK), t1 = min(p + n, (j + 1) * BLOCK);
  if (t0 >= t1) return;
  const CacheSide& sd = a.side[kv];
  float* const sp = sd.scale + b * sd.s_b + j * sd.s_blk + h * sd.s_h;
  const bool history = t0 > j * BLOCK;
  const float s_old = history ? *sp : 0.f;
  const int row0 = threadIdx.x / 16, col = (threadIdx.x % 16) * 8;
  const __nv_bfloat16* const x = a.x[kv] + b * a.x_b[kv] + h * a.x_h[kv] + col;
  uint4 v[ITERS];
  uint32_t m2 = 0;
#pragma unroll
  for (int i = 0; i < ITERS; i++) {
    const int t = j * BLOCK + i * ROWS + row0;
    v[i] = make_uint4(0, 0, 0, 0);
    if (t >= t0 && t < t1) v[i] = __ldg(reinterpret_cast<const uint4*>(x + (long long)(t - p) * a.x_tok[kv]));
  }
#pragma unroll
  for (int i = 0; i < ITERS; i++) {
    m2 = __vmaxu2(m2, __vmaxu2(__vmaxu2(v[i].x & 0x7fff7fffu, v[i].y & 0x7fff7fffu),
                               __vmaxu2(v[i].z & 0x7fff7fffu, v[i].w & 0x7fff7fffu)));
  }
  uint32_t m = __reduce_max_sync(0xffffffffu, max(m2 & 0xffffu, m2 >> 16));
  if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
  __syncthreads();  // also: every thread has read the old scale
#pragma unroll
  for (int w = 0; w < THREADS / 32; w++) m = max(m, warp_max[w]);
  const float s_new = pow2_scale<FMT>(m);
  const float s = s_old != s_old ? s_old : (s_new != s_new ? s_new : fmaxf(s_old, s_new));
  const bool bad = s != s;
  const float inv = bad ? 0.f : (s > 0.f ? 1.f / s : 0.f);
  uint8_t* const out = sd.codes + b * sd.c_b + h * sd.c_h + col;
  if (history && s != s_old) {
    const float ratio = bad ? 0.f : s_old * inv;
    for (int t = j * BLOCK + row0; t < t0; t += ROWS) {
      uint2* const w = reinterpret_cast<uint2*>(out + (long long)t * sd.c_tok);
      const uint2 o = *w;
      *w = bad ? make_uint2(0, 0) : make_uint2(recode4<FMT>(o.x, ratio), recode4<FMT>(o.y, ratio));
    }
  }
  if (threadIdx.x == 0) *sp = s;
#pragma unroll
  for (int i = 0; i < ITERS; i++) {
    const int t = j * BLOCK + i * ROWS + row0;
    if (t < t0 || t >= t1) continue;
    const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
    float f[8];
#pragma unroll
    for (int e = 0; e < 4; e++) {
      f[2 * e] = __uint_as_float(w[e] << 16) * inv;
      f[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u) * inv;
    }
    uint2 o = make_uint2(encode4<FMT>(f[0], f[1], f[2], f[3]), encode4<FMT>(f[4], f[5], f[6], f[7]));
    if (bad) o = make_uint2(0, 0);
    *reinterpret_cast<uint2*>(out + (long long)t * sd.c_tok) = o;
  }
}

template <int BLOCK>
cudaError_t launch_append(const AppendArgs& a, int format, cudaStream_t stream) {
  const long long grid = (long long)a.B * 2 * a.n_rel * a.Hk;
  if (grid > 0x7fffffffLL) return cudaErrorInvalidValue;
  const int threads = BLOCK <= 64 ? 128 : 256;
  if (format == CACHE_INT8) cache_append_kernel<BLOCK, CACHE_INT8><<<(unsigned)grid, threads, 0, stream>>>(a);
  else cache_append_kernel<BLOCK, CACHE_E4M3><<<(unsigned)grid, threads, 0, stream>>>(a);
  return cudaGetLastError();
}

// ------------------------------------------------------------------------------------ attention
constexpr int KT = 32;       // keys of a tile
constexpr int NWARP = 8;
constexpr int STAGES = 3;    // per warp
constexpr int SIDE_BYTES = KT * HD;
constexpr int STAGE_BYTES = 2 * SIDE_BYTES;  // keys, values
constexpr int MERGE_WARPS = 8;

struct DecArgs {
  int B, Sq, Hq, Hk, L, G, R, n_group;  // R = Sq * G query rows of a KV head in n_group groups of 8 * NT
  int block_shift;
  int runs;                             // warps that may take a run
  const __nv_bfloat16* q;
  long long q_b, q_tok, q_h;
  __nv_bfloat16* o;
  long long o_b, o_tok, o_h;
  CacheSide k, v;
  int one_b[2], one_h[2];               // keys / values: the cache is broadcast over sequences / heads (stride 0)
  const int* kv_len;
  int len_all, max_len;
  float scale_log2;                     // softmax scale * log2(e)
  float* part_o;                        // [units + runs][8 * NT][128]
  float2* part_ml;                      // [units + runs][8 * NT] reference and sum
  int merge_per_row;                    // warps that share a row of the merge
};

__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2f(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// maximum that keeps a NaN (fmaxf drops it): a NaN score has to reach its row's output
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// D += A(16x16, row) * B(16x8, col), f16 inputs, fp32 accumulators
__device__ __forceinline__ void mma16816_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Codes (bytes 0, 1) and (bytes 2, 3) of a word as two f16 pairs. int8: a byte with its sign bit
// flipped is u = code + 128, and 0x6400 | u is the f16 number 1024 + u, so one subtraction of 1152
// gives the code exactly.
template <int FMT>
__device__ __forceinline__ void decode4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (FMT == CACHE_INT8) {
    const uint32_t u = w ^ 0x80808080u;
    const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
    uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    __half2 ha = __hsub2(*reinterpret_cast<__half2*>(&a), off), hb = __hsub2(*reinterpret_cast<__half2*>(&b), off);
    lo = *reinterpret_cast<uint32_t*>(&ha);
    hi = *reinterpret_cast<uint32_t*>(&hb);
  } else {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(w));
  }
}

// The queries of a warp's 8 * NT rows as B operands. Row r of the KV head is query token r / G,
// head h * G + r % G; rows at or past R are zero.
template <int NT>
struct QueryFrag {
  uint32_t b[NT][8][2];
  float fac[NT][2];  // score factor of accumulator columns 2c, 2c+1: softmax scale * log2(e) / the row's power of two
  int row[NT][2];    // rows of those columns
};

template <int NT>
__device__ __forceinline__ void load_queries(QueryFrag<NT>& f, const DecArgs& a, int b, int h, int row0, int lane) {
  const int g = lane >> 2, c = lane & 3;
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    const int r = row0 + nt * 8 + g;
    uint4 w[4] = {};
    if (r < a.R) {
      const uint4* p = reinterpret_cast<const uint4*>(a.q + b * a.q_b + (long long)(r / a.G) * a.q_tok +
                                                      (long long)(h * a.G + r % a.G) * a.q_h + 32 * c);
#pragma unroll
      for (int i = 0; i < 4; i++) w[i] = p[i];
    }
    const uint32_t* x = reinterpret_cast<const uint32_t*>(w);
    uint32_t m2 = 0;
#pragma unroll
    for (int i = 0; i < 16; i++) m2 = __vmaxu2(m2, x[i] & 0x7fff7fffu);
    uint32_t m = max(m2 & 0xffffu, m2 >> 16);
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    // bring the row's largest magnitude to 1 .. 4 by a power of two whose inverse is a normal
    // number too; a row with NaN or infinity stays as it is
    const int e = m >= 0x7f80u ? 0 : min(126, max(-126, (int)(m >> 7) - 127));
    const float up = __int_as_float((127 - e) << 23), down = __int_as_float((127 + e) << 23);
#pragma unroll
    for (int j = 0; j < 8; j++) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const uint32_t y = x[2 * j + i];
        __half2 hh = __floats2half2_rn(__uint_as_float(y << 16) * up, __uint_as_float(y & 0xffff0000u) * up);
        f.b[nt][j][i] = *reinterpret_cast<uint32_t*>(&hh);
      }
    }
    // the factors of columns 2c, 2c+1 live in the lanes of rows g = 2c, 2c+1
#pragma unroll
    for (int i = 0; i < 2; i++) {
      f.fac[nt][i] = __shfl_sync(0xffffffffu, down, (2 * c + i) * 4) * a.scale_log2;
      f.row[nt][i] = row0 + nt * 8 + 2 * c + i;
    }
  }
}

// Running softmax of a warp: accumulators O^T (dims 16g + 2j (+1) x columns 2c (+1)), reference m
// and this lane's part of the sum for the two columns.
template <int NT>
struct RowState {
  float o[8][NT][4];
  float m[NT][2], l[NT][2];
};

// One tile of KT keys: `kt`/`vt` give 16-byte pieces (row, piece) of the tile's codes, `lim` the
// number of keys of the tile that each column sees (KT or more: all).
template <int NT, int FMT, class KLoad, class VLoad>
__device__ __forceinline__ void attend_tile(RowState<NT>& st, const QueryFrag<NT>& qf, KLoad kt, VLoad vt,
                                            const float (&ks)[KT / 16], const float (&vs)[KT / 16],
                                            const int (&lim)[NT][2], bool masked, int lane) {
  const int g = lane >> 2, c = lane & 3;
  constexpr int MT = KT / 16;
  float s[MT][NT][4];
#pragma unroll
  for (int mt = 0; mt < MT; mt++) {
#pragma unroll
    for (int nt = 0; nt < NT; nt++) s[mt][nt][0] = s[mt][nt][1] = s[mt][nt][2] = s[mt][nt][3] = 0.f;
#pragma unroll
    for (int hh = 0; hh < 2; hh++) {
      const uint4 x = kt(mt * 16 + g, 2 * c + hh), y = kt(mt * 16 + g + 8, 2 * c + hh);
      const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int w = 0; w < 4; w++) {
        uint32_t a0, a1, a2, a3;
        decode4<FMT>(xw[w], a0, a2);
        decode4<FMT>(yw[w], a1, a3);
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
          mma16816_f16(s[mt][nt], a0, a1, a2, a3, qf.b[nt][hh * 4 + w][0], qf.b[nt][hh * 4 + w][1]);
      }
    }
  }
  float lv[MT];
#pragma unroll
  for (int mt = 0; mt < MT; mt++) lv[mt] = lg2f(fmaxf(vs[mt], 0x1p-100f));
  uint32_t pb[MT][NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        float z = s[mt][nt][e] * (ks[mt] * qf.fac[nt][e & 1]);
        if (masked && mt * 16 + g + 8 * (e >> 1) >= lim[nt][e & 1]) z = -INFINITY;
        s[mt][nt][e] = z;
        top[e & 1] = max_nan(top[e & 1], z + lv[mt]);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
      top[i] = max_nan(top[i], __shfl_xor_sync(0xffffffffu, top[i], 4));
      top[i] = max_nan(top[i], __shfl_xor_sync(0xffffffffu, top[i], 8));
      top[i] = max_nan(top[i], __shfl_xor_sync(0xffffffffu, top[i], 16));
      const float m_new = max_nan(st.m[nt][i], top[i]);
      const float ref = m_new == -INFINITY ? 0.f : m_new;
      const float al = st.m[nt][i] == -INFINITY ? 0.f : ex2f(st.m[nt][i] - ref);
      st.m[nt][i] = m_new;
      st.l[nt][i] *= al;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        st.o[j][nt][i] *= al;
        st.o[j][nt][2 + i] *= al;
      }
      top[i] = ref;
    }
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
      float w[4];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const float p = ex2f(s[mt][nt][e] - top[e & 1]);
        st.l[nt][e & 1] += p;
        // a key that the column does not see weighs exactly 0, whatever its block's scale
        w[e] = masked && mt * 16 + g + 8 * (e >> 1) >= lim[nt][e & 1] ? 0.f : p * vs[mt];
      }
      __half2 h0 = __floats2half2_rn(w[0], w[1]), h1 = __floats2half2_rn(w[2], w[3]);
      pb[mt][nt][0] = transpose8x8(*reinterpret_cast<uint32_t*>(&h0));
      pb[mt][nt][1] = transpose8x8(*reinterpret_cast<uint32_t*>(&h1));
    }
  }
#pragma unroll
  for (int mt = 0; mt < MT; mt++) {
    const uint4 v0 = vt(mt * 16 + 2 * c, g), v1 = vt(mt * 16 + 2 * c + 1, g);
    const uint4 v2 = vt(mt * 16 + 2 * c + 8, g), v3 = vt(mt * 16 + 2 * c + 9, g);
    const uint32_t w0[4] = {v0.x, v0.y, v0.z, v0.w}, w1[4] = {v1.x, v1.y, v1.z, v1.w};
    const uint32_t w2[4] = {v2.x, v2.y, v2.z, v2.w}, w3[4] = {v3.x, v3.y, v3.z, v3.w};
#pragma unroll
    for (int w = 0; w < 4; w++) {
      uint32_t a0, a1, a2, a3, b0, b1, b2, b3;
      decode4<FMT>(__byte_perm(w0[w], w1[w], 0x5140), a0, a1);
      decode4<FMT>(__byte_perm(w2[w], w3[w], 0x5140), a2, a3);
      decode4<FMT>(__byte_perm(w0[w], w1[w], 0x7362), b0, b1);
      decode4<FMT>(__byte_perm(w2[w], w3[w], 0x7362), b2, b3);
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        mma16816_f16(st.o[2 * w][nt], a0, a1, a2, a3, pb[mt][nt][0], pb[mt][nt][1]);
        mma16816_f16(st.o[2 * w + 1][nt], b0, b1, b2, b3, pb[mt][nt][0], pb[mt][nt][1]);
      }
    }
  }
}

__device__ __forceinline__ int seq_len(const DecArgs& a, int b) {
  return max(0, min(a.kv_len ? __ldg(a.kv_len + b) : a.len_all, a.max_len));
}
__device__ __forceinline__ int seq_tiles(const DecArgs& a, int b) { return (seq_len(a, b) + KT - 1) / KT; }

// sum of the tiles of sequences [0, end) of one KV head and row group, by a whole warp
__device__ __forceinline__ long long tiles_before(const DecArgs& a, int end, int lane) {
  if (a.kv_len == nullptr) return (long long)end * seq_tiles(a, 0);
  long long sum = 0;
  for (int b = lane; b < end; b += 32) sum += seq_tiles(a, b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}

// The sequence of tiles and its division into runs.
struct Runs {
  long long total;
  int n;
  __device__ __forceinline__ Runs(long long t, int most) : total(t), n((int)min((long long)most, t)) {}
  __device__ __forceinline__ long long begin(int r) const { return total * r / n; }
  __device__ __forceinline__ int owner(long long i) const { return (int)(((i + 1) * n - 1) / total); }
};

// A place in the sequence of tiles.
struct Cursor {
  int b, hg, t, n;  // sequence, head * n_group + group, tile of the unit, tiles of a unit of this sequence
  __device__ __forceinline__ void next(const DecArgs& a) {
    if (++t < n) return;
    t = 0;
    if (++hg < a.Hk * a.n_group) return;
    hg = 0;
    do {
      if (++b >= a.B) return;
      n = seq_tiles(a, b);
    } while (n == 0);
  }
};

// the place of tile i, by a whole warp
__device__ __forceinline__ Cursor locate(const DecArgs& a, long long i, int lane) {
  Cursor c;
  const int per = a.Hk * a.n_group;
  if (a.kv_len == nullptr) {
    c.n = seq_tiles(a, 0);
    c.b = (int)(i / ((long long)c.n * per));
    i -= (long long)c.b * c.n * per;
  } else {
    long long before = 0;
    for (int b0 = 0;; b0 += 32) {  // i lies before the total, so some sequence holds it
      const int n = b0 + lane < a.B ? seq_tiles(a, b0 + lane) : 0;
      long long end = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, end, o);
        if (lane >= o) end += up;
      }
      const unsigned int hit = __ballot_sync(0xffffffffu, (before + end) * per > i);
      if (hit || b0 + 32 >= a.B) {
        const int at = hit ? __ffs(hit) - 1 : 31;
        c.b = b0 + at;
        c.n = __shfl_sync(0xffffffffu, n, at);
        i -= (before + __shfl_sync(0xffffffffu, end - n, at)) * per;
        break;
      }
      before += __shfl_sync(0xffffffffu, end, 31);
    }
  }
  c.hg = (int)(i / c.n);
  c.t = (int)(i % c.n);
  return c;
}

__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ void tma_load_4d(void* dst, const void* tmap, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

// A wait that runs out (2 s) is recorded and answered with false.
__device__ __forceinline__ bool bounded_wait(uint64_t* bar, uint32_t phase) {
  const uint32_t a = smem_u32(bar);
  if (mbar_try_wait(a, phase)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait(a, phase)) {
    if ((unsigned long long)(clock64() - t0) > FT_WAIT_LIMIT_CYCLES) {
      record_error(kErrWaitTimeout);
      return false;
    }
  }
  return true;
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}

struct DecSmem {
  uint8_t stage[NWARP][STAGES][STAGE_BYTES];
  uint64_t full[NWARP][STAGES];
};

struct TileScales {
  float k[KT / 16], v[KT / 16];
};

// 16 keys never straddle a block; a tile's tail past the length takes the last block's scale
__device__ __forceinline__ TileScales load_scales(const DecArgs& a, const Cursor& c) {
  TileScales s;
  const int h = c.hg / a.n_group, last = seq_len(a, c.b) - 1;
#pragma unroll
  for (int i = 0; i < KT / 16; i++) {
    const long long blk = min(c.t * KT + 16 * i, last) >> a.block_shift;
    s.k[i] = __ldg(a.k.scale + c.b * a.k.s_b + blk * a.k.s_blk + h * a.k.s_h);
    s.v[i] = __ldg(a.v.scale + c.b * a.v.s_b + blk * a.v.s_blk + h * a.v.s_h);
  }
  return s;
}

template <int NT, int FMT>
__global__ void __launch_bounds__(32 * NWARP, 1)
    cache_decode_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, DecArgs a) {
  extern __shared__ uint8_t smem_raw[];
  DecSmem& sm = *reinterpret_cast<DecSmem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  pdl_launch();
  const Runs runs(tiles_before(a, a.B, lane) * a.Hk * a.n_group, a.runs);
  const int run = warp * gridDim.x + blockIdx.x;  // neighbouring runs on different SMs: few runs spread out
  if (run >= runs.n) return;
  const long long first = runs.begin(run);
  const int n = (int)(runs.begin(run + 1) - first);
  uint64_t* const full = sm.full[warp];
  if (lane == 0) {
    for (int s = 0; s < STAGES; s++) mbar_init(&full[s], 1);
    fence_barrier_init();
  }
  __syncwarp();
  Cursor at = locate(a, first, lane), ahead = at;
  auto fetch = [&](int s) {  // one lane: the tile at `ahead` into stage s
    const int h = ahead.hg / a.n_group, key0 = ahead.t * KT;
    uint8_t* const dst = sm.stage[warp][s];
    mbar_arrive_expect_tx(&full[s], STAGE_BYTES);
    tma_load_4d(dst, &tm_k, &full[s], 0, a.one_h[0] ? 0 : h, key0, a.one_b[0] ? 0 : ahead.b);
    tma_load_4d(dst + SIDE_BYTES, &tm_v, &full[s], 0, a.one_h[1] ? 0 : h, key0, a.one_b[1] ? 0 : ahead.b);
  };
  for (int s = 0; s < STAGES && s < n; s++) {
    if (lane == 0) fetch(s);
    ahead.next(a);
  }
  QueryFrag<NT> qf;
  RowState<NT> st;
  int sees[NT][2], len = 0;
  auto enter = [&]() {  // a new unit: its queries, empty accumulators
    len = seq_len(a, at.b);
    load_queries<NT>(qf, a, at.b, at.hg / a.n_group, at.hg % a.n_group * 8 * NT, lane);
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        st.m[nt][i] = -INFINITY;
        st.l[nt][i] = 0.f;
        sees[nt][i] = len - a.Sq + 1 + min(qf.row[nt][i], a.R - 1) / a.G;
#pragma unroll
        for (int j = 0; j < 8; j++) st.o[j][nt][i] = st.o[j][nt][2 + i] = 0.f;
      }
    }
  };
  enter();
  TileScales sc = load_scales(a, at);
  bool ok = true;
  int s = 0;
  uint32_t ph = 0;
  for (int i = 0; i < n; i++) {
    Cursor then = at;
    then.next(a);
    const TileScales sc_next = i + 1 < n ? load_scales(a, then) : sc;
    if (ok) ok = __all_sync(0xffffffffu, bounded_wait(&full[s], ph));
    if (ok) {
      const int key0 = at.t * KT;
      const uint32_t kb = smem_u32(sm.stage[warp][s]), vb = kb + SIDE_BYTES;
      int lim[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; nt++) lim[nt][0] = sees[nt][0] - key0, lim[nt][1] = sees[nt][1] - key0;
      const bool masked = key0 + KT > len - a.Sq + 1;
      const int valid = len - key0;
      auto kt = [&](int r, int piece) { return lds128(kb + r * 128 + ((piece ^ (r & 7)) << 4)); };
      auto vt = [&](int r, int piece) {
        uint4 v = lds128(vb + r * 128 + ((piece ^ (r & 7)) << 4));
        // e4m3 bytes past the length may be NaN codes, which a weight of 0 would not cancel
        if (FMT == CACHE_E4M3 && r >= valid) v = make_uint4(0, 0, 0, 0);
        return v;
      };
      attend_tile<NT, FMT>(st, qf, kt, vt, sc.k, sc.v, lim, masked, lane);
      __syncwarp();  // every lane has read the stage
      if (i + STAGES < n) {
        if (lane == 0) fetch(s);
        ahead.next(a);
      }
    }
    if (++s == STAGES) {
      s = 0;
      ph ^= 1;
    }
    if (i + 1 == n || then.t == 0) {  // the unit, or this run's part of it, ends here
      // u + run grows from one piece of the sequence to the next, so it numbers the partial results
      const long long slot = (long long)at.b * a.Hk * a.n_group + at.hg + run;
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float l = st.l[nt][e];
          l += __shfl_xor_sync(0xffffffffu, l, 4);
          l += __shfl_xor_sync(0xffffffffu, l, 8);
          l += __shfl_xor_sync(0xffffffffu, l, 16);
          if (qf.row[nt][e] >= a.R) continue;
          const long long row = slot * (8 * NT) + nt * 8 + 2 * c + e;
          if (g == 0) __stcg(a.part_ml + row, make_float2(ok ? st.m[nt][e] : -INFINITY, l));
          float4* const dst = reinterpret_cast<float4*>(a.part_o + row * HD + 16 * g);
#pragma unroll
          for (int j = 0; j < 8; j += 2)
            __stcg(dst + j / 2, make_float4(st.o[j][nt][e], st.o[j][nt][2 + e], st.o[j + 1][nt][e], st.o[j + 1][nt][2 + e]));
        }
      }
      if (i + 1 < n) {
        at = then;
        enter();
      }
    }
    at = then;
    sc = sc_next;
  }
  if (!ok) {  // let this warp's copies in flight land before the shared memory goes away
    const long long t0 = clock64();
    while ((unsigned long long)(clock64() - t0) < FT_WAIT_LIMIT_CYCLES / 4) __nanosleep(1000);
  }
}

// Rows of the output: each row's partial results in run order, `merge_per_row` warps a row (each a
// contiguous part of them), four dims a lane.
template <int NT>
__global__ void __launch_bounds__(32 * MERGE_WARPS) cache_merge_kernel(DecArgs a) {
  __shared__ float4 so[MERGE_WARPS][32];
  __shared__ float2 sml[MERGE_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = a.merge_per_row, rows_here = MERGE_WARPS / per, part = warp % per;
  const long long rows = (long long)a.B * a.Hk * a.R;
  const long long row = (long long)blockIdx.x * rows_here + warp / per;  // (b * Hk + h) * R + r
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float M = -INFINITY, L = 0.f;
  int r = 0, h = 0, b = 0, len = 0;
  if (row < rows) {
    r = (int)(row % a.R);
    h = (int)(row / a.R % a.Hk);
    b = (int)(row / a.R / a.Hk);
    len = seq_len(a, b);
    const int n = (len + KT - 1) / KT, hg = h * a.n_group + r / (8 * NT);
    const Runs runs(tiles_before(a, a.B, lane) * a.Hk * a.n_group, a.runs);
    const long long f = tiles_before(a, b, lane) * a.Hk * a.n_group + (long long)hg * n;
    pdl_wait();
    if (n > 0) {
      const int r0 = runs.owner(f), r1 = runs.owner(f + n - 1) + 1, cnt = r1 - r0;
      const int lo = r0 + cnt * part / per, hi = r0 + cnt * (part + 1) / per;
      const long long base = ((long long)b * a.Hk * a.n_group + hg) * (8 * NT) + r % (8 * NT);
      for (int i0 = lo; i0 < hi; i0 += 32) {  // references of 32 partials at once, then their rows
        const float2 ml = i0 + lane < hi ? __ldcg(a.part_ml + base + (long long)(i0 + lane) * (8 * NT)) : make_float2(-INFINITY, 0.f);
        float top = ml.x;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float m_new = max_nan(M, top), ref = m_new == -INFINITY ? 0.f : m_new;
        const float al = M == -INFINITY ? 0.f : ex2f(M - ref), w = ml.x == -INFINITY ? 0.f : ex2f(ml.x - ref);
        float l = w * ml.y;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        M = m_new;
        L = L * al + l;
        acc.x *= al;
        acc.y *= al;
        acc.z *= al;
        acc.w *= al;
        const int m = min(32, hi - i0);
#pragma unroll 4
        for (int i = 0; i < m; i++) {
          const float wi = __shfl_sync(0xffffffffu, w, i);
          const float4 v = __ldcg(reinterpret_cast<const float4*>(a.part_o + (base + (long long)(i0 + i) * (8 * NT)) * HD) + lane);
          acc.x = fmaf(wi, v.x, acc.x);
          acc.y = fmaf(wi, v.y, acc.y);
          acc.z = fmaf(wi, v.z, acc.z);
          acc.w = fmaf(wi, v.w, acc.w);
        }
      }
    }
  }
  if (per > 1) {
    so[warp][lane] = acc;
    if (lane == 0) sml[warp] = make_float2(M, L);
    __syncthreads();
    if (part != 0) return;
    float top = M;
    for (int i = 1; i < per; i++) top = max_nan(top, sml[warp + i].x);
    const float ref = top == -INFINITY ? 0.f : top;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
    L = 0.f;
    for (int i = 0; i < per; i++) {
      const float w = sml[warp + i].x == -INFINITY ? 0.f : ex2f(sml[warp + i].x - ref);
      const float4 v = so[warp + i][lane];
      acc.x = fmaf(w, v.x, acc.x);
      acc.y = fmaf(w, v.y, acc.y);
      acc.z = fmaf(w, v.z, acc.z);
      acc.w = fmaf(w, v.w, acc.w);
      L += w * sml[warp + i].y;
    }
  }
  if (row >= rows) return;
  const float inv = 1.f / L;
  uint2 out = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
  if (len - a.Sq + 1 + r / a.G <= 0) out = make_uint2(0, 0);  // the row sees no key
  *reinterpret_cast<uint2*>(a.o + b * a.o_b + (long long)(r / a.G) * a.o_tok + (long long)(h * a.G + r % a.G) * a.o_h + 4 * lane) = out;
}

int rows_of(const CacheDecodeProblem& p) { return p.Sq * (p.Hq / p.Hk); }
int col_tiles(const CacheDecodeProblem& p) { return rows_of(p) > 8 ? 2 : 1; }
int groups_of(const CacheDecodeProblem& p) { return (rows_of(p) + 8 * col_tiles(p) - 1) / (8 * col_tiles(p)); }

long long units_of(const CacheDecodeProblem& p) { return (long long)p.B * p.Hk * groups_of(p); }
int runs_of(const CacheDecodeProblem& p) { return p.num_sms * NWARP; }
long long partials_of(const CacheDecodeProblem& p) { return (units_of(p) + runs_of(p)) * 8 * col_tiles(p); }

// One map of a cache side: [128 bytes][heads][tokens][sequences]. A broadcast dimension (stride 0)
// is mapped with one entry.
bool side_map(CUtensorMap* m, const CacheSide& s, const CacheDecodeProblem& p, int& one_b, int& one_h) {
  one_b = p.B == 1 || s.c_b == 0;
  one_h = p.Hk == 1 || s.c_h == 0;
  return make_tmap_4d_u8(m, s.codes, HD, one_h ? 1 : p.Hk, p.L, one_b ? 1 : p.B, one_h ? HD : s.c_h,
                         p.L == 1 ? HD : s.c_tok, one_b ? HD : s.c_b, HD, 1, KT, 1);
}

template <int NT, int FMT>
cudaError_t launch_decode(const CUtensorMap& tk, const CUtensorMap& tv, const DecArgs& a, int sms, cudaStream_t stream) {
  const int smem = (int)sizeof(DecSmem) + 1024;
  static bool attr = false;
  if (!attr) {
    const cudaError_t e = cudaFuncSetAttribute(cache_decode_kernel<NT, FMT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    attr = true;
  }
  cache_decode_kernel<NT, FMT><<<sms, 32 * NWARP, smem, stream>>>(tk, tv, a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  // the merge may start while the first kernel's last CTAs run; it waits for them before it reads
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  const long long rows = (long long)a.B * a.Hk * a.R;
  cfg.gridDim = dim3((unsigned)((rows * a.merge_per_row + MERGE_WARPS - 1) / MERGE_WARPS));
  cfg.blockDim = dim3(32 * MERGE_WARPS);
  cfg.stream = stream;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, cache_merge_kernel<NT>, a);
}

}  // namespace

size_t cache_decode_scratch_floats(const CacheDecodeProblem& p) { return (size_t)partials_of(p) * (HD + 2); }

cudaError_t cache_append(const CacheAppendProblem& p, cudaStream_t stream) {
  if (p.B <= 0 || p.S <= 0 || p.Hk <= 0) return cudaSuccess;
  AppendArgs a;
  a.B = p.B;
  a.S = p.S;
  a.Hk = p.Hk;
  a.L = p.L;
  for (int i = 0; i < 2; i++) {
    a.x[i] = p.x[i];
    a.x_b[i] = p.x_b[i];
    a.x_tok[i] = p.x_tok[i];
    a.x_h[i] = p.x_h[i];
    a.side[i] = p.side[i];
  }
  a.pos = p.pos;
  a.pos_all = p.pos_all;
  a.n_new = p.n_new;
  // blocks that S tokens can touch; a known position says exactly how many
  a.n_rel = p.pos ? (p.S + p.block - 2) / p.block + 1 : (p.pos_all % p.block + p.S + p.block - 1) / p.block;
  switch (p.block) {
    case 16: return launch_append<16>(a, p.format, stream);
    case 32: return launch_append<32>(a, p.format, stream);
    case 64: return launch_append<64>(a, p.format, stream);
    case 128: return launch_append<128>(a, p.format, stream);
    case 256: return launch_append<256>(a, p.format, stream);
  }
  return cudaErrorInvalidValue;
}

cudaError_t cache_decode(const CacheDecodeProblem& p, cudaStream_t stream) {
  if (p.B <= 0 || p.Sq <= 0 || p.Hq <= 0) return cudaSuccess;
  if (p.Hk <= 0 || p.Hq % p.Hk) return cudaErrorInvalidValue;
  DecArgs a;
  a.B = p.B;
  a.Sq = p.Sq;
  a.Hq = p.Hq;
  a.Hk = p.Hk;
  a.L = p.L;
  a.G = p.Hq / p.Hk;
  a.R = rows_of(p);
  a.n_group = groups_of(p);
  a.block_shift = 31 - __builtin_clz((unsigned)p.block);
  a.q = p.q;
  a.q_b = p.q_b;
  a.q_tok = p.q_tok;
  a.q_h = p.q_h;
  a.o = p.o;
  a.o_b = p.o_b;
  a.o_tok = p.o_tok;
  a.o_h = p.o_h;
  a.k = p.side[0];
  a.v = p.side[1];
  a.kv_len = p.kv_len;
  a.len_all = p.len_all;
  a.max_len = p.max_len;
  a.scale_log2 = p.scale * 1.4426950408889634f;
  a.runs = runs_of(p);
  const long long rows = (long long)p.B * p.Hk * a.R;
  // units, runs and rows are numbered in 32 bits on the way
  if (rows > 0x3fffffffLL || units_of(p) > 0x3fffffffLL || p.B > (1 << 24)) return cudaErrorInvalidValue;
  if (p.scratch == nullptr) return cudaErrorInvalidValue;
  a.part_o = p.scratch;
  a.part_ml = reinterpret_cast<float2*>(p.scratch + (size_t)partials_of(p) * HD);
  // a row has about runs / units partials; warps that share it take a few each
  const long long expect = a.runs / units_of(p);
  a.merge_per_row = expect >= 64 ? 8 : expect >= 16 ? 4 : expect >= 8 ? 2 : 1;
  CUtensorMap tk, tv;
  if (p.L > 0 && (!side_map(&tk, p.side[0], p, a.one_b[0], a.one_h[0]) || !side_map(&tv, p.side[1], p, a.one_b[1], a.one_h[1])))
    return cudaErrorInvalidValue;
  const bool i8 = p.format == CACHE_INT8;
  if (col_tiles(p) == 1)
    return i8 ? launch_decode<1, CACHE_INT8>(tk, tv, a, p.num_sms, stream) : launch_decode<1, CACHE_E4M3>(tk, tv, a, p.num_sms, stream);
  return i8 ? launch_decode<2, CACHE_INT8>(tk, tv, a, p.num_sms, stream) : launch_decode<2, CACHE_E4M3>(tk, tv, a, p.num_sms, stream);
}

}  // namespace ft
