// Key/value cache in 8 bits with one scale per block of tokens and head: writing tokens into it
// and decode attention over it, head_dim 128, for sm_100a.
//
// Writing. A block's scale is the smallest power of two s with max|x| <= qmax * s (qmax 127 for
// int8, 448 for e4m3), so x / s is exact and a block written at once has codes that depend on its
// values alone. A block that already holds tokens keeps the larger of its old scale and the new
// tokens', and its old codes are rounded again when the scale grew: written in several calls, its
// codes depend on their order too (by at most one step of the last scale). The largest magnitude is found on the bf16 bit patterns
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
// Work. The eight warps of a CTA (one CTA an SM) take tiles of as many heads side by side as divide
// the heads (8, 4, 2 or 1), and consecutive tiles of a head where that leaves warps over. The units
// of 32 keys of those heads, in the order sequence, heads, keys, are divided into equal contiguous
// runs, one per CTA, so ragged batches and few long sequences load every SM alike. Heads side by side
// matter because one token's heads are neighbours in memory: with a run per warp, each in its own
// head, the same copies took 34.8 us instead of 26.5 (32 x 2304 tokens, 8 heads) and 54 us instead of
// 42 (131071 tokens) without any arithmetic. A warp streams its tiles by itself through three 8 KB
// slots that hold 64 keys and their values in turn (TMA, 128-byte swizzle; the warp's own program
// order says when a slot is free, so there is no producer and no barrier between warps) and writes
// fp32 partial results where its head or its run end; a second kernel, launched so that its start
// overlaps the first one's end, merges the partials of each row in a fixed order.
//
// Scales: a score is (q . codes) * ks, and the weight of a value's codes is p * vs. The running
// reference is 7 below the maximum of score + log2(vs) (in log2 units), so that p * vs is at most 2^15
// whatever the scales are and f16 holds it to 2^-11, or to 2^-32 of the largest weight where that is
// more (a million keys that weigh less together still add up to 2^-12); the sum l takes p in fp32. q is
// scaled by a power of two per row into f16, the row's largest element to 1 .. 2: elements below 2^-17 of it
// lose bits there, by at most 2^-25 of the largest (f16's numbers are 2^-24 apart below 2^-14).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "ft_cache.h"
#include "ft_ops.h"
#include "sm100_common.cuh"

namespace ft {

FT_DEFINE_ERROR_READER(cache_device_error)

namespace {

constexpr int HD = 128;  // head dim

// Every kernel here is launched so that it may start while the kernel before it in the stream ends
// (programmatic serialization): it waits for that kernel's results before it reads any memory. No load
// takes the non-coherent path, which that wait says nothing about.

// ------------------------------------------------------------------------------------ writing
struct AppendArgs {
  int B, S, Hk, L, n_rel;  // n_rel: groups of blocks a sequence can touch, one a CTA
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

// Four values to codes, rounded to nearest even. int8: the sum with 1.5 * 2^23 has the rounded number in
// its low bits; values are within +-128 by the choice of the scale. (The integer conversion runs at a
// quarter of the rate: prompts took 72 us with it, 61 without.)
template <int FMT>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  if (FMT == CACHE_INT8) {
    const uint32_t ia = __float_as_uint(a + 12582912.f), ib = __float_as_uint(b + 12582912.f);
    const uint32_t ic = __float_as_uint(c + 12582912.f), id = __float_as_uint(d + 12582912.f);
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

// A block belongs to BLOCK / 16 warps, whose lanes hold its new tokens in registers (eight 16-byte pieces
// each) between the maximum and the rounding, so they are read once; a CTA of at least four warps takes
// consecutive blocks of one sequence and KV head, keys or values. Bound by HBM for prompts (32 x 2048
// tokens, 8 heads: 403 MB in 60-61 us at blocks of 16 to 64 tokens, the rate of a copy; 66 at 128, 94 at
// 256: 512 threads of 80 and more registers leave room for one CTA an SM, whose loads, barrier and stores
// then overlap with no other's) and by the launch for single tokens (3.0 us on the device).
template <int BLOCK>
struct AppendShape {
  static constexpr int WARPS_PER_BLOCK = BLOCK / 16, WARPS = WARPS_PER_BLOCK > 4 ? WARPS_PER_BLOCK : 4;
  static constexpr int BLOCKS = WARPS / WARPS_PER_BLOCK;  // of a CTA
};

template <int BLOCK, int FMT>
__global__ void __launch_bounds__(32 * AppendShape<BLOCK>::WARPS) cache_append_kernel(const __grid_constant__ AppendArgs a) {
  using Shape = AppendShape<BLOCK>;
  constexpr int WPB = Shape::WARPS_PER_BLOCK, STEP = 2 * WPB, ITERS = 8;  // a warp's pass is two token rows
  __shared__ uint32_t warp_max[Shape::WARPS];
  pdl_wait();
  pdl_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  long long id = blockIdx.x;
  const int h = (int)(id % a.Hk);
  id /= a.Hk;
  const int rel = (int)(id % a.n_rel) * Shape::BLOCKS + warp / WPB;
  id /= a.n_rel;
  const int kv = (int)(id & 1), b = (int)(id >> 1);
  const int p = a.pos ? a.pos[b] : a.pos_all, n = a.n_new ? a.n_new[b] : a.S;
  if (p < 0 || n < 0 || n > a.S || p > a.L - n) {  // nothing of such a sequence is written
    if (threadIdx.x == 0) record_error(kErrBadArgs);
    return;
  }
  const int j = p / BLOCK + rel;
  const int t0 = max(p, j * BLOCK), t1 = min(p + n, (j + 1) * BLOCK);  // new tokens of the block; t0 >= t1: none
  const CacheSide& sd = a.side[kv];
  float* const sp = sd.scale + b * sd.s_b + j * sd.s_blk + h * sd.s_h;
  const bool some = t0 < t1, history = some && t0 > j * BLOCK;
  const float s_old = history ? *sp : 0.f;
  const int row0 = j * BLOCK + (warp % WPB) * 2 + lane / 16, col = (lane % 16) * 8;
  const __nv_bfloat16* const x = a.x[kv] + b * a.x_b[kv] + h * a.x_h[kv] + col;
  uint4 v[ITERS];
  uint32_t m2 = 0;
#pragma unroll
  for (int i = 0; i < ITERS; i++) {
    const int t = row0 + i * STEP;
    v[i] = make_uint4(0, 0, 0, 0);
    if (t >= t0 && t < t1) v[i] = *reinterpret_cast<const uint4*>(x + (long long)(t - p) * a.x_tok[kv]);
  }
#pragma unroll
  for (int i = 0; i < ITERS; i++) {
    m2 = __vmaxu2(m2, __vmaxu2(__vmaxu2(v[i].x & 0x7fff7fffu, v[i].y & 0x7fff7fffu),
                               __vmaxu2(v[i].z & 0x7fff7fffu, v[i].w & 0x7fff7fffu)));
  }
  uint32_t m = __reduce_max_sync(0xffffffffu, max(m2 & 0xffffu, m2 >> 16));
  if (WPB > 1) {
    if (lane == 0) warp_max[warp] = m;
    __syncthreads();  // also: every thread has read the old scale
#pragma unroll
    for (int w = 0; w < WPB; w++) m = max(m, warp_max[warp / WPB * WPB + w]);
  } else {
    __syncwarp();
  }
  if (!some) return;
  const float s_new = pow2_scale<FMT>(m);
  const float s = s_old != s_old ? s_old : (s_new != s_new ? s_new : fmaxf(s_old, s_new));
  const bool bad = s != s;
  const float inv = bad ? 0.f : (s > 0.f ? 1.f / s : 0.f);
  uint8_t* const out = sd.codes + b * sd.c_b + h * sd.c_h + col;
  if (history && s != s_old) {
    const float ratio = bad ? 0.f : s_old * inv;
    for (int t = row0; t < t0; t += STEP) {
      uint2* const w = reinterpret_cast<uint2*>(out + (long long)t * sd.c_tok);
      const uint2 o = *w;
      *w = bad ? make_uint2(0, 0) : make_uint2(recode4<FMT>(o.x, ratio), recode4<FMT>(o.y, ratio));
    }
  }
  if (lane == 0 && warp % WPB == 0) *sp = s;
#pragma unroll
  for (int i = 0; i < ITERS; i++) {
    const int t = row0 + i * STEP;
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
cudaError_t launch_append(AppendArgs a, int format, cudaStream_t stream) {
  using Shape = AppendShape<BLOCK>;
  a.n_rel = (a.n_rel + Shape::BLOCKS - 1) / Shape::BLOCKS;
  const long long grid = (long long)a.B * 2 * a.n_rel * a.Hk;
  if (grid > 0x7fffffffLL) return cudaErrorInvalidValue;
  return launch_overlapped(format == CACHE_INT8 ? cache_append_kernel<BLOCK, CACHE_INT8> : cache_append_kernel<BLOCK, CACHE_E4M3>,
                           dim3((unsigned)grid), 32 * Shape::WARPS, 0, stream, a);
}

// ------------------------------------------------------------------------------------ attention
constexpr int UNIT = 32;     // keys: what runs are made of
constexpr int WARPS = 8;
constexpr int SLOTS = 3;     // per warp, keys and values in turn
// Units of a tile: two column tiles leave registers for one
constexpr int units_of_tile(int column_tiles) { return column_tiles == 1 ? 2 : 1; }
constexpr int UNIT_BYTES = UNIT * HD;
// What entering a head costs a warp (its queries, its partial result, a tile cut short), in units: runs
// are equal in units plus this much for each head and sequence
constexpr int ENTRY = 2;
constexpr int MERGE_WARPS = 16;  // at most

struct DecArgs {
  int B, Hq, Hk, L, G, R, n_group;      // R query rows of a KV head (queries x G) in n_group groups of 8 * NT
  int to_end;                           // tokens of a sequence from the first query's to its last
  int block_shift;
  int heads, keys;                      // (head, group) units and key tiles side by side in a CTA: heads * keys = WARPS
  int per;                              // Hk * n_group / heads: steps of heads in a sequence
  int runs;                             // CTAs
  const __nv_bfloat16* q;
  long long q_b, q_tok, q_h;
  __nv_bfloat16* o;
  long long o_b, o_tok, o_h;
  CacheSide k, v;
  int one_b[2], one_h[2];               // keys / values: the cache is broadcast over sequences / heads (stride 0)
  const int* kv_len;
  int len_all, max_len;
  float scale_log2;                     // softmax scale * log2(e)
  float* part_o;                        // [steps of heads + runs][WARPS][8 * NT][128]
  float2* part_ml;                      // [steps of heads + runs][WARPS][8 * NT] reference and sum
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

// 2^(d/2) for a difference of references d down to -252: sums are scaled by it twice. A block of zeros puts
// its reference up to 181 below that of values beside it while its keys' p are as large, and 2^d by itself
// would be 0 there; for the outputs, which are in the unit of the reference, that is right.
__device__ __forceinline__ float root_of_scale(float d) { return ex2f(0.5f * d); }

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

// Their bf16 rows as they lie in memory: 64 bytes a lane and row. Loaded apart from their conversion,
// so that the loads are on their way before the keys and values that fill the memory's queues.
template <int NT>
struct RawQueries {
  uint4 w[NT][4];
  int row0;
};

template <int NT>
__device__ __forceinline__ void load_queries(RawQueries<NT>& raw, const DecArgs& a, int b, int h, int row0, int lane) {
  const int g = lane >> 2, c = lane & 3;
  raw.row0 = row0;
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    const int r = row0 + nt * 8 + g;
    const uint4* p = reinterpret_cast<const uint4*>(a.q + b * a.q_b + (long long)(r / a.G) * a.q_tok +
                                                    (long long)(h * a.G + r % a.G) * a.q_h + 32 * c);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      raw.w[nt][i] = make_uint4(0, 0, 0, 0);
      if (r < a.R) raw.w[nt][i] = p[i];
    }
  }
}

template <int NT>
__device__ __forceinline__ void convert_queries(QueryFrag<NT>& f, const RawQueries<NT>& raw, const DecArgs& a, int lane) {
  const int c = lane & 3, row0 = raw.row0;
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    const uint4(&w)[4] = raw.w[nt];
    const uint32_t x[16] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w,
                            w[2].x, w[2].y, w[2].z, w[2].w, w[3].x, w[3].y, w[3].z, w[3].w};
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

// The scales of a tile's 16-key groups, keys' and values'.
// In the reference a value scale counts as at least 2^-60, so a key's p is at most 2^75 (blocks of zeros), and
// as finite, so that an infinite one stays with the rows that see it. Tiles with a scale outside 2^+-30 compute
// p by itself, the others as (p * vs) / vs, which has fp32's precision beside value scales up to 2^90 times
// larger. Values of scales below 2^-84 underflow to 0.
constexpr float V_SCALE_MIN = 0x1p-60f, V_SCALE_MAX = 0x1.fffffep127f, V_SCALE_ODD = 0x1p30f;
// p and its sums are kept 2^20 times larger: at most 2^127 over 2^32 keys. The key that weighs most has
// 2^(27 - 122) or more beside bf16's largest values (whose scale is 2^122 in int8), and one 2^31 times lighter
// is still a normal number; beside the largest scale that fp32 holds, one 2^25 times lighter.
constexpr float SUM_LOG2 = 20.f, SUM_UNIT = 0x1p20f;

template <int MT>
struct TileScales {
  float k[MT], v[MT];
};

// One tile of 16 * MT keys: `kt`/`vt` give 16-byte pieces (row, piece) of the tile's codes, `lim` the
// number of keys of the tile that each column sees (16 * MT or more: all). `keys_read` is called when
// the keys have been read, `values_here` before the values are.
template <int NT, int MT, int FMT, class KLoad, class VLoad, class KDone, class VReady>
__device__ __forceinline__ void attend_tile(RowState<NT>& st, const QueryFrag<NT>& qf, KLoad kt, VLoad vt,
                                            const TileScales<MT>& sc, const int (&lim)[NT][2], bool masked, int lane,
                                            KDone keys_read, VReady values_here) {
  const int g = lane >> 2, c = lane & 3;
  float s[MT][NT][4];
#pragma unroll
  for (int mt = 0; mt < MT; mt++)
#pragma unroll
    for (int nt = 0; nt < NT; nt++) s[mt][nt][0] = s[mt][nt][1] = s[mt][nt][2] = s[mt][nt][3] = 0.f;
#pragma unroll
  for (int hh = 0; hh < 2; hh++) {
    uint4 x[MT], y[MT];
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
      x[mt] = kt(mt * 16 + g, 2 * c + hh);
      y[mt] = kt(mt * 16 + g + 8, 2 * c + hh);
    }
#pragma unroll
    for (int w = 0; w < 4; w++) {
#pragma unroll
      for (int mt = 0; mt < MT; mt++) {  // MT independent chains
        const uint32_t xw[4] = {x[mt].x, x[mt].y, x[mt].z, x[mt].w}, yw[4] = {y[mt].x, y[mt].y, y[mt].z, y[mt].w};
        uint32_t a0, a1, a2, a3;
        decode4<FMT>(xw[w], a0, a2);
        decode4<FMT>(yw[w], a1, a3);
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
          mma16816_f16(s[mt][nt], a0, a1, a2, a3, qf.b[nt][hh * 4 + w][0], qf.b[nt][hh * 4 + w][1]);
      }
    }
  }
  keys_read();
  float lv[MT], iv[MT];
  bool odd = false;  // a value scale that is 0, small, large or NaN
#pragma unroll
  for (int mt = 0; mt < MT; mt++) {
    odd |= !(sc.v[mt] >= 1.f / V_SCALE_ODD && sc.v[mt] <= V_SCALE_ODD);
    const float v = fminf(fmaxf(sc.v[mt], V_SCALE_MIN), V_SCALE_MAX);
    lv[mt] = lg2f(v);
    iv[mt] = __fdividef(SUM_UNIT, v);
  }
  uint32_t pb[MT][NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
      const float f0 = sc.k[mt] * qf.fac[nt][0], f1 = sc.k[mt] * qf.fac[nt][1];
      s[mt][nt][0] *= f0;
      s[mt][nt][1] *= f1;
      s[mt][nt][2] *= f0;
      s[mt][nt][3] *= f1;
    }
    if (masked) {
#pragma unroll
      for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (mt * 16 + g + 8 * (e >> 1) >= lim[nt][e & 1]) s[mt][nt][e] = -INFINITY;
    }
    float top[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
      top[i] = max_nan(s[0][nt][i], s[0][nt][2 + i]) + lv[0];
#pragma unroll
      for (int mt = 1; mt < MT; mt++) top[i] = max_nan(top[i], max_nan(s[mt][nt][i], s[mt][nt][2 + i]) + lv[mt]);
    }
    // the reference moves only when a weight would pass 2^15, so the accumulators are seldom rescaled;
    // all lanes of a column take the same one
    const bool grow = !(top[0] <= st.m[nt][0] + 15.f) || !(top[1] <= st.m[nt][1] + 15.f);
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        top[i] = max_nan(top[i], __shfl_xor_sync(0xffffffffu, top[i], 4));
        top[i] = max_nan(top[i], __shfl_xor_sync(0xffffffffu, top[i], 8));
        top[i] = max_nan(top[i], __shfl_xor_sync(0xffffffffu, top[i], 16));
        const float m_new = max_nan(st.m[nt][i], top[i] - 7.f);
        const float root = st.m[nt][i] == -INFINITY ? 0.f : root_of_scale(st.m[nt][i] - m_new), al = root * root;
        st.m[nt][i] = m_new;
        st.l[nt][i] = st.l[nt][i] * root * root;
#pragma unroll
        for (int j = 0; j < 8; j++) {
          st.o[j][nt][i] *= al;
          st.o[j][nt][2 + i] *= al;
        }
      }
    }
    const float ref[2] = {st.m[nt][0] == -INFINITY ? 0.f : st.m[nt][0], st.m[nt][1] == -INFINITY ? 0.f : st.m[nt][1]};
    auto weights = [&](int mt, float w0, float w1, float w2, float w3) {
      __half2 h0 = __floats2half2_rn(w0, w1), h1 = __floats2half2_rn(w2, w3);
      pb[mt][nt][0] = transpose8x8(*reinterpret_cast<uint32_t*>(&h0));
      pb[mt][nt][1] = transpose8x8(*reinterpret_cast<uint32_t*>(&h1));
    };
    if (!odd) {  // two loops: a branch inside one kept scores alive and cost 2 us of 53
#pragma unroll
      for (int mt = 0; mt < MT; mt++) {
        const float d0 = lv[mt] - ref[0], d1 = lv[mt] - ref[1];
        const float w[4] = {ex2f(s[mt][nt][0] + d0), ex2f(s[mt][nt][1] + d1), ex2f(s[mt][nt][2] + d0), ex2f(s[mt][nt][3] + d1)};
        st.l[nt][0] = fmaf(w[0] + w[2], iv[mt], st.l[nt][0]);
        st.l[nt][1] = fmaf(w[1] + w[3], iv[mt], st.l[nt][1]);
        weights(mt, w[0], w[1], w[2], w[3]);
      }
    } else {  // p * vs is 0 for a scale of 0, NaN for NaN, and 0 for what the column does not see
#pragma unroll
      for (int mt = 0; mt < MT; mt++) {
        const float v = sc.v[mt] * (1.f / SUM_UNIT);
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float p = ex2f(s[mt][nt][e] + (SUM_LOG2 - ref[e & 1]));
          st.l[nt][e & 1] += p;
          w[e] = masked && mt * 16 + g + 8 * (e >> 1) >= lim[nt][e & 1] ? 0.f : p * v;
        }
        weights(mt, w[0], w[1], w[2], w[3]);
      }
    }
  }
  if (!values_here()) return;
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
  return max(0, min(a.kv_len ? a.kv_len[b] : a.len_all, a.max_len));
}
__device__ __forceinline__ int seq_units(const DecArgs& a, int b) { return (seq_len(a, b) + UNIT - 1) / UNIT; }

// the length of a sequence's share of the work in one step of heads: ENTRY places for the entry, then its units
__device__ __forceinline__ int seq_cost(const DecArgs& a, int b) {
  const int n = seq_units(a, b);
  return n ? n + ENTRY : 0;
}

// sum of the costs of sequences [0, end) over all steps of heads, by a whole warp
__device__ __forceinline__ int cost_before(const DecArgs& a, int end, int lane) {
  if (a.kv_len == nullptr) return end * seq_cost(a, 0) * a.per;
  int sum = 0;
  for (int b = lane; b < end; b += 32) sum += seq_cost(a, b);
  return __reduce_add_sync(0xffffffffu, sum) * a.per;
}

// The sequence of places (fewer than 2^30, the host checks) and its division into runs, the first
// `rem` of them one place longer.
struct Runs {
  int n, base, rem;
  __device__ __forceinline__ Runs(int total, int most) : n(min(most, total)) {
    base = n ? total / n : 0;
    rem = total - base * n;
  }
  __device__ __forceinline__ int begin(int r) const { return r * base + min(r, rem); }
  __device__ __forceinline__ int owner(int i) const {
    const int longer = rem * (base + 1);
    return i < longer ? i / (base + 1) : rem + (i - longer) / base;
  }
};

// A warp's place in its CTA's run: a tile of units [t, min(t + units of a tile, end)) of a piece, the
// run's part of one step of heads of one sequence. The tiles of a piece go to the warps of a head in
// turn, beginning with the one after the piece before: tile i of a piece is warp (i + turn) % keys'.
struct Cursor {
  int b, j, t, from, end, left;  // sequence, step of heads, unit, the piece's units [from, end), places of the run after it
  int turn;

  // this warp's place in the turn, which numbers its partial result of the piece
  __device__ __forceinline__ int key(const DecArgs& a, int warp_key) const { return (warp_key - turn) & (a.keys - 1); }

  // this warp's next tile (its first where t is the piece's begin and `first`); false at the run's end
  template <int UT>
  __device__ __forceinline__ bool next(const DecArgs& a, int warp_key, bool first) {
    t += first ? key(a, warp_key) * UT : a.keys * UT;
    while (t >= end) {
      if (left == 0) return false;
      turn += max(0, (end - from + UT - 1) / UT);
      int n = 0;
      if (++j == a.per) j = 0, b++;
      while ((n = seq_cost(a, b)) == 0) b++;  // places are left, so a sequence with some follows
      n = min(n, left);
      left -= n;
      from = 0;
      end = n - ENTRY;
      t = key(a, warp_key) * UT;
    }
    return true;
  }
};

// place i, the first of a run of `count`, by a whole warp
__device__ __forceinline__ Cursor locate(const DecArgs& a, int i, int count, int lane) {
  Cursor c;
  int n;
  if (a.kv_len == nullptr) {
    n = seq_cost(a, 0);
    c.b = i / (n * a.per);
    i -= c.b * n * a.per;
  } else {
    int before = 0;
    for (int b0 = 0;; b0 += 32) {  // i lies before the total, so some sequence holds it
      const int mine = b0 + lane < a.B ? seq_cost(a, b0 + lane) : 0;
      int end = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, end, o);
        if (lane >= o) end += up;
      }
      const unsigned int hit = __ballot_sync(0xffffffffu, (before + end) * a.per > i);
      if (hit || b0 + 32 >= a.B) {
        const int at = hit ? __ffs(hit) - 1 : 31;
        c.b = b0 + at;
        n = __shfl_sync(0xffffffffu, mine, at);
        i -= (before + __shfl_sync(0xffffffffu, end - mine, at)) * a.per;
        break;
      }
      before += __shfl_sync(0xffffffffu, end, 31);
    }
  }
  c.j = i / n;
  i -= c.j * n;
  c.left = count - (min(n, i + count) - i);
  c.from = c.t = max(0, i - ENTRY);
  c.turn = 0;
  c.end = min(n, i + count) - ENTRY;
  return c;
}

__device__ __forceinline__ void tma_load_4d(void* dst, const void* tmap, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}

template <int NT>
struct DecSmem {
  uint8_t slot[WARPS][SLOTS][units_of_tile(NT) * UNIT_BYTES];
  uint64_t full[WARPS][SLOTS];
};

// Bound by HBM where sequences are long (131071 tokens, 8 heads, e4m3: 268 MB in 51-53 us with the merge,
// 5.1-5.3 TB/s; 32 x 2304 tokens, int8: 152 MB in 35 us, of which 24 us stream) and by latency where they
// are short. The loads of a head's queries and scales come before the copies, which would hold them
// up for 5 us in the memory's queues.
template <int NT, int FMT>
__global__ void __launch_bounds__(32 * WARPS, 1)
    cache_decode_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                        const __grid_constant__ DecArgs a) {
  constexpr int UT = units_of_tile(NT), MT = UT * UNIT / 16;
  extern __shared__ uint8_t smem_raw[];
  DecSmem<NT>& sm = *reinterpret_cast<DecSmem<NT>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  uint64_t* const full = sm.full[warp];
  if (lane == 0) {
    for (int s = 0; s < SLOTS; s++) mbar_init(&full[s], 1);
    fence_barrier_init();
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  __syncwarp();
  pdl_wait();
  pdl_launch();
  const Runs runs(cost_before(a, a.B, lane), a.runs);
  const int run = blockIdx.x;
  if (run >= runs.n) return;
  const int first = runs.begin(run), count = runs.begin(run + 1) - first;
  const int my_head = warp % a.heads, my_key = warp / a.heads;
  Cursor at = locate(a, first, count, lane);
  if (!at.next<UT>(a, my_key, true)) return;  // a run too short for this warp
  Cursor ahead = at;
  auto fetch = [&](int s, bool values) {  // keys or values of the tile at `ahead` into slot s
    if (lane == 0) {
      const int hg = ahead.j * a.heads + my_head, h = a.n_group == 1 ? hg : hg / a.n_group;
      const int z = a.one_h[values] ? 0 : h, w = a.one_b[values] ? 0 : ahead.b;
      const CUtensorMap* const map = values ? &tm_v : &tm_k;
      uint8_t* const dst = sm.slot[warp][s];
      const bool two = UT == 2 && ahead.t + 1 < ahead.end;
      mbar_arrive_expect_tx(&full[s], two ? 2 * UNIT_BYTES : UNIT_BYTES);
      tma_load_4d(dst, map, &full[s], 0, z, ahead.t * UNIT, w);
      if (two) tma_load_4d(dst + UNIT_BYTES, map, &full[s], 0, z, (ahead.t + 1) * UNIT, w);
    }
  };
  QueryFrag<NT> qf;
  RawQueries<NT> raw;
  RowState<NT> st;
  int sees[NT][2], len = 0, len_next = 0;
  const float *ksp = nullptr, *vsp = nullptr;  // the head's scales
  TileScales<MT> sc;
  // The scales of the tile at unit t of a sequence of n keys. 16 keys never straddle a block, and a
  // tile of a whole block or less takes one scale; what lies past the length takes the last block's.
  auto scales = [&](int t, int n) {
    if (16 * MT <= 1 << a.block_shift) {
      const int blk = (t * UNIT) >> a.block_shift, blk2 = min(t * UNIT + 16 * MT - 1, n - 1) >> a.block_shift;
      const float k0 = ksp[(long long)blk * a.k.s_blk], v0 = vsp[(long long)blk * a.v.s_blk];
      const float k1 = ksp[(long long)blk2 * a.k.s_blk], v1 = vsp[(long long)blk2 * a.v.s_blk];
#pragma unroll
      for (int i = 0; i < MT; i++) {  // a tile that starts at an odd unit may lie in two blocks, half in each
        sc.k[i] = i < MT / 2 ? k0 : k1;
        sc.v[i] = i < MT / 2 ? v0 : v1;
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < MT; i++) {
      const int blk = min(t * UNIT + 16 * i, n - 1) >> a.block_shift;
      sc.k[i] = ksp[(long long)blk * a.k.s_blk];
      sc.v[i] = vsp[(long long)blk * a.v.s_blk];
    }
  };
  auto prepare = [&](const Cursor& x) {  // the loads for a new head, whose first tile is at x
    const int hg = x.j * a.heads + my_head, h = hg / a.n_group;
    len_next = seq_len(a, x.b);
    ksp = a.k.scale + x.b * a.k.s_b + h * a.k.s_h;
    vsp = a.v.scale + x.b * a.v.s_b + h * a.v.s_h;
    load_queries<NT>(raw, a, x.b, h, (hg - h * a.n_group) * 8 * NT, lane);
    scales(x.t, len_next);
  };
  auto enter = [&]() {  // the new head: its queries, empty accumulators
    len = len_next;
    convert_queries<NT>(qf, raw, a, lane);
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        st.m[nt][i] = -INFINITY;
        st.l[nt][i] = 0.f;
        sees[nt][i] = len - a.to_end + 1 + min(qf.row[nt][i], a.R - 1) / a.G;
#pragma unroll
        for (int j = 0; j < 8; j++) st.o[j][nt][i] = st.o[j][nt][2 + i] = 0.f;
      }
    }
  };
  prepare(at);  // before the copies: behind 192 KB an SM of them these loads took 5 us
  fetch(0, false);
  fetch(1, true);
  bool more = ahead.next<UT>(a, my_key, false);  // whether `ahead` is a tile after `at`
  if (more) fetch(2, false);
  enter();
  bool ok = true;
  int s = 0;        // slot of the next piece to read
  uint32_t ph = 0;  // and its phase
  auto turn = [&]() {
    if (++s == SLOTS) {
      s = 0;
      ph ^= 1;
    }
  };
  for (;;) {
    const bool last = !more || ahead.j != at.j || ahead.b != at.b;  // tile of this head
    const int key0 = at.t * UNIT, here = min((at.end - at.t) * UNIT, 16 * MT);  // keys of the tile that are this run's
    if (ok) ok = __all_sync(0xffffffffu, bounded_wait(&full[s], ph));
    const int sk = s;
    turn();
    if (ok) {
      int lim[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        lim[nt][0] = min(sees[nt][0] - key0, here);
        lim[nt][1] = min(sees[nt][1] - key0, here);
      }
      const bool masked = here < 16 * MT || key0 + 16 * MT > len - a.to_end + 1;
      const int valid = min(len - key0, here);
      const uint32_t kb = smem_u32(sm.slot[warp][sk]), vb = smem_u32(sm.slot[warp][s]);
      auto kt = [&](int r, int piece) { return lds128(kb + r * 128 + ((piece ^ (r & 7)) << 4)); };
      auto vt = [&](int r, int piece) {
        uint4 v = lds128(vb + r * 128 + ((piece ^ (r & 7)) << 4));
        // e4m3 bytes past the length may be NaN codes, which a weight of 0 would not cancel
        if (FMT == CACHE_E4M3 && r >= valid) v = make_uint4(0, 0, 0, 0);
        return v;
      };
      auto keys_read = [&]() {  // the slot takes the values of the next tile
        __syncwarp();
        if (more) fetch(sk, true);
      };
      auto values_here = [&]() { return ok = __all_sync(0xffffffffu, bounded_wait(&full[s], ph)); };
      const TileScales<MT> now = sc;
      if (!last) scales(ahead.t, len);  // in flight during the tile
      else if (more) prepare(ahead);
      attend_tile<NT, MT, FMT>(st, qf, kt, vt, now, lim, masked, lane, keys_read, values_here);
      __syncwarp();
    }
    if (last) {
      // step of heads + run grows from one piece to the next: it numbers the pieces
      const long long piece = ((long long)at.b * a.per + at.j + run) * WARPS + at.key(a, my_key) * a.heads + my_head;
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float l = st.l[nt][e];
          l += __shfl_xor_sync(0xffffffffu, l, 4);
          l += __shfl_xor_sync(0xffffffffu, l, 8);
          l += __shfl_xor_sync(0xffffffffu, l, 16);
          if (qf.row[nt][e] >= a.R) continue;
          const long long row = piece * (8 * NT) + nt * 8 + 2 * c + e;
          if (g == 0) __stcg(a.part_ml + row, make_float2(ok ? st.m[nt][e] : -INFINITY, l));
          float4* const dst = reinterpret_cast<float4*>(a.part_o + row * HD + 16 * g);
#pragma unroll
          for (int j = 0; j < 8; j += 2)
            __stcg(dst + j / 2, make_float4(st.o[j][nt][e], st.o[j][nt][2 + e], st.o[j + 1][nt][e], st.o[j + 1][nt][2 + e]));
        }
      }
    }
    if (!more) break;
    at = ahead;
    more = ahead.next<UT>(a, my_key, false);
    if (more && ok) fetch(s, false);
    turn();
    if (last) enter();
  }
  if (!ok) {  // let this warp's copies in flight land before the shared memory goes away
    const long long t0 = clock64();
    while ((unsigned long long)(clock64() - t0) < FT_WAIT_LIMIT_CYCLES / 4) __nanosleep(1000);
  }
}

// Rows of the output: each row's partial results in the order of runs and warps, `merge_per_row` warps a
// row (each a contiguous part of them), four dims a lane, eight partials in flight. Bound by latency:
// 1.6 us after its wait for 2048 rows of some six partials each.
template <int NT>
__global__ void __launch_bounds__(32 * MERGE_WARPS) cache_merge_kernel(const __grid_constant__ DecArgs a) {
  __shared__ float4 so[MERGE_WARPS][32];
  __shared__ float2 sml[MERGE_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = a.merge_per_row, rows_here = blockDim.x / 32 / per, part = warp % per;
  const int row = blockIdx.x * rows_here + warp / per, rows = a.B * a.Hk * a.R;  // (b * Hk + h) * R + r
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float M = -INFINITY, L = 0.f;
  int r = 0, h = 0, b = 0, len = 0;
  // The lengths are there: this kernel starts only after every CTA of the first one has waited for what
  // was before it. (Without a first one no key may count, whatever they are.)
  int r0 = 0, lo = 0, hi = 0, f = 0, n = 0, stride = 0;
  long long base = 0;
  Runs runs(0, 0);
  if (row < rows) {
    r = row % a.R;
    h = row / a.R % a.Hk;
    b = row / a.R / a.Hk;
    len = seq_len(a, b);
    const int hg = h * a.n_group + r / (8 * NT), j = hg / a.heads;
    n = seq_cost(a, b);
    runs = Runs(cost_before(a, a.B, lane), a.runs);
    f = cost_before(a, b, lane) + j * n;
    if (n > 0) {
      r0 = runs.owner(f);
      const int cnt = (runs.owner(f + n - 1) + 1 - r0) * a.keys;
      lo = cnt * part / per;
      hi = cnt * (part + 1) / per;
      // partial i: run r0 + i / keys, the warp of this head that is i % keys in turn
      base = (((long long)b * a.per + j + r0) * WARPS + hg - j * a.heads) * (8 * NT) + r % (8 * NT);
      stride = a.heads * 8 * NT;
    }
  }
  pdl_wait();
  pdl_launch();
  for (int i0 = lo; i0 < hi; i0 += 8) {
    float4 v[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
      v[i] = __ldcg(reinterpret_cast<const float4*>(a.part_o + (base + (long long)min(i0 + i, hi - 1) * stride) * HD) + lane);
    float2 ml = make_float2(-INFINITY, 0.f);
    const int mine = i0 + lane;
    if (lane < 8 && mine < hi) {
      // the warp wrote a partial if the run's part of the head reaches its first tile
      const int run = r0 + mine / a.keys, from = max(f, runs.begin(run)) - f, to = min(f + n, runs.begin(run + 1)) - f;
      if (max(0, from - ENTRY) + mine % a.keys * units_of_tile(NT) < to - ENTRY)
        ml = __ldcg(a.part_ml + base + (long long)mine * stride);
    }
    float top = ml.x;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    top = __shfl_sync(0xffffffffu, top, 0);
    const float m_new = max_nan(M, top), ref = m_new == -INFINITY ? 0.f : m_new;
    const float root = M == -INFINITY ? 0.f : root_of_scale(M - ref), al = root * root;
    const bool none = ml.x == -INFINITY;  // nothing was written there, or nothing of it counts
    const float wr = root_of_scale(ml.x - ref), w = none ? -1.f : wr * wr, lw = none ? 0.f : ml.y * wr * wr;
    L = L * root * root;
    M = m_new;
    acc.x *= al;
    acc.y *= al;
    acc.z *= al;
    acc.w *= al;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float wi = __shfl_sync(0xffffffffu, w, i), li = __shfl_sync(0xffffffffu, lw, i);
      if (wi < 0.f) continue;
      L += li;
      acc.x = fmaf(wi, v[i].x, acc.x);
      acc.y = fmaf(wi, v[i].y, acc.y);
      acc.z = fmaf(wi, v[i].z, acc.z);
      acc.w = fmaf(wi, v[i].w, acc.w);
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
      if (sml[warp + i].x == -INFINITY) continue;
      const float wr = root_of_scale(sml[warp + i].x - ref), w = wr * wr;
      const float4 v = so[warp + i][lane];
      acc.x = fmaf(w, v.x, acc.x);
      acc.y = fmaf(w, v.y, acc.y);
      acc.z = fmaf(w, v.z, acc.z);
      acc.w = fmaf(w, v.w, acc.w);
      L += sml[warp + i].y * wr * wr;
    }
  }
  if (row >= rows) return;
  const float inv = 1.f / L;
  uint2 out = make_uint2(pack_bf16x2(acc.x * SUM_UNIT * inv, acc.y * SUM_UNIT * inv),
                         pack_bf16x2(acc.z * SUM_UNIT * inv, acc.w * SUM_UNIT * inv));
  if (len - a.to_end + 1 + r / a.G <= 0) out = make_uint2(0, 0);  // the row sees no key
  *reinterpret_cast<uint2*>(a.o + b * a.o_b + (long long)(r / a.G) * a.o_tok + (long long)(h * a.G + r % a.G) * a.o_h + 4 * lane) = out;
}

int rows_of(const CacheDecodeProblem& p) { return p.Sq * (p.Hq / p.Hk); }
int col_tiles(const CacheDecodeProblem& p) { return rows_of(p) > 8 ? 2 : 1; }
int groups_of(const CacheDecodeProblem& p) { return (rows_of(p) + 8 * col_tiles(p) - 1) / (8 * col_tiles(p)); }

// as many (head, group) units side by side as divide their number
int heads_of(const CacheDecodeProblem& p) {
  const int u = p.Hk * groups_of(p);
  for (int h = WARPS; h > 1; h /= 2)
    if (u % h == 0) return h;
  return 1;
}
long long head_steps_of(const CacheDecodeProblem& p) { return (long long)p.B * (p.Hk * groups_of(p) / heads_of(p)); }
long long partials_of(const CacheDecodeProblem& p) { return (head_steps_of(p) + p.num_sms) * WARPS * 8 * col_tiles(p); }

// One map of a cache side: [128 bytes][heads][tokens][sequences]. A broadcast dimension (stride 0)
// is mapped with one entry.
bool side_map(CUtensorMap* m, const CacheSide& s, const CacheDecodeProblem& p, int& one_b, int& one_h) {
  one_b = p.B == 1 || s.c_b == 0;
  one_h = p.Hk == 1 || s.c_h == 0;
  return make_tmap_4d_u8(m, s.codes, HD, one_h ? 1 : p.Hk, p.L, one_b ? 1 : p.B, one_h ? HD : s.c_h,
                         p.L == 1 ? HD : s.c_tok, one_b ? HD : s.c_b, HD, 1, UNIT, 1);
}

template <int NT, int FMT>
cudaError_t launch_decode(const CUtensorMap& tk, const CUtensorMap& tv, const DecArgs& a, int sms, cudaStream_t stream) {
  const int smem = (int)sizeof(DecSmem<NT>) + 1024;
  static std::atomic<bool> ready[64];  // the attribute belongs to a kernel on one device
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err == cudaSuccess && (dev >= 64 || !ready[dev])) {
    err = cudaFuncSetAttribute(cache_decode_kernel<NT, FMT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (err == cudaSuccess && dev < 64) ready[dev] = true;
  }
  if (err != cudaSuccess) return err;
  return launch_overlapped(cache_decode_kernel<NT, FMT>, dim3((unsigned)sms), 32 * WARPS, smem, stream, tk, tv, a);
}

template <int NT>
cudaError_t launch_merge(const DecArgs& a, cudaStream_t stream) {
  // CTAs of four warps, or of one row's where that is more: small ones fill the SMs evenly
  const int warps = std::max(4, a.merge_per_row), rows_here = warps / a.merge_per_row;
  const int rows = a.B * a.Hk * a.R;
  return launch_overlapped(cache_merge_kernel<NT>, dim3((unsigned)((rows + rows_here - 1) / rows_here)), 32 * warps, 0, stream, a);
}

}  // namespace

size_t cache_decode_scratch_floats(const CacheDecodeProblem& p) { return (size_t)partials_of(p) * (HD + 2); }

CacheDecodePlan cache_decode_plan(CacheDecodeProblem p, size_t most) {
  CacheDecodePlan plan;
  auto bytes = [&] { return cache_decode_scratch_floats(p) * sizeof(float); };
  for (int rest = p.Sq, step = p.Sq; rest > 0; rest -= p.Sq) {
    p.Sq = std::min(step, rest);
    while (p.Sq > 1 && bytes() > most) p.Sq = (p.Sq + 1) / 2;
    if (plan.queries.empty()) step = p.Sq;
    plan.queries.push_back(p.Sq);
    plan.scratch_bytes = std::max(plan.scratch_bytes, bytes());
  }
  return plan;
}

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
  a.to_end = p.Sq + p.later;
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
  a.heads = heads_of(p);
  a.keys = WARPS / a.heads;
  a.per = p.Hk * a.n_group / a.heads;
  a.runs = p.num_sms;
  const long long rows = (long long)p.B * p.Hk * a.R;
  const long long places = head_steps_of(p) * ((p.max_len + UNIT - 1) / UNIT + ENTRY);
  if (rows > 0x3fffffffLL || places > 0x3fffffffLL) return cudaErrorInvalidValue;  // both are numbered in 32 bits
  if (p.scratch == nullptr) return cudaErrorInvalidValue;
  a.part_o = p.scratch;
  a.part_ml = reinterpret_cast<float2*>(p.scratch + (size_t)partials_of(p) * HD);
  // a row has at most about this many partials; warps that share it take a few each
  const long long expect = (a.runs / head_steps_of(p) + 1) * a.keys;
  a.merge_per_row = expect >= 64 ? 16 : expect >= 32 ? 8 : expect >= 16 ? 4 : expect >= 8 ? 2 : 1;
  const bool one = col_tiles(p) == 1;
  if (p.max_len > 0) {  // without keys there may be no memory to map; the merge alone writes the zeros
    CUtensorMap tk, tv;
    if (!side_map(&tk, p.side[0], p, a.one_b[0], a.one_h[0]) || !side_map(&tv, p.side[1], p, a.one_b[1], a.one_h[1]))
      return cudaErrorInvalidValue;
    const bool i8 = p.format == CACHE_INT8;
    const cudaError_t e =
        one ? (i8 ? launch_decode<1, CACHE_INT8>(tk, tv, a, p.num_sms, stream) : launch_decode<1, CACHE_E4M3>(tk, tv, a, p.num_sms, stream))
            : (i8 ? launch_decode<2, CACHE_INT8>(tk, tv, a, p.num_sms, stream) : launch_decode<2, CACHE_E4M3>(tk, tv, a, p.num_sms, stream));
    if (e != cudaSuccess) return e;
  }
  return one ? launch_merge<1>(a, stream) : launch_merge<2>(a, stream);
}

}  // namespace ft
