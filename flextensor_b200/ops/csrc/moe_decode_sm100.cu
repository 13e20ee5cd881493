// A whole mixture-of-experts feed-forward for a few tokens (at most 64), for sm_100a:
//   ids, w = softmax over the top-k of x router^T
//   out    = residual + sum_k w_k  W_down[e_k] ( silu(x Wg[e_k]^T) * (x Wu[e_k]^T) )
//
// Every weight of every expert that a token chose is read once and meets a handful of tokens, so
// the layer is bound by the HBM stream of the weights. Launches:
//   logits   x router^T in fp32, one CTA per expert and four tokens;
//   gate/up  D[weight row, token] = W x^T on tcgen05 (weights are the 128-row operand, the tokens
//            the narrow one), SwiGLU on the accumulator, h as a sum of two bf16 numbers;
//   down     the same product with both parts of h, fp32 partial sums;
//   combine  the partial sums of a token's experts with their weights and the residual.
// Each may start while the one before it ends (programmatic serialization). The choice of experts
// is a few hundred numbers, so every CTA of both products makes it for itself from the logits;
// the down product fills its stages with weights before it waits for h.
// h in one bf16 number would add an error as large as the output's own rounding; its second half
// costs one more MMA per tile and a few KB from L2.
// The two products split the stream of 128-row x 64-column weight tiles of all chosen experts into
// equal contiguous runs, one per CTA (a CTA per SM), whatever the expert and tile boundaries: every
// SM reads the same number of bytes. A weight tile that several CTAs share part of is summed in
// fp32 in the order of the CTAs, by the CTA that finishes last, so results do not depend on timing
// and no CTA waits for another.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "ft_moe_decode.h"
#include "ft_ops.h"
#include "sm100_common.cuh"

namespace ft {

FT_DEFINE_ERROR_READER(moe_decode_device_error)

namespace {

constexpr int BM = 128;                 // weight rows of a tile
constexpr int BK = 64;                  // columns of a tile (128 bytes)
constexpr int A_BYTES = BM * BK * 2;
constexpr int MAX_T = kMoeDecMaxTokens;
constexpr int MAX_E = kMoeDecMaxExperts;
constexpr int MAX_K = kMoeDecMaxTopk;
constexpr int MAX_SLOTS = MAX_T * MAX_K;
constexpr int EPI_WARPS = 4;
constexpr int NTHREADS = 256;           // warp 0 TMA, 1 MMA, 2-5 epilogue; all of them build the tables
constexpr int MAX_STAGES = 12;
constexpr int MIN_CHUNKS = 4;           // a CTA takes at least this many weight tiles
constexpr int TMEM_COLS = 2 * MAX_T;    // two accumulators
constexpr int RING_BUDGET = 200 * 1024;
static_assert(MAX_T * MAX_E * 4 <= RING_BUDGET, "the ring holds the logits first");

struct Args {
  int T, D, F, E, topk, slots;          // slots = T * topk (token, choice) pairs
  const __nv_bfloat16* x;
  long long ldx;
  const __nv_bfloat16* router;
  long long ldr;
  const __nv_bfloat16* residual;
  long long ldres;
  __nv_bfloat16* out;
  long long ldo;
  float* logits;                        // [T, E]
  float* wts;                           // [slots]
  int* place;                           // [slots] slot | position of its expert among the chosen << 16; [slots] their number
  unsigned int* done;                   // per weight tile of the gate/up product: segments finished
  int n_done;
  __nv_bfloat16* h;                     // [2][slots, F], high and low parts, slots ordered by expert, then token
  float* part;                          // gate/up: [2 * CTAs][cols][128] partial tiles
  float* y;                             // down: [splits][slots][D] partial sums
  int cols;                             // token columns of an MMA: T rounded up to 16
  int one_map;                          // one tensor map for all experts
};

template <int N>
struct Maps {
  CUtensorMap w[N];
};

__device__ __forceinline__ void fence_proxy_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ------------------------------------------------------------------------------------ routing
constexpr int LOGIT_WARPS = 8;
constexpr int LOGIT_TOKENS = 4;

// CTA (expert, four tokens): the router's row is read once for the four
__global__ void __launch_bounds__(32 * LOGIT_WARPS) moe_logits_kernel(const __grid_constant__ Args a) {
  __shared__ float part[LOGIT_WARPS][LOGIT_TOKENS];
  const int e = blockIdx.x, t0 = blockIdx.y * LOGIT_TOKENS, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch();
  const int id = (blockIdx.y * gridDim.x + blockIdx.x) * blockDim.x + threadIdx.x;
  for (int i = id; i < a.n_done; i += gridDim.x * gridDim.y * blockDim.x) a.done[i] = 0;
  const uint4* const r = reinterpret_cast<const uint4*>(a.router + e * a.ldr);
  float s[LOGIT_TOKENS] = {};
#pragma unroll 2
  for (int i = threadIdx.x; i < a.D / 8; i += 32 * LOGIT_WARPS) {
    const uint4 v = r[i];
    const uint32_t vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int t = 0; t < LOGIT_TOKENS; t++) {
      const uint4 u = reinterpret_cast<const uint4*>(a.x + min(t0 + t, a.T - 1) * a.ldx)[i];
      const uint32_t uw[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < 4; j++) {
        s[t] = fmaf(__uint_as_float(uw[j] << 16), __uint_as_float(vw[j] << 16), s[t]);
        s[t] = fmaf(__uint_as_float(uw[j] & 0xffff0000u), __uint_as_float(vw[j] & 0xffff0000u), s[t]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < LOGIT_TOKENS; t++) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s[t] += __shfl_xor_sync(0xffffffffu, s[t], o);
    if (lane == 0) part[warp][t] = s[t];
  }
  __syncthreads();
  if (threadIdx.x < LOGIT_TOKENS && t0 + threadIdx.x < a.T) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < LOGIT_WARPS; w++) v += part[w][threadIdx.x];
    a.logits[(t0 + threadIdx.x) * a.E + e] = v;
  }
}

// Two tokens' experts by repeated maximum, by a whole warp (two, because each step waits for the one
// before it): equal logits go to the lower expert, NaN counts as the largest. Lane k < topk gets choice
// k of each and its logit.
template <int PER>  // experts a lane
__device__ __forceinline__ void choose(const Args& a, const float* first, const float* second, int lane, int (&mine_e)[2],
                                       float (&mine)[2]) {
  float v[2][PER];
  uint32_t key[2][PER];
#pragma unroll
  for (int n = 0; n < 2; n++) {
#pragma unroll
    for (int i = 0; i < PER; i++) {
      v[n][i] = i * 32 + lane < a.E ? (n ? second : first)[i * 32 + lane] : 0.f;
      const uint32_t b = __float_as_uint(v[n][i]);
      key[n][i] = v[n][i] != v[n][i] ? 0xffffffffu : (v[n][i] == 0.f ? 0x80000000u : (b & 0x80000000u ? ~b : b | 0x80000000u));
      if (i * 32 + lane >= a.E) key[n][i] = 0;  // below every number: -infinity is 0x007fffff
    }
    mine_e[n] = 0;
    mine[n] = 0.f;
  }
  for (int k = 0; k < a.topk; k++) {
    uint32_t best[2];
    int chosen[2];
    float val[2];
#pragma unroll
    for (int n = 0; n < 2; n++) {
      best[n] = key[n][0];
#pragma unroll
      for (int i = 1; i < PER; i++) best[n] = max(best[n], key[n][i]);
      best[n] = __reduce_max_sync(0xffffffffu, best[n]);
    }
#pragma unroll
    for (int n = 0; n < 2; n++) {
      chosen[n] = 0;
      val[n] = 0.f;
#pragma unroll
      for (int i = PER - 1; i >= 0; i--) {  // the lowest group that holds it, and its lowest lane
        const unsigned int m = __ballot_sync(0xffffffffu, key[n][i] == best[n]);
        if (m) chosen[n] = i * 32 + __ffs(m) - 1, val[n] = v[n][i];
      }
      val[n] = __shfl_sync(0xffffffffu, val[n], chosen[n] & 31);
    }
#pragma unroll
    for (int n = 0; n < 2; n++) {
#pragma unroll
      for (int i = 0; i < PER; i++)
        if (i * 32 + lane == chosen[n]) key[n][i] = 0;
      if (lane == k) {
        mine[n] = val[n];
        mine_e[n] = chosen[n];
      }
    }
  }
}

// ------------------------------------------------------------------------------------ the products
struct Tables {
  short id[MAX_SLOTS];        // expert of each (token, choice) pair
  unsigned long long tokens[MAX_E];  // the tokens that chose each expert: a token chooses it once at most
  int warp_sum[MAX_E / 32];
  short pair[MAX_SLOTS];      // pairs ordered by expert, then token
  short token[MAX_SLOTS];     // and their tokens
  short off[MAX_E + 1];       // first slot of each expert
  short act[MAX_E];           // the experts that were chosen
  unsigned int used[MAX_E / 32];
  int n_act;
  int most;                   // tokens of the expert with the most
};

// The stream of weight tiles (fewer than 2^31: a tile is 16 KB): item = (chosen expert, row tile), kc
// tiles along the inner dimension. CTA c takes tiles [begin(c), begin(c + 1)), the first `rem` CTAs one
// more than the others.
struct Stream {
  int rt, kc, ctas, base, rem;
  __device__ __forceinline__ Stream(int n_act, int row_tiles, int k_chunks, int grid) : rt(row_tiles), kc(k_chunks) {
    const int total = n_act * row_tiles * k_chunks;
    ctas = min(grid, max(1, total / MIN_CHUNKS));
    base = total / ctas;
    rem = total - base * ctas;
  }
  __device__ __forceinline__ int begin(int c) const { return c * base + min(c, rem); }
  // the CTA whose run holds tile i
  __device__ __forceinline__ int owner(int i) const {
    const int longer = rem * (base + 1);
    return i < longer ? i / (base + 1) : rem + (i - longer) / base;
  }
};

// expert tables of every CTA, from the logits, which are brought to shared memory in one go (T * E
// floats, at most 32 KB of the ring that is still idle): tokens read one after the other from global
// memory cost 0.8 us each
__device__ void build_tables(Tables& tb, float* logits, const Args& a, bool keep_weights) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  static_assert(MAX_T == 64 && NTHREADS >= MAX_E, "a mask holds the tokens, a thread an expert");
  if (threadIdx.x == 0) tb.most = 0;
  if (threadIdx.x < MAX_E) tb.tokens[threadIdx.x] = 0;
#pragma unroll 4
  for (int i = threadIdx.x; i < a.T * a.E; i += NTHREADS) logits[i] = __ldcg(a.logits + i);
  __syncthreads();
  for (int t = warp; t < a.T; t += 2 * (NTHREADS / 32)) {
    const int u = t + NTHREADS / 32, us = min(u, a.T - 1);  // the second token, if there is one
    int e[2];
    float v[2];
    if (a.E <= 32) choose<1>(a, logits + t * a.E, logits + us * a.E, lane, e, v);
    else choose<MAX_E / 32>(a, logits + t * a.E, logits + us * a.E, lane, e, v);
#pragma unroll
    for (int n = 0; n < 2; n++) {
      const int token = n ? u : t;
      const bool mine = lane < a.topk && token < a.T;
      if (mine) {
        tb.id[token * a.topk + lane] = (short)e[n];
        atomicOr(&tb.tokens[e[n]], 1ull << token);
      }
      if (keep_weights) {  // softmax over the choices; the first is the largest
        const float top = __shfl_sync(0xffffffffu, v[n], 0);  // by every lane: a shuffle in a branch would wait for the others
        const float p = lane < a.topk ? expf(v[n] - top) : 0.f;
        float sum = p;
#pragma unroll
        for (int o = MAX_K / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (mine) a.wts[token * a.topk + lane] = p / sum;
      }
    }
  }
  __syncthreads();
  // experts: first slots and the list of the chosen, by a scan over four warps
  int count = 0, scan = 0;
  unsigned int used = 0;
  if (threadIdx.x < MAX_E) {
    count = __popcll(tb.tokens[threadIdx.x]);  // none for those that do not exist
    scan = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += up;
    }
    used = __ballot_sync(0xffffffffu, count > 0);
    const int most = __reduce_max_sync(0xffffffffu, count);
    if (lane == 31) tb.warp_sum[warp] = scan;
    if (lane == 0) {
      tb.used[warp] = used;
      atomicMax(&tb.most, most);
    }
  }
  __syncthreads();
  if (threadIdx.x < MAX_E) {
    int off = scan - count, at = __popc(used & ((1u << lane) - 1));
    for (int w = 0; w < warp; w++) off += tb.warp_sum[w], at += __popc(tb.used[w]);
    tb.off[threadIdx.x] = (short)off;
    if (count > 0) tb.act[at] = (short)threadIdx.x;
    if (threadIdx.x == MAX_E - 1) {
      tb.off[MAX_E] = (short)a.slots;
      tb.n_act = at + (count > 0);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.slots; i += NTHREADS) {  // a pair's slot: its expert's first, and the earlier tokens there
    const int e = tb.id[i], t = i / a.topk, at = tb.off[e] + __popcll(tb.tokens[e] & ((1ull << t) - 1));
    tb.pair[at] = (short)i;
    tb.token[at] = (short)t;
  }
  __syncthreads();
}

struct Ctrl {
  Tables tb;
  uint64_t full[MAX_STAGES], empty[MAX_STAGES], tfull[2], tempty[2], drain;
  uint32_t tmem;
  int last;
};

__device__ __forceinline__ void tmem_ld_x1(uint32_t taddr, uint32_t& r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr));
}

// Bound by HBM: at the Mixtral-8x22B shape with one token the gate/up product streams 805 MB in 121 us
// and the down product 403 MB in 61 us (6.6 TB/s both, above the rate of a copy), the whole layer 1208
// MB in 192 us; 64 experts of 2048 x 1024 and 7 tokens, 401 MB on average, take 78 us, of which about
// 20 us are the four launches' latencies.
// UP: the gate/up product (operand x, K = D, 2F weight rows); else the down product (operand h,
// K = F, D weight rows).
template <bool UP, int N_MAPS>
__global__ void __launch_bounds__(NTHREADS, 1)
    moe_product_kernel(const __grid_constant__ CUtensorMap tm_b, const __grid_constant__ CUtensorMap tm_lo,
                       const __grid_constant__ Maps<N_MAPS> maps, const __grid_constant__ Args a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ Ctrl sm;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < MAX_STAGES; s++) {
      mbar_init(&sm.full[s], 1);
      mbar_init(&sm.empty[s], 1);
    }
    for (int b = 0; b < 2; b++) {
      mbar_init(&sm.tfull[b], 1);
      mbar_init(&sm.tempty[b], EPI_WARPS);
    }
    mbar_init(&sm.drain, 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&sm.tmem, TMEM_COLS);
    tmem_relinquish();
  }
  // The logits are there: the gate/up product waits for their kernel, and the down product starts
  // only after every CTA of the gate/up product has done so.
  if (UP) {
    pdl_wait();
    pdl_launch();
  }
  build_tables(sm.tb, reinterpret_cast<float*>(ring), a, UP && blockIdx.x == 0);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const Tables& tb = sm.tb;
  const uint32_t tmem_base = sm.tmem;
  const int rows = UP ? 2 * a.F : a.D, K = UP ? a.D : a.F;
  const Stream st(tb.n_act, (rows + BM - 1) / BM, (K + BK - 1) / BK, gridDim.x);
  // a stage holds a weight tile and the token columns that go with it, for the down product both parts
  // of the rows of the largest group
  const int cols = UP ? a.cols : (tb.most + 15) / 16 * 16, stage_bytes = A_BYTES + cols * 128 * (UP ? 1 : 2);
  const int stages = min(MAX_STAGES, RING_BUDGET / stage_bytes);
  const int cta = blockIdx.x;
  const int begin = cta < st.ctas ? st.begin(cta) : 0, end = cta < st.ctas ? st.begin(cta + 1) : 0;

  if (UP && cta == 0) {  // where each pair's row of h and of the partial sums is, for the combine kernel
    for (int s = threadIdx.x; s < a.slots; s += NTHREADS) {
      const int e = tb.id[tb.pair[s]];
      int ai = __popc(tb.used[e / 32] & ((1u << (e % 32)) - 1));  // its place among the chosen experts
      for (int w = 0; w < e / 32; w++) ai += __popc(tb.used[w]);
      a.place[tb.pair[s]] = s | ai << 16;
    }
    if (threadIdx.x == 0) a.place[a.slots] = tb.n_act;
  }

  if (warp == 0) {
    if (elect_one()) {
      fence_proxy_async_shared();  // the ring held the logits
      int s = 0;
      uint32_t ph = 0, pend = 0, pend_ph = 0;
      bool ok = true;
      // weights of tile i of the run, tokens of it: a down tile takes both parts of the expert's rows of h, 16 a copy
      auto place_of = [&](int i, int& ai, int& rt, int& kb) {
        const int item = i / st.kc;
        ai = item / st.rt;
        rt = item - ai * st.rt;
        kb = i - item * st.kc;
      };
      auto tokens_bytes = [&](int e) {
        return UP ? cols * 128 : (tb.off[e + 1] - tb.off[e] + 15) / 16 * (2 * 16 * 128);
      };
      auto load_weights = [&](int s, int e, int rt, int kb) {
        mbar_arrive_expect_tx(&sm.full[s], A_BYTES + tokens_bytes(e));
        tma_load_3d(ring + (size_t)s * stage_bytes, &maps.w[a.one_map ? 0 : e], &sm.full[s], kb * BK, rt * BM, a.one_map ? e : 0);
      };
      auto load_tokens = [&](int s, int e, int kb) {
        uint8_t* const dst = ring + (size_t)s * stage_bytes + A_BYTES;
        if (UP) {
          tma_load_2d(dst, &tm_b, &sm.full[s], kb * BK, 0);
        } else {
          for (int r = tb.off[e], at = 0; r < tb.off[e + 1]; r += 16, at += 16 * 128) {
            tma_load_2d(dst + at, &tm_b, &sm.full[s], kb * BK, r);
            tma_load_2d(dst + cols * 128 + at, &tm_lo, &sm.full[s], kb * BK, r);
          }
        }
      };
      int i = begin;
      if (!UP) {  // the first stages' weights do not depend on h
        const int n = min(stages, end - begin);
        int ai, rt, kb;
        for (int b = 0; b < n; b++) {
          place_of(begin + b, ai, rt, kb);
          load_weights(b, tb.act[ai], rt, kb);
        }
        pdl_wait();
        fence_proxy_async_global();
        for (int b = 0; b < n; b++) {
          place_of(begin + b, ai, rt, kb);
          load_tokens(b, tb.act[ai], kb);
        }
        i += n;
        pend = (1u << n) - 1;
        s = n % stages;
        ph = n == stages;
      }
      while (i < end && ok) {
        int ai, rt, kb;
        place_of(i, ai, rt, kb);
        const int e = tb.act[ai];
        const int stop = min(end, i - kb + st.kc);
        for (; i < stop; i++, kb++) {
          if (!bounded_wait(&sm.empty[s], ph ^ 1)) {
            ok = false;
            break;
          }
          load_weights(s, e, rt, kb);
          load_tokens(s, e, kb);
          pend |= 1u << s;
          pend_ph = (pend_ph & ~(1u << s)) | (ph << s);
          if (++s == stages) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      if (!ok) {  // let the copies in flight land before the CTA's shared memory goes away
        const long long t0 = clock64();
        for (int b = 0; b < stages; b++)
          if (pend >> b & 1)
            while (!mbar_try_wait(smem_u32(&sm.full[b]), (pend_ph >> b) & 1) &&
                   (unsigned long long)(clock64() - t0) < FT_WAIT_LIMIT_CYCLES / 4) {
            }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      int s = 0, acc = 0;
      uint32_t ph = 0, acc_ph = 0;
      bool ok = true;
      for (int i = begin; i < end && ok;) {
        const int first = i, item = i / st.kc, stop = min(end, (item + 1) * st.kc);
        if (!bounded_wait(&sm.tempty[acc], acc_ph ^ 1)) break;
        tc_fence_after();
        const uint32_t dt = tmem_base + acc * MAX_T;
        const int e = tb.act[item / st.rt];
        const int here = UP ? cols : (tb.off[e + 1] - tb.off[e] + 15) / 16 * 16;
        const uint32_t idesc = umma_idesc_bf16_f32(BM, 0) | ((uint32_t)(here >> 3) << 17);
        for (; i < stop; i++) {
          if (!bounded_wait(&sm.full[s], ph)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a0 = smem_u32(ring) + s * stage_bytes, b0 = a0 + A_BYTES;
#pragma unroll
          for (int k = 0; k < BK / 16; k++)
            umma_bf16_ss(dt, umma_desc_kmajor_sw128(a0 + k * 32), umma_desc_kmajor_sw128(b0 + k * 32), idesc,
                         i != first || k != 0);
          if constexpr (!UP) {
            const uint32_t l0 = b0 + cols * 128;
#pragma unroll
            for (int k = 0; k < BK / 16; k++)
              umma_bf16_ss(dt, umma_desc_kmajor_sw128(a0 + k * 32), umma_desc_kmajor_sw128(l0 + k * 32), idesc, 1);
          }
          umma_commit(&sm.empty[s]);
          if (++s == stages) {
            s = 0;
            ph ^= 1;
          }
        }
        if (!ok) break;
        umma_commit(&sm.tfull[acc]);
        acc ^= 1;
        if (acc == 0) acc_ph ^= 1;
      }
      if (!ok) {
        umma_commit(&sm.drain);
        const long long t0 = clock64();
        while (!mbar_try_wait(smem_u32(&sm.drain), 0) &&
               (unsigned long long)(clock64() - t0) < FT_WAIT_LIMIT_CYCLES / 4) {
        }
      }
    }
  } else if (warp < 2 + EPI_WARPS) {
    if (!UP) {
      pdl_wait();  // the partial sums' memory may be in use until here
      pdl_launch();
    }
    const int q = warp & 3, row_in = q * 32 + lane;
    int acc = 0;
    uint32_t acc_ph = 0;
    bool ok = true;  // after a wait that ran out, no accumulator is read, but every barrier below is kept
    for (int i = begin; i < end;) {
      const int item = i / st.kc, stop = min(end, (item + 1) * st.kc);
      const int ai = item / st.rt, row = (item - ai * st.rt) * BM + row_in, e = tb.act[ai];
      const int off = tb.off[e], n = tb.off[e + 1] - off;
      const bool whole = stop - i == st.kc;
      if (ok) ok = __all_sync(0xffffffffu, bounded_wait(&sm.tfull[acc], acc_ph));
      tc_fence_after();
      const uint32_t src = tmem_base + acc * MAX_T + ((uint32_t)(q * 32) << 16);
      // this warp's 32 rows x the expert's tokens, eight columns at a time
      auto columns = [&](auto&& use) {
        if (!ok) return;
        for (int j0 = 0; j0 < n; j0 += 8) {
          uint32_t v[8];
#pragma unroll
          for (int u = 0; u < 8; u++) {
            const int j = min(j0 + u, n - 1);
            tmem_ld_x1(src + (UP ? tb.token[off + j] : j), v[u]);
          }
          tmem_ld_wait();
#pragma unroll
          for (int u = 0; u < 8; u++)
            if (j0 + u < n) use(j0 + u, __uint_as_float(v[u]));
        }
      };
      auto release = [&]() {  // the accumulator may be written again
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.tempty[acc]);
      };
      // gate row and up row are neighbouring lanes; four lanes give two outputs of one store
      auto swiglu = [&](int j, float v) {
        const float up = __shfl_down_sync(0xffffffffu, v, 1);
        const float h = v / (1.f + __expf(-v)) * up;
        const float next = __shfl_down_sync(0xffffffffu, h, 2);
        if ((lane & 3) == 0 && row < rows) {
          const uint32_t hi = pack_bf16x2(h, next);
          auto rest = [](float x, uint32_t bits) {  // an infinite high part is the whole of it
            return (bits & 0x7f800000u) == 0x7f800000u ? 0.f : x - __uint_as_float(bits);
          };
          __nv_bfloat16* const dst = a.h + (long long)(off + j) * a.F + row / 2;
          *reinterpret_cast<uint32_t*>(dst) = hi;
          *reinterpret_cast<uint32_t*>(dst + (long long)a.slots * a.F) =
              pack_bf16x2(rest(h, hi << 16), rest(next, hi & 0xffff0000u));
        }
      };
      if constexpr (UP) {
        if (whole) {
          columns(swiglu);
          release();
        } else {
          const int c0 = st.owner(item * st.kc), c1 = st.owner((item + 1) * st.kc - 1);
          auto tile = [&](int c) {  // a CTA's run cuts at most two tiles: its first and its last
            return a.part + ((long long)(2 * c + (st.begin(c) / st.kc == item ? 0 : 1)) * a.cols) * BM + row_in;
          };
          float* const mine = tile(cta);
          columns([&](int j, float v) { __stcg(mine + (long long)j * BM, v); });
          release();
          asm volatile("bar.sync 1, %0;" ::"n"(32 * EPI_WARPS) : "memory");  // with the fence: every thread's part is there before the count
          if (threadIdx.x == 64) {
            __threadfence();
            sm.last = atomicAdd(a.done + item, 1u) == (unsigned)(c1 - c0);
            __threadfence();
          }
          asm volatile("bar.sync 1, %0;" ::"n"(32 * EPI_WARPS) : "memory");
          if (sm.last) {
            constexpr int COLS = 8;  // columns in flight, of two runs
            for (int j0 = 0; j0 < n; j0 += COLS) {
              float v[COLS] = {};
              for (int c = c0; c <= c1; c += 2) {
                const float *const from = tile(c), *const next = tile(min(c + 1, c1));
                float x[COLS], y[COLS];
#pragma unroll
                for (int u = 0; u < COLS; u++) {
                  x[u] = __ldcg(from + (long long)min(j0 + u, n - 1) * BM);
                  y[u] = __ldcg(next + (long long)min(j0 + u, n - 1) * BM);
                }
#pragma unroll
                for (int u = 0; u < COLS; u++) {
                  v[u] += x[u];
                  if (c < c1) v[u] += y[u];
                }
              }
#pragma unroll
              for (int u = 0; u < COLS; u++)
                if (j0 + u < n) swiglu(j0 + u, v[u]);
            }
          }
        }
      } else {
        float* const dst = a.y + ((long long)(cta - st.owner(item * st.kc)) * a.slots + off) * a.D + row;
        columns([&](int j, float v) {
          if (row < rows) __stcg(dst + (long long)j * a.D, v);
        });
        release();
      }
      acc ^= 1;
      if (acc == 0) acc_ph ^= 1;
      i = stop;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

__global__ void __launch_bounds__(128) moe_combine_kernel(const __grid_constant__ Args a, int grid) {
  const int t = blockIdx.y, d = (blockIdx.x * 128 + threadIdx.x) * 2;
  // The choices and the residual are there: this kernel starts only after every CTA of the down product
  // has waited for the gate/up product. Only the partial sums are read after its own wait, the first
  // two of every choice before their first use.
  const bool mine = d < a.D;
  int at[MAX_K], n[MAX_K];
  float w[MAX_K];
#pragma unroll
  for (int k = 0; k < MAX_K; k++) {
    const int i = t * a.topk + min(k, a.topk - 1);
    at[k] = __ldcg(a.place + i);
    w[k] = __ldcg(a.wts + i);
  }
  const uint32_t r = a.residual && mine ? *reinterpret_cast<const uint32_t*>(a.residual + t * a.ldres + d) : 0u;
  const Stream st(__ldcg(a.place + a.slots), (a.D + BM - 1) / BM, (a.F + BK - 1) / BK, grid);
#pragma unroll
  for (int k = 0; k < MAX_K; k++) {
    const int item = (at[k] >> 16) * st.rt + min(d, a.D - 1) / BM;
    n[k] = st.owner((item + 1) * st.kc - 1) - st.owner(item * st.kc) + 1;
    at[k] &= 0xffff;
  }
  pdl_wait();
  pdl_launch();
  if (!mine) return;
  const float* const y = a.y + d;
  const long long part = (long long)a.slots * a.D;
  float2 v[MAX_K], u[MAX_K];
#pragma unroll
  for (int k = 0; k < MAX_K; k++) {
    if (k >= a.topk) break;
    v[k] = __ldcg(reinterpret_cast<const float2*>(y + (long long)at[k] * a.D));
    u[k] = make_float2(0.f, 0.f);
    if (n[k] > 1) u[k] = __ldcg(reinterpret_cast<const float2*>(y + part + (long long)at[k] * a.D));
  }
  float s0 = 0.f, s1 = 0.f;
#pragma unroll
  for (int k = 0; k < MAX_K; k++) {
    if (k >= a.topk) break;
    float y0 = v[k].x + u[k].x, y1 = v[k].y + u[k].y;
    for (int c = 2; c < n[k]; c++) {
      const float2 x = __ldcg(reinterpret_cast<const float2*>(y + c * part + (long long)at[k] * a.D));
      y0 += x.x;
      y1 += x.y;
    }
    s0 = fmaf(w[k], y0, s0);
    s1 = fmaf(w[k], y1, s1);
  }
  s0 += __uint_as_float(r << 16);
  s1 += __uint_as_float(r & 0xffff0000u);
  *reinterpret_cast<uint32_t*>(a.out + t * a.ldo + d) = pack_bf16x2(s0, s1);
}

// ------------------------------------------------------------------------------------ host side
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

struct Layout {
  size_t logits, wts, place, done, h, part, y, bytes;
  int n_done;
};

// CTAs that can share one row tile of the down product. Runs are at least m tiles long: MIN_CHUNKS,
// or total / SMs where that is more, and a token's topk experts differ, so at least topk are chosen.
int max_splits(const MoeDecodeProblem& p) {
  const long long rt = (p.D + BM - 1) / BM, kc = (p.F + BK - 1) / BK;
  const long long m = std::max<long long>(MIN_CHUNKS, rt * kc * p.topk / p.num_sms);
  return (int)((kc - 1 + m - 1) / m + 1);
}

Layout layout_of(const MoeDecodeProblem& p) {
  Layout l;
  const size_t slots = (size_t)p.T * p.topk, cols = (p.T + 15) / 16 * 16;
  l.n_done = (int)(std::min<size_t>(p.E, slots) * ((2 * (size_t)p.F + BM - 1) / BM));
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t r = at;
    at += up256(n);
    return r;
  };
  l.logits = take((size_t)p.T * p.E * 4);
  l.wts = take(slots * 4);
  l.place = take((slots + 1) * 4);
  l.done = take((size_t)l.n_done * 4);
  l.h = take(2 * slots * p.F * 2);
  l.part = take((size_t)p.num_sms * 2 * cols * BM * 4);
  l.y = take((size_t)max_splits(p) * slots * p.D * 4);
  l.bytes = at;
  return l;
}

// N = 1: the experts' weights lie at equal distances and one map covers them all
template <int N>
bool weight_maps(Maps<N>& m, const __nv_bfloat16* const* w, int E, int inner, int rows, long long ld) {
  if constexpr (N == 1) {
    return make_tmap_3d_bf16(&m.w[0], w[0], inner, rows, E, ld, E > 1 ? w[1] - w[0] : 0, BK, BM);
  } else {
    for (int e = 0; e < E; e++)
      if (!make_tmap_3d_bf16(&m.w[e], w[e], inner, rows, 1, ld, 0, BK, BM)) return false;
    return true;
  }
}

template <bool UP, int N>
cudaError_t launch_product(const MoeDecodeProblem& p, Args a, cudaStream_t stream) {
  const int inner = UP ? p.D : p.F, rows = UP ? 2 * p.F : p.D;
  const __nv_bfloat16* const* w = UP ? p.w_gate_up : p.w_down;
  Maps<N> maps;
  a.one_map = N == 1;
  if (!weight_maps<N>(maps, w, p.E, inner, rows, UP ? p.ld_gate_up : p.ld_down)) return cudaErrorInvalidValue;
  CUtensorMap tm_b, tm_lo;
  bool ok;
  if (UP) {
    ok = make_tmap_2d_bf16_swz(&tm_b, p.x, inner, p.T, p.ldx, BK, a.cols, 128);
    tm_lo = tm_b;
  } else {
    ok = make_tmap_2d_bf16_swz(&tm_b, a.h, inner, a.slots, p.F, BK, 16, 128) &&
         make_tmap_2d_bf16_swz(&tm_lo, a.h + (size_t)a.slots * p.F, inner, a.slots, p.F, BK, 16, 128);
  }
  if (!ok) return cudaErrorInvalidValue;
  const int smem = RING_BUDGET + 1024;
  static std::atomic<bool> ready[64];  // the attribute belongs to a kernel on one device
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err == cudaSuccess && (dev >= 64 || !ready[dev])) {
    err = cudaFuncSetAttribute(moe_product_kernel<UP, N>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (err == cudaSuccess && dev < 64) ready[dev] = true;
  }
  if (err != cudaSuccess) return err;
  return launch_overlapped(moe_product_kernel<UP, N>, dim3((unsigned)p.num_sms), NTHREADS, smem, stream, tm_b, tm_lo, maps, a);
}

template <bool UP>
cudaError_t launch_product_for(const MoeDecodeProblem& p, const Args& a, cudaStream_t stream) {
  if (moe_decode_one_map(UP ? p.w_gate_up : p.w_down, p.E)) return launch_product<UP, 1>(p, a, stream);
  if (p.E <= 8) return launch_product<UP, 8>(p, a, stream);
  if (p.E <= 32) return launch_product<UP, 32>(p, a, stream);
  return launch_product<UP, MAX_E>(p, a, stream);
}

}  // namespace

bool moe_decode_one_map(const __nv_bfloat16* const* w, int E) {
  if (E == 1) return true;
  const long long d = reinterpret_cast<intptr_t>(w[1]) - reinterpret_cast<intptr_t>(w[0]);  // bytes
  if (d <= 0 || d % 16 || d >= (1LL << 40)) return false;
  for (int e = 2; e < E; e++)
    if (reinterpret_cast<intptr_t>(w[e]) - reinterpret_cast<intptr_t>(w[e - 1]) != d) return false;
  return true;
}

size_t moe_decode_workspace(const MoeDecodeProblem& p) { return layout_of(p).bytes; }

cudaError_t moe_decode(const MoeDecodeProblem& p, cudaStream_t stream) {
  if (p.T <= 0) return cudaSuccess;
  if (p.T > MAX_T || p.E < 1 || p.E > MAX_E || p.topk < 1 || p.topk > MAX_K || p.topk > p.E || p.D < 8 || p.F < 8 ||
      p.D % 8 || p.F % 8 || p.workspace == nullptr)
    return cudaErrorInvalidValue;
  // tiles are numbered in 32 bits
  const long long tiles = (long long)p.E * std::max(((2 * p.F + BM - 1) / BM) * (long long)((p.D + BK - 1) / BK),
                                                    ((p.D + BM - 1) / BM) * (long long)((p.F + BK - 1) / BK));
  if (tiles > 0x7fffffffLL) return cudaErrorInvalidValue;
  const Layout l = layout_of(p);
  uint8_t* const ws = static_cast<uint8_t*>(p.workspace);
  Args a;
  a.T = p.T;
  a.D = p.D;
  a.F = p.F;
  a.E = p.E;
  a.topk = p.topk;
  a.slots = p.T * p.topk;
  a.x = p.x;
  a.ldx = p.ldx;
  a.router = p.router;
  a.ldr = p.ldr;
  a.residual = p.residual;
  a.ldres = p.ldres;
  a.out = p.out;
  a.ldo = p.ldo;
  a.logits = reinterpret_cast<float*>(ws + l.logits);
  a.wts = reinterpret_cast<float*>(ws + l.wts);
  a.place = reinterpret_cast<int*>(ws + l.place);
  a.done = reinterpret_cast<unsigned int*>(ws + l.done);
  a.n_done = l.n_done;
  a.h = reinterpret_cast<__nv_bfloat16*>(ws + l.h);
  a.part = reinterpret_cast<float*>(ws + l.part);
  a.y = reinterpret_cast<float*>(ws + l.y);
  a.cols = (p.T + 15) / 16 * 16;
  cudaError_t e = launch_overlapped(moe_logits_kernel, dim3((unsigned)p.E, (unsigned)((p.T + LOGIT_TOKENS - 1) / LOGIT_TOKENS)),
                                    32 * LOGIT_WARPS, 0, stream, a);
  if (e == cudaSuccess) e = launch_product_for<true>(p, a, stream);
  if (e == cudaSuccess) e = launch_product_for<false>(p, a, stream);
  if (e != cudaSuccess) return e;
  return launch_overlapped(moe_combine_kernel, dim3((unsigned)((p.D + 255) / 256), (unsigned)p.T), 128, 0, stream, a, p.num_sms);
}

}  // namespace ft
