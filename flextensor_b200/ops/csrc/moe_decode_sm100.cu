// A whole mixture-of-experts feed-forward for a few tokens (at most 64), for sm_100a:
//   ids, w = softmax over the top-k of x router^T
//   out    = residual + sum_k w_k  W_down[e_k] ( silu(x Wg[e_k]^T) * (x Wu[e_k]^T) )
//
// Every weight of every expert that a token chose is read once and meets a handful of tokens, so
// the layer is bound by the HBM stream of the weights. Launches:
//   route    one CTA a token: logits in fp32, top-k, softmax;
//   gate/up  D[weight row, token] = W x^T on tcgen05 (weights are the 128-row operand, the tokens
//            the narrow one), SwiGLU on the accumulator, h in bf16;
//   down     the same product with h, fp32 partial sums;
//   combine  the partial sums of a token's experts with their weights and the residual.
// The two products split the stream of 128-row x 64-column weight tiles of all chosen experts into
// equal contiguous runs, one per CTA (a CTA per SM), whatever the expert and tile boundaries: every
// SM reads the same number of bytes. A weight tile that several CTAs share part of is summed in
// fp32 in the order of the CTAs, by the CTA that finishes last, so results do not depend on timing
// and no CTA waits for another.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>

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
constexpr int NTHREADS = 192;           // warp 0 TMA, 1 MMA, 2-5 epilogue
constexpr int MAX_STAGES = 12;
constexpr int MIN_CHUNKS = 4;           // a CTA takes at least this many weight tiles
constexpr int TMEM_COLS = 2 * MAX_T;    // two accumulators
constexpr int RING_BUDGET = 200 * 1024;

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
  int* ids;                             // [slots] expert of each pair
  float* wts;                           // [slots]
  int* place;                           // [slots] slot | position of its expert among the chosen << 16; [slots] their number
  unsigned int* done;                   // per weight tile of the gate/up product: segments finished
  int n_done;
  __nv_bfloat16* h;                     // [slots, F], slots ordered by expert, then token
  float* part;                          // gate/up: [2 * CTAs][cols][128] partial tiles
  float* y;                             // down: [splits][slots][D] partial sums
  int cols;                             // token columns of an MMA: T rounded up to 16
  int stages, stage_bytes;
  int one_map;                          // the experts' weights are equally spaced: one tensor map
};

template <int N>
struct Maps {
  CUtensorMap w[N];
};

// A wait that runs out (2 s) is recorded; the caller then skips its work but keeps its barriers.
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

// ------------------------------------------------------------------------------------ routing
constexpr int ROUTE_WARPS = 8;

__global__ void __launch_bounds__(32 * ROUTE_WARPS) moe_route_kernel(Args a) {
  __shared__ float logit[MAX_E];
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < a.n_done; i += gridDim.x * blockDim.x) a.done[i] = 0;
  const uint4* x = reinterpret_cast<const uint4*>(a.x + t * a.ldx);
  for (int e = warp; e < a.E; e += ROUTE_WARPS) {
    const uint4* r = reinterpret_cast<const uint4*>(a.router + e * a.ldr);
    float s = 0.f;
#pragma unroll 4
    for (int i = lane; i < a.D / 8; i += 32) {
      const uint4 u = x[i], v = r[i];
      const uint32_t uw[4] = {u.x, u.y, u.z, u.w}, vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; j++) {
        s = fmaf(__uint_as_float(uw[j] << 16), __uint_as_float(vw[j] << 16), s);
        s = fmaf(__uint_as_float(uw[j] & 0xffff0000u), __uint_as_float(vw[j] & 0xffff0000u), s);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) logit[e] = s;
  }
  __syncthreads();
  if (warp != 0) return;
  // top-k by repeated maximum; equal logits go to the lower expert, NaN counts as the largest
  float mine = 0.f, top = 0.f, sum = 0.f;
  int mine_e = 0;
  unsigned int taken = 0;  // this lane's experts lane, lane + 32, ...
  for (int k = 0; k < a.topk; k++) {
    uint32_t best = 0;
    int be = MAX_E;
    for (int i = 0; i * 32 + lane < a.E; i++) {
      if (taken >> i & 1) continue;
      const float v = logit[i * 32 + lane];
      const uint32_t b = __float_as_uint(v);
      const uint32_t key = v != v ? 0xffffffffu : (v == 0.f ? 0x80000000u : (b & 0x80000000u ? ~b : b | 0x80000000u));
      if (key > best || be == MAX_E) {
        best = key;
        be = i * 32 + lane;
      }
    }
    const uint32_t m = __reduce_max_sync(0xffffffffu, be < MAX_E ? best : 0u);
    const int e = (int)__reduce_min_sync(0xffffffffu, be < MAX_E && best == m ? (unsigned)be : (unsigned)MAX_E);
    if ((e & 31) == lane) taken |= 1u << (e >> 5);
    const float v = logit[e];
    if (k == 0) top = v;
    const float p = expf(v - top);
    sum += p;
    if (lane == k) {
      mine = p;
      mine_e = e;
    }
  }
  if (lane < a.topk) {
    a.ids[t * a.topk + lane] = mine_e;
    a.wts[t * a.topk + lane] = mine / sum;
  }
}

// ------------------------------------------------------------------------------------ the products
struct Tables {
  short id[MAX_SLOTS];        // expert of each (token, choice) pair
  short pair[MAX_SLOTS];      // pairs ordered by expert, then token
  short off[MAX_E + 1];       // first slot of each expert
  short act[MAX_E];           // the experts that were chosen
  int n_act;
};

// The stream of weight tiles: item = (chosen expert, row tile), KC tiles along the inner dimension.
struct Stream {
  int rt, kc, ctas;
  long long total;
  __device__ __forceinline__ Stream(int n_act, int row_tiles, int k_chunks, int grid) : rt(row_tiles), kc(k_chunks) {
    total = (long long)n_act * row_tiles * k_chunks;
    ctas = (int)min((long long)grid, max(1LL, total / MIN_CHUNKS));
  }
  __device__ __forceinline__ long long begin(int c) const { return total * c / ctas; }
  // the CTA whose run holds tile i
  __device__ __forceinline__ int owner(long long i) const { return (int)(((i + 1) * ctas - 1) / total); }
};

// expert tables of every CTA, from the router's choices (a few hundred numbers)
__device__ void build_tables(Tables& tb, const Args& a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < a.slots; i += NTHREADS) tb.id[i] = (short)__ldcg(a.ids + i);
  __syncthreads();
  for (int e = warp; e < a.E; e += NTHREADS / 32) {
    int n = 0;
    for (int i = 0; i < a.slots; i += 32) n += __popc(__ballot_sync(0xffffffffu, i + lane < a.slots && tb.id[i + lane] == e));
    if (lane == 0) tb.off[e + 1] = (short)n;
  }
  __syncthreads();
  if (warp == 0) {
    constexpr int PER = MAX_E / 32;
    int n[PER], sum = 0, used = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const int e = lane * PER + i;
      n[i] = e < a.E ? tb.off[e + 1] : 0;
      sum += n[i];
      used += n[i] > 0;
    }
    int s = sum, u = used;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int sv = __shfl_up_sync(0xffffffffu, s, o), uv = __shfl_up_sync(0xffffffffu, u, o);
      if (lane >= o) s += sv, u += uv;
    }
    if (lane == 31) tb.n_act = u;
    if (lane == 0) tb.off[0] = 0;
    s -= sum;
    u -= used;
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const int e = lane * PER + i;
      if (e >= a.E) break;
      s += n[i];
      if (n[i] > 0) tb.act[u++] = (short)e;
      tb.off[e + 1] = (short)s;
    }
  }
  __syncthreads();
  for (int e = warp; e < a.E; e += NTHREADS / 32) {
    int at = tb.off[e];
    if (at == tb.off[e + 1]) continue;
    for (int i = 0; i < a.slots; i += 32) {
      const bool hit = i + lane < a.slots && tb.id[i + lane] == e;
      const unsigned int m = __ballot_sync(0xffffffffu, hit);
      if (hit) tb.pair[at + __popc(m & ((1u << lane) - 1))] = (short)(i + lane);
      at += __popc(m);
    }
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

// UP: the gate/up product (operand x, K = D, 2F weight rows); else the down product (operand h,
// K = F, D weight rows).
template <bool UP, int N_MAPS>
__global__ void __launch_bounds__(NTHREADS, 1)
    moe_product_kernel(const __grid_constant__ CUtensorMap tm_b, const __grid_constant__ Maps<N_MAPS> maps,
                       const __grid_constant__ Args a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ Ctrl sm;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; s++) {
      mbar_init(&sm.full[s], 1);
      mbar_init(&sm.empty[s], 1);
    }
    for (int b = 0; b < 2; b++) {
      mbar_init(&sm.tfull[b], 1);
      mbar_init(&sm.tempty[b], 4);
    }
    mbar_init(&sm.drain, 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&sm.tmem, TMEM_COLS);
    tmem_relinquish();
  }
  build_tables(sm.tb, a);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const Tables& tb = sm.tb;
  const uint32_t tmem_base = sm.tmem;
  const int rows = UP ? 2 * a.F : a.D, K = UP ? a.D : a.F;
  const Stream st(tb.n_act, (rows + BM - 1) / BM, (K + BK - 1) / BK, gridDim.x);
  const int cta = blockIdx.x;
  const long long begin = cta < st.ctas ? st.begin(cta) : 0, end = cta < st.ctas ? st.begin(cta + 1) : 0;

  if (UP && cta == 0) {  // where each pair's row of h and of the partial sums is, for the combine kernel
    for (int ai = warp; ai < tb.n_act; ai += NTHREADS / 32)
      for (int s = tb.off[tb.act[ai]] + lane; s < tb.off[tb.act[ai] + 1]; s += 32) a.place[tb.pair[s]] = s | ai << 16;
    if (threadIdx.x == 0) a.place[a.slots] = tb.n_act;
  }

  if (warp == 0) {
    if (elect_one()) {
      const uint32_t tile_bytes = A_BYTES + a.cols * BK * 2;
      int s = 0;
      uint32_t ph = 0, pend = 0, pend_ph = 0;
      bool ok = true;
      for (long long i = begin; i < end && ok;) {
        const long long item = i / st.kc;
        const int ai = (int)(item / st.rt), rt = (int)(item % st.rt), e = tb.act[ai];
        const long long stop = min(end, (item + 1) * st.kc);
        const CUtensorMap* tm_a = &maps.w[a.one_map ? 0 : e];
        const int z = a.one_map ? e : 0, brow = UP ? 0 : tb.off[e];
        for (int kb = (int)(i - item * st.kc); i < stop; i++, kb++) {
          if (!bounded_wait(&sm.empty[s], ph ^ 1)) {
            ok = false;
            break;
          }
          uint8_t* const dst = ring + (size_t)s * a.stage_bytes;
          mbar_arrive_expect_tx(&sm.full[s], tile_bytes);
          tma_load_3d(dst, tm_a, &sm.full[s], kb * BK, rt * BM, z);
          tma_load_2d(dst + A_BYTES, &tm_b, &sm.full[s], kb * BK, brow);
          pend |= 1u << s;
          pend_ph = (pend_ph & ~(1u << s)) | (ph << s);
          if (++s == a.stages) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      if (!ok) {  // let the copies in flight land before the CTA's shared memory goes away
        const long long t0 = clock64();
        for (int b = 0; b < a.stages; b++)
          if (pend >> b & 1)
            while (!mbar_try_wait(smem_u32(&sm.full[b]), (pend_ph >> b) & 1) &&
                   (unsigned long long)(clock64() - t0) < FT_WAIT_LIMIT_CYCLES / 4) {
            }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = umma_idesc_bf16_f32(BM, 0) | ((uint32_t)(a.cols >> 3) << 17);
      int s = 0, acc = 0;
      uint32_t ph = 0, acc_ph = 0;
      bool ok = true;
      for (long long i = begin; i < end && ok;) {
        const long long first = i, stop = min(end, (i / st.kc + 1) * st.kc);
        if (!bounded_wait(&sm.tempty[acc], acc_ph ^ 1)) break;
        tc_fence_after();
        const uint32_t dt = tmem_base + acc * MAX_T;
        for (; i < stop; i++) {
          if (!bounded_wait(&sm.full[s], ph)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a0 = smem_u32(ring) + s * a.stage_bytes, b0 = a0 + A_BYTES;
#pragma unroll
          for (int k = 0; k < BK / 16; k++)
            umma_bf16_ss(dt, umma_desc_kmajor_sw128(a0 + k * 32), umma_desc_kmajor_sw128(b0 + k * 32), idesc,
                         i != first || k != 0);
          umma_commit(&sm.empty[s]);
          if (++s == a.stages) {
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
  } else {
    const int q = warp & 3, row_in = q * 32 + lane;
    int acc = 0;
    uint32_t acc_ph = 0;
    bool ok = true;  // after a wait that ran out, no accumulator is read, but every barrier below is kept
    for (long long i = begin; i < end;) {
      const long long item = i / st.kc, stop = min(end, (item + 1) * st.kc);
      const int ai = (int)(item / st.rt), row = (int)(item % st.rt) * BM + row_in, e = tb.act[ai];
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
            tmem_ld_x1(src + (UP ? tb.pair[off + j] / a.topk : j), v[u]);
          }
          tmem_ld_wait();
#pragma unroll
          for (int u = 0; u < 8; u++)
            if (j0 + u < n) use(j0 + u, __uint_as_float(v[u]));
        }
      };
      // gate row and up row are neighbouring lanes; four lanes give two outputs of one store
      auto swiglu = [&](int j, float v) {
        const float up = __shfl_down_sync(0xffffffffu, v, 1);
        const float h = v / (1.f + __expf(-v)) * up;
        const float next = __shfl_down_sync(0xffffffffu, h, 2);
        if ((lane & 3) == 0 && row < rows)
          *reinterpret_cast<uint32_t*>(a.h + (long long)(off + j) * a.F + row / 2) = pack_bf16x2(h, next);
      };
      if constexpr (UP) {
        if (whole) {
          columns(swiglu);
        } else {
          const int c0 = st.owner(item * st.kc), c1 = st.owner((item + 1) * st.kc - 1);
          auto tile = [&](int c) {  // a CTA's run cuts at most two tiles: its first and its last
            return a.part + ((long long)(2 * c + (st.begin(c) / st.kc == item ? 0 : 1)) * a.cols) * BM + row_in;
          };
          float* const mine = tile(cta);
          columns([&](int j, float v) { __stcg(mine + (long long)j * BM, v); });
          __threadfence();
          asm volatile("bar.sync 1, 128;" ::: "memory");
          if (threadIdx.x == 64) sm.last = atomicAdd(a.done + item, 1u) == (unsigned)(c1 - c0);
          asm volatile("bar.sync 1, 128;" ::: "memory");
          if (sm.last) {
            __threadfence();
            for (int j = 0; j < n; j++) {
              float v = 0.f;
              for (int c = c0; c <= c1; c++) v += __ldcg(tile(c) + (long long)j * BM);
              swiglu(j, v);
            }
          }
        }
      } else {
        float* const dst = a.y + ((long long)(cta - st.owner(item * st.kc)) * a.slots + off) * a.D + row;
        columns([&](int j, float v) {
          if (row < rows) __stcg(dst + (long long)j * a.D, v);
        });
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.tempty[acc]);
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

__global__ void __launch_bounds__(128) moe_combine_kernel(Args a, int grid) {
  const int t = blockIdx.y, d = (blockIdx.x * 128 + threadIdx.x) * 2;
  if (d >= a.D) return;
  const Stream st(a.place[a.slots], (a.D + BM - 1) / BM, (a.F + BK - 1) / BK, grid);
  float s0 = 0.f, s1 = 0.f;
  for (int k = 0; k < a.topk; k++) {
    const int at = a.place[t * a.topk + k], slot = at & 0xffff;
    const float w = a.wts[t * a.topk + k];
    const long long item = (long long)(at >> 16) * st.rt + d / BM;
    const int n = st.owner((item + 1) * st.kc - 1) - st.owner(item * st.kc) + 1;
    float y0 = 0.f, y1 = 0.f;
    for (int c = 0; c < n; c++) {
      const float2 v = __ldcg(reinterpret_cast<const float2*>(a.y + ((long long)c * a.slots + slot) * a.D + d));
      y0 += v.x;
      y1 += v.y;
    }
    s0 = fmaf(w, y0, s0);
    s1 = fmaf(w, y1, s1);
  }
  if (a.residual) {
    const uint32_t r = *reinterpret_cast<const uint32_t*>(a.residual + t * a.ldres + d);
    s0 += __uint_as_float(r << 16);
    s1 += __uint_as_float(r & 0xffff0000u);
  }
  *reinterpret_cast<uint32_t*>(a.out + t * a.ldo + d) = pack_bf16x2(s0, s1);
}

// ------------------------------------------------------------------------------------ host side
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

struct Layout {
  size_t ids, wts, place, done, h, part, y, bytes;
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
  l.ids = take(slots * 4);
  l.wts = take(slots * 4);
  l.place = take((slots + 1) * 4);
  l.done = take((size_t)l.n_done * 4);
  l.h = take(slots * p.F * 2);
  l.part = take((size_t)p.num_sms * 2 * cols * BM * 4);
  l.y = take((size_t)max_splits(p) * slots * p.D * 4);
  l.bytes = at;
  return l;
}

template <int N>
bool weight_maps(Maps<N>& m, const __nv_bfloat16* const* w, int E, int inner, int rows, long long ld, bool one) {
  if (one)
    return make_tmap_3d_bf16(&m.w[0], w[0], inner, rows, E, ld, E > 1 ? w[1] - w[0] : 0, BK, BM);
  for (int e = 0; e < E; e++)
    if (!make_tmap_3d_bf16(&m.w[e], w[e], inner, rows, 1, ld, 0, BK, BM)) return false;
  return true;
}

// one tensor map serves all experts when their weights lie at equal distances
bool evenly_spaced(const __nv_bfloat16* const* w, int E) {
  if (E == 1) return true;
  const long long d = w[1] - w[0];
  if (d <= 0 || d % 8) return false;
  for (int e = 2; e < E; e++)
    if (w[e] - w[e - 1] != d) return false;
  return true;
}

template <bool UP, int N>
cudaError_t launch_product(const MoeDecodeProblem& p, Args a, cudaStream_t stream) {
  const int inner = UP ? p.D : p.F, rows = UP ? 2 * p.F : p.D;
  const __nv_bfloat16* const* w = UP ? p.w_gate_up : p.w_down;
  Maps<N> maps;
  a.one_map = evenly_spaced(w, p.E);
  if (!weight_maps<N>(maps, w, p.E, inner, rows, UP ? p.ld_gate_up : p.ld_down, a.one_map)) return cudaErrorInvalidValue;
  CUtensorMap tm_b;
  const bool ok = UP ? make_tmap_2d_bf16_swz(&tm_b, p.x, inner, p.T, p.ldx, BK, a.cols, 128)
                     : make_tmap_2d_bf16_swz(&tm_b, a.h, inner, a.slots, p.F, BK, a.cols, 128);
  if (!ok) return cudaErrorInvalidValue;
  const int smem = a.stages * a.stage_bytes + 1024;
  static bool attr = false;
  if (!attr) {
    const cudaError_t e =
        cudaFuncSetAttribute(moe_product_kernel<UP, N>, cudaFuncAttributeMaxDynamicSharedMemorySize, RING_BUDGET + 1024);
    if (e != cudaSuccess) return e;
    attr = true;
  }
  moe_product_kernel<UP, N><<<p.num_sms, NTHREADS, smem, stream>>>(tm_b, maps, a);
  return cudaGetLastError();
}

template <int N>
cudaError_t launch_all(const MoeDecodeProblem& p, const Args& a, cudaStream_t stream) {
  moe_route_kernel<<<p.T, 32 * ROUTE_WARPS, 0, stream>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) e = launch_product<true, N>(p, a, stream);
  if (e == cudaSuccess) e = launch_product<false, N>(p, a, stream);
  if (e != cudaSuccess) return e;
  moe_combine_kernel<<<dim3((p.D + 255) / 256, p.T), 128, 0, stream>>>(a, p.num_sms);
  return cudaGetLastError();
}

}  // namespace

size_t moe_decode_workspace(const MoeDecodeProblem& p) { return layout_of(p).bytes; }

cudaError_t moe_decode(const MoeDecodeProblem& p, cudaStream_t stream) {
  if (p.T <= 0) return cudaSuccess;
  if (p.T > MAX_T || p.E < 1 || p.E > MAX_E || p.topk < 1 || p.topk > MAX_K || p.topk > p.E || p.D < 8 || p.F < 8 ||
      p.D % 8 || p.F % 8 || p.workspace == nullptr)
    return cudaErrorInvalidValue;
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
  a.ids = reinterpret_cast<int*>(ws + l.ids);
  a.wts = reinterpret_cast<float*>(ws + l.wts);
  a.place = reinterpret_cast<int*>(ws + l.place);
  a.done = reinterpret_cast<unsigned int*>(ws + l.done);
  a.n_done = l.n_done;
  a.h = reinterpret_cast<__nv_bfloat16*>(ws + l.h);
  a.part = reinterpret_cast<float*>(ws + l.part);
  a.y = reinterpret_cast<float*>(ws + l.y);
  a.cols = (p.T + 15) / 16 * 16;
  a.stage_bytes = A_BYTES + a.cols * BK * 2;
  a.stages = std::min(MAX_STAGES, RING_BUDGET / a.stage_bytes);
  a.one_map = 0;
  if (p.E <= 8) return launch_all<8>(p, a, stream);
  if (p.E <= 32) return launch_all<32>(p, a, stream);
  return launch_all<MAX_E>(p, a, stream);
}

}  // namespace ft
