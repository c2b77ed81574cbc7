// Windowed attention, dK and dV (see attn_window.cuh).
//
// One CTA per (128 keys, key head, sequence) walks the 64-query blocks that see
// its keys, of every query head of the group:
//   S^T = K Q^T, dP^T = V dO^T;  P^T and dS^T over them in TMEM;
//   dV += P^T dO, dK += dS^T Q
// Warp 0 issues MMAs, warp 1 copies, the others (two threads per key row and
// buffer, 32 query columns each) compute P and dS. At head size 128 the sums take
// half of TMEM and one CTA an SM, which then keeps two blocks in flight in two
// pairs of score buffers; at 64 two CTAs share the SM, one pair each. The scores
// of a block overwrite P and dS of an earlier one, each as soon as its own product
// is done, so the tensor core always has the other one to work on.
//
// 8192 tokens, 16 heads of 128, window 1024, 4 sinks: 187 us, 695 TFLOP/s of its 4
// products (floor 80 us); 8 x 1024 tokens, 12 heads of 64, window 256: 57 us. An MMA
// with N = 64 and A in shared memory is bound by reading A (3x its multiplications),
// which makes about 1100 of the 2300 cycles a step at head size 128. One pair of
// buffers and four warps took 637 us there.
#include "attn_window.cuh"

namespace dst {
namespace attn_window {

template <int DP>
struct DkdvCfg {
  static constexpr int kAt = DP / 64;
  static constexpr int kKV = kAt * kRowAtom;  // 128 keys x DP
  static constexpr int kQ = kAt * kBlkAtom;   // 64 queries x DP
  static constexpr int NB = DP == 64 ? 1 : 2;  // pairs of score buffers
  static constexpr int NS = 3;                 // query stages
  static constexpr int kThreads = 64 + 256 * NB;
  static constexpr int kSmem = 2 * kKV + NS * (2 * kQ + 512) + 1024 + 256;
  static constexpr int kTmem = DP == 64 ? 256 : 512;
  static constexpr int kCtas = DP == 64 ? 2 : 1;
};

template <int DP>
__global__ void __launch_bounds__(DkdvCfg<DP>::kThreads, DkdvCfg<DP>::kCtas)
    dkdv_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmDO,
                const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                const __grid_constant__ CUtensorMap tmDK, const __grid_constant__ CUtensorMap tmDV,
                const float* __restrict__ lse, const float* __restrict__ di, const SinkChunks sinks, const Shape s) {
  using C = DkdvCfg<DP>;
  constexpr int NB = C::NB, NS = C::NS;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sK = smem;
  uint8_t* sV = sK + C::kKV;
  uint8_t* sQ = sV + C::kKV;        // [NS]
  uint8_t* sDO = sQ + NS * C::kQ;   // [NS]
  float* sL = reinterpret_cast<float*>(sDO + NS * C::kQ);  // [NS][64]
  float* sDi = sL + NS * 64;                               // [NS][64]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sDi + NS * 64);
  uint64_t* kv_full = bars;
  uint64_t* q_full = bars + 1;        // [NS]
  uint64_t* q_empty = q_full + NS;    // [NS]
  uint64_t* s_full = q_empty + NS;    // [NB]
  uint64_t* p_full = s_full + NB;     // [NB]
  uint64_t* v_done = p_full + NB;     // [NB] dV += P^T dO: S may be overwritten
  uint64_t* k_done = v_done + NB;     // [NB] dK += dS^T Q: dP may be overwritten
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(k_done + NB);

  // key block and its queries: its window, or a chunk of those past it that see
  // its sinks
  const int key_blocks = s.Tp / 128, extra = static_cast<int>(blockIdx.x) - key_blocks;
  const int kb = extra < 0 ? blockIdx.x : extra / sinks.chunks;
  const int chunk = extra < 0 ? 0 : extra % sinks.chunks + 1;
  const int k0 = kb * 128, hk = blockIdx.y, b = blockIdx.z;
  const bool cut = kb < sinks.blocks;  // this block's sinks have chunks of their own
  const int last_block = (s.T - 1) >> 6;
  int qb0 = k0 >> 6, qb1 = ((cut || k0 >= s.S) ? last_window_query(s, k0) : s.T - 1) >> 6;  // inclusive
  if (chunk > 0) {
    qb0 = qb1 + 1 + (chunk - 1) * sinks.steps;
    qb1 = min(qb0 + sinks.steps - 1, last_block);
    if (qb0 > last_block) return;
  }
  const int nq = qb1 - qb0 + 1, n = nq * s.G;
  const int warp = __shfl_sync(0xffffffff, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 32) {
    mbar_init(kv_full, 1);
    for (int i = 0; i < NS; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
    }
    for (int i = 0; i < NB; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 256);
      mbar_init(&v_done[i], 1);
      mbar_init(&k_done[i], 1);
    }
    fence_barrier_init();
  }
  int loaded = 0;  // query blocks whose copies were started (warp 1)
  auto load_q = [&](uint32_t el) {
    const int st = loaded % NS, h = hk * s.G + loaded / nq, q0 = (qb0 + loaded % nq) * 64;
    expect_tx(el, &q_full[st], 2 * C::kQ + 512);
#pragma unroll
    for (int a = 0; a < C::kAt; ++a) {
      tma_load_4d(el, sQ + st * C::kQ + a * kBlkAtom, &tmQ, &q_full[st], a * 64, q0, h, b);
      tma_load_4d(el, sDO + st * C::kQ + a * kBlkAtom, &tmDO, &q_full[st], a * 64, q0, h, b);
    }
    const int64_t row = (static_cast<int64_t>(b) * s.H + h) * s.Tp + q0;
    if (el) {
      bulk_load(sL + st * 64, lse + row, 256, &q_full[st]);
      bulk_load(sDi + st * 64, di + row, 256, &q_full[st]);
    }
    __syncwarp();
    ++loaded;
  };
  if (warp == 1) {  // the first copies travel while TMEM is allocated
    __syncwarp();
    const uint32_t el = elect_one();
    expect_tx(el, kv_full, 2 * C::kKV);
#pragma unroll
    for (int a = 0; a < C::kAt; ++a) {
      tma_load_4d(el, sK + a * kRowAtom, &tmK, kv_full, a * 64, k0, hk, b);
      tma_load_4d(el, sV + a * kRowAtom, &tmV, kv_full, a * 64, k0, hk, b);
    }
    while (loaded < min(n, NS)) load_q(el);
  }
  if (warp == 0) {
    __syncwarp();
    tmem_alloc(tmem_slot, C::kTmem);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  bool done = warp < 2;  // this thread's part of the result is staged
  const uint32_t tmem = __shfl_sync(0xffffffff, *tmem_slot, 0);
  // pair i: S^T in columns 128 i.., dP^T in 128 i + 64..; then dV, dK
  const uint32_t tDV = tmem + 128 * NB, tDK = tDV + DP;

  if (warp == 1) {
    const uint32_t el = elect_one();
    while (loaded < n && warp_wait(&q_empty[loaded % NS], ((loaded / NS) & 1) ^ 1, s.status, kTimeoutSmemEmpty)) load_q(el);
    // no copy may land after the CTA is gone
    mbar_wait(kv_full, 0, s.status, kTimeoutTmaFull);
    for (int i = max(0, loaded - NS); i < loaded; ++i)
      mbar_wait(&q_full[i % NS], (i / NS) & 1, s.status, kTimeoutTmaFull);
    __syncwarp();
  } else if (warp == 0) {
    constexpr uint32_t id_s = idesc_bf16_f32(128, 64, false, false), id_g = idesc_bf16_f32(128, DP, false, true);
    const uint32_t el = elect_one();
    bool ok = warp_wait(kv_full, 0, s.status, kTimeoutTmaFull);
    for (int i = 0; i < n + NB - 1 && ok; ++i) {
      if (i < n) {
        const int st = i % NS, bf = i % NB;
        const uint32_t ph = ((i / NB) & 1) ^ 1;
        ok = warp_wait(&q_full[st], (i / NS) & 1, s.status, kTimeoutTmaFull) &&
             warp_wait(&v_done[bf], ph, s.status, kTimeoutTmemEmpty);
        if (!ok) break;
        tc_fence_after();
        product<DP>(el, tmem + 128 * bf, sK, sQ + st * C::kQ, kBlkAtom, id_s);
        if (!(ok = warp_wait(&k_done[bf], ph, s.status, kTimeoutTmemEmpty))) break;
        tc_fence_after();
        product<DP>(el, tmem + 128 * bf + 64, sV, sDO + st * C::kQ, kBlkAtom, id_s);
        mma_commit(el, &s_full[bf]);
      }
      const int g = i - (NB - 1);
      if (g >= 0) {
        const int st = g % NS, bf = g % NB;
        if (!(ok = warp_wait(&p_full[bf], (g / NB) & 1, s.status, kTimeoutTmemFull))) break;
        tc_fence_after();
        const uint32_t q = desc_lo(sQ + st * C::kQ, kBlkAtom), go = desc_lo(sDO + st * C::kQ, kBlkAtom);
        // k-step kk: queries 16 kk.., columns of the half that computed them
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          mma_ts(el, tDV, tmem + 128 * bf + (kk >> 1) * 32 + (kk & 1) * 8, go + ((kk * 2048) >> 4), id_g,
                 (g > 0 || kk > 0) ? 1u : 0u);
        mma_commit(el, &v_done[bf]);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          mma_ts(el, tDK, tmem + 128 * bf + 64 + (kk >> 1) * 32 + (kk & 1) * 8, q + ((kk * 2048) >> 4), id_g,
                 (g > 0 || kk > 0) ? 1u : 0u);
        mma_commit(el, &k_done[bf]);
        mma_commit(el, &q_empty[st]);
      }
    }
    __syncwarp();
  } else {
    const int group = (warp - 2) >> 2, bf = group >> 1, half = group & 1, quad = warp & 3;
    const int r = quad * 32 + lane, key = k0 + r;
    const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t t_s = tmem + 128 * bf + half * 32 + lane_off, t_dp = t_s + 64;
    bool ok = true;
    for (int i = bf; i < n; i += NB) {
      const int st = i % NS;
      ok = __all_sync(0xffffffff, ok && mbar_wait(&q_full[st], (i / NS) & 1, s.status, kTimeoutTmaFull) &&
                                      mbar_wait(&s_full[bf], (i / NB) & 1, s.status, kTimeoutTmemFull));
      if (!ok) break;
      tc_fence_after();
      const int q0 = (qb0 + i % nq) * 64;
      const float4* l4 = reinterpret_cast<const float4*>(sL + st * 64 + half * 32);
      const float4* d4 = reinterpret_cast<const float4*>(sDi + st * 64 + half * 32);
      float p[32], ds[32];
      tmem_ld32x2_sync(t_s, t_dp, p, ds);
      // full unless some query comes before a key or is past a key's window
      if (q0 < k0 + 127 || (q0 + 63 - k0 >= s.W && k0 + 128 > s.S)) {
        const int from = key - q0 - half * 32;
        const int to = key < s.S ? 64 : static_cast<int>(min(static_cast<int64_t>(key) + s.W - q0 - half * 32, int64_t(64)));
#pragma unroll
        for (int c = 0; c < 32; ++c)
          if (c < from || c >= to) p[c] = -INFINITY;
      }
#pragma unroll
      for (int c4 = 0; c4 < 8; ++c4) {
        const float4 l = l4[c4], d = d4[c4];
        const float lv[4] = {l.x, l.y, l.z, l.w}, dv4[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = c4 * 4 + e;
          p[c] = exp2f(fmaf(p[c], s.scale_log2, -lv[e]));
          // a masked or vanished probability has no gradient, whatever dP is
          ds[c] = p[c] == 0.f ? 0.f : p[c] * (ds[c] - dv4[e]);
        }
      }
      tmem_put32(t_s, p);  // over this half's own scores
      tmem_put32(t_dp, ds);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&p_full[bf]);
    }
    // every product: the last of each buffer
    for (int i = max(0, n - NB); i < n; ++i)
      ok = __all_sync(0xffffffff, ok && mbar_wait(&k_done[i % NB], (i / NB) & 1, s.status, kTimeoutTmemFull) &&
                                      mbar_wait(&v_done[i % NB], (i / NB) & 1, s.status, kTimeoutTmemFull));
    if (ok) {
      tc_fence_after();
      // 2 NB threads a row, each a share of the columns of dK and dV
      constexpr int kShare = DP / (2 * NB);
      const int c0 = group * kShare;
      // sink rows of a cut block are sums of a chunk only: joined over the stored tile later
      const bool to_partial = cut && key < s.S;
#pragma unroll
      for (int ch = 0; ch < kShare / 32; ++ch) {
        const int c = c0 + ch * 32;
        float x[32];
#pragma unroll
        for (int which = 0; which < 2; ++which) {
          tmem_ld32_sync((which ? tDV : tDK) + c + lane_off, x);
          if (to_partial) {
            float4* dst = reinterpret_cast<float4*>(sinks.sums<DP>(b, gridDim.y, hk, chunk, which, key) + c);
#pragma unroll
            for (int j = 0; j < 8; ++j) dst[j] = make_float4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
          }
          if (chunk == 0) stage_cols(which ? sV : sK, r, c, x, which ? 1.f : s.scale);
        }
      }
      fence_proxy_async_smem();
      done = true;
    }
  }
  tc_fence_before();
  if (__syncthreads_and(done) && warp == 1 && chunk == 0) {
    const uint32_t el = elect_one();
    store_tile<DP>(el, &tmDK, sK, k0, hk, b);
    store_tile<DP>(el, &tmDV, sV, k0, hk, b);
    if (el) {
      bulk_commit();
      bulk_wait_read<0>();
    }
  }
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmem);
  }
}

// di[b, h, t] = sum_d dO O (0 for the rows past the end). DP/8 threads a row. O is the
// result as it was rounded to bf16, which the layer keeps anyway; that adds to the
// gradients' error (these roundings modelled in 64 bits, 1024 tokens, window 256: dQ
// 0.0028 of its norm, with an unrounded O 0.0025, the rest from P and dS; rounding the
// result alone 0.0017). An O in more bits would be one more tensor kept per layer. 8192
// tokens, 16 heads of 128: 15 us, 4.3 TB/s.
template <int DP>
__global__ void rowdot_kernel(const __nv_bfloat16* __restrict__ dout, const __nv_bfloat16* __restrict__ out,
                              float* __restrict__ di, int64_t rows, const Shape s) {
  constexpr int kPer = DP / 8;
  const int64_t gt = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t w = gt / kPer;  // (b, t, h) with t up to Tp, as dO and O lie
  const int part = static_cast<int>(gt % kPer);
  const int h = static_cast<int>(w % s.H), t = static_cast<int>(w / s.H % s.Tp);
  const int64_t b = w / s.H / s.Tp;
  float acc = 0.f;
  if (w < rows && t < s.T && part * 8 < s.D) {
    const int64_t off = ((b * s.T + t) * s.H + h) * s.D + part * 8;
    const uint4 a = *reinterpret_cast<const uint4*>(dout + off);
    const uint4 c = *reinterpret_cast<const uint4*>(out + off);
    const __nv_bfloat162* ah = reinterpret_cast<const __nv_bfloat162*>(&a);
    const __nv_bfloat162* ch = reinterpret_cast<const __nv_bfloat162*>(&c);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 x = __bfloat1622float2(ah[j]), y = __bfloat1622float2(ch[j]);
      acc += x.x * y.x + x.y * y.y;
    }
  }
#pragma unroll
  for (int o = kPer / 2; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffff, acc, o);
  if (w < rows && part == 0) di[(b * s.H + h) * s.Tp + t] = acc;
}

template <int DP>
void launch_rowdot(const __nv_bfloat16* dout, const __nv_bfloat16* out, float* di, int64_t B, const Shape& s,
                   cudaStream_t stream) {
  const int64_t rows = B * s.H * s.Tp;
  rowdot_kernel<DP><<<static_cast<unsigned>((rows * (DP / 8) + 255) / 256), 256, 0, stream>>>(dout, out, di, rows, s);
}

template <int DP>
void launch_dkdv(const CUtensorMap& q64, const CUtensorMap& dout64, const CUtensorMap& k128, const CUtensorMap& v128,
                 const float* lse, const float* di, const CUtensorMap& dk128, const CUtensorMap& dv128, int64_t B,
                 const SinkChunks& sinks, const Shape& s, cudaStream_t stream) {
  using C = DkdvCfg<DP>;
  if (allow_smem<dkdv_kernel<DP>>(C::kSmem) != cudaSuccess) return;
  const dim3 grid(s.Tp / 128 + sinks.blocks * sinks.chunks, s.H / s.G, static_cast<unsigned>(B));
  dkdv_kernel<DP><<<grid, C::kThreads, C::kSmem, stream>>>(q64, dout64, k128, v128, dk128, dv128, lse, di, sinks, s);
}

#define INSTANCES(DP)                                                                                                   \
  template void launch_rowdot<DP>(const __nv_bfloat16*, const __nv_bfloat16*, float*, int64_t, const Shape&,            \
                                  cudaStream_t);                                                                        \
  template void launch_dkdv<DP>(const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&,         \
                                const float*, const float*, const CUtensorMap&, const CUtensorMap&, int64_t,            \
                                const SinkChunks&, const Shape&, cudaStream_t);
INSTANCES(64)
INSTANCES(128)

}  // namespace attn_window
}  // namespace dst
