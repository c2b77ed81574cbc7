// Windowed attention, dQ (see attn_window.cuh).
//
// One CTA per (128 queries, head, sequence), two per SM, walks the 64-key blocks
// of its window and sinks:
//   S = Q K^T, dP = dO V^T;  dS over S in TMEM;  dQ += dS K
// Warp 0 copies and issues MMAs; the others (two threads a row, 32 key columns
// each) compute dS. dP of the next block runs beside dQ += dS K, the next S after
// it, so the tensor core has no gap of its own between blocks.
//
// 8192 tokens, 16 heads of 128, window 1024: 137 us, 710 TFLOP/s of its 3 products
// (floor 60 us); 8 x 1024 tokens, 12 heads of 64, window 256: 39 us. Bound like
// dK and dV by the two products with A in shared memory.
#include "attn_window.cuh"

namespace dst {
namespace attn_window {

constexpr int kThreads = 32 + 256;

template <int DP>
struct DqCfg {
  static constexpr int kAt = DP / 64;
  static constexpr int kQ = kAt * kRowAtom;   // 128 queries x DP
  static constexpr int kKV = kAt * kBlkAtom;  // 64 keys x DP
  static constexpr int NV = DP == 64 ? 2 : 1;  // value stages; keys have two
  // At head size 128 two CTAs leave no room to align the start by hand; with no
  // static shared memory it lies on a 1024-byte boundary, and the kernel checks.
  static constexpr int kSmem = 2 * kQ + (2 + NV) * kKV + 128;
};

template <int DP>
__global__ void __launch_bounds__(kThreads, 2)
    dq_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmDO,
              const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
              const __grid_constant__ CUtensorMap tmDQ, const float* __restrict__ lse, const float* __restrict__ di,
              const Operand dk, const Operand dv, const SinkChunks sinks, const Shape s) {
  using C = DqCfg<DP>;
  constexpr int NV = C::NV;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int tiles = s.Tp / 128, h = blockIdx.y, b = blockIdx.z, hk = h / s.G;

  if (static_cast<int>(blockIdx.x) >= tiles) {
    // The sums for the sinks of one key block, chunk after chunk.
    if (h % s.G != 0) return;
    const int kb = blockIdx.x - tiles, k0 = kb * 128, rows = min(128, s.S - k0);
    const int first = (last_window_query(s, k0) >> 6) + 1, far = ((s.T - 1) >> 6) - first + 1;
    const int parts = 1 + (far + sinks.steps - 1) / sinks.steps;
    constexpr int V = DP / 32;  // channels a lane; a warp takes a row
    const int c0 = (threadIdx.x & 31) * V;
    const int64_t step = static_cast<int64_t>(sinks.rows) * 2 * DP;
    for (int i = threadIdx.x >> 5; i < 2 * rows; i += kThreads / 32) {
      const int which = i >= rows, r = i - which * rows;
      const float* part = sinks.sums<DP>(b, s.H / s.G, hk, 0, which, k0 + r) + c0;
      float x[V] = {};
#pragma unroll 4
      for (int c = 0; c < parts; ++c) {
#pragma unroll
        for (int j = 0; j < V; j += 2) {
          const float2 y = *reinterpret_cast<const float2*>(part + c * step + j);
          x[j] += y.x;
          x[j + 1] += y.y;
        }
      }
      const Operand& g = which ? dv : dk;
      const float scale = which ? 1.f : s.scale;
      __nv_bfloat16* out = g.p + b * g.s.b + static_cast<int64_t>(k0 + r) * g.s.t + hk * g.s.h + c0;
      if (c0 < s.D)
#pragma unroll
        for (int j = 0; j < V; j += 2)
          *reinterpret_cast<uint32_t*>(out + j) = pack_bf16(x[j] * scale, x[j + 1] * scale);
    }
    return;
  }
  if (smem_u32(smem) & 1023) {
    if (threadIdx.x == 0) record_status(s.status, kBadArgument);
    return;
  }
  uint8_t* sQ = smem;
  uint8_t* sDO = sQ + C::kQ;
  uint8_t* sK = sDO + C::kQ;      // [2]
  uint8_t* sV = sK + 2 * C::kKV;  // [NV]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + NV * C::kKV);
  uint64_t* q_full = bars;
  uint64_t* k_full = bars + 1;  // [2]
  uint64_t* v_full = bars + 3;  // [NV]
  uint64_t* s_full = bars + 5;
  uint64_t* p_full = bars + 6;
  uint64_t* g_full = bars + 7;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 8);

  const int q0 = (tiles - 1 - static_cast<int>(blockIdx.x)) * 128;
  const int warp = __shfl_sync(0xffffffff, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const KeyBlocks<64> blocks(s, q0);
  const int n = blocks.n;

  int ks = 0, vs = 0;  // copies started (warp 0)
  auto load = [&](uint32_t el, const CUtensorMap* map, uint8_t* dst, uint64_t* bar, int j) {
    expect_tx(el, bar, C::kKV);
#pragma unroll
    for (int a = 0; a < C::kAt; ++a) tma_load_4d(el, dst + a * kBlkAtom, map, bar, a * 64, blocks.at(j) * 64, hk, b);
  };
  auto load_k = [&](uint32_t el) { load(el, &tmK, sK + (ks % 2) * C::kKV, &k_full[ks % 2], ks), ++ks; };
  auto load_v = [&](uint32_t el) { load(el, &tmV, sV + (vs % NV) * C::kKV, &v_full[vs % NV], vs), ++vs; };
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&v_full[i], 1);
    }
    mbar_init(s_full, 1);
    mbar_init(p_full, 256);
    mbar_init(g_full, 1);
    fence_barrier_init();
  }
  if (warp == 0) {  // the first copies travel while TMEM is allocated
    __syncwarp();
    const uint32_t el = elect_one();
    expect_tx(el, q_full, 2 * C::kQ);
#pragma unroll
    for (int a = 0; a < C::kAt; ++a) {
      tma_load_4d(el, sDO + a * kRowAtom, &tmDO, q_full, a * 64, q0, h, b);
      tma_load_4d(el, sQ + a * kRowAtom, &tmQ, q_full, a * 64, q0, h, b);
    }
    while (vs < min(n, NV)) load_v(el);
    while (ks < min(n, 2)) load_k(el);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  bool done = warp == 0;  // this thread's part of the result is staged
  const uint32_t tmem = __shfl_sync(0xffffffff, *tmem_slot, 0);
  const uint32_t tDP = tmem + 64, tDQ = tmem + 128;  // S, and dS over it, from 0

  if (warp == 0) {
    const uint32_t el = elect_one();
    constexpr uint32_t id_s = idesc_bf16_f32(128, 64, false, false), id_g = idesc_bf16_f32(128, DP, false, true);
    bool ok = warp_wait(q_full, 0, s.status, kTimeoutTmaFull);
    for (int j = 0; j <= n && ok; ++j) {
      if (j > 0) {
        const int g = j - 1;
        // dP_g has been read by its product
        ok = warp_wait(s_full, g & 1, s.status, kTimeoutTmemFull);
        if (ok && vs < n) load_v(el);
        ok = ok && warp_wait(p_full, g & 1, s.status, kTimeoutTmemFull);
        if (!ok) break;
        tc_fence_after();
        const uint32_t k = desc_lo(sK + (g % 2) * C::kKV, kBlkAtom);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          mma_ts(el, tDQ, tmem + (kk >> 1) * 32 + (kk & 1) * 8, k + ((kk * 2048) >> 4), id_g,
                 (g > 0 || kk > 0) ? 1u : 0u);
        mma_commit(el, g_full);
      }
      if (j < n) {
        if (!(ok = warp_wait(&v_full[j % NV], (j / NV) & 1, s.status, kTimeoutTmaFull))) break;
        product<DP>(el, tDP, sDO, sV + (j % NV) * C::kKV, kBlkAtom, id_s);
        if (j > 0) {  // dS over S, and K of the block before
          ok = warp_wait(g_full, (j - 1) & 1, s.status, kTimeoutTmemFull);
          if (ok && ks < n) load_k(el);
        }
        ok = ok && warp_wait(&k_full[j % 2], (j / 2) & 1, s.status, kTimeoutTmaFull);
        if (!ok) break;
        tc_fence_after();
        product<DP>(el, tmem, sQ, sK + (j % 2) * C::kKV, kBlkAtom, id_s);
        mma_commit(el, s_full);
      }
    }
    if (!ok) {  // a wait expired: no copy may land after the CTA is gone
      for (int j = max(0, ks - 2); j < ks; ++j) mbar_wait(&k_full[j % 2], (j / 2) & 1, s.status, kTimeoutTmaFull);
      for (int j = max(0, vs - NV); j < vs; ++j) mbar_wait(&v_full[j % NV], (j / NV) & 1, s.status, kTimeoutTmaFull);
    }
    __syncwarp();
  } else {
    const int half = (warp - 1) >> 2, quad = warp & 3;
    const int r = quad * 32 + lane, q = q0 + r;
    const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
    const int64_t row = (static_cast<int64_t>(b) * s.H + h) * s.Tp + q;
    const float lq = lse[row], dq_i = di[row];
    const uint32_t t_s = tmem + half * 32 + lane_off, t_dp = t_s + 64;
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      ok = __all_sync(0xffffffff, ok && mbar_wait(s_full, j & 1, s.status, kTimeoutTmemFull));
      if (!ok) break;
      tc_fence_after();
      const int k0 = blocks.at(j) * 64 + half * 32;
      float p[32], ds[32];
      tmem_ld32x2_sync(t_s, t_dp, p, ds);
      if (KeyBlocks<64>::partial<32>(s, q0, k0)) mask_keys(p, s, q, k0);
#pragma unroll
      for (int c = 0; c < 32; ++c) {
        const float e = exp2f(fmaf(p[c], s.scale_log2, -lq));
        // a masked or vanished probability has no gradient, whatever dP is
        ds[c] = e == 0.f ? 0.f : e * (ds[c] - dq_i);
      }
      tmem_put32(t_s, ds);  // over this half's own scores
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(p_full);
    }
    if (__all_sync(0xffffffff, ok && mbar_wait(g_full, (n - 1) & 1, s.status, kTimeoutTmemFull))) {
      tc_fence_after();
#pragma unroll
      for (int ch = 0; ch < DP / 64; ++ch) {
        const int c = half * (DP / 2) + ch * 32;
        float x[32];
        tmem_ld32_sync(tDQ + c + lane_off, x);
        stage_cols(sQ, r, c, x, s.scale);
      }
      fence_proxy_async_smem();
      done = true;
    }
  }
  tc_fence_before();
  if (__syncthreads_and(done) && warp == 0) {
    const uint32_t el = elect_one();
    store_tile<DP>(el, &tmDQ, sQ, q0, h, b);
    if (el) {
      bulk_commit();
      bulk_wait_read<0>();
    }
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

template <int DP>
void launch_dq(const CUtensorMap& q128, const CUtensorMap& dout128, const CUtensorMap& k64, const CUtensorMap& v64,
               const float* lse, const float* di, const CUtensorMap& dq128, const Operand& dk, const Operand& dv,
               int64_t B, const SinkChunks& sinks, const Shape& s, cudaStream_t stream) {
  if (allow_smem<dq_kernel<DP>>(DqCfg<DP>::kSmem) != cudaSuccess) return;
  const dim3 grid(s.Tp / 128 + sinks.blocks, s.H, static_cast<unsigned>(B));
  dq_kernel<DP><<<grid, kThreads, DqCfg<DP>::kSmem, stream>>>(q128, dout128, k64, v64, dq128, lse, di, dk, dv, sinks, s);
}

#define INSTANCE(DP)                                                                                                  \
  template void launch_dq<DP>(const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&,         \
                              const float*, const float*, const CUtensorMap&, const Operand&, const Operand&,         \
                              int64_t,                                                                                \
                              const SinkChunks&, const Shape&, cudaStream_t);
INSTANCE(64)
INSTANCE(128)

}  // namespace attn_window
}  // namespace dst
