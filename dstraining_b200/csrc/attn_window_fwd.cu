// Windowed attention, forward (see attn_window.cuh).
//
// One CTA per (128 queries, head, sequence), two per SM, blocks of 64 keys in two
// score buffers: warp 0 copies and issues S = Q K^T and O += P V; warps 1-4 and
// 5-8 are the softmax of the left and the right 32 columns of a block, a thread
// per row. Scores of the next block are computed while the softmax works on this
// one. The two halves of a row only meet where its maximum may have to move: a row
// keeps its reference maximum until a block exceeds it by 8 (in log2), so P stays
// below 2^8 and in most blocks one barrier between two warps is all they exchange.
//
// 8192 tokens, 16 heads of 128, window 1024: 94 us, 690 TFLOP/s of the visible
// pairs (floor 40 us of tensor time); 8 x 1024 tokens, 12 heads of 64, window 256:
// 34 us. A block takes about 800 cycles of an SM: 512 of them the exponentials (16 a
// cycle; at head size 128 the tensor core needs as much), the rest the chain from
// scores to sums where two tiles do not fill each other's gaps; 3 to 5 thousand
// cycles a tile go to start and end. Tried: blocks of 128 keys (121 us: one score
// buffer, the chain is exposed), a thread per row (144 us).
#include "attn_window.cuh"

namespace dst {
namespace attn_window {

constexpr int kThreads = 32 + 256;

template <int DP>
struct FwdCfg {
  static constexpr int kAt = DP / 64;
  static constexpr int kQ = kAt * kRowAtom;     // 128 queries x DP
  static constexpr int kKV = kAt * kBlkAtom;    // 64 keys x DP
  static constexpr int NS = 2;                  // key and value stages
  static constexpr int kRed = 2 * 2 * 128 * 4;  // [maxima, sums][half][row]
  static constexpr int kSmem = kQ + 2 * NS * kKV + kRed + 1024 + 128;
  static constexpr int kO = 128;  // TMEM: S, and P over it, in columns 0..63 and 64..127; O
};

template <int DP>
__global__ void __launch_bounds__(kThreads, 2)
    fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
               const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO,
               float* __restrict__ lse, const Shape s) {
  using C = FwdCfg<DP>;
  constexpr int NS = C::NS;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + C::kQ;        // [NS]
  uint8_t* sV = sK + NS * C::kKV;  // [NS]
  float* red = reinterpret_cast<float*>(sV + NS * C::kKV);
  uint64_t* bars = reinterpret_cast<uint64_t*>(red + 512);
  uint64_t* q_full = bars;
  uint64_t* k_full = bars + 1;  // [NS]
  uint64_t* v_full = bars + 3;  // [NS]
  uint64_t* s_full = bars + 5;  // [2]
  uint64_t* p_full = bars + 7;  // [2]
  uint64_t* o_full = bars + 9;
  uint64_t* o_last = bars + 10;  // the product of the last block
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 11);

  const int q0 = (gridDim.x - 1 - blockIdx.x) * 128;
  const int h = blockIdx.y, b = blockIdx.z, hk = h / s.G;
  const int warp = __shfl_sync(0xffffffff, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const KeyBlocks<64> blocks(s, q0);
  const int n = blocks.n;

  int ks = 0, vs = 0;  // copies started (warp 0)
  auto load = [&](uint32_t el, const CUtensorMap* map, uint8_t* dst, uint64_t* bar, int j) {
    expect_tx(el, bar, C::kKV);
#pragma unroll
    for (int a = 0; a < C::kAt; ++a) tma_load_4d(el, dst + a * kBlkAtom, map, bar, a * 64, blocks.at(j) * 64, hk, b);
  };
  auto load_k = [&](uint32_t el) { load(el, &tmK, sK + (ks % NS) * C::kKV, &k_full[ks % NS], ks), ++ks; };
  auto load_v = [&](uint32_t el) { load(el, &tmV, sV + (vs % NS) * C::kKV, &v_full[vs % NS], vs), ++vs; };
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < NS; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&v_full[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 256);
    }
    mbar_init(o_full, 1);
    mbar_init(o_last, 1);
    fence_barrier_init();
  }
  if (warp == 0) {  // the first copies travel while TMEM is allocated
    __syncwarp();
    const uint32_t el = elect_one();
    expect_tx(el, q_full, C::kQ);
#pragma unroll
    for (int a = 0; a < C::kAt; ++a) tma_load_4d(el, sQ + a * kRowAtom, &tmQ, q_full, a * 64, q0, h, b);
    while (ks < min(n, NS)) {
      load_k(el);
      load_v(el);
    }
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

  if (warp == 0) {
    const uint32_t el = elect_one();
    constexpr uint32_t id_s = idesc_bf16_f32(128, 64, false, false), id_o = idesc_bf16_f32(128, DP, false, true);
    auto issue_s = [&](int j) -> bool {  // S = Q K_j^T
      if (!warp_wait(&k_full[j % NS], (j / NS) & 1, s.status, kTimeoutTmaFull)) return false;
      tc_fence_after();
      product<DP>(el, tmem + 64 * (j & 1), sQ, sK + (j % NS) * C::kKV, kBlkAtom, id_s);
      mma_commit(el, &s_full[j & 1]);
      return true;
    };
    bool ok = warp_wait(q_full, 0, s.status, kTimeoutTmaFull) && issue_s(0) && (n == 1 || issue_s(1));
    for (int j = 0; j < n && ok; ++j) {
      ok = warp_wait(&v_full[j % NS], (j / NS) & 1, s.status, kTimeoutTmaFull) &&
           warp_wait(&p_full[j & 1], (j >> 1) & 1, s.status, kTimeoutTmemFull);
      if (!ok) break;
      if (ks < n) load_k(el);  // into K_j's stage: its scores are long done
      tc_fence_after();
      const uint32_t v = desc_lo(sV + (j % NS) * C::kKV, kBlkAtom);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)  // O (+)= P V_j; k-step kk: columns of the half that computed it
        mma_ts(el, tmem + C::kO, tmem + 64 * (j & 1) + (kk >> 1) * 32 + (kk & 1) * 8, v + ((kk * 2048) >> 4), id_o,
               (j > 0 || kk > 0) ? 1u : 0u);
      mma_commit(el, j + 1 < n ? o_full : o_last);
      if (j + 2 < n) {  // V_j, and the buffer of S_j and P_j, are free once this is done
        ok = warp_wait(o_full, j & 1, s.status, kTimeoutTmemFull);
        if (ok) load_v(el);
        ok = ok && issue_s(j + 2);
      }
    }
    if (!ok) {  // a wait expired: no copy may land after the CTA is gone
      for (int j = max(0, ks - NS); j < ks; ++j) mbar_wait(&k_full[j % NS], (j / NS) & 1, s.status, kTimeoutTmaFull);
      for (int j = max(0, vs - NS); j < vs; ++j) mbar_wait(&v_full[j % NS], (j / NS) & 1, s.status, kTimeoutTmaFull);
    }
    __syncwarp();
  } else {
    const int half = (warp - 1) >> 2, quad = warp & 3;  // a warp reads TMEM lanes 32 (warp % 4) ..
    const int r = quad * 32 + lane, q = q0 + r;
    const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
    float m_ref = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      ok = __all_sync(0xffffffff, ok && mbar_wait(&s_full[j & 1], (j >> 1) & 1, s.status, kTimeoutTmemFull));
      tc_fence_after();
      const uint32_t t_s = tmem + 64 * (j & 1) + half * 32 + lane_off;
      float v[32], m_blk = -INFINITY;
      const int k0 = blocks.at(j) * 64 + half * 32;
      if (ok) {
        tmem_ld32_sync(t_s, v);
        if (KeyBlocks<64>::partial<32>(s, q0, k0)) mask_keys(v, s, q, k0);
        float mx[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
        for (int i = 4; i < 32; ++i) mx[i & 3] = fmaxf(mx[i & 3], v[i]);
        m_blk = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * s.scale_log2;
      }
      float c = 1.f;
      if (pair_any(1 + quad, m_blk > m_ref + 8.f)) {
        red[half * 128 + r] = m_blk;
        pair_any(1 + quad, false);
        m_blk = fmaxf(m_blk, red[(half ^ 1) * 128 + r]);
        if (m_blk > m_ref + 8.f) {
          c = exp2f(m_ref - m_blk);
          l *= c;
          m_ref = m_blk;
        }
        // O holds P V of the blocks before: wait for the last of them, then rescale
        // this half's columns.
        if (j > 0) {
          ok = __all_sync(0xffffffff, ok && mbar_wait(o_full, (j - 1) & 1, s.status, kTimeoutTmemFull));
          tc_fence_after();
          if (ok) {
#pragma unroll 1
            for (int ch = 0; ch < DP / 32; ++ch) tmem_scale16(tmem + C::kO + half * (DP / 2) + ch * 16 + lane_off, c);
            tmem_wait_st();
          }
        }
        pair_any(1 + quad, false);  // red may be written again
      }
      const float m_use = m_ref == -INFINITY ? 0.f : m_ref;  // nothing visible so far
      float rs[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        v[i] = exp2f(fmaf(v[i], s.scale_log2, -m_use));
        rs[i & 3] += v[i];
      }
      l += (rs[0] + rs[1]) + (rs[2] + rs[3]);
      if (ok) {
        tmem_put32(t_s, v);  // over this half's own scores
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&p_full[j & 1]);
      }
    }
    red[256 + half * 128 + r] = l;
    pair_any(1 + quad, false);
    l += red[256 + (half ^ 1) * 128 + r];
    if (__all_sync(0xffffffff, ok && mbar_wait(o_last, 0, s.status, kTimeoutTmemFull))) {
      tc_fence_after();
      const float inv = 1.f / l;
#pragma unroll
      for (int ch = 0; ch < DP / 64; ++ch) {
        float o[32];
        tmem_ld32_sync(tmem + C::kO + half * (DP / 2) + ch * 32 + lane_off, o);
        stage_cols(sQ, r, half * (DP / 2) + ch * 32, o, inv);
      }
      fence_proxy_async_smem();
      done = true;
      // rows past the end: +inf, so that their probabilities are 0 in backward
      if (half == 0)
        lse[(static_cast<int64_t>(b) * s.H + h) * s.Tp + q] = q < s.T ? m_ref + log2f(l) : INFINITY;
    }
  }
  tc_fence_before();
  if (__syncthreads_and(done) && warp == 0) {
    const uint32_t el = elect_one();
    store_tile<DP>(el, &tmO, sQ, q0, h, b);
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
void launch_fwd(const CUtensorMap& q128, const CUtensorMap& k64, const CUtensorMap& v64, const CUtensorMap& out128,
                float* lse, int64_t B, const Shape& s, cudaStream_t stream) {
  if (allow_smem<fwd_kernel<DP>>(FwdCfg<DP>::kSmem) != cudaSuccess) return;
  fwd_kernel<DP><<<dim3(s.Tp / 128, s.H, static_cast<unsigned>(B)), kThreads, FwdCfg<DP>::kSmem, stream>>>(
      q128, k64, v64, out128, lse, s);
}
template void launch_fwd<64>(const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, float*,
                             int64_t, const Shape&, cudaStream_t);
template void launch_fwd<128>(const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, float*,
                              int64_t, const Shape&, cudaStream_t);
}  // namespace attn_window
}  // namespace dst
