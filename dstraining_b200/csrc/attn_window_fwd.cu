// Windowed attention, forward (see attn_window.cuh).
//
// One CTA per (128 queries, head, sequence), two per SM, blocks of 128 keys:
// warp 0 copies and issues S = Q K^T and O += P V; warps 1-4 and 5-8 are the
// softmax of the left and the right 64 columns of a block, a thread per row. The
// two halves of a row only meet where its maximum may have to move: a row keeps
// its reference maximum until a block exceeds it by 8 (in log2), so P stays below
// 2^8 and in most blocks one barrier between two warps is all they exchange.
// Blocks of 128 keys because an MMA with N = 64 reads its A tile from shared
// memory for half the work: scores of 128 x 64 took 3x the tensor time of their
// multiplications, of 128 x 128 2x.
#include "attn_window.cuh"

namespace dst {
namespace attn_window {

constexpr int kThreads = 32 + 256;

template <int DP>
struct FwdCfg {
  static constexpr int kAt = DP / 64;
  static constexpr int kTile = kAt * kRowAtom;  // 128 rows x DP
  static constexpr int NS = DP == 64 ? 2 : 1;   // key and value stages
  static constexpr int kRed = 2 * 2 * 128 * 4;  // [maxima, sums][half][row]
  static constexpr int kSmem = kTile * (1 + 2 * NS) + kRed + 1024 + 128;
  // TMEM: S in columns 0..127, O from 128. P beside them where there is room (DP 64:
  // 192..255), else each half of it over the same half of S.
  static constexpr bool kBeside = DP == 64;
  static constexpr int kO = 128;
  static constexpr int kP = kBeside ? 192 : 0;
  static constexpr int kPHalf = kBeside ? 32 : 64;
};

template <int DP>
__global__ void __launch_bounds__(kThreads, 2)
    fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
               const __grid_constant__ CUtensorMap tmV, __nv_bfloat16* __restrict__ out, float* __restrict__ lse,
               const Shape s) {
  using C = FwdCfg<DP>;
  constexpr int NS = C::NS;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + C::kTile;       // [NS]
  uint8_t* sV = sK + NS * C::kTile;  // [NS]
  float* red = reinterpret_cast<float*>(sV + NS * C::kTile);
  uint64_t* bars = reinterpret_cast<uint64_t*>(red + 512);
  uint64_t* q_full = bars;
  uint64_t* k_full = bars + 1;  // [NS]
  uint64_t* v_full = bars + 3;  // [NS]
  uint64_t* s_full = bars + 5;
  uint64_t* s_free = bars + 6;
  uint64_t* p_full = bars + 7;
  uint64_t* o_full = bars + 8;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 9);

  const int q0 = (gridDim.x - 1 - blockIdx.x) * 128;
  const int h = blockIdx.y, b = blockIdx.z, hk = h / s.G;
  const int warp = __shfl_sync(0xffffffff, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const KeyBlocks<128> blocks(s, q0);
  const int n = blocks.n;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < NS; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&v_full[i], 1);
    }
    mbar_init(s_full, 1);
    mbar_init(s_free, 256);
    mbar_init(p_full, 256);
    mbar_init(o_full, 1);
    fence_barrier_init();
  }
  if (warp == 0) {
    __syncwarp();
    tmem_alloc(tmem_slot, 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffff, *tmem_slot, 0);

  if (warp == 0) {
    const uint32_t el = elect_one();
    auto load = [&](const CUtensorMap* map, uint8_t* dst, uint64_t* bar, int row, int head) {
      expect_tx(el, bar, C::kTile);
#pragma unroll
      for (int a = 0; a < C::kAt; ++a) tma_load_4d(el, dst + a * kRowAtom, map, bar, a * 64, row, head, b);
    };
    auto load_k = [&](int j) { load(&tmK, sK + (j % NS) * C::kTile, &k_full[j % NS], blocks.at(j) * 128, hk); };
    auto load_v = [&](int j) { load(&tmV, sV + (j % NS) * C::kTile, &v_full[j % NS], blocks.at(j) * 128, hk); };
    auto issue_s = [&](int j) -> bool {  // S = Q K_j^T
      if (!warp_wait(&k_full[j % NS], (j / NS) & 1, s.status, kTimeoutTmaFull)) return false;
      tc_fence_after();
      product<DP>(el, tmem, sQ, sK + (j % NS) * C::kTile, kRowAtom, idesc_bf16_f32(128, 128, false, false));
      mma_commit(el, s_full);
      return true;
    };
    int ks = 0, vs = 0;  // copies started
    load(&tmQ, sQ, q_full, q0, h);
    for (; ks < min(n, NS); ++ks) {
      load_k(ks);
      load_v(vs++);
    }
    bool ok = warp_wait(q_full, 0, s.status, kTimeoutTmaFull) && issue_s(0);
    for (int j = 0; j < n && ok; ++j) {
      if (C::kBeside && j + 1 < n) {  // the next scores while the softmax works on these
        ok = warp_wait(s_free, j & 1, s.status, kTimeoutTmemEmpty) && issue_s(j + 1);
      } else if (!C::kBeside) {
        ok = warp_wait(s_full, j & 1, s.status, kTimeoutTmemFull);  // K_j has been read
        if (ok && ks < n) load_k(ks++);
      }
      ok = ok && warp_wait(&v_full[j % NS], (j / NS) & 1, s.status, kTimeoutTmaFull) &&
           warp_wait(p_full, j & 1, s.status, kTimeoutTmemFull);
      if (!ok) break;
      if (C::kBeside && ks < n) load_k(ks++);  // into K_j's stage: its scores are long done
      tc_fence_after();
      constexpr uint32_t id = idesc_bf16_f32(128, DP, false, true);
      const uint32_t v = desc_lo(sV + (j % NS) * C::kTile, kRowAtom);
      uint32_t acc = j > 0;
#pragma unroll
      for (int half = 0; half < 2; ++half) {  // O (+)= P V_j, without a half that no row sees
        if (!KeyBlocks<128>::seen<64>(s, q0, blocks.at(j) * 128 + half * 64)) continue;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          mma_ts(el, tmem + C::kO, tmem + C::kP + half * C::kPHalf + kk * 8, v + (((half * 4 + kk) * 2048) >> 4), id, acc);
          acc = 1;
        }
      }
      mma_commit(el, o_full);
      if (j + 1 < n) {  // V_j, and P over S, are free once this is done
        ok = warp_wait(o_full, j & 1, s.status, kTimeoutTmemFull);
        if (ok && vs < n) load_v(vs++);
        if (ok && !C::kBeside) ok = issue_s(j + 1);
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
      ok = __all_sync(0xffffffff, ok && mbar_wait(s_full, j & 1, s.status, kTimeoutTmemFull));
      tc_fence_after();
      float v[64], m_blk = -INFINITY;
      const int k0 = blocks.at(j) * 128 + half * 64;
      const bool seen = ok && KeyBlocks<128>::seen<64>(s, q0, k0);
      if (seen) {
        tmem_ld64_sync(tmem + half * 64 + lane_off, v);
        if (KeyBlocks<128>::partial<64>(s, q0, k0)) mask_keys(v, s, q, k0);
        float mx[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
        for (int i = 4; i < 64; ++i) mx[i & 3] = fmaxf(mx[i & 3], v[i]);
        m_blk = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * s.scale_log2;
      }
      tc_fence_before();
      if (C::kBeside && ok) mbar_arrive(s_free);  // the scores are in registers
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
      if (seen) {
        const float m_use = m_ref == -INFINITY ? 0.f : m_ref;  // nothing visible so far
        float rs[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          v[i] = exp2f(fmaf(v[i], s.scale_log2, -m_use));
          rs[i & 3] += v[i];
        }
        l += (rs[0] + rs[1]) + (rs[2] + rs[3]);
      }
      // P beside S is read by the product of the block before: wait for it
      if (C::kBeside && j > 0) ok = __all_sync(0xffffffff, ok && mbar_wait(o_full, (j - 1) & 1, s.status, kTimeoutTmemFull));
      if (ok) {
        tc_fence_after();
        if (seen) {
          tmem_put32(tmem + C::kP + half * C::kPHalf + lane_off, v);
          tmem_put32(tmem + C::kP + half * C::kPHalf + 16 + lane_off, v + 32);
          tmem_wait_st();
        }
        tc_fence_before();
        mbar_arrive(p_full);
      }
    }
    red[256 + half * 128 + r] = l;
    pair_any(1 + quad, false);
    l += red[256 + (half ^ 1) * 128 + r];
    if (__all_sync(0xffffffff, ok && mbar_wait(o_full, (n - 1) & 1, s.status, kTimeoutTmemFull))) {
      tc_fence_after();
      const float inv = 1.f / l;
      __nv_bfloat16* row = out + ((static_cast<int64_t>(b) * s.T + q) * s.H + h) * s.D;
#pragma unroll
      for (int ch = 0; ch < DP / 64; ++ch) {
        float o[32];
        tmem_ld32_sync(tmem + C::kO + half * (DP / 2) + ch * 32 + lane_off, o);
        if (q < s.T) store_cols(row, half * (DP / 2) + ch * 32, s.D, o, inv);
      }
      // rows past the end: +inf, so that their probabilities are 0 in backward
      if (half == 0)
        lse[(static_cast<int64_t>(b) * s.H + h) * s.Tp + q] = q < s.T ? m_ref + log2f(l) : INFINITY;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

template <int DP>
void launch_fwd(const CUtensorMap& q128, const CUtensorMap& k, const CUtensorMap& v, __nv_bfloat16* out, float* lse,
                int64_t B, const Shape& s, cudaStream_t stream) {
  if (allow_smem<fwd_kernel<DP>>(FwdCfg<DP>::kSmem) != cudaSuccess) return;
  fwd_kernel<DP><<<dim3(s.Tp / 128, s.H, static_cast<unsigned>(B)), kThreads, FwdCfg<DP>::kSmem, stream>>>(q128, k, v, out,
                                                                                                       lse, s);
}
template void launch_fwd<64>(const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, __nv_bfloat16*, float*, int64_t,
                             const Shape&, cudaStream_t);
template void launch_fwd<128>(const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, __nv_bfloat16*, float*, int64_t,
                              const Shape&, cudaStream_t);
}  // namespace attn_window
}  // namespace dst
