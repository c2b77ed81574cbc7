// Attention with a sliding window and a few first tokens (sinks) that stay
// visible, forward and backward, on the sm_100a tensor cores.
//
//   visible(i, j)  <=>  j <= i  and  (i - j < W  or  j < S)
//   O = softmax(scale * Q K^T over the visible keys) V,  L = log2-sum-exp2
//   dV = P^T dO,  dP = dO V^T,  dS = P * (dP - rowsum(dO * O)),
//   dQ = scale * dS K,  dK = scale * dS^T Q   (dK, dV summed over the query
//   heads that share a key head)
//
// A query tile visits only the key blocks it can see: the blocks that hold
// sinks, then those from its window's first key to its diagonal; a key block
// likewise visits only the query blocks that see it. Work and traffic are
// O(T (W + S)) instead of O(T^2).
//
// Every kernel is one small CTA of four warps in which a thread owns a row of
// the 128-row tile and thread 0 also issues the TMA copies and the MMAs. Within
// a CTA the steps of a block (scores, softmax, product) follow one another;
// several CTAs share an SM and fill each other's gaps, also across prologue and
// epilogue, which count for much when a window is only a few blocks long.
// P (and dS) go back to the tensor core as the A operand in TMEM, in the columns
// of the scores they came from, so they never touch shared memory.
//
// q, k, v are reached through 4-D tensor maps (channel, token, head, batch), so
// any layout with 16-byte aligned strides works and rows past the end of a
// sequence read as zeros. Scores, softmax statistics and all sums are fp32; P
// and dS are rounded to bf16 as operands of the second product (relative 2^-9,
// the precision of the inputs), with the row sum taken before the rounding.
// No atomics: results do not depend on scheduling. All waits are bounded.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "common.h"
#include "ptx.cuh"

namespace dst {
namespace attn_window {

constexpr int kThreads = 128;      // one per row of a 128-row tile
constexpr int kRowAtom = 128 * 128;  // 128 rows x 64 channels, 128B-swizzled
constexpr int kBlkAtom = 64 * 128;   // 64 rows x 64 channels

struct Shape {
  int T, Tp;    // tokens; rounded up to a multiple of 128 (rows of lse and di)
  int H, G;     // query heads; query heads per key head
  int D;        // real head size (<= the padded DP of the kernel)
  int W, S;     // window, sinks (both clipped to T)
  float scale, scale_log2;
  int* status;
};

struct Strides {  // in elements
  int64_t t, h, b;
};

// 4-D tiled load: channel, token, head, batch. The channel coordinate is a
// multiple of 64, so every copy starts on a 16-byte boundary.
__device__ __forceinline__ void tma_load_4d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int c, int t, int h,
                                            int b) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
      "[%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c), "r"(t), "r"(h), "r"(b)
      : "memory");
}

// D[tmem] (+)= A[tmem] * B[smem]: row i of A in lane i, two bf16 of consecutive
// k per 32-bit column.
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}

// A row of 64 values as bf16 pairs into 32 TMEM columns.
__device__ __forceinline__ void tmem_put_row64(uint32_t taddr, const float (&v)[64]) {
  float pk[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) pk[i] = __uint_as_float(pack_bf16(v[2 * i], v[2 * i + 1]));
  tmem_st32_sync(taddr, pk);
}

// Columns [c0, c0 + 32) of a row to global memory as bf16, up to D.
__device__ __forceinline__ void store_cols(__nv_bfloat16* row, int c0, int D, const float (&v)[32], float scale) {
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    if (c0 + i < D) {
      uint4 pk;
      uint32_t* w = reinterpret_cast<uint32_t*>(&pk);
#pragma unroll
      for (int t = 0; t < 4; ++t) w[t] = pack_bf16(v[i + 2 * t] * scale, v[i + 2 * t + 1] * scale);
      *reinterpret_cast<uint4*>(row + c0 + i) = pk;
    }
  }
}

// Key blocks (64 keys) that a tile of 128 queries from q0 visits: n in all,
// block j of the list is key block `at(j)`.
struct KeyBlocks {
  int sink_blocks, first, n;
  __device__ __forceinline__ KeyBlocks(const Shape& s, int q0) {
    const int q_last = min(q0 + 127, s.T - 1);
    first = max(0, q0 - s.W + 1) >> 6;
    sink_blocks = min((s.S + 63) >> 6, first);
    n = sink_blocks + (q_last >> 6) - first + 1;
  }
  __device__ __forceinline__ int at(int j) const { return j < sink_blocks ? j : first + j - sink_blocks; }
};

// Zero what this row may not see among 64 keys from k0 (as -inf scores).
__device__ __forceinline__ void mask_keys(float (&v)[64], const Shape& s, int q, int k0) {
  const int last = q - k0, low = q - s.W + 1 - k0, sink = s.S - k0;
#pragma unroll
  for (int i = 0; i < 64; ++i)
    if (i > last || (i < low && i >= sink)) v[i] = -INFINITY;
}

// Whether some row of the tile from q0 misses some key of the block from k0.
__device__ __forceinline__ bool block_is_partial(const Shape& s, int q0, int k0) {
  return k0 + 63 > q0 || (k0 < q0 + 127 - s.W + 1 && k0 + 64 > s.S);
}

// ------------------------------------------------------------------ forward
template <int DP>
struct FwdCfg {
  static constexpr int kAt = DP / 64;
  static constexpr int kQ = kAt * kRowAtom;   // 128 queries x DP
  static constexpr int kKV = kAt * kBlkAtom;  // 64 keys x DP
  static constexpr int kSmem = kQ + 4 * kKV + 1024 + 128;
  static constexpr int kTmem = DP == 64 ? 128 : 256;  // S (and P): 0..63, O: from kO
  static constexpr int kO = DP == 64 ? 64 : 128;
  static constexpr int kCtas = DP == 64 ? 4 : 2;
};

template <int DP>
__global__ void __launch_bounds__(kThreads, FwdCfg<DP>::kCtas)
    fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
               const __grid_constant__ CUtensorMap tmV, __nv_bfloat16* __restrict__ out, float* __restrict__ lse,
               const Shape s) {
  using C = FwdCfg<DP>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + C::kQ;       // [2]
  uint8_t* sV = sK + 2 * C::kKV;  // [2]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + 2 * C::kKV);
  uint64_t* q_full = bars;
  uint64_t* k_full = bars + 1;  // [2]
  uint64_t* v_full = bars + 3;  // [2]
  uint64_t* s_full = bars + 5;
  uint64_t* o_full = bars + 6;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 7);

  const int q0 = (gridDim.x - 1 - blockIdx.x) * 128;
  const int h = blockIdx.y, b = blockIdx.z, hk = h / s.G;
  const int warp = threadIdx.x >> 5;
  const KeyBlocks blocks(s, q0);
  const int n = blocks.n;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&v_full[i], 1);
    }
    mbar_init(s_full, 1);
    mbar_init(o_full, 1);
    fence_barrier_init();
  }
  if (warp == 0) {
    __syncwarp();
    tmem_alloc(tmem_slot, C::kTmem);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t lane_off = static_cast<uint32_t>(warp * 32) << 16;

  auto load_kv = [&](int j) {
    const int st = j & 1, k0 = blocks.at(j) * 64;
    mbar_arrive_expect_tx(&k_full[st], C::kKV);
#pragma unroll
    for (int a = 0; a < C::kAt; ++a)
      tma_load_4d(sK + st * C::kKV + a * kBlkAtom, &tmK, &k_full[st], a * 64, k0, hk, b);
    mbar_arrive_expect_tx(&v_full[st], C::kKV);
#pragma unroll
    for (int a = 0; a < C::kAt; ++a)
      tma_load_4d(sV + st * C::kKV + a * kBlkAtom, &tmV, &v_full[st], a * 64, k0, hk, b);
  };
  auto issue_s = [&](int j) {  // S = Q K_j^T
    constexpr uint32_t id = idesc_bf16_f32(128, 64, false, false);
    const uint32_t q_addr = smem_u32(sQ), k_addr = smem_u32(sK + (j & 1) * C::kKV);
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk)
      umma_f16_ss(tmem, smem_desc_sw128(q_addr + (kk >> 2) * kRowAtom + (kk & 3) * 32, 16, 1024),
                  smem_desc_sw128(k_addr + (kk >> 2) * kBlkAtom + (kk & 3) * 32, 16, 1024), id, kk > 0 ? 1u : 0u);
    umma_commit(s_full);
  };
  auto issue_pv = [&](int j) {  // O (+)= P V_j
    constexpr uint32_t id = idesc_bf16_f32(128, DP, false, true);
    const uint32_t v_addr = smem_u32(sV + (j & 1) * C::kKV);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
      umma_f16_ts(tmem + C::kO, tmem + kk * 8, smem_desc_sw128(v_addr + kk * 2048, kBlkAtom, 1024), id,
                  (j > 0 || kk > 0) ? 1u : 0u);
    umma_commit(o_full);
  };

  bool ok = true;  // a bounded wait of this thread has expired once it is false
  int loaded = 0;  // thread 0: K/V blocks whose copies were started
  if (threadIdx.x == 0) {
    mbar_arrive_expect_tx(q_full, C::kQ);
#pragma unroll
    for (int a = 0; a < C::kAt; ++a) tma_load_4d(sQ + a * kRowAtom, &tmQ, q_full, a * 64, q0, h, b);
    for (; loaded < min(n, 2); ++loaded) load_kv(loaded);
    ok = mbar_wait(q_full, 0, s.status, kTimeoutTmaFull) && mbar_wait(&k_full[0], 0, s.status, kTimeoutTmaFull);
    if (ok) issue_s(0);
  }
  __syncwarp();

  const int q = q0 + threadIdx.x;
  float m_ref = -INFINITY, l = 0.f;
  for (int j = 0; j < n; ++j) {
    // tcgen05.ld / st are warp-collective: the whole warp decides together
    const bool good = __all_sync(0xffffffff, ok && mbar_wait(s_full, j & 1, s.status, kTimeoutTmemFull));
    ok = ok && good;
    if (good) {
      tc_fence_after();
      float v[64];
      tmem_ld64_sync(tmem + lane_off, v);
      const int k0 = blocks.at(j) * 64;
      if (block_is_partial(s, q0, k0)) mask_keys(v, s, q, k0);
      float mx[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
      for (int i = 4; i < 64; ++i) mx[i & 3] = fmaxf(mx[i & 3], v[i]);
      const float m_blk = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * s.scale_log2;
      // A row keeps its reference maximum until a block exceeds it by 8 (in
      // log2), so P stays below 2^8 and O is rarely rescaled.
      const bool need = m_blk > m_ref + 8.f;
      const float c = need ? exp2f(m_ref - m_blk) : 1.f;
      if (need) {
        l *= c;
        m_ref = m_blk;
      }
      const float m_use = m_ref == -INFINITY ? 0.f : m_ref;  // nothing visible so far
      float rs[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 64; ++i) {
        v[i] = exp2f(fmaf(v[i], s.scale_log2, -m_use));
        rs[i & 3] += v[i];
      }
      l += (rs[0] + rs[1]) + (rs[2] + rs[3]);
      tmem_put_row64(tmem + lane_off, v);  // P over S: this lane's scores are in registers
      // S_j was issued after P_{j-1} V_{j-1} had completed, so O may change here.
      if (j > 0 && __any_sync(0xffffffff, need)) {
#pragma unroll 1
        for (int ch = 0; ch < DP / 32; ++ch) {
          float o[32];
          tmem_ld32_sync(tmem + C::kO + ch * 32 + lane_off, o);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] *= c;
          tmem_st32_sync(tmem + C::kO + ch * 32 + lane_off, o);
        }
      }
    }
    tc_fence_before();
    const bool all_ok = __syncthreads_and(ok);
    ok = all_ok;
    if (threadIdx.x == 0 && ok) {
      tc_fence_after();
      ok = mbar_wait(&v_full[j & 1], (j >> 1) & 1, s.status, kTimeoutTmaFull);
      if (ok) {
        issue_pv(j);
        if (j + 1 < n) {
          // the scores of block j + 1 overwrite P_j, and its copies V_j, K_j
          ok = mbar_wait(o_full, j & 1, s.status, kTimeoutTmemFull) &&
               mbar_wait(&k_full[(j + 1) & 1], ((j + 1) >> 1) & 1, s.status, kTimeoutTmaFull);
          if (ok) {
            if (loaded < n) load_kv(loaded++);
            issue_s(j + 1);
          }
        }
      }
    }
    __syncwarp();
  }
  const bool done = __all_sync(0xffffffff, ok && mbar_wait(o_full, (n - 1) & 1, s.status, kTimeoutTmemFull));
  if (done) {
    tc_fence_after();
    const float inv = 1.f / l;
    __nv_bfloat16* row = out + ((static_cast<int64_t>(b) * s.T + q) * s.H + h) * s.D;
#pragma unroll
    for (int ch = 0; ch < DP / 32; ++ch) {
      float o[32];
      tmem_ld32_sync(tmem + C::kO + ch * 32 + lane_off, o);
      if (q < s.T) store_cols(row, ch * 32, s.D, o, inv);
    }
    // rows past the end: +inf, so that their probabilities are 0 in backward
    lse[(static_cast<int64_t>(b) * s.H + h) * s.Tp + q] = q < s.T ? m_ref + log2f(l) : INFINITY;
  }
  if (threadIdx.x == 0 && !ok)  // a wait expired: no copy may land after the CTA is gone
    for (int j = max(0, loaded - 2); j < loaded; ++j) {
      mbar_wait(&k_full[j & 1], (j >> 1) & 1, s.status, kTimeoutTmaFull);
      mbar_wait(&v_full[j & 1], (j >> 1) & 1, s.status, kTimeoutTmaFull);
    }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmem);
  }
}

// ----------------------------------------------------------------- backward
// di[b, h, t] = sum_d dO O (0 for the rows past the end). DP/8 threads a row.
template <int DP>
__global__ void rowdot_kernel(const __nv_bfloat16* __restrict__ dout, const __nv_bfloat16* __restrict__ out,
                              float* __restrict__ di, int64_t rows, const Shape s) {
  constexpr int kPer = DP / 8;
  const int64_t gt = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t w = gt / kPer;  // (b, h, t) with t up to Tp
  const int part = static_cast<int>(gt % kPer);
  const int t = static_cast<int>(w % s.Tp);
  float acc = 0.f;
  if (w < rows && t < s.T && part * 8 < s.D) {
    const int64_t bh = w / s.Tp, off = ((bh / s.H * s.T + t) * s.H + bh % s.H) * s.D + part * 8;
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
  if (w < rows && part == 0) di[w] = acc;
}

// dK, dV of 128 keys: walks the 64-query blocks that see them, of every query
// head of the group. Per block
//   S^T = K Q^T, dP^T = V dO^T;  P^T, dS^T into TMEM;  dV += P^T dO, dK += dS^T Q
template <int DP>
struct DkdvCfg {
  static constexpr int kAt = DP / 64;
  static constexpr int kKV = kAt * kRowAtom;
  static constexpr int kQ = kAt * kBlkAtom;
  static constexpr int kSmem = 2 * kKV + 4 * kQ + 4 * 64 * 4 + 1024 + 128;
  static constexpr int kTmem = DP == 64 ? 256 : 512;  // S^T, dP^T, dV, dK
  static constexpr int kCtas = DP == 64 ? 2 : 1;
};

template <int DP>
__global__ void __launch_bounds__(kThreads, DkdvCfg<DP>::kCtas)
    dkdv_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmDO,
                const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                const float* __restrict__ lse, const float* __restrict__ di, __nv_bfloat16* __restrict__ dk,
                __nv_bfloat16* __restrict__ dv, const Strides sk, const Strides sv, const Shape s) {
  using C = DkdvCfg<DP>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sK = smem;
  uint8_t* sV = sK + C::kKV;
  uint8_t* sQ = sV + C::kKV;       // [2]
  uint8_t* sDO = sQ + 2 * C::kQ;   // [2]
  float* sL = reinterpret_cast<float*>(sDO + 2 * C::kQ);  // [2][64]
  float* sDi = sL + 128;                                  // [2][64]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sDi + 128);
  uint64_t* kv_full = bars;
  uint64_t* q_full = bars + 1;  // [2]
  uint64_t* s_full = bars + 3;
  uint64_t* g_full = bars + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 5);

  const int k0 = blockIdx.x * 128;  // block 0 (the sinks) has the most queries: first
  const int hk = blockIdx.y, b = blockIdx.z;
  const int warp = threadIdx.x >> 5;
  const int k_last = min(k0 + 127, s.T - 1);
  // queries from the block's first key to the last that sees a key of it
  const int q_last = k0 < s.S ? s.T - 1 : static_cast<int>(min(static_cast<int64_t>(s.T) - 1, static_cast<int64_t>(k_last) + s.W - 1));
  const int qb0 = k0 >> 6, nq = (q_last >> 6) - qb0 + 1;
  const int n = nq * s.G;

  if (threadIdx.x == 0) {
    mbar_init(kv_full, 1);
    for (int i = 0; i < 2; ++i) mbar_init(&q_full[i], 1);
    mbar_init(s_full, 1);
    mbar_init(g_full, 1);
    fence_barrier_init();
  }
  if (warp == 0) {
    __syncwarp();
    tmem_alloc(tmem_slot, C::kTmem);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tS = tmem, tDP = tmem + 64, tDV = tmem + 128, tDK = tmem + 128 + DP;
  const uint32_t lane_off = static_cast<uint32_t>(warp * 32) << 16;

  auto load_q = [&](int i) {
    const int st = i & 1, h = hk * s.G + i / nq, q0 = (qb0 + i % nq) * 64;
    mbar_arrive_expect_tx(&q_full[st], 2 * C::kQ + 2 * 64 * 4);
#pragma unroll
    for (int a = 0; a < C::kAt; ++a) {
      tma_load_4d(sQ + st * C::kQ + a * kBlkAtom, &tmQ, &q_full[st], a * 64, q0, h, b);
      tma_load_4d(sDO + st * C::kQ + a * kBlkAtom, &tmDO, &q_full[st], a * 64, q0, h, b);
    }
    const int64_t row = (static_cast<int64_t>(b) * s.H + h) * s.Tp + q0;
    bulk_load(sL + st * 64, lse + row, 256, &q_full[st]);
    bulk_load(sDi + st * 64, di + row, 256, &q_full[st]);
  };
  auto issue_s = [&](int i) {
    constexpr uint32_t id = idesc_bf16_f32(128, 64, false, false);
    const uint32_t k_addr = smem_u32(sK), v_addr = smem_u32(sV);
    const uint32_t q_addr = smem_u32(sQ + (i & 1) * C::kQ), do_addr = smem_u32(sDO + (i & 1) * C::kQ);
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      const uint32_t ao = (kk >> 2) * kRowAtom + (kk & 3) * 32, bo = (kk >> 2) * kBlkAtom + (kk & 3) * 32;
      umma_f16_ss(tS, smem_desc_sw128(k_addr + ao, 16, 1024), smem_desc_sw128(q_addr + bo, 16, 1024), id,
                  kk > 0 ? 1u : 0u);
      umma_f16_ss(tDP, smem_desc_sw128(v_addr + ao, 16, 1024), smem_desc_sw128(do_addr + bo, 16, 1024), id,
                  kk > 0 ? 1u : 0u);
    }
    umma_commit(s_full);
  };
  auto issue_g = [&](int i) {
    constexpr uint32_t id = idesc_bf16_f32(128, DP, false, true);
    const uint32_t q_addr = smem_u32(sQ + (i & 1) * C::kQ), do_addr = smem_u32(sDO + (i & 1) * C::kQ);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      const uint32_t acc = (i > 0 || kk > 0) ? 1u : 0u;
      umma_f16_ts(tDV, tS + kk * 8, smem_desc_sw128(do_addr + kk * 2048, kBlkAtom, 1024), id, acc);
      umma_f16_ts(tDK, tDP + kk * 8, smem_desc_sw128(q_addr + kk * 2048, kBlkAtom, 1024), id, acc);
    }
    umma_commit(g_full);
  };

  bool ok = true;
  int loaded = 0;
  if (threadIdx.x == 0) {
    mbar_arrive_expect_tx(kv_full, 2 * C::kKV);
#pragma unroll
    for (int a = 0; a < C::kAt; ++a) {
      tma_load_4d(sK + a * kRowAtom, &tmK, kv_full, a * 64, k0, hk, b);
      tma_load_4d(sV + a * kRowAtom, &tmV, kv_full, a * 64, k0, hk, b);
    }
    for (; loaded < min(n, 2); ++loaded) load_q(loaded);
    ok = mbar_wait(kv_full, 0, s.status, kTimeoutTmaFull) && mbar_wait(&q_full[0], 0, s.status, kTimeoutTmaFull);
    if (ok) issue_s(0);
  }
  __syncwarp();

  const int key = k0 + threadIdx.x;
  for (int i = 0; i < n; ++i) {
    const int st = i & 1;
    const bool good =
        __all_sync(0xffffffff, ok && mbar_wait(&q_full[st], (i >> 1) & 1, s.status, kTimeoutTmaFull) &&
                                   mbar_wait(s_full, i & 1, s.status, kTimeoutTmemFull));
    ok = ok && good;
    if (good) {
      tc_fence_after();
      const int q0 = (qb0 + i % nq) * 64;
      // query column c is visible from c >= key - q0 on, below key + W - q0 (no upper end for a sink)
      const int from = key - q0;
      const int64_t to64 = key < s.S ? INT32_MAX : static_cast<int64_t>(key) + s.W - q0;
      const int to = static_cast<int>(min(to64, static_cast<int64_t>(INT32_MAX)));
      float p[64], ds[64];
      tmem_ld64_sync(tS + lane_off, p);
      tmem_ld64_sync(tDP + lane_off, ds);
#pragma unroll
      for (int c = 0; c < 64; ++c) {
        const float e = exp2f(fmaf(p[c], s.scale_log2, -sL[st * 64 + c]));
        const bool seen = c >= from && c < to;
        p[c] = seen ? e : 0.f;
        ds[c] = seen ? e * (ds[c] - sDi[st * 64 + c]) : 0.f;
      }
      tmem_put_row64(tS + lane_off, p);
      tmem_put_row64(tDP + lane_off, ds);
    }
    tc_fence_before();
    ok = __syncthreads_and(ok);
    if (threadIdx.x == 0 && ok) {
      tc_fence_after();
      issue_g(i);
      if (i + 1 < n) {
        ok = mbar_wait(g_full, i & 1, s.status, kTimeoutTmemFull) &&
             mbar_wait(&q_full[(i + 1) & 1], ((i + 1) >> 1) & 1, s.status, kTimeoutTmaFull);
        if (ok) {
          if (loaded < n) load_q(loaded++);
          issue_s(i + 1);
        }
      }
    }
    __syncwarp();
  }
  if (__all_sync(0xffffffff, ok && mbar_wait(g_full, (n - 1) & 1, s.status, kTimeoutTmemFull))) {
    tc_fence_after();
    __nv_bfloat16* krow = dk + b * sk.b + static_cast<int64_t>(key) * sk.t + hk * sk.h;
    __nv_bfloat16* vrow = dv + b * sv.b + static_cast<int64_t>(key) * sv.t + hk * sv.h;
#pragma unroll
    for (int ch = 0; ch < DP / 32; ++ch) {
      float x[32];
      tmem_ld32_sync(tDK + ch * 32 + lane_off, x);
      if (key < s.T) store_cols(krow, ch * 32, s.D, x, s.scale);
      tmem_ld32_sync(tDV + ch * 32 + lane_off, x);
      if (key < s.T) store_cols(vrow, ch * 32, s.D, x, 1.f);
    }
  }
  if (threadIdx.x == 0 && !ok)
    for (int i = max(0, loaded - 2); i < loaded; ++i) mbar_wait(&q_full[i & 1], (i >> 1) & 1, s.status, kTimeoutTmaFull);
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmem);
  }
}

// dQ of 128 queries: walks the key blocks of the forward pass. Per block
//   S = Q K^T, dP = dO V^T;  dS into TMEM;  dQ += dS K
template <int DP>
struct DqCfg {
  static constexpr int kAt = DP / 64;
  static constexpr int kQ = kAt * kRowAtom;
  static constexpr int kKV = kAt * kBlkAtom;
  static constexpr int kStages = DP == 64 ? 2 : 1;
  static constexpr int kSmem = 2 * kQ + 2 * kStages * kKV + 1024 + 128;
  static constexpr int kCtas = 2;  // S, dP, dQ: 256 TMEM columns
};

template <int DP>
__global__ void __launch_bounds__(kThreads, DqCfg<DP>::kCtas)
    dq_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmDO,
              const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
              const float* __restrict__ lse, const float* __restrict__ di, __nv_bfloat16* __restrict__ dq,
              const Strides sq, const Shape s) {
  using C = DqCfg<DP>;
  constexpr int NS = C::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sDO = sQ + C::kQ;
  uint8_t* sK = sDO + C::kQ;        // [NS]
  uint8_t* sV = sK + NS * C::kKV;   // [NS]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + NS * C::kKV);
  uint64_t* q_full = bars;
  uint64_t* kv_full = bars + 1;  // [NS]
  uint64_t* s_full = bars + 3;
  uint64_t* g_full = bars + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 5);

  const int q0 = (gridDim.x - 1 - blockIdx.x) * 128;
  const int h = blockIdx.y, b = blockIdx.z, hk = h / s.G;
  const int warp = threadIdx.x >> 5;
  const KeyBlocks blocks(s, q0);
  const int n = blocks.n;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < NS; ++i) mbar_init(&kv_full[i], 1);
    mbar_init(s_full, 1);
    mbar_init(g_full, 1);
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
  const uint32_t tmem = *tmem_slot;
  const uint32_t tS = tmem, tDP = tmem + 64, tDQ = tmem + 128;
  const uint32_t lane_off = static_cast<uint32_t>(warp * 32) << 16;

  auto load_kv = [&](int j) {
    const int st = j % NS, k0 = blocks.at(j) * 64;
    mbar_arrive_expect_tx(&kv_full[st], 2 * C::kKV);
#pragma unroll
    for (int a = 0; a < C::kAt; ++a) {
      tma_load_4d(sK + st * C::kKV + a * kBlkAtom, &tmK, &kv_full[st], a * 64, k0, hk, b);
      tma_load_4d(sV + st * C::kKV + a * kBlkAtom, &tmV, &kv_full[st], a * 64, k0, hk, b);
    }
  };
  auto issue_s = [&](int j) {
    constexpr uint32_t id = idesc_bf16_f32(128, 64, false, false);
    const uint32_t q_addr = smem_u32(sQ), do_addr = smem_u32(sDO);
    const uint32_t k_addr = smem_u32(sK + (j % NS) * C::kKV), v_addr = smem_u32(sV + (j % NS) * C::kKV);
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      const uint32_t ao = (kk >> 2) * kRowAtom + (kk & 3) * 32, bo = (kk >> 2) * kBlkAtom + (kk & 3) * 32;
      umma_f16_ss(tS, smem_desc_sw128(q_addr + ao, 16, 1024), smem_desc_sw128(k_addr + bo, 16, 1024), id,
                  kk > 0 ? 1u : 0u);
      umma_f16_ss(tDP, smem_desc_sw128(do_addr + ao, 16, 1024), smem_desc_sw128(v_addr + bo, 16, 1024), id,
                  kk > 0 ? 1u : 0u);
    }
    umma_commit(s_full);
  };
  auto issue_g = [&](int j) {
    constexpr uint32_t id = idesc_bf16_f32(128, DP, false, true);
    const uint32_t k_addr = smem_u32(sK + (j % NS) * C::kKV);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
      umma_f16_ts(tDQ, tDP + kk * 8, smem_desc_sw128(k_addr + kk * 2048, kBlkAtom, 1024), id,
                  (j > 0 || kk > 0) ? 1u : 0u);
    umma_commit(g_full);
  };

  bool ok = true;
  int loaded = 0;
  if (threadIdx.x == 0) {
    mbar_arrive_expect_tx(q_full, 2 * C::kQ);
#pragma unroll
    for (int a = 0; a < C::kAt; ++a) {
      tma_load_4d(sQ + a * kRowAtom, &tmQ, q_full, a * 64, q0, h, b);
      tma_load_4d(sDO + a * kRowAtom, &tmDO, q_full, a * 64, q0, h, b);
    }
    for (; loaded < min(n, NS); ++loaded) load_kv(loaded);
    ok = mbar_wait(q_full, 0, s.status, kTimeoutTmaFull) && mbar_wait(&kv_full[0], 0, s.status, kTimeoutTmaFull);
    if (ok) issue_s(0);
  }
  __syncwarp();

  const int q = q0 + threadIdx.x;
  const int64_t row = (static_cast<int64_t>(b) * s.H + h) * s.Tp + q;
  const float lq = lse[row], dq_i = di[row];
  for (int j = 0; j < n; ++j) {
    const bool good = __all_sync(0xffffffff, ok && mbar_wait(s_full, j & 1, s.status, kTimeoutTmemFull));
    ok = ok && good;
    if (good) {
      tc_fence_after();
      const int k0 = blocks.at(j) * 64;
      float p[64], ds[64];
      tmem_ld64_sync(tS + lane_off, p);
      tmem_ld64_sync(tDP + lane_off, ds);
      if (block_is_partial(s, q0, k0)) mask_keys(p, s, q, k0);
#pragma unroll
      for (int c = 0; c < 64; ++c) {
        const float e = exp2f(fmaf(p[c], s.scale_log2, -lq));
        ds[c] = e == 0.f ? 0.f : e * (ds[c] - dq_i);
      }
      tmem_put_row64(tDP + lane_off, ds);
    }
    tc_fence_before();
    ok = __syncthreads_and(ok);
    if (threadIdx.x == 0 && ok) {
      tc_fence_after();
      issue_g(j);
      if (j + 1 < n) {
        ok = mbar_wait(g_full, j & 1, s.status, kTimeoutTmemFull);
        if (ok && loaded < n) load_kv(loaded++);
        ok = ok && mbar_wait(&kv_full[(j + 1) % NS], ((j + 1) / NS) & 1, s.status, kTimeoutTmaFull);
        if (ok) issue_s(j + 1);
      }
    }
    __syncwarp();
  }
  if (__all_sync(0xffffffff, ok && mbar_wait(g_full, (n - 1) & 1, s.status, kTimeoutTmemFull))) {
    tc_fence_after();
    __nv_bfloat16* qrow = dq + b * sq.b + static_cast<int64_t>(q) * sq.t + h * sq.h;
#pragma unroll
    for (int ch = 0; ch < DP / 32; ++ch) {
      float x[32];
      tmem_ld32_sync(tDQ + ch * 32 + lane_off, x);
      if (q < s.T) store_cols(qrow, ch * 32, s.D, x, s.scale);
    }
  }
  if (threadIdx.x == 0 && !ok)
    for (int j = max(0, loaded - NS); j < loaded; ++j)
      mbar_wait(&kv_full[j % NS], (j / NS) & 1, s.status, kTimeoutTmaFull);
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

// -------------------------------------------------------------------- host
// Where q, k or v (or a gradient of one) lies: [B, T, heads, D] with unit inner
// stride; the other strides and the start are multiples of 16 bytes, so that
// tensor maps and 16-byte vectors can address it.
struct Operand {
  __nv_bfloat16* p;
  Strides s;
};

bool addressable(const at::Tensor& x) {
  if (x.stride(3) != 1 || reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 != 0) return false;
  for (int i = 0; i < 3; ++i)
    if (x.size(i) != 1 && (x.stride(i) <= 0 || x.stride(i) % 8 != 0)) return false;
  return true;
}

at::Tensor as_addressable(const at::Tensor& x) {
  return addressable(x) ? x : x.clone(at::MemoryFormat::Contiguous);
}

Operand operand(const at::Tensor& x) {
  return {static_cast<__nv_bfloat16*>(x.data_ptr()), {x.stride(1), x.stride(2), x.stride(0)}};
}

// q, k or v of a buffer [B, T, heads, 3, D].
Operand part_of(const at::Tensor& qkv, int which, int64_t D) {
  return {static_cast<__nv_bfloat16*>(qkv.data_ptr()) + which * D, {qkv.stride(1), 3 * D, qkv.stride(0)}};
}

CUtensorMap map_of(const Operand& x, int64_t B, int64_t T, int64_t heads, int64_t D, int rows) {
  const uint64_t dims[4] = {static_cast<uint64_t>(D), static_cast<uint64_t>(T), static_cast<uint64_t>(heads),
                            static_cast<uint64_t>(B)};
  const int64_t st[3] = {x.s.t, x.s.h, x.s.b};
  uint64_t strides[3];
  for (int i = 0; i < 3; ++i) strides[i] = dims[i + 1] == 1 ? 16 : static_cast<uint64_t>(st[i]) * 2;
  const uint32_t box[4] = {64, static_cast<uint32_t>(rows), 1, 1};
  return make_tmap_bf16_4d(x.p, dims, strides, box);
}

void check_bf16(const at::Tensor& x, const char* name) {
  TORCH_CHECK(x.is_cuda() && x.scalar_type() == at::kBFloat16, "window attention: ", name, " must be a CUDA bf16 tensor");
}

Shape shape_of(int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t D, int64_t window, int64_t sinks) {
  TORCH_CHECK(D >= 8 && D <= 128 && D % 8 == 0, "window attention: head_dim must be a multiple of 8 up to 128, got ",
              std::to_string(D));
  TORCH_CHECK(T >= 1 && T < (int64_t(1) << 30) && B >= 1, "window attention: T and B must be positive");
  TORCH_CHECK(H <= 65535 && B <= 65535, "window attention: more than 65535 heads or sequences");
  TORCH_CHECK(Hk >= 1 && H >= 1 && H % Hk == 0,
              "window attention: the number of query heads must be a multiple of the number of key heads");
  TORCH_CHECK(window >= 1 && sinks >= 0, "window attention: window >= 1 and sinks >= 0 required");
  Shape s;
  s.T = static_cast<int>(T);
  s.Tp = static_cast<int>((T + 127) / 128 * 128);
  s.H = static_cast<int>(H);
  s.G = static_cast<int>(H / Hk);
  s.D = static_cast<int>(D);
  s.W = static_cast<int>(std::min(window, T));
  s.S = static_cast<int>(std::min(sinks, T));
  const double sc = 1.0 / std::sqrt(static_cast<double>(D));
  s.scale = static_cast<float>(sc);
  s.scale_log2 = static_cast<float>(sc * 1.4426950408889634);
  s.status = status_ptr();
  return s;
}

template <auto kKernel>
void allow_smem(int bytes) {  // once per kernel and device
  static bool done[64] = {false};
  int dev;
  C10_CUDA_CHECK(cudaGetDevice(&dev));
  if (!done[dev]) C10_CUDA_CHECK(cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  done[dev] = true;
}

template <int DP>
void run_fwd(const Operand& q, const Operand& k, const Operand& v, __nv_bfloat16* out, float* lse, int64_t B,
             const Shape& s) {
  constexpr int smem = FwdCfg<DP>::kSmem;
  allow_smem<fwd_kernel<DP>>(smem);
  const int Hk = s.H / s.G;
  fwd_kernel<DP><<<dim3(s.Tp / 128, s.H, static_cast<unsigned>(B)), kThreads, smem, at::cuda::getCurrentCUDAStream()>>>(
      map_of(q, B, s.T, s.H, s.D, 128), map_of(k, B, s.T, Hk, s.D, 64), map_of(v, B, s.T, Hk, s.D, 64), out, lse, s);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

template <int DP>
void run_bwd(__nv_bfloat16* dout, const Operand& q, const Operand& k, const Operand& v, __nv_bfloat16* out,
             const float* lse, float* di, const Operand& dq, const Operand& dk, const Operand& dv, int64_t B,
             const Shape& s) {
  auto st = at::cuda::getCurrentCUDAStream();
  const int Hk = s.H / s.G;
  const int64_t rows = B * s.H * s.Tp;
  const int64_t blocks = (rows * (DP / 8) + 255) / 256;
  TORCH_CHECK(blocks < (int64_t(1) << 31), "window attention: too many rows");
  const Operand go = {dout, {static_cast<int64_t>(s.H) * s.D, s.D, static_cast<int64_t>(s.T) * s.H * s.D}};
  rowdot_kernel<DP><<<static_cast<unsigned>(blocks), 256, 0, st>>>(dout, out, di, rows, s);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  allow_smem<dkdv_kernel<DP>>(DkdvCfg<DP>::kSmem);
  dkdv_kernel<DP><<<dim3(s.Tp / 128, Hk, static_cast<unsigned>(B)), kThreads, DkdvCfg<DP>::kSmem, st>>>(
      map_of(q, B, s.T, s.H, s.D, 64), map_of(go, B, s.T, s.H, s.D, 64), map_of(k, B, s.T, Hk, s.D, 128),
      map_of(v, B, s.T, Hk, s.D, 128), lse, di, dk.p, dv.p, dk.s, dv.s, s);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  allow_smem<dq_kernel<DP>>(DqCfg<DP>::kSmem);
  dq_kernel<DP><<<dim3(s.Tp / 128, s.H, static_cast<unsigned>(B)), kThreads, DqCfg<DP>::kSmem, st>>>(
      map_of(q, B, s.T, s.H, s.D, 128), map_of(go, B, s.T, s.H, s.D, 128), map_of(k, B, s.T, Hk, s.D, 64),
      map_of(v, B, s.T, Hk, s.D, 64), lse, di, dq.p, dq.s, s);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// out [B, T, H, D] and the base-2 log-sum-exp [B, H, T rounded up to 128].
std::pair<at::Tensor, at::Tensor> forward(const Operand& q, const Operand& k, const Operand& v, int64_t B,
                                          const Shape& s, const at::TensorOptions& options) {
  at::Tensor out = at::empty({B, s.T, s.H, s.D}, options);
  at::Tensor lse = at::empty({B, s.H, s.Tp}, options.dtype(at::kFloat));
  auto* o = static_cast<__nv_bfloat16*>(out.data_ptr());
  if (s.D <= 64)
    run_fwd<64>(q, k, v, o, lse.data_ptr<float>(), B, s);
  else
    run_fwd<128>(q, k, v, o, lse.data_ptr<float>(), B, s);
  return {out, lse};
}

void backward(const at::Tensor& dout, const Operand& q, const Operand& k, const Operand& v, const at::Tensor& out,
              const at::Tensor& lse, const Operand& dq, const Operand& dk, const Operand& dv, int64_t B, const Shape& s) {
  at::Tensor go = dout.contiguous();
  if (reinterpret_cast<uintptr_t>(go.data_ptr()) % 16) go = go.clone();
  at::Tensor di = at::empty_like(lse);
  auto *g = static_cast<__nv_bfloat16*>(go.data_ptr()), *o = static_cast<__nv_bfloat16*>(out.data_ptr());
  if (s.D <= 64)
    run_bwd<64>(g, q, k, v, o, lse.data_ptr<float>(), di.data_ptr<float>(), dq, dk, dv, B, s);
  else
    run_bwd<128>(g, q, k, v, o, lse.data_ptr<float>(), di.data_ptr<float>(), dq, dk, dv, B, s);
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Separate q, k, v. The autograd nodes are C++: a Python node costs more host
// time per call than a short sequence takes on the GPU.
struct SeparateFn : public torch::autograd::Function<SeparateFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& v_,
                            int64_t window, int64_t sinks) {
    c10::cuda::CUDAGuard guard(q_.device());
    const int64_t B = q_.size(0), T = q_.size(1), D = q_.size(3);
    const Shape s = shape_of(B, T, q_.size(2), k_.size(2), D, window, sinks);
    const at::Tensor q = as_addressable(q_), k = as_addressable(k_), v = as_addressable(v_);
    auto [out, lse] = attn_window::forward(operand(q), operand(k), operand(v), B, s, q.options());
    ctx->save_for_backward({q, k, v, out, lse});
    ctx->saved_data["window"] = window;
    ctx->saved_data["sinks"] = sinks;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &q = saved[0], &k = saved[1], &v = saved[2], &out = saved[3], &lse = saved[4];
    c10::cuda::CUDAGuard guard(q.device());
    const Shape s = shape_of(q.size(0), q.size(1), q.size(2), k.size(2), q.size(3), ctx->saved_data["window"].toInt(),
                             ctx->saved_data["sinks"].toInt());
    at::Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()),
               dv = at::empty(v.sizes(), v.options());
    attn_window::backward(grads[0], operand(q), operand(k), operand(v), out, lse, operand(dq), operand(dk), operand(dv),
                          q.size(0), s);
    debug_check("window_attention backward");
    return {dq, dk, dv, at::Tensor(), at::Tensor()};
  }
};

// q, k, v interleaved head by head in one buffer, and their gradients likewise.
struct FusedFn : public torch::autograd::Function<FusedFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& qkv_, int64_t n_head, int64_t head_dim,
                            int64_t window, int64_t sinks) {
    c10::cuda::CUDAGuard guard(qkv_.device());
    const int64_t B = qkv_.size(0), T = qkv_.size(1);
    const Shape s = shape_of(B, T, n_head, n_head, head_dim, window, sinks);
    at::Tensor qkv = qkv_.contiguous();
    if (reinterpret_cast<uintptr_t>(qkv.data_ptr()) % 16) qkv = qkv.clone();
    auto [out, lse] = attn_window::forward(part_of(qkv, 0, head_dim), part_of(qkv, 1, head_dim),
                                           part_of(qkv, 2, head_dim), B, s, qkv.options());
    ctx->save_for_backward({qkv, out, lse});
    ctx->saved_data["window"] = window;
    ctx->saved_data["sinks"] = sinks;
    return out.view({B, T, n_head * head_dim});
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &qkv = saved[0], &out = saved[1], &lse = saved[2];
    c10::cuda::CUDAGuard guard(qkv.device());
    const int64_t B = out.size(0), D = out.size(3);
    const Shape s = shape_of(B, out.size(1), out.size(2), out.size(2), D, ctx->saved_data["window"].toInt(),
                             ctx->saved_data["sinks"].toInt());
    at::Tensor dqkv = at::empty(qkv.sizes(), qkv.options());
    attn_window::backward(grads[0], part_of(qkv, 0, D), part_of(qkv, 1, D), part_of(qkv, 2, D), out, lse,
                          part_of(dqkv, 0, D), part_of(dqkv, 1, D), part_of(dqkv, 2, D), B, s);
    debug_check("window_attention backward");
    return {dqkv, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

}  // namespace attn_window
}  // namespace dst

using namespace dst;

// q [B, T, H, D], k and v [B, T, Hk, D], any strides -> [B, T, H, D], differentiable.
at::Tensor window_attention_qkv(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, int64_t window,
                                int64_t sinks) {
  attn_window::check_bf16(q, "q");
  attn_window::check_bf16(k, "k");
  attn_window::check_bf16(v, "v");
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && k.sizes() == v.sizes() && k.size(0) == q.size(0) &&
                  k.size(1) == q.size(1) && k.size(3) == q.size(3),
              "window attention: q [B, T, H, D] and k, v [B, T, Hk, D] must agree");
  TORCH_CHECK(k.device() == q.device() && v.device() == q.device(), "window attention: q, k, v on one device");
  return attn_window::SeparateFn::apply(q, k, v, window, sinks);
}

// qkv [B, T, n_head * 3 * head_dim] -> [B, T, n_head * head_dim], differentiable.
at::Tensor window_attention(const at::Tensor& qkv, int64_t n_head, int64_t head_dim, int64_t window, int64_t sinks) {
  attn_window::check_bf16(qkv, "qkv");
  TORCH_CHECK(qkv.dim() == 3 && n_head >= 1 && head_dim >= 1 && qkv.size(2) == 3 * n_head * head_dim,
              "window attention: qkv must be [B, T, n_head * 3 * head_dim]");
  return attn_window::FusedFn::apply(qkv, n_head, head_dim, window, sinks);
}

void register_attn_window(pybind11::module& m) {
  m.def("window_attention_qkv", &window_attention_qkv, "sliding-window attention with sinks", pybind11::arg("q"),
        pybind11::arg("k"), pybind11::arg("v"), pybind11::arg("window"), pybind11::arg("sinks"));
  m.def("window_attention", &window_attention, "sliding-window attention with sinks over a fused qkv buffer",
        pybind11::arg("qkv"), pybind11::arg("n_head"), pybind11::arg("head_dim"), pybind11::arg("window"),
        pybind11::arg("sinks"));
}
