// Attention with a sliding window and a few first tokens (sinks) that stay
// visible: what its kernels share.
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
// A CTA owns a 128-row tile: warp 0 issues the TMA copies and the tcgen05 MMAs,
// the other warps turn scores into probabilities (two threads a row, each half
// of a block's columns). Within a tile a block's steps (scores, softmax,
// product) mostly follow one another, so two tiles share an SM and fill each
// other's gaps - also across prologue and epilogue, which count for much when a
// window is only a few blocks long. P (and dS) go back to the tensor core as the
// A operand in TMEM and never touch shared memory.
//
// q, k, v are reached through 4-D tensor maps (channel, token, head, batch), so
// any layout with 16-byte aligned strides works and rows past the end of a
// sequence read as zeros. Scores, softmax statistics and all sums are fp32; P
// and dS are rounded to bf16 as operands of the second product (relative 2^-8 at most,
// the precision of the inputs), with the row sum taken before the rounding.
// No atomics on data: results do not depend on scheduling. All waits are bounded.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#ifdef __CUDACC__
#include "ptx.cuh"
#endif

namespace dst {
namespace attn_window {

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

struct Operand {  // q, k, v or a gradient: [B, T, heads, D], unit inner stride
  __nv_bfloat16* p;
  Strides s;
};

// Sinks are seen by every later query, so their key blocks would walk the whole
// sequence alone. The queries past the blocks' windows are cut into chunks of
// `steps` 64-query blocks (per query head), each its own CTA, whose sums for the
// sink rows are joined in order. Chunk 0 is the block's own window. Of many sinks
// the blocks are CTAs enough, so rows (1 + chunks) stays within T, or chunks is 1:
// the sums take no more than twice dK and dV in fp32, whatever S.
struct SinkChunks {
  int blocks;  // key blocks of 128 that hold sinks and have queries past their window
  int rows;    // sinks in these blocks
  int chunks;  // CTAs per such block beside its own
  int steps;
  float* partial;  // [B, Hk, 1 + chunks, 2, rows, DP]: dK (0) and dV (1) of a chunk
  template <int DP>
  __host__ __device__ float* sums(int b, int key_heads, int hk, int chunk, int which, int key) const {
    const int64_t unit = static_cast<int64_t>(b) * key_heads + hk;
    return partial + (((unit * (1 + chunks) + chunk) * 2 + which) * rows + key) * DP;
  }
};

__host__ __device__ inline int last_window_query(const Shape& s, int k0) {  // of the key block from k0
  const int64_t k_last = k0 + 127 < s.T - 1 ? k0 + 127 : s.T - 1;
  const int64_t q = k_last + s.W - 1;
  return q < s.T - 1 ? static_cast<int>(q) : s.T - 1;
}

#ifdef __CUDACC__

// The issuing warp runs its loop with all lanes and lets one elected lane (`el`)
// issue. That keeps addresses and descriptors warp-uniform, where the tensor core
// and TMA instructions want them: issued from a one-lane branch with 64-bit
// descriptors built for each, an MMA took the warp about 100 cycles, more than
// its multiplications.

// 4-D tiled load: channel, token, head, batch. The channel coordinate is a
// multiple of 64, so every copy starts on a 16-byte boundary.
__device__ __forceinline__ void tma_load_4d(uint32_t el, void* smem_dst, const CUtensorMap* map, uint64_t* bar, int c,
                                            int t, int h, int b) {
  asm volatile(
      "{\n\t.reg .pred pe;\n\t"
      "setp.ne.b32 pe, %7, 0;\n\t"
      "@pe cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
      "[%2];\n\t}" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c), "r"(t), "r"(h), "r"(b), "r"(el)
      : "memory");
}

// 4-D tiled store of a 128-row tile's 64-channel atom; rows and channels past the
// tensor's end are clipped.
__device__ __forceinline__ void tma_store_4d(uint32_t el, const CUtensorMap* map, const void* smem_src, int c, int t,
                                             int h, int b) {
  asm volatile(
      "{\n\t.reg .pred pe;\n\t"
      "setp.ne.b32 pe, %6, 0;\n\t"
      "@pe cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];\n\t}" ::"l"(
          reinterpret_cast<uint64_t>(map)),
      "r"(smem_u32(smem_src)), "r"(c), "r"(t), "r"(h), "r"(b), "r"(el)
      : "memory");
}

__device__ __forceinline__ void expect_tx(uint32_t el, uint64_t* bar, uint32_t bytes) {
  if (el) mbar_arrive_expect_tx(bar, bytes);
}

// Shared-memory descriptors of 128B-swizzled tiles (groups of 8 rows 1024 bytes
// apart): the low word holds address and leading offset, the high word is fixed.
constexpr uint32_t kDescHi = (1024 >> 4) | (1u << 14) | (2u << 29);

__device__ __forceinline__ uint32_t desc_lo(const void* tile, uint32_t lbo) {
  return ((smem_u32(tile) >> 4) & 0x3FFF) | ((lbo >> 4) << 16);
}

// D[tmem] (+)= A[smem] * B[smem]
__device__ __forceinline__ void mma_ss(uint32_t el, uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred pe, p;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 pe, %0, 0;\n\tsetp.ne.b32 p, %6, 0;\n\t"
      "mov.b64 da, {%2, %4};\n\tmov.b64 db, {%3, %4};\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f16 [%1], da, db, %5, p;\n\t}" ::"r"(el),
      "r"(d), "r"(a_lo), "r"(b_lo), "r"(kDescHi), "r"(idesc), "r"(accumulate)
      : "memory");
}

// D[tmem] (+)= A[tmem] * B[smem]: row i of A in lane i, two bf16 of consecutive
// k per 32-bit column.
__device__ __forceinline__ void mma_ts(uint32_t el, uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred pe, p;\n\t.reg .b64 db;\n\t"
      "setp.ne.b32 pe, %0, 0;\n\tsetp.ne.b32 p, %6, 0;\n\t"
      "mov.b64 db, {%3, %4};\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f16 [%1], [%2], db, %5, p;\n\t}" ::"r"(el),
      "r"(d), "r"(a_tmem), "r"(b_lo), "r"(kDescHi), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void mma_commit(uint32_t el, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred pe;\n\t"
      "setp.ne.b32 pe, %1, 0;\n\t"
      "@pe tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(el)
      : "memory");
}

// mbar_wait of a whole warp; the result is the same in every lane.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* status, int code) {
  return __all_sync(0xffffffff, mbar_wait(bar, parity, status, code));
}

// D = R C^T over DP channels: R a tile of 128 rows, C one whose 64-channel atoms
// are `col_atom` bytes.
template <int DP>
__device__ __forceinline__ void product(uint32_t el, uint32_t d, const void* rows, const void* cols, uint32_t col_atom,
                                        uint32_t idesc) {
  const uint32_t a = desc_lo(rows, 16), c = desc_lo(cols, 16);
#pragma unroll
  for (int kk = 0; kk < DP / 16; ++kk)
    mma_ss(el, d, a + (((kk >> 2) * kRowAtom + (kk & 3) * 32) >> 4), c + (((kk >> 2) * col_atom + (kk & 3) * 32) >> 4),
           idesc, kk > 0 ? 1u : 0u);
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}

// 32 values of a row as bf16 pairs into 16 TMEM columns.
__device__ __forceinline__ void tmem_put32(uint32_t taddr, const float* v) {
  uint32_t r[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) r[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Columns [c0, c0 + 32) of row r of a 128B-swizzled result tile, as bf16.
__device__ __forceinline__ void stage_cols(uint8_t* tile, int r, int c0, const float (&v)[32], float scale) {
  uint8_t* row = tile + (c0 >> 6) * kRowAtom + r * 128;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint4 pk;
    uint32_t* w = reinterpret_cast<uint32_t*>(&pk);
#pragma unroll
    for (int t = 0; t < 4; ++t) w[t] = pack_bf16(v[8 * i + 2 * t] * scale, v[8 * i + 2 * t + 1] * scale);
    *reinterpret_cast<uint4*>(row + (((((c0 >> 3) & 7) + i) ^ (r & 7)) << 4)) = pk;
  }
}

// The whole warp: a staged tile of DP channels to rows t.. of (head, sequence).
template <int DP>
__device__ __forceinline__ void store_tile(uint32_t el, const CUtensorMap* map, const uint8_t* tile, int t, int h, int b) {
#pragma unroll
  for (int a = 0; a < DP / 64; ++a) tma_store_4d(el, map, tile + a * kRowAtom, a * 64, t, h, b);
}

// 16 columns of a row, scaled in place.
__device__ __forceinline__ void tmem_scale16(uint32_t taddr, float c) {
  uint32_t r[16];
  asm volatile(
      "{\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;\n\t}"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * c);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Barrier of the two warps that share 32 rows; true if some thread brought true.
__device__ __forceinline__ bool pair_any(int id, bool x) {
  int r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, %2, 64, p;\n\t"
      "selp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(static_cast<int>(x)), "r"(id)
      : "memory");
  return r != 0;
}

// Key blocks of BN keys that a tile of 128 queries from q0 visits: n in all,
// block j of the list is key block `at(j)`.
template <int BN>
struct KeyBlocks {
  int sink_blocks, first, n;
  __device__ __forceinline__ KeyBlocks(const Shape& s, int q0) {
    const int q_last = min(q0 + 127, s.T - 1);
    first = max(0, q0 - s.W + 1) / BN;
    sink_blocks = min((s.S + BN - 1) / BN, first);
    n = sink_blocks + q_last / BN - first + 1;
  }
  __device__ __forceinline__ int at(int j) const { return j < sink_blocks ? j : first + j - sink_blocks; }
  // Whether some row of the tile misses some of the N keys from k0.
  template <int N>
  static __device__ __forceinline__ bool partial(const Shape& s, int q0, int k0) {
    return k0 + N - 1 > q0 || (k0 < q0 + 127 - s.W + 1 && k0 + N > s.S);
  }
};

// -inf for what query q may not see among N keys from k0.
template <int N>
__device__ __forceinline__ void mask_keys(float (&v)[N], const Shape& s, int q, int k0) {
  const int last = q - k0, low = q - s.W + 1 - k0, sink = s.S - k0;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i > last || (i < low && i >= sink)) v[i] = -INFINITY;
}

#endif  // __CUDACC__

// Launches (padded head size DP = 64 or 128), on `stream`.
template <int DP>
void launch_fwd(const CUtensorMap& q128, const CUtensorMap& k64, const CUtensorMap& v64, const CUtensorMap& out128,
                float* lse, int64_t B, const Shape& s, cudaStream_t stream);
template <int DP>
void launch_rowdot(const __nv_bfloat16* dout, const __nv_bfloat16* out, float* di, int64_t B, const Shape& s,
                   cudaStream_t stream);
template <int DP>
void launch_dkdv(const CUtensorMap& q64, const CUtensorMap& dout64, const CUtensorMap& k128, const CUtensorMap& v128,
                 const float* lse, const float* di, const CUtensorMap& dk128, const CUtensorMap& dv128, int64_t B,
                 const SinkChunks& sinks, const Shape& s, cudaStream_t stream);
template <int DP>
void launch_dq(const CUtensorMap& q128, const CUtensorMap& dout128, const CUtensorMap& k64, const CUtensorMap& v64,
               const float* lse, const float* di, const CUtensorMap& dq128, const Operand& dk, const Operand& dv,
               int64_t B, const SinkChunks& sinks, const Shape& s, cudaStream_t stream);

// Dynamic shared memory above 48 KB has to be allowed once per kernel and device.
template <auto kKernel>
cudaError_t allow_smem(int bytes) {
  static bool done[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || done[dev]) return e;
  e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  done[dev] = e == cudaSuccess;
  return e;
}

}  // namespace attn_window
}  // namespace dst
