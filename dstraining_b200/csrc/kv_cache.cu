// The rolling key/value cache of windowed attention with sinks, in bf16 or
// 4 bits, and the attention of one new token per sequence over it.
//
// Slots: S + W per (sequence, key head); token p lies in slot p while p < S and
// in S + (p - S) % W after, so once the ring is full a new token takes the slot
// of the one that leaves the window, and every filled slot is visible.
//
// 4 bits: each 32 channels of a row share a step = bf16((max - min) / 15) and
// their least value (bf16, exact: it is one of them); a channel is stored as
// code = clamp(rint((x - min) / step), 0, 15) and stands for min + code * step.
// 32 channels cost 20 bytes instead of 64. A group with an infinity or NaN
// stands for NaN.
//
// The single-token step reads every held row once and is bound by that traffic,
// so it has to keep many bytes in flight and spend few instructions on them:
//   * each warp streams tiles of keys through its own ring of shared-memory
//     stages with bulk copies (no barriers between warps, loads far ahead);
//   * the up to 8 query heads that share a key head are the rows of
//     mma.m16n8k16 (one query row per head: a 128-row tcgen05 tile would be
//     empty for the most part, and at 8 rows the instruction is not the bound);
//     4-bit codes become bf16 operands with one bit operation per pair (128 + code
//     is exact in bf16) and for values a subtraction (code - 8 is too), the steps
//     and least values are applied to the fp32 scores and to the probabilities,
//     never to rounded keys or values;
//   * probabilities enter the second product as the sum of two bf16 numbers in
//     the unused rows 8..15 (relative error 2^-16 at most), so the result carries the
//     precision of fp32 probabilities.
// A long cache is split over CTAs; the last one to finish joins the partial
// results in the order of the splits (fixed order: no run-to-run differences).
//
// Measured: bf16, 64 sequences x 16 heads of 128 x 4096 slots, 70% of them held (ragged
// lengths, 4 idle) 216 us, 6.95 TB/s (above the rate of a copy: it only reads); all held
// 332 us, 6.47 TB/s. 4 bits the same 119 us, 3.9 TB/s (all held 166 us, 4.05 TB/s), bound
// by the integer pipe that makes operands of the codes (64% of its cycles, DRAM 47%).
// 16 sequences x 2 key heads x 8 query heads x 16384 slots, 64% held, 49 us, 1.1 TB/s
// (all held 61 us): each sequence is cut into as many parts as all slots would be, so the
// longest CTA has 1280 keys where an even division of the held ones is 759, and the SMs
// are active half of the time. One sequence x 12 heads of 64 x 32768 slots 21 us,
// 1.5 TB/s, latency (SMs active 58%); one sequence x 12 heads x 700 slots in bf16 7 us,
// latency.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <map>
#include <string>
#include <utility>

#include "common.h"
#include "ptx.cuh"

namespace dst {
namespace kv_cache {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kRows = 8;  // query heads per CTA
constexpr int kMostCtas = 4;  // CTAs per SM of any step kernel

// ------------------------------------------------------------ row formats
// 8 channels of a row as one lane holds them.
__device__ __forceinline__ void unpack8(const uint4& u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

struct Quant8 {
  uint32_t code[8];
  uint32_t param;  // step (low half) and least value (high half), bf16
};

// Codes of this lane's 8 channels; the 4 lanes of an aligned quad hold a group.
// Division and rounding are the IEEE operations, so any implementation of the
// definition gets the same codes.
__device__ __forceinline__ Quant8 quantize8(const float (&x)[8]) {
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = min_nan(lo, x[i]);
    hi = max_nan(hi, x[i]);
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffff, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffff, hi, o));
  }
  const __nv_bfloat16 step16 = __float2bfloat16_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.f));
  const __nv_bfloat16 low16 = __float2bfloat16_rn(lo);
  const float step = __bfloat162float(step16);
  Quant8 q;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float c = step > 0.f ? __fdiv_rn(__fsub_rn(x[i], lo), step) : 0.f;
    q.code[i] = static_cast<uint32_t>(fminf(fmaxf(rintf(c), 0.f), 15.f));
  }
  q.param = static_cast<uint32_t>(__bfloat16_as_ushort(step16)) |
            (static_cast<uint32_t>(__bfloat16_as_ushort(low16)) << 16);
  return q;
}

__device__ __forceinline__ float param_step(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float param_low(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }
// What code 8 stands for.
__device__ __forceinline__ float param_middle(uint32_t p) { return fmaf(8.f, param_step(p), param_low(p)); }

// Layout of a packed row of DP channels, NG = DP / 32 groups.
//   keys:   word (t, g), t = 0..3, at 4 (t NG + g): the channels g*32 + t*8 + c;
//           nibble c/2 + 4 (c & 1), so that (word >> 4 i) & 0x000f000f is the
//           pair of channels 2 i, 2 i + 1
//   values: half-word (n, g), n = 0..7, at 2 (n NG + g): channels g*32 + n*4 + j
// Both are what one thread of the mma needs of a row, side by side.
__device__ __forceinline__ uint32_t key_word(const uint32_t (&c)[8]) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) w |= c[i] << (4 * ((i >> 1) + 4 * (i & 1)));
  return w;
}

template <int DP>
__device__ __forceinline__ void put_key8(uint8_t* row, int i, const uint32_t (&c)[8]) {
  *reinterpret_cast<uint32_t*>(row + 4 * ((i & 3) * (DP / 32) + (i >> 2))) = key_word(c);
}

template <int DP>
__device__ __forceinline__ void put_value8(uint8_t* row, int i, const uint32_t (&c)[8]) {
  constexpr int NG = DP / 32;
  const int g = i >> 2, n = (i & 3) * 2;
#pragma unroll
  for (int e = 0; e < 2; ++e)
    *reinterpret_cast<uint16_t*>(row + 2 * ((n + e) * NG + g)) =
        static_cast<uint16_t>(c[4 * e] | (c[4 * e + 1] << 4) | (c[4 * e + 2] << 8) | (c[4 * e + 3] << 12));
}

template <int DP>
__device__ __forceinline__ void get_key8(const uint8_t* row, int i, uint32_t (&c)[8]) {
  const uint32_t w = *reinterpret_cast<const uint32_t*>(row + 4 * ((i & 3) * (DP / 32) + (i >> 2)));
#pragma unroll
  for (int j = 0; j < 8; ++j) c[j] = (w >> (4 * ((j >> 1) + 4 * (j & 1)))) & 15u;
}

template <int DP>
__device__ __forceinline__ void get_value8(const uint8_t* row, int i, uint32_t (&c)[8]) {
  constexpr int NG = DP / 32;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const uint32_t w = *reinterpret_cast<const uint16_t*>(row + 2 * (((i & 3) * 2 + e) * NG + (i >> 2)));
#pragma unroll
    for (int j = 0; j < 4; ++j) c[4 * e + j] = (w >> (4 * j)) & 15u;
  }
}

__device__ __forceinline__ void store8f(float* dst, const float (&x)[8]) {
  *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
  *reinterpret_cast<float4*>(dst + 4) = make_float4(x[4], x[5], x[6], x[7]);
}

__device__ __forceinline__ void values8(const Quant8& q, float (&x)[8]) {
  const float step = param_step(q.param), low = param_low(q.param);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = fmaf(static_cast<float>(q.code[i]), step, low);  // the product is exact
}

// Where the cache of one operand (keys or values) lies: rows of `slots_alloc`
// (a multiple of the tile) per (sequence, key head).
struct Store {
  uint8_t* rows;     // bf16 rows of DP, or packed rows of DP / 2 bytes
  uint32_t* params;  // 4 bits: NG per row
};

struct Ring {
  int64_t W, S;
  int alloc;  // rows allocated per (sequence, key head)
  __device__ __forceinline__ int64_t slot(int64_t p) const { return p < S ? p : S + (p - S) % W; }
};

struct Positions {  // int64, one per sequence
  int64_t* p;
  int64_t stride;
  __device__ __forceinline__ int64_t& operator[](int b) const { return p[b * stride]; }
};

struct View {  // k or v rows: element strides, unit inner stride
  const __nv_bfloat16* p;
  int64_t b, h, t;
};

__device__ __forceinline__ uint4 load8(const __nv_bfloat16* row, int i, int D) {
  return i * 8 < D ? *reinterpret_cast<const uint4*>(row + i * 8) : make_uint4(0, 0, 0, 0);
}

// ------------------------------------------------------------- fill and read
// The rows of the prompts' visible tokens into their slots. DP/8 lanes per row;
// row i of a (sequence, head) is token i while that is a sink, then the tokens
// of the last window.
template <int DP, int BITS>
__global__ void __launch_bounds__(256)
    fill_kernel(const View k, const View v, const Positions lengths, const Positions pos, Store ks, Store vs,
                const Ring ring, int T, int rows, int Hk, int D, int* status) {
  constexpr int L = DP / 8;
  const int64_t r = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / L;
  const int i = threadIdx.x % L;
  const int b = blockIdx.z, hk = blockIdx.y >> 1;
  const bool value = blockIdx.y & 1;
  int64_t len = lengths.p ? lengths[b] : T;
  if (len < 0 || len > T) {
    if (threadIdx.x == 0) record_status(status, kBadArgument);
    len = len < 0 ? 0 : T;
  }
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) pos[b] = len;
  const int64_t tail = len - ring.W > ring.S ? len - ring.W : ring.S;
  const int64_t token = r < ring.S ? r : tail + (r - ring.S);
  const bool there = r < rows && token < len;
  if (!__any_sync(0xffffffff, there)) return;
  const View& x = value ? v : k;
  const Store& s = value ? vs : ks;
  const int64_t row = (static_cast<int64_t>(b) * Hk + hk) * ring.alloc + (there ? ring.slot(token) : 0);
  const uint4 u = there ? load8(x.p + b * x.b + token * x.t + hk * x.h, i, D) : make_uint4(0, 0, 0, 0);
  if (BITS == 16) {
    if (there) *reinterpret_cast<uint4*>(s.rows + row * (DP * 2) + i * 16) = u;
  } else {
    float f[8];
    unpack8(u, f);
    const Quant8 q = quantize8(f);
    if (there) {
      uint8_t* dst = s.rows + row * (DP / 2);
      if (value)
        put_value8<DP>(dst, i, q.code);
      else
        put_key8<DP>(dst, i, q.code);
      if ((i & 3) == 0) s.params[row * (DP / 32) + (i >> 2)] = q.param;
    }
  }
}

// The held rows in slot order (0 where no token is): bf16, or fp32 for 4 bits.
template <int DP, int BITS>
__global__ void __launch_bounds__(256)
    read_kernel(const Store ks, const Store vs, const Positions pos, void* __restrict__ ko, void* __restrict__ vo,
                const Ring ring, int slots, int Hk, int D) {
  constexpr int L = DP / 8;
  const int64_t r = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / L;
  const int i = threadIdx.x % L;
  if (r >= slots || i * 8 >= D) return;
  const int b = blockIdx.z, hk = blockIdx.y >> 1;
  const bool value = blockIdx.y & 1;
  const Store& s = value ? vs : ks;
  const bool there = r < pos[b];
  const int64_t bh = static_cast<int64_t>(b) * Hk + hk, row = bh * ring.alloc + r;
  const int64_t dst = (bh * slots + r) * D + i * 8;
  if (BITS == 16) {
    *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(value ? vo : ko) + dst) =
        there ? *reinterpret_cast<const uint4*>(s.rows + row * (DP * 2) + i * 16) : make_uint4(0, 0, 0, 0);
  } else {
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (there) {
      Quant8 q;
      if (value)
        get_value8<DP>(s.rows + row * (DP / 2), i, q.code);
      else
        get_key8<DP>(s.rows + row * (DP / 2), i, q.code);
      q.param = s.params[row * (DP / 32) + (i >> 2)];
      values8(q, f);
    }
    store8f(reinterpret_cast<float*>(value ? vo : ko) + dst, f);
  }
}

// ------------------------------------------------------------------- step
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0,
                                         float c1, float c2, float c3) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

// 8 x 8 b16 matrix, a row per 4 lanes, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}

// x and y as sums of two bf16 numbers each: hi pair, lo pair.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = pack2(x, y);
  lo = pack2(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xffff0000u));
}

// What the 8 query rows of the mma are.
enum Rows {
  kBf16Heads,      // bf16 cache: a head each
  kPackedHeads,    // 4 bits: a head each; every thread handles all groups of its keys
  kPackedGroups,   // 4 bits, few heads per key head: (head, group of 32 channels) each, so that a
                   // thread applies the steps and least values of its own group only (16 heads
                   // of 128 without sharing: 153 us against 198 with a row per head)
};

template <int DP, int ROWS>
struct StepCfg {
  static constexpr bool kPacked = ROWS != kBf16Heads;
  static constexpr int NG = DP / 32;
  static constexpr int kHeads = ROWS == kPackedGroups ? kRows / NG : kRows;  // per CTA
  static constexpr int kRowBytes = kPacked ? DP / 2 : DP * 2;
  static constexpr int kParamBytes = kPacked ? NG * 4 : 0;
  // keys per stage of a warp's ring
  static constexpr int KT = kPacked ? (DP == 64 ? 64 : 32) : (DP == 64 ? 32 : 16);
  static constexpr int kStages = kPacked ? 2 : 3;
  static constexpr int kOperand = KT * kRowBytes;  // keys or values of a stage
  static constexpr int kStage = 2 * kOperand + 2 * KT * kParamBytes;
  static constexpr int kRingBytes = kWarps * kStages * kStage;
  // the new token's row, laid out like a stage of 16 keys
  static constexpr int kNew = 2 * 16 * (kRowBytes + kParamBytes);
  static constexpr int kJoin = kWarps * kRows * (DP + 2) * 4;  // over the ring at the end
  static constexpr int kSumStages = 256 / KT;  // packed: the mma sums go to fp32 sums after so many
  static constexpr int kSums = kPacked ? kThreads * (ROWS == kPackedGroups ? 4 : DP / 8) * 2 * 4 : 0;
  static constexpr int kMaxSplits = kRingBytes / (4 * kRows) - 1;  // their weights too
  static constexpr int kSmem = (kRingBytes > kJoin ? kRingBytes : kJoin) + kNew + kSums + kWarps * kStages * 8 + 16 + 1024;
  static constexpr int kCtas = !kPacked ? 2 : ROWS == kPackedGroups ? 4 : DP == 64 ? 4 : 3;  // per SM
  static_assert(kCtas <= kMostCtas, "the arrival counters are too few");
  static constexpr int kSub = ROWS == kPackedHeads ? 1 : KT % 32 == 0 ? 2 : 1;  // subtiles of 16 keys at a time
};

struct StepArgs {
  const __nv_bfloat16* q;
  int64_t q_b, q_h;
  View k, v;  // the new token's rows
  Positions pos;
  Store ks, vs;
  __nv_bfloat16* out;      // [B, H, D]
  float *stored_k, *stored_v;  // optional [B, Hk, D]: what the new row stands for
  float* partial;          // [B * Hk * chunks][splits][kRows][DP + 2]
  int* arrived;            // [B * Hk * chunks] where splits > 1, 0 between launches
  Ring ring;
  int slots, Hk, G, D, chunks, splits;
  float scale_log2;
  int* status;
};

// The warp's running result for the 8 query rows: thread (n = lane / 4, t =
// lane % 4) holds for row n the output channels of columns 2t, 2t + 1 of each
// 8-column tile.
//
// Packed rows: the scores are computed transposed (a row of the mma is a key, so
// all 16 rows are used and the codes of a key go in as they come), so a thread's
// m and l are those of the query rows 2t, 2t + 1, over its keys n, n + 8. The codes of
// keys enter as 128 + code, those of values as code - 8; what code 8 stands for makes a
// term that is the same for all channels of a group, the sum over keys of
// p (low + 8 step), in each group's own fp32 sum (one that the groups share would spread
// a group that stands for NaN over all). Values have to lie around zero: each
// accumulation of the mma cuts the sum's low bits, so a sum over thousands of keys that a
// bias makes larger than the result loses the result's. With 128 + code, and the bias
// taken back by a sum of its own, the error grew with the keys a warp adds up, to 11% at
// 8192. For the same reason the sums go on to fp32 sums every 256 keys. A score is a sum of 4 or 8 products, where the bias costs nothing that shows (the
// same error to 6 digits, also for queries 16 times as large) and the subtraction 3%.
template <int DP, int ROWS>
struct State {
  static constexpr int NG = DP / 32;
  // packed groups: columns 2t, 2t + 1 are groups of one head, and the output is of the
  // row's own group
  static constexpr int kHeads = ROWS == kPackedHeads ? 2 : 1;
  static constexpr int kTiles = ROWS == kPackedGroups ? 4 : DP / 8;
  float m[kHeads], l[kHeads];
  float o[kTiles][4];  // [tile]: 0, 1 high parts, 2, 3 low parts of the probabilities
  float low[ROWS == kPackedHeads ? NG : 1][2];  // sum p (low + 8 step) of (group,) query row 2t, 2t + 1
};

// The query rows as mma operands. Packed: also -128 times their sums over groups for
// the query rows 2t, 2t + 1 (packed groups: once), and those sums to be multiplied with the least
// values of a key (packed heads: as three bf16 parts).
template <int DP, int ROWS>
struct Query {
  uint32_t a[DP / 16][2];
  float off[ROWS == kPackedHeads ? DP / 32 : 1][2];
  uint32_t sum[2];
};

// One 16-byte chunk `c` of row `r` of a 128B-swizzled tile of 64 channels.
__device__ __forceinline__ const uint4* swz(const uint8_t* tile, int r, int c) {
  return reinterpret_cast<const uint4*>(tile + r * 128 + ((c ^ (r & 7)) << 4));
}

// As in the prompt's kernel a row keeps its reference maximum until a tile exceeds
// it by 8 (in log2); then the sums of that row are rescaled by this factor.
__device__ __forceinline__ float move_max(float& m, float& l, float mx) {
  if (!(mx > m + 8.f)) return 1.f;
  const float c = exp2f(m - mx);
  m = mx;
  l *= c;
  return c;
}

// NS subtiles of 16 keys each: keys and values at `sk`, `sv`, `tile_rows` rows per
// swizzled tile; bit i of `valid` says whether key i takes part.
template <int DP, int NS>
__device__ __forceinline__ void attend_bf16(State<DP, kBf16Heads>& st, const Query<DP, kBf16Heads>& q,
                                            const uint8_t* sk, const uint8_t* sv, int tile_rows, uint32_t valid,
                                            float scale_log2) {
  const int lane = threadIdx.x & 31, n = lane >> 2, t = lane & 3;
  constexpr uint32_t kAll = NS == 2 ? 0xffffffffu : 0xffffu;
  float s[2 * NS][2];  // scores of columns 2t, 2t + 1 of each 8 keys, row n
#pragma unroll
  for (int i = 0; i < 2 * NS; ++i) {
    const int r = i * 8 + n;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int a = 0; a < DP / 64; ++a) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint4 w = *swz(sk + a * tile_rows * 128, r, 2 * t + c);
        mma16816(acc, q.a[a * 4 + c * 2][0], 0u, q.a[a * 4 + c * 2][1], 0u, w.x, w.y);
        mma16816(acc, q.a[a * 4 + c * 2 + 1][0], 0u, q.a[a * 4 + c * 2 + 1][1], 0u, w.z, w.w);
      }
    }
    s[i][0] = acc[0];
    s[i][1] = acc[1];
  }
  float mx = -INFINITY;
  if (valid != kAll) {
#pragma unroll
    for (int i = 0; i < 2 * NS; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (!((valid >> (i * 8 + 2 * t + e)) & 1u)) s[i][e] = -INFINITY;
  }
#pragma unroll
  for (int i = 0; i < 2 * NS; ++i) mx = fmaxf(mx, fmaxf(s[i][0], s[i][1]));
  mx = fmaxf(mx, __shfl_xor_sync(0xffffffff, mx, 1));
  mx = fmaxf(mx, __shfl_xor_sync(0xffffffff, mx, 2)) * scale_log2;
  if (__any_sync(0xffffffff, mx > st.m[0] + 8.f)) {
    const float c = move_max(st.m[0], st.l[0], mx);
#pragma unroll
    for (int i = 0; i < DP / 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) st.o[i][j] *= c;
  }
  const float m_use = st.m[0] == -INFINITY ? 0.f : st.m[0];
#pragma unroll
  for (int i = 0; i < 2 * NS; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      s[i][e] = exp2f(fmaf(s[i][e], scale_log2, -m_use));
      st.l[0] += s[i][e];
    }
#pragma unroll
  for (int u = 0; u < NS; ++u) {
    const int r0 = u * 16 + 2 * t;  // this thread's keys: r0, r0 + 1, r0 + 8, r0 + 9
    const uint32_t in = valid >> r0;
    uint32_t a0, a1, a2, a3;
    split2(s[2 * u][0], s[2 * u][1], a0, a1);
    split2(s[2 * u + 1][0], s[2 * u + 1][1], a2, a3);
#pragma unroll
    for (int a = 0; a < DP / 64; ++a) {
      const uint8_t* tile = sv + a * tile_rows * 128;
      uint4 x[4] = {*swz(tile, r0, n), *swz(tile, r0 + 1, n), *swz(tile, r0 + 8, n), *swz(tile, r0 + 9, n)};
      if (valid != kAll) {  // what lies in a masked row must not meet its zero probability
        const uint4 z = make_uint4(0, 0, 0, 0);
        if (!(in & 1u)) x[0] = z;
        if (!(in & 2u)) x[1] = z;
        if (!(in & 0x100u)) x[2] = z;
        if (!(in & 0x200u)) x[3] = z;
      }
      const uint32_t* w[4] = {&x[0].x, &x[1].x, &x[2].x, &x[3].x};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        mma16816(st.o[a * 8 + 2 * j], a0, a1, a2, a3, __byte_perm(w[0][j], w[1][j], 0x5410),
                 __byte_perm(w[2][j], w[3][j], 0x5410));
        mma16816(st.o[a * 8 + 2 * j + 1], a0, a1, a2, a3, __byte_perm(w[0][j], w[1][j], 0x7632),
                 __byte_perm(w[2][j], w[3][j], 0x7632));
      }
    }
  }
}

// Codes i and i + 4 of a word as a bf16 pair of 128 + code: a shift, and one
// three-input operation for mask and exponent (with both constants in registers; as
// immediates they took one each). Centred: code - 8, by a subtraction (exact).
struct Codes {
  uint32_t mask, exponent, middle;
  __device__ __forceinline__ Codes() {
    asm volatile("mov.u32 %0, 0x000f000f;" : "=r"(mask));
    asm volatile("mov.u32 %0, 0x43004300;" : "=r"(exponent));
    asm volatile("mov.u32 %0, 0x43084308;" : "=r"(middle));
  }
  __device__ __forceinline__ uint32_t first(uint32_t w) const {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "r"(mask), "r"(exponent));
    return r;
  }
  __device__ __forceinline__ void all(uint32_t w, uint32_t (&pair)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) pair[i] = first(w >> (4 * i));
  }
  __device__ __forceinline__ void centred(uint32_t w, uint32_t (&pair)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      pair[i] = first(w >> (4 * i));
      asm("sub.bf16x2 %0, %0, %1;" : "+r"(pair[i]) : "r"(middle));
    }
  }
};

// The same over packed rows with parameters `pk`, `pv`. Thread (n, t) computes the
// scores of keys n and n + 8 of a subtile for query rows 2t, 2t + 1.
template <int DP, int ROWS, int NS>
__device__ __forceinline__ void attend_packed(State<DP, ROWS>& st, const Query<DP, ROWS>& q, const uint8_t* sk,
                                              const uint8_t* sv, const uint32_t* pk, const uint32_t* pv, uint32_t valid,
                                              float scale_log2) {
  using St = State<DP, ROWS>;
  constexpr int NG = DP / 32, NH = St::kHeads;
  const int lane = threadIdx.x & 31, n = lane >> 2, t = lane & 3;
  const Codes codes;
  const int g0 = (2 * t) & (NG - 1);  // packed groups: column 2t + e is group g0 + e
  constexpr uint32_t kAll = NS == 2 ? 0xffffffffu : 0xffffu;
  float s[NS][2][NH];  // [subtile][key n, n + 8][head]
#pragma unroll
  for (int u = 0; u < NS; ++u) {
    uint32_t w[2][NG];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint8_t* p = sk + (u * 16 + k * 8 + n) * (DP / 2) + t * (DP / 8);
      if constexpr (NG == 2) {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        w[k][0] = x.x, w[k][1] = x.y;
      } else {
        const uint4 x = *reinterpret_cast<const uint4*>(p);
        w[k][0] = x.x, w[k][1] = x.y, w[k][2] = x.z, w[k][3] = x.w;
      }
    }
    // A operands of group g: 16 keys x its first and its last 16 channels
    auto key_codes = [&](int g, uint32_t (&a)[4], uint32_t (&b)[4]) {
      uint32_t x[4], y[4];
      codes.all(w[0][g], x);
      codes.all(w[1][g], y);
      a[0] = x[0], a[1] = y[0], a[2] = x[1], a[3] = y[1];
      b[0] = x[2], b[1] = y[2], b[2] = x[3], b[3] = y[3];
    };
    const uint32_t* par = pk + (u * 16 + n) * NG;  // of key n; key n + 8: 8 NG further
    if constexpr (ROWS == kPackedGroups) {
      float acc[4] = {q.off[0][0] * -128.f, q.off[0][1] * -128.f, q.off[0][0] * -128.f, q.off[0][1] * -128.f};
#pragma unroll
      for (int g = 0; g < NG; ++g) {  // columns of other groups hold zeros there
        uint32_t a[4], b[4];
        key_codes(g, a, b);
        mma16816(acc, a, q.a[2 * g][0], q.a[2 * g][1], acc[0], acc[1], acc[2], acc[3]);
        mma16816(acc, b, q.a[2 * g + 1][0], q.a[2 * g + 1][1], acc[0], acc[1], acc[2], acc[3]);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint2 x = *reinterpret_cast<const uint2*>(par + k * 8 * NG + g0);
        float v = fmaf(param_step(x.x), acc[2 * k], param_low(x.x) * q.off[0][0]) +
                  fmaf(param_step(x.y), acc[2 * k + 1], param_low(x.y) * q.off[0][1]);
        if (NG == 4) v += __shfl_xor_sync(0xffffffff, v, 1);  // the head's other two groups
        s[u][k][0] = v;
      }
    } else {
      // least values times query sums: k-slots (2t, 2t + 1) and (2t + 8, 2t + 9)
      uint32_t low[4];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint2 x = *reinterpret_cast<const uint2*>(par + k * 8 * NG + (NG == 4 ? 2 * (t & 1) : 0));
        low[k] = __byte_perm(x.x, x.y, 0x7632);
        low[2 + k] = NG == 4 && t < 2 ? low[k] : 0u;
      }
      float sc[4];
      mma16816(sc, low, q.sum[0], q.sum[1], 0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float acc[4];
        uint32_t a[4], b[4];
        key_codes(g, a, b);
        mma16816(acc, a, q.a[2 * g][0], q.a[2 * g][1], q.off[g][0], q.off[g][1], q.off[g][0], q.off[g][1]);
        mma16816(acc, b, q.a[2 * g + 1][0], q.a[2 * g + 1][1], acc[0], acc[1], acc[2], acc[3]);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float step = param_step(par[k * 8 * NG + g]);
          sc[2 * k] = fmaf(step, acc[2 * k], sc[2 * k]);
          sc[2 * k + 1] = fmaf(step, acc[2 * k + 1], sc[2 * k + 1]);
        }
      }
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < NH; ++e) s[u][k][e] = sc[2 * k + e];
    }
  }
  const bool masked = valid != kAll;
  if (masked) {
#pragma unroll
    for (int u = 0; u < NS; ++u)
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (!((valid >> (u * 16 + k * 8 + n)) & 1u)) {
#pragma unroll
          for (int e = 0; e < NH; ++e) s[u][k][e] = -INFINITY;
        }
  }
  float mx[NH], m_use[NH];
  bool need = false;
#pragma unroll
  for (int e = 0; e < NH; ++e) {
    mx[e] = -INFINITY;
#pragma unroll
    for (int u = 0; u < NS; ++u) mx[e] = fmaxf(mx[e], fmaxf(s[u][0][e], s[u][1][e]));
    mx[e] *= scale_log2;
    need = need || mx[e] > st.m[e] + 8.f;
  }
  if (__any_sync(0xffffffff, need)) {  // only now the maxima of all keys are needed
    float c[NH];
#pragma unroll
    for (int e = 0; e < NH; ++e) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffff, mx[e], o));
      c[e] = move_max(st.m[e], st.l[e], mx[e]);
    }
    // the factor of output row n lies with the threads that hold column n
    const float even = __shfl_sync(0xffffffff, c[0], n >> 1), odd = __shfl_sync(0xffffffff, c[NH - 1], n >> 1);
    const float cn = (n & 1) ? odd : even;
#pragma unroll
    for (int i = 0; i < St::kTiles; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) st.o[i][j] *= cn;
#pragma unroll
    for (int g = 0; g < (ROWS == kPackedHeads ? NG : 1); ++g)
#pragma unroll
      for (int e = 0; e < 2; ++e) st.low[g][e] *= c[NH == 2 ? e : 0];
  }
#pragma unroll
  for (int e = 0; e < NH; ++e) {
    m_use[e] = st.m[e] == -INFINITY ? 0.f : st.m[e];
#pragma unroll
    for (int u = 0; u < NS; ++u)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        s[u][k][e] = exp2f(fmaf(s[u][k][e], scale_log2, -m_use[e]));
        st.l[e] += s[u][k][e];
      }
  }
#pragma unroll
  for (int u = 0; u < NS; ++u) {
    const int r0 = u * 16 + 2 * t;  // values of this thread: keys r0, r0 + 1, r0 + 8, r0 + 9
    uint32_t w[4][NG / 2];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint8_t* x = sv + (r0 + (j & 1) + (j >> 1) * 8) * (DP / 2) + n * (DP / 16);
      if constexpr (NG == 2) {
        w[j][0] = *reinterpret_cast<const uint32_t*>(x);
      } else {
        const uint2 y = *reinterpret_cast<const uint2*>(x);
        w[j][0] = y.x, w[j][1] = y.y;
      }
    }
    bool on[2] = {true, true};
    if (masked) {  // what lies in a masked row must not meet its zero probability
      on[0] = (valid >> (u * 16 + n)) & 1u;
      on[1] = (valid >> (u * 16 + 8 + n)) & 1u;
    }
    const uint32_t* par = pv + (u * 16 + n) * NG;
    auto values = [&](int g, int tile0, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
      const uint32_t lo = __byte_perm(w[0][g >> 1], w[1][g >> 1], (g & 1) ? 0x7632 : 0x5410);
      const uint32_t hi = __byte_perm(w[2][g >> 1], w[3][g >> 1], (g & 1) ? 0x7632 : 0x5410);
      uint32_t x[4], y[4];
      codes.centred(lo, x);
      codes.centred(hi, y);
#pragma unroll
      for (int j = 0; j < 4; ++j) mma16816(st.o[tile0 + j], a0, a1, a2, a3, x[j], y[j]);
    };
    if constexpr (ROWS == kPackedGroups) {
      uint32_t hi[2], lo[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint2 x = *reinterpret_cast<const uint2*>(par + k * 8 * NG + g0);
        if (masked && !on[k]) x = make_uint2(0u, 0u);
        const float p = s[u][k][0];
        st.low[0][0] = fmaf(p, param_middle(x.x), st.low[0][0]);
        st.low[0][1] = fmaf(p, param_middle(x.y), st.low[0][1]);
        split2(p * param_step(x.x), p * param_step(x.y), hi[k], lo[k]);
      }
      const uint32_t a0 = transpose8(hi[0]), a1 = transpose8(lo[0]), a2 = transpose8(hi[1]), a3 = transpose8(lo[1]);
#pragma unroll
      for (int g = 0; g < NG; ++g) {  // into the rows of group g alone: one set of sums for all
        const bool mine = (n & (NG - 1)) == g;
        values(g, 0, mine ? a0 : 0u, mine ? a1 : 0u, mine ? a2 : 0u, mine ? a3 : 0u);
      }
    } else {
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        uint32_t hi[2], lo[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t x = par[k * 8 * NG + g];
          if (masked && !on[k]) x = 0u;
          const float step = param_step(x);
#pragma unroll
          for (int e = 0; e < 2; ++e) st.low[g][e] = fmaf(s[u][k][e], param_middle(x), st.low[g][e]);
          split2(s[u][k][0] * step, s[u][k][1] * step, hi[k], lo[k]);
        }
        const uint32_t a0 = transpose8(hi[0]), a1 = transpose8(lo[0]), a2 = transpose8(hi[1]), a3 = transpose8(lo[1]);
        values(g, g * 4, a0, a1, a2, a3);
      }
    }
  }
}

// The output sums so far into fp32 sums in shared memory (first: nothing is there yet),
// or at the end those added to what the mma holds; `m` are the maxima they go by.
// Rounded to nearest, a few hundred keys at a time, they do not lose what the mma cuts
// off: with a constant large channel in a group, whose other codes are far from the
// middle, 8192 keys in one mma sum cost the other channels 1%.
template <int DP, int ROWS>
__device__ __forceinline__ float sums_factor(const State<DP, ROWS>& st, float (&m)[State<DP, ROWS>::kHeads]) {
  constexpr int NH = State<DP, ROWS>::kHeads;
  const int n = (threadIdx.x & 31) >> 2;
  float c[NH];
#pragma unroll
  for (int e = 0; e < NH; ++e) {
    c[e] = m[e] == st.m[e] ? 1.f : exp2f(m[e] - st.m[e]);
    m[e] = st.m[e];
  }
  // the factor of output row n lies with the threads that hold column n
  const float even = __shfl_sync(0xffffffff, c[0], n >> 1), odd = __shfl_sync(0xffffffff, c[NH - 1], n >> 1);
  return (n & 1) ? odd : even;
}

template <int DP, int ROWS>
__device__ __forceinline__ void put_sums(State<DP, ROWS>& st, float* sums, float (&m)[State<DP, ROWS>::kHeads], bool first) {
  const float c = sums_factor<DP, ROWS>(st, m);
#pragma unroll
  for (int i = 0; i < State<DP, ROWS>::kTiles; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float* x = sums + (2 * i + j) * kThreads;
      const float now = st.o[i][j] + st.o[i][j + 2];
      *x = first ? now : fmaf(*x, c, now);
      st.o[i][j] = st.o[i][j + 2] = 0.f;
    }
}

template <int DP, int ROWS>
__device__ __forceinline__ void add_sums(State<DP, ROWS>& st, const float* sums, float (&m)[State<DP, ROWS>::kHeads]) {
  const float c = sums_factor<DP, ROWS>(st, m);
#pragma unroll
  for (int i = 0; i < State<DP, ROWS>::kTiles; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) st.o[i][j] = fmaf(sums[(2 * i + j) * kThreads], c, st.o[i][j]);
}

template <int DP, int ROWS, int NS>
__device__ __forceinline__ void attend(State<DP, ROWS>& st, const Query<DP, ROWS>& q, const uint8_t* sk,
                                       const uint8_t* sv, const uint32_t* pk, const uint32_t* pv, int tile_rows,
                                       uint32_t valid, float scale_log2) {
  if constexpr (ROWS == kBf16Heads)
    attend_bf16<DP, NS>(st, q, sk, sv, tile_rows, valid, scale_log2);
  else
    attend_packed<DP, ROWS, NS>(st, q, sk, sv, pk, pv, valid, scale_log2);
}

// Output channel of tile `tile`, column `n`.
template <int DP, int ROWS>
__device__ __forceinline__ int channel_of(int tile, int n) {
  return ROWS == kBf16Heads ? (tile >> 3) * 64 + n * 8 + (tile & 7) : (tile >> 2) * 32 + n * 4 + (tile & 3);
}

template <int DP, int ROWS>
__global__ void __launch_bounds__(kThreads, StepCfg<DP, ROWS>::kCtas)
    step_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const StepArgs a) {
  using C = StepCfg<DP, ROWS>;
  constexpr int NG = C::NG, KT = C::KT, ST = C::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* fresh = smem + (C::kRingBytes > C::kJoin ? C::kRingBytes : C::kJoin);
  float* sums = reinterpret_cast<float*>(fresh + C::kNew) + threadIdx.x;  // this thread's, kThreads apart
  uint64_t* bars = reinterpret_cast<uint64_t*>(fresh + C::kNew + C::kSums);
  int* last_flag = reinterpret_cast<int*>(bars + kWarps * ST);

  const int split = blockIdx.x, b = blockIdx.z;
  const int hk = blockIdx.y / a.chunks, chunk = blockIdx.y % a.chunks;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = lane >> 2, t = lane & 3;
  const int heads = min(C::kHeads, a.G - chunk * C::kHeads);  // query heads of this CTA
  const int h0 = hk * a.G + chunk * C::kHeads;
  const int64_t p = a.pos[b];
  if (p < 0) {  // an idle sequence: nothing to see, nothing to store
    if (split == 0) {
      for (int i = threadIdx.x; i < heads * a.D; i += kThreads)
        a.out[(static_cast<int64_t>(b) * a.Hk * a.G + h0) * a.D + i] = __float2bfloat16(0.f);
      if (a.stored_k && chunk == 0)
        for (int i = threadIdx.x; i < a.D; i += kThreads) {
          a.stored_k[(static_cast<int64_t>(b) * a.Hk + hk) * a.D + i] = 0.f;
          a.stored_v[(static_cast<int64_t>(b) * a.Hk + hk) * a.D + i] = 0.f;
        }
    }
    return;
  }
  // the held rows, without the new token and without the row it replaces
  const int held = static_cast<int>(p < a.slots ? p : a.slots);
  const int fresh_slot = static_cast<int>(a.ring.slot(p));
  int per = (held + a.splits - 1) / a.splits;
  per = max((per + KT - 1) / KT * KT, kWarps * KT);
  const int active = max(1, (held + per - 1) / per);
  if (split >= active) return;
  const int first = split * per, last = min(held, first + per);
  const int tiles = (last - first + KT - 1) / KT;  // of this CTA; warp w takes w, w + 4, ...
  const int64_t bh = static_cast<int64_t>(b) * a.Hk + hk;
  const int64_t base = bh * a.ring.alloc;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kWarps * ST; ++i) mbar_init(&bars[i], 1);
    fence_barrier_init();
  }
  __syncthreads();

  uint8_t* ring = smem + warp * ST * C::kStage;
  uint64_t* full = bars + warp * ST;
  auto load = [&](int i) {  // tile i of this warp (one lane)
    const int stage = i % ST;
    const int64_t row = base + first + (warp + i * kWarps) * KT;
    uint8_t* dst = ring + stage * C::kStage;
    mbar_arrive_expect_tx(&full[stage], C::kStage);
    if (!C::kPacked) {
#pragma unroll
      for (int c = 0; c < DP / 64; ++c) {
        tma_load_2d(dst + c * KT * 128, &tmK, &full[stage], c * 64, static_cast<int>(row));
        tma_load_2d(dst + C::kOperand + c * KT * 128, &tmV, &full[stage], c * 64, static_cast<int>(row));
      }
    } else {
      bulk_load(dst, a.ks.rows + row * C::kRowBytes, C::kOperand, &full[stage]);
      bulk_load(dst + C::kOperand, a.vs.rows + row * C::kRowBytes, C::kOperand, &full[stage]);
      bulk_load(dst + 2 * C::kOperand, a.ks.params + row * NG, KT * C::kParamBytes, &full[stage]);
      bulk_load(dst + 2 * C::kOperand + KT * C::kParamBytes, a.vs.params + row * NG, KT * C::kParamBytes, &full[stage]);
    }
  };
  const int mine = tiles > warp ? (tiles - warp + kWarps - 1) / kWarps : 0;
  int loaded = 0;
  if (lane == 0)
    for (; loaded < min(mine, ST); ++loaded) load(loaded);
  __syncwarp();

  // Query rows as the A operand. Channels of k-step kk that thread t holds: for
  // bf16 keys (kk/4)*64 + t*16 + (kk%4)*4 + 0..3, for packed keys (kk/2)*32 +
  // t*8 + (kk%2)*4 + 0..3. Where rows are (head, group), a row's other groups are 0.
  const int row_head = ROWS == kPackedGroups ? n / NG : n, row_group = n & (NG - 1);
  Query<DP, ROWS> q;
  {
    const __nv_bfloat16* qrow = a.q + b * a.q_b + (h0 + row_head) * a.q_h;
    float sum[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) sum[g] = 0.f;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      const int c = C::kPacked ? (kk >> 1) * 32 + t * 8 + (kk & 1) * 4 : (kk >> 2) * 64 + t * 16 + (kk & 3) * 4;
      const bool on = row_head < heads && c < a.D && (ROWS != kPackedGroups || (kk >> 1) == row_group);
      const uint2 w = on ? *reinterpret_cast<const uint2*>(qrow + c) : make_uint2(0u, 0u);
      q.a[kk][0] = w.x;
      q.a[kk][1] = w.y;
      if (C::kPacked)
        sum[kk >> 1] += (__uint_as_float(w.x << 16) + __uint_as_float(w.x & 0xffff0000u)) +
                        (__uint_as_float(w.y << 16) + __uint_as_float(w.y & 0xffff0000u));
    }
    if (C::kPacked) {
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        sum[g] += __shfl_xor_sync(0xffffffff, sum[g], 1);
        sum[g] += __shfl_xor_sync(0xffffffff, sum[g], 2);
      }
      if constexpr (ROWS == kPackedGroups) {
        float own = 0.f;  // zero but for the row's own group
#pragma unroll
        for (int g = 0; g < NG; ++g) own += sum[g];
#pragma unroll
        for (int e = 0; e < 2; ++e) q.off[0][e] = __shfl_sync(0xffffffff, own, (2 * t + e) * 4);
      } else if constexpr (ROWS == kPackedHeads) {
        // three bf16 parts of each sum; thread t holds part t / 2 of groups 2 (t % 2), + 1
        // and, for t < 2, the third part (two groups: part t)
        const int pair = NG == 4 ? 2 * (t & 1) : 0, part = NG == 4 ? t >> 1 : t;
        const float s0 = pair ? sum[NG - 2] : sum[0], s1 = pair ? sum[NG - 1] : sum[1];
        uint32_t hi, mid, lo, rest;
        split2(s0, s1, hi, mid);
        const float r0 = s0 - __uint_as_float(hi << 16), r1 = s1 - __uint_as_float(hi & 0xffff0000u);
        split2(r0 - __uint_as_float(mid << 16), r1 - __uint_as_float(mid & 0xffff0000u), lo, rest);
        q.sum[0] = part == 0 ? hi : part == 1 ? mid : (NG == 2 && part == 2) ? lo : 0u;
        q.sum[1] = NG == 4 && t < 2 ? lo : 0u;
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
          for (int e = 0; e < 2; ++e) q.off[g][e] = -128.f * __shfl_sync(0xffffffff, sum[g], (2 * t + e) * 4);
      }
    }
  }

  State<DP, ROWS> st;
#pragma unroll
  for (int e = 0; e < State<DP, ROWS>::kHeads; ++e) st.m[e] = -INFINITY, st.l[e] = 0.f;
#pragma unroll
  for (int g = 0; g < (ROWS == kPackedHeads ? NG : 1); ++g) st.low[g][0] = st.low[g][1] = 0.f;
#pragma unroll
  for (int i = 0; i < State<DP, ROWS>::kTiles; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) st.o[i][j] = 0.f;

  // The new token: its row into the cache (once) and, laid out as a tile of one
  // key, into this warp's result.
  if (split == 0 && warp == 0) {
    constexpr int L = DP / 8;
    const bool value = lane >= L;
    const int i = lane % L;
    const View& x = value ? a.v : a.k;
    const Store& s = value ? a.vs : a.ks;
    const bool on = lane < 2 * L;
    const uint4 u = on ? load8(x.p + b * x.b + hk * x.h, i, a.D) : make_uint4(0, 0, 0, 0);
    const int64_t row = base + fresh_slot;
    uint8_t* tile = fresh + (value ? 16 * C::kRowBytes : 0);
    uint32_t* params = reinterpret_cast<uint32_t*>(fresh + 32 * C::kRowBytes) + (value ? 16 * NG : 0);
    float f[8];
    unpack8(u, f);
    if (!C::kPacked) {
      if (on) {
        *reinterpret_cast<uint4*>(tile + (i >> 3) * 16 * 128 + ((i & 7) << 4)) = u;  // row 0: chunks in order
        if (chunk == 0) *reinterpret_cast<uint4*>(s.rows + row * C::kRowBytes + i * 16) = u;
      }
    } else {
      const Quant8 code = quantize8(f);
      values8(code, f);
      if (on) {
        uint8_t* dst = s.rows + row * C::kRowBytes;
        if (value) {
          put_value8<DP>(tile, i, code.code);
          if (chunk == 0) put_value8<DP>(dst, i, code.code);
        } else {
          put_key8<DP>(tile, i, code.code);
          if (chunk == 0) put_key8<DP>(dst, i, code.code);
        }
        if ((i & 3) == 0) {
          params[i >> 2] = code.param;
          if (chunk == 0) s.params[row * NG + (i >> 2)] = code.param;
        }
      }
    }
    if (a.stored_k && chunk == 0 && on && i * 8 < a.D)
      store8f((value ? a.stored_v : a.stored_k) + bh * a.D + i * 8, f);
    __syncwarp();
    const uint32_t* fp = reinterpret_cast<const uint32_t*>(fresh + 32 * C::kRowBytes);
    attend<DP, ROWS, 1>(st, q, fresh, fresh + 16 * C::kRowBytes, fp, fp + 16 * NG, 16, 1u, a.scale_log2);
  }

  bool ok = true;
  float m_sums[State<DP, ROWS>::kHeads];  // the maxima that the sums in shared memory go by
#pragma unroll
  for (int e = 0; e < State<DP, ROWS>::kHeads; ++e) m_sums[e] = -INFINITY;
  for (int i = 0; i < mine && ok; ++i) {
    const int stage = i % ST;
    ok = __all_sync(0xffffffff, mbar_wait(&full[stage], (i / ST) & 1, a.status, kTimeoutTmaFull));
    if (!ok) break;
    const uint8_t* src = ring + stage * C::kStage;
    const uint32_t* pk = reinterpret_cast<const uint32_t*>(src + 2 * C::kOperand);
    const uint32_t* pv = pk + KT * NG;
    const int row = first + (warp + i * kWarps) * KT;
    constexpr int NS = C::kSub;
#pragma unroll 1
    for (int u = 0; u < KT / (16 * NS); ++u) {
      const int r = row + u * 16 * NS;
      if (r >= last) break;
      constexpr uint32_t kAll = NS == 2 ? 0xffffffffu : 0xffffu;
      uint32_t valid = last - r >= 16 * NS ? kAll : (1u << (last - r)) - 1u;
      if (fresh_slot >= r && fresh_slot < r + 16 * NS) valid &= ~(1u << (fresh_slot - r));
      const int off = u * 16 * NS;
      attend<DP, ROWS, NS>(st, q, src + off * (C::kPacked ? C::kRowBytes : 128),
                           src + C::kOperand + off * (C::kPacked ? C::kRowBytes : 128), pk + off * NG, pv + off * NG,
                           KT, valid, a.scale_log2);
    }
    __syncwarp();
    if (lane == 0 && loaded < mine) load(loaded++);
    __syncwarp();
    if constexpr (C::kPacked)
      if ((i + 1) % C::kSumStages == 0) put_sums<DP, ROWS>(st, sums, m_sums, i + 1 == C::kSumStages);
  }
  if constexpr (C::kPacked)
    if (ok && mine >= C::kSumStages) add_sums<DP, ROWS>(st, sums, m_sums);
  if (!ok && lane == 0)  // a wait expired: no copy may land after the CTA is gone
    for (int i = max(0, loaded - ST); i < loaded; ++i) mbar_wait(&full[i % ST], (i / ST) & 1, a.status, kTimeoutTmaFull);

  // Row n's m, l and constant terms, over all keys of the warp.
  float row_m, row_l, add[NG];
#pragma unroll
  for (int g = 0; g < NG; ++g) add[g] = 0.f;
  if constexpr (ROWS == kBf16Heads) {  // keys were spread over 4 lanes
    row_m = st.m[0];
    row_l = st.l[0];
    row_l += __shfl_xor_sync(0xffffffff, row_l, 1);
    row_l += __shfl_xor_sync(0xffffffff, row_l, 2);
  } else {  // keys were spread over 8 groups of 4 lanes, query rows 2t, 2t + 1 over the 4
    auto over_keys = [](float x) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffff, x, o);
      return x;
    };
    auto to_row = [&](float even, float odd) {
      even = __shfl_sync(0xffffffff, even, n >> 1);
      odd = __shfl_sync(0xffffffff, odd, n >> 1);
      return (n & 1) ? odd : even;
    };
    constexpr int kLast = State<DP, ROWS>::kHeads - 1;
    row_m = to_row(st.m[0], st.m[kLast]);
    row_l = to_row(over_keys(st.l[0]), over_keys(st.l[kLast]));
    if constexpr (ROWS == kPackedHeads) {
#pragma unroll
      for (int g = 0; g < NG; ++g) add[g] = to_row(over_keys(st.low[g][0]), over_keys(st.low[g][1]));
    } else {
      add[0] = to_row(over_keys(st.low[0][0]), over_keys(st.low[0][1]));
    }
  }
  __syncthreads();  // every ring has been read
  float* join = reinterpret_cast<float*>(smem);  // [warp][row][DP + 2]: output, m, l
  if (row_head < heads) {
    float* row = join + (warp * kRows + row_head) * (DP + 2);
#pragma unroll
    for (int i = 0; i < State<DP, ROWS>::kTiles; ++i) {
      const int tile = ROWS == kPackedGroups ? row_group * 4 + i : i;
      const float c = C::kPacked ? add[ROWS == kPackedGroups ? 0 : i >> 2] : 0.f;
      row[channel_of<DP, ROWS>(tile, 2 * t)] = st.o[i][0] + st.o[i][2] + c;
      row[channel_of<DP, ROWS>(tile, 2 * t + 1)] = st.o[i][1] + st.o[i][3] + c;
    }
    if (t == 0 && (ROWS != kPackedGroups || row_group == 0)) {
      row[DP] = row_m;
      row[DP + 1] = row_l;
    }
  }
  __syncthreads();
  const int64_t unit = bh * a.chunks + chunk;
  float* part = a.partial + (unit * a.splits + split) * (kRows * (DP + 2));
  for (int i = threadIdx.x; i < heads * DP; i += kThreads) {
    const int r = i / DP, d = i % DP;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, join[(w * kRows + r) * (DP + 2) + DP]);
    const float m_use = m == -INFINITY ? 0.f : m;
    float o = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float* row = join + (w * kRows + r) * (DP + 2);
      const float c = exp2f(row[DP] - m_use);
      o += c * row[d];
      l += c * row[DP + 1];
    }
    if (active == 1) {
      if (d < a.D) a.out[(static_cast<int64_t>(b) * a.Hk * a.G + h0 + r) * a.D + d] = __float2bfloat16(o / l);
    } else {
      part[r * (DP + 2) + d] = o;
      if (d == 0) {
        part[r * (DP + 2) + DP] = m;
        part[r * (DP + 2) + DP + 1] = l;
      }
    }
  }
  if (active == 1) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    const int before = atomicAdd(&a.arrived[unit], 1);
    *last_flag = before == active - 1;
    if (before == active - 1) a.arrived[unit] = 0;  // ready for the next launch
  }
  __syncthreads();
  if (!*last_flag) return;
  __threadfence();
  const float* all = a.partial + unit * a.splits * (kRows * (DP + 2));
  constexpr int kStep = kRows * (DP + 2);
  if (active <= 8) {  // few splits: at once (6 splits of one sequence: 7.0 us against 7.9)
    for (int i = threadIdx.x; i < heads * DP; i += kThreads) {
      const int r = i / DP, d = i % DP;
      const float* row = all + r * (DP + 2);
      float m = -INFINITY, o = 0.f, l = 0.f;
      for (int s = 0; s < active; ++s) m = fmaxf(m, __ldcg(row + s * kStep + DP));
#pragma unroll 4
      for (int s = 0; s < active; ++s) {
        const float c = exp2f(__ldcg(row + s * kStep + DP) - m);
        o += c * __ldcg(row + s * kStep + d);
        l += c * __ldcg(row + s * kStep + DP + 1);
      }
      if (d < a.D) a.out[(static_cast<int64_t>(b) * a.Hk * a.G + h0 + r) * a.D + d] = __float2bfloat16(o / l);
    }
    return;
  }
  // many: the splits' weights first (a warp per query row), then the outputs, with
  // the loads of several splits in flight (13 splits: 48.9 us against 53.9)
  float* weight = join;                     // [row][split]
  float* inverse = join + kRows * active;   // [row]
  for (int r = warp; r < heads; r += kWarps) {
    const float* row = all + r * (DP + 2) + DP;
    float m = -INFINITY, l = 0.f;
    for (int s = lane; s < active; s += 32) m = fmaxf(m, __ldcg(row + static_cast<int64_t>(s) * kStep));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffff, m, o));
    for (int s = lane; s < active; s += 32) {
      const float c = exp2f(__ldcg(row + static_cast<int64_t>(s) * kStep) - m);
      weight[r * active + s] = c;
      l += c * __ldcg(row + static_cast<int64_t>(s) * kStep + 1);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffff, l, o);
    if (lane == 0) inverse[r] = 1.f / l;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * DP; i += kThreads) {
    const int r = i / DP, d = i % DP;
    const float* row = all + r * (DP + 2) + d;
    float o = 0.f;
#pragma unroll 8
    for (int s = 0; s < active; ++s) o += weight[r * active + s] * __ldcg(row + static_cast<int64_t>(s) * kStep);
    if (d < a.D)
      a.out[(static_cast<int64_t>(b) * a.Hk * a.G + h0 + r) * a.D + d] = __float2bfloat16(o * inverse[r]);
  }
}

// -------------------------------------------------------------------- host
// Operands the kernels can address as they are: unit inner stride, other strides
// and the start multiples of 16 bytes. Anything else is copied.
at::Tensor as_rows(const at::Tensor& x) {
  bool ok = x.stride(-1) == 1 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
  for (int i = 0; i + 1 < x.dim(); ++i) ok = ok && (x.size(i) == 1 || x.stride(i) % 8 == 0);
  return ok ? x : x.clone(at::MemoryFormat::Contiguous);
}

std::string sizes_text(at::IntArrayRef x) {
  std::string s = "[";
  for (size_t i = 0; i < x.size(); ++i) s += (i ? ", " : "") + std::to_string(x[i]);
  return s + "]";
}

// The rows of one layer's cache and what a step over them needs.
class KVCache {
 public:
  KVCache(int64_t batch, int64_t kv_heads, int64_t head_dim, int64_t window, int64_t sinks, int64_t bits, at::Tensor pos)
      : B_(batch), Hk_(kv_heads), D_(head_dim), bits_(static_cast<int>(bits)), pos_(std::move(pos)) {
    TORCH_CHECK_VALUE(D_ >= 8 && D_ <= 128 && D_ % 8 == 0 && (bits == 16 || (bits == 4 && D_ % 32 == 0)),
                      "kv cache: the CUDA cache takes head sizes that are multiples of 8 up to 128 (of 32 in 4 bits), got ",
                      std::to_string(D_));
    TORCH_CHECK_VALUE(window >= 1 && sinks >= 0 && window < (int64_t(1) << 31) && sinks < (int64_t(1) << 31),
                      "kv cache: window >= 1 and sinks >= 0 required");
    slots_ = window + sinks;
    DP_ = D_ <= 64 ? 64 : 128;
    const int64_t alloc = (slots_ + 63) / 64 * 64;  // whole tiles; rows past the last slot are never visible
    TORCH_CHECK_VALUE(B_ >= 1 && B_ <= 65535 && Hk_ >= 1 && Hk_ <= 32767 && alloc < (int64_t(1) << 31) / (B_ * Hk_),
                      "kv cache: batch, heads or slots out of range (2^31 rows at most)");
    check_positions(pos_, "pos");
    ring_ = {window, sinks, static_cast<int>(alloc)};
    c10::cuda::CUDAGuard guard(pos_.device());
    const auto options = pos_.options();
    for (int i = 0; i < 2; ++i) {
      rows_[i] = bits == 16 ? at::zeros({B_, Hk_, alloc, DP_}, options.dtype(at::kBFloat16))
                            : at::zeros({B_, Hk_, alloc, DP_ / 2}, options.dtype(at::kByte));
      if (bits == 4) params_[i] = at::zeros({B_, Hk_, alloc, DP_ / 32}, options.dtype(at::kInt));
      store_[i] = {static_cast<uint8_t*>(rows_[i].data_ptr()),
                   bits == 4 ? static_cast<uint32_t*>(params_[i].data_ptr()) : nullptr};
    }
    // Not with the first step: that may be one that a graph captures, and the counters
    // have to be 0 for steps outside of it too. Units that share the GPU among more than
    // one CTA each are at most half as many as fit on it.
    arrived_ = at::zeros({kMostCtas * num_sms() / 2}, options.dtype(at::kInt));
    dispatch([&](auto dp, auto bits_c) {
      if constexpr (bits_c() == 16) {
        const uint64_t n = static_cast<uint64_t>(B_) * Hk_ * alloc;
        for (int i = 0; i < 2; ++i)
          map_[i] = make_tmap_bf16(rows_[i].data_ptr(), dp(), n, dp(), 64, StepCfg<dp(), kBf16Heads>::KT);
      }
    });
  }

  // k, v [B, T, Hk, D]: the visible tokens of each prompt; pos[b] = its length.
  void fill(const at::Tensor& k_, const at::Tensor& v_, const c10::optional<at::Tensor>& lengths) {
    TORCH_CHECK_VALUE(k_.dim() == 4, "k must be [B, T, Hk, D], got ", sizes_text(k_.sizes()));
    const int64_t T = k_.size(1);
    TORCH_CHECK_VALUE(T < (int64_t(1) << 31), "kv cache: prompt too long");
    check_rows(k_, {B_, T, Hk_, D_}, "k");
    check_rows(v_, {B_, T, Hk_, D_}, "v");
    if (lengths) check_positions(*lengths, "lengths");
    c10::cuda::CUDAGuard guard(pos_.device());
    if (T == 0) {
      pos_.zero_();
      return;
    }
    const at::Tensor k = as_rows(k_), v = as_rows(v_);
    const int rows = static_cast<int>(std::min<int64_t>(T, slots_));
    const View kv = {static_cast<const __nv_bfloat16*>(k.data_ptr()), k.stride(0), k.stride(2), k.stride(1)};
    const View vv = {static_cast<const __nv_bfloat16*>(v.data_ptr()), v.stride(0), v.stride(2), v.stride(1)};
    dispatch([&](auto dp, auto bits) {
      const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(rows) * (dp() / 8) + 255) / 256),
                      static_cast<unsigned>(2 * Hk_), static_cast<unsigned>(B_));
      fill_kernel<dp(), bits()><<<grid, 256, 0, at::cuda::getCurrentCUDAStream()>>>(
          kv, vv, lengths ? positions(*lengths) : Positions{nullptr, 0}, positions(pos_), store_[0], store_[1], ring_,
          static_cast<int>(T), rows, static_cast<int>(Hk_), static_cast<int>(D_), status_ptr());
    });
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    debug_check("kv_cache fill");
  }

  // The held rows [B, Hk, slots, D] in slot order: bf16, or fp32 for 4 bits.
  std::pair<at::Tensor, at::Tensor> read() {
    c10::cuda::CUDAGuard guard(pos_.device());
    const auto options = pos_.options().dtype(bits_ == 16 ? at::kBFloat16 : at::kFloat);
    at::Tensor k = at::empty({B_, Hk_, slots_, D_}, options), v = at::empty({B_, Hk_, slots_, D_}, options);
    dispatch([&](auto dp, auto bits) {
      const dim3 grid(static_cast<unsigned>((slots_ * (dp() / 8) + 255) / 256), static_cast<unsigned>(2 * Hk_),
                      static_cast<unsigned>(B_));
      read_kernel<dp(), bits()><<<grid, 256, 0, at::cuda::getCurrentCUDAStream()>>>(
          store_[0], store_[1], positions(pos_), k.data_ptr(), v.data_ptr(), ring_, static_cast<int>(slots_),
          static_cast<int>(Hk_), static_cast<int>(D_));
    });
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    debug_check("kv_cache read");
    return {k, v};
  }

  // One token per sequence: q [B, H, D], k and v [B, Hk, D], pos [B] (-1: idle).
  // The attention [B, H, D] over the cache with the token in it and, on request,
  // what the stored rows stand for (fp32 [B, Hk, D]).
  std::vector<at::Tensor> step(const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& v_, const at::Tensor& pos,
                               bool return_stored) {
    TORCH_CHECK_VALUE(q_.dim() == 3 && q_.size(1) >= 1 && q_.size(1) % Hk_ == 0, "q must be [B, H, D] with H a multiple of ",
                      std::to_string(Hk_), ", got ", sizes_text(q_.sizes()));
    const int64_t H = q_.size(1), G = H / Hk_;
    const Rows rows = rows_for(G);
    const int64_t per = rows == kPackedGroups ? kRows / (DP_ / 32) : kRows, chunks = (G + per - 1) / per;
    check_rows(q_, {B_, H, D_}, "q");
    check_rows(k_, {B_, Hk_, D_}, "k");
    check_rows(v_, {B_, Hk_, D_}, "v");
    check_positions(pos, "pos");
    TORCH_CHECK_VALUE(Hk_ * chunks <= 65535, "kv cache: too many query heads");
    c10::cuda::CUDAGuard guard(pos_.device());
    const at::Tensor q = as_rows(q_), k = as_rows(k_), v = as_rows(v_);
    const Work& work = work_for(chunks, rows);
    at::Tensor out = at::empty({B_, H, D_}, q.options());
    std::vector<at::Tensor> result = {out};
    StepArgs a;
    a.q = static_cast<const __nv_bfloat16*>(q.data_ptr());
    a.q_b = q.stride(0), a.q_h = q.stride(1);
    a.k = {static_cast<const __nv_bfloat16*>(k.data_ptr()), k.stride(0), k.stride(1), 0};
    a.v = {static_cast<const __nv_bfloat16*>(v.data_ptr()), v.stride(0), v.stride(1), 0};
    a.pos = positions(pos);
    a.ks = store_[0], a.vs = store_[1];
    a.out = static_cast<__nv_bfloat16*>(out.data_ptr());
    a.stored_k = a.stored_v = nullptr;
    if (return_stored) {
      for (int i = 0; i < 2; ++i) result.push_back(at::empty({B_, Hk_, D_}, q.options().dtype(at::kFloat)));
      a.stored_k = result[1].data_ptr<float>();
      a.stored_v = result[2].data_ptr<float>();
    }
    a.partial = work.partial.data_ptr<float>();
    a.arrived = arrived_.data_ptr<int>();
    a.ring = ring_;
    a.slots = static_cast<int>(slots_), a.Hk = static_cast<int>(Hk_), a.G = static_cast<int>(G);
    a.D = static_cast<int>(D_), a.chunks = static_cast<int>(chunks), a.splits = work.splits;
    a.scale_log2 = static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(D_)));
    a.status = status_ptr();
    const dim3 grid(static_cast<unsigned>(work.splits), static_cast<unsigned>(Hk_ * chunks), static_cast<unsigned>(B_));
    dispatch_step(rows, [&](auto dp, auto rows_c) {
      using C = StepCfg<dp(), static_cast<int>(rows_c())>;
      auto kernel = step_kernel<dp(), static_cast<int>(rows_c())>;
      static bool configured[64] = {false};
      const int dev = pos_.device().index();
      if (!configured[dev])
        C10_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
      configured[dev] = true;
      kernel<<<grid, kThreads, C::kSmem, at::cuda::getCurrentCUDAStream()>>>(map_[0], map_[1], a);
    });
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    debug_check("kv_cache step");
    return result;
  }

  const at::Tensor& rows(int i) const { return rows_[i]; }
  const at::Tensor& params(int i) const { return params_[i]; }

 private:
  struct Work {  // joining the CTAs that share a cache
    int splits;
    at::Tensor partial;
  };

  template <typename F>
  void dispatch(F&& f) const {
    using std::integral_constant;
    if (DP_ == 64 && bits_ == 16) f(integral_constant<int, 64>(), integral_constant<int, 16>());
    if (DP_ == 64 && bits_ == 4) f(integral_constant<int, 64>(), integral_constant<int, 4>());
    if (DP_ == 128 && bits_ == 16) f(integral_constant<int, 128>(), integral_constant<int, 16>());
    if (DP_ == 128 && bits_ == 4) f(integral_constant<int, 128>(), integral_constant<int, 4>());
  }

  // 4 bits: rows of (head, group) as long as a key head's query heads fit in one CTA.
  Rows rows_for(int64_t G) const {
    if (bits_ == 16) return kBf16Heads;
    return G <= kRows / (DP_ / 32) ? kPackedGroups : kPackedHeads;
  }

  template <typename F>
  void dispatch_step(Rows rows, F&& f) const {
    using std::integral_constant;
    auto with = [&](auto dp) {
      if (rows == kBf16Heads) f(dp, integral_constant<int, kBf16Heads>());
      if (rows == kPackedHeads) f(dp, integral_constant<int, kPackedHeads>());
      if (rows == kPackedGroups) f(dp, integral_constant<int, kPackedGroups>());
    };
    DP_ == 64 ? with(integral_constant<int, 64>()) : with(integral_constant<int, 128>());
  }

  // How many CTAs share the slots of one (sequence, key head): as many as fit on the
  // GPU at once (a few more would run after all others: 57 us against 54 for 16
  // sequences of 2 key heads), each with at least one tile per warp.
  // It depends on the number of query heads alone, so by no earlier call's.
  const Work& work_for(int64_t chunks, Rows rows) {
    const auto key = std::make_pair(chunks, rows);
    auto it = work_.find(key);
    if (it != work_.end()) return it->second;
    const int64_t units = B_ * Hk_ * chunks;
    int64_t splits = 1;
    dispatch_step(rows, [&](auto dp, auto rows_c) {
      using C = StepCfg<dp(), static_cast<int>(rows_c())>;
      const int64_t most = (slots_ + kWarps * C::KT - 1) / (kWarps * C::KT);
      splits = std::min({most, std::max<int64_t>(1, C::kCtas * num_sms() / units), int64_t(C::kMaxSplits)});
    });
    Work w = {static_cast<int>(splits), at::empty({units * splits * kRows * (DP_ + 2)}, pos_.options().dtype(at::kFloat))};
    return work_.emplace(key, std::move(w)).first->second;
  }

  void check_rows(const at::Tensor& x, std::initializer_list<int64_t> sizes, const char* name) const {
    TORCH_CHECK_VALUE(x.sizes() == at::IntArrayRef(sizes) && x.scalar_type() == at::kBFloat16 && x.device() == pos_.device(),
                      name, " must be a bf16 tensor ", sizes_text(at::IntArrayRef(sizes)), " on the cache's device, got ",
                      sizes_text(x.sizes()), " ", c10::toString(x.scalar_type()));
  }

  void check_positions(const at::Tensor& x, const char* name) const {
    TORCH_CHECK_VALUE(x.is_cuda() && (!pos_.defined() || x.device() == pos_.device()) && x.scalar_type() == at::kLong &&
                          x.dim() == 1 && x.size(0) == B_,
                      name, " must be an int64 tensor [", std::to_string(B_), "] on the cache's device");
  }

  static Positions positions(const at::Tensor& x) { return {x.data_ptr<int64_t>(), x.stride(0)}; }

  int64_t B_, Hk_, D_, slots_, DP_;
  int bits_;
  at::Tensor pos_, rows_[2], params_[2];
  at::Tensor arrived_;  // per unit of a step, 0 between launches
  Store store_[2];
  Ring ring_;
  CUtensorMap map_[2] = {};
  std::map<std::pair<int64_t, Rows>, Work> work_;  // by chunks and row form
};

}  // namespace kv_cache
}  // namespace dst

using namespace dst;

void register_kv_cache(pybind11::module& m) {
  namespace py = pybind11;
  using kv_cache::KVCache;
  py::class_<KVCache>(m, "KVCache", "rolling key/value cache of one layer (bf16 or 4 bits)")
      .def(py::init<int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, at::Tensor>(), py::arg("batch"),
           py::arg("kv_heads"), py::arg("head_dim"), py::arg("window"), py::arg("sinks"), py::arg("bits"), py::arg("pos"))
      .def("fill", &KVCache::fill, py::arg("k"), py::arg("v"), py::arg("lengths"))
      .def("read", &KVCache::read)
      .def("step", &KVCache::step, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("pos"), py::arg("return_stored"))
      .def("rows", [](const KVCache& c) { return py::make_tuple(c.rows(0), c.rows(1)); })
      .def("params", [](const KVCache& c) { return py::make_tuple(c.params(0), c.params(1)); });
}
