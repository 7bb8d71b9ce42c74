// Attention over cached sequences for passes of more than one token: whole
// prompts packed back to back (causal, each over its own keys) and trees of
// drafted tokens over a cache. The reference runs both through transformers'
// attention modules, one sequence at a time (its engine hooks them,
// afterimage/runtime/streaming_engine.py:1871-1915; the speculation loop
// re-runs the whole sequence, :2488-2575).
//
// Row i of a sequence with m queries and L keys, head h, kv head h / (nh/nkv):
//   out = sum over seen j of exp(z_j - z_max) v_j / sum over seen j of exp(z_j - z_max),  z_j = scale q.k_j
// A prompt's row i sees the keys j <= L - m + i. A tree's row i sees every
// cache slot before pos, and slot pos + j where mask[i, j]. A row that sees
// nothing is zero. What a row does not see cannot reach it: masked scores are
// replaced, not added to; the plain kernel never multiplies a masked v_j, and
// the tensor-core kernel, whose masked weights are zeros that are multiplied,
// first takes out of V what is not finite (warps 10-11).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <mutex>
#include <type_traits>

#include "aib_internal.h"

namespace aibseq {

__device__ __forceinline__ float b2f(uint16_t v) { return __uint_as_float(static_cast<uint32_t>(v) << 16); }
__device__ __forceinline__ uint16_t f2b(float f) { return __bfloat16_as_ushort(__float2bfloat16_rn(f)); }

__device__ __forceinline__ int64_t clamp64(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : (v > hi ? hi : v); }

// One sequence: where its queries and keys are and what its rows see. Every
// value is cut to the extents that the host checked, so that lengths on the
// device cannot lead outside a tensor.
// (32 bits: the host limits tokens, sequences and key rows; only offsets in memory need more.)
struct Seq {
  int q0, m;    // first query row (within the q batch of a tree: 0) and number of queries
  int qb;       // q batch
  int kb, k0;   // k batch and first key row
  int L;        // keys
  int off;      // prompt: row i sees keys < off + i + 1; tree: slot of the drafted column 0
};

__device__ __forceinline__ int cut(int64_t v, int64_t lo, int64_t hi) { return static_cast<int>(clamp64(v, lo, hi)); }

__device__ __forceinline__ Seq sequence(const aib_attn_desc &p, int b) {
  Seq s;
  if (p.mask) {
    s.q0 = 0;
    s.m = static_cast<int>(p.tokens);
    s.qb = s.kb = b;
    s.k0 = 0;
    // a position outside [-columns, rows] means nothing more than its end of that range
    s.off = cut(p.pos[b], -p.mask_cols, p.key_rows);
    s.L = cut(s.off + p.mask_cols, 0, p.key_rows);
    return s;
  }
  s.q0 = cut(p.cu_q[b], 0, p.tokens);
  s.m = cut(p.cu_q[b + 1], s.q0, p.tokens) - s.q0;
  s.qb = 0;
  if (p.len_k) {
    s.kb = b;
    s.k0 = 0;
    s.L = cut(p.len_k[b], 0, p.key_rows);
  } else {
    s.kb = 0;
    s.k0 = cut(p.cu_k[b], 0, p.key_rows);
    s.L = cut(p.cu_k[b + 1], s.k0, p.key_rows) - s.k0;
  }
  s.off = s.L - s.m;
  return s;
}

// does row i of sequence s see key j (0 <= j < s.L)?
__device__ __forceinline__ bool sees(const aib_attn_desc &p, const Seq &s, int64_t i, int64_t j) {
  if (!p.mask) return j <= s.off + i;
  if (j < s.off) return true;
  const int64_t c = j - s.off;
  return c < p.mask_cols &&
         p.mask[static_cast<int64_t>(s.qb) * p.mask_batch_stride + i * p.mask_row_stride + c * p.mask_col_stride] != 0;
}

// ---------------------------------------------------------------------------
// The plain kernel: one warp for one row of one head, 32 keys at a time (a
// lane takes one key's score, then the warp adds the seen keys' values, a
// lane per value column). It takes every head size up to 256 and every
// stride; scores, sums and the running output are fp32, the result is
// rounded once. It is there to be right, not fast (a warp reads every key for
// one row): 1024 tokens of 16 heads of 256 on 8 take 8.3 ms, 26 nodes over
// 4000 slots 3.2 ms, where the same heads of 128 take 16 us each on the tensor
// cores; a second O of 256 columns beside the scores would need another layout
// of tensor memory, and no model shape of this package has such heads.
// ---------------------------------------------------------------------------
constexpr int kPlainMaxHd = 256;
constexpr int kPlainWarps = 4;

__global__ void __launch_bounds__(kPlainWarps * 32) attn_plain_kernel(const aib_attn_desc p) {
  __shared__ float qs[kPlainWarps][kPlainMaxHd];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t rows = (p.mask ? p.batch : 1) * p.tokens;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * kPlainWarps + w;
  if (r >= rows * p.nh) return;
  const int64_t tok = r / p.nh;
  const int h = static_cast<int>(r - tok * p.nh);
  const int kvh = h / (p.nh / p.nkv);
  Seq s;
  int64_t i;
  if (p.mask) {
    s = sequence(p, static_cast<int>(tok / p.tokens));
    i = tok % p.tokens;
  } else {
    int b = 0;
    while (b < p.batch && p.cu_q[b + 1] <= tok) ++b;
    if (b == p.batch) return;  // behind the last sequence: left as it is
    s = sequence(p, b);
    i = tok - s.q0;
    if (i < 0 || i >= s.m) return;
  }
  const uint16_t *q = static_cast<const uint16_t *>(p.q) + s.qb * p.q_batch_stride + (s.q0 + i) * p.q_token_stride +
                      h * p.q_head_stride;
  uint16_t *out = static_cast<uint16_t *>(p.out) + s.qb * p.out_batch_stride + (s.q0 + i) * p.out_token_stride +
                  h * p.out_head_stride;
  const uint16_t *k = static_cast<const uint16_t *>(p.k) + s.kb * p.k_batch_stride + s.k0 * p.k_token_stride +
                      kvh * p.k_head_stride;
  const uint16_t *v = static_cast<const uint16_t *>(p.v) + s.kb * p.v_batch_stride + s.k0 * p.v_token_stride +
                      kvh * p.v_head_stride;
  for (int d = lane; d < p.hd; d += 32) qs[w][d] = b2f(q[d]) * p.scale;
  __syncwarp();
  float acc[kPlainMaxHd / 32] = {};
  float m = -INFINITY, l = 0.f;
  const int64_t end = p.mask ? s.L : clamp64(s.off + i + 1, 0, s.L);
  for (int64_t j0 = 0; j0 < end; j0 += 32) {
    const int64_t j = j0 + lane;
    const bool seen = j < end && sees(p, s, i, j);
    float z = -INFINITY;
    if (seen) {
      z = 0.f;
      for (int d = 0; d < p.hd; ++d) z += qs[w][d] * b2f(k[j * p.k_token_stride + d]);
    }
    float top = z;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float mn = fmaxf(m, top);
    const float ref = mn == -INFINITY ? 0.f : mn;
    const float pr = seen ? expf(z - ref) : 0.f;
    const float a = expf(m - ref);
    float sum = pr;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    l = l * a + sum;
    m = mn;
#pragma unroll
    for (int c = 0; c < kPlainMaxHd / 32; ++c) acc[c] *= a;
    unsigned left = __ballot_sync(0xffffffffu, seen);
    while (left) {
      const int t = __ffs(left) - 1;
      left &= left - 1;
      const float pt = __shfl_sync(0xffffffffu, pr, t);
      const uint16_t *vr = v + (j0 + t) * p.v_token_stride;
#pragma unroll
      for (int c = 0; c < kPlainMaxHd / 32; ++c) {
        const int d = lane + 32 * c;
        if (d < p.hd) acc[c] += pt * b2f(vr[d]);
      }
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int c = 0; c < kPlainMaxHd / 32; ++c) {
    const int d = lane + 32 * c;
    if (d < p.hd) out[d] = f2b(l == 0.f ? 0.f : acc[c] * inv);
  }
}

// ---------------------------------------------------------------------------
// The tensor-core kernel (head sizes that are multiples of 8, up to 128).
//
// A tile is 128 rows: the G = nh / nkv heads that share a kv head, for
// 128 / G tokens (row r = token r / G, head r mod G). Sharing heads fills the
// rows of the matrix instructions for short prompts and drafted trees, and
// makes one pass over a kv head's keys serve all its queries. A CTA takes two
// tiles of consecutive tokens over the same keys ("pair"), or one tile whose
// key tiles two streams take in turn and join at the end ("solo"), and,
// where that would leave SMs empty, a share of the key axis; the shares join
// through a cluster's shared memory or in a second kernel.
//
// Per CTA, 128 keys at a time:
//   S = Q K^T         tcgen05.mma, both operands in shared memory -> tensor memory
//   P = exp2(S - m)   one thread per row: running maximum and sum, P as BF16
//                     over S's columns in tensor memory, or beside them
//   O = O + P V       tcgen05.mma, P from tensor memory, V as it lies in
//                     shared memory (keys x head size)
// The running maximum is only followed when it would leave P above 2^8: any
// reference m gives the same quotient, and rescaling O costs a pass over it.
//
// Warps 0-3 and 4-7: the softmax of stream 0 and 1; warp 8: TMA loads into a
// ring of K and V tiles; warp 9: the matrix instructions; warps 10-11: where
// a key tile is not seen in full, they replace what is not finite in V by
// zero, since a masked weight of zero times NaN is NaN; what of it is seen by
// some row is added back, row by row, at the end.
// Every wait is bounded; one that gives up sets AIB_STATUS_WAIT_TIMEOUT and
// the CTA unwinds.
//
// What bounds it. For a pair, 128 keys are 32 matrix instructions of 64 clocks
// each (2048 clocks) and 256 exponentials a scheduler at 8 clocks each (2048
// clocks); the two would have to overlap in full, and tensor memory has no room
// for a second S beside two O of 128 columns, so that a stream's next scores
// wait for its product with V (64 columns leave the room). Measured: about
// 3600 clocks, tensor pipe and exponential unit both busy half of the time. One
// prompt of 16384 tokens, 40 heads of 128 on 8 kv heads, causal: 2.15 ms in a
// burst (1280 TFLOP/s, 0.77 of the measured cuBLAS burst), 2.65 ms in a loop of
// seconds (1040, 0.75 of cuBLAS in such a loop), where the power limit holds
// the clock at 1.67 GHz.
// What was tried and did not pay there: exponentials by a polynomial on the
// multiply-add pipe for 1/8 or 2/8 of the weights (2.14 -> 2.16 and 2.19 ms); S
// in halves of 64 keys, the two in turn (2.41 against 2.31 ms then: a product
// with 64 columns reads Q as often as one with 128); a sixth ring tile, and
// prefetches into L2, where there is one Q tile (no change).
// A drafted tree of 64 nodes over 32,000 slots (three tiles a kv head, six
// shares): 53 us, of which the join is 5; the keys and values are read from
// HBM once (133 MB by the counters, 2.5 TB/s) and from L2 three times.
// Short calls are a chain of waits: set-up 1 us, first tiles 1.5, a tile's
// scores, softmax and product 2, the output 1, joining the shares 1 to 4. One
// token over 1000 slots: 9.4 us; a chain of five over 4099: 13.1 us.
// ---------------------------------------------------------------------------
constexpr int kTile = 128;
constexpr int kThreads = 384;
constexpr int kMaxSlots = 8;
constexpr unsigned kWaitLimit = AIB_WAIT_LIMIT_POLLS;
constexpr float kFollow = 8.f;  // log2 of how far above 1 a weight may come before the maximum is followed

template <int HDP, bool kOwnP>
struct Cfg {
  static constexpr int kHalves = HDP / 64;             // 128-byte-swizzled column blocks of a tile
  static constexpr int kSlotBytes = kHalves * 16384;   // one K, V or Q tile
  static constexpr int kSlots = HDP == 128 ? 5 : 8;
  static constexpr int kSmem = (2 + kSlots) * kSlotBytes + 1024;
  // With O of 64 columns P can have columns of its own (kOwnP): a stream's next scores are made as soon as the last
  // ones are in registers, and the softmax does not wait for them, for one more signal and wait a tile. With O of 128
  // P lies over S, and the scores wait for its product. Two tiles on the same keys gain by it, one tile does not: 8192
  // tokens, 32 heads of 64 on 8: 401 -> 373 us, seven prompts of 1 to 3000: 121 -> 115, 32 trees of 49 nodes: 53 -> 51;
  // 64 trees of 8: 79 -> 81, 317 queries over 8000 and 4100 keys: 55.5 -> 59.4. So items of two tiles have it.
  static_assert(!kOwnP || HDP == 64);
  static constexpr int kColO = 256, kColP = 384;  // tensor-memory columns; S of stream s at 128 s
  static constexpr int kStepO = kOwnP ? 64 : 128, kStepP = kOwnP ? 64 : 128;
};

struct TcParams {
  aib_attn_desc d;
  int group, tt;       // heads per kv head, tokens per tile
  int group_rcp;       // r / group is r * group_rcp >> 16 for r < 128
  int tpi;             // tiles an item may hold: 2 or 1
  int splits;          // shares of the key axis
  int cluster;         // the shares are one cluster's CTAs and join through its shared memory, without a second kernel
  float scale_log2;
  int vec_out;         // output rows allow 16-byte stores
  float *workspace;    // shares: O, maximum and sum of their rows
  int32_t *status;
};

// What one CTA works on.
struct Item {
  Seq s;
  int shares;          // shares of the key axis that hold any of the item's key tiles
  int t0;              // first token of tile 0 within the sequence
  int cnt0, cnt1;      // tokens in each tile
  int end0, end1;      // keys that some row of the tile sees lie before this
  int low0, low1;      // every row of the tile sees the keys before this
  int ta, tb;          // key tiles of this share
  bool live;
};

// Items of sequence i.
__device__ __forceinline__ int items_of(const TcParams &p, int i) {
  const int unit = p.tt * p.tpi;
  const int q0 = cut(p.d.cu_q[i], 0, p.d.tokens);
  return (cut(p.d.cu_q[i + 1], q0, p.d.tokens) - q0 + unit - 1) / unit;
}

// Item number -> sequence and first tile. Prompts: items are numbered from
// the last tiles of the longest prompts down (they see the most keys; the
// hardware hands CTAs out in order, so the longest run first). With P_b items
// in sequence b, the items at level l (the l-th of their sequence) or above
// are F(l) = sum_b max(0, P_b - l); a binary search finds the item's level.
// Collective over the warp.
__device__ __forceinline__ bool find_among_prompts(const TcParams &p, int item, int &b, int &level) {
  const int lane = threadIdx.x & 31, batch = static_cast<int>(p.d.batch);
  const int first = lane < batch ? items_of(p, lane) : 0;  // up to 32 sequences need no second read
  int lo = 0, hi = __reduce_max_sync(0xffffffffu, first);
  int all = __reduce_add_sync(0xffffffffu, first);
#pragma unroll 1
  for (int i = lane + 32; i - lane < batch; i += 32) {
    const int n = i < batch ? items_of(p, i) : 0;
    hi = max(hi, __reduce_max_sync(0xffffffffu, n));
    all += __reduce_add_sync(0xffffffffu, n);
  }
  if (all <= item) return false;
  int above = 0;  // F(hi); F(lo) > item >= F(hi)
#pragma unroll 1
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    int f = max(0, first - mid);
#pragma unroll 1
    for (int i = lane + 32; i < batch; i += 32) f += max(0, items_of(p, i) - mid);
    f = __reduce_add_sync(0xffffffffu, f);
    if (f > item) lo = mid; else hi = mid, above = f;
  }
  int rank = item - above;  // among the sequences that reach level lo (hi = lo + 1)
  level = lo;
#pragma unroll 1
  for (int i0 = 0; i0 < batch; i0 += 32) {
    const int n = i0 == 0 ? first : (i0 + lane < batch ? items_of(p, i0 + lane) : 0);
    unsigned has = __ballot_sync(0xffffffffu, n > lo);
    if (rank < __popc(has)) {
#pragma unroll 1
      for (; rank > 0; --rank) has &= has - 1;
      b = i0 + __ffs(has) - 1;
      return true;
    }
    rank -= __popc(has);
  }
  return false;
}
__device__ __forceinline__ bool find_item(const TcParams &p, int item, int &b, int &level) {
  if (p.d.mask) {
    const int unit = p.tt * p.tpi, tokens = static_cast<int>(p.d.tokens);
    const int per = tokens <= unit ? 1 : (tokens + unit - 1) / unit;
    b = per == 1 ? item : item / per;
    level = item - b * per;
    return b < static_cast<int>(p.d.batch);
  }
  if (p.d.batch == 1) {
    b = 0;
    level = items_of(p, 0) - 1 - item;
    return level >= 0;
  }
  return find_among_prompts(p, item, b, level);
}

__device__ __forceinline__ void make_tile(const TcParams &p, const Seq &s, int t, bool used, int &cnt, int &end,
                                          int &low) {
  cnt = used ? max(0, min(p.tt, s.m - t)) : 0;
  end = p.d.mask ? s.L : max(0, min(s.off + t + cnt, s.L));
  low = max(0, min(p.d.mask ? s.off : s.off + t + 1, s.L));
  if (cnt == 0) end = 0;
}

__device__ __forceinline__ Item make_item(const TcParams &p, int item, int split) {
  Item w;
  int b = 0, level = 0;
  w.live = find_item(p, item, b, level);
  if (!w.live) return w;
  w.s = sequence(p.d, b);
  w.t0 = level * p.tt * p.tpi;
  make_tile(p, w.s, w.t0, true, w.cnt0, w.end0, w.low0);
  make_tile(p, w.s, w.t0 + p.tt, p.tpi > 1, w.cnt1, w.end1, w.low1);
  const int tiles = (max(w.end0, w.end1) + kTile - 1) / kTile;
  const int per = p.splits == 1 ? tiles : (tiles + p.splits - 1) / p.splits;
  w.shares = per ? (tiles + per - 1) / per : 0;
  w.ta = min(tiles, split * per);
  w.tb = min(tiles, w.ta + per);
  return w;
}

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void mbar_init(uint32_t bar, unsigned count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, unsigned parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// Waits, as a whole warp, for the phase of `parity`; false when the bound is
// reached or another role gave up. One answer for all lanes: what follows
// stays uniform, which the warp-wide instructions need and the issue of the
// matrix and copy instructions (their operands are uniform registers) is
// faster for.
__device__ __forceinline__ bool warp_wait(uint32_t bar, unsigned parity, volatile int *gave_up) {
#pragma unroll 1
  for (unsigned n = 0; n < kWaitLimit; ++n) {
    if (__all_sync(0xffffffffu, mbar_try(bar, parity))) return true;
    if (n > 256) {
      if (__any_sync(0xffffffffu, *gave_up)) break;
      __nanosleep(32);
    }
  }
  *gave_up = 1;
  return false;
}
// one lane of a converged warp
__device__ __forceinline__ bool elect() {
  uint32_t yes;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(yes));
  return yes != 0;
}
// a value that is the same in all lanes, known to be so
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, int w,
                                            uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}

// shared-memory matrix descriptors, 128-byte swizzle. K-major (Q, K): 128-byte
// rows, 8-row groups 1024 bytes apart. MN-major (V, rows are keys): 64 columns
// a block, blocks of 64 columns 16 KiB apart, 8-key groups 1024 bytes apart.
// Only the low word differs between tiles: it holds address / 16, so that a
// step inside a tile is one addition. (One thread issues every matrix
// instruction of the CTA, between softmax warps that keep its scheduler busy:
// with the descriptors built for each instruction it was what the 16384-token
// prompt waited for.)
constexpr uint32_t kDescHigh = (1024 >> 4) | (1u << 14) | (2u << 29);
// (in a cluster the high bits of a shared address say whose memory it is)
__device__ __forceinline__ uint32_t desc_kmajor(uint32_t addr) { return (addr >> 4 & 0x3fff) | 1u << 16; }
__device__ __forceinline__ uint32_t desc_mnmajor(uint32_t addr) { return (addr >> 4 & 0x3fff) | (16384u >> 4) << 16; }

// BF16 x BF16 -> F32, M = 128
__host__ __device__ constexpr uint32_t idesc_bf16(int n, int b_mn_major) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(b_mn_major) << 16) |
         (static_cast<uint32_t>(n >> 3) << 17) | ((kTile >> 4) << 24);
}

// descriptors by their low words; `acc` 0: the first of a sum
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 da, db;\n setp.ne.b32 p, %4, 0;\n mov.b64 da, {%1, %5};\n mov.b64 db, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 db;\n setp.ne.b32 p, %4, 0;\n mov.b64 db, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

#define AIB_R8(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3]), "=r"(v[i + 4]), "=r"(v[i + 5]), "=r"(v[i + 6]), "=r"(v[i + 7])
#define AIB_I8(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]), "r"(v[i + 4]), "r"(v[i + 5]), "r"(v[i + 6]), "r"(v[i + 7])

// 32 tensor-memory columns of this thread's lane
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t *v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : AIB_R8(v, 0), AIB_R8(v, 8), AIB_R8(v, 16), AIB_R8(v, 24)
      : "r"(addr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t *v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : AIB_R8(v, 0), AIB_R8(v, 8)
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t *v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      AIB_I8(v, 0), AIB_I8(v, 8), AIB_I8(v, 16), AIB_I8(v, 24)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t *v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          addr),
      AIB_I8(v, 0), AIB_I8(v, 8)
      : "memory");
}
__device__ __forceinline__ float tmem_ld1(uint32_t addr) {
  float v;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n tcgen05.wait::ld.sync.aligned;" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void tmem_st1(uint32_t addr, float v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two floats as packed BF16, `lo` in the low half
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// two floats side by side, for the packed fp32 instructions
__device__ __forceinline__ uint64_t two(uint32_t lo, uint32_t hi) {
  return static_cast<uint64_t>(hi) << 32 | lo;
}
__device__ __forceinline__ uint64_t two(float v) { return two(__float_as_uint(v), __float_as_uint(v)); }
__device__ __forceinline__ float low_of(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float high_of(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_nan3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// shared memory of another CTA of the cluster: the address there of what is at `addr` here
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ bool not_finite_bf16(uint32_t h) { return (h & 0x7f80u) == 0x7f80u; }

__device__ __forceinline__ void lds128(uint32_t addr, uint32_t (&x)[4]) {
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void sts128(uint32_t addr, uint4 x) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
}

// What the warps of a CTA share of its item, in shared memory; read where it is needed, so that it takes no registers
// beside a tile of scores.
enum Field { kLive, kQ0, kQb, kKb, kK0, kKeys, kOff, kT0, kCnt0, kCnt1, kEnd, kLow0, kLow1, kTa, kPairs, kTiles, kTiles0, kSeenInFull, kShares, kFields };
__device__ __forceinline__ int lds32(uint32_t addr) {
  int v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// bits of the seen keys among the four 32-key words of key tile t, for this
// thread's row (token tok of the tile; first token of the tile is ti within
// the sequence). Collective over the warp for trees.
__device__ __forceinline__ void seen_words(const TcParams &p, const Seq &s, int t0, int tok, int warp_tok0,
                                           int warp_tok1, int t, uint32_t (&bits)[4]) {
  const int key0 = t * kTile;
  if (!p.d.mask) {
    const int n = max(0, min(s.off + t0 + tok + 1, s.L)) - key0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int k = n - 32 * c;
      bits[c] = k >= 32 ? 0xffffffffu : (k <= 0 ? 0u : (1u << k) - 1u);
    }
    return;
  }
  const int lane = threadIdx.x & 31;
  const uint8_t *m = p.d.mask + static_cast<int64_t>(s.qb) * p.d.mask_batch_stride;
#pragma unroll
  for (int c = 0; c < 4; ++c) bits[c] = 0;
#pragma unroll 1
  for (int a = warp_tok0; a <= warp_tok1; ++a) {
    const uint8_t *row = m + static_cast<int64_t>(t0 + a) * p.d.mask_row_stride;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int key = key0 + 32 * c + lane;
      const int64_t col = static_cast<int64_t>(key) - s.off;
      bool seen = key < s.L && col < p.d.mask_cols;
      if (seen && col >= 0) seen = row[col * p.d.mask_col_stride] != 0;
      const uint32_t word = __ballot_sync(0xffffffffu, seen);
      if (a == tok) bits[c] = word;
    }
  }
}

// What V held that is not finite (warps 10-11 took it out of the key tiles
// first .. last - 1 of the stream) and this thread's row sees is added to its
// row of O: whatever its weight, the sum is not finite there. Rare and slow.
// Collective over the warp.
template <int HDP>
__device__ __forceinline__ void add_not_finite(const TcParams &p, const Seq &s, int t0, int kvh, int tok, int warp_tok0,
                                            int warp_tok1, int first, int last, int step, uint32_t to) {
  const uint16_t *v = static_cast<const uint16_t *>(p.d.v) + s.kb * p.d.v_batch_stride + s.k0 * p.d.v_token_stride +
                      kvh * p.d.v_head_stride;
#pragma unroll 1
  for (int c = 0; c < p.d.hd; ++c) {
    float o = tmem_ld1(to + c);
#pragma unroll 1
    for (int t = first; t < last; t += step) {
      uint32_t bits[4];
      seen_words(p, s, t0, tok, warp_tok0, warp_tok1, t, bits);
#pragma unroll 1
      for (int i = 0; i < kTile; ++i) {
        const int key = t * kTile + i;
        const uint32_t word = i < 64 ? (i < 32 ? bits[0] : bits[1]) : (i < 96 ? bits[2] : bits[3]);
        if (key >= s.L || !((word >> (i & 31)) & 1u)) continue;
        const uint16_t x = v[key * p.d.v_token_stride + c];
        if (not_finite_bf16(x)) o += b2f(x);
      }
    }
    __syncwarp();  // the lanes went their own ways, and tensor memory is written by a converged warp
    tmem_st1(to + c, o);
  }
  tmem_wait_st();
}

// Joins a cluster's shares: out = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s, each CTA for HDP / shares columns,
// two threads to a row. `part`: where each CTA has its share's O (four columns of a row side by side), maxima and
// sums.
template <int HDP, typename F>
__device__ __forceinline__ void join_cluster(const TcParams &p, uint32_t part, int kvh, int rank, const F &field) {
  const int row = threadIdx.x & (kTile - 1);
  if (row >= field(kCnt0) * p.group) return;
  const int shares = min(p.splits, field(kShares));
  // columns of a thread: 4 to 32; four columns of a CTA (16 shares, heads of 64) are the first half's alone
  const int columns = HDP / p.splits, width = max(4, columns / 2);
  const int c0 = rank * columns + static_cast<int>(threadIdx.x >> 7) * width, c1 = min(c0 + width, (rank + 1) * columns);
  float m = -INFINITY;
#pragma unroll 4
  for (int s = 0; s < shares; ++s) m = fmaxf(m, ld_cluster(in_cta(part, s) + (HDP * kTile + row) * 4));
  const float ref = m == -INFINITY ? 0.f : m;
  const int tok = (row * p.group_rcp) >> 16;
  uint16_t *out = static_cast<uint16_t *>(p.d.out) + field(kQb) * p.d.out_batch_stride +
                  static_cast<int64_t>(field(kQ0) + field(kT0) + tok) * p.d.out_token_stride +
                  static_cast<int64_t>(kvh * p.group + row - tok * p.group) * p.d.out_head_stride;
#pragma unroll 1
  for (int c = c0; c < c1 && c < p.d.hd; c += 4) {
    float l = 0.f, o[4] = {};
#pragma unroll 4
    for (int s = 0; s < shares; ++s) {
      const uint32_t at = in_cta(part, s);
      const float a = ex2(ld_cluster(at + (HDP * kTile + row) * 4) - ref);
      const float4 x = ld_cluster4(at + (c / 4 * kTile + row) * 16);
      l += a * ld_cluster(at + ((HDP + 1) * kTile + row) * 4);
      o[0] += a * x.x;
      o[1] += a * x.y;
      o[2] += a * x.z;
      o[3] += a * x.w;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const uint32_t lo = pack_bf16(o[0] * inv, o[1] * inv), hi = pack_bf16(o[2] * inv, o[3] * inv);
    if (p.vec_out) {
      *reinterpret_cast<uint2 *>(out + c) = make_uint2(lo, hi);
    } else {
      out[c] = static_cast<uint16_t>(lo), out[c + 1] = static_cast<uint16_t>(lo >> 16);
      out[c + 2] = static_cast<uint16_t>(hi), out[c + 3] = static_cast<uint16_t>(hi >> 16);
    }
  }
}

template <int HDP, bool kOwnP>
__global__ void __launch_bounds__(kThreads, 1)
    attn_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v, const __grid_constant__ TcParams p) {
  using C = Cfg<HDP, kOwnP>;
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) uint64_t bar_full[kMaxSlots], bar_empty[kMaxSlots];
  __shared__ __align__(8) uint64_t bar_q, bar_s[2], bar_taken[2], bar_p[2][2], bar_pv[2];
  __shared__ __align__(8) uint64_t bar_drain, bar_dirty, bar_clean;
  __shared__ uint32_t tmem_base;
  __shared__ int gave_up, bad_seen;
  __shared__ int fields[kFields];

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  // (all kv heads of the largest item first: with the items of one head after the other the mixed prompts took a
  // sixth longer)
  const int item = blockIdx.x / p.d.nkv, kvh = blockIdx.x - item * p.d.nkv, split = blockIdx.y;
  const uint32_t smem_q = (smem_u32(raw) + 1023u) & ~1023u;
  const uint32_t ring = smem_q + 2 * C::kSlotBytes;

  if (warp == 8 && elect()) {
    for (int i = 0; i < C::kSlots; ++i) {
      mbar_init(smem_u32(&bar_full[i]), 1);
      mbar_init(smem_u32(&bar_empty[i]), 1);
    }
    mbar_init(smem_u32(&bar_q), 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(smem_u32(&bar_s[s]), 1);
      mbar_init(smem_u32(&bar_p[s][0]), 4);
      mbar_init(smem_u32(&bar_p[s][1]), 4);
      mbar_init(smem_u32(&bar_taken[s]), 4);
      mbar_init(smem_u32(&bar_pv[s]), 1);
    }
    mbar_init(smem_u32(&bar_drain), 1);
    mbar_init(smem_u32(&bar_dirty), 1);
    mbar_init(smem_u32(&bar_clean), 2);
    gave_up = 0;
    bad_seen = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_q) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_base))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    fence_before();
  }
  const auto field = [&](int f) { return lds32(smem_u32(&fields[f])); };
  int pairs, n_k, k_row = 0, k_b = 0;
  if (warp == 8) {
    // looks up what the CTA works on and asks for the first tiles; the others take it from there (all twelve warps
    // looking it up took each other's issue slots)
    const Item w = make_item(p, item, split);
    const bool pair = w.live && w.cnt1 > 0;
    // pair: key tiles of each stream (the second tile's tokens are later: they see as many or more);
    // solo: the tiles that both streams take in turn
    const int n0 = !w.live ? 0 : max(0, min((w.end0 + kTile - 1) / kTile, w.tb) - w.ta);
    const int nk = !w.live ? 0 : pair ? max(n0, min((w.end1 + kTile - 1) / kTile, w.tb) - w.ta) : n0;
    if (elect()) {
      fields[kLive] = w.live;
      fields[kQ0] = w.s.q0;
      fields[kQb] = w.s.qb;
      fields[kKb] = w.s.kb;
      fields[kK0] = w.s.k0;
      fields[kKeys] = w.s.L;
      fields[kOff] = w.s.off;
      fields[kT0] = w.t0;
      fields[kCnt0] = w.cnt0;
      fields[kCnt1] = w.cnt1;
      fields[kEnd] = max(w.end0, w.end1);
      fields[kLow0] = w.low0;
      fields[kLow1] = w.low1;
      fields[kTa] = w.ta;
      fields[kPairs] = pair;
      fields[kTiles] = nk;
      fields[kTiles0] = n0;
      fields[kShares] = w.live ? w.shares : 0;
      // the first key tile of this share that some row does not see in full
      fields[kSeenInFull] = max(0, (pair ? min(w.low0, w.low1) : w.low0) / kTile - w.ta);
    }
    __syncwarp();
    asm volatile("bar.arrive 2, 384;" ::: "memory");
    pairs = uniform(pair);
    n_k = uniform(nk);
    k_row = uniform(w.s.k0 + w.ta * kTile);
    k_b = uniform(w.s.kb);
  } else {
    asm volatile("bar.sync 2, 384;" ::: "memory");
    fence_after();
    pairs = uniform(field(kPairs));
    n_k = uniform(field(kTiles));
  }
  // The ring holds the tiles in the order in which the matrix instructions want them: `ahead` K tiles, then the next K
  // and a V in turn, then the V that are left.
  const int ahead = (pairs ? 0 : 1) + (kOwnP ? 1 : 0);
  const auto pos_v = [&](int j) { return j + ahead < n_k ? ahead + 2 * j + 1 : n_k + j; };
  const auto at = [&](int pos, int &j) {  // what is at a ring position: tile number, and whether it is V's
    if (pos < min(ahead, n_k)) {
      j = pos;
      return false;
    }
    const int q = max(0, pos - ahead);
    if (q / 2 + ahead < n_k) {
      j = q / 2 + (q & 1 ? 0 : ahead);
      return (q & 1) != 0;
    }
    j = pos - n_k;
    return true;
  };
  const int early = min(2 * n_k, C::kSlots);  // tiles that fit the empty ring: asked for before anything else
  const auto fetch = [&](const CUtensorMap *map, int j, int slot) {
    if (elect()) {
      const uint32_t fb = smem_u32(&bar_full[slot]);
      mbar_expect(fb, C::kSlotBytes);
#pragma unroll
      for (int h = 0; h < C::kHalves; ++h)
        tma_load_4d(ring + slot * C::kSlotBytes + h * 16384, map, h * 64, k_row + j * kTile, kvh, k_b, fb);
    }
    __syncwarp();
  };
  if (warp == 8 && n_k > 0) {
    const int q_row = uniform(field(kQ0) + field(kT0)), q_b = uniform(field(kQb));
    if (elect()) {
      const uint32_t qbar = smem_u32(&bar_q);
      const uint32_t bytes = static_cast<uint32_t>(p.group * p.tt * 128 * C::kHalves);
      mbar_expect(qbar, pairs ? 2 * bytes : bytes);
      for (int s = 0; s < (pairs ? 2 : 1); ++s)
        for (int h = 0; h < C::kHalves; ++h)
          tma_load_4d(smem_q + s * C::kSlotBytes + h * 16384, &map_q, h * 64, kvh * p.group, q_row + s * p.tt, q_b,
                      qbar);
    }
    __syncwarp();
#pragma unroll 1
    for (int pos = 0; pos < early; ++pos) {
      int j;
      const bool is_v = at(pos, j);
      fetch(is_v ? &map_v : &map_k, j, pos);
    }
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // the whole tensor memory is taken, so it starts at column 0 (Cfg has what lies where)

  // 384 threads start with 168 registers each; the softmax warps take over what the others leave
  // (256 x 216 + 128 x 72 = 384 x 168)
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 8) {
      if (n_k > 0) {
        int slot = 0, issued = early;
        unsigned phase = 0;  // of the slot's release that the next load waits for
#pragma unroll 1
        for (; issued < 2 * n_k; ++issued) {
          int j;
          const bool is_v = at(issued, j);
          if (!warp_wait(smem_u32(&bar_empty[slot]), phase, &gave_up)) break;
          fetch(is_v ? &map_v : &map_k, j, slot);
          if (++slot == C::kSlots) slot = 0, phase ^= 1u;
        }
        // copies in flight land before the CTA can end (bounded)
        (void)warp_wait(smem_u32(&bar_q), 0, &gave_up);
#pragma unroll 1
        for (int pos = max(0, issued - C::kSlots); pos < issued; ++pos)
#pragma unroll 1
          for (unsigned i = 0; i < kWaitLimit; ++i) {
            if (__all_sync(0xffffffffu, mbar_try(smem_u32(&bar_full[pos % C::kSlots]),
                                                 static_cast<unsigned>(pos / C::kSlots) & 1u)))
              break;
            __nanosleep(32);
          }
      }
    } else if (warp == 9) {
      if (n_k > 0) {
        constexpr uint32_t id_s = idesc_bf16(kTile, 0), id_o = idesc_bf16(HDP, 1);
        const uint32_t dq = desc_kmajor(smem_q), dk = desc_kmajor(ring), dv = desc_mnmajor(ring);
        constexpr uint32_t kSlotStep = C::kSlotBytes >> 4;
        const int n_0 = uniform(field(kTiles0)), n_full = uniform(field(kSeenInFull));
        unsigned clean_ph = 0, p_ph = 0, open = 0;  // p_ph, open: a bit per stream; open: its O has been written
        int slot = 0, k = 0, v = 0;
        unsigned phase = 0;
        bool ok = warp_wait(smem_u32(&bar_q), 0, &gave_up);
        // K and V tiles are taken in ring order: waits for the next one, returns its slot
        const auto next = [&](int &taken) {
          taken = slot;
          const bool r = warp_wait(smem_u32(&bar_full[slot]), phase, &gave_up);
          if (++slot == C::kSlots) slot = 0, phase ^= 1u;
          return r;
        };
        // Step u: the product with V of key tile j and the scores of that stream's next tile js; the scores first where
        // they need not wait for the product. A pair's streams share key tile j = u div 2; solo, tile j = u belongs to
        // stream j mod 2. The first two steps only make scores.
        const int total = pairs ? 2 * n_k : n_k;
        unsigned taken_ph = 0;
        const auto scores = [&](const int s, int js, int mine, bool takes, bool leaves) {
          if (js >= n_k) return true;
          if (takes && !next(k)) return false;
          if (js < mine) {
            fence_after();
            if (elect()) {
              const uint32_t a = dq + (pairs ? s * kSlotStep : 0), b = dk + k * kSlotStep;
#pragma unroll
              for (int i = 0; i < C::kHalves * 4; ++i)
                mma_ss(s * 128, a + (i / 4) * 1024 + (i % 4) * 2, b + (i / 4) * 1024 + (i % 4) * 2, id_s, i > 0);
              mma_commit(smem_u32(&bar_s[s]));
              if (leaves) mma_commit(smem_u32(&bar_empty[k]));
            }
            __syncwarp();
          }
          return true;
        };
        // (two steps to an iteration: the streams' addresses are constants then)
        const auto step = [&](const int u, const int s) {
          const int j = pairs ? u >> 1 : u, js = pairs ? j + 1 : j + 2;
          const int mine = pairs && s == 0 ? n_0 : n_k;  // this stream's tiles lie before this one
          const bool takes = !pairs || s == 0, leaves = !pairs || s == 1;
          const uint32_t ts = (kOwnP ? C::kColP : 0) + s * C::kStepP, to = C::kColO + s * C::kStepO;
          if (kOwnP) {
            if (j >= 0 && js < mine) {
              if (!warp_wait(smem_u32(&bar_taken[s]), taken_ph >> s & 1u, &gave_up)) return false;
              taken_ph ^= 1u << s;
            }
            if (!scores(s, js, mine, takes, leaves)) return false;
          }
          if (j >= 0) {
            if (takes) {
              if (!next(v)) return false;
              // warps 10-11 look V over (while the softmax runs) where some row does not see all of it
              if (j >= n_full && elect()) mbar_arrive(smem_u32(&bar_dirty));
              __syncwarp();
            }
            if (j < mine && !warp_wait(smem_u32(&bar_p[s][0]), p_ph >> s & 1u, &gave_up)) return false;
            if (takes && j >= n_full) {
              if (!warp_wait(smem_u32(&bar_clean), clean_ph, &gave_up)) return false;
              clean_ph ^= 1u;
            }
            if (j < mine) {
              // 64 keys, and then the other 64, whose weights may still be on their way
              fence_after();
              const uint32_t b = dv + v * kSlotStep;
              if (elect()) {
                mma_ts(to, ts, b, id_o, open >> s & 1u);
#pragma unroll
                for (int i = 1; i < kTile / 32; ++i) mma_ts(to, ts + i * 8, b + i * 128, id_o, 1);
              }
              __syncwarp();
              open |= 1u << s;
              if (!warp_wait(smem_u32(&bar_p[s][1]), p_ph >> s & 1u, &gave_up)) return false;
              p_ph ^= 1u << s;
              fence_after();
              if (elect()) {
#pragma unroll
                for (int i = kTile / 32; i < kTile / 16; ++i) mma_ts(to, ts + i * 8, b + i * 128, id_o, 1);
                if (leaves) mma_commit(smem_u32(&bar_empty[v]));
                if (kOwnP || js >= mine) mma_commit(smem_u32(&bar_pv[s]));
              }
              __syncwarp();
            }
          }
          return kOwnP || scores(s, js, mine, takes, leaves);
        };
#pragma unroll 1
        for (int u = -2; ok && u < total; u += 2) {
          ok = step(u, 0);
          if (ok && u + 1 < total) ok = step(u + 1, 1);
        }
        // nothing of this CTA is in flight in the tensor core when it ends
        if (elect()) mma_commit(smem_u32(&bar_drain));
        __syncwarp();
#pragma unroll 1
        for (unsigned i = 0; i < kWaitLimit; ++i) {
          if (__all_sync(0xffffffffu, mbar_try(smem_u32(&bar_drain), 0))) break;
          __nanosleep(32);
        }
      }
    } else {
      // ---- V tiles that some row does not see in full: what is not finite becomes zero
      const int seen_end = field(kEnd), ta = field(kTa), first_masked = field(kSeenInFull);
      const int self = static_cast<int>(threadIdx.x) - 320;
      for (int j = first_masked; j < n_k; ++j) {
        if (!warp_wait(smem_u32(&bar_dirty), (j - first_masked) & 1u, &gave_up)) break;
        const uint32_t base = ring + (pos_v(j) % C::kSlots) * C::kSlotBytes;
        const int rows_seen = seen_end - (ta + j) * kTile;
        // a value times zero is zero unless it is not finite: one multiply-add for two values finds whether any is
        const __nv_bfloat162 zero = __floats2bfloat162_rn(0.f, 0.f);
        __nv_bfloat162 any = zero;
#pragma unroll 4
        for (int e = self; e < C::kSlotBytes / 16; e += 64) {
          uint32_t x[4];
          lds128(base + e * 16, x);
#pragma unroll
          for (int i = 0; i < 4; ++i) any = __hfma2(*reinterpret_cast<__nv_bfloat162 *>(&x[i]), zero, any);
        }
        if (__hisnan(any.x) || __hisnan(any.y)) {
#pragma unroll 1
          for (int e = self; e < C::kSlotBytes / 16; e += 64) {
            uint32_t x[4];
            lds128(base + e * 16, x);
            bool found = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (not_finite_bf16(x[i])) x[i] &= 0xffff0000u, found = true;
              if (not_finite_bf16(x[i] >> 16)) x[i] &= 0x0000ffffu, found = true;
            }
            if (!found) continue;
            sts128(base + e * 16, make_uint4(x[0], x[1], x[2], x[3]));
            if ((e % 1024) / 8 < rows_seen) bad_seen = 1;
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_clean));
      }
    }
  } else if (field(kLive)) {  // uniform over the CTA
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ---- softmax: one thread per row of the stream's tile
    const int s = warp >> 2;
    const bool pair = pairs;
    const int nk = n_k, tile = pair ? s : 0;
    const int cnt = field(tile ? kCnt1 : kCnt0);
    const int wrow = (warp & 3) * 32, row = wrow + lane;
    const int rows = cnt * p.group;
    const bool active = wrow < rows;  // a warp without rows only keeps the barriers going
    const int tok = min((row * p.group_rcp) >> 16, cnt - 1);
    const int tok0 = (wrow * p.group_rcp) >> 16, tok1 = min(((wrow + 31) * p.group_rcp) >> 16, cnt - 1);
    const uint32_t lanes = static_cast<uint32_t>(wrow) << 16;
    const uint32_t ts = s * 128 + lanes, to = C::kColO + s * C::kStepO + lanes;
    const uint32_t tp = (kOwnP ? C::kColP : 0) + s * C::kStepP + lanes;
    const float sl = p.scale_log2;
    float m = -INFINITY, l = 0.f;
    const int mine = pair ? (s ? nk : field(kTiles0)) : (nk + 1 - s) / 2;
    bool ok = true;
    const auto seq = [&] {
      Seq r;
      r.q0 = field(kQ0), r.m = 0, r.qb = field(kQb), r.kb = field(kKb), r.k0 = field(kK0), r.L = field(kKeys);
      r.off = field(kOff);
      return r;
    };
    // one tile; a copy of its own for the tiles that every row sees in full (all but the last few of a long prompt)
    const auto softmax_tile = [&](int it, auto masked) {
      constexpr bool kMasked = decltype(masked)::value;
      uint32_t bits[4] = {~0u, ~0u, ~0u, ~0u};
      if (kMasked && active)
        seen_words(p, seq(), field(kT0) + tile * p.tt, tok, tok0, tok1, field(kTa) + (pair ? it : 2 * it + s), bits);
      if (!warp_wait(smem_u32(&bar_s[s]), it & 1, &gave_up)) return false;
      fence_after();
      if (active) {
        uint32_t x[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(ts + 32 * c, x + 32 * c);
        tmem_wait_ld();
        if (kOwnP) {
          fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&bar_taken[s]));
        }
        if (kMasked) {
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (!((bits[i / 32] >> (i % 32)) & 1u)) x[i] = 0xff800000u;  // -infinity
        }
        // a NaN among the scores makes the row's maximum, and with it the row, NaN
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 128; i += 2)
          top[i / 2 % 4] = max_nan3(top[i / 2 % 4], __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
        const float mz = max_nan(max_nan(top[0], top[1]), max_nan(top[2], top[3])) * sl;
        const bool follow = !(mz <= m + kFollow);
        // P and O are free once the product of the stream's previous tile is done (where P lies over S, this tile's
        // scores were ready only after it)
        if (kOwnP && it > 0) {
          if (!warp_wait(smem_u32(&bar_pv[s]), (it - 1) & 1, &gave_up)) return false;
          fence_after();
        }
        if (__any_sync(0xffffffffu, follow)) {
          const float mn = follow ? mz : m;
          const float a = m == -INFINITY ? 0.f : ex2(m - mn);
          if (it > 0) {
#pragma unroll 1
            for (int c = 0; c < HDP / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(to + 32 * c, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * a);
              tmem_st32(to + 32 * c, o);
            }
          }
          l *= a;
          m = mn;
        }
        // nothing seen yet: any finite reference; a score of infinity: NaN, as infinity minus itself
        const float ref = m == -INFINITY ? 0.f : (m == INFINITY ? __uint_as_float(0x7fffffffu) : m);
        const uint64_t sl2 = two(sl), ref2 = two(-ref);
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint64_t z = fma2(two(x[32 * c + 2 * i], x[32 * c + 2 * i + 1]), sl2, ref2);
            const float e0 = ex2(low_of(z)), e1 = ex2(high_of(z));
            sum[i % 2] = add2(sum[i % 2], two(__float_as_uint(e0), __float_as_uint(e1)));
            pk[i] = pack_bf16(e0, e1);  // the matrix product takes BF16; the sum keeps fp32
          }
          tmem_st16(tp + 16 * c, pk);
          if (c == 1) {  // the first 64 keys' weights can be used
            tmem_wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bar_p[s][0]));
          }
        }
        const uint64_t both = add2(sum[0], sum[1]);
        l += low_of(both) + high_of(both);
        tmem_wait_st();
      } else {
        if (kOwnP) {
          if (lane == 0) mbar_arrive(smem_u32(&bar_taken[s]));
          // no further than the warps with rows: an arrival counts for the phase that is open
          if (it > 0 && !warp_wait(smem_u32(&bar_pv[s]), (it - 1) & 1, &gave_up)) return false;
        }
        if (lane == 0) mbar_arrive(smem_u32(&bar_p[s][0]));
      }
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bar_p[s][1]));
      return true;
    };
    int it = 0;
    const int in_full = field(tile ? kLow1 : kLow0) / kTile - field(kTa);
    const int full = max(0, min(mine, pair ? in_full : (in_full - s + 1) / 2));
#pragma unroll 1
    for (; ok && it < full; ++it) ok = softmax_tile(it, std::false_type{});
#pragma unroll 1
    for (; ok && it < mine; ++it) ok = softmax_tile(it, std::true_type{});
    // a stream without tiles has no products to wait for; its Q tile, which its rows go out through, still has to land
    if (ok && mine > 0) ok = warp_wait(smem_u32(&bar_pv[s]), kOwnP ? (mine - 1) & 1 : 0, &gave_up);
    if (ok && mine == 0 && nk > 0) ok = warp_wait(smem_u32(&bar_q), 0, &gave_up);
    fence_after();

    if (mine > 0 && active && ok && __any_sync(0xffffffffu, *static_cast<volatile int *>(&bad_seen) != 0)) {
      const int step = pair ? 1 : 2, first_masked = field(kSeenInFull), ta = field(kTa);
      int first = pair ? 0 : s;
      if (first < first_masked) first += (first_masked - first + step - 1) / step * step;
      add_not_finite<HDP>(p, seq(), field(kT0) + tile * p.tt, kvh, tok, tok0, tok1, ta + first,
                          ta + (pair ? mine : nk), step, to);
    }
    // Solo: the two streams' sums over the same rows are joined through shared memory (over the ring, whose last tile
    // both have waited for): each stream hands over the half of its columns that the other one finishes.
    constexpr int kHalf = HDP / 2;
    float *joined = reinterpret_cast<float *>(raw + (ring - smem_u32(raw)));  // [HDP][128]
    float *join = joined + HDP * kTile;  // maximum and sum of each stream's rows
    const bool second = !pair && nk > 1;
    float a0 = 1.f, a1 = 0.f;
    if (second) {
      asm volatile("bar.sync 1, 256;" ::: "memory");
      join[2 * s * kTile + row] = m;
      join[(2 * s + 1) * kTile + row] = l;
      if (active && ok) {
#pragma unroll 1
        for (int c = 0; c < kHalf; c += 16) {
          const int col = (1 - s) * kHalf + c;
          uint32_t o[16];
          tmem_ld16(to + col, o);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) joined[(col + i) * kTile + row] = __uint_as_float(o[i]);
        }
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
      const float m1 = join[(2 - 2 * s) * kTile + row], mm = fmaxf(m, m1);
      const float ref = mm == -INFINITY ? 0.f : mm;
      a0 = ex2(m - ref);
      a1 = ex2(m1 - ref);
      l = l * a0 + join[(3 - 2 * s) * kTile + row] * a1;
      m = mm;
    }
    if ((pair || s == 0 || second) && active && ok) {
      const bool valid = row < rows;
      const float inv = p.splits > 1 ? 1.f : (l == 0.f ? 0.f : 1.f / l);
      a0 *= inv;
      a1 *= inv;
      const int64_t unit = ((static_cast<int64_t>(item) * p.splits + split) * p.d.nkv + kvh) * p.tpi + tile;
      float *part = p.cluster ? joined + (HDP + 4) * kTile : p.workspace + unit * (kTile * (HDP + 2));
      uint16_t *out = static_cast<uint16_t *>(p.d.out) + field(kQb) * p.d.out_batch_stride +
                      static_cast<int64_t>(field(kQ0) + field(kT0) + tile * p.tt) * p.d.out_token_stride +
                      static_cast<int64_t>(kvh * p.group) * p.d.out_head_stride;  // the tile's first row
      const uint32_t stage = smem_q + s * C::kSlotBytes + wrow * (2 * HDP);  // 32 rows of HDP values
      const int c_end = second ? (s + 1) * kHalf : HDP;
      int c = second ? s * kHalf : 0;
      if (!second && p.splits == 1 && mine > 0) {  // the whole row at once
        uint32_t o[HDP];
#pragma unroll
        for (int i = 0; i < HDP; i += 32) tmem_ld32(to + i, o + i);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < HDP; i += 8) {
          uint32_t x[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            x[k] = pack_bf16(__uint_as_float(o[i + 2 * k]) * a0, __uint_as_float(o[i + 2 * k + 1]) * a0);
          sts128(stage + lane * (2 * HDP) + (((i / 8) ^ (lane & 7)) * 16), make_uint4(x[0], x[1], x[2], x[3]));
        }
        c = c_end;
      }
#pragma unroll 1
      for (; c < c_end; c += 16) {
        float o[16];
        __syncwarp();  // lanes without a row left the last round early
        if (mine > 0) {
          tmem_ld16(to + c, reinterpret_cast<uint32_t *>(o));
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          o[i] *= a0;
          if (second) o[i] += joined[(c + i) * kTile + row] * a1;
        }
        if (p.splits > 1) {
          if (mine == 0 || !valid) continue;  // (the sum of zero written below says that there is nothing)
          // four columns of a row side by side, rows next to each other: 512 bytes to a store of the warp
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            reinterpret_cast<float4 *>(part)[(c + i) / 4 * kTile + row] = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        } else {
#pragma unroll
          for (int i = 0; i < 16; i += 8)
            sts128(stage + lane * (2 * HDP) + ((((c + i) / 8) ^ (lane & 7)) * 16),
                   make_uint4(pack_bf16(o[i], o[i + 1]), pack_bf16(o[i + 2], o[i + 3]), pack_bf16(o[i + 4], o[i + 5]),
                              pack_bf16(o[i + 6], o[i + 7])));
        }
      }
      if (p.splits == 1) {
        // a thread holds a row: written as they are, every store of a warp would touch 32 lines. Through the warp's
        // part of the Q tile (nothing reads it any more) a row's 16-byte pieces go out together.
        __syncwarp();
        const int per = second ? kHalf / 8 : HDP / 8;  // pieces of a row; a power of two
        const int at_once = 32 / per;                  // rows that the warp writes in one go
        const int q = (second ? s * per : 0) + lane % per;
        int r = lane / per;
        int head = wrow + r - ((wrow + r) * p.group_rcp >> 16) * p.group;
        uint16_t *to_row = out + static_cast<int64_t>((wrow + r) * p.group_rcp >> 16) * p.d.out_token_stride +
                           head * p.d.out_head_stride + q * 8;
        const int64_t next_token = p.d.out_token_stride - p.group * p.d.out_head_stride;
        if (q * 8 < p.d.hd) {
#pragma unroll 4
          for (; r < 32 && wrow + r < rows; r += at_once) {
            uint32_t x[4];
            lds128(stage + r * (2 * HDP) + ((q ^ (r & 7)) * 16), x);
            if (p.vec_out) {
              *reinterpret_cast<uint4 *>(to_row) = make_uint4(x[0], x[1], x[2], x[3]);
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i) to_row[i] = static_cast<uint16_t>(x[i / 2] >> (16 * (i & 1)));
            }
            to_row += at_once * p.d.out_head_stride;
            for (head += at_once; head >= p.group; head -= p.group) to_row += next_token;
          }
        }
      }
      if (p.splits > 1 && valid && (pair || s == 0)) {
        part[HDP * kTile + row] = m;
        part[(HDP + 1) * kTile + row] = l;
      }
    }
    fence_before();
  }
  __syncwarp();
  if (p.cluster) {
    cluster_barrier();  // every share's rows are in its CTA's shared memory
    if (warp < 8 && field(kLive)) join_cluster<HDP>(p, ring + (HDP + 4) * kTile * 4, kvh, split, field);
    __syncwarp();
    cluster_barrier();  // and none leaves while another one reads it
  }
  __syncthreads();
  if (threadIdx.x == 0 && gave_up && p.status) atomicOr(p.status, AIB_STATUS_WAIT_TIMEOUT);
  if (warp == 9) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem_base) : "memory");
  }
}

// Joins the shares of the key axis: out = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s.
// A block takes 32 rows and 32 columns of one tile: the weights of all shares
// first, then a warp for 8 columns, a lane for a row, the loads of 8 shares at
// once (one after the other they are all this kernel waits for).
constexpr int kMaxSplits = 64, kJoinThreads = 128, kJoinBatch = 8;

template <int HDP>
__global__ void __launch_bounds__(kJoinThreads) attn_join_kernel(const __grid_constant__ TcParams p) {
  __shared__ float weight[kMaxSplits][32], sums[kMaxSplits][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int item = blockIdx.x, kvh = blockIdx.y, quarter = blockIdx.z & 3, tile = blockIdx.z / 4 % p.tpi;
  const int c0 = (blockIdx.z / 4 / p.tpi) * 32 + warp * 8;
  const Item w = make_item(p, item, 0);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!w.live) return;
  const int rows = (tile ? w.cnt1 : w.cnt0) * p.group;
  if (quarter * 32 >= rows) return;
  const int row = quarter * 32 + lane;
  const bool valid = row < rows;
  const int64_t share = static_cast<int64_t>(p.d.nkv) * p.tpi * (kTile * (HDP + 2));
  const float *part = p.workspace + (static_cast<int64_t>(item) * p.splits * p.d.nkv * p.tpi + kvh * p.tpi + tile) *
                                        (kTile * (HDP + 2));
  // shares that the item's key tiles do not reach are not read; every other CTA wrote its rows in full
  const int last = w.shares - 1;
#pragma unroll 1
  for (int s0 = warp; s0 < w.shares; s0 += kJoinBatch * (kJoinThreads / 32)) {
    float x[kJoinBatch], y[kJoinBatch];
#pragma unroll
    for (int b = 0; b < kJoinBatch; ++b) {
      const float *r = part + min(s0 + b * (kJoinThreads / 32), last) * share + HDP * kTile + row;
      x[b] = __ldcg(r);
      y[b] = __ldcg(r + kTile);
    }
#pragma unroll
    for (int b = 0; b < kJoinBatch; ++b) {
      const int sp = min(s0 + b * (kJoinThreads / 32), last);
      weight[sp][lane] = x[b];
      sums[sp][lane] = y[b];
    }
  }
  __syncthreads();
  if (!valid || c0 >= p.d.hd) return;
  float m = -INFINITY;
#pragma unroll 4
  for (int sp = 0; sp < w.shares; ++sp) m = fmaxf(m, weight[sp][lane]);
  const float ref = m == -INFINITY ? 0.f : m;
  float l = 0.f, o[8] = {};
  const float4 *q = reinterpret_cast<const float4 *>(part) + c0 / 4 * kTile + row;
#pragma unroll 1
  for (int s0 = 0; s0 < w.shares; s0 += kJoinBatch) {
    float4 x[kJoinBatch][2];
#pragma unroll
    for (int b = 0; b < kJoinBatch; ++b) {
      const float4 *r = q + min(s0 + b, last) * (share / 4);  // behind the last share: again the last, not added
      x[b][0] = __ldcg(r);
      x[b][1] = __ldcg(r + kTile);
    }
#pragma unroll
    for (int b = 0; b < kJoinBatch; ++b) {
      if (s0 + b > last) break;
      const float a = ex2(weight[s0 + b][lane] - ref);
      l += a * sums[s0 + b][lane];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        o[4 * i] += a * x[b][i].x;
        o[4 * i + 1] += a * x[b][i].y;
        o[4 * i + 2] += a * x[b][i].z;
        o[4 * i + 3] += a * x[b][i].w;
      }
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] *= inv;
  const int tok = row / p.group;
  const int64_t token = w.s.q0 + w.t0 + tile * p.tt + tok;
  uint16_t *out = static_cast<uint16_t *>(p.d.out) + w.s.qb * p.d.out_batch_stride + token * p.d.out_token_stride +
                  static_cast<int64_t>(kvh * p.group + row - tok * p.group) * p.d.out_head_stride + c0;
  if (p.vec_out) {
    *reinterpret_cast<uint4 *>(out) = make_uint4(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]), pack_bf16(o[4], o[5]),
                                                 pack_bf16(o[6], o[7]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c0 + i < p.d.hd) out[i] = f2b(o[i]);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
static int check_common(const aib_attn_desc *p, const char *who) {
  if (!p) return aib_set_errorf("%s: null descriptor", who), AIB_EINVAL;
  if (p->tokens < 0 || p->batch < 0 || p->key_rows < 0 || p->nh < 1 || p->nkv < 1 || p->nh % p->nkv || p->hd < 1 ||
      p->hd > kPlainMaxHd)
    return aib_set_errorf("%s: bad shape (tokens %lld, batch %lld, key rows %lld, heads %d / %d, head size %d of at "
                          "most %d)", who, (long long)p->tokens, (long long)p->batch, (long long)p->key_rows, p->nh,
                          p->nkv, p->hd, kPlainMaxHd), AIB_EINVAL;
  const int64_t big = INT32_MAX - 1024;  // room for a tile behind the last row
  if (p->tokens > big || p->batch > big || p->key_rows > big)
    return aib_set_errorf("%s: tokens, batch and key rows must fit in 32 bits (below 2^31 - 1024)", who), AIB_EINVAL;
  if (p->sms < 0) return aib_set_errorf("%s: sms is negative", who), AIB_EINVAL;
  if (!std::isfinite(p->scale)) return aib_set_errorf("%s: scale is not finite", who), AIB_EINVAL;
  return AIB_OK;
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_fn() {
  static EncodeTiled fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiled>(p);
  });
  return fn;
}

// 4-D BF16 tensor (innermost first), box 64 columns x box1 x box2, 128-byte swizzle, zero fill outside
static bool make_map(CUtensorMap *map, const void *base, const int64_t (&size)[4], const int64_t (&stride)[3], int box1,
                     int box2) {
  EncodeTiled enc = encode_fn();
  if (!enc) return false;
  cuuint64_t dims[4], strides[3];
  for (int i = 0; i < 4; ++i) dims[i] = static_cast<cuuint64_t>(size[i]);
  // the stride of a dimension of one is never used
  for (int i = 0; i < 3; ++i) strides[i] = size[i + 1] > 1 ? static_cast<cuuint64_t>(stride[i]) * 2 : 16;
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box1), static_cast<cuuint32_t>(box2), 1};
  const cuuint32_t step[4] = {1, 1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void *>(base), dims, strides, box, step,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// a dimension that the TMA can step over: 16-byte steps, forward, no expanded tensor
static bool tma_stride(int64_t size, int64_t stride) {
  return size <= 1 || (stride > 0 && stride % 8 == 0 && stride < (1LL << 38));
}
static bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// The tensor-core kernel takes head sizes that are multiples of 8 up to 128,
// at most 128 heads per kv head, a positive scale (the maximum of the scores
// is taken before it) and what the TMA can address; the plain kernel takes
// the rest.
static bool tensor_cores(const aib_attn_desc &d, bool tree) {
  const int64_t b = tree ? d.batch : 1, kb = tree || d.len_k ? d.batch : 1;
  return d.hd % 8 == 0 && d.hd <= 128 && d.nh / d.nkv <= kTile && d.nkv <= 65535 && d.scale > 0.f && d.key_rows > 0 && aligned16(d.q) &&
         aligned16(d.k) && aligned16(d.v) && tma_stride(d.tokens, d.q_token_stride) &&
         tma_stride(d.nh, d.q_head_stride) && tma_stride(b, d.q_batch_stride) &&
         tma_stride(d.key_rows, d.k_token_stride) && tma_stride(d.nkv, d.k_head_stride) &&
         tma_stride(kb, d.k_batch_stride) && tma_stride(d.key_rows, d.v_token_stride) &&
         tma_stride(d.nkv, d.v_head_stride) && tma_stride(kb, d.v_batch_stride);
}

struct TcPlan {
  int group, tt, tpi, splits;
  bool cluster;
  int64_t items;
};

// clusters of `shares` CTAs of the attention kernel that the current device holds at once (0: none, or not known)
static int clusters_at_once(int hd, int shares);

static int64_t item_bound(const aib_attn_desc &d, bool tree, int64_t unit) {
  if (tree) return d.batch * ((d.tokens + unit - 1) / unit);
  // the sum of ceil(m_b / unit) over sequences whose m_b add up to at most `tokens`
  return std::min(d.tokens, (d.tokens + d.batch * (unit - 1)) / unit);
}

static TcPlan tc_plan(const aib_attn_desc &d, bool tree, int device_sms) {
  const int sms = d.sms > 0 ? static_cast<int>(std::min<int64_t>(d.sms, device_sms)) : device_sms;
  TcPlan pl;
  pl.group = d.nh / d.nkv;
  pl.tt = kTile / pl.group;
  pl.tpi = tree && d.tokens <= pl.tt ? 1 : 2;
  pl.splits = 1;
  pl.cluster = false;
  pl.items = item_bound(d, tree, 2LL * pl.tt);
  // Two tiles over the same keys halve the loads, but only where that still gives every SM an item. Where it does
  // not, one tile a CTA and a share of the key axis. 64 nodes over 32,000 slots: 497 us with two tiles and no shares,
  // 253 us with one tile and none, 86 us with two and nine shares, 63 us with one and six; 317 queries of two prompts
  // over 8000 and 4100 keys, one kv head: 134, 77, 31 and 28 us. Sixteen sequences of 26 nodes fill 128 of 148 SMs
  // and are not shared out: 32 us, with two and four shares in clusters 37 and 50 us, and with two, three and four
  // joined by a second kernel 1, 4 and 7 us more.
  if (pl.items * d.nkv < sms) {
    pl.tpi = 1;
    pl.items = item_bound(d, tree, pl.tt);
    const int64_t units = std::max<int64_t>(1, pl.items * d.nkv);
    // shares of at least two key tiles (one for each stream), at most one CTA per SM. The lengths are on the device, so
    // the tiles are those of the whole cache: one token over 1000 slots takes 9.5 us in a cache of 1152 rows, 9.6 in
    // one of 8192 and 12.2 in one of 32,768; 26 nodes 15.0, 15.5 and 15.5.
    const int64_t tiles = (d.key_rows + kTile - 1) / kTile;
    const int64_t cap = std::max<int64_t>(1, sms / units);
    pl.splits = static_cast<int>(std::min<int64_t>(std::min<int64_t>(cap, (tiles + 1) / 2), kMaxSplits));
    // Shares that are one cluster join in its shared memory and need no second kernel and no workspace. A cluster has
    // 2, 4, 8 or 16 CTAs of one GPC, so there are fewer shares; taken where that costs at most three more rounds of two
    // key tiles, which is what the second kernel costs (a round is 1.2 us, its start and its work 3 to 4). One token
    // over 1000 slots: 9.4 us, against 10.9 with a second kernel; a chain of five over 4099 (8 shares, against 18):
    // 13.1 and 15.2; 317 queries over 8000 and 4100 keys (8, against 10): 19.9 and 22.4; but 64 nodes over 32,000 slots
    // (4, against 6): 68 and 53.
    if (pl.splits > 1) {
      int s = 2;
      while (s < pl.splits && s < 16) s *= 2;
      if (s > cap) s /= 2;
      while (s > 1 && clusters_at_once(d.hd, s) < units) s /= 2;  // all at once, or the last ones wait for the first
      const auto rounds = [&](int64_t shares) { return ((tiles + shares - 1) / shares + 1) / 2; };
      if (d.sms == 0 && s > 1 && rounds(s) <= rounds(pl.splits) + 3) {
        pl.splits = s;
        pl.cluster = true;
      }
    }
  }
  return pl;
}

static int64_t tc_floats(const aib_attn_desc &d, const TcPlan &pl) {
  if (pl.splits == 1 || pl.cluster) return 0;
  const int hdp = d.hd <= 64 ? 64 : 128;
  return pl.items * pl.splits * d.nkv * pl.tpi * kTile * (hdp + 2);
}

static int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

// once per device: the shared-memory limit, and clusters of 16
template <int HDP, bool kOwnP>
static cudaError_t prepare_kernel() {
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !(ready.load() >> dev & 1))) {
    e = cudaFuncSetAttribute(attn_tc_kernel<HDP, kOwnP>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<HDP, kOwnP>::kSmem);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(attn_tc_kernel<HDP, kOwnP>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess && dev < 64) ready.fetch_or(1ull << dev);
  }
  return e;
}

static cudaLaunchAttribute cluster_of(int shares) {
  cudaLaunchAttribute a;
  a.id = cudaLaunchAttributeClusterDimension;
  a.val.clusterDim.x = 1;
  a.val.clusterDim.y = static_cast<unsigned>(shares);
  a.val.clusterDim.z = 1;
  return a;
}

template <int HDP>
static int query_clusters(int shares) {
  if (prepare_kernel<HDP, false>() != cudaSuccess) return (void)cudaGetLastError(), 0;
  cudaLaunchAttribute a = cluster_of(shares);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1, static_cast<unsigned>(shares));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Cfg<HDP, false>::kSmem;
  cfg.attrs = &a;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, attn_tc_kernel<HDP, false>, &cfg) != cudaSuccess) return (void)cudaGetLastError(), 0;
  return n;
}

static int clusters_at_once(int hd, int shares) {
  static std::atomic<int> known[64][2][17];  // 0: not asked yet; n + 1 otherwise
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return (void)cudaGetLastError(), 0;
  const bool wide = hd > 64;
  if (dev < 64) {
    const int k = known[dev][wide][shares].load();
    if (k) return k - 1;
  }
  const int n = wide ? query_clusters<128>(shares) : query_clusters<64>(shares);
  if (dev < 64) known[dev][wide][shares].store(n + 1);
  return n;
}

constexpr int kNoMaps = -1;  // the driver takes no tensor map of this layout: the plain kernel does the call

template <int HDP, bool kOwnP>
static int launch_tc(const aib_attn_desc &d, bool tree, const TcPlan &pl, const char *who, float *workspace,
                     int32_t *status, cudaStream_t st) {
  cudaError_t e = prepare_kernel<HDP, kOwnP>();
  if (e != cudaSuccess) return aib_set_errorf("%s: %s", who, cudaGetErrorString(e)), AIB_ECUDA;
  const int64_t kb = tree || d.len_k ? d.batch : 1;
  CUtensorMap mq, mk, mv;
  if (!make_map(&mq, d.q, {d.hd, d.nh, d.tokens, tree ? d.batch : 1},
                {d.q_head_stride, d.q_token_stride, d.q_batch_stride}, pl.group, pl.tt) ||
      !make_map(&mk, d.k, {d.hd, d.key_rows, d.nkv, kb}, {d.k_token_stride, d.k_head_stride, d.k_batch_stride}, kTile,
                1) ||
      !make_map(&mv, d.v, {d.hd, d.key_rows, d.nkv, kb}, {d.v_token_stride, d.v_head_stride, d.v_batch_stride}, kTile,
                1))
    return kNoMaps;
  TcParams p;
  p.d = d;
  p.group = pl.group;
  p.group_rcp = (65536 + pl.group - 1) / pl.group;
  p.tt = pl.tt;
  p.tpi = pl.tpi;
  p.splits = pl.splits;
  p.cluster = pl.cluster;
  p.scale_log2 = d.scale * 1.4426950408889634f;
  p.vec_out = aligned16(d.out) && d.out_token_stride % 8 == 0 && d.out_head_stride % 8 == 0 &&
              d.out_batch_stride % 8 == 0;
  p.workspace = workspace;
  p.status = status;
  const dim3 grid(static_cast<unsigned>(pl.items * d.nkv), static_cast<unsigned>(pl.splits));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr = cluster_of(pl.splits);
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Cfg<HDP, kOwnP>::kSmem;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = pl.cluster ? 1 : 0;
  e = cudaLaunchKernelEx(&cfg, attn_tc_kernel<HDP, kOwnP>, mq, mk, mv, p);
  if (e == cudaSuccess && pl.splits > 1 && !pl.cluster) {
    // started while the last shares still run (it waits for them before it reads)
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(pl.items), static_cast<unsigned>(d.nkv), 4 * pl.tpi * (HDP / 32));
    cfg.blockDim = dim3(kJoinThreads);
    cfg.dynamicSmemBytes = 0;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, attn_join_kernel<HDP>, p);
  }
  if (e != cudaSuccess) return aib_set_errorf("%s: %s", who, cudaGetErrorString(e)), AIB_ECUDA;
  return AIB_OK;
}

static int launch(const aib_attn_desc &d, const char *who, float *workspace, int64_t floats, int32_t *status,
                  cudaStream_t st) {
  const bool tree = d.mask != nullptr;
  if (tensor_cores(d, tree)) {
    const TcPlan pl = tc_plan(d, tree, sm_count());
    if (pl.items * pl.splits * d.nkv * 4 * pl.tpi > INT32_MAX) return aib_set_errorf("%s: too many rows", who), AIB_EINVAL;
    const int64_t need = tc_floats(d, pl);
    if (need && (!workspace || floats < need))
      return aib_set_errorf("%s: needs a workspace of %lld floats", who, (long long)need), AIB_EINVAL;
    if (need && !aligned16(workspace))  // shares are written and read four floats at a time
      return aib_set_errorf("%s: the workspace must start on a 16-byte boundary", who), AIB_EINVAL;
    const bool own = d.hd <= 64 && pl.tpi == 2;  // (Cfg has both sides)
    const int rc = own          ? launch_tc<64, true>(d, tree, pl, who, workspace, status, st)
                   : d.hd <= 64 ? launch_tc<64, false>(d, tree, pl, who, workspace, status, st)
                                : launch_tc<128, false>(d, tree, pl, who, workspace, status, st);
    if (rc != kNoMaps) return rc;
  }
  const int64_t rows = (tree ? d.batch : 1) * d.tokens * d.nh;
  const int64_t blocks = (rows + kPlainWarps - 1) / kPlainWarps;
  if (blocks > INT32_MAX) return aib_set_errorf("%s: too many rows", who), AIB_EINVAL;
  attn_plain_kernel<<<static_cast<unsigned>(blocks), kPlainWarps * 32, 0, st>>>(d);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return aib_set_errorf("%s: %s", who, cudaGetErrorString(e)), AIB_ECUDA;
  return AIB_OK;
}

}  // namespace aibseq

using namespace aibseq;

AIB_API int aib_prompt_attention_bf16(const aib_attn_desc *desc, float *workspace, int64_t workspace_floats,
                                      int32_t *d_status, void *stream) {
  const char *who = "prompt_attention";
  if (const int rc = check_common(desc, who)) return rc;
  aib_attn_desc p = *desc;
  p.mask = nullptr;
  if (p.tokens == 0 || p.batch == 0) return AIB_OK;
  if (!p.q || !p.out || !p.cu_q || (p.key_rows && (!p.k || !p.v)))
    return aib_set_errorf("%s: null pointer", who), AIB_EINVAL;
  if (!p.len_k && !p.cu_k) return aib_set_errorf("%s: give cu_k (packed keys) or len_k (caches)", who), AIB_EINVAL;
  return launch(p, who, workspace, workspace_floats, d_status, static_cast<cudaStream_t>(stream));
}

AIB_API int aib_tree_attention_bf16(const aib_attn_desc *desc, float *workspace, int64_t workspace_floats,
                                    int32_t *d_status, void *stream) {
  const char *who = "tree_attention";
  if (const int rc = check_common(desc, who)) return rc;
  const aib_attn_desc &p = *desc;
  if (p.mask_cols < 0 || p.mask_cols > p.key_rows)
    return aib_set_errorf("%s: %lld mask columns for caches of %lld rows", who, (long long)p.mask_cols,
                          (long long)p.key_rows), AIB_EINVAL;
  if (p.tokens == 0 || p.batch == 0) return AIB_OK;
  if (!p.q || !p.out || !p.pos || !p.mask || (p.key_rows && (!p.k || !p.v)))
    return aib_set_errorf("%s: null pointer", who), AIB_EINVAL;
  return launch(p, who, workspace, workspace_floats, d_status, static_cast<cudaStream_t>(stream));
}

AIB_API int64_t aib_attention_workspace_floats(const aib_attn_desc *d) {
  if (check_common(d, "attention_workspace_floats") || d->tokens == 0 || d->batch == 0) return 0;
  const auto floats = [&](bool tree) {
    return tensor_cores(*d, tree) ? tc_floats(*d, tc_plan(*d, tree, sm_count())) : 0;
  };
  // the prompt entry does not look at the mask, nor the tree entry at cu_q: what has both does for either
  if (!d->mask) return floats(false);
  return d->cu_q ? std::max(floats(false), floats(true)) : floats(true);
}
