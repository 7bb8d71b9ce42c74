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
// replaced, not added to, and a masked v_j is never multiplied.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "aib_internal.h"

namespace aibseq {

__device__ __forceinline__ float b2f(uint16_t v) { return __uint_as_float(static_cast<uint32_t>(v) << 16); }
__device__ __forceinline__ uint16_t f2b(float f) { return __bfloat16_as_ushort(__float2bfloat16_rn(f)); }

__device__ __forceinline__ int64_t clamp64(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : (v > hi ? hi : v); }

// One sequence: where its queries and keys are and what its rows see. Every
// value is cut to the extents that the host checked, so that lengths on the
// device cannot lead outside a tensor.
struct Seq {
  int64_t q0, m;    // first query row (within the q batch of a tree: 0) and number of queries
  int64_t qb;       // q batch
  int64_t kb, k0;   // k batch and first key row
  int64_t L;        // keys
  int64_t off;      // prompt: row i sees keys < off + i + 1; tree: slot of the drafted column 0 (unclamped)
};

__device__ __forceinline__ Seq sequence(const aib_attn_desc &p, int64_t b) {
  Seq s;
  if (p.mask) {
    s.q0 = 0;
    s.m = p.tokens;
    s.qb = s.kb = b;
    s.k0 = 0;
    // a position outside [-columns, rows] means nothing more than its end of that range
    s.off = clamp64(p.pos[b], -p.mask_cols, p.key_rows);
    s.L = clamp64(s.off + p.mask_cols, 0, p.key_rows);
    return s;
  }
  s.q0 = clamp64(p.cu_q[b], 0, p.tokens);
  s.m = clamp64(p.cu_q[b + 1], s.q0, p.tokens) - s.q0;
  s.qb = 0;
  if (p.len_k) {
    s.kb = b;
    s.k0 = 0;
    s.L = clamp64(p.len_k[b], 0, p.key_rows);
  } else {
    s.kb = 0;
    s.k0 = clamp64(p.cu_k[b], 0, p.key_rows);
    s.L = clamp64(p.cu_k[b + 1], s.k0, p.key_rows) - s.k0;
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
         p.mask[s.qb * p.mask_batch_stride + i * p.mask_row_stride + c * p.mask_col_stride] != 0;
}

// ---------------------------------------------------------------------------
// The plain kernel: one warp for one row of one head, 32 keys at a time (a
// lane takes one key's score, then the warp adds the seen keys' values, a
// lane per value column). It takes every head size up to 256 and every
// stride; scores, sums and the running output are fp32, the result is
// rounded once.
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
    s = sequence(p, tok / p.tokens);
    i = tok % p.tokens;
  } else {
    int64_t b = 0;
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
// host side
// ---------------------------------------------------------------------------
static int check_common(const aib_attn_desc *p, const char *who) {
  if (!p) return aib_set_errorf("%s: null descriptor", who), AIB_EINVAL;
  if (p->tokens < 0 || p->batch < 0 || p->key_rows < 0 || p->nh < 1 || p->nkv < 1 || p->nh % p->nkv || p->hd < 1 ||
      p->hd > kPlainMaxHd)
    return aib_set_errorf("%s: bad shape (tokens %lld, batch %lld, key rows %lld, heads %d / %d, head size %d of at "
                          "most %d)", who, (long long)p->tokens, (long long)p->batch, (long long)p->key_rows, p->nh,
                          p->nkv, p->hd, kPlainMaxHd), AIB_EINVAL;
  const int64_t big = INT32_MAX;
  if (p->tokens > big || p->batch > big || p->key_rows > big)
    return aib_set_errorf("%s: tokens, batch and key rows must fit in 32 bits", who), AIB_EINVAL;
  if (!std::isfinite(p->scale)) return aib_set_errorf("%s: scale is not finite", who), AIB_EINVAL;
  return AIB_OK;
}

static int launch(const aib_attn_desc &p, const char *who, cudaStream_t st) {
  const int64_t rows = (p.mask ? p.batch : 1) * p.tokens * p.nh;
  const int64_t blocks = (rows + kPlainWarps - 1) / kPlainWarps;
  if (blocks > INT32_MAX) return aib_set_errorf("%s: too many rows", who), AIB_EINVAL;
  attn_plain_kernel<<<static_cast<unsigned>(blocks), kPlainWarps * 32, 0, st>>>(p);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return aib_set_errorf("%s: %s", who, cudaGetErrorString(e)), AIB_ECUDA;
  return AIB_OK;
}

}  // namespace aibseq

using namespace aibseq;

AIB_API int aib_prompt_attention_bf16(const aib_attn_desc *desc, int32_t *, void *stream) {
  const char *who = "prompt_attention";
  if (const int rc = check_common(desc, who)) return rc;
  aib_attn_desc p = *desc;
  p.mask = nullptr;
  if (p.tokens == 0 || p.batch == 0) return AIB_OK;
  if (!p.q || !p.out || !p.cu_q || (p.key_rows && (!p.k || !p.v)))
    return aib_set_errorf("%s: null pointer", who), AIB_EINVAL;
  if (!p.len_k && !p.cu_k) return aib_set_errorf("%s: give cu_k (packed keys) or len_k (caches)", who), AIB_EINVAL;
  return launch(p, who, static_cast<cudaStream_t>(stream));
}

AIB_API int aib_tree_attention_bf16(const aib_attn_desc *desc, int32_t *, void *stream) {
  const char *who = "tree_attention";
  if (const int rc = check_common(desc, who)) return rc;
  const aib_attn_desc &p = *desc;
  if (p.mask_cols < 0 || p.mask_cols > p.key_rows)
    return aib_set_errorf("%s: %lld mask columns for caches of %lld rows", who, (long long)p.mask_cols,
                          (long long)p.key_rows), AIB_EINVAL;
  if (p.tokens == 0 || p.batch == 0) return AIB_OK;
  if (!p.q || !p.out || !p.pos || !p.mask || (p.key_rows && (!p.k || !p.v)))
    return aib_set_errorf("%s: null pointer", who), AIB_EINVAL;
  return launch(p, who, static_cast<cudaStream_t>(stream));
}

AIB_API int64_t aib_attention_workspace_floats(const aib_attn_desc *) { return 0; }
