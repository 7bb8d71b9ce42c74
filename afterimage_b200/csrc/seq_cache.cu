// What stands around the attention over cached sequences (seq_attn.cu): the
// q/k norms, rotary embedding and cache write of packed prompts and drafted
// trees in front of it, and the rows of a cache that stay after a draft was
// accepted behind it. The reference leaves the first to transformers' modules
// (hooked at afterimage/runtime/streaming_engine.py:1871-1915) and has no
// cache in its speculation loop (:2488-2575).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "aib_internal.h"

namespace aibseqc {

__device__ __forceinline__ float b2f(uint16_t v) { return __uint_as_float(static_cast<uint32_t>(v) << 16); }
__device__ __forceinline__ uint16_t f2b(float f) { return __bfloat16_as_ushort(__float2bfloat16_rn(f)); }

struct RopeParams {
  const uint16_t *qkv;
  int64_t qkv_stride;
  const int64_t *cu, *start, *depth;
  const uint16_t *qn, *kn;
  const float *inv_freq;
  uint16_t *q_out, *k, *v;
  int64_t k_bs, k_hs, k_ts, v_bs, v_hs, v_ts;  // element strides of the caches: batch, head, row
  int64_t n, batch, max_len;
  int nh, nkv, hd;
  float eps;
};

// cos and sin of place * inv_freq. A far place leaves no digits of the angle
// in an fp32 product (at 100,000 it is 1/256 off), so the product and its
// reduction to one turn are done in 64 bits; what is left is below pi and
// fp32 from here on.
__device__ __forceinline__ void turn(int64_t place, float inv_freq, float &c, float &s) {
  const double a = static_cast<double>(place) * static_cast<double>(inv_freq);
  const double r = a - rint(a * 0.15915494309189535) * 6.283185307179586;
  sincosf(static_cast<float>(r), &s, &c);
}

// the sequence that row n belongs to: the last b with cu[b] <= n < cu[b + 1], or -1
__device__ __forceinline__ int64_t find_sequence(const int64_t *cu, int64_t batch, int64_t n) {
  int64_t lo = 0, hi = batch;  // cu[lo] <= n < cu[hi] where the row is in a sequence
  if (n < cu[0] || n >= cu[batch]) return -1;
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (cu[mid] <= n) lo = mid; else hi = mid;
  }
  return lo;
}

// One block per token: its angles once, then a warp per head. Row values in
// fp32 (norm, rotation), one rounding at the write.
__global__ void rope_cache_kernel(const RopeParams p) {
  extern __shared__ float cs[];  // cos[half], sin[half]
  const int64_t n = blockIdx.x;
  const int64_t b = find_sequence(p.cu, p.batch, n);
  if (b < 0) return;
  const int64_t at = n - p.cu[b];
  const int64_t slot = p.start[b] + at;
  const int64_t place = p.start[b] + (p.depth ? p.depth[n] : at);
  const bool in_cache = slot >= 0 && slot < p.max_len;
  const int half = p.hd / 2;
  for (int d = threadIdx.x; d < half; d += blockDim.x) turn(place, p.inv_freq[d], cs[d], cs[half + d]);
  __syncthreads();
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  for (int h = w; h < p.nh + 2 * p.nkv; h += nw) {
    const uint16_t *x = p.qkv + n * p.qkv_stride + static_cast<int64_t>(h) * p.hd;
    if (h >= p.nh + p.nkv) {
      if (!in_cache) continue;
      uint16_t *o = p.v + b * p.v_bs + (h - p.nh - p.nkv) * p.v_hs + slot * p.v_ts;
      for (int d = lane; d < p.hd; d += 32) o[d] = x[d];
      continue;
    }
    const bool is_q = h < p.nh;
    if (!is_q && !in_cache) continue;
    const uint16_t *nw_ = is_q ? p.qn : p.kn;
    float r = 1.f;
    if (nw_) {
      float ss = 0.f;
      for (int d = lane; d < p.hd; d += 32) ss += b2f(x[d]) * b2f(x[d]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      r = rsqrtf(ss / static_cast<float>(p.hd) + p.eps);
    }
    uint16_t *o = is_q ? p.q_out + (n * p.nh + h) * p.hd : p.k + b * p.k_bs + (h - p.nh) * p.k_hs + slot * p.k_ts;
    for (int d = lane; d < half; d += 32) {
      float lo = b2f(x[d]) * r, hi = b2f(x[d + half]) * r;
      if (nw_) lo *= b2f(nw_[d]), hi *= b2f(nw_[d + half]);
      const float c = cs[d], s = cs[half + d];
      o[d] = f2b(lo * c - hi * s);
      o[d + half] = f2b(hi * c + lo * s);
    }
  }
}

// ---------------------------------------------------------------------------
constexpr int kMaxTensors = 256;
constexpr int kMaxKeep = 256;
constexpr int kKeepBytes = 48 * 1024;  // rows that one block holds between its reads and its writes

struct KeepParams {
  void *t[kMaxTensors];
  const int64_t *pos, *keep;
  int64_t bs, hs, ts;  // strides in units of the copied type
  int64_t max_len;
  int n, cols;         // kept rows, units per row
  int slice;           // units of a row that one block takes
};

// row pos + i <- row pos + keep[i], as the rows were before the call: a block
// takes one head's rows (or a slice of their columns) of one tensor, reads
// all, then writes.
template <typename T>
__global__ void keep_rows_kernel(const __grid_constant__ KeepParams p) {
  extern __shared__ __align__(16) unsigned char raw[];
  T *buf = reinterpret_cast<T *>(raw);
  const int64_t b = blockIdx.z;
  T *base = static_cast<T *>(p.t[blockIdx.y]) + b * p.bs;
  const int slices = (p.cols + p.slice - 1) / p.slice;
  const int head = blockIdx.x / slices, c0 = (blockIdx.x % slices) * p.slice;
  const int cols = min(p.slice, p.cols - c0);
  base += head * p.hs + c0;
  const int64_t pos = p.pos[b];
  const int64_t *keep = p.keep + b * p.n;
  for (int e = threadIdx.x; e < p.n * cols; e += blockDim.x) {
    const int i = e / cols, c = e - i * cols;
    const int64_t s = keep[i], src = pos + s;
    if (s >= 0 && src >= 0 && src < p.max_len) buf[e] = base[src * p.ts + c];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.n * cols; e += blockDim.x) {
    const int i = e / cols, c = e - i * cols;
    const int64_t s = keep[i], src = pos + s, dst = pos + i;
    if (s >= 0 && s != i && src >= 0 && src < p.max_len && dst >= 0 && dst < p.max_len) base[dst * p.ts + c] = buf[e];
  }
}

template <typename T>
static cudaError_t launch_keep(KeepParams p, int tensors, int64_t batch, int nkv, int hd, int64_t bs, int64_t hs,
                               int64_t ts, cudaStream_t st) {
  const int per = sizeof(T) / 2;
  p.cols = hd / per;
  p.bs = bs / per;
  p.hs = hs / per;
  p.ts = ts / per;
  p.slice = p.cols;
  while (static_cast<int64_t>(p.slice) * p.n * sizeof(T) > kKeepBytes) p.slice = (p.slice + 1) / 2;
  const int slices = (p.cols + p.slice - 1) / p.slice;
  const dim3 grid(static_cast<unsigned>(nkv * slices), static_cast<unsigned>(tensors), static_cast<unsigned>(batch));
  keep_rows_kernel<T><<<grid, 128, static_cast<size_t>(p.slice) * p.n * sizeof(T), st>>>(p);
  return cudaGetLastError();
}

}  // namespace aibseqc

using namespace aibseqc;

AIB_API int aib_rope_cache_packed_bf16(const void *qkv, int64_t qkv_stride, int64_t n, int64_t batch, int nh, int nkv,
                                       int hd, const int64_t *cu, const int64_t *start, const int64_t *depth,
                                       const void *q_norm_w, const void *k_norm_w, float eps, const float *inv_freq,
                                       void *q_out, void *k_cache, void *v_cache, const int64_t *k_strides,
                                       const int64_t *v_strides, int64_t max_len, void *stream) {
  if (n < 0 || batch < 0 || nh < 1 || nkv < 1 || hd < 2 || hd % 2 || hd > 1024 || max_len < 1 || n > INT32_MAX ||
      nh + 2LL * nkv > 65535)
    return aib_set_error("rope_cache_packed: bad shape"), AIB_EINVAL;
  if (n == 0 || batch == 0) return AIB_OK;
  if (!qkv || !cu || !start || !inv_freq || !q_out || !k_cache || !v_cache || !k_strides || !v_strides)
    return aib_set_error("rope_cache_packed: null pointer"), AIB_EINVAL;
  if ((q_norm_w == nullptr) != (k_norm_w == nullptr))
    return aib_set_error("rope_cache_packed: give both q and k norm weights or neither"), AIB_EINVAL;
  RopeParams p;
  p.qkv = static_cast<const uint16_t *>(qkv);
  p.qkv_stride = qkv_stride;
  p.cu = cu;
  p.start = start;
  p.depth = depth;
  p.qn = static_cast<const uint16_t *>(q_norm_w);
  p.kn = static_cast<const uint16_t *>(k_norm_w);
  p.inv_freq = inv_freq;
  p.q_out = static_cast<uint16_t *>(q_out);
  p.k = static_cast<uint16_t *>(k_cache);
  p.v = static_cast<uint16_t *>(v_cache);
  p.k_bs = k_strides[0], p.k_hs = k_strides[1], p.k_ts = k_strides[2];
  p.v_bs = v_strides[0], p.v_hs = v_strides[1], p.v_ts = v_strides[2];
  p.n = n;
  p.batch = batch;
  p.max_len = max_len;
  p.nh = nh;
  p.nkv = nkv;
  p.hd = hd;
  p.eps = eps;
  rope_cache_kernel<<<static_cast<unsigned>(n), 256, static_cast<size_t>(hd) * sizeof(float),
                      static_cast<cudaStream_t>(stream)>>>(p);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return aib_set_errorf("rope_cache_packed: %s", cudaGetErrorString(e)), AIB_ECUDA;
  return AIB_OK;
}

AIB_API int aib_keep_cache_rows_bf16(void *const *tensors, int count, int64_t batch, int nkv, int64_t max_len, int hd,
                                     const int64_t *strides, const int64_t *pos, const int64_t *keep, int n,
                                     void *stream) {
  if (count < 0 || batch < 0 || nkv < 1 || max_len < 1 || hd < 1 || hd > 1024 || n < 0 || nkv > 65535 / 16)
    return aib_set_error("keep_cache_rows: bad shape"), AIB_EINVAL;
  if (n > kMaxKeep) return aib_set_errorf("keep_cache_rows: %d rows, at most %d", n, kMaxKeep), AIB_EINVAL;
  if (batch > 65535) return aib_set_error("keep_cache_rows: batch above 65535"), AIB_EINVAL;
  if (count == 0 || batch == 0 || n == 0) return AIB_OK;
  if (!tensors || !strides || !pos || !keep) return aib_set_error("keep_cache_rows: null pointer"), AIB_EINVAL;
  uintptr_t low = static_cast<uintptr_t>(strides[0] | strides[1] | strides[2] | hd) * 2;
  for (int i = 0; i < count; ++i) {
    if (!tensors[i]) return aib_set_errorf("keep_cache_rows: null tensor %d", i), AIB_EINVAL;
    low |= reinterpret_cast<uintptr_t>(tensors[i]);
  }
  KeepParams p;
  p.pos = pos;
  p.keep = keep;
  p.max_len = max_len;
  p.n = n;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  for (int i0 = 0; i0 < count; i0 += kMaxTensors) {
    const int m = count - i0 < kMaxTensors ? count - i0 : kMaxTensors;
    for (int i = 0; i < m; ++i) p.t[i] = tensors[i0 + i];
    // 16-byte copies where every base, stride and row allows them
    const cudaError_t e = low % 16 == 0
                              ? launch_keep<uint4>(p, m, batch, nkv, hd, strides[0], strides[1], strides[2], st)
                              : launch_keep<uint16_t>(p, m, batch, nkv, hd, strides[0], strides[1], strides[2], st);
    if (e != cudaSuccess) return aib_set_errorf("keep_cache_rows: %s", cudaGetErrorString(e)), AIB_ECUDA;
  }
  return AIB_OK;
}
