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

__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  return static_cast<uint32_t>(f2b(hi)) << 16 | f2b(lo);
}
__device__ __forceinline__ void unpack(const uint4 &v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}

// Head sizes 16 LPR (64, 128, 256) with everything on 16-byte boundaries. One
// block per token; LPR lanes to a head, a lane with eight values of the first
// half and their eight partners of the second, so that the rotation stays in
// the lane and the norm takes log2(LPR) shuffles. Bound by memory: the rows
// are asked for before the block looks up its sequence and makes its angles
// (a chain of loads of its own), two rows to a thread at once, and the angles
// are read from shared memory where they are used, which lets five blocks
// share an SM: 8192 tokens of 48 heads of 128 (201 MB) take 34.6 us (5.82
// TB/s, 0.89 of the measured copy rate), 37.4 us at four blocks, 42 us at
// three, 86 us with a warp per head in turn. 26 tokens: 3.4 us, of which the
// chain of loads is most.
template <int LPR>
__global__ void __launch_bounds__(256, 5) rope_cache_vec_kernel(const RopeParams p) {
  constexpr int kHalf = 8 * LPR, kHd = 16 * LPR, kRows = 256 / LPR, kAtOnce = 2;
  __shared__ __align__(16) float cs[kHalf], sn[kHalf];
  const int64_t n = blockIdx.x;
  const int l = threadIdx.x % LPR, r = threadIdx.x / LPR;
  const int heads = p.nh + 2 * p.nkv;
  const uint16_t *x = p.qkv + n * p.qkv_stride + 8 * l;
  uint4 lo[kAtOnce], hi[kAtOnce];
  const auto load = [&](int h0) {
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int h = h0 + i * kRows + r;
      if (h < heads) {
        lo[i] = *reinterpret_cast<const uint4 *>(x + static_cast<int64_t>(h) * kHd);
        hi[i] = *reinterpret_cast<const uint4 *>(x + static_cast<int64_t>(h) * kHd + kHalf);
      }
    }
  };
  load(0);
  const float f = threadIdx.x < kHalf ? p.inv_freq[threadIdx.x] : 0.f;
  const int64_t depth = p.depth ? p.depth[n] : 0;
  const int64_t b = find_sequence(p.cu, p.batch, n);
  if (b < 0) return;  // uniform over the block
  const int64_t first = p.start[b], at = n - p.cu[b];
  const int64_t slot = first + at, place = first + (p.depth ? depth : at);
  const bool in_cache = slot >= 0 && slot < p.max_len;
  if (threadIdx.x < kHalf) turn(place, f, cs[threadIdx.x], sn[threadIdx.x]);
  __syncthreads();
  for (int h0 = 0; h0 < heads; h0 += kAtOnce * kRows) {
    if (h0) load(h0);
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int h = h0 + i * kRows + r;
      const bool is_q = h < p.nh, is_k = !is_q && h < p.nh + p.nkv;
      float u[8], v[8];
      unpack(lo[i], u);
      unpack(hi[i], v);
      if (p.qn) {  // every lane of a warp takes part in the sums
        float ss = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) ss += u[k] * u[k] + v[k] * v[k];
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float norm = rsqrtf(ss / static_cast<float>(kHd) + p.eps);
        if (is_q || is_k) {
          const uint16_t *w = (is_q ? p.qn : p.kn) + 8 * l;
          float wu[8], wv[8];
          unpack(*reinterpret_cast<const uint4 *>(w), wu);
          unpack(*reinterpret_cast<const uint4 *>(w + kHalf), wv);
#pragma unroll
          for (int k = 0; k < 8; ++k) u[k] *= norm * wu[k], v[k] *= norm * wv[k];
        }
      }
      if (h >= heads || (!is_q && !in_cache)) continue;
      uint16_t *o = is_q   ? p.q_out + (n * p.nh + h) * kHd
                    : is_k ? p.k + b * p.k_bs + (h - p.nh) * p.k_hs + slot * p.k_ts
                           : p.v + b * p.v_bs + (h - p.nh - p.nkv) * p.v_hs + slot * p.v_ts;
      uint4 a = lo[i], z = hi[i];
      if (is_q || is_k) {
        float c[8], s[8];
#pragma unroll
        for (int k = 0; k < 8; k += 4) {
          *reinterpret_cast<float4 *>(c + k) = *reinterpret_cast<const float4 *>(cs + 8 * l + k);
          *reinterpret_cast<float4 *>(s + k) = *reinterpret_cast<const float4 *>(sn + 8 * l + k);
        }
        uint32_t *aw = reinterpret_cast<uint32_t *>(&a), *zw = reinterpret_cast<uint32_t *>(&z);
#pragma unroll
        for (int k = 0; k < 8; k += 2) {
          aw[k / 2] = pack(u[k] * c[k] - v[k] * s[k], u[k + 1] * c[k + 1] - v[k + 1] * s[k + 1]);
          zw[k / 2] = pack(v[k] * c[k] + u[k] * s[k], v[k + 1] * c[k + 1] + u[k + 1] * s[k + 1]);
        }
      }
      *reinterpret_cast<uint4 *>(o + 8 * l) = a;
      *reinterpret_cast<uint4 *>(o + 8 * l + kHalf) = z;
    }
  }
}

// Every other head size and alignment. One block per token: its angles once,
// then a warp per head. Row values in fp32 (norm, rotation), one rounding at
// the write.
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

// The common case, an accepted path of a few rows: a warp takes one head's
// rows of one tensor and holds them all in registers between its reads and
// its writes (no other warp touches them), so nothing but the chain position
// -> row -> write is waited for.
constexpr int kKeepHeld = 8;  // units of a row that a lane holds

template <typename T>
__global__ void __launch_bounds__(256) keep_few_rows_kernel(const __grid_constant__ KeepParams p, int nkv) {
  const int head = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (head >= nkv) return;
  const int64_t b = blockIdx.z;
  T *base = static_cast<T *>(p.t[blockIdx.y]) + b * p.bs + head * p.hs;
  const int64_t pos = p.pos[b];
  const int64_t *keep = p.keep + b * p.n;
  T held[kKeepHeld];
  T *to[kKeepHeld];
#pragma unroll
  for (int k = 0; k < kKeepHeld; ++k) {
    const int e = lane + 32 * k, i = e / p.cols, c = e - i * p.cols;
    to[k] = nullptr;
    if (i >= p.n) continue;
    const int64_t s = keep[i], src = pos + s, dst = pos + i;
    if (s >= 0 && s != i && src >= 0 && src < p.max_len && dst >= 0 && dst < p.max_len) {
      held[k] = base[src * p.ts + c];
      to[k] = base + dst * p.ts + c;
    }
  }
  __syncwarp();
#pragma unroll
  for (int k = 0; k < kKeepHeld; ++k)
    if (to[k]) *to[k] = held[k];
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
  if (static_cast<int64_t>(p.n) * p.cols <= 32 * kKeepHeld) {
    const dim3 few(static_cast<unsigned>((nkv + 7) / 8), static_cast<unsigned>(tensors), static_cast<unsigned>(batch));
    keep_few_rows_kernel<T><<<few, 256, 0, st>>>(p, nkv);
    return cudaGetLastError();
  }
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
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(n);
  const uintptr_t low = reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out) |
                        reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |
                        reinterpret_cast<uintptr_t>(q_norm_w) | reinterpret_cast<uintptr_t>(k_norm_w) |
                        static_cast<uintptr_t>(qkv_stride | p.k_bs | p.k_hs | p.k_ts | p.v_bs | p.v_hs | p.v_ts) * 2;
  if (low % 16 == 0 && hd == 64)
    rope_cache_vec_kernel<4><<<grid, 256, 0, st>>>(p);
  else if (low % 16 == 0 && hd == 128)
    rope_cache_vec_kernel<8><<<grid, 256, 0, st>>>(p);
  else if (low % 16 == 0 && hd == 256)
    rope_cache_vec_kernel<16><<<grid, 256, 0, st>>>(p);
  else
    rope_cache_kernel<<<grid, 256, static_cast<size_t>(hd) * sizeof(float), st>>>(p);
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
