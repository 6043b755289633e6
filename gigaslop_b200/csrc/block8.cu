// The block-scaled FP8 format and the element-wise operators on it: E4M3 elements with one fp32 scale per block of 128 consecutive
// elements of a row (activations, gradients, checkpoints) or per 128 x 128 tile (weights).
//
//   quantise     s = 2^t, t the least integer with max|x| <= 448 2^t over the block's finite elements (s = 1 for a block without any that
//                is not zero; t >= -126), q = e4m3(x / s); NaN and infinities become NaN
//   restore      x^ = q s
//   SwiGLU       h = g sigmoid(g) u, quantised, together with the checkpoints of g and u
//   its gradient from the checkpoints: du = dh g^ sigmoid(g^),  dg = dh u^ sigmoid(g^) (1 + g^ sigmoid(-g^))
//
// A scale that is a power of two costs E4M3, a floating-point format, no relative precision; the division is exact, so the one rounding
// is the conversion, and a restored element is exact in fp32, in bf16, and in fp16 within its range (the weight gradient extends that: wgrad.cu).
//
// All of them are bound by HBM.  A lane owns 8 consecutive elements, so a block is half a warp, and its maximum four shuffles.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "capi_internal.h"
#include "ptx.cuh"

namespace gsb {

constexpr int B8 = 128;                       // elements of a block along a row
constexpr int B8_WARPS = 4;                   // (eight: the same or up to 4 % slower)
// Blocks per SM that the compiler leaves registers for: 40 warps for the kernels that reach it without spilling (SwiGLU gradient, M = 65536, F =
// 2048, bf16: 193 -> 174 us).
template <typename T, int V> constexpr int b8_resident(bool quant = false) { return sizeof(T) == 2 && V == 2 && !quant ? 10 : 1; }

// ---- 8 consecutive elements ------------------------------------------------------------------------------------------
template <typename T> struct Raw8 { uint4 w[sizeof(T) / 2]; };      // as loaded

__device__ __forceinline__ float2 pair_f32(uint32_t w, __half) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
__device__ __forceinline__ float2 pair_f32(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float (&v)[8]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = pair_f32(w[i], T{});
      v[2 * i] = f.x; v[2 * i + 1] = f.y;
    }
  }
}
template <typename T>
__device__ __forceinline__ Raw8<T> pack8(const float (&v)[8]) {
  Raw8<T> r;
  uint32_t* w = reinterpret_cast<uint32_t*>(&r);
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(v[i]);
  } else if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack_half2(v[2 * i], v[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
  }
  return r;
}

// Elements [c, c + 8) of a row of `cols`; what lies behind the row counts as zero.  V: 0 any rows, 1 rows that start on 16-byte (E4M3: 8-byte)
// boundaries, 2 such rows of whole vectors (no tail).
// First the whole vectors (load_row8, a predicated load each, so that many are in flight), then what is left (tail_row8): the vector in
// which the row ends, whole where the buffer goes on behind it (`room` elements from the row's start: the row stride, for the last row its
// length), and what has no alignment, one by one.
template <typename T, int V>
__device__ __forceinline__ Raw8<T> load_row8(const T* row, int c, int cols) {
  constexpr int W = sizeof(T) / 2;
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    r.w[i] = make_uint4(0u, 0u, 0u, 0u);
    if (V && c + 8 <= cols) r.w[i] = __ldcs(reinterpret_cast<const uint4*>(row + c) + i);
  }
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void tail_row8(Raw8<T>& r, const T* row, int c, int cols, long long room) {
  constexpr int W = sizeof(T) / 2;
  if (V == 2 || c >= cols || (V && c + 8 <= cols)) return;
  uint32_t w[4 * W];
#pragma unroll
  for (int i = 0; i < 4 * W; ++i) w[i] = 0u;
  if (V && c + 8 <= room) {
    const int n = cols - c;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const uint4 v = __ldcs(reinterpret_cast<const uint4*>(row + c) + i);
      w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
#pragma unroll
    for (int i = 0; i < 4 * W; ++i) {
      if constexpr (W == 1) w[i] = 2 * i + 1 < n ? w[i] : 2 * i < n ? w[i] & 0xffffu : 0u;
      else w[i] = i < n ? w[i] : 0u;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < cols) {
        if constexpr (W == 1) w[i >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(row)[c + i] << (16 * (i & 1));
        else w[i] = reinterpret_cast<const uint32_t*>(row)[c + i];
      }
  }
#pragma unroll
  for (int i = 0; i < W; ++i) r.w[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
}
template <typename T, int V>
__device__ __forceinline__ void store_row8(T* row, int c, int cols, const Raw8<T>& r) {
  constexpr int W = sizeof(T) / 2;
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
  if (V && c + 8 <= cols) {
#pragma unroll
    for (int i = 0; i < W; ++i) reinterpret_cast<uint4*>(row + c)[i] = r.w[i];
  } else if (V != 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < cols) {
        if constexpr (W == 1) reinterpret_cast<uint16_t*>(row)[c + i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
        else reinterpret_cast<uint32_t*>(row)[c + i] = w[i];
      }
  }
}
template <int V>
__device__ __forceinline__ uint2 load_q8(const uint8_t* row, int c, int cols) {
  uint2 q = make_uint2(0u, 0u);
  if (V && c + 8 <= cols) q = __ldcs(reinterpret_cast<const uint2*>(row + c));
  return q;
}
template <int V>
__device__ __forceinline__ void tail_q8(uint2& q, const uint8_t* row, int c, int cols, long long room) {
  if (V == 2 || c >= cols || (V && c + 8 <= cols)) return;
  if (V && c + 8 <= room) {
    const int n = cols - c;
    q = __ldcs(reinterpret_cast<const uint2*>(row + c));
    q.y = n <= 4 ? 0u : q.y & (0xffffffffu >> (8 * (8 - n)));
    q.x = n >= 4 ? q.x : q.x & (0xffffffffu >> (8 * (4 - n)));
  } else {
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < cols) w[i >> 2] |= (uint32_t)row[c + i] << (8 * (i & 3));
    q = make_uint2(w[0], w[1]);
  }
}
template <int V>
__device__ __forceinline__ void store_q8(uint8_t* row, int c, int cols, uint2 q) {
  if (V && c + 8 <= cols) {
    *reinterpret_cast<uint2*>(row + c) = q;
  } else if (V != 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < cols) row[c + i] = (uint8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
  }
}

// ---- the format ----------------------------------------------------------------------------------------------------------
// The scale of a block whose largest finite magnitude is amax: 448 = 1.75 2^8, so t is amax's exponent - 8, and one more where the
// significand is above 1.75.  The biased exponent of the scale is at least 1 (2^-126: its reciprocal is finite).
__device__ __forceinline__ float block_scale(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = (int)(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return amax > 0.f ? __uint_as_float((uint32_t)max(e, 1) << 23) : 1.f;
}
__device__ __forceinline__ float pow2_reciprocal(float s) { return __uint_as_float(0x7f000000u - __float_as_uint(s)); }     // 2^-t
__device__ __forceinline__ uint2 to_e4m3(const float (&v)[8], float inv) {
  uint32_t w[4];
  const float2 i2 = make_float2(inv, inv);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = __nv_cvt_float2_to_fp8x2(__fmul2_rn(make_float2(v[2 * i], v[2 * i + 1]), i2), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}
__device__ __forceinline__ void from_e4m3(uint2 q, float s, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = i < 2 ? q.x : q.y;
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * (i & 1))), __NV_E4M3);
    const float2 f = fmul2(__half22float2(__half2(h)), make_float2(s, s));
    v[2 * i] = f.x; v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ float half_warp_max(float m) {
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  return m;
}
__device__ __forceinline__ float max8(const float (&v)[8]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[i]));          // (fmaxf passes a NaN by)
  return m;
}
// Largest magnitude of 8 16-bit values as loaded, in both halves of a word (packed: exact, and half the instructions).
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b, __half) {
  const __half2 m = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b, __nv_bfloat16) {
  const __nv_bfloat162 m = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
template <typename T>
__device__ __forceinline__ uint32_t max8_packed(const Raw8<T>& r) {
  const uint4 w = r.w[0];
  uint32_t m = 0u;                                                 // (starts from 0: a NaN loses against it)
  m = max2(m, w.x & 0x7fff7fffu, T{});
  m = max2(m, w.y & 0x7fff7fffu, T{});
  m = max2(m, w.z & 0x7fff7fffu, T{});
  return max2(m, w.w & 0x7fff7fffu, T{});
}
// The block maxima of two tensors' vectors at once (of one: b = a).
template <typename T>
__device__ __forceinline__ float2 half_warp_max2(const Raw8<T>& a, const Raw8<T>& b) {
  const uint32_t ma = max8_packed<T>(a), mb = max8_packed<T>(b);
  uint32_t m = max2(__byte_perm(ma, mb, 0x5410), __byte_perm(ma, mb, 0x7632), T{});     // a in the low half, b in the high one
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) m = max2(m, __shfl_xor_sync(0xffffffffu, m, d), T{});
  return pair_f32(m, T{});
}
constexpr float FMAX = 3.402823466e38f;
// Infinities become NaN: they count for no maximum, and the conversion would saturate them.
__device__ __forceinline__ void drop_infinities(float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (fabsf(v[i]) > FMAX) v[i] = __int_as_float(0x7fffffff);
}
// For the block of a half-warp in which an infinity was found (all 32 lanes take part).
__device__ __forceinline__ float finite_half_warp_max(float (&v)[8]) {
  drop_infinities(v);
  return half_warp_max(max8(v));
}
// This lane's 8 values and the largest magnitude of its block
template <typename T>
__device__ __forceinline__ float values_and_max(const Raw8<T>& r, float (&v)[8]) {
  unpack8<T>(r, v);
  if constexpr (sizeof(T) == 2) return half_warp_max2<T>(r, r).x;
  else return half_warp_max(max8(v));
}

// The rows and blocks of a warp.  A warp owns a row and its half-warps every second block of it; where a row is one block, a row per
// half-warp.  Rows are walked from the last to the first, as the other quantisers do (the consumer reads upwards and finds in L2
// what was written last).
struct RowWalk {
  long long row;                        // the first; the others row_step apart
  int row_step, blk, blk_step;          // this half-warp's blocks
  __device__ __forceinline__ RowWalk(int nb, int rows = 1) {
    const int half = (threadIdx.x >> 4) & 1;
    const long long w = ((long long)(gridDim.x - 1 - blockIdx.x) * B8_WARPS + (threadIdx.x >> 5)) * rows;
    if (nb == 1) { row = 2 * w + half; row_step = 2; blk = 0; blk_step = 1; }
    else { row = w; row_step = 1; blk = half; blk_step = 2; }
  }
  // Row j, or the last one where there are not so many (all lanes take part in the shuffles)
  __device__ __forceinline__ long long in(int j, long long M) const {
    const long long r = row + j * row_step;
    return r < M ? r : M - 1;
  }
};
static long long row_walk_blocks(long long M, int nb, int rows_per_warp = 1) {
  const long long rows = (long long)B8_WARPS * rows_per_warp * (nb == 1 ? 2 : 1);
  return (M + rows - 1) / rows;
}

// ---- quantise, a block per row ---------------------------------------------------------------------------------------------
// A warp takes ROWS rows (or pairs of one-block rows) at a time, and all NV blocks of a half-warp in each are loaded before the first is used: four
// vectors in flight per lane.
template <typename T, int V, int NV, int ROWS>
__global__ void __launch_bounds__(B8_WARPS * 32)
block_quantize_kernel(const T* x, long long ldx, uint8_t* q, long long ldq, float* scale, long long lds, long long M, int K) {
  const int nb = (K + B8 - 1) / B8, sub = threadIdx.x & 15;
  const RowWalk w(nb, ROWS);
  pdl_wait();
  pdl_trigger();
  for (int b0 = 0; b0 < nb; b0 += NV * w.blk_step) {
    Raw8<T> raw[ROWS][NV];
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      const T* xr = x + w.in(j, M) * ldx;
#pragma unroll
      for (int i = 0; i < NV; ++i) raw[j][i] = load_row8<T, V>(xr, (b0 + w.blk + i * w.blk_step) * B8 + sub * 8, K);
    }
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      const long long row = w.in(j, M);
      const bool mine = w.row + j * w.row_step < M;
      const long long room = row + 1 < M ? ldx : K;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int b = b0 + w.blk + i * w.blk_step;
        tail_row8<T, V>(raw[j][i], x + row * ldx, b * B8 + sub * 8, K, room);
        float v[8];
        float m = values_and_max<T>(raw[j][i], v);
        if (__any_sync(0xffffffffu, m > FMAX)) m = finite_half_warp_max(v);
        const float s = block_scale(m);
        if (mine && b < nb) {
          store_q8<V>(q + row * ldq, b * B8 + sub * 8, K, to_e4m3(v, pow2_reciprocal(s)));
          if (sub == 0) scale[row * lds + b] = s;
        }
      }
    }
  }
}

// ---- quantise, a block per 128 x 128 tile ------------------------------------------------------------------------------------
// One CTA per tile, which it holds in registers: 16 lanes x 8 elements = a row of the tile, 32 rows per pass of 512 threads.
constexpr int B8T_THREADS = 512;
template <typename T, int V>
__global__ void __launch_bounds__(B8T_THREADS)
tile_quantize_kernel(const T* x, long long ldx, uint8_t* q, long long ldq, float* scale, long long lds, long long M, int K) {
  __shared__ float red[B8T_THREADS / 32];
  const int nb = (K + B8 - 1) / B8, kb = blockIdx.x % nb;
  const long long mb = blockIdx.x / nb;
  const int c = kb * B8 + (threadIdx.x & 15) * 8;
  const long long r0 = mb * B8 + (threadIdx.x >> 4);
  pdl_wait();
  pdl_trigger();
  Raw8<T> raw[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) raw[i] = load_row8<T, V>(x + (r0 + 32 * i < M ? r0 + 32 * i : M - 1) * ldx, c, r0 + 32 * i < M ? K : 0);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    tail_row8<T, V>(raw[i], x + (r0 + 32 * i < M ? r0 + 32 * i : M - 1) * ldx, c, r0 + 32 * i < M ? K : 0, r0 + 32 * i + 1 < M ? ldx : K);
  float v[4][8];
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    unpack8<T>(raw[i], v[i]);
    m = fmaxf(m, max8(v[i]));
  }
  auto tile_max = [&](float t) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, d));
    __syncthreads();                                               // (the previous use of `red` is over)
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = t;
    __syncthreads();
    t = red[threadIdx.x & (B8T_THREADS / 32 - 1)];
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, d));
    return t;
  };
  m = tile_max(m);
  if (m > FMAX) {                                                  // (the same for the whole CTA)
    m = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      drop_infinities(v[i]);
      m = fmaxf(m, max8(v[i]));
    }
    m = tile_max(m);
  }
  const float s = block_scale(m), inv = pow2_reciprocal(s);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (r0 + 32 * i < M) store_q8<V>(q + (r0 + 32 * i) * ldq, c, K, to_e4m3(v[i], inv));
  if (threadIdx.x == 0) scale[mb * lds + kb] = s;
}

// ---- restore -------------------------------------------------------------------------------------------------------------------
template <typename T, int V, int NV>
__global__ void __launch_bounds__(B8_WARPS * 32)
block_dequantize_kernel(const uint8_t* q, long long ldq, const float* scale, long long lds, T* x, long long ldx, long long M, int K, int row_shift) {
  const int nb = (K + B8 - 1) / B8, sub = threadIdx.x & 15;
  const RowWalk w(nb);
  pdl_wait();
  pdl_trigger();
  if (w.row >= M) return;
  const uint8_t* qr = q + w.row * ldq;
  const float* sr = scale + (w.row >> row_shift) * lds;
  T* xr = x + w.row * ldx;
  const long long room = w.row + 1 < M ? ldq : K;
  for (int b0 = w.blk; b0 < nb; b0 += NV * w.blk_step) {
    uint2 raw[NV];
    float s[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int b = b0 + i * w.blk_step;
      raw[i] = load_q8<V>(qr, b * B8 + sub * 8, K);
      s[i] = b < nb ? sr[b] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) tail_q8<V>(raw[i], qr, (b0 + i * w.blk_step) * B8 + sub * 8, K, room);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int b = b0 + i * w.blk_step;
      float v[8];
      from_e4m3(raw[i], s[i], v);
      if (b < nb) store_row8<T, V>(xr, b * B8 + sub * 8, K, pack8<T>(v));
    }
  }
}

// ---- SwiGLU ----------------------------------------------------------------------------------------------------------------------
// 1 / (1 + e^-g).  fp32: with t = e^-|g|, which never leaves fp32, 1 / (1 + t) or t / (1 + t): the exponential, a reciprocal between 1/2 and 1, a sum and a
// product, 2^-22 + 2^-23 + 2^-23 relative down to fp32's subnormal numbers (us, gradient of M = 9001, F = 2048 / M = 333, F = 1000 both ways: 1 / (1 + e^-g) with a fast
// division, 0 below g = -87.3, 44.4 / 8.0, with an exact one 47.0 / 10.6, this 44.4 / 8.0).  16-bit types: e^-g as 2^(-g log2 e) and the reciprocal on the special-function
// unit, in the forms that flush subnormal numbers (four instructions where the exact treatment of e^-g < 2^-126 and of sums > 2^126 takes fourteen; both
// kernels are bound by instruction issue: M = 65536, F = 2048, bf16 172 -> 164 us, gradient 172 -> 170).  Off by up to |g| 2^-24 relative (the rounding of
// the exponent) beside some 2^-22, far below what the results are rounded to; 0 below g = -87.3, where the sigmoid is below 2^-125.
__device__ __forceinline__ float fast_reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
template <typename T>
__device__ __forceinline__ float sigmoid_of(float g) {
  if constexpr (sizeof(T) == 4) {
    const float t = expf(-fabsf(g)), r = fast_reciprocal(1.f + t);
    return g >= 0.f ? r : t * r;
  } else {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
    return fast_reciprocal(1.f + e);
  }
}

struct SwigluFwd {
  const void* gate; long long ldg; const void* up; long long ldu;
  uint8_t* q[3]; float* s[3];                 // h, gate, up
  long long ldq, lds, M; int F;
};
template <typename T, int V>
__global__ void __launch_bounds__(B8_WARPS * 32, b8_resident<T, V>())
swiglu_block_kernel(const SwigluFwd p) {
  const int nb = (p.F + B8 - 1) / B8, sub = threadIdx.x & 15;
  const RowWalk w(nb);
  pdl_wait();
  pdl_trigger();
  const long long row = w.row < p.M ? w.row : p.M - 1;
  const bool mine = w.row < p.M;
  const T* gr = static_cast<const T*>(p.gate) + row * p.ldg;
  const T* ur = static_cast<const T*>(p.up) + row * p.ldu;
  const long long room_g = row + 1 < p.M ? p.ldg : p.F, room_u = row + 1 < p.M ? p.ldu : p.F;
  // (the next block's vectors are asked for before this one's are worked on)
  Raw8<T> ng = load_row8<T, V>(gr, w.blk * B8 + sub * 8, p.F), nu = load_row8<T, V>(ur, w.blk * B8 + sub * 8, p.F);
  for (int b0 = 0; b0 < nb; b0 += w.blk_step) {
    const int b = b0 + w.blk, c = b * B8 + sub * 8;
    Raw8<T> rg = ng, ru = nu;
    ng = load_row8<T, V>(gr, c + w.blk_step * B8, p.F);
    nu = load_row8<T, V>(ur, c + w.blk_step * B8, p.F);
    tail_row8<T, V>(rg, gr, c, p.F, room_g);
    tail_row8<T, V>(ru, ur, c, p.F, room_u);
    float v[3][8], m[3];
    unpack8<T>(rg, v[1]);
    unpack8<T>(ru, v[2]);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float2 g = make_float2(v[1][i], v[1][i + 1]);
      const float2 h = fmul2(fmul2(g, make_float2(sigmoid_of<T>(g.x), sigmoid_of<T>(g.y))), make_float2(v[2][i], v[2][i + 1]));
      v[0][i] = h.x; v[0][i + 1] = h.y;
    }
    if constexpr (sizeof(T) == 2) {
      const float2 gu = half_warp_max2<T>(rg, ru);
      m[1] = gu.x; m[2] = gu.y;
    } else {
      m[1] = half_warp_max(max8(v[1])); m[2] = half_warp_max(max8(v[2]));
    }
    m[0] = half_warp_max(max8(v[0]));
    if (__any_sync(0xffffffffu, fmaxf(m[0], fmaxf(m[1], m[2])) > FMAX)) {
#pragma unroll
      for (int t = 0; t < 3; ++t) m[t] = finite_half_warp_max(v[t]);
    }
#pragma unroll
    for (int t = 0; t < 3; ++t) {
      const float s = block_scale(m[t]);
      if (mine && b < nb) {
        store_q8<V>(p.q[t] + row * p.ldq, c, p.F, to_e4m3(v[t], pow2_reciprocal(s)));
        if (sub == 0) p.s[t][row * p.lds + b] = s;
      }
    }
  }
}

template <typename T, int V, bool QUANT>
__global__ void __launch_bounds__(B8_WARPS * 32, b8_resident<T, V>(QUANT))
swiglu_block_bwd_kernel(const SwigluBwd p) {
  const int nb = (p.F + B8 - 1) / B8, sub = threadIdx.x & 15;
  const RowWalk w(nb);
  pdl_wait();
  pdl_trigger();
  const long long row = w.row < p.M ? w.row : p.M - 1;
  const bool mine = w.row < p.M, last = row + 1 == p.M;
  const T* dr = static_cast<const T*>(p.dh) + row * p.lddh;
  const uint8_t* gr = p.gq + row * p.ldgq;
  const uint8_t* ur = p.uq + row * p.lduq;
  const float* gsr = p.gs + row * p.ldgs;
  const float* usr = p.us + row * p.ldus;
  // (the next block's vectors and scales are asked for before this one's are worked on)
  Raw8<T> nd;
  uint2 ng, nu;
  float nsg, nsu;
  auto fetch = [&](int b) {
    const int c = b * B8 + sub * 8;
    nd = load_row8<T, V>(dr, c, p.F);
    ng = load_q8<V>(gr, c, p.F);
    nu = load_q8<V>(ur, c, p.F);
    nsg = b < nb ? gsr[b] : 0.f;
    nsu = b < nb ? usr[b] : 0.f;
  };
  fetch(w.blk);
  for (int b0 = 0; b0 < nb; b0 += w.blk_step) {
    const int b = b0 + w.blk, c = b * B8 + sub * 8;
    const bool on = mine && b < nb;
    Raw8<T> rd = nd;
    uint2 qg = ng, qu = nu;
    const float sg = nsg, su = nsu;
    fetch(b + w.blk_step);
    tail_row8<T, V>(rd, dr, c, p.F, last ? p.F : p.lddh);
    tail_q8<V>(qg, gr, c, p.F, last ? p.F : p.ldgq);
    tail_q8<V>(qu, ur, c, p.F, last ? p.F : p.lduq);
    float d[8], g[8], u[8];
    unpack8<T>(rd, d);
    from_e4m3(qg, sg, g);
    from_e4m3(qu, su, u);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float2 gi = make_float2(g[i], g[i + 1]), ui = make_float2(u[i], u[i + 1]);
      const float2 sig = make_float2(sigmoid_of<T>(gi.x), sigmoid_of<T>(gi.y));
      const float2 ds = fmul2(make_float2(d[i], d[i + 1]), sig);
      const float2 one = make_float2(1.f, 1.f);
      const float2 slope = __ffma2_rn(gi, make_float2(1.f - sig.x, 1.f - sig.y), one);            // 1 + g (1 - sigmoid)
      const float2 dg = fmul2(fmul2(ds, ui), slope), du = fmul2(ds, gi);
      g[i] = dg.x; g[i + 1] = dg.y;
      u[i] = du.x; u[i + 1] = du.y;
    }
    const Raw8<T> og = pack8<T>(g), ou = pack8<T>(u);
    if (on) {
      store_row8<T, V>(static_cast<T*>(p.dg) + row * p.lddg, c, p.F, og);
      store_row8<T, V>(static_cast<T*>(p.du) + row * p.lddu, c, p.F, ou);
    }
    if constexpr (QUANT) {                      // from the rounded values, as quantising the outputs would give
      float m[2];
      unpack8<T>(og, g);
      unpack8<T>(ou, u);
      if constexpr (sizeof(T) == 2) {
        const float2 gu = half_warp_max2<T>(og, ou);
        m[0] = gu.x; m[1] = gu.y;
      } else {
        m[0] = half_warp_max(max8(g)); m[1] = half_warp_max(max8(u));
      }
      if (__any_sync(0xffffffffu, fmaxf(m[0], m[1]) > FMAX)) { m[0] = finite_half_warp_max(g); m[1] = finite_half_warp_max(u); }
      const float s0 = block_scale(m[0]), s1 = block_scale(m[1]);
      if (on) {
        store_q8<V>(p.q[0] + row * p.ldq, c, p.F, to_e4m3(g, pow2_reciprocal(s0)));
        store_q8<V>(p.q[1] + row * p.ldq, c, p.F, to_e4m3(u, pow2_reciprocal(s1)));
        if (sub == 0) { p.s[0][row * p.lds + b] = s0; p.s[1][row * p.lds + b] = s1; }
      }
    }
  }
}

// ---- host side ---------------------------------------------------------------------------------------------------------------------
static int elem_size(int dt) { return dt == GSB200_F32 ? 4 : dt == GSB200_F16 || dt == GSB200_BF16 ? 2 : 0; }
// Rows that the 16-byte (E4M3: 8-byte) accesses may take.
static bool wide_rows(const void* p, long long ld, int esz) {
  const long long a = esz == 1 ? 8 : 16;
  return (reinterpret_cast<uintptr_t>(p) % a) == 0 && (ld * esz) % a == 0;
}
static bool elem_aligned(const void* p, int esz) { return (reinterpret_cast<uintptr_t>(p) % esz) == 0; }
static bool grid_fits(long long blocks) { return blocks > 0 && blocks <= 0x7fffffffll; }
#define GSB_BY_V(v, K, T, ...) ((v) == 2 ? K<T, 2, ##__VA_ARGS__> : (v) == 1 ? K<T, 1, ##__VA_ARGS__> : K<T, 0, ##__VA_ARGS__>)
#define GSB_BY_TYPE(dt, CALL)                                   \
  ((dt) == GSB200_F16 ? CALL(__half) : (dt) == GSB200_BF16 ? CALL(__nv_bfloat16) : CALL(float))

int32_t launch_block_quantize(const void* x, int dt, long long ldx, uint8_t* q, long long ldq, float* scale, long long lds, long long M, int K,
                              int block_rows, cudaStream_t st) {
  if (M == 0) return GSB200_OK;
  const int esz = elem_size(dt), nb = K > 0 ? (int)(((long long)K + B8 - 1) / B8) : 0;
  if (!esz || !x || !q || !scale || M < 0 || K <= 0 || ldx < K || ldq < K || lds < nb) return GSB200_ERR_BAD_ARG;
  if (block_rows != 1 && block_rows != B8) return GSB200_ERR_BAD_ARG;
  if (K > (1 << 30) || !elem_aligned(x, esz) || !elem_aligned(scale, 4)) return GSB200_ERR_BAD_ARG;
  const bool aligned = wide_rows(x, ldx, esz) && wide_rows(q, ldq, 1);
  const int v = !aligned ? 0 : K % 8 == 0 ? 2 : 1;
  if (block_rows == B8) {
    const long long blocks = (M + B8 - 1) / B8 * nb;
    if (!grid_fits(blocks)) return GSB200_ERR_BAD_ARG;
#define CALL(T) launch_dependent(GSB_BY_V(v, tile_quantize_kernel, T), (unsigned)blocks, B8T_THREADS, 0, st, \
                                 static_cast<const T*>(x), ldx, q, ldq, scale, lds, M, K)
    return cuda_status(GSB_BY_TYPE(dt, CALL), "block quantise launch");
#undef CALL
  }
  // Several short rows a warp once they fill the SMs all the same (us, one row / several, bf16: M = 65536, K = 128 9.2 / 5.5, K = 512 18.9 / 16.3; M = 333,
  // K = 512 1.4 / 1.9)
  const bool many = M >= 16384;
  const long long blocks = row_walk_blocks(M, nb, !many || nb > 4 ? 1 : nb <= 2 ? 4 : 2);
  if (!grid_fits(blocks)) return GSB200_ERR_BAD_ARG;
#define CALL(T) launch_dependent(nb <= 2 ? (many ? GSB_BY_V(v, block_quantize_kernel, T, 1, 4) : GSB_BY_V(v, block_quantize_kernel, T, 1, 1))   \
                                 : nb <= 4 ? (many ? GSB_BY_V(v, block_quantize_kernel, T, 2, 2) : GSB_BY_V(v, block_quantize_kernel, T, 2, 1)) \
                                           : GSB_BY_V(v, block_quantize_kernel, T, 4, 1),                                                       \
                                 (unsigned)blocks, B8_WARPS * 32, 0, st, static_cast<const T*>(x), ldx, q, ldq, scale, lds, M, K)
  return cuda_status(GSB_BY_TYPE(dt, CALL), "block quantise launch");
#undef CALL
}

int32_t launch_block_dequantize(const uint8_t* q, long long ldq, const float* scale, long long lds, void* x, int dt, long long ldx, long long M,
                                int K, int block_rows, cudaStream_t st) {
  if (M == 0) return GSB200_OK;
  const int esz = elem_size(dt), nb = K > 0 ? (int)(((long long)K + B8 - 1) / B8) : 0;
  if (!esz || !x || !q || !scale || M < 0 || K <= 0 || ldx < K || ldq < K || lds < nb) return GSB200_ERR_BAD_ARG;
  if (block_rows != 1 && block_rows != B8) return GSB200_ERR_BAD_ARG;
  if (K > (1 << 30) || !elem_aligned(x, esz) || !elem_aligned(scale, 4)) return GSB200_ERR_BAD_ARG;
  const long long blocks = row_walk_blocks(M, nb);
  if (!grid_fits(blocks)) return GSB200_ERR_BAD_ARG;
  const bool aligned = wide_rows(x, ldx, esz) && wide_rows(q, ldq, 1);
  const int v = !aligned ? 0 : K % 8 == 0 ? 2 : 1;
  const int shift = block_rows == B8 ? 7 : 0;
#define CALL(T) launch_dependent(nb <= 2 ? GSB_BY_V(v, block_dequantize_kernel, T, 1)  \
                                 : nb <= 4 ? GSB_BY_V(v, block_dequantize_kernel, T, 2) \
                                         : GSB_BY_V(v, block_dequantize_kernel, T, 4), \
                                 (unsigned)blocks, B8_WARPS * 32, 0, st, q, ldq, scale, lds, static_cast<T*>(x), ldx, M, K, shift)
  return cuda_status(GSB_BY_TYPE(dt, CALL), "block restore launch");
#undef CALL
}

int32_t launch_swiglu_block(const void* gate, long long ldg, const void* up, long long ldu, int dt, uint8_t* hq, float* hs, uint8_t* gq, float* gs,
                            uint8_t* uq, float* us, long long ldq, long long lds, long long M, int F, cudaStream_t st) {
  if (M == 0) return GSB200_OK;
  const int esz = elem_size(dt), nb = F > 0 ? (int)(((long long)F + B8 - 1) / B8) : 0;
  if (!esz || !gate || !up || !hq || !hs || !gq || !gs || !uq || !us || M < 0 || F <= 0 || F > (1 << 30)) return GSB200_ERR_BAD_ARG;
  if (ldg < F || ldu < F || ldq < F || lds < nb) return GSB200_ERR_BAD_ARG;
  if (!elem_aligned(gate, esz) || !elem_aligned(up, esz) || !elem_aligned(hs, 4) || !elem_aligned(gs, 4) || !elem_aligned(us, 4)) return GSB200_ERR_BAD_ARG;
  const long long blocks = row_walk_blocks(M, nb);
  if (!grid_fits(blocks)) return GSB200_ERR_BAD_ARG;
  const bool aligned = wide_rows(gate, ldg, esz) && wide_rows(up, ldu, esz) && wide_rows(hq, ldq, 1) && wide_rows(gq, ldq, 1) && wide_rows(uq, ldq, 1);
  const int v = !aligned ? 0 : F % 8 == 0 ? 2 : 1;
  const SwigluFwd p{gate, ldg, up, ldu, {hq, gq, uq}, {hs, gs, us}, ldq, lds, M, F};
#define CALL(T) launch_dependent(GSB_BY_V(v, swiglu_block_kernel, T), (unsigned)blocks, B8_WARPS * 32, 0, st, p)
  return cuda_status(GSB_BY_TYPE(dt, CALL), "SwiGLU launch");
#undef CALL
}

int32_t launch_swiglu_block_bwd(const SwigluBwd& p, int dt, cudaStream_t st) {
  if (p.M == 0) return GSB200_OK;
  const int esz = elem_size(dt), nb = p.F > 0 ? (int)(((long long)p.F + B8 - 1) / B8) : 0;
  if (!esz || !p.dh || !p.gq || !p.gs || !p.uq || !p.us || !p.dg || !p.du || p.M < 0 || p.F <= 0 || p.F > (1 << 30)) return GSB200_ERR_BAD_ARG;
  if (p.lddh < p.F || p.ldgq < p.F || p.lduq < p.F || p.ldgs < nb || p.ldus < nb || p.lddg < p.F || p.lddu < p.F) return GSB200_ERR_BAD_ARG;
  if (!elem_aligned(p.dh, esz) || !elem_aligned(p.dg, esz) || !elem_aligned(p.du, esz) || !elem_aligned(p.gs, 4) || !elem_aligned(p.us, 4)) return GSB200_ERR_BAD_ARG;
  const bool quant = p.q[0] || p.q[1] || p.s[0] || p.s[1];
  if (quant && (!p.q[0] || !p.q[1] || !p.s[0] || !p.s[1] || p.ldq < p.F || p.lds < nb || !elem_aligned(p.s[0], 4) || !elem_aligned(p.s[1], 4))) return GSB200_ERR_BAD_ARG;
  const long long blocks = row_walk_blocks(p.M, nb);
  if (!grid_fits(blocks)) return GSB200_ERR_BAD_ARG;
  const bool aligned = wide_rows(p.dh, p.lddh, esz) && wide_rows(p.gq, p.ldgq, 1) && wide_rows(p.uq, p.lduq, 1) && wide_rows(p.dg, p.lddg, esz) &&
                   wide_rows(p.du, p.lddu, esz) && (!quant || (wide_rows(p.q[0], p.ldq, 1) && wide_rows(p.q[1], p.ldq, 1)));
  const int v = !aligned ? 0 : p.F % 8 == 0 ? 2 : 1;
#define CALL(T) launch_dependent(quant ? GSB_BY_V(v, swiglu_block_bwd_kernel, T, true) : GSB_BY_V(v, swiglu_block_bwd_kernel, T, false), \
                                 (unsigned)blocks, B8_WARPS * 32, 0, st, p)
  return cuda_status(GSB_BY_TYPE(dt, CALL), "SwiGLU gradient launch");
#undef CALL
}

}  // namespace gsb
