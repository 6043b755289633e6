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
// is the conversion, and a restored element is exact in fp32, in bf16, and in fp16 within its range.
//
// All of them are bound by HBM.  A lane owns 8 consecutive elements, so a block is half a warp, and its maximum four shuffles.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "capi_internal.h"
#include "ptx.cuh"

namespace gsb {

constexpr int B8 = 128;                       // elements of a block along a row
constexpr int B8_WARPS = 8;

// ---- 8 consecutive elements ------------------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }

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

// Elements [c, c + 8) of a row of `cols`: in 16-byte pieces where VEC (the row starts on a 16-byte boundary) and all are there,
// one by one otherwise; what lies behind the row reads as zero and is not written.
template <typename T, bool VEC>
__device__ __forceinline__ Raw8<T> load_row8(const T* row, int c, int cols) {
  Raw8<T> r;
  if (VEC && c + 8 <= cols) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) r.w[i] = __ldcs(reinterpret_cast<const uint4*>(row + c) + i);
  } else {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) r.w[i] = make_uint4(0u, 0u, 0u, 0u);
    T* e = reinterpret_cast<T*>(&r);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < cols) e[i] = row[c + i];
  }
  return r;
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_row8(T* row, int c, int cols, const Raw8<T>& r) {
  if (VEC && c + 8 <= cols) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(row + c)[i] = r.w[i];
  } else {
    const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < cols) row[c + i] = e[i];
  }
}
template <bool VEC>
__device__ __forceinline__ uint2 load_q8(const uint8_t* row, int c, int cols) {
  if (VEC && c + 8 <= cols) return __ldcs(reinterpret_cast<const uint2*>(row + c));
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (c + i < cols) w[i >> 2] |= (uint32_t)row[c + i] << (8 * (i & 3));
  return make_uint2(w[0], w[1]);
}
template <bool VEC>
__device__ __forceinline__ void store_q8(uint8_t* row, int c, int cols, uint2 q) {
  if (VEC && c + 8 <= cols) {
    *reinterpret_cast<uint2*>(row + c) = q;
  } else {
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
constexpr float FMAX = 3.402823466e38f;
// Infinities become NaN: they count for no maximum, and the conversion would saturate them.
__device__ __forceinline__ void drop_infinities(float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (fabsf(v[i]) > FMAX) v[i] = __int_as_float(0x7fffffff);
}
// Scale of this lane's block (all 32 lanes take part).
__device__ __forceinline__ float half_warp_scale(float (&v)[8]) {
  float m = half_warp_max(max8(v));
  if (__any_sync(0xffffffffu, m > FMAX)) {                         // rare: an infinity somewhere
    drop_infinities(v);
    m = half_warp_max(max8(v));
  }
  return block_scale(m);
}

// The rows and blocks of a warp.  A warp owns a row and its half-warps every second block of it; where a row is one block, a row per
// half-warp.  Rows are walked from the last to the first, as the other quantisers do (the consumer reads upwards and finds in L2
// what was written last).
struct RowWalk {
  long long row;
  int blk, blk_step;                    // this half-warp's blocks
  __device__ __forceinline__ RowWalk(int nb) {
    const int half = (threadIdx.x >> 4) & 1;
    const long long w = (long long)(gridDim.x - 1 - blockIdx.x) * B8_WARPS + (threadIdx.x >> 5);
    if (nb == 1) { row = 2 * w + half; blk = 0; blk_step = 1; }
    else { row = w; blk = half; blk_step = 2; }
  }
};
static long long row_walk_blocks(long long M, int nb) {
  const long long rows = B8_WARPS * (nb == 1 ? 2 : 1);
  return (M + rows - 1) / rows;
}

// ---- quantise, a block per row ---------------------------------------------------------------------------------------------
// NV blocks of a half-warp are loaded before the first is used.
template <typename T, bool VEC, int NV>
__global__ void __launch_bounds__(B8_WARPS * 32)
block_quantize_kernel(const T* x, long long ldx, uint8_t* q, long long ldq, float* scale, long long lds, long long M, int K) {
  const int nb = (K + B8 - 1) / B8, sub = threadIdx.x & 15;
  const RowWalk w(nb);
  pdl_wait();
  pdl_trigger();
  const long long row = w.row < M ? w.row : M - 1;                 // (all lanes take part in the shuffles)
  const bool mine = w.row < M;
  const T* xr = x + row * ldx;
  uint8_t* qr = q + row * ldq;
  float* sr = scale + row * lds;
  for (int b0 = 0; b0 < nb; b0 += NV * w.blk_step) {
    Raw8<T> raw[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) raw[i] = load_row8<T, VEC>(xr, (b0 + w.blk + i * w.blk_step) * B8 + sub * 8, K);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int b = b0 + w.blk + i * w.blk_step;
      float v[8];
      unpack8<T>(raw[i], v);
      const float s = half_warp_scale(v);
      if (mine && b < nb) {
        store_q8<VEC>(qr, b * B8 + sub * 8, K, to_e4m3(v, pow2_reciprocal(s)));
        if (sub == 0) sr[b] = s;
      }
    }
  }
}

// ---- quantise, a block per 128 x 128 tile ------------------------------------------------------------------------------------
// One CTA per tile, which it holds in registers: 16 lanes x 8 elements = a row of the tile, 32 rows per pass of 512 threads.
constexpr int B8T_THREADS = 512;
template <typename T, bool VEC>
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
  for (int i = 0; i < 4; ++i) raw[i] = load_row8<T, VEC>(x + (r0 + 32 * i < M ? r0 + 32 * i : M - 1) * ldx, c, r0 + 32 * i < M ? K : 0);
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
    if (r0 + 32 * i < M) store_q8<VEC>(q + (r0 + 32 * i) * ldq, c, K, to_e4m3(v[i], inv));
  if (threadIdx.x == 0) scale[mb * lds + kb] = s;
}

// ---- restore -------------------------------------------------------------------------------------------------------------------
template <typename T, bool VEC, int NV>
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
  for (int b0 = w.blk; b0 < nb; b0 += NV * w.blk_step) {
    uint2 raw[NV];
    float s[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int b = b0 + i * w.blk_step;
      raw[i] = load_q8<VEC>(qr, b * B8 + sub * 8, K);
      s[i] = b < nb ? sr[b] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int b = b0 + i * w.blk_step;
      float v[8];
      from_e4m3(raw[i], s[i], v);
      if (b < nb) store_row8<T, VEC>(xr, b * B8 + sub * 8, K, pack8<T>(v));
    }
  }
}

// ---- SwiGLU ----------------------------------------------------------------------------------------------------------------------
// 1 / (1 + e^-g) from the exponential and one division: within a few ulp of fp32 over the whole range (e^-g = inf gives 0).
__device__ __forceinline__ float sigmoid_f32(float g) { return __fdividef(1.f, 1.f + expf(-g)); }

struct SwigluFwd {
  const void* gate; long long ldg; const void* up; long long ldu;
  uint8_t* q[3]; float* s[3];                 // h, gate, up
  long long ldq, lds, M; int F;
};
template <typename T, bool VEC>
__global__ void __launch_bounds__(B8_WARPS * 32)
swiglu_block_kernel(const SwigluFwd p) {
  const int nb = (p.F + B8 - 1) / B8, sub = threadIdx.x & 15;
  const RowWalk w(nb);
  pdl_wait();
  pdl_trigger();
  const long long row = w.row < p.M ? w.row : p.M - 1;
  const bool mine = w.row < p.M;
  const T* gr = static_cast<const T*>(p.gate) + row * p.ldg;
  const T* ur = static_cast<const T*>(p.up) + row * p.ldu;
  for (int b0 = 0; b0 < nb; b0 += w.blk_step) {
    const int b = b0 + w.blk, c = b * B8 + sub * 8;
    const Raw8<T> rg = load_row8<T, VEC>(gr, c, p.F), ru = load_row8<T, VEC>(ur, c, p.F);
    float v[3][8];
    unpack8<T>(rg, v[1]);
    unpack8<T>(ru, v[2]);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[0][i] = v[1][i] * sigmoid_f32(v[1][i]) * v[2][i];
#pragma unroll
    for (int t = 0; t < 3; ++t) {
      const float s = half_warp_scale(v[t]);
      if (mine && b < nb) {
        store_q8<VEC>(p.q[t] + row * p.ldq, c, p.F, to_e4m3(v[t], pow2_reciprocal(s)));
        if (sub == 0) p.s[t][row * p.lds + b] = s;
      }
    }
  }
}

template <typename T, bool VEC, bool QUANT>
__global__ void __launch_bounds__(B8_WARPS * 32)
swiglu_block_bwd_kernel(const SwigluBwd p) {
  const int nb = (p.F + B8 - 1) / B8, sub = threadIdx.x & 15;
  const RowWalk w(nb);
  pdl_wait();
  pdl_trigger();
  const long long row = w.row < p.M ? w.row : p.M - 1;
  const bool mine = w.row < p.M;
  for (int b0 = 0; b0 < nb; b0 += w.blk_step) {
    const int b = b0 + w.blk, c = b * B8 + sub * 8;
    const bool on = mine && b < nb;
    const Raw8<T> rd = load_row8<T, VEC>(static_cast<const T*>(p.dh) + row * p.lddh, c, p.F);
    const uint2 qg = load_q8<VEC>(p.gq + row * p.ldgq, c, p.F), qu = load_q8<VEC>(p.uq + row * p.lduq, c, p.F);
    const float sg = b < nb ? p.gs[row * p.ldgs + b] : 0.f, su = b < nb ? p.us[row * p.ldus + b] : 0.f;
    float d[8], g[8], u[8];
    unpack8<T>(rd, d);
    from_e4m3(qg, sg, g);
    from_e4m3(qu, su, u);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float sig = sigmoid_f32(g[i]), ds = d[i] * sig;
      const float dg = ds * u[i] * (1.f + g[i] * (1.f - sig));
      u[i] = ds * g[i];
      g[i] = dg;
    }
    const Raw8<T> og = pack8<T>(g), ou = pack8<T>(u);
    if (on) {
      store_row8<T, VEC>(static_cast<T*>(p.dg) + row * p.lddg, c, p.F, og);
      store_row8<T, VEC>(static_cast<T*>(p.du) + row * p.lddu, c, p.F, ou);
    }
    if constexpr (QUANT) {                      // from the rounded values, as quantising the outputs would give
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float v[8];
        unpack8<T>(t == 0 ? og : ou, v);
        const float s = half_warp_scale(v);
        if (on) {
          store_q8<VEC>(p.q[t] + row * p.ldq, c, p.F, to_e4m3(v, pow2_reciprocal(s)));
          if (sub == 0) p.s[t][row * p.lds + b] = s;
        }
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
#define GSB_BY_TYPE(dt, CALL)                                   \
  ((dt) == GSB200_F16 ? CALL(__half) : (dt) == GSB200_BF16 ? CALL(__nv_bfloat16) : CALL(float))

int32_t launch_block_quantize(const void* x, int dt, long long ldx, uint8_t* q, long long ldq, float* scale, long long lds, long long M, int K,
                              int block_rows, cudaStream_t st) {
  if (M == 0) return GSB200_OK;
  const int esz = elem_size(dt), nb = K > 0 ? (int)(((long long)K + B8 - 1) / B8) : 0;
  if (!esz || !x || !q || !scale || M < 0 || K <= 0 || ldx < K || ldq < K || lds < nb) return GSB200_ERR_BAD_ARG;
  if (block_rows != 1 && block_rows != B8) return GSB200_ERR_BAD_ARG;
  if (K > (1 << 30) || !elem_aligned(x, esz) || !elem_aligned(scale, 4)) return GSB200_ERR_BAD_ARG;
  const bool vec = wide_rows(x, ldx, esz) && wide_rows(q, ldq, 1);
  if (block_rows == B8) {
    const long long blocks = (M + B8 - 1) / B8 * nb;
    if (!grid_fits(blocks)) return GSB200_ERR_BAD_ARG;
#define CALL(T) launch_dependent(vec ? tile_quantize_kernel<T, true> : tile_quantize_kernel<T, false>, (unsigned)blocks, B8T_THREADS, 0, st, \
                                 static_cast<const T*>(x), ldx, q, ldq, scale, lds, M, K)
    return cuda_status(GSB_BY_TYPE(dt, CALL), "block quantise launch");
#undef CALL
  }
  const long long blocks = row_walk_blocks(M, nb);
  if (!grid_fits(blocks)) return GSB200_ERR_BAD_ARG;
#define CALL(T) launch_dependent(nb <= 2 ? (vec ? block_quantize_kernel<T, true, 1> : block_quantize_kernel<T, false, 1>)      \
                                 : nb <= 4 ? (vec ? block_quantize_kernel<T, true, 2> : block_quantize_kernel<T, false, 2>)    \
                                           : (vec ? block_quantize_kernel<T, true, 4> : block_quantize_kernel<T, false, 4>),   \
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
  const bool vec = wide_rows(x, ldx, esz) && wide_rows(q, ldq, 1);
  const int shift = block_rows == B8 ? 7 : 0;
#define CALL(T) launch_dependent(nb <= 2 ? (vec ? block_dequantize_kernel<T, true, 1> : block_dequantize_kernel<T, false, 1>)  \
                                         : (vec ? block_dequantize_kernel<T, true, 4> : block_dequantize_kernel<T, false, 4>), \
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
  const bool vec = wide_rows(gate, ldg, esz) && wide_rows(up, ldu, esz) && wide_rows(hq, ldq, 1) && wide_rows(gq, ldq, 1) && wide_rows(uq, ldq, 1);
  const SwigluFwd p{gate, ldg, up, ldu, {hq, gq, uq}, {hs, gs, us}, ldq, lds, M, F};
#define CALL(T) launch_dependent(vec ? swiglu_block_kernel<T, true> : swiglu_block_kernel<T, false>, (unsigned)blocks, B8_WARPS * 32, 0, st, p)
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
  const bool vec = wide_rows(p.dh, p.lddh, esz) && wide_rows(p.gq, p.ldgq, 1) && wide_rows(p.uq, p.lduq, 1) && wide_rows(p.dg, p.lddg, esz) &&
                   wide_rows(p.du, p.lddu, esz) && (!quant || (wide_rows(p.q[0], p.ldq, 1) && wide_rows(p.q[1], p.ldq, 1)));
#define CALL(T) launch_dependent(vec ? (quant ? swiglu_block_bwd_kernel<T, true, true> : swiglu_block_bwd_kernel<T, true, false>)          \
                                     : (quant ? swiglu_block_bwd_kernel<T, false, true> : swiglu_block_bwd_kernel<T, false, false>),       \
                                 (unsigned)blocks, B8_WARPS * 32, 0, st, p)
  return cuda_status(GSB_BY_TYPE(dt, CALL), "SwiGLU gradient launch");
#undef CALL
}

}  // namespace gsb
