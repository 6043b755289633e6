// Weight gradient from an 8-bit activation checkpoint:
//
//   dW[n, k] (+)= sum over m of dY[m, n] x^[m, k],     x^[m, k] = s[m, k / 128] q[m, k]
//
// dY is 16-bit, x^ is restored on chip: E4M3 times a power of two is exact in 16 bits (fp16: inside its range), so nothing is lost
// against a 16-bit copy of the checkpoint that never exists in memory.  (A scale that is no power of two rounds the product to dY's
// type.)  The reduction runs over the rows of both operands, which the tensor core reads "MN-major".
//
// A CTA computes 256 x 256 of dW (two accumulators of 128 rows, all of TMEM) over a range of rows of the batch, 64 rows per step:
//   warp 0      TMA producer: dY, boxes of 64 rows x 64 columns
//   warp 1      MMA issue: 2 x 4 MMAs (M = 128, N = 256, K = 16) per step, 1024 tensor clocks
//   warps 4..11 restore the step's 64 x 256 elements of x^ from global memory into the operand tile; at the end they write dW
// Few tiles are cut over the batch: each part writes its sums to the workspace, and a second launch adds them in order.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <atomic>

#include "capi_internal.h"
#include "ptx.cuh"

namespace gsb {

constexpr int WG_BN = 256, WG_BK = 256, WG_BM = 64;        // columns of dY, columns of x^, rows per step
constexpr int WG_A_BYTES = WG_BM * WG_BN * 2;              // 32 KiB
constexpr int WG_B_BYTES = WG_BM * WG_BK * 2;              // 32 KiB
constexpr int WG_STAGE = WG_A_BYTES + WG_B_BYTES;
constexpr int WG_STAGES = 3;
constexpr int WG_BAR = WG_STAGES * WG_STAGE;
constexpr int WG_BYTES = WG_BAR + 256 + 1024;
constexpr int WG_WARPS = 8, WG_FRONT = 4, WG_THREADS = 32 * (WG_WARPS + WG_FRONT);
constexpr int WG_CHUNK = WG_BM * 128;                      // a 64-column chunk of an operand tile: 64 rows of 128 bytes
static_assert(WG_BYTES <= 227 * 1024, "shared memory budget");

struct WgParams {
  const uint8_t* q; long long ldq; const float* s; long long lds;
  float* out; long long ldo;                               // dW, or this part's sums in the workspace
  long long part_stride;                                   // elements between the parts
  long long M; int N, K, k_tiles, tiles, steps, parts;     // steps of 64 rows in all
  int accumulate;
};

// 16 E4M3 values -> 16 values of T, times s (T's own rounding of the product; exact for a power of two)
template <typename T> __device__ __forceinline__ void restore16(uint4 r, float s, uint4& lo, uint4& hi);
template <>
__device__ __forceinline__ void restore16<__half>(uint4 r, float s, uint4& lo, uint4& hi) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
  uint32_t o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i >> 1] >> (16 * (i & 1))), __NV_E4M3)));
    o[i] = pack_half2(f.x * s, f.y * s);
  }
  lo = make_uint4(o[0], o[1], o[2], o[3]); hi = make_uint4(o[4], o[5], o[6], o[7]);
}
template <>
__device__ __forceinline__ void restore16<__nv_bfloat16>(uint4 r, float s, uint4& lo, uint4& hi) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
  uint32_t o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i >> 1] >> (16 * (i & 1))), __NV_E4M3)));
    const __nv_bfloat162 b = __floats2bfloat162_rn(f.x * s, f.y * s);
    o[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  lo = make_uint4(o[0], o[1], o[2], o[3]); hi = make_uint4(o[4], o[5], o[6], o[7]);
}

template <typename T>
__global__ void __launch_bounds__(WG_THREADS, 1)
wgrad_kernel(const __grid_constant__ CUtensorMap tm_dy, const WgParams p) {
  extern __shared__ uint8_t wg_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(wg_smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_a = reinterpret_cast<uint64_t*>(smem + WG_BAR);
  uint64_t* full_b = full_a + WG_STAGES;
  uint64_t* empty = full_b + WG_STAGES;
  uint64_t* acc_full = empty + WG_STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  const AbortFlag abort_flag{smem_u32(tmem_slot + 1)};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = (int)(blockIdx.x % p.tiles), part = (int)(blockIdx.x / p.tiles);
  const int n0 = tile / p.k_tiles * WG_BN, k0 = tile % p.k_tiles * WG_BK;
  const int step0 = (int)((long long)p.steps * part / p.parts), step1 = (int)((long long)p.steps * (part + 1) / p.parts);
  const bool two = n0 + 128 < p.N;                         // the second accumulator has columns of dY

  if (threadIdx.x == 0) {
    for (int s = 0; s < WG_STAGES; ++s) { mbar_init(&full_a[s], 1); mbar_init(&full_b[s], WG_WARPS); mbar_init(&empty[s], 1); }
    mbar_init(acc_full, 1);
    abort_flag.set(0);
    fence_mbar_init();
    prefetch_tmap(&tm_dy);
  }
  if (warp == 1) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  pdl_wait();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const unsigned int budget = spin_budget();

  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      int s = 0; uint32_t ph = 0;
      for (int i = step0; i < step1; ++i) {
        if (!mbar_wait(&empty[s], ph ^ 1, abort_flag, ST_TIMEOUT_PRODUCER, 0xF00 | s, budget)) { ok = false; break; }
        uint8_t* st = smem + s * WG_STAGE;
        const int chunks = two ? 4 : 2;
        mbar_arrive_expect_tx(&full_a[s], chunks * WG_CHUNK);
        for (int j = 0; j < chunks; ++j) tma_load_2d(st + j * WG_CHUNK, &tm_dy, &full_a[s], n0 + 64 * j, i * WG_BM);
        if (++s == WG_STAGES) { s = 0; ph ^= 1; }
      }
      if (!ok) { const long long t0 = clock64(); while (clock64() - t0 < 2000000) { } }
    }
  } else if (warp == 1) {
    constexpr uint32_t fmt = std::is_same<T, __half>::value ? 0u : 1u;
    constexpr uint32_t idesc = umma_idesc(1, fmt, fmt, 128, WG_BK) | UMMA_A_MN | UMMA_B_MN;
    bool ok = true;
    int s = 0; uint32_t ph = 0;
    for (int i = step0; i < step1; ++i) {
      if (!__all_sync(0xffffffffu, mbar_wait(&full_a[s], ph, abort_flag, ST_TIMEOUT_MMA, 0xF10 | s, budget)) ||
          !__all_sync(0xffffffffu, mbar_wait(&full_b[s], ph, abort_flag, ST_TIMEOUT_MMA, 0xF20 | s, budget))) { ok = false; break; }
      tc_fence_after();
      const uint32_t st = smem_u32(smem + s * WG_STAGE);
      const uint64_t a_desc = umma_smem_desc_mn<128>(st, WG_CHUNK), b_desc = umma_smem_desc_mn<128>(st + WG_A_BYTES, WG_CHUNK);
      constexpr uint64_t step = (16 * 128) >> 4;           // K = 16: 16 rows of 128 bytes
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        umma_f16_elect(tmem_base, a_desc + step * k, b_desc + step * k, idesc, i != step0 || k != 0);
        if (two) umma_f16_elect(tmem_base + 256, a_desc + (2 * WG_CHUNK >> 4) + step * k, b_desc + step * k, idesc, i != step0 || k != 0);
      }
      umma_commit_elect(&empty[s]);
      if (++s == WG_STAGES) { s = 0; ph ^= 1; }
    }
    if (ok) umma_commit_elect(acc_full);
  } else if (warp >= WG_FRONT) {
    // Thread: 16 columns of x^ (two 16-byte pieces of a row of the tile), rows r, r + 16, ... of the step.
    const int tid = threadIdx.x - 32 * WG_FRONT, c = tid & 15, r = tid >> 4;
    const int k = k0 + 16 * c;
    const int have = p.K - k;                              // columns left from k on
    const uint8_t* qk = p.q + k;
    const float* sk = p.s + (k < p.K ? (k >> 7) : 0);
    uint4 raw[4];
    float sc[4];
    auto fetch = [&](int i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const long long m = (long long)i * WG_BM + r + 16 * j;
        raw[j] = make_uint4(0u, 0u, 0u, 0u);
        sc[j] = 0.f;
        if (i < step1 && m < p.M && have > 0) {
          sc[j] = sk[m * p.lds];
          if (have >= 16) raw[j] = *reinterpret_cast<const uint4*>(qk + m * p.ldq);
          else {
            uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int b = 0; b < 15; ++b)
              if (b < have) w[b >> 2] |= (uint32_t)qk[m * p.ldq + b] << (8 * (b & 3));
            raw[j] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
    };
    fetch(step0);
    bool ok = true;
    int s = 0; uint32_t ph = 0;
    for (int i = step0; i < step1; ++i) {
      if (!__all_sync(0xffffffffu, mbar_wait(&empty[s], ph ^ 1, abort_flag, ST_TIMEOUT_EPILOGUE, 0xF30 | s, budget))) { ok = false; break; }
      uint8_t* tile_b = smem + s * WG_STAGE + WG_A_BYTES + (c >> 2) * WG_CHUNK;
      const int swap = (c >> 2) & 1;                       // half of the lanes store their second piece first: no bank conflicts
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint4 lo, hi;
        restore16<T>(raw[j], sc[j], lo, hi);
        const int row = r + 16 * j, pc = 2 * (c & 3);
        uint8_t* line = tile_b + row * 128;
        *reinterpret_cast<uint4*>(line + (((pc + swap) ^ (row & 7)) << 4)) = swap ? hi : lo;
        *reinterpret_cast<uint4*>(line + (((pc + 1 - swap) ^ (row & 7)) << 4)) = swap ? lo : hi;
      }
      fetch(i + 1);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full_b[s]);
      if (++s == WG_STAGES) { s = 0; ph ^= 1; }
    }
    // dW: lane quarter (rows of 32 columns of dY), one accumulator per four warps
    const int q = warp & 3, half = (warp - WG_FRONT) >> 2;
    const int n = n0 + 128 * half + 32 * q + lane;
    const bool any = step1 > step0;                        // (a batch of no rows: all sums are zero)
    if (ok) ok = !any || __all_sync(0xffffffffu, mbar_wait(acc_full, 0, abort_flag, ST_TIMEOUT_EPILOGUE, 0xF40, budget));
    if (ok && (half == 0 || two)) {
      tc_fence_after();
      const uint32_t t = tmem_base + 256 * half + ((uint32_t)(q * 32) << 16);
      float* o = p.out + part * p.part_stride + (long long)n * p.ldo;
      const bool wide = ((reinterpret_cast<uintptr_t>(p.out) | (uintptr_t)(p.ldo * 4) | (uintptr_t)(p.part_stride * 4)) & 31) == 0;
      for (int c0 = 0; c0 < WG_BK && k0 + c0 < p.K; c0 += 32) {
        uint32_t v[32];
        tmem_ld_32x32b_x32(t + c0, v);
        tmem_ld_wait(v);
        if (n >= p.N) continue;
        float* oc = o + k0 + c0;
        if (wide && k0 + c0 + 32 <= p.K) {
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            uint4 x = make_uint4(v[8 * b], v[8 * b + 1], v[8 * b + 2], v[8 * b + 3]), y = make_uint4(v[8 * b + 4], v[8 * b + 5], v[8 * b + 6], v[8 * b + 7]);
            if (p.accumulate) {
              uint4 ox, oy;
              ldg_v8(oc + 8 * b, ox, oy);
              x = make_uint4(__float_as_uint(__uint_as_float(x.x) + __uint_as_float(ox.x)), __float_as_uint(__uint_as_float(x.y) + __uint_as_float(ox.y)),
                             __float_as_uint(__uint_as_float(x.z) + __uint_as_float(ox.z)), __float_as_uint(__uint_as_float(x.w) + __uint_as_float(ox.w)));
              y = make_uint4(__float_as_uint(__uint_as_float(y.x) + __uint_as_float(oy.x)), __float_as_uint(__uint_as_float(y.y) + __uint_as_float(oy.y)),
                             __float_as_uint(__uint_as_float(y.z) + __uint_as_float(oy.z)), __float_as_uint(__uint_as_float(y.w) + __uint_as_float(oy.w)));
            }
            stg_v8(oc + 8 * b, x, y);
          }
        } else {
#pragma unroll
          for (int b = 0; b < 32; ++b)
            if (k0 + c0 + b < p.K) oc[b] = p.accumulate ? oc[b] + __uint_as_float(v[b]) : __uint_as_float(v[b]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem_base, 512); }
}

// dW = (dW +) the parts' sums, in order.
__global__ void wgrad_reduce_kernel(const float* ws, long long ld, long long part_stride, int parts, float* out, long long ldo, int N, int K, int accumulate) {
  const int per_row = (K + 3) / 4;
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  pdl_wait();
  if (i >= (long long)N * per_row) return;
  const int n = (int)(i / per_row), k = (int)(i % per_row) * 4;
  const float* w = ws + (long long)n * ld + k;            // (the workspace's rows are padded to whole vectors)
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int j = 0; j < parts; ++j) {
    const float4 v = *reinterpret_cast<const float4*>(w + j * part_stride);
    a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
  }
  const float e[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (k + j < K) {
      float* o = out + (long long)n * ldo + k + j;
      *o = accumulate ? *o + e[j] : e[j];
    }
}

// Parts the batch is cut into: what fills the SMs with tiles, at least four steps each.  A function of the sizes alone: a workspace
// asked for before a device is chosen fits, and the sums have the same order everywhere.
constexpr int WG_FILL = 148;
static void wgrad_plan(long long M, int N, int K, int& tiles, int& steps, int& parts, long long& ld, long long& part_stride) {
  const int kt = (K + WG_BK - 1) / WG_BK;
  tiles = (N + WG_BN - 1) / WG_BN * kt;
  steps = (int)((M + WG_BM - 1) / WG_BM);
  parts = WG_FILL / tiles;
  if (parts > steps / 4) parts = steps / 4;
  if (parts < 1) parts = 1;
  ld = ((long long)K + 7) / 8 * 8;
  part_stride = ld * N;
}
static bool wgrad_shape_ok(long long M, int N, int K) {
  return M >= 0 && M <= 0x7fffff00ll && N > 0 && K > 0 && N <= (1 << 24) && K <= (1 << 24) &&
         (long long)((N + WG_BN - 1) / WG_BN) * ((K + WG_BK - 1) / WG_BK) <= (1 << 24);
}
int64_t wgrad_workspace_bytes(long long M, int N, int K) {
  if (!wgrad_shape_ok(M, N, K)) return 0;
  int tiles, steps, parts; long long ld, stride;
  wgrad_plan(M, N, K, tiles, steps, parts, ld, stride);
  return parts > 1 ? 4 * stride * parts : 0;
}

int32_t launch_wgrad(const void* dy, int dt, long long lddy, const uint8_t* q, long long ldq, const float* s, long long lds, float* dw, long long lddw,
                     int accumulate, void* ws, long long ws_bytes, long long M, int N, int K, cudaStream_t st) {
  if (!wgrad_shape_ok(M, N, K) || !dw || lddw < K || (reinterpret_cast<uintptr_t>(dw) & 3)) return GSB200_ERR_BAD_ARG;
  if (dt != GSB200_F16 && dt != GSB200_BF16) return GSB200_ERR_BAD_ARG;
  if (M == 0) {                                            // no rows: the gradient is zero
    if (accumulate) return GSB200_OK;
    return cuda_status(cudaMemset2DAsync(dw, (size_t)lddw * 4, 0, (size_t)K * 4, (size_t)N, st), "weight gradient of no rows");
  }
  if (!dy || !q || !s || lddy < N || ldq < K || lds < (K + 127) / 128) return GSB200_ERR_BAD_ARG;
  if (((reinterpret_cast<uintptr_t>(dy) | reinterpret_cast<uintptr_t>(q)) & 15) || lddy % 8 != 0 || ldq % 16 != 0 || (reinterpret_cast<uintptr_t>(s) & 3))
    return GSB200_ERR_BAD_ARG;
  const int32_t rc = ensure_device();
  if (rc != GSB200_OK) return rc;
  WgParams p{};
  long long ld, stride;
  wgrad_plan(M, N, K, p.tiles, p.steps, p.parts, ld, stride);
  const long long need = wgrad_workspace_bytes(M, N, K);
  if (need > 0 && (!ws || ws_bytes < need || (reinterpret_cast<uintptr_t>(ws) & 31))) return GSB200_ERR_BAD_ARG;
  static std::atomic<int> attr_done[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return GSB200_ERR_DEVICE;
  if (!attr_done[dev].load(std::memory_order_acquire)) {
    cudaError_t e = cudaFuncSetAttribute(wgrad_kernel<__half>, cudaFuncAttributeMaxDynamicSharedMemorySize, WG_BYTES);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(wgrad_kernel<__nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize, WG_BYTES);
    if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute(weight gradient)");
    attr_done[dev].store(1, std::memory_order_release);
  }
  CUtensorMap tm;
  if (!tmap_2d(&tm, dt == GSB200_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, dy, (uint64_t)M, (uint64_t)N,
               (uint64_t)lddy, 64, WG_BM, CU_TENSOR_MAP_SWIZZLE_128B)) return GSB200_ERR_BAD_ARG;
  p.q = q; p.ldq = ldq; p.s = s; p.lds = lds; p.M = M; p.N = N; p.K = K; p.k_tiles = (K + WG_BK - 1) / WG_BK;
  const bool cut = p.parts > 1;
  p.out = cut ? static_cast<float*>(ws) : dw; p.ldo = cut ? ld : lddw; p.part_stride = cut ? stride : 0;
  p.accumulate = cut ? 0 : accumulate;
  const long long grid = (long long)p.tiles * p.parts;
  if (grid > 0x7fffffffll) return GSB200_ERR_BAD_ARG;
  cudaError_t e = dt == GSB200_F16 ? launch_dependent(wgrad_kernel<__half>, (unsigned)grid, WG_THREADS, (size_t)WG_BYTES, st, tm, p)
                                   : launch_dependent(wgrad_kernel<__nv_bfloat16>, (unsigned)grid, WG_THREADS, (size_t)WG_BYTES, st, tm, p);
  if (e == cudaSuccess && cut) {
    const long long n4 = (long long)N * ((K + 3) / 4);
    e = launch_dependent(wgrad_reduce_kernel, (unsigned)((n4 + 255) / 256), 256, 0, st, static_cast<const float*>(ws), ld, stride, p.parts, dw, lddw, N, K, accumulate);
  }
  return cuda_status(e, "weight gradient launch");
}

}  // namespace gsb
