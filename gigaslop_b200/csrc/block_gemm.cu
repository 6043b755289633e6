// FP8 GEMM with one fp32 scale per block of 128 along the reduction:
//
//   C[m, n] = sum over b of  sa[m, b] sb[n / 128, b]  (sum over k in block b of A[m, k] B[n, k])
//
// A holds activations or gradients (a scale per row and block), B a weight (a scale per 128 x 128 tile), [N, K] or, for the
// input gradient, [K, N] as the forward pass has it (its rows are then the reduction; the tensor core reads it "MN-major").
//
// The scales change along the reduction, so the tensor core cannot carry a sum over a whole row: each 128-wide K block is multiplied into a
// tensor-memory stage of its own (four MMAs of K = 32 that start from zero), and the epilogue warps add it, times its scale, to fp32 sums
// in registers: one fused multiply-add per element and K block, since a thread holds one row and 128 columns that share a B scale.
// Tile 128 rows x 256 columns: per K block 512 tensor clocks, and for the eight epilogue warps 256 clocks of multiply-adds and as many
// of tensor-memory reads.  Two stages of 256 TMEM columns let both sides run at once.
//   warp 0      TMA producer (one lane)       warp 1   MMA issue (converged, one elected lane)
//   warps 4..11 epilogue: lane quarter e % 4, column half e / 4
#include <atomic>

#include "capi_internal.h"
#include "ptx.cuh"

namespace gsb {

constexpr int BG_BM = 128, BG_BK = 128;
constexpr int BG_EPI_WARPS = 8, BG_FRONT_WARPS = 4;
constexpr int BG_THREADS = 32 * (BG_EPI_WARPS + BG_FRONT_WARPS);
constexpr int BG_A_BYTES = BG_BM * BG_BK;                  // 16 KiB
constexpr int BG_STAGES = 4;
constexpr int BG_OUT_BUF = 4096;                           // per epilogue warp: 32 rows of 128 bytes

template <int BN>
struct BgSmem {
  static constexpr int STAGE = BG_A_BYTES + BN * BG_BK;
  static constexpr int OUT = BG_STAGES * STAGE;
  static constexpr int BAR = OUT + BG_EPI_WARPS * BG_OUT_BUF;
  static constexpr int BYTES = BAR + 256 + 1024;
  static_assert(BYTES <= 227 * 1024, "shared memory budget");
};

struct BgParams {
  int M, N, m_blocks, n_blocks, k_blocks;
  const float* sa; long long ld_sa;
  const float* sb; long long ld_sb_n, ld_sb_k;             // B scale of (column block, K block): sb[cb * ld_sb_n + kb * ld_sb_k]
  void* C; long long ldc; int c_type;
  int n_tma;                                               // the columns before it leave through TMA boxes, the others element by element
};

// KN: B is [K, N].  Its stage holds boxes of 128 K rows x 128 columns.
template <int BN, bool KN>
__global__ void __launch_bounds__(BG_THREADS, 1)
block_gemm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const __grid_constant__ CUtensorMap tm_c,
                  const BgParams p) {
  extern __shared__ uint8_t bg_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(bg_smem_raw) + 1023) & ~uintptr_t(1023));
  using L = BgSmem<BN>;
  constexpr int ACC = 512 / BN > 4 ? 4 : 512 / BN;         // accumulator stages
  constexpr int CW = BN / 2;                               // columns of an epilogue warp
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BAR);
  uint64_t* empty = full + BG_STAGES;
  uint64_t* acc_full = empty + BG_STAGES;
  uint64_t* acc_empty = acc_full + ACC;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + ACC);
  const AbortFlag abort_flag{smem_u32(tmem_slot + 1)};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int num_tiles = p.m_blocks * p.n_blocks;           // (the host keeps this below 2^31)

  if (threadIdx.x == 0) {
    for (int s = 0; s < BG_STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int s = 0; s < ACC; ++s) { mbar_init(&acc_full[s], 1); mbar_init(&acc_empty[s], BG_EPI_WARPS); }
    abort_flag.set(0);
    fence_mbar_init();
    prefetch_tmap(&tm_a); prefetch_tmap(&tm_b); prefetch_tmap(&tm_c);
  }
  if (warp == 1) { tmem_alloc(tmem_slot, ACC * BN); tmem_relinquish(); }
  pdl_wait();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const unsigned int budget = spin_budget();

  if (warp < BG_FRONT_WARPS) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0) {
      if (lane == 0) {
        bool ok = true;
        int s = 0; uint32_t ph = 0;
        for (int t = blockIdx.x; ok && t < num_tiles; t += gridDim.x) {
          const int m0 = t / p.n_blocks * BG_BM, n0 = t % p.n_blocks * BN;
          for (int kb = 0; kb < p.k_blocks; ++kb) {
            if (!mbar_wait(&empty[s], ph ^ 1, abort_flag, ST_TIMEOUT_PRODUCER, 0xE00 | s, budget)) { ok = false; break; }
            uint8_t* st = smem + s * L::STAGE;
            mbar_arrive_expect_tx(&full[s], L::STAGE);
            tma_load_2d(st, &tm_a, &full[s], kb * BG_BK, m0);
            if constexpr (KN) {
#pragma unroll
              for (int j = 0; j < (BN + 127) / 128; ++j) tma_load_2d(st + BG_A_BYTES + j * 128 * BG_BK, &tm_b, &full[s], n0 + 128 * j, kb * BG_BK);
            } else {
              tma_load_2d(st + BG_A_BYTES, &tm_b, &full[s], kb * BG_BK, n0);
            }
            if (++s == BG_STAGES) { s = 0; ph ^= 1; }
          }
        }
        if (!ok) { const long long t0 = clock64(); while (clock64() - t0 < 2000000) { } }     // loads in flight land before the CTA exits
      }
    } else if (warp == 1) {
      constexpr uint32_t idesc = umma_idesc(1, 0, 0, BG_BM, BN) | (KN ? UMMA_B_MN : 0u);
      bool ok = true;
      int s = 0, as = 0; uint32_t ph = 0, aph = 0;
      for (int t = blockIdx.x; ok && t < num_tiles; t += gridDim.x) {
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!__all_sync(0xffffffffu, mbar_wait(&acc_empty[as], aph ^ 1, abort_flag, ST_TIMEOUT_MMA, 0xE10 | as, budget)) ||
              !__all_sync(0xffffffffu, mbar_wait(&full[s], ph, abort_flag, ST_TIMEOUT_MMA, 0xE20 | s, budget))) { ok = false; break; }
          tc_fence_after();
          const uint32_t st = smem_u32(smem + s * L::STAGE);
          const uint64_t a_desc = umma_smem_desc_sw128(st);
          const uint64_t b_desc = KN ? umma_smem_desc_mn(st + BG_A_BYTES, 128 * BG_BK) : umma_smem_desc_sw128(st + BG_A_BYTES);
          constexpr uint64_t b_step = KN ? (32 * 128) >> 4 : 2;           // K = 32: 32 rows of 128 bytes, or 32 bytes of a row
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_f8_elect(tmem_base + as * BN, a_desc + 2 * k, b_desc + b_step * k, idesc, k != 0);
          umma_commit_elect(&empty[s]);
          umma_commit_elect(&acc_full[as]);
          if (++s == BG_STAGES) { s = 0; ph ^= 1; }
          if (++as == ACC) { as = 0; aph ^= 1; }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int e = warp - BG_FRONT_WARPS, q = warp & 3, half = e >> 2;
    uint8_t* const out_buf = smem + L::OUT + e * BG_OUT_BUF;
    const uint32_t t_lane = tmem_base + ((uint32_t)(q * 32) << 16) + half * CW;
    bool ok = true;
    int as = 0; uint32_t aph = 0;
    for (int t = blockIdx.x; ok && t < num_tiles; t += gridDim.x) {
      const int m0 = t / p.n_blocks * BG_BM + q * 32, n0 = t % p.n_blocks * BN + half * CW;
      const int row = m0 + lane;
      const bool live = m0 < p.M && n0 < p.N;                // (uniform) this warp has something to write
      const float* sa = p.sa + (long long)(row < p.M ? row : p.M - 1) * p.ld_sa;
      const float* sb = p.sb + (long long)((n0 < p.N ? n0 : 0) >> 7) * p.ld_sb_n;
      float acc[CW];
#pragma unroll
      for (int i = 0; i < CW; ++i) acc[i] = 0.f;
      float na = sa[0], nb = sb[0];                          // the next K block's scales
      for (int kb = 0; kb < p.k_blocks; ++kb) {
        const float sc = na * nb;
        if (kb + 1 < p.k_blocks) { na = sa[kb + 1]; nb = sb[(long long)(kb + 1) * p.ld_sb_k]; }
        if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[as], aph, abort_flag, ST_TIMEOUT_EPILOGUE, 0xE30 | as, budget))) { ok = false; break; }
        tc_fence_after();
        if (live) {
          const uint32_t ta = t_lane + as * BN;
          const float2 s2 = pk2(sc, sc);
          constexpr int NC = CW / 32;
          uint32_t v[2][32];
          tmem_ld_32x32b_x32(ta, v[0]);
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            tmem_ld_wait(v[c & 1]);
            if (c + 1 < NC) tmem_ld_32x32b_x32(ta + 32 * (c + 1), v[(c + 1) & 1]);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 r = __ffma2_rn(pk2(__uint_as_float(v[c & 1][2 * i]), __uint_as_float(v[c & 1][2 * i + 1])), s2,
                                          pk2(acc[32 * c + 2 * i], acc[32 * c + 2 * i + 1]));
              acc[32 * c + 2 * i] = r.x; acc[32 * c + 2 * i + 1] = r.y;
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[as]);
        if (++as == ACC) { as = 0; aph ^= 1; }
      }
      if (!ok || !live) continue;
      // 32 columns at a time.  Boxes of 32 rows x 128 bytes (32 columns of fp32, 64 of 16 bits) in the 128-byte swizzle.
      const bool f32 = p.c_type == GSB200_F32;
#pragma unroll
      for (int b = 0; b < CW / 32; ++b) {
        const int n = n0 + 32 * b, box = f32 ? n : n0 + 32 * (b & ~1);
        if (n >= p.N) break;
        if (box >= p.n_tma) {
          if (row < p.M) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              if (n + i >= p.N) continue;
              const long long o = (long long)row * p.ldc + n + i;
              const float v = acc[32 * b + i];
              if (f32) static_cast<float*>(p.C)[o] = v;
              else if (p.c_type == GSB200_F16) static_cast<__half*>(p.C)[o] = __float2half_rn(v);
              else static_cast<__nv_bfloat16*>(p.C)[o] = __float2bfloat16_rn(v);
            }
          }
          continue;
        }
        if (f32 || (b & 1) == 0) {
          if (lane == 0) tma_store_wait_read<0>();           // the previous box has left the buffer
          __syncwarp();
        }
        if (f32) {
#pragma unroll
          for (int pc = 0; pc < 8; ++pc)
            *reinterpret_cast<float4*>(out_buf + lane * 128 + ((pc ^ (lane & 7)) << 4)) =
                make_float4(acc[32 * b + 4 * pc], acc[32 * b + 4 * pc + 1], acc[32 * b + 4 * pc + 2], acc[32 * b + 4 * pc + 3]);
        } else {
#pragma unroll
          for (int pc = 0; pc < 4; ++pc) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float lo = acc[32 * b + 8 * pc + 2 * j], hi = acc[32 * b + 8 * pc + 2 * j + 1];
              if (p.c_type == GSB200_F16) w[j] = pack_half2(lo, hi);
              else { const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi); w[j] = *reinterpret_cast<const uint32_t*>(&h); }
            }
            *reinterpret_cast<uint4*>(out_buf + lane * 128 + (((4 * (b & 1) + pc) ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        if (f32 || (b & 1) == 1 || n + 32 >= p.N || b + 1 == CW / 32) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) { tma_store_2d(&tm_c, out_buf, box, m0); tma_store_commit(); }
        }
      }
    }
    if (lane == 0) tma_store_wait_all<0>();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem_base, ACC * BN); }
}

template <int BN, bool KN>
static cudaError_t launch_bg(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, const BgParams& p, int dev, cudaStream_t st) {
  static std::atomic<int> attr_done[64];
  auto k = block_gemm_kernel<BN, KN>;
  if (!attr_done[dev].load(std::memory_order_acquire)) {
    // the re-split of the registers waits until the block's own pool covers it
    cudaFuncAttributes fa{};
    cudaError_t e = cudaFuncGetAttributes(&fa, k);
    if (e == cudaSuccess && fa.numRegs * BG_THREADS < 32 * (BG_FRONT_WARPS * 56 + BG_EPI_WARPS * 224)) e = cudaErrorInvalidConfiguration;
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, BgSmem<BN>::BYTES);
    if (e != cudaSuccess) return e;
    attr_done[dev].store(1, std::memory_order_release);
  }
  const long long tiles = (long long)p.m_blocks * p.n_blocks;
  const int grid = (int)(tiles < sm_count() ? tiles : sm_count());
  return launch_dependent(k, (unsigned)grid, BG_THREADS, (size_t)BgSmem<BN>::BYTES, st, ta, tb, tc, p);
}

int32_t launch_block_gemm(const uint8_t* A, long long lda, const float* sa, long long ld_sa, const uint8_t* B, long long ldb, const float* sb,
                          long long ld_sb, void* C, long long ldc, int c_type, long long M, int N, int K, int flags, cudaStream_t st) {
  if (M == 0) return GSB200_OK;
  if (M < 0 || M > 0x7fffff00ll || N <= 0 || K <= 0 || N > (1 << 30) || K > (1 << 30)) return GSB200_ERR_BAD_ARG;
  if (flags & ~GSB200_FLAG_B_KN) return GSB200_ERR_BAD_ARG;
  const bool kn = (flags & GSB200_FLAG_B_KN) != 0;
  const int nb = (N + 127) / 128, kb = (K + 127) / 128;
  const int esz = c_type == GSB200_F32 ? 4 : c_type == GSB200_F16 || c_type == GSB200_BF16 ? 2 : 0;
  if (!A || !sa || !B || !sb || !C || !esz) return GSB200_ERR_BAD_ARG;
  if (((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(B)) & 15) || lda % 16 != 0 || ldb % 16 != 0) return GSB200_ERR_BAD_ARG;
  if (lda < K || ldb < (kn ? N : K) || ldc < N || ld_sa < kb || ld_sb < (kn ? nb : kb)) return GSB200_ERR_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(sa) & 3) || (reinterpret_cast<uintptr_t>(sb) & 3) || (reinterpret_cast<uintptr_t>(C) & (esz - 1))) return GSB200_ERR_BAD_ARG;
  const int32_t rc = ensure_device();
  if (rc != GSB200_OK) return rc;
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return GSB200_ERR_DEVICE;
  constexpr int BN = 256;
  BgParams p{};
  p.M = (int)M; p.N = N; p.m_blocks = (int)((M + BG_BM - 1) / BG_BM); p.n_blocks = (N + BN - 1) / BN; p.k_blocks = kb;
  if ((long long)p.m_blocks * p.n_blocks > 0x7fffffffll) return GSB200_ERR_BAD_ARG;
  p.sa = sa; p.ld_sa = ld_sa; p.sb = sb; p.ld_sb_n = kn ? 1 : ld_sb; p.ld_sb_k = kn ? ld_sb : 1;
  p.C = C; p.ldc = ldc; p.c_type = c_type;
  // TMA writes whole 16-byte pieces: where a row of C ends inside one, the last box goes element by element
  const bool tma_out = (reinterpret_cast<uintptr_t>(C) & 15) == 0 && (ldc * esz) % 16 == 0;
  p.n_tma = !tma_out ? 0 : (N * esz) % 16 == 0 ? N : N / (128 / esz) * (128 / esz);
  const CUtensorMapDataType u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  const CUtensorMapDataType ct = c_type == GSB200_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                               : c_type == GSB200_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUtensorMap ta, tb, tc;
  if (!tmap_2d(&ta, u8, 1, A, (uint64_t)M, (uint64_t)K, (uint64_t)lda, BG_BK, BG_BM, CU_TENSOR_MAP_SWIZZLE_128B)) return GSB200_ERR_BAD_ARG;
  if (kn ? !tmap_2d(&tb, u8, 1, B, (uint64_t)K, (uint64_t)N, (uint64_t)ldb, 128, BG_BK, CU_TENSOR_MAP_SWIZZLE_128B)
         : !tmap_2d(&tb, u8, 1, B, (uint64_t)N, (uint64_t)K, (uint64_t)ldb, BG_BK, BN, CU_TENSOR_MAP_SWIZZLE_128B)) return GSB200_ERR_BAD_ARG;
  if (p.n_tma == 0) tc = ta;
  else if (!tmap_2d(&tc, ct, esz, C, (uint64_t)M, (uint64_t)N, (uint64_t)ldc, 128 / esz, 32, CU_TENSOR_MAP_SWIZZLE_128B)) return GSB200_ERR_BAD_ARG;
  return cuda_status(kn ? launch_bg<BN, true>(ta, tb, tc, p, dev, st) : launch_bg<BN, false>(ta, tb, tc, p, dev, st), "block-scaled gemm launch");
}

}  // namespace gsb
