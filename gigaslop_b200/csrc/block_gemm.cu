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
//
// Four forms: up to four rows on plain fp32 (block_gemv_kernel), few tiles of 128 rows x 32 to 128 columns (block_gemm_small_kernel), and CTA pairs
// with tiles of 256 or 128 columns (block_gemm_kernel), which this is about:
// Tile 256 rows x 256 columns, 128 x 256 per CTA (cta_group::2), two tensor-memory stages of 256 columns (or four of 128).
//   warp 0      TMA producer (one lane); a CTA loads its 128 rows of A and half of the tile's B, 32 KiB per K block
//   warp 1      MMA issue (first CTA of the pair; converged, one elected lane)
//   warps 2, 3  products of the scales, loaded four K blocks ahead, through shared memory
//   warps 4..11 epilogue: lane quarter e % 4, column half e / 4
// A K block takes about 850 clocks where its MMAs take 512.  The round trip of a stage, two of which are all that tensor memory holds, accounts for that: MMAs
// (512 clocks and about 230 until the last one shows), the epilogue's wake-up, four reads of 32 columns (300), the return to the MMA warp (230), 1700
// clocks for two K blocks.  But it is not shown to be the only bound: tiles of 128 columns have four stages and half the MMAs, and still take some 600 clocks a K
// block (0.69 of a wide tile's time, below), in which a CTA loads the same 40 bytes a clock; the operands' feed or a fixed cost per K block in the epilogue would explain
// both.  Out of the stage's chain are the scales (their address arithmetic,
// loads and products), the wait for the operands (before that for the stage), the multiply-adds of a chunk (behind the read of the next one,
// the last ones behind the release).  us, M = 65536, N = 1536, K = 512 / N = 512, K = 2048: single CTAs with 256 columns that load their own scales
// 91 / 80; pairs 95 / 80; scales through shared memory 78 / 76; two staging boxes per warp instead of one 72 / 74, filled before one fence 70 / 72.
// Tried and dropped: results straight from registers in 32-byte sectors (92 / 78).
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <atomic>

#include "capi_internal.h"
#include "ptx.cuh"

namespace gsb {

constexpr int BG_BM = 128, BG_BK = 128;
constexpr int BG_EPI_WARPS = 8, BG_FRONT_WARPS = 4;
constexpr int BG_FRONT_REGS = 56, BG_EPI_REGS = 224;
constexpr int BG_THREADS = 32 * (BG_EPI_WARPS + BG_FRONT_WARPS);
constexpr int BG_A_BYTES = BG_BM * BG_BK;                  // 16 KiB
constexpr int BG_OUT_BUF = 2 * 4096;                       // per epilogue warp: two boxes of 32 rows x 128 bytes
// The large form with tiles of BN columns
template <int BN>
struct BgSmem {
  static constexpr int ACC = 512 / BN;                     // tensor-memory stages
  static constexpr int STAGE = BG_A_BYTES + BN / 2 * BG_BK;               // a CTA of the pair holds half of the tile's columns: 32 or 24 KiB
  static constexpr int STAGES = BN == 256 ? 4 : 6;
  static constexpr int SC = 2 * ACC;                       // K blocks of scales in shared memory
  static constexpr int OUT = STAGES * STAGE;
  static constexpr int SCALES = OUT + BG_EPI_WARPS * BG_OUT_BUF;          // [SC][2][BG_BM] products of the scales
  static constexpr int BAR = SCALES + SC * 2 * BG_BM * 4;
  static constexpr int BYTES = BAR + 256 + 1024;
  static_assert(BYTES <= 227 * 1024 && (2 * STAGES + 2 * ACC + SC) * 8 + 8 <= 256, "shared memory budget");
};

__device__ __forceinline__ uint32_t pack_bf2(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Two E4M3 values (the low 16 bits) as fp32
__device__ __forceinline__ float2 e4m3x2_f32(uint32_t w) {
  return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)w, __NV_E4M3)));
}

// Rows of C that no wide store may take: a warp's 32 rows of up to 128 bytes go through its 4 KiB box of shared memory, so that a store
// covers one row's neighbours instead of a column of 32 rows (us, contiguous rows of fp16, element by element / so: M = 65536, N = 1535, K = 512 979 / 131; M = 371,
// N = 3287, K = 640 23.1 / 6.1).  pieces(pc): 16-byte piece pc of this lane's row, NP of them.
template <typename E, int NP, typename P>
__device__ __forceinline__ void store_by_rows(uint8_t* box, int lane, P pieces, E* c, long long ldc, int rows, int cols) {
  __syncwarp();
#pragma unroll
  for (int pc = 0; pc < NP; ++pc) *reinterpret_cast<uint4*>(box + lane * 128 + ((pc ^ (lane & 7)) << 4)) = pieces(pc);
  __syncwarp();
#pragma unroll 4
  for (int r = 0; r < rows; ++r) {
#pragma unroll
    for (int x = lane; x < NP * 16 / (int)sizeof(E); x += 32) {
      const int b = x * (int)sizeof(E);
      if (x < cols) c[r * ldc + x] = *reinterpret_cast<const E*>(box + r * 128 + (((b >> 4) ^ (r & 7)) << 4) + (b & 15));
    }
  }
}

struct BgParams {
  int M, N, m_blocks, n_blocks, k_blocks;                  // a pair's row block is 256 rows, 128 per CTA
  const float* sa; long long ld_sa;
  const float* sb; long long ld_sb_n, ld_sb_k;             // B scale of (column block, K block): sb[cb * ld_sb_n + kb * ld_sb_k]
  void* C; long long ldc; int c_type;
  int a_rows;                                              // few-tile form: rows of the boxes of A
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
  constexpr int ACC = L::ACC, STAGES = L::STAGES, SC = L::SC;
  constexpr int CW = BN / 2;                               // columns of an epilogue warp
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BAR);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint64_t* acc_empty = acc_full + ACC;
  uint64_t* sc_empty = acc_empty + ACC;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sc_empty + SC);
  float* sc_smem = reinterpret_cast<float*>(smem + L::SCALES);
  const AbortFlag abort_flag{smem_u32(tmem_slot + 1)};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int num_tiles = p.m_blocks * p.n_blocks;           // (the host keeps this below 2^31)
  const int rank = (int)cluster_ctarank();      // the pair's first CTA issues the MMAs; its barriers collect both CTAs' loads and releases
  const int unit = (int)(blockIdx.x >> 1), units = (int)(gridDim.x >> 1);
  auto tile_row = [&](int t) { return t / p.n_blocks * 2 * BG_BM + rank * BG_BM; };      // this CTA's first row
  auto tile_col = [&](int t) { return t % p.n_blocks * BN; };

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int s = 0; s < ACC; ++s) { mbar_init(&acc_full[s], 1 + 2); mbar_init(&acc_empty[s], 2 * BG_EPI_WARPS); }
    for (int s = 0; s < SC; ++s) mbar_init(&sc_empty[s], BG_EPI_WARPS);
    abort_flag.set(0);
    fence_mbar_init();
    prefetch_tmap(&tm_a); prefetch_tmap(&tm_b); prefetch_tmap(&tm_c);
  }
  if (warp == 1) { tmem_alloc_pair(tmem_slot, ACC * BN); tmem_relinquish_pair(); }
  pdl_wait();
  tc_fence_before();
  cluster_sync_all();                                      // (a __syncthreads of both CTAs) the other's barriers are initialised before anything arrives at them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const unsigned int budget = spin_budget();

  if (warp < BG_FRONT_WARPS) {
    if constexpr (BN == 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(BG_FRONT_REGS));
    if (warp == 0) {
      if (lane == 0) {
        bool ok = true;
        int s = 0; uint32_t ph = 0;
        for (int t = unit; ok && t < num_tiles; t += units) {
          const int m0 = tile_row(t), n0 = tile_col(t) + rank * (BN / 2);
          for (int kb = 0; kb < p.k_blocks; ++kb) {
            if (!mbar_wait(&empty[s], ph ^ 1, abort_flag, ST_TIMEOUT_PRODUCER, 0xE00 | s, budget)) { ok = false; break; }
            uint8_t* st = smem + s * L::STAGE;
            auto load = [&](void* dst, const CUtensorMap* m, int x, int y) {
              tma_load_2d_pair(dst, m, mapa_shared(smem_u32(&full[s]), 0), x, y);
            };
            if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * L::STAGE);
            load(st, &tm_a, kb * BG_BK, m0);
            if constexpr (KN) load(st + BG_A_BYTES, &tm_b, n0, kb * BG_BK);
            else load(st + BG_A_BYTES, &tm_b, kb * BG_BK, n0);
            if (++s == STAGES) { s = 0; ph ^= 1; }
          }
        }
        if (!ok) { const long long t0 = clock64(); while (clock64() - t0 < 2000000) { } }     // loads in flight land before the CTA exits
      }
    } else if (warp == 1 && rank == 0) {
      constexpr uint32_t idesc = umma_idesc(1, 0, 0, 2 * BG_BM, BN) | (KN ? UMMA_B_MN : 0u);
      bool ok = true;
      int s = 0, as = 0; uint32_t ph = 0, aph = 0;
      for (int t = unit; ok && t < num_tiles; t += units) {
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          // (the stage's return last: it is what the MMAs wait for)
          if (!__all_sync(0xffffffffu, mbar_wait<true>(&full[s], ph, abort_flag, ST_TIMEOUT_MMA, 0xE20 | s, budget))) { ok = false; break; }
          const uint32_t st = smem_u32(smem + s * L::STAGE);
          const uint64_t a_desc = umma_smem_desc_sw128(st);
          const uint64_t b_desc = KN ? umma_smem_desc_mn<BN / 2>(st + BG_A_BYTES, 0) : umma_smem_desc_sw128(st + BG_A_BYTES);
          if (!__all_sync(0xffffffffu, mbar_wait<true>(&acc_empty[as], aph ^ 1, abort_flag, ST_TIMEOUT_MMA, 0xE10 | as, budget))) { ok = false; break; }
          tc_fence_after();
          constexpr uint64_t b_step = KN ? (32 * (BN / 2)) >> 4 : 2;      // K = 32: 32 rows of BN / 2 bytes, or 32 bytes of a row
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_f8_pair_elect(tmem_base + as * BN, a_desc + 2 * k, b_desc + b_step * k, idesc, k != 0);
          umma_commit_pair_both_elect(&acc_full[as]);
          umma_commit_pair_both_elect(&empty[s]);
          if (++s == STAGES) { s = 0; ph ^= 1; }
          if (++as == ACC) { as = 0; aph ^= 1; }
        }
      }
    } else if (warp >= 2) {
      // The products of the scales, ahead of the MMAs: two rows and both column halves per lane, loaded ahead.  A K
      // block's arrival completes acc_full together with the MMAs' (the one wait of the epilogue covers both), and must follow the
      // barrier's previous phase, ACC K blocks back.  The place that it takes in shared memory held the K block 2 ACC back.  The epilogue warps hand it back
      // on a barrier of its own (sc_empty): the arrival that returns their stage is relaxed and orders no read of shared memory.  They do so behind the K
      // block's multiply-adds, off the chain (us, M = 65536, N = 1536, K = 512 / N = 512, K = 2048 / N = 640, K = 512: so 71.7 / 75.1 / 45.8; right behind the
      // read 73.3 / 75.9 / 45.0; a barrier for half of the places 73.1 / 75.2 / 44.3).
      const int r = (warp - 2) * 64 + lane;
      constexpr int FAR = 4;                                 // K blocks that are loaded ahead
      float a0[FAR], a1[FAR], b0[FAR], b1[FAR];
      int ft = unit, fkb = 0;                                // what is fetched next
      auto fetch_next = [&](int j) {
        if (ft < num_tiles) {
          const int m = tile_row(ft) + r, n = tile_col(ft);
          a0[j] = ldg_f_here(p.sa + (long long)(m < p.M ? m : p.M - 1) * p.ld_sa + fkb);
          a1[j] = ldg_f_here(p.sa + (long long)(m + 32 < p.M ? m + 32 : p.M - 1) * p.ld_sa + fkb);
          const float* sb = p.sb + (long long)fkb * p.ld_sb_k + (long long)(n >> 7) * p.ld_sb_n;
          b0[j] = ldg_f_here(sb);
          b1[j] = BN == 128 ? b0[j] : n + 128 < p.N ? ldg_f_here(sb + p.ld_sb_n) : 0.f;
        }
        if (++fkb == p.k_blocks) { fkb = 0; ft += units; }
      };
#pragma unroll
      for (int j = 0; j < FAR; ++j) { a0[j] = a1[j] = b0[j] = b1[j] = 0.f; fetch_next(j); }
      bool ok = true;
      uint32_t i = 0;
      auto put = [&](int j) {
        const uint32_t as = i % ACC, place = i % SC;
        if (i >= SC && !__all_sync(0xffffffffu, mbar_wait<true>(&sc_empty[place], (i / SC - 1) & 1, abort_flag, ST_TIMEOUT_PRODUCER, 0xE48 | place, budget))) { ok = false; return; }
        if (i >= ACC && !__all_sync(0xffffffffu, mbar_wait<true>(&acc_full[as], (i / ACC - 1) & 1, abort_flag, ST_TIMEOUT_PRODUCER, 0xE40 | as, budget))) { ok = false; return; }
        float* d = sc_smem + place * 2 * BG_BM + r;
        d[0] = a0[j] * b0[j]; d[32] = a1[j] * b0[j]; d[BG_BM] = a0[j] * b1[j]; d[BG_BM + 32] = a1[j] * b1[j];
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_full[as]);
        fetch_next(j);
        ++i;
      };
      const uint32_t all = (uint32_t)((num_tiles - unit + units - 1) / units) * (uint32_t)p.k_blocks;      // (unit < num_tiles; bounded by the host)
      while (ok && i < all) {
#pragma unroll
        for (int j = 0; j < FAR; ++j)
          if (ok && i < all) put(j);
      }
    }
  } else {
    if constexpr (BN == 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(BG_EPI_REGS));      // (128 sums; with 64 the even share is enough)
    const int e = warp - BG_FRONT_WARPS, q = warp & 3, half = e >> 2;
    const uint32_t t_lane = tmem_base + ((uint32_t)(q * 32) << 16) + half * CW;
    bool ok = true;
    const float* const sc_lane = sc_smem + half * BG_BM + q * 32 + lane;
    const uint32_t release_addr = mapa_shared(smem_u32(&acc_empty[0]), 0);
    uint32_t it = 0;                                         // K blocks so far: stage it % ACC, phase it / ACC % 2
    for (int t = unit; ok && t < num_tiles; t += units) {
      const int m0 = tile_row(t) + q * 32, n0 = tile_col(t) + half * CW;
      const int row = m0 + lane;
      const bool live = m0 < p.M && n0 < p.N;                // (uniform) this warp has something to write
      float acc[CW];
#pragma unroll
      for (int i = 0; i < CW; ++i) acc[i] = 0.f;
      // A chain of 32-column chunks: while one is added, the next is on its way from tensor memory, across K blocks too if the next
      // stage is there already; a stage goes back as soon as its last chunk is in registers.
      uint32_t v[2][32];
      auto stage_there = [&]() { return __all_sync(0xffffffffu, mbar_wait<true>(&acc_full[it % ACC], (it / ACC) & 1, abort_flag, ST_TIMEOUT_EPILOGUE, 0xE30, budget)); };
      ok = stage_there();
      if (!ok) break;
      tc_fence_after();
      tmem_ld_32x32b_x32(t_lane + it % ACC * BN, v[0]);
      for (int kb = 0; kb < p.k_blocks; ++kb) {
        const float sc = sc_lane[it % SC * 2 * BG_BM];
        const bool more = kb + 1 < p.k_blocks;
        const float2 s2 = pk2(sc, sc);
        bool there = false;
#pragma unroll
        for (int c = 0; c < CW / 32; ++c) {
          tmem_ld_wait(v[c & 1]);
          if (c + 1 < CW / 32) {
            tmem_ld_32x32b_x32(t_lane + it % ACC * BN + 32 * (c + 1), v[(c + 1) & 1]);
          } else {
            tc_fence_before();
            if (lane == 0) mbar_arrive_remote_relaxed(release_addr + 8 * (it % ACC));
            ++it;
            there = more && __all_sync(0xffffffffu, mbar_test_wait(&acc_full[it % ACC], (it / ACC) & 1));
            if (there) {
              tc_fence_after();
              tmem_ld_32x32b_x32(t_lane + it % ACC * BN, v[0]);
            }
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 r = __ffma2_rn(pk2(__uint_as_float(v[c & 1][2 * i]), __uint_as_float(v[c & 1][2 * i + 1])), s2,
                                        pk2(acc[32 * c + 2 * i], acc[32 * c + 2 * i + 1]));
            acc[32 * c + 2 * i] = r.x; acc[32 * c + 2 * i + 1] = r.y;
          }
        }
        __syncwarp();                                        // (every lane has read its scale)
        if (lane == 0) mbar_arrive(&sc_empty[(it - 1) % SC]);
        if (more && !there) {
          ok = stage_there();
          if (!ok) break;
          tc_fence_after();
          tmem_ld_32x32b_x32(t_lane + it % ACC * BN, v[0]);
        }
      }
      if (!ok || !live) continue;
      // Boxes of 32 rows x 128 bytes (32 columns of fp32, 64 of 16 bits) in the 128-byte swizzle, two at a time.
      uint8_t* const out_buf = smem + L::OUT + e * BG_OUT_BUF;
      uint8_t* const line = out_buf + lane * 128;
      const int wide = p.c_type == GSB200_F32 ? 32 : 64;       // columns of a box
      auto boxes = [&](auto pack8, auto most, int first, int n_boxes) {        // pack8(bx, pc): 16-byte piece pc of a row of box bx
        if (lane == 0) tma_store_wait_read<0>();             // the previous boxes have left the buffer
        __syncwarp();
#pragma unroll
        for (int bx = 0; bx < decltype(most)::value; ++bx)
#pragma unroll
          for (int pc = 0; pc < 8; ++pc) *reinterpret_cast<uint4*>(line + bx * (BG_OUT_BUF / 2) + ((pc ^ (lane & 7)) << 4)) = pack8(bx, pc);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          for (int bx = 0; bx < n_boxes; ++bx) tma_store_2d(&tm_c, out_buf + bx * (BG_OUT_BUF / 2), first + bx * wide, m0);
          tma_store_commit();
        }
      };
      const int tma_cols = p.n_tma - n0;                       // columns of this warp that leave through boxes
      if (tma_cols > 0) {
        if (p.c_type == GSB200_F32) {
#pragma unroll
          for (int c0 = 0; c0 < CW; c0 += 64) {
            if (c0 >= tma_cols) break;
            boxes([&](int bx, int pc) {
              const float* a = acc + c0 + 32 * bx + 4 * pc;
              return make_uint4(__float_as_uint(a[0]), __float_as_uint(a[1]), __float_as_uint(a[2]), __float_as_uint(a[3]));
            }, std::integral_constant<int, 2>{}, n0 + c0, tma_cols - c0 > 32 ? 2 : 1);
          }
        } else if (p.c_type == GSB200_F16) {
          boxes([&](int bx, int pc) {
            const float* a = acc + 64 * bx + 8 * pc;
            return make_uint4(pack_half2(a[0], a[1]), pack_half2(a[2], a[3]), pack_half2(a[4], a[5]), pack_half2(a[6], a[7]));
          }, std::integral_constant<int, CW / 64>{}, n0, CW > 64 && tma_cols > 64 ? 2 : 1);
        } else {
          boxes([&](int bx, int pc) {
            const float* a = acc + 64 * bx + 8 * pc;
            return make_uint4(pack_bf2(a[0], a[1]), pack_bf2(a[2], a[3]), pack_bf2(a[4], a[5]), pack_bf2(a[6], a[7]));
          }, std::integral_constant<int, CW / 64>{}, n0, CW > 64 && tma_cols > 64 ? 2 : 1);
        }
      }
      if (tma_cols < CW && p.n_tma < p.N) {                    // what TMA cannot address (n_tma is a whole number of boxes)
        if (lane == 0) tma_store_wait_read<0>();
        const int rows = p.M - m0 < 32 ? p.M - m0 : 32;
        const long long o = (long long)m0 * p.ldc + n0;
        if (p.c_type == GSB200_F32) {
#pragma unroll
          for (int c0 = 0; c0 < CW; c0 += 32) {
            if (c0 < tma_cols || n0 + c0 >= p.N) continue;
            store_by_rows<uint32_t, 8>(out_buf, lane, [&](int pc) {
              const float* a = acc + c0 + 4 * pc;
              return make_uint4(__float_as_uint(a[0]), __float_as_uint(a[1]), __float_as_uint(a[2]), __float_as_uint(a[3]));
            }, static_cast<uint32_t*>(p.C) + o + c0, p.ldc, rows, p.N - n0 - c0);
          }
        } else {
          const bool f16 = p.c_type == GSB200_F16;
#pragma unroll
          for (int c0 = 0; c0 < CW; c0 += 64) {
            if (c0 < tma_cols || n0 + c0 >= p.N) continue;
            store_by_rows<uint16_t, 8>(out_buf, lane, [&](int pc) {
              const float* a = acc + c0 + 8 * pc;
              return f16 ? make_uint4(pack_half2(a[0], a[1]), pack_half2(a[2], a[3]), pack_half2(a[4], a[5]), pack_half2(a[6], a[7]))
                         : make_uint4(pack_bf2(a[0], a[1]), pack_bf2(a[2], a[3]), pack_bf2(a[4], a[5]), pack_bf2(a[6], a[7]));
            }, static_cast<uint16_t*>(p.C) + o + c0, p.ldc, rows, p.N - n0 - c0);
          }
        }
        __syncwarp();                                          // (the next tile's boxes go into the same buffer)
      }
    }
    if (lane == 0) tma_store_wait_all<0>();
  }
  tc_fence_before();
  // neither CTA leaves (or frees tensor memory) while the other may still arrive at its barriers or its MMAs write here
  cluster_sync_all();
  if (warp == 1) { tc_fence_after(); tmem_dealloc_pair(tmem_base, ACC * BN); }
}

// ---- few tiles ---------------------------------------------------------------------------------------------------------
// One tile of 128 rows x BN columns per CTA.  With few rows the time is a chain of latencies: the narrow tile spreads the weight over the SMs,
// a K block takes BN tensor-memory columns, so that up to 512 / BN of them are multiplied before the first has been added, and of a single
// row block only the rows that are there are loaded.  N = 2048, K = 512: 64 rows 3.1 us, 333 3.7, 1000 4.7 (single CTAs with 256 columns 6.2, 6.6, 6.8).
//   warp 0 TMA producer, warp 1 MMA issue, warps 2..9 epilogue (lane quarter w % 4, column half), results straight from registers
constexpr int BS_THREADS = 32 * 10;
template <int BN>
struct BsSmem {
  static constexpr int STAGE = BG_A_BYTES + BN * BG_BK;                    // 20, 24 or 32 KiB
  static constexpr int STAGES = BN == 128 ? 6 : 8;
  static constexpr int ACC = 512 / BN;                                     // tensor-memory stages: 16, 8, 4
  static constexpr int BAR = STAGES * STAGE;
  static constexpr int BYTES = BAR + (2 * STAGES + 2 * ACC) * 8 + 16 + 1024;
  static_assert(BYTES <= 227 * 1024, "shared memory budget");
};

template <int BN, bool KN>
__global__ void __launch_bounds__(BS_THREADS, 1)
block_gemm_small_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const BgParams p) {
  extern __shared__ uint8_t bs_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(bs_smem_raw) + 1023) & ~uintptr_t(1023));
  using L = BsSmem<BN>;
  constexpr int STAGES = L::STAGES, ACC = L::ACC, CW = BN / 2;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BAR);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint64_t* acc_empty = acc_full + ACC;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + ACC);
  const AbortFlag abort_flag{smem_u32(tmem_slot + 1)};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m0 = (int)(blockIdx.x / p.n_blocks) * BG_BM, n0 = (int)(blockIdx.x % p.n_blocks) * BN;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int s = 0; s < ACC; ++s) { mbar_init(&acc_full[s], 1); mbar_init(&acc_empty[s], BG_EPI_WARPS); }
    abort_flag.set(0);
    fence_mbar_init();
    prefetch_tmap(&tm_a); prefetch_tmap(&tm_b);
  }
  if (warp == 1) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_trigger();                                           // (after the tensor memory is in hand: see launch_gemm_small)
  pdl_wait();
  const unsigned int budget = spin_budget();

  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      int s = 0; uint32_t ph = 0;
      for (int kb = 0; kb < p.k_blocks; ++kb) {
        if (kb >= STAGES && !mbar_wait<true>(&empty[s], ph ^ 1, abort_flag, ST_TIMEOUT_PRODUCER, 0xE50 | s, budget)) { ok = false; break; }
        uint8_t* st = smem + s * L::STAGE;
        // (of a single row block only the rows that are there: what the others hold stays in rows that are not written)
        mbar_arrive_expect_tx(&full[s], p.a_rows * BG_BK + BN * BG_BK);
        tma_load_2d(st, &tm_a, &full[s], kb * BG_BK, m0);
        if constexpr (KN) tma_load_2d(st + BG_A_BYTES, &tm_b, &full[s], n0, kb * BG_BK);
        else tma_load_2d(st + BG_A_BYTES, &tm_b, &full[s], kb * BG_BK, n0);
        if (++s == STAGES) { s = 0; ph ^= 1; }
      }
      if (!ok) { const long long t0 = clock64(); while (clock64() - t0 < 2000000) { } }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = umma_idesc(1, 0, 0, BG_BM, BN) | (KN ? UMMA_B_MN : 0u);
    int s = 0, as = 0; uint32_t ph = 0, aph = 0;
    for (int kb = 0; kb < p.k_blocks; ++kb) {
      if (!__all_sync(0xffffffffu, mbar_wait<true>(&full[s], ph, abort_flag, ST_TIMEOUT_MMA, 0xE60 | s, budget))) break;
      if (kb >= ACC && !__all_sync(0xffffffffu, mbar_wait<true>(&acc_empty[as], aph ^ 1, abort_flag, ST_TIMEOUT_MMA, 0xE70 | as, budget))) break;
      tc_fence_after();
      const uint32_t st = smem_u32(smem + s * L::STAGE);
      const uint64_t a_desc = umma_smem_desc_sw128(st);
      const uint64_t b_desc = KN ? umma_smem_desc_mn<BN>(st + BG_A_BYTES, 0) : umma_smem_desc_sw128(st + BG_A_BYTES);
      constexpr uint64_t b_step = KN ? (32 * BN) >> 4 : 2;                  // K = 32: 32 rows of BN bytes, or 32 bytes of a row
#pragma unroll
      for (int k = 0; k < 4; ++k) umma_f8_elect(tmem_base + as * BN, a_desc + 2 * k, b_desc + b_step * k, idesc, k != 0);
      umma_commit_elect(&acc_full[as]);
      if (kb + STAGES < p.k_blocks) umma_commit_elect(&empty[s]);
      if (++s == STAGES) { s = 0; ph ^= 1; }
      if (++as == ACC) { as = 0; aph ^= 1; }
    }
  } else {
    const int q = warp & 3, half = warp >= 6 ? 1 : 0;      // warps 2..5 and 6..9: each quarter once
    const int row = m0 + q * 32 + lane, n = n0 + half * CW;
    const bool live = m0 + q * 32 < p.M && n < p.N;
    const float* sa = p.sa + (long long)(row < p.M ? row : p.M - 1) * p.ld_sa;
    const float* sb = p.sb + (long long)((n < p.N ? n : 0) >> 7) * p.ld_sb_n;
    const uint32_t t_lane = tmem_base + ((uint32_t)(q * 32) << 16) + half * CW;
    constexpr int AHEAD = 4;                               // scales are loaded so many K blocks ahead
    float sc[AHEAD], sd[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      sc[j] = j < p.k_blocks ? ldg_f_here(sa + j) : 0.f;
      sd[j] = j < p.k_blocks ? ldg_f_here(sb + (long long)j * p.ld_sb_k) : 0.f;
    }
    float acc[CW];
#pragma unroll
    for (int i = 0; i < CW; ++i) acc[i] = 0.f;
    bool ok = true;
    int as = 0; uint32_t aph = 0;
    for (int kb0 = 0; ok && kb0 < p.k_blocks; kb0 += AHEAD) {
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int kb = kb0 + j;
        if (kb >= p.k_blocks) break;
        const float s1 = sc[j] * sd[j];
        if (kb + AHEAD < p.k_blocks) {
          sc[j] = ldg_f_here(sa + kb + AHEAD);
          sd[j] = ldg_f_here(sb + (long long)(kb + AHEAD) * p.ld_sb_k);
        }
        ok = __all_sync(0xffffffffu, mbar_wait<true>(&acc_full[as], aph, abort_flag, ST_TIMEOUT_EPILOGUE, 0xE80 | as, budget));
        if (!ok) break;
        tc_fence_after();
        constexpr int CH = CW < 32 ? 16 : 32;
#pragma unroll
        for (int c = 0; c < CW / CH; ++c) {
          uint32_t v[CH];
          if constexpr (CH == 16) tmem_ld_32x32b_x16(t_lane + as * BN + CH * c, v);
          else tmem_ld_32x32b_x32(t_lane + as * BN + CH * c, v);
          tmem_ld_wait(v);
          if (c + 1 == CW / CH) {
            tc_fence_before();
            if (lane == 0) mbar_arrive(&acc_empty[as]);
          }
#pragma unroll
          for (int i = 0; i < CH; ++i) acc[CH * c + i] = fmaf(__uint_as_float(v[i]), s1, acc[CH * c + i]);
        }
        if (++as == ACC) { as = 0; aph ^= 1; }
      }
    }
    const int esz = p.c_type == GSB200_F32 ? 4 : 2;
    uint8_t* dst = static_cast<uint8_t*>(p.C) + ((long long)row * p.ldc + n) * esz;
    // 32 or 16 bytes at a time, as C's rows allow (M = 371, N = 3288, K = 640, fp16: element by element 23.5 us, 16 bytes 5.2)
    const uintptr_t at = reinterpret_cast<uintptr_t>(p.C) | (uintptr_t)(p.ldc * esz);
    const bool wide = (at & 31) == 0;
    if (ok && live && (at & 15) == 0) {
      if (row < p.M && p.c_type == GSB200_F32) {
#pragma unroll
        for (int b = 0; b < CW / 8; ++b) {
          const uint4 v[2] = {make_uint4(__float_as_uint(acc[8 * b]), __float_as_uint(acc[8 * b + 1]), __float_as_uint(acc[8 * b + 2]), __float_as_uint(acc[8 * b + 3])),
                              make_uint4(__float_as_uint(acc[8 * b + 4]), __float_as_uint(acc[8 * b + 5]), __float_as_uint(acc[8 * b + 6]), __float_as_uint(acc[8 * b + 7]))};
          if (wide && n + 8 * b + 8 <= p.N) {
            stg_v8(dst + 32 * b, v[0], v[1]);
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (n + 8 * b + 4 * h + 4 <= p.N) {
                *reinterpret_cast<uint4*>(dst + 32 * b + 16 * h) = v[h];
              } else {
#pragma unroll
                for (int i = 4 * h; i < 4 * h + 4; ++i)
                  if (n + 8 * b + i < p.N) reinterpret_cast<float*>(dst)[8 * b + i] = acc[8 * b + i];
              }
            }
          }
        }
      } else if (row < p.M) {
#pragma unroll
        for (int b = 0; b < CW / 16; ++b) {
          uint32_t w[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = p.c_type == GSB200_F16 ? pack_half2(acc[16 * b + 2 * i], acc[16 * b + 2 * i + 1]) : pack_bf2(acc[16 * b + 2 * i], acc[16 * b + 2 * i + 1]);
          if (wide && n + 16 * b + 16 <= p.N) {
            stg_v8(dst + 32 * b, make_uint4(w[0], w[1], w[2], w[3]), make_uint4(w[4], w[5], w[6], w[7]));
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (n + 16 * b + 8 * h + 8 <= p.N) {
                *reinterpret_cast<uint4*>(dst + 32 * b + 16 * h) = make_uint4(w[4 * h], w[4 * h + 1], w[4 * h + 2], w[4 * h + 3]);
              } else {
#pragma unroll
                for (int i = 8 * h; i < 8 * h + 8; ++i)
                  if (n + 16 * b + i < p.N) reinterpret_cast<uint16_t*>(dst)[16 * b + i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
              }
            }
          }
        }
      }
    } else if (ok && live) {                               // through the operands' memory: the last sums are here, so nothing reads or writes it any more
      static_assert(BG_EPI_WARPS * 4096 <= STAGES * L::STAGE, "a box per warp");
      uint8_t* const box = smem + (warp - 2) * 4096;
      const int rows = p.M - (m0 + q * 32) < 32 ? p.M - (m0 + q * 32) : 32;
      const long long o = (long long)(m0 + q * 32) * p.ldc + n;
      if (p.c_type == GSB200_F32) {
        constexpr int W = CW < 32 ? CW : 32;
#pragma unroll
        for (int c0 = 0; c0 < CW; c0 += W) {
          if (n + c0 >= p.N) continue;
          store_by_rows<uint32_t, W / 4>(box, lane, [&](int pc) {
            const float* a = acc + c0 + 4 * pc;
            return make_uint4(__float_as_uint(a[0]), __float_as_uint(a[1]), __float_as_uint(a[2]), __float_as_uint(a[3]));
          }, static_cast<uint32_t*>(p.C) + o + c0, p.ldc, rows, p.N - n - c0);
        }
      } else {
        const bool f16 = p.c_type == GSB200_F16;
        store_by_rows<uint16_t, CW / 8>(box, lane, [&](int pc) {
          const float* a = acc + 8 * pc;
          return f16 ? make_uint4(pack_half2(a[0], a[1]), pack_half2(a[2], a[3]), pack_half2(a[4], a[5]), pack_half2(a[6], a[7]))
                     : make_uint4(pack_bf2(a[0], a[1]), pack_bf2(a[2], a[3]), pack_bf2(a[4], a[5]), pack_bf2(a[6], a[7]));
        }, static_cast<uint16_t*>(p.C) + o, p.ldc, rows, p.N - n);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem_base, 512); }
}

template <int BN, bool KN>
static cudaError_t launch_bs(const CUtensorMap& ta, const CUtensorMap& tb, const BgParams& p, int dev, int grid, cudaStream_t st) {
  static std::atomic<int> attr_done[64];
  auto k = block_gemm_small_kernel<BN, KN>;
  if (!attr_done[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, BsSmem<BN>::BYTES);
    if (e != cudaSuccess) return e;
    attr_done[dev].store(1, std::memory_order_release);
  }
  return launch_dependent(k, (unsigned)grid, BS_THREADS, (size_t)BsSmem<BN>::BYTES, st, ta, tb, p);
}

// ---- a few rows -----------------------------------------------------------------------------------------------------------
// Up to four rows, B [N, K] (a decoder's products): the time is the read of the weight, and a tensor-core tile would spend 0.3 us on each
// K block of a chain.  A warp owns a column: a lane reads 16 consecutive elements of it per 512, multiplies them in fp32 with A's (as fp32 in shared
// memory, in the order in which the lanes read them without conflicts), and the 16 products' sum, times the block's scale, goes to the lane's sum;
// the lanes' are added at the end, in a fixed order.  us, this / the few-tile form: one row N = 2048, K = 512 2.0 / 3.1, N = 512, K = 2048 2.8 / 6.3, N = 4096,
// K = 4096 6.9 / 11.6; two rows 2.3 / 3.1, 3.5 / 6.3, 10.4 / 11.6; four 3.0 / 3.1, 5.1 / 6.3 and, N = 4096, K = 1024, 6.2 / 4.3 (every CTA lays A out): three
// and four rows up to a million weights.
constexpr int GV_WARPS = 8;
constexpr int GV_MAX = 10240;                              // elements of A in shared memory (rows x K, K rounded up to 512)
template <int ROWS>
__global__ void __launch_bounds__(GV_WARPS * 32)
block_gemv_kernel(const uint8_t* A, long long lda, const uint8_t* B, long long ldb, int K, const BgParams p) {
  __shared__ float4 a_s[GV_MAX / 4];                       // [K / 512][row][4][lane]: elements 512 i + 16 lane + 4 j ..
  __shared__ float sc_s[GV_MAX / 128];                     // [row][K block] products of the scales
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n_base = blockIdx.x * GV_WARPS, n = n_base + warp;
  const int rounds = (K + 511) / 512;
  pdl_wait();
  pdl_trigger();
  // the column's first elements are on their way while A is laid out
  const uint8_t* b = B + (long long)(n < p.N ? n : p.N - 1) * ldb;
  auto load_b = [&](int i) {
    const int k = 512 * i + 16 * lane;
    if (k + 16 <= K) return *reinterpret_cast<const uint4*>(b + k);
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < 15; ++j)
      if (k + j < K) w[j >> 2] |= (uint32_t)b[k + j] << (8 * (j & 3));
    return make_uint4(w[0], w[1], w[2], w[3]);
  };
  uint4 next = load_b(0);
  for (int i = threadIdx.x; i < ROWS * rounds * 128; i += GV_WARPS * 32) {      // four elements at a time
    const int l = i & 31, j = (i >> 5) & 3, m = (i >> 7) % ROWS, r = (i >> 7) / ROWS;
    const int k = 512 * r + 16 * l + 4 * j;
    uint32_t w = 0u;
    if (m < p.M && k < K) {
      const uint8_t* a = A + (long long)m * lda + k;
      if (k + 4 <= K) w = *reinterpret_cast<const uint32_t*>(a);
      else {
#pragma unroll
        for (int t = 0; t < 3; ++t)
          if (k + t < K) w |= (uint32_t)a[t] << (8 * t);
      }
    }
    const float2 lo = e4m3x2_f32(w), hi = e4m3x2_f32(w >> 16);
    a_s[i] = make_float4(lo.x, lo.y, hi.x, hi.y);
  }
  for (int i = threadIdx.x; i < ROWS * p.k_blocks; i += GV_WARPS * 32) {
    const int m = i / p.k_blocks, kb = i % p.k_blocks;
    sc_s[i] = m < p.M ? p.sa[(long long)m * p.ld_sa + kb] * p.sb[(long long)(n_base >> 7) * p.ld_sb_n + kb] : 0.f;
  }
  __syncthreads();
  float sum[ROWS];
#pragma unroll
  for (int m = 0; m < ROWS; ++m) sum[m] = 0.f;
  for (int r = 0; r < rounds; ++r) {
    const uint32_t w[4] = {next.x, next.y, next.z, next.w};
    if (r + 1 < rounds) next = load_b(r + 1);
    const int kb = 4 * r + (lane >> 3);
    float2 part[ROWS];
#pragma unroll
    for (int m = 0; m < ROWS; ++m) part[m] = make_float2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 lo = e4m3x2_f32(w[j]), hi = e4m3x2_f32(w[j] >> 16);
#pragma unroll
      for (int m = 0; m < ROWS; ++m) {
        const float4 a = a_s[((r * ROWS + m) * 4 + j) * 32 + lane];
        part[m] = __ffma2_rn(make_float2(a.x, a.y), lo, part[m]);
        part[m] = __ffma2_rn(make_float2(a.z, a.w), hi, part[m]);
      }
    }
    if (kb < p.k_blocks) {
#pragma unroll
      for (int m = 0; m < ROWS; ++m) sum[m] = fmaf(part[m].x + part[m].y, sc_s[m * p.k_blocks + kb], sum[m]);
    }
  }
#pragma unroll
  for (int m = 0; m < ROWS; ++m) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum[m] += __shfl_xor_sync(0xffffffffu, sum[m], d);
    if (lane == 0 && n < p.N && m < p.M) {
      const long long o = (long long)m * p.ldc + n;
      if (p.c_type == GSB200_F32) static_cast<float*>(p.C)[o] = sum[m];
      else if (p.c_type == GSB200_F16) static_cast<__half*>(p.C)[o] = __float2half_rn(sum[m]);
      else static_cast<__nv_bfloat16*>(p.C)[o] = __float2bfloat16_rn(sum[m]);
    }
  }
}

// Launches `units` pairs; units = 0 asks how many can be resident (0: this form must not be launched here).
template <int BN, bool KN>
static cudaError_t launch_bg(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, const BgParams& p, int dev, int units, int* capacity,
                             cudaStream_t st) {
  static std::atomic<int> cap[64];
  auto k = block_gemm_kernel<BN, KN>;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(BG_THREADS); cfg.dynamicSmemBytes = BgSmem<BN>::BYTES; cfg.stream = st;
  cfg.attrs = attr; cfg.numAttrs = 2;
  int c = cap[dev].load(std::memory_order_acquire);
  if (c == 0) {
    // the re-split of the registers waits until the block's own pool covers it
    cudaFuncAttributes fa{};
    cudaError_t e = cudaFuncGetAttributes(&fa, k);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, BgSmem<BN>::BYTES);
    if (e != cudaSuccess) return e;
    cfg.gridDim = dim3((unsigned)(sm_count_physical() / 2 * 2));
    int n = 0;
    const bool pool = BN != 256 || (fa.numRegs * BG_THREADS >= 32 * (BG_FRONT_WARPS * BG_FRONT_REGS + BG_EPI_WARPS * BG_EPI_REGS) && fa.numRegs * BG_THREADS <= 65536);
    c = pool && cudaOccupancyMaxActiveClusters(&n, k, &cfg) == cudaSuccess && n > 0 ? n : -1;
    (void)cudaGetLastError();
    cap[dev].store(c, std::memory_order_release);
  }
  if (units == 0) { *capacity = c > 0 ? c : 0; return cudaSuccess; }
  cfg.gridDim = dim3((unsigned)(2 * units));
  return cudaLaunchKernelEx(&cfg, k, ta, tb, tc, p);
}

static cudaError_t launch_bg_form(int pn, bool kn, const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, const BgParams& p, int dev, int units,
                                  int* capacity, cudaStream_t st) {
  return pn == 256 ? (kn ? launch_bg<256, true>(ta, tb, tc, p, dev, units, capacity, st) : launch_bg<256, false>(ta, tb, tc, p, dev, units, capacity, st))
                   : (kn ? launch_bg<128, true>(ta, tb, tc, p, dev, units, capacity, st) : launch_bg<128, false>(ta, tb, tc, p, dev, units, capacity, st));
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
  CUtensorMap ta{}, tb{}, tc{};
  BgParams p{};
  p.M = (int)M; p.N = N; p.k_blocks = kb;
  p.sa = sa; p.ld_sa = ld_sa; p.sb = sb; p.ld_sb_n = kn ? 1 : ld_sb; p.ld_sb_k = kn ? ld_sb : 1;
  p.C = C; p.ldc = ldc; p.c_type = c_type;
  const long long a_elems = (long long)(K + 511) / 512 * 512 * (M <= 2 ? M : 4);
  if (!kn && a_elems <= GV_MAX && (M <= 2 || (M <= 4 && (long long)N * K <= (1 << 20)))) {
    const unsigned g = (unsigned)((N + GV_WARPS - 1) / GV_WARPS);
    const cudaError_t e = M == 1 ? launch_dependent(block_gemv_kernel<1>, g, GV_WARPS * 32, 0, st, A, lda, B, ldb, K, p)
                        : M == 2 ? launch_dependent(block_gemv_kernel<2>, g, GV_WARPS * 32, 0, st, A, lda, B, ldb, K, p)
                                 : launch_dependent(block_gemv_kernel<4>, g, GV_WARPS * 32, 0, st, A, lda, B, ldb, K, p);
    return cuda_status(e, "block-scaled gemm launch");
  }
  const CUtensorMapDataType u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  const int sms = sm_count();
  const long long rb = (M + BG_BM - 1) / BG_BM;
  int bn = 0;                                                // the narrowest tile of which all are resident at once; none: pairs
  for (int w = 32; w <= 128 && bn == 0; w *= 2)
    if (rb * ((N + w - 1) / w) <= sms) bn = w;
  int units = 0, pn = 256;                                   // pairs, and the columns of their tiles
  if (bn == 0) {
    const long long rb2 = (M + 2 * BG_BM - 1) / (2 * BG_BM);
    // 128 columns where their rounds are cheaper: a tile takes 0.57 of the time of a 256-column one up to K = 512, 0.69 from there on (us, 256 / 128
    // columns, M = 65536: K = 512 N = 128 16.0 / 12.9, 640 41.0 / 40.4, 1536 70.6 / 80.2; K = 384, N = 384 25.9 / 23.4; K = 2048, N = 512 71.1 / 98.5)
    const long long pairs = sms / 2 > 0 ? sms / 2 : 1;
    const long long r256 = (rb2 * ((N + 255) / 256) + pairs - 1) / pairs, r128 = (rb2 * nb + pairs - 1) / pairs;
    if (r128 * (kb <= 4 ? 60 : 69) < r256 * 100) pn = 128;
    int cap = 0;
    const cudaError_t e = launch_bg_form(pn, kn, ta, ta, ta, p, dev, 0, &cap, st);
    if (e != cudaSuccess) return cuda_status(e, "block-scaled gemm set-up");
    units = (int)(pairs < cap ? pairs : cap);
    if (units == 0) bn = 128;                                // (pairs cannot be launched here)
  }
  if (bn != 0) {
    p.m_blocks = (int)rb; p.n_blocks = (N + bn - 1) / bn;
    const long long tiles = rb * p.n_blocks;
    if (tiles > 0x7fffffffll) return GSB200_ERR_BAD_ARG;
    p.a_rows = M < BG_BM ? (int)((M + 7) / 8 * 8) : BG_BM;
    if (!tmap_2d(&ta, u8, 1, A, (uint64_t)M, (uint64_t)K, (uint64_t)lda, BG_BK, (uint32_t)p.a_rows, CU_TENSOR_MAP_SWIZZLE_128B)) return GSB200_ERR_BAD_ARG;
    const CUtensorMapSwizzle sw = bn == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : bn == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B;
    if (kn ? !tmap_2d(&tb, u8, 1, B, (uint64_t)K, (uint64_t)N, (uint64_t)ldb, (uint32_t)bn, BG_BK, sw)
           : !tmap_2d(&tb, u8, 1, B, (uint64_t)N, (uint64_t)K, (uint64_t)ldb, BG_BK, (uint32_t)bn, CU_TENSOR_MAP_SWIZZLE_128B)) return GSB200_ERR_BAD_ARG;
    const int g = (int)tiles;
    const cudaError_t e = bn == 32 ? (kn ? launch_bs<32, true>(ta, tb, p, dev, g, st) : launch_bs<32, false>(ta, tb, p, dev, g, st))
                        : bn == 64 ? (kn ? launch_bs<64, true>(ta, tb, p, dev, g, st) : launch_bs<64, false>(ta, tb, p, dev, g, st))
                                   : (kn ? launch_bs<128, true>(ta, tb, p, dev, g, st) : launch_bs<128, false>(ta, tb, p, dev, g, st));
    return cuda_status(e, "block-scaled gemm launch");
  }
  p.m_blocks = (int)((M + 2 * BG_BM - 1) / (2 * BG_BM)); p.n_blocks = (N + pn - 1) / pn;
  const long long tiles = (long long)p.m_blocks * p.n_blocks;
  if (tiles > 0x7fffffffll) return GSB200_ERR_BAD_ARG;
  if (!tmap_2d(&ta, u8, 1, A, (uint64_t)M, (uint64_t)K, (uint64_t)lda, BG_BK, BG_BM, CU_TENSOR_MAP_SWIZZLE_128B)) return GSB200_ERR_BAD_ARG;
  // TMA writes whole 16-byte pieces: where a row of C ends inside one, the last box goes element by element
  const bool tma_out = (reinterpret_cast<uintptr_t>(C) & 15) == 0 && (ldc * esz) % 16 == 0;
  p.n_tma = !tma_out ? 0 : (N * esz) % 16 == 0 ? N : N / (128 / esz) * (128 / esz);
  const CUtensorMapDataType ct = c_type == GSB200_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                               : c_type == GSB200_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  if (kn ? !tmap_2d(&tb, u8, 1, B, (uint64_t)K, (uint64_t)N, (uint64_t)ldb, (uint32_t)(pn / 2), BG_BK, pn == 256 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B)
         : !tmap_2d(&tb, u8, 1, B, (uint64_t)N, (uint64_t)K, (uint64_t)ldb, BG_BK, (uint32_t)(pn / 2), CU_TENSOR_MAP_SWIZZLE_128B)) return GSB200_ERR_BAD_ARG;
  if (p.n_tma == 0) tc = ta;
  else if (!tmap_2d(&tc, ct, esz, C, (uint64_t)M, (uint64_t)N, (uint64_t)ldc, 128 / esz, 32, CU_TENSOR_MAP_SWIZZLE_128B)) return GSB200_ERR_BAD_ARG;
  if (tiles < units) units = (int)tiles;
  return cuda_status(launch_bg_form(pn, kn, ta, tb, tc, p, dev, units, nullptr, st), "block-scaled gemm launch");
}

}  // namespace gsb
