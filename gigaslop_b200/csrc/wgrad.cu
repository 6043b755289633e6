// Weight gradient from an 8-bit activation checkpoint:
//
//   dW[n, k] (+)= sum over m of dY[m, n] x^[m, k],     x^[m, k] = s[m, k / 128] q[m, k]
//
// dY is 16-bit, x^ is restored on chip: E4M3 times a power of two is exact in 16 bits, so nothing is lost
// against a 16-bit copy of the checkpoint that never exists in memory.  (A scale that is no power of two rounds the product to dY's
// type.)  The reduction runs over the rows of both operands, which the tensor core reads "MN-major".
//
// fp16 has not the range for that, and both operands of an MMA have one type.  So x^ is restored times a power of two, and the sums are divided by
// it, both exact.  A pass over the batch takes the rows whose scales, in these 128 columns, lie in a window of 22 powers of two: the largest become at most 2^7, 448
// of which fit, and the smallest keep all bits of E4M3.  The window is laid about the scales of 32 rows of the part, with more room above them than below; a row
// outside counts as zeros in the pass.  Where there was one, the scales are looked through, and passes with windows above and below follow as far as rows that are
// not all zeros need them.  us, fp16, without all this / with: M = 65536, N = 2048, K = 512 114.5 / 113.3, N = 512 43.0 / 40.9, M = 9001, N = 1000, K = 520 23.8 / 24.4 (one more window
// looked for and passed 68, five more 139), M = 1, N = 512, K = 512 7.7 / 8.2.  (The range of all scales looked up first: 4096 x 4096 x 4096 106 / 121, a column of scales is a load per row.)
//
// A CTA pair (cta_group::2) computes 512 x 256 of dW (two accumulators of 128 rows in each CTA, all of its tensor memory; narrow layers
// 256 x 256, one accumulator) over a range of rows of the batch, 64 rows per step.  A CTA holds its own rows of dW, i.e. columns of dY, and half
// of the tile's columns of x^, so an element of x^ is restored once per 512 columns of dY:
//   warp 0      TMA producer: dY, boxes of 64 rows x 64 columns
//   warp 1      MMA issue (first CTA): 4 MMAs (M = 256, N = 256, K = 16) per accumulator and step, 512 tensor clocks
//   warps 4..11 restore the step's 64 x 128 elements of x^ from global memory into the operand tile; at the end they write dW
// Few tiles are cut over the batch: each part writes its sums to the workspace, and a second launch adds them in order.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <atomic>

#include "capi_internal.h"
#include "ptx.cuh"

namespace gsb {

constexpr int WG_BK = 256, WG_BM = 64;                     // columns of x^ (a pair's), rows per step
constexpr int WG_WARPS = 8, WG_FRONT = 4, WG_THREADS = 32 * (WG_WARPS + WG_FRONT);
constexpr int WG_CHUNK = WG_BM * 128;                      // a 64-column chunk of an operand tile: 64 rows of 128 bytes
// Steps of 64 rows that the tensor core sums by itself.  Its fp32 additions truncate, which takes a little off a sum with each, fp16's longer products
// more than bf16's, so what it has summed is added to dW in segments, in fp32 as the parts are.  They are as long as keeps the error of random terms
// below 2^-19 in the 2-norm, whatever the batch.  Error / us (each segment costs 7, the time of 256 KiB per CTA through L2; written by the threads instead of by
// TMA 15 to 30) at M = 65536, N = 2048, K = 512, segments of 32, 48, 64, 128 steps: bf16 6.1e-7 / 126, 9.9e-7 / 118, 1.4e-6 / 112, 3.2e-6 (unsegmented) / 103; fp16
// 1.7e-6 / 126, 2.6e-6 / 119, 3.5e-6 / 112.  M = 65536, N = 4096, K = 4096: bf16 6.5e-7, 1.1e-6, 1.5e-6, 3.7e-6, fp16 1.8e-6, 2.8e-6, 3.9e-6; plain fp32
// products 1.5e-6 and 3.0e-6 (2e-7 where the batch is short).
template <typename T> constexpr int WG_SEGMENT = std::is_same<T, __half>::value ? 32 : 64;
constexpr int WG_AHEAD = 4;                                // steps of x^ in flight to the registers
constexpr int WG_B_BYTES = 2 * WG_CHUNK;                   // a CTA's 128 columns of x^
template <int ACC>                                         // accumulators (128 rows of dW per CTA each)
struct WgSmem {
  static constexpr int A_BYTES = ACC * 2 * WG_CHUNK;
  static constexpr int STAGE = A_BYTES + WG_B_BYTES;       // 48 or 32 KiB
  static constexpr int STAGES = ACC == 2 ? 4 : 5;
  static constexpr int OUT = STAGES * STAGE;               // per warp a box of 32 rows x 32 columns of dW
  static constexpr int BAR = OUT + WG_WARPS * 4096;
  static constexpr int BYTES = BAR + 256 + 1024;
  static_assert(BYTES <= 227 * 1024, "shared memory budget");
};

struct WgParams {
  const uint8_t* q; long long ldq; const float* s; long long lds;
  float* out; long long ldo;                               // dW, or this part's sums in the workspace
  long long part_rows;                                     // rows between the parts
  int tma_out;                                             // dW goes out in boxes
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
    o[i] = pack_half2_from(fmul2(f, make_float2(s, s)));
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
    const float2 v = fmul2(f, make_float2(s, s));
    o[i] = pack_bf2(v.x, v.y);
  }
  lo = make_uint4(o[0], o[1], o[2], o[3]); hi = make_uint4(o[4], o[5], o[6], o[7]);
}

constexpr int WG_WINDOW = 22;                              // fp16: powers of two that a pass covers
__device__ __forceinline__ int scale_exponent(float s) { return (int)(__float_as_uint(s) >> 23) & 255; }

template <typename T, int ACC>
__global__ void __launch_bounds__(WG_THREADS, 1)
wgrad_kernel(const __grid_constant__ CUtensorMap tm_dy, const __grid_constant__ CUtensorMap tm_out, const WgParams p) {
  extern __shared__ uint8_t wg_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(wg_smem_raw) + 1023) & ~uintptr_t(1023));
  using L = WgSmem<ACC>;
  constexpr int STAGES = L::STAGES, WG_SEG = WG_SEGMENT<T>;
  constexpr bool WINDOWS = std::is_same<T, __half>::value;
  uint64_t* full_a = reinterpret_cast<uint64_t*>(smem + L::BAR);
  uint64_t* full_b = full_a + STAGES;
  uint64_t* empty = full_b + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint64_t* acc_empty = acc_full + 1;
  uint64_t* missed_full = acc_empty + 1;                   // (fp16) missed[0] is known: whether either CTA has left scales out of the first pass
  uint64_t* more_full = missed_full + 1;                   // if so, missed[1] and missed[2]: how many passes above and below it their rows need
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(more_full + 1);
  int* missed = reinterpret_cast<int*>(tmem_slot + 2);
  static_assert((3 * STAGES + 4) * 8 + 8 + 12 <= 256, "room for the barriers");
  const AbortFlag abort_flag{smem_u32(tmem_slot + 1)};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_ctarank();                 // the pair's first CTA issues the MMAs; its barriers collect both CTAs' operands
  const int unit = (int)(blockIdx.x >> 1), tile = unit % p.tiles, part = unit / p.tiles;
  const int n0 = tile / p.k_tiles * (256 * ACC) + rank * 128, k0 = tile % p.k_tiles * WG_BK;      // accumulator j: columns n0 + 256 j .. of dY
  const int step0 = (int)((long long)p.steps * part / p.parts), step1 = (int)((long long)p.steps * (part + 1) / p.parts);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full_a[s], 1); mbar_init(&full_b[s], 2 * WG_WARPS); mbar_init(&empty[s], 1); }
    mbar_init(acc_full, 1); mbar_init(acc_empty, 2 * WG_WARPS); mbar_init(missed_full, 2 * WG_WARPS); mbar_init(more_full, 2 * WG_WARPS);
    missed[0] = missed[1] = missed[2] = 0;
    abort_flag.set(0);
    fence_mbar_init();
    prefetch_tmap(&tm_dy); prefetch_tmap(&tm_out);
  }
  if (warp == 1) { tmem_alloc_pair(tmem_slot, 256 * ACC); tmem_relinquish_pair(); }
  pdl_wait();
  float sample[2] = {0.f, 0.f};                            // scales of a row in both CTAs' columns: every warp looks at the same 32 rows of the part
  if (WINDOWS && warp >= WG_FRONT) {
    const long long r0 = (long long)step0 * WG_BM, r1 = (long long)step1 * WG_BM < p.M ? (long long)step1 * WG_BM : p.M;
    const float* const f = p.s + (r0 + (r1 - r0) * lane / 32) * p.lds + (k0 >> 7);
    sample[0] = f[0];
    if (k0 + 128 < p.K) sample[1] = f[1];
  }
  tc_fence_before();
  cluster_sync_all();                                      // (a __syncthreads of both CTAs) the other's barriers are initialised before anything arrives at them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const unsigned int budget = spin_budget();
  // Passes behind the first one (-1: gave up).
  auto missed_any = [&]() { return mbar_wait_cluster(missed_full, 0, abort_flag, ST_TIMEOUT_PRODUCER, 0xF50, budget) ? missed[0] : -1; };
  auto more_passes = [&]() {
    if constexpr (!WINDOWS) return 0;
    const int n = missed_any();
    return n <= 0 ? n : mbar_wait_cluster(more_full, 0, abort_flag, ST_TIMEOUT_PRODUCER, 0xF58, budget) ? missed[1] + missed[2] : -1;
  };

  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      int s = 0; uint32_t ph = 0;
      auto feed = [&]() {
        for (int i = step0; i < step1; ++i) {
          if (!mbar_wait(&empty[s], ph ^ 1, abort_flag, ST_TIMEOUT_PRODUCER, 0xF00 | s, budget)) { ok = false; break; }
          uint8_t* st = smem + s * L::STAGE;
          const uint32_t bar = mapa_shared(smem_u32(&full_a[s]), 0);
          if (rank == 0) mbar_arrive_expect_tx(&full_a[s], 2 * L::A_BYTES);
#pragma unroll
          for (int j = 0; j < 2 * ACC; ++j) tma_load_2d_pair(st + j * WG_CHUNK, &tm_dy, bar, n0 + 256 * (j >> 1) + 64 * (j & 1), i * WG_BM);
          if (++s == STAGES) { s = 0; ph ^= 1; }
        }
      };
      feed();
      for (int n = ok ? more_passes() : 0; ok && n > 0; --n) feed();
      if (!ok || abort_flag.get()) { const long long t0 = clock64(); while (clock64() - t0 < 2000000) { } }      // loads in flight land before the CTA exits
    }
  } else if (warp == 1 && rank == 0) {
    constexpr uint32_t fmt = std::is_same<T, __half>::value ? 0u : 1u;
    constexpr uint32_t idesc = umma_idesc(1, fmt, fmt, 256, WG_BK) | UMMA_A_MN | UMMA_B_MN;
    bool ok = true;
    int s = 0, segs = 0; uint32_t ph = 0;                   // segs: accumulations started
    auto multiply = [&]() {
      for (int i = step0; i < step1; ++i) {
        // x^ of the second CTA lies in that CTA's shared memory, and it is that SM's tensor core that reads it there.  The stores are in place when
        // the arrival leaves the SM: each writer passes them to the async proxy and its warp arrives behind that.  (An arrival with a
        // release to the cluster also waits for the loads in flight, 1400 clocks of each step: 184 us instead of 106 at M = 65536, N = 2048, K = 512.)
        if (!__all_sync(0xffffffffu, mbar_wait<true>(&full_a[s], ph, abort_flag, ST_TIMEOUT_MMA, 0xF10 | s, budget)) ||
            !__all_sync(0xffffffffu, mbar_wait<true>(&full_b[s], ph, abort_flag, ST_TIMEOUT_MMA, 0xF20 | s, budget))) { ok = false; break; }
        const int in_seg = (i - step0) % WG_SEG;
        if (in_seg == 0 && segs++ != 0 &&                      // the accumulators' previous sums are out
            !__all_sync(0xffffffffu, mbar_wait<true>(acc_empty, segs & 1, abort_flag, ST_TIMEOUT_MMA, 0xF60, budget))) { ok = false; break; }
        tc_fence_after();
        const uint32_t st = smem_u32(smem + s * L::STAGE);
        const uint64_t a_desc = umma_smem_desc_mn<128>(st, WG_CHUNK), b_desc = umma_smem_desc_mn<128>(st + L::A_BYTES, WG_CHUNK);
        constexpr uint64_t step = (16 * 128) >> 4;           // K = 16: 16 rows of 128 bytes
#pragma unroll
        for (int k = 0; k < 4; ++k) {
#pragma unroll
          for (int j = 0; j < ACC; ++j)
            umma_f16_pair_elect(tmem_base + 256 * j, a_desc + (j * 2 * WG_CHUNK >> 4) + step * k, b_desc + step * k, idesc, in_seg != 0 || k != 0);
        }
        umma_commit_pair_both_elect(&empty[s]);
        if (in_seg == WG_SEG - 1 || i + 1 == step1) umma_commit_pair_both_elect(acc_full);
        if (++s == STAGES) { s = 0; ph ^= 1; }
      }
    };
    multiply();
    for (int n = ok ? __shfl_sync(0xffffffffu, more_passes(), 0) : 0; ok && n > 0; --n) multiply();
  } else if (warp >= WG_FRONT) {
    // Thread: 16 columns of x^ (two 16-byte pieces of a row of the tile), rows r and r + 32 of the step, loaded WG_AHEAD steps ahead (a step is
    // shorter than a read of HBM).
    const int tid = threadIdx.x - 32 * WG_FRONT, c = tid & 7, r = tid >> 3;
    const int k = k0 + 128 * rank + 16 * c;
    const int have = p.K - k;                              // columns left from k on
    const long long dq = 32 * p.ldq, ds = 32 * p.lds;      // (to the thread's other row)
    const uint8_t* qp;
    const float* sp;
    auto rewind = [&]() {
      qp = p.q + ((long long)step0 * WG_BM + r) * p.ldq + (have > 0 ? k : 0);
      sp = p.s + ((long long)step0 * WG_BM + r) * p.lds + (have > 0 ? k >> 7 : 0);
    };
    rewind();
    uint4 raws[WG_AHEAD][2];
    float scs[WG_AHEAD][2];
    auto fetch = [&](int i, uint4 (&raw)[2], float (&sc)[2]) {
      raw[0] = raw[1] = make_uint4(0u, 0u, 0u, 0u);
      sc[0] = sc[1] = 0.f;
      if (i < step1 && have > 0) {
        // Whole 16-byte pieces: a row's stride holds them (columns behind K end in columns of dW that are not written), only the last row may end
        // before.
        const long long left = p.M - ((long long)i * WG_BM + r);     // rows from the thread's first on
        if ((long long)(i + 1) * WG_BM < p.M) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            raw[j] = *reinterpret_cast<const uint4*>(qp + j * dq);
            sc[j] = sp[j * ds];
          }
        } else {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            if (left <= 32 * j) continue;
            sc[j] = sp[j * ds];
            if (left > 32 * j + 1 || have >= 16) {
              raw[j] = *reinterpret_cast<const uint4*>(qp + j * dq);
            } else {
              uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
              for (int b = 0; b < 15; ++b)
                if (b < have) w[b >> 2] |= (uint32_t)qp[j * dq + b] << (8 * (b & 3));
              raw[j] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
      }
      qp += 2 * dq;
      sp += 2 * ds;
    };
#pragma unroll
    for (int a = 0; a < WG_AHEAD; ++a) fetch(step0 + a, raws[a], scs[a]);
    int tops[2] = {0, 0};                                  // greatest exponents of the pass, in both CTAs' columns of x^
    if constexpr (WINDOWS) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int e = scale_exponent(sample[i]);
        const bool counts = sample[i] != 0.f && e != 255;
        const int h = __reduce_max_sync(0xffffffffu, counts ? e : -1), l = __reduce_min_sync(0xffffffffu, counts ? e : 256);
        const int room = WG_WINDOW - 1 - (h - l);
        tops[i] = h < l ? 130 : h + (room > 0 ? room * 2 / 3 : 0);
      }
    }
    const uint32_t arrive_b = mapa_shared(smem_u32(full_b), 0);
    const int swap = (c >> 2) & 1, pc = 2 * (c & 3);       // half of the lanes store their second piece first: no bank conflicts
    bool ok = true;
    int top = 0;                                           // of this CTA's columns
    float up = 1.f;                                        // the factor on them
    auto factor_exponent = [](int e) { return max(min(260 - e, 253), 1); };        // 2^(133 - e): scales of exponent e become 2^6 .. 2^7
    uint32_t outside = 0;                                  // bits of the scales outside the pass
    // The factor of a row.  (Without a branch: the loads ahead wait at one, M = 9001, N = 1000, K = 520 26.1 us.  Infinite and NaN scales have a pass of their own.)
    auto factor = [&](float sc) {
      if constexpr (!WINDOWS) return sc;
      const bool in = (unsigned)(top - scale_exponent(sc)) < (unsigned)WG_WINDOW;
      outside |= in ? 0u : __float_as_uint(sc) & 0x7fffffffu;
      return in ? sc * up : 0.f;
    };
    // Segment `seg` of the sums to dW.  Warp: lane quarter; of two accumulators one per four warps, of one its column halves.
    auto drain = [&](int seg) {
      const int q = warp & 3, half = (warp - WG_FRONT) >> 2;
      const int n = n0 + (ACC == 2 ? 256 * half : 0) + 32 * q + lane;
      constexpr int COLS = ACC == 2 ? WG_BK : WG_BK / 2;
      const int cb = ACC == 2 ? 0 : half * COLS;           // first column of the warp
      if (!__all_sync(0xffffffffu, mbar_wait(acc_full, seg & 1, abort_flag, ST_TIMEOUT_EPILOGUE, 0xF40, budget))) { ok = false; return; }
      tc_fence_after();
      const uint32_t t = tmem_base + (ACC == 2 ? 256 * half : cb) + ((uint32_t)(q * 32) << 16);
      const bool add = p.accumulate || seg > 0;
      uint8_t* const box = smem + L::OUT + (warp - WG_FRONT) * 4096;
      float* o = p.out + (part * p.part_rows + n) * p.ldo + k0 + cb;
      if (seg > 0 && lane == 0) tma_store_wait_all<0>();   // the segment before is in memory
      for (int c0 = 0; c0 < COLS && k0 + cb + c0 < p.K; c0 += 32) {
        uint32_t v[32];
        __syncwarp();
        tmem_ld_32x32b_x32(t + c0, v);
        tmem_ld_wait(v);
        if constexpr (WINDOWS) {
          const float down = __uint_as_float((uint32_t)(254 - factor_exponent(cb + c0 < 128 ? tops[0] : tops[1])) << 23);
#pragma unroll
          for (int b = 0; b < 32; ++b) v[b] = __float_as_uint(__uint_as_float(v[b]) * down);
        }
        if (p.tma_out) {
          if (lane == 0) tma_store_wait_read<0>();         // the previous box has left the buffer
          __syncwarp();
#pragma unroll
          for (int pc = 0; pc < 8; ++pc)
            *reinterpret_cast<uint4*>(box + lane * 128 + ((pc ^ (lane & 7)) << 4)) = make_uint4(v[4 * pc], v[4 * pc + 1], v[4 * pc + 2], v[4 * pc + 3]);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            const int x = k0 + cb + c0, y = (int)(part * p.part_rows) + n;     // (lane 0's n: the warp's first row)
            if (add) tma_add_f32_2d(&tm_out, box, x, y);
            else tma_store_2d(&tm_out, box, x, y);
            tma_store_commit();
          }
        } else if (n < p.N) {
          float* oc = o + c0;
#pragma unroll
          for (int b = 0; b < 32; ++b)
            if (k0 + cb + c0 + b < p.K) oc[b] = add ? oc[b] + __uint_as_float(v[b]) : __uint_as_float(v[b]);
        }
      }
    };
    const uint32_t drained = mapa_shared(smem_u32(acc_empty), 0);
    static_assert(WG_SEG % WG_AHEAD == 0 && WG_AHEAD <= STAGES, "a segment is whole rounds of the loop below, and a round fits the ring");
    int s = 0, seg0 = 0; uint32_t ph = 0;                  // seg0: segments before the pass
    auto run_pass = [&](auto first_pass) {
      constexpr bool FIRST = decltype(first_pass)::value;
      if constexpr (WINDOWS) {
        top = rank == 0 ? tops[0] : tops[1];
        up = __uint_as_float((uint32_t)factor_exponent(top) << 23);
        if constexpr (!FIRST) {
          rewind();
#pragma unroll
          for (int a = 0; a < WG_AHEAD; ++a) fetch(step0 + a, raws[a], scs[a]);
          tc_fence_before();                               // the pass before has read its last sums
          __syncwarp();
          if (lane == 0) mbar_arrive_remote(drained);
        }
      }
      for (int i0 = step0; ok && i0 < step1; i0 += WG_AHEAD) {
        // (the next segment's first steps are in shared memory before: its MMAs start as soon as the sums are out)
        if (i0 - step0 > WG_SEG && (i0 - step0) % WG_SEG == WG_AHEAD) {
          drain(seg0 + (i0 - step0) / WG_SEG - 1);
          if (!ok) break;
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_remote(drained);
        }
#pragma unroll
        for (int a = 0; a < WG_AHEAD; ++a) {
          const int i = i0 + a;
          if (i >= step1) break;
          uint4 lo[2], hi[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) restore16<T>(raws[a][j], factor(scs[a][j]), lo[j], hi[j]);
          fetch(i + WG_AHEAD, raws[a], scs[a]);
          ok = __all_sync(0xffffffffu, mbar_wait<true>(&empty[s], ph ^ 1, abort_flag, ST_TIMEOUT_EPILOGUE, 0xF30 | s, budget));
          if (!ok) break;
          uint8_t* tile_b = smem + s * L::STAGE + L::A_BYTES + (c >> 2) * WG_CHUNK;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int row = r + 32 * j;
            uint8_t* line = tile_b + row * 128;
            *reinterpret_cast<uint4*>(line + (((pc + swap) ^ (row & 7)) << 4)) = swap ? hi[j] : lo[j];
            *reinterpret_cast<uint4*>(line + (((pc + 1 - swap) ^ (row & 7)) << 4)) = swap ? lo[j] : hi[j];
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive_remote(arrive_b + 8 * s);
          if (++s == STAGES) { s = 0; ph ^= 1; }
        }
      }
      // (the last segment; and the one before it, if this one was too short to come to that above)
      const int last = (step1 - step0 - 1) / WG_SEG;
      if (ok && last > 0 && step1 - step0 - last * WG_SEG <= WG_AHEAD) {
        drain(seg0 + last - 1);
        tc_fence_before();
        __syncwarp();
        if (ok && lane == 0) mbar_arrive_remote(drained);
      }
      if constexpr (WINDOWS && FIRST) {
        const bool any = __any_sync(0xffffffffu, outside != 0u);
        if (lane == 0) {
#pragma unroll
          for (uint32_t to = 0; to < 2; ++to) {
            const uint32_t bar = mapa_shared(smem_u32(missed_full), to);
            if (any) {
              red_max_cluster(mapa_shared(smem_u32(missed), to), 1);
              mbar_arrive_remote_release(bar);
            } else {
              mbar_arrive_remote_relaxed(bar);             // (nothing to order, and a release takes a microsecond)
            }
          }
        }
      }
      if (ok) drain(seg0 + last);
      seg0 += last + 1;
    };
    run_pass(std::true_type{});
    if constexpr (WINDOWS) {
      if (ok && __shfl_sync(0xffffffffu, missed_any(), 0) > 0) {
        int above = 0, below = 0;                          // (infinite and NaN scales have the greatest exponent, 255)
        rewind();
        for (int i = step0; i < step1; i += WG_AHEAD) {
#pragma unroll
          for (int a = 0; a < WG_AHEAD; ++a) fetch(i + a, raws[a], scs[a]);
#pragma unroll
          for (int a = 0; a < WG_AHEAD; ++a) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint4 q = raws[a][j];
              const int e = scale_exponent(scs[a][j]);
              if (scs[a][j] == 0.f || (e != 255 && ((q.x | q.y | q.z | q.w) & 0x7f7f7f7fu) == 0u)) continue;
              above = max(above, (e - top + WG_WINDOW - 1) / WG_WINDOW);
              below = max(below, (top - e) / WG_WINDOW);
            }
          }
        }
        above = __reduce_max_sync(0xffffffffu, above);
        below = __reduce_max_sync(0xffffffffu, below);
        if (lane == 0) {
          for (uint32_t to = 0; to < 2; ++to) {
            red_max_cluster(mapa_shared(smem_u32(missed + 1), to), above);
            red_max_cluster(mapa_shared(smem_u32(missed + 2), to), below);
            mbar_arrive_remote_release(mapa_shared(smem_u32(more_full), to));
          }
        }
        const int n = __shfl_sync(0xffffffffu, more_passes(), 0), up_to = n > 0 ? missed[1] : 0;
        for (int i = 1; ok && i <= n; ++i) {               // upwards, then from the first one downwards
          const int by = (i <= up_to ? 1 : i == up_to + 1 ? -1 - up_to : -1) * WG_WINDOW;
          tops[0] += by;
          tops[1] += by;
          run_pass(std::false_type{});
        }
      }
    }
    if (lane == 0) tma_store_wait_all<0>();
  }
  tc_fence_before();
  cluster_sync_all();                                      // neither CTA leaves while the other may still arrive at its barriers or its MMAs read here
  if (warp == 1) { tc_fence_after(); tmem_dealloc_pair(tmem_base, 256 * ACC); }
}

// dW = (dW +) the parts' sums, in order.  A thread's loads are what it waits for: eight parts' at a time, dW as vectors where its rows allow
// (accumulating, scalar by scalar / so: N = 2048 K = 512 M = 9001 29.8 / 28.5 us, N = 512 16.7 / 15.7).
__global__ void wgrad_reduce_kernel(const float* ws, long long ld, long long part_stride, int parts, float* out, long long ldo, int N, int K, int accumulate, int vec) {
  const int per_row = (K + 3) / 4;
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  pdl_wait();
  if (i >= (long long)N * per_row) return;
  const int n = (int)(i / per_row), k = (int)(i % per_row) * 4;
  const float* w = ws + (long long)n * ld + k;            // (the workspace's rows are padded to whole vectors)
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  int j = 0;
  for (; j + 8 <= parts; j += 8) {                        // eight parts' loads in flight
    float4 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = *reinterpret_cast<const float4*>(w + (j + u) * part_stride);
#pragma unroll
    for (int u = 0; u < 8; ++u) { a.x += v[u].x; a.y += v[u].y; a.z += v[u].z; a.w += v[u].w; }
  }
#pragma unroll 4
  for (; j < parts; ++j) {
    const float4 v = *reinterpret_cast<const float4*>(w + j * part_stride);
    a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
  }
  float* o = out + (long long)n * ldo + k;
  if (vec) {                                              // (dW's rows are whole aligned vectors)
    float4 d = accumulate ? *reinterpret_cast<const float4*>(o) : make_float4(0.f, 0.f, 0.f, 0.f);
    *reinterpret_cast<float4*>(o) = accumulate ? make_float4(d.x + a.x, d.y + a.y, d.z + a.z, d.w + a.w) : a;
    return;
  }
  const float e[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (k + u < K) o[u] = accumulate ? o[u] + e[u] : e[u];
}

// Accumulators per CTA, tiles, and the parts the batch is cut into: what fills the SMs with pairs, at least four steps each.  Two accumulators use
// the restored elements twice, but take half as many pairs for the same tiles and longer to write (us, K = 512, bf16, one / two accumulators: N = 2048
// M = 333 10.2 / 13.4, 3000 17.6 / 19.6, 9001 31.0 / 28.9, 65536 188 / 113; N = 512 M = 9001 15.9 / 19.5, 65536 54.4 / 43.0): two from 14 steps a part.  A function of the
// sizes alone: a workspace asked for before a device is chosen fits, and the sums have the same order everywhere.
constexpr int WG_FILL = 74;
static void wgrad_plan(long long M, int N, int K, int& acc, int& tiles, int& steps, int& parts, long long& ld, long long& part_rows) {
  const int kt = (K + WG_BK - 1) / WG_BK;
  steps = (int)((M + WG_BM - 1) / WG_BM);
  for (acc = N > 256 ? 2 : 1; ; acc = 1) {
    tiles = (N + 256 * acc - 1) / (256 * acc) * kt;
    parts = WG_FILL / tiles;
    if (parts > steps / 4) parts = steps / 4;
    if (parts < 1) parts = 1;
    if (acc == 1 || steps >= 14 * parts) break;
  }
  ld = ((long long)K + 7) / 8 * 8;
  part_rows = (long long)(N + 256 * acc - 1) / (256 * acc) * (256 * acc);      // (whole tiles: what lies behind N stays in its part)
}
static bool wgrad_shape_ok(long long M, int N, int K) {
  return M >= 0 && M <= 0x7fffff00ll && N > 0 && K > 0 && N <= (1 << 24) && K <= (1 << 24) &&
         (long long)((N + 255) / 256) * ((K + WG_BK - 1) / WG_BK) <= (1 << 24);
}
// What goes through the workspace: parts, and sums whose rows TMA could not write to a dW of their own width (us, M = 4096, N = 4096, K = 4095, written element by
// element by the kernel 184, so 130; M = 8300, N = 9704, K = 1001, fp16, in segments, 890 and 253).
static bool wgrad_by_workspace(int K, int parts) { return parts > 1 || K % 4 != 0; }
int64_t wgrad_workspace_bytes(long long M, int N, int K) {
  if (!wgrad_shape_ok(M, N, K)) return 0;
  int acc, tiles, steps, parts; long long ld, rows;
  wgrad_plan(M, N, K, acc, tiles, steps, parts, ld, rows);
  return wgrad_by_workspace(K, parts) ? 4 * ld * rows * parts : 0;
}

template <typename T, int ACC>
static cudaError_t launch_wg(const CUtensorMap& tm, const CUtensorMap& to, const WgParams& p, int dev, unsigned grid, cudaStream_t st) {
  static std::atomic<int> attr_done[64];
  auto k = wgrad_kernel<T, ACC>;
  if (!attr_done[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, WgSmem<ACC>::BYTES);
    if (e != cudaSuccess) return e;
    attr_done[dev].store(1, std::memory_order_release);
  }
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid); cfg.blockDim = dim3(WG_THREADS); cfg.dynamicSmemBytes = WgSmem<ACC>::BYTES; cfg.stream = st;
  cfg.attrs = attr; cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, k, tm, to, p);
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
  int acc;
  long long ld, rows;
  wgrad_plan(M, N, K, acc, p.tiles, p.steps, p.parts, ld, rows);
  const long long need = wgrad_workspace_bytes(M, N, K);
  if (need > 0 && (!ws || ws_bytes < need || (reinterpret_cast<uintptr_t>(ws) & 31))) return GSB200_ERR_BAD_ARG;
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return GSB200_ERR_DEVICE;
  CUtensorMap tm;
  if (!tmap_2d(&tm, dt == GSB200_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, dy, (uint64_t)M, (uint64_t)N,
               (uint64_t)lddy, 64, WG_BM, CU_TENSOR_MAP_SWIZZLE_128B)) return GSB200_ERR_BAD_ARG;
  p.q = q; p.ldq = ldq; p.s = s; p.lds = lds; p.M = M; p.N = N; p.K = K; p.k_tiles = (K + WG_BK - 1) / WG_BK;
  const bool cut = wgrad_by_workspace(K, p.parts);
  p.out = cut ? static_cast<float*>(ws) : dw; p.ldo = cut ? ld : lddw; p.part_rows = cut ? rows : 0;
  // (TMA writes whole 16-byte pieces)
  p.tma_out = cut || ((reinterpret_cast<uintptr_t>(dw) & 15) == 0 && lddw % 4 == 0 && K % 4 == 0);
  p.accumulate = cut ? 0 : accumulate;
  CUtensorMap to = tm;
  if (p.tma_out && !tmap_2d(&to, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, p.out, (uint64_t)(cut ? rows * p.parts : N), (uint64_t)(cut ? ld : K), (uint64_t)p.ldo, 32, 32,
                            CU_TENSOR_MAP_SWIZZLE_128B)) return GSB200_ERR_BAD_ARG;
  const long long grid = 2ll * p.tiles * p.parts;
  if (grid > 0x7fffffffll) return GSB200_ERR_BAD_ARG;
  const bool f16 = dt == GSB200_F16;
  cudaError_t e = acc == 2 ? (f16 ? launch_wg<__half, 2>(tm, to, p, dev, (unsigned)grid, st) : launch_wg<__nv_bfloat16, 2>(tm, to, p, dev, (unsigned)grid, st))
                           : (f16 ? launch_wg<__half, 1>(tm, to, p, dev, (unsigned)grid, st) : launch_wg<__nv_bfloat16, 1>(tm, to, p, dev, (unsigned)grid, st));
  if (e == cudaSuccess && cut) {
    const long long n4 = (long long)N * ((K + 3) / 4);
    const int vec = (reinterpret_cast<uintptr_t>(dw) & 15) == 0 && lddw % 4 == 0 && K % 4 == 0;
    e = launch_dependent(wgrad_reduce_kernel, (unsigned)((n4 + 255) / 256), 256, 0, st, static_cast<const float*>(ws), ld, rows * ld, p.parts, dw, lddw, N, K, accumulate, vec);
  }
  return cuda_status(e, "weight gradient launch");
}

}  // namespace gsb
