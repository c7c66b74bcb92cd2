// out[m, n] = round(act(acc * x_scale[m] * w_scale[n] + bias[n]) + residual[m, n]),
// acc = sum over k of x[m, k] * w[n, k] in fp32: a linear layer with everything behind the product in
// its epilogue (q4t_linear).  Operands both bf16 (tcgen05 kind::f16) or both e4m3 (kind::f8f6f4).
//
// The weight is the 128-row side of the MMA and up to 256 token rows are its columns, at every
// batch size: one token costs a 16-column MMA.
//
// Roles (one CTA per SM, persistent over the tiles): warp 0 streams 128-byte-wide k-blocks of both
// operands by TMA through a ring, warp 1 issues the MMAs into two accumulators in turn, warps 2-17 drain
// the finished one (four warps per quadrant of tensor-memory lanes, 32 columns each in turn) and store it.
// Rows and k past the ends of the operands are zeros from TMA; nothing is stored for them.
//
// On a B200 (copy 6.47 TB/s, cuBLAS bf16 1670 TFLOP/s in a burst and 1400 under the power cap): 16384 x 2048 x 2048 bf16 100 us
// (1370 TFLOP/s; 105 with a residual; cuBLAS without one 100), 122 under the power cap (cuBLAS 115 to 118); 8192^3 bf16 1254
// TFLOP/s under the cap (cuBLAS 1391); 8001 x 5120 x 2560 e4m3 89 us (2360 TFLOP/s; 98 with bias and GELU); 128 x 131072 x 2048 e4m3
// 56 us (5.4 TB/s), 66 repeated under the power cap; one token against 2048 x 2048 3.3 us (linear_row_kernel).
#include <cuda_fp16.h>

#include "kernels.h"
#include "q4t_device.cuh"

namespace q4t {

namespace {

// Epilogue warps: sixteen, or eight where each keeps 128 sums a lane (LONG below).
constexpr int lin_epi_warps(bool long_sums) { return long_sums ? 8 : 16; }
constexpr int lin_threads(bool long_sums) { return 64 + 32 * lin_epi_warps(long_sums); }
constexpr int kLinMaxStages = 8;
constexpr uint32_t kLinABytes = 128 * 128;
constexpr uint32_t kLinSmem = 220 * 1024;   // the operand ring at most

// Raised when a bounded wait of this kernel ran out (read and cleared by linear_timed_out).
__device__ int g_linear_timeout;

struct LinBars {
  uint64_t full[kLinMaxStages], empty[kLinMaxStages];
  uint64_t acc_full[2], acc_empty[2];
  uint32_t tmem_base;
  uint32_t abort_flag;
};

__device__ __forceinline__ void tc_mma_fp8(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{ .reg .pred p; setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p; }" ::"r"(d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tc_mma_fp8_pair(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                                uint32_t accumulate) {
  asm volatile(
      "{ .reg .pred p; setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p; }" ::"r"(d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ __half2 e4m3x2_to_half2(uint32_t two) {   // the low 16 bits; exact
  uint32_t r;
  asm("{ .reg .b16 lo, hi; mov.b32 {lo, hi}, %1; cvt.rn.f16x2.e4m3x2 %0, lo; }" : "=r"(r) : "r"(two));
  return *reinterpret_cast<const __half2*>(&r);
}

// Arrivals that hand an accumulator back.  Nothing in memory goes with them (the accumulator has been read when tcgen05.wait
// returns), and a releasing arrival waits until the warp's stores of the tile have landed: 6000 clocks a tile.
__device__ __forceinline__ void arrive_relaxed(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cta.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void arrive_relaxed_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// v * sigmoid(s), s = v (SiLU) or 2 sqrt(2/pi) (v + 0.044715 v^3) (GELU, 0.5 v (1 + tanh(s/2))), from exp(-|s|), times 2^7 while it is a
// number of its own: neither it nor the denominator, 1 .. 2, leaves fp32 before the result does.  (v / (1 + exp(-s)) by the fast division
// is 0 where 1 + exp(-s) is above 2^126: SiLU of -88, 5e-37.)  Two special-function operations an element, good to 2^-22, instead of a
// division routine, which cost more than the e4m3 mainloop of a K = 2560 tile.
template <int ACT>
__device__ __forceinline__ float activate(float v) {
  if (ACT != kLinSilu && ACT != kLinGelu) return v;
  const float u = ACT == kLinSilu ? v : fmaf(0.044715f * v * v, v, v);
  const float e = ex2(fmaf(-fabsf(u), ACT == kLinSilu ? 1.4426950408889634f : 2.302208198144325f, 7.0f));   // log2(e), 2 sqrt(2/pi) log2(e)
  return (v >= 0.0f ? v : v * e * 0.0078125f) * rcp(fmaf(e, 0.0078125f, 1.0f));
}

// The row's four values at a.residual + ..[m, n .. n + 3] as bf16 pairs; those past N read as zeros.
__device__ __forceinline__ uint2 residual4(const LinearArgs& a, int m, int n, int n_left, bool vec) {
  const uint16_t* p = a.residual + static_cast<size_t>(m) * a.ldr + n;
  if (vec) return *reinterpret_cast<const uint2*>(p);
  uint2 r = make_uint2(0, 0);
  if (n_left > 0) r.x = p[0];
  if (n_left > 1) r.x |= static_cast<uint32_t>(p[1]) << 16;
  if (n_left > 2) r.y = p[2];
  if (n_left > 3) r.y |= static_cast<uint32_t>(p[3]) << 16;
  return r;
}

// Finishes and stores out[m, n .. n + 3] (n_left of them exist).
template <bool FP8, int ACT>
__device__ __forceinline__ void finish4(const LinearArgs& a, int m, int n, int n_left, bool vec, float (&o)[4], float xs,
                                        const float (&ws)[4], const float (&bias)[4], uint2 res) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (FP8) o[i] = o[i] * xs * ws[i];   // in turn: the scales' product may leave fp32 where the result does not
    o[i] = activate<ACT>(o[i] + bias[i]);
  }
  o[0] += bf16x2_lo(res.x);
  o[1] += bf16x2_hi(res.x);
  o[2] += bf16x2_lo(res.y);
  o[3] += bf16x2_hi(res.y);
  const size_t at = static_cast<size_t>(m) * a.ldo + n;
  if (a.out_f32) {
    float* p = static_cast<float*>(a.out) + at;
    if (vec) {
      *reinterpret_cast<float4*>(p) = make_float4(o[0], o[1], o[2], o[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < n_left) p[i] = o[i];
    }
  } else {
    uint16_t* p = static_cast<uint16_t*>(a.out) + at;
    if (vec) {
      *reinterpret_cast<uint2*>(p) = make_uint2(f32x2_to_bf16x2(o[0], o[1]), f32x2_to_bf16x2(o[2], o[3]));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < n_left) p[i] = f32_to_bf16(o[i]);
    }
  }
}

// Where a tile lies: bands of kBand token tiles, in a band all weight tiles, token tiles first.  The tiles in flight then
// form a block of about 8 x 9 and share 17 tiles' operands through L2; token tiles straight through would keep the whole of
// x moving instead.
constexpr int kBand = 8;
__device__ __forceinline__ void tile_place(int tile, int m_tiles, int n_tiles, int& nt, int& mt) {
  const int band = tile / (kBand * n_tiles), first = band * kBand, high = min(kBand, m_tiles - first);
  const int in = tile - first * n_tiles;
  nt = in / high;
  mt = first + in - nt * high;
}

// One CTA per tile; or two CTAs of a cluster sharing a tile of 256 outputs (tcgen05 cta_group::2); or a cluster of
// up to eight CTAs sharing a tile's K.
//   kPair: each CTA loads its own 128 weight rows and half of the token rows, the leader issues the MMAs for both,
// each drains its own 128 accumulator lanes.  The leader owns the "full" and "accumulator empty" barriers; the MMAs'
// completion is signalled to both CTAs.
//   kSplit: few tiles and a long K (one token against a 2048 x 2048 weight is 16 tiles for 148 SMs).  Each CTA of the cluster
// accumulates its share of the k-blocks and stores the partial sums of outputs [r * 128 / split, ..) into CTA r's shared
// memory; behind a cluster barrier CTA r adds the shares in rank order (always the same order: deterministic, no
// atomics, no workspace) and finishes its outputs.
enum LinMode { kSingle = 0, kPair = 1, kSplit = 2 };
// LONG: the tensor cores add to their accumulator by truncation, for bf16 operands a bias of 1e-9 of the sum per element of K
// (4.4e-6 at K = 4096).  Where that shows, in fp32 outputs, the accumulator changes every kSegment k-blocks (768 elements: 7e-7)
// and the epilogue adds the segments in registers, rounding to nearest: eight warps with 128 sums a lane.  16384
// x 2048 x 2048 takes 138 us instead of 105, 128 x 131072 x 2048 106 instead of 97.  e4m3 products need fewer and exact steps (2.3e-7 at K = 4096).
constexpr int kSegment = 12;
template <bool FP8, int ACT, int MODE, bool LONG>
__global__ void __launch_bounds__(lin_threads(LONG), 1)
linear_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
              const __grid_constant__ LinearArgs a) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ LinBars bars;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile uint32_t* abort_flag = &bars.abort_flag;
  constexpr bool PAIR = MODE == kPair, SPLIT = MODE == kSplit;
  constexpr int kEpiWarps = lin_epi_warps(LONG);
  const uint32_t cta = MODE == kSingle ? 0u : cluster_cta_rank();   // rank in the cluster
  const uint32_t rank = PAIR ? cta : 0u;
  const bool leader = rank == 0;
  constexpr int kTileN = PAIR ? 256 : 128;
  [[maybe_unused]] const uint32_t red = smem_base + static_cast<uint32_t>(a.stages) * (kLinABytes + static_cast<uint32_t>(a.bn) * 128u);
  const int bn_load = PAIR ? a.bn >> 1 : a.bn;        // token rows this CTA loads
  const uint32_t stage_bytes = kLinABytes + static_cast<uint32_t>(bn_load) * 128u;
  const int nkb = (a.K * (FP8 ? 1 : 2) + 127) >> 7;   // k-blocks of 128 bytes
  const int n_tiles = (a.N + kTileN - 1) / kTileN, m_tiles = (a.M + a.bn - 1) / a.bn;
  const int tiles = n_tiles * m_tiles;
  const int per_tile = PAIR ? 2 : (SPLIT ? a.split : 1);
  const int first_tile = static_cast<int>(blockIdx.x) / per_tile;
  const int tile_step = static_cast<int>(gridDim.x) / per_tile;   // kSplit: one tile per cluster
  const int kb_begin = SPLIT ? static_cast<int>(cta) * nkb / a.split : 0;
  const int kb_end = SPLIT ? static_cast<int>(cta + 1) * nkb / a.split : nkb;

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(smem_u32(&bars.full[s]), 1);
      mbar_init(smem_u32(&bars.empty[s]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bars.acc_full[i]), 1);
      mbar_init(smem_u32(&bars.acc_empty[i]), PAIR ? 2 * kEpiWarps : kEpiWarps);
    }
    bars.abort_flag = 0;
    mbar_fence_init();
    prefetch_tmap(&tmap_w);
    prefetch_tmap(&tmap_x);
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(smem_u32(&bars.tmem_base), a.tmem_cols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_u32(&bars.tmem_base), a.tmem_cols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if constexpr (MODE != kSingle) cluster_sync(); else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem_base;
  chain_wait();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = first_tile; tile < tiles && ok; tile += tile_step) {
        int nt, mt;
        tile_place(tile, m_tiles, n_tiles, nt, mt);
        for (int kb = kb_begin; kb < kb_end; ++kb) {
          const uint32_t full = smem_u32(&bars.full[stage]), empty = smem_u32(&bars.empty[stage]);
          if (!mbar_wait(empty, phase ^ 1u, abort_flag)) {
            ok = false;
            break;
          }
          const uint32_t sa = smem_base + static_cast<uint32_t>(stage) * stage_bytes;
          const int kc = kb * (FP8 ? 128 : 64);
          const int wrow = nt * kTileN + static_cast<int>(rank) * 128, xrow = mt * a.bn + static_cast<int>(rank) * bn_load;
          if constexpr (PAIR) {
            const uint32_t sig = cluster_map(full, 0);
            if (leader) mbar_expect_tx(full, 2u * stage_bytes);
            tma_load_2d_pair(sa, &tmap_w, kc, wrow, sig);
            tma_load_2d_pair(sa + kLinABytes, &tmap_x, kc, xrow, sig);
          } else {
            mbar_expect_tx(full, stage_bytes);
            tma_load_2d(sa, &tmap_w, kc, wrow, full);
            tma_load_2d(sa + kLinABytes, &tmap_x, kc, xrow, full);
          }
          if (++stage == a.stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok) {
        atomicExch(&g_linear_timeout, 1);
        // no CTA leaves while its own copies are in flight (bounded as well; a pair's copies signal the leader,
        // and its CTAs leave together)
        for (int s = 0; leader && s < a.stages; ++s)
          for (uint32_t i = 0; i < (1u << 20) && !mbar_try_wait(smem_u32(&bars.full[s]), phase); ++i) {}
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && leader) {
      // M = 128 (pair: 256) weight rows, N = bn token rows, fp32 accumulation, both operands K-major
      const uint32_t idesc = (1u << 4) | (FP8 ? 0u : ((1u << 7) | (1u << 10))) | ((static_cast<uint32_t>(a.bn) >> 3) << 17) |
                             ((static_cast<uint32_t>(kTileN) >> 4) << 24);
      int stage = 0, it = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = first_tile; tile < tiles && ok; tile += tile_step) {
        for (int kb = kb_begin; kb < kb_end && ok; ++it) {   // one accumulator: a tile, or a segment of its K
          const int buf = it & 1, kb_first = kb, kb_stop = LONG ? min(kb + kSegment, kb_end) : kb_end;
          if (!mbar_wait(smem_u32(&bars.acc_empty[buf]), ((it >> 1) & 1u) ^ 1u, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d = tmem + static_cast<uint32_t>(buf) * a.bn;
          for (; kb < kb_stop; ++kb) {
            if (!mbar_wait(smem_u32(&bars.full[stage]), phase, abort_flag)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t sa = smem_base + static_cast<uint32_t>(stage) * stage_bytes;
            const uint64_t adesc = umma_desc_sw128(sa), bdesc = umma_desc_sw128(sa + kLinABytes);
#pragma unroll
            for (uint32_t u = 0; u < 4; ++u) {   // 32 bytes of K per instruction; past K both operands are zeros
              const uint32_t accumulate = kb != kb_first || u != 0;
              if constexpr (PAIR) {
                if (FP8) tc_mma_fp8_pair(d, adesc + 2u * u, bdesc + 2u * u, idesc, accumulate);
                else tc_mma_f16_pair(d, adesc + 2u * u, bdesc + 2u * u, idesc, accumulate);
              } else {
                if (FP8) tc_mma_fp8(d, adesc + 2u * u, bdesc + 2u * u, idesc, accumulate);
                else tc_mma_f16(d, adesc + 2u * u, bdesc + 2u * u, idesc, accumulate);
              }
            }
            if constexpr (PAIR) tc_commit_pair(smem_u32(&bars.empty[stage]), 3); else tc_commit(smem_u32(&bars.empty[stage]));
            if (++stage == a.stages) {
              stage = 0;
              phase ^= 1u;
            }
          }
          if (ok) {
            if constexpr (PAIR) tc_commit_pair(smem_u32(&bars.acc_full[buf]), 3); else tc_commit(smem_u32(&bars.acc_full[buf]));
          }
        }
      }
      if (!ok) atomicExch(&g_linear_timeout, 1);
    }
  } else {
    // A warp may touch the tensor-memory lanes of quadrant warp % 4.  It takes 32 columns (token rows) at a
    // time: a lane has one n of each, a 4x4 transpose among four lanes (four shuffles for four columns)
    // gives it four consecutive n of every fourth row, which is what it then loads and stores with
    // one 8- or 16-byte access (a warp: 64 or 128 bytes of four rows).
    const int quad = warp & 3, part = (warp - 2) >> 2;
    const int r4 = lane & 3, n4 = (lane >> 2) * 4;
    constexpr int kParts = kEpiWarps / 4, kChunks = 8 / kParts;   // chunks of 32 columns of a warp in one tile
    int it = 0;
    bool ok = true;
    for (int tile = first_tile; tile < tiles && ok; tile += tile_step) {
      int nt, mt;
      tile_place(tile, m_tiles, n_tiles, nt, mt);
      const int n = nt * kTileN + static_cast<int>(rank) * 128 + quad * 32 + n4;
      const int n_left = a.N - n;                       // of the lane's four outputs
      const bool vec = a.vec && n_left >= 4;
      float ws[4], bias[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ws[i] = !SPLIT && !LONG && FP8 && a.w_scale && i < n_left ? a.w_scale[n + i] : 1.0f;
        bias[i] = !SPLIT && !LONG && a.bias && i < n_left ? bf16_to_f32(a.bias[n + i]) : 0.0f;
      }
      const int m_base = mt * a.bn, cols = min(a.bn, a.M - m_base);
      // the tile's chunks of 32 columns of this warp: everything they read from memory is requested before
      // the wait for the accumulator and the first store (out may be residual)
      // (LONG reads its residual late: its registers are the sums')
      constexpr int kRead = LONG || SPLIT ? 1 : kChunks;
      float xs_lane[kRead];
      uint2 res[kRead][8];
#pragma unroll
      for (int h = 0; h < kRead; ++h) {
        const int c0 = part * 32 + h * (32 * kParts);
        xs_lane[h] = !SPLIT && FP8 && a.x_scale && c0 + lane < cols ? a.x_scale[m_base + c0 + lane] : 1.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int c = c0 + 4 * k + r4;
          res[h][k] = make_uint2(0, 0);
          if (!SPLIT && !LONG && a.residual && c < cols) res[h][k] = residual4(a, m_base + c, n, n_left, vec);
        }
      }
      uint32_t columns[LONG ? kChunks : 1][32];   // a chunk's columns of this lane; LONG: all chunks' sums over the segments so far
      for (int kb = kb_begin; kb < kb_end; kb += LONG ? kSegment : kb_end - kb_begin, ++it) {
        const int buf = it & 1;
        if (!mbar_wait(smem_u32(&bars.acc_full[buf]), (it >> 1) & 1u, abort_flag)) {
          if (lane == 0) atomicExch(&g_linear_timeout, 1);
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll
        for (int h = 0; h < kChunks; ++h) {
          const int c0 = part * 32 + h * (32 * kParts);
          if (c0 >= cols) break;
          const uint32_t tacc = tmem + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(buf * a.bn + c0);
          const bool wide = c0 + 16 < a.bn;
          uint32_t (&v)[32] = columns[LONG ? h : 0];
          if constexpr (LONG) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              uint32_t t[16];
              if (g == 0 || wide) tmem_ld16(tacc + 16u * g, t);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const float p = g == 0 || wide ? __uint_as_float(t[j]) : 0.0f;
                v[16 * g + j] = __float_as_uint(kb == kb_begin ? p : __uint_as_float(v[16 * g + j]) + p);
              }
            }
            if (kb + kSegment < kb_end) continue;
          } else {
            tmem_ld16(tacc, *reinterpret_cast<uint32_t (*)[16]>(&v[0]));
            if (wide) {
              tmem_ld16(tacc + 16u, *reinterpret_cast<uint32_t (*)[16]>(&v[16]));
            } else {
#pragma unroll
              for (int j = 16; j < 32; ++j) v[j] = 0;
            }
            tmem_ld_wait();
          }
          if constexpr (SPLIT) {
            // the 32 partial sums of this lane's output go to the CTA that finishes it
            const int rows = 128 / a.split, out_row = quad * 32 + lane, owner = out_row / rows;
            const uint32_t dst = cluster_map(red, static_cast<uint32_t>(owner)) +
                                 static_cast<uint32_t>((static_cast<int>(cta) * a.bn + c0) * rows + out_row - owner * rows) * 4u;
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (c0 + j < cols)
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(dst + static_cast<uint32_t>(j * rows) * 4u),
                             "r"(v[j])
                             : "memory");
          } else if constexpr (LONG) {
            // fp32 rows need no transpose: a column's 32 lanes are 128 consecutive bytes
            const int own = nt * kTileN + static_cast<int>(rank) * 128 + quad * 32 + lane;
            if (own < a.N) {
              const float b = a.bias ? bf16_to_f32(a.bias[own]) : 0.0f;
              float* out = static_cast<float*>(a.out) + static_cast<size_t>(m_base + c0) * a.ldo + own;
              const uint16_t* add = a.residual ? a.residual + static_cast<size_t>(m_base + c0) * a.ldr + own : nullptr;
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                if (c0 + j < cols) {
                  float o = activate<ACT>(__uint_as_float(v[j]) + b);
                  if (add) o += bf16_to_f32(add[j * a.ldr]);
                  out[j * a.ldo] = o;
                }
              }
            }
          } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const uint32_t* q = &v[4 * k];
              float o[4];
              {
                const bool odd = lane & 1, high = lane & 2;
                const uint32_t t0 = __shfl_xor_sync(0xffffffffu, odd ? q[0] : q[1], 1);
                const uint32_t t1 = __shfl_xor_sync(0xffffffffu, odd ? q[2] : q[3], 1);
                const uint32_t p0 = odd ? t0 : q[0], p1 = odd ? q[1] : t0, p2 = odd ? t1 : q[2], p3 = odd ? q[3] : t1;
                const uint32_t u0 = __shfl_xor_sync(0xffffffffu, high ? p0 : p2, 2);
                const uint32_t u1 = __shfl_xor_sync(0xffffffffu, high ? p1 : p3, 2);
                o[0] = __uint_as_float(high ? u0 : p0);
                o[1] = __uint_as_float(high ? u1 : p1);
                o[2] = __uint_as_float(high ? p2 : u0);
                o[3] = __uint_as_float(high ? p3 : u1);
              }
              const int c = c0 + 4 * k + r4;
              const float xs = FP8 ? __shfl_sync(0xffffffffu, xs_lane[h], 4 * k + r4) : 1.0f;
              if (c < cols) finish4<FP8, ACT>(a, m_base + c, n, n_left, vec, o, xs, ws, bias, res[h][k]);
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (PAIR) arrive_relaxed_cluster(cluster_map(smem_u32(&bars.acc_empty[buf]), 0));
          else arrive_relaxed(smem_u32(&bars.acc_empty[buf]));
        }
      }
    }
  }

  tc_fence_before();
  // neither CTA of a pair frees its tensor memory or leaves while the other may still touch it or its barriers; behind
  // this barrier the partial sums of a split tile are in place
  __syncwarp();
  if constexpr (MODE != kSingle) cluster_sync(); else __syncthreads();
  if constexpr (SPLIT) {
    int nt, mt;
    tile_place(first_tile, m_tiles, n_tiles, nt, mt);
    const int m_base = mt * a.bn, cols = min(a.bn, a.M - m_base);
    const int rows = 128 / a.split, groups = rows >> 2;
    for (int u = threadIdx.x; u < cols * groups; u += lin_threads(LONG)) {
      const int c = u / groups, g = (u - c * groups) * 4;
      const int n = nt * 128 + static_cast<int>(cta) * rows + g, n_left = a.N - n;
      if (n_left <= 0) continue;
      float o[4] = {0.0f, 0.0f, 0.0f, 0.0f}, ws[4], bias[4];
      for (int s = 0; s < a.split; ++s) {
        float p[4];
        asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];"
                     : "=f"(p[0]), "=f"(p[1]), "=f"(p[2]), "=f"(p[3])
                     : "r"(red + static_cast<uint32_t>((s * a.bn + c) * rows + g) * 4u)
                     : "memory");
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] += p[i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ws[i] = FP8 && a.w_scale && i < n_left ? a.w_scale[n + i] : 1.0f;
        bias[i] = a.bias && i < n_left ? bf16_to_f32(a.bias[n + i]) : 0.0f;
      }
      const bool vec = a.vec && n_left >= 4;
      finish4<FP8, ACT>(a, m_base + c, n, n_left, vec, o, FP8 && a.x_scale ? a.x_scale[m_base + c] : 1.0f, ws, bias,
                        a.residual ? residual4(a, m_base + c, n, n_left, vec) : make_uint2(0, 0));
    }
  }
  if (warp == 1) {
    __syncwarp();
    if constexpr (PAIR) tmem_dealloc_pair(tmem, a.tmem_cols); else tmem_dealloc(tmem, a.tmem_cols);
  }
}

// One token row without tensor cores: a warp takes R outputs and a share of K, requests kAhead pieces (16 bytes a lane)
// of each weight row and of the token row at once, and sums in fp32 in fixed order; the `ksplit` warps of a block that share
// outputs meet in shared memory.  Bound by the weight's bytes; at 2048 x 2048 by one memory round trip.
template <bool FP8, int R>
__global__ void __launch_bounds__(256) linear_row_kernel(const __grid_constant__ LinearRowArgs r) {
  constexpr int E = FP8 ? 16 : 8, kAhead = 8 / R;
  __shared__ float s_part[8][R];
  chain_wait();
  const LinearArgs& a = r.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int share = warp & (r.ksplit - 1), n0 = (blockIdx.x * (static_cast<int>(blockDim.x >> 5) / r.ksplit) + warp / r.ksplit) * R;
  const int full = a.K / E;   // whole pieces of a row
  auto widen = [](const uint4& v, float (&f)[E]) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (FP8) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float2 d = __half22float2(e4m3x2_to_half2(h ? u[j] >> 16 : u[j]));
          f[4 * j + 2 * h] = d.x;
          f[4 * j + 2 * h + 1] = d.y;
        }
      } else {
        f[2 * j] = bf16x2_lo(u[j]);
        f[2 * j + 1] = bf16x2_hi(u[j]);
      }
    }
  };
  const int64_t pitch = r.ldw * (FP8 ? 1 : 2);
  const uint8_t* const w0 = static_cast<const uint8_t*>(r.w) + n0 * pitch;
  // what the epilogue reads is requested with the operands: lane i of the first share finishes output n0 + i
  const int n = n0 + lane;
  const bool finishes = lane < R && share == 0 && n < a.N;
  const float xs = FP8 && finishes && a.x_scale ? a.x_scale[0] : 1.0f, ws = FP8 && finishes && a.w_scale ? a.w_scale[n] : 1.0f;
  const float bias = finishes && a.bias ? bf16_to_f32(a.bias[n]) : 0.0f;
  const float residual = finishes && a.residual ? bf16_to_f32(a.residual[n]) : 0.0f;
  float acc[R];
#pragma unroll
  for (int i = 0; i < R; ++i) acc[i] = 0.0f;
  for (int p0 = share * 32 + lane; p0 < full && n0 < a.N; p0 += 32 * r.ksplit * kAhead) {
    uint4 w[kAhead][R], x[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int p = p0 + 32 * r.ksplit * k;
      x[k] = p < full ? static_cast<const uint4*>(r.x)[p] : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < R; ++i)
        w[k][i] = p < full && n0 + i < a.N ? reinterpret_cast<const uint4*>(w0 + i * pitch)[p] : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      float xf[E];
      widen(x[k], xf);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        float wf[E];
        widen(w[k][i], wf);
#pragma unroll
        for (int j = 0; j < E; ++j) acc[i] = fmaf(wf[j], xf[j], acc[i]);
      }
    }
  }
  // the last K % E elements, one a lane of the first share
  const int k = full * E + lane;
  if (share == 0 && k < a.K) {
    auto one = [&](const void* row) {
      if constexpr (FP8) return __low2float(e4m3x2_to_half2(static_cast<const uint8_t*>(row)[k]));
      else return bf16_to_f32(static_cast<const uint16_t*>(row)[k]);
    };
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (n0 + i < a.N) acc[i] = fmaf(one(w0 + i * pitch), one(r.x), acc[i]);
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], off);
    if (r.ksplit > 1 && lane == 0) s_part[warp][i] = acc[i];
  }
  if (r.ksplit > 1) {
    __syncthreads();
    if (share != 0) return;
#pragma unroll
    for (int i = 0; i < R; ++i)
      for (int q = 1; q < r.ksplit; ++q) acc[i] += s_part[warp + q][i];
  }
  if (finishes) {
    float v = acc[0];
#pragma unroll
    for (int i = 1; i < R; ++i)
      if (lane == i) v = acc[i];
    if (FP8) v = v * xs * ws;   // in turn, see finish4
    v += bias;
    v = a.act == kLinSilu ? activate<kLinSilu>(v) : a.act == kLinGelu ? activate<kLinGelu>(v) : v;
    v += residual;
    if (a.out_f32) static_cast<float*>(a.out)[n] = v;
    else static_cast<uint16_t*>(a.out)[n] = f32_to_bf16(v);
  }
}

using LinearKernel = void (*)(CUtensorMap, CUtensorMap, LinearArgs);
template <bool FP8, int MODE, bool LONG>
LinearKernel linear_by_act(int act) {
  return act == kLinSilu ? linear_kernel<FP8, kLinSilu, MODE, LONG>
                         : act == kLinGelu ? linear_kernel<FP8, kLinGelu, MODE, LONG> : linear_kernel<FP8, 0, MODE, LONG>;
}
template <int MODE>
LinearKernel linear_by_sums(bool fp8, bool long_sums, int act) {
  return fp8 ? linear_by_act<true, MODE, false>(act)
             : long_sums ? linear_by_act<false, MODE, true>(act) : linear_by_act<false, MODE, false>(act);
}
LinearKernel linear_pick(bool fp8, bool long_sums, int mode, int act) {
  switch (mode) {
    case kPair: return linear_by_sums<kPair>(fp8, long_sums, act);
    case kSplit: return linear_by_sums<kSplit>(fp8, long_sums, act);
    default: return linear_by_sums<kSingle>(fp8, long_sums, act);
  }
}

}  // namespace

// Clusters of 2, 4 and 8 CTAs (one per SM) that can be resident at once, per device: clusters do not cross the
// boundaries between groups of SMs, so this is less than the SM count divided by the size (8: 14 on a B200 of 148 SMs).
int g_linear_clusters[16][4] = {};

cudaError_t linear_set_attributes() {
  cudaError_t e;
  for (int v = 0; v < 27; ++v)   // e4m3, bf16, bf16 in segments; modes; activations
    if ((e = cudaFuncSetAttribute(linear_pick(v % 3 == 0, v % 3 == 2, v / 3 % 3, v / 9), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  kLinSmem + 1024)) != cudaSuccess)
      return e;
  int dev = 0, n = 0;
  if ((e = cudaGetDevice(&dev)) != cudaSuccess) return e;
  for (int i = 1; i < 4 && dev >= 0 && dev < 16; ++i) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(1u << i);
    cfg.blockDim = dim3(lin_threads(false));
    cfg.dynamicSmemBytes = kLinSmem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1u << i;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, i == 1 ? linear_kernel<false, 0, kPair, false> : linear_kernel<false, 0, kSplit, false>, &cfg) ==
            cudaSuccess && n > 0)
      g_linear_clusters[dev][i] = n;
    else
      cudaGetLastError();   // the query is advisory
  }
  return cudaSuccess;
}

// How many clusters of 2^i CTAs run at once.
int linear_resident(int i, int num_sms) {
  int dev = 0;
  cudaGetDevice(&dev);
  const int most = num_sms >> i;
  return dev >= 0 && dev < 16 && g_linear_clusters[dev][i] > 0 && g_linear_clusters[dev][i] < most ? g_linear_clusters[dev][i] : most;
}

// The cheapest of the forms by what a k-block costs a CTA, measured on a B200 (microseconds): 0.25 for five tcgen05 issues and
// a barrier round trip (0.35 across a pair); its bytes at 105 GB/s per SM and 12.5 TB/s for all of them (L2); the MMAs; a
// launch is 4.2, joining a split tile 0.5 and 0.012 per token row.  At K = 2048, N = 2048, bf16 (form: us):
//   M = 1: split 4: 6.6, split 2: 8.7, single: 12.7 (split 8: 10.2, its 16 clusters do not fit at once);  M = 128: 64 rows a
//   tile, split 4: 7.8, 128 rows, split 4: 8.7, single 13.8;  M = 512: 128 rows, split 2: 12.4, single 14.2, pair 15.5;
//   M = 1024: 128 rows, single 14.6, pair 15.8;  M = 2048: pair 17.8, single 18.3.  128 x 131072 x 2048 e4m3: pair 54.9, single 68.
LinearPlan linear_plan(int M, int N, int K, bool fp8, bool out_f32, int num_sms) {
  const int nkb = (K * (fp8 ? 1 : 2) + 127) / 128;
  const bool long_sums = out_f32 && !fp8 && nkb > kSegment;
  const int least = (M + 255) / 256;
  const int resident[4] = {num_sms, linear_resident(1, num_sms), linear_resident(2, num_sms), linear_resident(3, num_sms)};
  LinearPlan best{};
  float best_us = 0.0f;
  for (int form = 0; form < 5; ++form) {           // split 1, 2, 4, 8, pair
    const bool pair = form == 4;
    const int i = pair ? 1 : form, split = pair ? 1 : 1 << form, ctas = 1 << i, step = pair ? 32 : 16;
    if (split > 1 && split * 2 > nkb) break;       // at least two k-blocks each
    if (pair && N <= 128) break;
    for (int cut = 1; cut <= 8; cut *= 2) {        // token rows in equal parts of at most 256, 128, ..
      const int64_t parts = static_cast<int64_t>(least) * cut;
      const int bn = static_cast<int>((M + parts - 1) / parts + step - 1) / step * step;
      const int64_t tiles = static_cast<int64_t>((N + (pair ? 255 : 127)) / (pair ? 256 : 128)) * ((M + bn - 1) / bn);
      const int64_t waves = (tiles + resident[i] - 1) / resident[i];
      if (split > 1 && waves > 1) break;
      // the partial sums take shared memory from the ring: one stage is left beside 256 token rows (5616 x 82 x 5856 e4m3: 21.6 us,
      // 128 rows and four stages 14.5)
      if (split > 1 && kLinSmem < 512u * static_cast<uint32_t>(bn) + 3u * (kLinABytes + 128u * static_cast<uint32_t>(bn))) continue;
      const float kb = static_cast<float>(nkb / split + (nkb % split != 0)), bytes = 16384.0f + 128.0f * static_cast<float>(pair ? bn / 2 : bn);
      const float running = static_cast<float>((tiles < resident[i] ? tiles : resident[i]) * ctas);
      float us = pair ? 0.35f : 0.25f;
      us = fmaxf(us, bytes * 9.5e-6f);
      us = fmaxf(us, bytes * running * 8.0e-8f);
      us = fmaxf(us, static_cast<float>(bn) * (pair ? 1.65e-3f : 1.4e-3f));
      us = 4.2f + static_cast<float>(waves) * kb * us + (split > 1 ? 0.5f + 0.012f * static_cast<float>(bn) : 0.0f);
      if (best_us == 0.0f || us < best_us) {
        best_us = us;
        best = LinearPlan{pair, long_sums, split, bn, pair ? bn / 2 : bn};
      }
      if (bn <= 32) break;
    }
  }
  return best;
}

// Where the row kernel beats the tensor cores (microseconds on a B200, row / tensor).  bf16: 2048 x 2048 3.5 / 7.1, 8192 x 2048
// 5.6 / 9.4, 2048 x 8192 5.9 / 13.4, 16384 x 2048 9.2 / 13.3, 32768 x 2048 29.0 / 26.8, 131072 x 2048 106 / 83.  e4m3: 2048 x 2048
// 3.0 / 6.2, 8192 x 2048 5.1 / 7.4, 2048 x 8192 5.4 / 9.4, 16384 x 2048 7.7 / 9.0, 32768 x 2048 14.2 / 14.1, 131072 x 2048 57 / 47.
bool linear_row_fits(int M, int N, int K) { return M == 1 && static_cast<int64_t>(N) * K < int64_t{1} << 26; }

cudaError_t launch_linear_row(const LinearRowArgs& args, bool fp8, cudaStream_t stream) {
  LinearRowArgs r = args;
  // Two outputs a warp share the token row's loads and conversions (e4m3, 4096 x 2048: 3.6 us, one 5.5; bf16 8192 x 2048 5.6, 6.1;
  // four hold too many registers: 5.6, 8.7), except where K is long and the outputs too few for the machine (512 x 16384 bf16: one
  // 4.1, two 5.2).  K is shared by more warps of a block as long as each has a full round of loads (half of one where
  // there are very few outputs) and the machine has room for them.
  const int64_t pieces = r.a.K / (fp8 ? 16 : 8);
  const bool two = r.a.N >= 1024 || pieces <= 1024;
  const int R = two ? 2 : 1;
  const int64_t groups = (static_cast<int64_t>(r.a.N) + R - 1) / R;
  r.ksplit = 1;
  while (r.ksplit < 8 && groups * r.ksplit < 4096 && pieces > (groups * r.ksplit < 1024 ? 64 : 128) * r.ksplit) r.ksplit *= 2;
  // four warps a block spread better over the SMs than eight (4096 x 2048 bf16: 3.95 us, 4.08)
  const int warps = r.ksplit == 8 ? 8 : 4, per_block = warps / r.ksplit * R;
  const dim3 grid((static_cast<unsigned>(r.a.N) + per_block - 1) / per_block);
  if (two)
    return fp8 ? launch_chained(linear_row_kernel<true, 2>, grid, dim3(32u * static_cast<unsigned>(warps)), 0, stream, r)
               : launch_chained(linear_row_kernel<false, 2>, grid, dim3(32u * static_cast<unsigned>(warps)), 0, stream, r);
  return fp8 ? launch_chained(linear_row_kernel<true, 1>, grid, dim3(32u * static_cast<unsigned>(warps)), 0, stream, r)
             : launch_chained(linear_row_kernel<false, 1>, grid, dim3(32u * static_cast<unsigned>(warps)), 0, stream, r);
}

cudaError_t launch_linear(const CUtensorMap& tmap_w, const CUtensorMap& tmap_x, const LinearArgs& args, const LinearPlan& plan,
                          bool fp8, int num_sms, cudaStream_t stream) {
  LinearArgs a = args;
  a.bn = plan.bn;
  a.split = plan.split;
  const int nkb = (a.K * (fp8 ? 1 : 2) + 127) / 128;
  const bool split = plan.split > 1;
  if (a.M <= 0 || a.N <= 0 || a.K <= 0 || a.bn < 16 || a.bn > 256 || (plan.long_sums && fp8) || a.bn % (plan.pair ? 32 : 16) || (split && plan.pair) ||
      plan.split < 1 || plan.split > 8 || 128 % plan.split || plan.split > nkb)
    return cudaErrorInvalidValue;
  const uint32_t stage = kLinABytes + static_cast<uint32_t>(plan.box_rows) * 128u;
  const uint32_t red = split ? 512u * static_cast<uint32_t>(a.bn) : 0u;   // partial sums of 128 / split outputs from each CTA
  a.stages = static_cast<int>((kLinSmem - red) / stage);
  if (a.stages > kLinMaxStages) a.stages = kLinMaxStages;
  if (split && a.stages > (nkb + plan.split - 1) / plan.split) a.stages = (nkb + plan.split - 1) / plan.split;
  a.tmem_cols = 32;
  while (a.tmem_cols < (split && !plan.long_sums ? 1u : 2u) * static_cast<uint32_t>(a.bn)) a.tmem_cols <<= 1;
  const int tile_n = plan.pair ? 256 : 128;
  const int64_t tiles = static_cast<int64_t>((a.N + tile_n - 1) / tile_n) * ((a.M + a.bn - 1) / a.bn);
  if (tiles * plan.split > (1 << 30)) return cudaErrorInvalidValue;
  const size_t smem = static_cast<size_t>(a.stages) * stage + red + 1024;
  const dim3 block(static_cast<unsigned>(lin_threads(plan.long_sums)));
  const LinearKernel kernel = linear_pick(fp8, plan.long_sums, plan.pair ? kPair : (split ? kSplit : kSingle), a.act);
  if (plan.pair) {
    int pairs = linear_resident(1, num_sms);
    if (tiles < pairs) pairs = static_cast<int>(tiles);
    return launch_chained_cluster(kernel, dim3(2u * static_cast<unsigned>(pairs)), block, smem, stream, 2, tmap_w, tmap_x, a);
  }
  if (split)
    return launch_chained_cluster(kernel, dim3(static_cast<unsigned>(tiles * plan.split)), block, smem, stream,
                                  static_cast<unsigned>(plan.split), tmap_w, tmap_x, a);
  return launch_chained(kernel, dim3(static_cast<unsigned>(tiles < num_sms ? tiles : num_sms)), block, smem, stream,
                        tmap_w, tmap_x, a);
}

// *out: did a launch of the kernels above give up on a bounded wait since the last call?
cudaError_t linear_timed_out(bool* out) {
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_linear_timeout, sizeof(v));
  if (e == cudaSuccess && v) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_linear_timeout, &zero, sizeof(zero));
  }
  *out = v != 0;
  return e;
}

}  // namespace q4t
