// bf16 rows to e4m3 rows with one fp32 scale each, plain (the weights and activations of an
// e4m3 product) or behind the residual addition and the RMSNorm that precede such a product.
//
//   r = bf16(x + y)                      the residual stream (r = x without y)
//   v = r * rsqrt(mean(r^2) + eps) * (weight + weight_offset)   (v = r for the plain quantiser)
//   scale = max(max|v|, 2^-64) / 448,  code = e4m3(v / scale)
//
// v, its sum of squares and its maximum are fp32; the codes are rounded from v itself, not from
// its bf16 copy (a bf16 step is 2^-8 of the value, an e4m3 one 2^-3, so going through bf16 would move
// codes that lie within 2^-9 of a rounding border).  The floor under the maximum keeps 1/scale
// finite: an all-zero row gets the smallest scale and zero codes.  A row with a NaN or an
// infinity, or whose sum of squares leaves fp32, gets a NaN scale and NaN codes (0x7F): the maximum
// is taken over the bit patterns of |v|, where infinities and NaNs order above every number.
//
// What bounds it: bytes (3 to 9 per element) at large T, launch latency at small T.  A block (or a
// warp) keeps its row in registers between the passes over it (sum of squares, maximum, codes).
// On a B200 (6.47 TB/s copies), back to back in a graph: 16384 x 2560 with y 50 us, 5.8 TB/s; 131072 x 2048 plain 115 us (134 us a
// call in a loop, 6.0 TB/s: the shorter time leaves a tenth of the stores in L2).
#include "kernels.h"
#include "q4t_device.cuh"

namespace q4t {

namespace {

constexpr float kE4m3Max = 448.0f;
constexpr float kMinAmax = 5.42101086242752217e-20f;  // 2^-64

// Four fp32 -> four e4m3 codes, round to nearest even, saturating; NaN gives 0x7F.
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  uint32_t r;
  asm("{ .reg .b16 lo, hi; cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1; cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3; "
      "mov.b32 %0, {lo, hi}; }"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}

// The codes of v / scale from ninv, minus the rounded 1 / scale: the product's error comes back as an exact remainder (Markstein's
// correction of a quotient).  Checked against the division for all 2^23 mantissas of scale around the rounding borders of e4m3: of the
// seven values of v next to a border the product alone puts 8 % on its wrong side, this none; bf16 rows lie on the borders often (four to
// seven codes in ten thousand differed).  The quotients are formed negated, Q = v * ninv, Q - (v + Q scale) / scale, and the codes' signs
// flipped back (flip: 0x80808080, or 0 in a row of NaNs): so an exact remainder, which is always +0, leaves the sign of a zero alone.
__device__ __forceinline__ uint32_t quotients4(const float* v, uint64_t scale2, uint64_t ninv2, uint32_t flip) {
  float q[4];
#pragma unroll
  for (int j = 0; j < 4; j += 2) {
    const uint64_t v2 = f32x2(v[j], v[j + 1]), q2 = mul2(v2, ninv2);
    f32x2_split(fma2(fma2(q2, scale2, v2), ninv2, q2), q[j], q[j + 1]);
  }
  return e4m3x4(q[0], q[1], q[2], q[3]) ^ flip;
}

// bf16(a + b) of a pair, added in fp32.
__device__ __forceinline__ uint32_t add_bf16x2(uint32_t a, uint32_t b) {
  return f32x2_to_bf16x2(bf16x2_lo(a) + bf16x2_lo(b), bf16x2_hi(a) + bf16x2_hi(b));
}

// WARPS: every warp of the block has a row of its own (no barriers); otherwise the block has one row.
template <bool NORM, int G, bool WARPS>
__global__ void __launch_bounds__(WARPS ? 256 : 1024, WARPS || NORM ? 1 : 2) fp8_rows_kernel(const Fp8RowsArgs a, int rows) {
  __shared__ float s_sum[32];
  __shared__ uint32_t s_max[32];
  chain_wait();
  const int n8 = a.hs >> 3, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nw = WARPS ? 1 : static_cast<int>(blockDim.x) >> 5;
  const int tid = WARPS ? lane : static_cast<int>(threadIdx.x), threads = WARPS ? 32 : static_cast<int>(blockDim.x);
  const size_t row = WARPS ? static_cast<size_t>(blockIdx.x) * (blockDim.x >> 5) + warp : blockIdx.x;
  if (WARPS && row >= static_cast<size_t>(rows)) return;
  const uint4* xr = reinterpret_cast<const uint4*>(a.x + row * a.hs);
  const uint4* yr = NORM && a.y ? reinterpret_cast<const uint4*>(a.y + row * a.hs) : nullptr;
  uint4* xo = NORM && a.x_out ? reinterpret_cast<uint4*>(a.x_out + row * a.hs) : nullptr;

  // everything the row needs is requested at once: x, y and the weights
  uint4 keep[G], add[NORM ? G : 1], weight[NORM ? G : 1];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int i = g * threads + tid;
    keep[g] = make_uint4(0, 0, 0, 0);
    if (i < n8) keep[g] = xr[i];
    if constexpr (NORM) {
      add[g] = weight[g] = make_uint4(0, 0, 0, 0);
      if (i < n8 && yr) add[g] = yr[i];
      if (i < n8 && a.weight) weight[g] = reinterpret_cast<const uint4*>(a.weight)[i];
    }
  }
  float rn = 1.0f;
  if constexpr (NORM) {
    float acc = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if (yr) {
        keep[g].x = add_bf16x2(keep[g].x, add[g].x);
        keep[g].y = add_bf16x2(keep[g].y, add[g].y);
        keep[g].z = add_bf16x2(keep[g].z, add[g].z);
        keep[g].w = add_bf16x2(keep[g].w, add[g].w);
      }
      const uint32_t u[4] = {keep[g].x, keep[g].y, keep[g].z, keep[g].w};
      float s = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s = fmaf(bf16x2_lo(u[j]), bf16x2_lo(u[j]), s);
        s = fmaf(bf16x2_hi(u[j]), bf16x2_hi(u[j]), s);
      }
      acc += s;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
    if (nw > 1) {
      if (lane == 0) s_sum[warp] = acc;
      __syncthreads();
      acc = lane < nw ? s_sum[lane] : 0.0f;
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
    }
    rn = __frsqrt_rn(__fdiv_rn(acc, static_cast<float>(a.hs)) + a.eps);
    if (!(acc <= 3.402823466e38f)) rn = __int_as_float(0x7fc00000);
    if (xo) {
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const int i = g * threads + tid;
        if (i < n8) xo[i] = keep[g];
      }
    }
  }

  float v[NORM ? G : 1][8];   // the plain quantiser unpacks its row where it needs it: registers are resident blocks
  uint32_t top = 0;
  auto unpack = [&](int g, float (&f)[8]) {
    const uint32_t u[4] = {keep[g].x, keep[g].y, keep[g].z, keep[g].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[2 * j] = bf16x2_lo(u[j]);
      f[2 * j + 1] = bf16x2_hi(u[j]);
    }
  };
  if constexpr (NORM) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      unpack(g, v[g]);
      const uint32_t w[4] = {weight[g].x, weight[g].y, weight[g].z, weight[g].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[g][2 * j] *= rn;
        v[g][2 * j + 1] *= rn;
        if (a.weight) {
          v[g][2 * j] *= bf16x2_lo(w[j]) + a.weight_offset;
          v[g][2 * j + 1] *= bf16x2_hi(w[j]) + a.weight_offset;
        }
      }
      if (g * threads + tid < n8) {   // past the row 0 * rn may be a NaN
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[g][j]) & 0x7fffffffu);
      }
    }
  } else {   // the bf16 patterns themselves, two at a time; past the row they are zeros
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const uint32_t u[4] = {keep[g].x, keep[g].y, keep[g].z, keep[g].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) top = __vmaxu2(top, u[j] & 0x7fff7fffu);
    }
    top = max(top & 0xffffu, top >> 16) << 16;
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (nw > 1) {
    if (lane == 0) s_max[warp] = top;
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, lane < nw ? s_max[lane] : 0u);
  }
  float scale = __fdiv_rn(fmaxf(__uint_as_float(top), kMinAmax), kE4m3Max);
  if (top >= 0x7f800000u) scale = __int_as_float(0x7fc00000);
  const uint32_t flip = top >= 0x7f800000u ? 0u : 0x80808080u;
  const float ninv = -__frcp_rn(scale);
  const uint64_t scale2 = f32x2(scale, scale), ninv2 = f32x2(ninv, ninv);
  if (tid == 0) a.scales[row] = scale;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int i = g * threads + tid;
    if (i < n8) {
      float(&f)[8] = v[NORM ? g : 0];
      if constexpr (!NORM) unpack(g, f);
      reinterpret_cast<uint2*>(a.codes + row * a.hs)[i] =
          make_uint2(quotients4(&f[0], scale2, ninv2, flip), quotients4(&f[4], scale2, ninv2, flip));
      if (NORM && a.h)
        reinterpret_cast<uint4*>(a.h + row * a.hs)[i] =
            make_uint4(f32x2_to_bf16x2(f[0], f[1]), f32x2_to_bf16x2(f[2], f[3]), f32x2_to_bf16x2(f[4], f[5]),
                       f32x2_to_bf16x2(f[6], f[7]));
    }
  }
}

template <bool NORM, int G>
cudaError_t launch_groups(const Fp8RowsArgs& a, bool warps, int rows, cudaStream_t stream) {
  if (warps)
    return launch_chained(fp8_rows_kernel<NORM, G, true>, dim3((static_cast<unsigned>(rows) + 7) / 8), dim3(256), 0, stream, a, rows);
  const unsigned threads = ((static_cast<unsigned>(a.hs) / 8 + G - 1) / G + 31) & ~31u;
  return launch_chained(fp8_rows_kernel<NORM, G, false>, dim3(static_cast<unsigned>(rows)), dim3(threads), 0, stream, a, rows);
}

template <bool NORM>
cudaError_t launch_rows(const Fp8RowsArgs& a, int rows, cudaStream_t stream) {
  // groups of eight elements a thread.  Few rows: one, the shortest chain of loads (one row of 2048: 1.8 us, four
  // groups 2.8).  Many rows: two, more bytes in flight without spending the registers that keep blocks resident (16384 x
  // 2560: 50 us, one group 57, four 65).  Short rows with a warp each: 100000 blocks of one row of 72 took 53 us, this 15.
  if (rows > 1024 && a.hs <= 256) return launch_groups<NORM, 1>(a, true, rows, stream);
  if (rows > 1024 && a.hs <= 512) return launch_groups<NORM, 2>(a, true, rows, stream);
  if constexpr (!NORM)   // 20000 x 1016: 10.8 us, a block each 12.5; the norm's x, y and weights would be 86 registers: 24.1, 21.3
    if (rows > 1024 && a.hs <= 1024) return launch_groups<NORM, 4>(a, true, rows, stream);
  if (rows <= 1024 && a.hs <= 8192) return launch_groups<NORM, 1>(a, false, rows, stream);
  if (a.hs <= 16384) return launch_groups<NORM, 2>(a, false, rows, stream);
  return launch_groups<NORM, 4>(a, false, rows, stream);
}

}  // namespace

cudaError_t launch_fp8_rows(const Fp8RowsArgs& a, bool norm, int rows, cudaStream_t stream) {
  if (rows <= 0 || a.hs <= 0 || a.hs % 8 || a.hs > kFp8RowsMaxHs) return cudaErrorInvalidValue;
  return norm ? launch_rows<true>(a, rows, stream) : launch_rows<false>(a, rows, stream);
}

}  // namespace q4t
