// Verification of drafted tokens (speculative sampling): which of a sequence's drafts stand under
// the target's distribution, and the token that follows them.
//
//   p_i = softmax(target row i / T), q_i = softmax(draft row i / T), or the single draft id itself
//   when there are no draft logits; draft i stands when u_i * q_i(x_i) < p_i(x_i) and every draft before it
//   stands; a = the first that does not (or the sequence's number of drafts)
//   r = max(p_a - q_a, 0) when draft a was refused (p_a itself where that leaves nothing: 2^-40 or less), p_a otherwise
//   token = the first t with r_0 + .. + r_t > u_n * sum(r)
//
// T <= 0 (or NaN) means greedy decoding: p is one at the row's first maximum, the drafts are taken as
// certain and the uniforms are not read.  NaN and -inf logits have no probability, +inf counts as the
// largest finite value.  A row without any probability refuses its draft and draws the token -1.
//
// Two kernels.  The first reads every row once, a warp per part of one or two 2-KB chunks, and leaves each part's
// maximum and sum of exponentials; they only decide acceptances, where an error of 1e-7 moves a border by as much, so
// the exponentials are fp32 and only their sums 64-bit.  The second draws, a cluster of CTAs per sequence: which
// token a uniform falls on hangs on a sum of up to V weights next to a border, and with V borders fp32 sums would
// miss one in a hundred draws, so the drawn row's weights, sums and differences are 64-bit throughout.
//
// On a B200, 32 sequences of 3 drafts over 131072 tokens, bf16 with draft logits (58.7 MB, 9.1 us at the copy rate): 35.5 us, 16 of
// them the first kernel; one sequence over 32003 tokens, fp32: 10.2 us, nearly all of it latency.
//
// One pass over the drawn row is enough although p - q needs both sums first: a weight is counted into
// P = sum of e^p and Q = sum of e^q over the tokens with p > q by the first kernel's sums (good to 1e-7), while the exact
// sums A and B of all e^p and e^q are formed beside them; then sum(r) = P / A - Q / B.  A token on the wrong side of the
// comparison has |p - q| <= d p, d the relative error of the first kernel's ratio of sums (1e-7), so no border of the draw is off by
// more than d, and where p / q spreads by much more than d by about d^2.  d is known once the exact sums are; where it is more
// than 2^-16 of what there is to draw from (distributions that agree to a percent, whose drafts are as rarely refused), a second pass
// compares with the exact ratio.  (Before that, rows that agreed to 1e-7 drew one token in ten wrongly; 0.2 to 0.5 us a call.)
#include <math_constants.h>

#include "kernels.h"
#include "q4t_device.cuh"

namespace q4t {

namespace {

constexpr int kStatThreads = 128;
constexpr int kDrawMaxWarps = 32;
constexpr int kDrawCtas = 8;   // most CTAs of a sequence
constexpr float kF32Max = 3.402823466e38f;
// A difference p - q that adds up to this (2^-40) or less is what 64-bit sums of equal distributions leave.
constexpr double kNothing = 9.094947017729282e-13;
// How far tokens on the wrong side of the comparison p > q may shift a border of the draw, relative to what is drawn from: 2^-16.
constexpr double kShift = 1.52587890625e-5;

// NaN -> -inf, +inf -> the largest finite value.
__device__ __forceinline__ float clean_logit(float l) { return fminf(fmaxf(l, -CUDART_INF_F), kF32Max); }

// log2(e) / T for a positive T, kept where products with logit differences cannot become 0 * inf.
__device__ __forceinline__ double inv_temperature(float T) {
  return fmin(fmax(CUDART_L2E / static_cast<double>(T), 1e-30), 1e30);
}
__device__ __forceinline__ bool is_greedy(const VerifyArgs& a, int b) { return a.temperature && !(a.temperature[b] > 0.0f); }
__device__ __forceinline__ float temperature_of(const VerifyArgs& a, int b) { return a.temperature ? a.temperature[b] : 1.0f; }
__device__ __forceinline__ int drafts_of(const VerifyArgs& a, int b) {
  return a.draft_len ? min(max(a.draft_len[b], 0), a.n) : a.n;
}

// A row of logits seen in 16-byte pieces that start at aligned addresses (a row may start anywhere).
template <bool F32>
struct Row {
  static constexpr int kE = F32 ? 4 : 8;
  const uint8_t* base;   // the row's first element rounded down to 16 bytes
  int skip, V;           // elements of piece 0 that lie before the row
  __device__ __forceinline__ Row(const void* logits, int64_t row, int64_t ld, int v) : V(v) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(logits) + static_cast<uintptr_t>(row * ld) * (F32 ? 4 : 2);
    skip = static_cast<int>(p & 15) / (F32 ? 4 : 2);
    base = reinterpret_cast<const uint8_t*>(p & ~static_cast<uintptr_t>(15));
  }
  __device__ __forceinline__ int pieces() const { return (skip + V + kE - 1) / kE; }
  __device__ __forceinline__ float one(int t) const {
    const size_t i = static_cast<size_t>(skip + t);
    return clean_logit(F32 ? reinterpret_cast<const float*>(base)[i] : bf16_to_f32(reinterpret_cast<const uint16_t*>(base)[i]));
  }
  __device__ __forceinline__ int first(int piece) const { return piece * kE - skip; }   // token of a piece's first element
  // Do `count` pieces from p on lie inside the row?  Then whole() reads them.
  __device__ __forceinline__ bool inside(int p, int count) const { return first(p) >= 0 && first(p + count) <= V; }
  __device__ __forceinline__ const uint4* whole(int p) const { return reinterpret_cast<const uint4*>(base) + p; }
  // The piece's bits; elements outside the row read as -inf.
  __device__ __forceinline__ uint4 piece(int p) const {
    const int t = first(p);
    if (t >= 0 && t + kE <= V) return reinterpret_cast<const uint4*>(base)[p];
    uint32_t u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (F32) {
        u[j] = t + j >= 0 && t + j < V ? reinterpret_cast<const uint32_t*>(base)[static_cast<size_t>(p) * 4 + j] : 0xff800000u;
      } else {
        u[j] = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int e = t + 2 * j + h;
          const uint32_t v = e >= 0 && e < V ? reinterpret_cast<const uint16_t*>(base)[static_cast<size_t>(p) * 8 + 2 * j + h] : 0xff80u;
          u[j] |= v << (16 * h);
        }
      }
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
  static __device__ __forceinline__ void unpack(const uint4& v, float (&l)[kE]) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (F32) {
        l[j] = __uint_as_float(u[j]);
      } else {
        l[2 * j] = bf16x2_lo(u[j]);
        l[2 * j + 1] = bf16x2_hi(u[j]);
      }
    }
  }
  // The kE logits from token first(p) on, cleaned; -inf outside the row.
  __device__ __forceinline__ int load(int p, float (&l)[kE]) const {
    unpack(piece(p), l);
#pragma unroll
    for (int j = 0; j < kE; ++j) l[j] = clean_logit(l[j]);
    return first(p);
  }
  // The kE elements that start s (1 .. kE - 1) elements into piece a, b the piece behind it.
  static __device__ __forceinline__ uint4 shifted(const uint4& a, const uint4& b, int s) {
    uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    const int words = F32 ? s : s >> 1;
    if (words & 2) {
#pragma unroll
      for (int j = 0; j < 6; ++j) u[j] = u[j + 2];
    }
    if (words & 1) {
#pragma unroll
      for (int j = 0; j < 5; ++j) u[j] = u[j + 1];
    }
    if (!F32 && (s & 1)) {
#pragma unroll
      for (int j = 0; j < 4; ++j) u[j] = __funnelshift_r(u[j], u[j + 1], 16);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
};

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

constexpr int kChunkLoads = 4;           // 16-byte loads of a lane in a chunk
constexpr float kLeastRef = -1048576.0f;  // a reference beyond this (either way) is not exact enough
template <bool F32>
constexpr int chunk_len() { return 32 * kChunkLoads * Row<F32>::kE; }   // logits of a chunk


// Maximum of a lane's logits; NaNs do not count.  bf16 pairs are compared as pairs.
template <bool F32, int N>
__device__ __forceinline__ float part_max(const uint4 (&raw)[N]) {
  if constexpr (F32) {
    float m = -CUDART_INF_F;
#pragma unroll
    for (int k = 0; k < N; ++k)
      m = fmaxf(fmaxf(m, fmaxf(__uint_as_float(raw[k].x), __uint_as_float(raw[k].y))),
                fmaxf(__uint_as_float(raw[k].z), __uint_as_float(raw[k].w)));
    return m;
  } else {
    auto pair = [](uint32_t v) { return *reinterpret_cast<const __nv_bfloat162*>(&v); };
    __nv_bfloat162 m = __hmax2(pair(raw[0].x), pair(raw[0].y));
#pragma unroll
    for (int k = 0; k < N; ++k) {
      if (k > 0) m = __hmax2(m, __hmax2(pair(raw[k].x), pair(raw[k].y)));
      m = __hmax2(m, __hmax2(pair(raw[k].z), pair(raw[k].w)));
    }
    return fmaxf(__low2float(m), __high2float(m));
  }
}

// Rows: the target's B * (n + 1) first, then the draft's B * n.  A warp walks through `chunks` chunks of a row (its part), a
// chunk's loads in flight while the one before is summed.  z = l c - R with c = log2(e) / T as two floats and R = fl(m c),
// m the largest logit that the lane has met: two fused steps an element (two elements an instruction), exact up to the
// rounding of z itself; a lane's sum is relative to 2^R and rescaled when m grows.  What this does not cover (NaN, +inf,
// nothing but masked logits, an R whose rounding is no longer a fraction of one) shows as a NaN, in R or in the maximum, and
// takes the careful loop, as greedy sequences do, which need the maximum's place instead.
// 224 rows of 131072 bf16 logits: 16 us, 3.7 TB/s.  The bytes take 9.1 us and one special-function operation a logit 6.5; the rest
// is start, the first loads' latency and the warps' joins.  Half of the exponentials as polynomials on the FMA pipe: 17.9 us.
template <bool F32>
__global__ void __launch_bounds__(kStatThreads) verify_stats_kernel(const VerifyArgs a, int parts, int chunks) {
  constexpr int E = Row<F32>::kE, kPieces = 32 * kChunkLoads;   // 16-byte pieces of a chunk
  chain_wait();
  chain_release_next();   // the draw's CTAs set up and read their drafts' logits while this kernel runs
  const int row = blockIdx.y, targets = a.B * (a.n + 1), lane = threadIdx.x & 31;
  const int part = blockIdx.x * (kStatThreads / 32) + (threadIdx.x >> 5);
  const bool target = row < targets;
  const int b = target ? row / (a.n + 1) : (row - targets) / a.n;
  const int i = target ? row - b * (a.n + 1) : row - targets - b * a.n;
  const bool greedy = is_greedy(a, b);
  if (part >= parts || (target ? i > drafts_of(a, b) : (i >= drafts_of(a, b) || greedy))) return;
  const Row<F32> r(target ? a.target : a.draft, target ? row : row - targets, target ? a.target_ld : a.draft_ld, a.V);
  const double c = greedy ? 1.0 : inv_temperature(temperature_of(a, b));
  const int p0 = part * chunks * kPieces + lane;
  // the remainder of c is positive, so that -inf stays -inf through both steps
  const float c_hi = __uint_as_float(__float_as_uint(__double2float_rz(c)) - 1u);
  const float c_lo = static_cast<float>(c - static_cast<double>(c_hi));

  VerifyPart out{-CUDART_INF_F, 0x7fffffff, 0.0, CUDART_NAN};
  bool careful = greedy;
  if (!greedy) {
    const uint64_t chi2 = f32x2(c_hi, c_hi), clo2 = f32x2(c_lo, c_lo);
    float m = -CUDART_INF_F, ref = kLeastRef;
    double sum = 0.0;
    auto fetch = [&](int chunk, uint4 (&v)[kChunkLoads]) {
      const int p = p0 + chunk * kPieces;
      if (chunk >= chunks) return;
      if (r.inside(p - lane, kPieces)) {
        const uint4* q = r.whole(p);
#pragma unroll
        for (int k = 0; k < kChunkLoads; ++k) v[k] = q[32 * k];
      } else {
#pragma unroll
        for (int k = 0; k < kChunkLoads; ++k) v[k] = r.piece(p + 32 * k);
      }
    };
    auto add = [&](const uint4 (&raw)[kChunkLoads]) {
      const float top = part_max<F32>(raw);
      if (top > m) {
        m = top;
        const float grown = fmaxf(m * c_hi, kLeastRef);
        sum *= static_cast<double>(ex2(ref - grown));
        ref = grown;
      }
      const uint64_t nref2 = f32x2(-ref, -ref);
      uint64_t s2[2] = {0, 0};
#pragma unroll
      for (int k = 0; k < kChunkLoads; ++k) {
        float l[E];
        r.unpack(raw[k], l);
#pragma unroll
        for (int j = 0; j < E; j += 2) {
          float z0, z1;
          const uint64_t l2 = f32x2(l[j], l[j + 1]);
          f32x2_split(fma2(l2, clo2, fma2(l2, chi2, nref2)), z0, z1);
          s2[k & 1] = add2(s2[k & 1], f32x2(ex2(z0), ex2(z1)));
        }
      }
      float s0, s1, s3, s4;
      f32x2_split(s2[0], s0, s1);
      f32x2_split(s2[1], s3, s4);
      sum += static_cast<double>((s0 + s1) + (s3 + s4));
    };
    uint4 even[kChunkLoads], odd[kChunkLoads];
    fetch(0, even);
#pragma unroll 1
    for (int chunk = 0; chunk < chunks; chunk += 2) {
      fetch(chunk + 1, odd);
      add(even);
      fetch(chunk + 2, even);
      if (chunk + 1 < chunks) add(odd);
    }
    float wm = m;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, off));
    const float wref = fmaxf(wm * c_hi, kLeastRef);
    sum *= static_cast<double>(ex2(ref - wref));
    sum = warp_sum(sum);
    out = VerifyPart{wm, 0x7fffffff, sum, wref};
    careful = !(sum >= 0.0 && sum <= 1e300 && wm < kF32Max && wref > kLeastRef && wref < -kLeastRef);
  }
  if (careful) {
    float best = -CUDART_INF_F;
    int at = 0x7fffffff;
#pragma unroll 1
    for (int k = 0; k < chunks * kChunkLoads; ++k) {
      float l[E];
      const int first = r.load(p0 + 32 * k, l);
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (l[j] > best) {
          best = l[j];
          at = first + j;
        }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, best, off);
      const int i2 = __shfl_xor_sync(0xffffffffu, at, off);
      if (m2 > best || (m2 == best && i2 < at)) {
        best = m2;
        at = i2;
      }
    }
    out = VerifyPart{best, at, 0.0, CUDART_NAN};
    if (!greedy && best > -CUDART_INF_F) {
      // relative to the maximum itself, differences first
      double sum = 0.0;
#pragma unroll 1
      for (int k = 0; k < chunks * kChunkLoads; ++k) {
        float l[E], s = 0.0f;
        r.load(p0 + 32 * k, l);
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const float d = fmaxf(l[j] - best, -kF32Max), z = d * c_hi;
          s += l[j] == -CUDART_INF_F ? 0.0f : exp2f(z < -1000.0f ? -1000.0f : fmaf(d, c_hi, d * c_lo));
        }
        sum += static_cast<double>(s);
      }
      out.sum = warp_sum(sum);
    }
  }
  if (lane == 0) a.parts[static_cast<size_t>(row) * parts + part] = out;
}

__device__ __forceinline__ double warp_scan(double v) {   // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const double o = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += o;
  }
  return v;
}

__constant__ double kRoots[16] = {   // 2^(i/16)
    1.0, 1.0442737824274138, 1.0905077326652577, 1.1387886347566916,
    1.189207115002721, 1.241857812073484, 1.2968395546510096, 1.3542555469368927,
    1.4142135623730951, 1.4768261459394993, 1.5422108254079407, 1.6104903319492543,
    1.681792830507429, 1.7562521603732995, 1.8340080864093424, 1.9152065613971474};

// 2^z for -1010 <= z <= 2: 2^(k/16) from a table of sixteen (one shared-memory word pair per bank pair: no
// conflicts) times the series of 2^r, |r| <= 1/32, to the fifth order (remainder below 1.5e-13 of the value, 2e-14 on
// average and nearly the same for all).  Ten 64-bit operations where the library's exp2 takes twice as many.
__device__ __forceinline__ double exp2_table(double z, const double* table) {
  const double magic = 6755399441055744.0;   // 1.5 * 2^52: rounds to an integer in the low word
  const double t = fma(z, 16.0, magic);
  const int k = __double2loint(t);
  const double r = fma(t - magic, -0.0625, z);
  double p = fma(r, 1.3333558146428443e-3, 9.618129107628477e-3);   // ln(2)^i / i!
  p = fma(p, r, 5.550410866482158e-2);
  p = fma(p, r, 2.402265069591007e-1);
  p = fma(p, r, 6.931471805599453e-1);
  // the table's entry i is 2^(i/16) with i * 2^16 taken from its high word: adding k * 2^16 puts k/16 into the exponent
  const double entry = table[k & 15], base = __hiloint2double(__double2hiint(entry) + (k << 16), __double2loint(entry));
  return fma(base * r, p, base);
}

__device__ __forceinline__ double exp2_low(double z, const double* table) { return z > -1000.0 ? exp2_table(z, table) : 0.0; }

// The weights 2^((l - ref) log2(e) / T) of one row, least 2^-1000: masked logits are raised to the one that gives it.  ref is
// the row's maximum, or 0 (see WeightTable).  Weights and sums of weights up to kTiny of the row's sum count as none (2^30
// of the least are below it).
constexpr double kTiny = 1.0e-265;   // about 2^-880
__device__ __forceinline__ double row_weight(float l, float ref, double c, const double* table) {
  const float v = clean_logit(l);
  const double z = (static_cast<double>(v) - static_cast<double>(ref)) * c;
  return v > -CUDART_INF_F && z > -1000.0 ? exp2_table(z, table) : 0.0;
}
struct RowWeights {
  double c, mc, cs;       // mc = ref c; cs = c * 2^896: a float's bits moved into a double's places are its value times 2^-896
  float m, ref, least;
  uint32_t m2, least2;    // the bounds as bf16 pairs
  bool regular;           // the bounds are exact bf16 values and near enough to 2^-1000
  __device__ __forceinline__ RowWeights(float top, float reference, double factor, bool f32)
      : c(factor), mc(static_cast<double>(reference) * factor), m(top), ref(reference) {
    cs = factor * 5.282945311356653e+269;
    const float low = reference - __fdividef(1000.0f, static_cast<float>(factor));
    least = f32 ? low : __bfloat162float(__float2bfloat16_ru(low));
    const double depth = (static_cast<double>(reference) - static_cast<double>(least)) * factor;
    // and the product's rounding, 2^-53 of m c in every weight alike, is nothing beside what a draw can see
    regular = depth > 920.0 && depth < 1001.0 && fabs(mc) < 4096.0 && fabsf(top) < 1e30f && factor > 1e-6 && factor < 1e6;
    m2 = f32x2_to_bf16x2(top, top);
    least2 = f32x2_to_bf16x2(least, least);
  }
  // any row, one logit at a time
  __device__ __forceinline__ double operator()(float l, const double* table) const { return row_weight(l, ref, c, table); }
  // the logits of one word of a regular row: E / 4 of them
  template <bool F32>
  __device__ __forceinline__ void word(uint32_t w, const double* table, double* e) const {
    if constexpr (F32) {
      const uint32_t u = __float_as_uint(fminf(fmaxf(__uint_as_float(w), least), m));   // NaN becomes the least
      e[0] = scaled(static_cast<int>(u) >> 3, static_cast<int>(u << 29), 0x8fffffffu, table);
    } else {
      auto pair = [](uint32_t v) { return *reinterpret_cast<const __nv_bfloat162*>(&v); };
      const __nv_bfloat162 v = __hmin2(__hmax2(pair(w), pair(least2)), pair(m2));
      const uint32_t u = *reinterpret_cast<const uint32_t*>(&v);
      e[0] = scaled(static_cast<int>(u << 16) >> 3, 0, 0x8fffe000u, table);
      e[1] = scaled(static_cast<int>(u) >> 3, 0, 0x8fffe000u, table);
    }
  }
  __device__ __forceinline__ double scaled(int hi, int lo, uint32_t mask, const double* table) const {
    return exp2_table(fma(__hiloint2double(static_cast<int>(static_cast<uint32_t>(hi) & mask), lo), cs, -mc), table);
  }
};

// The weights 2^(l log2(e) / T) of bf16 logits, looked up: one per value of either sign from 2^-12 up to 2^11, 47 KB of shared
// memory that hold for every row of the sequence.  Computing a weight takes 35 instructions, looking it up a dozen and the six
// cycles that 32 lanes at random places of shared memory cost.  Smaller magnitudes and NaN give a negative entry and are
// computed.  Logits below -2040 (masked ones) count as -2040, the least weight as long as 2^(-2040 c) is nothing beside the
// row's largest: see usable().
struct WeightTable {
  static constexpr int kLow = (115 << 7) - 1, kHigh = (138 << 7) - 1;   // bf16 bits: below 2^-12, 2040
  static constexpr int kEntries = 2 * (kHigh - kLow + 1);               // positive and negative values in turn
  static constexpr int kBytes = (kEntries + 23 * 48) * 8;               // with the factors that build() needs
  static __device__ __forceinline__ bool built(double c) { return c > 0.49 && c < 7.0; }   // 2040 c > 999, 128 c < 900
  static __device__ __forceinline__ bool usable(float m, double c) { return m < 128.0f && static_cast<double>(m) * c > -30.0; }
  // A value is (128 + 16 x + y) 2^(e - 7), so an entry is a product of one of 8 and one of 16 exponentials of its binary order e and
  // sign: 1104 exponentials instead of 5888.  Products that leave the range become zero, or infinite above any usable maximum.
  static constexpr int kOrders = 23, kFactors = kOrders * 48;   // of an order: 8 and 16, each of both signs
  template <int THREADS>
  static __device__ __forceinline__ void build(double* entries, double c, const double* table) {
    double* factors = entries + kEntries;
    for (int i = threadIdx.x; i < kFactors; i += THREADS) {
      const int order = i / 48, k = i - order * 48, n = k < 16 ? 128 + 16 * (k >> 1) : (k - 16) >> 1;
      const float mag = static_cast<float>(n) * __uint_as_float(static_cast<uint32_t>(127 - 12 - 7 + order) << 23);
      const double z = static_cast<double>(k & 1 ? -mag : mag) * c;
      factors[i] = exp2_table(fmin(fmax(z, -1000.0), 1000.0), table);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kEntries - 2; i += THREADS) {   // i: order, x, y, sign
      const double* f = factors + (i >> 8) * 48 + (i & 1);
      entries[i + 2] = f[(i >> 5 & 7) * 2] * f[16 + (i >> 1 & 15) * 2];
    }
    if (threadIdx.x < 2) entries[threadIdx.x] = -1.0;
  }
  // the weights of one word's two logits
  static __device__ __forceinline__ void look(uint32_t w, const double* entries, double (&e)[2]) {
    auto pair = [](uint32_t v) { return *reinterpret_cast<const __nv_bfloat162*>(&v); };
    const __nv_bfloat162 mag = __hmin2(__hmax2(__habs2(pair(w)), pair(kLow * 0x10001u)), pair(kHigh * 0x10001u));
    const uint32_t bits = *reinterpret_cast<const uint32_t*>(&mag) | (w & 0x80008000u);
    // a half's sign and magnitude doubled, then moved so that (magnitude, sign) is the entry's place in bytes
    const uint32_t lo = (__byte_perm(bits, 0, 0x1010) >> 12) & 0x7fff8u, hi = (__byte_perm(bits, 0, 0x3232) >> 12) & 0x7fff8u;
    const uint8_t* base = reinterpret_cast<const uint8_t*>(entries) - 16 * kLow;
    e[0] = *reinterpret_cast<const double*>(base + lo);
    e[1] = *reinterpret_cast<const double*>(base + hi);
  }
};

// a += x, b += y where `yes`: predicated sums (a conditional sum otherwise becomes four selects).
__device__ __forceinline__ void add_if(bool yes, double& a, double x, double& b, double y) {
  asm("{ .reg .pred p; setp.ne.s32 p, %4, 0; @p add.rn.f64 %0, %0, %2; @p add.rn.f64 %1, %1, %3; }"
      : "+d"(a), "+d"(b)
      : "d"(x), "d"(y), "r"(static_cast<int>(yes)));
}

struct DrawShared {
  VerifyPart p[kVerifyMaxDrafts + 1], q[kVerifyMaxDrafts];   // the sequence's rows
  double px[kVerifyMaxDrafts], ratio[kVerifyMaxDrafts];      // of draft i: its probability; the draft row's sum over the target row's
  uint8_t ok[kVerifyMaxDrafts];
  double table[16];
  double warp_sums[4][kDrawMaxWarps];                        // A, B, P, Q of each warp
  double all[2][kDrawCtas][4];                               // and of each CTA of the cluster, in either pass
  double lower, goal, sum, scale_q;                          // found by the first warp: see there
  int share, plain, again;
  int token;
  double prob;
};

__device__ __forceinline__ void st_cluster_f64(uint32_t addr, double v) {
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(v) : "memory");
}

// The sum over the eight lanes that differ in their lowest three bits.
__device__ __forceinline__ double sum8(double v) {
#pragma unroll
  for (int off = 1; off < 8; off <<= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// The four sums of a warp's tokens [t0, t1), token by token, with the exact scale of the draft row's weights.
struct Sums {
  double a, b, p, q;
};
template <bool F32>
__device__ __noinline__ Sums exact_sums(Row<F32> rp, Row<F32> rq, int t0, int t1, double c, float ref_p, float ref_q, double scale_q,
                                        const double* table) {
  Sums s{0.0, 0.0, 0.0, 0.0};
  for (int t = t0 + (threadIdx.x & 31); t < t1; t += 32) {
    const double ep = row_weight(rp.one(t), ref_p, c, table), eq = row_weight(rq.one(t), ref_q, c, table);
    s.a += ep;
    s.b += eq;
    if (ep > __dmul_rn(eq, scale_q)) {
      s.p += ep;
      s.q += eq;
    }
  }
  return s;
}

// A cluster of gridDim.x CTAs per sequence: join the parts (1.3 us), accept, one pass over the drawn row, exchange the sums
// through distributed shared memory (1.5 us), find CTA, warp and token (2.5 us).  The pass over 131072 bf16 tokens takes 9 us
// where p - q needs two rows and 5.5 where it does not: random shared-memory look-ups (6 cycles for 32) are 6.6 us of the 9; weights computed
// in 64 bits took 12.8 and 7.
template <bool F32, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) verify_draw_kernel(const VerifyArgs a, int parts) {
  constexpr int kDrawThreads = THREADS, kDrawWarps = THREADS / 32;
  constexpr bool TABLE = !F32 && THREADS == 1024;   // with 512 threads the table costs what it saves
  constexpr int E = Row<F32>::kE;
  __shared__ DrawShared sh;
  extern __shared__ double weight_entries[];   // TABLE: WeightTable::kEntries
  const int b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ctas = static_cast<int>(gridDim.x), cta = static_cast<int>(blockIdx.x);
  if (threadIdx.x < 16) {   // see exp2_table
    const double root = kRoots[threadIdx.x];
    sh.table[threadIdx.x] = __hiloint2double(__double2hiint(root) - (static_cast<int>(threadIdx.x) << 16), __double2loint(root));
  }
  if (threadIdx.x == 32) sh.token = -1;
  // what does not come from the first kernel is requested before the wait for it: each draft's logits, a thread per draft
  const int len = drafts_of(a, b), targets = a.B * (a.n + 1);
  const bool greedy = is_greedy(a, b);
  const double c = greedy ? 1.0 : inv_temperature(temperature_of(a, b));
  const bool has_q = a.draft != nullptr && !greedy;
  int x = -1;
  float lx = -CUDART_INF_F, lqx = -CUDART_INF_F, ux = 0.0f;
  if (static_cast<int>(threadIdx.x) < len) {
    const int64_t i = threadIdx.x;
    x = a.draft_ids[static_cast<size_t>(b) * a.n + i];
    ux = a.uniforms[static_cast<size_t>(b) * (a.n + 1) + i];
    if (x >= 0 && x < a.V) {
      lx = Row<F32>(a.target, static_cast<int64_t>(b) * (a.n + 1) + i, a.target_ld, a.V).one(x);
      if (has_q) lqx = Row<F32>(a.draft, static_cast<int64_t>(b) * a.n + i, a.draft_ld, a.V).one(x);
    }
  }
  const float u_draw = a.uniforms[static_cast<size_t>(b) * (a.n + 1) + a.n];
  __syncthreads();   // the table
  cluster_arrive();  // this CTA runs
  if (TABLE && !greedy && WeightTable::built(c)) WeightTable::build<THREADS>(weight_entries, c, sh.table);
  chain_wait();

  // the rows' parts joined, one warp per row: maximum and sum relative to it
  const int rows = (len + 1) + (has_q ? len : 0);
  for (int k = warp; k < rows; k += kDrawWarps) {
    const bool tgt = k <= len;
    const int i = tgt ? k : k - len - 1;
    const VerifyPart* part = a.parts + static_cast<size_t>(tgt ? b * (a.n + 1) + i : targets + b * a.n + i) * parts;
    float m = -CUDART_INF_F;
    int at = 0x7fffffff;
    double sum = 0.0;
    for (int s0 = 0; s0 < parts; s0 += 128) {   // 128 parts at a time, four a lane, joined to what the lane has
      VerifyPart v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int s = s0 + 32 * k + lane;
        v[k] = s < parts ? part[s] : VerifyPart{-CUDART_INF_F, 0x7fffffff, 0.0, 0.0};
      }
      float top = m;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (v[k].m > top || (v[k].m == top && v[k].at < at)) {
          top = v[k].m;
          at = v[k].at;
        }
      if (!greedy && top > -CUDART_INF_F) {
        const double tc = static_cast<double>(top) * c;
        if (m < top) sum *= m > -CUDART_INF_F ? exp2_low(static_cast<double>(m) * c - tc, sh.table) : 0.0;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (v[k].sum > 0.0) sum += v[k].sum * exp2_low((isnan(v[k].ref) ? static_cast<double>(v[k].m) * c : v[k].ref) - tc, sh.table);
      }
      m = top;
    }
    const float own = m;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, m, off);
      const int i2 = __shfl_xor_sync(0xffffffffu, at, off);
      if (m2 > m || (m2 == m && i2 < at)) {
        m = m2;
        at = i2;
      }
    }
    if (own < m) sum *= own > -CUDART_INF_F ? exp2_low((static_cast<double>(own) - static_cast<double>(m)) * c, sh.table) : 0.0;
    sum = warp_sum(sum);
    if (lane == 0) (tgt ? sh.p[i] : sh.q[i]) = VerifyPart{m, at, sum, 0.0};
  }
  __syncthreads();

  // acceptance, one thread per draft
  if (static_cast<int>(threadIdx.x) < len) {
    const int i = threadIdx.x;
    auto prob = [&](float l, const VerifyPart& st) {
      const double z = (static_cast<double>(l) - static_cast<double>(st.m)) * c;
      return l > -CUDART_INF_F && st.m > -CUDART_INF_F && z > -1000.0 ? exp2_table(z, sh.table) / st.sum : 0.0;
    };
    double px, qx = 1.0;
    if (greedy) {
      px = x >= 0 && x == sh.p[i].at ? 1.0 : 0.0;
    } else {
      px = prob(lx, sh.p[i]);
      if (has_q) {
        qx = prob(lqx, sh.q[i]);
        sh.ratio[i] = sh.q[i].sum / sh.p[i].sum;
      }
    }
    sh.px[i] = px;
    sh.ok[i] = greedy ? px > 0.0 : static_cast<double>(ux) * qx < px;
  }
  __syncthreads();
  cluster_wait();   // every CTA of the cluster runs: its shared memory may be written
  int at = 0;
  while (at < len && sh.ok[at]) ++at;

  // the draw
  const VerifyPart st = sh.p[at];
  int token = -1;
  double prob = 0.0;
  bool mine = cta == 0;   // this CTA writes the sequence's outputs
  if (st.m > -CUDART_INF_F && greedy) {
    token = st.at;
    prob = 1.0;
  } else if (st.m > -CUDART_INF_F) {
    const Row<F32> rp(a.target, static_cast<int64_t>(b) * (a.n + 1) + at, a.target_ld, a.V);
    const bool refused = at < len;
    const bool minus_q = refused && has_q && sh.q[at].m > -CUDART_INF_F;
    const Row<F32> rq(minus_q ? a.draft : a.target, minus_q ? static_cast<int64_t>(b) * a.n + at : 0,
                      minus_q ? a.draft_ld : a.target_ld, a.V);
    const int without = refused && !has_q ? a.draft_ids[static_cast<size_t>(b) * a.n + at] : -1;
    const float mq = minus_q ? sh.q[at].m : st.m;
    const bool looked = TABLE && WeightTable::built(c) && WeightTable::usable(st.m, c) && WeightTable::usable(mq, c);
    const RowWeights wp(st.m, looked ? 0.0f : st.m, c, F32), wq(mq, looked ? 0.0f : mq, c, F32);    // p > q by the first kernel's sums: e^p * ratio > e^q
    double ratio = minus_q ? sh.ratio[at] : 0.0;
    if (looked) ratio *= exp2_table((static_cast<double>(mq) - static_cast<double>(st.m)) * c, sh.table);

    // this warp's share: consecutive pieces of the target's row
    const int pieces = rp.pieces(), shares = ctas * kDrawWarps;
    const int per = (pieces + shares - 1) / shares;
    const int first_piece = min((cta * kDrawWarps + warp) * per, pieces), end_piece = min(first_piece + per, pieces);
    double sa = 0.0, sb = 0.0, sp = 0.0, sq = 0.0;
    // a piece of the target's row and the same tokens of the draft's, which may lie `shift` elements into two pieces
    const int apart = rq.skip - rp.skip, step = apart < 0 ? -1 : 0, shift = apart - step * E;
    auto pass = [&](auto weights_p, auto weights_q) {
      for (int p = first_piece + lane; p < end_piece; p += 32) {
        const int p0 = p - lane;
        const bool in = rp.inside(p0, 32) && (!minus_q || rq.inside(p0 + step, 33));
        const uint4 vp = in ? *rp.whole(p) : rp.piece(p);
        const uint32_t up[4] = {vp.x, vp.y, vp.z, vp.w};
        if (minus_q) {
          uint4 vq = in ? *rq.whole(p + step) : rq.piece(p + step);
          if (shift != 0) vq = Row<F32>::shifted(vq, in ? *rq.whole(p + step + 1) : rq.piece(p + step + 1), shift);
          const uint32_t uq[4] = {vq.x, vq.y, vq.z, vq.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            double ep[E / 4], eq[E / 4];
            weights_p(up[k], ep);
            weights_q(uq[k], eq);
#pragma unroll
            for (int j = 0; j < E / 4; ++j) {
              sa += ep[j];
              sb += eq[j];
              add_if(__double2hiint(fma(ep[j], ratio, -eq[j])) > 0, sp, ep[j], sq, eq[j]);   // the sign, without a 64-bit comparison
            }
          }
        } else {
          double own = 0.0;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            double ep[E / 4];
            weights_p(up[k], ep);
#pragma unroll
            for (int j = 0; j < E / 4; ++j) own += ep[j];
          }
          sa += own;
          const int first = rp.first(p);
          if (without >= first && without < first + E) {   // the piece of the token that is left out
            own = 0.0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              double ep[E / 4];
              weights_p(up[k], ep);
#pragma unroll
              for (int j = 0; j < E / 4; ++j)
                if (first + k * (E / 4) + j != without) own += ep[j];
            }
          }
          sp += own;
        }
      }
    };
    bool done = false;
    if constexpr (TABLE) {
      if (looked && wp.regular && wq.regular) {
        auto weights = [&](const RowWeights& row, uint32_t w, double (&e)[E / 4]) {
          WeightTable::look(w, weight_entries, e);
          if ((__double2hiint(e[0]) | __double2hiint(e[1])) < 0) row.template word<F32>(w, sh.table, e);
        };
        pass([&](uint32_t w, double (&e)[E / 4]) { weights(wp, w, e); }, [&](uint32_t w, double (&e)[E / 4]) { weights(wq, w, e); });
        done = true;
      }
    }
    if (done) {
    } else if (wp.regular && wq.regular) {
      pass([&](uint32_t w, double* e) { wp.template word<F32>(w, sh.table, e); },
           [&](uint32_t w, double* e) { wq.template word<F32>(w, sh.table, e); });
    } else {
      auto careful = [&](const RowWeights& row, uint32_t w, double* e) {
        if constexpr (F32) {
          e[0] = row(__uint_as_float(w), sh.table);
        } else {
          e[0] = row(bf16x2_lo(w), sh.table);
          e[1] = row(bf16x2_hi(w), sh.table);
        }
      };
      pass([&](uint32_t w, double* e) { careful(wp, w, e); }, [&](uint32_t w, double* e) { careful(wq, w, e); });
    }
    // The share (one a lane) that `goal` falls into, with what lies before it; rounding may leave the goal behind the last
    // share that holds anything.
    auto find = [&](double w, double upto, double goal, double none, double& lower) {
      const unsigned some = __ballot_sync(0xffffffffu, w > none), over = __ballot_sync(0xffffffffu, w > none && upto > goal);
      const int k = over ? __ffs(over) - 1 : (some ? 31 - __clz(some) : 0);
      lower = __shfl_sync(0xffffffffu, upto - w, k);
      return k;
    };
    // one turn, and in rare cases a second with the exact sums' ratio: see kShift
#pragma unroll 1
    for (int turn = 0;; ++turn) {
      sa = warp_sum(sa);
      sb = warp_sum(sb);
      sp = warp_sum(sp);
      sq = warp_sum(sq);
      if (lane == 0) {
        sh.warp_sums[0][warp] = sa;
        sh.warp_sums[1][warp] = sb;
        sh.warp_sums[2][warp] = sp;
        sh.warp_sums[3][warp] = sq;
      }
      __syncthreads();
      if (warp < 4) {   // a sum each, to every CTA
        const double t = warp_sum(lane < kDrawWarps ? sh.warp_sums[warp][lane] : 0.0);
        if (lane < ctas) st_cluster_f64(cluster_map(smem_u32(&sh.all[turn][cta][warp]), static_cast<uint32_t>(lane)), t);
      }
      __syncwarp();
      cluster_sync();
      if (warp == 0) {   // the first warp of every CTA adds the CTAs' shares in the same order, a lane per share
        const int c8 = lane & (kDrawCtas - 1);
        const bool have_cta = c8 < ctas;
        const double ka = have_cta ? sh.all[turn][c8][0] : 0.0, kb = have_cta ? sh.all[turn][c8][1] : 0.0;
        const double kp = have_cta ? sh.all[turn][c8][2] : 0.0, kq = have_cta ? sh.all[turn][c8][3] : 0.0;
        const double A = sum8(ka), B = sum8(kb), P = sum8(kp), Q = sum8(kq);
        // everything in the measure of the target's weights, whose sum is A
        const double scale_q = minus_q ? A / B : 0.0, none = kTiny * A;
        const bool plain = !(P - Q * scale_q > kNothing * A);   // the difference leaves nothing: the target's own distribution
        auto mass = [&](double wa, double wp_, double wq_) { return plain ? wa : fmax(wp_ - wq_ * scale_q, 0.0); };
        const double wk = lane < ctas ? mass(ka, kp, kq) : 0.0, upto = warp_scan(wk);
        const double goal = static_cast<double>(u_draw) * __shfl_sync(0xffffffffu, upto, 31);
        const bool again = turn == 0 && minus_q && fabs(ratio * scale_q - 1.0) * A > kShift * (P - Q * scale_q);
        double lower;
        int share = -1;
        if (find(wk, upto, goal, none, lower) == cta) {
          const double ww = lane < kDrawWarps ? mass(sh.warp_sums[0][lane], sh.warp_sums[2][lane], sh.warp_sums[3][lane]) : 0.0;
          share = find(ww, lower + warp_scan(ww), goal, none, lower);
        }
        if (lane == 0) {
          sh.share = share;
          sh.plain = plain;
          sh.lower = lower;
          sh.goal = goal;
          sh.sum = A;
          sh.scale_q = scale_q;
          sh.again = again;
        }
      }
      __syncthreads();
      if (!sh.again) break;
      const Sums sums = exact_sums<F32>(rp, rq, max(rp.first(first_piece), 0), min(rp.first(end_piece), a.V), c, wp.ref, wq.ref, sh.scale_q, sh.table);
      sa = sums.a;
      sb = sums.b;
      sp = sums.p;
      sq = sums.q;
    }
    const int share = sh.share;
    mine = share >= 0;
    if (mine) {
      const bool plain = sh.plain != 0;
      const double lower = sh.lower, goal = sh.goal, A = sh.sum, scale_q = sh.scale_q, none = kTiny * A;
      // token by token within the share, with the exact sums: each warp a run of consecutive tokens
      const int s0 = min((cta * kDrawWarps + share) * per, pieces), s1 = min(s0 + per, pieces);
      const int t0 = max(rp.first(s0), 0), t1 = min(rp.first(s1), a.V);
      const int run = (t1 - t0 + kDrawWarps - 1) / kDrawWarps;
      const int r0 = t0 + warp * run, r1 = min(r0 + run, t1);
      auto token_weight = [&](int t, double& p) {   // p: the target's probability
        p = wp(rp.one(t), sh.table);
        if (plain) return p;
        if (minus_q) return fmax(p - __dmul_rn(wq(rq.one(t), sh.table), scale_q), 0.0);
        return t == without ? 0.0 : p;
      };
      double w = 0.0, mine_w = 0.0, mine_p = 0.0;
      for (int t = r0 + lane; t < r1; t += 32) {
        mine_w = token_weight(t, mine_p);   // kept for the last token: the only one where a run is at most a warp long
        w += mine_w;
      }
      w = warp_sum(w);
      if (lane == 0) sh.warp_sums[0][warp] = w;
      __syncthreads();
      // the run, then the token: one warp
      const double wr = lane < kDrawWarps ? sh.warp_sums[0][lane] : 0.0;
      double upto;
      if (find(wr, lower + warp_scan(wr), goal, none, upto) == warp) {
        for (int tb = r0; tb < r1; tb += 32) {
          const int t = tb + lane;
          double own = 0.0, p = 0.0;
          if (t < r1) {
            if (run <= 32) {
              own = mine_w;
              p = mine_p;
            } else {
              own = token_weight(t, p);
            }
          }
          const double scan = upto + warp_scan(own);
          const unsigned some = __ballot_sync(0xffffffffu, own > none), over = __ballot_sync(0xffffffffu, own > none && scan > goal);
          // the first that crosses; the last with a weight stands in where rounding leaves the goal behind all of them
          const int k = over ? __ffs(over) - 1 : (some ? 31 - __clz(some) : -1);
          if (lane == k) {
            sh.token = t;
            sh.prob = p / A;
          }
          if (over) break;
          upto = __shfl_sync(0xffffffffu, scan, 31);
        }
      }
      __syncthreads();
      token = sh.token;
      if (token >= 0) prob = sh.prob;
    }
  }
  if (!mine) return;

  int32_t* out = a.tokens + static_cast<size_t>(b) * (a.n + 1);
  for (int i = threadIdx.x; i <= a.n; i += kDrawThreads) {
    out[i] = i < at ? a.draft_ids[static_cast<size_t>(b) * a.n + i] : (i == at ? token : -1);
    if (a.probs)
      a.probs[static_cast<size_t>(b) * (a.n + 1) + i] =
          static_cast<float>(i < at ? sh.px[i] : (i == at ? prob : 0.0));
  }
  if (threadIdx.x == 0) a.accepted[b] = at;
}

template <bool F32>
cudaError_t launch(const VerifyArgs& a, cudaStream_t stream) {
  const unsigned rows = static_cast<unsigned>(a.B) * static_cast<unsigned>(a.n + 1 + (a.draft ? a.n : 0));
  // Two consecutive chunks of a row to a warp where every SM still has its warps then (224 rows of 131072: one 18.6 us, two
  // 16.0, four 17, eight 19.7: long parts leave the memory system with scattered streams).  A row may start inside a 16-byte
  // piece and reach into one more than its length needs.
  const int all = static_cast<int>((static_cast<int64_t>(a.V) + 8 + chunk_len<F32>() - 1) / chunk_len<F32>());
  const int chunks = static_cast<int64_t>(rows) * all / 2 >= 148 * 20 ? 2 : 1;
  const int parts = (all + chunks - 1) / chunks;
  const unsigned warps = kStatThreads / 32;
  cudaError_t e = launch_chained(verify_stats_kernel<F32>, dim3((static_cast<unsigned>(parts) + warps - 1) / warps, rows),
                                 dim3(kStatThreads), 0, stream, a, parts, chunks);
  if (e != cudaSuccess) return e;
  // a CTA per 4096 tokens, at most kDrawCtas, and no more than one per SM: the clusters' CTAs are placed two to an SM
  // while others stay idle otherwise
  unsigned ctas = 1;
  const unsigned seqs = static_cast<unsigned>(a.B);
  while (ctas < kDrawCtas && static_cast<int64_t>(ctas) * 4096 < a.V && 2 * ctas * seqs <= 148) ctas *= 2;
  // 32 warps where each has tokens for several rounds and all clusters run at once with one CTA to an SM, which 14 of 8
  // and 33 of 4 do; 16 with more registers elsewhere (V 32003: 8.6 us, with 32 10.2; 16 sequences of 100000: 25.4, 29.5)
  const dim3 grid(ctas, seqs);
  const bool resident = ctas == 8 ? seqs <= 14 : ctas * seqs <= 132;
  const bool many = a.V / static_cast<int>(ctas) > 8192;
  if (many && resident)
    return launch_chained_cluster(verify_draw_kernel<F32, 1024>, grid, dim3(1024), F32 ? 0 : WeightTable::kBytes, stream, ctas, a, parts);
  return launch_chained_cluster(verify_draw_kernel<F32, 512>, grid, dim3(512), 0, stream, ctas, a, parts);
}

}  // namespace

// The most parts of a row: one chunk each, fp32.
int verify_parts(int V) { return static_cast<int>((static_cast<int64_t>(V) + 8 + chunk_len<true>() - 1) / chunk_len<true>()); }

cudaError_t launch_verify(const VerifyArgs& a, bool f32, cudaStream_t stream) {
  return f32 ? launch<true>(a, stream) : launch<false>(a, stream);
}

cudaError_t verify_set_attributes() {
  return cudaFuncSetAttribute(verify_draw_kernel<false, 1024>, cudaFuncAttributeMaxDynamicSharedMemorySize, WeightTable::kBytes);
}

}  // namespace q4t
