// Norms before and after an FFN block, fused with the block's gate and
// residual scale, and the int8 quantisation of rows.
//
// For every row t (all sums and products in fp32, each output rounded once):
//   b = N_post(y_t)                                   branch, after its norm
//   r = residual_scale * res_t + branch_scale * act(g_t) * b
//   residual_out_t = r
//   x = N_next(r)                                     input of the next block
//   out_t = x, or q = round_half_even(127 x / amax|x|) with row_scale = amax / 127
// N is the identity, the RMS norm v * rsqrt(mean v^2 + eps) * (o + w) + b or
// the layer norm (v - mean) * rsqrt(var + eps) * (o + w) + b.  The next norm
// takes r before residual_out's rounding.
//
// One pass: a row's values stay in registers between the reductions (the
// layer norm's variance is a second sum over centred values, not a difference
// of moments), so DRAM sees each input once and each output once, and the
// bytes are the bound.
//
// A row is cut into granules of 8 elements that start on 16 bytes; its first
// and last granule may be partial (rows of odd width start anywhere).  Three
// kernels share the arithmetic:
//   warp_kernel   a warp a row, rows up to 128 granules (more where there are
//                 many rows);
//   ring_kernel   a block a row, rows through a shared-memory ring of bulk
//                 copies that runs ahead of the arithmetic;
//   plain_kernel  single elements, read again in each pass: rows of tensors
//                 that do not share their granules (mixed alignments), mixes of
//                 three element types, and rows beyond the ring's (up to
//                 131071 values for rows that are quantised as they are).
//
// Each type of the branch (or of the rows to norm) has a translation unit of
// its own (block_norm_bf16.cu, _f16, _f32), compiled side by side.
#pragma once

#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "block_norm.h"
#include "qcc_common.cuh"
#include "qcc_host.h"

namespace qcc {

namespace {

constexpr uint64_t kDrainNs = 2000000000ull;  // for copies in flight after a wait that ran out
// A row whose largest magnitude is below this is stored as zeros: its scale
// (and 127 / amax) would leave the normal fp32 range.
constexpr float kSmallestAmax = 1.504632769052528e-36f;   // 2^-119

// ---------------------------------------------------------------------------
// Which elements a thread holds.
// ---------------------------------------------------------------------------

// Granule i of member `id` of a team of `width` threads: elements first(i) .. + 7.  EXACT: rows without a shift and
// with a multiple of 8 elements, whose granules (and those of 16-byte aligned parameters) exist whole or not at all.
template <bool EXACT>
struct GranuleMap {
  int n, shift, id, width;
  __device__ __forceinline__ int first(int i) const { return (i * width + id) * 8 - (EXACT ? 0 : shift); }
  __device__ __forceinline__ int element(int i, int j) const { return first(i) + j; }
  __device__ __forceinline__ bool has(int i, int j) const {
    return static_cast<unsigned>(element(i, j)) < static_cast<unsigned>(n);
  }
  // All of the granule exists.
  __device__ __forceinline__ bool whole(int i) const {
    return EXACT ? first(i) < n : first(i) >= 0 && first(i) + 8 <= n;
  }
};

// Two elements an instruction, each rounded as the single one: the kernels are short of issue slots, not of
// arithmetic (join of 8192 x 5120 bf16: 63.3 us with single instructions, 61.5 with these).
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{.reg .b64 a, b, r; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; add.rn.f32x2 r, a, b; mov.b64 {%0, %1}, r;}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{.reg .b64 a, b, r; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; mul.rn.f32x2 r, a, b; mov.b64 {%0, %1}, r;}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{.reg .b64 a, b, c, r; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; mov.b64 c, {%6, %7};"
      " fma.rn.f32x2 r, a, b, c; mov.b64 {%0, %1}, r;}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
// Elements 2 j and 2 j + 1 of a granule.
__device__ __forceinline__ float2 pair(const float (&v)[8], int j) { return make_float2(v[2 * j], v[2 * j + 1]); }
__device__ __forceinline__ void set_pair(float (&v)[8], int j, float2 p) { v[2 * j] = p.x, v[2 * j + 1] = p.y; }

__device__ __forceinline__ uint32_t half_bits(__nv_bfloat16 v) { return __bfloat16_as_ushort(v); }
__device__ __forceinline__ uint32_t half_bits(__half v) { return __half_as_ushort(v); }

// Elements as a granule's words.
template <typename T>
__device__ __forceinline__ Pack8<T> to_words(const T (&e)[8]) {
  Pack8<T> p;
  p.w[0] = make_uint4(half_bits(e[0]) | half_bits(e[1]) << 16, half_bits(e[2]) | half_bits(e[3]) << 16,
                      half_bits(e[4]) | half_bits(e[5]) << 16, half_bits(e[6]) | half_bits(e[7]) << 16);
  return p;
}
__device__ __forceinline__ Pack8<float> to_words(const float (&e)[8]) {
  Pack8<float> p;
  p.w[0] = make_uint4(__float_as_uint(e[0]), __float_as_uint(e[1]), __float_as_uint(e[2]), __float_as_uint(e[3]));
  p.w[1] = make_uint4(__float_as_uint(e[4]), __float_as_uint(e[5]), __float_as_uint(e[6]), __float_as_uint(e[7]));
  return p;
}

// Granule i of a row (zeros outside of it): one wide load where all of it exists.  Kept as words: 16-bit elements
// held one by one would be taken apart and put together again.
template <typename T, bool EXACT>
__device__ __forceinline__ Pack8<T> load_granule(const T* row, const GranuleMap<EXACT>& m, int i) {
  if (m.whole(i)) return load_pack8<T>(row + m.first(i));
  if (!EXACT) {
    T e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = m.has(i, j) ? row[m.element(i, j)] : T(0.f);
    return to_words(e);
  }
  Pack8<T> p;
#pragma unroll
  for (int k = 0; k < Pack8<T>::kWords; ++k) p.w[k] = make_uint4(0, 0, 0, 0);
  return p;
}

// Elements 8 - shift .. 15 - shift of two granules that follow each other, shift 1..7: words are selected two steps
// down, 16-bit elements then brought together across words.
template <typename P>
__device__ __forceinline__ Pack8<P> straddle(const Pack8<P>& lo, const Pack8<P>& hi, int shift) {
  constexpr int kWords = sizeof(P) * 2;  // of a granule
  uint32_t w[2 * kWords];
#pragma unroll
  for (int k = 0; k < Pack8<P>::kWords; ++k) {
    w[4 * k] = lo.w[k].x, w[4 * k + 1] = lo.w[k].y, w[4 * k + 2] = lo.w[k].z, w[4 * k + 3] = lo.w[k].w;
    w[kWords + 4 * k] = hi.w[k].x, w[kWords + 4 * k + 1] = hi.w[k].y;
    w[kWords + 4 * k + 2] = hi.w[k].z, w[kWords + 4 * k + 3] = hi.w[k].w;
  }
  const int first = sizeof(P) == 4 ? 8 - shift : (8 - shift) >> 1;  // the first word wanted
#pragma unroll
  for (int step = kWords / 2; step > 0; step >>= 1)
#pragma unroll
    for (int j = 0; j + step < 2 * kWords; ++j) w[j] = (first & step) != 0 ? w[j + step] : w[j];
  if (sizeof(P) == 2) {
    const int bits = (shift & 1) * 16;
#pragma unroll
    for (int j = 0; j < kWords; ++j) w[j] = __funnelshift_r(w[j], w[j + 1], bits);
  }
  Pack8<P> r;
#pragma unroll
  for (int k = 0; k < Pack8<P>::kWords; ++k) r.w[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
  return r;
}

// A parameter vector's elements of granule i.  Without EXACT they straddle two of its own granules (when it starts on
// 16 bytes and both lie inside of it), or are single elements.
template <typename P, bool EXACT>
__device__ __forceinline__ void load_param8(const P* p, const GranuleMap<EXACT>& m, int i, float (&f)[8]) {
  if (EXACT) {
    widen(load_granule(p, m, i), f);
    return;
  }
  const int e = m.first(i) + m.shift;  // the later granule's first element
  if (m.first(i) >= 0 && e + 8 <= m.n && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    const Pack8<P> hi = load_pack8<P>(p + e);
    widen(m.shift == 0 ? hi : straddle(load_pack8<P>(p + e - 8), hi, m.shift), f);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = m.has(i, j) ? to_f32<P>(p[m.element(i, j)]) : 0.f;
  }
}

// The same for a parameter in P or fp32.
template <typename P, bool EXACT>
__device__ __forceinline__ void load_param8(const void* p, int dtype, const GranuleMap<EXACT>& m, int i,
                                            float (&f)[8]) {
  if (sizeof(P) == 4 || dtype == QCC_DTYPE_F32)
    load_param8(static_cast<const float*>(p), m, i, f);
  else
    load_param8(static_cast<const P*>(p), m, i, f);
}

__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16*) {
  __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&p);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half*) {
  __half2 p = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&p);
}

template <typename T>
__device__ __forceinline__ void store_vec8(T* p, const float* f) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack2(f[0], f[1], p), pack2(f[2], f[3], p), pack2(f[4], f[5], p), pack2(f[6], f[7], p));
}
__device__ __forceinline__ void store_vec8(float* p, const float* f) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}

template <typename T, bool EXACT>
__device__ __forceinline__ void store_granule(T* row, const GranuleMap<EXACT>& m, int i, const float* f) {
  if (m.whole(i)) {
    store_vec8(row + m.first(i), f);
  } else if (!EXACT) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (m.has(i, j)) row[m.element(i, j)] = static_cast<T>(f[j]);
  }
}

// max(|a|, |f|, |g|), NaN if any is.
__device__ __forceinline__ float larger(float a, float f, float g) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(f), "f"(g));
  return r;
}

// Bits of |f|: ordered like the magnitudes, infinities and then NaNs above all finite values.
__device__ __forceinline__ uint32_t magnitude(float f) { return __float_as_uint(f) & 0x7FFFFFFFu; }

// What a row's largest magnitude (its bits) makes of its int8 form, for values that `factor` (1 to 2) still has to
// multiply: a factor of a whole row changes its scale and none of its quotients.
struct RowScale {
  float amax, scale, inverse, inverse_rest;  // inverse 0: the row is stored as zeros
  __device__ __forceinline__ explicit RowScale(uint32_t bits, float factor = 1.f) {
    amax = __uint_as_float(bits);
    const bool finite = bits <= 0x7F7FFFFFu, kept = finite && amax * factor >= kSmallestAmax;
    inverse = kept ? 127.f / amax : 0.f;
    inverse_rest = kept ? fmaf(-inverse, amax, 127.f) / amax : 0.f;
    scale = kept ? amax / 127.f * factor : finite ? 0.f : NAN;
  }
};

// round_half_even(127 x / amax) from the remainder 127 x - q amax of a rounding q that may be one off: an exact pair
// d + e, since q amax and 127 x are multiples of amax's last place and d is at most amax.
__device__ __forceinline__ int settle_border(float x, float amax, int q) {
  if (amax > 0x1p100f) x *= 0x1p-20f, amax *= 0x1p-20f;  // keeps 127 x finite; exact
  const float p = 127.f * x, e = fmaf(127.f, x, -p);
  const float d = fmaf(-static_cast<float>(q), amax, p);
  const float side = d < 0.f ? -1.f : 1.f;
  const float over = fmaf(2.f, fabsf(d), -amax) + 2.f * side * e;  // twice the remainder's size beyond half a step
  return over > 0.f || (over == 0.f && (q & 1) != 0) ? q + static_cast<int>(side) : q;
}

constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: adding it rounds to whole numbers, held in the low bits

// int8 of computed values (norms), in the low bytes: round_half_even of 127 x / amax rounded to fp32.  The reciprocal's
// remainder brings the quotient within 2^-47 of itself before its rounding, or 2^-28 where the remainder is no longer a
// normal number (amax above 2^109 or so), so a border k + 1/2 comes out as such.
__device__ __forceinline__ float2 quotient2(float2 x, const RowScale& s) {
  return fma2(x, both(s.inverse), mul2(x, both(s.inverse_rest)));
}
__device__ __forceinline__ void quantize8(const float (&f)[8], const RowScale& s, uint32_t (&q)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 r = add2(quotient2(pair(f, j), s), both(kMagic));
    q[2 * j] = __float_as_uint(r.x), q[2 * j + 1] = __float_as_uint(r.y);
  }
}

// The low bytes of four words.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// int8 of rows as they are: round_half_even(127 x / amax), of the exact quotient, for |x| <= amax.  Before its one
// rounding to fp32 the quotient is within 2^-28 of itself (see quotient2), less than half a last place, so a border
// k + 1/2 comes out as such, and what does not come out as one lies on its own side of it.  Values of 16-bit types lie
// on borders in earnest (small whole numbers times powers of two), and no other quotient of theirs rounds to one: with
// 11-bit significands those in [2^k, 2^(k+1)) are 2^(k-20) or more away from a border, and fp32 and the quotient before
// it are off by 2^(k-23) together there.  fp32 values that round to a border need the exact remainder.
template <typename T>
__device__ __forceinline__ void quantize8_exact(const float (&f)[8], const RowScale& s, uint32_t (&q)[8]) {
  bool border = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 t = quotient2(pair(f, j), s);
    const float2 r = add2(t, both(kMagic));
    q[2 * j] = __float_as_uint(r.x), q[2 * j + 1] = __float_as_uint(r.y);
    if (sizeof(T) == 4) border |= fabsf(t.x - (r.x - kMagic)) == 0.5f || fabsf(t.y - (r.y - kMagic)) == 0.5f;
  }
  if (sizeof(T) == 4 && border)
#pragma unroll
    for (int j = 0; j < 8; ++j)
      q[j] = static_cast<uint32_t>(settle_border(f[j], s.amax, __float2int_rn(f[j] * s.inverse)));
}

template <bool EXACT>
__device__ __forceinline__ void store_int8x8(int8_t* row, const GranuleMap<EXACT>& m, int i, const uint32_t (&q)[8]) {
  if (m.whole(i) && (EXACT || (reinterpret_cast<uintptr_t>(row + m.first(i)) & 7) == 0)) {
    *reinterpret_cast<uint2*>(row + m.first(i)) =
        make_uint2(low_bytes(q[0], q[1], q[2], q[3]), low_bytes(q[4], q[5], q[6], q[7]));
  } else if (!EXACT) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (m.has(i, j)) row[m.element(i, j)] = static_cast<int8_t>(q[j]);
  }
}

// ---------------------------------------------------------------------------
// Reductions over the team of a row, in a fixed order.
// ---------------------------------------------------------------------------

__device__ __forceinline__ uint32_t warp_max(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }

struct WarpTeam {
  __device__ __forceinline__ float sum(float v) { return warp_sum(v); }
  __device__ __forceinline__ uint32_t max(uint32_t v) { return warp_max(v); }
};

// One barrier a reduction: the halves of `scratch` [2][kMaxWarps] are used in turn, and a half's readers have passed
// the next reduction's barrier before it is written again.  Up to kFewWarps every thread joins the warps' parts from
// wide loads, beyond them a warp's lanes by shuffles (layer norm of 2048 x 5120, 10 warps: 13.5 and 14.0 us; norm of
// 4096 x 8001, 16 warps: 33.9 and 33.3 us).
constexpr int kMaxWarps = 20, kFewWarps = 12;

struct BlockTeam {
  float* scratch;
  int half = 0;
  // Before the kernel's first barrier: the parts of warps that the block does not have are neutral.
  static __device__ __forceinline__ void clear(float* scratch) {
    for (int i = threadIdx.x; i < 2 * kMaxWarps; i += blockDim.x) scratch[i] = 0.f;
  }
  __device__ __forceinline__ const float* exchange(float v) {
    float* s = scratch + half * kMaxWarps;
    half ^= 1;
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    return s;
  }
  __device__ __forceinline__ float lane_part(const float* s) const {
    const int lane = threadIdx.x & 31, warps = static_cast<int>(blockDim.x) >> 5;
    return lane < warps ? s[lane] : 0.f;  // 0: neutral for sums and for maxima of magnitudes
  }
  __device__ __forceinline__ float sum(float v) {
    const float* s = exchange(warp_sum(v));
    if (blockDim.x > kFewWarps * 32) return warp_sum(lane_part(s));
    float2 lo = both(0.f), hi = both(0.f);
#pragma unroll
    for (int k = 0; k < kFewWarps / 4; ++k) {
      const float4 p = reinterpret_cast<const float4*>(s)[k];
      lo = add2(lo, make_float2(p.x, p.y)), hi = add2(hi, make_float2(p.z, p.w));
    }
    lo = add2(lo, hi);
    return lo.x + lo.y;
  }
  __device__ __forceinline__ uint32_t max(uint32_t v) {
    const float* s = exchange(__uint_as_float(warp_max(v)));
    return warp_max(__float_as_uint(lane_part(s)));
  }
};

// ---------------------------------------------------------------------------
// The arithmetic of a row.
// ---------------------------------------------------------------------------

// The int8 form of an RMS norm without a bias needs the quotients of the products value * weight only: 1 / rms is a
// factor of the whole row.  Products of two 16-bit values are exact in fp32, and those of half the largest one's
// magnitude lie on the border 63.5 in earnest (one in 10 000 of 5120 wide bf16 rows), where a rounding by 1 / rms
// would decide.  So the values are multiplied by a power of two, which rounds nothing, and the rest of 1 / rms, in
// [1, 2), goes into the row's scale.
__device__ __forceinline__ bool keeps_ratios(const qcc_norm_params& a) {
  return a.kind == QCC_NORM_RMS && a.bias == nullptr;
}
__device__ __forceinline__ float power_part(float rstd) {
  return __uint_as_float(__float_as_uint(rstd) & 0x7F800000u);
}
__device__ __forceinline__ float factor_part(float rstd) {
  return __uint_as_float((__float_as_uint(rstd) & 0x007FFFFFu) | 0x3F800000u);
}

// v <- N(v) over the row's values (entries outside the row are 0 on entry, and stay so where they are summed).
// Returns 1 / its deviation; with `ratios` only that one's power of two has been applied.
template <typename P, int VPT, bool EXACT, typename Team>
__device__ __forceinline__ float normalise(float (&v)[VPT][8], const qcc_norm_params& a, float inv_n,
                                           const GranuleMap<EXACT>& m, Team& team, bool ratios = false) {
  if (a.kind == QCC_NORM_NONE) return 1.f;
  if (a.kind == QCC_NORM_LAYER) {
    float2 s = both(0.f);
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s = add2(s, pair(v[i], j));
    const float mean = team.sum(s.x + s.y) * inv_n;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) set_pair(v[i], j, add2(pair(v[i], j), both(-mean)));
      if (!m.whole(i))
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (EXACT || !m.has(i, j)) v[i][j] = 0.f;
    }
  }
  float2 s = both(0.f);
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) s = fma2(pair(v[i], j), pair(v[i], j), s);
  const float rstd = rsqrtf(team.sum(s.x + s.y) * inv_n + a.eps);
  const float by = ratios ? power_part(rstd) : rstd;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    float w[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) set_pair(v[i], j, mul2(pair(v[i], j), both(by)));
    if (a.weight != nullptr) {
      load_param8<P>(a.weight, a.dtype, m, i, w);
      if (a.weight_offset != 0.f)
#pragma unroll
        for (int j = 0; j < 4; ++j) set_pair(w, j, add2(pair(w, j), both(a.weight_offset)));
#pragma unroll
      for (int j = 0; j < 4; ++j) set_pair(v[i], j, mul2(pair(v[i], j), pair(w, j)));
    }
    if (a.bias != nullptr) {
      load_param8<P>(a.bias, a.dtype, m, i, w);
#pragma unroll
      for (int j = 0; j < 4; ++j) set_pair(v[i], j, add2(pair(v[i], j), pair(w, j)));
    }
  }
  return rstd;
}

__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t e) {
  if (dtype == QCC_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[e]);
  if (dtype == QCC_DTYPE_F16) return __half2float(static_cast<const __half*>(p)[e]);
  return static_cast<const float*>(p)[e];
}

__device__ __forceinline__ float gate_value(float g, int act) {
  // The fast exponential and quotient are off by |g| + 8 roundings at most, and exact at the ends (0 and 1).  From
  // exp(-|g|): beyond 2^126, as 1 + exp(-g) is below g = -87.3, the fast quotient is 0.
  if (act == QCC_GATE_SIGMOID) {
    const float e = __expf(-fabsf(g));
    return __fdividef(g < 0.f ? e : 1.f, 1.f + e);
  }
  if (act == QCC_GATE_TANH) return tanhf(g);
  return g;
}

// v <- act(gate) * v.
template <typename T, int VPT, bool EXACT>
__device__ __forceinline__ void apply_gate(float (&v)[VPT][8], const BlockNormArgs& a, int64_t t,
                                           const GranuleMap<EXACT>& m) {
  if (a.gate.values == nullptr) return;
  const int64_t row = (t / a.gate.rows_each) * a.gate.ld;
  if (a.gate.cols == 1) {
    const float s = gate_value(load_any(a.gate.values, a.gate.dtype, row), a.gate.act);
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) set_pair(v[i], j, mul2(pair(v[i], j), both(s)));
    return;
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    float g[8];
    if (a.gate_in_granules)  // in T
      widen(load_granule(static_cast<const T*>(a.gate.values) + row, m, i), g);
    else
      load_param8<T>(static_cast<const char*>(a.gate.values) + row * (a.gate.dtype == QCC_DTYPE_F32 ? 4 : 2),
                     a.gate.dtype, m, i, g);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] *= gate_value(g[j], a.gate.act);
  }
}

// residual_out[t] <- v <- residual_scale * r + branch_scale * v, for granule i (0 outside of the row, as r and v are).
template <typename R, bool EXACT>
__device__ __forceinline__ void join8(float (&v)[8], const float (&r)[8], const BlockNormArgs& a, int64_t t,
                                      const GranuleMap<EXACT>& m, int i) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    set_pair(v, j, fma2(both(a.residual_scale), pair(r, j), mul2(both(a.branch_scale), pair(v, j))));
  store_granule(static_cast<R*>(a.res_out) + t * a.ld_res_out, m, i, v);
}

// out[t] (P, fp32 or int8) from N_next(v).
template <typename P, int VPT, bool EXACT, typename Team>
__device__ __forceinline__ void finish_row(float (&v)[VPT][8], const BlockNormArgs& a, int64_t t,
                                           const GranuleMap<EXACT>& m, Team& team) {
  if (a.out == nullptr) return;
  if (a.out_dtype == QCC_DTYPE_I8) {
    const bool ratios = keeps_ratios(a.next);
    const float rstd = normalise<P>(v, a.next, a.inv_hidden, m, team, ratios);
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < 8; j += 2) amax = larger(amax, v[i][j], v[i][j + 1]);
    const RowScale s(team.max(__float_as_uint(amax)), ratios ? factor_part(rstd) : 1.f);
    if (m.id == 0) a.row_scale[t] = s.scale;
    int8_t* row = static_cast<int8_t*>(a.out) + t * a.ld_out;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (s.inverse == 0.f)  // also takes the NaNs and infinities out
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
      uint32_t q[8];
      quantize8(v[i], s, q);
      store_int8x8(row, m, i, q);
    }
    return;
  }
  normalise<P>(v, a.next, a.inv_hidden, m, team);
  if (a.out_dtype == QCC_DTYPE_F32) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) store_granule(static_cast<float*>(a.out) + t * a.ld_out, m, i, v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < VPT; ++i) store_granule(static_cast<P*>(a.out) + t * a.ld_out, m, i, v[i]);
  }
}

// ---------------------------------------------------------------------------
// Rows as they are to int8: the words stay as they came, and 16-bit magnitudes are compared two at a time.
// ---------------------------------------------------------------------------

__device__ __forceinline__ uint32_t larger2(uint32_t a, uint32_t w, __nv_bfloat16*) {  // NaN if either is
  const __nv_bfloat162 r =
      __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&a), __habs2(*reinterpret_cast<__nv_bfloat162*>(&w)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t larger2(uint32_t a, uint32_t w, __half*) {
  const __half2 r = __hmax2_nan(*reinterpret_cast<__half2*>(&a), __habs2(*reinterpret_cast<__half2*>(&w)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ void widen2(uint32_t w, float& lo, float& hi, __nv_bfloat16*) { bf16x2_to_f32(w, lo, hi); }
__device__ __forceinline__ void widen2(uint32_t w, float& lo, float& hi, __half*) { half2_to_f32(w, lo, hi); }

// Bits of the largest magnitude of the words.
template <typename T, int VPT>
__device__ __forceinline__ uint32_t largest(const Pack8<T> (&y)[VPT]) {
  if constexpr (sizeof(T) == 4) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int k = 0; k < 2; ++k)
        top = max(max(max(top, y[i].w[k].x & 0x7FFFFFFFu), max(y[i].w[k].y & 0x7FFFFFFFu, y[i].w[k].z & 0x7FFFFFFFu)),
                  y[i].w[k].w & 0x7FFFFFFFu);
    return top;
  } else {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      top = larger2(top, y[i].w[0].x, static_cast<T*>(nullptr));
      top = larger2(top, y[i].w[0].y, static_cast<T*>(nullptr));
      top = larger2(top, y[i].w[0].z, static_cast<T*>(nullptr));
      top = larger2(top, y[i].w[0].w, static_cast<T*>(nullptr));
    }
    float lo, hi;
    widen2(top, lo, hi, static_cast<T*>(nullptr));
    return max(magnitude(lo), magnitude(hi));
  }
}

template <typename T, int VPT, bool EXACT, typename Team>
__device__ __forceinline__ void quantize_row(const Pack8<T> (&y)[VPT], const BlockNormArgs& a, int64_t t,
                                             const GranuleMap<EXACT>& m, Team& team) {
  const RowScale s(team.max(largest(y)));
  if (m.id == 0) a.row_scale[t] = s.scale;
  int8_t* row = static_cast<int8_t*>(a.out) + t * a.ld_out;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    float f[8];
    uint32_t q[8];
    widen(y[i], f);
    if (s.inverse == 0.f)  // also takes the NaNs and infinities out
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = 0.f;
    quantize8_exact<T>(f, s, q);
    store_int8x8(row, m, i, q);
  }
}

// ---------------------------------------------------------------------------
// Kernels.  T: the branch's (or x's) type, R: the residual's in a join.
// ---------------------------------------------------------------------------

enum Mode { kNorm, kJoin, kQuantize };

// The 16-bit type that parameters and outputs may have besides fp32: T, or for the norm of fp32 rows R (an fp32
// residual stream normed for 16-bit weights).
template <typename T, typename R, Mode MODE>
using ParamType = std::conditional_t<sizeof(T) == 4 && MODE == kNorm, R, T>;

__device__ __forceinline__ int row_shift(const BlockNormArgs& a, int64_t t) {
  return static_cast<int>((a.shift0 + t * a.ldy) & 7);
}

constexpr int kWarpRows = 4;  // rows (warps) of a block
constexpr int kManyRows = 2048;  // from here on a warp takes rows beyond 128 granules too

// A warp a row: no barriers, every load of the row in flight at once.  Bound by latency at these sizes (8192 x 128
// bf16: 2.4 us, 1.7 TB/s).
template <typename T, typename R, Mode MODE, int VPT, bool EXACT>
__global__ void __launch_bounds__(32 * kWarpRows) warp_kernel(const BlockNormArgs a) {
  using P = ParamType<T, R, MODE>;
  grid_dependency_wait();
  grid_dependency_trigger();
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kWarpRows + (threadIdx.x >> 5);
  if (t >= a.rows) return;
  const GranuleMap<EXACT> m = {a.hidden, EXACT ? 0 : row_shift(a, t), static_cast<int>(threadIdx.x & 31), 32};
  WarpTeam team;
  Pack8<T> y[VPT];
  Pack8<R> r[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) y[i] = load_granule(static_cast<const T*>(a.y) + t * a.ldy, m, i);
  if (MODE == kQuantize) {
    quantize_row(y, a, t, m, team);
    return;
  }
  if (MODE == kJoin)
#pragma unroll
    for (int i = 0; i < VPT; ++i) r[i] = load_granule(static_cast<const R*>(a.res) + t * a.ld_res, m, i);
  float v[VPT][8];
#pragma unroll
  for (int i = 0; i < VPT; ++i) widen(y[i], v[i]);
  if (MODE == kJoin) {
    normalise<P>(v, a.post, a.inv_hidden, m, team);
    apply_gate<T>(v, a, t, m);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float f[8];
      widen(r[i], f);
      join8<R>(v[i], f, a, t, m, i);
    }
  }
  finish_row<P>(v, a, t, m, team);
}

// One norm's row statistics and an element's normed value, without `factor` where the norm's ratios are wanted.
struct RowNorm {
  float mean = 0.f, rstd = 1.f, factor = 1.f;
  template <typename F>
  __device__ __forceinline__ RowNorm(const qcc_norm_params& p, int n, BlockTeam& team, F value, bool ratios = false) {
    if (p.kind == QCC_NORM_NONE) return;
    float s = 0.f;
    if (p.kind == QCC_NORM_LAYER) {
      for (int e = threadIdx.x; e < n; e += blockDim.x) s += value(e);
      mean = team.sum(s) / static_cast<float>(n);
    }
    s = 0.f;
    for (int e = threadIdx.x; e < n; e += blockDim.x) {
      const float d = value(e) - mean;
      s += d * d;
    }
    rstd = 1.f / sqrtf(team.sum(s) / static_cast<float>(n) + p.eps);
    if (ratios) factor = factor_part(rstd), rstd = power_part(rstd);
  }
  __device__ __forceinline__ float apply(const qcc_norm_params& p, float v, int e) const {
    if (p.kind == QCC_NORM_NONE) return v;
    v = (v - mean) * rstd;
    if (p.weight != nullptr) v *= p.weight_offset + load_any(p.weight, p.dtype, e);
    return p.bias == nullptr ? v : v + load_any(p.bias, p.dtype, e);
  }
};

// One block a row; outputs are written in the last pass, so they may be the inputs themselves.  Single elements and
// repeated reads make it slow (join of 4096 x 5120 with a residual off by 6 bytes: 167 us, 32 us on shared granules;
// of fp32 rows with bf16 weights and output 191 us; rows to int8 of 4096 x 36864 543 us, 70 us of bytes).
__global__ void __launch_bounds__(512) plain_kernel(const BlockNormArgs a, int dtype, int res_dtype) {
  __shared__ __align__(16) float scratch[2 * kMaxWarps];
  BlockTeam::clear(scratch);
  __syncthreads();
  grid_dependency_wait();
  grid_dependency_trigger();
  const int64_t t = blockIdx.x;
  const int n = a.hidden;
  BlockTeam team = {scratch};
  const auto branch = [&](int e) { return load_any(a.y, dtype, t * a.ldy + e); };
  const RowNorm post(a.post, n, team, branch);
  const auto joined = [&](int e) {
    float v = branch(e);
    if (a.res == nullptr) return v;
    v = post.apply(a.post, v, e);
    if (a.gate.values != nullptr)
      v *= gate_value(load_any(a.gate.values, a.gate.dtype,
                               (t / a.gate.rows_each) * a.gate.ld + (a.gate.cols == 1 ? 0 : e)), a.gate.act);
    return a.residual_scale * load_any(a.res, res_dtype, t * a.ld_res + e) + a.branch_scale * v;
  };
  const bool to_int8 = a.out != nullptr && a.out_dtype == QCC_DTYPE_I8, ratios = to_int8 && keeps_ratios(a.next);
  const RowNorm next(a.next, n, team, joined, ratios);
  const bool as_is = a.res == nullptr && a.next.kind == QCC_NORM_NONE;
  RowScale s(0u);
  if (to_int8) {
    uint32_t amax = 0;
    for (int e = threadIdx.x; e < n; e += blockDim.x) amax = max(amax, magnitude(next.apply(a.next, joined(e), e)));
    s = RowScale(team.max(amax), next.factor);
    if (threadIdx.x == 0) a.row_scale[t] = s.scale;
  }
  for (int e = threadIdx.x; e < n; e += blockDim.x) {
    const float r = joined(e);
    if (a.res != nullptr) store_as(a.res_out, t * a.ld_res_out + e, res_dtype, r);
    if (a.out == nullptr) continue;
    const float x = next.apply(a.next, r, e);
    if (to_int8)
      static_cast<int8_t*>(a.out)[t * a.ld_out + e] = static_cast<int8_t>(
          s.inverse == 0.f ? 0
          : as_is          ? settle_border(x, s.amax, __float2int_rn(x * s.inverse))
                           : __float2int_rn(quotient2(both(x), s).x));
    else
      store_as(a.out, t * a.ld_out + e, a.out_dtype, x);
  }
}

// Bytes of a ring slot's part for a row of es-byte elements: its granules.
__host__ __device__ __forceinline__ int slot_bytes(int hidden, int es) { return (hidden + 14) / 8 * 8 * es; }

constexpr int kMaxDepth = 8;
// Shared memory that a ring kernel's blocks on an SM share: two rows each in kRoom, more rows each only within
// kDeepRoom (what is left caches the parameters: 208 KB of rings cost the norm of 8192 x 5120 rows 10 %).
constexpr int kRoom = 208 << 10, kDeepRoom = 128 << 10;
// Threads of an SM's ring blocks together: more blocks leave each a shallower ring (norm of 8192 x 5120, blocks of 320
// threads: 30.7 us with four and three rows each, 35.6 with five and two).
constexpr int kMostThreads = 1344;

// Threads of a ring block, at most; and blocks of that size an SM that its registers allow with no more than 8 bytes of
// spills.  Two
// granules a thread up to 640 threads for norms (8192 x 5120 bf16: 31.8 us, 34.4 us with four; fp32 60.6 and 76.2 us),
// four from 192 threads on for plain quantisation, whose threads do little else (4096 x 5120: 12.5 us, 17 with two).
template <Mode MODE, int VPT, bool EXACT>
struct RingShape {
  static constexpr int kThreads = VPT == 2 ? (MODE == kQuantize ? 192 : 640) : VPT == 4 ? 576 : 512;
  static_assert(kThreads <= 32 * kMaxWarps);
  static constexpr int kBlocks = EXACT && (VPT == 2 || (VPT == 4 && MODE != kJoin)) ? 2 : 1;
};

// The granules of row t that a bulk copy brings, [lo, hi): all of them, except that the partial granules at the two
// ends of the tensor would read outside of it (inside the tensor they read a neighbour's elements, ignored).
struct RowCopy {
  int lo, hi;
  __device__ __forceinline__ RowCopy(const BlockNormArgs& a, int64_t t, int shift) {
    lo = t == 0 && shift != 0 ? 1 : 0;
    hi = t == a.rows - 1 ? (a.hidden + shift) / 8 : (a.hidden + shift + 7) / 8;
  }
};

template <typename E>
__device__ __forceinline__ void copy_row(uint8_t* slot, const E* row, const RowCopy& c, int shift, uint64_t* bar,
                                         uint64_t policy) {
  if (c.lo < c.hi)
    bulk_load(slot + c.lo * 8 * sizeof(E), row + (c.lo * 8 - shift),
              static_cast<uint32_t>((c.hi - c.lo) * 8 * sizeof(E)), bar, policy);
}

// Granule i of the row from the ring slot; the tensor's partial end granules from global memory.
template <typename E, bool EXACT>
__device__ __forceinline__ Pack8<E> load_slot(const uint8_t* slot, const E* row, const RowCopy& c,
                                              const GranuleMap<EXACT>& m, int i) {
  const E* const there = reinterpret_cast<const E*>(slot);
  if (EXACT) return load_granule(there, m, i);
  const int g = i * m.width + m.id;
  if (m.whole(i)) return load_pack8<E>(there + g * 8);  // copied: only partial granules are left out
  const E* const from = g >= c.lo && g < c.hi ? there + m.shift : row;
  E e[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) e[j] = m.has(i, j) ? from[m.element(i, j)] : E(0.f);
  return to_words(e);
}

template <typename T>
__host__ __device__ constexpr int code_of() {
  return std::is_same_v<T, __nv_bfloat16> ? QCC_DTYPE_BF16 : std::is_same_v<T, __half> ? QCC_DTYPE_F16 : QCC_DTYPE_F32;
}

// The end of a block whose wait for row t (slot s) ran out: its rows from t on become NaN (int8: zeros, and NaN as the
// scale), and thread 0 sees the copies in flight in, which would land in the shared memory of a later block.
__device__ __forceinline__ void give_up(const BlockNormArgs& a, int res_dtype, uint64_t* full, int depth, int64_t t,
                                        int s, int phase) {
  if (threadIdx.x == 0)
    for (int64_t u = t, k = 0; k < depth && u < a.rows; ++k, u += gridDim.x) {
      mbar_wait_suspended(&full[s], phase, kDrainNs);
      if (++s == depth) s = 0, phase ^= 1;
    }
  for (; t < a.rows; t += gridDim.x) {
    for (int e = threadIdx.x; e < a.hidden; e += blockDim.x) {
      if (a.res_out != nullptr) store_as(a.res_out, t * a.ld_res_out + e, res_dtype, NAN);
      if (a.out == nullptr) continue;
      if (a.out_dtype == QCC_DTYPE_I8)
        static_cast<int8_t*>(a.out)[t * a.ld_out + e] = 0;
      else
        store_as(a.out, t * a.ld_out + e, a.out_dtype, NAN);
    }
    if (threadIdx.x == 0 && a.out != nullptr && a.out_dtype == QCC_DTYPE_I8) a.row_scale[t] = NAN;
  }
}

__device__ __noinline__ void give_up_call(const BlockNormArgs& a, int res_dtype, uint64_t* full, int depth, int64_t t,
                                          int s, int phase) {
  give_up(a, res_dtype, full, depth, t, s, phase);
}

// A block a row at a time, rows gridDim.x apart; thread 0 keeps `depth` rows of bulk copies ahead, so DRAM is busy
// while the block reduces.  Several small blocks an SM hide each other's reductions.  Measured (bf16): norm of
// 8192 x 5120 31.0 us (5.4 of 6.45 TB/s), join 59.8 us (5.6 TB/s), int8 rows of 4096 x 17408 34.9 us (6.1 TB/s).
// The issue slots are 65 to 69 % busy then, 17 instructions an element of the norm, 33 of the join: they and the
// reductions' latency bound it, not DRAM.
// Layer norms take a second reduction (43.4 us), norms to int8 another and three more instructions a value (42.6 us),
// odd widths two loads for eight parameters (4096 x 8001: 34.0 us, 8000: 27.8 us) and a store a value to int8 (74 us).
template <typename T, typename R, Mode MODE, int VPT, bool EXACT>
__global__ void __launch_bounds__(RingShape<MODE, VPT, EXACT>::kThreads, RingShape<MODE, VPT, EXACT>::kBlocks)
    ring_kernel(const __grid_constant__ BlockNormArgs a, int depth) {
  using P = ParamType<T, R, MODE>;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ uint64_t full[kMaxDepth];
  __shared__ volatile int missing[2][kMaxDepth];  // by the phase and slot of a row whose copies did not arrive
  __shared__ __align__(16) float scratch[2 * kMaxWarps];
  constexpr int kResidual = MODE == kJoin ? sizeof(R) : 0;
  const int y_bytes = slot_bytes(a.hidden, sizeof(T)), bytes = y_bytes + slot_bytes(a.hidden, kResidual);
  const uint64_t policy = policy_evict_first();
  BlockTeam::clear(scratch);
  if (threadIdx.x == 0) {
    for (int s = 0; s < depth; ++s) mbar_init(&full[s], 1), missing[0][s] = missing[1][s] = 0;
    fence_barrier_init();
  }
  __syncthreads();
  grid_dependency_wait();
  grid_dependency_trigger();
  const T* y = static_cast<const T*>(a.y);
  const R* res = static_cast<const R*>(a.res);
  const auto fetch = [&](int64_t t, int s) {
    const int shift = EXACT ? 0 : row_shift(a, t);
    const RowCopy c(a, t, shift);
    mbar_arrive_expect_tx(&full[s], max(0, c.hi - c.lo) * 8 * (static_cast<int>(sizeof(T)) + kResidual));
    copy_row(ring + s * bytes, y + t * a.ldy, c, shift, &full[s], policy);
    if (MODE == kJoin) copy_row(ring + s * bytes + y_bytes, res + t * a.ld_res, c, shift, &full[s], policy);
  };
  if (threadIdx.x == 0)
    for (int s = 0; s < depth; ++s) {
      const int64_t t = blockIdx.x + static_cast<int64_t>(s) * gridDim.x;
      if (t < a.rows) fetch(t, s);
    }
  BlockTeam team = {scratch};
  int s = 0, phase = 0;
  // Where the way out of a wait that ran out stands decides the loop's registers: behind the loop for norms of two
  // whole granules a thread (4096 x 8000 27.8 us, 34.8 with a call from inside), a call for the others (norm of 4096 x
  // 8001 34.0 and 48.4 us; join of 4096 x 12288 73.4 and 85.7, rows to int8 of 4096 x 17408 34.9 and 36.0).  Inline
  // inside the loop it costs the norms 15 %.
  constexpr bool kGiveUpLast = EXACT && VPT == 2 && MODE == kNorm;
  int64_t lost = a.rows;
  for (int64_t t = blockIdx.x; t < a.rows; t += gridDim.x) {
    const int shift = EXACT ? 0 : row_shift(a, t);
    const GranuleMap<EXACT> m = {a.hidden, shift, static_cast<int>(threadIdx.x), static_cast<int>(blockDim.x)};
    const RowCopy c(a, t, shift);
    const uint8_t* slot = ring + s * bytes;
    if (!mbar_wait_suspended<true>(&full[s], phase, a.wait_ns)) missing[phase][s] = 1;
    Pack8<T> words[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) words[i] = load_slot(slot, y + t * a.ldy, c, m, i);
    float v[VPT][8];
    if (MODE != kQuantize)
#pragma unroll
      for (int i = 0; i < VPT; ++i) widen(words[i], v[i]);
    if (MODE == kJoin) {
      normalise<T>(v, a.post, a.inv_hidden, m, team);
      apply_gate<T>(v, a, t, m);
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        float r[8];
        widen(load_slot(slot + y_bytes, res + t * a.ld_res, c, m, i), r);
        join8<R>(v[i], r, a, t, m, i);
      }
    }
    // The slot has been read; by a thread whose wait ran out perhaps too early, and then the block writes NaN over what
    // it made of the row.  A thread that is a row ahead of this test marks that row's own entry.
    __syncthreads();
    if (missing[phase][s] != 0) {
      if (kGiveUpLast) {
        lost = t;
        break;
      }
      give_up_call(a, code_of<R>(), full, depth, t, s, phase);
      return;
    }
    const int64_t ahead = t + static_cast<int64_t>(depth) * gridDim.x;
    if (threadIdx.x == 0 && ahead < a.rows) fetch(ahead, s);
    if (MODE == kQuantize)
      quantize_row(words, a, t, m, team);
    else
      finish_row<P>(v, a, t, m, team);
    if (++s == depth) s = 0, phase ^= 1;
  }
  if (kGiveUpLast && lost < a.rows) give_up(a, code_of<R>(), full, depth, lost, s, phase);
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------

// Whether a tensor's rows (es-byte elements, ld apart) start on 16 bytes in the granules of x's rows.
bool same_granules(const void* p, int64_t ld, int es, const BlockNormArgs& a) {
  return (reinterpret_cast<uintptr_t>(p) - static_cast<uintptr_t>(a.shift0) * es) % 16 == 0 &&
         (a.rows == 1 || ((ld - a.ldy) * es) % 16 == 0);
}

// A launch that may start while the launch ahead of it finishes.
template <typename K, typename... A>
bool launch_early(K kernel, unsigned grid, int threads, size_t smem, cudaStream_t stream, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_ok(cudaLaunchKernelEx(&cfg, kernel, args...));
}

template <typename T, typename R, Mode MODE, int VPT, bool EXACT>
bool launch_ring(const BlockNormArgs& a, int granules, int device, cudaStream_t stream) {
  auto* kernel = ring_kernel<T, R, MODE, VPT, EXACT>;
  if (!ensure_max_dynamic_smem(reinterpret_cast<const void*>(kernel), device)) return false;
  const int threads = ((granules + VPT - 1) / VPT + 31) / 32 * 32;
  const int slot = slot_bytes(a.hidden, sizeof(T)) + (MODE == kJoin ? slot_bytes(a.hidden, sizeof(R)) : 0);
  // Blocks an SM: as many as their registers allow, with at least two rows each in the ring's room; what is left
  // deepens the rings.
  static const int regs = [&] {
    cudaFuncAttributes attr;
    return cudaFuncGetAttributes(&attr, kernel) == cudaSuccess ? (attr.numRegs + 7) / 8 * 8 : 128;
  }();
  const int resident = std::max(1, std::min(65536 / (regs * threads), kMostThreads / threads));
  const int blocks = std::max(1, std::min(resident, kRoom / (2 * slot)));
  const int64_t grid = std::min<int64_t>(a.rows, static_cast<int64_t>(device_info(device).num_sms) * blocks);
  const int64_t each = (a.rows + grid - 1) / grid;
  const int rows_each = std::max(kDeepRoom / (blocks * slot), std::min(2, kRoom / (blocks * slot)));
  const int depth = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({kMaxDepth, rows_each, each})));
  return launch_early(kernel, static_cast<unsigned>(grid), threads, static_cast<size_t>(depth) * slot, stream, a,
                      depth);
}

template <typename T, typename R, Mode MODE, bool EXACT>
bool launch_granules(const BlockNormArgs& a, int granules, int device, cudaStream_t stream) {
  const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(a.rows) + kWarpRows - 1) / kWarpRows);
  if (granules <= 32) return launch_early(warp_kernel<T, R, MODE, 1, EXACT>, grid, 32 * kWarpRows, 0, stream, a);
  if (granules <= 64) return launch_early(warp_kernel<T, R, MODE, 2, EXACT>, grid, 32 * kWarpRows, 0, stream, a);
  if (granules <= 128) return launch_early(warp_kernel<T, R, MODE, 4, EXACT>, grid, 32 * kWarpRows, 0, stream, a);
  if constexpr (EXACT) {
    // Many rows: a warp takes up to 192 granules, or 256 when it only quantises (8192 rows of 1536 bf16: norm 11.5 us
    // against the ring's 14.8, int8 7.3 against 10.8; 2048: int8 9.3 against 11.9, but norm 15.7 against 15.4).  Few
    // rows: a block's more threads have less latency (500 layer norms of 1536: 3.8 us and 3.3 us).  Around kManyRows, a
    // warp and the ring: 2048 rows of 1536 norm 4.1 and 3.7 us, join 6.1 and 6.9, int8 2.4 and 3.8; 4096 rows 5.1 and
    // 6.0, 10.7 and 12.2, 3.7 and 5.6; 1024 rows 3.6 and 2.9, 4.8 and 5.1, 1.9 and 2.9.
    if (a.rows >= kManyRows && granules <= 192)
      return launch_early(warp_kernel<T, R, MODE, 6, EXACT>, grid, 32 * kWarpRows, 0, stream, a);
    if constexpr (MODE == kQuantize)
      if (a.rows >= kManyRows && granules <= 256)
        return launch_early(warp_kernel<T, R, MODE, 8, EXACT>, grid, 32 * kWarpRows, 0, stream, a);
  }
  if (granules <= 2 * RingShape<MODE, 2, EXACT>::kThreads)
    return launch_ring<T, R, MODE, 2, EXACT>(a, granules, device, stream);
  if (granules <= 4 * RingShape<MODE, 4, EXACT>::kThreads)
    return launch_ring<T, R, MODE, 4, EXACT>(a, granules, device, stream);
  return launch_ring<T, R, MODE, 8, EXACT>(a, granules, device, stream);
}

template <typename T, typename R, Mode MODE>
bool launch_rows(BlockNormArgs a, int dtype, int res_dtype, int device, cudaStream_t stream) {
  constexpr int es = sizeof(T), rs = sizeof(R);
  // The granule kernels take parameters and outputs in ParamType or fp32, gates in T or fp32.
  constexpr int kParams = code_of<ParamType<T, R, MODE>>();
  const auto known = [&](int d) { return d == kParams || d == QCC_DTYPE_F32; };
  const auto known_norm = [&](const qcc_norm_params& p) {
    return (p.weight == nullptr && p.bias == nullptr) || known(p.dtype);
  };
  a.inv_hidden = 1.f / static_cast<float>(a.hidden);
  a.wait_ns = wait_limit_ns();
  a.shift0 = static_cast<int>(reinterpret_cast<uintptr_t>(a.y) / es % 8);
  const bool row_gate = a.gate.values != nullptr && a.gate.cols > 1;
  const bool together =
      known_norm(a.post) && known_norm(a.next) && (!row_gate || known(a.gate.dtype)) &&
      same_granules(a.y, a.ldy, es, a) &&
      (MODE != kJoin || (same_granules(a.res, a.ld_res, rs, a) && same_granules(a.res_out, a.ld_res_out, rs, a))) &&
      (a.out == nullptr || a.out_dtype == QCC_DTYPE_I8 ||
       (known(a.out_dtype) && same_granules(a.out, a.ld_out, dtype_bytes(a.out_dtype), a)));
  const bool shifted = a.shift0 != 0 || (a.rows > 1 && a.ldy % 8 != 0);
  const int granules = (a.hidden + (shifted ? 14 : 7)) / 8;
  const int slot = slot_bytes(a.hidden, es) + (MODE == kJoin ? slot_bytes(a.hidden, rs) : 0);
  const bool fits = granules <= 4096 && slot <= kRoom;
  if (!together || !fits) {
    const int threads = std::min(512, (a.hidden + 31) / 32 * 32);
    return launch_early(plain_kernel, static_cast<unsigned>(a.rows), threads, 0, stream, a, dtype, res_dtype);
  }
  a.gate_in_granules =
      row_gate && a.gate.rows_each == 1 && a.gate.dtype == dtype && same_granules(a.gate.values, a.gate.ld, es, a);
  const bool gate_exact = !row_gate || a.gate_in_granules ||
                          (aligned16(a.gate.values) && (a.gate.ld * dtype_bytes(a.gate.dtype)) % 16 == 0);
  const bool exact = !shifted && a.hidden % 8 == 0 && aligned16(a.post.weight) && aligned16(a.post.bias) &&
                     aligned16(a.next.weight) && aligned16(a.next.bias) && gate_exact &&
                     (a.out == nullptr || a.out_dtype != QCC_DTYPE_I8 || (aligned16(a.out) && a.ld_out % 8 == 0));
  return exact ? launch_granules<T, R, MODE, true>(a, granules, device, stream)
               : launch_granules<T, R, MODE, false>(a, granules, device, stream);
}

}  // namespace
}  // namespace qcc
