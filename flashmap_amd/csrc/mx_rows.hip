// Rows to microscaled form (mx_device.h) and back: quantization with an MLP's activation on
// the way, and the two norms in front of the projections (root mean square with the
// residual's addition; the DiT's gated residual and modulated LayerNorm), which then write
// 8 (or 4) bits a value in place of 16.
//
// Bound: HBM for prompts and full batches, latency for one user's 16 rows. A thread holds 8
// consecutive values (one 16-byte load of bf16), so that a block of 32 is four neighbouring
// lanes and its maximum two DPP steps.
//
// Everything between the inputs and the codes is float32, rounded once: the residual stream
// is stored rounded to bf16, the norm is taken of the unrounded sum.
#include <limits.h>

#include <type_traits>

#include "fm_host.h"
#include "mx_device.h"

namespace fm {

constexpr int ROW_THREADS = 256;
constexpr int64_t MAX_ITEMS = (int64_t)1 << 30;  // threads per launch (a launch counts at most 2^32)

// Quad-wide maximum (lanes 4 i .. 4 i + 3), the same bits in all four.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  const uint32_t a = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, true);  // quad_perm [1, 0, 3, 2]
  v = v > a ? v : a;
  const uint32_t b = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, true);  // quad_perm [2, 3, 0, 1]
  return v > b ? v : b;
}

// 8 values of a row from column c, zeros from `cols` on; `vec`: 16-byte loads are aligned.
template <typename T>
__device__ __forceinline__ float to_f32(T v);
struct bf16_raw { uint16_t v; };
template <>
__device__ __forceinline__ float to_f32<bf16_raw>(bf16_raw v) { return bf16_to_f32(v.v); }
template <>
__device__ __forceinline__ float to_f32<_Float16>(_Float16 v) { return (float)v; }
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }

template <typename T>
__device__ __forceinline__ void load8(const T *row, int32_t c, int32_t cols, bool vec, float (&v)[8]) {
  if (vec && c + 8 <= cols) {
    if constexpr (sizeof(T) == 4) {
      const f32x4_t a = *reinterpret_cast<const f32x4_t *>(row + c), b = *reinterpret_cast<const f32x4_t *>(row + c + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
    } else {
      const u32x4_t a = load16(row + c);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, bf16_raw>::value)
          v[2 * i] = bf16_lo(a[i]), v[2 * i + 1] = bf16_hi(a[i]);
        else
          v[2 * i] = f16_lo(a[i]), v[2 * i + 1] = f16_hi(a[i]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? to_f32(row[c + i]) : 0.f;
  }
}

__device__ __forceinline__ void store8_bf16(uint16_t *row, int32_t c, int32_t cols, bool vec, const float (&v)[8]) {
  if (vec && c + 8 <= cols) {
    u32x4_t w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
    store16(row + c, w);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < cols) row[c + i] = (uint16_t)(pack_bf16x2(v[i], 0.f) & 0xffffu);
  }
}

// The codes of 8 values (four neighbouring lanes hold a block) and, from the block's first
// lane, its scale byte. Every lane of the quad has to call this.
template <int BITS>
__device__ __forceinline__ void store_block(const float (&v)[8], int32_t c, uint8_t *codes, uint8_t *scales) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t m = magnitude(v[i]);
    top = top > m ? top : m;
  }
  const uint32_t byte = mx_scale_byte<BITS>(quad_max(top));
  const float scale = mx_scale_value(byte);
  if constexpr (BITS == 8)
    *reinterpret_cast<u32x2_t *>(codes + c) =
        u32x2_t{mx_pack_e4m3x4(v[0], v[1], v[2], v[3], scale), mx_pack_e4m3x4(v[4], v[5], v[6], v[7], scale)};
  else
    *reinterpret_cast<uint32_t *>(codes + (c >> 1)) = mx_pack_e2m1x8(v, scale);
  if ((c & 31) == 0) scales[c >> 5] = (uint8_t)byte;
}

// item / chunks for item < 2^30 and 16 <= chunks <= 2^23, by a multiplication: with 2^l >= chunks
// and magic = floor(2^(30 + l) / chunks) + 1 the quotient is off by less than 2^-l <= 1 / chunks,
// and never past the next integer.
struct RowOf {
  uint32_t magic, shift;
  explicit RowOf(uint32_t chunks) {
    shift = 0;
    while ((1u << shift) < chunks) ++shift;
    magic = (uint32_t)(((uint64_t)1 << (30 + shift)) / chunks + 1);
    shift -= 2;
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t item) const { return __umulhi(item, magic) >> shift; }
};

// -------------------------------------------------------------------------- quantization

struct QuantArgs {
  const void *x;
  uint8_t *codes, *scales;
  int64_t xs, cs, ss;  // row strides (elements, bytes, bytes)
  int64_t rows;
  int32_t cols;
  uint32_t chunks;  // 8-value chunks of a stored row
  RowOf row_of;
  int32_t vec;
};

enum { ACT_NONE = 0, ACT_GELU = 1, ACT_SWIGLU = 2 };

// x Phi(x) = max(x, 0) - h, h = |x| / 2 erfc(|x| / sqrt 2): nothing cancels (h is at most half of
// |x|). erfc(z) = exp(-z^2) erfcx(z), and erfcx(a / sqrt 2) / 2 is a polynomial in 1 / (1 + 0.23 a),
// fitted to 5e-8 of its value for a up to 14.5 (least squares in Chebyshev polynomials,
// reweighted towards the largest relative error). Over all bf16 x, with a correctly rounded
// reciprocal and exponential, h comes to 5.4e-7 of its value for |x| below 4 and 3.8e-6 below 13.2
// (the rounding of the exponential's argument, which grows with x^2); beyond it is 0 (the
// exponential is below 2^-126). 16 of the 65280 finite bf16 x get another e4m3 code than the value
// rounded to float32 has, 5 another e2m1 code: a midpoint lies between the two. A third of erfcf's
// instructions, which bounded the pass (1024 x 8192, 25 MB: 14.9 us). Infinities and NaN give NaN.
__device__ __forceinline__ float gelu(float x) {
#pragma clang fp contract(off)
  const float a = fabsf(x);
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.23f, a, 1.f));
  float p = -0.0784958884f;
  p = __builtin_fmaf(p, t, 0.290552796f);
  p = __builtin_fmaf(p, t, -0.278415741f);
  p = __builtin_fmaf(p, t, 0.301807729f);
  p = __builtin_fmaf(p, t, -0.0331565229f);
  p = __builtin_fmaf(p, t, 0.119617817f);
  p = __builtin_fmaf(p, t, 0.0857352587f);
  p = __builtin_fmaf(p, t, 0.0923825472f);
  p = __builtin_fmaf(p, t, -2.80193462e-5f);
  const float e = __builtin_amdgcn_exp2f(a * a * -0.721347520f);  // exp(-a^2 / 2)
  return fmaxf(x, 0.f) - a * (e * p);
}
// gate / (1 + exp(-gate)) * up for gate from -87 on: the exponential with what its argument lost
// put back, the quotient by a refined reciprocal. The quotient is a normal float of at most 1 (a
// gate past 104 has 1), so that only the result can overflow.
__device__ __forceinline__ float swiglu(float gate, float up) {
#pragma clang fp contract(off)
  const float y = fmaxf(-gate, -104.f);
  const float u = y * 1.44269504f;
  const float r = __builtin_fmaf(y, 1.92596299e-8f, __builtin_fmaf(y, 1.44269504f, -u));
  const float e = __builtin_amdgcn_exp2f(u);
  const float d = 1.f + __builtin_fmaf(e * 0.693147182f, r, e);
  float q = __builtin_amdgcn_rcpf(d);
  q = __builtin_fmaf(__builtin_fmaf(-d, q, 1.f), q, q);
  return gate * q * up;
}
// The gates whose quotient is subnormal (or whose gate times quotient may be) while the result
// need not be: mantissas are multiplied and exponents added, for negative gates as gate
// exp(gate) / (1 + exp(gate)) * up with exp(-|gate|) = 2^n e, e from 0.7 to 1.42. -200 stands
// for what lies below it: with any up the result is below half of the smallest float. -inf gives
// NaN, as -inf times 0 does. Taken for every value this makes the pass a third longer (1024 x 8192);
// where no gate needs it the test for it is 5 %.
__device__ __forceinline__ bool swiglu_is_wide(float gate) { return gate < -87.f || fabsf(gate) < 0x1p-100f; }
__device__ __forceinline__ float swiglu_wide(float gate, float up) {
#pragma clang fp contract(off)
  const float g = gate < -200.f ? (gate - gate) - 200.f : gate;
  const float y = fminf(fabsf(gate), 200.f);
  const float u = y * -1.44269504f;
  const float r = __builtin_fmaf(y, -1.92596299e-8f, __builtin_fmaf(y, -1.44269504f, -u));
  const float n = rintf(u);
  const float p = __builtin_amdgcn_exp2f(u - n);
  const float e = __builtin_fmaf(p * 0.693147182f, r, p);
  const float d = 1.f + __builtin_ldexpf(e, (int)n);
  const float v = __builtin_amdgcn_frexp_mantf(g) * __builtin_amdgcn_frexp_mantf(up) * __fdiv_rn(gate < 0.f ? e : 1.f, d);
  return __builtin_ldexpf(v, __builtin_amdgcn_frexp_expf(g) + __builtin_amdgcn_frexp_expf(up) + (gate < 0.f ? (int)n : 0));
}

// A thread per 8 values, no loop: every load of the call is in flight at once, and the rows need
// nothing of each other. Bound: HBM without an activation (24576 x 2048 bf16 to 4 bits and back
// 42.5 us, 6.0 TB/s, a copy's rate at this size) and with SwiGLU (1024 x 8192 bf16 8.8 us, 4.8 TB/s), VALU
// issue with GELU (1024 x 8192 bf16 to 8 bits 8.6 us, 2.9 TB/s, 32 instructions a value).
template <typename T, int BITS, int ACT>
__global__ __launch_bounds__(ROW_THREADS) void mx_quantize_kernel(const QuantArgs a) {
  const uint32_t item = blockIdx.x * ROW_THREADS + threadIdx.x;
  const uint32_t row = a.row_of(item);
  if (row >= a.rows) return;  // chunks of a row are a multiple of 16: whole quads leave
  const int32_t c = 8 * (int32_t)(item - row * a.chunks);
  const T *x = (const T *)a.x + row * a.xs;
  float v[8];
  load8(x, c, a.cols, a.vec != 0, v);
  if constexpr (ACT == ACT_GELU) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = gelu(v[i]);
  } else if constexpr (ACT == ACT_SWIGLU) {
    float u[8], w[8], low = 0.f, least = 1.f;
    load8(x + a.cols, c, a.cols, a.vec != 0 && a.cols % 8 == 0, u);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      low = fminf(low, v[i]), least = fminf(least, fabsf(v[i]));
      w[i] = swiglu(v[i], u[i]);
    }
    if (c < a.cols && (low < -87.f || least < 0x1p-100f)) {  // rare
      for (int i = 0; i < 8; ++i)
        if (swiglu_is_wide(v[i])) w[i] = swiglu_wide(v[i], u[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = w[i];
  }
  store_block<BITS>(v, c, a.codes + row * a.cs, a.scales + row * a.ss);
}

// ------------------------------------------------------------------------- reading back

struct DequantArgs {
  const uint8_t *codes, *scales;
  void *out;
  int64_t cs, ss, os;
  int64_t rows;
  int32_t cols;
  uint32_t chunks;
  RowOf row_of;
  int32_t vec;
};

// Bound: HBM to bf16 (24576 x 2048 of 4 bits 19.7 us, 6.5 TB/s); fp16 and fp32 leave value by value, 62
// and 121 us, 2 TB/s.
template <typename T, int BITS>
__global__ __launch_bounds__(ROW_THREADS) void mx_dequantize_kernel(const DequantArgs a) {
  const uint32_t item = blockIdx.x * ROW_THREADS + threadIdx.x;
  const uint32_t row = a.row_of(item);
  if (row >= a.rows) return;
  const int32_t c = 8 * (int32_t)(item - row * a.chunks);
  if (c >= a.cols) return;
  const uint32_t byte = a.scales[row * a.ss + (c >> 5)];
  const float scale = byte == 255u ? __uint_as_float(0x7fc00000u) : mx_scale_value(byte);
  float v[8];
  typedef __attribute__((ext_vector_type(2))) float f32x2_t;
  if constexpr (BITS == 8) {
    const u32x2_t w = *reinterpret_cast<const u32x2_t *>(a.codes + row * a.cs + c);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
      v[4 * i] = lo[0] * scale, v[4 * i + 1] = lo[1] * scale, v[4 * i + 2] = hi[0] * scale, v[4 * i + 3] = hi[1] * scale;
    }
  } else {
    const uint32_t w = *reinterpret_cast<const uint32_t *>(a.codes + row * a.cs + (c >> 1));
    const f32x2_t p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 1);
    const f32x2_t p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 3);
    v[0] = p0[0] * scale, v[1] = p0[1] * scale, v[2] = p1[0] * scale, v[3] = p1[1] * scale;
    v[4] = p2[0] * scale, v[5] = p2[1] * scale, v[6] = p3[0] * scale, v[7] = p3[1] * scale;
  }
  if constexpr (std::is_same<T, bf16_raw>::value) {
    store8_bf16((uint16_t *)a.out + row * a.os, c, a.cols, a.vec != 0, v);
  } else {
    T *out = (T *)a.out + row * a.os;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < a.cols) out[c + i] = (T)v[i];
  }
}

// --------------------------------------------------------------------------------- norms

struct NormArgs {
  const uint16_t *x, *y;          // y NULL: nothing is added
  const uint16_t *gate;           // NULL: y is added as it is
  const float *weight;            // root mean square: the weights; else NULL
  const uint16_t *scale, *shift;  // modulated LayerNorm
  uint16_t *x_out;                // NULL: the stream is not stored
  uint8_t *codes, *scales;
  int64_t xs, ys, xos, cs, ss;
  int64_t rows;
  int32_t cols, gate_rows;
  uint32_t chunks;
  int32_t vec_x, vec_y, vec_p, vec_o;  // which rows may be read or written 16 bytes at a time
  float eps;
};

// The sum over a wavefront, the same bits in every lane.
__device__ __forceinline__ float wave_sum(float v) {
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x128, 0xf, 0xf, true));  // row_ror 8
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x124, 0xf, 0xf, true));
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x122, 0xf, 0xf, true));
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x121, 0xf, 0xf, true));
  return sum_over_groups(v);
}
// The sum over a row's TPR threads; lds: a place of its own per sum.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float *lds) {
  v = wave_sum(v);
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) lds[wave_id()] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < TPR / 64; ++w) v += lds[w];
  }
  return v;
}

// s = x + y or x + gate y, the stream; then s rsqrt(mean s^2 + eps) weight (RMS), or the LayerNorm
// (s - mean) rsqrt(var + eps) (1 + scale) + shift, its variance of the differences from the mean.
// TPR threads a row, NCH 8-value pieces each, held in registers between the one read and the one
// write. Bound: HBM for many rows (8192 x 4096 with a residual 42.3 us, 5.6 TB/s), a launch and a
// round trip for few (16 x 2048 3.0 us, 1024 x 2048 5.3 us).
// EARLY: the row-independent operands are loaded with the row, not after its statistics (one
// round trip less, for as many registers).
template <int TPR, int NCH, bool RMS, int BITS, bool EARLY>
__global__ __launch_bounds__(ROW_THREADS) void mx_norm_kernel(const NormArgs a) {
  __shared__ float lds[2][ROW_THREADS / 64];
  const int t = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * (ROW_THREADS / TPR) + threadIdx.x / TPR;
  if (row >= a.rows) return;  // a whole wavefront, and with TPR 256 a whole workgroup
  float v[NCH][8], p[EARLY ? NCH : 1][8], q[EARLY && !RMS ? NCH : 1][8];
  auto operands = [&](int32_t c, float (&pc)[8], float (&qc)[8]) {
    if constexpr (RMS) {
      load8(a.weight, c, a.cols, a.vec_p != 0, pc);
    } else {
      load8((const bf16_raw *)a.scale, c, a.cols, a.vec_p != 0, pc);
      load8((const bf16_raw *)a.shift, c, a.cols, a.vec_p != 0, qc);
    }
  };
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int32_t c = 8 * (t + TPR * i);
    load8((const bf16_raw *)a.x + row * a.xs, c, a.cols, a.vec_x != 0, v[i]);
    if (a.y != nullptr) {
      float y[8], g[8];
      load8((const bf16_raw *)a.y + row * a.ys, c, a.cols, a.vec_y != 0, y);
      if (a.gate == nullptr) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] += y[j];
      } else {
        if (a.gate_rows) {
          const float gr = bf16_to_f32(a.gate[row]);
#pragma unroll
          for (int j = 0; j < 8; ++j) g[j] = gr;
        } else {
          load8((const bf16_raw *)a.gate, c, a.cols, a.vec_p != 0, g);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = __builtin_fmaf(g[j], y[j], v[i][j]);
      }
    }
    if constexpr (EARLY) operands(c, p[i], q[RMS ? 0 : i]);
  }
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int32_t c = 8 * (t + TPR * i);
    if (a.x_out != nullptr && c < a.cols) store8_bf16(a.x_out + row * a.xos, c, a.cols, a.vec_o != 0, v[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += RMS ? v[i][j] * v[i][j] : v[i][j];
  }
  const float n = (float)a.cols;
  sum = row_sum<TPR>(sum, lds[0]);
  float mean = 0.f;
  if constexpr (!RMS) {
    mean = __fdiv_rn(sum, n);
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float d = 8 * (t + TPR * i) + j < a.cols ? v[i][j] - mean : 0.f;
        sum += d * d;
      }
    sum = row_sum<TPR>(sum, lds[1]);
  }
  // Rounded correctly: an ulp here moves every value of the row, and codes past their midpoints.
  const float r = __fdiv_rn(1.f, __fsqrt_rn(__fdiv_rn(sum, n) + a.eps));
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int32_t c = 8 * (t + TPR * i);
    if (c >= 8 * (int32_t)a.chunks) break;  // whole quads: chunks is a multiple of 16
    if constexpr (!EARLY) operands(c, p[0], q[0]);
    float(&pc)[8] = p[EARLY ? i : 0], (&qc)[8] = q[EARLY && !RMS ? i : 0];
    if constexpr (RMS) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] * r * pc[j];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[i][j] = c + j < a.cols ? __builtin_fmaf((v[i][j] - mean) * r, 1.f + pc[j], qc[j]) : 0.f;
    }
    store_block<BITS>(v[i], c, a.codes + row * a.cs, a.scales + row * a.ss);
  }
}

static bool aligned(const void *p, int64_t n) { return ((uintptr_t)p % (uintptr_t)n) == 0; }
static bool vec_rows(const void *p, int64_t stride, int64_t size) { return aligned(p, 16) && stride * size % 16 == 0; }

// What every call checks of its microscaled rows.
static int check_rows(const void *codes, int64_t codes_stride, const void *scales, int64_t scales_stride, int32_t bits,
                      int64_t cols) {
  FM_REQUIRE(bits == 4 || bits == 8, "bits %d: 4 or 8", bits);
  FM_REQUIRE(codes && scales, "NULL codes or scales");
  FM_REQUIRE(aligned(codes, 16) && codes_stride % 16 == 0 && codes_stride >= mx_padded(cols) * bits / 8,
             "codes must be 16-byte aligned rows of %lld bytes", (long long)(mx_padded(cols) * bits / 8));
  FM_REQUIRE(aligned(scales, 4) && scales_stride % 4 == 0 && scales_stride >= mx_padded(cols) / MX_BLOCK,
             "scales must be 4-byte aligned rows of %lld bytes", (long long)(mx_padded(cols) / MX_BLOCK));
  return FM_OK;
}

// f(first row, rows) for slices of at most MAX_ITEMS threads.
template <typename F>
static int by_slices(int64_t rows, int64_t threads_per_row, F f) {
  const int64_t most = MAX_ITEMS / threads_per_row;
  for (int64_t first = 0; first < rows; first += most) {
    f(first, rows - first < most ? rows - first : most);
    FM_CHECK_HIP(hipGetLastError());
  }
  return FM_OK;
}

template <typename F>
static void by_dtype(int32_t dtype, F f) {
  if (dtype == 0)
    f(bf16_raw{});
  else if (dtype == 1)
    f((_Float16)0);
  else
    f(0.f);
}

static int launch_norm(const NormArgs &base, bool rms, int32_t bits, hipStream_t stream) {
  // Rows of up to 512 values: a wavefront each; longer ones: a workgroup each.
  const int tpr = base.chunks <= 64 ? 64 : 256;
  const int nch = (int)((base.chunks + tpr - 1) / tpr);
  return by_slices(base.rows, tpr, [&](int64_t first, int64_t rows) {
    NormArgs a = base;
    a.rows = rows;
    a.x += first * a.xs;
    if (a.y) a.y += first * a.ys;
    if (a.gate && a.gate_rows) a.gate += first;
    if (a.x_out) a.x_out += first * a.xos;
    a.codes += first * a.cs;
    a.scales += first * a.ss;
    const int per = ROW_THREADS / tpr;
    const dim3 grid((unsigned)((rows + per - 1) / per));
    auto go = [&](auto t, auto c, auto r, auto b) {
      constexpr int NCH = decltype(c)::value;
      mx_norm_kernel<decltype(t)::value, NCH, decltype(r)::value, decltype(b)::value, NCH <= 2>
          <<<grid, dim3(ROW_THREADS), 0, stream>>>(a);
    };
    auto with_bits = [&](auto t, auto c, auto r) {
      if (bits == 8)
        go(t, c, r, std::integral_constant<int, 8>{});
      else
        go(t, c, r, std::integral_constant<int, 4>{});
    };
    auto with_kind = [&](auto t, auto c) {
      if (rms)
        with_bits(t, c, std::true_type{});
      else
        with_bits(t, c, std::false_type{});
    };
    if (tpr == 64)
      with_kind(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
    else if (nch <= 1)
      with_kind(std::integral_constant<int, 256>{}, std::integral_constant<int, 1>{});
    else if (nch <= 2)
      with_kind(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
    else if (nch <= 4)
      with_kind(std::integral_constant<int, 256>{}, std::integral_constant<int, 4>{});
    else
      with_kind(std::integral_constant<int, 256>{}, std::integral_constant<int, 8>{});
  });
}

}  // namespace fm

extern "C" int fm_mx_quantize(const void *x, int32_t dtype, int64_t x_stride, int32_t activation, int32_t bits,
                              void *codes, int64_t codes_stride, void *scales, int64_t scales_stride, int64_t rows,
                              int64_t cols, void *stream) {
  using namespace fm;
  FM_REQUIRE(rows >= 0 && cols > 0, "bad sizes: rows=%lld cols=%lld", (long long)rows, (long long)cols);
  if (rows == 0) return FM_OK;
  FM_REQUIRE(dtype >= 0 && dtype <= 2, "dtype %d: 0 bf16, 1 fp16, 2 fp32", dtype);
  FM_REQUIRE(activation >= 0 && activation <= 2, "activation %d: 0 none, 1 gelu, 2 swiglu", activation);
  if (cols > 1 << 26) return fail(FM_ERR_UNSUPPORTED, "rows of %lld values: at most 2^26", (long long)cols);
  const int64_t width = activation == ACT_SWIGLU ? 2 * cols : cols;
  const int64_t size = dtype == 2 ? 4 : 2;
  FM_REQUIRE(x != nullptr, "NULL tensor pointer");
  FM_REQUIRE(aligned(x, size) && (rows == 1 || x_stride >= width), "rows of x overlap: stride %lld, %lld values",
             (long long)x_stride, (long long)width);
  const int rc = check_rows(codes, codes_stride, scales, scales_stride, bits, cols);
  if (rc != FM_OK) return rc;
  const int64_t chunks = mx_padded(cols) / 8;
  return by_slices(rows, chunks, [&](int64_t first, int64_t n) {
    by_dtype(dtype, [&](auto tag) {
      typedef decltype(tag) T;
      QuantArgs a{(const T *)x + first * x_stride, (uint8_t *)codes + first * codes_stride,
                  (uint8_t *)scales + first * scales_stride, x_stride, codes_stride, scales_stride, n, (int32_t)cols,
                  (uint32_t)chunks, RowOf((uint32_t)chunks), vec_rows(x, x_stride, size)};
      const dim3 grid((unsigned)((n * chunks + ROW_THREADS - 1) / ROW_THREADS));
      auto go = [&](auto b, auto act) {
        mx_quantize_kernel<T, decltype(b)::value, decltype(act)::value>
            <<<grid, dim3(ROW_THREADS), 0, (hipStream_t)stream>>>(a);
      };
      auto with_act = [&](auto b) {
        if (activation == ACT_GELU)
          go(b, std::integral_constant<int, ACT_GELU>{});
        else if (activation == ACT_SWIGLU)
          go(b, std::integral_constant<int, ACT_SWIGLU>{});
        else
          go(b, std::integral_constant<int, ACT_NONE>{});
      };
      if (bits == 8)
        with_act(std::integral_constant<int, 8>{});
      else
        with_act(std::integral_constant<int, 4>{});
    });
  });
}

extern "C" int fm_mx_dequantize(const void *codes, int64_t codes_stride, const void *scales, int64_t scales_stride,
                                int32_t bits, void *out, int32_t dtype, int64_t out_stride, int64_t rows, int64_t cols,
                                void *stream) {
  using namespace fm;
  FM_REQUIRE(rows >= 0 && cols > 0, "bad sizes: rows=%lld cols=%lld", (long long)rows, (long long)cols);
  if (rows == 0) return FM_OK;
  FM_REQUIRE(dtype >= 0 && dtype <= 2, "dtype %d: 0 bf16, 1 fp16, 2 fp32", dtype);
  if (cols > 1 << 26) return fail(FM_ERR_UNSUPPORTED, "rows of %lld values: at most 2^26", (long long)cols);
  const int64_t size = dtype == 2 ? 4 : 2;
  FM_REQUIRE(out != nullptr, "NULL tensor pointer");
  FM_REQUIRE(aligned(out, size) && (rows == 1 || out_stride >= cols), "rows of out overlap: stride %lld, %lld values",
             (long long)out_stride, (long long)cols);
  const int rc = check_rows(codes, codes_stride, scales, scales_stride, bits, cols);
  if (rc != FM_OK) return rc;
  const int64_t chunks = mx_padded(cols) / 8;
  return by_slices(rows, chunks, [&](int64_t first, int64_t n) {
    by_dtype(dtype, [&](auto tag) {
      typedef decltype(tag) T;
      DequantArgs a{(const uint8_t *)codes + first * codes_stride, (const uint8_t *)scales + first * scales_stride,
                    (T *)out + first * out_stride, codes_stride, scales_stride, out_stride, n, (int32_t)cols,
                    (uint32_t)chunks, RowOf((uint32_t)chunks), vec_rows(out, out_stride, size)};
      const dim3 grid((unsigned)((n * chunks + ROW_THREADS - 1) / ROW_THREADS));
      if (bits == 8)
        mx_dequantize_kernel<T, 8><<<grid, dim3(ROW_THREADS), 0, (hipStream_t)stream>>>(a);
      else
        mx_dequantize_kernel<T, 4><<<grid, dim3(ROW_THREADS), 0, (hipStream_t)stream>>>(a);
    });
  });
}

extern "C" int fm_rms_norm_mx(const void *x, int64_t x_stride, const void *residual, int64_t residual_stride,
                              const float *weight, float eps, void *x_out, int64_t x_out_stride, int32_t bits,
                              void *codes, int64_t codes_stride, void *scales, int64_t scales_stride, int64_t rows,
                              int32_t cols, void *stream) {
  using namespace fm;
  FM_REQUIRE(rows >= 0 && cols > 0, "bad sizes: rows=%lld cols=%d", (long long)rows, cols);
  if (rows == 0) return FM_OK;
  if (cols > 16384) return fail(FM_ERR_UNSUPPORTED, "rows of %d values: at most 16384", cols);
  FM_REQUIRE(x && weight && aligned(x, 2) && aligned(weight, 4), "x and weight must be given, aligned to their values");
  FM_REQUIRE((residual != nullptr) == (x_out != nullptr), "a residual and the stream x_out go together");
  FM_REQUIRE(rows == 1 || (x_stride >= cols && (!residual || (residual_stride >= cols && x_out_stride >= cols))),
             "row strides must cover a row");
  const int rc = check_rows(codes, codes_stride, scales, scales_stride, bits, cols);
  if (rc != FM_OK) return rc;
  NormArgs a{};
  a.x = (const uint16_t *)x, a.y = (const uint16_t *)residual, a.weight = weight, a.x_out = (uint16_t *)x_out;
  a.codes = (uint8_t *)codes, a.scales = (uint8_t *)scales;
  a.xs = x_stride, a.ys = residual_stride, a.xos = x_out_stride, a.cs = codes_stride, a.ss = scales_stride;
  a.rows = rows, a.cols = cols, a.chunks = (uint32_t)(mx_padded(cols) / 8), a.eps = eps;
  a.vec_x = vec_rows(x, x_stride, 2), a.vec_y = vec_rows(residual, residual_stride, 2);
  a.vec_p = aligned(weight, 16), a.vec_o = vec_rows(x_out, x_out_stride, 2);
  return launch_norm(a, true, bits, (hipStream_t)stream);
}

extern "C" int fm_adaln_residual_mx(const void *x, int64_t x_stride, const void *y, int64_t y_stride, const void *gate,
                                    int32_t gate_per_row, const void *scale, const void *shift, void *x_out,
                                    int64_t x_out_stride, float eps, int32_t bits, void *codes, int64_t codes_stride,
                                    void *scales, int64_t scales_stride, int64_t rows, int32_t cols, void *stream) {
  using namespace fm;
  FM_REQUIRE(rows >= 0 && cols > 0, "bad sizes: rows=%lld cols=%d", (long long)rows, cols);
  if (rows == 0) return FM_OK;
  if (cols > 16384) return fail(FM_ERR_UNSUPPORTED, "rows of %d values: at most 16384", cols);
  FM_REQUIRE(x && scale && shift, "NULL tensor pointer");
  FM_REQUIRE(!y || (gate && x_out), "a residual needs its gate and x_out");
  FM_REQUIRE(y || !x_out, "x_out without a residual");
  FM_REQUIRE(aligned(x, 2) && aligned(y, 2) && aligned(gate, 2) && aligned(scale, 2) && aligned(shift, 2) && aligned(x_out, 2),
             "tensors must be aligned to their values");
  FM_REQUIRE(x_stride == 0 || rows == 1 || x_stride >= cols, "row strides must cover a row");
  FM_REQUIRE(rows == 1 || !y || (y_stride >= cols && x_out_stride >= cols), "row strides must cover a row");
  FM_REQUIRE(x_stride != 0 || x != x_out || rows == 1, "x_out may not alias a shared x row");
  const int rc = check_rows(codes, codes_stride, scales, scales_stride, bits, cols);
  if (rc != FM_OK) return rc;
  NormArgs a{};
  a.x = (const uint16_t *)x, a.y = (const uint16_t *)y, a.gate = (const uint16_t *)gate;
  a.scale = (const uint16_t *)scale, a.shift = (const uint16_t *)shift, a.x_out = (uint16_t *)x_out;
  a.codes = (uint8_t *)codes, a.scales = (uint8_t *)scales;
  a.xs = x_stride, a.ys = y_stride, a.xos = x_out_stride, a.cs = codes_stride, a.ss = scales_stride;
  a.rows = rows, a.cols = cols, a.gate_rows = gate_per_row, a.chunks = (uint32_t)(mx_padded(cols) / 8), a.eps = eps;
  a.vec_x = vec_rows(x, x_stride, 2), a.vec_y = vec_rows(y, y_stride, 2), a.vec_o = vec_rows(x_out, x_out_stride, 2);
  a.vec_p = aligned(scale, 16) && aligned(shift, 16) && (!y || gate_per_row || aligned(gate, 16));
  return launch_norm(a, false, bits, (hipStream_t)stream);
}
