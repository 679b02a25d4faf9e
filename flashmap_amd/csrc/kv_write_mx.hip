// Appending to a context cache in microscaled 4 bits (mx_device.h): every position's keys are
// normed, rotated to the position and stored with its values,
//
//   r = 1 / sqrt(sum(k^2) / D + eps),  y = (k r) w,  (y_2i, y_2i+1) turned by the angle of pair i
//
// then blocks of 32 of y and of the values quantized, in float32 from one end to the other and
// rounded once, to the code. A cache row (block, head, position in the page) is the D key codes
// and the D value codes, D bytes, and its 2 D / 32 scale bytes apart from it.
//
// One wavefront takes 16 (token, layer, head) rows in the row-quad layout (fm_device.h): the 32
// values of a block lie 8 each in the four lanes of a row, whose codes are one dword each. A
// transposition of 4 x 4 dwords between those lanes (four lane swaps) turns the dwords of four
// blocks into 16 consecutive bytes a lane: 16 rows of 64 bytes leave in one store.
//
// 8192 tokens, 6 layers of 16 heads, D 128: 133 us, 3.8 TB/s of the 510 MB that the call cannot do without (99 us at
// a copy's 5.12 TB/s). Neither memory nor instructions fill that time: scales leave 8 bytes a row, each a request
// of 32 (538 MB in all, 105 us), some 820 instructions a wavefront take 65 us to issue, and with 130
// registers three wavefronts a SIMD, which ask for all their rows at the start, overlap the two only in part. 777
// tokens, a quarter not kept: 14 us for 46 MB (9 at a copy's rate). One token: 5.4, a launch and its chain of loads.
#include "fm_host.h"
#include "mx_device.h"

namespace fm {

constexpr int MX_KV_LAYERS = 32;  // layers of one launch: their addresses travel with it

struct KvWriteMxArgs {
  const uint16_t *kv;  // (tokens, layers, 2, heads, D)
  int64_t rows;        // tokens * count * heads
  int32_t layers, first, count, heads;
  const int64_t *positions, *slots;
  const float *k_norm;  // (layers, D)
  Rope rope;
  float eps;
  int64_t num_blocks, stride, scales_stride;  // strides of a cache row, bytes
  int32_t page;
  uint8_t *codes[MX_KV_LAYERS], *scales[MX_KV_LAYERS];
};

// RMSNorm + RoPE in fp32 from one end to the other: y = (x r) w, rotated, every step rounded as
// written and nothing to bf16: the codes are the one rounding to fewer bits.
template <int D>
__device__ __forceinline__ void norm_rope_exact(const u32x4_t (&x)[D / 32], const PrologueOps<D> &ops, float eps,
                                                float (&y)[D / 32][8]) {
  constexpr int KT = D / 32;
  // The row's sum of squares in float64 (products of bf16 are exact in float32): its rounding to
  // float32 is then the same whatever the order, and with it the codes next to a midpoint.
  double ss = 0;
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float e = bf16_lo(x[t][q]), o = bf16_hi(x[t][q]);
      ss += (double)(e * e);
      ss += (double)(o * o);
    }
  ss += __shfl_xor(ss, 16);
  ss += __shfl_xor(ss, 32);
  const float r = __fdiv_rn(1.0f, __fsqrt_rn(add_rn(__fdiv_rn((float)ss, (float)D), eps)));
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float e = mul_rn(mul_rn(bf16_lo(x[t][q]), r), ops.w[t][2 * q]);
      const float o = mul_rn(mul_rn(bf16_hi(x[t][q]), r), ops.w[t][2 * q + 1]);
      const float c = ops.c[t][q], s = ops.s[t][q];
      y[t][2 * q] = sub_rn(mul_rn(e, c), mul_rn(o, s));
      y[t][2 * q + 1] = add_rn(mul_rn(o, c), mul_rn(e, s));
    }
}

// Lane g of a row holds dword g of blocks 0 .. 3 in w[0 .. 3]; afterwards block g's dwords 0 .. 3.
__device__ __forceinline__ u32x4_t transpose_quad(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3) {
  const auto a = __builtin_amdgcn_permlane32_swap(w0, w2, false, false);
  const auto b = __builtin_amdgcn_permlane32_swap(w1, w3, false, false);
  const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  const auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  return u32x4_t{c[0], c[1], d[0], d[1]};
}

// Eight of a block's 32 values in each of a row's four lanes: this lane's codes, the scale byte.
__device__ __forceinline__ uint32_t quantize_block(const float (&v)[8], uint32_t &byte) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, magnitude(v[j]));
  auto p = __builtin_amdgcn_permlane16_swap(top, top, false, false);
  top = max(p[0], p[1]);
  p = __builtin_amdgcn_permlane32_swap(top, top, false, false);
  byte = mx_scale_byte<4>(max(p[0], p[1]));
  return mx_pack_e2m1x8(v, mx_scale_value(byte));
}

template <int D>
__global__ __launch_bounds__(256) void kv_write_mx_kernel(const KvWriteMxArgs a) {
  constexpr int KT = D / 32;
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int n = lane & 15, g = lane >> 4;
  const int64_t row = ((int64_t)blockIdx.x * 4 + wave) * 16 + n;
  bool live = row < a.rows;
  const int64_t lh = (int64_t)a.count * a.heads;
  const int64_t token = live ? row / lh : 0;
  const int gh = live ? (int)(row - token * lh) : 0;
  const int index = gh / a.heads, h = gh - index * a.heads, layer = a.first + index;
  const uint16_t *krow = a.kv + ((token * a.layers + layer) * 2ll * a.heads + h) * D + 8 * g;
  const uint16_t *vrow = krow + (int64_t)a.heads * D;
  u32x4_t kf[KT], vf[KT];
#pragma unroll
  for (int t = 0; t < KT; ++t) kf[t] = load16(krow + 32 * t), vf[t] = load16(vrow + 32 * t);
  const int64_t slot = a.slots[token];
  const int64_t rr = clamp_row(a.rope, a.positions[token]);
  PrologueOps<D> ops;
  load_prologue_ops<D>(ops, a.k_norm + (int64_t)layer * D, a.rope, rr, g);
  float ky[KT][8];
  norm_rope_exact<D>(kf, ops, a.eps, ky);
  uint32_t w[2 * KT], sc[2] = {0, 0};  // key blocks, then value blocks
#pragma unroll
  for (int t = 0; t < KT; ++t) {
    uint32_t byte;
    w[t] = quantize_block(ky[t], byte);
    sc[0] |= byte << 8 * t;
    float y[8];
#pragma unroll
    for (int q = 0; q < 4; ++q) y[2 * q] = bf16_lo(vf[t][q]), y[2 * q + 1] = bf16_hi(vf[t][q]);
    w[KT + t] = quantize_block(y, byte);
    sc[1] |= byte << 8 * t;
  }
  u32x4_t out[D / 64];
#pragma unroll
  for (int i = 0; i < D / 64; ++i) out[i] = transpose_quad(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  live = live && slot >= 0 && slot < a.num_blocks * a.page;
  if (!live) return;
  const int64_t block = slot / a.page;
  const int64_t at = (block * a.heads + h) * a.page + (slot - block * a.page);
  uint8_t *dst = a.codes[index] + at * a.stride + 16 * g;
#pragma unroll
  for (int i = 0; i < D / 64; ++i) store16(dst + 64 * i, out[i]);
  if (g != 0) return;
  uint8_t *sdst = a.scales[index] + at * a.scales_stride;
  if constexpr (D == 128) {
    *reinterpret_cast<uint32_t *>(sdst) = sc[0];
    *reinterpret_cast<uint32_t *>(sdst + 4) = sc[1];
  } else {
    *reinterpret_cast<uint32_t *>(sdst) = sc[0] | sc[1] << 16;
  }
}

}  // namespace fm

using namespace fm;

extern "C" int fm_write_context_kv_mx(const void *kv, int64_t tokens, int32_t layers, int32_t heads, int32_t head_dim,
                                      const int64_t *positions, const int64_t *slots, const float *k_norm_weight,
                                      const float *rope_cos, const float *rope_sin, int64_t rope_row_stride,
                                      int64_t rope_pair_stride, int64_t rope_rows, void *const *codes,
                                      void *const *scales, int64_t row_stride, int64_t scales_stride,
                                      int64_t num_blocks, int32_t page_size, float eps, void *stream) {
  clear_error();
  FM_REQUIRE(tokens >= 0 && layers > 0 && heads > 0, "bad sizes");
  if (tokens == 0) return FM_OK;
  if (head_dim != 64 && head_dim != 128)
    return fail(FM_ERR_UNSUPPORTED, "head_dim %d not supported (64 or 128)", head_dim);
  FM_REQUIRE(kv && positions && slots && k_norm_weight && rope_cos && rope_sin && codes && scales, "NULL pointer");
  FM_REQUIRE(((uintptr_t)kv & 15) == 0, "kv must be 16-byte aligned");
  FM_REQUIRE(num_blocks >= 0 && page_size > 0, "bad cache geometry");
  FM_REQUIRE(row_stride % 16 == 0 && row_stride >= head_dim && scales_stride % 4 == 0 && scales_stride >= head_dim / 16,
             "cache rows hold %d code bytes at a stride of a multiple of 16 and %d scale bytes at one of 4", head_dim,
             head_dim / 16);
  FM_REQUIRE(tokens <= INT64_MAX / 4 / layers / heads && (tokens * layers * heads + 63) / 64 < (1ll << 24),
             "too many rows: at most 2^30 - 64 of tokens, layers and heads");
  for (int i = 0; i < layers; ++i)
    FM_REQUIRE(codes[i] && scales[i] && ((uintptr_t)codes[i] & 15) == 0 && ((uintptr_t)scales[i] & 3) == 0,
               "the codes of layer %d must be 16-byte aligned, its scales 4-byte aligned", i);
  KvWriteMxArgs a{};
  a.kv = (const uint16_t *)kv;
  a.layers = layers;
  a.heads = heads;
  a.positions = positions;
  a.slots = slots;
  a.k_norm = k_norm_weight;
  a.rope = Rope{rope_cos, rope_sin, rope_row_stride, rope_pair_stride, rope_rows};
  a.eps = eps;
  a.num_blocks = num_blocks;
  a.stride = row_stride;
  a.scales_stride = scales_stride;
  a.page = page_size;
  for (a.first = 0; a.first < layers; a.first += MX_KV_LAYERS) {
    a.count = layers - a.first < MX_KV_LAYERS ? layers - a.first : MX_KV_LAYERS;
    a.rows = tokens * a.count * heads;
    for (int i = 0; i < a.count; ++i) a.codes[i] = (uint8_t *)codes[a.first + i], a.scales[i] = (uint8_t *)scales[a.first + i];
    const dim3 grid((unsigned)((a.rows + 63) / 64));
    if (head_dim == 128)
      kv_write_mx_kernel<128><<<grid, dim3(256), 0, (hipStream_t)stream>>>(a);
    else
      kv_write_mx_kernel<64><<<grid, dim3(256), 0, (hipStream_t)stream>>>(a);
    FM_CHECK_HIP(hipGetLastError());
  }
  return FM_OK;
}
