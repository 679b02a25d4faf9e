// out = x W^T + bias with W in microscaled 4 bits (e2m1, mx_device.h) and x in microscaled 8
// or 4 bits, on the block-scaled matrix instruction:
//
//   out[m][n] = sum over blocks b of 2^(ex[m][b] + ew[n][b]) * sum over i in b of qx[m][i] qw[n][i]
//
// v_mfma_scale_f32_16x16x128_f8f6f4 takes both code formats and both scales as they are
// stored. Its operands, lane (r = lane % 16, g = lane / 16) for row r of a 16-row block:
//   e2m1  16 bytes, the codes of k = 32 g .. 32 g + 31
//   e4m3  32 bytes, the codes of k = 16 g .. 16 g + 15 and of k = 64 + 16 g .. 64 + 16 g + 15
//   scale one byte, that of row r's block k = 32 g .. 32 g + 31, for either format
// (checked lane by lane against the formula). Its sums, probed with single products: groups of
// 8 products are aligned to the group's largest, cut below 2^-13 of its power of two (an e2m1
// product spans less and is exact), and the groups and steps added as floats. With an e4m3
// operand that costs 4e-6 to 9e-6 of a result (hidden states with outlying channels, sums of
// 128 to 65536 products) and at most 3e-5 of the absolute sum (sums made to cancel; 6e-7 in the
// mean), against 2^-9 for its rounding to bf16 and 2^-5 for the operand's own.
//
// Rows are padded with zeros to multiples of 128 values, so the loops over k have no tail.
#include <stdint.h>

#include <type_traits>

#include "fm_host.h"
#include "mx_device.h"

namespace fm {

constexpr int MX_BF16_ROWS = 16;  // bf16 rows that the kernel quantizes itself

struct MxLinearArgs {
  const uint8_t *x, *xsc, *w, *wsc;
  const uint16_t *bias;
  uint16_t *out;
  int64_t xs, xss, ws, wss, os;  // row strides (bytes; out: elements)
  int64_t rows;
  int32_t n;
  int32_t k, steps;  // steps: of 128 along k
  int32_t out_unit;  // values of out that may be written at once: 8, 4, 2 or 1
  float *part;  // NULL, or the sums of a part of k: (parts, rows, part_stride) fp32
  int64_t part_stride;
};

// D(16x16 f32) += A(16x128 e2m1) * B(128x16 e4m3 or e2m1), block scales in byte 0 of sa, sb.
template <int XBITS>
__device__ __forceinline__ f32x4_t mfma_mx(const i32x8_t &a, const i32x8_t &b, f32x4_t c, int sa, int sb) {
  if constexpr (XBITS == 8)
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 0, 0, sa, 0, sb);
  else
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 4, 0, sa, 0, sb);
}

// The same with the scales in byte OP.
template <int XBITS, int OP>
__device__ __forceinline__ f32x4_t mfma_mx_op(const i32x8_t &a, const i32x8_t &b, f32x4_t c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, XBITS == 8 ? 0 : 4, OP, sa, OP, sb);
}

__device__ __forceinline__ i32x8_t operand(u32x4_t lo) {
  return i32x8_t{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], 0, 0, 0, 0};
}
__device__ __forceinline__ i32x8_t operand(u32x4_t lo, u32x4_t hi) {
  return i32x8_t{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}

// ------------------------------------------------------------------------- loads into LDS

// One 16-byte-per-lane load straight into LDS: lane l's bytes go to lds + 16 l. Inline asm, so
// that the compiler, which cannot tell the stages apart, does not wait for the loads in
// flight before every LDS read; the waits are counted by hand (wait_vm before the barrier
// that publishes a stage).
typedef __attribute__((address_space(3))) char lds_char_t;
__device__ __forceinline__ void dma16(const uint8_t *base, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(lds), "v"(offset), "s"(base)
               : "memory", "m0");
}
__device__ __forceinline__ void dma4(const uint8_t *base, uint32_t offset, uint32_t lds) {  // 4 bytes a lane
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
               :
               : "s"(lds), "v"(offset), "s"(base)
               : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void wait_vm() {
  static_assert(N >= 0 && N < 64, "vmcnt holds 6 bits");
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

// Where a row's 16-byte pieces lie in LDS. A load's neighbouring lanes take a row's neighbouring
// pieces (whole 64- or 128-byte segments: with a row a lane every lane's 16 bytes are a request
// of their own), so a stage holds rows of 4 or 8 pieces, piece c of row r at place c ^ swizzle(r).
// ds_read_b128 serves 16 lanes at a time, and not neighbours: lanes 0-3, 12-15, 20-23, 24-27,
// then the other 16 of the lower half, then the upper half alike (measured by which lanes'
// conflicts add up). The 16 rows of an operand read are then all different, half of them one
// piece on; with these places they fall on all 64 banks.
__device__ __forceinline__ int swizzle4(int r) { return r >> 3 ? 3 : 0; }
__device__ __forceinline__ int swizzle8(int r) { return r >> 1 ^ ((r >> 2 ^ r >> 3) & 1); }

// ------------------------------------------------------------- few rows: the reduction split

// 128 values of 16 rows in bf16 (lane (r, g): k = 16 g .. 16 g + 15 in v[0], v[1] and 64 + 16 g
// .. in v[2], v[3]) as the 8-bit operand and its scale, bit for bit what fm_mx_quantize
// stores. A block of 32 is two neighbouring lane groups' halves; magnitudes are compared and
// saturated as integers, two bf16 at a time.
__device__ __forceinline__ void quantize_operand(const u32x4_t (&v)[4], int g, i32x8_t &codes, int &scale) {
  typedef __attribute__((ext_vector_type(2))) uint16_t u16x2_t;
  typedef __attribute__((ext_vector_type(2))) short s16x2_t;
  uint32_t byte[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t mag[8];
    u16x2_t top = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      mag[i] = v[2 * h + (i >> 2)][i & 3] & 0x7fff7fffu;
      top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2_t, mag[i]));
    }
    uint32_t m = top[0] > top[1] ? top[0] : top[1];
    const auto pair = __builtin_amdgcn_permlane16_swap(m, m, false, false);
    m = pair[0] > pair[1] ? pair[0] : pair[1];
    byte[h] = mx_scale_byte<8>(m << 16);
    const float f = mx_scale_value(byte[h]);
    const uint32_t lim = byte[h] == 255u ? 0x7fffu : (byte[h] + 8) << 7 | 0x60u;  // 448 scales
    const u16x2_t lim2 = {(uint16_t)lim, (uint16_t)lim};
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      s16x2_t w = {0, 0};
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const uint32_t sat = __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(u16x2_t, mag[i + q]), lim2));
        const uint32_t d = sat | (v[2 * h + ((i + q) >> 2)][(i + q) & 3] & 0x80008000u);
        w = q == 0 ? __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, __builtin_bit_cast(bf16x2_t, d), f, false)
                   : __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, __builtin_bit_cast(bf16x2_t, d), f, true);
      }
      codes[4 * h + (i >> 1)] = __builtin_bit_cast(int, w);
    }
  }
  // byte[0]: block 0 in lane groups 0, 1 and block 1 in 2, 3; byte[1]: blocks 2 and 3. Group g
  // supplies block g's.
  const auto swapped = __builtin_amdgcn_permlane32_swap(byte[0], byte[1], false, false);
  scale = (int)(g & 1 ? swapped[1] : swapped[0]);
}

// A workgroup owns 16 NB rows of W against up to 16 rows of x; its wavefronts split k and meet in
// LDS in a fixed order. XBITS 16: x in bf16, quantized in registers. Bound: latency (a launch, the
// loads of a wavefront's share of k, all in flight at once, and the join): 1 x 2048 -> 2048 3.8 us,
// 16 x 2048 -> 8192 6.5 us, 9.3 MB.
template <int XBITS, int NB, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void mx_linear_rows_kernel(const MxLinearArgs a) {
  __shared__ f32x4_t part[WAVES][NB][64];
  constexpr int XL = XBITS == 16 ? 4 : XBITS == 8 ? 2 : 1;  // 16-byte loads of x a step
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int r = lane & 15, g = lane >> 4;
  const int32_t n0 = (int32_t)blockIdx.x * 16 * NB;
  const int32_t s0 = (int32_t)((int64_t)a.steps * wave / WAVES), s1 = (int32_t)((int64_t)a.steps * (wave + 1) / WAVES);
  // Rows past the end read the last one: their results are not stored.
  const uint8_t *w[NB], *wsc[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int64_t n = n0 + 16 * j + r < a.n ? n0 + 16 * j + r : a.n - 1;
    w[j] = a.w + n * a.ws + 16 * g, wsc[j] = a.wsc + n * a.wss + g;
  }
  const int64_t row = r < a.rows ? r : a.rows - 1;
  const uint8_t *const x = a.x + row * a.xs + (XBITS == 16 ? 32 : 16) * g;
  const uint8_t *const xsc = XBITS == 16 ? nullptr : a.xsc + row * a.xss + g;
  f32x4_t acc[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) acc[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  auto take = [&](auto group, int32_t s) {  // steps s .. s + G - 1, all their loads in flight at once
    constexpr int G = decltype(group)::value;
    u32x4_t wf[G][NB], xf[G][XL];
    int sw[G][NB], sx[G];
#pragma unroll
    for (int t = 0; t < G; ++t) {
      const int64_t at = s + t;
#pragma unroll
      for (int j = 0; j < NB; ++j) wf[t][j] = load16(w[j] + 64 * at), sw[t][j] = wsc[j][4 * at];
    }
#pragma unroll
    for (int t = 0; t < G; ++t) {
      const int64_t at = s + t;
      if constexpr (XBITS == 16) {
        // k is a multiple of 8: a 16-byte load past the row's end is zeros
        const int32_t k0 = 128 * (int32_t)at + 16 * g;
#pragma unroll
        for (int l = 0; l < 4; ++l) {
          const int o = 64 * (l >> 1) + 8 * (l & 1);
          xf[t][l] = k0 + o < a.k ? load16(x + 256 * at + 2 * o) : u32x4_t{0, 0, 0, 0};
        }
      } else {
#pragma unroll
        for (int l = 0; l < XL; ++l) xf[t][l] = load16(x + 64 * XL * at + 64 * l);
        sx[t] = xsc[4 * at];
      }
    }
#pragma unroll
    for (int t = 0; t < G; ++t) {
      i32x8_t xo;
      if constexpr (XBITS == 16)
        quantize_operand(xf[t], g, xo, sx[t]);
      else if constexpr (XBITS == 8)
        xo = operand(xf[t][0], xf[t][1]);
      else
        xo = operand(xf[t][0]);
#pragma unroll
      for (int j = 0; j < NB; ++j)
        acc[j] = mfma_mx<XBITS == 4 ? 4 : 8>(operand(wf[t][j]), xo, acc[j], sw[t][j], sx[t]);
    }
  };
  int32_t s = s0;
  for (; s + 4 <= s1; s += 4) take(std::integral_constant<int, 4>{}, s);
  if (s1 - s & 2) take(std::integral_constant<int, 2>{}, s), s += 2;
  if (s1 - s & 1) take(std::integral_constant<int, 1>{}, s);
#pragma unroll
  for (int j = 0; j < NB; ++j) part[wave][j][lane] = acc[j];
  __syncthreads();
  for (int b = wave; b < NB; b += WAVES) {
    f32x4_t sum = part[0][b][lane];
#pragma unroll
    for (int q = 1; q < WAVES; ++q) sum += part[q][b][lane];
    // Lane: row r of out, columns n .. n + 3.
    const int32_t n = n0 + 16 * b + 4 * g;
    if (r >= a.rows) continue;
    uint16_t *dst = a.out + r * a.os + n;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (a.bias != nullptr && n + i < a.n) sum[i] += bf16_to_f32(a.bias[n + i]);
    if (a.out_unit >= 4 && n + 4 <= a.n) {
      *reinterpret_cast<u32x2_t *>(dst) = u32x2_t{pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3])};
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < a.n) dst[i] = (uint16_t)(pack_bf16x2(sum[i], 0.f) & 0xffffu);
    }
  }
}

template <int XBITS, int NB, int WAVES>
static int launch_rows(const MxLinearArgs &a, hipStream_t stream) {
  const unsigned tiles = (unsigned)((a.n + 16 * NB - 1) / (16 * NB));
  mx_linear_rows_kernel<XBITS, NB, WAVES><<<dim3(tiles), dim3(64 * WAVES), 0, stream>>>(a);
  FM_CHECK_HIP(hipGetLastError());
  return FM_OK;
}

// ----------------------------------------------------------- few rows, many columns: streams

// Weights larger than what is in flight at once (a head over the vocabulary): a wavefront
// streams whole 16-row blocks of W through a ring of its own in LDS, D groups of four steps
// deep, and needs nobody: x, up to 16 rows of it, lies in LDS for the workgroup's whole
// life, quantized once. A group: 16 rows of 256 bytes, as four loads of eight 128-byte
// segments, and their scales, 16 bytes a row. Bound: HBM; 16 x 2048 -> 151936, 170 MB, 37 to 38 us,
// 4.4 to 4.6 TB/s (with a workgroup per 16 columns and k split, 61.5 us).
template <int XBITS, int WAVES, int D>
struct Stream {
  static constexpr int GROUP = 4096 + 256, RING = D * GROUP;
  static constexpr int XSTEP = 16 * (XBITS == 4 ? 64 : 128);  // bytes of a step of x
  static size_t lds(int32_t steps) { return WAVES * RING + (size_t)steps * XSTEP + (size_t)((steps + 3) / 4) * 256; }
};

template <int XBITS, int WAVES, int D>
__global__ __launch_bounds__(64 * WAVES) void mx_linear_stream_kernel(const MxLinearArgs a) {
  using T = Stream<XBITS, WAVES, D>;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int r = lane & 15, g = lane >> 4;
  const int at4 = 64 * r + 16 * (g ^ swizzle4(r));
  const int at8 = 128 * r + 16 * (g ^ swizzle8(r)), at8h = at8 ^ 64;
  char *const xl = lds + WAVES * T::RING, *const xsl = xl + a.steps * T::XSTEP;
  const int64_t row = r < a.rows ? r : a.rows - 1;
  for (int32_t s = wave; s < a.steps; s += WAVES) {
    i32x8_t codes;
    int scale;
    if constexpr (XBITS == 16) {
      u32x4_t v[4];
#pragma unroll
      for (int l = 0; l < 4; ++l) {
        const int32_t k = 128 * s + 16 * g + 64 * (l >> 1) + 8 * (l & 1);  // zeros past the row's end
        v[l] = k < a.k ? load16(a.x + row * a.xs + 2 * (int64_t)k) : u32x4_t{0, 0, 0, 0};
      }
      quantize_operand(v, g, codes, scale);
    } else {
      const uint8_t *x = a.x + row * a.xs + (XBITS == 8 ? 128 : 64) * (int64_t)s + 16 * g;
      codes = XBITS == 8 ? operand(load16(x), load16(x + 64)) : operand(load16(x));
      scale = a.xsc[row * a.xss + 4 * (int64_t)s + g];
    }
    char *const to = xl + s * T::XSTEP;
    store16(to + (XBITS == 4 ? at4 : at8), u32x4_t{(uint32_t)codes[0], (uint32_t)codes[1], (uint32_t)codes[2], (uint32_t)codes[3]});
    if constexpr (XBITS != 4)
      store16(to + at8h, u32x4_t{(uint32_t)codes[4], (uint32_t)codes[5], (uint32_t)codes[6], (uint32_t)codes[7]});
    xsl[(s >> 2) * 256 + 16 * r + 4 * g + (s & 3)] = (char)scale;
  }
  __syncthreads();

  const int32_t groups = (a.steps + 3) >> 2, blocks = (a.n + 15) >> 4;
  const int64_t waves = (int64_t)gridDim.x * WAVES, id = (int64_t)blockIdx.x * WAVES + wave;
  const int32_t b0 = (int32_t)(blocks * id / waves), b1 = (int32_t)(blocks * (id + 1) / waves);
  if (b0 == b1) return;
  const uint32_t ring = (uint32_t)(uintptr_t)(lds_char_t *)lds + wave * T::RING;
  const int64_t total = (int64_t)(b1 - b0) * groups;
  // The next group to load: block lb, group lg. Pieces past the row's end repeat its last ones.
  int32_t lb = b0, lg = 0, lslot = 0;
  const int32_t wlast = 64 * a.steps - 16, slast = 4 * a.steps - 4;
  auto issue = [&]() {
    const uint32_t to = ring + lslot * T::GROUP;
    const uint8_t *w = a.w + (int64_t)(16 * lb) * a.ws, *sc = a.wsc + (int64_t)(16 * lb) * a.wss;
    const int32_t last = a.n - 1 - 16 * lb;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int row = 8 * (u & 1) + (lane >> 3), piece = (lane & 7) ^ swizzle8(row);
      const int32_t at = 256 * lg + 128 * (u >> 1) + 16 * piece;
      dma16(w, (uint32_t)((row < last ? row : last) * (int32_t)a.ws + (at < wlast ? at : wlast)), to + 1024 * u);
    }
    const int row = lane >> 2;
    const int32_t at = 16 * lg + 4 * (lane & 3);
    dma4(sc, (uint32_t)((row < last ? row : last) * (int32_t)a.wss + (at < slast ? at : slast)), to + 4096);
    if (++lg == groups) lg = 0, ++lb;
    lslot = lslot == D - 1 ? 0 : lslot + 1;
  };
#pragma unroll
  for (int d = 0; d < D; ++d)
    if (d < total) issue();
  const uint32_t pick = 0x0400u + 0x0101u * (uint32_t)g;
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
  int32_t block = b0, grp = 0, slot = 0;
  for (int64_t t = 0; t < total; ++t) {
    // In flight behind this group: up to D - 1 groups, 5 loads each (and results being stored,
    // which only make the wait longer).
    if (t + D <= total)
      wait_vm<5 * (D - 1)>();
    else
      wait_vm<0>();
    const char *wl = lds + wave * T::RING + slot * T::GROUP;
    const u32x4_t d = *(const u32x4_t *)(wl + 4096 + 16 * r);
    const uint32_t a01 = __builtin_amdgcn_perm(d[1], d[0], pick), a23 = __builtin_amdgcn_perm(d[3], d[2], pick);
    const int sw = (int)__builtin_amdgcn_perm(a23, a01, 0x05040100);
    const int sx = *(const int *)(xsl + grp * 256 + 16 * r + 4 * g);
    auto step = [&](auto jc) {
      constexpr int J = decltype(jc)::value;
      const int32_t s = 4 * grp + J;
      if (s >= a.steps) return;
      const i32x8_t wf = operand(load16(wl + 2048 * (J >> 1) + (J & 1 ? at8h : at8)));
      const char *x = xl + s * T::XSTEP;
      i32x8_t xf;
      if constexpr (XBITS == 4)
        xf = operand(load16(x + at4));
      else
        xf = operand(load16(x + at8), load16(x + at8h));
      acc = mfma_mx_op<XBITS == 4 ? 4 : 8, J>(wf, xf, acc, sw, sx);
    };
    step(std::integral_constant<int, 0>{});
    step(std::integral_constant<int, 1>{});
    step(std::integral_constant<int, 2>{});
    step(std::integral_constant<int, 3>{});
    // The slot has been read (its values are operands by now): the group D on takes it.
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (t + D < total) issue();
    slot = slot == D - 1 ? 0 : slot + 1;
    if (++grp == groups) {
      // Lane: row r of out, columns n .. n + 3.
      const int32_t n = 16 * block + 4 * g;
      if (r < a.rows) {
        uint16_t *dst = a.out + r * a.os + n;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (a.bias != nullptr && n + q < a.n) acc[q] += bf16_to_f32(a.bias[n + q]);
        if (a.out_unit >= 4 && n + 4 <= a.n) {
          *reinterpret_cast<u32x2_t *>(dst) = u32x2_t{pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3])};
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (n + q < a.n) dst[q] = (uint16_t)(pack_bf16x2(acc[q], 0.f) & 0xffffu);
        }
      }
      acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
      grp = 0, ++block;
    }
  }
}

template <int XBITS, int WAVES, int D>
static int launch_stream(const MxLinearArgs &a, hipStream_t stream) {
  DeviceInfo info;
  const int rc = device_info(&info);
  if (rc != FM_OK) return rc;
  mx_linear_stream_kernel<XBITS, WAVES, D>
      <<<dim3((unsigned)info.cus), dim3(64 * WAVES), Stream<XBITS, WAVES, D>::lds(a.steps), stream>>>(a);
  FM_CHECK_HIP(hipGetLastError());
  return FM_OK;
}

// ------------------------------------------------------------------------ many rows: tiles
//
// Steps of 128 along k, three stages in LDS. A wavefront reads its rows and columns of a stage and
// multiplies all of one by all of the other, so larger shares need fewer bytes of LDS a product;
// at 256 x 256 LDS and the matrix instruction are busy alike. Bound, large products: the
// instruction, whose clock falls under it (random codes, nothing but the instruction on every
// SIMD: 17.5 ns with 8-bit x, 10.1 ns with 4-bit x, 3.8 and 6.6 PFLOP/s). Reached at 4096 x 20480
// -> 4096: 252 and 188 us, 2.7 and 3.65 PFLOP/s; storing results takes 25 us per 100 MB (with k =
// 128), partly beside other tiles' products (1024 x 2048 -> 151936 of 8-bit x 284 us, 8192 x 2048
// -> 24576 of 8-bit x 326 us, of 4-bit x 254 us). Small products (1024 x 8192 -> 2048: 25 to 28 us) are bound by a step's way
// through a workgroup, 0.41 us for 8 instructions a wavefront, however many workgroups run.
// Measured and not taken: a persistent grid that starts the next tile's loads before this one's
// stores (1 % either way; the stores count among the loads awaited), four and more stages (+6 %
// at 256 x 256, none below), 4-bit rows read two steps at a time in whole cache lines (4-bit x
// -4 %, 8-bit x +5 %), the next step's operands read among this one's products (none).

template <int XBITS, int BM, int BN, int WM, int WN>
struct Tile {
  static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
  static constexpr int XU = BM / 16 * (XBITS == 8 ? 2 : 1), WU = BN / 16;  // 1 KiB units of a stage
  static constexpr int XPW = XU / WAVES, WPW = WU / WAVES, PER = XPW + WPW;  // units a wavefront loads
  static constexpr int STAGE = 1024 * (XU + WU), STAGES = 3;
  static constexpr int SCALES = 16 * (BM + BN);  // one chunk of four steps
  static constexpr int LDS = STAGES * STAGE + SCALES > 2 * BM * BN ? STAGES * STAGE + SCALES : 2 * BM * BN;
  static constexpr int MF = BM / WM / 16, NF = BN / WN / 16;  // 16-row blocks of a wavefront
  static_assert(XU % WAVES == 0 && WU % WAVES == 0 && (BM + BN) % 64 == 0, "whole units a wavefront");
  static constexpr int SW = (BM + BN) / 64;  // wavefronts that load scales (one row a lane)
  static_assert(SW <= WAVES, "a row a lane");
};

// The row of W (in its 32-row group pair) that block f holds at index r: lane group g of the
// accumulators then holds 8 consecutive columns of out in blocks 2 p and 2 p + 1, 16 bytes.
__device__ __forceinline__ int w_row(int f, int r) { return 32 * (f >> 1) + 8 * (r >> 2) + 4 * (f & 1) + (r & 3); }

template <int XBITS, int BM, int BN, int WM, int WN, bool TURNS>
__global__ __launch_bounds__(64 * WM * WN, 2) void mx_linear_tile_kernel(const MxLinearArgs a, const int32_t tiles_m,
                                                                         const int32_t tiles_n) {
  using T = Tile<XBITS, BM, BN, WM, WN>;
  __shared__ __attribute__((aligned(1024))) char lds[T::LDS];
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int r = lane & 15, g = lane >> 4;
  const int wm = wave % WM, wn = wave / WM;
  // Consecutive workgroups go to the eight XCDs in turn: each XCD takes a consecutive part of
  // the tiles, in groups of up to 8 row tiles, rows first, so that what runs at once on an
  // XCD shares its reads of x and W in that XCD's L2.
  const uint32_t total = (uint32_t)tiles_m * (uint32_t)tiles_n;
  const uint32_t id = blockIdx.x, xcd = id & 7, base = total >> 3, rest = total & 7;
  const uint32_t at = xcd * base + (xcd < rest ? xcd : rest) + (id >> 3);
  const uint32_t group = at / (8u * (uint32_t)tiles_n), gm = group * 8;
  const uint32_t in = at - group * 8u * (uint32_t)tiles_n;
  const uint32_t high = (uint32_t)tiles_m - gm < 8u ? (uint32_t)tiles_m - gm : 8u;
  const int64_t m0 = (int64_t)(gm + in % high) * BM;
  const int32_t n0 = (int32_t)(in / high) * BN;

  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_char_t *)lds;
  const uint32_t sc0 = lds0 + T::STAGES * T::STAGE;
  // This workgroup's part of k, in whole chunks of four steps.
  const int32_t chunks_all = (a.steps + 3) >> 2;
  const int32_t first = 4 * (int32_t)((int64_t)chunks_all * blockIdx.y / gridDim.y);
  const int32_t end = 4 * (int32_t)((int64_t)chunks_all * (blockIdx.y + 1) / gridDim.y);
  const int32_t steps = (end < a.steps ? end : a.steps) - first;
  // Offsets from the tile's first row stay below 2^32 (strides are below 2^24, rows at most 256).
  const uint8_t *xbase = a.x + m0 * a.xs + (XBITS == 8 ? 128 : 64) * (int64_t)first;
  const uint8_t *wbase = a.w + (int64_t)n0 * a.ws + 64 * (int64_t)first;
  const int32_t mlast = (int32_t)(a.rows - 1 - m0 < BM ? a.rows - 1 - m0 : BM - 1);
  const int32_t nlast = a.n - 1 - n0 < BN ? a.n - 1 - n0 : BN - 1;
  uint32_t src[T::PER];
#pragma unroll
  for (int u = 0; u < T::XPW; ++u) {
    const int unit = wave * T::XPW + u;
    const int row = XBITS == 8 ? 8 * unit + (lane >> 3) : 16 * unit + (lane >> 2);
    const int piece = XBITS == 8 ? (lane & 7) ^ swizzle8(row & 15) : (lane & 3) ^ swizzle4(row & 15);
    src[u] = (uint32_t)(row < mlast ? row : mlast) * (uint32_t)a.xs + 16 * piece;
  }
#pragma unroll
  for (int u = 0; u < T::WPW; ++u) {
    const int row = w_row(wave * T::WPW + u, lane >> 2);
    src[T::XPW + u] = (uint32_t)(row < nlast ? row : nlast) * (uint32_t)a.ws + 16 * ((lane & 3) ^ swizzle4(lane >> 2));
  }
  // Where this lane's operands lie in a 16-row block.
  const int at4 = 64 * r + 16 * (g ^ swizzle4(r));
  const int at8 = 128 * r + 16 * (g ^ swizzle8(r)), at8h = at8 ^ 64;
  // Four steps' scales of a row at once, x's rows, then W's, 64 rows a wavefront. The last
  // chunk's 16 bytes end with the row: they hold `back` steps of the chunk before it first.
  const int32_t back = -steps & 3;
  static_assert(BM % 64 == 0, "a wavefront's rows are all x's or all W's");
  const bool of_x = 64 * wave < BM;
  const uint8_t *sbase = (of_x ? a.xsc + m0 * a.xss : a.wsc + (int64_t)n0 * a.wss) + 4 * (int64_t)first;
  uint32_t ssrc;
  {
    const int row = 64 * wave + lane - (of_x ? 0 : BM);
    ssrc = of_x ? (uint32_t)(row < mlast ? row : mlast) * (uint32_t)a.xss : (uint32_t)(row < nlast ? row : nlast) * (uint32_t)a.wss;
  }
  auto issue = [&](int stage) {  // the next step, into `stage`
    const uint32_t dst = lds0 + stage * T::STAGE;
#pragma unroll
    for (int u = 0; u < T::XPW; ++u) dma16(xbase, src[u], dst + 1024 * (wave * T::XPW + u));
#pragma unroll
    for (int u = 0; u < T::WPW; ++u) dma16(wbase, src[T::XPW + u], dst + 1024 * (T::XU + wave * T::WPW + u));
    xbase += XBITS == 8 ? 128 : 64;
    wbase += 64;
  };
  auto issue_scales = [&](int32_t chunk) {
    if (wave < T::SW) dma16(sbase + 16 * (int64_t)chunk - (4 * chunk + 4 > steps ? 4 * back : 0), ssrc, sc0 + 1024 * wave);
  };
  // A row's 16 scale bytes, (step, block) as stored: lane group g keeps block g's, whose byte
  // `step` the instruction selects; `shift` drops the bytes of the chunk before.
  const uint32_t pick = 0x0400u + 0x0101u * (uint32_t)g;
  auto scales_of = [&](int row, uint32_t shift) {
    const u32x4_t d = *(const u32x4_t *)(lds + T::STAGES * T::STAGE + 16 * row);
    const uint32_t a01 = __builtin_amdgcn_perm(d[1], d[0], pick), a23 = __builtin_amdgcn_perm(d[3], d[2], pick);
    return (int)(__builtin_amdgcn_perm(a23, a01, 0x05040100) >> shift);
  };

  f32x4_t acc[T::NF][T::MF];
#pragma unroll
  for (int j = 0; j < T::NF; ++j)
#pragma unroll
    for (int i = 0; i < T::MF; ++i) acc[j][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  if (steps >= 4) {
    issue_scales(0);
  } else if (wave < T::SW) {  // rows shorter than 16 bytes: dword by dword
    u32x4_t d = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (i < steps) d[i] = *(const uint32_t *)(sbase + ssrc + 4 * i);
    *(u32x4_t *)(lds + T::STAGES * T::STAGE + 1024 * wave + 16 * lane) = d;
  }
  issue(0);
  if (steps > 1) issue(1);
  int sx[T::MF], sw[T::NF];
  int stage = 0;  // of step s
  // This wavefront's loads of step s have landed; step s + 1's, and scales issued since, may be
  // in flight.
  auto landed = [&](int32_t s, bool scales) {
    if (s + 1 >= steps)
      wait_vm<0>();
    else if (scales && T::SW == T::WAVES)
      wait_vm<T::PER + 1>();
    else
      wait_vm<T::PER>();
  };
  auto barrier = [&]() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  // TURNS: the wavefronts of a SIMD take turns. While one half of the workgroup multiplies, the
  // other reads its operands from LDS into registers and starts the loads of two steps on.
  // Phase 2 s is the first half's reads of step s, phase 2 s + 1 its products and the second
  // half's reads; a barrier ends each phase. The loads of a step are in flight for three
  // phases, awaited before the barrier that ends the phase before the first half's reads. A
  // step's stage is free once the second half has read it, before either half loads the stage
  // three steps on. Else every wavefront reads and multiplies between the step's barriers.
  const bool late = TURNS && wave >= T::WAVES / 2;
  if (TURNS) {
    landed(0, false);
    barrier();
    if (late) barrier();
  }
  auto step = [&](auto jc, int32_t chunk) {
    constexpr int J = decltype(jc)::value;
    const int32_t s = 4 * chunk + J;
    if (s >= steps) return;
    const bool more = 4 * chunk + 4 < steps;
    if (!TURNS) {
      landed(s, J >= 2 && more);
      barrier();
      if (s + 2 < steps) issue(stage == 0 ? 2 : stage - 1);
      if (J == 1 && more) issue_scales(chunk + 1);
    }
    const char *xs = lds + stage * T::STAGE + 1024 * (XBITS == 8 ? 2 : 1) * wm * T::MF;
    const char *ws = lds + stage * T::STAGE + 1024 * (T::XU + wn * T::NF) + at4;
    if constexpr (J == 0) {
      const uint32_t shift = more || steps < 4 ? 0 : 8 * back;
#pragma unroll
      for (int i = 0; i < T::MF; ++i) {
        sx[i] = scales_of(16 * (wm * T::MF + i) + r, shift);
        if ((i & 3) == 3) __builtin_amdgcn_sched_barrier(0);  // few of their 16 bytes a row at a time
      }
#pragma unroll
      for (int j = 0; j < T::NF; ++j) {
        sw[j] = scales_of(BM + w_row(wn * T::NF + j, r), shift);
        if ((j & 3) == 3) __builtin_amdgcn_sched_barrier(0);
      }
    }
    i32x8_t xf[T::MF], wf[T::NF];
#pragma unroll
    for (int i = 0; i < T::MF; ++i) {
      if constexpr (XBITS == 8)
        xf[i] = operand(load16(xs + 2048 * i + at8), load16(xs + 2048 * i + at8h));
      else
        xf[i] = operand(load16(xs + 1024 * i + at4));
    }
#pragma unroll
    for (int j = 0; j < T::NF; ++j) wf[j] = operand(load16(ws + 1024 * j));
    if (TURNS) {
      if (s + 2 < steps) issue(stage == 0 ? 2 : stage - 1);
      if (J == 1 && more) issue_scales(chunk + 1);
      if (late && s + 1 < steps) landed(s + 1, (J == 1 || J == 2) && more);
      barrier();
      __builtin_amdgcn_s_setprio(1);
    }
#pragma unroll
    for (int j = 0; j < T::NF; ++j)
#pragma unroll
      for (int i = 0; i < T::MF; ++i) acc[j][i] = mfma_mx_op<XBITS, J>(wf[j], xf[i], acc[j][i], sw[j], sx[i]);
    if (TURNS) {
      __builtin_amdgcn_s_setprio(0);
      if (!late && s + 1 < steps) landed(s + 1, (J == 1 || J == 2) && more);
      barrier();
    }
    stage = stage == 2 ? 0 : stage + 1;
  };
  for (int32_t chunk = 0; 4 * chunk < steps; ++chunk) {
    step(std::integral_constant<int, 0>{}, chunk);
    step(std::integral_constant<int, 1>{}, chunk);
    step(std::integral_constant<int, 2>{}, chunk);
    step(std::integral_constant<int, 3>{}, chunk);
  }
  if (TURNS ? !late : a.part == nullptr) barrier();  // nobody reads the stages any more

  // Lane (r, g) holds row m of out, 8 columns from 8 g on in each 32-column group. (Found anew,
  // not kept in registers through the loop.)
  int out_lane = threadIdx.x & 63;
  asm volatile("" : "+v"(out_lane));
  const int out_r = out_lane & 15, out_g = out_lane >> 4;
  if (a.part != nullptr) {  // rows padded to whole groups of 8 columns
#pragma unroll
    for (int p = 0; p < T::NF / 2; ++p) {
      const int32_t n = n0 + 32 * (wn * (T::NF / 2) + p) + 8 * out_g;
#pragma unroll
      for (int i = 0; i < T::MF; ++i) {
        const int64_t m = m0 + 16 * (wm * T::MF + i) + out_r;
        if (m >= a.rows || n >= a.n) continue;
        float *to = a.part + (blockIdx.y * a.rows + m) * a.part_stride + n;
        *reinterpret_cast<f32x4_t *>(to) = acc[2 * p][i];
        *reinterpret_cast<f32x4_t *>(to + 4) = acc[2 * p + 1][i];
      }
    }
    return;
  }
  // The results go through LDS, so that a wavefront stores whole rows of the tile; a row's
  // 16-byte pieces lie at place piece ^ (row % 8). Stored from the lanes as they are, 64 bytes a
  // row at a time, 8192 x 24576 results of k = 128 take 157 us instead of 104 (fill: 63).
  constexpr int PIECES = BN / 8, ROWS = 64 / PIECES;
#pragma unroll
  for (int p = 0; p < T::NF / 2; ++p) {
    const int piece = 4 * (wn * (T::NF / 2) + p) + out_g;
    const int32_t n = n0 + 8 * piece;
    float b[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (a.bias != nullptr) {
#pragma unroll
      for (int q = 0; q < 8; ++q) b[q] = bf16_to_f32(a.bias[n + q < a.n ? n + q : a.n - 1]);
    }
#pragma unroll
    for (int i = 0; i < T::MF; ++i) {
      const f32x4_t lo = acc[2 * p][i], hi = acc[2 * p + 1][i];
      const int row = 16 * (wm * T::MF + i) + out_r;
      store16(lds + 2 * BN * row + 16 * (piece ^ (out_r & 7)),
              u32x4_t{pack_bf16x2(lo[0] + b[0], lo[1] + b[1]), pack_bf16x2(lo[2] + b[2], lo[3] + b[3]),
                      pack_bf16x2(hi[0] + b[4], hi[1] + b[5]), pack_bf16x2(hi[2] + b[6], hi[3] + b[7])});
    }
  }
  barrier();
  if (a.out_unit == 8) {
    const int piece = out_lane % PIECES;
    const int32_t n = n0 + 8 * piece;
#pragma unroll
    for (int q = 0; q < BM / T::WAVES / ROWS; ++q) {
      const int row = (q * T::WAVES + wave) * ROWS + out_lane / PIECES;
      if (m0 + row >= a.rows) continue;
      const u32x4_t v = load16(lds + 2 * BN * row + 16 * (piece ^ (row & 7)));
      uint16_t *dst = a.out + (m0 + row) * a.os + n;
      if (n + 8 <= a.n) {
        // Tiles this large are chosen for results that no cache holds.
        if (BM == 256)
          store16_nt(dst, v);
        else
          store16(dst, v);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (n + e < a.n) dst[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
      }
    }
    return;
  }
  // Rows that are not 16-byte aligned: as many values a lane as they allow, neighbouring lanes'
  // side by side.
  auto loose = [&](auto type) {
    typedef decltype(type) U;
    constexpr int W = sizeof(U) / 2;
    for (int q = wave; q < BM * BN / (64 * W); q += T::WAVES) {
      const int at = W * (64 * q + out_lane), row = at / BN, c = at % BN;
      const int32_t n = n0 + c;
      if (m0 + row >= a.rows || n >= a.n) continue;
      const U v = *reinterpret_cast<const U *>(lds + 2 * BN * row + 16 * ((c >> 3) ^ (row & 7)) + 2 * (c & 7));
      uint16_t *dst = a.out + (m0 + row) * a.os + n;
      if (n + W <= a.n) {
        *reinterpret_cast<U *>(dst) = v;
      } else {
        for (int e = 0; n + e < a.n; ++e) dst[e] = (uint16_t)(v >> (16 * e));
      }
    }
  };
  if (a.out_unit == 4)
    loose((uint64_t)0);
  else if (a.out_unit == 2)
    loose((uint32_t)0);
  else
    loose((uint16_t)0);
}

// The parts' sums, in their order, plus the bias: 8 columns a thread.
__global__ __launch_bounds__(256) void mx_linear_join_kernel(const MxLinearArgs a, const int32_t parts, const uint32_t groups) {
  const uint32_t item = blockIdx.x * 256 + threadIdx.x, m = item / groups;
  if (m >= a.rows) return;
  const int32_t n = 8 * (int32_t)(item - m * groups);
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const float *p = a.part + m * a.part_stride + n;
  for (int32_t z = 0; z < parts; ++z, p += a.rows * a.part_stride) {
    const f32x4_t lo = *reinterpret_cast<const f32x4_t *>(p), hi = *reinterpret_cast<const f32x4_t *>(p + 4);
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] += lo[q], v[4 + q] += hi[q];
  }
#pragma unroll
  for (int q = 0; q < 8; ++q)
    if (a.bias != nullptr && n + q < a.n) v[q] += bf16_to_f32(a.bias[n + q]);
  uint16_t *dst = a.out + m * a.os + n;
  if (a.out_unit == 8 && n + 8 <= a.n) {
    store16(dst, u32x4_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])});
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (n + q < a.n) dst[q] = (uint16_t)(pack_bf16x2(v[q], 0.f) & 0xffffu);
  }
}

// `parts` > 1: a.part holds parts * rows * part_stride floats (rows at most 2^22 / tiles of n).
template <int XBITS, int BM, int BN, int WM, int WN, bool TURNS>
static int launch_tiles(const MxLinearArgs &a, int32_t parts, hipStream_t stream) {
  const int64_t tm = (a.rows + BM - 1) / BM, tn = ((int64_t)a.n + BN - 1) / BN;
  // At most 2^22 workgroups a launch: slices of whole groups of row tiles.
  const int64_t most = (1 << 22) / tn < 8 ? 8 : (1 << 22) / tn / 8 * 8;
  for (int64_t first = 0; first < tm; first += most) {
    MxLinearArgs slice = a;
    const int64_t rows = a.rows - first * BM, here = tm - first < most ? tm - first : most;
    slice.x += first * BM * a.xs, slice.xsc += first * BM * a.xss, slice.out += first * BM * a.os;
    slice.rows = rows < here * BM ? rows : here * BM;
    if (parts == 1) slice.part = nullptr;
    mx_linear_tile_kernel<XBITS, BM, BN, WM, WN, TURNS>
        <<<dim3((unsigned)(here * tn), (unsigned)parts), dim3(64 * WM * WN), 0, stream>>>(slice, (int32_t)here, (int32_t)tn);
    FM_CHECK_HIP(hipGetLastError());
  }
  if (parts > 1) {
    const uint32_t groups = (uint32_t)(a.part_stride / 8);
    mx_linear_join_kernel<<<dim3((unsigned)((a.rows * groups + 255) / 256)), dim3(256), 0, stream>>>(a, parts, groups);
    FM_CHECK_HIP(hipGetLastError());
  }
  return FM_OK;
}

static bool aligned(const void *p, int64_t n) { return ((uintptr_t)p % (uintptr_t)n) == 0; }

// Which kernel a product runs on, by its sizes (MI355X: 256 CUs).
struct MxPlan {
  enum Kind { ROWS, STREAM, TILES } kind;
  int bm, bn;     // tiles
  int32_t parts;  // of k
};

constexpr size_t LDS_BYTES = 160 * 1024;
constexpr int64_t CUS = 256;
constexpr int STREAM_WAVES = 8, STREAM_GROUPS = 2;

template <int XBITS>
static bool streams(int32_t steps) {
  return Stream<XBITS, STREAM_WAVES, STREAM_GROUPS>::lds(steps) <= LDS_BYTES;
}

// Measured, us, weights from HBM (copies past the caches in turn, in a graph), x in 8 bits (bf16 x:
// the same order):
//   16 rows, k 2048:  n 4096  rows 4.9, stream 6.4, tiles 8.1;  n 8192  6.4, 7.1, 8.8
//                     n 12288 9.4, 7.4, 8.9;  n 151936 61.5, 36.8, 37.7
//   16 rows, n 2048:  k 4096  rows 7.0, stream 9.5, tiles 10.6;  k 8192 11.5, -, 12.1;  k 20480 26.9, -, 15.1
//   more rows, tiles of 64 x 64, 64 x 128, 128 x 128 and 256 x 256:
//     64 x 2048 -> 2048 6.9, 8.5, 11.7, 22;  64 x 2048 -> 24576 11.8, 10.8, 13.0, 23;  1024 x 8192 -> 2048 29.6, 27.9, 38.6, 73
//     1024 x 2048 -> 8192 27.9, 24.4, 21.6, 25.1;  512 x 8192 -> 8192 56, 46.8, 40.1, 74;  4096 x 2048 -> 4096 51, 43, 38.3, 30.6
//     300 x 2048 -> 151936 (a last row tile of 44) 150, 123, 124, 137
//   k in parts of at least 2048 values, tiles of 64 x 64: 64 x 8192 -> 2048 1 part 25.0, 2 17.7, 4 12.7, 8 12.1;
//     64 x 20480 -> 2048 4 parts 21.2, 8 15.7, 16 18.5;  64 x 2048 -> 2048 1 part 6.9, 4 7.9
static MxPlan plan_of(int64_t rows, int64_t n, int64_t k, int32_t x_bits) {
  const int32_t steps = (int32_t)(mx_padded(k) / MX_PAD);
  if (rows <= 16) {
    const bool fits = x_bits == 4 ? streams<4>(steps) : streams<8>(steps);
    if (n > 8192 && fits) return {MxPlan::STREAM, 0, 0, 1};
    if (x_bits == 16 || (k < 8192 && n <= 8192)) return {MxPlan::ROWS, 0, 0, 1};
  }
  // A tile size is worth taking if it fills the chip and its last row tile is not mostly air.
  auto fills = [&](int64_t bm, int64_t bn, int64_t least, double full) {
    const int64_t tiles = ((rows + bm - 1) / bm) * ((n + bn - 1) / bn);
    return tiles >= least && (double)(rows * n) >= full * (double)(tiles * bm * bn);
  };
  if (fills(256, 256, 192, 0.8)) return {MxPlan::TILES, 256, 256, 1};
  if (fills(128, 128, 256, 0.75)) return {MxPlan::TILES, 128, 128, 1};
  if (fills(64, 128, 192, 0.0)) return {MxPlan::TILES, 64, 128, 1};
  const int64_t tiles = ((rows + 63) / 64) * ((n + 63) / 64);
  int64_t parts = steps / 16 < 512 / tiles ? steps / 16 : 512 / tiles;
  parts = parts > 8 ? 8 : parts < 1 ? 1 : parts;
  return {MxPlan::TILES, 64, 64, (int32_t)parts};
}

static int64_t part_stride(int64_t n) { return (n + 7) / 8 * 8; }

template <int XBITS>
static int run_plan(const MxPlan &plan, const MxLinearArgs &a, hipStream_t stream) {
  if (plan.kind == MxPlan::STREAM) return launch_stream<XBITS, STREAM_WAVES, STREAM_GROUPS>(a, stream);
  if (plan.kind == MxPlan::ROWS)
    return a.n <= 4096 ? launch_rows<XBITS, 1, 8>(a, stream) : launch_rows<XBITS, 2, 8>(a, stream);
  if constexpr (XBITS != 16) {
    if (plan.bm == 256) {
      // A tile a CU: where the last round is for few, its columns' tiles go to a launch of smaller
      // ones. Measured, 1024 to 4096 rows, 1 / 4 / 9 whole rounds and a last one of
      //   16 tiles  8-bit x -23 / -8 / -2 %, 4-bit x -18 / -8 / -1 %;  48   -13 / -5 / -2, -9 / -4 / +1
      //   80        -5 / -3 / -2, -1 / -1 / +1;  112  -3 / -1 / -1, +3 / 0 / +3;  144 and more  +3 and more
      const int64_t tm = (a.rows + 255) / 256, tn = ((int64_t)a.n + 255) / 256, last = tm * tn % CUS;
      const int64_t moved = (last + tm - 1) / tm;
      const int64_t most = XBITS == 8 ? 96 : tm * tn < 8 * CUS ? 64 : 0;
      if (tm * tn > CUS && last > 0 && last <= most && moved < tn) {
        MxLinearArgs body = a, tail = a;
        body.n = (int32_t)(256 * (tn - moved)), tail.n = a.n - body.n;
        tail.w += body.n * a.ws, tail.wsc += body.n * a.wss, tail.out += body.n;
        if (a.bias != nullptr) tail.bias += body.n;
        const int rc = launch_tiles<XBITS, 256, 256, 4, 2, true>(body, 1, stream);
        if (rc != FM_OK) return rc;
        MxPlan rest = plan_of(a.rows, tail.n, a.k, XBITS);
        rest.parts = 1;
        return rest.bm == 256 ? launch_tiles<XBITS, 256, 256, 4, 2, true>(tail, 1, stream)
                              : run_plan<XBITS>(rest, tail, stream);
      }
      return launch_tiles<XBITS, 256, 256, 4, 2, true>(a, 1, stream);
    }
    if (plan.bm == 128) return launch_tiles<XBITS, 128, 128, 2, 2, false>(a, 1, stream);
    if (plan.bn == 128) return launch_tiles<XBITS, 64, 128, 1, 4, false>(a, 1, stream);
    return launch_tiles<XBITS, 64, 64, 2, 2, false>(a, plan.parts, stream);
  }
  return fail(FM_ERR_UNSUPPORTED, "bf16 x of more than %d rows", MX_BF16_ROWS);
}

// Whether the kernel quantizes bf16 rows itself: for longer sums a pass of its own in front is
// cheaper (16 rows, us: 8192 -> 2048 15.6 / 14, 20480 -> 2048 33.7 / 19), and so it is for more rows,
// where every workgroup would quantize them again. With more than 8192 columns 5632 values are the
// longest rows that lie in LDS beside the streams' rings.
static bool quantizes(int64_t rows, int64_t n, int64_t k) {
  return rows <= MX_BF16_ROWS && k % 8 == 0 && (n <= 8192 ? k < 8192 : k <= 5632);
}

static int32_t out_unit(const void *out, int64_t stride) {
  for (int32_t unit = 8; unit > 1; unit /= 2)
    if (aligned(out, 2 * unit) && stride % unit == 0) return unit;
  return 1;
}

// The workspace: the sums of parts of k, then bf16 rows as 8-bit codes and scales.
struct MxWorkspace {
  size_t parts, codes, scales;  // bytes
};
static MxWorkspace workspace_of(int64_t rows, int64_t n, int64_t k, int32_t x_bits) {
  const bool first = x_bits == 16 && !quantizes(rows, n, k);
  const MxPlan plan = plan_of(rows, n, k, first ? 8 : x_bits);
  const int64_t kp = mx_padded(k);
  return {plan.parts == 1 ? 0 : (size_t)(plan.parts * rows * part_stride(n)) * sizeof(float),
          first ? (size_t)(rows * kp) : 0, first ? (size_t)(rows * kp / MX_BLOCK) : 0};
}

}  // namespace fm

extern "C" size_t fm_mx_linear_workspace_bytes(int64_t rows, int64_t n, int64_t k, int32_t x_bits) {
  using namespace fm;
  if (rows <= 0 || n <= 0 || k <= 0 || k > 1 << 22 || n > 1 << 26 || rows > 1 << 26) return 0;
  const MxWorkspace ws = workspace_of(rows, n, k, x_bits);
  return ws.parts + ws.codes + ws.scales;
}

extern "C" int fm_mx_linear(const void *x, int32_t x_bits, int64_t x_stride, const void *x_scales,
                            int64_t x_scales_stride, const void *w, int64_t w_stride, const void *w_scales,
                            int64_t w_scales_stride, const void *bias, void *out, int64_t out_stride, int64_t rows,
                            int64_t n, int64_t k, void *workspace, size_t workspace_bytes, void *stream) {
  using namespace fm;
  FM_REQUIRE(rows >= 0 && n >= 0 && k > 0, "bad sizes: rows=%lld n=%lld k=%lld", (long long)rows, (long long)n,
             (long long)k);
  FM_REQUIRE(x_bits == 4 || x_bits == 8 || x_bits == 16, "x_bits %d: 4, 8 or 16 (bf16)", x_bits);
  if (rows == 0 || n == 0) return FM_OK;
  if (k > 1 << 22 || n > 1 << 26 || rows > 1 << 26)
    return fail(FM_ERR_UNSUPPORTED, "%lld rows, %lld columns: at most 2^26; sums of %lld: at most 2^22", (long long)rows,
                (long long)n, (long long)k);
  FM_REQUIRE(x && w && w_scales && out, "NULL tensor pointer");
  const int64_t kp = mx_padded(k);
  FM_REQUIRE(aligned(w, 16) && w_stride % 16 == 0 && w_stride >= kp / 2 && aligned(w_scales, 4) &&
                 w_scales_stride % 4 == 0 && w_scales_stride >= kp / MX_BLOCK,
             "w: 16-byte aligned rows of %lld bytes, 4-byte aligned scales of %lld", (long long)(kp / 2),
             (long long)(kp / MX_BLOCK));
  // The tiles' offsets from their first row are 32 bits.
  FM_REQUIRE(w_stride < 1 << 24 && w_scales_stride < 1 << 24 && (x_bits == 16 || (x_stride < 1 << 24 && x_scales_stride < 1 << 24)),
             "rows of codes and scales: strides below 2^24 bytes");
  FM_REQUIRE(aligned(out, 2) && aligned(bias, 2) && (rows == 1 || out_stride >= n), "out rows must cover %lld values",
             (long long)n);
  if (x_bits == 16 && quantizes(rows, n, k)) {
    FM_REQUIRE(aligned(x, 16) && x_stride % 8 == 0 && (rows == 1 || x_stride >= k),
               "bf16 x: 16-byte aligned rows, a stride of a multiple of 8 values");
  } else if (x_bits != 16) {
    FM_REQUIRE(x_scales && aligned(x, 16) && x_stride % 16 == 0 && x_stride >= kp * x_bits / 8 && aligned(x_scales, 4) &&
                   x_scales_stride % 4 == 0 && x_scales_stride >= kp / MX_BLOCK,
               "x: 16-byte aligned rows of %lld bytes, 4-byte aligned scales of %lld", (long long)(kp * x_bits / 8),
               (long long)(kp / MX_BLOCK));
  }
  const MxWorkspace ws = workspace_of(rows, n, k, x_bits);
  const size_t need = ws.parts + ws.codes + ws.scales;
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(FM_ERR_WORKSPACE, "workspace of %zu bytes, need %zu (16-byte aligned)", workspace_bytes, need);
  if (ws.codes > 0) {
    uint8_t *codes = (uint8_t *)workspace + ws.parts, *scales = codes + ws.codes;
    const int rc = fm_mx_quantize(x, 0, x_stride, 0, 8, codes, kp, scales, kp / MX_BLOCK, rows, k, stream);
    if (rc != FM_OK) return rc;
    x = codes, x_bits = 8, x_stride = kp, x_scales = scales, x_scales_stride = kp / MX_BLOCK;
  }
  const MxPlan plan = plan_of(rows, n, k, x_bits);
  const MxLinearArgs a{(const uint8_t *)x, (const uint8_t *)x_scales, (const uint8_t *)w, (const uint8_t *)w_scales,
                       (const uint16_t *)bias, (uint16_t *)out, x_bits == 16 ? 2 * x_stride : x_stride, x_scales_stride,
                       w_stride, w_scales_stride, out_stride, rows, (int32_t)n, (int32_t)k, (int32_t)(kp / MX_PAD),
                       out_unit(out, out_stride), (float *)workspace, part_stride(n)};
  const hipStream_t st = (hipStream_t)stream;
  return x_bits == 16 ? run_plan<16>(plan, a, st) : x_bits == 8 ? run_plan<8>(plan, a, st) : run_plan<4>(plan, a, st);
}
