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
// (checked lane by lane against the formula). Sums of e2m1 products are exact until they pass
// 24 bits; with an e4m3 operand the instruction aligns a step's 128 products to the largest
// of them and drops what lies about 2^-17 below it (measured, sums of 128 to 65536 products:
// 4e-6 to 9e-6 of the result; the rounding to bf16 is 2^-9 on average).
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
  int32_t vec_out;  // rows of out may be written 16 bytes at a time
};

// D(16x16 f32) += A(16x128 e2m1) * B(128x16 e4m3 or e2m1), block scales in byte 0 of sa, sb.
template <int XBITS>
__device__ __forceinline__ f32x4_t mfma_mx(const i32x8_t &a, const i32x8_t &b, f32x4_t c, int sa, int sb) {
  if constexpr (XBITS == 8)
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 0, 0, sa, 0, sb);
  else
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 4, 0, sa, 0, sb);
}

__device__ __forceinline__ i32x8_t operand(u32x4_t lo) {
  return i32x8_t{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], 0, 0, 0, 0};
}
__device__ __forceinline__ i32x8_t operand(u32x4_t lo, u32x4_t hi) {
  return i32x8_t{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}

// -------------------------------------------------------------------- few rows: streaming

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

// A workgroup owns 16 NB rows of W against 16 MB rows of x; its wavefronts split k and meet in
// LDS in a fixed order. XBITS 16: x in bf16, quantized in registers.
template <int XBITS, int MB, int NB, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void mx_linear_rows_kernel(const MxLinearArgs a) {
  __shared__ f32x4_t part[WAVES][NB * MB][64];
  constexpr int XL = XBITS == 16 ? 4 : XBITS == 8 ? 2 : 1;  // 16-byte loads of x a step
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int r = lane & 15, g = lane >> 4;
  const int32_t n0 = (int32_t)blockIdx.x * 16 * NB;
  const int32_t s0 = (int32_t)((int64_t)a.steps * wave / WAVES), s1 = (int32_t)((int64_t)a.steps * (wave + 1) / WAVES);
  // Rows past the end read the last one: their results are not stored.
  const uint8_t *w[NB], *wsc[NB], *x[MB], *xsc[MB];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int64_t n = n0 + 16 * j + r < a.n ? n0 + 16 * j + r : a.n - 1;
    w[j] = a.w + n * a.ws + 16 * g, wsc[j] = a.wsc + n * a.wss + g;
  }
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    const int64_t m = 16 * i + r < a.rows ? 16 * i + r : a.rows - 1;
    x[i] = a.x + m * a.xs + (XBITS == 16 ? 32 : 16) * g;
    xsc[i] = XBITS == 16 ? nullptr : a.xsc + m * a.xss + g;
  }
  f32x4_t acc[NB][MB];
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int i = 0; i < MB; ++i) acc[j][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  auto take = [&](auto group, int32_t s) {  // steps s .. s + G - 1, all their loads in flight at once
    constexpr int G = decltype(group)::value;
    u32x4_t wf[G][NB], xf[G][MB][XL];
    int sw[G][NB], sx[G][MB];
#pragma unroll
    for (int t = 0; t < G; ++t) {
      const int64_t at = s + t;
#pragma unroll
      for (int j = 0; j < NB; ++j) wf[t][j] = load16(w[j] + 64 * at), sw[t][j] = wsc[j][4 * at];
    }
#pragma unroll
    for (int t = 0; t < G; ++t) {
      const int64_t at = s + t;
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        if constexpr (XBITS == 16) {
          // k is a multiple of 8: a 16-byte load past the row's end is zeros
          const int32_t k0 = 128 * (int32_t)at + 16 * g;
#pragma unroll
          for (int l = 0; l < 4; ++l) {
            const int o = 64 * (l >> 1) + 8 * (l & 1);
            xf[t][i][l] = k0 + o < a.k ? load16(x[i] + 256 * at + 2 * o) : u32x4_t{0, 0, 0, 0};
          }
        } else {
#pragma unroll
          for (int l = 0; l < XL; ++l) xf[t][i][l] = load16(x[i] + 64 * XL * at + 64 * l);
          sx[t][i] = xsc[i][4 * at];
        }
      }
    }
#pragma unroll
    for (int t = 0; t < G; ++t) {
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        i32x8_t xo;
        if constexpr (XBITS == 16)
          quantize_operand(xf[t][i], g, xo, sx[t][i]);
        else if constexpr (XBITS == 8)
          xo = operand(xf[t][i][0], xf[t][i][1]);
        else
          xo = operand(xf[t][i][0]);
#pragma unroll
        for (int j = 0; j < NB; ++j)
          acc[j][i] = mfma_mx<XBITS == 4 ? 4 : 8>(operand(wf[t][j]), xo, acc[j][i], sw[t][j], sx[t][i]);
      }
    }
  };
  int32_t s = s0;
  for (; s + 4 <= s1; s += 4) take(std::integral_constant<int, 4>{}, s);
  if (s1 - s & 2) take(std::integral_constant<int, 2>{}, s), s += 2;
  if (s1 - s & 1) take(std::integral_constant<int, 1>{}, s);
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int i = 0; i < MB; ++i) part[wave][j * MB + i][lane] = acc[j][i];
  __syncthreads();
  for (int b = wave; b < NB * MB; b += WAVES) {
    f32x4_t sum = part[0][b][lane];
#pragma unroll
    for (int q = 1; q < WAVES; ++q) sum += part[q][b][lane];
    // Lane: row m of out, columns n .. n + 3.
    const int32_t m = 16 * (b % MB) + r, n = n0 + 16 * (b / MB) + 4 * g;
    if (m >= a.rows) continue;
    uint16_t *dst = a.out + m * a.os + n;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (a.bias != nullptr && n + i < a.n) sum[i] += bf16_to_f32(a.bias[n + i]);
    if (a.vec_out && n + 4 <= a.n) {
      *reinterpret_cast<u32x2_t *>(dst) = u32x2_t{pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3])};
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < a.n) dst[i] = (uint16_t)(pack_bf16x2(sum[i], 0.f) & 0xffffu);
    }
  }
}

template <int XBITS, int MB, int NB, int WAVES>
static int launch_rows(const MxLinearArgs &a, hipStream_t stream) {
  const unsigned tiles = (unsigned)((a.n + 16 * NB - 1) / (16 * NB));
  mx_linear_rows_kernel<XBITS, MB, NB, WAVES><<<dim3(tiles), dim3(64 * WAVES), 0, stream>>>(a);
  FM_CHECK_HIP(hipGetLastError());
  return FM_OK;
}

// ------------------------------------------------------------------------ many rows: tiles

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
template <int N>
__device__ __forceinline__ void wait_vm() {
  static_assert(N >= 0 && N < 64, "vmcnt holds 6 bits");
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

template <int XBITS, int BM, int BN, int WM, int WN>
struct Tile {
  static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
  static constexpr int XU = BM / 16 * (XBITS == 8 ? 2 : 1), WU = BN / 16;  // 1 KiB units of a stage
  static constexpr int XPW = XU / WAVES, WPW = WU / WAVES, PER = XPW + WPW;  // units a wavefront loads
  static constexpr int STAGE = 1024 * (XU + WU), STAGES = 3;
  static constexpr int SCALES = 16 * (BM + BN);  // one chunk of four steps
  static constexpr int LDS = STAGES * STAGE + SCALES;
  static constexpr int MF = BM / WM / 16, NF = BN / WN / 16;  // 16-row blocks of a wavefront
  static_assert(XU % WAVES == 0 && WU % WAVES == 0 && (BM + BN) % 64 == 0, "whole units a wavefront");
  static constexpr int SW = (BM + BN) / 64;  // wavefronts that load scales (one row a lane)
  static_assert(SW <= WAVES, "a row a lane");
};

// Where a row's 16-byte pieces lie in LDS. A load's neighbouring lanes take a row's neighbouring
// pieces (whole 64- or 128-byte segments: with a row a lane every lane's 16 bytes are a request
// of their own), so a stage holds rows of 4 or 8 pieces, piece c of row r at place c ^ swizzle(r).
// ds_read_b128 serves 16 lanes at a time, and not neighbours: lanes 0-3, 12-15, 20-23, 24-27,
// then the other 16 of the lower half, then the upper half alike (measured by which lanes'
// conflicts add up). The 16 rows of an operand read are then all different, half of them one
// piece on; with these places they fall on all 64 banks.
__device__ __forceinline__ int swizzle4(int r) { return r >> 3 ? 3 : 0; }
__device__ __forceinline__ int swizzle8(int r) { return r >> 1 ^ ((r >> 2 ^ r >> 3) & 1); }

// The row of W (in its 32-row group pair) that block f holds at index r: lane group g of the
// accumulators then holds 8 consecutive columns of out in blocks 2 p and 2 p + 1, which are
// stored 16 bytes at a time, 64 consecutive bytes a row.
__device__ __forceinline__ int w_row(int f, int r) { return 32 * (f >> 1) + 8 * (r >> 2) + 4 * (f & 1) + (r & 3); }

template <int XBITS, int OP>
__device__ __forceinline__ f32x4_t mfma_mx_op(const i32x8_t &a, const i32x8_t &b, f32x4_t c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, XBITS == 8 ? 0 : 4, OP, sa, OP, sb);
}

template <int XBITS, int BM, int BN, int WM, int WN, bool TURNS>
__global__ __launch_bounds__(64 * WM * WN, 2) void mx_linear_tile_kernel(const MxLinearArgs a,
                                                                                       const int32_t tiles_m,
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
  // This wavefront's units: x's first, then W's. Rows past the end read the last one.
  // Offsets from the tile's first row stay below 2^32 (k is at most 2^22, rows at most 256).
  const uint8_t *xbase = a.x + m0 * a.xs, *wbase = a.w + (int64_t)n0 * a.ws;
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
  const int32_t steps = a.steps, back = -steps & 3;
  static_assert(BM % 64 == 0, "a wavefront's rows are all x's or all W's");
  const bool of_x = 64 * wave < BM;
  const uint8_t *sbase = of_x ? a.xsc + m0 * a.xss : a.wsc + (int64_t)n0 * a.wss;
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
  if (TURNS && !late) barrier();

  // Lane (r, g): row m of out, 8 columns from 8 g on in each 32-column group.
  const bool vec = a.vec_out != 0;
#pragma unroll
  for (int p = 0; p < T::NF / 2; ++p) {
    const int32_t n = n0 + 32 * (wn * (T::NF / 2) + p) + 8 * g;
    float b[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) b[q] = a.bias != nullptr && n + q < a.n ? bf16_to_f32(a.bias[n + q]) : 0.f;
#pragma unroll
    for (int i = 0; i < T::MF; ++i) {
      const int64_t m = m0 + 16 * (wm * T::MF + i) + r;
      if (m >= a.rows) continue;
      float v[8];
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = acc[2 * p][i][q] + b[q], v[4 + q] = acc[2 * p + 1][i][q] + b[4 + q];
      uint16_t *dst = a.out + m * a.os + n;
      if (vec && n + 8 <= a.n) {
        store16(dst, u32x4_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                             pack_bf16x2(v[6], v[7])});
      } else {
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (n + q < a.n) dst[q] = (uint16_t)(pack_bf16x2(v[q], 0.f) & 0xffffu);
      }
    }
  }
}

template <int XBITS, int BM, int BN, int WM, int WN, bool TURNS>
static int launch_tiles(const MxLinearArgs &a, hipStream_t stream) {
  const int64_t tm = (a.rows + BM - 1) / BM, tn = ((int64_t)a.n + BN - 1) / BN;
  // At most 2^22 workgroups a launch: slices of whole groups of row tiles.
  const int64_t most = (1 << 22) / tn < 8 ? 8 : (1 << 22) / tn / 8 * 8;
  for (int64_t first = 0; first < tm; first += most) {
    MxLinearArgs part = a;
    const int64_t rows = a.rows - first * BM, here = tm - first < most ? tm - first : most;
    part.x += first * BM * a.xs, part.xsc += first * BM * a.xss, part.out += first * BM * a.os;
    part.rows = rows < here * BM ? rows : here * BM;
    mx_linear_tile_kernel<XBITS, BM, BN, WM, WN, TURNS>
        <<<dim3((unsigned)(here * tn)), dim3(64 * WM * WN), 0, stream>>>(part, (int32_t)here, (int32_t)tn);
    FM_CHECK_HIP(hipGetLastError());
  }
  return FM_OK;
}

static bool aligned(const void *p, int64_t n) { return ((uintptr_t)p % (uintptr_t)n) == 0; }

}  // namespace fm

extern "C" size_t fm_mx_linear_workspace_bytes(int64_t rows, int64_t n, int64_t k, int32_t x_bits) {
  return 0;
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
  if (x_bits == 16) {
    if (rows > MX_BF16_ROWS || k % 8 != 0)
      return fail(FM_ERR_UNSUPPORTED, "bf16 x of %lld rows of %lld: at most %d rows, a multiple of 8 values",
                  (long long)rows, (long long)k, MX_BF16_ROWS);
    FM_REQUIRE(aligned(x, 16) && x_stride % 8 == 0 && (rows == 1 || x_stride >= k),
               "bf16 x: 16-byte aligned rows, a stride of a multiple of 8 values");
  } else {
    FM_REQUIRE(x_scales && aligned(x, 16) && x_stride % 16 == 0 && x_stride >= kp * x_bits / 8 && aligned(x_scales, 4) &&
                   x_scales_stride % 4 == 0 && x_scales_stride >= kp / MX_BLOCK,
               "x: 16-byte aligned rows of %lld bytes, 4-byte aligned scales of %lld", (long long)(kp * x_bits / 8),
               (long long)(kp / MX_BLOCK));
  }
  const MxLinearArgs a{(const uint8_t *)x, (const uint8_t *)x_scales, (const uint8_t *)w, (const uint8_t *)w_scales,
                       (const uint16_t *)bias, (uint16_t *)out, x_bits == 16 ? 2 * x_stride : x_stride, x_scales_stride,
                       w_stride, w_scales_stride, out_stride, rows, (int32_t)n, (int32_t)k, (int32_t)(kp / MX_PAD),
                       aligned(out, 16) && out_stride % 8 == 0};
  const hipStream_t st = (hipStream_t)stream;
  if (rows > 64) {
    const bool large = ((rows + 255) / 256) * ((n + 255) / 256) >= 256;
    if (x_bits == 8) return large ? launch_tiles<8, 256, 256, 4, 2, true>(a, st) : launch_tiles<8, 128, 128, 2, 2, false>(a, st);
    return large ? launch_tiles<4, 256, 256, 4, 2, true>(a, st) : launch_tiles<4, 128, 128, 2, 2, false>(a, st);
  }
  auto few = [&](auto xb) {
    constexpr int XB = decltype(xb)::value;
    if (rows <= 16) {
      if (n <= 16 * 256) return launch_rows<XB, 1, 1, 16>(a, st);
      if (n <= 64 * 256) return launch_rows<XB, 1, 2, 8>(a, st);
      return launch_rows<XB, 1, 4, 4>(a, st);
    }
    if constexpr (XB != 16) {
      if (rows <= 32) return launch_rows<XB, 2, 2, 4>(a, st);
      return launch_rows<XB, 4, 2, 4>(a, st);
    }
    return (int)FM_ERR_UNSUPPORTED;
  };
  return x_bits == 16 ? few(std::integral_constant<int, 16>{})
         : x_bits == 8 ? few(std::integral_constant<int, 8>{})
                       : few(std::integral_constant<int, 4>{});
}
