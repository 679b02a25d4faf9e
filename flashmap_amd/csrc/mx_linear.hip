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

struct MxLinearArgs {
  const uint8_t *x, *xsc, *w, *wsc;
  const uint16_t *bias;
  uint16_t *out;
  int64_t xs, xss, ws, wss, os;  // row strides (bytes; out: elements)
  int64_t rows;
  int32_t n;
  int32_t steps;  // of 128 along k
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

// A workgroup owns 16 rows of W and 16 of x; its wavefronts split k and meet in LDS in a
// fixed order.
constexpr int MX_WAVES = 4;

template <int XBITS>
__global__ __launch_bounds__(64 * MX_WAVES) void mx_linear_rows_kernel(const MxLinearArgs a) {
  __shared__ f32x4_t part[MX_WAVES][64];
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int r = lane & 15, g = lane >> 4;
  const int32_t n0 = (int32_t)blockIdx.x * 16;
  const int64_t m0 = (int64_t)blockIdx.y * 16;
  // Rows past the end read the last one: their results are not stored.
  const int64_t nr = n0 + r < a.n ? n0 + r : a.n - 1, mr = m0 + r < a.rows ? m0 + r : a.rows - 1;
  const uint8_t *w = a.w + nr * a.ws + 16 * g, *wsc = a.wsc + nr * a.wss + g;
  const uint8_t *x = a.x + mr * a.xs + 16 * g, *xsc = a.xsc + mr * a.xss + g;
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
  for (int32_t s = wave; s < a.steps; s += MX_WAVES) {
    const i32x8_t wf = operand(load16(w + 64 * (int64_t)s));
    i32x8_t xf;
    if constexpr (XBITS == 8)
      xf = operand(load16(x + 128 * (int64_t)s), load16(x + 128 * (int64_t)s + 64));
    else
      xf = operand(load16(x + 64 * (int64_t)s));
    acc = mfma_mx<XBITS>(wf, xf, acc, wsc[4 * (int64_t)s], xsc[4 * (int64_t)s]);
  }
  part[wave][lane] = acc;
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int i = 1; i < MX_WAVES; ++i) acc += part[i][lane];
  // Lane: row m of out, columns n0 + 4 g .. + 3.
  const int64_t m = m0 + r;
  if (m >= a.rows) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int32_t n = n0 + 4 * g + i;
    if (n >= a.n) break;
    const float v = a.bias != nullptr ? acc[i] + bf16_to_f32(a.bias[n]) : acc[i];
    a.out[m * a.os + n] = (uint16_t)(pack_bf16x2(v, 0.f) & 0xffffu);
  }
}

// ------------------------------------------------------------------------ many rows: tiles

// One 16-byte-per-lane load straight into LDS: lane l's bytes go to lds + 16 l. Inline asm, so
// that the compiler, which cannot tell the stages apart, does not wait for the loads in
// flight before every LDS read; the waits are counted by hand (wait_vm before the barrier
// that publishes a stage).
typedef __attribute__((address_space(3))) char lds_char_t;
__device__ __forceinline__ void dma16(const void *src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds), "v"(src) : "memory", "m0");
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
  static constexpr int LDS = STAGES * STAGE + 2 * SCALES;
  static constexpr int MF = BM / WM / 16, NF = BN / WN / 16;  // 16-row blocks of a wavefront
  static_assert(XU % WAVES == 0 && WU % WAVES == 0 && (BM + BN) % 64 == 0, "whole units a wavefront");
  static constexpr int SW = (BM + BN) / 64;  // wavefronts that load scales (one row a lane)
  static_assert(SW <= WAVES, "a row a lane");
};

// The row of W (in its 32-row group pair) that block f holds at index r: lane group g of the
// accumulators then holds 8 consecutive columns of out in blocks 2 p and 2 p + 1, which are
// stored 16 bytes at a time, 64 consecutive bytes a row.
__device__ __forceinline__ int w_row(int f, int r) { return 32 * (f >> 1) + 8 * (r >> 2) + 4 * (f & 1) + (r & 3); }

template <int XBITS, int OP>
__device__ __forceinline__ f32x4_t mfma_mx_op(const i32x8_t &a, const i32x8_t &b, f32x4_t c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, XBITS == 8 ? 0 : 4, OP, sa, OP, sb);
}

template <int XBITS, int BM, int BN, int WM, int WN>
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
  const uint8_t *src[T::PER];
#pragma unroll
  for (int u = 0; u < T::XPW; ++u) {
    const int unit = wave * T::XPW + u, f = XBITS == 8 ? unit >> 1 : unit, h = XBITS == 8 ? unit & 1 : 0;
    const int64_t m = m0 + 16 * f + r;
    src[u] = a.x + (m < a.rows ? m : a.rows - 1) * a.xs + 64 * h + 16 * g;
  }
#pragma unroll
  for (int u = 0; u < T::WPW; ++u) {
    const int32_t n = n0 + w_row(wave * T::WPW + u, r);
    src[T::XPW + u] = a.w + (int64_t)(n < a.n ? n : a.n - 1) * a.ws + 16 * g;
  }
  const uint8_t *ssrc;  // this lane's row of scales: x's rows, then W's
  {
    const int row = 64 * wave + lane;
    const int64_t m = m0 + row;
    const int32_t n = n0 + row - BM;
    ssrc = row < BM ? a.xsc + (m < a.rows ? m : a.rows - 1) * a.xss
                    : a.wsc + (int64_t)(n < a.n ? n : a.n - 1) * a.wss;
  }
  auto issue = [&](int stage) {  // the next step, into `stage`
    const uint32_t dst = lds0 + stage * T::STAGE;
#pragma unroll
    for (int u = 0; u < T::XPW; ++u) {
      dma16(src[u], dst + 1024 * (wave * T::XPW + u));
      src[u] += XBITS == 8 ? 128 : 64;
    }
#pragma unroll
    for (int u = 0; u < T::WPW; ++u) {
      dma16(src[T::XPW + u], dst + 1024 * (T::XU + wave * T::WPW + u));
      src[T::XPW + u] += 64;
    }
  };
  // Four steps' scales of a row at once. The last chunk's 16 bytes end with the row: they hold
  // `back` steps of the chunk before it first.
  const int32_t steps = a.steps, back = -steps & 3;
  auto issue_scales = [&](int32_t chunk) {
    const int64_t from = 16 * (int64_t)chunk - (4 * chunk + 4 > steps ? 4 * back : 0);
    if (wave < T::SW) dma16(ssrc + from, sc0 + (chunk & 1) * T::SCALES + 1024 * wave);
  };
  // A row's 16 scale bytes, (step, block) as stored, to (block, step): lane group g then reads
  // one dword a row, whose byte `step` the instruction selects. A lane turns the row that it
  // loaded itself.
  auto turn_scales = [&](int32_t chunk) {
    if (wave >= T::SW) return;
    u32x4_t *p = (u32x4_t *)(lds + T::STAGES * T::STAGE + (chunk & 1) * T::SCALES + 1024 * wave + 16 * lane);
    u32x4_t d;
    if (steps < 4) {  // a row shorter than 16 bytes: read dword by dword
#pragma unroll
      for (int i = 0; i < 3; ++i) d[i] = i < steps ? *(const uint32_t *)(ssrc + 4 * i) : 0u;
      d[3] = 0u;
    } else {
      d = *p;
      if (4 * chunk + 4 > steps)
        d = back == 1 ? u32x4_t{d[1], d[2], d[3], 0u} : back == 2 ? u32x4_t{d[2], d[3], 0u, 0u} : u32x4_t{d[3], 0u, 0u, 0u};
    }
    const uint32_t a01 = __builtin_amdgcn_perm(d[1], d[0], 0x05010400), b01 = __builtin_amdgcn_perm(d[1], d[0], 0x07030602);
    const uint32_t a23 = __builtin_amdgcn_perm(d[3], d[2], 0x05010400), b23 = __builtin_amdgcn_perm(d[3], d[2], 0x07030602);
    *p = u32x4_t{__builtin_amdgcn_perm(a23, a01, 0x05040100), __builtin_amdgcn_perm(a23, a01, 0x07060302),
                 __builtin_amdgcn_perm(b23, b01, 0x05040100), __builtin_amdgcn_perm(b23, b01, 0x07060302)};
  };

  f32x4_t acc[T::NF][T::MF];
#pragma unroll
  for (int j = 0; j < T::NF; ++j)
#pragma unroll
    for (int i = 0; i < T::MF; ++i) acc[j][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  if (steps >= 4) issue_scales(0);
  issue(0);
  if (steps > 1) {
    issue(1);
    wait_vm<T::PER>();
  } else {
    wait_vm<0>();
  }
  turn_scales(0);
  int sx[T::MF], sw[T::NF];
  int stage = 0;  // of step s
  // Step s = 4 chunk + J: its stage has landed (what is still in flight is the next step's);
  // past the barrier nobody reads the stage of step s - 1 any more, which takes step s + 2.
  auto step = [&](auto jc, int32_t chunk) {
    constexpr int J = decltype(jc)::value;
    const int32_t s = 4 * chunk + J;
    if (s >= steps) return;
    if (s + 1 < steps)
      wait_vm<T::PER>();
    else
      wait_vm<0>();
    if (J == 2 && 4 * chunk + 4 < steps) turn_scales(chunk + 1);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (J == 0 && 4 * chunk + 4 < steps) issue_scales(chunk + 1);
    if (s + 2 < steps) issue(stage == 0 ? 2 : stage - 1);
    const char *xs = lds + stage * T::STAGE + 1024 * (XBITS == 8 ? 2 : 1) * wm * T::MF + 16 * lane;
    const char *ws = lds + stage * T::STAGE + 1024 * (T::XU + wn * T::NF) + 16 * lane;
    if constexpr (J == 0) {
      const char *sc = lds + T::STAGES * T::STAGE + (chunk & 1) * T::SCALES + 4 * g;
#pragma unroll
      for (int i = 0; i < T::MF; ++i) sx[i] = *(const int *)(sc + 16 * (16 * (wm * T::MF + i) + r));
#pragma unroll
      for (int j = 0; j < T::NF; ++j) sw[j] = *(const int *)(sc + 16 * (BM + w_row(wn * T::NF + j, r)));
    }
    i32x8_t xf[T::MF];
#pragma unroll
    for (int i = 0; i < T::MF; ++i) {
      if constexpr (XBITS == 8)
        xf[i] = operand(load16(xs + 2048 * i), load16(xs + 2048 * i + 1024));
      else
        xf[i] = operand(load16(xs + 1024 * i));
    }
#pragma unroll
    for (int j = 0; j < T::NF; ++j) {
      const i32x8_t wf = operand(load16(ws + 1024 * j));
#pragma unroll
      for (int i = 0; i < T::MF; ++i) acc[j][i] = mfma_mx_op<XBITS, J>(wf, xf[i], acc[j][i], sw[j], sx[i]);
    }
    stage = stage == 2 ? 0 : stage + 1;
  };
  for (int32_t chunk = 0; 4 * chunk < steps; ++chunk) {
    step(std::integral_constant<int, 0>{}, chunk);
    step(std::integral_constant<int, 1>{}, chunk);
    step(std::integral_constant<int, 2>{}, chunk);
    step(std::integral_constant<int, 3>{}, chunk);
  }

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

template <int XBITS, int BM, int BN, int WM, int WN>
static int launch_tiles(const MxLinearArgs &a, hipStream_t stream) {
  const int64_t tm = (a.rows + BM - 1) / BM, tn = ((int64_t)a.n + BN - 1) / BN;
  // At most 2^22 workgroups a launch: slices of whole groups of row tiles.
  const int64_t most = (1 << 22) / tn < 8 ? 8 : (1 << 22) / tn / 8 * 8;
  for (int64_t first = 0; first < tm; first += most) {
    MxLinearArgs part = a;
    const int64_t rows = a.rows - first * BM, here = tm - first < most ? tm - first : most;
    part.x += first * BM * a.xs, part.xsc += first * BM * a.xss, part.out += first * BM * a.os;
    part.rows = rows < here * BM ? rows : here * BM;
    mx_linear_tile_kernel<XBITS, BM, BN, WM, WN>
        <<<dim3((unsigned)(here * tn)), dim3(64 * WM * WN), 0, stream>>>(part, (int32_t)here, (int32_t)tn);
    FM_CHECK_HIP(hipGetLastError());
  }
  return FM_OK;
}

static bool aligned(const void *p, int64_t n) { return ((uintptr_t)p % (uintptr_t)n) == 0; }

}  // namespace fm

extern "C" size_t fm_mx_linear_workspace_bytes(int64_t rows, int64_t n, int64_t k, int32_t x_bits) {
  using namespace fm;
  if (rows <= 0 || n <= 0 || k <= 0 || x_bits != 16) return 0;
  const int64_t kp = mx_padded(k);
  return (size_t)(rows * (kp + kp / MX_BLOCK));
}

extern "C" int fm_mx_linear(const void *x, int32_t x_bits, int64_t x_stride, const void *x_scales,
                            int64_t x_scales_stride, const void *w, int64_t w_stride, const void *w_scales,
                            int64_t w_scales_stride, const void *bias, void *out, int64_t out_stride, int64_t rows,
                            int64_t n, int64_t k, void *workspace, size_t workspace_bytes, void *stream) {
  using namespace fm;
  FM_REQUIRE(rows >= 0 && n >= 0 && k > 0, "bad sizes: rows=%lld n=%lld k=%lld", (long long)rows, (long long)n, (long long)k);
  FM_REQUIRE(x_bits == 4 || x_bits == 8 || x_bits == 16, "x_bits %d: 4, 8 or 16 (bf16)", x_bits);
  if (rows == 0 || n == 0) return FM_OK;
  if (k > 1 << 26 || n > 1 << 26 || rows > 1 << 26)
    return fail(FM_ERR_UNSUPPORTED, "%lld rows, %lld columns of %lld: at most 2^26 each", (long long)rows, (long long)n, (long long)k);
  FM_REQUIRE(x && w && w_scales && out, "NULL tensor pointer");
  const int64_t kp = mx_padded(k);
  FM_REQUIRE(aligned(w, 16) && w_stride % 16 == 0 && w_stride >= kp / 2 && aligned(w_scales, 4) && w_scales_stride % 4 == 0 &&
                 w_scales_stride >= kp / MX_BLOCK,
             "w: 16-byte aligned rows of %lld bytes, 4-byte aligned scales of %lld", (long long)(kp / 2), (long long)(kp / MX_BLOCK));
  FM_REQUIRE(aligned(out, 2) && aligned(bias, 2) && (rows == 1 || out_stride >= n), "out rows must cover %lld values", (long long)n);
  if (x_bits == 16) {
    const size_t need = fm_mx_linear_workspace_bytes(rows, n, k, x_bits);
    if (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16))
      return fail(FM_ERR_WORKSPACE, "workspace of %zu bytes, need %zu (16-byte aligned)", workspace_bytes, need);
    uint8_t *codes = (uint8_t *)workspace, *scales = codes + rows * kp;
    const int rc = fm_mx_quantize(x, 0, x_stride, 0, 8, codes, kp, scales, kp / MX_BLOCK, rows, k, stream);
    if (rc != FM_OK) return rc;
    x = codes, x_stride = kp, x_scales = scales, x_scales_stride = kp / MX_BLOCK;
    x_bits = 8;
  }
  FM_REQUIRE(x_scales && aligned(x, 16) && x_stride % 16 == 0 && x_stride >= kp * x_bits / 8 && aligned(x_scales, 4) &&
                 x_scales_stride % 4 == 0 && x_scales_stride >= kp / MX_BLOCK,
             "x: 16-byte aligned rows of %lld bytes, 4-byte aligned scales of %lld", (long long)(kp * x_bits / 8),
             (long long)(kp / MX_BLOCK));
  MxLinearArgs a{(const uint8_t *)x, (const uint8_t *)x_scales, (const uint8_t *)w, (const uint8_t *)w_scales,
                 (const uint16_t *)bias, (uint16_t *)out, x_stride, x_scales_stride, w_stride, w_scales_stride,
                 out_stride, rows, (int32_t)n, (int32_t)(kp / MX_PAD), aligned(out, 16) && out_stride % 8 == 0};
  if (rows > 64) {
    const bool large = ((rows + 255) / 256) * ((n + 255) / 256) >= 256;
    auto go = [&](auto xb) {
      constexpr int XB = decltype(xb)::value;
      return large ? launch_tiles<XB, 256, 256, 4, 2>(a, (hipStream_t)stream)
                   : launch_tiles<XB, 128, 128, 2, 2>(a, (hipStream_t)stream);
    };
    return x_bits == 8 ? go(std::integral_constant<int, 8>{}) : go(std::integral_constant<int, 4>{});
  }
  const int64_t nt = (n + 15) / 16;  // at most 2^22 workgroups of 256 threads along n: 2^30 threads
  int64_t mt = (1 << 22) / nt;
  mt = mt < 1 ? 1 : mt > 65535 ? 65535 : mt;
  for (int64_t first = 0; first < rows; first += 16 * mt) {
    MxLinearArgs part = a;
    part.x += first * x_stride, part.xsc += first * x_scales_stride, part.out += first * out_stride;
    part.rows = rows - first < 16 * mt ? rows - first : 16 * mt;
    const dim3 grid((unsigned)nt, (unsigned)((part.rows + 15) / 16));
    if (x_bits == 8)
      mx_linear_rows_kernel<8><<<grid, dim3(64 * MX_WAVES), 0, (hipStream_t)stream>>>(part);
    else
      mx_linear_rows_kernel<4><<<grid, dim3(64 * MX_WAVES), 0, (hipStream_t)stream>>>(part);
    FM_CHECK_HIP(hipGetLastError());
  }
  return FM_OK;
}
