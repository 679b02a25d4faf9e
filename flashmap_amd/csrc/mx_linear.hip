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
                 out_stride, rows, (int32_t)n, (int32_t)(kp / MX_PAD)};
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
