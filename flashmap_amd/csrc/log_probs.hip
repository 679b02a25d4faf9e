// What a row of logits says about a token, in one pass over it:
//
//   lp(t) = (x_t - m) / T - log S,   S = sum_j exp((x_j - m) / T),   m = max_j x_j
//   entropy = log S - D / (T S),     D = sum_j (x_j - m) exp((x_j - m) / T)
//   rank(t) = 1 + #{j : x_j > x_t},  and the largest logits with their lp, the lower index first
//   among equals, a NaN before any number.
//
// A workgroup takes a tile of a row: its maximum, then its S, D, count and largest logits, as one
// record; wavefronts then put 64 records together at a time until a row has one. A logit and its
// index are one 64-bit key, whose order is the order of the list.
#include <math.h>

#include "fm_host.h"
#include "logits_device.h"

namespace fm {

constexpr int LP_THREADS = 256, LP_WAVES = LP_THREADS / 64;
constexpr int LP_IT = 4;                          // chunks of 8 logits a thread
constexpr int LP_TILE = 8 * LP_IT * LP_THREADS;   // logits of a workgroup
constexpr int LP_TOP = 32;                        // the longest list
constexpr int LP_JOIN = 64;                       // records that a wavefront puts together

struct LogProbsArgs {
  const char *logits;
  int64_t row_bytes, vocab;
  const int64_t *tokens;  // or NULL
  const float *temps;     // or NULL
  int32_t top;
  int64_t first_row;  // of this launch
  // outputs
  float *token, *entropy, *top_lp;
  int64_t *rank, *top_ids;
  // records of this step and of the next: (rows, parts) of float4 and (rows, parts, top) of keys
  float4 *stats, *stats_out;
  uint64_t *keys, *keys_out;
  int32_t parts, parts_out;
};

__device__ __forceinline__ uint32_t logit_order(float x) {
  x += 0.f;  // -0 is 0
  const uint32_t u = __float_as_uint(x);
  return x != x ? 0xffffffffu : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t o) {
  return __uint_as_float(o >> 31 ? o ^ 0x80000000u : ~o);
}
// 0: no logit.
__device__ __forceinline__ uint64_t logit_key(float x, uint32_t col) { return (uint64_t)logit_order(x) << 32 | (uint32_t)~col; }

__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t w = __shfl_xor((unsigned long long)v, o);
    v = w > v ? w : v;
  }
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}
template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// The logit of the row's token (NaN: the token is none).
template <int TY>
__device__ __forceinline__ float token_logit(const LogProbsArgs &a, int64_t row) {
  const int64_t t = a.tokens == nullptr ? -1 : a.tokens[row];
  if (t < 0 || t >= a.vocab) return NAN;
  const char *src = a.logits + row * a.row_bytes;
  if (TY == LOGITS_BF16) return bf16_to_f32(reinterpret_cast<const uint16_t *>(src)[t]);
  if (TY == LOGITS_F16) return (float)reinterpret_cast<const _Float16 *>(src)[t];
  return reinterpret_cast<const float *>(src)[t];
}

// Part blockIdx.x of row blockIdx.y.
template <int TY>
__global__ __launch_bounds__(LP_THREADS) void log_probs_tile_kernel(const LogProbsArgs a) {
  __shared__ float red[3][LP_WAVES];
  __shared__ int32_t counts[LP_WAVES];
  __shared__ uint64_t best[2][LP_WAVES];
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int64_t row = a.first_row + blockIdx.y;
  const RowView<TY> view(a.logits + row * a.row_bytes, a.vocab);
  const uint32_t g0 = blockIdx.x * (LP_IT * LP_THREADS);
  Chunk<TY> x[LP_IT];
#pragma unroll
  for (int it = 0; it < LP_IT; ++it) x[it] = view.chunk(g0 + it * LP_THREADS + threadIdx.x);
  const float mine = token_logit<TY>(a, row);
  const float inv_t = a.temps == nullptr ? 1.f : 1.f / a.temps[row];
  const float c = inv_t * 1.44269504f;
  if (view.edge(g0, LP_IT * LP_THREADS)) {
#pragma unroll
    for (int it = 0; it < LP_IT; ++it) view.trim(x[it], g0 + it * LP_THREADS + threadIdx.x);
  }
  float m = -INFINITY;
#pragma unroll
  for (int it = 0; it < LP_IT; ++it)
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, x[it].at(j));
  m = wave_max(m);
  if (lane == 0) red[0][wave] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < LP_WAVES; ++w) m = fmaxf(m, red[0][w]);
  // A tile of -inf alone: every exponential is 0, none is of inf - inf.
  const float from = m == -INFINITY ? 0.f : m;
  float s = 0.f, d = 0.f;
  int32_t above = 0;
#pragma unroll
  for (int it = 0; it < LP_IT; ++it)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float v = x[it].at(j), t = v - from;
      const float e = __builtin_amdgcn_exp2f(t * c);
      s += e;
      d = __builtin_fmaf(fmaxf(t, -3e38f), e, d);  // -inf stands for 0 here
      above += v > mine;
    }
  s = wave_sum(s), d = wave_sum(d), above = wave_sum(above);
  if (lane == 0) red[1][wave] = s, red[2][wave] = d, counts[wave] = above;
  __syncthreads();
  const int64_t record = (int64_t)blockIdx.y * a.parts + blockIdx.x;
  if (threadIdx.x == 0) {
    s = d = 0.f, above = 0;
    for (int w = 0; w < LP_WAVES; ++w) s += red[1][w], d += red[2][w], above += counts[w];
    a.stats[record] = make_float4(m, s, d, __int_as_float(above));
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < a.top; ++k) {
    uint64_t top = 0;
#pragma unroll
    for (int it = 0; it < LP_IT; ++it)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t col = 8 * (g0 + it * LP_THREADS + threadIdx.x) - view.skip + j;
        const uint64_t key = col < view.vocab ? logit_key(x[it].at(j), col) : 0;
        if (key < last && key > top) top = key;
      }
    top = wave_max(top);
    if (lane == 0) best[k & 1][wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < LP_WAVES; ++w) top = best[k & 1][w] > top ? best[k & 1][w] : top;
    last = top;
    if (threadIdx.x == 0) a.keys[record * a.top + k] = top;
    if (top == 0) last = 1;  // none left: zeros to the list's end
  }
}

// Records blockIdx.x * 64 to that + 63 of row blockIdx.y; where they are all, the row's results.
template <int TY>
__global__ __launch_bounds__(64) void log_probs_join_kernel(const LogProbsArgs a) {
  __shared__ uint64_t lists[LP_JOIN * LP_TOP];
  const int lane = threadIdx.x;
  const int64_t row = a.first_row + blockIdx.y;
  const int first = blockIdx.x * LP_JOIN, n = a.parts - first < LP_JOIN ? a.parts - first : LP_JOIN;
  const int64_t record = (int64_t)blockIdx.y * a.parts + first;
  for (int i = lane; i < n * a.top; i += 64) lists[i] = a.keys[record * a.top + i];
  const bool results = a.parts_out == 1;
  const float mine = results ? token_logit<TY>(a, row) : 0.f;
  const float temp = a.temps == nullptr ? 1.f : a.temps[row];
  float4 st = lane < n ? a.stats[record + lane] : make_float4(-INFINITY, 0.f, 0.f, 0.f);
  const float m = wave_max(st.x);
  const float off = fmaxf(st.x - m, -3e38f), f = __builtin_amdgcn_exp2f(off * (1.44269504f / temp));
  // A record of -inf alone has S 0 (and f NaN where all are).
  float s = st.y == 0.f ? 0.f : st.y * f;
  float d = st.y == 0.f ? 0.f : __builtin_fmaf(off, s, st.z * f);
  s = wave_sum(s), d = wave_sum(d);
  const int32_t above = wave_sum(lane < n ? __float_as_int(st.w) : 0);
  const int64_t to = (int64_t)blockIdx.y * a.parts_out + blockIdx.x;
  const float log_s = logf(s);
  if (lane == 0) {
    if (!results) {
      a.stats_out[to] = make_float4(m, s, d, __int_as_float(above));
    } else {
      a.entropy[row] = log_s - d / (temp * s);
      if (a.tokens != nullptr) {
        const int64_t t = a.tokens[row];
        a.token[row] = (mine - m) / temp - log_s;
        a.rank[row] = t < 0 || t >= a.vocab ? 0 : (int64_t)above + 1;
      }
    }
  }
  __syncthreads();
  int at = 0;
  for (int k = 0; k < a.top; ++k) {
    const uint64_t head = lane < n && at < a.top ? lists[lane * a.top + at] : 0;
    const uint64_t top = wave_max(head);
    if (head == top) ++at;
    if (lane != 0) continue;
    if (!results) {
      a.keys_out[to * a.top + k] = top;
    } else {
      a.top_ids[row * a.top + k] = (int64_t)(uint32_t)~(uint32_t)top;
      a.top_lp[row * a.top + k] = (logit_of((uint32_t)(top >> 32)) - m) / temp - log_s;
    }
  }
}

static int64_t lp_parts(int64_t vocab) { return (vocab + 7 + LP_TILE - 1) / LP_TILE; }  // rows may start inside a granule

// Rows of one pass: what a launch's grid and the workspace are made for.
static int64_t lp_rows(int64_t rows) { return rows < 32768 ? rows : 32768; }

static size_t lp_bytes(int64_t records, int64_t top) { return (size_t)records * (16 + 8 * (size_t)top); }

template <int TY>
static int run_log_probs(LogProbsArgs a, int64_t rows, char *ws, hipStream_t stream) {
  const int64_t parts = lp_parts(a.vocab), joined = (parts + LP_JOIN - 1) / LP_JOIN, most = lp_rows(rows);
  for (int64_t first = 0; first < rows; first += most) {
    const unsigned n = (unsigned)(rows - first < most ? rows - first : most);
    a.first_row = first;
    a.parts = (int32_t)parts;
    auto set = [&](float4 *&stats, uint64_t *&keys, int64_t at, int64_t records) {
      stats = (float4 *)(ws + at);
      keys = (uint64_t *)(stats + records);
    };
    // Two areas that take turns: the tiles' records, and a 64th of them.
    const int64_t area[2] = {0, (int64_t)lp_bytes(most * parts, a.top)}, room[2] = {most * parts, most * joined};
    int from = 0;
    set(a.stats, a.keys, area[0], room[0]);
    log_probs_tile_kernel<TY><<<dim3((unsigned)parts, n), dim3(LP_THREADS), 0, stream>>>(a);
    FM_CHECK_HIP(hipGetLastError());
    do {
      a.parts_out = (a.parts + LP_JOIN - 1) / LP_JOIN;
      set(a.stats, a.keys, area[from], room[from]);
      set(a.stats_out, a.keys_out, area[1 - from], room[1 - from]);
      log_probs_join_kernel<TY><<<dim3((unsigned)a.parts_out, n), dim3(64), 0, stream>>>(a);
      FM_CHECK_HIP(hipGetLastError());
      a.parts = a.parts_out;
      from = 1 - from;
    } while (a.parts > 1);
  }
  return FM_OK;
}

}  // namespace fm

using namespace fm;

extern "C" size_t fm_log_probs_workspace_bytes(int64_t rows, int64_t vocab, int32_t top) {
  if (rows <= 0 || vocab <= 0 || vocab > INT32_MAX || top < 0 || top > LP_TOP) return 0;
  const int64_t parts = lp_parts(vocab);
  return lp_bytes(lp_rows(rows) * (parts + (parts + LP_JOIN - 1) / LP_JOIN), top);
}

extern "C" int fm_log_probs_rows(const void *logits, int32_t dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                                 const int64_t *tokens, const float *temperatures, int32_t top, float *token,
                                 int64_t *rank, float *entropy, int64_t *top_ids, float *top_log_probs, void *workspace,
                                 size_t workspace_bytes, void *stream) {
  clear_error();
  FM_REQUIRE(rows >= 0 && vocab >= 0, "bad sizes");
  FM_REQUIRE(dtype == LOGITS_BF16 || dtype == LOGITS_F16 || dtype == LOGITS_F32, "unknown logits dtype %d", dtype);
  FM_REQUIRE(top >= 0 && top <= LP_TOP, "top %d: 0 to %d", top, LP_TOP);
  if (rows == 0) return FM_OK;
  FM_REQUIRE(vocab > 0 && vocab <= INT32_MAX, "a vocabulary of 1 to 2^31 - 1, got %lld", (long long)vocab);
  FM_REQUIRE(top <= vocab, "top %d of a vocabulary of %lld", top, (long long)vocab);
  FM_REQUIRE(row_stride >= vocab, "row stride %lld below the vocabulary %lld", (long long)row_stride, (long long)vocab);
  const int es = dtype == LOGITS_F32 ? 4 : 2;
  FM_REQUIRE(logits && entropy && workspace, "NULL logits/entropy/workspace");
  FM_REQUIRE((uintptr_t)logits % es == 0 && (uintptr_t)workspace % 16 == 0,
             "logits must be aligned to their values, the workspace to 16 bytes");
  FM_REQUIRE(tokens == nullptr || (token && rank), "tokens need their outputs");
  FM_REQUIRE(top == 0 || (top_ids && top_log_probs), "a list needs its outputs");
  const size_t need = fm_log_probs_workspace_bytes(rows, vocab, top);
  if (workspace_bytes < need) return fail(FM_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
  LogProbsArgs a{};
  a.logits = (const char *)logits, a.row_bytes = row_stride * es, a.vocab = vocab;
  a.tokens = tokens, a.temps = temperatures, a.top = top;
  a.token = token, a.entropy = entropy, a.top_lp = top_log_probs, a.rank = rank, a.top_ids = top_ids;
  if (dtype == LOGITS_BF16) return run_log_probs<LOGITS_BF16>(a, rows, (char *)workspace, (hipStream_t)stream);
  if (dtype == LOGITS_F16) return run_log_probs<LOGITS_F16>(a, rows, (char *)workspace, (hipStream_t)stream);
  return run_log_probs<LOGITS_F32>(a, rows, (char *)workspace, (hipStream_t)stream);
}
