// What a row of logits says about a token, in one pass over it:
//
//   lp(t) = (x_t - m) / T - log S,   S = sum_j exp((x_j - m) / T),   m = max_j x_j
//   entropy = log S - D / (T S),     D = sum_j (x_j - m) exp((x_j - m) / T)
//   rank(t) = 1 + #{j : x_j > x_t},  and the largest logits with their lp, the lower index first
//   among equals, a NaN before any number.
//
// A row is cut into parts, one where there are rows for the whole chip, and a part is a workgroup's:
// its lanes keep a maximum, S and D of their own, put in line with each new maximum, so that nothing is
// joined before the part's end; the next tile's logits travel meanwhile. Parts leave records, which a
// workgroup a row puts together the same way; a row of one part is done at once.
// 1024 rows of 151936 bf16 logits with a list of 8: 84 us (3.7 TB/s); without a list 67, with loads
// alone 61: the exponentials and the list's tests (10 to 14 operations a logit) are nearly as long
// as the loads, and only partly hidden by them.
// The list: a logit and its index are one 64-bit key, whose order is the order of the list. A
// wavefront meets its columns in rising order and keeps the keys that may be among its largest in LDS. A
// tile whose maximum does not pass the last of them is left at once. Where many lanes pass (the first
// tile), the k-th largest of the lanes' own largest keys, found a bit at a time by ballots, bounds the k-th
// largest of all: about k keys of 2048 remain. They are put in order by counting: a key's place is the
// number of keys above it. What costs most is rising logits, whose tiles all pass.
#include <math.h>

#include "fm_host.h"
#include "logits_device.h"
#include "wave_device.h"

namespace fm {

constexpr int LP_THREADS = 256, LP_WAVES = LP_THREADS / 64;
constexpr int LP_TOP = 32;        // the longest list
constexpr int LP_KEPT = 64;       // keys that a wavefront keeps before it puts them in order
constexpr int LP_ROOM = LP_KEPT + 8 * 64;  // and those that one step may add
constexpr int LP_GROUPS = 1024;   // workgroups that few rows are cut into: 4 a CU
constexpr int LP_SMALL = 8 * LP_THREADS, LP_WIDE = 2 * LP_SMALL;  // logits of a tile

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
  // records of the parts, (rows, parts) of (m, S, D, count) and (rows, parts, top) of keys
  float4 *stats;
  uint64_t *keys;
  int32_t parts, tiles;  // tiles: of a part
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

// log2(e) / T, inside float32 where T is so small (below 5e-39) that it is not: the largest logit's
// exponent is 0 then too, and of any other one the exponential is 0 either way.
__device__ __forceinline__ float exponent_factor(float temp) { return fminf(1.f / temp * 1.44269504f, 3e38f); }

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

// The largest t below 2^bits that at least k lanes' v reach, two bits at a time.
__device__ __forceinline__ uint32_t kth_largest(uint32_t v, int k, int bits) {
  uint32_t t = 0;
#pragma nounroll
  for (int at = bits - 2; at >= 0; at -= 2) {
    int more = 0;
#pragma unroll
    for (uint32_t q = 1; q < 4; ++q) more += __popcll(__ballot(v >= (t | q << at))) >= k;
    t |= (uint32_t)more << at;
  }
  return t;
}

// A wavefront's largest keys. Keys of no logit are 0 and never kept.
template <int TY>
struct LpList {
  // Bits of logit_order() in which logits of the type differ, from the highest: below them negative
  // ones have ones, the others zeros.
  static constexpr int BITS = TY == LOGITS_F32 ? 32 : TY == LOGITS_BF16 ? 16 : 20;
  uint64_t *kept;      // LP_ROOM and then LP_TOP places in LDS
  int top, n;          // n: kept so far, uniform
  uint64_t least;      // keys up to this are not among the largest (0: nothing is known)
  float least_logit;   // its logit, NaN where that says nothing

  __device__ __forceinline__ void start(uint64_t *lds, int k) { kept = lds, top = k, n = 0, least = 0, least_logit = NAN; }
  __device__ __forceinline__ void raise(uint64_t to) {
    if (to <= least) return;
    least = to;
    least_logit = logit_of((uint32_t)(to >> 32));
  }
  // `order`: of a lane's largest logit of those that are about to come; low(order): the low word of its
  // largest key with that logit.
  template <typename F>
  __device__ __forceinline__ void bound(uint32_t order, const F &low) {
    const uint32_t v = order >> (32 - BITS), t = kth_largest(v, top, BITS);
    if (t == 0) return;
    uint64_t to = (uint64_t)t << (64 - BITS);
    if (t >> (BITS - 1) == 0) to |= (uint64_t)((1ull << (32 - BITS)) - 1) << 32;
    if (__popcll(__ballot(v >= t)) > top)  // equals: by their columns
      to |= kth_largest(v == t ? low(order) : 0, top - __popcll(__ballot(v > t)), 32);
    raise(to - 1);
  }
  __device__ __forceinline__ void add(uint64_t key) {
    const bool pass = key > least;
    const uint64_t mask = __ballot(pass);
    if (pass) kept[n + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0))] = key;
    n += __popcll(mask);
  }
  // The largest in order at the front, the others gone.
  __device__ __forceinline__ void order(int lane) {
    wave_fence();
    uint64_t *const sorted = kept + LP_ROOM;
#pragma nounroll
    for (int from = 0; from < n; from += 64) {
      const uint64_t key = from + lane < n ? kept[from + lane] : 0;
      int place = 0;
#pragma unroll 4
      for (int i = 0; i < n; ++i) place += kept[i] > key;
      if (key != 0 && place < top) sorted[place] = key;
    }
    n = n < top ? n : top;
    wave_fence();
    const uint64_t key = lane < n ? sorted[lane] : 0;
    if (lane < LP_TOP) kept[lane] = key;  // and none behind them
    wave_fence();
    if (n == top) raise(kept[top - 1]);
  }
};

// A lane's share of m, S, D and the count, and another one in.
struct LpSums {
  float m, s, d;
  int32_t above;
  // Everything in line with the maximum `to`; c: log2(e) / T.
  __device__ __forceinline__ void line(float to, float c) {
    const float from = to == -INFINITY ? 0.f : to;  // of -inf alone every exponential is 0, none is of inf - inf
    const float off = fmaxf(m - from, -3e38f), f = __builtin_amdgcn_exp2f((m - from) * c);
    s *= f;
    d = __builtin_fmaf(off, s, d * f);  // off is as low as -3e38 where f is 0
    m = to;
  }
  __device__ __forceinline__ void add(float m2, float s2, float d2, int32_t above2, float c) {
    LpSums other{m2, s2, d2, above2};
    const float to = fmaxf(m, m2);
    line(to, c), other.line(to, c);
    s += other.s, d += other.d, above += above2;
  }
};

struct LpShared {
  uint64_t keys[LP_WAVES][LP_ROOM + LP_TOP];
  float sums[LP_WAVES][4];
};

// The lanes' sums and the wavefronts' lists to one record, or to the row's results.
template <int TY, bool RESULTS>
__device__ __forceinline__ void finish(const LogProbsArgs &a, LpShared &lds, LpSums sums, LpList<TY> &list, float mine, int64_t row,
                                       int64_t record) {
  const int lane = threadIdx.x & 63, wave = wave_id();
  const float temp = a.temps == nullptr ? 1.f : a.temps[row], c = exponent_factor(temp);
  sums.line(wave_max(sums.m), c);
  const float s = wave_sum(sums.s), d = wave_sum(sums.d);
  const int32_t above = wave_sum(sums.above);
  if (lane == 0) *reinterpret_cast<float4 *>(lds.sums[wave]) = make_float4(sums.m, s, d, __int_as_float(above));
  if (a.top > 0) list.order(lane);
  __syncthreads();
  LpSums all{-INFINITY, 0.f, 0.f, 0};
#pragma unroll
  for (int w = 0; w < LP_WAVES; ++w) {
    const float4 v = *reinterpret_cast<const float4 *>(lds.sums[w]);
    all.add(v.x, v.y, v.z, __float_as_int(v.w), c);
  }
  const float log_s = logf(all.s);
  if (threadIdx.x == 0) {
    if constexpr (!RESULTS) {
      a.stats[record] = make_float4(all.m, all.s, all.d, __int_as_float(all.above));
    } else {
      a.entropy[row] = log_s - all.d / (temp * all.s);
      if (a.tokens != nullptr) {
        const int64_t t = a.tokens[row];
        a.token[row] = (mine - all.m) / temp - log_s;
        a.rank[row] = t < 0 || t >= a.vocab ? 0 : (int64_t)all.above + 1;
      }
    }
  }
  if (lane >= a.top) return;
  // A key's place among all wavefronts' lists; those of no logit last, in any order of their own.
  const uint64_t key = lds.keys[wave][lane];
  int place = 0;
#pragma unroll 4
  for (int i = 0; i < a.top; ++i)
#pragma unroll
    for (int w = 0; w < LP_WAVES; ++w) {
      const uint64_t other = lds.keys[w][i];
      place += other > key || (other == key && (w < wave || (w == wave && i < lane)));
    }
  if (place >= a.top) return;
  if constexpr (!RESULTS) {
    a.keys[record * a.top + place] = key;
  } else {
    a.top_ids[row * a.top + place] = (int64_t)(uint32_t)~(uint32_t)key;
    a.top_lp[row * a.top + place] = (logit_of((uint32_t)(key >> 32)) - all.m) / temp - log_s;
  }
}

// Part blockIdx.x of row blockIdx.y, tiles of IT chunks of 8 logits a thread.
template <int TY, int IT, bool RESULTS>
__global__ __launch_bounds__(LP_THREADS, 4) void log_probs_part_kernel(const LogProbsArgs a) {
  __shared__ LpShared lds;
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int64_t row = a.first_row + blockIdx.y;
  const RowView<TY> view(a.logits + row * a.row_bytes, a.vocab);
  const uint32_t first = blockIdx.x * (uint32_t)a.tiles * (IT * LP_THREADS);
  Chunk<TY> next[IT];
#pragma unroll
  for (int it = 0; it < IT; ++it) next[it] = view.chunk(first + it * LP_THREADS + threadIdx.x);
  const float mine = token_logit<TY>(a, row);
  const float c = a.temps == nullptr ? 1.44269504f : exponent_factor(a.temps[row]);
  LpSums sums{-INFINITY, 0.f, 0.f, 0};
  LpList<TY> list;
  list.start(lds.keys[wave], a.top);
  int32_t above = 0;  // of the wavefront
#pragma nounroll
  for (int32_t t = 0; t < a.tiles; ++t) {
    const uint32_t g0 = first + t * (IT * LP_THREADS);
    if ((uint64_t)g0 * 8 >= (uint64_t)view.skip + view.vocab) break;  // behind the row
    Chunk<TY> x[IT];
#pragma unroll
    for (int it = 0; it < IT; ++it) x[it] = next[it];
    if (t + 1 < a.tiles) {
#pragma unroll
      for (int it = 0; it < IT; ++it) next[it] = view.chunk(g0 + (IT + it) * LP_THREADS + threadIdx.x);
    }
    if (view.edge(g0, IT * LP_THREADS)) {
#pragma unroll
      for (int it = 0; it < IT; ++it) view.trim(x[it], g0 + it * LP_THREADS + threadIdx.x);
    }
    float m = -INFINITY, chunk[IT];
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      chunk[it] = x[it].at(0);
#pragma unroll
      for (int j = 1; j < 8; ++j) chunk[it] = fmaxf(chunk[it], x[it].at(j));
      m = fmaxf(m, chunk[it]);
    }
    if (__ballot(m > sums.m) != 0) sums.line(fmaxf(m, sums.m), c);
    const float from = sums.m == -INFINITY ? 0.f : sums.m;
    float s[2] = {sums.s, 0.f}, d[2] = {sums.d, 0.f};
#pragma unroll
    for (int it = 0; it < IT; ++it) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float v = x[it].at(j), off = v - from;
        const float e = __builtin_amdgcn_exp2f(off * c);
        s[j & 1] += e;
        d[j & 1] = __builtin_fmaf(fmaxf(off, -3e38f), e, d[j & 1]);  // -inf stands for 0 here
      }
    }
    sums.s = s[0] + s[1], sums.d = d[0] + d[1];
    if (__ballot(m > mine) != 0) {  // without a token it is NaN
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        x[it].forget();
#pragma unroll
        for (int j = 0; j < 8; ++j) above += __popcll(__ballot(x[it].at(j) > mine));
      }
    }
    // All columns kept lie before this tile's: an equal logit comes behind them.
    const bool none = sums.s != sums.s;  // there may be NaNs, which no maximum shows
    const uint64_t passed = a.top == 0 ? 0 : __ballot(!(m <= list.least_logit) || none);
    if (passed == 0) continue;
    // Columns are worked out anew where they are asked for: kept, they would take 32 registers.
    auto column = [&](int it) {
      uint32_t col = 8 * (g0 + it * LP_THREADS + threadIdx.x) - view.skip;
      asm volatile("" : "+v"(col));
      return col;
    };
    auto key_at = [&](int it, int j, uint32_t col) {
      return col + j < view.vocab ? logit_key(x[it].at(j), col + j) : 0;
    };
    if (__popcll(passed) > 16) {  // each lane that passes adds a key or more: worth a bound
      list.bound(logit_order(m), [&](uint32_t order) {  // rare: from memory again, or it takes 60 registers
        uint32_t low = 0;
#pragma nounroll
        for (int it = 0; it < IT; ++it) {
          const Chunk<TY> again = view.chunk(g0 + it * LP_THREADS + threadIdx.x);
          const uint32_t col = column(it);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (col + j < view.vocab && logit_order(again.at(j)) == order && ~(col + j) > low) low = ~(col + j);
        }
        return low;
      });
    }
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      if (__ballot(!(chunk[it] < list.least_logit) || none) == 0) continue;
      x[it].forget();
      const uint32_t col = column(it);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (__ballot(!(x[it].at(j) < list.least_logit)) != 0) list.add(key_at(it, j, col));
      if (list.n > LP_KEPT) list.order(lane);
    }
    if (list.least == 0 || list.n > 2 * a.top) list.order(lane);
  }
  sums.above = lane == 0 ? above : 0;
  finish<TY, RESULTS>(a, lds, sums, list, mine, row, (int64_t)blockIdx.y * a.parts + blockIdx.x);
}

// The records of row blockIdx.x. Of one row of 75 parts with lists of 20: 9.8 us (the parts take 12), loads that follow
// one another (token, its logit, records, then keys) and every key's way through the bound and the order.
template <int TY>
__global__ __launch_bounds__(LP_THREADS) void log_probs_join_kernel(const LogProbsArgs a) {
  __shared__ LpShared lds;
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int64_t row = a.first_row + blockIdx.x, record = (int64_t)blockIdx.x * a.parts;
  const float mine = threadIdx.x == 0 ? token_logit<TY>(a, row) : 0.f;
  const float c = a.temps == nullptr ? 1.44269504f : exponent_factor(a.temps[row]);
  LpSums sums{-INFINITY, 0.f, 0.f, 0};
  LpList<TY> list;
  list.start(lds.keys[wave], a.top);
  for (int32_t r = threadIdx.x; r < a.parts; r += LP_THREADS) {
    const float4 v = a.stats[record + r];
    sums.add(v.x, v.y, v.z, __float_as_int(v.w), c);
  }
  const int32_t total = a.parts * a.top;
#pragma nounroll
  for (int32_t at = 0; at < total; at += 8 * LP_THREADS) {
    uint64_t key[8], largest = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int32_t i = at + j * LP_THREADS + (int32_t)threadIdx.x;
      key[j] = i < total ? a.keys[record * a.top + i] : 0;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) largest = key[j] > largest ? key[j] : largest;
    list.bound((uint32_t)(largest >> 32), [&](uint32_t) { return (uint32_t)largest; });
#pragma unroll
    for (int j = 0; j < 8; ++j) list.add(key[j]);
    if (list.n > LP_KEPT) list.order(lane);
  }
  finish<TY, true>(a, lds, sums, list, mine, row, 0);
}

// How a call is cut: rows for 4 workgroups a CU are a part each, fewer are cut into parts for as many,
// of whole tiles: with parts for 6 or 8 a CU, 1024 rows of 151936 bf16 logits take 100 or 156 us instead of
// 84, with tiles twice as long 84. Where there are fewer tiles than that, they are halved (one such row: 75
// parts of 2048 logits).
struct LpCut {
  int64_t parts;
  int32_t tiles;
  bool small;
  LpCut(int64_t rows, int64_t vocab) {
    const int64_t n = vocab + 7;  // rows may start inside a granule
    const int64_t most = rows >= LP_GROUPS ? 1 : (LP_GROUPS + rows - 1) / rows;
    small = (n + LP_WIDE - 1) / LP_WIDE < most;
    const int64_t tile = small ? LP_SMALL : LP_WIDE, all = (n + tile - 1) / tile;
    tiles = (int32_t)((all + most - 1) / most);
    parts = (all + tiles - 1) / tiles;
  }
};

// Rows of one launch.
constexpr int64_t LP_ROWS = 32768;

static size_t lp_bytes(int64_t records, int64_t top) { return (size_t)records * (16 + 8 * (size_t)top); }

template <int TY>
static int run_log_probs(LogProbsArgs a, int64_t rows, char *ws, hipStream_t stream) {
  constexpr int IT = LP_WIDE / LP_SMALL;
  const LpCut cut(rows, a.vocab);
  a.parts = (int32_t)cut.parts, a.tiles = cut.tiles;
  a.stats = (float4 *)ws;
  a.keys = (uint64_t *)(a.stats + rows * cut.parts);
  for (int64_t first = 0; first < rows; first += LP_ROWS) {
    a.first_row = first;
    const dim3 grid((unsigned)cut.parts, (unsigned)(rows - first < LP_ROWS ? rows - first : LP_ROWS));
    if (cut.parts == 1) {
      if (cut.small)
        log_probs_part_kernel<TY, 1, true><<<grid, LP_THREADS, 0, stream>>>(a);
      else
        log_probs_part_kernel<TY, IT, true><<<grid, LP_THREADS, 0, stream>>>(a);
    } else {
      if (cut.small)
        log_probs_part_kernel<TY, 1, false><<<grid, LP_THREADS, 0, stream>>>(a);
      else
        log_probs_part_kernel<TY, IT, false><<<grid, LP_THREADS, 0, stream>>>(a);
      FM_CHECK_HIP(hipGetLastError());
      log_probs_join_kernel<TY><<<dim3(grid.y), LP_THREADS, 0, stream>>>(a);
    }
    FM_CHECK_HIP(hipGetLastError());
  }
  return FM_OK;
}

}  // namespace fm

using namespace fm;

extern "C" size_t fm_log_probs_workspace_bytes(int64_t rows, int64_t vocab, int32_t top) {
  if (rows <= 0 || vocab <= 0 || vocab > INT32_MAX || top < 0 || top > LP_TOP) return 0;
  const LpCut cut(rows, vocab);
  return cut.parts == 1 ? 16 : lp_bytes(rows * cut.parts, top);
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
