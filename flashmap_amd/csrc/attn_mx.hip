// Non-causal attention over a paged context in microscaled 4 bits (mx_device.h):
//
//   s_ij = scale q_i . k_j,  p_ij = exp(s_ij - m_i),  o_i = sum_j p_ij v_j / sum_j p_ij
//
// A cache row (block, head, position in the page) holds D key codes and D value codes, D bytes, and
// apart from them 2 D / 32 scale bytes: 17/64 of a bf16 row.
//
// A unit is (sequence, KV head, up to 16 RB query rows). Its positions are taken 128 a step, 32 by
// each of a workgroup's four wavefronts, and all units' steps form one line that is cut into
// equal shares, one per workgroup: a unit cut by a share's end leaves partial sums that
// attn_mx_join_kernel puts together. A wavefront needs nobody between the ends of a unit: it
// streams its own cache rows into its own ring in LDS (loads straight into LDS, NS tiles deep,
// across the ends of units), and keeps all 16 RB rows, so that a value is widened to bf16 once
// for all of them.
//
// Scores: K on the block-scaled matrix instruction as it is stored, against the query as a sum of
// two e4m3 operands, hi = e4m3(q / 2^e) and lo = e4m3((q - hi 2^e) / 2^(e - 5)): 4 + 4 significant
// bits (2^e puts a block's largest magnitude to [128, 256); a value below 2^-13 of that loses at most 2^-22
// of it). The query is scaled by log2(e) softmax_scale in float32, behind its norm and rotation where
// they go with the call, and rounded only there, by at most 2^-8: as many bits as bf16 has. K needs no
// conversion and no register but the 16 bytes a
// lane that it comes in. S^T = K Q^T leaves a query row's scores in the lanes that take that row's
// probabilities in O^T = V^T P^T: nothing crosses lanes.
// Values: each lane widens 8 tokens' dwords (8 channels each) with their block's scale, exactly, to
// bf16 pairs, and pairs of tokens by byte permutes. Probabilities are rounded to bf16 (2^-8 of each at
// most, as the bf16 attention does) and summed as they were rounded; maxima, sums and outputs are float32.
// A row's maximum is a reference that moves only when a score passes it by 2^8: the sums stay far
// inside float32 and bf16 keeps its 8 bits wherever its exponent is. A tile's scores start from less
// their rows' references, so that a probability is one exponential, and one test of the tile's
// exponents finds those that passed.
//
// What bounds it: with 16 rows a head the cache's bytes (8 contexts of 131072 positions, 16 query rows on
// each of 8 heads: 221 us, 5.2 TB/s, what a copy reaches); with 64 rows a head matrix and vector instructions
// and the loads take nearly equal times that overlap only in part (the same contexts 320 us: 238 for the loads
// alone, 267 for the instructions alone), and a unit's end, four wavefronts' sums of 64 rows, some microseconds
// a share (8 contexts of 32768 positions: 98 us). Row blocks of a unit share its loads and the widening of its
// values, so a unit takes up to four: as two units of two, the second reads everything again (419 us).
// One or two keep the queries' operands in registers and leave LDS for three workgroups a CU (mx_resident), three
// or four keep them in LDS, with a tile more in each ring. Four of 128 channels take all 256 registers: 29 that
// are not used among the tiles are spilled and come back between units.
// Nothing among the tiles may be loaded through registers: a wait for it would wait for the whole
// ring (8 contexts of 32768 positions: 8 % more with one such wait).
#include <math.h>

#include <type_traits>

#include "fm_host.h"
#include "mx_device.h"
#include "wave_device.h"

namespace fm {

constexpr int MXA_WAVES = 4;
constexpr int MXA_TILE = 32;                     // positions of a wavefront's tile
constexpr int MXA_STEP = MXA_WAVES * MXA_TILE;   // of a workgroup's step
constexpr int MXA_BATCH = 256;                   // sequences of one launch: their steps lie in LDS
constexpr int MXA_GROUPS = 1024;                 // row groups of one launch: their parts lie in the workspace
constexpr int MXA_UNIT_COST = 6;                 // steps that a unit's start and end cost
constexpr float MXA_SLACK = 8.f;                 // log2 that scores may pass their row's reference by

struct MxAttnArgs {
  const uint16_t *q;
  int64_t q_st, q_sh;  // token and head strides, elements
  uint16_t *o;
  int64_t o_st, o_sh;
  const int32_t *cu_q;  // NULL: sequence b's tokens start at token0 + b q_len
  int64_t token0, q_tokens;  // q_tokens: rows of q and out; what cu_q says past them is left alone
  int32_t q_len, group, hkv;
  int32_t rgroup0, rgroups;  // row groups of this launch: the first and how many
  uint32_t q_mul, q_shift;  // n / q_len, as n / page below
  const uint8_t *codes, *scales;
  uint32_t cs16, ss4;  // row strides in 16 and in 4 bytes (the last row's offsets in them below 2^32)
  uint32_t num_blocks, page, head_rows;  // head_rows: rows of a block, hkv page
  uint32_t page_mul, page_shift;  // n / page = mulhi(2 n, page_mul) >> page_shift for n < 2^31
  const int32_t *table;
  int64_t table_stride;
  int32_t table_width;
  const int32_t *lens;
  int32_t batch, max_len;  // max_len: positions that the table and the caller's bound allow
  float scale_log2;
  const float *qn_w;  // non-NULL: the queries' norm and rotation
  Rope rope;
  const int64_t *q_pos;
  float eps;
  float *part_o;   // (2 shares, 16 RB, D), relative to the row's reference
  float *part_ml;  // (2 shares, 16 RB, 2): the reference (log2) and the sum
  int32_t shares;  // of a row group
  double per_share;  // 1 / shares
};

// Workgroups a CU, as registers and LDS allow. Two row blocks of 128 channels need more registers than three
// workgroups leave (43 would be spilled): 64 requests of 256 to 8192 positions, 32 query rows on each of 8 heads, 90 us
// with two, 114 with three. One row block (256 requests of 16 to 512 positions, 16 rows: 60 with two, 55 with
// three) and 64 channels (32 rows of the 64 requests: 60 and 55) gain from the third.
constexpr int mx_resident(int d, int rb) { return rb == 1 || (rb == 2 && d == 64) ? 3 : 2; }

template <int D, int RB>
struct MxGeo {
  static constexpr int NF = D / 16;                       // 16-channel fragments
  static constexpr int CODES = MXA_TILE * D, SCALES = MXA_TILE * (D / 16);
  static constexpr int DMAS = CODES / 1024;               // 16-byte loads a lane of a tile's codes
  static constexpr int LOADS = DMAS + 2;                  // and its scales, and later page ids
  static constexpr int SLOT = CODES + SCALES + 4 * MXA_TILE;
  static constexpr int RESIDENT = mx_resident(D, RB);
  static constexpr int NS = RB <= 2 ? 2 : 3;              // tiles in a wavefront's ring
  static constexpr int RING = MXA_WAVES * NS * SLOT;
  static constexpr int QN = D == 128 ? 4 : 2;             // 16-byte operands a lane of a row block's queries
  static constexpr int QOP = QN * 1024 + 128;             // and the bytes of their two scales
  static constexpr int MF = RB <= 2 ? 2 : 4;              // fragments that are joined at a time
  static constexpr int MERGE = MXA_WAVES * MF * 1024;
  static constexpr int SHARED = RB * QOP > MERGE ? RB * QOP : MERGE;  // one after the other
  static constexpr int ML = MXA_WAVES * RB * 16 * 8;
  static constexpr int LINE = 4 * (MXA_BATCH + 4) * 4;    // the sequences (MxLine)
  static constexpr int SMEM = RING + SHARED + ML + LINE + 4 * D;
  static_assert(SMEM <= 160 * 1024 / RESIDENT, "LDS");
};

// ------------------------------------------------------------------------------ pieces

typedef __attribute__((address_space(3))) char lds_char_t;
// Loads straight into LDS, lane l's bytes at lds + 16 l (4 l). Inline asm, so that the compiler
// does not wait for the loads in flight before every LDS read; the waits are counted by hand.
__device__ __forceinline__ void ring_load16(const uint8_t *p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds), "v"(p) : "memory", "m0");
}
__device__ __forceinline__ void ring_load4(const void *p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(lds), "v"(p) : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void ring_wait() {
  static_assert(N >= 0 && N < 64, "vmcnt holds 6 bits");
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}
// Every LDS read issued so far has its data: what lies there may be loaded over.
__device__ __forceinline__ void ring_read_done() { asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory"); }
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ int32_t context_len(const MxAttnArgs &a, int b) {
  const int32_t n = a.lens[b];
  return n < 0 ? 0 : n < a.max_len ? n : a.max_len;
}
__device__ __forceinline__ int32_t steps_of(int32_t len) { return (len + MXA_STEP - 1) / MXA_STEP; }
// Query tokens [first, stop) of the caller's rows: the first and how many the call takes.
__device__ __forceinline__ int32_t tokens_in(const MxAttnArgs &a, int64_t first, int64_t stop) {
  const int64_t n = (stop < a.q_tokens ? stop : a.q_tokens) - first;
  return n < 0 || first < 0 ? 0 : n < a.q_len ? (int32_t)n : a.q_len;
}
__device__ __forceinline__ int32_t divided(int32_t n, uint32_t mul, uint32_t shift) {  // n < 2^31
  return (int32_t)(__umulhi((uint32_t)n << 1, mul) >> shift);
}

// floor(a / b) for 0 <= a < 2^50, b > 0 and a quotient below 2^24.
__device__ __forceinline__ int32_t quotient(int64_t a, int64_t b) {
  int32_t q = (int32_t)((float)a * __builtin_amdgcn_rcpf((float)b));
  while ((int64_t)q * b > a) --q;
  while ((int64_t)(q + 1) * b <= a) ++q;
  return q;
}

// The line of a row group's steps, all heads of all sequences, cut into n shares by cost: a unit counts
// its steps and, in front of them, c more for its start and end (0 where shares are a few steps). Of
// 64 requests of 256 to 8192 positions the shares that hold the short ones would otherwise take
// twice the others' time. With fewer steps than shares each is one.
struct MxPlan {
  int64_t total, each;  // share s starts at s total / n = s each + s over / n
  int32_t n, c, over;
  bool few;
  __device__ __forceinline__ MxPlan(const MxAttnArgs &a, int32_t steps, int32_t sequences) {
    const int64_t all = (int64_t)a.hkv * steps;
    few = all < a.shares;
    n = few ? (int32_t)all : a.shares;
    const int64_t fair = few ? 0 : (int64_t)((double)all * a.per_share) >> 2;
    c = fair < MXA_UNIT_COST ? (int32_t)fair : MXA_UNIT_COST;
    total = all + (int64_t)a.hkv * c * sequences;
    each = (int64_t)((double)total * a.per_share);  // within 1: total is below 2^46
    while (each * a.shares > total) --each;
    while ((each + 1) * a.shares <= total) ++each;
    over = (int32_t)(total - each * a.shares);
  }
  __device__ __forceinline__ int64_t share(int32_t s) const { return few ? s : s * each + quotient(s * over, n); }
  // The share that `at` lies in: the last that starts there or before.
  __device__ __forceinline__ int32_t share_of(int64_t at) const {
    if (few) return (int32_t)at;
    int32_t w = (int32_t)((float)at * (float)n * __builtin_amdgcn_rcpf((float)total));
    while (share(w) > at) --w;
    while (share(w + 1) <= at) ++w;
    return w;
  }
};

// A place on the line: step lt of unit (b, h).
struct MxCursor {
  int b, h, lt, steps, len;
};

// In LDS, by sequence: the steps, and the sequences with steps, before it; its length; its first token.
struct MxLine {
  int32_t *pre, *some, *len, *cu;
  __device__ __forceinline__ void load(MxCursor &c) const {
    c.len = uniform(len[c.b]);
    c.steps = steps_of(c.len);
  }
};

__device__ __forceinline__ void advance(const MxAttnArgs &a, const MxLine &line, MxCursor &c) {
  if (++c.lt < c.steps) return;
  c.lt = 0;
  if (++c.h < a.hkv) return;
  c.h = 0;
  for (++c.b; c.b < a.batch; ++c.b) {  // sequences without context have no units
    line.load(c);
    if (c.steps > 0) break;
  }
}

// The step at which `at` of the cost line lies, and its number; the sequences are tested 64 at a time.
__device__ __forceinline__ int64_t locate(const MxAttnArgs &a, const MxPlan &plan, const MxLine &line, int64_t at,
                                          MxCursor &c) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const int b = b0 + lane < a.batch ? b0 + lane : 0;
    before += __popcll(__ballot(b0 + lane < a.batch && (int64_t)a.hkv * (line.pre[b] + plan.c * line.some[b]) <= at));
  }
  c.b = uniform(before - 1);  // the last that starts there or before: those without steps start where the next does
  line.load(c);
  const int32_t pre = uniform(line.pre[c.b]);
  const int64_t off = at - (int64_t)a.hkv * (pre + plan.c * uniform(line.some[c.b]));
  c.h = uniform(quotient(off, c.steps + plan.c));
  const int in = (int)(off - (int64_t)c.h * (c.steps + plan.c)) - plan.c;
  c.lt = in > 0 ? in : 0;
  return (int64_t)a.hkv * pre + (int64_t)c.h * c.steps + c.lt;
}

// LDS place of the 16-byte piece c of tile row r: rows of 128 bytes (D 128) or 64. Operand
// reads take 16 rows at once, value reads one dword of four rows: both then fall on all banks.
template <int D>
__device__ __forceinline__ int place(int r, int c) {
  return D == 128 ? 128 * r + 16 * (c ^ (r >> 1 & 7)) : 64 * r + 16 * (c ^ (r >> 2 & 3));
}
// The tile row of operand row m of a 16-position block: the four lane groups' rows of one value
// read are then neighbours and 8 apart.
__device__ __forceinline__ int row_of(int m) { return (m >> 2 & 1) + 8 * (m >> 3) + 2 * (m & 3); }

// D(16x16 f32) += A(16x128 e2m1) B(128x16 e4m3), a scale byte for each lane's 32 values.
__device__ __forceinline__ f32x4_t mfma_k_q(u32x4_t k, u32x4_t q0, u32x4_t q1, f32x4_t c, int sk, int sq) {
  const i32x8_t a = {(int)k[0], (int)k[1], (int)k[2], (int)k[3], 0, 0, 0, 0};
  const i32x8_t b = {(int)q0[0], (int)q0[1], (int)q0[2], (int)q0[3], (int)q1[0], (int)q1[1], (int)q1[2], (int)q1[3]};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 0, 0, sk, 0, sq);
}

__device__ __forceinline__ uint32_t lo_byte(uint32_t byte) { return byte == 255u ? 255u : byte - 5; }

// load_rope_ops for tables whose pairs lie side by side, or interleaved (the entry refuses others: their
// addresses alone would take half the registers).
template <int D>
__device__ __forceinline__ void load_rope(PrologueOps<D> &ops, const Rope &rope, int64_t row, int g) {
  const float *cs = rope.cos + row * rope.row_stride;
  const bool apart = rope.pair_stride == 1;
  const float *second = apart ? rope.sin + row * rope.row_stride : cs + 4;
#pragma unroll
  for (int t = 0; t < D / 32; ++t) {
    const int at = apart ? 16 * t + 4 * g : 32 * t + 8 * g;
    const f32x4u_t v = *(g_f32x4u_t *)(cs + at), w = *(g_f32x4u_t *)(second + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) ops.c[t][i] = v[i], ops.s[t][i] = w[i];
  }
}
// As they were loaded: pairs apart, or two (cos, sin) in ops.c and two in ops.s.
template <int D>
__device__ __forceinline__ void sort_rope(PrologueOps<D> &ops, const Rope &rope) {
  if (rope.pair_stride == 1) return;
#pragma unroll
  for (int t = 0; t < D / 32; ++t) {
    const float c1 = ops.c[t][2], s0 = ops.c[t][1], s1 = ops.c[t][3], c2 = ops.s[t][0], c3 = ops.s[t][2], s2 = ops.s[t][1];
    ops.c[t][1] = c1, ops.c[t][2] = c2, ops.c[t][3] = c3;
    ops.s[t][0] = s0, ops.s[t][1] = s1, ops.s[t][2] = s2;
  }
}

// The writer's norm and rotation (kv_write_mx.hip) where the result is rounded to 8 bits, not 2: sums in float32 as
// they come, the root's reciprocal by its instruction (1 ulp), products fused.
template <int D>
__device__ __forceinline__ void norm_rope_query(const u32x4_t (&x)[D / 32], const PrologueOps<D> &ops, float eps,
                                                float (&y)[D / 32][8]) {
  float ss = 0.f;
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      y[t][2 * q] = bf16_lo(x[t][q]), y[t][2 * q + 1] = bf16_hi(x[t][q]);
      ss += y[t][2 * q] * y[t][2 * q] + y[t][2 * q + 1] * y[t][2 * q + 1];
    }
  ss = sum_over_groups(ss);
  const float r = __builtin_amdgcn_rsqf(ss * (1.f / D) + eps);
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float e = y[t][2 * q] * r * ops.w[t][2 * q], o = y[t][2 * q + 1] * r * ops.w[t][2 * q + 1];
      y[t][2 * q] = e * ops.c[t][q] - o * ops.s[t][q];
      y[t][2 * q + 1] = o * ops.c[t][q] + e * ops.s[t][q];
    }
}

// Eight of a block's 32 values in each of a row's four lanes, as two e4m3 operands and the scale byte
// of the first.
__device__ __forceinline__ void split_query(const float (&x)[8], u32x2_t &hi, u32x2_t &lo, uint32_t &byte) {
  typedef __attribute__((ext_vector_type(2))) short s16x2_t;
  typedef __attribute__((ext_vector_type(2))) float f32x2_t;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, magnitude(x[i]));
  auto p = __builtin_amdgcn_permlane16_swap(top, top, false, false);
  top = max(p[0], p[1]);
  p = __builtin_amdgcn_permlane32_swap(top, top, false, false);
  top = max(p[0], p[1]) >> 23;
  // At least 6, so that lo's scale is a byte too; 255 (an infinity or a NaN) makes the scores NaN.
  byte = top == 255 ? 255u : top < 13 ? 6u : top - 7;
  const float sh = mx_scale_value(byte), sl = mx_scale_value(lo_byte(byte));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float *v = x + 4 * i;
    s16x2_t h = {0, 0}, l = {0, 0};
    h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(h, v[0], v[1], sh, false);
    h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(h, v[2], v[3], sh, true);
    const uint32_t hw = __builtin_bit_cast(uint32_t, h);
    const f32x2_t b0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hw, sh, false);
    const f32x2_t b1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hw, sh, true);
    l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l, v[0] - b0[0], v[1] - b0[1], sl, false);
    l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l, v[2] - b1[0], v[3] - b1[1], sl, true);
    hi[i] = hw;
    lo[i] = __builtin_bit_cast(uint32_t, l);
  }
}

// Two value codes (byte SEL of w) times the scale, as bf16.
template <int SEL>
__device__ __forceinline__ uint32_t widen(uint32_t w, float scale) {
  const bf16x2_t v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL);
  return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ uint32_t both_lo(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t both_hi(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// sum + both bf16 values of p (v_dot2_f32_bf16 with ones).
__device__ __forceinline__ float add_both(uint32_t p, float sum) {
  typedef __attribute__((ext_vector_type(2))) __bf16 b2_t;
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2_t, p), __builtin_bit_cast(b2_t, 0x3f803f80u), sum, false);
}

// The float of a scale byte, of which the widening takes the exponent (0: 2^-127; 255: NaN).
__device__ __forceinline__ float mx_scale_float(uint32_t byte) { return __uint_as_float(byte << 23); }

// The sum over the lanes up to this one.
template <int CTRL, int ROWS>
__device__ __forceinline__ int32_t shifted(int32_t v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int32_t wave_prefix(int32_t v) {
  v += shifted<0x111, 0xf>(v);  // from the lane 1, 2, 4 and 8 before, in rows of 16
  v += shifted<0x112, 0xf>(v);
  v += shifted<0x114, 0xf>(v);
  v += shifted<0x118, 0xf>(v);
  v += shifted<0x142, 0xa>(v);  // the row before's last, into rows 1 and 3
  v += shifted<0x143, 0xc>(v);  // lane 31, into rows 2 and 3
  return v;
}

// The workgroup's LDS writes are everybody's; loads in flight go on.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory"); }

// The oldest tile in flight is there, `behind` younger ones (MOST at most) with LOADS loads each are not waited for.
template <int LOADS, int MOST>
__device__ __forceinline__ void wait_tiles(int32_t behind) {
  if constexpr (MOST == 0)
    ring_wait<0>();
  else if (behind >= MOST)
    ring_wait<LOADS * MOST>();
  else
    wait_tiles<LOADS, MOST - 1>(behind);
}

// --------------------------------------------------------------------------- the kernel

template <int D, int RB>
__global__ __launch_bounds__(64 * MXA_WAVES, (MxGeo<D, RB>::RESIDENT)) void attn_mx_kernel(const MxAttnArgs a) {
  using G = MxGeo<D, RB>;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int n = lane & 15, g = lane >> 4;
  char *const ring = lds + wave * G::NS * G::SLOT;
  const uint32_t ring_at = (uint32_t)(uintptr_t)(lds_char_t *)ring;
  char *const shared = lds + G::RING, *const qop = shared;
  float *const ml = reinterpret_cast<float *>(shared + G::SHARED);
  int32_t *const first = reinterpret_cast<int32_t *>(shared + G::SHARED + G::ML);
  const MxLine line{first, first + (MXA_BATCH + 4), first + 2 * (MXA_BATCH + 4), first + 3 * (MXA_BATCH + 4)};
  float *const qn_w = reinterpret_cast<float *>(first + 4 * (MXA_BATCH + 4));

  // The steps before each sequence, and the sequences with steps, by every wavefront for itself (all
  // write the same): a prefix sum of 64 sequences at a time.
  int32_t steps_all = 0, some_all = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const int b = b0 + lane;
    const int32_t l = b < a.batch ? context_len(a, b) : 0, s = steps_of(l);
    if (a.cu_q != nullptr && b < a.batch) line.cu[b] = a.cu_q[b];
    const int32_t sum = wave_prefix(s) + steps_all;
    const uint64_t has = __ballot(s > 0);
    line.len[b] = l;
    line.pre[b] = sum - s;
    line.some[b] = some_all + __popcll(has & ((1ull << lane) - 1));
    steps_all = __builtin_amdgcn_readlane(sum, 63);
    some_all += __popcll(has);
  }
  if (a.cu_q != nullptr) line.cu[a.batch] = a.cu_q[a.batch];
  if (a.qn_w != nullptr && threadIdx.x < D) qn_w[threadIdx.x] = a.qn_w[threadIdx.x];
  wave_fence();
  const MxPlan plan(a, steps_all, some_all);
  // Neighbouring shares, and a share's row groups, on one XCD (workgroups go to the 8 XCDs in turn, and
  // the grid's x is a multiple of 8): they read the same cache rows, the row groups at the same time.
  const int32_t rg = blockIdx.y, share = (int32_t)((blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3));
  if (share >= plan.n) return;
  MxCursor cc, ci;
  const int64_t end = share + 1 < plan.n ? locate(a, plan, line, plan.share(share + 1), ci) : (int64_t)a.hkv * steps_all;
  const int32_t count = uniform((int)(end - locate(a, plan, line, plan.share(share), cc)));
  if (count == 0) return;  // a part of a unit's start alone

  // ---- the queries: a wavefront holds the 16 rows of its row block on their way from memory
  const int32_t rows = a.group * a.q_len;  // of a sequence's KV head
  auto row_token = [&](const MxCursor &c, int rb, int32_t &head) {  // of this lane's row of a row block; -1: none
    int64_t from = a.token0 + (int64_t)c.b * a.q_len;
    int32_t tokens = a.q_len;
    if (a.cu_q != nullptr) {
      from = uniform(line.cu[c.b]);
      tokens = tokens_in(a, from, uniform(line.cu[c.b + 1]));
    }
    const int32_t r = ((a.rgroup0 + rg) * RB + rb) * 16 + n;
    head = divided(r, a.q_mul, a.q_shift);
    const int32_t tok = r - head * a.q_len;
    return r < rows && tok < tokens ? from + tok : -1;
  };
  u32x4_t qx[D / 32];
  PrologueOps<D> ops;
  int32_t rope_row = 0;
  auto fetch_position = [&](const MxCursor &c) {
    if (a.qn_w == nullptr || wave >= RB) return;
    int32_t head;
    const int64_t token = row_token(c, wave, head);
    int64_t pos = token < 0 ? 0 : token;
    if (a.q_pos != nullptr) pos = a.q_pos[pos];
    rope_row = (int32_t)clamp_row(a.rope, pos);
  };
  auto fetch_query = [&](const MxCursor &c) {
    // Whatever the branches below leave out is new here: nothing of the last rows is kept for it.
#pragma unroll
    for (int t = 0; t < D / 32; ++t) {
      qx[t] = u32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < 4; ++i) ops.c[t][i] = ops.s[t][i] = 0.f;
    }
    if (wave >= RB) return;
    int32_t head;
    const int64_t token = row_token(c, wave, head);
    const bool live = token >= 0;
    const uint16_t *src = a.q + (live ? token : 0) * a.q_st + ((int64_t)c.h * a.group + (live ? head : 0)) * a.q_sh + 8 * g;
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
      if (live) qx[t] = load16(src + 32 * t);
    if (a.qn_w != nullptr) load_rope(ops, a.rope, rope_row, g);
  };
  // ---- the ring. A tile's page ids lie in its slot before its rows are asked for: those of tile
  // t + NS travel with the rows of tile t.
  MxCursor cd = ci = cc;
  int32_t ids_left = count;
  auto page_of = [&](const MxCursor &c, uint32_t lane, uint32_t &t) {  // of this lane's position, t, of the tile
    t = c.lt * MXA_STEP + wave * MXA_TILE + (lane & (MXA_TILE - 1));
    t = min(t, (uint32_t)c.len - 1);
    return (uint32_t)divided(t, a.page_mul, a.page_shift);
  };
  auto load_ids = [&](uint32_t to, uint32_t lane) {  // of the tile at ci; past the share's end its last tile's again
    uint32_t t;
    const uint32_t col = page_of(ci, lane, t);
    if (lane < MXA_TILE) ring_load4(a.table + (int64_t)ci.b * a.table_stride + col, to + G::CODES + G::SCALES);
    if (--ids_left > 0) advance(a, line, ci);
  };
  int32_t load_at = 0;  // the slot of the tile at cd
  // Lane constants of both steps are worked out anew for every tile: kept, they would go to scratch
  // memory, whose reloads wait for the whole ring.
  struct Rows {
    uint32_t at16, at4;  // where this lane's position of the tile lies: codes in 16 bytes, scales in 4
  };
  auto find_rows = [&]() {  // of the tile at cd, whose ids lie in its slot
    uint32_t lane = threadIdx.x & 63, t;
    asm volatile("" : "+v"(lane));
    const uint32_t col = page_of(cd, lane, t);
    uint32_t id = *reinterpret_cast<const uint32_t *>(ring + load_at + G::CODES + G::SCALES + 4 * (lane & (MXA_TILE - 1)));
    id = id < a.num_blocks ? id : 0;  // a page that the cache does not have: its first
    const uint32_t row = id * a.head_rows + (cd.h * a.page + (t - __umul24(col, a.page)));
    return Rows{row * a.cs16, row * a.ss4};
  };
  auto load_tile = [&](const Rows &rows) {
    const uint32_t to = ring_at + load_at;
    uint32_t lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    constexpr uint32_t LPR = D / 16;  // lanes of a row
    const uint32_t r = lane / LPR, piece = lane % LPR ^ (D == 128 ? r >> 1 : r >> 2 & 3);  // as place() says
    uint32_t from[G::DMAS], scale_from = rows.at4;
#pragma unroll
    for (int u = 0; u < G::DMAS; ++u)
      from[u] = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * (r + u * (64 / LPR)), (int)rows.at16);
    if constexpr (D == 128) scale_from = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * (lane >> 1), (int)rows.at4);
    ring_read_done();  // all of them, and whoever read this slot's last tile is done
#pragma unroll
    for (int u = 0; u < G::DMAS; ++u) {
      const uint32_t c = D == 128 ? piece ^ (u & 1) << 2 : piece;
      ring_load16(a.codes + 16 * c + ((uint64_t)from[u] << 4), to + 1024 * u);
    }
    if (D == 128 || lane < MXA_TILE)
      ring_load4(a.scales + (D == 128 ? 4 * (lane & 1) : 0) + ((uint64_t)scale_from << 2), to + G::CODES);
    load_ids(to, lane);
    advance(a, line, cd);
    load_at = load_at == (G::NS - 1) * G::SLOT ? 0 : load_at + G::SLOT;
  };
  const int32_t ahead = count < G::NS ? count : G::NS;
  for (int32_t i = 0; i < ahead; ++i) load_ids(ring_at + i * G::SLOT, lane);
  fetch_position(cc);
  ring_wait<0>();
  fetch_query(cc);
  for (int32_t i = 0; i < ahead; ++i) load_tile(find_rows());

  // Where this lane's operands lie in a tile: key row row_of(n) and its scale; value dwords of rows
  // row_of(4 g + i), i the last two bits of what follows, and their scales.
  const uint32_t key_at = place<D>(row_of(n), D == 128 ? g : g & 1);
  const uint32_t key_scale_at = G::CODES + row_of(n) * (D / 16) + (D == 128 ? g : g & 1);
  const uint32_t value_row = (g & 1) + 8 * (g >> 1), value_block = D == 128 ? n >> 2 : n >> 3;
  uint32_t value_at[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    value_at[i] = place<D>(value_row + 2 * i, D / 32 + value_block) + (D == 128 ? 4 * (n & 3) : 2 * (n & 7));
  const uint32_t value_scale_at = G::CODES + value_row * (D / 16) + D / 32 + value_block;

  // ---- the share, unit by unit
  int32_t read_at = 0;  // the slot of the tile to take
  for (int32_t k = 0; k < count;) {
    const int32_t seg = cc.steps - cc.lt < count - k ? cc.steps - cc.lt : count - k;
    const int32_t part = 2 * (rg * a.shares + share) + (k > 0 ? 1 : 0);  // where the unit's sums go if it is not whole
    const bool whole = seg == cc.steps, more = k + seg < count;
    MxCursor next = cc;
    next.lt += seg - 1;
    if (more) advance(a, line, next);

    if (more) fetch_position(next);
    // The unit's queries as operands: a wavefront a row block.
    lds_barrier();  // nobody joins the last unit any more
    // On every path the loads of the query end here, not where the tiles next write their registers.
#pragma unroll
    for (int t = 0; t < D / 32; ++t) {
      asm volatile("" : "+v"(qx[t]));
#pragma unroll
      for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(ops.c[t][i]), "+v"(ops.s[t][i]));
    }
    if (wave < RB) {
      float y[D / 32][8];
      if (a.qn_w != nullptr) {
#pragma unroll
        for (int t = 0; t < D / 32; ++t)
#pragma unroll
          for (int i = 0; i < 8; ++i) ops.w[t][i] = qn_w[32 * t + 8 * g + i];
        sort_rope(ops, a.rope);
        norm_rope_query<D>(qx, ops, a.eps, y);
      } else {
#pragma unroll
        for (int t = 0; t < D / 32; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) y[t][2 * i] = bf16_lo(qx[t][i]), y[t][2 * i + 1] = bf16_hi(qx[t][i]);
      }
      // A row's hi and lo codes, 2 D bytes, then all rows in the operands' order in their place.
      char *const to = qop + wave * G::QOP, *const stage = to + n * 2 * D;
      uint32_t mine = 0;  // the byte of block g
#pragma unroll
      for (int t = 0; t < D / 32; ++t) {
        u32x2_t hi, lo;
        uint32_t byte;
#pragma unroll
        for (int i = 0; i < 8; ++i) y[t][i] *= a.scale_log2;
        split_query(y[t], hi, lo, byte);
        mine = t == (g & (D / 32 - 1)) ? byte : mine;
        *reinterpret_cast<u32x2_t *>(stage + 32 * t + 8 * g) = hi;
        *reinterpret_cast<u32x2_t *>(stage + D + 32 * t + 8 * g) = lo;
      }
      wave_fence();
      // The operand of lane group g: channels 16 g to 16 g + 15 and, in its second half, 64 on; its
      // scale byte that of channels 32 g on. D 64: hi in the first half, lo in the second.
      u32x4_t op[G::QN];
#pragma unroll
      for (int i = 0; i < G::QN; ++i) op[i] = load16(stage + 64 * i + 16 * g);
      wave_fence();
#pragma unroll
      for (int i = 0; i < G::QN; ++i) store16(to + 1024 * i + 16 * lane, op[i]);
      const uint32_t low = lo_byte(mine);
      *reinterpret_cast<uint16_t *>(to + G::QN * 1024 + 2 * lane) =
          (uint16_t)(D == 128 ? mine | low << 8 : g < 2 ? mine : low);
    }
    lds_barrier();
    constexpr bool QR = RB <= 2;  // the queries stay in registers, else in LDS
    u32x4_t qr[QR ? RB : 1][G::QN];
    int qrs[QR ? RB : 1];
    if constexpr (QR) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        qrs[rb] = *reinterpret_cast<const uint16_t *>(qop + rb * G::QOP + G::QN * 1024 + 2 * lane);
#pragma unroll
        for (int i = 0; i < G::QN; ++i) qr[rb][i] = load16(qop + rb * G::QOP + 1024 * i + 16 * lane);
      }
    }
    f32x4_t o[RB][G::NF];
    f32x4_t minus[RB];  // less a row's reference, four times: what its scores' sums start from
    float sum[RB];      // of a row's probabilities in this lane
    bool fresh = true;  // no tile yet
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      minus[rb] = f32x4_t{0.f, 0.f, 0.f, 0.f}, sum[rb] = 0.f;
#pragma unroll
      for (int f = 0; f < G::NF; ++f) o[rb][f] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }

    // The next unit's positions are there before the tiles: a load that the compiler waits for among
    // them would wait for the whole ring every time.
    asm volatile("" : "+v"(rope_row));
    for (int32_t i = 0; i < seg; ++i, ++k) {
      wait_tiles<G::LOADS, G::NS - 1>(count - k - 1);
      const bool again = k + G::NS < count;
      Rows rows{0, 0};
      if (again) rows = find_rows();
      const int32_t live = cc.len - (cc.lt + i) * MXA_STEP - wave * MXA_TILE;  // positions of the tile
      if (live > 0) {
        const char *const slot = ring + read_at;
        u32x4_t kf[2];
        int ks[2];
#pragma unroll
        for (int tb = 0; tb < 2; ++tb) {
          kf[tb] = load16(slot + key_at + 16 * D * tb);
          ks[tb] = *reinterpret_cast<const uint8_t *>(slot + key_scale_at + D * tb);
        }
        // The log2 of row block rb's probabilities: scores less the references. Positions past the context
        // repeat its last one.
        auto scores = [&](int rb, f32x4_t (&s)[2]) {
          u32x4_t q[G::QN];
          int qs;
          if constexpr (QR) {
#pragma unroll
            for (int x = 0; x < G::QN; ++x) q[x] = qr[rb][x];
            qs = qrs[rb];
          } else {
#pragma unroll
            for (int x = 0; x < G::QN; ++x) q[x] = load16(qop + rb * G::QOP + 1024 * x + 16 * lane);
            qs = *reinterpret_cast<const uint16_t *>(qop + rb * G::QOP + G::QN * 1024 + 2 * lane);
          }
#pragma unroll
          for (int tb = 0; tb < 2; ++tb) s[tb] = mfma_k_q(kf[tb], q[0], q[1], minus[rb], ks[tb], qs);
          if constexpr (D == 128) {
#pragma unroll
            for (int tb = 0; tb < 2; ++tb) s[tb] = mfma_k_q(kf[tb], q[2], q[3], s[tb], ks[tb], qs >> 8);
          }
        };
        // References of rows that have none yet or are passed by: the tile's largest score, and what
        // was summed in line with it.
        auto refer = [&]() {
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) {
            f32x4_t s[2];
            scores(rb, s);
            if constexpr (!QR) __builtin_amdgcn_sched_barrier(0);
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; j += 2) top = fmaxf(fmaxf(top, s[j >> 2][j & 3]), s[j >> 2][(j & 3) + 1]);
            top = max_over_groups(top);
            const float by = (fresh ? top > -INFINITY : top >= 1.f) ? top + MXA_SLACK - 1.f : 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) minus[rb][i] -= by;
            if (!fresh) {
              const float f = __builtin_amdgcn_exp2f(-by);
              sum[rb] *= f;
#pragma unroll
              for (int c = 0; c < G::NF; ++c) o[rb][c] *= f;
            }
          }
          fresh = false;
        };
        u32x4_t p[RB];
#pragma nounroll
        for (int told = fresh ? 1 : 0;; told = 2) {
          if (told) refer();
          uint32_t any = 0;
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) {
            f32x4_t s[2];
            scores(rb, s);
            float e[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) e[j] = __builtin_amdgcn_exp2f(s[j >> 2][j & 3]);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              p[rb][c] = pack_bf16x2(e[2 * c], e[2 * c + 1]);
              any |= p[rb][c];
            }
            if constexpr (!QR)  // two row blocks' scores at a time: registers
              if (rb & 1) __builtin_amdgcn_sched_barrier(0);
          }
          // The highest exponent bit: a probability of 2 or more, 2^8 times what its row's reference meant.
          if (told == 2 || __ballot((any & 0x40004000u) != 0) == 0) break;
        }
        if (live < MXA_TILE) {
          int32_t left = live - (int)value_row;
          asm volatile("" : "+v"(left));  // the comparisons stay in here
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int r = 16 * (c >> 1) + 4 * (c & 1);
            const uint32_t kept = (r < left ? 0xffffu : 0u) | (r + 2 < left ? 0xffff0000u : 0u);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) p[rb][c] &= kept;
          }
        }
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int c = 0; c < 4; ++c) sum[rb] = add_both(p[rb][c], sum[rb]);
        if constexpr (!QR) __builtin_amdgcn_sched_barrier(0);  // the values are read behind the scores: registers
        typedef typename std::conditional<D == 128, uint32_t, uint16_t>::type vword_t;
        uint32_t vw[8];
        float vs[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int i = j & 3, tb = j >> 2;
          vw[j] = *reinterpret_cast<const vword_t *>(slot + value_at[i] + 16 * D * tb);
          vs[j] = mx_scale_float(*reinterpret_cast<const uint8_t *>(slot + value_scale_at + (D / 16) * (16 * tb + 2 * i)));
        }
        auto channels = [&](auto sel) {  // two of this lane's channels
          constexpr int B = decltype(sel)::value;
          uint32_t w[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) w[j] = widen<B>(vw[j], vs[j]);
          const u32x4_t v0 = {both_lo(w[0], w[1]), both_lo(w[2], w[3]), both_lo(w[4], w[5]), both_lo(w[6], w[7])};
          const u32x4_t v1 = {both_hi(w[0], w[1]), both_hi(w[2], w[3]), both_hi(w[4], w[5]), both_hi(w[6], w[7])};
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) o[rb][2 * B] = mfma_16x16x32(v0, p[rb], o[rb][2 * B]);
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) o[rb][2 * B + 1] = mfma_16x16x32(v1, p[rb], o[rb][2 * B + 1]);
        };
        channels(std::integral_constant<int, 0>{});
        channels(std::integral_constant<int, 1>{});
        if constexpr (D == 128) {
          channels(std::integral_constant<int, 2>{});
          channels(std::integral_constant<int, 3>{});
        }
      }
      read_at = read_at == (G::NS - 1) * G::SLOT ? 0 : read_at + G::SLOT;
      if (again) load_tile(rows);
    }

    fetch_query(more ? next : cc);  // on its way while this unit is joined
    // The four wavefronts' parts of the unit together, MF fragments at a time.
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      sum[rb] = sum_over_groups(sum[rb]);
      if (g == 0) *reinterpret_cast<float2 *>(ml + 2 * ((wave * RB + rb) * 16 + n)) = make_float2(fresh ? -INFINITY : -minus[rb][0], sum[rb]);
    }
    lds_barrier();  // and the queries have been read: their place takes the fragments
    float scale[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {  // a row's reference and sum over the wavefronts
      float2 v[MXA_WAVES];
#pragma unroll
      for (int w = 0; w < MXA_WAVES; ++w) v[w] = *reinterpret_cast<const float2 *>(ml + 2 * ((w * RB + rb) * 16 + n));
      float m = v[0].x, l = 0.f;
#pragma unroll
      for (int w = 1; w < MXA_WAVES; ++w) m = fmaxf(m, v[w].x);
#pragma unroll
      for (int w = 0; w < MXA_WAVES; ++w) l += v[w].y * __builtin_amdgcn_exp2f(v[w].x - m);
      scale[rb] = fresh ? 0.f : __builtin_amdgcn_exp2f(-minus[rb][0] - m);
      minus[rb][0] = m, sum[rb] = l;
    }
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const float inv = 1.f / sum[rb];
      const int64_t at = (int64_t)part * RB + rb;
      float *const part_o = a.part_o + at * 16 * D + 4 * lane;  // fragment 0's place
      auto row_out = [&]() {  // row n's channels, or NULL
        int32_t head;
        const int64_t token = row_token(cc, rb, head);
        return token >= 0 ? a.o + token * a.o_st + ((int64_t)cc.h * a.group + head) * a.o_sh : nullptr;
      };
      if (!whole && wave == 0 && g == 0)
        *reinterpret_cast<float2 *>(a.part_ml + 2 * (at * 16 + n)) = make_float2(minus[rb][0], sum[rb]);
      if constexpr (G::MF == 2) {
        // Fragments f and f + 1, of which each wavefront joins one of the lanes' four values.
        uint16_t *const dst = whole ? row_out() : nullptr;
#pragma unroll
        for (int f = 0; f < G::NF; f += 2) {
          if (rb + f > 0) lds_barrier();  // the last two have been read
#pragma unroll
          for (int q = 0; q < 2; ++q)
            *reinterpret_cast<f32x4_t *>(shared + ((q * MXA_WAVES + wave) * 64 + lane) * 16) = o[rb][f + q] * scale[rb];
          lds_barrier();
          float v[2] = {0.f, 0.f};
#pragma unroll
          for (int w = 0; w < MXA_WAVES; ++w)
#pragma unroll
            for (int q = 0; q < 2; ++q)
              v[q] += *reinterpret_cast<const float *>(shared + ((q * MXA_WAVES + w) * 64 + lane) * 16 + 4 * wave);
          if (!whole)
            part_o[f * 256 + wave] = v[0], part_o[(f + 1) * 256 + wave] = v[1];
          else if (dst != nullptr)
            *reinterpret_cast<uint32_t *>(dst + (4 * g + wave) * G::NF + f) = pack_bf16x2(v[0] * inv, v[1] * inv);
        }
      } else {
        // Every FWth fragment from h on, one for each wavefront: FW in all, whose channels lie side by side.
        constexpr int FW = G::NF / 4;
        f32x4_t v[FW];
#pragma unroll
        for (int h = 0; h < FW; ++h) {
          if (rb + h > 0) lds_barrier();  // the last four have been read
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<f32x4_t *>(shared + ((q * MXA_WAVES + wave) * 64 + lane) * 16) = o[rb][q * FW + h] * scale[rb];
          lds_barrier();
          v[h] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int w = 0; w < MXA_WAVES; ++w)
            v[h] += *reinterpret_cast<const f32x4_t *>(shared + ((wave * MXA_WAVES + w) * 64 + lane) * 16);
        }
        if (!whole) {
#pragma unroll
          for (int h = 0; h < FW; ++h) *reinterpret_cast<f32x4_t *>(part_o + (wave * FW + h) * 256) = v[h];
        } else if (uint16_t *const dst = row_out()) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint16_t *const to = dst + (4 * g + i) * G::NF + wave * FW;
            const uint32_t d = pack_bf16x2(v[0][i] * inv, v[FW - 1][i] * inv);
            if constexpr (FW == 2)
              *reinterpret_cast<uint32_t *>(to) = d;
            else
              *to = (uint16_t)d;
          }
        }
      }
    }

    cc = next;
  }
}

// The units that shares cut, from their parts, and zeros for the sequences without context. A
// workgroup a 16-row block of a unit, a wavefront a quarter of its fragments, as the parts hold them:
// they are written and read whole lines at a time. SPLIT: the quarters lie with four workgroups, whose
// wavefronts take every fourth part (calls of few units, which are cut into many).
template <int D, bool SPLIT>
__global__ __launch_bounds__(64 * MXA_WAVES) void attn_mx_join_kernel(const MxAttnArgs a, int rb_unit) {
  constexpr int NF = D / 16, FW = NF / 4;
  constexpr int STEP = SPLIT ? MXA_WAVES : 1;
  __shared__ int32_t sums[4][MXA_WAVES];
  __shared__ f32x4_t parts_sum[MXA_WAVES][64][FW + 1];
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int b = (int)blockIdx.x / a.hkv, h = (int)blockIdx.x - b * a.hkv;
  const int block = blockIdx.y, rg = block / rb_unit, rb = block - rg * rb_unit;
  const int32_t steps = steps_of(context_len(a, b));
  int64_t token0 = a.token0 + (int64_t)b * a.q_len;
  int32_t tokens = a.q_len;
  if (a.cu_q != nullptr) token0 = a.cu_q[b], tokens = tokens_in(a, token0, a.cu_q[b + 1]);
  const int32_t mine = (int)threadIdx.x < a.batch ? steps_of(context_len(a, threadIdx.x)) : 0;
  const int32_t upto = wave_prefix(mine);
  const uint64_t has = __ballot(mine > 0);
  if (lane == 63) sums[0][wave] = upto, sums[1][wave] = __popcll(has);
  if ((int)threadIdx.x == b) sums[2][0] = upto - mine, sums[3][0] = __popcll(has & ((1ull << lane) - 1));
  __syncthreads();
  int32_t all[4] = {0, sums[2][0], 0, sums[3][0]};  // steps, of them before b, sequences with steps, of them before b
#pragma unroll
  for (int w = 0; w < MXA_WAVES; ++w) {
    all[0] += sums[0][w], all[2] += sums[1][w];
    if (w < (b >> 6)) all[1] += sums[0][w], all[3] += sums[1][w];
  }
  // This thread: channels (4 g + i) NF + quarter FW + f of row n.
  const int n = lane & 15, g = lane >> 4, quarter = SPLIT ? (int)blockIdx.z : wave;
  const int32_t r = (a.rgroup0 * rb_unit + block) * 16 + n;
  const int32_t head = divided(r, a.q_mul, a.q_shift), tok = r - head * a.q_len;
  const bool live = r < a.group * a.q_len && tok < tokens && (!SPLIT || wave == 0);
  f32x4_t v[FW];
#pragma unroll
  for (int f = 0; f < FW; ++f) v[f] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  auto store = [&]() {
    if (!live) return;
    uint16_t *dst = a.o + (token0 + tok) * a.o_st + ((int64_t)h * a.group + head) * a.o_sh + 4 * g * NF + quarter * FW;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t d = pack_bf16x2(v[0][i], v[FW - 1][i]);
      if constexpr (FW == 2)
        *reinterpret_cast<uint32_t *>(dst + i * NF) = d;
      else
        dst[i * NF] = (uint16_t)d;
    }
  };
  if (steps == 0) return store();
  const MxPlan plan(a, all[0], all[2]);
  const int64_t from = (int64_t)a.hkv * (all[1] + plan.c * all[3]) + (int64_t)h * (steps + plan.c);
  const int32_t w0 = plan.share_of(from + plan.c), w1 = plan.share_of(from + plan.c + steps - 1);
  if (w0 == w1) return;  // whole in one share
  // Share w0's part lies behind that of the unit it starts with, if that is another.
  const int32_t p0 = 2 * (rg * a.shares + w0), behind = plan.share(w0) < from ? 1 : 0, parts = w1 - w0 + 1;
  float m = -INFINITY, l = 0.f;
  // Four parts at a time, their loads in flight together.
  for (int32_t i0 = SPLIT ? wave : 0; i0 < parts; i0 += 4 * STEP) {
    float2 ml[4];
    f32x4_t pv[4][FW];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int32_t i = i0 + u * STEP < parts ? i0 + u * STEP : i0;
      const int64_t at = (int64_t)(p0 + 2 * i + (i == 0 ? behind : 0)) * rb_unit + rb;
      ml[u] = *reinterpret_cast<const float2 *>(a.part_ml + 2 * (at * 16 + n));
      if (i0 + u * STEP >= parts) ml[u] = make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int f = 0; f < FW; ++f)
        pv[u][f] = *reinterpret_cast<const f32x4_t *>(a.part_o + ((at * NF + quarter * FW + f) * 64 + lane) * 4);
    }
    float top = m;
#pragma unroll
    for (int u = 0; u < 4; ++u) top = fmaxf(top, ml[u].x);
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
    l *= f;
#pragma unroll
    for (int c = 0; c < FW; ++c) v[c] *= f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (i0 + u * STEP >= parts) continue;
      const float fu = __builtin_amdgcn_exp2f(ml[u].x - top);
      l += ml[u].y * fu;
#pragma unroll
      for (int c = 0; c < FW; ++c) v[c] += pv[u][c] * fu;
    }
    m = top;
  }
  if constexpr (SPLIT) {
    f32x4_t *const to = parts_sum[wave][lane];
    to[0] = f32x4_t{m, l, 0.f, 0.f};
#pragma unroll
    for (int f = 0; f < FW; ++f) to[1 + f] = v[f];
    __syncthreads();
    if (wave != 0) return;
    float top = m;
#pragma unroll
    for (int w = 1; w < MXA_WAVES; ++w) top = fmaxf(top, parts_sum[w][lane][0][0]);
    l = 0.f;
#pragma unroll
    for (int f = 0; f < FW; ++f) v[f] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < MXA_WAVES; ++w) {
      const f32x4_t *src = parts_sum[w][lane];
      if (src[0][0] == -INFINITY) continue;  // took no part
      const float by = __builtin_amdgcn_exp2f(src[0][0] - top);
      l += src[0][1] * by;
#pragma unroll
      for (int f = 0; f < FW; ++f) v[f] += src[1 + f] * by;
    }
  }
  const float inv = 1.f / l;
#pragma unroll
  for (int f = 0; f < FW; ++f) v[f] *= inv;
  store();
}

constexpr int64_t MXA_ROWS = 1 << 20;  // query rows of a KV head

// How a KV head's query rows are cut: row blocks of a unit (up to 4, all units alike where the rows fill more
// than one), the row groups that they make, and those of one launch (even slices of at most MXA_GROUPS). A
// launch has a tail: one row of a head each, 300 positions, 65536 rows take 239 us in one launch and 275 in
// four, 200000 rows 725 in one and 750 in four.
struct MxRows {
  int32_t rb, rgroups, slice;
  explicit MxRows(int64_t rows) {
    const int32_t blocks = (int32_t)((rows + 15) / 16);
    rgroups = (blocks + 3) / 4;
    rb = (blocks + rgroups - 1) / rgroups;
    const int32_t launches = (rgroups + MXA_GROUPS - 1) / MXA_GROUPS;
    slice = (rgroups + launches - 1) / launches;
  }
};

// Shares of a row group: as many workgroups as the chip holds at once, by eights (a share an XCD).
static int32_t mx_attn_shares(int d, int rb, int32_t rgroups) {
  DeviceInfo info;
  const int cus = device_info(&info) == FM_OK ? info.cus : 256;
  const int32_t n = mx_resident(d, rb) * cus / rgroups / 8 * 8;
  return n < 8 ? 8 : n;
}

static size_t mx_attn_part_floats(int d, int rb, int32_t rgroups) {
  return (size_t)2 * mx_attn_shares(d, rb, rgroups) * rgroups * 16 * rb * (d + 2);
}

template <int D, int RB>
static int launch_attn_mx(const MxAttnArgs &a, hipStream_t stream) {
  attn_mx_kernel<D, RB><<<dim3(a.shares, a.rgroups), dim3(64 * MXA_WAVES), MxGeo<D, RB>::SMEM, stream>>>(a);
  FM_CHECK_HIP(hipGetLastError());
  const unsigned units = (unsigned)(a.batch * a.hkv), blocks = (unsigned)(a.rgroups * RB);
  // With fewer row blocks than the chip takes workgroups at once they are cut into many parts.
  if (units * blocks < 512)
    attn_mx_join_kernel<D, true><<<dim3(units, blocks, 4), dim3(64 * MXA_WAVES), 0, stream>>>(a, RB);
  else
    attn_mx_join_kernel<D, false><<<dim3(units, blocks), dim3(64 * MXA_WAVES), 0, stream>>>(a, RB);
  FM_CHECK_HIP(hipGetLastError());
  return FM_OK;
}

template <int D>
static int run_attn_mx(const MxAttnArgs &a, int rb, hipStream_t stream) {
  switch (rb) {
    case 1: return launch_attn_mx<D, 1>(a, stream);
    case 2: return launch_attn_mx<D, 2>(a, stream);
    case 3: return launch_attn_mx<D, 3>(a, stream);
    default: return launch_attn_mx<D, 4>(a, stream);
  }
}

}  // namespace fm

using namespace fm;

extern "C" size_t fm_block_attn_paged_mx_workspace_bytes(int32_t max_seqlen_q, int32_t num_q_heads,
                                                         int32_t num_kv_heads, int32_t head_dim) {
  if (max_seqlen_q <= 0 || num_kv_heads <= 0 || num_q_heads < num_kv_heads || head_dim <= 0) return 0;
  const int64_t rows = (int64_t)(num_q_heads / num_kv_heads) * max_seqlen_q;
  if (rows > MXA_ROWS) return 0;
  const MxRows cut(rows);
  return sizeof(float) * mx_attn_part_floats(head_dim, cut.rb, cut.slice);
}

extern "C" int fm_block_attn_paged_mx(
    const void *q, int64_t q_tokens, int64_t q_stride_token, int64_t q_stride_head, void *out, int64_t out_stride_token,
    int64_t out_stride_head, const int32_t *cu_seqlens_q, const void *codes, int64_t row_stride, const void *scales,
    int64_t scales_stride, int64_t num_blocks, int32_t page_size, const int32_t *block_table,
    int64_t block_table_stride, int64_t block_table_width, const int32_t *seqused_k, int32_t batch,
    int32_t max_seqlen_q, int32_t max_seqlen_k, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    float softmax_scale, const float *q_norm_weight, const float *rope_cos, const float *rope_sin,
    int64_t rope_row_stride, int64_t rope_pair_stride, int64_t rope_rows, const int64_t *q_positions, float eps,
    void *workspace, size_t workspace_bytes, void *stream) {
  clear_error();
  FM_REQUIRE(batch >= 0 && max_seqlen_q >= 0 && max_seqlen_k >= 0, "bad sizes");
  if (batch == 0 || max_seqlen_q == 0) return FM_OK;
  if (head_dim != 64 && head_dim != 128)
    return fail(FM_ERR_UNSUPPORTED, "head_dim %d not supported (64 or 128)", head_dim);
  FM_REQUIRE(num_kv_heads > 0 && num_q_heads > 0 && num_q_heads % num_kv_heads == 0,
             "%d query heads do not divide into %d KV heads", num_q_heads, num_kv_heads);
  // Where no context has a position the table is not read, and an empty one may have no address.
  FM_REQUIRE(q && out && codes && scales && seqused_k && workspace &&
                 (block_table || block_table_width == 0 || max_seqlen_k == 0),
             "NULL pointer");
  FM_REQUIRE(((uintptr_t)q & 15) == 0 && ((uintptr_t)out & 15) == 0 && ((uintptr_t)codes & 15) == 0 &&
                 ((uintptr_t)scales & 3) == 0 && ((uintptr_t)workspace & 15) == 0,
             "q, out, codes and workspace must be 16-byte aligned, scales 4-byte aligned");
  FM_REQUIRE(q_stride_token % 8 == 0 && q_stride_head % 8 == 0 && out_stride_token % 8 == 0 && out_stride_head % 8 == 0,
             "token and head strides must be multiples of 8 elements");
  FM_REQUIRE(row_stride % 16 == 0 && row_stride >= head_dim && scales_stride % 4 == 0 && scales_stride >= head_dim / 16,
             "cache rows hold %d code bytes at a stride of a multiple of 16 and %d scale bytes at one of 4", head_dim,
             head_dim / 16);
  FM_REQUIRE(num_blocks > 0 && page_size > 0 && page_size < (1 << 24) &&
                 num_blocks <= ((int64_t)UINT32_MAX / num_kv_heads) / page_size,
             "a cache of 1 to 2^32 - 1 rows, got %lld blocks of %d heads and %d positions", (long long)num_blocks,
             num_kv_heads, page_size);
  FM_REQUIRE(block_table_width >= 0 && (batch == 1 || block_table_stride >= 0), "bad block table");
  FM_REQUIRE(softmax_scale >= 0.f && softmax_scale <= 3e38f, "softmax_scale must be finite and not negative");
  FM_REQUIRE(q_norm_weight == nullptr || (rope_cos && rope_sin && rope_rows > 0 && rope_rows < (1ll << 31)),
             "a query norm needs its rotary table of 1 to 2^31 - 1 rows");
  if (q_norm_weight != nullptr && rope_pair_stride != 1 && !(rope_pair_stride == 2 && rope_sin == rope_cos + 1))
    return fail(FM_ERR_UNSUPPORTED, "rotary tables of pairs side by side, or (cos, sin) interleaved");
  FM_REQUIRE(q_tokens >= 0 && (cu_seqlens_q || q_tokens >= (int64_t)batch * max_seqlen_q),
             "without cu_seqlens_q the query holds batch x max_seqlen_q = %lld rows, got %lld",
             (long long)batch * max_seqlen_q, (long long)q_tokens);
  const int64_t rows = (int64_t)(num_q_heads / num_kv_heads) * max_seqlen_q;
  FM_REQUIRE(rows <= MXA_ROWS, "at most 2^20 query rows for a KV head, got %lld", (long long)rows);
  MxAttnArgs a{};
  const MxRows cut(rows);
  const int64_t units = (int64_t)(batch < MXA_BATCH ? batch : MXA_BATCH) * num_kv_heads;  // of a launch and row group
  FM_REQUIRE(units < (1 << 24), "%lld KV heads of a launch's sequences, at most 2^24 - 1", (long long)units);
  a.q_tokens = q_tokens;
  a.q = (const uint16_t *)q, a.q_st = q_stride_token, a.q_sh = q_stride_head;
  a.o = (uint16_t *)out, a.o_st = out_stride_token, a.o_sh = out_stride_head;
  a.q_len = max_seqlen_q, a.group = num_q_heads / num_kv_heads, a.hkv = num_kv_heads;
  a.codes = (const uint8_t *)codes, a.scales = (const uint8_t *)scales;
  const int64_t cache_rows = num_blocks * num_kv_heads * page_size, cs16 = row_stride / 16, ss4 = scales_stride / 4;
  FM_REQUIRE(cs16 <= UINT32_MAX / cache_rows && ss4 <= UINT32_MAX / cache_rows,
             "a cache of less than 2^36 bytes of code rows and 2^34 of scale rows");
  a.cs16 = (uint32_t)cs16, a.ss4 = (uint32_t)ss4, a.num_blocks = (uint32_t)num_blocks, a.page = page_size;
  a.head_rows = (uint32_t)num_kv_heads * page_size;
  auto divisor = [](int64_t d, uint32_t &mul, uint32_t &shift) {
    for (shift = 0; (1ll << shift) < d;) ++shift;
    mul = (uint32_t)(((1ull << (31 + shift)) + d - 1) / d);
  };
  divisor(page_size, a.page_mul, a.page_shift);
  divisor(max_seqlen_q, a.q_mul, a.q_shift);
  a.table_stride = block_table_stride;
  const int64_t held = block_table_width * page_size;
  const int64_t most = held < max_seqlen_k ? held : max_seqlen_k;
  FM_REQUIRE(most <= (1 << 24), "contexts of at most 2^24 positions, got %lld", (long long)most);
  a.max_len = (int32_t)most;
  a.scale_log2 = softmax_scale * 1.44269504088896341f;
  a.qn_w = q_norm_weight;
  a.rope = Rope{rope_cos, rope_sin, rope_row_stride, rope_pair_stride, rope_rows};
  a.q_pos = q_positions, a.eps = eps;
  a.shares = mx_attn_shares(head_dim, cut.rb, cut.slice);
  // A share's steps are counted in 32 bits.
  FM_REQUIRE(units * ((most + MXA_STEP - 1) / MXA_STEP) / a.shares < INT32_MAX, "too many positions for one launch");
  a.per_share = 1.0 / a.shares;
  const size_t need = sizeof(float) * mx_attn_part_floats(head_dim, cut.rb, cut.slice);
  if (workspace_bytes < need) return fail(FM_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
  a.part_o = (float *)workspace;
  a.part_ml = a.part_o + (size_t)2 * a.shares * cut.slice * 16 * cut.rb * head_dim;
  // Launches of up to MXA_BATCH sequences and MXA_GROUPS row groups, one after another: they share the workspace.
  for (int32_t b0 = 0; b0 < batch; b0 += MXA_BATCH) {
    a.batch = batch - b0 < MXA_BATCH ? batch - b0 : MXA_BATCH;
    a.cu_q = cu_seqlens_q == nullptr ? nullptr : cu_seqlens_q + b0;
    a.token0 = (int64_t)b0 * max_seqlen_q;
    a.table = block_table == nullptr ? nullptr : block_table + b0 * block_table_stride;
    a.lens = seqused_k + b0;
    for (a.rgroup0 = 0; a.rgroup0 < cut.rgroups; a.rgroup0 += cut.slice) {
      a.rgroups = cut.rgroups - a.rgroup0 < cut.slice ? cut.rgroups - a.rgroup0 : cut.slice;
      const int rc = head_dim == 128 ? run_attn_mx<128>(a, cut.rb, (hipStream_t)stream)
                                     : run_attn_mx<64>(a, cut.rb, (hipStream_t)stream);
      if (rc != FM_OK) return rc;
    }
  }
  return FM_OK;
}
