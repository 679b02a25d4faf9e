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
// bits, all 8 of a bf16 (2^e puts a block's largest magnitude to [128, 256); a value below 2^-13 of
// that loses at most 2^-22 of it). The query's norm and rotation, where they go with the call, are
// float32 and rounded only there, by at most 2^-8. K needs no conversion and no register but the 16 bytes a
// lane that it comes in. S^T = K Q^T leaves a query row's scores in the lanes that take that row's
// probabilities in O^T = V^T P^T: nothing crosses lanes.
// Values: each lane widens 8 tokens' dwords (8 channels each) with their block's scale, exactly, to
// bf16 pairs, and pairs of tokens by byte permutes. Probabilities are rounded to bf16 (2^-9 of each, as
// the bf16 attention does); maxima, sums and outputs are float32.
// A row's maximum is a reference that moves only when a score passes it by 2^8: the sums stay far
// inside float32 and bf16 keeps its 8 bits wherever its exponent is.
#include <math.h>

#include <type_traits>

#include "fm_host.h"
#include "mx_device.h"

namespace fm {

constexpr int MXA_WAVES = 4;
constexpr int MXA_TILE = 32;                     // positions of a wavefront's tile
constexpr int MXA_STEP = MXA_WAVES * MXA_TILE;   // of a workgroup's step
constexpr int MXA_BATCH = 256;                   // sequences of one launch: their steps lie in LDS
constexpr float MXA_SLACK = 8.f;                 // log2 that scores may pass their row's reference by

struct MxAttnArgs {
  const uint16_t *q;
  int64_t q_st, q_sh;  // token and head strides, elements
  uint16_t *o;
  int64_t o_st, o_sh;
  const int32_t *cu_q;  // NULL: sequence b's tokens start at token0 + b q_len
  int64_t token0, q_tokens;  // q_tokens: rows of q and out; what cu_q says past them is left alone
  int32_t q_len, group, hkv, rgroups;
  const uint8_t *codes, *scales;
  int64_t cs, ss;  // row strides, bytes
  int64_t num_blocks;
  int32_t page;
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
  int32_t shares;
};

template <int D, int RB>
struct MxGeo {
  static constexpr int KB = D / 2;                        // bytes of a row's keys, and of its values
  static constexpr int NF = D / 16;                       // 16-channel fragments
  static constexpr int CODES = MXA_TILE * D, SCALES = MXA_TILE * (D / 16);
  static constexpr int DMAS = CODES / 1024;               // 16-byte loads a lane of a tile's codes
  static constexpr int LOADS = DMAS + 2;                  // and its scales, and later page ids
  static constexpr int SLOT = CODES + SCALES + 4 * MXA_TILE;
  static constexpr int NS = 3;                            // tiles in a wavefront's ring
  static constexpr int RING = MXA_WAVES * NS * SLOT;
  static constexpr int QN = D == 128 ? 4 : 2;             // 16-byte operands a lane of a row block's queries
  static constexpr int QOP = QN * 1024 + 128;             // and the bytes of their two scales
  static constexpr int MERGE = MXA_WAVES * 4 * 1024;      // four fragments of every wavefront
  static constexpr int SHARED = RB * QOP > MERGE ? RB * QOP : MERGE;  // one after the other
  static constexpr int ML = MXA_WAVES * RB * 16 * 8;
  static constexpr int PRE = (MXA_BATCH + 4) * 4 + MXA_BATCH * 4;
  static constexpr int SMEM = RING + SHARED + ML + PRE;
  static_assert(SMEM <= 80 * 1024, "two workgroups a CU");
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
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ int32_t context_len(const MxAttnArgs &a, int b) {
  const int32_t n = a.lens[b];
  return n < 0 ? 0 : n < a.max_len ? n : a.max_len;
}
__device__ __forceinline__ int32_t steps_of(int32_t len) { return (len + MXA_STEP - 1) / MXA_STEP; }
__device__ __forceinline__ int32_t tokens_of(const MxAttnArgs &a, int b) {  // query tokens of sequence b
  if (a.cu_q == nullptr) return a.q_len;
  const int64_t first = a.cu_q[b], end = a.cu_q[b + 1], n = (end < a.q_tokens ? end : a.q_tokens) - first;
  return n < 0 || first < 0 ? 0 : n < a.q_len ? (int32_t)n : a.q_len;
}
__device__ __forceinline__ int64_t first_token(const MxAttnArgs &a, int b) {
  return a.cu_q == nullptr ? a.token0 + (int64_t)b * a.q_len : (int64_t)a.cu_q[b];
}

// The line's share s: [s total / n, (s + 1) total / n).
__device__ __forceinline__ int64_t share_at(int64_t s, int64_t total, int64_t n) { return s * total / n; }

// A place on the line: step lt of unit (b, h, rg).
struct MxCursor {
  int b, h, rg, lt, steps, len;
};

struct MxLine {  // in LDS: steps of the sequences before b, and their lengths
  const int32_t *pre, *len;
  __device__ __forceinline__ void load(MxCursor &c) const {
    c.steps = uniform(pre[c.b + 1] - pre[c.b]);
    c.len = uniform(len[c.b]);
  }
};

__device__ __forceinline__ bool advance(const MxAttnArgs &a, const MxLine &line, MxCursor &c) {  // true: a new unit
  if (++c.lt < c.steps) return false;
  c.lt = 0;
  if (++c.rg < a.rgroups) return true;
  c.rg = 0;
  if (++c.h < a.hkv) return true;
  c.h = 0;
  for (++c.b; c.b < a.batch; ++c.b) {  // sequences without context have no units
    line.load(c);
    if (c.steps > 0) break;
  }
  return true;
}

// Where step t of the line lies, the sequences tested 64 at a time.
__device__ __forceinline__ MxCursor cursor_at(const MxAttnArgs &a, const MxLine &line, int64_t t) {
  const int64_t ups = (int64_t)a.hkv * a.rgroups;
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64)
    before += __popcll(__ballot(b0 + lane < a.batch && ups * line.pre[b0 + lane < a.batch ? b0 + lane : 0] <= t));
  // The last sequence that starts at or before t; those without steps start where the next does.
  MxCursor c;
  c.b = uniform(before - 1);
  line.load(c);
  const int64_t off = t - ups * uniform(line.pre[c.b]);
  const int unit = (int)(off / c.steps);
  c.lt = (int)(off - (int64_t)unit * c.steps);
  c.h = unit / a.rgroups;
  c.rg = unit - c.h * a.rgroups;
  return c;
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

// The float of a scale byte, of which the widening takes the exponent (0: 2^-127; 255: NaN).
__device__ __forceinline__ float mx_scale_float(uint32_t byte) { return __uint_as_float(byte << 23); }

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
__global__ __launch_bounds__(64 * MXA_WAVES, 2) void attn_mx_kernel(const MxAttnArgs a) {
  using G = MxGeo<D, RB>;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int n = lane & 15, g = lane >> 4;
  char *const ring = lds + wave * G::NS * G::SLOT;
  const uint32_t ring_at = (uint32_t)(uintptr_t)(lds_char_t *)ring;
  char *const shared = lds + G::RING, *const qop = shared;
  float *const ml = reinterpret_cast<float *>(shared + G::SHARED);
  int32_t *const pre = reinterpret_cast<int32_t *>(shared + G::SHARED + G::ML);
  int32_t *const len = pre + MXA_BATCH + 4;

  // The steps of the sequences before each: a prefix sum, a sequence a thread.
  {
    static_assert(MXA_BATCH == 64 * MXA_WAVES, "a sequence a thread");
    const int b = threadIdx.x;
    const int32_t l = b < a.batch ? context_len(a, b) : 0, s = steps_of(l);
    int32_t sum = s;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int32_t v = __shfl_up(sum, o);
      if (lane >= o) sum += v;
    }
    int32_t *const totals = reinterpret_cast<int32_t *>(ml);
    if (lane == 63) totals[wave] = sum;
    __syncthreads();
    for (int w = 0; w < wave; ++w) sum += totals[w];
    len[b] = l;
    pre[b] = sum - s;
    if (b == MXA_BATCH - 1) pre[MXA_BATCH] = sum;
    __syncthreads();
  }
  const MxLine line{pre, len};
  const int64_t total = (int64_t)a.hkv * a.rgroups * uniform(pre[a.batch]);
  const int64_t shares = total < a.shares ? total : a.shares;
  // Neighbouring shares on one XCD (workgroups go to the 8 XCDs in turn): the row groups of a head
  // and the ends of units read the same cache rows.
  const int64_t wg = blockIdx.x, per = gridDim.x >> 3;
  const int64_t share = wg < 8 * per ? (wg & 7) * per + (wg >> 3) : wg;
  if (share >= shares) return;
  const int64_t t0 = share_at(share, total, shares), t1 = share_at(share + 1, total, shares);
  const int32_t count = (int32_t)(t1 - t0);

  // ---- the ring. A tile's page ids lie in its slot before its rows are asked for: those of tile
  // t + NS travel with the rows of tile t.
  const MxCursor start = cursor_at(a, line, t0);
  MxCursor ci = start, cd = start, cc = start;
  int32_t ids_left = count;
  auto page_of = [&](const MxCursor &c, int32_t &t) {  // of this lane's position, t, of the wavefront's tile
    t = c.lt * MXA_STEP + wave * MXA_TILE + (lane & (MXA_TILE - 1));
    t = t < c.len ? t : c.len - 1;
    return __umulhi((uint32_t)t << 1, a.page_mul) >> a.page_shift;
  };
  auto load_ids = [&](uint32_t to) {  // of the tile at ci; past the share's end its last tile's again
    int32_t t;
    const uint32_t col = page_of(ci, t);
    if (lane < MXA_TILE) ring_load4(a.table + (int64_t)ci.b * a.table_stride + col, to + G::CODES + G::SCALES);
    if (--ids_left > 0) advance(a, line, ci);
  };
  int32_t load_at = 0;  // the slot of the tile at cd
  auto load_tile = [&]() {
    const uint32_t to = ring_at + load_at;
    int32_t t;
    const uint32_t col = page_of(cd, t);
    uint32_t id = *reinterpret_cast<const uint32_t *>(ring + load_at + G::CODES + G::SCALES + 4 * (lane & (MXA_TILE - 1)));
    ring_read_done();                           // and whoever read this slot's last tile is done
    id = id < (uint32_t)a.num_blocks ? id : 0;  // a page that the cache does not have: its first
    const uint32_t row = (id * (uint32_t)a.hkv + cd.h) * (uint32_t)a.page + ((uint32_t)t - col * (uint32_t)a.page);
    constexpr int LPR = D / 16;  // lanes of a row
#pragma unroll
    for (int u = 0; u < G::DMAS; ++u) {
      const int r = (64 / LPR) * u + lane / LPR;
      const uint32_t from = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * r, (int)row);
      const int piece = (lane % LPR) ^ (D == 128 ? r >> 1 & 7 : r >> 2 & 3);  // as place() says
      ring_load16(a.codes + (uint64_t)from * (uint64_t)a.cs + 16 * piece, to + 1024 * u);
    }
    if constexpr (D == 128) {
      const uint32_t from = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * (lane >> 1), (int)row);
      ring_load4(a.scales + (uint64_t)from * (uint64_t)a.ss + 4 * (lane & 1), to + G::CODES);
    } else {
      if (lane < MXA_TILE) ring_load4(a.scales + (uint64_t)row * (uint64_t)a.ss, to + G::CODES);
    }
    load_ids(to);
    advance(a, line, cd);
    load_at = load_at == (G::NS - 1) * G::SLOT ? 0 : load_at + G::SLOT;
  };
  const int32_t ahead = count < G::NS ? count : G::NS;
  for (int32_t i = 0; i < ahead; ++i) load_ids(ring_at + i * G::SLOT);
  ring_wait<0>();
  for (int32_t i = 0; i < ahead; ++i) load_tile();

  // ---- the share, unit by unit
  const int32_t rows = a.group * a.q_len;  // of a sequence's KV head
  int32_t read_at = 0;                     // the slot of the tile to take
  for (int32_t k = 0; k < count;) {
    const int32_t seg = cc.steps - cc.lt < count - k ? cc.steps - cc.lt : count - k;
    const bool whole = seg == cc.steps;
    const int32_t row0 = cc.rg * RB * 16, tokens = tokens_of(a, cc.b);
    const int64_t token0 = first_token(a, cc.b);

    // The unit's queries as operands: a wavefront a row block.
    lds_barrier();  // nobody joins the last unit any more
    if (wave < RB) {
      const int32_t r = row0 + 16 * wave + n, head = r / a.q_len, tok = r - head * a.q_len;
      const bool live = r < rows && tok < tokens;
      const int64_t token = live ? token0 + tok : 0;
      const uint16_t *src = a.q + token * a.q_st + ((int64_t)cc.h * a.group + (live ? head : 0)) * a.q_sh + 8 * g;
      u32x4_t x[D / 32];
#pragma unroll
      for (int t = 0; t < D / 32; ++t) x[t] = live ? load16(src + 32 * t) : u32x4_t{0, 0, 0, 0};
      float y[D / 32][8];
      if (a.qn_w != nullptr) {
        const int64_t pos = live ? (a.q_pos != nullptr ? a.q_pos[token] : token) : 0;
        PrologueOps<D> ops;
        load_prologue_ops<D>(ops, a.qn_w, a.rope, clamp_row(a.rope, pos), g);
        norm_rope_exact<D>(x, ops, a.eps, y);
      } else {
#pragma unroll
        for (int t = 0; t < D / 32; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) y[t][2 * i] = bf16_lo(x[t][i]), y[t][2 * i + 1] = bf16_hi(x[t][i]);
      }
      // A row's hi and lo codes, 2 D bytes, then all rows in the operands' order in their place.
      char *const to = qop + wave * G::QOP, *const stage = to + n * 2 * D;
      uint32_t mine = 0;  // the byte of block g
#pragma unroll
      for (int t = 0; t < D / 32; ++t) {
        u32x2_t hi, lo;
        uint32_t byte;
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
    u32x4_t qr[RB <= 2 ? RB : 1][G::QN];
    if constexpr (RB <= 2) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int i = 0; i < G::QN; ++i) qr[rb][i] = load16(qop + rb * G::QOP + 1024 * i + 16 * lane);
    }

    f32x4_t o[RB][G::NF];
    float ref[RB], sum[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      ref[rb] = -INFINITY, sum[rb] = 0.f;
#pragma unroll
      for (int f = 0; f < G::NF; ++f) o[rb][f] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }

    for (int32_t i = 0; i < seg; ++i, ++k) {
      wait_tiles<G::LOADS, G::NS - 1>(count - k - 1);
      const int32_t live = cc.len - (cc.lt + i) * MXA_STEP - wave * MXA_TILE;  // positions of the tile
      if (live > 0) {
        const char *const slot = ring + read_at;
        u32x4_t kf[2];
        int ks[2];
#pragma unroll
        for (int tb = 0; tb < 2; ++tb) {
          const int r = 16 * tb + row_of(n), c = D == 128 ? g : g & 1;
          kf[tb] = load16(slot + place<D>(r, c));
          ks[tb] = *reinterpret_cast<const uint8_t *>(slot + G::CODES + r * (D / 16) + c);
        }
        u32x4_t p[RB];
        auto scores = [&](auto from) {  // of two row blocks (or the last one)
          constexpr int R0 = decltype(from)::value, R1 = R0 + 2 < RB ? R0 + 2 : RB, R = R1 - R0;
          f32x4_t s[R][2];
#pragma unroll
          for (int i = 0; i < R; ++i) {
            u32x4_t q[G::QN];
#pragma unroll
            for (int x = 0; x < G::QN; ++x) {
              if constexpr (RB <= 2)
                q[x] = qr[R0 + i][x];
              else
                q[x] = load16(qop + (R0 + i) * G::QOP + 1024 * x + 16 * lane);
            }
            const int qs = *reinterpret_cast<const uint16_t *>(qop + (R0 + i) * G::QOP + G::QN * 1024 + 2 * lane);
#pragma unroll
            for (int tb = 0; tb < 2; ++tb) {
              s[i][tb] = mfma_k_q(kf[tb], q[0], q[1], f32x4_t{0.f, 0.f, 0.f, 0.f}, ks[tb], qs);
              if constexpr (D == 128) s[i][tb] = mfma_k_q(kf[tb], q[2], q[3], s[i][tb], ks[tb], qs >> 8);
            }
          }
          if (live < MXA_TILE) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int r = 16 * (j >> 2) + (g & 1) + 8 * (g >> 1) + 2 * (j & 3);
#pragma unroll
              for (int i = 0; i < R; ++i)
                if (r >= live) s[i][j >> 2][j & 3] = -INFINITY;
            }
          }
          float top[R];
          bool passed = false;
#pragma unroll
          for (int i = 0; i < R; ++i) {
            top[i] = s[i][0][0];
#pragma unroll
            for (int j = 1; j < 8; ++j) top[i] = fmaxf(top[i], s[i][j >> 2][j & 3]);
            top[i] *= a.scale_log2;
            passed |= top[i] > ref[R0 + i] + MXA_SLACK;
          }
          if (__ballot(passed) != 0) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
              const float m = fmaxf(fmaxf(ref[R0 + i], max_over_groups(top[i])), -3.0e38f);
              const float f = __builtin_amdgcn_exp2f(ref[R0 + i] - m);
              ref[R0 + i] = m;
              sum[R0 + i] *= f;
#pragma unroll
              for (int c = 0; c < G::NF; ++c) o[R0 + i][c] *= f;
            }
          }
#pragma unroll
          for (int i = 0; i < R; ++i) {
            float e[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              e[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][j >> 2][j & 3], a.scale_log2, -ref[R0 + i]));
              sum[R0 + i] += e[j];
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) p[R0 + i][c] = pack_bf16x2(e[2 * c], e[2 * c + 1]);
          }
        };
        scores(std::integral_constant<int, 0>{});
        if constexpr (RB > 2) scores(std::integral_constant<int, 2>{});
        asm volatile("" : : : "memory");  // the values are read behind the scores: registers
        typedef typename std::conditional<D == 128, uint32_t, uint16_t>::type vword_t;
        uint32_t vw[8];
        float vs[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int r = 16 * (j >> 2) + (g & 1) + 8 * (g >> 1) + 2 * (j & 3);
          const int c = D == 128 ? n >> 2 : n >> 3, in = D == 128 ? 4 * (n & 3) : 2 * (n & 7);
          vw[j] = *reinterpret_cast<const vword_t *>(slot + place<D>(r, D / 32 + c) + in);
          vs[j] = mx_scale_float(*reinterpret_cast<const uint8_t *>(slot + G::CODES + r * (D / 16) + D / 32 + c));
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
      if (k + G::NS < count) load_tile();
    }

    // The four wavefronts' parts of the unit together, four fragments of each at a time.
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      sum[rb] = sum_over_groups(sum[rb]);
      if (g == 0) *reinterpret_cast<float2 *>(ml + 2 * ((wave * RB + rb) * 16 + n)) = make_float2(ref[rb], sum[rb]);
    }
    lds_barrier();
    auto joined = [&](int row, float &m, float &l) {  // a row's reference and sum over the wavefronts
      float2 v[MXA_WAVES];
#pragma unroll
      for (int w = 0; w < MXA_WAVES; ++w) v[w] = *reinterpret_cast<const float2 *>(ml + 2 * (w * RB * 16 + row));
      m = v[0].x;
#pragma unroll
      for (int w = 1; w < MXA_WAVES; ++w) m = fmaxf(m, v[w].x);
      l = 0.f;
#pragma unroll
      for (int w = 0; w < MXA_WAVES; ++w) l += v[w].y * __builtin_amdgcn_exp2f(v[w].x - m);
    };
    const int64_t part = 2 * share + (k == seg ? 0 : 1);
    constexpr int FW = G::NF / 4;  // fragments of a row block that a wavefront joins
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const int32_t r = row0 + 16 * rb + n, head = r / a.q_len, tok = r - head * a.q_len;
      const bool live = r < rows && tok < tokens;
      float m, l;
      joined(rb * 16 + n, m, l);
      const float scale = __builtin_amdgcn_exp2f(ref[rb] - m);
      f32x4_t v[FW];
#pragma unroll
      for (int h = 0; h < FW; ++h) {
        lds_barrier();  // the last four fragments (the queries, at first) have been read
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<f32x4_t *>(shared + ((q * MXA_WAVES + wave) * 64 + lane) * 16) = o[rb][q * FW + h] * scale;
        lds_barrier();
        v[h] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < MXA_WAVES; ++w)
          v[h] += *reinterpret_cast<const f32x4_t *>(shared + ((wave * MXA_WAVES + w) * 64 + lane) * 16);
      }
      // Channels (4 g + i) NF + wave FW + h of row n.
      if (whole) {
        if (live) {
          const float inv = 1.f / l;
          uint16_t *dst = a.o + (token0 + tok) * a.o_st + ((int64_t)cc.h * a.group + head) * a.o_sh + 4 * g * G::NF + wave * FW;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t d = pack_bf16x2(v[0][i] * inv, v[FW - 1][i] * inv);
            if constexpr (FW == 2)
              *reinterpret_cast<uint32_t *>(dst + i * G::NF) = d;
            else
              dst[i * G::NF] = (uint16_t)d;
          }
        }
      } else {
        const int64_t at = part * RB + rb;
#pragma unroll
        for (int h = 0; h < FW; ++h)
          *reinterpret_cast<f32x4_t *>(a.part_o + ((at * G::NF + wave * FW + h) * 64 + lane) * 4) = v[h];
        if (wave == 0 && g == 0) *reinterpret_cast<float2 *>(a.part_ml + 2 * (at * 16 + n)) = make_float2(m, l);
      }
    }
    cc.lt += seg - 1;
    advance(a, line, cc);
  }
}

// The units that shares cut, from their parts, and zeros for the sequences without context. A
// workgroup a 16-row block of a unit, laid out as the parts are: a wavefront D / 64 fragments.
template <int D>
__global__ __launch_bounds__(64 * MXA_WAVES) void attn_mx_join_kernel(const MxAttnArgs a, int rb_unit) {
  constexpr int NF = D / 16, FW = NF / 4;
  __shared__ int32_t sums[2][MXA_WAVES];
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int n = lane & 15, g = lane >> 4;
  const int64_t ups = (int64_t)a.hkv * a.rgroups;
  const int b = (int)(blockIdx.x / ups), u = (int)(blockIdx.x - b * ups), h = u / a.rgroups, rg = u - h * a.rgroups;
  const int rb = blockIdx.y;
  int32_t before = 0, all = 0;
  if ((int)threadIdx.x < a.batch) all = steps_of(context_len(a, threadIdx.x));
  before = (int)threadIdx.x < b ? all : 0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) before += __shfl_xor(before, o), all += __shfl_xor(all, o);
  if (lane == 0) sums[0][wave] = before, sums[1][wave] = all;
  __syncthreads();
  before = all = 0;
#pragma unroll
  for (int w = 0; w < MXA_WAVES; ++w) before += sums[0][w], all += sums[1][w];
  const int64_t total = ups * all, shares = total < a.shares ? total : a.shares;
  const int32_t steps = steps_of(context_len(a, b));
  const int32_t tokens = tokens_of(a, b);
  const int32_t r = (rg * rb_unit + rb) * 16 + n, head = r / a.q_len, tok = r - head * a.q_len;
  const bool live = r < a.group * a.q_len && tok < tokens;
  f32x4_t v[FW];
#pragma unroll
  for (int f = 0; f < FW; ++f) v[f] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float inv = 0.f;
  if (steps > 0) {
    const int64_t s = ups * before + (int64_t)u * steps, e = s + steps;
    const int64_t w0 = ((s + 1) * shares - 1) / total, w1 = (e * shares - 1) / total;
    if (w0 == w1) return;
    float m = -INFINITY, l = 0.f;
    for (int64_t w = w0; w <= w1; ++w) {
      const int64_t at = (2 * w + (share_at(w, total, shares) < s ? 1 : 0)) * rb_unit + rb;
      const float2 ml = *reinterpret_cast<const float2 *>(a.part_ml + 2 * (at * 16 + n));
      const float top = fmaxf(m, ml.x), f0 = __builtin_amdgcn_exp2f(m - top), f1 = __builtin_amdgcn_exp2f(ml.x - top);
      l = l * f0 + ml.y * f1;
#pragma unroll
      for (int f = 0; f < FW; ++f)
        v[f] = v[f] * f0 + *reinterpret_cast<const f32x4_t *>(a.part_o + ((at * NF + wave * FW + f) * 64 + lane) * 4) * f1;
      m = top;
    }
    inv = 1.f / l;
  }
  if (!live) return;
  uint16_t *dst = a.o + (first_token(a, b) + tok) * a.o_st + ((int64_t)h * a.group + head) * a.o_sh + 4 * g * NF + wave * FW;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t d = pack_bf16x2(v[0][i] * inv, v[FW - 1][i] * inv);
    if constexpr (FW == 2)
      *reinterpret_cast<uint32_t *>(dst + i * NF) = d;
    else
      dst[i * NF] = (uint16_t)d;
  }
}

// Row blocks of a unit: up to 4, all units alike where the rows fill more than one.
static int unit_blocks(int32_t rows, int32_t *rgroups) {
  const int32_t blocks = (rows + 15) / 16;
  *rgroups = (blocks + 3) / 4;
  return (blocks + *rgroups - 1) / *rgroups;
}

static int mx_attn_shares(int rb) {
  DeviceInfo info;
  const int cus = device_info(&info) == FM_OK ? info.cus : 256;
  (void)rb;
  return 2 * cus;
}

static size_t mx_attn_part_floats(int rb, int d) { return (size_t)2 * mx_attn_shares(rb) * 16 * rb * (d + 2); }

template <int D, int RB>
static int launch_attn_mx(const MxAttnArgs &a, hipStream_t stream) {
  attn_mx_kernel<D, RB><<<dim3((unsigned)a.shares), dim3(64 * MXA_WAVES), MxGeo<D, RB>::SMEM, stream>>>(a);
  FM_CHECK_HIP(hipGetLastError());
  const int64_t units = (int64_t)a.batch * a.hkv * a.rgroups;
  attn_mx_join_kernel<D><<<dim3((unsigned)units, RB), dim3(256), 0, stream>>>(a, RB);
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
  if (rows > (1 << 24)) return 0;
  int32_t rgroups;
  return sizeof(float) * mx_attn_part_floats(unit_blocks((int32_t)rows, &rgroups), head_dim);
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
  FM_REQUIRE(q && out && codes && scales && block_table && seqused_k && workspace, "NULL pointer");
  FM_REQUIRE(((uintptr_t)q & 15) == 0 && ((uintptr_t)out & 15) == 0 && ((uintptr_t)codes & 15) == 0 &&
                 ((uintptr_t)scales & 3) == 0 && ((uintptr_t)workspace & 15) == 0,
             "q, out, codes and workspace must be 16-byte aligned, scales 4-byte aligned");
  FM_REQUIRE(q_stride_token % 8 == 0 && q_stride_head % 8 == 0 && out_stride_token % 8 == 0 && out_stride_head % 8 == 0,
             "token and head strides must be multiples of 8 elements");
  FM_REQUIRE(row_stride % 16 == 0 && row_stride >= head_dim && scales_stride % 4 == 0 && scales_stride >= head_dim / 16,
             "cache rows hold %d code bytes at a stride of a multiple of 16 and %d scale bytes at one of 4", head_dim,
             head_dim / 16);
  FM_REQUIRE(num_blocks > 0 && page_size > 0 && page_size < (1 << 30) &&
                 num_blocks <= ((int64_t)UINT32_MAX / num_kv_heads) / page_size,
             "a cache of 1 to 2^32 - 1 rows, got %lld blocks of %d heads and %d positions", (long long)num_blocks,
             num_kv_heads, page_size);
  FM_REQUIRE(block_table_width >= 0 && (batch == 1 || block_table_stride >= 0), "bad block table");
  FM_REQUIRE(softmax_scale >= 0.f && softmax_scale <= 3e38f, "softmax_scale must be finite and not negative");
  FM_REQUIRE(q_norm_weight == nullptr || (rope_cos && rope_sin), "a query norm needs its rotary table");
  FM_REQUIRE(q_tokens >= 0 && (cu_seqlens_q || q_tokens >= (int64_t)batch * max_seqlen_q),
             "without cu_seqlens_q the query holds batch x max_seqlen_q = %lld rows, got %lld",
             (long long)batch * max_seqlen_q, (long long)q_tokens);
  const int64_t rows = (int64_t)(num_q_heads / num_kv_heads) * max_seqlen_q;
  FM_REQUIRE(rows <= (1 << 24), "at most 2^24 query rows for a KV head, got %lld", (long long)rows);
  MxAttnArgs a{};
  const int rb = unit_blocks((int32_t)rows, &a.rgroups);
  FM_REQUIRE((int64_t)MXA_BATCH * num_kv_heads * a.rgroups < (1ll << 31), "too many units");
  a.q_tokens = q_tokens;
  a.q = (const uint16_t *)q, a.q_st = q_stride_token, a.q_sh = q_stride_head;
  a.o = (uint16_t *)out, a.o_st = out_stride_token, a.o_sh = out_stride_head;
  a.q_len = max_seqlen_q, a.group = num_q_heads / num_kv_heads, a.hkv = num_kv_heads;
  a.codes = (const uint8_t *)codes, a.scales = (const uint8_t *)scales;
  a.cs = row_stride, a.ss = scales_stride, a.num_blocks = num_blocks, a.page = page_size;
  while ((1ll << a.page_shift) < page_size) ++a.page_shift;
  a.page_mul = (uint32_t)(((1ull << (31 + a.page_shift)) + page_size - 1) / page_size);
  a.table_stride = block_table_stride;
  const int64_t held = block_table_width * page_size;
  const int64_t most = held < max_seqlen_k ? held : max_seqlen_k;
  FM_REQUIRE(most <= (1 << 29), "contexts of at most 2^29 positions, got %lld", (long long)most);
  a.max_len = (int32_t)most;
  a.scale_log2 = softmax_scale * 1.44269504088896341f;
  a.qn_w = q_norm_weight;
  a.rope = Rope{rope_cos, rope_sin, rope_row_stride, rope_pair_stride, rope_rows};
  a.q_pos = q_positions, a.eps = eps;
  a.shares = mx_attn_shares(rb);
  const size_t need = sizeof(float) * mx_attn_part_floats(rb, head_dim);
  if (workspace_bytes < need) return fail(FM_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
  a.part_o = (float *)workspace;
  a.part_ml = a.part_o + (size_t)2 * a.shares * 16 * rb * head_dim;
  // Launches of up to MXA_BATCH sequences, one after another: they share the workspace.
  for (int32_t b0 = 0; b0 < batch; b0 += MXA_BATCH) {
    a.batch = batch - b0 < MXA_BATCH ? batch - b0 : MXA_BATCH;
    a.cu_q = cu_seqlens_q == nullptr ? nullptr : cu_seqlens_q + b0;
    a.token0 = (int64_t)b0 * max_seqlen_q;
    a.table = block_table + b0 * block_table_stride;
    a.lens = seqused_k + b0;
    const int rc = head_dim == 128 ? run_attn_mx<128>(a, rb, (hipStream_t)stream) : run_attn_mx<64>(a, rb, (hipStream_t)stream);
    if (rc != FM_OK) return rc;
  }
  return FM_OK;
}
