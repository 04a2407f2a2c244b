// GQA attention of the last tokens of each sequence over a 4-bit KV cache (format and layout: tdist/kv4.hpp).
//
// One workgroup of four waves takes one (sequence, KV head, block of query columns, KV split); a column is one (new token,
// query head) of the `group` heads that share the KV head.  A wave walks 32-token blocks, 128 tokens apart, with a softmax
// state of its own; the four states are merged through LDS, the splits by a second launch.
//
//   S^T[token, column] = K . Q^T.  A dword of K codes becomes four registers of two fp16 numbers, 1024 + code or 64 + code: the
//   code is put into the significand, one and-or for two codes and one shift for eight.  They are exact, and what a 16x16x32
//   MFMA takes.  The accumulator starts at -1024 and -64 times the sums of q that the offsets add, so what comes out is
//   sum(q code), and with a token's scale and low
//       s = scale * sum(q code) + low * sum(q).
//   O^T[channel, column] = V^T . P^T.  The scale belongs to a token, the axis that is summed: it goes into P, and P * scale is
//   rounded to fp16.  A step of that, 2^-11 of a weight, is an eighth of the bf16 result's own; for fp16 caches, whose result
//   has steps of 2^-11 too, the remainder is a second fp16 number.  A product of the same P with -1024 or -64 takes the
//   offsets off in the accumulator, where they and the code have met the same rounded weight.  sum(p low) is kept beside.
//   The 32 tokens of a block are contracted in the order in which the S^T accumulators hold them, which is how the V codes
//   are stored, so neither side moves between lanes.
// The reference m of the exponentials is raised only when a P * scale would pass 2^14 (fp16 ends at 2^16), and then put where
// the largest is 2^6: the cross-lane maximum leaves the loop, and a weight keeps all its bits down to 2^-20 of the largest
// (2^-8 in a group of 2^-12 of the widest scale; groups further apart, or far from 1, get a power of two each).
//
// What bounds it (calls in a row; from a graph over three caches in turn 58 .. 59 and 36 .. 38 us for the first two): many
// sequences, the bytes of the cache (64 x 4096 tokens, 8 heads of 128: 286 MB in 55 us, 5.2 TB/s, where a copy reaches 4.9 and reading
// alone 5.3 .. 5.6); one long sequence of 131072, those and the two launches' start and end (151 MB in 35 us, 4.3 TB/s); a few
// tokens, the launches (6.5 us); many columns, the vector instructions of unpacking and softmax (1024 new tokens over 16384, 266
// GFLOP: 511 .. 560 us, 520 TFLOP/s at best, and 740 in fp16; kv4_chunk.hip takes 295 for bf16 and gets such calls, but for capped
// ones: 915).  bf16 high and low parts of 16 + code, what this began with, took 103 us for the first of these.
//
// What is held in fewer bits than a sum in fp32, and shows: P * scale as one fp16 number over bf16 caches, which puts errors against 64
// bits 2 to 4 % above those of 32-bit arithmetic rounded once.  P is 2^34 at most, so that |low| up to 2^94 keeps its sums finite.
//
// Registers.  Spilled ones, of 256 (scratch, bytes a lane): heads of 256 in groups of 32 103 .. 156 (364 .. 512), in groups of 64
// 1 .. 37 (8 .. 136), heads of 128 in groups of 32 with two column blocks 41 .. 48 (152 .. 180), others none.  16 x 4096 tokens, 4 heads of 256:
// 42.7 us in groups of 32 where groups of 64 take 22.9 and of 128 20.2; 5 new tokens over 16 x 4096, 8 heads of 128: 41.7 and 30.0 us
// in groups of 32 and 64.
#include <algorithm>

#include "tdist/kv4.hpp"

namespace {

using namespace tdist::kv4;
typedef __attribute__((ext_vector_type(4))) float f32x4;
struct AttnArgs {
  Cache c;
  const uint16_t* q;        // [batch, S, q_heads, D]
  float* partial;           // splits > 1: [rows, splits, D] sums over their own weight, rows = batch * S * q_heads
  float* partial_lse;       // and [rows, splits] log2-sum-exp2 (-inf: no token)
  void* out;                // [batch, S, q_heads, D] (out_mode 1) or fp32 [.., D + 1] with the log-sum-exp (out_mode 2)
  long long q_sb, q_ss, q_sh;
  int table_stride, max_pages;
  int page_tiles;           // 16-token tiles of a page,
  uint32_t page_magic;      // and floor(2^32 / page_tiles) + 1 (0: one tile a page)
  int batch, S, q_heads, group, splits, causal, out_mode;
  int first;                // of this launch's (column block, sequence) pairs
  const int* flags;         // where given: [blocks of flag_columns * batch, splits, kv_heads], 0: another kernel has done it
  int flag_columns;
  float scale, soft_cap, inv_cap;     // (inv_cap: 1 / soft_cap)
};

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

// Blocks a wave has in flight.  Three where the registers hold them (131072 tokens: 37.5 us); one with two column blocks or heads of
// 256 channels, whose sums leave less room (chunk of 1024 511 us against 531 with two, heads of 256 50.3 against 53.9) - and not
// enough: see above for what is spilled even so.
constexpr int ring_of(int D, int CB) { return CB == 2 || D == 256 ? 1 : 3; }

#define INLINE __attribute__((always_inline))     // (lambdas: a call would put what they capture into memory)

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_fast(float x) { return __builtin_amdgcn_logf(x); }
__device__ __forceinline__ f32x4 mfma(const u32x4& a, const u32x4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// The masks and offsets of the unpacking, kept in registers (a literal each would keep the and-or from being one instruction)
struct Unpack {
  uint32_t m0, m1, o0, o1;
  __device__ __forceinline__ Unpack() {
    asm volatile("s_mov_b32 %0, 0x000f000f" : "=s"(m0));
    asm volatile("s_mov_b32 %0, 0x00f000f0" : "=s"(m1));
    asm volatile("v_mov_b32 %0, 0x64006400" : "=v"(o0));
    asm volatile("v_mov_b32 %0, 0x54005400" : "=v"(o1));
  }
  // nibbles n and n + 4 of a dword as two fp16 numbers: 1024 + code (n even) or 64 + code (n odd).  w8 = w >> 8.
  __device__ __forceinline__ uint32_t even(uint32_t w) const { return (w & m0) | o0; }
  __device__ __forceinline__ uint32_t odd(uint32_t w) const { return (w & m1) | o1; }
};

// One block of 32 tokens as it comes from the cache: two tiles of sixteen.  The parameters come one dword a lane and
// group (lanes 0 .. 31 the tokens' of K, 32 .. 63 of V) and reach the lanes that need them through LDS.
template <int D, int NG>
struct Raw {
  uint32_t k[2][D / 32], v[2][D / 32], params[NG];
};
// Where its tiles are: the first row of (page, KV head), the tile's first token in the page, and whether there is a page.
struct Where {
  long long row0[2];
  int off[2];
  bool there[2];
};

// the largest of a value over lanes 32 .. 63 (NaN only if all are)
__device__ __forceinline__ float max_upper_half(float v) {
  auto with = [&](int moved) { v = fmaxf(v, __builtin_bit_cast(float, moved)); };
  with(__builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0xb1, 0xf, 0xf, true));       // neighbours
  with(__builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x4e, 0xf, 0xf, true));       // pairs of them
  with(__builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x141, 0xf, 0xf, true));      // fours (mirrored eight)
  with(__builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x140, 0xf, 0xf, true));      // eights (mirrored sixteen)
  return fmaxf(__builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 32)),
               __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 48)));
}

template <int N>
__device__ __forceinline__ void load_words(uint32_t (&dst)[N], const uint8_t* base, uint32_t lane_off) {
  if constexpr (N == 2) {
    const uint2 v = *(const uint2*)(base + lane_off);
    dst[0] = v.x, dst[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const u32x4 v = *(const u32x4*)(base + lane_off + 16 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) dst[4 * i + j] = v[j];
    }
  }
}

// cap tanh(score / cap).  tanh is 1 - 2 / (e^2x + 1), which is off by 2^-24 of 1 however small x is: times a large cap that would
// be more than the scores themselves.  Up to x = 1 / 4 it is x (1 - x^2 / 3 + 2 x^4 / 15 - 17 x^6 / 315), the next term 62 x^8 / 2835 < 2^-21,
// and with it the score times what stands in brackets, which is the score itself under a cap that is far above it.
__device__ __forceinline__ float capped(float score, float cap, float inv_cap) {
  const float x = score * inv_cap, x2 = x * x;
  const float near = score * __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(x2, -17.f / 315.f, 2.f / 15.f), x2, -1.f / 3.f), x2, 1.f);
  const float far = cap * (1.f - 2.f * __builtin_amdgcn_rcpf(exp2_fast(2.f * 1.4426950408889634f * x) + 1.f));
  return fabsf(x) < 0.25f ? near : far;
}

// The larger of an op's two sides over the sixteen lanes of a row; every lane gets it.
template <class Op>
__device__ __forceinline__ float over_row(float v, Op op) {
  auto with = [&](int moved) { v = op(v, __builtin_bit_cast(float, moved)); };
  with(__builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0xb1, 0xf, 0xf, true));
  with(__builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x4e, 0xf, 0xf, true));
  with(__builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x141, 0xf, 0xf, true));
  with(__builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x140, 0xf, 0xf, true));
  return v;
}

// R = 0: CB blocks of sixteen columns share what a wave unpacks; scores as S^T[token, column].  Two blocks where there are more
// than sixteen columns (chunk of 1024: 1007 us with one, 532 with two and the loop as straight code); for heads of 256 the
// second block's sums do not fit the registers, and one is faster.
//
// R = 1, 2: at most 4 R columns (a decode step of grouped heads).  S^T would leave three quarters or half of every register idle,
// and all the work per score is done on registers.  Here it is S[column, token]: Q is the first operand, its columns spread
// over the rows 4 g + i, i < R, so that lane group g holds R columns of sixteen tokens - R registers a tile where S^T has four,
// and one token's parameters a lane where it has four's.  P goes to the second product through LDS.  Everything else is the same.
// 131072 tokens, four heads to a KV head: 37.5 us with it, 39.4 without (another card 35.4); 512 tokens 6.5 and 6.8.
template <bool IS_BF16, int D, int G, int CB, int R = 0>
__global__ __launch_bounds__(256, 2) void kv4_attn_kernel(AttnArgs a, const int* __restrict__ block_table,
                                                           const int* __restrict__ kv_len) {
  constexpr int KS = D / 32;            // MFMA steps over the head dim = dwords of a lane per K row
  constexpr int NT = D / 16;            // 16-channel tiles of V
  constexpr int NG = D / G;
  constexpr int GS = G / 32, GT = G / 16;
  constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
  constexpr float NONE = -1e30f;        // the reference before the first token
  constexpr float WIDE = 0x1p3f, NARROW = 0x1p-9f;      // V scales that are taken as they are
  constexpr float AT = 6.f, MOST = 14.f;  // log2 of the largest P: where a new reference puts it, and where it may grow to
  constexpr int DC = D < 128 ? D : 128; // channels merged at a time
  constexpr int W = R > 0 ? R : CB;     // columns of which a lane holds scores
  static_assert(R == 0 || CB == 1, "");
  __shared__ float s_m[4][16], s_l[4][16];
  __shared__ __attribute__((aligned(16))) float s_o[4][16][DC + 4];
  __shared__ __attribute__((aligned(16))) uint32_t s_params[4][2][NG][32];
  __shared__ __attribute__((aligned(16))) uint16_t s_p[R > 0 ? 4 : 1][NG][IS_BF16 ? 1 : 2][R > 0 ? 4 * R : 1][32];

  const int kvh = blockIdx.x, split = blockIdx.y;       // (kv heads first: what shares a cache line's XCD shares its L2)
  const int z = a.first + (int)blockIdx.z;
  const int cblk = a.batch == 1 ? z : z / a.batch, b = z - cblk * a.batch;
  const int group = a.group, columns = group * a.S;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, lg = lane >> 4;
  constexpr int COLUMNS = R > 0 ? 4 * R : 16 * CB;
  const int col0 = cblk * COLUMNS;
  if (a.flags && !a.flags[(((long long)(col0 / a.flag_columns) * a.batch + b) * a.splits + split) * gridDim.x + kvh]) return;

  // tokens: a column sees [0, limit), the workgroup's columns [0, len), none of them misses one below `full`
  const long long room = (long long)a.max_pages * a.c.page_size;
  const int L = (int)min((long long)max(kv_len[b], 0), room);
  const bool one = a.S == 1;                  // (columns are heads: no division by a variable on the way to the first load)
  const int s_first = one ? 0 : col0 / group, s_last = one ? 0 : min(col0 + COLUMNS - 1, columns - 1) / group;
  const int len = max(0, a.causal ? L - a.S + s_last + 1 : L);
  const int full = a.causal ? L - a.S + s_first + 1 : L;
  int whole = len;                            // what is split: with flags, what the flagged block of columns sees
  if (a.flags && a.causal) whole = max(0, L - a.S + min((col0 / a.flag_columns + 1) * a.flag_columns - 1, columns - 1) / group + 1);
  const int per = a.splits == 1 ? whole : ((whole + a.splits - 1) / a.splits + 127) & ~127;
  const int start = (int)min((long long)split * per, (long long)len), end = min(len, start + per);
  if (a.splits > 1 && start >= end) {         // (the merge does not look at the sums of a split without tokens)
    const int col = col0 + (int)threadIdx.x;
    if (threadIdx.x < COLUMNS && col < columns)
      a.partial_lse[(((long long)b * a.S + (one ? 0 : col / group)) * a.q_heads + kvh * group + (one ? col : col % group)) * a.splits +
                    split] = -INFINITY;
    return;
  }

  // Q as fp16: bf16 rows are brought near 2^8 by a power of two per column, which loses nothing that a score could show
  // (numbers 2^-32 of the column's largest).  A negative scale turns Q's sign, so that larger scores are larger weights.
  int limit[W];
  u32x4 q[CB][KS];
  float qsum[W][NG], qk[W];
  f32x4 c0[CB][NG];                           // what the accumulators start at
  u32x4 raw[CB][KS];
  auto fetch_q = [&]() INLINE {
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      // the column of this lane's operand row, and of its scores
      const int col = R > 0 ? col0 + (li >> 2) * R + (li & 3) : col0 + cb * 16 + li;
      const bool col_ok = col < columns && (R == 0 || (li & 3) < R);
      const int row_s = one || !col_ok ? 0 : col / group, head = kvh * group + (col_ok ? col - row_s * group : 0);
      if constexpr (R == 0) {
        limit[cb] = !col_ok ? 0 : a.causal ? L - a.S + row_s + 1 : L;
      } else {
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const int mine = col0 + lg * R + i;
          limit[i] = mine >= columns ? 0 : a.causal && !one ? L - a.S + mine / group + 1 : L;
        }
      }
      const uint16_t* qp = a.q + b * a.q_sb + row_s * a.q_ss + head * a.q_sh + lg * 8;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        raw[cb][s] = u32x4{0, 0, 0, 0};
        if (col_ok) raw[cb][s] = *(const u32x4*)(qp + 32 * s);
      }
    }
  };
  auto prepare_q = [&]() INLINE {
    const float sign = a.scale < 0.f ? -1.f : 1.f;
    const float lead = fabsf(a.soft_cap > 0.f ? a.scale : a.scale * LOG2E);
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      float mul = sign, back = 1.f;
      if (IS_BF16) {
        float top = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            top = fmaxf(top, fmaxf(fabsf(from16<IS_BF16>(raw[cb][s][i] & 0xffffu)), fabsf(low_of<IS_BF16>(raw[cb][s][i]))));
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        int e = (int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127;       // top in [2^e, 2^(e+1))
        e = e < -100 ? -100 : e;
        mul = sign * __builtin_bit_cast(float, (uint32_t)(127 + 8 - e) << 23);
        back = __builtin_bit_cast(float, (uint32_t)(127 - 8 + e) << 23);
      }
      const float factor = fminf(fmaxf(lead * back, 1e-37f), 1e37f);     // (a masked score is -inf, a 0 is 0: they stay that)
      if constexpr (R == 0) {
        qk[cb] = factor;
      } else {
#pragma unroll
        for (int i = 0; i < R; ++i) qk[i] = __shfl(factor, 4 * lg + i);
      }
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float sum0 = 0.f, sum1 = 0.f;         // of the channels that unpack as 1024 + code, and as 64 + code
#pragma unroll
        for (int s = g * GS; s < (g + 1) * GS; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t w = to16<false>(from16<IS_BF16>(raw[cb][s][i] & 0xffffu) * mul) |
                               to16<false>(low_of<IS_BF16>(raw[cb][s][i]) * mul) << 16;
            q[cb][s][i] = w;
            (i & 1 ? sum1 : sum0) += from16<false>(w & 0xffffu) + from16<false>(w >> 16);
          }
        sum0 += __shfl_xor(sum0, 16);
        sum0 += __shfl_xor(sum0, 32);
        sum1 += __shfl_xor(sum1, 16);
        sum1 += __shfl_xor(sum1, 32);
        const float c = -1024.f * sum0 - 64.f * sum1;
        if constexpr (R == 0) {
          qsum[cb][g] = sum0 + sum1;
          c0[cb][g] = f32x4{c, c, c, c};
        } else {
          c0[cb][g] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < R; ++i) qsum[i][g] = __shfl(sum0 + sum1, 4 * lg + i), c0[cb][g][i] = __shfl(c, 4 * lg + i);
        }
      }
    }
  };

  float m[W], l[W], corr[W][NG], vs[NG];
  f32x4 o[CB][NT];
#pragma unroll
  for (int cb = 0; cb < CB; ++cb)
#pragma unroll
    for (int j = 0; j < NT; ++j) o[cb][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < W; ++i) {
    m[i] = NONE, l[i] = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g) corr[i][g] = 0.f;
  }
  // a value of column li's score lane, for R > 0 (R registers of lane group li / R)
  auto of_column = [&](const float (&v)[W]) INLINE -> float {
    const int from = 16 * ((li / (R > 0 ? R : 1)) & 3);
    float r = __shfl(v[0], from);
    if constexpr (R == 2) {
      const float other = __shfl(v[W - 1], from);
      r = li & 1 ? other : r;
    }
    return r;
  };
#pragma unroll
  for (int g = 0; g < NG; ++g) vs[g] = 1.f;
  const Unpack u;
  u32x4 neg0, neg1;                     // -1024 and -64
#pragma unroll
  for (int i = 0; i < 4; ++i) neg0[i] = 0xe400e400u, neg1[i] = 0xd400d400u;

  const int* table = block_table + (long long)b * a.table_stride;
  const int last_tile = (end - 1) >> 4;
  auto lookup = [&](int n0) INLINE -> Where {
    Where w;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int want = (n0 >> 4) + t, tile = min(want, last_tile);
      uint32_t i = a.page_magic ? (uint32_t)(((uint64_t)(uint32_t)tile * a.page_magic) >> 32) : (uint32_t)tile;
      if (i * (uint32_t)a.page_tiles > (uint32_t)tile) --i;     // the quotient, or one more
      const int page = table[i];
      w.there[t] = want <= last_tile && page >= 0 && page < a.c.pages;
      w.row0[t] = ((long long)(w.there[t] ? page : 0) * a.c.kv_heads + kvh) * a.c.page_size;
      w.off[t] = (tile - (int)i * a.page_tiles) * 16;
    }
    return w;
  };
  const uint32_t k_lane = li * (D / 2) + lg * (D / 8), v_lane = lg * (2 * D) + li * (D / 8);
  const uint32_t* p_lane = (lane < 32 ? a.c.k_params : a.c.v_params) + li;      // lane: token lane & 31 of K or V
  uint32_t(*const params)[NG][32] = s_params[wave];
  auto load_k = [&](const Where& w, Raw<D, NG>& r) INLINE {         // and the parameters of both
#pragma unroll
    for (int t = 0; t < 2; ++t) load_words(r.k[t], a.c.k_codes + (w.row0[t] + w.off[t]) * (D / 2), k_lane);
    const long long at0 = w.row0[0] * NG + w.off[0], at1 = w.row0[1] * NG + w.off[1];
    const uint32_t* p = p_lane + (lane & 16 ? at1 : at0);
#pragma unroll
    for (int g = 0; g < NG; ++g) r.params[g] = p[(long long)g * a.c.page_size];
  };
  auto load_v = [&](const Where& w, Raw<D, NG>& r) INLINE {
#pragma unroll
    for (int t = 0; t < 2; ++t) load_words(r.v[t], a.c.v_codes + (w.row0[t] + w.off[t]) * (D / 2), v_lane);
  };
  auto load = [&](const Where& w, Raw<D, NG>& r) INLINE {
    load_k(w, r);
    load_v(w, r);
  };
  // V scales far from 1 are brought there by a power of two per group, the same for all columns; `widest` becomes the widest
  // after that.  false: they are far from 1, and the block is not treated as one that needs care.
  auto rescale = [&](auto careful, const uint32_t (&param)[NG], float (&ratio)[NG], float& widest) INLINE -> bool {
    constexpr bool CAREFUL = decltype(careful)::value;
    if (!CAREFUL) {
      bool off = false;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const float w = max_upper_half(fmaxf(0.f, scale_of<IS_BF16>(param[g])));
        off |= w > WIDE || (w > 0.f && w < NARROW);
      }
      if (off) return false;
    }
    widest = 0x1p-20f;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      ratio[g] = 1.f;
      const float w = max_upper_half(fmaxf(0.f, scale_of<IS_BF16>(param[g]) * vs[g]));
      if (CAREFUL && (w > WIDE || (w > 0.f && w < NARROW))) {
        const int have = (int)(__builtin_bit_cast(uint32_t, vs[g]) >> 23) - 127;
        int e = (int)(__builtin_bit_cast(uint32_t, w) >> 23) - 127;
        e = min(max(e, -60), 60);           // (what is further off takes several blocks to arrive)
        e = min(max(e, have - 120), have + 120);
        ratio[g] = __builtin_bit_cast(float, (uint32_t)(127 - e) << 23);
        vs[g] *= ratio[g];
      }
      widest = fmaxf(widest, w * ratio[g]);
    }
    return true;
  };
  // O^T += V^T . P^T for the channels of group g
  auto multiply_v = [&](int g, const Raw<D, NG>& r, const u32x4 (&hi)[CB], const u32x4 (&lo)[CB]) INLINE {
#pragma unroll
    for (int j = g * GT; j < (g + 1) * GT; ++j) {
      const int h = j / 4, n = j % 4;
      uint32_t w[4] = {r.v[0][2 * h], r.v[0][2 * h + 1], r.v[1][2 * h], r.v[1][2 * h + 1]};
      if (n >= 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] >>= 8;
      }
      const u32x4 v = n & 1 ? u32x4{u.odd(w[0]), u.odd(w[1]), u.odd(w[2]), u.odd(w[3])}
                            : u32x4{u.even(w[0]), u.even(w[1]), u.even(w[2]), u.even(w[3])};
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) {
        o[cb][j] = mfma(n & 1 ? neg1 : neg0, hi[cb], o[cb][j]);
        o[cb][j] = mfma(v, hi[cb], o[cb][j]);
        if constexpr (!IS_BF16) {
          o[cb][j] = mfma(n & 1 ? neg1 : neg0, lo[cb], o[cb][j]);
          o[cb][j] = mfma(v, lo[cb], o[cb][j]);
        }
      }
    }
  };
  // the rest of a block, its parameters in LDS (R = 0)
  auto by_columns = [&](auto careful, int n0, bool there0, bool there1, const Raw<D, NG>& r, const uint32_t (&param)[NG],
                        float widest, auto after_k) INLINE -> bool {
    constexpr bool CAREFUL = decltype(careful)::value;
    // ---- scores of token n0 + 16 t + 4 lg + i, column li of each block: sum(q value), still to be times qk
    float sc[CB][8];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f32x4 acc[CB];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const u32x4 kp = *(const u32x4*)&params[0][g][16 * t + 4 * lg];
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) acc[cb] = c0[cb][g];
#pragma unroll
        for (int s = g * GS; s < (g + 1) * GS; ++s) {
          const uint32_t w = r.k[t][s], w8 = w >> 8;
          const u32x4 k = u32x4{u.even(w), u.odd(w), u.even(w8), u.odd(w8)};
#pragma unroll
          for (int cb = 0; cb < CB; ++cb) acc[cb] = mfma(k, q[cb][s], acc[cb]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float s = scale_of<IS_BF16>(kp[i]), low = low_of<IS_BF16>(kp[i]);
#pragma unroll
          for (int cb = 0; cb < CB; ++cb) {
            const float first = g == 0 ? low * qsum[cb][g] : __builtin_fmaf(low, qsum[cb][g], sc[cb][4 * t + i]);
            sc[cb][4 * t + i] = __builtin_fmaf(s, acc[cb][i], first);
          }
        }
      }
    }
    after_k();
    if (CAREFUL && a.soft_cap > 0.f) {
#pragma unroll
      for (int cb = 0; cb < CB; ++cb)
#pragma unroll
        for (int i = 0; i < 8; ++i) sc[cb][i] = LOG2E * capped(qk[cb] * sc[cb][i], a.soft_cap, a.inv_cap);
    }
    float x_mul[CB];
    uint32_t seen[CB];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) x_mul[cb] = CAREFUL && a.soft_cap > 0.f ? 1.f : qk[cb], seen[cb] = 255u;
    if (CAREFUL) {
#pragma unroll
      for (int cb = 0; cb < CB; ++cb)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int tok = n0 + 16 * (i >> 2) + 4 * lg + (i & 3);
          const bool see = (i < 4 ? there0 : there1) && tok < min(limit[cb], end);
          sc[cb][i] = see ? sc[cb][i] : -INFINITY;
          if (!see) seen[cb] &= ~(1u << i);
        }
    }
    // ---- the references: P times a scale stays below 2^MOST (fp16), with as much room below for the small ones
    const float wide = log2_fast(widest);
    bool raise = false;
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      float top = sc[cb][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) top = fmaxf(top, sc[cb][i]);
      raise |= __builtin_fmaf(top, x_mul[cb], wide) > m[cb] + MOST;
    }
    if (__any(raise)) {
      float ratio[NG];
      if (!rescale(careful, param, ratio, widest)) return false;
      const float now = log2_fast(widest);
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) {
        float top = sc[cb][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) top = fmaxf(top, sc[cb][i]);
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float at = __builtin_fmaf(top, x_mul[cb], now);
        const float to = at > m[cb] + MOST ? at - AT : m[cb];
        const float f = exp2_fast(m[cb] - to);
        m[cb] = to;
        l[cb] *= f;
#pragma unroll
        for (int g = 0; g < NG; ++g) corr[cb][g] *= f;
#pragma unroll
        for (int j = 0; j < NT; ++j) o[cb][j] *= f * ratio[j / GT];
      }
    }
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sc[cb][i] = exp2_fast(__builtin_fmaf(sc[cb][i], x_mul[cb], -m[cb]));      // P from here on
        l[cb] += sc[cb][i];
      }
    // ---- O^T += V^T . P^T, group by group
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float sv[8], low[8];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const u32x4 vp = *(const u32x4*)&params[1][g][16 * t + 4 * lg];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sv[4 * t + i] = scale_of<IS_BF16>(vp[i]);
          low[4 * t + i] = low_of<IS_BF16>(vp[i]);
        }
      }
      if (CAREFUL) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sv[i] *= vs[g];
      }
      u32x4 hi[CB], lo[CB];
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          float s2[2], c2[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) s2[k] = sc[cb][i + k] * sv[i + k], c2[k] = sc[cb][i + k] * low[i + k];
          if (CAREFUL) {                      // 0 times the NaN of a token that only other columns see
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const bool see = seen[cb] >> (i + k) & 1;
              s2[k] = see ? s2[k] : 0.f, c2[k] = see ? c2[k] : 0.f;
            }
          }
          corr[cb][g] += c2[0];
          corr[cb][g] += c2[1];
          typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
          const f16x2 h = f16x2{(_Float16)s2[0], (_Float16)s2[1]};
          hi[cb][i / 2] = __builtin_bit_cast(uint32_t, h);
          if constexpr (!IS_BF16) {
            const f16x2 rest = f16x2{(_Float16)(s2[0] - (float)h[0]), (_Float16)(s2[1] - (float)h[1])};
            lo[cb][i / 2] = __builtin_bit_cast(uint32_t, rest);
          }
        }
      }
      multiply_v(g, r, hi, lo);
    }
    return true;
  };
  // the same for R > 0
  auto by_tokens = [&](auto careful, int n0, bool there0, bool there1, const Raw<D, NG>& r, const uint32_t (&param)[NG],
                       float widest, auto after_k) INLINE -> bool {
    constexpr bool CAREFUL = decltype(careful)::value;
    // ---- scores of token n0 + 16 t + li, column lg R + i
    float sc[2][W];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint32_t kp = params[0][g][16 * t + li];
        f32x4 acc = c0[0][g];
#pragma unroll
        for (int s = g * GS; s < (g + 1) * GS; ++s) {
          const uint32_t w = r.k[t][s], w8 = w >> 8;
          acc = mfma(q[0][s], u32x4{u.even(w), u.odd(w), u.even(w8), u.odd(w8)}, acc);
        }
        const float s = scale_of<IS_BF16>(kp), low = low_of<IS_BF16>(kp);
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const float first = g == 0 ? low * qsum[i][g] : __builtin_fmaf(low, qsum[i][g], sc[t][i]);
          sc[t][i] = __builtin_fmaf(s, acc[i], first);
        }
      }
    }
    after_k();
    if (CAREFUL && a.soft_cap > 0.f) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < W; ++i) sc[t][i] = LOG2E * capped(qk[i] * sc[t][i], a.soft_cap, a.inv_cap);
    }
    float x_mul[W];
    bool seen[2][W];
#pragma unroll
    for (int i = 0; i < W; ++i) {
      x_mul[i] = CAREFUL && a.soft_cap > 0.f ? 1.f : qk[i];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        seen[t][i] = !CAREFUL || ((t ? there1 : there0) && n0 + 16 * t + li < min(limit[i], end));
        if (CAREFUL) sc[t][i] = seen[t][i] ? sc[t][i] : -INFINITY;
      }
    }
    const float wide = log2_fast(widest);
    bool raise = false;
#pragma unroll
    for (int i = 0; i < W; ++i) raise |= __builtin_fmaf(fmaxf(sc[0][i], sc[1][i]), x_mul[i], wide) > m[i] + MOST;
    if (__any(raise)) {
      float ratio[NG];
      if (!rescale(careful, param, ratio, widest)) return false;
      const float now = log2_fast(widest);
      float f[W];
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const float top = over_row(fmaxf(sc[0][i], sc[1][i]), [](float a, float b) { return fmaxf(a, b); });
        const float at = __builtin_fmaf(top, x_mul[i], now);
        const float to = at > m[i] + MOST ? at - AT : m[i];
        f[i] = exp2_fast(m[i] - to);
        m[i] = to;
        l[i] *= f[i];
#pragma unroll
        for (int g = 0; g < NG; ++g) corr[i][g] *= f[i];
      }
      const float mine = of_column(f);
#pragma unroll
      for (int j = 0; j < NT; ++j) o[0][j] *= mine * ratio[j / GT];
    }
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        sc[t][i] = exp2_fast(__builtin_fmaf(sc[t][i], x_mul[i], -m[i]));        // P from here on
        l[i] += sc[t][i];
      }
    // P to the order in which V's tokens are contracted: token 4 g + k of tile t is element 8 g + 4 t + k
    uint16_t(*const ps)[IS_BF16 ? 1 : 2][R > 0 ? 4 * R : 1][32] = s_p[R > 0 ? wave : 0];
    const int put = (li >> 2) * 8 + (li & 3), column = li & (4 * W - 1);
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint32_t vp = params[1][g][16 * t + li];
        float sv = scale_of<IS_BF16>(vp);
        const float low = low_of<IS_BF16>(vp);
        if (CAREFUL) sv *= vs[g];
#pragma unroll
        for (int i = 0; i < W; ++i) {
          float s1 = sc[t][i] * sv, c1 = sc[t][i] * low;
          if (CAREFUL) s1 = seen[t][i] ? s1 : 0.f, c1 = seen[t][i] ? c1 : 0.f;
          corr[i][g] += c1;
          const _Float16 h = (_Float16)s1;
          ps[g][0][lg * W + i][put + 4 * t] = __builtin_bit_cast(uint16_t, h);
          if constexpr (!IS_BF16) ps[g][1][lg * W + i][put + 4 * t] = __builtin_bit_cast(uint16_t, (_Float16)(s1 - (float)h));
        }
      }
    lanes_meet();
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      u32x4 hi[CB], lo[CB];
      hi[0] = *(const u32x4*)&ps[g][0][column][8 * lg];
      if constexpr (!IS_BF16) lo[0] = *(const u32x4*)&ps[g][1][column][8 * lg];
      multiply_v(g, r, hi, lo);
    }
    return true;
  };
  // CAREFUL: the block has tokens that are not there or not seen by every column, the scores are capped, or V's scales are
  // brought near 1.  Without it the block is straight code but for the one branch on the references; false: nothing has been
  // done, the block needs care.  after_k() is called when K's registers are free.
  auto compute_as = [&](auto careful, int n0, bool there0, bool there1, const Raw<D, NG>& r, auto after_k) INLINE -> bool {
    constexpr bool CAREFUL = decltype(careful)::value;
    // ---- the block's widest V scale; the parameters of tokens that are not there may hold anything
    uint32_t param[NG];
    float widest = 0x1p-20f;
#pragma unroll
    for (int g = 0; g < NG; ++g) param[g] = r.params[g];
    if (CAREFUL) {
      const bool live = (lane & 16 ? there1 : there0) && n0 + (lane & 31) < end;
#pragma unroll
      for (int g = 0; g < NG; ++g) param[g] = live ? param[g] : 0u;
    }
    lanes_meet();                       // (the block before)
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      params[lane >> 5][g][lane & 31] = param[g];
      widest = fmaxf(widest, CAREFUL ? scale_of<IS_BF16>(param[g]) * vs[g] : scale_of<IS_BF16>(param[g]));
    }
    lanes_meet();
    widest = max_upper_half(widest);
    if constexpr (R > 0) {
      return by_tokens(careful, n0, there0, there1, r, param, widest, after_k);
    } else {
      return by_columns(careful, n0, there0, there1, r, param, widest, after_k);
    }
  };
  // A wave's blocks are 128 tokens apart.  RING of them are in flight: while one is multiplied the next ones are on their way,
  // and the pages of the one behind them are looked up.  With RING 1 the next block's K is fetched into the registers of this
  // one's as soon as the scores are there, and V after the products: where two column blocks need the registers.  Plain blocks
  // first; from the first one that needs care on, all of them get it.
  int n0 = start + 32 * wave;
  if (n0 < end) {
    fetch_q();
    constexpr int RING = ring_of(D, CB);
    Raw<D, NG> ring[RING];
    bool there[RING];
    auto nothing = [] {};
    const int plain_end = a.soft_cap > 0.f ? 0 : min(full, end);
    if constexpr (RING == 1) {
      Where w = lookup(n0);
      load(w, ring[0]);
      there[0] = w.there[0] && w.there[1];
      w = lookup(n0 + 128);
      prepare_q();
      while (n0 + 32 <= plain_end && there[0]) {
        if (!compute_as(std::false_type{}, n0, true, true, ring[0], [&]() INLINE { load_k(w, ring[0]); })) break;
        load_v(w, ring[0]);                   // (behind the last block: the last tile's page once more)
        there[0] = w.there[0] && w.there[1];
        w = lookup(n0 + 256);
        n0 += 128;
      }
    } else {
#pragma unroll
      for (int i = 0; i < RING - 1; ++i) {
        const Where w = lookup(n0 + 128 * i);
        load(w, ring[i]);
        there[i] = w.there[0] && w.there[1];
      }
      there[RING - 1] = false;
      Where ahead = lookup(n0 + 128 * (RING - 1));
      prepare_q();
      auto plain = [&](auto slot) INLINE -> bool {
        constexpr int I = decltype(slot)::value, AHEAD = (I + RING - 1) % RING;
        if (n0 + 32 > plain_end || !there[I]) return false;
        load(ahead, ring[AHEAD]);
        there[AHEAD] = ahead.there[0] && ahead.there[1];
        ahead = lookup(n0 + 128 * RING);
        if (!compute_as(std::false_type{}, n0, true, true, ring[I], nothing)) return false;
        n0 += 128;
        return true;
      };
      for (;;) {
        if (!plain(std::integral_constant<int, 0>{})) break;
        if (!plain(std::integral_constant<int, 1>{})) break;
        if constexpr (RING > 2) {
          if (!plain(std::integral_constant<int, 2>{})) break;
        }
      }
    }
    if (n0 < end) {
      Raw<D, NG> r, next;
      Where w = lookup(n0);
      load(w, r);
      bool there0 = w.there[0], there1 = w.there[1];
      w = lookup(n0 + 128);
      for (;;) {
        load(w, next);
        const bool next0 = w.there[0], next1 = w.there[1];
        w = lookup(n0 + 256);
        compute_as(std::true_type{}, n0, there0, there1, r, nothing);
        n0 += 128;
        if (n0 >= end) break;
        r = next, there0 = next0, there1 = next1;
      }
    }
  }

  // ---- merge: one column's sums are spread over the four lane groups, then over the four waves
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    float low_sum[NG];                        // of column li
    if (cb) __syncthreads();
    if constexpr (R == 0) {
      l[cb] += __shfl_xor(l[cb], 16);
      l[cb] += __shfl_xor(l[cb], 32);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        low_sum[g] = corr[cb][g] + __shfl_xor(corr[cb][g], 16);
        low_sum[g] += __shfl_xor(low_sum[g], 32);
      }
      if (lg == 0) s_m[wave][li] = m[cb], s_l[wave][li] = l[cb];
    } else {
      auto add = [](float a, float b) { return a + b; };
#pragma unroll
      for (int i = 0; i < W; ++i) {
        l[i] = over_row(l[i], add);
        if (li == 0) s_m[wave][lg * W + i] = m[i], s_l[wave][lg * W + i] = l[i];
      }
      if (lg == 0 && li >= 4 * W) s_m[wave][li] = NONE, s_l[wave][li] = 0.f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float v[W];
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = over_row(corr[i][g], add);
        low_sum[g] = of_column(v);
      }
    }
    __syncthreads();
    // thread (column mc, part): channels part * 4 + 64 i of that column
    const int mc = threadIdx.x >> 4, part = threadIdx.x & 15;
    const int mcol = col0 + cb * 16 + mc;
    const float m_all = fmaxf(fmaxf(s_m[0][mc], s_m[1][mc]), fmaxf(s_m[2][mc], s_m[3][mc]));
    float f[4], l_all = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      f[w] = exp2_fast(s_m[w][mc] - m_all);
      l_all += s_l[w][mc] * f[w];
    }
    const float inv = l_all != 0.f ? 1.f / l_all : 0.f;
    const float lse = l_all != 0.f ? m_all + log2_fast(l_all) : -INFINITY;
    const int ms = one ? 0 : mcol / group, mh = kvh * group + (mcol - ms * group);
    const long long row = ((long long)b * a.S + ms) * a.q_heads + mh;
    float* prow = a.partial + (row * a.splits + split) * D;
#pragma unroll
    for (int d0 = 0; d0 < D; d0 += DC) {
      if (d0) __syncthreads();
#pragma unroll
      for (int j = d0 / 16; j < (d0 + DC) / 16; ++j) {
        f32x4 v = o[cb][j];
        const float undo = 1.f / vs[j / GT];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __builtin_fmaf(v[i], undo, low_sum[j / GT]);
        *(f32x4*)&s_o[wave][li][(j - d0 / 16) * 16 + 4 * lg] = v;
      }
      __syncthreads();
      if (mcol < columns && mc < COLUMNS) {
#pragma unroll
        for (int i = 0; i < DC / 64; ++i) {
          const int ch = part * 4 + 64 * i;
          f32x4 r = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int w = 0; w < 4; ++w) r += *(const f32x4*)&s_o[w][mc][ch] * f[w];
          r *= inv;
          if (a.splits > 1) {
            *(f32x4*)(prow + d0 + ch) = r;
          } else if (a.out_mode == 2) {
#pragma unroll
            for (int k = 0; k < 4; ++k) ((float*)a.out)[row * (D + 1) + d0 + ch + k] = r[k];
          } else {
            const uint2 v = uint2{to16<IS_BF16>(r[0]) | to16<IS_BF16>(r[1]) << 16, to16<IS_BF16>(r[2]) | to16<IS_BF16>(r[3]) << 16};
            *(uint2*)((uint16_t*)a.out + row * D + d0 + ch) = v;
          }
        }
      }
    }
    if (mcol < columns && mc < COLUMNS && part == 0) {
      if (a.splits > 1) a.partial_lse[row * a.splits + split] = lse;
      else if (a.out_mode == 2) ((float*)a.out)[row * (D + 1) + D] = lse * LN2;
    }
  }
}

constexpr int FEW_SPLITS = 8;

// One workgroup merges the splits of one row.  D / 4 lanes hold a split's sums, so 1024 / D splits are read at a time; eight
// rounds of loads are issued before the first is used (64 splits of 128 channels: one trip to memory).
template <bool IS_BF16, int D>
__global__ __launch_bounds__(256) void kv4_merge_kernel(const float* __restrict__ partial, const float* __restrict__ lse, int splits,
                                                        void* __restrict__ out, int out_mode) {
  constexpr int LANES = D / 4, AT_ONCE = 256 / LANES, ROUNDS = 8;
  __shared__ __attribute__((aligned(16))) float s_acc[AT_ONCE][D];
  const long long row = blockIdx.x;
  const int lane = threadIdx.x & 63, c4 = threadIdx.x % LANES, first = threadIdx.x / LANES;
  const float* l = lse + row * splits;
  const float* sums = partial + row * splits * D + c4 * 4;
  f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
  float top = -INFINITY, sum = 0.f;
  for (int s0 = 0; s0 < splits; s0 += AT_ONCE * ROUNDS) {
    f32x4 v[ROUNDS];
    float mine[ROUNDS];
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
      const int s = s0 + first + AT_ONCE * i;
      v[i] = *(const f32x4*)(sums + (long long)min(s, splits - 1) * D);
      mine[i] = s < splits ? l[s] : -INFINITY;
    }
    float peak = top;                     // over all of this pass's splits: every lane reads some of them
    for (int s = s0 + lane; s < min(splits, s0 + AT_ONCE * ROUNDS); s += 64) peak = fmaxf(peak, l[s]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) peak = fmaxf(peak, __shfl_xor(peak, o));
    // As long as no split has had a token (or only NaN, which the weights keep), what is subtracted is 0, but `top` stays where
    // it is: a 0 kept there would be the reference of all later passes, however far below it their sums are.
    const float from = peak == -INFINITY ? 0.f : peak;
    const float f = exp2_fast(top - from);
    sum *= f;
    acc *= f;
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
      const float w = exp2_fast(mine[i] - from);
      sum += w;
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[k] += w != 0.f ? w * v[i][k] : 0.f;      // (a split without tokens has written no sums)
    }
    top = peak;
  }
  *(f32x4*)&s_acc[first][c4 * 4] = acc;
  __shared__ float s_sum[AT_ONCE];
  if (c4 == 0) s_sum[first] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < AT_ONCE; ++i) sum += s_sum[i];
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  for (int c = threadIdx.x; c < D; c += 256) {
    float r = 0.f;
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) r += s_acc[i][c];
    r *= inv;
    if (out_mode == 2) ((float*)out)[row * (D + 1) + c] = r;
    else ((uint16_t*)out)[row * D + c] = to16<IS_BF16>(r);
  }
  if (out_mode == 2 && threadIdx.x == 0)
    ((float*)out)[row * (D + 1) + D] = sum != 0.f ? (top + log2_fast(sum)) * 0.6931471805599453f : -INFINITY;
}

// The same for few splits: D / 4 lanes take a row, a workgroup 1024 / D rows, and all splits are read at once.  32768 rows of 2
// splits, 128 channels: 8.4 us (42 MB, 5.0 TB/s) where a workgroup for each row takes 50.
template <bool IS_BF16, int D>
__global__ __launch_bounds__(256) void kv4_merge_few_kernel(const float* __restrict__ partial, const float* __restrict__ lse, int splits,
                                                            long long rows, void* __restrict__ out, int out_mode) {
  constexpr int LANES = D / 4, AT_ONCE = FEW_SPLITS;
  const long long row = (long long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  if (row >= rows) return;
  const int c = threadIdx.x % LANES * 4;
  f32x4 v[AT_ONCE];
  float w[AT_ONCE], top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int s = 0; s < AT_ONCE; ++s) {
    w[s] = s < splits ? lse[row * splits + s] : -INFINITY;
    if (s < splits) v[s] = *(const f32x4*)(partial + (row * splits + s) * D + c);
    top = fmaxf(top, w[s]);
  }
  if (top == -INFINITY) top = 0.f;        // no split has a token (or what they have is NaN, which the weights keep)
  f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < AT_ONCE; ++s) {
    w[s] = exp2_fast(w[s] - top);
    sum += w[s];
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] += w[s] != 0.f ? w[s] * v[s][k] : 0.f;    // (a split without tokens has written no sums)
  }
  acc *= sum != 0.f ? 1.f / sum : 0.f;
  if (out_mode == 2) {
    float* to = (float*)out + row * (D + 1);
#pragma unroll
    for (int k = 0; k < 4; ++k) to[c + k] = acc[k];
    if (c == 0) to[D] = sum != 0.f ? (top + log2_fast(sum)) * 0.6931471805599453f : -INFINITY;
  } else {
    *(uint2*)((uint16_t*)out + row * D + c) =
        uint2{to16<IS_BF16>(acc[0]) | to16<IS_BF16>(acc[1]) << 16, to16<IS_BF16>(acc[2]) | to16<IS_BF16>(acc[3]) << 16};
  }
}

template <class Fn>
bool dispatch(int dtype, int D, int G, Fn&& fn) {
  auto typed = [&](auto d, auto g) {
    if (dtype == 0) fn(std::true_type{}, d, g); else fn(std::false_type{}, d, g);
    return true;
  };
#define TDIST_KV4_CASE(DD, GG) \
  if (D == DD && G == GG) return typed(std::integral_constant<int, DD>{}, std::integral_constant<int, GG>{});
  TDIST_KV4_CASE(64, 32) TDIST_KV4_CASE(64, 64)
  TDIST_KV4_CASE(128, 32) TDIST_KV4_CASE(128, 64) TDIST_KV4_CASE(128, 128)
  TDIST_KV4_CASE(256, 32) TDIST_KV4_CASE(256, 64) TDIST_KV4_CASE(256, 128)
#undef TDIST_KV4_CASE
  return false;
}

}  // namespace

// partial (splits > 1): batch * S * q_heads * splits * (head_dim + 1) floats.
// out_mode 1: out [batch, S, q_heads, D] in q's type; 2: fp32 [batch, S, q_heads, D + 1], natural-log LSE last.
// flags (or null): what tdist_kv4_chunk, run before with the same arguments, has left undone; only that is done here, and the merge.
TDIST_API int tdist_kv4_attn(const void* k_codes, const void* v_codes, const void* k_params, const void* v_params, int pages,
                             int kv_heads, int page_size, int head_dim, int group, const void* q, long long q_sb, long long q_ss,
                             long long q_sh, const int* table, int table_stride, int max_pages, const int* kv_len, float* partial,
                             void* out, int batch, int S, int q_heads, int splits, int causal, int out_mode, float scale,
                             float soft_cap, int dtype, const int* flags, int flag_columns, void* stream) {
  AttnArgs a;
  a.c = Cache{(uint8_t*)k_codes, (uint8_t*)v_codes, (uint32_t*)k_params, (uint32_t*)v_params, pages, kv_heads, page_size};
  TDIST_REQUIRE(k_codes && v_codes && k_params && v_params && pages > 0 && kv_heads > 0 && page_size > 0 && page_size % 16 == 0 &&
                    (((uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_params | (uintptr_t)v_params) & 15) == 0,
                "a 4-bit cache needs four 16-byte aligned tensors, pages of a multiple of 16 tokens");
  TDIST_REQUIRE(batch >= 0 && S >= 0 && q_heads > 0 && q_heads % kv_heads == 0 && max_pages >= 0 &&
                    (long long)max_pages * page_size <= (1ll << 30), "bad head counts, or more than 2^30 tokens in a row of the table");
  TDIST_REQUIRE(splits >= 1 && splits <= 65535 && (splits == 1 || partial), "splits need their partial rows");
  TDIST_REQUIRE(!flags || (flag_columns > 0 && flag_columns % 32 == 0), "flags are for blocks of a multiple of 32 columns");
  TDIST_REQUIRE((out_mode == 1 || out_mode == 2) && (dtype == 0 || dtype == 1), "out_mode must be 1 or 2, dtype 0 (bf16) or 1 (fp16)");
  if (batch == 0 || S == 0) return 0;
  TDIST_REQUIRE(q && (table || max_pages == 0) && kv_len && out, "null argument");
  TDIST_REQUIRE(((uintptr_t)q & 15) == 0 && ((uintptr_t)out & 7) == 0 && ((q_sb | q_ss | q_sh) & 7) == 0,
                "q rows must keep 16-byte alignment");
  const long long columns = (long long)(q_heads / kv_heads) * S;
  const long long per_group = columns <= 4 ? 4 : columns <= 8 ? 8 : columns > 16 && head_dim <= 128 ? 32 : 16;
  const long long blocks = (columns + per_group - 1) / per_group * batch;
  TDIST_REQUIRE(blocks < (1ll << 31) && columns < (1ll << 30) && (long long)batch * S * q_heads < (1ll << 31), "too many query rows");
  a.q = (const uint16_t*)q, a.partial = partial, a.out = out;
  a.page_tiles = page_size / 16;
  a.page_magic = a.page_tiles == 1 ? 0u : (uint32_t)((1ull << 32) / a.page_tiles) + 1u;
  a.partial_lse = partial ? partial + (long long)batch * S * q_heads * splits * head_dim : nullptr;
  a.q_sb = q_sb, a.q_ss = q_ss, a.q_sh = q_sh, a.table_stride = table_stride, a.max_pages = max_pages;
  a.batch = batch, a.S = S, a.q_heads = q_heads, a.group = q_heads / kv_heads, a.splits = splits, a.causal = causal, a.out_mode = out_mode;
  a.scale = scale, a.soft_cap = soft_cap, a.inv_cap = std::min(1.f / soft_cap, 1e38f), a.flags = flags, a.flag_columns = flag_columns;
  const bool ok = dispatch(dtype, head_dim, group, [&](auto bf, auto d, auto g) {
    auto launch = [&](auto kernel) {
      for (a.first = 0; a.first < blocks; a.first += 65535)       // (the limit of a grid's third dimension)
        hipLaunchKernelGGL(kernel, dim3(kv_heads, splits, (unsigned)std::min(65535ll, blocks - a.first)), dim3(256), 0,
                           (hipStream_t)stream, a, table, kv_len);
    };
    constexpr bool BF = decltype(bf)::value;
    constexpr int D = decltype(d)::value, G = decltype(g)::value;
    if constexpr (D <= 128) {
      if (per_group == 32) return launch(kv4_attn_kernel<BF, D, G, 2>);
    }
    if (per_group == 4) launch(kv4_attn_kernel<BF, D, G, 1, 1>);
    else if (per_group == 8) launch(kv4_attn_kernel<BF, D, G, 1, 2>);
    else launch(kv4_attn_kernel<BF, D, G, 1>);
  });
  TDIST_REQUIRE(ok, "head_dim 64 / 128 / 256 with groups of 32 / 64 / 128 channels (at most head_dim)");
  TDIST_HIP_TRY(hipGetLastError());
  if (splits == 1) return 0;
  const long long rows = (long long)batch * S * q_heads;
  dispatch(dtype, head_dim, group, [&](auto bf, auto d, auto) {
    constexpr int per_block = 1024 / decltype(d)::value;
    if (splits <= FEW_SPLITS) {
      hipLaunchKernelGGL((kv4_merge_few_kernel<decltype(bf)::value, decltype(d)::value>), dim3((unsigned)((rows + per_block - 1) / per_block)),
                         dim3(256), 0, (hipStream_t)stream, a.partial, a.partial_lse, splits, rows, out, out_mode);
      return;
    }
    hipLaunchKernelGGL((kv4_merge_kernel<decltype(bf)::value, decltype(d)::value>), dim3((unsigned)rows), dim3(256), 0,
                       (hipStream_t)stream, a.partial, a.partial_lse, splits, out, out_mode);
  });
  TDIST_HIP_TRY(hipGetLastError());
  return 0;
}
