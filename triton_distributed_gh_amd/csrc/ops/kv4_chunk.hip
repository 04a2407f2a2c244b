// GQA attention over a 4-bit KV cache for many query columns (a chunk of a prompt, long drafts): what attention over a few
// columns (kv4_attn.hip) does anew for every sixteen or thirty-two of them - unpacking, a token's scale and low - is done once
// for a workgroup's columns, and handed out through LDS.
//
// A workgroup of NW waves takes one (sequence, KV head, NW x CB x 16 query columns, KV split), every wave its CB x 16 columns
// over all tokens, 64 at a time.  The waves share the work of turning the next 64 tokens' codes into fp16 values
//     value = fp16(scale * code + low)              (1024 + code or 64 + code from the bits, minus that, one fused multiply-add)
// in the order in which 16x16x32 MFMAs take them, so that a wave then reads its operands as straight 16-byte runs:
//   S^T[token, column] = K . Q^T,   P = exp2(scale log2(e) s - m) in fp16,   O^T[channel, column] = V^T . P^T,
// and the sums of P come out of one more product with ones, of the same rounded P that O is made of: what rounding does to a
// weight cancels where that weight is nearly all of the sum.  The reference m moves as in kv4_attn.hip.
//
// For bf16 caches: values rounded to fp16 are within 2^-11 of themselves (but for small ones, see below) and a weight within 2^-11,
// where the result is rounded to 2^-8; 1024 tokens over 16384 are 1.9e-3 off at most with it and with the plain form in 32 bits
// (relative to a row's norm), at three times the scores, in groups of 32, 2.5e-3 for 2.0e-3.  A fp16 result has steps of 2^-11
// itself, and these roundings would be most of its error: 5.8e-4 for 2.7e-4, three times the scores 1.6e-3 for 2.4e-4, where
// kv4_attn.hip comes to 2.8e-4 and 2.5e-4.  So fp16 caches stay there, which costs them 740 us where this kernel took 351.
//
// fp16 does not reach as far as bf16.  Below 2^-14 its numbers are 2^-24 apart, and a value is then off by as much as 17 * 2^-25:
// a code's 15 times what the scale lost, what low lost, and the result's own rounding.  Whose group is how large against that
// is asked of every token by itself, as a row may see that token alone.
//   V: an answer's own size counts.  V is held times 2^7, which puts the numbers of trained models in the middle of fp16's range;
//      a group of less than 2^-16 and not 0 is flagged (at 2^-9 as it is held, 17 * 2^-25 are 2^-11.9 of it), one of 2^8 too.
//   K: a score's absolute error counts, the sum of scale |q| times what K is off by.  While that sum is under 2^8 for every column of the
//      workgroup (about 10 for queries of size 1), 17 * 2^-25 of it are less than 2^-12 of a nat whatever K's size.  Beyond it, groups of
//      less than 2^-9 and not 0 are flagged; groups of 2^15 always.
// (A group's size: 15 scale + |low|, one to three times its largest value.)  A NaN in a scale and a page that is none are flagged too.
// `flags` has one int per workgroup, written by every launch; kv4_attn.hip runs behind this kernel and takes just the flagged
// workgroups' columns.
//
// What bounds it: 1024 new tokens over 16384, 32 / 8 heads of 128 (266 GFLOP): 294 .. 307 us in all, 870 .. 905 TFLOP/s where a
// large bf16 matrix product reaches 1203; the other kernel takes 511.  (A dozen calls in a row: the same call after a pause, or with
// a wait for each, takes 350 .. 390 us until the card is busy again.)  Of a SIMD's cycles its matrix unit has 37 %, vector
// instructions 48 %, and two waves hardly overlap the two.  Timing-only builds of 349 us (launches apart from each other): 279
// without the unpacking, 294 without V's way back from LDS, 311 with half of the second product, 334 without the exponentials.
// Eight waves with one set of buffers against twice four: 346 and 367 us (with half the columns for a workgroup, unpacking costs
// twice as much); scores of the next 32 tokens made ahead of time from a third buffer: 348, and 99 for 77 where heads of 256 then
// need shorter blocks; all 64 tokens' scores at once spill registers; operands read ahead of the references 346.
#include <algorithm>

#include "tdist/kv4.hpp"

namespace {

using namespace tdist::kv4;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
#define INLINE __attribute__((always_inline))     // (lambdas: a call would put what they capture into memory)

struct ChunkArgs {
  Cache c;
  const uint16_t* q;        // [batch, S, q_heads, D]
  float* partial;           // splits > 1: [rows, splits, D] sums over their own weight, rows = batch * S * q_heads
  float* partial_lse;       // and [rows, splits] log2-sum-exp2 (-inf: no token)
  void* out;                // [batch, S, q_heads, D] (out_mode 1) or fp32 [.., D + 1] with the log-sum-exp (out_mode 2)
  int* flags;               // [column blocks * batch, splits, kv_heads]
  long long q_sb, q_ss, q_sh;
  int table_stride, max_pages;
  int page_tiles;           // 16-token tiles of a page,
  uint32_t page_magic;      // and floor(2^32 / page_tiles) + 1 (0: one tile a page)
  int batch, S, q_heads, group, splits, causal, out_mode;
  int first;                // of this launch's (column block, sequence) pairs
  float scale;
};

__device__ __forceinline__ f32x4 mfma(const u32x4& a, const u32x4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f16x2 both(float a, float b) { return f16x2{(_Float16)a, (_Float16)b}; }

// The masks and offsets of the unpacking, kept in registers (a literal each would keep the and-or from being one instruction)
struct Unpack {
  uint32_t m0, m1, o0, o1;
  __device__ __forceinline__ Unpack() {
    asm volatile("s_mov_b32 %0, 0x000f000f" : "=s"(m0));
    asm volatile("s_mov_b32 %0, 0x00f000f0" : "=s"(m1));
    asm volatile("v_mov_b32 %0, 0x64006400" : "=v"(o0));
    asm volatile("v_mov_b32 %0, 0x54005400" : "=v"(o1));
  }
  // nibbles n and n + 4 (n even / odd) of a dword, scaled and moved
  __device__ __forceinline__ uint32_t even(uint32_t w, f16x2 scale, f16x2 low) const {
    const f16x2 code = __builtin_bit_cast(f16x2, (w & m0) | o0) - (_Float16)1024.f;
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(code, scale, low));
  }
  __device__ __forceinline__ uint32_t odd(uint32_t w, f16x2 scale, f16x2 low) const {
    const f16x2 code = __builtin_bit_cast(f16x2, (w & m1) | o1) - (_Float16)64.f;
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(code, scale, low));
  }
};

constexpr int WAVES = 8;                // of a workgroup
template <int D>
constexpr int column_blocks() { return D <= 128 ? 2 : 1; }          // of sixteen, per wave: what its registers hold
template <int D, int NW>
constexpr int columns_of() { return 16 * column_blocks<D>() * NW; }

template <int D, int G, int NW>
__global__ __launch_bounds__(NW * 64, 2) void kv4_chunk_kernel(ChunkArgs a, const int* __restrict__ block_table,
                                                               const int* __restrict__ kv_len) {
  constexpr int CB = column_blocks<D>(), COLUMNS = columns_of<D, NW>();
  constexpr int KS = D / 32;            // MFMA steps over the head dim = dwords of a lane per K row
  constexpr int NT = D / 16;            // 16-channel tiles of V
  constexpr int NG = D / G;
  constexpr int TOK = 64;               // tokens at a time: four tiles, two pairs of them
  // K: a wave unpacks KP steps of one tile; V: 64 / VS channels of one pair, VN times
  constexpr int KPARTS = NW / 4, KP = KS / KPARTS, KG = KP * 32 > G ? KP * 32 / G : 1;
  constexpr int H = D / 64, VS = NW > 2 * H ? 2 : 1, UNITS = 2 * H * VS, VN = UNITS > NW ? UNITS / NW : 1;
  constexpr int VG = 64 / VS > G ? 64 / VS / G : 1;
  static_assert(NW % 4 == 0 && KS % KPARTS == 0 && (UNITS % NW == 0 || UNITS < NW), "");
  constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
  constexpr float NONE = -1e30f;        // the reference before the first token
  constexpr float AT = 6.f, MOST = 14.f;  // log2 of the largest P: where a new reference puts it, and where it may grow to
  constexpr float FAR = 0x1p15f, NEAR = 0x1p-9f;        // sizes, as they are held, that are flagged from there on / below
  constexpr float BOOST = 0x1p7f;       // V is held times that
  constexpr float WIDE_Q = 0x1p8f;      // sums of scale |q| for which small K is looked for
  __shared__ __attribute__((aligned(16))) u32x4 s_k[2][4][KS][64];
  __shared__ __attribute__((aligned(16))) u32x4 s_v[2][2][NT][64];
  __shared__ int s_bad, s_wide;

  const int kvh = blockIdx.x, split = blockIdx.y;
  const int z = a.first + (int)blockIdx.z;
  const int cblk = a.batch == 1 ? z : z / a.batch, b = z - cblk * a.batch;
  const int group = a.group, columns = group * a.S;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, lg = lane >> 4;
  const int block0 = cblk * COLUMNS, col0 = block0 + wave * 16 * CB;
  int* const flag = a.flags + ((long long)z * a.splits + split) * gridDim.x + kvh;

  // tokens: a column sees [0, limit), the workgroup's columns [0, len), this wave's none beyond `most`, all of them [0, plain_end)
  const long long room = (long long)a.max_pages * a.c.page_size;
  const int L = (int)min((long long)max(kv_len[b], 0), room);
  const int len = max(0, a.causal ? L - a.S + min(block0 + COLUMNS - 1, columns - 1) / group + 1 : L);
  const int per = a.splits == 1 ? len : ((len + a.splits - 1) / a.splits + 127) & ~127;
  const int start = (int)min((long long)split * per, (long long)len), end = min(len, start + per);
  const int plain_end = min(end, a.causal ? L - a.S + block0 / group + 1 : L);
  const int most = col0 >= columns ? 0 : min(end, a.causal ? L - a.S + min(col0 + 16 * CB - 1, columns - 1) / group + 1 : L);
  if (threadIdx.x == 0) s_bad = s_wide = 0;
  bool wide_q = false;

  // Q in fp16: rows are brought near 2^8 by a power of two per column, which loses nothing that a score could show
  // (numbers 2^-32 of the column's largest).  A negative scale turns Q's sign, so that larger scores are larger weights.
  int limit[CB];
  u32x4 q[CB][KS];
  float qk[CB];
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    const int col = col0 + cb * 16 + li;
    const bool col_ok = col < columns;
    const int row_s = col_ok ? col / group : 0, head = kvh * group + (col_ok ? col - row_s * group : 0);
    limit[cb] = !col_ok ? 0 : a.causal ? L - a.S + row_s + 1 : L;
    const uint16_t* qp = a.q + b * a.q_sb + row_s * a.q_ss + head * a.q_sh + lg * 8;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      q[cb][s] = u32x4{0, 0, 0, 0};
      if (col_ok) q[cb][s] = *(const u32x4*)(qp + 32 * s);
    }
    float all = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) all += fabsf(from16<true>(q[cb][s][i] & 0xffffu)) + fabsf(low_of<true>(q[cb][s][i]));
    all += __shfl_xor(all, 16);
    all += __shfl_xor(all, 32);
    wide_q |= !(all * fabsf(a.scale) < WIDE_Q);
    float mul = a.scale < 0.f ? -1.f : 1.f;
    float top = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        top = fmaxf(top, fmaxf(fabsf(from16<true>(q[cb][s][i] & 0xffffu)), fabsf(low_of<true>(q[cb][s][i]))));
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    int e = (int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127;           // top in [2^e, 2^(e+1))
    e = e < -100 ? -100 : e;
    mul *= __builtin_bit_cast(float, (uint32_t)(127 + 8 - e) << 23);
    const float back = __builtin_bit_cast(float, (uint32_t)(127 - 8 + e) << 23);
    qk[cb] = fminf(fmaxf(fabsf(a.scale * LOG2E) * back, 1e-37f), 1e37f);    // (a masked score is -inf: it stays that)
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        q[cb][s][i] = __builtin_bit_cast(uint32_t, both(from16<true>(q[cb][s][i] & 0xffffu) * mul,
                                                        low_of<true>(q[cb][s][i]) * mul));
  }

  // ---- the codes of 64 tokens on their way: where they are, and what this wave fetches of them
  const int* table = block_table + (long long)b * a.table_stride;
  const int last_tile = (end - 1) >> 4;
  bool bad = false;
  struct Spot {
    long long row0;                     // the first row of (page, KV head)
    int off;                            // the tile's first token in the page
  };
  struct Spots {
    Spot k, v[VN][2];
  };
  struct Raw {
    uint32_t k[KP], kp[KG];
    u32x2 v[VN][2];
    u32x4 vp[VN][2][VG];
  };
  // the parts that are this wave's
  const int k_tile = wave & 3, k_part = wave >> 2;
  auto v_pair = [&](int n) INLINE { return (wave + n * NW) / (H * VS) & 1; };
  auto v_h = [&](int n) INLINE { return (wave + n * NW) / VS % H; };
  auto v_sub = [&](int n) INLINE { return (wave + n * NW) % VS; };
  const bool has_v = UNITS >= NW || wave < UNITS;
  auto spot = [&](int n0, int tile_of) INLINE -> Spot {
    const int want = (n0 >> 4) + tile_of, tile = min(want, last_tile);
    uint32_t i = a.page_magic ? (uint32_t)(((uint64_t)(uint32_t)tile * a.page_magic) >> 32) : (uint32_t)tile;
    if (i * (uint32_t)a.page_tiles > (uint32_t)tile) --i;       // the quotient, or one more
    const int page = table[i];
    const bool there = page >= 0 && page < a.c.pages;
    bad |= !there;
    return Spot{((long long)(there ? page : 0) * a.c.kv_heads + kvh) * a.c.page_size, (tile - (int)i * a.page_tiles) * 16};
  };
  const bool whole = (a.page_tiles & 3) == 0;
  auto lookup = [&](int n0) INLINE -> Spots {
    Spots w;
    if (whole) {                        // 64 tokens on one page (the tiles behind the last one are read, but not taken)
      const Spot at = spot(n0, 0);
      const int first = at.off & ~(TOK - 1);
      w.k = Spot{at.row0, first + 16 * k_tile};
#pragma unroll
      for (int n = 0; n < VN; ++n)
#pragma unroll
        for (int t = 0; t < 2; ++t) w.v[n][t] = Spot{at.row0, first + 32 * v_pair(n) + 16 * t};
      return w;
    }
    w.k = spot(n0, k_tile);
#pragma unroll
    for (int n = 0; n < VN; ++n)
#pragma unroll
      for (int t = 0; t < 2; ++t) w.v[n][t] = spot(n0, 2 * v_pair(n) + t);
    return w;
  };
  const uint32_t k_lane = li * (D / 2) + lg * (D / 8) + k_part * (KP * 4), v_lane = lg * (2 * D) + li * (D / 8);
  auto load = [&](const Spots& w, Raw& r) INLINE {
    const uint8_t* kb = a.c.k_codes + (w.k.row0 + w.k.off) * (D / 2) + k_lane;
    if constexpr (KP == 1) {
      r.k[0] = *(const uint32_t*)kb;
    } else if constexpr (KP == 2) {
      const u32x2 v = *(const u32x2*)kb;
      r.k[0] = v[0], r.k[1] = v[1];
    } else {
#pragma unroll
      for (int i = 0; i < KP / 4; ++i) {
        const u32x4 v = *(const u32x4*)(kb + 16 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) r.k[4 * i + j] = v[j];
      }
    }
    const uint32_t* kp = a.c.k_params + w.k.row0 * NG + w.k.off + li;
#pragma unroll
    for (int g = 0; g < KG; ++g) r.kp[g] = kp[(long long)(k_part * KP * 32 / G + g) * a.c.page_size];
    if (has_v) {
#pragma unroll
      for (int n = 0; n < VN; ++n)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const Spot& s = w.v[n][t];
          r.v[n][t] = *(const u32x2*)(a.c.v_codes + (s.row0 + s.off) * (D / 2) + v_lane + 8 * v_h(n));
          const uint32_t* vp = a.c.v_params + s.row0 * NG + s.off + 4 * lg;
#pragma unroll
          for (int g = 0; g < VG; ++g)
            r.vp[n][t][g] = *(const u32x4*)(vp + (long long)((64 * v_h(n) + 64 / VS * v_sub(n)) / G + g) * a.c.page_size);
        }
    }
  };
  const Unpack u;
  float near_k = 0.f;                   // K below this and not 0 is flagged
  auto unpack = [&](int buf, int n0, Raw& r) INLINE {
    if (n0 + TOK > end) {               // tokens behind the end: zeros, whatever the page holds there
      const bool live = n0 + 16 * k_tile + li < end;
#pragma unroll
      for (int g = 0; g < KG; ++g) r.kp[g] = live ? r.kp[g] : 0u;
#pragma unroll
      for (int n = 0; n < VN; ++n)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int g = 0; g < VG; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              r.vp[n][t][g][i] = n0 + 32 * v_pair(n) + 16 * t + 4 * lg + i < end ? r.vp[n][t][g][i] : 0u;
    }
    f16x2 scale[KG], low[KG];
#pragma unroll
    for (int g = 0; g < KG; ++g) {
      const float s = scale_of<true>(r.kp[g]), l = low_of<true>(r.kp[g]);
      const float size = __builtin_fmaf(15.f, s, fabsf(l));
      bad |= !(size < FAR) | (size < near_k & size > 0.f);
      scale[g] = both(s, s), low[g] = both(l, l);
    }
#pragma unroll
    for (int s = 0; s < KP; ++s) {
      constexpr int per_group = G / 32;
      const int g = s / per_group;
      const uint32_t w = r.k[s], w8 = w >> 8;
      s_k[buf][k_tile][k_part * KP + s][lane] = u32x4{u.even(w, scale[g], low[g]), u.odd(w, scale[g], low[g]),
                                                      u.even(w8, scale[g], low[g]), u.odd(w8, scale[g], low[g])};
    }
    if (has_v) {
#pragma unroll
      for (int n = 0; n < VN; ++n) {
        f16x2 sv[VG][4], lv[VG][4];     // of tokens 4 lg + 2 (k & 1), + 1 of tile k >> 1
#pragma unroll
        for (int g = 0; g < VG; ++g) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float s[2], l[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t p = r.vp[n][k >> 1][g][2 * (k & 1) + i];
              s[i] = scale_of<true>(p) * BOOST, l[i] = low_of<true>(p) * BOOST;
              const float size = __builtin_fmaf(15.f, s[i], fabsf(l[i]));
              bad |= !(size < FAR) | (size < NEAR & size > 0.f);
            }
            sv[g][k] = both(s[0], s[1]), lv[g][k] = both(l[0], l[1]);
          }
        }
        const u32x2 v0 = r.v[n][0], v1 = r.v[n][1];
        uint32_t w[4] = {v0[0], v0[1], v1[0], v1[1]};
        if constexpr (VS == 2) {
          const int by = 8 * v_sub(n);
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] >>= by;
        }
        u32x4* const to = &s_v[buf][v_pair(n)][4 * v_h(n) + 4 / VS * v_sub(n)][lane];
#pragma unroll
        for (int i = 0; i < 4 / VS; ++i) {
          const int g = 16 * i / G;
          u32x4 v;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            v[k] = i & 1 ? u.odd(i >= 2 ? w[k] >> 8 : w[k], sv[g][k], lv[g][k]) : u.even(i >= 2 ? w[k] >> 8 : w[k], sv[g][k], lv[g][k]);
          to[64 * i] = v;
        }
      }
    }
  };

  float m[CB];
  f32x4 o[CB][NT], l[CB];
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    m[cb] = NONE, l[cb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NT; ++j) o[cb][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  u32x4 ones;
#pragma unroll
  for (int i = 0; i < 4; ++i) ones[i] = 0x3c003c00u;

  // MASKED: some column does not see some of the 32 tokens of pair p
  auto compute = [&](auto masked, int buf, int p, int n0) INLINE {
    float sc[CB][8];                    // of token n0 + 16 (i / 4) + 4 lg + i % 4, column li of each block
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f32x4 acc[CB];
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) acc[cb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const u32x4 k = s_k[buf][2 * p + t][s][lane];
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) acc[cb] = mfma(k, q[cb][s], acc[cb]);
      }
#pragma unroll
      for (int cb = 0; cb < CB; ++cb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sc[cb][4 * t + i] = acc[cb][i];
          if (decltype(masked)::value && n0 + 16 * t + 4 * lg + i >= min(limit[cb], end)) sc[cb][4 * t + i] = -INFINITY;
        }
    }
    float top[CB];
    bool raise = false;
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      top[cb] = sc[cb][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) top[cb] = fmaxf(top[cb], sc[cb][i]);
      raise |= top[cb] * qk[cb] > m[cb] + MOST;
    }
    if (__any(raise)) {
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) {
        float t = fmaxf(top[cb], __shfl_xor(top[cb], 16));
        t = fmaxf(t, __shfl_xor(t, 32)) * qk[cb];
        const float to = t > m[cb] + MOST ? t - AT : m[cb];
        const float f = __builtin_amdgcn_exp2f(m[cb] - to);
        m[cb] = to;
        l[cb] *= f;
#pragma unroll
        for (int j = 0; j < NT; ++j) o[cb][j] *= f;
      }
    }
    u32x4 w[CB];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[cb][2 * i], qk[cb], -m[cb]));
        const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[cb][2 * i + 1], qk[cb], -m[cb]));
        w[cb][i] = __builtin_bit_cast(uint32_t, both(x, y));
      }
      l[cb] = mfma(ones, w[cb], l[cb]);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const u32x4 v = s_v[buf][p][j][lane];
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) o[cb][j] = mfma(v, w[cb], o[cb][j]);
    }
  };

  // Two buffers: while one block of 64 is multiplied the next one is written, and the codes of the one behind it are on their
  // way.  Every wave takes every block, so all of them meet at every barrier.
  if (start < end) {
    Raw raw;
    load(lookup(start), raw);
    __syncthreads();                    // (s_bad, s_wide are 0)
    if (__any(wide_q) && lane == 0) s_wide = 1;
    __syncthreads();
    near_k = s_wide ? NEAR : 0.f;
    unpack(0, start, raw);
    load(lookup(start + TOK), raw);     // (behind the last block: its last tile's page once more)
    Spots next = lookup(start + 2 * TOK);
    __syncthreads();
    int buf = 0, n0 = start;
    auto ahead = [&]() INLINE {
      unpack(buf ^ 1, n0 + TOK, raw);
      load(next, raw);
      next = lookup(n0 + 3 * TOK);
    };
    // what all columns see, then the rest
    for (; n0 + TOK <= plain_end; n0 += TOK, buf ^= 1) {
      ahead();
      compute(std::false_type{}, buf, 0, n0);
      compute(std::false_type{}, buf, 1, n0 + 32);
      __syncthreads();
    }
    for (; n0 < end; n0 += TOK, buf ^= 1) {
      ahead();
      if (n0 < most) {
        compute(std::true_type{}, buf, 0, n0);
        compute(std::true_type{}, buf, 1, n0 + 32);
      }
      __syncthreads();
    }
    if (__any(bad) && lane == 0) s_bad = 1;
  }
  __syncthreads();
  const int is_bad = s_bad;
  if (threadIdx.x == 0) *flag = is_bad;
  if (is_bad) return;

#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    const int col = col0 + cb * 16 + li, row_s = col / group;
    if (col >= columns) continue;
    const long long at = ((long long)b * a.S + row_s) * a.q_heads + kvh * group + col - row_s * group;
    const float sum = l[cb][0], inv = sum != 0.f ? 1.f / BOOST / sum : 0.f;
    const float lse = sum != 0.f ? m[cb] + __builtin_amdgcn_logf(sum) : -INFINITY;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const f32x4 r = o[cb][j] * inv;
      const int ch = 16 * j + 4 * lg;
      if (a.splits > 1) {
        *(f32x4*)(a.partial + (at * a.splits + split) * D + ch) = r;
      } else if (a.out_mode == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) ((float*)a.out)[at * (D + 1) + ch + i] = r[i];
      } else {
        *(u32x2*)((uint16_t*)a.out + at * D + ch) =
            u32x2{to16<true>(r[0]) | to16<true>(r[1]) << 16, to16<true>(r[2]) | to16<true>(r[3]) << 16};
      }
    }
    if (lg == 0) {
      if (a.splits > 1) a.partial_lse[at * a.splits + split] = lse;
      else if (a.out_mode == 2) ((float*)a.out)[at * (D + 1) + D] = lse * LN2;
    }
  }
}

template <class Fn>
bool dispatch(int D, int G, Fn&& fn) {
  auto typed = [&](auto d, auto g) {
    fn(d, g);
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

// The same arguments as tdist_kv4_attn, for a bf16 cache and without a cap.  flags: one int for every (block of columns, sequence, split, KV head),
// `flag_columns` columns to a block; tdist_kv4_attn with them, on the same stream, then does what is flagged and the merge.
TDIST_API int tdist_kv4_chunk(const void* k_codes, const void* v_codes, const void* k_params, const void* v_params, int pages,
                              int kv_heads, int page_size, int head_dim, int group, const void* q, long long q_sb, long long q_ss,
                              long long q_sh, const int* table, int table_stride, int max_pages, const int* kv_len, float* partial,
                              void* out, int batch, int S, int q_heads, int splits, int causal, int out_mode, float scale,
                              int dtype, int* flags, int flag_columns, void* stream) {
  ChunkArgs a;
  a.c = Cache{(uint8_t*)k_codes, (uint8_t*)v_codes, (uint32_t*)k_params, (uint32_t*)v_params, pages, kv_heads, page_size};
  TDIST_REQUIRE(k_codes && v_codes && k_params && v_params && pages > 0 && kv_heads > 0 && page_size > 0 && page_size % 16 == 0 &&
                    (((uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_params | (uintptr_t)v_params) & 15) == 0,
                "a 4-bit cache needs four 16-byte aligned tensors, pages of a multiple of 16 tokens");
  TDIST_REQUIRE(batch >= 0 && S >= 0 && q_heads > 0 && q_heads % kv_heads == 0 && max_pages >= 0 &&
                    (long long)max_pages * page_size <= (1ll << 30), "bad head counts, or more than 2^30 tokens in a row of the table");
  TDIST_REQUIRE(splits >= 1 && splits <= 65535 && (splits == 1 || partial), "splits need their partial rows");
  TDIST_REQUIRE((out_mode == 1 || out_mode == 2) && dtype == 0, "out_mode must be 1 or 2, dtype 0 (bf16)");
  if (batch == 0 || S == 0) return 0;
  TDIST_REQUIRE(q && (table || max_pages == 0) && kv_len && out && flags, "null argument");
  TDIST_REQUIRE(((uintptr_t)q & 15) == 0 && ((uintptr_t)out & 7) == 0 && ((q_sb | q_ss | q_sh) & 7) == 0,
                "q rows must keep 16-byte alignment");
  const long long columns = (long long)(q_heads / kv_heads) * S;
  TDIST_REQUIRE(columns < (1ll << 30) && (long long)batch * S * q_heads < (1ll << 31), "too many query rows");
  a.q = (const uint16_t*)q, a.partial = partial, a.out = out, a.flags = flags;
  a.page_tiles = page_size / 16;
  a.page_magic = a.page_tiles == 1 ? 0u : (uint32_t)((1ull << 32) / a.page_tiles) + 1u;
  a.partial_lse = partial ? partial + (long long)batch * S * q_heads * splits * head_dim : nullptr;
  a.q_sb = q_sb, a.q_ss = q_ss, a.q_sh = q_sh, a.table_stride = table_stride, a.max_pages = max_pages;
  a.batch = batch, a.S = S, a.q_heads = q_heads, a.group = q_heads / kv_heads, a.splits = splits, a.causal = causal, a.out_mode = out_mode;
  a.scale = scale;
  bool same = true;
  const bool ok = dispatch(head_dim, group, [&](auto d, auto g) {
    constexpr int D = decltype(d)::value, NW = WAVES;
    constexpr int per_group = columns_of<D, NW>();
    same = flag_columns == per_group;
    if (!same) return;
    const long long blocks = (columns + per_group - 1) / per_group * batch;
    for (a.first = 0; a.first < blocks; a.first += 65535)       // (the limit of a grid's third dimension)
      hipLaunchKernelGGL((kv4_chunk_kernel<D, decltype(g)::value, NW>),
                         dim3(kv_heads, splits, (unsigned)std::min(65535ll, blocks - a.first)), dim3(NW * 64), 0, (hipStream_t)stream,
                         a, table, kv_len);
  });
  TDIST_REQUIRE(ok, "head_dim 64 / 128 / 256 with groups of 32 / 64 / 128 channels (at most head_dim)");
  TDIST_REQUIRE(same, "flag_columns must be the columns of a workgroup");
  TDIST_HIP_TRY(hipGetLastError());
  return 0;
}
