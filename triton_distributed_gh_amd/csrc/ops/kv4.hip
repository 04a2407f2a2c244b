// Writing and reading a 4-bit KV cache (format and layout: tdist/kv4.hpp).
//
//   kv4_append    K / V rows of new tokens -> codes and group parameters
//   kv4_qkv_prep  the same from a QKV projection, with the heads' RMSNorm and rotation in front (and q out)
//   kv4_read      pages -> 16-bit rows, the sequences packed one behind the other
//
// All three move rows once and are bound by memory; a lane works on eight neighbouring channels (16 bytes of a 16-bit
// row), D / 8 lanes on a row, so a group's minimum and maximum are G / 8 lanes' and stay inside a wave.
//
// Measured, 8 KV heads of 128: append of 8 ragged prompts of up to 4001 tokens (groups of 128, 89 MB in and out) 25 us, 3.5 TB/s,
// where the simple form (a lane group per row, V written unit by unit) took 40; read of 16 ragged sequences of up to 8192
// (groups of 64, 351 MB) 79 .. 82 us, 4.3 TB/s of a copy's 4.9, simple form 199; projection epilogue of 2 x 1500 tokens, 64 query
// heads, groups of 32 (about 115 MB) 33 us, 3.5 TB/s, simple form 65.  Append is held by the ten or so vector operations a channel
// that exact codes take, next to its bytes.  What the projection's epilogue waits for, 33 us where its bytes take 23.5, is not known: of
// its 80 heads here 64 are Q's, without codes and in 32 bits.  One token of a sequence (6 us for write and read, 7.5 with the
// projection) is held by the launches.
// This file is compiled without fast-math: the code of a value next to a border is decided by IEEE arithmetic and is
// the same on every path that writes a cache, the CPU's included.
#include <algorithm>

#include "tdist/kv4.hpp"

namespace {

using namespace tdist::kv4;

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

// A wave works on a tile of TILE tokens in PASSES passes of ROWS rows of LANES lanes.
template <int D, int MOST = 16>
struct Tile {
  static constexpr int LANES = D / 8, ROWS = 64 / LANES, TILE = MOST < 4 * ROWS ? MOST : 4 * ROWS, PASSES = TILE / ROWS;
};
template <int D>
using PrepTile = Tile<D, 8>;        // (the rotation's factors of a tile are kept in registers)

template <bool IS_BF16>
__device__ __forceinline__ void unpack_row8(const u32x4& v, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = from16<IS_BF16>(v[i] & 0xffffu);
    x[2 * i + 1] = low_of<IS_BF16>(v[i]);
  }
}
template <bool IS_BF16>
__device__ __forceinline__ u32x4 pack_row8(const float (&x)[8]) {
  u32x4 u;
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = to16<IS_BF16>(x[2 * i]) | to16<IS_BF16>(x[2 * i + 1]) << 16;
  return u;
}

// Lane exchanges inside a row of sixteen without LDS.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true);
}
constexpr int XOR1 = 0xb1, XOR2 = 0x4e, XOR3 = 0x1b, XOR7 = 0x141, XOR15 = 0x140, ROR8 = 0x128;
__device__ __forceinline__ uint32_t xor4(uint32_t v) { return dpp<XOR7>(dpp<XOR3>(v)); }
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, dpp<CTRL>(__builtin_bit_cast(uint32_t, v)));
}
template <int CTRL>
__device__ __forceinline__ double dpp(double v) {
  const uint2 u = __builtin_bit_cast(uint2, v);
  return __builtin_bit_cast(double, uint2{dpp<CTRL>(u.x), dpp<CTRL>(u.y)});
}
// op over N neighbouring lanes (N = 4 .. 32); every lane gets the result.  (Once fours agree, the mirrored eight is one, and
// so on.)
template <int N, class T, class Op>
__device__ __forceinline__ T over_lanes(T v, Op op) {
  v = op(v, dpp<XOR1>(v));
  v = op(v, dpp<XOR2>(v));
  if constexpr (N >= 8) v = op(v, dpp<XOR7>(v));
  if constexpr (N >= 16) v = op(v, dpp<XOR15>(v));
  if constexpr (N >= 32) v = op(v, __shfl_xor(v, 16));
  return v;
}

// A group's range over the G / 8 lanes that hold it, and its smallest value; `nan`: one of the lane's values is a NaN (which
// minimum and maximum pass over).  An infinite value makes the range infinite or NaN.
template <int G>
__device__ __forceinline__ float range_of(const float (&x)[8], float& lo, bool& nan) {
  float hi = x[0];
  lo = x[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) lo = fminf(lo, x[e]), hi = fmaxf(hi, x[e]);
  lo = over_lanes<G / 8>(lo, [](float a, float b) { return fminf(a, b); });
  hi = over_lanes<G / 8>(hi, [](float a, float b) { return fmaxf(a, b); });
  nan = __builtin_isunordered(x[0], x[1]) | __builtin_isunordered(x[2], x[3]) | __builtin_isunordered(x[4], x[5]) |
        __builtin_isunordered(x[6], x[7]);
  return hi - lo;
}
__device__ __forceinline__ bool ordinary(float range) { return range == 0.f || (range > 0x1p-96f && range < 0x1p110f); }

// Codes of the lane's eight channels, as floats, and the parameter dword of their group.
//
// Both quotients, range / 15 and (x - low) / scale, have to be the IEEE ones.  With r = RN(1 / s) and q0 = RN(d r),
// which is within an ulp of the quotient, d - q0 s is exact in one fma and RN(q0 + (d - q0 s) r) is the correctly rounded
// quotient (Markstein's theorem); r itself comes from the hardware's reciprocal by one step of the same kind.  Its one
// exception, a divisor whose significand is all ones, is neither 15 nor a 16-bit number.  That is three operations a channel
// where a division takes ten.  PLAIN: the range is ordinary, no intermediate can leave the normal numbers; the others divide.
template <bool IS_BF16, int G, bool PLAIN>
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], float lo, float range, bool nan, float (&code)[8]) {
  uint32_t s16;
  if (PLAIN) {
    constexpr float R15 = 1.f / 15.f;
    const float s0 = range * R15;
    s16 = to16<IS_BF16>(__builtin_fmaf(__builtin_fmaf(-s0, 15.f, range), R15, s0));
    const float s = from16<IS_BF16>(s16);
    float r = __builtin_amdgcn_rcpf(s);
    r = __builtin_fmaf(__builtin_fmaf(-s, r, 1.f), r, r);
    r = s > 0.f ? r : 0.f;                            // no range, or a scale that rounds to 0: codes 0
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = x[e] - lo;
      const float q0 = d * r;
      code[e] = __builtin_rintf(__builtin_fmaf(__builtin_fmaf(-q0, s, d), r, q0));
      if constexpr (!IS_BF16) code[e] = fminf(code[e], 15.f);   // a subnormal scale may be rounded down a long way
    }
  } else {
    range += over_lanes<G / 8>(nan ? NAN : 0.f, [](float a, float b) { return a + b; });
    s16 = range < INFINITY ? to16<IS_BF16>(range / 15.f) : to16<IS_BF16>(NAN);
    const float s = from16<IS_BF16>(s16);
#pragma unroll
    for (int e = 0; e < 8; ++e) code[e] = s > 0.f ? fminf(__builtin_rintf((x[e] - lo) / s), 15.f) : 0.f;
  }
  return s16 | to16<IS_BF16>(lo) << 16;               // (lo is one of the row's 16-bit values)
}

// Quantises a tile of rows of one head and writes rows lo .. hi - 1 of it.  `at`: the place of the tile's first token (a
// multiple of TILE, so all of them are in one page).  rows(p, x): the lane's eight channels of pass p.  `stage`: TILE D / 2 bytes
// of LDS of the wave's own.
//
// K rows are runs of their own.  A 16-byte run of V is one channel lane's four tokens: a whole tile is brought into that
// order in LDS and leaves as 16-byte stores; the first and last tile of a sequence, whose runs are shared with other calls, are
// written unit by unit.  The passes of a whole tile are one stretch of straight code.
template <bool IS_BF16, int D, int G, bool IS_V, class T, class Rows>
__device__ __forceinline__ void store_tile(const Cache& c, const Place& at, int head, int lo, int hi, char* stage, Rows&& rows) {
  const int lane = threadIdx.x & 63, l8 = lane % T::LANES;
  const long long row0 = ((long long)at.page * c.kv_heads + head) * c.page_size;   // first token of (page, head)
  uint8_t* const vbase = c.v_codes + (row0 + at.off) * (D / 2);
  uint32_t* const params = (IS_V ? c.v_params : c.k_params) + row0 * (D / G) + (long long)(l8 / (G / 8)) * c.page_size + at.off;

  auto write = [&](auto whole_, int p, uint32_t param, const float (&code)[8]) __attribute__((always_inline)) {
    constexpr bool WHOLE = decltype(whole_)::value;
    const int i = p * T::ROWS + lane / T::LANES;
    const bool live = WHOLE || (i >= lo && i < hi);
    if constexpr (!IS_V) {
      // (codes are put together as floats, exactly: one conversion for four)
      float even = code[6], odd = code[7];
#pragma unroll
      for (int n = 4; n >= 0; n -= 2) even = __builtin_fmaf(even, 16.f, code[n]), odd = __builtin_fmaf(odd, 16.f, code[n + 1]);
      const uint32_t w = (uint32_t)even | (uint32_t)odd << 16;
      const int word = (l8 & 3) * (D / 32) + (l8 >> 2);
      if (live) *(uint32_t*)(c.k_codes + (row0 + at.off + i) * (D / 2) + word * 4) = w;
    } else {
      // the four lanes n = 0 .. 3 of a unit hold its four 16-channel tiles: two steps of exchange, in each of which a lane
      // keeps half of what it has and gives the other half away, leave each lane two whole units
      const int n = (l8 >> 1) & 3;
      uint32_t u[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) u[k] = (uint32_t)__builtin_fmaf(code[2 * k + 1], 65536.f, code[2 * k]) << (4 * n);
      const bool up1 = n & 1, up2 = n & 2;
      const uint32_t a0 = (up1 ? u[2] : u[0]) | dpp<XOR2>(up1 ? u[0] : u[2]);
      const uint32_t a1 = (up1 ? u[3] : u[1]) | dpp<XOR2>(up1 ? u[1] : u[3]);
      const uint32_t b = (up2 ? a1 : a0) | xor4(up2 ? a0 : a1);
      const int ch = (l8 & 1) * 8 + (up1 ? 4 : 0) + (up2 ? 2 : 0);                  // this lane's units: channels ch, ch + 1
      const int to = (i >> 2) * (2 * D) + ch * (D / 8) + (l8 >> 3) * 8 + (i & 3) * 2;
      if (WHOLE) {
        *(uint16_t*)(stage + to) = (uint16_t)b;
        *(uint16_t*)(stage + to + D / 8) = (uint16_t)(b >> 16);
      } else if (live) {
        *(uint16_t*)(vbase + to) = (uint16_t)b;
        *(uint16_t*)(vbase + to + D / 8) = (uint16_t)(b >> 16);
      }
    }
    if (live && l8 % (G / 8) == 0) params[i] = param;
  };

  if (lo <= 0 && hi >= T::TILE) {
    float x[T::PASSES][8], low[T::PASSES], range[T::PASSES];
    bool nan[T::PASSES], odd = false;
#pragma unroll
    for (int p = 0; p < T::PASSES; ++p) {
      rows(p, x[p]);
      range[p] = range_of<G>(x[p], low[p], nan[p]);
      odd |= nan[p] | !ordinary(range[p]);
    }
    if (!__any(odd)) {
#pragma unroll
      for (int p = 0; p < T::PASSES; ++p) {
        float code[8];
        const uint32_t param = quantise8<IS_BF16, G, true>(x[p], low[p], range[p], false, code);
        write(std::true_type{}, p, param, code);
      }
    } else {
#pragma unroll
      for (int p = 0; p < T::PASSES; ++p) {
        float code[8];
        const uint32_t param = quantise8<IS_BF16, G, false>(x[p], low[p], range[p], nan[p], code);
        write(std::true_type{}, p, param, code);
      }
    }
    if constexpr (IS_V) {
      lanes_meet();
      if (lane * 16 < T::TILE * (D / 2)) *(u32x4*)(vbase + lane * 16) = *(const u32x4*)(stage + lane * 16);
      lanes_meet();                     // (the next head's tile)
    }
  } else {
#pragma unroll
    for (int p = 0; p < T::PASSES; ++p) {
      if (hi <= p * T::ROWS || lo >= (p + 1) * T::ROWS) continue;                  // (uniform)
      float x[8], code[8], low;
      bool nan;
      rows(p, x);
      const float range = range_of<G>(x, low, nan);
      uint32_t param;
      if (!__any(nan | !ordinary(range))) {
        param = quantise8<IS_BF16, G, true>(x, low, range, false, code);
      } else {
        param = quantise8<IS_BF16, G, false>(x, low, range, nan, code);
      }
      write(std::false_type{}, p, param, code);
    }
  }
}

// A wave per tile and head; workgroups with neighbouring numbers take the heads (Hkv of K, then Hkv of V) of the same tokens,
// whose rows are neighbours in memory.  Tiles are aligned in the sequence.  grid: (tiles x heads, batch)
template <bool IS_BF16, int D, int G>
__global__ __launch_bounds__(256) void kv4_append_kernel(Cache c, const uint16_t* __restrict__ k, const uint16_t* __restrict__ v,
                                                         long long k_sb, long long k_ss, long long k_sh, long long v_sb,
                                                         long long v_ss, long long v_sh, const int* __restrict__ kv_offset,
                                                         const int* __restrict__ new_lens, const int* __restrict__ table,
                                                         int table_stride, int max_pages, int S) {
  using T = Tile<D>;
  __shared__ __attribute__((aligned(16))) char stage[4][T::TILE * D / 2];
  const int b = blockIdx.y, lane = threadIdx.x & 63, l8 = lane % T::LANES;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t tile = blockIdx.x / (2u * c.kv_heads), which = blockIdx.x - tile * 2u * c.kv_heads;
  const bool is_v = (int)which >= c.kv_heads;
  const int head = which - (is_v ? c.kv_heads : 0);
  const int offset = kv_offset[b], count = new_lens ? min(new_lens[b], S) : S;
  const long long s0 = ((long long)tile * (blockDim.x >> 6) + wave) * T::TILE - (offset & (T::TILE - 1));   // the tile's first row
  if (s0 >= count) return;
  const Place at = place_of(c, table + (long long)b * table_stride, offset + s0, max_pages);
  if (at.page < 0) return;
  const int lo = s0 < 0 ? (int)-s0 : 0, hi = (int)min((long long)T::TILE, count - s0);
  const uint16_t* src = is_v ? v + b * v_sb + head * v_sh : k + b * k_sb + head * k_sh;
  const long long ss = is_v ? v_ss : k_ss;
  u32x4 raw[T::PASSES];
#pragma unroll
  for (int p = 0; p < T::PASSES; ++p) {
    const int i = p * T::ROWS + lane / T::LANES;
    raw[p] = u32x4{0, 0, 0, 0};
    if (i >= lo && i < hi) raw[p] = *(const u32x4*)(src + (s0 + i) * ss + l8 * 8);
  }
  auto rows = [&](int p, float (&x)[8]) { unpack_row8<IS_BF16>(raw[p], x); };
  if (is_v) {
    store_tile<IS_BF16, D, G, true, T>(c, at, head, lo, hi, stage[wave], rows);
  } else {
    store_tile<IS_BF16, D, G, false, T>(c, at, head, lo, hi, stage[wave], rows);
  }
}

// grid: (tiles of tokens x blocks of `heads_each` of the Hq + 2 Hkv heads, batch), a wave per tile and block: the rotation's
// factors of a tile are fetched once for the heads of the block.  K's mean square and rotation are taken in 64 bits, so that a
// stored code does not depend on the order of a sum; Q's in 32.
template <int D, int G>
__global__ __launch_bounds__(256) void kv4_qkv_prep_kernel(Cache c, const uint16_t* __restrict__ qkv, long long q_sb,
                                                           long long q_ss, const uint16_t* __restrict__ q_w,
                                                           const uint16_t* __restrict__ k_w, float q_eps, float k_eps,
                                                           const long long* __restrict__ positions,
                                                           const float* __restrict__ cos_t, const float* __restrict__ sin_t,
                                                           long long rope_rows, uint16_t* __restrict__ q_out,
                                                           const int* __restrict__ kv_offset, int* __restrict__ total_out,
                                                           const int* __restrict__ table, int table_stride, int max_pages,
                                                           int S, int q_heads, int heads_each) {
  using T = PrepTile<D>;
  __shared__ __attribute__((aligned(16))) char stage[4][T::TILE * D / 2];
  const int b = blockIdx.y, lane = threadIdx.x & 63, l8 = lane % T::LANES;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int heads = q_heads + 2 * c.kv_heads;
  const uint32_t blocks = (heads + heads_each - 1) / heads_each, tile = blockIdx.x / blocks, block = blockIdx.x - tile * blocks;
  const int offset = kv_offset[b];
  if (blockIdx.x == 0 && threadIdx.x == 0) total_out[b] = offset + S;
  const long long s0 = ((long long)tile * (blockDim.x >> 6) + wave) * T::TILE - (offset & (T::TILE - 1));
  if (s0 >= S) return;
  const int lo = s0 < 0 ? (int)-s0 : 0, hi = (int)min((long long)T::TILE, S - s0);
  const int head0 = block * heads_each, head1 = min(head0 + heads_each, heads);
  Place at = Place{-1, 0};
  if (head1 > q_heads) at = place_of(c, table + (long long)b * table_stride, offset + s0, max_pages);
  float cs[T::PASSES][8], sn[T::PASSES][8];
  if (head0 < q_heads + c.kv_heads) {
#pragma unroll
    for (int p = 0; p < T::PASSES; ++p) {
      const int i = p * T::ROWS + lane / T::LANES;
      long long pos = i >= lo && i < hi ? positions[(long long)b * S + s0 + i] : 0;
      pos = pos < 0 ? 0 : pos < rope_rows ? pos : rope_rows - 1;
      const long long from = pos * (D / 2) + (l8 * 8) % (D / 2);
#pragma unroll
      for (int e = 0; e < 8; ++e) cs[p][e] = cos_t[from + e], sn[p][e] = sin_t[from + e];
    }
  }
  const uint16_t* src = qkv + b * q_sb + l8 * 8;
  auto fetch = [&](int head, u32x4 (&raw)[T::PASSES]) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < T::PASSES; ++p) {
      const int i = p * T::ROWS + lane / T::LANES;
      raw[p] = u32x4{0, 0, 0, 0};
      if (i >= lo && i < hi) raw[p] = *(const u32x4*)(src + (s0 + i) * q_ss + (long long)head * D);
    }
  };
  u32x4 raw[T::PASSES], next[T::PASSES] = {};
  fetch(head0, raw);
  for (int head = head0; head < head1; ++head) {
    if (head + 1 < head1) fetch(head + 1, next);
    const bool is_q = head < q_heads, is_v = head >= q_heads + c.kv_heads;
    const uint16_t* w = is_q ? q_w : is_v ? nullptr : k_w;
    float g[8];
    if (w) unpack_row8<true>(*(const u32x4*)(w + l8 * 8), g);
    auto rows = [&](int p, float (&x)[8]) __attribute__((always_inline)) {
      unpack_row8<true>(raw[p], x);
      if (is_v) return;
      if (w) {
        float inv;
        if (is_q) {
          float ss = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(x[e], x[e], ss);
          ss = over_lanes<T::LANES>(ss, [](float a, float b) { return a + b; });
          inv = __builtin_amdgcn_rsqf(ss * (1.f / D) + q_eps);
        } else {
          double ss = 0.;
#pragma unroll
          for (int e = 0; e < 8; ++e) ss = __builtin_fma((double)x[e], (double)x[e], ss);
          ss = over_lanes<T::LANES>(ss, [](double a, double b) { return a + b; });
          inv = (float)(1. / __builtin_sqrt(ss / D + (double)k_eps));
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = from16<true>(to16<true>(x[e] * inv * g[e]));
      }
      // pairs (i, i + D / 2) are the same element of lanes l8 and l8 ^ (D / 16)
      float other[8], y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (D == 128) {
          other[e] = dpp<ROR8>(x[e]);
        } else if constexpr (D == 64) {
          other[e] = dpp<XOR7>(dpp<XOR3>(x[e]));
        } else {
          other[e] = __shfl_xor(x[e], 16);
        }
        if (l8 < T::LANES / 2) other[e] = -other[e];
      }
      if (is_q) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = __builtin_fmaf(x[e], cs[p][e], other[e] * sn[p][e]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float co = cs[p][e], si = sn[p][e];
          asm volatile("" : "+v"(co), "+v"(si));      // (not all of them as 64-bit numbers ahead of the loop over the heads)
          y[e] = (float)__builtin_fma((double)x[e], (double)co, (double)other[e] * si);
          asm volatile("" : "+v"(y[e]));        // 64 -> 32 -> 16 bits as two roundings, which the compiler would merge
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = from16<true>(to16<true>(y[e]));
    };
    if (is_q) {
#pragma unroll
      for (int p = 0; p < T::PASSES; ++p) {
        if (hi <= p * T::ROWS || lo >= (p + 1) * T::ROWS) continue;
        const int i = p * T::ROWS + lane / T::LANES;
        float x[8];
        rows(p, x);
        if (i >= lo && i < hi) *(u32x4*)(q_out + (((long long)b * S + s0 + i) * q_heads + head) * D + l8 * 8) = pack_row8<true>(x);
      }
    } else if (at.page >= 0) {
      if (is_v) {
        store_tile<true, D, G, true, T>(c, at, head - q_heads - c.kv_heads, lo, hi, stage[wave], rows);
      } else {
        store_tile<true, D, G, false, T>(c, at, head - q_heads, lo, hi, stage[wave], rows);
      }
    }
#pragma unroll
    for (int p = 0; p < T::PASSES; ++p) raw[p] = next[p];
  }
}

// Row r of the output belongs to the sequence b with cu[b] <= r < cu[b + 1].  A wave takes `rows_each` rows (TILE, or ROWS) of
// one head of K or V, sequence by sequence (one row of each of many sequences: 26 us with TILE, 4 with ROWS); workgroups with
// neighbouring numbers take the heads of the same rows, which are neighbours in the output.  V's runs of four tokens are turned into rows in LDS.
template <bool IS_BF16, int D, int G>
__global__ __launch_bounds__(256) void kv4_read_kernel(Cache c, const int* __restrict__ table, int table_stride, int max_pages,
                                                       const int* __restrict__ cu, const int* __restrict__ starts, int batch,
                                                       long long total, int rows_each, uint16_t* __restrict__ k_out,
                                                       uint16_t* __restrict__ v_out, long long k_st, long long k_sh,
                                                       long long v_st, long long v_sh) {
  using T = Tile<D>;
  constexpr float MOST = IS_BF16 ? 0x1.fep127f : 65504.f;
  constexpr int QUADS = T::TILE / 4 + 1;        // of an unaligned tile
  constexpr int ROW = D / 2 + 16;               // bytes of a token's units in LDS, and a gap so that neighbours meet other banks
  __shared__ __attribute__((aligned(16))) char stages[4][QUADS * 4 * ROW];
  const int lane = threadIdx.x & 63, l8 = lane % T::LANES;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  char* const stage = stages[wave];
  const uint32_t tile = blockIdx.x / (2u * c.kv_heads), which = blockIdx.x - tile * 2u * c.kv_heads;
  const bool is_v = (int)which >= c.kv_heads;
  const int head = which - (is_v ? c.kv_heads : 0);
  const long long end = min(total, (long long)cu[batch]);
  long long r = max(((long long)tile * (blockDim.x >> 6) + wave) * rows_each, (long long)cu[0]);
  const long long stop = min(((long long)tile * (blockDim.x >> 6) + wave + 1) * rows_each, end);
  if (r >= stop) return;
  int b = 0, b_last = 0;                        // how many sequences end at or before r, and before the last row
  for (int i = 0; i < batch; i += 64) {
    const int ends = i + lane < batch ? cu[i + lane + 1] : 0x7fffffff;
    b += __popcll(__ballot(ends <= r));
    b_last += __popcll(__ballot(ends < stop));
  }
  b = min(__builtin_amdgcn_readfirstlane(b), batch - 1);
  b_last = min(__builtin_amdgcn_readfirstlane(b_last), batch - 1);
  const uint8_t* const codes = is_v ? c.v_codes : c.k_codes;
  const uint32_t* const params = is_v ? c.v_params : c.k_params;
  uint16_t* const out = (is_v ? v_out + head * v_sh : k_out + head * k_sh) + l8 * 8;
  const long long st = is_v ? v_st : k_st;

  if (b_last > b + 1) {
    // rows of many sequences (a decode step's, one each): every row finds its own place, V channel by channel
    const int ends = b + lane < batch ? cu[b + lane + 1] : 0x7fffffff;
#pragma unroll
    for (int p = 0; p < T::PASSES; ++p) {
      if (r + p * T::ROWS >= stop) break;
      const long long mine = r + p * T::ROWS + lane / T::LANES;
      int at_b = b;
#pragma unroll
      for (int j = 0; j < T::ROWS; ++j) {
        const int passed = __popcll(__ballot(ends <= r + p * T::ROWS + j));
        if (lane / T::LANES == j) at_b = b + passed;
      }
      if (b_last - b >= 64) {                   // (sixty sequences without rows between these: a lane each does not reach)
        at_b = b;
        for (int top = b_last + 1; top - at_b > 1;) {
          const int mid = (at_b + top) >> 1;
          if (cu[mid] <= mine) at_b = mid; else top = mid;
        }
      }
      if (mine >= stop) continue;
      const long long pos = (starts ? (long long)starts[at_b] : 0) + (mine - cu[at_b]);
      const Place at = place_of(c, table + (long long)at_b * table_stride, pos, max_pages);
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = 0.f;
      if (at.page >= 0) {
        const long long row0 = ((long long)at.page * c.kv_heads + head) * c.page_size;
        const uint32_t param = params[row0 * (D / G) + (long long)(l8 / (G / 8)) * c.page_size + at.off];
        const float s = scale_of<IS_BF16>(param), low = low_of<IS_BF16>(param);
        const uint8_t* k_at = codes + (row0 + at.off) * (D / 2) + ((l8 & 3) * (D / 32) + (l8 >> 2)) * 4;
        const uint8_t* v_at = codes + row0 * (D / 2) + (at.off >> 2) * (2 * D) + (l8 & 1) * D + (l8 >> 3) * 8 + (at.off & 3) * 2;
        const uint32_t w = is_v ? 0u : *(const uint32_t*)k_at;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t unit = is_v ? (uint32_t)*(const uint16_t*)(v_at + e * (D / 8)) >> (4 * ((l8 >> 1) & 3))
                                     : w >> (4 * (e >> 1) + 16 * (e & 1));
          x[e] = __builtin_fmaf(s, (float)(unit & 15u), low);
          x[e] = x[e] > MOST ? MOST : x[e];
        }
      }
      *(u32x4*)(out + mine * st) = pack_row8<IS_BF16>(x);
    }
    return;
  }
  while (r < stop && b < batch) {
    const long long pos = (starts ? (long long)starts[b] : 0) + (r - cu[b]);
    int n = (int)min(stop, (long long)cu[b + 1]) - (int)r;               // rows of this sequence
    if (pos < 0) n = (int)min((long long)n, -pos);                       // (in front of its first token, on their own)
    if (n <= 0) {
      ++b;
    } else {
      // at most two pages: rows below `cut` are in the first
      const int* row = table + (long long)b * table_stride;
      const Place first = place_of(c, row, pos, max_pages);
      const int off = (int)((uint32_t)(pos < 0 ? 0 : pos) % (uint32_t)c.page_size), cut = c.page_size - off;
      const Place second = n > cut ? place_of(c, row, pos + cut, max_pages) : Place{-1, 0};
      const long long row_a = ((long long)first.page * c.kv_heads + head) * c.page_size + off;
      const long long row_b = ((long long)second.page * c.kv_heads + head) * c.page_size - cut;
      const long long top_a = row_a - off, top_b = row_b + cut;           // first rows of the pages
      if (is_v) {
        // quads q = 0 .. of the tokens off & ~3 ..; row i is token (off & 3) + i of them
        const int shift = off & 3;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int quad = k * (T::TILE / 4) + (lane >> 4), i = quad * 4 - shift;      // i: its first token's row
          if (quad < QUADS && (T::TILE / 4 == 4 || k == 1 || quad < T::TILE / 4) && i < n && i > -4) {
            const bool in_b = i >= cut;
            if ((in_b ? second.page : first.page) >= 0) {
              const uint8_t* p = codes + ((in_b ? row_b : row_a) + i) * (D / 2) + (lane & 15) * (D / 8);
              uint32_t w[D / 32];
              if constexpr (D == 64) {
                const uint2 v = *(const uint2*)p;
                w[0] = v.x, w[1] = v.y;
              } else {
#pragma unroll
                for (int j = 0; j < D / 128; ++j) {
                  const u32x4 v = *(const u32x4*)(p + 16 * j);
#pragma unroll
                  for (int m = 0; m < 4; ++m) w[4 * j + m] = v[m];
                }
              }
#pragma unroll
              for (int h = 0; h < D / 64; ++h)
#pragma unroll
                for (int t = 0; t < 4; ++t)
                  *(uint16_t*)(stage + (quad * 4 + t) * ROW + h * 32 + (lane & 15) * 2) = (uint16_t)(w[2 * h + (t >> 1)] >> (16 * (t & 1)));
            }
          }
        }
        lanes_meet();
      }
      uint32_t word[T::PASSES], param[T::PASSES];
#pragma unroll
      for (int p = 0; p < T::PASSES; ++p) {
        const int i = p * T::ROWS + lane / T::LANES;
        const bool in_b = i >= cut;
        word[p] = param[p] = 0;                 // (no page: zeros)
        if (i < n && (in_b ? second.page : first.page) >= 0) {
          const long long at = (in_b ? row_b : row_a) + i, page_top = in_b ? top_b : top_a;
          if (!is_v) word[p] = *(const uint32_t*)(codes + at * (D / 2) + ((l8 & 3) * (D / 32) + (l8 >> 2)) * 4);
          param[p] = params[page_top * (D / G) + (long long)(l8 / (G / 8)) * c.page_size + (at - page_top)];
        }
      }
#pragma unroll
      for (int p = 0; p < T::PASSES; ++p) {
        const int i = p * T::ROWS + lane / T::LANES;
        uint32_t lo4, hi4;                      // codes of channels (0, 4, 1, 5) and (2, 6, 3, 7), a byte each
        if (is_v) {
          const u32x4 v = *(const u32x4*)(stage + ((off & 3) + i) * ROW + (l8 >> 3) * 32 + (l8 & 1) * 16);
          const int by = 4 * ((l8 >> 1) & 3);
          const uint32_t a = v[0] >> by & 0x000f000fu, b2 = v[1] >> by & 0x000f000fu, c2 = v[2] >> by & 0x000f000fu,
                         d = v[3] >> by & 0x000f000fu;
          lo4 = a | c2 << 8, hi4 = b2 | d << 8;
        } else {
          lo4 = word[p] & 0x0f0f0f0fu, hi4 = word[p] >> 4 & 0x0f0f0f0fu;
        }
        const float s = scale_of<IS_BF16>(param[p]), low = low_of<IS_BF16>(param[p]);
        const float code[8] = {(float)(lo4 & 0xffu), (float)(lo4 >> 16 & 0xffu), (float)(hi4 & 0xffu), (float)(hi4 >> 16 & 0xffu),
                               (float)(lo4 >> 8 & 0xffu), (float)(lo4 >> 24), (float)(hi4 >> 8 & 0xffu), (float)(hi4 >> 24)};
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __builtin_fmaf(s, code[e], low);
        if (__any(__builtin_fmaf(s, 15.f, low) > MOST)) {                // (a scale that was rounded up)
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = x[e] > MOST ? MOST : x[e];  // a NaN stays one
        }
        if (is_v && (i >= cut ? second.page : first.page) < 0) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = 0.f;
        }
        if (i < n) *(u32x4*)(out + (r + i) * st) = pack_row8<IS_BF16>(x);
      }
      lanes_meet();                     // (the next sequence's rows)
      r += n;
    }
  }
}

// fn(<IS_BF16>, <D>, <G>) for the supported combinations; false if there is none.
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

bool cache_ok(const Cache& c) {
  return c.k_codes && c.v_codes && c.k_params && c.v_params && c.pages > 0 && c.kv_heads > 0 && c.kv_heads <= 16384 &&
         c.page_size > 0 && c.page_size % 16 == 0 &&
         (((uintptr_t)c.k_codes | (uintptr_t)c.v_codes | (uintptr_t)c.k_params | (uintptr_t)c.v_params) & 15) == 0;
}

// tiles that S tokens can touch, wherever the first one falls
int tiles_of(int S, int tile) { return (int)(((long long)S + tile - 1 + tile - 1) / tile); }

// a grid's second dimension, and the threads of its first
constexpr int MOST_SEQUENCES = 65535;
bool grid_ok(long long blocks, int waves) { return blocks * waves * 64 < (1ll << 32); }

// tokens are counted in 32 bits, with room for whole blocks behind the last one
bool room_ok(const Cache& c, int max_pages) { return (long long)max_pages * c.page_size <= (1ll << 30); }

constexpr const char* TOO_MANY = "too many rows for one call";
constexpr const char* BAD_CACHE = "a 4-bit cache needs four 16-byte aligned tensors, pages of a multiple of 16 tokens";
constexpr const char* BAD_FORM = "head_dim 64 / 128 / 256 with groups of 32 / 64 / 128 channels (at most head_dim), dtype 0 (bf16) or 1 (fp16)";

}  // namespace

TDIST_API int tdist_kv4_append(void* k_codes, void* v_codes, void* k_params, void* v_params, int pages, int kv_heads,
                               int page_size, int head_dim, int group, const void* k, const void* v, long long k_sb,
                               long long k_ss, long long k_sh, long long v_sb, long long v_ss, long long v_sh,
                               const int* kv_offset, const int* new_lens, const int* table, int table_stride, int max_pages,
                               int batch, int S, int dtype, void* stream) {
  const Cache c{(uint8_t*)k_codes, (uint8_t*)v_codes, (uint32_t*)k_params, (uint32_t*)v_params, pages, kv_heads, page_size};
  TDIST_REQUIRE(cache_ok(c), BAD_CACHE);
  TDIST_REQUIRE(dtype == 0 || dtype == 1, BAD_FORM);
  TDIST_REQUIRE(batch >= 0 && S >= 0 && max_pages >= 0 && room_ok(c, max_pages) && (long long)S * kv_heads < (1ll << 31),
                "bad batch / token count");
  if (batch == 0 || S == 0) return 0;
  TDIST_REQUIRE(k && v && kv_offset && (table || max_pages == 0), "null argument");
  TDIST_REQUIRE((((uintptr_t)k | (uintptr_t)v) & 15) == 0 && ((k_sb | k_ss | k_sh | v_sb | v_ss | v_sh) & 7) == 0,
                "k / v rows must keep 16-byte alignment");
  bool fits = true;
  const bool ok = dispatch(dtype, head_dim, group, [&](auto bf, auto d, auto g) {
    const int tiles = tiles_of(S, Tile<decltype(d)::value>::TILE), waves = std::min(tiles, 4);
    const int blocks = (tiles + waves - 1) / waves * 2 * kv_heads;
    fits = grid_ok(blocks, waves);
    for (long long b = 0; fits && b < batch; b += MOST_SEQUENCES)
      hipLaunchKernelGGL((kv4_append_kernel<decltype(bf)::value, decltype(d)::value, decltype(g)::value>),
                         dim3(blocks, (unsigned)std::min<long long>(MOST_SEQUENCES, batch - b)),
                         dim3(64 * waves), 0, (hipStream_t)stream, c, (const uint16_t*)k + b * k_sb, (const uint16_t*)v + b * v_sb, k_sb,
                         k_ss, k_sh, v_sb, v_ss, v_sh, kv_offset + b, new_lens ? new_lens + b : nullptr, table + b * table_stride,
                         table_stride, max_pages, S);
  });
  TDIST_REQUIRE(ok, BAD_FORM);
  TDIST_REQUIRE(fits, TOO_MANY);
  TDIST_HIP_TRY(hipGetLastError());
  return 0;
}

TDIST_API int tdist_kv4_qkv_prep(void* k_codes, void* v_codes, void* k_params, void* v_params, int pages, int kv_heads,
                                 int page_size, int head_dim, int group, const void* qkv, long long q_sb, long long q_ss,
                                 const void* q_w, const void* k_w, float q_eps, float k_eps, const long long* positions,
                                 const float* cos_t, const float* sin_t, long long rope_rows, void* q_out,
                                 const int* kv_offset, int* total_out, const int* table, int table_stride, int max_pages,
                                 int batch, int S, int q_heads, void* stream) {
  const Cache c{(uint8_t*)k_codes, (uint8_t*)v_codes, (uint32_t*)k_params, (uint32_t*)v_params, pages, kv_heads, page_size};
  TDIST_REQUIRE(cache_ok(c), BAD_CACHE);
  TDIST_REQUIRE(batch >= 0 && S >= 0 && max_pages >= 0 && room_ok(c, max_pages) && q_heads > 0 && q_heads <= 32767 && rope_rows > 0 &&
                    (long long)S * (q_heads + 2 * kv_heads) < (1ll << 31),
                "bad batch / token / head count");
  if (batch == 0 || S == 0) return 0;
  TDIST_REQUIRE(qkv && positions && cos_t && sin_t && q_out && kv_offset && total_out && (table || max_pages == 0), "null argument");
  TDIST_REQUIRE((((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)q_w | (uintptr_t)k_w) & 15) == 0 && ((q_sb | q_ss) & 7) == 0,
                "qkv rows, norm weights and q must keep 16-byte alignment");
  bool fits = true;
  const bool ok = dispatch(0, head_dim, group, [&](auto bf, auto d, auto g) {
    if constexpr (decltype(bf)::value) {
      const int tiles = tiles_of(S, PrepTile<decltype(d)::value>::TILE), waves = std::min(tiles, 4), heads = q_heads + 2 * kv_heads;
      // heads that share a fetch of the rotation's factors, where there is work for the chip without that
      const int each = (int)std::max(1ll, std::min(8ll, (long long)tiles * heads * batch / 6144));
      const int blocks = (tiles + waves - 1) / waves * ((heads + each - 1) / each);
      fits = grid_ok(blocks, waves);
      for (long long b = 0; fits && b < batch; b += MOST_SEQUENCES)
        hipLaunchKernelGGL((kv4_qkv_prep_kernel<decltype(d)::value, decltype(g)::value>),
                           dim3(blocks, (unsigned)std::min<long long>(MOST_SEQUENCES, batch - b)),
                           dim3(64 * waves), 0, (hipStream_t)stream, c, (const uint16_t*)qkv + b * q_sb, q_sb, q_ss, (const uint16_t*)q_w,
                           (const uint16_t*)k_w, q_eps, k_eps, positions + b * S, cos_t, sin_t, rope_rows,
                           (uint16_t*)q_out + b * S * q_heads * head_dim, kv_offset + b, total_out + b, table + b * table_stride,
                           table_stride, max_pages, S, q_heads, each);
    }
  });
  TDIST_REQUIRE(ok, BAD_FORM);
  TDIST_REQUIRE(fits, TOO_MANY);
  TDIST_HIP_TRY(hipGetLastError());
  return 0;
}

TDIST_API int tdist_kv4_read(const void* k_codes, const void* v_codes, const void* k_params, const void* v_params, int pages,
                             int kv_heads, int page_size, int head_dim, int group, const int* table, int table_stride,
                             int max_pages, const int* cu, const int* starts, int batch, long long total, void* k_out,
                             void* v_out, long long k_st, long long k_sh, long long v_st, long long v_sh, int dtype,
                             void* stream) {
  const Cache c{(uint8_t*)k_codes, (uint8_t*)v_codes, (uint32_t*)k_params, (uint32_t*)v_params, pages, kv_heads, page_size};
  TDIST_REQUIRE(cache_ok(c), BAD_CACHE);
  TDIST_REQUIRE(dtype == 0 || dtype == 1, BAD_FORM);
  TDIST_REQUIRE(batch >= 0 && total >= 0 && total < (1ll << 31) && max_pages >= 0 && room_ok(c, max_pages), "bad batch / row count");
  if (batch == 0 || total == 0) return 0;
  TDIST_REQUIRE((table || max_pages == 0) && cu && k_out && v_out, "null argument");
  TDIST_REQUIRE((((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0 && ((k_st | k_sh | v_st | v_sh) & 7) == 0,
                "output rows must keep 16-byte alignment");
  TDIST_REQUIRE(total * kv_heads < (1ll << 31), TOO_MANY);
  bool fits = true;
  const bool ok = dispatch(dtype, head_dim, group, [&](auto bf, auto d, auto g) {
    // short sequences: as few of them in a wave as there can be
    using T = Tile<decltype(d)::value>;
    const int rows_each = total <= 4ll * batch ? T::ROWS : T::TILE;
    const long long tiles = (total + rows_each - 1) / rows_each;
    const int waves = (int)std::min(tiles, 4ll);
    fits = grid_ok((tiles + waves - 1) / waves * 2 * kv_heads, waves);
    if (!fits) return;
    hipLaunchKernelGGL((kv4_read_kernel<decltype(bf)::value, decltype(d)::value, decltype(g)::value>),
                       dim3((unsigned)((tiles + waves - 1) / waves * 2 * kv_heads)), dim3(64 * waves), 0, (hipStream_t)stream, c,
                       table, table_stride, max_pages, cu, starts, batch, total, rows_each, (uint16_t*)k_out, (uint16_t*)v_out, k_st, k_sh,
                       v_st, v_sh);
  });
  TDIST_REQUIRE(ok, BAD_FORM);
  TDIST_REQUIRE(fits, TOO_MANY);
  TDIST_HIP_TRY(hipGetLastError());
  return 0;
}
