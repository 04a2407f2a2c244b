// GQA attention of the last tokens of each sequence over a 4-bit KV cache (format and layout: tdist/kv4.hpp).
//
// One workgroup of four waves takes one (sequence, KV head, block of sixteen query columns, KV split); a column is one
// (new token, query head) of the `group` heads that share the KV head.  A wave walks 32-token blocks with a softmax state
// of its own; the four states are merged through LDS, the splits by a second launch.
//
//   S^T[token, column] = K . Q^T.  A dword of K codes becomes four registers of two 16-bit numbers 16 + code (the code
//   is put into the significand of 16.0: a shift and one and-or each), which is what a 16x16x32 MFMA takes.  The
//   accumulator starts at -16 sum(q) of the group, so what comes out is sum(q code), and with a token's scale and low
//       s = scale * sum(q code) + low * sum(q).
//   O^T[channel, column] = V^T . P^T.  The scale belongs to a token, the axis that is summed: it goes into P.  P * scale is
//   split into two bf16 numbers (high and low part, 16 significant bits together) and multiplied twice: a single 8-bit
//   rounding of P would be as large as the rounding of the result.  The 16 of 16 + code and low come off at the end:
//       O = sum(p scale (16 + code)) + sum(p (low - 16 scale)).
//   The 32 tokens of a block are contracted in the order in which the S^T accumulators hold them, which is how the V
//   codes are stored, so neither side moves between lanes.
// The running maximum is only raised (and the sums rescaled) when a score exceeds it by 2^8: P up to 256 costs nothing
// in floating point, and the cross-lane maximum leaves the loop.
#include "tdist/gemm_gfx950.hpp"
#include "tdist/kv4.hpp"

namespace {

using namespace tdist::kv4;
using tdist::gemm::f32x4;
using tdist::gemm::Frag;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;

struct AttnArgs {
  Cache c;
  const uint16_t* q;        // [batch, S, q_heads, D]
  const int* table;         // [batch, max_pages]
  const int* kv_len;        // [batch], the S new tokens included
  float* partial;           // splits > 1: [rows, splits, D] sums over their own weight, rows = batch * S * q_heads
  float* partial_lse;       // and [rows, splits] log2-sum-exp2 (-inf: no token)
  void* out;                // [batch, S, q_heads, D] (out_mode 1) or fp32 [.., D + 1] with the log-sum-exp (out_mode 2)
  long long q_sb, q_ss, q_sh;
  int table_stride, max_pages;
  int batch, S, q_heads, splits, causal, out_mode;
  float scale, soft_cap;
};

// 16 + code as 16-bit numbers: the code sits below the leading significand bit of 16.0, at bit POS
template <bool IS_BF16>
struct Unpack {
  static constexpr uint32_t MAGIC = IS_BF16 ? 0x41804180u : 0x4c004c00u;
  static constexpr int POS = IS_BF16 ? 3 : 6;
  template <int N>        // nibbles N and N + 4 of w
  static __device__ __forceinline__ uint32_t pair(uint32_t w) {
    constexpr uint32_t MASK = 0x000f000fu << POS;
    if constexpr (POS > 4 * N) {
      return ((w << (POS - 4 * N)) & MASK) | MAGIC;
    } else {
      return ((w >> (4 * N - POS)) & MASK) | MAGIC;
    }
  }
};

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_fast(float x) { return __builtin_amdgcn_logf(x); }

template <bool IS_BF16, int D, int G>
__global__ __launch_bounds__(256) void kv4_attn_kernel(AttnArgs a) {
  using F = Frag<IS_BF16>;
  using QT = typename F::T;
  constexpr int KS = D / 32;            // MFMA steps over the head dim = dwords of a lane per K row
  constexpr int NT = D / 16;            // 16-channel tiles of V
  constexpr int NG = D / G;
  constexpr int GS = G / 32, GT = G / 16;
  constexpr int VW = D / 32;            // dwords of V codes per lane and four tokens
  constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
  constexpr float NONE = -1e30f;        // the running maximum before the first token
  constexpr int DC = D < 128 ? D : 128; // channels merged at a time
  __shared__ float s_m[4][16], s_l[4][16];
  __shared__ __attribute__((aligned(16))) float s_o[4][16][DC + 4];

  const int pairs = a.batch * a.c.kv_heads;
  const int cblk = blockIdx.x / pairs, pair = blockIdx.x - cblk * pairs;    // (columns of one KV head: on the same XCD if pairs % 8 == 0)
  const int b = pair / a.c.kv_heads, kvh = pair - b * a.c.kv_heads;
  const int group = a.q_heads / a.c.kv_heads, columns = group * a.S;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, lg = lane >> 4;
  const int col = cblk * 16 + li;
  const bool col_ok = col < columns;
  const int row_s = col_ok ? col / group : 0, head = kvh * group + (col_ok ? col - row_s * group : 0);

  // tokens: this column sees [0, limit), the block of columns [0, len), none of them masked below `full`
  const long long room = (long long)a.max_pages * a.c.page_size;
  const int L = (int)min((long long)max(a.kv_len[b], 0), room);
  const int s_first = cblk * 16 / group, s_last = min(cblk * 16 + 15, columns - 1) / group;
  const int limit = !col_ok ? 0 : a.causal ? L - a.S + row_s + 1 : L;
  const int len = max(0, a.causal ? L - a.S + s_last + 1 : L);
  const int full = a.causal ? L - a.S + s_first + 1 : L;
  const int per = ((len + a.splits - 1) / a.splits + 127) & ~127;
  const int start = (int)blockIdx.y * per, end = min(len, start + per);
  if (a.splits > 1 && start >= end) {       // (the merge does not look at the sums of a split without tokens)
    if (wave == 0 && lg == 0 && col_ok)
      a.partial_lse[(((long long)b * a.S + row_s) * a.q_heads + head) * a.splits + blockIdx.y] = -INFINITY;
    return;
  }

  QT qreg[KS];
  float qsum[NG];
  {
    const uint16_t* qp = a.q + b * a.q_sb + row_s * a.q_ss + head * a.q_sh + lg * 8;
    float part[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) part[g] = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      u32x4 v = u32x4{0, 0, 0, 0};
      if (col_ok) v = *(const u32x4*)(qp + 32 * s);
      qreg[s] = __builtin_bit_cast(QT, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) part[s / GS] += from16<IS_BF16>(v[i] & 0xffffu) + low_of<IS_BF16>(v[i]);
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      part[g] += __shfl_xor(part[g], 16);
      qsum[g] = part[g] + __shfl_xor(part[g], 32);
    }
  }

  float m = NONE, l = 0.f, corr[NG];
  f32x4 o[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) o[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int g = 0; g < NG; ++g) corr[g] = 0.f;
  const float qk = a.soft_cap > 0.f ? a.scale / a.soft_cap : a.scale * LOG2E;
  const int* table = a.table + (long long)b * a.table_stride;

  for (int n0 = start + 32 * wave; n0 < end; n0 += 128) {
    uint32_t kw[2][KS], vw[2][VW], kp[2][NG][4], vp[2][NG][4];
    bool there[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int tok = __builtin_amdgcn_readfirstlane(n0 + 16 * t);
      const Place at = place_of(a.c, table, tok < end ? tok : -1, a.max_pages);
      there[t] = at.page >= 0;
      const long long row0 = ((long long)max(at.page, 0) * a.c.kv_heads + kvh) * a.c.page_size;
      const uint32_t* kc = (const uint32_t*)(a.c.k_codes + (row0 + at.off + li) * (D / 2)) + lg * KS;
      const uint32_t* vc = (const uint32_t*)(a.c.v_codes + (row0 + at.off + 4 * lg) * (D / 2)) + li * VW;
#pragma unroll
      for (int i = 0; i < KS; ++i) kw[t][i] = kc[i];
#pragma unroll
      for (int i = 0; i < VW; ++i) vw[t][i] = vc[i];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const long long at_p = row0 * NG + (long long)g * a.c.page_size + at.off + 4 * lg;
        const u32x4 kk = *(const u32x4*)(a.c.k_params + at_p), vv = *(const u32x4*)(a.c.v_params + at_p);
#pragma unroll
        for (int i = 0; i < 4; ++i) kp[t][g][i] = kk[i], vp[t][g][i] = vv[i];
      }
    }

    // ---- scores (in units of log2): token n0 + 16 t + 4 lg + i, column li
    float sc[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[t][i] = 0.f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const float c0 = -16.f * qsum[g];
        f32x4 acc = f32x4{c0, c0, c0, c0};
#pragma unroll
        for (int s = g * GS; s < (g + 1) * GS; ++s) {
          using U = Unpack<IS_BF16>;
          const uint32_t w = kw[t][s];
          const u32x4 k = u32x4{U::template pair<0>(w), U::template pair<1>(w), U::template pair<2>(w), U::template pair<3>(w)};
          acc = F::mfma(__builtin_bit_cast(QT, k), qreg[s], acc);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          sc[t][i] += scale_of<IS_BF16>(kp[t][g][i]) * acc[i] + low_of<IS_BF16>(kp[t][g][i]) * qsum[g];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[t][i] *= qk;
      if (a.soft_cap > 0.f) {
#pragma unroll
        for (int i = 0; i < 4; ++i)       // cap tanh(x) = cap (1 - 2 / (e^2x + 1))
          sc[t][i] = a.soft_cap * LOG2E * (1.f - 2.f / (exp2_fast(2.f * LOG2E * sc[t][i]) + 1.f));
      }
    }
    // ---- masks: the parameters of tokens that are not there may hold anything, so they are cleared, not multiplied away
    const bool masked = n0 + 32 > min(full, end) || !there[0] || !there[1];
    if (masked) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int tok = n0 + 16 * t + 4 * lg + i;
          if (!there[t] || tok >= min(limit, end)) sc[t][i] = -INFINITY;
        }
    }
    float top = sc[0][0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, sc[i >> 2][i & 3]);
    if (__any(top > m + 8.f)) {
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float m_new = fmaxf(m, top), f = exp2_fast(m - m_new);
      m = m_new;
      l *= f;
#pragma unroll
      for (int g = 0; g < NG; ++g) corr[g] *= f;
#pragma unroll
      for (int j = 0; j < NT; ++j) o[j] *= f;
    }
    float p[2][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i >> 2][i & 3] = exp2_fast(sc[i >> 2][i & 3] - m);
      l += p[i >> 2][i & 3];
    }
    // ---- O^T += V^T . P^T
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      bf16x8 hi, lo;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float s = scale_of<IS_BF16>(vp[i >> 2][g][i & 3]), low = low_of<IS_BF16>(vp[i >> 2][g][i & 3]);
        if (masked) {
          const bool off = sc[i >> 2][i & 3] == -INFINITY;
          s = off ? 0.f : s, low = off ? 0.f : low;
        }
        const float ps = p[i >> 2][i & 3] * s;
        corr[g] += p[i >> 2][i & 3] * low - 16.f * ps;
        hi[i] = (__bf16)ps;
        lo[i] = (__bf16)(ps - (float)hi[i]);
      }
#pragma unroll
      for (int j = g * GT; j < (g + 1) * GT; ++j) {
        using U = Unpack<true>;
        const uint32_t w0 = vw[0][j / 4 * 2], w1 = vw[0][j / 4 * 2 + 1], w2 = vw[1][j / 4 * 2], w3 = vw[1][j / 4 * 2 + 1];
        u32x4 v;
        if (j % 4 == 0) v = u32x4{U::pair<0>(w0), U::pair<0>(w1), U::pair<0>(w2), U::pair<0>(w3)};
        else if (j % 4 == 1) v = u32x4{U::pair<1>(w0), U::pair<1>(w1), U::pair<1>(w2), U::pair<1>(w3)};
        else if (j % 4 == 2) v = u32x4{U::pair<2>(w0), U::pair<2>(w1), U::pair<2>(w2), U::pair<2>(w3)};
        else v = u32x4{U::pair<3>(w0), U::pair<3>(w1), U::pair<3>(w2), U::pair<3>(w3)};
        o[j] = Frag<true>::mfma(__builtin_bit_cast(typename Frag<true>::T, v), __builtin_bit_cast(typename Frag<true>::T, hi), o[j]);
        o[j] = Frag<true>::mfma(__builtin_bit_cast(typename Frag<true>::T, v), __builtin_bit_cast(typename Frag<true>::T, lo), o[j]);
      }
    }
  }

  // ---- one column's sums are spread over the four lane groups
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    corr[g] += __shfl_xor(corr[g], 16);
    corr[g] += __shfl_xor(corr[g], 32);
  }
  if (lg == 0) s_m[wave][li] = m, s_l[wave][li] = l;
  __syncthreads();

  // thread (column c, part): merges the four waves' states for channels part * 4 + 64 i
  const int mc = threadIdx.x >> 4, part = threadIdx.x & 15;
  const int mcol = cblk * 16 + mc;
  const float m_all = fmaxf(fmaxf(s_m[0][mc], s_m[1][mc]), fmaxf(s_m[2][mc], s_m[3][mc]));
  float f[4], l_all = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[w] = exp2_fast(s_m[w][mc] - m_all);
    l_all += s_l[w][mc] * f[w];
  }
  const float inv = l_all != 0.f ? 1.f / l_all : 0.f;
  const float lse = l_all != 0.f ? m_all + log2_fast(l_all) : -INFINITY;
  const int ms = mcol / group, mh = kvh * group + (mcol - ms * group);
  const long long row = ((long long)b * a.S + ms) * a.q_heads + mh;
  float* prow = a.partial + (row * a.splits + blockIdx.y) * D;
#pragma unroll
  for (int d0 = 0; d0 < D; d0 += DC) {
    if (d0) __syncthreads();
#pragma unroll
    for (int j = d0 / 16; j < (d0 + DC) / 16; ++j) {
      f32x4 v = o[j];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += corr[j / GT];
      *(f32x4*)&s_o[wave][li][(j - d0 / 16) * 16 + 4 * lg] = v;
    }
    __syncthreads();
    if (mcol < columns) {
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
  if (mcol < columns && part == 0) {
    if (a.splits > 1) a.partial_lse[row * a.splits + blockIdx.y] = lse;
    else if (a.out_mode == 2) ((float*)a.out)[row * (D + 1) + D] = lse * LN2;
  }
}

// One workgroup merges the splits of one row; wave w takes splits w, w + 4, ...
template <bool IS_BF16, int D>
__global__ __launch_bounds__(256) void kv4_merge_kernel(const float* __restrict__ partial, const float* __restrict__ lse, int splits,
                                                        void* __restrict__ out, int out_mode) {
  constexpr int V = D / 64;             // channels of a lane
  __shared__ float s_acc[4][D];
  const long long row = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float* l = lse + row * splits;
  float top = -INFINITY;
  for (int s = lane; s < splits; s += 64) top = fmaxf(top, l[s]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  if (top == -INFINITY) top = 0.f;      // no split has a token (or what they have is NaN, which the weights keep)
  float sum = 0.f;
  for (int s = lane; s < splits; s += 64) sum += exp2_fast(l[s] - top);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  float acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll 4
  for (int s = wave; s < splits; s += 4) {
    const float w = exp2_fast(l[s] - top);
    const float* p = partial + (row * splits + s) * D + lane * V;
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] += w != 0.f ? w * p[i] : 0.f;     // (a split without tokens has written no sums)
  }
#pragma unroll
  for (int i = 0; i < V; ++i) s_acc[wave][lane * V + i] = acc[i];
  __syncthreads();
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  for (int c = threadIdx.x; c < D; c += 256) {
    const float r = (s_acc[0][c] + s_acc[1][c] + s_acc[2][c] + s_acc[3][c]) * inv;
    if (out_mode == 2) ((float*)out)[row * (D + 1) + c] = r;
    else ((uint16_t*)out)[row * D + c] = to16<IS_BF16>(r);
  }
  if (out_mode == 2 && threadIdx.x == 0)
    ((float*)out)[row * (D + 1) + D] = sum != 0.f ? (top + log2_fast(sum)) * 0.6931471805599453f : -INFINITY;
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
TDIST_API int tdist_kv4_attn(const void* k_codes, const void* v_codes, const void* k_params, const void* v_params, int pages,
                             int kv_heads, int page_size, int head_dim, int group, const void* q, long long q_sb, long long q_ss,
                             long long q_sh, const int* table, int table_stride, int max_pages, const int* kv_len, float* partial,
                             void* out, int batch, int S, int q_heads, int splits, int causal, int out_mode, float scale,
                             float soft_cap, int dtype, void* stream) {
  AttnArgs a;
  a.c = Cache{(uint8_t*)k_codes, (uint8_t*)v_codes, (uint32_t*)k_params, (uint32_t*)v_params, pages, kv_heads, page_size};
  TDIST_REQUIRE(k_codes && v_codes && k_params && v_params && pages > 0 && kv_heads > 0 && page_size > 0 && page_size % 16 == 0 &&
                    (((uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_params | (uintptr_t)v_params) & 15) == 0,
                "a 4-bit cache needs four 16-byte aligned tensors, pages of a multiple of 16 tokens");
  TDIST_REQUIRE(batch >= 0 && S >= 0 && q_heads > 0 && q_heads % kv_heads == 0 && max_pages >= 0, "bad head counts");
  TDIST_REQUIRE(splits >= 1 && splits <= 65535 && (splits == 1 || partial), "splits need their partial rows");
  TDIST_REQUIRE((out_mode == 1 || out_mode == 2) && (dtype == 0 || dtype == 1), "out_mode must be 1 or 2, dtype 0 (bf16) or 1 (fp16)");
  if (batch == 0 || S == 0) return 0;
  TDIST_REQUIRE(q && table && kv_len && out, "null argument");
  TDIST_REQUIRE(((uintptr_t)q & 15) == 0 && ((uintptr_t)out & 7) == 0 && ((q_sb | q_ss | q_sh) & 7) == 0,
                "q rows must keep 16-byte alignment");
  const long long cblocks = ((long long)(q_heads / kv_heads) * S + 15) / 16, blocks = cblocks * batch * kv_heads;
  TDIST_REQUIRE(blocks < (1ll << 31) && (long long)batch * S * q_heads < (1ll << 31), "too many query rows");
  a.q = (const uint16_t*)q, a.table = table, a.kv_len = kv_len, a.partial = partial, a.out = out;
  a.partial_lse = partial ? partial + (long long)batch * S * q_heads * splits * head_dim : nullptr;
  a.q_sb = q_sb, a.q_ss = q_ss, a.q_sh = q_sh, a.table_stride = table_stride, a.max_pages = max_pages;
  a.batch = batch, a.S = S, a.q_heads = q_heads, a.splits = splits, a.causal = causal, a.out_mode = out_mode;
  a.scale = scale, a.soft_cap = soft_cap;
  const bool ok = dispatch(dtype, head_dim, group, [&](auto bf, auto d, auto g) {
    hipLaunchKernelGGL((kv4_attn_kernel<decltype(bf)::value, decltype(d)::value, decltype(g)::value>),
                       dim3((unsigned)blocks, splits), dim3(256), 0, (hipStream_t)stream, a);
  });
  TDIST_REQUIRE(ok, "head_dim 64 / 128 / 256 with groups of 32 / 64 / 128 channels (at most head_dim)");
  TDIST_HIP_TRY(hipGetLastError());
  if (splits == 1) return 0;
  const long long rows = (long long)batch * S * q_heads;
  dispatch(dtype, head_dim, group, [&](auto bf, auto d, auto) {
    hipLaunchKernelGGL((kv4_merge_kernel<decltype(bf)::value, decltype(d)::value>), dim3((unsigned)rows), dim3(256), 0,
                       (hipStream_t)stream, a.partial, a.partial_lse, splits, out, out_mode);
  });
  TDIST_HIP_TRY(hipGetLastError());
  return 0;
}
