// Writing and reading a 4-bit KV cache (format and layout: tdist/kv4.hpp).
//
//   kv4_append    K / V rows of new tokens -> codes and group parameters
//   kv4_qkv_prep  the same from a QKV projection, with the heads' RMSNorm and rotation in front (and q out)
//   kv4_read      pages -> 16-bit rows, the sequences packed one behind the other
//
// All three move rows once and are bound by memory; a lane works on eight neighbouring channels (16 bytes of a 16-bit
// row), D / 8 lanes on a row, so a group's minimum and maximum are G / 8 lanes' and stay inside a wave.
// This file is compiled without fast-math: the code of a value next to a border is decided by IEEE arithmetic and is
// the same on every path that writes a cache, the CPU's included.
#include "tdist/kv4.hpp"

namespace {

using namespace tdist::kv4;

template <bool IS_BF16>
__device__ __forceinline__ void unpack_row8(const uint4& v, float (&x)[8]) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = from16<IS_BF16>(u[i] & 0xffffu);
    x[2 * i + 1] = low_of<IS_BF16>(u[i]);
  }
}
template <bool IS_BF16>
__device__ __forceinline__ uint4 pack_row8(const float (&x)[8]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = to16<IS_BF16>(x[2 * i]) | to16<IS_BF16>(x[2 * i + 1]) << 16;
  return uint4{u[0], u[1], u[2], u[3]};
}

// Codes of the lane's eight channels and the parameter dword of their group.
//
// The quotient has to be the IEEE one.  With r = RN(1 / s), q0 = RN(d r) is within an ulp of it, d - q0 s is exact in
// one fma and q = RN(q0 + (d - q0 s) r) is the correctly rounded quotient (Markstein's theorem; its one exception, a
// divisor whose significand is all ones, cannot be a 16-bit number).  That is three operations a channel instead of
// a division's ten; scales so small or large that an intermediate could leave the normal range take the division.
template <bool IS_BF16, int G>
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], uint32_t (&code)[8]) {
  float lo = x[0], hi = x[0], odd = x[0] * 0.f;       // odd: NaN if any value is an infinity or a NaN
#pragma unroll
  for (int e = 1; e < 8; ++e) lo = fminf(lo, x[e]), hi = fmaxf(hi, x[e]), odd += x[e] * 0.f;
#pragma unroll
  for (int o = 1; o < G / 8; o <<= 1) {
    lo = fminf(lo, __shfl_xor(lo, o));
    hi = fmaxf(hi, __shfl_xor(hi, o));
    odd += __shfl_xor(odd, o);
  }
  const float range = (hi - lo) + odd;
  const uint32_t s16 = range < INFINITY ? to16<IS_BF16>(range / 15.f) : to16<IS_BF16>(NAN);
  const float s = from16<IS_BF16>(s16);
  if (s > 0x1p-100f && s < 0x1p100f) {
    const float r = 1.f / s;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = x[e] - lo;
      const float q0 = d * r;
      const float q = __builtin_fmaf(__builtin_fmaf(-q0, s, d), r, q0);
      code[e] = (uint32_t)fminf(__builtin_rintf(q), 15.f);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) code[e] = s > 0.f ? (uint32_t)fminf(__builtin_rintf((x[e] - lo) / s), 15.f) : 0u;
  }
  return s16 | to16<IS_BF16>(lo) << 16;               // (lo is one of the row's 16-bit values)
}

// Quantises a row held eight channels a lane (lane l8 of D / 8) and writes it to (page, head, token `off` of the page).
// Every lane of the wave calls it; rows that go nowhere have page < 0.
template <bool IS_BF16, int D, int G, bool IS_V>
__device__ __forceinline__ void store_row(const Cache& c, const float (&x)[8], int l8, int page, int head, int off) {
  uint32_t code[8];
  const uint32_t param = quantise8<IS_BF16, G>(x, code);
  const long long row0 = ((long long)page * c.kv_heads + head) * c.page_size;      // first token of (page, head)
  if constexpr (!IS_V) {
    if (page < 0) return;
    uint32_t w = 0;
#pragma unroll
    for (int n = 0; n < 4; ++n) w |= code[2 * n] << (4 * n) | code[2 * n + 1] << (16 + 4 * n);
    const int word = (l8 & 3) * (D / 32) + (l8 >> 2);
    *(uint32_t*)(c.k_codes + (row0 + off) * (D / 2) + word * 4) = w;
  } else {
    // the four lanes n = 0 .. 3 of a unit hold its four 16-channel tiles: two steps of exchange, in each of which a lane
    // keeps half of what it has and gives the other half away, leave each lane two whole units
    const int n = (l8 >> 1) & 3;
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = (code[2 * i] | code[2 * i + 1] << 16) << (4 * n);
    const bool up1 = n & 1, up2 = n & 2;
    const uint32_t a0 = (up1 ? u[2] : u[0]) | __shfl_xor(up1 ? u[0] : u[2], 2);
    const uint32_t a1 = (up1 ? u[3] : u[1]) | __shfl_xor(up1 ? u[1] : u[3], 2);
    const uint32_t b = (up2 ? a1 : a0) | __shfl_xor(up2 ? a0 : a1, 4);
    if (page < 0) return;
    const int ch = (l8 & 1) * 8 + (up1 ? 4 : 0) + (up2 ? 2 : 0);                    // this lane's units: channels ch, ch + 1
    uint8_t* p = c.v_codes + row0 * (D / 2) + (long long)(off >> 2) * (2 * D) + (l8 >> 3) * 8 + (off & 3) * 2;
    *(uint16_t*)(p + ch * (D / 8)) = (uint16_t)b;
    *(uint16_t*)(p + (ch + 1) * (D / 8)) = (uint16_t)(b >> 16);
  }
  if (l8 % (G / 8) == 0) {
    uint32_t* params = IS_V ? c.v_params : c.k_params;
    params[row0 * (D / G) + (long long)(l8 / (G / 8)) * c.page_size + off] = param;
  }
}

// grid: (tiles of tokens, Hkv heads of K then Hkv of V, batch)
template <bool IS_BF16, int D, int G>
__global__ __launch_bounds__(256) void kv4_append_kernel(Cache c, const uint16_t* __restrict__ k, const uint16_t* __restrict__ v,
                                                         long long k_sb, long long k_ss, long long k_sh, long long v_sb,
                                                         long long v_ss, long long v_sh, const int* __restrict__ kv_offset,
                                                         const int* __restrict__ new_lens, const int* __restrict__ table,
                                                         int table_stride, int max_pages, int S) {
  constexpr int LANES = D / 8;
  const int b = blockIdx.z, l8 = threadIdx.x % LANES;
  const int s = blockIdx.x * (blockDim.x / LANES) + threadIdx.x / LANES;
  const bool is_v = (int)blockIdx.y >= c.kv_heads;
  const int head = blockIdx.y - (is_v ? c.kv_heads : 0);
  const int count = new_lens ? min(new_lens[b], S) : S;
  const bool live = s < count;
  const long long pos = (long long)kv_offset[b] + s;
  const Place at = place_of(c, table + (long long)b * table_stride, live ? pos : -1, max_pages);
  float x[8];
  uint4 raw = uint4{0, 0, 0, 0};
  if (live)
    raw = *(const uint4*)((is_v ? v + b * v_sb + s * v_ss + head * v_sh : k + b * k_sb + s * k_ss + head * k_sh) + l8 * 8);
  unpack_row8<IS_BF16>(raw, x);
  if (is_v) {
    store_row<IS_BF16, D, G, true>(c, x, l8, at.page, head, at.off);
  } else {
    store_row<IS_BF16, D, G, false>(c, x, l8, at.page, head, at.off);
  }
}

// grid: (tiles of tokens, Hq heads of q, Hkv of K, Hkv of V, batch).  The norm's mean square and the rotation are taken in
// 64 bits, so that a stored code does not depend on the order of a sum.
template <int D, int G>
__global__ __launch_bounds__(256) void kv4_qkv_prep_kernel(Cache c, const uint16_t* __restrict__ qkv, long long q_sb,
                                                           long long q_ss, const uint16_t* __restrict__ q_w,
                                                           const uint16_t* __restrict__ k_w, float q_eps, float k_eps,
                                                           const long long* __restrict__ positions,
                                                           const float* __restrict__ cos_t, const float* __restrict__ sin_t,
                                                           long long rope_rows, uint16_t* __restrict__ q_out,
                                                           const int* __restrict__ kv_offset, int* __restrict__ total_out,
                                                           const int* __restrict__ table, int table_stride, int max_pages,
                                                           int S, int q_heads) {
  constexpr int LANES = D / 8;
  const int b = blockIdx.z, l8 = threadIdx.x % LANES;
  const int s = blockIdx.x * (blockDim.x / LANES) + threadIdx.x / LANES;
  const int head = blockIdx.y;
  const int offset = kv_offset[b];
  if (head == 0 && s == 0 && l8 == 0) total_out[b] = offset + S;
  const bool live = s < S, is_q = head < q_heads, is_v = head >= q_heads + c.kv_heads;
  const long long pos = (long long)offset + s;
  const Place at = place_of(c, table + (long long)b * table_stride, live && !is_q ? pos : -1, max_pages);
  float x[8];
  uint4 raw = uint4{0, 0, 0, 0};
  if (live) raw = *(const uint4*)(qkv + b * q_sb + s * q_ss + (long long)head * D + l8 * 8);
  unpack_row8<true>(raw, x);
  if (is_v) {
    store_row<true, D, G, true>(c, x, l8, at.page, head - q_heads - c.kv_heads, at.off);
    return;
  }
  const uint16_t* w = is_q ? q_w : k_w;
  if (w) {
    double ss = 0.;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += (double)x[e] * x[e];
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) ss += __shfl_xor(ss, o);
    const float inv = (float)(1. / __builtin_sqrt(ss / D + (double)(is_q ? q_eps : k_eps)));
    float g[8];
    unpack_row8<true>(*(const uint4*)(w + l8 * 8), g);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = from16<true>(to16<true>(x[e] * inv * g[e]));
  }
  {
    // pairs (i, i + D / 2) are the same element of lanes l8 and l8 ^ (D / 16)
    long long p = live ? positions[(long long)b * S + s] : 0;
    p = p < 0 ? 0 : p < rope_rows ? p : rope_rows - 1;
    const int i0 = (l8 * 8) % (D / 2);
    const float* cs = cos_t + p * (D / 2) + i0;
    const float* sn = sin_t + p * (D / 2) + i0;
    const double sign = l8 < LANES / 2 ? -1. : 1.;
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float other = __shfl_xor(x[e], LANES / 2);
      y[e] = (float)((double)x[e] * cs[e] + sign * other * sn[e]);
      asm volatile("" : "+v"(y[e]));          // 64 -> 32 -> 16 bits as two roundings, which the compiler would merge
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = from16<true>(to16<true>(y[e]));
  }
  if (is_q) {
    if (live) *(uint4*)(q_out + (((long long)b * S + s) * q_heads + head) * D + l8 * 8) = pack_row8<true>(x);
    return;
  }
  store_row<true, D, G, false>(c, x, l8, at.page, head - q_heads, at.off);
}

// grid: (tiles of output rows, Hkv heads of K then Hkv of V).  Row r belongs to the sequence b with cu[b] <= r < cu[b + 1].
template <bool IS_BF16, int D, int G>
__global__ __launch_bounds__(256) void kv4_read_kernel(Cache c, const int* __restrict__ table, int table_stride, int max_pages,
                                                       const int* __restrict__ cu, const int* __restrict__ starts, int batch,
                                                       long long total, uint16_t* __restrict__ k_out,
                                                       uint16_t* __restrict__ v_out, long long k_st, long long k_sh,
                                                       long long v_st, long long v_sh) {
  constexpr int LANES = D / 8;
  constexpr float MOST = IS_BF16 ? 0x1.fep127f : 65504.f;
  const int l8 = threadIdx.x % LANES;
  const long long r = (long long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const bool is_v = (int)blockIdx.y >= c.kv_heads;
  const int head = blockIdx.y - (is_v ? c.kv_heads : 0);
  const long long end = min(total, (long long)cu[batch]);
  if (r >= end || r < cu[0]) return;
  int b = 0, top = batch;                 // cu[b] <= r < cu[top]
  while (top - b > 1) {
    const int mid = (b + top) >> 1;
    if (cu[mid] <= r) b = mid; else top = mid;
  }
  const long long pos = (starts ? (long long)starts[b] : 0) + (r - cu[b]);
  const Place at = place_of(c, table + (long long)b * table_stride, pos, max_pages);
  const int off = at.off;
  float x[8];
  if (at.page < 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.f;
  } else {
    const long long row0 = ((long long)at.page * c.kv_heads + head) * c.page_size;
    uint32_t code[8];
    if (!is_v) {
      const int word = (l8 & 3) * (D / 32) + (l8 >> 2);
      const uint32_t w = *(const uint32_t*)(c.k_codes + (row0 + off) * (D / 2) + word * 4);
#pragma unroll
      for (int n = 0; n < 4; ++n) code[2 * n] = w >> (4 * n) & 15u, code[2 * n + 1] = w >> (16 + 4 * n) & 15u;
    } else {
      const uint8_t* p = c.v_codes + row0 * (D / 2) + (long long)(off >> 2) * (2 * D) + (l8 >> 3) * 8 + (off & 3) * 2;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        code[e] = (uint32_t)*(const uint16_t*)(p + ((l8 & 1) * 8 + e) * (D / 8)) >> (4 * ((l8 >> 1) & 3)) & 15u;
    }
    const uint32_t param = (is_v ? c.v_params : c.k_params)[row0 * (D / G) + (long long)(l8 / (G / 8)) * c.page_size + off];
    const float s = scale_of<IS_BF16>(param), lo = low_of<IS_BF16>(param);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float value = __builtin_fmaf(s, (float)code[e], lo);
      x[e] = value > MOST ? MOST : value;               // (a scale that was rounded up; a NaN stays one)
    }
  }
  uint16_t* dst = is_v ? v_out + r * v_st + head * v_sh : k_out + r * k_st + head * k_sh;
  *(uint4*)(dst + l8 * 8) = pack_row8<IS_BF16>(x);
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
  TDIST_REQUIRE(batch >= 0 && batch <= 65535 && S >= 0 && max_pages >= 0, "bad batch / token count");
  if (batch == 0 || S == 0) return 0;
  TDIST_REQUIRE(k && v && kv_offset && table, "null argument");
  TDIST_REQUIRE((((uintptr_t)k | (uintptr_t)v) & 15) == 0 && ((k_sb | k_ss | k_sh | v_sb | v_ss | v_sh) & 7) == 0,
                "k / v rows must keep 16-byte alignment");
  const int threads = (long long)S * head_dim <= 512 ? 64 : 256;      // (a decode step's one token fills part of a wave)
  const int rows = threads / (head_dim / 8 > 0 ? head_dim / 8 : 1);
  const bool ok = dispatch(dtype, head_dim, group, [&](auto bf, auto d, auto g) {
    hipLaunchKernelGGL((kv4_append_kernel<decltype(bf)::value, decltype(d)::value, decltype(g)::value>),
                       dim3((S + rows - 1) / rows, 2 * kv_heads, batch), dim3(threads), 0, (hipStream_t)stream, c,
                       (const uint16_t*)k, (const uint16_t*)v, k_sb, k_ss, k_sh, v_sb, v_ss, v_sh, kv_offset, new_lens, table,
                       table_stride, max_pages, S);
  });
  TDIST_REQUIRE(ok, BAD_FORM);
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
  TDIST_REQUIRE(batch >= 0 && batch <= 65535 && S >= 0 && max_pages >= 0 && q_heads > 0 && q_heads <= 32767 && rope_rows > 0,
                "bad batch / token / head count");
  if (batch == 0 || S == 0) return 0;
  TDIST_REQUIRE(qkv && positions && cos_t && sin_t && q_out && kv_offset && total_out && table, "null argument");
  TDIST_REQUIRE((((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)q_w | (uintptr_t)k_w) & 15) == 0 && ((q_sb | q_ss) & 7) == 0,
                "qkv rows, norm weights and q must keep 16-byte alignment");
  const int threads = (long long)S * head_dim <= 512 ? 64 : 256;
  const int rows = threads / (head_dim / 8 > 0 ? head_dim / 8 : 1);
  const bool ok = dispatch(0, head_dim, group, [&](auto bf, auto d, auto g) {
    if constexpr (decltype(bf)::value)
      hipLaunchKernelGGL((kv4_qkv_prep_kernel<decltype(d)::value, decltype(g)::value>),
                         dim3((S + rows - 1) / rows, q_heads + 2 * kv_heads, batch), dim3(threads), 0, (hipStream_t)stream, c,
                         (const uint16_t*)qkv, q_sb, q_ss, (const uint16_t*)q_w, (const uint16_t*)k_w, q_eps, k_eps, positions,
                         cos_t, sin_t, rope_rows, (uint16_t*)q_out, kv_offset, total_out, table, table_stride, max_pages, S,
                         q_heads);
  });
  TDIST_REQUIRE(ok, BAD_FORM);
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
  TDIST_REQUIRE(batch >= 0 && total >= 0 && total < (1ll << 31) && max_pages >= 0, "bad batch / row count");
  if (batch == 0 || total == 0) return 0;
  TDIST_REQUIRE(table && cu && k_out && v_out, "null argument");
  TDIST_REQUIRE((((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0 && ((k_st | k_sh | v_st | v_sh) & 7) == 0,
                "output rows must keep 16-byte alignment");
  const int rows = 256 / (head_dim / 8 > 0 ? head_dim / 8 : 1);
  const bool ok = dispatch(dtype, head_dim, group, [&](auto bf, auto d, auto g) {
    hipLaunchKernelGGL((kv4_read_kernel<decltype(bf)::value, decltype(d)::value, decltype(g)::value>),
                       dim3((unsigned)((total + rows - 1) / rows), 2 * kv_heads), dim3(256), 0, (hipStream_t)stream, c, table,
                       table_stride, max_pages, cu, starts, batch, total, (uint16_t*)k_out, (uint16_t*)v_out, k_st, k_sh, v_st,
                       v_sh);
  });
  TDIST_REQUIRE(ok, BAD_FORM);
  TDIST_HIP_TRY(hipGetLastError());
  return 0;
}
