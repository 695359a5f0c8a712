// mac_paged_cache.hip -- the 8-bit paged K/V cache for MI355X (gfx950): rows
// quantised as they are written, decode RoPE with the write, and reading back.
//
// Format.  K and V pages hold OCP e4m3 codes [pages, P, Hkv, D].  Row-scaled
// form: kv_scales [pages, Hkv, P, 2] holds one E8M0 byte e per row of K and of
// V, and an element is code * 2^(e - 127), with 2^(e - 127) the smallest power
// of two s for which max |x| <= 448 s over the row's finite elements (at least
// 2^-126).  A power of two keeps e4m3's relative precision (a scale only moves
// the exponents), makes x / s exact, so the one rounding is the code's, and
// code * s exact in bf16; gfx950's conversions apply it for nothing.  K's and
// V's bytes lie together, and a page's rows of one head after one another, so
// that attention reads both with one 2-byte load from 2 P consecutive bytes.
// Static form (kv_scales NULL): element = code * k_scale or v_scale, code =
// e4m3(x / scale) by an IEEE division.  Codes round to nearest even and
// saturate at 448; NaN and infinities become the NaN code.
//
// Layout.  A group of W lanes (the power of two that holds D / 8) owns one row,
// 8 elements per lane: one 16-byte load per 16-bit row, a maximum over the
// group, four conversions, one 8-byte store.  K and V rows of a (token, head)
// go together, so both scale bytes leave in one 2-byte store.  The kernels are
// bound by their bytes (or, for a decode batch, by the launch): a lane has all
// of its loads in flight at once and there is no loop.  Measured, 8 KV heads of
// 128 dims: 32768 tokens written in 43 us (4.7 TB/s where a device copy reaches
// 4.9), 65536 read back to bf16 in 80 (5.1 TB/s); RoPE with the write, 32 query
// heads, 2048 tokens 15 us from a warm cache (3.1 TB/s); 64 tokens, either write, 4
// to 5 us.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "mac_attention_amd.h"
#include "mac_common.h"

// Every product and sum rounds on its own (RoPE's rotated keys decide codes,
// which a contraction would make depend on the compiler's choice).
#pragma clang fp contract(off)

namespace mac {
int fail(int code, const char* fmt, ...);
}  // namespace mac

namespace {

using namespace mac;

constexpr int kThreads = 256;
constexpr float kTop = 448.0f;  // the largest e4m3 value

struct CacheParams {
  // input rows (elements): token and head strides
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;
  int q_vec, kv_vec;  // rows move as 16-byte vectors
  // cache (bytes = codes): page, slot and head strides
  uint8_t* kc;
  uint8_t* vc;
  uint16_t* scales;  // [pages, Hkv, P] (K byte low, V byte high), or NULL
  int64_t k_ps, k_ss, k_chs, v_ps, v_ss, v_chs;
  int64_t slots;  // pages * P
  int page_shift;
  const void* locs;
  int locs_i64;
  float k_scale, v_scale;
  uint32_t items;  // (token, head) rows of the launch
  int Hq, Hkv, D;
  // RoPE
  uint16_t* q_out;
  const float* cs;
  int64_t cs_stride, cs_rows;
  const void* positions;
  int pos_i64, rot, neox, cs_vec;
  // read back
  void* out_k;
  void* out_v;
};

__device__ __forceinline__ int64_t index_at(const void* p, int is_i64, int64_t n) {
  return is_i64 ? static_cast<const int64_t*>(p)[n] : static_cast<const int32_t*>(p)[n];
}

// 16-bit element types by C ABI code.
template <int kT>
__device__ __forceinline__ float to_f32(uint16_t b) {
  if constexpr (kT == MAC_DTYPE_BF16) return bf16_to_f32(b);
  else return static_cast<float>(__builtin_bit_cast(_Float16, b));
}
template <int kT>
__device__ __forceinline__ uint16_t from_f32(float f) {
  if constexpr (kT == MAC_DTYPE_BF16) return f32_to_bf16(f);
  else return __builtin_bit_cast(uint16_t, static_cast<_Float16>(f));
}

// Eight elements of a row: one 16-byte load, or one by one for rows that do
// not start on 16 bytes.
template <int kT>
__device__ __forceinline__ void load8(const uint16_t* at, int vec, float (&x)[8]) {
  uint16_t u[8];
  if (vec) {
    const uint4 w = *reinterpret_cast<const uint4*>(at);
    const uint32_t d[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u[2 * i] = static_cast<uint16_t>(d[i]);
      u[2 * i + 1] = static_cast<uint16_t>(d[i] >> 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = at[i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_f32<kT>(u[i]);
}

__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// Largest finite magnitude of the row, in every lane of its group of W.
template <int W>
__device__ __forceinline__ float row_amax(const float (&x)[8]) {
  float a = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = fmaxf(a, finite(x[i]) ? fabsf(x[i]) : 0.0f);
#pragma unroll
  for (int off = 1; off < W; off <<= 1) a = fmaxf(a, __shfl_xor(a, off));
  return a;
}

// E8M0 byte of the smallest power of two s >= 2^-126 with amax <= 448 s: 448 =
// 1.75 * 2^8, so s has amax's exponent less 8, or less 7 past a mantissa of 1.75.
__device__ __forceinline__ uint32_t scale_byte(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = static_cast<int>(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return static_cast<uint32_t>(max(e, 1));
}

// Codes of eight elements x whose quotients by their scale are y (infinite where a
// static scale is too small: those saturate).
__device__ __forceinline__ uint2 encode8(const float (&x)[8], const float (&y)[8]) {
  float c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = finite(x[i]) ? fminf(fmaxf(y[i], -kTop), kTop) : __uint_as_float(0x7fc00000u);
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(c[4], c[5], 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(c[6], c[7], hi, true);
  return make_uint2(static_cast<uint32_t>(lo), static_cast<uint32_t>(hi));
}

// Codes of a lane's eight elements and the row's scale byte.
template <int W>
__device__ __forceinline__ uint2 quantise8(const float (&x)[8], bool scaled, float factor, uint32_t& byte) {
  float y[8];
  if (scaled) {
    byte = scale_byte(row_amax<W>(x));
    const float inv = __uint_as_float((254u - byte) << 23);  // 2^(127 - byte): byte is 1 .. 247
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = x[i] * inv;
  } else {
    byte = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __fdiv_rn(x[i], factor);
  }
  return encode8(x, y);
}

// Stores a (token, head)'s lane: codes of K and V and the scale bytes.  Locs
// outside the cache are skipped.
__device__ __forceinline__ void store_row(const CacheParams& p, int64_t loc, int h, int lane8, uint2 kq, uint2 vq,
                                          uint32_t kb, uint32_t vb) {
  if (loc < 0 || loc >= p.slots) return;
  const int64_t page = loc >> p.page_shift;
  const int64_t slot = loc & ((int64_t{1} << p.page_shift) - 1);
  *reinterpret_cast<uint2*>(p.kc + page * p.k_ps + slot * p.k_ss + h * p.k_chs + 8 * lane8) = kq;
  *reinterpret_cast<uint2*>(p.vc + page * p.v_ps + slot * p.v_ss + h * p.v_chs + 8 * lane8) = vq;
  if (p.scales != nullptr && lane8 == 0)
    p.scales[((page * p.Hkv + h) << p.page_shift) + slot] = static_cast<uint16_t>(kb | (vb << 8));
}

// One group of W lanes per (token, KV head).
template <int kT, int W>
__global__ void __launch_bounds__(kThreads) cache_write_kernel(CacheParams p) {
  const uint32_t item = blockIdx.x * (kThreads / W) + threadIdx.x / W;
  const int lane8 = threadIdx.x % W;
  if (item >= p.items) return;  // (whole groups)
  const uint32_t row = item / p.Hkv;
  const int h = static_cast<int>(item - row * p.Hkv);
  const int64_t n = row;
  const bool in = 8 * lane8 < p.D;  // (a row of fewer than 8 W elements: the other lanes hold zeros)
  float kx[8] = {}, vx[8] = {};
  const int64_t loc = index_at(p.locs, p.locs_i64, n);
  if (in) {
    load8<kT>(p.k + n * p.k_ts + h * p.k_hs + 8 * lane8, p.kv_vec, kx);
    load8<kT>(p.v + n * p.v_ts + h * p.v_hs + 8 * lane8, p.kv_vec, vx);
  }
  uint32_t kb, vb;
  const uint2 kq = quantise8<W>(kx, p.scales != nullptr, p.k_scale, kb);
  const uint2 vq = quantise8<W>(vx, p.scales != nullptr, p.v_scale, vb);
  if (in) store_row(p, loc, h, lane8, kq, vq, kb, vb);
}

// RoPE of a lane's eight elements x at dims d0 .. d0 + 7 of the row at `row`:
// the pair partners come from the row itself (another lane's elements in the
// half-split style: read again, they are in the cache).
template <int kT>
__device__ __forceinline__ void rope8(const CacheParams& p, const uint16_t* row, int vec, const float* cs, int d0,
                                      float (&x)[8]) {
  const int half = p.rot >> 1;
  if (d0 >= p.rot) return;
  if (p.neox && (half & 7) == 0) {  // the lane's partners are eight elements in one run
    const bool first = d0 < half;
    const int i0 = first ? d0 : d0 - half;
    float y[8], c[8], s[8];
    load8<kT>(row + (first ? d0 + half : d0 - half), vec, y);
    if (p.cs_vec) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4 a = *reinterpret_cast<const float4*>(cs + i0 + 4 * j);
        const float4 b = *reinterpret_cast<const float4*>(cs + half + i0 + 4 * j);
        c[4 * j] = a.x; c[4 * j + 1] = a.y; c[4 * j + 2] = a.z; c[4 * j + 3] = a.w;
        s[4 * j] = b.x; s[4 * j + 1] = b.y; s[4 * j + 2] = b.z; s[4 * j + 3] = b.w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        c[e] = cs[i0 + e];
        s[e] = cs[half + i0 + e];
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = first ? x[e] * c[e] - y[e] * s[e] : x[e] * c[e] + y[e] * s[e];
    return;
  }
  if (p.neox) {  // rotary sizes whose halves the lanes' runs do not divide
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = d0 + e;
      if (d >= p.rot) break;
      const bool first = d < half;
      const int i = first ? d : d - half;
      const float y = to_f32<kT>(row[first ? d + half : d - half]);
      x[e] = first ? x[e] * cs[i] - y * cs[half + i] : x[e] * cs[i] + y * cs[half + i];
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; e += 2) {  // adjacent pairs
    if (d0 + e >= p.rot) break;
    const int i = (d0 + e) >> 1;
    const float x0 = x[e], x1 = x[e + 1], c = cs[i], s = cs[half + i];
    x[e] = x0 * c - x1 * s;
    x[e + 1] = x1 * c + x0 * s;
  }
}

// One group of W lanes per (token, head): query heads first (rotated rows to
// q_out), then KV heads (rotated K and V to the cache).
template <int kT, int W>
__global__ void __launch_bounds__(kThreads) rope_write_kernel(CacheParams p) {
  const uint32_t item = blockIdx.x * (kThreads / W) + threadIdx.x / W;
  const int lane8 = threadIdx.x % W;
  const uint32_t heads = p.Hq + p.Hkv;
  if (item >= p.items) return;
  const uint32_t token = item / heads;
  const int r = static_cast<int>(item - token * heads);
  const int64_t n = token;
  const bool in = 8 * lane8 < p.D;
  int64_t pos = index_at(p.positions, p.pos_i64, n);
  pos = pos < 0 ? 0 : (pos >= p.cs_rows ? p.cs_rows - 1 : pos);
  const float* cs = p.cs + pos * p.cs_stride;
  if (r < p.Hq) {
    if (!in) return;
    const uint16_t* row = p.q + n * p.q_ts + r * p.q_hs;
    float x[8];
    load8<kT>(row + 8 * lane8, p.q_vec, x);
    rope8<kT>(p, row, p.q_vec, cs, 8 * lane8, x);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = from_f32<kT>(x[2 * i]) | (static_cast<uint32_t>(from_f32<kT>(x[2 * i + 1])) << 16);
    *reinterpret_cast<uint4*>(p.q_out + (n * p.Hq + r) * p.D + 8 * lane8) = make_uint4(w[0], w[1], w[2], w[3]);
    return;
  }
  const int h = r - p.Hq;
  const int64_t loc = index_at(p.locs, p.locs_i64, n);
  float kx[8] = {}, vx[8] = {};
  if (in) {
    const uint16_t* row = p.k + n * p.k_ts + h * p.k_hs;
    load8<kT>(row + 8 * lane8, p.kv_vec, kx);
    load8<kT>(p.v + n * p.v_ts + h * p.v_hs + 8 * lane8, p.kv_vec, vx);
    rope8<kT>(p, row, p.kv_vec, cs, 8 * lane8, kx);
  }
  uint32_t kb, vb;
  const uint2 kq = quantise8<W>(kx, p.scales != nullptr, p.k_scale, kb);
  const uint2 vq = quantise8<W>(vx, p.scales != nullptr, p.v_scale, vb);
  if (in) store_row(p, loc, h, lane8, kq, vq, kb, vb);
}

// Eight codes as f32 times their scale: the power of two inside the
// conversion (exact), a static factor by one product.
__device__ __forceinline__ void decode8(uint2 w, bool scaled, uint32_t byte, float factor, float (&x)[8]) {
  const float s = scaled ? __uint_as_float(byte << 23) : 1.0f;  // (the conversion reads the exponent: byte 0 is 2^-127)
  const uint32_t d[2] = {w.x, w.y};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(d[i], s, false);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(d[i], s, true);
    x[4 * i] = a[0]; x[4 * i + 1] = a[1]; x[4 * i + 2] = b[0]; x[4 * i + 3] = b[1];
  }
  if (!scaled) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= factor;
  }
}

template <int kT>
__device__ __forceinline__ void put8(void* out, int64_t at, const float (&x)[8]) {
  if constexpr (kT == MAC_DTYPE_F32) {
    float4* o = reinterpret_cast<float4*>(static_cast<float*>(out) + at);
    o[0] = make_float4(x[0], x[1], x[2], x[3]);
    o[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = from_f32<kT>(x[2 * i]) | (static_cast<uint32_t>(from_f32<kT>(x[2 * i + 1])) << 16);
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// One group of W lanes per (listed row, KV head); rows outside the cache read
// as zeros.
template <int kT, int W>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(CacheParams p) {
  const uint32_t item = blockIdx.x * (kThreads / W) + threadIdx.x / W;
  const int lane8 = threadIdx.x % W;
  if (item >= p.items || 8 * lane8 >= p.D) return;
  const uint32_t row = item / p.Hkv;
  const int h = static_cast<int>(item - row * p.Hkv);
  const int64_t n = row;
  const int64_t loc = index_at(p.locs, p.locs_i64, n);
  float kx[8] = {}, vx[8] = {};
  if (loc >= 0 && loc < p.slots) {
    const int64_t page = loc >> p.page_shift;
    const int64_t slot = loc & ((int64_t{1} << p.page_shift) - 1);
    const uint2 kq = *reinterpret_cast<const uint2*>(p.kc + page * p.k_ps + slot * p.k_ss + h * p.k_chs + 8 * lane8);
    const uint2 vq = *reinterpret_cast<const uint2*>(p.vc + page * p.v_ps + slot * p.v_ss + h * p.v_chs + 8 * lane8);
    const uint32_t b = p.scales != nullptr ? p.scales[((page * p.Hkv + h) << p.page_shift) + slot] : 0;
    decode8(kq, p.scales != nullptr, b & 255u, p.k_scale, kx);
    decode8(vq, p.scales != nullptr, b >> 8, p.v_scale, vx);
  }
  const int64_t at = (n * p.Hkv + h) * p.D + 8 * lane8;
  put8<kT>(p.out_k, at, kx);
  put8<kT>(p.out_v, at, vx);
}

bool aligned(const void* ptr, int n) { return (reinterpret_cast<uintptr_t>(ptr) & (n - 1)) == 0; }
bool vec16(const void* ptr, int64_t ts, int64_t hs) { return aligned(ptr, 16) && ((ts | hs) & 7) == 0; }

// Whether rows [tokens, heads, D] of 2-byte elements end before the n at out, or begin after them.
bool apart(const void* rows, int64_t ts, int64_t hs, int64_t tokens, int64_t heads, int64_t D, const void* out, int64_t n) {
  const int64_t a = (tokens - 1) * ts, b = (heads - 1) * hs;
  const int64_t lo = std::min<int64_t>(a, 0) + std::min<int64_t>(b, 0), hi = std::max<int64_t>(a, 0) + std::max<int64_t>(b, 0) + D;
  const intptr_t r = reinterpret_cast<intptr_t>(rows), o = reinterpret_cast<intptr_t>(out);
  return r + 2 * hi <= o || r + 2 * lo >= o + 2 * n;
}

// Launches kern<kT, W> for the row size.
template <typename Launch>
void by_width(int D, Launch launch) {
  if (D <= 64) launch(std::integral_constant<int, 8>{});
  else if (D <= 128) launch(std::integral_constant<int, 16>{});
  else launch(std::integral_constant<int, 32>{});
}

unsigned groups_grid(uint32_t items, int w) {
  return static_cast<unsigned>((static_cast<int64_t>(items) * w + kThreads - 1) / kThreads);
}

}  // namespace

#define REQUIRE(cond, ...) \
  do {                     \
    if (!(cond)) return mac::fail(MAC_ERR_INVALID_ARGUMENT, __VA_ARGS__); \
  } while (0)

#define HIP_OK(call)                                                                      \
  do {                                                                                    \
    hipError_t e_ = (call);                                                               \
    if (e_ != hipSuccess) return mac::fail(MAC_ERR_HIP, "%s: %s", #call, hipGetErrorString(e_)); \
  } while (0)

namespace {

// The cache block shared by the three calls; fills p.
int check_cache(const MacPagedCache* c, CacheParams& p) {
  REQUIRE(c != nullptr, "cache is NULL");
  REQUIRE(c->struct_size == sizeof(MacPagedCache), "struct_size mismatch (%u vs %zu)", c->struct_size, sizeof(MacPagedCache));
  REQUIRE(c->abi_version == MAC_ABI_VERSION, "abi_version mismatch");
  REQUIRE(c->k_cache && c->v_cache, "null pointer argument");
  REQUIRE(c->cache_dtype == MAC_DTYPE_E4M3, "the cache must hold e4m3 codes");
  REQUIRE(c->num_pages > 0 && c->Hkv > 0, "num_pages and Hkv must be positive");
  REQUIRE(c->page_size > 0 && (c->page_size & (c->page_size - 1)) == 0, "page_size must be a power of two (got %d)",
          c->page_size);
  REQUIRE(c->D >= 16 && c->D <= 256 && c->D % 16 == 0, "head_dim must be a multiple of 16 up to 256 (got %d)", c->D);
  REQUIRE(aligned(c->k_cache, 16) && aligned(c->v_cache, 16), "k_cache and v_cache must be 16-byte aligned");
  REQUIRE(((c->k_page_stride | c->k_slot_stride | c->k_head_stride | c->v_page_stride | c->v_slot_stride |
            c->v_head_stride) & 15) == 0,
          "cache strides must be multiples of 16 bytes");
  REQUIRE(aligned(c->kv_scales, 2), "kv_scales must be 2-byte aligned");
  if (c->kv_scales == nullptr)
    REQUIRE(c->k_scale > 0 && std::isfinite(c->k_scale) && c->v_scale > 0 && std::isfinite(c->v_scale),
            "k_scale and v_scale must be positive");
  else
    REQUIRE(c->k_scale == 1.0f && c->v_scale == 1.0f, "a row-scaled cache takes no k_scale / v_scale");
  p.kc = static_cast<uint8_t*>(c->k_cache);
  p.vc = static_cast<uint8_t*>(c->v_cache);
  p.scales = static_cast<uint16_t*>(c->kv_scales);
  p.k_ps = c->k_page_stride;
  p.k_ss = c->k_slot_stride;
  p.k_chs = c->k_head_stride;
  p.v_ps = c->v_page_stride;
  p.v_ss = c->v_slot_stride;
  p.v_chs = c->v_head_stride;
  p.page_shift = __builtin_ctz(c->page_size);
  p.slots = c->num_pages << p.page_shift;
  p.k_scale = c->k_scale;
  p.v_scale = c->v_scale;
  p.Hkv = c->Hkv;
  p.D = c->D;
  return MAC_OK;
}

// (a launch has fewer than 2^32 threads, a row at most 32 of them)
int check_items(int64_t tokens, int64_t heads, CacheParams& p) {
  constexpr int64_t kMost = (int64_t{1} << 27) - 8;
  REQUIRE(tokens >= 0, "tokens must be >= 0");
  REQUIRE(heads < INT_MAX && tokens <= kMost / heads, "too many rows (tokens * heads must be less than 2^27)");
  p.items = static_cast<uint32_t>(tokens * heads);
  return MAC_OK;
}

}  // namespace

extern "C" int mac_paged_cache_write_fp8(const MacPagedCache* c, const void* k, int64_t k_stride0, int64_t k_stride1,
                                         const void* v, int64_t v_stride0, int64_t v_stride1, int32_t dtype,
                                         const void* cache_locs, int32_t cache_locs_is_i64, int64_t tokens,
                                         void* stream) {
  CacheParams p{};
  if (int rc = check_cache(c, p)) return rc;
  REQUIRE(dtype == MAC_DTYPE_BF16 || dtype == MAC_DTYPE_F16, "k and v must be bfloat16 or float16");
  if (int rc = check_items(tokens, c->Hkv, p)) return rc;
  if (tokens == 0) return MAC_OK;
  REQUIRE(k && v && cache_locs, "null pointer argument");
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.k_ts = k_stride0;
  p.k_hs = k_stride1;
  p.v_ts = v_stride0;
  p.v_hs = v_stride1;
  p.kv_vec = vec16(k, k_stride0, k_stride1) && vec16(v, v_stride0, v_stride1);
  p.locs = cache_locs;
  p.locs_i64 = cache_locs_is_i64;
  hipStream_t s = static_cast<hipStream_t>(stream);
  by_width(p.D, [&](auto w) {
    constexpr int W = decltype(w)::value;
    const dim3 grid(groups_grid(p.items, W));
    if (dtype == MAC_DTYPE_BF16) hipLaunchKernelGGL((cache_write_kernel<MAC_DTYPE_BF16, W>), grid, dim3(kThreads), 0, s, p);
    else hipLaunchKernelGGL((cache_write_kernel<MAC_DTYPE_F16, W>), grid, dim3(kThreads), 0, s, p);
  });
  HIP_OK(hipGetLastError());
  return MAC_OK;
}

extern "C" int mac_paged_rope_write_fp8(const MacPagedCache* c, const MacPagedRopeArgs* a, void* stream) {
  REQUIRE(a != nullptr, "args is NULL");
  REQUIRE(a->struct_size == sizeof(MacPagedRopeArgs), "struct_size mismatch (%u vs %zu)", a->struct_size, sizeof(MacPagedRopeArgs));
  REQUIRE(a->abi_version == MAC_ABI_VERSION, "abi_version mismatch");
  CacheParams p{};
  if (int rc = check_cache(c, p)) return rc;
  REQUIRE(a->dtype == MAC_DTYPE_BF16 || a->dtype == MAC_DTYPE_F16, "q, k and v must be bfloat16 or float16");
  REQUIRE(a->Hq > 0, "Hq must be positive");
  if (int rc = check_items(a->tokens, static_cast<int64_t>(a->Hq) + c->Hkv, p)) return rc;
  REQUIRE(a->rotary_dim > 0 && a->rotary_dim <= c->D && a->rotary_dim % 2 == 0, "invalid rotary_dim");
  if (a->tokens == 0) return MAC_OK;
  REQUIRE(a->cos_sin_rows > 0, "cos_sin_cache must not be empty");
  REQUIRE(a->q && a->k && a->v && a->q_out && a->cos_sin_cache && a->positions && a->cache_locs, "null pointer argument");
  REQUIRE(aligned(a->q_out, 16), "q_out must be 16-byte aligned");
  // (a rotated element's partner is read from the row itself)
  const int64_t out_n = a->tokens * a->Hq * c->D;
  REQUIRE(apart(a->q, a->q_stride0, a->q_stride1, a->tokens, a->Hq, c->D, a->q_out, out_n) &&
              apart(a->k, a->k_stride0, a->k_stride1, a->tokens, c->Hkv, c->D, a->q_out, out_n) &&
              apart(a->v, a->v_stride0, a->v_stride1, a->tokens, c->Hkv, c->D, a->q_out, out_n),
          "q_out must not overlap q, k or v");
  p.q = static_cast<const uint16_t*>(a->q);
  p.k = static_cast<const uint16_t*>(a->k);
  p.v = static_cast<const uint16_t*>(a->v);
  p.q_ts = a->q_stride0;
  p.q_hs = a->q_stride1;
  p.k_ts = a->k_stride0;
  p.k_hs = a->k_stride1;
  p.v_ts = a->v_stride0;
  p.v_hs = a->v_stride1;
  p.q_vec = vec16(a->q, a->q_stride0, a->q_stride1);
  p.kv_vec = vec16(a->k, a->k_stride0, a->k_stride1) && vec16(a->v, a->v_stride0, a->v_stride1);
  p.locs = a->cache_locs;
  p.locs_i64 = a->cache_locs_is_i64;
  p.Hq = a->Hq;
  p.q_out = static_cast<uint16_t*>(a->q_out);
  p.cs = a->cos_sin_cache;
  p.cs_stride = a->cos_sin_stride0;
  p.cs_rows = a->cos_sin_rows;
  p.positions = a->positions;
  p.pos_i64 = a->positions_is_i64;
  p.rot = a->rotary_dim;
  p.neox = a->is_neox;
  p.cs_vec = aligned(a->cos_sin_cache, 16) && a->cos_sin_stride0 % 4 == 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  by_width(p.D, [&](auto w) {
    constexpr int W = decltype(w)::value;
    const dim3 grid(groups_grid(p.items, W));
    if (a->dtype == MAC_DTYPE_BF16) hipLaunchKernelGGL((rope_write_kernel<MAC_DTYPE_BF16, W>), grid, dim3(kThreads), 0, s, p);
    else hipLaunchKernelGGL((rope_write_kernel<MAC_DTYPE_F16, W>), grid, dim3(kThreads), 0, s, p);
  });
  HIP_OK(hipGetLastError());
  return MAC_OK;
}

extern "C" int mac_paged_cache_read_fp8(const MacPagedCache* c, const void* kv_indices, int32_t kv_indices_is_i64,
                                        int64_t rows, void* out_k, void* out_v, int32_t dtype, void* stream) {
  CacheParams p{};
  if (int rc = check_cache(c, p)) return rc;
  REQUIRE(dtype >= MAC_DTYPE_F32 && dtype <= MAC_DTYPE_F16, "dtype must be float32, bfloat16 or float16");
  if (int rc = check_items(rows, c->Hkv, p)) return rc;
  if (rows == 0) return MAC_OK;
  REQUIRE(kv_indices && out_k && out_v, "null pointer argument");
  REQUIRE(aligned(out_k, 16) && aligned(out_v, 16), "out_k and out_v must be 16-byte aligned");
  p.locs = kv_indices;
  p.locs_i64 = kv_indices_is_i64;
  p.out_k = out_k;
  p.out_v = out_v;
  hipStream_t s = static_cast<hipStream_t>(stream);
  by_width(p.D, [&](auto w) {
    constexpr int W = decltype(w)::value;
    const dim3 grid(groups_grid(p.items, W));
    if (dtype == MAC_DTYPE_F32) hipLaunchKernelGGL((cache_read_kernel<MAC_DTYPE_F32, W>), grid, dim3(kThreads), 0, s, p);
    else if (dtype == MAC_DTYPE_BF16) hipLaunchKernelGGL((cache_read_kernel<MAC_DTYPE_BF16, W>), grid, dim3(kThreads), 0, s, p);
    else hipLaunchKernelGGL((cache_read_kernel<MAC_DTYPE_F16, W>), grid, dim3(kThreads), 0, s, p);
  });
  HIP_OK(hipGetLastError());
  return MAC_OK;
}
