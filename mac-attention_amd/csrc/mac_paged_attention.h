// mac_paged_attention.h -- parameters, planning and element types shared by
// the paged chunk attention's entry point and kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mac_attention_amd.h"
#include "mac_common.h"

namespace mac {

// Plain form: workgroups take whole tasks in turn.  kEither: the device decides, from
// the lengths that the host does not know (paged_plan).
enum { kPlain = 0, kStream = 1, kEither = 2 };
constexpr int kShortKeys = 1024;  // keys that streaming has to save a workgroup

// What the kernels read.  A call's queries are cut into tasks of `cols`
// (row, head) columns of one request and KV head; stream form: the tasks' keys
// laid end to end in units of 2^unit_shift keys, dealt to the workgroups in
// equal runs.
struct PagedParams {
  const uint16_t* q;
  const char* k;
  const char* v;
  const uint16_t* scales;  // [pages, Hkv, P] (K byte low, V byte high), or NULL
  const int32_t* qo_indptr;
  const int32_t* kv_lens;
  const int32_t* table;
  const int32_t* req_ids;  // row of the table for each request, or NULL: the request's number
  uint16_t* out;
  float* lse;
  float* part_o;   // stream form: [2 grid][heads][body's columns][D] unnormalised partial outputs
  float* part_ml;  // [2 grid][heads][columns][2] their reference points (log2 units) and sums
  int32_t* plan;   // [B + 1] units before each request, for the combining launch; whether there are any
  int64_t q_ts, q_hs;                          // elements
  uint32_t kv_ps, kv_ss, kv_hs;  // bytes: page, slot and head strides of K and of V
  int64_t table_stride;
  int64_t total_q;
  uint32_t num_pages;
  int B, Hq, Hkv, G;
  int table_rows, table_cols, page_shift;
  int window_left;  // < 0: none
  int cols;         // columns of a task per KV head (whole rows where a row's heads fit one)
  int heads_shift;  // a task takes 2^heads_shift KV heads (stream body)
  int task_rows;    // most rows that a task's columns touch
  int unit_shift;   // stream form
  int stream;       // kPlain, kStream or kEither
  int spare;        // kEither: 1: the tasks leave part of the GPU idle
  int by_rows;      // stream form: 1: partial states combined a row, 0: a row and head per workgroup
  int grid;         // workgroups (stream form: slots hold 2 partials of each)
  float q_scale;    // sm_scale k_scale log2(e); with a cap: 1 (scores are capped to log2 units)
  float cap_in, cap_out;  // 2 log2(e) sm_scale k_scale / cap, cap log2(e); 0: no cap
  float v_scale;
};

// The kernels read their parameters where the launch put them.  A fresh pointer
// is opaque to the compiler: what is read through it is loaded where it is used,
// not kept in scalar registers over the key loop (which spilled some 80 of them).
typedef const __attribute__((address_space(4))) PagedParams PagedArgs;
__device__ __forceinline__ PagedArgs& fresh_args() {
  PagedArgs* a = (PagedArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(a));
  return *a;
}

// A request's rows, keys and tasks; all 0 for one whose rows do not lie in the
// buffers.
struct PagedRequest {
  int q0, n;    // first row, rows
  int len;      // kv length (row r sits at position len - n + r)
  int keys;     // cached keys that the table can name
  int tasks;    // column tasks per KV head (or group of 2^heads_shift)
  int units;    // stream form: units per task
};

__device__ __forceinline__ PagedRequest paged_request(PagedArgs& p, int b) {
  PagedRequest r;
  r.q0 = p.qo_indptr[b];
  const int q1 = p.qo_indptr[b + 1];
  r.len = max(p.kv_lens[b], 0);
  const int row = p.req_ids != nullptr ? p.req_ids[b] : b;
  r.n = r.q0 >= 0 && q1 > r.q0 && q1 <= p.total_q ? q1 - r.q0 : 0;
  // (the table holds fewer than 2^30 keys a request, checked on the host)
  r.keys = row >= 0 && row < p.table_rows ? min(r.len, p.table_cols << p.page_shift) : 0;
  r.tasks = static_cast<int>((static_cast<int64_t>(r.n) * p.G + p.cols - 1) / p.cols);
  const int span = p.window_left < 0 ? r.keys : min(r.keys, p.window_left + p.task_rows);
  r.units = max((span + (1 << p.unit_shift) - 1) >> p.unit_shift, 1);
  return r;
}

// Exclusive prefix of the requests' units (stream form) or tasks (plain form) in
// s_pre[B + 1], by a workgroup of 256 threads; ends with a barrier.  s_tmp: 4
// entries.  Returns the units of the thread's longest task.
__device__ __forceinline__ int paged_prefix(PagedArgs& p, bool stream, int* s_pre, int* s_tmp) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per = ceil_div(p.B, 256);
  const int b0 = min(p.B, tid * per), b1 = min(p.B, b0 + per);
  int sum = 0, longest = 0;
  for (int b = b0; b < b1; ++b) {
    const PagedRequest r = paged_request(p, b);
    const int w = r.tasks * (p.Hkv >> p.heads_shift) * (stream ? r.units : 1);
    if (w != 0) longest = max(longest, r.units);
    s_pre[b] = w;
    sum += w;
  }
  int x = sum;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(x, off);
    if (lane >= off) x += y;
  }
  if (lane == 63) s_tmp[wave] = x;
  __syncthreads();
  int acc = x - sum, total = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < wave) acc += s_tmp[w];
    total += s_tmp[w];
  }
  for (int b = b0; b < b1; ++b) {
    const int w = s_pre[b];
    s_pre[b] = acc;
    acc += w;
  }
  if (tid == 0) s_pre[p.B] = total;
  __syncthreads();
  return longest;
}

// The prefix, and the form: where a choice is left, the stream form if a task is
// longer than a workgroup's share of the units and kShortKeys more, which pay for the
// partial states; where whole tasks would leave part of the GPU idle, than one and a
// half times the share, for a workgroup alone on its CU is the faster one.  Every
// workgroup decides alike.  Whole / streamed, 8 KV heads of 4 query heads (us): a chunk
// of 2048 rows over its own keys and one token over 128K 3365 / 299, and 63 tokens over
// 16K (a task is as long as the share) 593 / 716; 5 requests of 512 rows over 4K to 32K
// 990 / 750, 12 such 1717 / 1839; part of the GPU: 2 of 334 rows over 500 keys 38 / 62,
// 2000 79 / 82, 8000 238 / 163; 256 rows over 1000 keys 49 / 61, 2000 77 / 65, 8000 231
// / 93; 8 of 40 rows over 500 36 / 47, 2000 77 / 61.
template <bool kEitherForm>
__device__ __forceinline__ bool paged_plan(PagedArgs& p, int* s_pre, int* s_tmp) {
  if constexpr (!kEitherForm) {
    paged_prefix(p, true, s_pre, s_tmp);
    return true;
  }
  const int longest = paged_prefix(p, p.stream != kPlain, s_pre, s_tmp);
  if (p.stream != kEither) return p.stream == kStream;
  const int total = s_pre[p.B];
  const int more = longest - max(kShortKeys >> p.unit_shift, 1);
  if (__syncthreads_or(2 * static_cast<int64_t>(more) * p.grid > (2 + p.spare) * static_cast<int64_t>(total))) return true;
  paged_prefix(p, false, s_pre, s_tmp);
  return false;
}

// Largest b < B with pre[b] <= x.
__device__ __forceinline__ int paged_find(const int* s_pre, int B, int x) {
  int lo = 0, hi = B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (s_pre[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Stream form: the units dealt to the workgroups in equal runs, the first `more` of
// them with one unit more.
struct Deal {
  uint32_t groups, each, more;
  __device__ __forceinline__ int begin(uint32_t w) const { return static_cast<int>(w * each + min(w, more)); }
  // the workgroup whose run holds unit x
  __device__ __forceinline__ int owner(uint32_t x) const {
    const uint32_t longer = more * (each + 1);
    return static_cast<int>(x < longer ? x / (each + 1) : more + (x - longer) / each);
  }
};
__device__ __forceinline__ Deal stream_deal(PagedArgs& p, int total) {
  Deal d;
  d.groups = min(p.grid, max(total, 1));
  d.each = static_cast<uint32_t>(total) / d.groups;
  d.more = total - d.each * d.groups;
  return d;
}

// One of a task's runs of keys.
struct PagedTask {
  int b, hkv, gc0;      // request, (first) KV head, first column of the request's rows x G
  int q0, n, len;       // of the request
  int nc;               // columns
  int row0, row1;       // first and last row
  int klo, khi;         // keys to attend over in this run
  const int32_t* table;
};

__device__ __forceinline__ PagedTask paged_task(PagedArgs& p, int b, const PagedRequest& r, int index) {
  PagedTask t;
  t.b = b;
  const int group = index / r.tasks;
  const int ct = index - group * r.tasks;
  t.hkv = group << p.heads_shift;
  t.q0 = r.q0;
  t.n = r.n;
  t.len = r.len;
  // (columns of a request fit 31 bits, checked on the host)
  t.gc0 = ct * p.cols;
  t.nc = min(p.cols, r.n * p.G - t.gc0);
  t.row0 = t.gc0 / p.G;
  t.row1 = (t.gc0 + t.nc - 1) / p.G;
  const int first = r.len - r.n + t.row0, last = r.len - r.n + t.row1;
  t.klo = p.window_left < 0 ? 0 : max(first - p.window_left, 0);
  t.khi = min(max(last + 1, 0), r.keys);
  const int row = p.req_ids != nullptr ? p.req_ids[b] : b;
  t.table = p.table + static_cast<int64_t>(row < 0 || row >= p.table_rows ? 0 : row) * p.table_stride;
  return t;
}

// Registers of raw bits: native vectors (HIP's uint4 is a struct, whose arrays
// the compiler left in scratch memory).
typedef uint32_t pa_u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t pa_u32x4 __attribute__((ext_vector_type(4)));

// 16-bit element types.
typedef __bf16 pa_bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 pa_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 pa_f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 pa_f16x8 __attribute__((ext_vector_type(8)));
typedef float pa_f32x4 __attribute__((ext_vector_type(4)));

template <int kT>
struct PagedElem;

template <>
struct PagedElem<MAC_DTYPE_BF16> {
  static __device__ __forceinline__ pa_f32x4 mfma(const pa_u32x4& a, const pa_u32x4& b, pa_f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pa_bf16x8, a), __builtin_bit_cast(pa_bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack2(float a, float b) {
    const pa_bf16x2 v = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
    return __builtin_bit_cast(uint32_t, v);
  }
  // two codes (the low or the high half of w) times the power of two s: exact
  template <bool kHigh>
  static __device__ __forceinline__ uint32_t decode2(uint32_t w, float s) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, kHigh));
  }
  static __device__ __forceinline__ float low(uint32_t w) { return bf16_lo(w); }
  static __device__ __forceinline__ float high(uint32_t w) { return bf16_hi(w); }
  static __device__ __forceinline__ bool not_finite(uint32_t w) {
    return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
  }
};

template <>
struct PagedElem<MAC_DTYPE_F16> {
  static __device__ __forceinline__ pa_f32x4 mfma(const pa_u32x4& a, const pa_u32x4& b, pa_f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pa_f16x8, a), __builtin_bit_cast(pa_f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack2(float a, float b) {
    const pa_f16x2 v = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
    return __builtin_bit_cast(uint32_t, v);
  }
  template <bool kHigh>
  static __device__ __forceinline__ uint32_t decode2(uint32_t w, float s) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, kHigh));
  }
  static __device__ __forceinline__ float low(uint32_t w) { return static_cast<float>(__builtin_bit_cast(pa_f16x2, w)[0]); }
  static __device__ __forceinline__ float high(uint32_t w) { return static_cast<float>(__builtin_bit_cast(pa_f16x2, w)[1]); }
  static __device__ __forceinline__ bool not_finite(uint32_t w) {
    return (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u;
  }
};

// Sixteen codes as two vectors of eight 16-bit values.
template <int kT>
__device__ __forceinline__ void decode16(const pa_u32x4& w, float s, pa_u32x4& a, pa_u32x4& b) {
  typedef PagedElem<kT> E;
  a = pa_u32x4{E::template decode2<false>(w.x, s), E::template decode2<true>(w.x, s),
                 E::template decode2<false>(w.y, s), E::template decode2<true>(w.y, s)};
  b = pa_u32x4{E::template decode2<false>(w.z, s), E::template decode2<true>(w.z, s),
                 E::template decode2<false>(w.w, s), E::template decode2<true>(w.w, s)};
}
template <int kT>
__device__ __forceinline__ bool not_finite(const pa_u32x4& w) {
  typedef PagedElem<kT> E;
  return E::not_finite(w.x) || E::not_finite(w.y) || E::not_finite(w.z) || E::not_finite(w.w);
}

// Host: launch of one variant (mac_paged_attention.hip is compiled once for
// each of them).
enum { kBodyStream16 = 0, kBodyStream32 = 1, kBodyTile64 = 2, kBodyTile128 = 3, kBodies = 4 };
constexpr int kBodyCols[kBodies] = {16, 32, 64, 128};

// Resident workgroups of a body on the current device, and its launch (with
// the combining one in the stream form).
#define MAC_PAGED_VARIANT_DECL(name)                 \
  int paged_resident_##name(int D, int body, int B); \
  hipError_t paged_launch_##name(const PagedParams& p, int D, int body, hipStream_t stream);
MAC_PAGED_VARIANT_DECL(bf16)
MAC_PAGED_VARIANT_DECL(f16)
MAC_PAGED_VARIANT_DECL(bf16_fp8)
MAC_PAGED_VARIANT_DECL(f16_fp8)

}  // namespace mac
