// mac_paged_api.hip -- entry points of the paged chunk attention: argument
// checks, the choice of the kernel body and of the stream form, the workspace.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>

#include "mac_paged_attention.h"

namespace mac {
int fail(int code, const char* fmt, ...);
}  // namespace mac

namespace {

using namespace mac;

#define REQUIRE(cond, ...) \
  do {                     \
    if (!(cond)) return mac::fail(MAC_ERR_INVALID_ARGUMENT, __VA_ARGS__); \
  } while (0)

bool aligned16(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0; }

constexpr int kMaxB = 4096;  // requests handled by the in-workgroup plan
constexpr int kMaxQ = 1 << 24;  // workgroups: a launch has fewer than 2^32 threads

struct Choice {
  int body = 0, cols = 0, heads_shift = 0, task_rows = 0, unit_shift = 0, stream = kPlain, spare = 0, by_rows = 0, grid = 0;
  size_t plan_bytes = 0, ml_bytes = 0, o_bytes = 0;
  size_t bytes() const { return plan_bytes + ml_bytes + o_bytes; }
};

struct Variant {
  int (*resident)(int, int, int);
  hipError_t (*launch)(const PagedParams&, int, int, hipStream_t);
};

Variant variant(int q_dtype, int cache_dtype) {
  if (q_dtype == MAC_DTYPE_BF16)
    return cache_dtype == MAC_DTYPE_E4M3 ? Variant{paged_resident_bf16_fp8, paged_launch_bf16_fp8}
                                         : Variant{paged_resident_bf16, paged_launch_bf16};
  return cache_dtype == MAC_DTYPE_E4M3 ? Variant{paged_resident_f16_fp8, paged_launch_f16_fp8}
                                       : Variant{paged_resident_f16, paged_launch_f16};
}

size_t up16(size_t n) { return (n + 15) / 16 * 16; }

// Body, task size and form for a call's shapes; false: too large.
bool choose(const MacPagedCache& c, int q_dtype, int Hq, int64_t total_q, int B, int64_t max_keys, Choice& ch) {
  const int G = Hq / c.Hkv;
  const int64_t cols = (total_q + B - 1) / B * G;  // columns of a request of average length
  // 17 to 32 columns: the stream body where a wave's registers hold them (32 requests
  // of 4 rows of 8 heads, stream / tile, us: 8-bit rows of 128 dims over 16K keys 129 /
  // 147, of 64 over 26K 123 / 131, 16-bit of 64 175 / 186; 16-bit of 128 dims 272 / 237)
  const bool stream32 = cols <= 32 && (c.cache_dtype == MAC_DTYPE_E4M3 || c.D == 64);
  ch.body = cols <= 16 ? kBodyStream16 : (stream32 ? kBodyStream32 : (cols <= 64 ? kBodyTile64 : kBodyTile128));
  if (c.D > 128) ch.body = kBodyTile64;  // (the only one whose states and operands of 256 dims fit a wave's registers)
  const int room = kBodyCols[ch.body];
  ch.cols = G <= room ? room / G * G : room;  // whole rows where a row's heads fit
  ch.task_rows = G <= room ? ch.cols / G : 2;
  // The stream body's waves read 256 bytes of a token at a time: two or four heads'
  // rows where they lie side by side.  8 KV heads of 128 dims, 8-bit, one head / two
  // (us): 64 requests over 26K keys 645 / 600, 16 over 32K 227 / 211, 4 over 128K 219 /
  // 199, 64 over 1K 46 / 48; of 64 dims, one / four: 573 / 466, 194 / 148, 164 / 156, 48 /
  // 41.  Not where few tasks share the keys among many workgroups (fewer, larger
  // partial states then): 1 request over 128K keys 75 / 80, over 4K 27 / 32.
  const int64_t row = static_cast<int64_t>(c.D) * (c.cache_dtype == MAC_DTYPE_E4M3 ? 1 : 2);
  const int64_t head_tasks = std::min<int64_t>(total_q, total_q * G / ch.cols + B) * c.Hkv;
  if (ch.body <= kBodyStream32 && c.k_head_stride == row && head_tasks >= 32)
    while (row << ch.heads_shift < 256 && c.Hkv % (2 << ch.heads_shift) == 0) ++ch.heads_shift;
  // bounds on the tasks: of this batch's rows, and of any row offsets (a
  // request's rows lie within total_q)
  const int64_t tasks = (std::min<int64_t>(total_q, total_q * G / ch.cols + B)) * (c.Hkv >> ch.heads_shift);
  const int64_t worst = static_cast<int64_t>(B) * ((total_q * G + ch.cols - 1) / ch.cols) * c.Hkv;
  if (worst >= INT_MAX) return false;
  const int resident = variant(q_dtype, c.cache_dtype).resident(c.D, ch.body, B);
  // The stream body streams its keys.  The tile body does where whole tasks would leave
  // much of the GPU idle or take very different times, which the lengths decide, on the
  // device (paged_plan); else workgroups that take whole tasks, in step over the same
  // keys, share them in L2 and write no partial states (streamed / whole, 4 heads per
  // group, us: 2048 rows over 2K keys, 512 tasks of 512 resident, 116 / 84, over 8K 364 /
  // 320, 4 x 2048 of 64 dims, 1024 of 768, 482 / 408).  One request's tasks are about as
  // long as each other: enough of them are taken whole, and so are tasks of tables too
  // short for the device to stream any (256 rows over their own keys 35 -> 29 without
  // the combining launch).
  const bool fits = 2 * worst < INT_MAX;  // (the units of a task and its partial states)
  ch.spare = tasks < resident;
  if (ch.body <= kBodyStream32) {
    if (!fits) return false;
    ch.stream = kStream;
  } else {
    ch.stream = (B > 1 || ch.spare) && fits && max_keys > kShortKeys ? kEither : kPlain;
  }
  ch.grid = resident;
  if (ch.stream == kPlain) {
    ch.grid = static_cast<int>(std::min<int64_t>(tasks, resident));
    return true;
  }
  // Partial states of up to four pieces a task: a wave per row and head joins them, else
  // a workgroup.  Wave / workgroup (us): 24 ragged requests of 64 dims (1.3 pieces) 106 /
  // 151, 512 rows of 4 heads over 32K keys (4) 373 / 389, 256 (8) 226 / 220, 128 (16) 171
  // / 129, 64 (64) 192 / 86; a token of 256 dims over 8K (256) 144 / 33.
  ch.by_rows = ch.body >= kBodyTile64 && ch.grid <= 4 * tasks;
  if (!ch.by_rows && total_q * Hq >= kMaxQ) return false;
  ch.unit_shift = 7 - ch.heads_shift;  // one block of each wave
  while (ch.unit_shift < 30 && (((max_keys + (int64_t{1} << ch.unit_shift) - 1) >> ch.unit_shift) + 1) * worst >= INT_MAX) ++ch.unit_shift;
  ch.plan_bytes = up16(sizeof(int) * (static_cast<size_t>(B) + 2));
  const size_t slots = 2 * static_cast<size_t>(ch.grid) * (room << ch.heads_shift);
  ch.ml_bytes = slots * 2 * sizeof(float);
  ch.o_bytes = slots * c.D * sizeof(float);
  return true;
}

int check(const MacPagedCache* c, const MacPagedAttentionArgs* a) {
  REQUIRE(c != nullptr && a != nullptr, "cache / args is NULL");
  REQUIRE(c->struct_size == sizeof(MacPagedCache), "struct_size mismatch (%u vs %zu)", c->struct_size, sizeof(MacPagedCache));
  REQUIRE(a->struct_size == sizeof(MacPagedAttentionArgs), "struct_size mismatch (%u vs %zu)", a->struct_size,
          sizeof(MacPagedAttentionArgs));
  REQUIRE(c->abi_version == MAC_ABI_VERSION && a->abi_version == MAC_ABI_VERSION, "abi_version mismatch");
  REQUIRE(a->q_dtype == MAC_DTYPE_BF16 || a->q_dtype == MAC_DTYPE_F16, "q must be bfloat16 or float16");
  REQUIRE(c->cache_dtype == MAC_DTYPE_E4M3 || c->cache_dtype == a->q_dtype, "the cache must hold e4m3 codes or q's type");
  REQUIRE(c->D == 64 || c->D == 128 || c->D == 256, "head_dim must be 64, 128 or 256 (got %d)", c->D);
  REQUIRE(a->Hq > 0 && c->Hkv > 0 && a->Hq % c->Hkv == 0, "Hq must be a positive multiple of Hkv");
  REQUIRE(a->B >= 0 && a->B <= kMaxB, "B must be in [0, %d] (got %d)", kMaxB, a->B);
  REQUIRE(a->total_q >= 0 && a->total_q < kMaxQ && a->total_q <= INT_MAX / a->Hq, "total_q too large");
  REQUIRE(c->num_pages > 0 && c->num_pages <= INT_MAX, "num_pages must be positive (and fit 31 bits)");
  REQUIRE(c->page_size > 0 && (c->page_size & (c->page_size - 1)) == 0, "page_size must be a power of two (got %d)",
          c->page_size);
  REQUIRE(a->table_rows >= 0 && a->table_cols >= 0 &&
              static_cast<int64_t>(a->table_cols) * c->page_size < (int64_t{1} << 30),
          "page_table must name fewer than 2^30 keys per request");
  REQUIRE(static_cast<int64_t>(c->Hkv) * c->page_size <= INT_MAX, "pages too large");
  REQUIRE(a->sm_scale > 0 && std::isfinite(a->sm_scale), "sm_scale must be positive");
  REQUIRE(a->logit_cap >= 0 && std::isfinite(a->logit_cap), "logit_cap must be >= 0");
  REQUIRE(c->k_scale > 0 && std::isfinite(c->k_scale) && c->v_scale > 0 && std::isfinite(c->v_scale),
          "k_scale and v_scale must be positive");
  if (c->kv_scales != nullptr) {
    REQUIRE(c->cache_dtype == MAC_DTYPE_E4M3, "kv_scales belong to an e4m3 cache");
    REQUIRE(c->k_scale == 1.0f && c->v_scale == 1.0f, "a row-scaled cache takes no k_scale / v_scale");
    REQUIRE((reinterpret_cast<uintptr_t>(c->kv_scales) & 1) == 0, "kv_scales must be 2-byte aligned");
  }
  return MAC_OK;
}

}  // namespace

extern "C" int64_t mac_paged_chunk_attention_workspace(const MacPagedCache* c, const MacPagedAttentionArgs* a) {
  if (check(c, a) != MAC_OK) return -1;
  if (a->B == 0 || a->total_q == 0) return 0;
  Choice ch;
  if (!choose(*c, a->q_dtype, a->Hq, a->total_q, a->B, static_cast<int64_t>(a->table_cols) * c->page_size, ch)) return 0;
  return static_cast<int64_t>(ch.bytes());
}

extern "C" int mac_paged_chunk_attention(const MacPagedCache* c, const MacPagedAttentionArgs* a, void* workspace,
                                         int64_t workspace_bytes, void* stream) {
  if (int rc = check(c, a)) return rc;
  if (a->B == 0 || a->total_q == 0) return MAC_OK;
  REQUIRE(a->q && c->k_cache && c->v_cache && a->qo_indptr && a->kv_lens && a->out && a->out_lse, "null pointer argument");
  REQUIRE(a->page_table || a->table_cols == 0 || a->table_rows == 0, "null pointer argument");
  REQUIRE(aligned16(a->q) && ((a->q_stride0 | a->q_stride1) & 7) == 0, "q rows must be 16-byte aligned");
  REQUIRE(aligned16(c->k_cache) && aligned16(c->v_cache), "k_cache and v_cache must be 16-byte aligned");
  REQUIRE(((c->k_page_stride | c->k_slot_stride | c->k_head_stride) & 15) == 0,
          "cache strides must be multiples of 16 bytes");
  REQUIRE(c->k_page_stride == c->v_page_stride && c->k_slot_stride == c->v_slot_stride && c->k_head_stride == c->v_head_stride,
          "k_cache and v_cache must have the same strides");
  for (const int64_t s : {c->k_page_stride, c->k_slot_stride, c->k_head_stride})
    REQUIRE(s >= 0 && s <= UINT_MAX, "cache strides must be less than 2^32 bytes");
  REQUIRE(aligned16(a->out), "out must be 16-byte aligned");
  Choice ch;
  REQUIRE(choose(*c, a->q_dtype, a->Hq, a->total_q, a->B, static_cast<int64_t>(a->table_cols) * c->page_size, ch),
          "batch too large");
  REQUIRE(aligned16(workspace) && workspace_bytes >= static_cast<int64_t>(ch.bytes()) && (workspace || ch.bytes() == 0),
          "workspace too small or misaligned (needs %zu bytes)", ch.bytes());
  const int G = a->Hq / c->Hkv;
  const double log2e = 1.4426950408889634;
  PagedParams p{};
  p.q = static_cast<const uint16_t*>(a->q);
  p.k = static_cast<const char*>(c->k_cache);
  p.v = static_cast<const char*>(c->v_cache);
  p.scales = static_cast<const uint16_t*>(c->kv_scales);
  p.qo_indptr = a->qo_indptr;
  p.kv_lens = a->kv_lens;
  p.table = a->page_table;
  p.req_ids = a->req_ids;
  p.out = static_cast<uint16_t*>(a->out);
  p.lse = a->out_lse;
  if (ch.stream != kPlain) {
    char* w = static_cast<char*>(workspace);
    p.plan = reinterpret_cast<int32_t*>(w);
    p.part_ml = reinterpret_cast<float*>(w + ch.plan_bytes);
    p.part_o = reinterpret_cast<float*>(w + ch.plan_bytes + ch.ml_bytes);
  }
  p.q_ts = a->q_stride0;
  p.q_hs = a->q_stride1;
  p.kv_ps = static_cast<uint32_t>(c->k_page_stride);
  p.kv_ss = static_cast<uint32_t>(c->k_slot_stride);
  p.kv_hs = static_cast<uint32_t>(c->k_head_stride);
  p.table_stride = a->table_stride;
  p.total_q = a->total_q;
  p.num_pages = static_cast<uint32_t>(c->num_pages);
  p.B = a->B;
  p.Hq = a->Hq;
  p.Hkv = c->Hkv;
  p.G = G;
  p.table_rows = a->table_rows;
  p.table_cols = a->table_cols;
  p.page_shift = __builtin_ctz(c->page_size);
  // (a window of 2^30 keys or more covers any request's)
  p.window_left = a->window_left < 0 || a->window_left >= (1 << 30) ? -1 : a->window_left;
  p.cols = ch.cols;
  p.heads_shift = ch.heads_shift;
  p.task_rows = ch.task_rows;
  p.unit_shift = ch.unit_shift;
  p.stream = ch.stream;
  p.spare = ch.spare;
  p.by_rows = ch.by_rows;
  p.grid = ch.grid;
  const double raw = a->sm_scale * c->k_scale;
  p.q_scale = static_cast<float>(a->logit_cap > 0 ? 1.0 : raw * log2e);
  p.cap_in = a->logit_cap > 0 ? static_cast<float>(2.0 * log2e * raw / a->logit_cap) : 0.0f;
  p.cap_out = static_cast<float>(a->logit_cap * log2e);
  // (scores are scaled in fp32: a factor that is 0 or infinite there would turn
  // masked scores into NaN)
  REQUIRE(p.q_scale >= FLT_MIN && std::isfinite(p.q_scale), "sm_scale * k_scale does not fit fp32");
  REQUIRE(a->logit_cap == 0 || (p.cap_in >= FLT_MIN && std::isfinite(p.cap_in) && p.cap_out >= FLT_MIN && std::isfinite(p.cap_out)),
          "logit_cap does not fit fp32 with sm_scale");
  p.v_scale = c->v_scale;
  const hipError_t e = variant(a->q_dtype, c->cache_dtype).launch(p, c->D, ch.body, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return mac::fail(MAC_ERR_HIP, "paged chunk attention: %s", hipGetErrorString(e));
  return MAC_OK;
}
