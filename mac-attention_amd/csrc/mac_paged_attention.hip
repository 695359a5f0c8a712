// mac_paged_attention.hip -- attention of a chunk of new tokens over a paged
// K/V cache for MI355X (gfx950).  Compiled once per variant (queries bf16 or
// fp16; cache of the same type or e4m3): MAC_PAGED_T, MAC_PAGED_F8 and
// MAC_PAGED_NAME come from the build.
//
// Row r of a request with n new rows and a cache of len keys sits at position
// len - n + r and attends to the keys [max(pos - window, 0), pos]:
//   s_k = q . k_k sm_scale     (or cap tanh(q . k_k sm_scale / cap))
//   out = sum_k e^(s_k - m) v_k / l,  lse = m + log l,  l = sum_k e^(s_k - m)
// in one pass over the keys with a running reference point m and sum l in fp32.
//
// Columns.  A GQA group's heads share their keys, so the (row, head) pairs of a
// request and KV head are the columns of S^T = K Q^T and O^T += V^T P^T on
// v_mfma_f32_16x16x32: 16 consecutive columns a tile, whatever the group size
// (one token of 4 heads, five drafted tokens of 8, a chunk's rows).  The lane
// (quad, col) = (lane / 16, lane % 16) holds column col: its scores of keys 16 t
// + 4 quad + (0..3), and of the output dims 16 dt + 4 quad + (0..3).
//
// 8-bit rows become 16-bit values when they are staged: every e4m3 value times
// a power of two is exact in bf16, and gfx950 converts two codes and applies
// the row's scale in one instruction, so the products run as for 16-bit rows.
// A static k_scale is part of the softmax scale, v_scale of the final
// normalisation.  P is rounded to the queries' type for its product (2^-8 or
// 2^-11 of each weight, as much as the output's own rounding); sums are fp32.
//
// Masked keys: keys past a row's range, past the cache or without a page get
// s = -inf, and V of keys that no row may see is zeroed when staged.  A key that
// some rows see and others do not would reach them all through 0 x NaN if its V
// is not finite: such a key is masked for every row and added at the end of the
// run, for the rows that see it (add_key).

#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "mac_paged_attention.h"

namespace {

using namespace mac;

constexpr int kT = MAC_PAGED_T;
constexpr bool kF8 = MAC_PAGED_F8;
typedef PagedElem<kT> E;
typedef pa_f32x4 f32x4;

// An index times a byte stride: both fit 32 bits, their product need not.
__device__ __forceinline__ uint64_t at64(uint32_t i, uint32_t stride) { return static_cast<uint64_t>(i) * stride; }

// Four dims of V, one row each of four: the transposing LDS read (lds_read_tr16)
// of 16-bit elements of either type.
__device__ __forceinline__ pa_u32x2 read_tr(const uint16_t* at) { return __builtin_bit_cast(pa_u32x2, lds_read_tr16(at)); }
__device__ __forceinline__ pa_u32x4 join(const pa_u32x2& a, const pa_u32x2& b) { return pa_u32x4{a.x, a.y, b.x, b.y}; }

// Softmax state of one column tile: raw-score reference point m (-inf: no key
// seen), the scaled score past which it moves, the lane's part of the sum.
struct Column {
  float m, past, l;
};
__device__ __forceinline__ Column fresh_column() { return Column{-INFINITY, -INFINITY, 0.0f}; }
// A reference point so large that m scale, rounded on its own, would be off by
// whole powers of two (2^20 leaves 2^-4 of one): then (s - m) scale is formed
// instead of one fma.
constexpr float kFar = 1048576.0f;

// Scores of 16 kKt keys (s[c][t][r]: key 16 t + 4 quad + r) to weights in f, moving
// the reference points where a score exceeds one by 2^8 (lazily: p <= 2^8 is as
// exact, and most blocks rescale nothing).  Called by whole waves; far: some
// reference point of the wave is.  One branch each for all of the wave's columns:
// the exponentials share a basic block with the products around them.
template <int kPer, int kKt, int kDT>
__device__ __forceinline__ void weigh(const f32x4 (&s)[kPer][kKt], float scale, Column (&st)[kPer], bool& far,
                                      f32x4 (&acc)[kPer][kDT], float (&f)[kPer][4 * kKt]) {
  float top[kPer];
  bool past = false;
#pragma unroll
  for (int c = 0; c < kPer; ++c) {
    top[c] = s[c][0][0];
#pragma unroll
    for (int e = 1; e < 4 * kKt; e += 2) {
      const float a = s[c][e >> 2][e & 3], b = e + 1 < 4 * kKt ? s[c][(e + 1) >> 2][(e + 1) & 3] : a;
      top[c] = max3_nonan(top[c], a, b);
    }
    past = past || top[c] * scale > st[c].past;
  }
  if (__any(past)) {
    bool big = false;
#pragma unroll
    for (int c = 0; c < kPer; ++c) {
      const float bm = quad_max(top[c]);
      const float m_new = max3_nonan(st[c].m, bm, bm);
      const float alpha = st[c].m == m_new ? 1.0f : fast_exp2((st[c].m - m_new) * scale);
      st[c].m = m_new;
      st[c].past = m_new * scale + 8.0f;
      big = big || (fabsf(m_new) * scale > kFar && m_new != -INFINITY);
      st[c].l *= alpha;
#pragma unroll
      for (int dt = 0; dt < kDT; ++dt) acc[c][dt] *= alpha;
    }
    far = __any(big);
  }
  if (far) {
#pragma unroll
    for (int c = 0; c < kPer; ++c)
#pragma unroll
      for (int e = 0; e < 4 * kKt; ++e) f[c][e] = (st[c].m == -INFINITY ? s[c][e >> 2][e & 3] : s[c][e >> 2][e & 3] - st[c].m) * scale;
  } else {
#pragma unroll
    for (int c = 0; c < kPer; ++c) {
      const float mo = st[c].m == -INFINITY ? 0.0f : -st[c].m * scale;
#pragma unroll
      for (int e = 0; e < 4 * kKt; ++e) f[c][e] = fmaf(s[c][e >> 2][e & 3], scale, mo);
    }
  }
#pragma unroll
  for (int c = 0; c < kPer; ++c) {
    float sum[2] = {0.0f, 0.0f};  // (two chains)
#pragma unroll
    for (int e = 0; e < 4 * kKt; ++e) {
      f[c][e] = fast_exp2(f[c][e]);
      sum[e & 1] = e < 2 ? f[c][e] : sum[e & 1] + f[c][e];
    }
    st[c].l += sum[0] + sum[1];
  }
}

__device__ __forceinline__ pa_u32x4 pack8(const float* f) {
  return pa_u32x4{E::pack2(f[0], f[1]), E::pack2(f[2], f[3]), E::pack2(f[4], f[5]), E::pack2(f[6], f[7])};
}

// Logit cap: raw scores to capped ones in log2 units, cap log2(e) tanh(x) with
// tanh(x) = 1 - 2 / (1 + e^2x) (off by 2^-23 of the cap: the scores are fp32).
__device__ __forceinline__ float capped(float x, float cap_in, float cap_out) {
  return cap_out * (1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + fast_exp2(x * cap_in)));
}
template <int kKt>
__device__ __forceinline__ void cap_scores(f32x4 (&c)[kKt], float cap_in, float cap_out) {
#pragma unroll
  for (int t = 0; t < kKt; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) c[t][r] = capped(c[t][r], cap_in, cap_out);
}

// The keys of 32 from `base` that a row with the range [lo, hi) sees, less
// `bad`, as bits of the lane's own keys: bit 16 t + r.
__device__ __forceinline__ uint32_t seen_keys(int base, int lo, int hi, uint32_t bad, int quad) {
  const int a = min(max(lo - base, 0), 32), z = min(max(hi - base, 0), 32);
  const uint64_t range = ((1ull << z) - 1) & ~((1ull << a) - 1);
  return (static_cast<uint32_t>(range) & ~bad) >> (4 * quad);
}
// Masks the scores c[0], c[1] of 32 keys.
__device__ __forceinline__ void mask_scores(f32x4* c, uint32_t seen) {
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) c[t][r] = (seen >> (16 * t + r)) & 1 ? c[t][r] : -INFINITY;
}

// Column c of a task: its row in the request and head in the group (a column past
// the task computes its last one and stores nothing).
__device__ __forceinline__ void lane_column(PagedArgs& p, const PagedTask& t, int c, int& row, int& head) {
  const int gc = t.gc0 + min(c, t.nc - 1);
  row = gc / p.G;
  head = gc - row * p.G;
}
// First key that the row at a position sees.
__device__ __forceinline__ int first_key(int pos, int window) { return window < 0 ? 0 : max(pos - window, 0); }

// Eight consecutive elements of a cached row from dim d, in fp32.
__device__ __forceinline__ void row8(const char* row, int d, float scale, float (&x)[8]) {
  pa_u32x4 w;
  if constexpr (kF8) {
    const pa_u32x2 c = *reinterpret_cast<const pa_u32x2*>(row + d);
    w = pa_u32x4{E::decode2<false>(c.x, scale), E::decode2<true>(c.x, scale), E::decode2<false>(c.y, scale), E::decode2<true>(c.y, scale)};
  } else {
    w = *reinterpret_cast<const pa_u32x4*>(row + 2 * d);
  }
  x[0] = E::low(w.x); x[1] = E::high(w.x); x[2] = E::low(w.y); x[3] = E::high(w.y);
  x[4] = E::low(w.z); x[5] = E::high(w.z); x[6] = E::low(w.w); x[7] = E::high(w.w);
}

// Adds one key of KV head hkv to the states of the rows that see it, in fp32 on the
// vector units.  kSplitQ: q's chunks in the order of the 8-bit stream body.
template <int D, int kPer, bool kSplitQ>
__device__ __forceinline__ void add_key(PagedArgs& p, const PagedTask& t, int hkv, int key, const pa_u32x4 (&q)[kPer][D / 32],
                                        const int (&pos)[kPer], Column (&st)[kPer], f32x4 (&acc)[kPer][D / 16], int quad) {
  const int page = t.table[key >> p.page_shift];
  const int slot = key & ((1 << p.page_shift) - 1);
  const uint64_t row = at64(page, p.kv_ps) + at64(slot, p.kv_ss) + at64(hkv, p.kv_hs);
  const char* kr = p.k + row;
  const char* vr = p.v + row;
  const uint32_t sc = kF8 && p.scales != nullptr ? p.scales[((static_cast<int64_t>(page) * p.Hkv + hkv) << p.page_shift) + slot] : 0x7f7fu;
  const float ks = __uint_as_float((sc & 255u) << 23), vs = __uint_as_float((sc >> 8) << 23);
  float s[kPer] = {};
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    float k[8];
    row8(kr, kSplitQ ? 64 * (i >> 1) + 16 * quad + 8 * (i & 1) : 32 * i + 8 * quad, ks, k);
#pragma unroll
    for (int c = 0; c < kPer; ++c) {
      const uint32_t w[4] = {q[c][i].x, q[c][i].y, q[c][i].z, q[c][i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) s[c] = fmaf(E::high(w[e]), k[2 * e + 1], fmaf(E::low(w[e]), k[2 * e], s[c]));
    }
  }
#pragma unroll
  for (int c = 0; c < kPer; ++c) {
    float x = quad_sum(s[c]);
    if (p.cap_out != 0.0f) x = capped(x, p.cap_in, p.cap_out);
    if (key < first_key(pos[c], p.window_left) || key > pos[c]) continue;
    const float m = max3_nonan(st[c].m, x, x);
    const float alpha = st[c].m == m ? 1.0f : fast_exp2((st[c].m - m) * p.q_scale);
    const float f = x == m ? (m == -INFINITY ? 0.0f : 1.0f) : fast_exp2((x - m) * p.q_scale);
    st[c].m = m;
    st[c].l = st[c].l * alpha + (quad == 0 ? f : 0.0f);  // (a lane holds its part of the sum)
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) {
      const int d = 16 * dt + 4 * quad;
      pa_u32x2 w;
      if constexpr (kF8) {
        const uint32_t x = *reinterpret_cast<const uint32_t*>(vr + d);
        w = pa_u32x2{E::decode2<false>(x, vs), E::decode2<true>(x, vs)};
      } else {
        w = *reinterpret_cast<const pa_u32x2*>(vr + 2 * d);
      }
      const f32x4 v = {E::low(w.x), E::high(w.x), E::low(w.y), E::high(w.y)};
      acc[c][dt] = acc[c][dt] * alpha + v * f;
    }
  }
}

// One run's place in the stream or in the task list.
struct Run {
  PagedTask task;
  bool whole;  // the task's keys are all here: results go straight out
  int slot;    // else the partial state's place
};

// This workgroup's next run.  Stream form: x is the unit it starts at (moved past
// the run), x0 and x1 the workgroup's first and last.  Plain form: x is the round
// of tasks, x1 the number of tasks.  Tasks go longest rows first within a request,
// its KV heads side by side (with 8 of them, each on an XCD whose L2 its rows then
// share); every other whole round is dealt backwards, in eights, or the same
// workgroups would take the longer tasks of each (4 x 4096 rows 826 -> 777 us; a last,
// partial round goes to the first workgroups, which a CU serves first: 4 x 2048 rows of
// 64 dims 468 -> 413).  False: no more.
__device__ __forceinline__ bool next_run(PagedArgs& p, bool stream, const int* s_pre, int x0, int x1, int& x, Run& r) {
  int at = x;
  if (!stream) {
    const int grid = gridDim.x, w = blockIdx.x;
    const int64_t round = static_cast<int64_t>(x) * grid;
    const bool back = (x & 1) && grid % 8 == 0 && round + grid <= x1;
    const int64_t task = round + (back ? grid - 8 - (w & ~7) + (w & 7) : w);
    if (task >= x1) return false;
    at = static_cast<int>(task);
    ++x;
  } else if (x >= x1) {
    return false;
  }
  const int b = __builtin_amdgcn_readfirstlane(paged_find(s_pre, p.B, at));
  PagedRequest q = paged_request(p, b);
  q.q0 = __builtin_amdgcn_readfirstlane(q.q0);
  q.n = __builtin_amdgcn_readfirstlane(q.n);
  q.len = __builtin_amdgcn_readfirstlane(q.len);
  q.keys = __builtin_amdgcn_readfirstlane(q.keys);
  q.tasks = __builtin_amdgcn_readfirstlane(q.tasks);
  q.units = __builtin_amdgcn_readfirstlane(q.units);
  at -= __builtin_amdgcn_readfirstlane(s_pre[b]);
  if (!stream) {
    const int index = at / p.Hkv, h = at - index * p.Hkv;
    r.task = paged_task(p, b, q, h * q.tasks + (q.tasks - 1 - index));
    r.whole = true;
    r.slot = 0;
    return true;
  }
  const int index = at / q.units, unit = at - index * q.units;
  const int end = min(x1, x + q.units - unit);
  r.task = paged_task(p, b, q, index);
  r.whole = unit == 0 && end - x == q.units;
  r.slot = 2 * static_cast<int>(blockIdx.x) + (x == x0 ? 0 : 1);
  const int lo = r.task.klo + static_cast<int>(min(static_cast<int64_t>(unit) << p.unit_shift, int64_t{1} << 30));
  const int hi = r.task.klo + static_cast<int>(min(static_cast<int64_t>(unit + end - x) << p.unit_shift, int64_t{1} << 30));
  r.task.klo = min(lo, r.task.khi);
  r.task.khi = min(hi, r.task.khi);
  x = end;
  return true;
}

// ------------------------------------------------------------ stream body ---

// Few columns (16 kPer): the bytes of K and V bound the call, so the four waves
// take different keys, 32 at a time, and meet once, at the end of a run.  Rows of
// fewer than 256 bytes are read with their neighbours': two (four) waves take two
// (four) KV heads of the same keys, and a token's heads, which lie side by side,
// come from memory together (64 requests over 26K 8-bit keys of 8 heads of 128 dims
// 645 -> 600 us).  A wave needs no barrier on its way: it loads whole rows (a
// quarter of a wave reads one or two of them; operand order, a row per lane, takes
// eight times the cache lookups per byte and ran at 4.2 TB/s where this runs at
// 6.1), and stages them in tiles of LDS of its own, K as cached in XOR-swizzled
// chunks, V as 16-bit values for the transposing reads.  A block's registers are
// free for the next one's loads as soon as it is staged, so those are in flight
// while it is computed (a second block in flight, of 8-bit rows: 595 -> 643 us, for
// the registers); their page entries went out a block before.
//
// A wave's blocks that hold keys which only some rows see: a task has at most 32
// rows, so 31 such keys at either end, 2 blocks each (3 in all under a window
// shorter than that).
constexpr int kOddBlocks = 4;

template <int D, int kPer>
__global__ void __launch_bounds__(256, 2) stream_kernel(PagedParams) {
  constexpr int kS = D / 32;                // k-steps of a score
  constexpr int kRL = D * (kF8 ? 1 : 2) / 16;  // lanes (16-byte chunks) per cached row
  constexpr int kRI = 64 / kRL;             // rows per load
  constexpr int kNI = 32 / kRI;             // loads per block
  constexpr int kW = kF8 ? 2 : 1;           // staged V vectors, and k-steps, per chunk
  constexpr int kVU = D / 8 + 2;            // 16-byte units per staged V row
  constexpr int kDT = D / 16;
  constexpr int kC = 16 * kPer;
  constexpr int kOut = D + 4;               // floats per column of the joined state
  extern __shared__ int s_pre[];
  __shared__ int s_tmp[4];
  __shared__ pa_u32x4 s_k[4][32 * kRL];
  __shared__ pa_u32x4 s_v[4][32 * kVU];
  __shared__ float s_m[4][kC], s_l[4][kC];
  __shared__ pa_u32x2 s_odd[4][kOddBlocks];  // per wave: first key and key bits of blocks with keys to add apart
  static_assert(16 * kOut * 4 <= 32 * kVU * 16, "a wave's state fits its V tile");

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, quad = lane >> 4, col = lane & 15;
  PagedArgs& a0 = fresh_args();
  paged_plan<false>(a0, s_pre, s_tmp);
  const int total = __builtin_amdgcn_readfirstlane(s_pre[a0.B]);
  const Deal deal = stream_deal(a0, total);
  if (blockIdx.x == 0)
    for (int b = tid; b <= a0.B; b += 256) a0.plan[b] = s_pre[b];
  if (blockIdx.x >= deal.groups) return;
  const int x0 = deal.begin(blockIdx.x), x1 = deal.begin(blockIdx.x + 1);

  // chunk c of staged K row r lies at c ^ swizzle(r): eight rows' chunks on different banks
  auto swizzle = [](int r) { return kRL >= 16 ? r & 15 : (kRL == 8 ? r & 7 : (r >> 2) & 3); };
  const int ld_row = lane / kRL, ld_ch = lane % kRL;  // the lane's row of a load, its chunk
  const uint16_t* const vr = reinterpret_cast<const uint16_t*>(&s_v[wave][0]) + (4 * quad + (col >> 2)) * (kVU * 8) + 4 * (col & 3);

  // the wave's head in the task and its share of the keys
  const int heads_shift = a0.heads_shift, heads = 1 << heads_shift;
  const int own_head = wave & (heads - 1), key_step = 128 >> heads_shift;

  int x = x0;
  Run run;
  while (next_run(fresh_args(), true, s_pre, x0, x1, x, run)) {
    const PagedTask& t = run.task;
    PagedArgs& p = fresh_args();
    const int hkv = t.hkv + own_head;
    const float scale = p.q_scale;
    const int window = p.window_left;
    // (a static cache loads a word of K in the scale's place: a load that only
    // some calls make would leave the waits behind it uncounted)
    const bool scaled = kF8 && p.scales != nullptr;
    const uint16_t* const scales = scaled ? p.scales + (hkv << p.page_shift) : reinterpret_cast<const uint16_t*>(p.k);
    const uint32_t sc_ps = scaled ? static_cast<uint32_t>(p.Hkv) << p.page_shift : 0;  // scale words per page
    const int page_shift = p.page_shift, slot_mask = (1 << p.page_shift) - 1;
    const uint32_t num_pages = p.num_pages, kv_ps = p.kv_ps, kv_ss = p.kv_ss;
    // the wave's columns
    int pos[kPer];
    pa_u32x4 q[kPer][kS];
#pragma unroll
    for (int c = 0; c < kPer; ++c) {
      int row, head;
      lane_column(p, t, 16 * c + col, row, head);
      pos[c] = t.len - t.n + row;
      const uint16_t* at = p.q + static_cast<int64_t>(t.q0 + row) * p.q_ts + (hkv * p.G + head) * p.q_hs;
#pragma unroll
      for (int s = 0; s < kS; ++s)
        q[c][s] = *reinterpret_cast<const pa_u32x4*>(at + (kF8 ? 64 * (s >> 1) + 16 * quad + 8 * (s & 1) : 32 * s + 8 * quad));
    }
    // keys that every row of the task sees
    const int all_lo = first_key(t.len - t.n + t.row1, window);
    const int all_hi = t.len - t.n + t.row0 + 1;

    const char* const kb = p.k + at64(hkv, p.kv_hs) + 16 * ld_ch;
    const int64_t v_minus_k = p.v - p.k;
    const int last_entry = p.table_cols - 1;
    // the block in flight
    struct Flight {
      pa_u32x4 k[kNI], v[kNI];
      uint32_t sc, bad;  // scale bytes of key lane % 32, keys without a row
    };
    Flight fl;
    auto entry = [&](int base) {
      return t.table[static_cast<uint32_t>(min((base + (lane & 31)) >> page_shift, last_entry))];
    };
    auto load = [&](int base, int e) {
      const int key = base + (lane & 31);
      const bool ok = key < t.khi && static_cast<uint32_t>(e) < num_pages;
      fl.bad = ~static_cast<uint32_t>(__ballot(ok));
      const uint32_t page = ok ? e : 0;  // (a key without a row reads page 0: its weight is 0, its V zeroed)
#pragma unroll
      for (int i = 0; i < kNI; ++i) {
        const int src = kRI * i + ld_row;
        const char* at = kb + at64(__shfl(page, src), kv_ps) + at64((base + src) & slot_mask, kv_ss);
        fl.k[i] = __builtin_nontemporal_load(reinterpret_cast<const pa_u32x4*>(at));
        fl.v[i] = __builtin_nontemporal_load(reinterpret_cast<const pa_u32x4*>(at + v_minus_k));
      }
      if constexpr (kF8) fl.sc = scales[static_cast<uint64_t>(page) * sc_ps + (scaled ? key & slot_mask : 0)];
    };

    Column st[kPer];
    f32x4 acc[kPer][kDT];
#pragma unroll
    for (int c = 0; c < kPer; ++c) {
      st[c] = fresh_column();
#pragma unroll
      for (int dt = 0; dt < kDT; ++dt) acc[c][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    bool far = false;
    int n_odd = 0;  // blocks in s_odd
    // the wave's blocks: every fourth of the run's (of two heads: every second)
    int base = t.klo + 32 * (wave >> heads_shift);
    int e_next = 0;  // entries of the block to load next
    if (base < t.khi) {
      const int e = entry(base);
      e_next = entry(base + key_step);
      load(base, e);
    }
    auto step = [&]() {  // (written out in the loop, rows of 64 bytes took 488 us for 432)
      const uint32_t bad = __builtin_amdgcn_readfirstlane(fl.bad);
      const bool part = base < all_lo || base + 32 > all_hi;  // some row of the task does not see some key
      const bool masked = part || bad != 0;
      const uint32_t sc = kF8 && scaled ? fl.sc : 0x7f7fu;
      // rows to LDS
      pa_u32x4 w[kNI][kW];
#pragma unroll
      for (int i = 0; i < kNI; ++i) {
        if constexpr (kF8) decode16<kT>(fl.v[i], __uint_as_float((__shfl(sc, kRI * i + ld_row) >> 8) << 23), w[i][0], w[i][1]);
        else w[i][0] = fl.v[i];
      }
      uint32_t odd = 0;  // keys with V that is not finite
      if (masked) {
#pragma unroll
        for (int i = 0; i < kNI; ++i) {
          const bool ok = !((bad >> (kRI * i + ld_row)) & 1);
          bool odd_row = false;
#pragma unroll
          for (int h = 0; h < kW; ++h) {
            const bool nf = ok && part && not_finite<kT>(w[i][h]);
            odd_row = odd_row || nf;
            const uint32_t z = ok && !nf ? 0xffffffffu : 0u;
            w[i][h] = pa_u32x4{w[i][h].x & z, w[i][h].y & z, w[i][h].z & z, w[i][h].w & z};
          }
          const uint64_t o = __ballot(odd_row);
          if (o != 0) {
#pragma unroll
            for (int r = 0; r < kRI; ++r) odd |= static_cast<uint32_t>(((o >> (kRL * r)) & ((1ull << kRL) - 1)) != 0) << (kRI * i + r);
          }
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (the block before is read)
#pragma unroll
      for (int i = 0; i < kNI; ++i) {
        const int r = kRI * i + ld_row;
        s_k[wave][r * kRL + (ld_ch ^ swizzle(r))] = fl.k[i];
#pragma unroll
        for (int h = 0; h < kW; ++h) s_v[wave][r * kVU + kW * ld_ch + h] = w[i][h];
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_sched_barrier(0);
      if (base + key_step < t.khi) {
        const int e_after = entry(base + 2 * key_step);  // (ahead of the rows: the wait for it is no wait for them)
        load(base + key_step, e_next);
        e_next = e_after;
      }
      __builtin_amdgcn_sched_barrier(0);
      if (odd != 0) {
        if (lane == 0) s_odd[wave][n_odd] = pa_u32x2{static_cast<uint32_t>(base), odd};
        ++n_odd;
      }
      // scores
      f32x4 s4[kPer][2];
#pragma unroll
      for (int c = 0; c < kPer; ++c)
#pragma unroll
        for (int i = 0; i < 2; ++i) s4[c][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      float ks[2] = {1.0f, 1.0f};
      if constexpr (kF8) {
#pragma unroll
        for (int i = 0; i < 2; ++i) ks[i] = __uint_as_float((__shfl(sc, 16 * i + col) & 255u) << 23);
      }
#pragma unroll
      for (int ch = 0; ch < kRL / 4; ++ch) {
        pa_u32x4 a[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const pa_u32x4 raw = s_k[wave][(16 * i + col) * kRL + ((4 * ch + quad) ^ swizzle(16 * i + col))];
          if constexpr (kF8) decode16<kT>(raw, ks[i], a[i][0], a[i][1]);
          else a[i][0] = raw;
        }
#pragma unroll
        for (int h = 0; h < kW; ++h)
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int c = 0; c < kPer; ++c) s4[c][i] = E::mfma(a[i][h], q[c][kW * ch + h], s4[c][i]);
      }
      if (p.cap_out != 0.0f) {
#pragma unroll
        for (int c = 0; c < kPer; ++c) cap_scores(s4[c], p.cap_in, p.cap_out);
      }
      if (masked) {
#pragma unroll
        for (int c = 0; c < kPer; ++c)
          mask_scores(&s4[c][0], seen_keys(base, first_key(pos[c], window), min(pos[c] + 1, t.khi), bad | odd, quad));
      }
      float f[kPer][8];
      weigh(s4, scale, st, far, acc, f);
      pa_u32x4 pb[kPer];
#pragma unroll
      for (int c = 0; c < kPer; ++c) pb[c] = pack8(f[c]);
#pragma unroll
      for (int dt = 0; dt < kDT; ++dt) {
        const pa_u32x4 a = join(read_tr(vr + 16 * dt), read_tr(vr + 16 * kVU * 8 + 16 * dt));
#pragma unroll
        for (int c = 0; c < kPer; ++c) acc[c][dt] = E::mfma(a, pb[c], acc[c][dt]);
      }
    };
    while (base < t.khi) {
      step();
      base += key_step;
    }

    PagedArgs& e = fresh_args();
    for (int i = 0; i < n_odd; ++i) {
      const pa_u32x2 o = s_odd[wave][i];
      const int first = __builtin_amdgcn_readfirstlane(o.x);
      for (uint32_t left = __builtin_amdgcn_readfirstlane(o.y); left != 0; left &= left - 1)
        add_key<D, kPer, kF8>(e, t, hkv, first + __builtin_ctz(left), q, pos, st, acc, quad);
    }

    // the four waves' states joined
#pragma unroll
    for (int c = 0; c < kPer; ++c) {
      const float l = quad_sum(st[c].l);
      if (quad == 0) {
        s_m[wave][16 * c + col] = st[c].m * scale;  // (-inf: no key)
        s_l[wave][16 * c + col] = l;
      }
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < kPer; ++c) {
      float m = s_m[own_head][16 * c + col];
      for (int w = own_head + heads; w < 4; w += heads) m = fmaxf(m, s_m[w][16 * c + col]);
      const float own = s_m[wave][16 * c + col];
      // (-inf for a state without keys: weight 0, or 1 where no wave has any)
      const float f = own == m ? 1.0f : fast_exp2(own - m);
      float* o = reinterpret_cast<float*>(&s_v[wave][0]) + col * kOut + 4 * quad;
#pragma unroll
      for (int dt = 0; dt < kDT; ++dt) *reinterpret_cast<f32x4*>(o + 16 * dt) = acc[c][dt] * f;
      __syncthreads();
      // 16 threads per column, D / 16 dims each
      const int cc = tid >> 4, d0 = (tid & 15) * kDT;
      const int gcol = 16 * c + cc;
      for (int h = 0; h < heads; ++h) {
        float mx = s_m[h][gcol], l = 0.0f;
        for (int w = h + heads; w < 4; w += heads) mx = fmaxf(mx, s_m[w][gcol]);
        for (int w = h; w < 4; w += heads) l += s_l[w][gcol] * (s_m[w][gcol] == mx ? 1.0f : fast_exp2(s_m[w][gcol] - mx));
        if (gcol < t.nc) {
          float r[kDT];
#pragma unroll
          for (int i = 0; i < kDT; i += 4) {
            f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int w = h; w < 4; w += heads) sum += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(&s_v[w][0]) + cc * kOut + d0 + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) r[i + j] = sum[j];
          }
          if (run.whole) {
            int row, head;
            lane_column(e, t, gcol, row, head);
            const int64_t at = static_cast<int64_t>(t.q0 + row) * e.Hq + (t.hkv + h) * e.G + head;
            const float inv = l == 0.0f ? 0.0f : e.v_scale / l;
#pragma unroll
            for (int i = 0; i < kDT; i += 4)
              *reinterpret_cast<pa_u32x2*>(e.out + at * D + d0 + i) =
                  pa_u32x2{E::pack2(r[i] * inv, r[i + 1] * inv), E::pack2(r[i + 2] * inv, r[i + 3] * inv)};
            if (d0 == 0) e.lse[at] = l == 0.0f ? -INFINITY : (mx + fast_log2(l)) * kLn2;
          } else {
            const int64_t at = (static_cast<int64_t>(run.slot) * heads + h) * kC + gcol;
#pragma unroll
            for (int i = 0; i < kDT; i += 4)
              *reinterpret_cast<f32x4*>(e.part_o + at * D + d0 + i) = f32x4{r[i], r[i + 1], r[i + 2], r[i + 3]};
            if (d0 == 0) {
              e.part_ml[at * 2] = mx;
              e.part_ml[at * 2 + 1] = l;
            }
          }
        }
      }
      __syncthreads();  // the tiles and sums are free again
    }
  }
}

// -------------------------------------------------------------- tile body ---

// Many columns (64 kPer): the matrix cores bound the call, so the four waves
// take different columns, kPer tiles each, and share K and V tiles of kBlk keys
// in double-buffered LDS.  K chunk c (16 bytes) of key k lies at position c ^ (k
// & 15) (& 7 for 64 dims) of its row, so that the 16 keys an operand reads lie
// on different banks; V rows are padded by 32 bytes for the transposing reads.
template <int D, int kPer, int kBlk, int kOcc>
__global__ void __launch_bounds__(256, kOcc) tile_kernel(PagedParams) {
  constexpr int kS = D / 32;
  constexpr int kDT = D / 16;
  constexpr int kKU = D / 8;               // 16-byte units per staged K row
  constexpr int kVU = D / 8 + 2;
  constexpr int kSwz = kKU < 16 ? kKU - 1 : 15;
  constexpr int kRowCh = kF8 ? D / 16 : D / 8;  // 16-byte chunks of a cached row
  constexpr int kStep = 256 / kRowCh;           // keys per pass of the workgroup
  constexpr int kLd = kBlk / kStep;
  constexpr int kSub = kBlk / 32;
  constexpr int kW = kF8 ? 2 : 1;  // staged vectors per chunk
  // blocks in flight.  64 columns are for calls that the bytes of K and V bound: a
  // second block where one has 16 KiB (32 requests of 5 rows of 8 heads over 16K 8-bit
  // keys of 128 dims 182 -> 158 us, over 26K 16-bit ones of 64 dims 207 -> 192), not
  // where it has 32 (235 -> 243) or rows of 64 bytes, half of a memory line (151 -> 175)
  constexpr int kSets = kPer == 1 && D * (kF8 ? 1 : 2) == 128 ? 2 : 1;
  static_assert(kLd >= 1, "a block is at least one pass");
  // blocks in which some row of the task misses some key: at either end of its
  // keys the rows' 64 kPer - 1 and one block's
  constexpr int kOdd = 2 * ((64 * kPer + kBlk - 1) / kBlk + 2);
  extern __shared__ int s_pre[];
  __shared__ int s_tmp[4];
  __shared__ pa_u32x4 s_k[2][kBlk * kKU];
  __shared__ pa_u32x4 s_v[2][kBlk * kVU];
  __shared__ pa_u32x4 s_bad[2][kSub];  // per wave: its keys (of each 32) without a row
  __shared__ pa_u32x4 s_odd[kOdd][kSub];  // and, of the blocks at the rows' edges, its keys to add apart
  __shared__ int s_odd_at[kOdd];       // the blocks' first keys

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, quad = lane >> 4, col = lane & 15;
  PagedArgs& a0 = fresh_args();
  const bool stream = paged_plan<true>(a0, s_pre, s_tmp);
  const int total = __builtin_amdgcn_readfirstlane(s_pre[a0.B]);
  int x0 = 0, x1 = total;
  if (a0.stream != kPlain && blockIdx.x == 0) {
    for (int b = tid; b <= a0.B; b += 256) a0.plan[b] = s_pre[b];
    if (tid == 0) a0.plan[a0.B + 1] = stream;
  }
  if (stream) {
    const Deal deal = stream_deal(a0, total);
    if (blockIdx.x >= deal.groups) return;
    x0 = deal.begin(blockIdx.x);
    x1 = deal.begin(blockIdx.x + 1);
  }
  // loader: thread t stages chunk t % kRowCh of keys t / kRowCh + kStep i
  const int ld_key = tid / kRowCh, ld_ch = tid % kRowCh;
  // compute: the lane's V^T read position
  const int rd_v = (4 * quad + (col >> 2)) * (kVU * 8) + 4 * (col & 3);

  int x = x0;
  Run run;
  while (next_run(fresh_args(), stream, s_pre, x0, x1, x, run)) {
    const PagedTask& t = run.task;
    PagedArgs& p = fresh_args();
    const float scale = p.q_scale;
    const int window = p.window_left;
    // (a static cache loads a word of K in the scale's place: a load that only
    // some calls make would leave the waits behind it uncounted)
    const bool scaled = kF8 && p.scales != nullptr;
    const uint16_t* const scales = scaled ? p.scales + (t.hkv << p.page_shift) : reinterpret_cast<const uint16_t*>(p.k);
    const uint32_t sc_ps = scaled ? static_cast<uint32_t>(p.Hkv) << p.page_shift : 0;  // scale words per page
    const int page_shift = p.page_shift, slot_mask = (1 << p.page_shift) - 1;
    const uint32_t num_pages = p.num_pages, kv_ps = p.kv_ps, kv_ss = p.kv_ss;
    int pos[kPer];
    pa_u32x4 q[kPer][kS];
#pragma unroll
    for (int c = 0; c < kPer; ++c) {
      int row, head;
      lane_column(p, t, 16 * (kPer * wave + c) + col, row, head);
      pos[c] = t.len - t.n + row;
      const uint16_t* at = p.q + static_cast<int64_t>(t.q0 + row) * p.q_ts + (t.hkv * p.G + head) * p.q_hs;
#pragma unroll
      for (int s = 0; s < kS; ++s) q[c][s] = *reinterpret_cast<const pa_u32x4*>(at + 32 * s + 8 * quad);
    }
    // the wave's first and last row, and the keys they leave unmasked or need
    const int c0 = 16 * kPer * wave;
    const bool live = c0 < t.nc;
    const int pf = t.len - t.n + (t.gc0 + min(c0, t.nc - 1)) / p.G;
    const int pl = t.len - t.n + (t.gc0 + min(c0 + 16 * kPer, t.nc) - 1) / p.G;  // (of no use to a wave that is not live)
    const int all_lo = first_key(pl, window), all_hi = pf + 1;
    const int any_lo = first_key(pf, window), any_hi = min(pl + 1, t.khi);
    // keys past which some row of the task is masked (for the staging's look at V)
    const int task_lo = first_key(t.len - t.n + t.row1, window);
    const int task_hi = t.len - t.n + t.row0 + 1;

    const char* const kb = p.k + at64(t.hkv, p.kv_hs) + 16 * ld_ch;
    const int64_t v_minus_k = p.v - p.k;
    const int last_entry = p.table_cols - 1;
    // the blocks in flight
    struct Flight {
      pa_u32x4 k[kLd], v[kLd];
      uint32_t sc[kLd];
      uint32_t ok;  // bit i: key i of the thread's has a row
    };
    Flight flight[kSets];
    int en[kLd], en_after[kLd];  // entries of the block to load next, and of the one after
    auto entries = [&](int base, int (&en)[kLd]) {
#pragma unroll
      for (int i = 0; i < kLd; ++i)
        en[i] = t.table[static_cast<uint32_t>(min((base + ld_key + kStep * i) >> page_shift, last_entry))];
    };
    auto load = [&](int base, const int (&en)[kLd], Flight& fl) {
      fl.ok = 0;
#pragma unroll
      for (int i = 0; i < kLd; ++i) {
        const int key = base + ld_key + kStep * i;
        const bool in = key < t.khi && static_cast<uint32_t>(en[i]) < num_pages;
        fl.ok |= in ? 1u << i : 0u;
        const uint32_t page = in ? en[i] : 0;  // (a key without a row reads page 0: its weight is 0, its V zeroed)
        const char* at = kb + at64(page, kv_ps) + at64(key & slot_mask, kv_ss);
        fl.k[i] = *reinterpret_cast<const pa_u32x4*>(at);
        fl.v[i] = *reinterpret_cast<const pa_u32x4*>(at + v_minus_k);
        if constexpr (kF8) fl.sc[i] = scales[static_cast<uint64_t>(page) * sc_ps + (scaled ? key & slot_mask : 0)];
      }
    };

    Column st[kPer];
    f32x4 acc[kPer][kDT];
#pragma unroll
    for (int c = 0; c < kPer; ++c) {
      st[c] = fresh_column();
#pragma unroll
      for (int dt = 0; dt < kDT; ++dt) acc[c][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    const int nblk = t.khi > t.klo ? ceil_div(t.khi - t.klo, kBlk) : 0;
    if (nblk > 0) {
#pragma unroll
      for (int i = 0; i < kSets; ++i) {
        entries(t.klo + kBlk * i, en);
        if (i == kSets - 1) entries(t.klo + kBlk * kSets, en_after);
        load(t.klo + kBlk * i, en, flight[i]);
      }
    }
    int n_part = 0;
    bool far = false;
    __syncthreads();  // the run before is done with the tiles
    int bi = 0;
    auto step = [&](Flight& fl) {
      const int buf = bi & 1;
      const int base = t.klo + bi * kBlk;
      const bool part = base < task_lo || base + kBlk > task_hi;
      {
        uint32_t odd_rows = 0;  // bit i: the thread's part of row i
        const bool whole = __all(fl.ok == (1u << kLd) - 1u);
#pragma unroll
        for (int i = 0; i < kLd; ++i) {
          const int key = ld_key + kStep * i;
          pa_u32x4* const kd = &s_k[buf][key * kKU];
          pa_u32x4* const vd = &s_v[buf][key * kVU];
          pa_u32x4 k2[kW], v2[kW];
          if constexpr (kF8) {
            const uint32_t b2 = scaled ? fl.sc[i] : 0x7f7fu;
            decode16<kT>(fl.k[i], __uint_as_float((b2 & 255u) << 23), k2[0], k2[1]);
            decode16<kT>(fl.v[i], __uint_as_float((b2 >> 8) << 23), v2[0], v2[1]);
          } else {
            k2[0] = fl.k[i];
            v2[0] = fl.v[i];
          }
          if (part || !whole) {
            const bool in = (fl.ok >> i) & 1;
#pragma unroll
            for (int h = 0; h < kW; ++h) {
              const bool nf = in && part && not_finite<kT>(v2[h]);
              odd_rows |= nf ? 1u << i : 0u;
              const uint32_t z = in && !nf ? 0xffffffffu : 0u;
              v2[h] &= pa_u32x4{z, z, z, z};
            }
          }
#pragma unroll
          for (int h = 0; h < kW; ++h) {
            const int u = kW * ld_ch + h;
            kd[u ^ (key & kSwz)] = k2[h];
            vd[u] = v2[h];
          }
        }
        // the wave's keys: 64 / kRowCh of each pass
        uint64_t bad = 0, odd = 0;
        if (!whole || (part && __any(odd_rows))) {
#pragma unroll
          for (int i = 0; i < kLd; ++i) {
            const uint64_t no = __ballot(((fl.ok >> i) & 1) == 0), od = __ballot((odd_rows >> i) & 1);
#pragma unroll
            for (int r = 0; r < 64 / kRowCh; ++r) {
              const int key = kStep * i + (64 / kRowCh) * wave + r;
              bad |= ((no >> (kRowCh * r)) & 1) << key;
              odd |= static_cast<uint64_t>(((od >> (kRowCh * r)) & ((1ull << kRowCh) - 1)) != 0) << key;
            }
          }
        }
        if (lane == 0) {
#pragma unroll
          for (int h = 0; h < kSub; ++h) {
            reinterpret_cast<uint32_t*>(&s_bad[buf][h])[wave] = static_cast<uint32_t>((bad | odd) >> (32 * h));
            if (part) reinterpret_cast<uint32_t*>(&s_odd[n_part][h])[wave] = static_cast<uint32_t>(odd >> (32 * h));
          }
          if (part && wave == 0) s_odd_at[n_part] = base;
        }
        if (part) ++n_part;
      }
      __syncthreads();  // the block is visible; every wave is done with the block before last
      // (with two in flight, blocks past the run are loaded too, the cache's first
      // page: behind a branch their number would be unknown to the waits for the
      // one before)
      if (kSets > 1 || bi + 1 < nblk) {
#pragma unroll
        for (int i = 0; i < kLd; ++i) en[i] = en_after[i];
        entries(base + kBlk * (kSets + 1), en_after);  // (ahead of the rows: the wait for them is no wait for those)
        load(base + kBlk * kSets, en, fl);
      }
      if (!live || base + kBlk <= any_lo || base >= any_hi) return;
      // both products take all of the block's keys, so that one vote and one set
      // of branches serves them and the exponentials of one half overlap the other's
      // products
      uint32_t bad[kSub];
      bool masked = base < all_lo || base + kBlk > all_hi;
      const pa_u32x4* const kt = &s_k[buf][col * kKU];
      const uint16_t* const vt = reinterpret_cast<const uint16_t*>(&s_v[buf][0]) + rd_v;
      pa_u32x4 bw[kSub];
#pragma unroll
      for (int h = 0; h < kSub; ++h) bw[h] = s_bad[buf][h];
      f32x4 s4[kPer][2 * kSub];
#pragma unroll
      for (int c = 0; c < kPer; ++c)
#pragma unroll
        for (int i = 0; i < 2 * kSub; ++i) s4[c][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int h = 0; h < kSub; ++h)
#pragma unroll
        for (int s = 0; s < kS; ++s)
#pragma unroll
          for (int i = 2 * h; i < 2 * h + 2; ++i) {
            const pa_u32x4 a = kt[16 * i * kKU + ((4 * s + quad) ^ (col & kSwz))];
#pragma unroll
            for (int c = 0; c < kPer; ++c) s4[c][i] = E::mfma(a, q[c][s], s4[c][i]);
          }
#pragma unroll
      for (int h = 0; h < kSub; ++h) {
        bad[h] = __builtin_amdgcn_readfirstlane(bw[h].x | bw[h].y | bw[h].z | bw[h].w);
        masked = masked || bad[h] != 0;
      }
      if (p.cap_out != 0.0f) {
#pragma unroll
        for (int c = 0; c < kPer; ++c) cap_scores(s4[c], p.cap_in, p.cap_out);
      }
      if (masked) {
#pragma unroll
        for (int c = 0; c < kPer; ++c)
#pragma unroll
          for (int h = 0; h < kSub; ++h)
            mask_scores(&s4[c][2 * h], seen_keys(base + 32 * h, first_key(pos[c], window), min(pos[c] + 1, t.khi), bad[h], quad));
      }
      float f[kPer][8 * kSub];
      weigh(s4, scale, st, far, acc, f);
#pragma unroll
      for (int h = 0; h < kSub; ++h) {
        pa_u32x4 pb[kPer];
#pragma unroll
        for (int c = 0; c < kPer; ++c) pb[c] = pack8(&f[c][8 * h]);
#pragma unroll
        for (int dt = 0; dt < kDT; ++dt) {
          const uint16_t* const at = vt + 32 * h * kVU * 8 + 16 * dt;
          const pa_u32x4 a = join(read_tr(at), read_tr(at + 16 * kVU * 8));
#pragma unroll
          for (int c = 0; c < kPer; ++c) acc[c][dt] = E::mfma(a, pb[c], acc[c][dt]);
        }
      }
    };
    while (bi < nblk) {
      step(flight[0]);
      ++bi;
      if constexpr (kSets > 1) {
        if (bi >= nblk) break;
        step(flight[1]);
        ++bi;
      }
    }
    if (!live) continue;
    PagedArgs& e = fresh_args();
    for (int i = 0; i < n_part; ++i)
#pragma unroll 1
      for (int h = 0; h < kSub; ++h) {
        const pa_u32x4 o = s_odd[i][h];
        const int first = __builtin_amdgcn_readfirstlane(s_odd_at[i]) + 32 * h;
        for (uint32_t left = __builtin_amdgcn_readfirstlane(o.x | o.y | o.z | o.w); left != 0; left &= left - 1)
          add_key<D, kPer, false>(e, t, t.hkv, first + __builtin_ctz(left), q, pos, st, acc, quad);
      }
#pragma unroll
    for (int c = 0; c < kPer; ++c) {
      const float l = quad_sum(st[c].l);
      const int cc = 16 * (kPer * wave + c) + col;
      if (cc >= t.nc) continue;
      const float m = st[c].m * e.q_scale;
      if (run.whole) {
        int row, head;
        lane_column(e, t, cc, row, head);
        const int64_t at = static_cast<int64_t>(t.q0 + row) * e.Hq + t.hkv * e.G + head;
        const float inv = l == 0.0f ? 0.0f : e.v_scale / l;
        uint16_t* o = e.out + at * D + 4 * quad;
#pragma unroll
        for (int dt = 0; dt < kDT; ++dt)
          *reinterpret_cast<pa_u32x2*>(o + 16 * dt) = pa_u32x2{E::pack2(acc[c][dt][0] * inv, acc[c][dt][1] * inv),
                                                              E::pack2(acc[c][dt][2] * inv, acc[c][dt][3] * inv)};
        if (quad == 0) e.lse[at] = l == 0.0f ? -INFINITY : (m + fast_log2(l)) * kLn2;
      } else {
        const int64_t at = static_cast<int64_t>(run.slot) * (64 * kPer) + cc;
        float* o = e.part_o + at * D + 4 * quad;
#pragma unroll
        for (int dt = 0; dt < kDT; ++dt) *reinterpret_cast<f32x4*>(o + 16 * dt) = acc[c][dt];
        if (quad == 0) {
          e.part_ml[at * 2] = m;
          e.part_ml[at * 2 + 1] = l;
        }
      }
    }
  }
}

// ---------------------------------------------------------------- combine ---

// Stream form, second launch: the partial states of a task that several
// workgroups shared.  Rows of whole tasks return at once.
//
// Where the pieces of query row `row` and head `head` of request b lie: the
// workgroups first .. first + n - 1, n = 0 for a task that one workgroup had.
struct Pieces {
  int first, n;
  bool at_start;  // the first one's run begins with the task
  int offset;      // of the column in a slot
  __device__ __forceinline__ int64_t place(int i, int64_t slot_columns) const {
    const int64_t slot = 2 * static_cast<int64_t>(first + i) + (i == 0 && !at_start ? 1 : 0);
    return slot * slot_columns + offset;
  }
};
__device__ __forceinline__ Pieces find_pieces(PagedArgs& p, const PagedRequest& r, int before, const Deal& deal, int row, int head, int kc) {
  const int hkv = head / p.G;
  const int gc = (row - r.q0) * p.G + head - hkv * p.G;
  const int ct = gc / p.cols, col = gc - ct * p.cols;
  const int group = hkv >> p.heads_shift;
  const int unit = before + (group * r.tasks + ct) * r.units;
  Pieces x;
  x.first = deal.owner(unit);
  x.n = deal.owner(unit + r.units - 1) - x.first;
  x.n = x.n > 0 ? x.n + 1 : 0;
  x.at_start = deal.begin(x.first) == unit;
  x.offset = (hkv - (group << p.heads_shift)) * kc + col;
  return x;
}
// The request that a row belongs to (-1: none), for a whole workgroup.
__device__ __forceinline__ int request_of_row(PagedArgs& p, int row) {
  __shared__ int s_b;
  if (threadIdx.x == 0) s_b = -1;
  __syncthreads();
  for (int b = threadIdx.x; b < p.B; b += 256)
    if (p.qo_indptr[b] <= row && row < p.qo_indptr[b + 1]) s_b = b;
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(s_b);
}
// A wave's state over the pieces i0, i0 + step, ..: lane l holds dims l + 64 j.
template <int kV>
struct Joined {
  float m, l, o[kV];
};
template <int kV>
__device__ __forceinline__ Joined<kV> join_pieces(PagedArgs& p, const Pieces& x, int64_t slot_columns, int i0, int step) {
  constexpr int D = 64 * kV, kB = 4;  // pieces' loads in flight
  const int lane = threadIdx.x & 63;
  Joined<kV> s = {-INFINITY, 0.0f, {}};
  for (; i0 < x.n; i0 += step * kB) {
    float pm[kB], pl[kB], po[kB][kV];
#pragma unroll
    for (int u = 0; u < kB; ++u) {
      const int64_t at = x.place(min(i0 + step * u, x.n - 1), slot_columns);
      pm[u] = p.part_ml[2 * at];
      pl[u] = p.part_ml[2 * at + 1];
#pragma unroll
      for (int j = 0; j < kV; ++j) po[u][j] = p.part_o[at * D + 64 * j + lane];
    }
#pragma unroll
    for (int u = 0; u < kB; ++u) {
      if (i0 + step * u >= x.n) break;
      const float mn = max3_nonan(s.m, pm[u], pm[u]);
      const float fa = s.m == mn ? 1.0f : fast_exp2(s.m - mn), fb = pm[u] == mn ? 1.0f : fast_exp2(pm[u] - mn);
      s.m = mn;
      s.l = s.l * fa + pl[u] * fb;
#pragma unroll
      for (int j = 0; j < kV; ++j) s.o[j] = s.o[j] * fa + po[u][j] * fb;
    }
  }
  return s;
}

// Rows in many pieces: one workgroup per (row, query head), its waves take every
// fourth piece.
template <int D>
__global__ void __launch_bounds__(256) combine_kernel(PagedParams, int kc) {
  PagedArgs& p = fresh_args();
  constexpr int kV = D / 64;
  __shared__ float s_o[4][D], s_m[4], s_l[4];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (p.stream == kEither && p.plan[p.B + 1] == 0) return;  // plain form
  const int row = blockIdx.x / p.Hq, head = blockIdx.x - row * p.Hq;
  const int b = request_of_row(p, row);
  if (b < 0) return;
  const PagedRequest r = paged_request(p, b);
  if (r.n == 0) return;
  const Pieces x = find_pieces(p, r, p.plan[b], stream_deal(p, p.plan[p.B]), row, head, kc);
  if (x.n == 0) return;  // stored by its workgroup
  const Joined<kV> s = join_pieces<kV>(p, x, static_cast<int64_t>(kc) << p.heads_shift, wave, 4);
#pragma unroll
  for (int j = 0; j < kV; ++j) s_o[wave][64 * j + lane] = s.o[j];
  if (lane == 0) {
    s_m[wave] = s.m;
    s_l[wave] = s.l;
  }
  __syncthreads();
  float mx = s_m[0], lt = 0.0f;
#pragma unroll
  for (int w = 1; w < 4; ++w) mx = max3_nonan(mx, s_m[w], s_m[w]);
  float f[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[w] = s_m[w] == mx ? 1.0f : fast_exp2(s_m[w] - mx);
    lt += s_l[w] * f[w];
  }
  const int64_t at = static_cast<int64_t>(row) * p.Hq + head;
  const float inv = lt == 0.0f ? 0.0f : p.v_scale / lt;
  for (int d = 2 * tid; d < D; d += 512) {
    float y[2] = {0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      y[0] += s_o[w][d] * f[w];
      y[1] += s_o[w][d + 1] * f[w];
    }
    *reinterpret_cast<uint32_t*>(p.out + at * D + d) = E::pack2(y[0] * inv, y[1] * inv);
  }
  if (tid == 0) p.lse[at] = lt == 0.0f ? -INFINITY : (mx + fast_log2(lt)) * kLn2;
}

// Rows in few pieces: gridDim.y workgroups per row, a wave per query head in turn;
// 64 heads' pieces are looked up together, one in a lane.
template <int D>
__global__ void __launch_bounds__(256) combine_rows_kernel(PagedParams, int kc) {
  PagedArgs& p = fresh_args();
  constexpr int kV = D / 64;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (p.plan[p.B + 1] == 0) return;  // plain form
  const int row = blockIdx.x;
  const int b = request_of_row(p, row);
  if (b < 0) return;
  const PagedRequest r = paged_request(p, b);
  if (r.n == 0) return;
  const int before = p.plan[b];
  const Deal deal = stream_deal(p, p.plan[p.B]);
  const int step = 4 * gridDim.y;
  Pieces found = {};
  for (int i = 0, head = 4 * blockIdx.y + wave; head < p.Hq; ++i, head += step) {
    if (i % 64 == 0) found = find_pieces(p, r, before, deal, row, min(head + step * lane, p.Hq - 1), kc);
    Pieces x;
    x.n = __builtin_amdgcn_readlane(found.n, i % 64);
    if (x.n == 0) continue;
    x.first = __builtin_amdgcn_readlane(found.first, i % 64);
    x.at_start = __builtin_amdgcn_readlane(found.at_start, i % 64);
    x.offset = __builtin_amdgcn_readlane(found.offset, i % 64);
    const Joined<kV> s = join_pieces<kV>(p, x, static_cast<int64_t>(kc) << p.heads_shift, 0, 1);
    const int64_t at = static_cast<int64_t>(row) * p.Hq + head;
    const float inv = s.l == 0.0f ? 0.0f : p.v_scale / s.l;
#pragma unroll
    for (int j = 0; j < kV; ++j) p.out[at * D + 64 * j + lane] = static_cast<uint16_t>(E::pack2(s.o[j] * inv, 0.0f));
    if (lane == 0) p.lse[at] = s.l == 0.0f ? -INFINITY : (s.m + fast_log2(s.l)) * kLn2;
  }
}

// ----------------------------------------------------------------- launch ---

typedef void (*Kernel)(PagedParams);
typedef void (*Kernel2)(PagedParams, int);

template <int D>
Kernel body_kernel(int body) {
  if constexpr (D <= 128) {
    switch (body) {
      case kBodyStream16: return stream_kernel<D, 1>;
      case kBodyStream32:
        if constexpr (kF8 || D == 64) return stream_kernel<D, 2>;
        return nullptr;
      case kBodyTile64: return tile_kernel<D, 1, 64, 2>;
      default: return tile_kernel<D, 2, 64, (D == 64 ? 3 : 2)>;
    }
  } else {
    return tile_kernel<D, 1, 32, 2>;  // (the other bodies' states and operands of 256 dims exceed a wave's registers)
  }
}
Kernel body_of(int D, int body) {
  return D == 64 ? body_kernel<64>(body) : (D == 128 ? body_kernel<128>(body) : body_kernel<256>(body));
}
template <int D>
Kernel2 combine_of(bool by_rows) {
  return by_rows ? combine_rows_kernel<D> : combine_kernel<D>;
}
size_t plan_bytes(int B) { return sizeof(int) * (static_cast<size_t>(B) + 1); }

}  // namespace

#define MAC_PAGED_CAT2(a, b) a##b
#define MAC_PAGED_CAT(a, b) MAC_PAGED_CAT2(a, b)

namespace mac {

int MAC_PAGED_CAT(paged_resident_, MAC_PAGED_NAME)(int D, int body, int B) {
  // (queries of the runtime, some microseconds each: once per device for plans of
  // up to 4 KiB, which take a workgroup's room from none of the bodies)
  constexpr int kDevices = 64;
  constexpr size_t kPlan = 4096;
  static std::atomic<int> known[kDevices][3][kBodies];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return 1;
  const size_t bytes = std::max(plan_bytes(B), kPlan);
  std::atomic<int>* slot = bytes == kPlan && dev >= 0 && dev < kDevices ? &known[dev][D == 64 ? 0 : (D == 128 ? 1 : 2)][body] : nullptr;
  if (slot != nullptr)
    if (const int n = slot->load(std::memory_order_relaxed)) return n;
  int cus = 256, v = 0, per = 1;
  if (hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && v > 0) cus = v;
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&per, reinterpret_cast<const void*>(body_of(D, body)), 256, bytes) != hipSuccess ||
      per < 1)
    per = 1;
  if (slot != nullptr) slot->store(cus * per, std::memory_order_relaxed);
  return cus * per;
}

hipError_t MAC_PAGED_CAT(paged_launch_, MAC_PAGED_NAME)(const PagedParams& p, int D, int body, hipStream_t stream) {
  hipLaunchKernelGGL(body_of(D, body), dim3(p.grid), dim3(256), plan_bytes(p.B), stream, p);
  if (p.stream != kPlain) {
    const Kernel2 kern = D == 64 ? combine_of<64>(p.by_rows) : (D == 128 ? combine_of<128>(p.by_rows) : combine_of<256>(p.by_rows));
    const unsigned rows = static_cast<unsigned>(p.total_q), heads = p.Hq;
    // (a row's heads spread over up to 4096 workgroups: a chunk of 512 rows and one token
    // over 128K keys, in 40 pieces, 313 us with 1024, 170; with 16384 155, but 24 ragged
    // requests of 1876 rows 112 where 4096 takes 109)
    const dim3 grid = p.by_rows ? dim3(rows, std::clamp(4096u / rows, 1u, (heads + 3) / 4)) : dim3(rows * heads);
    hipLaunchKernelGGL(kern, grid, dim3(256), 0, stream, p, kBodyCols[body]);
  }
  return hipGetLastError();
}

}  // namespace mac
