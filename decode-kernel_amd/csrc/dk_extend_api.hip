// dk_extend_api.hip — the extend (prefill) attention's C ABI (include/dk_decode.h:
// dk_extend_attention): argument checks and launches.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

#include "dk_args.h"
#include "dk_decode.h"
#include "dk_extend.h"
#include "dk_extend_kv4.h"
#include "dk_launch.h"

namespace dk {
namespace {

// Workgroups per query tile (kExtendFill): 1 = the keys are not split.
int extend_split(int32_t batch, const int32_t* new_lens, const int32_t* all_lens, int32_t hkv,
                 int32_t group, int32_t window) {
  int64_t groups = 0, keys = 0;
  for (int32_t b = 0; b < batch; ++b) {
    if (new_lens[b] <= 0) continue;
    groups += ((int64_t)new_lens[b] * group + kExtendRows - 1) / kExtendRows * hkv;
    // a tile of 128 rows spans up to 128 / group + 1 positions beyond its window
    const int64_t seen = window > 0 ? (int64_t)window + kExtendRows / group + 1 : INT32_MAX;
    keys = std::max<int64_t>(keys, std::min<int64_t>(all_lens[b], seen));
  }
  if (groups == 0) return 1;
  const int64_t s = std::min<int64_t>(kExtendFill / groups, keys / kExtendSplitKeys);
  return (int)std::min<int64_t>(std::max<int64_t>(s, 1), kExtendMaxSplit);
}

// The same over a 4-bit cache: of the splits up to that one, the one with the least time, its parts
// being the longest query tile's keys (kKv4TileCost per 64 of them, more where two workgroups share a
// CU) and, split, the partials' way through memory and the merge's launch. us, this choice and the one
// above: one request of 512 tokens (32/8/128 fp16) 19.7 and 27.8, of 1024 33.3 and 52.1, (32/8/64)
// 24.6 and 34.7; 64 new of 4064 22.5 both, in one part 99.6; 512 of 2512 51.7 both, in one part 68.3.
int extend_split_kv4(int32_t batch, const int32_t* new_lens, const int32_t* all_lens, int32_t hkv,
                     int32_t group, int32_t head_dim, int32_t window) {
  const int most = extend_split(batch, new_lens, all_lens, hkv, group, window);
  if (most == 1) return 1;
  const double per_tile = head_dim == 64 ? 1.6 : head_dim == 128 ? 2.1 : 4.6;   // us per 64 keys
  const double shared = head_dim == 256 ? 2.0 : 1.5;   // where two workgroups take turns on a CU
  constexpr double kMerge = 4.5, kPartials = 4.0e6;    // us; bytes per us
  int64_t groups = 0, keys = 0, tokens = 0;
  for (int32_t b = 0; b < batch; ++b) {
    if (new_lens[b] <= 0) continue;
    groups += ((int64_t)new_lens[b] * group + kExtendRows - 1) / kExtendRows * hkv;
    const int64_t seen = window > 0 ? (int64_t)window + kExtendRows / group + 1 : INT32_MAX;
    keys = std::max<int64_t>(keys, std::min<int64_t>(all_lens[b], seen));
    tokens += new_lens[b];
  }
  const double tiles = (double)((keys + 63) / 64);
  const double part = (double)tokens * hkv * group * head_dim * 2 * sizeof(float) / kPartials;
  int best = 1;
  double least = 0;
  for (int s = 1; s <= most; ++s) {
    const double turns = groups * s > kExtendFill / 2 ? shared : 1.0;
    const double cost = std::ceil(tiles / s) * per_tile * turns + (s > 1 ? kMerge + part * s : 0.0);
    if (s == 1 || cost < least) {
      least = cost;
      best = s;
    }
  }
  return best;
}

template <class T>
hipError_t merge(const ExtendArgs& a, int64_t tokens, int d, bool keep_nan, hipStream_t stream) {
  MergeArgs m{};
  m.po = a.part_o;
  m.pm = a.part_m;
  m.pl = a.part_l;
  m.out = a.out;
  m.o_b = a.o_b;
  m.o_h = a.o_h;
  m.batch = (int32_t)tokens;
  m.hq = a.hkv * a.group;
  m.split = a.split;
  m.sinks = a.sinks;
  m.keep_nan = keep_nan;
  return launch_merge<T>(m, d, false, stream);
}

// Sizes of each request, in range of the map (rows of `width` entries' tokens) and of q; *first:
// the new tokens in all.
int check_requests(int32_t batch, const int32_t* rows, const int32_t* new_lens,
                   const int32_t* all_lens, int64_t num_rows, int32_t group, int64_t num_tokens,
                   int64_t width, int64_t* first) {
  *first = 0;
  for (int32_t b = 0; b < batch; ++b) {
    if (new_lens[b] < 0 || all_lens[b] < new_lens[b] || all_lens[b] > INT32_MAX - 1024 ||
        (int64_t)new_lens[b] * group > INT32_MAX - 1024)
      return set_error(DK_EINVAL, "request %d: %d new of %d tokens", b, new_lens[b], all_lens[b]);
    if (rows[b] < 0 || rows[b] >= num_rows || all_lens[b] > width)
      return set_error(DK_EINVAL, "request %d: row %d or its length exceeds the map", b, rows[b]);
    *first += new_lens[b];
  }
  if (*first > num_tokens)
    return set_error(DK_EINVAL, "%lld new tokens in q rows for %lld", (long long)*first,
                     (long long)num_tokens);
  return DK_OK;
}

// Deals a call's query tiles (n of them) to `slots` workgroups per kv head, of which `period` start
// on a CU each before the next: the longest tiles first, one per workgroup, then the next to the
// workgroups in reverse, and so on; then the workgroups by their load, every second `period` of
// them reversed, so that a CU's workgroups add up to much the same.
void deal_tiles(ExtendKv4Args& ka, int n, int slots, int period) {
  const ExtendArgs& a = ka.e;
  constexpr int kLevels = 256;
  int32_t load[kKv4ExtendOrder] = {};
  uint16_t work[kKv4ExtendOrder], tile[kKv4ExtendOrder], rank[kKv4ExtendOrder];
  // ranks of `count` items by falling size
  auto sort = [&](const auto* size, int count, int64_t most) {
    int at[kLevels + 1] = {};
    auto level = [&](int i) { return kLevels - 1 - (int)((int64_t)size[i] * (kLevels - 1) / most); };
    for (int i = 0; i < count; ++i) ++at[level(i) + 1];
    for (int i = 0; i < kLevels; ++i) at[i + 1] += at[i];
    for (int i = 0; i < count; ++i) rank[i] = (uint16_t)at[level(i)]++;
  };
  int64_t most = 1;
  for (int r = 0, i = 0; r < a.num_reqs; ++r) {
    const ExtendReq& q = a.req[r];
    const int64_t rows = (int64_t)q.n_new * a.group;
    const int tiles = (int)((rows + kExtendRows - 1) / kExtendRows);
    for (int k = 0; k < tiles; ++k, ++i) {         // a request's n-th tile counts from its end
      const int64_t row0 = (int64_t)(tiles - 1 - k) * kExtendRows;
      const int64_t last = std::min(row0 + kExtendRows, rows) - 1;
      int64_t keys = q.n_all - q.n_new + last / a.group + 1;
      if (a.window > 0) keys = std::min<int64_t>(keys, a.window + kExtendRows / a.group + 1);
      work[i] = (uint16_t)std::min<int64_t>(keys / 32 + 2, 32767);   // and a tile's fixed cost
      tile[i] = (uint16_t)(r * kKv4ExtendOrder + k);
      most = std::max<int64_t>(most, work[i]);
    }
  }
  sort(work, n, most);
  uint16_t owner[kKv4ExtendOrder], next[kKv4ExtendOrder] = {};
  most = 1;
  for (int i = 0; i < n; ++i) {
    const int turn = rank[i] / slots, x = rank[i] % slots;
    owner[i] = (uint16_t)(turn & 1 ? slots - 1 - x : x);
    load[owner[i]] += work[i];
    most = std::max<int64_t>(most, load[owner[i]]);
  }
  sort(load, slots, most);
  for (int i = 0; i < slots; ++i) {
    const int first = rank[i] / period * period, end = std::min(first + period, slots);
    if (rank[i] / period & 1) rank[i] = (uint16_t)(end - 1 - (rank[i] - first));
  }
  for (int i = 0; i <= slots; ++i) ka.start[i] = 0;
  for (int i = 0; i < n; ++i) ++ka.start[rank[owner[i]] + 1];
  for (int i = 0; i < slots; ++i) ka.start[i + 1] += ka.start[i];
  for (int i = 0; i < n; ++i) {
    const int x = rank[owner[i]];
    ka.list[ka.start[x] + next[x]++] = tile[i];
  }
}

// The split of the keys, its workspace and the launches of a call whose arguments are checked;
// first: its new tokens.
int launch_extend(ExtendArgs& a, ExtendKv4Args* kv4, const void* fn, const int32_t* rows, const int32_t* new_lens,
                  const int32_t* all_lens, void* workspace, size_t workspace_bytes, int32_t batch,
                  int64_t first, int32_t head_dim, int32_t dtype, void* hip_stream) {
  // without a workspace for the partials the keys are not split
  a.split = kv4 ? extend_split_kv4(batch, new_lens, all_lens, a.hkv, a.group, head_dim, a.window)
                : extend_split(batch, new_lens, all_lens, a.hkv, a.group, a.window);
  if (a.split > 1) {
    size_t off_o, off_m, off_l, total;
    partials_layout_rows(first * (a.hkv * a.group) * a.split, head_dim, &off_o, &off_m, &off_l, &total);
    if (!workspace || workspace_bytes < total || (uintptr_t)workspace % 256 != 0) {
      a.split = 1;
    } else {
      uint8_t* ws = static_cast<uint8_t*>(workspace);
      a.part_o = reinterpret_cast<float*>(ws + off_o);
      a.part_m = reinterpret_cast<float*>(ws + off_m);
      a.part_l = reinterpret_cast<float*>(ws + off_l);
    }
  }
  // kExtendMaxReqs requests per launch: their sizes travel as kernel arguments, so a call
  // copies nothing to the device
  int32_t b = 0;
  int64_t q0 = 0;
  while (b < batch) {
    int32_t n = 0;
    int64_t tiles = 0;
    for (; b < batch && n < kExtendMaxReqs; ++b) {
      if (new_lens[b] == 0) continue;
      const int64_t t = ((int64_t)new_lens[b] * a.group + kExtendRows - 1) / kExtendRows;
      if ((tiles + t) * a.hkv > INT32_MAX) {
        if (n == 0) return set_error(DK_EUNSUPPORTED, "request %d has too many new tokens", b);
        break;
      }
      a.req[n++] = ExtendReq{rows[b], (int32_t)q0, new_lens[b], all_lens[b], (int32_t)tiles};
      tiles += t;
      q0 += new_lens[b];
    }
    if (n == 0) break;
    a.num_reqs = n;
    a.tiles = (int32_t)tiles;
    int64_t slots = tiles;
    if (kv4) {
      const int period = std::max(256 / a.hkv, 1);
      kv4->dealt = a.split == 1 && tiles <= kKv4ExtendOrder;
      if (kv4->dealt) {
        slots = std::min<int64_t>(tiles, kv4_extend_resident(head_dim, a.cap_out != 0.f) * period);
        deal_tiles(*kv4, (int)tiles, (int)slots, period);
      }
    }
    void* args[] = {kv4 ? (void*)kv4 : (void*)&a};
    const hipError_t e =
        hipLaunchKernel(fn, dim3((uint32_t)(slots * a.hkv), a.split), dim3(kExtendThreads), args, 0,
                        static_cast<hipStream_t>(hip_stream));
    if (e != hipSuccess) return set_error((int)e, "extend launch: %s", hipGetErrorString(e));
  }
  if (a.split > 1) {
    const hipStream_t st = static_cast<hipStream_t>(hip_stream);
    const hipError_t e =
        dtype == DK_BF16 ? merge<BF16>(a, first, head_dim, kv4 != nullptr, st)
                         : merge<F16>(a, first, head_dim, kv4 != nullptr, st);
    if (e != hipSuccess) return set_error((int)e, "extend merge launch: %s", hipGetErrorString(e));
  }
  return DK_OK;
}

}  // namespace
}  // namespace dk

namespace {
size_t extend_workspace(int32_t batch, const int32_t* new_lens, const int32_t* all_lens,
                        int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t window,
                        bool kv4) {
  using namespace dk;
  if (batch <= 0 || !new_lens || !all_lens || num_q_heads <= 0 || num_kv_heads <= 0 ||
      num_q_heads % num_kv_heads != 0 || head_dim <= 0 || window < 0)
    return 0;
  const int32_t group = num_q_heads / num_kv_heads;
  const int s = kv4 ? extend_split_kv4(batch, new_lens, all_lens, num_kv_heads, group, head_dim, window)
                    : extend_split(batch, new_lens, all_lens, num_kv_heads, group, window);
  if (s == 1) return 0;
  int64_t tokens = 0;
  for (int32_t b = 0; b < batch; ++b) tokens += std::max(new_lens[b], 0);
  size_t o, m, l, total;
  partials_layout_rows(tokens * num_q_heads * s, head_dim, &o, &m, &l, &total);
  return total;
}
}  // namespace

extern "C" size_t dk_extend_workspace_bytes(int32_t batch, const int32_t* new_lens,
                                            const int32_t* all_lens, int32_t num_q_heads,
                                            int32_t num_kv_heads, int32_t head_dim,
                                            int32_t window) {
  return extend_workspace(batch, new_lens, all_lens, num_q_heads, num_kv_heads, head_dim, window, false);
}

extern "C" size_t dk_extend_kv4_workspace_bytes(int32_t batch, const int32_t* new_lens,
                                                const int32_t* all_lens, int32_t num_q_heads,
                                                int32_t num_kv_heads, int32_t head_dim,
                                                int32_t window) {
  return extend_workspace(batch, new_lens, all_lens, num_q_heads, num_kv_heads, head_dim, window, true);
}

extern "C" int dk_extend_attention(
    const void* q, const void* k_pool, const void* v_pool, const int32_t* req_to_token,
    int64_t req_stride, int64_t num_rows, const int32_t* rows, const int32_t* new_lens,
    const int32_t* all_lens, void* out, void* workspace, size_t workspace_bytes, int32_t batch,
    int64_t num_tokens, int32_t num_q_heads,
    int32_t num_kv_heads, int32_t head_dim, int64_t num_slots, int32_t dtype, int32_t kv_dtype,
    const dk_extend_strides* strides, float score_scale, float v_scale, float logit_cap,
    int32_t window, const float* sinks, void* hip_stream) {
  using namespace dk;
  clear_error();
  if (!strides) return set_error(DK_ENULL, "strides must be non-NULL");
  if (batch < 0 || num_tokens < 0 || num_tokens > INT32_MAX || num_q_heads <= 0 ||
      num_kv_heads <= 0 || num_q_heads % num_kv_heads != 0 || window < 0 || num_rows < 0 ||
      num_rows > INT32_MAX || num_slots < 0 || num_slots > INT32_MAX || req_stride < 0 ||
      req_stride >= kMaxStride)
    return set_error(DK_EINVAL, "dk_extend_attention: bad sizes");
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return set_error(DK_EINVAL, "head_dim must be 64, 128 or 256; got %d", head_dim);
  if (dtype != DK_F16 && dtype != DK_BF16)
    return set_error(DK_EINVAL, "dtype must be DK_F16 or DK_BF16; got %d", dtype);
  if (kv_dtype != DK_KV_SAME && kv_dtype != DK_KV_FP8_E4M3)
    return set_error(DK_EINVAL, "kv_dtype must be DK_KV_SAME or DK_KV_FP8_E4M3");
  if (!std::isfinite(score_scale) || !(score_scale > 0.f) || !std::isfinite(v_scale) ||
      !std::isfinite(logit_cap))
    return set_error(DK_EINVAL, "score_scale must be finite and > 0, v_scale and logit_cap finite");
  if (batch == 0) return DK_OK;
  if (!rows || !new_lens || !all_lens)
    return set_error(DK_ENULL, "dk_extend_attention: NULL pointer");
  const int64_t kes = kv_dtype == DK_KV_FP8_E4M3 ? 1 : 2;
  const dk_extend_strides& s = *strides;
  if (!extent_ok(num_tokens, s.q_b, num_q_heads, s.q_h, head_dim, 2) ||
      !extent_ok(num_tokens, s.o_b, num_q_heads, s.o_h, head_dim, 2) ||
      !extent_ok(num_slots, s.k_s, num_kv_heads, s.k_h, head_dim, kes) ||
      !extent_ok(num_slots, s.v_s, num_kv_heads, s.v_h, head_dim, kes))
    return set_error(DK_EUNSUPPORTED, "strides must be non-negative and below 2^40 elements");
  for (int64_t b : {s.q_b * 2, s.q_h * 2, s.o_b * 2, s.o_h * 2, s.k_s * kes, s.k_h * kes,
                    s.v_s * kes, s.v_h * kes, (int64_t)((uintptr_t)q % 16),
                    (int64_t)((uintptr_t)out % 16), (int64_t)((uintptr_t)k_pool % 16),
                    (int64_t)((uintptr_t)v_pool % 16)})
    if (b % 16 != 0)
      return set_error(DK_EUNSUPPORTED, "q, out and the pools must be 16-byte aligned, and "
                                        "their strides multiples of 16 bytes");
  if (s.k_s * kes > INT32_MAX || s.v_s * kes > INT32_MAX)
    return set_error(DK_EUNSUPPORTED, "pool slots must be less than 2^31 bytes apart");
  const int32_t group = num_q_heads / num_kv_heads;
  int64_t first = 0;
  if (const int rc = check_requests(batch, rows, new_lens, all_lens, num_rows, group, num_tokens,
                                    num_rows > 1 ? req_stride : INT32_MAX, &first))
    return rc;
  if (first == 0) return DK_OK;
  if (!q || !k_pool || !v_pool || !req_to_token || !out)
    return set_error(DK_ENULL, "dk_extend_attention: NULL pointer");
  if (num_slots == 0) return set_error(DK_EINVAL, "the token pool is empty");

  ExtendArgs a{};
  a.q = static_cast<const uint8_t*>(q);
  a.k = static_cast<const uint8_t*>(k_pool);
  a.v = static_cast<const uint8_t*>(v_pool);
  a.req_to_token = req_to_token;
  a.out = static_cast<uint8_t*>(out);
  a.sinks = sinks;
  a.q_b = s.q_b * 2;
  a.q_h = s.q_h * 2;
  a.o_b = s.o_b * 2;
  a.o_h = s.o_h * 2;
  a.k_s = (uint32_t)(s.k_s * kes);
  a.k_h = s.k_h * kes;
  a.v_s = (uint32_t)(s.v_s * kes);
  a.v_h = s.v_h * kes;
  a.req_stride = req_stride;
  a.group = group;
  a.hkv = num_kv_heads;
  a.window = window;
  a.num_slots = (uint32_t)num_slots;
  a.kscale = kLog2e * score_scale;
  a.cap_in = logit_cap != 0.f ? score_scale / logit_cap : 0.f;
  a.cap_out = kLog2e * logit_cap;
  a.vscale = v_scale;
  const bool bf16 = dtype == DK_BF16, kv8 = kes == 1, cap = logit_cap != 0.f;
  const void* fn = head_dim == 64    ? extend_symbol<64>(bf16, kv8, cap)
                   : head_dim == 128 ? extend_symbol<128>(bf16, kv8, cap)
                                     : extend_symbol<256>(bf16, kv8, cap);
  return launch_extend(a, nullptr, fn, rows, new_lens, all_lens, workspace, workspace_bytes, batch,
                       first, head_dim, dtype, hip_stream);
}

extern "C" int dk_extend_attention_kv4(
    const void* q, const void* cache, int64_t kv_p, int64_t kv_h, const int32_t* block_table,
    int64_t table_stride, int64_t num_rows, int32_t max_blocks, const int32_t* rows,
    const int32_t* new_lens, const int32_t* all_lens, void* out, void* workspace,
    size_t workspace_bytes, int32_t batch, int64_t num_tokens, int32_t num_q_heads,
    int32_t num_kv_heads, int32_t head_dim, int64_t num_pages, int32_t dtype,
    const dk_extend_strides* strides, float score_scale, float logit_cap, int32_t window,
    const float* sinks, void* hip_stream) {
  using namespace dk;
  clear_error();
  if (!strides) return set_error(DK_ENULL, "strides must be non-NULL");
  if (batch < 0 || num_tokens < 0 || num_tokens > INT32_MAX || num_q_heads <= 0 ||
      num_kv_heads <= 0 || num_q_heads % num_kv_heads != 0 || window < 0 || num_rows < 0 ||
      num_rows > INT32_MAX || num_pages < 0 || num_pages > INT32_MAX || table_stride < 0 ||
      table_stride >= kMaxStride || max_blocks < 0 || (num_rows > 1 && max_blocks > table_stride))
    return set_error(DK_EINVAL, "dk_extend_attention_kv4: bad sizes");
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return set_error(DK_EINVAL, "head_dim must be 64, 128 or 256; got %d", head_dim);
  if (dtype != DK_F16 && dtype != DK_BF16)
    return set_error(DK_EINVAL, "dtype must be DK_F16 or DK_BF16; got %d", dtype);
  if (!std::isfinite(score_scale) || !(score_scale > 0.f) || !std::isfinite(logit_cap))
    return set_error(DK_EINVAL, "score_scale must be finite and > 0, logit_cap finite");
  if (batch == 0) return DK_OK;
  if (!rows || !new_lens || !all_lens)
    return set_error(DK_ENULL, "dk_extend_attention_kv4: NULL pointer");
  const dk_extend_strides& s = *strides;
  if (!extent_ok(num_tokens, s.q_b, num_q_heads, s.q_h, head_dim, 2) ||
      !extent_ok(num_tokens, s.o_b, num_q_heads, s.o_h, head_dim, 2))
    return set_error(DK_EUNSUPPORTED, "strides must be non-negative and below 2^40 elements");
  for (int64_t b : {s.q_b, s.q_h, s.o_b, s.o_h, (int64_t)((uintptr_t)q % 16) / 2,
                    (int64_t)((uintptr_t)out % 16) / 2})
    if (b % 8 != 0 || (uintptr_t)q % 2 || (uintptr_t)out % 2)
      return set_error(DK_EUNSUPPORTED, "q and out must be 16-byte aligned, and their strides "
                                        "multiples of 16 bytes");
  if (!kv4_pool_ok(cache, num_pages, kv_p, num_kv_heads, kv_h, head_dim))
    return set_error(DK_EUNSUPPORTED, "the 4-bit cache must be 16-byte aligned, with page and head "
                                      "strides that are non-negative multiples of 16 bytes");
  if (!rows_apart(num_tokens, s.o_b, num_q_heads, s.o_h, head_dim))
    return set_error(DK_EUNSUPPORTED, "the rows of out overlap");
  const int32_t group = num_q_heads / num_kv_heads;
  int64_t first = 0;
  if (const int rc = check_requests(batch, rows, new_lens, all_lens, num_rows, group, num_tokens,
                                    (int64_t)max_blocks * kPageSize, &first))
    return rc;
  if (first == 0) return DK_OK;
  if (!q || !cache || !block_table || !out)
    return set_error(DK_ENULL, "dk_extend_attention_kv4: NULL pointer");
  if (num_pages == 0) return set_error(DK_EINVAL, "the page pool is empty");

  ExtendKv4Args ka{};
  ExtendArgs& a = ka.e;
  a.q = static_cast<const uint8_t*>(q);
  a.k = static_cast<const uint8_t*>(cache);
  a.req_to_token = block_table;
  a.out = static_cast<uint8_t*>(out);
  a.sinks = sinks;
  a.q_b = s.q_b * 2;
  a.q_h = s.q_h * 2;
  a.o_b = s.o_b * 2;
  a.o_h = s.o_h * 2;
  a.k_h = kv_h;
  ka.kv_p = kv_p;
  a.req_stride = table_stride;
  a.group = group;
  a.hkv = num_kv_heads;
  a.window = window;
  a.num_slots = (uint32_t)num_pages;
  const bool bf16 = dtype == DK_BF16, cap = logit_cap != 0.f;
  const float stage = (float)(1 << (bf16 ? kv4_stage_exp<BF16>() : kv4_stage_exp<F16>()));
  a.kscale = kLog2e * score_scale;
  a.cap_in = cap ? score_scale / logit_cap : 0.f;
  a.cap_out = kLog2e * logit_cap;
  a.vscale = stage;
  const void* fn = head_dim == 64    ? extend_kv4_symbol<64>(bf16, cap)
                   : head_dim == 128 ? extend_kv4_symbol<128>(bf16, cap)
                                     : extend_kv4_symbol<256>(bf16, cap);
  return launch_extend(a, &ka, fn, rows, new_lens, all_lens, workspace, workspace_bytes, batch, first,
                       head_dim, dtype, hip_stream);
}
