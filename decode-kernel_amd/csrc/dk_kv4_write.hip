// dk_kv4_write.hip — writing and reading the 4-bit cache by token (C ABI in include/dk_decode.h:
// dk_kv4_write, dk_kv4_append, dk_kv4_read). The format is dk_kv4.h's.
//
// Write: each token's K row (rotated) and V row become E2M1 codes and E8M0 scales in the token's
// slot of its page block, and q (optional) is rotated in place. A block of 32 dims with the
// largest magnitude m = f 2^e, 1 <= f < 2, has the scale 2^(e - 2), or 2^(e - 1) where f >= 7/4: then
// m is no further from a code than half a step (E2M1 ends at 6 = 1.5 * 2^2; 7 lies half way to the 8
// that the next scale has). Codes are x / scale rounded to the nearest, ties to the even code. A
// block with a NaN or an infinity gets the NaN scale, so that it reads as NaN.
//
// Rotation as in dk_append_kv (rotate-half pairs or interleaved ones, fp32, one rounding of q), but
// for the angle: position * inv_freq is formed in double and reduced in turns, so that a position of
// 100,000 keeps the fp32 accuracy of a near one (an fp32 product of 1e5 is off by up to 4e-3).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "dk_args.h"
#include "dk_decode.h"
#include "dk_kv4.h"

namespace dk {
namespace {

constexpr int kWriteThreads = 256;
// From this many tokens on a workgroup takes several, fewer than fill the chip take one each.
constexpr int64_t kWriteManyTokens = 4096;
constexpr int kWriteGroupTokens = 4;

struct Kv4WriteArgs {
  uint8_t* q;                 // may be null
  const uint8_t* k_new;
  const uint8_t* v_new;
  uint8_t* cache;
  const void* slots;          // int32 or int64, or null: the page table's last token
  const int32_t* indptr;
  const int32_t* indices;
  const int32_t* last_len;
  const void* positions;      // int32 or int64; null: the token's index in its sequence (table)
  const float* inv_freq;      // null: no rotation
  int64_t q_b, q_h, n_b, n_h, kv_p, kv_h;   // bytes
  int32_t tokens, hq, hkv, rope_style, num_indices;
  int32_t slots64, positions64;
  uint32_t num_pages;
  int32_t per_group;          // tokens per workgroup
};

// (cos, sin) of position * f: whole turns leave in double (exact product, error 2^-52 of the
// turns), then a quarter turn's polynomial: Taylor series to x^11 / x^12 over |x| <= pi/4, off by
// less than 1e-9 before rounding.
__device__ __forceinline__ void cos_sin(double position, float f, float* cs, float* sn) {
  const double turns = position * (double)f * 0.15915494309189535;
  const double part = turns - __builtin_rint(turns);         // in [-1/2, 1/2]
  const double quarter = __builtin_rint(part * 4.0);         // -2 .. 2
  const float x = (float)((part - 0.25 * quarter) * 6.283185307179586);
  const float x2 = x * x;
  float s = -2.5052108e-8f, c = 2.0876757e-9f;               // -1/11!, 1/12!
  s = __builtin_fmaf(s, x2, 2.7557319e-6f);
  s = __builtin_fmaf(s, x2, -1.9841270e-4f);
  s = __builtin_fmaf(s, x2, 8.3333333e-3f);
  s = __builtin_fmaf(s, x2, -1.6666667e-1f);
  s = __builtin_fmaf(s * x2, x, x);
  c = __builtin_fmaf(c, x2, -2.7557319e-7f);
  c = __builtin_fmaf(c, x2, 2.4801587e-5f);
  c = __builtin_fmaf(c, x2, -1.3888889e-3f);
  c = __builtin_fmaf(c, x2, 4.1666667e-2f);
  c = __builtin_fmaf(c, x2, -0.5f);
  c = __builtin_fmaf(c, x2, 1.0f);
  const int n = (int)quarter & 3;
  const float a = n & 1 ? s : c, b = n & 1 ? c : s;          // |cos|, |sin| of the quadrant
  *cs = n == 1 || n == 2 ? -a : a;
  *sn = n >= 2 ? -b : b;
}

template <class E>
using Run8 = E __attribute__((ext_vector_type(8)));

// Largest magnitude of 8 values and those of the 3 neighbouring lanes of the quad (32 dims), as
// float bits (a NaN is larger than an infinity, an infinity than any number)
__device__ __forceinline__ u32 block_top(const float (&x)[8]) {
  u32 m = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __builtin_bit_cast(u32, x[i]) & 0x7fffffffu);
  m = max(m, dpp_u<0xB1>(m));
  return max(m, dpp_u<0x4E>(m));
}
__device__ __forceinline__ u32 block_scale(u32 top) {
  if (top >= 0x7f800000u) return 255u;
  return (u32)min(max((int)((top + 0x200000u) >> 23) - 2, 1), 252);
}
// 8 values as a word of codes
__device__ __forceinline__ u32 codes8(const float (&x)[8], u32 scale) {
  const float sc = __builtin_bit_cast(float, min(scale, 254u) << 23);
  u32 w = 0u;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], sc, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], sc, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], sc, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], sc, 3);
}

// 8 values of dims i .. i+7 of token t's row into the page block
template <int D, bool V>
__device__ __forceinline__ void put8(uint8_t* blk, int t, int i, const float (&x)[8]) {
  const u32 scale = block_scale(block_top(x));
  const u32 w = codes8(x, scale);
  if constexpr (!V) {
    *reinterpret_cast<u32*>(blk + t * (D / 2) + i / 2) = w;
  } else if constexpr (D == 64) {                            // two runs of 4 dims
    uint8_t* p = blk + kv4_v_at(D) + kv4_v_off(D, t, i);
    *reinterpret_cast<uint16_t*>(p) = (uint16_t)w;
    *reinterpret_cast<uint16_t*>(p + 8) = (uint16_t)(w >> 16);
  } else {
    *reinterpret_cast<u32*>(blk + kv4_v_at(D) + kv4_v_off(D, t, i)) = w;
  }
  if ((i & 31) == 0) blk[(V ? kv4_vs_at(D) : kv4_ks_at(D)) + (i >> 5) * 16 + t] = (uint8_t)scale;
}

__device__ __forceinline__ int64_t index_at(const void* p, int32_t wide, int64_t i) {
  return wide ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}

// Workgroup: per_group consecutive tokens (blockIdx.x), slice blockIdx.y of their units. A unit is 8
// + 8 dims of one q or K head (its pairs), or 8 dims of a V head; 4 neighbouring lanes hold a block's
// 32 dims. The tokens' cosines and sines are formed once, in LDS, for all heads. With inv_freq and q null
// the K rows are written as they are.
template <class E, int D>
__global__ __launch_bounds__(kWriteThreads) void dk_kv4_write_kernel(Kv4WriteArgs a) {
  constexpr int HU = D / 16;                                 // units of a q or K head
  constexpr int VU = D / 8;
  extern __shared__ float trig[];                            // per token: D/2 cosines, D/2 sines
  const int t0 = blockIdx.x * a.per_group;
  const int nt = min(a.per_group, a.tokens - t0);
  const bool rot = a.inv_freq != nullptr;
  const int qu = a.q && rot ? a.hq * HU : 0, ku = a.hkv * HU;
  const int units = qu + ku + a.hkv * VU;

  auto where = [&](int t, int* slot, int64_t* pos) -> uint8_t* {
    *slot = 0;
    if (a.slots) {
      const int64_t s = index_at(a.slots, a.slots64, t);
      if (pos) *pos = a.positions ? index_at(a.positions, a.positions64, t) : 0;
      if (s < 0 || s >= (int64_t)a.num_pages * kPage) return nullptr;
      *slot = (int)(s % kPage);
      return a.cache + s / kPage * a.kv_p;
    }
    const int s0 = min(max(a.indptr[t], 0), a.num_indices);
    const int s1 = min(max(a.indptr[t + 1], 0), a.num_indices);
    if (pos) *pos = 0;
    if (s1 <= s0) return nullptr;
    *slot = min(max(a.last_len[t] - 1, 0), kPage - 1);
    if (pos) *pos = a.positions ? index_at(a.positions, a.positions64, t)
                                : (int64_t)(s1 - s0 - 1) * kPage + *slot;
    const u32 page = (u32)a.indices[s1 - 1];
    return page < a.num_pages ? a.cache + (int64_t)page * a.kv_p : nullptr;
  };

  if (rot) {
    for (int i = threadIdx.x; i < nt * (D / 2); i += kWriteThreads) {
      const int t = i / (D / 2), f = i % (D / 2);
      int slot;
      int64_t pos;
      where(t0 + t, &slot, &pos);
      float c, s;
      cos_sin((double)pos, a.inv_freq[f], &c, &s);
      trig[t * D + f] = c;
      trig[t * D + D / 2 + f] = s;
    }
    __syncthreads();
  }
  for (int u = blockIdx.y * kWriteThreads + threadIdx.x; u < nt * units;
       u += gridDim.y * kWriteThreads) {
    const int tl = u / units, t = t0 + tl;
    int x = u - tl * units;
    int slot;
    uint8_t* blk = where(t, &slot, nullptr);
    // a sequence without pages has no token to append: its q row stays (as in dk_append_kv)
    const bool none = !a.slots && a.indptr[t + 1] <= a.indptr[t];
    if (x < qu + ku) {
      const bool is_q = x < qu;
      if (!is_q) x -= qu;
      const int h = x / HU, n = x % HU;                      // head, 8-pair column
      uint8_t* row = is_q ? a.q + (int64_t)t * a.q_b + (int64_t)h * a.q_h
                          : const_cast<uint8_t*>(a.k_new) + (int64_t)t * a.n_b + (int64_t)h * a.n_h;
      // two runs of 8 dims: their pairs lie across them (rotate half) or inside (interleaved)
      const int i0 = 8 * n, i1 = 8 * n + D / 2;
      const Run8<E> lo = *reinterpret_cast<const Run8<E>*>(row + 2 * i0);
      const Run8<E> hi = *reinterpret_cast<const Run8<E>*>(row + 2 * i1);
      float y0[8], y1[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y0[e] = (float)lo[e];
        y1[e] = (float)hi[e];
      }
      if (rot) {
        const float* cs = trig + tl * D;
        const float* sn = cs + D / 2;
        if (a.rope_style == 0) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float c = cs[i0 + e], s = sn[i0 + e], p = y0[e], q = y1[e];
            y0[e] = __builtin_fmaf(p, c, -(q * s));
            y1[e] = __builtin_fmaf(p, s, q * c);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const float c0 = cs[i0 / 2 + e / 2], s0 = sn[i0 / 2 + e / 2];
            const float c1 = cs[i1 / 2 + e / 2], s1 = sn[i1 / 2 + e / 2];
            const float p0 = y0[e], q0 = y0[e + 1], p1 = y1[e], q1 = y1[e + 1];
            y0[e] = __builtin_fmaf(p0, c0, -(q0 * s0));
            y0[e + 1] = __builtin_fmaf(p0, s0, q0 * c0);
            y1[e] = __builtin_fmaf(p1, c1, -(q1 * s1));
            y1[e + 1] = __builtin_fmaf(p1, s1, q1 * c1);
          }
        }
      }
      if (is_q) {
        if (!none) {
          Run8<E> o0, o1;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            o0[e] = (E)y0[e];
            o1[e] = (E)y1[e];
          }
          *reinterpret_cast<Run8<E>*>(row + 2 * i0) = o0;
          *reinterpret_cast<Run8<E>*>(row + 2 * i1) = o1;
        }
      } else if (blk) {                                      // the same for a block's 4 lanes
        put8<D, false>(blk + (int64_t)h * a.kv_h, slot, i0, y0);
        put8<D, false>(blk + (int64_t)h * a.kv_h, slot, i1, y1);
      }
    } else if (blk) {
      x -= qu + ku;
      const int h = x / VU, i = 8 * (x % VU);
      const Run8<E> v = *reinterpret_cast<const Run8<E>*>(a.v_new + (int64_t)t * a.n_b +
                                                          (int64_t)h * a.n_h + 2 * i);
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = (float)v[e];
      put8<D, true>(blk + (int64_t)h * a.kv_h, slot, i, y);
    }
  }
}

struct Kv4ReadArgs {
  const uint8_t* cache;
  const void* slots;
  uint8_t* k;
  uint8_t* v;
  int64_t kv_p, kv_h, o_b, o_h;   // bytes
  int64_t rows;
  int32_t hkv, slots64;
  uint32_t num_pages;
};

// A thread reads 8 dims of a token's K and V rows of one head; a slot outside the pool reads as zeros.
// Bound by memory: 8192 tokens of 8 heads, D = 128, 10.0 us (42 MB, of which 33 written); a row of K
// or V per thread, with 64-bit indexes, 11.5.
template <class T, int D>
__global__ __launch_bounds__(kWriteThreads) void dk_kv4_read_kernel(Kv4ReadArgs a) {
  constexpr int RU = D / 8;
  const int64_t row = (int64_t)blockIdx.x * (kWriteThreads / RU) + threadIdx.x / RU;
  if (row >= a.rows) return;
  const int i = 8 * (int)(threadIdx.x % RU);
  int64_t t;
  int h;
  if (a.rows <= UINT32_MAX) {
    t = (u32)row / (u32)a.hkv;
    h = (int)((u32)row - (u32)t * (u32)a.hkv);
  } else {
    t = row / a.hkv;
    h = (int)(row - t * a.hkv);
  }
  const int64_t s = index_at(a.slots, a.slots64, t);
  u32x4 k = {0u, 0u, 0u, 0u}, v = {0u, 0u, 0u, 0u};
  if (s >= 0 && s < (int64_t)a.num_pages * kPage) {
    const uint8_t* blk = a.cache + (s >> 4) * a.kv_p + (int64_t)h * a.kv_h;
    const int slot = (int)(s & (kPage - 1));
    const u32 kw = *reinterpret_cast<const u32*>(blk + slot * (D / 2) + i / 2);
    u32 vw;
    const uint8_t* p = blk + kv4_v_at(D) + kv4_v_off(D, slot, i);
    if constexpr (D == 64)
      vw = (u32)*reinterpret_cast<const uint16_t*>(p) |
           (u32)*reinterpret_cast<const uint16_t*>(p + 8) << 16;
    else
      vw = *reinterpret_cast<const u32*>(p);
    const u32 ks = (u32)blk[kv4_ks_at(D) + (i >> 5) * 16 + slot] << 23;
    const u32 vs = (u32)blk[kv4_vs_at(D) + (i >> 5) * 16 + slot] << 23;
    k = u32x4{from_fp4<T, 0>(kw, ks), from_fp4<T, 1>(kw, ks), from_fp4<T, 2>(kw, ks),
              from_fp4<T, 3>(kw, ks)};
    v = u32x4{from_fp4<T, 0>(vw, vs), from_fp4<T, 1>(vw, vs), from_fp4<T, 2>(vw, vs),
              from_fp4<T, 3>(vw, vs)};
  }
  const int64_t at = t * a.o_b + (int64_t)h * a.o_h + 2 * i;
  *reinterpret_cast<u32x4*>(a.k + at) = k;
  *reinterpret_cast<u32x4*>(a.v + at) = v;
}

const void* write_symbol(int32_t dtype, int d) {
  const bool f = dtype == DK_F16;
  switch (d) {
    case 64: return f ? (const void*)dk_kv4_write_kernel<_Float16, 64> : (const void*)dk_kv4_write_kernel<__bf16, 64>;
    case 128: return f ? (const void*)dk_kv4_write_kernel<_Float16, 128> : (const void*)dk_kv4_write_kernel<__bf16, 128>;
    default: return f ? (const void*)dk_kv4_write_kernel<_Float16, 256> : (const void*)dk_kv4_write_kernel<__bf16, 256>;
  }
}
const void* read_symbol(int32_t dtype, int d) {
  const bool f = dtype == DK_F16;
  switch (d) {
    case 64: return f ? (const void*)dk_kv4_read_kernel<F16, 64> : (const void*)dk_kv4_read_kernel<BF16, 64>;
    case 128: return f ? (const void*)dk_kv4_read_kernel<F16, 128> : (const void*)dk_kv4_read_kernel<BF16, 128>;
    default: return f ? (const void*)dk_kv4_read_kernel<F16, 256> : (const void*)dk_kv4_read_kernel<BF16, 256>;
  }
}

// Checks shared by the three entry points
int check_sizes(const char* what, int64_t tokens, int32_t hq, int32_t hkv, int32_t d,
                int64_t num_pages, int32_t dtype) {
  if (tokens < 0 || tokens > INT32_MAX || hq <= 0 || hkv <= 0 || num_pages < 0 ||
      (int64_t)hq + 2 * (int64_t)hkv > (1 << 16))
    return set_error(DK_EINVAL, "%s: bad token, head or page count", what);
  if (d != 64 && d != 128 && d != 256)
    return set_error(DK_EINVAL, "head_dim must be 64, 128 or 256; got %d", d);
  if (dtype != DK_F16 && dtype != DK_BF16)
    return set_error(DK_EINVAL, "dtype must be DK_F16 or DK_BF16; got %d", dtype);
  return DK_OK;
}

// 16-byte aligned rows of 16-bit elements below 2^62 bytes
bool rows_ok(const void* p, int64_t tokens, int64_t s_t, int32_t heads, int64_t s_h, int32_t d) {
  return s_t >= 0 && s_h >= 0 && s_t % 8 == 0 && s_h % 8 == 0 && (uintptr_t)p % 16 == 0 &&
         extent_ok(tokens, s_t, heads, s_h, d, 2);
}

int write_impl(const char* what, void* q, const void* k_new, const void* v_new, int64_t new_b,
               int64_t new_h, void* cache, Kv4WriteArgs a, int64_t tokens, int32_t hq, int32_t hkv,
               int32_t d, int64_t num_pages, int32_t dtype, const dk_strides* strides,
               hipStream_t stream) {
  if (!strides) return set_error(DK_ENULL, "strides must be non-NULL");
  if (const int rc = check_sizes(what, tokens, hq, hkv, d, num_pages, dtype)) return rc;
  if (a.rope_style != 0 && a.rope_style != 1)
    return set_error(DK_EINVAL, "rope_style must be 0 (rotate half) or 1 (interleaved)");
  if (tokens == 0) return DK_OK;
  if (!k_new || !v_new || (num_pages > 0 && !cache))
    return set_error(DK_ENULL, "%s: NULL pointer", what);
  const dk_strides& s = *strides;
  if ((q && !rows_ok(q, tokens, s.q_b, hq, s.q_h, d)) ||
      !rows_ok(k_new, tokens, new_b, hkv, new_h, d) || !rows_ok(v_new, tokens, new_b, hkv, new_h, d))
    return set_error(DK_EUNSUPPORTED, "q, k_new and v_new must be 16-byte aligned, with strides that "
                                      "are non-negative multiples of 8 elements");
  if (!kv4_pool_ok(cache, num_pages, s.kv_p, hkv, s.kv_h, d))
    return set_error(DK_EUNSUPPORTED, "the 4-bit cache must be 16-byte aligned, with page and head "
                                      "strides that are non-negative multiples of 16 bytes");
  a.q = static_cast<uint8_t*>(q);
  a.k_new = static_cast<const uint8_t*>(k_new);
  a.v_new = static_cast<const uint8_t*>(v_new);
  a.cache = static_cast<uint8_t*>(cache);
  a.q_b = s.q_b * 2;
  a.q_h = s.q_h * 2;
  a.n_b = new_b * 2;
  a.n_h = new_h * 2;
  a.kv_p = s.kv_p;
  a.kv_h = s.kv_h;
  a.tokens = (int32_t)tokens;
  a.hq = hq;
  a.hkv = hkv;
  a.num_pages = (uint32_t)std::min<int64_t>(num_pages, (int64_t)1 << 31);
  // few tokens: one per workgroup, its units over as many workgroups as they fill; many: several
  // tokens per workgroup
  const int64_t units = (int64_t)(q && a.inv_freq ? hq : 0) * (d / 16) + (int64_t)hkv * (d / 16 + d / 8);
  a.per_group = tokens >= kWriteManyTokens ? kWriteGroupTokens : 1;
  const int64_t groups = (tokens + a.per_group - 1) / a.per_group;
  const int64_t slices = a.per_group > 1 ? 1 : (units + kWriteThreads - 1) / kWriteThreads;
  void* args[] = {&a};
  const hipError_t e = hipLaunchKernel(
      write_symbol(dtype, d), dim3((uint32_t)groups, (uint32_t)std::min<int64_t>(slices, 65535)),
      dim3(kWriteThreads), args, a.inv_freq ? (size_t)a.per_group * d * sizeof(float) : 0, stream);
  if (e != hipSuccess) return set_error((int)e, "%s launch: %s", what, hipGetErrorString(e));
  return DK_OK;
}

}  // namespace
}  // namespace dk

extern "C" int dk_kv4_write(void* q, const void* k_new, const void* v_new, int64_t new_t,
                            int64_t new_h, void* cache, const void* slots, int32_t slots_int64,
                            const void* positions, int32_t positions_int64, const float* inv_freq,
                            int32_t rope_style, int64_t num_tokens, int32_t num_q_heads,
                            int32_t num_kv_heads, int32_t head_dim, int64_t num_pages,
                            int32_t dtype, const dk_strides* strides, void* hip_stream) {
  using namespace dk;
  clear_error();
  if (num_tokens > 0 && (!slots || (inv_freq && !positions)))
    return set_error(DK_ENULL, "dk_kv4_write: slots, and positions with inv_freq, must be non-NULL");
  Kv4WriteArgs a{};
  a.slots = slots;
  a.slots64 = slots_int64 != 0;
  a.positions = positions;
  a.positions64 = positions_int64 != 0;
  a.inv_freq = inv_freq;
  a.rope_style = rope_style;
  return write_impl("dk_kv4_write", q, k_new, v_new, new_t, new_h, cache, a, num_tokens, num_q_heads,
                    num_kv_heads, head_dim, num_pages, dtype, strides,
                    static_cast<hipStream_t>(hip_stream));
}

extern "C" int dk_kv4_append(void* q, const void* k_new, const void* v_new, int64_t new_b,
                             int64_t new_h, void* cache, const int32_t* kv_indptr,
                             const int32_t* kv_indices, const int32_t* kv_last_page_len,
                             const int32_t* positions, const float* inv_freq, int32_t rope_style,
                             int32_t batch, int32_t num_q_heads, int32_t num_kv_heads,
                             int32_t head_dim, int64_t num_pages, int64_t num_indices,
                             int32_t dtype, const dk_strides* strides, void* hip_stream) {
  using namespace dk;
  clear_error();
  if (num_indices < 0 || num_indices > INT32_MAX)
    return set_error(DK_EINVAL, "dk_kv4_append: bad num_indices");
  if (batch > 0 && (!kv_indptr || !kv_last_page_len || (num_indices > 0 && !kv_indices)))
    return set_error(DK_ENULL, "dk_kv4_append: NULL pointer");
  Kv4WriteArgs a{};
  a.indptr = kv_indptr;
  a.indices = kv_indices;
  a.last_len = kv_last_page_len;
  a.num_indices = (int32_t)num_indices;
  a.positions = positions;
  a.inv_freq = inv_freq;
  a.rope_style = rope_style;
  return write_impl("dk_kv4_append", q, k_new, v_new, new_b, new_h, cache, a, batch, num_q_heads,
                    num_kv_heads, head_dim, num_pages, dtype, strides,
                    static_cast<hipStream_t>(hip_stream));
}

extern "C" int dk_kv4_read(const void* cache, int64_t kv_p, int64_t kv_h, const void* slots,
                           int32_t slots_int64, void* k_out, void* v_out, int64_t out_t,
                           int64_t out_h, int64_t num_tokens, int32_t num_kv_heads,
                           int32_t head_dim, int64_t num_pages, int32_t dtype, void* hip_stream) {
  using namespace dk;
  clear_error();
  if (const int rc = check_sizes("dk_kv4_read", num_tokens, 1, num_kv_heads, head_dim, num_pages, dtype))
    return rc;
  if (num_tokens == 0) return DK_OK;
  if (!slots || !k_out || !v_out || (num_pages > 0 && !cache))
    return set_error(DK_ENULL, "dk_kv4_read: NULL pointer");
  if (!rows_ok(k_out, num_tokens, out_t, num_kv_heads, out_h, head_dim) ||
      !rows_ok(v_out, num_tokens, out_t, num_kv_heads, out_h, head_dim))
    return set_error(DK_EUNSUPPORTED, "k_out and v_out must be 16-byte aligned, with strides that are "
                                      "non-negative multiples of 8 elements");
  if (!kv4_pool_ok(cache, num_pages, kv_p, num_kv_heads, kv_h, head_dim))
    return set_error(DK_EUNSUPPORTED, "the 4-bit cache must be 16-byte aligned, with page and head "
                                      "strides that are non-negative multiples of 16 bytes");
  Kv4ReadArgs a{};
  a.cache = static_cast<const uint8_t*>(cache);
  a.slots = slots;
  a.slots64 = slots_int64 != 0;
  a.k = static_cast<uint8_t*>(k_out);
  a.v = static_cast<uint8_t*>(v_out);
  a.kv_p = kv_p;
  a.kv_h = kv_h;
  a.o_b = out_t * 2;
  a.o_h = out_h * 2;
  a.rows = num_tokens * num_kv_heads;
  a.hkv = num_kv_heads;
  a.num_pages = (uint32_t)std::min<int64_t>(num_pages, (int64_t)1 << 31);
  const int64_t rows = kWriteThreads / (head_dim / 8), groups = (a.rows + rows - 1) / rows;
  if (groups > UINT32_MAX / kWriteThreads) return set_error(DK_EUNSUPPORTED, "dk_kv4_read: too many rows");
  void* args[] = {&a};
  const hipError_t e = hipLaunchKernel(read_symbol(dtype, head_dim), dim3((uint32_t)groups),
                                       dim3(kWriteThreads), args, 0,
                                       static_cast<hipStream_t>(hip_stream));
  if (e != hipSuccess) return set_error((int)e, "kv4 read launch: %s", hipGetErrorString(e));
  return DK_OK;
}
