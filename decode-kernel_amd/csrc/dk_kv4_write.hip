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
// Rotation as in dk_append_kv (rotate-half pairs or interleaved ones, one rounding of q), but for the
// angle: position * inv_freq is formed and reduced in double, so that a position of 100,000 keeps the
// accuracy of a near one (an fp32 product of 1e5 is off by up to 4e-3). q is rotated in fp32, K in
// double: an fp32 rotation puts about one K element of 8 million on the other side of a boundary
// between two codes, a whole step of E2M1 away. Bound by memory: 8192 tokens of 32/8/128 40.8 us (176
// MB, 4.3 TB/s, where a large copy reaches 4.9), with K in fp32 too 38.5.
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
// From this many tokens on a workgroup takes several (its angles serve more rows and its loads overlap:
// 8192 tokens of 32/8/128, us, 2 / 4 / 8 tokens 44.3 / 41.4 / 40.8; 16384 of 32/8/64 54.4 / 49.0 / 46.3);
// fewer take one each, their rows over as many workgroups as they fill.
constexpr int64_t kWriteManyTokens = 8192;
constexpr int kWriteGroupTokens = 8;

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

// (cos, sin) of position * f in double: the product is exact, quarter turns leave it in two parts of
// pi / 2 (the second what the first lacks of it), then the Taylor series to x^16 / x^17 over
// |x| <= pi / 4, off by less than 1e-16.
__device__ __forceinline__ void cos_sin(double position, float f, double* cs, double* sn) {
  const double angle = position * (double)f;
  const double quarter = __builtin_rint(angle * 0.6366197723675814);   // 2 / pi
  const double x = __builtin_fma(-quarter, 6.123233995736766e-17,
                                 __builtin_fma(-quarter, 1.5707963267948966, angle));
  const double x2 = x * x;
  double s = 2.8114572543455206e-15, c = 4.779477332387385e-14;        // 1/17!, 1/16!
  s = __builtin_fma(s, x2, -7.647163731819816e-13);
  s = __builtin_fma(s, x2, 1.6059043836821613e-10);
  s = __builtin_fma(s, x2, -2.505210838544172e-08);
  s = __builtin_fma(s, x2, 2.7557319223985893e-06);
  s = __builtin_fma(s, x2, -1.984126984126984e-04);
  s = __builtin_fma(s, x2, 8.333333333333333e-03);
  s = __builtin_fma(s, x2, -1.6666666666666666e-01);
  s = __builtin_fma(s * x2, x, x);
  c = __builtin_fma(c, x2, -1.1470745597729725e-11);
  c = __builtin_fma(c, x2, 2.08767569878681e-09);
  c = __builtin_fma(c, x2, -2.755731922398589e-07);
  c = __builtin_fma(c, x2, 2.48015873015873e-05);
  c = __builtin_fma(c, x2, -1.388888888888889e-03);
  c = __builtin_fma(c, x2, 4.1666666666666664e-02);
  c = __builtin_fma(c, x2, -0.5);
  c = __builtin_fma(c, x2, 1.0);
  const int n = (int)((int64_t)quarter & 3);
  const double a = n & 1 ? s : c, b = n & 1 ? c : s;         // |cos|, |sin| of the quadrant
  *cs = n == 1 || n == 2 ? -a : a;
  *sn = n >= 2 ? -b : b;
}

// y in fp32 such that a rounding to fewer bits gives what it gives for y: cut towards zero, the last
// bit set where something was cut (NaN and infinities stay)
__device__ __forceinline__ float to_odd(double y) {
  const float f = (float)y;
  const double back = f;
  u32 b = __builtin_bit_cast(u32, f);
  b -= __builtin_fabs(back) > __builtin_fabs(y) ? 1u : 0u;
  b |= back != y ? 1u : 0u;
  return __builtin_bit_cast(float, b);
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

// turn(f, p, q, &u, &v) for the pairs (p, q) of two runs of 8 dims from i0 and i1: across them (style
// 0), or neighbours within each; f: the pair's frequency
template <class F>
__device__ __forceinline__ void turn_pairs(int style, int i0, int i1, float (&y0)[8], float (&y1)[8],
                                           F&& turn) {
  if (style == 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      turn(i0 + e, y0[e], y1[e], &y0[e], &y1[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      turn(i0 / 2 + e / 2, y0[e], y0[e + 1], &y0[e], &y0[e + 1]);
      turn(i1 / 2 + e / 2, y1[e], y1[e + 1], &y1[e], &y1[e + 1]);
    }
  }
}

// Workgroup: per_group consecutive tokens (blockIdx.x), slice blockIdx.y of their units. A unit is 8
// + 8 dims of one head's row (a rotated one's pairs); 4 neighbouring lanes hold a block's 32 dims. The
// tokens' cosines and sines are formed once, in LDS, for all heads. Without inv_freq q is left alone
// and K is written as it is.
template <class E, int D>
__global__ __launch_bounds__(kWriteThreads) void dk_kv4_write_kernel(Kv4WriteArgs a) {
  constexpr int HU = D / 16;                                 // units of a q or K head
  extern __shared__ __attribute__((aligned(8))) float trig[];   // per token: D/2 cosines, D/2 sines;
  double* const trig64 = reinterpret_cast<double*>(trig + a.per_group * D);   // the same in double
  const int t0 = blockIdx.x * a.per_group;
  const int nt = min(a.per_group, a.tokens - t0);
  const bool rot = a.inv_freq != nullptr;
  const int qu = a.q && rot ? a.hq * HU : 0, ku = a.hkv * HU;
  const int units = qu + 2 * ku;

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

  // two runs of 8 dims of a row: rotated pairs lie across them (rotate half) or inside (interleaved)
  struct Unit {
    int t, x;                                                // token of the group, unit of the token
    Run8<E> lo, hi;
  };
  auto row_of = [&](const Unit& u) -> uint8_t* {
    const int h = (u.x < qu ? u.x : u.x < qu + ku ? u.x - qu : u.x - qu - ku) / HU;
    const int64_t t = t0 + u.t;
    if (u.x < qu) return a.q + t * a.q_b + (int64_t)h * a.q_h;
    return const_cast<uint8_t*>(u.x < qu + ku ? a.k_new : a.v_new) + t * a.n_b + (int64_t)h * a.n_h;
  };
  auto fetch = [&](int at, Unit& u) {
    u.t = at / units;
    u.x = at - u.t * units;
    const uint8_t* row = row_of(u) + 16 * (u.x % HU);        // qu and ku are multiples of HU
    u.lo = *reinterpret_cast<const Run8<E>*>(row);
    u.hi = *reinterpret_cast<const Run8<E>*>(row + D);
  };
  Unit u0, u1;
  const int first = blockIdx.y * kWriteThreads + threadIdx.x;
  if (first < nt * units) fetch(first, u0);                  // in flight while the angles are formed
  if (rot) {
    for (int i = threadIdx.x; i < nt * (D / 2); i += kWriteThreads) {
      const int t = i / (D / 2), f = i % (D / 2);
      int slot;
      int64_t pos;
      where(t0 + t, &slot, &pos);
      double c, s;
      cos_sin((double)pos, a.inv_freq[f], &c, &s);
      trig[t * D + f] = (float)c;
      trig[t * D + D / 2 + f] = (float)s;
      trig64[t * D + f] = c;
      trig64[t * D + D / 2 + f] = s;
    }
    __syncthreads();
  }
  auto put = [&](const Unit& u) {
    const int t = t0 + u.t, x = u.x, n = x % HU;
    const int i0 = 8 * n, i1 = 8 * n + D / 2;
    const bool is_q = x < qu, is_k = !is_q && x < qu + ku;
    int slot;
    uint8_t* blk = where(t, &slot, nullptr);
    // a sequence without pages has no token to append: its q row stays (as in dk_append_kv)
    if (is_q ? !a.slots && a.indptr[t + 1] <= a.indptr[t] : !blk) return;
    const int tl = u.t;
    const Run8<E> &lo = u.lo, &hi = u.hi;
    float y0[8], y1[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y0[e] = (float)lo[e];
      y1[e] = (float)hi[e];
    }
    if (rot && is_q) {
      const float *cs = trig + tl * D, *sn = cs + D / 2;
      turn_pairs(a.rope_style, i0, i1, y0, y1, [&](int f, float p, float q, float* u, float* v) {
        *u = __builtin_fmaf(p, cs[f], -(q * sn[f]));
        *v = __builtin_fmaf(p, sn[f], q * cs[f]);
      });
    } else if (rot && is_k) {
      const double *cs = trig64 + tl * D, *sn = cs + D / 2;
      turn_pairs(a.rope_style, i0, i1, y0, y1, [&](int f, double p, double q, float* u, float* v) {
        *u = (float)(p * cs[f] - q * sn[f]);
        *v = (float)(p * sn[f] + q * cs[f]);
      });
      // every boundary between codes, and between scales, is a float of at most 2 mantissa bits: only
      // one that came out as such may lie on its other side
      u32 low = ~0u;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        low = min(low, min(__builtin_bit_cast(u32, y0[e]) & 0x1fffffu,
                           __builtin_bit_cast(u32, y1[e]) & 0x1fffffu));
      if (__builtin_amdgcn_ballot_w64(low == 0u)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          y0[e] = (float)lo[e];
          y1[e] = (float)hi[e];
        }
        turn_pairs(a.rope_style, i0, i1, y0, y1, [&](int f, double p, double q, float* u, float* v) {
          *u = to_odd(p * cs[f] - q * sn[f]);
          *v = to_odd(p * sn[f] + q * cs[f]);
        });
      }
    }
    if (is_q) {
      Run8<E> o0, o1;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        o0[e] = (E)y0[e];
        o1[e] = (E)y1[e];
      }
      uint8_t* row = row_of(u);
      *reinterpret_cast<Run8<E>*>(row + 2 * i0) = o0;
      *reinterpret_cast<Run8<E>*>(row + 2 * i1) = o1;
    } else if (is_k) {                                       // the same for a block's 4 lanes
      blk += (int64_t)((x - qu) / HU) * a.kv_h;
      put8<D, false>(blk, slot, i0, y0);
      put8<D, false>(blk, slot, i1, y1);
    } else {
      blk += (int64_t)((x - qu - ku) / HU) * a.kv_h;
      put8<D, true>(blk, slot, i0, y0);
      put8<D, true>(blk, slot, i1, y1);
    }
  };
  // the next unit's rows are in flight while one is put
  const int step = gridDim.y * kWriteThreads, all = nt * units;
  for (int at = first; at < all; at += 2 * step) {
    if (at + step < all) fetch(at + step, u1);
    put(u0);
    if (at + 2 * step < all) fetch(at + 2 * step, u0);
    if (at + step < all) put(u1);
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
  if ((q && a.inv_freq && !rows_apart(tokens, s.q_b, hq, s.q_h, d)) ||
      !rows_apart(num_pages, s.kv_p, hkv, s.kv_h, 17 * d))
    return set_error(DK_EUNSUPPORTED, "%s: rows of q, or blocks of the cache, overlap", what);
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
  const int64_t units = ((int64_t)(q && a.inv_freq ? hq : 0) + 2 * (int64_t)hkv) * (d / 16);
  a.per_group = tokens >= kWriteManyTokens ? kWriteGroupTokens : 1;
  const int64_t groups = (tokens + a.per_group - 1) / a.per_group;
  const int64_t slices = a.per_group > 1 ? 1 : (units + kWriteThreads - 1) / kWriteThreads;
  void* args[] = {&a};
  const hipError_t e = hipLaunchKernel(
      write_symbol(dtype, d), dim3((uint32_t)groups, (uint32_t)std::min<int64_t>(slices, 65535)),
      dim3(kWriteThreads), args, a.inv_freq ? (size_t)a.per_group * d * (sizeof(float) + sizeof(double)) : 0, stream);
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
  if (!rows_apart(num_tokens, out_t, num_kv_heads, out_h, head_dim))
    return set_error(DK_EUNSUPPORTED, "dk_kv4_read: the rows of k_out and v_out overlap");
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
