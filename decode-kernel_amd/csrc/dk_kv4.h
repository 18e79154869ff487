// dk_kv4.h — the 4-bit paged cache (OCP MXFP4) and decode attention over it (gfx950, wave64).
//
// A page block holds one kv head's 16 tokens in 17 * D bytes: the K codes, the V codes, the K
// scales and the V scales. Codes are E2M1 (two per byte, the even dim in the low nibble), scales
// E8M0, one per 32 dims of a row. Every part lies as the kernels' lanes load it, so that a page
// block is read by whole-line loads whatever the other heads hold:
//   * K codes row by row: lane (r, c) of a wavefront (r = lane / 16, c = lane % 16) takes token
//     c's block r, 16 bytes, the fp4 operand of v_mfma_scale_f32_16x16x128_f8f6f4;
//   * V codes in runs of 4 tokens x W / 16 dims (W = min(D, 128)): lane (r, c) takes tokens
//     4r .. 4r+3, dims c * W / 16 .., as one load;
//   * scales block by block, 16 tokens each: a lane's K scale is a byte, its 4 V scales a word.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dk_kernels.h"

namespace dk {

constexpr int kv4_bytes(int d) { return 17 * d; }          // of a page block
constexpr int kv4_v_at(int d) { return 8 * d; }            // V codes
constexpr int kv4_ks_at(int d) { return 16 * d; }          // K scales
constexpr int kv4_vs_at(int d) { return 16 * d + d / 2; }  // V scales
// Bytes from the V codes' start to the run of token t (its 4-token group) that holds dim i, i a
// multiple of W / 16 or inside the run
__device__ __forceinline__ int kv4_v_off(int d, int t, int i) {
  const int w = d < 128 ? d : 128, s = i / w, j = i - s * w, run = w / 16;
  return s * 8 * w + (t >> 2) * 2 * w + j / run * (w / 8) + (t & 3) * (w / 32) + j % run / 2;
}

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef short i16x2 __attribute__((ext_vector_type(2)));

// C += A.B: A 16 tokens x 128 dims of E2M1 (16 bytes per lane), B 128 dims x 16 columns of E4M3
// (32 bytes per lane). sa / sb: E8M0 scales of the lane's row / column and 32-dim block (byte
// GB of sb). The lanes' k index: fp4 lane r holds k = 32 r .. 32 r + 31; fp8 lane r holds k =
// 16 r .. 16 r + 15 and 64 + 16 r .. 64 + 16 r + 15.
template <int GB>
__device__ __forceinline__ f32x4 mfma_mx(u32x4 a, i32x8 b, f32x4 c, u32 sa, u32 sb) {
  const i32x8 av = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, b, c, 4, 0, 0, (int)sa, GB, (int)sb);
}

// bf16 pair (dims 2B, 2B+1 of the word's 8) of E2M1 codes times the scale whose exponent field
// `sc` holds (sign and mantissa are not read; all ones gives NaN)
template <int B>
__device__ __forceinline__ u32 fp4_bf16(u32 w, u32 sc) {
  return __builtin_bit_cast(
      u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, __builtin_bit_cast(float, sc), B));
}

// The same pair in T (fp16: values beyond its range become infinities)
template <class T, int B>
__device__ __forceinline__ u32 from_fp4(u32 w, u32 sc) {
  if constexpr (__is_same(T, F16))
    return __builtin_bit_cast(
        u32, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, __builtin_bit_cast(float, sc), B));
  else
    return fp4_bf16<B>(w, sc);
}

// E8M0 byte B of w moved to a float's exponent field (other bits arbitrary)
template <int B>
__device__ __forceinline__ u32 e8m0_exp(u32 w) {
  if constexpr (B == 3) return w >> 1;
  else return w << (23 - 8 * B);
}

// q enters the MX products as QParts parts of E4M3, each with a power-of-two scale per 32-dim
// block. v_mfma_scale adds the products of a group of dims in a window of 13 bits below the
// largest (measured: next to 2^8, 2^-5 counts and 2^-6 is lost). So the first part is a fixed-point
// digit, whose products fill at most 8 bits and add up exactly: q to the nearest multiple of 1/16
// of the power of two above the block's largest magnitude. The others are the remainder's leading 4
// bits each time, with the sign of the next remainder 9 bits (bf16, 2 parts) or 13 (fp16, 3), so
// that q's own 8 or 11 bits are held wherever it lies, and what the window drops is below 2^-18 of a
// product of the largest magnitudes.
template <class T>
struct QParts {
  static constexpr int n = 3;
};
template <>
struct QParts<F16> {
  static constexpr int n = 4;
};
// Part i's scale exponent below the block's largest exponent
__device__ __forceinline__ constexpr int q_part_exp(int i) { return i == 0 ? 3 : 8 + 4 * i; }

// Max over the lanes that hold one q head of HP (columns agreeing modulo HP)
template <int HP>
__device__ __forceinline__ float max_head(float x) {
  if constexpr (HP <= 4) x = fmaxf(x, row_ror<4>(x));
  if constexpr (HP <= 8) x = fmaxf(x, row_ror<8>(x));
  return max_xor32(max_xor16(x));
}
template <int HP>
__device__ __forceinline__ float sum_head(float x) {
  if constexpr (HP <= 4) x += row_ror<4>(x);
  if constexpr (HP <= 8) x += row_ror<8>(x);
  return sum_xor32(sum_xor16(x));
}

// One wavefront over pages of one kv head, kStep at a time, for up to HP (4, 8 or 16) q heads.
//   * q.k: K's codes and scales are MFMA operands as they lie; q enters as E4M3 parts with
//     scales of its own, one MFMA each. The 16 columns are HP heads x U = 16 / HP pages: for a
//     page's MFMAs the scale of every other page's columns is 0 (2^-127), so U pages accumulate
//     into one set of scores and every lane's 4 scores count: lane (r, c) holds tokens
//     4r .. 4r+3 of page c / HP of the set, head c % HP.
//   * softmax as in Wave: fp32, log2 domain, a reference that moves by more than 2^8 only.
//   * P.V in bf16, whatever q's type: E2M1 times a power of two is exact there, and p as hi + lo
//     parts keeps 16 bits at any magnitude. v_mfma_f32_16x16x32 over two pages: a lane's V words
//     widened with their scales (v_cvt_scalef32_pk_bf16_fp4) and paired by token (v_perm). Rows
//     are the heads again, so for HP < 16 hi and lo share one MFMA, lo in rows of its own.
template <class T, int D, int HP, bool CAP>
struct Kv4Wave {
  static constexpr int kStep = D <= 128 ? 4 : 2;   // pages per step
  static constexpr int U = 16 / HP < kStep ? 16 / HP : kStep;   // pages per set of scores
  static constexpr int SETS = kStep / U;
  static constexpr int NH = D <= 128 ? 1 : D / 128;   // 128-dim parts
  static constexpr int KWD = D == 64 ? 2 : 4;      // K words per lane, page and part
  static constexpr int VWD = D == 64 ? 2 : 4;
  static constexpr int W = D < 128 ? D : 128;
  static constexpr int JN = W / 16;                // dims per lane and part
  static constexpr int QP = QParts<T>::n;
  static constexpr int ACC = HP == 16 ? 2 : 1;     // MFMAs per V operand (hi, lo)

  i32x8 qf[NH][QP];
  u32 qs[NH][QP];          // q's scales: byte g for the columns of page group g, 0 elsewhere
  f32x4 o[NH][JN];         // row 4r + i (head (4r + i) % HP), dim 128 h + c * JN + j
  float mref, lsum;
  u32x4 k[kStep][NH], v[kStep][NH];
  u32 ks[kStep][NH], vs[kStep][NH];
  int r, c;
  u32 koff, voff, ksoff, vsoff;
  float kscale, cap_in, cap_out;

  __device__ __forceinline__ void init(const Pass1Args& a) {
    const int lane = threadIdx.x & 63;
    r = lane >> 4;
    c = lane & 15;
    koff = (u32)(c * (D / 2) + r * 4 * KWD);
    voff = (u32)(kv4_v_at(D) + lane * 4 * VWD);
    ksoff = (u32)(kv4_ks_at(D) + (D == 64 ? r / 2 : r) * 16 + c);
    vsoff = (u32)(kv4_vs_at(D) + (D == 64 ? c / 8 : c / 4) * 16 + 4 * r);
    kscale = a.kscale;
    cap_in = a.cap_in;
    cap_out = a.cap_out;
  }

  // q rows of the chunk's hv valid heads from qbase, q_h bytes apart, as E4M3 parts (QParts). A
  // block with a NaN or an infinity gets the NaN scale.
  __device__ __forceinline__ void load_q(const uint8_t* qbase, int64_t q_h, int hv) {
    const int h = c % HP;
#pragma unroll
    for (int p = 0; p < NH; ++p) {
      // this lane's dims (see mfma_mx): 16 from d0 in bytes 0 .. 15, 16 from d1 in 16 .. 31; at
      // D = 64 lane row r of K holds dims 16 r .. 16 r + 15 in the first half of its block
      const int d0 = D == 64 ? 8 * r : 128 * p + 16 * r;
      const int d1 = D == 64 ? 32 + 8 * r : d0 + 64;
      const bool live = h < hv && (D != 64 || (r & 1) == 0);
      float x[2][16];
      u32 top[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        u32 w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = 0u;
        if (live) ld_words_cached<8>(w, qbase + (int64_t)h * q_h + 2 * (e ? d1 : d0));
        top[e] = 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          unpack2(w[i], &x[e][2 * i], &x[e][2 * i + 1]);
          top[e] = max(top[e], __builtin_bit_cast(u32, x[e][2 * i]) & 0x7fffffffu);
          top[e] = max(top[e], __builtin_bit_cast(u32, x[e][2 * i + 1]) & 0x7fffffffu);
        }
        // a 32-dim block of q: lane rows 2 (r / 2) and 2 (r / 2) + 1 (D = 64: rows 0 and 2)
        top[e] = max(top[e], (u32)__shfl_xor((int)top[e], D == 64 ? 32 : 16, 64));
        if constexpr (D == 64) top[e] = max(top[e], (u32)__shfl_xor((int)top[e], 16, 64));
      }
      int ex[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int b = (int)(top[e] >> 23);
        ex[e] = top[e] == 0u ? 127 : max(b, q_part_exp(QP - 1) + 1);   // 255: NaN or infinity
      }
#pragma unroll
      for (int i = 0; i < QP; ++i) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float sc = __builtin_bit_cast(float, (u32)(min(ex[e], 254) - q_part_exp(i)) << 23);
          float y4[16];
          if (i == 0) {                              // 1 / sc is a power of two too
            const float inv = __builtin_bit_cast(
                float, (u32)(254 - (min(ex[e], 254) - q_part_exp(0))) << 23);
#pragma unroll
            for (int y = 0; y < 16; ++y) y4[y] = __builtin_rintf(x[e][y] * inv) * sc;
          } else {
#pragma unroll
            for (int y = 0; y < 16; ++y) y4[y] = x[e][y];
          }
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            i16x2 q8 = {0, 0};
            q8 = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(q8, y4[4 * y], y4[4 * y + 1], sc, false);
            q8 = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(q8, y4[4 * y + 2], y4[4 * y + 3], sc, true);
            const u32 word = __builtin_bit_cast(u32, q8);
            qf[p][i][4 * e + y] = (int)word;
            const f32x2 a0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(word, sc, false);
            const f32x2 a1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(word, sc, true);
            x[e][4 * y] -= a0[0];
            x[e][4 * y + 1] -= a0[1];
            x[e][4 * y + 2] -= a1[0];
            x[e][4 * y + 3] -= a1[1];
          }
        }
      }
      // the scale of this lane's column and block r (D = 64: block r / 2): held by lane row
      // 2 (r % 2) (D = 64: by every row), first half for r < 2
      int e0 = ex[0], e1 = ex[1];
      if constexpr (D != 64) {
        const int src = ((r & 1) << 5) | c;
        e0 = __shfl(ex[0], src, 64);
        e1 = __shfl(ex[1], src, 64);
      }
      const int mine = r < 2 ? e0 : e1;
#pragma unroll
      for (int i = 0; i < QP; ++i)
        qs[p][i] = (u32)(mine == 255 ? 255 : mine - q_part_exp(i)) << (8 * (c / HP));
    }
  }

  static __device__ __forceinline__ void unpack2(u32 w, float* x, float* y) {
    if constexpr (__is_same(T, F16)) {
      const f16x2 hh = __builtin_bit_cast(f16x2, w);
      *x = (float)hh[0];
      *y = (float)hh[1];
    } else {
      *x = __builtin_bit_cast(float, w << 16);
      *y = __builtin_bit_cast(float, w & 0xffff0000u);
    }
  }

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int p = 0; p < NH; ++p)
#pragma unroll
      for (int j = 0; j < JN; ++j) o[p][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    mref = kMinit;
    lsum = 0.f;
  }

  // loads of page slot I (a block that does not exist: a zero extent, zeros and no access)
  template <int I>
  __device__ __forceinline__ void load_k(const uint8_t* blk, bool live) {
    const __amdgpu_buffer_rsrc_t rs = page_rsrc(blk, live ? (u32)kv4_bytes(D) : 0u);
    static_for<NH>([&](auto pc) {
      constexpr int p = decltype(pc)::value;
      u32 w[4] = {0u, 0u, 0u, 0u};
      ld_buf<KWD>(w, rs, koff, 64 * p);
      k[I][p] = u32x4{w[0], w[1], w[2], w[3]};
      ks[I][p] = (u32)__builtin_amdgcn_raw_buffer_load_b8(rs, (int)ksoff, 64 * p, kBufNT);
    });
  }
  template <int I>
  __device__ __forceinline__ void load_v(const uint8_t* blk, bool live) {
    const __amdgpu_buffer_rsrc_t rs = page_rsrc(blk, live ? (u32)kv4_bytes(D) : 0u);
    static_for<NH>([&](auto pc) {
      constexpr int p = decltype(pc)::value;
      u32 w[4] = {0u, 0u, 0u, 0u};
      ld_buf<VWD>(w, rs, voff, 1024 * p);
      v[I][p] = u32x4{w[0], w[1], w[2], w[3]};
      vs[I][p] = (u32)__builtin_amdgcn_raw_buffer_load_b32(rs, (int)vsoff, 64 * p, kBufNT);
    });
  }

  // Tokens of page slot I outside [lo, hi): their scales may hold anything, so K's becomes 1 (a
  // NaN would reach the scores of the set's other pages) and V's 0.
  template <int I>
  __device__ __forceinline__ void mask_scales(int lo, int hi) {
    u32 m = 0u;
#pragma unroll
    for (int t = 0; t < 4; ++t) m |= 4 * r + t >= lo && 4 * r + t < hi ? 0xffu << (8 * t) : 0u;
#pragma unroll
    for (int p = 0; p < NH; ++p) {
      ks[I][p] = c >= lo && c < hi ? ks[I][p] : 127u;
      vs[I][p] &= m;
    }
  }

  // Scores of the step's pages
  __device__ __forceinline__ void scores(f32x4 (&s)[SETS]) {
    static_for<SETS>([&](auto xc) {
      constexpr int x = decltype(xc)::value;
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
      static_for<U>([&](auto gc) {
        constexpr int g = decltype(gc)::value;
#pragma unroll
        for (int p = 0; p < NH; ++p)
#pragma unroll
          for (int i = 0; i < QP; ++i)
            acc = mfma_mx<g>(k[x * U + g][p], qf[p][i], acc, ks[x * U + g][p], qs[p][i]);
      });
      s[x] = acc;
    });
  }

  // The running softmax over the step's scores: s becomes p. valid: of page slot i in 16 bits
  // from bit 16 i.
  __device__ __forceinline__ void softmax(f32x4 (&s)[SETS], bool edge, uint64_t valid) {
    float mx = kNegInf;
#pragma unroll
    for (int x = 0; x < SETS; ++x) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[x][i] = CAP ? cap_out * tanh_approx(s[x][i] * cap_in) : s[x][i] * kscale;
      }
    }
    if constexpr (U * HP < 16) {                   // columns without a page
#pragma unroll
      for (int i = 0; i < 4; ++i) s[0][i] = c < U * HP ? s[0][i] : kNegInf;
    }
    if (edge) {
#pragma unroll
      for (int x = 0; x < SETS; ++x) {
        const int vl = (int)(valid >> (16 * (x * U + c / HP % U)));   // this lane's page
        const int lo = vl >> 8 & 255, hi = vl & 255;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          s[x][i] = 4 * r + i >= lo && 4 * r + i < hi && (U * HP == 16 || c < U * HP) ? s[x][i]
                                                                                     : kNegInf;
      }
    }
#pragma unroll
    for (int x = 0; x < SETS; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[x][i]);
    if (__builtin_amdgcn_ballot_w64(mx > mref + kSlack)) {
      const float mn = fmaxf(mref, max_head<HP>(mx));
      const float al = __builtin_amdgcn_exp2f(mref - mn);
      lsum *= al;
      mref = mn;
#pragma unroll
      for (int i = 0; i < 4; ++i) {                // row 4r + i's head is column (4r + i) % HP's
        const float f = __shfl(al, (4 * r + i) % HP, 16);
#pragma unroll
        for (int p = 0; p < NH; ++p)
#pragma unroll
          for (int j = 0; j < JN; ++j) o[p][j][i] *= f;
      }
    }
#pragma unroll
    for (int x = 0; x < SETS; ++x) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[x][i] = __builtin_amdgcn_exp2f(s[x][i] - mref);
      lsum += (s[x][0] + s[x][1]) + (s[x][2] + s[x][3]);
    }
  }

  // The A operands of P.V: pair m holds pages 2m (words 0, 1) and 2m + 1 (words 2, 3), rows =
  // columns of the scores. HP = 16: hi in pa[m][0], lo in pa[m][1]. HP = 8: rows of group g hold
  // page 2m + g's hi and the other page's lo. HP = 4: page i's hi in rows of group i, its lo in
  // rows of group i ^ 2, zero in the other pages' rows.
  __device__ __forceinline__ void weights(const f32x4 (&s)[SETS], u32x4 (&pa)[kStep / 2][ACC]) const {
    u32 hi[SETS][2], lo[SETS][2];
#pragma unroll
    for (int x = 0; x < SETS; ++x)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float h0, h1, l0, l1;
        hi[x][e] = BF16::pack2(s[x][2 * e], s[x][2 * e + 1], &h0, &h1);
        lo[x][e] = BF16::pack2(s[x][2 * e] - h0, s[x][2 * e + 1] - h1, &l0, &l1);
      }
    if constexpr (HP == 16) {
#pragma unroll
      for (int m = 0; m < kStep / 2; ++m) {
        pa[m][0] = u32x4{hi[2 * m][0], hi[2 * m][1], hi[2 * m + 1][0], hi[2 * m + 1][1]};
        pa[m][1] = u32x4{lo[2 * m][0], lo[2 * m][1], lo[2 * m + 1][0], lo[2 * m + 1][1]};
      }
    } else {
#pragma unroll
      for (int x = 0; x < SETS; ++x)
#pragma unroll
        for (int e = 0; e < 2; ++e) lo[x][e] = dpp_u<0x128>(lo[x][e]);   // from column c ^ 8
      if constexpr (HP == 8) {
#pragma unroll
        for (int m = 0; m < SETS; ++m)
          pa[m][0] = u32x4{c < 8 ? hi[m][0] : lo[m][0], c < 8 ? hi[m][1] : lo[m][1],
                           c < 8 ? lo[m][0] : hi[m][0], c < 8 ? lo[m][1] : hi[m][1]};
      } else {
        const u32 even = (c >> 2 & 1) ? 0u : ~0u, own = c < 8 ? ~0u : 0u;
        const u32 d0 = hi[0][0] ^ lo[0][0], d1 = hi[0][1] ^ lo[0][1];
        static_for<kStep / 2>([&](auto mc) {         // pages 0, 1 then 2, 3
          constexpr int m = decltype(mc)::value;
          const u32 pick = m == 0 ? own : ~own;      // hi there, lo elsewhere
          const u32 x0 = lo[0][0] ^ (d0 & pick), x1 = lo[0][1] ^ (d1 & pick);
          pa[m][0] = u32x4{x0 & even, x1 & even, x0 & ~even, x1 & ~even};
        });
      }
    }
  }

  // dims 2b, 2b+1 of this lane's run (part p) for its 4 tokens of page slot i: words (tokens
  // 0, 1) and (2, 3) of the even dim in e, of the odd dim in d
  template <int B>
  __device__ __forceinline__ void widen(int i, int p, u32 (&e)[2], u32 (&d)[2]) const {
    u32 t[4];
    static_for<4>([&](auto tc) {
      constexpr int x = decltype(tc)::value;
      const u32 sc = e8m0_exp<x>(vs[i][p]);
      if constexpr (D == 64) t[x] = fp4_bf16<2 * (x % 2) + B>(v[i][p][x / 2], sc);
      else t[x] = fp4_bf16<B>(v[i][p][x], sc);
    });
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      e[x] = __builtin_amdgcn_perm(t[2 * x + 1], t[2 * x], 0x05040100u);
      d[x] = __builtin_amdgcn_perm(t[2 * x + 1], t[2 * x], 0x07060302u);
    }
  }

  __device__ __forceinline__ void accumulate(const u32x4 (&pa)[kStep / 2][ACC]) {
    static_for<kStep / 2>([&](auto mc) {
      constexpr int m = decltype(mc)::value;
#pragma unroll
      for (int p = 0; p < NH; ++p)
        static_for<JN / 2>([&](auto bc) {
          constexpr int b = decltype(bc)::value;
          u32 e0[2], d0[2], e1[2], d1[2];
          widen<b>(2 * m, p, e0, d0);
          widen<b>(2 * m + 1, p, e1, d1);
          const u32x4 ve = {e0[0], e0[1], e1[0], e1[1]}, vd = {d0[0], d0[1], d1[0], d1[1]};
#pragma unroll
          for (int x = 0; x < ACC; ++x) {
            o[p][2 * b] = BF16::mfma(pa[m][x], ve, o[p][2 * b]);
            o[p][2 * b + 1] = BF16::mfma(pa[m][x], vd, o[p][2 * b + 1]);
          }
        });
    });
  }

  // Pages 0 .. n-1 of a run, groups of kStep first + w, + NW, ...; block(i): the page block of
  // page i; valid(i): its tokens, hi | lo << 8. K's next loads are issued when the scores have
  // read the registers, V's when P.V has: the other half of a step covers each.
  template <class BlockFn, class ValidFn>
  __device__ __forceinline__ void stream(int NW, int w, int n, BlockFn block, ValidFn valid) {
    const int groups = (n + kStep - 1) / kStep;
    if (w >= groups) return;
    const uint8_t* at[kStep];
    static_for<kStep>([&](auto ic) {
      constexpr int i = decltype(ic)::value;
      at[i] = block(min(kStep * w + i, n - 1));
      load_k<i>(at[i], kStep * w + i < n);
    });
    static_for<kStep>([&](auto ic) {
      constexpr int i = decltype(ic)::value;
      load_v<i>(at[i], kStep * w + i < n);
    });
    for (int g = w; g < groups; g += NW) {
      const int next = g + NW;
      uint64_t vl = 0;
      static_for<kStep>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        vl |= (uint64_t)(kStep * g + i < n ? valid(kStep * g + i) : 0) << (16 * i);
        at[i] = block(min(kStep * next + i, n - 1));
      });
      const bool edge = vl != (kStep == 4 ? 0x0010001000100010u : 0x00100010u);
      if (edge) {
        static_for<kStep>([&](auto ic) {
          constexpr int i = decltype(ic)::value;
          mask_scales<i>((int)(vl >> (16 * i + 8)) & 255, (int)(vl >> (16 * i)) & 255);
        });
      }
      f32x4 s[SETS];
      scores(s);
      static_for<kStep>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        load_k<i>(at[i], kStep * next + i < n);
      });
      softmax(s, edge, vl);
      u32x4 pa[kStep / 2][ACC];
      weights(s, pa);
      accumulate(pa);
      static_for<kStep>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        load_v<i>(at[i], kStep * next + i < n);
      });
    }
  }
};

// LDS for the wavefronts' results: o's 16 rows, references and sums per head
template <int D, int NW>
struct Kv4Smem {
  alignas(16) float o[NW][16][D];
  float m[NW][16], l[NW][16];
};

// The workgroup's result for hv heads: normalised to out, or a partial (head h at row
// prow0 + h * phstride). Holds workgroup barriers.
template <class T, int D, int HP, int NW, class WV>
__device__ __forceinline__ void kv4_store(WV& wv, Kv4Smem<D, NW>& sm, const Pass1Args& a,
                                          bool direct, uint8_t* out, int64_t prow0,
                                          int64_t phstride, int hv, int w, int tid, int qh0) {
  const float l = sum_head<HP>(wv.lsum);
  if (wv.r == 0 && wv.c < HP) {
    sm.m[w][wv.c] = wv.mref;
    sm.l[w][wv.c] = l;
  }
#pragma unroll
  for (int p = 0; p < WV::NH; ++p)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < WV::JN; j += 4)
        *reinterpret_cast<f32x4*>(&sm.o[w][4 * wv.r + i][128 * p + wv.c * WV::JN + j]) =
            f32x4{wv.o[p][j][i], wv.o[p][j + 1][i], wv.o[p][j + 2][i], wv.o[p][j + 3][i]};
  __syncthreads();
  const float* sink = a.sinks ? a.sinks + qh0 : nullptr;
  const bool out8 = (((uintptr_t)out | (uintptr_t)a.o_h) & 7) == 0;
  for (int idx = tid; idx < hv * (D / 4); idx += NW * 64) {
    const int h = idx / (D / 4), d = 4 * (idx % (D / 4));
    float mt = kMinit;
#pragma unroll
    for (int ww = 0; ww < NW; ++ww) mt = fmaxf(mt, sm.m[ww][h]);
    float L = 0.f;
    f32x4 O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ww = 0; ww < NW; ++ww) {
      const float f = __builtin_amdgcn_exp2f(sm.m[ww][h] - mt);
      L += sm.l[ww][h] * f;
      f32x4 x = *reinterpret_cast<const f32x4*>(&sm.o[ww][h][d]);
#pragma unroll
      for (int g = 1; g < 16 / HP; ++g) x += *reinterpret_cast<const f32x4*>(&sm.o[ww][g * HP + h][d]);
      O += x * f;
    }
    const bool empty = !(mt > kMinit) && L == 0.f;
    if (direct) {
      if (sink) L += __builtin_amdgcn_exp2f(sink[h] * kLog2e - mt);   // +inf when empty
      uint8_t* op = out + (int64_t)h * a.o_h + 2 * d;
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = L == 0.f ? 0.f : O[e] / L;
      if (out8) {
        float t0, t1;
        *reinterpret_cast<u32x2*>(op) =
            u32x2{T::pack2(x[0], x[1], &t0, &t1), T::pack2(x[2], x[3], &t0, &t1)};
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) T::store(op + 2 * e, x[e]);
      }
    } else {
      const int64_t row = prow0 + h * phstride;
      *reinterpret_cast<f32x4*>(a.part_o + row * D + d) = O;
      if (d == 0) {
        a.part_m[row] = empty ? kEmptyM : mt * kLn2;
        a.part_l[row] = L;
      }
    }
  }
  __syncthreads();   // the LDS is reused by the next segment
}

// Explicit split: workgroup = (head chunk, kv head, split, sequence), as dk_pass1_split
template <class T, int D, int HP, bool CAP, int NW>
__global__ __launch_bounds__(NW * 64, 2) void dk_kv4_split(Pass1Args a) {
  __shared__ Kv4Smem<D, NW> sm;
  Kv4Wave<T, D, HP, CAP> wv;
  wv.init(a);
  const int w = uniform(threadIdx.x >> 6);
  int hc = 0, t = blockIdx.x;
  if (a.chunks > 1) {
    const int x = t % kXcds, y = t / kXcds;
    hc = y % a.chunks;
    t = (y / a.chunks) * kXcds + x;
    if (t >= a.batch * a.hkv * a.split) return;   // padding of the last XCD round
  }
  const int kvh = t % a.hkv;
  t /= a.hkv;
  const int s = t % a.split, b = t / a.split;
  const int seq0 = seq_begin(a, b);
  const int npages = max(seq_begin(a, b + 1), seq0) - seq0;
  const int last = min(max(ld_const(a.last_len, b), 0), kPage);
  int first_page = 0, first_tok = 0;
  if (a.window > 0 && npages > 0) {
    const int t0 = max((npages - 1) * kPage + last - a.window, 0);
    first_page = t0 / kPage;
    first_tok = t0 % kPage;
  }
  const int npw = npages - first_page;
  const int pps = (npw + a.split - 1) / a.split;
  const int p0 = first_page + min(s * pps, npw);
  const int n = max(min(p0 + pps, npages) - p0, 0);
  const int qh0 = kvh * a.group + hc * a.per;
  const int hv = min(a.per, a.group - hc * a.per);
  wv.load_q(a.q + (int64_t)b * a.q_b + (int64_t)qh0 * a.q_h, a.q_h, hv);
  wv.reset();
  const uint8_t* base = a.kv + (int64_t)kvh * a.kv_h;
  auto block = [&](int i) -> const uint8_t* {
    u32 pid = (u32)uniform(ld_const(a.indices, seq0 + p0 + i));
    pid = pid < a.num_pages ? pid : 0u;
    return base + (int64_t)pid * a.kv_p;
  };
  auto valid = [&](int i) -> int {
    const int pg = p0 + i;
    return (pg == npages - 1 ? last : kPage) | (pg == first_page ? first_tok << 8 : 0);
  };
  wv.stream(NW, w, n, block, valid);
  kv4_store<T, D, HP, NW>(wv, sm, a, a.direct != 0,
                          a.out + (int64_t)b * a.o_b + (int64_t)qh0 * a.o_h,
                          ((int64_t)b * a.hq + qh0) * a.split + s, a.split, hv, w,
                          (int)threadIdx.x, qh0);
}

// Balanced: the page ranges, segments and partial slots of dk_pass1_balanced (one kv head per
// workgroup; the range split that charges sequence starts when a.seg_cost > 0)
template <class T, int D, int HP, bool CAP, int NW>
__global__ __launch_bounds__(NW * 64, 2) void dk_kv4_balanced(Pass1Args a, int heads) {
  __shared__ Kv4Smem<D, NW> sm;
  Kv4Wave<T, D, HP, CAP> wv;
  wv.init(a);
  const int w = uniform(threadIdx.x >> 6);
  const int Wg = a.ranges;
  int hc, j;
  if (a.chunks > 1) {
    const int x = (int)blockIdx.x % kXcds, y = (int)blockIdx.x / kXcds;
    const int un = (y / a.chunks) * kXcds + x;
    if (un >= a.hkv * Wg) return;
    j = un / a.hkv;
    hc = (y % a.chunks) * a.hkv + un % a.hkv;
  } else {
    hc = (int)blockIdx.x % a.hkv;
    j = (int)blockIdx.x / a.hkv;
  }
  const int base = seq_begin(a, 0);
  const int P = max(seq_begin(a, a.batch) - base, 0);
  const int A = a.seg_cost;
  int u, u_end, b = 0, L = 0;
  int64_t Lc = 0;
  if (A == 0) {
    L = (P + Wg - 1) / Wg;
    if (L <= 0) return;
    u = (int)min((int64_t)j * L, (int64_t)P);
    u_end = min(u + L, P);
  } else {
    Lc = range_cost_len(P, A, a.batch, Wg);
    if (Lc <= 0) return;
    u = cost_boundary(a, base, P, A, (int64_t)j * Lc, &b);
    int b_end;
    u_end = (int64_t)(j + 1) * Lc >= (int64_t)P + (int64_t)A * max(a.batch - 1, 0)
                ? P : cost_boundary(a, base, P, A, (int64_t)(j + 1) * Lc, &b_end);
  }
  if (u >= u_end) return;
  const int kvh = hc % a.hkv, chunk = hc / a.hkv;
  const int qh0 = kvh * a.group + chunk * a.per;
  const int hv = min(a.per, a.group - chunk * a.per);
  const uint8_t* kbase = a.kv + (int64_t)kvh * a.kv_h;
  if (A == 0) {
    int lo = 0, hi = a.batch - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (seq_begin(a, mid) - base <= u) lo = mid; else hi = mid - 1;
    }
    b = lo;
  }
  int seq0 = seq_begin(a, b);
  int np = max(seq_begin(a, b + 1), seq0) - seq0;
  int pg = u - (seq0 - base);
  while (A != 0 && pg >= np && b < a.batch - 1) {
    ++b;
    seq0 = seq_begin(a, b);
    np = max(seq_begin(a, b + 1), seq0) - seq0;
    pg = u - (seq0 - base);
  }
  if (np <= 0 || pg < 0 || pg >= np) return;   // only for a decreasing kv_indptr (invalid)
  while (true) {
    const int n = min(np - pg, u_end - u);
    wv.load_q(a.q + (int64_t)b * a.q_b + (int64_t)qh0 * a.q_h, a.q_h, hv);
    wv.reset();
    const int last = min(max(ld_const(a.last_len, b), 0), kPage);
    const int idx0 = seq0 + pg, left = np - 1 - pg;
    auto block = [&](int i) -> const uint8_t* {
      u32 pid = (u32)uniform(ld_const(a.indices, idx0 + i));
      pid = pid < a.num_pages ? pid : 0u;
      return kbase + (int64_t)pid * a.kv_p;
    };
    auto valid = [&](int i) -> int { return i == left ? last : kPage; };
    wv.stream(NW, w, n, block, valid);
    // ranges holding this sequence's units
    const int start = seq0 - base;
    int nslots;
    if (A == 0) {
      nslots = (start + np - 1) / L - start / L + 1;
    } else {
      const int64_t c0 = (int64_t)start + (int64_t)A * b;
      nslots = (int)((c0 + np - 1) / Lc - c0 / Lc + 1);
    }
    kv4_store<T, D, HP, NW>(wv, sm, a, nslots == 1,
                            a.out + (int64_t)b * a.o_b + (int64_t)qh0 * a.o_h,
                            ((int64_t)hc * (Wg + a.batch) + j + b) * heads, 1, hv, w,
                            (int)threadIdx.x, qh0);
    u += n;
    if (u >= u_end) break;
    do {
      ++b;
      seq0 = seq_begin(a, b);
      np = max(seq_begin(a, b + 1), seq0) - seq0;
    } while (np == 0 && b < a.batch - 1);
    if (np <= 0) break;                        // only for an invalid kv_indptr
    pg = 0;
  }
}

// Kernel symbols of one head_dim (dk_kv4.hip, compiled once per head_dim); hp 4, 8 or 16 q heads
template <int D>
const void* kv4_symbol(bool bf16, int hp, bool cap, int waves, bool balanced);
extern template const void* kv4_symbol<64>(bool, int, bool, int, bool);
extern template const void* kv4_symbol<128>(bool, int, bool, int, bool);
extern template const void* kv4_symbol<256>(bool, int, bool, int, bool);

}  // namespace dk
