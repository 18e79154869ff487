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
typedef u32 u32x6 __attribute__((ext_vector_type(6)));
typedef float f32x16v __attribute__((ext_vector_type(16)));
typedef float f32x32v __attribute__((ext_vector_type(32)));

// C += A.B: A 16 tokens x 128 dims of E2M1 (16 bytes per lane), B 128 dims x 16 columns of E2M3
// (24 bytes per lane); lane row r holds k = 32 r .. 32 r + 31 of both. sa / sb: E8M0 scales of the
// lane's row / column for those 32 (byte GB of sb). The products are multiples of 1/16 up to 45 (times
// the scales), and the MFMA adds them exactly.
template <int GB>
__device__ __forceinline__ f32x4 mfma_mx(u32x4 a, u32x6 b, f32x4 c, u32 sa, u32 sb) {
  const i32x8 av = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8 bv = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], (int)b[4], (int)b[5], 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 2, 0, (int)sa, GB, (int)sb);
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

// q enters the MX products as QParts parts of E2M3 (steps of 1/8 up to 2, 1/4 up to 4), each with a
// power-of-two scale per 32-dim block: the first puts the block's largest magnitude in [2, 4), each
// next one is 2^-5 of the last and holds what that left (at most 1/8 of its scale, so 4 of the next). 3
// parts leave at most 2^-14 of the power of two below the block's largest magnitude, 4 parts 2^-19:
// bf16's 8 bits are whole down to 2^-7 of the largest and fp16's 11 bits down to 2^-9, and what smaller
// elements lose is no more than the largest one's own last bit. fp6 operands multiply at twice
// the rate of fp8 ones, whose sums the MFMA also cuts 13 bits below a group's largest product.
template <class T>
struct QParts {
  static constexpr int n = 3;
};
template <>
struct QParts<F16> {
  static constexpr int n = 4;
};
// Part i's scale exponent below the block's largest exponent
__device__ __forceinline__ constexpr int q_part_exp(int i) { return 1 + 5 * i; }

// One wavefront over pages of one kv head, kStep at a time, for up to HP (4, 8 or 16) q heads.
//   * q.k: K's codes and scales are MFMA operands as they lie; q enters as E2M3 parts with
//     scales of its own, one MFMA each. The 16 columns are HP heads x U pages: for a page's MFMAs
//     the scale of every other page's columns is 0 (2^-127), so U pages accumulate into one set of
//     scores and every lane's 4 scores count: lane (r, c) holds tokens 4r .. 4r+3 of page group(c) of
//     the set, head head(c).
//   * softmax as in Wave: fp32, log2 domain, a reference that moves by more than 2^8 only.
//   * P.V in bf16, whatever q's type: E2M1 times a power of two is exact there, and p as hi + lo
//     parts keeps 16 bits at any magnitude. A lane's V words are widened with their scales by
//     v_cvt_scalef32_pk_bf16_fp4, two neighbouring dims of one token each, on v_mfma_f32_16x16x32.
//     HP = 4: k = (token, parity): the pair is the operand as it is, and a row that is to sum the even
//     dims has p in the even k and 0 in the odd ones. The 16 rows are 4 heads x (parity, part).
//     HP = 8, 16: k = tokens of two pages, the pairs regrouped by token (v_perm); rows are the heads,
//     and for HP = 8 the parts share an MFMA, each page's lo in the rows of the other page.
// Bound by HBM reads at D = 128 and 256 with up to 4 heads: 32 x 8192 tokens of 32/8/128 fp16 48 us (286
// MB; 6.5 TB/s between start and end, where reads of this page pattern without arithmetic reach 6.8). At
// D = 64, whose pages hold half the bytes per instruction, by instruction issue (79 % of the cycles): 128
// x 128..8192 tokens of 64/8/64 bf16 65 us and a merge (292 MB, 4.5 TB/s; the pattern 6.2); three
// wavefronts per SIMD instead of two 73 against 71. With 8 and 16 heads by the matrix instructions'
// dependent chains: 16 x 32768 of 64/8/128 fp16 94 us, 8 x 65536 of 128/8/128 bf16 97 (6.1 and 5.9 TB/s).
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
  static constexpr bool PAIR = HP == 4;            // P.V over (token, parity)
  static constexpr int ACC = HP == 16 ? 2 : 1;     // MFMAs per V operand (hi, lo)
  static constexpr int OV = PAIR ? JN / 2 : JN;    // accumulators per part
  static constexpr int kBatch = 64 / kStep;        // steps whose page offsets the lanes hold

  struct Pages {           // a step's pages as loaded
    u32x4 k[kStep][NH], v[kStep][NH];
    u32 ks[kStep][NH], vs[kStep][NH];
  };
  u32x6 qf[NH][QP];
  u32 qs[NH][QP];          // q's scales: byte g for the columns of page group g, 0 elsewhere
  f32x4 o[NH][OV];         // PAIR: head r, dims 2j + {0, 1, 0, 1} of the lane's run, parts hi, hi, lo,
                           // lo; else row 4r + i (head (4r + i) % HP), dim 128 h + c * JN + j
  float mref, lsum;
  int r, c;
  u32 koff, voff, ksoff, vsoff;
  float kscale, cap_in, cap_out;
  // the pages of a run: their ids from indices[idx0], n of them; steps w, w + NW, ...
  const int32_t* ids;
  const uint8_t* base;     // the kv head's block of page 0
  uint64_t page_bytes;
  uint32_t num_pages;
  u32 off_lo, off_hi;      // lane l: byte offset of page l % kStep of step l / kStep of the batch
  int32_t next_id;         // the next batch's page id

  static __device__ __forceinline__ int head(int c) { return PAIR ? c >> 2 : c % HP; }
  static __device__ __forceinline__ int group(int c) { return PAIR ? c & 3 : c / HP; }
  // over the lanes that hold one q head
  static __device__ __forceinline__ float max_head(float x) {
    if constexpr (PAIR) {
      x = fmaxf(x, xor1(x));
      x = fmaxf(x, xor2(x));
    }
    if constexpr (HP == 8) x = fmaxf(x, row_ror<8>(x));
    return max_xor32(max_xor16(x));
  }
  static __device__ __forceinline__ float sum_head(float x) {
    if constexpr (PAIR) {
      x += xor1(x);
      x += xor2(x);
    }
    if constexpr (HP == 8) x += row_ror<8>(x);
    return sum_xor32(sum_xor16(x));
  }

  __device__ __forceinline__ void init(const Pass1Args& a, int kvh) {
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
    base = a.kv + (int64_t)kvh * a.kv_h;
    page_bytes = (uint64_t)a.kv_p;
    num_pages = a.num_pages;
  }

  // q rows of the chunk's hv valid heads from qbase, q_h bytes apart, as E2M3 parts (QParts). A
  // block with a NaN or an infinity gets the NaN scale.
  __device__ __forceinline__ void load_q(const uint8_t* qbase, int64_t q_h, int hv) {
    const int h = head(c);
    constexpr int NW_ = D == 64 ? 8 : 16;          // q words per lane and part
#pragma unroll
    for (int p = 0; p < NH; ++p) {
      // the dims that K's lane row r holds: 32 from 128 p + 32 r (D = 64: 16 from 16 r, and zeros)
      u32 w[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = 0u;
      if (h < hv) ld_words_cached<NW_>(w, qbase + (int64_t)h * q_h + 4 * NW_ * (4 * p + r));
      f32x16v lo, hi;                              // even and odd dims
      u32 top = 0u;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float x, y;
        unpack2(w[i], &x, &y);
        lo[i] = x;
        hi[i] = y;
        top = max(top, __builtin_bit_cast(u32, x) & 0x7fffffffu);
        top = max(top, __builtin_bit_cast(u32, y) & 0x7fffffffu);
      }
      if constexpr (D == 64) top = max(top, (u32)__shfl_xor((int)top, 16, 64));   // the other half
      const int e = (int)(top >> 23);
      const int ex = top == 0u ? 127 : max(e, q_part_exp(QP - 1) + 1);   // 255: NaN or infinity
      static_for<QP>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        const float sc = __builtin_bit_cast(float, (u32)(min(ex, 254) - q_part_exp(i)) << 23);
        const u32x6 q6 = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(lo, hi, sc);
        // the conversion writes its result before it has read all its inputs, which the compiler
        // does not know: inputs that live on share no register with it (measured: a result over the
        // scale's or a source's register was wrong)
        asm volatile("" ::"v"(lo), "v"(hi), "v"(sc), "v"(q6));
        qf[p][i] = q6;
        qs[p][i] = (u32)(ex == 255 ? 255 : ex - q_part_exp(i)) << (8 * group(c));
        if constexpr (i + 1 < QP) {
          const f32x32v back = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(q6, sc);
          asm volatile("" ::"v"(q6), "v"(sc), "v"(back));
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            lo[j] -= back[2 * j];
            hi[j] -= back[2 * j + 1];
          }
        }
      });
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
      for (int j = 0; j < OV; ++j) o[p][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    mref = kMinit;
    lsum = 0.f;
  }

  // ---- pages
  // This lane's page of the batch from step k0: id of page l % kStep of step k0 + l / kStep of the run
  // (past its end: the last one's)
  __device__ __forceinline__ int32_t lane_id(int NW, int w, int n, int k0) const {
    const int lane = threadIdx.x & 63;
    return ids[min(kStep * (w + NW * (k0 + lane / kStep)) + lane % kStep, n - 1)];
  }
  __device__ __forceinline__ void take_ids() {     // next_id becomes the batch's offsets
    const uint64_t pid = (u32)next_id < num_pages ? (u32)next_id : 0u;
    const uint64_t off = pid * page_bytes;
    off_lo = (u32)off;
    off_hi = (u32)(off >> 32);
  }
  // loads of page slot I from the lanes' offsets (live == false: a zero extent, zeros and no access)
  template <int I>
  __device__ __forceinline__ void load(Pages& b, int lane, bool live) const {
    const uint64_t off = (u32)__builtin_amdgcn_readlane((int)off_lo, lane) |
                         (uint64_t)(u32)__builtin_amdgcn_readlane((int)off_hi, lane) << 32;
    const __amdgpu_buffer_rsrc_t rs = page_rsrc(base + off, live ? (u32)kv4_bytes(D) : 0u);
    static_for<NH>([&](auto pc) {
      constexpr int p = decltype(pc)::value;
      u32 w[4] = {0u, 0u, 0u, 0u}, x[4] = {0u, 0u, 0u, 0u};
      ld_buf<KWD>(w, rs, koff, 64 * p);
      b.k[I][p] = u32x4{w[0], w[1], w[2], w[3]};
      b.ks[I][p] = (u32)__builtin_amdgcn_raw_buffer_load_b8(rs, (int)ksoff, 64 * p, kBufNT);
      ld_buf<VWD>(x, rs, voff, 1024 * p);
      b.v[I][p] = u32x4{x[0], x[1], x[2], x[3]};
      b.vs[I][p] = (u32)__builtin_amdgcn_raw_buffer_load_b32(rs, (int)vsoff, 64 * p, kBufNT);
    });
  }
  // step k of this wavefront (its pages' offsets are in the lanes), which is global step w + NW * k
  __device__ __forceinline__ void fetch(Pages& b, int NW, int w, int n, int k) const {
    const int first = kStep * (w + NW * k), lane = kStep * (k % kBatch);
    static_for<kStep>([&](auto ic) {
      constexpr int i = decltype(ic)::value;
      load<i>(b, lane + i, first + i < n);
    });
  }

  // Tokens of page slot I outside [lo, hi) of the page: their scales may hold anything, so K's becomes
  // 1 (a NaN would reach the scores of the set's other pages) and V's 0.
  template <int I>
  __device__ __forceinline__ void mask_scales(Pages& b, int lo, int hi) const {
    u32 m = 0u;
#pragma unroll
    for (int t = 0; t < 4; ++t) m |= 4 * r + t >= lo && 4 * r + t < hi ? 0xffu << (8 * t) : 0u;
#pragma unroll
    for (int p = 0; p < NH; ++p) {
      b.ks[I][p] = c >= lo && c < hi ? b.ks[I][p] : 127u;
      b.vs[I][p] &= m;
    }
  }

  // Scores of the step's pages
  __device__ __forceinline__ void scores(const Pages& b, f32x4 (&s)[SETS]) const {
    static_for<SETS>([&](auto xc) {
      constexpr int x = decltype(xc)::value;
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
      static_for<U>([&](auto gc) {
        constexpr int g = decltype(gc)::value;
#pragma unroll
        for (int p = 0; p < NH; ++p)
#pragma unroll
          for (int i = 0; i < QP; ++i)
            acc = mfma_mx<g>(b.k[x * U + g][p], qf[p][i], acc, b.ks[x * U + g][p], qs[p][i]);
      });
      s[x] = acc;
    });
  }

  // The running softmax over the step's scores: s becomes p. edge: the step's tokens outside
  // [lo, hi) (from the step's first) do not count.
  __device__ __forceinline__ void softmax(f32x4 (&s)[SETS], bool edge, int lo, int hi) {
    float mx = kNegInf;
#pragma unroll
    for (int x = 0; x < SETS; ++x) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[x][i] = CAP ? cap_out * tanh_approx(s[x][i] * cap_in) : s[x][i] * kscale;
        if constexpr (U * HP < 16) s[x][i] = group(c) < U ? s[x][i] : kNegInf;   // no such page
      }
    }
    if (edge) {
#pragma unroll
      for (int x = 0; x < SETS; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int t = kPage * (x * U + group(c)) + 4 * r + i;
          s[x][i] = t >= lo && t < hi ? s[x][i] : kNegInf;
        }
    }
#pragma unroll
    for (int x = 0; x < SETS; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[x][i]);
    if (__builtin_amdgcn_ballot_w64(mx > mref + kSlack)) {
      const float mn = fmaxf(mref, max_head(mx));
      const float al = __builtin_amdgcn_exp2f(mref - mn);
      lsum *= al;
      mref = mn;
      if constexpr (PAIR) {                          // the accumulators are head r's
        const float f = __shfl(al, 4 * r, 16);
#pragma unroll
        for (int p = 0; p < NH; ++p)
#pragma unroll
          for (int j = 0; j < OV; ++j) o[p][j] *= f;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float f = __shfl(al, (4 * r + i) % HP, 16);
#pragma unroll
          for (int p = 0; p < NH; ++p)
#pragma unroll
            for (int j = 0; j < OV; ++j) o[p][j][i] *= f;
        }
      }
    }
#pragma unroll
    for (int x = 0; x < SETS; ++x) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[x][i] = __builtin_amdgcn_exp2f(s[x][i] - mref);
      lsum += (s[x][0] + s[x][1]) + (s[x][2] + s[x][3]);
    }
  }

  // ---- P.V over (token, parity)
  __device__ __forceinline__ void accumulate_pair(const Pages& b, const f32x4 (&s)[SETS]) {
    // a token's p as (hi, lo) in one word: hi rounded to the nearest, lo the remainder cut to bf16
    u32 t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = s[0][i];
      const u32 h = (__builtin_bit_cast(u32, x) + 0x8000u) & 0xffff0000u;
      const float l = x - __builtin_bit_cast(float, h);
      t[i] = __builtin_amdgcn_perm(__builtin_bit_cast(u32, l), h, 0x07060302u);
    }
    // row 4 head + x: parity x & 1, part x >> 1: this lane's part of the word to its parity's half
    const u32 sel = (c & 1) ? ((c & 2) ? 0x03020c0cu : 0x01000c0cu) : ((c & 2) ? 0x0c0c0302u : 0x0c0c0100u);
    static_for<kStep>([&](auto uc) {
      constexpr int u = decltype(uc)::value;
      u32x4 pa;                                      // page u's weights lie in lane u of each quad
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const u32 y = quad_bcast_u<u>(t[i]);
        pa[i] = __builtin_amdgcn_perm(y, y, sel);
      }
#pragma unroll
      for (int p = 0; p < NH; ++p)
        static_for<OV>([&](auto jc) {
          constexpr int j = decltype(jc)::value;
          u32 v[4];
          widen<j>(b, u, p, v);
          o[p][j] = BF16::mfma(pa, u32x4{v[0], v[1], v[2], v[3]}, o[p][j]);
        });
    });
  }

  // ---- P.V over the tokens of two pages
  // The A operands: pair m holds pages 2m (words 0, 1) and 2m + 1 (words 2, 3), rows = columns of
  // the scores. HP = 16: hi in pa[m][0], lo in pa[m][1]. HP = 8: rows of group g hold page 2m + g's
  // hi and the other page's lo.
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
      for (int m = 0; m < SETS; ++m) {
        const u32 l0 = dpp_u<0x128>(lo[m][0]), l1 = dpp_u<0x128>(lo[m][1]);   // from column c ^ 8
        pa[m][0] = u32x4{c < 8 ? hi[m][0] : l0, c < 8 ? hi[m][1] : l1, c < 8 ? l0 : hi[m][0],
                         c < 8 ? l1 : hi[m][1]};
      }
    }
  }
  __device__ __forceinline__ void accumulate_tokens(const Pages& b, const f32x4 (&s)[SETS]) {
    u32x4 pa[kStep / 2][ACC];
    weights(s, pa);
    static_for<kStep / 2>([&](auto mc) {
      constexpr int m = decltype(mc)::value;
#pragma unroll
      for (int p = 0; p < NH; ++p)
        static_for<JN / 2>([&](auto bc) {
          constexpr int j = decltype(bc)::value;
          u32 x[4], y[4];
          widen<j>(b, 2 * m, p, x);
          widen<j>(b, 2 * m + 1, p, y);
          const u32x4 ve = {pair_lo(x[0], x[1]), pair_lo(x[2], x[3]), pair_lo(y[0], y[1]), pair_lo(y[2], y[3])};
          const u32x4 vd = {pair_hi(x[0], x[1]), pair_hi(x[2], x[3]), pair_hi(y[0], y[1]), pair_hi(y[2], y[3])};
#pragma unroll
          for (int e = 0; e < ACC; ++e) {
            o[p][2 * j] = BF16::mfma(pa[m][e], ve, o[p][2 * j]);
            o[p][2 * j + 1] = BF16::mfma(pa[m][e], vd, o[p][2 * j + 1]);
          }
        });
    });
  }
  static __device__ __forceinline__ u32 pair_lo(u32 a, u32 b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
  static __device__ __forceinline__ u32 pair_hi(u32 a, u32 b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

  // dims 2J, 2J+1 of this lane's run (part p) for its 4 tokens of page slot i, as bf16 pairs
  template <int J>
  static __device__ __forceinline__ void widen(const Pages& b, int i, int p, u32 (&t)[4]) {
    static_for<4>([&](auto tc) {
      constexpr int x = decltype(tc)::value;
      const u32 sc = e8m0_exp<x>(b.vs[i][p]);
      if constexpr (D == 64) t[x] = fp4_bf16<2 * (x % 2) + J>(b.v[i][p][x / 2], sc);
      else t[x] = fp4_bf16<J>(b.v[i][p][x], sc);
    });
  }

  // One loaded step, its pages from page `first` of the run; tokens [lo, hi) of the run count
  __device__ __forceinline__ void compute(Pages& b, int first, int lo, int hi) {
    lo -= kPage * first;
    hi -= kPage * first;
    const bool edge = lo > 0 || hi < kStep * kPage;
    if (edge) {
      static_for<kStep>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        mask_scales<i>(b, lo - kPage * i, hi - kPage * i);
      });
    }
    f32x4 s[SETS];
    scores(b, s);
    softmax(s, edge, lo, hi);
    if constexpr (PAIR) accumulate_pair(b, s);
    else accumulate_tokens(b, s);
  }

  // The run's first loads: the ids of the first batch of steps of pages indices[0 .. n)
  __device__ __forceinline__ void start(const int32_t* indices, int NW, int w, int n, Pages& b) {
    ids = indices;
    next_id = lane_id(NW, w, n, 0);
    take_ids();
    fetch(b, NW, w, n, 0);
  }
  // Steps of a run of n pages after start(), whose n may have been larger; tokens [lo, hi) count. The
  // next step's loads are in flight while one is computed.
  __device__ __forceinline__ void stream(int NW, int w, int n, int lo, int hi, Pages& b0) {
    const int all = (n + kStep - 1) / kStep;
    const int steps = all > w ? (all - w + NW - 1) / NW : 0;
    if (steps == 0) return;
    if (steps > kBatch - 1) next_id = lane_id(NW, w, n, kBatch);
    Pages b1;
    auto step = [&](Pages& cur, Pages& nxt, int k) {
      const int kn = k + 1;
      if (kn % kBatch == 0) {                        // the lanes' batch of offsets is used up
        take_ids();
        next_id = lane_id(NW, w, n, kn + kBatch);
      }
      fetch(nxt, NW, w, n, kn);
      compute(cur, kStep * (w + NW * k), lo, hi);
    };
    for (int k = 0;;) {
      step(b0, b1, k);
      if (++k >= steps) break;
      step(b1, b0, k);
      if (++k >= steps) break;
    }
  }
};

// LDS for the wavefronts' results: the accumulators' rows, references and sums per head
template <int D, int HP, int NW>
struct Kv4Smem {
  static constexpr int ROWS = HP == 4 ? 4 : 16;
  alignas(16) float o[NW][ROWS][D];
  float m[NW][16], l[NW][16];
};

// The workgroup's result for hv heads: normalised to out, or a partial (head h at row
// prow0 + h * phstride). Holds workgroup barriers.
template <class T, int D, int HP, int NW, class WV>
__device__ __forceinline__ void kv4_store(WV& wv, Kv4Smem<D, HP, NW>& sm, const Pass1Args& a,
                                          bool direct, uint8_t* out, int64_t prow0,
                                          int64_t phstride, int hv, int w, int tid, int qh0) {
  const float l = WV::sum_head(wv.lsum);
  if (wv.r == 0 && WV::group(wv.c) == 0) {
    sm.m[w][WV::head(wv.c)] = wv.mref;
    sm.l[w][WV::head(wv.c)] = l;
  }
#pragma unroll
  for (int p = 0; p < WV::NH; ++p) {
    if constexpr (WV::PAIR) {
#pragma unroll
      for (int j = 0; j < WV::OV; j += 2) {
        const f32x4 x = wv.o[p][j], y = wv.o[p][j + 1];
        *reinterpret_cast<f32x4*>(&sm.o[w][wv.r][128 * p + wv.c * WV::JN + 2 * j]) =
            f32x4{x[0] + x[2], x[1] + x[3], y[0] + y[2], y[1] + y[3]};
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < WV::JN; j += 4)
          *reinterpret_cast<f32x4*>(&sm.o[w][4 * wv.r + i][128 * p + wv.c * WV::JN + j]) =
              f32x4{wv.o[p][j][i], wv.o[p][j + 1][i], wv.o[p][j + 2][i], wv.o[p][j + 3][i]};
    }
  }
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
      if constexpr (HP == 8) x += *reinterpret_cast<const f32x4*>(&sm.o[ww][8 + h][d]);
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

// Wavefronts per SIMD that the kernels are compiled for: two, but for D = 256 with 8 or 16 heads, whose
// accumulators and pages need more than 256 registers
template <int D, int HP>
constexpr int kv4_waves() { return D == 256 && HP > 4 ? 1 : 2; }

// Explicit split: workgroup = (head chunk, kv head, split, sequence), as dk_pass1_split
template <class T, int D, int HP, bool CAP, int NW>
__global__ __launch_bounds__(NW * 64, (kv4_waves<D, HP>())) void dk_kv4_split(Pass1Args a) {
  using WV = Kv4Wave<T, D, HP, CAP>;
  __shared__ Kv4Smem<D, HP, NW> sm;
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
  WV wv;
  wv.init(a, kvh);
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
  typename WV::Pages pages;
  if (n > 0) wv.start(a.indices + seq0 + p0, NW, w, n, pages);
  wv.load_q(a.q + (int64_t)b * a.q_b + (int64_t)qh0 * a.q_h, a.q_h, hv);
  wv.reset();
  const int lo = p0 == first_page ? first_tok : 0;
  const int hi = p0 + n == npages ? kPage * (n - 1) + last : kPage * n;
  wv.stream(NW, w, n, lo, hi, pages);
  kv4_store<T, D, HP, NW>(wv, sm, a, a.direct != 0,
                          a.out + (int64_t)b * a.o_b + (int64_t)qh0 * a.o_h,
                          ((int64_t)b * a.hq + qh0) * a.split + s, a.split, hv, w,
                          (int)threadIdx.x, qh0);
}

// The sequence that holds unit u of the linear (sequence, page) space: the largest b with
// start(b) <= u, by one wavefront's search over kv_indptr, 64 candidates per step (one dependent
// read up to 64 sequences, two up to 4096); every lane returns it.
__device__ __forceinline__ int kv4_sequence_of(const Pass1Args& a, int base, int u) {
  const int lane = threadIdx.x & 63;
  int lo = 0, S = a.batch;
  while (S > 1) {
    const int st = (S + 63) / 64;
    const bool in = lane * st < S;
    const int at = min(max(a.indptr[min(lo + lane * st, a.batch)], 0), a.num_indices) - base;
    const uint64_t m = __builtin_amdgcn_ballot_w64(in && at <= u);
    const int k = m ? 63 - __builtin_clzll(m) : 0;
    lo += k * st;
    S = min(st, S - k * st);
  }
  return uniform(lo);
}

// Balanced: the page ranges, segments and partial slots of dk_pass1_balanced (one kv head per
// workgroup; the range split that charges sequence starts when a.seg_cost > 0). A range's first pages
// are on their way while its first sequence is looked up.
template <class T, int D, int HP, bool CAP, int NW>
__global__ __launch_bounds__(NW * 64, (kv4_waves<D, HP>())) void dk_kv4_balanced(Pass1Args a, int heads) {
  using WV = Kv4Wave<T, D, HP, CAP>;
  __shared__ Kv4Smem<D, HP, NW> sm;
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
  const int kvh = hc % a.hkv, chunk = hc / a.hkv;
  WV wv;
  wv.init(a, kvh);
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
  const int qh0 = kvh * a.group + chunk * a.per;
  const int hv = min(a.per, a.group - chunk * a.per);
  typename WV::Pages pages;
  wv.start(a.indices + base + u, NW, w, u_end - u, pages);
  if (A == 0) b = kv4_sequence_of(a, base, u);
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
    const int hi = pg + n == np ? kPage * (n - 1) + last : kPage * n;
    wv.stream(NW, w, n, 0, hi, pages);
    // ranges holding this sequence's units
    const int start = seq0 - base, cur = b;
    int nslots;
    if (A == 0) {
      nslots = (start + np - 1) / L - start / L + 1;
    } else {
      const int64_t c0 = (int64_t)start + (int64_t)A * b;
      nslots = (int)((c0 + np - 1) / Lc - c0 / Lc + 1);
    }
    u += n;
    bool more = u < u_end;
    if (more) {                                // the next sequence's first pages
      do {
        ++b;
        seq0 = seq_begin(a, b);
        np = max(seq_begin(a, b + 1), seq0) - seq0;
      } while (np == 0 && b < a.batch - 1);
      more = np > 0;                           // else only for an invalid kv_indptr
      pg = 0;
    }
    kv4_store<T, D, HP, NW>(wv, sm, a, nslots == 1,
                            a.out + (int64_t)cur * a.o_b + (int64_t)qh0 * a.o_h,
                            ((int64_t)hc * (Wg + a.batch) + j + cur) * heads, 1, hv, w,
                            (int)threadIdx.x, qh0);
    if (!more) break;
    wv.start(a.indices + seq0, NW, w, min(np, u_end - u), pages);
  }
}

// Kernel symbols of one head_dim (dk_kv4.hip, compiled once per head_dim); hp 4, 8 or 16 q heads
template <int D>
const void* kv4_symbol(bool bf16, int hp, bool cap, int waves, bool balanced);
extern template const void* kv4_symbol<64>(bool, int, bool, int, bool);
extern template const void* kv4_symbol<128>(bool, int, bool, int, bool);
extern template const void* kv4_symbol<256>(bool, int, bool, int, bool);

}  // namespace dk
