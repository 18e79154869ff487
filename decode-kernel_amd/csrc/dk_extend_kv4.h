// dk_extend_kv4.h — extend (prefill) attention over a 4-bit cache (dk_kv4.h), gfx950, wave64.
//
// dk_extend.h's mathematics (S^T = K.Q^T, O^T += V^T.P^T, 128 query rows of one kv head per workgroup,
// 32 per wavefront), over page blocks found through a block table:
//   * q.k on v_mfma_scale_f32_32x32x64_f8f6f4, at four times the rate of 16-bit operands: K's codes and
//     scales as they lie in the page, q as 3 parts of E2M3 with scales of their own, so three quarters
//     of the 16-bit time, a quarter of the LDS traffic and no widening (2048 new of 8192 tokens, fp16
//     322 -> 298 us; with K widened to q's type);
//   * V is widened to q's type on its way into LDS, in pieces between the last P.V products of the tile
//     before, whose MFMAs leave the VALU free; a wavefront loads a page's 17 D bytes a tile ahead;
//   * a tile's A operands are read from LDS several steps ahead of the MFMA that takes them, and its
//     two 32-key blocks are staggered: the second's weights are formed beside the first's products;
//   * LDS rows are padded rather than swizzled: 16 rows' 16-byte chunks (K) and 4 rows' 64-byte runs
//     (V, transpose reads) lie in different banks, and every address is a base and a constant;
//   * a weight enters as two parts of q's type: 22 bits in fp16 (ExtendParts<F16>), in bf16 16, off by
//     at most 2^-16 of itself where the output's own rounding is 2^-8 (a third part takes 1e-6 off the
//     error of the norm and costs 12 %).
// Bound by the card's power where a call is long: the clock settles at 1.6 to 2.0 GHz, and a variant
// with a third less MFMA work was only 16 % faster, one without exponentials 7 %. 32/8/128, 2048 new of
// 8192 tokens, us: fp16 298, bf16 291 (dk_extend over 16-bit rows 376, 441). 8 requests of 79-730 new
// tokens over up to 500 (32/8/64 bf16) 37.8: bound by the VALU, 1.0 us per workgroup and 64-key tile on a
// CU that holds three, and by the longest workgroup, 16 tiles of 1.75 us each. Tiles dealt to the
// workgroups that the chip holds (ExtendKv4Args) against one workgroup per tile: 38.6 and 42.6 there,
// one request of 2048 tokens (32/8/128 fp16) 65.3 and 67.8.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dk_extend.h"
#include "dk_kv4.h"

namespace dk {

constexpr int kKv4ExtendOrder = 256;  // query tiles that a call deals out itself (ExtendKv4Args)

// E2M3 parts of q (QParts): what 3 leave of an element is at most 2^-15 of the power of two below its 32
// dims' largest magnitude. bf16 is whole down to 2^-7 of that, fp16 down to 2^-4, and what smaller
// elements lose is a sixteenth of the largest one's own rounding. A fourth part for fp16 (as in decode,
// which waits for memory) costs 4.5 %: 312 us against 298 for 2048 new of 8192 tokens.
constexpr int kKv4ExtendQParts = 3;

// Workgroups that a CU holds at once
constexpr int kv4_extend_resident(int d, bool cap) { return d == 64 ? (cap ? 2 : 3) : d == 128 ? 2 : 1; }

struct ExtendKv4Args {
  ExtendArgs e;                         // k: the page pool, k_h: its kv heads' stride, req_to_token:
                                        // page ids, num_slots: pages; vscale: undoes kv4_stage_exp
  int64_t kv_p;                         // bytes between pages
  // dealt != 0: a workgroup takes the query tiles list[start[i]] .. list[start[i + 1] - 1] of its
  // head, i = its index in the grid; a tile: request * kKv4ExtendOrder + its n-th tile
  int32_t dealt;
  uint16_t list[kKv4ExtendOrder], start[kKv4ExtendOrder + 1];
};

// V is staged in q's type, in fp16 at half its size (exact, the factor returned by the output's
// scale): E2M1's 6 times the largest scale of an fp16 value, 4 * 2^14, is past
// fp16's range.
template <class T>
constexpr int kv4_stage_exp() { return __is_same(T, F16) ? 1 : 0; }
// A float whose exponent field is an E8M0 byte (other bits arbitrary), halved for fp16; the NaN byte stays
template <class T>
__device__ __forceinline__ u32 kv4_stage_scale(u32 sc) {
  if constexpr (kv4_stage_exp<T>() == 0) return sc;
  return __builtin_bit_cast(u32, __builtin_bit_cast(float, sc) * 0.5f);
}

// f(Index<0>{}) .. f(Index<N - 1>{})
template <int I>
struct Index {
  static constexpr int value = I;
};
template <int N, int I = 0, class F>
__device__ __forceinline__ void for_each(F&& f) {
  if constexpr (I < N) {
    f(Index<I>{});
    for_each<N, I + 1>(f);
  }
}

// x less half H of a packed pair, exact where the half is x rounded: one instruction each
template <int H>
__device__ __forceinline__ float less(F16, float x, u32 pair) {
  float r;
  if constexpr (H == 0)
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(pair), "v"(x));
  else
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(pair), "v"(x));
  return r;
}
template <int H>
__device__ __forceinline__ float less(BF16, float x, u32 pair) {
  u32 minus;   // -1 and 0, in a register: an inline -1.0 is an fp32 one
  if constexpr (H == 0) asm("s_mov_b32 %0, 0xbf80" : "=s"(minus));
  else asm("s_mov_b32 %0, 0xbf800000" : "=s"(minus));
  return BF16::dot2(pair, minus, x);
}

// C += A.B: A 32 keys x 64 dims of E2M1, B 64 dims x 32 rows of E2M3; lane half h holds dims 32 h .. of
// both. Byte GA of sa / GB of sb: the E8M0 scale of the lane's key / row for those 32.
template <int GA, int GB>
__device__ __forceinline__ f32x16 mfma_mx32(u32x4 a, u32x6 b, f32x16 c, u32 sa, u32 sb) {
  const i32x8 av = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8 bv = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], (int)b[4], (int)b[5], 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, c, 4, 2, GA, (int)sa, GB, (int)sb);
}

// 32 values of q (16 words) as QP parts of E2M3 and their scales' bytes (QParts; a block with a NaN
// or an infinity gets the NaN scale)
template <class T, int QP>
__device__ __forceinline__ void q_parts(const u32 (&w)[16], u32x6 (&part)[QP], u32* scales) {
  f32x16v lo, hi;                                // even and odd dims
  u32 top = 0u;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float x, y;
    if constexpr (__is_same(T, F16)) {
      const f16x2 v = __builtin_bit_cast(f16x2, w[i]);
      x = (float)v[0];
      y = (float)v[1];
    } else {
      x = __builtin_bit_cast(float, w[i] << 16);
      y = __builtin_bit_cast(float, w[i] & 0xffff0000u);
    }
    lo[i] = x;
    hi[i] = y;
    top = max(top, max(__builtin_bit_cast(u32, x) & 0x7fffffffu, __builtin_bit_cast(u32, y) & 0x7fffffffu));
  }
  const int ex = top == 0u ? 127 : max((int)(top >> 23), q_part_exp(QP - 1) + 1);
  *scales = 0u;
  for_each<QP>([&](auto ic) {
    constexpr int i = ic.value;
    const float sc = __builtin_bit_cast(float, (u32)(min(ex, 254) - q_part_exp(i)) << 23);
    const u32x6 q6 = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(lo, hi, sc);
    asm volatile("" ::"v"(lo), "v"(hi), "v"(sc), "v"(q6));   // no shared register (Kv4Wave::load_q)
    part[i] = q6;
    *scales |= (u32)(ex == 255 ? 255 : ex - q_part_exp(i)) << (8 * i);
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

template <class T, int D, bool CAP>
__global__ __launch_bounds__(kExtendThreads, (kv4_extend_resident(D, CAP))) void dk_extend_kv4(ExtendKv4Args ka) {
  const ExtendArgs& a = ka.e;
  constexpr int NB = D <= 128 ? 2 : 1;            // 32-key blocks per tile
  constexpr int BN = 32 * NB;
  // Bytes per LDS row, padded so that 16 rows' chunks of 16 bytes (K) and 4 rows' runs of 64 (V) fall
  // into different banks: every offset is then a constant of the instruction
  constexpr int DB = D / 32;                      // 32-dim blocks
  constexpr int KB = D / 2 + 16, VB = 2 * D + 64;
  constexpr int KS = BN * KB, KT = KS + BN * DB;   // K's scales (DB bytes per key), V's tile
  constexpr int BUF = KT + BN * VB;
  constexpr int KM = D / 64;                      // 64-dim parts of a row
  constexpr int QP = kKv4ExtendQParts;
  constexpr int PV = D / 16;                      // steps of a 32-key block's V: 16 keys x 32 dims
  constexpr int kAhead = D > 64 ? 4 : __is_same(T, BF16) ? 3 : 2;   // what the registers hold
  constexpr int WP = D == 256 ? 2 : 1;            // wavefronts that stage a page, 128 dims (64) each
  constexpr int BW = D == 64 ? 2 : 4;             // words of a lane's K codes and V codes
  __shared__ __attribute__((aligned(16))) uint8_t smem[2 * BUF];
  // NaN values (V's NaN scale) are staged as zeros, as 0 * NaN would reach the queries that do not
  // attend to them; which 32-dim blocks of which tokens they were lies here, by the wavefront that
  // staged them and where its entry of nan_tile names the tile (its number + 1)
  __shared__ u32 nan_tile[2][4], nan_blocks[2][4][kPage];

  // workgroup -> (kv head, query tile): the kv head is fastest, so with 8 kv heads every XCD
  // streams one head and its L2 holds that head's K and V for all tiles of a request
  const int kvh = (int)blockIdx.x % a.hkv;
  const int t = (int)blockIdx.x / a.hkv;
  int entry = ka.dealt ? ka.start[t] : 0;
  const int entries = ka.dealt ? ka.start[t + 1] : 1;
  do {
  // the lane's places, formed again for each tile: held from one to the next they would spill
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  const int lane = tid & 63, w = uniform(tid >> 6);
  const int h = lane >> 5, c = lane & 31;
  int lo = 0, nth;                     // the request, and which of its tiles
  if (ka.dealt) {
    lo = ka.list[entry] / kKv4ExtendOrder;
    nth = ka.list[entry] % kKv4ExtendOrder;
  } else {
    int hi = a.num_reqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.req[mid].tile0 <= t) lo = mid; else hi = mid - 1;
    }
    nth = t - a.req[lo].tile0;
  }
  const ExtendReq rq = a.req[lo];
  const int G = a.group, rows = rq.n_new * G;
  // the last tiles of a request see the most keys: they start first
  const int ntile = (rows + kExtendRows - 1) / kExtendRows;
  const int row0 = (ntile - 1 - nth) * kExtendRows;
  const int prefix = rq.n_all - rq.n_new;

  const int rr = min(row0 + 32 * w + c, rows - 1);               // this lane's row of q
  const int pos = prefix + rr / G;                               // and its position
  // key range of the workgroup and of this wavefront (uniform)
  const int wrow = min(row0 + 32 * w, rows - 1);
  const int wpos0 = prefix + wrow / G, wpos1 = prefix + min(row0 + 32 * w + 31, rows - 1) / G;
  const bool active = row0 + 32 * w < rows;
  const int bpos0 = prefix + row0 / G, bpos1 = prefix + min(row0 + kExtendRows - 1, rows - 1) / G;
  const int win = a.window > 0 ? a.window : INT32_MAX;
  int kbeg = max(bpos0 - win + 1, 0) / BN;
  int kend = bpos1 / BN + 1;
  if (a.split > 1) {                   // this workgroup's range of key tiles (may be empty)
    const int per = (kend - kbeg + a.split - 1) / a.split;
    kbeg += (int)blockIdx.y * per;
    kend = min(kbeg + per, kend);
  }

  // q as E2M3 parts (QParts), lane (h, c): dims 64 m + 32 h .. of row c
  u32x6 qf[KM][QP];
  u32 qs[KM];                          // their scales, a byte each
  {
    const uint8_t* qp = a.q + (int64_t)(rq.q0 + rr / G) * a.q_b +
                        (int64_t)(kvh * G + rr % G) * a.q_h + 64 * h;
#pragma unroll
    for (int m = 0; m < KM; ++m) {
      u32 words[16];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(qp + 128 * m + 16 * i);
        words[4 * i] = x[0];
        words[4 * i + 1] = x[1];
        words[4 * i + 2] = x[2];
        words[4 * i + 3] = x[3];
      }
      q_parts<T, QP>(words, qf[m], &qs[m]);
    }
  }

  // ---- loads: wavefront w takes page pg of the tile, part sp of its dims. Lane (sr, st): block sr
  // (D = 64: half of one) of K token st, and dims st * W / 16 .. of V tokens 4 sr .. 4 sr + 3.
  const int32_t* map = a.req_to_token + (int64_t)rq.row * a.req_stride;
  const uint8_t* kbase = a.k + (int64_t)kvh * a.k_h;
  const int pg = w / WP, sp = w % WP, st = lane & 15, sr = lane >> 4;
  const int last_block = (rq.n_all - 1) / kPage;
  int page = 0;                       // id that the table holds for the tile loaded next
  bool bad = false;                   // the loaded page's id lies outside the pool
  u32 kr[BW], vr[BW];
  u32 ksc, vsc;                       // K's scale, V's 4 scales
  const u32 k_off = st * (D / 2) + 64 * sp + 4 * BW * sr;
  const u32 v_off = kv4_v_at(D) + 1024 * sp + 4 * BW * lane;
  const u32 ks_off = kv4_ks_at(D) + 16 * (D == 64 ? sr / 2 : 4 * sp + sr) + st;
  const u32 vs_off = kv4_vs_at(D) + 16 * (D == 64 ? st / 8 : 4 * sp + st / 4) + 4 * sr;
  auto load_id = [&](int j) { page = map[min(j * (BN / kPage) + pg, last_block)]; };
  auto load_tile = [&]() {            // outside the pool page 0 is read instead
    bad = (uint32_t)uniform(page) >= a.num_slots;
    const uint8_t* blk = kbase + (int64_t)(bad ? 0 : uniform(page)) * ka.kv_p;
    typedef u32 Run __attribute__((ext_vector_type(BW)));
    const Run kw = *reinterpret_cast<const Run*>(blk + k_off);
    const Run vw = *reinterpret_cast<const Run*>(blk + v_off);
#pragma unroll
    for (int x = 0; x < BW; ++x) {
      kr[x] = kw[x];
      vr[x] = vw[x];
    }
    ksc = blk[ks_off];
    vsc = *reinterpret_cast<const u32*>(blk + vs_off);
  };
  // keys past the request's last are zeros; a page outside the pool has K = NaN and V = 0, so that
  // every query that attends to it gives NaN. By the scales: codes of +-0 for a zero, the NaN scale.
  auto any_nan = [&]() {              // some scale of V is the NaN byte (a zero byte of its inverse)
    return __builtin_amdgcn_ballot_w64(((~vsc - 0x01010101u) & vsc & 0x80808080u) != 0u) != 0u;
  };
  auto fix_tile = [&](int j, int buf) {
    const int key = j * BN + pg * kPage;
    const bool gone = key + st >= rq.n_all;
    u32* const blocks = nan_blocks[buf != 0][w];
    blocks[st] = 0u;
    bool found = false;
#pragma unroll
    for (int x = 0; x < BW; ++x) kr[x] = gone ? 0u : kr[x];
    ksc = gone ? 127u : bad ? 255u : ksc;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      bool out = bad || key + 4 * sr + x >= rq.n_all;
      if (!out && (vsc >> (8 * x) & 255u) == 255u) {
        atomicOr(&blocks[4 * sr + x], 1u << (D == 64 ? st / 8 : 4 * sp + st / 4));
        out = found = true;
      }
      vsc = out ? (vsc & ~(0xffu << (8 * x))) | 127u << (8 * x) : vsc;
      if constexpr (D == 64)
        vr[x / 2] = out ? vr[x / 2] & (x & 1 ? 0xffffu : 0xffff0000u) : vr[x / 2];
      else
        vr[x] = out ? 0u : vr[x];
    }
    if (__builtin_amdgcn_ballot_w64(found)) nan_tile[buf != 0][w] = (u32)j + 1u;
  };
  // Staging, in pieces: K's codes and scale as they are, V's 4 tokens
  constexpr int PIECES = 5;
  uint8_t* const kput = smem + (pg * kPage + st) * KB + 64 * sp + 4 * BW * sr;
  uint8_t* const ksput = smem + KS + (pg * kPage + st) * DB + (D == 64 ? sr / 2 : 4 * sp + sr);
  uint8_t* const vput = smem + KT + (pg * kPage + 4 * sr) * VB + 256 * sp + (D == 64 ? 8 : 16) * st;
  auto store_piece = [&](auto piece, int buf) {
    constexpr int p = decltype(piece)::value;
    if constexpr (p == 0) {
      typedef u32 Run __attribute__((ext_vector_type(BW)));
      Run x;
#pragma unroll
      for (int i = 0; i < BW; ++i) x[i] = kr[i];
      *reinterpret_cast<Run*>(kput + buf) = x;
      ksput[buf] = (uint8_t)ksc;
    } else {
      constexpr int x = p - 1;
      const u32 sc = kv4_stage_scale<T>(e8m0_exp<x>(vsc));
      if constexpr (D == 64) {
        const u32 v = vr[x / 2] >> (16 * (x & 1));
        *reinterpret_cast<u32x2*>(vput + buf + x * VB) =
            u32x2{from_fp4<T, 0>(v, sc), from_fp4<T, 1>(v, sc)};
      } else {
        *reinterpret_cast<u32x4*>(vput + buf + x * VB) =
            u32x4{from_fp4<T, 0>(vr[x], sc), from_fp4<T, 1>(vr[x], sc), from_fp4<T, 2>(vr[x], sc),
                  from_fp4<T, 3>(vr[x], sc)};
      }
    }
  };
  auto store_tile = [&](int buf) {
    for_each<PIECES>([&](auto p) { store_piece(p, buf); });
  };

  f32x16 o[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[b][i] = 0.f;
  float mref = kMinit, lsum = 0.f;
  u32 nans = 0u;                      // 32-dim blocks in which this row attends to a NaN

  // this lane's places in the tiles it reads (dk_extend.h)
  const uint8_t* const kget = smem + c * KB + 16 * h;
  const uint8_t* const ksget = smem + KS + c * DB;
  const uint8_t* const vget = smem + KT + (4 * h + ((lane & 15) >> 2)) * VB +
                              32 * ((lane >> 4) & 1) + 8 * (lane & 3);

  // A operands: 64 dims (part m) of block n's keys, and their scales (byte 0: 64 m + 32 h .. of an even
  // m, byte 2 of an odd one); 16 keys' 32 dims (step y of PV) of its V
  auto read_k = [&](int n, int m, int buf) {
    return *reinterpret_cast<const u32x4*>(kget + buf + 32 * n * KB + 32 * m);
  };
  auto read_ks = [&](int n, int buf, u32 (&sc)[(KM + 1) / 2]) {
    const uint8_t* p = ksget + buf + 32 * n * DB;
    if constexpr (D == 64) {
      sc[0] = (u32)*reinterpret_cast<const uint16_t*>(p) >> (8 * h);
    } else {
#pragma unroll
      for (int i = 0; i < KM / 2; ++i) sc[i] = reinterpret_cast<const u32*>(p)[i] >> (8 * h);
    }
  };
  auto read_v = [&](int n, int y, int buf) {
    const uint8_t* vp = vget + buf + (32 * n + 16 * (y / DB)) * VB + 64 * (y % DB);
    const u32x2 v0 = lds_read_tr(vp), v1 = lds_read_tr(vp + 8 * VB);
    return u32x4{v0[0], v0[1], v1[0], v1[1]};
  };
  // pair x (0..7) of a block's weights in this lane, split into two parts
  auto weigh = [&](int x, const f32x16& s, u32x4 (&pp)[2][2]) {
    float r0 = __builtin_amdgcn_exp2f(CAP ? s[2 * x] - mref : __builtin_fmaf(s[2 * x], a.kscale, -mref));
    float r1 = __builtin_amdgcn_exp2f(CAP ? s[2 * x + 1] - mref
                                          : __builtin_fmaf(s[2 * x + 1], a.kscale, -mref));
    lsum += r0 + r1;
    float t0, t1;
    const u32 top = T::pack2(r0, r1, &t0, &t1);
    pp[x / 4][0][x % 4] = top;
    pp[x / 4][1][x % 4] = T::pack2(less<0>(T{}, r0, top), less<1>(T{}, r1, top), &t0, &t1);
    // computed here, beside the MFMAs around, and not where it is used first
    asm volatile("" : "+v"(pp[x / 4][0][x % 4]), "+v"(pp[x / 4][1][x % 4]), "+v"(lsum));
  };
  auto pv = [&](int y, u32x4 vf, const u32x4 (&pp)[2][2]) {
    o[y % DB] = mfma32(T{}, vf, pp[y / DB][0], o[y % DB]);
    o[y % DB] = mfma32(T{}, vf, pp[y / DB][1], o[y % DB]);
  };
  // cap and mask of a block's scores; what its keys mean for `nans`
  auto mask = [&](int k0, f32x16& s, uint64_t nan_pages, int buf) {
    if constexpr (CAP) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = a.cap_out * tanhf(s[i] * a.cap_in);
    }
    if (k0 + 31 > wpos0) {
      const int rel = pos - k0 - 4 * h;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = 8 * (i / 4) + i % 4 > rel ? kNegInf : s[i];
    }
    if (k0 <= wpos1 - win) {
      const int rel = pos - win - k0 - 4 * h;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = 8 * (i / 4) + i % 4 <= rel ? kNegInf : s[i];
    }
    if (nan_pages) {
      u32 seen = 0u;
#pragma unroll
      for (int i = 0; i < 16; ++i) seen |= s[i] != kNegInf ? 1u << i : 0u;
#pragma unroll 1
      for (int i = 0; i < 16; ++i) {
        const int key = (k0 & (BN - 1)) + 8 * (i / 4) + 4 * h + i % 4;
#pragma unroll
        for (int x = 0; x < WP; ++x) {
          const int from = key / kPage * WP + x;
          if (nan_pages >> from & 1)
            nans |= seen >> i & 1u ? nan_blocks[buf != 0][from][key % kPage] : 0u;
        }
      }
    }
  };
  auto top_of = [&](const f32x16& s) {
    float mx = kNegInf;
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[i]);
    return mx;
  };
  // mx, of this lane's scores: the row's; true: the reference has to move
  auto moves = [&](float* mx) -> bool {
    *mx = max_xor32(*mx);
    if constexpr (!CAP) *mx *= a.kscale;
    const bool move = ExtendParts<T>::n == 2 ? fabsf(*mx - (mref + kExtendTop / 2)) > kExtendTop / 2
                                             : *mx > mref + kSlack;
    return __builtin_amdgcn_ballot_w64(move);
  };
  auto move_ref = [&](float mx) {
    float mn = fmaxf(mref, mx);
    if constexpr (ExtendParts<T>::n == 2) {   // the reference follows the blocks (ExtendParts<F16>)
      const float to = mx - (mx > mref + kExtendTop + kExtendMid ? kExtendJump : kExtendMid);
      const float room = __builtin_amdgcn_logf(sum_xor32(lsum)) - kExtendRoom;   // log2
      mn = mx > kNegInf ? fmaxf(to, mref + room) : mref;   // no key of the block seen: stays
    }
    const float al = __builtin_amdgcn_exp2f(mref - mn);
    lsum *= al;
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[b][i] *= al;
    mref = mn;
  };
  auto pin = [] { __builtin_amdgcn_sched_barrier(0x4); };   // scalar code may cross

  load_id(kbeg);
  load_tile();
  load_id(kbeg + 1);
  if (lane < 2) nan_tile[lane][w] = 0u;
  if ((kbeg + 1) * BN > rq.n_all || bad || any_nan()) fix_tile(kbeg, 0);
  store_tile(0);
  __syncthreads();
  for (int j = kbeg; j < kend; ++j) {
    const int buf = (j - kbeg) & 1 ? BUF : 0;
    auto fix = [&] {
      if ((j + 2) * BN > rq.n_all || bad || any_nan()) fix_tile(j + 1, BUF - buf);
    };
    // a wavefront whose rows see none of the tile's keys skips it
    if (active && j * BN <= wpos1 && j * BN + BN - 1 > wpos0 - win) {
      const uint64_t nan_pages =
          __builtin_amdgcn_ballot_w64(nan_tile[buf != 0][lane & 3] == (u32)j + 1u) & 15u;
      f32x16 s0, s1;
      u32x4 p0[2][2], p1[2][2];
      float mx;
      // the tile's A operands, read kAhead steps before their use: all keys, then all values
      u32x4 ahead[kAhead];
      u32 ks0[(KM + 1) / 2], ks1[(KM + 1) / 2];
      auto fetch = [&](int g) {
        if (g < NB * (KM + PV))
          ahead[g % kAhead] = g < NB * KM ? read_k(g / KM, g % KM, buf)
                                          : read_v((g - NB * KM) / PV, (g - NB * KM) % PV, buf);
      };
      read_ks(0, buf, ks0);
      if constexpr (NB == 2) read_ks(1, buf, ks1);
#pragma unroll
      for (int g = 0; g < kAhead; ++g) fetch(g);
      load_tile();                    // after the last tile a page of the request again, for nobody
      load_id(j + 2);
      for_each<NB * KM>([&](auto g) {
        constexpr int n = g.value / KM, m = g.value % KM;
        f32x16& x = n ? s1 : s0;
        const u32 sc = n ? ks1[m / 2] : ks0[m / 2];
        for_each<QP>([&](auto i) {
          x = mfma_mx32<2 * (m % 2), i.value>(ahead[g.value % kAhead], qf[m][i.value],
                                              m || i.value ? x : f32x16{}, sc, qs[m]);
        });
        fetch(g.value + kAhead);
        pin();
      });
      mask(j * BN, s0, nan_pages, buf);
      mx = top_of(s0);
      if constexpr (NB == 2) {
        mask(j * BN + 32, s1, nan_pages, buf);
        mx = fmaxf(mx, top_of(s1));
      }
      if (moves(&mx)) move_ref(mx);
      for_each<8>([&](auto x) { weigh(x.value, s0, p0); });
      pin();
      if constexpr (NB == 2) {
        // the first block's V products beside the second's weights
        for_each<8>([&](auto x) {
#pragma unroll
          for (int y = x.value * PV / 8; y < (x.value + 1) * PV / 8; ++y) {
            pv(y, ahead[(NB * KM + y) % kAhead], p0);
            fetch(NB * KM + y + kAhead);
          }
          weigh(x.value, s1, p1);
          pin();
        });
      }
      // the last block's V products beside the staging of the next tile
      fix();
      for_each<PIECES>([&](auto p) {
        constexpr int at = NB * KM + (NB - 1) * PV;
#pragma unroll
        for (int y = p.value * PV / PIECES; y < (p.value + 1) * PV / PIECES; ++y) {
          pv(y, ahead[(at + y) % kAhead], NB == 2 ? p1 : p0);
          fetch(at + y + kAhead);
        }
        store_piece(p, BUF - buf);
        pin();
      });
    } else {
      load_tile();
      load_id(j + 2);
      fix();
      store_tile(BUF - buf);
    }
    __syncthreads();
  }

  if (__builtin_amdgcn_ballot_w64(nans != 0u)) {
    nans |= (u32)__shfl_xor((int)nans, 32);
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[b][i] = nans >> b & 1u ? __builtin_nanf("") : o[b][i];
  }
  lsum = sum_xor32(lsum);
  // this lane's row again: held over the loop it would cost registers that spill
  int base = row0;
  asm volatile("" : "+s"(base));
  const int row = base + 32 * w + c, tok = min(row, rows - 1) / G, head = min(row, rows - 1) - tok * G;
  if (a.split > 1) {
    // relative to this range's reference; dk_merge_split adds the sinks and normalises
    if (row < rows) {
      const int64_t r = ((int64_t)(rq.q0 + tok) * (a.hkv * G) + kvh * G + head) * a.split +
                        blockIdx.y;
#pragma unroll
      for (int b = 0; b < DB; ++b)
#pragma unroll
        for (int x = 0; x < 4; ++x)
          *reinterpret_cast<f32x4*>(a.part_o + r * D + 32 * b + 8 * x + 4 * h) =
              f32x4{o[b][4 * x] * a.vscale, o[b][4 * x + 1] * a.vscale, o[b][4 * x + 2] * a.vscale,
                    o[b][4 * x + 3] * a.vscale};
      if (h == 0) {
        a.part_m[r] = mref * kLn2;
        a.part_l[r] = lsum;
      }
    }
    return;                            // such a call deals nothing out
  }
  if (a.sinks) lsum += __builtin_amdgcn_exp2f(a.sinks[kvh * G + head] * kLog2e - mref);
  const float inv = lsum == 0.f ? 0.f : a.vscale / lsum;
  if (row < rows) {
    uint8_t* op = a.out + (int64_t)(rq.q0 + tok) * a.o_b + (int64_t)(kvh * G + head) * a.o_h;
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        float e0, e1;
        const u32x2 v = {T::pack2(o[b][4 * x] * inv, o[b][4 * x + 1] * inv, &e0, &e1),
                         T::pack2(o[b][4 * x + 2] * inv, o[b][4 * x + 3] * inv, &e0, &e1)};
        *reinterpret_cast<u32x2*>(op + 2 * (32 * b + 8 * x + 4 * h)) = v;
      }
  }
  } while (++entry < entries);
}

// Kernel symbol of one head_dim (dk_extend_kv4.hip, compiled once per head_dim)
template <int D>
const void* extend_kv4_symbol(bool bf16, bool cap);
extern template const void* extend_kv4_symbol<64>(bool, bool);
extern template const void* extend_kv4_symbol<128>(bool, bool);
extern template const void* extend_kv4_symbol<256>(bool, bool);

}  // namespace dk
