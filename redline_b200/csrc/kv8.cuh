// What the kernels of the 8-bit cache share: its format, conversions, and how a launch's keys are shared out.
//
// A page of one kv head holds page_size rows of kD e4m3 bytes and has one scale for its keys and one for its values,
// a power of two kept as its exponent plus 127 (e8m0).  A block x is stored as x / 2^e rounded to e4m3, 2^e the smallest
// power of two with max |x| <= 448 * 2^e.  A power of two and no other number, because then
//   - raising the scale of a page that has room left rescales the bytes that are in it exactly (but for numbers that fall
//     below e4m3's normal range, which are off by at most 2^-10 of the unit, 2^-18 of the block's largest), so that what is
//     stored hardly depends on how the tokens were cut into steps;
//   - the values that the bytes stand for are numbers of 4 significant bits: exact in bfloat16, half and float.
// An e4m3 number has its 3 bits of mantissa at any size, so a scale between two powers would gain nothing.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace rl {

constexpr int kKv8MaxPage = 64;

// 2^e for -127 <= e <= 127, by its bits.
__device__ __forceinline__ float kv8_exp2i(int e) {
  return e >= -126 ? __uint_as_float(static_cast<uint32_t>(e + 127) << 23) : __uint_as_float(0x00400000u);
}
// The value of a scale's byte: 2^(code - 127); 255 is not a number in e8m0.
__device__ __forceinline__ float kv8_scale(int code) {
  return code == 255 ? __uint_as_float(0x7fc00000u) : kv8_exp2i(code - 127);
}
// The byte of the scale of a block whose largest finite magnitude is `amax`: the smallest power of two 2^e with
// amax <= 448 * 2^e = 1.75 * 2^(e + 8).  At least 2^-126 (a normal float) and at most 2^119, for which 448 * 2^e is
// still finite: a block of larger numbers saturates.
__device__ __forceinline__ int kv8_code(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int code = static_cast<int>(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(code, 1), 246);
}

// Two e4m3 bytes (the low one first) as two halves: exact.
__device__ __forceinline__ uint32_t kv8_h2(uint32_t two) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(two)));
  return h;
}
// Four e4m3 bytes as two words of two halves.
__device__ __forceinline__ void halves4(uint32_t four, uint32_t& lo, uint32_t& hi) {
  asm("{\n"
      ".reg .b16 a, b;\n"
      "mov.b32 {a, b}, %2;\n"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n"
      "cvt.rn.f16x2.e4m3x2 %1, b;\n"
      "}\n"
      : "=r"(lo), "=r"(hi)
      : "r"(four));
}
__device__ __forceinline__ uint32_t pack_halves(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Four e4m3 bytes as floats.
__device__ __forceinline__ void kv8_f4(uint32_t four, float* f) {
  const uint32_t a = kv8_h2(four), b = kv8_h2(four >> 16);
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a)), y = __half22float2(*reinterpret_cast<const __half2*>(&b));
  f[0] = x.x;
  f[1] = x.y;
  f[2] = y.x;
  f[3] = y.y;
}
__device__ __forceinline__ void kv8_f16(uint4 v, float* f) {
  kv8_f4(v.x, f);
  kv8_f4(v.y, f + 4);
  kv8_f4(v.z, f + 8);
  kv8_f4(v.w, f + 12);
}
// Two floats rounded to e4m3 (to nearest, ties to even; beyond 448: 448), the first in the low byte.
__device__ __forceinline__ uint32_t kv8_pack2(float lo, float hi) {
  uint16_t d;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ uint32_t kv8_pack4(const float* f) { return kv8_pack2(f[0], f[1]) | kv8_pack2(f[2], f[3]) << 16; }

// A page id of a block table, if the pool has such a page; else page 0, the one that belongs to nobody, and `bad` is set.
__device__ __forceinline__ int kv8_page(int page, int pages, bool& bad) {
  const bool in = static_cast<unsigned>(page) < static_cast<unsigned>(pages);
  bad |= !in;
  return in ? page : 0;
}

constexpr int kKv8BadPage = 16;      // the bit of the tcgen05 kernels' status that a page id beyond the pool sets

// ---- rows by a warp: without the limits of the kernels that are built for speed, for the rows that meet them
//
// R query rows over the keys of one kv head of a sequence, in float32 throughout: scores by exponents of q and the page apart, values as
// they are, a key that a row does not see not looked at.  Lane i has the entries i E .. of every row.  Four keys at a time: their 4 R
// partial products meet in 31 shuffles (every step leaves a lane half of the values), so that a score, its weight and its row's m and l
// are one lane's (row_of, key_of); the weights go round for the values.  (A row at a time, with five shuffles and every lane's exponentials for
// each key: 333 rows behind 1,000 keys 10.7 ms.)
template <int D>
struct Kv8Rows {
  static constexpr int E = D <= 32 ? 1 : D <= 64 ? 2 : D <= 128 ? 4 : 8;
  static constexpr int R = E <= 2 ? 8 : E == 4 ? 4 : 2;
  static constexpr int L = 8 / R;                          // lanes that have the same score
  static __device__ __forceinline__ bool in_head(int lane) { return lane * E < D; }
  static __device__ __forceinline__ int row_of(int lane) { return lane / (4 * L); }
  static __device__ __forceinline__ int key_of(int lane) { return lane / L & 3; }
};

template <int E>
__device__ __forceinline__ void kv8_row_load(const uint8_t* p, float* f) {
  if constexpr (E == 1) {
    const uint32_t h = kv8_h2(*p);
    f[0] = __low2float(*reinterpret_cast<const __half2*>(&h));
  } else if constexpr (E == 2) {
    const uint32_t h = kv8_h2(*reinterpret_cast<const uint16_t*>(p));
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h));
    f[0] = x.x;
    f[1] = x.y;
  } else {
#pragma unroll
    for (int e = 0; e < E; e += 4) kv8_f4(*reinterpret_cast<const uint32_t*>(p + e), f + e);
  }
}

// Keys [lo, hi) of the lane's row (none: lo = hi).  q comes as it is and is lost; the numerators are left in o, relative to 2^m, the lane's
// row's reference (log2 units, as c is), and l is that row's denominator.
template <int D, typename Args>
__device__ __forceinline__ void kv8_rows(const Args& a, int seq, int kvh, int lo, int hi, float c, int lane,
                                         float (&q)[Kv8Rows<D>::R][Kv8Rows<D>::E], float (&o)[Kv8Rows<D>::R][Kv8Rows<D>::E], float& m, float& l) {
  constexpr int E = Kv8Rows<D>::E, R = Kv8Rows<D>::R, L = Kv8Rows<D>::L;
  const bool in = Kv8Rows<D>::in_head(lane);
  const int mine = Kv8Rows<D>::row_of(lane), u_mine = Kv8Rows<D>::key_of(lane);
  const uint8_t *kc = reinterpret_cast<const uint8_t*>(a.kcache), *vc = reinterpret_cast<const uint8_t*>(a.vcache);
  const int32_t* bt = a.block_table + static_cast<size_t>(seq) * a.max_blocks;
  int ex = 0;                                              // of the lane's row: its largest entry is 1.f * 2^ex
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float amax = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      amax = fmaxf(amax, in ? fabsf(q[r][e]) : 0.f);
      o[r][e] = 0.f;
    }
    amax = warp_max(amax);
    const int x = amax > 0.f && amax < INFINITY ? ilogbf(amax) : 0;
    if (r == mine) ex = x;
#pragma unroll
    for (int e = 0; e < E; ++e) q[r][e] = in ? ldexpf(q[r][e], -x) : 0.f;
  }
  m = -INFINITY;
  l = 0.f;
  const int end = __reduce_max_sync(0xffffffffu, hi), begin = __reduce_min_sync(0xffffffffu, lo < hi ? lo : 0x7fffffff);
#pragma unroll 1
  for (int j0 = begin & ~15; j0 < end; j0 += 16) {         // 16 keys of one page
    bool bad = false;                                      // (told by whoever went over the keys before)
    const size_t block = static_cast<size_t>(kv8_page(bt[j0 >> a.page_shift], a.pages, bad)) * a.hkv + kvh;
    const int kcode = a.kscale[block], e2 = max(ex + kcode - 127, -252);
    const float f1 = kv8_exp2i(e2 >> 1), f2 = kcode == 255 ? __uint_as_float(0x7fc00000u) : kv8_exp2i(e2 - (e2 >> 1));
    const float fv = kv8_scale(a.vscale[block]);
    const size_t base = ((block << a.page_shift) + (j0 & ((1 << a.page_shift) - 1))) * D + (in ? lane * E : 0);
#pragma unroll 1
    for (int j = 0; j < 16; j += 4) {
      float s[4 * R], v[4][E];                             // s: row by row, its four keys
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        float k[E];
        kv8_row_load<E>(kc + base + static_cast<size_t>(j + u) * D, k);
        kv8_row_load<E>(vc + base + static_cast<size_t>(j + u) * D, v[u]);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          s[r * 4 + u] = 0.f;
#pragma unroll
          for (int e = 0; e < E; ++e) s[r * 4 + u] += in ? q[r][e] * k[e] : 0.f;
        }
      }
      int n = 4 * R;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) {
        if (n > 1) {
          n >>= 1;
          const bool up = lane & x;
#pragma unroll
          for (int i = 0; i < 2 * R; ++i)
            if (i < n) {
              const float keep = up ? s[n + i] : s[i], send = up ? s[i] : s[n + i];
              s[i] = keep + __shfl_xor_sync(0xffffffffu, send, x);
            }
        } else {
          s[0] += __shfl_xor_sync(0xffffffffu, s[0], x);
        }
      }
      const int key = j0 + j + u_mine;
      const bool seen = key >= lo && key < hi;
      const float score = seen ? s[0] * c * f1 * f2 : -INFINITY;
      float top = fmaxf(m, score);
#pragma unroll
      for (int x = L; x < 4 * L; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      const float use = top == -INFINITY ? 0.f : top, f = m == -INFINITY ? 0.f : exp2f(m - use);
      const float p = seen ? exp2f(score - use) : -1.f;    // (-1: a key that the row does not see)
      l = l * f + fmaxf(p, 0.f) + (p != p ? p : 0.f);
      if (__any_sync(0xffffffffu, f != 1.f))
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float fr = __shfl_sync(0xffffffffu, f, r * 4 * L);
#pragma unroll
          for (int e = 0; e < E; ++e) o[r][e] *= fr;
        }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
#pragma unroll
        for (int e = 0; e < E; ++e) v[u][e] *= fv;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float w = __shfl_sync(0xffffffffu, p, (r * 4 + u) * L);
#pragma unroll
          for (int e = 0; e < E; ++e) o[r][e] = w < 0.f ? o[r][e] : o[r][e] + w * v[u][e];
        }
      }
      m = top;
    }
  }
#pragma unroll
  for (int x = L; x < 4 * L; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
}

// ---- single tokens: how the keys of a launch are shared out
//
// A row is an (item, kv head): the query heads of one kv head of one sequence's token.  Its live keys are counted in
// units of kUnit keys from an absolute boundary.  The units of all rows, one after another, are cut into as many
// equal shares as there are groups of warps at work: a share holds whole rows, and at its two ends at most one row
// each that is cut.  A whole row is written by its group; of a cut row every group leaves its piece in a
// place of its own in the workspace (two places a share: 0 for the row that goes on from the share before, 1 for a row
// that begins here and goes on), counts itself, and the last one to count adds the pieces in the order of the keys.  Nobody waits
// for anybody.
struct Kv8Args {
  const void* q;               // [tokens, q_stride], head h at column h * D
  int q_stride;
  const uint8_t* kcache;       // [pages, Hkv, page_size, D] e4m3
  const uint8_t* vcache;
  const uint8_t* kscale;       // [pages, Hkv] e8m0
  const uint8_t* vscale;
  const int32_t* block_table;  // [seqs, max_blocks]
  int max_blocks;
  const int4* items;           // (token index of the query, sequence index, context length, 0)
  int nitems;
  int before;                  // items of the call before these (launches before this one have taken them)
  float* part;                 // [shares, 2, G, D + 4] pieces: numerators, d, m, denominator
  int* counters;               // [items * Hkv], zero between launches
  void* out;                   // [tokens, out_stride]
  int out_stride;
  int hq, hkv, page_shift, window;
  float scale;
  const float* cos;            // q is rotated by the kernel if given (position: context - 1)
  const float* sin;
  int max_pos;
  int store;                   // q holds rows [q | k | v]: the tokens' keys and values are stored by the attention's kernel
  int pages;                   // of the pool
  int* status;
  int bad_page;                // the bit of *status that a page id beyond the pool sets
};

// What a part of a row's keys comes to, for one head, is left as D numerators times 2^(m + d) and a denominator times 2^m (log2
// units).  Two references, because a numerator's terms carry the scales of their pages; the second as a distance from
// the first, so that it keeps its bits when the scores are large.  A part without keys has m = -inf and denominator 0.

}  // namespace rl
