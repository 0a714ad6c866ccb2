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

// ---- one row by a warp: without the limits of the kernels that are built for speed, for the rows that meet them
//
// A query row of one head over the keys [lo, hi), in float32 throughout: scores by exponents of q and the page apart, values as they are,
// a key that the row does not see not looked at.  Lane i has entries i E .. of q (`q`, as they are) and gets the numerators there (`o`,
// relative to 2^m, m in log2 units as c is) and the denominator l.  Some 50 times slower than the kernels' own ways.
template <int D>
struct Kv8Row {
  static constexpr int E = D <= 32 ? 1 : D <= 64 ? 2 : D <= 128 ? 4 : 8;
  static __device__ __forceinline__ bool in_head(int lane) { return lane * E < D; }
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

template <int D, typename Args>
__device__ __forceinline__ void kv8_row(const Args& a, int seq, int kvh, int lo, int hi, float c, int lane, float* q, float* o, float& m, float& l) {
  constexpr int E = Kv8Row<D>::E;
  const bool in = Kv8Row<D>::in_head(lane);
  const uint8_t *kc = reinterpret_cast<const uint8_t*>(a.kcache), *vc = reinterpret_cast<const uint8_t*>(a.vcache);
  const int32_t* bt = a.block_table + static_cast<size_t>(seq) * a.max_blocks;
  float amax = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    amax = fmaxf(amax, in ? fabsf(q[e]) : 0.f);
    o[e] = 0.f;
  }
  amax = warp_max(amax);
  const int ex = amax > 0.f && amax < INFINITY ? ilogbf(amax) : 0;
#pragma unroll
  for (int e = 0; e < E; ++e) q[e] = in ? ldexpf(q[e], -ex) : 0.f;
  m = -INFINITY;
  l = 0.f;
#pragma unroll 1
  for (int j0 = lo & ~15; j0 < hi; j0 += 16) {             // 16 keys of one page
    bool bad = false;                                      // (told by whoever went over the keys before)
    const size_t block = static_cast<size_t>(kv8_page(bt[j0 >> a.page_shift], a.pages, bad)) * a.hkv + kvh;
    const int kcode = a.kscale[block];
    const float fv = kv8_scale(a.vscale[block]);
    const size_t base = ((block << a.page_shift) + (j0 & ((1 << a.page_shift) - 1))) * D + (in ? lane * E : 0);
#pragma unroll 1
    for (int j = 0; j < 16; j += 4) {
      float x[4], v[4][E];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        float k[E];
        kv8_row_load<E>(kc + base + static_cast<size_t>(j + u) * D, k);
        kv8_row_load<E>(vc + base + static_cast<size_t>(j + u) * D, v[u]);
        x[u] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) x[u] += in ? q[e] * k[e] : 0.f;
      }
      float top = m;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int key = j0 + j + u;
        x[u] = ldexpf(warp_sum(x[u]) * c, ex + kcode - 127);
        if (kcode == 255) x[u] = __uint_as_float(0x7fc00000u);
        if (key < lo || key >= hi) x[u] = -INFINITY;
        top = fmaxf(top, x[u]);
      }
      const float use = top == -INFINITY ? 0.f : top, f = m == -INFINITY ? 0.f : exp2f(m - use);
      l *= f;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] *= f;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int key = j0 + j + u;
        if (key < lo || key >= hi) continue;
        const float p = exp2f(x[u] - use);
        l += p;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] += p * (v[u][e] * fv);
      }
      m = top;
    }
  }
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
