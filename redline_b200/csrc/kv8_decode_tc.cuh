// Single tokens over the 8-bit cache on the tensor cores (bfloat16 rows, head size 64 or 128, up to 16 query heads to a kv head).
//
// Included by kv8.cu.  A row is a (item, kv head).  A GROUP of warps takes a row, or a share of one, at a time; its live keys
// are cut into as many equal runs of sub-blocks (32 keys) as the group has warps.  Every warp is a pipeline of its own:
// the sub-blocks of its run come by 16-byte asynchronous copies into a private ring, 8 to 16 KB on their way while one is worked on
// (44 KB an SM cover the way from DRAM at full rate).  A sub-block:
//   S = K Q^T    mma.sync.m16n8k16 on halves, 16 keys x 8 query heads: an e4m3 number is a half exactly (one conversion for two); q is
//                scaled by a power of two per row to at most 256 and rounded to 11 bits.  (The instruction on e4m3 bytes, k = 32, takes
//                1.26 times as long as this one and would want q in three parts of four bits; with the heads as the wide side, half of
//                its rows empty, there were twice as many products.)  Which entries of the head a k index of the product
//                stands for is free, so a lane's 16 bytes of a key are four k steps of the A fragment as they lie.
//   softmax      online, in log2 units, against a reference that moves only when some score exceeds it by 2^10: one vote a sub-block
//                instead of shuffles.  The weights are halves, 2^5 at the reference: 11 bits down to 2^-19 of it, steps of 2^-29 below.
//                For the product they carry the value scale of their page relative to the largest so far.  A run that meets pages more than
//                2^10 apart is left and done in float32 (kv8_rows); a page whose scale is the smallest counts as zeros
//   O^T += V^T P^T   ldmatrix transposes 16 x 16 bytes of V: four keys of an entry in a word; movmatrix transposes P
// With the rotation in the kernel (a.store) the warp that has a row's newest page also stores the token's key and value there: it
// takes that sub-block first, puts the token over what the copy brought, rescales the page if its scale rises, and goes on
// with the bytes as they are stored.
// Page ids and scales are fetched a window of 32 pages at a time, a page to a lane, ahead of their use.
//
// A launch of few keys is a chain of trips to memory (item, page ids, keys; then the results' way to their row), so whatever does not
// depend on one another is asked for together, and results meet in two steps: weights by a warp a head, then sums of 16 bytes a
// thread.
//
// What bounds a long launch is the copies' rate; a short one its chain of trips (0.7 us each) and the one fetch of every
// instruction.  32 / 8 heads, the token's own write included at head size 64: one sequence of 513 keys 8.5 us, 8 of 4,096 17.0 us (1.9 TB/s),
// 64 of 516 to 768 19.4; head size 128: one of 131,072 keys 58 us (4.6 TB/s), 24 of 64 to 8,192 62 us (3.6 TB/s).
//
// Where rows are shared out (see kv8_choice in kv8.cu for which):
//   rows    a cluster of up to 8 CTAs to a row, whose partial results meet in the first one's shared memory; or, with more rows
//           than clusters can be resident, CTAs whose warps form groups that take a row each, one after another
//   pieces  every row in as many pieces as there are CTAs for, which meet in global memory: few rows, and long ones
//   shares  the launch's keys in equal shares, one to a group (kv8.cuh): for rows of very different lengths
#pragma once

#include "cp_async.cuh"
#include "tma.cuh"

namespace rl {

constexpr int kDecWarps = kD == 64 ? 12 : 8, kDecThreads = kDecWarps * 32;
constexpr int kSub = 32;                                 // keys of a sub-block
constexpr int kSubBytes = kSub * kD;                     // K (or V) of one
constexpr int kRing = kD == 64 ? 4 : 3;                  // (192 KB for all warps either way)
constexpr int kRingBytes = kRing * 2 * kSubBytes;
constexpr int kMaxCluster = 8;
constexpr int kPartLd = kD + 4;                          // floats to a head in a warp's partial result: kd numerators, d, m, denominator
static_assert(16 * kPartLd * 4 <= kRingBytes, "a warp's partial result lies in its own ring");

__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
// 16 rows of 16 bytes, a row's address in each of lanes 0 .. 15, and 16 more in lanes 16 .. 31: lane (g, t) gets rows
// 4 t .. 4 t + 3 of column g in v[0], of column g + 8 in v[1], and of the second rows likewise in v[2] and v[3].
__device__ __forceinline__ void ldmatrix_trans(uint32_t* v, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0, %1, %2, %3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(addr));
}
__device__ __forceinline__ void mma_f16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// An 8 x 8 tile of halves, a row's two to a lane, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// (volatile: asked for where it stands)
__device__ __forceinline__ uint4 ldg16(const void* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ void mma_f16_first(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
// (nothing to be seen yet: only that the others have begun)
__device__ __forceinline__ void cluster_arrive_begun() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Four floats to this CTA's address p in CTA `rank` of the cluster.
__device__ __forceinline__ void store_cluster(float* p, uint32_t rank, float4 v) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(remote), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}

constexpr float kDecGrow = 10.f;        // log2 of how far a score may exceed the reference
constexpr int kDecBase = 5;             // log2 of a weight at the reference: 2^15 at most
constexpr int kDecSpread = 10;          // log2 of how far the value scales of a run's pages may be apart

// One warp's result for its run.  Thread (g, t) holds entries 16 c + g (o[c][i][0 and 1]) and 16 c + 8 + g (2 and 3) of the heads
// 8 i + 2 t and 8 i + 2 t + 1, and those heads' references and denominators (of its own keys until the end).
template <bool HI>
struct TcState {
  float o[kD / 16][HI ? 2 : 1][4];
  float m[HI ? 2 : 1][2], l[HI ? 2 : 1][2];
  int vref;                            // the exponent that the numerators' values are relative to (the same for the warp)
};

// A row of the token (a query head's, or its own key or value) is taken by 8 lanes, kRowPart entries d .. and as many D/2 further to a
// lane, so that both entries of a rotated pair are there; four rows at a time.  What it takes is asked for before the first
// copies and used when those are on their way.
constexpr int kRowPart = kD / 16;
struct TcRaw {
  uint32_t lo[kRowPart / 2], hi[kRowPart / 2];
};
struct TcAngles {
  float c[kRowPart], n[kRowPart];
};
template <int N>
__device__ __forceinline__ void ldg_words(const void* p, uint32_t* v) {      // (volatile: asked for where it stands)
  if constexpr (N == 2) {
    asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "l"(p));
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 x = ldg16(static_cast<const char*>(p) + i * 4);
      v[i] = x.x;
      v[i + 1] = x.y;
      v[i + 2] = x.z;
      v[i + 3] = x.w;
    }
  }
}
__device__ __forceinline__ void tc_fetch_row(const Kv8Args& a, const Kv8Segment& s, int head, int lane, TcRaw& r) {
  const bf16* p = static_cast<const bf16*>(a.q) + static_cast<size_t>(s.tok) * a.q_stride + head * kD + (lane & 7) * kRowPart;
  ldg_words<kRowPart / 2>(p, r.lo);
  ldg_words<kRowPart / 2>(p + kD / 2, r.hi);
}
__device__ __forceinline__ void tc_fetch_angles(const Kv8Args& a, const Kv8Segment& s, int lane, TcAngles& t) {
  const size_t at = static_cast<size_t>(s.ctx - 1 < a.max_pos ? s.ctx - 1 : 0) * (kD / 2) + (lane & 7) * kRowPart;
  ldg_words<kRowPart>(a.cos + at, reinterpret_cast<uint32_t*>(t.c));
  ldg_words<kRowPart>(a.sin + at, reinterpret_cast<uint32_t*>(t.n));
}
// (rounded as the write rounds them: kv8_rotate8)
__device__ __forceinline__ void tc_make_row(const TcRaw& r, const TcAngles& t, bool turn, float* x0, float* x1) {
#pragma unroll
  for (int e = 0; e < kRowPart; e += 2) {
    x0[e] = __uint_as_float(r.lo[e / 2] << 16);
    x0[e + 1] = __uint_as_float(r.lo[e / 2] & 0xffff0000u);
    x1[e] = __uint_as_float(r.hi[e / 2] << 16);
    x1[e + 1] = __uint_as_float(r.hi[e / 2] & 0xffff0000u);
  }
  if (turn) {
#pragma unroll
    for (int e = 0; e < kRowPart; ++e) {
      const float lo = x0[e], hi = x1[e];
      x0[e] = __fsub_rn(__fmul_rn(lo, t.c[e]), __fmul_rn(hi, t.n[e]));
      x1[e] = __fadd_rn(__fmul_rn(hi, t.c[e]), __fmul_rn(lo, t.n[e]));
    }
  }
}

// q of the segment's token as halves into `area` (shared memory, [heads][D]), scaled by a power of two per row to at most 256, and
// the factors of the exponents behind them.  `row` is the lane's first row.
template <bool HI>
__device__ __forceinline__ void tc_make_q(const Kv8Args& a, const Kv8Segment& s, int lane, uint32_t area, TcRaw& row, const TcAngles& t) {
  constexpr float kLog2e = 1.4426950408889634f;
  const int G = a.hq / a.hkv;
  if (a.cos != nullptr && s.ctx > a.max_pos && lane == 0) atomicOr(a.status, 2);
#pragma unroll 1
  for (int r0 = 0; r0 < G; r0 += 4) {
    const int r = min(r0 + (lane >> 3), G - 1);          // (lanes without a row of their own repeat the last)
    float x0[kRowPart], x1[kRowPart];
    tc_make_row(row, t, a.cos != nullptr, x0, x1);
    if (r0 + 4 < G) tc_fetch_row(a, s, s.kvh * G + min(r + 4, G - 1), lane, row);
    // (the largest of the bits of the magnitudes is that of the magnitudes, and beyond the finite ones for what is not)
    uint32_t most = 0;
#pragma unroll
    for (int e = 0; e < kRowPart; ++e)
      most = max(most, max(__float_as_uint(x0[e]) & 0x7fffffffu, __float_as_uint(x1[e]) & 0x7fffffffu));
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    const int ex = static_cast<int>(most >> 23);         // the largest entry is 1.m * 2^(ex - 127)
    const int up = ex == 0 ? 0 : min(134 - ex, 127);     // ... and is scaled to 1.m * 2^7
    const float mul = kv8_exp2i(max(up, -126));
    // (a row that is not finite is not a number, not a large one)
    const float f = ex == 255 ? __uint_as_float(0x7fc00000u) : a.scale * kLog2e * kv8_exp2i(-up);
    const uint32_t at = area + r * (kD * 2) + (lane & 7) * (kRowPart * 2);
#pragma unroll
    for (int e = 0; e < kRowPart; e += 4) {
      asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at + 2 * e), "r"(pack_halves(x0[e] * mul, x0[e + 1] * mul)),
                   "r"(pack_halves(x0[e + 2] * mul, x0[e + 3] * mul)) : "memory");
      asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at + kD + 2 * e), "r"(pack_halves(x1[e] * mul, x1[e + 1] * mul)),
                   "r"(pack_halves(x1[e + 2] * mul, x1[e + 3] * mul)) : "memory");
    }
    asm volatile("st.shared.f32 [%0], %1;" ::"r"(area + (HI ? 16 : 8) * (kD * 2) + r * 4), "f"(f) : "memory");
  }
  __syncwarp();
}

// Where 16-byte piece ch of row r of a sub-block lies in its stage (K, V): the fragment reads are free of bank conflicts.
__device__ __forceinline__ uint32_t tc_place(bool is_v, int r, int ch) {
  const int sw = kD == 64 ? (is_v ? (r >> 1) & 3 : 0) : (is_v ? r & 7 : (r & 1) << 2);
  return static_cast<uint32_t>((is_v ? kSubBytes : 0) + r * kD + ((ch ^ sw) << 4));
}
// Stores the token's key (lanes 0 .. 7) and value (8 .. 15; the others repeat) into its page, in the cache (if `mine`) and in the stage that
// holds the page.  codes: the bytes of the page's scales (K, then V); they come back as they are now.
__device__ __forceinline__ uint32_t tc_store_token(const Kv8Args& a, const Kv8Segment& s, int page, uint32_t stage, int lane, bool mine,
                                                   const TcRaw& token, const TcAngles& t, uint32_t codes) {
  constexpr int CH = kD / 16;
  const int ps = 1 << a.page_shift, pos = s.ctx - 1, off = pos & (ps - 1), row = pos % kSub, row0 = row - off;
  const int which = (lane >> 3) & 1;
  float x0[kRowPart], x1[kRowPart], amax = 0.f;
  tc_make_row(token, t, which == 0, x0, x1);
#pragma unroll
  for (int e = 0; e < kRowPart; ++e) {
    const float u = fabsf(x0[e]), v = fabsf(x1[e]);
    amax = fmaxf(amax, fmaxf(u < INFINITY ? u : 0.f, v < INFINITY ? v : 0.f));
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  const size_t block = static_cast<size_t>(page) * a.hkv + s.kvh;
  const int old = min(static_cast<int>((codes >> (8 * which)) & 255), 254);
  int code = kv8_code(amax);
  if (off > 0) code = max(code, old);
  const int kcode = __shfl_sync(0xffffffffu, code, 0), vcode = __shfl_sync(0xffffffffu, code, 8);
  if (off > 0) {                                         // what is in the page goes over to a larger scale
#pragma unroll 1
    for (int is_v = 0; is_v < 2; ++is_v) {
      const int was = min(static_cast<int>((codes >> (8 * is_v)) & 255), 254), now = is_v ? vcode : kcode;
      if (now == was) continue;
      uint4* base = reinterpret_cast<uint4*>(const_cast<uint8_t*>(is_v ? a.vcache : a.kcache) + block * ps * kD);
      const float f = kv8_exp2i(max(was - now, -127));
#pragma unroll 1
      for (int c = lane; c < off * CH; c += 32) {
        const uint32_t at = stage + tc_place(is_v, row0 + c / CH, c % CH);
        float y[16];
        kv8_f16(lds16(at), y);
#pragma unroll
        for (int e = 0; e < 16; ++e) y[e] *= f;
        const uint4 w = make_uint4(kv8_pack4(y), kv8_pack4(y + 4), kv8_pack4(y + 8), kv8_pack4(y + 12));
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w) : "memory");
        if (mine) base[c] = w;
      }
    }
  }
  if (lane < 16) {
    const float inv = kv8_exp2i(127 - code);
#pragma unroll
    for (int e = 0; e < kRowPart; ++e) {
      x0[e] = fabsf(x0[e]) < INFINITY ? x0[e] * inv : __uint_as_float(0x7fc00000u);
      x1[e] = fabsf(x1[e]) < INFINITY ? x1[e] * inv : __uint_as_float(0x7fc00000u);
    }
    uint8_t* dst = const_cast<uint8_t*>(which ? a.vcache : a.kcache) + (block * ps + off) * kD;
#pragma unroll
    for (int e = 0; e < kRowPart; e += 4)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int d = (lane & 7) * kRowPart + e + half * (kD / 2);
        const uint32_t w = kv8_pack4((half ? x1 : x0) + e);
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(stage + tc_place(which, row, d >> 4) + (d & 15)), "r"(w) : "memory");
        if (mine) *reinterpret_cast<uint32_t*>(dst + d) = w;
      }
    if (mine && (lane & 7) == 0) const_cast<uint8_t*>(which ? a.vscale : a.kscale)[block] = static_cast<uint8_t>(code);
  }
  __syncwarp();
  return static_cast<uint32_t>(kcode) | static_cast<uint32_t>(vcode) << 8;
}

// The run of sub-blocks [sb0, sb0 + n) of the segment, the last one first, through the warp's ring.  False: the pages are too far apart
// (the token is stored, the result of no use).
template <bool HI>
__device__ __forceinline__ bool tc_run(const Kv8Args& a, const Kv8Segment& s, int sb0, int n, uint32_t ring, int lane, TcState<HI>& st) {
  constexpr int KS = kD / 16, NC = kD / 16, NR = HI ? 2 : 1;
  constexpr int CPR = kD / 16;                           // 16-byte pieces of a key
  const int shift = a.page_shift, ps = 1 << shift;
#pragma unroll
  for (int h = 0; h < NR; ++h) {
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) st.o[c][h][e] = 0.f;
    st.m[h][0] = st.m[h][1] = -INFINITY;
    st.l[h][0] = st.l[h][1] = 0.f;
  }
  st.vref = -1000;
  uint32_t vleast = 0x3fffffff;                          // the smallest exponent of a page's values, plus 125 (a page of zeros: a large number)
  bool near = true;
  if (n <= 0) return true;
  const int32_t* bt = a.block_table + static_cast<size_t>(s.seq) * a.max_blocks;
  // (a sub-block may reach over either end of the live keys, into pages that need not be there any more: their places are
  // filled from the nearest live page)
  const int page_first = s.key_lo >> shift, page_last = min(s.key_hi - 1, (sb0 + n) * kSub - 1) >> shift;
  auto page_of = [&](int key) { return page_last - min(max(key >> shift, page_first), page_last); };     // counted from the last
  // a window of 32 pages, a page to a lane: its id and the bytes of its scales (K, V), those of the window before, and the
  // ids of the next; and the scales of the window that the sums are in
  bool bad = false;                                      // a page id beyond the pool
  int window = 0, my_page = kv8_page(bt[max(page_last - lane, page_first)], a.pages, bad), next_page = 0;
  const int top = sb0 + n - 1;
  const bool store = a.store && s.key_hi == s.ctx && top == (s.ctx - 1) / kSub;      // the newest page is this warp's
  TcRaw row, token;
  TcAngles angles;
  tc_fetch_row(a, s, s.kvh * (a.hq / a.hkv) + min(lane >> 3, a.hq / a.hkv - 1), lane, row);
  if (a.cos != nullptr) tc_fetch_angles(a, s, lane, angles);
  if (store) tc_fetch_row(a, s, a.hq + ((lane >> 3) & 1) * a.hkv + s.kvh, lane, token);
  auto codes_of = [&](int page) -> uint32_t {
    const size_t at = static_cast<size_t>(page) * a.hkv + s.kvh;
    return static_cast<uint32_t>(__ldcg(a.kscale + at)) | static_cast<uint32_t>(__ldcg(a.vscale + at)) << 8;
  };
  uint32_t my_codes = codes_of(my_page), old_codes = 0;
  if (page_last - 32 >= page_first) next_page = bt[max(page_last - 32 - lane, page_first)];
  // Copies sub-block sb into stage `stage`.  16 keys of a page are contiguous; the places in shared memory are swizzled so that
  // the fragment reads are free of bank conflicts.  Bytes behind the segment's last key are copied too (they lie in the page).
  const uint32_t ch = lane % CPR, in = lane / CPR;       // this lane's piece of a row, its row of a round
  // (rows of 128 bytes: K piece ^ 4 in odd rows, V piece ^ row; rows of 64: V piece ^ half of the row)
  const uint32_t koff = in * kD + (kD == 64 ? ch : ch ^ ((in & 1) << 2)) * 16;
  const uint32_t voff = in * kD + (kD == 64 ? ch ^ ((in >> 1) & 3) : ch ^ (in & 3)) * 16;
  const size_t page_bytes = static_cast<size_t>(a.hkv) * ps * kD;
  const uint8_t* kbase = a.kcache + static_cast<size_t>(s.kvh) * ps * kD + lane * 16;
  const uint8_t* vbase = a.vcache + static_cast<size_t>(s.kvh) * ps * kD + lane * 16;
  auto issue = [&](int sb, int stage) {
    const uint32_t kdst = ring + stage * (2 * kSubBytes) + koff, vdst = ring + stage * (2 * kSubBytes) + kSubBytes + voff;
#pragma unroll
    for (int b = 1; b >= 0; --b) {
      const int key = sb * kSub + b * 16;
      const int idx = page_of(key);
      if ((idx >> 5) != window) {
        window = idx >> 5;
        my_page = kv8_page(next_page, a.pages, bad);
        old_codes = my_codes;
        my_codes = codes_of(my_page);
        next_page = bt[max(page_last - window * 32 - 32 - lane, page_first)];
      }
      const int page = __shfl_sync(0xffffffffu, my_page, idx & 31);
      const size_t at = page * page_bytes + (key & (ps - 1)) * kD;
      const uint8_t *kp = kbase + at, *vp = vbase + at;
#pragma unroll
      for (int i = 0; i < CPR / 2; ++i) {
        cp_async16_s(kdst + b * (16 * kD) + i * 512, kp + i * 512);
        // (a round is 4 rows of 128 bytes or 8 of 64: only the first changes the swizzle, by bit 2 of the row)
        cp_async16_s((kD == 64 ? vdst : vdst ^ ((i & 1) << 6)) + b * (16 * kD) + i * 512, vp + i * 512);
      }
    }
  };
  const int token_page = __shfl_sync(0xffffffffu, my_page, 0);
  bool mine = true;
  if (store) {                                           // (of several items of one page or sequence the first stores: see kv8_write_kernel)
#pragma unroll 1
    for (int i = lane - a.before; i < s.item; i += 32) {
      const int4 other = a.items[i];
      if (other.z > 0 && (other.y == s.seq
                          || a.block_table[static_cast<size_t>(other.y) * a.max_blocks + ((other.z - 1) >> shift)] == token_page))
        mine = false;
    }
    if (lane == 0 && bad) mine = false;                  // (a page beyond the pool stands as page 0 here, but nothing is stored there)
    mine = __all_sync(0xffffffffu, mine);
    if (!mine && token_page != 0 && lane == 0) atomicOr(a.status, 8);
  }
  // lane addresses: key 4 (g / 2) + g % 2 of K and the one 2 further (so that the weights of keys 4 t .. 4 t + 3 meet in a lane
  // once they are transposed), key lane of V
  const uint32_t kr = 4 * (lane >> 3) + ((lane >> 2) & 1);
  const uint32_t krow = kr * kD + (kD == 64 ? lane & 3 : (lane & 3) ^ ((kr & 1) << 2)) * 16;
  const uint32_t vrow = lane * kD, vsw = kD == 64 ? (lane >> 1) & 3 : lane & 7;
  uint32_t qf[NR][KS][2];
  float factor[NR][2];
  int stage = 0, ahead = 0;
#pragma unroll 1
  for (int i = 1 - kRing; i < n; ++i) {
    const int k0 = (top - i) * kSub;
    if (i == 0) {                                        // the first copies are on their way: q, by way of the stage that is still free
      const uint32_t area = ring + (kRing - 1) * (2 * kSubBytes);
      tc_make_q<HI>(a, s, lane, area, row, angles);
#pragma unroll
      for (int h = 0; h < NR; ++h) {
        const int r = (lane >> 2) + 8 * h;
        const bool has = r < a.hq / a.hkv;
#pragma unroll
        for (int c = 0; c < KS / 4; ++c)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint4 x = lds16(area + r * (kD * 2) + c * 128 + (lane & 3) * 32 + u * 16);
            qf[h][c * 4 + 2 * u][0] = has ? x.x : 0u;
            qf[h][c * 4 + 2 * u][1] = has ? x.y : 0u;
            qf[h][c * 4 + 2 * u + 1][0] = has ? x.z : 0u;
            qf[h][c * 4 + 2 * u + 1][1] = has ? x.w : 0u;
          }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int hd = 8 * h + (lane & 3) * 2 + e;
          float f;
          asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f) : "r"(area + (HI ? 16 : 8) * (kD * 2) + hd * 4));
          factor[h][e] = hd < a.hq / a.hkv ? f : 0.f;
        }
      }
    }
    if (i >= 0) {
      cp_async_wait<kRing - 2>();
      __syncwarp();                                      // (every lane's copies; and every lane is through with the sub-block before)
    }
    if (i == 0 && store) {
      const uint32_t codes = tc_store_token(a, s, token_page, ring, lane, mine, token, angles, __shfl_sync(0xffffffffu, my_codes, 0));
      if (lane == 0) my_codes = codes;
    }
    if (i + kRing - 1 < n) issue(top - i - (kRing - 1), ahead);
    ahead = ahead + 1 == kRing ? 0 : ahead + 1;
    cp_async_commit();                                     // (a group to a sub-block, empty behind the last)
    if (i < 0) continue;
    const uint32_t kst = ring + stage * (2 * kSubBytes) + krow, vst = ring + stage * (2 * kSubBytes) + kSubBytes + vrow;
    stage = stage + 1 == kRing ? 0 : stage + 1;
    const bool whole = k0 >= s.key_lo && k0 + kSub <= s.key_hi;
    if (!whole) {
      // a key that is not seen may hold anything, what is not a number included: its weight of 0 does not cover that
      const int key = k0 + lane;
      if (key < s.key_lo || key >= s.key_hi) {
#pragma unroll
        for (int c = 0; c < CPR; ++c)
          asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(vst + c * 16), "r"(0u) : "memory");
      }
      __syncwarp();
    }
    // ---- S: 16 keys b (rows 4 (g / 2) + g % 2, and 2 further: c0 and c2), heads 8 h + 2 t (c0) and 8 h + 2 t + 1
    float sv[2][NR][4];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int c = 0; c < KS / 4; ++c) {
        const uint4 k0w = lds16((c ? kst ^ 64u : kst) + b * 16 * kD), k1w = lds16((c ? kst ^ 64u : kst) + (b * 16 + 2) * kD);
        const uint32_t w0[4] = {k0w.x, k0w.y, k0w.z, k0w.w}, w1[4] = {k1w.x, k1w.y, k1w.z, k1w.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t a0, a1, a2, a3;
          halves4(w0[k], a0, a2);
          halves4(w1[k], a1, a3);
#pragma unroll
          for (int h = 0; h < NR; ++h) {
            const uint32_t* q2 = qf[h][c * 4 + k];
            if (c == 0 && k == 0) mma_f16_first(sv[b][h], a0, a1, a2, a3, q2[0], q2[1]);
            else mma_f16(sv[b][h], a0, a1, a2, a3, q2[0], q2[1]);
          }
        }
      }
    // ---- V^T as A fragments: entries 16 c + g and 16 c + 8 + g, keys 4 t .. + 3 and 16 further
    uint32_t v[NC][4];
#pragma unroll
    for (int c = 0; c < NC; ++c) ldmatrix_trans(v[c], vst + ((c ^ vsw) << 4));
    // the scales of the first and the second 16 keys (the copies are at most one window ahead)
    float kf[2];
    int ve[2];
    bool odd = false;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int idx = page_of(k0 + b * 16);
      const uint32_t c = __shfl_sync(0xffffffffu, (idx >> 5) == window ? my_codes : old_codes, idx & 31);
      kf[b] = kv8_scale(c & 255);
      ve[b] = static_cast<int>(c >> 8) - 127;
      odd |= ve[b] == 128;
    }
    const int vref = max(st.vref, max(ve[0], ve[1]));
    const uint32_t least = min(static_cast<uint32_t>(ve[0] + 125), static_cast<uint32_t>(ve[1] + 125));
    if (vref != st.vref || least < vleast) {             // (the same for the warp)
      vleast = min(vleast, least);
      if (vref + 125 - static_cast<int>(vleast) > kDecSpread) {
        near = false;
        break;
      }
      const float f = kv8_exp2i(max(st.vref - vref, -127));
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int h = 0; h < NR; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) st.o[c][h][e] *= f;
      st.vref = vref;
    }
    if (!whole) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int key = k0 + b * 16 + static_cast<int>(kr) + 2 * r;
          if (key < s.key_lo || key >= s.key_hi)
#pragma unroll
            for (int h = 0; h < NR; ++h) sv[b][h][2 * r] = sv[b][h][2 * r + 1] = -INFINITY;
        }
    }
    float f[2][NR][2], y[2][NR][4];
    bool grown = false;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int h = 0; h < NR; ++h) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          f[b][h][e] = factor[h][e] * kf[b];
          // (times -inf it has to be -inf; so small a factor makes every score 0)
          if (f[b][h][e] < 1.2e-38f) f[b][h][e] = 1.2e-38f;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[b][h][e] = fmaf(sv[b][h][e], f[b][h][e & 1], -st.m[h][e & 1]);
          grown |= y[b][h][e] > kDecGrow;
        }
      }
    if (__any_sync(0xffffffffu, grown)) {                // (the first sub-block among them: the reference is -inf)
#pragma unroll
      for (int h = 0; h < NR; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float m = st.m[h][e];
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              y[b][h][2 * r + e] = sv[b][h][2 * r + e] * f[b][h][e];
              m = fmaxf(m, y[b][h][2 * r + e]);
            }
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
          const float alpha = m == st.m[h][e] ? 1.f : ex2_approx(st.m[h][e] - m);
          st.m[h][e] = m;
          st.l[h][e] *= alpha;
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            st.o[c][h][e] *= alpha;
            st.o[c][h][2 + e] *= alpha;
          }
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 2; ++r) y[b][h][2 * r + e] -= m;
        }
    }
    // ---- the weights as B fragments: keys 4 t, 4 t + 1 and 4 t + 2, 4 t + 3 of head 8 h + g
    uint32_t pf[2][NR][2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      float w = kv8_exp2i(max(ve[b] - vref + kDecBase, -127));
      if (odd && ve[b] == 128) w = __uint_as_float(0x7fc00000u);
#pragma unroll
      for (int h = 0; h < NR; ++h)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float p0 = ex2_approx(y[b][h][2 * r]), p1 = ex2_approx(y[b][h][2 * r + 1]);
          st.l[h][0] += p0;
          st.l[h][1] += p1;
          pf[b][h][r] = transposed(pack_halves(p0 * w, p1 * w));
        }
    }
    // ---- O^T += V^T P^T
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        uint32_t a0, a1, a2, a3;
        halves4(v[c][2 * b], a0, a2);
        halves4(v[c][2 * b + 1], a1, a3);
#pragma unroll
        for (int h = 0; h < NR; ++h) mma_f16(st.o[c][h], a0, a1, a2, a3, pf[b][h][0], pf[b][h][1]);
      }
  }
  cp_async_wait<0>();
  if (bad) atomicOr(a.status, a.bad_page);
#pragma unroll
  for (int h = 0; h < NR; ++h)                           // the eight lanes of a head
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) st.l[h][e] += __shfl_xor_sync(0xffffffffu, st.l[h][e], o);
  __syncwarp();
  return near;
}

// The same run in float32, into the place of the warp's partial result.
__device__ __noinline__ void tc_run_far(const Kv8Args& a, Kv8Segment s, int sb0, int n, int lane, float* to) {
  typedef Kv8Rows<kD> Rows;
  const int G = a.hq / a.hkv, at = lane * Rows::E, dh = at % (kD / 2);
#pragma unroll 1
  for (int r0 = 0; r0 < G; r0 += Rows::R) {
    float x[Rows::R][Rows::E] = {}, o[Rows::R][Rows::E], m, l;
#pragma unroll
    for (int r = 0; r < Rows::R; ++r) {
      if (r0 + r >= G) continue;
      const bf16* row = static_cast<const bf16*>(a.q) + static_cast<size_t>(s.tok) * a.q_stride + (s.kvh * G + r0 + r) * kD;
#pragma unroll
      for (int e = 0; e < Rows::E; ++e) {
        x[r][e] = to_float(row[at + e]);
        if (a.cos != nullptr) {
          const size_t i = static_cast<size_t>(s.ctx - 1 < a.max_pos ? s.ctx - 1 : 0) * (kD / 2) + dh + e;
          const float other = to_float(row[at < kD / 2 ? at + e + kD / 2 : dh + e]);
          x[r][e] = at < kD / 2 ? x[r][e] * a.cos[i] - other * a.sin[i] : x[r][e] * a.cos[i] + other * a.sin[i];
        }
      }
    }
    const int mine = r0 + Rows::row_of(lane);
    kv8_rows<kD>(a, s.seq, s.kvh, max(s.key_lo, sb0 * kSub), mine < G ? min(s.key_hi, (sb0 + n) * kSub) : 0, a.scale * 1.4426950408889634f, lane,
                 x, o, m, l);
#pragma unroll
    for (int r = 0; r < Rows::R; ++r)
      if (r0 + r < G)
#pragma unroll
        for (int e = 0; e < Rows::E; ++e) to[(r0 + r) * kPartLd + at + e] = o[r][e];
    if (mine < G && lane % (4 * Rows::L) == 0) *reinterpret_cast<float4*>(to + mine * kPartLd + kD) = make_float4(0.f, m, l, 0.f);
  }
}

__device__ __forceinline__ void tc_group_barrier(int bar, int gsize) {
  asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(gsize * 32) : "memory");
}
// Adds up `n` partial results ([G][kPartLd] floats, `stride` bytes apart in shared memory; the first one's references are
// overwritten) in order and leaves the sums: as the row's result (`out`; to == nullptr), as a partial result in global memory, or (rank >= 0)
// in the shared memory of CTA `rank` of the cluster.  The `gsize` warps that call it meet at barrier `bar`.
// (One piece of code for all of them, and little of it: code that a launch runs once comes from L2 or memory, a microsecond for some
// hundreds of instructions.)
__device__ __noinline__ void tc_fold(unsigned char* parts, int stride, int n, int wg, int gsize, int bar, int G, bf16* out, float* to, int rank) {
  const int lane = threadIdx.x & 31;
  // weights: a warp to a head, a lane to a partial result
#pragma unroll 1
  for (int r = wg; r < G; r += gsize) {
    float* p = reinterpret_cast<float*>(parts + min(lane, n - 1) * stride) + r * kPartLd + kD;
    const float4 x = *reinterpret_cast<const float4*>(p);                // d, m, denominator
    const bool none = lane >= n || (x.y == -INFINITY && x.z == 0.f);     // (a part without keys)
    const float top = warp_max(x.y), dm = none ? 0.f : x.y - top;
    const float dtop = warp_max(none ? -INFINITY : x.x + dm);
    const float den = warp_sum(none ? 0.f : x.z * ex2_approx(dm));
    if (lane < n) p[0] = none ? 0.f : ex2_approx(x.x + dm - dtop);
    if (lane == 0) {
      p[1] = top;
      p[2] = dtop;
      p[3] = den;
    }
  }
  tc_group_barrier(bar, gsize);
#pragma unroll 1
  for (int i = wg * 32 + lane; i < G * (kD / 4); i += gsize * 32) {
    const int r = i / (kD / 4), d = (i - r * (kD / 4)) * 4;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    const float* p = reinterpret_cast<const float*>(parts) + r * kPartLd;
    const float4 ref = *reinterpret_cast<const float4*>(p + kD);         // weight, m, d, denominator
#pragma unroll 1
    for (int w = 0; w < n; ++w) {
      const float f = p[kD];
      const float4 x = *reinterpret_cast<const float4*>(p + d);
      p += stride / 4;
      sum.x += f * x.x;
      sum.y += f * x.y;
      sum.z += f * x.z;
      sum.w += f * x.w;
    }
    if (to == nullptr) {
      const float f = __fdividef(ex2_approx(ref.z), ref.w);
      const float v[4] = {sum.x * f, sum.y * f, sum.z * f, sum.w * f};
      store4(out + r * kD + d, v);
    } else {
      float* q = to + r * kPartLd;
      const float4 refs = make_float4(ref.z, ref.y, ref.w, 0.f);
      if (rank >= 0) {
        store_cluster(q + d, rank, sum);
        if (d == 0) store_cluster(q + kD, rank, refs);
      } else {
        *reinterpret_cast<float4*>(q + d) = sum;
        if (d == 0) *reinterpret_cast<float4*>(q + kD) = refs;
      }
    }
  }
}

// groups: of the CTA's warps, a divisor of their number.  parts: 0 rows, > 0 pieces of a row (one to a CTA), -1 shares.
template <bool HI>
__global__ void __launch_bounds__(kDecThreads, 1)
kv8_decode_tc_kernel(const __grid_constant__ Kv8Args a, int groups, int parts) {
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int start[kMaxItems + 1];
  __shared__ int last[kDecWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int G = a.hq / a.hkv;
  const int csize = static_cast<int>(cluster_size()), rank = static_cast<int>(cluster_rank());
  const int gsize = kDecWarps / groups, gi = warp / gsize, wg = warp - gi * gsize;
  const int gtid = wg * 32 + lane;
  const int nclusters = gridDim.x / csize;
  float* slots = reinterpret_cast<float*>(smem + kDecWarps * kRingBytes);      // [csize][G][kPartLd], of the first CTA of a cluster
  if (csize > 1) cluster_arrive_begun();                       // (met before the first store into another CTA: it has begun by then)
  pdl_wait();
  const bool by_shares = parts < 0;
  const Kv8Cut cut(by_shares ? kv8_units(a, start) : 0, nclusters * groups);
  const int share = gi * nclusters + blockIdx.x;          // (neighbouring shares lie on different SMs)
  int u = by_shares && share < cut.shares ? cut.begin(share) : 0;
  const int share_first = u, end = by_shares && share < cut.shares ? cut.begin(share + 1) : 0;
  const int nrows = a.nitems * a.hkv;
  int rowi = parts > 0 ? blockIdx.x / parts : gi * nclusters + blockIdx.x / csize;
#pragma unroll 1
  for (;;) {
    Kv8Segment s;
    if (by_shares) {
      if (u >= end) break;
      s = kv8_segment(a, start, u, end);
    } else {
      if (rowi >= nrows) break;
      s.item = rowi / a.hkv;
      s.kvh = rowi - s.item * a.hkv;
      const int4 info = a.items[s.item];
      s.tok = info.x;
      s.seq = info.y;
      s.ctx = info.z;
      s.key_lo = a.window > 0 && s.ctx > a.window ? s.ctx - a.window : 0;
      s.key_hi = s.ctx;
      s.whole = parts == 0;
      rowi = parts > 0 ? nrows : rowi + groups * nclusters;
      if (s.ctx <= 0) {                                  // (the same for the whole cluster)
        if (csize > 1) cluster_wait();
        continue;
      }
      if (parts > 0) {                                   // this CTA's piece, in whole sub-blocks
        const int j = blockIdx.x % parts, first = s.key_lo / kSub, all = (s.key_hi - 1) / kSub - first + 1;
        const int b0 = first + static_cast<int>(static_cast<long long>(all) * j / parts);
        const int b1 = first + static_cast<int>(static_cast<long long>(all) * (j + 1) / parts);
        s.key_lo = max(s.key_lo, b0 * kSub);
        s.key_hi = min(s.key_hi, b1 * kSub);
      }
    }
    // ---- this warp's run of sub-blocks
    const int W = csize * gsize, wi = rank * gsize + wg;
    const int first = s.key_lo / kSub, all = s.key_hi > s.key_lo ? (s.key_hi - 1) / kSub - first + 1 : 0;
    const int per = all / W, rem = all - per * W;
    TcState<HI> st;
    const int sb0 = first + wi * per + min(wi, rem), sbs = per + (wi < rem ? 1 : 0);
    const bool near = tc_run<HI>(a, s, sb0, sbs, smem_u32(smem) + warp * kRingBytes, lane, st);
    bf16* out = static_cast<bf16*>(a.out) + static_cast<size_t>(s.tok) * a.out_stride + s.kvh * G * kD;
    // ---- its partial result into its ring
    float* mine = reinterpret_cast<float*>(smem + warp * kRingBytes);
    const int g = lane >> 2, t = lane & 3;
    if (!near) tc_run_far(a, s, sb0, sbs, lane, mine);
#pragma unroll
    for (int h = 0; h < (HI ? 2 : 1); ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * h + 2 * t + e;
        if (r >= G || !near) continue;
#pragma unroll
        for (int c = 0; c < kD / 16; ++c) {
          mine[r * kPartLd + 16 * c + g] = st.o[c][h][e];
          mine[r * kPartLd + 16 * c + 8 + g] = st.o[c][h][2 + e];
        }
        if (g == 0) *reinterpret_cast<float4*>(mine + r * kPartLd + kD) = make_float4(static_cast<float>(st.vref - kDecBase), st.m[h][e], st.l[h][e], 0.f);
      }
    if (csize > 1) {
      // ---- the CTA's sums into a slot of the cluster's first CTA, which adds the slots in order
      __syncthreads();
      cluster_wait();
      tc_fold(smem, kRingBytes, kDecWarps, warp, kDecWarps, 1, G, nullptr, slots + rank * G * kPartLd, 0);
      cluster_arrive();
      cluster_wait();
      if (rank == 0) tc_fold(reinterpret_cast<unsigned char*>(slots), G * kPartLd * 4, csize, warp, kDecWarps, 1, G, out, nullptr, -1);
      continue;                                          // (one row to a cluster: see the launch)
    }
    tc_group_barrier(1 + gi, gsize);
    // (with pieces CTA x leaves the piece of share x)
    float* piece = !s.whole ? a.part + (static_cast<size_t>(share) * 2 + (u == share_first ? 0 : 1)) * (G * (kD + 4)) : nullptr;
    tc_fold(smem + gi * gsize * kRingBytes, kRingBytes, gsize, wg, gsize, 1 + gi, G, out, piece, -1);
    if (piece != nullptr) {
      __threadfence();                                   // the piece, before it is counted
      tc_group_barrier(1 + gi, gsize);
      const int s0 = parts > 0 ? blockIdx.x / parts * parts : cut.of(s.row_begin);
      const int s1 = parts > 0 ? s0 + parts - 1 : cut.of(s.row_end - 1);
      if (gtid == 0) {
        int* c = a.counters + static_cast<size_t>(s.item) * a.hkv + s.kvh;
        const int done = atomicAdd(c, 1) == s1 - s0;
        if (done) *c = 0;
        last[gi] = done;
      }
      tc_group_barrier(1 + gi, gsize);
      if (last[gi]) {
        __threadfence();
        kv8_merge<bf16>(a.part, G, s0, s1, parts < 0 && cut.begin(s0) != s.row_begin ? 1 : 0, out, wg, gsize);
      }
    }
    tc_group_barrier(1 + gi, gsize);                     // before the rings are used again
    if (by_shares) u = s.next;
  }
}

}  // namespace rl
