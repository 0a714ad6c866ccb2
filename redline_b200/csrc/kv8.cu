// The paged cache that is held in 8 bits (format: kv8.cuh): its write, and the attention that reads it.
//
//   kv8_write_kernel     rotates q and k, stores k and v with a scale for every page and kv head
//   kv8_decode_kernel    single tokens on the CUDA cores: any head size in steps of 16 up to 256, float32 or bfloat16
//   kv8_prefill_kernel   portions of prompts on the CUDA cores, for the same types and sizes
#include <mutex>

#include "kv8.cuh"

#ifndef RL_HEAD_DIM
#define RL_HEAD_DIM 64
#endif

namespace rl {

constexpr int kD = RL_HEAD_DIM;
static_assert(kD % 16 == 0 && kD >= 16 && kD <= 256, "head size must be a multiple of 16, at most 256");

// ------------------------------------------------------------------------------------------------ write

// Eight consecutive elements.
__device__ __forceinline__ void load8(const float* p, float* out) {
  load16(p, out);
  load16(p + 4, out + 4);
}
__device__ __forceinline__ void load8(const bf16* p, float* out) { load16(p, out); }
__device__ __forceinline__ void store8(float* p, const float* in) {
  store16(p, in);
  store16(p + 4, in + 4);
}
__device__ __forceinline__ void store8(bf16* p, const float* in) { store16(p, in); }

// Entries i and i + D/2 of a head by the angle's cosine and sine.  (Each product is rounded before the sum: what is
// stored next is rounded to 4 bits, and a fused sum would land on the other side of a border now and then.)
__device__ __forceinline__ void kv8_rotate8(float* x0, float* x1, const float* c, const float* s) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = x0[i], b = x1[i];
    x0[i] = __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i]));
    x1[i] = __fadd_rn(__fmul_rn(b, c[i]), __fmul_rn(a, s[i]));
  }
}

template <typename T>
struct Kv8WriteArgs {
  const T* qkv;                // [tokens, qkv_stride]: q heads, then k heads, then v heads
  int qkv_stride;
  const int32_t* positions;
  const int32_t* slots;        // [tokens] place in the cache; negative: none.  With items instead: null
  const int4* items;           // (token, sequence, context): the slot is that of position context - 1
  const int32_t* block_table;
  int max_blocks;
  const float* cos;            // [max_pos, D/2], null: no rotation
  const float* sin;
  uint8_t* kcache;
  uint8_t* vcache;
  uint8_t* kscale;
  uint8_t* vscale;
  T* q_out;                    // [tokens, q_stride], null: q is left alone
  int q_stride;
  int tokens, hq, hkv, page_shift, max_pos;
  long long num_slots;
  int* status;
};

// Slot of token t (-1: none).
template <typename T>
__device__ __forceinline__ long long kv8_slot(const Kv8WriteArgs<T>& a, int t) {
  if (a.slots != nullptr) return a.slots[t];
  const int4 info = a.items[t];
  if (info.z <= 0) return -1;
  const int pos = info.z - 1;
  return (static_cast<long long>(a.block_table[static_cast<size_t>(info.y) * a.max_blocks + (pos >> a.page_shift)])
          << a.page_shift) + (pos & ((1 << a.page_shift) - 1));
}

// A position whose angles the tables have.
template <typename T>
__device__ __forceinline__ int kv8_position(const Kv8WriteArgs<T>& a, int pos) {
  if (pos >= 0 && pos < a.max_pos) return pos;
  atomicOr(a.status, 2);
  return 0;
}

constexpr int kWriteThreads = 256, kWriteWarps = kWriteThreads / 32;
constexpr int kWriteTokens = 32 / (kD / 16);       // tokens that a warp takes at once: each D/16 lanes, 8 entries of either half of the head
// Rounds of them that are kept between the two passes over a run: a page of 16 tokens at head sizes up to 128.  (As floats, and with three CTAs an SM
// a thread has 80 registers: 32 bytes of them are spilled at head size 64, 424 at 128.)
constexpr int kWriteRounds = kD <= 64 ? 2 : 4;

// gridDim.y = tasks + 1.  CTAs (x, y < tasks) store: where a RUN begins among the `span` tokens from x * span, the tokens that follow one
// another in one page, a warp takes the keys or the values of one kv head of the run.  CTAs (x, tasks) rotate the q of those
// tokens, eight pairs of entries to a thread.
// Where runs begin is not known to the host.  One token to a CTA as long as all are resident at once: each of a decode batch is a
// run of its own, and four runs one after another take four times as long.  Four to a CTA beyond: most tokens of a prompt
// begin no run, and the CTAs are handed out one by one.
// What bounds it is the way from the slots to the rows to the block's largest magnitude to the bytes; what does not depend on one
// another is asked for together.  32 / 8 heads of 64: 8 single tokens 3.7 us, a prompt of 2,048 tokens 11.4 us (2.0 TB/s); nine portions
// of 1 to 700 tokens at head size 128 26.7 us (2.3 TB/s).  The look at all earlier tokens before a run is stored grows with the square: 16,384
// tokens 94 us (1.9 TB/s), 65,536 679 us (1.1 TB/s).
template <typename T>
__global__ void __launch_bounds__(kWriteThreads, 3)
kv8_write_kernel(const Kv8WriteArgs<T> a, int span, int tasks) {
  pdl_wait();
  pdl_launch();
  constexpr int CH = kD / 16, TPR = kWriteTokens;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t0 = blockIdx.x * span, ps = 1 << a.page_shift;
  if (static_cast<int>(blockIdx.y) == tasks) {
    if (a.q_out == nullptr) return;
    const int per = a.hq * CH, n = min(span, a.tokens - t0) * per;
#pragma unroll 2
    for (int i = threadIdx.x; i < n; i += kWriteThreads) {
      const int t = t0 + i / per, rest = i % per, col = rest / CH * kD + rest % CH * 8;
      const T* src = a.qkv + static_cast<size_t>(t) * a.qkv_stride + col;
      float x0[8], x1[8];
      load8(src, x0);
      load8(src + kD / 2, x1);
      if (a.cos != nullptr) {
        const size_t at = static_cast<size_t>(kv8_position(a, a.positions[t])) * (kD / 2) + rest % CH * 8;
        float c[8], s[8];
        load8(a.cos + at, c);
        load8(a.sin + at, s);
        kv8_rotate8(x0, x1, c, s);
      }
      T* dst = a.q_out + static_cast<size_t>(t) * a.q_stride + col;
      store8(dst, x0);
      store8(dst + kD / 2, x1);
    }
    return;
  }
  // the slots of the token before, of the CTA's and of those after them (lane l: token t0 - 1 + l)
  long long theirs = -1;
  if (t0 - 1 + lane >= 0 && t0 - 1 + lane < a.tokens) theirs = kv8_slot(a, t0 - 1 + lane);
  const int w = blockIdx.y * kWriteWarps + warp;           // keys of kv head w, or values of kv head w - hkv
  const bool busy = w < 2 * a.hkv, is_v = w >= a.hkv;
  const int h = is_v ? w - a.hkv : w;
  const int tl = lane / CH, ch = lane - tl * CH;
  for (int l = 1; l <= span; ++l) {                        // (the same for the whole CTA)
    const int t = t0 + l - 1;
    const long long slot = __shfl_sync(0xffffffffu, theirs, l);
    if (slot < 0) continue;
    if (slot >= a.num_slots) {
      if (threadIdx.x == 0) atomicOr(a.status, 4);
      continue;
    }
    const int off = static_cast<int>(slot & (ps - 1));
    const long long page = slot >> a.page_shift;
    // (an item is a run of its own: the attention's kernel, where it stores itself, could not take two)
    if (a.items == nullptr && off > 0 && __shfl_sync(0xffffffffu, theirs, l - 1) == slot - 1) continue;      // not the first of its run
    int n = 1;                                             // tokens of the run
    if (a.items == nullptr) {
      // (lane l has its first token; those before stand for themselves)
      unsigned m = __ballot_sync(0xffffffffu, lane < l || (off + lane - l < ps && theirs == slot + lane - l));
      n = m == 0xffffffffu ? 32 - l : __ffs(~m) - 1 - l;
      while (n >= 32 - l && off + n < ps) {
        const int i = n + lane;
        m = __ballot_sync(0xffffffffu, t + i < a.tokens && off + i < ps && kv8_slot(a, t + i) == slot + i);
        if (m != 0xffffffffu) {
          n += __ffs(~m) - 1;
          break;
        }
        n += 32;
      }
    }
    const T* src = a.qkv + static_cast<size_t>(a.hq + w) * kD + ch * 8;
    const bool turn = !is_v && a.cos != nullptr;
    auto load = [&](int i, float* x) {                     // token i of the run
      const T* p = src + static_cast<size_t>(a.items != nullptr ? a.items[t + i].x : t + i) * a.qkv_stride;
      load8(p, x);
      load8(p + kD / 2, x + 8);
      if (turn) {
        const int pos = a.items != nullptr ? a.items[t + i].z - 1 : a.positions[t + i];
        const size_t at = static_cast<size_t>(kv8_position(a, pos)) * (kD / 2) + ch * 8;
        float c[8], s[8];
        load8(a.cos + at, c);
        load8(a.sin + at, s);
        kv8_rotate8(x, x + 8, c, s);
      }
    };
    const bool lanes = busy && tl < TPR;
    float kept[kWriteRounds][16];
#pragma unroll
    for (int r = 0; r < kWriteRounds; ++r)
      if (lanes && tl + r * TPR < n) load(tl + r * TPR, kept[r]);
    uint8_t* scale = (is_v ? a.vscale : a.kscale) + static_cast<size_t>(page) * a.hkv + h;
    const int old = busy && off > 0 ? min(static_cast<int>(*scale), 254) : 0;
    // Two runs of one page in one call would each set its scale without the other's: only the first is stored.  (Page 0
    // is the reserved one that padding rows write to: nothing to tell of there.)  Two items of one sequence likewise.
    bool before = false;
    const int seq = a.items != nullptr ? a.items[t].y : 0;
    for (int i = threadIdx.x; i < t; i += kWriteThreads) {
      const long long s = kv8_slot(a, i);
      before |= s >= 0 && (s >> a.page_shift) == page;
    }
    if (a.items != nullptr)
      for (int i = threadIdx.x; i < t; i += kWriteThreads) before |= a.items[i].z > 0 && a.items[i].y == seq;
    if (__syncthreads_or(before)) {                        // (every thread has read its scale)
      if (threadIdx.x == 0 && page != 0) atomicOr(a.status, 8);
      continue;
    }
    if (!busy) continue;
    float amax = 0.f;
    auto largest = [&](const float* x) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float u = fabsf(x[e]);
        amax = fmaxf(amax, u < INFINITY ? u : 0.f);
      }
    };
#pragma unroll
    for (int r = 0; r < kWriteRounds; ++r)
      if (lanes && tl + r * TPR < n) largest(kept[r]);
    if (lanes)
      for (int i = tl + kWriteRounds * TPR; i < n; i += TPR) {
        float x[16];
        load(i, x);
        largest(x);
      }
    amax = warp_max(amax);
    uint8_t* cache = is_v ? a.vcache : a.kcache;
    uint8_t* base = cache + (static_cast<size_t>(page) * a.hkv + h) * (static_cast<size_t>(ps) * kD);
    const int code = max(kv8_code(amax), old);
    if (off > 0 && code > old) {                           // what is in the page goes over to the larger scale
      const float f = kv8_exp2i(max(old - code, -127));
      for (int c = lane; c < off * (kD / 16); c += 32) {
        uint4* p = reinterpret_cast<uint4*>(base) + c;
        float x[16];
        kv8_f16(*p, x);
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] *= f;
        *p = make_uint4(kv8_pack4(x), kv8_pack4(x + 4), kv8_pack4(x + 8), kv8_pack4(x + 12));
      }
    }
    if (lane == 0) *scale = static_cast<uint8_t>(code);
    const float inv = kv8_exp2i(127 - code);
    auto put = [&](int i, float* x) {
#pragma unroll
      for (int e = 0; e < 16; ++e)                         // (what is not finite is stored as not a number, and left out of the scale)
        x[e] = fabsf(x[e]) < INFINITY ? x[e] * inv : __uint_as_float(0x7fc00000u);
      uint8_t* dst = base + static_cast<size_t>(off + i) * kD + ch * 8;
      *reinterpret_cast<uint2*>(dst) = make_uint2(kv8_pack4(x), kv8_pack4(x + 4));
      *reinterpret_cast<uint2*>(dst + kD / 2) = make_uint2(kv8_pack4(x + 8), kv8_pack4(x + 12));
    };
#pragma unroll
    for (int r = 0; r < kWriteRounds; ++r)
      if (lanes && tl + r * TPR < n) put(tl + r * TPR, kept[r]);
    if (lanes)
      for (int i = tl + kWriteRounds * TPR; i < n; i += TPR) {
        float x[16];
        load(i, x);
        put(i, x);
      }
  }
}

// ------------------------------------------------------------------------------------------------ single tokens

constexpr int kUnit = 64;                  // keys of a unit of work (an absolute boundary; the largest page)
constexpr int kMaxItems = 1024;            // items whose first units are kept in shared memory

// The launch's units: start[i] is the first unit of item i (all its kv heads), start[nitems] their number.
// Called by all threads of the CTA; `start` is shared memory for nitems + 1.
__device__ __forceinline__ int kv8_units(const Kv8Args& a, int* start) {
  __shared__ int warp_sums[33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
  int run = 0;
  for (int i0 = 0; i0 < a.nitems; i0 += blockDim.x) {
    const int i = i0 + threadIdx.x;
    int n = 0;
    if (i < a.nitems) {
      const int ctx = a.items[i].z;
      if (ctx > 0) {
        const int lo = a.window > 0 && ctx > a.window ? ctx - a.window : 0;
        n = ((ctx - 1) / kUnit - lo / kUnit + 1) * a.hkv;
      }
    }
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    int below = 0, all = 0;
    for (int w = 0; w < nwarps; ++w) {
      if (w < warp) below += warp_sums[w];
      all += warp_sums[w];
    }
    if (i < a.nitems) start[i] = run + below + inc - n;
    run += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) start[a.nitems] = run;
  __syncthreads();
  return run;
}

// A share's part of one row: keys [key_lo, key_hi).
struct Kv8Segment {
  int item, kvh, tok, seq, ctx;
  int key_lo, key_hi;
  int next;                 // the unit after the segment
  int row_begin, row_end;   // the row's units
  bool whole;
};

// The shares: of q + 1 units the first `rem`, of q the others (never more shares than units).
struct Kv8Cut {
  int shares, q, rem;
  __device__ __forceinline__ Kv8Cut(int units, int most) {
    shares = min(most, units);
    q = shares > 0 ? units / shares : 0;
    rem = units - q * shares;
  }
  __device__ __forceinline__ int begin(int s) const { return s * q + min(s, rem); }
  __device__ __forceinline__ int of(int u) const {         // the share that unit u lies in
    const int big = rem * (q + 1);
    return u < big ? u / (q + 1) : rem + (u - big) / q;
  }
};

__device__ __forceinline__ Kv8Segment kv8_segment(const Kv8Args& a, const int* start, int u, int end) {
  int lo = 0, hi = a.nitems - 1;            // the largest i with start[i] <= u (items without keys have no units)
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (start[mid] <= u) lo = mid; else hi = mid - 1;
  }
  Kv8Segment g;
  g.item = lo;
  const int4 info = a.items[lo];
  g.tok = info.x;
  g.seq = info.y;
  g.ctx = info.z;
  const int first = a.window > 0 && g.ctx > a.window ? g.ctx - a.window : 0;
  const int u0 = first / kUnit, n = (g.ctx - 1) / kUnit - u0 + 1;
  g.kvh = (u - start[lo]) / n;
  g.row_begin = start[lo] + g.kvh * n;
  g.row_end = g.row_begin + n;
  g.next = min(end, g.row_end);
  g.key_lo = max(first, (u0 + u - g.row_begin) * kUnit);
  g.key_hi = min(g.ctx, (u0 + g.next - g.row_begin) * kUnit);
  g.whole = u == g.row_begin && g.next == g.row_end;
  return g;
}

// The pieces of a cut row, which shares s0 .. s1 have left, added in the order of the keys and written out, by `nwarps` warps: a warp to
// 32 (or 16) entries of a head.  First a lane to a piece, for the references and the weights, then an entry to a lane, the pieces' loads in
// flight together.  (place: of the first share, which ends with the row unless it begins with it; the others' is 0.)
template <typename T>
__device__ __noinline__ void kv8_merge(const float* part, int G, int s0, int s1, int place, T* out, int warp, int nwarps) {
  constexpr int W = kD % 32 == 0 ? 32 : 16, NB = kD / W;
  const int lane = threadIdx.x & 31;
  const int row = G * (kD + 4);
#pragma unroll 1
  for (int i = warp; i < G * NB; i += nwarps) {
    const int r = i / NB, d = (i - r * NB) * W + lane % W;
    const float* base = part + r * (kD + 4);
    auto piece = [&](int s) { return base + (static_cast<size_t>(s) * 2 + (s == s0 ? place : 0)) * row; };
    float top = -INFINITY, dtop = -INFINITY, den = 0.f, num = 0.f;
#pragma unroll 1
    for (int c = s0; c <= s1; c += 32) {                 // (32 pieces at a time; the sums so far are carried over)
      const bool in = c + lane <= s1;
      const float4 x = in ? __ldcg(reinterpret_cast<const float4*>(piece(c + lane) + kD)) : make_float4(-INFINITY, -INFINITY, 0.f, 0.f);
      const bool none = x.y == -INFINITY && x.z == 0.f;
      const float t = fmaxf(top, warp_max(x.y));
      const float dm = none ? 0.f : x.y - t, od = top == -INFINITY ? 0.f : top - t;
      const float dt = fmaxf(dtop + od, warp_max(none ? -INFINITY : x.x + dm));
      const float w = none ? 0.f : exp2f(x.x + dm - dt);
      num *= dtop == -INFINITY ? 0.f : exp2f(dtop + od - dt);
      den = den * exp2f(od) + warp_sum(none ? 0.f : x.z * exp2f(dm));
      top = t;
      dtop = dt;
      const int n = min(32, s1 - c + 1);
#pragma unroll 8
      for (int k = 0; k < n; ++k) num += __shfl_sync(0xffffffffu, w, k) * __ldcg(piece(c + k) + d);
    }
    if (lane < W)
      out[r * kD + d] = from_float<T>(num * exp2f(dtop) / den);
  }
}

constexpr int kGenThreads = 128;
constexpr int kGenHeads = 4;               // query heads in one pass over the keys
constexpr int kGenLanes = kD <= 16 ? 1 : kD <= 32 ? 2 : kD <= 64 ? 4 : kD <= 128 ? 8 : 16;     // lanes to a key: 16 entries each

// Single tokens on the CUDA cores.  A CTA to a share; a key to kGenLanes lanes of a warp, each with 16 entries of four
// query heads and their numerators in registers and a running (max, denominator) of its own keys.  For float32 and the head sizes and groups
// that the tensor-core kernel does not take; what bounds it is the conversions and products, 0.5 to 0.9 TB/s of the cache (32 / 8 heads in
// bfloat16: 8 x 4,096 keys at head size 64 69 us against 17, 1 x 131,072 at 128 353 against 58; 8 x 4,096 in float32 60 us, in
// bfloat16 with 10 / 2 heads of 80 70).
template <typename T>
__global__ void __launch_bounds__(kGenThreads)
kv8_decode_kernel(const Kv8Args a) {
  __shared__ int start[kMaxItems + 1];
  __shared__ float parts[kGenThreads / 32][kGenHeads][kD + 2];
  __shared__ int last;
  pdl_launch();
  pdl_wait();
  constexpr float kLog2e = 1.4426950408889634f;
  constexpr int KPW = 32 / kGenLanes;       // keys that a warp takes at once
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int G = a.hq / a.hkv, ps = 1 << a.page_shift;
  const int ch = lane % kGenLanes, slot = lane / kGenLanes;
  const bool in_head = ch * 16 < kD;
  const Kv8Cut cut(kv8_units(a, start), gridDim.x);
  if (static_cast<int>(blockIdx.x) >= cut.shares) return;
  bool bad = false;                          // a page id beyond the pool
  const int begin = cut.begin(blockIdx.x), end = cut.begin(blockIdx.x + 1);
  for (int u = begin; u < end;) {
    const Kv8Segment g = kv8_segment(a, start, u, end);
    const int32_t* bt = a.block_table + static_cast<size_t>(g.seq) * a.max_blocks;
    float* piece = a.part + (static_cast<size_t>(blockIdx.x) * 2 + (u == begin ? 0 : 1)) * (G * (kD + 4));
    for (int g0 = 0; g0 < G; g0 += kGenHeads) {
      const int ng = min(kGenHeads, G - g0);
      float q[kGenHeads][16], acc[kGenHeads][16], m[kGenHeads], l[kGenHeads];
#pragma unroll
      for (int h = 0; h < kGenHeads; ++h) {
        m[h] = -INFINITY;
        l[h] = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) q[h][e] = acc[h][e] = 0.f;
        if (h < ng && in_head) {
          const T* row = static_cast<const T*>(a.q) + static_cast<size_t>(g.tok) * a.q_stride + (g.kvh * G + g0 + h) * kD;
          load8(row + ch * 16, q[h]);
          load8(row + ch * 16 + 8, q[h] + 8);
          if (a.cos != nullptr) {           // the other half's entries come from the row, too
            int pos = g.ctx - 1;
            if (pos >= a.max_pos) {
              atomicOr(a.status, 2);
              pos = 0;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int d = ch * 16 + e, dh = d < kD / 2 ? d : d - kD / 2;
              const float other = to_float(row[d < kD / 2 ? d + kD / 2 : dh]);
              const float c = a.cos[static_cast<size_t>(pos) * (kD / 2) + dh], s = a.sin[static_cast<size_t>(pos) * (kD / 2) + dh];
              q[h][e] = d < kD / 2 ? q[h][e] * c - other * s : q[h][e] * c + other * s;
            }
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) q[h][e] *= a.scale * kLog2e;
        }
      }
      // (the trip count is the same for all lanes of a warp: the shuffles below need all of them)
      for (int k0 = g.key_lo + warp * KPW; k0 < g.key_hi; k0 += KPW * (kGenThreads / 32)) {
        const int key = k0 + slot;
        const bool live = key < g.key_hi;
        const size_t block = static_cast<size_t>(kv8_page(bt[(live ? key : k0) >> a.page_shift], a.pages, bad)) * a.hkv + g.kvh;
        const size_t at = (block * ps + (key & (ps - 1))) * kD + ch * 16;
        float s[kGenHeads] = {};
        uint4 vraw = make_uint4(0, 0, 0, 0);
        if (live && in_head) {
          const uint4 kraw = *reinterpret_cast<const uint4*>(a.kcache + at);
          vraw = *reinterpret_cast<const uint4*>(a.vcache + at);
          float k[16];
          kv8_f16(kraw, k);
#pragma unroll
          for (int h = 0; h < kGenHeads; ++h)
#pragma unroll
            for (int e = 0; e < 16; ++e) s[h] += q[h][e] * k[e];
        }
#pragma unroll
        for (int h = 0; h < kGenHeads; ++h)
#pragma unroll
          for (int o = 1; o < kGenLanes; o <<= 1) s[h] += __shfl_xor_sync(0xffffffffu, s[h], o);
        if (live) {
          const float ks = kv8_scale(a.kscale[block]), vs = kv8_scale(a.vscale[block]);
          float v[16];
          kv8_f16(vraw, v);
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] *= vs;
#pragma unroll
          for (int h = 0; h < kGenHeads; ++h) {
            const float x = s[h] * ks;
            if (x > m[h]) {
              const float f = exp2f(m[h] - x);           // 0 the first time
              l[h] *= f;
#pragma unroll
              for (int e = 0; e < 16; ++e) acc[h][e] *= f;
              m[h] = x;
            }
            // (a score that is not a number makes the row not a number; one of -inf weighs nothing)
            const float p = x == -INFINITY ? 0.f : exp2f(x - m[h]);
            l[h] += p;
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[h][e] += p * v[e];
          }
        }
      }
      // the warp's slots, then its partial result
#pragma unroll
      for (int h = 0; h < kGenHeads; ++h) {
#pragma unroll
        for (int o = kGenLanes; o < 32; o <<= 1) {
          const float om = __shfl_xor_sync(0xffffffffu, m[h], o), ol = __shfl_xor_sync(0xffffffffu, l[h], o);
          const float mn = fmaxf(m[h], om);
          const float f = m[h] == -INFINITY ? 0.f : exp2f(m[h] - mn), w = om == -INFINITY ? 0.f : exp2f(om - mn);
          l[h] = l[h] * f + ol * w;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float oa = __shfl_xor_sync(0xffffffffu, acc[h][e], o);
            acc[h][e] = acc[h][e] * f + oa * w;
          }
          m[h] = mn;
        }
        if (slot == 0 && in_head) {
#pragma unroll
          for (int e = 0; e < 16; ++e) parts[warp][h][ch * 16 + e] = acc[h][e];
          if (ch == 0) {
            parts[warp][h][kD] = m[h];
            parts[warp][h][kD + 1] = l[h];
          }
        }
      }
      __syncthreads();
      for (int i = threadIdx.x; i < ng * kD; i += kGenThreads) {
        const int h = i / kD, d = i - h * kD;
        float mx = -INFINITY, den = 0.f, num = 0.f;
#pragma unroll
        for (int w = 0; w < kGenThreads / 32; ++w) mx = fmaxf(mx, parts[w][h][kD]);
#pragma unroll
        for (int w = 0; w < kGenThreads / 32; ++w) {
          const float f = parts[w][h][kD] == -INFINITY ? 0.f : exp2f(parts[w][h][kD] - mx);
          den += f * parts[w][h][kD + 1];
          num += f * parts[w][h][d];
        }
        const int r = g0 + h;
        if (g.whole) {
          static_cast<T*>(a.out)[static_cast<size_t>(g.tok) * a.out_stride + (g.kvh * G + r) * kD + d] = from_float<T>(num / den);
        } else {
          piece[r * (kD + 4) + d] = num;
          if (d == 0) *reinterpret_cast<float4*>(piece + r * (kD + 4) + kD) = make_float4(0.f, mx, den, 0.f);
        }
      }
      __syncthreads();
    }
    if (!g.whole) {
      __threadfence();                       // the piece, before it is counted
      __syncthreads();
      if (threadIdx.x == 0) {
        int* c = a.counters + static_cast<size_t>(g.item) * a.hkv + g.kvh;
        last = atomicAdd(c, 1) == cut.of(g.row_end - 1) - cut.of(g.row_begin);
        if (last) *c = 0;
      }
      __syncthreads();
      if (last) {
        __threadfence();
        const int s0 = cut.of(g.row_begin);
        kv8_merge<T>(a.part, G, s0, cut.of(g.row_end - 1), cut.begin(s0) != g.row_begin ? 1 : 0,
                     static_cast<T*>(a.out) + static_cast<size_t>(g.tok) * a.out_stride + g.kvh * G * kD, warp, kGenThreads / 32);
      }
      __syncthreads();
    }
    u = g.next;
  }
  if (bad) atomicOr(a.status, a.bad_page);
}

template <typename T>
struct Kv8PrefillArgs {
  static constexpr bool kEightBit = true;      // (what the kernel of prefill_tc.cuh goes by)
  const T* q;
  int q_stride;
  const uint8_t* kcache;
  const uint8_t* vcache;
  const uint8_t* kscale;
  const uint8_t* vscale;
  const int32_t* block_table;
  int max_blocks;
  const int32_t* tile_seq;
  const int32_t* tile_tok;
  const int32_t* tile_rows;
  const int32_t* positions;
  T* out;
  int out_stride;
  int hq, hkv, page_shift, window;
  float scale;
  int pages;                                   // of the pool
};

}  // namespace rl

#if RL_HEAD_DIM == 64 || RL_HEAD_DIM == 128
#include "kv8_decode_tc.cuh"
#include "prefill_tc.cuh"
#define RL_KV8_TC 1
#endif

namespace rl {

// ------------------------------------------------------------------------------------------------ portions of prompts

constexpr int kPR = 64, kPK = 64, kPreThreads = 256;      // query rows and keys of a tile
constexpr int kPLd = 68;                                  // floats to a row of 64 in shared memory
constexpr size_t kPreSmem = sizeof(float) * (2 * kD * kPLd + kPK * kD + kPK * kPLd);

// Rows tok0 .. + rows of one head once more, R to a warp.
template <typename T>
__device__ __noinline__ void kv8_prefill_again(const Kv8PrefillArgs<T>& a, int seq, int tok0, int rows, int pos0, int head) {
  typedef Kv8Rows<kD> Rows;
  const int lane = threadIdx.x & 31, at = head * kD + lane * Rows::E;
#pragma unroll 1
  for (int r0 = (threadIdx.x >> 5) * Rows::R; r0 < rows; r0 += kPreThreads / 32 * Rows::R) {
    float q[Rows::R][Rows::E] = {}, o[Rows::R][Rows::E], top, den;
#pragma unroll
    for (int r = 0; r < Rows::R; ++r)
      if (Rows::in_head(lane) && r0 + r < rows)
#pragma unroll
        for (int e = 0; e < Rows::E; ++e) q[r][e] = to_float(a.q[static_cast<size_t>(tok0 + r0 + r) * a.q_stride + at + e]);
    const int mine = r0 + Rows::row_of(lane), pos = pos0 + mine;
    kv8_rows<kD>(a, seq, head / (a.hq / a.hkv), a.window > 0 && pos + 1 > a.window ? pos + 1 - a.window : 0, mine < rows ? pos + 1 : 0,
                 a.scale * 1.4426950408889634f, lane, q, o, top, den);
#pragma unroll
    for (int r = 0; r < Rows::R; ++r) {
      const float d = __shfl_sync(0xffffffffu, den, r * 4 * Rows::L);
      if (Rows::in_head(lane) && r0 + r < rows)
#pragma unroll
        for (int e = 0; e < Rows::E; ++e) a.out[static_cast<size_t>(tok0 + r0 + r) * a.out_stride + at + e] = from_float<T>(o[r][e] / d);
    }
  }
}

// Portions of prompts on the CUDA cores: a CTA to 64 consecutive query rows (half a tile of the launch) of one head;
// keys in tiles of 64.  Thread (ty, tx) has rows 4 ty .. + 3; of S their keys 4 tx .. + 3 (operands as four rows and four
// keys side by side: two 16-byte reads for 16 products), of O their columns tx + 16 j.  For float32 and the head sizes that the tcgen05
// kernel does not take (bfloat16 at 64: 2,048 tokens behind 6,144 keys 5,520 us against 254); float32, four portions of 33 to 129 tokens, 3 / 1
// heads of 128: 46 us; 512 tokens behind 512 in bfloat16, 12 / 4 heads of 96, 243 us.  What bounds it is the FFMA pipe and the
// reads of its operands from shared memory; few items do not fill the SMs.
template <typename T>
__global__ void __launch_bounds__(kPreThreads)
kv8_prefill_kernel(const __grid_constant__ Kv8PrefillArgs<T> a, int* status) {
  extern __shared__ __align__(16) float tiles[];
  float* qs = tiles;                        // [D][68], scaled
  float* ks = qs + kD * kPLd;               // [D][68]
  float* vs = ks + kD * kPLd;               // [64][D]
  float* ps = vs + kPK * kD;                // [64 keys][68]
  constexpr float kLog2e = 1.4426950408889634f;
  constexpr int NC = kD / 16;
  pdl_launch();
  pdl_wait();
  const int tile = blockIdx.x >> 1, head = blockIdx.y, kvh = head / (a.hq / a.hkv);
  const int half = (blockIdx.x & 1) * kPR;
  const int rows = min(a.tile_rows[tile] - half, kPR);
  if (rows <= 0) return;
  const int tok0 = a.tile_tok[tile] + half;
  const int pos0 = a.positions[tok0], page = 1 << a.page_shift;
  const int32_t* bt = a.block_table + static_cast<size_t>(a.tile_seq[tile]) * a.max_blocks;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  for (int i = threadIdx.x; i < kPR * (kD / 8); i += kPreThreads) {
    const int r = i % kPR, c = i / kPR;
    float x[8] = {};
    if (r < rows) load8(a.q + static_cast<size_t>(tok0 + r) * a.q_stride + head * kD + c * 8, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) qs[(c * 8 + e) * kPLd + r] = x[e] * (a.scale * kLog2e);
  }
  const int k_end = pos0 + rows;
  const int first = a.window > 0 && pos0 + 1 > a.window ? pos0 + 1 - a.window : 0;
  float m[4], l[4], acc[4][NC];
  bool bad = false;                                       // a page id beyond the pool
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int j = 0; j < NC; ++j) acc[i][j] = 0.f;
  }
  for (int k0 = first / kPK * kPK; k0 < k_end; k0 += kPK) {
    __syncthreads();
    for (int i = threadIdx.x; i < kPK * (kD / 16); i += kPreThreads) {
      const int key = i % kPK, c = i / kPK, j = k0 + key;
      float k[16] = {}, v[16] = {};
      if (j < k_end && j >= first) {
        const size_t block = static_cast<size_t>(kv8_page(bt[j >> a.page_shift], a.pages, bad)) * a.hkv + kvh;
        const size_t at = (block * page + (j & (page - 1))) * kD + c * 16;
        const float fk = kv8_scale(a.kscale[block]), fv = kv8_scale(a.vscale[block]);
        kv8_f16(*reinterpret_cast<const uint4*>(a.kcache + at), k);
        kv8_f16(*reinterpret_cast<const uint4*>(a.vcache + at), v);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          k[e] *= fk;
          v[e] *= fv;
        }
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        ks[(c * 16 + e) * kPLd + key] = k[e];
        vs[key * kD + c * 16 + e] = v[e];
      }
    }
    __syncthreads();
    float s[4][4] = {};
#pragma unroll 4
    for (int d = 0; d < kD; ++d) {
      const float4 x = *reinterpret_cast<const float4*>(qs + d * kPLd + ty * 4);
      const float4 y = *reinterpret_cast<const float4*>(ks + d * kPLd + tx * 4);
      const float xr[4] = {x.x, x.y, x.z, x.w}, yr[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] += xr[i] * yr[j];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int pos = pos0 + ty * 4 + i;
      const int lo = a.window > 0 && pos + 1 > a.window ? pos + 1 - a.window : 0;
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = k0 + tx * 4 + j;
        if (key > pos || key < lo) s[i][j] = -INFINITY;
        top = fmaxf(top, s[i][j]);
      }
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float mn = fmaxf(m[i], top);
      const float use = mn == -INFINITY ? 0.f : mn;       // (no key of the row yet)
      const float f = m[i] == -INFINITY ? 0.f : exp2f(m[i] - use);
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = exp2f(s[i][j] - use);
        sum += s[i][j];
      }
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      l[i] = l[i] * f + sum;
      m[i] = mn;
#pragma unroll
      for (int j = 0; j < NC; ++j) acc[i][j] *= f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<float4*>(ps + (tx * 4 + j) * kPLd + ty * 4) = make_float4(s[0][j], s[1][j], s[2][j], s[3][j]);
    __syncwarp();                                          // (a row's sixteen threads are half a warp)
#pragma unroll 4
    for (int c = 0; c < kPK; ++c) {
      const float4 p = *reinterpret_cast<const float4*>(ps + c * kPLd + ty * 4);
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        const float v = vs[c * kD + tx + 16 * j];
        acc[0][j] += p.x * v;
        acc[1][j] += p.y * v;
        acc[2][j] += p.z * v;
        acc[3][j] += p.w * v;
      }
    }
  }
  if (bad) atomicOr(status, kKv8BadPage);
  // A value that is not a number reaches the rows that see its key and no others, which a weight of 0 does not see to: rows that come out
  // not finite are done once more by themselves.  (With a look at every weight in the tiles that reach past a row's own key four short
  // portions took 59 us instead of 51.)
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NC; ++j) odd |= !(fabsf(acc[i][j]) < INFINITY);
  if (__syncthreads_or(odd)) {
    kv8_prefill_again<T>(a, a.tile_seq[tile], tok0, rows, pos0, head);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = ty * 4 + i;
    if (r >= rows) continue;
    const float inv = 1.f / l[i];
#pragma unroll
    for (int j = 0; j < NC; ++j)
      a.out[static_cast<size_t>(tok0 + r) * a.out_stride + head * kD + tx + 16 * j] = from_float<T>(acc[i][j] * inv);
  }
}

}  // namespace rl

using namespace rl;

namespace {

constexpr int kMaxDevices = 64;

int device_sms(int* sms) {
  static int sms_of[kMaxDevices];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (dev < 0 || dev >= kMaxDevices) return static_cast<int>(cudaErrorInvalidDevice);
  if (sms_of[dev] == 0) {
    int n = 0;
    e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return static_cast<int>(e);
    sms_of[dev] = n > 0 ? n : 1;
  }
  *sms = sms_of[dev];
  return 0;
}

int shift_of(int page_size) {
  int s = 0;
  while ((1 << s) < page_size) ++s;
  return s;
}

template <typename T>
int launch_write(const void* qkv, int qkv_stride, const int32_t* positions, const int32_t* slots, const int4* items,
                 const int32_t* bt, int max_blocks, const float* cos, const float* sin, uint8_t* kc, uint8_t* vc, uint8_t* ks,
                 uint8_t* vs, void* q_out, int q_stride, int tokens, int hq, int hkv, int page_size, int max_pos,
                 long long num_slots, int* status, cudaStream_t stream) {
  Kv8WriteArgs<T> a;
  a.qkv = static_cast<const T*>(qkv);
  a.qkv_stride = qkv_stride;
  a.positions = positions;
  a.slots = slots;
  a.items = items;
  a.block_table = bt;
  a.max_blocks = max_blocks;
  a.cos = cos;
  a.sin = sin;
  a.kcache = kc;
  a.vcache = vc;
  a.kscale = ks;
  a.vscale = vs;
  a.q_out = static_cast<T*>(q_out);
  a.q_stride = q_stride;
  a.tokens = tokens;
  a.hq = hq;
  a.hkv = hkv;
  a.page_shift = shift_of(page_size);
  a.max_pos = max_pos;
  a.num_slots = num_slots;
  a.status = status;
  if (tokens == 0 || (slots == nullptr && items == nullptr && q_out == nullptr)) return 0;
  int sms = 0;
  const int e = device_sms(&sms);
  if (e) return e;
  const int tasks = slots != nullptr || items != nullptr ? (2 * hkv + kWriteWarps - 1) / kWriteWarps : 0;
  const int span = static_cast<long long>(tokens) * (tasks + 1) <= 4 * sms ? 1 : 4;
  launch_kernel(kv8_write_kernel<T>, dim3((tokens + span - 1) / span, tasks + (q_out != nullptr ? 1 : 0)), dim3(kWriteThreads), 0, stream, a,
                span, tasks);
  return static_cast<int>(cudaGetLastError());
}

// The largest number of shares that a launch is cut into, whatever the device: the workspace has two places for each.  (148 SMs
// times the 12 groups of a CTA.)
constexpr int kMaxShares = 1776;

// CTAs of a launch in shares, `groups` to a CTA, and pieces of a row, one to a CTA: as many as the device holds at once and the
// workspace has places for.
int shares_ctas(int resident, int groups) { return resident < kMaxShares / groups ? resident : kMaxShares / groups; }
int most_pieces(int resident, long long rows) {
  const long long k = (resident < kMaxShares ? resident : kMaxShares) / rows;
  return static_cast<int>(k < 48 ? k : 48);
}

#ifdef RL_KV8_TC

typedef void (*TcKernel)(Kv8Args, int, int);
const TcKernel kTcKernels[2] = {kv8_decode_tc_kernel<false>, kv8_decode_tc_kernel<true>};      // (true: groups of more than 8 heads)

struct TcDevice {
  bool ready;
  int sms;
  int resident[kMaxCluster + 1];     // clusters of so many CTAs that fit the device at once (one row's slots of 16 heads)
  int smem_most;
};

size_t tc_smem(int csize, int G) {
  return static_cast<size_t>(kDecWarps) * kRingBytes + (csize > 1 ? sizeof(float) * csize * G * kPartLd : 0);
}

// What is asked of the device once.
int tc_device(const TcDevice** out) {
  static TcDevice devices[kMaxDevices];
  static std::mutex lock;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (dev < 0 || dev >= kMaxDevices) return static_cast<int>(cudaErrorInvalidDevice);
  std::lock_guard<std::mutex> guard(lock);
  TcDevice& d = devices[dev];
  if (!d.ready) {
    int n = 0, most = 0;
    e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev);
    cudaFuncAttributes fa;
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&fa, kTcKernels[0]);
    if (e != cudaSuccess) return static_cast<int>(e);
    d.sms = n > 0 ? n : 1;
    d.smem_most = most - static_cast<int>(fa.sharedSizeBytes);
    for (TcKernel k : kTcKernels) {
      e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, d.smem_most);
      if (e != cudaSuccess) return static_cast<int>(e);
    }
    for (int c = 1; c <= kMaxCluster; ++c) {
      cudaLaunchConfig_t q = {};
      q.gridDim = dim3(c);
      q.blockDim = dim3(kDecThreads);
      q.dynamicSmemBytes = tc_smem(c, 1);
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim.x = c;
      at[0].val.clusterDim.y = 1;
      at[0].val.clusterDim.z = 1;
      q.attrs = at;
      q.numAttrs = 1;
      int k = 0;
      if (cudaOccupancyMaxActiveClusters(&k, kTcKernels[0], &q) != cudaSuccess) {
        cudaGetLastError();
        k = 0;
      }
      d.resident[c] = k;
    }
    if (d.resident[1] < 1) return static_cast<int>(cudaErrorNotSupported);
    d.ready = true;
  }
  *out = &d;
  return 0;
}

// How a launch's rows are shared out; see kv8_decode_tc_kernel.
struct TcPlan {
  int csize, groups, ctas, parts;      // parts: 0 rows, > 0 pieces of a row, -1 shares
};

// The CTAs of a row's cluster, and as few groups (a divisor of the warps) as give every row one at once, else a warp to a row.
void tc_rows(const TcDevice* d, long long rows, int G, int* csize, int* groups) {
  *csize = *groups = 1;
  for (int c = kMaxCluster; c > 1; --c)
    if (d->resident[c] >= rows && tc_smem(c, G) <= static_cast<size_t>(d->smem_most)) {
      *csize = c;
      return;
    }
  if (rows > d->resident[1]) {
    *groups = kDecWarps;
    for (int k = 2; k < kDecWarps; ++k)
      if (kDecWarps % k == 0 && static_cast<long long>(d->resident[1]) * k >= rows) {
        *groups = k;
        break;
      }
  }
}

// The pieces of a row where there is a CTA for each; the last to arrive adds them up, which takes some 0.2 us a piece.
int tc_pieces(const TcDevice* d, long long rows) { return most_pieces(d->resident[1], rows); }

// Which of rows (2), shares (3) and pieces (4) is expected to take the shortest, in us: a start; then the longest of a warp's
// run of sub-blocks, what the busiest SM reads and what all bytes take.  Fitted to 1017 launches (kv heads 1, 2 and 8, groups of
// four, 1 to 128 sequences of 256 to 131,072 keys, all equal or spread over L / 8 or L / 64 to L), over which the choice is 0.2 % longer
// than the best (1.19 times at the worst).  Rows / shares / pieces, us, with 8 kv heads: one sequence of 65,536 keys 33 / 34 / 25 at head
// size 64 and 47 / 48 / 38 at 128; 8 of 4,096 at head size 64 16 / 26 / 20; 24 of 1,024 to 8,192 at 128 76 / 62 / -.
int kv8_choice(const TcDevice* d, int nitems, int hq, int hkv, int max_ctx, double mean) {
  if (mean <= 0.0) return 2;
  const long long rows = static_cast<long long>(nitems) * hkv;
  int csize, groups;
  tc_rows(d, rows, hq / hkv, &csize, &groups);
  const bool narrow = kD == 64;
  const double lat = narrow ? 0.81 : 1.20, sm_rate = narrow ? 42e3 : 58e3, rate = narrow ? 20e6 : 6.4e6;
  const double key = kD * 2.0, bytes = rows * mean * key;
  auto longest = [](double a, double b, double c) { return a > b ? (a > c ? a : c) : (b > c ? b : c); };
  const double turns = csize == 1 ? (rows + static_cast<long long>(d->resident[1]) * groups - 1) / (static_cast<long long>(d->resident[1]) * groups) : 1;
  const int per_row = csize * (kDecWarps / groups);
  const double run = (max_ctx / kSub + per_row) / per_row + (turns - 1) * mean / kSub / per_row;
  const double by_rows = (narrow ? 6.5 : 7.4) + longest(run * lat, (max_ctx + (groups * turns - 1) * mean) * key / csize / sm_rate, bytes / rate);
  const double by_shares = (narrow ? 17.1 : 21.5) + bytes / (narrow ? 4.12e6 : 5.09e6);
  double by_pieces = 1e30;
  if (const int k = tc_pieces(d, rows)) {
    by_pieces = (narrow ? 11.7 : 14.6) + longest((max_ctx / kSub + k * kDecWarps) / (k * kDecWarps) * lat, max_ctx * key / k / sm_rate, bytes / (narrow ? 7.1e6 : 7.8e6));
  }
  return by_rows <= by_shares && by_rows <= by_pieces ? 2 : (by_pieces <= by_shares ? 4 : 3);
}

// impl 2: rows; 3: shares; 4: every row in as many pieces as there are CTAs for; 0: the one that is expected to be the
// fastest, from the longest context and the sum of all as the host knows them (sum_ctx 0: unknown).
int tc_plan(int nitems, int hq, int hkv, int max_ctx, long long sum_ctx, int impl, TcPlan* plan) {
  const TcDevice* d = nullptr;
  const int err = tc_device(&d);
  if (err) return err;
  const long long rows = static_cast<long long>(nitems) * hkv;
  const int resident = d->resident[1];
  plan->csize = 1;
  plan->groups = 1;
  plan->parts = 0;
  if (impl == 0) impl = kv8_choice(d, nitems, hq, hkv, max_ctx, static_cast<double>(sum_ctx) / nitems);
  if (impl == 4 && tc_pieces(d, rows) < 1) impl = 2;
  if (impl == 4) {
    plan->parts = tc_pieces(d, rows);
    plan->ctas = static_cast<int>(rows * plan->parts);
    return 0;
  }
  tc_rows(d, rows, hq / hkv, &plan->csize, &plan->groups);
  if (impl == 3) {
    plan->csize = 1;
    plan->parts = -1;
    plan->ctas = shares_ctas(resident, plan->groups);
    return 0;
  }
  const long long wanted = plan->csize > 1 ? rows : (rows + plan->groups - 1) / plan->groups;
  plan->ctas = static_cast<int>((wanted < resident || plan->csize > 1 ? wanted : resident) * plan->csize);
  return 0;
}

int launch_decode_tc(Kv8Args a, int max_ctx, long long sum_ctx, int impl, cudaStream_t stream) {
  TcPlan plan;
  const int err = tc_plan(a.nitems, a.hq, a.hkv, max_ctx, sum_ctx, impl, &plan);
  if (err) return err;
  const int G = a.hq / a.hkv, csize = plan.csize;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(plan.ctas);
  cfg.blockDim = dim3(kDecThreads);
  cfg.dynamicSmemBytes = tc_smem(csize, G);
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = csize;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kTcKernels[G > 8 ? 1 : 0], a, plan.groups, plan.parts));
}

#endif

}  // namespace

extern "C" {

// The arguments of the entry points: fields of eight bytes, packed by the caller.  (A foreign call with 30 arguments of its own
// took 8 us of one core, one with a packed argument takes 2.)
struct Kv8WriteCall {
  int64_t dtype;
  const void* qkv;
  int64_t qkv_stride;
  const int32_t *positions, *slots;
  const float *cos, *sin;
  uint8_t *kc, *vc, *ks, *vs;
  void* q_out;
  int64_t q_stride, tokens, hq, hkv, page_size, max_pos, num_slots;
  int* status;
  cudaStream_t stream;
};

// store: q holds the unrotated rows [q | k | v]; the tokens' keys and values are stored first (by the attention's kernel itself or a launch of
// their own), and the attention rotates q on its way in.
struct Kv8DecodeCall {
  int64_t dtype;
  const void* q;
  int64_t q_stride;
  uint8_t *kc, *vc, *ks, *vs;
  const int32_t* block_table;
  int64_t max_blocks;
  const int4* items;
  int64_t nitems;
  float* part;
  int* counters;
  void* out;
  int64_t out_stride, hq, hkv, page_size, window;
  double scale;
  const float *cos, *sin;
  int64_t max_pos, store, num_slots;
  int* status;
  int64_t max_ctx, sum_ctx, impl;
  int64_t bad_page;
  cudaStream_t stream;
};

struct Kv8PrefillCall {
  int64_t dtype;
  const void* q;
  int64_t q_stride;
  const uint8_t *kc, *vc, *ks, *vs;
  const int32_t* block_table;
  int64_t max_blocks;
  const int32_t *tile_seq, *tile_tok, *tile_rows, *positions;
  void* out;
  int64_t out_stride, tiles, hq, hkv, page_size, window;
  double scale;
  int64_t impl, pages;
  int* status;
  cudaStream_t stream;
};
static_assert(sizeof(Kv8WriteCall) == 21 * 8 && sizeof(Kv8DecodeCall) == 31 * 8 && sizeof(Kv8PrefillCall) == 25 * 8, "as they are packed");

// Which way of sharing out (2, 3 or 4; 0: the CUDA cores) a launch on the tensor cores would go by impl 0, or an error as a negative number.
int rl_kv8_decode_choice(int dtype, int nitems, int hq, int hkv, int max_ctx, long long sum_ctx) {
  if (hkv < 1 || hq < hkv) return -static_cast<int>(cudaErrorInvalidValue);
#ifdef RL_KV8_TC
  if (dtype == 1 && hq / hkv <= 16 && nitems > 0) {
    const TcDevice* d = nullptr;
    const int err = tc_device(&d);
    if (err) return -err;
    return kv8_choice(d, nitems, hq, hkv, max_ctx, static_cast<double>(sum_ctx) / nitems);
  }
#endif
  return 0;
}

// The most pieces that a launch leaves in the workspace on a device that holds `resident` CTAs of `groups` groups at once: in shares
// (rows 0) or with so many rows in pieces.
long long rl_kv8_most_pieces(int resident, int groups, int rows) {
  if (resident < 1 || groups < 1 || rows < 0) return -1;
  return rows == 0 ? static_cast<long long>(shares_ctas(resident, groups)) * groups : static_cast<long long>(rows) * most_pieces(resident, rows);
}

// The floats of the workspace for groups of G heads (kv8.cuh: Kv8Args::part).
long long rl_kv8_part_floats(int G) { return static_cast<long long>(kMaxShares) * 2 * G * (kD + 4); }

int rl_kv8_write(const Kv8WriteCall* c) {
  auto run = c->dtype == 0 ? launch_write<float> : launch_write<bf16>;
  return run(c->qkv, static_cast<int>(c->qkv_stride), c->positions, c->slots, nullptr, nullptr, 0, c->cos, c->sin, c->kc, c->vc, c->ks,
             c->vs, c->q_out, static_cast<int>(c->q_stride), static_cast<int>(c->tokens), static_cast<int>(c->hq),
             static_cast<int>(c->hkv), static_cast<int>(c->page_size), static_cast<int>(c->max_pos), c->num_slots, c->status, c->stream);
}

int rl_kv8_attn_decode(const Kv8DecodeCall* c) {
  const int nitems = static_cast<int>(c->nitems), hq = static_cast<int>(c->hq), hkv = static_cast<int>(c->hkv);
  const int page_size = static_cast<int>(c->page_size), impl = static_cast<int>(c->impl), max_pos = static_cast<int>(c->max_pos);
  const int max_ctx = static_cast<int>(c->max_ctx), q_stride = static_cast<int>(c->q_stride);
  const bool store = c->store != 0, single = c->dtype == 0;
  if (hkv < 1 || hq < hkv) return static_cast<int>(cudaErrorInvalidValue);
#ifdef RL_KV8_TC
  const bool takes = !single && hq / hkv <= 16;
#else
  const bool takes = false;
#endif
  if (impl > 1 && !takes) return static_cast<int>(cudaErrorInvalidValue);      // (before anything is stored)
  const bool tc = takes && impl != 1;
  int sms = 0;
  int e = device_sms(&sms);
  if (e) return e;
  // (pages of 64 tokens reach over two sub-blocks, which may be two warps': their tokens are stored by a kernel of its own)
  const bool fused = store && tc && page_size <= 32;
  if (store && !fused) {
    auto run = single ? launch_write<float> : launch_write<bf16>;
    e = run(c->q, q_stride, nullptr, nullptr, c->items, c->block_table, static_cast<int>(c->max_blocks), c->cos, c->sin, c->kc, c->vc,
            c->ks, c->vs, nullptr, 0, nitems, hq, hkv, page_size, max_pos, c->num_slots, c->status, c->stream);
    if (e) return e;
  }
  Kv8Args a;
  a.q = c->q;
  a.q_stride = q_stride;
  a.kcache = c->kc;
  a.vcache = c->vc;
  a.kscale = c->ks;
  a.vscale = c->vs;
  a.block_table = c->block_table;
  a.max_blocks = static_cast<int>(c->max_blocks);
  a.items = c->items;
  a.nitems = nitems;
  a.part = c->part;
  a.counters = c->counters;
  a.out = c->out;
  a.out_stride = static_cast<int>(c->out_stride);
  a.hq = hq;
  a.hkv = hkv;
  a.page_shift = shift_of(page_size);
  a.window = static_cast<int>(c->window);
  a.scale = static_cast<float>(c->scale);
  a.cos = store ? c->cos : nullptr;
  a.store = fused ? 1 : 0;
  a.sin = c->sin;
  a.max_pos = max_pos;
  a.pages = static_cast<int>(c->num_slots / page_size);
  a.status = c->status;
  a.bad_page = static_cast<int>(c->bad_page);
  for (int i0 = 0; i0 < nitems; i0 += kMaxItems) {         // (one launch unless there are very many items)
    a.items = c->items + i0;
    a.before = i0;
    a.nitems = nitems - i0 < kMaxItems ? nitems - i0 : kMaxItems;
#ifdef RL_KV8_TC
    if (tc) {
      e = launch_decode_tc(a, max_ctx, c->sum_ctx / nitems * a.nitems, impl, c->stream);
      if (e) return e;
      continue;
    }
#endif
    // a CTA to a unit, as far as they are resident together
    const long long max_units = static_cast<long long>(a.nitems) * hkv * (max_ctx / kUnit + 2);
    const int most = shares_ctas(sms * 2, 1);
    const int ctas = static_cast<int>(max_units < most ? max_units : most);
    if (single)
      launch_kernel(kv8_decode_kernel<float>, dim3(ctas), dim3(kGenThreads), 0, c->stream, a);
    else
      launch_kernel(kv8_decode_kernel<bf16>, dim3(ctas), dim3(kGenThreads), 0, c->stream, a);
    e = static_cast<int>(cudaGetLastError());
    if (e) return e;
  }
  return 0;
}

}  // extern "C"

namespace {

template <typename T>
int launch_prefill(const void* q, int q_stride, const void* kc, const void* vc, const void* ks, const void* vs, const int32_t* bt,
                   int max_blocks, const int32_t* tile_seq, const int32_t* tile_tok, const int32_t* tile_rows,
                   const int32_t* positions, void* out, int out_stride, int tiles, int hq, int hkv, int page_size, int window,
                   float scale, int impl, int pages, int* status, cudaStream_t stream) {
  Kv8PrefillArgs<T> a;
  a.q = static_cast<const T*>(q);
  a.q_stride = q_stride;
  a.kcache = static_cast<const uint8_t*>(kc);
  a.vcache = static_cast<const uint8_t*>(vc);
  a.kscale = static_cast<const uint8_t*>(ks);
  a.vscale = static_cast<const uint8_t*>(vs);
  a.block_table = bt;
  a.max_blocks = max_blocks;
  a.tile_seq = tile_seq;
  a.tile_tok = tile_tok;
  a.tile_rows = tile_rows;
  a.positions = positions;
  a.out = static_cast<T*>(out);
  a.out_stride = out_stride;
  a.hq = hq;
  a.hkv = hkv;
  a.page_shift = shift_of(page_size);
  a.window = window;
  a.scale = scale;
  a.pages = pages;
  static bool simt_set[kMaxDevices];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (dev < 0 || dev >= kMaxDevices) return static_cast<int>(cudaErrorInvalidDevice);
#ifdef RL_KV8_TC
  if constexpr (sizeof(T) == 2) {
    if (impl != 1) {
      int sms = 0;
      const int err = device_sms(&sms);
      if (err) return err;
      static bool tc_set[kMaxDevices];
      if (!tc_set[dev]) {
        e = cudaFuncSetAttribute(prefill_attn_tc_kernel<Kv8PrefillArgs<bf16>>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(kPrefillTcSmem8));
        if (e != cudaSuccess) return static_cast<int>(e);
        tc_set[dev] = true;
      }
      const long long work = static_cast<long long>(tiles) * hkv * ((hq / hkv + 1) / 2);     // (tile, kv head, pair of heads)
      launch_kernel(prefill_attn_tc_kernel<Kv8PrefillArgs<bf16>>, dim3(static_cast<unsigned>(work < sms ? work : sms)), dim3(kTcThreads8),
                    kPrefillTcSmem8, stream, a, tiles, status);
      return static_cast<int>(cudaGetLastError());
    }
  }
#endif
  if (impl > 1) return static_cast<int>(cudaErrorInvalidValue);
  if (!simt_set[dev]) {
    e = cudaFuncSetAttribute(kv8_prefill_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kPreSmem));
    if (e != cudaSuccess) return static_cast<int>(e);
    simt_set[dev] = true;
  }
  launch_kernel(kv8_prefill_kernel<T>, dim3(tiles * 2, hq), dim3(kPreThreads), kPreSmem, stream, a, status);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace

extern "C" int rl_kv8_attn_prefill(const Kv8PrefillCall* c) {
  if (c->hkv < 1 || c->hq < c->hkv) return static_cast<int>(cudaErrorInvalidValue);
  auto run = c->dtype == 0 ? launch_prefill<float> : launch_prefill<bf16>;
  return run(c->q, static_cast<int>(c->q_stride), c->kc, c->vc, c->ks, c->vs, c->block_table, static_cast<int>(c->max_blocks), c->tile_seq,
             c->tile_tok, c->tile_rows, c->positions, c->out, static_cast<int>(c->out_stride), static_cast<int>(c->tiles),
             static_cast<int>(c->hq), static_cast<int>(c->hkv), static_cast<int>(c->page_size), static_cast<int>(c->window),
             static_cast<float>(c->scale), static_cast<int>(c->impl), static_cast<int>(c->pages), c->status, c->stream);
}
