// Single tokens over the 8-bit cache on the tensor cores (bfloat16 rows, head size 64 or 128, up to 16 query heads to a kv head).
//
// Included by kv8.cu.  A row is a (item, kv head).  A GROUP of warps takes a row, or a share of one, at a time; its live keys
// are cut into as many equal runs of sub-blocks (32 keys) as the group has warps.  Every warp is a pipeline of its own:
// the sub-blocks of its run come by 16-byte asynchronous copies into a private ring, 8 to 16 KB on their way while one is worked on
// (44 KB an SM cover the way from DRAM at full rate).  A sub-block:
//   S = Q K^T    mma.sync.m16n8k16 on halves: an e4m3 number is a half exactly (one conversion for two); q is scaled by a power of
//                two per row to at most 256 and rounded to 11 bits.  (The same instruction on e4m3 bytes is put together from
//                conversions, two products on halves and sums on this machine; it took 1.5 times as long.)  Which entries of the head a
//                k index of the product stands for is free, so a lane's 16 bytes of a key are four k steps of the B
//                fragment as they lie.
//   softmax      online, in log2 units: the denominator sums 2^(x - m), m the largest score; the weights for the product are
//                2^(x - m + e - d), e the exponent of the page's value scale and d the largest x - m + e, so that they keep
//                their bits whatever scales lie side by side (pages of zeros among them) and O needs no factor a page
//   O += P V     P as halves, scaled to at most 2^14: 11 bits down to 2^-28 of the run's largest weight.  ldmatrix transposes 16 x 16
//                bytes of V: four keys of an entry in a word
// Page ids and scales are fetched a window of 32 pages at a time, a page to a lane, and the window after it behind that.
//
// Where rows are shared out (see launch_decode_tc for the choice):
//   rows    a cluster of up to 8 CTAs to a row, whose partial results meet in the first one's shared memory; or, with more rows
//           than clusters can be resident, CTAs whose warps form groups that take a row each, one after another
//   shares  the launch's keys in equal shares, one to a group (kv8.cuh): for rows of very different lengths
#pragma once

namespace rl {

constexpr int kTcWarps = kD == 64 ? 12 : 8, kTcThreads = kTcWarps * 32;
constexpr int kSub = 32;                                 // keys of a sub-block
constexpr int kSubBytes = kSub * kD;                     // K (or V) of one
constexpr int kRing = kD == 64 ? 4 : 3;                  // (192 KB for all warps either way)
constexpr int kRingBytes = kRing * 2 * kSubBytes;
constexpr int kHeadBytes = kRing * 16;                   // the scales of a warp's stages: (K, log2 of V) of the first 16 keys and of the second
constexpr int kMaxCluster = 8;
constexpr int kPartLd = kD + 4;                          // floats to a head in a warp's partial result: kd numerators, d, m, denominator
static_assert(16 * kPartLd * 4 <= kRingBytes, "a warp's partial result lies in its own ring");

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void copy16(uint32_t smem, const void* gmem) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(smem), "l"(gmem));
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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
__device__ __forceinline__ void mma_f16_first(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
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
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// A float to this CTA's address p in CTA `rank` of the cluster.
__device__ __forceinline__ void store_cluster(float* p, uint32_t rank, float v) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_addr(p)), "r"(rank));
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote), "f"(v) : "memory");
}

// One warp's result for its run; thread (g, t) holds, of head g, entries 8 j + 2 t + e at o[j][e], and of head g + 8 (HI)
// at o[j][2 + e].
struct TcState {
  float o[kD / 8][4];
  float m[2], d[2], l[2];        // (the same for a row's four lanes, but for the denominator of the lane's own keys)
};

// q of the segment's token as A fragments (k step by k step; the rows g and g + 8, and both once more for the step's second
// half), rotated on the way if the tables are given, and the factor of the exponent.
template <bool HI>
__device__ __forceinline__ void tc_load_q(const Kv8Args& a, const Kv8Segment& s, int lane, uint32_t (*qf)[HI ? 4 : 2], float* factor) {
  constexpr float kLog2e = 1.4426950408889634f;
  constexpr int NC = kD / 64;                            // 16-entry pieces of a head to a lane: entries 64 c + 16 t ..
  const int g = lane >> 2, t = lane & 3, G = a.hq / a.hkv;
#pragma unroll
  for (int h = 0; h < (HI ? 2 : 1); ++h) {
    const int r = g + 8 * h;
    float x[NC][16];
    if (r < G) {
      const bf16* row = static_cast<const bf16*>(a.q) + static_cast<size_t>(s.tok) * a.q_stride + (s.kvh * G + r) * kD + t * 16;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        load16(row + c * 64, x[c]);
        load16(row + c * 64 + 8, x[c] + 8);
      }
    } else {
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[c][e] = 0.f;
    }
    if (a.cos != nullptr) {
      int pos = s.ctx - 1;
      if (pos >= a.max_pos) {
        if (lane == 0) atomicOr(a.status, 2);
        pos = 0;
      }
      // entry i turns with i + D/2: at head size 64 that is lane t ^ 2's, at 128 the lane's own other piece
      const int d0 = (kD == 64 ? t & 1 : t) * 16;
#pragma unroll
      for (int e0 = 0; e0 < 16; e0 += 4) {
        float cs[4], sn[4];
        load16(a.cos + static_cast<size_t>(pos) * (kD / 2) + d0 + e0, cs);
        load16(a.sin + static_cast<size_t>(pos) * (kD / 2) + d0 + e0, sn);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int e = e0 + i;
          if constexpr (kD == 64) {
            const float other = __shfl_xor_sync(0xffffffffu, x[0][e], 2);
            x[0][e] = t < 2 ? x[0][e] * cs[i] - other * sn[i] : x[0][e] * cs[i] + other * sn[i];
          } else {
            const float lo = x[0][e], hi = x[NC - 1][e];
            x[0][e] = lo * cs[i] - hi * sn[i];
            x[NC - 1][e] = hi * cs[i] + lo * sn[i];
          }
        }
      }
    }
    float most = 0.f;
    bool odd = false;                                    // (a row that is not finite is not a number, not a large one)
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        most = fmaxf(most, fabsf(x[c][e]));
        odd |= !(fabsf(x[c][e]) < INFINITY);
      }
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    odd = ((__ballot_sync(0xffffffffu, odd) >> (g * 4)) & 15u) != 0;
    const int ex = static_cast<int>(__float_as_uint(most) >> 23);        // the largest entry is 1.m * 2^(ex - 127)
    const int up = ex == 0 ? 0 : min(134 - ex, 127);                     // ... and is scaled to 1.m * 2^7
    const float mul = kv8_exp2i(max(up, -126));
    factor[h] = odd ? __uint_as_float(0x7fc00000u) : a.scale * kLog2e * kv8_exp2i(-up);
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = odd ? 0.f : x[c][4 * k + e] * mul;
        qf[c * 4 + k][h] = pack_halves(y[0], y[1]);
        qf[c * 4 + k][h + (HI ? 2 : 1)] = pack_halves(y[2], y[3]);
      }
  }
}

// The run of sub-blocks [sb0, sb0 + n) of the segment through the warp's ring (`ring`, its stages' scales at `head`).
// `waited`: the kernels before this one are done; if they are not, the first copies are those of pages that the one before
// does not write.
template <bool HI>
__device__ __forceinline__ void tc_run(const Kv8Args& a, const Kv8Segment& s, int sb0, int n, uint32_t ring, uint32_t head, int lane,
                                       bool& waited, TcState& st) {
  constexpr int KS = kD / 16, NJ = kD / 8, NR = HI ? 2 : 1;
  constexpr int CPR = kD / 16;                           // 16-byte pieces of a key
  const int g = lane >> 2, t = lane & 3;
  const int shift = a.page_shift, ps = 1 << shift;
  const int32_t* bt = a.block_table + static_cast<size_t>(s.seq) * a.max_blocks;
#pragma unroll
  for (int j = 0; j < NJ; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) st.o[j][e] = 0.f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    st.m[h] = st.d[h] = -INFINITY;
    st.l[h] = 0.f;
  }
  // (a sub-block may reach over either end of the live keys, into pages that need not be there any more: their places are
  // filled from the nearest live page)
  const int page_first = s.key_lo >> shift, page_last = (s.key_hi - 1) >> shift;
  const int page0 = n > 0 ? max((sb0 * kSub) >> shift, page_first) : 0;
  // a window of 32 pages, a page to a lane: its id and its scales; and the next window's
  int window = 0, my_page = 0, next_page = 0;
  float my_kf = 0.f, my_ve = 0.f, next_kf = 0.f, next_ve = 0.f;
  auto fetch = [&](int w, int& page, float& kf, float& ve) {
    page = bt[min(page0 + w * 32 + lane, page_last)];
    const size_t at = static_cast<size_t>(page) * a.hkv + s.kvh;
    const int kc = __ldcg(a.kscale + at), vc = __ldcg(a.vscale + at);
    kf = kv8_scale(kc);
    ve = vc == 255 ? __uint_as_float(0x7fc00000u) : static_cast<float>(vc - 127);
  };
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
    for (int b = 0; b < 2; ++b) {
      const int key = sb * kSub + b * 16;
      const int idx = min(max(key >> shift, page_first), page_last) - page0;
      if ((idx >> 5) != window) {
        window = idx >> 5;
        my_page = next_page;
        my_kf = next_kf;
        my_ve = next_ve;
        fetch(window + 1, next_page, next_kf, next_ve);
      }
      const int page = __shfl_sync(0xffffffffu, my_page, idx & 31);
      const size_t at = page * page_bytes + (key & (ps - 1)) * kD;
      const uint8_t *kp = kbase + at, *vp = vbase + at;
#pragma unroll
      for (int i = 0; i < CPR / 2; ++i) {
        copy16(kdst + b * (16 * kD) + i * 512, kp + i * 512);
        // (a round is 4 rows of 128 bytes or 8 of 64: only the first changes the swizzle, by bit 2 of the row)
        copy16((kD == 64 ? vdst : vdst ^ ((i & 1) << 6)) + b * (16 * kD) + i * 512, vp + i * 512);
      }
      if (lane == (idx & 31))
        asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(head + stage * 16 + b * 8), "f"(my_kf), "f"(my_ve) : "memory");
    }
  };
  int loaded = 0;
  if (n > 0) {
    fetch(0, my_page, my_kf, my_ve);
    if (page0 + 32 <= page_last) fetch(1, next_page, next_kf, next_ve);
  }
  if (!waited) {
    const int newest = (s.ctx - 1) >> shift;             // the page that the kernel before this one may be writing to
#pragma unroll 1
    for (; loaded < min(n, kRing - 1) && (((sb0 + loaded) * kSub + kSub - 1) >> shift) < newest; ++loaded) {
      issue(sb0 + loaded, loaded);
      copies_commit();
    }
    pdl_wait();
    waited = true;
    if (n > 0 && page0 + window * 32 + 63 >= newest) {   // its scales are there now
      fetch(window, my_page, my_kf, my_ve);
      if (page0 + 32 <= page_last) fetch(window + 1, next_page, next_kf, next_ve);
    }
  }
  if (n <= 0) return;
#pragma unroll 1
  for (; loaded < kRing - 1; ++loaded) {
    if (loaded < n) issue(sb0 + loaded, loaded);
    copies_commit();                                     // (a group to a sub-block, empty behind the last)
  }
  uint32_t qf[KS][HI ? 4 : 2];
  float factor[NR];
  tc_load_q<HI>(a, s, lane, qf, factor);

  // lane addresses: key 4 (g / 2) + g % 2 of K (so that a lane's scores are those of keys 4 t .. 4 t + 3), key lane of V
  const uint32_t kr = 4 * (g >> 1) + (g & 1);
  const uint32_t krow = kr * kD + (kD == 64 ? t : t ^ ((kr & 1) << 2)) * 16;
  const uint32_t vrow = lane * kD, vsw = kD == 64 ? (lane >> 1) & 3 : lane & 7;
  int stage = 0, ahead = kRing - 1;
#pragma unroll 1
  for (int i = 0; i < n; ++i) {
    const int k0 = (sb0 + i) * kSub;
    copies_wait<kRing - 2>();
    __syncwarp();                                        // (every lane's copies; and every lane is through with the sub-block before)
    if (i + kRing - 1 < n) issue(sb0 + i + kRing - 1, ahead);
    copies_commit();
    const uint32_t kst = ring + stage * (2 * kSubBytes) + krow, vst = ring + stage * (2 * kSubBytes) + kSubBytes + vrow;
    const uint4 hd = lds16(head + stage * 16);
    const float kf[2] = {__uint_as_float(hd.x), __uint_as_float(hd.z)}, ve[2] = {__uint_as_float(hd.y), __uint_as_float(hd.w)};
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
    ahead = stage;
    stage = stage + 1 == kRing ? 0 : stage + 1;
    // ---- S: rows g (and g + 8), keys 16 (nt / 2) + 4 t + 2 (nt % 2) + e
    float sv[4][4];
#pragma unroll
    for (int nt = 0; nt < 4; ++nt) {
#pragma unroll
      for (int c = 0; c < KS / 4; ++c) {
        const uint4 kw = lds16((c ? kst ^ 64u : kst) + ((nt >> 1) * 16 + (nt & 1) * 2) * kD);
        const uint32_t w[4] = {kw.x, kw.y, kw.z, kw.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t* q = qf[c * 4 + k];
          uint32_t b0, b1;
          halves4(w[k], b0, b1);
          if (c == 0 && k == 0) mma_f16_first(sv[nt], q[0], HI ? q[1] : 0u, q[HI ? 2 : 1], HI ? q[HI ? 3 : 0] : 0u, b0, b1);
          else mma_f16(sv[nt], q[0], HI ? q[1] : 0u, q[HI ? 2 : 1], HI ? q[HI ? 3 : 0] : 0u, b0, b1);
        }
      }
    }
    // ---- V as B fragments: entries 16 c + g and 16 c + 8 + g, keys 4 t .. + 3 and 16 further
    uint32_t v[kD / 16][4];
#pragma unroll
    for (int c = 0; c < kD / 16; ++c) ldmatrix_trans(v[c], vst + ((c ^ vsw) << 4));
    if (!whole) {
#pragma unroll
      for (int nt = 0; nt < 4; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int key = k0 + (nt >> 1) * 16 + t * 4 + (nt & 1) * 2 + e;
          if (key < s.key_lo || key >= s.key_hi) {
            sv[nt][e] = -INFINITY;
            if (HI) sv[nt][2 + e] = -INFINITY;
          }
        }
    }
    float alpha[NR];
    uint32_t pf[2][4] = {};                              // the weights as A fragments of 16 keys each
#pragma unroll
    for (int h = 0; h < NR; ++h) {
      float mx[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        float f = factor[h] * kf[b];
        f = f < 1.2e-38f ? 1.2e-38f : f;                 // (times -inf it has to be -inf; so small a factor makes every score 0)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 2; ++e) sv[2 * b + u][2 * h + e] *= f;
        mx[b] = fmaxf(fmaxf(sv[2 * b][2 * h], sv[2 * b][2 * h + 1]), fmaxf(sv[2 * b + 1][2 * h], sv[2 * b + 1][2 * h + 1]));
        mx[b] = fmaxf(mx[b], __shfl_xor_sync(0xffffffffu, mx[b], 1));
        mx[b] = fmaxf(mx[b], __shfl_xor_sync(0xffffffffu, mx[b], 2));
      }
      const float m = fmaxf(st.m[h], fmaxf(mx[0], mx[1]));
      const float dm = st.m[h] - m;                      // -inf the first time
      const float d = fmaxf(st.d[h] + dm, fmaxf(mx[0] - m + ve[0], mx[1] - m + ve[1]));
      alpha[h] = exp2_fast(st.d[h] + dm - d);
      float sum = 0.f;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        // (a block whose best score is 2^-112 of the row's best and whose scale is as many times larger would need more)
        const float w = exp2_fast(fminf(ve[b] - d + 14.f, 126.f));
        float p[4];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float x = exp2_fast(sv[2 * b + u][2 * h + e] - m);
            sum += x;
            p[2 * u + e] = x * w;
          }
        pf[b][h] = pack_halves(p[0], p[1]);
        pf[b][2 + h] = pack_halves(p[2], p[3]);
      }
      st.l[h] = st.l[h] * exp2_fast(dm) + sum;
      st.m[h] = m;
      st.d[h] = d;
    }
    if (__any_sync(0xffffffffu, alpha[0] != 1.f || (HI && alpha[NR - 1] != 1.f))) {
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < (HI ? 4 : 2); ++e) st.o[j][e] *= alpha[HI ? e >> 1 : 0];
    }
    // ---- O += P V
#pragma unroll
    for (int c = 0; c < kD / 16; ++c)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float* o = st.o[2 * c + u];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          uint32_t b0, b1;
          halves4(v[c][2 * b + u], b0, b1);
          mma_f16(o, pf[b][0], pf[b][1], pf[b][2], pf[b][3], b0, b1);
        }
      }
  }
  copies_wait<0>();
#pragma unroll
  for (int h = 0; h < NR; ++h) {                         // the row's four lanes
    st.l[h] += __shfl_xor_sync(0xffffffffu, st.l[h], 1);
    st.l[h] += __shfl_xor_sync(0xffffffffu, st.l[h], 2);
  }
#pragma unroll
  for (int j = 0; j < NJ; ++j)
#pragma unroll
    for (int e = 0; e < (HI ? 4 : 2); ++e) st.o[j][e] *= 6.103515625e-5f;        // 2^-14
  __syncwarp();
}

// Adds up the partial results of warps [w0, w0 + nw) for head r, entry d (they are in the warps' rings).
__device__ __forceinline__ Kv8Piece tc_fold(const unsigned char* smem, int w0, int nw, int r, int d) {
  Kv8Piece sum;
  for (int w = w0; w < w0 + nw; ++w)
    sum.m = fmaxf(sum.m, (reinterpret_cast<const float*>(smem + w * kRingBytes) + r * kPartLd)[kD + 1]);
  for (int w = w0; w < w0 + nw; ++w) {
    const float* p = reinterpret_cast<const float*>(smem + w * kRingBytes) + r * kPartLd;
    sum.d = fmaxf(sum.d, p[kD] + (p[kD + 1] - sum.m));
  }
  for (int w = w0; w < w0 + nw; ++w) {
    const float* p = reinterpret_cast<const float*>(smem + w * kRingBytes) + r * kPartLd;
    if (p[kD + 1] == -INFINITY && p[kD + 2] == 0.f) continue;        // (a warp without keys)
    const float dm = p[kD + 1] - sum.m;
    sum.num += exp2f(p[kD] + dm - sum.d) * p[d];
    sum.den += exp2f(dm) * p[kD + 2];
  }
  return sum;
}

// groups: of the CTA's warps, a divisor of their number.  shares: the keys in equal shares (else: rows).
template <bool HI>
__global__ void __launch_bounds__(kTcThreads, 1)
kv8_decode_tc_kernel(const Kv8Args a, int groups, int by_shares) {
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int start[kMaxItems + 1];
  __shared__ int last[kTcWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int G = a.hq / a.hkv;
  const int csize = static_cast<int>(cluster_size()), rank = static_cast<int>(cluster_rank());
  const int gsize = kTcWarps / groups, gi = warp / gsize, wg = warp - gi * gsize;
  const int gthreads = gsize * 32, gtid = wg * 32 + lane;
  const int nclusters = gridDim.x / csize;
  float* slots = reinterpret_cast<float*>(smem + kTcWarps * (kRingBytes + kHeadBytes));      // [csize][G][kD + 3], of the first CTA of a cluster
  // With the rotation in this kernel the one before it is the write of the tokens' keys (launch_decode_tc), and what came
  // before that is done: only the newest pages have to wait.  Without, anything may be under way.
  if (csize > 1) cluster_arrive();                       // (met before the first store into another CTA: it has begun by then)
  bool waited = false;
  if (a.cos == nullptr) {
    pdl_wait();
    waited = true;
  }
  int units = 0, shares = 0, u = 0, end = 0;
  if (by_shares) {
    units = kv8_units(a, start);
    shares = min(nclusters * groups, units);
    const int mine = gi * nclusters + blockIdx.x;        // (neighbouring shares lie on different SMs)
    if (mine < shares) {
      u = kv8_share_begin(mine, units, shares);
      end = kv8_share_begin(mine + 1, units, shares);
    }
  }
  const int share = gi * nclusters + blockIdx.x, share_first = u;
  const int nrows = a.nitems * a.hkv;
  int rowi = gi * nclusters + blockIdx.x / csize;
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
      s.whole = true;
      rowi += groups * nclusters;
      if (s.ctx <= 0) {                                  // (the same for the whole cluster)
        if (csize > 1) cluster_wait();
        continue;
      }
    }
    // ---- this warp's run of sub-blocks
    const int W = csize * gsize, wi = rank * gsize + wg;
    const int first = s.key_lo / kSub, all = (s.key_hi - 1) / kSub - first + 1;
    const int per = all / W, rem = all - per * W;
    TcState st;
    tc_run<HI>(a, s, first + wi * per + min(wi, rem), per + (wi < rem ? 1 : 0), smem_addr(smem) + warp * kRingBytes,
                      smem_addr(smem) + kTcWarps * kRingBytes + warp * kHeadBytes, lane, waited, st);
    // ---- its partial result into its ring
    float* mine = reinterpret_cast<float*>(smem + warp * kRingBytes);
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int h = 0; h < (HI ? 2 : 1); ++h) {
      const int r = g + 8 * h;
      if (r < G) {
#pragma unroll
        for (int j = 0; j < kD / 8; ++j)
          *reinterpret_cast<float2*>(mine + r * kPartLd + 8 * j + 2 * t) = make_float2(st.o[j][2 * h], st.o[j][2 * h + 1]);
        if (t == 0) {
          mine[r * kPartLd + kD] = st.d[h];
          mine[r * kPartLd + kD + 1] = st.m[h];
          mine[r * kPartLd + kD + 2] = st.l[h];
        }
      }
    }
    if (csize > 1) {
      // ---- the CTA's sums into a slot of the cluster's first CTA, which adds the slots in order
      __syncthreads();
      cluster_wait();
      for (int i = threadIdx.x; i < G * kD; i += kTcThreads) {
        const int r = i / kD, d = i - r * kD;
        const Kv8Piece x = tc_fold(smem, 0, kTcWarps, r, d);
        float* slot = slots + (rank * G + r) * (kD + 3);
        store_cluster(slot + d, 0, x.num);
        if (d == 0) {
          store_cluster(slot + kD, 0, x.d);
          store_cluster(slot + kD + 1, 0, x.m);
          store_cluster(slot + kD + 2, 0, x.den);
        }
      }
      cluster_arrive();
      cluster_wait();
      if (rank == 0)
        for (int i = threadIdx.x; i < G * kD; i += kTcThreads) {
          const int r = i / kD, d = i - r * kD;
          Kv8Piece x;
          for (int c = 0; c < csize; ++c) {
            const float* p = slots + (c * G + r) * (kD + 3);
            x.add(p[kD], p[kD + 1], p[kD + 2], p[d]);
          }
          static_cast<bf16*>(a.out)[static_cast<size_t>(s.tok) * a.out_stride + (s.kvh * G + r) * kD + d] = __float2bfloat16_rn(x.value());
        }
      continue;                                          // (one row to a cluster: see the launch)
    }
    asm volatile("bar.sync %0, %1;" ::"r"(1 + gi), "r"(gthreads) : "memory");
    float* piece = by_shares && !s.whole ? a.part + (static_cast<size_t>(share) * 2 + (u == share_first ? 0 : 1)) * (G * (kD + 3)) : nullptr;
    for (int i = gtid; i < G * kD; i += gthreads) {
      const int r = i / kD, d = i - r * kD;
      const Kv8Piece x = tc_fold(smem, gi * gsize, gsize, r, d);
      if (piece == nullptr)
        static_cast<bf16*>(a.out)[static_cast<size_t>(s.tok) * a.out_stride + (s.kvh * G + r) * kD + d] = __float2bfloat16_rn(x.value());
      else
        kv8_leave(piece + r * (kD + 3), kD, d, x);
    }
    if (piece != nullptr) {
      __threadfence();                                   // the piece, before it is counted
      asm volatile("bar.sync %0, %1;" ::"r"(1 + gi), "r"(gthreads) : "memory");
      if (gtid == 0) {
        const int pieces = kv8_share_of(s.row_end - 1, units, shares) - kv8_share_of(s.row_begin, units, shares) + 1;
        int* c = a.counters + static_cast<size_t>(s.item) * a.hkv + s.kvh;
        const int done = atomicAdd(c, 1) == pieces - 1;
        if (done) *c = 0;
        last[gi] = done;
      }
      asm volatile("bar.sync %0, %1;" ::"r"(1 + gi), "r"(gthreads) : "memory");
      if (last[gi]) {
        __threadfence();
        kv8_merge<bf16>(a, s, units, shares, gtid, gthreads);
      }
    }
    asm volatile("bar.sync %0, %1;" ::"r"(1 + gi), "r"(gthreads) : "memory");      // before the rings are used again
    if (by_shares) u = s.next;
  }
  if (!waited) pdl_wait();                               // (nothing of this launch ends before what it follows)
}

}  // namespace rl
