// Attention over the paged 8-bit KV cache, sm_100a: few query rows (single tokens, drafted tokens).
//
// For the rows r = (query token i, query head of the K/V head) of one K/V head:
//   x_j = q_r . c_j * (amax_k * softmax scale * log2 e / Q)     c_j: K codes of key j, amax_k of its page
//   m = max x_j;  l = sum 2^(x_j - m);  o = sum 2^(x_j - m) * (amax_v / Q) * d_j / l     d_j: V codes
// over the visible keys (j < kv_len; causal: j <= kv_len - q_len + i), one pass with the running maximum and sum in
// fp32. The 8-bit codes are widened to fp16, which holds every one of them exactly, and multiplied on the tensor
// cores with fp32 sums. A bf16 query row is first scaled by a power of two to a maximum in [1, 2), which fp16 holds
// to 2^-25 of the row's maximum; the weights 2^(x - m) in [0, 1] are rounded to fp16 (2^-12 relative, below the
// rounding of a bf16 or fp16 result). The scale of V is applied to each page's product in fp32, so pages of any two
// magnitudes mix without loss.
//
// Bound by memory: 256 bytes of codes a (key, K/V head) against 512 flops a row; with 16 rows that is 32 flops a
// byte, far under what even mma.sync gives, and its fragments live in registers: no round trip through tensor memory
// for rows that would fill an eighth of a 128-row tile. One CTA: 16 rows x one key split, 4 warps, each taking whole
// pages (64 keys) in turn from a ring of 6 page slots (K and V 8 KB each, TMA, 128-byte swizzle); a warp refills the
// slot it has consumed, so there is no producer warp and no empty barrier, and warps meet only to merge at the end.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "lbq_kernels.h"
#include "lbq_paged.h"
#include "lbq_paged.cuh"
#include "lbq_ptx.cuh"

namespace lbq {

constexpr int kDecWarps = 4;
constexpr int kDecSlots = 6;
constexpr int kDecRows = 16;
constexpr int kMergePitch = 132;                       // floats of a merged row in shared memory
constexpr size_t kDecSmem = 1024 + size_t(kDecSlots) * 2 * kPageBytes;
static_assert(size_t(kDecWarps) * kDecRows * kMergePitch * 4 <= size_t(kDecSlots) * 2 * kPageBytes, "merge area");

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Channels 4 * (lane % 4) .. + 3 of every 16 of one query row as the A fragments of 8 MMA steps (the channel order
// inside a step is the one in which ldmatrix hands out four consecutive bytes of K; a dot product does not mind),
// scaled by a power of two to a largest magnitude in [1, 2); returns the factor that undoes it.
template <int kDt>
__device__ __forceinline__ float load_query(const uint16_t* row, int quad, uint2 (&frag)[8]) {
  uint2 raw[8];
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    raw[k] = row ? *reinterpret_cast<const uint2*>(row + 16 * k + 4 * quad) : make_uint2(0u, 0u);
    if constexpr (kDt == 0) {
      const uint32_t w[4] = {raw[k].x << 16, raw[k].x & 0xffff0000u, raw[k].y << 16, raw[k].y & 0xffff0000u};
#pragma unroll
      for (int i = 0; i < 4; ++i) top = max(top, w[i] & 0x7fffffffu);
    }
  }
  if constexpr (kDt == 1) {
#pragma unroll
    for (int k = 0; k < 8; ++k) frag[k] = raw[k];
    return 1.f;
  } else {
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // exponent field e of the maximum: scale by 2^(127 - e); zero, subnormal and non-finite rows go unscaled
    uint32_t e = top >> 23;
    const bool plain = e == 0 || e == 255;
    if (e == 254) e = 253;                               // 2^(127 - 254) is no normal float: a maximum in [2, 4)
    const float down = plain ? 1.f : __uint_as_float((254u - e) << 23);
    const float up = plain ? 1.f : __uint_as_float(e << 23);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const __half2 lo = __floats2half2_rn(__uint_as_float(raw[k].x << 16) * down, __uint_as_float(raw[k].x & 0xffff0000u) * down);
      const __half2 hi = __floats2half2_rn(__uint_as_float(raw[k].y << 16) * down, __uint_as_float(raw[k].y & 0xffff0000u) * down);
      frag[k] = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
    return up;
  }
}

// out row (query token i, head) of 16 channels from channel 16 * seg.
template <int kDt>
__device__ __forceinline__ void store_out16(const PagedAttnArgs& a, int b, int i, int head, int seg, const float (&o)[16]) {
  uint16_t* p = static_cast<uint16_t*>(a.out) + b * a.so[0] + i * a.so[1] + head * a.so[2] + seg * 16;
  uint32_t w[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) w[k] = pack_act2(o[2 * k], o[2 * k + 1], kDt);
  reinterpret_cast<uint4*>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
  reinterpret_cast<uint4*>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
}
struct DecShared {
  uint64_t full[kDecSlots];
  int issued[kDecSlots];
  int abort;
  float m[kDecWarps][kDecRows];
  float l[kDecWarps][kDecRows];
};

template <int kFmt, int kDt>
__global__ void __launch_bounds__(kDecWarps * 32, 2)
    paged_decode_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                        const PagedAttnArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ DecShared sh;
  volatile int* abort_flag = &sh.abort;
  const int tile = blockIdx.x % a.tiles, h = blockIdx.x / a.tiles, split = blockIdx.y, b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane & 3, r0 = lane >> 2;
  const TileKeys tk = tile_keys(a, b, tile);
  const int pages = int((tk.visible + kPageTokens - 1) / kPageTokens);
  const int p0 = split * a.split_pages;
  const int n = max(0, min(pages - p0, a.split_pages));
  if (split > 0 && n == 0) return;
  const bool single = pages <= a.split_pages;
  const int32_t* table = a.pt.table + b * a.pt.st_b + p0;

  // Page ids outside the pool are recorded and read as page 0 with every key masked.
  auto page_id = [&](int i, bool& ok) {
    const int id = table[i];
    ok = id >= 0 && id < a.pt.num_pages;
    if (!ok && a.status) atomicCAS(a.status, 0, kDevBadPage);
    return ok ? id : 0;
  };
  auto issue = [&](int i, int id) {
    const int s = i % kDecSlots;
    mbar_arrive_expect_tx(&sh.full[s], 2 * kPageBytes);
    const int row = (id * a.heads + h) * kPageTokens;
    tma_load_3d(ring + s * 2 * kPageBytes, &tm_k, &sh.full[s], 0, row, 0);
    tma_load_3d(ring + s * 2 * kPageBytes + kPageBytes, &tm_v, &sh.full[s], 0, row, 0);
    sh.issued[s] = i / kDecSlots + 1;
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < kDecSlots; ++s) {
      mbar_init(&sh.full[s], 1);
      sh.issued[s] = 0;
    }
    sh.abort = 0;
    fence_mbar_init();
  }
  __syncthreads();
  if (warp == 0 && lane < min(n, kDecSlots)) {
    bool ok;
    const int id = page_id(lane, ok);
    issue(lane, id);
  }

  uint32_t qa[8][4];
  float unit[2];                                         // per row: undo the power of two, softmax scale, 1 / Q
  int64_t limit[2];                                      // last visible key
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = tile * kDecRows + r0 + 8 * e, i = r / a.group, g = r - i * a.group;
    const bool on = i < tk.qn;
    const uint16_t* row = on ? static_cast<const uint16_t*>(a.q) + b * a.sq[0] + i * a.sq[1] + (h * a.group + g) * a.sq[2]
                             : nullptr;
    uint2 frag[8];
    unit[e] = load_query<kDt>(row, quad, frag) * a.score_log2;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      qa[k][e] = frag[k].x;
      qa[k][2 + e] = frag[k].y;
    }
    limit[e] = !on ? -1 : (a.causal ? tk.kv - tk.qn + i : tk.kv - 1);
  }
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float o[16][4];
#pragma unroll
  for (int c = 0; c < 16; ++c)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[c][e] = 0.f;

  // The scales of this warp's next page are loaded one page ahead, its page id two pages ahead.
  const int64_t hs = a.heads;
  bool ok_cur = false, ok_next = false;
  int id_next = 0;
  float ka = 0.f, va = 0.f;
  if (warp < n) {
    const int id = page_id(warp, ok_cur);
    ka = a.ka[id * hs + h];
    va = a.va[id * hs + h];
  }
  if (warp + kDecWarps < n) id_next = page_id(warp + kDecWarps, ok_next);
  for (int i = warp; i < n; i += kDecWarps) {
    const int s = i % kDecSlots;
    float ka_next = 0.f, va_next = 0.f;
    bool ok_after = false, ok_fill = false;
    int id_after = 0, id_fill = 0;
    if (i + kDecWarps < n) {
      ka_next = a.ka[id_next * hs + h];
      va_next = a.va[id_next * hs + h];
    }
    if (i + 2 * kDecWarps < n) id_after = page_id(i + 2 * kDecWarps, ok_after);
    if (i + kDecSlots < n) id_fill = page_id(i + kDecSlots, ok_fill);
    if (!mbar_wait(&sh.full[s], (i / kDecSlots) & 1, abort_flag, a.status, kDevTimeoutKV)) break;
    const uint32_t kb = smem_u32(ring + s * 2 * kPageBytes), vb = kb + kPageBytes;

    // scores of the 64 keys: tile nt holds keys 8 nt .. 8 nt + 7
    float x[8][4];
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[nt][e] = 0.f;
#pragma unroll
      for (int kq = 0; kq < 2; ++kq) {
        const int key = nt * 8 + (lane & 7), c = kq * 4 + (lane >> 3);
        uint32_t r[4];
        ldsm4(kb + key * 128 + ((c ^ (key & 7)) << 4), r);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t w = bias<kFmt>(r[k]);
          mma_f16(x[nt], qa[kq * 4 + k], widen<kFmt, 0, 1>(w), widen<kFmt, 2, 3>(w));
        }
      }
    }
    const float c0 = ka * unit[0], c1 = ka * unit[1];
    const int64_t j0 = int64_t(p0 + i) * kPageTokens + 2 * quad;
    const bool whole = ok_cur && min(limit[0], limit[1]) >= j0 + 63;
    float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        x[nt][e] *= c0;
        x[nt][2 + e] *= c1;
        if (!whole) {
          const int64_t j = j0 + nt * 8 + e;
          if (!ok_cur || j > limit[0]) x[nt][e] = -INFINITY;
          if (!ok_cur || j > limit[1]) x[nt][2 + e] = -INFINITY;
        }
        t0 = fmaxf(t0, x[nt][e]);
        t1 = fmaxf(t1, x[nt][2 + e]);
      }
    }
    t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 1));
    t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 1));
    t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 2));
    t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 2));
    t0 = fmaxf(t0, m[0]);
    t1 = fmaxf(t1, m[1]);
    // a row that has seen no key yet keeps m = -inf; its exponents are taken against 0 and give 0
    const float n0 = t0 == -INFINITY ? 0.f : t0, n1 = t1 == -INFINITY ? 0.f : t1;
    const float al0 = ex2_approx(m[0] - n0), al1 = ex2_approx(m[1] - n1);
    m[0] = t0;
    m[1] = t1;
    float s0 = 0.f, s1 = 0.f;
    uint32_t pa[4][4];
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) {
      const float w0 = ex2_approx(x[nt][0] - n0), w1 = ex2_approx(x[nt][1] - n0);
      const float w2 = ex2_approx(x[nt][2] - n1), w3 = ex2_approx(x[nt][3] - n1);
      s0 += w0 + w1;
      s1 += w2 + w3;
      pa[nt >> 1][(nt & 1) * 2] = pack_act2(w0, w1, 1);
      pa[nt >> 1][(nt & 1) * 2 + 1] = pack_act2(w2, w3, 1);
    }
    l[0] = l[0] * al0 + s0;
    l[1] = l[1] * al1 + s1;
    // o = o * alpha + (P . D) * v: channels 16 c + 2 n (even) and 16 c + 2 n + 1 (odd) are two MMA column tiles
    const float v = va * a.v_unit;
    // rows of V past the sequence's tokens hold whatever the page held before: weight 0 times a NaN code (e4m3; int8 has
    // none) would be NaN, so they are read as 0
    const int64_t rest = ok_cur ? tk.kv - int64_t(p0 + i) * kPageTokens : 0;
    const bool clip = kFmt == 1 && rest < kPageTokens;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      float ev[4] = {0.f, 0.f, 0.f, 0.f}, od[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int key = half * 32 + lane;
        uint32_t r[4];
        ldsm4_t(vb + key * 128 + ((c ^ (key & 7)) << 4), r);
        if (clip) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int j = half * 32 + k * 8 + 2 * quad;
            r[k] &= (j < rest ? 0x0000ffffu : 0u) | (j + 1 < rest ? 0xffff0000u : 0u);
          }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t w0 = bias<kFmt>(r[2 * k]), w1 = bias<kFmt>(r[2 * k + 1]);
          mma_f16(ev, pa[half * 2 + k], widen<kFmt, 0, 2>(w0), widen<kFmt, 0, 2>(w1));
          mma_f16(od, pa[half * 2 + k], widen<kFmt, 1, 3>(w0), widen<kFmt, 1, 3>(w1));
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float al = e < 2 ? al0 : al1;
        o[2 * c][e] = fmaf(ev[e], v, o[2 * c][e] * al);
        o[2 * c + 1][e] = fmaf(od[e], v, o[2 * c + 1][e] * al);
      }
    }
    __syncwarp();                                          // every lane has read the slot
    if (lane == 0 && i + kDecSlots < n) issue(i + kDecSlots, id_fill);
    ok_cur = ok_next;
    ok_next = ok_after;
    id_next = id_after;
    ka = ka_next;
    va = va_next;
  }
  __syncthreads();
  if (*abort_flag) {                                       // let copies in flight land before the CTA goes away
    if (threadIdx.x == 0)
      for (int s = 0; s < kDecSlots; ++s)
        if (sh.issued[s]) mbar_drain_wait(&sh.full[s], (sh.issued[s] - 1) & 1);
    return;
  }

  // merge the warps: rows of 128 channels in the ring, which nothing reads any more
  float* mo = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
    if (quad == 0) {
      sh.m[warp][r0 + 8 * e] = m[e];
      sh.l[warp][r0 + 8 * e] = l[e];
    }
    float* row = mo + (warp * kDecRows + r0 + 8 * e) * kMergePitch;
#pragma unroll
    for (int c = 0; c < 8; ++c)
      *reinterpret_cast<float4*>(row + 16 * c + 4 * quad) =
          make_float4(o[2 * c][2 * e], o[2 * c + 1][2 * e], o[2 * c][2 * e + 1], o[2 * c + 1][2 * e + 1]);
  }
  __syncthreads();
  const int rr = threadIdx.x >> 3, seg = threadIdx.x & 7;
  const int row = tile * kDecRows + rr, qi = row / a.group, head = h * a.group + row % a.group;
  float mm = -INFINITY;
#pragma unroll
  for (int w = 0; w < kDecWarps; ++w) mm = fmaxf(mm, sh.m[w][rr]);
  const float ref = mm == -INFINITY ? 0.f : mm;
  float ll = 0.f, acc[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) acc[k] = 0.f;
#pragma unroll
  for (int w = 0; w < kDecWarps; ++w) {
    const float f = ex2_approx(sh.m[w][rr] - ref);
    ll += sh.l[w][rr] * f;
    const float4* p = reinterpret_cast<const float4*>(mo + (w * kDecRows + rr) * kMergePitch + 16 * seg);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float4 x = p[k];
      acc[4 * k] += x.x * f;
      acc[4 * k + 1] += x.y * f;
      acc[4 * k + 2] += x.z * f;
      acc[4 * k + 3] += x.w * f;
    }
  }
  if (single) {
    if (qi >= a.q_len) return;
    const float inv = ll == 0.f ? 0.f : 1.f / ll;
#pragma unroll
    for (int k = 0; k < 16; ++k) acc[k] = ll == 0.f ? 0.f : acc[k] * inv;
    store_out16<kDt>(a, b, qi, head, seg, acc);
    if (a.lse && seg == 0) a.lse[(int64_t(b) * a.q_len + qi) * (a.heads * a.group) + head] = natural_lse(mm, ll);
  } else {
    const int64_t at = (int64_t(split) * a.batch * a.heads + int64_t(b) * a.heads + h) * (int64_t(a.tiles) * a.tile_rows) + row;
    float4* p = reinterpret_cast<float4*>(a.o_part + at * 128 + 16 * seg);
#pragma unroll
    for (int k = 0; k < 4; ++k) p[k] = make_float4(acc[4 * k], acc[4 * k + 1], acc[4 * k + 2], acc[4 * k + 3]);
    if (seg == 0) a.ml_part[at] = make_float2(mm, ll);
  }
}

// Merge of the key splits: one warp a row, 4 channels a lane. Rows whose tile fits one split were finished by the
// attention kernel.
template <int kDt>
__global__ void __launch_bounds__(128) paged_combine_kernel(const PagedAttnArgs a) {
  const int64_t rows = int64_t(a.q_len) * a.group;
  const int64_t item = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (item >= rows * a.heads * a.batch) return;
  const int64_t bh = item / rows;
  const int row = int(item - bh * rows), b = int(bh / a.heads), h = int(bh - int64_t(b) * a.heads);
  const TileKeys tk = tile_keys(a, b, row / a.tile_rows);
  const int pages = int((tk.visible + kPageTokens - 1) / kPageTokens);
  if (pages <= a.split_pages) return;
  const int n = (pages + a.split_pages - 1) / a.split_pages;
  const int64_t step = int64_t(a.batch) * a.heads * a.tiles * a.tile_rows;
  const int64_t at = bh * (int64_t(a.tiles) * a.tile_rows) + row;
  float m = -INFINITY;
  for (int s = lane; s < n; s += 32) m = fmaxf(m, a.ml_part[s * step + at].x);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  const float ref = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = 0; s < n; ++s) {
    const float2 ml = a.ml_part[s * step + at];
    const float4 x = *reinterpret_cast<const float4*>(a.o_part + (s * step + at) * 128 + 4 * lane);
    const float f = ex2_approx(ml.x - ref);
    l += ml.y * f;
    o.x += x.x * f;
    o.y += x.y * f;
    o.z += x.z * f;
    o.w += x.w * f;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int i = row / a.group, head = h * a.group + row % a.group;
  uint16_t* p = static_cast<uint16_t*>(a.out) + b * a.so[0] + i * a.so[1] + head * a.so[2] + 4 * lane;
  uint2 w = make_uint2(0u, 0u);
  if (l != 0.f) w = make_uint2(pack_act2(o.x * inv, o.y * inv, kDt), pack_act2(o.z * inv, o.w * inv, kDt));
  *reinterpret_cast<uint2*>(p) = w;
  if (a.lse && lane == 0) a.lse[(int64_t(b) * a.q_len + i) * (a.heads * a.group) + head] = natural_lse(m, l);
}

template <int kFmt, int kDt>
cudaError_t launch_decode_as(const PagedAttnArgs& a, const CUtensorMap& tm_k, const CUtensorMap& tm_v, cudaStream_t st) {
  if (cudaError_t e = allow_dynamic_smem<paged_decode_kernel<kFmt, kDt>>(int(kDecSmem)); e != cudaSuccess) return e;
  const dim3 grid(unsigned(a.heads) * a.tiles, a.splits, a.batch);
  paged_decode_kernel<kFmt, kDt><<<grid, kDecWarps * 32, kDecSmem, st>>>(tm_k, tm_v, a);
  return cudaGetLastError();
}
cudaError_t launch_paged_decode(const PagedAttnArgs& a, const CUtensorMap& tm_k, const CUtensorMap& tm_v,
                                cudaStream_t st) {
  if (a.fmt) return a.dtype ? launch_decode_as<1, 1>(a, tm_k, tm_v, st) : launch_decode_as<1, 0>(a, tm_k, tm_v, st);
  return a.dtype ? launch_decode_as<0, 1>(a, tm_k, tm_v, st) : launch_decode_as<0, 0>(a, tm_k, tm_v, st);
}
cudaError_t launch_paged_combine(const PagedAttnArgs& a, cudaStream_t st) {
  const int64_t items = int64_t(a.q_len) * a.group * a.heads * a.batch;
  if (a.dtype) paged_combine_kernel<1><<<unsigned((items + 3) / 4), 128, 0, st>>>(a);
  else paged_combine_kernel<0><<<unsigned((items + 3) / 4), 128, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace lbq
