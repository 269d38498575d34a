// Attention over the paged 8-bit KV cache, sm_100a: few query rows (single tokens, drafted tokens), and the merge of key
// splits for both attention kernels.
//
// For the rows r = (query token i, query head of the K/V head) of one K/V head, over the visible keys j (j < kv_len;
// causal: j <= kv_len - q_len + i):
//   x_j = q_r . c_j * (amax_k * softmax scale * log2 e / Q)          c_j: K codes of key j, amax_k of its page
//   m = running maximum of x_j + log2 amax_v;  w_j = 2^(x_j + log2 amax_v - m + 7)
//   o = sum w_j d_j (d_j: V codes);  l = sum w_j / amax_v;  out = o / (Q l)
// The codes are widened to fp16, which holds every one exactly, and multiplied on the tensor cores with fp32 sums. A bf16
// query row is first scaled by a power of two to a maximum in [1, 2), which fp16 holds to 2^-25 of the row's maximum.
// The scale of V rides in the exponent, so the weights that matter are those nearest 2^7 whatever the pages' magnitudes;
// m moves only when exceeded by more than 2^8, so weights stay below 2^15 and o, l are rescaled rarely. Weights are
// rounded to fp16 for the product (off by 2^-11 relative at most, and by 2^-32 of the row's largest where that is more); l sums
// them before the rounding. A second product for what the rounding leaves would double this one's work; an output in bf16 (off
// by 2^-8) hides the rounding, one in fp16 shows it slightly. Where V scales lie further apart than fp32's exponents, see
// kFaint (lbq_paged.cuh).
//
// Bound by memory: 256 bytes of codes a (key, K/V head) against 512 flops a row. The keys are the M side of the products
// (S^T = C Q^T, O^T = D^T W^T, mma.sync m16n8k16) and the queries the N side: 8 rows fill a tile, a widened fragment serves
// every tile of 8, and the fragments stay in registers (tcgen05 would want 128 query rows and a round trip through tensor
// memory). One CTA: 8 * kNT rows x one key split, 4 warps, each taking whole pages (64 keys) in turn from a ring of 6 page
// slots (K and V 8 KB each, TMA, 128-byte swizzle); a warp refills the slot it has consumed, so there is no producer warp
// and no empty barrier, and warps meet only to merge at the end. The slots' next users are other warps, which may be a lap
// ahead: they look at the slot's count of fills first, since a barrier's parity alone would let them pass on the phase
// before the last.
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
constexpr int kMergePitch = 132;                       // floats of a merged row in shared memory
constexpr size_t kDecSmem = 1024 + size_t(kDecSlots) * 2 * kPageBytes;
static_assert(size_t(kDecWarps * kMergePitch + 128) * 16 * 4 <= size_t(kDecSlots) * 2 * kPageBytes, "merge area");

// Volatile, so that they stay between the wait for a slot and its refill; not the products, which may move freely.
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Transposes an 8 x 8 matrix of 16-bit elements held as two of a row per lane.
__device__ __forceinline__ uint32_t movmatrix_t(uint32_t v) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}
// Channels 4 * (lane % 4) .. + 3 of every 16 of one query row as the B fragments of 8 MMA steps (the channel order
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
    float up;
    const float down = row_scale(top, up);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const __half2 lo = __floats2half2_rn(__uint_as_float(raw[k].x << 16) * down, __uint_as_float(raw[k].x & 0xffff0000u) * down);
      const __half2 hi = __floats2half2_rn(__uint_as_float(raw[k].y << 16) * down, __uint_as_float(raw[k].y & 0xffff0000u) * down);
      frag[k] = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
    return up;
  }
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The float(s) at `p` of CTA `rank` of the cluster.
__device__ __forceinline__ float2 peer_f2(const float* p, int rank) {
  float2 v;
  asm volatile(
      "{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %2, %3;\n\tld.shared::cluster.v2.f32 {%0, %1}, [ra];\n\t}"
      : "=f"(v.x), "=f"(v.y)
      : "r"(smem_u32(p)), "r"(rank)
      : "memory");
  return v;
}

__device__ __forceinline__ void st_release(int* p, int v) {
  asm volatile("st.release.cta.shared.s32 [%0], %1;" ::"r"(smem_u32(p)), "r"(v) : "memory");
}
__device__ __forceinline__ int ld_acquire(const int* p) {
  int v;
  asm volatile("ld.acquire.cta.shared.s32 %0, [%1];" : "=r"(v) : "r"(smem_u32(p)) : "memory");
  return v;
}

struct DecShared {
  uint64_t full[kDecSlots];
  int issued[kDecSlots];
  int abort;
  float m[kDecWarps][16];
  float l[kDecWarps][16];
  float2 ml[16];                                         // clustered splits: this CTA's maximum and sum of each row
};

template <int kFmt, int kDt, int kNT>
__global__ void __launch_bounds__(kDecWarps * 32, 2)
    paged_decode_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                        const PagedAttnArgs a) {
  constexpr int kRows = 8 * kNT;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ DecShared sh;
  volatile int* abort_flag = &sh.abort;
  const int tile = blockIdx.x % a.tiles, h = blockIdx.x / a.tiles, split = blockIdx.y, b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane & 3, r0 = lane >> 2;
  if (threadIdx.x == 32) {
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  after_previous_grid();
  const int p0 = split * a.split_pages;
  const int32_t* table = a.pt.table + b * a.pt.st_b + p0;
  // the first page ids, before it is known whether the sequence has them: one load's latency less until data flows
  const int id_early = threadIdx.x < kDecSlots && p0 + int(threadIdx.x) < a.pt.width ? table[threadIdx.x] : 0;
  const TileKeys tk = tile_keys(a, b, tile);
  const int pages = int((tk.visible + kPageTokens - 1) / kPageTokens);
  const int n = max(0, min(pages - p0, a.split_pages));
  const bool single = pages <= a.split_pages;            // of the whole tile, so of every CTA of its cluster
  if (split > 0 && (single || (n == 0 && !a.clustered))) return;
  const uint32_t pool = uint32_t(a.pt.num_pages);

  // Page ids are loaded well before they are looked at. One outside the pool is recorded, and read as page 0 with every
  // key masked.
  auto known = [&](int id) {
    const bool ok = uint32_t(id) < pool;
    if (!ok && a.status) atomicCAS(a.status, 0, kDevBadPage);
    return ok;
  };
  auto issue = [&](int i, int id) {
    const int s = i % kDecSlots;
    mbar_arrive_expect_tx(&sh.full[s], 2 * kPageBytes);
    const int row = ((known(id) ? id : 0) * a.heads + h) * kPageTokens;
    tma_load_3d(ring + s * 2 * kPageBytes, &tm_k, &sh.full[s], 0, row, 0);
    tma_load_3d(ring + s * 2 * kPageBytes + kPageBytes, &tm_v, &sh.full[s], 0, row, 0);
    st_release(&sh.issued[s], i / kDecSlots + 1);
  };
  // The slot's fill number i / kDecSlots has been issued (bounded, like every wait).
  auto filled = [&](int i) {
    const int s = i % kDecSlots, want = i / kDecSlots + 1;
    if (ld_acquire(&sh.issued[s]) >= want) return true;
    const uint64_t t0 = globaltimer_ns();
    for (uint32_t k = 1; k < LBQ_SPIN_LIMIT; ++k) {
      if (ld_acquire(&sh.issued[s]) >= want) return true;
      if (*abort_flag) return false;
      if ((k & 255) == 0 && globaltimer_ns() - t0 > LBQ_WAIT_LIMIT_NS) break;
    }
    *abort_flag = 1;
    if (a.status) atomicCAS(a.status, 0, kDevTimeoutKV);
    return false;
  };
  if (threadIdx.x < kDecSlots) {
    // each slot's barrier is set up by the lane that first fills the slot
    const int s = threadIdx.x;
    mbar_init(&sh.full[s], 1);
    sh.issued[s] = 0;
    if (s == 0) sh.abort = 0;
    fence_mbar_init();
    if (s < n) issue(s, id_early);
  }

  uint2 qb[kNT][8];
  float unit[kNT][2];                                    // per query column
  int limit[kNT][2];                                     // last visible key of the split (a table has under 2^24 pages)
#pragma unroll
  for (int t = 0; t < kNT; ++t) {
    const int r = tile * kRows + 8 * t + r0, i = r / a.group, g = r - i * a.group;
    const uint16_t* row = i < tk.qn ? static_cast<const uint16_t*>(a.q) + b * a.sq[0] + i * a.sq[1] + (h * a.group + g) * a.sq[2]
                                    : nullptr;
    const float u = row_factor(load_query<kDt>(row, quad, qb[t]), a.score_log2);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      unit[t][e] = __shfl_sync(0xffffffffu, u, 8 * quad + 4 * e);      // column 2 quad + e is row r0 of that lane
      const int qi = (tile * kRows + 8 * t + 2 * quad + e) / a.group;
      limit[t][e] = qi >= tk.qn ? -1 : int((a.causal ? tk.kv - tk.qn + qi : tk.kv - 1) - int64_t(p0) * kPageTokens);
    }
  }
  float m[kNT][2], l[kNT][2], o[8][kNT][4];
#pragma unroll
  for (int t = 0; t < kNT; ++t) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      m[t][e] = -INFINITY;
      l[t][e] = 0.f;
    }
#pragma unroll
    for (int c = 0; c < 8; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[c][t][e] = 0.f;
  }
  __syncthreads();                                       // barriers set up

  // The scales of this warp's next page are loaded one page ahead, its page id two pages ahead.
  const int64_t hs = a.heads;
  int id_cur = warp < n ? table[warp] : 0, id_next = warp + kDecWarps < n ? table[warp + kDecWarps] : 0;
  float ka = 0.f, va = 0.f;
  {
    const int64_t id = uint32_t(id_cur) < pool ? id_cur : 0;
    ka = a.ka[id * hs + h];
    va = a.va[id * hs + h];
  }
  for (int i = warp; i < n; i += kDecWarps) {
    const int s = i % kDecSlots;
    const int64_t idn = uint32_t(id_next) < pool ? id_next : 0;
    const float ka_next = a.ka[idn * hs + h], va_next = a.va[idn * hs + h];
    const int id_after = i + 2 * kDecWarps < n ? table[i + 2 * kDecWarps] : 0;
    const int id_fill = i + kDecSlots < n ? table[i + kDecSlots] : 0;
    if (!filled(i) || !mbar_wait(&sh.full[s], (i / kDecSlots) & 1, abort_flag, a.status, kDevTimeoutKV)) break;
    const uint32_t kb = smem_u32(ring + s * 2 * kPageBytes), vb = kb + kPageBytes;
    const bool ok = known(id_cur);

    // scores: tile mt holds keys 16 mt + r0 (elements 0, 1) and 16 mt + r0 + 8 (2, 3) of queries 2 quad, 2 quad + 1
    float x[kNT][4][4];
#pragma unroll
    for (int t = 0; t < kNT; ++t)
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[t][mt][e] = 0.f;
#pragma unroll
    for (int c2 = 0; c2 < 4; ++c2) {
      uint32_t r[4][4];                                  // [key tile]: keys 0-7 and 8-15 of piece 2 c2, then of 2 c2 + 1
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        const int key = mt * 16 + (lane & 15), c = 2 * c2 + (lane >> 4);
        ldsm4(kb + key * 128 + ((c ^ (key & 7)) << 4), r[mt]);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
          const uint32_t w0 = bias<kFmt>(r[mt][2 * k]), w1 = bias<kFmt>(r[mt][2 * k + 1]);
          const uint32_t f[4] = {widen<kFmt, 0, 1>(w0), widen<kFmt, 0, 1>(w1), widen<kFmt, 2, 3>(w0), widen<kFmt, 2, 3>(w1)};
#pragma unroll
          for (int t = 0; t < kNT; ++t) mma_f16(x[t][mt], f, qb[t][2 * c2 + k].x, qb[t][2 * c2 + k].y);
        }
    }
    const float kat = fmaxf(ka, kTinyScale), vat = fmaxf(va, kTinyScale);
    const float lv = __log2f(vat);
    const int j0 = i * kPageTokens;
    uint32_t pb[kNT][4][2];
#pragma unroll
    for (int t = 0; t < kNT; ++t) {
      if (!ok || min(limit[t][0], limit[t][1]) < j0 + 63) {
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = j0 + mt * 16 + r0 + 8 * (e >> 1);
            if (!ok || j > limit[t][e & 1]) x[t][mt][e] = -INFINITY;
          }
      }
      float c[2], bb[2], half[2], is[2];
      bool grow = false;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float top = fmaxf(x[t][0][e], x[t][0][2 + e]);
#pragma unroll
        for (int mt = 1; mt < 4; ++mt) top = fmax3(top, x[t][mt][e], x[t][mt][2 + e]);
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        c[e] = score_factor(kat, unit[t][e]);
        top = fmaf(top, c[e], lv);
        half[e] = 1.f;
        if (top > m[t][e] + kSlack) {                    // also from m = -inf
          half[e] = half_ex2(m[t][e] - top);
          m[t][e] = top;
          grow = true;
        }
        const float lift = lv + faint_exponent(top - m[t][e]);
        is[e] = ex2_approx(kSumBits - lift);
        // a query that has seen no key yet: its exponents are taken against 0 and are -inf
        bb[e] = lift - ((m[t][e] == -INFINITY ? 0.f : m[t][e]) - kWeightBits);
      }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          l[t][e] = l[t][e] * half[e] * half[e];
          half[e] *= half[e];
        }
#pragma unroll
        for (int c8 = 0; c8 < 8; ++c8)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[c8][t][e] *= half[e & 1];
      }
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] = ex2_approx(fmaf(x[t][mt][e], c[e & 1], bb[e & 1]));
          sum[e & 1] += w[e];
        }
        pb[t][mt][0] = movmatrix_t(pack_act2(w[0], w[1], 1));
        pb[t][mt][1] = movmatrix_t(pack_act2(w[2], w[3], 1));
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) l[t][e] = fmaf(sum[e], is[e], l[t][e]);
    }
    // rows of V past the sequence's tokens hold whatever the page held before: weight 0 times a NaN code (e4m3; int8 has
    // none) would be NaN, so they are read as 0
    const int rest = ok ? int(tk.kv - (int64_t(p0) * kPageTokens + j0)) : 0;
    const bool clip = kFmt == 1 && rest < kPageTokens;
    // o: rows r0 and r0 + 8 of a tile are channels 16 c + 2 r0 and 16 c + 2 r0 + 1, columns the queries
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int key = half * 32 + lane;
#pragma unroll
      for (int c4 = 0; c4 < 2; ++c4) {
        uint32_t r[4][4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          ldsm4_t(vb + key * 128 + (((4 * c4 + c) ^ (key & 7)) << 4), r[c]);
          if (clip) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int j = half * 32 + k * 8 + 2 * quad;
              r[c][k] &= (j < rest ? 0x0000ffffu : 0u) | (j + 1 < rest ? 0xffff0000u : 0u);
            }
          }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t w0 = bias<kFmt>(r[c][2 * k]), w1 = bias<kFmt>(r[c][2 * k + 1]);
            const uint32_t f[4] = {widen<kFmt, 0, 2>(w0), widen<kFmt, 1, 3>(w0), widen<kFmt, 0, 2>(w1), widen<kFmt, 1, 3>(w1)};
#pragma unroll
            for (int t = 0; t < kNT; ++t) mma_f16(o[4 * c4 + c][t], f, pb[t][half * 2 + k][0], pb[t][half * 2 + k][1]);
          }
      }
    }
    __syncwarp();                                          // every lane has read the slot
    if (lane == 0 && i + kDecSlots < n) issue(i + kDecSlots, id_fill);
    id_cur = id_next;
    id_next = id_after;
    ka = ka_next;
    va = va_next;
  }
  __syncthreads();
  const bool aborted = *abort_flag;
  if (aborted) {                                           // let copies in flight land before the CTA goes away
    if (threadIdx.x == 0)
      for (int s = 0; s < kDecSlots; ++s)
        if (sh.issued[s]) mbar_drain_wait(&sh.full[s], (sh.issued[s] - 1) & 1);
    if (single || !a.clustered) return;
    __syncthreads();                                       // the cluster's other CTAs wait for this one
  }

  // merge the warps: rows of 128 channels in the ring, which nothing reads any more
  float* mo = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int t = 0; t < kNT; ++t) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], d);
      const int q = 8 * t + 2 * quad + e;
      if (r0 == 0) {
        sh.m[warp][q] = m[t][e];
        sh.l[warp][q] = l[t][e] * kSumUnit;
      }
      float* row = mo + (warp * kRows + q) * kMergePitch + 2 * r0;
#pragma unroll
      for (int c = 0; c < 8; ++c) *reinterpret_cast<float2*>(row + 16 * c) = make_float2(o[c][t][e], o[c][t][2 + e]);
    }
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < kNT; ++t) {
    const int rr = 8 * t + (threadIdx.x >> 4), seg = threadIdx.x & 15;   // 8 channels a thread
    const int row = tile * kRows + rr, qi = row / a.group, head = h * a.group + (row - qi * a.group);
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) mm = fmaxf(mm, sh.m[w][rr]);
    const float ref = mm == -INFINITY ? 0.f : mm;
    float ll = 0.f, acc[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[k] = 0.f;
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
      const float half = half_ex2(sh.m[w][rr] - ref), f = half * half;
      ll += sh.l[w][rr] * half * half;
      const float4* p = reinterpret_cast<const float4*>(mo + (w * kRows + rr) * kMergePitch + 8 * seg);
      const float4 x = p[0], y = p[1];
      acc[0] += x.x * f;
      acc[1] += x.y * f;
      acc[2] += x.z * f;
      acc[3] += x.w * f;
      acc[4] += y.x * f;
      acc[5] += y.y * f;
      acc[6] += y.z * f;
      acc[7] += y.w * f;
    }
    if (single) {
      if (qi < a.q_len) {
        const float inv = ll == 0.f ? 0.f : a.v_unit / ll;
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          w[k] = ll == 0.f ? 0u : pack_act2(acc[2 * k] * inv, acc[2 * k + 1] * inv, kDt);
        uint16_t* p = static_cast<uint16_t*>(a.out) + b * a.so[0] + qi * a.so[1] + head * a.so[2] + seg * 8;
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        if (a.lse && seg == 0) a.lse[(int64_t(b) * a.q_len + qi) * (a.heads * a.group) + head] = natural_lse(mm - kWeightBits, ll);
      }
    } else if (a.clustered) {
      // this split's row, unscaled, behind the merge area
      float* p = mo + kDecWarps * kRows * kMergePitch + rr * 128 + 8 * seg;
      *reinterpret_cast<float4*>(p) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      *reinterpret_cast<float4*>(p + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
      if (seg == 0) sh.ml[rr] = make_float2(mm, ll);
    } else {
      const int64_t at = (int64_t(split) * a.batch * a.heads + int64_t(b) * a.heads + h) * (int64_t(a.tiles) * a.tile_rows) + row;
      float4* p = reinterpret_cast<float4*>(a.o_part + at * 128 + 8 * seg);
      p[0] = make_float4(acc[0] * a.v_unit, acc[1] * a.v_unit, acc[2] * a.v_unit, acc[3] * a.v_unit);
      p[1] = make_float4(acc[4] * a.v_unit, acc[5] * a.v_unit, acc[6] * a.v_unit, acc[7] * a.v_unit);
      if (seg == 0) a.ml_part[at] = make_float2(mm - kWeightBits, ll);
    }
  }
  if (single || !a.clustered) return;
  // The cluster's CTAs share the rows out, two at a time with two channels a thread, and read one another's splits.
  cluster_sync();
  const int ch = 2 * (threadIdx.x & 63);
  for (int rr = 2 * split + (threadIdx.x >> 6); rr < kRows; rr += 2 * a.splits) {
    const int row = tile * kRows + rr, qi = row / a.group, head = h * a.group + (row - qi * a.group);
    float2 ml[8], x[8];
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      ml[s] = make_float2(-INFINITY, 0.f);
      x[s] = make_float2(0.f, 0.f);
      if (s < a.splits) {
        ml[s] = peer_f2(&sh.ml[rr].x, s);
        x[s] = peer_f2(mo + kDecWarps * kRows * kMergePitch + rr * 128 + ch, s);
      }
    }
    float mm = -INFINITY;
#pragma unroll
    for (int s = 0; s < 8; ++s) mm = fmaxf(mm, ml[s].x);
    const float ref = mm == -INFINITY ? 0.f : mm;
    float ll = 0.f;
    float2 o2 = make_float2(0.f, 0.f);
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const float half = half_ex2(ml[s].x - ref), f = half * half;
      ll += ml[s].y * half * half;
      o2.x += x[s].x * f;
      o2.y += x[s].y * f;
    }
    if (qi < a.q_len) {
      const float inv = ll == 0.f ? 0.f : a.v_unit / ll;
      uint16_t* p = static_cast<uint16_t*>(a.out) + b * a.so[0] + qi * a.so[1] + head * a.so[2] + ch;
      *reinterpret_cast<uint32_t*>(p) = ll == 0.f ? 0u : pack_act2(o2.x * inv, o2.y * inv, kDt);
      if (a.lse && ch == 0) a.lse[(int64_t(b) * a.q_len + qi) * (a.heads * a.group) + head] = natural_lse(mm - kWeightBits, ll);
    }
  }
  cluster_sync();                                          // nobody reads this CTA's memory any more
}

// Merge of the key splits: one CTA a row, its 4 warps take the splits in turn, 4 channels a lane. A split's weight is
// 2^(m_s - max m). Rows whose tile fits one split were finished by the attention kernel. Few rows with many splits are
// the common case (a decoded token): what counts is latency, so up to 32 splits' loads go out together.
template <int kDt>
__global__ void __launch_bounds__(128) paged_combine_kernel(const PagedAttnArgs a) {
  const int row = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // the lengths are the caller's, written before the attention kernel, which let this grid start only after it had waited
  const TileKeys tk = tile_keys(a, b, row / a.tile_rows);
  after_previous_grid();
  const int pages = int((tk.visible + kPageTokens - 1) / kPageTokens);
  if (pages <= a.split_pages) return;
  const int n = (pages + a.split_pages - 1) / a.split_pages;
  const int64_t step = int64_t(a.batch) * a.heads * a.tiles * a.tile_rows;
  const int64_t at = (int64_t(b) * a.heads + h) * (int64_t(a.tiles) * a.tile_rows) + row;
  __shared__ float sm[4], sl[4];
  __shared__ float4 so[4][32];
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int kRound = 8;                                // splits a warp loads at once
  for (int s0 = warp; s0 < n; s0 += 4 * kRound) {
    float2 ml[kRound];
    float4 x[kRound];
#pragma unroll
    for (int k = 0; k < kRound; ++k) {
      const int s = s0 + 4 * k;
      ml[k] = make_float2(-INFINITY, 0.f);
      x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (s < n) {
        ml[k] = a.ml_part[s * step + at];
        x[k] = *reinterpret_cast<const float4*>(a.o_part + (s * step + at) * 128 + 4 * lane);
      }
    }
    float top = m;
#pragma unroll
    for (int k = 0; k < kRound; ++k) top = fmaxf(top, ml[k].x);
    const float ref = top == -INFINITY ? 0.f : top, half = half_ex2(m - ref), al = half * half;
    m = top;
    l = l * half * half;
    o = make_float4(o.x * al, o.y * al, o.z * al, o.w * al);
#pragma unroll
    for (int k = 0; k < kRound; ++k) {
      const float half_k = half_ex2(ml[k].x - ref), f = half_k * half_k;
      l += ml[k].y * half_k * half_k;
      o.x += x[k].x * f;
      o.y += x[k].y * f;
      o.z += x[k].z * f;
      o.w += x[k].w * f;
    }
  }
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
  so[warp][lane] = o;
  __syncthreads();
  if (warp != 0) return;
  const float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3])), ref = top == -INFINITY ? 0.f : top;
  l = 0.f;
  o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float half = half_ex2(sm[w] - ref), f = half * half;
    const float4 x = so[w][lane];
    l += sl[w] * half * half;
    o.x += x.x * f;
    o.y += x.y * f;
    o.z += x.z * f;
    o.w += x.w * f;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int i = row / a.group, head = h * a.group + (row - i * a.group);
  uint16_t* p = static_cast<uint16_t*>(a.out) + b * a.so[0] + i * a.so[1] + head * a.so[2] + 4 * lane;
  uint2 w = make_uint2(0u, 0u);
  if (l != 0.f) w = make_uint2(pack_act2(o.x * inv, o.y * inv, kDt), pack_act2(o.z * inv, o.w * inv, kDt));
  *reinterpret_cast<uint2*>(p) = w;
  if (a.lse && lane == 0) a.lse[(int64_t(b) * a.q_len + i) * (a.heads * a.group) + head] = natural_lse(top, l);
}

template <int kFmt, int kDt, int kNT>
cudaError_t launch_decode_as(const PagedAttnArgs& a, const CUtensorMap& tm_k, const CUtensorMap& tm_v, cudaStream_t st) {
  if (cudaError_t e = allow_dynamic_smem<paged_decode_kernel<kFmt, kDt, kNT>>(int(kDecSmem)); e != cudaSuccess) return e;
  const dim3 grid(unsigned(a.heads) * a.tiles, a.splits, a.batch);
  return launch_after_clustered(paged_decode_kernel<kFmt, kDt, kNT>, dim3(1, a.clustered ? a.splits : 1), grid,
                                dim3(kDecWarps * 32), kDecSmem, st, tm_k, tm_v, a);
}
template <int kFmt, int kDt>
cudaError_t launch_decode_rows(const PagedAttnArgs& a, const CUtensorMap& tm_k, const CUtensorMap& tm_v, cudaStream_t st) {
  return a.tile_rows == 8 ? launch_decode_as<kFmt, kDt, 1>(a, tm_k, tm_v, st) : launch_decode_as<kFmt, kDt, 2>(a, tm_k, tm_v, st);
}
cudaError_t launch_paged_decode(const PagedAttnArgs& a, const CUtensorMap& tm_k, const CUtensorMap& tm_v,
                                cudaStream_t st) {
  if (a.fmt) return a.dtype ? launch_decode_rows<1, 1>(a, tm_k, tm_v, st) : launch_decode_rows<1, 0>(a, tm_k, tm_v, st);
  return a.dtype ? launch_decode_rows<0, 1>(a, tm_k, tm_v, st) : launch_decode_rows<0, 0>(a, tm_k, tm_v, st);
}
cudaError_t launch_paged_combine(const PagedAttnArgs& a, cudaStream_t st) {
  const dim3 grid(unsigned(a.q_len) * a.group, a.heads, a.batch);
  return a.dtype ? launch_after(paged_combine_kernel<1>, grid, dim3(128), 0, st, a)
                 : launch_after(paged_combine_kernel<0>, grid, dim3(128), 0, st, a);
}

}  // namespace lbq
