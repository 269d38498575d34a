// Attention over the paged 8-bit KV cache, sm_100a: many query rows (prompts, whole chunks).
//
// The formulas of pattn.cu with both products on tcgen05. Per page (64 keys) and 128-row query tile:
//   S = Q . C^T (kind::f16, fp32 in tensor memory): C the K codes widened to fp16 (exact), Q in fp16 with a power of two
//       per row taken out; score x = S * c, c = amax_k * 2^e * softmax scale * log2 e / Q one factor a row and page
//   P = 2^(x + log2 amax_v - m + 7) as fp16 in tensor memory, over S; O += P . D (D the V codes in fp16)
//   l += sum P / amax_v (fp32, before the rounding);  out = O / (Q l)
// P in fp16 is off by 2^-11 relative, as in pattn.cu (bf16 would be off by 2^-8, and tf32 has half the rate).
//
// Bound by the tensor pipe and by exp2 alike: a page and 256 rows are 1024 clocks of MMA (8192 flops a clock) and 1024
// clocks of MUFU. CTA = two 128-row query tiles of one K/V head and key split, 512 threads:
//   warps 0-3 / 4-7  softmax of tile A / B, one thread a row (= TMEM lane): also load and scale Q, rescale O, and store the
//                    result;
//   warps 8-11       widen the pages: global memory -> registers (one page ahead) -> fp16 tiles in shared memory. The
//                    codes must pass through registers to be widened, so they are loaded there and not staged by TMA;
//   warp 12          MMA issuer and tensor-memory owner.
// Shared memory: Q 64 KB, K and V four fp16 stages (pages) of 16 KB each. K tiles are K-major, V tiles MN-major, and both
// have one layout: 128-byte rows of 64 channels of a key, 128-byte swizzle, the two channel halves 8 KB apart. Tensor
// memory: S_A, S_B two 64-column buffers each (pages u and u + 1), O_A, O_B 128 columns, P over the first half of its S
// buffer. The product P.D of a page must be complete before scores of page u + 2 overwrite P (different accumulators give
// no order); meanwhile the softmax works on page u + 1. With one 128-key buffer a tile (no second page in hand) every
// product's latency lay bare between two softmax steps: 5800 clocks for 128 keys, 1539 us for a chunk of 6032 queries x
// 30160 keys x 12 heads.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "lbq_kernels.h"
#include "lbq_paged.h"
#include "lbq_paged.cuh"
#include "lbq_ptx.cuh"

namespace lbq {

namespace {

constexpr int kRowThreads = 512;
constexpr int kQHalf = 128 * 128;                // bytes of 128 query rows of 64 fp16 channels
constexpr int kQTile = 2 * kQHalf;
constexpr int kHalf = 64 * 128;                  // bytes of 64 keys of 64 fp16 channels
constexpr int kPage16 = 2 * kHalf;               // a page of fp16 values
constexpr int kRowStages = 4;
constexpr uint32_t kIdescScores = idesc_m128(64, 1, 0, 0);     // f32 <- f16 x f16, N = 64 keys
constexpr uint32_t kRegSoftmax = 168, kRegWiden = 104, kRegIssue = 72;
static_assert(128 * (2 * kRegSoftmax + kRegWiden + kRegIssue) <= kRowThreads * 128, "register split");
struct RowsShared {
  uint64_t q_full;                               // both query tiles in shared memory (256 threads)
  uint64_t k_full[kRowStages], v_full[kRowStages];      // 128 widening threads
  uint64_t k_empty[kRowStages], v_empty[kRowStages];    // MMAs that read the stage complete
  uint64_t s_full[2][2];                         // [tile][page & 1]: scores complete
  uint64_t p_full[2][2];                         // weights written, O rescaled (128 threads)
  uint64_t o_done[2][2];                         // product complete
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
};
constexpr size_t kRowsSmem = 1024 + 2 * kQTile + 2 * kRowStages * kPage16 + sizeof(RowsShared);
static_assert(kRowsSmem <= 232448, "shared memory");

// 8 codes -> 8 fp16 values.
template <int kFmt>
__device__ __forceinline__ uint4 widen8(const uint2 r) {
  const uint32_t a = bias<kFmt>(r.x), b = bias<kFmt>(r.y);
  return make_uint4(widen<kFmt, 0, 1>(a), widen<kFmt, 2, 3>(a), widen<kFmt, 0, 1>(b), widen<kFmt, 2, 3>(b));
}

// One query row (null: zeros) as fp16 into row rl of a swizzled tile, scaled by a power of two to a maximum in [1, 2)
// (bf16; fp16 rows go as they are); returns the factor that undoes it.
template <int kDt>
__device__ __forceinline__ float stage_query(const uint16_t* row, uint8_t* tile, int rl) {
  float down = 1.f, up = 1.f;
  if constexpr (kDt == 0) {
    uint32_t top = 0;
    if (row != nullptr) {
#pragma unroll 4
      for (int c = 0; c < 16; ++c) {
        const uint4 r = reinterpret_cast<const uint4*>(row)[c];
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, max((w[i] << 16) & 0x7fffffffu, w[i] & 0x7fff0000u));
      }
    }
    down = row_scale(top, up);
  }
#pragma unroll 4
  for (int c = 0; c < 16; ++c) {
    uint4 r = row != nullptr ? reinterpret_cast<const uint4*>(row)[c] : make_uint4(0u, 0u, 0u, 0u);
    if constexpr (kDt == 0) {
      uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = pack_act2(__uint_as_float(w[i] << 16) * down, __uint_as_float(w[i] & 0xffff0000u) * down, 1);
      r = make_uint4(w[0], w[1], w[2], w[3]);
    }
    *reinterpret_cast<uint4*>(tile + (c >> 3) * kQHalf + rl * 128 + (((c & 7) ^ (rl & 7)) << 4)) = r;
  }
  return up;
}

template <int kFmt, int kDt>
__global__ void __launch_bounds__(kRowThreads, 1) paged_rows_kernel(const PagedAttnArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = smem + 2 * kQTile;
  uint8_t* sV = sK + kRowStages * kPage16;
  RowsShared* sh = reinterpret_cast<RowsShared*>(sV + kRowStages * kPage16);
  volatile int* abort_flag = &sh->abort;
  after_previous_grid();
  // the last row tiles see the most keys under a causal mask: they start first
  const int tile = a.tiles - 1 - int(blockIdx.x % a.tiles), h = blockIdx.x / a.tiles, split = blockIdx.y, b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const TileKeys tk = tile_keys(a, b, tile);
  const int pages = int((tk.visible + kPageTokens - 1) / kPageTokens);
  const int p0 = split * a.split_pages;
  const int n = max(0, min(pages - p0, a.split_pages));
  if (split > 0 && n == 0) return;
  const bool single = pages <= a.split_pages;
  const int32_t* table = a.pt.table + b * a.pt.st_b + p0;
  const uint32_t pool = uint32_t(a.pt.num_pages);

  if (threadIdx.x == 0) {
    mbar_init(&sh->q_full, 256);
    for (int s = 0; s < kRowStages; ++s) {
      mbar_init(&sh->k_full[s], 128);
      mbar_init(&sh->v_full[s], 128);
      mbar_init(&sh->k_empty[s], 1);
      mbar_init(&sh->v_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      for (int e = 0; e < 2; ++e) {
        mbar_init(&sh->s_full[t][e], 1);
        mbar_init(&sh->p_full[t][e], 128);
        mbar_init(&sh->o_done[t][e], 1);
      }
    }
    mbar_init(&sh->drain, 1);
    sh->abort = 0;
    fence_mbar_init();
  }
  if (warp == 12) {
    tmem_alloc(&sh->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem_base;

  if (warp >= 12) {
    reg_dealloc<kRegIssue>();
    if (warp == 12 && n > 0) {
      // ---------------------------------------------------------- MMA issuer (one lane issues)
      const uint64_t qd = smem_desc_sw128(smem_u32(sQ)), kd = smem_desc_sw128(smem_u32(sK));
      const uint64_t vd = smem_desc_sw128_mn(smem_u32(sV), kHalf);
      auto scores = [&](int t, int u) {
        const uint64_t q0 = qd + t * (kQTile >> 4), k0 = kd + (u % kRowStages) * (kPage16 >> 4);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 8; ++k)                    // 16 channels a step, 4 steps a 64-channel half
            mma_f16_ss(tmem + 128 * t + 64 * (u & 1), q0 + (k >> 2) * (kQHalf >> 4) + 2 * (k & 3),
                       k0 + (k >> 2) * (kHalf >> 4) + 2 * (k & 3), kIdescScores, k > 0);
          tc_commit(&sh->s_full[t][u & 1]);
        }
        __syncwarp();
      };
      auto have_k = [&](int u) {
        return mbar_wait(&sh->k_full[u % kRowStages], (u / kRowStages) & 1, abort_flag, a.status, kDevTimeoutKV);
      };
      bool ok = mbar_wait_role(&sh->q_full, 0, abort_flag, a.status, kDevTimeoutQ);
      for (int u = 0; ok && u < min(n, 2); ++u) {
        if (!(ok = have_k(u))) break;
        tc_fence_after();
        scores(0, u);
        scores(1, u);
        if (elect_one()) tc_commit(&sh->k_empty[u]);
        __syncwarp();
      }
      for (int u = 0; ok && u < n; ++u) {
        const int s = u % kRowStages, e = u & 1;
        const uint32_t phase = (u >> 1) & 1;
        if (!(ok = mbar_wait(&sh->v_full[s], (u / kRowStages) & 1, abort_flag, a.status, kDevTimeoutKV))) break;
        for (int t = 0; ok && t < 2; ++t) {
          if (!(ok = mbar_wait(&sh->p_full[t][e], phase, abort_flag, a.status, kDevTimeoutP))) break;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 4; ++k)                  // 16 keys a step: 8 columns of P, 2 groups of 8 rows of V
              mma_f16_ts(tmem + 256 + 128 * t, tmem + 128 * t + 64 * e + 8 * k, vd + s * (kPage16 >> 4) + k * (2048 >> 4),
                         kIdescF16BMn, u > 0 || k > 0);
            tc_commit(&sh->o_done[t][e]);
          }
          __syncwarp();
        }
        if (!ok) break;
        if (elect_one()) tc_commit(&sh->v_empty[s]);
        __syncwarp();
        if (u + 2 < n) {
          if (!(ok = have_k(u + 2))) break;
          for (int t = 0; ok && t < 2; ++t) {
            if (!(ok = mbar_wait(&sh->o_done[t][e], phase, abort_flag, a.status, kDevTimeoutO))) break;
            tc_fence_after();
            scores(t, u + 2);
          }
          if (!ok) break;
          if (elect_one()) tc_commit(&sh->k_empty[(u + 2) % kRowStages]);
          __syncwarp();
        }
      }
      if (elect_one()) tc_commit(&sh->drain);            // every MMA has completed once it flips
      __syncwarp();
      mbar_drain_wait(&sh->drain, 0);
    }
  } else if (warp >= 8) {
    // ------------------------------------------------------------ widening warps
    reg_dealloc<kRegWiden>();
    const int w = warp - 8, c = lane & 7, half = c >> 2;
    // piece i of a page: key 16 i + 4 w + lane / 8, 16-byte piece c of its row: a load takes four whole 128-byte rows.
    // Its 16 values are two 16-byte pieces of the key's row in channel half `half`; the lanes of one half store the first
    // one first and those of the other the second, so that the eight lanes of a key take all eight bank groups at once.
    auto load = [&](const uint8_t* base, int u, int id, uint4 (&r)[4]) {
      const bool ok = uint32_t(id) < pool;
      if (!ok && a.status) atomicCAS(a.status, 0, kDevBadPage);
      const uint8_t* pg = base + (int64_t(ok ? id : 0) * a.heads + h) * kPageBytes;
      // rows past the sequence hold what the page held before: a NaN code times a weight of 0 would be NaN
      const int64_t rest = ok ? tk.kv - int64_t(p0 + u) * kPageTokens : 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = 16 * i + 4 * w + (lane >> 3);
        r[i] = key < rest ? *reinterpret_cast<const uint4*>(pg + key * 128 + c * 16) : make_uint4(0u, 0u, 0u, 0u);
      }
    };
    auto store = [&](uint8_t* dst, const uint4 (&r)[4]) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = 16 * i + 4 * w + (lane >> 3), k7 = key & 7, at = 2 * (c & 3);
        uint8_t* row = dst + half * kHalf + key * 128;
        const uint2 first = half ? make_uint2(r[i].z, r[i].w) : make_uint2(r[i].x, r[i].y);
        const uint2 second = half ? make_uint2(r[i].x, r[i].y) : make_uint2(r[i].z, r[i].w);
        *reinterpret_cast<uint4*>(row + (((at + half) ^ k7) << 4)) = widen8<kFmt>(first);
        *reinterpret_cast<uint4*>(row + (((at + 1 - half) ^ k7) << 4)) = widen8<kFmt>(second);
      }
      fence_proxy_async_smem();
    };
    uint4 kreg[4], vreg[4];
    int id_next = 0;
    if (n > 0) {
      const int id = table[0];
      load(a.k_pages, 0, id, kreg);
      load(a.v_pages, 0, id, vreg);
      if (n > 1) id_next = table[1];
    }
    for (int u = 0; u < n; ++u) {
      const int s = u % kRowStages;
      const uint32_t phase = ((u / kRowStages) & 1) ^ 1;
      const int id = id_next;
      if (u + 2 < n) id_next = table[u + 2];
      if (!mbar_wait_role(&sh->k_empty[s], phase, abort_flag, a.status, kDevTimeoutKV)) break;
      store(sK + s * kPage16, kreg);
      mbar_arrive(&sh->k_full[s]);
      if (u + 1 < n) load(a.k_pages, u + 1, id, kreg);
      if (!mbar_wait_role(&sh->v_empty[s], phase, abort_flag, a.status, kDevTimeoutKV)) break;
      store(sV + s * kPage16, vreg);
      mbar_arrive(&sh->v_full[s]);
      if (u + 1 < n) load(a.v_pages, u + 1, id, vreg);
    }
  } else {
    // ------------------------------------------------------------ softmax warps
    reg_alloc<kRegSoftmax>();
    const int t = warp >> 2, quarter = warp & 3, rl = quarter * 32 + lane;
    const uint32_t lane_off = uint32_t(quarter * 32) << 16;
    const uint32_t tS0 = tmem + 128 * t + lane_off, tO = tmem + 256 + 128 * t + lane_off;
    const int row = tile * kManyTile + t * 128 + rl, qi = row / a.group, head = h * a.group + (row - qi * a.group);
    const bool on = qi < tk.qn;
    const uint16_t* qrow = on ? static_cast<const uint16_t*>(a.q) + b * a.sq[0] + qi * a.sq[1] + head * a.sq[2] : nullptr;
    const float unit = row_factor(stage_query<kDt>(qrow, sQ + t * kQTile, rl), a.score_log2);
    fence_proxy_async_smem();
    mbar_arrive(&sh->q_full);
    const int limit = !on ? -1 : int((a.causal ? tk.kv - tk.qn + qi : tk.kv - 1) - int64_t(p0) * kPageTokens);
    float m = -INFINITY, l = 0.f;
    // The scales of the next page are loaded one page ahead, its id two pages ahead. They are kept above 0 (a written
    // page's are at least 2^-40): the logarithm of va is taken.
    int id_next = n > 0 ? table[0] : 0;
    float ka_next = 1.f, va_next = 1.f;
    bool ok_next = false;
    auto scales = [&](int u) {
      ok_next = uint32_t(id_next) < pool;
      const int64_t at = int64_t(ok_next ? id_next : 0) * a.heads + h;
      ka_next = a.ka[at];
      va_next = a.va[at];
      if (u + 1 < n) id_next = table[u + 1];
    };
    if (n > 0) scales(0);
    bool ok = true;
    for (int u = 0; u < n; ++u) {
      const bool known = ok_next;
      const float ka = fmaxf(ka_next, kTinyScale), va = fmaxf(va_next, kTinyScale);
      if (u + 1 < n) scales(u + 1);
      const uint32_t tS = tS0 + 64 * (u & 1);
      if (!(ok = mbar_wait(&sh->s_full[t][u & 1], (u >> 1) & 1, abort_flag, a.status, kDevTimeoutS))) break;
      tc_fence_after();
      uint32_t sv[64];
      auto& sv0 = *reinterpret_cast<uint32_t(*)[32]>(&sv[0]);
      auto& sv1 = *reinterpret_cast<uint32_t(*)[32]>(&sv[32]);
      tmem_ld32(tS, sv0);
      tmem_ld32(tS + 32, sv1);
      tmem_ld_wait(sv0);
      reg_anchor(sv1);
      auto F = [&](int i) { return __uint_as_float(sv[i]); };
      const int rest = limit - u * kPageTokens;           // last visible key of the page
      if (!__all_sync(0xffffffffu, rest >= 63 && known)) {
        const int last = known ? min(rest, 63) : -1;
#pragma unroll
        for (int i = 0; i < 64; ++i)
          if (i > last) sv[i] = 0xff800000u;
      }
      float r[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) r[q] = fmaxf(F(2 * q), F(2 * q + 1));
#pragma unroll
      for (int i = 8; i < 64; i += 8) {
#pragma unroll
        for (int q = 0; q < 4; ++q) r[q] = fmax3(r[q], F(i + 2 * q), F(i + 2 * q + 1));
      }
      const float c = score_factor(ka, unit), lv = __log2f(va);
      const float top = fmaf(fmax3(r[0], r[1], fmaxf(r[2], r[3])), c, lv);
      const bool grow = top > m + kSlack;                 // also from m = -inf
      if (__any_sync(0xffffffffu, grow)) {
        const float half = grow ? half_ex2(m - top) : 1.f, alpha = half * half;
        if (grow) m = top;
        l = l * half * half;
        if (u > 0) {                                      // products up to page u - 2 are complete, as its scores are
          if (!(ok = mbar_wait(&sh->o_done[t][(u - 1) & 1], ((u - 1) >> 1) & 1, abort_flag, a.status, kDevTimeoutO))) break;
          tc_fence_after();
#pragma unroll 1
          for (int cc = 0; cc < 4; ++cc) {
            uint32_t ov[32];
            tmem_ld32(tO + 32 * cc, ov);
            tmem_ld_wait(ov);
#pragma unroll
            for (int e = 0; e < 32; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
            tmem_st32(tO + 32 * cc, ov);
          }
        }
      }
      const float lift = lv + faint_exponent(top - m);
      const float ref = lift - ((m == -INFINITY ? 0.f : m) - kWeightBits);
      const uint64_t c2 = f2_pack(c, c), b2 = f2_pack(ref, ref);
      uint64_t acc[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        float w0, w1;
        f2_unpack(f2_fma(f2_pack(F(2 * i), F(2 * i + 1)), c2, b2), w0, w1);
        w0 = ex2_approx(w0);
        w1 = ex2_approx(w1);
        acc[i & 1] = f2_add(acc[i & 1], f2_pack(w0, w1));
        sv[i] = pack_act2(w0, w1, 1);
      }
      tmem_st32(tS, sv0);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&sh->p_full[t][u & 1]);
      float s[4];
      f2_unpack(acc[0], s[0], s[1]);
      f2_unpack(acc[1], s[2], s[3]);
      l = fmaf((s[0] + s[1]) + (s[2] + s[3]), ex2_approx(kSumBits - lift), l);
    }
    l *= kSumUnit;
    if (ok && n > 0) ok = mbar_wait(&sh->o_done[t][(n - 1) & 1], ((n - 1) >> 1) & 1, abort_flag, a.status, kDevTimeoutO);
    tc_fence_after();
    // ---------------------------------------------------------- result: O / (Q l), or the split's O / Q, m - 7, l
    const bool row_ok = ok && qi < a.q_len;
    const float inv = single ? (l == 0.f ? 0.f : __fdividef(a.v_unit, l)) : a.v_unit;
    const int64_t at = (int64_t(split) * a.batch * a.heads + int64_t(b) * a.heads + h) * (int64_t(a.tiles) * a.tile_rows) + row;
    uint16_t* orow = static_cast<uint16_t*>(a.out) + b * a.so[0] + qi * a.so[1] + head * a.so[2];
    float* prow = a.o_part + at * 128;
    if (ok) {
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t ov[32];
        if (n > 0) {
          tmem_ld32(tO + 32 * c, ov);
          tmem_ld_wait(ov);
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float x = __uint_as_float(ov[e]) * inv;
          ov[e] = n == 0 || l == 0.f ? 0u : __float_as_uint(x);
        }
        if (single && row_ok) {
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = pack_act2(__uint_as_float(ov[2 * e]), __uint_as_float(ov[2 * e + 1]), kDt);
          if (a.wide_out) {
            st_global_v8(orow + 32 * c, w);
            st_global_v8(orow + 32 * c + 16, w + 8);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              reinterpret_cast<uint4*>(orow + 32 * c)[e] = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
          }
        } else if (!single) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            reinterpret_cast<uint4*>(prow + 32 * c)[e] = make_uint4(ov[4 * e], ov[4 * e + 1], ov[4 * e + 2], ov[4 * e + 3]);
        }
      }
      if (single) {
        if (row_ok && a.lse) a.lse[(int64_t(b) * a.q_len + qi) * (a.heads * a.group) + head] = natural_lse(m - kWeightBits, l);
      } else {
        a.ml_part[at] = make_float2(m - kWeightBits, l);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 12) tmem_dealloc(tmem, 512);
}

template <int kFmt, int kDt>
cudaError_t launch_rows_as(const PagedAttnArgs& a, cudaStream_t st) {
  if (cudaError_t e = allow_dynamic_smem<paged_rows_kernel<kFmt, kDt>>(int(kRowsSmem)); e != cudaSuccess) return e;
  return launch_after(paged_rows_kernel<kFmt, kDt>, dim3(unsigned(a.heads) * a.tiles, a.splits, a.batch), dim3(kRowThreads),
                      kRowsSmem, st, a);
}

}  // namespace

cudaError_t launch_paged_rows(const PagedAttnArgs& a, cudaStream_t st) {
  if (a.fmt) return a.dtype ? launch_rows_as<1, 1>(a, st) : launch_rows_as<1, 0>(a, st);
  return a.dtype ? launch_rows_as<0, 1>(a, st) : launch_rows_as<0, 0>(a, st);
}

}  // namespace lbq
