// Attention over the paged 8-bit KV cache, sm_100a: many query rows (prompts, whole chunks).
//
// The formulas of pattn.cu with both products on tcgen05. Per 128-key tile (two pages) and 128-row query tile:
//   S = Q . C^T (kind::f16, fp32 in tensor memory): C the K codes widened to fp16 (exact), Q in fp16 with a power of two
//       per row taken out; score x = S * c, c = amax_k * 2^e * softmax scale * log2 e / Q one factor a row and page
//   P = 2^(x + log2 amax_v - m) as fp16 in tensor memory, over S; O += P . D (D the V codes in fp16)
//   l += sum P / amax_v (fp32, before the rounding);  out = O / (Q l)
// The scale of a V page rides in the exponent, so m is the running maximum of x + log2 amax_v: the weights that the
// product needs are those nearest 1 and nothing overflows fp16 whatever the pages' magnitudes. m moves only when a
// row's maximum exceeds it by more than 2^8 (weights carry a factor 2^7 and stay below 2^15), which is when O and l are
// rescaled; the rounding of a weight is 2^-12 relative down to 2^-21 of the row's largest.
//
// Bound by the tensor pipe and by exp2 alike: a step (128 keys, 256 rows) has 2048 clocks of MMA (8192 flops a clock) and
// 2048 clocks of MUFU. CTA = two 128-row query tiles of one K/V head and key split, 512 threads:
//   warps 0-3 / 4-7  softmax of tile A / B, one thread a row (= TMEM lane): also load and scale Q, rescale O (its last
//                    product is complete by the time the next scores are), and store the result;
//   warps 8-11       widen the pages: global memory -> registers (one tile ahead) -> fp16 tiles in shared memory. The
//                    codes must pass through registers to be widened, so they are loaded there and not staged by TMA;
//   warp 12          MMA issuer and tensor-memory owner.
// Shared memory: Q 64 KB, K and V two fp16 stages of 32 KB each. K tiles are K-major, V tiles MN-major, and both have one
// layout: 128-byte rows of 64 channels of a key, 128-byte swizzle, the two channel halves 16 KB apart. Tensor memory:
// S_A, S_B, O_A, O_B, 128 columns each, P_t over the first 64 columns of S_t: the product P.D of a tile must be complete
// before the next scores of that tile are issued (different accumulators give no order), and while it is waited for, the
// other tile's softmax runs.
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
constexpr int kHalf = 128 * 128;                 // bytes of 128 rows of 64 fp16 channels
constexpr int kTile16 = 2 * kHalf;               // a 128 x 128 fp16 tile
constexpr int kRowStages = 2;
constexpr uint32_t kRegSoftmax = 168, kRegWiden = 128, kRegIssue = 48;
static_assert(128 * (2 * kRegSoftmax + kRegWiden + kRegIssue) <= kRowThreads * 128, "register split");
struct RowsShared {
  uint64_t q_full;                               // both query tiles in shared memory (256 threads)
  uint64_t k_full[kRowStages], v_full[kRowStages];      // 128 widening threads
  uint64_t k_empty[kRowStages], v_empty[kRowStages];    // MMAs that read the stage complete
  uint64_t s_full[2];                            // scores of tile t complete
  uint64_t p_full[2];                            // weights of tile t written, O rescaled (128 threads)
  uint64_t o_done[2];                            // product of tile t complete
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
};
constexpr size_t kRowsSmem = 1024 + 2 * kTile16 + 2 * kRowStages * kTile16 + sizeof(RowsShared);
static_assert(kRowsSmem <= 232448, "shared memory");

// 16 codes -> 16 fp16 values (two 16-byte pieces).
template <int kFmt>
__device__ __forceinline__ void widen16(const uint4 r, uint4& lo, uint4& hi) {
  const uint32_t w[4] = {bias<kFmt>(r.x), bias<kFmt>(r.y), bias<kFmt>(r.z), bias<kFmt>(r.w)};
  lo = make_uint4(widen<kFmt, 0, 1>(w[0]), widen<kFmt, 2, 3>(w[0]), widen<kFmt, 0, 1>(w[1]), widen<kFmt, 2, 3>(w[1]));
  hi = make_uint4(widen<kFmt, 0, 1>(w[2]), widen<kFmt, 2, 3>(w[2]), widen<kFmt, 0, 1>(w[3]), widen<kFmt, 2, 3>(w[3]));
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
    uint32_t e = top >> 23;
    const bool plain = e == 0 || e == 255;
    if (e == 254) e = 253;
    if (!plain) {
      down = __uint_as_float((254u - e) << 23);
      up = __uint_as_float(e << 23);
    }
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
    *reinterpret_cast<uint4*>(tile + (c >> 3) * kHalf + rl * 128 + (((c & 7) ^ (rl & 7)) << 4)) = r;
  }
  return up;
}

// Page ids and scales of one 128-key tile.
struct TileScale {
  float ka[2], va[2];
  bool ok[2];
};

template <int kFmt, int kDt>
__global__ void __launch_bounds__(kRowThreads, 1) paged_rows_kernel(const PagedAttnArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = smem + 2 * kTile16;
  uint8_t* sV = sK + kRowStages * kTile16;
  RowsShared* sh = reinterpret_cast<RowsShared*>(sV + kRowStages * kTile16);
  volatile int* abort_flag = &sh->abort;
  asm volatile("griddepcontrol.launch_dependents;");     // a merge of key splits may be launched; it waits for the end
  // the last row tiles see the most keys under a causal mask: they start first
  const int tile = a.tiles - 1 - int(blockIdx.x % a.tiles), h = blockIdx.x / a.tiles, split = blockIdx.y, b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const TileKeys tk = tile_keys(a, b, tile);
  const int pages = int((tk.visible + kPageTokens - 1) / kPageTokens);
  const int p0 = split * a.split_pages;
  const int np = max(0, min(pages - p0, a.split_pages));
  if (split > 0 && np == 0) return;
  const int n = (np + 1) / 2;                            // 128-key tiles
  const bool single = pages <= a.split_pages;
  const int32_t* table = a.pt.table + b * a.pt.st_b + p0;
  // A page of the split, 0 with ok = false past its end or outside the pool (recorded).
  auto page_id = [&](int i, bool& ok) {
    ok = false;
    if (i >= np) return 0;
    const int id = table[i];
    ok = id >= 0 && id < a.pt.num_pages;
    if (!ok && a.status) atomicCAS(a.status, 0, kDevBadPage);
    return ok ? id : 0;
  };

  if (threadIdx.x == 0) {
    mbar_init(&sh->q_full, 256);
    for (int s = 0; s < kRowStages; ++s) {
      mbar_init(&sh->k_full[s], 128);
      mbar_init(&sh->v_full[s], 128);
      mbar_init(&sh->k_empty[s], 1);
      mbar_init(&sh->v_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&sh->s_full[t], 1);
      mbar_init(&sh->p_full[t], 128);
      mbar_init(&sh->o_done[t], 1);
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
      const uint32_t tS[2] = {tmem, tmem + 128}, tO[2] = {tmem + 256, tmem + 384};
      const uint64_t qd = smem_desc_sw128(smem_u32(sQ)), kd = smem_desc_sw128(smem_u32(sK));
      const uint64_t vd = smem_desc_sw128_mn(smem_u32(sV), kHalf);
      constexpr uint64_t kTileDesc = kTile16 >> 4, kHalfDesc = kHalf >> 4;
      auto scores = [&](int t, int j) {
        const uint64_t q0 = qd + t * kTileDesc, k0 = kd + (j % kRowStages) * kTileDesc;
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 8; ++k)                    // 16 channels a step, 4 steps a 64-channel half
            mma_f16_ss(tS[t], q0 + (k >> 2) * kHalfDesc + 2 * (k & 3), k0 + (k >> 2) * kHalfDesc + 2 * (k & 3), kIdescF16,
                       k > 0);
          tc_commit(&sh->s_full[t]);
        }
        __syncwarp();
      };
      bool ok = mbar_wait_role(&sh->q_full, 0, abort_flag, a.status, kDevTimeoutQ) &&
                mbar_wait_role(&sh->k_full[0], 0, abort_flag, a.status, kDevTimeoutKV);
      tc_fence_after();
      if (ok) {
        scores(0, 0);
        scores(1, 0);
        if (elect_one()) tc_commit(&sh->k_empty[0]);
        __syncwarp();
      }
      for (int j = 0; ok && j < n; ++j) {
        const int s = j % kRowStages;
        if (!(ok = mbar_wait(&sh->v_full[s], (j / kRowStages) & 1, abort_flag, a.status, kDevTimeoutKV))) break;
        const bool more = j + 1 < n;
        if (more && !(ok = mbar_wait(&sh->k_full[(j + 1) % kRowStages], ((j + 1) / kRowStages) & 1, abort_flag, a.status,
                                     kDevTimeoutKV)))
          break;
        for (int t = 0; ok && t < 2; ++t) {
          if (!(ok = mbar_wait(&sh->p_full[t], j & 1, abort_flag, a.status, kDevTimeoutP))) break;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 8; ++k)                  // 16 keys a step: 8 columns of P, 2 groups of 8 rows of V
              mma_f16_ts(tO[t], tS[t] + 8 * k, vd + s * kTileDesc + k * (2048 >> 4), kIdescF16BMn, j > 0 || k > 0);
            tc_commit(&sh->o_done[t]);
          }
          __syncwarp();
          if (more) {
            if (!(ok = mbar_wait(&sh->o_done[t], j & 1, abort_flag, a.status, kDevTimeoutO))) break;
            tc_fence_after();
            scores(t, j + 1);
          }
        }
        if (!ok) break;
        if (elect_one()) {
          tc_commit(&sh->v_empty[s]);
          if (more) tc_commit(&sh->k_empty[(j + 1) % kRowStages]);
        }
        __syncwarp();
      }
      if (elect_one()) tc_commit(&sh->drain);            // every MMA has completed once it flips
      __syncwarp();
      mbar_drain_wait(&sh->drain, 0);
    }
  } else if (warp >= 8) {
    // ------------------------------------------------------------ widening warps
    reg_dealloc<kRegWiden>();
    const int w = warp - 8, kr = lane & 7, c4 = lane >> 3;
    // piece i of a tile: key 8 * (u / 2) + kr, 16-byte piece 4 * (u % 2) + c4 of its row, u = 4 i + w. Eight lanes of a
    // store take eight keys, whose swizzle spreads them over all banks.
    auto load = [&](const uint8_t* base, int j, uint4 (&r)[8]) {
      bool ok[2];
      const uint8_t* pg[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int64_t id = page_id(2 * j + e, ok[e]);
        pg[e] = base + (id * a.heads + h) * kPageBytes;
      }
      const int64_t k0 = int64_t(p0 + 2 * j) * kPageTokens;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int u = 4 * i + w, key = (u >> 1) * 8 + kr;
        // rows past the sequence hold what the page held before: a NaN code times a weight of 0 would be NaN
        r[i] = ok[i >> 2] && k0 + key < tk.kv
                   ? *reinterpret_cast<const uint4*>(pg[i >> 2] + (key & 63) * 128 + ((u & 1) * 4 + c4) * 16)
                   : make_uint4(0u, 0u, 0u, 0u);
      }
    };
    auto store = [&](uint8_t* dst, const uint4 (&r)[8]) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int u = 4 * i + w, key = (u >> 1) * 8 + kr;
        uint4 lo, hi;
        widen16<kFmt>(r[i], lo, hi);
        uint8_t* row = dst + (u & 1) * kHalf + key * 128;
        *reinterpret_cast<uint4*>(row + (((2 * c4) ^ kr) << 4)) = lo;
        *reinterpret_cast<uint4*>(row + (((2 * c4 + 1) ^ kr) << 4)) = hi;
      }
      fence_proxy_async_smem();
    };
    uint4 kreg[8], vreg[8];
    if (n > 0) {
      load(a.k_pages, 0, kreg);
      load(a.v_pages, 0, vreg);
    }
    for (int j = 0; j < n; ++j) {
      const int s = j % kRowStages;
      const uint32_t phase = ((j / kRowStages) & 1) ^ 1;
      if (!mbar_wait_role(&sh->k_empty[s], phase, abort_flag, a.status, kDevTimeoutKV)) break;
      store(sK + s * kTile16, kreg);
      mbar_arrive(&sh->k_full[s]);
      if (j + 1 < n) load(a.k_pages, j + 1, kreg);
      if (!mbar_wait_role(&sh->v_empty[s], phase, abort_flag, a.status, kDevTimeoutKV)) break;
      store(sV + s * kTile16, vreg);
      mbar_arrive(&sh->v_full[s]);
      if (j + 1 < n) load(a.v_pages, j + 1, vreg);
    }
  } else {
    // ------------------------------------------------------------ softmax warps
    reg_alloc<kRegSoftmax>();
    const int t = warp >> 2, quarter = warp & 3, rl = quarter * 32 + lane;
    const uint32_t lane_off = uint32_t(quarter * 32) << 16;
    const uint32_t tS = tmem + 128 * t + lane_off, tO = tmem + 256 + 128 * t + lane_off;
    const int row = tile * kManyTile + t * 128 + rl, qi = row / a.group, head = h * a.group + (row - qi * a.group);
    const bool on = qi < tk.qn;
    const uint16_t* qrow = on ? static_cast<const uint16_t*>(a.q) + b * a.sq[0] + qi * a.sq[1] + head * a.sq[2] : nullptr;
    const float unit = stage_query<kDt>(qrow, sQ + t * kTile16, rl) * a.score_log2;
    fence_proxy_async_smem();
    mbar_arrive(&sh->q_full);
    const int64_t limit = (!on ? -1 : (a.causal ? tk.kv - tk.qn + qi : tk.kv - 1)) - int64_t(p0) * kPageTokens;
    float m = -INFINITY, l = 0.f;
    auto scales = [&](int j) {
      TileScale x;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int64_t id = page_id(2 * j + e, x.ok[e]);
        // kept above 0 (a written page's are at least 2^-40): a masked score is -inf times ka, and va is divided by
        x.ka[e] = x.ok[e] ? fmaxf(a.ka[id * a.heads + h], kTinyScale) : 1.f;
        x.va[e] = x.ok[e] ? fmaxf(a.va[id * a.heads + h], kTinyScale) : 1.f;
      }
      return x;
    };
    TileScale next{};
    if (n > 0) next = scales(0);
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      const TileScale sc = next;
      if (j + 1 < n) next = scales(j + 1);
      if (!(ok = mbar_wait(&sh->s_full[t], j & 1, abort_flag, a.status, kDevTimeoutS))) break;
      tc_fence_after();
      uint32_t sv[128];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(tS + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&sv[32 * c]));
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        auto& part = *reinterpret_cast<uint32_t(*)[32]>(&sv[32 * c]);
        if (c == 0) tmem_ld_wait(part);
        else reg_anchor(part);
      }
      auto F = [&](int i) { return __uint_as_float(sv[i]); };
      const int64_t rest = limit - int64_t(j) * 128;      // last visible key of the tile
      if (!__all_sync(0xffffffffu, rest >= 127 && sc.ok[0] && sc.ok[1])) {
        const int last0 = sc.ok[0] ? int(rest < 64 ? rest : 63) : -1, last1 = sc.ok[1] ? int(rest < 128 ? rest : 127) : -1;
#pragma unroll
        for (int i = 0; i < 128; ++i)
          if (i > (i < 64 ? last0 : last1)) sv[i] = 0xff800000u;
      }
      float r[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) r[q] = fmaxf(F(64 * (q >> 2) + 2 * (q & 3)), F(64 * (q >> 2) + 2 * (q & 3) + 1));
#pragma unroll
      for (int i = 8; i < 64; i += 8) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          r[q] = fmax3(r[q], F(i + 2 * q), F(i + 2 * q + 1));
          r[4 + q] = fmax3(r[4 + q], F(64 + i + 2 * q), F(64 + i + 2 * q + 1));
        }
      }
      const float c0 = sc.ka[0] * unit, c1 = sc.ka[1] * unit;
      const float lv0 = __log2f(sc.va[0]), lv1 = __log2f(sc.va[1]);
      const float x0 = fmax3(r[0], r[1], fmaxf(r[2], r[3])), x1 = fmax3(r[4], r[5], fmaxf(r[6], r[7]));
      const float top = fmaxf(fmaf(x0, c0, lv0), fmaf(x1, c1, lv1));
      const bool grow = top > m + kSlack;                 // also from m = -inf
      if (__any_sync(0xffffffffu, grow)) {
        const float alpha = grow ? ex2_approx(m - top) : 1.f;
        if (grow) m = top;
        l *= alpha;
        if (j > 0) {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t ov[32];
            tmem_ld32(tO + 32 * c, ov);
            tmem_ld_wait(ov);
#pragma unroll
            for (int e = 0; e < 32; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
            tmem_st32(tO + 32 * c, ov);
          }
        }
      }
      const float ref = (m == -INFINITY ? 0.f : m) - kWeightBits;
      const uint64_t cc[2] = {f2_pack(c0, c0), f2_pack(c1, c1)};
      const uint64_t bb[2] = {f2_pack(lv0 - ref, lv0 - ref), f2_pack(lv1 - ref, lv1 - ref)};
      uint64_t acc[4] = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < 64; ++i) {
        const int e = i >> 5;
        float w0, w1;
        f2_unpack(f2_fma(f2_pack(F(2 * i), F(2 * i + 1)), cc[e], bb[e]), w0, w1);
        w0 = ex2_approx(w0);
        w1 = ex2_approx(w1);
        acc[2 * e + (i & 1)] = f2_add(acc[2 * e + (i & 1)], f2_pack(w0, w1));
        sv[i] = pack_act2(w0, w1, 1);
      }
      tmem_st32(tS, *reinterpret_cast<uint32_t(*)[32]>(&sv[0]));
      tmem_st32(tS + 32, *reinterpret_cast<uint32_t(*)[32]>(&sv[32]));
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&sh->p_full[t]);
      float s[8];
#pragma unroll
      for (int q = 0; q < 4; ++q) f2_unpack(acc[q], s[2 * q], s[2 * q + 1]);
      l += __fdividef((s[0] + s[1]) + (s[2] + s[3]), sc.va[0]) + __fdividef((s[4] + s[5]) + (s[6] + s[7]), sc.va[1]);
    }
    if (ok && n > 0) ok = mbar_wait(&sh->o_done[t], (n - 1) & 1, abort_flag, a.status, kDevTimeoutO);
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
  paged_rows_kernel<kFmt, kDt><<<dim3(unsigned(a.heads) * a.tiles, a.splits, a.batch), kRowThreads, kRowsSmem, st>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_paged_rows(const PagedAttnArgs& a, cudaStream_t st) {
  if (a.fmt) return a.dtype ? launch_rows_as<1, 1>(a, st) : launch_rows_as<1, 0>(a, st);
  return a.dtype ? launch_rows_as<0, 1>(a, st) : launch_rows_as<0, 0>(a, st);
}

}  // namespace lbq
