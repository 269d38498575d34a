// Device pieces that the two attention kernels over the paged cache share.
#pragma once
#include <cuda_fp16.h>
#include <cstdint>

#include "lbq_paged.h"
#include "lbq_ptx.cuh"

namespace lbq {

// Start of every kernel of this family: nothing is read or written before the grid that it follows in its stream has
// ended; then the next launch may take its place on the GPU as SMs allow. They are launched with programmatic stream
// serialization (launch_after below), so the launch latency and the set-up of one overlap the run of the one before. Every
// thread comes through here, so that a grid never ends before the grids it follows, and when a grid starts all but the one
// directly before it have ended.
__device__ __forceinline__ void after_previous_grid() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

constexpr float kTinyScale = 5.421010862427522e-20f;   // 2^-64: scales are kept above it (a written page's are >= 2^-40)
constexpr float kMinFactor = 1.1754943508222875e-38f;  // 2^-126
// The factor of a row's scores of one page is page (its scale) * row (the power of two taken out of the row) * scale (softmax
// scale * log2 e / Q). Row and scale are multiplied first, with 2^6 moved from the page's part to theirs, so that the smallest
// rows keep 16 bits and the largest do not overflow. It never is 0, which times the -inf of a masked score would be NaN
// (scores stay below 2^33 in magnitude: at the smallest factor they are 0 to any precision).
__device__ __forceinline__ float row_factor(float row, float scale) { return fminf(row * (64.f * scale), 3.402823466e38f); }
__device__ __forceinline__ float score_factor(float page, float row) { return fmaxf(page * (1.f / 64.f) * row, kMinFactor); }
// The power of two that scales a bf16 query row of largest magnitude `top` (the bits of the fp32 value) to a maximum in
// [1, 2), and its inverse `up`. With the exponent field e that is 2^(127 - e); 2^(127 - 254) is no normal float: a maximum
// in [2, 4) there. A row of subnormals, 2^-126 at most, goes up by 2^127; non-finite rows go as they are.
__device__ __forceinline__ float row_scale(uint32_t top, float& up) {
  const uint32_t e = min(top >> 23, 253u);
  const bool finite = top < 0x7f800000u;
  up = !finite ? 1.f : e == 0 ? 5.877471754111438e-39f : __uint_as_float(e << 23);      // 2^-127
  return finite ? __uint_as_float((254u - e) << 23) : 1.f;
}
constexpr float kWeightBits = 7.f;               // weights are scaled by 2^7 ...
constexpr float kSlack = 8.f;                    // ... and the running maximum may lag by 2^8: below 2^15, fp16's range

// A page whose largest weight lies more than 2^kFaint below 2^kWeightBits adds nothing to o, but may hold most of the sum
// when its V are that much smaller (weights carry the scale of V, a page of zeros has 2^-40): its weights would underflow
// before the division by va. The binary exponent that they, and va, are raised by; `far` is the page's maximum less the
// row's. (400: the page's part of the sum is 0 then, and masked pages, top = -inf, stay finite.) While sums are taken they
// are scaled by 2^kSumBits, so that 1 / va (2^128 at most) is no subnormal.
constexpr float kFaint = 100.f;
constexpr float kSumBits = 8.f, kSumUnit = 1.f / 256.f;
__device__ __forceinline__ float faint_exponent(float far) { return fminf(fmaxf(-far - kFaint, 0.f), 400.f); }
// 2^(e / 2): l times it twice. 2^e alone can underflow where the maximum moves for a V scale and not for a score.
__device__ __forceinline__ float half_ex2(float e) { return ex2_approx(0.5f * e); }

// Keys [0, visible) are seen by some row of the tile; 0 when every row is empty or past the sequence's queries.
struct TileKeys {
  int64_t kv;
  int qn;
  int64_t visible;
};
__device__ __forceinline__ TileKeys tile_keys(const PagedAttnArgs& a, int b, int tile) {
  TileKeys t;
  const int64_t most = int64_t(a.pt.width) * kPageTokens;
  t.kv = a.kv_lens ? a.kv_lens[b] : a.kv_len0;
  t.qn = a.q_lens ? a.q_lens[b] : a.q_len;               // both loads before anything waits for one
  if ((t.kv < 0) | (t.kv > most) | (t.qn < 0) | (t.qn > a.q_len)) {
    if (a.status) atomicCAS(a.status, 0, kDevBadPage);
    t.kv = t.kv < 0 ? 0 : min(t.kv, most);
    t.qn = t.qn < 0 ? 0 : min(t.qn, a.q_len);
  }
  const int first = tile * a.tile_rows / a.group;                        // first and last query token of the tile
  const int last = min((tile * a.tile_rows + a.tile_rows - 1) / a.group, t.qn - 1);
  if (first > last) t.visible = 0;
  else t.visible = a.causal ? min(t.kv, max(t.kv - t.qn + last + 1, int64_t(0))) : t.kv;
  return t;
}

// Bytes (s0, s1) of r as a pair of fp16 values: int8 by the magic-number conversion (a byte put into the low mantissa bits of
// 1024 is 1024 + (c + 128), and the subtraction is exact), e4m3 by the converter.
template <int kFmt, int kS0, int kS1>
__device__ __forceinline__ uint32_t widen(uint32_t r) {
  uint32_t d;
  if constexpr (kFmt == 0) {
    const uint32_t p = __byte_perm(r, 0x64646464u, 0x4040 | kS0 | (kS1 << 8));
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&p), __half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
    d = *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const uint16_t p = uint16_t(__byte_perm(r, 0u, kS0 | (kS1 << 4)));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"(p));
  }
  return d;
}
template <int kFmt>
__device__ __forceinline__ uint32_t bias(uint32_t r) { return kFmt == 0 ? r ^ 0x80808080u : r; }

__device__ __forceinline__ float natural_lse(float m, float l) {
  return l > 0.f ? (m + __log2f(l)) * 0.6931471805599453f : (l == l ? -INFINITY : l);
}

template <class... Params, class... Args>
cudaError_t launch_after_clustered(void (*kernel)(Params...), dim3 cluster, dim3 grid, dim3 block, size_t smem,
                                   cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2] = {};
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = cluster.x;
  at[1].val.clusterDim.y = cluster.y;
  at[1].val.clusterDim.z = cluster.z;
  cfg.attrs = at;
  cfg.numAttrs = cluster.x * cluster.y * cluster.z > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, Params(args)...);
}

template <class... Params, class... Args>
cudaError_t launch_after(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args&&... args) {
  return launch_after_clustered(kernel, dim3(1), grid, block, smem, st, args...);
}

}  // namespace lbq
