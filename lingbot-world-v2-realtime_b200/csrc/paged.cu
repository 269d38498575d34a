// Paged 8-bit KV cache, sm_100a: the quantizing write, the read-back of a window, and page copies (layout and
// formulas in lbq_paged.h).
//
// Write. For a page and head that new tokens x enter: a = max(a_old, max finite |x|, 2^-40), where a_old is the page's stored
// amax if it holds tokens before the new ones, else 0 (so it keeps the magnitude of tokens that are replaced now: what was
// rounded to their scale cannot be had back); held codes c become rnd(c * a_old / a) when a grew, new tokens rnd(x * Q / a)
// (rnd: round half to even for int8, round to nearest for e4m3); infinities become +-Q and NaN 0, so a cache never holds a
// non-finite value.
//
// The codes are those of exact arithmetic, without a division a value. x and a have at most 11 significant bits, a code
// at most 7, so a quotient V = x Q / a or c a_old / a is either exactly half way between two codes, or off it by at least
// V / (127 * 2047) or 1 / (2 * 2047) (numerators are integers), which for |V| < 128 is at least 16 units in the last
// place of an fp32 V; for e4m3, with 31 * 2047 in place of 127 * 2047, more. V computed as x * fl(Q / a) is off by at
// most 2 such units. Rounded to a multiple of 16 units, a half way case, which has 9 significant bits at most, becomes
// exact again, and any other stays on its side. A pool that was filled by other means may hold an amax with more bits:
// its pages take an IEEE division a value, which decides alike but within 2^-24 of a border. (On 6032 tokens x 12 heads
// the division a value cost 28 us a write.)
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>
#include <type_traits>

#include "lbq_kernels.h"
#include "lbq_paged.h"
#include "lbq_paged.cuh"
#include "lbq_ptx.cuh"

namespace lbq {

// Page of block `blk` of sequence b, or -1 (recording the status) when the table or the pool has no such page.
__device__ __forceinline__ int page_of(const PageTable& pt, int b, int64_t blk, int* status) {
  int id = -1;
  if (uint64_t(blk) < uint64_t(pt.width)) id = pt.table[b * pt.st_b + blk];
  if (id < 0 || id >= pt.num_pages) {
    if (status) atomicCAS(status, 0, kDevBadPage);
    return -1;
  }
  return id;
}

// Four values in [-127.5, 127.5] to int8 codes, round half to even, packed: adding 1.5 * 2^23 leaves the integer's
// two's-complement byte in the low mantissa bits.
__device__ __forceinline__ uint32_t pack_s8x4(float a, float b, float c, float d) {
  const uint32_t ua = __float_as_uint(__fadd_rn(a, 12582912.f)), ub = __float_as_uint(__fadd_rn(b, 12582912.f));
  const uint32_t uc = __float_as_uint(__fadd_rn(c, 12582912.f)), ud = __float_as_uint(__fadd_rn(d, 12582912.f));
  return __byte_perm(__byte_perm(ua, ub, 0x0040), __byte_perm(uc, ud, 0x0040), 0x5410);
}
template <int kFmt>
__device__ __forceinline__ uint32_t pack_codes(float a, float b, float c, float d) {
  if constexpr (kFmt == 0) return pack_s8x4(a, b, c, d);
  else return pack_e4m3x2(a, b) | (pack_e4m3x2(c, d) << 16);
}
// Four codes as floats.
template <int kFmt>
__device__ __forceinline__ void unpack_codes(uint32_t w, float (&f)[4]) {
  if constexpr (kFmt == 0) {
    // the float 2^23 + (c + 128), then exactly less 2^23 + 128: two issues a code on full-rate pipes, none on the converter
    const uint32_t u = w ^ 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7540 + i)) - 8388736.f;
  } else {
    uint32_t h[2];
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h[0]) : "h"(uint16_t(w)));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h[1]) : "h"(uint16_t(w >> 16)));
    const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&h[0]));
    const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&h[1]));
    f[0] = lo.x; f[1] = lo.y; f[2] = hi.x; f[3] = hi.y;
  }
}

// x * r on the side of every code border that the exact quotient is on (see above).
__device__ __forceinline__ float quotient(float x, float r) {
  return __uint_as_float((__float_as_uint(__fmul_rn(x, r)) + 8u) & ~15u);
}

template <int kDt>
__device__ __forceinline__ void unpack_act8(const uint4 r, float (&f)[8]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) act2_to_f32(w[i], kDt, f[2 * i], f[2 * i + 1]);
}
template <int kDt>
__device__ __forceinline__ uint4 pack_act8(const float (&f)[8]) {
  return make_uint4(pack_act2(f[0], f[1], kDt), pack_act2(f[2], f[3], kDt), pack_act2(f[4], f[5], kDt),
                    pack_act2(f[6], f[7], kDt));
}

// One thread's part of a table row: the cosines and sines of its 8 channels (4 pairs of neighbours, or 8 pairs whose other
// half another thread holds).
template <int kRope>
struct Turn {
  static constexpr int kN = kRope == 2 ? 8 : 4;
  float4 c[kN / 4], s[kN / 4];
  __device__ __forceinline__ void load(const float* cs, const float* sn) {
#pragma unroll
    for (int i = 0; i < kN / 4; ++i) {
      c[i] = reinterpret_cast<const float4*>(cs)[i];
      s[i] = reinterpret_cast<const float4*>(sn)[i];
    }
  }
};
// Rotates 8 channels (rope.cu's arithmetic: products and sums rounded one by one, the result rounded to the activation
// type). `other`: the same channels of the pairs' other half, `low`: x is the first half (half layout).
template <int kDt, int kRope>
__device__ __forceinline__ uint4 rotate8(const uint4 raw, const uint4 other, bool low, const Turn<kRope>& t) {
  float x[8];
  unpack_act8<kDt>(raw, x);
  if constexpr (kRope == 1) {
    const float c[4] = {t.c[0].x, t.c[0].y, t.c[0].z, t.c[0].w}, s[4] = {t.s[0].x, t.s[0].y, t.s[0].z, t.s[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p = x[2 * i], q = x[2 * i + 1];
      x[2 * i] = __fsub_rn(__fmul_rn(p, c[i]), __fmul_rn(q, s[i]));
      x[2 * i + 1] = __fadd_rn(__fmul_rn(p, s[i]), __fmul_rn(q, c[i]));
    }
  } else {
    float o[8];
    unpack_act8<kDt>(other, o);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 cv = t.c[i >> 2], sv = t.s[i >> 2];
      const float c = (i & 3) == 0 ? cv.x : (i & 3) == 1 ? cv.y : (i & 3) == 2 ? cv.z : cv.w;
      const float s = (i & 3) == 0 ? sv.x : (i & 3) == 1 ? sv.y : (i & 3) == 2 ? sv.z : sv.w;
      // the first half x c - o s, the second o s + x c: one sign apart, and a sum of two products commutes
      const float os = __fmul_rn(o[i], s);
      x[i] = __fadd_rn(__fmul_rn(x[i], c), low ? -os : os);
    }
  }
  return pack_act8<kDt>(x);
}

// The codes of one thread's rows by IEEE divisions, for any scale and any value; kept out of line, away from the
// registers and the instruction stream of the usual path (and given its rows by value: a reference would put them in local
// memory, 64 bytes a thread written and read for nothing).
template <int kFmt, int kDt>
__device__ __noinline__ void general_codes(uint4 r0, uint4 r1, uint4 r2, uint4 r3, uint8_t* codes, int rg, int c16, int lo,
                                           int hi, float amax, float old) {
  constexpr float kQ = kFmt ? 448.f : 127.f;
  // both operands scaled by 2^-64 where x * Q could overflow
  const float f = amax > 1.8446744073709552e19f ? 5.421010862427522e-20f : 1.f;      // 2^64, 2^-64
#pragma unroll 1
  for (int i = 0; i < 4; ++i) {
    const int r = rg + 16 * i;
    uint2* dst = reinterpret_cast<uint2*>(codes + r * 128 + c16 * 8);
    float x[8];
    if (r >= lo && r < hi) {
      unpack_act8<kDt>(i == 0 ? r0 : i == 1 ? r1 : i == 2 ? r2 : r3, x);
      for (int j = 0; j < 8; ++j) {
        const float v = x[j] != x[j] ? 0.f : fminf(fmaxf(x[j], -amax), amax);
        x[j] = __fdiv_rn(__fmul_rn(v, f * kQ), amax * f);
      }
    } else if (r < lo && amax > old) {
      const uint2 c = *dst;
      float y[4], z[4];
      unpack_codes<kFmt>(c.x, y);
      unpack_codes<kFmt>(c.y, z);
      for (int j = 0; j < 4; ++j) {
        x[j] = __fdiv_rn(__fmul_rn(y[j], old * f), amax * f);
        x[4 + j] = __fdiv_rn(__fmul_rn(z[j], old * f), amax * f);
      }
    } else {
      continue;
    }
    *dst = make_uint2(pack_codes<kFmt>(x[0], x[1], x[2], x[3]), pack_codes<kFmt>(x[4], x[5], x[6], x[7]));
  }
}

// One CTA per (touched page, head, sequence) and tensor. 256 threads = 16 chunks of 8 channels x 16 row groups; a thread
// takes rows rg + 16 i. The new rows stay in registers between the maximum and the codes, so each value is read once; all
// loads go out before the page is looked up.
template <int kFmt, int kDt, int kRope>
__device__ __forceinline__ void write_page(const PageWriteArgs& a, const int w, uint32_t* red) {
  const int h = blockIdx.y, b = blockIdx.z;
  const int t = threadIdx.x, c16 = t & 15, rg = t >> 4;
  const int64_t start = a.start ? a.start[b] : a.start0;
  int n = a.lens ? a.lens[b] : a.len;
  if (start < 0 || n < 0 || n > a.len) {
    if (a.status && t == 0) atomicCAS(a.status, 0, kDevBadPage);
    if (start < 0 || n < 0) return;
    n = a.len;
  }
  const int off = int(start % kPageTokens);                              // the first touched page's held rows
  const int l0 = int(blockIdx.x >> 1) * kPageTokens - off;               // source row of this page's row 0
  const int lo = l0 < 0 ? -l0 : 0, hi = min(n - l0, kPageTokens);        // rows [lo, hi) are new
  if (hi <= lo) return;
  const int64_t blk = start / kPageTokens + (blockIdx.x >> 1);
  const int64_t sl = a.ss[w][1];
  const uint16_t* src = static_cast<const uint16_t*>(a.src[w]) + b * a.ss[w][0] + h * a.ss[w][2] + (l0 + rg) * sl + c16 * 8;
  uint4 raw[4];
  bool on[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    on[i] = rg + 16 * i >= lo && rg + 16 * i < hi;
    raw[i] = make_uint4(0u, 0u, 0u, 0u);
    if (on[i]) raw[i] = *reinterpret_cast<const uint4*>(src + 16 * i * sl);
  }
  const int page = page_of(a.pt, b, blk, a.status);
  if constexpr (kRope != 0) {
    if (c16 * 8 < a.rope.rot) {
      const int half = a.rope.rot / 2, ch = c16 * 8;
      const bool low = kRope == 1 || ch < half;
      const int col = kRope == 1 ? ch / 2 : (low ? ch : ch - half);
#pragma unroll
      for (int i2 = 0; i2 < 4; i2 += 2) {                                // two rows at a time
        Turn<kRope> turn[2];
        uint4 other[2];
        bool in[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int i = i2 + k, l = l0 + rg + 16 * i;
          int64_t at = start + l;
          in[k] = false;
          if (on[i]) {
            if (a.rope.pos != nullptr) {
              const int64_t o = b * a.rope.sp_b + l * a.rope.sp_l;
              at = a.rope.pos64 ? static_cast<const int64_t*>(a.rope.pos)[o] : static_cast<const int32_t*>(a.rope.pos)[o];
            }
            in[k] = at >= 0 && at < a.rope.rows;
            if (!in[k] && a.status) atomicCAS(a.status, 0, kDevBadPosition);
          }
          if (in[k]) {
            turn[k].load(a.rope.cos + at * a.rope.stride + col, a.rope.sin + at * a.rope.stride + col);
            if (kRope == 2) other[k] = *reinterpret_cast<const uint4*>(src + 16 * i * sl + (low ? half : -half));
          }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k)
          if (in[k]) raw[i2 + k] = rotate8<kDt, kRope>(raw[i2 + k], other[k], low, turn[k]);
      }
    }
  }
  if (page < 0) return;
  const int64_t ph = int64_t(page) * a.heads + h;
  uint8_t* codes = a.codes[w] + ph * kPageBytes;
  float* amax_p = a.amax[w] + ph;
  const float old = lo > 0 ? *amax_p : 0.f;
  // largest magnitude, two values at a time: as bits, which order like the magnitudes
  uint32_t top2 = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    top2 = __vmaxu2(top2, __vmaxu2(__vmaxu2(raw[i].x & 0x7fff7fffu, raw[i].y & 0x7fff7fffu),
                                   __vmaxu2(raw[i].z & 0x7fff7fffu, raw[i].w & 0x7fff7fffu)));
  uint32_t top = __reduce_max_sync(0xffffffffu, max(top2 & 0xffffu, top2 >> 16));
  if ((t & 31) == 0) red[t >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, red[i]);
  const bool odd = top >= (kDt ? 0x7c00u : 0x7f80u);                     // an infinity or a NaN among them
  if (odd) {                                                             // uniform over the CTA: the finite ones' maximum
    top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t m = (v[j >> 1] >> (16 * (j & 1))) & 0x7fffu;
        top = max(top, m < (kDt ? 0x7c00u : 0x7f80u) ? m : 0u);
      }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    __syncthreads();
    if ((t & 31) == 0) red[t >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, red[i]);
  }
  float amax, unused;
  act2_to_f32(top, kDt, amax, unused);
  amax = fmaxf(fmaxf(amax, old), kAmaxFloor);
  if (t == 0) *amax_p = amax;
  constexpr float kQ = kFmt ? 448.f : 127.f;
  // more than 11 significant bits in a scale, or values that are not finite: the general path
  const bool wide = ((__float_as_uint(amax) | __float_as_uint(old)) & 0x1fffu) != 0;
  if (wide || odd) {
    general_codes<kFmt, kDt>(raw[0], raw[1], raw[2], raw[3], codes, rg, c16, lo, hi, amax, old);
    return;
  }
  const float r_new = __fdiv_rn(kQ, amax);
  uint2* dst = reinterpret_cast<uint2*>(codes + rg * 128 + c16 * 8);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (on[i]) {
      float x[8];
      unpack_act8<kDt>(raw[i], x);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = quotient(x[j], r_new);
      dst[256 * i] = make_uint2(pack_codes<kFmt>(x[0], x[1], x[2], x[3]), pack_codes<kFmt>(x[4], x[5], x[6], x[7]));
    }
  }
  if (lo > 0 && amax > old) {
    const float r_old = __fdiv_rn(old, amax);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (rg + 16 * i >= lo) break;
      const uint2 c = dst[256 * i];
      float x[4], y[4];
      unpack_codes<kFmt>(c.x, x);
      unpack_codes<kFmt>(c.y, y);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = quotient(x[j], r_old);
        y[j] = quotient(y[j], r_old);
      }
      dst[256 * i] = make_uint2(pack_codes<kFmt>(x[0], x[1], x[2], x[3]), pack_codes<kFmt>(y[0], y[1], y[2], y[3]));
    }
  }
}
template <int kFmt, int kDt, int kRope>
__global__ void __launch_bounds__(256) page_write_kernel(const __grid_constant__ PageWriteArgs a) {
  __shared__ uint32_t red[8];
  after_previous_grid();
  if (blockIdx.x & 1) write_page<kFmt, kDt, 0>(a, 1, red);
  else write_page<kFmt, kDt, kRope>(a, 0, red);
}

// One CTA per (64 tokens read, head, sequence), both tensors: 8 codes in, 8 values out a thread, row and tensor, so that a
// half warp writes a whole 256-byte row (16 codes a thread, as two 16-byte stores, would write every 32-byte sector twice);
// four rows a thread, all loads before the first store.
template <int kFmt, int kDt>
__global__ void __launch_bounds__(256) page_read_kernel(const __grid_constant__ PageReadArgs a) {
  const int h = blockIdx.y, b = blockIdx.z;
  const int t = threadIdx.x, c16 = t & 15, rg = t >> 4;
  after_previous_grid();
  const int64_t start = a.start ? a.start[b] : a.start0;
  int n = a.lens ? a.lens[b] : a.len;
  n = n < 0 ? 0 : (n > a.len ? a.len : n);
  if (start < 0) {
    if (a.status && t == 0) atomicCAS(a.status, 0, kDevBadPage);
    n = 0;
  }
  const int l0 = int(blockIdx.x) * 64 + rg;
  uint2 c[4][2];
  float unit[4][2];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int l = l0 + 16 * i;
    const int64_t tok = start + l;
    int page = -1;
    if (l < n) page = page_of(a.pt, b, tok / kPageTokens, a.status);
    const int64_t ph = int64_t(page < 0 ? 0 : page) * a.heads + h;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      c[i][w] = make_uint2(0u, 0u);
      unit[i][w] = 0.f;
      if (page >= 0) {
        c[i][w] = *reinterpret_cast<const uint2*>(a.codes[w] + ph * kPageBytes + int(tok % kPageTokens) * 128 + c16 * 8);
        unit[i][w] = a.amax[w][ph];
      }
    }
  }
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    uint16_t* dst = static_cast<uint16_t*>(a.dst[w]) + b * a.sd[w][0] + l0 * a.sd[w][1] + h * a.sd[w][2] + c16 * 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (l0 + 16 * i >= a.len) break;
      const float u = __fdiv_rn(unit[i][w], kFmt ? 448.f : 127.f);
      float lo[4], hi[4];
      unpack_codes<kFmt>(c[i][w].x, lo);
      unpack_codes<kFmt>(c[i][w].y, hi);
      const float x[8] = {lo[0] * u, lo[1] * u, lo[2] * u, lo[3] * u, hi[0] * u, hi[1] * u, hi[2] * u, hi[3] * u};
      *reinterpret_cast<uint4*>(dst + 16 * i * a.sd[w][1]) = pack_act8<kDt>(x);
    }
  }
}

// Copies whole pages (all heads, both tensors, amax) of every layer. grid: (16 KB pieces of a page, pair, layer * 2 +
// tensor); the pair list travels in the parameters, so nothing is read before the data.
__global__ void __launch_bounds__(256) page_copy_kernel(const __grid_constant__ PageCopyArgs a) {
  const int w = blockIdx.z & 1, layer = blockIdx.z >> 1;
  after_previous_grid();
  const int64_t page = int64_t(a.heads) * kPageBytes;
  const int64_t src = a.src[blockIdx.y], dst = a.dst[blockIdx.y];
  uint8_t* base = a.codes[w] + layer * a.layer_codes;
  const uint4* from = reinterpret_cast<const uint4*>(base + src * page);
  uint4* to = reinterpret_cast<uint4*>(base + dst * page);
  const int64_t n = page / 16;
  uint4 v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t o = int64_t(blockIdx.x) * 1024 + i * 256 + threadIdx.x;
    if (o < n) v[i] = from[o];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t o = int64_t(blockIdx.x) * 1024 + i * 256 + threadIdx.x;
    if (o < n) to[o] = v[i];
  }
  if (blockIdx.x == 0) {
    float* am = a.amax[w] + layer * a.layer_amax;
    for (int h = threadIdx.x; h < a.heads; h += 256) am[dst * a.heads + h] = am[src * a.heads + h];
  }
}

// ------------------------------------------------------------------ launchers
cudaError_t launch_page_write(const PageWriteArgs& a, cudaStream_t st) {
  // tokens of a sequence lie in at most (len + 62) / 64 + 1 pages
  const dim3 grid(unsigned((a.len + 62) / 64 + 1) * 2, a.heads, a.batch);
  const int rope = a.rope.cos == nullptr ? 0 : (a.rope.interleaved ? 1 : 2);
  auto pick = [&](auto fmt, auto dt) {
    constexpr int kF = decltype(fmt)::value, kD = decltype(dt)::value;
    return rope == 0 ? page_write_kernel<kF, kD, 0> : (rope == 1 ? page_write_kernel<kF, kD, 1> : page_write_kernel<kF, kD, 2>);
  };
  using Zero = std::integral_constant<int, 0>;
  using One = std::integral_constant<int, 1>;
  auto kern = a.fmt ? (a.dtype ? pick(One{}, One{}) : pick(One{}, Zero{})) : (a.dtype ? pick(Zero{}, One{}) : pick(Zero{}, Zero{}));
  return launch_after(kern, grid, dim3(256), 0, st, a);
}
cudaError_t launch_page_read(const PageReadArgs& a, cudaStream_t st) {
  const dim3 grid(unsigned((a.len + 63) / 64), a.heads, a.batch);
  auto kern = a.fmt ? (a.dtype ? page_read_kernel<1, 1> : page_read_kernel<1, 0>)
                    : (a.dtype ? page_read_kernel<0, 1> : page_read_kernel<0, 0>);
  return launch_after(kern, grid, dim3(256), 0, st, a);
}
cudaError_t launch_page_copy(const PageCopyArgs& a, cudaStream_t st) {
  const dim3 grid(unsigned((int64_t(a.heads) * kPageBytes / 16 + 1023) / 1024), a.pairs, a.layers * 2);
  return launch_after(page_copy_kernel, grid, dim3(256), 0, st, a);
}

}  // namespace lbq
