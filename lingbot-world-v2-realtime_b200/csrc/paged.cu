// Paged 8-bit KV cache, sm_100a: the quantizing write, the read-back of a window, and page copies (layout and
// formulas in lbq_paged.h).
//
// Write. For a page and head that new tokens x enter: a = max(amax of the tokens it already holds, max finite |x|,
// 2^-40); held codes c become rnd(c * a_old / a) when a grew, new tokens rnd(x * Q / a) (rnd: round half to even for
// int8, round to nearest for e4m3); infinities become +-Q and NaN 0, so a cache never holds a non-finite value.
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

#include "lbq_kernels.h"
#include "lbq_paged.h"
#include "lbq_ptx.cuh"

namespace lbq {

// Page of block `blk` of sequence b, or -1 (recording the status) when the table or the pool has no such page.
__device__ __forceinline__ int page_of(const PageTable& pt, int b, int64_t blk, int* status) {
  int id = -1;
  if (blk < pt.width) id = pt.table[b * pt.st_b + blk];
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

// Rotates the 8 channels 8 * c16 .. of one K row (rope.cu's arithmetic: products and sums rounded one by one, the
// result rounded to the activation type). `row`: the head's 128 channels in memory, for the half layout's partners.
template <int kDt>
__device__ __forceinline__ uint4 rope_row8(const uint4 raw, const uint16_t* row, int c16, const RopeTable& r,
                                           int64_t at) {
  float x[8];
  unpack_act8<kDt>(raw, x);
  const int ch = c16 * 8, half = r.rot / 2;
  if (r.interleaved) {
    const float4 c = *reinterpret_cast<const float4*>(r.cos + at * r.stride + ch / 2);
    const float4 s = *reinterpret_cast<const float4*>(r.sin + at * r.stride + ch / 2);
    const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p = x[2 * i], q = x[2 * i + 1];
      x[2 * i] = __fsub_rn(__fmul_rn(p, cc[i]), __fmul_rn(q, ss[i]));
      x[2 * i + 1] = __fadd_rn(__fmul_rn(p, ss[i]), __fmul_rn(q, cc[i]));
    }
  } else {
    const bool low = ch < half;
    const int k0 = low ? ch : ch - half;
    float o[8];
    unpack_act8<kDt>(*reinterpret_cast<const uint4*>(row + (low ? ch + half : ch - half)), o);
#pragma unroll
    for (int q4 = 0; q4 < 2; ++q4) {
      const float4 c = *reinterpret_cast<const float4*>(r.cos + at * r.stride + k0 + 4 * q4);
      const float4 s = *reinterpret_cast<const float4*>(r.sin + at * r.stride + k0 + 4 * q4);
      const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = 4 * q4 + i;
        x[j] = low ? __fsub_rn(__fmul_rn(x[j], cc[i]), __fmul_rn(o[j], ss[i]))
                   : __fadd_rn(__fmul_rn(o[j], ss[i]), __fmul_rn(x[j], cc[i]));
      }
    }
  }
  return pack_act8<kDt>(x);
}

// The codes of one thread's rows by IEEE divisions, for any scale and any value; kept out of line, away from the
// registers and the instruction stream of the usual path.
template <int kFmt, int kDt>
__device__ __noinline__ void general_codes(const uint4 (&raw)[4], uint8_t* codes, int rg, int c16, int lo, int hi, float amax,
                                           float old) {
  constexpr float kQ = kFmt ? 448.f : 127.f;
  // both operands scaled by 2^-64 where x * Q could overflow
  const float f = amax > 1.8446744073709552e19f ? 5.421010862427522e-20f : 1.f;      // 2^64, 2^-64
#pragma unroll 1
  for (int i = 0; i < 4; ++i) {
    const int r = rg + 16 * i;
    uint2* dst = reinterpret_cast<uint2*>(codes + r * 128 + c16 * 8);
    float x[8];
    if (r >= lo && r < hi) {
      unpack_act8<kDt>(raw[i], x);
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

// One CTA per (touched page, head, sequence) and tensor (grid.x even: K, odd: V). 256 threads = 16 chunks of 8
// channels x 16 row groups; a thread takes rows rg + 16 i. The new rows stay in registers between the maximum and
// the codes, so each value is read once.
template <int kFmt, int kDt>
__global__ void __launch_bounds__(256) page_write_kernel(const PageWriteArgs a) {
  const int w = blockIdx.x & 1, h = blockIdx.y, b = blockIdx.z;
  const int t = threadIdx.x, c16 = t & 15, rg = t >> 4;
  const int64_t start = a.start ? a.start[b] : a.start0;
  int n = a.lens ? a.lens[b] : a.len;
  n = n < 0 ? 0 : (n > a.len ? a.len : n);
  const int64_t blk = start / kPageTokens + (blockIdx.x >> 1);
  const int64_t t0 = blk * kPageTokens;
  const int lo = int(start > t0 ? start - t0 : 0);                       // rows held before
  const int64_t end = start + n - t0;
  const int hi = int(end < kPageTokens ? end : kPageTokens);             // rows [lo, hi) are new
  if (start < 0) {
    if (a.status && t == 0) atomicCAS(a.status, 0, kDevBadPage);
    return;
  }
  if (hi <= lo) return;
  const int64_t* ss = a.ss[w];
  const uint16_t* src = static_cast<const uint16_t*>(a.src[w]) + b * ss[0] + h * ss[2];
  const bool rope = w == 0 && a.rope.cos != nullptr && c16 * 8 < a.rope.rot;
  // rows outside [lo, hi) load a neighbour's, so that no load waits for a branch, and count as 0
  uint4 raw[4];
  int64_t at[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t l = t0 + min(max(rg + 16 * i, lo), hi - 1) - start;
    raw[i] = *reinterpret_cast<const uint4*>(src + l * ss[1] + c16 * 8);
    at[i] = start + l;
    if (rope && a.rope.pos != nullptr) {
      const int64_t o = b * a.rope.sp_b + l * a.rope.sp_l;
      at[i] = a.rope.pos64 ? static_cast<const int64_t*>(a.rope.pos)[o] : static_cast<const int32_t*>(a.rope.pos)[o];
    }
  }
  const int page = page_of(a.pt, b, blk, a.status);
  if (page < 0) return;
  const int64_t ph = int64_t(page) * a.heads + h;
  uint8_t* codes = a.codes[w] + ph * kPageBytes;
  float* amax_p = a.amax[w] + ph;
  const float old = lo > 0 ? *amax_p : 0.f;
  if (rope) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool in = at[i] >= 0 && at[i] < a.rope.rows;
      if (!in && a.status) atomicCAS(a.status, 0, kDevBadPosition);
      const int64_t l = t0 + min(max(rg + 16 * i, lo), hi - 1) - start;
      const uint4 turned = rope_row8<kDt>(raw[i], src + l * ss[1], c16, a.rope, in ? at[i] : 0);
      if (in) raw[i] = turned;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (rg + 16 * i < lo || rg + 16 * i >= hi) raw[i] = make_uint4(0u, 0u, 0u, 0u);
  // largest magnitude, two values at a time: as bits, which order like the magnitudes
  uint32_t top2 = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    top2 = __vmaxu2(top2, __vmaxu2(__vmaxu2(raw[i].x & 0x7fff7fffu, raw[i].y & 0x7fff7fffu),
                                   __vmaxu2(raw[i].z & 0x7fff7fffu, raw[i].w & 0x7fff7fffu)));
  uint32_t top = __reduce_max_sync(0xffffffffu, max(top2 & 0xffffu, top2 >> 16));
  __shared__ uint32_t red[8];
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
    general_codes<kFmt, kDt>(raw, codes, rg, c16, lo, hi, amax, old);
    return;
  }
  const float r_new = __fdiv_rn(kQ, amax), r_old = __fdiv_rn(old, amax);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = rg + 16 * i;
    uint2* dst = reinterpret_cast<uint2*>(codes + r * 128 + c16 * 8);
    if (r >= lo && r < hi) {
      float x[8];
      unpack_act8<kDt>(raw[i], x);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = quotient(x[j], r_new);
      *dst = make_uint2(pack_codes<kFmt>(x[0], x[1], x[2], x[3]), pack_codes<kFmt>(x[4], x[5], x[6], x[7]));
    } else if (r < lo && amax > old) {
      const uint2 c = *dst;
      float x[4], y[4];
      unpack_codes<kFmt>(c.x, x);
      unpack_codes<kFmt>(c.y, y);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = quotient(x[j], r_old);
        y[j] = quotient(y[j], r_old);
      }
      *dst = make_uint2(pack_codes<kFmt>(x[0], x[1], x[2], x[3]), pack_codes<kFmt>(y[0], y[1], y[2], y[3]));
    }
  }
}

// One CTA per (64 tokens read, head, sequence), both tensors: 16 codes in, 16 values (two 16-byte stores) out a thread,
// row and tensor, two rows a thread, all loads before the first store.
template <int kFmt, int kDt>
__global__ void __launch_bounds__(256) page_read_kernel(const PageReadArgs a) {
  const int h = blockIdx.y, b = blockIdx.z;
  const int t = threadIdx.x, c8 = t & 7, rg = t >> 3;
  const int64_t start = a.start ? a.start[b] : a.start0;
  int n = a.lens ? a.lens[b] : a.len;
  n = n < 0 ? 0 : (n > a.len ? a.len : n);
  if (start < 0) {
    if (a.status && t == 0) atomicCAS(a.status, 0, kDevBadPage);
    n = 0;
  }
  uint4 c[2][2];
  float unit[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t l = int64_t(blockIdx.x) * 64 + rg + 32 * i;
    int page = -1;
    const int64_t tok = start + l;
    if (l < n) page = page_of(a.pt, b, tok / kPageTokens, a.status);
    const int64_t ph = int64_t(page < 0 ? 0 : page) * a.heads + h;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      c[i][w] = make_uint4(0u, 0u, 0u, 0u);
      unit[i][w] = 0.f;
      if (page >= 0) {
        c[i][w] = *reinterpret_cast<const uint4*>(a.codes[w] + ph * kPageBytes + (tok % kPageTokens) * 128 + c8 * 16);
        unit[i][w] = a.amax[w][ph];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t l = int64_t(blockIdx.x) * 64 + rg + 32 * i;
    if (l >= a.len) break;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const float u = __fdiv_rn(unit[i][w], kFmt ? 448.f : 127.f);
      const uint32_t q[4] = {c[i][w].x, c[i][w].y, c[i][w].z, c[i][w].w};
      uint32_t v[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float f[4];
        unpack_codes<kFmt>(q[k], f);
        v[2 * k] = pack_act2(f[0] * u, f[1] * u, kDt);
        v[2 * k + 1] = pack_act2(f[2] * u, f[3] * u, kDt);
      }
      uint16_t* dst = static_cast<uint16_t*>(a.dst[w]) + b * a.sd[w][0] + l * a.sd[w][1] + h * a.sd[w][2] + c8 * 16;
      reinterpret_cast<uint4*>(dst)[0] = make_uint4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<uint4*>(dst)[1] = make_uint4(v[4], v[5], v[6], v[7]);
    }
  }
}

// Copies whole pages (all heads, both tensors, amax) of every layer. grid: (16 KB pieces of a page, pair, layer * 2 +
// tensor); the pair list travels in the parameters, so nothing is read before the data.
__global__ void __launch_bounds__(256) page_copy_kernel(const __grid_constant__ PageCopyArgs a) {
  const int w = blockIdx.z & 1, layer = blockIdx.z >> 1;
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
  auto kern = a.fmt ? (a.dtype ? page_write_kernel<1, 1> : page_write_kernel<1, 0>)
                    : (a.dtype ? page_write_kernel<0, 1> : page_write_kernel<0, 0>);
  kern<<<grid, 256, 0, st>>>(a);
  return cudaGetLastError();
}
cudaError_t launch_page_read(const PageReadArgs& a, cudaStream_t st) {
  const dim3 grid(unsigned((a.len + 63) / 64), a.heads, a.batch);
  auto kern = a.fmt ? (a.dtype ? page_read_kernel<1, 1> : page_read_kernel<1, 0>)
                    : (a.dtype ? page_read_kernel<0, 1> : page_read_kernel<0, 0>);
  kern<<<grid, 256, 0, st>>>(a);
  return cudaGetLastError();
}
cudaError_t launch_page_copy(const PageCopyArgs& a, cudaStream_t st) {
  const dim3 grid(unsigned((int64_t(a.heads) * kPageBytes / 16 + 1023) / 1024), a.pairs, a.layers * 2);
  page_copy_kernel<<<grid, 256, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace lbq
