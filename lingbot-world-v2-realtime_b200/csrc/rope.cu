// Rotary positions for sm_100a: (x0, x1) -> (x0 c - x1 s, x0 s + x1 c) for the pairs of the first `rot` channels of
// every head, (2i, 2i + 1) (interleaved) or (i, i + rot / 2) (half), with c, s = row pos of the fp32 tables. Products
// and sums are rounded one by one in fp32 (no fma), then once to the tensor's type, so that the page write's fused
// rotation and a product-by-product evaluation give the same bits. The inverse rotation (s -> -s) is also the
// gradient: a rotation's transpose.
//
// Bound by memory: 2 x 2 bytes an element and 4 bytes a table entry against 1.5 flops. One CTA per token: a thread
// keeps the c, s of its channels in registers and walks the heads of both tensors, so a table row is read once a
// token, not once a head.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "lbq_kernels.h"
#include "lbq_paged.h"
#include "lbq_ptx.cuh"

namespace lbq {

template <int kDt> struct ActType { using T = uint16_t; };
template <> struct ActType<2> { using T = float; };

template <int kDt>
__device__ __forceinline__ float act_load(const typename ActType<kDt>::T* p) {
  if constexpr (kDt == 2) return *p;
  else if constexpr (kDt == 1) return __half2float(__ushort_as_half(*p));
  else return __uint_as_float(uint32_t(*p) << 16);
}
template <int kDt>
__device__ __forceinline__ void act_store(typename ActType<kDt>::T* p, float v) {
  if constexpr (kDt == 2) *p = v;
  else if constexpr (kDt == 1) *p = __half_as_ushort(__float2half_rn(v));
  else *p = __bfloat16_as_ushort(__float2bfloat16_rn(v));
}

// kN consecutive channels; 16-byte accesses where kN of them fill 16 bytes.
template <int kDt, int kN>
__device__ __forceinline__ void load_n(const typename ActType<kDt>::T* p, float (&f)[kN]) {
  if constexpr (kN * sizeof(typename ActType<kDt>::T) == 16) {
    const uint4 r = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
    if constexpr (kDt == 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) act2_to_f32(w[i], kDt, f[2 * i], f[2 * i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kN; ++i) f[i] = act_load<kDt>(p + i);
  }
}
template <int kDt, int kN>
__device__ __forceinline__ void store_n(typename ActType<kDt>::T* p, const float (&f)[kN]) {
  if constexpr (kN * sizeof(typename ActType<kDt>::T) == 16) {
    uint32_t w[4];
    if constexpr (kDt == 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(f[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = pack_act2(f[2 * i], f[2 * i + 1], kDt);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < kN; ++i) act_store<kDt>(p + i, f[i]);
  }
}

constexpr int kBatch = 2;

// Block (units, heads in flight): unit u of a head is kN channels (interleaved) or kN pairs (half) of the rotated
// part, or kN channels of the rest, which is copied unless the call is in place.
template <int kDt, bool kInter, int kN>
__global__ void rope_kernel(const RopeArgs a) {
  using T = typename ActType<kDt>::T;
  const int u = threadIdx.x;
  const int b = int(blockIdx.x / a.len), l = int(blockIdx.x - int64_t(b) * a.len);
  const int rot_units = kInter ? a.rope.rot / kN : a.rope.rot / (2 * kN);
  bool turn = u < rot_units;
  constexpr int kPairs = kInter ? kN / 2 : kN;
  float c[kPairs], s[kPairs];
#pragma unroll
  for (int i = 0; i < kPairs; ++i) { c[i] = 1.f; s[i] = 0.f; }
  if (turn) {
    int64_t row = a.start + l;
    if (a.rope.pos != nullptr) {
      const int64_t at = b * a.rope.sp_b + l * a.rope.sp_l;
      row = a.rope.pos64 ? static_cast<const int64_t*>(a.rope.pos)[at] : static_cast<const int32_t*>(a.rope.pos)[at];
    }
    if (row >= 0 && row < a.rope.rows) {
      const float* cp = a.rope.cos + row * a.rope.stride + u * kPairs;
      const float* sp = a.rope.sin + row * a.rope.stride + u * kPairs;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        c[i] = cp[i];
        s[i] = a.inverse ? -sp[i] : sp[i];
      }
    } else {
      if (u == 0 && threadIdx.y == 0 && a.status) atomicCAS(a.status, 0, kDevBadPosition);
    }
  }
  const int heads = a.heads[0] + a.heads[1];
  const int ch = turn ? u * kN : a.rope.rot + (u - rot_units) * kN;
  // kBatch heads at a time, all their loads first: one head a thread leaves too few bytes in flight (4.5 TB/s on 6032
  // tokens of 24 heads)
  for (int h0 = threadIdx.y; h0 < heads; h0 += kBatch * blockDim.y) {
    const T* x[kBatch];
    T* y[kBatch];
    float f[kBatch][kN], g[kBatch][kInter ? 1 : kN];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int hh = h0 + k * blockDim.y;
      if (hh >= heads) break;
      const int w = hh >= a.heads[0];
      const int h = w ? hh - a.heads[0] : hh;
      x[k] = static_cast<const T*>(a.x[w]) + b * a.sx[w][0] + l * a.sx[w][1] + h * a.sx[w][2] + ch;
      y[k] = static_cast<T*>(a.y[w]) + b * a.sy[w][0] + l * a.sy[w][1] + h * a.sy[w][2] + ch;
      load_n<kDt, kN>(x[k], f[k]);
      if constexpr (!kInter) {
        if (turn) load_n<kDt, kN>(x[k] + a.rope.rot / 2, g[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (h0 + k * int(blockDim.y) >= heads) break;
      if (turn) {
        if constexpr (kInter) {
#pragma unroll
          for (int i = 0; i < kPairs; ++i) {
            const float p = f[k][2 * i], q = f[k][2 * i + 1];
            f[k][2 * i] = __fsub_rn(__fmul_rn(p, c[i]), __fmul_rn(q, s[i]));
            f[k][2 * i + 1] = __fadd_rn(__fmul_rn(p, s[i]), __fmul_rn(q, c[i]));
          }
        } else {
#pragma unroll
          for (int i = 0; i < kN; ++i) {
            const float p = f[k][i], q = g[k][i];
            f[k][i] = __fsub_rn(__fmul_rn(p, c[i]), __fmul_rn(q, s[i]));
            g[k][i] = __fadd_rn(__fmul_rn(p, s[i]), __fmul_rn(q, c[i]));
          }
          store_n<kDt, kN>(y[k] + a.rope.rot / 2, g[k]);
        }
      }
      store_n<kDt, kN>(y[k], f[k]);
    }
  }
}

template <int kDt, bool kInter, int kN>
cudaError_t launch_rope_as(const RopeArgs& a, cudaStream_t st) {
  const int units = (kInter ? a.rope.rot / kN : a.rope.rot / (2 * kN)) + (a.in_place ? 0 : (a.dim - a.rope.rot) / kN);
  const int heads = a.heads[0] + a.heads[1];
  int hy = units >= 256 ? 1 : 256 / units;
  if (hy > heads) hy = heads;
  const int per = (heads + hy - 1) / hy;
  hy = (heads + per - 1) / per;
  rope_kernel<kDt, kInter, kN><<<dim3(unsigned(int64_t(a.batch) * a.len)), dim3(units, hy), 0, st>>>(a);
  return cudaGetLastError();
}
template <int kDt>
cudaError_t launch_rope_dt(const RopeArgs& a, cudaStream_t st) {
  constexpr int kVec = kDt == 2 ? 4 : 8;
  if (a.rope.interleaved) return a.vec ? launch_rope_as<kDt, true, kVec>(a, st) : launch_rope_as<kDt, true, 2>(a, st);
  return a.vec ? launch_rope_as<kDt, false, kVec>(a, st) : launch_rope_as<kDt, false, 1>(a, st);
}
cudaError_t launch_rope(const RopeArgs& a, cudaStream_t st) {
  if (a.dtype == 2) return launch_rope_dt<2>(a, st);
  return a.dtype ? launch_rope_dt<1>(a, st) : launch_rope_dt<0>(a, st);
}

}  // namespace lbq
