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
#include "lbq_paged.cuh"
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

// kN table entries, in 16-byte pieces where the table allows.
template <int kN>
__device__ __forceinline__ void load_f32(const float* p, bool wide, float (&f)[kN]) {
  if constexpr (kN % 4 == 0) {
    if (wide) {
#pragma unroll
      for (int i = 0; i < kN; i += 4) {
        const float4 v = *reinterpret_cast<const float4*>(p + i);
        f[i] = v.x;
        f[i + 1] = v.y;
        f[i + 2] = v.z;
        f[i + 3] = v.w;
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < kN; ++i) f[i] = p[i];
}

// kN consecutive channels as they lie in memory: one 16-byte access where they fill it.
template <int kDt, int kN>
struct Piece {
  using T = typename ActType<kDt>::T;
  static constexpr bool kWide = kN * sizeof(T) == 16;
  uint4 raw;
  T each[kWide ? 1 : kN];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kWide) {
      raw = *reinterpret_cast<const uint4*>(p);
    } else {
#pragma unroll
      for (int i = 0; i < kN; ++i) each[i] = p[i];
    }
  }
  __device__ __forceinline__ void get(float (&f)[kN]) const {
    if constexpr (kWide) {
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
      if constexpr (kDt == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) act2_to_f32(w[i], kDt, f[2 * i], f[2 * i + 1]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kN; ++i) f[i] = act_load<kDt>(&each[i]);
    }
  }
  static __device__ __forceinline__ void store(T* p, const float (&f)[kN]) {
    if constexpr (kWide) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (kDt == 2) w[i] = __float_as_uint(f[i]);
        else w[i] = pack_act2(f[2 * i], f[2 * i + 1], kDt);
      }
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int i = 0; i < kN; ++i) act_store<kDt>(p + i, f[i]);
    }
  }
};

// Block (units, heads in flight) at grid (token, sequence): unit u of a head is kN channels (interleaved) or kN pairs
// (half) of the rotated part, or kN channels of the rest, which is copied unless the call is in place. A thread takes
// every blockDim.y-th head of each tensor, two at a time: the loads of two heads of both tensors go out before the table
// row is there, and the addresses advance by one addition a head.
template <int kDt, bool kInter, int kN>
__global__ void __launch_bounds__(512) rope_kernel(const __grid_constant__ RopeArgs a) {
  using T = typename ActType<kDt>::T;
  constexpr int kPairs = kInter ? kN / 2 : kN;
  const int u = threadIdx.x, l = blockIdx.x, b = blockIdx.y;
  const int half = a.rope.rot / 2;
  const int rot_units = kInter ? a.rope.rot / kN : half / kN;
  const bool turn = u < rot_units;
  const int ch = turn ? u * kN : a.rope.rot + (u - rot_units) * kN;
  after_previous_grid();
  int64_t row = a.start + l;
  if (a.rope.pos != nullptr) {
    const int64_t at = b * a.rope.sp_b + l * a.rope.sp_l;
    row = a.rope.pos64 ? static_cast<const int64_t*>(a.rope.pos)[at] : static_cast<const int32_t*>(a.rope.pos)[at];
  }
  const T* x[2];
  T* y[2];
  int64_t dx[2], dy[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    x[w] = static_cast<const T*>(a.x[w]) + b * a.sx[w][0] + l * a.sx[w][1] + threadIdx.y * a.sx[w][2] + ch;
    y[w] = static_cast<T*>(a.y[w]) + b * a.sy[w][0] + l * a.sy[w][1] + threadIdx.y * a.sy[w][2] + ch;
    dx[w] = blockDim.y * a.sx[w][2];
    dy[w] = blockDim.y * a.sy[w][2];
  }
  using P = Piece<kDt, kN>;
  P f[2][2], g[2][2];                                    // g: the pairs' other halves (half layout)
  auto load = [&](int h0) {
#pragma unroll
    for (int w = 0; w < 2; ++w) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (h0 + k * int(blockDim.y) < a.heads[w]) {
          f[w][k].load(x[w] + k * dx[w]);
          if constexpr (!kInter) {
            if (turn) g[w][k].load(x[w] + k * dx[w] + half);
          }
        }
      }
      x[w] += 2 * dx[w];
    }
  };
  load(threadIdx.y);
  float c[kPairs], s[kPairs];
  const bool in = row >= 0 && row < a.rope.rows;
  if (!in && u == 0 && threadIdx.y == 0 && a.status) atomicCAS(a.status, 0, kDevBadPosition);
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    c[i] = 1.f;
    s[i] = 0.f;
  }
  if (turn && in) {
    load_f32<kPairs>(a.rope.cos + row * a.rope.stride + u * kPairs, a.wide_table, c);
    load_f32<kPairs>(a.rope.sin + row * a.rope.stride + u * kPairs, a.wide_table, s);
    if (a.inverse) {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) s[i] = -s[i];
    }
  }
  const int most = max(a.heads[0], a.heads[1]);
  for (int h0 = threadIdx.y; h0 < most; h0 += 2 * blockDim.y) {
    if (h0 != threadIdx.y) load(h0);
#pragma unroll
    for (int w = 0; w < 2; ++w) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (h0 + k * int(blockDim.y) >= a.heads[w]) continue;
        float v[kN];
        f[w][k].get(v);
        if (turn) {
          if constexpr (kInter) {
#pragma unroll
            for (int i = 0; in && i < kPairs; ++i) {
              const float p = v[2 * i], q = v[2 * i + 1];
              v[2 * i] = __fsub_rn(__fmul_rn(p, c[i]), __fmul_rn(q, s[i]));
              v[2 * i + 1] = __fadd_rn(__fmul_rn(p, s[i]), __fmul_rn(q, c[i]));
            }
          } else {
            float z[kN];
            g[w][k].get(z);
#pragma unroll
            for (int i = 0; in && i < kN; ++i) {
              const float p = v[i], q = z[i];
              v[i] = __fsub_rn(__fmul_rn(p, c[i]), __fmul_rn(q, s[i]));
              z[i] = __fadd_rn(__fmul_rn(p, s[i]), __fmul_rn(q, c[i]));
            }
            P::store(y[w] + k * dy[w] + half, z);
          }
        }
        P::store(y[w] + k * dy[w], v);
      }
      y[w] += 2 * dy[w];
    }
  }
}

template <int kDt, bool kInter, int kN>
cudaError_t launch_rope_as(const RopeArgs& a, cudaStream_t st) {
  const int units = (kInter ? a.rope.rot / kN : a.rope.rot / (2 * kN)) + (a.in_place ? 0 : (a.dim - a.rope.rot) / kN);
  const int most = a.heads[0] > a.heads[1] ? a.heads[0] : a.heads[1];
  // many tokens: two heads of each tensor a thread; few: as many threads as a CTA of 512 takes
  int hy = int64_t(a.batch) * a.len >= 1024 ? (most + 1) / 2 : most;
  const int fit = units >= 512 ? 1 : 512 / units;
  if (hy > fit) hy = fit;
  return launch_after(rope_kernel<kDt, kInter, kN>, dim3(a.len, a.batch), dim3(units, hy), 0, st, a);
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
