// C ABI of the paged 8-bit KV cache and of rotary positions (declared in include/lbq.h): argument checks and
// launches. Errors go to lbq_last_error(); nothing allocates or synchronises.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/lbq.h"
#include "lbq_kernels.h"
#include "lbq_paged.h"

namespace {

using lbq::set_error;

constexpr int kMaxGrid = 65535;
constexpr int64_t kMaxStart = int64_t(1) << 62;      // a token index behind it could pass 64 bits

int check_start(int64_t start) {
  return start >= 0 && start < kMaxStart ? LBQ_OK : set_error(LBQ_ERR_ARG, "start must be >= 0 and below 2^62");
}

bool aligned(const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int check_rows(const char* name, const void* p, int64_t sb, int64_t sl, int64_t sh) {
  if (p == nullptr) return set_error(LBQ_ERR_ARG, "%s is null", name);
  if (!aligned(p, 16)) return set_error(LBQ_ERR_ALIGN, "%s is not 16-byte aligned", name);
  if (sb % 8 || sl % 8 || sh % 8 || sb < 0 || sl < 0 || sh < 0)
    return set_error(LBQ_ERR_ALIGN, "%s strides (%lld, %lld, %lld) must be non-negative multiples of 8 elements", name,
                     (long long)sb, (long long)sl, (long long)sh);
  return LBQ_OK;
}

int check_pool(const void* k_pages, const float* k_amax, const void* v_pages, const float* v_amax, int64_t num_pages,
               int heads, int fmt) {
  if (!k_pages || !v_pages || !k_amax || !v_amax) return set_error(LBQ_ERR_ARG, "k_pages, v_pages, k_amax or v_amax is null");
  if (!aligned(k_pages, 128) || !aligned(v_pages, 128) || !aligned(k_amax, 4) || !aligned(v_amax, 4))
    return set_error(LBQ_ERR_ALIGN, "pages must be 128-byte aligned, their amax 4-byte aligned");
  if (heads <= 0 || heads > kMaxGrid) return set_error(LBQ_ERR_ARG, "heads %d outside [1, %d]", heads, kMaxGrid);
  if (fmt != LBQ_PAGE_INT8 && fmt != LBQ_PAGE_E4M3) return set_error(LBQ_ERR_ARG, "fmt %d is neither int8 nor e4m3", fmt);
  if (num_pages <= 0 || num_pages * heads > (int64_t(1) << 31) / lbq::kPageTokens - 1)
    return set_error(LBQ_ERR_ARG, "%lld pages of %d heads: pages * heads * 64 must stay below 2^31", (long long)num_pages, heads);
  return LBQ_OK;
}

int check_table(const int32_t* table, int64_t st_b, int width, int batch) {
  if (table == nullptr || !aligned(table, 4)) return set_error(LBQ_ERR_ARG, "page table is null or not 4-byte aligned");
  if (width <= 0 || st_b < 0 || (batch > 1 && st_b < width && st_b != 0))
    return set_error(LBQ_ERR_ARG, "page table of width %d with row stride %lld", width, (long long)st_b);
  return LBQ_OK;
}

int check_batch(int batch, int len, const char* what) {
  if (batch <= 0 || batch > kMaxGrid) return set_error(LBQ_ERR_ARG, "batch %d outside [1, %d]", batch, kMaxGrid);
  if (len < 0 || len > (1 << 28)) return set_error(LBQ_ERR_ARG, "%s %d out of range", what, len);
  return LBQ_OK;
}

int check_act16(int dtype) {
  return dtype == LBQ_DTYPE_BF16 || dtype == LBQ_DTYPE_F16 ? LBQ_OK
                                                           : set_error(LBQ_ERR_ARG, "dtype %d is neither bf16 nor fp16", dtype);
}

// A rotary table of any even `rot` up to `dim`, and its positions.
int make_rope(lbq::RopeTable* r, const float* cs, const float* sn, int64_t stride, int64_t rows, int rot, int interleaved,
              const void* pos, int pos64, int64_t sp_b, int64_t sp_l, int dim) {
  if (!cs || !sn) return set_error(LBQ_ERR_ARG, "rope_cos or rope_sin is null");
  if (!aligned(cs, 4) || !aligned(sn, 4)) return set_error(LBQ_ERR_ALIGN, "rope tables are not 4-byte aligned");
  if (rot <= 0 || rot % 2 || rot > dim) return set_error(LBQ_ERR_ARG, "rot %d must be even and in [2, %d]", rot, dim);
  if (rows <= 0 || stride < rot / 2)
    return set_error(LBQ_ERR_ARG, "rope tables of %lld rows with stride %lld for rot %d", (long long)rows, (long long)stride, rot);
  if (pos != nullptr && (!aligned(pos, pos64 ? 8 : 4) || sp_b < 0 || sp_l < 0))
    return set_error(LBQ_ERR_ARG, "positions must be aligned with non-negative strides");
  *r = lbq::RopeTable{cs, sn, stride, rows, rot, interleaved != 0, pos, pos64 != 0, sp_b, sp_l};
  return LBQ_OK;
}

int finish(cudaError_t e, const char* what) {
  return e == cudaSuccess ? LBQ_OK : set_error(LBQ_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

// Query rows (token, query head of the K/V head) that one CTA takes, by the rows of a K/V head: the few-row kernel (8 or 16
// a CTA) up to 64, the many-row kernel (256) above. Measured, us, few / many: 64 rows of 12 heads x 30160 keys 63 / 72, of 32
// batch heads x 8192 keys 54 / 63; 72 rows 93 / 72 and 94 / 63.
constexpr int64_t kFewRows = 64;
int attn_tile_rows(int64_t rows) { return rows <= 8 ? 8 : (rows <= kFewRows ? 16 : lbq::kManyTile); }

// At most 8 key splits whose CTAs fit the GPU at once as clusters are one cluster a tile, which merges them itself: no
// workspace, no second launch. Two CTAs an SM, 296, are more than clusters can fill, since one lies in one group of SMs: up to
// 256 CTAs they fit and gain 0.5 to 1 us, from 280 on some wait for a second wave (alike, one token x 4096 keys, clustered /
// not: 64 x 4 CTAs 14.1 / 16.7 us, 32 x 8 10.3 / 11.1, 80 x 3 17.9 / 19.5, 56 x 5 17.1 / 15.7, 72 x 4 22.2 / 16.9, 96 x 3 30.1 /
// 20.6, 36 x 8 17.6 / 11.5). CTAs of several waves are left to be scheduled one by one.
constexpr int64_t kFewCtas = 2 * 148;
constexpr int64_t kClusterCtas = 256;
bool attn_clustered(int64_t rows, int heads, int batch, int splits) {
  const int tile = attn_tile_rows(rows);
  return tile != lbq::kManyTile && splits > 1 && splits <= 8 &&
         (rows + tile - 1) / tile * heads * batch * splits <= kClusterCtas;
}

}  // namespace

extern "C" {

int lbq_rope(const void* x, int64_t sx_b, int64_t sx_l, int64_t sx_h, void* y, int64_t sy_b, int64_t sy_l, int64_t sy_h,
             int heads, const void* x2, int64_t sx2_b, int64_t sx2_l, int64_t sx2_h, void* y2, int64_t sy2_b,
             int64_t sy2_l, int64_t sy2_h, int heads2, int batch, int len, int dim, const float* rope_cos,
             const float* rope_sin, int64_t rope_stride, int64_t rope_rows, int rot, int interleaved, const void* pos,
             int pos64, int64_t sp_b, int64_t sp_l, int64_t start, int inverse, int dtype, void* stream) {
  int r;
  if (x == nullptr || y == nullptr) return set_error(LBQ_ERR_ARG, "x or y is null");
  if (dtype < LBQ_DTYPE_BF16 || dtype > 2) return set_error(LBQ_ERR_ARG, "dtype %d is not bf16 (0), fp16 (1) or fp32 (2)", dtype);
  if ((x2 == nullptr) != (y2 == nullptr) || (x2 != nullptr) != (heads2 > 0))
    return set_error(LBQ_ERR_ARG, "x2, y2 and heads2: give all or none");
  if (heads <= 0 || heads > kMaxGrid || heads2 < 0 || heads2 > kMaxGrid) return set_error(LBQ_ERR_ARG, "heads out of range");
  if ((r = check_batch(batch, len, "len"))) return r;
  if (dim <= 0 || dim > 512 || dim % 2) return set_error(LBQ_ERR_ARG, "dim %d must be even and in [2, 512]", dim);
  const int size = dtype == 2 ? 4 : 2;
  const void* ptrs[4] = {x, y, x2, y2};
  const int64_t strides[4][3] = {{sx_b, sx_l, sx_h}, {sy_b, sy_l, sy_h}, {sx2_b, sx2_l, sx2_h}, {sy2_b, sy2_l, sy2_h}};
  bool wide = true;
  for (int i = 0; i < (x2 ? 4 : 2); ++i) {
    if (!aligned(ptrs[i], size)) return set_error(LBQ_ERR_ALIGN, "a tensor is not aligned to its elements");
    wide = wide && aligned(ptrs[i], 16);
    for (int64_t s : strides[i]) {
      if (s < 0) return set_error(LBQ_ERR_ARG, "negative stride");
      wide = wide && s * size % 16 == 0;
    }
  }
  lbq::RopeArgs a{};
  if ((r = make_rope(&a.rope, rope_cos, rope_sin, rope_stride, rope_rows, rot, interleaved, pos, pos64, sp_b, sp_l, dim)))
    return r;
  if ((r = check_start(start))) return r;
  if (len == 0) return LBQ_OK;
  const int vec = 16 / size;
  // 16-byte accesses where a 16-byte piece lies wholly in the rotated part (or in one half of it) or in the rest
  a.vec = wide && rot % (interleaved ? vec : 2 * vec) == 0 && (dim - rot) % vec == 0;
  a.wide_table = rope_stride % 4 == 0 && aligned(rope_cos, 16) && aligned(rope_sin, 16);
  for (int i = 0; i < 2; ++i) {
    a.x[i] = i ? x2 : x;
    a.y[i] = i ? y2 : y;
    for (int k = 0; k < 3; ++k) {
      a.sx[i][k] = strides[2 * i][k];
      a.sy[i][k] = strides[2 * i + 1][k];
    }
  }
  a.heads[0] = heads;
  a.heads[1] = heads2;
  a.in_place = x == y && sx_b == sy_b && sx_l == sy_l && sx_h == sy_h &&
               (x2 == nullptr || (x2 == y2 && sx2_b == sy2_b && sx2_l == sy2_l && sx2_h == sy2_h));
  a.batch = batch;
  a.len = len;
  a.dim = dim;
  a.dtype = dtype;
  a.inverse = inverse != 0;
  a.start = start;
  a.status = lbq::device_status_ptr();
  return finish(lbq::launch_rope(a, static_cast<cudaStream_t>(stream)), "rope launch");
}

int lbq_page_write(const void* k, int64_t sk_b, int64_t sk_l, int64_t sk_h, const void* v, int64_t sv_b, int64_t sv_l,
                   int64_t sv_h, void* k_pages, float* k_amax, void* v_pages, float* v_amax, int64_t num_pages, int heads,
                   int fmt, const int32_t* table, int64_t st_b, int width, const int32_t* start, int64_t start0,
                   const int32_t* lens, int batch, int len, const float* rope_cos, const float* rope_sin,
                   int64_t rope_stride, int64_t rope_rows, int rot, int interleaved, const void* pos, int pos64,
                   int64_t sp_b, int64_t sp_l, int dtype, void* stream) {
  int r;
  if ((r = check_act16(dtype)) || (r = check_rows("k", k, sk_b, sk_l, sk_h)) || (r = check_rows("v", v, sv_b, sv_l, sv_h)) ||
      (r = check_pool(k_pages, k_amax, v_pages, v_amax, num_pages, heads, fmt)) ||
      (r = check_batch(batch, len, "len")) || (r = check_table(table, st_b, width, batch)))
    return r;
  if ((r = check_start(start0))) return r;
  if (start == nullptr && lens == nullptr && start0 + len > int64_t(width) * lbq::kPageTokens)
    return set_error(LBQ_ERR_ARG, "tokens [%lld, %lld) outside the %d-page table", (long long)start0,
                     (long long)(start0 + len), width);
  lbq::PageWriteArgs a{};
  if (rope_cos != nullptr || rope_sin != nullptr) {
    if ((r = make_rope(&a.rope, rope_cos, rope_sin, rope_stride, rope_rows, rot, interleaved, pos, pos64, sp_b, sp_l, 128)))
      return r;
    if (rot % (interleaved ? 8 : 16) || rope_stride % 4 || !aligned(rope_cos, 16) || !aligned(rope_sin, 16))
      return set_error(LBQ_ERR_ALIGN, "rope in the write: rot a multiple of %d, 16-byte aligned tables with a row "
                       "stride of a multiple of 4", interleaved ? 8 : 16);
  }
  if (len == 0) return LBQ_OK;
  a.src[0] = k;
  a.src[1] = v;
  const int64_t ss[2][3] = {{sk_b, sk_l, sk_h}, {sv_b, sv_l, sv_h}};
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 3; ++j) a.ss[i][j] = ss[i][j];
  a.codes[0] = static_cast<uint8_t*>(k_pages);
  a.codes[1] = static_cast<uint8_t*>(v_pages);
  a.amax[0] = k_amax;
  a.amax[1] = v_amax;
  a.pt = lbq::PageTable{table, st_b, width, num_pages};
  a.start = start;
  a.start0 = start0;
  a.lens = lens;
  a.batch = batch;
  a.len = len;
  a.heads = heads;
  a.fmt = fmt;
  a.dtype = dtype;
  a.status = lbq::device_status_ptr();
  return finish(lbq::launch_page_write(a, static_cast<cudaStream_t>(stream)), "page_write launch");
}

int lbq_page_read(const void* k_pages, const float* k_amax, const void* v_pages, const float* v_amax, int64_t num_pages,
                  int heads, int fmt, const int32_t* table, int64_t st_b, int width, const int32_t* start, int64_t start0,
                  const int32_t* lens, int batch, int len, void* k_out, int64_t sk_b, int64_t sk_l, int64_t sk_h,
                  void* v_out, int64_t sv_b, int64_t sv_l, int64_t sv_h, int dtype, void* stream) {
  int r;
  if ((r = check_act16(dtype)) || (r = check_rows("k_out", k_out, sk_b, sk_l, sk_h)) ||
      (r = check_rows("v_out", v_out, sv_b, sv_l, sv_h)) ||
      (r = check_pool(k_pages, k_amax, v_pages, v_amax, num_pages, heads, fmt)) ||
      (r = check_batch(batch, len, "len")) || (r = check_table(table, st_b, width, batch)))
    return r;
  if ((r = check_start(start0))) return r;
  if (start == nullptr && lens == nullptr && start0 + len > int64_t(width) * lbq::kPageTokens)
    return set_error(LBQ_ERR_ARG, "tokens [%lld, %lld) outside the %d-page table", (long long)start0,
                     (long long)(start0 + len), width);
  if (len == 0) return LBQ_OK;
  lbq::PageReadArgs a{};
  a.codes[0] = static_cast<const uint8_t*>(k_pages);
  a.codes[1] = static_cast<const uint8_t*>(v_pages);
  a.amax[0] = k_amax;
  a.amax[1] = v_amax;
  a.dst[0] = k_out;
  a.dst[1] = v_out;
  const int64_t sd[2][3] = {{sk_b, sk_l, sk_h}, {sv_b, sv_l, sv_h}};
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 3; ++j) a.sd[i][j] = sd[i][j];
  a.pt = lbq::PageTable{table, st_b, width, num_pages};
  a.start = start;
  a.start0 = start0;
  a.lens = lens;
  a.batch = batch;
  a.len = len;
  a.heads = heads;
  a.fmt = fmt;
  a.dtype = dtype;
  a.status = lbq::device_status_ptr();
  return finish(lbq::launch_page_read(a, static_cast<cudaStream_t>(stream)), "page_read launch");
}

int lbq_page_copy(void* k_pages, float* k_amax, void* v_pages, float* v_amax, int64_t num_pages, int heads, int layers,
                  int64_t layer_bytes, int64_t layer_amax, const int32_t* src, const int32_t* dst, int pairs,
                  void* stream) {
  int r;
  if ((r = check_pool(k_pages, k_amax, v_pages, v_amax, num_pages, heads, LBQ_PAGE_INT8))) return r;
  if (layers <= 0 || layers > kMaxGrid / 2) return set_error(LBQ_ERR_ARG, "layers %d outside [1, %d]", layers, kMaxGrid / 2);
  if (layers > 1 && (layer_bytes < num_pages * heads * lbq::kPageBytes || layer_bytes % 128 || layer_amax < num_pages * heads))
    return set_error(LBQ_ERR_ARG, "layer strides (%lld bytes, %lld amax) are smaller than a layer or not aligned",
                     (long long)layer_bytes, (long long)layer_amax);
  if (pairs < 0 || (pairs > 0 && (!src || !dst))) return set_error(LBQ_ERR_ARG, "src or dst is null");
  for (int i = 0; i < pairs; ++i)
    if (src[i] < 0 || src[i] >= num_pages || dst[i] < 0 || dst[i] >= num_pages)
      return set_error(LBQ_ERR_ARG, "pair %d: page %d -> %d outside the pool of %lld", i, src[i], dst[i], (long long)num_pages);
  lbq::PageCopyArgs a{};
  a.codes[0] = static_cast<uint8_t*>(k_pages);
  a.codes[1] = static_cast<uint8_t*>(v_pages);
  a.amax[0] = k_amax;
  a.amax[1] = v_amax;
  a.layer_codes = layer_bytes;
  a.layer_amax = layer_amax;
  a.heads = heads;
  a.layers = layers;
  for (int at = 0; at < pairs; at += lbq::kCopyPairs) {
    a.pairs = pairs - at < lbq::kCopyPairs ? pairs - at : lbq::kCopyPairs;
    for (int i = 0; i < a.pairs; ++i) {
      a.src[i] = src[at + i];
      a.dst[i] = dst[at + i];
    }
    if ((r = finish(lbq::launch_page_copy(a, static_cast<cudaStream_t>(stream)), "page_copy launch"))) return r;
  }
  return LBQ_OK;
}

int lbq_paged_attn_splits(int batch, int q_len, int heads, int group, int64_t max_kv_len, int ragged) {
  if (batch <= 0 || q_len <= 0 || heads <= 0 || group <= 0 || max_kv_len <= 0) return 1;
  const int64_t rows = int64_t(q_len) * group;
  const int tile = attn_tile_rows(rows);
  const int64_t ctas = (rows + tile - 1) / tile * heads * batch;
  const int64_t pages = (max_kv_len + lbq::kPageTokens - 1) / lbq::kPageTokens;
  // Few rows: two CTAs an SM (296 at once), a split keeps at least 4 pages, one for each warp. Many rows: one CTA an SM, at
  // least 8 pages to pay for the query tiles. Ragged batches (mean length under two thirds of the longest) get more and
  // shorter splits, which balance the long sequences (measured, us: CTAs before splitting x longest sequence, with 1 / 2 / 4 / 8
  // splits. 256 x 8192 keys, all alike 84 / 93 / 100; ragged 74 / 65 / 60 / 62; 512 x 8192 ragged 117 / 107 / 103; 1024 x 4096
  // ragged 98 / 104 / 113; 128 x 8192 ragged 51 / 41 / 28 / 32; 64 x 30000 ragged - / 91 / 70 / 48; 96 x 4100 with 3 / 4 / 6
  // splits, ragged 24 / 21 / 17, all alike 26 / 38 / 31). More CTAs than SMs want splits of 32 pages and more (ragged, 1 / 2 / 4:
  // 192 x 2048 keys 23 / 20 / 22, 480 x 3000 45 / 48 / 49, 512 x 2048 35 / 39 / 44, 512 x 30000 366 / 330 / 312).
  const bool few = tile != lbq::kManyTile;
  int64_t n = (few ? kFewCtas : 148) / ctas;
  if (few && ragged && pages >= 32 && ctas >= 64 && ctas <= 600) {
    if (ctas <= 148) n *= 2;
    else n = std::max<int64_t>(std::min<int64_t>(4, pages / 32), ctas <= 400 ? 2 : 1);
  }
  const int64_t least = few ? 4 : 8;
  if (n > pages / least) n = pages / least;
  if (few && n > 8 && n <= 16 && pages <= 96) n = 8;      // one cluster's worth: no merge launch (16 splits of 64 pages: alike)
  return int(n < 1 ? 1 : (n > 1024 ? 1024 : n));
}

size_t lbq_paged_attn_workspace(int batch, int q_len, int heads, int group, int num_splits) {
  if (batch <= 0 || q_len < 0 || heads <= 0 || group <= 0 || num_splits <= 1) return 0;
  const uint64_t rows = uint64_t(q_len) * group;
  const uint64_t tile = attn_tile_rows(int64_t(rows));
  if (attn_clustered(int64_t(rows), heads, batch, num_splits)) return 0;
  uint64_t n, bytes;
  if (__builtin_mul_overflow((rows + tile - 1) / tile * tile, uint64_t(batch) * heads, &n) ||
      __builtin_mul_overflow(n, uint64_t(num_splits), &n) || __builtin_mul_overflow(n, uint64_t(128 * 4 + 8), &bytes))
    return SIZE_MAX;
  return size_t(bytes);
}

int lbq_paged_attn(const void* q, int64_t sq_b, int64_t sq_l, int64_t sq_h, const void* k_pages, const float* k_amax,
                   const void* v_pages, const float* v_amax, int64_t num_pages, int heads, int fmt, const int32_t* table,
                   int64_t st_b, int width, const int32_t* kv_lens, int64_t kv_len0, const int32_t* q_lens, int batch,
                   int q_len, int group, int causal, float sm_scale, void* out, int64_t so_b, int64_t so_l, int64_t so_h,
                   float* lse, int num_splits, void* workspace, size_t workspace_bytes, int dtype, void* stream) {
  int r;
  if ((r = check_act16(dtype)) || (r = check_rows("q", q, sq_b, sq_l, sq_h)) ||
      (r = check_rows("out", out, so_b, so_l, so_h)) ||
      (r = check_pool(k_pages, k_amax, v_pages, v_amax, num_pages, heads, fmt)) ||
      (r = check_batch(batch, q_len, "q_len")) || (r = check_table(table, st_b, width, batch)))
    return r;
  if (group <= 0 || int64_t(group) * heads > (1 << 24))
    return set_error(LBQ_ERR_ARG, "group %d: at least 1 and at most 2^24 query heads in all", group);
  if (int64_t(q_len) * group > (1 << 30)) return set_error(LBQ_ERR_ARG, "q_len * group too large");
  if (kv_lens == nullptr && (kv_len0 < 0 || kv_len0 > int64_t(width) * lbq::kPageTokens))
    return set_error(LBQ_ERR_ARG, "kv_len %lld outside the %d-page table", (long long)kv_len0, width);
  if (width > (1 << 24)) return set_error(LBQ_ERR_ARG, "page table of width %d", width);
  if (lse != nullptr && !aligned(lse, 4)) return set_error(LBQ_ERR_ALIGN, "lse is not 4-byte aligned");
  if (q_len == 0) return LBQ_OK;
  lbq::PagedAttnArgs a{};
  const int64_t rows = int64_t(q_len) * group;
  a.tile_rows = attn_tile_rows(rows);
  a.tiles = int((rows + a.tile_rows - 1) / a.tile_rows);
  if (int64_t(a.tiles) * heads > (int64_t(1) << 31) - 1) return set_error(LBQ_ERR_ARG, "too many row tiles");
  int pages = width;                                        // most pages that a sequence can have
  if (kv_lens == nullptr) pages = kv_len0 > 0 ? int((kv_len0 + lbq::kPageTokens - 1) / lbq::kPageTokens) : 1;
  if (num_splits < 1) num_splits = 1;
  if (num_splits > pages) num_splits = pages;
  a.split_pages = (pages + num_splits - 1) / num_splits;
  a.splits = (pages + a.split_pages - 1) / a.split_pages;
  if (a.splits > kMaxGrid) return set_error(LBQ_ERR_ARG, "too many key splits");
  a.clustered = attn_clustered(rows, heads, batch, a.splits);
  if (a.splits > 1 && !a.clustered) {
    const size_t need = lbq_paged_attn_workspace(batch, q_len, heads, group, a.splits);
    if (workspace == nullptr || workspace_bytes < need)
      return set_error(LBQ_ERR_ARG, "workspace of %zu bytes is smaller than the %zu needed", workspace_bytes, need);
    if (!aligned(workspace, 16)) return set_error(LBQ_ERR_ALIGN, "workspace is not 16-byte aligned");
    const int64_t n = int64_t(a.splits) * batch * heads * a.tiles * a.tile_rows;
    a.o_part = static_cast<float*>(workspace);
    a.ml_part = reinterpret_cast<float2*>(a.o_part + n * 128);
  }
  if (!(sm_scale > 0.f)) sm_scale = 0.08838834764831845f;   // 128 ** -0.5
  a.q = q;
  a.out = out;
  const int64_t sq[3] = {sq_b, sq_l, sq_h}, so[3] = {so_b, so_l, so_h};
  for (int i = 0; i < 3; ++i) {
    a.sq[i] = sq[i];
    a.so[i] = so[i];
  }
  a.lse = lse;
  a.ka = k_amax;
  a.va = v_amax;
  a.pt = lbq::PageTable{table, st_b, width, num_pages};
  a.k_pages = static_cast<const uint8_t*>(k_pages);
  a.v_pages = static_cast<const uint8_t*>(v_pages);
  a.wide_out = aligned(out, 32) && so_b % 16 == 0 && so_l % 16 == 0 && so_h % 16 == 0;
  a.kv_lens = kv_lens;
  a.kv_len0 = kv_len0;
  a.q_lens = q_lens;
  a.batch = batch;
  a.q_len = q_len;
  a.heads = heads;
  a.group = group;
  a.causal = causal != 0;
  a.fmt = fmt;
  a.dtype = dtype;
  a.score_log2 = float(double(sm_scale) * 1.4426950408889634 / lbq::code_max(fmt));
  a.v_unit = 1.f / lbq::code_max(fmt);
  a.status = lbq::device_status_ptr();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a.tile_rows != lbq::kManyTile) {
    CUtensorMap tk, tv;
    const uint64_t prows = uint64_t(num_pages) * heads * lbq::kPageTokens;
    if ((r = lbq::make_page_map(&tk, k_pages, prows, "k_pages", lbq::kPageTokens)) ||
        (r = lbq::make_page_map(&tv, v_pages, prows, "v_pages", lbq::kPageTokens)))
      return r;
    r = finish(lbq::launch_paged_decode(a, tk, tv, st), "paged_attn launch");
  } else {
    r = finish(lbq::launch_paged_rows(a, st), "paged_attn launch");
  }
  if (r) return r;
  if (a.splits > 1 && !a.clustered) return finish(lbq::launch_paged_combine(a, st), "paged_attn merge launch");
  return LBQ_OK;
}

}  // extern "C"
