// Argument blocks and launchers of the paged 8-bit KV cache and of the rotary kernel (internal header).
//
// Cache layout: a page holds 64 tokens of every K/V head. Codes [pages][heads][64][128] are int8 (fmt 0) or
// e4m3 (fmt 1); amax [pages][heads] (f32) is the largest magnitude of a page and head, and
// value = code * amax / Q with Q = 127 (int8) or 448 (e4m3). Token t of sequence b is row t % 64 of page
// table[b][t / 64].
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace lbq {

constexpr int kPageTokens = 64;
constexpr int kPageBytes = 64 * 128;          // codes of one page, head and tensor
constexpr float kAmaxFloor = 9.094947017729282379150390625e-13f;   // 2^-40

__host__ __device__ inline float code_max(int fmt) { return fmt ? 448.f : 127.f; }

struct PageTable {
  const int32_t* table;         // [batch][st_b], `width` entries used a row
  int64_t st_b;
  int width;
  int64_t num_pages;
};

struct RopeTable {
  const float* cos;             // null: no rotation; else [rows][rot / 2], row stride `stride`
  const float* sin;
  int64_t stride, rows;
  int rot;
  int interleaved;              // pairs (2i, 2i + 1); else (i, i + rot / 2)
  const void* pos;              // [batch][len] table rows (null: start + i)
  int pos64;                    // pos is int64, else int32
  int64_t sp_b, sp_l;
};

struct RopeArgs {
  const void* x[2];             // two tensors of one call ([B, L, heads, dim]); the second may have no heads
  void* y[2];
  int64_t sx[2][3], sy[2][3];
  int heads[2];
  int in_place;                 // y is x: channels past `rot` stay
  int batch, len, dim;
  int dtype;                    // 0 bf16, 1 fp16, 2 fp32
  int vec;                      // 16-byte accesses
  int wide_table;               // the tables' rows are 16-byte aligned
  int inverse;
  int64_t start;                // position of token 0 when the table has no `pos`
  RopeTable rope;
  int* status;
};

struct PageWriteArgs {
  const void* src[2];           // K, V [B, L, heads, 128]
  int64_t ss[2][3];
  uint8_t* codes[2];
  float* amax[2];
  PageTable pt;
  const int32_t* start;         // [B] tokens held before (null: start0 for all)
  int64_t start0;
  const int32_t* lens;          // [B] new tokens (null: len)
  int batch, len, heads, fmt, dtype;
  RopeTable rope;               // of K
  int* status;
};

struct PageReadArgs {
  const uint8_t* codes[2];
  const float* amax[2];
  void* dst[2];                 // K, V [B, L, heads, 128]
  int64_t sd[2][3];
  PageTable pt;
  const int32_t* start;         // first token read (null: start0)
  int64_t start0;
  const int32_t* lens;          // [B] tokens read (null: len); rows past them are 0
  int batch, len, heads, fmt, dtype;
  int* status;
};

constexpr int kManyTile = 256;                  // query rows of a CTA of the many-row attention kernel

constexpr int kCopyPairs = 480;               // page pairs of one launch (they travel as kernel parameters)
struct PageCopyArgs {
  uint8_t* codes[2];
  float* amax[2];
  int64_t layer_codes, layer_amax;            // bytes / floats from one layer's pages to the next's
  int heads, layers, pairs;
  int32_t src[kCopyPairs], dst[kCopyPairs];
};

struct PagedAttnArgs {
  const void* q;                // [B, Lq, heads * group, 128]
  int64_t sq[3];
  void* out;
  int64_t so[3];
  float* lse;                   // null, or [B, Lq, heads * group]
  const uint8_t* k_pages;
  const uint8_t* v_pages;
  const float* ka;
  const float* va;
  PageTable pt;
  const int32_t* kv_lens;       // null: kv_len0
  int64_t kv_len0;
  const int32_t* q_lens;        // null: q_len
  int batch, q_len, heads, group, causal, fmt, dtype;
  float score_log2;             // softmax scale * log2(e) / Q
  float v_unit;                 // 1 / Q
  int tile_rows, tiles;         // rows (query token, query head of the K/V head) of a CTA, tiles of a K/V head
  int splits, split_pages;      // key splits, and the pages of one
  int clustered;                // the splits of a tile are one cluster, which merges them (few rows, at most 8 splits)
  float* o_part;                // [splits][batch * heads][tiles * tile_rows][128] (splits > 1, not clustered)
  float2* ml_part;              // the same rows' (max in log2 units, sum)
  int wide_out;                 // out's base and strides are 32-byte aligned
  int* status;
};

cudaError_t launch_rope(const RopeArgs& a, cudaStream_t st);
cudaError_t launch_page_write(const PageWriteArgs& a, cudaStream_t st);
cudaError_t launch_page_read(const PageReadArgs& a, cudaStream_t st);
cudaError_t launch_page_copy(const PageCopyArgs& a, cudaStream_t st);
cudaError_t launch_paged_decode(const PagedAttnArgs& a, const CUtensorMap& tm_k, const CUtensorMap& tm_v,
                                cudaStream_t st);
cudaError_t launch_paged_rows(const PagedAttnArgs& a, cudaStream_t st);
cudaError_t launch_paged_combine(const PagedAttnArgs& a, cudaStream_t st);

// Tensor map of `rows` x 128 bytes, box 64 x 128 bytes, 128-byte swizzle; 0 or an LBQ_ERR_* code.
int make_page_map(CUtensorMap* m, const void* base, uint64_t rows, const char* name, uint32_t box_rows);

}  // namespace lbq
