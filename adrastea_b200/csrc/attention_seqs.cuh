// Arguments of the attention over sequences of different lengths, shared by its kernels.
#pragma once

#include "paged.cuh"

namespace adr {

struct SeqAttention {
  __half* out;
  const __half *q, *k, *v;
  long long so[2], sq[2];        // row, head
  long long sk[3], sv[3];        // page, row, head (without pages: -, row, head)
  const int *cu_q, *kv_len;      // kv_len null: the keys are the sequence's own rows
  const int* block_table;        // null: k and v are rows like q
  int tokens, n_seqs, n_heads, n_kv_heads, group, head_dim;
  int max_pages, page_size, n_pages;
  int causal;
  float scale;
  unsigned int* status;
};

// A copy of `rows` slots of one head of a page: [64 columns, 1 head, rows, 1 page] of a pool with strides page, slot,
// head.  (A dimension of one element is given a stride that the copy engine takes.)
inline int pool_map(adr_ctx* ctx, CUtensorMap* map, const __half* base, const long long* s, const SeqAttention& a,
                    int rows) {
  const uint64_t dims[4] = {(uint64_t)a.head_dim, (uint64_t)a.n_kv_heads, (uint64_t)a.page_size, (uint64_t)a.n_pages};
  const long long st[3] = {s[2], s[1], s[0]};
  uint64_t strides[3];
  for (int i = 0; i < 3; ++i) strides[i] = dims[i + 1] > 1 ? (uint64_t)st[i] * 2 : (uint64_t)a.head_dim * 2;
  const uint32_t box[4] = {64u, 1u, (uint32_t)rows, 1u};
  return tma_encode(ctx, map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Kernels of a few rows per sequence (attention_few.cu): `rows` rows of a key head at most chooses the tile,
// sequences with more than max_rows are passed over.
// attention_few_takes: whether its counts fit (`one_tile_each`: no sequence has more than `rows` rows).
bool attention_few_takes(const SeqAttention& a, int rows, bool one_tile_each);
size_t attention_few_workspace(const adr_ctx* ctx, int head_dim);
int launch_attention_few(adr_ctx* ctx, cudaStream_t stream, const SeqAttention& a, int rows, int max_rows,
                         void* workspace);

// Tiles of many rows (attention_tiles.cu): sequences with fewer than min_rows rows of a key head are passed over.  The
// workspace is used over pages only.
// attention_tiles_splits: how many CTAs share a tile's keys over pages; more than one: all tiles are on the GPU at once.
int attention_tiles_splits(const adr_ctx* ctx, const SeqAttention& a);
size_t attention_tiles_workspace(const adr_ctx* ctx, int head_dim);
int launch_attention_tiles(adr_ctx* ctx, cudaStream_t stream, const SeqAttention& a, int max_q, int min_rows,
                           void* workspace);

}  // namespace adr
