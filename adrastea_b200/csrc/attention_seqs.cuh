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

}  // namespace adr
