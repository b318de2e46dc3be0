// Attention over sequences of different lengths: the entry points and the choice of a kernel.
#include <algorithm>
#include <climits>
#include <cmath>

#include "paged.cuh"
#include "attention_seqs.cuh"

namespace adr {

namespace {

// Rows of a key head up to which the kernel of few rows takes a sequence.  (32 rows over 32768 positions: 38 against 85 us
// in tiles, 32 x 1000: 46 against 40; from 40 rows on the tiles are ahead nearly everywhere, 32 x 1000: 160 against 143.  Fitted to
// head_dim 128: of 64, 32 x 1000 takes 31.5 us here and 18.7 in tiles.)
constexpr int FEW_ROWS = 32;

// Keys of a tile's part up to which a second kernel for the sequences of few rows costs more than their tiles (6 sequences of
// up to 100 tokens over up to 4096 positions, 32/8 heads: 43 against 56 us; a single token's tile over more would be what all
// others wait for).  By the table's width, as the number of parts is: the figures are of tables as wide as the longest sequence.
constexpr int ALONE_KEYS = 4096;

// The strides of n dimensions of the given extents: not negative, and 16-byte steps where a dimension has more
// than one element.
int check_steps(const void* base, const long long* strides, int n, const int* extents) {
  if (!strides) return ADR_ERR_INVALID;
  for (int i = 0; i < n; ++i)
    if (strides[i] < 0) return ADR_ERR_INVALID;
  if (reinterpret_cast<uintptr_t>(base) & 15u) return ADR_ERR_SHAPE;
  for (int i = 0; i < n; ++i)
    if (extents[i] > 1 && (strides[i] % 8 != 0 || strides[i] == 0)) return ADR_ERR_SHAPE;
  return ADR_OK;
}

int check_heads(int n_heads, int n_kv_heads, int head_dim) {
  if (n_heads <= 0 || n_kv_heads <= 0 || head_dim <= 0) return ADR_ERR_INVALID;
  if (head_dim != 64 && head_dim != 128) return ADR_ERR_SHAPE;
  if (n_heads % n_kv_heads != 0 || n_heads / n_kv_heads > 64 || n_kv_heads > 65535) return ADR_ERR_SHAPE;
  return ADR_OK;
}

}  // namespace

}  // namespace adr

using namespace adr;

extern "C" int adr_attention_packed(adr_ctx* ctx, adr_stream stream, void* out, const void* q, const void* k,
                                    const void* v, int tokens, int n_seqs, int max_q, int n_heads, int n_kv_heads,
                                    int head_dim, const long long* strides_o, const long long* strides_q,
                                    const long long* strides_k, const long long* strides_v, const int32_t* cu_q,
                                    float scale, uint32_t mask_op) {
  if (!out || !q || !k || !v || !cu_q || tokens <= 0 || n_seqs <= 0 || max_q <= 0) return ADR_ERR_INVALID;
  if (mask_op > ADR_MASK_CAUSAL || !std::isfinite(scale)) return ADR_ERR_INVALID;
  if (int rc = check_heads(n_heads, n_kv_heads, head_dim); rc != ADR_OK) return rc;
  const int eq[2] = {tokens, n_heads}, ek[2] = {tokens, n_kv_heads};
  if (int rc = check_steps(out, strides_o, 2, eq); rc != ADR_OK) return rc;
  if (int rc = check_steps(q, strides_q, 2, eq); rc != ADR_OK) return rc;
  if (int rc = check_steps(k, strides_k, 2, ek); rc != ADR_OK) return rc;
  if (int rc = check_steps(v, strides_v, 2, ek); rc != ADR_OK) return rc;
  if (!on_elements(cu_q)) return ADR_ERR_SHAPE;
  if (!ctx) return ADR_ERR_INVALID;
  DeviceGuard guard(ctx);
  SeqAttention p = {};
  p.out = (__half*)out;
  p.q = (const __half*)q;
  p.k = (const __half*)k;
  p.v = (const __half*)v;
  p.cu_q = cu_q;
  p.tokens = tokens;
  p.n_seqs = n_seqs;
  p.n_heads = n_heads;
  p.n_kv_heads = n_kv_heads;
  p.group = n_heads / n_kv_heads;
  p.head_dim = head_dim;
  p.causal = mask_op == ADR_MASK_CAUSAL;
  for (int i = 0; i < 2; ++i) {
    p.so[i] = strides_o[i];
    p.sq[i] = strides_q[i];
    p.sk[i + 1] = strides_k[i];
    p.sv[i + 1] = strides_v[i];
  }
  p.scale = scale;
  p.status = ctx->d_status;
  return launch_attention_tiles(ctx, (cudaStream_t)stream, p, max_q, 1, nullptr);
}

extern "C" size_t adr_attention_paged_workspace(const adr_ctx* ctx, int n_heads, int n_kv_heads, int head_dim) {
  if (!ctx || check_heads(n_heads, n_kv_heads, head_dim) != ADR_OK) return 0;
  return std::max(attention_few_workspace(ctx, head_dim), attention_tiles_workspace(ctx, head_dim));
}

extern "C" int adr_attention_paged(adr_ctx* ctx, adr_stream stream, void* out, const void* q, const void* k_pages,
                                   const void* v_pages, int tokens, int n_seqs, int max_q, int n_heads,
                                   int n_kv_heads, int head_dim, const long long* strides_o,
                                   const long long* strides_q, const long long* strides_kp,
                                   const long long* strides_vp, const int32_t* block_table, const int32_t* cu_q,
                                   const int32_t* kv_len, int max_pages, int page_size, int n_pages, float scale,
                                   void* workspace, size_t workspace_bytes) {
  if (!out || !q || !k_pages || !v_pages || !block_table || !cu_q || !kv_len || !workspace) return ADR_ERR_INVALID;
  if (tokens <= 0 || n_seqs <= 0 || max_q <= 0 || max_pages <= 0 || page_size <= 0 || n_pages <= 0)
    return ADR_ERR_INVALID;
  if (!std::isfinite(scale)) return ADR_ERR_INVALID;
  if (int rc = check_heads(n_heads, n_kv_heads, head_dim); rc != ADR_OK) return rc;
  if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)) != 0) return ADR_ERR_SHAPE;
  if ((long long)max_pages * page_size > (1LL << 30)) return ADR_ERR_SHAPE;
  const int eq[2] = {tokens, n_heads}, ek[3] = {n_pages, page_size, n_kv_heads};
  if (int rc = check_steps(out, strides_o, 2, eq); rc != ADR_OK) return rc;
  if (int rc = check_steps(q, strides_q, 2, eq); rc != ADR_OK) return rc;
  if (int rc = check_steps(k_pages, strides_kp, 3, ek); rc != ADR_OK) return rc;
  if (int rc = check_steps(v_pages, strides_vp, 3, ek); rc != ADR_OK) return rc;
  if ((reinterpret_cast<uintptr_t>(workspace) & 15u) || !on_elements(block_table, cu_q, kv_len)) return ADR_ERR_SHAPE;
  if (!ctx) return ADR_ERR_INVALID;
  if (workspace_bytes < adr_attention_paged_workspace(ctx, n_heads, n_kv_heads, head_dim)) return ADR_ERR_SHAPE;
  DeviceGuard guard(ctx);
  SeqAttention p = {};
  p.out = (__half*)out;
  p.q = (const __half*)q;
  p.k = (const __half*)k_pages;
  p.v = (const __half*)v_pages;
  p.cu_q = cu_q;
  p.kv_len = kv_len;
  p.block_table = block_table;
  p.tokens = tokens;
  p.n_seqs = n_seqs;
  p.n_heads = n_heads;
  p.n_kv_heads = n_kv_heads;
  p.group = n_heads / n_kv_heads;
  p.head_dim = head_dim;
  p.max_pages = max_pages;
  p.page_size = page_size;
  p.n_pages = n_pages;
  p.causal = 1;
  for (int i = 0; i < 2; ++i) {
    p.so[i] = strides_o[i];
    p.sq[i] = strides_q[i];
  }
  for (int i = 0; i < 3; ++i) {
    p.sk[i] = strides_kp[i];
    p.sv[i] = strides_vp[i];
  }
  p.scale = scale;
  p.status = ctx->d_status;
  const long long rows = (long long)max_q * p.group;
  if (rows <= FEW_ROWS && attention_few_takes(p, (int)rows, false))
    return launch_attention_few(ctx, (cudaStream_t)stream, p, (int)rows, INT_MAX, workspace);
  // All sequences of one length, or all tiles on the GPU at once with at most ALONE_KEYS keys each: tiles for all.  Otherwise
  // those of few rows go to the other kernel.
  const int splits = attention_tiles_splits(ctx, p);
  const bool at_once = splits > 1 && (long long)max_pages * page_size <= (long long)splits * ALONE_KEYS;
  if ((long long)n_seqs * max_q == tokens || at_once || !attention_few_takes(p, FEW_ROWS, true))
    return launch_attention_tiles(ctx, (cudaStream_t)stream, p, max_q, 1, workspace);
  if (int rc = launch_attention_tiles(ctx, (cudaStream_t)stream, p, max_q, FEW_ROWS + 1, workspace); rc != ADR_OK)
    return rc;
  return launch_attention_few(ctx, (cudaStream_t)stream, p, FEW_ROWS, FEW_ROWS, workspace);
}
