// Attention over sequences of different lengths: the entry points, and a kernel that is right for every case.
#include <algorithm>
#include <climits>
#include <cmath>

#include "paged.cuh"
#include "attention_seqs.cuh"

namespace adr {

namespace {

// One warp per (row, query head): the keys one after the other with a running maximum and sum.
template <int HD>
__global__ void __launch_bounds__(128) attention_seqs_simple_kernel(SeqAttention p) {
  constexpr int PER = HD / 32;
  pdl_wait_trigger();
  const int t = blockIdx.x, lane = threadIdx.x & 31;
  const int s = find_sequence(p.cu_q, p.n_seqs, t, lane);
  if (s >= p.n_seqs) return;
  const SeqSpan span = seq_span(p.cu_q, p.kv_len, s, p.tokens, p.max_pages * p.page_size, p.status);
  if (t < span.q0 || t >= span.q0 + span.lq) return;
  const int limit = p.causal ? max(0, span.lk - span.lq + (t - span.q0) + 1) : span.lk;
  for (int h = threadIdx.x >> 5; h < p.n_heads; h += 4) {
    const int kh = h / p.group;
    const __half* q = p.q + t * p.sq[0] + h * p.sq[1] + lane * PER;
    float qf[PER], o[PER], m = -INFINITY, l = 0.0f;
    for (int i = 0; i < PER; ++i) qf[i] = __half2float(q[i]), o[i] = 0.0f;
    for (int j = 0; j < limit; ++j) {
      long long ko, vo;
      bool real = true;
      if (p.block_table) {
        const int page = __ldg(p.block_table + (long long)s * p.max_pages + j / p.page_size);
        real = page >= 0 && page < p.n_pages;
        if (!real) atomicOr(p.status, PAGED_BAD);
        ko = page * p.sk[0] + (j % p.page_size) * p.sk[1] + kh * p.sk[2];
        vo = page * p.sv[0] + (j % p.page_size) * p.sv[1] + kh * p.sv[2];
      } else {
        ko = (long long)(span.q0 + j) * p.sk[1] + kh * p.sk[2];
        vo = (long long)(span.q0 + j) * p.sv[1] + kh * p.sv[2];
      }
      float x = 0.0f;
      for (int i = 0; i < PER; ++i) x += real ? qf[i] * __half2float(p.k[ko + lane * PER + i]) : 0.0f;
      for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
      x *= p.scale;
      const float mn = fmaxf(m, x), mu = mn == -INFINITY ? 0.0f : mn;
      const float a = expf(m - mu), w = expf(x - mu);
      l = l * a + w;
      for (int i = 0; i < PER; ++i) o[i] = o[i] * a + (real ? w * __half2float(p.v[vo + lane * PER + i]) : 0.0f);
      m = mn;
    }
    __half* dst = p.out + t * p.so[0] + h * p.so[1] + lane * PER;
    for (int i = 0; i < PER; ++i) dst[i] = __float2half_rn(limit > 0 ? o[i] / l : 0.0f);
  }
}

int launch_simple(adr_ctx* ctx, cudaStream_t stream, const SeqAttention& p) {
  if (p.head_dim == 64) attention_seqs_simple_kernel<64><<<p.tokens, 128, 0, stream>>>(p);
  else attention_seqs_simple_kernel<128><<<p.tokens, 128, 0, stream>>>(p);
  return after_launch(ctx);
}

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
  return launch_simple(ctx, (cudaStream_t)stream, p);
}

extern "C" size_t adr_attention_paged_workspace(const adr_ctx* ctx, int n_heads, int n_kv_heads, int head_dim) {
  if (!ctx || check_heads(n_heads, n_kv_heads, head_dim) != ADR_OK) return 0;
  return attention_few_workspace(ctx, head_dim);
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
  if (reinterpret_cast<uintptr_t>(workspace) & 15u) return ADR_ERR_SHAPE;
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
  return launch_attention_few(ctx, (cudaStream_t)stream, p, (int)std::min<long long>((long long)max_q * p.group, 64),
                              INT_MAX, workspace);
}
