// What the operators over sequences of different lengths share: finding a row's sequence, its span, its pages.
//
// The new tokens of all sequences lie one behind the other in the rows of q: sequence s has the rows
// cu_q[s] .. cu_q[s + 1] - 1 and kv_len[s] positions of which its rows are the last.  Position p of it lies in
// slot p % page_size of page block_table[s][p / page_size].  The three arrays are device memory, so their
// contents are checked here, where they are read: spans are cut to the rows there are, lengths to the table's
// capacity, and a page outside the pool is neither read nor written (status bit PAGED_BAD).
#pragma once

#include "tma.cuh"

namespace adr {

constexpr unsigned PAGED_BAD = 1u << 20;  // a length or page outside what the tables and the pool hold

struct SeqSpan {
  int q0, lq;  // its first row and their number
  int lk;      // its positions; row i is at position lk - lq + i
};

__device__ __forceinline__ SeqSpan seq_span(const int* cu_q, const int* kv_len, int s, int tokens, int capacity,
                                            unsigned int* status) {
  SeqSpan r;
  r.q0 = min(max(__ldg(cu_q + s), 0), tokens);
  r.lq = min(max(__ldg(cu_q + s + 1), r.q0), tokens) - r.q0;
  r.lk = r.lq;
  if (kv_len) {
    const int n = __ldg(kv_len + s);
    r.lk = min(max(n, 0), capacity);
    if (r.lk != n) atomicOr(status, PAGED_BAD);
  }
  return r;
}

// The sequence that row t belongs to, found by a whole warp: the first s with t < cu_q[s + 1], 32 probes at a time
// (a lane's probe is one load, so 32 sequences cost one round trip to L2 and 1024 cost two).  n_seqs if there is none.
__device__ __forceinline__ int find_sequence(const int* cu_q, int n_seqs, int t, int lane) {
  int lo = 0, hi = n_seqs;  // the answer lies in [lo, hi]
  while (lo < hi) {
    const int step = (hi - lo + 31) / 32;
    const int probe = lo + lane * step + step - 1;  // last sequence of this lane's share
    const bool above = probe >= hi || t < __ldg(cu_q + probe + 1);
    const unsigned m = __ballot_sync(0xffffffffu, above);
    const int first = m ? __ffs(m) - 1 : 32;  // the first share that reaches past t
    lo = min(lo + first * step, hi);
    hi = min(lo + step - 1, hi);
  }
  return lo;
}

// Whether the arrays begin where their elements may: from elsewhere the GPU cannot read one.
template <typename... T>
bool on_elements(const T*... arrays) {
  return ((reinterpret_cast<uintptr_t>(arrays) % alignof(T) == 0) && ...);
}

// A launch that may begin while the one before it in its stream ends: the kernels here wait for that one's end before
// they read or write any memory, so it need not be the caller's choice as it is for kernels that fetch weights ahead (in
// a stream of equal calls: 4111 rows rotated 21.6 against 22.8 us, a token over 131072 keys 98.0 against 99.9).
// `fills`: what note_filling_launch wants to know; 0 for a kernel that does not fill the GPU.
template <typename... KArgs, typename... Args>
int launch_serving(adr_ctx* ctx, cudaStream_t stream, void (*kfn)(KArgs...), dim3 grid, unsigned threads, size_t smem,
                   int fills, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kfn, static_cast<KArgs>(args)...);
  if (e != cudaSuccess) {
    ctx->last_cuda_error = (int)e;
    return ADR_ERR_CUDA;
  }
  if (fills) note_filling_launch(ctx, stream, fills);
  return after_launch(ctx);
}

}  // namespace adr
