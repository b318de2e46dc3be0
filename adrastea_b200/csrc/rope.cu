// Rotary positions of packed rows: pairs (2i, 2i + 1) or (i, i + d/2), all or the first part of a head, angles
// scaled for long contexts; alone, or for the new tokens of sequences whose k and v go to a paged cache.
//
// The angle of pair i at position p is p * f_i.  A 32-bit f_i would lose it at far positions (2^-24 relative of
// 10^6 radians), and a 64-bit product costs the GPU's few fp64 units.  So the table holds f_i / (2 pi), the turns
// per position, as a 64-bit fixed-point fraction; p times it modulo 2^64 is then the fraction of a turn, exact to
// |p| * 2^-65, by integer multiplication, whatever the position's size or sign.  Its upper 32 bits become the
// argument of sincospif: what remains is the 2^-24 of a 32-bit float.
#include <cmath>

#include "paged.cuh"

namespace adr {

namespace {

constexpr int ROPE_THREADS = 256;
constexpr int ROPE_MAX_HD = 256;

struct RopePlan {
  const unsigned long long* turns;  // [rotary / 2]
  int rotary;
  float amplitude;
  int head_dim;
};

struct Strided {  // [tokens, heads, head_dim], unit innermost stride
  long long token, head;
};

__device__ __forceinline__ float2 turn_at(const RopePlan& r, int pair, int position) {
  const unsigned long long a = (unsigned long long)(long long)position * __ldg(r.turns + pair);
  float s, c;
  sincospif((float)(int)(a >> 32) * 0x1p-31f, &s, &c);
  return make_float2(c * r.amplitude, s * r.amplitude);
}

__device__ __forceinline__ void turn_pair(__half& a, __half& b, float2 w) {
  const float x = __half2float(a), y = __half2float(b);
  a = __float2half_rn(x * w.x - y * w.y);
  b = __float2half_rn(y * w.x + x * w.y);
}

// A unit is what one thread rotates at once: 16-byte pieces (one with its pairs inside, or the piece of the first
// and that of the second half) where VEC, single pairs otherwise; behind the rotated units come those copied.
template <bool HALF, bool VEC>
struct Unit {
  static constexpr int PAIRS = VEC ? (HALF ? 8 : 4) : 1;
  static constexpr int COPY = VEC ? 8 : 1;
  __host__ __device__ static int rotated(int rotary) { return rotary / (2 * PAIRS); }
  __host__ __device__ static int count(int rotary, int head_dim) {
    return rotated(rotary) + (head_dim - rotary) / COPY;
  }
  struct Data {
    uint4 a, b;
  };
  __device__ static Data load(const __half* head, int u, const RopePlan& r) {
    Data d;
    const int nr = rotated(r.rotary);
    if constexpr (VEC) {
      if (u >= nr) {
        d.a = *reinterpret_cast<const uint4*>(head + r.rotary + (u - nr) * 8);
      } else {
        d.a = *reinterpret_cast<const uint4*>(head + u * 8);
        if constexpr (HALF) d.b = *reinterpret_cast<const uint4*>(head + r.rotary / 2 + u * 8);
      }
    } else {
      const unsigned short* h = reinterpret_cast<const unsigned short*>(head);
      if (u >= nr) {
        d.a.x = h[r.rotary + (u - nr)];
      } else {
        d.a.x = h[HALF ? u : 2 * u];
        d.b.x = h[HALF ? u + r.rotary / 2 : 2 * u + 1];
      }
    }
    return d;
  }
  __device__ static void store(__half* head, int u, const RopePlan& r, Data d, const float2* turns) {
    const int nr = rotated(r.rotary);
    if constexpr (VEC) {
      if (u >= nr) {
        *reinterpret_cast<uint4*>(head + r.rotary + (u - nr) * 8) = d.a;
        return;
      }
      __half* x = reinterpret_cast<__half*>(&d.a);
      __half* y = reinterpret_cast<__half*>(&d.b);
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        const float2 w = turns[u * PAIRS + i];
        if constexpr (HALF) turn_pair(x[i], y[i], w);
        else turn_pair(x[2 * i], x[2 * i + 1], w);
      }
      *reinterpret_cast<uint4*>(head + u * 8) = d.a;
      if constexpr (HALF) *reinterpret_cast<uint4*>(head + r.rotary / 2 + u * 8) = d.b;
    } else {
      if (u >= nr) {
        head[r.rotary + (u - nr)] = __ushort_as_half((unsigned short)d.a.x);
        return;
      }
      __half x = __ushort_as_half((unsigned short)d.a.x), y = __ushort_as_half((unsigned short)d.b.x);
      turn_pair(x, y, turns[u]);
      head[HALF ? u : 2 * u] = x;
      head[HALF ? u + r.rotary / 2 : 2 * u + 1] = y;
    }
  }
};

// Rotates `heads` heads of one row, src to dst (which may be the same), with the turns in shared memory.
template <bool HALF, bool VEC>
__device__ __forceinline__ void rotate_heads(__half* dst, long long dst_head, const __half* src, long long src_head,
                                             int heads, const RopePlan& r, const float2* turns) {
  using U = Unit<HALF, VEC>;
  const int n = heads * U::count(r.rotary, r.head_dim), per = U::count(r.rotary, r.head_dim);
  for (int i = threadIdx.x; i < n; i += ROPE_THREADS) {
    const int h = i / per, u = i - h * per;
    U::store(dst + h * dst_head, u, r, U::load(src + h * src_head, u, r), turns);
  }
}

__device__ __forceinline__ void fill_turns(float2* turns, const RopePlan& r, int position) {
  for (int i = threadIdx.x; i < r.rotary / 2; i += ROPE_THREADS) turns[i] = turn_at(r, i, position);
  __syncthreads();
}

// One row per block.
template <bool HALF, bool VEC>
__global__ void __launch_bounds__(ROPE_THREADS)
    rope_kernel(__half* out, const __half* in, Strided so, Strided si, int heads, const int* positions, RopePlan r) {
  __shared__ float2 turns[ROPE_MAX_HD / 2];
  pdl_wait_trigger();
  const long long t = blockIdx.x;
  fill_turns(turns, r, __ldg(positions + t));
  rotate_heads<HALF, VEC>(out + t * so.token, so.head, in + t * si.token, si.head, heads, r, turns);
}

struct PagePool {
  __half* base;
  long long page, token, head;
};

struct AppendParams {
  __half* q_out;
  const __half *q, *k, *v;
  Strided sqo, sq, sk, sv;
  PagePool kp, vp;
  const int *block_table, *cu_q, *kv_len;
  int tokens, n_seqs, heads, kv_heads, max_pages, page_size, n_pages;
  RopePlan r;
  unsigned int* status;
};

template <bool HALF, bool VEC>
__global__ void __launch_bounds__(ROPE_THREADS) rope_append_kernel(AppendParams p) {
  __shared__ float2 turns[ROPE_MAX_HD / 2];
  pdl_wait_trigger();
  const int t = blockIdx.x;
  const int s = find_sequence(p.cu_q, p.n_seqs, t, threadIdx.x & 31);
  if (s >= p.n_seqs) return;  // rows behind the last sequence
  const SeqSpan span = seq_span(p.cu_q, nullptr, s, p.tokens, 0, p.status);
  if (t < span.q0 || t >= span.q0 + span.lq) return;
  const int position = __ldg(p.kv_len + s) - span.lq + (t - span.q0);
  fill_turns(turns, p.r, position);
  rotate_heads<HALF, VEC>(p.q_out + t * p.sqo.token, p.sqo.head, p.q + t * p.sq.token, p.sq.head, p.heads, p.r, turns);
  int page = -1;
  if (position >= 0 && position / p.page_size < p.max_pages)
    page = __ldg(p.block_table + (long long)s * p.max_pages + position / p.page_size);
  if (page < 0 || page >= p.n_pages) {
    if (threadIdx.x == 0) atomicOr(p.status, PAGED_BAD);
    return;
  }
  const int slot = position % p.page_size;
  __half* kd = p.kp.base + page * p.kp.page + slot * p.kp.token;
  __half* vd = p.vp.base + page * p.vp.page + slot * p.vp.token;
  rotate_heads<HALF, VEC>(kd, p.kp.head, p.k + t * p.sk.token, p.sk.head, p.kv_heads, p.r, turns);
  RopePlan copy = p.r;
  copy.rotary = 0;
  rotate_heads<HALF, VEC>(vd, p.vp.head, p.v + t * p.sv.token, p.sv.head, p.kv_heads, copy, turns);
}

template <typename... KArgs, typename... Args>
int launch_rows(adr_ctx* ctx, cudaStream_t stream, void (*kfn)(KArgs...), int rows, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows);
  cfg.blockDim = dim3(ROPE_THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ctx->tune_pdl.load() ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kfn, static_cast<KArgs>(args)...);
  if (e != cudaSuccess) {
    ctx->last_cuda_error = (int)e;
    return ADR_ERR_CUDA;
  }
  // (as for the other row kernels: with a block per SM and more it fills the GPU)
  if (rows >= ctx->sm_count) note_filling_launch(ctx, stream, 4);
  else ctx->small_before = 1;
  return after_launch(ctx);
}

int check_rotation(const uint64_t* turns, int head_dim, int rotary_dim, float amplitude, uint32_t layout) {
  if (!turns || head_dim <= 0 || rotary_dim <= 0 || layout > ADR_ROPE_HALF) return ADR_ERR_INVALID;
  if (!std::isfinite(amplitude)) return ADR_ERR_INVALID;
  if (rotary_dim % 2 != 0 || rotary_dim > head_dim || head_dim > ROPE_MAX_HD) return ADR_ERR_SHAPE;
  return ADR_OK;
}

int check_strides(const long long* s, int n) {
  if (!s) return ADR_ERR_INVALID;
  for (int i = 0; i < n; ++i)
    if (s[i] < 0) return ADR_ERR_INVALID;
  return ADR_OK;
}

// 16-byte pieces: every row and head starts on one, and so does every part of a head
bool in_pieces(const void* p, const long long* s, int n) {
  if (reinterpret_cast<uintptr_t>(p) & 15u) return false;
  for (int i = 0; i < n; ++i)
    if (s[i] % 8 != 0) return false;
  return true;
}
bool parts_in_pieces(int head_dim, int rotary_dim, uint32_t layout) {
  return head_dim % 8 == 0 && rotary_dim % (layout == ADR_ROPE_HALF ? 16 : 8) == 0;
}

}  // namespace

}  // namespace adr

using namespace adr;

extern "C" int adr_rope_turns(uint64_t* turns, float* amplitude, int rotary_dim, double theta, uint32_t scaling,
                              double factor, double original, double low, double high) {
  if (!turns || !amplitude || rotary_dim <= 0 || scaling > ADR_ROPE_SCALE_YARN) return ADR_ERR_INVALID;
  if (rotary_dim % 2 != 0) return ADR_ERR_SHAPE;
  if (!(theta > 1.0) || !std::isfinite(theta)) return ADR_ERR_INVALID;
  if (scaling != ADR_ROPE_SCALE_NONE && (!(factor >= 1.0) || !std::isfinite(factor))) return ADR_ERR_INVALID;
  if (scaling == ADR_ROPE_SCALE_BASE && rotary_dim < 4) return ADR_ERR_SHAPE;
  if (scaling == ADR_ROPE_SCALE_BANDS || scaling == ADR_ROPE_SCALE_YARN) {
    if (!(original > 0.0) || !(low > 0.0) || !(high > low) || !std::isfinite(original) || !std::isfinite(high))
      return ADR_ERR_INVALID;
  }
  // long double: 64 bits of mantissa, one more than the fraction keeps of the first pair's
  const long double two_pi = 2.0L * acosl(-1.0L);
  const long double d = rotary_dim, s = factor, L = original;
  long double base = theta;
  if (scaling == ADR_ROPE_SCALE_BASE) base *= powl(s, d / (d - 2));
  // YaRN: the pairs that turn `high` and `low` times within the original context bound the ramp
  long double ramp_lo = 0, ramp_hi = 0;
  if (scaling == ADR_ROPE_SCALE_YARN) {
    auto pair_of = [&](long double n) { return d * logl(L / (n * two_pi)) / (2 * logl(base)); };
    ramp_lo = fmaxl(floorl(pair_of(high)), 0);
    ramp_hi = fminl(ceill(pair_of(low)), d - 1);
    if (ramp_hi - ramp_lo < 0.001L) ramp_hi = ramp_lo + 0.001L;
  }
  for (int i = 0; i < rotary_dim / 2; ++i) {
    long double f = powl(base, -2.0L * i / d);
    if (scaling == ADR_ROPE_SCALE_LINEAR) {
      f /= s;
    } else if (scaling == ADR_ROPE_SCALE_BANDS) {
      const long double n = L * f / two_pi;  // turns within the original context
      const long double w = fminl(1, fmaxl(0, (n - low) / ((long double)high - low)));
      f = f / s * (1 - w) + f * w;
    } else if (scaling == ADR_ROPE_SCALE_YARN) {
      const long double w = fminl(1, fmaxl(0, (i - ramp_lo) / (ramp_hi - ramp_lo)));
      f = f / s * w + f * (1 - w);
    }
    turns[i] = (uint64_t)(f / two_pi * 0x1p64L);  // f <= 1: below 2^62
  }
  *amplitude = scaling == ADR_ROPE_SCALE_YARN ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
  return ADR_OK;
}

extern "C" int adr_rope_f16(adr_ctx* ctx, adr_stream stream, void* out, const void* in, int tokens, int n_heads,
                            int head_dim, const long long* strides_o, const long long* strides_i,
                            const int32_t* positions, const uint64_t* turns, int rotary_dim, float amplitude,
                            uint32_t layout) {
  if (!out || !in || !positions || tokens <= 0 || n_heads <= 0) return ADR_ERR_INVALID;
  if (int rc = check_rotation(turns, head_dim, rotary_dim, amplitude, layout); rc != ADR_OK) return rc;
  if (check_strides(strides_o, 2) != ADR_OK || check_strides(strides_i, 2) != ADR_OK) return ADR_ERR_INVALID;
  if ((long long)n_heads * head_dim > (1 << 30)) return ADR_ERR_SHAPE;
  if (!ctx) return ADR_ERR_INVALID;
  DeviceGuard guard(ctx);
  const bool vec = parts_in_pieces(head_dim, rotary_dim, layout) && in_pieces(out, strides_o, 2) &&
                   in_pieces(in, strides_i, 2);
  const RopePlan r{reinterpret_cast<const unsigned long long*>(turns), rotary_dim, amplitude, head_dim};
  const Strided so{strides_o[0], strides_o[1]}, si{strides_i[0], strides_i[1]};
  auto kfn = layout == ADR_ROPE_HALF ? (vec ? rope_kernel<true, true> : rope_kernel<true, false>)
                                     : (vec ? rope_kernel<false, true> : rope_kernel<false, false>);
  return launch_rows(ctx, (cudaStream_t)stream, kfn, tokens, (__half*)out, (const __half*)in, so, si, n_heads,
                     (const int*)positions, r);
}

extern "C" int adr_rope_append_paged(adr_ctx* ctx, adr_stream stream, void* q_out, const void* q, const void* k,
                                     const void* v, void* k_pages, void* v_pages, int tokens, int n_seqs,
                                     int n_heads, int n_kv_heads, int head_dim, const long long* strides_qo,
                                     const long long* strides_q, const long long* strides_k,
                                     const long long* strides_v, const long long* strides_kp,
                                     const long long* strides_vp, const int32_t* block_table, const int32_t* cu_q,
                                     const int32_t* kv_len, int max_pages, int page_size, int n_pages,
                                     const uint64_t* turns, int rotary_dim, float amplitude, uint32_t layout) {
  if (!q_out || !q || !k || !v || !k_pages || !v_pages || !block_table || !cu_q || !kv_len) return ADR_ERR_INVALID;
  if (tokens <= 0 || n_seqs <= 0 || n_heads <= 0 || n_kv_heads <= 0 || max_pages <= 0 || page_size <= 0 || n_pages <= 0)
    return ADR_ERR_INVALID;
  if (int rc = check_rotation(turns, head_dim, rotary_dim, amplitude, layout); rc != ADR_OK) return rc;
  const long long* rows[4] = {strides_qo, strides_q, strides_k, strides_v};
  for (const long long* s : rows)
    if (check_strides(s, 2) != ADR_OK) return ADR_ERR_INVALID;
  if (check_strides(strides_kp, 3) != ADR_OK || check_strides(strides_vp, 3) != ADR_OK) return ADR_ERR_INVALID;
  if (((long long)n_heads + n_kv_heads) * head_dim > (1 << 30)) return ADR_ERR_SHAPE;
  if (!ctx) return ADR_ERR_INVALID;
  DeviceGuard guard(ctx);
  const bool vec = parts_in_pieces(head_dim, rotary_dim, layout) && in_pieces(q_out, strides_qo, 2) &&
                   in_pieces(q, strides_q, 2) && in_pieces(k, strides_k, 2) && in_pieces(v, strides_v, 2) &&
                   in_pieces(k_pages, strides_kp, 3) && in_pieces(v_pages, strides_vp, 3);
  AppendParams p;
  p.q_out = (__half*)q_out;
  p.q = (const __half*)q;
  p.k = (const __half*)k;
  p.v = (const __half*)v;
  p.sqo = {strides_qo[0], strides_qo[1]};
  p.sq = {strides_q[0], strides_q[1]};
  p.sk = {strides_k[0], strides_k[1]};
  p.sv = {strides_v[0], strides_v[1]};
  p.kp = {(__half*)k_pages, strides_kp[0], strides_kp[1], strides_kp[2]};
  p.vp = {(__half*)v_pages, strides_vp[0], strides_vp[1], strides_vp[2]};
  p.block_table = block_table;
  p.cu_q = cu_q;
  p.kv_len = kv_len;
  p.tokens = tokens;
  p.n_seqs = n_seqs;
  p.heads = n_heads;
  p.kv_heads = n_kv_heads;
  p.max_pages = max_pages;
  p.page_size = page_size;
  p.n_pages = n_pages;
  p.r = {reinterpret_cast<const unsigned long long*>(turns), rotary_dim, amplitude, head_dim};
  p.status = ctx->d_status;
  auto kfn = layout == ADR_ROPE_HALF ? (vec ? rope_append_kernel<true, true> : rope_append_kernel<true, false>)
                                     : (vec ? rope_append_kernel<false, true> : rope_append_kernel<false, false>);
  return launch_rows(ctx, (cudaStream_t)stream, kfn, tokens, p);
}
