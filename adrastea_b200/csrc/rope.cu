// Rotary positions of packed rows: pairs (2i, 2i + 1) or (i, i + d/2), all or the first part of a head, angles
// scaled for long contexts; alone, or for the new tokens of sequences whose k and v go to a paged cache.
//
// The angle of pair i at position p is p * f_i.  A 32-bit f_i would lose it at far positions (2^-24 relative of
// 10^6 radians), and a 64-bit product costs the GPU's few fp64 units.  So the table holds f_i / (2 pi), the turns
// per position, as a 64-bit fixed-point fraction (cut off); p times it modulo 2^64 is then the fraction of a turn, off by
// |p| * 2^-64 at most, by integer multiplication, whatever the position's size or sign.  Its upper 32 bits become the
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
  __device__ static void store(__half* head, int u, const RopePlan& r, Data d, const float2 (&turns)[PAIRS]) {
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
        const float2 w = turns[i];
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
      turn_pair(x, y, turns[0]);
      head[HALF ? u : 2 * u] = x;
      head[HALF ? u + r.rotary / 2 : 2 * u + 1] = y;
    }
  }
};

// A block takes R rows.  With one row each (few rows: latency counts) a thread's first piece is on its way while it is
// looked up where the row stands, a chain of two or three loads of about a microsecond each; with four the chain and the
// 64 or so turns of each row are computed by as many threads as there are turns, and each row has two warps of its own.
// (Single columns, not 16-byte pieces: one row, whose units can be more than two warps.)
constexpr int ROPE_FEW = 1, ROPE_MANY = 4;

// The place of thread `id` of a row's `threads`: unit u of heads h, h + step, ...  (threads that do not make up a whole
// head are idle)
struct Place {
  int u, h, step;
  __device__ Place(int per, int id, int threads) : u(id % per), h(id / per), step(threads / per) {
    if (h >= step) h = 1 << 30;
  }
};

// The heads from `at.h` on of one row, two at a time: src_of and dst_of give a head's columns.
template <bool HALF, bool VEC, typename Src, typename Dst>
__device__ __forceinline__ void turn_heads(const Place& at, int h, int heads, const RopePlan& r, const float2* turns,
                                           const Src& src_of, const Dst& dst_of) {
  using U = Unit<HALF, VEC>;
  float2 w[U::PAIRS];
  if (at.u < U::rotated(r.rotary) && h < heads) {
#pragma unroll
    for (int i = 0; i < U::PAIRS; ++i) w[i] = turns[at.u * U::PAIRS + i];
  }
  for (; h < heads; h += 2 * at.step) {
    const bool two = h + at.step < heads;
    typename U::Data a = U::load(src_of(h), at.u, r), b;
    if (two) b = U::load(src_of(h + at.step), at.u, r);
    U::store(dst_of(h), at.u, r, a, w);
    if (two) U::store(dst_of(h + at.step), at.u, r, b, w);
  }
}
template <bool HALF, bool VEC>
__device__ __forceinline__ void turn_one(const Place& at, const RopePlan& r, const float2* turns,
                                         const typename Unit<HALF, VEC>::Data& d, __half* dst) {
  using U = Unit<HALF, VEC>;
  float2 w[U::PAIRS];
#pragma unroll
  for (int i = 0; i < U::PAIRS; ++i) w[i] = at.u < U::rotated(r.rotary) ? turns[at.u * U::PAIRS + i] : make_float2(1.0f, 0.0f);
  U::store(dst, at.u, r, d, w);
}

// The turns of R rows, by as many threads as there are.
template <int R>
__device__ __forceinline__ void fill_turns(float2 (*turns)[ROPE_MAX_HD / 2], const RopePlan& r, const int* position) {
  const int n = r.rotary / 2;
  for (int i = threadIdx.x; i < R * n; i += ROPE_THREADS) turns[i / n][i % n] = turn_at(r, i % n, position[i / n]);
  __syncthreads();
}

// Bound by memory where rows are many (8000 rows of 64 heads of 128: 44 us, 5.9 TB/s).  A block is over in a few chains of
// loads, so what counts is how many an SM holds: four of the halves (64 registers; at 72 there are three: 4111 rows of 40
// heads 19.1 against 21.6 us), five of the interleaved (48).
template <bool HALF, bool VEC, int R>
__global__ void __launch_bounds__(ROPE_THREADS, HALF ? 4 : 5)
    rope_kernel(__half* out, const __half* in, Strided so, Strided si, int rows, int heads, const int* positions, RopePlan r) {
  using U = Unit<HALF, VEC>;
  __shared__ float2 turns[R][ROPE_MAX_HD / 2];
  __shared__ int position[R];
  pdl_wait_trigger();
  constexpr int ROW_THREADS = ROPE_THREADS / R;
  const int i = threadIdx.x / ROW_THREADS;  // this thread's row
  const Place at(U::count(r.rotary, r.head_dim), threadIdx.x % ROW_THREADS, ROW_THREADS);
  const long long t0 = (long long)blockIdx.x * R;
  typename U::Data ahead;
  if (R == 1 && at.h < heads) ahead = U::load(in + t0 * si.token + at.h * si.head, at.u, r);
  if (threadIdx.x < R) position[threadIdx.x] = __ldg(positions + min(t0 + threadIdx.x, (long long)rows - 1));
  __syncthreads();
  fill_turns<R>(turns, r, position);
  if (t0 + i >= rows) return;
  const __half* src = in + (t0 + i) * si.token;
  __half* dst = out + (t0 + i) * so.token;
  if (R == 1 && at.h < heads) turn_one<HALF, VEC>(at, r, turns[i], ahead, dst + at.h * so.head);
  turn_heads<HALF, VEC>(at, at.h + (R == 1 ? at.step : 0), heads, r, turns[i], [&](int h) { return src + h * si.head; },
                        [&](int h) { return dst + h * so.head; });
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

// Four blocks to an SM, 64 registers (8000 rows of 32/8 heads: 66 us against 74 at 72 registers).  Bound by memory: 5.7 TB/s
// of rows read and written, of 6.55.
template <bool HALF, bool VEC, int R>
__global__ void __launch_bounds__(ROPE_THREADS, 4) rope_append_kernel(const __grid_constant__ AppendParams p) {
  using U = Unit<HALF, VEC>;
  __shared__ float2 turns[R][ROPE_MAX_HD / 2];
  __shared__ int position[R], page_of[R];  // page: below 0 there is none, below -1 the row is no sequence's
  pdl_wait_trigger();
  const RopePlan& r = p.r;
  RopePlan copy = r;
  copy.rotary = 0;
  constexpr int ROW_THREADS = ROPE_THREADS / R;
  const int i = threadIdx.x / ROW_THREADS, in_row = threadIdx.x % ROW_THREADS;  // this thread's row
  const Place at(U::count(r.rotary, r.head_dim), in_row, ROW_THREADS), at_v(U::count(0, r.head_dim), in_row, ROW_THREADS);
  const int t0 = blockIdx.x * R, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, heads = p.heads + p.kv_heads;
  // query heads, then key heads
  auto head_src = [&](long long t, int h) {
    return h < p.heads ? p.q + t * p.sq.token + h * p.sq.head : p.k + t * p.sk.token + (h - p.heads) * p.sk.head;
  };
  typename U::Data ahead;
  if (R == 1 && at.h < heads) ahead = U::load(head_src(t0, at.h), at.u, r);
  // a warp looks up one row
  if (warp < R) {
    const int t = t0 + warp;
    int at_position = 0, page = -2;
    const int s = t < p.tokens ? find_sequence(p.cu_q, p.n_seqs, t, lane) : p.n_seqs;
    if (s < p.n_seqs) {
      const int positions = __ldg(p.kv_len + s);
      const SeqSpan span = seq_span(p.cu_q, nullptr, s, p.tokens, 0, p.status);
      if (t >= span.q0 && t < span.q0 + span.lq) {
        at_position = positions - span.lq + (t - span.q0);
        page = -1;
        if (at_position >= 0 && at_position / p.page_size < p.max_pages)
          page = __ldg(p.block_table + (long long)s * p.max_pages + at_position / p.page_size);
        if (page < 0 || page >= p.n_pages) {
          page = -1;
          if (lane == 0) atomicOr(p.status, PAGED_BAD);
        }
      }
    }
    if (lane == 0) position[warp] = at_position, page_of[warp] = page;
  }
  __syncthreads();
  fill_turns<R>(turns, r, position);
  const long long t = t0 + i;
  const int page = page_of[i];
  if (page < -1) return;
  const int slot = position[i] % p.page_size;
  __half* qd = p.q_out + t * p.sqo.token;
  __half* kd = p.kp.base + (page >= 0 ? page * p.kp.page + slot * p.kp.token : 0);
  __half* vd = p.vp.base + (page >= 0 ? page * p.vp.page + slot * p.vp.token : 0);
  const int n = page >= 0 ? heads : p.heads;  // (without a page only the queries)
  auto head_dst = [&](int h) { return h < p.heads ? qd + h * p.sqo.head : kd + (h - p.heads) * p.kp.head; };
  if (R == 1 && at.h < n) turn_one<HALF, VEC>(at, r, turns[i], ahead, head_dst(at.h));
  turn_heads<HALF, VEC>(at, at.h + (R == 1 ? at.step : 0), n, r, turns[i], [&](int h) { return head_src(t, h); }, head_dst);
  const __half* vs = p.v + t * p.sv.token;
  turn_heads<HALF, VEC>(at_v, at_v.h, page >= 0 ? p.kv_heads : 0, copy, turns[i], [&](int h) { return vs + h * p.sv.head; },
                        [&](int h) { return vd + h * p.vp.head; });
}

// (as for the other row kernels: with a block per SM and more it fills the GPU)
template <typename K, typename... Args>
int launch_rows(adr_ctx* ctx, cudaStream_t stream, K kfn, int blocks, const Args&... args) {
  const bool fills = blocks >= ctx->sm_count;
  if (int rc = launch_serving(ctx, stream, kfn, dim3(blocks), ROPE_THREADS, 0, fills ? 4 : 0, args...); rc != ADR_OK) return rc;
  if (!fills) ctx->small_before = 1;
  return ADR_OK;
}

// From two rows to an SM on they go four to a block (600 rows of 32/8 heads: 5.7 against 8.3 us; 148 rows would take 4.0 either
// way, and below that the single rows' first loads are worth more).
bool many_rows(const adr_ctx* ctx, int rows) { return rows >= 2 * ctx->sm_count; }

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
  if (!on_elements((const __half*)out, (const __half*)in, positions, turns)) return ADR_ERR_SHAPE;
  if (!ctx) return ADR_ERR_INVALID;
  DeviceGuard guard(ctx);
  const bool vec = parts_in_pieces(head_dim, rotary_dim, layout) && in_pieces(out, strides_o, 2) &&
                   in_pieces(in, strides_i, 2);
  const RopePlan r{reinterpret_cast<const unsigned long long*>(turns), rotary_dim, amplitude, head_dim};
  const Strided so{strides_o[0], strides_o[1]}, si{strides_i[0], strides_i[1]};
  auto go = [&](auto kfn, int per) {
    return launch_rows(ctx, (cudaStream_t)stream, kfn, (tokens - 1) / per + 1, (__half*)out, (const __half*)in, so, si,
                       tokens, n_heads, (const int*)positions, r);
  };
  const bool many = vec && many_rows(ctx, tokens), half = layout == ADR_ROPE_HALF;
  if (many) return half ? go(rope_kernel<true, true, ROPE_MANY>, ROPE_MANY) : go(rope_kernel<false, true, ROPE_MANY>, ROPE_MANY);
  if (vec) return half ? go(rope_kernel<true, true, ROPE_FEW>, ROPE_FEW) : go(rope_kernel<false, true, ROPE_FEW>, ROPE_FEW);
  return half ? go(rope_kernel<true, false, ROPE_FEW>, ROPE_FEW) : go(rope_kernel<false, false, ROPE_FEW>, ROPE_FEW);
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
  if (!on_elements((const __half*)q_out, (const __half*)q, (const __half*)k, (const __half*)v, (const __half*)k_pages,
                   (const __half*)v_pages, block_table, cu_q, kv_len, turns))
    return ADR_ERR_SHAPE;
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
  auto go = [&](auto kfn, int per) { return launch_rows(ctx, (cudaStream_t)stream, kfn, (tokens - 1) / per + 1, p); };
  const bool many = vec && many_rows(ctx, tokens), half = layout == ADR_ROPE_HALF;
  if (many)
    return half ? go(rope_append_kernel<true, true, ROPE_MANY>, ROPE_MANY)
                : go(rope_append_kernel<false, true, ROPE_MANY>, ROPE_MANY);
  if (vec)
    return half ? go(rope_append_kernel<true, true, ROPE_FEW>, ROPE_FEW)
                : go(rope_append_kernel<false, true, ROPE_FEW>, ROPE_FEW);
  return half ? go(rope_append_kernel<true, false, ROPE_FEW>, ROPE_FEW)
              : go(rope_append_kernel<false, false, ROPE_FEW>, ROPE_FEW);
}
