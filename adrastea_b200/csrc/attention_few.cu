// Attention of a few new rows per sequence over a paged cache: single tokens, and a few at a time.
//
// The rows of one key head (its query heads times the new tokens, up to 64) share every key and value, so one pass
// over the cache serves them all: what bounds this kernel is reading the cache once.
//   * Work is counted in units of 64 keys of one (sequence, key head, tile of rows).  Every CTA computes from the
//     lengths on the device where the 1/Gth part of all units that is its own begins, so the cache of a batch of very
//     different lengths, or of one long sequence, is spread evenly over the SMs with no plan from the host.
//   * A producer warp copies pages by TMA into a ring of stages (64 keys and values), across the borders of items.
//   * Four warps compute: S = Q K^T and O += P V by mma.sync m16n8k16 with the 16 (32, 64) rows as M and a running
//     maximum and sum.  (tcgen05 wants 64 or 128 rows: at up to 16 live ones the tensor work is 5 % of the time that
//     the keys take to arrive.)  With 16 rows the warps share a stage's keys, with 64 its rows.
//   * An item that lies within one CTA is finished there.  Otherwise each part stores its maximum, sum and unscaled
//     output, and the CTA that arrives last (a counter per border) joins the parts in their order: same bits each run.
#include <algorithm>

#include "attention_seqs.cuh"

namespace adr {

namespace {

constexpr int FEW_KB = 64;          // keys of a stage, and of a unit of work
constexpr int FEW_THREADS = 160;    // four computing warps and the producer
constexpr int FEW_MAX_ROWS = 64;

template <int HD, int WM>
struct FewCfg {
  static constexpr int ROWS = 16 * WM;
  static constexpr int WK = 4 / WM;             // warps that share a stage's keys
  static constexpr int KEYS = FEW_KB / WK;      // of a stage, for one warp
  static constexpr int CH = HD / 64;            // 64-column chunks of a head
  static constexpr int TILE = FEW_KB * HD * 2;  // bytes of a stage's keys
  static constexpr int STAGES = HD == 128 ? 3 : 6;
  static constexpr int MERGE = WK == 1 ? 0 : 4 * (HD / 8) * 32 * 8;  // eight rows of every warp
  static constexpr size_t SMEM = (size_t)STAGES * 2 * TILE + MERGE + 4 * 16 * 8 + 16 * STAGES + 160;
};

struct FewParams {
  SeqAttention a;
  int max_rows;  // sequences with more rows of a key head than this are left to another kernel
  int page_rows; // rows of a copy: a page, 64 at most
  int min_units; // of a CTA, where there are few
  float* part_ml;
  float* part_o;
  unsigned int* counters;
};

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Nonzero if one of the two halves is infinite or not a number (its exponent bits are all ones: adding one to them
// carries into the sign, which was masked away).
__device__ __forceinline__ uint32_t not_finite2(uint32_t x) { return ((x & 0x7C007C00u) + 0x04000400u) & 0x80008000u; }
// The computing warps only.
__device__ __forceinline__ void few_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// Where in the list of all units (sequence by sequence, key head by key head, tile by tile, 64 keys each) a CTA is.
struct Walk {
  SeqSpan span;
  int s, head, tile, blk;
  int tiles, blks;
};

// How the units are shared out: CTA c begins with unit begin(c).
struct Share {
  long long per;
  int ctas, more;
  __device__ long long begin(int c) const { return c * per + min(c, more); }
  __device__ int owner(long long u) const {
    const long long big = more * (per + 1);
    return u < big ? (int)(u / (per + 1)) : more + (int)((u - big) / per);
  }
};

template <int ROWS>
struct FewWork {
  const FewParams& p;
  __device__ explicit FewWork(const FewParams& p_) : p(p_) {}
  __device__ SeqSpan span(int s) const {
    return seq_span(p.a.cu_q, p.a.kv_len, s, p.a.tokens, p.a.max_pages * p.a.page_size, p.a.status);
  }
  __device__ int tiles(const SeqSpan& v) const {
    const long long rows = (long long)v.lq * p.a.group;
    return rows > p.max_rows ? 0 : (int)((rows + ROWS - 1) / ROWS);
  }
  __device__ static int blocks(const SeqSpan& v) { return max(1, (v.lk + FEW_KB - 1) / FEW_KB); }
  __device__ long long units(int s) const {
    if (s >= p.a.n_seqs) return 0;
    const SeqSpan v = span(s);
    return (long long)tiles(v) * blocks(v) * p.a.n_kv_heads;
  }
  // by a whole warp
  __device__ long long total(int lane) const {
    long long n = 0;
    for (int s = lane; s < p.a.n_seqs; s += 32) n += units(s);
    for (int d = 16; d > 0; d >>= 1) n += __shfl_xor_sync(0xffffffffu, n, d);
    return n;
  }
  __device__ void enter(Walk& w, int s) const {
    w.s = s;
    w.span = span(s);
    w.tiles = tiles(w.span);
    w.blks = blocks(w.span);
  }
  // Unit u of all, by a whole warp.  (The loops over sequences end behind the last one whatever the arrays hold; no
  // tiles: there is no such unit.)
  __device__ Walk find(long long u, int lane) const {
    Walk w = {};
    for (int s0 = 0; s0 < p.a.n_seqs; s0 += 32) {
      const long long mine = units(s0 + lane);
      long long upto = mine;
      for (int d = 1; d < 32; d <<= 1) {
        const long long o = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += o;
      }
      const unsigned m = __ballot_sync(0xffffffffu, u < upto);
      if (m) {
        const int l = __ffs(m) - 1;
        const long long rest = u - __shfl_sync(0xffffffffu, upto - mine, l);
        enter(w, s0 + l);
        w.head = (int)(rest / ((long long)w.tiles * w.blks));
        const int in_head = (int)(rest - (long long)w.head * w.tiles * w.blks);
        w.tile = in_head / w.blks;
        w.blk = in_head - w.tile * w.blks;
        return w;
      }
      u -= __shfl_sync(0xffffffffu, upto, 31);
    }
    return w;
  }
  // the item behind w's; no tiles: there is none
  __device__ void next(Walk& w) const {
    w.blk = 0;
    if (++w.tile < w.tiles) return;
    w.tile = 0;
    if (++w.head < p.a.n_kv_heads) return;
    w.head = 0;
    w.tiles = 0;
    for (int s = w.s + 1; s < p.a.n_seqs && w.tiles == 0; ++s) enter(w, s);
  }
};

template <int HD, int WM>
__global__ void __launch_bounds__(FEW_THREADS, 2)
    attention_few_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                         const __grid_constant__ FewParams p) {
  using Cfg = FewCfg<HD, WM>;
  constexpr int STAGES = Cfg::STAGES, WK = Cfg::WK, NT = HD / 8;
  extern __shared__ __align__(1024) uint8_t few_smem[];  // (the swizzle's atoms begin on 1024 bytes)
  uint8_t* ring = few_smem;
  float2* merge = reinterpret_cast<float2*>(ring + (size_t)STAGES * 2 * Cfg::TILE);   // [4 warps][NT][32]
  float2* ml = merge + Cfg::MERGE / 8;                                                // [4 warps][16 rows]
  uint64_t* full = reinterpret_cast<uint64_t*>(ml + 4 * 16);
  uint64_t* empty = full + STAGES;
  long long& s_total = *reinterpret_cast<long long*>(empty + STAGES);
  volatile unsigned int& s_last = *reinterpret_cast<unsigned int*>(empty + STAGES + 1);
  Walk* s_walk = reinterpret_cast<Walk*>(empty + STAGES + 2);  // [3]: the first item, then alternately the next ones
  static_assert(sizeof(Walk) * 3 + 16 <= 160, "what a CTA's warps share");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 4);
    }
    mbar_fence_init();
  }
  pdl_wait_trigger();

  // One warp looks up what is to be done, so that the warps that meet at barriers agree on it whatever happens to
  // the arrays meanwhile.  No more CTAs than units; the first `total % ctas` CTAs have one unit more than the others.
  const FewWork<Cfg::ROWS> work(p);
  auto share_of = [&](long long n) {
    Share r;
    r.ctas = (int)min((long long)gridDim.x, (n + p.min_units - 1) / p.min_units);
    r.per = r.ctas ? n / r.ctas : 0;
    r.more = (int)(n - r.per * r.ctas);
    return r;
  };
  if (warp == 0) {
    const long long n = work.total(lane);
    const Share sh = share_of(n);
    Walk f = {};
    if ((int)blockIdx.x < sh.ctas) f = work.find(sh.begin(blockIdx.x), lane);
    if (lane == 0) s_total = n, s_walk[2] = f;
  }
  __syncthreads();
  const Share share = share_of(s_total);
  Walk w = s_walk[2];
  if ((int)blockIdx.x >= share.ctas || w.tiles == 0) return;
  const long long u0 = share.begin(blockIdx.x), u1 = share.begin(blockIdx.x + 1);
  bool ok = true;

  if (warp == 4) {
    // ------------------------------- producer -------------------------------
    const int pr = p.page_rows, page_size = p.a.page_size;
    int st = 0;
    unsigned use = 0;
    long long issued = 0;
    for (long long u = u0; u < u1;) {
      const int last = (int)min((long long)w.blks, w.blk + (u1 - u));
      const int* row = p.a.block_table + (long long)w.s * p.a.max_pages;
      for (int b = w.blk; b < last; ++b) {
        const int keys = min(FEW_KB, w.span.lk - b * FEW_KB);
        if (keys <= 0) break;  // a sequence without positions
        const int copies = (keys + pr - 1) / pr;
        const int pos = b * FEW_KB + lane * pr;
        int page = 0;
        if (lane < copies) {
          page = __ldg(row + pos / page_size);
          if (page < 0 || page >= p.a.n_pages) {
            page = p.a.n_pages;  // outside the map: zeros arrive
            atomicOr(p.a.status, PAGED_BAD);
          }
        }
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&empty[st], (use & 1u) ^ 1u));
        if (!ok) break;
        if (lane == 0) mbar_expect_tx(&full[st], (unsigned)(copies * pr * HD * 2 * 2));
        __syncwarp();
        if (lane < copies) {
          uint8_t* k_sm = ring + (size_t)st * 2 * Cfg::TILE + lane * pr * 128;
          const int slot = pos % page_size;
#pragma unroll
          for (int c = 0; c < Cfg::CH; ++c) {
            tma_load_4d(k_sm + c * FEW_KB * 128, &map_k, c * 64, w.head, slot, page, &full[st]);
            tma_load_4d(k_sm + Cfg::TILE + c * FEW_KB * 128, &map_v, c * 64, w.head, slot, page, &full[st]);
          }
        }
        ++issued;
        if (++st == STAGES) st = 0, ++use;
      }
      if (!ok) break;
      u += last - w.blk;
      if (u < u1) work.next(w);
      if (w.tiles == 0) break;
    }
    // every copy has landed before the CTA may end
    for (long long i = max(0LL, issued - STAGES); i < issued; ++i)
      if (!mbar_wait(&full[i % STAGES], (unsigned)(i / STAGES) & 1u)) ok = false;
    if (!ok && lane == 0) atomicOr(p.a.status, 1u << 21);
    return;
  }

  // ------------------------------- computing warps -------------------------------
  const int wm = warp / WK, wk = warp % WK;
  const float scale2 = p.a.scale * 1.4426950408889634f;  // scores in powers of two
  const int quad = lane >> 2, pairc = (lane & 3) * 2;
  // ldmatrix lane addresses inside a 64-column chunk: keys by keys (K), and transposed (V)
  const int k_key = ((lane >> 4) << 3) + (lane & 7), k_col = (lane >> 3) & 1;
  const int v_key = (((lane >> 3) & 1) << 3) + (lane & 7), v_col = lane >> 4;
  // the thread's two rows of an item: how many positions they see, where their output goes; their queries
  auto rows_of = [&](const Walk& x) { return min(Cfg::ROWS, x.span.lq * p.a.group - x.tile * Cfg::ROWS); };
  auto enter = [&](const Walk& x, int (&limit)[2], __half* (&dst)[2], uint32_t (&qa)[HD / 16][4]) {
    const __half* src[2];
    const int live = rows_of(x);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = x.tile * Cfg::ROWS + min(wm * 16 + quad + 8 * i, live - 1);  // rows past the last repeat it, unstored
      const int tok = r / p.a.group, h = x.head * p.a.group + r - tok * p.a.group;
      limit[i] = max(0, x.span.lk - x.span.lq + tok + 1);
      src[i] = p.a.q + (long long)(x.span.q0 + tok) * p.a.sq[0] + h * p.a.sq[1];
      dst[i] = p.a.out + (long long)(x.span.q0 + tok) * p.a.so[0] + h * p.a.so[1];
    }
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        qa[kk][i] = *reinterpret_cast<const uint32_t*>(src[i & 1] + kk * 16 + (i >> 1) * 8 + pairc);
  };
  int st = 0, turn = 0, limit[2];
  unsigned use = 0;
  __half* dst[2];
  uint32_t qa[HD / 16][4];
  enter(w, limit, dst, qa);
  for (long long u = u0;;) {
    const int first = w.blk, last = (int)min((long long)w.blks, w.blk + (u1 - u));
    const bool more = u + (last - first) < u1;
    if (warp == 0 && more) {
      Walk n = w;
      work.next(n);
      if (lane == 0) s_walk[turn] = n;
    }
    const int lk = w.span.lk, live = rows_of(w);
    // positions that every row of the tile sees (an earlier token sees fewer)
    const int all_see = max(0, lk - w.span.lq + w.tile * Cfg::ROWS / p.a.group + 1);
    float o[NT][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[t][i] = 0.0f;

    for (int b = first; b < last && lk > 0; ++b) {
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&full[st], use & 1u));
      const uint32_t k_sm = smem_u32(ring + (size_t)st * 2 * Cfg::TILE);
      const uint32_t v_sm = k_sm + Cfg::TILE;
#pragma unroll 1
      for (int step = 0; step < Cfg::KEYS; step += 16) {
        const int kb = wk * Cfg::KEYS + step;  // of the stage
        const int key0 = b * FEW_KB + kb;      // position of its first key
        if (key0 >= lk) break;
        float s[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[t][i] = 0.0f;
        const uint32_t k_row = k_sm + (kb + k_key) * 128;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          uint32_t kf[4];
          ldsm_x4(k_row + (kk / 4) * FEW_KB * 128 + ((((kk & 3) * 2 + k_col) ^ (k_key & 7)) << 4), kf);
          mma_16816(s[0], qa[kk], kf[0], kf[1]);
          mma_16816(s[1], qa[kk], kf[2], kf[3]);
        }
        const bool partly = key0 + 16 > all_see;  // some row does not see some of these keys
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[t][i] *= scale2;
            if (partly && key0 + t * 8 + pairc + (i & 1) >= limit[i >> 1]) s[t][i] = -INFINITY;
            top[i >> 1] = fmaxf(top[i >> 1], s[t][i]);
          }
        bool moved = false;
        float use_m[2], alpha[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
          top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
          const float mn = fmaxf(m[i], top[i]);
          use_m[i] = mn == -INFINITY ? 0.0f : mn;
          alpha[i] = exp2_fast(m[i] - use_m[i]);
          moved = moved || mn != m[i];
          m[i] = mn;
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[t][i] *= alpha[i >> 1];
          l[0] *= alpha[0];
          l[1] *= alpha[1];
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[t][i] = exp2_fast(s[t][i] - use_m[i >> 1]);
            l[i >> 1] += s[t][i];
          }
        // probabilities are rounded to fp16 for the tensor cores (2^-11 of each: as much as the output's own rounding)
        const uint32_t pa[4] = {pack_half2(s[0][0], s[0][1]), pack_half2(s[0][2], s[0][3]),
                                pack_half2(s[1][0], s[1][1]), pack_half2(s[1][2], s[1][3])};
        const uint32_t v_row = v_sm + (kb + v_key) * 128;
        auto v_addr = [&](int d16) {
          return v_row + (d16 / 4) * FEW_KB * 128 + ((((d16 & 3) * 2 + v_col) ^ (v_key & 7)) << 4);
        };
        if (!partly) {
#pragma unroll
          for (int d = 0; d < HD / 16; ++d) {
            uint32_t vf[4];
            ldsm_x4_t(v_addr(d), vf);
            mma_16816(o[2 * d], pa, vf[0], vf[1]);
            mma_16816(o[2 * d + 1], pa, vf[2], vf[3]);
          }
          continue;
        }
        // A probability of zero does not silence a value that is infinite or not a number.  Values behind the last
        // position (whatever the page holds there) are cleared; if one that only some rows see is not finite, the
        // step is done key by key, for the rows that see it.
        uint32_t keep[2], odd = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int key = key0 + pairc + 8 * i;
          keep[i] = (key < lk ? 0xFFFFu : 0u) | (key + 1 < lk ? 0xFFFF0000u : 0u);
        }
        if (all_see < min(lk, key0 + 16)) {
#pragma unroll 1
          for (int d = 0; d < HD / 16; ++d) {
            uint32_t vf[4];
            ldsm_x4_t(v_addr(d), vf);
#pragma unroll
            for (int i = 0; i < 4; ++i) odd |= not_finite2(vf[i] & keep[i & 1]);
          }
        }
        if (!__any_sync(0xffffffffu, odd != 0)) {
#pragma unroll
          for (int d = 0; d < HD / 16; ++d) {
            uint32_t vf[4];
            ldsm_x4_t(v_addr(d), vf);
            mma_16816(o[2 * d], pa, vf[0] & keep[0], vf[1] & keep[1]);
            mma_16816(o[2 * d + 1], pa, vf[2] & keep[0], vf[3] & keep[1]);
          }
          continue;
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const int from = (lane & ~3) | ((k & 7) >> 1);
          float pk[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float x = __shfl_sync(0xffffffffu, s[k >> 3][2 * i + (k & 1)], from);
            pk[i] = __half2float(__float2half_rn(x));
          }
          const bool see0 = key0 + k < limit[0], see1 = key0 + k < limit[1];
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            uint32_t raw;
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(raw)
                         : "r"(v_sm + (kb + k) * 128 + (t / 8) * FEW_KB * 128 + (((t & 7) ^ ((kb + k) & 7)) << 4) + pairc * 2));
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&raw));
            if (see0) o[t][0] = fmaf(pk[0], v.x, o[t][0]), o[t][1] = fmaf(pk[0], v.y, o[t][1]);
            if (see1) o[t][2] = fmaf(pk[1], v.x, o[t][2]), o[t][3] = fmaf(pk[1], v.y, o[t][3]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
      if (++st == STAGES) st = 0, ++use;
    }

    // ---- the warps that shared the keys agree on maximum and sum ----
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
    if (WK > 1 && (lane & 3) == 0) {
      ml[warp * 16 + quad] = make_float2(m[0], l[0]);
      ml[warp * 16 + quad + 8] = make_float2(m[1], l[1]);
    }
    few_sync();
    // the queries of the next item are on their way while this one is put together
    int next_limit[2];
    __half* next_dst[2];
    Walk next_w = w;
    if (more) {
      next_w = s_walk[turn];
      turn ^= 1;
      if (next_w.tiles != 0) enter(next_w, next_limit, next_dst, qa);
    }
    if constexpr (WK > 1) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int j = 0; j < WK; ++j) top = fmaxf(top, ml[(wm * WK + j) * 16 + quad + 8 * i].x);
        const float um = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int j = 0; j < WK; ++j) {
          const float2 x = ml[(wm * WK + j) * 16 + quad + 8 * i];
          sum += x.y * exp2_fast(x.x - um);
        }
        const float f = exp2_fast(m[i] - um);
#pragma unroll
        for (int t = 0; t < NT; ++t) o[t][2 * i] *= f, o[t][2 * i + 1] *= f;
        m[i] = top;
        l[i] = sum;
      }
    }

    // ---- the item is finished here, or this part of it is put down ----
    const bool whole = first == 0 && last == w.blks;
    // a CTA has at most two parts: one that begins with its units, one that begins behind them
    const size_t slot = 2 * (size_t)blockIdx.x + (u == u0 ? 0 : 1);
    float* po = p.part_o + slot * (FEW_MAX_ROWS * HD);
    if (!whole && wk == 0 && (lane & 3) == 0) {
      float2* pml = reinterpret_cast<float2*>(p.part_ml + slot * (FEW_MAX_ROWS * 2));
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (wm * 16 + quad + 8 * i < live) __stcg(pml + wm * 16 + quad + 8 * i, make_float2(m[i], l[i]));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (WK > 1 && i > 0) {
        if (WM == 1 && live <= 8) break;
        few_sync();  // the first eight rows have been read
      }
      if constexpr (WK > 1) {
        float2* mine = merge + warp * NT * 32 + lane;
#pragma unroll
        for (int t = 0; t < NT; ++t) mine[t * 32] = make_float2(o[t][2 * i], o[t][2 * i + 1]);
        few_sync();
      }
      const int r = wm * 16 + quad + 8 * i;
      // no visible position: zeros
      const float inv = limit[i] > 0 ? 1.0f / l[i] : 0.0f;
      // every warp adds up and stores its share of the columns
#pragma unroll
      for (int tt = 0; tt < NT / WK; ++tt) {
        const int t = WK > 1 ? wk * (NT / WK) + tt : tt;
        float2 x = make_float2(0.0f, 0.0f);
        if constexpr (WK > 1) {
          const float2* from = merge + (wm * WK * NT + t) * 32 + lane;
#pragma unroll
          for (int j = 0; j < WK; ++j) {
            const float2 y = from[j * NT * 32];
            x.x += y.x;
            x.y += y.y;
          }
        } else {
          x = make_float2(o[tt][2 * i], o[tt][2 * i + 1]);
        }
        if (r < live) {
          if (whole) *reinterpret_cast<uint32_t*>(dst[i] + t * 8 + pairc) = pack_half2(x.x * inv, x.y * inv);
          else __stcg(reinterpret_cast<float2*>(po + r * HD + t * 8 + pairc), x);
        }
      }
    }
    if (!whole) {
      // the CTAs that hold parts: from that of the item's first unit to that of its last
      const long long i0 = u - first;
      const int c0 = share.owner(i0), c1 = share.owner(i0 + w.blks - 1);
      __threadfence();
      few_sync();
      if (threadIdx.x == 0) {
        const bool is_last = atomicAdd(p.counters + c0, 1u) == (unsigned)(c1 - c0);
        if (is_last) p.counters[c0] = 0;  // as the next call finds it
        __threadfence();
        s_last = is_last ? 1u : 0u;
      }
      few_sync();
      if (s_last) {
        // a row to a warp, HD / 32 columns to a lane; eight parts' loads in flight
        constexpr int PER = HD / 32, DEEP = 8;
        const int parts = c1 - c0 + 1;
        const size_t slot0 = 2 * (size_t)c0 + (share.begin(c0) < i0 ? 1 : 0);  // the others are their CTAs' first
        auto slot_of = [&](int j) { return j == 0 ? slot0 : 2 * (size_t)(c0 + j); };
        for (int r = warp; r < live; r += 4) {
          float top = -INFINITY;
          for (int j = lane; j < parts; j += 32)
            top = fmaxf(top, __ldcg(reinterpret_cast<const float2*>(p.part_ml + slot_of(j) * (FEW_MAX_ROWS * 2)) + r).x);
          for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
          const float um = top == -INFINITY ? 0.0f : top;
          float sum = 0.0f, acc[PER];
#pragma unroll
          for (int i = 0; i < PER; ++i) acc[i] = 0.0f;
          for (int j0 = 0; j0 < parts; j0 += 32) {
            float factor = 0.0f;
            if (j0 + lane < parts) {
              const float2 x = __ldcg(reinterpret_cast<const float2*>(p.part_ml + slot_of(j0 + lane) * (FEW_MAX_ROWS * 2)) + r);
              factor = exp2_fast(x.x - um);
              sum += x.y * factor;
            }
            const int n = min(32, parts - j0);
            for (int j = 0; j < n; j += DEEP) {
              float4 v[DEEP];
#pragma unroll
              for (int d = 0; d < DEEP; ++d) {
                v[d] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (j + d < n) {
                  const float* src = p.part_o + slot_of(j0 + j + d) * (FEW_MAX_ROWS * HD) + r * HD + lane * PER;
                  if constexpr (PER == 4) {
                    v[d] = __ldcg(reinterpret_cast<const float4*>(src));
                  } else {
                    const float2 y = __ldcg(reinterpret_cast<const float2*>(src));
                    v[d].x = y.x, v[d].y = y.y;
                  }
                }
              }
#pragma unroll
              for (int d = 0; d < DEEP; ++d) {
                const float f = __shfl_sync(0xffffffffu, factor, j + d);
                if (j + d >= n) break;
                acc[0] += v[d].x * f, acc[1] += v[d].y * f;
                if constexpr (PER == 4) acc[2] += v[d].z * f, acc[3] += v[d].w * f;
              }
            }
          }
          for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
          const int rr = w.tile * Cfg::ROWS + r, tok = rr / p.a.group;
          const float inv = lk - w.span.lq + tok + 1 > 0 ? 1.0f / sum : 0.0f;
          __half* at = p.a.out + (long long)(w.span.q0 + tok) * p.a.so[0] +
                       (long long)(w.head * p.a.group + rr - tok * p.a.group) * p.a.so[1] + lane * PER;
#pragma unroll
          for (int i = 0; i < PER; i += 2)
            *reinterpret_cast<uint32_t*>(at + i) = pack_half2(acc[i] * inv, acc[i + 1] * inv);
        }
      }
    }
    u += last - first;
    if (!more || next_w.tiles == 0) break;
    w = next_w;
#pragma unroll
    for (int i = 0; i < 2; ++i) limit[i] = next_limit[i], dst[i] = next_dst[i];
  }
  if (!ok && lane == 0) atomicOr(p.a.status, 1u << 22);
}

int few_ctas(const adr_ctx* ctx) { return 2 * (ctx->sm_count > 0 ? ctx->sm_count : 148); }

template <int HD, int WM>
int launch_few_as(adr_ctx* ctx, cudaStream_t stream, const CUtensorMap& mk, const CUtensorMap& mv, const FewParams& p) {
  using Cfg = FewCfg<HD, WM>;
  auto kfn = attention_few_kernel<HD, WM>;
  if (int rc = opt_in_smem(ctx, kfn, Cfg::SMEM); rc != ADR_OK) return rc;
  return launch_whole_sm(ctx, stream, kfn, dim3(few_ctas(ctx)), FEW_THREADS, Cfg::SMEM, 1, true, mk, mv, p);
}

}  // namespace

size_t attention_few_workspace(const adr_ctx* ctx, int head_dim) {
  const size_t g = few_ctas(ctx);
  return (g * sizeof(unsigned) + 255) / 256 * 256 + 2 * g * FEW_MAX_ROWS * (head_dim + 2) * sizeof(float);
}

int launch_attention_few(adr_ctx* ctx, cudaStream_t stream, const SeqAttention& a, int rows, int max_rows, void* workspace) {
  FewParams p;
  p.a = a;
  p.max_rows = max_rows;
  p.min_units = std::max(1, ctx->tune_att_cs.load());
  p.page_rows = a.page_size < FEW_KB ? a.page_size : FEW_KB;
  const size_t g = few_ctas(ctx);
  p.counters = static_cast<unsigned int*>(workspace);
  p.part_ml = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + (g * sizeof(unsigned) + 255) / 256 * 256);
  p.part_o = p.part_ml + 2 * g * FEW_MAX_ROWS * 2;
  CUtensorMap mk, mv;
  if (int rc = pool_map(ctx, &mk, a.k, a.sk, a, p.page_rows); rc != ADR_OK) return rc;
  if (int rc = pool_map(ctx, &mv, a.v, a.sv, a, p.page_rows); rc != ADR_OK) return rc;
  if (a.head_dim == 128)
    return rows <= 16   ? launch_few_as<128, 1>(ctx, stream, mk, mv, p)
           : rows <= 32 ? launch_few_as<128, 2>(ctx, stream, mk, mv, p)
                        : launch_few_as<128, 4>(ctx, stream, mk, mv, p);
  return rows <= 16   ? launch_few_as<64, 1>(ctx, stream, mk, mv, p)
         : rows <= 32 ? launch_few_as<64, 2>(ctx, stream, mk, mv, p)
                      : launch_few_as<64, 4>(ctx, stream, mk, mv, p);
}

}  // namespace adr
