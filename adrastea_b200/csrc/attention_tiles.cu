// Attention of many rows per sequence, causal or not, over rows of a projection or over a paged cache.
//
// A tile is 128 rows of one key head: its `group` query heads times 128 / group tokens, token by token, so that the
// heads that share keys share their loads and a causal tile spans few tokens.  A CTA takes NT = 2 tiles (neighbouring
// tokens) over the same keys: while the softmax warps of one tile work, the tensor cores work for the other.
//   * producer: Q once, then K and V in blocks of 128 keys through a ring of shared-memory slots, by TMA (whole boxes
//     of rows, or page by page), in the 128-byte swizzle;
//   * S = Q K^T by tcgen05.mma into tensor memory; P = exp2(scale2 (S - m)) written back over S by one thread per row;
//     O += P V with P from tensor memory and V as it lies in memory (N-major), O staying in tensor memory;
//   * the maximum m that a row is scaled by is moved only when a score passes it by more than 2^8 (P then stays within
//     fp16's range, and the sums are fp32): the rescaling of O in tensor memory is rare;
//   * when S of a block is complete, so is the product with V before it (the tensor cores run in order), so the softmax
//     warps may touch O and no further barrier is needed.
// What a causal row does not see must not reach it even if it is infinite or not a number; a probability of zero does
// not see to that.  Keys are masked by selection.  Values behind the sequence's end are cleared in shared memory; a
// block of which some rows see only a part is searched, and where a value that some row does not see is not finite the
// softmax warps do that block's product themselves, each row with the keys it sees.
#include <algorithm>

#include "attention_seqs.cuh"
#include "tcgen05.cuh"

namespace adr {

namespace {

constexpr int TL_M = 128;   // rows of a tile
constexpr int TL_N = 128;   // keys of a block

template <int HD, int NT>
struct TileCfg {
  static constexpr int CH = HD / 64;
  static constexpr int TILE = 128 * HD * 2;
  static constexpr int SLOTS = NT == 2 ? (HD == 128 ? 5 : 8) : (HD == 128 ? 2 : 4);
  static constexpr int THREADS = NT * 128 + 64;
  static constexpr uint32_t COLS = NT == 2 ? 512 : 256;
  static constexpr uint32_t O_COL = NT * 128;
  static constexpr size_t SMEM = 1024 + (size_t)TILE * (NT + SLOTS) + 8 * (3 * NT + NT + 2 * SLOTS) + 64;
};

struct TileParams {
  SeqAttention a;
  int tokens_tile;   // tokens of a tile: 128 / group
  int min_rows;      // sequences with fewer rows of a key head than this are left to another kernel
  int page_rows;     // rows of a copy of keys: a page, 128 at most
};

__device__ __forceinline__ void tmem_ld_x32(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
      "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_x32(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
      "%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_ld_x8(uint32_t addr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_st_x8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// A from tensor memory
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
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
// Nonzero if one of the two halves is infinite or not a number (see attention_few.cu).
__device__ __forceinline__ uint32_t not_finite2(uint32_t x) { return ((x & 0x7C007C00u) + 0x04000400u) & 0x80008000u; }
// Whether the predicate holds for any of the 128 threads of a tile's softmax warps.
__device__ __forceinline__ bool tile_any(int tile, bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred a, b;\n\tsetp.ne.u32 a, %1, 0;\n\t"
      "barrier.cta.red.or.pred b, %2, 128, a;\n\tselp.u32 %0, 1, 0, b;\n\t}"
      : "=r"(r) : "r"((uint32_t)x), "r"(tile + 1) : "memory");
  return r != 0;
}

struct TileJob {
  SeqSpan span;
  int s, token0;  // first token of the CTA's tiles
};

template <int HD, int NT, bool PAGED>
__global__ void __launch_bounds__(TileCfg<HD, NT>::THREADS, NT == 2 ? 1 : 2)
    attention_tiles_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                           const __grid_constant__ CUtensorMap map_v, const __grid_constant__ TileParams p) {
  using Cfg = TileCfg<HD, NT>;
  constexpr int CH = Cfg::CH, SLOTS = Cfg::SLOTS, TILE = Cfg::TILE;
  extern __shared__ uint8_t tile_smem[];
  uint8_t* q_sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(tile_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* ring = q_sm + NT * TILE;  // K of block 0, V of block 0, K of block 1 ...
  uint64_t* q_full = reinterpret_cast<uint64_t*>(ring + SLOTS * TILE);  // [NT]
  uint64_t* s_ready = q_full + NT;   // [NT] scores of a tile are complete
  uint64_t* p_ready = s_ready + NT;  // [NT] its probabilities are
  uint64_t* o_done = p_ready + NT;   // [NT] its output is
  uint64_t* full = o_done + NT;      // [SLOTS]
  uint64_t* empty = full + SLOTS;    // [SLOTS]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(empty + SLOTS);
  volatile uint32_t* by_hand = tmem_slot + 1;  // [NT] the softmax warps did this block's product with V
  __shared__ TileJob s_job;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int W_MMA = NT * 4, W_TMA = NT * 4 + 1;
  if (warp == W_TMA && lane == 0) {
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
    for (int i = 0; i < NT; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&s_ready[i], 1);
      mbar_init(&p_ready[i], 4);
      mbar_init(&o_done[i], 1);
    }
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_fence_init();
  }
  if (warp == W_MMA) tmem_alloc(tmem_slot, Cfg::COLS);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  // (only now: a launch behind this one may not take the tensor memory that this CTA is waiting for)
  pdl_wait_trigger();
  const int head = blockIdx.x % p.a.n_kv_heads;
  if (warp == 0) {
    // the CTA's tiles: the last ones of a sequence, which see most keys, come first
    int id = blockIdx.x / p.a.n_kv_heads;
    const int per = NT * p.tokens_tile;
    TileJob job = {};
    job.s = p.a.n_seqs;
    for (int s0 = 0; s0 < p.a.n_seqs; s0 += 32) {
      int mine = 0;
      if (s0 + lane < p.a.n_seqs) {
        const int lq = min(max(__ldg(p.a.cu_q + s0 + lane + 1), 0), p.a.tokens) -
                       min(max(__ldg(p.a.cu_q + s0 + lane), 0), p.a.tokens);
        if (lq > 0 && (long long)lq * p.a.group >= p.min_rows) mine = (lq + per - 1) / per;
      }
      int upto = mine;
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += o;
      }
      const unsigned m = __ballot_sync(0xffffffffu, id < upto);
      if (m) {
        const int l = __ffs(m) - 1;
        const int behind = __shfl_sync(0xffffffffu, upto, l) - 1 - id;  // tiles of the sequence that come later
        job.s = s0 + l;
        job.span = seq_span(p.a.cu_q, p.a.kv_len, job.s, p.a.tokens, p.a.max_pages * p.a.page_size, p.a.status);
        job.token0 = behind * per;
        break;
      }
      id -= __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) s_job = job;
  }
  __syncthreads();
  const uint32_t tmem = *tmem_slot;
  const SeqSpan span = s_job.span;
  const int lq = span.lq, lk = span.lk, token0 = s_job.token0;
  const bool any = s_job.s < p.a.n_seqs && token0 < lq;
  // per tile: its tokens, the keys that its last row sees, the blocks of them
  int n_tok[NT], kend[NT], nb[NT], nb_max = 0;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int first = token0 + t * p.tokens_tile;
    n_tok[t] = any ? min(p.tokens_tile, max(0, lq - first)) : 0;
    kend[t] = n_tok[t] == 0 ? 0 : p.a.causal ? max(0, lk - lq + first + n_tok[t]) : lk;
    nb[t] = (kend[t] + TL_N - 1) / TL_N;
    nb_max = max(nb_max, nb[t]);
  }
  // keys of a block as the tensor cores take them, in steps of 16
  auto block_n = [&](int t, int j) { return min(TL_N, (kend[t] - j * TL_N + 15) & ~15); };

  if (warp == W_TMA) {
    // ------------------------------- producer -------------------------------
    bool ok = true;
    if (nb_max > 0) {
      if (lane == 0) {
        for (int t = 0; t < NT; ++t) {
          if (nb[t] == 0) continue;
          mbar_expect_tx(&q_full[t], (unsigned)(CH * p.tokens_tile * p.a.group * 128));
          for (int c = 0; c < CH; ++c)
            tma_load_3d(q_sm + t * TILE + c * (TL_M * 128), &map_q, c * 64, head * p.a.group,
                        span.q0 + token0 + t * p.tokens_tile, &q_full[t]);
        }
      }
      int issued = 0;
      for (int i = 0; i < 2 * nb_max; ++i) {
        const int st = i % SLOTS, j = i >> 1;
        uint8_t* dst = ring + st * TILE;
        const CUtensorMap* map = (i & 1) ? &map_v : &map_k;
        if constexpr (PAGED) {
          const int pr = p.page_rows;
          const int copies = (min(TL_N, lk - j * TL_N) + pr - 1) / pr;
          const int pos = j * TL_N + lane * pr;
          int page = 0;
          if (lane < copies) {
            page = __ldg(p.a.block_table + (long long)s_job.s * p.a.max_pages + pos / p.a.page_size);
            if (page < 0 || page >= p.a.n_pages) {
              page = p.a.n_pages;  // outside the map: zeros arrive
              atomicOr(p.a.status, PAGED_BAD);
            }
          }
          if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&empty[st], ((unsigned)(i / SLOTS) & 1u) ^ 1u));
          if (!ok) break;
          if (lane == 0) mbar_expect_tx(&full[st], (unsigned)(copies * pr * HD * 2));
          __syncwarp();
          if (lane < copies)
            for (int c = 0; c < CH; ++c)
              tma_load_4d(dst + c * (TL_N * 128) + lane * pr * 128, map, c * 64, head, pos % p.a.page_size, page, &full[st]);
        } else {
          if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&empty[st], ((unsigned)(i / SLOTS) & 1u) ^ 1u));
          if (!ok) break;
          if (lane == 0) {
            mbar_expect_tx(&full[st], TILE);
            for (int c = 0; c < CH; ++c)
              tma_load_3d(dst + c * (TL_N * 128), map, c * 64, head, span.q0 + j * TL_N, &full[st]);
          }
        }
        issued = i + 1;
      }
      // every copy has landed and every slot's last reader is done before the CTA may end
      for (int t = 0; t < NT; ++t)
        if (nb[t] > 0 && !mbar_wait(&q_full[t], 0)) ok = false;
      for (int i = max(0, issued - SLOTS); i < issued; ++i) {
        if (!mbar_wait(&full[i % SLOTS], (unsigned)(i / SLOTS) & 1u)) ok = false;
        if (ok && !mbar_wait(&empty[i % SLOTS], (unsigned)(i / SLOTS) & 1u)) ok = false;
      }
    }
    if (!ok && lane == 0) atomicOr(p.a.status, 1u << 23);
  } else if (warp == W_MMA) {
    // ------------------------------- tensor cores -------------------------------
    if (lane == 0 && nb_max > 0) {
      bool ok = true;
      uint32_t have_o[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) have_o[t] = 0;
      auto wait_full = [&](int i) { ok = ok && mbar_wait(&full[i % SLOTS], (unsigned)(i / SLOTS) & 1u); };
      // the last tile that uses block j (tile 1 sees at least what tile 0 sees)
      auto last_of = [&](int j) { return NT == 2 && j < nb[NT - 1] ? 1 : 0; };
      auto scores = [&](int t, int j) {
        if (j == 0) ok = ok && mbar_wait(&q_full[t], 0);
        wait_full(2 * j);
        if (!ok) return;
        tc_fence_after_sync();
        const uint32_t idesc = umma_idesc_f16(block_n(t, j), false);
        const uint32_t qa = smem_u32(q_sm + t * TILE), ka = smem_u32(ring + ((2 * j) % SLOTS) * TILE);
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_f16(tmem + t * 128, umma_desc_k_sw128(qa + c * (TL_M * 128)) + (uint64_t)(kk * 2),
                     umma_desc_k_sw128(ka + c * (TL_N * 128)) + (uint64_t)(kk * 2), idesc, (c | kk) ? 1u : 0u);
        umma_commit(&s_ready[t]);
        if (t == last_of(j)) umma_commit(&empty[(2 * j) % SLOTS]);
      };
      auto output = [&](int t, int j) {
        ok = ok && mbar_wait(&p_ready[t], (unsigned)j & 1u);
        wait_full(2 * j + 1);
        if (!ok) return;
        tc_fence_after_sync();
        if (by_hand[t] == 0) {
          constexpr uint32_t idesc = umma_idesc_f16(HD, true);
          const uint64_t vd = umma_desc_mn_sw128(smem_u32(ring + ((2 * j + 1) % SLOTS) * TILE), TL_N * 128);
          const int steps = block_n(t, j) / 16;
          for (int ks = 0; ks < steps; ++ks)
            umma_ts(tmem + Cfg::O_COL + t * HD, tmem + t * 128 + ks * 8, vd + (uint64_t)ks * 128, idesc,
                    (have_o[t] | (uint32_t)ks) ? 1u : 0u);
        }
        have_o[t] = 1;
        if (t == last_of(j)) umma_commit(&empty[(2 * j + 1) % SLOTS]);
        if (j == nb[t] - 1) umma_commit(&o_done[t]);
      };
#pragma unroll
      for (int t = 0; t < NT; ++t)
        if (nb[t] > 0) scores(t, 0);
      for (int j = 0; j < nb_max && ok; ++j) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if (j < nb[t]) output(t, j);
          if (j + 1 < nb[t]) scores(t, j + 1);
        }
      }
      if (!ok) atomicOr(p.a.status, 1u << 24);
    }
  } else {
    // ------------------------------- softmax and output -------------------------------
    const int t = NT == 2 ? warp >> 2 : 0;
    const int row = (warp & 3) * 32 + lane;  // of the tile, and lane of tensor memory
    const int my_nb = NT == 2 && t == 1 ? nb[NT - 1] : nb[0];
    const int my_tok = NT == 2 && t == 1 ? n_tok[NT - 1] : n_tok[0];
    const int first = token0 + t * p.tokens_tile;
    const int tok = row / p.a.group;
    const bool live = tok < my_tok;
    const bool warp_live = __any_sync(0xffffffffu, live);
    const int limit = !live ? 0 : p.a.causal ? max(0, lk - lq + first + tok + 1) : lk;
    const int all_see = p.a.causal ? max(0, lk - lq + first + 1) : lk;  // keys that every row of the tile sees
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lanes + (uint32_t)(t * 128), o_at = tmem + lanes + Cfg::O_COL + (uint32_t)(t * HD);
    // scores in powers of two; the sign of the scale goes into the scores so that the largest product is the maximum
    // (a scale of zero, which would make NaN of what is masked, is as good as one of 1e-30: exp2 is 1 for every score)
    const float scale2 = fmaxf(fabsf(p.a.scale) * 1.4426950408889634f, 1e-30f);
    const bool negative = p.a.scale < 0.0f;
    const float slack = 8.0f / scale2;
    float m = -INFINITY, l = 0.0f;
    bool ok = true;

    for (int j = 0; j < my_nb; ++j) {
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&s_ready[t], (unsigned)j & 1u));
      tc_fence_after_sync();
      const int key0 = j * TL_N;
      const bool partly = key0 + TL_N > all_see;  // some row does not see some key of the block
      bool hand = false;
      if (ok && warp_live) {
        uint32_t s[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_x32(s_at + c * 32, s + c * 32);
        tmem_ld_wait();
        if (negative) {
#pragma unroll
          for (int i = 0; i < 128; ++i) s[i] ^= 0x80000000u;
        }
        if (partly) {
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (key0 + i >= limit) s[i] = 0xFF800000u;  // -infinity
        }
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 128; ++i) top[i & 3] = fmaxf(top[i & 3], __uint_as_float(s[i]));
        const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        // (a first maximum moves from -infinity: nothing is summed or in O yet but zeros)
        const bool move = mx > m + slack || (m == -INFINITY && mx > m);
        if (__any_sync(0xffffffffu, move)) {
          const float alpha = move ? (m == -INFINITY ? 0.0f : exp2_fast((m - mx) * scale2)) : 1.0f;
          if (move) m = mx;
          l *= alpha;
          if (j > 0) {
#pragma unroll 1
            for (int c = 0; c < HD; c += 8) {
              uint32_t o[8];
              tmem_ld_x8(o_at + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st_x8(o_at + c, o);
            }
          }
        }
        const float base = m == -INFINITY ? 0.0f : m * scale2;
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t pk[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float a = exp2_fast(fmaf(__uint_as_float(s[c * 64 + 2 * i]), scale2, -base));
            const float b = exp2_fast(fmaf(__uint_as_float(s[c * 64 + 2 * i + 1]), scale2, -base));
            sum[i & 3] += a + b;
            pk[i] = pack_half2(a, b);
          }
          tmem_st_x32(s_at + c * 32, pk);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      }
      tmem_wait_st();
      if (partly) {
        // V: wait for it, clear what lies behind the end, look for what may not be multiplied by zero
        uint8_t* v = ring + ((2 * j + 1) % SLOTS) * TILE;
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&full[(2 * j + 1) % SLOTS], (unsigned)((2 * j + 1) / SLOTS) & 1u));
        const int from = max(0, all_see - key0), end = min(TL_N, lk - key0);
        uint32_t odd = 0;
        // a thread takes a 16-byte piece of every 128 / (HD / 8)-th row (the swizzle only permutes a row's pieces)
        constexpr int LPR = HD / 8;
        for (int r = from + row / LPR; r < TL_N; r += 128 / LPR) {
          uint4* at = reinterpret_cast<uint4*>(v + ((row % LPR) / 8) * (TL_N * 128) + r * 128 + (row % 8) * 16);
          if (r >= end) {
            *at = make_uint4(0, 0, 0, 0);
          } else {
            const uint4 x = *at;
            odd |= not_finite2(x.x) | not_finite2(x.y) | not_finite2(x.z) | not_finite2(x.w);
          }
        }
        fence_proxy_async();
        hand = tile_any(t, odd != 0);
        if (hand && ok && warp_live) {
          // this block's product by hand
#pragma unroll 1
          for (int c = 0; c < HD; c += 8) {
            uint32_t o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = 0;
            if (j > 0) {
              tmem_ld_x8(o_at + c, o);
              tmem_ld_wait();
            }
#pragma unroll 1
            for (int k0 = 0; k0 < end; k0 += 16) {
              uint32_t pk[8];
              __syncwarp();
              tmem_ld_x8(s_at + k0 / 2, pk);
              tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 16; ++k) {
                const __half2 ph = *reinterpret_cast<const __half2*>(&pk[k >> 1]);
                const float w = (k & 1) ? __high2float(ph) : __low2float(ph);
                const int r = k0 + k;
                if (key0 + r >= limit) continue;  // (also what lies behind the end)
                const uint4 x = *reinterpret_cast<const uint4*>(v + (c / 64) * (TL_N * 128) + r * 128 + (((c / 8) ^ r) & 7) * 16);
                const __half2* h = reinterpret_cast<const __half2*>(&x);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float2 f = __half22float2(h[i]);
                  o[2 * i] = __float_as_uint(fmaf(w, f.x, __uint_as_float(o[2 * i])));
                  o[2 * i + 1] = __float_as_uint(fmaf(w, f.y, __uint_as_float(o[2 * i + 1])));
                }
              }
            }
            __syncwarp();
            tmem_st_x8(o_at + c, o);
          }
          tmem_wait_st();
        }
      }
      if (row == 0) by_hand[t] = hand ? 1u : 0u;
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_ready[t]);
    }
    if (my_nb > 0) {
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&o_done[t], 0));
      tc_fence_after_sync();
    }
    if (ok && warp_live) {
      // a row that sees no key gets zeros
      const float inv = limit > 0 ? 1.0f / l : 0.0f;
      __half* dst = p.a.out + (long long)(span.q0 + first + tok) * p.a.so[0] +
                    (long long)(head * p.a.group + row - tok * p.a.group) * p.a.so[1];
#pragma unroll
      for (int c = 0; c < HD; c += 32) {
        uint32_t o[32];
        if (my_nb > 0) {
          tmem_ld_x32(o_at + c, o);
          tmem_ld_wait();
        }
        if (live) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (limit > 0) {
              w.x = pack_half2(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv);
              w.y = pack_half2(__uint_as_float(o[i + 2]) * inv, __uint_as_float(o[i + 3]) * inv);
              w.z = pack_half2(__uint_as_float(o[i + 4]) * inv, __uint_as_float(o[i + 5]) * inv);
              w.w = pack_half2(__uint_as_float(o[i + 6]) * inv, __uint_as_float(o[i + 7]) * inv);
            }
            *reinterpret_cast<uint4*>(dst + c + i) = w;
          }
        }
        __syncwarp();
      }
    }
    if (!ok && lane == 0) atomicOr(p.a.status, 1u << 25);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == W_MMA) {
    __syncwarp();
    tc_fence_after_sync();
    tmem_dealloc(tmem, Cfg::COLS);
  }
}

// Rows of a projection, [64 columns, heads, rows] boxes of a [tokens, heads, head_dim] view.
int rows_map(adr_ctx* ctx, CUtensorMap* map, const __half* base, const SeqAttention& a, int n_heads, long long s_row,
             long long s_head, int box_heads, int box_rows) {
  const uint64_t dims[3] = {(uint64_t)a.head_dim, (uint64_t)n_heads, (uint64_t)a.tokens};
  const uint64_t strides[2] = {n_heads > 1 ? (uint64_t)s_head * 2 : (uint64_t)a.head_dim * 2,
                               a.tokens > 1 ? (uint64_t)s_row * 2 : (uint64_t)a.head_dim * 2};
  const uint32_t box[3] = {64u, (uint32_t)box_heads, (uint32_t)box_rows};
  return tma_get(ctx, map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int HD, int NT, bool PAGED>
int launch_tiles_as(adr_ctx* ctx, cudaStream_t stream, const SeqAttention& a, int min_rows) {
  using Cfg = TileCfg<HD, NT>;
  auto kfn = attention_tiles_kernel<HD, NT, PAGED>;
  if (int rc = opt_in_smem(ctx, kfn, Cfg::SMEM); rc != ADR_OK) return rc;
  TileParams p;
  p.a = a;
  p.tokens_tile = TL_M / a.group;
  p.min_rows = min_rows;
  p.page_rows = std::min(a.page_size, TL_N);
  CUtensorMap mq, mk, mv;
  if (int rc = rows_map(ctx, &mq, a.q, a, a.n_heads, a.sq[0], a.sq[1], a.group, p.tokens_tile); rc != ADR_OK) return rc;
  if constexpr (PAGED) {
    if (int rc = pool_map(ctx, &mk, a.k, a.sk, a, p.page_rows); rc != ADR_OK) return rc;
    if (int rc = pool_map(ctx, &mv, a.v, a.sv, a, p.page_rows); rc != ADR_OK) return rc;
  } else {
    if (int rc = rows_map(ctx, &mk, a.k, a, a.n_kv_heads, a.sk[1], a.sk[2], 1, TL_N); rc != ADR_OK) return rc;
    if (int rc = rows_map(ctx, &mv, a.v, a, a.n_kv_heads, a.sv[1], a.sv[2], 1, TL_N); rc != ADR_OK) return rc;
  }
  // as many CTAs as there can be: a sequence fills up its last one
  const long long per = NT * p.tokens_tile;
  const long long tiles = std::min<long long>(a.tokens, (a.tokens + a.n_seqs * (per - 1)) / per);
  if (tiles * a.n_kv_heads > 0x7fffffffLL) return ADR_ERR_SHAPE;
  return launch_whole_sm(ctx, stream, kfn, dim3((unsigned)(tiles * a.n_kv_heads)), Cfg::THREADS, Cfg::SMEM, 1, true, mq,
                         mk, mv, p);
}

}  // namespace

int launch_attention_tiles(adr_ctx* ctx, cudaStream_t stream, const SeqAttention& a, int max_q, int min_rows) {
  const bool paged = a.block_table != nullptr;
  const bool one = (long long)max_q * a.group <= TL_M;
  if (a.head_dim == 128) {
    if (one) return paged ? launch_tiles_as<128, 1, true>(ctx, stream, a, min_rows) : launch_tiles_as<128, 1, false>(ctx, stream, a, min_rows);
    return paged ? launch_tiles_as<128, 2, true>(ctx, stream, a, min_rows) : launch_tiles_as<128, 2, false>(ctx, stream, a, min_rows);
  }
  if (one) return paged ? launch_tiles_as<64, 1, true>(ctx, stream, a, min_rows) : launch_tiles_as<64, 1, false>(ctx, stream, a, min_rows);
  return paged ? launch_tiles_as<64, 2, true>(ctx, stream, a, min_rows) : launch_tiles_as<64, 2, false>(ctx, stream, a, min_rows);
}

}  // namespace adr
