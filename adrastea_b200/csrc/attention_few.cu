// Attention of a few new rows per sequence over a paged cache: single tokens, and a few at a time.
//
// The rows of one key head (its query heads times the new tokens, up to 32) share every key and value, so one pass
// over the cache serves them all: what bounds this kernel is reading the cache once (64 sequences of 128 to 8192
// positions, 32/8 heads of 128: 91 us, 512 MB at 5.6 TB/s of 6.55).
//   * Work is counted in units of one (sequence, key head, tile of rows), 64 keys of 128 columns or 128 of 64, and cut
//     into one chunk for each CTA by the lengths on the device, so the cache of a batch of very different lengths, or of
//     one long sequence, is spread evenly with no plan from the host.  (SMs do not get equal shares of the memory's
//     bandwidth; but to keep an eighth of the work back in small chunks, for CTAs to take as they get done, cost as much
//     as it gave: 64 sequences 90.7 against 88.4 us, one of 131072 positions 93.4 against 90.1, eight tokens of 64
//     sequences 130 against 138.)
//   * The producer warp looks up what comes next and copies pages by TMA into a ring of stages (a unit's keys and values),
//     across the borders of items.
//   * Four warps compute: S = Q K^T and O += P V by mma.sync m16n8k16 with the 16 (32) rows as M and a running
//     maximum and sum.  (tcgen05 wants 64 or 128 rows: at up to 16 live ones the tensor work is 17 % of the time that
//     the keys take to arrive.  With 64 rows, a row tile to each warp, this kernel took 1.3 to 2.5 times what the tiles of
//     attention_tiles.cu take.)  With 16 rows the warps share a stage's keys among them, with 32 two by two.
//   * An item that lies within one chunk is finished there.  Otherwise each part stores its maximum, sum and unscaled
//     output, and a second kernel, which is resident before the first one ends, joins them in their order.  (Joined by
//     the CTA that came last, 111 parts took 65 us: a join is a chain of loads of about a microsecond each, and one CTA
//     has too few of them in flight.)  What is cut where does not depend on who computes it: same bits each run.
#include <algorithm>

#include "attention_seqs.cuh"

namespace adr {

namespace {

constexpr int FEW_THREADS = 160;       // four computing warps and the producer
constexpr int MOST_UNITS = 2000000000;  // units of work that can be counted

// Probabilities and their sums are carried times 2^15: fp16 holds that (up to just below 2^16), and what is small keeps as
// many bits as there are, 11 down to 2^-29 of a row's largest weight and 2^-40 of it below.
constexpr float FEW_UP = 15.0f;

constexpr int few_kb(int head_dim) { return 8192 / head_dim; }  // 64 keys of 128 columns, 128 of 64

template <int HD, int WM>
struct FewCfg {
  static constexpr int KB = few_kb(HD);         // keys of a stage, and of a unit of work
  static constexpr int ROWS = 16 * WM;
  static constexpr int WK = 4 / WM;             // warps that share a stage's keys
  static constexpr int KEYS = KB / WK;          // of a stage, for one warp
  static constexpr int SK = KEYS < 32 ? KEYS : 32;  // of a step of a warp
  static constexpr int CH = HD / 64;            // 64-column chunks of a head
  static constexpr int TILE = KB * HD * 2;      // bytes of a stage's keys: 16 KB
  static constexpr int STAGES = 3;
  static constexpr int MERGE = WK == 1 ? 0 : 4 * (HD / 8) * 32 * 8;  // eight rows of every warp
  // Stages of an item after which a warp's sums begin anew: 32768 keys of its own (see take_mean).
  static constexpr int FOLD = 32768 / KEYS;
  static constexpr int SEGS = STAGES + 2;       // descriptors in flight (a segment has at least one stage)
  static constexpr size_t SMEM = (size_t)STAGES * 2 * TILE + MERGE + 4 * 16 * 8 + 16 * STAGES + 8 * SEGS +
                                 SEGS * 48;
  static_assert(WM == 1 || WM == 2, "");
};

struct Segment;

struct FewParams {
  SeqAttention a;
  int max_rows;  // sequences with more rows of a key head than this are left to another kernel
  int page_rows; // rows of a copy: a page, a stage at most
  int most_units;  // of all sequences together, by the arguments
  float* part_ml;          // [slots][ROWS][2]: two slots to a chunk
  float* part_o;           // [slots][ROWS][head_dim]
  int* chunks;             // their number in this call
  Segment* begins;  // the first segment of every chunk
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
// The tensor cores' sums round towards zero, 1e-7 of a sum for every 16 products: 2e-4 after 32768 keys, values of one sign were
// off by 1.7e-3 after a million.  So after that many a thread takes out of its part of a row's sum what the row's mean so far
// stands for (`l` times it), keeps that mean in 16 bits, zero where it would not be finite, and the sum begins anew.  In
// kernels of their own (LONG): with that code 64 sequences took 94.1 instead of 89.5 us, 94 short ones 16.4 instead of 15.2.
__device__ __forceinline__ uint32_t take_mean(float& a, float& b, float l, float inv) {
  float2 x = make_float2(a * inv, b * inv);
  if (!(fabsf(x.x) <= 65504.0f)) x.x = 0.0f;
  if (!(fabsf(x.y) <= 65504.0f)) x.y = 0.0f;
  const __half2 h = __floats2half2_rn(x.x, x.y);
  x = __half22float2(h);
  a = fmaf(-l, x.x, a);
  b = fmaf(-l, x.y, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void add_mean(float& a, float& b, float l, uint32_t mean) {
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&mean));
  a = fmaf(l, x.x, a);
  b = fmaf(l, x.y, b);
}
// The computing warps only: a barrier, and one that says whether the predicate holds for all of them.
__device__ __forceinline__ void few_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ bool few_all(bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred a, b;\n\tsetp.ne.u32 a, %1, 0;\n\t"
      "barrier.cta.red.and.pred b, 1, 128, a;\n\tselp.u32 %0, 1, 0, b;\n\t}"
      : "=r"(r) : "r"((uint32_t)x) : "memory");
  return r != 0;
}

// Where in the list of all units (sequence by sequence, key head by key head, tile by tile, KB keys each) one is.
struct Walk {
  SeqSpan span;
  int s, head, tile, blk;
  int tiles, blks;
};

// How the units are cut: the list is divided evenly into `ctas` chunks (the first `more` have one more than `per`).
struct Share {
  int total, ctas, per, more;
  __device__ int begin(int c) const { return c * per + min(c, more); }
  __device__ int chunk_of(int u) const {
    const int big = more * (per + 1);
    return u < big ? u / (per + 1) : more + (u - big) / per;
  }
};

// A run of units of one item, as the producer hands it to the computing warps.
struct Segment {
  int q0, lq, lk;           // of the sequence
  int head, tile;
  int first, last, blks;    // blocks of this run, of the item; blks == 0: there is no more
  int slot;                 // where a part goes (slots are in the order of the units)
  int chunk0, parts;        // chunks of the item's parts
  int slot0;                // slot of the first one; the others are the first slots of their chunks
};
static_assert(sizeof(Segment) == 48, "");

template <int ROWS, int KB>
struct FewWork {
  const FewParams& p;
  const int lane, q;  // a lane stands for q sequences
  int before, upto;   // units before and up to the end of its sequences
  __device__ FewWork(const FewParams& p_, int lane_) : p(p_), lane(lane_), q((p_.a.n_seqs + 31) / 32) {
    int mine = 0;
#pragma unroll 4
    for (int i = 0; i < q; ++i) mine = sum_of(mine, units(lane * q + i));
    upto = scan(mine);
    before = upto - mine;
  }
  // of two numbers up to MOST_UNITS, staying there (a sequence has fewer units; all of them may not, if spans overlap)
  __device__ static int sum_of(int a, int b) { return (int)min((unsigned)a + (unsigned)b, (unsigned)MOST_UNITS); }
  __device__ int scan(int x) const {
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x = sum_of(x, o);
    }
    return x;
  }
  __device__ SeqSpan span(int s) const {
    return seq_span(p.a.cu_q, p.a.kv_len, s, p.a.tokens, p.a.max_pages * p.a.page_size, p.a.status);
  }
  __device__ int tiles(const SeqSpan& v) const {
    const long long rows = (long long)v.lq * p.a.group;
    return rows > p.max_rows ? 0 : (int)((rows + ROWS - 1) / ROWS);
  }
  __device__ static int blocks(const SeqSpan& v) { return max(1, (v.lk + KB - 1) / KB); }
  __device__ int units(int s) const {
    if (s >= p.a.n_seqs) return 0;
    const SeqSpan v = span(s);
    return tiles(v) * blocks(v) * p.a.n_kv_heads;
  }
  __device__ Share share() const {
    Share r;
    r.total = __shfl_sync(0xffffffffu, upto, 31);
    if (r.total > p.most_units) {  // more than sequences side by side can have: cu_q is wrong, and nothing is done
      if (lane == 0) atomicOr(p.a.status, PAGED_BAD);
      r.total = 0;
    }
    r.ctas = min((int)gridDim.x, r.total);
    r.per = r.ctas ? r.total / r.ctas : 0;
    r.more = r.total - r.per * r.ctas;
    return r;
  }
  __device__ void enter(Walk& w, int s) const {
    w.s = s;
    w.span = span(s);
    w.tiles = tiles(w.span);
    w.blks = blocks(w.span);
  }
  // Unit u of all, by the whole warp.  (The loops over sequences end behind the last one whatever happens to the arrays
  // meanwhile; no tiles: there is no such unit.)
  __device__ Walk find(int u) const {
    Walk w = {};
    const unsigned m = __ballot_sync(0xffffffffu, u < upto);
    if (!m) return w;
    const int l = __ffs(m) - 1;
    u -= __shfl_sync(0xffffffffu, before, l);
    int s = l * q;
    if (q > 1) {
      const int end = min(p.a.n_seqs, s + q);
      for (;; s += 32) {
        if (s >= end) return w;
        const int mine = s + lane < end ? units(s + lane) : 0;
        const int sum = scan(mine);
        const unsigned h = __ballot_sync(0xffffffffu, u < sum);
        if (h) {
          const int f = __ffs(h) - 1;
          u -= __shfl_sync(0xffffffffu, sum - mine, f);
          s += f;
          break;
        }
        u -= __shfl_sync(0xffffffffu, sum, 31);
      }
    }
    enter(w, s);
    if (w.tiles == 0) return w;
    const int per_head = w.tiles * w.blks;
    w.head = u / per_head;
    const int in_head = u - w.head * per_head;
    w.tile = in_head / w.blks;
    w.blk = in_head - w.tile * w.blks;
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

// Joins parts.  Block j stands for the border before chunk j: if an item goes across it, the blocks of its borders share
// its rows.  Few parts: a row to a warp; many: a row to the block, the parts shared out among its warps.  All loads of
// eight parts are in flight at once.  (What is read here was written by the launch before, or, if that gave up, is left
// from another call: nothing is stored outside the rows there are.)
template <int HD, int ROWS, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) few_join_kernel(const __grid_constant__ FewParams p) {
  constexpr int PER = HD / 32, DEEP = 8;
  __shared__ float part[WARPS][HD];
  __shared__ float2 part_ml[WARPS];
  pdl_wait_trigger();
  const int j = blockIdx.x + 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = p.a.group;
  const int n = min(*p.chunks, (int)gridDim.x + 1);
  const Segment g = p.begins[j];
  if (j >= n || g.first == 0) return;  // no item goes across
  const int border = j - 1 - g.chunk0;
  if (g.chunk0 < 0 || border < 0 || g.parts > n || border > g.parts - 2 || g.chunk0 + g.parts > n || g.slot0 >> 1 != g.chunk0)
    return;
  const int live = min(ROWS, g.lq * group - g.tile * ROWS);
  const bool many = g.parts > DEEP;
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml);
  for (int r = many ? border : border * WARPS + warp; r < live; r += (g.parts - 1) * (many ? 1 : WARPS)) {
    float m = -INFINITY, l = 0.0f, acc[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] = 0.0f;
    const int step = many ? WARPS : 1;
    for (int j0 = many ? warp : 0; j0 < g.parts; j0 += DEEP * step) {
      float2 x[DEEP];
      float4 v[DEEP];
#pragma unroll
      for (int d = 0; d < DEEP; ++d) {
        const int at = j0 + d * step;
        const size_t row = (size_t)(at == 0 ? g.slot0 : 2 * (g.chunk0 + min(at, g.parts - 1))) * ROWS + r;
        x[d] = __ldcg(ml + row);
        if constexpr (PER == 4) {
          v[d] = __ldcg(reinterpret_cast<const float4*>(p.part_o + row * HD + lane * PER));
        } else {
          const float2 y = __ldcg(reinterpret_cast<const float2*>(p.part_o + row * HD + lane * PER));
          v[d] = make_float4(y.x, y.y, 0.0f, 0.0f);
        }
      }
      float top = m;
#pragma unroll
      for (int d = 0; d < DEEP; ++d) {
        if (j0 + d * step >= g.parts) x[d] = make_float2(-INFINITY, 0.0f);
        top = fmaxf(top, x[d].x);
      }
      const float um = top == -INFINITY ? 0.0f : top, alpha = exp2_fast(m - um);
      l *= alpha;
#pragma unroll
      for (int i = 0; i < PER; ++i) acc[i] *= alpha;
#pragma unroll
      for (int d = 0; d < DEEP; ++d) {
        if (j0 + d * step >= g.parts) break;
        const float f = exp2_fast(x[d].x - um);
        l += x[d].y * f;
        acc[0] += v[d].x * f, acc[1] += v[d].y * f;
        if constexpr (PER == 4) acc[2] += v[d].z * f, acc[3] += v[d].w * f;
      }
      m = top;
    }
    if (many) {
      __syncthreads();  // (the row before has been read)
      if (lane == 0) part_ml[warp] = make_float2(m, l);
#pragma unroll
      for (int i = 0; i < PER; ++i) part[warp][lane * PER + i] = acc[i];
      __syncthreads();
      if (warp != 0) continue;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) top = fmaxf(top, part_ml[w].x);
      const float um = top == -INFINITY ? 0.0f : top;
      l = 0.0f;
#pragma unroll
      for (int i = 0; i < PER; ++i) acc[i] = 0.0f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float f = exp2_fast(part_ml[w].x - um);
        l += part_ml[w].y * f;
#pragma unroll
        for (int i = 0; i < PER; ++i) acc[i] += part[w][lane * PER + i] * f;
      }
    }
    const int rr = g.tile * ROWS + r, tok = rr / group, row = g.q0 + tok, head = g.head * group + rr - tok * group;
    if (row < 0 || row >= p.a.tokens || head < 0 || head >= p.a.n_heads) continue;
    const float inv = g.lk - g.lq + tok + 1 > 0 ? 1.0f / l : 0.0f;
    __half* at = p.a.out + (long long)row * p.a.so[0] + (long long)head * p.a.so[1] + lane * PER;
#pragma unroll
    for (int i = 0; i < PER; i += 2) *reinterpret_cast<uint32_t*>(at + i) = pack_half2(acc[i] * inv, acc[i + 1] * inv);
  }
}

template <int HD, int WM, bool LONG>
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
  uint64_t* seg_full = empty + STAGES;                              // [SEGS]
  Segment* segs = reinterpret_cast<Segment*>(seg_full + Cfg::SEGS);  // [SEGS]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 4);
    }
    for (int i = 0; i < Cfg::SEGS; ++i) mbar_init(&seg_full[i], 1);
    mbar_fence_init();
  }
  __syncthreads();
  pdl_wait_trigger();
  bool ok = true;

  if (warp == 4) {
    // ------------------------------- producer -------------------------------
    // It alone looks up what is to be done, so that the warps that meet at barriers agree on it.
    const FewWork<Cfg::ROWS, Cfg::KB> work(p, lane);
    const Share share = work.share();
    const int pr = p.page_rows, page_size = p.a.page_size;
    int st = 0, issued = 0, seg = 0;
    unsigned use = 0;
    auto publish = [&](const Segment& g) {
      if (lane == 0) {
        segs[seg % Cfg::SEGS] = g;
        mbar_arrive(&seg_full[seg % Cfg::SEGS]);
      }
      ++seg;
    };
    auto wait_empty = [&] { return ok && __all_sync(0xffffffffu, mbar_wait(&empty[st], (use & 1u) ^ 1u)); };
    if (blockIdx.x == 0 && lane == 0) *p.chunks = share.ctas;
    const int chunk = blockIdx.x, begin = share.begin(chunk), end = chunk < share.ctas ? share.begin(chunk + 1) : begin;
    Walk w = {};
    if (begin < end) w = work.find(begin);
    for (int u = begin; u < end && w.tiles != 0 && ok;) {
      const int last = min(w.blks, w.blk + end - u);
      Segment g;
      g.q0 = w.span.q0, g.lq = w.span.lq, g.lk = w.span.lk;
      g.head = w.head, g.tile = w.tile;
      g.first = w.blk, g.last = last, g.blks = w.blks;
      // a chunk has at most two parts: one that begins with it, one that begins behind its beginning
      g.slot = 2 * chunk + (u == begin ? 0 : 1);
      g.chunk0 = chunk, g.parts = 1, g.slot0 = g.slot;
      if (w.blk != 0 || last != w.blks) {
        const int i0 = u - w.blk;
        g.chunk0 = share.chunk_of(i0);
        g.parts = share.chunk_of(i0 + w.blks - 1) - g.chunk0 + 1;
        if (w.blk != 0) {
          const int before_i0 = i0 > 0 ? share.chunk_of(i0 - 1) : -1;
          g.slot0 = 2 * g.chunk0 + (before_i0 == g.chunk0 ? 1 : 0);
        }
      }
      publish(g);
      if (u == begin && lane == 0) p.begins[chunk] = g;
      const int* row = p.a.block_table + (long long)w.s * p.a.max_pages;
      for (int b = w.blk; b < last; ++b) {
        const int keys = min(Cfg::KB, w.span.lk - b * Cfg::KB);
        const int copies = (max(keys, 0) + pr - 1) / pr;  // none: a sequence without positions
        const int pos = b * Cfg::KB + lane * pr;
        int page = 0;
        if (lane < copies) {
          page = __ldg(row + pos / page_size);
          if (page < 0 || page >= p.a.n_pages) {
            page = p.a.n_pages;  // outside the map: zeros arrive
            atomicOr(p.a.status, PAGED_BAD);
          }
        }
        ok = wait_empty();
        if (!ok) break;
        if (lane == 0) mbar_expect_tx(&full[st], (unsigned)(copies * pr * HD * 2 * 2));
        __syncwarp();
        if (lane < copies) {
          uint8_t* k_sm = ring + (size_t)st * 2 * Cfg::TILE + lane * pr * 128;
          const int slot = pos % page_size;
#pragma unroll
          for (int c = 0; c < Cfg::CH; ++c) {
            tma_load_4d(k_sm + c * Cfg::KB * 128, &map_k, c * 64, w.head, slot, page, &full[st]);
            tma_load_4d(k_sm + Cfg::TILE + c * Cfg::KB * 128, &map_v, c * 64, w.head, slot, page, &full[st]);
          }
        }
        ++issued;
        if (++st == STAGES) st = 0, ++use;
      }
      u += last - w.blk;
      if (u < end) work.next(w);
    }
    const Segment none = {};
    publish(none);
    // every copy has landed before the CTA may end
    for (int i = max(0, issued - STAGES); i < issued; ++i)
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
  auto rows_of = [&](const Segment& x) { return min(Cfg::ROWS, x.lq * p.a.group - x.tile * Cfg::ROWS); };
  auto enter = [&](const Segment& x, int (&limit)[2], __half* (&dst)[2], uint32_t (&qa)[HD / 16][4]) {
    const __half* src[2];
    const int live = rows_of(x);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = x.tile * Cfg::ROWS + min(wm * 16 + quad + 8 * i, live - 1);  // rows past the last repeat it, unstored
      const int tok = r / p.a.group, h = x.head * p.a.group + r - tok * p.a.group;
      limit[i] = max(0, x.lk - x.lq + tok + 1);
      src[i] = p.a.q + (long long)(x.q0 + tok) * p.a.sq[0] + h * p.a.sq[1];
      dst[i] = p.a.out + (long long)(x.q0 + tok) * p.a.so[0] + h * p.a.so[1];
    }
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        qa[kk][i] = *reinterpret_cast<const uint32_t*>(src[i & 1] + kk * 16 + (i >> 1) * 8 + pairc);
  };
  int st = 0, seg = 0, limit[2];
  unsigned use = 0;
  __half* dst[2];
  uint32_t qa[HD / 16][4];
  ok = mbar_wait(&seg_full[0], 0);
  if (!few_all(ok)) {
    if (threadIdx.x == 0) atomicOr(p.a.status, 1u << 22);
    return;
  }
  Segment w = segs[0];
  if (w.blks != 0) enter(w, limit, dst, qa);
  while (w.blks != 0) {
    const int lk = w.lk, live = rows_of(w);
    // positions that every row of the tile sees (an earlier token sees fewer)
    const int all_see = max(0, lk - w.lq + w.tile * Cfg::ROWS / p.a.group + 1);
    float o[NT][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[t][i] = 0.0f;

    // the thread's means, and what they stand for, in room that the warps use when they put an item together (all are past
    // the one before: the ring lets none be more than a few stages ahead)
    uint2* const mean = reinterpret_cast<uint2*>(merge) + warp * NT * 32 + lane;
    float2* const weight = ml + warp * 16 + quad;
    auto add_means = [&] {
      __syncwarp();
      const float l0 = weight[0].x, l1 = weight[8].x;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const uint2 c = mean[t * 32];
        add_mean(o[t][0], o[t][1], l0, c.x);
        add_mean(o[t][2], o[t][3], l1, c.y);
      }
      __syncwarp();
    };
    for (int b = w.first; b < w.last; ++b) {  // (without positions: one empty stage)
      if (LONG && b > w.first && (b - w.first) % Cfg::FOLD == 0) {
        if (b - w.first > Cfg::FOLD) add_means();
        float sum[2], inv[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          sum[i] = l[i] + __shfl_xor_sync(0xffffffffu, l[i], 1);
          sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
          inv[i] = 1.0f / sum[i];
          if ((lane & 3) == 0) weight[8 * i].x = sum[i];
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
          mean[t * 32] = make_uint2(take_mean(o[t][0], o[t][1], sum[0], inv[0]), take_mean(o[t][2], o[t][3], sum[1], inv[1]));
      }
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&full[st], use & 1u));
      const uint32_t k_sm = smem_u32(ring + (size_t)st * 2 * Cfg::TILE);
      const uint32_t v_sm = k_sm + Cfg::TILE;
#pragma unroll 1
      for (int step = 0; step < Cfg::KEYS; step += Cfg::SK) {
        const int kb = wk * Cfg::KEYS + step;  // of the stage
        const int key0 = b * Cfg::KB + kb;      // position of its first key
        if (key0 >= lk) break;
        constexpr int SK = Cfg::SK, G = SK / 16;
        float s[2 * G][4];
#pragma unroll
        for (int t = 0; t < 2 * G; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[t][i] = 0.0f;
        const uint32_t k_row = k_sm + (kb + k_key) * 128;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
          for (int g = 0; g < G; ++g) {
            uint32_t kf[4];
            ldsm_x4(k_row + g * 16 * 128 + (kk / 4) * Cfg::KB * 128 + ((((kk & 3) * 2 + k_col) ^ (k_key & 7)) << 4), kf);
            mma_16816(s[2 * g], qa[kk], kf[0], kf[1]);
            mma_16816(s[2 * g + 1], qa[kk], kf[2], kf[3]);
          }
        const bool partly = key0 + SK > all_see;  // some row does not see some of these keys
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int t = 0; t < 2 * G; ++t)
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
          if (LONG && b - w.first >= Cfg::FOLD && (lane & 3) == 0) weight[0].x *= alpha[0], weight[8].x *= alpha[1];
        }
#pragma unroll
        for (int t = 0; t < 2 * G; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[t][i] = exp2_fast(s[t][i] - use_m[i >> 1] + FEW_UP);  // (in this order: maxima can be large)
            l[i >> 1] += s[t][i];
          }
        // probabilities are rounded to fp16 for the tensor cores (2^-11 of each, as much as the output's own rounding; see
        // FEW_UP for the smallest)
        uint32_t pa[G][4];
#pragma unroll
        for (int g = 0; g < G; ++g) {
          pa[g][0] = pack_half2(s[2 * g][0], s[2 * g][1]), pa[g][1] = pack_half2(s[2 * g][2], s[2 * g][3]);
          pa[g][2] = pack_half2(s[2 * g + 1][0], s[2 * g + 1][1]), pa[g][3] = pack_half2(s[2 * g + 1][2], s[2 * g + 1][3]);
        }
        const uint32_t v_row = v_sm + (kb + v_key) * 128;
        auto v_addr = [&](int g, int d16) {
          return v_row + g * 16 * 128 + (d16 / 4) * Cfg::KB * 128 + ((((d16 & 3) * 2 + v_col) ^ (v_key & 7)) << 4);
        };
        if (!partly) {
#pragma unroll
          for (int d = 0; d < HD / 16; ++d)
#pragma unroll
            for (int g = 0; g < G; ++g) {
              uint32_t vf[4];
              ldsm_x4_t(v_addr(g, d), vf);
              mma_16816(o[2 * d], pa[g], vf[0], vf[1]);
              mma_16816(o[2 * d + 1], pa[g], vf[2], vf[3]);
            }
          continue;
        }
        // A probability of zero does not silence a value that is infinite or not a number.  Values behind the last
        // position (whatever the page holds there) are cleared; if one that only some rows see is not finite, the
        // sixteen keys are done one by one, for the rows that see them.
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const int first = key0 + 16 * g;
          if (first >= lk) break;
          uint32_t keep[2], odd = 0;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int key = first + pairc + 8 * i;
            keep[i] = (key < lk ? 0xFFFFu : 0u) | (key + 1 < lk ? 0xFFFF0000u : 0u);
          }
          if (all_see < min(lk, first + 16)) {
#pragma unroll 1
            for (int d = 0; d < HD / 16; ++d) {
              uint32_t vf[4];
              ldsm_x4_t(v_addr(g, d), vf);
#pragma unroll
              for (int i = 0; i < 4; ++i) odd |= not_finite2(vf[i] & keep[i & 1]);
            }
          }
          if (!__any_sync(0xffffffffu, odd != 0)) {
#pragma unroll
            for (int d = 0; d < HD / 16; ++d) {
              uint32_t vf[4];
              ldsm_x4_t(v_addr(g, d), vf);
              mma_16816(o[2 * d], pa[g], vf[0] & keep[0], vf[1] & keep[1]);
              mma_16816(o[2 * d + 1], pa[g], vf[2] & keep[0], vf[3] & keep[1]);
            }
            continue;
          }
#pragma unroll 1
          for (int k = 0; k < 16; ++k) {
            const int from = (lane & ~3) | ((k & 7) >> 1);
            float pk[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float even = k < 8 ? s[2 * g][2 * i] : s[2 * g + 1][2 * i];
              const float uneven = k < 8 ? s[2 * g][2 * i + 1] : s[2 * g + 1][2 * i + 1];
              const float x = __shfl_sync(0xffffffffu, (k & 1) ? uneven : even, from);
              pk[i] = __half2float(__float2half_rn(x));
            }
            const int at = kb + 16 * g + k;
            const bool see0 = first + k < limit[0], see1 = first + k < limit[1];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              uint32_t raw;
              asm volatile("ld.shared.u32 %0, [%1];" : "=r"(raw)
                           : "r"(v_sm + at * 128 + (t / 8) * Cfg::KB * 128 + (((t & 7) ^ (at & 7)) << 4) + pairc * 2));
              const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&raw));
              if (see0) o[t][0] = fmaf(pk[0], v.x, o[t][0]), o[t][1] = fmaf(pk[0], v.y, o[t][1]);
              if (see1) o[t][2] = fmaf(pk[1], v.x, o[t][2]), o[t][3] = fmaf(pk[1], v.y, o[t][3]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
      if (++st == STAGES) st = 0, ++use;
    }

    if (LONG && w.last - w.first > Cfg::FOLD) add_means();
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
    ++seg;
    if (ok) ok = mbar_wait(&seg_full[seg % Cfg::SEGS], (unsigned)(seg / Cfg::SEGS) & 1u);
    ok = few_all(ok);  // (all warps go on, or none does)
    if (!ok) break;
    // the queries of the next item are on their way while this one is put together
    int next_limit[2];
    __half* next_dst[2];
    const Segment next_w = segs[seg % Cfg::SEGS];
    if (next_w.blks != 0) enter(next_w, next_limit, next_dst, qa);
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
    const bool whole = w.first == 0 && w.last == w.blks;
    float* po = p.part_o + (size_t)w.slot * (Cfg::ROWS * HD);
    if (!whole && wk == 0 && (lane & 3) == 0) {
      float2* pml = reinterpret_cast<float2*>(p.part_ml) + (size_t)w.slot * Cfg::ROWS;
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
    w = next_w;
#pragma unroll
    for (int i = 0; i < 2; ++i) limit[i] = next_limit[i], dst[i] = next_dst[i];
  }
  if (!ok && lane == 0) atomicOr(p.a.status, 1u << 22);
}

int few_ctas(const adr_ctx* ctx) { return 2 * (ctx->sm_count > 0 ? ctx->sm_count : 148); }

// Two slots to each of the chunks, ROWS rows to a slot.
template <int HD, int WM>
constexpr size_t few_rows(size_t ctas) {
  using Cfg = FewCfg<HD, WM>;
  return 2 * ctas * Cfg::ROWS;
}
// The number of chunks, then their first segments.
constexpr size_t FEW_HEAD = 256;
size_t few_begins(size_t ctas) { return (ctas * sizeof(Segment) + 255) / 256 * 256; }

template <int HD, int WM>
int launch_few_as(adr_ctx* ctx, cudaStream_t stream, const CUtensorMap& mk, const CUtensorMap& mv, FewParams p,
                  double units) {
  using Cfg = FewCfg<HD, WM>;
  const int g = few_ctas(ctx);
  // (whether some CTA may have more than FOLD stages of one item: by the table's width, and by what all sequences are to each)
  const bool many = (long long)p.a.max_pages * p.a.page_size > (long long)Cfg::FOLD * Cfg::KB && units > (double)g * Cfg::FOLD;
  auto kfn = many ? attention_few_kernel<HD, WM, true> : attention_few_kernel<HD, WM, false>;
  if (int rc = opt_in_smem(ctx, kfn, Cfg::SMEM); rc != ADR_OK) return rc;
  p.most_units = (int)units;
  p.part_ml = p.part_o + few_rows<HD, WM>(g) * HD;
  const int ctas = (int)std::min<double>(g, units);
  if (int rc = launch_serving(ctx, stream, kfn, dim3(ctas), FEW_THREADS, Cfg::SMEM, 2, mk, mv, p); rc != ADR_OK) return rc;
  // the borders between the chunks: none where a CTA is all there is, and none inside an item of one block
  const int borders = ctas - 1;
  if (borders < 1 || (long long)p.a.max_pages * p.a.page_size <= Cfg::KB) return ADR_OK;
  // More warps to a row where an item may have many parts (one sequence of 20000 positions, one key head: 29 -> 20 us; of few
  // parts four are faster: 32 heads over 600 positions 10.1 against 10.9).
  const bool many_parts = (long long)p.a.n_seqs * p.a.n_kv_heads * 32 <= ctas;
  return launch_serving(ctx, stream, many_parts ? few_join_kernel<HD, Cfg::ROWS, 8> : few_join_kernel<HD, Cfg::ROWS, 4>,
                        dim3(borders), many_parts ? 256 : 128, 0, 0, p);
}

// What the units of the launch can be at most: tiles of `rows` rows, blocks of the longest table row.
double few_units(const SeqAttention& a, int rows, bool one_tile_each) {
  const int tile = rows <= 16 ? 16 : 32;
  const double tiles = one_tile_each ? a.n_seqs : (double)a.tokens * a.group / tile + a.n_seqs;
  const int kb = few_kb(a.head_dim);
  const double blocks = (double)(((long long)a.max_pages * a.page_size + kb - 1) / kb);
  return tiles * blocks * a.n_kv_heads;
}

}  // namespace

size_t attention_few_workspace(const adr_ctx* ctx, int head_dim) {
  const size_t g = few_ctas(ctx);
  const size_t rows = std::max(few_rows<128, 1>(g), few_rows<128, 2>(g));
  return FEW_HEAD + few_begins(g) + rows * (head_dim + 2) * sizeof(float);
}

bool attention_few_takes(const SeqAttention& a, int rows, bool one_tile_each) {
  return few_units(a, rows, one_tile_each) < MOST_UNITS;
}

int launch_attention_few(adr_ctx* ctx, cudaStream_t stream, const SeqAttention& a, int rows, int max_rows, void* workspace) {
  FewParams p;
  p.a = a;
  p.max_rows = max_rows;
  p.page_rows = std::min(a.page_size, few_kb(a.head_dim));
  uint8_t* at = static_cast<uint8_t*>(workspace);
  p.chunks = reinterpret_cast<int*>(at);
  p.begins = reinterpret_cast<Segment*>(at + FEW_HEAD);
  p.part_o = reinterpret_cast<float*>(at + FEW_HEAD + few_begins(few_ctas(ctx)));
  CUtensorMap mk, mv;
  if (int rc = pool_map(ctx, &mk, a.k, a.sk, a, p.page_rows); rc != ADR_OK) return rc;
  if (int rc = pool_map(ctx, &mv, a.v, a.sv, a, p.page_rows); rc != ADR_OK) return rc;
  const double units = few_units(a, rows, max_rows <= rows);
  if (a.head_dim == 128)
    return rows <= 16 ? launch_few_as<128, 1>(ctx, stream, mk, mv, p, units)
                      : launch_few_as<128, 2>(ctx, stream, mk, mv, p, units);
  return rows <= 16 ? launch_few_as<64, 1>(ctx, stream, mk, mv, p, units)
                    : launch_few_as<64, 2>(ctx, stream, mk, mv, p, units);
}

}  // namespace adr
