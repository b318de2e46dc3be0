// Attention of many rows per sequence, causal or not, over rows of a projection or over a paged cache.
//
// A tile is 128 rows of one key head: its `group` query heads times 128 / group tokens, token by token, so that the
// heads that share keys share their loads and a causal tile spans few tokens.  A CTA takes NT tiles over the same keys: with
// two of them (neighbouring tokens) the tensor cores work for one while the softmax warps of the other work; with one, two
// or four CTAs to an SM do that for each other (launch_attention_tiles has the choice).
//   * producer: Q once, then K and V in blocks of N = 128 (64) keys through a ring of shared-memory slots, by TMA (whole
//     boxes of rows, or page by page), in the 128-byte swizzle; with N = 64 the tensor-core warp does that too (160
//     threads: four CTAs to an SM have 96 registers a thread, of 192 they would have 80);
//   * S = Q K^T by tcgen05.mma into tensor memory; P = 2^7 exp2(scale2 (S - m)) written back over S by one thread per row;
//     O += P V with P from tensor memory and V as it lies in memory (N-major), O staying in tensor memory;
//   * the product with V begins when half a block's probabilities are there;
//   * the maximum m that a row is scaled by is moved only when a score passes it by more than 2^8: the rescaling of O in
//     tensor memory is rare.  P and the sums are carried times 2^7, so that they end at 2^15, within fp16's range, and what
//     is small keeps as many bits as there are: 11 down to 2^-21 of a row's largest weight, 2^-32 of it below;
//   * the tensor cores' sums round towards zero, 1e-7 of a sum for every 16 products (values of one sign were off by 8.4e-4
//     after 131072 keys, by 7e-3 after a million): every 32768 keys, where that is 2^-12 of the sum, the softmax warps take out
//     of O what a row's mean so far stands for, and the sum begins anew;
//   * when S of a block is complete, so is the product with V before it (the tensor cores run in order), so the softmax
//     warps may touch O and no further barrier is needed;
//   * few tiles over many pages: the keys of each are shared out among CTAs, and a second kernel joins the parts.
// What bounds it: no unit alone.  Two prompts of 8192 tokens, 64/8 heads of 128: 1.9 ms, 1160 TFLOP/s of 1625 in short runs
// and 2.2 to 2.3 ms at the power limit, where the clock falls to 1.62 GHz; the tensor cores are busy for half of the time, the
// exponential unit for 43 %, issue slots for 36 % (2 x 4096 tokens, 32/8 heads), each softmax pass waiting for the product
// before it.  Of 257 tokens and head_dim 64 (images): 39 us where memory wants 10: each CTA begins and ends in about 5
// us of latency, a third of which the other three hide, and every third tile has one row.
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
constexpr size_t TL_PARTS_AT = 16384;  // of the workspace: jobs, then parts
// Probabilities are at most 2^8 (see above); fp16 holds up to just below 2^16.
constexpr float TL_UP = 7.0f;
// From this size on, in powers of two, the maximum is subtracted from the scores before the scale is applied.  Below, one
// fused operation does both, and what the product of maximum and scale loses in fp32 (2^-5 at most) is a factor that a
// row's probabilities and their sum share; above, it would grow past what fp16 and exp2 hold.
constexpr float TL_FAR = 0x1p20f;
__device__ __forceinline__ bool is_far(float base) {  // (not infinity, nor what is not a number)
  return __float_as_uint(fabsf(base)) - __float_as_uint(TL_FAR) < 0x7F800000u - __float_as_uint(TL_FAR);
}
// Keys after which the sum in O begins anew (2048 sums of 16 products lose 2e-4 of what they begin from zero), in kernels of
// their own: with that code 32 x 257 tokens took 41.9 instead of 39.2 us, 4 chunks of 512 over up to 16384 295 instead of 281.
constexpr int TL_LONG = 32768;
// Of every eight pairs of probabilities, those that the FMA units compute; the others go to the exponential unit.
constexpr int BY_FMA = 1;

// N: keys of a block.
template <int HD, int NT, int N>
struct TileCfg {
  static constexpr int CH = HD / 64;
  static constexpr int Q_TILE = TL_M * HD * 2, TILE = N * HD * 2;  // bytes of a tile's queries, of a block's keys
  static constexpr int SLOTS = NT == 2 ? 5 : (HD == 128 ? 2 : 4);
  static constexpr bool ONE = N == 64;  // one warp loads and issues the products
  static constexpr int THREADS = NT * 128 + (ONE ? 32 : 64);
  static constexpr int CTAS = NT == 2 ? 1 : (N == 64 ? 4 : 2);  // to an SM
  static constexpr uint32_t COLS = NT == 2 ? 512 : (N + HD <= 128 ? 128 : 256);  // of tensor memory: N + HD for a tile
  static constexpr uint32_t O_COL = NT * N;
  static constexpr size_t SMEM = 1024 + (size_t)Q_TILE * NT + (size_t)TILE * SLOTS + 8 * (5 * NT + 2 * SLOTS) + 64;
};

struct TileJob {
  SeqSpan span;
  int s, token0;  // first token of the CTA's tiles; s past the last sequence: nothing to do
};

struct TileParams {
  SeqAttention a;
  int tokens_tile;   // tokens of a tile: 128 / group
  int min_rows;      // sequences with fewer rows of a key head than this are left to another kernel
  int page_rows;     // rows of a copy of keys: a page, 128 at most
  int splits;        // parts of a job's keys, each for a CTA of its own
  float2* part_ml;   // [jobs * splits][128]
  float* part_o;     // [jobs * splits][128][head_dim]
  TileJob* job_of;   // [jobs]
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
__device__ __forceinline__ void tmem_st_x16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
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
// The tensor-core warp runs its code with all lanes, so that addresses and descriptors are the same for all of them and
// live in uniform registers; only the instructions themselves are one lane's.  (With one lane in a branch of its own
// each of these instructions was preceded by moves of its six operands: 80 to 110 cycles where the tensor cores take 64.)
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}" : "=r"(r));
  return r;
}
// Lower words of the descriptors of tcgen05.cuh; the upper word is the same for both kinds.
constexpr uint32_t DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) { return ((addr & 0x3FFFFu) >> 4) | ((lbo >> 4) << 16); }
template <bool ACC>
__device__ __forceinline__ void umma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred e, p;\n\t.reg .b64 a, b;\n\tsetp.ne.u32 e, %5, 0;\n\tsetp.ne.u32 p, %6, 0;\n\t"
      "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "n"(DESC_HI), "r"(idesc), "r"(leader), "n"(ACC ? 1 : 0)
      : "memory");
}
// A from tensor memory
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, uint32_t accumulate,
                                        uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred e, p;\n\t.reg .b64 b;\n\tsetp.ne.u32 e, %5, 0;\n\tsetp.ne.u32 p, %6, 0;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b_lo), "n"(DESC_HI), "r"(idesc), "r"(leader), "r"(accumulate)
      : "memory");
}
// mbar_wait in few instructions where the phase is complete, and with no call in it (a call would cost the caller its
// uniform registers): the clock is looked at every 256th time only.
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity) {
  long long t0 = 0;
  for (uint32_t n = 0;; ++n) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    if (done) return true;
    if ((n & 255u) == 255u) {
      const long long t = clock64();
      if (t0 == 0) t0 = t;
      else if (t - t0 > kWaitLimitCycles) return false;
    }
  }
}
__device__ __forceinline__ void arrive_bar(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void commit_one(uint32_t bar, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred e;\n\tsetp.ne.u32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(leader)
      : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 of_pair(uint64_t x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// 2^x of both by the FMA units: x = n + f with n the nearest integer (the rounding of a sum with 1.5 * 2^23, whose low
// bits are n), 2^f on [-1/2, 1/2] by the polynomial of degree 4 of least relative error (Remez exchange in 64 bits:
// 2.6e-6, below the 2^-11 that the result is rounded to), times 2^n.  Below -126 the result is 2^-126, which is zero in
// fp16; NaN stays NaN.
__device__ __forceinline__ uint64_t exp2_fma2(uint64_t x2) {
  float2 x = of_pair(x2);
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.x) : "f"(-126.0f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.y) : "f"(-126.0f));
  x2 = pair_of(x.x, x.y);
  const uint64_t t = add2(x2, pair_of(12582912.0f, 12582912.0f));
  const uint64_t n = add2(t, pair_of(-12582912.0f, -12582912.0f));
  const uint64_t f = fma2(n, pair_of(-1.0f, -1.0f), x2);
  uint64_t q = fma2(f, pair_of(0.009570102207f, 0.009570102207f), pair_of(0.055917859077f, 0.055917859077f));
  q = fma2(f, q, pair_of(0.240247443318f, 0.240247443318f));
  q = fma2(f, q, pair_of(0.693121790886f, 0.693121790886f));
  q = fma2(f, q, pair_of(0.999999284744f, 0.999999284744f));
  const float2 tf = of_pair(t);
  return mul2(q, pair_of(__int_as_float((__float_as_int(tf.x) << 23) + 0x3F800000),
                         __int_as_float((__float_as_int(tf.y) << 23) + 0x3F800000)));
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

// Eight columns of a row's mean, which stand for what has been taken out of the sum in O: kept where the row's output goes
// (16-bit, and zeros where it would not be finite), or its part (32-bit).  `o` comes back as what is left of the sum.
template <bool SPLIT>
__device__ __forceinline__ void add_mean(const uint8_t* at, float weight, uint32_t* o) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 x = SPLIT ? reinterpret_cast<const float2*>(at)[i / 2] : __half22float2(reinterpret_cast<const __half2*>(at)[i / 2]);
    o[i] = __float_as_uint(fmaf(weight, x.x, __uint_as_float(o[i])));
    o[i + 1] = __float_as_uint(fmaf(weight, x.y, __uint_as_float(o[i + 1])));
  }
}
template <bool SPLIT>
__device__ __forceinline__ void take_mean(uint8_t* at, float l, float inv, uint32_t* o) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    float2 x = make_float2(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv);
    if (!(fabsf(x.x) <= 65504.0f)) x.x = 0.0f;
    if (!(fabsf(x.y) <= 65504.0f)) x.y = 0.0f;
    if constexpr (SPLIT) {
      reinterpret_cast<float2*>(at)[i / 2] = x;
    } else {
      const __half2 h = __floats2half2_rn(x.x, x.y);
      reinterpret_cast<__half2*>(at)[i / 2] = h;
      x = __half22float2(h);
    }
    o[i] = __float_as_uint(fmaf(-l, x.x, __uint_as_float(o[i])));
    o[i + 1] = __float_as_uint(fmaf(-l, x.y, __uint_as_float(o[i + 1])));
  }
}

template <int HD, int NT, int N, bool PAGED, bool SPLIT, bool LONG>
__global__ void __launch_bounds__(TileCfg<HD, NT, N>::THREADS, TileCfg<HD, NT, N>::CTAS)
    attention_tiles_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                           const __grid_constant__ CUtensorMap map_v, const __grid_constant__ TileParams p) {
  using Cfg = TileCfg<HD, NT, N>;
  constexpr int CH = Cfg::CH, SLOTS = Cfg::SLOTS, TILE = Cfg::TILE, Q_TILE = Cfg::Q_TILE;
  extern __shared__ uint8_t tile_smem[];
  uint8_t* q_sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(tile_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* ring = q_sm + NT * Q_TILE;  // K of block 0, V of block 0, K of block 1 ...
  uint64_t* q_full = reinterpret_cast<uint64_t*>(ring + SLOTS * TILE);  // [NT]
  uint64_t* s_ready = q_full + NT;   // [NT] scores of a tile are complete
  uint64_t* p_ready = s_ready + NT;  // [NT] its probabilities are
  uint64_t* p_half = p_ready + NT;   // [NT] those of the first 64 keys are
  uint64_t* o_done = p_half + NT;    // [NT] its output is
  uint64_t* full = o_done + NT;      // [SLOTS]
  uint64_t* empty = full + SLOTS;    // [SLOTS]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(empty + SLOTS);
  volatile uint32_t* by_hand = tmem_slot + 1;  // [NT] the softmax warps did this block's product with V
  __shared__ TileJob s_job;
  __shared__ float s_mean[LONG ? NT * TL_M : 1];  // the sum of probabilities that a row's mean (see take_mean) stands for

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr bool ONE = Cfg::ONE;
  constexpr int W_MMA = NT * 4, W_TMA = NT * 4 + (ONE ? 0 : 1);
  if (warp == W_TMA && lane == 0) {
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
    for (int i = 0; i < NT; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&s_ready[i], 1);
      mbar_init(&p_ready[i], 4);
      mbar_init(&p_half[i], 4);
      mbar_init(&o_done[i], 1);
    }
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_fence_init();
  }
  // (The launch before this one may be anyone's and not have its tensor memory yet: none is held while it is waited for.)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __syncwarp();
  if (warp == W_MMA) tmem_alloc(tmem_slot, Cfg::COLS);
  const int job_id = SPLIT ? blockIdx.x / p.splits : blockIdx.x;
  const int head = job_id % p.a.n_kv_heads;
  if (warp == 0) {
    // The CTA's tiles.  The last ones of a sequence, which see most keys, come first, and so do the longest sequences (of
    // 32 at most: of more there are enough to average out): what starts last should be short.
    int id = job_id / p.a.n_kv_heads;
    const int per = NT * p.tokens_tile;
    TileJob job = {};
    job.s = p.a.n_seqs;
    for (int s0 = 0; s0 < p.a.n_seqs; s0 += 32) {
      int mine = 0, keys = 0;
      if (s0 + lane < p.a.n_seqs) {
        const int lq = min(max(__ldg(p.a.cu_q + s0 + lane + 1), 0), p.a.tokens) -
                       min(max(__ldg(p.a.cu_q + s0 + lane), 0), p.a.tokens);
        keys = PAGED ? __ldg(p.a.kv_len + s0 + lane) : lq;
        if (lq > 0 && (long long)lq * p.a.group >= p.min_rows) mine = (lq + per - 1) / per;
      }
      int before = 0;  // tiles of sequences that come before the lane's
      const int first_keys = __shfl_sync(0xffffffffu, keys, 0);
      const bool differ = __any_sync(0xffffffffu, lane < p.a.n_seqs && keys != first_keys);
      if (p.a.n_seqs <= 32 && differ) {
        for (int i = 0; i < p.a.n_seqs; ++i) {
          const int k = __shfl_sync(0xffffffffu, keys, i), n = __shfl_sync(0xffffffffu, mine, i);
          if (k > keys || (k == keys && i < lane)) before += n;
        }
      } else {
        int upto = mine;
        for (int d = 1; d < 32; d <<= 1) {
          const int o = __shfl_up_sync(0xffffffffu, upto, d);
          if (lane >= d) upto += o;
        }
        before = upto - mine;
      }
      const unsigned m = __ballot_sync(0xffffffffu, id >= before && id < before + mine);
      if (m) {
        const int l = __ffs(m) - 1;
        const int behind = __shfl_sync(0xffffffffu, before + mine, l) - 1 - id;  // tiles of the sequence that come later
        job.s = s0 + l;
        job.span = seq_span(p.a.cu_q, p.a.kv_len, job.s, p.a.tokens, p.a.max_pages * p.a.page_size, p.a.status);
        job.token0 = behind * per;
        break;
      }
      if (p.a.n_seqs <= 32) break;
      id -= __shfl_sync(0xffffffffu, before + mine, 31);
    }
    if (lane == 0) {
      s_job = job;
      if (SPLIT && blockIdx.x % p.splits == 0) p.job_of[job_id] = job;
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  // (only now: a launch behind this one may not take the tensor memory that this CTA is waiting for)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
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
    nb[t] = (kend[t] + N - 1) / N;
    nb_max = max(nb_max, nb[t]);
  }
  int j0 = 0;  // this CTA's first block; blocks are counted from it
  if constexpr (SPLIT) {
    const int part = blockIdx.x % p.splits, all = nb[0];
    j0 = all * part / p.splits;
    nb[0] = nb_max = all * (part + 1) / p.splits - j0;
  }
  // keys of a block as the tensor cores take them, in steps of 16
  auto block_n = [&](int t, int j) { return min(N, (kend[t] - (j0 + j) * N + 15) & ~15); };

  if (!ONE && warp == W_TMA) {
    // ------------------------------- producer -------------------------------
    bool ok = true;
    if (nb_max > 0) {
      if (lane == 0) {
        for (int t = 0; t < NT; ++t) {
          if (nb[t] == 0) continue;
          mbar_expect_tx(&q_full[t], (unsigned)(CH * p.tokens_tile * p.a.group * 128));
          for (int c = 0; c < CH; ++c)
            tma_load_3d(q_sm + t * Q_TILE + c * (TL_M * 128), &map_q, c * 64, head * p.a.group,
                        span.q0 + token0 + t * p.tokens_tile, &q_full[t]);
        }
      }
      int issued = 0;
      for (int i = 0; i < 2 * nb_max; ++i) {
        const int st = i % SLOTS, j = j0 + (i >> 1);
        uint8_t* dst = ring + st * TILE;
        const CUtensorMap* map = (i & 1) ? &map_v : &map_k;
        if constexpr (PAGED) {
          const int pr = p.page_rows;
          const int copies = (min(N, lk - j * N) + pr - 1) / pr;
          const int pos = j * N + lane * pr;
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
              tma_load_4d(dst + c * (N * 128) + lane * pr * 128, map, c * 64, head, pos % p.a.page_size, page, &full[st]);
        } else {
          if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&empty[st], ((unsigned)(i / SLOTS) & 1u) ^ 1u));
          if (!ok) break;
          if (lane == 0) {
            mbar_expect_tx(&full[st], TILE);
            for (int c = 0; c < CH; ++c)
              tma_load_3d(dst + c * (N * 128), map, c * 64, head, span.q0 + j * N, &full[st]);
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
    if (nb_max > 0) {
      // (Nothing here leaves the loops early: a lane whose wait ran out skips the waits and instructions that follow.)
      bool ok = true;
      const uint32_t leader = elect_one();
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      const uint32_t q_lo = desc_lo(smem_u32(q_sm), 16), k_lo = desc_lo(smem_u32(ring), 16),
                     v_lo = desc_lo(smem_u32(ring), N * 128);
      const uint32_t b_q = smem_u32(q_full), b_s = smem_u32(s_ready), b_p = smem_u32(p_ready), b_h = smem_u32(p_half),
                     b_o = smem_u32(o_done), b_full = smem_u32(full), b_empty = smem_u32(empty);
      constexpr uint32_t CHUNK = N * 128 / 16, Q_CHUNK = TL_M * 128 / 16, SLOT = TILE / 16;  // steps of a descriptor
      int all_see[NT];  // keys that every row of a tile sees
#pragma unroll
      for (int t = 0; t < NT; ++t) all_see[t] = p.a.causal ? max(0, lk - lq + token0 + t * p.tokens_tile + 1) : lk;
      uint32_t have_o[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) have_o[t] = 0;
      // (the vote tells the compiler, too, that the lanes are together again)
      auto wait = [&](uint32_t bar, uint32_t parity) { ok = __all_sync(0xffffffffu, ok && wait_bar(bar, parity)); };
      auto k_slot = [](int j) { return (uint32_t)(2 * j) % SLOTS; };
      auto v_slot = [](int j) { return (uint32_t)(2 * j + 1) % SLOTS; };
      auto wait_k = [&](int j) { wait(b_full + k_slot(j) * 8, ((uint32_t)(2 * j) / SLOTS) & 1u); };
      auto wait_v = [&](int j) { wait(b_full + v_slot(j) * 8, ((uint32_t)(2 * j + 1) / SLOTS) & 1u); };
      auto scores = [&](int t, int j, bool last) {
        tc_fence_after_sync();
        if (!ok) return;
        const uint32_t idesc = umma_idesc_f16(block_n(t, j), false), go = leader;
        const uint32_t qa = q_lo + t * (Q_TILE / 16), ka = k_lo + k_slot(j) * SLOT;
        umma_ss<false>(tm + t * N, qa, ka, idesc, go);
#pragma unroll
        for (int i = 1; i < CH * 4; ++i)
          umma_ss<true>(tm + t * N, qa + (i / 4) * Q_CHUNK + (i % 4) * 2, ka + (i / 4) * CHUNK + (i % 4) * 2, idesc, go);
        commit_one(b_s + t * 8, go);
        if (last) commit_one(b_empty + k_slot(j) * 8, go);
      };
      auto output = [&](int t, int j, bool last) {
        wait(b_h + t * 8, (uint32_t)j & 1u);
        tc_fence_after_sync();
        constexpr uint32_t idesc = umma_idesc_f16(HD, true);
        const uint32_t vd = v_lo + v_slot(j) * SLOT, d = tm + Cfg::O_COL + t * HD, a = tm + t * N;
        if ((j0 + j + 1) * N <= all_see[t]) {
          if (!ok) return;
          const uint32_t go = leader;
          umma_ts(d, a, vd, idesc, have_o[t], go);
#pragma unroll
          for (int i = 1; i < N / 32; ++i) umma_ts(d, a + i * 8, vd + i * 128, idesc, 1u, go);
          wait(b_p + t * 8, (uint32_t)j & 1u);
          tc_fence_after_sync();
          if (!ok) return;
          const uint32_t go2 = leader;
#pragma unroll
          for (int i = N / 32; i < N / 16; ++i) umma_ts(d, a + i * 8, vd + i * 128, idesc, 1u, go2);
        } else {
          // a block that not every row sees whole: it may be short, or done already
          wait(b_p + t * 8, (uint32_t)j & 1u);
          tc_fence_after_sync();
          if (!ok) return;
          const uint32_t go = __shfl_sync(0xffffffffu, by_hand[t], 0) == 0 ? leader : 0;
          const int n = block_n(t, j) / 16;
          for (int i = 0; i < n; ++i) umma_ts(d, a + i * 8, vd + i * 128, idesc, have_o[t] | (uint32_t)i, go);
        }
        have_o[t] = 1;
        const uint32_t go = leader;
        if (last) commit_one(b_empty + v_slot(j) * 8, go);
        if (j == nb[t] - 1) commit_one(b_o + t * 8, go);
      };
      // tile 1 sees at least what tile 0 sees, so a block's last user is tile 1 where it takes part
      auto last = [&](int t, int j) { return !ONE && (NT == 1 || t == 1 || j >= nb[NT - 1]); };
      // Without a producer: copy i of K of block 0, V of block 0, K of block 1 ..., into a slot that is free.
      int issued = 0;
      auto load = [&](int i) {
        if (!ok || i >= 2 * nb_max) return;
        if (leader) {
          mbar_expect_tx(&full[i % SLOTS], TILE);
          for (int c = 0; c < CH; ++c)
            tma_load_3d(ring + (i % SLOTS) * TILE + c * (N * 128), (i & 1) ? &map_v : &map_k, c * 64, head,
                        span.q0 + (i >> 1) * N, &full[i % SLOTS]);
        }
        issued = i + 1;
        __syncwarp();
      };
      if constexpr (ONE) {
        static_assert(NT == 1 && !PAGED && !SPLIT && SLOTS == 4, "");
        if (leader) {
          mbar_expect_tx(q_full, (unsigned)(CH * p.tokens_tile * p.a.group * 128));
          for (int c = 0; c < CH; ++c)
            tma_load_3d(q_sm + c * (TL_M * 128), &map_q, c * 64, head * p.a.group, span.q0 + token0, q_full);
        }
        __syncwarp();
        for (int i = 0; i < SLOTS; ++i) load(i);
      }
      wait_k(0);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (nb[t] == 0) continue;
        wait(b_q + t * 8, 0);
        scores(t, 0, last(t, 0));
      }
#pragma unroll 1
      for (int j = 0; j < nb_max && ok; ++j) {
        wait_v(j);
        if (j + 1 < nb_max) wait_k(j + 1);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if (j < nb[t]) output(t, j, last(t, j));
          if (j + 1 < nb[t]) scores(t, j + 1, last(t, j + 1));
        }
        if constexpr (ONE) {
          // The probabilities of block j are there, so its scores are, and what was issued before them: the product with V of
          // block j - 1.  Their slots are free.
          if (j > 0) load(2 * j + 3);
          load(2 * j + 4);
        }
      }
      if constexpr (ONE) {
        // every copy has landed before the CTA may end
        bool landed = mbar_wait(q_full, 0);
        for (int i = max(0, issued - SLOTS); i < issued; ++i)
          if (!mbar_wait(&full[i % SLOTS], (unsigned)(i / SLOTS) & 1u)) landed = false;
        ok = __all_sync(0xffffffffu, ok && landed);
      }
      if (!ok && lane == 0) atomicOr(p.a.status, 1u << 24);
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
    const int warp_most = __reduce_max_sync(0xffffffffu, limit);  // keys that some row of the warp sees
    const int my_end = NT == 2 && t == 1 ? kend[NT - 1] : kend[0];
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lanes + (uint32_t)(t * N), o_at = tmem + lanes + Cfg::O_COL + (uint32_t)(t * HD);
    // scores in powers of two; the sign of the scale, and a scale of zero, go into the scores, so that the largest product is
    // the maximum, what is masked stays infinite, and zero times infinity is not a number
    const float scale2 = fmaxf(fabsf(p.a.scale) * 1.4426950408889634f, 1e-30f);
    const float sign = p.a.scale > 0.0f ? 1.0f : p.a.scale < 0.0f ? -1.0f : 0.0f;
    const float slack = 8.0f / scale2;
    float m = -INFINITY, l = 0.0f;
    bool ok = true;

    // where the row's output goes, or its part; computed anew (the compiler would hold it in registers through the loop)
    auto row_at = [&]() -> uint8_t* {
      int r = row;
      asm volatile("" : "+r"(r));
      if constexpr (SPLIT) return reinterpret_cast<uint8_t*>(p.part_o + ((size_t)blockIdx.x * TL_M + r) * HD);
      const int tk = r / p.a.group;
      return reinterpret_cast<uint8_t*>(p.a.out + (long long)(span.q0 + first + tk) * p.a.so[0] +
                                        (long long)(head * p.a.group + r - tk * p.a.group) * p.a.so[1]);
    };
    constexpr int MEAN = SPLIT ? 4 : 2;  // bytes of a column there
    constexpr int FOLD = TL_LONG / N;
    const uint32_t b_s = smem_u32(&s_ready[t]), b_p = smem_u32(&p_ready[t]), b_h = smem_u32(&p_half[t]);
    for (int j = 0; j < my_nb; ++j) {
      const int key0 = (j0 + j) * N;
      const bool partly = key0 + N > all_see;  // some row does not see some key of the block
      uint8_t* v = ring + ((2 * j + 1) % SLOTS) * TILE;
      bool hand = false;
      // V is waited for, cleared behind the end, and searched for what may not be multiplied by zero.  A thread takes a
      // 16-byte piece of every 128 / (HD / 8)-th row (the swizzle only permutes a row's pieces).
      auto look_at_values = [&] {
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&full[(2 * j + 1) % SLOTS], (unsigned)((2 * j + 1) / SLOTS) & 1u));
        const int from = max(0, all_see - key0), end = min(N, lk - key0);
        const int read = min(N, (my_end - key0 + 15) & ~15);  // rows that the tensor cores read
        constexpr int LPR = HD / 8, STEP = 128 / LPR;
        uint4* at = reinterpret_cast<uint4*>(v + ((row % LPR) / 8) * (N * 128) + (row % 8) * 16);
        uint32_t odd = 0;
        int r = from + row / LPR;
        for (; r + 3 * STEP < min(end, read); r += 4 * STEP) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint4 x = at[(r + i * STEP) * 8];
            odd |= not_finite2(x.x) | not_finite2(x.y) | not_finite2(x.z) | not_finite2(x.w);
          }
        }
#pragma unroll 1
        for (; r < read; r += STEP) {
          if (r >= end) {
            at[r * 8] = make_uint4(0, 0, 0, 0);
          } else {
            const uint4 x = at[r * 8];
            odd |= not_finite2(x.x) | not_finite2(x.y) | not_finite2(x.z) | not_finite2(x.w);
          }
        }
        fence_proxy_async();
        hand = tile_any(t, odd != 0);
      };
      // While the scores are computed; but with two slots a block's V is loaded only when the product with the one before
      // is done: it is looked at behind the probabilities then.  (Nor may it be waited for before the scores: a barrier's
      // phase can be told from the next but one only when the one between is known to be complete.)
      const bool early = SLOTS > 2 || j == 0;
      if (partly && early) look_at_values();
      if (ok) ok = __all_sync(0xffffffffu, wait_bar(b_s, (unsigned)j & 1u));
      tc_fence_after_sync();
      if (ok && warp_live) {
        const int chunks = partly ? (min(N, my_end - key0) + 31) / 32 : N / 32;  // of 32 keys
        // the row's maximum
        float mx;
        if (!partly && sign == 1.0f) {
          uint32_t s[N];
#pragma unroll
          for (int c = 0; c < N / 32; ++c) tmem_ld_x32(s_at + c * 32, s + c * 32);
          tmem_ld_wait();
          float top[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) top[i] = fmaxf(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1]));
#pragma unroll
          for (int i = 16; i < N; i += 2)
            top[(i >> 1) & 7] = max3(top[(i >> 1) & 7], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
          mx = max3(max3(top[0], top[1], top[2]), max3(top[3], top[4], top[5]), fmaxf(top[6], top[7]));
        } else {
          // the scores as they are to be, written back; what no row of the warp sees is passed over
          mx = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < chunks; ++c) {
            const int k = key0 + c * 32;
            if (k >= warp_most) break;
            uint32_t s[32];
            tmem_ld_x32(s_at + c * 32, s);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              s[i] = __float_as_uint(__uint_as_float(s[i]) * sign);
              if (k + i >= limit) s[i] = 0xFF800000u;  // -infinity
              mx = fmaxf(mx, __uint_as_float(s[i]));
            }
            tmem_st_x32(s_at + c * 32, s);
          }
          tmem_wait_st();
        }
        // (a first maximum moves from -infinity: nothing is summed or in O yet but zeros.  The difference is exact where
        // it matters; a sum with the slack would round it away in large maxima.)
        const bool move = mx - m > slack;
        float base = m * scale2;
        const bool fold = LONG && j % FOLD == 0 && j > 0;
        if (__any_sync(0xffffffffu, move || fold || is_far(base))) {
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
            if (LONG && j > FOLD) s_mean[t * TL_M + row] *= alpha;
          }
          if (fold) {
            const float weight = j > FOLD ? s_mean[t * TL_M + row] : 0.0f, inv = 1.0f / l;
            uint8_t* at = row_at();
            tmem_wait_st();
#pragma unroll 1
            for (int c = 0; c < HD; c += 8, at += 8 * MEAN) {
              uint32_t o[8];
              tmem_ld_x8(o_at + c, o);
              tmem_ld_wait();
              if (live) {
                if (j > FOLD) add_mean<SPLIT>(at, weight, o);
                take_mean<SPLIT>(at, l, inv, o);
              }
              __syncwarp();
              tmem_st_x8(o_at + c, o);
            }
            s_mean[t * TL_M + row] = l;
          }
          base = m * scale2;
          if (__any_sync(0xffffffffu, is_far(base))) {
            const float zero = m == -INFINITY ? 0.0f : m;
#pragma unroll 1
            for (int c = 0; c < chunks * 32 && key0 + c < warp_most; c += 8) {
              uint32_t s[8];
              tmem_ld_x8(s_at + c, s);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 8; ++i) s[i] = __float_as_uint(__uint_as_float(s[i]) - zero);
              tmem_st_x8(s_at + c, s);
            }
            tmem_wait_st();
            base = 0.0f;
          }
        }
        if (m == -INFINITY) base = 0.0f;
        const uint64_t mul = pair_of(scale2, scale2), sub = pair_of(TL_UP - base, TL_UP - base);
        uint64_t sum[2] = {0, 0};
        auto powers = [&](const uint32_t (&s)[32], uint32_t (&pk)[16]) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            uint64_t x = fma2(pair_of(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), mul, sub);
            if ((i & 7) >= 8 - BY_FMA) {
              x = exp2_fma2(x);
            } else {
              const float2 e = of_pair(x);
              x = pair_of(exp2_fast(e.x), exp2_fast(e.y));
            }
            sum[i & 1] = add2(sum[i & 1], x);
            const float2 e = of_pair(x);
            pk[i] = pack_half2(e.x, e.y);
          }
        };
        // The scores are read a second time, 32 at a time and 32 ahead, rather than kept: that leaves registers for many
        // exponentials at once.  Probabilities are written over scores that have been read.
        if (!partly) {
          constexpr bool AHEAD = N == 128;  // (registers for that are there where few CTAs share an SM)
          uint32_t s[AHEAD ? 2 : 1][32];
          tmem_ld_x32(s_at, s[0]);
#pragma unroll
          for (int c = 0; c < N / 32; ++c) {
            tmem_ld_wait();
            if (AHEAD && c + 1 < N / 32) tmem_ld_x32(s_at + (c + 1) * 32, s[(c + 1) & 1]);
            uint32_t pk[16];
            powers(s[AHEAD ? c & 1 : 0], pk);
            tmem_st_x16(s_at + c * 16, pk);
            if (!AHEAD && c + 1 < N / 32) tmem_ld_x32(s_at + (c + 1) * 32, s[0]);
            if (c == N / 64 - 1) {
              // the tensor cores may begin
              tmem_wait_st();
              tc_fence_before_sync();
              __syncwarp();
              if (lane == 0) arrive_bar(b_h);
            }
          }
        } else {
#pragma unroll 1
          for (int c = 0; c < chunks; ++c) {
            uint32_t pk[16];
            if (key0 + c * 32 < warp_most) {
              uint32_t s[32];
              tmem_ld_x32(s_at + c * 32, s);
              tmem_ld_wait();
              powers(s, pk);
            } else {
#pragma unroll
              for (int i = 0; i < 16; ++i) pk[i] = 0;
            }
            tmem_st_x16(s_at + c * 16, pk);
          }
        }
        const float2 total = of_pair(add2(sum[0], sum[1]));
        l += total.x + total.y;
      }
      tmem_wait_st();
      if (partly && !early) look_at_values();
      if (hand && ok && warp_live) {
        // this block's product by hand
        const int end = min(N, my_end - key0);
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
              const uint4 x = *reinterpret_cast<const uint4*>(v + (c / 64) * (N * 128) + r * 128 + (((c / 8) ^ r) & 7) * 16);
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
      if (partly && row == 0) by_hand[t] = hand ? 1u : 0u;
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if (partly || !ok || !warp_live) arrive_bar(b_h);
        arrive_bar(b_p);
      }
    }
    if (my_nb > 0) {
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&o_done[t], 0));
      tc_fence_after_sync();
    }
    if (SPLIT && ok && live) p.part_ml[(size_t)blockIdx.x * TL_M + row] = make_float2(m * scale2, l);
    if (ok && warp_live) {
      // A row that sees no key gets zeros; one whose scores are all -infinity has no softmax, and is not a number.  (Its sum
      // is not zero: see exp2_fma2.)
      const float inv = limit > 0 ? 1.0f / (m == -INFINITY ? 0.0f : l) : 0.0f;
      __half* dst = p.a.out + (long long)(span.q0 + first + tok) * p.a.so[0] +
                    (long long)(head * p.a.group + row - tok * p.a.group) * p.a.so[1];
      const bool folded = LONG && my_nb > FOLD;
#pragma unroll
      for (int c = 0; c < HD; c += 32) {
        uint32_t o[32];
        if (my_nb > 0) {
          tmem_ld_x32(o_at + c, o);
          tmem_ld_wait();
        }
        if (folded && live) {
          const float weight = s_mean[t * TL_M + row];
          const uint8_t* at = row_at() + c * MEAN;
#pragma unroll
          for (int i = 0; i < 32; i += 8) add_mean<SPLIT>(at + i * MEAN, weight, o + i);
        }
        if (SPLIT && live && my_nb > 0) {
          float4* to = reinterpret_cast<float4*>(p.part_o + ((size_t)blockIdx.x * TL_M + row) * HD + c);
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            __stcg(to + i / 4, make_float4(__uint_as_float(o[i]), __uint_as_float(o[i + 1]), __uint_as_float(o[i + 2]),
                                           __uint_as_float(o[i + 3])));
        }
        if (!SPLIT && live) {
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

// Joins a job's parts in their order: a block has 16 rows of a job, a warp one row at a time, HD / 32 columns to a lane.
constexpr int TJ_ROWS = 16, TJ_THREADS = 128, TL_MAX_SPLITS = 32;
template <int HD>
__global__ void __launch_bounds__(TJ_THREADS) tiles_join_kernel(const __grid_constant__ TileParams p) {
  constexpr int PER = HD / 32, DEEP = 8;  // columns of a lane, parts whose loads are in flight
  pdl_wait_trigger();
  const int id = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const TileJob job = p.job_of[id];
  const int head = id % p.a.n_kv_heads;
  const int n_tok = job.s < p.a.n_seqs ? min(p.tokens_tile, job.span.lq - job.token0) : 0;
  for (int r = blockIdx.y * TJ_ROWS + warp; r < min(n_tok * p.a.group, (int)(blockIdx.y + 1) * TJ_ROWS); r += TJ_THREADS / 32) {
    float m = -INFINITY, l = 0.0f, acc[PER] = {};
    for (int s0 = 0; s0 < p.splits; s0 += DEEP) {
      float2 x[DEEP];
      float v[DEEP][PER];
#pragma unroll
      for (int i = 0; i < DEEP; ++i) {
        const size_t at = ((size_t)id * p.splits + min(s0 + i, p.splits - 1)) * TL_M + r;
        x[i] = __ldcg(p.part_ml + at);
        if constexpr (PER == 4) {
          const float4 y = __ldcg(reinterpret_cast<const float4*>(p.part_o + at * HD + lane * PER));
          v[i][0] = y.x, v[i][1] = y.y, v[i][2] = y.z, v[i][3] = y.w;
        } else {
          const float2 y = __ldcg(reinterpret_cast<const float2*>(p.part_o + at * HD + lane * PER));
          v[i][0] = y.x, v[i][1] = y.y;
        }
      }
      float top = m;
#pragma unroll
      for (int i = 0; i < DEEP; ++i) {
        if (s0 + i >= p.splits) x[i] = make_float2(-INFINITY, 0.0f);
        top = fmaxf(top, x[i].x);
      }
      const float um = top == -INFINITY ? 0.0f : top, alpha = exp2_fast(m - um);
      l *= alpha;
#pragma unroll
      for (int c = 0; c < PER; ++c) acc[c] *= alpha;
#pragma unroll
      for (int i = 0; i < DEEP; ++i) {
        if (x[i].x == -INFINITY && x[i].y == 0.0f) continue;  // a part that saw nothing has put down no output
        const float f = exp2_fast(x[i].x - um);
        l += x[i].y * f;
#pragma unroll
        for (int c = 0; c < PER; ++c) acc[c] += v[i][c] * f;
      }
      m = top;
    }
    const int tok = job.token0 + r / p.a.group, row = job.span.q0 + tok;
    if (row < 0 || row >= p.a.tokens) continue;  // (what another call left, if this one gave up)
    const float inv = job.span.lk - job.span.lq + tok + 1 > 0 ? 1.0f / l : 0.0f;
    __half* to = p.a.out + (long long)row * p.a.so[0] + (long long)(head * p.a.group + r % p.a.group) * p.a.so[1] + lane * PER;
#pragma unroll
    for (int c = 0; c < PER; c += 2) *reinterpret_cast<uint32_t*>(to + c) = pack_half2(acc[c] * inv, acc[c + 1] * inv);
  }
}

// Rows of a projection, [64 columns, heads, rows] boxes of a [tokens, heads, head_dim] view.
int rows_map(adr_ctx* ctx, CUtensorMap* map, const __half* base, const SeqAttention& a, int n_heads, long long s_row,
             long long s_head, int box_heads, int box_rows) {
  const uint64_t dims[3] = {(uint64_t)a.head_dim, (uint64_t)n_heads, (uint64_t)a.tokens};
  const uint64_t strides[2] = {n_heads > 1 ? (uint64_t)s_head * 2 : (uint64_t)a.head_dim * 2,
                               a.tokens > 1 ? (uint64_t)s_row * 2 : (uint64_t)a.head_dim * 2};
  const uint32_t box[3] = {64u, (uint32_t)box_heads, (uint32_t)box_rows};
  return tma_encode(ctx, map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Jobs that there can be at most: each sequence fills up its last one.
long long most_jobs(const SeqAttention& a, int nt) {
  const long long per = nt * (TL_M / a.group);
  return std::min<long long>(a.tokens, (a.tokens + a.n_seqs * (per - 1)) / per) * a.n_kv_heads;
}

template <int HD, int NT, int N, bool PAGED, bool SPLIT, bool LONG>
int launch_tiles_as(adr_ctx* ctx, cudaStream_t stream, const SeqAttention& a, int min_rows, int splits = 1,
                    uint8_t* workspace = nullptr) {
  using Cfg = TileCfg<HD, NT, N>;
  auto kfn = attention_tiles_kernel<HD, NT, N, PAGED, SPLIT, LONG>;
  if (int rc = opt_in_smem(ctx, kfn, Cfg::SMEM); rc != ADR_OK) return rc;
  TileParams p = {};
  p.a = a;
  p.tokens_tile = TL_M / a.group;
  p.min_rows = min_rows;
  p.page_rows = std::min(a.page_size, N);
  CUtensorMap mq, mk, mv;
  if (int rc = rows_map(ctx, &mq, a.q, a, a.n_heads, a.sq[0], a.sq[1], a.group, p.tokens_tile); rc != ADR_OK) return rc;
  if constexpr (PAGED) {
    if (int rc = pool_map(ctx, &mk, a.k, a.sk, a, p.page_rows); rc != ADR_OK) return rc;
    if (int rc = pool_map(ctx, &mv, a.v, a.sv, a, p.page_rows); rc != ADR_OK) return rc;
  } else {
    if (int rc = rows_map(ctx, &mk, a.k, a, a.n_kv_heads, a.sk[1], a.sk[2], 1, N); rc != ADR_OK) return rc;
    if (int rc = rows_map(ctx, &mv, a.v, a, a.n_kv_heads, a.sv[1], a.sv[2], 1, N); rc != ADR_OK) return rc;
  }
  const long long jobs = most_jobs(a, NT);
  if (jobs > 0x40000000LL) return ADR_ERR_SHAPE;
  p.splits = splits;
  if constexpr (SPLIT) {
    p.job_of = reinterpret_cast<TileJob*>(workspace);
    p.part_ml = reinterpret_cast<float2*>(workspace + TL_PARTS_AT);
    p.part_o = reinterpret_cast<float*>(p.part_ml + jobs * splits * TL_M);
  }
  const dim3 ctas((unsigned)(jobs * splits));
  if (int rc = launch_serving(ctx, stream, kfn, ctas, Cfg::THREADS, Cfg::SMEM, 2, mq, mk, mv, p); rc != ADR_OK || !SPLIT)
    return rc;
  return launch_serving(ctx, stream, tiles_join_kernel<HD>, dim3((unsigned)jobs, TL_M / TJ_ROWS), TJ_THREADS, 0, 0, p);
}

// Parts at once: as many as CTAs that the GPU holds, two to an SM.
int tile_parts(const adr_ctx* ctx) { return 2 * (ctx->sm_count > 0 ? ctx->sm_count : 148); }

}  // namespace

size_t attention_tiles_workspace(const adr_ctx* ctx, int head_dim) {
  return TL_PARTS_AT + (size_t)tile_parts(ctx) * TL_M * (head_dim + 2) * sizeof(float);
}

int attention_tiles_splits(const adr_ctx* ctx, const SeqAttention& a) {
  // Few tiles over many keys: the keys of each are shared out among CTAs, at least 256 to each (220 tokens over 1423 positions,
  // 16/16 heads: 23.8 us, of 512 to each 27.2).
  const long long jobs = most_jobs(a, 1), keys = (long long)a.max_pages * a.page_size;
  if ((size_t)jobs * sizeof(TileJob) > TL_PARTS_AT) return 1;
  const long long splits = std::min<long long>({tile_parts(ctx) / std::max(jobs, 1LL), keys / 256, TL_MAX_SPLITS});
  return (int)std::max(splits, 1LL);
}

int launch_attention_tiles(adr_ctx* ctx, cudaStream_t stream, const SeqAttention& a, int max_q, int min_rows, void* workspace) {
  // One tile to a CTA and two CTAs to an SM, or two tiles that share their keys.  The former hides one CTA's start and
  // end behind the other's work, the latter halves what is loaded; measured on 32/32 and 32/8 heads: head_dim 64 in one
  // tile everywhere (4 x 2048 tokens 135 against 146 us); head_dim 128 of prompts up to 2048 tokens in one (16 x 512: 96
  // against 111 us, 2 x 6000: 576 against 544), over pages, whose copies are many, up to 512 positions only (16 x 200: 42
  // against 43 us, 4 x 512 over 1024: 64 against 59).
  // Blocks of 64 keys take half the tensor memory where head_dim is 64, and without a warp for the copies four CTAs fit on an
  // SM.  Worth it where there are enough tiles for all of them, of long causal ones, which differ, twice as many: 16/16 heads,
  // causal: 4 x 2048 tokens (1024 tiles) 93 against 78 us, 16 x 512 (1024) 39 against 39; all keys seen: 16 x 512 36 against
  // 42, 4 x 2048 107 against 120; 32/32 heads, causal: 1 x 2048 (512 tiles) 46 against 42, 2 x 8192 (4096) 749 against 813.
  if (a.block_table == nullptr) {
    const bool many_keys = max_q > TL_LONG;
    if (a.head_dim == 64) {
      if (most_jobs(a, 1) > (a.causal && max_q > 512 ? 4 : 2) * tile_parts(ctx))
        return many_keys ? launch_tiles_as<64, 1, 64, false, false, true>(ctx, stream, a, min_rows)
                         : launch_tiles_as<64, 1, 64, false, false, false>(ctx, stream, a, min_rows);
      return many_keys ? launch_tiles_as<64, 1, 128, false, false, true>(ctx, stream, a, min_rows)
                       : launch_tiles_as<64, 1, 128, false, false, false>(ctx, stream, a, min_rows);
    }
    if (many_keys) return launch_tiles_as<128, 2, 128, false, false, true>(ctx, stream, a, min_rows);
    return max_q <= 2048 ? launch_tiles_as<128, 1, 128, false, false, false>(ctx, stream, a, min_rows)
                         : launch_tiles_as<128, 2, 128, false, false, false>(ctx, stream, a, min_rows);
  }
  const int splits = attention_tiles_splits(ctx, a);
  const long long keys = (long long)a.max_pages * a.page_size;
  const bool many_keys = keys > (long long)splits * TL_LONG;
  uint8_t* const ws = static_cast<uint8_t*>(workspace);
  if (splits > 1) {
    if (a.head_dim == 64)
      return many_keys ? launch_tiles_as<64, 1, 128, true, true, true>(ctx, stream, a, min_rows, splits, ws)
                       : launch_tiles_as<64, 1, 128, true, true, false>(ctx, stream, a, min_rows, splits, ws);
    return many_keys ? launch_tiles_as<128, 1, 128, true, true, true>(ctx, stream, a, min_rows, splits, ws)
                     : launch_tiles_as<128, 1, 128, true, true, false>(ctx, stream, a, min_rows, splits, ws);
  }
  if (a.head_dim == 64)
    return many_keys ? launch_tiles_as<64, 1, 128, true, false, true>(ctx, stream, a, min_rows)
                     : launch_tiles_as<64, 1, 128, true, false, false>(ctx, stream, a, min_rows);
  if (many_keys) return launch_tiles_as<128, 2, 128, true, false, true>(ctx, stream, a, min_rows);
  return keys <= 512 ? launch_tiles_as<128, 1, 128, true, false, false>(ctx, stream, a, min_rows)
                     : launch_tiles_as<128, 2, 128, true, false, false>(ctx, stream, a, min_rows);
}

}  // namespace adr
