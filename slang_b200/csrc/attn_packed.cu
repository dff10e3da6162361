// Causal attention of packed prompts on tcgen05 (sb_attn_prefill_packed):
// sequences of different lengths end to end in one tensor, grouped heads, a
// sliding window, more keys than queries (a cached prefix).
//
// The rows of a query tile are (token, query head of the kv head's group): 128 /
// group tokens of all heads that share K and V, so each K/V block serves the
// whole group.  Two kernels:
//
// attn_packed_pair_kernel (head_dim 128 and 256): a CTA pair (cta_group::2) takes
// two query tiles, one per CTA.  The pair's MMAs run over 256 rows; each CTA holds
// half of a block's keys and half of its values' dims, so a block is loaded and read
// from shared memory half as often.  One CTA alone is bound by shared memory,
// not by its tensor cores: at head_dim 256 a block costs it 128 KB of operand reads for
// Q K^T, 64 KB for P V and 128 KB of TMA writes, 2560 cycles at 128 bytes per cycle
// against 2048 of MMA (measured 1.70 us = 3200 cycles); the pair needs 1536.
//   warp 0        TMA: this CTA's Q tile, then its halves of K and V through a ring
//                 of slots whose arrival is counted in the even CTA.
//   warp 1        even CTA, one thread: tcgen05.mma S = Q K^T, then O += P V (P from
//                 tensor memory).
//   warps 2, 3    zero the V rows past the sequence's end in its last block: those
//                 rows belong to another sequence, and 0 times a NaN there would
//                 reach this one.
//   warps 4 .. 7  softmax, a thread per query row: the block's scores of the row from
//                 tensor memory, running maximum m (raised, with O rescaled, only when a
//                 score passes it by 2^8) and sum l, p = 2^(s - m) in the input
//                 type to tensor memory; after the last block O / l to the output.
// P has buffers of its own, so the next block's scores are issued as soon as every
// row has read this block's, and run under its softmax; P V follows when P is
// there.  At 256 (blocks of 128 keys) O, the scores and two P buffers fill tensor
// memory; at 128 (blocks of 64) two pairs fit an SM pair, and one's MMAs run under
// the other's softmax and output.
//
// attn_packed_64_kernel (head_dim 64): one CTA takes two query tiles, each with its
// own softmax warps; while one tile is in its softmax the other's products run.  P
// takes the place of the scores it was made from: MMAs execute in the order of
// their issue, so the next scores may overwrite it by an MMA issued after the one
// that reads it.
//
// Both kernels stay over the plan: a CTA or pair takes one (tile pair, kv head) after
// another, its next K, V and Q on their way while the last output is written.
//
// Work per 128 x 128 block and head dim HD: 2 * 128 * 128 * HD multiply-adds = 8 HD
// cycles at 4096 per cycle and SM, and 128 * 128 exponentials = 1024 cycles at 16:
// tensor-bound at 256, even at 128, bound by the exponentials at 64.  Measured (in graphs
// of such calls where nothing else is said):
//   256  one prompt of 15001 tokens, 8 heads over one: 2570 cycles per block of 128
//        keys (2048 of MMA), 720 to 728 us = 1.27 to 1.28 PFLOP/s (0.77 of the cuBLAS rate,
//        0.92 of the sustained one), when the power limit takes the clock to 1.6 GHz and
//        below; 687 us in calls 30 ms apart, some 20 of them the launch.
//   128  8 prompts, 8003 tokens, 32 heads over 8: 1710 cycles per block of 64 keys with
//        two CTAs on an SM (512 each of MMA, 512 each of exponentials): 860 in the
//        exponentials, 300 for the scores, 150 for the maximum, 100 each for
//        reading, for handing the scores back and for P.  105 us = 820 TFLOP/s (122 us in
//        a row of calls from the host); bound by that chain, with the tensor pipe and the special-function unit 43 %
//        busy each.  Two threads per row (half the chain, one exchange of the
//        maximum) took an eighth longer, a third CTA does not fit tensor memory.
//    64  one prompt of 8000 tokens, 16 heads: 218 us in f16, 216 in bf16 = 600 TFLOP/s
//        (110 us of exponentials, 79 of MMA at the cuBLAS rate); 8 prompts, 8003 tokens,
//        16 heads over 4: 51.5 us.
// With a window of 512, 4 prompts of 2000 tokens: 50 us (8 heads of 256 over one), 94 (32 of
// 128 over 8); 8 times 128 tokens behind a cached prefix to 4096 (32 of 128 over 8): 79 us.
//
// S, O, m and l are f32; p is rounded to the input type for the second product
// (its relative error is that of the output's own rounding; f16 weights are lifted, see
// kLift).  Every wait is bounded (2 s): a stuck pipeline records SB_ERR_TIMEOUT and unwinds.
#include <cudaTypedefs.h>

#include <algorithm>
#include <vector>

#include "paged.cuh"
#include "tmap.cuh"

namespace {

constexpr int QR = 128;  // query rows per tile
constexpr float kLog2e = 1.4426950408889634f;
using sbp::kRise;

// head_dim 64, one CTA
struct Cfg64 {
  static constexpr int HD = 64, NQ = 2, KB = 128;  // KB: keys per block
  static constexpr int THREADS = 128 + 128 * NQ;
  static constexpr int Q_BYTES = QR * HD * 2;
  static constexpr int SLOT = KB * HD * 2;  // a block of K or of V
  static constexpr int NSLOT = 8;
  static constexpr int OFF_SLOT = NQ * Q_BYTES;
  static constexpr int OFF_BAR = OFF_SLOT + NSLOT * SLOT;
  static constexpr int SMEM = OFF_BAR + 256 + 1024;  // + alignment slack
  static constexpr uint32_t TM_S = NQ * HD;          // S buffers (and P) after the O accumulators
};

// head_dim 128 and 256, a CTA pair
template <int HD>
struct PairCfg {
  static constexpr int CTAS = HD == 256 ? 1 : 2;   // per SM
  static constexpr int KB = HD == 256 ? 128 : 64;  // keys per block
  static constexpr int Q_BYTES = QR * HD * 2;
  static constexpr int SLOT = KB / 2 * HD * 2;    // this CTA's half of a block of K or of V
  static constexpr int NSLOT = HD == 256 ? 5 : 8;
  static constexpr int OFF_BAR = Q_BYTES + NSLOT * SLOT;
  static constexpr int SMEM = OFF_BAR + 256 + 1024;
  static constexpr uint32_t TM_S = HD, TM_P = HD + KB, TM_COLS = HD + 2 * KB;  // scores, two P buffers of KB / 2
};

struct Bars {
  uint64_t q_full, q_free;
  uint64_t full[8], empty[8];
  uint64_t s_full[2], s_free, p_full[2], pv_done[2];
  uint64_t dirty, clean, drain;
  uint32_t tmem_slot;
  int abort;
};
static_assert(sizeof(Bars) <= 256, "barrier block");

struct Tile {  // two query tiles, as sb_attn_packed_plan lays them out
  int q0, n_tok, k0, k_len, pos0, pad[3];
};

struct PackedParams {
  void* out;
  int64_t out_token, out_head;  // strides, elements
  const Tile* tiles;
  int* err;
  int t_q, t_k, n_tiles, nkv, group, tpt, window;
  float scale2;  // scale * log2(e)
};

// 32 lanes x 16 consecutive columns (thread t -> lane base + t).
__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void tma_load_3d(const CUtensorMap* map, uint64_t* bar, void* dst, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(sbd::smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(sbd::smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

__device__ __forceinline__ bool drain_wait(uint64_t* bar, uint32_t parity) {
  const uint64_t t0 = sbd::global_ns();
  while (!sbd::mbar_try_wait(bar, parity)) {
    if (sbd::global_ns() - t0 > sbd::kWaitLimitNs) return false;
  }
  return true;
}

// Both operands f16, or both bf16.
template <typename T>
constexpr uint32_t idesc(int m, int n, int b_mn) {
  const uint32_t bf = std::is_same<T, __half>::value ? 0u : 1u;
  return sbd::umma_idesc_f16(m, n, 0, b_mn) | bf << 7 | bf << 10;
}

// The pair's forms: completion counted on a barrier of the pair's even CTA (`bar`: a shared::cluster address), and
// both operands from shared memory (A: this CTA's 128 rows in each CTA; B: N / 2 rows in each).
__device__ __forceinline__ void tma_load_3d_pair(const CUtensorMap* map, uint32_t bar, void* dst, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(sbd::smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void umma_f16_ss_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                                 uint32_t accumulate) {
  const uint32_t z = 0;  // no output lanes disabled
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8, %9, %10, %11, %12}, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(z), "r"(z), "r"(z), "r"(z), "r"(z), "r"(z), "r"(z), "r"(z)
      : "memory");
}

// ---- pairs of f32 in one 64-bit register (the packed FMA-pipe forms)
__device__ __forceinline__ uint64_t pack_f2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack_f2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma_f2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_f2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// n low bits set, none below 0 and all from 32 on
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xFFFFFFFFu : n > 0 ? (1u << n) - 1u : 0u; }

// One query row's part in a block: reads the scores (then `loaded()`), masks them (keys [lo, hi) of the sequence;
// `whole`: all of them), raises the running maximum and rescales O where a score asks for it, once `pv_before()`
// says that the P V of the block before is complete, writes P to `tp` and adds to the sum.  Warp-collective; false when a wait failed.
template <typename T, int HD, int KB, typename Loaded, typename Before>
__device__ __forceinline__ bool softmax_block(uint32_t ts, uint32_t tp, uint32_t to, int kb, int lo, int hi, bool whole,
                                              float scale2, float& m, float& l, Loaded loaded, Before pv_before) {
  constexpr int CH = KB / 32;
  uint32_t sv[CH][32];
#pragma unroll
  for (int c = 0; c < CH; ++c) sbd::tmem_ld_32x32b_x32(ts + 32 * c, sv[c]);
  sbd::tmem_wait_ld();
  loaded();
  if (!whole) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const uint32_t seen = low_bits(hi - kb - 32 * c) & ~low_bits(lo - kb - 32 * c);
#pragma unroll
      for (int e = 0; e < 32; ++e) sv[c][e] = seen & (1u << e) ? sv[c][e] : 0xFF800000u;  // -inf
    }
  }
  float mx[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    mx[c] = __uint_as_float(sv[0][c]);
#pragma unroll
    for (int e = 4 + c; e < KB; e += 4) mx[c] = fmaxf(mx[c], __uint_as_float(sv[e >> 5][e & 31]));
  }
  const float mx2 = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale2;
  const bool start = m == -INFINITY;  // O is still zero in this row
  const bool rise = !start && mx2 > m + kRise;
  if (__any_sync(0xFFFFFFFFu, rise)) {
    // O += P V of the block before has to be complete before it is scaled
    if (!__all_sync(0xFFFFFFFFu, pv_before())) return false;
    sbd::tc_fence_after();
    const float alpha = rise ? ex2(m - mx2) : 1.f;
#pragma unroll 1
    for (int c = 0; c < HD / 16; ++c) {
      uint32_t ov[16];
      tmem_ld_x16(to + 16 * c, ov);
      sbd::tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 16; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
      sbd::tmem_st_32x32b_x16(to + 16 * c, ov);
    }
    sbd::tmem_wait_st();
    l *= alpha;
  }
  if (start || rise) m = mx2;
  const float mu = (m == -INFINITY ? 0.f : m) - sbp::kLift<T>;
  const uint64_t scale_2 = pack_f2(scale2, scale2), shift_2 = pack_f2(-mu, -mu);
  uint64_t sum[2] = {0, 0};  // pairs of zeros
  // All exponentials in the special-function unit, 16 a cycle and SM.  Some of them by a polynomial on the FMA pipe cost
  // more issue slots than they save even at head_dim 64, and need a way of their own for scores that are not finite: one
  // prompt of 8000 tokens and 16 heads takes 221 us with none, 228 with 3 of 16, 237 with 5 and 247 with 9.
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    uint32_t pk[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float2 p = unpack_f2(fma_f2(pack_f2(__uint_as_float(sv[c][2 * e]), __uint_as_float(sv[c][2 * e + 1])), scale_2, shift_2));
      p = make_float2(ex2(p.x), ex2(p.y));
      sum[e & 1] = add_f2(sum[e & 1], pack_f2(p.x, p.y));
      pk[e] = sbp::pack2<T>(p.x, p.y);
    }
    sbd::tmem_st_32x32b_x16(tp + 16 * c, pk);
  }
  const float2 s0 = unpack_f2(sum[0]), s1 = unpack_f2(sum[1]);
  l += (s0.x + s0.y) + (s1.x + s1.y);
  sbd::tmem_wait_st();
  sbd::tc_fence_before();
  return true;
}

// A warp's 32 finished rows: O / l to memory (zeros where a row saw no key), `dst` and `store` each lane's own row's.
// Four lanes exchange the 64 bytes that each has of its row at a time, so that a store instruction writes 64 bytes of
// 8 rows in place of 16 bytes of 32 (a lane's own row straight from registers).
template <typename T, int HD>
__device__ __forceinline__ void store_rows(uint32_t to, float l, T* dst, bool store) {
  const int lane = threadIdx.x & 31;
  const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
  const unsigned stored = __ballot_sync(0xFFFFFFFFu, store) >> (lane & 28);
  unsigned long long row[4];
#pragma unroll
  for (int r = 0; r < 4; ++r)
    row[r] = __shfl_sync(0xFFFFFFFFu, reinterpret_cast<unsigned long long>(dst), (lane & 28) + r) + (lane & 3) * 16;
#pragma unroll 2
  for (int c = 0; c < HD / 32; ++c) {
    uint32_t ov[32], w[4][4];
    sbd::tmem_ld_32x32b_x32(to + 32 * c, ov);
    sbd::tmem_wait_ld();
#pragma unroll
    for (int e = 0; e < 32; e += 2)
      w[e / 8][e / 2 % 4] = l == 0.f ? 0u : sbp::pack2<T>(__uint_as_float(ov[e]) * inv, __uint_as_float(ov[e + 1]) * inv);
    // w[i]: chunk i of this lane's row -> chunk (lane & 3) of the group's row i
#pragma unroll
    for (int b = 1; b < 4; b *= 2)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i & b) continue;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t got = __shfl_xor_sync(0xFFFFFFFFu, lane & b ? w[i][q] : w[i + b][q], b);
          if (lane & b) w[i][q] = got;
          else w[i + b][q] = got;
        }
      }
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (stored >> r & 1) *reinterpret_cast<uint4*>(row[r] + c * 64) = make_uint4(w[r][0], w[r][1], w[r][2], w[r][3]);
  }
}

// Zeroes rows [from, KB) of a V block of `boxes` boxes [KB rows x 128 bytes]: whole rows, the swizzle only permutes
// inside them.  64 threads.
template <int KB>
__device__ __forceinline__ void zero_rows(uint8_t* vs, int boxes, int from, int thread) {
  for (int b = 0; b < boxes; ++b)
    for (int x = from * 8 + thread; x < KB * 8; x += 64) *reinterpret_cast<uint4*>(vs + b * (KB * 128) + x * 16) = make_uint4(0, 0, 0, 0);
  sbd::fence_proxy_async_smem();
  __syncwarp();
}

// A query row as its softmax thread sees it.
struct Row {
  int tok, head;           // of its tile and of the group
  int lo, hi;              // keys [lo, hi) of the sequence
  int all_lo, all_hi;      // keys that every row of the tile sees
  bool ok;
};
__device__ __forceinline__ Row row_of(const PackedParams& p, const Tile& tl, int i, int row, int k_len) {
  Row r;
  r.tok = row / p.group, r.head = row - r.tok * p.group;
  const int n_tok = min(p.tpt, tl.n_tok - i * p.tpt), pos0 = tl.pos0 + i * p.tpt, pos = pos0 + r.tok;
  r.ok = r.tok < n_tok;
  r.hi = r.ok ? min(pos + 1, k_len) : 0;
  r.lo = p.window > 0 ? pos + 1 - p.window : 0;
  r.all_hi = min(pos0 + 1, k_len);
  r.all_lo = p.window > 0 ? pos0 + n_tok - p.window : 0;
  return r;
}

// What a CTA or a pair does at a time: a plan's tile and a kv head.  It stays and takes one item after another, there
// and back over the plan (`units` of them do): the tiles come in falling order of their keys, so the sums are about the
// same.  Each role walks the items by itself, so the loads and scores of one run ahead into the softmax and output of
// the one before; the rings and the barriers' phases carry on.  Against a CTA or pair per item 8 packed prompts of
// 32 x 128 heads, 8003 tokens, take 15 % less time, of 16 x 64 heads 11 %.
struct Item {
  Tile tl;
  int kv;
};
__device__ __forceinline__ bool plan_item(const PackedParams& p, int n, int units, int unit, Item& it) {
  const int64_t i = static_cast<int64_t>(n) * units + (n & 1 ? units - 1 - unit : unit);
  if (i >= static_cast<int64_t>(p.n_tiles) * p.nkv) return false;
  it.kv = static_cast<int>(i) % p.nkv;
  it.tl = p.tiles[i / p.nkv];
  return true;
}

// Key blocks [j0, j0 + of[i]) of an item's two tiles, nb of them in all; `unclean`: the one that holds the sequence's
// end inside it, -1 if none does.
struct Blocks {
  int k_len, j0, of[2], nb, unclean;
};
template <int KB>
__device__ __forceinline__ Blocks blocks_of(const PackedParams& p, const Tile& tl) {
  Blocks b;
  b.k_len = min(tl.k_len, p.t_k);
  b.j0 = p.window > 0 ? max(0, tl.pos0 + 1 - p.window) / KB : 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int n = min(p.tpt, tl.n_tok - i * p.tpt);
    const int last = min(tl.pos0 + i * p.tpt + n - 1, b.k_len - 1);  // the tile's furthest key
    b.of[i] = n > 0 ? max(0, (last >= 0 ? last / KB + 1 : 0) - b.j0) : 0;
  }
  b.nb = max(b.of[0], b.of[1]);
  b.unclean = b.k_len % KB ? b.k_len / KB - b.j0 : -1;
  if (b.unclean >= b.nb) b.unclean = -1;
  return b;
}

template <typename T, int HD>
__global__ void __launch_bounds__(256, PairCfg<HD>::CTAS)
    attn_packed_pair_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                            const __grid_constant__ CUtensorMap tmV, const PackedParams p) {
  using C = PairCfg<HD>;
  constexpr int KB = C::KB, NSLOT = C::NSLOT;
  constexpr uint16_t kBoth = 3;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Bars* bars = reinterpret_cast<Bars*>(smem + C::OFF_BAR);
  volatile int* abort = &bars->abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(sbd::cluster_ctarank());
  const bool lead = rank == 0;
  sbd::griddep_launch_dependents();

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      sbd::mbar_init(&bars->p_full[i], 8);
      sbd::mbar_init(&bars->pv_done[i], 1);
    }
    for (int i = 0; i < NSLOT; ++i) {
      sbd::mbar_init(&bars->full[i], 1);
      sbd::mbar_init(&bars->empty[i], 1);
    }
    sbd::mbar_init(&bars->q_full, 1);
    sbd::mbar_init(&bars->q_free, 1);
    sbd::mbar_init(&bars->s_full[0], 1);
    sbd::mbar_init(&bars->s_free, 8);
    sbd::mbar_init(&bars->dirty, 1);
    sbd::mbar_init(&bars->clean, 4);
    sbd::mbar_init(&bars->drain, 1);
    bars->abort = 0;
    sbd::fence_mbar_init();
    sbd::fence_proxy_async_smem();
    sbd::prefetch_tmap(&tmQ);
    sbd::prefetch_tmap(&tmK);
    sbd::prefetch_tmap(&tmV);
  }
  if (warp == 1) {
    sbd::tmem_alloc_pair(&bars->tmem_slot, C::TM_COLS);
    sbd::tmem_relinquish_pair();
  }
  sbd::griddep_wait();
  sbd::tc_fence_before();
  sbd::cluster_sync_all();  // both CTAs' barriers exist
  sbd::tc_fence_after();
  const uint32_t tmem = bars->tmem_slot;
  // the pair's items, one after another
  auto item_at = [&](int n, Item& it) { return plan_item(p, n, gridDim.x >> 1, blockIdx.x >> 1, it); };

  if (warp < 4) {
    if (warp == 0) {
      // ------------------------------------------------------------ TMA producer
      if (lane == 0) {
        const int q_bytes = p.tpt * p.group * HD * 2;  // a box of tpt tokens x group heads; tokens past the tensor read as zero
        const uint32_t q_bar = sbd::mapa_shared(sbd::smem_u32(&bars->q_full), 0);
        int it = 0, nq = 0;
        bool ok = true;
        Item w;
        for (int n = 0; ok && item_at(n, w); ++n) {
          const Blocks blk = blocks_of<KB>(p, w.tl);
          if (blk.nb == 0) continue;
          auto load = [&](bool is_v, int j) {  // this CTA's half of block j of K or V into the next slot
            const int st = it % NSLOT;
            ok = ok && sbd::mbar_wait(&bars->empty[st], ((it / NSLOT) & 1) ^ 1, abort, p.err);
            if (!ok) return;
            uint8_t* dst = smem + C::Q_BYTES + st * C::SLOT;
            if (lead) sbd::mbar_arrive_expect_tx(&bars->full[st], 2 * C::SLOT);
            const uint32_t bar = sbd::mapa_shared(sbd::smem_u32(&bars->full[st]), 0);
            if (is_v) {  // KB keys, dims rank * HD / 2 ...
              for (int b = 0; b < HD / 128; ++b)
                tma_load_3d_pair(&tmV, bar, dst + b * (KB * 128), rank * (HD / 2) + 64 * b, w.kv, w.tl.k0 + j * KB);
            } else {  // keys rank * KB / 2 ..., all dims
              for (int b = 0; b < HD / 64; ++b)
                tma_load_3d_pair(&tmK, bar, dst + b * (KB / 2 * 128), 64 * b, w.kv, w.tl.k0 + j * KB + rank * (KB / 2));
            }
            ++it;
          };
          for (int j = 0; j <= blk.nb && ok; ++j) {
            if (j < blk.nb) load(false, blk.j0 + j);
            if (j == 0) {  // Q, once the scores of the tile before are done with it
              ok = ok && sbd::mbar_wait(&bars->q_free, (nq & 1) ^ 1, abort, p.err);
              if (!ok) break;
              if (lead) sbd::mbar_arrive_expect_tx(&bars->q_full, 2 * q_bytes);
              for (int b = 0; b < HD / 64; ++b)
                tma_load_3d_pair(&tmQ, q_bar, smem + b * (QR * 128), 64 * b, w.kv * p.group, w.tl.q0 + rank * p.tpt);
              ++nq;
            } else {
              load(true, blk.j0 + j - 1);  // the next block's scores come before this block's P V
            }
          }
        }
        if (*abort && lead) {  // copies in flight land before shared memory is released (the even CTA counts both CTAs')
          if (nq > 0) drain_wait(&bars->q_full, (nq - 1) & 1);
          for (int i = max(0, it - NSLOT); i < it; ++i) drain_wait(&bars->full[i % NSLOT], (i / NSLOT) & 1);
        }
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------ MMA issuer (even CTA)
      if (lane == 0 && lead) {
        constexpr uint32_t idesc_s = idesc<T>(2 * QR, KB, 0), idesc_o = idesc<T>(2 * QR, HD, 1);
        const uint64_t qd = sbd::umma_desc(sbd::smem_u32(smem), 16, 1024, sbd::kLayoutSwizzle128B);
        const uint64_t kd = sbd::umma_desc(sbd::smem_u32(smem + C::Q_BYTES), 16, 1024, sbd::kLayoutSwizzle128B);
        const uint64_t vd = sbd::umma_desc(sbd::smem_u32(smem + C::Q_BYTES), KB * 128, 1024, sbd::kLayoutSwizzle128B);
        int it = 0, nq = 0, g = 0;  // ring items, tiles with keys and blocks so far
        bool ok = true;
        auto slot_wait = [&](int i) { ok = ok && sbd::mbar_wait(&bars->full[i % NSLOT], (i / NSLOT) & 1, abort, p.err); };
        auto scores = [&](bool last) {  // S = Q K_j^T, once every row has read the scores of the block before
          ok = ok && sbd::mbar_wait(&bars->s_free, (g & 1) ^ 1, abort, p.err);
          slot_wait(it);
          if (!ok) return;
          sbd::tc_fence_after();
          const uint32_t d = tmem + C::TM_S;
          const uint64_t k = kd + static_cast<uint64_t>((it % NSLOT) * (C::SLOT >> 4));
  #pragma unroll
          for (int s = 0; s < HD / 16; ++s)
            umma_f16_ss_pair(d, qd + (s >> 2) * (QR * 128 >> 4) + (s & 3) * 2, k + (s >> 2) * (KB / 2 * 128 >> 4) + (s & 3) * 2,
                             idesc_s, s > 0 ? 1u : 0u);
          sbd::umma_commit_pair(&bars->empty[it % NSLOT], kBoth);
          if (last) sbd::umma_commit_pair(&bars->q_free, kBoth);
          sbd::umma_commit_pair(&bars->s_full[0], kBoth);
          ++it, ++g;
        };
        Item w;
        for (int n = 0; ok && item_at(n, w); ++n) {
          const Blocks blk = blocks_of<KB>(p, w.tl);
          if (blk.nb == 0) continue;
          ok = sbd::mbar_wait(&bars->q_full, nq & 1, abort, p.err);
          scores(blk.nb == 1);
          for (int j = 0; j < blk.nb && ok; ++j) {
            if (j + 1 < blk.nb) scores(j + 2 == blk.nb);
            slot_wait(it);
            if (ok && j == (blk.unclean >= 0 ? blk.unclean : blk.nb - 1)) {
              ok = sbd::mbar_wait_cluster(&bars->clean, (nq & 1) ^ 1, abort, p.err);  // the cleaners' answer for the tile before
              sbd::mbar_arrive(&bars->dirty);
              sbd::mbar_arrive_remote(sbd::mapa_shared(sbd::smem_u32(&bars->dirty), 1));
              if (blk.unclean >= 0)  // shared memory that the other CTA wrote
                ok = ok && sbd::mbar_wait_cluster(&bars->clean, nq & 1, abort, p.err);
            }
            const int at = j + 1 < blk.nb ? g - 2 : g - 1, buf = at & 1;  // this block's number
            ok = ok && sbd::mbar_wait(&bars->p_full[buf], (at >> 1) & 1, abort, p.err);
            if (!ok) break;
            sbd::tc_fence_after();
            // O += P V_j.  The first of a tile overwrites the last tile's O: whoever wrote P had read it.
            const uint64_t v = vd + static_cast<uint64_t>((it % NSLOT) * (C::SLOT >> 4));
  #pragma unroll
            for (int s = 0; s < KB / 16; ++s)
              sbd::umma_f16_ts_pair(tmem, tmem + C::TM_P + buf * (KB / 2) + s * 8, v + s * (2048 >> 4), idesc_o, j > 0 || s > 0 ? 1u : 0u);
            sbd::umma_commit_pair(&bars->empty[it % NSLOT], kBoth);
            sbd::umma_commit_pair(&bars->pv_done[buf], kBoth);
            ++it;
          }
          ++nq;
        }
        // every MMA issued has finished before tensor and shared memory are released
        sbd::umma_commit_pair(&bars->drain, kBoth);
        drain_wait(&bars->drain, 0);
      }
    } else {
      // ------------------------------------------------------------ V rows past the sequence's end
      // asked once per tile, also where there is nothing to do: no wait here lasts longer than a tile
      int it = 0, nq = 0;
      Item w;
      for (int n = 0; item_at(n, w); ++n) {
        const Blocks blk = blocks_of<KB>(p, w.tl);
        if (blk.nb == 0) continue;
        if (!__all_sync(0xFFFFFFFFu, sbd::mbar_wait(&bars->dirty, nq & 1, abort, p.err))) break;
        if (blk.unclean >= 0) {
          const int item = it + min(blk.unclean + 2, blk.nb) + blk.unclean;  // in the producer's order
          zero_rows<KB>(smem + C::Q_BYTES + item % NSLOT * C::SLOT, HD / 128, blk.k_len % KB, threadIdx.x - 64);
        }
        if (lane == 0) {
          if (lead) sbd::mbar_arrive(&bars->clean);
          else sbd::mbar_arrive_remote(sbd::mapa_shared(sbd::smem_u32(&bars->clean), 0));
        }
        it += 2 * blk.nb;
        ++nq;
      }
    }
  } else {
    // ------------------------------------------------------------ softmax and output
    // P V of block j completes in the phases of a barrier per P buffer: the scores of block j + 1 do not wait for P V
    // of block j, and one barrier's phases could be mistaken two blocks apart.  They do follow P V of block j - 1
    // in the order of issue, and a commit counts every MMA before it: scores of block j in place say that P V of block
    // j - 2 is done, so its P buffer is free, and that no wait on pv_done is more than a phase behind.
    const int quad = warp & 3;
    const uint32_t tm = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const uint32_t lead_bar = sbd::mapa_shared(sbd::smem_u32(bars), 0);
    // a warp's arrival on a barrier of the even CTA
    auto arrive = [&](uint64_t* bar) {
      __syncwarp();
      if (lane == 0) {
        if (lead) sbd::mbar_arrive(bar);
        else sbd::mbar_arrive_remote_cta(lead_bar + static_cast<uint32_t>(reinterpret_cast<uint8_t*>(bar) - reinterpret_cast<uint8_t*>(bars)));
      }
    };
    auto pv_complete = [&](int j) { return sbd::mbar_wait(&bars->pv_done[j & 1], (j >> 1) & 1, abort, p.err); };
    int g = 0;  // blocks so far
    bool ok = true;
    Item w;
    bool more = item_at(0, w);
    for (int n = 1; ok && more; ++n) {
      const Blocks blk = blocks_of<KB>(p, w.tl);
      const Row r = row_of(p, w.tl, rank, quad * 32 + lane, blk.k_len);
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < blk.nb; ++j, ++g) {
        const int kb = (blk.j0 + j) * KB;
        ok = __all_sync(0xFFFFFFFFu, sbd::mbar_wait(&bars->s_full[0], g & 1, abort, p.err));
        if (!ok) break;
        sbd::tc_fence_after();
        ok = softmax_block<T, HD, KB>(
            tm + C::TM_S, tm + C::TM_P + (g & 1) * (KB / 2), tm, kb, r.lo, r.hi, kb + KB <= r.all_hi && kb >= r.all_lo, p.scale2, m, l,
            [&] {
              sbd::tc_fence_before();
              arrive(&bars->s_free);
            },
            [&] { return pv_complete(g - 1); });
        if (!ok) break;
        arrive(&bars->p_full[g & 1]);
      }
      const int64_t token = static_cast<int64_t>(w.tl.q0) + rank * p.tpt + r.tok;
      T* dst = static_cast<T*>(p.out) + token * p.out_token + static_cast<int64_t>(w.kv * p.group + r.head) * p.out_head;
      more = item_at(n, w);  // on its way while P V completes
      if (ok && blk.nb > 0) ok = __all_sync(0xFFFFFFFFu, pv_complete(g - 1));
      if (!ok) break;
      sbd::tc_fence_after();
      store_rows<T, HD>(tm, l, dst, r.ok && token >= 0 && token < p.t_q);
    }
  }

  // both CTAs are done with each other's barriers and with tensor memory (the MMAs have completed)
  sbd::tc_fence_before();
  sbd::cluster_sync_all();
  if (warp == 1) {
    sbd::tc_fence_after();
    sbd::tmem_dealloc_pair(tmem, C::TM_COLS);
  }
}

template <typename T>
__global__ void __launch_bounds__(Cfg64::THREADS, 1)
    attn_packed_64_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                          const __grid_constant__ CUtensorMap tmV, const PackedParams p) {
  using C = Cfg64;
  constexpr int NQ = C::NQ, NSLOT = C::NSLOT, HD = C::HD, KB = C::KB;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Bars* bars = reinterpret_cast<Bars*>(smem + C::OFF_BAR);
  volatile int* abort = &bars->abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  sbd::griddep_launch_dependents();

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      sbd::mbar_init(&bars->s_full[i], 1);
      sbd::mbar_init(&bars->p_full[i], 4);
      sbd::mbar_init(&bars->pv_done[i], 1);
    }
    for (int i = 0; i < NSLOT; ++i) {
      sbd::mbar_init(&bars->full[i], 1);
      sbd::mbar_init(&bars->empty[i], 1);
    }
    sbd::mbar_init(&bars->q_full, 1);
    sbd::mbar_init(&bars->q_free, 1);
    sbd::mbar_init(&bars->dirty, 1);
    sbd::mbar_init(&bars->clean, 2);
    sbd::mbar_init(&bars->drain, 1);
    bars->abort = 0;
    sbd::fence_mbar_init();
    sbd::fence_proxy_async_smem();
    sbd::prefetch_tmap(&tmQ);
    sbd::prefetch_tmap(&tmK);
    sbd::prefetch_tmap(&tmV);
  }
  if (warp == 1) {
    sbd::tmem_alloc(&bars->tmem_slot, 512);
    sbd::tmem_relinquish();
  }
  sbd::griddep_wait();
  sbd::tc_fence_before();
  __syncthreads();
  sbd::tc_fence_after();
  const uint32_t tmem = bars->tmem_slot;
  // the CTA's items, one after another; the ring holds K_0, V_0, K_1, V_1, ... (one slot each)
  auto item_at = [&](int n, Item& it) { return plan_item(p, n, gridDim.x, blockIdx.x, it); };

  // 168 registers a thread at launch, then 72 in the first warpgroup and 216 in the softmax's two
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 0) {
      // ------------------------------------------------------------ TMA producer
      if (lane == 0) {
        int it = 0, nq = 0;
        bool ok = true;
        Item w;
        for (int n = 0; ok && item_at(n, w); ++n) {
          const Blocks blk = blocks_of<KB>(p, w.tl);
          for (int x = 0; x < 2 * blk.nb; ++x) {
            const int st = it % NSLOT;
            ok = sbd::mbar_wait(&bars->empty[st], ((it / NSLOT) & 1) ^ 1, abort, p.err);
            if (!ok) break;
            sbd::mbar_arrive_expect_tx(&bars->full[st], C::SLOT);
            tma_load_3d(x & 1 ? &tmV : &tmK, &bars->full[st], smem + C::OFF_SLOT + st * C::SLOT, 0, w.kv, w.tl.k0 + (blk.j0 + x / 2) * KB);
            ++it;
            if (x > 0) continue;  // Q, once the scores of the item before are done with it
            ok = sbd::mbar_wait(&bars->q_free, (nq & 1) ^ 1, abort, p.err);
            if (!ok) break;
            sbd::mbar_arrive_expect_tx(&bars->q_full, NQ * p.tpt * p.group * HD * 2);
            for (int i = 0; i < NQ; ++i)
              tma_load_3d(&tmQ, &bars->q_full, smem + i * C::Q_BYTES, 0, w.kv * p.group, w.tl.q0 + i * p.tpt);
            ++nq;
          }
        }
        if (*abort) {  // copies in flight land before this CTA's shared memory is released
          if (nq > 0) drain_wait(&bars->q_full, (nq - 1) & 1);
          for (int i = max(0, it - NSLOT); i < it; ++i) drain_wait(&bars->full[i % NSLOT], (i / NSLOT) & 1);
        }
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------ MMA issuer
      if (lane == 0) {
        constexpr uint32_t idesc_s = idesc<T>(QR, KB, 0), idesc_o = idesc<T>(QR, HD, 1);
        bool ok = true;
        auto slot_wait = [&](int i) {
          ok = ok && sbd::mbar_wait(&bars->full[i % NSLOT], (i / NSLOT) & 1, abort, p.err);
          return sbd::smem_u32(smem + C::OFF_SLOT + (i % NSLOT) * C::SLOT);
        };
        auto issue_s = [&](int i, uint32_t ks) {  // S_i = Q_i K^T
          const uint32_t qb = sbd::smem_u32(smem + i * C::Q_BYTES);
  #pragma unroll
          for (int s = 0; s < HD / 16; ++s)
            sbd::umma_f16(tmem + C::TM_S + i * KB, sbd::umma_desc(qb + s * 32, 16, 1024, sbd::kLayoutSwizzle128B),
                          sbd::umma_desc(ks + s * 32, 16, 1024, sbd::kLayoutSwizzle128B), idesc_s, s > 0 ? 1u : 0u);
          sbd::umma_commit(&bars->s_full[i]);
        };
        int it = 0, nq = 0, g[NQ] = {0, 0};  // ring items, items with keys, blocks of each tile so far
        Item w;
        for (int n = 0; ok && item_at(n, w); ++n) {
          const Blocks blk = blocks_of<KB>(p, w.tl);
          if (blk.nb == 0) continue;
          ok = sbd::mbar_wait(&bars->q_full, nq & 1, abort, p.err);
          const uint32_t ks = slot_wait(it);
          if (ok) {
            sbd::tc_fence_after();
            for (int i = 0; i < NQ; ++i)
              if (blk.of[i] > 0) issue_s(i, ks);
            sbd::umma_commit(&bars->empty[it % NSLOT]);
            if (blk.nb == 1) sbd::umma_commit(&bars->q_free);
          }
          ++it;
          for (int j = 0; j < blk.nb && ok; ++j) {
            const bool next = j + 1 < blk.nb;
            const uint32_t vs = slot_wait(it);
            if (ok && j == (blk.unclean >= 0 ? blk.unclean : blk.nb - 1)) {
              ok = sbd::mbar_wait(&bars->clean, (nq & 1) ^ 1, abort, p.err);  // the cleaners' answer for the item before
              sbd::mbar_arrive(&bars->dirty);
              if (blk.unclean >= 0) ok = ok && sbd::mbar_wait(&bars->clean, nq & 1, abort, p.err);
            }
            const uint32_t kn = next ? slot_wait(it + 1) : 0;
            for (int i = 0; i < NQ && ok; ++i) {
              if (j >= blk.of[i]) continue;
              ok = sbd::mbar_wait(&bars->p_full[i], g[i] & 1, abort, p.err);
              if (!ok) break;
              ++g[i];
              sbd::tc_fence_after();
              // O_i += P_i V.  The first of an item overwrites the last one's O: whoever wrote P had read it.
  #pragma unroll
              for (int s = 0; s < KB / 16; ++s)
                sbd::umma_f16_ts(tmem + i * HD, tmem + C::TM_S + i * KB + s * 8,
                                 sbd::umma_desc(vs + s * 2048, KB * 128, 1024, sbd::kLayoutSwizzle128B), idesc_o, j > 0 || s > 0 ? 1u : 0u);
              sbd::umma_commit(&bars->pv_done[i]);
              if (j + 1 < blk.of[i]) issue_s(i, kn);
            }
            if (!ok) break;
            sbd::umma_commit(&bars->empty[it % NSLOT]);
            if (next) sbd::umma_commit(&bars->empty[(it + 1) % NSLOT]);
            if (j + 2 == blk.nb) sbd::umma_commit(&bars->q_free);
            it += next ? 2 : 1;
          }
          ++nq;
        }
        // every MMA issued has finished before tensor and shared memory are released
        sbd::umma_commit(&bars->drain);
        drain_wait(&bars->drain, 0);
      }
    } else {
      // ------------------------------------------------------------ V rows past the sequence's end
      // (the issuer, which follows the slots' phases, says when they have landed: once per item, also where there is
      // nothing to do, so that no wait here lasts longer than an item)
      int it = 0, nq = 0;
      Item w;
      for (int n = 0; item_at(n, w); ++n) {
        const Blocks blk = blocks_of<KB>(p, w.tl);
        if (blk.nb == 0) continue;
        if (!__all_sync(0xFFFFFFFFu, sbd::mbar_wait(&bars->dirty, nq & 1, abort, p.err))) break;
        if (blk.unclean >= 0)
          zero_rows<KB>(smem + C::OFF_SLOT + (it + 2 * blk.unclean + 1) % NSLOT * C::SLOT, 1, blk.k_len % KB, threadIdx.x - 64);
        if (lane == 0) sbd::mbar_arrive(&bars->clean);
        it += 2 * blk.nb;
        ++nq;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ------------------------------------------------------------ softmax and output
    const int i = (warp - 4) >> 2, quad = warp & 3;  // tile, lane quadrant
    const uint32_t tm = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    int g = 0;  // this tile's blocks so far
    bool ok = true;
    Item w;
    bool more = item_at(0, w);
    for (int n = 1; ok && more; ++n) {
      const Blocks blk = blocks_of<KB>(p, w.tl);
      const Row r = row_of(p, w.tl, i, quad * 32 + lane, blk.k_len);
      const int nb = blk.of[i];
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < nb; ++j, ++g) {
        const int kb = (blk.j0 + j) * KB;
        ok = __all_sync(0xFFFFFFFFu, sbd::mbar_wait(&bars->s_full[i], g & 1, abort, p.err));
        if (!ok) break;
        sbd::tc_fence_after();
        const uint32_t ts = tm + C::TM_S + i * KB;  // P takes the place of the scores it was made from
        ok = softmax_block<T, HD, KB>(
            ts, ts, tm + i * HD, kb, r.lo, r.hi, kb + KB <= r.all_hi && kb >= r.all_lo, p.scale2, m, l, [] {}, [] { return true; });
        if (!ok) break;
        __syncwarp();
        if (lane == 0) sbd::mbar_arrive(&bars->p_full[i]);
      }
      const int64_t token = static_cast<int64_t>(w.tl.q0) + i * p.tpt + r.tok;
      T* dst = static_cast<T*>(p.out) + token * p.out_token + static_cast<int64_t>(w.kv * p.group + r.head) * p.out_head;
      more = item_at(n, w);  // on its way while P V completes
      if (ok && nb > 0) ok = __all_sync(0xFFFFFFFFu, sbd::mbar_wait(&bars->pv_done[i], (g - 1) & 1, abort, p.err));
      if (!ok) break;
      sbd::tc_fence_after();
      store_rows<T, HD>(tm + i * HD, l, dst, r.ok && token >= 0 && token < p.t_q);
    }
  }

  sbd::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    sbd::tc_fence_after();
    sbd::tmem_dealloc(tmem, 512);
  }
}

// [tokens][heads][HD] of 16-bit elements, copied in boxes of 64 x box_heads x box_tokens.
int make_map3(CUtensorMap* map, bool bf16, const void* base, int hd, int heads, int tokens, int64_t head_stride,
              int64_t token_stride, int box_heads, int box_tokens) {
  auto fn = sb::encode_fn();
  if (!fn) return sb::fail(SB_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(hd), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(tokens)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(head_stride) * 2, static_cast<cuuint64_t>(token_stride) * 2};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_tokens)};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base),
                  dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return sb::fail(SB_ERR_ARG, "cuTensorMapEncodeTiled failed (CUresult %d)", static_cast<int>(r));
  return SB_OK;
}

struct Strides {
  int64_t q_token, q_head, k_token, k_head;
};

template <typename K>
int raise_smem(K kernel, int bytes, bool (&set)[64]) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && set[dev]) return SB_OK;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return sb::cuda_fail(e, "attn_packed smem attribute");
  if (dev >= 0 && dev < 64) set[dev] = true;
  return SB_OK;
}

// K in boxes of k_rows keys, V of v_rows.
template <typename T>
int make_maps(const void* q, const void* k, const void* v, const Strides& st, const PackedParams& p, int hd, int k_rows,
              int v_rows, CUtensorMap (&m)[3]) {
  constexpr bool bf = !std::is_same<T, __half>::value;
  const int t_k = std::max(p.t_k, 1);
  int rc = make_map3(&m[0], bf, q, hd, p.group * p.nkv, p.t_q, st.q_head, st.q_token, p.group, p.tpt);
  if (!rc) rc = make_map3(&m[1], bf, k, hd, p.nkv, t_k, st.k_head, st.k_token, 1, k_rows);
  if (!rc) rc = make_map3(&m[2], bf, v, hd, p.nkv, t_k, st.k_head, st.k_token, 1, v_rows);
  return rc;
}

template <typename T>
int launch_64(const void* q, const void* k, const void* v, const Strides& st, const PackedParams& p, int n_tiles, cudaStream_t stream) {
  static bool set[64] = {};
  CUtensorMap m[3];
  int rc = make_maps<T>(q, k, v, st, p, 64, Cfg64::KB, Cfg64::KB, m);
  if (!rc) rc = raise_smem(attn_packed_64_kernel<T>, Cfg64::SMEM, set);
  if (rc) return rc;
  cudaError_t e = sb::launch_pdl(attn_packed_64_kernel<T>, dim3(std::min(n_tiles * p.nkv, sb::num_sms())), dim3(Cfg64::THREADS), Cfg64::SMEM, stream, m[0], m[1], m[2], p);
  if (e != cudaSuccess) return sb::cuda_fail(e, "attn_packed_64_kernel");
  return sb::launch_status("attn_packed_64_kernel");
}

template <typename T, int HD>
int launch_pair(const void* q, const void* k, const void* v, const Strides& st, const PackedParams& p, int n_tiles, cudaStream_t stream) {
  using C = PairCfg<HD>;
  static bool set[64] = {};
  CUtensorMap m[3];
  int rc = make_maps<T>(q, k, v, st, p, HD, C::KB / 2, C::KB, m);
  if (!rc) rc = raise_smem(attn_packed_pair_kernel<T, HD>, C::SMEM, set);
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * std::min(n_tiles * p.nkv, sb::num_sms() / 2 * C::CTAS));
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaError_t e = cudaLaunchKernelEx(&cfg, attn_packed_pair_kernel<T, HD>, m[0], m[1], m[2], p);
  if (e != cudaSuccess) return sb::cuda_fail(e, "attn_packed_pair_kernel");
  return sb::launch_status("attn_packed_pair_kernel");
}

template <typename T>
int launch_packed_hd(int hd, const void* q, const void* k, const void* v, const Strides& st, const PackedParams& p,
                     int n_tiles, cudaStream_t s) {
  if (hd == 64) return launch_64<T>(q, k, v, st, p, n_tiles, s);
  if (hd == 128) return launch_pair<T, 128>(q, k, v, st, p, n_tiles, s);
  return launch_pair<T, 256>(q, k, v, st, p, n_tiles, s);
}

// Query tokens per tile of the plan: two query tiles, of one CTA or of a pair.
int tokens_per_tile(int group) { return 2 * (QR / group); }

int check_heads(const char* who, int n_heads, int n_kv_heads, int hd) {
  SB_CHECK_ARG(hd == 64 || hd == 128 || hd == 256, "%s: head_dim %d not in {64, 128, 256}", who, hd);
  SB_CHECK_ARG(n_kv_heads >= 1 && n_heads >= 1 && n_heads % n_kv_heads == 0 && n_heads / n_kv_heads <= QR,
               "%s: %d query heads over %d kv heads", who, n_heads, n_kv_heads);
  return SB_OK;
}

}  // namespace

extern "C" int sb_attn_packed_plan(const int32_t* q_lens, const int32_t* kv_lens, int n, int n_heads, int n_kv_heads,
                                   int head_dim, int window, int32_t* tiles, int max_tiles, int* n_tiles) {
  int rc = check_heads("sb_attn_packed_plan", n_heads, n_kv_heads, head_dim);
  if (rc) return rc;
  SB_CHECK_ARG(n >= 0 && window >= 0 && max_tiles >= 0 && n_tiles && (n == 0 || q_lens), "sb_attn_packed_plan: bad arguments");
  const int per = tokens_per_tile(n_heads / n_kv_heads);
  int64_t count = 0, tq = 0, tk = 0;
  for (int i = 0; i < n; ++i) {
    const int kl = kv_lens ? kv_lens[i] : q_lens[i];
    SB_CHECK_ARG(q_lens[i] >= 0 && kl >= 0, "sb_attn_packed_plan: negative length of sequence %d", i);
    count += (q_lens[i] + per - 1) / per;
    tq += q_lens[i];
    tk += kl;
  }
  SB_CHECK_ARG(tq < (1ll << 31) && tk < (1ll << 31) && count * n_kv_heads < (1ll << 30), "sb_attn_packed_plan: too many tokens");
  *n_tiles = static_cast<int>(count);
  if (!tiles) return SB_OK;  // the count alone
  SB_CHECK_ARG(count <= max_tiles, "sb_attn_packed_plan: %lld tiles, room for %d", static_cast<long long>(count), max_tiles);
  Tile* out = reinterpret_cast<Tile*>(tiles);
  int at = 0, q0 = 0, k0 = 0;
  for (int i = 0; i < n; ++i) {
    const int ql = q_lens[i], kl = kv_lens ? kv_lens[i] : ql;
    for (int t = 0; t < ql; t += per) out[at++] = Tile{q0 + t, std::min(per, ql - t), k0, kl, kl - ql + t, {0, 0, 0}};
    q0 += ql;
    k0 += kl;
  }
  // the tiles that see the most keys first: the last CTAs to start are the short ones
  auto keys = [&](const Tile& t) {
    const int hi = std::min(t.pos0 + t.n_tok, t.k_len);
    return hi - (window > 0 ? std::max(0, t.pos0 + 1 - window) : 0);
  };
  std::stable_sort(out, out + at, [&](const Tile& a, const Tile& b) { return keys(a) > keys(b); });
  return SB_OK;
}

extern "C" int sb_attn_prefill_packed(const void* q, int64_t q_token, int64_t q_head, const void* k, const void* v,
                                      int64_t k_token, int64_t k_head, void* out, int64_t out_token, int64_t out_head,
                                      int dtype, int t_q, int t_k, int n_heads, int n_kv_heads, int head_dim,
                                      int window, float scale, const int32_t* tiles, int n_tiles, void* stream) {
  int rc = check_heads("sb_attn_prefill_packed", n_heads, n_kv_heads, head_dim);
  if (rc) return rc;
  SB_CHECK_ARG(dtype == SB_F16 || dtype == SB_BF16, "sb_attn_prefill_packed: q, k, v and out are f16 or bf16");
  SB_CHECK_ARG(t_q >= 0 && t_k >= 0 && window >= 0 && n_tiles >= 0 &&
                   static_cast<int64_t>(n_tiles) * n_kv_heads < (1ll << 30), "sb_attn_prefill_packed: bad sizes");
  SB_CHECK_ARG(scale > 0.f && scale <= 3.0e38f, "sb_attn_prefill_packed: scale must be positive and finite");
  if (t_q == 0 || n_tiles == 0) return SB_OK;
  SB_CHECK_ARG(q && out && tiles && (t_k == 0 || (k && v)), "sb_attn_prefill_packed: null pointer");
  if (!sb::aligned(q, 16) || !sb::aligned(k, 16) || !sb::aligned(v, 16) || !sb::aligned(out, 16) || q_token % 8 ||
      q_head % 8 || k_token % 8 || k_head % 8 || out_token % 8 || out_head % 8 || !sb::aligned(tiles, 4))
    return sb::fail(SB_ERR_ALIGN, "sb_attn_prefill_packed: rows must start on 16-byte boundaries");
  SB_CHECK_ARG(q_token > 0 && q_head > 0 && k_token > 0 && k_head > 0 && out_token > 0 && out_head > 0,
               "sb_attn_prefill_packed: strides must be positive");
  PackedParams p{};
  p.out = out, p.out_token = out_token, p.out_head = out_head, p.tiles = reinterpret_cast<const Tile*>(tiles);
  p.err = sb::device_error_word();
  p.t_q = t_q, p.t_k = t_k, p.n_tiles = n_tiles, p.nkv = n_kv_heads, p.group = n_heads / n_kv_heads, p.tpt = QR / p.group;
  p.window = window, p.scale2 = scale * kLog2e;
  if (t_k == 0) k = v = q;  // nothing is read; the maps need an address
  const Strides st{q_token, q_head, k_token, k_head};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == SB_F16 ? launch_packed_hd<__half>(head_dim, q, k, v, st, p, n_tiles, s)
                         : launch_packed_hd<__nv_bfloat16>(head_dim, q, k, v, st, p, n_tiles, s);
}
