// Causal attention of packed prompts on tcgen05 (sb_attn_prefill_packed):
// sequences of different lengths end to end in one tensor, grouped heads, a
// sliding window, more keys than queries (a cached prefix).
//
// The rows of a query tile are (token, query head of the kv head's group), 128 /
// group tokens of all heads that share K and V, so each K/V block serves the
// whole group.  A CTA owns NQ tiles of 128 rows (two for head_dim 64 and 128,
// one for 256) and walks the key blocks of 128 that its tokens see:
//   warp 0        TMA: the Q tiles once, then K and V through a ring of slots.
//   warp 1        one thread issues tcgen05.mma: S = Q K^T (both operands in
//                 shared memory) and O += P V (P from tensor memory).
//   warps 2, 3    zero the V rows past the sequence's end in its last block: those
//                 rows belong to another sequence, and 0 times a NaN there would
//                 reach this one.
//   warps 4 ...   softmax, a thread per query row of its tile: the row's 128
//                 scores from tensor memory, running maximum m (raised, with O
//                 rescaled, only when a score passes it by 2^8) and sum l,
//                 p = 2^(s - m) in the input type back into the scores' columns.
// While the softmax works on one block the tensor cores run the other tile's
// products (two tiles), or the next block's scores (one tile, two score
// buffers).  The issuing thread's MMAs execute in order, so a score buffer may
// be overwritten by an MMA issued after the one that reads the P in it.
//
// Work per 128 x 128 block and head dim HD: 2 * 128 * 128 * HD multiply-adds = 8 HD
// cycles at 4096 per cycle and SM, and 128 * 128 exponentials = 1024 cycles at 16:
// tensor-bound at 256, even at 128, bound by the exponentials at 64.
//
// S, O, m and l are f32; p is rounded to the input type for the second product
// (its relative error is that of the output's own rounding).  Every wait is
// bounded (2 s): a stuck pipeline records SB_ERR_TIMEOUT and unwinds.
#include <cudaTypedefs.h>

#include <algorithm>
#include <vector>

#include "paged.cuh"
#include "tmap.cuh"

namespace {

constexpr int QR = 128;  // query rows per tile
constexpr int KB = 128;  // keys per block
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRise = 8.f;  // log2 units: p stays below 2^8

template <int HD>
struct Cfg {
  static constexpr int NQ = HD == 256 ? 1 : 2;
  static constexpr int THREADS = 128 + 128 * NQ;
  static constexpr int Q_BYTES = QR * HD * 2;
  static constexpr int SLOT = HD == 64 ? 16384 : 32768;  // a K block, or half of one (256)
  static constexpr int PER = KB * HD * 2 / SLOT;         // slots per K or V block
  static constexpr int NSLOT = HD == 64 ? 8 : 5;
  static constexpr int VK = KB / PER;  // keys of V per slot
  static constexpr int OFF_SLOT = NQ * Q_BYTES;
  static constexpr int OFF_BAR = OFF_SLOT + NSLOT * SLOT;
  static constexpr int SMEM = OFF_BAR + 256 + 1024;  // + alignment slack
  static constexpr uint32_t TM_S = NQ * HD;          // S buffers (and P) after the O accumulators
};

struct Bars {
  uint64_t q_full[2];
  uint64_t full[8], empty[8];
  uint64_t s_full[2], p_full[2], pv_done[2];
  uint64_t dirty, clean, drain;
  uint32_t tmem_slot;
  int abort;
};
static_assert(sizeof(Bars) <= 256, "barrier block");

struct Tile {  // one CTA's queries, as sb_attn_packed_plan lays them out
  int q0, n_tok, k0, k_len, pos0, pad[3];
};

struct PackedParams {
  void* out;
  int64_t out_token, out_head;  // strides, elements
  const Tile* tiles;
  int* err;
  int t_q, t_k, nkv, group, tpt, window;
  float scale2;  // scale * log2(e)
};

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

template <typename T>
constexpr uint32_t idesc(int n, int b_mn) {
  const uint32_t bf = sizeof(T) == 2 && !std::is_same<T, __half>::value ? 1u : 0u;
  return sbd::umma_idesc_f16(QR, n, 0, b_mn) | bf << 7 | bf << 10;
}

template <typename T, int HD>
__global__ void __launch_bounds__(Cfg<HD>::THREADS, 1)
    attn_packed_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                       const __grid_constant__ CUtensorMap tmV, const PackedParams p) {
  using C = Cfg<HD>;
  constexpr int NQ = C::NQ, PER = C::PER, NSLOT = C::NSLOT;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Bars* bars = reinterpret_cast<Bars*>(smem + C::OFF_BAR);
  volatile int* abort = &bars->abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  sbd::griddep_launch_dependents();
  const int kv = blockIdx.x % p.nkv;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      sbd::mbar_init(&bars->q_full[i], 1);
      sbd::mbar_init(&bars->s_full[i], 1);
      sbd::mbar_init(&bars->p_full[i], 4);
      sbd::mbar_init(&bars->pv_done[i], 1);
    }
    for (int i = 0; i < NSLOT; ++i) {
      sbd::mbar_init(&bars->full[i], 1);
      sbd::mbar_init(&bars->empty[i], 1);
    }
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
  const Tile tl = p.tiles[blockIdx.x / p.nkv];
  sbd::tc_fence_before();
  __syncthreads();
  sbd::tc_fence_after();
  const uint32_t tmem = bars->tmem_slot;

  // key blocks [j0, j0 + nb[i]) of tile i; rows see keys (pos - window, pos] of [0, k_len)
  const int k_len = min(tl.k_len, p.t_k);
  int nb[2] = {0, 0}, j0 = 0, nb_all = 0;
  {
    const int first = tl.pos0;
    j0 = p.window > 0 ? max(0, first + 1 - p.window) / KB : 0;
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const int n = min(p.tpt, tl.n_tok - i * p.tpt);
      const int last = min(first + i * p.tpt + n - 1, k_len - 1);  // the tile's furthest key
      nb[i] = n > 0 ? max(0, (last >= 0 ? last / KB + 1 : 0) - j0) : 0;
      nb_all = max(nb_all, nb[i]);
    }
  }
  // the block that holds the sequence's end inside it, if this CTA reads it
  const int j_end = k_len % KB ? k_len / KB : -1;
  const bool cleans = j_end >= j0 && j_end < j0 + nb_all;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0 && nb_all > 0) {
      for (int i = 0; i < NQ; ++i) {
        if (nb[i] == 0) continue;
        // a box of tpt tokens x group heads; tokens past the tensor read as zero
        sbd::mbar_arrive_expect_tx(&bars->q_full[i], p.tpt * p.group * HD * 2);
        for (int b = 0; b < HD / 64; ++b)
          tma_load_3d(&tmQ, &bars->q_full[i], smem + i * C::Q_BYTES + b * (QR * 128), 64 * b, kv * p.group,
                      tl.q0 + i * p.tpt);
      }
      int it = 0;
      bool ok = true;
      auto load = [&](bool is_v, int j, int c) {  // part c of block j of K or V into the next slot
        const int st = it % NSLOT;
        ok = ok && sbd::mbar_wait(&bars->empty[st], ((it / NSLOT) & 1) ^ 1, abort, p.err);
        if (!ok) return;
        uint8_t* dst = smem + C::OFF_SLOT + st * C::SLOT;
        sbd::mbar_arrive_expect_tx(&bars->full[st], C::SLOT);
        if (is_v) {
          for (int b = 0; b < HD / 64; ++b)
            tma_load_3d(&tmV, &bars->full[st], dst + b * (C::VK * 128), 64 * b, kv, tl.k0 + j * KB + c * C::VK);
        } else {
          for (int b = 0; b < HD / 64 / PER; ++b)
            tma_load_3d(&tmK, &bars->full[st], dst + b * (KB * 128), 64 * (c * (HD / 64 / PER) + b), kv, tl.k0 + j * KB);
        }
        ++it;
      };
      for (int j = 0; j <= nb_all && ok; ++j) {
        if (j < nb_all)
          for (int c = 0; c < PER; ++c) load(false, j0 + j, c);
        const int vj = NQ == 1 ? j - 1 : j;  // one tile: the next block's scores come before this block's P V
        if (vj >= 0 && vj < nb_all)
          for (int c = 0; c < PER; ++c) load(true, j0 + vj, c);
      }
      if (*abort) {  // copies in flight land before this CTA's shared memory is released
        for (int i = 0; i < NQ; ++i)
          if (nb[i] > 0) drain_wait(&bars->q_full[i], 0);
        for (int i = max(0, it - NSLOT); i < it; ++i) drain_wait(&bars->full[i % NSLOT], (i / NSLOT) & 1);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0 && nb_all > 0) {
      constexpr uint32_t idesc_s = idesc<T>(KB, 0), idesc_o = idesc<T>(HD, 1);
      int it = 0;
      bool ok = true;
      auto slot_wait = [&](int i) {
        ok = ok && sbd::mbar_wait(&bars->full[i % NSLOT], (i / NSLOT) & 1, abort, p.err);
        return smem + C::OFF_SLOT + (i % NSLOT) * C::SLOT;
      };
      // block j's V has landed (its items start at `at`); if it holds the sequence's end, also cleaned
      auto v_ready = [&](int j, int at) {
        if (!cleans || j0 + j != j_end) return;
        for (int c = 0; c < PER && ok; ++c) slot_wait(at + c);
        if (!ok) return;
        sbd::mbar_arrive(&bars->dirty);
        ok = sbd::mbar_wait(&bars->clean, 0, abort, p.err);
      };
      // part c of S_i(buf) = Q_i K^T from slot `ks`
      auto issue_s = [&](int i, int buf, int c, const uint8_t* ks) {
        const uint32_t qb = sbd::smem_u32(smem + i * C::Q_BYTES), kb = sbd::smem_u32(ks);
        constexpr int STEPS = HD / 16 / PER;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
          const int gs = c * STEPS + s;  // k-step of 16 dims
          const uint64_t ad = sbd::umma_desc(qb + (gs >> 2) * (QR * 128) + (gs & 3) * 32, 16, 1024, sbd::kLayoutSwizzle128B);
          const uint64_t bd = sbd::umma_desc(kb + (s >> 2) * (KB * 128) + (s & 3) * 32, 16, 1024, sbd::kLayoutSwizzle128B);
          sbd::umma_f16(tmem + C::TM_S + buf * KB, ad, bd, idesc_s, gs > 0 ? 1u : 0u);
        }
      };
      // O_i += P(buf) V for part c of the block, from slot `vs`
      auto issue_pv = [&](int i, int buf, int c, const uint8_t* vs, bool first) {
        const uint32_t vb = sbd::smem_u32(vs);
#pragma unroll
        for (int s = 0; s < C::VK / 16; ++s) {
          const uint64_t bd = sbd::umma_desc(vb + s * 2048, C::VK * 128, 1024, sbd::kLayoutSwizzle128B);
          sbd::umma_f16_ts(tmem + i * HD, tmem + C::TM_S + buf * KB + c * (C::VK / 2) + s * 8, bd, idesc_o,
                           first && c == 0 && s == 0 ? 0u : 1u);
        }
      };
      for (int i = 0; i < NQ && ok; ++i)
        if (nb[i] > 0) ok = sbd::mbar_wait(&bars->q_full[i], 0, abort, p.err);
      if constexpr (NQ == 1) {
        auto scores = [&](int j) {
          for (int c = 0; c < PER && ok; ++c) {
            const uint8_t* ks = slot_wait(it);
            if (!ok) return;
            sbd::tc_fence_after();
            issue_s(0, j & 1, c, ks);
            sbd::umma_commit(&bars->empty[it % NSLOT]);
            ++it;
          }
          if (ok) sbd::umma_commit(&bars->s_full[j & 1]);
        };
        if (ok) scores(0);
        for (int j = 0; j < nb_all && ok; ++j) {
          if (j + 1 < nb_all) scores(j + 1);
          if (ok) v_ready(j, it);
          ok = ok && sbd::mbar_wait(&bars->p_full[j & 1], (j >> 1) & 1, abort, p.err);
          for (int c = 0; c < PER && ok; ++c) {
            const uint8_t* vs = slot_wait(it);
            if (!ok) break;
            sbd::tc_fence_after();
            issue_pv(0, j & 1, c, vs, j == 0);
            sbd::umma_commit(&bars->empty[it % NSLOT]);
            ++it;
          }
          if (ok) sbd::umma_commit(&bars->pv_done[0]);
        }
      } else {
        // items: K_0, V_0, K_1, V_1, ... (one slot each)
        const uint8_t* ks = slot_wait(0);
        if (ok) {
          sbd::tc_fence_after();
          for (int i = 0; i < NQ; ++i)
            if (nb[i] > 0) {
              issue_s(i, i, 0, ks);
              sbd::umma_commit(&bars->s_full[i]);
            }
          sbd::umma_commit(&bars->empty[0]);
        }
        for (int j = 0; j < nb_all && ok; ++j) {
          const uint8_t* vs = slot_wait(2 * j + 1);
          if (ok) v_ready(j, 2 * j + 1);
          const uint8_t* kn = j + 1 < nb_all ? slot_wait(2 * j + 2) : nullptr;
          for (int i = 0; i < NQ && ok; ++i) {
            if (j >= nb[i]) continue;
            ok = sbd::mbar_wait(&bars->p_full[i], j & 1, abort, p.err);
            if (!ok) break;
            sbd::tc_fence_after();
            issue_pv(i, i, 0, vs, j == 0);
            sbd::umma_commit(&bars->pv_done[i]);
            if (j + 1 < nb[i]) {
              issue_s(i, i, 0, kn);
              sbd::umma_commit(&bars->s_full[i]);
            }
          }
          if (!ok) break;
          sbd::umma_commit(&bars->empty[(2 * j + 1) % NSLOT]);
          if (j + 1 < nb_all) sbd::umma_commit(&bars->empty[(2 * j + 2) % NSLOT]);
        }
      }
      // every MMA issued has finished before tensor and shared memory are released
      sbd::umma_commit(&bars->drain);
      drain_wait(&bars->drain, 0);
    }
  } else if (warp < 4) {
    // ------------------------------------------------------------ V rows past the sequence's end
    if (cleans) {
      const int j = j_end - j0, from = k_len % KB;
      // V_j's first item in the producer's order
      const int item = NQ == 1 ? PER * (min(j + 2, nb_all) + j) : 2 * j + 1;
      // the issuer, which follows the slots' phases, says when they have landed
      const bool ok = __all_sync(0xFFFFFFFFu, sbd::mbar_wait(&bars->dirty, 0, abort, p.err));
      for (int c = 0; c < PER && ok; ++c) {
        uint8_t* vs = smem + C::OFF_SLOT + (item + c) % NSLOT * C::SLOT;
        // whole rows of 128 bytes per box: the swizzle only permutes inside them
        const int lo = max(0, from - c * C::VK);
        for (int b = 0; b < HD / 64; ++b)
          for (int x = lo * 8 + (threadIdx.x - 64); x < C::VK * 8; x += 64)
            *reinterpret_cast<uint4*>(vs + b * (C::VK * 128) + x * 16) = make_uint4(0, 0, 0, 0);
      }
      sbd::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0 && ok) sbd::mbar_arrive(&bars->clean);
    }
  } else {
    // ------------------------------------------------------------ softmax and output
    const int i = (warp - 4) >> 2;  // tile
    const int quad = warp & 3, row = quad * 32 + lane;
    const int tok = row / p.group, head = row - tok * p.group;
    const int n_tok = min(p.tpt, tl.n_tok - i * p.tpt);
    const bool row_ok = tok < n_tok;
    const int pos = tl.pos0 + i * p.tpt + tok;
    // keys [lo, hi) of the sequence
    const int hi = row_ok ? min(pos + 1, k_len) : 0;
    const int lo = p.window > 0 ? pos + 1 - p.window : 0;
    // blocks that every row of the tile sees whole need no mask
    const int all_hi = min(tl.pos0 + i * p.tpt + 1, k_len);
    const int all_lo = p.window > 0 ? tl.pos0 + i * p.tpt + n_tok - p.window : 0;
    const uint32_t tm = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < nb[i] && ok; ++j) {
      const int buf = NQ == 1 ? j & 1 : i;
      const uint32_t ph = NQ == 1 ? (j >> 1) & 1 : j & 1;
      ok = __all_sync(0xFFFFFFFFu, sbd::mbar_wait(&bars->s_full[buf], ph, abort, p.err));
      if (!ok) break;
      sbd::tc_fence_after();
      const uint32_t ts = tm + C::TM_S + buf * KB;
      uint32_t sv[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) sbd::tmem_ld_32x32b_x32(ts + 32 * c, sv[c]);
      sbd::tmem_wait_ld();
      const int kb = (j0 + j) * KB;
      if (kb + KB > all_hi || kb < all_lo) {
        const int v0 = lo - kb, v1 = hi - kb;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            sv[c][e] = 32 * c + e >= v0 && 32 * c + e < v1 ? sv[c][e] : 0xFF800000u;  // -inf
      }
      float mx[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        mx[c] = __uint_as_float(sv[c][0]);
#pragma unroll
        for (int e = 1; e < 32; ++e) mx[c] = fmaxf(mx[c], __uint_as_float(sv[c][e]));
      }
      const float mx2 = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale2;
      const bool start = m == -INFINITY;  // O is still zero in this row
      const bool rise = !start && mx2 > m + kRise;
      if (__any_sync(0xFFFFFFFFu, rise)) {
        // O += P_{j-1} V_{j-1} has to be complete before it is scaled
        ok = __all_sync(0xFFFFFFFFu, sbd::mbar_wait(&bars->pv_done[i], (j - 1) & 1, abort, p.err));
        if (!ok) break;
        sbd::tc_fence_after();
        const float alpha = rise ? ex2(m - mx2) : 1.f;
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t ov[32];
          sbd::tmem_ld_32x32b_x32(tm + i * HD + 32 * c, ov);
          sbd::tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
          sbd::tmem_st_32x32b_x16(tm + i * HD + 32 * c, *reinterpret_cast<const uint32_t(*)[16]>(&ov[0]));
          sbd::tmem_st_32x32b_x16(tm + i * HD + 32 * c + 16, *reinterpret_cast<const uint32_t(*)[16]>(&ov[16]));
        }
        sbd::tmem_wait_st();
        l *= alpha;
      }
      if (start || rise) m = mx2;
      const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t pk[16];
        float ls[2] = {0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float p0 = ex2(fmaf(__uint_as_float(sv[c][2 * e]), p.scale2, -mu));
          const float p1 = ex2(fmaf(__uint_as_float(sv[c][2 * e + 1]), p.scale2, -mu));
          ls[0] += p0;
          ls[1] += p1;
          pk[e] = sbp::pack2<T>(p0, p1);
        }
        l += ls[0] + ls[1];
        sbd::tmem_st_32x32b_x16(ts + 16 * c, pk);
      }
      sbd::tmem_wait_st();
      sbd::tc_fence_before();
      __syncwarp();
      if (lane == 0) sbd::mbar_arrive(&bars->p_full[buf]);
    }
    // ------------------------------------------------------------ O / l
    if (ok && nb[i] > 0) ok = __all_sync(0xFFFFFFFFu, sbd::mbar_wait(&bars->pv_done[i], (nb[i] - 1) & 1, abort, p.err));
    if (ok) {
      sbd::tc_fence_after();
      const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
      const int64_t token = static_cast<int64_t>(tl.q0) + i * p.tpt + tok;
      T* dst = static_cast<T*>(p.out) + token * p.out_token + static_cast<int64_t>(kv * p.group + head) * p.out_head;
      const bool store = row_ok && token >= 0 && token < p.t_q;
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t ov[32];
        if (nb[i] > 0) {
          sbd::tmem_ld_32x32b_x32(tm + i * HD + 32 * c, ov);
          sbd::tmem_wait_ld();
        }
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          uint32_t w[4];
#pragma unroll
          for (int q = 0; q < 4; ++q)
            w[q] = l == 0.f ? 0u : sbp::pack2<T>(__uint_as_float(ov[e + 2 * q]) * inv, __uint_as_float(ov[e + 2 * q + 1]) * inv);
          if (store) *reinterpret_cast<uint4*>(dst + 32 * c + e) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
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

template <typename T, int HD>
int launch_packed(const void* q, const void* k, const void* v, const Strides& st, const PackedParams& p, int n_tiles,
                  cudaStream_t stream) {
  using C = Cfg<HD>;
  constexpr bool bf = !std::is_same<T, __half>::value;
  CUtensorMap tq, tk, tv;
  int rc = make_map3(&tq, bf, q, HD, p.group * p.nkv, p.t_q, st.q_head, st.q_token, p.group, p.tpt);
  const int t_k = std::max(p.t_k, 1);
  if (!rc) rc = make_map3(&tk, bf, k, HD, p.nkv, t_k, st.k_head, st.k_token, 1, KB);
  if (!rc) rc = make_map3(&tv, bf, v, HD, p.nkv, t_k, st.k_head, st.k_token, 1, C::VK);
  if (rc) return rc;
  static bool set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(attn_packed_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return sb::cuda_fail(e, "attn_packed_kernel smem attribute");
    if (dev >= 0 && dev < 64) set[dev] = true;
  }
  cudaError_t e = sb::launch_pdl(attn_packed_kernel<T, HD>, dim3(n_tiles * p.nkv), dim3(C::THREADS), C::SMEM, stream, tq, tk, tv, p);
  if (e != cudaSuccess) return sb::cuda_fail(e, "attn_packed_kernel");
  return sb::launch_status("attn_packed_kernel");
}

template <typename T>
int launch_packed_hd(int hd, const void* q, const void* k, const void* v, const Strides& st, const PackedParams& p,
                     int n_tiles, cudaStream_t s) {
  if (hd == 64) return launch_packed<T, 64>(q, k, v, st, p, n_tiles, s);
  if (hd == 128) return launch_packed<T, 128>(q, k, v, st, p, n_tiles, s);
  return launch_packed<T, 256>(q, k, v, st, p, n_tiles, s);
}

// Query tokens per CTA.
int tokens_per_cta(int group, int hd) { return (hd == 256 ? 1 : 2) * (QR / group); }

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
  const int per = tokens_per_cta(n_heads / n_kv_heads, head_dim);
  int64_t count = 0, tq = 0, tk = 0;
  for (int i = 0; i < n; ++i) {
    const int kl = kv_lens ? kv_lens[i] : q_lens[i];
    SB_CHECK_ARG(q_lens[i] >= 0 && kl >= 0, "sb_attn_packed_plan: negative length of sequence %d", i);
    count += (q_lens[i] + per - 1) / per;
    tq += q_lens[i];
    tk += kl;
  }
  SB_CHECK_ARG(tq < (1ll << 31) && tk < (1ll << 31) && count * n_kv_heads < (1ll << 31), "sb_attn_packed_plan: too many tokens");
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
                   static_cast<int64_t>(n_tiles) * n_kv_heads < (1ll << 31), "sb_attn_prefill_packed: bad sizes");
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
  p.t_q = t_q, p.t_k = t_k, p.nkv = n_kv_heads, p.group = n_heads / n_kv_heads, p.tpt = QR / p.group;
  p.window = window, p.scale2 = scale * kLog2e;
  if (t_k == 0) k = v = q;  // nothing is read; the maps need an address
  const Strides st{q_token, q_head, k_token, k_head};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == SB_F16 ? launch_packed_hd<__half>(head_dim, q, k, v, st, p, n_tiles, s)
                         : launch_packed_hd<__nv_bfloat16>(head_dim, q, k, v, st, p, n_tiles, s);
}
