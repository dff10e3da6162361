// Attention of one new token per sequence over a paged key-value cache
// (sb_attn_decode_paged): out[b, h] = softmax_t(scale q[b, h] . K_t) V over the
// keys t in [lo, pos[b]] of the sequence's pages, lo = 0 or pos + 1 - window.
//
// Bound by reading K and V once.  The cached keys of every (sequence, kv head)
// are cut into blocks of KB keys, the blocks of all of them are laid end to
// end, and each CTA of one resident wave takes an equal run of blocks: the SMs
// stay busy to the end whatever the lengths are, and the split needs no host
// knowledge of them.  A (sequence, kv head) that ends up in several CTAs is
// joined by the CTA that finishes it last (a counter, no waiting):
//   out = sum_c 2^(m_c - M) O_c / sum_c 2^(m_c - M) l_c,   M = max m_c.
//
// A warp reads K and V straight into registers in the layout of the tensor
// cores' operands (mma.sync m16n8k16): per CTA nothing is staged in shared
// memory and no warp waits for another until the join.  With t = lane % 4 and
// g = lane / 4:
//   S = Q K^T   A = Q (rows = the kv head's query heads, at most 8 or 16),
//               B = K: lane (g, t) loads 16 bytes of key g, dims 8 (t + 4 i) ...;
//               the contraction runs over the same permutation of the dims
//               on both sides, so whole vectors are the fragments.
//   O^T = V^T P^T  B = P^T, which is S's accumulator layout as it stands;
//               A = V^T: lane (g, t) loads 16 bytes (dims 64 c + 8 g ...) of keys
//               2t, 2t+1, 2t+8, 2t+9 and pairs neighbouring keys with byte permutes.
// The legacy tensor path suffices: 8 query heads per kv head need 51 TFLOP/s at
// the full memory rate.
//
// p = 2^(s - m) is rounded to the cache's type for the second product (its
// relative error is that of the output's own rounding; f16 weights are lifted, see
// kLift); m, l, S and O are f32.
// m only rises when a score passes it by 2^8, so O is rarely rescaled.
//
// Measured in a graph of such calls: 96 sequences of 4096 keys on average (ragged, 32 heads
// of 128 over 8, bf16) 269 us (1.61 GB, 6.0 TB/s, 0.93 of a copy's rate); one sequence of
// 130001 keys (8 heads of 256 over one) 35 us, 21 of them its bytes: about 5 until the first
// keys arrive (positions, page table, keys: each needs the one before), 2 to 3 for two
// joins, 2 for the launch.  One sequence of 1091 keys 10.7 us: the same latencies.  More than
// 16 query heads per kv head read K and V once per 16: 64 sequences of 4000 keys with 48
// heads of 128 over one take 78 us, with 32 over two 58 (twice the bytes, read once).
#include <algorithm>

#include "paged.cuh"

namespace {

constexpr int W = 4;  // warps per CTA
// Partials one CTA joins: more than the square root of the grid, so two levels suffice.  One sequence of 130001 keys
// (8 heads of 256 over one): 35.2 us with 24, 36.0 with 32, 35.9 with 12.
constexpr int JOIN = 24;
// Keys that a CTA has at least.  One sequence of 1091 keys (17 CTAs of 64): 10.9 us, 12.1 with 128, the same with 32.
constexpr int MIN_KEYS = 64;
constexpr float kLog2e = 1.4426950408889634f;
using sbp::kRise;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                 uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

struct DecodeParams {
  const void* q;
  int64_t q_stride;  // elements between sequences
  void* out;         // [b][nh][hd]
  sbp::Pages pages;
  const int32_t* pos;
  unsigned int* group_count;  // [grid / JOIN + 1][2], zero between calls
  unsigned int* count;        // [grid], of the split segment that starts in that CTA; zero between calls
  float* part;                // [grid][2][HT * (hd + 2)]
  int b, nkv, group, htiles, window;  // htiles: tiles of HT query heads per kv head
  float scale2;                       // scale * log2(e)
};

// Keys [lo, hi) of sequence b, hi clamped to what its pages hold.
__device__ __forceinline__ void key_range(const DecodeParams& p, int b, int* lo, int* hi) {
  const int pos = p.pos[b];
  const int64_t held = static_cast<int64_t>(p.pages.max_pages) << p.pages.shift;
  const int end = pos < 0 ? 0 : (pos < held ? pos + 1 : static_cast<int>(held));
  *hi = end;
  // the window ends at the token's own position, even when that lies past the pages
  *lo = p.window > 0 && pos >= p.window ? (pos + 1 - p.window < end ? pos + 1 - p.window : end) : 0;
}

// HD: head_dim.  HS: warps that share a key tile, each with HD / HS of the dims.
// NT: tiles of 8 query heads (HT = 8 NT heads per CTA).
template <typename T, int HD, int HS, int NT>
struct Shape {
  static constexpr int HDW = HD / HS;
  static constexpr int NS = 256 / HDW;     // 16-key subtiles per iteration: 8 KB of K and of V in flight per warp
  static constexpr int TK = 16 * NS;       // keys per warp (team) and iteration
  static constexpr int TEAMS = W / HS;
  static constexpr int KB = TK * TEAMS;    // keys per block
  static_assert(KB >= 32, "the entry point's bound on the number of blocks");
  static constexpr int HT = 8 * NT;
  static constexpr int PART = HT * (HD + 2);       // a partial: O [HT][HD], m [HT], l [HT]
  static constexpr int HP = HD + 4;                // a head's row in shared memory: neighbouring heads in other banks
  static constexpr int SM_O = TEAMS * HT * HP;     // each team's O
  static_assert(SM_O >= (JOIN + 2) * HT && JOIN <= 32 && HT % W == 0, "the join's weights lie there too; a lane per part");
  static constexpr int SM_F = SM_O + 2 * TEAMS * HT + (HS > 1 ? W * 32 * 4 * NS * NT : 0);
};

template <typename T, int HD, int HS, int NT>
__global__ void __launch_bounds__(W * 32, 2) attn_decode_paged_kernel(const DecodeParams p) {
  using C = Shape<T, HD, HS, NT>;
  constexpr int HDW = C::HDW, NS = C::NS, TK = C::TK, TEAMS = C::TEAMS, KB = C::KB, HT = C::HT;
  constexpr int KC = HDW / 32, VC = HDW / 64;  // 16-byte vectors of a key / of a value row per lane
  extern __shared__ float sm[];
  float* sm_o = sm;
  float* sm_m = sm + C::SM_O;
  float* sm_l = sm_m + TEAMS * HT;
  float* sm_x = sm_l + TEAMS * HT;  // HS > 1: the teams' partial scores
  __shared__ int sh_last;
  __shared__ int sh_scan[W], sh_first[4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int team = warp / HS, half = warp % HS;
  sbd::griddep_launch_dependents();
  sbd::griddep_wait();

  // total blocks of all sequences, this CTA's run of them [r0, r1) and the sequence that holds r0: each
  // thread counts a few neighbouring sequences, whose loads are one latency (the entry point has checked
  // that they number below 2^31)
  auto blocks_of = [&](int lo, int hi) { return (hi - lo + KB - 1) / KB * (p.nkv * p.htiles); };
  const int per = (p.b + W * 32 - 1) / (W * 32), b0 = threadIdx.x * per, b1 = min(b0 + per, p.b);
  int own = 0;
#pragma unroll 4
  for (int b = b0; b < b1; ++b) {
    int lo, hi;
    key_range(p, b, &lo, &hi);
    own += blocks_of(lo, hi);
  }
  int inc = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
    if (lane >= o) inc += v;
  }
  if (lane == 31) sh_scan[warp] = inc;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w == warp) inc += total;
    total += sh_scan[w];
  }
  // CTAs that work: each has at least MIN_KEYS keys to itself, so that joining does not cost more than it saves;
  // the first `more` of them hold `share` + 1 blocks, the others `share`
  constexpr int MIN_BLOCKS = MIN_KEYS > KB ? MIN_KEYS / KB : 1;
  const int n_cta = min(static_cast<int>(gridDim.x), (total + MIN_BLOCKS - 1) / MIN_BLOCKS);
  const int share = n_cta ? total / n_cta : 0, more = total - share * n_cta;
  auto start_of = [&](int c) { return c * share + min(c, more); };
  auto cta_of = [&](int r) { return r < more * (share + 1) ? r / (share + 1) : more + (r - more * (share + 1)) / share; };
  const bool works = static_cast<int>(blockIdx.x) < n_cta;
  const int r0 = works ? start_of(blockIdx.x) : 0, r1 = works ? start_of(blockIdx.x + 1) : 0;
  if (works && inc - own <= r0 && r0 < inc) {
    int at = inc - own, b = b0, lo, hi;
    for (;; ++b) {
      key_range(p, b, &lo, &hi);
      if (r0 < at + blocks_of(lo, hi)) break;
      at += blocks_of(lo, hi);
    }
    sh_first[0] = b, sh_first[1] = at, sh_first[2] = lo, sh_first[3] = hi;
  }
  __syncthreads();
  // The sequence in 64 bits where that saves spilled registers: 64 sequences of 4000 keys with 4 heads of 64 per kv head
  // take 59.6 us in place of 64.0; with two tiles of heads it costs some (16 heads of 512: 83.4 in place of 80.2).
  std::conditional_t<NT == 1, int64_t, int> b = sh_first[0];
  int seq_start = sh_first[1], lo = sh_first[2], hi = sh_first[3];  // seq_start: its first block
  const T* kbase = static_cast<const T*>(p.pages.k);
  const T* vbase = static_cast<const T*>(p.pages.v);
  const int pmask = (1 << p.pages.shift) - 1;

  for (int r = r0; r < r1;) {
    const int nblk = (hi - lo + KB - 1) / KB;
    if (r >= seq_start + nblk * (p.nkv * p.htiles)) {
      seq_start += nblk * (p.nkv * p.htiles);
      key_range(p, static_cast<int>(++b), &lo, &hi);
      continue;
    }
    const int hidx = (r - seq_start) / nblk;  // (kv head, head tile)
    const int seg0 = seq_start + hidx * nblk, seg1 = seg0 + nblk;
    const int e = min(r1, seg1);
    const int kv = hidx / p.htiles, h0 = (hidx % p.htiles) * HT;  // query heads kv * group + h0 ...
    const int nheads = min(HT, p.group - h0);
    const int k_begin = lo + (r - seg0) * KB, k_end = min(hi, lo + (e - seg0) * KB);
    const int32_t* row = p.pages.table + static_cast<int64_t>(b) * p.pages.max_pages;

    // Q fragments: vector i of lane (g, t) is dims half * HDW + 8 (t + 4 i) ... of heads g (and g + 8)
    uint4 qf[NT][KC];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int h = g + 8 * n;
      const T* qp = static_cast<const T*>(p.q) + b * p.q_stride + static_cast<int64_t>(kv * p.group + h0 + h) * HD + half * HDW + 8 * t;
#pragma unroll
      for (int i = 0; i < KC; ++i)
        qf[n][i] = h < nheads ? *reinterpret_cast<const uint4*>(qp + 32 * i) : make_uint4(0, 0, 0, 0);
    }
    float o[4 * VC][NT][4];
#pragma unroll
    for (int i = 0; i < 4 * VC; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[i][n][x] = 0.f;
    float m[NT], l[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) m[n] = -INFINITY, l[n] = 0.f;

    // page of key `key`, -1 for a key that takes no part
    auto page_of = [&](int key) {
      if (key >= k_end) return -1;
      const int pg = row[key >> p.pages.shift];
      return pg >= 0 && pg < p.pages.n_pages ? pg : -1;
    };
    // this lane holds the pages of keys base + lane (and + 32 when a tile has 64 keys)
    struct Held {
      int a, b;
    };
    auto fetch_page = [&](int base) {
      return Held{lane < TK ? page_of(base + lane) : -1, lane + 32 < TK ? page_of(base + lane + 32) : -1};
    };
    auto row_of = [&](const T* basep, int key, int page) {
      return basep + page * p.pages.page_stride + kv * p.pages.head_stride + (key & pmask) * p.pages.token_stride;
    };
    uint4 kf[2 * NS][KC];
    auto load_k = [&](int base, const Held& pages) {
#pragma unroll
      for (int j = 0; j < 2 * NS; ++j) {
        const int in = 8 * j + g;
        const int page = __shfl_sync(0xFFFFFFFFu, 8 * j >= 32 ? pages.b : pages.a, in & 31);
        const T* src = row_of(kbase, base + in, page) + half * HDW + 8 * t;
#pragma unroll
        for (int i = 0; i < KC; ++i) kf[j][i] = page >= 0 ? sbd::ldg_nc_v4(src + 32 * i) : make_uint4(0, 0, 0, 0);
      }
    };
    int base = k_begin + team * TK;
    Held pg = fetch_page(base);
    load_k(base, pg);
    Held pg_next = fetch_page(base + KB);
    for (; base < k_end; base += KB) {
      // V of this tile: keys 16 s + {2t, 2t+1, 2t+8, 2t+9}
      uint4 vf[NS][4][VC];
      uint32_t okmask = 0;  // bit 4 s + x: that key takes part
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int in = 16 * s + 2 * t + (x & 1) + 8 * (x >> 1);
          const int page = __shfl_sync(0xFFFFFFFFu, 16 * s >= 32 ? pg.b : pg.a, in & 31);
          const T* src = row_of(vbase, base + in, page) + half * HDW + 8 * g;
          okmask |= page >= 0 ? 1u << (4 * s + x) : 0u;
#pragma unroll
          for (int c = 0; c < VC; ++c) vf[s][x][c] = page >= 0 ? sbd::ldg_nc_v4(src + 64 * c) : make_uint4(0, 0, 0, 0);
        }
      // S: rows = heads (g, g + 8), columns = keys 2t, 2t+1 of each 8-key tile
      float sc[2 * NS][4];
#pragma unroll
      for (int j = 0; j < 2 * NS; ++j) {
#pragma unroll
        for (int x = 0; x < 4; ++x) sc[j][x] = 0.f;
#pragma unroll
        for (int i = 0; i < KC; ++i) {
          mma16816<T>(sc[j], qf[0][i].x, NT > 1 ? qf[NT - 1][i].x : 0u, qf[0][i].y, NT > 1 ? qf[NT - 1][i].y : 0u,
                      kf[j][i].x, kf[j][i].y);
          mma16816<T>(sc[j], qf[0][i].z, NT > 1 ? qf[NT - 1][i].z : 0u, qf[0][i].w, NT > 1 ? qf[NT - 1][i].w : 0u,
                      kf[j][i].z, kf[j][i].w);
        }
      }
      // the next tile's K while the softmax and the second product run
      load_k(base + KB, pg_next);
      pg = pg_next;
      pg_next = fetch_page(base + 2 * KB);
      if constexpr (HS > 1) {  // the sum of the team's shares of the dims, in one order for all of them
        constexpr int N = 4 * NS * NT;
        float* share = sm_x + (team * HS * 32 + lane) * N;
#pragma unroll
        for (int j = 0; j < 2 * NS; ++j)
#pragma unroll
          for (int x = 0; x < 2 * NT; ++x) share[half * 32 * N + j * 2 * NT + x] = sc[j][x];
        sbd::named_bar_sync(1 + team, HS * 32);
#pragma unroll
        for (int j = 0; j < 2 * NS; ++j)
#pragma unroll
          for (int x = 0; x < 2 * NT; ++x) {
            float sum = share[j * 2 * NT + x];
#pragma unroll
            for (int w = 1; w < HS; ++w) sum += share[w * 32 * N + j * 2 * NT + x];
            sc[j][x] = sum;
          }
        sbd::named_bar_sync(1 + team, HS * 32);  // the buffer is free for the next tile
      }
      uint32_t pb[2 * NS][NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < 2 * NS; ++j)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const bool ok = (okmask >> (4 * (j >> 1) + 2 * (j & 1) + x)) & 1u;
            float& v = sc[j][2 * n + x];
            v = ok ? v * p.scale2 : -INFINITY;
            mx = fmaxf(mx, v);
          }
        mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 2));
        const bool rise = mx > m[n] + kRise || (m[n] == -INFINITY && mx > -INFINITY);
        if (__any_sync(0xFFFFFFFFu, rise)) {
          const float alpha = rise ? (m[n] == -INFINITY ? 0.f : ex2(m[n] - mx)) : 1.f;
          l[n] *= alpha;
          if (rise) m[n] = mx;
          const float a0 = __shfl_sync(0xFFFFFFFFu, alpha, 8 * t), a1 = __shfl_sync(0xFFFFFFFFu, alpha, 8 * t + 4);
#pragma unroll
          for (int i = 0; i < 4 * VC; ++i) {
            o[i][n][0] *= a0, o[i][n][2] *= a0;
            o[i][n][1] *= a1, o[i][n][3] *= a1;
          }
        }
        const float mu = (m[n] == -INFINITY ? 0.f : m[n]) - sbp::kLift<T>;
#pragma unroll
        for (int j = 0; j < 2 * NS; ++j) {
          const float p0 = ex2(sc[j][2 * n] - mu), p1 = ex2(sc[j][2 * n + 1] - mu);
          l[n] += p0 + p1;
          pb[j][n] = sbp::pack2<T>(p0, p1);
        }
      }
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int c = 0; c < VC; ++c) {
          const uint32_t* r0v = reinterpret_cast<const uint32_t*>(&vf[s][0][c]);
          const uint32_t* r1v = reinterpret_cast<const uint32_t*>(&vf[s][1][c]);
          const uint32_t* r2v = reinterpret_cast<const uint32_t*>(&vf[s][2][c]);
          const uint32_t* r3v = reinterpret_cast<const uint32_t*>(&vf[s][3][c]);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t a0 = __byte_perm(r0v[w], r1v[w], 0x5410), a1 = __byte_perm(r0v[w], r1v[w], 0x7632);
            const uint32_t a2 = __byte_perm(r2v[w], r3v[w], 0x5410), a3 = __byte_perm(r2v[w], r3v[w], 0x7632);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma16816<T>(o[4 * c + w][n], a0, a1, a2, a3, pb[2 * s][n], pb[2 * s + 1][n]);
          }
        }
    }

    // join the CTA's teams: every team's O, m, l in shared memory
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      l[n] += __shfl_xor_sync(0xFFFFFFFFu, l[n], 1);
      l[n] += __shfl_xor_sync(0xFFFFFFFFu, l[n], 2);
      if (half == 0 && t == 0) {
        sm_m[team * HT + 8 * n + g] = m[n];
        sm_l[team * HT + 8 * n + g] = l[n];
      }
      // lane (g, t): heads 8 n + 2t, + 1; dims half * HDW + 64 c + 8 g + 0..7
#pragma unroll
      for (int c = 0; c < VC; ++c)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          float* dst = sm_o + (team * HT + 8 * n + 2 * t + hh) * C::HP + half * HDW + 64 * c + 8 * g;
          *reinterpret_cast<float4*>(dst) = make_float4(o[4 * c][n][hh], o[4 * c][n][2 + hh], o[4 * c + 1][n][hh], o[4 * c + 1][n][2 + hh]);
          *reinterpret_cast<float4*>(dst + 4) = make_float4(o[4 * c + 2][n][hh], o[4 * c + 2][n][2 + hh], o[4 * c + 3][n][hh], o[4 * c + 3][n][2 + hh]);
        }
    }
    __syncthreads();
    const bool whole = r == seg0 && e == seg1;
    float* part = p.part + (static_cast<int64_t>(blockIdx.x) * 2 + (r == r0 ? 0 : 1)) * C::PART;
    T* out = static_cast<T*>(p.out) + (static_cast<int64_t>(b) * p.nkv * p.group + kv * p.group + h0) * HD;
    for (int i = threadIdx.x; i < nheads * (HD / 8); i += W * 32) {
      const int h = i / (HD / 8), d = 8 * (i % (HD / 8));
      float M = sm_m[h];
#pragma unroll
      for (int w = 1; w < TEAMS; ++w) M = fmaxf(M, sm_m[w * HT + h]);
      const float mu = M == -INFINITY ? 0.f : M;
      float L = 0.f, acc[8] = {};
#pragma unroll
      for (int w = 0; w < TEAMS; ++w) {
        const float f = ex2(sm_m[w * HT + h] - mu);
        L += f * sm_l[w * HT + h];
        float v[8];
        sbp::load8(sm_o + (w * HT + h) * C::HP + d, v);
#pragma unroll
        for (int x = 0; x < 8; ++x) acc[x] += f * v[x];
      }
      if (whole) {
        const float inv = L > 0.f ? 1.f / L : (L == L ? 0.f : L);
#pragma unroll
        for (int x = 0; x < 8; ++x) acc[x] *= inv;
        sbp::store8(out + h * HD + d, acc);
      } else {
        float4* dst = reinterpret_cast<float4*>(part + h * HD + d);
        dst[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
        dst[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
        if (d == 0) part[HT * HD + h] = M, part[HT * HD + HT + h] = L;
      }
    }
    if (!whole) {
      // the CTAs that hold blocks of this segment: [c0, c1]
      const int c0 = cta_of(seg0), c1 = cta_of(seg1 - 1);
      const bool first_aligned = start_of(c0) == seg0;  // c0's run begins with this segment
      auto slot = [&](int c) { return p.part + (static_cast<int64_t>(c) * 2 + (c > c0 || first_aligned ? 0 : 1)) * C::PART; };
      // true in the last of `n` CTAs to arrive at a counter; everything they wrote before is visible to it
      auto last_of = [&](unsigned int* cnt, int n) {
        __syncthreads();
        if (threadIdx.x == 0) {  // one release / acquire for the CTA, around whose barriers its threads' accesses stand
          unsigned int seen;
          asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(seen) : "l"(cnt) : "memory");
          sh_last = seen == static_cast<unsigned int>(n - 1);
          if (sh_last) *cnt = 0;  // ready for the next call
        }
        __syncthreads();
        return sh_last != 0;
      };
      // joins the partials of n CTAs (at most JOIN), the i-th in slot(of(i)): into the output, or into the first one's slot
      auto join = [&](int n, auto of, bool final) {
        float* wgt = sm_o;  // [n][HT] weights, [HT] sums, [HT] maxima; the teams' O is no longer needed
        // Every thread has the loads of several parts of its vectors in flight at once, the first of them before the
        // weights are known.
        constexpr int VPT = HT * HD / 4 / (W * 32), UX = VPT >= 16 ? 2 : 32 / VPT > 8 ? 8 : 32 / VPT;
        float4 acc[VPT], v[UX][VPT];
        auto fetch = [&](int x) {
#pragma unroll
          for (int y = 0; y < UX; ++y) {
            const float4* src = reinterpret_cast<const float4*>(slot(of(min(x + y, n - 1)))) + threadIdx.x;
#pragma unroll
            for (int u = 0; u < VPT; ++u) v[y][u] = __ldcg(src + u * W * 32);
          }
        };
        fetch(0);
        // a warp's heads, a lane per part; rows of heads that are not there hold anything: no weight
        constexpr int HW = HT / W;
        const int at = min(lane, n - 1);
        const float* src = slot(of(at)) + HT * HD + warp * HW;
        float pm[HW], pl[HW];
#pragma unroll
        for (int x = 0; x < HW; ++x) pm[x] = __ldcg(src + x), pl[x] = __ldcg(src + HT + x);
#pragma unroll
        for (int x = 0; x < HW; ++x) {
          const int h = warp * HW + x;
          float M = pm[x];
#pragma unroll
          for (int o = 16; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xFFFFFFFFu, M, o));
          const float f = h < nheads && lane < n ? ex2(pm[x] - (M == -INFINITY ? 0.f : M)) : 0.f;
          float L = h < nheads && lane < n ? f * pl[x] : 0.f;
#pragma unroll
          for (int o = 16; o >= 1; o >>= 1) L += __shfl_xor_sync(0xFFFFFFFFu, L, o);
          if (lane < n) wgt[lane * HT + h] = f;
          if (lane == 0) wgt[n * HT + h] = L, wgt[(n + 1) * HT + h] = M;
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < VPT; ++u) acc[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int x = 0; x < n; x += UX) {
          if (x) fetch(x);
#pragma unroll
          for (int y = 0; y < UX; ++y)
#pragma unroll
            for (int u = 0; u < VPT; ++u) {
              const float f = x + y < n ? wgt[(x + y) * HT + (threadIdx.x + u * W * 32) / (HD / 4)] : 0.f;
              if (f == 0.f) continue;  // a part without weight, or of a head that is not there
              acc[u].x += f * v[y][u].x, acc[u].y += f * v[y][u].y, acc[u].z += f * v[y][u].z, acc[u].w += f * v[y][u].w;
            }
        }
#pragma unroll
        for (int u = 0; u < VPT; ++u) {
          const int i = threadIdx.x + u * W * 32, h = i / (HD / 4), d = 4 * (i % (HD / 4));
          if (h >= nheads) continue;
          const float L = wgt[n * HT + h];
          if (final) {
            const float inv = L > 0.f ? 1.f / L : (L == L ? 0.f : L);
            *reinterpret_cast<uint2*>(out + h * HD + d) =
                make_uint2(sbp::pack2<T>(acc[u].x * inv, acc[u].y * inv), sbp::pack2<T>(acc[u].z * inv, acc[u].w * inv));
          } else {
            float* dst = slot(of(0));
            *reinterpret_cast<float4*>(dst + h * HD + d) = acc[u];
            if (d == 0) dst[HT * HD + h] = wgt[(n + 1) * HT + h], dst[HT * HD + HT + h] = L;
          }
        }
      };
      unsigned int* cnt = p.count + c0;  // only the last segment that starts in a CTA reaches past it
      if (c1 - c0 < JOIN) {
        if (last_of(cnt, c1 - c0 + 1)) join(c1 - c0 + 1, [&](int i) { return c0 + i; }, true);
      } else {
        // a long segment: CTAs of each group of JOIN neighbours join first, so that no CTA reads them all.  A
        // group touches two long segments at most: one from its left, one that starts in it.
        const int grp = static_cast<int>(blockIdx.x) / JOIN, g0 = max(c0, grp * JOIN), g1 = min(c1, grp * JOIN + JOIN - 1);
        if (last_of(p.group_count + 2 * grp + (c0 < grp * JOIN ? 0 : 1), g1 - g0 + 1)) {
          join(g1 - g0 + 1, [&](int i) { return g0 + i; }, false);
          const int first = c0 / JOIN, n = c1 / JOIN - first + 1;
          if (last_of(cnt, n)) join(n, [&](int i) { return max(c0, (first + i) * JOIN); }, true);
        }
      }
    }
    __syncthreads();  // shared memory is free for the next segment
    r = e;
  }
  // sequences with no key at all: zero rows
  for (int b = blockIdx.x; b < p.b; b += gridDim.x) {
    key_range(p, b, &lo, &hi);
    if (hi > lo) continue;
    uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + static_cast<int64_t>(b) * p.nkv * p.group * HD);
    for (int i = threadIdx.x; i < p.nkv * p.group * HD / 8; i += W * 32) dst[i] = make_uint4(0, 0, 0, 0);
  }
}

int head_tile(int group) { return group <= 8 ? 8 : 16; }

// CTAs of one resident wave.
int grid_of() { return 2 * sb::num_sms(); }

// The workspace: counters of the groups and of the CTAs, then the partials.  Where each lies and how many counters
// there are depends on the GPU alone, so calls of any batch, head counts and head_dim follow each other on one
// workspace that is large enough for them: none writes a partial over another's counters.
size_t group_bytes(int grid) { return (static_cast<size_t>(grid) / JOIN + 1) * 8; }
size_t counter_bytes(int grid) { return (group_bytes(grid) + static_cast<size_t>(grid) * 4 + 255) / 256 * 256; }

template <typename T, int HD, int HS, int NT>
int launch_decode(const DecodeParams& p, int grid, cudaStream_t stream) {
  using C = Shape<T, HD, HS, NT>;
  constexpr int smem = C::SM_F * 4;
  static bool set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(attn_decode_paged_kernel<T, HD, HS, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return sb::cuda_fail(e, "attn_decode_paged_kernel smem attribute");
    if (dev >= 0 && dev < 64) set[dev] = true;
  }
  cudaError_t e = sb::launch_pdl(attn_decode_paged_kernel<T, HD, HS, NT>, dim3(grid), dim3(W * 32), smem, stream, p);
  if (e != cudaSuccess) return sb::cuda_fail(e, "attn_decode_paged_kernel");
  return sb::launch_status("attn_decode_paged_kernel");
}

template <typename T>
int launch_decode_hd(int hd, int ht, const DecodeParams& p, int grid, cudaStream_t s) {
  switch (hd) {
    case 64: return ht == 8 ? launch_decode<T, 64, 1, 1>(p, grid, s) : launch_decode<T, 64, 1, 2>(p, grid, s);
    case 128: return ht == 8 ? launch_decode<T, 128, 1, 1>(p, grid, s) : launch_decode<T, 128, 1, 2>(p, grid, s);
    case 256: return ht == 8 ? launch_decode<T, 256, 1, 1>(p, grid, s) : launch_decode<T, 256, 2, 2>(p, grid, s);
    default: return ht == 8 ? launch_decode<T, 512, 2, 1>(p, grid, s) : launch_decode<T, 512, 4, 2>(p, grid, s);
  }
}

}  // namespace

extern "C" size_t sb_attn_decode_paged_workspace_size(const sb_paged_kv* kv, int n_heads, int b) {
  if (!kv || kv->n_kv_heads < 1 || n_heads < 1 || n_heads % kv->n_kv_heads || b < 1) return 0;
  const int ht = head_tile(n_heads / kv->n_kv_heads), grid = grid_of();
  return counter_bytes(grid) + static_cast<size_t>(grid) * 2 * ht * (kv->head_dim + 2) * sizeof(float);
}

extern "C" int sb_attn_decode_paged(const sb_paged_kv* kv, const int32_t* page_table, int max_pages, const int32_t* pos,
                                    int b, const void* q, int64_t q_stride, int n_heads, int window, float scale,
                                    void* out, void* workspace, size_t workspace_bytes, void* stream) {
  DecodeParams p{};
  int rc = sbp::check_pages("sb_attn_decode_paged", kv, page_table, max_pages, &p.pages);
  if (rc) return rc;
  SB_CHECK_ARG(b >= 0 && n_heads >= 1 && n_heads % kv->n_kv_heads == 0 && window >= 0,
               "sb_attn_decode_paged: %d query heads over %d kv heads, or bad sizes", n_heads, kv->n_kv_heads);
  SB_CHECK_ARG(b <= 1 || q_stride >= static_cast<int64_t>(n_heads) * kv->head_dim, "sb_attn_decode_paged: q_stride is shorter than a row");
  if (b == 0) return SB_OK;
  SB_CHECK_ARG(pos && q && out && workspace, "sb_attn_decode_paged: null pointer");
  if (!sb::aligned(q, 16) || q_stride % 8 || !sb::aligned(out, 16) || !sb::aligned(workspace, 16))
    return sb::fail(SB_ERR_ALIGN, "sb_attn_decode_paged: q rows, out and the workspace must start on 16-byte boundaries");
  if (workspace_bytes < sb_attn_decode_paged_workspace_size(kv, n_heads, b))
    return sb::fail(SB_ERR_WORKSPACE, "sb_attn_decode_paged: workspace of %zu bytes, %zu needed", workspace_bytes,
                    sb_attn_decode_paged_workspace_size(kv, n_heads, b));
  const int group = n_heads / kv->n_kv_heads, ht = head_tile(group);
  p.q = q, p.q_stride = q_stride, p.out = out, p.pos = pos, p.b = b, p.nkv = kv->n_kv_heads, p.group = group;
  p.htiles = (group + ht - 1) / ht, p.window = window, p.scale2 = scale * kLog2e;
  // what the table's rows can hold, in the kernel's 32-bit numbers of keys and of blocks (of 32 keys at least)
  const int64_t held = static_cast<int64_t>(max_pages) * kv->page_size;
  SB_CHECK_ARG(held <= (1ll << 31) - 4096 && (held / 32 + 1) * p.nkv * p.htiles < (1ll << 31) / b,
               "sb_attn_decode_paged: a page table for %d sequences of %lld keys is too large", b, static_cast<long long>(held));
  const int grid = grid_of();
  p.group_count = static_cast<unsigned int*>(workspace);
  p.count = p.group_count + group_bytes(grid) / 4;
  p.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + counter_bytes(grid));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return kv->dtype == SB_F16 ? launch_decode_hd<__half>(kv->head_dim, ht, p, grid, s)
                             : launch_decode_hd<__nv_bfloat16>(kv->head_dim, ht, p, grid, s);
}
