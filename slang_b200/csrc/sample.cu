// Sampling of the next token (sb_sample): temperature, then top-k, then top-p of
// the top-k's mass, then min-p, drawn by a race that random numbers decide.
//
// With w_i = exp((x_i - max x) / T) and E_i = -log(1 - u_i) exponential waiting
// times, the token with the smallest E_i / w_i among the kept ones is a draw
// with probabilities w_i / sum of the kept w (the minimum of exponentials of
// rates w_i).  u_i = (word i + 1/2) 2^-32 of Philox4x32-10 (Salmon, Moraes, Dror
// and Shaw, SC 2011) under the row's seed as the key and (i / 4, position) as
// the counter, so nothing random is stored and a row's draw depends on its own
// seed, position and logits alone.  Unlike inverting the cumulative
// distribution this needs no sum over the vocabulary in some order, and it makes
// top-p cheap: the nucleus is a prefix of the ranking, so
//   race among all; if the mass ranked before the winner reaches p of the
//   total, the winner and all that rank behind it are out: race again among
//   those before it
// ends with the nucleus' own winner, after 1 / p rounds or so.
//
// Bound by reading the logits once.  A row is cut into segments of 1024 values, a
// warp takes whole segments, and a row's CTAs (one, or a thread-block cluster when
// the rows are few) exchange a few words through distributed shared memory.  The
// one pass over the row leaves each lane's maximum of its 32 values of a segment
// and each segment's mass in shared memory; what follows reads again only the
// lanes whose maximum can matter, mostly from the L2 cache:
//   the race      needs every token's random word, but no logit: a token can win only
//                 if u <= t w, where t is a time already reached and w at most
//                 that of its lane's maximum, one integer comparison per word.
//                 Only the few that pass are read and get their logarithm.
//   top-p         one pass sums what ranks before the winner.  A token below (1 - p) / V of
//                 the total is out from the start: all such tokens together
//                 weigh less than 1 - p, so the prefix above them holds the nucleus.
//   min-p         a token below w = min_p is out (min_p <= 1 here: above it the largest is drawn).
//   top-k         the k-th largest of the lanes' maxima is a lower bound of
//                 the k-th largest value; what reaches it (a little more than
//                 k tokens) is sorted by one CTA, which finishes the row alone.
// Masses are added as integers, those of a segment in one order, so neither the
// order of arrival nor the number of CTAs shows in the result.
//
// One row of 262144 f32 logits with top-p takes 11.5 us where the first winner stands:
// 2.2 for the pass, 2.8 for the random words on the row's 16 SMs, the rest three joins
// of its CTAs; 14 to 16 on average over rows that race again.  128 such rows with mixed
// settings take 61 to 65 us by their draws (2.1 TB/s): greedy rows alone 26 (5.1 TB/s),
// min-p 37, top-k of 20 to 200 61, no filter 64, top-p 92 to 101; mixed with the softcap,
// whose tanhf is taken of every value that is read, 120 to 132.  The random words bound
// the rows without a filter and with top-p: twenty 32 x 32 -> 64 products per four
// tokens, 16 a cycle and SM, are 37 us for 33.5 million tokens.  (High words through f64
// multiply-adds rounded down are exact too and took 8 % longer without a filter.)
//
// Rows whose top-k has more than 1024 candidates (k near 870 and above of 262144 such
// logits, or thousands of equal values) are searched bit by bit, some 50 passes each:
// 128 rows with k = 1100 take 1750 us, with k = 850, where a few rows are among them, 95 to
// 480.
#include <algorithm>

#include "paged.cuh"

namespace {

constexpr int NT = 256;         // threads per CTA
constexpr int CTAS = 4;         // CTAs per SM
constexpr int NW = NT / 32;
constexpr int MAX_CS = 16;      // CTAs per row
constexpr int SEG = 1024;       // values per segment: 32 per lane, in 8 vectors
constexpr int MAX_V = 800 * SEG;  // 25600 lane maxima: 100 KB in one CTA
constexpr int BINS = 256;       // of maxima, 1/8 octave of w each
constexpr int SORT = 1024;      // candidates of a top-k row that one CTA sorts
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLargest = 3.402823466e38f;  // bounds stay finite: -inf (banned, padding) is below them
// Masses in units of 2^-40 of the largest token's: a row's stay below 2^60, and 819200 tokens below a unit each
// weigh less than 2^-20 of it.
constexpr float kUnit = 1099511627776.f;

struct SampleParams {
  const void* x;
  int64_t ld;
  int v, segs;   // segs: segments of a row
  int vec;       // rows start on a 4-value boundary
  int sorted;    // the costly rows first
  float softcap; // 0: off
  const int64_t* seeds;
  const int32_t* pos;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int32_t* tokens;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Ranking bits of a value; -0 ranks with 0.
__device__ __forceinline__ uint32_t order_of(float x) { return sbd::orderable(x + 0.f); }

// What the CTAs of a cluster exchange in one step: a sum, the smallest key with
// a value that goes with it, and a count with the part that lower ranks hold.
struct Word {
  unsigned long long sum, key;
  unsigned int aux, count;
};

struct Shared {
  Word slot[2][MAX_CS * NW];  // the words of all warps of the cluster, in turn
  unsigned long long scan[NW];
  unsigned int n;      // entries of this CTA's list
  int bin;
  unsigned int hist[BINS];
  unsigned long long list[SORT];  // candidates here: (inverted ranking bits, index), smaller ranks before
  alignas(16) unsigned long long keys[SORT];  // a top-k row's, in the CTA of rank 0
};

// Philox4x32-10 under one key: the keys of its ten rounds are kept, a call is
// twenty 64-bit products and as many three-way exclusive ors.
struct Philox {
  uint32_t k0[10], k1[10], c1;
  __device__ __forceinline__ Philox(uint64_t seed, uint32_t pos) : c1(pos) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
      k0[r] = static_cast<uint32_t>(seed) + r * 0x9E3779B9u;
      k1[r] = static_cast<uint32_t>(seed >> 32) + r * 0xBB67AE85u;
    }
  }
  __device__ __forceinline__ uint4 operator()(uint32_t c0) const {
    uint4 c = make_uint4(c0, c1, 0, 0);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
      const uint64_t a = static_cast<uint64_t>(c.x) * 0xD2511F53u, b = static_cast<uint64_t>(c.z) * 0xCD9E8D57u;
      c = make_uint4(static_cast<uint32_t>(b >> 32) ^ c.y ^ k0[r], static_cast<uint32_t>(b),
                     static_cast<uint32_t>(a >> 32) ^ c.w ^ k1[r], static_cast<uint32_t>(a));
    }
    return c;
  }
};

// The join of a warp's words, in every lane: the 64-bit parts in pieces that the
// 32-bit warp reductions take (sums below 2^60 in pieces of 20 bits).
__device__ __forceinline__ Word warp_join(Word w) {
  constexpr unsigned kAll = 0xFFFFFFFFu;
  Word r;
  r.sum = __reduce_add_sync(kAll, static_cast<unsigned>(w.sum & 0xFFFFFu)) +
          (static_cast<unsigned long long>(__reduce_add_sync(kAll, static_cast<unsigned>(w.sum >> 20 & 0xFFFFFu))) << 20) +
          (static_cast<unsigned long long>(__reduce_add_sync(kAll, static_cast<unsigned>(w.sum >> 40))) << 40);
  const unsigned hi = __reduce_min_sync(kAll, static_cast<unsigned>(w.key >> 32));
  const unsigned lo = __reduce_min_sync(kAll, static_cast<unsigned>(w.key >> 32) == hi ? static_cast<unsigned>(w.key) : ~0u);
  r.key = static_cast<unsigned long long>(hi) << 32 | lo;
  r.aux = __shfl_sync(kAll, w.aux, __ffs(__ballot_sync(kAll, w.key == r.key)) - 1);
  r.count = __reduce_add_sync(kAll, w.count);
  return r;
}

// Joins the words of all threads of the cluster (keys differ, or are ~0).  Each warp puts its word into every CTA's
// shared memory and, after one barrier, joins what has arrived in its own.  Two buffers in turn: a word is replaced
// only after a barrier that its readers reach once they have read it.  `lower`: the count in CTAs of lower rank.
__device__ Word reduce(Shared& sh, Word w, int cs, int& turn, unsigned* lower = nullptr) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = cs > 1 ? static_cast<int>(sbd::cluster_ctarank()) : 0;
  Word* slot = sh.slot[turn];
  turn ^= 1;
  w = warp_join(w);
  if (cs > 1) {
    if (lane < cs) {
      const uint32_t a = sbd::mapa_shared(sbd::smem_u32(slot + rank * NW + warp), lane);
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(w.sum) : "memory");
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a + 8), "l"(w.key) : "memory");
      asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(a + 16), "r"(w.aux), "r"(w.count) : "memory");
    }
    sbd::cluster_sync_all();
  } else {
    if (lane == 0) slot[warp] = w;
    __syncthreads();
  }
  w = Word{0, ~0ull, 0, 0};
  unsigned below = 0;
  for (int i = lane; i < cs * NW; i += 32) {
    const Word o = slot[i];
    w.sum += o.sum, w.count += o.count;
    if (o.key < w.key) w.key = o.key, w.aux = o.aux;
    below += i < rank * NW ? o.count : 0;
  }
  if (lower) *lower = __reduce_add_sync(0xFFFFFFFFu, below);
  return warp_join(w);
}

// Settings that keep the largest logit alone (of equal ones the first).  No weight reaches a min_p above 1.
__device__ __forceinline__ bool is_greedy(float temp, float top_p, float min_p, int top_k) {
  return !(temp > 0.f) || top_p <= 0.f || !(min_p <= 1.f) || top_k == 1;
}

// The row of this cluster when the rows are more than one wave of CTAs: within NT neighbours those that take longest
// come first (top-p without top-k, no filter, top-k, min-p, greedy; stable), so that the last ones to start are short.
// Rows of 262144 with mixed settings: 128 of them 63.6 us in place of 66.4, with the softcap 122 in place of 141, 256 of
// them 101 in place of 111; rows all of one kind pay 2 us, of 25 (greedy) to 100.
__device__ __forceinline__ int sorted_row(const SampleParams& p, Shared& sh) {
  constexpr int KINDS = 6;  // the last: past the last row
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = static_cast<int>(blockIdx.y) / NT * NT, r = first + threadIdx.x;
  int kind = KINDS - 1;
  if (r < static_cast<int>(gridDim.y)) {
    const float temp = p.temperature ? p.temperature[r] : 1.f, top_p = p.top_p ? p.top_p[r] : 1.f;
    const float min_p = p.min_p ? p.min_p[r] : 0.f;
    const int top_k = p.top_k ? p.top_k[r] : 0;
    if (is_greedy(temp, top_p, min_p, top_k)) kind = 4;
    else if (top_k > 0) kind = 2;
    else if (min_p > 0.f) kind = 3;
    else kind = top_p < 1.f ? 0 : 1;
  }
  unsigned* count = reinterpret_cast<unsigned*>(sh.keys);  // [KINDS][NW]
  unsigned before = 0;
#pragma unroll
  for (int k = 0; k < KINDS; ++k) {
    const unsigned m = __ballot_sync(0xFFFFFFFFu, kind == k);
    if (lane == 0) count[k * NW + warp] = __popc(m);
    if (kind == k) before = __popc(m & ((1u << lane) - 1u));
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < KINDS * NW; i += 4) {
    const uint4 c = *reinterpret_cast<const uint4*>(count + i);
    const int n = kind * NW + warp - i;  // the counts before this warp's of its kind
    before += (n > 0 ? c.x : 0) + (n > 1 ? c.y : 0) + (n > 2 ? c.z : 0) + (n > 3 ? c.w : 0);
  }
  if (before == blockIdx.y - first) sh.bin = r;
  __syncthreads();
  return sh.bin;
}

template <typename T>
__global__ void __launch_bounds__(NT, CTAS) sample_kernel(const SampleParams p) {
  extern __shared__ __align__(16) float lane_max[];  // [local segment][lane], then [local segment] {largest, mass}
  __shared__ Shared sh;
  const int cs = gridDim.x, rank = blockIdx.x;  // a cluster spans the x axis
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rounds = (p.segs + cs * NW - 1) / (cs * NW);  // segments per warp; local segment l = round * NW + warp
  float2* seg_mass = reinterpret_cast<float2*>(lane_max + rounds * NW * 32);
  auto seg_of = [&](int round) { return (round * cs + rank) * NW + warp; };
  sbd::griddep_launch_dependents();
  if (cs > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
  if (threadIdx.x < BINS) sh.hist[threadIdx.x] = 0;
  if (threadIdx.x == 0) sh.n = 0;
  sbd::griddep_wait();
  const int row = p.sorted ? sorted_row(p, sh) : blockIdx.y;
  const float temp = p.temperature ? p.temperature[row] : 1.f;
  const float top_p = p.top_p ? p.top_p[row] : 1.f, min_p = p.min_p ? p.min_p[row] : 0.f;
  const int top_k = p.top_k ? p.top_k[row] : 0;
  const int64_t seed = p.seeds[row];
  const int pos = p.pos[row];
  const T* src = static_cast<const T*>(p.x) + row * p.ld;
  const bool greedy = is_greedy(temp, top_p, min_p, top_k);
  const float inv = fmaxf(kLog2e / temp, 1e-45f);  // above zero, so that -inf stays -inf at any temperature
  int turn = 0;

  // This lane's values of a segment: v[4 j + e] is value seg * SEG + 128 j + 4 lane + e, -inf for NaN and past the end.
  auto load = [&](int seg, float (&v)[32]) {
    const int at = seg * SEG + 4 * lane;
    if (p.vec && seg * SEG + SEG <= p.v) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (sizeof(T) == 4) {
          const uint4 r = sbd::ldg_nc_v4(src + at + 128 * j);
          v[4 * j] = __uint_as_float(r.x), v[4 * j + 1] = __uint_as_float(r.y);
          v[4 * j + 2] = __uint_as_float(r.z), v[4 * j + 3] = __uint_as_float(r.w);
        } else {
          const uint2 r = __ldg(reinterpret_cast<const uint2*>(src + at + 128 * j));
          const float2 a = sbp::unpack2<T>(r.x), b = sbp::unpack2<T>(r.y);
          v[4 * j] = a.x, v[4 * j + 1] = a.y, v[4 * j + 2] = b.x, v[4 * j + 3] = b.y;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const int idx = at + 128 * (i >> 2) + (i & 3);
        v[i] = idx < p.v ? static_cast<float>(src[idx]) : -INFINITY;
      }
    }
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = fmaxf(v[i], -INFINITY);  // NaN
    if (p.softcap > 0.f) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = v[i] == -INFINITY ? v[i] : p.softcap * tanhf(v[i] / p.softcap);
    }
  };
  auto fetch = [&](int idx) {  // one of them, as `load` gives it
    const float x = fmaxf(static_cast<float>(src[idx]), -INFINITY);
    return p.softcap > 0.f && x > -INFINITY ? p.softcap * tanhf(x / p.softcap) : x;
  };
  auto index_of = [&](int seg, int i) { return seg * SEG + 128 * (i >> 2) + 4 * lane + (i & 3); };

  // ---- the pass over the row: the largest value (ties: the lowest index), lane maxima, segment masses
  float wmax = -INFINITY;  // this warp's, with its index
  unsigned widx = ~0u;
  for (int r = 0; r < rounds; ++r) {
    const int seg = seg_of(r);
    float m = -INFINITY, sm = -INFINITY, sum = 0.f;
    if (seg < p.segs) {
      float v[32];
      load(seg, v);
#pragma unroll
      for (int i = 0; i < 32; ++i) m = fmaxf(m, v[i]);
      sm = m;
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) sm = fmaxf(sm, __shfl_xor_sync(0xFFFFFFFFu, sm, o));
      if (sm > wmax) {  // segments come in rising order: an equal value later has a higher index
        unsigned idx = ~0u;
        if (m == sm) {
#pragma unroll
          for (int i = 31; i >= 0; --i) idx = v[i] == m ? index_of(seg, i) : idx;
        }
        wmax = sm;
        widx = __reduce_min_sync(0xFFFFFFFFu, idx);
      }
      if (top_p < 1.f && !greedy && sm > -INFINITY) {
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 32; ++i) part[i & 3] += ex2(fminf((v[i] - sm) * inv, 0.f));
        sum = (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
      }
    }
    lane_max[(r * NW + warp) * 32 + lane] = m;
    if (lane == 0) seg_mass[r * NW + warp] = make_float2(sm, sum);
  }
  Word w0{0, ~0ull, 0, 0};
  if (widx != ~0u && wmax > -INFINITY) w0.key = static_cast<unsigned long long>(~order_of(wmax)) << 32 | widx, w0.aux = __float_as_uint(wmax);
  if (cs > 1) asm volatile("barrier.cluster.wait;" ::: "memory");  // the CTAs whose memory takes the words have started
  w0 = reduce(sh, w0, cs, turn);
  int token = static_cast<int>(w0.key & 0xFFFFFFFFu);  // -1 when no value is above -inf
  const float mx = __uint_as_float(w0.aux);
  if (w0.key == ~0ull || greedy) {
    if (rank == 0 && threadIdx.x == 0) p.tokens[row] = token;
    return;  // what other CTAs write here has arrived
  }
  // log2 of w; fminf gives the maximum itself 0 even where it is infinite (inf - inf)
  auto z2_of = [&](float x) { return fminf((x - mx) * inv, 0.f); };
  // race key of a token with random word q: its waiting time over its rate, then its index; ~0 below min_p
  auto race = [&](float x, int idx, uint32_t q) {
    const float wx = expf(x == mx ? 0.f : (x - mx) / temp);
    if (!(wx >= min_p && wx > 0.f) && x != mx) return ~0ull;
    const float u = fminf((__uint2float_rn(q) + 0.5f) * 2.3283064365386963e-10f, 0.99999994f);
    return static_cast<unsigned long long>(__float_as_uint(-log1pf(-u) / wx)) << 32 | static_cast<uint32_t>(idx);
  };
  const Philox philox(static_cast<uint64_t>(seed), static_cast<uint32_t>(pos));
  auto word_of = [&](int idx) {
    const uint4 r = philox(static_cast<uint32_t>(idx) >> 2);
    const uint32_t lo = idx & 1 ? r.y : r.x, hi = idx & 1 ? r.w : r.z;
    return idx & 2 ? hi : lo;
  };
  auto mass_of = [&](float z2) { return __float2ull_rn(ex2(z2) * kUnit); };
  auto value_bits = [](uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o); };
  auto value_of = [&](unsigned long long key) { return value_bits(~static_cast<uint32_t>(key >> 32)); };
  // a value below every x with log2 w >= c, whatever the rounding on either side
  auto floor_of = [&](float c) { return mx == INFINITY ? kLargest : fmaxf(mx + (c - 0.01f) / inv - fabsf(mx) * 0x1p-21f, -kLargest); };
  // Calls f(seg, v) with the segments of this warp that hold a value of at least `least`; the values of
  // lanes without one are -inf.
  auto visit = [&](float least, auto f, unsigned limit = ~0u) {
    for (int r = 0; r < rounds; ++r) {
      // one read for the whole warp, whose lanes have to leave together
      if (__shfl_sync(0xFFFFFFFFu, *static_cast<volatile unsigned*>(&sh.n), 0) > limit) break;
      const int seg = seg_of(r);
      const bool hit = lane_max[(r * NW + warp) * 32 + lane] >= least;  // -inf past the last segment
      if (!__any_sync(0xFFFFFFFFu, hit)) continue;
      float v[32];
      if (hit) {
        load(seg, v);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = -INFINITY;
      }
      f(seg, v);
    }
  };
  // the keys of this CTA's values of at least `least` into sh.list, sh.n of them; beyond SORT it gives up.  A
  // lane's hits become a bit mask, so that a warp takes its places with one atomic.
  auto collect = [&](float least) {
    visit(least, [&](int seg, float (&v)[32]) {
      uint32_t hits = 0;
#pragma unroll
      for (int i = 0; i < 32; ++i) hits |= v[i] >= least ? 1u << i : 0u;
      const unsigned mine = __popc(hits);
      unsigned inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned c = __shfl_up_sync(0xFFFFFFFFu, inc, o);
        if (lane >= o) inc += c;
      }
      unsigned base = 0;
      if (lane == 31 && inc) base = atomicAdd(&sh.n, inc);
      base = __shfl_sync(0xFFFFFFFFu, base, 31) + inc - mine;
      if (base + mine > SORT) hits = 0;  // the list will not be used
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (hits >> i & 1) sh.list[base++] = static_cast<unsigned long long>(~order_of(v[i])) << 32 | static_cast<uint32_t>(index_of(seg, i));
    }, SORT);
    __syncthreads();
  };

  auto bin_of = [&](float x) { return static_cast<int>(fminf(-8.f * z2_of(x), static_cast<float>(BINS - 1))); };
  auto count_maxima = [&] {
    for (int r = 0; r < rounds; ++r) {
      const float m = lane_max[(r * NW + warp) * 32 + lane];
      if (m > -INFINITY) atomicAdd(&sh.hist[bin_of(m)], 1u);
    }
  };
  // after a barrier of the cluster: thread b < BINS gets the row's count of bin b
  auto bin_count = [&] {
    unsigned cnt = 0;
    for (int r = 0; r < cs; ++r) {
      unsigned c;
      asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(c) : "r"(sbd::mapa_shared(sbd::smem_u32(&sh.hist[threadIdx.x]), r)) : "memory");
      cnt += c;
    }
    return cnt;
  };
  static_assert(BINS == NT, "a bin per thread");
  // inclusive sum over the threads
  auto scan = [&](unsigned long long v, unsigned long long* whole) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long c = __shfl_up_sync(0xFFFFFFFFu, v, o);
      if (lane >= o) v += c;
    }
    if (lane == 31) sh.scan[warp] = v;
    __syncthreads();
    *whole = 0;
    for (int w = 0; w < NW; ++w) {
      const unsigned long long c = sh.scan[w];
      v += w < warp ? c : 0;
      *whole += c;
    }
    __syncthreads();
    return v;
  };

  uint32_t xl = 0;  // the race is among tokens that rank before (xl, il): ranking bits, index
  int il = p.v;
  if (top_k > 0 && top_k < p.v) {
    // ---- top-k: the bin of the lanes' maxima (of all values where the maxima are too few) that reaches k;
    // every value in it or above is a candidate
    if (top_k <= p.v / 64) {
      count_maxima();
    } else {
      visit(-kLargest, [&](int, float (&v)[32]) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (v[i] > -INFINITY) atomicAdd(&sh.hist[bin_of(v[i])], 1u);
      });
    }
    if (threadIdx.x == 0) sh.bin = BINS - 1;  // not reached (fewer than k finite values): everything
    __syncthreads();
    if (cs > 1) sbd::cluster_sync_all();
    const unsigned cnt = bin_count();
    unsigned long long finite;
    const unsigned upto = static_cast<unsigned>(scan(cnt, &finite)), k = static_cast<unsigned>(top_k);
    if (upto >= k && upto - cnt < k) sh.bin = threadIdx.x;
    __syncthreads();
    const int bin = sh.bin;
    collect(bin == BINS - 1 ? -kLargest : floor_of(-0.125f * (bin + 1)));
    const unsigned mine = sh.n;
    unsigned at;
    const unsigned total = reduce(sh, Word{0, ~0ull, 0, threadIdx.x ? 0u : min(mine, SORT + 1u)}, cs, turn, &at).count;
    if (total <= SORT) {
      if (cs > 1) {
        const uint32_t dst = sbd::mapa_shared(sbd::smem_u32(sh.keys), 0);
        for (unsigned i = threadIdx.x; i < mine; i += NT)
          asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(dst + 8 * (at + i)), "l"(sh.list[i]) : "memory");
        sbd::cluster_sync_all();
        if (rank) return;  // from here on nobody reads this CTA's memory
      } else {
        for (unsigned i = threadIdx.x; i < mine; i += NT) sh.keys[i] = sh.list[i];
      }
      unsigned size = 2;
      while (size < total) size *= 2;
      for (unsigned i = total + threadIdx.x; i < size; i += NT) sh.keys[i] = ~0ull;
      __syncthreads();
      unsigned long long* key = sh.keys;
      for (unsigned k = 2; k <= size; k *= 2)  // bitonic
        for (unsigned j = k / 2; j; j /= 2) {
          for (unsigned t = threadIdx.x; t < size / 2; t += NT) {
            const unsigned a = 2 * j * (t / j) + t % j, b = a + j;
            const unsigned long long ka = key[a], kb = key[b];
            if ((ka > kb) == !(a & k)) key[a] = kb, key[b] = ka;
          }
          __syncthreads();
        }
      // E neighbouring ranks are this thread's; the mass before each
      constexpr int E = SORT / NT;
      const unsigned members = min(total, static_cast<unsigned>(top_k)), r0 = E * threadIdx.x, r1 = min(r0 + E, members);
      unsigned long long own = 0, all;
#pragma unroll 1
      for (unsigned r = r0; r < r1; ++r) own += mass_of(z2_of(value_of(key[r])));
      unsigned long long before = scan(own, &all) - own;
      const double limit = static_cast<double>(top_p) * static_cast<double>(all);
      Word best{0, ~0ull, 0, 0};
#pragma unroll 1
      for (unsigned r = r0; r < r1; ++r) {
        const float x = value_of(key[r]);
        const int idx = static_cast<int>(key[r] & 0xFFFFFFFFu);
        if (x > -INFINITY && (!(top_p < 1.f) || static_cast<double>(before) < limit)) best.key = min(best.key, race(x, idx, word_of(idx)));
        before += mass_of(z2_of(x));
      }
      int none = 0;
      best = reduce(sh, best, 1, none);
      if (threadIdx.x == 0) p.tokens[row] = static_cast<int>(best.key & 0xFFFFFFFFu);
      return;
    }
    // more candidates than one CTA sorts (a large k, or thousands of equal values): the largest value that at
    // least top_k values reach, bit by bit, then the index up to which those equal to it are in
    auto count = [&](auto in) {
      unsigned cnt = 0;
      visit(-INFINITY, [&](int seg, float (&v)[32]) {
#pragma unroll
        for (int i = 0; i < 32; ++i) cnt += index_of(seg, i) < p.v && in(order_of(v[i]), index_of(seg, i));
      });
      return reduce(sh, Word{0, ~0ull, 0, cnt}, cs, turn).count;
    };
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t c = xl | 1u << bit;
      if (count([&](uint32_t o, int) { return o >= c; }) >= static_cast<unsigned>(top_k)) xl = c;
    }
    const unsigned above = count([&](uint32_t o, int) { return o > xl; });
    int lo = 0, hi = p.v - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (above + count([&](uint32_t o, int idx) { return o == xl && idx <= mid; }) >= static_cast<unsigned>(top_k)) hi = mid;
      else lo = mid + 1;
    }
    il = lo + 1;  // ranks before (xl, il): the k in
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
  }

  // ---- the race among the tokens that rank before (xl, il)
  bool all = xl == 0;  // every token does
  auto in = [&](float x, int idx) {
    const uint32_t o = order_of(x);
    return o > xl || (o == xl && idx < il);
  };
  // log2 of the smallest w that can be kept (see above; the total is at least the largest token's 1)
  float cut = min_p > 0.f ? __log2f(min_p) : -INFINITY;
  if (top_p < 1.f) cut = fmaxf(cut, __log2f((1.f - top_p) / static_cast<float>(p.v)));
  const float least = cut > -INFINITY ? floor_of(cut) : -kLargest;
  // The largest logit's own time bounds the winner's: it is in every race that is not empty.  E >= u, so a token
  // with u > bound w is out (with a margin over what ex2 and the product are off).
  const float bound = __uint_as_float(static_cast<uint32_t>(race(mx, token, word_of(token)) >> 32));
  const float reach = __log2f(bound) + 32.01f;  // 2^(reach + log2 w): the largest word that may win
  Word w{0, ~0ull, 0, 0};
  auto enter = [&](int idx) {
    if (idx >= p.v) return;  // padding of the last segment
    const float x = fetch(idx);
    const uint32_t q = word_of(idx);
    if (x == -INFINITY || !(all || in(x, idx)) || __uint2float_rn(q) > ex2(z2_of(x) + reach)) return;
    const unsigned long long k = race(x, idx, q);
    if (k < w.key) w.key = k, w.aux = order_of(x);
  };
  // the race among values of at least `from` that rank before (xl, il)
  auto race_all = [&](float from) {
    for (int r = 0; r < rounds; ++r) {
      const float m = lane_max[(r * NW + warp) * 32 + lane];  // -inf past the last segment
      const bool hit = m >= from;
      if (!__any_sync(0xFFFFFFFFu, hit)) continue;
      const uint32_t top = __float2uint_ru(ex2(z2_of(m) + reach));
      const int seg = seg_of(r);
      uint32_t may = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint4 q = philox(static_cast<uint32_t>(index_of(seg, 4 * j)) >> 2);
        may |= (q.x <= top ? 1u << (4 * j) : 0u) | (q.y <= top ? 2u << (4 * j) : 0u) | (q.z <= top ? 4u << (4 * j) : 0u) |
               (q.w <= top ? 8u << (4 * j) : 0u);
      }
      // These are read.  A lane of a likely token passes most of its words: the warp takes its values side by
      // side, one latency for all; the stray ones of other lanes are their own.
      if (!hit) may = 0;
      for (unsigned busy = __ballot_sync(0xFFFFFFFFu, __popc(may) > 2); busy; busy &= busy - 1) {
        const int of = __ffs(busy) - 1;
        const uint32_t his = __shfl_sync(0xFFFFFFFFu, may, of);
        if (his >> lane & 1) enter(index_of(seg, lane) + 4 * (of - lane));
        if (lane == of) may = 0;
      }
      for (; may; may &= may - 1) enter(index_of(seg, __ffs(may) - 1));
    }
  };
  // the mass of what ranks before (xl, il); lanes below it are not read again.  A lane's values of a segment are
  // summed in f32, as in the segments' own masses, and rounded to units once.
  auto mass_all = [&] {
    visit(fmaxf(-kLargest, value_bits(xl)), [&](int seg, float (&v)[32]) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (in(v[i], index_of(seg, i))) sum += ex2(z2_of(v[i]));
      w.sum += __float2ull_rn(sum * kUnit);
    });
  };
  if (top_p < 1.f) {  // the whole: of all tokens from the segments, of a top-k's by a pass
    if (all) {
      for (int i = threadIdx.x; i < rounds * NW; i += NT) {
        const float2 f = seg_mass[i];
        if (f.x > -INFINITY) w.sum += __float2ull_rn(f.y * ex2(z2_of(f.x)) * kUnit);
      }
    } else {
      mass_all();
    }
  }
  race_all(least);
  w = reduce(sh, w, cs, turn);
  token = static_cast<int>(w.key & 0xFFFFFFFFu);
  const double enough = static_cast<double>(top_p) * static_cast<double>(w.sum);
  while (top_p < 1.f) {
    // the mass before the winner; below p of the whole it stands, else the race goes on among what ranks before it
    xl = w.aux, il = token, all = false;
    w = Word{0, ~0ull, 0, 0};
    mass_all();
    w = reduce(sh, w, cs, turn);
    if (static_cast<double>(w.sum) < enough) break;
    w = Word{0, ~0ull, 0, 0};
    race_all(fmaxf(least, value_bits(xl)));
    w = reduce(sh, w, cs, turn);
    if (w.key == ~0ull) break;  // nothing before it
    token = static_cast<int>(w.key & 0xFFFFFFFFu);
  }
  if (rank == 0 && threadIdx.x == 0) p.tokens[row] = token;
}

template <typename T>
int launch_sample(SampleParams& p, int rows, int cs, cudaStream_t stream) {
  const int local = (p.segs + cs * NW - 1) / (cs * NW) * NW;  // segments of a CTA
  const int smem = local * (32 * 4 + 8);
  static bool set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_V / SEG * (32 * 4 + 8));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return sb::cuda_fail(e, "sample_kernel attributes");
    if (dev >= 0 && dev < 64) set[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cs, rows);
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cs;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel<T>, static_cast<const SampleParams>(p));
  if (e != cudaSuccess) return sb::cuda_fail(e, "sample_kernel");
  return sb::launch_status("sample_kernel");
}

}  // namespace

extern "C" int sb_sample(const void* logits, int dtype, int64_t ld, int rows, int vocab, const int64_t* seeds,
                         const int32_t* pos, const float* temperature, const int32_t* top_k, const float* top_p,
                         const float* min_p, float softcap, int32_t* tokens, void* stream) {
  SB_CHECK_ARG(dtype == SB_F16 || dtype == SB_BF16 || dtype == SB_F32, "sb_sample: bad logits dtype");
  SB_CHECK_ARG(rows >= 0 && rows <= 65535 && vocab >= 1 && vocab <= MAX_V,
               "sb_sample: %d rows of %d logits (at most 65535 rows, %d logits)", rows, vocab, MAX_V);
  SB_CHECK_ARG(softcap >= 0.f && softcap <= kLargest, "sb_sample: softcap must be 0 (off) or positive and finite");
  SB_CHECK_ARG(rows <= 1 || ld >= vocab, "sb_sample: ld is shorter than a row");
  if (rows == 0) return SB_OK;
  SB_CHECK_ARG(logits && seeds && pos && tokens, "sb_sample: null pointer");
  const int size = dtype == SB_F32 ? 4 : 2;
  if (!sb::aligned(logits, size)) return sb::fail(SB_ERR_ALIGN, "sb_sample: logits are not aligned to their type");
  SampleParams p{};
  p.x = logits, p.ld = ld, p.v = vocab, p.seeds = seeds, p.pos = pos, p.temperature = temperature, p.top_k = top_k;
  p.top_p = top_p, p.min_p = min_p, p.tokens = tokens;
  p.vec = sb::aligned(logits, 4 * size) && (rows == 1 || ld % 4 == 0);
  p.segs = (vocab + SEG - 1) / SEG;
  p.softcap = softcap;
  // CTAs per row: as many as make about seven per SM in all, while each warp has a segment.  Rows of 262144 with mixed
  // settings: 64 of them 46 us with 16 per row (the rule's), 51 with 4; 128 of them 64 with 8 (the rule's, two waves,
  // whose phases overlap), 85 with 4, 75 with 16; 256 of them 101 with 4 (the rule's), 93 with 8, 140 with 16.  The bound
  // is met by powers of two just so: 130 rows get 4 and take 76 to 96 by their draws, where 8 took 66.
  int cs = 1;
  while (cs < MAX_CS && p.segs >= cs * 2 * NW && static_cast<int64_t>(rows) * cs * 2 <= 7 * sb::num_sms()) cs *= 2;
  p.sorted = static_cast<int64_t>(rows) * cs > CTAS * sb::num_sms() && (temperature || top_k || top_p || min_p);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == SB_F32) return launch_sample<float>(p, rows, cs, s);
  if (dtype == SB_F16) return launch_sample<__half>(p, rows, cs, s);
  return launch_sample<__nv_bfloat16>(p, rows, cs, s);
}
