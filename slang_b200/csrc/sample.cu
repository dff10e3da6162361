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
// Bound by reading the logits once.  A row belongs to one thread-block cluster
// that holds it in shared memory, a slice per CTA; every later pass reads the
// slices, and the CTAs exchange a few words each through distributed shared
// memory.  What the passes cost is kept small by working on short lists:
//   min-p, top-p  a token below w = min_p is out, and so is one below (1 - p) / V of
//                 the total: all such tokens together weigh less than 1 - p, so
//                 the prefix above them already holds the nucleus.
//   top-k         the k-th largest of the threads' own maxima is a lower bound of
//                 the k-th largest value; what reaches it (a little more than
//                 k tokens) is sorted by one CTA, which finishes the row alone.
// Masses are added as integers (w in units of 2^-40), so no order of addition
// shows in the result.
#include <algorithm>

#include "paged.cuh"

namespace {

constexpr int NT = 512;       // threads per CTA
constexpr int MAX_CS = 16;    // CTAs per row
constexpr int MAX_SLICE = 51200;  // values per CTA: 200 KB
constexpr int BINS = 256;     // of the threads' maxima, 1/8 octave of w each
constexpr int SORT = 1024;    // candidates of a top-k row that one CTA sorts
constexpr int MINE = 512;     // of those in one slice
// Candidates per CTA of other rows (16-bit offsets into the slice).  Beyond this
// many of a 16384-value slice a pass over all of it costs no more: one Philox call
// serves four values there, one here.
constexpr int LIST = 3072;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLargest = 3.402823466e38f;  // bounds stay finite: -inf (banned, padding) is below them
constexpr float kUnit = 1099511627776.f;  // 2^40

struct SampleParams {
  const void* x;
  int64_t ld;
  int v, slice;  // slice: values per CTA, a multiple of 4
  int vec;       // rows start on a 4-value boundary
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
  Word slot[2];        // this CTA's contribution, in turn
  Word warp[NT / 32];
  Word all;
  unsigned int lower;  // the count in CTAs of lower rank
  unsigned int n;      // entries of this CTA's list
  int bin;
  unsigned int hist[BINS];
  union {
    uint16_t list[LIST];
    struct {
      unsigned long long keys[SORT];  // of the whole row, in the CTA of rank 0
      uint16_t mine[MINE];
    } top;
  };
};
static_assert(sizeof(Shared) <= 11 * 1024, "three CTAs of 64 KB slices per SM");

// One counter's four words of Philox4x32-10.
__device__ __forceinline__ uint4 philox(uint32_t c0, uint32_t c1, uint32_t k0, uint32_t k1) {
  uint32_t c2 = 0, c3 = 0;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = static_cast<uint64_t>(c0) * 0xD2511F53u, b = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(b);
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

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

// Joins the words of all threads of the cluster (keys differ, or are ~0).  Two
// slots in turn: a CTA writes one again only after a barrier that every other
// CTA reaches once it has read it.
__device__ Word reduce(Shared& sh, Word w, int cs, int& turn) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  w = warp_join(w);
  if (lane == 0) sh.warp[warp] = w;
  __syncthreads();
  if (warp == 0) {
    w = warp_join(lane < NT / 32 ? sh.warp[lane] : Word{0, ~0ull, 0, 0});
    if (lane == 0) {
      (cs > 1 ? sh.slot[turn] : sh.all) = w;
      sh.lower = 0;
    }
  }
  if (cs > 1) {
    sbd::cluster_sync_all();
    if (warp == 0) {
      w = Word{0, ~0ull, 0, 0};
      if (lane < cs) {
        const uint32_t a = sbd::mapa_shared(sbd::smem_u32(&sh.slot[turn]), lane);
        asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(w.sum) : "r"(a) : "memory");
        asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(w.key) : "r"(a + 8) : "memory");
        asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(w.aux), "=r"(w.count) : "r"(a + 16) : "memory");
      }
      const unsigned lower = __reduce_add_sync(0xFFFFFFFFu, lane < static_cast<int>(sbd::cluster_ctarank()) ? w.count : 0u);
      w = warp_join(w);
      if (lane == 0) sh.all = w, sh.lower = lower;
    }
    turn ^= 1;
  }
  __syncthreads();
  return sh.all;
}

template <typename T>
__global__ void __launch_bounds__(NT, 3) sample_kernel(const SampleParams p) {
  extern __shared__ __align__(16) float xs[];  // this CTA's slice of the row, NaN as -inf, padded with -inf to a multiple of 4
  __shared__ Shared sh;
  const int cs = gridDim.x, rank = blockIdx.x, row = blockIdx.y;  // a cluster spans the x axis
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  sbd::griddep_launch_dependents();
  if (threadIdx.x < BINS) sh.hist[threadIdx.x] = 0;
  if (threadIdx.x == 0) sh.n = 0;
  sbd::griddep_wait();
  const float temp = p.temperature ? p.temperature[row] : 1.f;
  const float top_p = p.top_p ? p.top_p[row] : 1.f, min_p = p.min_p ? p.min_p[row] : 0.f;
  const int top_k = p.top_k ? p.top_k[row] : 0;
  const uint32_t k0 = static_cast<uint32_t>(p.seeds[row]), k1 = static_cast<uint32_t>(p.seeds[row] >> 32);
  const uint32_t c1 = static_cast<uint32_t>(p.pos[row]);
  const int first = rank * p.slice, n = max(0, min(p.slice, p.v - first)), n4 = (n + 3) / 4;
  const T* src = static_cast<const T*>(p.x) + row * p.ld + first;
  int turn = 0;

  // ---- the slice into shared memory; this thread's largest value, ties to the lowest index
  float tmax = -INFINITY;
  int tquad = -1;
  auto take = [&](int i, float4 f) {
    f.x = fmaxf(f.x, -INFINITY), f.y = fmaxf(f.y, -INFINITY), f.z = fmaxf(f.z, -INFINITY), f.w = fmaxf(f.w, -INFINITY);  // NaN
    const float m = fmaxf(fmaxf(f.x, f.y), fmaxf(f.z, f.w));
    if (m > tmax) tmax = m, tquad = i;
    *reinterpret_cast<float4*>(xs + 4 * i) = f;
  };
  auto quad = [&](int i) {
    if constexpr (sizeof(T) == 4) {
      const uint4 r = sbd::ldg_nc_v4(src + 4 * i);
      return make_float4(__uint_as_float(r.x), __uint_as_float(r.y), __uint_as_float(r.z), __uint_as_float(r.w));
    } else {
      const uint2 r = __ldg(reinterpret_cast<const uint2*>(src + 4 * i));
      const float2 a = sbp::unpack2<T>(r.x), b = sbp::unpack2<T>(r.y);
      return make_float4(a.x, a.y, b.x, b.y);
    }
  };
  int i0 = threadIdx.x;
  if (p.vec) {
    constexpr int U = 8;  // vectors in flight per thread
    for (; i0 + (U - 1) * NT < n / 4; i0 += U * NT) {
      float4 f[U];
#pragma unroll
      for (int u = 0; u < U; ++u) f[u] = quad(i0 + u * NT);
#pragma unroll
      for (int u = 0; u < U; ++u) take(i0 + u * NT, f[u]);
    }
    for (; i0 < n / 4; i0 += NT) take(i0, quad(i0));
  }
  for (; i0 < n4; i0 += NT) {
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = 4 * i0 + e < n ? static_cast<float>(src[4 * i0 + e]) : -INFINITY;
    take(i0, make_float4(v[0], v[1], v[2], v[3]));
  }
  Word w0{0, ~0ull, 0, 0};
  if (tquad >= 0) {
    const float4 f = *reinterpret_cast<const float4*>(xs + 4 * tquad);  // this thread's own store
    const int idx = first + 4 * tquad + (f.x == tmax ? 0 : f.y == tmax ? 1 : f.z == tmax ? 2 : 3);
    w0.key = static_cast<unsigned long long>(~order_of(tmax)) << 32 | static_cast<uint32_t>(idx), w0.aux = __float_as_uint(tmax);
  }
  w0 = reduce(sh, w0, cs, turn);
  int token = static_cast<int>(w0.key & 0xFFFFFFFFu);  // -1 when no value is above -inf
  const float mx = __uint_as_float(w0.aux);
  if (w0.key == ~0ull || !(temp > 0.f) || top_p <= 0.f || top_k == 1) {
    if (rank == 0 && threadIdx.x == 0) p.tokens[row] = token;
    if (cs > 1) sbd::cluster_sync_all();  // no CTA leaves while another may read its slot
    return;
  }
  // log2 of w; fminf gives the maximum itself 0 even where it is infinite (inf - inf)
  const float inv = fmaxf(kLog2e / temp, 1e-37f);  // above zero, so that -inf stays -inf
  auto z2_of = [&](float x) { return fminf((x - mx) * inv, 0.f); };
  // race key of a token with random word q: its waiting time over its rate, then its index; ~0 below min_p
  auto race = [&](float x, int idx, uint32_t q) {
    const float wx = expf(x == mx ? 0.f : (x - mx) / temp);
    if (!(wx >= min_p && wx > 0.f) && x != mx) return ~0ull;
    const float u = fminf((__uint2float_rn(q) + 0.5f) * 2.3283064365386963e-10f, 0.99999994f);
    return static_cast<unsigned long long>(__float_as_uint(-log1pf(-u) / wx)) << 32 | static_cast<uint32_t>(idx);
  };
  auto word_of = [&](int idx) {
    const uint4 r = philox(static_cast<uint32_t>(idx) >> 2, c1, k0, k1);
    const uint32_t lo = idx & 1 ? r.y : r.x, hi = idx & 1 ? r.w : r.z;
    return idx & 2 ? hi : lo;
  };
  // a value below every x with log2 w >= c, whatever the rounding on either side
  auto floor_of = [&](float c) { return mx == INFINITY ? kLargest : fmaxf(mx + (c - 0.01f) / inv - fabsf(mx) * 0x1p-21f, -kLargest); };
  // offsets of this CTA's values of at least `least` into list[cap]; sh.n counts them all.  Up to 32 values
  // per thread become a bit mask, so that a warp takes its places in the list with one atomic.
  auto collect = [&](uint16_t* list, int cap, float least, auto also) {
    for (int i0 = 0; i0 < n4; i0 += 8 * NT) {
      uint32_t hits = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = i0 + j * NT + threadIdx.x;
        if (i < n4) {
          const float4 f = *reinterpret_cast<const float4*>(xs + 4 * i);
          const float v[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            hits |= v[e] >= least ? 1u << (4 * j + e) : 0u;
            also(v[e], 4 * i + e);
          }
        }
      }
      const unsigned mine = __popc(hits);
      unsigned inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
        if (lane >= o) inc += v;
      }
      unsigned base = 0;
      if (lane == 31 && inc) base = atomicAdd(&sh.n, inc);
      base = __shfl_sync(0xFFFFFFFFu, base, 31) + inc - mine;
      if (base + mine > static_cast<unsigned>(cap)) hits = 0;  // the list will not be used
      for (; hits; hits &= hits - 1, ++base) {
        const int bit = __ffs(hits) - 1;
        list[base] = static_cast<uint16_t>(4 * (i0 + (bit >> 2) * NT + threadIdx.x) + (bit & 3));
      }
    }
    __syncthreads();
  };

  uint32_t xl = 0;  // the race is among tokens that rank before (xl, il): orderable value, index
  int il = p.v;
  if (top_k > 0 && top_k < p.v) {
    // ---- top-k: the bin of the threads' maxima that reaches k; every value in it or above is a candidate
    auto bin_of = [&](float x) { return static_cast<int>(fminf(-8.f * z2_of(x), static_cast<float>(BINS - 1))); };
    if (tquad >= 0) atomicAdd(&sh.hist[bin_of(tmax)], 1u);
    __syncthreads();
    if (cs > 1) sbd::cluster_sync_all();
    unsigned cnt = 0;
    if (threadIdx.x < BINS) {
      if (cs > 1) {
        for (int r = 0; r < cs; ++r) {
          unsigned c;
          asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(c) : "r"(sbd::mapa_shared(sbd::smem_u32(&sh.hist[threadIdx.x]), r)) : "memory");
          cnt += c;
        }
      } else {
        cnt = sh.hist[threadIdx.x];
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned c = __shfl_up_sync(0xFFFFFFFFu, cnt, o);
        if (lane >= o) cnt += c;
      }
      if (lane == 31) sh.warp[warp].count = cnt;
    }
    if (threadIdx.x == 0) sh.bin = BINS - 1;  // too few maxima: everything
    __syncthreads();
    if (threadIdx.x < BINS) {
      unsigned before = 0;
      for (int x = 0; x < warp; ++x) before += sh.warp[x].count;
      const unsigned up = __shfl_up_sync(0xFFFFFFFFu, cnt, 1);
      const unsigned k = static_cast<unsigned>(top_k);
      if (before + cnt >= k && (lane ? before + up : before) < k) sh.bin = threadIdx.x;
    }
    __syncthreads();
    const int bin = sh.bin;
    collect(sh.top.mine, MINE, bin == BINS - 1 ? -kLargest : floor_of(-0.125f * (bin + 1)), [](float, int) {});
    const unsigned mine = sh.n;  // a list that does not fit counts as too many candidates
    const unsigned total = reduce(sh, Word{0, ~0ull, 0, threadIdx.x ? 0u : mine > MINE ? SORT + 1u : mine}, cs, turn).count;
    if (total <= SORT) {
      auto key_of = [&](int i) { return static_cast<unsigned long long>(~order_of(xs[i])) << 32 | static_cast<uint32_t>(first + i); };
      const unsigned at = sh.lower;
      if (cs > 1) {
        const uint32_t dst = sbd::mapa_shared(sbd::smem_u32(sh.top.keys), 0);
        for (unsigned i = threadIdx.x; i < mine; i += NT)
          asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(dst + 8 * (at + i)), "l"(key_of(sh.top.mine[i])) : "memory");
        sbd::cluster_sync_all();
        if (rank) return;  // from here on nobody reads this CTA's memory
      } else {
        for (unsigned i = threadIdx.x; i < mine; i += NT) sh.top.keys[i] = key_of(sh.top.mine[i]);
      }
      unsigned size = 2;
      while (size < total) size *= 2;
      for (unsigned i = total + threadIdx.x; i < size; i += NT) sh.top.keys[i] = ~0ull;
      __syncthreads();
      unsigned long long* key = sh.top.keys;
      for (unsigned k = 2; k <= size; k *= 2)  // bitonic
        for (unsigned j = k / 2; j; j /= 2) {
          if (threadIdx.x < size / 2) {
            const unsigned a = 2 * j * (threadIdx.x / j) + threadIdx.x % j, b = a + j;
            const unsigned long long ka = key[a], kb = key[b];
            if ((ka > kb) == !(a & k)) key[a] = kb, key[b] = ka;
          }
          __syncthreads();
        }
      // ranks 2 t and 2 t + 1 are this thread's; the mass before each
      float x[2] = {-INFINITY, -INFINITY};
      int idx[2] = {0, 0};
      unsigned long long mass[2] = {0, 0};
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const unsigned r = 2 * threadIdx.x + e;
        if (r < total && r < static_cast<unsigned>(top_k)) {
          const uint32_t o = ~static_cast<uint32_t>(key[r] >> 32);
          x[e] = __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
          idx[e] = static_cast<int>(key[r] & 0xFFFFFFFFu);
          mass[e] = __float2ull_rn(ex2(z2_of(x[e])) * kUnit);
        }
      }
      unsigned long long inc = mass[0] + mass[1];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
        if (lane >= o) inc += v;
      }
      if (lane == 31) sh.warp[warp].sum = inc;
      __syncthreads();
      unsigned long long before = inc - mass[0] - mass[1], all = 0;
      for (int r = 0; r < NT / 32; ++r) {
        const unsigned long long v = sh.warp[r].sum;
        before += r < warp ? v : 0;
        all += v;
      }
      __syncthreads();
      const double limit = static_cast<double>(top_p) * static_cast<double>(all);
      Word best{0, ~0ull, 0, 0};
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (x[e] > -INFINITY && (top_p >= 1.f || static_cast<double>(before) < limit)) best.key = min(best.key, race(x[e], idx[e], word_of(idx[e])));
        before += mass[e];
      }
      int none = 0;
      best = reduce(sh, best, 1, none);
      if (threadIdx.x == 0) p.tokens[row] = static_cast<int>(best.key & 0xFFFFFFFFu);
      return;
    }
    // more candidates than one CTA sorts (a large k, or thousands of equal values): the largest value that at
    // least top_k values reach, bit by bit, then the index up to which those equal to it are in
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t c = xl | 1u << bit;
      unsigned cnt = 0;
      for (int i = threadIdx.x; i < n; i += NT) cnt += order_of(xs[i]) >= c;
      if (reduce(sh, Word{0, ~0ull, 0, cnt}, cs, turn).count >= static_cast<unsigned>(top_k)) xl = c;
    }
    unsigned above = 0;
    for (int i = threadIdx.x; i < n; i += NT) above += order_of(xs[i]) > xl;
    above = reduce(sh, Word{0, ~0ull, 0, above}, cs, turn).count;
    int lo = 0, hi = p.v - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      unsigned cnt = 0;
      for (int i = threadIdx.x; i < n && first + i <= mid; i += NT) cnt += order_of(xs[i]) == xl;
      if (above + reduce(sh, Word{0, ~0ull, 0, cnt}, cs, turn).count >= static_cast<unsigned>(top_k)) hi = mid;
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
  // log2 of the smallest w that can be kept (see above)
  float cut = min_p > 0.f ? __log2f(min_p) : -INFINITY;
  if (top_p < 1.f) cut = fmaxf(cut, __log2f((1.f - top_p) / static_cast<float>(p.v)));
  bool listed = false;
  Word w{0, ~0ull, 0, 0};
  if (cut > -INFINITY) {
    float sum = 0.f;
    const float least = floor_of(cut);
    if (top_p >= 1.f) collect(sh.list, LIST, least, [](float, int) {});
    else if (all) collect(sh.list, LIST, least, [&](float x, int) { sum += ex2(z2_of(x)); });
    else collect(sh.list, LIST, least, [&](float x, int i) { sum += in(x, first + i) ? ex2(z2_of(x)) : 0.f; });
    w.sum = __float2ull_rn(sum * kUnit);
    listed = sh.n <= LIST;
  }
  // The largest logit's own time bounds the winner's: it is in every race that is not empty.  A token can
  // only win when E / w <= bound; E >= u, so nearly all are out by u > bound w, two operations and an ex2 (with
  // a margin over what those are off); the logarithm, the exponential and the division are for the rest.
  const float bound = __uint_as_float(static_cast<uint32_t>(race(mx, token, word_of(token)) >> 32));
  const float reach = __log2f(bound) + 32.01f;
  auto loses = [&](float z2, uint32_t q) { return __uint2float_rn(q) > ex2(z2 + reach); };
  double mass = 0.0;
  for (int round = 0;; ++round) {
    auto run = [&](float x, int idx, uint32_t q) {
      const unsigned long long k = race(x, idx, q);
      if (k < w.key) w.key = k, w.aux = order_of(x);
    };
    if (listed) {
      const unsigned m = sh.n;
      for (unsigned i = threadIdx.x; i < m; i += NT) {
        const int at = sh.list[i], idx = first + at;
        const float x = xs[at], z = z2_of(x);
        if (!all) {
          if (!in(x, idx)) continue;
          if (round) w.sum += __float2ull_rn(ex2(z) * kUnit);
        }
        const uint32_t q = word_of(idx);
        if (!loses(z, q)) run(x, idx, q);
      }
    } else {
      float sum = 0.f;
      for (int i = threadIdx.x; i < n4; i += NT) {
        const float4 f = *reinterpret_cast<const float4*>(xs + 4 * i);
        const float v[4] = {f.x, f.y, f.z, f.w};
        float z[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] = z2_of(v[e]);
        if (!all) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            z[e] = in(v[e], first + 4 * i + e) ? z[e] : -INFINITY;
            sum += ex2(z[e]);
          }
          if (fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])) == -INFINITY) continue;
        }
        const uint4 r = philox(static_cast<uint32_t>(first / 4 + i), c1, k0, k1);
        const uint32_t q[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!loses(z[e], q[e]) && z[e] > -INFINITY) run(v[e], first + 4 * i + e, q[e]);
      }
      if (round) w.sum = __float2ull_rn(sum * kUnit);
    }
    w = reduce(sh, w, cs, turn);
    if (round && (w.key == ~0ull || static_cast<double>(w.sum) < static_cast<double>(top_p) * mass)) break;  // the last winner stands
    token = static_cast<int>(w.key & 0xFFFFFFFFu);
    if (top_p >= 1.f) break;
    if (!round) mass = static_cast<double>(w.sum);
    // next: what ranks before the winner, its mass and the winner among it
    xl = w.aux, il = token, all = false;
    w = Word{0, ~0ull, 0, 0};
  }
  if (rank == 0 && threadIdx.x == 0) p.tokens[row] = token;
  if (cs > 1) sbd::cluster_sync_all();  // no CTA leaves while another may read its slot
}

template <typename T>
int launch_sample(SampleParams& p, int rows, int cs, cudaStream_t stream) {
  const int smem = p.slice * 4;
  static bool set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SLICE * 4);
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
                         const float* min_p, int32_t* tokens, void* stream) {
  SB_CHECK_ARG(dtype == SB_F16 || dtype == SB_BF16 || dtype == SB_F32, "sb_sample: bad logits dtype");
  SB_CHECK_ARG(rows >= 0 && rows <= 65535 && vocab >= 1 && vocab <= MAX_CS * MAX_SLICE,
               "sb_sample: %d rows of %d logits (at most 65535 rows, %d logits)", rows, vocab, MAX_CS * MAX_SLICE);
  SB_CHECK_ARG(rows <= 1 || ld >= vocab, "sb_sample: ld is shorter than a row");
  if (rows == 0) return SB_OK;
  SB_CHECK_ARG(logits && seeds && pos && tokens, "sb_sample: null pointer");
  const int size = dtype == SB_F32 ? 4 : 2;
  if (!sb::aligned(logits, size)) return sb::fail(SB_ERR_ALIGN, "sb_sample: logits are not aligned to their type");
  SampleParams p{};
  p.x = logits, p.ld = ld, p.v = vocab, p.seeds = seeds, p.pos = pos, p.temperature = temperature, p.top_k = top_k;
  p.top_p = top_p, p.min_p = min_p, p.tokens = tokens;
  p.vec = sb::aligned(logits, 4 * size) && (rows == 1 || ld % 4 == 0);
  // CTAs per row: as many as leave 1024 values or more to each, up to 16
  int cs = 1;
  while (cs < MAX_CS && vocab > cs * 1024) cs *= 2;
  p.slice = ((vocab + cs - 1) / cs + 3) / 4 * 4;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == SB_F32) return launch_sample<float>(p, rows, cs, s);
  if (dtype == SB_F16) return launch_sample<__half>(p, rows, cs, s);
  return launch_sample<__nv_bfloat16>(p, rows, cs, s);
}
