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
// memory.
#include <algorithm>

#include "paged.cuh"

namespace {

constexpr int NT = 512;       // threads per CTA
constexpr int MAX_CS = 16;    // CTAs per row
constexpr int MAX_SLICE = 51200;  // values per CTA: 200 KB

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

// What the CTAs of a cluster exchange in one step.
struct Word {
  double sum;
  unsigned long long key;
  unsigned int count, pad;
};

struct Shared {
  Word slot[3];        // this CTA's contribution, in turn
  Word warp[NT / 32];
  Word all;
};

// One counter word quadruple of Philox4x32-10.
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

// Adds sums and counts and takes the smallest key over the cluster.  `turn`
// counts the calls: three slots in turn, so that one barrier per call is
// enough (a CTA can be at most one call ahead of another's reads).
__device__ Word reduce(Shared& sh, double sum, unsigned long long key, unsigned int count, int cs, int& turn) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    const unsigned long long k = __shfl_xor_sync(0xFFFFFFFFu, key, o);
    key = k < key ? k : key;
    count += __shfl_xor_sync(0xFFFFFFFFu, count, o);
  }
  if (lane == 0) sh.warp[warp] = Word{sum, key, count, 0};
  __syncthreads();
  if (warp == 0) {
    Word w = lane < NT / 32 ? sh.warp[lane] : Word{0.0, ~0ull, 0u, 0u};
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) {
      w.sum += __shfl_xor_sync(0xFFFFFFFFu, w.sum, o);
      const unsigned long long k = __shfl_xor_sync(0xFFFFFFFFu, w.key, o);
      w.key = k < w.key ? k : w.key;
      w.count += __shfl_xor_sync(0xFFFFFFFFu, w.count, o);
    }
    if (lane == 0) (cs > 1 ? sh.slot[turn] : sh.all) = w;
  }
  if (cs > 1) {
    sbd::cluster_sync_all();
    if (warp == 0) {
      Word w{0.0, ~0ull, 0u, 0u};
      if (lane < cs) {
        const uint32_t a = sbd::mapa_shared(sbd::smem_u32(&sh.slot[turn]), lane);
        uint32_t lo, hi;
        asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(w.sum) : "r"(a) : "memory");
        asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(lo), "=r"(hi) : "r"(a + 8) : "memory");
        w.key = static_cast<unsigned long long>(hi) << 32 | lo;
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(w.count) : "r"(a + 16) : "memory");
      }
#pragma unroll
      for (int o = 8; o >= 1; o >>= 1) {  // every CTA adds in the same order
        w.sum += __shfl_xor_sync(0xFFFFFFFFu, w.sum, o);
        const unsigned long long k = __shfl_xor_sync(0xFFFFFFFFu, w.key, o);
        w.key = k < w.key ? k : w.key;
        w.count += __shfl_xor_sync(0xFFFFFFFFu, w.count, o);
      }
      if (lane == 0) sh.all = w;
    }
    turn = turn == 2 ? 0 : turn + 1;
  }
  __syncthreads();
  return sh.all;
}

template <typename T>
__global__ void __launch_bounds__(NT) sample_kernel(const SampleParams p) {
  extern __shared__ float xs[];  // this CTA's slice of the row, NaN as -inf, padded with -inf to a multiple of 4
  __shared__ Shared sh;
  const int cs = gridDim.x, rank = blockIdx.x, row = blockIdx.y;  // a cluster spans the x axis
  sbd::griddep_launch_dependents();
  sbd::griddep_wait();
  const int first = rank * p.slice, n = max(0, min(p.slice, p.v - first)), n4 = (n + 3) / 4;
  const T* src = static_cast<const T*>(p.x) + row * p.ld + first;
  int turn = 0;

  // ---- the slice into shared memory; the largest value, ties to the lowest index
  unsigned long long best = ~0ull;
  for (int i = threadIdx.x; i < n4; i += NT) {
    float v[4];
    if (p.vec && 4 * i + 4 <= n) {
      if constexpr (sizeof(T) == 4) {
        const uint4 r = sbd::ldg_nc_v4(src + 4 * i);
        v[0] = __uint_as_float(r.x), v[1] = __uint_as_float(r.y), v[2] = __uint_as_float(r.z), v[3] = __uint_as_float(r.w);
      } else {
        const uint2 r = __ldg(reinterpret_cast<const uint2*>(src + 4 * i));
        const float2 a = sbp::unpack2<T>(r.x), b = sbp::unpack2<T>(r.y);
        v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = 4 * i + e < n ? static_cast<float>(src[4 * i + e]) : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = v[e] != v[e] ? -INFINITY : v[e] + 0.f;  // -0 ranks with 0
      const unsigned long long key = static_cast<unsigned long long>(~sbd::orderable(v[e])) << 32 | static_cast<uint32_t>(first + 4 * i + e);
      best = 4 * i + e < n && key < best ? key : best;
    }
    *reinterpret_cast<float4*>(xs + 4 * i) = make_float4(v[0], v[1], v[2], v[3]);
  }
  best = reduce(sh, 0.0, best, 0, cs, turn).key;
  const uint32_t mx_bits = ~static_cast<uint32_t>(best >> 32);
  const float mx = __uint_as_float(mx_bits & 0x80000000u ? mx_bits & 0x7FFFFFFFu : ~mx_bits);
  const float temp = p.temperature ? p.temperature[row] : 1.f;
  const float top_p = p.top_p ? p.top_p[row] : 1.f, min_p = p.min_p ? p.min_p[row] : 0.f;
  const int top_k = p.top_k ? p.top_k[row] : 0;
  int token;
  if (mx == -INFINITY) {
    token = -1;  // no token may be drawn
  } else if (!(temp > 0.f) || top_p <= 0.f || top_k == 1) {
    token = static_cast<int>(best & 0xFFFFFFFFu);
  } else {
    // distance below the maximum in units of the temperature (0 for the maximum itself, whatever its size)
    auto z_of = [&](float x) { return x == mx ? 0.f : (x - mx) / temp; };
    constexpr float kLog2e = 1.4426950408889634f;
    const float inv = kLog2e / temp;
    auto w_fast = [&](float x) { return x == mx ? 1.f : ex2((x - mx) * inv); };

    // ---- top-k: the rank's last member (xk, ik); a token is in when it does not rank behind it
    uint32_t xk = 0;  // orderable bits
    int ik = p.v;
    if (top_k > 0 && top_k < p.v) {
      // the largest key that at least top_k values reach, bit by bit
      for (int bit = 31; bit >= 0; --bit) {
        const uint32_t c = xk | 1u << bit;
        unsigned int cnt = 0;
        for (int i = threadIdx.x; i < n; i += NT) cnt += sbd::orderable(xs[i]) >= c;
        if (reduce(sh, 0.0, ~0ull, cnt, cs, turn).count >= static_cast<unsigned int>(top_k)) xk = c;
      }
      unsigned int cnt = 0;
      for (int i = threadIdx.x; i < n; i += NT) cnt += sbd::orderable(xs[i]) > xk;
      const unsigned int above = reduce(sh, 0.0, ~0ull, cnt, cs, turn).count;
      // of those equal to it the lowest indices: the smallest index bound that lets enough of them in
      int lo = 0, hi = p.v - 1;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        cnt = 0;
        for (int i = threadIdx.x; i < n && first + i <= mid; i += NT) cnt += sbd::orderable(xs[i]) == xk;
        if (above + reduce(sh, 0.0, ~0ull, cnt, cs, turn).count >= static_cast<unsigned int>(top_k)) hi = mid;
        else lo = mid + 1;
      }
      ik = lo;
    }
    auto before = [](uint32_t a, int ia, uint32_t b, int ib) { return a > b || (a == b && ia < ib); };

    // ---- the race among (x, i) up to and including (xl, il) in rank, and the mass before or up to it
    uint32_t xl = xk;
    int il = ik;
    double total = 0.0;
    const uint32_t k0 = static_cast<uint32_t>(p.seeds[row]), k1 = static_cast<uint32_t>(p.seeds[row] >> 32);
    const uint32_t c1 = static_cast<uint32_t>(p.pos[row]);
    for (int round = 0;; ++round) {
      float sum = 0.f;
      unsigned long long win = ~0ull;
      for (int i = threadIdx.x; i < n4; i += NT) {
        const float4 f = *reinterpret_cast<const float4*>(xs + 4 * i);
        const float v[4] = {f.x, f.y, f.z, f.w};
        bool in[4], any = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t o = sbd::orderable(v[e]);
          const int idx = first + 4 * i + e;
          in[e] = 4 * i + e < n && (before(o, idx, xl, il) || (round == 0 && o == xl && idx == il));
          const float w = in[e] ? w_fast(v[e]) : 0.f;
          sum += w;
          in[e] = in[e] && w > 0.f;
          any |= in[e];
        }
        if (!any) continue;
        const uint4 r = philox(static_cast<uint32_t>(first / 4 + i), c1, k0, k1);
        const uint32_t word[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (!in[e]) continue;
          const float w = expf(z_of(v[e]));
          if (!(w >= min_p) && v[e] != mx) continue;  // min-p never drops the maximum
          const float u = fminf((__uint2float_rn(word[e]) + 0.5f) * 2.3283064365386963e-10f, 0.99999994f);
          const float t = -log1pf(-u) / w;
          const unsigned long long key = static_cast<unsigned long long>(__float_as_uint(t)) << 32 | static_cast<uint32_t>(first + 4 * i + e);
          win = key < win ? key : win;
        }
      }
      const Word all = reduce(sh, static_cast<double>(sum), win, 0, cs, turn);
      if (round == 0) {
        total = all.sum;
      } else if (all.sum < static_cast<double>(top_p) * total || all.key == ~0ull) {
        token = il;  // the mass before the last winner is below p of the total: it stands
        break;
      }
      // the winner of this round becomes the bound of the next
      il = static_cast<int>(all.key & 0xFFFFFFFFu);
      if (top_p >= 1.f) {
        token = il;
        break;
      }
      // its value, from the CTA that holds it
      {
        const bool mine = threadIdx.x == 0 && il >= first && il < first + n;
        const unsigned long long bits = mine ? sbd::orderable(xs[il - first]) : ~0ull;
        xl = static_cast<uint32_t>(reduce(sh, 0.0, bits, 0, cs, turn).key);
      }
    }
  }
  if (rank == 0 && threadIdx.x == 0) p.tokens[row] = token;
  if (cs > 1) sbd::cluster_sync_all();  // no CTA leaves while another may read its slots
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
