// Append of new tokens to a paged key-value cache (sb_kv_append_paged): per
// head of a token's q|k|v row
//   y = x / sqrt(mean(x^2) + eps) * w            (q, k with their weights, v with none; optional)
//   (y_i, y_{i+r}) -> (y_i cos - y_{i+r} sin, y_{i+r} cos + y_i sin)   for i < r = rot / 2 (q, k)
// then q goes to its output row and k, v to page table[seq][pos / page_size],
// row pos % page_size.
//
// Every value is read and written once: bound by memory for many tokens and by
// launch latency for a few.  A lane holds eight neighbouring values (one
// 16-byte vector in 16 bits), so a head takes head_dim / 8 lanes and a warp
// holds 256 / head_dim heads (or one head of 512 as two vectors per lane); the
// rotation's partner value sits r / 8 lanes away and comes by shuffle, which
// keeps every load and store a full vector whatever rot is.
#include "paged.cuh"

namespace {

struct AppendParams {
  const void* qkv;
  int64_t ld;
  void* q_out;
  const float *q_norm, *k_norm, *cos_t, *sin_t;
  const int32_t *seq, *pos;
  sbp::Pages pages;
  int t, n_seqs, nh, nkv, rot, max_pos, v_norm, units;  // units: warp-wide pieces of a token's row
  float eps;
};

// VPT: vectors of eight per lane (2 for head_dim 512, else 1).
template <int HD, typename S, typename D>
__global__ void __launch_bounds__(256) kv_append_kernel(const AppendParams p) {
  constexpr int VPT = HD > 256 ? 2 : 1;
  constexpr int LPH = HD / (8 * VPT);  // lanes per head
  constexpr int HPW = 32 / LPH;        // heads per warp
  sbd::griddep_launch_dependents();
  sbd::griddep_wait();
  const int lane = threadIdx.x & 31;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int tok = static_cast<int>(unit / p.units);
  if (tok >= p.t) return;  // whole warps
  const int heads = p.nh + 2 * p.nkv;
  const int head = static_cast<int>(unit - static_cast<int64_t>(tok) * p.units) * HPW + lane / LPH;
  const int sub = lane % LPH;  // vector j of this lane covers values 8 * (sub + j * LPH) ...
  const bool live = head < heads;
  const int pos = p.pos[tok];
  const int seq = p.seq ? p.seq[tok] : tok;
  const bool place = pos >= 0 && pos < p.max_pos;

  float x[VPT][8];
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    if (live) {
      sbp::load8(static_cast<const S*>(p.qkv) + tok * p.ld + static_cast<int64_t>(head) * HD + 8 * (sub + j * LPH), x[j]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[j][e] = 0.f;
    }
  }
  const bool is_q = head < p.nh, is_v = head >= p.nh + p.nkv;
  const float* w = is_q ? p.q_norm : is_v ? nullptr : p.k_norm;
  if (p.q_norm || p.k_norm || p.v_norm) {  // uniform over the warp: the shuffles below meet every lane
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < VPT; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += x[j][e] * x[j][e];
#pragma unroll
    for (int o = LPH / 2; o >= 1; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
    const float rd = 1.0f / sqrtf(ss / HD + p.eps);
    if (w || (is_v && p.v_norm)) {
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        float wv[8];
        if (w) sbp::load8(w + 8 * (sub + j * LPH), wv);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[j][e] *= w ? rd * wv[e] : rd;
      }
    }
  }
  // rotation: value i < rot/2 pairs with i + rot/2, a whole number of vectors away
  const int hv = p.rot >> 4;  // vectors in half the rotated part
  float y[VPT][8];
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int vec = sub + j * LPH;
    const bool rotates = vec < 2 * hv, low = vec < hv;
    const int other = rotates ? (low ? vec + hv : vec - hv) : vec;  // the partner's vector
    const int src = (lane - sub) + other % LPH;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float o = __shfl_sync(0xFFFFFFFFu, x[0][e], src);
      if constexpr (VPT == 2) {
        const float o1 = __shfl_sync(0xFFFFFFFFu, x[1][e], src);
        o = other >= LPH ? o1 : o;
      }
      y[j][e] = o;
    }
    if (rotates && live && !is_v && place) {
      const size_t at = static_cast<size_t>(pos) * (p.rot >> 1) + 8 * (low ? vec : other);
      float c[8], s[8];
      sbp::load8(p.cos_t + at, c);
      sbp::load8(p.sin_t + at, s);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[j][e] = low ? x[j][e] * c[e] - y[j][e] * s[e] : x[j][e] * c[e] + y[j][e] * s[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[j][e] = x[j][e];
    }
  }
  if (!live) return;
  if (is_q) {
    if (!p.q_out) return;
    D* dst = static_cast<D*>(p.q_out) + (static_cast<int64_t>(tok) * p.nh + head) * HD;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      if (!place) {  // a padding token's q is zero
#pragma unroll
        for (int e = 0; e < 8; ++e) y[j][e] = 0.f;
      }
      sbp::store8(dst + 8 * (sub + j * LPH), y[j]);
    }
    return;
  }
  // a token out of place, a sequence without the page, or a page the cache does not have: nothing is written
  if (!place || seq < 0 || seq >= p.n_seqs || (pos >> p.pages.shift) >= p.pages.max_pages) return;
  const int page = p.pages.table[static_cast<int64_t>(seq) * p.pages.max_pages + (pos >> p.pages.shift)];
  if (page < 0 || page >= p.pages.n_pages) return;
  const int g = head - p.nh - (is_v ? p.nkv : 0);
  D* dst = static_cast<D*>(const_cast<void*>(is_v ? p.pages.v : p.pages.k)) + page * p.pages.page_stride +
           g * p.pages.head_stride + (pos & ((1 << p.pages.shift) - 1)) * p.pages.token_stride;
#pragma unroll
  for (int j = 0; j < VPT; ++j) sbp::store8(dst + 8 * (sub + j * LPH), y[j]);
}

template <int HD, typename S, typename D>
int launch_append(AppendParams& p, cudaStream_t stream) {
  constexpr int HPW = HD > 256 ? 1 : 256 / HD;
  const int heads = p.nh + 2 * p.nkv;
  p.units = (heads + HPW - 1) / HPW;
  const int64_t warps = static_cast<int64_t>(p.t) * p.units;
  const int64_t blocks = (warps + 7) / 8;
  SB_CHECK_ARG(blocks < (1ll << 31), "sb_kv_append_paged: too many tokens");
  cudaError_t e = sb::launch_pdl(kv_append_kernel<HD, S, D>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, p);
  if (e != cudaSuccess) return sb::cuda_fail(e, "kv_append_kernel");
  return sb::launch_status("kv_append_kernel");
}

template <typename S, typename D>
int launch_append_hd(int hd, AppendParams& p, cudaStream_t stream) {
  switch (hd) {
    case 64: return launch_append<64, S, D>(p, stream);
    case 128: return launch_append<128, S, D>(p, stream);
    case 256: return launch_append<256, S, D>(p, stream);
    default: return launch_append<512, S, D>(p, stream);
  }
}

template <typename D>
int launch_append_src(int src, int hd, AppendParams& p, cudaStream_t stream) {
  if (src == SB_F32) return launch_append_hd<float, D>(hd, p, stream);
  if (src == SB_F16) return launch_append_hd<__half, D>(hd, p, stream);
  return launch_append_hd<__nv_bfloat16, D>(hd, p, stream);
}

}  // namespace

extern "C" int sb_kv_append_paged(const sb_paged_kv* kv, const int32_t* page_table, int n_seqs, int max_pages,
                                  const void* qkv, int qkv_dtype, int64_t ld, int t, int n_heads, const int32_t* seq,
                                  const int32_t* pos, const float* q_norm, const float* k_norm, int v_norm, float eps,
                                  const float* cos_t, const float* sin_t, int rot, int max_pos, void* q_out,
                                  void* stream) {
  AppendParams p{};
  int rc = sbp::check_pages("sb_kv_append_paged", kv, page_table, max_pages, &p.pages);
  if (rc) return rc;
  SB_CHECK_ARG(qkv_dtype == SB_F16 || qkv_dtype == SB_F32 || qkv_dtype == SB_BF16, "sb_kv_append_paged: bad q|k|v dtype");
  SB_CHECK_ARG(t >= 0 && n_seqs >= 0 && n_heads >= 0 && max_pos >= 0, "sb_kv_append_paged: bad sizes");
  SB_CHECK_ARG(rot >= 0 && rot <= kv->head_dim && rot % 16 == 0, "sb_kv_append_paged: rot %d is not a multiple of 16 up to head_dim", rot);
  SB_CHECK_ARG(ld >= static_cast<int64_t>(n_heads + 2 * kv->n_kv_heads) * kv->head_dim, "sb_kv_append_paged: ld is shorter than a row");
  if (t == 0) return SB_OK;
  SB_CHECK_ARG(qkv && pos && (rot == 0 || (cos_t && sin_t)), "sb_kv_append_paged: null pointer");
  SB_CHECK_ARG(seq || t <= n_seqs, "sb_kv_append_paged: without `seq`, token i is sequence i: %d tokens, %d sequences", t, n_seqs);
  const int vec = qkv_dtype == SB_F32 ? 4 : 8;
  if (!sb::aligned(qkv, 16) || ld % vec || !sb::aligned(q_out, 16) || !sb::aligned(cos_t, 16) || !sb::aligned(sin_t, 16) ||
      !sb::aligned(q_norm, 16) || !sb::aligned(k_norm, 16))
    return sb::fail(SB_ERR_ALIGN, "sb_kv_append_paged: rows, tables and norm weights must start on 16-byte boundaries");
  p.qkv = qkv, p.ld = ld, p.q_out = q_out, p.q_norm = q_norm, p.k_norm = k_norm, p.cos_t = cos_t, p.sin_t = sin_t;
  p.seq = seq, p.pos = pos, p.t = t, p.n_seqs = n_seqs, p.nh = n_heads, p.nkv = kv->n_kv_heads, p.rot = rot;
  p.max_pos = max_pos, p.v_norm = v_norm, p.eps = eps;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return kv->dtype == SB_F16 ? launch_append_src<__half>(qkv_dtype, kv->head_dim, p, s)
                             : launch_append_src<__nv_bfloat16>(qkv_dtype, kv->head_dim, p, s);
}
