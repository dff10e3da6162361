// Append of new tokens to a paged key-value cache (sb_kv_append_paged): per
// head of a token's q|k|v row
//   y = x / sqrt(mean(x^2) + eps) * w            (q, k with their weights, v with none; optional)
//   (y_i, y_{i+r}) -> (y_i cos - y_{i+r} sin, y_{i+r} cos + y_i sin)   for i < r = rot / 2 (q, k)
// then q goes to its output row and k, v to page table[seq][pos / page_size],
// row pos % page_size.
//
// Every value is read and written once: bound by memory for many tokens and by
// launch latency for a few.  A lane holds the two vectors of eight values that the
// rotation pairs, v and v + r / 8 (past the rotated part any two), so a pair
// shares its angles, nothing is exchanged between lanes but the norm's sum, and
// every load and store is a full vector whatever rot is.  A head takes
// head_dim / 16 lanes, a warp holds 512 / head_dim heads.  Measured in a graph of such
// calls: 16133 packed tokens of 48 x 128 bf16 values 74 us into pages laid out token by
// token, 78 head by head (397 MB, 5.4 and 5.1 TB/s, 0.84 and 0.79 of a copy's rate), 89
// with k_out and v_out too (463 MB); one token 2.2 us, 256 tokens 3.0.
#include "paged.cuh"

namespace {

struct AppendParams {
  const void* qkv;
  int64_t ld;
  void *q_out, *k_out, *v_out;
  const float *q_norm, *k_norm, *cos_t, *sin_t;
  const int32_t *seq, *pos;
  sbp::Pages pages;
  int t, n_seqs, nh, nkv, rot, max_pos, v_norm, units;  // units: warps per token
  float eps;
};

// R: pieces of 512 values of one token per warp, whose loads are all in flight at
// once and share the angles and the page.
template <int HD, int R, typename S, typename D>
__global__ void __launch_bounds__(256, 3) kv_append_kernel(const AppendParams p) {
  constexpr int LPH = HD / 16;   // lanes per head
  constexpr int HPW = 32 / LPH;  // heads per piece
  sbd::griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const unsigned warp = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int tok = static_cast<int>(warp / static_cast<unsigned>(p.units));
  const int heads = p.nh + 2 * p.nkv;
  const int head0 = (static_cast<int>(warp) - tok * p.units) * R * HPW + lane / LPH;  // piece r: head0 + r * HPW
  // this lane's pair of vectors: i and i + rot/2 for i < rot/2; past rot the halves of the rest
  const int sub = lane % LPH, hv = p.rot >> 4;
  const bool turns = sub < hv;
  const int at0 = 8 * (turns ? sub : sub + hv), at1 = 8 * (turns ? sub + hv : sub + LPH);
  sbd::griddep_wait();
  if (tok >= p.t) return;  // whole warps

  const S* src = static_cast<const S*>(p.qkv) + tok * p.ld;
  float x[R][2][8];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int head = min(head0 + r * HPW, heads - 1);  // a head past the last loads it again and stores nothing
    sbp::load8(src + head * HD + at0, x[r][0]);
    sbp::load8(src + head * HD + at1, x[r][1]);
  }
  const int pos = p.pos[tok];
  const int seq = p.seq ? p.seq[tok] : tok;
  // where a head's packed row goes: q, and k and v when they are wanted; null: nowhere
  auto out_row = [&](int head) -> D* {
    if (head < p.nh) return p.q_out ? static_cast<D*>(p.q_out) + (static_cast<int64_t>(tok) * p.nh + head) * HD : nullptr;
    const bool v = head >= p.nh + p.nkv;
    D* base = static_cast<D*>(v ? p.v_out : p.k_out);
    return base && head < heads ? base + (static_cast<int64_t>(tok) * p.nkv + head - p.nh - (v ? p.nkv : 0)) * HD : nullptr;
  };
  if (pos < 0 || pos >= p.max_pos) {  // padding (the whole warp): zero rows, nothing is appended
    const float zero[8] = {};
#pragma unroll
    for (int r = 0; r < R; ++r) {
      D* dst = out_row(head0 + r * HPW);
      if (!dst) continue;
      sbp::store8(dst + at0, zero);
      sbp::store8(dst + at1, zero);
    }
    return;
  }
  // the page of the token, -1 for a sequence without it or a page the cache does not have
  int page = -1;
  if (seq >= 0 && seq < p.n_seqs && (pos >> p.pages.shift) < p.pages.max_pages)
    page = p.pages.table[static_cast<int64_t>(seq) * p.pages.max_pages + (pos >> p.pages.shift)];
  if (page >= p.pages.n_pages) page = -1;
  float c[8], sn[8];
  if (turns) {
    const size_t at = static_cast<size_t>(pos) * (p.rot >> 1) + at0;
    sbp::load8(p.cos_t + at, c);
    sbp::load8(p.sin_t + at, sn);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = 1.f, sn[e] = 0.f;
  }
  const int64_t kv_row = page * p.pages.page_stride + (pos & ((1 << p.pages.shift) - 1)) * p.pages.token_stride;
  const bool norms = p.q_norm || p.k_norm || p.v_norm;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int head = head0 + r * HPW;
    const bool is_q = head < p.nh, is_v = head >= p.nh + p.nkv;
    if (norms) {  // uniform over the warp: the shuffles meet every lane
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += x[r][0][e] * x[r][0][e] + x[r][1][e] * x[r][1][e];
#pragma unroll
      for (int o = LPH / 2; o >= 1; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
      const float rd = 1.0f / sqrtf(ss / HD + p.eps);
      const float* w = is_q ? p.q_norm : is_v ? nullptr : p.k_norm;
      if (w) {
        float w0[8], w1[8];
        sbp::load8(w + at0, w0);
        sbp::load8(w + at1, w1);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[r][0][e] *= rd * w0[e], x[r][1][e] *= rd * w1[e];
      } else if (is_v && p.v_norm) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[r][0][e] *= rd, x[r][1][e] *= rd;
      }
    }
    if (!is_v) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = x[r][0][e], b = x[r][1][e];
        x[r][0][e] = a * c[e] - b * sn[e];
        x[r][1][e] = b * c[e] + a * sn[e];
      }
    }
    D* dst = out_row(head);
    if (dst) {
      sbp::store8(dst + at0, x[r][0]);
      sbp::store8(dst + at1, x[r][1]);
    }
    if (is_q || head >= heads || page < 0) continue;  // a key or value without a page is not appended
    dst = static_cast<D*>(const_cast<void*>(is_v ? p.pages.v : p.pages.k)) + kv_row +
          (head - p.nh - (is_v ? p.nkv : 0)) * p.pages.head_stride;
    sbp::store8(dst + at0, x[r][0]);
    sbp::store8(dst + at1, x[r][1]);
  }
}

template <int HD, int R, typename S, typename D>
int launch_append_r(AppendParams& p, int pieces, cudaStream_t stream) {
  p.units = (pieces + R - 1) / R;
  const int64_t blocks = (static_cast<int64_t>(p.t) * p.units + 7) / 8;
  SB_CHECK_ARG(blocks < (1ll << 28), "sb_kv_append_paged: too many tokens");
  cudaError_t e = sb::launch_pdl(kv_append_kernel<HD, R, S, D>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, p);
  if (e != cudaSuccess) return sb::cuda_fail(e, "kv_append_kernel");
  return sb::launch_status("kv_append_kernel");
}

// A piece per warp while they fit two full waves (the shortest chain of loads);
// beyond that three, which keep more bytes in flight.  16133 tokens of 48 heads of
// 128 in bf16, pages laid out head by head: 115 us with one piece, 87 with two, 78
// with three, 84 with four, whose registers leave one block less per SM.
template <int HD, typename S, typename D>
int launch_append(AppendParams& p, cudaStream_t stream) {
  constexpr int HPW = 512 / HD;
  const int pieces = (p.nh + 2 * p.nkv + HPW - 1) / HPW;
  if (static_cast<int64_t>(p.t) * pieces <= 64ll * 2 * sb::num_sms()) return launch_append_r<HD, 1, S, D>(p, pieces, stream);
  return launch_append_r<HD, 3, S, D>(p, pieces, stream);
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
                                  void* k_out, void* v_out, void* stream) {
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
  if (!sb::aligned(qkv, 16) || ld % vec || !sb::aligned(q_out, 16) || !sb::aligned(k_out, 16) ||
      !sb::aligned(v_out, 16) || !sb::aligned(cos_t, 16) || !sb::aligned(sin_t, 16) ||
      !sb::aligned(q_norm, 16) || !sb::aligned(k_norm, 16))
    return sb::fail(SB_ERR_ALIGN, "sb_kv_append_paged: rows, tables and norm weights must start on 16-byte boundaries");
  p.qkv = qkv, p.ld = ld, p.q_out = q_out, p.k_out = k_out, p.v_out = v_out, p.q_norm = q_norm, p.k_norm = k_norm, p.cos_t = cos_t, p.sin_t = sin_t;
  p.seq = seq, p.pos = pos, p.t = t, p.n_seqs = n_seqs, p.nh = n_heads, p.nkv = kv->n_kv_heads, p.rot = rot;
  p.max_pos = max_pos, p.v_norm = v_norm, p.eps = eps;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return kv->dtype == SB_F16 ? launch_append_src<__half>(qkv_dtype, kv->head_dim, p, s)
                             : launch_append_src<__nv_bfloat16>(qkv_dtype, kv->head_dim, p, s);
}
