// Attention over the paged 4-bit cache.
#include "kernels.h"
#include "paged_common.cuh"

namespace cutb {
namespace {

constexpr uint32_t PT_THREADS = 128;

// One block per row and query head: its warps take turns over the keys, each with a running maximum and sum, and meet at the end.
template <typename T, int N>  // N: groups of 32 elements of a head
__global__ void __launch_bounds__(PT_THREADS) paged_attention_kernel(const __grid_constant__ cutb_paged_desc d) {
  __shared__ float acc_s[4][32 * N], m_s[4], l_s[4];
  pdl_enter();
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32, row = blockIdx.x, h = blockIdx.y, dp = pg_pad(d.head_dim), groups = dp / 32;
  const uint32_t s = paged_seq_of(d, row);
  if (s >= d.n_seqs) return;
  const PagedSeq sq = paged_seq(d, s);
  if (sq.bad && threadIdx.x == 0) paged_report(d.status, CUTB_ERR_INVALID);
  if (row - sq.row0 >= sq.rows) return;
  const uint32_t pos = sq.len - sq.rows + (row - sq.row0), kvh = h / (d.n_heads / d.n_kv_heads);
  const uint32_t first = d.window && pos + 1 > d.window ? pos + 1 - d.window : 0;
  const T *q = reinterpret_cast<const T *>(d.q) + row * d.ldq + (uint64_t)h * d.head_dim;
  float x[N], acc[N], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) x[j] = 32 * j + lane < d.head_dim ? to_f(q[32 * j + lane]) * d.scale : 0.f, acc[j] = 0.f;
  for (uint32_t key = first + warp; key <= pos; key += 4) {
    const uint32_t page = __ldg(d.tables + sq.slot * d.ld_table + key / d.page_tokens), t = key % PG_UNIT;
    if (page >= d.n_pages) {
      if (lane == 0) paged_report(d.status, CUTB_ERR_INVALID);
      continue;
    }
    const uint8_t *unit = reinterpret_cast<const uint8_t *>(d.pages) + (uint64_t)page * d.page_bytes +
                          ((uint64_t)kvh * (d.page_tokens / PG_UNIT) + key % d.page_tokens / PG_UNIT) * pg_unit_bytes(dp);
    float score = 0.f, v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const __half2 sc = *reinterpret_cast<const __half2 *>(unit + pg_key_scales_at(dp) + 4 * (t * groups + j));
      const uint32_t w = reinterpret_cast<const uint32_t *>(unit)[pg_key_word(dp, t, j, lane / 8)] >> pg_key_bit(lane % 8) & 15u;
      score = fmaf(x[j], __half2float(__hfma(__uint2half_rn(w), __low2half(sc), __high2half(sc))), score);
      const __half *sv = reinterpret_cast<const __half *>(unit + pg_value_scales_at(dp)) + 8 * (j * 4 + t / 4) + t % 4;
      const uint32_t u = unit[pg_values_at(dp) + pg_value_byte(t, (32 * j + lane) / 16, lane % 8)] >> (lane & 8 ? 4 : 0) & 15u;
      v[j] = __half2float(__hfma(__uint2half_rn(u), sv[0], sv[4]));
    }
#pragma unroll
    for (int o = 16; o; o /= 2) score += __shfl_xor_sync(0xffffffffu, score, o);
    const float mn = fmaxf(m, score), f = expf(m - mn), p = expf(score - mn);
    m = mn, l = fmaf(l, f, p);
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = fmaf(acc[j], f, p * v[j]);
  }
#pragma unroll
  for (int j = 0; j < N; ++j) acc_s[warp][32 * j + lane] = acc[j];
  if (lane == 0) m_s[warp] = m, l_s[warp] = l;
  __syncthreads();
  const float top = fmaxf(fmaxf(m_s[0], m_s[1]), fmaxf(m_s[2], m_s[3]));
  float f[4], sum = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) f[w] = m_s[w] == -INFINITY ? 0.f : expf(m_s[w] - top), sum = fmaf(f[w], l_s[w], sum);
  T *out = reinterpret_cast<T *>(d.out) + row * d.ldo + (uint64_t)h * d.head_dim;
  for (uint32_t i = threadIdx.x; i < d.head_dim; i += PT_THREADS) {
    float y = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) y = fmaf(f[w], acc_s[w][i], y);
    out[i] = from_f<T>(sum > 0.f ? y / sum : 0.f);
  }
}

}  // namespace

uint64_t paged_attention_workspace(const cutb_paged_desc &) { return 0; }

int paged_attention_launch(const cutb_paged_desc &d, cudaStream_t stream) {
  return paged_with_type(d.dtype, [&](auto t) {
    using T = decltype(t);
    const dim3 grid(d.n_tokens, d.n_heads);
    switch (pg_pad(d.head_dim) / 64) {
      case 1: CUTB_CUDA_TRY(launch_pdl(paged_attention_kernel<T, 2>, grid, dim3(PT_THREADS), 0, stream, d)); break;
      case 2: CUTB_CUDA_TRY(launch_pdl(paged_attention_kernel<T, 4>, grid, dim3(PT_THREADS), 0, stream, d)); break;
      case 3: CUTB_CUDA_TRY(launch_pdl(paged_attention_kernel<T, 6>, grid, dim3(PT_THREADS), 0, stream, d)); break;
      default: CUTB_CUDA_TRY(launch_pdl(paged_attention_kernel<T, 8>, grid, dim3(PT_THREADS), 0, stream, d)); break;
    }
    return (int)CUTB_OK;
  });
}

}  // namespace cutb
