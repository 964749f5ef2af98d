// Attention over the paged 4-bit cache for a few rows of each sequence (single tokens, above all).
//
// scores^T = K Q^T and out^T = V^T P^T on warp MMAs (m16n8k16): the 16 tokens of a unit are the MMA's rows (then its depth), the query
// rows its 8 columns, so that keys and values are the A operands.  The units are laid out for that: a lane's words, nibbles turned into fp16 pairs
// in registers, are its A fragments, and nothing goes through shared memory twice.  P^T comes from the scores' accumulators by movmatrix.
// 16-bit rows take 8 columns.  fp32 rows enter as two fp16 terms: a tile of 8 columns has the high parts of four rows and then their low
// parts, and so have the weights (22 bits of each; the products are exact, the sums fp32).  Queries are scaled by a power of two so
// that the largest element is in [1, 2), weights by 2^15: fp16 holds 2^-24 of the former and 2^-39 of the largest weight.
//
// Bound by HBM: 2560 bytes of a 128-element unit are 4096 elements, and about 290 warp instructions.  Units are copied whole by bulk
// copies, each warp through a ring of its own, so that a block has up to 80 KB in flight and warps meet only at the ends.
// The units of all sequences and KV heads in a row are shared out evenly over the blocks.  Where a block's part begins or ends inside
// a KV head's units, its maxima, sums and values go to the workspace, and a second kernel joins them in their order.
#include "kernels.h"
#include "paged_common.cuh"

namespace cutb {
namespace {

constexpr uint32_t PT_WARPS = 8, PT_THREADS = 32 * PT_WARPS;

__host__ __device__ constexpr uint32_t pt_stages(uint32_t dp) { return dp == 64 ? 8 : dp == 128 ? 4 : dp == 192 ? 3 : 2; }
__host__ __device__ constexpr uint32_t pt_ring_bytes(uint32_t dp) { return PT_WARPS * pt_stages(dp) * pg_unit_bytes(dp); }

struct PtSeq {
  uint32_t slot, len, row0, rows;
};
// The shares: block b works on the units total b / shares .. total (b + 1) / shares of all, at least PT_WARPS each.
__device__ __forceinline__ uint32_t pt_shares(uint64_t total, uint32_t blocks) {
  const uint64_t most = (total + PT_WARPS - 1) / PT_WARPS;
  return (uint32_t)(most < blocks ? most : blocks);
}
__device__ __forceinline__ uint64_t pt_from(uint64_t total, uint32_t shares, uint32_t b) { return total * b / shares; }
// first unit that a sequence's rows see, and how many there are up to the last one
__device__ __forceinline__ void pt_units(const cutb_paged_desc &d, uint32_t len, uint32_t rows, uint32_t &first, uint32_t &n) {
  const uint32_t oldest = len - rows;  // position of the first row
  first = d.window && oldest + 1 > d.window ? (oldest + 1 - d.window) / PG_UNIT : 0;
  n = (len + PG_UNIT - 1) / PG_UNIT - first;
}

struct PtPlan {
  uint32_t rows;       // query rows of an item
  uint32_t blocks;     // at most
  uint64_t *prefix;    // workspace: units (times rows' chunks) of the sequences before
  float *part;         // workspace: [block][2][rows][dp + 2]
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float pt_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_half(float a, float b) { return h2_as_u32(__floats2half2_rn(a, b)); }

template <typename T, int DP, int NT>
__global__ void __launch_bounds__(PT_THREADS, DP * NT <= 128 ? 2 : 1) paged_attention_kernel(const __grid_constant__ cutb_paged_desc d, const PtPlan plan) {
  constexpr bool SPLIT = sizeof(T) == 4;
  constexpr uint32_t G = DP / 32, MT = DP / 16, S = pt_stages(DP), UB = pg_unit_bytes(DP), TILE = SPLIT ? 4 : 8, RI = TILE * NT, LD = DP + 4;
  extern __shared__ __align__(128) uint8_t pt_smem[];
  uint64_t *prefix = reinterpret_cast<uint64_t *>(pt_smem + pt_ring_bytes(DP));
  PtSeq *seqs = reinterpret_cast<PtSeq *>(prefix + d.n_seqs + 1);
  __shared__ __align__(8) uint64_t bars[PT_WARPS * S];
  __shared__ float m_s[PT_WARPS][8 * NT], l_s[PT_WARPS][8 * NT];
  __shared__ uint64_t sums[PT_WARPS], carry_s;
  const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid & 31, g = lane / 4, t = lane % 4;
  const uint32_t bar = smem_u32(bars) + warp * S * 8, ring = smem_u32(pt_smem) + warp * S * UB;
  if (lane == 0) {
    for (uint32_t i = 0; i < S; ++i) mbar_init(bar + 8 * i, 1);
    fence_mbar_init();
  }
  pdl_enter();
  const uint32_t rep = d.n_heads / d.n_kv_heads;
  auto chunks_of = [&](uint32_t rows) { return (rows * rep + RI - 1) / RI; };
  // units of the sequences before each
  if (tid == 0) carry_s = 0;
  for (uint32_t s0 = 0; s0 < d.n_seqs; s0 += PT_THREADS) {
    const uint32_t s = s0 + tid;
    uint64_t x = 0;
    if (s < d.n_seqs) {
      const PagedSeq q = paged_seq(d, s);
      if (q.bad && blockIdx.x == 0) paged_report(d.status, CUTB_ERR_INVALID);
      seqs[s] = PtSeq{q.slot, q.len, q.row0, q.rows};
      uint32_t first, n = 0;
      if (q.rows) pt_units(d, q.len, q.rows, first, n);
      x = (uint64_t)n * chunks_of(q.rows);
    }
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const uint64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) sums[warp] = x;
    __syncthreads();
    for (uint32_t w = 0; w < warp; ++w) x += sums[w];
    x += carry_s;
    if (s < d.n_seqs) prefix[s + 1] = x;
    __syncthreads();
    if (tid == PT_THREADS - 1) carry_s = x;
  }
  if (tid == 0) prefix[0] = 0;
  __syncthreads();
  if (blockIdx.x == 0)
    for (uint32_t s = tid; s <= d.n_seqs; s += PT_THREADS) plan.prefix[s] = prefix[s];
  const uint64_t total = prefix[d.n_seqs] * d.n_kv_heads;
  const uint32_t shares = pt_shares(total, plan.blocks);
  if (blockIdx.x >= shares) return;
  const uint64_t begin = pt_from(total, shares, blockIdx.x), end = pt_from(total, shares, blockIdx.x + 1);
  uint32_t s = 0;
  for (uint32_t hi = d.n_seqs; s + 1 < hi;) {  // the sequence that unit `begin` belongs to
    const uint32_t mid = (s + hi) / 2;
    if (prefix[mid] * d.n_kv_heads <= begin) s = mid;
    else hi = mid;
  }
  uint32_t stage = 0, phase = 0;
  bool dead = false;
  for (uint64_t x = begin; x < end;) {
    while (prefix[s + 1] * d.n_kv_heads <= x) ++s;  // (sequences without units are passed over)
    const PtSeq sq = seqs[s];
    uint32_t first, n;
    pt_units(d, sq.len, sq.rows, first, n);
    const uint64_t local = x - prefix[s] * d.n_kv_heads;
    const uint32_t chunks = chunks_of(sq.rows), item = (uint32_t)(local / n), ua = (uint32_t)(local % n), kvh = item / chunks, row_a = item % chunks * RI;
    const uint32_t ub = (uint32_t)min((uint64_t)n, ua + (end - x)), rows = min(RI, sq.rows * rep - row_a);
    const uint32_t *table = d.tables + sq.slot * d.ld_table;
    const uint8_t *base = reinterpret_cast<const uint8_t *>(d.pages) + (uint64_t)kvh * (d.page_tokens / PG_UNIT) * UB;
    // units of this warp: ua + warp, + 8, ...; the pages of 32 of them at a time are in the lanes
    const uint32_t mine = ub > ua + warp ? (ub - ua - warp + PT_WARPS - 1) / PT_WARPS : 0;
    auto unit_at = [&](uint32_t i) { return first + ua + warp + PT_WARPS * i; };
    uint32_t entry = 0;
    auto look_up = [&](uint32_t i) {
      entry = CUTB_NO_PAGE;
      if (i + lane < mine) entry = __ldg(table + unit_at(i + lane) * PG_UNIT / d.page_tokens);
    };
    auto issue = [&](uint32_t i, uint32_t to) {  // every lane; pages that do not exist arrive without bytes
      if (i % 32 == 0) look_up(i);
      const uint32_t page = __shfl_sync(0xffffffffu, entry, i % 32);
      if (lane == 0) {
        if (page < d.n_pages) {
          mbar_arrive_expect_tx(bar + 8 * to, UB);
          bulk_g2s(ring + to * UB, base + (uint64_t)page * d.page_bytes + unit_at(i) * PG_UNIT % d.page_tokens / PG_UNIT * UB, UB, bar + 8 * to);
        } else {
          mbar_arrive(bar + 8 * to);
          paged_report(d.status, CUTB_ERR_INVALID);
        }
      }
      return page < d.n_pages;
    };
    uint32_t there = 0;  // bit of a stage: its page exists
    uint32_t issued = 0;
    if (!dead)
      for (; issued < min(mine, S); ++issued) {
        const uint32_t to = (stage + issued) % S;
        there = issue(issued, to) ? there | 1u << to : there & ~(1u << to);
      }
    // this lane's columns: query row of column g (fragments) and of columns 2 t, 2 t + 1 (scores)
    uint32_t qf[NT][2 * G][2];
    float mult[NT][2];
    uint32_t at[NT][2];  // positions + 1; 0: no such row
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const uint32_t r = row_a + nt * TILE + (SPLIT ? g & 3 : g);
      const bool live = r < row_a + rows;
      const uint32_t tok = r / rep, hq = kvh * rep + r % rep;
      const T *src = reinterpret_cast<const T *>(d.q) + (uint64_t)(sq.row0 + (live ? tok : 0)) * d.ldq + (uint64_t)(live ? hq : 0) * d.head_dim;
      float v[G][8], top = 0.f;
#pragma unroll
      for (int j = 0; j < G; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t i = 32 * j + 8 * t + e;
          v[j][e] = live && i < d.head_dim ? to_f(src[i]) : 0.f;
          top = fmaxf(top, fabsf(v[j][e]));
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^-e of the largest element (of numbers too small or not finite: none)
      const uint32_t ex = __float_as_uint(top) >> 23;
      const float down = ex > 0 && ex < 254 ? __uint_as_float((254 - ex) << 23) : 1.f, up = ex > 0 && ex < 254 ? __uint_as_float(ex << 23) : 1.f;
#pragma unroll
      for (int j = 0; j < G; ++j)
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const float a = v[j][e] * down, b = v[j][e + 1] * down;
          uint32_t w = pack_half(a, b);
          if (SPLIT) {
            const float2 h = __half22float2(u32_as_h2(w));
            const uint32_t low = pack_half(a - h.x, b - h.y);
            w = g < 4 ? w : low;
          }
          qf[nt][2 * j + e / 4][e / 2 % 2] = w;
        }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t c = 2 * t + k, cr = SPLIT ? c & 3 : c, rr = row_a + nt * TILE + cr;
        mult[nt][k] = __shfl_sync(0xffffffffu, up, cr * 4) * d.scale * 1.4426950408889634f;
        at[nt][k] = cr < TILE && nt * TILE + cr < rows ? sq.len - sq.rows + rr / rep + 1 : 0;
      }
    }
    const uint32_t pos_min = sq.len - sq.rows + row_a / rep, pos_max = sq.len - sq.rows + (row_a + rows - 1) / rep;
    float m[NT][2], l[NT][2], o[NT][MT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY, l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int i = 0; i < MT; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
    }
    const uint32_t tk = 4 * (g / 2) + (g & 1);  // the token of MMA row g; row g + 8 is the second after it
    for (uint32_t i = 0; i < mine && !dead; ++i) {
      if (!warp_wait(bar + 8 * stage, phase)) {
        dead = true;
        break;
      }
      const uint8_t *u = pt_smem + (ring - smem_u32(pt_smem)) + stage * UB;
      const bool exists = there >> stage & 1;
      const uint32_t key0 = unit_at(i) * PG_UNIT;
      const bool edge = !exists || key0 + PG_UNIT - 1 > pos_min || (d.window && pos_max >= key0 && pos_max - key0 >= d.window);
      float sc[NT][4];
      {
        float acc[NT][2][4] = {};
        uint32_t w0[G], w1[G], s0[G], s1[G];
        const uint32_t *k0 = reinterpret_cast<const uint32_t *>(u) + tk * (DP / 8), *k1 = k0 + 2 * (DP / 8);
        if constexpr (DP % 128 == 0) {
#pragma unroll
          for (int j = 0; j < G; j += 4) {
            *reinterpret_cast<uint4 *>(w0 + j) = *reinterpret_cast<const uint4 *>(k0 + 4 * j + 4 * t);
            *reinterpret_cast<uint4 *>(w1 + j) = *reinterpret_cast<const uint4 *>(k1 + 4 * j + 4 * t);
          }
        } else {
#pragma unroll
          for (int j = 0; j < G; j += 2) {
            *reinterpret_cast<uint2 *>(w0 + j) = *reinterpret_cast<const uint2 *>(k0 + 4 * j + 2 * t);
            *reinterpret_cast<uint2 *>(w1 + j) = *reinterpret_cast<const uint2 *>(k1 + 4 * j + 2 * t);
          }
        }
        const uint32_t *ks = reinterpret_cast<const uint32_t *>(u + pg_key_scales_at(DP)) + tk * G;
#pragma unroll
        for (int j = 0; j < G; j += 2) {
          *reinterpret_cast<uint2 *>(s0 + j) = *reinterpret_cast<const uint2 *>(ks + j);
          *reinterpret_cast<uint2 *>(s1 + j) = *reinterpret_cast<const uint2 *>(ks + 2 * G + j);
        }
#pragma unroll
        for (int j = 0; j < G; ++j) {
          __half2 a[4], b[4];
          pg_quants(w0[j], a);
          pg_quants(w1[j], b);
          const __half2 x0 = u32_as_h2(s0[j]), x1 = u32_as_h2(s1[j]), d0 = __low2half2(x0), m0 = __high2half2(x0), d1 = __low2half2(x1), m1 = __high2half2(x1);
#pragma unroll
          for (int e = 0; e < 4; ++e) a[e] = __hfma2(a[e], d0, m0), b[e] = __hfma2(b[e], d1, m1);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_f16(acc[nt][0], h2_as_u32(a[0]), h2_as_u32(b[0]), h2_as_u32(a[1]), h2_as_u32(b[1]), qf[nt][2 * j][0], qf[nt][2 * j][1]);
            mma_f16(acc[nt][1], h2_as_u32(a[2]), h2_as_u32(b[2]), h2_as_u32(a[3]), h2_as_u32(b[3]), qf[nt][2 * j + 1][0], qf[nt][2 * j + 1][1]);
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float v = acc[nt][0][c] + acc[nt][1][c];
            if (SPLIT) v += __shfl_xor_sync(0xffffffffu, v, 2);
            sc[nt][c] = v * mult[nt][c & 1];
          }
      }
      if (edge) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t key = key0 + tk + (c & 2), p1 = at[nt][c & 1];
            if (!exists || key >= p1 || (d.window && p1 - key > d.window)) sc[nt][c] = -INFINITY;
          }
      }
      uint32_t bf[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float f[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float mx = fmaxf(sc[nt][k], sc[nt][k + 2]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          const float mn = fmaxf(m[nt][k], mx);
          f[k] = m[nt][k] == mn ? 1.f : pt_exp2(m[nt][k] - mn);
          m[nt][k] = mn;
        }
        if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {
          l[nt][0] *= f[0], l[nt][1] *= f[1];
#pragma unroll
          for (int i2 = 0; i2 < MT; ++i2) o[nt][i2][0] *= f[0], o[nt][i2][1] *= f[1], o[nt][i2][2] *= f[0], o[nt][i2][3] *= f[1];
        }
        float p[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float mm = m[nt][c & 1];
          p[c] = pt_exp2(sc[nt][c] - (mm == -INFINITY ? 0.f : mm - 15.f));
        }
        l[nt][0] += p[0] + p[2], l[nt][1] += p[1] + p[3];
        uint32_t h0 = pack_half(p[0], p[1]), h1 = pack_half(p[2], p[3]);
        if (SPLIT && t >= 2) {
          const float2 a = __half22float2(u32_as_h2(h0)), b = __half22float2(u32_as_h2(h1));
          h0 = pack_half(p[0] - a.x, p[1] - a.y), h1 = pack_half(p[2] - b.x, p[3] - b.y);
        }
        __syncwarp();
        bf[nt][0] = transposed(h0), bf[nt][1] = transposed(h1);
      }
      {
        const uint4 *vw = reinterpret_cast<const uint4 *>(u + pg_values_at(DP)) + lane;
        const uint4 *vs = reinterpret_cast<const uint4 *>(u + pg_value_scales_at(DP)) + t;
        const bool tail = !exists || key0 + PG_UNIT > sq.len;  // what is past the sequence may be anything
#pragma unroll
        for (int q4 = 0; q4 < MT / 4; ++q4) {
          const uint4 w = vw[32 * q4];
          const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint4 x = vs[4 * (2 * q4 + half)];
            if (tail) {
              const uint32_t left = !exists || sq.len <= key0 + 4 * t ? 0 : min(4u, sq.len - key0 - 4 * t);
              const uint32_t m01 = left >= 2 ? 0xffffffffu : left ? 0xffffu : 0u, m23 = left >= 4 ? 0xffffffffu : left == 3 ? 0xffffu : 0u;
              x.x &= m01, x.y &= m23, x.z &= m01, x.w &= m23;
            }
            const __half2 dA = u32_as_h2(x.x), dB = u32_as_h2(x.y), mA = u32_as_h2(x.z), mB = u32_as_h2(x.w);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              __half2 a[4];
              pg_quants(ws[2 * half + k], a);
              a[0] = __hfma2(a[0], dA, mA), a[1] = __hfma2(a[1], dA, mA), a[2] = __hfma2(a[2], dB, mB), a[3] = __hfma2(a[3], dB, mB);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma_f16(o[nt][4 * q4 + 2 * half + k], h2_as_u32(a[0]), h2_as_u32(a[1]), h2_as_u32(a[2]), h2_as_u32(a[3]), bf[nt][0], bf[nt][1]);
            }
          }
        }
      }
      __syncwarp();  // the unit is read
      if (issued < mine) {
        there = issue(issued, stage) ? there | 1u << stage : there & ~(1u << stage);
        ++issued;
      }
      if (++stage == S) stage = 0, phase ^= 1u;
    }
    if (dead) {
      for (uint32_t i = 0; i < S; ++i) mbar_drain(bar + 8 * i, i < stage ? phase ^ 1u : phase);  // nothing may land in a block that has ended
      if (lane == 0) paged_report(d.status, CUTB_ERR_TIMEOUT);
    }
    // the warps' parts meet: maxima and sums, then the values under the common maximum
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float v = l[nt][k];
        v += __shfl_xor_sync(0xffffffffu, v, 4), v += __shfl_xor_sync(0xffffffffu, v, 8), v += __shfl_xor_sync(0xffffffffu, v, 16);
        if (g == 0) m_s[warp][8 * nt + 2 * t + k] = m[nt][k], l_s[warp][8 * nt + 2 * t + k] = v;
      }
    __syncthreads();  // (and every warp is done with its ring)
    float *vals = reinterpret_cast<float *>(pt_smem);  // [warp][row][LD]; the low parts of fp32 rows join their high parts
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float f[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float top = -INFINITY;
        for (uint32_t w = 0; w < PT_WARPS; ++w) top = fmaxf(top, m_s[w][8 * nt + 2 * t + k]);
        f[k] = m[nt][k] == -INFINITY ? 0.f : pt_exp2(m[nt][k] - top);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        float y[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          y[c] = o[nt][i][c];
          if (SPLIT) y[c] += __shfl_xor_sync(0xffffffffu, y[c], 2);
          y[c] *= f[c & 1];
        }
        if (!SPLIT || t < 2) {
          float *to = vals + (warp * RI + nt * TILE + 2 * t) * LD + 16 * i + g;
          to[0] = y[0], to[LD] = y[1], to[8] = y[2], to[LD + 8] = y[3];
        }
      }
    }
    __syncthreads();
    const bool whole = ua == 0 && ub == n;
    float *part = plan.part + ((uint64_t)blockIdx.x * 2 + (ua == 0)) * RI * (DP + 2);
    for (uint32_t e = tid; e < RI * DP; e += PT_THREADS) {
      const uint32_t r = e / DP, i = e % DP, c = r / TILE * 8 + r % TILE;
      if (r >= rows) break;
      float y = 0.f, top = -INFINITY, sum = 0.f;
#pragma unroll
      for (uint32_t w = 0; w < PT_WARPS; ++w) y += vals[(w * RI + r) * LD + i], top = fmaxf(top, m_s[w][c]);
#pragma unroll
      for (uint32_t w = 0; w < PT_WARPS; ++w) sum += m_s[w][c] == -INFINITY ? 0.f : l_s[w][c] * pt_exp2(m_s[w][c] - top);
      if (whole) {
        const uint32_t rr = row_a + r;
        if (i < d.head_dim)
          reinterpret_cast<T *>(d.out)[(uint64_t)(sq.row0 + rr / rep) * d.ldo + (uint64_t)(kvh * rep + rr % rep) * d.head_dim + i] = from_f<T>(sum > 0.f ? y / sum : 0.f);
      } else {
        part[r * (DP + 2) + i] = y;
        if (i == 0) part[r * (DP + 2) + DP] = top, part[r * (DP + 2) + DP + 1] = sum;
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();  // the rings may be filled again
    x += ub - ua;
  }
}

// Joins the parts of the KV heads' units that several blocks worked on, in the order of the units.
template <typename T> __global__ void __launch_bounds__(128) paged_join_kernel(const __grid_constant__ cutb_paged_desc d, const PtPlan plan) {
  pdl_enter();
  const uint32_t of = gridDim.x / d.n_seqs, s = blockIdx.x / of, kvh = blockIdx.y, chunk = blockIdx.x % of, dp = pg_pad(d.head_dim), rep = d.n_heads / d.n_kv_heads, RI = plan.rows;
  const PagedSeq sq = paged_seq(d, s);
  const uint32_t chunks = (sq.rows * rep + RI - 1) / RI;
  if (chunk >= chunks) return;
  const uint64_t total = plan.prefix[d.n_seqs] * d.n_kv_heads;
  uint32_t first, n;
  pt_units(d, sq.len, sq.rows, first, n);
  const uint64_t a = plan.prefix[s] * d.n_kv_heads + (uint64_t)(kvh * chunks + chunk) * n;
  const uint32_t shares = pt_shares(total, plan.blocks);
  auto block_of = [&](uint64_t x) {
    uint32_t b = (uint32_t)(x * shares / total);
    while (pt_from(total, shares, b + 1) <= x) ++b;
    return b;
  };
  const uint32_t b0 = block_of(a), b1 = block_of(a + n - 1);
  if (b0 == b1) return;
  const uint32_t row_a = chunk * RI, rows = min(RI, sq.rows * rep - row_a);
  auto part = [&](uint32_t b, uint32_t r) { return plan.part + (((uint64_t)b * 2 + (b == b0)) * RI + r) * (dp + 2); };
  for (uint32_t e = threadIdx.x; e < rows * d.head_dim; e += 128) {
    const uint32_t r = e / d.head_dim, i = e % d.head_dim, rr = row_a + r;
    float top = -INFINITY, y = 0.f, sum = 0.f;
    for (uint32_t b = b0; b <= b1; ++b) top = fmaxf(top, part(b, r)[dp]);
    for (uint32_t b = b0; b <= b1; ++b) {
      const float *p = part(b, r), f = p[dp] == -INFINITY ? 0.f : pt_exp2(p[dp] - top);
      y = fmaf(f, p[i], y), sum = fmaf(f, p[dp + 1], sum);
    }
    reinterpret_cast<T *>(d.out)[(uint64_t)(sq.row0 + rr / rep) * d.ldo + (uint64_t)(kvh * rep + rr % rep) * d.head_dim + i] = from_f<T>(sum > 0.f ? y / sum : 0.f);
  }
}

// Two tiles of columns where one does not hold a sequence's rows: the cache is read once for 8 fp32 or 16 16-bit rows.  (Wider heads
// have no registers for it.)
uint32_t pt_tiles(const cutb_paged_desc &d) {
  const uint64_t rows = (uint64_t)d.max_new * (d.n_heads / d.n_kv_heads);
  return pg_pad(d.head_dim) <= 128 && rows > (d.dtype == CUTB_F32 ? 4 : 8) ? 2 : 1;
}
int pt_plan(const cutb_paged_desc &d, PtPlan *p, uint64_t *bytes) {
  DeviceInfo di;
  if (int rc = get_device_info(&di)) return rc;
  const uint32_t nt = pt_tiles(d), dp = pg_pad(d.head_dim);
  p->rows = (d.dtype == CUTB_F32 ? 4 : 8) * nt;
  p->blocks = di.sm_count * (dp * nt <= 128 ? 2 : 1);
  const uint64_t prefix = (8ull * (d.n_seqs + 1) + 255) / 256 * 256;
  p->prefix = reinterpret_cast<uint64_t *>(d.workspace);
  p->part = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(d.workspace) + prefix);
  *bytes = prefix + 4ull * p->blocks * 2 * p->rows * (dp + 2);
  return CUTB_OK;
}

template <typename T, int DP, int NT> int pt_launch(const cutb_paged_desc &d, const PtPlan &p, cudaStream_t stream) {
  const uint32_t smem = pt_ring_bytes(DP) + 8 * (d.n_seqs + 1) + (uint32_t)sizeof(PtSeq) * d.n_seqs;
  const uint32_t most = pt_ring_bytes(DP) + 8 * (PG_MAX_SEQS + 1) + (uint32_t)sizeof(PtSeq) * PG_MAX_SEQS;
  static_assert(PT_WARPS * (sizeof(T) == 4 ? 4 : 8) * NT * (DP + 4) * 4 <= pt_ring_bytes(DP), "the parts meet in the rings");
  CUTB_CUDA_TRY(cudaFuncSetAttribute(paged_attention_kernel<T, DP, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
  CUTB_CUDA_TRY(launch_pdl(paged_attention_kernel<T, DP, NT>, dim3(p.blocks), dim3(PT_THREADS), smem, stream, d, p));
  const uint32_t chunks = (uint32_t)(((uint64_t)(d.max_new < d.n_tokens ? d.max_new : d.n_tokens) * (d.n_heads / d.n_kv_heads) + p.rows - 1) / p.rows);
  CUTB_CUDA_TRY(launch_pdl(paged_join_kernel<T>, dim3(d.n_seqs * chunks, d.n_kv_heads), dim3(128), 0, stream, d, p));
  return CUTB_OK;
}

}  // namespace

uint64_t paged_attention_workspace(const cutb_paged_desc &d) {
  PtPlan p;
  uint64_t bytes = 0;
  return pt_plan(d, &p, &bytes) == CUTB_OK ? bytes : 0;
}

int paged_attention_launch(const cutb_paged_desc &d, cudaStream_t stream) {
  PtPlan p;
  uint64_t bytes;
  if (int rc = pt_plan(d, &p, &bytes)) return rc;
  return paged_with_type(d.dtype, [&](auto t) {
    using T = decltype(t);
    const bool two = pt_tiles(d) == 2;
    switch (pg_pad(d.head_dim)) {
      case 64: return two ? pt_launch<T, 64, 2>(d, p, stream) : pt_launch<T, 64, 1>(d, p, stream);
      case 128: return two ? pt_launch<T, 128, 2>(d, p, stream) : pt_launch<T, 128, 1>(d, p, stream);
      case 192: return pt_launch<T, 192, 1>(d, p, stream);
      default: return pt_launch<T, 256, 1>(d, p, stream);
    }
  });
}

}  // namespace cutb
