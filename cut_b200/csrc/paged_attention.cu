// Attention over the paged 4-bit cache for a few rows of each sequence (single tokens, above all).
//
// scores^T = K Q^T and out^T = V^T P^T on warp MMAs (m16n8k16): the 16 tokens of a unit are the MMA's rows (then its depth), the query
// rows its 8 columns, so that keys and values are the A operands.  The units are laid out for that: a lane's words, nibbles turned into fp16 pairs
// in registers, are its A fragments, and nothing goes through shared memory twice.  P^T comes from the scores' accumulators by movmatrix.
// 16-bit rows take 8 columns.  fp32 rows enter as two fp16 terms: a tile of 8 columns has the high parts of four rows and then their low
// parts, and so have the weights (22 bits of each; the products are exact, the sums fp32).  Queries are scaled by a power of two so
// that the largest element is in [1, 2), weights are kept between 2^8
// and 2^15 at their largest: fp16 holds 2^-24 of the former and 2^-32 of the largest weight.  The weights of 16-bit rows enter as one fp16 number,
// 11 bits: bf16 outputs are as far from the exact ones as rounding takes them, fp16 ones 2.7e-4 instead of 2.1e-4 (over 131072 keys); a second
// term would double the products of the values.
//
// A unit of 128-element heads is 2560 bytes and about 290 warp instructions.  Units are copied whole by bulk
// copies, each warp through a ring of its own, so that a block has up to 80 KB in flight and warps meet only at the ends.
// 64 sequences of 3000 tokens, 32 heads of 128 over 8 KV heads, in bf16: 68 us, 3.6 TB/s; of 8000 in fp32: 147 us, 4.4 TB/s; 2 of 131072 in
// fp16: 82 us, 4.1 TB/s.  What holds it back is that only four warps fit a scheduler (127 registers: the values' sums are in them), which issue in 57 %
// of the cycles, most of it nibbles becoming fp16; a token of 1500 takes 14 us, two launches' latencies.
// Two units a step: what a step costs besides its products (the copy, the maximum over the lanes) is paid half as often.
// The steps of all sequences and KV heads in a row are shared out evenly over the blocks.  Where a block's part begins or ends inside
// a KV head's units, its maxima, sums and values go to the workspace, and a second kernel joins them in their order.
#include "kernels.h"
#include "paged_common.cuh"

namespace cutb {
namespace {

constexpr uint32_t PT_WARPS = 8, PT_THREADS = 32 * PT_WARPS, PT_KEYS = 2 * PG_UNIT;

__host__ __device__ constexpr uint32_t pt_stages(uint32_t dp) { return dp == 64 ? 4 : dp == 128 ? 2 : 2; }
__host__ __device__ constexpr uint32_t pt_ring_bytes(uint32_t dp) { return PT_WARPS * pt_stages(dp) * 2 * pg_unit_bytes(dp); }

struct PtSeq {
  uint32_t slot, len, row0, rows;
};
__device__ __forceinline__ uint64_t pt_div(uint64_t a, uint64_t b) {  // (a 64-bit division takes some hundred cycles)
  return (a | b) >> 32 ? a / b : (uint32_t)a / (uint32_t)b;
}
// The shares of the blocks: `each` steps, the first `more` of them one more; a block for every PT_WARPS steps at most.
struct PtShares {
  uint64_t each, more;
  uint32_t n;
  __device__ __forceinline__ PtShares(uint64_t total, uint32_t blocks) {
    const uint64_t most = (total + PT_WARPS - 1) / PT_WARPS;
    n = (uint32_t)(most < blocks ? most : blocks);
    each = n ? pt_div(total, n) : 0, more = total - each * n;
  }
  __device__ __forceinline__ uint64_t from(uint32_t b) const { return each * b + (b < more ? b : more); }
  __device__ __forceinline__ uint32_t block_of(uint64_t x) const {
    const uint64_t big = more * (each + 1);
    return (uint32_t)(x < big ? pt_div(x, each + 1) : more + pt_div(x - big, each));
  }
};
// first step (two units) that a sequence's rows see, and how many there are up to the last one
__device__ __forceinline__ void pt_units(const cutb_paged_desc &d, uint32_t len, uint32_t rows, uint32_t &first, uint32_t &n) {
  const uint32_t oldest = len - rows;  // position of the first row
  first = d.window && oldest + 1 > d.window ? (oldest + 1 - d.window) / PT_KEYS : 0;
  n = (len + PT_KEYS - 1) / PT_KEYS - first;
}

struct PtPlan {
  uint32_t rows;       // query rows of an item
  uint32_t blocks;     // at most
  uint32_t vec;        // the queries may be read 16 bytes at a time
  float scale, sign;   // |scale| log2(e), and its sign, which goes to the queries (a scale of zero: queries of zero)
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
  __shared__ __align__(16) float2 part_s[8 * NT][PT_WARPS];  // of a column and a warp: what its weights are relative to, their sum
  __shared__ uint64_t sums[PT_WARPS], carry_s;
  const uint32_t tid = threadIdx.x, warp = warp_index(), lane = tid & 31, g = lane / 4, t = lane % 4;
  const uint32_t bar = smem_u32(bars) + warp * S * 8, ring = smem_u32(pt_smem) + warp * S * 2 * UB;
  const uint32_t page_units = d.page_tokens / PG_UNIT, page_mask = page_units - 1, page_shift = 31 - __clz(page_units);
  if (lane == 0) {
    for (uint32_t i = 0; i < S; ++i) mbar_init(bar + 8 * i, 2);
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
  const PtShares shares(total, plan.blocks);
  if (blockIdx.x >= shares.n) return;
  const uint64_t begin = shares.from(blockIdx.x), end = shares.from(blockIdx.x + 1);
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
    const uint32_t chunks = chunks_of(sq.rows), item = (uint32_t)pt_div(local, n), ua = (uint32_t)(local - (uint64_t)item * n), kvh = item / chunks, row_a = item % chunks * RI;
    const uint32_t ub = (uint32_t)min((uint64_t)n, ua + (end - x)), rows = min(RI, sq.rows * rep - row_a);
    const uint32_t *table = d.tables + sq.slot * d.ld_table;
    const uint8_t *base = reinterpret_cast<const uint8_t *>(d.pages) + (uint64_t)kvh * page_units * UB;
    // steps of this warp: ua + warp, + 8, ...; the pages of 16 of them at a time are in the lanes, one for each unit
    const uint32_t mine = ub > ua + warp ? (ub - ua - warp + PT_WARPS - 1) / PT_WARPS : 0;
    auto unit_at = [&](uint32_t i) { return 2 * (first + ua + warp + PT_WARPS * i); };
    const uint8_t *source = nullptr;  // of this lane's unit
    uint32_t pages_there = 0;         // of the 32 units
    // Starts the copies of step i into stage `to`, each by the lane that has the unit's address; bit u of the result: unit u has
    // keys and its page exists.
    auto issue = [&](uint32_t i, uint32_t to) {
      if (i % 16 == 0) {
        const uint32_t k = i + lane / 2, unit = unit_at(k) + (lane & 1);
        const bool keys = k < mine && unit * PG_UNIT < sq.len;
        const uint32_t page = keys ? table[unit >> page_shift] : CUTB_NO_PAGE;
        if (keys && page >= d.n_pages) paged_report(d.status, CUTB_ERR_INVALID);
        source = base + (uint64_t)page * d.page_bytes + (unit & page_mask) * UB;
        pages_there = __ballot_sync(0xffffffffu, page < d.n_pages);
      }
      if (lane / 2 == i % 16) {
        if (pages_there >> lane & 1) {
          mbar_arrive_expect_tx(bar + 8 * to, UB);
          bulk_g2s(ring + (to * 2 + (lane & 1)) * UB, source, UB, bar + 8 * to);
        } else {
          mbar_arrive(bar + 8 * to);
        }
      }
      return pages_there >> 2 * (i % 16) & 3u;
    };
    uint32_t there = 0;  // two bits of each stage
    uint32_t issued = 0;
    if (!dead)
      for (; issued < min(mine, S); ++issued) {
        const uint32_t to = (stage + issued) % S;
        there = (there & ~(3u << 2 * to)) | issue(issued, to) << 2 * to;
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
      for (int j = 0; j < G; ++j) {
        const uint32_t i = 32 * j + 8 * t;
        if (plan.vec) {  // eight elements that are there or not
          uint4 raw[sizeof(T) / 2] = {};
          if (live && i < d.head_dim)
#pragma unroll
            for (int k = 0; k < (int)sizeof(T) / 2; ++k) raw[k] = __ldg(reinterpret_cast<const uint4 *>(src + i) + k);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[j][e] = to_f(reinterpret_cast<const T *>(raw)[e]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[j][e] = live && i + e < d.head_dim ? to_f(src[i + e]) : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[j][e]));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^-e of the largest element (of numbers too small: none).  An infinite element makes every score infinite or NaN, and so the weights NaN
      // whatever the signs: the row enters as NaN.
      const uint32_t ex = __float_as_uint(top) >> 23;
      const float down = plan.sign * (ex > 0 && ex < 254 ? __uint_as_float((254 - ex) << 23) : ex == 255 ? NAN : 1.f), up = ex > 0 && ex < 254 ? __uint_as_float(ex << 23) : 1.f;
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
        mult[nt][k] = fmaxf(__shfl_sync(0xffffffffu, up, cr * 4) * plan.scale, 1.1754944e-38f);  // (above zero: minus infinity stays itself)
        at[nt][k] = cr < TILE && nt * TILE + cr < rows ? sq.len - sq.rows + rr / rep + 1 : 0;
      }
    }
    const uint32_t pos_min = sq.len - sq.rows + row_a / rep, pos_max = sq.len - sq.rows + (row_a + rows - 1) / rep;
    // Weights are taken relative to `low`: 2^8 for a score that is the largest so far, up to 2^15 before `low` follows it, so that the
    // values are rescaled rarely; fp16 pairs hold 2^-24 of that, and the sums are fp32 whatever their scale.
    float low[NT][2], from[NT][2], l[NT][2], o[NT][MT][4];  // from: low where there is one
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      low[nt][0] = low[nt][1] = -INFINITY, from[nt][0] = from[nt][1] = l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int i = 0; i < MT; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
    }
    const uint32_t tk = 4 * (g / 2) + (g & 1);  // the token of MMA row g; row g + 8 is the second after it
    for (uint32_t i = 0; i < mine && !dead; ++i) {
      if (!warp_wait(bar + 8 * stage, phase)) {
        dead = true;
        break;
      }
      const uint8_t *u0 = pt_smem + (ring - smem_u32(pt_smem)) + stage * 2 * UB;
      const uint32_t exists = there >> 2 * stage & 3;
      const uint32_t key0 = unit_at(i) * PG_UNIT;
      const bool edge = exists != 3 || key0 + PT_KEYS - 1 > pos_min || (d.window && pos_max >= key0 && pos_max - key0 >= d.window);
      float sc[NT][2][4] = {};  // (the two units' sums are independent chains)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint8_t *u = u0 + half * UB;
        alignas(16) uint32_t w0[G], w1[G], s0[G], s1[G];
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
        if constexpr (G % 4 == 0) {
#pragma unroll
          for (int j = 0; j < G; j += 4) {
            *reinterpret_cast<uint4 *>(s0 + j) = *reinterpret_cast<const uint4 *>(ks + j);
            *reinterpret_cast<uint4 *>(s1 + j) = *reinterpret_cast<const uint4 *>(ks + 2 * G + j);
          }
        } else {
#pragma unroll
          for (int j = 0; j < G; j += 2) {
            *reinterpret_cast<uint2 *>(s0 + j) = *reinterpret_cast<const uint2 *>(ks + j);
            *reinterpret_cast<uint2 *>(s1 + j) = *reinterpret_cast<const uint2 *>(ks + 2 * G + j);
          }
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
            mma_f16(sc[nt][half], h2_as_u32(a[0]), h2_as_u32(b[0]), h2_as_u32(a[1]), h2_as_u32(b[1]), qf[nt][2 * j][0], qf[nt][2 * j][1]);
            mma_f16(sc[nt][half], h2_as_u32(a[2]), h2_as_u32(b[2]), h2_as_u32(a[3]), h2_as_u32(b[3]), qf[nt][2 * j + 1][0], qf[nt][2 * j + 1][1]);
          }
        }
        if (SPLIT)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c) sc[nt][half][c] += __shfl_xor_sync(0xffffffffu, sc[nt][half][c], 2);
      }
      if (edge) {
        // what is past the sequence, or on a page that is not there, may be anything: its values become zeros
        if (exists != 3 || key0 + PT_KEYS > sq.len) {
          constexpr uint32_t WORDS = pg_unit_bytes(DP) / 10 / 4;  // of a unit's value scales, a word for two tokens
          for (uint32_t e = lane; e < 2 * WORDS; e += 32) {
            const uint32_t half = e / WORDS, w = e % WORDS, quad = w / 4 % 4, pair = w % 2;
            uint32_t *to = reinterpret_cast<uint32_t *>(const_cast<uint8_t *>(u0) + half * UB + pg_value_scales_at(DP)) + w;
            const uint32_t tok = key0 + half * PG_UNIT + 4 * quad + 2 * pair;
            const uint32_t keep = !(exists >> half & 1) || tok >= sq.len ? 0u : tok + 1 >= sq.len ? 0xffffu : 0xffffffffu;
            *to &= keep;
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const uint32_t key = key0 + c / 4 * PG_UNIT + tk + (c & 2), p1 = at[nt][c & 1];
            if (!(exists >> c / 4 & 1) || key >= p1 || (d.window && p1 - key > d.window)) sc[nt][c / 4][c % 4] = -INFINITY;
          }
      }
      uint32_t bf[NT][2][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float f[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) f[k] = fmaxf(fmaxf(sc[nt][0][k], sc[nt][0][k + 2]), fmaxf(sc[nt][1][k], sc[nt][1][k + 2]));
        if (__any_sync(0xffffffffu, fmaf(f[0], mult[nt][0], -15.f) > low[nt][0] || fmaf(f[1], mult[nt][1], -15.f) > low[nt][1])) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float mx = f[k];
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float to = fmaxf(low[nt][k], fmaf(mx, mult[nt][k], -8.f));
            f[k] = low[nt][k] == to ? 1.f : pt_exp2(low[nt][k] - to);
            low[nt][k] = to, l[nt][k] *= f[k];
            from[nt][k] = to == -INFINITY ? 0.f : to;
          }
#pragma unroll
          for (int i2 = 0; i2 < MT; ++i2) o[nt][i2][0] *= f[0], o[nt][i2][1] *= f[1], o[nt][i2][2] *= f[0], o[nt][i2][3] *= f[1];
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float p[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) p[c] = pt_exp2(fmaf(sc[nt][half][c], mult[nt][c & 1], -from[nt][c & 1]));
          l[nt][0] += p[0] + p[2], l[nt][1] += p[1] + p[3];
          uint32_t h0 = pack_half(p[0], p[1]), h1 = pack_half(p[2], p[3]);
          if (SPLIT) {
            const float2 a = __half22float2(u32_as_h2(h0)), b = __half22float2(u32_as_h2(h1));
            const uint32_t l0 = pack_half(p[0] - a.x, p[1] - a.y), l1 = pack_half(p[2] - b.x, p[3] - b.y);
            h0 = t < 2 ? h0 : l0, h1 = t < 2 ? h1 : l1;
          }
          bf[nt][half][0] = transposed(h0), bf[nt][half][1] = transposed(h1);
        }
      }
#pragma unroll
      for (int q4 = 0; q4 < MT / 4; ++q4) {
        uint4 w4[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) w4[half] = *(reinterpret_cast<const uint4 *>(u0 + half * UB + pg_values_at(DP)) + 32 * q4 + lane);
#pragma unroll
        for (int gr = 0; gr < 2; ++gr) {
          uint4 x[2];
#pragma unroll
          for (int half = 0; half < 2; ++half) x[half] = *(reinterpret_cast<const uint4 *>(u0 + half * UB + pg_value_scales_at(DP)) + 4 * (2 * q4 + gr) + t);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            // A step's values are added here, rounded: tensor cores cut off what a sum cannot hold, 2^-22 of it at every product, so that one
            // over a warp's 131072 keys came out 2^-10 too small.  (64 x 3000 tokens in bf16 77.8 us, 76.8 with one sum; heads of 256 140 and 136.)
            float fresh[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int c = 0; c < 4; ++c) fresh[nt][c] = 0.f;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const __half2 dA = u32_as_h2(x[half].x), dB = u32_as_h2(x[half].y), mA = u32_as_h2(x[half].z), mB = u32_as_h2(x[half].w);
              const uint32_t ws[4] = {w4[half].x, w4[half].y, w4[half].z, w4[half].w};
              __half2 a[4];
              pg_quants(ws[2 * gr + k], a);
              a[0] = __hfma2(a[0], dA, mA), a[1] = __hfma2(a[1], dA, mA), a[2] = __hfma2(a[2], dB, mB), a[3] = __hfma2(a[3], dB, mB);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma_f16(fresh[nt], h2_as_u32(a[0]), h2_as_u32(a[1]), h2_as_u32(a[2]), h2_as_u32(a[3]), bf[nt][half][0], bf[nt][half][1]);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int c = 0; c < 4; ++c) o[nt][4 * q4 + 2 * gr + k][c] += fresh[nt][c];
          }
        }
      }
      __syncwarp();  // the units are read
      if (issued < mine) {
        there = (there & ~(3u << 2 * stage)) | issue(issued, stage) << 2 * stage;
        ++issued;
      }
      if (++stage == S) stage = 0, phase ^= 1u;
    }
    if (dead) {
      for (uint32_t i = 0; i < S; ++i) mbar_drain(bar + 8 * i, i < stage ? phase ^ 1u : phase);  // nothing may land in a block that has ended
      if (lane == 0) paged_report(d.status, CUTB_ERR_TIMEOUT);
    }
    // the warps' parts meet, each in its warp's ring; the low parts of fp32 rows join their high parts
    float *vals = reinterpret_cast<float *>(pt_smem + warp * S * 2 * UB);  // [row][LD]
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float v = l[nt][k];
        v += __shfl_xor_sync(0xffffffffu, v, 4), v += __shfl_xor_sync(0xffffffffu, v, 8), v += __shfl_xor_sync(0xffffffffu, v, 16);
        if (g == 0) part_s[8 * nt + 2 * t + k][warp] = make_float2(low[nt][k], v);
      }
      const bool in0 = nt * TILE + 2 * t < rows, in1 = nt * TILE + 2 * t + 1 < rows;
      float *to = vals + (nt * TILE + 2 * t) * LD + g;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        float y[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          y[c] = o[nt][i][c];
          if (SPLIT) y[c] += __shfl_xor_sync(0xffffffffu, y[c], 2);
        }
        if (!SPLIT || t < 2) {
          if (in0) to[16 * i] = y[0], to[16 * i + 8] = y[2];
          if (in1) to[16 * i + LD] = y[1], to[16 * i + LD + 8] = y[3];
        }
      }
    }
    __syncthreads();
    const bool whole = ua == 0 && ub == n;
    float *part = plan.part + ((uint64_t)blockIdx.x * 2 + (ua == 0)) * RI * (DP + 2);
    for (uint32_t e = tid; e < rows * DP; e += PT_THREADS) {
      const uint32_t r = e / DP, i = e % DP, c = r / TILE * 8 + r % TILE;
      float2 w[PT_WARPS];
      float y = 0.f, top = -INFINITY, sum = 0.f;
#pragma unroll
      for (uint32_t k = 0; k < PT_WARPS; ++k) w[k] = part_s[c][k], top = fmaxf(top, w[k].x);
#pragma unroll
      for (uint32_t k = 0; k < PT_WARPS; ++k) {
        const float f = w[k].x == -INFINITY ? 0.f : pt_exp2(w[k].x - top);
        sum = fmaf(f, w[k].y, sum);
        y = fmaf(f, reinterpret_cast<const float *>(pt_smem + k * S * 2 * UB)[r * LD + i], y);
      }
      if (whole) {
        const uint32_t rr = row_a + r;
        if (i < d.head_dim)
          reinterpret_cast<T *>(d.out)[(uint64_t)(sq.row0 + rr / rep) * d.ldo + (uint64_t)(kvh * rep + rr % rep) * d.head_dim + i] = from_f<T>(sum == 0.f ? 0.f : y / sum);
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

// Joins the parts of the KV heads' steps that several blocks worked on, in the order of the steps: a block per query row, which
// weighs all parts first.
constexpr uint32_t PJ_THREADS = 128;
template <typename T> __global__ void __launch_bounds__(PJ_THREADS) paged_join_kernel(const __grid_constant__ cutb_paged_desc d, const PtPlan plan) {
  extern __shared__ float2 weight_s[];  // of part b: {largest score, sum}, then its weight
  __shared__ float warps[2][4];
  pdl_enter();
  const uint32_t dp = pg_pad(d.head_dim), rep = d.n_heads / d.n_kv_heads, tid = threadIdx.x;
  const uint32_t RI = plan.rows, token = blockIdx.x / rep, kvh = blockIdx.y, s = paged_seq_of(d, token);
  if (s >= d.n_seqs) return;
  const PagedSeq sq = paged_seq(d, s);
  if (token - sq.row0 >= sq.rows) return;
  const uint32_t row = blockIdx.x - sq.row0 * rep;
  const uint32_t chunks = (sq.rows * rep + RI - 1) / RI, chunk = row / RI, r = row % RI;
  const uint64_t total = plan.prefix[d.n_seqs] * d.n_kv_heads;
  uint32_t first, n;
  pt_units(d, sq.len, sq.rows, first, n);
  const uint64_t a = plan.prefix[s] * d.n_kv_heads + (uint64_t)(kvh * chunks + chunk) * n;
  const PtShares shares(total, plan.blocks);
  const uint32_t b0 = shares.block_of(a), parts = shares.block_of(a + n - 1) - b0 + 1;
  if (parts == 1) return;
  const uint64_t step = 2ull * RI * (dp + 2);
  const float *mid = plan.part + (uint64_t)b0 * step + (uint64_t)r * (dp + 2);  // of block b0 + k: k steps on; the first has its second slot
  auto part = [&](uint32_t k) { return mid + k * step + (k ? 0 : (uint64_t)RI * (dp + 2)); };
  float top = -INFINITY;
  for (uint32_t k = tid; k < parts; k += PJ_THREADS) {
    weight_s[k] = make_float2(part(k)[dp], part(k)[dp + 1]);
    top = fmaxf(top, weight_s[k].x);
  }
#pragma unroll
  for (int o = 16; o; o /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((tid & 31) == 0) warps[0][tid / 32] = top;
  __syncthreads();
  top = fmaxf(fmaxf(warps[0][0], warps[0][1]), fmaxf(warps[0][2], warps[0][3]));
  float sum = 0.f;
  for (uint32_t k = tid; k < parts; k += PJ_THREADS) {
    const float2 w = weight_s[k];
    const float f = w.x == -INFINITY ? 0.f : pt_exp2(w.x - top);
    weight_s[k].x = f, sum = fmaf(f, w.y, sum);
  }
#pragma unroll
  for (int o = 16; o; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((tid & 31) == 0) warps[1][tid / 32] = sum;
  __syncthreads();
  sum = (warps[1][0] + warps[1][1]) + (warps[1][2] + warps[1][3]);
  T *out = reinterpret_cast<T *>(d.out) + (uint64_t)(sq.row0 + row / rep) * d.ldo + (uint64_t)(kvh * rep + row % rep) * d.head_dim;
  for (uint32_t i = tid; i < d.head_dim; i += PJ_THREADS) {
    float y = 0.f;
#pragma unroll 8
    for (uint32_t k = 0; k < parts; ++k) y = fmaf(weight_s[k].x, part(k)[i], y);
    out[i] = from_f<T>(sum == 0.f ? 0.f : y / sum);
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
  p->scale = d.scale == 0.f ? 1.f : fabsf(d.scale) * 1.4426950408889634f, p->sign = d.scale == 0.f ? 0.f : d.scale < 0.f ? -1.f : 1.f;
  p->vec = d.head_dim % 8 == 0 && d.ldq * (d.dtype == CUTB_F32 ? 4 : 2) % 16 == 0 && reinterpret_cast<uintptr_t>(d.q) % 16 == 0;
  const uint64_t prefix = (8ull * (d.n_seqs + 1) + 255) / 256 * 256;
  p->prefix = reinterpret_cast<uint64_t *>(d.workspace);
  p->part = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(d.workspace) + prefix);
  *bytes = prefix + 4ull * p->blocks * 2 * p->rows * (dp + 2);
  return CUTB_OK;
}

template <typename T, int DP, int NT> int pt_launch(const cutb_paged_desc &d, const PtPlan &p, cudaStream_t stream) {
  const uint32_t smem = pt_ring_bytes(DP) + 8 * (d.n_seqs + 1) + (uint32_t)sizeof(PtSeq) * d.n_seqs;
  const uint32_t most = pt_ring_bytes(DP) + 8 * (PG_MAX_SEQS + 1) + (uint32_t)sizeof(PtSeq) * PG_MAX_SEQS;
  static_assert((sizeof(T) == 4 ? 4 : 8) * NT * (DP + 4) * 4 <= pt_ring_bytes(DP) / PT_WARPS, "a warp's part fits in its ring");
  CUTB_CUDA_TRY(cudaFuncSetAttribute(paged_attention_kernel<T, DP, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
  CUTB_CUDA_TRY(launch_pdl(paged_attention_kernel<T, DP, NT>, dim3(p.blocks), dim3(PT_THREADS), smem, stream, d, p));
  CUTB_CUDA_TRY(launch_pdl(paged_join_kernel<T>, dim3(d.n_tokens * (d.n_heads / d.n_kv_heads), d.n_kv_heads), dim3(PJ_THREADS), 8 * p.blocks, stream, d, p));
  return CUTB_OK;
}

}  // namespace

uint64_t paged_attention_workspace(const cutb_paged_desc &d) {
  if (paged_prefill_applies(d)) return paged_prefill_workspace(d);
  PtPlan p;
  uint64_t bytes = 0;
  return pt_plan(d, &p, &bytes) == CUTB_OK ? bytes : 0;
}

int paged_attention_launch(const cutb_paged_desc &d, cudaStream_t stream) {
  if (paged_prefill_applies(d)) return paged_prefill_launch(d, stream);
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
