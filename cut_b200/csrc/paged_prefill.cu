// Attention of prompts over the paged 4-bit cache, on the 5th-generation tensor cores.
//
// A block owns X tiles of 128 query rows of one KV head of a sequence (a row is a token and one of the query heads that share the KV
// head), and walks over tiles of 128 keys.
//   softmax warps   (4 X) a row per thread = tensor-memory lane: the scores are read twice, for their maximum and for the weights,
//                   which go back in their place as fp16 (fp32 rows: two terms, the low parts beside them).  As in the kernel for few
//                   rows, weights are relative to a reference that follows the maximum in steps of 2^7, so that the weighted values are rarely
//                   rescaled; what the scores lack to the reference is exact.
//   issuing warp    scores = Q K^T from shared memory, weighted values = P (tensor memory) V; fp32 rows with two terms of Q and of P
//   unpacking warps (7; 16 warps have 128 registers a thread) take turns over units of 16 tokens: nibbles from global memory (the next
//                   tile's are on their way while this one's are turned into fp16), written as the tensor cores read them: K with a token to a row, V with an element to a row, as
//                   its units keep four neighbouring tokens together; 128-byte swizzle.
// A tile of 128 keys costs 256 rows of 128 elements about 2000 cycles of tensor cores, as many of exponentials, and the unpacking 800
// issue slots a scheduler, which run beside one another: two row tiles alternate, and the weights of 64 keys at a time are handed over.
// 8192 tokens of 32 heads (8 KV heads) of 128 in bf16: 703 us, 782 TFLOP/s of the half that is seen; 4 x 1500 behind 1500 more: 362 us; 512
// tokens in fp32: 26 us, of which one tile's chain of products, exponentials and products is the most.
// Weights of 16-bit rows are one fp16 number, as in the kernel for few rows.
// The keys of a row tile are one block's work however many they are: a few rows behind a long cache that come here (more than 32 query rows of a
// KV head) leave most SMs idle, 5 rows of 64 heads behind 100000 keys 1803 us, 4 rows, by the other kernel, 89.
// Every wait is bounded; on expiry the block records CUTB_ERR_TIMEOUT, frees its tensor memory and returns (it has no copies in flight).
#include "kernels.h"
#include "paged_common.cuh"
#include "tcgen05.cuh"

namespace cutb {
namespace {

constexpr uint32_t PP_KEYS = 128, PP_UNITS = 8, PP_UNPACK = 7, PP_PLANE = 128 * 128;  // bytes of 64 columns of 128 rows

template <typename T, int DP> struct PpShape {
  static constexpr bool SPLIT = sizeof(T) == 4;
  static constexpr uint32_t X = SPLIT || DP > 128 ? 1 : 2, TERMS = SPLIT ? 2 : 1;
  static constexpr uint32_t SK = DP <= 192 ? 2 : 1, SV = DP <= 128 ? 2 : 1;
  static constexpr uint32_t QT = DP / 64 * PP_PLANE, KT = QT, VT = DP * 256;  // bytes of a tile
  static constexpr uint32_t SMEM = 1024 + X * TERMS * QT + SK * KT + SV * VT, WARPS = 4 * X + 1 + PP_UNPACK;
  // tensor memory columns: scores and weights from 0, low parts (X = 1), values, and (SPLIT) the values of the tiles before
  static constexpr uint32_t LOW = 128, OUT = 256, TOTAL = 384;
};

// Tensor cores cut a sum off at every product, by some 2^-22 of it: over 131072 keys the values of 16-bit rows came out 8.6e-4 too small, nearly
// twice half a step of fp16.  So a sum goes on there for this many tiles (6e-5), and then is added to fp32 totals in the workspace, which calls
// have that may see more keys.  fp32 rows are added up after every tile, in tensor memory; their sums and the weights' move to totals too (added one
// by one, a million weights came out 2e-5 too small).  The last 2048 rows of 32768 in bf16: 1381 us, 1336 with one sum.
constexpr uint32_t PP_SUM = 64;

struct PpParams {
  float scale, sign;  // |scale| log2(e), and its sign (a scale of zero: queries of zero)
  uint32_t vec, out_vec;
  float4 *totals;     // [block][DP / 4][row], where a row may see more than PP_SUM tiles
};

__device__ __forceinline__ float pp_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pp_pack(float a, float b) { return h2_as_u32(__floats2half2_rn(a, b)); }
__device__ __forceinline__ uint32_t pp_sw(uint32_t row, uint32_t chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }
__device__ __forceinline__ uint32_t pp_fma(__half2 q, __half2 d, __half2 m) { return h2_as_u32(__hfma2(q, d, m)); }
// Tensor memory into registers, the wait in the same statement: the loads write their registers whenever they come, and a copy of one that
// the compiler puts between two statements would read what was there before and free the register for something else.
__device__ __forceinline__ void pp_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
      "%30,%31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
        "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
        "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void pp_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                 "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void pp_sts16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void pp_sts8(uint32_t at, uint32_t a, uint32_t b) {
  asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at), "r"(a), "r"(b) : "memory");
}

template <typename T, int DP>
__global__ void __launch_bounds__(PpShape<T, DP>::WARPS * 32, 1) paged_prefill_kernel(const __grid_constant__ cutb_paged_desc d, const PpParams pp) {
  using S = PpShape<T, DP>;
  constexpr bool SPLIT = S::SPLIT;
  constexpr uint32_t X = S::X, SK = S::SK, SV = S::SV, QT = S::QT, KT = S::KT, VT = S::VT, G = DP / 32, UB = pg_unit_bytes(DP), ROWS = X * 128;
  extern __shared__ __align__(1024) uint8_t pp_raw[];
  const uint32_t smem = (smem_u32(pp_raw) + 1023) & ~1023u, q_u = smem, k_u = q_u + X * S::TERMS * QT, v_u = k_u + SK * KT;
  __shared__ __align__(8) uint64_t bars[2 * SK + 2 * SV + 4 * X + 2];
  __shared__ uint32_t tmem_slot, abort_flag, bad_s, seq_s, tile_s;
  __shared__ float mult_s[ROWS];
  __shared__ PagedSeq found_s;
  const uint32_t tid = threadIdx.x, warp = warp_index(), lane = tid & 31;
  const uint32_t kfull = smem_u32(bars), kempty = kfull + SK * 8, vfull = kempty + SK * 8, vempty = vfull + SV * 8;
  const uint32_t sfull = vempty + SV * 8, pready = sfull + X * 8, odone = pready + 2 * X * 8, qready = odone + X * 8, drained = qready + 8;
  if (tid == 0) {
    for (uint32_t i = 0; i < SK; ++i) mbar_init(kfull + i * 8, PP_UNITS), mbar_init(kempty + i * 8, 1);
    for (uint32_t i = 0; i < SV; ++i) mbar_init(vfull + i * 8, PP_UNITS), mbar_init(vempty + i * 8, 1);
    for (uint32_t x = 0; x < X; ++x) mbar_init(sfull + x * 8, 1), mbar_init(odone + x * 8, 1), mbar_init(pready + 2 * x * 8, 4), mbar_init(pready + (2 * x + 1) * 8, 4);
    mbar_init(qready, 4 * X), mbar_init(drained, 1);
    abort_flag = 0, bad_s = 0;
    fence_mbar_init();
  }
  pdl_enter();
  const uint32_t rep = d.n_heads / d.n_kv_heads, kvh = blockIdx.y;
  if (warp == 4 * X) {  // the sequence and the row tile that the block works on: 32 sequences at a time
    uint32_t before = 0;
    if (lane == 0) seq_s = d.n_seqs;
    __syncwarp();
    for (uint32_t s0 = 0; s0 < d.n_seqs; s0 += 32) {
      uint32_t tiles = 0;
      PagedSeq q = {};
      if (s0 + lane < d.n_seqs) {
        q = paged_seq(d, s0 + lane);
        if (q.bad && blockIdx.x == 0 && kvh == 0) paged_report(d.status, CUTB_ERR_INVALID);
        tiles = (q.rows * rep + ROWS - 1) / ROWS;
      }
      uint32_t sum = tiles;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += y;
      }
      const uint32_t mine = before + sum - tiles;
      if (blockIdx.x >= mine && blockIdx.x < mine + tiles) seq_s = s0 + lane, found_s = q, tile_s = tiles - 1 - (blockIdx.x - mine);  // the later tokens (more keys) first
      before += __shfl_sync(0xffffffffu, sum, 31);
      if (blockIdx.x < before && blockIdx.x) break;  // (block 0 looks at all of them)
    }
    __syncwarp();
  }
  __syncthreads();
  if (seq_s >= d.n_seqs) return;
  const PagedSeq sq = found_s;
  // (what every address below is made of, once more)
  if (sq.slot >= d.n_slots || sq.rows == 0 || sq.rows > d.n_tokens || sq.row0 > d.n_tokens - sq.rows || sq.len < sq.rows || sq.len > d.ld_table * d.page_tokens ||
      tile_s >= (sq.rows * rep + ROWS - 1) / ROWS) {
    if (tid == 0) paged_report(d.status, CUTB_ERR_INVALID);
    return;
  }
  const uint32_t row_a = tile_s * ROWS, n_rows = min(ROWS, sq.rows * rep - row_a), pos0 = sq.len - sq.rows;
  if (warp == 4 * X) {
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // first and one past the last key that each row tile sees; hi = 0: no rows
  uint32_t lo[2] = {0, 0}, hi[2] = {0, 0}, first_pos[2] = {0, 0};
#pragma unroll
  for (uint32_t x = 0; x < X; ++x) {
    if (x * 128 >= n_rows) continue;
    first_pos[x] = pos0 + (row_a + x * 128) / rep;
    hi[x] = pos0 + (row_a + min(n_rows, (x + 1) * 128) - 1) / rep + 1;
    lo[x] = d.window && first_pos[x] + 1 > d.window ? first_pos[x] + 1 - d.window : 0;
  }
  const uint32_t key_lo = lo[0], key_hi = max(hi[0], hi[1]), t_first = key_lo / PP_KEYS, t_end = (key_hi + PP_KEYS - 1) / PP_KEYS;
  const uint32_t *table = d.tables + sq.slot * d.ld_table;
  const uint32_t page_units = d.page_tokens / PG_UNIT, page_mask = page_units - 1, page_shift = 31 - __clz(page_units);
  for (uint32_t p = t_first * 8 / page_units + tid; p <= (key_hi - 1) / d.page_tokens; p += S::WARPS * 32)
    if (table[p] >= d.n_pages) bad_s = 1;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const bool any_bad = bad_s != 0;
  if (any_bad && tid == 0) paged_report(d.status, CUTB_ERR_INVALID);
  auto sees = [&](uint32_t x, uint32_t t) { return t * PP_KEYS < hi[x] && (t + 1) * PP_KEYS > lo[x]; };
  auto give_up = [&]() {
    paged_report(d.status, CUTB_ERR_TIMEOUT);
    atomicExch(&abort_flag, 1u);
  };
  auto aborted = [&]() { return *reinterpret_cast<volatile uint32_t *>(&abort_flag) != 0; };

  if (warp > 4 * X) {
    // ---- unpacking: the warps take turns over the units of all tiles ----
    constexpr uint32_t KQ = DP / 64;  // 16-byte pieces of a unit's keys, and of its values, in a lane
    const uint32_t r = lane / 4, quad = lane % 4, n_end = 8 * t_end;
    const uint8_t *base = reinterpret_cast<const uint8_t *>(d.pages) + (uint64_t)kvh * page_units * UB;
    uint4 kw[KQ], vw[KQ], vs[G];
    uint32_t ks[KQ][G];
    bool there_k = false, there_v = false;
    auto token_of = [&](uint32_t k) { return (128 * k + 4 * lane) / (DP / 8); };  // (a piece lies within one token)
    auto unit_of = [&](uint32_t unit, const uint8_t *&u) {
      u = base;
      if (unit * PG_UNIT >= sq.len) return false;
      const uint32_t page = table[unit >> page_shift];
      if (page >= d.n_pages) return false;
      u = base + (uint64_t)page * d.page_bytes + (unit & page_mask) * UB;
      return true;
    };
    auto load_keys = [&](uint32_t unit) {
      const uint8_t *u;
      if (!(there_k = unit_of(unit, u))) return;
#pragma unroll
      for (uint32_t k = 0; k < KQ; ++k) {
        kw[k] = __ldg(reinterpret_cast<const uint4 *>(u) + 32 * k + lane);
        const uint32_t *sc = reinterpret_cast<const uint32_t *>(u + pg_key_scales_at(DP)) + token_of(k) * G;
#pragma unroll
        for (uint32_t j = 0; j < G; j += 2) *reinterpret_cast<uint2 *>(&ks[k][j]) = __ldg(reinterpret_cast<const uint2 *>(sc + j));
      }
    };
    auto load_values = [&](uint32_t unit) {
      const uint8_t *u;
      if (!(there_v = unit_of(unit, u))) return;
#pragma unroll
      for (uint32_t k = 0; k < KQ; ++k) vw[k] = __ldg(reinterpret_cast<const uint4 *>(u + pg_values_at(DP)) + 32 * k + lane);
#pragma unroll
      for (uint32_t j = 0; j < G; ++j) vs[j] = __ldg(reinterpret_cast<const uint4 *>(u + pg_value_scales_at(DP)) + 4 * j + quad);
    };
    uint32_t unit = 8 * t_first + warp - 4 * X - 1;
    load_keys(unit);
    load_values(unit);
    for (; unit < n_end; unit += PP_UNPACK) {
      // (a fresh barrier lets a wait on the phase before its first pass)
      const uint32_t i0 = unit / 8 - t_first, dw = unit % 8, sk = i0 % SK, pk = ~(i0 / SK) & 1, sv = i0 % SV, pv = ~(i0 / SV) & 1, next = unit + PP_UNPACK;
      if (!__all_sync(0xffffffffu, mbar_wait_probe_first(kempty + sk * 8, pk) && !aborted())) {
        if (lane == 0) give_up();
        break;
      }
      if (there_k) {
#pragma unroll
        for (uint32_t k = 0; k < KQ; ++k) {
          const uint32_t tok = token_of(k), row = dw * 16 + tok, rem = (128 * k + 4 * lane) % (DP / 8);
          uint32_t w[4] = {kw[k].x, kw[k].y, kw[k].z, kw[k].w};
#pragma unroll
          for (uint32_t e = 0; e < 4; ++e) {
            // element e of the piece; tokens of odd places take their neighbours first, so that eight lanes fill a row of banks
            constexpr uint32_t W = DP % 128 == 0 ? 4 : 2;
            const bool odd = tok & 1;
            const uint32_t at = rem + e, j0 = at / (4 * W) * W + at % W, b = at / W % 4, j = odd ? j0 ^ 1 : j0;
            const uint32_t word = odd ? w[e ^ 1] : w[e];
            uint32_t scale = 0;
            if constexpr (DP == 128) {
              scale = odd ? ks[k][e ^ 1] : ks[k][e];
            } else {
#pragma unroll
              for (uint32_t g2 = 0; g2 < G; ++g2) scale = g2 == j ? ks[k][g2] : scale;
            }
            const __half2 s = u32_as_h2(scale), ds = __low2half2(s), ms = __high2half2(s);
            __half2 q[4];
            pg_quants(word, q);
            const uint32_t chunk = 4 * j + b;
            pp_sts16(k_u + sk * KT + chunk / 8 * PP_PLANE + pp_sw(row, chunk % 8), pp_fma(q[0], ds, ms), pp_fma(q[1], ds, ms), pp_fma(q[2], ds, ms), pp_fma(q[3], ds, ms));
          }
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(kfull + sk * 8);
      if (next < n_end) load_keys(next);
      if (!__all_sync(0xffffffffu, mbar_wait_probe_first(vempty + sv * 8, pv) && !aborted())) {
        if (lane == 0) give_up();
        break;
      }
      {
        const uint32_t tok0 = unit * PG_UNIT + 4 * quad, left = !there_v || tok0 >= sq.len ? 0 : min(4u, sq.len - tok0);
        const uint32_t m01 = left >= 2 ? 0xffffffffu : left ? 0xffffu : 0u, m23 = left >= 4 ? 0xffffffffu : left == 3 ? 0xffffu : 0u;
        const uint32_t dst = v_u + sv * VT + dw / 4 * (DP * 128) + (quad & 1) * 8, chunk = dw % 4 * 2 + quad / 2;
#pragma unroll
        for (uint32_t i = 0; i < DP / 16; ++i) {
          const uint4 v4 = vw[i / 4], x = vs[i / 2];
          const uint32_t w[4] = {v4.x, v4.y, v4.z, v4.w};
          const __half2 dA = u32_as_h2(x.x & m01), dB = u32_as_h2(x.y & m23), mA = u32_as_h2(x.z & m01), mB = u32_as_h2(x.w & m23);
          __half2 q[4];
          pg_quants(w[i % 4], q);
          const uint32_t at = dst + pp_sw(16 * i + r, chunk);  // (row r + 8 has the same swizzle)
          pp_sts8(at, pp_fma(q[0], dA, mA), pp_fma(q[2], dB, mB));
          pp_sts8(at + 8 * 128, pp_fma(q[1], dA, mA), pp_fma(q[3], dB, mB));
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(vfull + sv * 8);
      if (next < n_end) load_values(next);
    }
    __syncwarp();
  } else if (warp == 4 * X) {
    // ---- products: one lane waits and issues ----
    // (the other lanes have nothing to do: where they voted on every wait, a commit between two waits was carried out twice)
    const bool leader = elect_one();
    if (leader) {
      const uint64_t proto = umma_desc_sw128(0);
      const uint32_t desc_hi = (uint32_t)(proto >> 32), q_lo = (uint32_t)proto + ((q_u & 0x3FFFFu) >> 4), k_lo = (uint32_t)proto + ((k_u & 0x3FFFFu) >> 4);
      const uint32_t v_lo = (uint32_t)proto + ((v_u & 0x3FFFFu) >> 4);
      constexpr uint32_t id_s = umma_idesc_f16(128, 128), id_o = umma_idesc_f16(128, DP);
      uint32_t sk = 0, pk = 0, sv = 0, pv = 0, pp_[2] = {0, 0}, acc[2] = {0, 0};  // acc: tiles in the sums
      bool ok = mbar_spin_bounded(qready, 0);
      tc_fence_after();
      auto scores = [&](uint32_t x) {
#pragma unroll
        for (uint32_t term = 0; term < S::TERMS; ++term)
#pragma unroll
          for (uint32_t ks = 0; ks < DP / 16; ++ks) {
            const uint32_t off = (ks >> 2) * (PP_PLANE >> 4) + (ks & 3) * 2;
            // (low parts first, while the sum is small: tensor cores cut off what a sum cannot hold)
            umma_f16(tmem + x * 128, q_lo + (x * S::TERMS + S::TERMS - 1 - term) * (QT >> 4) + off, k_lo + sk * (KT >> 4) + off, desc_hi, id_s, term | ks ? 1u : 0u);
          }
        umma_commit(sfull + x * 8);
      };
      auto values = [&](uint32_t x, bool last) {
        ok = ok && mbar_spin_bounded(vfull + sv * 8, pv);
#pragma unroll
        for (uint32_t half = 0; half < 2; ++half) {
          ok = ok && mbar_spin_bounded(pready + (2 * x + half) * 8, pp_[x]);
          if (!ok) return;
          tc_fence_after();
#pragma unroll
          for (uint32_t term = 0; term < S::TERMS; ++term)
#pragma unroll
            for (uint32_t ks = 4 * half; ks < 4 * half + 4; ++ks)
              umma_ts(tmem + S::OUT + x * DP, tmem + (term + 1 < S::TERMS ? S::LOW : x * 128) + ks * 8, v_lo + sv * (VT >> 4) + (ks >> 2) * (DP * 128 >> 4) + (ks & 3) * 2, desc_hi, id_o,
                      term | ks ? 1u : acc[x] != 0);
        }
        pp_[x] ^= 1u;
        umma_commit(odone + x * 8);
        if (last) umma_commit(vempty + sv * 8);
        if (!SPLIT) acc[x] = (acc[x] + 1) % PP_SUM;
        if (last && ++sv == SV) sv = 0, pv ^= 1u;
      };
      bool pending = false;  // the second row tile's value product over the tile before
      for (uint32_t t = t_first; t < t_end && ok; ++t) {
        const bool s0 = sees(0, t), s1 = X > 1 && sees(1, t);
        ok = mbar_spin_bounded(kfull + sk * 8, pk);
        if (!ok) break;
        tc_fence_after();
        if (s0) {
          scores(0);
          if (!s1) umma_commit(kempty + sk * 8);
        }
        if (pending) values(1, true);
        pending = s1;
        if (!ok) break;
        if (s1) {
          scores(1);
          umma_commit(kempty + sk * 8);
        }
        if (s0) values(0, !s1);
        if (++sk == SK) sk = 0, pk ^= 1u;
      }
      if (ok && pending) values(1, true);
      if (!ok) give_up();
      // products in flight read this block's shared memory and write its tensor memory: they end before it does, whoever gave up
      umma_commit(drained);
      if (!mbar_test(drained, 0)) (void)mbar_wait_bounded(drained, 0, 1u << 10);
    }
    __syncwarp();
  } else {
    // ---- a row's queries, scaled by a power of two, as one or two fp16 terms; then its softmax ----
    const uint32_t x = warp >> 2, row = tid & 127, R = row_a + x * 128 + row, Rc = min(R, row_a + n_rows - 1);
    const bool live = x * 128 + row < n_rows;
    const uint32_t pos = pos0 + Rc / rep;
    const uint64_t token = sq.row0 + Rc / rep, head = (uint64_t)(kvh * rep + Rc % rep) * d.head_dim;
    {
      // The rows come as they are to the bytes that their terms will have (asynchronous copies, all at once); then a warp turns 32
      // rows of its own into terms.  Little code: straight-line code is fetched once per block, a few hundred cycles a line.
      constexpr uint32_t PIECES = DP * sizeof(T) / 16, E = DP / 32;  // 16-byte pieces of a row, elements of a lane
      auto place = [&](uint32_t r, uint32_t byte) {  // of a raw row's byte
        return q_u + (r >> 7) * S::TERMS * QT + byte / 128 * PP_PLANE + (r & 127) * 128 + byte % 128;
      };
      const uint32_t r0 = warp * 32;
#pragma unroll 1
      for (uint32_t i = lane; i < 32 * PIECES; i += 32) {
        const uint32_t r = r0 + i / PIECES, c = i % PIECES, Rr = row_a + min(r, n_rows - 1), e = c * 16 / sizeof(T);
        const T *src = reinterpret_cast<const T *>(d.q) + (uint64_t)(sq.row0 + Rr / rep) * d.ldq + (uint64_t)(kvh * rep + Rr % rep) * d.head_dim + e;
        const uint32_t dst = place(r, c * 16);
        if (pp.vec && e < d.head_dim) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
        } else {
          T raw[16 / sizeof(T)];
#pragma unroll
          for (uint32_t k = 0; k < 16 / sizeof(T); ++k) raw[k] = e + k < d.head_dim ? src[k] : from_f<T>(0.f);
          const uint4 w = *reinterpret_cast<const uint4 *>(raw);
          pp_sts16(dst, w.x, w.y, w.z, w.w);
        }
      }
      asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
      __syncwarp();
      constexpr uint32_t B = 4;  // rows at a time
#pragma unroll 1
      for (uint32_t r = r0; r < r0 + 32; r += B) {
        float v[B][E], top[B];
#pragma unroll
        for (uint32_t k = 0; k < B; ++k) {
          top[k] = 0.f;
#pragma unroll
          for (uint32_t i = 0; i < E; i += 2) {
            const uint32_t at = place(r + k, (E * lane + i) * sizeof(T));
            if constexpr (SPLIT) {
              asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v[k][i]), "=f"(v[k][i + 1]) : "r"(at) : "memory");
            } else {
              uint32_t w;
              asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(at) : "memory");
              const T *e = reinterpret_cast<const T *>(&w);
              v[k][i] = to_f(e[0]), v[k][i + 1] = to_f(e[1]);
            }
            top[k] = fmaxf(top[k], fmaxf(fabsf(v[k][i]), fabsf(v[k][i + 1])));
          }
        }
#pragma unroll
        for (int o = 16; o; o /= 2)
#pragma unroll
          for (uint32_t k = 0; k < B; ++k) top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], o));  // (and every lane has read)
#pragma unroll
        for (uint32_t k = 0; k < B; ++k) {
          const uint32_t ex = __float_as_uint(top[k]) >> 23;
          const bool fits = ex > 0 && ex < 254;
          // (an infinite element makes all weights NaN: the row enters as NaN, as in the kernel for few rows)
          const float down = (r + k < n_rows ? pp.sign : 0.f) * (fits ? __uint_as_float((254 - ex) << 23) : ex == 255 ? NAN : 1.f);
          if (lane == 0) mult_s[r + k] = fmaxf((fits ? __uint_as_float(ex << 23) : 1.f) * pp.scale, 1.1754944e-38f);  // (above zero: minus infinity stays itself)
#pragma unroll
          for (uint32_t i = 0; i < E; i += 2) {
            const float f0 = v[k][i] * down, f1 = v[k][i + 1] * down;
            const uint32_t h = pp_pack(f0, f1), c = E * lane + i;
            const uint32_t at = q_u + (r >> 7) * S::TERMS * QT + c / 64 * PP_PLANE + pp_sw((r + k) & 127, c % 64 / 8) + c % 8 * 2;
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(h) : "memory");
            if constexpr (SPLIT) {
              const float2 f = __half22float2(u32_as_h2(h));
              asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + QT), "r"(pp_pack(f0 - f.x, f1 - f.y)) : "memory");
            }
          }
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(qready);
      asm volatile("bar.sync 1, %0;" ::"n"(4 * X * 32) : "memory");
    }
    const float mult = mult_s[x * 128 + row];
    const uint32_t mine = tmem + ((warp & 3) << 21), s_t = mine + x * 128, l_t = mine + S::LOW, o_t = mine + S::OUT + x * DP, t_t = mine + S::TOTAL;
    float low = -INFINITY, from = 0.f, l = 0.f, low_sum = -INFINITY, l_sum = 0.f;  // low_sum: what the totals are relative to, l_sum: the weights'
    uint32_t ph = 0, done = 0;
    float4 *totals = pp.totals + ((uint64_t)blockIdx.x * gridDim.y + kvh) * (ROWS * DP / 4) + x * 128 + row;  // (this thread's own, ROWS apart)
    bool dead = false;
    const uint32_t my_hi = hi[x], my_lo = lo[x], my_first = first_pos[x];
    for (uint32_t t = t_first; t < t_end; ++t) {
      const uint32_t key0 = t * PP_KEYS;
      if (!(key0 < my_hi && key0 + PP_KEYS > my_lo)) continue;
      if (!__all_sync(0xffffffffu, mbar_wait_probe_first(sfull + x * 8, ph) && !aborted())) {
        dead = true;
        break;
      }
      ph ^= 1u;
      tc_fence_after();
      // does every row of the tile see every key?
      const bool all = !any_bad && key0 + PP_KEYS - 1 <= my_first && (!d.window || my_hi - 1 - key0 < d.window);
      uint32_t gone = 0;  // units on pages that do not exist
      if (any_bad)
        for (uint32_t u = 0; u < 8; ++u)
          if ((8 * t + u) * PG_UNIT < my_hi && table[(8 * t + u) >> page_shift] >= d.n_pages) gone |= 1u << u;
      const int last = (int)(pos - key0), oldest = d.window && pos >= d.window ? (int)(pos - d.window + 1 - key0) : -1;  // keys of the tile that the row sees
      auto masked = [&](uint32_t j, uint32_t (&s)[32]) {
        asm volatile("" ::: "memory");  // (a branch: as selects it would be carried out for every tile)
#pragma unroll
        for (int i = 0; i < 32; ++i) s[i] = (i > last - 32 * (int)j) | (i < oldest - 32 * (int)j) ? 0xff800000u : s[i];
        if (gone)
#pragma unroll
          for (uint32_t i = 0; i < 32; ++i) s[i] = gone >> (2 * j + i / 16) & 1 ? 0xff800000u : s[i];
      };
      float mx = -INFINITY;
#pragma unroll 1
      for (uint32_t j = 0; j < 4; ++j) {
        uint32_t s[32];
        pp_ld32(s_t + 32 * j, s);
        if (!all) masked(j, s);
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (uint32_t i = 0; i < 32; ++i) m4[i % 4] = fmaxf(m4[i % 4], __uint_as_float(s[i]));
        mx = fmaxf(mx, fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])));
      }
      const bool rises = __any_sync(0xffffffffu, fmaf(mx, mult, -15.f) > low);
      float f = 1.f;
      if (rises) {
        const float to = fmaxf(low, fmaf(mx, mult, -8.f));
        f = low == to ? 1.f : pp_exp2(low - to);
        low = to, l *= f, from = to == -INFINITY ? 0.f : to;
      }
      // The weighted values follow.  Those of fp32 rows leave the tensor cores after every tile and are added here, those of 16-bit rows after
      // PP_SUM tiles.
      const bool moves = done && done % PP_SUM == 0;  // the sums to the totals; the next tile begins anew
      if (done && (rises || SPLIT || moves)) {
        if (!warp_wait(odone + x * 8, (done - 1) & 1u)) {
          dead = true;
          break;
        }
        tc_fence_after();
        auto sums = [&](uint32_t c, uint32_t (&o)[16]) {
          pp_ld16(o_t + c, o);
          if constexpr (SPLIT) {
            if ((done - 1) % PP_SUM) {
              uint32_t y[16];
              pp_ld16(t_t + c, y);
#pragma unroll
              for (uint32_t i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) + __uint_as_float(y[i]));
            }
          }
        };
        if (moves) {
          const float ft = low_sum == low ? 1.f : pp_exp2(low_sum - low);
#pragma unroll 2
          for (uint32_t c = 0; c < DP; c += 16) {
            float4 y[4] = {};
            if (done > PP_SUM)
#pragma unroll
              for (uint32_t i = 0; i < 4; ++i) y[i] = totals[(c / 4 + i) * ROWS];
            uint32_t o[16];
            sums(c, o);
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
              totals[(c / 4 + i) * ROWS] = make_float4(fmaf(y[i].x, ft, __uint_as_float(o[4 * i]) * f), fmaf(y[i].y, ft, __uint_as_float(o[4 * i + 1]) * f),
                                                       fmaf(y[i].z, ft, __uint_as_float(o[4 * i + 2]) * f), fmaf(y[i].w, ft, __uint_as_float(o[4 * i + 3]) * f));
          }
          l_sum = fmaf(l_sum, ft, l), l = 0.f, low_sum = low;
        } else {
#pragma unroll 1
          for (uint32_t c = 0; c < DP; c += 16) {
            uint32_t o[16];
            sums(c, o);
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_st16(SPLIT ? t_t + c : o_t + c, o);
          }
          if constexpr (SPLIT) tmem_wait_st();
        }
      }
#pragma unroll 1
      for (uint32_t j = 0; j < 4; ++j) {
        uint32_t s[32], h[16];
        pp_ld32(s_t + 32 * j, s);
        if (!all) masked(j, s);
        float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i) {
          const float a = pp_exp2(fmaf(__uint_as_float(s[2 * i]), mult, -from)), b = pp_exp2(fmaf(__uint_as_float(s[2 * i + 1]), mult, -from));
          sum0 += a, sum1 += b;
          h[i] = pp_pack(a, b);
          if constexpr (SPLIT) s[2 * i] = __float_as_uint(a), s[2 * i + 1] = __float_as_uint(b);
        }
        l += sum0 + sum1;
        tmem_st16(s_t + 16 * j, h);
        if constexpr (SPLIT) {
#pragma unroll
          for (uint32_t i = 0; i < 16; ++i) {
            const float2 f = __half22float2(u32_as_h2(h[i]));
            h[i] = pp_pack(__uint_as_float(s[2 * i]) - f.x, __uint_as_float(s[2 * i + 1]) - f.y);
          }
          tmem_st16(l_t + 16 * j, h);
        }
        if (j & 1) {
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(pready + (2 * x + j / 2) * 8);
        }
      }
      ++done;
    }
    if (!dead && done && !warp_wait(odone + x * 8, (done - 1) & 1u)) dead = true;
    if (dead) {
      if (lane == 0) give_up();
    } else if (done) {
      tc_fence_after();
      const float ft = low_sum == low ? 1.f : pp_exp2(low_sum - low);
      l = fmaf(l_sum, ft, l);
      const float inv = l == 0.f ? 0.f : 1.f / l;
      T *out = reinterpret_cast<T *>(d.out) + token * d.ldo + head;
#pragma unroll 1
      for (uint32_t c = 0; c < DP; c += 32) {
        if (c >= d.head_dim) break;
        uint32_t o[32];
        __syncwarp();
        pp_ld32(o_t + c, o);
        if constexpr (SPLIT) {
          if ((done - 1) % PP_SUM) {
            uint32_t y[32];
            pp_ld32(t_t + c, y);
#pragma unroll
            for (uint32_t i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) + __uint_as_float(y[i]));
          }
        }
        if (!live) continue;
        if (done > PP_SUM) {
#pragma unroll
          for (uint32_t i = 0; i < 32; i += 4) {
            const float4 y = totals[(c + i) / 4 * ROWS];
            o[i] = __float_as_uint(fmaf(y.x, ft, __uint_as_float(o[i]))), o[i + 1] = __float_as_uint(fmaf(y.y, ft, __uint_as_float(o[i + 1])));
            o[i + 2] = __float_as_uint(fmaf(y.z, ft, __uint_as_float(o[i + 2]))), o[i + 3] = __float_as_uint(fmaf(y.w, ft, __uint_as_float(o[i + 3])));
          }
        }
        if (pp.out_vec) {
          constexpr uint32_t N = 16 / sizeof(T);
#pragma unroll
          for (uint32_t i = 0; i < 32; i += N) {
            if (c + i >= d.head_dim) break;
            uint4 raw;
            T *e = reinterpret_cast<T *>(&raw);
#pragma unroll
            for (uint32_t k = 0; k < N; ++k) e[k] = from_f<T>(__uint_as_float(o[i + k]) * inv);
            *reinterpret_cast<uint4 *>(out + c + i) = raw;
          }
        } else {
#pragma unroll
          for (uint32_t i = 0; i < 32; ++i)
            if (c + i < d.head_dim) out[c + i] = from_f<T>(__uint_as_float(o[i]) * inv);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4 * X) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// a tile of rows for every 128 X of them, and one more for what each sequence leaves over
uint64_t pp_row_tiles(const cutb_paged_desc &d, uint32_t X) { return (uint64_t)d.n_tokens * (d.n_heads / d.n_kv_heads) / (X * 128) + d.n_seqs; }

template <typename T, int DP> int pp_launch(const cutb_paged_desc &d, cudaStream_t stream) {
  using S = PpShape<T, DP>;
  auto aligned = [&](const void *p, uint64_t ld) { return d.head_dim % 8 == 0 && ld * sizeof(T) % 16 == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  PpParams pp;
  pp.scale = d.scale == 0.f ? 1.f : fabsf(d.scale) * 1.4426950408889634f, pp.sign = d.scale == 0.f ? 0.f : d.scale < 0.f ? -1.f : 1.f;
  pp.vec = aligned(d.q, d.ldq), pp.out_vec = aligned(d.out, d.ldo), pp.totals = reinterpret_cast<float4 *>(d.workspace);
  const uint64_t tiles = pp_row_tiles(d, S::X);
  CUTB_CUDA_TRY(cudaFuncSetAttribute(paged_prefill_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM));
  CUTB_CUDA_TRY(launch_pdl(paged_prefill_kernel<T, DP>, dim3((uint32_t)tiles, d.n_kv_heads), dim3(S::WARPS * 32), S::SMEM, stream, d, pp));
  return CUTB_OK;
}

}  // namespace

bool paged_prefill_applies(const cutb_paged_desc &d) {
  // (tensor memory does not hold the values of an fp32 tile of wider heads twice, beside its scores)
  if (d.dtype == CUTB_F32 && pg_pad(d.head_dim) > 128) return false;
  return (uint64_t)d.max_new * (d.n_heads / d.n_kv_heads) > 32;
}

// The totals of rows that may see more than PP_SUM tiles of keys: all the keys that a table holds, or a window's and those of the other
// rows of a tile.
uint64_t paged_prefill_workspace(const cutb_paged_desc &d) {
  const uint32_t dp = pg_pad(d.head_dim);
  uint64_t seen = (d.ld_table * d.page_tokens + PP_KEYS - 1) / PP_KEYS;
  if (d.window) seen = min(seen, ((uint64_t)d.window + 126) / PP_KEYS + 2);
  if (seen <= PP_SUM) return 0;
  const uint32_t X = d.dtype == CUTB_F32 ? PpShape<float, 128>::X : dp > 128 ? PpShape<__half, 256>::X : PpShape<__half, 128>::X;
  return pp_row_tiles(d, X) * d.n_kv_heads * X * 128 * dp * 4;
}

int paged_prefill_launch(const cutb_paged_desc &d, cudaStream_t stream) {
  return paged_with_type(d.dtype, [&](auto t) {
    using T = decltype(t);
    switch (pg_pad(d.head_dim)) {
      case 64: return pp_launch<T, 64>(d, stream);
      case 128: return pp_launch<T, 128>(d, stream);
      default:
        if constexpr (sizeof(T) == 2) return pg_pad(d.head_dim) == 192 ? pp_launch<T, 192>(d, stream) : pp_launch<T, 256>(d, stream);
        else return (int)CUTB_ERR_UNSUPPORTED;
    }
  });
}

}  // namespace cutb
