// The next token of each row of logits, by a given random number.
//
// A cluster of 1 to 8 blocks works on a row.  A block keeps its part as fp32 in shared memory, or where that would leave one block on
// an SM reads it again from L2.  Weights are integers of 2^-42 of the largest, so that sums do not depend on the order of additions and
// blocks (fp32 weights would move a choice among a hundred thousand even ones once in a few hundred draws).
// The cut-offs are places in the falling order: the key (a logit's bits as an ordered integer) where a count or a sum of weights has
// gone by.  A histogram of 2048 places of the weights' exponents (32-bit additions only: a weight as three times 16 bits, at most 2^16
// elements to a block; every block adds up the cluster's histograms for itself, one cluster barrier) gives a place, and the tokens there
// are compared with one another, or where they are many found by their keys, 11 bits at a time.  A top-k up to 256 needs a histogram of
// the threads' largest logits only.  Equal logits are cut off by their index.  The draw adds up the kept weights in the order of the indices.
// Bound by instructions and, for few rows, by barriers: 1 x 32000 fp32 logits with every cut-off 10 us, 64 of them 14 (with top-p alone
// 33), 256 x 128256 bf16 logits without cut-offs 68 us, with top-k and top-p 48, with top-p alone 291.
#include <cooperative_groups.h>

#include <type_traits>

#include "kernels.h"
#include "paged_common.cuh"

namespace cutb {
namespace {

namespace cg = cooperative_groups;

constexpr uint32_t SM_THREADS = 512, SM_WARPS = 16, SM_BINS = 2048, SM_LIST = SM_THREADS;
constexpr uint32_t SM_VOCAB = 1u << 19;        // an eighth of it is 2^16 elements to a block: their 16-bit pieces add up in 32 bits
constexpr uint32_t SM_SHARED = 100 * 1024;    // dynamic shared memory of a block, at most: two blocks on an SM
constexpr double SM_ONE = 4398046511104.0;  // 2^42
typedef unsigned long long u64;

// A logit as it counts: a NaN is minus infinity, minus zero is zero.
__device__ __forceinline__ float sm_logit(float v) { return fmaxf(v, -INFINITY) + 0.f; }
// larger logits have larger keys
__device__ __forceinline__ uint32_t sm_key(float v) {
  const uint32_t b = __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float sm_value(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }

struct SmShared {
  double powers[256];
  u64 sums[SM_WARPS], part[4];
  uint32_t max_s, found_s, bin_s, many_s, tally[4], range[2];
  u64 left_s, bin_sum;
};

// 2^42 2^(i / 256), summed up by the compiler
struct SmPowers {
  double v[256];
  constexpr SmPowers() : v() {
    for (int i = 0; i < 256; ++i) {
      const double x = i * 0.69314718055994530942 / 256;
      double term = 1, sum = 1;
      for (int k = 1; k < 24; ++k) term *= x / k, sum += term;
      v[i] = sum * SM_ONE;
    }
  }
};
__device__ const SmPowers sm_powers;

struct SmRow {
  float top;
  double rate, offset;   // log2(e) / temperature, and it times the largest logit
  const double *powers;  // 2^42 2^(i / 256)
  // exp((v - top) / temperature) in units of 2^-42, rounded: 2^t = 2^n 2^(i / 256) (1 + c), c = exp(r ln 2) - 1 to its third power for |r| <=
  // 1 / 512 (2^-42 is left).  Ten operations in 64 bits (with pairs of fp32 numbers it were 45 in all), the ends selected without
  // branches: 256 rows of 128256 bf16 logits without cut-offs take 68 us, where reading them takes 10.
  __device__ __forceinline__ u64 mass(float v) const {
    const double t = fma((double)v, rate, -offset);
    constexpr double BIG = 6755399441055744.0 / 256.0;  // 3 * 2^51 / 256: the last place of a sum with it is 1 / 256
    const double s = t + BIG, r = t - (s - BIG);
    const int k = __double2loint(s);
    const double at = powers[k & 255], p = __hiloint2double(__double2hiint(at) + ((k >> 8) << 20), __double2loint(at));  // (2^n: n >= -44)
    const double m = fma(p, r * fma(r, fma(r, 0.055504108664821580, 0.24022650695910071), 0.69314718055994531), p) + 4503599627370496.0;
    const u64 units = (u64)__double_as_longlong(m) & 0xfffffffffffffull;  // the last place of 2^52 is 1
    return v == top ? 1ull << 42 : t > -44.0 ? units : 0;  // (infinite logits too, and what is not a number: 0)
  }
};

// floor(f total) of 0 <= f < 1, and whether something is left over
__device__ __forceinline__ u64 sm_share(float f, u64 total, bool &rest) {
  const uint32_t b = __float_as_uint(f), e = b >> 23, m = e ? (b & 0x7fffffu) | 0x800000u : b & 0x7fffffu, down = 150 - (e ? e : 1);  // f = m 2^-down
  const u64 lo = total * m, hi = __umul64hi(total, m);
  if (down >= 128) return rest = lo | hi, 0;
  if (down >= 64) return rest = lo || (hi & ((1ull << (down - 64)) - 1)), hi >> (down - 64);
  return rest = lo & ((1ull << down) - 1), lo >> down | hi << (64 - down);  // (24 <= down)
}
// of a cut-off p < 1: the largest weight before a token that is kept (one below the target, a number above zero)
__device__ __forceinline__ u64 sm_before(float p, u64 total) {
  if (!(p > 0.f)) return 0;
  bool rest;
  const u64 w = sm_share(p, total, rest);
  return rest || !w ? w : w - 1;
}

// What is kept so far: keys above `key`, and of those equal to it the ones up to index `last`.
struct SmCut {
  uint32_t key, last;
  __device__ __forceinline__ bool keeps(uint32_t k, uint32_t i) const { return k > key || (k == key && i <= last); }
};

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o; o /= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ u64 warp_before(u64 v) {  // sum of the lanes up to and with this one
  const uint32_t lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const u64 y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= (uint32_t)o) v += y;
  }
  return v;
}

// RESIDENT: the block's part of the row is in shared memory; else it is read again, from L2
template <typename T, bool RESIDENT> __global__ void __launch_bounds__(SM_THREADS, 2) sample_kernel(const __grid_constant__ cutb_sample_desc d, uint32_t part) {
  extern __shared__ __align__(16) uint8_t sm_raw[];
  __shared__ SmShared sh;
  cg::cluster_group cl = cg::this_cluster();
  const uint32_t C = cl.num_blocks(), rank = cl.block_rank(), r = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = warp_index();
  float *x_s = reinterpret_cast<float *>(sm_raw);
  uint32_t *hist = reinterpret_cast<uint32_t *>(sm_raw + (RESIDENT ? (part * 4 + 15) / 16 * 16 : 0));  // two of three times SM_BINS
  if (tid < 256) sh.powers[tid] = sm_powers.v[tid];
  if (tid == 0) sh.max_s = 0;
  pdl_enter();
  __syncthreads();
  const uint32_t a = min(d.vocab, rank * part), n = min(d.vocab, a + part) - a;  // this block's part: a .. a + n - 1
  const T *src = reinterpret_cast<const T *>(d.logits) + r * d.ld + a;
  const float temp = d.temperature ? d.temperature[r] : 1.f, p = d.top_p ? d.top_p[r] : 1.f, least = d.min_p ? d.min_p[r] : 0.f, u = d.u[r];
  const uint32_t k = d.top_k ? d.top_k[r] : 0;
  const bool bad = !(temp >= 0.f && temp < INFINITY) || p != p || least != least || !(u >= 0.f && u < 1.f);
  float highest = -INFINITY;  // (fmaxf passes over what is not a number)
  auto take = [&](uint32_t i, float v) {
    if (RESIDENT) x_s[i] = sm_logit(v);
    highest = fmaxf(highest, v);
  };
  {
    constexpr uint32_t V = 16 / sizeof(T);  // elements of a load
    const uint32_t head = min(n, (uint32_t)((16 - reinterpret_cast<uintptr_t>(src) % 16) % 16 / sizeof(T))), vecs = (n - head) / V;
    if (tid < head) take(tid, to_f(src[tid]));
#pragma unroll 4
    for (uint32_t i = tid; i < vecs; i += SM_THREADS) {
      const uint4 w = __ldg(reinterpret_cast<const uint4 *>(src + head) + i);
      const T *e = reinterpret_cast<const T *>(&w);
#pragma unroll
      for (uint32_t j = 0; j < V; ++j) take(head + V * i + j, to_f(e[j]));
    }
    const uint32_t rest = head + V * vecs + tid;
    if (rest < n) take(rest, to_f(src[rest]));
  }
  uint32_t best = __reduce_max_sync(0xffffffffu, sm_key(sm_logit(highest)));
  if (lane == 0) atomicMax(&sh.max_s, best);
  auto logit = [&](uint32_t i) { return RESIDENT ? x_s[i] : sm_logit(to_f(src[i])); };
  // f(i, logit i) for first <= i < end (first a multiple of 8) by threads me, me + step, ..
  constexpr uint32_t V = 16 / sizeof(T);
  const bool vec = reinterpret_cast<uintptr_t>(src) % 16 == 0;
  auto sweep = [&](uint32_t first, uint32_t end, uint32_t me, uint32_t step, auto f) {
    if (RESIDENT || !vec) {
#pragma unroll 4
      for (uint32_t i = first + me; i < end; i += step) f(i, logit(i));
    } else {
#pragma unroll 2
      for (uint32_t i = first + V * me; i < end; i += V * step) {
        if (i + V <= end) {
          const uint4 w = __ldg(reinterpret_cast<const uint4 *>(src + i));
          const T *e = reinterpret_cast<const T *>(&w);
#pragma unroll
          for (uint32_t j = 0; j < V; ++j) f(i + j, sm_logit(to_f(e[j])));
        } else {
          for (uint32_t j = i; j < end; ++j) f(j, logit(j));
        }
      }
    }
  };
  cl.sync();  // (and the part is in shared memory)
  best = 0;
  for (uint32_t q = 0; q < C; ++q) best = max(best, *cl.map_shared_rank(&sh.max_s, q));
  SmRow row;
  row.top = sm_value(best), row.rate = temp > 0.f ? 1.4426950408889634074 / (double)temp : 0.0, row.offset = row.rate * (double)row.top, row.powers = sh.powers;
  const uint32_t top_key = best;

  // A block's sum of `counts`, warps over consecutive chunks whose sums stay in sh.sums.
  const uint32_t chunk = ((n + SM_WARPS - 1) / SM_WARPS + 7) / 8 * 8;
  auto counted = [&](auto counts) {
    const uint32_t b0 = min(n, warp * chunk), b1 = min(n, b0 + chunk);
    u64 v = 0;
    sweep(b0, b1, lane, 32, [&](uint32_t i, float x) { v += counts(i, x); });
    v = warp_sum(v);
    __syncthreads();
    if (lane == 0) sh.sums[warp] = v;
    __syncthreads();
    u64 t = 0;
    for (uint32_t w = 0; w < SM_WARPS; ++w) t += sh.sums[w];
    return t;
  };
  // Sums over the cluster: `stage` numbers the exchanges, so that none overwrites what is still read.
  auto exchange = [&](int stage, u64 mine, u64 &before) {  // all blocks' sum; `before`: that of the blocks before this one
    if (tid == 0) sh.part[stage] = mine;
    cl.sync();
    u64 total = 0;
    before = 0;
    for (uint32_t q = 0; q < C; ++q) {
      const u64 v = *cl.map_shared_rank(&sh.part[stage], q);
      if (q < rank) before += v;
      total += v;
    }
    return total;
  };
  // The first index (of the row) at which the running sum of `counts` over this block's part passes `target`; it lies in this part, and
  // counted(counts) came last.  The chunk where it happens is cut into one for each warp, and the warp where it happens walks its own.
  auto locate = [&](u64 target, auto counts) {
    uint32_t w = 0;
    for (; w + 1 < SM_WARPS && sh.sums[w] <= target; ++w) target -= sh.sums[w];
    const uint32_t c0 = min(n, w * chunk), c1 = min(n, c0 + chunk), each = (c1 - c0 + SM_WARPS - 1) / SM_WARPS;
    const uint32_t b0 = min(c1, c0 + warp * each), b1 = min(c1, b0 + each);
    u64 sum = 0;
    for (uint32_t i = b0 + lane; i < b1; i += 32) sum += counts(i, logit(i));
    sum = warp_sum(sum);
    __syncthreads();
    if (lane == 0) sh.sums[warp] = sum;
    __syncthreads();
    u64 before = 0;
    for (uint32_t q = 0; q < warp; ++q) before += sh.sums[q];
    if (before <= target && target < before + sum) {
      for (uint32_t i0 = b0; i0 < b1; i0 += 32) {
        const u64 upto = before + warp_before(i0 + lane < b1 ? counts(i0 + lane, logit(i0 + lane)) : 0);
        const uint32_t past = __ballot_sync(0xffffffffu, upto > target);
        if (past) {
          if (lane == 0) sh.found_s = i0 + __ffs(past) - 1;
          break;
        }
        before = __shfl_sync(0xffffffffu, upto, 31);
      }
    }
    __syncthreads();
    return a + sh.found_s;
  };
  // the same over the cluster: every block learns the index
  auto find = [&](int stage, u64 mine, u64 target, auto counts) {
    u64 before;
    (void)exchange(stage, mine, before);
    if (before <= target && target < before + mine) {
      const uint32_t at = locate(target - before, counts);
      if (tid < C) cl.map_shared_rank(&sh, tid)->tally[stage] = at;
    }
    cl.sync();
    return sh.tally[stage];
  };

  if (bad || row.top == -INFINITY) {
    if (rank == 0 && tid == 0) {
      if (bad) paged_report(d.status, CUTB_ERR_INVALID);
      d.tokens[r] = CUTB_NO_TOKEN;
      if (d.logprobs) d.logprobs[r] = -INFINITY;
    }
    cl.sync();
    return;
  }
  SmCut cut{0, d.vocab};
  uint32_t buffer = 0;
  // Places of the falling order: 2048 of the weights' exponents over 43.5 (the last: no weight).  clear() gives a histogram of WORDS times
  // SM_BINS, the two in turn; crossing() the place in the cluster's sum of them where goal(their total) is reached, `target`: what is left of
  // that there, and what is there.
  const float scale = (float)row.rate * (2 * (SM_BINS - 1) / 43.5f), half = 0.5f * row.top;  // (half the distance: two finite logits may be infinitely far apart)
  auto place = [&](float v) { return min(SM_BINS - 1, __float2uint_rd(fmaf(-0.5f, v, half) * scale)); };  // (what is not a number: 0)
  auto clear = [&](uint32_t words) {
    uint32_t *h = hist + buffer * 3 * SM_BINS;
    buffer ^= 1;
    for (uint32_t i = tid; i < words * SM_BINS / 4; i += SM_THREADS) reinterpret_cast<uint4 *>(h)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    return h;
  };
  auto crossing = [&](auto words_type, uint32_t *h, auto goal, u64 &target, u64 &there) {
    constexpr uint32_t WORDS = decltype(words_type)::value;
    if (tid == 0) sh.bin_s = SM_BINS;
    cl.sync();
    u64 mine[4] = {0, 0, 0, 0};
#pragma unroll
    for (uint32_t q = 0; q < 8; ++q) {  // (all loads on their way before the first is needed)
      if (q >= C) continue;
      const uint32_t *o = cl.map_shared_rank(h, q) + 4 * tid;
#pragma unroll
      for (uint32_t w = 0; w < WORDS; ++w) {
        const uint4 e = *reinterpret_cast<const uint4 *>(o + w * SM_BINS);
        mine[0] += (u64)e.x << 16 * w, mine[1] += (u64)e.y << 16 * w, mine[2] += (u64)e.z << 16 * w, mine[3] += (u64)e.w << 16 * w;
      }
    }
    const u64 sum = mine[0] + mine[1] + mine[2] + mine[3], upto = warp_before(sum);
    if (lane == 31) sh.sums[warp] = upto;
    __syncthreads();
    u64 before = upto - sum, total = 0;
    for (uint32_t w = 0; w < SM_WARPS; ++w) {
      if (w == warp) before += total;
      total += sh.sums[w];
    }
    target = goal(total);
    if (before <= target && target < before + sum) {
      uint32_t b = 0;
      for (; b < 3 && before + mine[b] <= target; ++b) before += mine[b];
      sh.bin_s = 4 * tid + b, sh.left_s = target - before, sh.bin_sum = mine[b];
    }
    __syncthreads();
    const uint32_t bin = sh.bin_s;
    target = sh.left_s, there = sh.bin_sum;
    return bin;
  };
  // The tokens that `wanted` names, {key, ~index} in no order, in a list of the first block's (in the histogram that is not in use): how many
  // there are, of which the list has the first SM_LIST.  sh.many_s is 0 in every block before the barrier that came last, and stays until the next.
  u64 *list = nullptr;
  auto gather = [&](auto wanted) {
    list = reinterpret_cast<u64 *>(hist + buffer * 3 * SM_BINS);
    u64 *to = cl.map_shared_rank(list, 0);
    uint32_t *many_at = cl.map_shared_rank(&sh.many_s, 0);
    sweep(0, n, tid, SM_THREADS, [&](uint32_t i, float v) {
      if (!wanted(i, v)) return;
      const auto together = cg::coalesced_threads();  // (rows of equal logits want every place)
      uint32_t at = 0;
      if (together.thread_rank() == 0) at = atomicAdd(many_at, together.size());
      at = together.shfl(at, 0) + together.thread_rank();
      if (at < SM_LIST) to[at] = (u64)sm_key(v) << 32 | ~(a + i);
    });
    cl.sync();
    return *many_at;
  };
  // The key whose place in the falling order is where goal(all) of the kept counts (COUNT) or weights has gone by; `left`: what of it
  // is left at that key, `there`: what is there.  Only tokens with a weight count; false: fewer than the target do.
  // First by the weights' exponents, then by comparing the tokens at that place, or where they are many by their keys, 11 bits at a time.
  auto select = [&](auto count_type, auto goal, uint32_t &key, u64 &left, u64 &there) {
    constexpr bool COUNT = decltype(count_type)::value;
    constexpr std::integral_constant<uint32_t, COUNT ? 1 : 3> words;
    auto add = [&](uint32_t *h, float v) {
      if (COUNT) {
        atomicAdd(h, 1u);
      } else {
        const u64 m = row.mass(v);
        if (m & 0xffffu) atomicAdd(h, (uint32_t)m & 0xffffu);
        if (m >> 16 & 0xffffu) atomicAdd(h + SM_BINS, (uint32_t)(m >> 16) & 0xffffu);
        if (m >> 32) atomicAdd(h + 2 * SM_BINS, (uint32_t)(m >> 32));
      }
    };
    uint32_t *h = clear(words.value);
    if (tid == 0) sh.range[0] = 0xffffffffu, sh.range[1] = 0, sh.many_s = 0;
    sweep(0, n, tid, SM_THREADS, [&](uint32_t i, float v) {
      const uint32_t b = place(v);
      if (b < SM_BINS - 1 && cut.keeps(sm_key(v), a + i)) add(h + b, v);
    });
    u64 target;
    const uint32_t bin = crossing(words, h, goal, target, there);
    if (bin == SM_BINS) return false;
    const uint32_t many = gather([&](uint32_t i, float v) {
      const uint32_t c = sm_key(v);
      if (place(v) != bin || !cut.keeps(c, a + i)) return false;
      atomicMin(&sh.range[0], top_key - c), atomicMax(&sh.range[1], top_key - c);
      return true;
    });
    if (many <= SM_LIST) {  // every block compares them all (64 x 32000 fp32 logits with top-p took 54 us by steps over the keys, then 37)
      u64 *masses = list + SM_LIST;
      const u64 entry = tid < many ? cl.map_shared_rank(list, 0)[tid] : 0;
      const uint32_t own = (uint32_t)(entry >> 32);
      if (tid < many) masses[tid] = COUNT ? 1 : row.mass(sm_value(own));
      if (rank && tid < many) list[tid] = entry;
      __syncthreads();
      if (tid < many) {
        u64 ahead = 0, same = 0;
#pragma unroll 4
        for (uint32_t j = 0; j < many; ++j) {
          const uint32_t o = (uint32_t)(list[j] >> 32);
          const u64 m = masses[j];
          ahead += o > own ? m : 0, same += o == own ? m : 0;
        }
        if (ahead <= target && target < ahead + same) sh.bin_s = own, sh.left_s = target - ahead, sh.bin_sum = same;  // (equal ones write the same)
      }
      __syncthreads();
      key = sh.bin_s, left = sh.left_s, there = sh.bin_sum;
      cl.sync();  // (the list is read)
      return true;
    }
    uint32_t base = 0xffffffffu, end = 0;
    for (uint32_t q = 0; q < C; ++q) base = min(base, cl.map_shared_rank(sh.range, q)[0]), end = max(end, cl.map_shared_rank(sh.range, q)[1]);
    uint32_t shift = end - base < SM_BINS ? 0 : 21 - __clz(end - base);
    for (bool more = end != base; more;) {
      h = clear(words.value);
      sweep(0, n, tid, SM_THREADS, [&](uint32_t i, float v) {
        const uint32_t c = sm_key(v), diff = top_key - c;
        if (diff >= base && (diff - base) >> shift < SM_BINS && diff <= end && cut.keeps(c, a + i)) add(h + ((diff - base) >> shift), v);
      });
      base += crossing(words, h, [&](u64) { return target; }, target, there) << shift;
      end = min(end, base + ((1u << shift) - 1));
      more = shift != 0;
      shift = shift > 11 ? shift - 11 : 0;
      __syncthreads();  // (the next step writes what this one has read)
    }
    key = top_key - base, left = target;
    cl.sync();  // (the ranges are read)
    return true;
  };

  bool rest;
  const u64 share = least > 0.f && least < 1.f ? sm_share(least, 1ull << 42, rest) : 0, fewest = least >= 1.f ? ~0ull : share + (share && rest);
  auto log_share = [&](float v, u64 total) {
    return (float)((v == row.top ? 0.0 : ((double)v - (double)row.top) / (double)temp) - log((double)total / SM_ONE));
  };
  // The rest of the work by the first block alone, where the list has every token that may be kept, `many` of them, of which the `limit` first
  // in the falling order are: a thread has one, and finds its place in that order and in the indices' by comparing.
  auto finish = [&](uint32_t many, uint32_t limit) {
    const bool have = tid < many;
    const u64 own = have ? list[tid] : 0;
    const float value = sm_value((uint32_t)(own >> 32));
    u64 *masses = list + SM_LIST;
    const u64 mass = have ? row.mass(value) : 0;
    masses[tid] = mass;
    auto block_sum = [&](u64 v) {
      v = warp_sum(v);
      __syncthreads();
      if (lane == 0) sh.sums[warp] = v;
      __syncthreads();
      u64 t = 0;
      for (uint32_t w = 0; w < SM_WARPS; ++w) t += sh.sums[w];
      return t;
    };
    __syncthreads();
    u64 ahead = 0;  // the weight before this token in the falling order
    uint32_t at = have ? 0 : limit;
    if (have)
#pragma unroll 4
      for (uint32_t j = 0; j < many; ++j) {
        const bool before = list[j] > own;
        ahead += before ? masses[j] : 0, at += before;
      }
    const u64 all = block_sum(at < limit ? mass : 0);
    bool keeps = at < limit && (mass >= fewest || value == row.top);
    if (p < 1.f && ahead > sm_before(p, all)) keeps = false;
    const u64 left = keeps ? mass : 0, total = block_sum(left);
    masses[tid] = left;  // (block_sum: the weights are read)
    __syncthreads();
    if (!left) return;
    u64 before = 0;
#pragma unroll 4
    for (uint32_t j = 0; j < many; ++j) before += (uint32_t)list[j] > (uint32_t)own ? masses[j] : 0;  // (~index)
    const u64 target = sm_share(u, total, rest);
    if (before <= target && target < before + left) {
      d.tokens[r] = ~(uint32_t)own;
      if (d.logprobs) d.logprobs[r] = log_share(value, total);
    }
  };

  if (temp == 0.f || least > 1.f) {  // (no weight comes up to more than the largest: its first place is kept)
    auto f = [&](uint32_t, float v) { return (u64)(v == row.top); };
    cut = SmCut{top_key, find(0, counted(f), 0, f)};
  } else {
    if (k && k < d.vocab) {
      u64 left, there;
      auto goal = [&](u64) -> u64 { return k - 1; };
      if (k <= SM_LIST / 2) {
        // Each thread's largest logit is known: the place of the k-th of those is not before that of the k-th logit, and few tokens come up to it
        // (256 x 128256 with k = 50: 44 us; by a histogram of all logits 211).
        uint32_t *h = clear(1);
        if (tid == 0) sh.many_s = 0;
        const uint32_t b = place(sm_logit(highest));
        if (b < SM_BINS - 1) atomicAdd(h + b, 1u);
        const uint32_t bin = crossing(std::integral_constant<uint32_t, 1>(), h, goal, left, there);
        if (bin < SM_BINS) {
          const uint32_t many = gather([&](uint32_t, float v) { return place(v) <= bin; });
          if (many <= SM_LIST) {
            if (rank == 0) finish(many, k);
            cl.sync();  // (every block has read the first one's count)
            return;
          }
          cl.sync();
        }
      }
      uint32_t key;
      if (select(std::true_type(), goal, key, left, there)) {
        cut = SmCut{key, d.vocab};
        if (left + 1 < there) {  // some of several equal ones
          auto f = [&](uint32_t, float v) { return (u64)(sm_key(v) == key); };
          cut.last = find(0, counted(f), left, f);
        }
        if (k <= SM_LIST) {
          if (tid == 0) sh.many_s = 0;
          cl.sync();
          const uint32_t many = gather([&](uint32_t i, float v) { return cut.keeps(sm_key(v), a + i); });
          if (rank == 0) finish(many, k);
          cl.sync();
          return;
        }
      }
    }
    if (p < 1.f) {
      u64 left, there;
      uint32_t key;
      (void)select(std::false_type(), [&](u64 total) { return sm_before(p, total); }, key, left, there);  // (the largest logit has a weight)
      const u64 one = row.mass(sm_value(key)), ties = one ? left / one : 0;  // kept before the last one
      const SmCut was = cut;
      cut = SmCut{key, key == was.key ? was.last : d.vocab};
      if ((ties + 1) * one < there) {
        auto g = [&](uint32_t i, float v) { return (u64)(sm_key(v) == key && was.keeps(key, a + i)); };
        cut.last = find(2, counted(g), ties, g);
      }
    }
  }
  auto draw = [&](auto kept) {
    const u64 mine = counted(kept);
    u64 before;
    const u64 total = exchange(3, mine, before);
    const u64 target = sm_share(u, total, rest);
    if (before <= target && target < before + mine) {
      const uint32_t token = locate(target - before, kept);
      if (tid == 0) {
        d.tokens[r] = token;
        if (d.logprobs) d.logprobs[r] = temp == 0.f ? 0.f : log_share(logit(token - a), total);
      }
    }
  };
  if (cut.key == 0 && fewest == 0) {
    draw([&](uint32_t, float v) -> u64 { return row.mass(v); });
  } else {
    draw([&](uint32_t i, float v) -> u64 {
      if (!cut.keeps(sm_key(v), a + i)) return 0;
      const u64 m = row.mass(v);
      return v == row.top || m >= fewest ? m : 0;
    });
  }
  cl.sync();  // the other blocks read this one's sums
}

// Blocks of a row: more than one where the rows alone would leave SMs without work, eight at most (which is what every device can launch
// together) and no fewer than 8192 logits to each (1 x 32000 fp32 logits, four blocks and eight: with every cut-off 9.9 and 10.9 us, with
// none 7.8 and 6.6).
uint32_t sm_cluster(uint32_t rows, uint32_t vocab, uint32_t sms) {
  uint32_t c = 1;
  while (c < 8 && ((uint64_t)rows * c < sms || (uint64_t)c * 65536 < vocab) && c * 8192u < vocab) c *= 2;
  return c;
}

template <typename T, bool RESIDENT> int sm_launch(const cutb_sample_desc &d, uint32_t cluster, uint32_t part, uint32_t smem, cudaStream_t stream) {
  // (one limit for all calls: another thread's may be set between this call's and its launch)
  CUTB_CUDA_TRY(cudaFuncSetAttribute(sample_kernel<T, RESIDENT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SM_SHARED));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(d.rows * cluster), cfg.blockDim = dim3(SM_THREADS), cfg.dynamicSmemBytes = smem, cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr, cfg.numAttrs = 2;
  CUTB_CUDA_TRY(cudaLaunchKernelEx(&cfg, sample_kernel<T, RESIDENT>, d, part));
  return CUTB_OK;
}

}  // namespace

int sample_launch(const cutb_sample_desc &d, cudaStream_t stream) {
  DeviceInfo di;
  if (int rc = get_device_info(&di)) return rc;
  const uint32_t cluster = sm_cluster(d.rows, d.vocab, di.sm_count), part = ((d.vocab + cluster - 1) / cluster + 7) / 8 * 8;
  const uint32_t hist = d.top_k || d.top_p ? 2 * 3 * SM_BINS * 4 : 0;
  const bool resident = (uint64_t)part * 4 + hist <= SM_SHARED;
  return paged_with_type(d.dtype, [&](auto t) {
    using T = decltype(t);
    return resident ? sm_launch<T, true>(d, cluster, part, (part * 4 + 15) / 16 * 16 + hist, stream) : sm_launch<T, false>(d, cluster, part, hist, stream);
  });
}

}  // namespace cutb

using namespace cutb;

extern "C" int cutb_sample(const cutb_sample_desc *d, void *stream) {
  if (!d || (d->dtype != CUTB_F32 && d->dtype != CUTB_F16 && d->dtype != CUTB_BF16)) {
    set_last_error("sample: null descriptor, or an element type that is not fp32, fp16 or bf16");
    return CUTB_ERR_INVALID;
  }
  if (d->rows == 0) return CUTB_OK;
  if (d->vocab == 0 || d->vocab > SM_VOCAB || (d->rows > 1 && d->ld < d->vocab) || d->rows > (1u << 24)) {
    set_last_error("sample: a row has 1 .. 524288 logits and a stride that holds them (vocab=%u ld=%llu)", d->vocab, (unsigned long long)d->ld);
    return CUTB_ERR_INVALID;
  }
  if (!d->logits || !d->u || !d->tokens || reinterpret_cast<uintptr_t>(d->logits) % (d->dtype == CUTB_F32 ? 4 : 2)) {
    set_last_error("sample: null pointer or misaligned logits");
    return CUTB_ERR_INVALID;
  }
  const void *words[] = {d->temperature, d->top_k, d->top_p, d->min_p, d->u, d->tokens, d->logprobs, d->status};
  for (const void *p : words)
    if (reinterpret_cast<uintptr_t>(p) % 4) {
      set_last_error("sample: settings and results are 4-byte aligned");
      return CUTB_ERR_INVALID;
    }
  return sample_launch(*d, reinterpret_cast<cudaStream_t>(stream));
}
