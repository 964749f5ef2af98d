// The next token of each row of logits, by a given random number.
#include "kernels.h"
#include "paged_common.cuh"

namespace cutb {
namespace {

constexpr uint32_t SM_THREADS = 1024, SM_WARPS = 32;
constexpr double SM_ONE = 4398046511104.0;  // 2^42: weights are added as integers of 2^-42, up to 2^20 of them
typedef unsigned long long u64;

// A logit as it counts: a NaN is minus infinity, minus zero is zero.
template <typename T> __device__ __forceinline__ float sm_logit(const T *x, uint32_t i) {
  const float v = to_f(x[i]) + 0.f;
  return v != v ? -INFINITY : v;
}
// larger logits have larger keys
__device__ __forceinline__ uint32_t sm_key(float v) {
  const uint32_t b = __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float sm_value(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }

struct SmRow {
  float top;
  double rate;  // 1 / temperature
  double least;
  __device__ __forceinline__ double weight(float v) const {
    if (v == top) return 1.0;  // (an infinite one too)
    return exp(((double)v - (double)top) * rate);
  }
  __device__ __forceinline__ u64 mass(float v) const { return (u64)__double2ll_rn(weight(v) * SM_ONE); }
};

// Sum over the block, to all of its threads.
__device__ __forceinline__ u64 sm_sum(u64 v, u64 *warps) {
#pragma unroll
  for (int o = 16; o; o /= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x / 32] = v;
  __syncthreads();
  u64 t = warps[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o; o /= 2) t += __shfl_xor_sync(0xffffffffu, t, o);
  return t;
}

// What is kept so far: keys above `key`, and of those equal to it the ones up to index `last`.
struct SmCut {
  uint32_t key, last;
  __device__ __forceinline__ bool keeps(uint32_t k, uint32_t i) const { return k > key || (k == key && i <= last); }
};

// The first index, counted over the places where `counts(i)` is above zero, at which the running sum passes `target`: warps take
// consecutive parts, the one where it happens walks its part.
template <typename F> __device__ uint32_t sm_find(uint32_t n, u64 target, u64 *warps, uint32_t *found, F counts) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32, part = (n + SM_WARPS - 1) / SM_WARPS, a = min(n, warp * part), b = min(n, a + part);
  u64 sum = 0;
  for (uint32_t i = a + lane; i < b; i += 32) sum += counts(i);
#pragma unroll
  for (int o = 16; o; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __syncthreads();
  if (lane == 0) warps[warp] = sum;
  if (threadIdx.x == 0) *found = 0xffffffffu;
  __syncthreads();
  u64 before = 0;
  for (uint32_t w = 0; w < warp; ++w) before += warps[w];
  if (before <= target && target < before + sum) {
    for (uint32_t i0 = a; i0 < b; i0 += 32) {
      u64 x = i0 + lane < b ? counts(i0 + lane) : 0;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const u64 y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, before + x > target);
      if (past) {
        if (lane == 0) *found = i0 + __ffs(past) - 1;
        break;
      }
      before += __shfl_sync(0xffffffffu, x, 31);
    }
  }
  __syncthreads();
  return *found;
}

// One block per row.
template <typename T> __global__ void __launch_bounds__(SM_THREADS) sample_kernel(const __grid_constant__ cutb_sample_desc d) {
  __shared__ u64 warps[SM_WARPS], bins[256], left_s;
  __shared__ uint32_t found_s, digit_s;
  pdl_enter();
  const uint32_t r = blockIdx.x, n = d.vocab, tid = threadIdx.x;
  const T *x = reinterpret_cast<const T *>(d.logits) + r * d.ld;
  const float temp = d.temperature ? d.temperature[r] : 1.f, p = d.top_p ? d.top_p[r] : 1.f, least = d.min_p ? d.min_p[r] : 0.f, u = d.u[r];
  const uint32_t k = d.top_k ? d.top_k[r] : 0;
  const bool bad = !(temp >= 0.f && temp < INFINITY) || p != p || least != least || !(u >= 0.f && u < 1.f);
  uint32_t best = 0;
  for (uint32_t i = tid; i < n; i += SM_THREADS) best = max(best, sm_key(sm_logit(x, i)));
#pragma unroll
  for (int o = 16; o; o /= 2) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if (tid == 0) found_s = 0;
  __syncthreads();
  if ((tid & 31) == 0) atomicMax(&found_s, best);
  __syncthreads();
  SmRow row;
  row.top = sm_value(found_s), row.rate = temp > 0.f ? 1.0 / (double)temp : 0.0, row.least = least;
  __syncthreads();
  if (bad || row.top == -INFINITY) {
    if (tid == 0) {
      if (bad) paged_report(d.status, CUTB_ERR_INVALID);
      d.tokens[r] = CUTB_NO_TOKEN;
      if (d.logprobs) d.logprobs[r] = -INFINITY;
    }
    return;
  }
  SmCut cut{0, n};
  if (temp == 0.f) {
    cut = SmCut{sm_key(row.top), sm_find(n, 0, warps, &found_s, [&](uint32_t i) { return (u64)(sm_logit(x, i) == row.top); })};
  } else {
    // the key whose place in the falling order is where `target` of the kept counts (or weights) has gone by, digit by digit; `left`:
    // what of the target is left at that key
    auto select = [&](u64 target, auto measure, u64 &left) {
      uint32_t key = 0, mask = 0;
      for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) bins[tid] = 0;
        __syncthreads();
        for (uint32_t i = tid; i < n; i += SM_THREADS) {
          const float v = sm_logit(x, i);
          const uint32_t c = sm_key(v);
          if ((c & mask) == key && cut.keeps(c, i)) atomicAdd(&bins[c >> shift & 255u], measure(v));
        }
        __syncthreads();
        if (tid == 0) {
          int b = 255;
          for (; b > 0 && bins[b] <= target; --b) target -= bins[b];
          digit_s = b, left_s = target;
        }
        __syncthreads();
        key |= digit_s << shift, mask |= 255u << shift, target = left_s;
      }
      left = target;
      return key;
    };
    if (k && k < n) {
      u64 left;
      const uint32_t key = select(k - 1, [](float) { return u64(1); }, left);
      cut = SmCut{key, sm_find(n, left, warps, &found_s, [&](uint32_t i) { return (u64)(sm_key(sm_logit(x, i)) == key); })};
    }
    if (p < 1.f) {
      u64 total = 0;
      for (uint32_t i = tid; i < n; i += SM_THREADS) {
        const float v = sm_logit(x, i);
        if (cut.keeps(sm_key(v), i)) total += row.mass(v);
      }
      total = sm_sum(total, warps);
      // a token is kept while the weight before it is below the target, a number above zero
      const double want = fmax((double)p, 0.0) * (double)total;
      const u64 target = want > 1.0 ? (u64)ceil(want) - 1 : 0;
      u64 left;
      const uint32_t key = select(target, [&](float v) { return row.mass(v); }, left);
      const u64 one = row.mass(sm_value(key));
      const u64 ties = one ? left / one : 0;  // kept before the last one
      cut = SmCut{key, sm_find(n, ties, warps, &found_s, [&](uint32_t i) {
                    const uint32_t c = sm_key(sm_logit(x, i));
                    return (u64)(c == key && cut.keeps(c, i));
                  })};
    }
  }
  auto kept = [&](uint32_t i) {
    const float v = sm_logit(x, i);
    return cut.keeps(sm_key(v), i) && (v == row.top || row.weight(v) >= row.least) ? row.mass(v) : 0;
  };
  u64 total = 0;
  for (uint32_t i = tid; i < n; i += SM_THREADS) total += kept(i);
  total = sm_sum(total, warps);
  const u64 target = (u64)floor((double)u * (double)total);
  const uint32_t token = sm_find(n, target, warps, &found_s, kept);
  if (tid == 0) {
    d.tokens[r] = token;
    if (d.logprobs) d.logprobs[r] = temp == 0.f ? 0.f : (float)log(row.weight(sm_logit(x, token)) * (SM_ONE / (double)total));
  }
}

}  // namespace

int sample_launch(const cutb_sample_desc &d, cudaStream_t stream) {
  return paged_with_type(d.dtype, [&](auto t) {
    using T = decltype(t);
    CUTB_CUDA_TRY(launch_pdl(sample_kernel<T>, dim3(d.rows), dim3(SM_THREADS), 0, stream, d));
    return (int)CUTB_OK;
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
  if (d->vocab == 0 || d->vocab > (1u << 20) || (d->rows > 1 && d->ld < d->vocab) || d->rows > 0x7fffffffu) {
    set_last_error("sample: a row has 1 .. 1048576 logits and a stride that holds them (vocab=%u ld=%llu)", d->vocab, (unsigned long long)d->ld);
    return CUTB_ERR_INVALID;
  }
  if (!d->logits || !d->u || !d->tokens || reinterpret_cast<uintptr_t>(d->logits) % (d->dtype == CUTB_F32 ? 4 : 2)) {
    set_last_error("sample: null pointer or misaligned logits");
    return CUTB_ERR_INVALID;
  }
  return sample_launch(*d, reinterpret_cast<cudaStream_t>(stream));
}
