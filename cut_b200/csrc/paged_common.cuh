// Layout of the paged 4-bit cache, and what its kernels share: the sequences of a call, element types, dequantisation.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace cutb {
namespace {

constexpr uint32_t PG_UNIT = 16;       // tokens of a unit
constexpr uint32_t PG_MAX_SEQS = 1024;  // sequences of a call
constexpr float PG_LIMIT = 32768.f;    // what a cached element may hold: 15 d + m stays below fp16's largest number

__host__ __device__ constexpr uint32_t pg_pad(uint32_t head_dim) { return (head_dim + 63) / 64 * 64; }
__host__ __device__ constexpr uint32_t pg_unit_bytes(uint32_t dp) { return 20 * dp; }
// offsets within a unit: keys, values (bytes), scales of the keys and of the values (bytes)
__host__ __device__ constexpr uint32_t pg_values_at(uint32_t dp) { return 8 * dp; }
__host__ __device__ constexpr uint32_t pg_key_scales_at(uint32_t dp) { return 16 * dp; }
__host__ __device__ constexpr uint32_t pg_value_scales_at(uint32_t dp) { return 18 * dp; }
// the word of token t that holds elements 32 j + 8 b .. + 7 of its key: the words that one lane of four (b) of an MMA fragment needs lie together
__host__ __device__ constexpr uint32_t pg_key_word(uint32_t dp, uint32_t t, uint32_t j, uint32_t b) {
  const uint32_t w = dp % 128 == 0 ? 4 : 2;
  return t * (dp / 8) + j / w * 4 * w + b * w + j % w;
}
// bit of element e of such a word: pairs of elements 16 bits apart, so that two logic operations give fp16 pairs in their order
__host__ __device__ constexpr uint32_t pg_key_bit(uint32_t e) { return (e & 1) * 16 + (e >> 1 & 1) * 4 + (e >> 2) * 8; }
// the byte of token t that holds elements 16 i + r (low half) and 16 i + r + 8 of its value, r < 8: a word is a lane's MMA fragment
__host__ __device__ constexpr uint32_t pg_value_byte(uint32_t t, uint32_t i, uint32_t r) {
  return 4 * (i / 4 * 128 + (r * 4 + t / 4) * 4 + i % 4) + (t & 1) * 2 + (t >> 1 & 1);
}

#ifdef __CUDACC__

// One sequence of a call: its table row, its length, its rows.  rows = 0 where it is empty or cannot be served (bad).
struct PagedSeq {
  uint32_t slot, len, row0, rows;
  bool bad;
};
__device__ __forceinline__ PagedSeq paged_seq(const cutb_paged_desc &d, uint32_t s) {
  PagedSeq q;
  q.row0 = d.starts ? d.starts[s] : s;
  const uint32_t end = d.starts ? d.starts[s + 1] : s + 1;
  q.slot = d.slots ? d.slots[s] : s;
  q.bad = end < q.row0 || end > d.n_tokens || end - q.row0 > d.max_new || q.slot >= d.n_slots;
  q.rows = q.bad ? 0 : end - q.row0;
  q.len = q.slot < d.n_slots ? d.lengths[q.slot] : 0;
  if (q.rows && (q.len < q.rows || q.len > d.ld_table * d.page_tokens)) q.bad = true, q.rows = 0;
  return q;
}
__device__ __forceinline__ void paged_report(int *status, int code) {
  if (status) atomicExch(status, code);
}
// The last sequence that starts at or before `row`, by a whole warp (every lane gets it); n_seqs if there is none.
__device__ __forceinline__ uint32_t paged_seq_of(const cutb_paged_desc &d, uint32_t row) {
  if (!d.starts) return row < d.n_seqs ? row : d.n_seqs;
  const uint32_t lane = threadIdx.x & 31;
  uint32_t lo = 0, hi = d.n_seqs;
  for (;;) {  // 32 places at a time
    const uint32_t step = (hi - lo + 31) / 32, at = lo + lane * step;
    const uint32_t n = __popc(__ballot_sync(0xffffffffu, at < hi && d.starts[min(at, hi - 1)] <= row));
    if (n == 0) return d.n_seqs;
    lo += (n - 1) * step, hi = min(lo + step, hi);
    if (step == 1) return lo;
  }
}

// This thread's warp, as a number that the compiler knows to be the same in all of its lanes.  Where roles are told apart by threadIdx.x / 32
// it must expect lanes that have parted: a shuffle then takes 230 cycles instead of 25, and every vote and matrix instruction as much.  (So it must
// behind a wait that one lane makes for the others: prompts of 8192 tokens 886 us with such waits, 700 with warp_wait.)
__device__ __forceinline__ uint32_t warp_index() { return __shfl_sync(0xffffffffu, threadIdx.x / 32, 0); }
template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f(float v) { return v; }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }

// Eight nibbles of a word as four pairs of the fp16 numbers d q + m: bits of q under the exponent of 1024 are 1024 + q (or 1024 + 16 q),
// from which q comes back exactly; the last step rounds once.
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {  // a & b | c, one instruction
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ void pg_quants(uint32_t w, __half2 (&q)[4]) {
  const __half2 k1024 = u32_as_h2(0x64006400u), k16th = u32_as_h2(0x2c002c00u), k64 = u32_as_h2(0xd400d400u);  // 1024, 1 / 16, -64
  const uint32_t v = w >> 8;
  q[0] = __hsub2(u32_as_h2(and_or(w, 0x000f000fu, 0x64006400u)), k1024);
  q[1] = __hfma2(u32_as_h2(and_or(w, 0x00f000f0u, 0x64006400u)), k16th, k64);
  q[2] = __hsub2(u32_as_h2(and_or(v, 0x000f000fu, 0x64006400u)), k1024);
  q[3] = __hfma2(u32_as_h2(and_or(v, 0x00f000f0u, 0x64006400u)), k16th, k64);
}

#endif  // __CUDACC__

}  // namespace

#ifdef __CUDACC__
// runs `f` with the element type of `dtype`
template <typename F> int paged_with_type(int dtype, F f) {
  if (dtype == CUTB_F32) return f(float());
  if (dtype == CUTB_F16) return f(__half());
  return f(__nv_bfloat16());
}
#endif

}  // namespace cutb
