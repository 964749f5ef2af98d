// The paged 4-bit cache: rows written and read back, and the bookkeeping of its pages.
#include "kernels.h"
#include "paged_common.cuh"

namespace cutb {
namespace {

// ---- rows --------------------------------------------------------------------------------------------------------------
// A lane holds four neighbouring elements of every 128 of a head, so that the eight lanes of a group of 32 meet in three shuffles and
// two lanes make a word.
template <typename T> __device__ __forceinline__ void load4(const T *p, uint32_t i, uint32_t n, bool vec, float (&x)[4]) {
  if (vec) {
    if (i >= n) {
      x[0] = x[1] = x[2] = x[3] = 0.f;
    } else if constexpr (sizeof(T) == 4) {
      const float4 f = __ldg(reinterpret_cast<const float4 *>(p + i));
      x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
    } else {
      const uint2 u = __ldg(reinterpret_cast<const uint2 *>(p + i));
      const T *e = reinterpret_cast<const T *>(&u);
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = to_f(e[k]);
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) x[k] = i + k < n ? to_f(p[i + k]) : 0.f;
}

template <typename T> __device__ __forceinline__ void store4(T *p, uint32_t i, uint32_t n, bool vec, const float (&x)[4]) {
  if (vec) {
    if (i >= n) return;
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4 *>(p + i) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
      uint2 u;
      T *e = reinterpret_cast<T *>(&u);
#pragma unroll
      for (int k = 0; k < 4; ++k) e[k] = from_f<T>(x[k]);
      *reinterpret_cast<uint2 *>(p + i) = u;
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (i + k < n) p[i + k] = from_f<T>(x[k]);
}

// elements i .. i + 3 of a head, turned: products and sums rounded one by one
__device__ __forceinline__ float turned(bool first, float x, float z, float c, float s) {
  return first ? __fsub_rn(__fmul_rn(x, c), __fmul_rn(z, s)) : __fadd_rn(__fmul_rn(z, s), __fmul_rn(x, c));
}
template <typename T, bool VEC>
__device__ __forceinline__ void turned4(const cutb_paged_desc &d, const T *p, uint32_t i, uint32_t pos, float (&x)[4]) {
  load4(p, i, d.head_dim, VEC, x);
  if (i >= d.rot_dims) return;
  const uint32_t half = d.rot_dims / 2;
  const float *cs = d.cos_table + (uint64_t)pos * half, *sn = d.sin_table + (uint64_t)pos * half;
  float y[4];
  if (VEC) {  // (rot_dims is a multiple of 8)
    if (d.rot_pairing) {
      const float2 c = __ldg(reinterpret_cast<const float2 *>(cs + i / 2)), n = __ldg(reinterpret_cast<const float2 *>(sn + i / 2));
      y[0] = turned(true, x[0], x[1], c.x, n.x), y[1] = turned(false, x[1], x[0], c.x, n.x);
      y[2] = turned(true, x[2], x[3], c.y, n.y), y[3] = turned(false, x[3], x[2], c.y, n.y);
    } else {
      const bool first = i < half;
      const uint32_t t = first ? i : i - half;
      const float4 c = __ldg(reinterpret_cast<const float4 *>(cs + t)), n = __ldg(reinterpret_cast<const float4 *>(sn + t));
      float z[4];
      load4(p, first ? i + half : t, d.head_dim, true, z);
      y[0] = turned(first, x[0], z[0], c.x, n.x), y[1] = turned(first, x[1], z[1], c.y, n.y);
      y[2] = turned(first, x[2], z[2], c.z, n.z), y[3] = turned(first, x[3], z[3], c.w, n.w);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t e = i + k;
      y[k] = x[k];
      if (e >= d.rot_dims) continue;
      const bool first = d.rot_pairing ? (e & 1) == 0 : e < half;
      const uint32_t t = d.rot_pairing ? e / 2 : (first ? e : e - half), other = d.rot_pairing ? e ^ 1u : (first ? e + half : e - half);
      y[k] = turned(first, x[k], to_f(p[other]), __ldg(cs + t), __ldg(sn + t));
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) x[k] = y[k];
}

// Four elements of a group, its other ones in the lanes beside: their numbers, and d and m of the group.  rint((x - m) / d) by the
// reciprocal of d, whose result is off by less than 2^-18; where that could round to the other side, by the quotient itself.
struct Coded {
  uint32_t code[4];
  __half d, m;
};
__device__ __forceinline__ Coded coded4(float (&x)[4], uint32_t i, uint32_t n, bool &changed) {
  Coded r;
  float lo = INFINITY, hi = -INFINITY;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (i + k >= n) continue;
    const float c = x[k] != x[k] ? 0.f : fminf(fmaxf(x[k], -PG_LIMIT), PG_LIMIT);
    changed |= !(c == x[k]);
    x[k] = c, lo = fminf(lo, c), hi = fmaxf(hi, c);
  }
#pragma unroll
  for (int o = 1; o < 8; o *= 2) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  if (lo > hi) lo = hi = 0.f;  // a group of padding
  r.m = __float2half_rn(lo);
  const float mf = __half2float(r.m);
  r.d = __float2half_rn(fmaxf(__fdiv_rn(__fsub_rn(hi, mf), 15.f), 0.f));
  const float df = __half2float(r.d), inv = df > 0.f ? __frcp_rn(df) : 0.f;
  bool close = false;
  float v[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    v[k] = fminf(fmaxf(__fmul_rn(__fsub_rn(x[k], mf), inv), 0.f), 15.f);
    close |= fabsf(v[k] - floorf(v[k]) - 0.5f) < 1e-5f;
  }
  if (close)
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = fminf(fmaxf(__fdiv_rn(__fsub_rn(x[k], mf), df), 0.f), 15.f);
#pragma unroll
  for (int k = 0; k < 4; ++k) r.code[k] = i + k < n ? (uint32_t)rintf(v[k]) : 0u;
  return r;
}
__device__ __forceinline__ uint32_t key_word(const Coded &c, uint32_t i) {  // of this lane and the next
  uint32_t part = 0;
#pragma unroll
  for (uint32_t k = 0; k < 4; ++k) part |= c.code[k] << pg_key_bit((i + k) % 8);
  return part | __shfl_xor_sync(0xffffffffu, part, 1);
}
__device__ __forceinline__ uint32_t value_bytes(const Coded &c) {  // the partners of bytes, eight elements on, are two lanes on
  const uint32_t mine = c.code[0] | c.code[1] << 8 | c.code[2] << 16 | c.code[3] << 24;
  return mine | __shfl_xor_sync(0xffffffffu, mine, 2) << 4;
}

// A row's head into its unit: codes and scales of the keys or of the values, in the cache itself or in a copy of theirs.
template <typename T, bool VEC>
__device__ __forceinline__ void write_head(const cutb_paged_desc &d, const T *src, uint32_t pos, bool value, uint8_t *codes, uint8_t *scales, bool &changed) {
  const uint32_t lane = threadIdx.x & 31, dp = pg_pad(d.head_dim), t = pos % PG_UNIT, groups = dp / 32;
  for (uint32_t i0 = 0; i0 < dp; i0 += 128) {
    const uint32_t i = i0 + 4 * lane, g = i / 32;
    float x[4];
    if (value) load4(src, i, d.head_dim, VEC, x);
    else turned4<T, VEC>(d, src, i, pos, x);
    const Coded c = coded4(x, i, d.head_dim, changed);
    if (value) {
      const uint32_t bytes = value_bytes(c);
      if (i < dp && (lane & 2) == 0)
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) codes[pg_value_byte(t, i / 16, (i + k) % 8)] = (uint8_t)(bytes >> 8 * k);
      if (i < dp && (lane & 7) == 0) {
        __half *sc = reinterpret_cast<__half *>(scales) + 8 * (g * 4 + t / 4) + t % 4;
        sc[0] = c.d, sc[4] = c.m;
      }
    } else {
      const uint32_t word = key_word(c, i);
      if (i < dp && (lane & 1) == 0) reinterpret_cast<uint32_t *>(codes)[pg_key_word(dp, t, g, i % 32 / 8)] = word;
      if (i < dp && (lane & 7) == 0) *reinterpret_cast<__half2 *>(scales + 4 * (t * groups + g)) = __halves2half2(c.d, c.m);
    }
  }
}

// Where the codes (and scales) of a head's keys or values of the unit at `pos` lie.
struct Unit {
  uint8_t *codes, *scales;
};
__device__ __forceinline__ Unit unit_of(const cutb_paged_desc &d, uint32_t page, uint32_t kvh, uint32_t pos, bool value) {
  const uint32_t dp = pg_pad(d.head_dim);
  uint8_t *u = reinterpret_cast<uint8_t *>(d.pages) + (uint64_t)page * d.page_bytes +
               ((uint64_t)kvh * (d.page_tokens / PG_UNIT) + pos % d.page_tokens / PG_UNIT) * pg_unit_bytes(dp);
  return value ? Unit{u + pg_values_at(dp), u + pg_value_scales_at(dp)} : Unit{u, u + pg_key_scales_at(dp)};
}

// Few rows: a warp per head of a row.
template <typename T, bool VEC> __global__ void __launch_bounds__(256) paged_kv_write_kernel(const __grid_constant__ cutb_paged_desc d) {
  pdl_enter();
  const uint32_t lane = threadIdx.x & 31, heads = 2 * d.n_kv_heads + (d.q ? d.n_heads : 0);
  const uint64_t item = (uint64_t)blockIdx.x * 8 + warp_index();
  const uint32_t row = (uint32_t)(item / heads), h = (uint32_t)(item % heads);
  if (row >= d.n_tokens) return;
  const uint32_t s = paged_seq_of(d, row);
  if (s >= d.n_seqs) return;
  const PagedSeq sq = paged_seq(d, s);
  bool bad = sq.bad;
  if (!bad && row - sq.row0 >= sq.rows) return;  // behind the last sequence
  const uint32_t pos = sq.len - sq.rows + (row - sq.row0);
  uint32_t page = 0;
  if (!bad) {
    page = d.tables[sq.slot * d.ld_table + pos / d.page_tokens];
    bad = page >= d.n_pages || (d.rot_dims && pos >= d.max_pos);
  }
  if (bad) {
    if (lane == 0) paged_report(d.status, CUTB_ERR_INVALID);
    return;
  }
  if (h >= 2 * d.n_kv_heads) {  // a query
    const T *src = reinterpret_cast<const T *>(d.q) + row * d.ldq + (uint64_t)(h - 2 * d.n_kv_heads) * d.head_dim;
    T *dst = reinterpret_cast<T *>(d.q_out) + row * d.ldq_out + (uint64_t)(h - 2 * d.n_kv_heads) * d.head_dim;
    for (uint32_t i = 4 * lane; i < d.head_dim; i += 128) {
      float x[4];
      turned4<T, VEC>(d, src, i, pos, x);
      store4(dst, i, d.head_dim, VEC, x);
    }
    return;
  }
  const bool value = h >= d.n_kv_heads;
  const uint32_t kvh = value ? h - d.n_kv_heads : h;
  const T *src = reinterpret_cast<const T *>(value ? d.v : d.k) + row * (value ? d.ldv : d.ldk) + (uint64_t)kvh * d.head_dim;
  const Unit u = unit_of(d, page, kvh, pos, value);
  bool changed = false;
  write_head<T, VEC>(d, src, pos, value, u.codes, u.scales, changed);
  if (__any_sync(0xffffffffu, changed) && lane == 0) paged_report(d.status, CUTB_ERR_RANGE);
}

// The pieces of sequences that begin among rows 16 c .. 16 c + 15: from a sequence's first row or the first one of a unit to the unit's
// end.  f(first row, its position, rows, page), by the whole warp.
template <typename F> __device__ __forceinline__ void for_pieces(const cutb_paged_desc &d, uint32_t c, F f) {
  const uint32_t lane = threadIdx.x & 31, end = (uint32_t)min((uint64_t)c * PG_UNIT + PG_UNIT, (uint64_t)d.n_tokens);
  for (uint32_t row = c * PG_UNIT; row < end;) {
    const uint32_t s = paged_seq_of(d, row);
    if (s >= d.n_seqs) {  // (before the first sequence)
      ++row;
      continue;
    }
    const PagedSeq sq = paged_seq(d, s);
    if (sq.bad || row - sq.row0 >= sq.rows) {
      if (sq.bad && lane == 0) paged_report(d.status, CUTB_ERR_INVALID);
      if (!sq.bad && s + 1 == d.n_seqs) return;  // behind the last sequence
      ++row;
      continue;
    }
    const uint32_t first = sq.len - sq.rows, past = sq.row0 + sq.rows;
    uint32_t pos = first + (row - sq.row0);
    if (row != sq.row0 && pos % PG_UNIT) row += PG_UNIT - pos % PG_UNIT;
    while (row < min(end, past)) {
      pos = first + (row - sq.row0);
      const uint32_t n = min(PG_UNIT - pos % PG_UNIT, past - row), page = d.tables[sq.slot * d.ld_table + pos / d.page_tokens];
      if (page < d.n_pages) f(row, pos, n, page);
      else if (lane == 0) paged_report(d.status, CUTB_ERR_INVALID);
      row += n;
    }
    row = past;  // (the next unit may lie behind it, another sequence's first row before that)
  }
}

// ---- many rows: a lane holds eight elements of one row, sixteen lanes a row, so that a warp works on two rows at a time (what is
// computed once for a group of 32 elements, and the shuffles, count four times less than in the form above)
template <typename T, bool VEC> __device__ __forceinline__ void load8(const T *p, uint32_t i, uint32_t n, float (&x)[8]) {
  if constexpr (VEC) {
    if constexpr (sizeof(T) == 4) {
      const float4 *q = reinterpret_cast<const float4 *>(p + (i < n ? i : 0));
      const float4 a = __ldg(q), b = __ldg(q + 1);
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
      const uint4 u = __ldg(reinterpret_cast<const uint4 *>(p + (i < n ? i : 0)));
      const T *e = reinterpret_cast<const T *>(&u);
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = to_f(e[k]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = i + k < n ? to_f(p[i + k]) : 0.f;
  }
}
template <typename T, bool VEC> __device__ __forceinline__ void store8(T *p, uint32_t i, uint32_t n, const float (&x)[8]) {
  if constexpr (VEC) {
    if (i >= n) return;
    if constexpr (sizeof(T) == 4) {
      float4 *q = reinterpret_cast<float4 *>(p + i);
      q[0] = make_float4(x[0], x[1], x[2], x[3]), q[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      uint4 u;
      T *e = reinterpret_cast<T *>(&u);
#pragma unroll
      for (int k = 0; k < 8; ++k) e[k] = from_f<T>(x[k]);
      *reinterpret_cast<uint4 *>(p + i) = u;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k < n) p[i + k] = from_f<T>(x[k]);
  }
}
// What turns elements i .. i + 7 at a position: cosines and sines, element by element.
struct Turn {
  float c[8], n[8];
};
template <bool VEC> __device__ __forceinline__ void turn_at(const cutb_paged_desc &d, uint32_t i, uint32_t pos, Turn &turn) {
  if (d.rot_dims == 0) return;
  const uint32_t half = d.rot_dims / 2;
  const float *cs = d.cos_table + (uint64_t)pos * half, *sn = d.sin_table + (uint64_t)pos * half;
  if constexpr (VEC) {  // (no branches: the loads of several rows go out together)
    const bool on = i < d.rot_dims;
    if (d.rot_pairing) {  // (rot_dims is a multiple of 8)
      const uint32_t t = on ? i / 2 : 0;
      const float4 c = __ldg(reinterpret_cast<const float4 *>(cs + t)), n = __ldg(reinterpret_cast<const float4 *>(sn + t));
      turn.c[0] = turn.c[1] = c.x, turn.c[2] = turn.c[3] = c.y, turn.c[4] = turn.c[5] = c.z, turn.c[6] = turn.c[7] = c.w;
      turn.n[0] = turn.n[1] = n.x, turn.n[2] = turn.n[3] = n.y, turn.n[4] = turn.n[5] = n.z, turn.n[6] = turn.n[7] = n.w;
    } else {  // (of 16)
      const uint32_t t = on ? (i < half ? i : i - half) : 0;
      load8<float, true>(cs, t, half, turn.c);
      load8<float, true>(sn, t, half, turn.n);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t e = min(i + k, d.rot_dims - 1), t = d.rot_pairing ? e / 2 : (e < half ? e : e - half);
      turn.c[k] = __ldg(cs + t), turn.n[k] = __ldg(sn + t);
    }
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void turned8(const cutb_paged_desc &d, const T *p, uint32_t i, const Turn &turn, float (&x)[8]) {
  load8<T, VEC>(p, i, d.head_dim, x);
  if (d.rot_dims == 0) return;
  const uint32_t half = d.rot_dims / 2;
  float z[8];
  if (VEC && d.rot_pairing) {
#pragma unroll
    for (int k = 0; k < 8; ++k) z[k] = x[k ^ 1];
  } else if constexpr (VEC) {
    load8<T, true>(p, i >= d.rot_dims ? 0 : i < half ? i + half : i - half, d.head_dim, z);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t e = i + k;
      z[k] = e >= d.rot_dims ? 0.f : to_f(p[d.rot_pairing ? e ^ 1u : (e < half ? e + half : e - half)]);
    }
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const bool first = d.rot_pairing ? (k & 1) == 0 : i + k < half;
    x[k] = i + k < d.rot_dims ? turned(first, x[k], z[k], turn.c[k], turn.n[k]) : x[k];
  }
}

// as coded4, of eight elements in each of four lanes; the codes as bytes
__device__ __forceinline__ float min3(float a, float b, float c) {  // NaN if one of them is
  float r;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
struct Coded8 {
  uint32_t lo, hi;
  __half d, m;
};
template <bool VEC> __device__ __forceinline__ void range8(const float (&x)[8], uint32_t i, uint32_t n, float &lo, float &hi) {
  if constexpr (VEC) {
    lo = min3(min3(x[0], x[1], x[2]), min3(x[3], x[4], x[5]), min3(x[6], x[7], x[7]));
    hi = max3(max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5]), max3(x[6], x[7], x[7]));
    if (i >= n) lo = INFINITY, hi = -INFINITY;
  } else {
    lo = INFINITY, hi = -INFINITY;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k < n) lo = min3(lo, x[k], x[k]), hi = max3(hi, x[k], x[k]);
  }
#pragma unroll
  for (int o = 1; o < 4; o *= 2) {
    const float l = __shfl_xor_sync(0xffffffffu, lo, o), u = __shfl_xor_sync(0xffffffffu, hi, o);
    lo = min3(lo, l, l), hi = max3(hi, u, u);
  }
}
template <bool VEC> __device__ __forceinline__ Coded8 coded8(float (&x)[8], uint32_t i, uint32_t n, bool &changed) {
  Coded8 r;
  float lo, hi;
  range8<VEC>(x, i, n, lo, hi);
  if (__any_sync(0xffffffffu, !(lo >= -PG_LIMIT && hi <= PG_LIMIT))) {  // (NaN too)
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float c = x[k] != x[k] ? 0.f : fminf(fmaxf(x[k], -PG_LIMIT), PG_LIMIT);
      changed |= (VEC ? i : i + k) < n && !(c == x[k]);
      x[k] = c;
    }
    range8<VEC>(x, i, n, lo, hi);
  }
  if (lo > hi) lo = hi = 0.f;  // a group of padding
  r.m = __float2half_rn(lo);
  const float mf = __half2float(r.m);
  r.d = __float2half_rn(fmaxf(__fdiv_rn(__fsub_rn(hi, mf), 15.f), 0.f));
  const float df = __half2float(r.d);
  float inv;  // of d, at least 2^-24: off by one step at most
  asm("rcp.approx.f32 %0, %1;" : "=f"(inv) : "f"(df));
  inv = df > 0.f ? __fmul_rn(inv, 1.f / 15.f) : 0.f;
  // a fifteenth of the number between 0 and 1, so that one multiplication cuts it off; five roundings leave 15 * 5 * 2^-24 = 5e-6
  constexpr float BIG = 12582912.f;  // 3 * 2^22: the last place of a sum with it is 1
  float v[8], off = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float f = __saturatef(__fmul_rn(__fsub_rn(x[k], mf), inv)), up = __fmaf_rn(f, 15.f, BIG);
    off = fmaxf(off, fabsf(__fmaf_rn(f, 15.f, __fsub_rn(BIG, up))));
    v[k] = up;
  }
  if (off > 0.49999f)
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = __fadd_rn(fminf(fmaxf(__fdiv_rn(__fsub_rn(x[k], mf), df), 0.f), 15.f), BIG);
  uint32_t c[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) c[k] = VEC || i + k < n ? __float_as_uint(v[k]) : 0u;
  r.lo = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
  r.hi = __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410);
  if (VEC && i >= n) r.lo = r.hi = 0;
  return r;
}

constexpr uint32_t PC_STAGE = 10 * 256;  // codes and scales of the keys or values of a unit, at most

// The queries of a row, by a warp: cosines and sines are fetched once for all heads, and the row is read from end to end (a warp per head
// of sixteen rows, 256 bytes at a time, turned 13426 rows of 32 heads in bf16 in 63 us).
template <typename T, bool VEC> __device__ __forceinline__ void turn_row(const cutb_paged_desc &d, uint32_t row) {
  const uint32_t lane = threadIdx.x & 31, hd = d.head_dim, s = paged_seq_of(d, row);
  if (s >= d.n_seqs) return;
  const PagedSeq sq = paged_seq(d, s);
  if (sq.bad || row - sq.row0 >= sq.rows) return;  // (the keys' warps report)
  const uint32_t pos = sq.len - sq.rows + (row - sq.row0);
  if ((d.rot_dims && pos >= d.max_pos) || d.tables[sq.slot * d.ld_table + pos / d.page_tokens] >= d.n_pages) return;
  const T *src = reinterpret_cast<const T *>(d.q) + row * d.ldq;
  T *dst = reinterpret_cast<T *>(d.q_out) + row * d.ldq_out;
  for (uint32_t i = 8 * (lane % 16); i < hd; i += 128) {
    Turn turn;
    turn_at<VEC>(d, i, pos, turn);
#pragma unroll 4
    for (uint32_t h = lane / 16; h < d.n_heads; h += 2) {
      float x[8];
      turned8<T, VEC>(d, src + h * hd, i, turn, x);
      store8<T, VEC>(dst + h * hd, i, hd, x);
    }
  }
}

// A warp per head of a piece: a whole unit is put together in shared memory, four tokens at a time, and stored in 16-byte pieces; the warps
// behind those turn the queries.  13426 rows of 32 + 2 * 8 heads of 128 in bf16: 94 us, 50 without queries, where reading them takes 9: loads
// that nothing covers are the longest wait (7.8 cycles an instruction, 52 % of the issue slots used; some 2000 instructions a unit).  A warp per head
// of a row, bytes stored one by one, took 400 with the reading.
template <typename T, bool VEC> __global__ void __launch_bounds__(256, 4) paged_kv_write_units_kernel(const __grid_constant__ cutb_paged_desc d) {
  __shared__ __align__(16) uint8_t stage_s[8][PC_STAGE];
  pdl_enter();
  const uint32_t lane = threadIdx.x & 31, warp = warp_index(), heads = 2 * d.n_kv_heads, hd = d.head_dim, dp = pg_pad(hd), groups = dp / 32, second = lane / 16;
  const uint64_t item = (uint64_t)blockIdx.x * 8 + warp, keys = ((uint64_t)d.n_tokens + PG_UNIT - 1) / PG_UNIT * heads;
  if (item >= keys) {
    if (d.q && item - keys < d.n_tokens) turn_row<T, VEC>(d, (uint32_t)(item - keys));
    return;
  }
  const uint32_t h = (uint32_t)(item % heads);
  uint8_t *stage = stage_s[warp];
  bool changed = false;
  for_pieces(d, (uint32_t)(item / heads), [&](uint32_t row, uint32_t pos, uint32_t n, uint32_t page) {
    if (d.rot_dims && pos + n > d.max_pos) {
      if (lane == 0) paged_report(d.status, CUTB_ERR_INVALID);
      n = pos < d.max_pos ? d.max_pos - pos : 0;
    }
    const bool value = h >= d.n_kv_heads;
    const uint32_t kvh = value ? h - d.n_kv_heads : h;
    const uint64_t ld = value ? d.ldv : d.ldk;
    const T *src = reinterpret_cast<const T *>(value ? d.v : d.k) + row * ld + (uint64_t)kvh * hd;
    const Unit u = unit_of(d, page, kvh, pos, value);
    if (n < PG_UNIT) {
      for (uint32_t r = 0; r < n; ++r) write_head<T, false>(d, src + r * ld, pos + r, value, u.codes, u.scales, changed);
      return;
    }
    uint8_t *scales = stage + 8 * dp;
    for (uint32_t i0 = 0; i0 < dp; i0 += 128) {
      const uint32_t i = i0 + 8 * (lane % 16), g = i / 32;
#pragma unroll 1
      for (uint32_t t0 = 0; t0 < PG_UNIT; t0 += 4) {
        const uint32_t t[2] = {t0 + second, t0 + 2 + second};
        float x[2][8];
        Coded8 c[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (value) load8<T, VEC>(src + t[k] * ld, i, hd, x[k]);
          else {
            Turn turn;
            turn_at<VEC>(d, i, pos + t[k], turn);
            turned8<T, VEC>(d, src + t[k] * ld, i, turn, x[k]);
          }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) c[k] = coded8<VEC>(x[k], i, hd, changed);
        if (value) {
          // byte r of a token: element r low, element r + 8, the next lane's, high; this lane stores four of them
          const bool odd = lane & 1;
          uint32_t b[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t other = __shfl_xor_sync(0xffffffffu, odd ? c[k].lo : c[k].hi, 1);
            b[k] = odd ? other | c[k].hi << 4 : c[k].lo | other << 4;
          }
          if (i < dp)
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)  // tokens 0, 2 of four, or 1, 3, lie together
              *reinterpret_cast<uint16_t *>(stage + pg_value_byte(t0, i / 16, 4 * odd + e) + 2 * second) =
                  (uint16_t)((b[0] >> 8 * e & 255u) | (b[1] >> 8 * e & 255u) << 8);
          if (i < dp && i % 32 == 0) {
            __half *sc = reinterpret_cast<__half *>(scales) + 8 * (g * 4 + t0 / 4);
#pragma unroll
            for (int k = 0; k < 2; ++k) sc[2 * k + second] = c[k].d, sc[4 + 2 * k + second] = c[k].m;
          }
        } else if (i < dp) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            reinterpret_cast<uint32_t *>(stage)[pg_key_word(dp, t[k], g, i % 32 / 8)] =  // the bits of pg_key_bit
                __byte_perm(c[k].lo, c[k].hi, 0x5140) | __byte_perm(c[k].lo, c[k].hi, 0x7362) << 4;
            if (i % 32 == 0) *reinterpret_cast<__half2 *>(scales + 4 * (t[k] * groups + g)) = __halves2half2(c[k].d, c[k].m);
          }
        }
      }
    }
    __syncwarp();
    for (uint32_t w = lane; w < dp / 2; w += 32) reinterpret_cast<uint4 *>(u.codes)[w] = reinterpret_cast<const uint4 *>(stage)[w];
    for (uint32_t w = lane; w < dp / 8; w += 32) reinterpret_cast<uint4 *>(u.scales)[w] = reinterpret_cast<const uint4 *>(scales)[w];
    __syncwarp();
  });
  if (__any_sync(0xffffffffu, changed) && lane == 0) paged_report(d.status, CUTB_ERR_RANGE);
}

// What the cache holds of head elements i .. i + 3 of token t of a unit.
__device__ __forceinline__ void read_head(uint32_t dp, uint32_t t, uint32_t i, bool value, const uint8_t *codes, const uint8_t *scales, float (&x)[4]) {
  const uint32_t g = i / 32, groups = dp / 32;
  __half dh, m;
  if (value) {
    const __half *sc = reinterpret_cast<const __half *>(scales) + 8 * (g * 4 + t / 4) + t % 4;
    dh = sc[0], m = sc[4];
  } else {
    const __half2 sc = *reinterpret_cast<const __half2 *>(scales + 4 * (t * groups + g));
    dh = __low2half(sc), m = __high2half(sc);
  }
  const uint32_t word = value ? 0u : reinterpret_cast<const uint32_t *>(codes)[pg_key_word(dp, t, g, i % 32 / 8)];
#pragma unroll
  for (uint32_t k = 0; k < 4; ++k) {
    const uint32_t q = value ? codes[pg_value_byte(t, i / 16, (i + k) % 8)] >> ((i & 8) ? 4 : 0) & 15u : word >> pg_key_bit((i + k) % 8) & 15u;
    x[k] = __half2float(__hfma(__uint2half_rn(q), dh, m));
  }
}

template <typename T, bool VEC> __global__ void __launch_bounds__(256) paged_kv_read_kernel(const __grid_constant__ cutb_paged_desc d) {
  pdl_enter();
  const uint32_t lane = threadIdx.x & 31, heads = 2 * d.n_kv_heads;
  const uint64_t item = (uint64_t)blockIdx.x * 8 + warp_index();
  const uint32_t row = (uint32_t)(item / heads), h = (uint32_t)(item % heads);
  if (row >= d.n_tokens) return;
  const uint32_t s = paged_seq_of(d, row);
  if (s >= d.n_seqs) return;
  const PagedSeq sq = paged_seq(d, s);
  if (!sq.bad && row - sq.row0 >= sq.rows) return;
  const uint32_t pos = sq.len - sq.rows + (row - sq.row0);
  const uint32_t page = sq.bad ? CUTB_NO_PAGE : d.tables[sq.slot * d.ld_table + pos / d.page_tokens];
  const bool value = h >= d.n_kv_heads;
  const uint32_t kvh = value ? h - d.n_kv_heads : h;
  T *dst = reinterpret_cast<T *>(value ? d.v_out : d.k_out) + row * (value ? d.ldv_out : d.ldk_out) + (uint64_t)kvh * d.head_dim;
  if (page >= d.n_pages) {
    if (lane == 0) paged_report(d.status, CUTB_ERR_INVALID);
    if (!d.starts)  // (the row is this sequence's whatever else is wrong: callers need not fill the rows first)
      for (uint32_t i = lane; i < d.head_dim; i += 32) dst[i] = from_f<T>(0.f);
    return;
  }
  const Unit u = unit_of(d, page, kvh, pos, value);
  for (uint32_t i = 4 * lane; i < d.head_dim; i += 128) {
    float x[4];
    read_head(pg_pad(d.head_dim), pos % PG_UNIT, i, value, u.codes, u.scales, x);
    store4(dst, i, d.head_dim, VEC, x);
  }
}

// Many rows: a lane takes whole words, eight elements of a key or the bytes of sixteen elements of four tokens' values.
template <typename T, bool VEC> __global__ void __launch_bounds__(256, 4) paged_kv_read_units_kernel(const __grid_constant__ cutb_paged_desc d, uint32_t each) {
  pdl_enter();
  const uint32_t lane = threadIdx.x & 31, heads = 2 * d.n_kv_heads;
  const uint64_t item = (uint64_t)blockIdx.x * 8 + warp_index();
  const uint32_t parts = (heads + each - 1) / each, h0 = (uint32_t)(item % parts), hd = d.head_dim, dp = pg_pad(hd), groups = dp / 32;
  for_pieces(d, (uint32_t)(item / parts), [&](uint32_t row, uint32_t pos, uint32_t n, uint32_t page) {
    for (uint32_t h = h0; h < heads; h += parts) {  // (neighbouring warps have neighbouring heads at a time)
      const bool value = h >= d.n_kv_heads;
      const uint32_t kvh = value ? h - d.n_kv_heads : h;
      const uint64_t ld = value ? d.ldv_out : d.ldk_out;
      const Unit u = unit_of(d, page, kvh, pos, value);
      const uint32_t *words = reinterpret_cast<const uint32_t *>(u.codes), t0 = pos % PG_UNIT;
      T *dst = reinterpret_cast<T *>(value ? d.v_out : d.k_out) + row * ld + (uint64_t)kvh * hd;
      if (!value) {
#pragma unroll 4
        for (uint32_t w = t0 * (dp / 8) + lane; w < (t0 + n) * (dp / 8); w += 32) {
          const uint32_t t = w / (dp / 8), at = w % (dp / 8) * 8, j = at / 32, b = at % 32 / 8;
          const __half2 sc = *reinterpret_cast<const __half2 *>(u.scales + 4 * (t * groups + j)), dd = __low2half2(sc), mm = __high2half2(sc);
          __half2 q[4];
          pg_quants(words[pg_key_word(dp, t, j, b)], q);
          float x[8];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 f = __half22float2(__hfma2(q[k], dd, mm));
            x[2 * k] = f.x, x[2 * k + 1] = f.y;
          }
          store8<T, VEC>(dst + (t - t0) * ld, at, hd, x);
        }
        continue;
      }
      for (uint32_t w = lane; w < dp / 4; w += 32) {  // sixteen elements i, four tokens t4
        const uint32_t i = w % (dp / 16), t4 = w / (dp / 16) * 4;
        if (t4 + 4 <= t0 || t4 >= t0 + n) continue;
        const __half2 *sc = reinterpret_cast<const __half2 *>(u.scales) + 4 * (i / 2 * 4 + t4 / 4);
        const __half2 d01 = sc[0], d23 = sc[1], m01 = sc[2], m23 = sc[3];
        uint32_t word[8];
#pragma unroll
        for (uint32_t r = 0; r < 8; ++r) word[r] = words[pg_value_byte(t4, i, r) / 4];
#pragma unroll
        for (uint32_t high = 0; high < 2; ++high) {
          float x[4][8];
#pragma unroll
          for (uint32_t r = 0; r < 8; ++r) {
            __half2 q[4];
            pg_quants(word[r], q);
            const float2 a = __half22float2(__hfma2(q[high], d01, m01)), b = __half22float2(__hfma2(q[2 + high], d23, m23));
            x[0][r] = a.x, x[1][r] = a.y, x[2][r] = b.x, x[3][r] = b.y;
          }
#pragma unroll
          for (uint32_t k = 0; k < 4; ++k)
            if (t4 + k >= t0 && t4 + k < t0 + n) store8<T, VEC>(dst + (uint64_t)(t4 + k - t0) * ld, 16 * i + 8 * high, hd, x[k]);
        }
      }
    }
  });
}

// By units where their warps are sixteen to an SM and sequences may have units (without starts they have a row each); else a warp per head of a row.
bool by_units(const cutb_paged_desc &d, uint64_t heads) { return d.starts && d.max_new >= PG_UNIT && (d.n_tokens + PG_UNIT - 1) / PG_UNIT * heads >= 148 * 16; }
uint32_t units_of(const cutb_paged_desc &d) { return (d.n_tokens + PG_UNIT - 1) / PG_UNIT; }
dim3 warps_grid(uint64_t warps) { return dim3((uint32_t)((warps + 7) / 8)); }

// ---- bookkeeping ---------------------------------------------------------------------------------------------------------
constexpr uint32_t PB_THREADS = 1024, PB_MOST = 1024;

// What a planning kernel leaves for the kernel that moves pages: {count, held pages}, then the pairs, then (compact) where a page goes.
struct PagesPlan {
  uint32_t *head, *src, *dst, *to;
};
__host__ __device__ inline PagesPlan pages_plan(void *ws, uint32_t n_pages) {
  uint32_t *w = reinterpret_cast<uint32_t *>(ws);
  const uint32_t most = n_pages > PB_MOST ? n_pages : PB_MOST;
  return PagesPlan{w, w + 64, w + 64 + most, w + 64 + 2ull * most};
}

// Exclusive sum over the block's threads; `total` to all.
__device__ __forceinline__ uint32_t block_sum_before(uint32_t v, uint32_t *warps, uint32_t &total) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  uint32_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // (the sums of a call before are read)
  if (lane == 31) warps[warp] = x;
  __syncthreads();
  uint32_t w = warps[lane];
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += y;
  }
  total = __shfl_sync(0xffffffffu, w, 31);
  const uint32_t before = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
  return x - v + (warp ? before : 0);
}

__device__ __forceinline__ uint32_t pages_of(uint32_t tokens, uint32_t page_tokens) { return tokens / page_tokens + (tokens % page_tokens != 0); }

// One block, a thread per entry; then its warps fill the tables entry by entry.
__global__ void __launch_bounds__(PB_THREADS) pages_reserve_kernel(const __grid_constant__ cutb_pages_desc d) {
  __shared__ uint32_t warps[32], slot_s[PB_MOST], last_s[PB_MOST], first_s[PB_MOST], have_s[PB_MOST], want_s[PB_MOST];
  pdl_enter();
  const PagesPlan plan = pages_plan(d.workspace, d.n_pages);
  const uint32_t i = threadIdx.x, lane = i & 31, P = d.page_tokens;
  const bool mine = i < d.n;
  const uint32_t s = mine ? d.items[i] : 0, grow = mine ? d.counts[i] : 0;
  slot_s[i] = mine ? s : 0xffffffffu;
  __syncthreads();
  bool ok = mine && s < d.n_slots;
  for (uint32_t j = 0; j < i && ok; ++j) ok = slot_s[j] != s;
  const uint32_t len = ok ? d.lengths[s] : 0;
  ok = ok && (uint64_t)len + grow <= (uint64_t)d.ld_table * P && (uint64_t)len + grow <= 0xffffffffu;
  const bool partial = ok && grow && len % P;
  uint32_t last = 0xffffffffu;
  if (partial) {
    last = d.tables[s * d.ld_table + len / P];
    if (last >= d.n_pages) ok = false, last = 0xffffffffu;
  }
  last_s[i] = last;
  if (mine && !ok) paged_report(d.status, CUTB_ERR_INVALID);
  __syncthreads();
  bool copied = false;
  if (last != 0xffffffffu) {  // all holders of a page but the last copy it
    const uint32_t refs = d.refs[last];
    uint32_t earlier = 0;
    for (uint32_t j = 0; j < i; ++j) earlier += last_s[j] == last;
    copied = refs > earlier + 1;
  }
  const uint32_t have = pages_of(len, P), want = ok ? pages_of(len + grow, P) : have, need = want - have + copied;
  uint32_t total;
  const uint32_t first = block_sum_before(need, warps, total);
  // the lowest free pages, 4096 at a time
  uint32_t found = 0;
  for (uint32_t p0 = 0; p0 < d.n_pages && found < total; p0 += 4 * PB_THREADS) {
    uint32_t free4 = 0;
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
      const uint32_t p = p0 + 4 * i + k;
      free4 |= (uint32_t)(p < d.n_pages && d.refs[p] == 0) << k;
    }
    uint32_t sum;
    uint32_t at = found + block_sum_before(__popc(free4), warps, sum);
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k)
      if (free4 >> k & 1) {
        if (at < total) plan.to[at] = p0 + 4 * i + k;
        ++at;
      }
    found += sum;
  }
  __syncthreads();  // (and the list is written)
  const bool granted = ok && first + need <= found;
  if (mine && ok && !granted) paged_report(d.status, CUTB_ERR_PAGES);
  const bool moves = granted && copied;
  uint32_t count;
  const uint32_t at = block_sum_before(moves, warps, count);
  if (moves) {
    plan.src[at] = last, plan.dst[at] = plan.to[first];
    d.tables[s * d.ld_table + len / P] = plan.to[first];
    d.refs[plan.to[first]] = 1;
    atomicSub(d.refs + last, 1u);
  }
  if (i == 0) plan.head[0] = count;
  if (granted) d.lengths[s] = len + grow;
  first_s[i] = first + copied, have_s[i] = have, want_s[i] = granted ? want : have;
  __syncthreads();
  for (uint32_t e = i / 32; e < d.n; e += PB_THREADS / 32) {
    const uint32_t from = have_s[e], n = want_s[e] - from;
    for (uint32_t k = lane; k < n; k += 32) {
      const uint32_t p = plan.to[first_s[e] + k];
      d.tables[slot_s[e] * d.ld_table + from + k] = p;
      d.refs[p] = 1;
    }
  }
}

__global__ void __launch_bounds__(PB_THREADS) pages_fork_kernel(const __grid_constant__ cutb_pages_desc d) {
  __shared__ uint32_t src_s[PB_MOST], dst_s[PB_MOST], n_s[PB_MOST];
  pdl_enter();
  const uint32_t i = threadIdx.x, lane = i & 31;
  const bool mine = i < d.n;
  const uint32_t src = mine ? d.items[i] : 0, dst = mine ? d.others[i] : 0;
  dst_s[i] = mine ? dst : 0xffffffffu, src_s[i] = src;
  __syncthreads();
  bool ok = mine && src < d.n_slots && dst < d.n_slots && src != dst;
  for (uint32_t j = 0; j < i && ok; ++j) ok = dst_s[j] != dst;
  const uint32_t len = ok ? d.lengths[src] : 0;
  ok = ok && d.lengths[dst] == 0 && len <= (uint64_t)d.ld_table * d.page_tokens;
  if (mine && !ok) paged_report(d.status, CUTB_ERR_INVALID);
  n_s[i] = ok ? pages_of(len, d.page_tokens) : 0;
  __syncthreads();  // every length is read as it was
  if (ok) d.lengths[dst] = len;
  for (uint32_t e = i / 32; e < d.n; e += PB_THREADS / 32)
    for (uint32_t k = lane; k < n_s[e]; k += 32) {
      const uint32_t p = d.tables[src_s[e] * d.ld_table + k];
      d.tables[dst_s[e] * d.ld_table + k] = p;
      if (p < d.n_pages) atomicAdd(d.refs + p, 1u);
      else paged_report(d.status, CUTB_ERR_INVALID);
    }
}

__global__ void __launch_bounds__(PB_THREADS) pages_free_kernel(const __grid_constant__ cutb_pages_desc d) {
  __shared__ uint32_t slot_s[PB_MOST], n_s[PB_MOST];
  pdl_enter();
  const uint32_t i = threadIdx.x, lane = i & 31;
  const bool mine = i < d.n;
  const uint32_t s = mine ? d.items[i] : 0;
  uint32_t n = 0;
  if (mine && s >= d.n_slots) paged_report(d.status, CUTB_ERR_INVALID);
  if (mine && s < d.n_slots) {
    const uint32_t len = atomicExch(d.lengths + s, 0u);  // (a slot named twice is empty the second time)
    n = pages_of(len, d.page_tokens);
    if (n > d.ld_table) n = (uint32_t)d.ld_table, paged_report(d.status, CUTB_ERR_INVALID);
  }
  slot_s[i] = s, n_s[i] = n;
  __syncthreads();
  for (uint32_t e = i / 32; e < d.n; e += PB_THREADS / 32)
    for (uint32_t k = lane; k < n_s[e]; k += 32) {
      uint32_t *entry = d.tables + slot_s[e] * d.ld_table + k;
      const uint32_t p = *entry;
      *entry = CUTB_NO_PAGE;
      if (p >= d.n_pages) {
        paged_report(d.status, CUTB_ERR_INVALID);
      } else if (atomicSub(d.refs + p, 1u) - 1 >= 0x7fffffffu) {  // nobody held it (or others have just taken off as much: each of them puts its own back)
        atomicAdd(d.refs + p, 1u);
        paged_report(d.status, CUTB_ERR_INVALID);
      }
    }
}

// One block: counts the held pages, pairs those past the count with the free places below it, and moves their counts.
__global__ void __launch_bounds__(PB_THREADS) pages_compact_kernel(const __grid_constant__ cutb_pages_desc d) {
  __shared__ uint32_t warps[32];
  pdl_enter();
  const PagesPlan plan = pages_plan(d.workspace, d.n_pages);
  const uint32_t i = threadIdx.x;
  uint32_t held = 0, unused;
  for (uint32_t p = i; p < d.n_pages; p += PB_THREADS) held += d.refs[p] != 0;
  (void)block_sum_before(held, warps, unused);
  held = unused;
  uint32_t holes = 0, late = 0;
  for (uint32_t p0 = 0; p0 < d.n_pages; p0 += PB_THREADS) {
    const uint32_t p = p0 + i;
    const bool in = p < d.n_pages, live = in && d.refs[p] != 0, hole = in && !live && p < held, moves = live && p >= held;
    uint32_t sum;
    uint32_t at = holes + block_sum_before(hole, warps, sum);
    if (hole) plan.dst[at] = p;
    holes += sum;
    at = late + block_sum_before(moves, warps, sum);
    if (moves) plan.src[at] = p;
    late += sum;
    if (in && p >= held && !live) plan.to[p] = p;
  }
  __syncthreads();
  for (uint32_t k = i; k < late; k += PB_THREADS) {
    const uint32_t from = plan.src[k], to = plan.dst[k];
    plan.to[from] = to;
    d.refs[to] = d.refs[from];
    d.refs[from] = 0;
  }
  if (i == 0) plan.head[0] = late, plan.head[1] = held;
}

// Moves the planned pages, PM_CHUNK bytes to a block at a time, and (remap) follows them in the tables.
constexpr uint32_t PM_THREADS = 256, PM_CHUNK = PM_THREADS * 16 * 4;
__global__ void __launch_bounds__(PM_THREADS) pages_move_kernel(const __grid_constant__ cutb_pages_desc d, const uint32_t *count, const uint32_t *src,
                                                                const uint32_t *dst, uint32_t fixed, const uint32_t *to) {
  pdl_enter();
  const uint32_t n = count ? count[0] : fixed, chunks = (uint32_t)((d.page_bytes + PM_CHUNK - 1) / PM_CHUNK);
  if (to) {
    const uint32_t held = count[1];
    const uint64_t entries = d.n_slots * d.ld_table;
    for (uint64_t e = (uint64_t)blockIdx.x * PM_THREADS + threadIdx.x; e < entries; e += (uint64_t)gridDim.x * PM_THREADS) {
      const uint32_t p = d.tables[e];
      if (p >= held && p < d.n_pages) d.tables[e] = to[p];
    }
  }
  for (uint64_t w = blockIdx.x; w < (uint64_t)n * chunks; w += gridDim.x) {
    const uint32_t k = (uint32_t)(w / chunks), from = src[k], into = dst[k];
    if (from >= d.n_pages || into >= d.n_pages) {
      if (threadIdx.x == 0) paged_report(d.status, CUTB_ERR_INVALID);
      continue;
    }
    const uint64_t at = w % chunks * (uint64_t)PM_CHUNK;
    const uint4 *a = reinterpret_cast<const uint4 *>(reinterpret_cast<const uint8_t *>(d.pages) + from * d.page_bytes + at);
    uint4 *b = reinterpret_cast<uint4 *>(reinterpret_cast<uint8_t *>(d.pages) + into * d.page_bytes + at);
    const uint64_t left = (d.page_bytes - at) / 16;
    uint4 v[4];
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j)
      if (threadIdx.x + j * PM_THREADS < left) v[j] = a[threadIdx.x + j * PM_THREADS];
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j)
      if (threadIdx.x + j * PM_THREADS < left) b[threadIdx.x + j * PM_THREADS] = v[j];
  }
}

bool aligned(const void *p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int move_blocks(uint64_t most, uint32_t *out) {
  DeviceInfo di;
  if (int rc = get_device_info(&di)) return rc;
  const uint64_t full = (uint64_t)di.sm_count * 8;
  *out = (uint32_t)(most < full ? (most ? most : 1) : full);
  return CUTB_OK;
}

}  // namespace

int paged_kv_write_launch(const cutb_paged_desc &d, cudaStream_t stream) {
  return paged_with_type(d.dtype, [&](auto t) {
    using T = decltype(t);
    const uint32_t heads = 2 * d.n_kv_heads + (d.q ? d.n_heads : 0);
    const uintptr_t a = 4 * sizeof(T);
    const bool vec = d.head_dim % 4 == 0 && d.ldk % 4 == 0 && d.ldv % 4 == 0 && aligned(d.k, a) && aligned(d.v, a) &&
                     (!d.q || (d.ldq % 4 == 0 && d.ldq_out % 4 == 0 && aligned(d.q, a) && aligned(d.q_out, a))) &&
                     (!d.rot_dims || (d.rot_dims % 8 == 0 && aligned(d.cos_table, 16) && aligned(d.sin_table, 16)));
    const bool wide = d.head_dim % 8 == 0 && d.ldk % 8 == 0 && d.ldv % 8 == 0 && aligned(d.k, 16) && aligned(d.v, 16) &&
                      (!d.q || (d.ldq % 8 == 0 && d.ldq_out % 8 == 0 && aligned(d.q, 16) && aligned(d.q_out, 16))) &&
                      (!d.rot_dims || (d.rot_dims % (d.rot_pairing ? 8 : 16) == 0 && aligned(d.cos_table, 16) && aligned(d.sin_table, 16)));
    if (by_units(d, 2 * d.n_kv_heads)) {
      const auto kernel = wide ? paged_kv_write_units_kernel<T, true> : paged_kv_write_units_kernel<T, false>;
      CUTB_CUDA_TRY(launch_pdl(kernel, warps_grid((uint64_t)units_of(d) * 2 * d.n_kv_heads + (d.q ? d.n_tokens : 0)), dim3(256), 0, stream, d));
    } else {
      const auto kernel = vec ? paged_kv_write_kernel<T, true> : paged_kv_write_kernel<T, false>;
      CUTB_CUDA_TRY(launch_pdl(kernel, warps_grid((uint64_t)d.n_tokens * heads), dim3(256), 0, stream, d));
    }
    return (int)CUTB_OK;
  });
}

int paged_kv_read_launch(const cutb_paged_desc &d, cudaStream_t stream) {
  return paged_with_type(d.dtype, [&](auto t) {
    using T = decltype(t);
    const uint32_t heads = 2 * d.n_kv_heads;
    const uintptr_t a = 4 * sizeof(T);
    const bool vec = d.head_dim % 4 == 0 && d.ldk_out % 4 == 0 && d.ldv_out % 4 == 0 && aligned(d.k_out, a) && aligned(d.v_out, a);
    const bool wide = d.head_dim % 8 == 0 && d.ldk_out % 8 == 0 && d.ldv_out % 8 == 0 && aligned(d.k_out, 16) && aligned(d.v_out, 16);
    if (by_units(d, heads)) {
      const uint32_t each = (uint64_t)units_of(d) * d.n_kv_heads >= 148 * 32 ? 2 : 1;  // (13426 rows of 8 heads: 33 us, 39 one by one)
      const auto kernel = wide ? paged_kv_read_units_kernel<T, true> : paged_kv_read_units_kernel<T, false>;
      CUTB_CUDA_TRY(launch_pdl(kernel, warps_grid((uint64_t)units_of(d) * (heads / each)), dim3(256), 0, stream, d, each));
    } else {
      const auto kernel = vec ? paged_kv_read_kernel<T, true> : paged_kv_read_kernel<T, false>;
      CUTB_CUDA_TRY(launch_pdl(kernel, warps_grid((uint64_t)d.n_tokens * heads), dim3(256), 0, stream, d));
    }
    return (int)CUTB_OK;
  });
}

int pages_reserve_launch(const cutb_pages_desc &d, cudaStream_t stream) {
  const PagesPlan plan = pages_plan(d.workspace, d.n_pages);
  uint32_t blocks;
  if (int rc = move_blocks((uint64_t)d.n * ((d.page_bytes + PM_CHUNK - 1) / PM_CHUNK), &blocks)) return rc;
  CUTB_CUDA_TRY(launch_pdl(pages_reserve_kernel, dim3(1), dim3(PB_THREADS), 0, stream, d));
  CUTB_CUDA_TRY(launch_pdl(pages_move_kernel, dim3(blocks), dim3(PM_THREADS), 0, stream, d, plan.head, plan.src, plan.dst, 0u, (const uint32_t *)nullptr));
  return CUTB_OK;
}

int pages_fork_launch(const cutb_pages_desc &d, cudaStream_t stream) {
  CUTB_CUDA_TRY(launch_pdl(pages_fork_kernel, dim3(1), dim3(PB_THREADS), 0, stream, d));
  return CUTB_OK;
}

int pages_free_launch(const cutb_pages_desc &d, cudaStream_t stream) {
  CUTB_CUDA_TRY(launch_pdl(pages_free_kernel, dim3(1), dim3(PB_THREADS), 0, stream, d));
  return CUTB_OK;
}

int pages_compact_launch(const cutb_pages_desc &d, cudaStream_t stream) {
  const PagesPlan plan = pages_plan(d.workspace, d.n_pages);
  uint32_t blocks;
  if (int rc = move_blocks(~0ull, &blocks)) return rc;
  CUTB_CUDA_TRY(launch_pdl(pages_compact_kernel, dim3(1), dim3(PB_THREADS), 0, stream, d));
  CUTB_CUDA_TRY(launch_pdl(pages_move_kernel, dim3(blocks), dim3(PM_THREADS), 0, stream, d, plan.head, plan.src, plan.dst, 0u, (const uint32_t *)plan.to));
  return CUTB_OK;
}

int pages_copy_launch(const cutb_pages_desc &d, cudaStream_t stream) {
  uint32_t blocks;
  if (int rc = move_blocks((uint64_t)d.n * ((d.page_bytes + PM_CHUNK - 1) / PM_CHUNK), &blocks)) return rc;
  CUTB_CUDA_TRY(launch_pdl(pages_move_kernel, dim3(blocks), dim3(PM_THREADS), 0, stream, d, (const uint32_t *)nullptr, d.items, d.others, d.n, (const uint32_t *)nullptr));
  return CUTB_OK;
}

}  // namespace cutb
