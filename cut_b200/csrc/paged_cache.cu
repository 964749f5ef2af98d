// The paged 4-bit cache: rows written and read back, and the bookkeeping of its pages.
#include "kernels.h"
#include "paged_common.cuh"

namespace cutb {
namespace {

// ---- rows --------------------------------------------------------------------------------------------------------------
// A warp per head of a token: the new keys and values (and the queries) of the token, then of the next one.  A lane holds four
// neighbouring elements of every 128, so that the eight lanes of a group of 32 meet in three shuffles and two lanes make a word.
template <typename T> __device__ __forceinline__ void load4(const T *p, uint32_t i, uint32_t n, bool vec, float (&x)[4]) {
  if (vec && i + 4 <= n) {
    if constexpr (sizeof(T) == 4) {
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
  if (vec && i + 4 <= n) {
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
template <typename T>
__device__ __forceinline__ void turned4(const cutb_paged_desc &d, const T *p, uint32_t i, uint32_t pos, bool vec, float (&x)[4]) {
  load4(p, i, d.head_dim, vec, x);
  if (i >= d.rot_dims) return;
  const uint32_t half = d.rot_dims / 2;
  const float *cs = d.cos_table + (uint64_t)pos * half, *sn = d.sin_table + (uint64_t)pos * half;
  float y[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t e = i + k;
    y[k] = x[k];
    if (e >= d.rot_dims) continue;
    const bool first = d.rot_pairing ? (e & 1) == 0 : e < half;
    const uint32_t t = d.rot_pairing ? e / 2 : (first ? e : e - half), other = d.rot_pairing ? e ^ 1u : (first ? e + half : e - half);
    const float z = to_f(p[other]), c = __ldg(cs + t), s = __ldg(sn + t);
    y[k] = first ? __fsub_rn(__fmul_rn(x[k], c), __fmul_rn(z, s)) : __fadd_rn(__fmul_rn(z, s), __fmul_rn(x[k], c));
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) x[k] = y[k];
}

template <typename T> __global__ void __launch_bounds__(256) paged_kv_write_kernel(const __grid_constant__ cutb_paged_desc d, int vec) {
  pdl_enter();
  const uint32_t lane = threadIdx.x & 31, heads = 2 * d.n_kv_heads + (d.q ? d.n_heads : 0);
  const uint64_t item = ((uint64_t)blockIdx.x * 256 + threadIdx.x) / 32;
  const uint32_t row = (uint32_t)(item / heads), h = (uint32_t)(item % heads);
  if (row >= d.n_tokens) return;
  const uint32_t s = paged_seq_of(d, row);
  if (s >= d.n_seqs) return;
  const PagedSeq sq = paged_seq(d, s);
  bool bad = sq.bad;
  if (!bad && row - sq.row0 >= sq.rows) return;  // behind the last sequence
  const uint32_t pos = sq.len - sq.rows + (row - sq.row0), dp = pg_pad(d.head_dim);
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
      turned4(d, src, i, pos, vec, x);
      store4(dst, i, d.head_dim, vec, x);
    }
    return;
  }
  const bool value = h >= d.n_kv_heads;
  const uint32_t kvh = value ? h - d.n_kv_heads : h, t = pos % PG_UNIT, groups = dp / 32;
  uint8_t *unit = reinterpret_cast<uint8_t *>(d.pages) + (uint64_t)page * d.page_bytes +
                  ((uint64_t)kvh * (d.page_tokens / PG_UNIT) + pos % d.page_tokens / PG_UNIT) * pg_unit_bytes(dp);
  const T *src = reinterpret_cast<const T *>(value ? d.v : d.k) + row * (value ? d.ldv : d.ldk) + (uint64_t)kvh * d.head_dim;
  bool changed = false;
  for (uint32_t i0 = 0; i0 < dp; i0 += 128) {
    const uint32_t i = i0 + 4 * lane;
    float x[4], lo = INFINITY, hi = -INFINITY;
    if (value) load4(src, i, d.head_dim, vec, x);
    else turned4(d, src, i, pos, vec, x);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (i + k >= d.head_dim) continue;
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
    const __half m = __float2half_rn(lo);
    const float mf = __half2float(m);
    const __half dh = __float2half_rn(fmaxf(__fdiv_rn(__fsub_rn(hi, mf), 15.f), 0.f));
    const float df = __half2float(dh);
    uint32_t code[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      code[k] = i + k < d.head_dim && df > 0.f ? (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[k], mf), df)), 0.f), 15.f) : 0u;
    const uint32_t g = i / 32;
    if (value) {
      // the partners of bytes, eight elements on, are two lanes on
      uint32_t mine = code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24;
      const uint32_t bytes = mine | __shfl_xor_sync(0xffffffffu, mine, 2) << 4;
      if (i < dp && (lane & 2) == 0)
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) unit[pg_values_at(dp) + pg_value_byte(t, i / 16, (i + k) % 8)] = (uint8_t)(bytes >> 8 * k);
      if (i < dp && (lane & 7) == 0) {
        __half *sc = reinterpret_cast<__half *>(unit + pg_value_scales_at(dp)) + 8 * (g * 4 + t / 4) + t % 4;
        sc[0] = dh, sc[4] = m;
      }
    } else {
      uint32_t part = 0;
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) part |= code[k] << pg_key_bit((i + k) % 8);
      const uint32_t word = part | __shfl_xor_sync(0xffffffffu, part, 1);
      if (i < dp && (lane & 1) == 0) reinterpret_cast<uint32_t *>(unit)[pg_key_word(dp, t, g, i % 32 / 8)] = word;
      if (i < dp && (lane & 7) == 0) *reinterpret_cast<__half2 *>(unit + pg_key_scales_at(dp) + 4 * (t * groups + g)) = __halves2half2(dh, m);
    }
  }
  if (__any_sync(0xffffffffu, changed) && lane == 0) paged_report(d.status, CUTB_ERR_RANGE);
}

template <typename T> __global__ void __launch_bounds__(256) paged_kv_read_kernel(const __grid_constant__ cutb_paged_desc d, int vec) {
  pdl_enter();
  const uint32_t lane = threadIdx.x & 31, heads = 2 * d.n_kv_heads;
  const uint64_t item = ((uint64_t)blockIdx.x * 256 + threadIdx.x) / 32;
  const uint32_t row = (uint32_t)(item / heads), h = (uint32_t)(item % heads);
  if (row >= d.n_tokens) return;
  const uint32_t s = paged_seq_of(d, row);
  if (s >= d.n_seqs) return;
  const PagedSeq sq = paged_seq(d, s);
  if (!sq.bad && row - sq.row0 >= sq.rows) return;
  const uint32_t pos = sq.len - sq.rows + (row - sq.row0), dp = pg_pad(d.head_dim), t = pos % PG_UNIT, groups = dp / 32;
  const uint32_t page = sq.bad ? CUTB_NO_PAGE : d.tables[sq.slot * d.ld_table + pos / d.page_tokens];
  if (page >= d.n_pages) {
    if (lane == 0) paged_report(d.status, CUTB_ERR_INVALID);
    return;
  }
  const bool value = h >= d.n_kv_heads;
  const uint32_t kvh = value ? h - d.n_kv_heads : h;
  T *dst = reinterpret_cast<T *>(value ? d.v_out : d.k_out) + row * (value ? d.ldv_out : d.ldk_out) + (uint64_t)kvh * d.head_dim;
  const uint8_t *unit = reinterpret_cast<const uint8_t *>(d.pages) + (uint64_t)page * d.page_bytes +
                        ((uint64_t)kvh * (d.page_tokens / PG_UNIT) + pos % d.page_tokens / PG_UNIT) * pg_unit_bytes(dp);
  for (uint32_t i = 4 * lane; i < d.head_dim; i += 128) {
    const uint32_t g = i / 32;
    __half dh, m;
    float x[4];
    if (value) {
      const __half *sc = reinterpret_cast<const __half *>(unit + pg_value_scales_at(dp)) + 8 * (g * 4 + t / 4) + t % 4;
      dh = sc[0], m = sc[4];
    } else {
      const __half2 sc = *reinterpret_cast<const __half2 *>(unit + pg_key_scales_at(dp) + 4 * (t * groups + g));
      dh = __low2half(sc), m = __high2half(sc);
    }
    const uint32_t word = value ? 0u : reinterpret_cast<const uint32_t *>(unit)[pg_key_word(dp, t, g, i % 32 / 8)];
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
      const uint32_t q = value ? unit[pg_values_at(dp) + pg_value_byte(t, i / 16, (i + k) % 8)] >> ((i & 8) ? 4 : 0) & 15u : word >> pg_key_bit((i + k) % 8) & 15u;
      x[k] = __half2float(__hfma(__uint2half_rn(q), dh, m));
    }
    store4(dst, i, d.head_dim, vec, x);
  }
}

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
      } else if (atomicSub(d.refs + p, 1u) == 0) {  // nobody held it
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
    const uint64_t items = (uint64_t)d.n_tokens * (2 * d.n_kv_heads + (d.q ? d.n_heads : 0));
    const uintptr_t a = 4 * sizeof(T);
    const bool vec = d.head_dim % 4 == 0 && d.ldk % 4 == 0 && d.ldv % 4 == 0 && aligned(d.k, a) && aligned(d.v, a) &&
                     (!d.q || (d.ldq % 4 == 0 && d.ldq_out % 4 == 0 && aligned(d.q, a) && aligned(d.q_out, a)));
    CUTB_CUDA_TRY(launch_pdl(paged_kv_write_kernel<T>, dim3((uint32_t)((items + 7) / 8)), dim3(256), 0, stream, d, (int)vec));
    return (int)CUTB_OK;
  });
}

int paged_kv_read_launch(const cutb_paged_desc &d, cudaStream_t stream) {
  return paged_with_type(d.dtype, [&](auto t) {
    using T = decltype(t);
    const uint64_t items = (uint64_t)d.n_tokens * 2 * d.n_kv_heads;
    const uintptr_t a = 4 * sizeof(T);
    const bool vec = d.head_dim % 4 == 0 && d.ldk_out % 4 == 0 && d.ldv_out % 4 == 0 && aligned(d.k_out, a) && aligned(d.v_out, a);
    CUTB_CUDA_TRY(launch_pdl(paged_kv_read_kernel<T>, dim3((uint32_t)((items + 7) / 8)), dim3(256), 0, stream, d, (int)vec));
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
