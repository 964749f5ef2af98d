// extern "C" entry points of the paged 4-bit cache: argument checks and launch.
#include "kernels.h"
#include "paged_common.cuh"

namespace cutb {
namespace {

bool misaligned(const void *p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }
bool page_size_ok(uint32_t t) { return t >= 16 && t <= 256 && (t & (t - 1)) == 0; }
uint32_t type_bytes(int t) { return t == CUTB_F32 ? 4 : 2; }

uint64_t layer_bytes(uint32_t n_kv_heads, uint32_t head_dim, uint32_t page_tokens) {
  return (uint64_t)n_kv_heads * (page_tokens / PG_UNIT) * pg_unit_bytes(pg_pad(head_dim));
}

// CUTB_OK with *nothing set: there are no rows
int check_paged(const cutb_paged_desc *d, const char *what) {
  if (!d || (d->dtype != CUTB_F32 && d->dtype != CUTB_F16 && d->dtype != CUTB_BF16)) {
    set_last_error("%s: null descriptor, or an element type that is not fp32, fp16 or bf16", what);
    return CUTB_ERR_INVALID;
  }
  if (!page_size_ok(d->page_tokens) || d->n_kv_heads == 0 || d->n_kv_heads > 65535 || d->head_dim == 0 || d->head_dim > 256 || d->n_pages == 0 ||
      d->n_pages == CUTB_NO_PAGE || d->ld_table == 0 || d->n_slots == 0) {
    set_last_error("%s: a page holds 16, 32, 64, 128 or 256 tokens, a head 1 .. 256 elements; pages, slots and heads are needed", what);
    return CUTB_ERR_INVALID;
  }
  if (!d->pages || !d->tables || !d->lengths || misaligned(d->pages, 16) || d->page_bytes % 16 ||
      d->page_bytes < layer_bytes(d->n_kv_heads, d->head_dim, d->page_tokens)) {
    set_last_error("%s: null pointer, pages that are not 16-byte aligned, or page_bytes short of a layer's %llu", what,
                   (unsigned long long)layer_bytes(d->n_kv_heads, d->head_dim, d->page_tokens));
    return CUTB_ERR_INVALID;
  }
  if (misaligned(d->tables, 4) || misaligned(d->lengths, 4) || misaligned(d->slots, 4) || misaligned(d->starts, 4) || misaligned(d->status, 4)) {
    set_last_error("%s: tables, lengths, slots, starts and the status word are 4-byte aligned", what);
    return CUTB_ERR_INVALID;
  }
  if (d->n_seqs > PG_MAX_SEQS || (!d->slots && d->n_seqs > d->n_slots) || (!d->starts && d->n_tokens < d->n_seqs) || (d->n_seqs && d->n_tokens && d->max_new == 0)) {
    set_last_error("%s: at most %u sequences, a slot and a row for each, and max_new at least 1", what, PG_MAX_SEQS);
    return CUTB_ERR_INVALID;
  }
  if (d->n_tokens > 0x7fffffffu || (uint64_t)d->ld_table * d->page_tokens > 0x7fffffffull) {
    set_last_error("%s: rows and a table's tokens are counted in 31 bits", what);
    return CUTB_ERR_INVALID;
  }
  if ((uint64_t)d->n_tokens * (2ull * d->n_kv_heads + d->n_heads) > 0x3ffffffffull) {
    set_last_error("%s: heads of rows are counted in 34 bits", what);
    return CUTB_ERR_INVALID;
  }
  return CUTB_OK;
}

int check_rows(const cutb_paged_desc *d, const char *what, const void *p, uint64_t ld, uint32_t heads) {
  if (!p || misaligned(p, type_bytes(d->dtype)) || (d->n_tokens > 1 && ld < (uint64_t)heads * d->head_dim)) {
    set_last_error("%s: null or misaligned rows, or a row stride (%llu) that does not hold %u heads", what, (unsigned long long)ld, heads);
    return CUTB_ERR_INVALID;
  }
  return CUTB_OK;
}

int check_heads(const cutb_paged_desc *d, const char *what) {
  if (d->n_heads == 0 || d->n_heads > 65535 || d->n_heads % d->n_kv_heads) {
    set_last_error("%s: n_heads (%u) must be a multiple of n_kv_heads (%u)", what, d->n_heads, d->n_kv_heads);
    return CUTB_ERR_INVALID;
  }
  return CUTB_OK;
}

int check_pages(const cutb_pages_desc *d, const char *what, bool slots, bool moves) {
  if (!d || d->n_pages == 0 || d->n_pages > 0x7fffffffu || (slots && (!d->tables || !d->lengths || !d->refs || d->ld_table == 0 || d->n_slots == 0 || !page_size_ok(d->page_tokens) ||
                                               (uint64_t)d->ld_table * d->page_tokens > 0x7fffffffull))) {
    set_last_error("%s: null pointer, no pages or slots, or a page that does not hold 16, 32, 64, 128 or 256 tokens", what);
    return CUTB_ERR_INVALID;
  }
  if (misaligned(d->tables, 4) || misaligned(d->lengths, 4) || misaligned(d->refs, 4) || misaligned(d->status, 4)) {
    set_last_error("%s: tables, lengths, refs and the status word are 4-byte aligned", what);
    return CUTB_ERR_INVALID;
  }
  if (moves && (!d->pages || misaligned(d->pages, 16) || d->page_bytes == 0 || d->page_bytes % 16 || d->page_bytes > (1ull << 40))) {
    set_last_error("%s: pages must be 16-byte aligned, page_bytes a multiple of 16", what);
    return CUTB_ERR_INVALID;
  }
  return CUTB_OK;
}

int check_items(const cutb_pages_desc *d, const char *what, uint32_t most, bool pairs, bool counts) {
  if (misaligned(d->items, 4) || misaligned(d->others, 4) || misaligned(d->counts, 4)) {
    set_last_error("%s: entries are 4-byte aligned", what);
    return CUTB_ERR_INVALID;
  }
  if (d->n > most || (d->n && (!d->items || (pairs && !d->others) || (counts && !d->counts)))) {
    set_last_error("%s: null entries, or more than %u of them", what, most);
    return CUTB_ERR_INVALID;
  }
  return CUTB_OK;
}

uint64_t pages_workspace(const cutb_pages_desc &d) {
  const uint64_t most = d.n_pages > 1024 ? d.n_pages : 1024;
  return 256 + 4 * (2 * most + (uint64_t)d.n_pages);
}

int check_workspace(const char *what, const void *ws, uint64_t have, uint64_t need) {
  if (need && (!ws || have < need || misaligned(ws, 256))) {
    set_last_error("%s: needs a 256-byte aligned workspace of %llu bytes", what, (unsigned long long)need);
    return CUTB_ERR_WORKSPACE;
  }
  return CUTB_OK;
}

}  // namespace
}  // namespace cutb

using namespace cutb;

extern "C" {

uint64_t cutb_paged_layer_bytes(uint32_t n_kv_heads, uint32_t head_dim, uint32_t page_tokens) {
  if (n_kv_heads == 0 || head_dim == 0 || head_dim > 256 || !page_size_ok(page_tokens)) return 0;
  return layer_bytes(n_kv_heads, head_dim, page_tokens);
}

int cutb_paged_kv_write(const cutb_paged_desc *d, void *stream) {
  const char *what = "paged_kv_write";
  if (int rc = check_paged(d, what)) return rc;
  if (d->n_tokens == 0 || d->n_seqs == 0) return CUTB_OK;
  if (int rc = check_rows(d, what, d->k, d->ldk, d->n_kv_heads)) return rc;
  if (int rc = check_rows(d, what, d->v, d->ldv, d->n_kv_heads)) return rc;
  if (d->q) {
    if (int rc = check_heads(d, what)) return rc;
    if (int rc = check_rows(d, what, d->q, d->ldq, d->n_heads)) return rc;
    if (int rc = check_rows(d, what, d->q_out, d->ldq_out, d->n_heads)) return rc;
  }
  if (d->q && d->q == d->q_out && d->rot_dims) {
    set_last_error("%s: the turned queries go to rows of their own", what);
    return CUTB_ERR_INVALID;
  }
  if (d->rot_dims % 2 || d->rot_dims > d->head_dim || (d->rot_dims && (!d->cos_table || !d->sin_table || misaligned(d->cos_table, 4) || misaligned(d->sin_table, 4) || d->max_pos == 0)) || d->rot_pairing < 0 || d->rot_pairing > 1) {
    set_last_error("%s: rot_dims must be even and at most head_dim, with tables and a pairing of 0 or 1", what);
    return CUTB_ERR_INVALID;
  }
  return paged_kv_write_launch(*d, reinterpret_cast<cudaStream_t>(stream));
}

int cutb_paged_kv_read(const cutb_paged_desc *d, void *stream) {
  const char *what = "paged_kv_read";
  if (int rc = check_paged(d, what)) return rc;
  if (d->n_tokens == 0 || d->n_seqs == 0) return CUTB_OK;
  if (int rc = check_rows(d, what, d->k_out, d->ldk_out, d->n_kv_heads)) return rc;
  if (int rc = check_rows(d, what, d->v_out, d->ldv_out, d->n_kv_heads)) return rc;
  return paged_kv_read_launch(*d, reinterpret_cast<cudaStream_t>(stream));
}

uint64_t cutb_paged_workspace_bytes(const cutb_paged_desc *d) {
  if (check_paged(d, "paged_attention") != CUTB_OK || check_heads(d, "paged_attention") != CUTB_OK || d->n_tokens == 0 || d->n_seqs == 0) return 0;
  return paged_attention_workspace(*d);
}

int cutb_paged_attention(const cutb_paged_desc *d, void *stream) {
  const char *what = "paged_attention";
  if (int rc = check_paged(d, what)) return rc;
  if (int rc = check_heads(d, what)) return rc;
  if (d->n_tokens == 0 || d->n_seqs == 0) return CUTB_OK;
  if (int rc = check_rows(d, what, d->q, d->ldq, d->n_heads)) return rc;
  if (int rc = check_rows(d, what, d->out, d->ldo, d->n_heads)) return rc;
  if ((uint64_t)d->n_tokens * (d->n_heads / d->n_kv_heads) > 0x7fffffffu) {
    set_last_error("%s: rows times query heads of a KV head are counted in 31 bits", what);
    return CUTB_ERR_INVALID;
  }
  if (!(d->scale - d->scale == 0.f)) {
    set_last_error("%s: the scale must be finite", what);
    return CUTB_ERR_INVALID;
  }
  if (int rc = check_workspace(what, d->workspace, d->workspace_bytes, paged_attention_workspace(*d))) return rc;
  return paged_attention_launch(*d, reinterpret_cast<cudaStream_t>(stream));
}

uint64_t cutb_pages_workspace_bytes(const cutb_pages_desc *d) { return d && d->n_pages && d->n_pages <= 0x7fffffffu ? pages_workspace(*d) : 0; }

int cutb_pages_reserve(const cutb_pages_desc *d, void *stream) {
  const char *what = "pages_reserve";
  if (int rc = check_pages(d, what, true, true)) return rc;
  if (int rc = check_items(d, what, 1024, false, true)) return rc;
  if ((uint64_t)d->n * (d->ld_table + 1) > 0xffffffffull) {
    set_last_error("%s: the entries' tables are counted in 32 bits together", what);
    return CUTB_ERR_INVALID;
  }
  if (int rc = check_workspace(what, d->workspace, d->workspace_bytes, pages_workspace(*d))) return rc;
  return d->n ? pages_reserve_launch(*d, reinterpret_cast<cudaStream_t>(stream)) : (int)CUTB_OK;
}

int cutb_pages_fork(const cutb_pages_desc *d, void *stream) {
  const char *what = "pages_fork";
  if (int rc = check_pages(d, what, true, false)) return rc;
  if (int rc = check_items(d, what, 1024, true, false)) return rc;
  return d->n ? pages_fork_launch(*d, reinterpret_cast<cudaStream_t>(stream)) : (int)CUTB_OK;
}

int cutb_pages_free(const cutb_pages_desc *d, void *stream) {
  const char *what = "pages_free";
  if (int rc = check_pages(d, what, true, false)) return rc;
  if (int rc = check_items(d, what, 1024, false, false)) return rc;
  return d->n ? pages_free_launch(*d, reinterpret_cast<cudaStream_t>(stream)) : (int)CUTB_OK;
}

int cutb_pages_compact(const cutb_pages_desc *d, void *stream) {
  const char *what = "pages_compact";
  if (int rc = check_pages(d, what, true, true)) return rc;
  if (int rc = check_workspace(what, d->workspace, d->workspace_bytes, pages_workspace(*d))) return rc;
  return pages_compact_launch(*d, reinterpret_cast<cudaStream_t>(stream));
}

int cutb_pages_copy(const cutb_pages_desc *d, void *stream) {
  const char *what = "pages_copy";
  if (int rc = check_pages(d, what, false, true)) return rc;
  if (int rc = check_items(d, what, 65535, true, false)) return rc;
  return d->n ? pages_copy_launch(*d, reinterpret_cast<cudaStream_t>(stream)) : (int)CUTB_OK;
}

}  // extern "C"
