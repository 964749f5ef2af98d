"""Refusals of the paged cache's and the sampler's entry points: host logic, answered without a GPU."""
import ctypes as C

import pytest
import torch

from cut_b200 import _lib as L
from cut_b200 import ops
from cut_b200.paged import PagedCache


def desc(**kw):
    d = L.PagedDesc()
    base = dict(pages=4096, page_bytes=81920, ld_table=8, n_pages=4, page_tokens=64, n_kv_heads=8, head_dim=128, tables=256, lengths=256,
                n_slots=2, n_seqs=2, n_tokens=2, max_new=1, dtype=L.F32, n_heads=32, q=256, ldq=4096, k=256, ldk=1024, v=256, ldv=1024,
                q_out=512, ldq_out=4096, k_out=256, ldk_out=1024, v_out=256, ldv_out=1024, out=256, ldo=4096, scale=0.1)
    for k, v in {**base, **kw}.items():
        setattr(d, k, v)
    return d


def refused(name, d, word, code=L.ERR_INVALID):
    lib = L.lib()
    assert getattr(lib, name)(C.byref(d) if d is not None else None, None) == code, (name, word, lib.cutb_last_error())
    assert word in lib.cutb_last_error().decode(), (word, lib.cutb_last_error())


CALLS = ("cutb_paged_kv_write", "cutb_paged_kv_read", "cutb_paged_attention")


def test_struct_sizes_are_the_headers():
    assert (C.sizeof(L.PagedDesc), C.sizeof(L.PagesDesc), C.sizeof(L.SampleDesc)) == (272, 112, 96)


def test_layer_bytes():
    f = L.lib().cutb_paged_layer_bytes
    assert f(8, 128, 64) == 8 * 4 * 20 * 128 and f(1, 1, 16) == 20 * 64 and f(3, 129, 256) == 3 * 16 * 20 * 192
    assert f(8, 128, 48) == f(8, 128, 8) == f(8, 128, 512) == f(0, 128, 64) == f(8, 257, 64) == f(8, 0, 64) == 0


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("kw,word", [({"dtype": 7}, "element type"), ({"page_tokens": 48}, "a page holds"), ({"head_dim": 257}, "a page holds"),
                                     ({"head_dim": 0}, "a page holds"), ({"n_pages": 0}, "a page holds"), ({"ld_table": 0}, "a page holds"),
                                     ({"pages": None}, "null pointer"), ({"pages": 4104}, "16-byte"), ({"page_bytes": 81904}, "short of"),
                                     ({"page_bytes": 81928}, "16-byte"), ({"tables": None}, "null pointer"), ({"lengths": None}, "null pointer"),
                                     ({"n_seqs": 3, "n_tokens": 3}, "sequences"), ({"n_tokens": 1}, "sequences"), ({"max_new": 0}, "max_new"),
                                     ({"n_seqs": 1025, "slots": 256, "n_tokens": 1025}, "sequences"), ({"ld_table": 1 << 30}, "31 bits")])
def test_caches_and_sequences_that_are_refused(name, kw, word):
    refused(name, desc(**kw), word)


def test_rows_that_are_refused():
    for name in CALLS:
        refused(name, None, "null descriptor")
        assert getattr(L.lib(), name)(C.byref(desc(n_tokens=0, n_seqs=0)), None) == L.OK  # nothing to do
    refused("cutb_paged_kv_write", desc(k=None), "rows")
    refused("cutb_paged_kv_write", desc(v=258), "rows")
    refused("cutb_paged_kv_write", desc(ldk=1023), "rows")
    refused("cutb_paged_kv_write", desc(n_heads=12), "multiple")
    refused("cutb_paged_kv_write", desc(q_out=None), "rows")
    refused("cutb_paged_kv_write", desc(rot_dims=3), "rot_dims")
    refused("cutb_paged_kv_write", desc(rot_dims=130, cos_table=256, sin_table=256, max_pos=9), "rot_dims")
    refused("cutb_paged_kv_write", desc(rot_dims=128), "tables")
    refused("cutb_paged_kv_write", desc(rot_dims=128, cos_table=256, sin_table=256, max_pos=9, rot_pairing=2), "pairing")
    refused("cutb_paged_kv_write", desc(rot_dims=128, cos_table=256, sin_table=256, max_pos=9, q_out=256), "of their own")
    refused("cutb_paged_kv_read", desc(v_out=None), "rows")
    refused("cutb_paged_attention", desc(n_heads=0), "multiple")
    refused("cutb_paged_attention", desc(out=None), "rows")
    refused("cutb_paged_attention", desc(ldq=4095), "rows")
    refused("cutb_paged_attention", desc(scale=float("nan")), "finite")
    refused("cutb_paged_attention", desc(scale=float("inf")), "finite")
    assert L.lib().cutb_paged_workspace_bytes(C.byref(desc(page_tokens=48))) == 0


def pages(**kw):
    d = L.PagesDesc()
    base = dict(pages=4096, page_bytes=4096, ld_table=8, n_pages=4, page_tokens=64, n_slots=2, n=1, tables=256, lengths=256, refs=256, items=256,
                others=256, counts=256, workspace=4096, workspace_bytes=1 << 20)
    for k, v in {**base, **kw}.items():
        setattr(d, k, v)
    return d


def test_bookkeeping_that_is_refused():
    for name in ("reserve", "fork", "free", "compact"):
        for kw in ({"tables": None}, {"lengths": None}, {"refs": None}, {"n_pages": 0}, {"n_slots": 0}, {"page_tokens": 12}, {"ld_table": 1 << 30}):
            refused("cutb_pages_" + name, pages(**kw), "a page that does not hold")
    for name in ("reserve", "compact", "copy"):
        for kw in ({"pages": None}, {"pages": 4104}, {"page_bytes": 4104}, {"page_bytes": 0}):
            refused("cutb_pages_" + name, pages(**kw), "16-byte")
    for name in ("reserve", "fork", "free"):
        refused("cutb_pages_" + name, pages(n=1025), "1024")
        refused("cutb_pages_" + name, pages(items=None), "null entries")
        assert getattr(L.lib(), "cutb_pages_" + name)(C.byref(pages(n=0)), None) == L.OK
    refused("cutb_pages_copy", pages(n=65536), "65535")
    refused("cutb_pages_copy", pages(others=None), "null entries")
    refused("cutb_pages_reserve", pages(counts=None), "null entries")
    for name in ("reserve", "compact"):
        refused("cutb_pages_" + name, pages(workspace_bytes=64), "workspace", L.ERR_WORKSPACE)
        refused("cutb_pages_" + name, pages(workspace=4100), "workspace", L.ERR_WORKSPACE)
    assert L.lib().cutb_pages_workspace_bytes(C.byref(pages())) >= 256 and L.lib().cutb_pages_workspace_bytes(None) == 0
    assert L.lib().cutb_status_string(L.ERR_PAGES) == b"too few free pages"


def test_sampling_that_is_refused():
    def s(**kw):
        d = L.SampleDesc()
        for k, v in {**dict(logits=256, ld=100, rows=2, vocab=100, dtype=L.F32, u=256, tokens=256), **kw}.items():
            setattr(d, k, v)
        return d

    refused("cutb_sample", None, "null descriptor")
    refused("cutb_sample", s(dtype=3), "element type")
    refused("cutb_sample", s(vocab=0), "logits")
    refused("cutb_sample", s(vocab=(1 << 19) + 1, ld=1 << 21), "logits")
    refused("cutb_sample", s(ld=99), "stride")
    refused("cutb_sample", s(u=None), "null")
    refused("cutb_sample", s(tokens=None), "null")
    refused("cutb_sample", s(logits=258), "misaligned")
    assert L.lib().cutb_sample(C.byref(s(rows=0)), None) == L.OK


def test_python_refuses_tensors_that_are_not_on_the_device_or_not_alike():
    z = lambda *shape, t=torch.int32: torch.zeros(shape, dtype=t)  # noqa: E731
    with pytest.raises(RuntimeError, match="uint8"):
        PagedCache(z(4, 64), z(2, 2), z(2), z(4))
    with pytest.raises(RuntimeError, match="per table row"):
        PagedCache(z(4, 64, t=torch.uint8), z(2, 2), z(3), z(4))
    with pytest.raises(RuntimeError, match="16 bytes"):
        PagedCache(z(4, 72, t=torch.uint8), z(2, 2), z(2), z(4))
    with pytest.raises(ValueError):
        PagedCache.allocate(4, 2, 64, 8, 257, device="cpu")
    c = PagedCache.allocate(4, 2, 200, 2, 32, n_layers=3, page_tokens=16, device="cpu")
    assert c.pages.shape == (4, 3 * 2 * 20 * 64) and c.tables.shape == (2, 13) and int(c.tables.max()) == -1 and c.layer_bytes() == 2 * 20 * 64
    f = lambda n: torch.zeros(1, n)  # noqa: E731
    with pytest.raises(RuntimeError, match="rows of 2 x 32"):
        ops.paged_kv_write(c, f(63), f(64))
    with pytest.raises(RuntimeError, match="one type"):
        ops.paged_kv_write(c, f(64), f(64).half())
    with pytest.raises(RuntimeError, match="tables"):
        ops.paged_kv_write(c, f(64), f(64), rot_dims=32, cos_t=torch.zeros(4, 8), sin_t=torch.zeros(4, 8))
    with pytest.raises(RuntimeError, match="current CUDA device"):
        ops.paged_kv_write(c, f(64), f(64))
    with pytest.raises(RuntimeError, match="current CUDA device"):
        ops.paged_attention(c, f(128), 4)
    with pytest.raises(RuntimeError, match="current CUDA device"):
        c.fork([0], [1])
    with pytest.raises(RuntimeError, match="one length"):
        c.reserve([0, 1], [1])
    with pytest.raises(RuntimeError, match="current CUDA device"):
        ops.sample(torch.zeros(2, 8), torch.zeros(2))
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        ops.sample(torch.zeros(2, 8, dtype=torch.float64), torch.zeros(2))


def test_misaligned_words_are_refused():
    for name in CALLS:
        for field in ("tables", "lengths", "slots", "starts", "status"):
            refused(name, desc(**{field: 258}), "4-byte aligned")
    refused("cutb_paged_kv_write", desc(rot_dims=128, cos_table=258, sin_table=256, max_pos=9), "tables")
    for name in ("reserve", "fork", "free", "compact"):
        for field in ("tables", "lengths", "refs", "status"):
            refused("cutb_pages_" + name, pages(**{field: 258}), "4-byte aligned")
    refused("cutb_pages_reserve", pages(counts=257), "4-byte aligned")
    refused("cutb_pages_copy", pages(others=258), "4-byte aligned")
    for field in ("temperature", "top_k", "top_p", "min_p", "u", "tokens", "logprobs", "status"):
        d = L.SampleDesc()
        for k, v in {**dict(logits=256, ld=100, rows=2, vocab=100, dtype=L.F32, u=256, tokens=256), field: 258}.items():
            setattr(d, k, v)
        refused("cutb_sample", d, "4-byte aligned")


def test_more_heads_of_rows_than_are_counted():
    for name in CALLS:
        refused(name, desc(n_tokens=0x7fffffff, n_kv_heads=8, n_heads=32, page_bytes=1 << 30), "34 bits")


def test_more_query_rows_than_are_counted():
    refused("cutb_paged_attention", desc(n_tokens=1 << 30, n_kv_heads=1, n_heads=4, head_dim=128, ldq=512, ldo=512), "31 bits")


def test_a_continuation_without_logits_is_refused():
    from cut_b200.decoding import Sampling

    with pytest.raises(RuntimeError, match="logits of the last token"):
        Sampling().decode(None, 1, None)


def test_tables_whose_entries_would_overflow_are_refused():
    refused("cutb_pages_reserve", pages(n=1024, ld_table=1 << 22, page_tokens=16), "32 bits")
    refused("cutb_pages_reserve", pages(n=100, ld_table=1 << 26, page_tokens=16), "32 bits")


def test_pages_that_are_parts_of_wider_ones_are_not_moved():
    """reserve (copy on write), compact and copy take a page whole: of a view of some layers that would be the neighbours' bytes too."""
    z = lambda *shape, t=torch.int32: torch.zeros(shape, dtype=t)  # noqa: E731
    pool = z(4, 256, t=torch.uint8)
    for part in (pool[:, :128], pool[:, 64:192], pool[::2], pool[:, 240:]):
        n = part.shape[0]
        c = PagedCache(part, z(2, 2), z(2), z(n), page_tokens=16)
        for call in (lambda: c.reserve([0], [1]), c.compact, lambda: c.copy([0], [1])):
            with pytest.raises(RuntimeError, match="moved whole"):
                call()
        for call in (lambda: c.fork([0], [1]), lambda: c.free([0])):  # (these touch tables and counts only; the tensors are on the host)
            with pytest.raises(RuntimeError, match="current CUDA device"):
                call()
    for whole in (pool, pool[1:3], pool[2:3, :128]):  # (of one page nothing goes to another)
        c = PagedCache(whole, z(2, 2), z(2), z(whole.shape[0]), page_tokens=16)
        with pytest.raises(RuntimeError, match="current CUDA device"):
            c.reserve([0], [1])
        assert c._desc().page_bytes == whole.shape[1]


def test_tables_that_are_parts_of_wider_ones_are_refused():
    """A sequence may grow to its table's end, and compact follows every entry: beyond a view's columns those are others' entries."""
    z = lambda *shape, t=torch.int32: torch.zeros(shape, dtype=t)  # noqa: E731
    wide, pool = z(4, 8), z(4, 256, t=torch.uint8)
    for tables in (wide[:, :3], wide[:, 5:], wide[::2], torch.as_strided(wide, (4, 8), (2, 1)), z(1, 8).expand(4, 8)):
        with pytest.raises(RuntimeError, match="parts of wider ones"):
            PagedCache(pool, tables, z(tables.shape[0]), z(4))
    for tables in (wide, wide[1:3], wide[3:, 5:], z(4, 1)):  # (one table ends where the view does)
        c = PagedCache(pool, tables, z(tables.shape[0]), z(4), page_tokens=16)
        assert c._desc().ld_table == tables.shape[1]


def test_a_layer_that_a_part_of_the_pages_does_not_hold_is_refused(monkeypatch):
    monkeypatch.setattr(ops, "_here", lambda *a: None)
    c = PagedCache.allocate(4, 2, 200, 2, 32, n_layers=3, page_tokens=16, device="cpu")
    part = c.layer_bytes()
    view = lambda a, b: PagedCache(c.pages[:, a:b], c.tables, c.lengths, c.refs, page_tokens=16, n_kv_heads=2, head_dim=32)  # noqa: E731
    for cache, layer in ((view(0, part - 16), 0), (view(part, 2 * part), 1), (view(0, 2 * part + 16), 2), (c, 3), (c, -1)):
        with pytest.raises(RuntimeError, match="no such layer"):
            ops.paged_desc(cache, 2, torch.float32, layer=layer)
    for cache, layer, at in ((view(part, 2 * part), 0, part), (view(part, 3 * part), 1, 2 * part), (c, 2, 2 * part), (c, 0, 0)):
        assert ops.paged_desc(cache, 2, torch.float32, layer=layer).pages == c.pages.data_ptr() + at


def test_rows_without_a_sequence_of_their_own_are_refused(monkeypatch):
    """Without starts a row belongs to a sequence each: rows that no slot stands for would be dropped, or come back as they were."""
    monkeypatch.setattr(ops, "_here", lambda *a: None)
    c = PagedCache.allocate(4, 4, 200, 2, 32, page_tokens=16, device="cpu")
    f, i32 = lambda n, w: torch.zeros(n, w), lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    for n, slots in ((10, None), (5, None), (3, i32(0, 1)), (1, i32(0, 1)), (1, i32())):
        for call in (lambda: ops.paged_attention(c, f(n, 128), 4, slots=slots), lambda: ops.paged_kv_read(c, n, slots=slots),
                     lambda: ops.paged_kv_write(c, f(n, 64), f(n, 64), slots=slots)):
            with pytest.raises(RuntimeError, match="as many rows as named slots"):
                call()
    with pytest.raises(RuntimeError, match="an entry more"):
        ops.paged_desc(c, 0, torch.float32, starts=i32())
    for n, kw in ((4, {}), (3, {}), (0, {}), (2, dict(slots=i32(3, 1))), (6, dict(slots=i32(0, 1, 2, 3, 3, 3))), (10, dict(starts=i32(0, 3)))):
        d = ops.paged_desc(c, n, torch.float32, **kw)
        assert (d.n_tokens, d.n_seqs) == (n, 1 if "starts" in kw else n)


def test_scratch_of_more_sequences_than_slots(monkeypatch):
    """A call may name a slot more than once: its scratch is that of as many sequences as it names."""
    monkeypatch.setattr(ops, "_here", lambda *a: None)
    seen = []
    monkeypatch.setattr(ops, "paged_workspace_bytes", lambda d: seen.append((d.n_seqs, d.n_tokens, d.n_heads, bool(d.slots))) or 512)
    c = PagedCache.allocate(4, 4, 200, 2, 32, page_tokens=16, device="cpu")
    assert ops.paged_workspace(c, 4, 100, torch.float32).numel() == 512 and seen == [(100, 100, 4, True)]


def test_rows_read_are_zero_where_nothing_is_read(monkeypatch):
    """What is wrong with sequences is found on the device, and with starts their rows are left as they are: not as memory happens to be.
    (Without starts the call itself writes every row.)"""
    monkeypatch.setattr(ops, "_here", lambda *a: None)
    monkeypatch.setattr(ops, "_stream_ptr", lambda: None)
    monkeypatch.setattr(ops.L, "check", lambda rc: None)
    c = PagedCache.allocate(4, 4, 200, 2, 32, page_tokens=16, device="cpu")
    monkeypatch.setattr(torch.Tensor, "new_empty", lambda self, *shape, **kw: self.new_full(shape[0], 7, **kw))

    class Skips:  # a call that reads nothing
        cutb_paged_layer_bytes = L.lib().cutb_paged_layer_bytes
        cutb_paged_kv_read = staticmethod(lambda d, s: 0)

    monkeypatch.setattr(ops.L, "lib", lambda: Skips)
    for starts in ([0, 2], [0, 3], [0]):
        k, v = ops.paged_kv_read(c, 3, dtype=torch.float32, starts=torch.tensor(starts, dtype=torch.int32))
        assert k.shape == v.shape == (3, 64) and k.is_contiguous() and v.is_contiguous() and not k.any() and not v.any()


def test_counts_below_zero_and_other_types_are_refused(monkeypatch):
    """They would come to the call as counts of thousands of millions."""
    monkeypatch.setattr(ops, "_here", lambda *a: None)
    c, q = PagedCache.allocate(4, 4, 200, 2, 32, page_tokens=16, device="cpu"), torch.zeros(2, 128)
    for window in (-1, 1 << 32):
        with pytest.raises(RuntimeError, match="window"):
            ops.paged_attention(c, q, 4, window=window)
    for max_new in (-1, 1 << 32):
        with pytest.raises(RuntimeError, match="max_new"):
            ops.paged_attention(c, q, 4, max_new=max_new)
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        ops.paged_kv_read(c, 2, dtype=torch.float64)


def test_scratch_of_prompts_behind_many_keys():
    """Rows that may see more than 8192 keys have their sums moved to totals in the scratch, 4 bytes an element of whole tiles of rows."""
    need = lambda **kw: L.lib().cutb_paged_workspace_bytes(C.byref(desc(**{**dict(n_seqs=1, n_tokens=1000, max_new=1000, starts=256), **kw})))  # noqa: E731
    tiles = {L.F16: 1000 * 4 // 256 + 1, L.F32: 1000 * 4 // 128 + 1}
    for kind, rows in ((L.F16, 256), (L.F32, 128)):
        assert need(dtype=kind, ld_table=128) == 0  # 8192 keys
        assert need(dtype=kind, ld_table=129) == tiles[kind] * 8 * rows * 128 * 4
        assert need(dtype=kind, ld_table=9999, window=62 * 128 + 1) == 0 and need(dtype=kind, ld_table=9999, window=8192) > 0
        refused("cutb_paged_attention", desc(n_seqs=1, n_tokens=1000, max_new=1000, starts=256, dtype=kind, ld_table=129), "workspace", L.ERR_WORKSPACE)
    assert need(dtype=L.BF16, ld_table=129, n_kv_heads=2, n_heads=6, head_dim=200, ldq=1200, ldo=1200) == (1000 * 3 // 128 + 1) * 2 * 128 * 256 * 4
