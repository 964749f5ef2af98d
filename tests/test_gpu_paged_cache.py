"""The paged 4-bit cache on the GPU: rows written and read back (the bytes too), attention over it, against a plain model in 64 bits."""
import numpy as np
import pytest

import paged_util as P

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def make_cache(lengths, kv, head, page, r, n_layers=1, layer=0, spare=2, fill=255):
    """A cache whose sequences hold pages in a random order; every byte of the pool is `fill` (as fp16 numbers NaN)."""
    from cut_b200.paged import PagedCache

    need = [-(-n // page) for n in lengths]
    order = r.permutation(sum(need) + spare)
    c = PagedCache.allocate(sum(need) + spare, len(lengths), max(1, max(need) + 1) * page, kv, head, n_layers=n_layers, page_tokens=page)
    t, at = -np.ones(tuple(c.tables.shape), dtype=np.int32), 0
    for s, k in enumerate(need):
        t[s, :k] = order[at: at + k]
        at += k
    c.tables.copy_(cuda(t))
    c.lengths.copy_(cuda(np.array(lengths, dtype=np.int32)))
    c.pages.fill_(fill)
    return c


def rows_of(new):
    return cuda(np.concatenate([[0], np.cumsum(new)]).astype(np.int32))


def fill_cache(c, lengths, kv, head, r, spread=1.0):
    """Writes every token; returns the values that the cache holds, [kv, tokens, head] for each sequence."""
    from cut_b200 import ops

    n = sum(lengths)
    if n == 0:
        return [np.zeros((kv, 0, head)) for _ in lengths], [np.zeros((kv, 0, head)) for _ in lengths]
    k, v = (spread * r.standard_normal((n, kv * head))).astype(np.float32), r.standard_normal((n, kv * head)).astype(np.float32)
    ops.paged_kv_write(c, cuda(k), cuda(v), starts=rows_of(lengths))
    cut = np.cumsum([0] + list(lengths))
    out = [[P.quantised(x.reshape(n, kv, head)[a:b])[0].transpose(1, 0, 2) for a, b in zip(cut, cut[1:])] for x in (k, v)]
    return out[0], out[1]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("head,kv,page,rot,pairing", [(128, 2, 64, 128, 0), (64, 1, 16, 32, 1), (40, 3, 32, 40, 0), (192, 2, 16, 64, 1), (256, 1, 128, 256, 0),
                                                      (33, 2, 16, 0, 0), (1, 1, 256, 0, 0), (80, 1, 16, 6, 0), (128, 1, 64, 2, 1)])
def test_written_rows_and_their_bytes(kind, head, kv, page, rot, pairing):
    from cut_b200 import ops

    r = np.random.default_rng(head + page)
    lengths, new, heads = [1, 37, 20, page + 1, 5], [1, 30, 0, page + 1, 2], 2 * kv
    c = make_cache(lengths, kv, head, page, r)
    before = c.pages.cpu().numpy().copy()
    n, t = sum(new), TYPES[kind]
    qkv = (3 * torch.from_numpy(r.standard_normal((n + 2, (heads + 2 * kv) * head)))).to(t).cuda()  # two rows behind the last sequence
    q, k, v = qkv[:, : heads * head], qkv[:, heads * head: (heads + kv) * head], qkv[:, (heads + kv) * head:]  # (strided)
    cos, sin = P.tables_of(head, rot, 300)
    q_out = torch.full((n + 2, heads * head), 7.0, dtype=t, device="cuda")
    kw = dict(rot_dims=rot, pairing=pairing, cos_t=cuda(cos), sin_t=cuda(sin)) if rot else {}
    ops.paged_kv_write(c, k, v, q=q, q_out=q_out, starts=rows_of(new), **kw)
    c.check()
    ko, vo = ops.paged_kv_read(c, n + 2, starts=rows_of(new), dtype=torch.float32)
    c.check()
    x = qkv.float().cpu().numpy()
    pool, tables = c.pages.cpu().numpy(), c.tables.cpu().numpy()
    want_k, want_v, row, touched = [], [], 0, np.zeros(pool.shape, dtype=bool)
    unit_bytes = 20 * P.pad(head)
    for s, m in enumerate(new):
        for i in range(m):
            pos = lengths[s] - m + i
            heads_x = P.turned(x[row, : (heads + kv) * head].reshape(-1, head), pos, cos, sin, rot, pairing)
            got_q = q_out[row].float().cpu().numpy()
            assert np.array_equal(got_q, torch.from_numpy(heads_x[:heads].reshape(-1)).to(t).float().numpy())
            want_k.append(P.quantised(heads_x[heads:])[0].reshape(-1))
            want_v.append(P.quantised(x[row, (heads + kv) * head:].reshape(kv, head))[0].reshape(-1))
            for h in range(kv):
                at = (h * (page // 16) + pos % page // 16) * unit_bytes
                touched[tables[s, pos // page], at: at + unit_bytes] = True
            if i % 7 == 0:  # the bytes, as the layout says
                at = (kv - 1) * (page // 16) * unit_bytes + pos % page // 16 * unit_bytes
                unit = pool[tables[s, pos // page], at: at + unit_bytes]
                assert np.array_equal(P.unit_values(unit, head, "k")[pos % 16], want_k[-1][(kv - 1) * head:])
                assert np.array_equal(P.unit_values(unit, head, "v")[pos % 16], want_v[-1][(kv - 1) * head:])
            row += 1
    assert np.array_equal(ko[:n].cpu().numpy(), np.array(want_k)) and np.array_equal(vo[:n].cpu().numpy(), np.array(want_v))
    assert not ko[n:].any() and not vo[n:].any() and bool((q_out[n:] == 7).all())
    assert np.array_equal(pool[~touched], before[~touched])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("head,kv,page,rot,pairing", [(128, 16, 64, 64, 1), (128, 16, 16, 128, 0), (40, 16, 32, 6, 0), (256, 16, 16, 40, 1), (192, 16, 128, 0, 0)])
def test_many_rows(kind, head, kv, page, rot, pairing):
    """Enough rows for the form that writes and reads whole units, with sequences that begin and end inside of them; in every third row
    numbers that lie halfway between two codes."""
    from cut_b200 import ops

    r = np.random.default_rng(head + rot)
    lengths, new = [400, 37, 30, 9, 160, 1, 75, 60, 51, 90], [333, 5, 0, 9, 160, 1, 75, 22, 50, 67]
    heads, at = 2 * kv, 3  # three rows before the first sequence
    c = make_cache(lengths, kv, head, page, r)
    n, t = sum(new), TYPES[kind]
    rows = at + n + 150
    x = r.standard_normal((rows, (heads + 2 * kv) * head))
    x[::3] = r.integers(0, 31, x[::3].shape)
    qkv = torch.from_numpy(x).to(t).cuda()
    q, k, v = qkv[:, : heads * head], qkv[:, heads * head: (heads + kv) * head], qkv[:, (heads + kv) * head:]
    cos, sin = P.tables_of(head, rot, 500)
    q_out = torch.full((rows, heads * head), 7.0, dtype=t, device="cuda")
    kw = dict(rot_dims=rot, pairing=pairing, cos_t=cuda(cos), sin_t=cuda(sin)) if rot else {}
    starts = rows_of(new) + at
    before = c.pages.clone()
    ops.paged_kv_write(c, k, v, q=q, q_out=q_out, starts=starts, **kw)
    ko, vo = ops.paged_kv_read(c, rows, starts=starts, dtype=torch.float32)
    c.check()
    x = qkv.float().cpu().numpy()
    pos = np.concatenate([np.arange(a - b, a) for a, b in zip(lengths, new)])
    turned = np.stack([P.turned(x[at + i, : (heads + kv) * head].reshape(-1, head), p, cos, sin, rot, pairing) for i, p in enumerate(pos)])
    got = q_out.float().cpu().numpy()
    assert np.array_equal(got[at: at + n], torch.from_numpy(turned[:, :heads].reshape(n, -1)).to(t).float().numpy())
    for out, want in ((ko, turned[:, heads:]), (vo, x[at: at + n, (heads + kv) * head:].reshape(n, kv, head))):
        out = out.cpu().numpy()
        assert np.array_equal(out[at: at + n], P.quantised(want)[0].reshape(n, -1)) and not out[:at].any() and not out[at + n:].any()
    assert (got[:at] == 7).all() and (got[at + n:] == 7).all()
    # the same bytes as from rows a few at a time, and nothing else
    whole = c.pages.clone()
    c.pages.copy_(before)
    cut = np.cumsum([at] + new)
    for s, m in enumerate(new):
        for a in range(0, m, 40):
            part = slice(int(cut[s]) + a, int(cut[s]) + min(a + 40, m))
            c.lengths.copy_(cuda(np.array([min(lengths[s] - m + a + 40, lengths[s]) if j == s else 0 for j in range(len(new))], dtype=np.int32)))
            ops.paged_kv_write(c, k[part], v[part], starts=rows_of([part.stop - part.start]), slots=cuda(np.array([s], dtype=np.int32)), **kw)
    c.check()
    assert torch.equal(c.pages, whole)


def test_values_that_the_cache_cannot_hold():
    from cut_b200 import _lib as L
    from cut_b200 import ops

    r = np.random.default_rng(0)
    c = make_cache([3], 1, 64, 16, r)
    x = r.standard_normal((3, 64)).astype(np.float32)
    x[0, 5], x[0, 40], x[1, 3], x[1, 33], x[2, :32], x[2, 32:] = np.inf, -1e30, np.nan, 7e4, 2.5, 1e-9
    ops.paged_kv_write(c, cuda(x), cuda(x), starts=rows_of([3]))
    with pytest.raises(L.CutbError) as e:
        c.check()
    assert e.value.status == L.ERR_RANGE
    k, v = ops.paged_kv_read(c, 3, starts=rows_of([3]), dtype=torch.float32)
    want, changed = P.quantised(x)
    assert changed and np.isfinite(want).all() and np.array_equal(k.cpu().numpy(), want) and torch.equal(k, v)
    c.check()


def test_values_that_the_cache_cannot_hold_among_many_rows():
    from cut_b200 import _lib as L
    from cut_b200 import ops

    r = np.random.default_rng(1)
    n, kv = 700, 32
    c = make_cache([n], kv, 64, 32, r)
    x = r.standard_normal((n, kv * 64)).astype(np.float32)
    at = r.integers(0, x.size, 400)
    x.reshape(-1)[at] = r.choice(np.array([np.inf, -np.inf, np.nan, 1e30, -7e4, 32768.0, 1e-40], dtype=np.float32), 400)
    x[5, :64], x[6, :32] = np.nan, np.inf
    ops.paged_kv_write(c, cuda(x), cuda(x), starts=rows_of([n]))
    with pytest.raises(L.CutbError) as e:
        c.check()
    assert e.value.status == L.ERR_RANGE
    k, v = ops.paged_kv_read(c, n, starts=rows_of([n]), dtype=torch.float32)
    c.check()
    want = P.quantised(x.reshape(n, kv, 64))[0].reshape(n, -1)
    assert np.isfinite(want).all() and np.array_equal(k.cpu().numpy(), want) and torch.equal(k, v)


CASES = [  # head, query heads, kv heads, page, lengths, new rows, window
    (128, 8, 2, 64, [1, 15, 16, 17, 64, 65, 300], [1] * 7, 0),
    (128, 8, 1, 16, [200, 33], [1, 1], 0),
    (128, 4, 4, 16, [70, 0, 129], [1, 0, 1], 0),
    (64, 6, 2, 32, [50, 100], [1, 1], 20),
    (40, 3, 1, 16, [31, 90], [1, 1], 0),
    (192, 14, 2, 16, [40, 21], [1, 1], 7),
    (256, 16, 1, 64, [100, 3], [1, 1], 0),
    (96, 24, 1, 32, [77], [1], 0),
    (128, 8, 2, 64, [40, 130, 9], [3, 5, 2], 0),
    (128, 32, 8, 64, [200, 70, 33], [150, 70, 1], 0),
    (128, 4, 2, 16, [333], [333], 0),
    (64, 4, 4, 16, [290, 60], [129, 60], 33),
    (256, 4, 1, 32, [150], [100], 0),
    (80, 5, 5, 16, [140, 12], [139, 12], 1),
    (192, 2, 2, 128, [260], [130], 100),
    (128, 20, 1, 64, [90], [50], 0),
]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("head,nh,kv,page,lengths,new,window", CASES)
def test_attention(kind, head, nh, kv, page, lengths, new, window):
    from cut_b200 import ops

    r = np.random.default_rng(head + nh + len(lengths))
    c = make_cache(lengths, kv, head, page, r)
    ks, vs = fill_cache(c, lengths, kv, head, r, spread=2.0)
    n, t = sum(new), TYPES[kind]
    q = torch.from_numpy(1.5 * r.standard_normal((n + 3, nh * head))).to(t).cuda()  # three rows behind the last sequence
    out = torch.full((n + 3, nh * head), 7.0, dtype=t, device="cuda")
    ops.paged_attention(c, q, nh, starts=rows_of(new), max_new=max(new), window=window, out=out)
    c.check()
    x, got, row, scale = q.double().cpu().numpy(), out.double().cpu().numpy(), 0, float(np.float32(head ** -0.5))
    for s, m in enumerate(new):
        for i in range(m):
            for h in range(nh):
                y, spread, products = P.attention(x[row, h * head: (h + 1) * head], ks[s][h * kv // nh], vs[s][h * kv // nh], lengths[s] - m + i, scale, window)
                off = np.abs(got[row, h * head: (h + 1) * head] - y) - P.tolerance(y, spread, products, scale, kind)
                assert off.max() <= 0, (s, i, h, off.max(), int(off.argmax()))
            row += 1
    assert bool((out[n:] == 7).all())


def test_one_row_each_slots_layers_and_strides():
    """Sequences by slot in an order of their own, one row each; the second layer of a cache; rows inside a wider matrix."""
    from cut_b200 import ops

    r = np.random.default_rng(5)
    lengths, kv, head, nh = [20, 60, 33, 90], 2, 64, 4
    c = make_cache(lengths, kv, head, 16, r, n_layers=3)
    part = c.layer_bytes()
    from cut_b200.paged import PagedCache

    second = PagedCache(c.pages[:, part: 2 * part], c.tables, c.lengths, c.refs, page_tokens=16, n_kv_heads=kv, head_dim=head, status=c.status)
    ks, vs = fill_cache(second, lengths, kv, head, r)
    assert bool((c.pages[:, :part] == 255).all()) and bool((c.pages[:, 2 * part:] == 255).all())
    wide = torch.from_numpy(r.standard_normal((2, nh * head + 24)).astype(np.float32)).cuda()
    q, slots = wide[:, 8: 8 + nh * head], [3, 1]
    out = ops.paged_attention(c, q, nh, slots=cuda(np.array(slots, dtype=np.int32)), layer=1, scale=-0.3)
    c.check()
    x, got = q.double().cpu().numpy(), out.double().cpu().numpy()
    for i, s in enumerate(slots):
        for h in range(nh):
            y, spread, products = P.attention(x[i, h * head: (h + 1) * head], ks[s][h // 2], vs[s][h // 2], lengths[s] - 1, float(np.float32(-0.3)), 0)
            assert (np.abs(got[i, h * head: (h + 1) * head] - y) <= P.tolerance(y, spread, products, 0.3, "f32")).all()


@pytest.mark.parametrize("new", [1, 40])
def test_bad_pages_slots_and_lengths_are_left_out_and_reported(new):
    from cut_b200 import _lib as L
    from cut_b200 import ops

    r = np.random.default_rng(6)
    lengths, kv, head, nh = [60, 60, 60, 60, 60, 60], 1, 64, 2
    c = make_cache(lengths, kv, head, 16, r)
    ks, vs = fill_cache(c, lengths, kv, head, r)
    c.check()
    c.tables[1, 1] = 1 << 20           # a page that does not exist: its keys are not there
    c.lengths[2] = 1 << 30             # longer than the table
    c.lengths[3] = new - 1             # shorter than the new rows
    slots = cuda(np.array([0, 1, 2, 3, 77, 5], dtype=np.int32))
    q = torch.from_numpy(r.standard_normal((6 * new, nh * head)).astype(np.float32)).cuda()
    starts = rows_of([new] * 6)
    out = torch.full_like(q, 7.0)
    ops.paged_attention(c, q, nh, starts=starts, slots=slots, max_new=new, out=out)
    with pytest.raises(L.CutbError) as e:
        c.check()
    assert e.value.status == L.ERR_INVALID
    x, got = q.double().cpu().numpy(), out.double().cpu().numpy()
    assert (got[2 * new: 5 * new] == 7).all()
    for s in (0, 1, 5):
        keep = np.r_[0:16, 32:60] if s == 1 else np.r_[0:60]
        for i in (0, new - 1):
            pos = 60 - new + i
            seen = keep[keep <= pos]
            for h in range(nh):
                y, spread, products = P.attention(x[s * new + i, h * head: (h + 1) * head], ks[s][0][seen], vs[s][0][seen], len(seen) - 1, 0.125, 0)
                assert (np.abs(got[s * new + i, h * head: (h + 1) * head] - y) <= P.tolerance(y, spread, products, 0.125, "f32")).all(), (s, i, h)
    # the same to be written: nothing of it is touched, the others are
    before = c.pages.clone()
    k = torch.from_numpy(r.standard_normal((6 * new, head)).astype(np.float32)).cuda()
    c.tables[0, 3] = -5  # (the last page of slot 0)
    ops.paged_kv_write(c, k, k, starts=starts, slots=slots, max_new=new)
    with pytest.raises(L.CutbError) as e:
        c.check()
    assert e.value.status == L.ERR_INVALID
    changed = (c.pages != before).any(1).nonzero().view(-1).tolist()
    own = set(c.tables[5, :4].tolist()) | set(c.tables[1, 2:4].tolist()) | (set(c.tables[0, 1:3].tolist()) | {int(c.tables[1, 0])} if new > 1 else set())
    assert set(changed) <= own and int(c.tables[5, 3]) in changed


def test_positions_past_the_tables_and_rows_past_the_call():
    from cut_b200 import _lib as L
    from cut_b200 import ops

    r = np.random.default_rng(7)
    c = make_cache([20, 20], 1, 64, 16, r)
    cos, sin = P.tables_of(64, 64, 18)
    k = torch.from_numpy(r.standard_normal((6, 64)).astype(np.float32)).cuda()
    ops.paged_kv_write(c, k, k, starts=rows_of([3, 3]), rot_dims=64, cos_t=cuda(cos), sin_t=cuda(sin))  # positions 17, 18, 19
    with pytest.raises(L.CutbError):
        c.check()
    ko, _ = ops.paged_kv_read(c, 6, starts=rows_of([3, 3]), dtype=torch.float32)
    assert np.isfinite(ko.cpu().numpy()[[0, 3]]).all() and np.isnan(ko.cpu().numpy()[[1, 2, 4, 5]]).all()
    for starts, max_new in (([0, 4, 9], 8), ([0, 2, 1], 8), ([0, 3, 6], 2)):  # behind the rows, falling, more than max_new
        out = torch.full((6, 64), 7.0, device="cuda")
        c.pages.zero_()
        ops.paged_attention(c, torch.ones(6, 64, device="cuda"), 1, starts=cuda(np.array(starts, dtype=np.int32)), max_new=max_new, out=out)
        with pytest.raises(L.CutbError):
            c.check()
        assert bool((out[4:] == 7).all())


def test_scores_that_jump_and_a_zero_scale():
    """Large scores that rise along the keys (the running maximum follows), and a scale of zero (the mean of the values)."""
    from cut_b200 import ops

    r = np.random.default_rng(8)
    n, head = 700, 128
    c = make_cache([n], 1, head, 64, r)
    direction = r.standard_normal(head)
    k = (np.linspace(-6, 6, n)[:, None] * direction + 0.1 * r.standard_normal((n, head))).astype(np.float32)
    v = r.standard_normal((n, head)).astype(np.float32)
    ops.paged_kv_write(c, cuda(k), cuda(v), starts=rows_of([n]))
    kq, vq = P.quantised(k)[0], P.quantised(v)[0]
    for rows in (1, 200):
        q = np.tile(direction.astype(np.float32), (rows, 4))
        q[:, head:] *= np.float32(-1)
        for scale in (1.0, 0.0):
            out = ops.paged_attention(c, cuda(q), 4, starts=rows_of([rows]), max_new=rows, scale=scale).double().cpu().numpy()
            for i in {0, rows - 1}:
                for h in (0, 1):
                    y, spread, products = P.attention(q[i, h * head: (h + 1) * head].astype(np.float64), kq, vq, n - rows + i, scale, 0)
                    assert (np.abs(out[i, h * head: (h + 1) * head] - y) <= P.tolerance(y, spread, products, scale, "f32")).all(), (rows, scale, i, h)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_long_sequences_share_their_work(kind):
    from cut_b200 import ops

    r = np.random.default_rng(9)
    lengths, kv, head, nh = [20000, 17, 5000], 1, 128, 4
    c = make_cache(lengths, kv, head, 64, r)
    ks, vs = fill_cache(c, lengths, kv, head, r)
    q = torch.from_numpy(r.standard_normal((3, nh * head))).to(TYPES[kind]).cuda()
    got = ops.paged_attention(c, q, nh).double().cpu().numpy()
    again = ops.paged_attention(c, q, nh).double().cpu().numpy()
    assert np.array_equal(got, again)
    x, scale = q.double().cpu().numpy(), float(np.float32(head ** -0.5))
    for s in range(3):
        for h in range(nh):
            y, spread, products = P.attention(x[s, h * head: (h + 1) * head], ks[s][0], vs[s][0], lengths[s] - 1, scale, 0)
            assert (np.abs(got[s, h * head: (h + 1) * head] - y) <= P.tolerance(y, spread, products, scale, kind)).all(), (s, h)


def test_offsets_past_32_bits():
    """A pool of over 4 GB, the sequence in its last pages."""
    from cut_b200 import ops
    from cut_b200.paged import PagedCache

    r = np.random.default_rng(10)
    c = PagedCache.allocate(4200, 1, 256, 1, 128, page_tokens=64)
    pages = torch.zeros((4200, 1 << 20), dtype=torch.uint8, device="cuda")
    c = PagedCache(pages, c.tables, c.lengths, c.refs, page_tokens=64, n_kv_heads=1, head_dim=128, status=c.status)
    c.tables[0, :3] = torch.tensor([4199, 1, 4198], dtype=torch.int32)
    c.lengths[0] = 150
    ks, vs = fill_cache(c, [150], 1, 128, r)
    q = torch.from_numpy(r.standard_normal((1, 256)).astype(np.float32)).cuda()
    got = ops.paged_attention(c, q, 2).double().cpu().numpy()
    for h in range(2):
        y, spread, products = P.attention(q.double().cpu().numpy()[0, h * 128: (h + 1) * 128], ks[0][0], vs[0][0], 149, 128 ** -0.5, 0)
        assert (np.abs(got[0, h * 128: (h + 1) * 128] - y) <= P.tolerance(y, spread, products, 128 ** -0.5, "f32")).all()
    c.check()


def test_recorded_calls_follow_the_lengths_and_streams_stay_apart():
    """A step recorded once serves later steps; two recorded calls with workspaces of their own run on two streams."""
    from cut_b200 import ops

    r = np.random.default_rng(11)
    kv, head, nh = 2, 128, 8
    lengths = [400, 100]
    c = make_cache([500, 500], kv, head, 64, r)
    ks, vs = fill_cache(c, [500, 500], kv, head, r)
    q = torch.from_numpy(r.standard_normal((2, nh * head)).astype(np.float32)).cuda()
    outs = [torch.zeros_like(q) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs = []
    for out, st in zip(outs, streams):
        with torch.cuda.stream(st):
            ops.paged_attention(c, q, nh, out=out)
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                ops.paged_attention(c, q, nh, out=out)
            graphs.append(g)
    for lengths in ([400, 100], [7, 500], [500, 1]):
        c.lengths.copy_(cuda(np.array(lengths, dtype=np.int32)))
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1])
        got, x = outs[0].double().cpu().numpy(), q.double().cpu().numpy()
        for s in range(2):
            for h in (0, nh - 1):
                y, spread, products = P.attention(x[s, h * head: (h + 1) * head], ks[s][h * kv // nh], vs[s][h * kv // nh], lengths[s] - 1, 128 ** -0.5, 0)
                assert (np.abs(got[s, h * head: (h + 1) * head] - y) <= P.tolerance(y, spread, products, 128 ** -0.5, "f32")).all()


def test_what_is_wrong_among_many_rows_is_left_out_and_reported():
    from cut_b200 import _lib as L
    from cut_b200 import ops

    r = np.random.default_rng(8)
    kv, head, new, page = 32, 64, 120, 16
    c = make_cache([150] * 6, kv, head, page, r)
    good = c.tables.clone()
    c.tables[1, 4] = 1 << 20   # a page that does not exist: tokens 64 .. 79
    c.tables[0, 9] = -5        # tokens 144 .. 149
    c.lengths[2] = 1 << 30     # longer than the table
    c.lengths[3] = new - 1     # shorter than the new rows
    slots = cuda(np.array([0, 1, 2, 3, 77, 5], dtype=np.int32))
    k, v, q = (torch.from_numpy(r.standard_normal((6 * new + 40, kv * head)).astype(np.float32)).cuda() for _ in range(3))
    cos, sin = P.tables_of(head, 16, 140)  # and no positions past 139
    starts, before = rows_of([new] * 6), c.pages.clone()
    q_out = torch.full_like(q, 7.0)
    ops.paged_kv_write(c, k, v, q=q, q_out=q_out, starts=starts, slots=slots, max_new=new, rot_dims=16, cos_t=cuda(cos), sin_t=cuda(sin))
    with pytest.raises(L.CutbError) as e:
        c.check()
    assert e.value.status == L.ERR_INVALID
    ko, vo = ops.paged_kv_read(c, 6 * new + 40, starts=starts, slots=slots, max_new=new, dtype=torch.float32)
    with pytest.raises(L.CutbError):
        c.check()
    ko, vo, q_out, x, y, z = (a.cpu().numpy() for a in (ko, vo, q_out, k, v, q))
    written, bad = np.zeros(6 * new + 40, dtype=bool), np.zeros(6 * new + 40, dtype=bool)
    for s in range(6):
        for i in range(new):
            pos, row = 150 - new + i, s * new + i
            bad[row] = s in (2, 3, 4) or (s == 1 and pos // page == 4) or (s == 0 and pos // page == 9)
            written[row] = not bad[row] and pos < 140
            if written[row]:
                assert np.array_equal(ko[row], P.quantised(P.turned(x[row].reshape(kv, head), pos, cos, sin, 16, 0))[0].reshape(-1)), row
                assert np.array_equal(q_out[row], P.turned(z[row].reshape(kv, head), pos, cos, sin, 16, 0).reshape(-1)), row
    assert np.array_equal(vo[written], P.quantised(y[written].reshape(-1, kv, head))[0].reshape(written.sum(), -1))
    assert (q_out[~written] == 7).all() and not ko[bad].any() and not vo[bad].any() and not ko[6 * new:].any()
    assert np.isnan(ko[: 6 * new][~written[: 6 * new] & ~bad[: 6 * new]]).all()  # the pool as it was
    changed = (c.pages != before).any(1).nonzero().view(-1).tolist()
    assert set(changed) <= set(good[0, 1:9].tolist()) | set(good[1, 1:4].tolist()) | set(good[1, 5:9].tolist()) | set(good[5, 1:9].tolist())


def test_many_rows_follow_a_recording_and_pages_past_32_bits():
    """The forms for many rows, recorded once and replayed at other lengths; pages more than 4 GB into the pool."""
    from cut_b200 import ops
    from cut_b200.paged import PagedCache

    r = np.random.default_rng(9)
    kv, head, page, new = 16, 128, 64, 700
    c = PagedCache.allocate(40000, 1, 2048, kv, head, page_tokens=page)
    assert c.pages.numel() > 6 << 30
    ids = (39999 - 1117 * np.arange(32)).astype(np.int32)
    c.tables[0, :32] = cuda(ids)
    k, v = (torch.from_numpy(r.standard_normal((new, kv * head)).astype(np.float32)).cuda() for _ in range(2))
    starts = rows_of([new])
    c.lengths.fill_(1500)
    ops.paged_kv_write(c, k, v, starts=starts)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.paged_kv_write(c, k, v, starts=starts)
        ko, vo = ops.paged_kv_read(c, new, starts=starts, dtype=torch.float32)
    for length in (700, 2048, 711):
        c.pages.fill_(255)
        c.lengths.fill_(length)
        k.copy_(torch.randn_like(k)), v.copy_(torch.randn_like(v))
        g.replay()
        c.check()
        for got, want in ((ko, k), (vo, v)):
            assert np.array_equal(got.cpu().numpy(), P.quantised(want.cpu().numpy().reshape(new, kv, head))[0].reshape(new, -1)), length
        touched = set((c.pages != 255).any(1).nonzero().view(-1).tolist())  # (a page that begins before the first row is changed in part)
        assert touched == set(ids[(length - new) // page: -(-length // page)].tolist())


def test_rows_of_slots_that_cannot_be_read_are_zero():
    from cut_b200 import _lib as L
    from cut_b200 import ops

    r = np.random.default_rng(12)
    lengths, kv, head = [20, 33, 0, 7], 2, 64
    c = make_cache(lengths, kv, head, 16, r)
    ks, vs = fill_cache(c, lengths, kv, head, r)
    c.tables[3, 0] = 1 << 20
    slots = cuda(np.array([1, 77, 2, 3, 0], dtype=np.int32))  # the second is none, the third empty, the fourth's page does not exist
    for _ in range(3):
        junk = torch.full((10 * kv * head,), 7.0, device="cuda")  # (what the allocator hands out next)
        del junk
        k, v = ops.paged_kv_read(c, 5, slots=slots, dtype=torch.float32)
        with pytest.raises(L.CutbError) as e:
            c.check()
        assert e.value.status == L.ERR_INVALID
        for got, want in ((k, ks), (v, vs)):
            got = got.cpu().numpy()
            assert not got[1:4].any()
            assert np.array_equal(got[0], want[1][:, -1].reshape(-1)) and np.array_equal(got[4], want[0][:, -1].reshape(-1))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("head,nh,kv,lengths,new", [(128, 4, 2, [90, 40, 33], 1), (128, 4, 2, [2500], 3), (64, 8, 2, [70, 300], 1), (256, 2, 1, [50], 1),
                                                    (128, 4, 2, [300, 90], 60), (64, 4, 4, [150], 150), (192, 4, 1, [100], 40)])
def test_queries_that_are_not_finite_give_nan(kind, head, nh, kv, lengths, new):
    """A NaN or an infinity among a head's queries makes its row NaN, whatever the signs of the scores, and no other row."""
    from cut_b200 import ops

    r = np.random.default_rng(head + new)
    c = make_cache(lengths, kv, head, 16, r)
    n, tokens = len(lengths) * new, sum(lengths)
    k = r.standard_normal((tokens, kv, head)).astype(np.float32)
    k[:, :, 3] = -1 - np.abs(k[:, :, 3])  # (an infinite query element there: minus infinity for all keys)
    v = r.standard_normal((tokens, kv, head)).astype(np.float32)
    ops.paged_kv_write(c, cuda(k.reshape(tokens, -1)), cuda(v.reshape(tokens, -1)), starts=rows_of(lengths))
    cut = np.cumsum([0] + lengths)
    q = torch.from_numpy(r.standard_normal((n, nh, head))).to(TYPES[kind]).cuda()
    bad = {}
    for i, (h, at, what) in enumerate([(0, 5, np.nan), (nh - 1, 3, np.inf), (1, 9, np.inf), (1, 9, -np.inf), (0, 3, -np.inf)]):
        row = i * 7 % n
        q[row, h, at] = what
        if i == 1:
            q[row, h, :3], q[row, h, 4:] = 0, 0
        bad.setdefault(row, set()).add(h)
    out = ops.paged_attention(c, q.view(n, -1), nh, starts=rows_of([new] * len(lengths)), max_new=new)
    c.check()
    x, got, scale = q.double().cpu().numpy(), out.double().cpu().numpy().reshape(n, nh, head), float(np.float32(head ** -0.5))
    kq, vq = P.quantised(k)[0], P.quantised(v)[0]
    for row in range(n):
        s = row // new
        for h in range(nh):
            if h in bad.get(row, ()):
                assert np.isnan(got[row, h]).all(), (row, h)
            elif row < 12 or row % 11 == 0:
                ks, vs = kq[cut[s]: cut[s + 1], h * kv // nh], vq[cut[s]: cut[s + 1], h * kv // nh]
                y, spread, products = P.attention(x[row, h], ks, vs, lengths[s] - new + row % new, scale, 0)
                assert (np.abs(got[row, h] - y) <= P.tolerance(y, spread, products, scale, kind)).all(), (row, h)


def repeated(c, tokens, kv, head, r):
    """Fills pages 0, 1, .. of a cache whose table names them over and over, with positive values: what the cache holds of its
    first `tokens` tokens, [kv, tokens, head] twice."""
    from cut_b200 import ops

    width = c.tables.shape[1]
    c.tables.copy_((torch.arange(width, dtype=torch.int32) % (tokens // c.page_tokens)).expand_as(c.tables))
    k, v = r.standard_normal((tokens, kv, head)).astype(np.float32), r.random((tokens, kv, head)).astype(np.float32)
    c.lengths.fill_(tokens)
    ops.paged_kv_write(c, cuda(k.reshape(tokens, -1)), cuda(v.reshape(tokens, -1)), starts=rows_of([tokens]), slots=rows_of([])[:1])
    return P.quantised(k)[0].transpose(1, 0, 2), P.quantised(v)[0].transpose(1, 0, 2)


def attention_repeated(q, k, v, pos, scale):
    """P.attention over keys 0 .. pos that are k, v [tokens, head] over and over."""
    n = len(k)
    s = k @ q * scale
    p = np.exp(s - s.max()) * ((pos + 1) // n + (np.arange(n) < (pos + 1) % n))
    p /= p.sum()
    return p @ v, p @ np.abs(v), float((np.abs(k) @ np.abs(q)).max())


@pytest.mark.parametrize("kind,head,nh", [("f16", 64, 1), ("bf16", 64, 1), ("f32", 64, 1), ("f16", 128, 16), ("f16", 256, 2)])
def test_single_rows_over_millions_of_keys(kind, head, nh):
    """A hundred sequences of four million keys (the same pages over and over), so that a warp adds up hundreds of thousands of them:
    values that are all positive, whose sum is large against each."""
    from cut_b200 import ops
    from cut_b200.paged import PagedCache

    r = np.random.default_rng(head + nh)
    n, base, length = 100, 4096, 4 << 20
    c = PagedCache.allocate(base // 256, n, length, 1, head, page_tokens=256)
    ks, vs = repeated(c, base, 1, head, r)
    lengths = length - r.integers(0, 5000, n)
    c.lengths.copy_(cuda(lengths.astype(np.int32)))
    q = torch.from_numpy(0.1 * r.standard_normal((n, nh * head))).to(TYPES[kind]).cuda()
    got, x, scale = ops.paged_attention(c, q, nh).double().cpu().numpy(), q.double().cpu().numpy(), float(np.float32(head ** -0.5))
    c.check()
    for s in range(n):
        for h in range(nh):
            part = slice(h * head, (h + 1) * head)
            y, spread, products = attention_repeated(x[s, part], ks[0], vs[0], int(lengths[s]) - 1, scale)
            off = np.abs(got[s, part] - y) - P.tolerance(y, spread, products, scale, kind)
            assert off.max() <= 0, (s, h, off.max(), float(np.mean(got[s, part] / y - 1)))


@pytest.mark.parametrize("kind,head,nh,new,length,window", [("f16", 64, 1, 64, 1 << 20, 0), ("bf16", 64, 1, 64, 1 << 20, 0), ("f32", 64, 1, 64, 1 << 20, 0),
                                                            ("f16", 128, 4, 100, 300000, 0), ("f16", 192, 4, 40, 280000, 0), ("f16", 256, 3, 50, 270000, 0),
                                                            ("f16", 128, 2, 300, 400000, 262144), ("f16", 128, 1, 64, 8192 + 64, 0), ("f16", 40, 1, 200, 16500, 8300)])
def test_prompts_behind_hundreds_of_thousands_of_keys(kind, head, nh, new, length, window):
    """Prompts whose rows add up many thousands of positive values, and ones just past the keys that one sum goes on for."""
    from cut_b200 import ops
    from cut_b200.paged import PagedCache

    r = np.random.default_rng(head + new)
    base = 2048
    c = PagedCache.allocate(base // 64, 3, length + 100, 1, head, page_tokens=64)
    ks, vs = repeated(c, base, 1, head, r)
    lengths, rows = [length, 1000, length - 3000], [new, 100, new // 2 + 33]  # (and a short one between them)
    c.lengths.copy_(cuda(np.array(lengths, dtype=np.int32)))
    n = sum(rows)
    q = torch.from_numpy(0.1 * r.standard_normal((n, nh * head))).to(TYPES[kind]).cuda()
    out = ops.paged_attention(c, q, nh, starts=rows_of(rows), max_new=max(rows), window=window)
    again = ops.paged_attention(c, q, nh, starts=rows_of(rows), max_new=max(rows), window=window)
    c.check()
    assert torch.equal(out, again)
    got, x, scale, row = out.double().cpu().numpy(), q.double().cpu().numpy(), float(np.float32(head ** -0.5)), 0
    for s, m in enumerate(rows):
        for i in range(m):
            pos = lengths[s] - m + i
            if i % 9 and i + 1 < m:
                row += 1
                continue
            for h in range(nh):
                part = slice(h * head, (h + 1) * head)
                if window and pos >= window:  # the keys from pos + 1 - window on
                    at = (pos + 1 - window) % base
                    y, spread, products = attention_repeated(x[row, part], np.roll(ks[0], -at, 0), np.roll(vs[0], -at, 0), window - 1, scale)
                else:
                    y, spread, products = attention_repeated(x[row, part], ks[0], vs[0], pos, scale)
                off = np.abs(got[row, part] - y) - P.tolerance(y, spread, products, scale, kind)
                assert off.max() <= 0, (s, i, h, off.max(), float(np.mean(got[row, part] / y - 1)))
            row += 1


def test_scores_that_rise_over_many_keys():
    """The reference of the weights moves while sums are on their way to the totals, and stays where rows have seen their largest early."""
    from cut_b200 import ops
    from cut_b200.paged import PagedCache

    r = np.random.default_rng(13)
    n, head, rows = 40000, 64, 130
    c = PagedCache.allocate(n // 64, 1, n, 1, head, page_tokens=64)
    c.tables[0] = torch.arange(n // 64, dtype=torch.int32)
    c.lengths.fill_(n)
    direction = r.standard_normal(head)
    k = (np.linspace(-40, 40, n)[:, None] * direction / head + 0.02 * r.standard_normal((n, head))).astype(np.float32)
    v = r.standard_normal((n, head)).astype(np.float32)
    ops.paged_kv_write(c, cuda(k), cuda(v), starts=rows_of([n]))
    kq, vq = P.quantised(k)[0], P.quantised(v)[0]
    q = np.tile(direction, (rows, 2)) * r.choice([-1.0, 0.02, 1.0, 0.3], (rows, 1))
    for kind in ("f16", "bf16"):
        x = torch.from_numpy(q).to(TYPES[kind]).cuda()
        got = ops.paged_attention(c, x, 2, starts=rows_of([rows]), max_new=rows, scale=1.0).double().cpu().numpy()
        x = x.double().cpu().numpy()
        for i in range(0, rows, 7):
            y, spread, products = P.attention(x[i, :head], kq, vq, n - rows + i, 1.0, 0)
            assert (np.abs(got[i, :head] - y) <= P.tolerance(y, spread, products, 1.0, kind)).all(), (kind, i)
    c.check()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("head,kv,n,max_new", [(64, 2, 6, None), (33, 3, 6, None), (128, 32, 900, 16)])
def test_every_row_that_is_read_without_starts_is_written(kind, head, kv, n, max_new):
    """Few rows, and as many as whole units would be read by: the rows of sequences that cannot be read are zero, whatever was there."""
    import ctypes as C

    from cut_b200 import _lib as L
    from cut_b200 import ops

    r = np.random.default_rng(14)
    lengths = [20, 33, 0, 7]
    c = make_cache(lengths, kv, head, 16, r)
    ks, vs = fill_cache(c, lengths, kv, head, r)
    c.tables[3, 0], slots = 1 << 20, r.choice([0, 1, 2, 3, 77, -1], n).astype(np.int32)
    slots[:3] = 2, 0, 77
    k, v = (torch.full((n, kv * head), 7.0, dtype=TYPES[kind], device="cuda") for _ in range(2))
    sl = cuda(slots)
    d = ops.paged_desc(c, n, TYPES[kind], slots=sl, max_new=max_new)
    d.k_out, d.ldk_out, d.v_out, d.ldv_out = k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0)
    L.check(L.lib().cutb_paged_kv_read(C.byref(d), ops._stream_ptr()))
    with pytest.raises(L.CutbError) as e:
        c.check()
    assert e.value.status == L.ERR_INVALID
    for got, held in ((k, ks), (v, vs)):
        want = np.stack([held[s][:, -1].reshape(-1) if s in (0, 1) else np.zeros(kv * head) for s in slots])
        assert torch.equal(got.cpu(), torch.from_numpy(want).to(TYPES[kind]))
