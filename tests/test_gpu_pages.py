"""The bookkeeping of a paged cache on the GPU against the same done by hand, and a run of a server's calls together."""
import numpy as np
import pytest

import paged_util as P

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def pair(n_pages, n_slots, width, page=16, page_bytes=4112, seed=0):
    """A cache and its model, with pages of random bytes."""
    from cut_b200.paged import PagedCache

    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = torch.randint(0, 256, (n_pages, page_bytes), dtype=torch.uint8, device="cuda", generator=g)
    c = PagedCache(pages, i32(n_slots, width).fill_(-1), i32(n_slots), i32(n_pages), page_tokens=page, status=i32(1))
    m = P.Pool(n_pages, n_slots, width, page)
    m.bytes = pages.cpu().numpy().copy()
    return c, m


def same(c, m, bytes_too=True):
    assert np.array_equal(c.lengths.cpu().numpy(), m.lengths)
    assert np.array_equal(c.refs.cpu().numpy(), m.refs)
    got = c.tables.cpu().numpy()
    for s in range(len(m.lengths)):
        n = m.count(s)
        assert np.array_equal(got[s, :n], m.tables[s, :n]), s
        assert (got[s, n:] == -1).all(), s
    if bytes_too:
        held = m.refs > 0
        assert np.array_equal(c.pages.cpu().numpy()[held], m.bytes[held])


def status(c):
    st = int(c.status.item())
    c.status.zero_()
    return st


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("seed", range(4))
def test_random_bookkeeping(page, seed):
    r = np.random.default_rng(seed)
    c, m = pair(200, 24, 12, page, seed=seed)
    for step in range(30):
        what = r.choice(["reserve", "reserve", "fork", "free", "compact"])
        if what == "reserve":
            slots = r.permutation(24)[: r.integers(1, 24)]
            counts = r.choice([0, 1, 2, page, 3 * page + 1], len(slots))
            keep = m.lengths[slots] + counts <= 12 * page
            c.reserve(slots[keep], counts[keep]), m.reserve(slots[keep], counts[keep])
        elif what == "fork":
            empty, full = np.flatnonzero(m.lengths == 0), np.flatnonzero(m.lengths)
            if len(empty) and len(full):
                dst = r.permutation(empty)[: r.integers(1, len(empty) + 1)]
                src = r.choice(full, len(dst))
                c.fork(src, dst), m.fork(src, dst)
        elif what == "free":
            slots = r.permutation(24)[: r.integers(1, 8)]
            c.free(slots), m.free(slots)
        else:
            c.compact(), m.compact()
        st = status(c)
        assert ("pages" in m.wrong) == (st == 7) and "invalid" not in m.wrong and st in (0, 7), (step, what, st, m.wrong)
        m.wrong.clear()
        same(c, m)


def test_holders_of_one_page_copy_it_but_the_last():
    c, m = pair(40, 8, 4)
    for f in (c, m):
        f.reserve([0], [20])
        f.fork([0, 0, 0, 0], [1, 2, 3, 4])
        f.reserve([3, 0, 4], [1, 1, 1])
        f.free([1])
        f.reserve([2], [1])  # the only holder left of the first copy
    assert status(c) == 0
    same(c, m)
    assert len({int(p) for p in c.tables[[0, 2, 3, 4], 1].tolist()}) == 4 and int(c.refs.sum()) == 4 + 4


def test_with_too_few_pages_the_first_come_are_served():
    c, m = pair(6, 6, 5)
    for f in (c, m):
        f.reserve([2, 0, 1, 3], [33, 16, 40, 0])  # 3, 1, 3 pages of six
    assert status(c) == 7 and "pages" in m.wrong
    same(c, m)
    assert c.lengths.tolist() == [16, 0, 33, 0, 0, 0]
    for f in (c, m):  # a copy that finds no page leaves the shared page as it is, for those behind it too
        f.reserve([1, 4], [32, 0])
        f.fork([2], [5])
        f.reserve([5, 2], [1, 1])
    assert status(c) == 7
    same(c, m)
    assert c.lengths.tolist()[2] == 33 and c.lengths.tolist()[5] == 33


def test_entries_that_cannot_be_served():
    from cut_b200 import _lib as L

    c, m = pair(20, 4, 3)
    for f in (c, m):
        f.reserve([0, 9, 0, 1, -1], [5, 1, 1, 100, 1])  # a slot that does not exist, one named twice, one longer than its table
    assert status(c) == L.ERR_INVALID and c.lengths.tolist() == [5, 0, 0, 0]
    same(c, m)
    for f in (c, m):
        f.fork([0, 0, 0, 0, 7], [1, 1, 0, 8, 2])
    assert status(c) == L.ERR_INVALID and c.lengths.tolist() == [5, 5, 0, 0]
    same(c, m)
    for f in (c, m):
        f.free([3, 1, 1])
    assert status(c) == 0
    same(c, m)
    c.free([40])
    assert status(c) == L.ERR_INVALID
    same(c, m)
    c.tables[0, 0] = 99  # a page that does not exist
    c.reserve([0], [1])
    assert status(c) == L.ERR_INVALID and c.lengths.tolist() == [5, 0, 0, 0]
    c.copy([0, 25], [1, 2])
    assert status(c) == L.ERR_INVALID and torch.equal(c.pages[0], c.pages[1])


@pytest.mark.parametrize("page_bytes", [16, 4096, 16384, 16400, 100000])
def test_copies(page_bytes):
    c, m = pair(50, 1, 1, page_bytes=page_bytes)
    r = np.random.default_rng(page_bytes)
    order = r.permutation(50)
    c.copy(order[:20], order[20:40])
    m.bytes[order[20:40]] = m.bytes[order[:20]]
    assert np.array_equal(c.pages.cpu().numpy(), m.bytes) and status(c) == 0
    c.copy([], [])


def test_many_pages_and_slots():
    c, m = pair(30000, 1000, 40, page_bytes=16)
    r = np.random.default_rng(3)
    slots, counts = r.permutation(1000), r.integers(0, 500, 1000)
    for f in (c, m):
        f.reserve(slots, counts)
        f.free(slots[::2])
        f.compact()
        f.reserve(slots[:100], np.full(100, 37))
    assert status(c) == 0
    same(c, m)


def test_recorded_bookkeeping():
    """fork, reserve and free recorded once and replayed: slots and counts are read on the device."""
    c, m = pair(64, 8, 8)
    c.reserve([0, 1], [20, 40]), m.reserve([0, 1], [20, 40])
    src, dst, every, one = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0, 1], [2, 3], [2, 3], [1, 17]))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.fork(src, dst)
        c.reserve(every, one)
        c.compact()
    for a, b in (([0, 1], [2, 3]), ([2, 0], [5, 4])):
        src.copy_(torch.tensor(a, dtype=torch.int32)), dst.copy_(torch.tensor(b, dtype=torch.int32)), every.copy_(dst)
        g.replay()
        m.fork(a, b), m.reserve(b, [1, 17]), m.compact()
        same(c, m)
    assert status(c) == 0


def test_a_server_of_three_sequences():
    """Prompts, a fork, single tokens, an end, a compaction, more tokens: attention and sampled tokens of every step against a model
    that keeps each sequence's values by itself."""
    from cut_b200 import ops
    from cut_b200.paged import PagedCache

    r = np.random.default_rng(1)
    kv, nh, head, page, vocab = 2, 4, 64, 16, 300
    c = PagedCache.allocate(24, 4, 96, kv, head, n_layers=2, page_tokens=page)
    cos, sin = P.tables_of(head, head, 96)
    cos_d, sin_d = (torch.from_numpy(t).cuda() for t in (cos, sin))
    held = {s: [[np.zeros((kv, 0, head))] * 2 for _ in range(2)] for s in range(4)}  # slot -> layer -> [keys, values]
    head_w = torch.from_numpy(r.standard_normal((nh * head, vocab)).astype(np.float32)).cuda()

    def step(slots, new):
        """`new[i]` further tokens of slots[i] through both layers; the next token of each."""
        c.reserve(slots, new)
        starts = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32).cuda() if max(new) > 1 else None
        sl = torch.tensor(slots, dtype=torch.int32).cuda()
        n = sum(new)
        for layer in range(2):
            x = r.standard_normal((n, (nh + 2 * kv) * head)).astype(np.float32)
            qkv = torch.from_numpy(x).cuda()
            q, k, v = qkv[:, : nh * head], qkv[:, nh * head: (nh + kv) * head], qkv[:, (nh + kv) * head:]
            q = ops.paged_kv_write(c, k, v, q=q, starts=starts, slots=sl, cos_t=cos_d, sin_t=sin_d, rot_dims=head, layer=layer)
            out = ops.paged_attention(c, q, nh, starts=starts, slots=sl, max_new=max(new), layer=layer)
            got, row = out.double().cpu().numpy(), 0
            for s, m in zip(slots, new):
                for i in range(m):
                    pos = held[s][layer][0].shape[1]
                    turned = P.turned(x[row, : (nh + kv) * head].reshape(-1, head), pos, cos, sin, head, 0)
                    for which, y in ((0, turned[nh:]), (1, x[row, (nh + kv) * head:].reshape(kv, head))):
                        held[s][layer][which] = np.concatenate([held[s][layer][which], P.quantised(y)[0][:, None]], axis=1)
                    for h in range(nh):
                        y, spread, products = P.attention(turned[h].astype(np.float64), held[s][layer][0][h // 2], held[s][layer][1][h // 2], pos, head ** -0.5, 0)
                        assert (np.abs(got[row, h * head: (h + 1) * head] - y) <= P.tolerance(y, spread, products, head ** -0.5, "f32")).all()
                    row += 1
        logits = out[torch.tensor(np.cumsum(new) - 1).cuda()] @ head_w
        u, t = r.random(len(slots)).astype(np.float32), np.full(len(slots), 0.8, np.float32)
        tokens = ops.sample(logits, torch.from_numpy(u).cuda(), temperature=torch.from_numpy(t).cuda())
        assert tokens.tolist() == [P.sampled(row, np.float64(np.float32(0.8)), 0, 1.0, 0.0, a)[0] for row, a in zip(logits.double().cpu().numpy(), u.astype(np.float64))]

    step([0, 2], [37, 18])
    c.fork([0], [1])
    held[1] = [[a for a in layer] for layer in held[0]]
    step([0, 1, 2], [1, 1, 1])
    step([1, 0], [1, 1])
    c.free([2])
    held[2] = [[np.zeros((kv, 0, head))] * 2 for _ in range(2)]
    c.compact()
    assert int((c.refs > 0).sum()) == int((c.refs[: int((c.refs > 0).sum())] > 0).sum())
    step([0, 1], [1, 20])
    step([2, 1, 0], [5, 1, 3])
    c.check()


def test_tables_that_name_a_page_more_often_than_it_is_held():
    """Freed at once, by many slots: the count ends at none, whatever order they come in, and the call reports it."""
    from cut_b200 import _lib as L

    for held in (0, 1, 3):
        c, _ = pair(8, 400, 4)
        c.tables[:, :2] = torch.tensor([5, 2], dtype=torch.int32)
        c.lengths.fill_(20)
        c.refs[5], c.refs[2] = held, 400
        c.free(list(range(400)))
        assert status(c) == L.ERR_INVALID
        assert c.refs.tolist() == [0] * 8 and not c.lengths.any() and bool((c.tables == -1).all())
