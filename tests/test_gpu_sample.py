"""Sampling on the GPU against the same in 64 bits: every choice equal, the logarithms to fp32's last digits."""
import numpy as np
import pytest

import paged_util as P

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def run(x, u, t=None, k=None, p=None, least=None):
    """x: torch logits on the GPU; the settings as lists or None -> (tokens, logprobs, status)"""
    from cut_b200 import ops

    dev = lambda v, kind: None if v is None else torch.tensor(np.asarray(v), dtype=kind).cuda()  # noqa: E731
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    tokens, logs = ops.sample(x, dev(u, torch.float32), temperature=dev(t, torch.float32), top_k=dev(k, torch.int32), top_p=dev(p, torch.float32),
                              min_p=dev(least, torch.float32), want_logprobs=True, status=st)
    return tokens.cpu().numpy(), logs.cpu().numpy(), int(st.item())


def check(x, u, t=None, k=None, p=None, least=None):
    n = len(u)
    got, logs, st = run(x, u, t, k, p, least)
    assert st == 0
    rows = x.double().cpu().numpy()
    f = lambda v, d: np.full(n, d) if v is None else np.asarray(v, dtype=np.float32).astype(np.float64)  # noqa: E731
    for r in range(n):
        tok, lp = P.sampled(rows[r], f(t, 1)[r], 0 if k is None else k[r], f(p, 1)[r], f(least, 0)[r], float(np.float32(u[r])))
        assert got[r] == (-1 if tok is None else tok), r
        # the shares are within 2^-40, the logarithm is rounded once
        assert (lp == logs[r]) or abs(logs[r] - lp) <= 2.0 ** -24 * abs(lp) + 2.0 ** -36, (r, logs[r], lp)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 32000, 50257, 128256])
def test_settings(kind, vocab):
    r = np.random.default_rng(vocab)
    n = 24
    x = torch.from_numpy(2.5 * r.standard_normal((n, vocab))).to(TYPES[kind]).cuda()
    x[::2, : max(1, vocab // 7)] += 5
    u = r.random(n).astype(np.float32)
    t, k = r.choice([0, 0.01, 0.7, 1, 1.3, 5], n), r.choice([0, 1, 5, 50, vocab - 1, vocab, vocab + 9], n).astype(int)
    p, least = r.choice([1.0, 0.0, 0.5, 0.9, 0.999, 2.0, -1.0], n), r.choice([0, 0, 1e-4, 0.05, 0.3, 1.0, 7.0], n)
    check(x, u)
    check(x, u, t=t)
    check(x, u, k=k)
    check(x, u, p=p)
    check(x, u, least=least)
    check(x, u, t, k, p, least)


def test_ties_and_ends_of_the_range():
    """Equal logits are taken in their order; u of zero and just below one; zeros of both signs are equal."""
    x = torch.zeros(12, 1000, device="cuda")
    x[1::2, ::3] = -0.0
    u = np.array([0, 1 - 2 ** -24, 0.5, 0.25, 0.125, 0.999, 0.3, 0.7, 0, 0.9999, 1e-30, 0.0625], dtype=np.float32)
    check(x, u)
    check(x, u, k=[1, 2, 3, 10, 33, 999, 1000, 500, 1, 7, 64, 5])
    check(x, u, p=[0.1, 0.5, 1e-9, 0.0105, 0.25, 0.75, 0.999, 0.0, 0.3, 0.2, 0.9, 0.0625])
    check(x, u, k=[100] * 12, p=[0.25] * 12)
    check(x, u, t=[0.0] * 12)
    x[:, 400:] = 3.0
    check(x, u, k=[600, 601, 599, 10, 700, 650, 1, 0, 900, 620, 3, 605], p=[1, 0.99, 0.5] * 4)


@pytest.mark.parametrize("kind", list(TYPES))
def test_masked_and_not_finite(kind):
    r = np.random.default_rng(1)
    inf, nan, low = float("inf"), float("nan"), torch.finfo(TYPES[kind]).min
    x = torch.from_numpy(r.standard_normal((8, 500))).to(TYPES[kind]).cuda()
    x[0, 3:] = -inf
    x[1, ::2] = nan
    x[2, [7, 70, 400]] = inf
    x[3] = -inf
    x[4] = nan
    x[5, :490] = low
    x[6] = low
    x[7, 5], x[7, 6] = inf, nan
    u = r.random(8)
    check(x, u)
    check(x, u, t=[0.5] * 8, k=[20] * 8, p=[0.9] * 8, least=[0.01] * 8)
    check(x, u, t=[0.0] * 8)
    check(x, u, k=[500, 499, 2, 1, 1, 495, 3, 2])


def test_settings_that_mean_nothing():
    from cut_b200 import _lib as L

    x = torch.randn(9, 50, device="cuda")
    nan, inf = float("nan"), float("inf")
    u, t, p, least = [0.5] * 9, [1.0] * 9, [0.9] * 9, [0.1] * 9
    u[0], u[1], u[2], t[3], t[4], t[5], p[6], least[7] = 1.0, -0.1, nan, -1.0, nan, inf, nan, nan
    got, logs, st = run(x, u, t, None, p, least)
    assert st == L.ERR_INVALID and (got[:8] == -1).all() and (logs[:8] == -np.inf).all() and 0 <= got[8] < 50


def test_many_choices_of_one_row():
    """The tokens that u from 0 to 1 gives, one after another, have the weights' shares."""
    r = np.random.default_rng(4)
    row = torch.from_numpy((3 * r.standard_normal(5000)).astype(np.float32)).cuda()
    n = 2000
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    x = row.expand(n, -1).contiguous()
    check(x, u)
    check(x, u, k=[100] * n, p=[0.8] * n)


def test_strides_offsets_streams_and_recordings():
    from cut_b200 import ops

    r = np.random.default_rng(5)
    wide = torch.from_numpy(r.standard_normal((5, 4099)).astype(np.float32)).cuda()
    for off in (0, 1, 2, 3):
        check(wide[:, off: off + 4001], r.random(5))
    half = wide.bfloat16()
    for off in (1, 2, 7):
        check(half[:, off: off + 4003], r.random(5), k=[50] * 5)
    u = torch.rand(5, device="cuda")
    tokens, s = torch.zeros(5, dtype=torch.int32, device="cuda"), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.sample(wide, u, tokens=tokens)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            ops.sample(wide, u, tokens=tokens)
    for _ in range(3):
        u.copy_(torch.rand(5))
        g.replay()
        torch.cuda.synchronize()
        assert tokens.tolist() == [P.sampled(row, 1.0, 0, 1.0, 0.0, a)[0] for row, a in zip(wide.double().cpu().numpy(), u.double().cpu().numpy())]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [300, 600, 5000, 40000, 128256])
def test_counts_of_every_size(kind, vocab):
    """Cut-offs by count on either side of what one block finishes alone, with and without the others, equal logits among them."""
    r = np.random.default_rng(vocab + 1)
    k = np.array([1, 2, 3, 17, 200, 255, 256, 257, 300, 511, 512, 513, 600, 1024, 2048, 5])
    n = len(k)
    x = 2.5 * r.standard_normal((n, vocab))
    x[1::3] = np.round(x[1::3])  # many equal ones
    x = torch.from_numpy(x).to(TYPES[kind]).cuda()
    u = r.random(n).astype(np.float32)
    check(x, u, k=k)
    check(x, u, t=r.choice([0.01, 0.5, 1, 2, 30], n), k=k, p=r.choice([0.3, 0.9, 0.999, 1.0], n), least=r.choice([0, 0.01, 0.2], n))


@pytest.mark.parametrize("kind", list(TYPES))
def test_largest_logits_side_by_side(kind):
    """The largest logits in a few threads' parts of the row, and a row whose logits but a few have no weight."""
    r = np.random.default_rng(5)
    vocab = 60000
    x = r.standard_normal((8, vocab))
    at = np.arange(vocab)
    x[:4, at // 8 % 512 < 8] += 20
    x[4, 20000:23000] += 20
    x[5:, 10:] -= 1000
    x = torch.from_numpy(x).to(TYPES[kind]).cuda()
    u = r.random(8).astype(np.float32)
    for k in ([50] * 8, [3, 9, 10, 11, 250, 10, 11, 12], [300, 500, 700, 900, 1100, 256, 257, 600]):
        check(x, u, k=k)
        check(x, u, k=k, p=[0.9] * 8, least=[0, 0.01] * 4)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("vocab", [40, 5000, 128256])
def test_least_weights_above_the_largest_with_ties(kind, vocab):
    """min_p above 1 leaves the first of the largest logits, at 1 all of them, whatever the other cut-offs do."""
    r = np.random.default_rng(vocab)
    x = r.standard_normal((12, vocab))
    for row in range(12):
        x[row, r.permutation(vocab)[: (2, 7, 30)[row % 3]]] = 6.0
    x[11] = 0.0
    x[10, [3, 17]] = np.inf
    x = torch.from_numpy(x).to(TYPES[kind]).cuda()
    u, least = np.linspace(0.05, 0.999, 12).astype(np.float32), [7.0, 1.0, 1.0000001] * 4
    check(x, u, least=least)
    check(x, u, least=least, k=[20] * 12)
    check(x, u, least=least, p=[0.6, 0.9, 1.0, 0.0] * 3)
    check(x, u, least=least, k=[300, 5, 0, 1000, 1, 20] * 2, p=[0.6, 0.9, 1.0, 0.01] * 3, t=[1, 0.5, 3, 0] * 3)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_logits_further_apart_than_the_type_holds(kind):
    """The distance of two finite logits may be past the largest number; at a high temperature both have weight."""
    r = np.random.default_rng(9)
    big = 3e38
    x = r.choice([big, -big, 0.0, 1e38, -2e38], (8, 3000))
    x[1] = -big
    x[1, 70], x[2, :] = big, np.linspace(-big, big, 3000)
    x[3, ::5] = -np.inf
    x = torch.from_numpy(x).to(TYPES[kind]).cuda()
    u, t = np.array([0.999, 0.999, 0.3, 0.9, 0.95, 0.5, 0.99, 0.999], dtype=np.float32), [big, big, 1e38, big, 2e38, 1e38, big, 3e38]
    for kw in (dict(), dict(p=[0.99, 0.999, 0.9, 0.97, 0.95, 0.999, 0.99, 0.97]), dict(k=[2000, 60, 700, 2900, 2500, 1300, 2999, 600]),
               dict(k=[2000, 300, 1500, 2900, 0, 511, 2999, 0], p=[0.99] * 8, least=[0, 0.1, 0.01, 0, 0, 0.001, 0, 0.1])):
        check(x, u, t=t, **kw)


def test_two_threads_draw_from_rows_of_different_sizes():
    """Calls at once from two threads, one with little shared memory to a block and one with much."""
    import ctypes as C
    import threading

    from cut_b200 import _lib as L

    r = np.random.default_rng(10)
    ready, wrong, call = threading.Barrier(2), [], L.lib().cutb_sample

    def work(vocab):
        try:
            x = torch.from_numpy(r.standard_normal((2, vocab)).astype(np.float32)).cuda()
            u, tokens, stream = torch.full((2,), 0.5, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), torch.cuda.Stream()
            d = L.SampleDesc(logits=x.data_ptr(), ld=vocab, rows=2, vocab=vocab, dtype=L.F32, u=u.data_ptr(), tokens=tokens.data_ptr())
            torch.cuda.synchronize()
            ready.wait(60)
            codes = [call(C.byref(d), stream.cuda_stream) for _ in range(20000)]
            stream.synchronize()
            assert set(codes) == {L.OK}
            assert tokens.tolist() == [P.sampled(row, 1.0, 0, 1.0, 0.0, 0.5)[0] for row in x.double().cpu().numpy()]
        except BaseException as e:  # noqa: BLE001 (handed to the test's thread)
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=(vocab,)) for vocab in (100, 8000)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong


def check_wide(x, u, t=None, k=None, p=None, least=None):
    """As check(), the logarithms as near as many small weights allow: a weight is a whole number of units of 2^-42 of the largest, off by half
    a unit (and what the exponential is off by, 2^-42 of the weight), so that the sum of n of them, which is at least 1, is off by n 2^-43
    + 2^-42 of itself and the logarithm by as much."""
    got, logs, st = run(x, u, t, k, p, least)
    assert st == 0
    rows, n = x.double().cpu().numpy(), len(u)
    f = lambda v, d: np.full(n, d) if v is None else np.asarray(v, dtype=np.float32).astype(np.float64)  # noqa: E731
    for r in range(n):
        tok, lp = P.sampled(rows[r], f(t, 1)[r], 0 if k is None else k[r], f(p, 1)[r], f(least, 0)[r], float(np.float32(u[r])))
        assert got[r] == tok, r
        assert abs(logs[r] - lp) <= 2.0 ** -24 * abs(lp) + x.shape[1] * 2.0 ** -43 + 2.0 ** -36, (r, logs[r], lp)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("off", [0, 1])
def test_rows_that_are_read_again_without_cut_offs(kind, off):
    """So many rows that two blocks have one, and so wide that a block reads its part again instead of keeping it."""
    r = np.random.default_rng(off)
    n, vocab = 150, 128256
    g = torch.Generator(device="cuda").manual_seed(off)
    x = (2.5 * torch.randn(n, vocab + 3, device="cuda", generator=g)).to(TYPES[kind])[:, off: off + vocab - off]
    u = r.random(n).astype(np.float32)
    check_wide(x, u, t=r.choice([0.0, 0.5, 1.0, 2.0], n))
    check_wide(x, u, t=r.choice([0.5, 1.0], n), least=r.choice([0.0, 0.01, 0.5, 1.0, 3.0], n))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [524288, 524287, 300001])
def test_the_widest_rows(kind, vocab):
    r = np.random.default_rng(vocab)
    x = torch.from_numpy(r.choice([0.05, 2.5], (5, 1)) * r.standard_normal((5, vocab))).to(TYPES[kind]).cuda()
    u = r.random(5).astype(np.float32)
    check_wide(x, u)
    check_wide(x, u, p=[0.9, 0.3, 0.999, 0.5, 0.95])
    check_wide(x, u, k=[0, 3, 1000, 40, 260000], p=[0.9, 1.0, 0.99, 0.5, 0.95], least=[0, 0.01, 0, 0, 0.2])


def test_the_widest_rows_whose_weights_fill_their_digits():
    """All logits but one equal, with a weight whose lower two digits of 16 bits are as large as a search finds them: a block's 65536 of
    them add up to just below 2^32 in either place."""
    vocab = 524288
    v = (1 + np.arange(1 << 22, dtype=np.float64) * 2.0 ** -23).astype(np.float32)
    w = np.rint(np.exp(-v.astype(np.longdouble)) * np.longdouble(2.0) ** 42).astype(np.int64)
    best = v[np.argmax(np.minimum(w & 0xffff, w >> 16 & 0xffff))]
    weight = int(w[np.argmax(np.minimum(w & 0xffff, w >> 16 & 0xffff))])
    assert min(weight & 0xffff, weight >> 16 & 0xffff) > 0xff00
    x = torch.full((4, vocab), 0.0, device="cuda")
    x[:] = -float(best)
    for row, at in enumerate((0, 70001, 262144, vocab - 1)):
        x[row, at] = 0.0
    check_wide(x, [0.3333, 0.7777, 0.12345, 0.987], p=[0.5000123, 0.9000123, 0.2500123, 0.9990123])
    check_wide(x, [0.3333, 0.7777, 0.12345, 0.987])
