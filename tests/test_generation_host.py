"""Sampled generation, as far as it needs no GPU: the settings' refusals, the queue, the command line."""
import pytest

from cut_b200.decoding import RequestQueue, Sampling, generate

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("bad", [dict(temperature=-0.1), dict(temperature=float("inf")), dict(temperature=float("nan")), dict(top_k=-1), dict(top_k=1 << 31),
                                 dict(top_p=-0.1), dict(top_p=1.1), dict(top_p=float("nan")), dict(min_p=-1.0), dict(min_p=1.5)])
def test_settings_that_are_refused(bad):
    with pytest.raises(ValueError):
        Sampling(**bad)


def test_queue_hands_the_last_logits_to_the_decoder():
    class Fake:
        def __init__(self):
            self.seen = []

        def open(self):
            return "s"

        def close(self, s):
            pass

        def forward(self, s, tokens, want):
            return torch.tensor([[float(tokens[w])] for w in want]) if want else None

        def decode_greedy(self, s, n):
            return [0] * n

        def decode_sampled(self, s, logits, n, sampling):
            self.seen.append((logits.tolist(), n, sampling))
            return [1] * n

    d, how = Fake(), Sampling(temperature=0.5, seed=3)
    q = RequestQueue(d, portion=2)
    a, b, c = q.submit([4, 5, 6], 2, how), q.submit([7], 3), q.submit([8], 0, how)
    q.run()
    assert (a.tokens, b.tokens, c.tokens) == ([1, 1], [0, 0, 0], []) and d.seen == [([[6.0]], 2, how)]
    assert generate(d, [9], 1, sampling=how) == [1] and generate(d, [9], 1) == [0]


@pytest.mark.parametrize("option", ["--temperature", "--top-k", "--top-p", "--min-p", "--seed"])
def test_the_runner_of_gguf_files_does_not_draw(option, capsys):
    from cut_b200.generate import main

    with pytest.raises(SystemExit):
        main(["--model", "m.gguf", "--tokens", "1", option, "1"])
    assert "likeliest" in capsys.readouterr().err


def test_a_page_of_the_decoder_is_a_page_of_the_cache():
    from cut_b200.paged import PagedCache

    with pytest.raises(ValueError):
        PagedCache.allocate(1, 1, 16, 1, 64, page_tokens=24, device="cpu")


def test_a_token_that_could_not_be_drawn_is_an_error():
    status = torch.zeros(1, dtype=torch.int32)
    assert Sampling.ids(torch.tensor([3, 0, 7], dtype=torch.int32), status) == [3, 0, 7] and Sampling.ids(torch.empty(0, dtype=torch.int32), status) == []
    with pytest.raises(RuntimeError, match="token 1 of 2"):
        Sampling.ids(torch.tensor([3, -1], dtype=torch.int32), status)
    status.fill_(1)
    with pytest.raises(RuntimeError, match="status 1"):
        Sampling.ids(torch.tensor([-1, -1], dtype=torch.int32), status)
    assert int(status) == 0


@pytest.mark.parametrize("temperature", [1e39, 3.5e38, 1 << 200])
def test_a_temperature_that_32_bits_do_not_hold_is_refused(temperature):
    with pytest.raises(ValueError, match="32 bits"):
        Sampling(temperature=temperature)
    assert Sampling(temperature=3.4e38).temperature == 3.4e38


def test_a_sequence_uses_up_its_seeds_numbers(monkeypatch):
    """What is drawn in pieces is drawn by the numbers that follow, not by the first ones again."""
    from cut_b200 import decoding

    seen = []
    monkeypatch.setattr(decoding.ops, "sample", lambda rows, u, *, tokens, **kw: (seen.append(float(u)), tokens.zero_()))
    logits, feed = torch.zeros(1, 4), lambda token: torch.zeros(1, 4)
    how = Sampling(seed=4)
    assert how.decode(logits, 12, feed).tolist() == [0] * 12
    at_once, at = list(seen), 0
    seen.clear()
    for n in (1, 1, 0, 5, 1, 4):
        how.decode(logits, n, feed, at)
        at += n
    assert seen == at_once and len(set(seen)) == 12
