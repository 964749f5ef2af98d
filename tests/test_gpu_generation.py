"""Generation over a 4-bit cache and with drawn tokens: a Llama-style decoder against a composition in 64 bits that attends to what the
cache holds, drawn tokens against the same draw in 64 bits from the logits of a decoder that is fed them one by one."""
import json
import os
import subprocess
import sys

import numpy as np
import pytest

import paged_util as P
from oracle import oracle as O

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def model(page, max_seq, fmt=0, layers=2, heads=4, kv=2, head=64, seed=3):
    from cut_b200.llama_decode import LlamaConfig, synthetic_weights

    cfg = LlamaConfig(n_layers=layers, hidden=256, n_heads=heads, n_kv_heads=kv, head_dim=head, ffn=512, vocab=512, max_seq=max_seq, fmt=fmt,
                      kv_page_tokens=page)
    w = synthetic_weights(cfg, seed=seed, scale_shift=4)
    w["embedding"] = (w["embedding"] * 50).astype(np.float32)
    return cfg, w


class Composed:
    """The model in 64 bits, keys and values as the decoder's cache holds them; those of the new rows have to be what the model's own
    stand for, but for a step of their group where a rounding went the other way."""

    def __init__(self, cfg, w, dec):
        from cut_b200.llama_decode import rope_tables

        deq = lambda raw, n, k: O.dequant_rows(cfg.fmt, raw, n, k).astype(np.float64)  # noqa: E731
        self.cfg, self.w, self.dec, self.tables = cfg, w, dec, rope_tables(cfg)
        shapes = dict(wqkv=(cfg.q_dim + 2 * cfg.kv_dim, cfg.hidden), wo=(cfg.hidden, cfg.q_dim), wgate=(cfg.ffn, cfg.hidden), wup=(cfg.ffn, cfg.hidden),
                      wdown=(cfg.hidden, cfg.ffn))
        self.layers = [{**{k: deq(l[k], *s) for k, s in shapes.items()}, **{k: l[k] for k in ("attn_norm", "ffn_norm")}} for l in w["layers"]]
        self.lm = deq(w["lm_head"], cfg.vocab, cfg.hidden)

    def held(self, n, l):
        """What the cache holds of the first n tokens: float64 [n, kv, head] twice.  (The decoder's position is n.)"""
        from cut_b200 import ops

        starts = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        self.dec.paged.lengths.fill_(n)
        rows = ops.paged_kv_read(self.dec.paged, n, starts=starts, dtype=torch.float32, layer=l)
        return [r.double().cpu().numpy().reshape(n, self.cfg.n_kv_heads, self.cfg.head_dim) for r in rows]

    def run(self, tokens, first, slack):
        """Logits of the rows of tokens that stand at first, first + 1, ...; the cache holds them all already."""
        cfg, (cos, sin) = self.cfg, self.tables
        n, hd, rep = len(tokens), cfg.head_dim, cfg.n_heads // cfg.n_kv_heads
        x = self.w["embedding"][np.asarray(tokens)].astype(np.float64)
        norm = lambda v, wt: v / np.sqrt((v * v).mean(-1, keepdims=True) + cfg.eps) * wt  # noqa: E731
        for l, lw in enumerate(self.layers):
            qkv = (norm(x, lw["attn_norm"]) @ lw["wqkv"].T).astype(np.float32).reshape(n, -1, hd)
            turned = np.stack([P.turned(qkv[i, : cfg.n_heads + cfg.n_kv_heads], first + i, cos, sin, hd, 0) for i in range(n)]).astype(np.float64)
            k, v = self.held(first + n, l)
            for got, own in ((k, turned[:, cfg.n_heads:]), (v, qkv[:, cfg.n_heads + cfg.n_kv_heads:])):
                step = np.repeat(np.ptp(own.reshape(n, cfg.n_kv_heads, -1, 32), axis=-1) / 15, 32, axis=-1)
                assert (np.abs(got[first:] - own) <= (0.51 + slack) * step + (2.0 ** -10 + slack) * np.abs(own).max()).all()
            a = np.empty((n, cfg.n_heads, hd))
            for i in range(n):
                for h in range(cfg.n_heads):
                    a[i, h] = P.attention(turned[i, h], k[:, h // rep], v[:, h // rep], first + i, hd ** -0.5, 0)[0]
            x = x + a.reshape(n, -1) @ lw["wo"].T
            h = norm(x, lw["ffn_norm"])
            g = h @ lw["wgate"].T
            x = x + ((g / (1.0 + np.exp(-g))) * (h @ lw["wup"].T)) @ lw["wdown"].T
        return norm(x, self.w["final_norm"]) @ self.lm.T


@pytest.mark.parametrize("page,fmt,heads,kv,head", [(16, 0, 4, 2, 64), (64, 2, 8, 2, 32), (32, 1, 4, 4, 128)])
def test_decode_steps_over_a_paged_cache(page, fmt, heads, kv, head):
    from cut_b200.llama_decode import LlamaDecoder

    cfg, w = model(page, 50, fmt, heads=heads, kv=kv, head=head)
    dec = LlamaDecoder(cfg, w)
    ref = Composed(cfg, w, dec)
    assert not hasattr(dec, "k_cache")
    tokens = [int(t) for t in np.random.default_rng(page).integers(0, cfg.vocab, 20)]
    for pos, tok in enumerate(tokens):
        got = dec.step(tok, pos).double().cpu().numpy()
        want = ref.run([tok], pos, 0.01)[0]
        rel = np.linalg.norm(got - want) / np.linalg.norm(want)
        assert np.isfinite(got).all() and rel <= 1e-3, (pos, rel)  # as with rows of fp16
    dec.check_status()
    eager, tok = [], 7
    for i in range(6):
        tok = int(torch.argmax(dec.step(tok, 20 + i)).item())
        eager.append(tok)
    dec.set_position(7, 20)
    dec.capture()
    got = []
    for _ in range(6):
        dec.replay(1)
        got.append(int(dec.token.item()))
    assert got == eager and int(dec.params[0].item()) == 26
    dec.check_status()


@pytest.mark.parametrize("T,portion", [(7, 7), (40, 40), (150, 64)])
def test_prompts_over_a_paged_cache(T, portion):
    from cut_b200.llama_decode import LlamaDecoder

    cfg, w = model(16, T + 9)
    dec = LlamaDecoder(cfg, w)
    ref = Composed(cfg, w, dec)
    tokens = [int(t) for t in np.random.default_rng(T).integers(0, cfg.vocab, T)]
    for at in range(0, T, portion):
        part = tokens[at: at + portion]
        got = dec.prefill(part, at).double().cpu().numpy()
        want = ref.run(part, at, 0.03)[-1]
        assert np.linalg.norm(got - want) / np.linalg.norm(want) <= 3e-3  # as with rows of fp16
        dec.params.copy_(torch.tensor([at + len(part), at + len(part) + 1], dtype=torch.int32))
    nxt = int(dec.token.item())
    got = dec.step(nxt, T).double().cpu().numpy()
    want = ref.run([nxt], T, 0.03)[0]
    assert np.linalg.norm(got - want) / np.linalg.norm(want) <= 3e-3
    dec.check_status()


def test_position_past_a_paged_cache_is_reported():
    from cut_b200 import _lib as L
    from cut_b200.llama_decode import LlamaDecoder

    cfg, w = model(16, 20, layers=1)  # two pages, of which twenty tokens count
    dec = LlamaDecoder(cfg, w)
    dec.step(1, 19)
    dec.check_status()
    dec.step(1, 20)
    with pytest.raises(L.CutbError):
        dec.check_status()


def draws(n, seed):
    return torch.rand(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).double().cpu().numpy()


def follow(step, logits, picks, how):
    """Every pick against the draw in 64 bits from the logits before it."""
    f = lambda v: float(np.float32(v))  # noqa: E731
    for i, u in enumerate(draws(len(picks), how.seed)):
        want, _ = P.sampled(logits.double().cpu().numpy().reshape(-1), f(how.temperature), how.top_k, f(how.top_p), f(how.min_p), u)
        assert picks[i] == want, i
        if i + 1 < len(picks):
            logits = step(picks[i])


@pytest.mark.parametrize("page", [0, 16])
def test_drawn_tokens_of_the_llama_decoder(page):
    from cut_b200.decoding import Sampling, generate
    from cut_b200.llama_decode import LlamaDecoder

    cfg, w = model(page, 64)
    dec, other = LlamaDecoder(cfg, w), LlamaDecoder(cfg, w)
    prompt, all_picks = [3, 500, 17, 17, 9], []
    for how in (Sampling(), Sampling(temperature=3.0, top_k=40, top_p=0.9, min_p=0.01, seed=5), Sampling(temperature=2.0, seed=6)):
        picks = generate(dec, prompt, 12, sampling=how)
        seq = other.open()
        follow(lambda t: other.forward(seq, [t], [0]), other.forward(seq, prompt, [4]), picks, how)
        other.close(seq)
        assert picks == generate(dec, prompt, 12, sampling=how)
        all_picks.append(tuple(picks))
    assert len(set(all_picks)) == 3
    assert generate(dec, prompt, 12, sampling=Sampling(temperature=0.0)) == generate(dec, prompt, 12)
    seq = dec.open()
    logits = dec.forward(seq, prompt, [4])
    assert dec.decode_sampled(seq, logits, 0, Sampling()) == [] and seq.pos == 5
    first = dec.decode_sampled(seq, logits, 3, Sampling(seed=1))
    assert seq.pos == 7 and dec.decode_greedy(seq, 1) == first[-1:]  # the last one drawn has not been fed yet
    with pytest.raises(ValueError):
        dec.decode_sampled(seq, logits, 64, Sampling())
    dec.close(seq)


def test_drawn_tokens_of_a_model_folder(tmp_path):
    import test_gpu_layer_list as T
    from cut_b200.decoding import Sampling, generate
    from cut_b200.models import load_model

    cfg = T.CONFIGS["wide"]
    folder = T.save_model(tmp_path / "model", cfg, T.random_weights(cfg, 5))
    dec, other = load_model(folder, "float32", max_seq=64), load_model(folder, "float32", max_seq=64)
    prompt, how = [5, 6, 7], Sampling(temperature=1.5, top_k=30, top_p=0.95, seed=11)
    picks = generate(dec, prompt, 10, sampling=how)
    seq = other.open()
    other.forward(seq, prompt[:2], [])
    follow(lambda t: other.forward(seq, [t], [0]), other.forward(seq, prompt[2:], [0]), picks, how)
    other.close(seq)
    assert generate(dec, prompt, 10, sampling=Sampling(temperature=0.0)) == generate(dec, prompt, 10)
    seq = dec.open()
    dec.forward(seq, prompt, [])
    with pytest.raises(RuntimeError, match="logits of the last token"):
        dec.decode_sampled(seq, torch.zeros(1, cfg["vocab"], device="cuda"), 2, how)
    dec.close(seq)
    run = [sys.executable, "-m", "cut_b200.generate", "--model", folder, "--tokens", "5,6,7", "--n", "10", "--dtype", "float32"]
    r = subprocess.run([*run, "--temperature", "1.5", "--top-k", "30", "--top-p", "0.95", "--min-p", "0", "--seed", "11"], capture_output=True, text=True,
                       timeout=600, cwd=ROOT)
    assert r.returncode == 0, r.stderr[-2000:]
    assert json.loads(r.stdout)["tokens"] == generate(dec, prompt, 10, sampling=how)


@pytest.mark.parametrize("n", [1, 3])
def test_logits_without_a_choice_are_an_error(n, tmp_path):
    """A diverged model's logits give no token: neither as the only one, nor as the next step's input; the decoder serves on."""
    import test_gpu_layer_list as T
    from cut_b200.decoding import Sampling, generate
    from cut_b200.llama_decode import LlamaDecoder
    from cut_b200.models import load_model

    cfg, w = model(0, 64)
    folder = T.save_model(tmp_path / "model", T.CONFIGS["wide"], T.random_weights(T.CONFIGS["wide"], 5))
    for dec in (LlamaDecoder(cfg, w), load_model(folder, "float32", max_seq=64)):
        for fill in (float("nan"), -float("inf")):
            before = generate(dec, [5, 6, 7], 4, sampling=Sampling(seed=1))
            seq = dec.open()
            logits = dec.forward(seq, [5, 6, 7], [2])
            with pytest.raises(RuntimeError, match=f"token 0 of {n}"):
                dec.decode_sampled(seq, torch.full_like(logits, fill), n, Sampling())
            dec.close(seq)
            assert generate(dec, [5, 6, 7], 4, sampling=Sampling(seed=1)) == before


def test_replies_drawn_in_pieces(tmp_path):
    """Token by token, or a few at a time, with the logits of every piece's last token asked for: the reply that is drawn at once."""
    import test_gpu_layer_list as T
    from cut_b200.decoding import Sampling, generate
    from cut_b200.llama_decode import LlamaDecoder
    from cut_b200.models import load_model

    cfg, w = model(16, 64)
    folder = T.save_model(tmp_path / "model", T.CONFIGS["wide"], T.random_weights(T.CONFIGS["wide"], 5))
    for dec in (LlamaDecoder(cfg, w), load_model(folder, "float32", max_seq=64)):
        for how in (Sampling(temperature=3.0, seed=8), Sampling(temperature=2.0, top_k=50, seed=9)):
            want = generate(dec, [5, 6, 7], 16, sampling=how)
            for pieces in ([1] * 16, [3, 1, 7, 0, 5]):
                seq, got = dec.open(), []
                logits = dec.forward(seq, [5, 6, 7], [2])
                for n in pieces:
                    got += dec.decode_sampled(seq, logits, n, how)
                    if n and len(got) < 16:
                        logits = dec.forward(seq, got[-1:], [0])  # (the last one drawn has not been fed yet)
                dec.close(seq)
                assert got == want, pieces
