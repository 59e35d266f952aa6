"""The decoder over a paged cache and with drafted tokens: append, attention
and verification together, as a user runs them."""
import json

import numpy as np
import pytest
import torch

from conftest import rel_err
from test_gpu_decoder import TOL, _check_against_oracle, _oracle_weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tiny():
    from riallm_b200 import decoder as D
    cfg = D.DecoderConfig()
    return cfg, D.quantize_weights(D.synthetic_weights(cfg, seed=0))


def _prompt(cfg, *shape, seed=1):
    return torch.randint(0, cfg.vocab, shape, generator=torch.Generator().manual_seed(seed))


def _near_greedy(O, cfg, qw, prompt, toks):
    """Every token is the oracle's argmax, or within the tolerance of it,
    given the tokens before it."""
    from oracle.decoder_ref import DecoderRef
    ref = DecoderRef(cfg, *_oracle_weights(O, qw))
    feed, pos = prompt, 0
    for t in toks:
        r = ref.forward(feed, pos, last_only=True)[0]
        pos += len(feed)
        assert (r.max() - r[t]) / np.abs(r).max() < TOL
        feed = np.array([t])


def test_paged_greedy_matches_oracle(rb, oracle_lib, tiny):
    """64-token prompt, 16 tokens, pages of 16, graph and eager."""
    from riallm_b200 import decoder as D
    cfg, qw = tiny
    model = D.Decoder(cfg, qw, max_seq=128, page_size=16)
    prompt = _prompt(cfg, 64)
    toks, logits = model.generate(prompt.cuda(), 16, keep_logits=True)
    _check_against_oracle(oracle_lib, cfg, qw, prompt.numpy(), toks, logits.cpu().numpy())
    assert model.generate(prompt.cuda(), 16, use_graph=False) == toks
    assert model.pages.free_pages == 8 - 5  # 79 positions held
    model.reset()
    assert model.pages.free_pages == 8
    model.close()


def test_paged_matches_contiguous_batch(rb, tiny):
    """Three sequences, a pool just large enough: the contiguous cache's
    logits to bf16 rounding."""
    from riallm_b200 import decoder as D
    cfg, qw = tiny
    prompt = _prompt(cfg, 3, 37, seed=4).cuda()
    out = []
    for kw in (dict(), dict(page_size=32, num_pages=6)):
        m = D.Decoder(cfg, qw, max_batch=3, max_seq=96, **kw)
        out.append(m.generate(prompt, 8, keep_logits=True))
        m.close()
    # The first step is from the same tokens.
    assert rel_err(out[1][1][:, 0].cpu().numpy(), out[0][1][:, 0].cpu().numpy()) < TOL
    same = (out[0][0] == out[1][0]).cumprod(1).bool()
    assert same[:, 0].all()


def test_window_recycles_pages(rb, tiny):
    """A window over a pool that holds a fifth of the sequence gives what the
    same window gives with every page kept, and a window longer than the
    sequence changes nothing."""
    from riallm_b200 import decoder as D
    cfg, qw = tiny
    prompt = _prompt(cfg, 40, seed=6).cuda()

    def run(**kw):
        m = D.Decoder(cfg, qw, max_seq=256, page_size=16, **kw)
        toks, logits = m.generate(prompt, 150, keep_logits=True)
        held = int((m.pages.table >= 0).sum())
        m.close()
        return toks, logits, held
    small, large = run(window=32, sinks=4, num_pages=5), run(window=32, sinks=4)
    assert small[0] == large[0] and torch.equal(small[1], large[1])
    assert small[2] <= 4 and large[2] <= 4  # one of sinks, three of the window
    plain, wide = run(), run(window=1000, sinks=2)
    assert plain[0] == wide[0]
    assert plain[0] != small[0]


def test_pool_exhausted_leaves_state(rb, tiny):
    from riallm_b200 import decoder as D
    cfg, qw = tiny
    m = D.Decoder(cfg, qw, max_seq=128, page_size=16, num_pages=3)
    with pytest.raises(rb.MemoryError_, match="pages wanted"):
        m.forward(_prompt(cfg, 64).cuda())
    assert m.length == 0 and m.pages.free_pages == 3
    assert m.forward(_prompt(cfg, 48).cuda()).shape == (1, cfg.vocab)
    with pytest.raises(rb.MemoryError_):
        m.forward(_prompt(cfg, 1).cuda())
    assert m.length == 48
    m.close()
    for bad in (dict(window=4), dict(sinks=1), dict(num_pages=3), dict(page_size=20), dict(page_size=16, window=-1)):
        with pytest.raises(rb.ConfigError):
            D.Decoder(cfg, qw, max_seq=64, **bad)


@pytest.mark.parametrize("kw", [dict(page_size=16), dict()], ids=["paged", "contiguous"])
def test_drafted_greedy(rb, oracle_lib, tiny, kw):
    """Right guesses are accepted, wrong ones are not, and the tokens are
    greedy ones either way."""
    from riallm_b200 import decoder as D
    cfg, qw = tiny
    m = D.Decoder(cfg, qw, max_seq=96, **kw)
    prompt = _prompt(cfg, 64)
    want = m.generate(prompt.cuda(), 16)

    def right(tokens, n):
        return want[len(tokens) - 64:][:n]

    toks = m.generate_drafted(prompt.cuda(), 16, drafts=5, propose=right)
    _near_greedy(oracle_lib, cfg, qw, prompt.numpy(), toks)
    if toks == want:  # a near tie may have gone the other way
        assert m.draft_stats["accepted"] == m.draft_stats["proposed"] == 12 and m.draft_stats["steps"] == 4
    wrong = m.generate_drafted(prompt.cuda(), 16, drafts=3, propose=lambda t, n: [(t[-1] + 1) % 7] * n)
    _near_greedy(oracle_lib, cfg, qw, prompt.numpy(), wrong)
    assert m.draft_stats["accepted"] <= 1 and m.draft_stats["steps"] >= 15
    # Half right: the first guess holds, the second does not.
    half = m.generate_drafted(prompt.cuda(), 16, drafts=2,
                              propose=lambda t, n: (right(t, 1) + [cfg.vocab + 5, 3])[:n])
    _near_greedy(oracle_lib, cfg, qw, prompt.numpy(), half)
    none = m.generate_drafted(prompt.cuda(), 5, drafts=0)
    _near_greedy(oracle_lib, cfg, qw, prompt.numpy(), none)
    assert len(none) == 5
    m.close()


def test_drafted_batch_sampled(rb, tiny):
    """A batch whose sequences accept different numbers of drafts: as long as
    asked, repeatable from a seed, and the default drafts are looked up in
    the sequence."""
    from riallm_b200 import decoder as D
    cfg, qw = tiny
    m = D.Decoder(cfg, qw, max_batch=3, max_seq=80, page_size=16, num_pages=15)
    prompt = _prompt(cfg, 3, 20, seed=9)
    prompt[0, 10:] = prompt[0, :10]  # repeats itself
    runs = [m.generate_drafted(prompt.cuda(), 24, drafts=4, temperature=0.7,
                               generator=torch.Generator(device="cuda").manual_seed(s)) for s in (3, 3, 4)]
    assert all(r.shape == (3, 24) and (r >= 0).all() and (r < cfg.vocab).all() for r in runs)
    assert torch.equal(runs[0], runs[1]) and not torch.equal(runs[0], runs[2])
    greedy = m.generate(prompt.cuda(), 10)
    drafted = m.generate_drafted(prompt.cuda(), 10, propose=lambda t, n: greedy[[int(t[0]) == int(p[0]) for p in prompt]
                                                                                .index(True)].tolist()[len(t) - 20:][:n])
    assert (greedy == drafted)[:, 0].all()
    assert m.draft_stats["accepted"] > 0
    # The last position of the cache is reached, not passed.
    full = m.generate_drafted(prompt.cuda(), 61, drafts=9, propose=lambda t, n: [1] * n)
    assert full.shape == (3, 61)
    with pytest.raises(rb.ConfigError, match="max_seq"):
        m.generate_drafted(prompt.cuda(), 62)
    m.close()


def test_tiny_temperature_is_greedy(rb, tiny):
    """Sampling at a temperature that leaves only the maximum any weight gives
    the greedy tokens; bad arguments are refused."""
    from riallm_b200 import decoder as D
    cfg, qw = tiny
    m = D.Decoder(cfg, qw, max_seq=64, page_size=64)
    prompt = _prompt(cfg, 30, seed=12).cuda()
    a = m.generate_drafted(prompt, 8, temperature=0.0)
    b = m.generate_drafted(prompt, 8, temperature=1e-6)
    assert a == b
    for bad in (dict(drafts=-1), dict(drafts=256), dict(new_tokens=0)):
        with pytest.raises(rb.ConfigError):
            m.generate_drafted(prompt, **dict(dict(new_tokens=3), **bad))
    m.close()


def test_from_pretrained_paged(rb, tmp_path):
    """page_size from the model factory: the config's sliding window, plain
    and drafted generation, against a decoder built in memory."""
    from riallm_b200 import decoder as D
    from test_gpu_auto_model import _write_checkpoint
    cfg = D.DecoderConfig(vocab=4096)
    w = D.synthetic_weights(cfg, seed=0)
    w = {k: (v if "norm" in k else v.to(torch.bfloat16).float()) for k, v in w.items()}
    _write_checkpoint(str(tmp_path), cfg, w)
    config = json.loads((tmp_path / "config.json").read_text())
    config["sliding_window"] = 24
    (tmp_path / "config.json").write_text(json.dumps(config))
    prompt = _prompt(cfg, 40)
    ref = D.Decoder(cfg, D.quantize_weights(w), max_seq=128, page_size=16, window=24, sinks=4)
    want = prompt.tolist() + ref.generate(prompt.cuda(), 8)
    ref.close()
    opts = rb.ModelOptions(compression=rb.CompressionType.FourBit, prefetch_layers=False)
    m = rb.AutoModel.from_pretrained(str(tmp_path), opts, cache_dir=str(tmp_path / "q"), max_seq=128, page_size=16,
                                     num_pages=6, sinks=4)
    assert m.decoder.window == 24 and m.decoder.pages.num_pages == 6
    assert m.generate(prompt, 8) == want
    drafted = m.generate_drafted(prompt, 8, drafts=3)
    assert len(drafted) == 48 and drafted[:41] == want[:41]
    assert m.generate_drafted(prompt, 6, temperature=0.9, seed=5) == m.generate_drafted(prompt, 6, temperature=0.9, seed=5)
    assert m.generate_drafted(prompt, 0) == prompt.tolist()
    m.close()
