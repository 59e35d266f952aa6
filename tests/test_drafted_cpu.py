"""generate_drafted's host side on the CPU, without its kernels: a decoder
whose model step is a table look-up and whose verification is the greedy
rule."""
import pytest
import torch


class Steps:
    """What a decoder's model step was given: (tokens a sequence, first
    positions)."""

    def __init__(self):
        self.calls = []


def stub(monkeypatch, rb, batch, max_seq, follow, vocab=50, page_size=0):
    """A decoder whose model answers follow(token) after every token."""
    from riallm_b200 import decoder as D
    m = object.__new__(D.Decoder)
    m.cfg = D.DecoderConfig(vocab=vocab)
    m.dev, m.ctx, m.ep, m.streamer = torch.device("cpu"), None, None, None
    m.max_batch, m.max_seq, m.window, m.sinks, m.pages = batch, max_seq, 0, 0, None
    m.pos, m.length, m._lengths = torch.zeros(batch, dtype=torch.int32), 0, [0] * batch
    if page_size:
        from riallm_b200.paged import PagedKVCache
        c = m.pages = object.__new__(PagedKVCache)
        c.page_size, c.max_pages = page_size, -(-max_seq // page_size)
        c.num_pages = batch * c.max_pages
        c.table = torch.full((batch, c.max_pages), -1, dtype=torch.int32)
        c._init_host(batch)
    log = Steps()

    def forward(ids, experts_used=None, all_logits=False):
        B, T = ids.shape
        log.calls.append((T, m.pos[:B].tolist()))
        m.pos[:B] += T
        logits = torch.nn.functional.one_hot(ids.apply_(follow), vocab).float()
        return logits if all_logits else logits[:, -1]

    def verify(logits, draft, accept_u, sample_u, temperature, draft_probs=None, ctx=None):
        top = logits.argmax(-1)
        B, n1 = top.shape
        tokens, accepted = torch.full((B, n1), -1, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)
        for b in range(B):
            a = 0
            while a < n1 - 1 and int(draft[b, a]) == int(top[b, a]):
                a += 1
            tokens[b, :a + 1], accepted[b] = top[b, :a + 1], a
        return tokens, accepted

    m._forward = forward
    monkeypatch.setattr(D, "verify_draft", verify)
    return m, log


def plain(prompt, new_tokens, follow):
    out = [int(prompt[-1])]
    for _ in range(new_tokens):
        out.append(follow(out[-1]))
    return out[1:]


def test_expert_parallel_is_refused(monkeypatch, rb):
    """Ranks would take steps of different sizes and numbers: refused before
    the model runs."""
    m, log = stub(monkeypatch, rb, 1, 64, lambda t: (t + 1) % 50)
    m.ep = object()
    with pytest.raises(rb.ConfigError, match="expert-parallel"):
        m.generate_drafted(torch.tensor([1, 2, 3]), 5)
    assert log.calls == [] and m.length == 0
