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


@pytest.mark.parametrize("page_size", [0, 16])
@pytest.mark.parametrize("prompt_len,new_tokens,max_seq", [(4, 13, 16), (5, 12, 16), (4, 12, 16), (4, 30, 64)])
def test_a_finished_sequence_holds_nobody_up(monkeypatch, rb, prompt_len, new_tokens, max_seq, page_size):
    """One sequence's drafts are all right and the others' are all wrong: the
    first ends early, with the cache full where its length is max_seq, and the
    others go on to the end, with drafts."""
    def follow(t):
        return (3 * t + 1) % 50

    m, log = stub(monkeypatch, rb, 3, max_seq, follow, page_size=page_size)
    prompt = torch.tensor([[1] * (prompt_len - 1) + [7], [2] * (prompt_len - 1) + [8], [3] * (prompt_len - 1) + [9]])
    want = [plain(p, new_tokens, follow) for p in prompt.tolist()]

    def propose(tokens, n):
        if tokens[0] == 2:
            return plain(tokens, n, follow)
        return [(follow(tokens[-1]) + 1) % 50] * n

    out = m.generate_drafted(prompt, new_tokens, drafts=4, propose=propose)
    assert out.tolist() == want
    steps = log.calls[1:]
    # The two that are left take one token a step, each with as many drafts as
    # the longest unfinished sequence has room for.
    full = prompt_len + new_tokens - 1
    assert len(steps) == new_tokens - 1
    for i, (T, pos) in enumerate(steps):
        longest = max(p for p in pos if p < full)
        assert pos[0] == pos[2] == prompt_len + i and T == 1 + min(4, new_tokens - i - 2, max_seq - longest - 1)
        assert longest + T <= max_seq
    assert m._lengths == [full] * 3 and m.length == full and m.pos.tolist() == [full] * 3


def test_room_is_asked_of_the_unfinished(monkeypatch, rb):
    """More tokens than the cache holds are refused as before."""
    m, _ = stub(monkeypatch, rb, 2, 16, lambda t: (t + 1) % 50)
    with pytest.raises(rb.ConfigError, match="max_seq"):
        m.generate_drafted(torch.tensor([[1, 2, 3, 4], [5, 6, 7, 8]]), 14)
