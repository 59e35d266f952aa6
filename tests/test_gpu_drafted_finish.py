"""generate_drafted where one sequence ends early with the cache full: the
others run on to their own ends."""
import pytest
import torch

from test_gpu_decoder_paged import _near_greedy, _prompt, tiny  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [dict(page_size=16), dict()], ids=["paged", "contiguous"])
def test_full_cache_beside_unfinished(rb, oracle_lib, tiny, kw):  # noqa: F811
    from riallm_b200 import decoder as D
    cfg, qw = tiny
    prompt, new = _prompt(cfg, 2, 37, seed=8), 12
    m = D.Decoder(cfg, qw, max_batch=2, max_seq=48, **kw)  # 37 + 12 - 1 positions
    greedy = m.generate(prompt.cuda(), new).tolist()
    first = prompt[0].tolist()

    def propose(tokens, n):
        if tokens[:37] == first:
            return greedy[0][len(tokens) - 37:][:n]
        return [(tokens[-1] + 1) % 7] * n

    toks = m.generate_drafted(prompt.cuda(), new, drafts=5, propose=propose)
    assert toks.shape == (2, new) and m.draft_stats["accepted"] >= 5
    assert m._lengths == [48, 48] and m.pos.tolist() == [48, 48]
    for b in range(2):
        _near_greedy(oracle_lib, cfg, qw, prompt[b].numpy(), toks[b].tolist())
    m.close()
