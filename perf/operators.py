"""Cases of the paged-cache decode operators: the rotary append into a paged
key-value cache, attention over it (with a sliding window and sinks), and the
verification of drafted tokens.

`run` computes an operator in elementary torch operations, or, with `own`
set, through riallm_b200's entry points. Attention heads are those of this
repository's configurations (32/8, 8/2 and 48/8 heads of 128, 32/4 and 16/2
of 64), vocabularies 32000 and generic ones.
"""
import math

import torch

own = False

_PHI = 0.6180339887498949


# ------------------------------------------------------------------ cases

def _attend(name, B, T, max_len, heads, kv_heads, head_dim, page_size, window=0, sinks=0):
    return {"name": name, "op": "attention", "B": B, "T": T, "max_len": max_len, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page_size": page_size, "window": window, "sinks": sinks}


def _append(name, B, T, max_len, heads, kv_heads, head_dim, page_size):
    return {"name": name, "op": "append", "B": B, "T": T, "max_len": max_len, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page_size": page_size}


def _verify(name, B, drafts, vocab, bf16, temperature, one_hot):
    return {"name": name, "op": "verify", "B": B, "drafts": drafts, "vocab": vocab, "bf16": bf16,
            "temperature": temperature, "one_hot": one_hot}


def listed():
    return [
        # One sequence just begun: nothing but latency counts.
        _attend("attend_one_short", 1, 1, 57, 32, 8, 128, 16),
        # The usual decode step: 32 sequences of up to 2000 tokens, small pages.
        _attend("attend_batch_32", 32, 1, 2000, 32, 8, 128, 16),
        # One long document: all parallelism comes from splitting its keys.
        _attend("attend_one_long", 1, 1, 131071, 32, 8, 128, 64),
        # A full server: 96 sequences, up to 16384 tokens each.
        _attend("attend_batch_96_long", 96, 1, 16384, 32, 8, 128, 32),
        # Window and sinks: the pages between them have been given back.
        _attend("attend_window_decode", 64, 1, 20011, 32, 8, 128, 16, 4096, 4),
        # A step that checks five drafted tokens per sequence.
        _attend("attend_drafted", 16, 6, 4001, 48, 8, 128, 32),
        # A prompt into an empty cache.
        _attend("attend_prompt_4096", 1, 4096, 4096, 32, 8, 128, 64),
        # The second part of two prompts, heads of 64, window and sinks.
        _attend("attend_prompt_window", 2, 2501, 9001, 16, 2, 64, 16, 2048, 4),
        # A decode step's append.
        _append("append_batch_64", 64, 1, 4000, 32, 8, 128, 16),
        # A prompt's append.
        _append("append_prompt_8192", 1, 8192, 8192, 32, 4, 64, 64),
        # One sequence, four drafted tokens.
        _verify("verify_one", 1, 4, 32000, False, 0.8, False),
        # A large batch, a large vocabulary, bf16 logits.
        _verify("verify_batch_128", 128, 5, 128001, True, 1.0, False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    nh, nkv, d = rng.choice([(32, 8, 128), (8, 2, 128), (48, 8, 128), (32, 4, 64), (16, 2, 64), (4, 4, 64)])
    ps = rng.choice([16, 32, 64, 128])
    kind = rng.choice(["decode", "decode", "decode", "drafted", "prompt", "prompt", "append", "verify"])
    if kind == "verify":
        B, n = _log(rng, 1, 128), rng.randint(1, 8)
        V = _log(rng, 1000, max(1001, min(150001, 128 * 6 * 128001 // (B * (n + 1)))))
        return {"op": "verify", "B": B, "drafts": n, "vocab": V, "bf16": rng.random() < 0.5,
                "temperature": rng.choice([0.0, 0.5, 0.8, 1.0, 1.3]), "one_hot": rng.random() < 0.25}
    if kind == "append":
        T = _log(rng, 1, 8192)
        B = _log(rng, 1, max(1, min(256, 8192 // T)))
        return {"op": "append", "B": B, "T": T, "max_len": T + _log(rng, 1, 100000 // B), "heads": nh,
                "kv_heads": nkv, "head_dim": d, "page_size": ps}
    window, sinks = (_log(rng, 64, 8192), rng.randint(0, 20)) if rng.random() < 0.4 else (0, 0)
    if kind == "prompt":
        most = 32 * 4096 * 2048  # (query, key) pairs of the largest listed prompt
        T = min(_log(rng, 9, 4096), math.isqrt(2 * most // nh))
        B = _log(rng, 1, max(1, min(4096 // T, 2 * most // (nh * T * T))))
        max_len = T + min(_log(rng, 1, 8192), most // (B * T * nh) - T // 2)
    else:
        T = 1 if kind == "decode" else rng.randint(2, 8)
        B = _log(rng, 1, 128)
        max_len = T + _log(rng, 1, min(131072, 96 * 16384 // B * 1024 // (nkv * d)))
    return {"op": "attention", "B": B, "T": T, "max_len": max_len, "heads": nh, "kv_heads": nkv, "head_dim": d,
            "page_size": ps, "window": window, "sinks": sinks}


def _lengths(case):
    """Tokens in the cache after this step's, per sequence: the first sequence has max_len, the others spread
    over [T, max_len]."""
    B, T, L = case["B"], case["T"], case["max_len"]
    return [T + int((L - T) * (1.0 - (b * _PHI) % 1.0)) for b in range(B)]


def _visible_keys(case):
    """(keys that any row of a sequence sees, (row, key) pairs that see each other), summed over the sequences."""
    T, w, s = case["T"], case["window"], case["sinks"]
    keys = pairs = 0
    for n in _lengths(case):
        first, last = n - T, n - 1
        keys += n if w == 0 else (n - max(0, first - w + 1)) + min(s, max(0, first - w + 1))
        if w == 0:
            pairs += (first + 1 + last + 1) * T // 2
        else:
            for p in range(first, last + 1):
                lo = max(0, p - w + 1)
                pairs += p - lo + 1 + min(s, lo)
    return keys, pairs


def work(case):
    if case["op"] == "verify":
        B, n, V = case["B"], case["drafts"], case["vocab"]
        # Every position's logits, and of the draft's distributions the row that the sample is taken from.
        return {"bytes": B * (n + 1) * V * (2 if case["bf16"] else 4) + (0 if case["one_hot"] else 4 * B * V),
                "flops": 3 * B * (n + 1) * V}
    nh, nkv, d, rows = case["heads"], case["kv_heads"], case["head_dim"], case["B"] * case["T"]
    if case["op"] == "append":
        return {"bytes": 4 * rows * (nh + 2 * nkv) * d + 4 * case["B"], "flops": 3 * rows * (nh + nkv) * d}
    keys, pairs = _visible_keys(case)
    return {"bytes": 4 * keys * nkv * d + 4 * rows * nh * d, "flops": 4 * pairs * nh * d}


# ----------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=g)

    if case["op"] == "verify":
        B, n, V = case["B"], case["drafts"], case["vocab"]
        # The draft model sees the target's logits through noise, and its tokens are drawn from its own distribution.
        target = normal(B, n + 1, V, dtype=torch.float32).mul_(2.5)
        guess = target[:, :n] + normal(B, n, V, dtype=torch.float32)
        noise = torch.empty((B, n, V), device="cuda").exponential_(generator=g).clamp_(min=1e-30)
        probs = torch.softmax(guess, -1)
        tokens = torch.argmax(probs / noise, -1).to(torch.int32)
        return {"case": case, "logits": target.to(torch.bfloat16) if case["bf16"] else target, "tokens": tokens,
                "probs": None if case["one_hot"] else probs,
                "temperature": torch.full((B,), case["temperature"], device="cuda"),
                "accept_u": torch.rand((B, n), device="cuda", generator=g),
                "sample_u": torch.rand((B,), device="cuda", generator=g)}

    B, T, nh, nkv, d, ps = (case[k] for k in ("B", "T", "heads", "kv_heads", "head_dim", "page_size"))
    lengths = torch.tensor(_lengths(case), device="cuda")
    pos = (lengths - T).to(torch.int32)
    per_seq = -(-max(_lengths(case)) // ps)
    page = torch.arange(per_seq, device="cuda")
    held = page[None, :] * ps < lengths[:, None]
    if case["op"] == "attention" and case["window"]:  # pages that no row sees any more have been given back
        seen = (page[None, :] * ps < case["sinks"]) | ((page[None, :] + 1) * ps > pos[:, None] - case["window"] + 1)
        held = held & seen
    count = int(held.sum())
    order = torch.randperm(count, device="cuda", generator=g).to(torch.int32)
    table = torch.full((B, per_seq), -1, dtype=torch.int32, device="cuda")
    table[held] = order
    state = {"case": case, "pos": pos, "table": table, "k_pages": normal(count, nkv, ps, d),
             "v_pages": normal(count, nkv, ps, d)}
    if case["op"] == "append":
        state["qkv"] = normal(B * T, (nh + 2 * nkv) * d)
        state["inv_freq"] = torch.tensor([1.0 / 1e6 ** (i / d) for i in range(0, d, 2)], dtype=torch.float32,
                                         device="cuda")
        state["q_out"] = torch.empty((B * T, nh * d), dtype=torch.bfloat16, device="cuda")
    else:
        # Queries of the size that makes a row's weights uneven, as trained ones are.
        state["q"] = normal(B * T, nh * d).mul_(1.5)
        state["out"] = torch.empty_like(state["q"])
    return state


# ------------------------------------------------------------ plain forms

def _rotate_plain(x, cos, sin):
    """x [rows, heads, d] in 64 bits; rotate-half."""
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _append_plain(s):
    c = s["case"]
    B, T, nh, nkv, d, ps = (c[k] for k in ("B", "T", "heads", "kv_heads", "head_dim", "page_size"))
    p = (s["pos"].long()[:, None] + torch.arange(T, device="cuda")).reshape(-1)          # [B*T]
    x = s["qkv"].view(B * T, nh + 2 * nkv, d)
    angle = p.double()[:, None] * s["inv_freq"].double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    r = _rotate_plain(x[:, :nh + nkv].float(), cos, sin).to(torch.bfloat16)
    s["q_out"].copy_(r[:, :nh].reshape(B * T, nh * d))
    row = torch.arange(B, device="cuda").repeat_interleave(T)
    page, slot = s["table"][row, p // ps].long(), p % ps
    s["k_pages"][page, :, slot] = r[:, nh:]
    s["v_pages"][page, :, slot] = x[:, nh + nkv:]
    return s["q_out"], s["k_pages"], s["v_pages"]


def _cache_rows(s, pages, dtype):
    """[B, nkv, positions, d] of the pages of each sequence, in order."""
    B, n = s["table"].shape
    x = pages[s["table"].clamp(min=0).long()].to(dtype)  # [B, n, nkv, page, d]
    return x.transpose(1, 2).reshape(B, x.shape[2], n * x.shape[3], x.shape[4])


def _mask(s):
    """[B, T, positions]: which keys each row sees."""
    c = s["case"]
    T, ps, w, sinks = c["T"], c["page_size"], c["window"], c["sinks"]
    j = torch.arange(s["table"].shape[1] * ps, device="cuda")
    p = s["pos"].long()[:, None, None] + torch.arange(T, device="cuda")[None, :, None]
    see = (j <= p) & (s["table"] >= 0).repeat_interleave(ps, 1)[:, None, :]
    if w:
        see = see & ((j > p - w) | (j < sinks))
    return see


def _attention_plain(s):
    c = s["case"]
    B, T, nh, nkv, d = (c[k] for k in ("B", "T", "heads", "kv_heads", "head_dim"))
    rep = nh // nkv
    k, v = _cache_rows(s, s["k_pages"], torch.float32), _cache_rows(s, s["v_pages"], torch.float32)
    see = _mask(s)
    v = v * see.any(1)[:, None, :, None]
    q = s["q"].view(B, T, nkv, rep, d).permute(0, 2, 3, 1, 4).reshape(B, nkv, rep * T, d).float()
    x = (q @ k.transpose(2, 3)).mul_(1.0 / math.sqrt(d)).view(B, nkv, rep, T, -1)
    x = x.masked_fill_(~see[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True).clamp(min=-3e38)
    e = x.sub_(m).exp_().view(B, nkv, rep * T, -1)
    o = (e @ v) / e.sum(-1, keepdim=True).clamp(min=1e-30)
    s["out"].copy_(o.view(B, nkv, rep, T, d).permute(0, 3, 1, 2, 4).reshape(B * T, nh * d))
    return s["out"]


def _first_true(x):
    """Index of the first true value along the last axis (its length where there is none)."""
    n = x.shape[-1]
    i = torch.arange(n, device=x.device)
    return torch.where(x, i, n).amin(-1)


def _verify_plain(s):
    logits, tokens, probs, temp = s["logits"], s["tokens"].long(), s["probs"], s["temperature"]
    B, n1, V = logits.shape
    n = n1 - 1
    x = logits.double()
    top = x.amax(-1, keepdim=True)
    greedy = torch.arange(V, device="cuda") == _first_true(x == top)[..., None]
    t = temp.double()[:, None, None]
    e = torch.exp((x - top) / torch.where(t > 0, t, 1.0))
    p = torch.where(t > 0, e / e.sum(-1, keepdim=True), greedy.double())                 # [B, n + 1, V]
    px = p[:, :n].gather(-1, tokens[..., None])[..., 0]
    qx = 1.0 if probs is None else probs.double().gather(-1, tokens[..., None])[..., 0]
    accepted = _first_true(~(s["accept_u"].double() * qx < px))                          # [B]
    b = torch.arange(B, device="cuda")
    row = p[b, accepted]
    at = accepted.clamp(max=n - 1)
    drop = (torch.arange(V, device="cuda") == tokens[b, at][:, None]).double() if probs is None else probs[b, at].double()
    rest = (row - drop * (accepted < n)[:, None]).clamp(min=0)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, row)
    upto = rest.cumsum(-1)
    hit = (upto > s["sample_u"].double()[:, None] * upto[:, -1:]) & (rest > 0)
    sample = _first_true(hit)
    i = torch.arange(n1, device="cuda")[None, :]
    drafted = torch.cat([tokens, tokens[:, :1]], 1)
    out = torch.where(i < accepted[:, None], drafted, torch.where(i == accepted[:, None], sample[:, None], -1))
    return out.to(torch.int32), accepted.to(torch.int32)


# -------------------------------------------------------------------- run

def run(state):
    op = state["case"]["op"]
    if own:
        from riallm_b200 import paged, sampling
        c = state["case"]
        if op == "attention":
            return paged.paged_attention(state["q"], state["pos"], state["table"], state["k_pages"], state["v_pages"],
                                         window=c["window"], sinks=c["sinks"], out=state["out"])
        if op == "append":
            q = paged.rope_paged_append(state["qkv"], state["pos"], state["table"], state["k_pages"],
                                        state["v_pages"], state["inv_freq"], q_out=state["q_out"])
            return q, state["k_pages"], state["v_pages"]
        return sampling.verify_draft(state["logits"], state["tokens"], state["accept_u"], state["sample_u"],
                                     temperature=state["temperature"], draft_probs=state["probs"])
    if op == "attention":
        return _attention_plain(state)
    return _append_plain(state) if op == "append" else _verify_plain(state)


# ------------------------------------------------------------------ exact

def _attention_exact(s):
    """Sequence by sequence and KV head by KV head, over the keys that exist."""
    c = s["case"]
    B, T, nh, nkv, d, ps = (c[k] for k in ("B", "T", "heads", "kv_heads", "head_dim", "page_size"))
    rep, w, sinks = nh // nkv, c["window"], c["sinks"]
    out = torch.zeros((B, T, nkv, rep, d), dtype=torch.float64, device="cuda")
    q = s["q"].double().view(B, T, nkv, rep, d)
    start = s["pos"].tolist()
    for b in range(B):
        n = start[b] + T
        j = torch.arange(n, device="cuda")
        entry = s["table"][b, j // ps].long()
        if w:
            kept = (entry >= 0) & ((j > start[b] - w) | (j < sinks))
            j, entry = j[kept], entry[kept]
        for h in range(nkv):
            k, v = s["k_pages"][entry, h, j % ps].double(), s["v_pages"][entry, h, j % ps].double()
            for t0 in range(0, T, 512):
                p = start[b] + torch.arange(t0, min(T, t0 + 512), device="cuda")
                score = torch.einsum("trd,jd->trj", q[b, t0:t0 + 512, h], k) / math.sqrt(d)
                hidden = j[None, :] > p[:, None]
                if w:
                    hidden = hidden | ((j[None, :] <= p[:, None] - w) & (j[None, :] >= sinks))
                score = torch.where(hidden[:, None, :], torch.full_like(score, -math.inf), score)
                out[b, t0:t0 + 512, h] = torch.einsum("trj,jd->trd", torch.softmax(score, -1), v)
    return out.view(B * T, nh * d)


def _append_exact(s):
    c = s["case"]
    B, T, nh, nkv, d, ps = (c[k] for k in ("B", "T", "heads", "kv_heads", "head_dim", "page_size"))
    k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    x = s["qkv"].double().view(B, T, nh + 2 * nkv, 2, d // 2)
    p = s["pos"].double()[:, None] + torch.arange(T, device="cuda", dtype=torch.float64)
    turn = torch.polar(torch.ones((B, T, 1, d // 2), dtype=torch.float64, device="cuda"),
                       p[:, :, None, None] * s["inv_freq"].double())
    z = torch.complex(x[:, :, :nh + nkv, 0], x[:, :, :nh + nkv, 1]) * turn
    y = torch.cat([z.real, z.imag], -1)
    for b in range(B):
        at = p[b].long()
        page = s["table"][b, at // ps].long()
        k_pages[page, :, at % ps] = y[b, :, nh:]
        v_pages[page, :, at % ps] = x[b, :, nh + nkv:].reshape(T, nkv, d)
    return y[:, :, :nh].reshape(B * T, nh * d), k_pages, v_pages



def exact(case, seed):
    if case["op"] == "verify":
        return None
    with torch.no_grad():
        s = prepare(case, seed)
        return _attention_exact(s) if case["op"] == "attention" else _append_exact(s)
