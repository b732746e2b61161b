"""Several answers to one prompt and several tokens at a time, as cases that can be timed and checked.

Two operators serve such steps.  *Attention of a batch that shares a prefix*: groups of sequences
whose first tokens lie once in the block cache (the same blocks in every table), each sequence with
tokens of its own behind them and one or a few new tokens, the last of which may be drafts.
*Verification of drafted tokens*: which of a sequence's drafts the model's probabilities let stand,
and the token behind the last of them, from uniform numbers that are inputs.

A case of attention: ``heads`` on ``kv_heads`` of ``dim`` channels, ``batch`` sequences of which
``loose`` share nothing and the rest form ``groups``; the first group's prefix has ``prefix`` tokens
(whole blocks of 64), the others' are shorter; up to ``own`` cached tokens of a sequence's own and up
to ``fresh`` new ones; ``sink``: a number per head that joins the softmax's denominator.
A case of verification: ``batch`` sequences of up to ``drafts`` drafts, ``vocab`` ids, ``temperature``
and ``top_k`` as the sampler takes them, ``proposed``: whether the drafts come with the logits that
they were drawn from (else they were looked up, and stand for certain).

Lengths follow from the case alone, so that its work does; values and the cache's order from the seed.
"""
from __future__ import annotations

import random

import torch

own = False

BLOCK = 64
DEVICE = "cuda"


# ------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------
def _attn(name, heads, kv_heads, dim, batch, prefix, own_tokens, fresh=1, groups=1, loose=0,
          sink=False, dtype="bfloat16"):
    return dict(name=name, op="attention", dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim,
                batch=batch, groups=groups, loose=loose, prefix=prefix, own=own_tokens, fresh=fresh,
                sink=sink)


def _verify(name, batch, drafts, vocab, temperature, top_k=0, proposed=True):
    return dict(name=name, op="verify", batch=batch, drafts=drafts, vocab=vocab,
                temperature=temperature, top_k=top_k, proposed=proposed)


def listed():
    return [
        # SmolLM2-135M, two answers to a short question: the call's latency
        _attn("two answers, short prompt", 9, 3, 64, batch=2, prefix=192, own_tokens=12),
        # the same model, eight answers to a prompt of some 2,000 tokens
        _attn("eight answers at 1984", 9, 3, 64, batch=8, prefix=1984, own_tokens=150),
        # SmolLM2-1.7B (a key/value head for every head), the best of 64 answers to a long prompt
        _attn("64 answers at 8000", 32, 32, 64, batch=64, prefix=8000, own_tokens=190),
        # SmolLM2-360M, 24 answers that bring up to four drafts beside their last token
        _attn("24 answers with drafts", 15, 5, 64, batch=24, prefix=4096, own_tokens=300, fresh=5),
        # heads of 128 with a sink, three prompts at once and two sequences that share nothing
        _attn("three prompts, two strangers", 16, 2, 128, batch=33, prefix=2432, own_tokens=500,
              fresh=3, groups=3, loose=2, sink=True),
        # the benchmark's wide layers (32 heads on 8), 64 answers with drafts behind a very long prompt
        _attn("64 answers with drafts at 30016", 32, 8, 64, batch=64, prefix=30016, own_tokens=500,
              fresh=5),
        # the 32-bit mode of SmolLM2-135M
        _attn("eight answers, float32", 9, 3, 64, batch=8, prefix=1984, own_tokens=150,
              dtype="float32"),
        # a single user's answer with four drafts: the call's latency
        _verify("one answer, four drafts", 1, 4, 49152, 0.8),
        # greedy answers: a draft stands where it is the arg max
        _verify("greedy, 16 answers", 16, 4, 49152, 0.0),
        # the command line's usual options, a batch of ordinary size
        _verify("top 40, 32 answers", 32, 4, 49152, 0.8, top_k=40),
        # drafts looked up in the prompt, a vocabulary of an odd size
        _verify("looked up, odd vocabulary", 12, 8, 32003, 0.7, proposed=False),
        # a full batch, seven drafts each, the whole vocabulary
        _verify("64 answers, seven drafts", 64, 7, 49152, 1.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    if rng.random() < 0.5:
        heads, kv, dim = rng.choice([(9, 3, 64), (15, 5, 64), (32, 32, 64), (32, 8, 64), (16, 2, 128),
                                     (4, 2, 16), (3, 1, 32), (10, 5, 80), (8, 8, 128)])
        dtype = "float32" if rng.random() < 0.2 else "bfloat16"
        batch = _log_int(rng, 1, 64)
        groups = rng.randint(1, max(1, min(4, batch // 2)))
        loose = rng.randint(0, max(0, (batch - groups) // 4))
        fresh = rng.choice([1, 1, 1, 2, 3, 5, 8, 11])
        # (at most the work of the largest listed case)
        longest = min(30000, int(64 * 320 * 32 * 30000 / (batch * fresh * heads * dim)),
                      int(64 * 40 * 30000 / (batch * kv * dim / 64) / 4),
                      4000 if dtype == "float32" else 30000)
        prefix = BLOCK * max(1, _log_int(rng, BLOCK, max(BLOCK, longest)) // BLOCK)
        case = _attn("", heads, kv, dim, batch, prefix, _log_int(rng, 1, 600), fresh, groups, loose,
                     rng.random() < 0.3, dtype)
        del case["name"]
        return case
    vocab = rng.choice([49152, 32003, 50001, 1000, 151, 128000])
    drafts = rng.choice([1, 2, 3, 4, 5, 7, 8, 12])
    batch = _log_int(rng, 1, max(1, min(100, int(64 * 15 * 49152 / (vocab * (2 * drafts + 1))))))
    mode = rng.random()
    temperature = 0.0 if mode < 0.2 else rng.choice([0.3, 0.7, 0.8, 1.0, 1.7])
    top_k = 0 if mode < 0.6 else _log_int(rng, 1, min(1000, vocab))
    case = _verify("", batch, drafts, vocab, temperature, top_k, rng.random() < 0.7)
    del case["name"]
    return case


def _key(case):
    return repr(sorted((k, v) for k, v in case.items() if k != "name"))


def _lengths(case):
    """(sequences of every group, its prefix), cached tokens and new tokens of every sequence."""
    rng = random.Random(_key(case))
    B, G = case["batch"], case["groups"]
    order = list(range(B))
    rng.shuffle(order)
    sharing = order[:B - case["loose"]]
    groups = []
    for g in range(G):
        members = sorted(sharing[g::G])
        blocks = case["prefix"] // BLOCK
        groups.append((members, BLOCK * (blocks if g == 0 else rng.randint(1, blocks))))
    start = [rng.randint(0, case["own"]) for _ in range(B)]
    new = [case["fresh"] if rng.random() < 0.5 else rng.randint(1, case["fresh"]) for _ in range(B)]
    for members, prefix in groups:
        for b in members:
            start[b] += prefix
    return groups, start, new


def _drafts(case):
    """How many drafts every sequence brings."""
    rng = random.Random(_key(case))
    K = case["drafts"]
    return [K if b == 0 or rng.random() < 0.6 else rng.randint(0, K) for b in range(case["batch"])]


# ------------------------------------------------------------------------------------------
# what a program has in hand
# ------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed))
    rng = random.Random(int(seed))
    return (_prepare_attention if case["op"] == "attention" else _prepare_verify)(case, gen, rng)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _prepare_attention(case, gen, rng):
    nh, nkv, hd, B = case["heads"], case["kv_heads"], case["dim"], case["batch"]
    dtype = getattr(torch, case["dtype"])
    groups, start, new = _lengths(case)
    prefix_of = [0] * B
    for members, prefix in groups:
        for b in members:
            prefix_of[b] = prefix
    need = [-(-(start[b] + new[b]) // BLOCK) for b in range(B)]
    total = sum(p // BLOCK for _, p in groups) + sum(need[b] - prefix_of[b] // BLOCK for b in range(B))
    blocks = list(range(total + 3))
    rng.shuffle(blocks)
    slots = rng.sample(range(B + 2), B)
    width = max(need) + 1
    table = [[-1] * width for _ in range(B + 2)]
    for members, prefix in groups:
        shared = [blocks.pop() for _ in range(prefix // BLOCK)]
        for b in members:
            table[slots[b]][:len(shared)] = shared
    for b in range(B):
        for i in range(prefix_of[b] // BLOCK, need[b]):
            table[slots[b]][i] = blocks.pop()
    n_blocks = total + 3

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).to(dtype)
    T = sum(new)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    packed = normal(T, (nh + 2 * nkv) * hd)             # rows q | k | v as a projection leaves them
    s = dict(case=case, q=packed[:, :nh * hd], kc=normal(n_blocks, nkv, BLOCK, hd),
             vc=normal(n_blocks, nkv, BLOCK, hd), table=_ints(table),
             tok_pos=_ints([start[b] + i for b in range(B) for i in range(new[b])]),
             tok_seq=_ints([b for b in range(B) for _ in range(new[b])]),
             tok_at=_ints([i for b in range(B) for i in range(new[b])]),
             cu_seqlens=_ints(cu), seq_slot=_ints(slots),
             scale=hd ** -0.5, fresh=max(new), blocks=max(need),
             sink=torch.randn(nh, generator=gen, device=DEVICE) if case["sink"] else None,
             out=torch.empty((T, nh * hd), dtype=dtype, device=DEVICE))
    if own:
        from cretif_b200.csrc import ops
        s["plan"] = ops.shared_prefix_plan(groups, new, start, nh, nkv, hd, dtype, DEVICE)
        s["fault"] = ops.fault_word(DEVICE)
    return s


def _prepare_verify(case, gen, rng):
    B, K, V = case["batch"], case["drafts"], case["vocab"]
    counts = _drafts(case)
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n + 1)
    R = cu[-1]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32)
    logits = 2.5 * normal(R, V)
    logits[torch.arange(R, device=DEVICE)[:, None],
           torch.randint(0, V, (R, 8), generator=gen, device=DEVICE)] += 9.0
    # a smaller model's opinion of the same places: the model's, blurred
    rows = torch.tensor([[min(cu[b] + j, cu[b + 1] - 1) for j in range(K)] for b in range(B)],
                        device=DEVICE)
    draft_logits = logits[rows] + 0.8 * normal(B, K, V)
    z = draft_logits
    if case["top_k"] and case["top_k"] < V:
        z = z.masked_fill(z < z.topk(case["top_k"], dim=-1).values[..., -1:], float("-inf"))
    if case["temperature"] > 0:
        noise = torch.rand((B, K, V), generator=gen, device=DEVICE).clamp_(1e-12, 1 - 1e-7)
        z = z / case["temperature"] - torch.log(-torch.log(noise))
    drafts = z.argmax(dim=-1).to(torch.int32)

    def uniform(*shape):
        return (torch.randint(0, 1 << 24, shape, generator=gen, device=DEVICE).float() + 0.5) / (1 << 24)
    s = dict(case=case, logits=logits, cu_rows=_ints(cu), drafts=drafts,
             draft_logits=draft_logits if case["proposed"] else None,
             accept_u=uniform(B, K), next_u=uniform(B),
             accepted=torch.empty(B, dtype=torch.int32, device=DEVICE),
             tokens=torch.empty((B, K + 1), dtype=torch.int32, device=DEVICE))
    if own:
        from cretif_b200.sampling import DraftVerifier, SamplingParams
        s["verifier"] = DraftVerifier(SamplingParams(case["temperature"], case["top_k"]), V)
    return s


# ------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    if case["op"] == "attention":
        if own:
            from cretif_b200.csrc import ops
            ops.attn_shared(s["q"], s["out"], s["kc"], s["vc"], s["table"], s["tok_pos"],
                            s["cu_seqlens"], s["seq_slot"], s["plan"], s["scale"], BLOCK, s["fault"],
                            sink=s["sink"])
            return s["out"]
        return _plain_attention(s)
    if own:
        s["verifier"](s["logits"], s["cu_rows"], s["drafts"], s["accept_u"], s["next_u"],
                      s["accepted"], s["tokens"], draft_logits=s["draft_logits"])
        return {"accepted": s["accepted"], "tokens": s["tokens"]}
    return _plain_verify(s)


def _plain_attention(s):
    """Every sequence's keys and values gathered out of the blocks, scores, softmax, sum."""
    case = s["case"]
    nh, nkv, hd, B = case["heads"], case["kv_heads"], case["dim"], case["batch"]
    g, N, nb = nh // nkv, s["fresh"], s["blocks"]
    tab = s["table"][s["seq_slot"].long(), :nb].long().clamp_min(0)
    K = s["kc"][tab].permute(0, 2, 1, 3, 4).reshape(B, nkv, nb * BLOCK, hd).float()
    V = s["vc"][tab].permute(0, 2, 1, 3, 4).reshape(B, nkv, nb * BLOCK, hd).float()
    cu = s["cu_seqlens"].long()
    at = torch.minimum(cu[:-1, None] + torch.arange(N, device=DEVICE), cu[1:, None] - 1)   # [B, N]
    q = s["q"][at].float().view(B, N, nkv, g, hd).permute(0, 2, 1, 3, 4).reshape(B, nkv, N * g, hd)
    z = (q @ K.transpose(2, 3)).view(B, nkv, N, g, nb * BLOCK) * s["scale"]
    hidden = torch.arange(nb * BLOCK, device=DEVICE) > s["tok_pos"][at][..., None]         # [B, N, L]
    z = z.masked_fill(hidden[:, None, :, None], float("-inf"))
    top = z.amax(dim=-1, keepdim=True)
    p = torch.exp(z - top)
    total = p.sum(dim=-1, keepdim=True)
    if s["sink"] is not None:
        total = total + torch.exp(s["sink"].view(1, nkv, 1, g, 1) - top)
    o = ((p / total).reshape(B, nkv, N * g, -1) @ V).view(B, nkv, N, g, hd)
    o = o[s["tok_seq"].long(), :, s["tok_at"].long()]
    return o.reshape(-1, nh * hd).to(s["out"].dtype)


def _probabilities(z, temperature, top_k):
    """Softmax over the kept ids of every row, in 64 bits."""
    z = z.double()
    if 0 < top_k < z.shape[-1]:
        order = torch.sort(z, dim=-1, descending=True, stable=True).indices
        keep = torch.zeros_like(z, dtype=torch.bool).scatter_(-1, order[..., :top_k], True)
        z = z.masked_fill(~keep, float("-inf"))
    e = torch.exp((z - z.amax(dim=-1, keepdim=True)) / temperature)
    return e / e.sum(dim=-1, keepdim=True)


def _plain_verify(s):
    case = s["case"]
    B, K, V = case["batch"], case["drafts"], case["vocab"]
    cu = s["cu_rows"].long()
    count = cu[1:] - cu[:-1] - 1
    place = torch.arange(K + 1, device=DEVICE)
    rows = torch.minimum(cu[:-1, None] + place, cu[1:, None] - 1)
    x = s["drafts"].long()
    live = place[:K] < count[:, None]
    if case["temperature"] <= 0:
        best = s["logits"].argmax(dim=-1)[rows]
        stands = live & (best[:, :K] == x)
        accepted = torch.cumprod(stands.long(), dim=1).sum(dim=1)
        token = best.gather(1, accepted[:, None])
    else:
        p = _probabilities(s["logits"][rows], case["temperature"], case["top_k"])
        if s["draft_logits"] is not None:
            q = _probabilities(s["draft_logits"], case["temperature"], case["top_k"])
        else:
            q = torch.zeros((B, K, V), dtype=torch.float64, device=DEVICE).scatter_(-1, x[..., None], 1.0)
        px, qx = p[:, :K].gather(-1, x[..., None])[..., 0], q.gather(-1, x[..., None])[..., 0]
        stands = live & (s["accept_u"].double() * qx < px)
        accepted = torch.cumprod(stands.long(), dim=1).sum(dim=1)
        each = torch.arange(B, device=DEVICE)
        r = p[each, accepted]
        left = (r - q[each, accepted.clamp_max(K - 1)]).clamp_min(0.0)
        r = torch.where((accepted < count)[:, None], left, r)
        run_sum = torch.cumsum(r, dim=-1)
        goal = s["next_u"].double()[:, None] * run_sum[:, -1:]
        token = (run_sum <= goal).sum(dim=-1, keepdim=True).clamp_max(V - 1)
    kept = torch.cat([x, x[:, :1]], dim=1)
    tokens = torch.where(place < accepted[:, None], kept,
                         torch.where(place == accepted[:, None], token, torch.full_like(kept, -1)))
    return {"accepted": accepted.to(torch.int32), "tokens": tokens.to(torch.int32)}


# ------------------------------------------------------------------------------------------
# what a pass cannot do without, and its answer in 64 bits
# ------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "attention":
        size = 4 if case["dtype"] == "float32" else 2
        nh, nkv, hd = case["heads"], case["kv_heads"], case["dim"]
        groups, start, new = _lengths(case)
        keys = sum(p for _, p in groups) + sum(a + n for a, n in zip(start, new)) \
            - sum(p * len(m) for m, p in groups)
        seen = sum(a + i + 1 for a, n in zip(start, new) for i in range(n))
        return {"bytes": size * (2 * keys * nkv * hd + 2 * sum(new) * nh * hd),
                "flops": 4 * seen * nh * hd}
    counts = _drafts(case)
    rows = sum(counts) + len(counts)
    proposed = sum(counts) if case["proposed"] and case["temperature"] > 0 else 0
    return {"bytes": 4 * case["vocab"] * (rows + proposed), "flops": 4 * case["vocab"] * (rows + proposed)}


def exact(case, seed):
    if case["op"] != "attention":
        return None                                   # ids and counts: whole numbers
    s = prepare(case, seed)
    nh, nkv, hd = case["heads"], case["kv_heads"], case["dim"]
    cu, slots, pos = s["cu_seqlens"].tolist(), s["seq_slot"].tolist(), s["tok_pos"].tolist()
    out = torch.zeros((cu[-1], nkv, nh // nkv, hd), dtype=torch.float64, device=DEVICE)
    for b, slot in enumerate(slots):
        t0, t1 = cu[b], cu[b + 1]
        length = pos[t1 - 1] + 1
        ids = s["table"][slot, :-(-length // BLOCK)].long()
        K, V = (torch.cat(list(c[ids].unbind(0)), dim=1)[:, :length].double() for c in (s["kc"], s["vc"]))
        for t in range(t0, t1):
            n = pos[t] + 1
            q = s["q"][t].double().view(nkv, nh // nkv, hd)
            a = torch.einsum("hgd,hnd->hgn", q, K[:, :n]) * s["scale"]
            if s["sink"] is not None:
                a = torch.cat([a, s["sink"].double().view(nkv, -1, 1)], dim=-1)
            out[t] = torch.einsum("hgn,hnd->hgd", torch.softmax(a, dim=-1)[..., :n], V[:, :n])
    return out.view(cu[-1], nh * hd)
