"""More operators of a batched serving step whose speed this repository is held to: a paged cache
that finds its scales while it is written, and the way from logits to tokens.

A case is a dict of plain values. `kind` says which operator it goes through:

  write       q/k norm per head, rotation and the write of k and v into pages whose codes have one
              scale for each block of 64 tokens and head, found from what is written
  read        keys and values read back from such pages as bf16 rows
  attention   one step of a batch over such a cache: every sequence brings its newest tokens and
              attends to its own keys and to the leading pages it shares with its group
  pick        penalties for repeated tokens, biases and grammar masks on a batch's logits, and each
              row's next token with its log-probability

`own` false: plain float32 torch. `own` true: hephaestus_amd.serve. exact() repeats a case in float64
from the definitions.

The cache: pages of 64 keys; K codes [pages, kv heads, 2, 64 keys, 64 dims] (dims in two halves), V
codes [pages, kv heads, 128 dims, 64 places], key j of the page at place v_place(j); a page's scales
[pages, 2 * kv heads], K's and then V's, are powers of two: 2^e with the least e in [-117, 119] for
which no value of the block is above 448 * 2^e. Tokens behind a page's first ones can only raise its
scale, and the codes that were there are then expressed in the new one; a call that writes a page's
key 0 begins the page anew. An attention call's tokens are its sequences' newest ones in order, so
token i of n attends to kv_len - n + i + 1 keys.

The pick: a token of the row's history (the prompt and what was answered) has its logit divided by the
repetition penalty if it is above zero, else multiplied by it; a token answered n > 0 times loses
n * frequency + presence; then the row's biases are added; tokens whose bit in the row's mask is 0
become -inf. The token is the lowest index of the largest.
"""
import math
import random

import torch

own = False

DEV = "cuda"
D = 128
PAGE = 64
EPS = 1e-6
THETA = 1e6
E4M3_MAX = 448.0
POSITIONS = 32768


def v_place(j):
    """Where a page's V rows hold key j (0..63): 16-byte runs of the keys that one lane of a
    matrix instruction takes."""
    return (j // 4 % 4) * 16 + (j // 32) * 8 + (j // 16 % 2) * 4 + j % 4


# ------------------------------------------------------------------ cases ----

def listed():
    return [
        # three decoding sequences, each somewhere in a page
        {"name": "write_t3", "kind": "write", "tokens": 3, "seqs": 3, "heads": 32, "kv_heads": 8},
        # a decode batch: a token of each of 128 sequences
        {"name": "write_t128", "kind": "write", "tokens": 128, "seqs": 128, "heads": 32,
         "kv_heads": 8},
        # a prefill chunk of several prompts, odd in all
        {"name": "write_t4090", "kind": "write", "tokens": 4090, "seqs": 6, "heads": 32,
         "kv_heads": 8},
        # a short prompt's keys, for a program that inspects or moves them
        {"name": "read_n100", "kind": "read", "rows": 100, "seqs": 1, "kv_heads": 8},
        # several long sequences leave the cache, odd in all
        {"name": "read_n65001", "kind": "read", "rows": 65001, "seqs": 5, "kv_heads": 8},
        # a few samples of one short prompt: the smallest step, where launches count
        {"name": "scaled_attn_b5_p704", "kind": "attention", "seqs": 5, "groups": 1, "prefix": 704,
         "suffix": 90, "new": 1, "heads": 32, "kv_heads": 8, "layers": 4},
        # a serving batch under three system prompts, ragged answers
        {"name": "scaled_attn_b96_p2048", "kind": "attention", "seqs": 96, "groups": 3,
         "prefix": 2048, "suffix": 1500, "new": 1, "heads": 32, "kv_heads": 8, "layers": 3},
        # one sequence decodes behind a very long document
        {"name": "scaled_attn_b1_p131008", "kind": "attention", "seqs": 1, "groups": 1,
         "prefix": 131008, "suffix": 500, "new": 1, "heads": 32, "kv_heads": 8, "layers": 2},
        # the requests' own prompts of ragged length enter behind a shared prefix
        {"name": "scaled_attn_extend_b6", "kind": "attention", "seqs": 6, "groups": 1,
         "prefix": 1024, "suffix": 900, "new": 700, "heads": 32, "kv_heads": 8, "layers": 2},
        # three greedy requests with penalties; their logits are of no further use
        {"name": "pick_r3", "kind": "pick", "rows": 3, "vocab": 151936, "history": 600, "bias": 0,
         "masks": 0, "out": False, "dtype": "float32"},
        # a decode batch that answers in grammars, its logits going on to a sampler
        {"name": "pick_r64_grammar", "kind": "pick", "rows": 64, "vocab": 151936, "history": 3500,
         "bias": 20, "masks": 9, "out": True, "dtype": "float32"},
        # the largest batch, long answers
        {"name": "pick_r256_h20000", "kind": "pick", "rows": 256, "vocab": 151936,
         "history": 20000, "bias": 0, "masks": 0, "out": False, "dtype": "float32"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["write", "read", "attention", "attention", "pick", "pick"])
    heads, kv = rng.choice([(32, 8), (32, 8), (16, 8), (16, 2), (40, 8), (8, 8)])
    if kind == "write":
        tokens = _log(rng, 1, 4096)
        return {"kind": kind, "tokens": tokens, "seqs": _log(rng, 1, min(tokens, 128)),
                "heads": min(heads, 32), "kv_heads": kv}
    if kind == "read":
        rows = _log(rng, 1, 65000)
        return {"kind": kind, "rows": rows, "seqs": _log(rng, 1, min(rows, 128)), "kv_heads": kv}
    if kind == "attention":
        seqs = _log(rng, 1, 128)
        prefix = PAGE * _log(rng, 1, 2000 if seqs < 4 else 250)
        new = 1 if rng.random() < 0.7 else _log(rng, 2, 700)
        suffix = max(_log(rng, 1, 2000), new)
        while seqs * new * (prefix + suffix) > 4_000_000:
            new = max(1, new // 2)
            prefix = max(PAGE, prefix // 2 // PAGE * PAGE) if new == 1 else prefix
        return {"kind": kind, "seqs": seqs, "groups": rng.randint(1, min(seqs, 3)),
                "prefix": prefix, "suffix": suffix, "new": new, "heads": heads, "kv_heads": kv,
                "layers": 2}
    return {"kind": kind, "rows": _log(rng, 1, 256), "vocab": _log(rng, 5000, 151936),
            "history": _log(rng, 1, 20000), "bias": rng.choice([0, 1, 20, 300]),
            "masks": rng.choice([0, 1, 9]), "out": rng.random() < 0.5,
            "dtype": rng.choice(["float32", "float32", "bfloat16"])}


# ----------------------------------------------------------------- inputs ----

def _codes(g, *shape):
    """E4M3 codes of normal values whose largest of a block lies near 448."""
    x = torch.randn(shape, generator=g, device=DEV) * 100
    return x.clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)


def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _pool(g, layers, pages, kv):
    """The pools of some layers. Blocks differ in scale: values of 1.75, 3.5 and 7 at most."""
    return {"k": _codes(g, *layers, pages, kv, 2, PAGE, D // 2),
            "v": _codes(g, *layers, pages, kv, D, PAGE),
            "scale": torch.randint(-8, -5, (*layers, pages, 2 * kv), generator=g,
                                   device=DEV).float().exp2()}


def _runs(rng, rows, seqs):
    """Runs of neighbouring positions of several sequences, and their slots in a scattered pool."""
    cuts = [0] + sorted(rng.sample(range(1, rows), seqs - 1)) + [rows]
    runs = [(rng.randint(0, max(0, POSITIONS - b + a)), b - a) for a, b in zip(cuts, cuts[1:])]
    pool = rows // PAGE + 2 * seqs + 3
    ids = rng.sample(range(pool), pool)
    positions, slots = [], []
    for first, n in runs:
        mine = {p: ids.pop() for p in range(first // PAGE, (first + n - 1) // PAGE + 1)}
        positions += range(first, first + n)
        slots += [mine[j // PAGE] * PAGE + j % PAGE for j in range(first, first + n)]
    return positions, slots, pool


def _prepare_write(case, seed, rng, g):
    tokens, heads, kv = case["tokens"], case["heads"], case["kv_heads"]
    positions, slots, pool = _runs(rng, tokens, case["seqs"])
    gamma = 1 + 0.1 * torch.randn(2, D, generator=g, device=DEV)
    return {**_pool(g, (), pool, kv),
            "qkv": torch.randn(tokens, heads + 2 * kv, D, generator=g,
                               device=DEV).to(torch.bfloat16),
            "q_gamma": gamma[0].to(torch.bfloat16), "k_gamma": gamma[1].to(torch.bfloat16),
            "positions": _int32(positions), "slots": _int32(slots),
            # a serving program keeps the rotation's cos and sin: [positions, 64 pairs, 2]
            "rope": _rope(torch.arange(POSITIONS, device=DEV)),
            "pages": torch.tensor(sorted({s // PAGE for s in slots}), device=DEV),
            "q": torch.zeros(tokens, heads, D, dtype=torch.bfloat16, device=DEV)}


def _prepare_read(case, seed, rng, g):
    _, slots, pool = _runs(rng, case["rows"], case["seqs"])
    shape = (2, case["rows"], case["kv_heads"], D)
    rows = torch.zeros(shape, dtype=torch.bfloat16, device=DEV)
    return {**_pool(g, (), pool, case["kv_heads"]), "slots": _int32(slots), "k_rows": rows[0],
            "v_rows": rows[1]}


def _batch(case, seed):
    """An attention batch on the host: per sequence its new tokens, its keys and its page ids; per
    group its sequences and shared pages."""
    seqs, groups = case["seqs"], case["groups"]
    rng = random.Random(seqs * case["new"] + 3)        # ragged, but as many tokens for every seed
    new = [1 if case["new"] == 1 else rng.randint(1, case["new"]) for _ in range(seqs)]
    rng = random.Random(seed * 7919 + 1)
    own_keys = [max(n, rng.randint(1, case["suffix"])) for n in new]
    start = [seqs * g // groups for g in range(groups + 1)]
    shared = [max(1, case["prefix"] // PAGE // (g + 1)) for g in range(groups)]
    pool = sum(shared) + sum(-(-n // PAGE) for n in own_keys) + 3
    ids = rng.sample(range(pool), pool)                # pages lie anywhere in the pool
    prefixes = [[ids.pop() for _ in range(n)] for n in shared]
    of = [g for g in range(groups) for _ in range(start[g], start[g + 1])]
    tables = [prefixes[g] + [ids.pop() for _ in range(-(-n // PAGE))]
              for g, n in zip(of, own_keys)]
    return {"new": new, "kv_len": [shared[g] * PAGE + n for g, n in zip(of, own_keys)],
            "tables": tables, "group_start": start, "shared": shared, "pool": pool,
            "q_start": [sum(new[:i]) for i in range(seqs + 1)], "of": of}


def _padded(tokens, pages, first_key, end_key):
    """Batches of ragged token and page lists, padded with their first entries: the tokens, where
    each token's row lies, the pages, and each batch's first and end key."""
    rows, cols = max(len(t) for t in tokens), max(len(p) for p in pages)
    where = [(t, i * rows + j) for i, ts in enumerate(tokens) for j, t in enumerate(ts)]
    return {"tokens": torch.tensor([t + t[:1] * (rows - len(t)) for t in tokens], device=DEV),
            "where": torch.tensor([w for _, w in sorted(where)], device=DEV),
            "pages": torch.tensor([p + p[:1] * (cols - len(p)) for p in pages], device=DEV),
            "first": torch.tensor(first_key, device=DEV), "end": torch.tensor(end_key, device=DEV)}


def _prepare_attention(case, seed, rng, g):
    b = _batch(case, seed)
    layers, tokens, at = case["layers"], b["q_start"][-1], b["q_start"]
    width = max(len(t) for t in b["tables"])
    seqs, shared = range(case["seqs"]), [b["shared"][g] for g in b["of"]]
    bounds = list(zip(b["group_start"], b["group_start"][1:]))
    limit = [b["kv_len"][s] - b["new"][s] + i + 1 for s in seqs for i in range(b["new"][s])]
    shape = (layers, tokens, case["heads"], D)
    return {**_pool(g, (layers,), b["pool"], case["kv_heads"]), "batch": b,
            "q": torch.randn(shape, generator=g, device=DEV).to(torch.bfloat16),
            "table": _int32([t + [-1] * (width - len(t)) for t in b["tables"]]),
            "q_start": _int32(b["q_start"]), "kv_len": _int32(b["kv_len"]),
            "group_start": _int32(b["group_start"]), "shared": _int32(b["shared"]),
            # index tensors of the plain form's two padded batches: all groups' prefixes, all
            # sequences' own keys
            "limit": torch.tensor(limit, device=DEV),
            "prefix": _padded([list(range(at[a], at[c])) for a, c in bounds],
                              [b["tables"][a][:n] for (a, _), n in zip(bounds, b["shared"])],
                              [0] * len(bounds), [n * PAGE for n in b["shared"]]),
            "suffix": _padded([list(range(at[s], at[s + 1])) for s in seqs],
                              [b["tables"][s][shared[s]:] for s in seqs],
                              [n * PAGE for n in shared], b["kv_len"]),
            "out": torch.zeros(shape, dtype=torch.bfloat16, device=DEV)}


def _prepare_pick(case, seed, rng, g):
    rows, vocab, cap, bias, masks = (case[f] for f in ("rows", "vocab", "history", "bias", "masks"))
    n_slots, words = rows + 3, -(-vocab // 32)
    length = [rng.randint(1, cap) for _ in range(n_slots)]
    # some words come often, most hardly ever
    u = torch.rand(n_slots, cap, generator=g, device=DEV)
    words_of = torch.randperm(vocab, generator=g, device=DEV)
    bits = torch.randint(0, 1 << 32, (3, max(masks, 1), words), generator=g, device=DEV)
    bits = bits[0] & bits[1] & bits[2]                 # a grammar allows an eighth of the tokens
    logits = torch.randn(rows, vocab, generator=g, device=DEV) * 3
    dtype = getattr(torch, case["dtype"])
    ids = torch.rand(n_slots, vocab, generator=g, device=DEV).topk(max(bias, 1)).indices
    penalties = torch.rand(n_slots, 3, generator=g, device=DEV) * 0.5
    penalties[:, 0] += 1
    return {"logits": logits.to(dtype), "slots": _int32(rng.sample(range(n_slots), rows)),
            "history": words_of[(vocab ** u).long() - 1].int(), "length": _int32(length),
            "n_prompt": _int32([rng.randint(0, n) for n in length]), "penalties": penalties,
            "bias_ids": ids.int(), "n_bias": _int32([rng.randint(0, bias) for _ in length]),
            "bias": torch.randn(n_slots, max(bias, 1), generator=g, device=DEV) * 4,
            "masks": (bits - ((bits >> 31) << 32)).int() if masks else None,
            "mask_ids": _int32([rng.randrange(-1, masks) for _ in range(rows)]) if masks else None,
            "out": torch.zeros(rows, vocab, dtype=dtype, device=DEV) if case["out"] else None,
            "tokens": torch.zeros(rows, dtype=torch.int32, device=DEV),
            "logprob": torch.zeros(rows, dtype=torch.float32, device=DEV)}


def prepare(case, seed):
    make = {"write": _prepare_write, "read": _prepare_read, "attention": _prepare_attention,
            "pick": _prepare_pick}[case["kind"]]
    g = torch.Generator(device=DEV).manual_seed(seed)
    return {**make(case, seed, random.Random(seed * 7919 + 2), g), "case": case}


# ------------------------------------------------------------- plain forms ----

def _rope(positions):
    freq = THETA ** (-torch.arange(0, D, 2, dtype=torch.float64, device=DEV) / D)
    angle = positions.to(torch.float64)[:, None] * freq
    return torch.stack([angle.cos(), angle.sin()], dim=-1).float()


def _values(codes):
    return codes.view(torch.float8_e4m3fn).float()


def _to_codes(x):
    return x.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)


def _norm_rope(x, gamma, cos, sin):
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gamma.float()
    a, b = y[..., :D // 2], y[..., D // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _places(key):
    return key // 4 % 4 * 16 + key // 32 * 8 + key // 16 % 2 * 4 + key % 4


def _write_plain(s):
    kv, heads = s["k"].shape[1], s["q"].shape[1]
    page, key = s["slots"].long() // PAGE, s["slots"].long() % PAGE
    x = s["qkv"].float()
    cos, sin = s["rope"][s["positions"].long()][:, None].unbind(-1)
    s["q"].copy_(_norm_rope(x[:, :heads], s["q_gamma"], cos, sin))
    k, v = _norm_rope(x[:, heads:heads + kv], s["k_gamma"], cos, sin), x[:, heads + kv:]
    # the blocks' new scales
    amax = torch.cat([k, v], 1).abs().amax(-1)
    amax = torch.zeros_like(s["scale"]).scatter_reduce(0, page[:, None].expand_as(amax), amax,
                                                       "amax")[s["pages"]]
    fraction, exponent = torch.frexp(amax.clamp_min(2.0 ** -112))
    scale = torch.ldexp(torch.ones_like(amax),
                        (exponent - 9 + (fraction > 0.875)).clamp(-117, 119))
    fresh = torch.zeros(len(s["k"]), device=DEV).scatter_reduce(0, page, (key == 0).float(), "amax")
    fresh, old = fresh[s["pages"], None] > 0, s["scale"][s["pages"]]
    scale = torch.where(fresh, scale, torch.maximum(scale, old))
    s["scale"][s["pages"]] = scale
    # the codes that were there in the new scales, and then the new ones
    grown = torch.where(fresh, 1.0, old / scale)[..., None, None]
    s["k"][s["pages"]] = _to_codes(_values(s["k"][s["pages"]]) * grown[:, :kv, :, None])
    s["v"][s["pages"]] = _to_codes(_values(s["v"][s["pages"]]) * grown[:, kv:])
    inv = 1 / s["scale"][page][..., None]
    s["k"][page, :, :, key] = _to_codes(k * inv[:, :kv]).view(-1, kv, 2, D // 2)
    s["v"][page, :, :, _places(key)] = _to_codes(v * inv[:, kv:])
    return (s["q"], s["k"].view(torch.float8_e4m3fn), s["v"].view(torch.float8_e4m3fn), s["scale"])


def _read_plain(s):
    kv = s["k"].shape[1]
    page, key = s["slots"].long() // PAGE, s["slots"].long() % PAGE
    scale = s["scale"][page][..., None]
    k = _values(s["k"][page, :, :, key]).flatten(2) * scale[:, :kv]
    v = _values(s["v"][page, :, :, _places(key)]) * scale[:, kv:]
    return k.to(torch.bfloat16), v.to(torch.bfloat16)


def _partial_attention(q, k, v, ix, limit):
    """Softmax numerator, denominator and maximum of every token over its batch's keys."""
    heads, kv = q.shape[1], k.shape[1]
    keys = k[ix["pages"]].transpose(1, 2).flatten(2, 3)            # [batch, kv, keys, 128]
    vals = v[ix["pages"]].transpose(1, 2).flatten(2, 3)
    batch, rows = ix["tokens"].shape
    qs = q[ix["tokens"]].view(batch, rows, kv, heads // kv, D).transpose(1, 2).flatten(2, 3)
    x = (qs @ keys.transpose(-1, -2).contiguous()).view(batch, kv, rows, heads // kv, -1) * D ** -0.5
    at = ix["first"][:, None] + torch.arange(keys.shape[2], device=DEV)
    seen = (at[:, None] < limit[ix["tokens"]][:, :, None]) & (at < ix["end"][:, None])[:, None]
    x = x.masked_fill(~seen[:, None, :, None], -torch.inf)
    m = x.amax(-1).clamp_min(-1e30)
    p = torch.exp(x - m[..., None])
    o = (p.flatten(2, 3) @ vals).view(batch, kv, rows, heads // kv, D)

    def of_tokens(t):
        return t.transpose(1, 2).reshape(batch * rows, heads, *t.shape[4:])[ix["where"]]

    return of_tokens(o), of_tokens(p.sum(-1)), of_tokens(m)


def _attention_plain(s, i):
    kv = s["k"].shape[2]
    scale = s["scale"][i][..., None, None]
    k = _values(s["k"][i])
    k = torch.cat([k[:, :, 0], k[:, :, 1]], dim=-1) * scale[:, :kv]
    v = _values(s["v"][i])[..., _places(torch.arange(PAGE, device=DEV))].transpose(-1, -2)
    v = v * scale[:, kv:]
    q = s["q"][i].float()
    o1, l1, m1 = _partial_attention(q, k, v, s["prefix"], s["limit"])
    o2, l2, m2 = _partial_attention(q, k, v, s["suffix"], s["limit"])
    m = torch.maximum(m1, m2)
    w1, w2 = torch.exp(m1 - m), torch.exp(m2 - m)
    o = (o1 * w1[..., None] + o2 * w2[..., None]) / (l1 * w1 + l2 * w2)[..., None]
    return o.to(torch.bfloat16)


def _pick_plain(s):
    rows, vocab = s["logits"].shape
    x, slot = s["logits"].float(), s["slots"].long()
    history, length = s["history"][slot].long(), s["length"][slot, None]
    at = torch.arange(history.shape[1], device=DEV)
    live = at < length
    count = torch.zeros(rows, vocab, dtype=torch.int32, device=DEV)
    seen = count.scatter_add(1, history, live.int()) > 0
    count = count.scatter_add(1, history, (live & (at >= s["n_prompt"][slot, None])).int())
    repetition, presence, frequency = s["penalties"][slot, :, None].unbind(1)
    x = torch.where(seen, torch.where(x > 0, x / repetition, x * repetition), x)
    x = torch.where(count > 0, x - (count * frequency + presence), x)
    entry = torch.arange(s["bias_ids"].shape[1], device=DEV) < s["n_bias"][slot, None]
    x = x.scatter_add(1, s["bias_ids"][slot].long(), torch.where(entry, s["bias"][slot], 0.0))
    if s["masks"] is not None:
        bits = s["masks"][s["mask_ids"].clamp_min(0).long()][..., None]
        bits = (bits >> torch.arange(32, device=DEV, dtype=torch.int32) & 1).flatten(1)[:, :vocab]
        x = x.masked_fill((bits == 0) & (s["mask_ids"] >= 0)[:, None], -torch.inf)
    top = x.amax(-1, keepdim=True)
    token = torch.where(x == top, torch.arange(vocab, device=DEV), vocab).amin(-1)
    logprob = -(x - top).exp().sum(-1).log()
    out = x.to(s["logits"].dtype) if s["out"] is not None else None
    return token.int(), logprob, out


# -------------------------------------------------------------------- run ----

def _run_own(s):
    from hephaestus_amd import serve
    case = s["case"]
    if case["kind"] == "write":
        serve.qk_norm_rope_pages_scaled(s["q"], s["qkv"], s["q_gamma"], s["k_gamma"], s["k"], s["v"],
                                        s["scale"], s["rope"], s["positions"], s["slots"], EPS)
        return (s["q"], s["k"].view(torch.float8_e4m3fn), s["v"].view(torch.float8_e4m3fn),
                s["scale"])
    if case["kind"] == "read":
        serve.read_pages(s["k_rows"], s["v_rows"], s["k"], s["v"], s["slots"],
                         page_scale=s["scale"])
        return s["k_rows"], s["v_rows"]
    if case["kind"] == "attention":
        if "plan" not in s:                                  # the step's workspaces
            s["plan"] = serve.AttentionPlan(case["seqs"], s["q"].shape[1], case["heads"],
                                            case["kv_heads"], s["table"].shape[1],
                                            n_groups=case["groups"])
        s["plan"].update(s["q_start"], s["kv_len"], s["group_start"], s["shared"])
        for i in range(case["layers"]):
            serve.attention_pages_scaled(s["out"][i], s["q"][i], s["k"][i], s["v"][i], s["scale"][i],
                                         s["table"], s["plan"])
        return s["out"]
    if "rules" not in s:                                     # the requests' rules, kept on the device
        s["rules"] = serve.TokenRules(len(s["length"]), case["vocab"], s["history"].shape[1],
                                      s["bias"].shape[1])
        for name in ("history", "length", "n_prompt", "penalties", "bias_ids", "bias", "n_bias"):
            getattr(s["rules"], name).copy_(s[name])
        s["ws"] = serve.pick_ws(case["rows"], case["vocab"])
    serve.pick_tokens(s["tokens"], s["logits"], s["rules"], s["slots"], masks=s["masks"],
                      mask_ids=s["mask_ids"], out=s["out"], logprob=s["logprob"], ws=s["ws"])
    return s["tokens"], s["logprob"], s["out"]


def run(state):
    kind = state["case"]["kind"]
    if own:
        return _run_own(state)
    if kind == "write":
        return _write_plain(state)
    if kind == "read":
        return _read_plain(state)
    if kind == "attention":
        return torch.stack([_attention_plain(state, i) for i in range(state["case"]["layers"])])
    return _pick_plain(state)


# ---------------------------------------------------------- work and exact ----

def work(case):
    kind, kv = case["kind"], case.get("kv_heads")
    if kind == "write":
        heads, t = case["heads"], case["tokens"]
        return {"bytes": t * (D * (2 * (heads + 2 * kv) + 2 * heads + 2 * kv) + D * 4 + 8),
                "flops": t * D * (heads + kv) * 8}
    if kind == "read":
        return {"bytes": case["rows"] * (kv * D * 6 + 4), "flops": case["rows"] * kv * D * 2}
    if kind == "attention":
        b = _batch(case, 1)
        keys = sum(b["shared"]) * PAGE + sum(n - PAGE * b["shared"][g]
                                             for n, g in zip(b["kv_len"], b["of"]))
        pairs = sum(n * (2 * k - n + 1) // 2 for n, k in zip(b["new"], b["kv_len"]))
        return {"bytes": case["layers"] * (keys * kv * D * 2 + sum(b["new"]) * case["heads"] * D * 4),
                "flops": case["layers"] * pairs * case["heads"] * D * 4}
    n, size = case["rows"] * case["vocab"], 4 if case["dtype"] == "float32" else 2
    return {"bytes": n * size * (2 if case["out"] else 1) + min(case["masks"], case["rows"])
            * case["vocab"] // 8 + case["rows"] * case["history"] * 2, "flops": n * 4}


def _exact_write(s):
    heads, kv = s["q"].shape[1], s["k"].shape[1]
    x = s["qkv"].double()
    gamma = torch.cat([s["q_gamma"].expand(heads, D), s["k_gamma"].expand(kv, D)]).double()
    y = x[:, :heads + kv]
    y = gamma * y / torch.sqrt((y * y).sum(-1, keepdim=True) / D + EPS)
    pair = torch.arange(D // 2, dtype=torch.float64, device=DEV)
    angle = s["positions"].double()[:, None, None] / torch.pow(THETA, 2 * pair / D)
    z = torch.complex(y[..., :D // 2], y[..., D // 2:]) * torch.polar(torch.ones_like(angle), angle)
    y = torch.cat([z.real, z.imag], -1)
    # cached values: the codes' own, where no rounding to codes is counted
    k, v = (s[f].view(torch.float8_e4m3fn).double() for f in ("k", "v"))
    scale, new = s["scale"].double(), torch.cat([y[:, heads:], x[:, heads + kv:]], 1)
    order = torch.argsort(s["slots"] // PAGE, stable=True)
    pages, counts = torch.unique_consecutive(s["slots"][order] // PAGE, return_counts=True)
    for p, rows in zip(pages.tolist(), order.split(counts.tolist())):
        e = torch.ceil(torch.log2(new[rows].abs().amax(0).amax(-1) / E4M3_MAX)).clamp(-117, 119)
        if not (s["slots"][rows] % PAGE == 0).any():
            e = torch.maximum(e, torch.log2(scale[p]))
            f = (scale[p] / 2 ** e)[:, None, None]
            k[p] *= f[:kv, :, None]
            v[p] *= f[kv:]
        scale[p] = 2 ** e
        key = s["slots"][rows].long() % PAGE
        value = (new[rows] / scale[p][:, None]).clamp(-E4M3_MAX, E4M3_MAX)
        k[p][:, :, key] = value[:, :kv].unflatten(-1, (2, D // 2)).permute(1, 2, 0, 3)
        place = torch.tensor([v_place(j) for j in range(PAGE)], device=DEV)[key]
        v[p][:, :, place] = value[:, kv:].permute(1, 2, 0)
    return y[:, :heads], k, v, scale


def _exact_read(s):
    kv, place = s["k"].shape[1], [v_place(j) for j in range(PAGE)]
    scale = s["scale"].double()[:, :, None, None]
    k = s["k"].view(torch.float8_e4m3fn).double().permute(0, 1, 3, 2, 4).flatten(3) * scale[:, :kv]
    v = s["v"].view(torch.float8_e4m3fn).double()[..., place].transpose(2, 3) * scale[:, kv:]
    return tuple(x.transpose(1, 2).flatten(0, 1)[s["slots"].long()] for x in (k, v))


def _exact_attention(s):
    b, case = s["batch"], s["case"]
    heads, kv, place = case["heads"], case["kv_heads"], [v_place(j) for j in range(PAGE)]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for layer in range(case["layers"]):
        for i, (table, n, keys) in enumerate(zip(b["tables"], b["new"], b["kv_len"])):
            t, scale = b["q_start"][i], s["scale"][layer, table].double()[:, :, None, None]
            # [pages, kv, 2, 64, 64] -> [kv, keys, 128]
            ks = s["k"][layer, table].view(torch.float8_e4m3fn).double().permute(0, 1, 3, 2, 4)
            ks = (ks.flatten(3) * scale[:, :kv]).transpose(0, 1).flatten(1, 2)[:, :keys]
            vs = s["v"][layer, table].view(torch.float8_e4m3fn).double()[..., place].transpose(2, 3)
            vs = (vs * scale[:, kv:]).transpose(0, 1).flatten(1, 2)[:, :keys]
            q = s["q"][layer, t:t + n].double().view(n, kv, heads // kv, D).permute(1, 2, 0, 3)
            x = q.reshape(kv, -1, D) @ ks.transpose(1, 2).contiguous() / math.sqrt(D)
            x = x.view(kv, heads // kv, n, keys)
            later = torch.arange(keys, device=DEV) > (torch.arange(n, device=DEV) + keys - n)[:, None]
            p = torch.softmax(x.masked_fill(later, -math.inf), -1)
            o = (p.view(kv, -1, keys) @ vs).view(kv, heads // kv, n, D)
            out[layer, t:t + n] = o.permute(2, 0, 1, 3).reshape(n, heads, D)
    return out


def _exact_pick(s):
    vocab, out, logprob = s["case"]["vocab"], [], []
    for r, slot in enumerate(s["slots"].tolist()):
        x, n, first = s["logits"][r].double(), int(s["length"][slot]), int(s["n_prompt"][slot])
        tokens = s["history"][slot, :n].long()
        repetition, presence, frequency = s["penalties"][slot].double()
        seen = torch.unique(tokens)
        x[seen] = torch.minimum(x[seen] / repetition, x[seen] * repetition)
        answered, times = torch.unique(tokens[first:], return_counts=True)
        x[answered] -= times * frequency + presence
        n = int(s["n_bias"][slot])
        x[s["bias_ids"][slot, :n].long()] += s["bias"][slot, :n].double()
        if s["masks"] is not None and int(s["mask_ids"][r]) >= 0:
            at = torch.arange(vocab, device=DEV)
            word = s["masks"][int(s["mask_ids"][r])].long()[at // 32]
            x[(word >> at % 32) % 2 == 0] = -math.inf
        out.append(x)
        logprob.append(x.max() - torch.logsumexp(x, 0))
    return None, torch.stack(logprob), torch.stack(out) if s["out"] is not None else None


def exact(case, seed):
    f = {"write": _exact_write, "read": _exact_read, "attention": _exact_attention,
         "pick": _exact_pick}
    return f[case["kind"]](prepare(case, seed))
