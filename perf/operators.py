"""The operators of a batched serving step whose speed this repository is held to.

A case is a dict of plain values. `kind` says which operator it goes through:

  attention   one step of a batch over the paged E4M3 cache: every sequence brings its newest tokens
              and attends to its own keys and to the leading pages it shares with its group
  qk          q/k norm per head, rotation and the write of k and v into pages, for a batch of tokens
  pages       pages of all layers copied within the pools (fork of a prefix's tail, compaction)
  lora        low-rank adapters of many requests added to the output of a shared projection

With several layers each has its own cache, weights and rows, as in a forward pass, and what one
step's layers share (the plan of the batch) is made once a pass, inside the pass.

`own` false: plain float32 torch. `own` true: hephaestus_amd.serve. exact() repeats a case in float64
from the definitions.

Layouts (64-key pages): K codes [pages, kv heads, 2, 64 keys, 64 dims] (dims in two halves); V codes
[pages, kv heads, 128 dims, 64 places], key j of the page at place v_place(j). An attention call's
tokens are its sequences' newest ones in order, so token i of n attends to kv_len - n + i + 1 keys.
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
KV_AMAX = 5.0          # the caches' scale is this / 448: about the amax of a few thousand normals


def v_place(j):
    """Where a page's V rows hold key j (0..63): 16-byte runs of the keys that one lane of a
    matrix instruction takes."""
    return (j // 4 % 4) * 16 + (j // 32) * 8 + (j // 16 % 2) * 4 + j % 4


# ------------------------------------------------------------------ cases ----

def listed():
    return [
        # a few samples of one short prompt: the smallest step, where launches count
        {"name": "attn_b4_p512", "kind": "attention", "seqs": 4, "groups": 1, "prefix": 512,
         "suffix": 100, "new": 1, "heads": 32, "kv_heads": 8, "layers": 4},
        # a serving batch under two system prompts, ragged answers
        {"name": "attn_b64_p4096", "kind": "attention", "seqs": 64, "groups": 2, "prefix": 4096,
         "suffix": 1000, "new": 1, "heads": 32, "kv_heads": 8, "layers": 4},
        # many questions about one long document
        {"name": "attn_b128_p19968", "kind": "attention", "seqs": 128, "groups": 1,
         "prefix": 19968, "suffix": 2000, "new": 1, "heads": 32, "kv_heads": 8, "layers": 2},
        # the requests' own prompts of ragged length enter behind a shared prefix
        {"name": "attn_extend_b8", "kind": "attention", "seqs": 8, "groups": 1, "prefix": 2048,
         "suffix": 600, "new": 500, "heads": 32, "kv_heads": 8, "layers": 2},
        # three decoding sequences
        {"name": "qk_t3", "kind": "qk", "tokens": 3, "seqs": 3, "heads": 32, "kv_heads": 8},
        # a decode batch at scattered positions
        {"name": "qk_t128", "kind": "qk", "tokens": 128, "seqs": 128, "heads": 32, "kv_heads": 8},
        # a prefill chunk of several prompts, odd in all
        {"name": "qk_t4090", "kind": "qk", "tokens": 4090, "seqs": 6, "heads": 32, "kv_heads": 8},
        # eight sequences fork off a prefix: its partly filled last page is copied for each
        {"name": "pages_fork_8", "kind": "pages", "copies": 8, "pages": 24, "kv_heads": 8,
         "layers": 36},
        # a fragmented pool is compacted: live pages move down into holes
        {"name": "pages_compact_64", "kind": "pages", "copies": 64, "pages": 160, "kv_heads": 8,
         "layers": 36},
        # five decoding requests with three adapters, beside the fused q|k|v projection
        {"name": "lora_qkv_m5", "kind": "lora", "m": 5, "n": 6144, "k": 2560, "rank": 16,
         "adapters": 3, "layers": 4},
        # a decode batch of many tenants beside gate|up
        {"name": "lora_gate_up_m64", "kind": "lora", "m": 64, "n": 19456, "k": 2560, "rank": 16,
         "adapters": 40, "layers": 2},
        # a prefill chunk of several tenants' prompts beside down_proj, odd in all
        {"name": "lora_down_m4090", "kind": "lora", "m": 4090, "n": 2560, "k": 9728, "rank": 64,
         "adapters": 5, "layers": 1},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "qk", "pages", "lora", "lora"])
    heads, kv = rng.choice([(32, 8), (32, 8), (16, 8), (16, 2), (40, 8), (8, 8)])
    if kind == "attention":
        seqs = _log(rng, 1, 128)
        prefix = PAGE * _log(rng, 1, 312)
        new = 1 if rng.random() < 0.7 else _log(rng, 2, 500)
        suffix = max(_log(rng, 1, 2000), new)
        while seqs * new * (prefix + suffix) > 4_000_000:      # the largest listed case's
            new = max(1, new // 2)
            prefix = max(PAGE, prefix // 2 // PAGE * PAGE) if new == 1 else prefix
        return {"kind": kind, "seqs": seqs, "groups": rng.randint(1, min(seqs, 3)),
                "prefix": prefix, "suffix": suffix, "new": new, "heads": heads, "kv_heads": kv,
                "layers": 2}
    if kind == "qk":
        tokens = _log(rng, 1, 4096)
        return {"kind": kind, "tokens": tokens, "seqs": _log(rng, 1, min(tokens, 128)),
                "heads": min(heads, 32), "kv_heads": kv}
    if kind == "pages":
        copies = _log(rng, 1, 64)
        return {"kind": kind, "copies": copies, "pages": 2 * copies + rng.randint(0, 24),
                "kv_heads": kv, "layers": rng.randint(1, 36)}
    m = _log(rng, 1, 4096)
    return {"kind": "lora", "m": m, "n": 16 * rng.randint(16, 160), "k": 128 * rng.randint(2, 76),
            "rank": 8 * _log(rng, 1, 8), "adapters": _log(rng, 1, min(m, 40) if m <= 256 else 8),
            "layers": 2 if m <= 256 else 1}


# ----------------------------------------------------------------- inputs ----

def _codes(g, *shape):
    """E4M3 codes of normal values under the scale KV_AMAX / 448."""
    x = torch.randn(shape, generator=g, device=DEV) * (E4M3_MAX / KV_AMAX)
    return x.clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)


def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _attention_shape(case, seed):
    """The batch on the host: per sequence its new tokens, its keys and its page ids; per group
    its sequences and shared pages."""
    seqs, groups = case["seqs"], case["groups"]
    rng = random.Random(seqs * case["new"])            # ragged, but as many tokens for every seed
    new = [1 if case["new"] == 1 else rng.randint(1, case["new"]) for _ in range(seqs)]
    rng = random.Random(seed * 7919 + 1)
    own_keys = [max(n, rng.randint(1, case["suffix"])) for n in new]
    start = [seqs * g // groups for g in range(groups + 1)]
    # the first prompt is the longest
    shared = [max(1, case["prefix"] // PAGE // (g + 1)) for g in range(groups)]
    need = sum(shared) + sum(-(-n // PAGE) for n in own_keys)
    ids = rng.sample(range(need + 3), need)            # pages lie anywhere in the pool
    tables, kv_len, at = [], [], 0
    for g in range(groups):
        prefix, at = ids[at:at + shared[g]], at + shared[g]
        for s in range(start[g], start[g + 1]):
            n = -(-own_keys[s] // PAGE)
            tables.append(prefix + ids[at:at + n])
            kv_len.append(shared[g] * PAGE + own_keys[s])
            at += n
    return {"new": new, "kv_len": kv_len, "tables": tables, "group_start": start,
            "shared": shared, "pool": need + 3}


def _prepare_attention(case, seed):
    b = _attention_shape(case, seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    layers, kv, tokens = case["layers"], case["kv_heads"], sum(b["new"])
    width = max(len(t) for t in b["tables"])
    q_start = [0]
    for n in b["new"]:
        q_start.append(q_start[-1] + n)
    return {"shape": b, "tokens": tokens,
            "q": torch.randn(layers, tokens, case["heads"], D, generator=g,
                             device=DEV).to(torch.bfloat16),
            "k": _codes(g, layers, b["pool"], kv, 2, PAGE, D // 2),
            "v": _codes(g, layers, b["pool"], kv, D, PAGE),
            "scale": torch.full((layers, 2 * kv), KV_AMAX / E4M3_MAX, device=DEV),
            "table": _int32([t + [-1] * (width - len(t)) for t in b["tables"]]),
            "q_start": _int32(q_start), "kv_len": _int32(b["kv_len"]),
            "group_start": _int32(b["group_start"]), "shared": _int32(b["shared"]),
            "out": torch.zeros(layers, tokens, case["heads"], D, dtype=torch.bfloat16,
                               device=DEV)}


def _prepare_qk(case, seed):
    rng = random.Random(seed * 7919 + 2)
    g = torch.Generator(device=DEV).manual_seed(seed)
    tokens, seqs, heads, kv = case["tokens"], case["seqs"], case["heads"], case["kv_heads"]
    cuts = [0] + sorted(rng.sample(range(1, tokens), seqs - 1)) + [tokens]
    positions, slots, pages = [], [], []
    for n in (b - a for a, b in zip(cuts, cuts[1:])):
        first = rng.randint(0, 32768 - n)
        positions += range(first, first + n)
        pages.append((first, n))
    pool = tokens // PAGE + 2 * seqs + 3
    ids = rng.sample(range(pool), pool)
    for f, n in pages:
        mine = {p: ids.pop() for p in range(f // PAGE, (f + n - 1) // PAGE + 1)}
        slots += [mine[j // PAGE] * PAGE + j % PAGE for j in range(f, f + n)]
    gamma = 1 + 0.1 * torch.randn(2, D, generator=g, device=DEV)
    return {"qkv": torch.randn(tokens, heads + 2 * kv, D, generator=g,
                               device=DEV).to(torch.bfloat16),
            "q_gamma": gamma[0].to(torch.bfloat16), "k_gamma": gamma[1].to(torch.bfloat16),
            "k": _codes(g, pool, kv, 2, PAGE, D // 2), "v": _codes(g, pool, kv, D, PAGE),
            "inv": torch.full((2 * kv,), E4M3_MAX / KV_AMAX, device=DEV),
            "positions": _int32(positions), "slots": _int32(slots),
            "q": torch.zeros(tokens, heads, D, dtype=torch.bfloat16, device=DEV)}


def _prepare_pages(case, seed):
    rng = random.Random(seed * 7919 + 3)
    g = torch.Generator(device=DEV).manual_seed(seed)
    ids = rng.sample(range(case["pages"]), 2 * case["copies"])
    return {"k": _codes(g, case["layers"], case["pages"], case["kv_heads"], 2, PAGE, D // 2),
            "v": _codes(g, case["layers"], case["pages"], case["kv_heads"], D, PAGE),
            "src": ids[::2], "dst": ids[1::2]}


def _prepare_lora(case, seed):
    rng = random.Random(seed * 7919 + 4)
    g = torch.Generator(device=DEV).manual_seed(seed)
    m, n, k, r, adapters, layers = (case[f] for f in ("m", "n", "k", "rank", "adapters", "layers"))
    if m <= 256:       # decoding: a row is a request; some requests have no adapter
        ids = [rng.randrange(-1, adapters) for _ in range(m)]
    else:              # prompts: runs of rows
        cuts = [0] + sorted(rng.sample(range(1, m), 2 * adapters - 1)) + [m]
        ids = []
        for a, b in zip(cuts, cuts[1:]):
            ids += [rng.randrange(-1, adapters)] * (b - a)

    def rand(std, *shape):
        return (torch.randn(shape, generator=g, device=DEV) * std).to(torch.bfloat16)

    return {"x": rand(1.0, layers, m, k), "a": rand(k ** -0.5, layers, adapters, r, k),
            "b": rand(1.0, layers, adapters, n, r), "base": rand(1.0, layers, m, n),
            "scale": torch.rand(adapters, generator=g, device=DEV) + 0.5,
            "ids": _int32(ids), "out": torch.zeros(layers, m, n, dtype=torch.bfloat16, device=DEV)}


def prepare(case, seed):
    state = {"attention": _prepare_attention, "qk": _prepare_qk, "pages": _prepare_pages,
             "lora": _prepare_lora}[case["kind"]](case, seed)
    if case["kind"] == "qk":
        # a serving program keeps the rotation's cos and sin: [positions, 64 pairs, 2]
        state["rope"] = _rope(torch.arange(32768, device=DEV))
    if case["kind"] == "attention":
        state["index"] = _attention_index(state["shape"])
    state["case"] = case
    return state


# ------------------------------------------------------------- plain forms ----

def _rope(positions):
    freq = THETA ** (-torch.arange(0, D, 2, dtype=torch.float64, device=DEV) / D)
    angle = positions.to(torch.float64)[:, None] * freq
    return torch.stack([angle.cos(), angle.sin()], dim=-1).float()


def _values(codes):
    return codes.view(torch.float8_e4m3fn).float()


def _k_rows(pages):
    """[..., pages, kv, 2, 64, 64] -> [..., pages, kv, 64 keys, 128]."""
    return torch.cat([pages[..., 0, :, :], pages[..., 1, :, :]], dim=-1)


def _v_rows(pages):
    """[..., pages, kv, 128, 64 places] -> [..., pages, kv, 64 keys, 128]."""
    place = torch.tensor([v_place(j) for j in range(PAGE)], device=DEV)
    return pages[..., place].transpose(-1, -2)


def _attention_index(b):
    """Index tensors of the padded batches that the plain form multiplies: one of all groups'
    prefixes, one of all sequences' own keys."""
    first = [0]
    for n in b["new"]:
        first.append(first[-1] + n)
    seqs = range(len(b["new"]))
    shared = [b["shared"][g] for g in range(len(b["shared"]))
              for _ in range(b["group_start"][g], b["group_start"][g + 1])]
    limit = [b["kv_len"][s] - b["new"][s] + i + 1 for s in seqs for i in range(b["new"][s])]
    tok = [[first[a] + i for i in range(first[c] - first[a])]
           for a, c in zip(b["group_start"], b["group_start"][1:])]
    return {"limit": torch.tensor(limit, device=DEV),
            "prefix": _padded(tok, [b["tables"][a][:n] for a, n in zip(b["group_start"],
                                                                       b["shared"])],
                              [0] * len(tok), [n * PAGE for n in b["shared"]]),
            "suffix": _padded([list(range(first[s], first[s + 1])) for s in seqs],
                              [b["tables"][s][shared[s]:] for s in seqs],
                              [shared[s] * PAGE for s in seqs], b["kv_len"])}


def _padded(tokens, pages, first_key, end_key):
    """Batches of ragged token and page lists, padded with their first entries: the tokens, where
    each token's row lies, the pages, and each batch's first and end key."""
    rows, cols = max(len(t) for t in tokens), max(len(p) for p in pages)
    where = [(t, i * rows + j) for i, ts in enumerate(tokens) for j, t in enumerate(ts)]
    return {"tokens": torch.tensor([t + t[:1] * (rows - len(t)) for t in tokens], device=DEV),
            "where": torch.tensor([w for _, w in sorted(where)], device=DEV),
            "pages": torch.tensor([p + p[:1] * (cols - len(p)) for p in pages], device=DEV),
            "first": torch.tensor(first_key, device=DEV), "end": torch.tensor(end_key, device=DEV)}


def _partial_attention(q, k, v, scale, ix, limit):
    """Softmax numerator, denominator and maximum of every token over its batch's keys."""
    heads, kv = q.shape[1], k.shape[1]
    keys = k[ix["pages"]].transpose(1, 2).flatten(2, 3)            # [batch, kv, keys, 128]
    vals = v[ix["pages"]].transpose(1, 2).flatten(2, 3)
    batch, rows = ix["tokens"].shape
    qs = q[ix["tokens"]].view(batch, rows, kv, heads // kv, D).transpose(1, 2).flatten(2, 3)
    s = qs @ keys.transpose(-1, -2).contiguous()
    s = s.view(batch, kv, rows, heads // kv, -1) * scale[None, :kv, None, None, None] * D ** -0.5
    at = ix["first"][:, None] + torch.arange(keys.shape[2], device=DEV)
    seen = (at[:, None] < limit[ix["tokens"]][:, :, None]) & (at < ix["end"][:, None])[:, None]
    s = s.masked_fill(~seen[:, None, :, None], -torch.inf)
    m = s.amax(-1).clamp_min(-1e30)
    p = torch.exp(s - m[..., None])
    o = (p.flatten(2, 3) @ vals).view(batch, kv, rows, heads // kv, D)

    def of_tokens(t):
        return t.transpose(1, 2).reshape(batch * rows, heads, *t.shape[4:])[ix["where"]]

    return of_tokens(o), of_tokens(p.sum(-1)), of_tokens(m)


def _attention_plain(q, k, v, scale, index):
    q, k, v = q.float(), _k_rows(_values(k)), _v_rows(_values(v)).contiguous()
    o1, l1, m1 = _partial_attention(q, k, v, scale, index["prefix"], index["limit"])
    o2, l2, m2 = _partial_attention(q, k, v, scale, index["suffix"], index["limit"])
    m = torch.maximum(m1, m2)
    w1, w2 = torch.exp(m1 - m), torch.exp(m2 - m)
    o = (o1 * w1[..., None] + o2 * w2[..., None]) / (l1 * w1 + l2 * w2)[..., None]
    kv = k.shape[1]
    return (o * scale[kv:].repeat_interleave(q.shape[1] // kv)[None, :, None]).to(torch.bfloat16)


def _norm_rope(x, gamma, cos, sin):
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gamma.float()
    a, b = y[..., :D // 2], y[..., D // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _to_codes(x):
    return x.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)


def _qk_plain(s):
    kv, heads = s["k"].shape[1], s["q"].shape[1]
    x = s["qkv"].float()
    cos, sin = s["rope"][s["positions"].long()][:, None].unbind(-1)
    s["q"].copy_(_norm_rope(x[:, :heads], s["q_gamma"], cos, sin))
    k = _norm_rope(x[:, heads:heads + kv], s["k_gamma"], cos, sin) * s["inv"][:kv, None]
    v = x[:, heads + kv:] * s["inv"][kv:, None]
    page, key = s["slots"].long() // PAGE, s["slots"].long() % PAGE
    place = key // 4 % 4 * 16 + key // 32 * 8 + key // 16 % 2 * 4 + key % 4
    s["k"][page, :, :, key] = _to_codes(k).view(-1, kv, 2, D // 2)
    s["v"][page, :, :, place] = _to_codes(v)
    return s["q"], s["k"].view(torch.float8_e4m3fn), s["v"].view(torch.float8_e4m3fn)


def _pages_plain(s):
    s["k"][:, s["dst"]] = s["k"][:, s["src"]]
    s["v"][:, s["dst"]] = s["v"][:, s["src"]]
    return s["k"].view(torch.float8_e4m3fn), s["v"].view(torch.float8_e4m3fn)


def _lora_plain(x, a, b, base, scale, ids):
    """Every row with every adapter, the others' columns then cleared."""
    adapters, r, k = a.shape
    t = (x.float() @ a.float().view(adapters * r, k).T).view(-1, adapters, r)
    mine = ids[:, None] == torch.arange(adapters, device=DEV)
    t = torch.where(mine[:, :, None], t * scale[:, None], 0.0).view(-1, adapters * r)
    delta = t @ b.float().transpose(1, 2).reshape(adapters * r, -1)
    return (base.float() + delta).to(torch.bfloat16)


# -------------------------------------------------------------------- run ----

def _run_own(s):
    from hephaestus_amd import serve
    case = s["case"]
    if case["kind"] == "attention":
        if "plan" not in s:                                  # the step's workspaces
            s["plan"] = serve.AttentionPlan(case["seqs"], s["tokens"], case["heads"],
                                            case["kv_heads"], s["table"].shape[1],
                                            n_groups=case["groups"])
        s["plan"].update(s["q_start"], s["kv_len"], s["group_start"], s["shared"])
        for i in range(case["layers"]):
            serve.attention_pages(s["out"][i], s["q"][i], s["k"][i], s["v"][i], s["scale"][i],
                                  s["table"], s["plan"])
        return s["out"]
    if case["kind"] == "qk":
        serve.qk_norm_rope_pages(s["q"], s["qkv"], s["q_gamma"], s["k_gamma"], s["k"], s["v"],
                                 s["inv"], s["rope"], s["positions"], s["slots"], EPS)
        return s["q"], s["k"].view(torch.float8_e4m3fn), s["v"].view(torch.float8_e4m3fn)
    if case["kind"] == "pages":
        serve.copy_pages(s["k"], s["v"], s["src"], s["dst"])
        return s["k"].view(torch.float8_e4m3fn), s["v"].view(torch.float8_e4m3fn)
    if "plan" not in s:
        s["plan"] = serve.LoraPlan(case["m"], case["adapters"], case["rank"], case["k"],
                                   case["n"])
    s["plan"].update(s["ids"])
    for i in range(case["layers"]):
        serve.lora_add(s["out"][i], s["base"][i], s["x"][i], s["a"][i], s["b"][i], s["scale"],
                       s["plan"])
    return s["out"]


def run(state):
    s = state
    kind, layers = s["case"]["kind"], range(s["case"].get("layers", 1))
    if own:
        return _run_own(s)
    if kind == "attention":
        return torch.stack([_attention_plain(s["q"][i], s["k"][i], s["v"][i], s["scale"][i],
                                             s["index"]) for i in layers])
    if kind == "qk":
        return _qk_plain(s)
    if kind == "pages":
        return _pages_plain(s)
    return torch.stack([_lora_plain(s["x"][i], s["a"][i], s["b"][i], s["base"][i], s["scale"],
                                    s["ids"]) for i in layers])


# ---------------------------------------------------------- work and exact ----

def work(case):
    kind = case["kind"]
    if kind == "attention":
        b = _attention_shape(case, 1)
        shared = [n for n, a, c in zip(b["shared"], b["group_start"], b["group_start"][1:])
                  for _ in range(a, c)]
        keys = sum(b["shared"]) * PAGE + sum(n - PAGE * p for n, p in zip(b["kv_len"], shared))
        pairs = sum(n * (2 * kv - n + 1) // 2 for n, kv in zip(b["new"], b["kv_len"]))
        return {"bytes": case["layers"] * (keys * case["kv_heads"] * D * 2
                                           + sum(b["new"]) * case["heads"] * D * 4),
                "flops": case["layers"] * pairs * case["heads"] * D * 4}
    if kind == "qk":
        heads, kv, t = case["heads"], case["kv_heads"], case["tokens"]
        return {"bytes": t * (D * (2 * (heads + 2 * kv) + 2 * heads + 2 * kv) + D * 4 + 8),
                "flops": t * D * (heads + kv) * 8}
    if kind == "pages":
        return {"bytes": 2 * case["layers"] * case["copies"] * case["kv_heads"] * 2 * PAGE * D,
                "flops": 0}
    m, n, k, r = case["m"], case["n"], case["k"], case["rank"]
    used = min(case["adapters"], m)
    return {"bytes": 2 * case["layers"] * (m * k + used * r * (k + n) + 2 * m * n),
            "flops": 2 * case["layers"] * m * r * (k + n)}


def _exact_attention(s):
    b, case = s["shape"], s["case"]
    heads, kv = case["heads"], case["kv_heads"]
    place = [v_place(j) for j in range(PAGE)]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for layer in range(case["layers"]):
        k = s["k"][layer].view(torch.float8_e4m3fn)
        v = s["v"][layer].view(torch.float8_e4m3fn)
        sk, sv = s["scale"][layer].double().view(2, kv, 1, 1)
        t = 0
        for table, n, keys in zip(b["tables"], b["new"], b["kv_len"]):
            # [pages, kv, 2, 64, 64] -> [kv, keys, 128]
            ks = k[table].double().permute(1, 0, 3, 2, 4).reshape(kv, -1, D)[:, :keys] * sk
            vs = v[table].double()[..., place].permute(1, 0, 3, 2).reshape(kv, -1, D)[:, :keys] * sv
            q = s["q"][layer, t:t + n].double().view(n, kv, heads // kv, D).permute(1, 2, 0, 3)
            x = q.reshape(kv, -1, D) @ ks.transpose(1, 2).contiguous() / math.sqrt(D)
            x = x.view(kv, heads // kv, n, keys)
            later = torch.arange(keys, device=DEV) > (torch.arange(n, device=DEV) + keys - n)[:, None]
            p = torch.softmax(x.masked_fill(later, -math.inf), -1)
            o = (p.view(kv, -1, keys) @ vs).view(kv, heads // kv, n, D)
            out[layer, t:t + n] = o.permute(2, 0, 1, 3).reshape(n, heads, D)
            t += n
    return out


def _exact_qk(s):
    heads, kv = s["q"].shape[1], s["k"].shape[1]
    x = s["qkv"].double()
    x = x[:, :heads + kv]
    gamma = torch.cat([s["q_gamma"].expand(heads, D), s["k_gamma"].expand(kv, D)]).double()
    y = gamma * x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS)
    pair = torch.arange(D // 2, dtype=torch.float64, device=DEV)
    angle = s["positions"].double()[:, None, None] / torch.pow(THETA, 2 * pair / D)
    z = torch.complex(y[..., :D // 2], y[..., D // 2:]) * torch.polar(torch.ones_like(angle), angle)
    y = torch.cat([z.real, z.imag], -1)
    # cached values: the codes' own, where no rounding to codes is counted
    k, v = (s[f].view(torch.float8_e4m3fn).double() for f in ("k", "v"))
    page, key = s["slots"].long() // PAGE, s["slots"].long() % PAGE
    where = torch.tensor([v_place(j) for j in range(PAGE)], device=DEV)[key]
    new_k = (y[:, heads:] * s["inv"].double()[:kv, None]).clamp(-E4M3_MAX, E4M3_MAX)
    new_v = (s["qkv"][:, heads + kv:].double() * s["inv"].double()[kv:, None])
    k[page, :, :, key] = new_k.view(-1, kv, 2, D // 2)
    v[page, :, :, where] = new_v.clamp(-E4M3_MAX, E4M3_MAX)
    return y[:, :heads], k, v


def _exact_lora(s):
    out = s["base"].double()
    for i in range(s["case"]["layers"]):
        for a in range(s["case"]["adapters"]):
            rows = (s["ids"] == a).nonzero().flatten()
            t = s["x"][i, rows].double() @ s["a"][i, a].double().T
            out[i, rows] += s["scale"][a].double() * (t @ s["b"][i, a].double().T)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attention":
        return _exact_attention(s)
    if case["kind"] == "qk":
        return _exact_qk(s)
    if case["kind"] == "lora":
        return _exact_lora(s)
    source = list(range(case["pages"]))
    for a, b in zip(s["src"], s["dst"]):
        source[b] = a
    return tuple(s[f].view(torch.float8_e4m3fn)[:, source].double() for f in ("k", "v"))
