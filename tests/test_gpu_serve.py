"""The batched serving ops against plain float64 restatements.

Tolerances are counted from the roundings each op documents (half a step is
2^-8 relative in bf16, 2^-4 in E4M3) plus the f32 sums' own bound: n terms
summed in f32 in any order are within n * 2^-24 of the sum of magnitudes.
"""
import math
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from hephaestus_amd import _lib as L
from hephaestus_amd import decode as DEC
from hephaestus_amd import serve as S
from hephaestus_amd.kernels import HephError
from hephaestus_amd.loader import Qwen3Config

pytestmark = pytest.mark.gpu

D, PAGE = 128, 64
E, B16, F32 = 2.0 ** -4, 2.0 ** -8, 2.0 ** -24      # half steps


def f64(t):
    if t.dtype in (torch.uint8, torch.float8_e4m3fn):
        t = t.view(torch.float8_e4m3fn).cpu().float()
    return t.detach().cpu().double()


def codes(g, *shape):
    return (torch.randn(shape, generator=g, device="cuda") * 90).clamp(-448, 448).to(
        torch.float8_e4m3fn).view(torch.uint8)


def k_rows(pages):
    """[n, kv, 2, 64, 64] codes -> [n * 64, kv, 128] values, float64."""
    p = f64(pages)
    return p.permute(0, 3, 1, 2, 4).reshape(p.shape[0] * PAGE, p.shape[1], D)


def v_rows(pages):
    p = f64(pages)[..., [S.v_place(j) for j in range(PAGE)]]
    return p.permute(0, 3, 1, 2).reshape(p.shape[0] * PAGE, p.shape[1], D)


# ------------------------------------------------------------ norm + rope ----

def norm_rope(x, gamma, pos, eps, theta=1e6):
    """float64 [T, heads, 128]."""
    y = gamma * x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    a = pos.double()[:, None] * theta ** (-torch.arange(0, D, 2).double() / D)
    c, s = a.cos()[:, None], a.sin()[:, None]
    lo, hi = y[..., :64], y[..., 64:]
    return torch.cat([lo * c - hi * s, hi * c + lo * s], -1)


def qk_case(T, H, KV, seed, n_pos=5000, pad=0, in_place=False, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    wide = (H + 2 * KV) * D + pad
    buf = (torch.randn(T, wide, generator=g, device="cuda") * scale).to(torch.bfloat16)
    qkv = buf[:, :(H + 2 * KV) * D].unflatten(1, (H + 2 * KV, D))
    gam = (1 + 0.1 * torch.randn(2, D, generator=g, device="cuda")).to(torch.bfloat16)
    n_pages = T // 16 + 3
    k, v = codes(g, n_pages, KV, 2, PAGE, 64), codes(g, n_pages, KV, D, PAGE)
    inv = torch.rand(2 * KV, generator=g, device="cuda") * 100 + 30
    pos = torch.randint(0, n_pos, (T,), generator=g, device="cuda", dtype=torch.int32)
    slot = torch.randperm(n_pages * PAGE, generator=g, device="cuda")[:T].int()
    q = qkv[:, :H] if in_place else torch.zeros(T, H, D, dtype=torch.bfloat16, device="cuda")
    return dict(qkv=qkv, gam=gam, k=k, v=v, inv=inv, pos=pos, slot=slot, q=q, n_pos=n_pos)


def check_qk(c, H, KV, eps=1e-6):
    T = c["qkv"].shape[0]
    x, k0, v0, q0 = f64(c["qkv"]).clone(), c["k"].clone(), c["v"].clone(), f64(c["q"]).clone()
    rope = S.rope_table_f32(c["n_pos"])
    S.qk_norm_rope_pages(c["q"], c["qkv"], c["gam"][0], c["gam"][1], c["k"], c["v"], c["inv"],
                         rope, c["pos"], c["slot"], eps)
    torch.cuda.synchronize()
    gam, inv, pos, slot = f64(c["gam"]), f64(c["inv"]), c["pos"].cpu().long(), c["slot"].cpu().long()
    live = (pos >= 0) & (pos < c["n_pos"])
    at = torch.where(live, pos, 0)
    # f32 inside: the norm's factor, table entries and four products, each within
    # a few 2^-24 of the pair's magnitude
    q = norm_rope(x[:, :H], gam[0], at, eps)
    slop = 32 * F32 * q.abs().amax(-1, keepdim=True) * 2
    got = f64(c["q"])
    assert ((got - q).abs() <= B16 * q.abs() + slop)[live].all()
    assert torch.equal(got[~live], q0[~live])
    cached = live & (slot >= 0) & (slot < k0.shape[0] * PAGE)
    kk = norm_rope(x[:, H:H + KV], gam[1], at, eps) * inv[:KV, None]
    vv = x[:, H + KV:] * inv[KV:, None]
    want_k, want_v = k_rows(k0), v_rows(v0)
    got_k, got_v = k_rows(c["k"]), v_rows(c["v"])
    for got, want, val in ((got_k, want_k, kk), (got_v, want_v, vv)):
        new = got[slot[cached]]
        val = val.clamp(-448, 448)[cached]
        tol = torch.maximum(E * val.abs(), torch.tensor(2.0 ** -10).double())
        tol = tol + 64 * F32 * val.abs().amax(-1, keepdim=True)
        assert ((new - val).abs() <= tol).all()
        rest = torch.ones(got.shape[0], dtype=torch.bool)
        rest[slot[cached]] = False
        assert torch.equal(got[rest], want[rest])          # every other key as it was
    # V codes are of one product: equal to torch's rounding of it in f32
    code = (x[:, H + KV:].float() * c["inv"].cpu()[KV:, None]).clamp(-448, 448)
    assert torch.equal(got_v[slot[cached]], code.to(torch.float8_e4m3fn).double()[cached])


@pytest.mark.parametrize("T,H,KV", [(1, 32, 8), (3, 8, 8), (17, 16, 2), (64, 40, 8), (130, 5, 1),
                                    (1000, 32, 8)])
def test_qk_norm_rope_pages(T, H, KV):
    check_qk(qk_case(T, H, KV, seed=T), H, KV)


@pytest.mark.parametrize("pad,in_place", [(0, True), (8, False), (264, True)])
def test_qk_strides_and_in_place(pad, in_place):
    check_qk(qk_case(33, 16, 4, seed=5, pad=pad, in_place=in_place), 16, 4)


def test_qk_runs_of_slots():
    # prompts: consecutive slots from any start, across pages, odd ends
    for first, n in ((0, 64), (64, 200), (5, 59), (63, 2), (60, 133), (17, 16), (16, 48)):
        c = qk_case(n, 8, 4, seed=first + n)
        c["slot"] = torch.arange(first, first + n, dtype=torch.int32, device="cuda")
        c["k"] = c["k"].new_zeros(6, *c["k"].shape[1:]).copy_(c["k"][:1])
        c["v"] = c["v"].new_zeros(6, *c["v"].shape[1:]).copy_(c["v"][:1])
        check_qk(c, 8, 4)
    # two prompts that meet in one call, the second in lower pages
    c = qk_case(100, 8, 4, seed=9)
    c["slot"] = torch.cat([torch.arange(140, 190), torch.arange(10, 60)]).int().cuda()
    check_qk(c, 8, 4)
    # descending slots, and runs with a hole
    c = qk_case(64, 8, 4, seed=10)
    c["slot"] = torch.arange(127, 63, -1, dtype=torch.int32, device="cuda")
    check_qk(c, 8, 4)
    c = qk_case(63, 8, 4, seed=11)
    c["slot"] = torch.cat([torch.arange(64, 90), torch.arange(91, 128)]).int().cuda()
    check_qk(c, 8, 4)


def test_qk_long_batches_in_runs():
    # windows of 64 tokens: prompts from any slot, some tokens left out, and the bytes
    # of a batch alike however its tokens are cut into calls
    for first in (0, 64, 37, 3):
        c = qk_case(777, 6, 3, seed=first)
        c["slot"] = torch.arange(first, first + 777, dtype=torch.int32, device="cuda")
        c["pos"][[0, 100, 101, 640]] = -1
        c["slot"][[7, 63, 64, 700]] = -1
        check_qk(c, 6, 3)
    c = qk_case(700, 8, 4, seed=20)
    a = torch.arange(2000, 2350)
    c["slot"] = torch.cat([a, torch.randperm(1800)[:200], torch.arange(1999, 1849, -1)]).int().cuda()
    check_qk(c, 8, 4)
    whole, parts = qk_case(600, 8, 4, seed=21), qk_case(600, 8, 4, seed=21)
    for d in (whole, parts):
        d["slot"] = torch.arange(5, 605, dtype=torch.int32, device="cuda")
    check_qk(whole, 8, 4)
    rope = S.rope_table_f32(whole["n_pos"])
    for lo in range(0, 600, 50):
        s = slice(lo, lo + 50)
        S.qk_norm_rope_pages(parts["q"][s], parts["qkv"][s], parts["gam"][0], parts["gam"][1],
                             parts["k"], parts["v"], parts["inv"], rope, parts["pos"][s].clone(),
                             parts["slot"][s].clone())
    torch.cuda.synchronize()
    assert torch.equal(whole["k"], parts["k"]) and torch.equal(whole["v"], parts["v"])
    assert torch.equal(whole["q"], parts["q"])


def test_qk_padding_rows():
    c = qk_case(40, 8, 4, seed=3)
    c["pos"][[0, 7, 39]] = torch.tensor([-1, 5000, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    c["slot"][[1, 8, 20]] = torch.tensor([-1, 2 ** 31 - 1, c["k"].shape[0] * PAGE],
                                         dtype=torch.int32, device="cuda")
    check_qk(c, 8, 4)
    # inside a run of slots too
    c = qk_case(64, 8, 4, seed=4)
    c["slot"] = torch.arange(64, 128, dtype=torch.int32, device="cuda")
    c["pos"][[5, 33]] = -1
    c["slot"][[9, 60]] = -5
    check_qk(c, 8, 4)


def test_qk_far_positions_and_extreme_values():
    c = qk_case(20, 8, 4, seed=6, n_pos=262144)
    c["pos"][:3] = torch.tensor([262143, 0, 200001], dtype=torch.int32, device="cuda")
    check_qk(c, 8, 4)
    for scale in (1e-18, 1e15):                   # sums of squares near f32's ends
        check_qk(qk_case(9, 8, 4, seed=7, scale=scale), 8, 4)
    c = qk_case(9, 8, 4, seed=8)
    c["qkv"][2] = 0
    check_qk(c, 8, 4)


def test_qk_nan_and_infinities():
    # a NaN of k or v becomes the code of -448 in the cache, an infinite v the largest code;
    # a NaN in a head of k reaches all of it (its norm), one in v no other element
    for T in (9, 600):                                     # both windows of V
        c = qk_case(T, 8, 4, seed=T)
        x = c["qkv"]
        x[1, 8 + 2, 77] = float("nan")
        x[2, 12 + 1, 5], x[2, 12 + 1, 6], x[2, 12 + 1, 7] = float("nan"), float("inf"), -float("inf")
        x[3, 4, 0] = float("nan")
        rope = S.rope_table_f32(c["n_pos"])
        clean = dict(c, k=c["k"].clone(), v=c["v"].clone(), q=c["q"].clone(), qkv=x.nan_to_num(0, 1, -1))
        for d in (c, clean):
            S.qk_norm_rope_pages(d["q"], d["qkv"], *d["gam"], d["k"], d["v"], d["inv"], rope, d["pos"],
                                 d["slot"])
        torch.cuda.synchronize()
        want_k, want_v, want_q = k_rows(clean["k"]), v_rows(clean["v"]), f64(clean["q"])
        slot = c["slot"].cpu().long()
        want_k[slot[1], 2] = -448
        want_v[slot[2], 1, 5:8] = torch.tensor([-448.0, 448.0, -448.0]).double()
        assert torch.equal(k_rows(c["k"]), want_k) and torch.equal(v_rows(c["v"]), want_v)
        got = f64(c["q"])
        assert torch.isnan(got[3, 4]).all()
        got[3, 4] = want_q[3, 4]
        assert torch.equal(got, want_q)


def test_rope_table_f32():
    t = f64(S.rope_table_f32(4100, 5e6))
    a = torch.arange(4100).double()[:, None] * 5e6 ** (-torch.arange(0, D, 2).double() / D)
    assert (t[..., 0] - a.cos()).abs().max() <= 2.0 ** -24
    assert (t[..., 1] - a.sin()).abs().max() <= 2.0 ** -24


# --------------------------------------------------------------- attention ----

def batch(new, own, shared=(), group_start=(), seed=0, H=32, KV=8, bad=(), garbage=True,
          extra_tokens=0, scale_q=1.0):
    """Sequences with new[s] tokens and own[s] keys of their own behind their
    group's shared[g] pages. Unused keys of the pools hold NaN codes."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = len(new)
    of = [next((i for i, a in enumerate(group_start[:-1]) if a <= s < group_start[i + 1]), -1)
          for s in range(n)]
    kv_len = [own[s] + (shared[of[s]] * PAGE if of[s] >= 0 else 0) for s in range(n)]
    need = sum(shared) + sum(-(-o // PAGE) for o in own)
    ids = torch.randperm(need + 2, generator=torch.Generator().manual_seed(seed)).tolist()
    prefix = [[ids.pop() for _ in range(p)] for p in shared]
    tables = [(list(prefix[of[s]]) if of[s] >= 0 else []) +
              [ids.pop() for _ in range(-(-own[s] // PAGE))] for s in range(n)]
    k, v = codes(g, need + 2, KV, 2, PAGE, 64), codes(g, need + 2, KV, D, PAGE)
    if garbage:
        used = torch.zeros(need + 2, PAGE, dtype=torch.bool)
        for s in range(n):
            for j in range(kv_len[s]):
                used[tables[s][j // PAGE], j % PAGE] = True
        k.permute(0, 3, 1, 2, 4)[~used.cuda()] = 0x7F
        place = [S.v_place(j) for j in range(PAGE)]
        vk = v[..., place]
        vk.permute(0, 3, 1, 2)[~used.cuda()] = 0xFF
        v[..., place] = vk
    width = max(1, max(len(t) for t in tables)) + 1
    table = torch.full((n, width), -1, dtype=torch.int32)
    for s, t in enumerate(tables):
        table[s, :len(t)] = torch.tensor(t, dtype=torch.int32)
    for s, p, val in bad:
        table[s, p] = val
    T = sum(new) + extra_tokens
    q = (torch.randn(T, H, D, generator=g, device="cuda") * scale_q).to(torch.bfloat16)
    return dict(new=new, kv_len=kv_len, table=table.cuda(), k=k, v=v, q=q, H=H, KV=KV, T=T,
                scale=(torch.rand(2 * KV, generator=g, device="cuda") + 0.5) / 90,
                q_start=torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32).cuda(),
                lens=torch.tensor(kv_len, dtype=torch.int32).cuda(),
                group_start=torch.tensor(group_start, dtype=torch.int32).cuda() if shared else None,
                shared=torch.tensor(shared, dtype=torch.int32).cuda() if shared else None)


def make_plan(b):
    plan = S.AttentionPlan(len(b["new"]), b["T"], b["H"], b["KV"], b["table"].shape[1],
                           n_groups=0 if b["shared"] is None else b["shared"].numel())
    plan.update(b["q_start"], b["lens"], b["group_start"], b["shared"])
    return plan


def run_attention(b, plan=None, fill=7.0):
    out = torch.full((b["T"], b["H"], D), fill, dtype=torch.bfloat16, device="cuda")
    S.attention_pages(out, b["q"], b["k"], b["v"], b["scale"], b["table"], plan or make_plan(b))
    return out


def check_attention(b, out, tokens=None):
    """All rows of out, or those of some tokens."""
    H, KV, G = b["H"], b["KV"], b["H"] // b["KV"]
    table, n_pages = b["table"].cpu(), b["k"].shape[0]
    sk, sv = f64(b["scale"])[:KV], f64(b["scale"])[KV:]
    got, t = f64(out), 0
    for s, n in enumerate(b["new"]):
        total = b["kv_len"][s]
        ids = table[s, :-(-total // PAGE)].long()
        ok = ((ids >= 0) & (ids < n_pages)).repeat_interleave(PAGE)[:total]
        ids = ids.clamp(0, n_pages - 1).cuda()
        ks = k_rows(b["k"][ids])[:total] * sk[:, None]
        vs = v_rows(b["v"][ids])[:total] * sv[:, None]
        for i in range(n):
            if tokens is not None and t not in tokens:
                t += 1
                continue
            see = ok & (torch.arange(total) <= total - n + i)
            q = f64(b["q"][t]).view(KV, G, D)
            x = torch.einsum("kgd,jkd->kgj", q, ks[see]) / math.sqrt(D)
            mag = torch.einsum("kgd,jkd->kgj", q.abs(), ks[see].abs()) / math.sqrt(D)
            if see.any():
                p = torch.softmax(x, -1)
                want = torch.einsum("kgj,jkd->kgd", p, vs[see]).reshape(H, D)
                weight = torch.einsum("kgj,jkd->kgd", p, vs[see].abs()).reshape(H, D)
                # a probability is off by its rounding to bf16 and by its score's f32
                # sum (and exp2's argument), numerator and denominator; then out's own rounding
                e = 2 * (140 * F32 * mag.amax(-1) + 2.0 ** -20).view(H, 1)
                tol = (B16 + e) * weight + B16 * want.abs() + (B16 * B16) * weight
            else:
                want, tol = torch.zeros(H, D).double(), torch.zeros(H, D).double()
            off = (got[t] - want).abs()
            assert (off <= tol).all(), (s, i, (off - tol).max().item())
            t += 1
    assert (got[t:] == 7.0).all()           # rows of no sequence stay as they were


@pytest.mark.parametrize("new,own", [
    ([1], [1]), ([1], [64]), ([1], [65]), ([1, 1, 1], [63, 1, 200]), ([1] * 5, [1, 64, 65, 128, 700]),
    ([1], [3000]), ([5, 1, 3], [5, 9, 70]), ([17], [17]), ([64], [300]), ([130, 1, 33], [130, 90, 64]),
    ([300], [300]),
])
def test_attention_no_groups(new, own):
    b = batch(new, own, seed=len(new) + own[0])
    check_attention(b, run_attention(b))


@pytest.mark.parametrize("H,KV", [(8, 8), (16, 8), (40, 8), (16, 2), (7, 1), (32, 1), (64, 1), (96, 4)])
def test_attention_head_layouts(H, KV):
    b = batch([1, 1, 4, 1], [70, 64, 100, 1], shared=[3], group_start=[0, 4], seed=H, H=H, KV=KV)
    check_attention(b, run_attention(b))
    b = batch([20, 1], [40, 100], seed=H + 1, H=H, KV=KV)
    check_attention(b, run_attention(b))


@pytest.mark.parametrize("new,own,shared,group_start", [
    ([1] * 4, [1, 30, 64, 100], [5], [0, 4]),
    ([1] * 9, [10, 20, 30, 40, 50, 60, 70, 80, 90], [2, 7, 1], [0, 4, 5, 9]),
    ([1] * 6, [10, 20, 30, 40, 500, 60], [4, 3], [1, 3, 5]),       # sequences in no group
    ([1] * 40, list(range(1, 41)), [20], [0, 40]),
    ([3, 40, 1, 70], [3, 45, 200, 100], [6], [0, 4]),
    ([1, 1], [5, 6], [0, 3], [0, 1, 2]),                           # a group that shares nothing
    ([1, 1], [5, 6], [3, 2], [0, 0, 2]),                           # a group of no sequence
    ([2, 1], [5, 6], [40], [0, 2]),
    ([1, 100, 1, 1], [3, 120, 70, 5], [25], [0, 4]),               # shared beside a long prompt
    ([1, 100, 1, 90], [3, 120, 70, 95], [4], [0, 4]),              # not shared for two prompts' sake
])
def test_attention_shared_prefix(new, own, shared, group_start):
    b = batch(new, own, shared, group_start, seed=sum(own))
    # the kv_len of sequences in no group has no prefix
    check_attention(b, run_attention(b))


def prefix_rows(plan):
    """Rows of the plan's units that work on a shared prefix."""
    words = plan.plan.cpu().numpy().view(np.int32)
    n_units, first = int(words[7]), 12 + 8 * plan.n_tok
    units = words[first:first + 8 * n_units].reshape(n_units, 8)      # rows: 3, prefix: 7
    return int(units[units[:, 7] != 0, 3].sum()) if n_units else 0


@pytest.mark.parametrize("n,new,H,KV,shared,planned", [
    (30, 1, 64, 1, 40, True),          # one token of 64 heads a kv head
    (6, 16, 32, 8, 40, True), (9, 8, 16, 2, 70, True),
    (30, 1, 64, 1, 31, False), (4, 16, 32, 8, 40, False),       # too short, too few
    (9, 4, 32, 8, 3, True),            # less than 64 rows: always
    (30, 17, 16, 4, 40, False),        # more than 64
])
def test_attention_sequences_of_64_rows_share_a_long_prefix(n, new, H, KV, shared, planned):
    b = batch([new] * n, [new + 7 * i % 90 for i in range(n)], [shared], [0, n], seed=n + new, H=H, KV=KV)
    plan = make_plan(b)
    assert prefix_rows(plan) % (n * new * H // KV) == 0 and (prefix_rows(plan) > 0) == planned
    rng = np.random.default_rng(n)
    check_attention(b, run_attention(b, plan), tokens=set(rng.integers(0, b["T"], 25).tolist()))


@pytest.mark.parametrize("scaled", [False, True])
@pytest.mark.parametrize("n,prefixes,H,KV", [(12, 1, 32, 8), (13, 2, 32, 8), (3, 1, 8, 8), (700, 3, 4, 1), (1024, 1, 4, 1)])
def test_attention_pages_that_recur(scaled, n, prefixes, H, KV):
    """Sequences that share their first pages without saying so read them through the caches, and
    those with copies of their own past them: the same bits."""
    b = batch([1] * n, [130 + i % 70 for i in range(n)], seed=n, H=H, KV=KV, garbage=False)
    shared = b["table"].clone()
    for s in range(n):
        shared[s, :2] = b["table"][s % prefixes, :2]
    ids = shared[:, :2].flatten().long()
    own = b["table"][:, :2].flatten().long()
    b["page_scale"] = torch.full((b["k"].shape[0], 2 * KV), 2.0 ** -7, device="cuda")
    for t in ("k", "v"):
        b[t][own] = b[t][ids]
    outs = []
    for table in (b["table"], shared):
        out = torch.zeros(b["T"], H, D, dtype=torch.bfloat16, device="cuda")
        if scaled:
            S.attention_pages_scaled(out, b["q"], b["k"], b["v"], b["page_scale"], table, make_plan(b))
        else:
            S.attention_pages(out, b["q"], b["k"], b["v"], b["scale"], table, make_plan(b))
        outs.append(out)
    assert torch.equal(*outs)
    if not scaled:
        check_attention(b, outs[0], tokens=set(range(0, n, max(n // 10, 1))))


def test_attention_shared_equals_unshared():
    # what is shared changes where keys are summed, not what is summed
    b = batch([1] * 12, [30 * i + 1 for i in range(12)], [9], [0, 12], seed=77)
    check_attention(b, run_attention(b))
    b["shared"] = b["group_start"] = None
    check_attention(b, run_attention(b))


def test_attention_shared_beyond_own_keys():
    # shared_pages past a sequence's keys: its own limit holds
    b = batch([1, 1, 2], [64 * 3, 64 * 2 + 5, 64 * 3], seed=5)
    for s in (1, 2):
        b["table"][s, :2] = b["table"][0, :2]
    b["table"][2, 2] = b["table"][0, 2]
    b["group_start"] = torch.tensor([0, 3], dtype=torch.int32).cuda()
    b["shared"] = torch.tensor([3], dtype=torch.int32).cuda()
    b["table"][1, 2] = b["table"][0, 2]
    check_attention(b, run_attention(b))
    b["shared"][0] = 1000                       # past the table
    check_attention(b, run_attention(b))


def test_attention_bad_metadata():
    # page ids outside the pool are left out; lengths are clamped
    b = batch([1, 1, 3], [300, 100, 80], bad=[(0, 1, -1), (0, 3, 10 ** 6), (1, 0, -7), (2, 0, 2 ** 31 - 1)],
              seed=3, garbage=False)
    check_attention(b, run_attention(b))
    b = batch([1, 1], [5, 64], bad=[(0, 0, -1), (1, 0, 99)], seed=4, garbage=False)
    check_attention(b, run_attention(b))                            # nothing left: zero rows
    # no keys; fewer keys than tokens; a sequence without tokens
    b = batch([1, 4, 2, 0], [1, 10, 70, 40], seed=5, garbage=False)
    b["kv_len"] = [0, 2, 70, 40]
    b["lens"] = torch.tensor([-3, 2, 70, 40], dtype=torch.int32).cuda()
    out = run_attention(b)
    assert (out[0] == 0).all() and (out[1:3] == 0).all()
    check_attention(dict(b, new=[2], kv_len=[2], table=b["table"][1:2], q=b["q"][3:5], T=2),
                    out[3:5])
    # a length past the table
    b = batch([1], [64 * 3], seed=6, garbage=False)
    b["table"] = b["table"][:, :3].contiguous()
    b["lens"][0] = 2 ** 31 - 1
    check_attention(b, run_attention(b))
    # q_start past the rows and falling
    b = batch([1, 1, 1], [50, 60, 70], seed=7, garbage=False)
    b["q_start"] = torch.tensor([0, 1, 0, 10 ** 6], dtype=torch.int32).cuda()
    plan = make_plan(b)
    run_attention(b, plan)
    torch.cuda.synchronize()


def same_pages(n_seqs, new, keys, H, KV, seed):
    """n_seqs sequences on the same pages, each with `new` tokens: long runs in a small pool."""
    b = batch([new], [keys], seed=seed, H=H, KV=KV, garbage=False)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    T = n_seqs * new
    b.update(new=[new] * n_seqs, kv_len=[keys] * n_seqs, table=b["table"].repeat(n_seqs, 1), T=T,
             q=torch.randn(T, H, D, generator=g, device="cuda").to(torch.bfloat16),
             q_start=(torch.arange(n_seqs + 1) * new).int().cuda(),
             lens=torch.full((n_seqs,), keys, dtype=torch.int32, device="cuda"))
    return b


def test_attention_units_of_more_than_64_pages():
    # narrow: 40 sequences in the 64 slots of a kv head, 130 pages each
    b = same_pages(40, 1, 64 * 130 - 7, 8, 8, seed=30)
    b["table"][3, 70] = -1                               # a page left out behind the first 64
    check_attention(b, run_attention(b), tokens=[0, 3, 39])
    # wide: nine tiles in the eight slots, eight whole and the last one cut
    b = same_pages(3, 300, 64 * 150 - 20, 64, 64, seed=31)
    b["table"][1, [0, 65, 149]] = torch.tensor([-1, 10 ** 6, -7], dtype=torch.int32, device="cuda")
    check_attention(b, run_attention(b), tokens=[0, 127, 128, 299, 300, 555, 599, 600, 899])


@pytest.mark.parametrize("new,H", [(1, 2), (1, 40), (90, 2)])
def test_attention_longest_sequences(new, H):
    # as many keys as an op takes: units of 64 pages and more, 64 of them a row
    keys = L.ATTN_MAX_KEYS
    b = batch([new, 1], [keys, 2], seed=41 + new, H=H, KV=1, garbage=False)
    b["table"] = b["table"][:, :keys // PAGE].contiguous()
    check_attention(b, run_attention(b), tokens=[0, new - 1, new])


def test_attention_wide_tiles_split_over_pages():
    # few tiles, long runs: units of a tile meet again in the merge
    for new, keys, H, KV in ((128, 64 * 40, 8, 2), (65, 64 * 33 + 1, 4, 4), (40, 5000, 28, 4)):
        b = batch([new, 1], [keys, 700], seed=new, H=H, KV=KV)
        check_attention(b, run_attention(b), tokens=[0, 1, new // 2, new - 1, new])


def test_attention_nan_and_bad_pages_in_wide_tiles():
    # a NaN in V behind one tile's edge, in a page that the run's other rows see, and
    # beside pages left out
    b = batch([150], [64 * 80], seed=33, H=8, KV=2)
    edges = []
    for key, dim in ((64 * 80 - 149, 5), (64 * 80 - 100, 77), (64 * 80 - 2, 127)):
        page = int(b["table"][0, key // PAGE])
        b["v"][page, 1, dim, S.v_place(key % PAGE)] = 0xFF
        edges.append((key - (64 * 80 - 150), dim))
    for p in (2, 66):
        b["table"][0, p] = -1
    out = run_attention(b).float()
    t = torch.arange(150, device="cuda")
    nan = torch.zeros(150, 8, D, dtype=torch.bool, device="cuda")
    for first, dim in edges:
        nan[t >= first, 4:, dim] = True
    assert torch.equal(torch.isnan(out), nan)
    for key, dim in ((64 * 80 - 149, 5), (64 * 80 - 100, 77), (64 * 80 - 2, 127)):
        b["v"][int(b["table"][0, key // PAGE]), 1, dim, S.v_place(key % PAGE)] = 0
    # (a code in place of the NaN: only rows that do not see it are compared)
    want = run_attention(b).float()
    assert torch.equal(out[~nan], want[~nan])
    check_attention(b, run_attention(b), tokens=[0, 60, 149])
    # a NaN key reaches all dims of the heads of its kv head, where it is seen
    key = 64 * 80 - 50
    b["k"][int(b["table"][0, key // PAGE]), 0, 1, key % PAGE, 3] = 0x7F
    out = run_attention(b)
    assert torch.isnan(out[100:, :4]).all() and torch.isfinite(out[:100]).all()
    assert torch.isfinite(out[100:, 4:]).all()


@pytest.mark.parametrize("n,G", [(1024, 1), (1024, 1024), (333, 70)])
def test_attention_many_sequences(n, G):
    rng = np.random.default_rng(n + G)
    own = [int(x) for x in rng.integers(1, 90, n)]
    cuts = sorted(int(x) for x in rng.integers(0, n + 1, G - 1))
    group_start = [0] + cuts + [n]
    shared = [int(x) for x in rng.integers(0, 4, G)]
    new = [min(o, int(x)) for o, x in zip(own, rng.integers(1, 4, n))]
    b = batch(new, own, shared, group_start, seed=n, H=4, KV=1)
    check_attention(b, run_attention(b), tokens=set(rng.integers(0, b["T"], 150).tolist()))


def test_attention_falling_starts_stay_in_bounds():
    # every second sequence has all the tokens, many times the rows that the plan was sized for
    b = batch([1] * 64 + [0] * 64, [64 * 3] * 128, seed=35, H=64, KV=1, garbage=False)
    b["q_start"] = torch.tensor([0, 64] * 64 + [0], dtype=torch.int32).cuda()
    plan = make_plan(b)
    guard = plan.ws.clone()
    extra = torch.full((1 << 20,), 0x5A, dtype=torch.uint8, device="cuda")
    plan.ws = torch.cat([guard, extra])
    kept, plan.plan = plan.plan, torch.cat([plan.plan, extra])
    S._bind(plan)
    plan.update(b["q_start"], b["lens"])
    run_attention(b, plan)
    torch.cuda.synchronize()
    assert (plan.ws[guard.numel():] == 0x5A).all() and (plan.plan[kept.numel():] == 0x5A).all()


def test_attention_pools_past_32_bits():
    # the last pages of pools of 5 GiB each, through all the ops that address them
    KV, n_pages = 8, (5 << 30) // (8 * 8192)
    k = torch.empty(1, n_pages, KV, 2, PAGE, 64, dtype=torch.uint8, device="cuda")
    v = torch.empty(1, n_pages, KV, D, PAGE, dtype=torch.uint8, device="cuda")
    small = batch([1, 40], [300, 200], seed=36, H=32, KV=KV, garbage=False)
    used = small["k"].shape[0]
    at = n_pages - used
    k[0, at:], v[0, at:] = small["k"], small["v"]
    far = dict(small, k=k[0], v=v[0], table=torch.where(small["table"] < 0, small["table"], small["table"] + at))
    assert torch.equal(run_attention(far), run_attention(small))
    S.copy_pages(k, v, list(range(at, n_pages)), list(range(used)))
    assert torch.equal(k[0, :used], small["k"]) and torch.equal(v[0, :used], small["v"])
    S.copy_pages(k, v, list(range(used)), list(range(at - used, at)))
    assert torch.equal(k[0, at - used:at], small["k"]) and torch.equal(v[0, at - used:at], small["v"])
    for T in (5, 600):
        c = qk_case(T, 32, KV, seed=37)
        lo = c["k"].shape[0]
        rope = S.rope_table_f32(c["n_pos"])
        for kk, vv, base in ((c["k"], c["v"], 0), (k[0], v[0], n_pages - lo)):
            kk[base:base + lo], vv[base:base + lo] = 0, 0
            S.qk_norm_rope_pages(c["q"], c["qkv"], *c["gam"], kk, vv, c["inv"], rope, c["pos"],
                                 c["slot"] + base * PAGE)
        assert torch.equal(k[0, -lo:], c["k"]) and torch.equal(v[0, -lo:], c["v"])


def test_two_plans_on_two_streams_at_once():
    bs = [batch([1] * 30, [100 * i + 1 for i in range(30)], [12], [0, 30], seed=38),
          batch([200, 3], [2000, 64], seed=39)]
    want = [run_attention(b) for b in bs]
    plans = [make_plan(b) for b in bs]
    outs = [[torch.zeros_like(w) for _ in range(8)] for w in want]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in bs]
    for i in range(8):
        for b, p, o, s in zip(bs, plans, outs, streams):
            with torch.cuda.stream(s):
                p.update(b["q_start"], b["lens"], b["group_start"], b["shared"])
                S.attention_pages(o[i], b["q"], b["k"], b["v"], b["scale"], b["table"], p)
    torch.cuda.synchronize()
    for w, os in zip(want, outs):
        for o in os:
            assert torch.equal(o, w)


def test_two_graphs_share_a_plan():
    # captured apart, replayed in turn on one stream, with eager calls of the same plan between
    bs = [batch([1] * 6, own, [5], [0, 6], seed=40) for own in ([1, 64, 200, 7, 900, 65], [3] * 6)]
    bs[1]["table"] = torch.nn.functional.pad(
        bs[1]["table"], (0, bs[0]["table"].shape[1] - bs[1]["table"].shape[1]), value=-1)
    want = [run_attention(b) for b in bs]
    plan, graphs, outs = make_plan(bs[0]), [], [torch.zeros_like(w) for w in want]
    torch.cuda.synchronize()
    for b, o in zip(bs, outs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            plan.update(b["q_start"], b["lens"], b["group_start"], b["shared"])
            S.attention_pages(o, b["q"], b["k"], b["v"], b["scale"], b["table"], plan)
    for i in range(6):
        for o in outs:
            o.zero_()
        graphs[i % 2].replay()
        graphs[1 - i % 2].replay()
        if i % 3 == 0:
            plan.update(bs[0]["q_start"], bs[0]["lens"], bs[0]["group_start"], bs[0]["shared"])
            assert torch.equal(run_attention(bs[0], plan), want[0])
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)


def test_attention_rows_behind_the_last_sequence():
    b = batch([1, 5], [64, 5], [2], [0, 2], seed=9, extra_tokens=6)
    check_attention(b, run_attention(b))


def test_attention_q_rows_apart():
    b = batch([1, 3, 1], [64, 5, 400], [2], [0, 3], seed=10)
    wide = torch.randn(b["T"], b["H"] + 2 * b["KV"], D, device="cuda").to(torch.bfloat16)
    wide[:, :b["H"]] = b["q"]
    out = run_attention(b)
    b["q"] = wide[:, :b["H"]]
    got = run_attention(b)
    check_attention(b, got)
    assert torch.equal(got, out)


def test_attention_extreme_scores():
    # one key far above the rest, all scores equal, scores of +-1000
    b = batch([1, 1, 2], [500, 64, 90], [4], [0, 3], seed=11, scale_q=30.0)
    check_attention(b, run_attention(b))
    b["q"].zero_()
    check_attention(b, run_attention(b))


def test_attention_nan_stays_with_its_row():
    b = batch([1] * 4 + [6], [64, 10, 30, 100, 50], [4], [0, 5], seed=12)
    b["q"][1, 3] = float("nan")
    b["q"][7, 5, 17] = float("inf")
    out = run_attention(b)
    assert torch.isnan(out[1, 3]).all() and torch.isnan(out[7, 5]).all()
    bad = torch.zeros(b["T"], b["H"], dtype=torch.bool, device="cuda")
    bad[1, 3] = bad[7, 5] = True
    assert torch.isfinite(out[~bad]).all()
    q2 = b["q"].clone()
    q2[bad] = 0
    want = run_attention(dict(b, q=q2))
    assert torch.equal(out[~bad], want[~bad])


def test_attention_nan_value_behind_the_causal_edge():
    # a NaN code at key 40 of 50 reaches the rows that see it and no other
    b = batch([20], [50], seed=13)
    page = int(b["table"][0, 0])
    b["v"][page, :, 5, S.v_place(40)] = 0x7F
    out = run_attention(b).float()
    t_sees = torch.arange(20) + 30 >= 40
    assert torch.isnan(out[t_sees.cuda()][:, :, 5]).all()
    out[:, :, 5] = 0
    assert torch.isfinite(out).all()
    assert not torch.isnan(run_attention(b)[~t_sees.cuda()]).any()


def test_attention_graph_replay_with_other_lengths():
    b = batch([1] * 8, [100, 1, 64, 300, 5, 6, 7, 640], [6], [0, 8], seed=14)
    plan = make_plan(b)
    out = torch.full((b["T"], b["H"], D), 7.0, dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        S.attention_pages(out, b["q"], b["k"], b["v"], b["scale"], b["table"], plan)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.update(b["q_start"], b["lens"], b["group_start"], b["shared"])
        S.attention_pages(out, b["q"], b["k"], b["v"], b["scale"], b["table"], plan)
    for cut in (0, 3, 50, 0):
        kv = [max(n - cut, 6 * PAGE + 1) for n in b["kv_len"]]
        b["lens"].copy_(torch.tensor(kv, dtype=torch.int32))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        check_attention(dict(b, kv_len=kv), out)
        want = run_attention(dict(b, kv_len=kv))
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_attention_repeats_bit_for_bit():
    b = batch([1] * 33 + [40], [50 * i + 1 for i in range(33)] + [70], [20], [0, 34], seed=15)
    first = run_attention(b)
    for _ in range(3):
        assert torch.equal(run_attention(b), first)


def test_attention_other_plan_writes_nothing():
    b = batch([1, 1], [64, 70], seed=16)
    other = batch([1, 1, 1], [64, 70, 3], seed=16)
    plan, big = make_plan(b), make_plan(other)
    big.n_seqs, big.n_tok = plan.n_seqs, plan.n_tok       # misused: sizes of another plan
    out = run_attention(b, big)
    assert (out == 7.0).all()
    fresh = S.AttentionPlan(2, 2, 32, 8, b["table"].shape[1])
    assert (run_attention(b, fresh) == 7.0).all()          # no plan yet


def test_attention_matches_single_row_op():
    # one sequence, against the single-token op on the same codes
    n, H, KV = 777, 32, 8
    b = batch([1], [n], seed=17, garbage=False)
    ids = b["table"][0, :-(-n // PAGE)].long()
    kc = b["k"][ids].permute(0, 3, 1, 2, 4).reshape(-1, KV, D).contiguous()
    vr = b["v"][ids][..., [S.v_place(j) for j in range(PAGE)]].permute(0, 3, 1, 2).reshape(-1, KV, D)
    out1 = torch.empty(H * D, dtype=torch.bfloat16, device="cuda")
    DEC.attention_fp8kv(out1, b["q"].reshape(-1), kc, DEC.v_blocks(vr[:n]), b["scale"], H, KV, n)
    out2 = run_attention(b)
    # each is within its probabilities' and its own bf16 rounding of the exact result
    diff = (f64(out1).view(H, D) - f64(out2)[0]).abs()
    assert (diff <= 4 * B16 * f64(b["v"]).abs().max() * f64(b["scale"]).max()).all()
    check_attention(b, out2)


# ------------------------------------------------------------------- pages ----

@pytest.mark.parametrize("layers,KV,n_pages,n", [(1, 1, 4, 1), (3, 8, 40, 16), (2, 5, 900, 300),
                                                 (36, 8, 8, 2)])
def test_copy_pages(layers, KV, n_pages, n):
    g = torch.Generator(device="cuda").manual_seed(n)
    k = torch.randint(0, 256, (layers, n_pages, KV, 2, PAGE, 64), generator=g, device="cuda",
                      dtype=torch.uint8)
    v = torch.randint(0, 256, (layers, n_pages, KV, D, PAGE), generator=g, device="cuda",
                      dtype=torch.uint8)
    ids = torch.randperm(n_pages, generator=torch.Generator().manual_seed(n)).tolist()
    src, dst = ids[:n], ids[n:2 * n]
    src[-1] = src[0]                                       # a source may repeat
    wk, wv = k.clone(), v.clone()
    wk[:, dst], wv[:, dst] = k[:, src], v[:, src]
    S.copy_pages(k, v, src, dst)
    torch.cuda.synchronize()
    assert torch.equal(k, wk) and torch.equal(v, wv)


def test_copy_pages_captured_keeps_its_pairs():
    k = torch.arange(6, dtype=torch.uint8, device="cuda").view(1, 6, 1, 1, 1, 1).expand(
        2, 6, 1, 2, PAGE, 64).contiguous()
    v = k.reshape(2, 6, 1, D, PAGE).clone()
    graph = torch.cuda.CUDAGraph()
    src = np.array([0, 1], np.int32)
    with torch.cuda.graph(graph):
        S.copy_pages(k, v, src, [4, 5])
    src[:] = 3
    for _ in range(3):
        k[:, 4:] = 9
        graph.replay()
        torch.cuda.synchronize()
        assert k[:, :, 0, 0, 0, 0].tolist() == [[0, 1, 2, 3, 0, 1]] * 2


# -------------------------------------------------------------------- lora ----

def lora_case(M, N, K, r, A, seed, dtype=torch.bfloat16, ids=None):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(std, *shape):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(torch.bfloat16)
    if ids is None:
        ids = torch.randint(-1, A, (M,), generator=g, device="cuda", dtype=torch.int32)
    else:
        ids = torch.tensor(ids, dtype=torch.int32).cuda()
    return dict(x=rand(1.0, M, K), a=rand(K ** -0.5, A, r, K), b=rand(1.0, A, N, r), ids=ids,
                base=rand(1.0, M, N).to(dtype), scale=torch.rand(A, generator=g, device="cuda") + 0.5)


def check_lora(c, in_place=False, plan=None):
    M, K = c["x"].shape
    A, N, r = c["b"].shape
    base = c["base"].clone()
    out = c["base"].clone() if in_place else torch.full_like(base, 3.0)
    if plan is None:
        plan = S.LoraPlan(M, A, r, K, N)
        plan.update(c["ids"])
    S.lora_add(out, out if in_place else c["base"], c["x"], c["a"], c["b"], c["scale"], plan)
    torch.cuda.synchronize()
    x, a, b, ids = f64(c["x"]), f64(c["a"]), f64(c["b"]), c["ids"].cpu().long()
    has = (ids >= 0) & (ids < A)
    at = torch.where(has, ids, 0)
    want, tol = f64(base), torch.zeros(M, N).double()
    half = B16 if out.dtype == torch.bfloat16 else F32
    for m in range(M):
        if has[m]:
            i, s = at[m], f64(c["scale"])[at[m]]
            t, mag = (a[i] @ x[m]) * s, (a[i].abs() @ x[m].abs()) * s
            want[m] += b[i] @ t
            # t: its f32 sum over K, the scale, and the 16 bits kept; then the sum over 2r
            tol[m] = b[i].abs() @ (mag * (K + 2) * F32 + t.abs() * (2.0 ** -16 + (2 * r + 2) * F32))
    tol += half * want.abs() + 2 * F32 * f64(base).abs()
    tol[~has] = 0
    off = (f64(out) - want).abs()
    assert (off <= tol).all(), (off - tol).max().item()
    return out


@pytest.mark.parametrize("M,N,K,r,A", [
    (1, 16, 16, 8, 1), (1, 6144, 2560, 16, 3), (5, 2560, 4096, 16, 2), (16, 48, 80, 24, 4),
    (17, 304, 176, 40, 1), (33, 512, 2560, 64, 33), (64, 1040, 9728, 8, 7), (100, 96, 144, 128, 5),
    (257, 2560, 1024, 32, 3), (600, 272, 528, 72, 2), (1, 16, 2560, 128, 9), (300, 16, 4096, 16, 50),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_lora_add(M, N, K, r, A, dtype):
    check_lora(lora_case(M, N, K, r, A, seed=M + N, dtype=dtype))


@pytest.mark.parametrize("M,N,K,r,A", [
    (2200, 48, 272, 16, 3), (1030, 1040, 976, 24, 4096), (700, 4096, 64, 128, 1), (4096, 16, 48, 40, 2),
    (256, 528, 976, 64, 2000), (513, 6144, 4112, 8, 2),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_lora_long_batches_and_many_adapters(M, N, K, r, A, dtype):
    if A > 1000:                      # (adapters beyond the few that are used need no values)
        c = lora_case(M, 16, 16, 8, A, seed=M, dtype=dtype)
        few = lora_case(M, N, K, r, 5, seed=M, dtype=dtype)
        far = torch.tensor([0, 17, 1000, A - 2, A - 1], device="cuda")
        c["a"] = torch.zeros(A, r, K, dtype=torch.bfloat16, device="cuda").index_copy_(0, far, few["a"])
        c["b"] = torch.zeros(A, N, r, dtype=torch.bfloat16, device="cuda").index_copy_(0, far, few["b"])
        c["ids"] = torch.where(few["ids"] < 0, -1, far[few["ids"].clamp(min=0).long()].int()).contiguous()
        c["x"], c["base"] = few["x"], few["base"]
        check_lora(c)
    else:
        check_lora(lora_case(M, N, K, r, A, seed=M, dtype=dtype), in_place=True)


def test_lora_infinite_products():
    # t of one rank overflows: an infinity of b's sign there, no NaN
    c = lora_case(20, 96, 256, 16, 2, seed=9, ids=[0] * 20)
    c["x"].zero_()
    c["a"].zero_()
    c["x"][4, 9], c["a"][0, 3, 9] = 3e38, 8.0
    plan = S.LoraPlan(20, 2, 16, 256)
    plan.update(c["ids"])
    out = torch.empty_like(c["base"])
    S.lora_add(out, c["base"], c["x"], c["a"], c["b"], c["scale"], plan)
    assert torch.equal(out[4].float(), torch.sign(c["b"][0, :, 3].float()) * float("inf"))
    rest = torch.arange(20) != 4
    assert torch.equal(out[rest], c["base"][rest])


def test_lora_on_two_streams_at_once():
    cs = [lora_case(500, 512, 1024, 16, 4, seed=10), lora_case(9, 2560, 4096, 64, 3, seed=11)]
    plans, outs, want = [], [], []
    for c in cs:
        M, K = c["x"].shape
        A, N, r = c["b"].shape
        plans.append(S.LoraPlan(M, A, r, K))
        want.append(check_lora(c))
        outs.append([torch.zeros_like(want[-1]) for _ in range(8)])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    for i in range(8):
        for c, p, o, s in zip(cs, plans, outs, streams):
            with torch.cuda.stream(s):
                p.update(c["ids"])
                S.lora_add(o[i], c["base"], c["x"], c["a"], c["b"], c["scale"], p)
    torch.cuda.synchronize()
    for w, os in zip(want, outs):
        for o in os:
            assert torch.equal(o, w)


@pytest.mark.parametrize("ids", [[-1] * 20, [0] * 20, [3, -1, 7, 2 ** 31 - 1, -2 ** 31] * 4,
                                 [1] * 17 + [0] * 3])
def test_lora_ids(ids):
    check_lora(lora_case(20, 96, 256, 16, 4, seed=1, ids=ids), in_place=True)
    check_lora(lora_case(20, 96, 256, 16, 4, seed=2, ids=ids))


def test_lora_plan_serves_other_projections():
    ids = [0, 2, 2, -1, 1, 0, 2]
    c1 = lora_case(7, 96, 256, 16, 3, seed=3, ids=ids)
    c2 = lora_case(7, 512, 2560, 64, 3, seed=4, ids=ids)
    plan = S.LoraPlan(7, 3, 64, 2560)
    plan.update(c1["ids"])
    check_lora(c1, plan=plan)
    check_lora(c2, plan=plan, in_place=True)
    check_lora(c1, plan=plan)


def test_lora_graph_replay_with_other_ids():
    c = lora_case(40, 320, 512, 16, 6, seed=5)
    plan = S.LoraPlan(40, 6, 16, 512)
    out = torch.zeros_like(c["base"])
    plan.update(c["ids"])
    S.lora_add(out, c["base"], c["x"], c["a"], c["b"], c["scale"], plan)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.update(c["ids"])
        S.lora_add(out, c["base"], c["x"], c["a"], c["b"], c["scale"], plan)
    for seed in range(4):
        c["ids"].copy_(torch.randint(-1, 6, (40,), generator=torch.Generator().manual_seed(seed)))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        want = check_lora(c)
        assert torch.equal(out, want)


def test_lora_repeats_bit_for_bit_and_rows_do_not_depend_on_their_batch():
    c = lora_case(200, 512, 2560, 32, 9, seed=6)
    first = check_lora(c)
    assert torch.equal(check_lora(c), first)
    # the same rows in another order
    perm = torch.randperm(200, generator=torch.Generator().manual_seed(1)).cuda()
    d = dict(c, x=c["x"][perm].contiguous(), ids=c["ids"][perm].contiguous(),
             base=c["base"][perm].contiguous())
    assert torch.equal(check_lora(d), first[perm])


def test_lora_nan_stays_with_its_row():
    c = lora_case(20, 96, 256, 16, 2, seed=7, ids=[0] * 10 + [1] * 10)
    c["x"][3, 5] = float("nan")
    c["b"][1, 7, 2] = float("inf")
    plan = S.LoraPlan(20, 2, 16, 256)
    plan.update(c["ids"])
    out = torch.empty_like(c["base"])
    S.lora_add(out, c["base"], c["x"], c["a"], c["b"], c["scale"], plan)
    bad = torch.zeros(20, 96, dtype=torch.bool, device="cuda")
    bad[3] = True
    bad[10:, 7] = True
    assert torch.isnan(out[3]).all() and not torch.isfinite(out[10:, 7]).any()
    assert torch.isfinite(out[~bad]).all()


def test_lora_other_plan_writes_nothing():
    c = lora_case(20, 96, 256, 16, 2, seed=8)
    plan = S.LoraPlan(24, 2, 16, 256)
    plan.m = 20
    out = torch.full_like(c["base"], 3.0)
    S.lora_add(out, c["base"], c["x"], c["a"], c["b"], c["scale"], plan)
    assert (out == 3.0).all()


# ---------------------------------------------------------- the whole step ----

CFG = Qwen3Config(vocab=512, hidden=256, n_layers=2, n_heads=8, n_kv_heads=2, inter=384)


def decoder(n_pages=40, seed=0, lora=None):
    w = DEC.random_init(CFG, seed)
    kv = S.PagedKVCache(CFG, n_pages)
    kv.scale.fill_(4.0 / 448)
    kv.inv.fill_(448 / 4.0)
    return S.Qwen3BatchDecoder(w, kv, n_pos=2048, lora=lora)


def step_reference(d, history, adapter=-1):
    """Logits after the last token of one sequence, every token recomputed in
    f64 from the dequantized weights (activations and cache quantized as the
    step quantizes them)."""
    cfg, w = d.w.cfg, d.w

    def deq(fw):
        s = f64(fw.scale).repeat_interleave(128, 0).repeat_interleave(128, 1)
        return f64(fw.w) * s[:fw.w.shape[0], :fw.w.shape[1]]

    def bf(x):
        return x.float().to(torch.bfloat16).double()

    def quant(x):
        g = x.view(x.shape[0], -1, 128)
        s = g.abs().amax(-1, keepdim=True).float() / 448
        s = torch.where(s < 1e-12, torch.ones_like(s), s)
        return ((g.float() * (1 / s)).to(torch.float8_e4m3fn).double() * s.double()).view(x.shape)

    def norm(x, gamma, eps):
        return bf(f64(gamma) * bf(x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)))

    def lin(x, fw, li=None, op=None):
        y = quant(x) @ deq(fw).T
        if adapter >= 0 and li is not None and op in d.lora.layers[li]:
            a, b = d.lora.layers[li][op]
            y = y + f64(d.lora.scale)[adapter] * (x @ f64(a[adapter]).T) @ f64(b[adapter]).T
        return y

    T, H, KV = len(history), cfg.n_heads, cfg.n_kv_heads
    x = bf(deq(w.embed)[history])
    pos = torch.arange(T)
    for li, lw in enumerate(w.layers):
        qkv = bf(lin(norm(x, lw.attn_norm, cfg.eps), lw.qkv, li, "qkv")).view(T, H + 2 * KV, D)
        q = bf(norm_rope(qkv[:, :H], f64(lw.q_norm), pos, cfg.eps, cfg.theta))
        k = norm_rope(qkv[:, H:H + KV], f64(lw.k_norm), pos, cfg.eps, cfg.theta)
        s, inv = f64(d.kv.scale[li]), f64(d.kv.inv[li])
        k = (k * inv[:KV, None]).clamp(-448, 448).float().to(torch.float8_e4m3fn).double() * s[:KV, None]
        v = (qkv[:, H + KV:] * inv[KV:, None]).clamp(-448, 448).float().to(
            torch.float8_e4m3fn).double() * s[KV:, None]
        G = H // KV
        sc = torch.einsum("tkgd,jkd->kgtj", q.view(T, KV, G, D), k) / math.sqrt(D)
        sc = sc.masked_fill(pos[None, :] > pos[:, None], -math.inf)
        att = bf(torch.einsum("kgtj,jkd->tkgd", sc.softmax(-1), v).reshape(T, H * D))
        x = bf(x + lin(att, lw.o, li, "o"))
        gu = bf(lin(norm(x, lw.ffn_norm, cfg.eps), lw.gate_up, li, "gate_up"))
        gate, up = gu.chunk(2, -1)
        act = bf(bf(gate / (1 + torch.exp(-gate))) * up)
        x = bf(x + lin(act, lw.down, li, "down"))
    return (quant(norm(x[-1:], w.final_norm, cfg.eps)) @ deq(w.embed).T)[0]


def lora_weights(n_adapters=3, rank=16, seed=5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    H, I, Q, KV = CFG.hidden, CFG.inter, CFG.q_out, CFG.kv_out

    def pair(n, k):
        return tuple((torch.randn(n_adapters, *s, generator=g, device="cuda") * std).to(torch.bfloat16)
                     for s, std in (((rank, k), k ** -0.5), ((n, rank), 0.05)))
    layers = [{"qkv": pair(Q + 2 * KV, H), "o": pair(H, Q), "down": pair(H, I)},
              {"gate_up": pair(2 * I, H), "qkv": pair(Q + 2 * KV, H)}]
    return S.LoraWeights(torch.tensor([0.5, 1.0, 2.0], device="cuda"), layers)


def near(got, want):
    # W8A8 flips of single codes between two correct orders of summation: the
    # logits agree as vectors
    got, want = f64(got), want
    return ((got - want).norm() / want.norm()).item()


def test_batch_decoder_prompts_fork_decode_compact_free():
    lora = lora_weights()
    d = decoder(lora=lora)
    rng = np.random.default_rng(0)
    prompt = rng.integers(0, CFG.vocab, 150).tolist()
    root = d.kv.new()
    logits = d.step([prompt], [root], [-1])
    assert near(logits[0], step_reference(d, prompt)) < 0.1
    forks = d.kv.fork(root, 3)
    assert all(s.pages[:2] == root.pages[:2] and s.pages[2] != root.pages[2] for s in forks)
    assert S._groups([root] + forks) == ([0, 4], [2])
    other = d.kv.new()
    hist = [list(prompt) for _ in range(3)] + [[]]
    seqs = forks + [other]
    adapters = [0, 2, -1, 1]
    # the forks' first step starts from the shared prompt without adapters: the
    # reference recomputes it with them, so it is compared for those without only
    new = [rng.integers(0, CFG.vocab, n).tolist() for n in (1, 5, 1, 70)]
    logits = d.step(new, seqs, adapters)
    for h, n in zip(hist, new):
        h += n
    for i in (2, 3):
        assert near(logits[i], step_reference(d, hist[i], adapters[i])) < 0.1, i
    d.kv.free(root)
    moved = d.kv.compact()
    assert max(p for s in seqs for p in s.pages) < d.kv.n_pages - d.kv.free_pages
    for _ in range(3):
        new = [[int(t)] for t in rng.integers(0, CFG.vocab, 4)]
        logits = d.step(new, seqs, adapters)
        for h, n in zip(hist, new):
            h += n
    for i in (2, 3):
        assert near(logits[i], step_reference(d, hist[i], adapters[i])) < 0.1, (i, moved)
    for s in seqs:
        d.kv.free(s)
    assert d.kv.free_pages == d.kv.n_pages


def test_batch_decoder_rows_do_not_depend_on_their_batch():
    # a forked sequence's step against the same tokens in a cache of its own
    d = decoder(seed=1)
    rng = np.random.default_rng(1)
    prompt = rng.integers(0, CFG.vocab, 100).tolist()
    root = d.kv.new()
    d.step([prompt], [root])
    a, b = d.kv.fork(root, 2)
    d.kv.free(root)
    got = d.step([[3], [9]], [a, b])
    alone = d.kv.new()
    want = d.step([prompt + [9]], [alone])
    assert near(got[1], f64(want[0])) < 0.1
    with pytest.raises(ValueError):
        d.step([[1], [2]], [a, a])
    with pytest.raises(ValueError):
        d.step([[1]], [root])
    with pytest.raises(MemoryError):
        d.step([[1] * 1900, [1] * 1900], [a, b])
    assert a.length == 101 and d.kv.free_pages == 40 - len(set(a.pages + b.pages + alone.pages))


def test_batch_decoder_gate_notices_mistakes():
    # the bound that the steps above are held to is one that a mistake breaks: each is planted in
    # the restatement (adapters of the feed-forward four times as strong, so that each counts)
    lora = lora_weights(seed=6)
    for layer in lora.layers:
        for op in ("gate_up", "down"):
            if op in layer:
                layer[op] = (layer[op][0], layer[op][1] * 4)
    d = decoder(seed=3, lora=lora)
    rng = np.random.default_rng(3)
    hist = [rng.integers(0, CFG.vocab, n).tolist() for n in (6, 70)]
    seqs, adapters = [d.kv.new() for _ in hist], [2, 1]
    d.step([h[:-1] for h in hist], seqs, adapters)
    got = d.step([h[-1:] for h in hist], seqs, adapters)

    def off(i, history=None, adapter=adapters, layers=lora.layers):
        other = SimpleNamespace(w=d.w, kv=d.kv, lora=SimpleNamespace(scale=lora.scale, layers=layers))
        return near(got[i], step_reference(other, history or hist[i], adapter[i]))
    assert off(0) < 0.1 and off(1) < 0.1
    for li, layer in enumerate(lora.layers):
        for op in layer:
            without = [dict(x) for x in lora.layers]
            del without[li][op]
            assert off(0, layers=without) > 0.1 and off(1, layers=without) > 0.1, (li, op)
    assert off(0, adapter=[1, 0]) > 0.1 and off(1, adapter=[1, 0]) > 0.1
    h = hist[0]
    for history in (h[1:], h[:-2] + h[-1:], [h[1], h[0]] + h[2:], h[:-1] + [(h[-1] + 1) % CFG.vocab]):
        assert off(0, history=history) > 0.1, history            # a key lost, two slots swapped


def test_captured_step_of_all_ops():
    # adapters -> q/k norm, rotation, pages -> attention -> adapters as one graph, replayed over
    # growing sequences, a padding row among them, with the same step run eagerly in between
    H, KV, K, T = 8, 2, 256, 6
    N, g = (H + 2 * KV) * D, torch.Generator(device="cuda").manual_seed(50)
    up, down = lora_case(T, N, K, 16, 3, seed=51), lora_case(T, K, H * D, 16, 3, seed=52)
    gam = torch.ones(2, D, dtype=torch.bfloat16, device="cuda")
    rope, inv = S.rope_table_f32(1000), torch.full((2 * KV,), 30.0, device="cuda")
    scale, table = 1 / inv, torch.arange(T * 4, dtype=torch.int32, device="cuda").view(T, 4).clone()
    table[1:4, 0] = 0                                    # a shared first page
    sides = []
    for _ in range(2):
        k, v = codes(g, T * 4, KV, 2, PAGE, 64), codes(g, T * 4, KV, D, PAGE)
        sides.append(dict(k=k, v=v, qkv=torch.zeros(T, N, dtype=torch.bfloat16, device="cuda"),
                          att=torch.zeros(T, H, D, dtype=torch.bfloat16, device="cuda"),
                          o=torch.zeros(T, K, dtype=torch.bfloat16, device="cuda"),
                          plan=S.AttentionPlan(T - 1, T, H, KV, 4, n_groups=2),
                          lplan=S.LoraPlan(T, 3, 16, H * D)))
    sides[1]["k"], sides[1]["v"] = sides[0]["k"].clone(), sides[0]["v"].clone()
    meta = {n: torch.zeros(m, dtype=torch.int32, device="cuda") for n, m in
            (("pos", T), ("slot", T), ("start", T), ("lens", T - 1), ("group", 3), ("shared", 2), ("ids", T))}

    def step(s):
        s["plan"].update(meta["start"], meta["lens"], meta["group"], meta["shared"])
        s["lplan"].update(meta["ids"])
        S.lora_add(s["qkv"], up["base"], up["x"], up["a"], up["b"], up["scale"], s["lplan"])
        x = s["qkv"].view(T, H + 2 * KV, D)
        S.qk_norm_rope_pages(x[:, :H], x, gam[0], gam[1], s["k"], s["v"], inv, rope, meta["pos"], meta["slot"])
        S.attention_pages(s["att"], x[:, :H], s["k"], s["v"], scale, table[:T - 1], s["plan"])
        S.lora_add(s["o"], down["base"], s["att"].view(T, H * D), down["a"], down["b"], down["scale"],
                   s["lplan"])

    def put(i):
        lens = [70 + i, 65 + i, 66 + 3 * i, 130 + i, 1 + i]
        own = [n - 1 for n in lens]                     # the new key of each sequence
        rows = dict(pos=own + [-1], lens=lens, start=list(range(T)), group=[0, 1, 4], shared=[0, 1],
                    slot=[int(table[s, j // PAGE]) * PAGE + j % PAGE for s, j in enumerate(own)] + [-1],
                    ids=[(i + s) % 4 - 1 for s in range(T)])
        for n, values in rows.items():
            meta[n].copy_(torch.tensor(values, dtype=torch.int32))
        up["x"].normal_(generator=g)

    put(0)
    for s in sides:
        step(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(sides[0])
    for i in range(1, 8):
        put(i)
        graph.replay()
        step(sides[1])
        torch.cuda.synchronize()
        for n in ("qkv", "k", "v", "att", "o"):
            assert torch.equal(sides[0][n], sides[1][n]), (i, n)
    assert torch.isfinite(sides[0]["o"].float()).all()


def test_batch_decoder_on_another_stream():
    rng = np.random.default_rng(2)
    prompts = [rng.integers(0, CFG.vocab, n).tolist() for n in (130, 70, 3)]
    got = []
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        d = decoder(seed=2)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            root = d.kv.new()
            d.step([prompts[0]], [root])
            seqs = d.kv.fork(root, 2) + [d.kv.new()]
            d.step([[5], prompts[1], prompts[2]], seqs)
            d.kv.free(seqs[0])
            d.kv.compact()
            got.append(d.step([[7], [8]], seqs[1:]))
        torch.cuda.synchronize()
    assert torch.equal(got[0], got[1])


def test_host_refusals_on_device_tensors():
    b = batch([1, 1], [64, 70], seed=1)
    plan = make_plan(b)
    out = torch.empty(2, 32, D, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):                       # another table
        S.attention_pages(out, b["q"], b["k"], b["v"], b["scale"], b["table"][:, :1].contiguous(), plan)
    with pytest.raises(ValueError):                       # out too small
        S.attention_pages(out[:1], b["q"], b["k"], b["v"], b["scale"], b["table"], plan)
    with pytest.raises(TypeError):
        S.attention_pages(out, b["q"].float(), b["k"], b["v"], b["scale"], b["table"], plan)
    with pytest.raises(ValueError):                       # groups not planned
        plan.update(b["q_start"], b["lens"], b["q_start"], b["lens"])
    with pytest.raises(ValueError):
        S.attention_pages(out, b["q"], b["v"], b["k"], b["scale"], b["table"], plan)
    k = b["k"].unsqueeze(0)
    v = b["v"].unsqueeze(0)
    for src, dst in (([0], [0]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([-1], [0]), ([0], [99])):
        with pytest.raises(HephError) as e:
            S.copy_pages(k, v, src, dst)
        assert e.value.status == L.HEPH_ERR_SHAPE
    S.copy_pages(k, v, [], [])
    with pytest.raises(ValueError):
        S.copy_pages(k, v, [0, 1], [2])
    with pytest.raises(TypeError):
        S.copy_pages(k, v, [0.0], [1])
    with pytest.raises(OverflowError):
        S.copy_pages(k, v, [2 ** 31], [1])
    c = lora_case(4, 96, 256, 16, 2, seed=1)
    plan = S.LoraPlan(4, 2, 16, 256)
    with pytest.raises(HephError):                        # a workspace planned for less
        S.lora_add(c["base"], c["base"], *[lora_case(4, 96, 4096, 128, 2, 1)[f] for f in "xab"],
                   c["scale"], plan)
    with pytest.raises(ValueError):
        S.lora_add(c["base"], c["base"], c["x"], c["a"][:1], c["b"][:1], c["scale"], plan)
    with pytest.raises(TypeError):
        S.lora_add(c["base"], c["base"].float(), c["x"], c["a"], c["b"], c["scale"], plan)
    with pytest.raises(ValueError, match="x of shape"):
        S.lora_add(c["base"], c["base"], torch.cat([c["x"], c["x"]], 1), c["a"], c["b"], c["scale"], plan)
    with pytest.raises(ValueError, match="c of shape"):
        S.lora_add(c["base"].t().contiguous(), c["base"], c["x"], c["a"], c["b"], c["scale"], plan)
    plan = make_plan(b)
    for q in (b["q"].transpose(1, 2).contiguous().transpose(1, 2), b["q"][:, ::2], b["q"][:, :, :64],
              b["q"].flatten(), b["q"][:1].expand(2, 32, D)):
        with pytest.raises((ValueError, HephError)):
            S.attention_pages(out, q, b["k"], b["v"], b["scale"], b["table"], plan)
    with pytest.raises(ValueError):                       # a pool with a layer dimension
        S.attention_pages(out, b["q"], k, v, b["scale"], b["table"], plan)
