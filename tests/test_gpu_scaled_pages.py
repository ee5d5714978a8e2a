"""The paged cache with scales of its own (found while written, read back, attended to, copied)
against plain restatements in 64 bits.

Tolerances are counted from the roundings each op documents (half a step is 2^-8 relative in bf16,
2^-4 in E4M3, and 2^-10 of the scale for subnormal codes) plus the f32 sums' own bound: n terms
summed in f32 in any order are within n * 2^-24 of the sum of magnitudes.
"""
import math

import numpy as np
import pytest
import torch

from hephaestus_amd import serve as S
from hephaestus_amd.kernels import HephError
from tests.test_gpu_serve import (B16, CFG, D, E, F32, PAGE, batch, codes, f64, k_rows, make_plan, near,
                                  norm_rope, v_rows)
from hephaestus_amd import decode as DEC

pytestmark = pytest.mark.gpu

I32 = dict(dtype=torch.int32, device="cuda")


def i32(x):
    return torch.tensor(x, **I32)


def e4m3(x):
    return x.float().to(torch.float8_e4m3fn).double()


# ------------------------------------------------------------------ write ----

def write_case(runs, H=8, KV=4, seed=0, n_pages=None, pad=0, in_place=False, n_pos=5000):
    """runs: (first key, tokens) of sequences, each on pages of its own."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    T = sum(n for _, n in runs)
    need = sum((f + n - 1) // PAGE - f // PAGE + 1 for f, n in runs)
    n_pages = n_pages or need + 3
    ids = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
    pos, slot = [], []
    for first, n in runs:
        mine = {p: ids.pop() for p in range(first // PAGE, (first + n - 1) // PAGE + 1)}
        pos += range(first, first + n)
        slot += [mine[j // PAGE] * PAGE + j % PAGE for j in range(first, first + n)]
    wide = (H + 2 * KV) * D + pad
    buf = torch.randn(T, wide, generator=g, device="cuda")
    # heads and tokens of other magnitudes: v's scales differ, and grow by one step or several
    buf *= torch.randint(-3, 4, (T, 1), generator=g, device="cuda").float().exp2()
    buf = buf.to(torch.bfloat16)
    qkv = buf[:, :(H + 2 * KV) * D].unflatten(1, (H + 2 * KV, D))
    gam = (1 + 0.3 * torch.randn(2, D, generator=g, device="cuda")).to(torch.bfloat16)
    q = qkv[:, :H] if in_place else torch.zeros(T, H, D, dtype=torch.bfloat16, device="cuda")
    return dict(qkv=qkv, gam=gam, k=codes(g, n_pages, KV, 2, PAGE, 64), v=codes(g, n_pages, KV, D, PAGE),
                scale=torch.randint(-11, -4, (n_pages, 2 * KV), generator=g, device="cuda").float().exp2(),
                pos=i32(pos), slot=i32(slot), q=q, n_pos=n_pos, H=H, KV=KV)


def write(c, s=slice(None), eps=1e-6):
    S.qk_norm_rope_pages_scaled(c["q"][s], c["qkv"][s], c["gam"][0], c["gam"][1], c["k"], c["v"], c["scale"],
                                S.rope_table_f32(c["n_pos"]), c["pos"][s].clone(), c["slot"][s].clone(), eps)


def old_exp(scale):
    """Exponents of scales as they may lie in memory."""
    bits = scale.cpu().view(torch.int32).long()
    return ((bits >> 23 & 0xFF) - 127).clamp(-117, 119)


def check_write(c, eps=1e-6):
    H, KV = c["H"], c["KV"]
    x, k0, v0, q0 = f64(c["qkv"]).clone(), k_rows(c["k"]), v_rows(c["v"]), f64(c["q"]).clone()
    s0 = c["scale"].cpu().clone()
    write(c, eps=eps)
    torch.cuda.synchronize()
    gam, pos, slot = f64(c["gam"]), c["pos"].cpu().long(), c["slot"].cpu().long()
    n_pages = c["k"].shape[0]
    live = (pos >= 0) & (pos < c["n_pos"])
    at = torch.where(live, pos, 0)
    q = norm_rope(x[:, :H], gam[0], at, eps)
    # f32 inside: the norm's factor, table entries and four products, each within a few 2^-24 of
    # the pair's magnitude
    slop = 64 * F32 * q.abs().amax(-1, keepdim=True)
    got = f64(c["q"])
    assert ((got - q).abs() <= B16 * q.abs() + slop)[live].all()
    assert torch.equal(got[~live], q0[~live])
    cached = live & (slot >= 0) & (slot < n_pages * PAGE)
    new = torch.cat([norm_rope(x[:, H:H + KV], gam[1], at, eps), x[:, H + KV:]], 1)      # [T, 2 KV, 128]
    got_k, got_v = k_rows(c["k"]).view(n_pages, PAGE, KV, D), v_rows(c["v"]).view(n_pages, PAGE, KV, D)
    got = torch.cat([got_k, got_v], 2)
    was = torch.cat([k0.view(n_pages, PAGE, KV, D), v0.view(n_pages, PAGE, KV, D)], 2)
    scale, e0 = f64(c["scale"]), old_exp(s0)
    for p in range(n_pages):
        mine = cached & (slot // PAGE == p)
        if not mine.any():                                   # as it was, to the last bit
            assert torch.equal(c["scale"][p].cpu().view(torch.int32), s0[p].view(torch.int32))
            assert torch.equal(torch.nan_to_num(got[p], 999.0), torch.nan_to_num(was[p], 999.0))
            continue
        y, key = new[mine], slot[mine] % PAGE
        amax = torch.where(torch.isfinite(y), y.abs(), 0).amax(0).amax(-1)
        e = torch.log2(scale[p])
        assert torch.equal(e, e.round()) and (e >= -117).all() and (e <= 119).all()
        fresh = bool((key == 0).any())
        floor = torch.full_like(e, -117.0) if fresh else e0[p].double()
        # the least 2^e that holds the values, up to k's f32 rounding of them, and no less than it was
        near_edge = torch.where(torch.arange(2 * KV) < KV, 64 * F32, 0.0)
        assert (e >= floor).all()
        assert ((amax <= 448 * 2.0 ** e * (1 + near_edge)) | (e == 119)).all()
        assert ((e == floor) | (amax > 224 * 2.0 ** e * (1 - near_edge))).all()
        # new codes
        val, scaled = got[p][key], y / 2.0 ** e[:, None]
        # (an infinity or NaN of a k head reaches all of it through its norm)
        bad = ~torch.isfinite(scaled)
        assert torch.isnan(val[bad]).all()
        scaled = torch.where(bad, 0, scaled).clamp(-448, 448)
        tol = torch.maximum(E * scaled.abs(), torch.tensor(2.0 ** -10).double())
        tol = tol + near_edge[:, None] * scaled.abs().amax(-1, keepdim=True)
        assert ((val - scaled).abs() <= tol)[~bad].all()
        assert torch.equal(val[:, KV:][~bad[:, KV:]], e4m3(scaled[:, KV:])[~bad[:, KV:]])   # v: one rounding
        # the other keys: rescaled codes, to the last bit
        rest = torch.ones(PAGE, dtype=torch.bool)
        rest[key] = False
        by = torch.ones(2 * KV).double() if fresh else 2.0 ** (e0[p] - e).clamp_min(-126)
        want = e4m3(was[p] * by[:, None])[rest]
        assert torch.equal(torch.isnan(got[p][rest]), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got[p][rest]), torch.nan_to_num(want))


@pytest.mark.parametrize("runs,H,KV", [
    ([(0, 1)], 32, 8), ([(63, 1)], 8, 8), ([(64, 1), (5, 1), (700, 1)], 16, 2), ([(0, 64)], 8, 4),
    ([(10, 54)], 8, 4), ([(10, 55)], 5, 1), ([(37, 200)], 40, 8), ([(0, 130), (63, 2), (64, 64), (1, 1)], 8, 4),
    ([(i * 7, 1) for i in range(130)], 32, 8), ([(i * 31, 3) for i in range(50)], 8, 4),
    ([(3, 300), (0, 200), (100, 500), (64, 1), (65, 63)], 16, 4),          # over 512 tokens
    ([(i * 3, 1) for i in range(600)], 8, 2), ([(0, 900)], 32, 8), ([(17, 1000), (40, 9)], 12, 12),
])
def test_write(runs, H, KV):
    check_write(write_case(runs, H, KV, seed=len(runs) + runs[0][1]))


@pytest.mark.parametrize("T", [70, 600])
@pytest.mark.parametrize("pad,in_place", [(0, True), (8, False), (264, True)])
def test_write_strides_and_in_place(T, pad, in_place):
    check_write(write_case([(20, T)], 16, 4, seed=5, pad=pad, in_place=in_place))


@pytest.mark.parametrize("value", [0.0, -0.0, -1.0, float("nan"), float("inf"), 1e-45, 3e38, 2.0 ** -120])
def test_write_over_scales_that_were_never_written(value):
    # pages begun anew do not look at what they held; others take its exponent, held to the range
    c = write_case([(0, 30), (64, 1), (70, 3)], seed=3)
    c["scale"].fill_(value)
    check_write(c)


def test_write_a_page_that_begins_behind_its_key_0():
    # its scale set to 0 first: the new values' own, as where key 0 is among them
    for T in (3, 40):
        c, d = write_case([(10, T)], seed=18), write_case([(0, T)], seed=18)
        for x in (c, d):
            x["qkv"][:, x["H"] + x["KV"]:] *= 2.0 ** -20
        c["scale"].zero_()
        check_write(c)
        write(d)
        page = [int(x["slot"][0]) // PAGE for x in (c, d)]
        assert torch.equal(c["scale"][page[0], c["KV"]:], d["scale"][page[1], d["KV"]:])


def test_write_slots_of_a_run_in_any_order():
    c = write_case([(0, 64), (70, 40)], seed=4)
    order = torch.cat([torch.randperm(64), 64 + torch.randperm(40).flip(0)]).cuda()
    for f in ("pos", "slot"):
        c[f] = c[f][order]
    # (the second run lies in one page up to key 127)
    check_write(c)
    c = write_case([(64, 64)] * 10, seed=6)                    # over 512 tokens, falling
    c["slot"] = c["slot"].view(10, 64).flip(1).reshape(-1).contiguous()
    check_write(c)


@pytest.mark.parametrize("T", [100, 700])
def test_write_padding_rows_and_bad_slots(T):
    c = write_case([(0, T)], seed=7)
    # (at page edges: a page's tokens stay neighbours)
    c["pos"][[0, 64, T - 1]] = i32([-1, 5000, 2 ** 31 - 1])
    c["slot"][[63, 65]] = i32([-1, 2 ** 31 - 1])
    c["slot"][62] = c["k"].shape[0] * PAGE
    check_write(c)
    c["pos"].fill_(-1)                                         # nothing to write
    check_write(c)


@pytest.mark.parametrize("T", [3, 70, 130, 600, 1100])
@pytest.mark.parametrize("first", [0, 5])
@pytest.mark.parametrize("holes", ["one", "third", "most", "edges", "long"])
def test_write_skipped_tokens_inside_pages(T, first, holes):
    """Tokens without a position or a slot among those of a page, also more of them than a window
    or two hold: the page's other tokens are still written as one."""
    c = write_case([(first, T)], seed=14)
    t = torch.arange(T)
    skip = {"one": t % 64 == 30, "third": t % 3 == 1, "most": t % 20 != 7, "edges": (t % 4 == 3) | (t % 64 == 0),
            "long": (t % 64 == 1) | (t % 64 == 40)}[holes]
    if holes == "long":                                        # 150 skipped ones in one place of each page
        n = 1 + 149 * skip.long()
        idx = torch.repeat_interleave(t, n).cuda()
        skip = torch.repeat_interleave(skip, n)
        for f in ("pos", "slot"):
            c[f] = c[f][idx].contiguous()
        c["qkv"], c["q"] = c["qkv"][idx].contiguous(), c["q"][idx].contiguous()
    bad = torch.nonzero(skip).flatten()
    for i, b in enumerate(bad.tolist()):
        if i % 3 == 0:
            c["pos"][b] = -1
        else:
            c["slot"][b] = (-1, c["k"].shape[0] * PAGE)[i % 2]
    check_write(c)


@pytest.mark.parametrize("T", [3, 600, 1100])
def test_write_skipped_tokens_between_sequences(T):
    # a padded batch: each sequence's rows are followed by rows of none
    runs = [(i * 5, 1 + i % 3) for i in range(T // 3 + 1)]
    c = write_case(runs, seed=15)
    idx, keep, at = [], [], 0
    for _, n in runs:
        idx += [*range(at, at + n), *[at] * (4 - n)]
        keep += [True] * n + [False] * (4 - n)
        at += n
    idx, off = torch.tensor(idx).cuda(), ~torch.tensor(keep).cuda()
    for f in ("pos", "slot", "qkv", "q"):
        c[f] = c[f][idx].contiguous()
    c["pos"][off] = -1
    check_write(c)


@pytest.mark.parametrize("T", [70, 600])
def test_write_nan_infinities_and_extremes(T):
    c = write_case([(5, T)], seed=8)
    x, H, KV = c["qkv"], c["H"], c["KV"]
    x[3, H + KV, 7], x[4, H + KV, 8], x[4, H + KV, 9] = float("nan"), float("inf"), float("-inf")
    x[6, H + 1, 0], x[7, H + 2, 5] = float("nan"), float("inf")
    x[8, H + KV + 1] = float("nan")                            # a whole row
    x[:, H + KV + 2] = 0                                       # a block of zeros
    x[10, H + KV + 3, 0], x[11, H + KV + 3, 0] = 3.3895313892515355e38, -448 * 2.0 ** 119
    check_write(c)
    c = write_case([(0, T)], seed=9)
    c["qkv"][:, c["H"] + c["KV"]:] *= 1e-38                    # down to subnormal bf16
    c["scale"].fill_(2.0 ** -126)
    check_write(c)
    c = write_case([(3, T)], seed=10)
    c["qkv"].zero_()
    check_write(c)


def test_write_edges_of_the_scale():
    # largest values of exactly 448 * 2^e and just above, e over the whole range
    for e in (-117, -20, -6, 0, 5, 100, 119):
        for f, step in ((1.0, 0), (1 + 2.0 ** -7, 1), (0.5, -1), (0.5 + 2.0 ** -8, 0)):
            if not -117 <= e + step <= 119:
                continue
            c = write_case([(0, 1)], 4, 2, seed=11)
            c["qkv"][0, 6:] = 0
            c["qkv"][0, 6, 3] = -448 * f * 2.0 ** e
            check_write(c)
            page = int(c["slot"][0]) // PAGE
            assert float(c["scale"][page, 2]) == 2.0 ** (e + step), (e, f)


def test_write_token_by_token_equals_at_once():
    # the same scales, and values that differ by what codes lost when their scale grew
    runs = [(0, 150)]
    whole, steps = write_case(runs, seed=12), write_case(runs, seed=12)
    write(whole)
    for t in range(150):
        write(steps, slice(t, t + 1))
    torch.cuda.synchronize()
    assert torch.equal(whole["scale"], steps["scale"]) and torch.equal(whole["q"], steps["q"])
    for rows, f in ((k_rows, "k"), (v_rows, "v")):
        slot = whole["slot"].cpu().long()
        a, b = rows(whole[f])[slot], rows(steps[f])[slot]
        # each growth rounds a code that becomes subnormal by half of 2^-9 at most, which the later
        # ones halve at least: in all below 2^-9, beside the first rounding's half step
        assert ((a - b).abs() <= 2.0 ** -9 + 2 * E * a.abs()).all()
        assert torch.equal(a[a.abs() >= 2.0 ** -2], b[a.abs() >= 2.0 ** -2])


def test_write_repeats_bit_for_bit_and_captured():
    a, b = (write_case([(5, 300), (64, 70), (1, 1)], seed=13) for _ in range(2))
    rope = S.rope_table_f32(a["n_pos"])

    def call(c):
        S.qk_norm_rope_pages_scaled(c["q"], c["qkv"], *c["gam"], c["k"], c["v"], c["scale"], rope, c["pos"], c["slot"])
    start = {f: a[f].clone() for f in ("k", "v", "scale", "qkv")}
    call(a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(a)
    for i in range(4):
        for c in (a, b):
            for f in start:
                c[f].copy_(start[f])
            c["qkv"][:, c["H"]:] *= 2.0 ** i                   # other scales each time
        graph.replay()
        call(b)
        torch.cuda.synchronize()
        for f in ("q", "k", "v", "scale"):
            assert torch.equal(a[f], b[f]), (i, f)


def test_write_and_read_pools_past_32_bits():
    KV, n_pages = 8, (5 << 30) // (8 * 8192)
    k = torch.empty(n_pages, KV, 2, PAGE, 64, dtype=torch.uint8, device="cuda")
    v = torch.empty(n_pages, KV, D, PAGE, dtype=torch.uint8, device="cuda")
    scale = torch.zeros(n_pages, 2 * KV, device="cuda")
    for T in (90, 600):
        c = write_case([(10, T)], 8, KV, seed=14)
        n = c["k"].shape[0]
        for name, pool in (("k", k), ("v", v), ("scale", scale)):
            pool[-n:] = c[name]
        far = dict(c, k=k, v=v, scale=scale, slot=c["slot"] + (n_pages - n) * PAGE, q=torch.zeros_like(c["q"]))
        write(far)
        write(c)
        rows = [[torch.zeros(T, KV, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)] for _ in range(2)]
        S.read_pages(*rows[0], k, v, far["slot"], page_scale=scale)
        S.read_pages(*rows[1], c["k"], c["v"], c["slot"], page_scale=c["scale"])
        torch.cuda.synchronize()
        for name, pool in (("k", k), ("v", v), ("scale", scale)):
            assert torch.equal(pool[-n:], c[name])
        assert torch.equal(rows[0][0], rows[1][0]) and torch.equal(rows[0][1], rows[1][1])


# ------------------------------------------------------------------- read ----

def check_read(slots, KV=4, seed=0, n_pages=9, static=False, nan=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    k, v = codes(g, n_pages, KV, 2, PAGE, 64), codes(g, n_pages, KV, D, PAGE)
    if nan:
        k[0, 0, 0, 3, 5], v[1, 1, 17, 8] = 0x7F, 0xFF
    n = len(slots)
    out = [torch.full((n, KV, D), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    if static:
        scale = torch.rand(2 * KV, generator=g, device="cuda") + 0.1
        S.read_pages(*out, k, v, i32(slots), kv_scale=scale)
        per_page = scale.cpu().expand(n_pages, 2 * KV)
    else:
        scale = torch.randint(-117, 120, (n_pages, 2 * KV), generator=g, device="cuda").double().exp2().float()
        S.read_pages(*out, k, v, i32(slots), page_scale=scale)
        per_page = scale.cpu()
    torch.cuda.synchronize()
    s = torch.tensor(slots).long()
    ok = (s >= 0) & (s < n_pages * PAGE)
    at = torch.where(ok, s, 0)
    for i, rows in enumerate((k_rows(k), v_rows(v))):
        # (a product in f32 and its rounding to bf16; with a power of two both are exact)
        want = rows[at].float() * per_page[at // PAGE, i * KV:(i + 1) * KV, None]
        want = torch.where(ok[:, None, None], want.to(torch.bfloat16), torch.tensor(7.0, dtype=torch.bfloat16))
        got = out[i].cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
        if not static:
            exact = rows[at] * per_page.double()[at // PAGE, i * KV:(i + 1) * KV, None]
            assert torch.equal(torch.nan_to_num(got.double()[ok]), torch.nan_to_num(exact[ok]))


@pytest.mark.parametrize("static", [False, True])
@pytest.mark.parametrize("n", [1, 64, 65, 3000])
def test_read(n, static):
    check_read([j % (9 * PAGE) for j in range(5, 5 + n)], seed=n, static=static)


@pytest.mark.parametrize("KV", [1, 3, 8, 64])
def test_read_heads(KV):
    check_read(list(range(60, 200)), KV=KV, seed=KV, nan=KV > 1)


def test_read_rounds_the_product_in_f32_and_then_to_bf16():
    # with one scale for all pages: scales whose product with 1.875 (code 0x3F) is, rounded to f32,
    # just between two bf16 values, while the exact product is not
    x = (np.arange(1, 4000, 4, dtype=np.uint32) << 16 | 0x3F808000).view(np.float32)     # halfway, odd above
    x = x[x < 4]
    s = (x.astype(np.float64) / 1.875).astype(np.float32)
    exact = s.astype(np.float64) * 1.875
    twice = (s * np.float32(1.875) == x) & (exact != x)
    s, exact = s[twice][:8], exact[twice][:8]
    assert len(s) == 8
    KV = 4
    k = torch.full((1, KV, 2, PAGE, 64), 0x3F, dtype=torch.uint8, device="cuda")
    v = torch.full((1, KV, D, PAGE), 0x3F, dtype=torch.uint8, device="cuda")
    out = [torch.zeros(3, KV, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    S.read_pages(*out, k, v, i32([0, 1, 63]), kv_scale=torch.from_numpy(s).cuda())
    want = torch.from_numpy(s * np.float32(1.875)).to(torch.bfloat16)
    once = torch.from_numpy(exact).to(torch.float64)
    got = torch.cat([out[0][0, :, 0], out[1][0, :, 0]]).cpu()
    assert torch.equal(got, want)
    # one step off the nearest at most: half a step of bf16 and half of one of f32
    assert ((got.double() - once).abs() <= (2.0 ** -8 + 2.0 ** -24) * once).all()
    for o in out:
        assert (o == o[:1, :, :1]).all()


def test_read_any_slots():
    rng = np.random.default_rng(0)
    check_read(rng.integers(0, 9 * PAGE, 500).tolist(), seed=1)                      # scattered, repeated
    check_read(rng.integers(0, 9 * PAGE, 2500).tolist(), seed=2)
    check_read([5] * 200 + list(range(100, 10, -1)), seed=3)
    bad = rng.integers(0, 9 * PAGE, 100)
    bad[[0, 5, 63, 64, 99]] = [-1, 9 * PAGE, 2 ** 31 - 1, -2 ** 31, -1]
    check_read(bad.tolist(), seed=4)
    check_read([-1, -2, -3, 0, 1, 2], seed=5)
    check_read([0, 1, 2, 63, 64, 65, 66, 128, 127], seed=6, nan=True)


# --------------------------------------------------------------- attention ----

def with_scales(b, seed=0, spread=3):
    g = torch.Generator(device="cuda").manual_seed(seed + 1000)
    n = b["k"].shape[0]
    b["page_scale"] = torch.randint(-7 - spread, -6, (n, 2 * b["KV"]), generator=g, device="cuda").float().exp2()
    return b


def attend(b, plan=None, fill=7.0):
    out = torch.full((b["T"], b["H"], D), fill, dtype=torch.bfloat16, device="cuda")
    S.attention_pages_scaled(out, b["q"], b["k"], b["v"], b["page_scale"], b["table"], plan or make_plan(b))
    return out


def check_attention(b, out, tokens=None):
    H, KV, G = b["H"], b["KV"], b["H"] // b["KV"]
    table, n_pages = b["table"].cpu(), b["k"].shape[0]
    got, t = f64(out), 0
    for s, n in enumerate(b["new"]):
        total = b["kv_len"][s]
        ids = table[s, :-(-total // PAGE)].long()
        ok = ((ids >= 0) & (ids < n_pages)).repeat_interleave(PAGE)[:total]
        ids = ids.clamp(0, n_pages - 1).cuda()
        scale = f64(b["page_scale"])[ids.cpu()].repeat_interleave(PAGE, 0)[:total]
        ks = k_rows(b["k"][ids])[:total] * scale[:, :KV, None]
        vs = v_rows(b["v"][ids])[:total] * scale[:, KV:, None]
        for i in range(n):
            if tokens is not None and t not in tokens:
                t += 1
                continue
            see = ok & (torch.arange(total) <= total - n + i)
            q = f64(b["q"][t]).view(KV, G, D)
            if see.any():
                x = torch.einsum("kgd,jkd->kgj", q, ks[see]) / math.sqrt(D)
                mag = torch.einsum("kgd,jkd->kgj", q.abs(), ks[see].abs()) / math.sqrt(D)
                p = torch.softmax(x, -1)
                want = torch.einsum("kgj,jkd->kgd", p, vs[see]).reshape(H, D)
                weight = torch.einsum("kgj,jkd->kgd", p, vs[see].abs()).reshape(H, D)
                # a probability is off by its rounding to bf16 and by its score's f32 sum (and
                # exp2's argument), numerator and denominator; then out's own rounding
                e = 2 * (140 * F32 * mag.amax(-1) + 2.0 ** -20).view(H, 1)
                tol = (B16 + e) * weight + B16 * want.abs() + (B16 * B16) * weight
            else:
                want, tol = torch.zeros(H, D).double(), torch.zeros(H, D).double()
            off = (got[t] - want).abs()
            assert (off <= tol).all(), (s, i, (off - tol).max().item())
            t += 1
    assert (got[t:] == 7.0).all()


@pytest.mark.parametrize("new,own,shared,group_start", [
    ([1], [1], (), ()), ([1], [64], (), ()), ([1, 1, 1], [63, 1, 200], (), ()),
    ([1], [64 * 70 + 3], (), ()), ([5, 1, 3], [5, 9, 70], (), ()), ([64], [300], (), ()),
    ([130, 1, 33], [130, 90, 64], (), ()), ([300], [64 * 9], (), ()),
    ([1] * 4, [1, 30, 64, 100], [5], [0, 4]),
    ([1] * 9, [10, 20, 30, 40, 50, 60, 70, 80, 90], [2, 7, 1], [0, 4, 5, 9]),
    ([1] * 40, list(range(1, 41)), [20], [0, 40]),
    ([3, 40, 1, 70], [3, 45, 200, 100], [6], [0, 4]),
    ([1, 100, 1, 1], [3, 120, 70, 5], [25], [0, 4]),
])
def test_attention(new, own, shared, group_start):
    b = with_scales(batch(new, own, shared, group_start, seed=sum(own)), seed=len(own))
    check_attention(b, attend(b))


@pytest.mark.parametrize("H,KV", [(8, 8), (40, 8), (16, 2), (7, 1), (64, 1), (96, 4)])
def test_attention_head_layouts(H, KV):
    b = with_scales(batch([1, 1, 4, 1], [70, 64, 100, 1], shared=[3], group_start=[0, 4], seed=H, H=H, KV=KV))
    check_attention(b, attend(b))
    b = with_scales(batch([20, 1], [40, 100], seed=H + 1, H=H, KV=KV))
    check_attention(b, attend(b))


def test_attention_scales_far_apart():
    # pages whose values are a million times others', both ways, wide and narrow units
    for new, own in (([1], [500]), ([1, 1], [64, 700]), ([90], [400])):
        b = with_scales(batch(new, own, seed=21), seed=21, spread=20)
        check_attention(b, attend(b))
        b["page_scale"][:, b["KV"]:] *= 2.0 ** 20
        check_attention(b, attend(b))


@pytest.mark.parametrize("lo,hi", [(105, 119), (60, 119), (-117, -100), (-117, -60), (-117, 119)])
def test_attention_values_at_the_ends_of_their_range(lo, hi):
    """Values up to 448 * 2^119, whose sums leave f32's range though their mean does not, and down to
    the smallest normal ones; in one unit, in parts that are merged, behind a prefix, wide and narrow."""
    for i, (new, own, shared, group_start) in enumerate([
            ([1], [300], (), ()), ([1], [64 * 70 + 3], (), ()), ([5, 40], [30, 200], (), ()), ([150], [700], (), ()),
            ([1] * 9, [10, 20, 30, 40, 50, 60, 70, 80, 90], [2, 7, 1], [0, 4, 5, 9]),
            ([1, 100, 1, 1], [3, 120, 70, 5], [25], [0, 4])]):
        b = with_scales(batch(new, own, shared, group_start, seed=50 + i), seed=50 + i)
        g = torch.Generator().manual_seed(i)
        scale = torch.randint(lo, hi + 1, (b["k"].shape[0], b["KV"]), generator=g).double().exp2()
        b["page_scale"][:, b["KV"]:] = scale.float().cuda()
        check_attention(b, attend(b))


@pytest.mark.parametrize("new", [1, 20])
def test_attention_values_grow_along_a_long_run(new):
    # more than 64 pages of one unit (as many sequences as there are places), the later ones' values
    # larger or smaller than the first ones'
    n, pages = 70, 70
    b = with_scales(batch([new] * n, [64 * pages - 5] * n, seed=60, H=8 if new == 1 else 32, garbage=False), seed=60)
    first = torch.zeros(b["k"].shape[0], dtype=torch.bool)
    first[b["table"][:, :64].flatten().cpu().long()] = True
    for early, late in ((110, 119), (119, 110), (-117, -85), (-90, -117), (0, 100), (0, 0)):
        e = torch.where(first, early, late).float()
        b["page_scale"][:, b["KV"]:] = e.exp2()[:, None].cuda()
        check_attention(b, attend(b), tokens=[0, 5 * new + new // 2, n * new - 1])


def test_attention_one_scale_equals_the_static_op():
    # with one power of two everywhere the codes enter as multiples of it: the products are the
    # same but for the order of the exact scaling, out to the last bit where nothing is rounded twice
    b = batch([1] * 5 + [90], [100, 1, 64, 700, 65, 200], [6], [0, 6], seed=22)
    b["page_scale"] = torch.full((b["k"].shape[0], 2 * b["KV"]), 2.0 ** -7, device="cuda")
    b["scale"] = torch.full((2 * b["KV"],), 2.0 ** -7, device="cuda")
    want = torch.empty(b["T"], b["H"], D, dtype=torch.bfloat16, device="cuda")
    S.attention_pages(want, b["q"], b["k"], b["v"], b["scale"], b["table"], make_plan(b))
    got = attend(b)
    assert torch.equal(got, want)


def test_attention_bad_pages_and_lengths():
    b = with_scales(batch([1, 1, 3], [300, 100, 80], seed=3, garbage=False,
                          bad=[(0, 1, -1), (0, 3, 10 ** 6), (1, 0, -7), (2, 0, 2 ** 31 - 1)]))
    check_attention(b, attend(b))
    b = with_scales(batch([1, 1], [5, 64], bad=[(0, 0, -1), (1, 0, 99)], seed=4, garbage=False))
    check_attention(b, attend(b))                              # nothing left: zero rows
    b = with_scales(batch([90, 1], [64 * 80, 70], seed=5, garbage=False))
    b["table"][0, [0, 64, 79]] = i32([-1, 10 ** 6, -7])
    check_attention(b, attend(b), tokens=[0, 40, 89, 90])
    b = with_scales(batch([1, 2], [50, 60], seed=6, garbage=False, extra_tokens=4))
    b["lens"][0], b["kv_len"][0] = -5, 0
    check_attention(b, attend(b))


def test_attention_nan_stays_with_its_rows():
    for new in (20, 100):
        b = with_scales(batch([new], [new + 30], seed=13))
        page = int(b["table"][0, 0])
        b["v"][page, :, 5, S.v_place(40)] = 0x7F
        out = attend(b).float()
        sees = torch.arange(new) + 30 >= 40
        assert torch.isnan(out[sees.cuda()][:, :, 5]).all()
        out[sees.cuda(), :, 5] = 0
        assert torch.isfinite(out).all()


def test_attention_many_sequences_and_longest():
    rng = np.random.default_rng(7)
    own = [int(x) for x in rng.integers(1, 90, 700)]
    b = with_scales(batch([1] * 700, own, [3, 2], [0, 300, 700], seed=8, H=4, KV=1))
    check_attention(b, attend(b), tokens=set(rng.integers(0, 700, 100).tolist()))
    b = with_scales(batch([1, 1], [262144, 2], seed=9, H=8, KV=1, garbage=False))
    b["table"] = b["table"][:, :4096].contiguous()
    check_attention(b, attend(b))


def test_attention_pools_past_32_bits():
    KV, n_pages = 8, (5 << 30) // (8 * 8192)
    k = torch.empty(n_pages, KV, 2, PAGE, 64, dtype=torch.uint8, device="cuda")
    v = torch.empty(n_pages, KV, D, PAGE, dtype=torch.uint8, device="cuda")
    scale = torch.empty(n_pages, 2 * KV, device="cuda")
    small = with_scales(batch([1, 40], [300, 200], seed=36, garbage=False))
    at = n_pages - small["k"].shape[0]
    k[at:], v[at:], scale[at:] = small["k"], small["v"], small["page_scale"]
    far = dict(small, k=k, v=v, page_scale=scale, table=torch.where(small["table"] < 0, small["table"], small["table"] + at))
    assert torch.equal(attend(far), attend(small))


def test_attention_two_streams_and_two_graphs_of_a_plan():
    bs = [with_scales(batch([1] * 6, own, [5], [0, 6], seed=40), seed=i)
          for i, own in enumerate(([1, 64, 200, 7, 900, 65], [3] * 6))]
    bs[1]["table"] = torch.nn.functional.pad(
        bs[1]["table"], (0, bs[0]["table"].shape[1] - bs[1]["table"].shape[1]), value=-1)
    want = [attend(b) for b in bs]
    plans, outs = [make_plan(b) for b in bs], [torch.zeros_like(w) for w in want]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in bs]
    for _ in range(8):
        for b, p, o, s in zip(bs, plans, outs, streams):
            with torch.cuda.stream(s):
                p.update(b["q_start"], b["lens"], b["group_start"], b["shared"])
                S.attention_pages_scaled(o, b["q"], b["k"], b["v"], b["page_scale"], b["table"], p)
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
    graphs = []
    for b, o in zip(bs, outs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            plans[0].update(b["q_start"], b["lens"], b["group_start"], b["shared"])
            S.attention_pages_scaled(o, b["q"], b["k"], b["v"], b["page_scale"], b["table"], plans[0])
    for i in range(4):
        for o in outs:
            o.zero_()
        graphs[i % 2].replay()
        graphs[1 - i % 2].replay()
        assert torch.equal(attend(bs[0], make_plan(bs[0])), want[0])
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))


# ------------------------------------------------- copies and the whole step ----

@pytest.mark.parametrize("layers,KV,n_pages,n", [(1, 1, 4, 1), (3, 8, 40, 16), (2, 5, 900, 300)])
def test_copy_pages_with_scales(layers, KV, n_pages, n):
    g = torch.Generator(device="cuda").manual_seed(n)
    k, v = codes(g, layers, n_pages, KV, 2, PAGE, 64), codes(g, layers, n_pages, KV, D, PAGE)
    scale = torch.rand(layers, n_pages, 2 * KV, generator=g, device="cuda")
    ids = torch.randperm(n_pages, generator=torch.Generator().manual_seed(n)).tolist()
    src, dst = [ids[i // 2] for i in range(n)], ids[n:2 * n]
    want = [t.clone() for t in (k, v, scale)]
    for t in want:
        t[:, dst] = t[:, src]
    S.copy_pages(k, v, src, dst, page_scale=scale)
    assert all(torch.equal(a, b) for a, b in zip((k, v, scale), want))


def decoder(seed=0, n_pages=40, page_scales=True):
    w = DEC.random_init(CFG, seed)
    kv = S.PagedKVCache(CFG, n_pages, page_scales=page_scales)
    if not page_scales:
        kv.scale.fill_(4.0 / 448)
        kv.inv.fill_(448 / 4.0)
    return S.Qwen3BatchDecoder(w, kv, n_pos=2048)


def reference(d, history):
    """Logits after the last token of one sequence: every token recomputed in f64 from the
    dequantized weights, activations quantized as the step does, keys and values by blocks of 64."""
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

    def block(x):
        out = torch.empty_like(x)
        for a in range(0, x.shape[0], PAGE):
            y = x[a:a + PAGE]
            s = 2.0 ** torch.ceil(torch.log2(y.abs().amax(0).amax(-1) / 448))[:, None]
            out[a:a + PAGE] = e4m3(y / s) * s
        return out

    def norm(x, gamma):
        return bf(f64(gamma) * bf(x / torch.sqrt((x * x).mean(-1, keepdim=True) + cfg.eps)))

    T, H, KV = len(history), cfg.n_heads, cfg.n_kv_heads
    x, pos, G = bf(deq(w.embed)[history]), torch.arange(T), H // KV
    for lw in w.layers:
        qkv = bf(quant(norm(x, lw.attn_norm)) @ deq(lw.qkv).T).view(T, H + 2 * KV, D)
        q = bf(norm_rope(qkv[:, :H], f64(lw.q_norm), pos, cfg.eps, cfg.theta))
        k = block(norm_rope(qkv[:, H:H + KV], f64(lw.k_norm), pos, cfg.eps, cfg.theta))
        v = block(qkv[:, H + KV:])
        sc = torch.einsum("tkgd,jkd->kgtj", q.view(T, KV, G, D), k) / math.sqrt(D)
        sc = sc.masked_fill(pos[None, :] > pos[:, None], -math.inf)
        att = bf(torch.einsum("kgtj,jkd->tkgd", sc.softmax(-1), v).reshape(T, H * D))
        x = bf(x + quant(att) @ deq(lw.o).T)
        gate, up = bf(quant(norm(x, lw.ffn_norm)) @ deq(lw.gate_up).T).chunk(2, -1)
        x = bf(x + quant(bf(bf(gate / (1 + torch.exp(-gate))) * up)) @ deq(lw.down).T)
    return (quant(norm(x[-1:], w.final_norm)) @ deq(w.embed).T)[0]


def test_decoder_prompts_fork_decode_compact():
    # the bound that a static cache's steps are held to (W8A8 flips of single codes); a cache
    # whose scales were lost on a fork or a compaction is far outside it
    d = decoder()
    rng = np.random.default_rng(0)
    prompt = rng.integers(0, CFG.vocab, 150).tolist()
    root = d.kv.new()
    assert near(d.step([prompt], [root])[0], reference(d, prompt)) < 0.1
    seqs = d.kv.fork(root, 2) + [d.kv.new()]
    hist = [list(prompt), list(prompt), []]
    for i, counts in enumerate(((1, 5, 70), (1, 1, 1), (3, 1, 1))):
        new = [rng.integers(0, CFG.vocab, n).tolist() for n in counts]
        logits = d.step(new, seqs)
        for h, n in zip(hist, new):
            h += n
        if i == 0:
            d.kv.free(root)
            assert d.kv.compact() > 0
    for i, h in enumerate(hist):
        assert near(logits[i], reference(d, h)) < 0.1, i
    d.kv.page_scale *= 4
    assert near(d.step([[1], [1], [1]], seqs)[0], reference(d, hist[0] + [1])) > 0.1
    for s in seqs:
        d.kv.free(s)
    assert d.kv.free_pages == d.kv.n_pages


def test_cache_reads_what_the_decoder_wrote():
    for page_scales in (True, False):
        d = decoder(seed=4, page_scales=page_scales)
        seq, other = d.kv.new(), d.kv.new()
        rng = np.random.default_rng(4)
        d.step([rng.integers(0, CFG.vocab, 100).tolist(), [3]], [seq, other])
        k, v = d.kv.read(seq, 1)
        assert k.shape == v.shape == (100, CFG.n_kv_heads, D)
        pages = torch.tensor(seq.pages).cuda()
        scale = (f64(d.kv.page_scale[1])[seq.pages].repeat_interleave(PAGE, 0)[:100] if page_scales
                 else f64(d.kv.scale[1])[None].expand(100, -1))
        for got, rows, s in ((k, k_rows(d.kv.k[1][pages]), scale[:, :CFG.n_kv_heads]),
                             (v, v_rows(d.kv.v[1][pages]), scale[:, CFG.n_kv_heads:])):
            want = rows[:100] * s[..., None]
            assert ((f64(got) - want).abs() <= (2.0 ** -24 + B16) * want.abs() * (not page_scales)).all()
        part = d.kv.read(seq, 1, 60, 9)
        assert torch.equal(part[0], k[60:69]) and torch.equal(part[1], v[60:69])
        assert d.kv.read(seq, 0, 100)[0].shape == (0, CFG.n_kv_heads, D)
        for args in ((seq, 2), (seq, -1), (seq, 0, 101), (seq, 0, 90, 11), (seq, 0, -1, 3), (seq, 0, 3, -1)):
            with pytest.raises(ValueError):
                d.kv.read(*args)


@pytest.mark.parametrize("fails", ["logits", "tokens", "scratch", "no masks"])
def test_a_step_without_memory_writes_no_keys(monkeypatch, fails):
    """A step that finds no memory for its logits, or for the pick behind them, has not touched the
    older keys of a partly filled page, whose scales and codes it would change."""
    d = decoder(seed=6, page_scales=True)
    seq = d.kv.new()
    rng = np.random.default_rng(6)
    d.step([rng.integers(0, CFG.vocab, 70).tolist()], [seq])
    kv, more = d.kv, rng.integers(0, CFG.vocab, 50).tolist()

    def state():
        return [t.clone() for t in (kv.k, kv.v, kv.page_scale)], seq.length, list(seq.pages), kv.free_pages
    before = state()
    empty, shape = torch.empty, {"logits": (1, CFG.vocab), "tokens": (1,)}.get(fails)

    def full(*args, **kw):
        if args == shape:
            raise torch.OutOfMemoryError("no memory")
        return empty(*args, **kw)

    def scratch(*args):
        raise torch.OutOfMemoryError("no memory")
    with monkeypatch.context() as m:
        m.setattr(torch, "empty", full)
        if fails == "scratch":
            m.setattr(S, "pick_ws", scratch)
        with pytest.raises(ValueError if fails == "no masks" else torch.OutOfMemoryError):
            if fails == "logits":
                d.step([more], [seq])
            elif fails == "no masks":
                d.next_tokens([more], [seq], masks=torch.zeros(0, -(-CFG.vocab // 32), **I32), mask_ids=[-1])
            else:
                d.next_tokens([more], [seq])
    after = state()
    assert after[1:] == before[1:] and all(torch.equal(a, b) for a, b in zip(after[0], before[0]))
    d.step([more], [seq])
    assert not torch.equal(kv.page_scale[:, before[2][1]], before[0][2][:, before[2][1]])


def test_cache_reads_on_another_stream():
    """Reads of two sequences on a stream that is busy, while the current one allocates and writes."""
    for page_scales in (True, False):
        d = decoder(seed=5, page_scales=page_scales)
        a, b = d.kv.new(), d.kv.new()
        rng = np.random.default_rng(5)
        d.step([rng.integers(0, CFG.vocab, n).tolist() for n in (200, 200)], [a, b])
        want = [d.kv.read(q, 1) for q in (a, b)]
        s, busy = torch.cuda.Stream(), torch.randn(4096, 4096, device="cuda")
        torch.cuda.synchronize()
        for ctx in (s, s.cuda_stream, 0):
            if ctx != 0:
                with torch.cuda.stream(s):
                    for _ in range(10):
                        busy = torch.mm(busy, busy).mul_(2.0 ** -12)
            got = [d.kv.read(q, 1, ctx=ctx) for q in (a, b)]
            full = [torch.full((n,), -1, dtype=torch.int32, device="cuda") for n in (200, 200, 200 * 128, 200 * 128)]
            torch.cuda.synchronize()
            for g, w in zip(got, want):
                assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])
            del full


def test_captured_step_of_write_attend_read():
    # the run of them as a serving step makes it, captured and replayed over growing sequences
    # (a page filled, one begun, a padding row), against the same run made eagerly
    H, KV, T, steps = 8, 2, 5, 70
    g = torch.Generator(device="cuda").manual_seed(60)
    rope, gam = S.rope_table_f32(1000), torch.ones(2, D, dtype=torch.bfloat16, device="cuda")
    table = torch.arange(T * 4, **I32).view(T, 4).clone()
    sides = [dict(k=torch.zeros(T * 4, KV, 2, PAGE, 64, dtype=torch.uint8, device="cuda"),
                  v=torch.zeros(T * 4, KV, D, PAGE, dtype=torch.uint8, device="cuda"),
                  s=torch.zeros(T * 4, 2 * KV, device="cuda"), plan=S.AttentionPlan(T - 1, T, H, KV, 4),
                  att=torch.zeros(T, H, D, dtype=torch.bfloat16, device="cuda"),
                  q=torch.zeros(T, H, D, dtype=torch.bfloat16, device="cuda"),
                  back=[torch.zeros(T, KV, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)])
             for _ in range(2)]
    qkv = torch.zeros(T, H + 2 * KV, D, dtype=torch.bfloat16, device="cuda")
    meta = {n: torch.zeros(m, **I32) for n, m in (("pos", T), ("slot", T), ("start", T), ("lens", T - 1))}

    def step(s):
        s["plan"].update(meta["start"], meta["lens"])
        S.qk_norm_rope_pages_scaled(s["q"], qkv, gam[0], gam[1], s["k"], s["v"], s["s"], rope, meta["pos"], meta["slot"])
        S.attention_pages_scaled(s["att"], s["q"], s["k"], s["v"], s["s"], table[:T - 1], s["plan"])
        S.read_pages(*s["back"], s["k"], s["v"], meta["slot"], page_scale=s["s"])

    def put(i):
        own = [i, i, i + 1 if i else 0, i]
        rows = dict(pos=own + [-1], lens=[n + 1 for n in own], start=list(range(T)),
                    slot=[int(table[s, j // PAGE]) * PAGE + j % PAGE for s, j in enumerate(own)] + [-1])
        for n, values in rows.items():
            meta[n].copy_(torch.tensor(values, dtype=torch.int32))
        qkv.normal_(generator=g)
        qkv[:, H + KV:] *= 2.0 ** (i % 5)

    put(0)
    for s in sides:
        step(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(sides[0])
    for i in range(1, steps):
        put(i)
        graph.replay()
        step(sides[1])
        torch.cuda.synchronize()
        for n in ("k", "v", "s", "att", "q"):
            assert torch.equal(sides[0][n], sides[1][n]), (i, n)
        assert all(torch.equal(a, b) for a, b in zip(sides[0]["back"], sides[1]["back"]))
    b = dict(new=[1] * (T - 1), kv_len=[int(x) for x in meta["lens"]], table=table[:T - 1], k=sides[0]["k"],
             v=sides[0]["v"], page_scale=sides[0]["s"], q=sides[0]["q"][:T - 1], T=T - 1, H=H, KV=KV)
    check_attention(b, sides[0]["att"][:T - 1])
    # what was read back is what was written, within its codes' rounding
    y = torch.cat([norm_rope(f64(qkv)[:, H:H + KV], f64(gam[1]), meta["pos"].cpu().clamp_min(0), 1e-6),
                   f64(qkv)[:, H + KV:]], 1)[:T - 1]
    got = torch.cat([f64(x) for x in sides[0]["back"]], 1)[:T - 1]
    scale = f64(sides[0]["s"])[meta["slot"].cpu().long()[:T - 1] // PAGE][..., None]
    tol = torch.maximum(E * y.abs(), 2.0 ** -10 * scale) + 64 * F32 * y.abs().amax(-1, keepdim=True)
    assert ((got - y).abs() <= tol).all()


def test_host_refusals_on_device_tensors():
    c = write_case([(0, 9)], seed=1)
    rope = S.rope_table_f32(c["n_pos"])

    def call(**kw):
        a = dict(c, **kw)
        S.qk_norm_rope_pages_scaled(a["q"], a["qkv"], *a["gam"], a["k"], a["v"], a["scale"], rope, a["pos"], a["slot"])
    for kw in (dict(scale=c["scale"][:-1]), dict(scale=c["scale"][:, :-1]), dict(scale=c["scale"].t().contiguous()),
               dict(scale=c["scale"].cpu()), dict(pos=c["pos"][:-1]), dict(k=c["k"][:-1])):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(TypeError):
        call(scale=c["scale"].half())
    rows = [torch.zeros(9, 4, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for args, kw in (((*rows, c["k"], c["v"], c["slot"]), {}),
                     ((*rows, c["k"], c["v"], c["slot"]), dict(kv_scale=c["scale"][0], page_scale=c["scale"])),
                     ((rows[0][:8], rows[1], c["k"], c["v"], c["slot"]), dict(page_scale=c["scale"])),
                     ((*rows, c["k"], c["v"], c["slot"]), dict(page_scale=c["scale"][:2])),
                     ((*rows, c["k"], c["v"], c["slot"]), dict(kv_scale=c["scale"][0, :5].clone())),
                     ((*rows, c["v"], c["k"], c["slot"]), dict(page_scale=c["scale"]))):
        with pytest.raises(ValueError):
            S.read_pages(*args, **kw)
    with pytest.raises(HephError):
        S.read_pages(rows[0], rows[0], c["k"], c["v"], c["slot"], page_scale=c["scale"])
    with pytest.raises(TypeError):
        S.read_pages(*rows, c["k"], c["v"], c["slot"].long(), page_scale=c["scale"])
    b = with_scales(batch([1, 1], [64, 70], seed=1))
    with pytest.raises(ValueError, match="page_scale of shape"):
        attend(dict(b, page_scale=b["scale"]))
    with pytest.raises(ValueError, match="page_scale of shape"):
        S.copy_pages(c["k"][None], c["v"][None], [0], [1], page_scale=c["scale"])
