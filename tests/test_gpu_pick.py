"""The pick of the next tokens against plain restatements.

The processed logits are compared with the same f32 operations of numpy (each correctly rounded, so
equal to the last bit), log-probabilities with 64 bits: a sum of n terms exp(l - top), each within
2^-21 (its argument's rounding, at most 2^-24 * 1.45 * 104, counts for the small ones only: a term
exp(-d) is off by d * exp(-d) * 2^-23, under 2^-24; exp2 itself by 2^-23), summed in f32 in chains of
at most 64 and trees behind them, and one log.
"""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from hephaestus_amd import _lib as L
from hephaestus_amd import decode as DEC
from hephaestus_amd import serve as S
from hephaestus_amd.kernels import HephError
from tests.test_gpu_serve import CFG

pytestmark = pytest.mark.gpu

REL = 2.0 ** -17          # of the sum: 64 + 20 additions of 2^-24 each, and a term's own 2^-22


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def bits_of(allowed):
    """bool [n, vocab] -> int32 words."""
    n, vocab = allowed.shape
    a = np.zeros((n, -(-vocab // 32) * 32), np.uint8)
    a[:, :vocab] = allowed
    return torch.from_numpy(np.packbits(a, axis=1, bitorder="little").view(np.int32).copy()).cuda()


def case(rows, vocab, history=50, max_bias=0, masks=0, seed=0, dtype=torch.float32, scale=3.0):
    rng = np.random.default_rng(seed)
    n_slots = rows + 2
    rules = S.TokenRules(n_slots, vocab, history, max_bias)
    h = rng.zipf(1.3, (n_slots, history)) % vocab
    length = rng.integers(0, history + 1, n_slots)
    rules.history.copy_(torch.from_numpy(h.astype(np.int32)))
    rules.length.copy_(torch.from_numpy(length.astype(np.int32)))
    rules.n_prompt.copy_(torch.from_numpy(rng.integers(0, length + 1).astype(np.int32)))
    rules.penalties.copy_(torch.from_numpy(
        np.stack([1 + rng.random(n_slots), rng.normal(0, 0.5, n_slots), rng.normal(0, 0.3, n_slots)], 1)))
    if max_bias:
        rules.bias_ids.copy_(torch.from_numpy(rng.integers(0, vocab, (n_slots, max_bias)).astype(np.int32)))
        rules.bias.normal_(0, 3)
        rules.n_bias.copy_(torch.from_numpy(rng.integers(0, max_bias + 1, n_slots).astype(np.int32)))
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = dict(logits=(torch.randn(rows, vocab, generator=g, device="cuda") * scale).to(dtype), rules=rules,
             slots=i32(rng.permutation(n_slots)[:rows]), masks=None, mask_ids=None)
    if masks:
        c["masks"] = bits_of(rng.random((masks, vocab)) < 0.3)
        c["mask_ids"] = i32(rng.integers(-1, masks, rows))
    return c


def reference(c):
    """f32 logits after the rules, as numpy rounds them."""
    x = c["logits"].float().cpu().numpy().copy()
    r, one = c["rules"], np.float32
    vocab = x.shape[1]
    for row in range(x.shape[0]):
        slot = int(c["slots"][row]) if c["slots"] is not None else -1
        if r is not None and 0 <= slot < r.n_slots:
            n = min(max(int(r.length[slot]), 0), r.max_tokens)
            h, first = r.history[slot, :n].cpu().numpy(), int(r.n_prompt[slot])
            rep, pres, freq = r.penalties[slot].cpu().numpy()
            inside = (h >= 0) & (h < vocab)
            answered = np.bincount(h[inside & (np.arange(n) >= first)], minlength=vocab)
            seen = np.bincount(h[inside], minlength=vocab) > 0
            with np.errstate(all="ignore"):
                y = np.where(x[row] > 0, x[row] / rep, x[row] * rep)
                x[row] = np.where(seen, y, x[row])
                y = x[row] - (answered.astype(one) * freq + pres)
                x[row] = np.where(answered > 0, y, x[row])
            ids, values = r.bias_ids[slot].tolist(), r.bias[slot].cpu().numpy()
            last = {t: values[i] for i, t in enumerate(ids[:min(max(int(r.n_bias[slot]), 0), r.max_bias)])}
            for t, b in last.items():
                if 0 <= t < vocab:
                    x[row, t] = one(x[row, t] + b)
        if c["masks"] is not None:
            m = int(c["mask_ids"][row])
            if 0 <= m < c["masks"].shape[0]:
                words = c["masks"][m].cpu().numpy().view(np.uint8)
                x[row, np.unpackbits(words, bitorder="little")[:vocab] == 0] = -np.inf
    return x


def pick(c, out=False, append=False, in_place=False):
    rows = c["logits"].shape[0]
    tokens, logprob = i32([-9] * rows), torch.full((rows,), 9.0, device="cuda")
    o = c["logits"] if in_place else torch.full_like(c["logits"], 55.0) if out else None
    S.pick_tokens(tokens, c["logits"], c["rules"], c["slots"], c["masks"], c["mask_ids"], out=o, logprob=logprob,
                  append=append)
    torch.cuda.synchronize()
    return tokens.cpu().numpy(), logprob.cpu().numpy(), o


def check(c, out=True, in_place=False, append=False):
    want = reference(c)
    tokens, logprob, o = pick(c, out, append, in_place)
    if o is not None:
        a = torch.from_numpy(want).to(o.dtype)
        got = o.cpu()
        assert torch.equal(torch.isnan(a), torch.isnan(got))
        assert torch.equal(torch.nan_to_num(a, 3.0), torch.nan_to_num(got, 3.0))
    clean = np.where(np.isnan(want), -np.inf, want)
    best = clean.argmax(1)                                  # the first of equal ones
    none = clean.max(1) == -np.inf
    assert np.array_equal(tokens, np.where(none, -1, best))
    top = clean.max(1)
    for r in range(len(tokens)):
        if np.isnan(want[r]).any() or top[r] == np.inf:
            assert np.isnan(logprob[r])
        elif none[r]:
            assert logprob[r] == -np.inf
        else:
            exact = -np.log(np.exp(want[r].astype(np.float64) - top[r]).sum())
            assert abs(logprob[r] - exact) <= REL + 2.0 ** -22 * abs(exact), (r, logprob[r], exact)
    return tokens


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,history,max_bias,masks", [
    (1, 1, 1, 0, 0), (1, 2, 5, 1, 1), (3, 31, 40, 3, 2), (2, 33, 1, 0, 1), (5, 5003, 600, 20, 3),
    (2, 16384, 300, 300, 2), (3, 16385, 70, 0, 0), (4, 32769, 5000, 5, 0), (2, 151936, 900, 300, 2),
    (70, 4097, 33, 7, 5), (300, 1000, 20, 2, 3),
])
def test_pick(rows, vocab, history, max_bias, masks, dtype):
    check(case(rows, vocab, history, max_bias, masks, seed=rows + vocab, dtype=dtype))


@pytest.mark.parametrize("rows", [1, 30, 200])
def test_pick_long_histories(rows):
    check(case(rows, 40000, 20000, 9, 0, seed=rows), out=rows < 100)


def test_pick_counts_past_sixteen_bits():
    c = case(1, 500, 262144, 1, 0, seed=2)
    c["rules"].history.fill_(123)
    c["rules"].length.fill_(262144)
    c["rules"].n_prompt.fill_(0)
    c["rules"].penalties[:, 2] = 1e-5
    c["rules"].bias_ids.fill_(123)
    check(c)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pick_repetition_below_one(dtype):
    # what was seen is preferred: positive logits grow, negative ones shrink towards 0
    c = case(6, 7001, 900, 20, 2, seed=17, dtype=dtype)
    c["rules"].penalties[:, 0] = torch.tensor([0.3, 0.5, 0.75, 0.999, 2.0 ** -20, 1e-30, 1.0, 0.1]).cuda()
    check(c)


def test_pick_without_rules_or_masks():
    for seed, kw in enumerate((dict(rules=None, slots=None), dict())):
        c = dict(case(5, 7001, 100, 3, 0, seed=seed), **kw)
        check(c, out=False)
    c = case(6, 7001, 100, 3, 2, seed=3)
    c["slots"] = i32([-1, 99, 2 ** 31 - 1, -2 ** 31, 8, 0])
    c["mask_ids"] = i32([0, 2, -1, 2 ** 31 - 1, 1, -2 ** 31])
    check(c)
    # tokens or out alone
    o = torch.zeros_like(c["logits"])
    S.pick_tokens(None, c["logits"], c["rules"], c["slots"], out=o)
    want = reference(dict(c, masks=None))
    assert np.array_equal(o.cpu().numpy(), want)


def test_pick_ties_go_to_the_lowest_index():
    for vocab in (64, 5000, 40000):
        c = dict(case(8, vocab, seed=vocab), rules=None, slots=None)
        c["logits"].fill_(1.5)
        for r in range(8):
            c["logits"][r, [int(x) for x in np.random.default_rng(r).integers(0, vocab, 5)]] = 2.5
        check(c)
    c["logits"].fill_(-0.0)
    c["logits"][:, 7:] = 0.0                                 # equal to -0
    assert (check(c) == 0).all()


def test_pick_masks_that_leave_nothing_or_one():
    c = case(6, 20001, 100, 4, 1, seed=5)
    allowed = np.zeros((6, 20001), bool)
    allowed[1, 20000] = allowed[2, 0] = allowed[3, 16384] = allowed[4, 16383] = True
    allowed[5] = True
    c["masks"], c["mask_ids"] = bits_of(allowed), i32([0, 1, 2, 3, 4, 5])
    tokens = check(c)
    assert tokens[:5].tolist() == [-1, 20000, 0, 16384, 16383]


def test_pick_nan_infinities_and_lowest_values():
    c = case(9, 20001, 100, 4, 1, seed=6)
    x = c["logits"]
    x[0, 17000] = float("nan")
    x[1, 5] = float("inf")
    x[2].fill_(float("-inf"))
    x[3].fill_(torch.finfo(torch.float32).min)
    x[4].fill_(float("nan"))
    x[5, :20000] = float("-inf")
    x[6, 11], x[6, 12] = float("nan"), float("inf")          # masked below
    x[7].fill_(3e38)
    x[8] *= 1e-42                                            # subnormals
    c["slots"] = i32([0, 1, 2, -1, 3, 4, 5, -1, -1])
    allowed = np.ones((1, 20001), bool)
    allowed[0, [11, 12]] = False
    c["masks"], c["mask_ids"] = bits_of(allowed), i32([-1, -1, -1, -1, -1, -1, 0, -1, -1])
    check(c)


def test_pick_bad_metadata_stays_in_bounds():
    c = case(5, 3001, 64, 8, 0, seed=7)
    r = c["rules"]
    r.length.copy_(i32([2 ** 31 - 1, -1, 65, -2 ** 31, 64, 3, 64]))
    r.n_prompt.copy_(i32([2 ** 31 - 1, 5, -7, 3, 1000, -2 ** 31, 64]))
    r.n_bias.copy_(i32([2 ** 31 - 1, -3, 9, -2 ** 31, 8, 3, 8]))
    r.history[:, ::7] = 3001
    r.history[:, 1::7] = -1
    r.history[:, 2::7] = -2 ** 31
    r.bias_ids[:, ::3] = -5
    r.bias_ids[:, 1::3] = 2 ** 31 - 1
    check(c)


def test_pick_a_bias_twice_the_last_one_counts():
    c = case(3, 20000, 10, 40, 0, seed=8)
    r = c["rules"]
    r.bias_ids[:] = i32([5, 19000] * 20)
    r.bias[:] = torch.arange(40, device="cuda").float()
    r.n_bias.copy_(i32([40, 39, 2, 1, 0]))
    check(c)


def test_pick_rows_apart_and_in_place():
    for dtype in (torch.float32, torch.bfloat16):
        c = case(7, 5003, 90, 5, 2, seed=9, dtype=dtype)
        wide = torch.randn(7, 5003 + 13, device="cuda").to(dtype)
        wide[:, 3:5006] = c["logits"]
        guard = wide.clone()
        c["logits"] = wide[:, 3:5006]
        want = reference(c)
        tokens, _, _ = pick(c)
        check(c)
        assert torch.equal(wide, guard)                      # inputs as they were
        check(c, in_place=True)
        assert torch.equal(wide[:, 3:5006].float().cpu(), torch.from_numpy(want).to(dtype).float())
        assert torch.equal(wide[:, :3], guard[:, :3]) and torch.equal(wide[:, 5006:], guard[:, 5006:])
    c = case(1, 5003, 90, 5, 2, seed=10)
    check(c, in_place=True)


def test_pick_appends_to_the_histories():
    c = case(6, 9000, 30, 0, 1, seed=11)
    r = c["rules"]
    c["masks"], c["mask_ids"] = bits_of(np.zeros((1, 9000), bool)), i32([-1, -1, 0, -1, -1, -1])
    c["slots"] = i32([3, 0, 1, -1, 99, 5])
    r.length.copy_(i32([4, 9, 2, 30, 6, 0, 0, 0]))           # slot 3 is full, row 2 has no token
    before, length = r.history.cpu().numpy().copy(), r.length.cpu().numpy().copy()
    tokens = check(c, append=True)
    want = before.copy()
    for row, slot in ((1, 0), (5, 5)):
        want[slot, length[slot]] = tokens[row]
        length[slot] += 1
    assert np.array_equal(r.history.cpu().numpy(), want) and np.array_equal(r.length.cpu().numpy(), length)


def test_pick_rows_that_share_a_request():
    # several rows of one slot (samples of one request) and one mask; nothing is appended
    c = case(6, 9001, 300, 5, 2, seed=17)
    c["slots"], c["mask_ids"] = i32([2, 2, 2, 0, 2, 0]), i32([1, 1, 1, 1, 0, 1])
    check(c)


def test_pick_scratch_of_a_larger_batch_serves_smaller_ones():
    ws = S.pick_ws(40, 151936)
    for rows, vocab in ((40, 151936), (27, 151936), (26, 151936), (13, 151936), (1, 151936), (14, 50000), (3, 9)):
        c = dict(case(rows, vocab, seed=rows), rules=None, slots=None)
        tokens = i32([0] * rows)
        S.pick_tokens(tokens, c["logits"], ws=ws)
        assert torch.equal(tokens.long(), c["logits"].argmax(1))
        assert S.pick_ws(rows, vocab).numel() <= ws.numel()


def test_pick_repeats_bit_for_bit():
    c = case(40, 30000, 3000, 50, 4, seed=12)
    first = pick(c, out=True)
    for _ in range(3):
        again = pick(c, out=True)
        assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])
        assert torch.equal(first[2], again[2])


def test_pick_captured_greedy_loop():
    # a loop on the device: logits that depend on the last token, histories that grow
    rows, vocab = 5, 20001
    g = torch.Generator(device="cuda").manual_seed(13)
    model = torch.randn(97, vocab, generator=g, device="cuda")
    masks = bits_of(np.random.default_rng(13).random((2, vocab)) < 0.2)
    mask_ids, slots = i32([0, -1, 1, -1, 0]), i32([4, 0, 2, 1, 3])
    sides = []
    for _ in range(2):
        rules = S.TokenRules(rows, vocab, 64, 4)
        for s in range(rows):
            rules.set(s, [s, 7, 7, s + 1], repetition=1.3, presence=0.4, frequency=0.2, bias={11: -2.0, s: 1.5})
        sides.append(SimpleNamespace(rules=rules, tokens=i32([1] * rows), lp=torch.zeros(rows, device="cuda"),
                                     logits=torch.zeros(rows, vocab, device="cuda"), ws=S.pick_ws(rows, vocab)))

    def step(s):
        torch.index_select(model, 0, s.tokens % 97, out=s.logits)
        S.pick_tokens(s.tokens, s.logits, s.rules, slots, masks, mask_ids, logprob=s.lp, append=True, ws=s.ws)
    for s in sides:
        step(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(sides[0])
    for i in range(70):                                      # past the histories' room
        c = dict(logits=model[(sides[1].tokens % 97).long()], rules=sides[1].rules, slots=slots, masks=masks,
                 mask_ids=mask_ids)
        want = reference(c).argmax(1)
        graph.replay()
        step(sides[1])
        torch.cuda.synchronize()
        assert np.array_equal(sides[1].tokens.cpu().numpy(), want), i
        assert torch.equal(sides[0].tokens, sides[1].tokens) and torch.equal(sides[0].lp, sides[1].lp)
        assert torch.equal(sides[0].rules.history, sides[1].rules.history)
    assert (sides[0].rules.length == 64).all()


def test_pick_on_two_streams_at_once():
    cs = [case(30, 40000, 2000, 9, 3, seed=14), case(4, 151936, 500, 0, 0, seed=15)]
    want = [pick(c, out=True) for c in cs]
    outs = [(i32([0] * len(w[0])), torch.zeros(len(w[0]), device="cuda"), torch.zeros_like(w[2])) for w in want]
    ws = [S.pick_ws(*c["logits"].shape) for c in cs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    for _ in range(6):
        for c, o, w, s in zip(cs, outs, ws, streams):
            with torch.cuda.stream(s):
                S.pick_tokens(o[0], c["logits"], c["rules"], c["slots"], c["masks"], c["mask_ids"], out=o[2],
                              logprob=o[1], ws=w)
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert np.array_equal(w[0], o[0].cpu().numpy()) and np.array_equal(w[1], o[1].cpu().numpy())
        assert torch.equal(w[2], o[2])


def test_pick_scratch_on_another_stream():
    """A call on another stream than the current one, whose scratch it allocates itself: what the
    current stream allocates and writes behind the call is other memory."""
    c = case(300, 20000, 100, seed=31)
    want, lp = torch.empty(2, 300, device="cuda").unbind()
    want = want.int()
    S.pick_tokens(want, c["logits"], c["rules"], c["slots"], logprob=lp)
    tokens, logprob = torch.zeros(300, dtype=torch.int32, device="cuda"), torch.zeros(300, device="cuda")
    s, busy = torch.cuda.Stream(), torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    for ctx in (s, s.cuda_stream):
        with torch.cuda.stream(s):
            for _ in range(10):
                busy = torch.mm(busy, busy).mul_(2.0 ** -12)
        S.pick_tokens(tokens, c["logits"], c["rules"], c["slots"], logprob=logprob, ctx=ctx)
        nb = S.pick_ws(300, 20000).numel()
        full = [torch.full((nb,), 0x41, dtype=torch.uint8, device="cuda") for _ in range(8)]
        torch.cuda.synchronize()
        assert torch.equal(tokens, want) and torch.equal(logprob, lp)
        assert all((f == 0x41).all() for f in full)
        tokens.zero_()
        logprob.zero_()
        torch.cuda.synchronize()
    S.pick_tokens(tokens, c["logits"], c["rules"], c["slots"], logprob=logprob, ctx=0)
    torch.cuda.synchronize()
    assert torch.equal(tokens, want) and torch.equal(logprob, lp)


@pytest.mark.parametrize("dtype,rows", [(torch.float32, 55), (torch.float32, 56), (torch.bfloat16, 111)])
def test_pick_logits_that_the_caches_hold_and_more(dtype, rows):
    # 32 MiB of logits after the rules are the border
    check(case(rows, 151937, 300, 20, 3, seed=rows, dtype=dtype))


def test_pick_rows_past_32_bits():
    # logits of 8.6 GB: the last rows equal the same rows alone
    rows, vocab = 14200, 151936
    x = torch.empty(rows, vocab, device="cuda")
    small = case(3, vocab, 100, 5, 2, seed=16)
    x[-3:] = small["logits"]
    rest = i32([-1] * (rows - 3))
    tokens = i32([0] * rows)
    S.pick_tokens(tokens, x, small["rules"], torch.cat([rest, small["slots"]]), small["masks"],
                  torch.cat([rest, small["mask_ids"]]), out=x)
    torch.cuda.synchronize()
    want = reference(small)
    assert np.array_equal(x[-3:].cpu().numpy(), want)
    assert np.array_equal(tokens[-3:].cpu().numpy(), want.argmax(1))


def test_rules_set():
    r = S.TokenRules(3, 100, 8, 2)
    r.set(1, [1, 2, 3], [4, 4], 1.5, 0.25, -0.5, {7: -float("inf"), 9: 2.0})
    assert r.history[1, :5].tolist() == [1, 2, 3, 4, 4] and r.length.tolist() == [0, 5, 0]
    assert r.n_prompt.tolist() == [0, 3, 0] and r.penalties[1].tolist() == [1.5, 0.25, -0.5]
    assert r.bias_ids[1].tolist() == [7, 9] and r.bias[1].tolist() == [-float("inf"), 2.0]
    assert r.n_bias.tolist() == [0, 2, 0] and r.penalties[0].tolist() == [1, 0, 0]
    c = dict(logits=torch.zeros(1, 100, device="cuda"), rules=r, slots=i32([1]), masks=None, mask_ids=None)
    assert check(c)[0] == 9
    r.set(1)                                                 # another request, without rules
    assert r.length[1] == 0 and r.n_bias[1] == 0 and check(c)[0] == 0


def test_next_tokens_follow_the_logits():
    # the decoder's steps with rules against its own logits and the restated rules
    def make():
        w = DEC.random_init(CFG, 7)
        d = S.Qwen3BatchDecoder(w, S.PagedKVCache(CFG, 40, page_scales=True), n_pos=2048)
        return d, [d.kv.new() for _ in range(3)]
    (a, seqs), (b, others) = make(), make()
    rules = S.TokenRules(4, CFG.vocab, 300, 3)
    prompts = [list(range(5, 90)), [3], [17, 17, 40]]
    for slot, p in zip((2, 0), prompts):
        rules.set(slot, p, repetition=1.8, presence=0.5, frequency=0.1, bias={1: 2.0})
    masks = bits_of(np.arange(CFG.vocab)[None] % 3 == 1)
    slots, mask_ids = [2, 0, -1], [-1, 0, 0]
    new = prompts
    for i in range(12):
        logits = b.step(new, others)
        want = reference(dict(logits=logits, rules=rules, slots=i32(slots), masks=masks, mask_ids=i32(mask_ids)))
        length = rules.length.tolist()
        tokens, logprob = a.next_tokens(new, seqs, None, rules, slots, masks, mask_ids)
        assert np.array_equal(tokens.cpu().numpy(), want.argmax(1)), i
        assert torch.isfinite(logprob).all() and (logprob <= 0).all()
        assert rules.length.tolist() == [length[0] + 1, 0, length[2] + 1, 0]
        new = [[t] for t in tokens.tolist()]
    assert (tokens[1:] % 3 == 1).all()
    assert rules.history[2, 85:97].tolist()[-1] == int(tokens[0])
    tokens, _ = a.next_tokens(new, seqs)                      # greedy, without rules
    assert torch.equal(tokens.long(), b.step(new, others).argmax(1))
    before = [s.length for s in seqs]
    for kw in (dict(rules=rules), dict(rules=rules, slots=[0, 1]), dict(rules=rules, slots=[1, 1, 0]),
               dict(rules=rules, slots=[0, 1, 4]), dict(masks=masks), dict(masks=masks, mask_ids=[0, 0, 1]),
               dict(masks=masks[:, :3], mask_ids=[0, 0, 0]), dict(masks=masks.cpu(), mask_ids=[0, 0, 0]),
               dict(rules=S.TokenRules(4, 100, 3), slots=[0, 1, 2])):
        with pytest.raises(ValueError):
            a.next_tokens(new, seqs, **kw)
    with pytest.raises(TypeError):
        a.next_tokens(new, seqs, masks=masks.long(), mask_ids=[0, 0, 0])
    assert [s.length for s in seqs] == before


def test_host_refusals_on_device_tensors():
    c = case(3, 500, 20, 2, 2, seed=1)
    tokens = i32([0, 0, 0])

    def call(tokens=tokens, logits=c["logits"], rules=c["rules"], slots=c["slots"], **kw):
        S.pick_tokens(tokens, logits, rules, slots, **kw)
    for kw in (dict(slots=None), dict(rules=None), dict(masks=c["masks"]), dict(mask_ids=c["mask_ids"]),
               dict(tokens=tokens[:2]), dict(slots=c["slots"][:2]), dict(out=c["logits"][:, :499]),
               dict(masks=c["masks"][:, :5].contiguous(), mask_ids=c["mask_ids"]), dict(logits=c["logits"].t()),
               dict(logits=c["logits"][:, ::2]), dict(rules=S.TokenRules(5, 499, 3)), dict(tokens=tokens.cpu()),
               dict(logprob=torch.zeros(2, device="cuda")), dict(logits=c["logits"].cpu())):
        with pytest.raises(ValueError):
            call(**kw)
    for kw in (dict(logits=c["logits"].half()), dict(logits=c["logits"][0]), dict(tokens=tokens.long()),
               dict(out=c["logits"].to(torch.bfloat16)), dict(slots=c["slots"].long())):
        with pytest.raises(TypeError):
            call(**kw)
    for kw in (dict(tokens=None), dict(ws=torch.empty(16, dtype=torch.uint8, device="cuda")),
               dict(append=True, rules=None, slots=None), dict(tokens=None, out=c["logits"], append=True)):
        with pytest.raises(HephError):
            call(**kw)
    with pytest.raises(HephError):
        S.pick_ws(0, 5)
    assert L.lib().heph_pick_ws_bytes(1, 0) == 0
