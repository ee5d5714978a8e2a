"""The serving ops' argument checks and the page bookkeeping, without a GPU."""
import ctypes
import time
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from hephaestus_amd import _lib as L
from hephaestus_amd import serve as S
from hephaestus_amd.loader import Qwen3Config

FAKE, ODD = 0x10000, 0x10008        # never dereferenced by validation
CFG = Qwen3Config(vocab=512, hidden=256, n_layers=2, n_heads=8, n_kv_heads=2, inter=384)


@pytest.fixture(scope="module")
def lib():
    return L.lib()


def qk(lib, **kw):
    a = dict(q=FAKE, qs=4096, x=FAKE * 2, xs=6144, qg=FAKE, kg=FAKE, k=FAKE, v=FAKE, np=4, inv=FAKE,
             rope=FAKE, nr=10, pos=FAKE, slot=FAKE, T=3, H=32, KV=8, D=128)
    a.update(kw)
    return lib.heph_qk_norm_rope_pages(a["q"], a["qs"], a["x"], a["xs"], a["qg"], a["kg"], a["k"],
                                       a["v"], a["np"], a["inv"], a["rope"], a["nr"], a["pos"],
                                       a["slot"], a["T"], a["H"], a["KV"], a["D"], 1e-6, None)


@pytest.mark.parametrize("kw,status", [
    *[({f: None}, L.HEPH_ERR_NULL) for f in ("q", "x", "qg", "kg", "k", "v", "inv", "rope", "pos",
                                             "slot")],
    *[({f: ODD}, L.HEPH_ERR_ALIGN) for f in ("q", "x", "qg", "kg", "k", "v", "rope")],
    (dict(qs=4088), L.HEPH_ERR_SHAPE), (dict(xs=6136), L.HEPH_ERR_SHAPE),
    (dict(qs=4100), L.HEPH_ERR_ALIGN), (dict(xs=6150), L.HEPH_ERR_ALIGN),
    (dict(T=0), L.HEPH_ERR_SHAPE), (dict(np=0), L.HEPH_ERR_SHAPE), (dict(nr=0), L.HEPH_ERR_SHAPE),
    (dict(D=64), L.HEPH_ERR_SHAPE), (dict(H=30), L.HEPH_ERR_SHAPE), (dict(KV=0), L.HEPH_ERR_SHAPE),
    (dict(H=130, KV=2, qs=1 << 20, xs=1 << 20), L.HEPH_ERR_SHAPE),
    (dict(q=FAKE * 2), L.HEPH_ERR_SHAPE),                       # in place with another stride
])
def test_qk_rejects(lib, kw, status):
    assert qk(lib, **kw) == status


def attn(lib, **kw):
    sizes = dict(T=3, S=2, G=0, H=32, KV=8)
    sizes.update({f: kw[f] for f in sizes if f in kw})
    a = dict(out=FAKE, q=FAKE * 4, qs=4096, k=FAKE, v=FAKE, np=4, sc=FAKE, table=FAKE, tp=5, plan=FAKE,
             pb=1 << 40, ws=FAKE, wb=1 << 40, D=128, **sizes)
    a.update(kw)
    return lib.heph_pages_attention(a["out"], a["q"], a["qs"], a["k"], a["v"], a["np"], a["sc"],
                                    a["table"], a["tp"], a["plan"], a["pb"], a["ws"], a["wb"],
                                    a["T"], a["S"], a["G"], a["H"], a["KV"], a["D"], None)


@pytest.mark.parametrize("kw,status", [
    *[({f: None}, L.HEPH_ERR_NULL) for f in ("out", "q", "k", "v", "sc", "table", "plan", "ws")],
    *[({f: ODD}, L.HEPH_ERR_ALIGN) for f in ("out", "q", "k", "v", "plan", "ws")],
    (dict(qs=4088), L.HEPH_ERR_SHAPE), (dict(qs=4100), L.HEPH_ERR_ALIGN),
    (dict(out=FAKE * 4), L.HEPH_ERR_SHAPE),                     # q's own buffer
    (dict(T=0), L.HEPH_ERR_SHAPE), (dict(S=0), L.HEPH_ERR_SHAPE),
    (dict(S=1025, T=2000), L.HEPH_ERR_SHAPE), (dict(G=3), L.HEPH_ERR_SHAPE),
    (dict(G=-1), L.HEPH_ERR_SHAPE), (dict(np=0), L.HEPH_ERR_SHAPE), (dict(tp=0), L.HEPH_ERR_SHAPE),
    (dict(tp=4097), L.HEPH_ERR_SHAPE), (dict(D=64), L.HEPH_ERR_SHAPE), (dict(H=36), L.HEPH_ERR_SHAPE),
    (dict(H=65, KV=1, qs=1 << 20), L.HEPH_ERR_SHAPE),
    (dict(pb=16), L.HEPH_ERR_WORKSPACE), (dict(wb=8), L.HEPH_ERR_WORKSPACE),
])
def test_attention_rejects(lib, kw, status):
    assert attn(lib, **kw) == status


def test_attention_plan_rejects(lib):
    def plan(p=FAKE, pb=1 << 40, qs=FAKE, kl=FAKE, gs=None, sh=None, T=3, S_=2, G=0, tp=5, H=32, KV=8):
        return lib.heph_pages_attention_plan(p, pb, qs, kl, gs, sh, T, S_, G, tp, H, KV, None)
    assert plan(p=None) == plan(qs=None) == plan(kl=None) == plan(G=1) == L.HEPH_ERR_NULL
    assert plan(G=1, gs=FAKE) == L.HEPH_ERR_NULL
    assert plan(p=ODD) == L.HEPH_ERR_ALIGN
    assert plan(pb=8) == L.HEPH_ERR_WORKSPACE
    for kw in (dict(T=0), dict(S_=0), dict(G=3, gs=FAKE, sh=FAKE), dict(tp=0), dict(H=33), dict(T=1 << 30)):
        assert plan(**kw) == L.HEPH_ERR_SHAPE, kw
    assert lib.heph_pages_attention_plan_bytes(0, 1, 0, 32, 8) == 0
    assert lib.heph_pages_attention_ws_bytes(1, 0, 0, 32, 8) == 0


def copy(lib, src, dst, k=FAKE, v=FAKE, layers=2, pages=8, kv=4, n=None):
    s, d = np.array(src, np.int32), np.array(dst, np.int32)
    return lib.heph_copy_pages(k, v, layers, pages, kv, s.ctypes.data, d.ctypes.data,
                               len(src) if n is None else n, None)


def test_copy_pages_rejects(lib):
    for src, dst in (([0], [0]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([-1], [0]), ([0], [8]),
                     ([8], [0]), ([0], [-1]), ([0, 1, 2], [4, 5, 0])):
        assert copy(lib, src, dst) == L.HEPH_ERR_SHAPE, (src, dst)
    assert copy(lib, [0], [1], k=None) == L.HEPH_ERR_NULL
    assert lib.heph_copy_pages(FAKE, FAKE, 1, 8, 4, None, FAKE, 1, None) == L.HEPH_ERR_NULL
    assert copy(lib, [0], [1], v=ODD) == L.HEPH_ERR_ALIGN
    for kw in (dict(layers=0), dict(pages=0), dict(kv=0), dict(n=-1)):
        assert copy(lib, [0], [1], **kw) == L.HEPH_ERR_SHAPE, kw
    assert copy(lib, [], []) == L.HEPH_OK


def lora(lib, **kw):
    a = dict(c=FAKE, dt=0, base=FAKE, x=FAKE, a=FAKE, b=FAKE, sc=FAKE, plan=FAKE, pb=1 << 40, ws=FAKE,
             wb=1 << 40, M=4, N=96, K=256, r=16, A=3)
    a.update(kw)
    return lib.heph_lora_add(a["c"], a["dt"], a["base"], a["x"], a["a"], a["b"], a["sc"], a["plan"],
                             a["pb"], a["ws"], a["wb"], a["M"], a["N"], a["K"], a["r"], a["A"], None)


@pytest.mark.parametrize("kw,status", [
    *[({f: None}, L.HEPH_ERR_NULL) for f in ("c", "base", "x", "a", "b", "sc", "plan", "ws")],
    *[({f: ODD}, L.HEPH_ERR_ALIGN) for f in ("c", "base", "x", "a", "b", "plan", "ws")],
    (dict(dt=2), L.HEPH_ERR_DTYPE), (dict(M=0), L.HEPH_ERR_SHAPE), (dict(N=40), L.HEPH_ERR_SHAPE),
    (dict(K=24), L.HEPH_ERR_SHAPE), (dict(r=12), L.HEPH_ERR_SHAPE), (dict(r=136), L.HEPH_ERR_SHAPE),
    (dict(r=0), L.HEPH_ERR_SHAPE), (dict(A=0), L.HEPH_ERR_SHAPE),
    (dict(pb=8), L.HEPH_ERR_WORKSPACE), (dict(wb=8), L.HEPH_ERR_WORKSPACE),
])
def test_lora_rejects(lib, kw, status):
    assert lora(lib, **kw) == status


def test_lora_plan_rejects(lib):
    assert lib.heph_lora_plan(None, 1 << 20, FAKE, 4, 3, None) == L.HEPH_ERR_NULL
    assert lib.heph_lora_plan(FAKE, 1 << 20, None, 4, 3, None) == L.HEPH_ERR_NULL
    assert lib.heph_lora_plan(ODD, 1 << 20, FAKE, 4, 3, None) == L.HEPH_ERR_ALIGN
    assert lib.heph_lora_plan(FAKE, 8, FAKE, 4, 3, None) == L.HEPH_ERR_WORKSPACE
    assert lib.heph_lora_plan(FAKE, 1 << 20, FAKE, 0, 3, None) == L.HEPH_ERR_SHAPE
    assert lib.heph_lora_plan_bytes(0, 3) == 0 and lib.heph_lora_ws_bytes(4, 3, 256, 12) == 0


def test_rope_table_rejects(lib):
    assert lib.heph_rope_table_f32(None, 4, 128, 1e6, None) == L.HEPH_ERR_NULL
    assert lib.heph_rope_table_f32(ODD, 4, 128, 1e6, None) == L.HEPH_ERR_ALIGN
    for n, d, th in ((0, 128, 1e6), (262145, 128, 1e6), (4, 64, 1e6), (4, 128, 0.0), (4, 128, float("nan"))):
        assert lib.heph_rope_table_f32(FAKE, n, d, th, None) == L.HEPH_ERR_SHAPE


def test_valid_calls_without_a_gpu_report_the_device(lib):
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert qk(lib) == attn(lib) == lora(lib) == copy(lib, [0, 0], [1, 2]) == L.HEPH_ERR_DEVICE
    assert lib.heph_lora_plan(FAKE, 1 << 20, FAKE, 4, 3, None) == L.HEPH_ERR_DEVICE


def test_python_rejects_host_tensors(monkeypatch):
    monkeypatch.setattr(S, "_at", lambda ctx: (0, 0))          # (no device to ask here)
    t = torch.zeros(2, 8, 128, dtype=torch.bfloat16)
    k, v = torch.zeros(4, 2, 2, 64, 64, dtype=torch.uint8), torch.zeros(4, 2, 128, 64, dtype=torch.uint8)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        S.qk_norm_rope_pages(t, torch.zeros(2, 12, 128, dtype=torch.bfloat16), t[0, 0], t[0, 0], k, v,
                             torch.ones(4), torch.zeros(4, 64, 2), i, i)
    with pytest.raises(ValueError):
        S.copy_pages(k[None], v[None], [0], [1])
    with pytest.raises(ValueError, match="pools of shapes"):
        S.attention_pages(t, t, k[None], v[None], torch.ones(4), i[None], SimpleNamespace(
            n_seqs=1, table_pages=2, n_tok=2, n_heads=8, n_kv=2))
    with pytest.raises(ValueError):
        plan = S.LoraPlan.__new__(S.LoraPlan)                  # (without its device buffers)
        plan.m, plan.n_adapters = 2, 2
        plan._dev, plan._bound = 0, (0, 0, 0, 0)
        S.lora_add(t[0], t[0], t[0], torch.zeros(2, 8, 128, dtype=torch.bfloat16),
                   torch.zeros(2, 128, 8, dtype=torch.bfloat16), torch.ones(2), plan)
    with pytest.raises(ValueError, match="no rows of 64"):
        S.lora_add(t[0], t[0], t[0], torch.zeros(2, 8, 128, dtype=torch.bfloat16),
                   torch.zeros(2, 64, 8, dtype=torch.bfloat16), torch.ones(2), plan)


def test_plan_refusals(lib):
    for args in ((1, 1, 8, 8, 0), (1, 1, 8, 8, 4097), (0, 1, 8, 8, 4), (1, 0, 8, 8, 4), (1025, 1, 8, 8, 4),
                 (1, 1, 8, 3, 4)):
        with pytest.raises(S.HephError) as e:
            S.AttentionPlan(*args, device="cpu")
        assert e.value.status == L.HEPH_ERR_SHAPE
    for args in ((0, 1, 8, 128), (1, 0, 8, 128), (1, 4097, 8, 128), (1, 1, 12, 128), (1, 1, 136, 128), (1, 1, 8, 8)):
        with pytest.raises(S.HephError):
            S.LoraPlan(*args, device="cpu")
    p = S.AttentionPlan(2, 3, 8, 8, 4, n_groups=1, device="cpu")
    with pytest.raises(ValueError, match="needs group_start"):
        p.update(torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))


def test_attention_buffers_of_extreme_batches(lib):
    plan, ws = lib.heph_pages_attention_plan_bytes, lib.heph_pages_attention_ws_bytes
    for sizes in ((1, 1, 0, 1, 1), (1024, 1024, 1024, 64, 1), (1 << 20, 1024, 3, 4096, 64), (7, 3, 1, 96, 96)):
        T, n_seqs, G, H, KV = sizes
        # at least a token's entry, a row's partial result behind a prefix and its own
        assert plan(*sizes) > 32 * T and ws(*sizes) >= 2 * T * H * (128 * 4 + 8)
    for sizes in ((0, 1, 0, 8, 8), (1, 0, 0, 8, 8), (1, 1025, 0, 8, 8), (1, 1, 2, 8, 8), (1, 1, -1, 8, 8),
                  ((1 << 20) + 1, 1, 0, 8, 8), (1, 1, 0, 130, 2), (1, 1, 0, 4160, 65), (1, 1, 0, 7, 2)):
        assert plan(*sizes) == 0 and ws(*sizes) == 0


def test_v_place_is_a_permutation_that_keeps_runs_of_four():
    p = [S.v_place(j) for j in range(64)]
    assert sorted(p) == list(range(64))
    assert all(p[j] == p[j - j % 4] + j % 4 for j in range(64))


# ---------------------------------------------------------- page bookkeeping ----

@pytest.fixture
def cache(monkeypatch):
    """A cache on the host whose page copies are torch's."""
    c = S.PagedKVCache(CFG, 12, device="cpu")
    c.copies = []

    def copy_pages(k, v, src, dst, ctx=None):
        assert not set(src) & set(dst) and len(set(dst)) == len(dst)
        c.copies.append((list(src), list(dst)))
        k[:, dst], v[:, dst] = k[:, src], v[:, src]
    monkeypatch.setattr(S, "copy_pages", copy_pages)
    return c


def check_counts(c):
    users = [0] * c.n_pages
    for s in c._seqs:
        assert len(s.pages) == -(-s.length // 64) and len(set(s.pages)) == len(s.pages)
        for p in s.pages:
            users[p] += 1
    assert users == c._users
    assert sorted(c._free) == [p for p in range(c.n_pages) if not users[p]]


def write(c, slots, value):
    for s in slots:
        c.k[:, s // 64, :, :, s % 64] = value
        c.v[:, s // 64, :, :, S.v_place(s % 64)] = value


def read(c, seq):
    k = [int(c.k[0, seq.pages[j // 64], 0, 0, j % 64, 0]) for j in range(seq.length)]
    v = [int(c.v[1, seq.pages[j // 64], 1, 5, S.v_place(j % 64)]) for j in range(seq.length)]
    assert k == v
    return k


def test_extend_fork_free_compact(cache):
    c = cache
    a = c.new()
    slots = c.extend(a, 100)
    assert slots == list(range(100)) and c.free_pages == 10
    write(c, slots, 1)
    b, d = c.fork(a, 2)
    assert c.copies == [([1, 1], [2, 3])] and b.pages == [0, 2] and d.pages == [0, 3]
    check_counts(c)
    write(c, c.extend(b, 30), 2)
    write(c, c.extend(d, 60), 3)
    write(c, c.extend(a, 1), 4)
    assert read(c, a) == [1] * 100 + [4]
    assert read(c, b) == [1] * 100 + [2] * 30 and read(c, d) == [1] * 100 + [3] * 60
    c.free(a)
    check_counts(c)
    assert c.free_pages == 12 - 6 + 1 and 0 not in c._free         # page 0 is still shared
    c.free(b)
    moved = c.compact()
    check_counts(c)
    assert moved == 2 and sorted(d.pages) == [0, 1, 2] and read(c, d) == [1] * 100 + [3] * 60
    assert c.compact() == 0
    c.free(d)
    assert c.free_pages == 12


def test_fork_of_full_pages_and_of_nothing(cache):
    c = cache
    a = c.new()
    e, = c.fork(a)
    assert e.pages == [] and c.copies == []
    c.extend(a, 128)
    f, g = c.fork(a, 2)
    assert f.pages == a.pages == g.pages and c.copies == []
    assert c.fork(a, 0) == []
    c.extend(f, 1)
    assert f.pages[:2] == a.pages and len(f.pages) == 3
    check_counts(c)


def test_bookkeeping_refusals(cache):
    c = cache
    a = c.new()
    with pytest.raises(MemoryError):
        c.extend(a, 12 * 64 + 1)
    assert a.length == 0 and a.pages == []
    c.extend(a, 11 * 64 + 5)
    with pytest.raises(MemoryError):
        c.fork(a)
    check_counts(c)
    with pytest.raises(ValueError):
        c.extend(a, -1)
    with pytest.raises(ValueError):
        c.fork(a, -1)
    c.free(a)
    for f in (c.free, c.fork, lambda s: c.extend(s, 1)):
        with pytest.raises(ValueError):
            f(a)
    with pytest.raises(ValueError):
        S.PagedKVCache(CFG, 0, device="cpu")


def test_a_fork_whose_copy_fails_changes_nothing(cache, monkeypatch):
    c = cache
    a = c.new()
    c.extend(a, 70)

    def fails(*args):
        raise S.HephError(L.HEPH_ERR_LAUNCH, "heph_copy_pages")
    monkeypatch.setattr(S, "copy_pages", fails)
    with pytest.raises(S.HephError):
        c.fork(a, 3)
    assert len(c._seqs) == 1 and c.free_pages == 10
    check_counts(c)


def test_step_refusals_leave_the_sequences(cache, monkeypatch):
    c = cache
    w = SimpleNamespace(cfg=CFG, embed=SimpleNamespace(block=True, w=torch.zeros(1)),
                        layers=[None] * CFG.n_layers)
    monkeypatch.setattr(S, "rope_table_f32", lambda n, theta, device: torch.zeros(n, 64, 2))
    lora = S.LoraWeights(torch.ones(3), [{}] * CFG.n_layers)
    d = S.Qwen3BatchDecoder(w, c, n_pos=300, lora=lora)
    a, b, other = c.new(), c.new(), S.PagedKVCache(CFG, 2, device="cpu").new()
    c.extend(a, 70)
    for tokens, seqs, adapters, error in (
            ([], [], None, ValueError), ([[1]], [a, b], None, ValueError),
            ([[1], []], [a, b], None, ValueError), ([[1], [2]], [a, a], None, ValueError),
            ([[1]], [other], None, ValueError), ([[512]], [a], None, ValueError),
            ([[1, -1]], [a], None, ValueError), ([[1]], [a], [0, 1], ValueError),
            ([[1]], [a], [3], ValueError), ([[1]], [a], [-2], ValueError),
            ([[0] * 231], [a], None, ValueError),                     # past the rotation table
            ([[0] * 230, [0] * 290], [a, b], [0, -1], None)):         # fails in its first launch
        def launches(*args):
            raise S.HephError(L.HEPH_ERR_LAUNCH, "step")
        monkeypatch.setattr(d, "_run", lambda t, s, ad: ([c.extend(i, len(j)) for i, j in zip(s, t)],
                                                         launches()))
        with pytest.raises(error or S.HephError):
            d.step(tokens, seqs, adapters)
        assert (a.length, b.length, len(a.pages), b.pages, c.free_pages) == (70, 0, 2, [], 10)
        check_counts(c)
    c.extend(b, 10 * 64)
    with pytest.raises(MemoryError):
        d.step([[0] * 100], [a])
    check_counts(c)


def test_random_use_keeps_every_sequence(cache):
    c, rng, want = cache, np.random.default_rng(0), {}
    value = 0
    for step in range(300):
        what, seqs = rng.integers(0, 5), list(c._seqs)
        if what == 0 or not seqs:
            s = c.new()
            want[id(s)] = []
            continue
        s = seqs[rng.integers(len(seqs))]
        try:
            if what == 1:
                n = int(rng.integers(0, 90))
                value = value % 100 + 1
                write(c, c.extend(s, n), value)
                want[id(s)] = want[id(s)] + [value] * n
            elif what == 2:
                for f in c.fork(s, int(rng.integers(0, 3))):
                    want[id(f)] = list(want[id(s)])
            elif what == 3:
                c.free(s)
                # (keep the object: ids are not reused)
                want[id(s)], want[("kept", step)] = [], s
            else:
                c.compact()
        except MemoryError:
            pass
        check_counts(c)
        for t in c._seqs:
            assert read(c, t) == want[id(t)]


def test_groups_of_sequences():
    def seq(*pages):
        s = S.Sequence()
        s.pages = list(pages)
        return s
    assert S._groups([seq(1)]) == ([0, 1], [0])
    assert S._groups([seq(1, 2, 3), seq(1, 2, 4), seq(1, 2, 5, 6)]) == ([0, 3], [2])
    assert S._groups([seq(1, 2), seq(3, 4), seq(3, 5), seq()]) == ([0, 1, 3, 4], [0, 1, 0])
    # a long common prefix is not given up for a member that shares little of it
    assert S._groups([seq(*range(9)), seq(*range(9)), seq(0, 20)]) == ([0, 2, 3], [9, 0])


def test_group_lists_fit_the_plan():
    rng = np.random.default_rng(1)
    for _ in range(50):
        seqs = []
        for _ in range(int(rng.integers(1, 12))):
            s = S.Sequence()
            s.pages = [int(rng.integers(0, 2)) * 100 + j for j in range(int(rng.integers(0, 6)))]
            seqs.append(s)
        start, shared = S._groups(seqs)
        assert start[0] == 0 and start[-1] == len(seqs) and len(shared) == len(start) - 1 <= len(seqs)
        for g, n in enumerate(shared):
            rows = [s.pages[:n] for s in seqs[start[g]:start[g + 1]]]
            assert all(r == rows[0] and len(r) == n for r in rows)


def test_ctypes_signatures_of_the_serving_ops():
    for name, nargs in (("heph_qk_norm_rope_pages", 20), ("heph_pages_attention", 20),
                        ("heph_pages_attention_plan", 13), ("heph_copy_pages", 9),
                        ("heph_lora_add", 17)):
        assert len(L.SIGNATURES[name][1]) == nargs
        assert getattr(L.lib(), name).restype is ctypes.c_int


# --------------------------------------------------------- the decoder's host side ----

def host_decoder(cache, monkeypatch, lora=None, n_pos=300):
    """A decoder without device memory: what a step does before its first launch."""
    H, I, Q, KV = CFG.hidden, CFG.inter, CFG.q_out, CFG.kv_out

    def weight(n, k):
        return SimpleNamespace(N=n, K=k)
    layer = SimpleNamespace(qkv=weight(Q + 2 * KV, H), o=weight(H, Q), gate_up=weight(2 * I, H),
                            down=weight(H, I))
    w = SimpleNamespace(cfg=CFG, embed=SimpleNamespace(block=True, w=torch.zeros(1)),
                        layers=[layer] * CFG.n_layers)
    monkeypatch.setattr(S, "rope_table_f32", lambda n, theta, device: torch.zeros(n, 64, 2))
    return S.Qwen3BatchDecoder(w, cache, n_pos=n_pos, lora=lora)


def pair(n, k, rank=16, n_adapters=3):
    return (torch.zeros(n_adapters, rank, k, dtype=torch.bfloat16),
            torch.zeros(n_adapters, n, rank, dtype=torch.bfloat16))


def test_lora_weights_that_no_projection_takes_are_refused(cache, monkeypatch):
    H, I, Q, KV = CFG.hidden, CFG.inter, CFG.q_out, CFG.kv_out
    good = {"qkv": pair(Q + 2 * KV, H), "o": pair(H, Q), "gate_up": pair(2 * I, H, rank=8),
            "down": pair(H, I)}
    scale = torch.ones(3)
    lora = S.LoraWeights(scale, [good, {}])
    assert (lora.n_adapters, lora.max_rank, lora.max_k) == (3, 16, max(Q, I))
    host_decoder(cache, monkeypatch, lora)
    for name in ("q", "q_proj", "gate", "up_proj", "Down", ""):
        with pytest.raises(ValueError, match="no projection"):
            S.LoraWeights(scale, [{}, {name: pair(H, I)}])
    a, b = pair(H, I)
    for bad in (pair(H, I, n_adapters=2), (a, b[:2]), (a[:, :8], b), pair(H, I, rank=12), pair(H, I, rank=136), (a[0], b), (a, b[0]), (b, a)):
        with pytest.raises(ValueError, match="layer 1, down"):
            S.LoraWeights(scale, [good, {"down": bad}])
    # sizes of another projection or of another model, before any step
    for name, wrong in (("qkv", pair(H, Q)), ("qkv", pair(Q, H)), ("o", pair(Q, H)),
                        ("gate_up", pair(I, H)), ("down", pair(H, I // 2))):
        lora = S.LoraWeights(scale, [good, dict(good, **{name: wrong})])
        with pytest.raises(ValueError, match=f"layer 1, {name}"):
            host_decoder(cache, monkeypatch, lora)


def chain(*shared_with_the_first):
    """Sequences of 64 pages; number i shares that many with the first one."""
    out = []
    for i, n in enumerate(shared_with_the_first):
        s = S.Sequence()
        s.pages = list(range(n)) + [1000 * (i + 1) + j for j in range(64 - n)]
        out.append(s)
    return out


def test_groups_do_not_shrink_step_by_step():
    # every neighbour halves the common prefix: the group ends at half of its first two's pages
    start, shared = S._groups(chain(*[64] * 32, 32, 16, 8, 4, 2, 1))
    assert start[:2] == [0, 33] and shared[0] == 32
    assert S._groups(chain(64, 40, 20, 19, 64)) == ([0, 3, 5], [20, 19])
    assert S._groups(chain(64, 41, 20)) == ([0, 2, 3], [41, 0])
    rng = np.random.default_rng(2)
    for _ in range(50):
        seqs = chain(*(int(n) for n in rng.integers(0, 65, 12)))
        start, shared = S._groups(seqs)
        for a, b, n in zip(start, start[1:], shared):
            rows = [s.pages for s in seqs[a:b]]
            first_two = next(i for i in range(65) if i == 64 or rows[0][i] != rows[1][i]) if b - a > 1 else 0
            assert all(r[:n] == rows[0][:n] for r in rows) and 2 * n >= first_two


@pytest.mark.parametrize("error", [KeyboardInterrupt, MemoryError])
def test_an_interrupted_step_or_fork_changes_nothing(cache, monkeypatch, error):
    c = cache
    d = host_decoder(c, monkeypatch)
    a, b = c.new(), c.new()
    c.extend(a, 70)

    def stops(*args):
        raise error()
    monkeypatch.setattr(d, "_run", lambda t, s, ad: ([c.extend(i, len(j)) for i, j in zip(s, t)], stops()))
    with pytest.raises(error):
        d.step([[1] * 100, [2]], [a, b])
    monkeypatch.setattr(S, "copy_pages", stops)
    with pytest.raises(error):
        c.fork(a, 2)
    assert (a.length, b.length, len(c._seqs), c.free_pages) == (70, 0, 2, 10)
    check_counts(c)


def test_layout_of_a_step(cache, monkeypatch):
    c = cache
    d = host_decoder(c, monkeypatch)
    a, b = c.new(), c.new()
    c.extend(a, 130)
    f, = c.fork(a)
    got = [np.asarray(p).tolist() for p in d._layout([[7], [8, 9], [1] * 3], [a, f, b], [2, -1, 0])]
    p, q, r = a.pages, f.pages, b.pages
    assert p[:2] == q[:2] and len(p) == len(q) == 3 and len(r) == 1
    assert got == [[7, 8, 9, 1, 1, 1], [130, 130, 131, 0, 1, 2],
                   [p[2] * 64 + 2, q[2] * 64 + 2, q[2] * 64 + 3] + [r[0] * 64 + i for i in range(3)],
                   [0, 1, 3, 6], [131, 132, 3], [0, 2, 3], [2, 0], [2, -1, -1, 0, 0, 0],
                   [p, q, r + [-1, -1]]]
    assert [len(x) for x in d._layout([[1]], [b], None)] == [1, 1, 1, 2, 1, 2, 1, 1, 1]
    check_counts(c)


def test_a_step_of_many_sequences_costs_the_host_in_proportion(monkeypatch):
    # eight times the sequences: eight times the time, not 64 (copies of a growing page table
    # took 98 times, 787 ms)
    def host_time(n_seqs, pages=312):
        # one kv head of one layer: the pools are untouched zeros
        c = S.PagedKVCache(Qwen3Config(vocab=512, hidden=128, n_layers=1, n_heads=1, n_kv_heads=1, inter=128),
                           n_seqs * 2 + pages, device="cpu")
        d = host_decoder(c, monkeypatch, n_pos=64 * 400)
        root = c.new()
        c.extend(root, 64 * (pages - 1))
        seqs = c.fork(root, n_seqs)
        best = 1e9
        for _ in range(3):
            monkeypatch.setattr(d, "_run", d._layout)
            t = time.process_time()
            d.step([[1]] * n_seqs, seqs)
            best = min(best, time.process_time() - t)
        return best
    assert host_time(1024) < 30 * host_time(128)


def test_common_pages():
    rng = np.random.default_rng(3)
    for _ in range(300):
        n, a, b = (int(x) for x in rng.integers(0, 9, 3))
        x, y = list(range(n)) + [100] * a, list(range(n)) + [200] * b
        assert S._common(x, y) == n
        assert S._common(x, x[:n]) == n and S._common(x, x + y) == len(x)


@pytest.mark.parametrize("tokens,adapters", [([[1.5]], None), ([[1, 2.0]], None), ([[3]], [0.5]), ([["1"]], None)])
def test_a_step_takes_whole_numbers_only(cache, monkeypatch, tokens, adapters):
    c = cache
    d = host_decoder(c, monkeypatch, lora=S.LoraWeights(torch.ones(3), [{}] * CFG.n_layers))
    monkeypatch.setattr(d, "_run", lambda *a: [np.asarray(p) for p in d._layout(*a)])
    a = c.new()
    c.extend(a, 70)
    with pytest.raises(TypeError):
        d.step(tokens, [a], adapters)
    assert (a.length, len(a.pages), c.free_pages) == (70, 2, 10)
    check_counts(c)
    tok, *_, ids, table = d.step([[np.int64(5), torch.tensor(6)]], [a], [np.int32(2)])
    assert tok.tolist() == [5, 6] and ids.tolist() == [2, 2] and tok.dtype == ids.dtype == table.dtype == np.int32
