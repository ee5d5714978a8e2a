"""The refusals of the cache with scales of its own and of the pick, without a GPU."""
import ctypes

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


def write(lib, **kw):
    a = dict(q=FAKE, qs=4096, x=FAKE * 2, xs=6144, qg=FAKE, kg=FAKE, k=FAKE, v=FAKE, np=4, sc=FAKE,
             rope=FAKE, nr=10, pos=FAKE, slot=FAKE, T=3, H=32, KV=8, D=128)
    a.update(kw)
    return lib.heph_qk_norm_rope_pages_scaled(a["q"], a["qs"], a["x"], a["xs"], a["qg"], a["kg"], a["k"],
                                              a["v"], a["np"], a["sc"], a["rope"], a["nr"], a["pos"],
                                              a["slot"], a["T"], a["H"], a["KV"], a["D"], 1e-6, None)


@pytest.mark.parametrize("kw,status", [
    *[({f: None}, L.HEPH_ERR_NULL) for f in ("q", "x", "qg", "kg", "k", "v", "sc", "rope", "pos", "slot")],
    *[({f: ODD}, L.HEPH_ERR_ALIGN) for f in ("q", "x", "qg", "kg", "k", "v", "rope")],
    (dict(sc=FAKE + 2), L.HEPH_ERR_ALIGN),
    (dict(qs=4088), L.HEPH_ERR_SHAPE), (dict(xs=6136), L.HEPH_ERR_SHAPE),
    (dict(qs=4100), L.HEPH_ERR_ALIGN), (dict(xs=6150), L.HEPH_ERR_ALIGN),
    (dict(T=0), L.HEPH_ERR_SHAPE), (dict(np=0), L.HEPH_ERR_SHAPE), (dict(np=1 << 25), L.HEPH_ERR_SHAPE),
    (dict(nr=0), L.HEPH_ERR_SHAPE), (dict(D=64), L.HEPH_ERR_SHAPE), (dict(H=30), L.HEPH_ERR_SHAPE),
    (dict(KV=0), L.HEPH_ERR_SHAPE), (dict(H=130, KV=2, qs=1 << 20, xs=1 << 20), L.HEPH_ERR_SHAPE),
    (dict(q=FAKE * 2), L.HEPH_ERR_SHAPE),                       # in place with another stride
])
def test_write_rejects(lib, kw, status):
    assert write(lib, **kw) == status


def read(lib, **kw):
    a = dict(ko=FAKE, vo=FAKE * 2, k=FAKE, v=FAKE, np=4, kv=None, sc=FAKE, slot=FAKE, n=3, KV=8, D=128)
    a.update(kw)
    return lib.heph_read_pages(a["ko"], a["vo"], a["k"], a["v"], a["np"], a["kv"], a["sc"], a["slot"], a["n"],
                               a["KV"], a["D"], None)


@pytest.mark.parametrize("kw,status", [
    *[({f: None}, L.HEPH_ERR_NULL) for f in ("ko", "vo", "k", "v", "sc", "slot")],
    *[({f: ODD}, L.HEPH_ERR_ALIGN) for f in ("ko", "vo", "k", "v")],
    (dict(kv=FAKE), L.HEPH_ERR_SHAPE), (dict(vo=FAKE), L.HEPH_ERR_SHAPE), (dict(np=0), L.HEPH_ERR_SHAPE),
    (dict(np=1 << 25), L.HEPH_ERR_SHAPE), (dict(n=0), L.HEPH_ERR_SHAPE), (dict(KV=0), L.HEPH_ERR_SHAPE),
    (dict(KV=5000), L.HEPH_ERR_SHAPE), (dict(D=64), L.HEPH_ERR_SHAPE),
    (dict(n=2 ** 31 - 1, KV=4096), L.HEPH_ERR_UNSUPPORTED),
])
def test_read_rejects(lib, kw, status):
    assert read(lib, **kw) == status


def attn(lib, **kw):
    a = dict(out=FAKE, q=FAKE * 4, qs=4096, k=FAKE, v=FAKE, np=4, sc=FAKE, table=FAKE, tp=5, plan=FAKE,
             pb=1 << 40, ws=FAKE, wb=1 << 40, T=3, S=2, G=0, H=32, KV=8, D=128)
    a.update(kw)
    return lib.heph_pages_attention_scaled(*(a[f] for f in (
        "out", "q", "qs", "k", "v", "np", "sc", "table", "tp", "plan", "pb", "ws", "wb", "T", "S", "G", "H",
        "KV", "D")), None)


@pytest.mark.parametrize("kw,status", [
    *[({f: None}, L.HEPH_ERR_NULL) for f in ("out", "q", "k", "v", "sc", "table", "plan", "ws")],
    *[({f: ODD}, L.HEPH_ERR_ALIGN) for f in ("out", "q", "k", "v", "plan", "ws")],
    (dict(qs=4088), L.HEPH_ERR_SHAPE), (dict(qs=4100), L.HEPH_ERR_ALIGN), (dict(out=FAKE * 4), L.HEPH_ERR_SHAPE),
    (dict(T=0), L.HEPH_ERR_SHAPE), (dict(S=0), L.HEPH_ERR_SHAPE), (dict(S=1025, T=2000), L.HEPH_ERR_SHAPE),
    (dict(G=3), L.HEPH_ERR_SHAPE), (dict(np=0), L.HEPH_ERR_SHAPE), (dict(tp=4097), L.HEPH_ERR_SHAPE),
    (dict(D=64), L.HEPH_ERR_SHAPE), (dict(H=36), L.HEPH_ERR_SHAPE),
    (dict(pb=16), L.HEPH_ERR_WORKSPACE), (dict(wb=8), L.HEPH_ERR_WORKSPACE),
])
def test_attention_rejects(lib, kw, status):
    assert attn(lib, **kw) == status


def test_copy_rejects(lib):
    def copy(src, dst, scale=FAKE, n=None):
        s, d = np.array(src, np.int32), np.array(dst, np.int32)
        return lib.heph_copy_pages_scaled(FAKE, FAKE, scale, 2, 8, 4, s.ctypes.data, d.ctypes.data,
                                          len(src) if n is None else n, None)
    assert copy([0], [1], scale=None) == L.HEPH_ERR_NULL
    assert copy([0], [1], scale=FAKE + 2) == L.HEPH_ERR_ALIGN
    for src, dst in (([0], [0]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([-1], [0]), ([0], [8])):
        assert copy(src, dst) == L.HEPH_ERR_SHAPE
    assert copy([], []) == L.HEPH_OK


def rules(**kw):
    a = dict(n_slots=4, max_tokens=10, max_bias=2, history=FAKE, length=FAKE, n_prompt=FAKE, penalties=FAKE,
             bias_ids=FAKE, bias=FAKE, n_bias=FAKE)
    a.update(kw)
    return L.TokenRulesArgs(**a)


def pick(lib, rules=rules(), **kw):
    a = dict(t=FAKE, lp=FAKE, out=None, os=0, x=FAKE * 2, xs=500, dt=1, rows=3, vocab=500, slots=FAKE, m=None,
             nm=0, mi=None, fl=0, ws=FAKE, wb=1 << 30)
    a.update(kw)
    return lib.heph_pick_tokens(a["t"], a["lp"], a["out"], a["os"], a["x"], a["xs"], a["dt"], a["rows"],
                                a["vocab"], None if rules is None else ctypes.byref(rules), a["slots"], a["m"],
                                a["nm"], a["mi"], a["fl"], a["ws"], a["wb"], None)


@pytest.mark.parametrize("kw,status", [
    (dict(x=None), L.HEPH_ERR_NULL), (dict(ws=None), L.HEPH_ERR_NULL), (dict(t=None), L.HEPH_ERR_NULL),
    (dict(fl=1, rules=None), L.HEPH_ERR_NULL), (dict(fl=1, slots=None), L.HEPH_ERR_NULL),
    (dict(fl=1, t=None, out=FAKE, os=500), L.HEPH_ERR_NULL),
    *[(dict(rules=rules(**{f: None})), L.HEPH_ERR_NULL) for f in ("history", "length", "n_prompt", "penalties",
                                                                 "bias_ids", "bias", "n_bias")],
    (dict(fl=2), L.HEPH_ERR_FLAGS), (dict(dt=2), L.HEPH_ERR_DTYPE),
    (dict(rows=0), L.HEPH_ERR_SHAPE), (dict(rows=(1 << 20) + 1), L.HEPH_ERR_SHAPE), (dict(vocab=0), L.HEPH_ERR_SHAPE),
    (dict(vocab=(1 << 24) + 1, xs=1 << 30), L.HEPH_ERR_SHAPE), (dict(xs=499), L.HEPH_ERR_SHAPE),
    (dict(out=FAKE, os=499), L.HEPH_ERR_SHAPE), (dict(out=FAKE * 2, os=501), L.HEPH_ERR_SHAPE),
    (dict(m=FAKE, mi=FAKE), L.HEPH_ERR_SHAPE),
    *[(dict(rules=rules(**kw)), L.HEPH_ERR_SHAPE) for kw in (dict(n_slots=0), dict(max_tokens=0), dict(max_bias=-1),
                                                            dict(max_tokens=262145), dict(max_bias=4096))],
    (dict(x=FAKE + 2), L.HEPH_ERR_ALIGN), (dict(out=FAKE + 1, os=500), L.HEPH_ERR_ALIGN),
    (dict(x=FAKE + 1, dt=0), L.HEPH_ERR_ALIGN), (dict(ws=ODD), L.HEPH_ERR_ALIGN),
    (dict(wb=8), L.HEPH_ERR_WORKSPACE),
    (dict(rows=1 << 20, vocab=1 << 24, xs=1 << 24, wb=1 << 60), L.HEPH_ERR_UNSUPPORTED),
])
def test_pick_rejects(lib, kw, status):
    assert pick(lib, **kw) == status


def test_pick_sizes(lib):
    ws = lib.heph_pick_ws_bytes
    assert ws(0, 5) == ws(5, 0) == ws((1 << 20) + 1, 5) == ws(5, (1 << 24) + 1) == 0
    assert ws(1, 1) > 0 and ws(100, 151936) >= 100 * 16


def test_valid_calls_without_a_gpu_report_the_device(lib):
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert write(lib) == read(lib) == attn(lib) == pick(lib) == L.HEPH_ERR_DEVICE
    # nothing of rules that no slots ask for is looked at; biases only where there are any
    none = dict(history=None, length=None, n_slots=0, max_bias=-5)
    assert pick(lib, rules=rules(**none), slots=None) == pick(lib, rules=None) == L.HEPH_ERR_DEVICE
    assert pick(lib, rules=rules(max_bias=0, bias_ids=None, bias=None, n_bias=None)) == L.HEPH_ERR_DEVICE
    assert pick(lib, t=None, out=FAKE * 2, os=500) == pick(lib, lp=None) == L.HEPH_ERR_DEVICE
    assert read(lib, kv=FAKE, sc=None) == L.HEPH_ERR_DEVICE


# ------------------------------------------------------------------ python ----

def test_rules_refuse():
    for args in ((0, 5, 5), (1, 0, 5), (1, 5, 0), (1, 5, 262145), (1, 5, 5, -1), (1, 5, 5, 4096)):
        with pytest.raises(ValueError):
            S.TokenRules(*args, device="cpu")
    r = S.TokenRules(2, 50, 4, 1, device="cpu")
    for args, kw in (((2,), {}), ((-1,), {}), ((0, [1] * 5), {}), ((0, [1, 2], [3, 4, 5]), {}), ((0, [50]), {}),
                     ((0, [-1]), {}), ((0,), dict(repetition=0)), ((0,), dict(repetition=-1)),
                     ((0,), dict(repetition=float("nan"))), ((0,), dict(presence=float("inf"))),
                     ((0,), dict(frequency=float("nan"))), ((0,), dict(bias={50: 1.0})),
                     ((0,), dict(bias={1: float("nan")})), ((0,), dict(bias={1: float("inf")})),
                     ((0,), dict(bias={1: 0.0, 2: 0.0}))):
        with pytest.raises(ValueError):
            r.set(*args, **kw)
    with pytest.raises(TypeError):
        r.set(0, [1.5])
    assert (r.length == 0).all() and (r.penalties == torch.tensor([1.0, 0, 0])).all()
    r.set(1, [1, 2], [3], 1.5, 0.1, 0.2, {4: -float("inf")})
    assert r.length.tolist() == [0, 3] and r.n_prompt.tolist() == [0, 2] and r.n_bias.tolist() == [0, 1]


def test_host_tensors_are_refused(monkeypatch):
    monkeypatch.setattr(S, "_at", lambda ctx: (0, 0))          # (no device to ask here)
    x, t = torch.zeros(2, 50), torch.zeros(2, dtype=torch.int32)
    k, v = torch.zeros(4, 2, 2, 64, 64, dtype=torch.uint8), torch.zeros(4, 2, 128, 64, dtype=torch.uint8)
    rows = torch.zeros(2, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        S.pick_tokens(t, x)
    with pytest.raises(ValueError):
        S.read_pages(rows, rows, k, v, t, page_scale=torch.ones(4, 4))
    with pytest.raises(ValueError):
        S.copy_pages(k[None], v[None], [0], [1], page_scale=torch.ones(1, 4, 4))
    with pytest.raises(ValueError):
        S.qk_norm_rope_pages_scaled(rows, torch.zeros(2, 6, 128, dtype=torch.bfloat16), rows[0, 0], rows[0, 0], k, v,
                                    torch.ones(4, 4), torch.zeros(4, 64, 2), t, t)


def test_fork_and_compaction_take_the_scales_with_them(monkeypatch):
    c = S.PagedKVCache(CFG, 12, device="cpu", page_scales=True)
    assert c.scale is None and c.inv is None and c.page_scale.shape == (2, 12, 4)

    def copy_pages(k, v, src, dst, ctx=None, page_scale=None):
        for t in (k, v, page_scale):
            t[:, dst] = t[:, src]
    monkeypatch.setattr(S, "copy_pages", copy_pages)
    a = c.new()
    c.extend(a, 100)
    c.page_scale[:] = torch.arange(12.0)[:, None]
    b, = c.fork(a)
    assert (c.page_scale[:, b.pages[1]] == 1).all()
    c.free(a)
    c.compact()
    assert (c.page_scale[:, b.pages[0]] == 0).all() and (c.page_scale[:, b.pages[1]] == 1).all()
    assert b.pages == [0, 1]


def test_next_tokens_that_fail_leave_the_sequences(monkeypatch):
    from types import SimpleNamespace
    c = S.PagedKVCache(CFG, 12, device="cpu", page_scales=True)
    w = SimpleNamespace(cfg=CFG, embed=SimpleNamespace(block=True, w=torch.zeros(1)), layers=[None] * CFG.n_layers)
    monkeypatch.setattr(S, "rope_table_f32", lambda n, theta, device: torch.zeros(n, 64, 2))
    d = S.Qwen3BatchDecoder(w, c, n_pos=300)
    a, b = c.new(), c.new()
    c.extend(a, 60)

    def run(tokens, seqs, adapters):
        d._layout(tokens, seqs, adapters)
        return torch.zeros(len(seqs), CFG.vocab)
    monkeypatch.setattr(d, "_run", run)

    def fails(*args, **kw):
        raise S.HephError(L.HEPH_ERR_LAUNCH, "heph_pick_tokens")
    monkeypatch.setattr(S, "pick_tokens", fails)
    with pytest.raises(S.HephError):
        d.next_tokens([[1] * 70, [2]], [a, b])
    assert (a.length, len(a.pages), b.length, b.pages) == (60, 1, 0, []) and c.free_pages == 11
    rules = S.TokenRules(2, CFG.vocab, 5, device="cpu")
    words = torch.zeros(1, CFG.vocab // 32, dtype=torch.int32)
    for kw in (dict(rules=rules), dict(slots=[0, 1]), dict(rules=rules, slots=[0]), dict(rules=rules, slots=[1, 1]),
               dict(rules=rules, slots=[0, 2]), dict(masks=words), dict(masks=words, mask_ids=[0]),
               dict(masks=words, mask_ids=[0, 1]), dict(masks=words[:, 1:], mask_ids=[0, 0]),
               dict(rules=S.TokenRules(2, 7, 5, device="cpu"), slots=[0, 1])):
        with pytest.raises(ValueError):
            d.next_tokens([[1], [2]], [a, b], **kw)
    assert (a.length, b.length, c.free_pages) == (60, 0, 11)


def test_what_a_call_allocates_is_its_streams(monkeypatch):
    """Scratch, slots and rows of a call with ctx are allocated and uploaded on that stream."""
    on = []

    class On:
        def __init__(self, stream):
            self.stream = stream

        def __enter__(self):
            on.append(self.stream)

        def __exit__(self, *exc):
            on.pop()
    monkeypatch.setattr(torch.cuda, "stream", On)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda handle: handle)
    monkeypatch.setattr(torch.cuda, "default_stream", lambda: 0)
    monkeypatch.setattr(S, "_at", lambda ctx: (0, ctx))
    made = []

    def watched(f):
        def make(*args, **kw):
            made.append(list(on))
            return f(*args, **kw)
        return make
    for name in ("empty", "tensor"):
        monkeypatch.setattr(torch, name, watched(getattr(torch, name)))
    c = S.PagedKVCache(CFG, 4, device="cpu")
    seq = c.new()
    c.extend(seq, 70)
    for ctx, want in ((77, [77]), (0, [0]), (None, [])):
        with pytest.raises(ValueError):                # (host tensors: refused behind the allocations)
            c.read(seq, 0, ctx=ctx)
        assert made == [want] * 3
        made.clear()
        with pytest.raises(ValueError):
            S.rope_table_f32(10, device="cpu", ctx=ctx)
        assert made == [want]
        made.clear()
        monkeypatch.setattr(S, "_rows", lambda t, *args: (FAKE, 512))
        with pytest.raises(ValueError):
            S.pick_tokens(torch.zeros(2, dtype=torch.int32), torch.zeros(2, 512), ctx=ctx)
        assert made == [want]
        made.clear()


def test_rules_refuse_what_f32_does_not_hold():
    r = S.TokenRules(1, 50, 4, 2, device="cpu")
    for kw in (dict(repetition=1e-50), dict(repetition=1e39), dict(presence=1e39), dict(frequency=-1e39),
               dict(bias={3: 1e39}), dict(bias={3: 1.0, 4: 3.5e38})):
        with pytest.raises(ValueError):
            r.set(0, [1], **kw)
    assert (r.length == 0).all() and (r.penalties == torch.tensor([1.0, 0, 0])).all()
    r.set(0, [1], repetition=1e-38, presence=3e38, bias={3: -1e39, 4: 1e-50})
    assert r.penalties.tolist() == [[float(np.float32(1e-38)), float(np.float32(3e38)), 0.0]]
    assert r.bias.tolist() == [[-float("inf"), 0.0]]
