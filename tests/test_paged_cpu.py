"""CPU: what the launchers and entry points of the paged cache and of draft verification refuse before they launch anything, and
the plain forms that their GPU tests compare with."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import cvattn as cv
from cvattn import _lib
from paged_reference import E4M3, PLACE, VALUES, Pool, assign, attention, nearest, verify

D = 64


class Device(torch.Tensor):
    """A host tensor that says it is a CUDA tensor: launchers can be built on it, not called."""
    is_cuda = property(lambda self: True)


def dev(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype).as_subclass(Device)


def i32(*shape):
    return dev(*shape, dtype=torch.int32)


def pool(pages=6, size=32, heads=2, fmt=cv.PAGE_I8):
    u8 = lambda: dev(pages, heads, size * D, dtype=torch.uint8)  # noqa: E731
    return cv.PagePool(u8(), u8(), dev(pages, heads, size // 16), dev(pages, heads, size // 16), fmt)


def append_arguments(S=2):
    return {"pool": pool(), "k": dev(S, 3, 2 * D), "v": dev(S, 3, 2 * D), "table": i32(S, 4), "kv_len": i32(S)}


def read_arguments(S=2):
    return {"pool": pool(), "k": dev(S, 3, 2 * D), "v": dev(S, 3, 2 * D), "table": i32(S, 4)}


def attention_arguments(S=2):
    return {"pool": pool(), "q": dev(S, 3, 14, D), "out": dev(S, 3, 14, D), "table": i32(S, 4), "kv_len": i32(S),
            "workspace": dev(max(1, cv.paged_attention_workspace_size(S, 3, 128, 14, 2)), dtype=torch.uint8)}


def assign_arguments(S=2):
    return {"pools": [pool()], "table": i32(S, 4), "keep": i32(S), "need": i32(S), "room": i32(S), "workspace": dev(4096, dtype=torch.uint8)}


def compact_arguments(S=2):
    return {"pools": [pool()], "table": i32(S, 4), "n_live": i32(1), "workspace": dev(4096, dtype=torch.uint8)}


def verify_arguments(S=2, n=4, V=50):
    return {"logits": dev(S, n, V), "tokens": i32(S, n), "accept_u": dev(S, n), "sample_u": dev(S), "accepted": i32(S, n), "n_accepted": i32(S),
            "next_token": i32(S), "workspace": dev(4096, dtype=torch.uint8)}


LAUNCHERS = [(cv.PageAppender, append_arguments, {"n_new": i32(2), "refs": i32(6)}), (cv.PageReader, read_arguments, {"first": i32(2), "n_rows": i32(2)}),
             (cv.PagedAttention, attention_arguments, {"lse": dev(2, 3, 14), "n_q": i32(2)}),
             (cv.PageAssigner, assign_arguments, {"src": i32(2), "table_out": i32(2, 4), "refs": i32(6)}),
             (cv.PageCompactor, compact_arguments, {"table_out": i32(2, 4), "refs": i32(6)}),
             (cv.DraftVerifier, verify_arguments, {"parents": i32(2, 4), "n_nodes": i32(2), "draft_probs": dev(2, 4, 50), "temperature": dev(2),
                                                   "log_probs": dev(2, 4)})]


@pytest.mark.parametrize("cls,arguments,more", LAUNCHERS, ids=lambda x: getattr(x, "__name__", ""))
def test_launchers_check_every_tensor(cls, arguments, more):
    """Built with all arguments; refused with any of them on the host, of another type, or of another length."""
    cls(None, **arguments())
    whole = {**arguments(), **more}
    cls(None, **whole)
    for name, t in whole.items():
        if not isinstance(t, torch.Tensor):
            continue
        plain = t.as_subclass(torch.Tensor)
        with pytest.raises(ValueError, match=name):
            cls(None, **{**whole, name: plain})
        if name == "workspace":
            continue
        with pytest.raises(ValueError):
            cls(None, **{**whole, name: plain.to(torch.float64).as_subclass(Device)})
        wider = torch.zeros((t.shape[0] + 1, *t.shape[1:]), dtype=t.dtype).as_subclass(Device)
        if name not in ("table", "k", "q", "logits"):  # (the ones that say how many sequences there are)
            with pytest.raises(ValueError):
                cls(None, **{**whole, name: wider})


def test_pools_are_checked():
    good = pool()
    u8 = lambda *s: dev(*s, dtype=torch.uint8)  # noqa: E731
    args = lambda **kw: {**{"k": u8(4, 2, 1024), "v": u8(4, 2, 1024), "k_scale": dev(4, 2, 1), "v_scale": dev(4, 2, 1), "format": 0}, **kw}  # noqa: E731
    cv.PagePool(**args())
    for bad in ({"k": u8(4, 2, 1000)}, {"k": u8(4, 2, 40 * D)}, {"k": u8(4, 2048)}, {"v": u8(4, 2, 2048)}, {"v": u8(4, 3, 1024)}, {"k_scale": dev(4, 2, 2)},
                {"v_scale": dev(4, 2, 1, dtype=torch.float16)}, {"v": torch.zeros(4, 2, 1024, dtype=torch.uint8)}, {"k": u8(4, 2, 2048)[:, :, ::2]},
                {"v": u8(4, 3, 1024)[:, :2]}):
        with pytest.raises(ValueError):
            cv.PagePool(**args(**bad))
    wide = cv.PagePool(u8(4, 5, 1024)[:, :2], u8(4, 5, 1024)[:, :2], dev(4, 2, 1), dev(4, 2, 1), 1)
    assert wide.desc.nb_page == 5 * 1024 and good.desc.nb_page == 2 * 32 * D
    with pytest.raises(ValueError):
        cv.PageAssigner(None, [], i32(2, 4), i32(2), i32(2))


# The entry points check before they touch a device: made-up addresses never reach one.
class Fake(ctypes.Structure):
    _fields_ = [("device", ctypes.c_int), ("status", ctypes.c_void_p)]


AT = 1 << 30


def c_pool(**kw):
    d = _lib.PagePoolDesc(AT, 2 * AT, 3 * AT, 4 * AT, 4096, 8, 0, 2, D, 32, 6, 0)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def c_append(**kw):
    p = _lib.PagedAppendParams(c_pool(), AT, 2 * AT, 128, 384, 5 * AT, 4, 4, 2, 6 * AT, None, None, 3, 0)
    return "cvattn_paged_append", p, kw


def c_read(**kw):
    p = _lib.PagedReadParams(c_pool(), AT, 2 * AT, 128, 384, 5 * AT, 4, 4, 2, None, None, 3, 0)
    return "cvattn_paged_read", p, kw


def c_attention(**kw):
    p = _lib.PagedAttentionParams(c_pool(), AT, 896, 2688, 2 * AT, 896, 2688, None, 5 * AT, 4, 6 * AT, None, 2, 3, 14, 128, 4, 0.125, 0, 0, 7 * AT, 1 << 24)
    return "cvattn_paged_attention", p, kw


def c_assign(**kw):
    pools = (_lib.PagePoolDesc * 2)(c_pool(), c_pool())
    p = _lib.PagesAssignParams(pools, 2, 2, 5 * AT, 6 * AT, 4, 4, 0, None, 7 * AT, 8 * AT, 9 * AT, None, 10 * AT, 1 << 20)
    return "cvattn_pages_assign", p, kw


def c_compact(**kw):
    pools = (_lib.PagePoolDesc * 2)(c_pool(), c_pool())
    p = _lib.PagesCompactParams(pools, 2, 2, 5 * AT, 6 * AT, 4, 4, 0, 7 * AT, None, 10 * AT, 1 << 20)
    return "cvattn_pages_compact", p, kw


def c_verify(**kw):
    p = _lib.VerifyParams(AT, 50, 200, None, 0, 0, 2 * AT, None, 0, None, 3 * AT, 4 * AT, None, 5 * AT, 4, 6 * AT, 7 * AT, None, 0, 2, 4, 50, 8 * AT, 1 << 20)
    return "cvattn_verify_drafts", p, kw


INVALID, UNSUPPORTED, LENGTH = 1, 2, 3
REFUSALS = [
    *[(c, {"pool": c_pool(**bad)}, s) for c in (c_append, c_read, c_attention) for bad, s in (
        ({"k": None}, INVALID), ({"v_scale": None}, INVALID), ({"k": AT + 8}, INVALID), ({"format": 2}, INVALID), ({"page_size": 48}, INVALID),
        ({"n_heads": 0}, INVALID), ({"n_pages": 0}, INVALID), ({"nb_page": 4096 - 16}, INVALID), ({"nb_page": 4100}, INVALID), ({"nb_scale": 3}, INVALID),
        ({"head_dim": 128}, UNSUPPORTED), ({"reserved": 1}, INVALID))],
    *[(c, bad, INVALID) for c in (c_append, c_read) for bad in ({"k": None}, {"v": AT + 4}, {"nb_row": 126}, {"nb_row": 124}, {"table": None},
                                                                {"table_nb_seq": 3}, {"table_width": 0}, {"n_seq": -1}, {"reserved": 1})],
    (c_append, {"kv_len": None}, INVALID), (c_append, {"max_new": 129}, LENGTH), (c_append, {"max_new": -1}, INVALID), (c_append, {"n_seq": 65536}, UNSUPPORTED),
    (c_read, {"nb_seq": 380}, INVALID), (c_read, {"max_rows": -1}, INVALID),
    *[(c_attention, bad, s) for bad, s in (
        ({"q": None}, INVALID), ({"out": AT + 4}, INVALID), ({"q_nb_tok": 892}, INVALID), ({"out_nb_tok": 892}, INVALID), ({"q_nb_seq": 2}, INVALID),
        ({"out_nb_seq": 896}, INVALID), ({"kv_len": None}, INVALID), ({"n_q_heads": 13}, UNSUPPORTED), ({"n_q_heads": 18, "q_nb_tok": 1152, "out_nb_tok": 1152,
                                                                                                     "out_nb_seq": 3456}, UNSUPPORTED),
        ({"max_kv_len": 129}, LENGTH), ({"max_kv_len": -1}, INVALID), ({"flags": 1}, INVALID), ({"workspace": AT + 4, "max_q": 2000, "out_nb_seq": 2000 * 896}, INVALID),
        ({"workspace_size": 16, "max_q": 2000, "max_kv_len": 128, "out_nb_seq": 2000 * 896}, INVALID))],
    *[(c, bad, INVALID) for c in (c_assign, c_compact) for bad in (
        {"pools": None}, {"n_pools": 0}, {"table": None}, {"table_out": None}, {"table_out": 5 * AT + 4}, {"table_nb_seq": 3}, {"workspace": None},
        {"workspace_size": 64}, {"refs": 5 * AT}, {"reserved": 1})],
    *[(c_assign, bad, INVALID) for bad in ({"keep": None}, {"need": None}, {"room": None}, {"room": 7 * AT}, {"room": 8 * AT + 4}, {"room": 5 * AT},
                                           {"refs": 7 * AT - 16}, {"keep": 6 * AT})],
    (c_compact, {"n_live": None}, INVALID), (c_compact, {"n_live": 6 * AT + 8}, INVALID), (c_compact, {"refs": 7 * AT - 4}, INVALID),
    *[(c_verify, bad, s) for bad, s in (
        ({"logits": None}, INVALID), ({"tokens": None}, INVALID), ({"logits_type": 2}, UNSUPPORTED), ({"logits": AT + 2}, INVALID), ({"logits_nb_node": 49}, INVALID),
        ({"draft_probs": AT + 2}, INVALID), ({"draft_probs": 9 * AT, "probs_nb_node": 49}, INVALID), ({"parents": 9 * AT, "parents_nb_seq": 3}, INVALID),
        ({"accepted_stride": 3}, INVALID), ({"n_accepted": 4 * AT}, INVALID), ({"accepted": 2 * AT + 16}, INVALID), ({"n_nodes": 7 * AT}, INVALID),
        ({"max_nodes": 257}, UNSUPPORTED), ({"vocab": 0}, INVALID), ({"vocab": 1 << 22, "logits_nb_node": 1 << 22}, UNSUPPORTED), ({"workspace": None}, INVALID),
        ({"workspace_size": 16}, INVALID))],
]


@pytest.mark.parametrize("make,bad,status", REFUSALS, ids=lambda x: getattr(x, "__name__", None))
def test_entry_points_refuse(make, bad, status):
    name, p, _ = make()
    ctx = Fake(0, None)
    for k, v in bad.items():
        if k == "pool":
            p.pool = v
        elif k == "pools":
            p.pools = ctypes.POINTER(_lib.PagePoolDesc)()
        else:
            setattr(p, k, v)
    fn = getattr(cv.lib, name)
    assert fn(ctypes.byref(ctx), None, ctypes.byref(p)) == status, bad
    assert fn(None, None, ctypes.byref(p)) == INVALID and fn(ctypes.byref(ctx), None, None) == INVALID


@pytest.mark.parametrize("make", [c_append, c_read, c_attention, c_assign, c_compact, c_verify], ids=lambda x: x.__name__)
def test_no_sequences_are_no_work(make):
    name, p, _ = make()
    p.n_seq = 0
    assert getattr(cv.lib, name)(ctypes.byref(Fake(0, None)), None, ctypes.byref(p)) == 0


def test_sizes_past_the_grids_and_32_bits_are_refused():
    ctx, most = Fake(0, None), 1 << 20
    rows = {"max_q": most, "out_nb_seq": most * 896, "workspace_size": 1 << 62}
    bad = [(c_attention, {"pool": c_pool(n_heads=1000, nb_page=1000 * 32 * D, nb_scale=2000), "n_q_heads": 1000, "n_seq": 1025, "max_q": 4161,
                          "q_nb_tok": 64000, "out_nb_tok": 64000, "out_nb_seq": 4161 * 64000, "workspace_size": 1 << 62}),
           (c_attention, {**rows, "max_kv_len": 0, "n_seq": 1}),
           (c_attention, {**rows, "max_q": most + 1}),
           (c_attention, {"max_kv_len": (1 << 30) + 1, "table_width": (1 << 31) // 32 - 1, "table_nb_seq": 1 << 26, "workspace_size": 1 << 62}),
           *[(c, {"pool": c_pool(n_pages=(1 << 30) + 1)}) for c in (c_append, c_read, c_attention)]]
    for make, values in bad:
        name, p, _ = make()
        for k, v in values.items():
            setattr(p, k, v)
        assert getattr(cv.lib, name)(ctypes.byref(ctx), None, ctypes.byref(p)) == UNSUPPORTED, values
    for make in (c_assign, c_compact):
        name, p, _ = make()
        p.n_seq, p.table_width, p.table_nb_seq = 1 << 20, 1025, 1025
        assert getattr(cv.lib, name)(ctypes.byref(ctx), None, ctypes.byref(p)) == INVALID


def test_pools_of_one_table_agree():
    for bad in (c_pool(page_size=16), c_pool(n_pages=7)):
        name, p, _ = c_assign()
        p.pools[1] = bad
        assert getattr(cv.lib, name)(ctypes.byref(Fake(0, None)), None, ctypes.byref(p)) == INVALID


def test_workspace_sizes():
    assert cv.paged_attention_workspace_size(0, 1, 1, 14, 2) == 0 and cv.paged_attention_workspace_size(1, 1, 100, 14, 3) == 0
    for S, n, L in ((1, 1, 300), (64, 1, 4096), (16, 16, 8192), (1, 1, 1 << 20), (200, 512, 4096)):
        size = cv.paged_attention_workspace_size(S, n, L, 14, 2)
        assert 0 <= size < 1 << 30
    assert cv.lib.cvattn_pages_workspace_size(0, 1, 1) == 0 < cv.lib.cvattn_pages_workspace_size(1, 1, 1)
    assert cv.lib.cvattn_verify_workspace_size(1, 0, 1) == 0 < cv.lib.cvattn_verify_workspace_size(1, 1, 1)


# ---------------------------------------------------------------------------------------------------- the plain forms

def test_formats():
    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(E4M3[np.isfinite(t)], t[np.isfinite(t)])
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.standard_normal(4000) * np.exp(rng.uniform(-8, 6, 4000)), E4M3[:126] * 0.5 + E4M3[1:127] * 0.5])
    want = torch.tensor(np.clip(x, -448, 448)).float().to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    exact = np.abs(x.astype(np.float32).astype(np.float64) - x) == 0
    assert np.array_equal(nearest(1, x)[exact], want[exact])
    assert np.array_equal(VALUES[0][nearest(0, np.array([0.5, 1.5, -2.5, 126.5, 127.5, -1e30]))], [0, 2, -2, 126, 127, -127])
    assert all(sorted(PLACE[k].ravel()) == list(range(1024)) for k in "kv")


@pytest.mark.parametrize("fmt", [0, 1])
def test_rounding_is_off_by_half_a_step(fmt):
    rng = np.random.default_rng(fmt)
    host = Pool(fmt, 2, 32, 2)
    x = rng.standard_normal((40, 2, D)).astype(np.float32)
    host.append("k", [1, 0], 0, x)
    for b in range(0, 40, 16):
        part, got = x[b:b + 16].astype(np.float64), host.rows("k", [1, 0], 40)[b:b + 16]
        most = np.abs(part).max((0, 2), keepdims=True)
        # int8: half of 1/127 of the block's largest; e4m3: 2^-4 of the value, or half a step of its smallest numbers
        half = most / 127 / 2 if fmt == 0 else np.maximum(np.abs(part) * 2.0 ** -4, most / 448 * 2.0 ** -10)
        assert np.all(np.abs(got - part) <= half * (1 + 1e-6))


def test_attention_of_the_plain_form():
    rng = np.random.default_rng(3)
    q, k, v = rng.standard_normal((2, 4, D)), rng.standard_normal((9, 2, D)), rng.standard_normal((9, 2, D))
    out, lse = attention(q, k, v, 2, 0.125)
    s = np.einsum("nhd,lhd->nhl", q, np.repeat(k, 2, 1)) * 0.125
    s[0, :, 8] = -np.inf
    p = np.exp(s - s.max(-1, keepdims=True))
    assert np.allclose(out, np.einsum("nhl,lhd->nhd", p / p.sum(-1, keepdims=True), np.repeat(v, 2, 1)))
    assert np.allclose(lse, np.log(np.exp(s).sum(-1)))


def test_verification_keeps_the_target_distribution():
    """Over many random numbers the first gained token is distributed as the target, whatever the drafts."""
    rng = np.random.default_rng(5)
    p, q = rng.dirichlet(np.ones(6)), rng.dirichlet(np.ones(6))
    logits = np.log(np.stack([p] * 4))
    n, gained = 40000, []
    for _ in range(n):
        tokens = np.concatenate([[0], rng.choice(6, 3, p=q)])
        path, end, _ = verify(logits, tokens, [-1, 0, 0, 0], 4, rng.random(4), rng.random(), 1.0, np.stack([q] * 4))
        gained.append(tokens[path[1]] if len(path) > 1 else end)
    share = np.bincount(gained, minlength=6) / n
    assert np.abs(share - p).max() < 5 * np.sqrt(0.25 / n)  # five standard deviations of a share


def test_assignment_of_the_plain_form():
    t = np.array([[4, 1, -1], [4, 1, -1]], np.int32)
    out, refs, room, moves = assign(t, [0, 0], [20, 20], [20, 21], 16, 6)
    assert out.tolist() == [[4, 1, -1], [4, 0, -1]] and moves == [(1, 0)] and list(refs) == [1, 1, 0, 0, 2, 0] and list(room) == [20, 21]
