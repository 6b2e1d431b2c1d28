"""Refusals of the paged-cache and sampling entry points, on the host: the C argument checks (before any device is
asked for) and the Python wrappers' shape, type and device checks; and the oracle of the GPU tests against itself."""
import ctypes
import math

import numpy as np
import pytest
import torch

from funasr_amd import runtime as rt
from oracle import serve_ref as ref

P16 = 0x10000   # an aligned address that no check may read
E_ARG = -1


def ref_(x):
    return None if x is None else ctypes.byref(x)


def cache(**kw):
    c = rt.PfmPagedKv()
    c.k, c.v, c.pages, c.page_size, c.heads, c.head_dim, c.dtype = P16, P16, 4, 16, 2, 64, rt.PFM_BF16
    c.k_stride[:], c.v_stride[:] = (2048, 128, 64), (2048, 128, 64)
    c.block_table, c.table_stride, c.table_width, c.kv_len, c.cu_q, c.batch, c.tokens = P16, 3, 3, P16, P16, 2, 5
    for k, v in kw.items():
        if k in ("k_stride", "v_stride"):
            getattr(c, k)[:] = v
        else:
            setattr(c, k, v)
    return ref_(c)


def rows(p=P16, ts=256, hs=64):
    return ref_(rt.PfmRows(p, ts, hs))


BAD_CACHE = [dict(dtype=2), dict(dtype=9), dict(batch=-1), dict(tokens=-1), dict(pages=-1), dict(table_width=-1),
             dict(page_size=0), dict(heads=0), dict(heads=70000), dict(head_dim=0), dict(head_dim=60), dict(head_dim=264),
             dict(k=None), dict(v=None), dict(block_table=None), dict(kv_len=None), dict(cu_q=None), dict(table_stride=2),
             dict(k=P16 + 8), dict(v=P16 + 2), dict(k_stride=(2048, 128, 60)), dict(v_stride=(2044, 128, 64)),
             dict(k_stride=(-2048, 128, 64)), dict(page_size=1 << 30, table_width=3),
             dict(page_size=(1 << 31) - 4096, table_width=1, k_stride=(1 << 38, 128, 64), v_stride=(1 << 38, 128, 64))]


@pytest.mark.parametrize("kw", BAD_CACHE, ids=str)
def test_bad_cache_refused(kw):
    lib = rt.load_library()
    c = cache(**kw)
    assert lib.pfm_op_kv_append(None, c, rows(), rows(), rows(), rows(), 4, None, 0, 0, None) == E_ARG
    assert b"pfm_op_kv_append" in lib.pfm_last_error()
    assert lib.pfm_op_paged_attention(None, c, rows(), rows(), 4, 1.0, 1, 0, P16, 1 << 40) == E_ARG
    assert b"pfm_op_paged_attention" in lib.pfm_last_error()


@pytest.mark.parametrize("k,v,q,qo,hq,freq,rot", [
    (None, rows(), rows(), rows(), 4, P16, 64), (rows(), None, rows(), rows(), 4, P16, 64),
    (rows(), rows(), None, rows(), 4, P16, 64), (rows(), rows(), rows(), None, 4, P16, 64),
    (rows(P16 + 4), rows(), rows(), rows(), 4, P16, 64), (rows(ts=250), rows(), rows(), rows(), 4, P16, 64),
    (rows(hs=-64), rows(), rows(), rows(), 4, P16, 64), (rows(), rows(), rows(), rows(hs=0), 4, P16, 64),
    (rows(), rows(), rows(), rows(ts=0), 4, P16, 64), (rows(), rows(), rows(), rows(), -1, P16, 64),
    (rows(), rows(), rows(), rows(), 4, P16, 8), (rows(), rows(), rows(), rows(), 4, P16, 24),
    (rows(), rows(), rows(), rows(), 4, P16, 80)])
def test_bad_append_refused(k, v, q, qo, hq, freq, rot):
    lib = rt.load_library()
    assert lib.pfm_op_kv_append(None, cache(), k, v, q, qo, hq, freq, rot, 0, None) == E_ARG


@pytest.mark.parametrize("kw", [dict(k_stride=(0, 128, 64)), dict(v_stride=(2048, 128, 0)), dict(k_stride=(2048, 0, 64))])
def test_append_to_overlapping_pages_refused(kw):
    lib = rt.load_library()
    assert lib.pfm_op_kv_append(None, cache(**kw), rows(), rows(), rows(), rows(), 4, None, 0, 0, None) == E_ARG


@pytest.mark.parametrize("q,out,hq,scale,window,ws,nb", [
    (None, rows(), 4, 1.0, 0, P16, 1 << 40), (rows(), None, 4, 1.0, 0, P16, 1 << 40),
    (rows(), rows(), 3, 1.0, 0, P16, 1 << 40), (rows(), rows(), 0, 1.0, 0, P16, 1 << 40),
    (rows(), rows(), 4, math.nan, 0, P16, 1 << 40), (rows(), rows(), 4, math.inf, 0, P16, 1 << 40),
    (rows(), rows(), 4, 1.0, -1, P16, 1 << 40), (rows(P16 + 2), rows(), 4, 1.0, 0, P16, 1 << 40),
    (rows(), rows(ts=0), 4, 1.0, 0, P16, 1 << 40), (rows(), rows(hs=0), 4, 1.0, 0, P16, 1 << 40)])
def test_bad_attention_refused(q, out, hq, scale, window, ws, nb):
    lib = rt.load_library()
    assert lib.pfm_op_paged_attention(None, cache(), q, out, hq, scale, 1, window, ws, nb) == E_ARG


def test_attention_workspace_refused():
    lib = rt.load_library()
    c = cache(table_width=4096, table_stride=4096, tokens=2)   # long caches, few rows: the keys are split
    need = lib.pfm_paged_attention_ws_bytes(c, 4)
    assert need > 0
    for ws, nb in ((None, need), (P16, need - 1), (P16 + 4, need)):
        assert lib.pfm_op_paged_attention(None, c, rows(), rows(), 4, 1.0, 1, 0, ws, nb) == E_ARG
        assert b"pace" in lib.pfm_last_error()
    assert lib.pfm_paged_attention_ws_bytes(None, 4) == 0
    assert lib.pfm_paged_attention_ws_bytes(cache(batch=0, tokens=0), 4) == 0


@pytest.mark.parametrize("kw", [dict(dtype=2), dict(B=-1), dict(V=0), dict(V=(1 << 20) + 1, ld=1 << 21), dict(ld=9),
                                dict(logits=None), dict(u=None), dict(token=None), dict(logits=P16 + 1)], ids=str)
def test_bad_sample_refused(kw):
    lib = rt.load_library()
    a = dict(dtype=rt.PFM_F32, logits=P16, ld=10, B=2, V=10, u=P16, token=P16) | kw
    assert lib.pfm_op_sample(None, a["dtype"], a["logits"], a["ld"], a["B"], a["V"], a["u"], None, None, None, None,
                             a["token"], None, P16, 1 << 40) == E_ARG
    assert b"pfm_op_sample" in lib.pfm_last_error()


def test_window_takes_the_workspace_of_no_window():
    """pfm_paged_attention_ws_bytes knows no window: with any, the call wants no more."""
    lib = rt.load_library()
    rng = np.random.default_rng(3)
    for _ in range(4000):
        width, n, heads, b = (int(rng.integers(1, x)) for x in (6000, 9000, 12, 9))
        c = cache(table_width=width, table_stride=width, tokens=n, heads=heads, batch=b,
                  head_dim=int(rng.choice([64, 128, 256])), k_stride=(1 << 20, 1 << 14, 256),
                  v_stride=(1 << 20, 1 << 14, 256), dtype=int(rng.choice([rt.PFM_F32, rt.PFM_BF16])))
        nb = lib.pfm_paged_attention_ws_bytes(c, heads * 2)
        window, causal = int(rng.integers(1, 16 * width + 1)), int(rng.integers(2))
        lib.pfm_op_paged_attention(None, c, rows(ts=1 << 14, hs=256), rows(ts=1 << 14, hs=256), heads * 2, 1.0, causal,
                                   window, P16, nb)
        assert b"workspace" not in lib.pfm_last_error(), (width, n, heads, b, window, causal)


def ws_bytes(batch, tokens, reach, heads=8, q_heads=32, dim=128, page=64, **kw):
    width = -(-reach // page)
    c = cache(batch=batch, tokens=tokens, table_width=width, table_stride=width, page_size=page, heads=heads, head_dim=dim, **kw)
    return rt.load_library().pfm_paged_attention_ws_bytes(c, q_heads)


@pytest.mark.parametrize("batch,tokens,reach", [(2, 8192, 8192), (8, 3500, 6720), (8, 4096, 4096), (3, 1500, 4000)])
def test_workspace_of_prompts(batch, tokens, reach):
    """Prompts whose row tiles are not split: the parts of sequences of at most 16 query rows alone, 256 at most (as many
    as a launch splits into) of 16 rows per sequence and kv head, whatever the number of tokens is."""
    nb = ws_bytes(batch, tokens, reach)
    assert nb <= min(256, reach // 256) * batch * 8 * 16 * (128 + 2) * 4
    assert nb <= tokens * 32 * 128 * 2                   # and less than the output


def test_workspace_is_bounded():
    """No call asks for more than the header says, whatever the table's reach: 2^18 or 2^19 rows of dims, maximum and sum."""
    rng = np.random.default_rng(8)
    size = lambda a, b: int(round(np.exp(rng.uniform(np.log(a), np.log(b)))))  # noqa: E731
    for _ in range(20000):
        heads, dim, batch = int(rng.choice([1, 2, 4, 8, 16, 32])), int(rng.choice([8, 64, 128, 136, 256])), size(1, 512)
        args = (batch, size(batch, 131072), size(64, 1 << 20), heads, heads * int(rng.choice([1, 2, 3, 8, 16])), dim)
        kw = dict(dtype=int(rng.choice([rt.PFM_F32, rt.PFM_BF16]))) | (dict(cu_q=None) if rng.random() < 0.3 else {})
        if "cu_q" in kw:
            args = (args[1], *args[1:])
        assert ws_bytes(*args, **kw) <= 4 * (dim + 2) << (19 if dim <= 128 else 18), (args, kw)


@pytest.mark.parametrize("kw", [dict(k_stride=(4096, 64, 64)), dict(v_stride=(2048, 64, 64)), dict(k_stride=(64, 128, 64)),
                                dict(k_stride=(1984, 128, 64))], ids=str)
def test_append_to_interleaved_pages_refused(kw):
    """strides that step over a head, but on the place of another slot, page or head"""
    lib = rt.load_library()
    assert lib.pfm_op_kv_append(None, cache(**kw), rows(), rows(), rows(), rows(), 4, None, 0, 0, None) == E_ARG
    assert b"overlap" in lib.pfm_last_error()


def test_outputs_on_each_other_refused():
    lib = rt.load_library()
    assert lib.pfm_op_kv_append(None, cache(), rows(), rows(), rows(), rows(ts=128), 4, None, 0, 0, None) == E_ARG
    assert lib.pfm_op_paged_attention(None, cache(), rows(), rows(ts=128), 4, 1.0, 1, 0, P16, 1 << 40) == E_ARG
    assert b"overlap" in lib.pfm_last_error()


def test_calls_past_a_launch_refused():
    """a grid of 2^32 threads or more"""
    lib = rt.load_library()
    big = dict(table_width=1, table_stride=1)
    for kw in (dict(batch=1 << 25, tokens=1 << 25, cu_q=None), dict(batch=1, tokens=(1 << 24) + 1)):
        c = cache(**big, **kw)
        assert lib.pfm_op_kv_append(None, c, rows(), rows(), rows(), rows(), 4, None, 0, 0, None) == E_ARG
        assert lib.pfm_op_paged_attention(None, c, rows(), rows(), 4, 1.0, 1, 0, P16, 1 << 60) == E_ARG
    c = cache(**big, batch=1 << 20, tokens=1 << 20, cu_q=None, heads=64, k_stride=(1 << 16, 1 << 12, 64),
              v_stride=(1 << 16, 1 << 12, 64))
    assert lib.pfm_op_paged_attention(None, c, rows(ts=1 << 13), rows(ts=1 << 13), 64, 1.0, 1, 0, P16, 1 << 60) == E_ARG
    assert b"one call" in lib.pfm_last_error()
    assert lib.pfm_op_sample(None, rt.PFM_F32, P16, 20000, (1 << 20) + 1, 20000, P16, None, None, None, None, P16, None,
                             P16, 1 << 60) == E_ARG
    assert b"2^20" in lib.pfm_last_error()


def test_calls_within_the_stated_limit_are_taken():
    """tokens * q_heads / 16 + 3 * batch * heads < 2^24 fits one launch's grid in every plan."""
    lib, rng, n = rt.load_library(), np.random.default_rng(5), 0
    size = lambda top: int(round(2 ** rng.uniform(0, top)))  # noqa: E731
    while n < 3000:
        heads, group, batch, dim = size(9), size(8), size(24), int(rng.choice([8, 128, 256]))
        tokens = max(batch, size(24)) if rng.random() < 0.7 else batch
        room = (1 << 24) - 1 - 3 * batch * heads
        if rng.random() < 0.5 and room * 16 >= batch * heads * group:
            tokens = min(1 << 24, room * 16 // (heads * group))              # at the limit
        if tokens * heads * group / 16 + 3 * batch * heads >= 1 << 24 or tokens < 1:
            continue
        n += 1
        width = size(14)
        c = cache(batch=batch, tokens=tokens, heads=heads, head_dim=dim, table_width=width, table_stride=width,
                  dtype=int(rng.choice([rt.PFM_F32, rt.PFM_F16])), **({"cu_q": None} if tokens == batch else {}))
        r = rows(ts=1 << 28, hs=1 << 10)
        lib.pfm_op_paged_attention(None, c, r, r, heads * group, 1.0, 1, 0, P16, 1 << 60)
        assert b"one call" not in lib.pfm_last_error(), (batch, tokens, heads, group, dim, width)
        assert b"2^31" not in lib.pfm_last_error()


def test_empty_batches_are_nothing():
    lib = rt.load_library()
    c = cache(batch=0, tokens=0)
    assert lib.pfm_op_kv_append(None, c, None, None, None, None, 0, None, 0, 0, None) == 0
    assert lib.pfm_op_paged_attention(None, c, None, None, 4, 1.0, 1, 0, None, 0) == 0
    assert lib.pfm_op_sample(None, rt.PFM_F32, None, 10, 0, 10, None, None, None, None, None, None, None, None, 0) == 0


def _args(N=3, B=3, W=2, P=8, page=4, hk=2, hq=4, D=16, dt=torch.float32):
    return dict(k=torch.zeros(N, hk, D, dtype=dt), v=torch.zeros(N, hk, D, dtype=dt), q=torch.zeros(N, hq, D, dtype=dt),
                kp=torch.zeros(P, page, hk, D, dtype=dt), vp=torch.zeros(P, page, hk, D, dtype=dt),
                table=torch.zeros(B, W, dtype=torch.int32), kv_len=torch.ones(B, dtype=torch.int32))


@pytest.mark.parametrize("change", [
    dict(k=torch.zeros(3, 2, 8)), dict(k=torch.zeros(2, 2, 16)), dict(k=torch.zeros(3, 2, 16).half()),
    dict(v=torch.zeros(3, 1, 16)), dict(q=torch.zeros(3, 4, 8)), dict(q=torch.zeros(4, 4, 16)), dict(q=torch.zeros(3, 64)),
    dict(kp=torch.zeros(8, 4, 32)), dict(vp=torch.zeros(8, 4, 2, 16).half()), dict(vp=torch.zeros(7, 4, 2, 16)),
    dict(kp=torch.zeros(8, 4, 2, 16).double(), vp=torch.zeros(8, 4, 2, 16).double()),
    dict(kp=torch.zeros(8, 4, 16, 2).transpose(2, 3), vp=torch.zeros(8, 4, 2, 16)),
    dict(table=torch.zeros(3, 2)), dict(table=torch.zeros(3, dtype=torch.int32)),
    dict(table=torch.zeros(2, 3, dtype=torch.int32).t()), dict(kv_len=torch.ones(3)),
    dict(kv_len=torch.ones(4, dtype=torch.int32)), dict(table=torch.zeros(2, 2, dtype=torch.int32), kv_len=torch.ones(2, dtype=torch.int32)),
    dict(cu_q=torch.zeros(3, dtype=torch.int32)), dict(cu_q=torch.zeros(4))], ids=lambda c: "-".join(f"{k}{tuple(v.shape)}" for k, v in c.items()))
def test_wrappers_refuse(change):
    a = _args() | change
    cu = a.get("cu_q")
    with pytest.raises(rt.PfmError):
        rt.op_kv_append(a["k"], a["v"], a["kp"], a["vp"], a["table"], a["kv_len"], cu, q=a["q"])
    if not {"k", "v"} & set(change):
        with pytest.raises(rt.PfmError):
            rt.op_paged_attention(a["q"], a["kp"], a["vp"], a["table"], a["kv_len"], cu)


def test_wrappers_refuse_host_tensors_and_extras():
    a = _args()
    with pytest.raises(rt.PfmError):
        rt.op_paged_attention(a["q"], a["kp"], a["vp"], a["table"], a["kv_len"])
    with pytest.raises(rt.PfmError):
        rt.op_kv_append(a["k"], a["v"], a["kp"], a["vp"], a["table"], a["kv_len"], q_out=a["q"])
    for bad in (torch.zeros(2, 8), torch.zeros(8).double()):
        with pytest.raises(rt.PfmError):
            rt.op_kv_append(a["k"], a["v"], a["kp"], a["vp"], a["table"], a["kv_len"], inv_freq=bad)
    x, u = torch.zeros(2, 10), torch.zeros(2)
    for call in (lambda: rt.op_sample(x, u), lambda: rt.op_sample(x.double(), u), lambda: rt.op_sample(x[0], u),
                 lambda: rt.op_sample(x.t(), torch.zeros(10)), lambda: rt.op_sample(x, None),
                 lambda: rt.op_sample(x, u.double()), lambda: rt.op_sample(x, u, top_k=u),
                 lambda: rt.op_sample(x, u, temperature=torch.zeros(3)), lambda: rt.op_sample(x, torch.zeros(4)[::2])):
        with pytest.raises(rt.PfmError):
            call()


@pytest.mark.parametrize("change", [dict(k=torch.tensor(0.0)), dict(k=torch.zeros(3)), dict(q=torch.zeros(3)), dict(q=torch.tensor(0.0)),
                                    dict(inv_freq=torch.tensor(1.0)), dict(v=torch.tensor(0.0))],
                         ids=lambda c: "-".join(f"{k}{tuple(v.shape)}" for k, v in c.items()))
def test_wrappers_refuse_other_ranks(change):
    a = _args() | change
    with pytest.raises(rt.PfmError):
        rt.op_kv_append(a["k"], a["v"], a["kp"], a["vp"], a["table"], a["kv_len"], q=a["q"], inv_freq=a.get("inv_freq"))


@pytest.mark.parametrize("window", [-1, 1 << 31, (1 << 32) + 5])
def test_wrapper_refuses_windows_past_32_bits(window):
    a = _args()
    with pytest.raises(rt.PfmError, match="window"):
        rt.op_paged_attention(a["q"], a["kp"], a["vp"], a["table"], a["kv_len"], window=window)


def test_struct_layout_matches_header():
    """ctypes layouts against the C compiler's, by the header's field order and sizes."""
    assert ctypes.sizeof(rt.PfmRows) == 24 and ctypes.sizeof(rt.PfmPagedKv) == 8 * 13 + 4 * 7 + 4
    assert rt.PfmPagedKv.dtype.offset == 104 and rt.PfmPagedKv.tokens.offset == 128


# ---- the oracle itself
def test_oracle_sample_by_hand():
    x = torch.log(torch.tensor([[0.1, 0.4, 0.2, 0.3]]))
    s = lambda u, **kw: ref.sample(x, torch.tensor([u]), **kw)  # noqa: E731
    assert s(0.05)[0] == [0] and s(0.3)[0] == [1] and s(0.6)[0] == [2] and s(0.99)[0] == [3]
    assert s(0.0, top_k=torch.tensor([2]))[0] == [1] and s(0.99, top_k=torch.tensor([2]))[0] == [3]
    t, p = s(0.99, top_p=torch.tensor([0.69]))
    assert t == [3] and p[0] == pytest.approx(0.3 / 0.7, rel=1e-6)
    assert s(0.0, min_p=torch.tensor([0.7]))[0] == [1]
    assert s(0.9, temperature=torch.tensor([0.0]))[0] == [1]
    assert ref.sample(torch.full((1, 3), -math.inf), torch.tensor([0.5])) == ([-1], [0.0])


def test_oracle_attend_and_append_by_hand():
    kp = torch.zeros(3, 2, 1, 8, dtype=torch.float64)
    vp = torch.zeros_like(kp)
    table = torch.tensor([[2, 0]], dtype=torch.int32)
    k = torch.arange(24.0).view(3, 1, 8)
    _, kp, vp = ref.append(k, 2 * k, kp, vp, table, torch.tensor([3]), torch.tensor([0, 3]))
    assert torch.equal(kp[2, 0, 0], k[0, 0].double()) and torch.equal(vp[0, 0, 0], 2 * k[2, 0].double())
    q = torch.zeros(3, 2, 8)
    o, _, _ = ref.attend(q, kp, vp, table, torch.tensor([3]), torch.tensor([0, 3]))
    assert torch.allclose(o[:, 0], torch.stack([2 * k[: i + 1, 0].double().mean(0) for i in range(3)]))
    r = ref.rotate(torch.ones(1, 16, dtype=torch.float64), 1, torch.tensor([math.pi / 2] * 8), False)
    assert torch.allclose(r, torch.tensor([[-1.0] * 8 + [1.0] * 8], dtype=torch.float64), atol=1e-6)
