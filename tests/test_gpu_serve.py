"""Decoding over a paged key / value cache on the MI355X: append with rotation, attention of new tokens, sampling, each
against its plain statement in 64 bits (oracle/serve_ref.py), and a run of them together as a decoder makes it.

Tolerances (a rounding to type t is off by at most u = finfo(t).eps / 2 relative to the value):
  append     one rounding u of the result; the products and the sum in f32 and the angle, reduced to a turn in 64 bits
             and rounded to f32, add under 2^-20 (|x1| + |x2|). Values and unrotated dims are copied: bit for bit.
  attention  the probabilities are rounded to a 16-bit type (u; in f32 not), the scores' f32 sums of D products are off
             by (D + 8) 2^-24 spread (spread = scale max_j sum_d |q_d k_jd|), which acts twice (numerator, sum), 2^-20
             covers exp2 and the base change, L 2^-24 the sums over L keys; all of it relative to sum_j p_j |v_j|.
             Then u relative to the result. f16's subnormal probabilities: 2^-25 absolute per key.
  sample     the token is exact; its probability is a ratio of whole numbers rounded to f32."""
import ctypes
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from funasr_amd import runtime as rt  # noqa: E402
from oracle import serve_ref as ref  # noqa: E402

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    rt.load_library()
    return torch.device("cuda", 0)


class Batch:
    """Sequences with `new` tokens and `kv` keys (the new ones included) in shuffled pages, as CPU tensors."""

    def __init__(self, new, kv, hq=4, hk=2, D=64, page=16, dt=BF16, seed=0, one=False, spare=2, width=None, layout="nhd"):
        g = torch.Generator().manual_seed(seed)
        self.new, self.kv, self.one, self.dt, self.layout = new, kv, one, dt, layout
        n = sum(new)
        self.q, self.k, self.v = (torch.randn(n, h, D, generator=g).to(dt) for h in (hq, hk, hk))
        need = [min(-(-m // page), width or m + 1) for m in kv]
        P = sum(need) + spare
        ids = torch.randperm(P, generator=g)
        W = max(max(need), 1) if width is None else width
        self.table = torch.full((len(kv), W), -1, dtype=torch.int32)
        at = 0
        for b, m in enumerate(need):
            self.table[b, :m] = ids[at:at + m].int()
            at += m
        self.kp, self.vp = (torch.randn(P, page, hk, D, generator=g).to(dt) for _ in range(2))
        self.kv_len = torch.tensor(kv, dtype=torch.int32)
        self.cu = None if one else torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32)

    def pages(self, t, dev):
        if self.layout == "hnd":      # heads outside the page's slots
            return t.to(dev).transpose(1, 2).contiguous().transpose(1, 2)
        if self.layout == "slice":    # one layer of many, in a wider row
            wide = torch.zeros(t.shape[0], 2, *t.shape[1:3], t.shape[3] + 16, dtype=t.dtype, device=dev)
            wide[:, 1, :, :, :t.shape[3]] = t.to(dev)
            return wide[:, 1, :, :, :t.shape[3]]
        return t.to(dev)

    def on(self, dev):
        cu = None if self.cu is None else self.cu.to(dev)
        return self.pages(self.kp, dev), self.pages(self.vp, dev), self.table.to(dev), self.kv_len.to(dev), cu


def half_step(dt):
    return torch.finfo(dt).eps / 2


def attend_check(B, dev, q=None, **kw):
    """The call as it is, and with a table whose further entries name no page: how far it reaches says which kernels run."""
    q = B.q if q is None else q
    kp, vp, table, kv_len, cu = B.on(dev)
    (n, hq, D), (_, page, hk) = q.shape, B.kp.shape[:3]
    far = 2 * 10 ** 7 // ((n * hq // hk // 16 + 1) * hk * D * page) + 1
    for wide in [torch.full((len(B.kv), 0), -1, dtype=torch.int32), torch.full((len(B.kv), far), -1, dtype=torch.int32)]:
        got = rt.op_paged_attention(q.to(dev), kp, vp, torch.cat([table, wide.to(dev)], 1), kv_len, cu, **kw)
        torch.cuda.synchronize()
        want, bound, spread = ref.attend(q, B.kp, B.vp, torch.cat([B.table, wide], 1), B.kv_len, B.cu, **kw)
        check_attend(got.cpu(), want, bound, spread, B, D)
        if not len(wide[0]):
            first = got
    return first


def check_attend(got, want, bound, spread, B, D):
    L = max(B.kv + [1])
    u = half_step(B.dt)
    d = (D + 8) * 2.0 ** -24 * spread[..., None] * 2 + 2.0 ** -20 + L * 2.0 ** -24
    tol = ((0 if B.dt == F32 else u) + d) * bound * 1.05 + u * want.abs() * 1.05 + 1e-30
    if B.dt == F16:
        tol = tol + 2.0 ** -25 * (1 + 6 * L)     # the tests' finite values stay under 6
    err = (got.double() - want).abs()
    assert torch.equal(torch.isnan(got.double()), torch.isnan(want))
    bad = ~(err <= tol) & ~torch.isnan(want) & ~(got.double() == want)
    assert not bad.any(), (int(bad.sum()), float((err / tol)[bad].max()), bad.nonzero()[:3].tolist())


# ---- append
@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("D,rot,page,inter,layout", [(64, 64, 16, False, "nhd"), (64, 32, 1, True, "nhd"), (80, 80, 17, False, "hnd"),
                                                     (96, 48, 24, True, "slice"), (128, 128, 64, False, "hnd"),
                                                     (256, 256, 5, True, "nhd"), (8, 0, 3, False, "nhd"), (32, 16, 16, False, "slice")])
def test_append(dev, dt, D, rot, page, inter, layout):
    new, kv = [3, 0, 1, 17, 40], [3, 5, 1000, 33, 90]
    B = Batch(new, kv, hq=6, hk=2, D=D, page=page, dt=dt, seed=D + rot, layout=layout)
    freq = (10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64) / max(rot // 2, 1))).float() if rot else None
    kp, vp, table, kv_len, cu = B.on(dev)
    qkv = torch.cat([B.q, B.k, B.v], 1).to(dev)         # slices of one projection
    q = rt.op_kv_append(qkv[:, 6:8], qkv[:, 8:], kp, vp, table, kv_len, cu, q=qkv[:, :6],
                        inv_freq=None if freq is None else freq.to(dev), interleaved=inter)
    torch.cuda.synchronize()
    wq, wk, wv = ref.append(B.k, B.v, B.kp, B.vp, B.table, B.kv_len, B.cu, q=B.q, inv_freq=freq, interleaved=inter,
                            q_out=torch.zeros_like(B.q))
    assert torch.equal(vp.cpu().double(), wv)
    for got, want, src in ((q, wq, B.q), (kp, wk, None)):
        got = got.cpu().double()
        most = 8.0 if src is None else float(src.double().abs().max())
        assert ((got - want).abs() <= half_step(dt) * want.abs() * 1.001 + (2.0 ** -20 * 2 * most if rot else 0)).all()
        assert torch.equal(got[..., rot:], want[..., rot:])
    untouched = (wk == B.kp.double()).all(-1)
    assert torch.equal(kp.cpu()[untouched], B.kp[untouched])


@pytest.mark.parametrize("dt", [F32, BF16])
def test_append_far_positions(dev, dt):
    """Angles of positions up to 2^31 - 1 and explicit positions, negative ones among them."""
    B = Batch([1] * 6, [4] * 6, D=64, dt=dt, one=True)
    pos = torch.tensor([0, 1, 12345678, 2 ** 31 - 1, -7, 2 ** 30 + 1], dtype=torch.int32)
    freq = torch.tensor([1.0, 0.7310585, 1e-3, 1e-6, 0.25, 3.0, 0.1, 1e-5] * 4)
    kp, vp, table, kv_len, cu = B.on(dev)
    q = rt.op_kv_append(B.k.to(dev), B.v.to(dev), kp, vp, table, kv_len, q=B.q.to(dev), inv_freq=freq.to(dev), pos=pos.to(dev))
    wq, wk, _ = ref.append(B.k, B.v, B.kp, B.vp, B.table, B.kv_len, q=B.q, inv_freq=freq, pos=pos, q_out=torch.zeros_like(B.q))
    for got, want in ((q, wq), (kp, wk)):
        assert ((got.cpu().double() - want).abs() <= half_step(dt) * want.abs() * 1.001 + 2.0 ** -20 * 8).all()


def test_append_leaves_what_is_not_its_own(dev):
    """Rows behind the last sequence, absent pages, positions before 0 and behind the table, sequences without rows; q
    rotated in place; keys alone."""
    B = Batch([2, 3, 1, 4], [2, 2, 90, 40], D=64, page=16, dt=F32, width=3)   # 3 new of 2 keys; 90 keys > 48 of the table
    B.table[3, 1], B.table[3, 2] = 999, -5
    q, k, v = (torch.cat([t, torch.full((5, *t.shape[1:]), 7.0)]) for t in (B.q, B.k, B.v))
    freq = torch.rand(32) + 0.1
    kp, vp, table, kv_len, cu = B.on(dev)
    qd = q.to(dev)
    out = rt.op_kv_append(k.to(dev), v.to(dev), kp, vp, table, kv_len, cu, q=qd, inv_freq=freq.to(dev), q_out=qd)
    assert out is qd
    wq, wk, wv = ref.append(k, v, B.kp, B.vp, B.table, B.kv_len, B.cu, q=q, inv_freq=freq, q_out=q)
    assert torch.equal(qd.cpu()[10:], q[10:])
    assert (qd.cpu().double() - wq).abs().max() <= 2.0 ** -20 * 10
    assert (kp.cpu().double() - wk).abs().max() <= 2.0 ** -20 * 10 and torch.equal(vp.cpu().double(), wv)
    kp2, vp2, *_ = B.on(dev)
    assert rt.op_kv_append(k.to(dev), v.to(dev), kp2, vp2, table, kv_len, cu, inv_freq=freq.to(dev)) is None
    assert torch.equal(kp, kp2) and torch.equal(vp, vp2)


@pytest.mark.parametrize("n", [1023, 1025, 2051])
def test_append_many_rows(dev, n):
    """Both sides of the rows-per-workgroup rule, over 130 sequences (more than one wave looks through at once)."""
    r = np.random.default_rng(n)
    cuts = np.sort(r.integers(0, n + 1, 129))
    new = np.diff(np.concatenate([[0], cuts, [n]])).tolist()
    B = Batch(new, [int(x + r.integers(0, 50)) for x in new], hq=1, hk=1, D=16, page=8, dt=F32, seed=n)
    freq = torch.rand(8)
    kp, vp, table, kv_len, cu = B.on(dev)
    q = rt.op_kv_append(B.k.to(dev), B.v.to(dev), kp, vp, table, kv_len, cu, q=B.q.to(dev), inv_freq=freq.to(dev))
    wq, wk, wv = ref.append(B.k, B.v, B.kp, B.vp, B.table, B.kv_len, B.cu, q=B.q, inv_freq=freq, q_out=torch.zeros_like(B.q))
    assert torch.equal(vp.cpu().double(), wv)
    assert (q.cpu().double() - wq).abs().max() <= 2.0 ** -19 * 6 and (kp.cpu().double() - wk).abs().max() <= 2.0 ** -19 * 6


@pytest.mark.parametrize("seqs", [1, 63, 64, 65, 128, 129])
@pytest.mark.parametrize("last", [0, 1, 30])
def test_batches_about_what_a_wave_looks_through(dev, seqs, last):
    """A wave looks through 64 sequences at a time for a row's own: batches that end there and just past it, with idle
    sequences at both sides of the border, rows behind the last sequence, and append and attention alike."""
    r = np.random.default_rng(seqs + last)
    new = r.choice([0, 1, 2, 19], seqs).tolist()
    new[-1] = last
    for i in (62, 63, 64):
        if i < seqs - 1:
            new[i] = (i + last) % 2
    B = Batch(new, [int(x + r.integers(0, 40)) for x in new], hq=2, hk=1, D=16, page=8, dt=F32, seed=seqs)
    n, freq = sum(new), torch.rand(8)
    more = lambda t: torch.cat([t, torch.full((5, *t.shape[1:]), 7.0)])  # noqa: E731
    q, k, v = more(B.q), more(B.k), more(B.v)
    kp, vp, table, kv_len, cu = B.on(dev)
    qd = q.to(dev)
    rt.op_kv_append(k.to(dev), v.to(dev), kp, vp, table, kv_len, cu, q=qd, inv_freq=freq.to(dev), q_out=qd)
    wq, wk, wv = ref.append(k, v, B.kp, B.vp, B.table, B.kv_len, B.cu, q=q, inv_freq=freq, q_out=q)
    assert torch.equal(vp.cpu().double(), wv) and torch.equal(qd.cpu()[n:], q[n:])
    assert (qd.cpu().double() - wq).abs().max() <= 2.0 ** -19 * 6 and (kp.cpu().double() - wk).abs().max() <= 2.0 ** -19 * 6
    out = torch.full((n + 5, 2, 16), 3.0, device=dev)
    rt.op_paged_attention(q.to(dev), kp, vp, table, kv_len, cu, out=out)
    assert (out[n:] == 3).all()
    B.kp, B.vp = kp.cpu(), vp.cpu()
    attend_check(B, dev)


@pytest.mark.parametrize("n", [2 ** 23 + 1, 2 ** 24])
def test_append_of_the_most_tokens(dev, n):
    """As many rows as the header allows, more than one launch has threads for: every row arrives, the last ones too."""
    page = 4096
    P = -(-n // page)
    qkv = torch.arange(3 * n, dtype=torch.int32, device=dev).view(n, 3, 1).expand(n, 3, 4).contiguous().view(F16)    # 8 dims
    q, k, v = qkv[:, :1], qkv[:, 1:2], qkv[:, 2:]
    kp = torch.zeros(P, page, 1, 8, dtype=F16, device=dev)
    vp = torch.zeros_like(kp)
    table = torch.arange(P, dtype=torch.int32, device=dev)[None].flip(1).contiguous()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    out = rt.op_kv_append(k, v, kp, vp, table, i32(n), i32(0, n), q=q)
    bits = lambda t: t.contiguous().view(torch.int16)  # noqa: E731
    assert torch.equal(bits(out), bits(q))
    for pages, src in ((kp, k), (vp, v)):
        got = bits(pages).flip(0).reshape(-1, 8)
        assert torch.equal(got[:n], bits(src)[:, 0]) and not got[n:].any()


# ---- attention
@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("D", [8, 32, 64, 80, 96, 128, 200, 256])
@pytest.mark.parametrize("page,layout", [(16, "nhd"), (7, "slice")])
def test_attend_one_token(dev, dt, D, page, layout):
    kv = [1, 2, 16, 31, 32, 33, 130, 500]
    attend_check(Batch([1] * 8, kv, hq=4, hk=2, D=D, page=page, dt=dt, seed=D, one=True, layout=layout), dev)


@pytest.mark.parametrize("hq,hk", [(1, 1), (4, 4), (6, 2), (7, 1), (8, 1), (16, 1), (17, 1), (40, 2), (64, 1)])
@pytest.mark.parametrize("dt", [BF16, F32])
def test_attend_groups(dev, hq, hk, dt):
    attend_check(Batch([1, 1, 1], [5, 77, 300], hq=hq, hk=hk, D=64, dt=dt, seed=hq, one=True), dev)
    attend_check(Batch([3, 1, 9], [5, 77, 60], hq=hq, hk=hk, D=64, dt=dt, seed=hq), dev)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("D", [64, 80, 128, 256])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 1), (True, 20), (False, 33), (True, 100000)])
def test_attend_chunks(dev, dt, D, causal, window):
    new, kv = [33, 0, 1, 70, 16, 5], [33, 12, 90, 129, 100, 5]
    attend_check(Batch(new, kv, hq=4, hk=2, D=D, page=16, dt=dt, seed=D + window), dev, causal=causal, window=window)


@pytest.mark.parametrize("page", [1, 3, 16, 31, 64, 100, 256])
@pytest.mark.parametrize("layout", ["nhd", "hnd", "slice"])
def test_attend_pages_and_layouts(dev, page, layout):
    B = Batch([40, 1, 130], [200, 77, 131], hq=6, hk=2, D=64, page=page, dt=BF16, seed=page, layout=layout)
    attend_check(B, dev)
    attend_check(B, dev, causal=False, window=50, scale=0.3)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-4, 1.0])
def test_attend_scales(dev, dt, scale):
    B = Batch([50, 1, 300], [70, 90, 310], hq=2, hk=1, D=64, dt=dt, seed=6)
    attend_check(B, dev, scale=scale)
    attend_check(B, dev, scale=scale, window=31)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("used,total", [(0, 40), (1, 40), (4, 300), (40, 41), (200, 300)])
def test_attend_one_sequence_in_a_padded_call(dev, dt, used, total):
    """One sequence whose rows fill a part of q: the rest of out stays."""
    B = Batch([used], [used + 30], hq=4, hk=1, D=64, dt=dt, seed=used)
    q = torch.randn(total, 4, 64).to(dt)
    kp, vp, table, kv_len, cu = B.on(dev)
    out = torch.full((total, 4, 64), 5.0, dtype=dt, device=dev)
    want, bound, spread = ref.attend(q, B.kp, B.vp, B.table, B.kv_len, B.cu, out=torch.full((total, 4, 64), 5.0))
    for more in (0, 20000):
        out.fill_(5)
        wide = torch.cat([table, torch.full((1, more), -1, dtype=torch.int32, device=dev)], 1)
        rt.op_paged_attention(q.to(dev), kp, vp, wide, kv_len, cu, out=out)
        assert (out[used:] == 5).all()
        check_attend(out.cpu(), want, bound, spread, B, 64)


def test_attend_empty_rows_and_absent_pages(dev):
    """More new tokens than keys, no keys, kv_len below 0 and above the table, pages that are not there, an idle slot."""
    B = Batch([4, 3, 2, 5, 2], [4, 3, 2, 64, 40], hq=4, hk=2, D=64, page=16, dt=BF16, width=4)
    B.kv_len = torch.tensor([2, 0, -3, 70, 40], dtype=torch.int32)
    B.table[4, 0], B.table[4, 1], B.table[3, 2] = -1, 10 ** 6, 77
    got = attend_check(B, dev)
    assert not got[:2].any() and not got[4:9].any()
    B.table[4, :] = -1
    assert not attend_check(B, dev)[14:].any()
    B = Batch([1] * 4, [3, 40, 1, 20], dt=F16, one=True)
    B.kv_len[1] = 0
    assert not attend_check(B, dev)[1].any()


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("causal", [True, False])
def test_attend_more_new_rows_than_keys(dev, dt, causal):
    """positions before the first key, under the longest window"""
    B = Batch([40, 3, 9], [7, 1, 0], D=64, dt=dt)
    for window in (2 ** 31 - 1, 2 ** 30, 3, 0):
        attend_check(B, dev, causal=causal, window=window)


def test_rows_that_descend_are_none(dev):
    """cu_q that goes back: the sequence has no rows, whatever the difference is"""
    B = Batch([2, 3], [5, 6], D=64)
    kp, vp, table, kv_len, _ = B.on(dev)
    cu = torch.tensor([4, -2 ** 31, 3], dtype=torch.int32)      # none, then rows 0 .. 2
    out = torch.full_like(B.q, 7.0)
    got = rt.op_paged_attention(B.q.to(dev), kp, vp, table, kv_len, cu.to(dev), out=out.to(dev))
    want, bound, spread = ref.attend(B.q, B.kp, B.vp, B.table, B.kv_len, cu, out=out)
    check_attend(got.cpu()[:3], want[:3], bound[:3], spread[:3], B, 64)
    assert (got[3:] == 7).all()
    rt.op_kv_append(B.k.to(dev), B.v.to(dev), kp, vp, table, kv_len, cu.to(dev))
    _, wk, wv = ref.append(B.k, B.v, B.kp, B.vp, B.table, B.kv_len, cu)
    assert torch.equal(kp.cpu().double(), wk) and torch.equal(vp.cpu().double(), wv)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_attend_rows_behind_the_last_sequence(dev, dt):
    for new, kv in (([5, 3], [50, 20]), ([1, 1], [3000, 2000])):    # unsplit and split keys
        B = Batch(new, kv, D=64, dt=dt)
        n = sum(new)
        q = torch.cat([B.q, torch.randn(7, 4, 64).to(dt)]).to(dev)
        kp, vp, table, kv_len, cu = B.on(dev)
        out = torch.full((n + 7, 4, 64), 3.0, dtype=dt, device=dev)
        assert rt.op_paged_attention(q, kp, vp, table, kv_len, cu, out=out) is out
        assert (out[n:] == 3).all()
        want, bound, spread = ref.attend(B.q, B.kp, B.vp, B.table, B.kv_len, B.cu)
        check_attend(out[:n].cpu(), want, bound, spread, B, 64)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_attend_hidden_garbage_stays_hidden(dev, dt, D):
    """NaN, infinities and the type's lowest value in slots behind the keys, in pages of nobody, and in keys and values
    that some queries of a tile see and others do not."""
    new, kv = [40, 20, 1], [75, 20, 33]
    B = Batch(new, kv, hq=4, hk=2, D=D, page=16, dt=dt, seed=5)
    flat = [math.nan, math.inf, -math.inf, torch.finfo(dt).min]
    used = torch.zeros(B.kp.shape[:2], dtype=torch.bool)
    for b, m in enumerate(kv):
        for t in range(m):
            used[B.table[b, t // 16].item(), t % 16] = True
    for i, (p, s) in enumerate((~used).nonzero().tolist()):
        B.kp[p, s], B.vp[p, s] = flat[i % 4], flat[(i + 1) % 4]
    attend_check(B, dev)
    attend_check(B, dev, causal=False)

    def at(b, t):
        return B.table[b, t // 16].item(), t % 16

    for b, t, kind in ((0, 60, math.nan), (0, 70, math.inf), (1, 7, -math.inf), (1, 19, math.nan)):
        B.vp[at(b, t)][..., ::3] = kind
    got = attend_check(B, dev)
    assert torch.isfinite(got[:25].float()).all() and torch.isfinite(got[40:47].float()).all()
    attend_check(B, dev, window=5)
    B.kp[at(0, 66)], B.kp[at(1, 15)] = math.nan, math.nan
    attend_check(B, dev)
    attend_check(B, dev, window=9)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_attend_scores_of_minus_infinity(dev, dt):
    """Keys whose score is -inf weigh nothing; a query whose scores all are gives zeros."""
    B = Batch([1, 2], [40, 35], hq=2, hk=1, D=64, dt=dt, seed=2)
    B.q = B.q.abs() + 0.1
    for t in range(0, 40, 2):
        B.kp[B.table[0, t // 16].item(), t % 16, :, 3] = -math.inf
    for t in range(35):
        B.kp[B.table[1, t // 16].item(), t % 16, :, 0] = -math.inf
    assert not attend_check(B, dev)[1:].any()


@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_attend_long_and_split(dev, dt):
    """Long caches with few rows: the keys are split and joined; some splits see no key."""
    attend_check(Batch([1, 1, 1], [9000, 130, 3], hq=4, hk=1, D=128, page=64, dt=dt, one=True, seed=1), dev)
    attend_check(Batch([2, 1, 3], [9000, 3, 700], hq=8, hk=2, D=64, page=16, dt=dt, seed=2), dev)
    attend_check(Batch([2, 1], [9000, 40], hq=2, hk=1, D=64, page=16, dt=dt, seed=3), dev, window=300)


@pytest.mark.parametrize("dt,D", [(F32, 64), (BF16, 128), (F16, 256)])
@pytest.mark.parametrize("far", [9000, 4000])
def test_attend_few_rows_over_long_caches_among_prompts(dev, dt, D, far):
    """Both kernels in one call, the few rows' keys split (into more and into fewer parts than 16): their parts in the
    workspace are numbered by row tiles. Sequences without rows and with more than one head group per tile among them."""
    B = Batch([1, 60, 0, 2, 3, 90], [far, 77, 500, far // 2, 130, 300], hq=8, hk=2, D=D, page=16, dt=dt, seed=far)
    lib, (kp, vp, table, kv_len, cu) = rt.load_library(), B.on(dev)
    kv = rt._paged_kv(torch, kp, vp, table, kv_len, cu, 156)
    assert lib.pfm_paged_attention_ws_bytes(kv, 8) > 0
    attend_check(B, dev)
    attend_check(B, dev, window=far // 2 + 9, causal=False)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("new,kv,one", [([1] * 3, [500, 480, 450], True), ([1, 1], [8192, 3000], True), ([70, 3], [4100, 9000], False),
                                        ([300], [1500], False)])
@pytest.mark.parametrize("sink", [0, 700])
@pytest.mark.parametrize("start", [-30.0, -5.0])
def test_attend_tail_behind_a_dominant_key(dev, dt, new, kv, one, sink, start):
    """One key takes nearly all the weight and has no value; thousands of keys at 2^-25 .. 2^-28 of it make the output. Each
    weight's rounding is relative down to 2^-29 of the largest (f16's normal range below 2^15), and absolute under it, 2^-40
    per key for single tokens and 2^-32 for chunks, so that the tail is summed as well as anything else: to f16 itself, under 2^-25 it is nothing. start:
    score of the first keys, under the dominant one's by less or by more than the kernels rescale at.
    Tolerance: as for all attention, those per key (values are under 2), and half a step of f16's subnormal results."""
    B = Batch(new, kv, hq=4, hk=2, D=64, dt=dt, one=one, seed=sink)
    g = torch.Generator().manual_seed(7)
    B.q[:] = 0
    B.q[..., 0] = 1
    for b, m in enumerate(kv):
        t = torch.arange(m)
        at = B.table[b, t // 16].long(), t % 16
        x = -math.log(2) * (25.2 + 2.8 * torch.rand(m, 2, generator=g))
        x[:5] = start
        x[min(sink, m // 2)] = 0
        v = 1 + torch.rand(m, 2, 64, generator=g)
        v[:5] = v[min(sink, m // 2)] = 0
        k = torch.zeros(m, 2, 64)
        k[..., 0] = x
        B.kp[at], B.vp[at] = k.to(dt), v.to(dt)
    kp, vp, table, kv_len, cu = B.on(dev)
    got = rt.op_paged_attention(B.q.to(dev), kp, vp, table, kv_len, cu, scale=1.0).cpu().double()
    want, bound, spread = ref.attend(B.q, B.kp, B.vp, B.table, B.kv_len, B.cu, scale=1.0)
    assert want.min() > 2.0 ** -18          # the tail is there: f16's smallest normal number is 2^-14, its half step 2^-25
    u, L = half_step(dt), max(kv)
    d = (64 + 8) * 2.0 ** -24 * spread[..., None] * 2 + 2.0 ** -20 + L * 2.0 ** -24
    tol = (u + d) * bound * 1.05 + u * want * 1.05 + L * 2.0 * 2.0 ** (-40 if one else -32) + 2.0 ** -25
    err = (got - want).abs()
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("dt,q,k", [(F16, 301, 299), (F16, 3001, 2999), (F16, 30016, 29984), (BF16, 3e4, 3e4), (BF16, 1e9, 3e9), (F32, 3001, 2999),
                                    (F32, 123456.7, 9876.5), (F32, 1e13, 7e13)])
@pytest.mark.parametrize("new,kv,one", [([1, 1], [300, 5000], True), ([200, 2], [700, 300], False)])
@pytest.mark.parametrize("sign", [1, -1])
def test_attend_scores_of_any_size(dev, dt, q, k, new, kv, one, sign):
    """Equal scores up to 10^28, where a step of a score is more than the exponential's whole range: all keys that a query
    sees weigh alike, whichever side of 0 they are on, and the first three, with scores of the other sign, or of 0, nothing
    or all. Weights are equal or 0, so the tolerance is that of the sums, of a weight's and of the result's rounding."""
    B = Batch(new, kv, hq=4, hk=2, D=64, dt=dt, one=one, seed=3)
    B.q[:], B.kp[:] = q, sign * k
    B.vp = (B.vp.float().abs() + 1).to(dt)
    for b in range(len(kv)):
        for t, f in ((0, -1), (1, 0), (2, -1)):
            B.kp[B.table[b, 0].item(), t] *= f
    kp, vp, table, kv_len, cu = B.on(dev)
    want, bound, _ = ref.attend(B.q, B.kp, B.vp, B.table, B.kv_len, B.cu)
    u = half_step(dt)
    tol = (u + 2.0 ** -20 + max(kv) * 2.0 ** -24) * bound * 1.05 + u * want * 1.05
    for far in (0, 1000):                   # further table entries of no page: how far it reaches says which kernels run
        wide = torch.cat([table, torch.full((len(kv), far), -1, dtype=torch.int32, device=dev)], 1)
        got = rt.op_paged_attention(B.q.to(dev), kp, vp, wide, kv_len, cu).cpu().double()
        assert torch.isfinite(got).all()
        assert ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol).max())


@pytest.mark.parametrize("new,one", [([1, 1], True), ([200, 2], False)])
def test_attend_scores_past_32_bits_are_no_numbers(dev, new, one):
    """q k is a number of 32 bits, its multiple in the exponent's base is not: NaN, as from inf - inf, and no zeros."""
    B = Batch(new, [300, 250], hq=4, hk=2, D=64, dt=F32, one=one, seed=3)
    B.q[:], B.kp[:] = 1e18, 3e38 / 64 / 1e18
    kp, vp, table, kv_len, cu = B.on(dev)
    for far in (0, 1000):
        wide = torch.cat([table, torch.full((2, far), -1, dtype=torch.int32, device=dev)], 1)
        assert torch.isnan(rt.op_paged_attention(B.q.to(dev), kp, vp, wide, kv_len, cu, scale=1.0)).all()


def test_attend_large_scores(dev):
    """Scores of thousands: one key takes all; the running maximum rises late."""
    B = Batch([1, 30], [200, 400], hq=2, hk=2, D=64, dt=F32, seed=3)
    B.q *= 30
    B.kp *= 30
    kp, vp, table, kv_len, cu = B.on(dev)
    got = rt.op_paged_attention(B.q.to(dev), kp, vp, table, kv_len, cu).cpu()
    want, bound, spread = ref.attend(B.q, B.kp, B.vp, B.table, B.kv_len, B.cu)
    check_attend(got, want, bound, spread, B, 64)


@pytest.mark.parametrize("n,mq", [(260, 40), (600, 9)])
def test_attend_many_sequences(dev, n, mq):
    """More sequences than a wave looks through at once, idle ones and single tokens among chunks."""
    r = np.random.default_rng(n)
    new = [int(x) for x in r.choice([0, 1, 1, 2, mq], n // 4)]
    new[0] = 1
    B = Batch(new, [int(x + r.integers(0, 60)) for x in new], hq=2, hk=1, D=32, page=8, dt=F32, seed=n)
    attend_check(B, dev)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("new", [0, 2])
def test_attend_one_long_among_many_short(dev, dt, new):
    """parts of the long cache alone; new 0: a token each, without cu_q"""
    kv = [3 + i % 90 for i in range(270)]
    kv[131], kv[7], kv[0] = 17000, 8193, 0
    B = Batch([1] * 270 if not new else [new - i % 2 for i in range(270)], kv, hq=16, hk=8, D=16, dt=dt, one=not new)
    attend_check(B, dev)
    attend_check(B, dev, window=9000, causal=bool(new))


def test_attend_shared_pages(dev):
    """Sequences that share a prefix's pages; one block table row for all (stride 0)."""
    B = Batch([1, 1, 1], [48, 48, 48], dt=BF16, one=True)
    B.table[1, :2], B.table[2, :2] = B.table[0, :2], B.table[0, :2]
    attend_check(B, dev)
    B.table[:] = B.table[0].clone()
    want, bound, spread = ref.attend(B.q, B.kp, B.vp, B.table, B.kv_len)
    kp, vp, table, kv_len, _ = B.on(dev)
    with pytest.raises(rt.PfmError):      # a table whose rows lie on each other is refused
        rt.op_paged_attention(B.q.to(dev), kp, vp, table[:1].expand(3, -1), kv_len)
    check_attend(rt.op_paged_attention(B.q.to(dev), kp, vp, table, kv_len).cpu(), want, bound, spread, B, 64)


@pytest.mark.parametrize("op", ["append", "attend"])
def test_offsets_past_32_bits(dev, op):
    """Pages beyond 2^31 elements of the pool (4.6 GB of it; only the last pages are used)."""
    pages, page, hk, D = 2 ** 31 // (64 * 8 * 128) + 40, 64, 8, 128
    B = Batch([3, 1], [100, 70], hq=16, hk=hk, D=D, page=page, dt=BF16)
    P = B.kp.shape[0]
    kp = torch.zeros((pages, page, hk, D), dtype=BF16, device=dev)
    vp = torch.zeros_like(kp)
    kp[-P:], vp[-P:] = B.kp.to(dev), B.vp.to(dev)
    table = torch.where(B.table >= 0, B.table + (pages - P), B.table).to(dev)
    args = (kp, vp, table, B.kv_len.to(dev), B.cu.to(dev))
    if op == "attend":
        want, bound, spread = ref.attend(B.q, B.kp, B.vp, B.table, B.kv_len, B.cu)
        check_attend(rt.op_paged_attention(B.q.to(dev), *args).cpu(), want, bound, spread, B, D)
    else:
        rt.op_kv_append(B.k.to(dev), B.v.to(dev), *args)
        _, wk, wv = ref.append(B.k, B.v, B.kp, B.vp, B.table, B.kv_len, B.cu)
        assert torch.equal(kp[-P:].cpu().double(), wk) and torch.equal(vp[-P:].cpu().double(), wv)
        assert not kp[:-P].any() and not vp[:-P].any()


# ---- sampling
def sample_check(dev, x, u, **kw):
    on = {k: None if v is None else v.to(dev) for k, v in kw.items()}
    t, p = rt.op_sample(x.to(dev), u.to(dev), **on)
    wt, wp = ref.sample(x, u, **kw)
    assert t.tolist() == wt
    assert np.allclose(p.cpu().numpy(), np.array(wp), rtol=2.0 ** -23, atol=0)
    return t


def settings(B, mode, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda a, b: a + (b - a) * torch.rand(B, generator=g)  # noqa: E731
    some = lambda t, off: torch.where(torch.rand(B, generator=g) < 0.6, t, torch.full_like(t, off))  # noqa: E731
    kw = {}
    if mode != "plain":
        kw["temperature"] = some(r(0.2, 1.6), 0.0 if mode == "mixed" else 1.0)
    if mode in ("topk", "mixed", "topk_topp"):
        kw["top_k"] = some(torch.randint(1, 300, (B,), generator=g, dtype=torch.int32), 0)
    if mode in ("topp", "mixed", "topk_topp"):
        kw["top_p"] = some(r(0.05, 0.999), 1.0)
    if mode in ("minp", "mixed"):
        kw["min_p"] = some(r(0.0, 0.3), 0.0)
    return kw


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("V", [1, 2, 63, 64, 1000, 8404, 25055, 100003])
@pytest.mark.parametrize("mode", ["plain", "topk", "topp", "minp", "topk_topp", "mixed"])
def test_sample(dev, dt, V, mode):
    B = 12
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(B, V, generator=g) * 2.5).to(dt)
    sample_check(dev, x, torch.rand(B, generator=g), **settings(B, mode, V))


@pytest.mark.parametrize("off", range(8))
@pytest.mark.parametrize("dt", [F32, BF16])
def test_sample_strided_rows(dev, off, dt):
    """Rows that begin anywhere in a 16-byte piece and are parts of longer ones; what lies around them is not read in."""
    g = torch.Generator().manual_seed(off)
    wide = torch.full((5, 3001 + off), 1e4).to(dt)
    x = (torch.randn(5, 2500, generator=g) * 3).to(dt)
    w = wide.to(dev)
    w[:, off:off + 2500] = x.to(dev)
    view = w[:, off:off + 2500]
    u = torch.rand(5, generator=g)
    for kw in ({}, dict(top_k=torch.full((5,), 40, dtype=torch.int32)), dict(top_p=torch.full((5,), 0.9))):
        t, _ = rt.op_sample(view, u.to(dev), **{k: v.to(dev) for k, v in kw.items()})
        assert t.tolist() == ref.sample(x, u, **kw)[0]


@pytest.mark.parametrize("V", [5, 3000, 50001])
def test_sample_ties_and_flat_rows(dev, V):
    """All logits equal (more in one bin than are sorted at once), two levels, and steps: ties go by index."""
    g = torch.Generator().manual_seed(V)
    rows = [torch.zeros(V), torch.full((V,), -3.5), (torch.arange(V) % 2).float(), (torch.arange(V) // 7).float() / V,
            torch.randint(0, 3, (V,), generator=g).float() * 1e-3, -(torch.arange(V) % 2).float() * 0.0]
    x = torch.stack(rows)
    for u in (0.0, 0.37, 0.99999994):
        uu = torch.full((len(rows),), u)
        sample_check(dev, x, uu)
        for k in (1, 2, V // 2 + 1, V, V + 7):
            sample_check(dev, x, uu, top_k=torch.full((len(rows),), k, dtype=torch.int32))
        for p in (0.0, 1e-6, 0.5, 0.9):
            sample_check(dev, x, uu, top_p=torch.full((len(rows),), p))
        sample_check(dev, x, uu, top_p=torch.full((len(rows),), 0.4), top_k=torch.full((len(rows),), V // 2 + 1, dtype=torch.int32),
                     min_p=torch.full((len(rows),), 0.999))


def test_sample_infinities_nan_and_empty_rows(dev):
    V, inf, nan = 4000, math.inf, math.nan
    x = torch.randn(9, V)
    x[0] = -inf
    x[1] = nan
    x[2, 5:] = -inf
    x[3, ::2] = nan
    x[4, 17] = x[4, 900] = inf
    x[5] = torch.finfo(F32).min
    x[6] = torch.finfo(F32).min
    x[6, 77] = torch.finfo(F32).max
    x[7] = -inf
    x[7, 3999] = -1e30
    x[8, :100] = -nan
    u = torch.rand(9)
    for kw in ({}, dict(temperature=torch.zeros(9)), dict(top_k=torch.full((9,), 3, dtype=torch.int32)),
               dict(top_p=torch.full((9,), 0.7)), dict(min_p=torch.full((9,), 0.2)), dict(temperature=torch.full((9,), 1e-30)),
               dict(temperature=torch.full((9,), 1e30), top_p=torch.full((9,), 0.5))):
        t = sample_check(dev, x, u, **kw)
        assert t[0] == -1 and t[1] == -1 and t[7] == 3999 and t[6] == 77 and t[4] in (17, 900)


def test_sample_settings_out_of_range(dev):
    """Settings that switch a filter off or are no numbers, uniform numbers at the ends."""
    V = 3000
    x = torch.randn(8, V) * 2
    full = lambda v: torch.full((8,), v)  # noqa: E731
    base = sample_check(dev, x, full(0.5))
    for kw in (dict(top_k=full(0).int()), dict(top_k=full(-4).int()), dict(top_k=full(V).int()), dict(top_p=full(1.0)),
               dict(top_p=full(2.0)), dict(top_p=full(math.nan)), dict(min_p=full(0.0)), dict(min_p=full(-1.0))):
        t, _ = rt.op_sample(x.to(dev), full(0.5).to(dev), **{k: v.to(dev) for k, v in kw.items()})
        assert torch.equal(t, base)
    best = x.argmax(-1).int().tolist()
    for kw in (dict(top_p=full(-1.0)), dict(min_p=full(5.0)), dict(temperature=full(-1.0)), dict(temperature=full(math.nan))):
        assert rt.op_sample(x.to(dev), full(0.5).to(dev), **{k: v.to(dev) for k, v in kw.items()})[0].tolist() == best
    assert rt.op_sample(x.to(dev), full(0.0).to(dev))[0].tolist() == [0] * 8
    for u in (1.0, 1.5, math.inf):
        assert rt.op_sample(x.to(dev), full(u).to(dev))[0].tolist() == ref.sample(x, full(min(u, 1.0)))[0]
    assert torch.equal(rt.op_sample(x.to(dev), full(math.nan).to(dev))[0], rt.op_sample(x.to(dev), full(0.0).to(dev))[0])


@pytest.mark.parametrize("V", [12287, 12288, 12289])
@pytest.mark.parametrize("mode", ["plain", "topp", "mixed"])
def test_sample_about_the_longest_row_of_one_workgroup(dev, V, mode):
    B = 9
    g = torch.Generator().manual_seed(V)
    x = torch.randn(B, V, generator=g) * 3
    sample_check(dev, x, torch.rand(B, generator=g), **settings(B, mode, V))


@pytest.mark.parametrize("V", [50, 8404, 20000])
@pytest.mark.parametrize("T", [math.inf, 1e30, 1e4])
def test_sample_high_temperatures(dev, V, T):
    """all logits above -inf alike; the order of tokens is still that of their logits"""
    B = 12
    g = torch.Generator().manual_seed(int(V))
    x = torch.randn(B, V, generator=g) * 5
    x[1, ::3], x[2, :V // 2], x[3] = -math.inf, -math.inf, 1.0
    u = torch.rand(B, generator=g)
    t = torch.full((B,), T)
    k, p = torch.tensor([0, V // 3 + 1, 2] * 4, dtype=torch.int32), torch.tensor([0.9, 0.5, 1.0, 0.01] * 3)
    sample_check(dev, x, u, temperature=t)
    sample_check(dev, x, u, temperature=t, top_p=p)
    sample_check(dev, x, u, temperature=t, top_k=k)
    sample_check(dev, x, u, temperature=t, top_k=k, top_p=p)


def test_sample_does_not_depend_on_the_batch(dev):
    g = torch.Generator().manual_seed(4)
    x = (torch.randn(64, 40000, generator=g) * 3).to(dev)
    u = torch.rand(64, generator=g).to(dev)
    kw = {k: v.to(dev) for k, v in settings(64, "mixed", 9).items()}
    t, p = rt.op_sample(x, u, **kw)
    for i in range(0, 64, 9):
        t1, p1 = rt.op_sample(x[i:i + 1], u[i:i + 1], **{k: v[i:i + 1] for k, v in kw.items()})
        assert t1[0] == t[i] and p1[0] == p[i]


def test_sample_follows_the_distribution(dev):
    """200,000 draws of one row: every count within 6 standard deviations of its expectation."""
    n, V = 200000, 50
    p = torch.softmax(torch.randn(V, generator=torch.Generator().manual_seed(0)), 0)
    t, _ = rt.op_sample(p.log()[None].repeat(n, 1).to(dev), ((torch.arange(n) + 0.5) / n).to(dev))
    c = torch.bincount(t.long().cpu(), minlength=V).double() / n
    assert ((c - p.double()).abs() <= 2.0 / n + 1e-6).all()      # u is evenly spaced: within one step at each end


# ---- together
def _decoder_step(x, w, state, u, set_, freq, heads, lens):
    """One token of every sequence through one attention layer of a small decoder."""
    hq, hk, D = heads
    kp, vp, table = state
    qkv = (x @ w["qkv"]).view(x.shape[0], hq + 2 * hk, D)
    q = rt.op_kv_append(qkv[:, hq:hq + hk], qkv[:, hq + hk:], kp, vp, table, lens, q=qkv[:, :hq], inv_freq=freq)
    o = rt.op_paged_attention(q, kp, vp, table, lens)
    logits = x @ w["skip"] + o.reshape(x.shape[0], hq * D) @ w["out"]
    return rt.op_sample(logits, u, **set_)


def _decoder(dev, dt, B=3, V=500, hq=4, hk=2, D=64, width=96):
    g = torch.Generator().manual_seed(11)
    w = {"emb": torch.randn(V, width, generator=g), "qkv": torch.randn(width, (hq + 2 * hk) * D, generator=g) / width ** 0.5,
         "out": torch.randn(hq * D, V, generator=g) / 4, "skip": torch.randn(width, V, generator=g) / width ** 0.5 * 2}
    return {k: v.to(dt).to(dev) for k, v in w.items()}, (1e4 ** (-torch.arange(D // 2) / (D // 2))).to(dev), (hq, hk, D)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_prompt_then_tokens_equals_all_at_once(dev, dt):
    """A prompt in one chunk, then tokens one by one: each step's attention equals the same rows of one pass over all
    the tokens (other tiles and splits: to the type's rounding), and append writes the same bits either way."""
    w, freq, (hq, hk, D) = _decoder(dev, dt)
    g = torch.Generator().manual_seed(3)
    n, prompt, page = 60, [37, 50, 1], 16
    ids = [torch.randint(0, 500, (n,), generator=g).to(dev) for _ in prompt]
    table = torch.randperm(12, generator=g)[:12].view(3, 4).int().to(dev)
    # the projections once for all rows: only the attention differs
    rows = [(w["emb"][i] @ w["qkv"]).view(n, hq + 2 * hk, D) for i in ids]

    def pages():
        return (torch.zeros(12, page, hk, D, dtype=dt, device=dev) for _ in range(2))

    def go(state, x, lens, cu):
        q = rt.op_kv_append(x[:, hq:hq + hk], x[:, hq + hk:], *state, table, lens, cu, q=x[:, :hq], inv_freq=freq)
        return rt.op_paged_attention(q, *state, table, lens, cu)

    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    whole = tuple(pages())
    want = go(whole, torch.cat(rows), i32([n] * 3), i32([0, n, 2 * n, 3 * n])).view(3, n, hq, D)
    parts = tuple(pages())
    o = go(parts, torch.cat([r[:p] for r, p in zip(rows, prompt)]), i32(prompt), i32([0, 37, 87, 88]))
    # two evaluations, each with a rounding of p and one of the result (sum_j p_j |v_j| < 1.5 here) and the f32 sums' part
    # of D + 8 = 72 products at a spread under 10
    tol = dict(rtol=0, atol=2 * (1.5 * 2 * half_step(dt) + 2 * 72 * 2.0 ** -24 * 10 * 1.5))
    at = 0
    for b, p in enumerate(prompt):
        torch.testing.assert_close(o[at:at + p], want[b, :p], **tol)
        at += p
    for t in range(n - max(prompt)):
        lens = [p + t + 1 for p in prompt]
        o = go(parts, torch.stack([r[m - 1] for r, m in zip(rows, lens)]), i32(lens), None)
        for b, m in enumerate(lens):
            torch.testing.assert_close(o[b], want[b, m - 1], **tol)
    for a, b in zip(whole, parts):
        for s in range(3):
            m = prompt[s] + n - max(prompt)
            flat = lambda x: x[table[s].long()].reshape(-1, hk, D)[:m]  # noqa: E731
            assert torch.equal(flat(a), flat(b))


def test_decode_loop_in_a_graph(dev):
    """The step captured once and replayed for every token, lengths and tokens in place, eager work between replays;
    two graphs of the same step share no workspace: replayed in turn they give the eager run's tokens."""
    dt, B, steps = BF16, 3, 12
    w, freq, heads = _decoder(dev, dt)
    hq, hk, D = heads
    g = torch.Generator().manual_seed(5)
    us = torch.rand(steps, B, generator=g).to(dev)
    table = torch.randperm(300, generator=g).view(3, 100).int().to(dev)
    start = [7, 1500, 400]
    fill = [torch.randn(300, 16, hk, D, generator=g).to(dt).to(dev) for _ in range(2)]
    set_ = dict(temperature=torch.tensor([0.8, 0.0, 1.1], device=dev), top_k=torch.tensor([40, 0, 0], dtype=torch.int32, device=dev),
                top_p=torch.tensor([0.9, 1.0, 0.8], device=dev))

    def eager():
        state, lens = (*(f.clone() for f in fill), table), torch.tensor(start, dtype=torch.int32, device=dev)
        tok, out = torch.tensor([1, 2, 3], device=dev), []
        for t in range(steps):
            lens += 1
            tok, prob = _decoder_step(w["emb"][tok.long()], w, state, us[t], set_, freq, heads, lens)
            out.append((tok.tolist(), prob.tolist()))
        return out

    want = eager()
    state, lens = (*(f.clone() for f in fill), table), torch.tensor(start, dtype=torch.int32, device=dev)
    tok, u = torch.tensor([1, 2, 3], device=dev, dtype=torch.int32), torch.zeros(B, device=dev)
    side = torch.cuda.Stream()
    graphs = []
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _decoder_step(w["emb"][tok.long()], w, state, u, set_, freq, heads, lens)   # warm-up (one slot, rewritten later)
    torch.cuda.synchronize()
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            lens += 1
            nt, prob = _decoder_step(w["emb"][tok.long()], w, state, u, set_, freq, heads, lens)
            tok.copy_(nt)
        graphs.append((gr, prob))
    for rep in range(2):
        for s, f in zip(state, fill):
            s.copy_(f)
        lens.copy_(torch.tensor(start, dtype=torch.int32))
        tok.copy_(torch.tensor([1, 2, 3]))
        for t in range(steps):
            u.copy_(us[t])
            gr, prob = graphs[t % 2]
            gr.replay()
            torch.cuda.synchronize()
            assert (tok.tolist(), prob.tolist()) == want[t], (rep, t)
            if t % 3 == 0:
                rt.op_sample(torch.randn(2, 700, device=dev), torch.rand(2, device=dev))   # eager work between replays
    assert eager() == want


@pytest.mark.parametrize("dt", [F32, BF16])
def test_chunks_in_a_graph(dev, dt):
    """One captured append and attention of chunks, replayed for batches of other lengths in the same buffers: single
    tokens over long caches, prompts, idle sequences and rows behind the last one, eager calls between the replays."""
    n, hq, hk, D, page, freq = 300, 8, 2, 64, 16, torch.rand(32)
    batches = [([1, 250, 0, 3], [9000, 400, 77, 500]), ([75] * 4, [75, 1000, 80, 3000]), ([300, 0, 0, 0], [4000, 1, 0, 30]),
               ([1, 1, 1, 1], [9000, 8000, 17, 1]), ([0, 0, 0, 0], [5, 5, 5, 5]), ([0, 120, 180, 0], [0, 9000, 180, 0])]
    state = lambda B: (B.q, B.k, B.v, B.kp, B.vp, B.table, B.kv_len, B.cu)  # noqa: E731
    P, W = 1500, -(-9000 // page)

    def padded(new, kv, seed):
        B = Batch(new, kv, hq=hq, hk=hk, D=D, page=page, dt=dt, seed=seed)
        fill = lambda t, m: torch.cat([t, torch.full((m - t.shape[0], *t.shape[1:]), 0.25, dtype=t.dtype)])  # noqa: E731
        B.q, B.k, B.v, B.kp, B.vp = fill(B.q, n), fill(B.k, n), fill(B.v, n), fill(B.kp, P), fill(B.vp, P)
        B.table = torch.cat([B.table, torch.full((4, W - B.table.shape[1]), -1, dtype=torch.int32)], 1)
        return state(B)

    hosts = [padded(*b, seed=i) for i, b in enumerate(batches)]
    freq = freq.to(dev)

    def step(q, k, v, kp, vp, table, lens, cu, qo, out):
        rt.op_kv_append(k, v, kp, vp, table, lens, cu, q=q, inv_freq=freq, q_out=qo)
        rt.op_paged_attention(qo, kp, vp, table, lens, cu, out=out)

    want = []
    for h in hosts:
        a = [t.to(dev) for t in h]
        qo, out = torch.full_like(a[0], 5.0), torch.full_like(a[0], 6.0)
        step(*a, qo, out)
        want.append((qo, out, a[3], a[4]))
    bufs = [t.to(dev) for t in hosts[0]]
    qo, out = torch.full_like(bufs[0], 5.0), torch.full_like(bufs[0], 6.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*bufs, qo, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*bufs, qo, out)
    for i in (0, 1, 2, 3, 4, 5, 3, 1, 0):
        for t, h in zip(bufs, hosts[i]):
            t.copy_(h)
        qo.fill_(5)
        out.fill_(6)
        graph.replay()
        torch.cuda.synchronize()
        for got, w in zip((qo, out, bufs[3], bufs[4]), want[i]):
            assert torch.equal(got, w), i
        rt.op_paged_attention(want[1][0], *[t.to(dev) for t in hosts[1][3:]])       # eager work between replays


@pytest.mark.parametrize("V", [5000, 60000])
def test_sampling_in_a_graph_follows_its_settings(dev, V):
    """One captured draw, replayed with other logits and settings in the same buffers: rows change between the largest
    logit, no filter, few candidates, a wide nucleus, +inf and none at all."""
    B, g = 12, torch.Generator().manual_seed(V)
    x, u = torch.zeros(B, V, device=dev), torch.zeros(B, device=dev)
    off = dict(temperature=torch.ones(B), top_k=torch.zeros(B, dtype=torch.int32), top_p=torch.ones(B), min_p=torch.zeros(B))
    kw = {k: v.to(dev) for k, v in off.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rt.op_sample(x, u, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        token, prob = rt.op_sample(x, u, **kw)
    for i, mode in enumerate(["mixed", "topp", "plain", "topk", "minp", "topk_topp", "mixed", "topp"]):
        h = torch.randn(B, V, generator=g) * (3 if i % 2 else 0.5)
        h[i] = -math.inf
        h[i + 1, 7::V // 3] = math.inf
        uu, s = torch.rand(B, generator=g), off | settings(B, mode, i)
        x.copy_(h)
        u.copy_(uu)
        for k, t in kw.items():
            t.copy_(s[k])
        graph.replay()
        torch.cuda.synchronize()
        wt, wp = ref.sample(h, uu, **s)
        assert token.tolist() == wt, mode
        assert np.allclose(prob.cpu().numpy(), np.array(wp), rtol=2.0 ** -23, atol=0)
        rt.op_sample(torch.randn(2, 70000, device=dev), torch.rand(2, device=dev), top_p=torch.full((2,), 0.9, device=dev))


def test_other_streams_at_once(dev):
    """Two streams with batches of their own, queued without waiting for each other."""
    B1 = Batch([1] * 4, [3000, 2000, 100, 7], hq=8, hk=2, D=128, page=64, dt=BF16, one=True, seed=1)
    B2 = Batch([30, 200], [900, 400], hq=8, hk=2, D=128, page=64, dt=BF16, seed=2)
    ins = [(B, B.q.to(dev), B.on(dev)) for B in (B1, B2)]
    alone = [rt.op_paged_attention(q, *a) for _, q, a in ins]
    x, u = torch.randn(8, 50000, device=dev), torch.rand(8, device=dev)
    tok = rt.op_sample(x, u)[0]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for st, (_, q, a) in zip(streams, ins):
            with torch.cuda.stream(st):
                got.append((rt.op_paged_attention(q, *a), rt.op_sample(x, u)[0]))
        torch.cuda.synchronize()
        for (o, t), w in zip(got, alone):
            assert torch.equal(o, w) and torch.equal(t, tok)


def test_host_memory_refused(dev):
    """Host tensors reach no kernel."""
    B = Batch([1, 1], [5, 6], one=True)
    kp, vp, table, kv_len, _ = B.on(dev)
    with pytest.raises(rt.PfmError):
        rt.op_paged_attention(B.q, kp, vp, table, kv_len)
    with pytest.raises(rt.PfmError):
        rt.op_paged_attention(B.q.to(dev), kp, vp, B.table, kv_len)
    lib, kv = rt.load_library(), rt.PfmPagedKv.from_buffer_copy(rt._paged_kv(torch, kp, vp, table, kv_len, None, 2))
    q, host = B.q.to(dev), torch.zeros(4, dtype=torch.int32)
    rows = rt._rows(q, (2, 4, 64), BF16, q.device, "q")
    kv.kv_len = host.data_ptr()
    assert lib.pfm_op_paged_attention(None, ctypes.byref(kv), rows, rows, 4, 1.0, 1, 0, None, 0) == -1
    assert b"kv_len" in lib.pfm_last_error()
