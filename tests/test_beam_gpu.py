"""The hypotheses' operators on the GPU against the 64-bit oracle (oracle/beam.py) and the one-row operators they extend.

Tolerances, from the arithmetic (u = half a step of a type: bf16 2^-8, fp16 2^-11, fp32 2^-24):
- RoPE: two fp32 products and their sum, then one rounding to the type.
- attention: a score is an fp32 sum of 128 products (each term passes at most 128 additions, and the scaling), so off by at
  most 132 u32 scale sum |q k|; exp of it in fp32 adds 2^-21 + |s| 2^-22 relative; a weight may be rounded to the
  activations' type, or to fp16 with an int8 V row's scale in it, before it meets V, u. Those perturb o = sum w v /
  sum w by at most twice their sum times sum w |v| / sum w (numerator and normaliser); fp32 sums over n slots by
  (n / 32 + 64) u32 of the same; the result is rounded once, u |o|.
- the selection: whole numbers equal (the inputs' values are far apart, or equal); a score is its fp32 rounding plus the
  error of log sum exp, whose fp32 sum of V terms is off by a relative 2^-18 at most.
"""
import math

import numpy as np
import pytest
import torch

import beam
import decode
import fused
import kv8
import mm_int4
import prefill
from oracle import beam as OB

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
U = {F16: 2.0 ** -11, BF16: 2.0 ** -8, torch.float32: 2.0 ** -24}
HD = 128


def i64(dev, *v):
    return torch.tensor(v, dtype=torch.int64, device=dev)


def as_cache(x, q8):
    """x on the GPU as a plain cache or an int8 one, and its values in float64"""
    if not q8:
        return x, x.double().cpu().numpy()
    a = torch.empty_like(x)
    c, c2 = kv8.empty(*x.shape, device=x.device), kv8.empty(*x.shape, device=x.device)
    a.copy_(x)
    kv8.quantize(a, a, c, c2)
    return c, (c[0].double() * c[1].double()[..., None]).cpu().numpy()


# -------------------------------------------------------------------------------------------------------------- post
def _post_case(dev, dt, B, nkv, rep, inter, T, q8, seed, stride=0, P=64):
    g = torch.Generator(device=dev).manual_seed(seed)
    NH = nkv * rep
    y = torch.randn(B, (NH + 2 * nkv) * HD + 2 * inter + stride, device=dev, dtype=dt, generator=g)
    cos, sin = decode.rope_tables(P, HD, 10000.0, dt, dev)
    if q8:
        ks, vs = (tuple(t.fill_(9) for t in kv8.empty(B, nkv, T, HD, device=dev)) for _ in range(2))
    else:
        ks, vs = (torch.full((B, nkv, T, HD), 9.0, device=dev, dtype=dt) for _ in range(2))
    q = torch.full((B, NH * HD), 9.0, device=dev, dtype=dt)
    act = torch.full((B, inter), 9.0, device=dev, dtype=dt)
    return y[:, :y.shape[1] - stride], cos, sin, ks, vs, q, act


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("B,nkv,rep,inter,T,stride", [(1, 1, 1, 8, 1, 0), (3, 4, 4, 100, 9, 0), (5, 2, 1, 7, 4, 3),
                                                      (17, 4, 2, 2056, 3, 8), (33, 1, 8, 64, 40, 0)])
@pytest.mark.parametrize("rope", [True, False])
def test_post(dt, q8, B, nkv, rep, inter, T, stride, rope, dev):
    NH, plen = nkv * rep, 11
    y, cos, sin, ks, vs, q, act = _post_case(dev, dt, B, nkv, rep, inter, T, q8, B, stride)
    slot = [(b * 7) % T for b in range(B)]
    beam.post(y, i64(dev, *slot), i64(dev, plen), cos, sin, ks, vs, q, act, NH=NH, NKV=nkv, HD=HD, ROPE=rope)
    yd = y.double().cpu().numpy()
    heads = yd[:, :(NH + 2 * nkv) * HD].reshape(B, -1, HD)
    want, err = heads.copy(), np.zeros_like(heads)
    if rope:
        at, n = np.array(slot) + plen, NH + nkv
        c, s = (t.double().cpu().numpy()[at][:, None, ::2] for t in (cos, sin))
        e, o = heads[:, :n, ::2], heads[:, :n, 1::2]
        want[:, :n, ::2], want[:, :n, 1::2] = e * c - o * s, o * c + e * s
        mag = np.abs(e * c) + np.abs(o * s), np.abs(o * c) + np.abs(e * s)
        for i in range(2):
            err[:, :n, i::2] = 2 * U[torch.float32] * mag[i] + U[dt] * np.abs(want[:, :n, i::2]) * (1 + 1e-6) + 1e-8
    got = q.double().cpu().numpy().reshape(B, NH, HD)
    assert np.all(np.abs(got - want[:, :NH]) <= err[:, :NH])
    for cache, lo in ((ks, NH), (vs, NH + nkv)):
        rows = cache[0] if q8 else cache
        for b in range(B):
            x = rows[b, :, slot[b]].double().cpu().numpy()
            if q8:
                scale = cache[1][b, :, slot[b]].cpu().numpy()
                x = x * scale[:, None].astype(np.float64)
                # a code step beside the rounding of the value that it stands for
                assert np.all(np.abs(x - want[b, lo:lo + nkv]) <= err[b, lo:lo + nkv] + scale[:, None] * (0.5 + 1e-6))
            else:
                assert np.all(np.abs(x - want[b, lo:lo + nkv]) <= err[b, lo:lo + nkv])
            others = [t for t in range(T) if t != slot[b]]
            assert (rows[b, :, others] == 9).all() and (not q8 or (cache[1][b, :, others] == 9).all())
    gate, up = yd[:, -2 * inter:-inter], yd[:, -inter:]
    ref = gate / (1 + np.exp(-gate)) * up
    assert np.all(np.abs(act.double().cpu().numpy() - ref) <= np.abs(ref) * (U[dt] + 2.0 ** -19) + 1e-7)


@pytest.mark.parametrize("dt", [F16, BF16])
def test_post_is_the_one_row_post(dt, dev):
    """B rows give what fused.post gives for each, bit for bit; an int8 cache holds that cache's codes."""
    B, nkv, rep, inter, S = 4, 4, 4, 264, 40
    y, cos, sin, ks, vs, q, act = _post_case(dev, dt, B, nkv, rep, inter, S, False, 3)
    _, _, _, k8, v8, q2, act2 = _post_case(dev, dt, B, nkv, rep, inter, S, True, 3)
    slot = i64(dev, 5)
    kw = dict(NH=nkv * rep, NKV=nkv, HD=HD, ROPE=True)
    beam.post(y, slot, None, cos, sin, ks, vs, q, act, **kw)
    beam.post(y, slot, None, cos, sin, k8, v8, q2, act2, **kw)
    for b in range(B):
        kc, vc = (torch.full((nkv, S, HD), 9.0, device=dev, dtype=dt) for _ in range(2))
        q1, a1 = torch.zeros_like(q[0]), torch.zeros_like(act[0])
        fused.post[(1,)](y[b].contiguous(), slot, cos, sin, kc, vc, q1, a1, S, inter, **kw)
        assert torch.equal(kc, ks[b]) and torch.equal(vc, vs[b]) and torch.equal(q1, q[b]) and torch.equal(a1, act[b])
    assert torch.equal(q, q2) and torch.equal(act, act2)
    e8, f8 = kv8.empty(B, nkv, S, HD, device=dev), kv8.empty(B, nkv, S, HD, device=dev)
    kv8.quantize(ks, vs, e8, f8, t0=5, n=1)
    for a, b in zip((*k8, *v8), (*e8, *f8)):
        assert torch.equal(a[:, :, 5], b[:, :, 5])


def test_post_rows_without_a_slot(dev):
    B, nkv, rep, inter, T = 6, 2, 2, 24, 8
    y, cos, sin, ks, vs, q, act = _post_case(dev, F16, B, nkv, rep, inter, T, False, 4, P=20)
    # beyond the cache, before it, beyond the RoPE tables (14 + 7 > 19), and three that fit
    slot = [8, -1, 7, 5, 0, 2 ** 40]
    beam.post(y, i64(dev, *slot), i64(dev, 14), cos, sin, ks, vs, q, act, NH=4, NKV=nkv, HD=HD, ROPE=True)
    ok = [3, 4]
    for b in range(B):
        assert bool((q[b] == 9).all()) == (b not in ok) and bool((ks[b] == 9).all()) == (b not in ok)
        assert bool((vs[b] == 9).all()) == (b not in ok) and not (act[b] == 9).all()
    # without RoPE only the cache bounds the slot
    beam.post(y, i64(dev, *slot), i64(dev, 14), cos, sin, ks, vs, q, act, NH=4, NKV=nkv, HD=HD, ROPE=False)
    assert not (q[2] == 9).all() and not (ks[2, :, 7] == 9).all()
    assert (q[0] == 9).all() and (q[1] == 9).all() and (q[5] == 9).all()
    # a prefix length beyond the tables, also one that a sum would wrap
    for p in (20, -1, 2 ** 63 - 1):
        q.fill_(9)
        beam.post(y, i64(dev, 3), i64(dev, p), cos, sin, ks, vs, q, act, NH=4, NKV=nkv, HD=HD, ROPE=True)
        assert (q == 9).all()


# -------------------------------------------------------------------------------------------------------- attention
def check_attn(o, q, kv, dt, scale, p_unit):
    """o [B, NH * HD] against the oracle; kv(b, g): (k, v) rows in float64"""
    B, NH = q.shape[0], q.shape[1] // HD
    qd, od = q.double().cpu().numpy().reshape(B, NH, HD), o.double().cpu().numpy().reshape(B, NH, HD)
    for b in range(B):
        for h in range(NH):
            k, v = kv(b, h)
            want, mag = OB.attend(qd[b, h], (k, v), scale)
            s = np.abs(k) @ np.abs(qd[b, h]) * abs(scale) if len(k) else np.zeros(1)
            rel = p_unit + 132 * U[torch.float32] * s.max() + 2.0 ** -21 + s.max() * 2.0 ** -22
            tol = 2 * rel * mag + (len(k) / 32 + 64) * U[torch.float32] * mag + U[dt] * np.abs(want) + 1e-7
            with np.errstate(invalid="ignore"):  # infinite values are held to be the same ones, NaN to be NaN
                same = (od[b, h] == want) | (np.isnan(od[b, h]) & np.isnan(want))
                off = np.where(same, 0.0, np.abs(od[b, h] - want))
            assert np.all(same | (off <= tol)), (b, h, len(k), float((off / (tol + 1e-30)).max()))


def attn_case(dev, dt, B, nkv, rep, S, T, plen, spos, p8=False, s8=False, table=None, seed=0, rows=None, sharp=2.0,
              junk=float("nan")):
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, device=dev, dtype=dt, generator=g)  # noqa: E731
    NH, rows = nkv * rep, rows or B
    q = r(B, NH * HD) * sharp
    n = min(max(plen, 0), S) if plen is not None else 0
    kc = vc = ks = vs = None
    kcd = vcd = ksd = vsd = None
    if S:
        (kc, kcd), (vc, vcd) = (as_cache(r(nkv, S, HD), p8) for _ in range(2))
        for c in (kc, vc):  # what lies behind the prefix does not matter
            if p8:
                c[1][:, n:] = junk
            else:
                c[:, n:] = junk
    used = None
    if T:
        (ks, ksd), (vs, vsd) = (as_cache(r(rows, nkv, T, HD), s8) for _ in range(2))
        used = torch.zeros(rows, T, dtype=torch.bool, device=dev)
        for b in range(B):
            for t in range(min(spos[b if len(spos) > 1 else 0] + 1, T)):
                w = b if table is None else int(table[b, t])
                if 0 <= w < rows:
                    used[w, t] = True
        for c in (ks, vs):
            if s8:
                c[1].masked_fill_(~used[:, None], junk)
            else:
                c.masked_fill_(~used[:, None, :, None], junk)
    src = None if table is None else torch.tensor(table, dtype=torch.int32, device=dev)
    o = torch.full((B, NH * HD), 7.0, device=dev, dtype=dt)
    pl = None if not S else i64(dev, plen)
    sp = None if not T else i64(dev, *spos)
    scale = HD ** -0.5
    run = lambda ws=None: beam.attn(q, kc, vc, pl, ks, vs, sp, o, scale, src=src, ws=ws)  # noqa: E731

    def kv(b, h):
        return OB.slots(kcd, vcd, plen, ksd, vsd, spos[b if len(spos) > 1 else 0] if T else -1,
                        None if table is None else table[b], b, h // rep)
    unit = U[dt]
    return dict(q=q, o=o, run=run, kv=kv, unit=unit, scale=scale, plen=pl, spos=sp, kc=kc, vc=vc, ks=ks, vs=vs, src=src)


def run_and_check(c, dt):
    c["run"]()
    check_attn(c["o"], c["q"], c["kv"], dt, c["scale"], c["unit"])


KINDS = [(F16, False, False), (BF16, False, False), (F16, True, True), (BF16, True, True), (F16, True, False),
         (BF16, False, True)]


@pytest.mark.parametrize("dt,p8,s8", KINDS)
@pytest.mark.parametrize("B,nkv,rep,plen,slen", [(1, 1, 1, 1, 1), (4, 4, 4, 34, 9), (3, 2, 8, 0, 5), (5, 2, 1, 63, 0),
                                                 (2, 4, 2, 129, 65), (9, 2, 4, 257, 33), (17, 1, 8, 200, 31),
                                                 (33, 2, 2, 95, 3)])
def test_attn(dt, p8, s8, B, nkv, rep, plen, slen, dev):
    run_and_check(attn_case(dev, dt, B, nkv, rep, plen + 3, slen + 2, plen, [slen - 1], p8, s8, seed=plen), dt)


@pytest.mark.parametrize("dt,p8", [(F16, False), (BF16, False), (F16, True), (BF16, True)])
@pytest.mark.parametrize("B,nkv,rep,plen", [(5, 1, 4, 4096), (17, 2, 1, 4095), (17, 1, 2, 4097), (16, 1, 4, 4160),
                                            (7, 2, 8, 4223), (33, 1, 4, 5001), (9, 3, 8, 8191), (65, 1, 2, 6000)])
def test_attn_long_prefix(dt, p8, B, nkv, rep, plen, dev):
    """Prefixes of some thousand slots, a suffix beside them."""
    run_and_check(attn_case(dev, dt, B, nkv, rep, plen + 5, 40, plen, [b % 40 for b in range(B)], p8, False, seed=plen), dt)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("B,nkv,rep,plen,p8", [
    (17, 8, 1, 12287, False), (17, 8, 1, 12288, False), (8, 8, 4, 12345, False),                   # blocks of 32 rows
    (33, 8, 1, 8193, False), (16, 8, 4, 24570, False), (16, 8, 4, 32769, True),                    # 32; 64
    (65, 8, 1, 5000, False), (20, 8, 4, 24600, False), (32, 8, 4, 17000, True), (20, 8, 4, 26300, True),  # 64; 128
    (32, 8, 8, 1537, False), (40, 8, 8, 9001, False), (129, 16, 1, 2000, False), (100, 4, 8, 4000, False),
    (72, 8, 8, 4001, True)])
def test_attn_wide_prefix(dt, B, nkv, rep, plen, p8, dev):
    """Prefixes long enough, for so many query rows, that blocks take them tile by tile through LDS; around the border,
    in each of its block sizes, with row groups that are not full and splits of unequal length."""
    c = attn_case(dev, dt, B, nkv, rep, plen + 5, 40, plen, [b % 40 for b in range(B)], p8, False, seed=plen)
    c["run"]()
    kd, vd = ((x[0][:, :plen].double() * x[1][:, :plen].double()[..., None] if p8 else x[:, :plen].double()).cpu().numpy()
              for x in (c["kc"], c["vc"]))
    ks, vs = c["ks"].double().cpu().numpy(), c["vs"].double().cpu().numpy()
    NH = nkv * rep
    rows = sorted({0, 1, B // 2, B - 1})
    for h in sorted({0, NH // 2 + rep // 2, NH - 1}):  # one head of some hypotheses, seen as a model of one head
        g = h // rep
        pick = lambda x: x.view(B, NH, HD)[rows, h].contiguous()  # noqa: E731
        check_attn(pick(c["o"]), pick(c["q"]),
                   lambda b, _: OB.slots(kd, vd, plen, ks, vs, rows[b] % 40, None, rows[b], g), dt, c["scale"], c["unit"])
    assert bool(torch.isfinite(c["o"]).all())


def test_attn_short_prefix_in_a_long_cache(dev):
    for p8 in (False, True):
        c = attn_case(dev, F16, 20, 2, 2, 9000, 10, 8999, [9], p8, False, seed=4, junk=0.0)
        for n in (8999, 4095, 4096, 1, 0, 5000, 20000):
            c["plen"].fill_(n)
            c["run"]()
            kd, vd = ((x[0].double() * x[1].double()[..., None] if p8 else x.double()).cpu().numpy()
                      for x in (c["kc"], c["vc"]))
            ks, vs = c["ks"].double().cpu().numpy(), c["vs"].double().cpu().numpy()
            check_attn(c["o"][:3], c["q"][:3], lambda b, h: OB.slots(kd, vd, n, ks, vs, 9, None, b, h // 2), F16,
                       c["scale"], c["unit"])


def test_attn_short_prefix_in_a_very_long_cache(dev):
    """The cache admits the LDS tiles, the prefix may not."""
    for p8, B, rep, S in ((False, 20, 1, 14000), (True, 20, 4, 27000)):
        c = attn_case(dev, F16, B, 8, rep, S, 10, S, [9], p8, False, seed=4, junk=0.0)
        for n in (S, 12287, 12288, 1, 0, 63, 26214, 26215, 5000, 200000):
            c["plen"].fill_(n)
            c["run"]()
            kd, vd = ((x[0].double() * x[1].double()[..., None] if p8 else x.double()).cpu().numpy()
                      for x in (c["kc"], c["vc"]))
            ks, vs = c["ks"].double().cpu().numpy(), c["vs"].double().cpu().numpy()
            for h in (0, 5 * rep):
                pick = lambda x: x.view(B, 8 * rep, HD)[:2, h].contiguous()  # noqa: E731
                check_attn(pick(c["o"]), pick(c["q"]),
                           lambda b, _: OB.slots(kd, vd, n, ks, vs, 9, None, b, h // rep), F16, c["scale"], c["unit"])


@pytest.mark.parametrize("dt,p8,s8", KINDS)
def test_attn_around_one_launch(dt, p8, s8, dev):
    """Caches of up to 256 slots are taken in one launch, its eight waves shared out by the lengths, 32 slots a step."""
    for S, T in ((128, 127), (128, 128), (129, 128), (255, 1), (256, 1), (1, 255), (1, 256), (33, 223), (224, 32)):
        run_and_check(attn_case(dev, dt, 3, 2, 4, S, T, S, [T - 1], p8, s8, seed=S), dt)
        run_and_check(attn_case(dev, dt, 2, 1, 8, S, T, S // 2, [T - 1, T // 3], p8, s8, seed=T), dt)
    for S, T in ((500, 268), (500, 269), (96, 672), (0, 768)):  # and of up to 768 for 128 to 256 rows of KV heads
        run_and_check(attn_case(dev, dt, 64, 2, 1, S, T, S - 1, [T - 1 - b for b in range(64)], p8, s8, seed=S), dt)
        run_and_check(attn_case(dev, dt, 17, 15, 1, S, T, S - 1, [T - 1], p8, s8, seed=T), dt)
    run_and_check(attn_case(dev, dt, 64, 8, 1, 200, 56, 199, [55], p8, s8, seed=1), dt)
    run_and_check(attn_case(dev, dt, 57, 9, 1, 200, 56, 199, [55], p8, s8, seed=1), dt)
    for n in (1, 31, 32, 33, 255, 256, 257):
        run_and_check(attn_case(dev, dt, 2, 1, 2, n, 0, n, [0], p8, False, seed=n), dt)
        run_and_check(attn_case(dev, dt, 2, 1, 2, 0, n, None, [n - 1], False, s8, seed=n), dt)


@pytest.mark.parametrize("dt,p8,s8", [(F16, False, False), (BF16, True, True)])
@pytest.mark.parametrize("B,nkv", [(127, 1), (64, 2), (128, 2), (257, 1)])
def test_attn_around_one_launch_of_three_steps(dt, p8, s8, B, nkv, dev):
    """127, 128, 256 and 257 pairs of hypothesis and KV head: one launch for up to 768 slots from 128 pairs to 256."""
    for S, T in ((300, 468), (300, 469)):
        c = attn_case(dev, dt, B, nkv, 1, S, T, S - 1, [T - 1 - b % 7 for b in range(B)], p8, s8, seed=S + T)
        c["run"]()
        rows = [0, 1, B // 2, B - 1]
        kv = c["kv"]
        check_attn(c["o"][rows], c["q"][rows], lambda b, h: kv(rows[b], h), dt, c["scale"], c["unit"])
        assert bool(torch.isfinite(c["o"]).all())


@pytest.mark.parametrize("dt,p8,s8", KINDS)
@pytest.mark.parametrize("B,rows,T,seed", [(4, 4, 40, 0), (6, 9, 131, 1), (8, 3, 17, 2)])
def test_attn_table(dt, p8, s8, B, rows, T, seed, dev):
    rng = np.random.default_rng(seed)
    table = rng.integers(0, rows, (B, T))
    table[rng.random((B, T)) < 0.1] = -1              # no slot
    table[rng.random((B, T)) < 0.1] = rows + seed * 2 ** 20
    spos = [int(x) for x in rng.integers(-1, T, B)]
    spos[0] = T - 1
    run_and_check(attn_case(dev, dt, B, 2, 4, 50, T, 37, spos, p8, s8, table=table, seed=seed, rows=rows), dt)


@pytest.mark.parametrize("dt,p8,s8", KINDS)
def test_attn_empty_and_clamped(dt, p8, s8, dev):
    # no slot at all for hypothesis 1; lengths beyond the caches; no prefix; no suffix
    c = attn_case(dev, dt, 3, 2, 4, 20, 10, 0, [4, -1, 9], p8, s8)
    run_and_check(c, dt)
    assert not c["o"][1].any()
    run_and_check(attn_case(dev, dt, 3, 2, 4, 20, 10, 1000, [4, -5, 77], p8, s8), dt)
    run_and_check(attn_case(dev, dt, 3, 2, 4, 20, 10, -3, [2 ** 40], p8, s8), dt)
    run_and_check(attn_case(dev, dt, 3, 2, 4, 0, 40, None, [4, 39, 9], False, s8), dt)
    c = attn_case(dev, dt, 3, 2, 4, 70, 0, 66, [0], p8, False)
    run_and_check(c, dt)
    c["plen"].zero_()
    c["run"]()
    assert not c["o"].any()


@pytest.mark.parametrize("dt", [F16, BF16])
def test_attn_every_split_boundary(dt, dev):
    """Prefix and suffix lengths around the pieces that waves and blocks take."""
    for n in (31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 512, 513):
        run_and_check(attn_case(dev, dt, 2, 1, 2, 600, 3, n, [1], seed=n), dt)
        run_and_check(attn_case(dev, dt, 2, 1, 2, 8, 600, 3, [n - 1], seed=n), dt)


@pytest.mark.parametrize("dt,p8", [(F16, False), (BF16, False), (F16, True), (BF16, True)])
def test_attn_scores_that_move(dt, p8, dev):
    """A running maximum that keeps rising, that falls, and one slot that outweighs all."""
    for shape in ("rise", "fall", "spike"):
        c = attn_case(dev, dt, 4, 2, 4, 700, 50, 650, [40], p8, False, seed=5, sharp=1.0)
        g = torch.Generator(device=dev).manual_seed(9)
        base = torch.randn(2, 1, HD, device=dev, generator=g)
        ramp = torch.linspace(0, 12, 700, device=dev)[None, :, None]
        ramp = {"rise": ramp, "fall": 12 - ramp, "spike": (ramp * 0 + (torch.arange(700, device=dev) == 333)[None, :, None] * 30)}[shape]
        k = (base * ramp + torch.randn(2, 700, HD, device=dev, generator=g) * 0.5).to(dt)
        c["q"].copy_((base.repeat_interleave(4, 0).reshape(1, -1) + torch.randn(4, 8 * HD, device=dev, generator=g)).to(dt))
        kc, kd = as_cache(k, p8)
        vd = (c["vc"][0].double() * c["vc"][1].double()[..., None] if p8 else c["vc"].double()).cpu().numpy()
        beam.attn(c["q"], kc, c["vc"], c["plen"], None, None, None, c["o"], c["scale"])
        check_attn(c["o"], c["q"], lambda b, h: (kd[h // 4, :650], vd[h // 4, :650]), dt, c["scale"], c["unit"])


@pytest.mark.parametrize("dt,p8", [(F16, False), (BF16, False), (F16, True), (BF16, True)])
def test_attn_low_scores(dt, p8, dev):
    """Scores far below zero throughout, over one to ten splits of prefix and suffix."""
    for plen, spos in ((100, -1), (0, 9), (300, 20), (300, 200), (500, 200), (900, 299)):
        c = attn_case(dev, dt, 3, 2, 2, 1000, 300, plen, [spos], p8, False, seed=plen, sharp=1.0, junk=0.0)
        c["q"][:, ::HD] = 60.0
        for x in (c["kc"], c["ks"]):
            x = x if isinstance(x, torch.Tensor) else x[0]
            x[..., 0] = -127 if x.dtype == torch.int8 else -100.0
        if p8:
            c["kc"][1].fill_(0.8)
        kd, vd = ((x[0].double() * x[1].double()[..., None] if p8 else x.double()).cpu().numpy()
                  for x in (c["kc"], c["vc"]))
        ks, vs = c["ks"].double().cpu().numpy(), c["vs"].double().cpu().numpy()
        c["run"]()
        check_attn(c["o"], c["q"], lambda b, h: OB.slots(kd, vd, plen, ks, vs, spos, None, b, h // 2), dt, c["scale"],
                   c["unit"])


@pytest.mark.parametrize("dt", [F16, BF16])
def test_attn_infinities(dt, dev):
    """Scores of -inf have no weight, a row of them gives zeros; NaN in a slot that counts gives NaN."""
    c = attn_case(dev, dt, 20, 1, 1, 4200, 4, 4190, [1])
    c["q"][:] = 1.0
    c["kc"][0, :, 0] = -float("inf")
    c["ks"][:, 0, :, 0] = -float("inf")
    c["run"]()
    assert not c["o"].any()
    c["kc"][0, 4189, 0] = 0  # one slot counts
    c["run"]()
    assert torch.equal(c["o"], c["vc"][0, 4189].expand(20, -1))
    c["vc"][0, 4189, 5] = float("inf")  # and nothing that lies behind it
    c["run"]()
    want = c["vc"][0, 4189].expand(20, -1)
    assert torch.equal(c["o"], want) and torch.isinf(want[:, 5]).all()
    c = attn_case(dev, dt, 2, 1, 1, 40, 4, 40, [1])
    inf = float("inf")
    c["q"][:] = 1.0
    c["kc"][0, 5:20, 0] = -inf
    c["run"]()
    k, v = c["kc"][0].double().cpu().numpy(), c["vc"][0].double().cpu().numpy()
    keep = np.r_[0:5, 20:40]

    def kv(b, h):
        ks, vs = c["ks"][b, 0, :2].double().cpu().numpy(), c["vs"][b, 0, :2].double().cpu().numpy()
        return np.concatenate((k[keep], ks)), np.concatenate((v[keep], vs))
    check_attn(c["o"], c["q"], kv, dt, c["scale"], c["unit"])
    c["kc"][0, :, 0] = -inf
    c["ks"][:, 0, :, 0] = -inf
    c["run"]()
    assert not c["o"].any()
    c["kc"][0, 7, 3] = float("nan")
    c["run"]()
    assert torch.isnan(c["o"]).all()
    c["kc"][0, 7, 3] = 0
    c["kc"][0, :, 0] = 0
    c["vc"][0, 7, 3] = float("nan")
    c["run"]()
    assert torch.isnan(c["o"][:, 3]).all() and torch.isfinite(c["o"][:, 4:]).all()


@pytest.mark.parametrize("dt", [F16, BF16])
def test_attn_wide_infinities(dt, dev):
    """The same where the prefix is taken tile by tile."""
    inf = float("inf")
    c = attn_case(dev, dt, 200, 8, 1, 2000, 4, 1990, [1])
    c["q"][:] = 1.0
    c["kc"][:, :, 0] = -inf
    c["ks"][..., 0] = -inf
    c["run"]()
    assert not c["o"].any()
    for at in (0, 63, 64, 1000, 1989):  # one slot counts
        c["kc"][:, at, 0] = 0
        c["run"]()
        assert torch.equal(c["o"].view(200, 8, HD), c["vc"][:, at].expand(200, -1, -1))
        c["kc"][:, at, 0] = -inf
    c["kc"][:, 700, 0] = 0
    c["vc"][:, 700, 5] = inf
    c["run"]()
    assert torch.equal(c["o"].view(200, 8, HD), c["vc"][:, 700].expand(200, -1, -1))
    c["kc"][:, :1990, 0] = 0
    c["vc"][:, 700, 5] = float("nan")
    c["run"]()
    o = c["o"].view(200, 8, HD)
    assert torch.isnan(o[..., 5]).all() and torch.isfinite(o[..., 6:]).all()
    c["kc"][3, 1989, 1] = float("nan")
    c["run"]()
    assert torch.isnan(o[:, 3]).all() and torch.isfinite(o[:, 4, 6:]).all()


@pytest.mark.parametrize("dt,p8", [(F16, False), (BF16, False), (F16, True), (BF16, True)])
def test_attn_wide_scores_that_move(dt, p8, dev):
    """Running maxima that move, and V rows of very different sizes, where the prefix is taken tile by tile."""
    B, nkv, S = 200, 8, 10500 if p8 else 2500
    for shape in ("rise", "fall", "spike"):
        c = attn_case(dev, dt, B, nkv, 1, S, 0, S - 3, [0], p8, False, seed=5, sharp=1.0)
        g = torch.Generator(device=dev).manual_seed(9)
        base = torch.randn(nkv, 1, HD, device=dev, generator=g)
        ramp = torch.linspace(0, 12, S, device=dev)[None, :, None]
        if shape == "fall":
            ramp = 12 - ramp
        elif shape == "spike":
            ramp = (torch.arange(S, device=dev) == S - 700)[None, :, None] * 30.0
        k = (base * ramp + torch.randn(nkv, S, HD, device=dev, generator=g) * 0.5).to(dt)
        c["q"].copy_((base.reshape(1, -1) + torch.randn(B, nkv * HD, device=dev, generator=g)).to(dt))
        size = torch.exp(torch.randn(nkv, S, 1, device=dev, generator=g) * 2)
        kc, kd = as_cache(k, p8)
        vc, vd = as_cache((torch.randn(nkv, S, HD, device=dev, generator=g) * size).to(dt), p8)
        beam.attn(c["q"], kc, vc, c["plen"], None, None, None, c["o"], c["scale"])
        for h in (0, 5):
            rows = [0, 17, 99, 199]
            pick = lambda x: x.view(B, nkv, HD)[rows, h].contiguous()  # noqa: E731
            check_attn(pick(c["o"]), pick(c["q"]), lambda b, _: (kd[h, :S - 3], vd[h, :S - 3]), dt, c["scale"], c["unit"])


def test_attn_wide_captured(dev):
    """A captured call whose prefix comes and goes past the length from which it is taken tile by tile; its result is the
    eager one's, every time, whatever the workspace held."""
    import _hiplib as HL
    c = attn_case(dev, F16, 200, 8, 1, 2000, 40, 2000, [10], seed=2, junk=0.0)
    n = HL.lib().rk_beam_attn_ws_bytes(200, 8, 8, 2000, 40)
    ws = torch.zeros(n, dtype=torch.uint8, device=dev)
    c["run"](ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c["run"](ws)
    for plen in (2000, 100, 1900, 1800, 0, 1999):
        c["plen"].fill_(plen)
        c["spos"].fill_(plen % 40)
        ws.fill_(255)
        graph.replay()
        got = c["o"].clone()
        c["o"].fill_(5)
        c["run"]()
        assert torch.equal(got, c["o"]) and bool(torch.isfinite(got).all())


def test_attn_quantised_row_of_nan(dev):
    c = attn_case(dev, F16, 2, 1, 2, 40, 4, 40, [1], p8=True)
    c["kc"][1][0, 39] = float("nan")
    c["run"]()
    assert torch.isnan(c["o"]).all()


@pytest.mark.parametrize("dt,p8,s8", KINDS)
def test_attn_small_and_large_values(dt, p8, s8, dev):
    """V rows of very different sizes (int8: of very different scales), queries near the types' ends."""
    for big in (1e-3, 3.0, 200.0):
        c = attn_case(dev, dt, 3, 2, 4, 90, 30, 80, [20], p8, s8, seed=6)
        g = torch.Generator(device=dev).manual_seed(7)
        size = torch.exp(torch.randn(2, 90, 1, device=dev, generator=g) * 2) * big
        v, vd = as_cache((torch.randn(2, 90, HD, device=dev, generator=g) * size).to(dt), p8)
        kd = (c["kc"][0].double() * c["kc"][1].double()[..., None] if p8 else c["kc"].double()).cpu().numpy()
        beam.attn(c["q"], c["kc"], v, c["plen"], None, None, None, c["o"], c["scale"])
        check_attn(c["o"], c["q"], lambda b, h: (kd[h // 4, :80], vd[h // 4, :80]), dt, c["scale"], c["unit"])


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("B,nkv,plen", [(3, 2, 90), (3, 2, 700), (9, 1, 4500)])
def test_attn_v_scales_far_apart(dt, B, nkv, plen, dev):
    """One int8 slot whose V is 2^20 times the others' but whose weight is next to none, at several places."""
    for at in (0, 40, plen - 1):
        c = attn_case(dev, dt, B, nkv, 4, plen, 0, plen, [0], True, False, seed=at, sharp=1.0)
        codes, scales = c["kc"]
        q = c["q"].view(B, nkv, 4, HD)
        q[..., 0] = 30.0
        codes[:, at].zero_()
        codes[:, at, 0] = -127
        scales[:, at] = 1.0
        c["vc"][1][:, at] *= 2.0 ** 20
        kd, vd = ((x[0].double() * x[1].double()[..., None]).cpu().numpy() for x in (c["kc"], c["vc"]))
        c["run"]()
        check_attn(c["o"], c["q"], lambda b, h: (kd[h // 4], vd[h // 4]), dt, c["scale"], c["unit"])


def test_attn_large_sizes_of_the_type(dev):
    """bf16 keys and queries beyond fp16's range, their scores brought back by the scale."""
    c = attn_case(dev, BF16, 2, 1, 2, 70, 5, 66, [3], seed=8)
    big = 2.0 ** 60
    c["q"].mul_(big)
    for k in (c["kc"], c["ks"]):
        k.mul_(big)
    kc, kd = as_cache(c["kc"][:, :66].contiguous(), False)
    vd = c["vc"].double().cpu().numpy()
    beam.attn(c["q"], c["kc"], c["vc"], c["plen"], None, None, None, c["o"], c["scale"] / big ** 2)
    check_attn(c["o"], c["q"], lambda b, h: (kd[0], vd[0, :66]), BF16, c["scale"] / big ** 2, c["unit"])


# paths of an attention call: one launch; split, with a join; the prefix tile by tile (plain; plain and int8)
PATHS = [(3, 2, 4, 100, 40), (3, 2, 4, 700, 300), (200, 8, 1, 2500, 40), (200, 8, 1, 10500, 40)]


def attend64(q, kv, suffix, scale):
    """softmax(scale q . k) v and sum w |v| beside it in float64, [B, NH, HD]: q [B, NH * HD] over the prefix rows kv = (k, v)
    [nkv, n, HD] and each hypothesis's own suffix = (k, v) [B, nkv, m, HD], all of them slots"""
    kd, vd = (x.double() for x in kv)
    ks, vs = (x.double() for x in suffix)
    nkv = kd.shape[0]
    qd = q.double().view(q.shape[0], nkv, -1, HD)
    sp = (qd[:, :, :, None] * kd[None, :, None]).sum(-1) if kd.shape[1] < 1000 else \
        torch.stack([qd[:, g] @ kd[g].t() for g in range(nkv)], 1)
    s = torch.cat((sp, (qd[:, :, :, None] * ks[:, :, None]).sum(-1)), -1) * scale
    w = torch.exp(s - s.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    n = kd.shape[1]
    both = []
    for x, y in ((vd, vs), (vd.abs(), vs.abs())):
        o = torch.stack([w[:, g, :, :n] @ x[g] for g in range(nkv)], 1) + (w[..., n:, None] * y[:, :, None]).sum(-2)
        both.append(o.flatten(1, 2))
    return both


def dense(c, *index):
    """a cache's values in float64, at the given index"""
    return (c[0].double() * c[1].double()[..., None] if isinstance(c, tuple) else c.double())[index]


@pytest.mark.parametrize("dt,p8,s8", KINDS)
@pytest.mark.parametrize("B,nkv,rep,S,T", PATHS)
def test_attn_large_scores(dt, p8, s8, B, nkv, rep, S, T, dev):
    """Scores of 2^29 and more (bf16: 2^83), of which an fp32 holds no fraction: a few slots of the one highest score share
    the row, wherever they lie. Every product here is exact, so the weights are, but for their rounding to 16 bits."""
    unit = 2.0 ** (13 if dt is F16 else 40)
    plen, slen = S - 1, T - 1
    c = attn_case(dev, dt, B, nkv, rep, S, T, plen, [slen - 1], p8, s8, seed=S, junk=0.0)
    size = unit * (1 + torch.arange(B * nkv * rep, device=dev) % 16 / 16)
    c["q"].copy_(size[:, None].expand(-1, HD).reshape(B, -1))
    tops, stops = sorted({0, 33, S // 2, S - 2}), [T // 2, T - 2]
    for cache, at, n in ((c["kc"], tops, plen), (c["ks"], stops, slen)):
        rows, of = (cache[0], 32) if isinstance(cache, tuple) else (cache, unit / 2)
        rows.fill_(of)
        rows[..., at, :] = 2 * of
        rows[..., n:, :] = 3 * of if of == 32 else 1.5 * unit  # behind the length
        if of == 32:
            cache[1].fill_(unit / 64)
    v = torch.cat((dense(c["vc"])[:, tops].expand(B, -1, -1, -1), dense(c["vs"])[:, :, stops]), 2)
    want, mag = (x.mean(2).repeat_interleave(rep, 1).reshape(B, -1) for x in (v, v.abs()))
    for sign in (1, -1):
        q = c["q"] * sign
        beam.attn(q, c["kc"], c["vc"], c["plen"], c["ks"], c["vs"], c["spos"], c["o"], sign * c["scale"])
        off = (c["o"].double() - want).abs()
        assert bool((off <= (2 * U[dt] + 2.0 ** -20) * mag + U[dt] * want.abs() + 1e-7).all()), float((off / mag).max())


@pytest.mark.parametrize("dt,p8,s8", KINDS)
@pytest.mark.parametrize("B,nkv,rep,S,T", [(64, 2, 1, 600, 100), (64, 4, 1, 300, 700), (3, 2, 4, 40000, 4),
                                           (200, 8, 1, 2500, 4), (200, 8, 1, 10500, 4)])
def test_attn_large_scores_that_rise(dt, p8, s8, B, nkv, rep, S, T, dev):
    """Scores around 2^27, where fp32 has every 16th number, that rise from 2^27 + 16 to the next one while a wave goes on;
    exactly so, in log2 units, by this scale."""
    scale = float(np.float32(math.log(2)))
    assert np.float32(scale) * np.float32(1.4426950408889634) == 1
    c = attn_case(dev, dt, B, nkv, rep, S, T, S - 1, [T - 2], p8, s8, seed=S, junk=0.0)
    c["q"].zero_()
    c["q"].view(B, -1, HD)[..., 0], c["q"].view(B, -1, HD)[..., 1] = 2.0 ** 12, 2.0 ** -5
    for k in (c["kc"], c["ks"]):
        rows, unit = (k[0], 1) if isinstance(k, tuple) else (k, 512)
        n = rows.shape[-2]
        rows.zero_()
        rows[..., 0] = 64 * unit
        rows[..., 1] = 1 * unit
        rows[..., n * 6 // 10:, 1] = 2 * unit
        if unit == 1:
            k[1].fill_(512.0)
    beam.attn(c["q"], c["kc"], c["vc"], c["plen"], c["ks"], c["vs"], c["spos"], c["o"], scale)
    want, mag = attend64(c["q"], [dense(c[k])[:, :S - 1] for k in ("kc", "vc")],
                         [dense(c[k])[:, :, :T - 1] for k in ("ks", "vs")], scale)
    off = (c["o"].double().view_as(want) - want).abs()
    assert bool((off <= (2 * U[dt] + 2.0 ** -17) * mag + U[dt] * want.abs() + 1e-7).all()), float((off / mag).max())


@pytest.mark.parametrize("S,T", [(60, 30), (400, 140)])
def test_attn_no_slot_beside_low_scores(S, T, dev):
    """A suffix whose table leads to no slot does not count as a score, however small the scale: scores of about -256 beside
    it, keys near the end of bf16's range."""
    c = attn_case(dev, BF16, 2, 1, 2, S, T, S - 3, [T - 1], False, True, table=np.full((2, T), -1), seed=S, sharp=1.0,
                  junk=0.0)
    q = c["q"].view(2, 2, HD)
    q[..., :16] = 16.0
    c["kc"].mul_(2.0 ** 116)
    c["kc"][..., :16] = -2.0 ** 118
    c["scale"] = 2.0 ** -118
    beam.attn(c["q"], c["kc"], c["vc"], c["plen"], c["ks"], c["vs"], c["spos"], c["o"], c["scale"], src=c["src"])
    kd, vd = (c[k][0, :S - 3].double().cpu().numpy() for k in ("kc", "vc"))
    check_attn(c["o"], c["q"], lambda b, h: (kd, vd), BF16, c["scale"], c["unit"])


@pytest.mark.parametrize("dt,p8,s8", KINDS)
@pytest.mark.parametrize("B,nkv,rep,S,T", PATHS)
@pytest.mark.parametrize("depth", [12.0, 16.203125, 17.40625, 20.0])
def test_attn_many_low_weights(dt, p8, s8, B, nkv, rep, S, T, depth, dev):
    """One slot leads by `depth`, all others have the same score: in the dims where the leading one's V is 0 the others are
    the result. A weight is held to within 2^-32 of the largest one (half a step of fp16 below 2^7), int8: 2^-31 with V's
    scale in it, besides its rounding."""
    plen, slen = S - 1, T - 1
    c = attn_case(dev, dt, B, nkv, rep, S, T, plen, [slen - 1], p8, s8, seed=S, junk=0.0)
    g = torch.Generator(device=dev).manual_seed(S)
    c["q"].zero_()
    c["q"].view(B, -1, HD)[..., 0] = 1.0
    v = (torch.rand(nkv, S, HD, device=dev, generator=g) + 1) * 1024
    v[:, 0, 64:] = 0
    vs = (torch.rand(B, nkv, T, HD, device=dev, generator=g) + 1) * 1024
    c["vc"], c["vs"] = as_cache(v.to(dt), p8)[0], as_cache(vs.to(dt), s8)[0]
    for k in (c["kc"], c["ks"]):
        (k[0] if isinstance(k, tuple) else k).zero_()
    top = torch.tensor(depth, dtype=dt).item()
    if p8:
        c["kc"][0][:, 0, 0] = 64
        c["kc"][1][:, 0] = top / 64
    else:
        c["kc"][:, 0, 0] = top
    beam.attn(c["q"], c["kc"], c["vc"], c["plen"], c["ks"], c["vs"], c["spos"], c["o"], 1.0)
    want, mag = attend64(c["q"], [dense(c[k])[:, :plen] for k in ("kc", "vc")],
                         [dense(c[k])[:, :, :slen] for k in ("ks", "vs")], 1.0)
    n, vmax = plen + slen, 2048 * (1 + 2.0 ** -8)
    grid = 2.0 ** (-31 if p8 or s8 else -32) * (127.5 if p8 or s8 else 1)  # int8: of the largest V scale, for codes to 127
    tol = 2 * (U[dt] + 2.0 ** -18) * mag + n * grid * (vmax / 127 if p8 or s8 else vmax) + U[dt] * want.abs() + 2.0 ** -25
    off = (c["o"].double().view_as(want) - want).abs()
    assert bool((off <= tol).all()), (float((off / tol).max()), float((off / mag).max()))


@pytest.mark.parametrize("B,nkv,rep,S,T", PATHS)
def test_attn_int8_weights_of_fp16(B, nkv, rep, S, T, dev):
    """Slots in pairs of nearly the same score and opposite V: a result far below its terms, which shows the weights' own
    roundings; with int8 caches and fp16 activations 2^-21 relative at most, and within 2^-32 of twice the largest V scale for
    codes to 127. The scores have one product: off by |s| 2^-22 (three roundings; a tenth of the weights at most has |s| > 9,
    and next to no weight), exp by 2^-21."""
    plen, slen = S - 2, T - 2
    c = attn_case(dev, F16, B, nkv, rep, S, T, plen, [slen - 1], True, True, seed=S, junk=0.0)
    g = torch.Generator(device=dev).manual_seed(S + 1)
    c["q"].zero_()
    c["q"].view(B, -1, HD)[..., 0] = 1.0
    for key, value, n in (("kc", "vc", S // 2), ("ks", "vs", T // 2)):
        lead = c[key][0].shape[:-2]
        score = -(8 if n < 2000 else 100) * torch.rand(*lead, n, device=dev, generator=g) - 0.5
        score = torch.stack((score, score * (1 - 2.0 ** -7 * torch.rand(*lead, n, device=dev, generator=g))), -1).flatten(-2)
        k = torch.zeros(*lead, 2 * n, HD, dtype=torch.int8, device=dev)
        k[..., 0] = -64
        v = torch.randn(*lead, n, HD, device=dev, generator=g).to(F16)
        c[key] = (k, (score / -64).contiguous())
        c[value] = as_cache(torch.stack((v, -v), -2).flatten(-3, -2).contiguous(), True)[0]
    beam.attn(c["q"], c["kc"], c["vc"], c["plen"], c["ks"], c["vs"], c["spos"], c["o"], 1.0)
    want, mag = attend64(c["q"], [dense(c[k])[:, :plen] for k in ("kc", "vc")],
                         [dense(c[k])[:, :, :slen] for k in ("ks", "vs")], 1.0)
    n, most = plen + slen, max(x[1].max().item() for x in (c["vc"], c["vs"]))
    tol = (2 * (2.0 ** -21 + 2.0 ** -21 + 9.1 * 2.0 ** -22) + (n / 32 + 64) * U[torch.float32]) * mag + \
        n * 2.0 ** -32 * 2 * most * 127 + U[F16] * want.abs() + 2.0 ** -25
    off = (c["o"].double().view_as(want) - want).abs()
    assert bool((off <= tol).all()), (float((off / tol).max()), float((off / mag).max()))


@pytest.mark.parametrize("B,nkv,rep,S,T", PATHS)
def test_attn_int8_one_slot_that_counts(B, nkv, rep, S, T, dev):
    """One slot outweighs all others by e^60: with fp16 activations the result is its V row, rounded once."""
    c = attn_case(dev, F16, B, nkv, rep, S, T, S, [T - 1], True, True, seed=S, junk=0.0)
    c["q"].zero_()
    c["q"].view(B, -1, HD)[..., 0] = 1.0
    for k in (c["kc"], c["ks"]):
        k[0].zero_()
    at = S * 2 // 3
    c["kc"][0][:, at, 0] = 60
    c["kc"][1][:, at] = 1.0
    beam.attn(c["q"], c["kc"], c["vc"], c["plen"], c["ks"], c["vs"], c["spos"], c["o"], 1.0)
    want = dense(c["vc"])[:, at].repeat_interleave(rep, 0).expand(B, -1, -1).reshape(B, -1)
    off = (c["o"].double() - want).abs()
    assert bool((off <= (U[F16] + 2.0 ** -20) * want.abs() + 2.0 ** -25).all()), float((off / want.abs()).max())


@pytest.mark.parametrize("p8", [False, True])
def test_attn_matches_the_one_row_attention(p8, dev):
    """A hypothesis by itself is fused.attn over one cache holding its prefix and suffix."""
    B, nkv, rep, plen, T = 4, 4, 4, 150, 30
    c = attn_case(dev, F16, B, nkv, rep, 200, T, plen, [T - 1], seed=11, junk=0.0)
    c["run"]()
    for b in range(B):
        kc = torch.cat((c["kc"][:, :plen], c["ks"][b]), 1).contiguous()
        vc = torch.cat((c["vc"][:, :plen], c["vs"][b]), 1).contiguous()
        o = torch.zeros(nkv * rep * HD, device=dev, dtype=F16)
        fused.attn(c["q"][b].contiguous(), kc, vc, i64(dev, plen + T - 1), o, plen + T, c["scale"], REP=rep, HD=HD)
        # two results within their tolerance of the truth; V is of size 1, weights sum to 1
        assert (o.float() - c["o"][b].float()).abs().max() <= 2 * (4 * U[F16] + 1e-4) * 4


def test_attn_offsets_beyond_32_bits(dev):
    """An int8 prefix of more than 2^31 bytes and elements, read at its end."""
    nkv, S = 1, (1 << 24) + 70000
    codes = torch.zeros(nkv, S, HD, dtype=torch.int8, device=dev)
    scales = torch.full((nkv, S), 0.05, device=dev)
    tail = torch.randint(-127, 128, (nkv, 500, HD), device=dev, generator=torch.Generator(device=dev).manual_seed(1))
    codes[:, S - 500:] = tail.to(torch.int8)
    q = torch.ones(2, HD, device=dev, dtype=F16) * 0.5
    q[1] *= -1
    o = torch.zeros(2, HD, device=dev, dtype=F16)
    # the scores of the zero rows are 0; those of the tail are made to outweigh them all
    codes[:, S - 500:, :64] = 127
    q[:, :64] = 6.0
    beam.attn(q, (codes, scales), (codes, scales), i64(dev, S), None, None, None, o, HD ** -0.5)
    kd = (codes[0, S - 500:].double() * 0.05).cpu().numpy()
    zeros = S - 500
    for b in range(2):
        s = (kd @ q[b].double().cpu().numpy()) * HD ** -0.5
        w = np.exp(s - s.max())
        want = (w @ kd) / (w.sum() + zeros * math.exp(-s.max()))
        mag = (w @ np.abs(kd)) / (w.sum() + zeros * math.exp(-s.max()))
        srel = 132 * U[torch.float32] * np.abs(kd).max() * HD * 6 * HD ** -0.5
        tol = 2 * (U[BF16] + srel) * mag + U[F16] * np.abs(want) + 1e-6
        assert np.all(np.abs(o[b].double().cpu().numpy() - want) <= tol)


@pytest.mark.parametrize("p8,B", [(False, 20), (True, 64)])
def test_attn_wide_offsets_beyond_32_bits(p8, B, dev):
    """The same for more query rows, where the prefix is taken tile by tile: a plain one of more than 2^32 bytes, an int8
    one of more than 2^31."""
    S = (1 << 24) + 70000
    g = torch.Generator(device=dev).manual_seed(1)
    kv = torch.zeros(1, S, HD, dtype=torch.int8 if p8 else F16, device=dev)
    tail = torch.randint(-127, 128, (1, 500, HD), device=dev, generator=g)
    tail[..., :64] = 127
    kv[:, S - 500:] = (tail if p8 else tail * 0.05).to(kv.dtype)
    kd = kv[0, S - 500:].double().cpu().numpy() * (0.05 if p8 else 1)
    cache = (kv, torch.full((1, S), 0.05, device=dev)) if p8 else kv
    q = torch.randn(B, HD, device=dev, generator=g).to(F16)
    q[:, :64] = 6.0
    o = torch.zeros(B, HD, device=dev, dtype=F16)
    beam.attn(q, cache, cache, i64(dev, S), None, None, None, o, HD ** -0.5)
    for b in range(0, B, 7):
        s = (kd @ q[b].double().cpu().numpy()) * HD ** -0.5
        w = np.exp(s - s.max())
        total = w.sum() + (S - 500) * math.exp(-s.max())
        want, mag = (w @ kd) / total, (w @ np.abs(kd)) / total
        srel = 132 * U[torch.float32] * np.abs(kd).max() * HD * 6 * HD ** -0.5
        tol = 2 * (U[F16] + srel) * mag + U[F16] * np.abs(want) + 1e-6
        assert np.all(np.abs(o[b].double().cpu().numpy() - want) <= tol)


def test_attn_captured(dev):
    """Two graphs with a workspace each, replayed in turn and beside each other as lengths and inputs change."""
    cs = [attn_case(dev, F16, 4, 2, 4, 300, 64, 200 + 50 * i, [10 + i], p8=bool(i), seed=i, junk=0.0) for i in range(2)]
    graphs, side = [], torch.cuda.Stream(device=dev)
    for c in cs:
        c["run"]()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c["run"]()
        graphs.append(g)
    for i in range(4):
        for c in cs:
            c["q"].copy_(torch.randn(4, 1024, generator=torch.Generator().manual_seed(i)).to(F16))
            c["plen"].fill_((7, 64, 199, 250)[i])
            c["spos"].fill_((-1, 0, 33, 63)[i])
            c["o"].fill_(5)
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        for c in cs:
            got = c["o"].clone()
            c["run"]()
            torch.cuda.synchronize()
            assert torch.equal(got, c["o"]) and not (got == 5).all()


def test_calls_beside_each_other(dev):
    """Calls on two streams, each with a workspace from the allocator, and calls one after the other give the same bits."""
    cs = [attn_case(dev, F16, 8, 4, 4, 900, 300, 800 - 60 * i, [100 + i], p8=bool(i), s8=bool(i), seed=i, junk=0.0)
          for i in range(2)]
    cs.append(attn_case(dev, BF16, 200, 8, 1, 2000, 40, 1990, [20], seed=4, junk=0.0))
    cs.append(attn_case(dev, BF16, 5, 2, 4, 100, 40, 90, [20], seed=5, junk=0.0))
    logits = [torch.randn(16, 20000, device=dev, generator=torch.Generator(device=dev).manual_seed(i)) for i in range(4)]
    states = [pick_state(dev, 16, 40, 9, i)[1] for i in range(4)]
    outs = [tuple(torch.zeros_like(s[k]) for k in ORDER[:6]) for s in states]

    def run(i):
        cs[i]["run"]()
        beam.pick(logits[i], *(states[i][k] for k in ORDER), END_IDX=7, out=outs[i])
    want = []
    for i in range(4):
        run(i)
        want.append([t.clone() for t in (cs[i]["o"], *outs[i])])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=dev) for _ in range(2)]
    for _ in range(20):
        for i in range(4):
            with torch.cuda.stream(streams[i % 2]):
                run(i)
    torch.cuda.synchronize()
    for i in range(4):
        assert all(torch.equal(a, b) for a, b in zip(want[i], (cs[i]["o"], *outs[i])))


def test_attn_same_inputs_same_bits(dev):
    c = attn_case(dev, BF16, 8, 4, 4, 1500, 300, 1400, [250], seed=3, table=np.random.default_rng(0).integers(0, 8, (8, 300)))
    first = c["run"]().clone()
    for _ in range(5):
        c["o"].zero_()
        assert torch.equal(c["run"](), first)


def test_attn_workspace_contents_do_not_matter(dev):
    import _hiplib as HL
    c = attn_case(dev, F16, 3, 2, 2, 400, 100, 333, [5, 70, -1])
    want = c["run"]().clone()
    n = HL.lib().rk_beam_attn_ws_bytes(3, 4, 2, 400, 100)
    for fill in (0, 255):
        c["o"].zero_()
        assert torch.equal(c["run"](torch.full((n + 16,), fill, dtype=torch.uint8, device=dev)), want)
    with pytest.raises(RuntimeError, match="workspace"):
        c["run"](torch.zeros(n - 1, dtype=torch.uint8, device=dev))


# ------------------------------------------------------------------------------------------------------------- pick
def pick_state(dev, B, T, step, seed, done=()):
    r = np.random.default_rng(seed)
    st = dict(score=(-r.random(B) * 4 - 0.1 * step).astype(np.float32), done=np.isin(np.arange(B), done),
              lens=np.where(np.isin(np.arange(B), done), r.integers(0, step + 1, B), step), step=step,
              hist=r.integers(0, 1000, (B, T)), src=r.integers(0, B, (B, T)).astype(np.int32))
    gpu = dict(score=torch.tensor(st["score"]), done=torch.tensor(st["done"]), lens=torch.tensor(st["lens"]),
               step=torch.tensor([step]), hist=torch.tensor(st["hist"]), src=torch.tensor(st["src"]))
    gpu = {k: v.to(dev) for k, v in gpu.items()}
    gpu["tok"] = torch.full((B,), -7, dtype=torch.int64, device=dev)
    gpu["parent"] = torch.full((B,), -7, dtype=torch.int32, device=dev)
    return st, gpu


def check_pick(g, want, V):
    assert g["parent"].tolist() == want["parent"].tolist() and g["tok"].tolist() == want["tok"].tolist()
    assert g["done"].tolist() == want["done"].tolist() and g["lens"].tolist() == want["lens"].tolist()
    assert g["step"].item() == want["step"]
    assert np.array_equal(g["hist"].cpu().numpy(), want["hist"]) and np.array_equal(g["src"].cpu().numpy(), want["src"])
    got, ref = g["score"].double().cpu().numpy(), want["score"]
    fin = np.isfinite(ref)
    assert np.array_equal(got[~fin], ref[~fin])
    assert np.all(np.abs(got[fin] - ref[fin]) <= 2.0 ** -18 + U[torch.float32] * np.abs(ref[fin]))


ORDER = ("score", "done", "lens", "step", "hist", "src", "tok", "parent")


@pytest.mark.parametrize("B", [2, 7, 32])
@pytest.mark.parametrize("V", [5000, 20000, 66000])
def test_pick_uneven(V, B, dev):
    """Hypotheses that are far apart, from none to all but a few of them without a chance, and logits in order, in runs
    and in periods: the best candidates lie close together in some lists, lanes or waves."""
    g = torch.Generator().manual_seed(V + B)
    v = torch.arange(V).float()
    shapes = {"random": torch.randn(B, V, generator=g) * 3, "up": (v / V * 9).expand(B, V), "down": (-v / V * 9).expand(B, V),
              "hump": (-((v - V // 3) / 300) ** 2).expand(B, V) + torch.randn(B, V, generator=g) * 0.01,
              "period": torch.where(v % 64 == 5, v / V + 5, -v / V).expand(B, V)}
    for name, x in shapes.items():
        x = x.contiguous()
        for lead in (0.0, 0.3, 4.0, 60.0):
            st, s = pick_state(dev, B, 16, 9, V + B)
            st["score"] = (-lead * np.arange(B)[::-1] - 0.37 * (np.arange(B) % 3)).astype(np.float32)
            s["score"].copy_(torch.tensor(st["score"]))
            want = OB.pick(x.double().numpy(), *(st[k] for k in ORDER[:6]), V - 1, 0)
            beam.pick(x.to(dev), *(s[k] for k in ORDER), END_IDX=V - 1)
            check_pick(s, want, V)


@pytest.mark.parametrize("residues", [2, 3, 16, 31, 32, 63])
@pytest.mark.parametrize("B,V", [(4, 8192), (32, 8192), (32, 40001)])
def test_pick_best_tokens_at_few_residues(B, V, residues, dev):
    """The best tokens, all different, at a few residues of the index modulo 64: more candidates than are gathered."""
    g = torch.Generator().manual_seed(V + residues)
    high = torch.zeros(64, dtype=torch.bool)
    high[torch.randperm(64, generator=g)[:residues]] = True
    x = torch.stack([torch.randperm(V, generator=g) for _ in range(B)]).float() / V
    x[:, high[torch.arange(V) % 64]] += 8.0
    for lead in (0.0, 0.4):
        st, s = pick_state(dev, B, 16, 9, V + B)
        st["score"] = (-lead * np.arange(B)[::-1] - 0.37 * (np.arange(B) % 3)).astype(np.float32)
        s["score"].copy_(torch.tensor(st["score"]))
        want = OB.pick(x.double().numpy(), *(st[k] for k in ORDER[:6]), V - 1, 0)
        beam.pick(x.to(dev), *(s[k] for k in ORDER), END_IDX=V - 1)
        check_pick(s, want, V)


@pytest.mark.parametrize("dt", [torch.float32, F16, BF16])
@pytest.mark.parametrize("B,V,T,step,done", [(1, 1, 1, 0, ()), (1, 700, 4, 3, ()), (4, 4096, 40, 7, (2,)),
                                             (8, 16385, 600, 599, (0, 5)), (32, 5000, 1025, 1000, (1, 2, 30)),
                                             (5, 1025, 513, 0, ()), (3, 64, 9, 8, (0, 1, 2)), (32, 70001, 33, 20, ()),
                                             (7, 31, 10, 5, (6,)), (32, 20, 8, 3, ())])
def test_pick(dt, B, V, T, step, done, dev):
    g = torch.Generator().manual_seed(V)
    logits = (torch.randn(B, V, generator=g) * 3).to(dt)
    ids = torch.randperm(V, generator=g) + 5
    for inplace in (True, False):
        st, s = pick_state(dev, B, T, step, V + B, done)
        want = OB.pick(logits.double().numpy(), *(st[k] for k in ORDER[:6]), V - 1, 8, ids=ids.numpy())
        out = None
        if not inplace:
            out = tuple(torch.full_like(s[k], 1) for k in ORDER[:6])
            out[4].copy_(s["hist"] + 1000)
            out[5].copy_(s["src"] + 1000)
            want["hist"][:, step + 1:] += 1000
            want["src"][:, step + 1:] += 1000
        before = {k: s[k].clone() for k in ORDER[:6]}
        beam.pick(logits.to(dev), *(s[k] for k in ORDER), END_IDX=V - 1, MIN_NEW=8, ids=ids.to(dev), out=out)
        if not inplace:
            assert all(torch.equal(before[k], s[k]) for k in before)
            s.update(zip(ORDER[:6], out))
        check_pick(s, want, V)


def test_pick_ties(dev):
    """Equal values, within a row and between rows: the lower hypothesis, then the lower token."""
    B, V = 6, 3000
    logits = torch.zeros(B, V)
    logits[:, 5::700] = 2.0
    logits[3, 1] = -0.0
    st, s = pick_state(dev, B, 10, 9, 0)
    st["score"][:] = -1
    s["score"].fill_(-1)
    want = OB.pick(logits.double().numpy(), *(st[k] for k in ORDER[:6]), V - 1)
    assert want["parent"].tolist() == [0] * 5 + [1] and want["tok"].tolist() == [5, 705, 1405, 2105, 2805, 5]
    beam.pick(logits.to(dev), *(s[k] for k in ORDER), END_IDX=V - 1)
    check_pick(s, want, V)
    # all logits equal: the lowest tokens; -0 is no less than 0
    st, s = pick_state(dev, B, 10, 9, 0)
    logits = torch.zeros(B, V)
    logits[:, ::2] = -0.0
    st["score"][:] = [-3, -1, -1, -1, -1, -1]
    s["score"].copy_(torch.tensor(st["score"]))
    want = OB.pick(logits.double().numpy(), *(st[k] for k in ORDER[:6]), V - 1)
    assert want["parent"].tolist() == [1] * 6 and want["tok"].tolist() == list(range(6))
    beam.pick(logits.to(dev), *(s[k] for k in ORDER), END_IDX=V - 1)
    check_pick(s, want, V)


@pytest.mark.parametrize("B,V", [(32, 100), (32, 5000), (9, 8193), (32, 270001)])
def test_pick_nothing_but_ties(B, V, dev):
    """Every candidate of every hypothesis equal; and all but a few."""
    for extra in (0, 3):
        logits = torch.zeros(B, V, dtype=F16)
        if extra:
            logits[B // 2, V // 2:V // 2 + extra] = 1
        st, s = pick_state(dev, B, 4, 2, 1)
        st["score"][:] = -2
        s["score"].fill_(-2)
        x = logits.double().numpy()
        if V > 10000:  # the oracle's own pick sorts every row
            val = -2 - math.log(V)
            val2 = -2 - math.log(V - extra + extra * math.e) if extra else val
            order = [(1 + val2, B // 2, V // 2 + i) for i in range(extra)] + [(val, 0, i) for i in range(B)]
            order = order[:B]
            assert s["hist"].shape == (B, 4)
            beam.pick(logits.to(dev), *(s[k] for k in ORDER), END_IDX=V - 1)
            assert s["parent"].tolist() == [o[1] for o in order] and s["tok"].tolist() == [o[2] for o in order]
            assert np.allclose(s["score"].cpu().numpy(), [o[0] for o in order], atol=2.0 ** -18)
            continue
        want = OB.pick(x, *(st[k] for k in ORDER[:6]), V - 1)
        beam.pick(logits.to(dev), *(s[k] for k in ORDER), END_IDX=V - 1)
        check_pick(s, want, V)


def test_pick_best_tokens_side_by_side(dev):
    """All the best of a row in one lane's, one wave's and one piece's reach, rising and falling."""
    V, B = 9000, 32
    for start, stepw in ((0, 1), (4000, 1), (8968, 1), (7, 64), (100, 256), (3, 128)):
        for sign in (1, -1):
            logits = torch.randn(B, V, generator=torch.Generator().manual_seed(start)) * 0.1
            at = torch.arange(B) * stepw + start
            at = at[at < V]
            logits[1, at] = 10 + sign * torch.arange(len(at)) * 0.25
            st, s = pick_state(dev, B, 4, 2, 1)
            st["score"][:] = 0
            s["score"].zero_()
            want = OB.pick(logits.double().numpy(), *(st[k] for k in ORDER[:6]), 0)
            beam.pick(logits.to(dev), *(s[k] for k in ORDER), END_IDX=0)
            check_pick(s, want, V)


def test_pick_special_logits(dev):
    inf, nan = float("inf"), float("nan")
    B, V = 5, 1500
    for dt in (torch.float32, F16, BF16):
        logits = (torch.randn(B, V, generator=torch.Generator().manual_seed(3)) * 2).to(dt)
        logits[0, ::3] = nan
        logits[1, :] = -inf
        logits[2, 100], logits[2, 1200] = inf, inf
        logits[3, :] = nan
        logits[4, 7], logits[4, 8] = -inf, nan
        st, s = pick_state(dev, B, 6, 5, 2)
        x = logits.double().numpy()
        x[2][x[2] == np.inf] = np.finfo(np.float32).max
        want = OB.pick(x, *(st[k] for k in ORDER[:6]), V - 1)
        beam.pick(logits.to(dev), *(s[k] for k in ORDER), END_IDX=V - 1)
        check_pick(s, want, V)


def test_pick_start_end_and_too_few_candidates(dev):
    """One live hypothesis fans out; with less than B tokens the others end and stay ended; NaN scores count for
    nothing."""
    B, V, T = 6, 4, 5
    search = beam.BeamSearch(B, T, torch.arange(V, device=dev) + 50, end_id=53, min_new=1)
    logits = torch.randn(B, V, generator=torch.Generator().manual_seed(0))
    st = dict(score=np.array([0] + [-np.inf] * (B - 1)), done=np.zeros(B, bool), lens=np.zeros(B, np.int64), step=0,
              hist=np.zeros((B, T), np.int64), src=np.zeros((B, T), np.int32))
    for i in range(T):
        want = OB.pick(logits.double().numpy(), *(st[k] for k in ORDER[:6]), V - 1, 1, ids=np.arange(V) + 50)
        search(logits.to(dev))
        got = {k: getattr(search, k) for k in ORDER}
        check_pick(got, want, V)
        st = {k: got[k].cpu().numpy() for k in ORDER[:6]}
        st["step"] = i + 1
        if i == 0:
            assert np.isinf(st["score"][3:]).all() and st["done"][3:].all()
    before = {k: getattr(search, k).clone() for k in ORDER}
    search(logits.to(dev))  # no column left: nothing is written
    assert all(torch.equal(before[k], getattr(search, k)) for k in ORDER)
    search.step.fill_(-1)
    search(logits.to(dev))
    assert all(torch.equal(before[k], getattr(search, k)) for k in ORDER if k != "step")
    search.reset()
    search.score.fill_(float("nan"))
    search(logits.to(dev))
    assert search.done.all() and torch.isinf(search.score).all()


def test_pick_strided_logits_and_own_ids(dev):
    B, V = 4, 999
    full = torch.randn(B, V + 37, generator=torch.Generator().manual_seed(1)).to(F16)
    full[:, V:] = 100
    st, s = pick_state(dev, B, 4, 1, 4)
    want = OB.pick(full[:, :V].double().numpy(), *(st[k] for k in ORDER[:6]), 3)
    beam.pick(full.to(dev)[:, :V], *(s[k] for k in ORDER), END_IDX=3)
    check_pick(s, want, V)


def test_pick_captured(dev):
    B, V, T = 8, 16385, 40
    search = beam.BeamSearch(B, T, torch.arange(V, device=dev), end_id=V - 1)
    eager = beam.BeamSearch(B, T, torch.arange(V, device=dev), end_id=V - 1)
    logits = torch.zeros(B, V, device=dev)
    search(logits)
    search.reset()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        search(logits)
    for i in range(12):
        logits.copy_(torch.randn(B, V, generator=torch.Generator().manual_seed(i)) * 3)
        g.replay()
        eager(logits)
        torch.cuda.synchronize()
        for k in ORDER:
            assert torch.equal(getattr(search, k), getattr(eager, k)), (i, k)


# --------------------------------------------------------------------------------------------------- a run of them
@pytest.mark.parametrize("q8", [False, True])
def test_beam_search_of_a_decoder(q8, dev):
    """A beam search over a small decoder, its steps captured in one graph: the prompt through the batched prefill, its
    cache quantised or plain, every step's rows through mm_int4, post, attn and pick. Every hypothesis, taken by itself
    through the batch-1 decode step over the same prompt, has the score that the search gave it."""
    B, T = 4, 6
    cfg = decode.Config(L=2, H=256, NH=4, NKV=2, inter=512, S=64, n_audio=300, vocab=400)
    w = decode.random_weights(cfg, 5, dev)
    prompt = [3, 77, 150, 9, 222]
    one = decode.DecodeStep(cfg, w, device=dev)
    pre = prefill.Prefill(cfg, w, one.kc, one.vc, one.cos, one.sin, max_T=16)
    hn = pre.run(prompt).clone()
    head = (w["head"][0].float() * w["head"][1].float()[:, None]).contiguous()
    ids = torch.arange(300, device=dev) + 40
    search = beam.BeamSearch(B, T, ids, end_id=339, min_new=T)
    plen, spos = i64(dev, len(prompt)), i64(dev, 0)
    if q8:
        kc, vc = kv8.empty(*one.kc.shape, device=dev), kv8.empty(*one.kc.shape, device=dev)
        kv8.quantize(one.kc, one.vc, kc, vc, n=len(prompt))
        ks, vs = kv8.empty(cfg.L, B, 2, T, HD, device=dev), kv8.empty(cfg.L, B, 2, T, HD, device=dev)
        layer = lambda c, i: (c[0][i], c[1][i])  # noqa: E731
    else:
        kc, vc = one.kc, one.vc
        ks, vs = (torch.full((cfg.L, B, 2, T, HD), float("nan"), device=dev, dtype=F16) for _ in range(2))
        layer = lambda c, i: c[i]  # noqa: E731
    zz = lambda n: torch.zeros(B, n, device=dev, dtype=F16)  # noqa: E731
    x, h, y, q, o, act, a, d = (zz(n) for n in (256, 256, cfg.n_in, 512, 512, 512, 256, 256))
    logits = torch.zeros(B, 300, device=dev)

    def step():
        prefill.embed_ln_rows(search.tok, w["emb"][0], w["emb"][1], w["ln"][0], x, h, cfg.eps)
        for i in range(cfg.L):
            mm_int4.mm_int4(h, *w["w_in"][i], out=y)
            beam.post(y, spos, plen, one.cos, one.sin, layer(ks, i), layer(vs, i), q, act, NH=4, NKV=2, HD=HD,
                      ROPE=cfg.sliding[i])
            beam.attn(q, layer(kc, i), layer(vc, i), plen, layer(ks, i), layer(vs, i), spos, o, HD ** -0.5,
                      src=search.src)
            mm_int4.mm_int4(o, *w["w_o"][i], out=a)
            mm_int4.mm_int4(act, *w["w_down"][i], out=d)
            prefill.add_ln_rows(x, a, d, w["norm"] if i == cfg.L - 1 else w["ln"][i + 1], h, B, cfg.eps)
        torch.matmul(h.float(), head.t(), out=logits)
        search(logits)
        fused.pos_advance(spos)

    first = (hn.float() @ head.t()).expand(B, -1).contiguous()
    # warm up and capture, then the search itself from its start
    search(first)
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    search.reset()
    spos.zero_()
    search(first)
    for _ in range(T - 1):
        g.replay()
    torch.cuda.synchronize()
    assert search.step.item() == T and search.lens.tolist() == [T] * B and not search.done.any()
    hist = search.hist.cpu()
    assert len({tuple(r.tolist()) for r in hist}) == B
    total = []
    for b in range(B):
        pre.run(prompt)
        lp = 0.0
        row = hn
        for t in range(T):
            p = torch.log_softmax(row.double() @ head.double().t(), -1)
            p_end = torch.log_softmax((row.double() @ head.double().t()).masked_fill(ids == 339, -math.inf), -1)
            lp += (p_end if t < T else p)[hist[b, t] - 40].item()
            one.set_state(int(hist[b, t]), len(prompt) + t)
            one.step()
            row = one.h
        total.append(lp)
    # fp16 activations over two layers in both paths, int8 caches in one of them
    assert np.allclose(search.score.cpu().numpy(), total, atol=0.15 if q8 else 0.05), (search.score, total)


@pytest.mark.parametrize("q8", [False, True])
def test_beam_search_step_by_step(q8, dev):
    """The same decoder, every captured step against the oracle's selection from the logits that the step itself made and
    the states before it; with an end token that some hypotheses take on the way."""
    B, T, V = 5, 9, 300
    cfg = decode.Config(L=2, H=256, NH=4, NKV=2, inter=512, S=64, n_audio=V, vocab=400)
    w = decode.random_weights(cfg, 5, dev)
    prompt = [11, 5, 140]
    one = decode.DecodeStep(cfg, w, device=dev)
    first = prefill.Prefill(cfg, w, one.kc, one.vc, one.cos, one.sin, max_T=16).run(prompt)
    head = (w["head"][0].float() * w["head"][1].float()[:, None]).contiguous()
    first = (first.float() @ head.t()).expand(B, -1).contiguous()
    ids = torch.arange(V, device=dev) + 40
    plen, spos = i64(dev, len(prompt)), i64(dev, 0)
    kc, vc = one.kc, one.vc
    cache = lambda: torch.full((cfg.L, B, 2, T, HD), float("nan"), device=dev, dtype=F16)  # noqa: E731
    layer = lambda c, i: c[i]  # noqa: E731
    if q8:
        kc, vc = kv8.empty(*one.kc.shape, device=dev), kv8.empty(*one.kc.shape, device=dev)
        kv8.quantize(one.kc, one.vc, kc, vc, n=len(prompt))
        cache = lambda: kv8.empty(cfg.L, B, 2, T, HD, device=dev)  # noqa: E731
        layer = lambda c, i: (c[0][i], c[1][i])  # noqa: E731
    ks, vs = cache(), cache()
    zz = lambda n: torch.zeros(B, n, device=dev, dtype=F16)  # noqa: E731
    x, h, y, q, o, act, a, d = (zz(n) for n in (256, 256, cfg.n_in, 512, 512, 512, 256, 256))
    logits = torch.zeros(B, V, device=dev)

    def step(search):
        prefill.embed_ln_rows(search.tok, w["emb"][0], w["emb"][1], w["ln"][0], x, h, cfg.eps)
        for i in range(cfg.L):
            mm_int4.mm_int4(h, *w["w_in"][i], out=y)
            beam.post(y, spos, plen, one.cos, one.sin, layer(ks, i), layer(vs, i), q, act, NH=4, NKV=2, HD=HD,
                      ROPE=cfg.sliding[i])
            beam.attn(q, layer(kc, i), layer(vc, i), plen, layer(ks, i), layer(vs, i), spos, o, HD ** -0.5,
                      src=search.src)
            mm_int4.mm_int4(o, *w["w_o"][i], out=a)
            mm_int4.mm_int4(act, *w["w_down"][i], out=d)
            prefill.add_ln_rows(x, a, d, w["norm"] if i == cfg.L - 1 else w["ln"][i + 1], h, B, cfg.eps)
        torch.matmul(h.float(), head.t(), out=logits)
        search(logits)
        fused.pos_advance(spos)

    # a first search tells which token some hypothesis takes as its fourth one: in the second it is the end
    end = 40
    for captured in (False, True):
        search = beam.BeamSearch(B, T, ids, end_id=end, min_new=2)
        if captured:
            search(first)
            step(search)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step(search)
            search.reset()
        spos.zero_()
        for t in range(T):
            before = [getattr(search, k).cpu().numpy().copy() for k in ORDER[:6]]
            before[3] = int(before[3][0])
            if t == 0:
                search(first)
            elif captured:
                graph.replay()
            else:
                step(search)
            torch.cuda.synchronize()
            want = OB.pick((logits if t else first).double().cpu().numpy(), *before, end - 40, 2, ids=ids.cpu().numpy())
            check_pick({k: getattr(search, k) for k in ORDER}, want, V)
        if captured:
            assert search.done.any() and search.lens.min() < T
        end = int(search.hist[0, 3])
