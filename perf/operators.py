"""Several hypotheses of one prompt, decoded side by side by a batch-1 int4 decoder (hidden 2048, 16 query / 4 KV heads
of 128, MLP 11008, 16385 audio logits, 2048 cache slots): the operators around the projections of such a step, as timed
cases.

  attn  decode attention of B hypotheses over a shared prompt cache (the prefix) and a cache of their own (the suffix),
        whose slots are found through a table once a beam search has reordered the hypotheses
  post  what follows the fused projection for B rows: RoPE of q and k, the K / V write into the suffix cache (as the
        activations' type or quantised to int8 with one scale per slot and head), SiLU(gate) * up
  kv8   a plain K / V cache quantised to int8 and read back
  pick  a beam search's selection over hypotheses and vocabulary, with the reordering of their states

listed() and draw() give cases as dicts of plain values, prepare() a case's inputs on the GPU, run() one pass: in plain
torch where `own` is false, through the package's entry points where it is true. work() is what a pass cannot do
without, exact() the same outputs in 64 bits.
"""
import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DEV = "cuda"
HD = 128
THETA = 10000.0
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
PKG = Path(__file__).resolve().parents[1] / "rumik-fast_amd"


def _modules():
    """the package's modules, imported by name as its users do"""
    for p in (PKG / "kernels", PKG / "engine"):
        if str(p) not in sys.path:
            sys.path.insert(0, str(p))
    import beam
    import kv8
    return beam, kv8


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the smallest attention call: four hypotheses of a usual sentence (34 prompt tokens), nine tokens in
        {"name": "attn_4x34", "op": "attn", "B": 4, "nkv": 4, "rep": 4, "S": 2048, "plen": 34, "T": 256, "slen": 9,
         "dtype": "fp16", "p8": False, "s8": False, "table": True},
        # a beam search over a long prompt, half a minute of audio tokens in
        {"name": "attn_8x512", "op": "attn", "B": 8, "nkv": 4, "rep": 4, "S": 2048, "plen": 512, "T": 1024,
         "slen": 700, "dtype": "bf16", "p8": False, "s8": False, "table": True},
        # best-of-16 over a cache filled to its last slot, everything in int8, hypotheses of different lengths
        {"name": "attn_16x2047_q8", "op": "attn", "B": 16, "nkv": 4, "rep": 4, "S": 2048, "plen": 2047, "T": 513,
         "slen": 513, "dtype": "bf16", "p8": True, "s8": True, "table": False},
        # a document as the prompt, quantised after its prefill; few hypotheses, short plain suffixes
        {"name": "attn_5x30001_q8", "op": "attn", "B": 5, "nkv": 8, "rep": 2, "S": 32768, "plen": 30001, "T": 64,
         "slen": 33, "dtype": "fp16", "p8": True, "s8": False, "table": True},
        # the largest: many hypotheses over the longest prompt, wide heads
        {"name": "attn_32x65536", "op": "attn", "B": 32, "nkv": 8, "rep": 4, "S": 65536, "plen": 65536, "T": 512,
         "slen": 300, "dtype": "fp16", "p8": False, "s8": False, "table": False},
        # one layer's rows after the projection, four hypotheses, plain suffix cache
        {"name": "post_4", "op": "post", "B": 4, "nkv": 4, "rep": 4, "inter": 11008, "T": 256, "slot": 9, "plen": 34,
         "dtype": "fp16", "s8": False, "rope": True},
        # 32 hypotheses into an int8 suffix cache, which is then read back
        {"name": "post_32_q8", "op": "post", "B": 32, "nkv": 4, "rep": 4, "inter": 11008, "T": 256, "slot": 200,
         "plen": 512, "dtype": "bf16", "s8": True, "rope": True},
        # a short prompt's slots of one layer, quantised and read back
        {"name": "kv8_34", "op": "kv8", "heads": 4, "S": 2048, "t0": 0, "n": 34, "dtype": "fp16"},
        # a long prompt's slots of all 36 layers in one call
        {"name": "kv8_36x1999", "op": "kv8", "heads": 144, "S": 2048, "t0": 1, "n": 1999, "dtype": "bf16"},
        # a small search over the text vocabulary, early on
        {"name": "pick_4x4096", "op": "pick", "B": 4, "V": 4096, "T": 256, "step": 3, "dtype": "fp32", "done": 0},
        # the audio head's logits, well into a sentence, two hypotheses ended
        {"name": "pick_8x16385", "op": "pick", "B": 8, "V": 16385, "T": 1024, "step": 700, "dtype": "fp32", "done": 2},
        # the widest search over a large vocabulary and a long history
        {"name": "pick_32x131101", "op": "pick", "B": 32, "V": 131101, "T": 4096, "step": 4001, "dtype": "bf16",
         "done": 5},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "post", "kv8", "pick", "pick"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "attn":
        rep = rng.choice([1, 2, 4, 8])
        nkv = rng.choice([1, 2, 4, 8] if rep < 8 else [1, 2, 4])
        plen = _log(rng, 1, 65536) if rng.random() < 0.9 else 0
        slen = _log(rng, 1, 1024) if plen == 0 or rng.random() < 0.9 else 0
        return {"op": op, "B": _log(rng, 1, 32), "nkv": nkv, "rep": rep, "S": plen + rng.randrange(1, 100),
                "plen": plen, "T": slen + rng.randrange(1, 100), "slen": slen, "dtype": dtype,
                "p8": rng.random() < 0.5, "s8": rng.random() < 0.5, "table": rng.random() < 0.5}
    if op == "post":
        T = _log(rng, 1, 512)
        return {"op": op, "B": _log(rng, 1, 64), "nkv": rng.choice([1, 2, 4, 8]), "rep": rng.choice([1, 2, 4]),
                "inter": _log(rng, 64, 16384), "T": T, "slot": rng.randrange(T), "plen": _log(rng, 1, 2048),
                "dtype": dtype, "s8": rng.random() < 0.6, "rope": rng.random() < 0.75}
    if op == "kv8":
        n, t0 = _log(rng, 1, 2048), rng.randrange(0, 20)
        return {"op": op, "heads": _log(rng, 1, 144), "S": t0 + n + rng.randrange(0, 50), "t0": t0, "n": n,
                "dtype": dtype}
    B, T = _log(rng, 1, 32), _log(rng, 2, 4096)
    return {"op": op, "B": B, "V": _log(rng, 50, 131072), "T": T, "step": rng.randrange(T),
            "dtype": rng.choice(["fp16", "bf16", "fp32"]), "done": rng.randrange(0, B // 3 + 1)}


# ------------------------------------------------------------------------------------------------------------ inputs
def _ancestry(B, n, seed):
    """table[b, t]: the hypothesis that wrote slot t of what is now hypothesis b, after n steps of a search whose
    survivors come from the better half of the hypotheses more often than from the others"""
    r = random.Random(seed)
    rows, cols = list(range(B)), []
    for _ in range(n):
        cols.append(rows)
        parent = sorted(min(r.randrange(B), r.randrange(B)) for _ in range(B))
        rows = [parent[b] for b in rows]
    return torch.tensor(cols[::-1], dtype=torch.int32).t().contiguous() if n else torch.zeros(B, 0, dtype=torch.int32)


def _table_rows(case):
    """distinct (row, slot) pairs of the case's table, from one such search"""
    t = _ancestry(case["B"], case["slen"], 1).numpy()
    return sum(len(np.unique(t[:, k])) for k in range(t.shape[1]))


def _cache(shape, dt, quantised, g):
    if not quantised:
        return torch.randn(shape, device=DEV, dtype=dt, generator=g)
    codes = (torch.randn(shape, device=DEV, dtype=torch.float16, generator=g) * 45).round().clamp(-127, 127)
    scales = torch.rand(shape[:-1], device=DEV, dtype=torch.float32, generator=g) * 0.02 + 0.012
    return codes.to(torch.int8), scales


def _rope_tables(n, dt):
    inv = 1.0 / (THETA ** (torch.arange(0, HD, 2, dtype=torch.float32) / HD))
    a = torch.outer(torch.arange(n, dtype=torch.float32), inv).repeat_interleave(2, -1)
    return a.cos().to(dt).to(DEV), a.sin().to(dt).to(DEV)


def prepare(case, seed):
    c, dt = case, DT[case["dtype"]]
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = random.Random(seed)
    s = {"c": dict(c)}
    if c["op"] == "attn":
        B, nkv, NH = c["B"], c["nkv"], c["nkv"] * c["rep"]
        s["q"] = torch.randn(B, NH * HD, device=DEV, dtype=dt, generator=g) * 2
        s["kc"], s["vc"] = (_cache((nkv, c["S"], HD), dt, c["p8"], g) for _ in range(2))
        s["ks"], s["vs"] = (_cache((B, nkv, c["T"], HD), dt, c["s8"], g) for _ in range(2))
        s["plen"] = torch.tensor([c["plen"]], device=DEV)
        # the slot of each hypothesis's newest token: the same where a table leads to the slots (a search in step),
        # else ragged, one hypothesis at the full length
        slots = [c["slen"] - 1] * B if c["table"] else [c["slen"] - 1] + [r.randrange(-1, c["slen"]) for _ in range(B - 1)]
        s["spos"] = torch.tensor(slots, device=DEV)
        s["src"] = None
        if c["table"]:
            src = torch.zeros(B, c["T"], dtype=torch.int32)
            src[:, :c["slen"]] = _ancestry(B, c["slen"], seed)
            s["src"] = src.to(DEV)
        s["o"] = torch.zeros(B, NH * HD, device=DEV, dtype=dt)
    elif c["op"] == "post":
        B, nkv, NH = c["B"], c["nkv"], c["nkv"] * c["rep"]
        s["y"] = torch.randn(B, (NH + 2 * nkv) * HD + 2 * c["inter"], device=DEV, dtype=dt, generator=g)
        s["cos"], s["sin"] = _rope_tables(c["plen"] + c["T"], dt)
        s["ks"], s["vs"] = (_cache((B, nkv, c["T"], HD), dt, c["s8"], g) for _ in range(2))
        s["plen"], s["spos"] = torch.tensor([c["plen"]], device=DEV), torch.tensor([c["slot"]], device=DEV)
        s["q"] = torch.zeros(B, NH * HD, device=DEV, dtype=dt)
        s["act"] = torch.zeros(B, c["inter"], device=DEV, dtype=dt)
        s["kr"], s["vr"] = (torch.zeros(B, nkv, c["T"], HD, device=DEV, dtype=dt) for _ in range(2))
    elif c["op"] == "kv8":
        shape = (c["heads"], c["S"], HD)
        # keys have a few large dims, values do not
        s["kc"], s["vc"] = (torch.randn(shape, device=DEV, dtype=dt, generator=g) for _ in range(2))
        s["kc"][..., ::37] *= 6
        s["k8"], s["v8"] = ((torch.zeros(shape, device=DEV, dtype=torch.int8),
                             torch.zeros(shape[:-1], device=DEV)) for _ in range(2))
        s["kr"], s["vr"] = (torch.zeros(shape, device=DEV, dtype=dt) for _ in range(2))
    else:
        B, V, T = c["B"], c["V"], c["T"]
        s["logits"] = (torch.randn(B, V, device=DEV, generator=g) * 3).to(dt)
        s["score"] = -torch.rand(B, device=DEV, generator=g) * 4 - 0.1 * c["step"]
        s["ids"] = torch.randperm(V, device=DEV, generator=g) + 7
        done = torch.zeros(B, dtype=torch.bool)
        done[r.sample(range(B), c["done"])] = True
        s["done"] = done.to(DEV)
        s["lens"] = torch.tensor([r.randrange(c["step"] + 1) if d else c["step"] for d in done.tolist()], device=DEV)
        s["step"] = torch.tensor([c["step"]], device=DEV)
        s["hist"] = torch.randint(0, V, (B, T), device=DEV, generator=g)
        s["src"] = torch.randint(0, B, (B, T), device=DEV, dtype=torch.int32, generator=g)
        s["tok"] = torch.zeros(B, device=DEV, dtype=torch.int64)
        s["parent"] = torch.zeros(B, device=DEV, dtype=torch.int32)
        s["out"] = tuple(torch.zeros_like(s[k]) for k in ("score", "done", "lens", "step", "hist", "src"))
        s["end"], s["min_new"] = V - 1, 8
    return s


# -------------------------------------------------------------------------------------------------------- plain forms
def _values(cache):
    return cache[0].float() * cache[1][..., None] if isinstance(cache, tuple) else cache.float()


def _cut(cache, n):
    """the first n slots (the next to last dim of the codes and values)"""
    return (cache[0][..., :n, :], cache[1][..., :n]) if isinstance(cache, tuple) else cache[..., :n, :]


def _gathered(cache, src, n):
    """[B, nkv, n, ...]: slot t of hypothesis b from row src[b, t]"""
    t = torch.arange(n, device=DEV)
    pick = lambda x: x[src[:, :n].long(), :, t].transpose(1, 2)  # noqa: E731
    return tuple(pick(x) for x in cache) if isinstance(cache, tuple) else pick(cache)


def _attn(s):
    c = s["c"]
    B, nkv, rep, n, m = c["B"], c["nkv"], c["rep"], c["plen"], c["slen"]
    q = s["q"].float().view(B, nkv, rep, HD)
    qg = q.transpose(0, 1).reshape(nkv, B * rep, HD)
    kp, vp = _values(_cut(s["kc"], n)), _values(_cut(s["vc"], n))
    sp = torch.matmul(qg, kp.transpose(1, 2).contiguous()).view(nkv, B, rep, n).transpose(0, 1) * HD ** -0.5
    ks, vs = ((_gathered(x, s["src"], m) if c["table"] else _cut(x, m)) for x in (s["ks"], s["vs"]))
    ks, vs = _values(ks), _values(vs)
    ss = torch.matmul(q, ks.transpose(2, 3).contiguous()) * HD ** -0.5
    empty = torch.arange(m, device=DEV) > s["spos"][:, None]
    ss = ss.masked_fill(empty[:, None, None], -math.inf)
    top = torch.cat((sp, ss), -1).amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    ep, es = torch.exp(sp - top), torch.exp(ss - top)
    total = ep.sum(-1, keepdim=True) + es.sum(-1, keepdim=True)
    o = torch.matmul(ep.transpose(0, 1).reshape(nkv, B * rep, n), vp).view(nkv, B, rep, HD).transpose(0, 1)
    o = (o + torch.matmul(es, vs)) / total
    s["o"].copy_(torch.where(total > 0, o, torch.zeros_like(o)).reshape(B, -1))
    return s["o"]


def _quantised(x):
    """int8 codes and one fp32 scale per row of HD values: the nearest codes, ties to even"""
    scale = (x.float().abs().amax(-1).double() / 127).float()
    code = (x.double() / scale.double()[..., None]).round()
    return torch.where(scale[..., None] > 0, code, torch.zeros_like(code)).to(torch.int8), scale


def _post(s):
    c, dt = s["c"], s["y"].dtype
    B, nkv, rep, slot = c["B"], c["nkv"], c["rep"], c["slot"]
    NH, inter = nkv * rep, c["inter"]
    y = s["y"].float()
    qk, v, gate, up = y.split([(NH + nkv) * HD, nkv * HD, inter, inter], -1)
    qk, v = qk.view(B, NH + nkv, HD), v.view(B, nkv, HD)
    if c["rope"]:
        cos, sin = (t.index_select(0, s["plen"] + s["spos"]).float()[:, None, 0::2] for t in (s["cos"], s["sin"]))
        e, o = qk[..., 0::2], qk[..., 1::2]
        qk = torch.stack((e * cos - o * sin, o * cos + e * sin), -1).flatten(-2)
    s["q"].copy_(qk[:, :NH].reshape(B, -1))
    s["act"].copy_(gate / (1 + torch.exp(-gate)) * up)
    k, v = qk[:, NH:].to(dt), v.to(dt)
    if not c["s8"]:
        s["ks"][:, :, slot], s["vs"][:, :, slot] = k, v
        return {"q": s["q"], "act": s["act"], "k": s["ks"], "v": s["vs"]}
    for cache, x, back in ((s["ks"], k, s["kr"]), (s["vs"], v, s["vr"])):
        cache[0][:, :, slot], cache[1][:, :, slot] = _quantised(x)
        back.copy_(_values(cache))
    return {"q": s["q"], "act": s["act"], "k": s["kr"], "v": s["vr"]}


def _kv8(s):
    c = s["c"]
    at = slice(c["t0"], c["t0"] + c["n"])
    for x, cache, back in ((s["kc"], s["k8"], s["kr"]), (s["vc"], s["v8"], s["vr"])):
        cache[0][:, at], cache[1][:, at] = _quantised(x[:, at])
        back[:, at] = _values((cache[0][:, at], cache[1][:, at])).to(back.dtype)
    return {"k": s["kr"], "v": s["vr"], "k_scale": s["k8"][1], "v_scale": s["v8"][1]}


def _pick(s):
    c, inf = s["c"], math.inf
    B, V, step = c["B"], c["V"], c["step"]
    score, done, lens, nstep, hist, src = s["out"]
    x = s["logits"].float() + 0.0  # -0 is 0
    if step < s["min_new"]:
        x[:, s["end"]] = -inf
    # every hypothesis's best tokens, the lowest index first where logits are equal: value and index as one key
    k = min(B, V)
    bits = x.view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    idx = 0xFFFFFFFF - (torch.topk((bits << 32) + (0xFFFFFFFF - torch.arange(V, device=DEV)), k, -1)[0] & 0xFFFFFFFF)
    # their scores in 64 bits: those of two hypotheses may be nearer to each other than fp32 sums tell
    x = x.double()
    x = x - x.amax(-1, keepdim=True)
    best = x.gather(-1, idx) - torch.log(torch.exp(x).sum(-1, keepdim=True)) + s["score"].double()[:, None]
    # a hypothesis that has ended goes on as it is
    best = torch.where(s["done"][:, None], torch.full_like(best, -inf), best)
    best[:, 0] = torch.where(s["done"], s["score"].double(), best[:, 0])
    idx[:, 0] = torch.where(s["done"], torch.full_like(idx[:, 0], s["end"]), idx[:, 0])
    top, at = torch.sort(best.reshape(-1), stable=True, descending=True)
    top, at = top[:B], at[:B]
    parent = torch.div(at, k, rounding_mode="floor")
    token = idx.reshape(-1)[at]
    was = s["done"][parent]
    score.copy_(top)
    lens.copy_(s["lens"][parent] + (~was).long())
    done.copy_(was | (token == s["end"]))
    s["tok"].copy_(s["ids"][token])
    s["parent"].copy_(parent)
    hist[:, :step] = s["hist"][parent, :step]
    src[:, :step] = s["src"][parent, :step]
    hist[:, step] = s["tok"]
    src[:, step] = torch.arange(B, device=DEV, dtype=torch.int32)
    nstep.copy_(s["step"] + 1)
    return {"tok": s["tok"], "parent": s["parent"], "state": s["out"]}


# ----------------------------------------------------------------------------------------------------- the package's
def _run_own(s):
    beam, kv8 = _modules()
    c = s["c"]
    if c["op"] == "attn":
        return beam.attn(s["q"], s["kc"], s["vc"], s["plen"], s["ks"], s["vs"], s["spos"], s["o"], HD ** -0.5,
                         src=s["src"])
    if c["op"] == "post":
        beam.post(s["y"], s["spos"], s["plen"], s["cos"], s["sin"], s["ks"], s["vs"], s["q"], s["act"],
                  NH=c["nkv"] * c["rep"], NKV=c["nkv"], HD=HD, ROPE=c["rope"])
        if not c["s8"]:
            return {"q": s["q"], "act": s["act"], "k": s["ks"], "v": s["vs"]}
        kv8.dequantize(s["ks"], s["vs"], s["kr"], s["vr"])
        return {"q": s["q"], "act": s["act"], "k": s["kr"], "v": s["vr"]}
    if c["op"] == "kv8":
        kv8.quantize(s["kc"], s["vc"], s["k8"], s["v8"], t0=c["t0"], n=c["n"])
        kv8.dequantize(s["k8"], s["v8"], s["kr"], s["vr"], t0=c["t0"], n=c["n"])
        return {"k": s["kr"], "v": s["vr"], "k_scale": s["k8"][1], "v_scale": s["v8"][1]}
    beam.pick(s["logits"], s["score"], s["done"], s["lens"], s["step"], s["hist"], s["src"], s["tok"], s["parent"],
              END_IDX=s["end"], MIN_NEW=s["min_new"], ids=s["ids"], out=s["out"])
    return {"tok": s["tok"], "parent": s["parent"], "state": s["out"]}


def run(state):
    if own:
        return _run_own(state)
    return {"attn": _attn, "post": _post, "kv8": _kv8, "pick": _pick}[state["c"]["op"]](state)


# -------------------------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    row8 = HD + 4  # a quantised slot of one head
    if c["op"] == "attn":
        NH = c["nkv"] * c["rep"]
        # ragged lengths are uniform below the longest
        slots = c["B"] * c["slen"] if c["table"] else c["slen"] + (c["B"] - 1) * (c["slen"] - 1) / 2
        rows = _table_rows(c) if c["table"] else slots
        kv = c["plen"] * (row8 if c["p8"] else 2 * HD) + rows * (row8 if c["s8"] else 2 * HD)
        return {"bytes": 2 * c["nkv"] * kv + 4 * c["B"] * NH * HD + 4 * (c["B"] * c["slen"] if c["table"] else 0),
                "flops": 4 * HD * NH * (c["B"] * c["plen"] + slots)}
    if c["op"] == "post":
        n = c["B"] * ((2 * c["rep"] + 2) * c["nkv"] * HD + 3 * c["inter"])  # q, k, v, gate, up in; q and act out
        kv = 2 * c["B"] * c["nkv"] * (c["T"] * (row8 + 2 * HD) + row8 if c["s8"] else 2 * HD)
        return {"bytes": 2 * n + kv, "flops": c["B"] * (3 * (c["rep"] + 1) * c["nkv"] * HD + 5 * c["inter"])}
    if c["op"] == "kv8":
        rows = 2 * c["heads"] * c["n"]
        return {"bytes": rows * 2 * (row8 + 2 * HD), "flops": rows * 4 * HD}
    size = {"fp16": 2, "bf16": 2, "fp32": 4}[c["dtype"]]
    return {"bytes": c["B"] * (c["V"] * size + 2 * 12 * c["step"] + 64), "flops": 4 * c["B"] * c["V"]}


# -------------------------------------------------------------------------------------------------- the same in 64 bits
def _double(cache):
    return cache[0].double() * cache[1].double()[..., None] if isinstance(cache, tuple) else cache.double()


def _codes(x):
    """int8 codes times their scale, in 64 bits, of the rows of x"""
    scale = (x.double().abs().amax(-1, keepdim=True) / 127).float().double()
    return torch.where(scale > 0, torch.round(x.double() / scale), torch.zeros_like(scale)) * scale, scale[..., 0]


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "attn":
        out = torch.zeros(c["B"], c["nkv"] * c["rep"], HD, dtype=torch.float64, device=DEV)
        kp, vp = (_double(_cut(x, c["plen"])) for x in (s["kc"], s["vc"]))
        slots = s["spos"].tolist()
        for b in range(c["B"]):
            m = slots[b] + 1
            if not c["plen"] + m:
                continue
            rows = s["src"][b, :m].long() if c["table"] else torch.full((m,), b, device=DEV)
            t = torch.arange(m, device=DEV)
            kb, vb = ((_double((x[0][rows, :, t], x[1][rows, :, t])) if c["s8"] else x[rows, :, t].double())
                      for x in (s["ks"], s["vs"]))
            for h in range(c["nkv"] * c["rep"]):
                j = h // c["rep"]
                k, v = torch.cat((kp[j], kb[:, j])), torch.cat((vp[j], vb[:, j]))
                a = torch.softmax((k * s["q"][b, h * HD:(h + 1) * HD].double()).sum(-1) / math.sqrt(HD), 0)
                out[b, h] = (a[:, None] * v).sum(0)
        return out.reshape(c["B"], -1)
    if c["op"] == "post":
        NH, dt = c["nkv"] * c["rep"], s["y"].dtype
        y = s["y"].double()
        heads = y[:, :(NH + 2 * c["nkv"]) * HD].reshape(c["B"], -1, HD).clone()
        if c["rope"]:
            at, n = c["plen"] + c["slot"], NH + c["nkv"]
            z = torch.complex(heads[:, :n, 0::2].contiguous(), heads[:, :n, 1::2].contiguous())
            z = z * torch.complex(s["cos"][at, 0::2].double(), s["sin"][at, 0::2].double())
            heads[:, :n] = torch.view_as_real(z).flatten(-2)
        gate, up = y[:, -2 * c["inter"]:].chunk(2, -1)
        out = {"q": heads[:, :NH].reshape(c["B"], -1), "act": gate * torch.sigmoid(gate) * up}
        for name, cache, x in (("k", s["ks"], heads[:, NH:NH + c["nkv"]]), ("v", s["vs"], heads[:, NH + c["nkv"]:])):
            out[name] = _double(cache)
            # an int8 cache holds the codes of the values that a plain one would hold
            out[name][:, :, c["slot"]] = _codes(x.to(dt))[0] if c["s8"] else x
        return out
    if c["op"] == "kv8":
        out = {}
        for name, x in (("k", s["kc"]), ("v", s["vc"])):
            back, scale = torch.zeros(x.shape, dtype=torch.float64, device=DEV), torch.zeros(x.shape[:-1], device=DEV).double()
            at = slice(c["t0"], c["t0"] + c["n"])
            back[:, at], scale[:, at] = _codes(x[:, at])
            out[name], out[name + "_scale"] = back, scale
        return out
    B, V, step = c["B"], c["V"], c["step"]
    x, score, done = s["logits"].double().cpu().numpy(), s["score"].double().cpu().numpy(), s["done"].cpu().numpy()
    if step < s["min_new"]:
        x[:, s["end"]] = -np.inf
    top = x.max(-1, keepdims=True)
    x = score[:, None] + x - (top + np.log(np.exp(x - top).sum(-1, keepdims=True)))
    x[done] = -np.inf
    x[done, s["end"]] = score[done]
    best = np.argsort(-x.reshape(-1), kind="stable")[:B]
    state = [torch.from_numpy(x.reshape(-1)[best])] + [None] * 5
    return {"tok": None, "parent": None, "state": state}
