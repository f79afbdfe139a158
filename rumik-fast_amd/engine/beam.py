"""Several hypotheses of one prompt decoded side by side on MI355X, as a beam search does: what stands between the
projections of such a step. The reference decodes one sequence (engine/rumik_fused.py:97-121); there post, the decode
attention and the sampler take one row, here B.

A layer's cache is in two parts: the prompt's (the prefix: kc / vc [NKV, S, 128], read once for all hypotheses) and one
per hypothesis (the suffix: ks / vs [B, NKV, T, 128], slot t the t-th new token). Each is a plain tensor in the
activations' type or an int8 pair (codes, scales) as in kv8. A step of B hypotheses, for every layer:

    y = mm_int4(h, *w_in)                                              # [B, q | k | v | gate | up]
    beam.post(y, spos, plen, cos, sin, ks, vs, q, act, NH=, NKV=, HD=, ROPE=)
    beam.attn(q, kc, vc, plen, ks, vs, spos, o, scale, src=search.src)
    ... mm_int4(o, *w_o), mm_int4(act, *w_down), add_ln over the rows

then the head, `search(logits)` and `fused.pos_advance(spos)`. (The head's product for B rows and, for best of n instead of
a search, the sampling are the caller's.) `plen` (the prompt's length) and `spos` (the newest
token's suffix slot, one for all or one each) are int64 on the device, so that one captured graph serves every step.
Reordering hypotheses moves no cache: pick permutes the table src, through which attn finds a hypothesis's slots in
the rows that wrote them.

Every call is asynchronous on the current torch stream and allocates at most its workspace (`ws=None`: from torch's
caching allocator per call, as mm_int4 does; calls that may overlap must not share one). There is no CPU path.
"""
import ctypes
import struct
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "kernels"))
import _hiplib as HL  # noqa: E402
import kv8  # noqa: E402

HD = 128
MAX_BEAMS = 32  # hypotheses that pick selects among

_p, _i = ctypes.c_void_p, ctypes.c_int
_INT = 2 ** 31 - 1  # the largest row stride that is passed as an int


class _AttnParams(ctypes.Structure):
    """rk_beam_attn_params"""
    _fields_ = ([(n, _p) for n in ("q", "o", "kc", "vc", "kc_scale", "vc_scale", "plen", "ks", "vs", "ks_scale",
                                   "vs_scale", "spos", "src", "ws")] +
                [("ws_bytes", ctypes.c_size_t), ("scale", ctypes.c_float)] +
                [(n, _i) for n in ("dt", "B", "NH", "NKV", "HD", "S", "T", "rows", "nspos", "src_ld")])


class _PickParams(ctypes.Structure):
    """rk_beam_pick_params"""
    _fields_ = ([(n, _p) for n in ("logits", "ids", "score", "done", "lens", "step", "hist", "src", "score_out",
                                   "done_out", "lens_out", "step_out", "hist_out", "src_out", "tok", "parent", "ws")] +
                [("ws_bytes", ctypes.c_size_t), ("ldl", ctypes.c_longlong)] +
                [(n, _i) for n in ("logits_dtype", "B", "V", "T", "end_idx", "min_new")])


def _packer(cls):
    """a struct of the class's fields packed in one call (setting ctypes fields one by one takes longer than a launch)"""
    codes = {_p: "P", _i: "i", ctypes.c_size_t: "N", ctypes.c_float: "f", ctypes.c_longlong: "q"}
    fmt = struct.Struct("@" + "".join(codes[t] for _, t in cls._fields_))
    assert fmt.size <= ctypes.sizeof(cls)
    tail = bytes(ctypes.sizeof(cls) - fmt.size)
    return lambda *values: fmt.pack(*values) + tail


_pack_attn, _pack_pick = _packer(_AttnParams), _packer(_PickParams)


def _need(ok, what="shape"):
    if not ok:
        raise RuntimeError(what)


def _typed(what, dtype, *ts):
    for t in ts:
        if t.dtype is not dtype or not t.is_contiguous():
            raise RuntimeError(f"{what}: contiguous {dtype} wanted, got {t.dtype}")


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _workspace(what, ws, nbytes, gpu):
    """(tensor, bytes): ws, or memory from torch's caching allocator, which is free for the stream's next calls afterwards"""
    if ws is None:
        return torch.empty(nbytes, dtype=torch.uint8, device=gpu), nbytes
    size = ws.numel() * ws.element_size()
    if not ws.is_contiguous() or ws.get_device() != gpu or size < nbytes:
        raise RuntimeError(f"{what}: the workspace is {nbytes} contiguous bytes on the tensors' GPU")
    return ws, size


def post(y, spos, plen, cos, sin, ks, vs, q, act, NH, NKV, HD, ROPE):
    """fused.post for B rows: row b of y [B, q | k | v | gate | up] at suffix slot spos[b], position plen + spos[b]:
    RoPE on q and k (ROPE), q -> q [B, NH * HD], k / v -> ks / vs [B, NKV, T, HD] (plain, or int8 pairs holding the codes
    of what a plain cache would hold), act [B, inter] = silu(gate) * up. y may have a row stride; spos int64 [1] or [B];
    plen int64 [1] or None (0); cos / sin [positions, HD] in y's type. A row without a slot or position gets act only."""
    _need(y.dim() == 2 and act.dim() == 2)
    dt = y.dtype
    kx, vx, kscale, vscale = kv8.pair(ks, vs, dt, "beam.post")
    (B, width), inter = y.shape, act.shape[-1]
    T = kx.shape[2] if kx.dim() == 4 else 0
    ns = spos.numel()
    ldy = y.stride(0) if B > 1 else width
    _need(kx.shape == (B, NKV, T, HD) and act.shape == (B, inter) and q.numel() == B * NH * HD and
          width == (NH + 2 * NKV) * HD + 2 * inter and width <= ldy <= _INT and (width == 1 or y.stride(1) == 1) and
          (ns == 1 or ns == B))
    _typed("beam.post", dt, q, act)
    _typed("beam.post", torch.int64, spos)
    if plen is not None:
        _need(plen.numel() == 1)
        _typed("beam.post", torch.int64, plen)
    P = 0
    if ROPE:
        _typed("beam.post", dt, cos, sin)
        P = cos.shape[0]
        _need(cos.shape == sin.shape == (P, HD))
    else:
        cos = sin = None
    gpu = HL.gpu_index("beam.post", y, spos, plen, cos, sin, kx, vx, kscale, vscale, q, act)
    HL.launch("beam.post", gpu, HL.lib().rk_beam_post, y.data_ptr(), ldy, spos.data_ptr(), ns, _ptr(plen), _ptr(cos),
              _ptr(sin), P, kx.data_ptr(), _ptr(kscale), vx.data_ptr(), _ptr(vscale), q.data_ptr(), act.data_ptr(),
              HL.dt(y), B, NH, NKV, HD, T, inter, 1 if ROPE else 0)


def attn(q, kc, vc, plen, ks, vs, spos, o, scale, src=None, ws=None):
    """Decode attention of B hypotheses: o [B, NH * 128] from q [B, NH * 128] over prefix slots [0, plen) of kc / vc
    [NKV, S, 128] and suffix slots t <= spos (its own, or the one) of ks / vs [rows, NKV, T, 128]; a hypothesis with no
    slot gets zeros. src int32 [B, >= T] (a row stride is taken): slot t of hypothesis b is slot t of row src[b, t], and
    none where that is outside [0, rows); None: row b. kc = vc = plen = None: no prefix, ks = vs = spos = None: no
    suffix. Either part is plain in q's type or int8 pairs. Returns o."""
    _need(q.dim() == 2)
    B, width = q.shape
    dt = q.dtype
    kx = vx = kxs = vxs = sx = wx = sxs = wxs = None
    NKV = S = T = rows = ns = ld = 0
    if kc is not None:
        kx, vx, kxs, vxs = kv8.pair(kc, vc, dt, "beam.attn prefix")
        _need(kx.dim() == 3 and plen is not None and plen.numel() == 1)
        _typed("beam.attn", torch.int64, plen)
        NKV, S, _ = kx.shape
    else:
        _need(ks is not None and vc is None)
        plen = None
    if ks is not None:
        sx, wx, sxs, wxs = kv8.pair(ks, vs, dt, "beam.attn suffix")
        _need(spos is not None)
        ns = spos.numel()
        _need(sx.dim() == 4 and (ns == 1 or ns == B) and (kc is None or sx.shape[1] == NKV))
        _typed("beam.attn", torch.int64, spos)
        rows, NKV, T, _ = sx.shape
        if src is not None:
            ld = src.stride(0) if B > 1 else src.shape[-1]
            _need(src.dim() == 2 and src.shape[0] == B and src.shape[1] >= T and src.stride(1) == 1 and T <= ld <= _INT)
            _need(src.dtype is torch.int32, "beam.attn: src is int32")
        else:
            _need(rows >= B)
    else:
        _need(vs is None)
        spos = src = None
    _need(o.numel() == B * width and NKV > 0 and width % (NKV * HD) == 0)
    _typed("beam.attn", dt, q, o)
    gpu = HL.gpu_index("beam.attn", q, kx, vx, kxs, vxs, plen, sx, wx, sxs, wxs, spos, src, o)
    lib, NH = HL.lib(), width // HD
    ws, nbytes = _workspace("beam.attn", ws, lib.rk_beam_attn_ws_bytes(B, NH, NKV, S, T), gpu)
    HL.launch("beam.attn", gpu, lib.rk_beam_attn, _pack_attn(
        q.data_ptr(), o.data_ptr(), _ptr(kx), _ptr(vx), _ptr(kxs), _ptr(vxs), _ptr(plen), _ptr(sx), _ptr(wx), _ptr(sxs),
        _ptr(wxs), _ptr(spos), _ptr(src), ws.data_ptr(), nbytes, scale, HL.dt(q), B, NH, NKV, HD, S, T, rows, ns, ld))
    return o


def _states(B, T, score, done, lens, step, hist, src):
    """the six state tensors' pointers, checked"""
    shape = (B, T)
    _need(score.numel() == B and done.numel() == B and lens.numel() == B and step.numel() == 1 and
          hist.shape == shape and src.shape == shape)
    _typed("beam.pick", torch.float32, score)
    _typed("beam.pick", torch.bool, done)
    _typed("beam.pick", torch.int64, lens, step, hist)
    _typed("beam.pick", torch.int32, src)
    return (score.data_ptr(), done.data_ptr(), lens.data_ptr(), step.data_ptr(), hist.data_ptr(), src.data_ptr())


def pick(logits, score, done, lens, step, hist, src, tok, parent, END_IDX, MIN_NEW=0, ids=None, out=None, ws=None):
    """A beam search's selection: the B best of score[b] + log softmax(logits[b])[v] over hypotheses and tokens (an ended
    hypothesis, done, competes with its own score) become the hypotheses, and their states are reordered.

    logits [B, V] fp16 / bf16 / fp32 (a row stride is taken), the end token END_IDX masked while step < MIN_NEW, NaN taken
    as -inf; score fp32 [B], done bool [B], lens int64 [B] (tokens, the end token among them), step int64 [1], hist
    int64 [B, T] (tokens), src int32 [B, T] (the suffix rows of their slots) -> out, the same six (None: in place);
    tok int64 [B] (ids[v], or v) and parent int32 [B]. Columns before `step` are those of the parents, column `step` the
    new token and the hypothesis's own row, step + 1. Equal values: the lower (hypothesis, token) first. With fewer than
    B candidates the others end at score -inf. At a step outside [0, T) nothing is written. B <= 32."""
    _need(logits.dim() == 2 and hist.dim() == 2)
    (B, V), (_, T) = logits.shape, hist.shape
    ldl = logits.stride(0) if B > 1 else V
    _need(1 <= B <= MAX_BEAMS and 0 <= END_IDX < V and T > 0 and ldl >= V and (V == 1 or logits.stride(1) == 1) and
          tok.numel() == B and parent.numel() == B)
    _typed("beam.pick", torch.int64, tok)
    _typed("beam.pick", torch.int32, parent)
    if ids is not None:
        _need(ids.numel() == V)
        _typed("beam.pick", torch.int64, ids)
    was = _states(B, T, score, done, lens, step, hist, src)
    if out is None:
        will = was
        gpu = HL.gpu_index("beam.pick", logits, ids, score, done, lens, step, hist, src, tok, parent)
    else:
        _need(len(out) == 6)
        will = _states(B, T, *out)
        gpu = HL.gpu_index("beam.pick", logits, ids, score, done, lens, step, hist, src, tok, parent, *out)
    lib = HL.lib()
    ws, nbytes = _workspace("beam.pick", ws, lib.rk_beam_pick_ws_bytes(B, V), gpu)
    HL.launch("beam.pick", gpu, lib.rk_beam_pick, _pack_pick(
        logits.data_ptr(), _ptr(ids), *was, *will, tok.data_ptr(), parent.data_ptr(), ws.data_ptr(), nbytes, ldl,
        HL.dt(logits), B, V, T, END_IDX, MIN_NEW))


class BeamSearch:
    """A search's states on the device (score, done, lens, step, hist, src, tok, parent) and its workspace; `__call__`
    picks from logits [B, len(audio_ids)] in place, as sample.FusedSampler samples for one sequence (but without its stop
    predictor: end_id alone ends a hypothesis). tok is the next step's input, hist[:, :step] the hypotheses' tokens, src
    what beam.attn takes, score the sum of log probabilities. hist and src have T columns, as the suffix caches have slots."""

    def __init__(self, B, T, audio_ids, end_id, min_new=0, device=None):
        dev = audio_ids.device if device is None else torch.device(device)
        _need(1 <= B <= MAX_BEAMS and T > 0)
        self.audio_ids = audio_ids.to(dev)
        ends = (self.audio_ids == end_id).nonzero().flatten().tolist()
        assert len(ends) == 1
        self.B, self.T, self.end_idx, self.min_new = B, T, ends[0], min_new
        self.score = torch.empty(B, dtype=torch.float32, device=dev)
        self.done = torch.empty(B, dtype=torch.bool, device=dev)
        self.lens = torch.empty(B, dtype=torch.int64, device=dev)
        self.step = torch.empty(1, dtype=torch.int64, device=dev)
        self.hist = torch.empty(B, T, dtype=torch.int64, device=dev)
        self.src = torch.empty(B, T, dtype=torch.int32, device=dev)
        self.tok = torch.empty(B, dtype=torch.int64, device=dev)
        self.parent = torch.empty(B, dtype=torch.int32, device=dev)
        nbytes = HL.lib().rk_beam_pick_ws_bytes(B, self.audio_ids.numel())
        self.ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        self.reset()

    def reset(self):
        """The start: one hypothesis, the empty one, with score 0; the others come from its first B tokens."""
        self.score.fill_(float("-inf"))
        self.score[:1].fill_(0)
        for t in (self.done, self.lens, self.step, self.hist, self.src, self.tok, self.parent):
            t.zero_()

    def __call__(self, logits):
        pick(logits, self.score, self.done, self.lens, self.step, self.hist, self.src, self.tok, self.parent,
             self.end_idx, self.min_new, ids=self.audio_ids, ws=self.ws)
        return self.tok
