"""Rotary positions with the append to a paged cache, attention over packed sequences, and attention of
new tokens over a paged cache, each against its formula in 64 bits.

Tolerances, per element, from the roundings alone (eps = finfo(dtype).eps, half a step is eps / 2):

* rotary: the result is rounded once, eps / 2 |y|.  Before that, in fp32: the angle (relative 2^-24 of at most
  pi, so pi 2^-24), cos and sin (a few 2^-24), two products and a sum: less than 16 * 2^-24 = 2^-20 of
  amplitude (|x1| + |x2|).  fp16 results below 2^-14 are rounded to steps of 2^-24: half a step more.
* attention: o = sum p v / sum p is rounded once, eps / 2 |o|.  Each weight is rounded to dtype once, eps / 2
  of p |v|, and may be missing from the sum of the weights in its rounded form, eps / 2 again: eps A with
  A = sum p |v| / sum p.  A score's fp32 sum over head_dim products is off by at most head_dim 2^-24 S,
  S = scale * sum |q| |k|, and its scaling and exponential by a few 2^-24 of |s| <= S more; that enters p
  and sum p: 2 (head_dim + 8) 2^-24 S A.  Sums over n keys in fp32: n 2^-24 each, 2 n 2^-24 A.  An fp16 weight
  below 2^-14 of the row's largest is rounded to steps of 2^-24: 2^-25 |v| over sum exp(s - max) for each key.
"""

import math

import pytest
import torch

from transformer_optimization_amd import _C
from _util import log

DTYPES = [torch.bfloat16, torch.float16]
gpu = pytest.mark.gpu


def _gen(seed):
    return torch.Generator("cpu").manual_seed(seed)


def _randn(shape, dtype, dev, seed, scale=1.0):
    return (torch.randn(shape, generator=_gen(seed)) * scale).to(dev, dtype)


def _cu(lens, dev, first=0):
    at = [first]
    for n in lens:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=dev)


def _i32(xs, dev):
    return torch.tensor(xs, dtype=torch.int32, device=dev)


# ------------------------------------------------------------------- oracle
def _attend(q, k, v, scale, causal, dtype):
    """64-bit attention of q [n, H, d] over k, v [m, Hk, d], rows aligned at the last key; masked keys are left
    out, not multiplied by 0.  Returns the result and its tolerance."""
    n, h, d = q.shape
    m, hk = k.shape[:2]
    out = torch.zeros(n, h, d, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    eps = torch.finfo(dtype).eps
    for x in range(h):
        qx, kx, vx = q[:, x].double(), k[:, x // (h // hk)].double(), v[:, x // (h // hk)].double()
        s = (qx @ kx.T) * scale
        size = (qx.abs() @ kx.abs().T) * scale
        seen = torch.ones(n, m, dtype=torch.bool, device=q.device)
        if causal:
            seen = seen.tril(m - n)
        s = s.masked_fill(~seen, -math.inf)
        some = seen.any(1)
        top = s.amax(1, keepdim=True) if m else s.new_zeros(n, 1)
        p = torch.where(some[:, None], torch.exp(s - top), torch.zeros_like(s))
        p = torch.where(seen, p, torch.zeros_like(p))
        w = p / torch.where(some, p.sum(1), torch.ones_like(top[:, 0]))[:, None]
        bad = ~torch.isfinite(vx)
        clean = vx.masked_fill(bad, 0.0)
        o = w @ clean
        # what is not finite reaches the rows that see it, and no others
        reach = (seen.double() @ bad.double()) > 0
        o = torch.where(reach, torch.full_like(o, math.nan), o)
        a = w @ clean.abs()
        big = size.masked_fill(~seen, 0.0).amax(1, keepdim=True) if m else s.new_zeros(n, 1)
        out[:, x] = o
        if dtype == torch.float16 and m:
            total = torch.where(some, p.sum(1), torch.ones_like(top[:, 0]))[:, None]
            a = a + 2.0**-25 / eps * (seen.double() @ clean.abs()) / total
        tol[:, x] = eps / 2 * o.abs() + a * (eps + 2 * (d + 8) * 2.0**-24 * big + 2 * m * 2.0**-24) + 2.0**-25
    return out, tol


def _same(got, want, tol, what):
    """Every element within its tolerance; where the formula is not finite, the result is not finite."""
    got, g = got.double(), ~torch.isfinite(got)
    w = ~torch.isfinite(want)
    assert torch.equal(g, w), f"{what}: {int((g ^ w).sum())} elements finite on one side only"
    d = torch.where(w, torch.zeros_like(want), (got - want).abs())
    over = torch.where(w, torch.zeros_like(want), d - tol)
    log(f"  {what}: max error {float(d.max()) if d.numel() else 0:.3e}, share of tolerance "
        f"{float((d / tol).nan_to_num().max()) if d.numel() else 0:.3f}")
    assert not d.numel() or float(over.max()) <= 0, what


def _paged(lens, kv_heads, page, hd, dtype, dev, seed, token_major=False, spare=3, fill=math.nan, width=None):
    """Keys and values of each sequence, and caches that hold them in shuffled pages.  Slots of no key hold
    `fill`; unused table entries point outside the pool."""
    counts = [(n + page - 1) // page for n in lens]
    pages = sum(counts) + spare
    order = torch.randperm(pages, generator=_gen(seed)).to(torch.int32)
    width = width or max(max(counts), 1)
    table = torch.full((len(lens), width), -7, dtype=torch.int32)
    table[:, 1::2] = 2**31 - 1
    shape = (pages, page, kv_heads, hd) if token_major else (pages, kv_heads, page, hd)
    caches = [torch.full(shape, fill, dtype=dtype) for _ in range(2)]
    views = [c.transpose(1, 2) if token_major else c for c in caches]
    ks, vs, at = [], [], 0
    for b, n in enumerate(lens):
        kv = [torch.randn(n, kv_heads, hd, generator=_gen(seed + 10 * b + i)).to(dtype) for i in (1, 2)]
        table[b, :counts[b]] = order[at:at + counts[b]]
        at += counts[b]
        for c, x in zip(views, kv):
            for i in range(counts[b]):
                part = x[i * page:(i + 1) * page]
                c[int(table[b, i]), :, :part.shape[0]] = part.transpose(0, 1)
        ks.append(kv[0].to(dev))
        vs.append(kv[1].to(dev))
    caches = [c.to(dev) for c in caches]
    views = [c.transpose(1, 2) if token_major else c for c in caches]
    return ks, vs, views[0], views[1], table.to(dev)


# ------------------------------------------------------------ steps (CPU)
@pytest.mark.parametrize("scaling", _C.ROTARY_SCALINGS)
@pytest.mark.parametrize("rotary,base", [(64, 10000.0), (128, 500000.0), (20, 10000.0)])
def test_rotary_steps_are_the_frequencies_in_turns(scaling, rotary, base):
    steps, amplitude = _C.rotary_steps(rotary, base, scaling=scaling, factor=8.0, original_len=4096)
    assert steps.dtype == torch.int64 and steps.shape == (rotary // 2,)
    assert amplitude == (pytest.approx(0.1 * math.log(8.0) + 1) if scaling == "ramp" else 1.0)
    plain = [base ** (-2 * i / rotary) for i in range(rotary // 2)]
    for i, (f, s) in enumerate(zip(plain, steps.tolist())):
        if scaling == "linear":
            f /= 8.0
        elif scaling == "base":
            f = (base * 8.0 ** (rotary / (rotary - 2))) ** (-2 * i / rotary)
        elif scaling == "ramp":
            turns = 4096 * f / (2 * math.pi)
            w = min(max((turns - 1) / 31, 0.0), 1.0)
            f = f * (w + (1 - w) / 8)
        assert s / 2.0**64 * 2 * math.pi == pytest.approx(f, rel=1e-13)


def test_rotary_steps_keep_only_the_fraction_of_a_turn():
    steps, _ = _C.rotary_steps(4, 0.01)  # frequencies 1 and 10 rad: 0.159 and 1.59 turns
    assert steps[1] / 2.0**64 == pytest.approx(10 / (2 * math.pi) - 2, rel=1e-12)


def test_rotary_steps_refusals():
    for kw in (dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=64, base=0.0), dict(rotary_dim=64, scaling="x"),
               dict(rotary_dim=64, factor=0.0), dict(rotary_dim=64, scaling="ramp"), dict(rotary_dim=2, scaling="base"),
               dict(rotary_dim=64, base=math.inf), dict(rotary_dim=64, scaling="ramp", original_len=8, low_turns=9.0,
                                                        high_turns=9.0)):
        with pytest.raises(ValueError):
            _C.rotary_steps(**{"base": 10000.0, **kw})


# -------------------------------------------------------- refusals (CPU)
FAKE = 1 << 20  # never dereferenced: validation comes first


class _Abi:
    """The C entry points on made-up addresses, one argument changed at a time."""

    def __init__(self):
        import ctypes
        self.lib, self.ct, self.keep = _C.load_library(), ctypes, []

    def st(self, *v):
        if v[0] is None:
            return None
        a = (self.ct.c_int64 * len(v))(*v)
        self.keep.append(a)
        return self.ct.addressof(a)

    def rotary(self, **kw):
        a = dict(q=FAKE, qs=(512, 64), qo=1 << 30, qos=(512, 64), k=1 << 31, ks=(128, 64), ko=None, kos=(128, 64),
                 v=3 << 30, vs=(128, 64), kc=1 << 33, kcs=(2048, 1024, 64), vc=1 << 34, vcs=(2048, 1024, 64), steps=FAKE,
                 pos=None, cu=FAKE, kvl=FAKE, table=FAKE, ld=8, t=64, b=2, h=8, hk=2, hd=64, r=64, np=32, ps=16, mp=8,
                 amp=1.0, dt=_C.TX_BF16)
        a.update(kw)
        return self.lib.tx_rotary_append(
            a["q"], self.st(*a["qs"]), a["qo"], self.st(*a["qos"]), a["k"], self.st(*a["ks"]), a["ko"], self.st(*a["kos"]),
            a["v"], self.st(*a["vs"]), a["kc"], self.st(*a["kcs"]), a["vc"], self.st(*a["vcs"]), a["steps"], a["pos"],
            a["cu"], a["kvl"], a["table"], a["ld"], a["t"], a["b"], a["h"], a["hk"], a["hd"], a["r"], a["np"], a["ps"],
            a["mp"], a["amp"], 0, a["dt"], None)

    def packed(self, **kw):
        a = dict(q=FAKE, qs=(512, 64), k=1 << 30, ks=(128, 64), v=1 << 31, vs=(128, 64), o=3 << 30, os=(512, 64), cu=FAKE,
                 t=64, b=2, h=8, hk=2, hd=64, scale=0.125, dt=_C.TX_BF16)
        a.update(kw)
        return self.lib.tx_flash_attn_packed(
            a["q"], self.st(*a["qs"]), a["k"], self.st(*a["ks"]), a["v"], self.st(*a["vs"]), a["o"], self.st(*a["os"]),
            a["cu"], a["t"], a["b"], a["h"], a["hk"], a["hd"], a["scale"], 1, a["dt"], None)

    def paged(self, **kw):
        a = dict(q=FAKE, qs=(512, 64), kc=1 << 33, kcs=(2048, 1024, 64), vc=1 << 34, vcs=(2048, 1024, 64), o=3 << 30,
                 os=(512, 64), cu=FAKE, kvl=FAKE, table=FAKE, ld=8, t=64, b=2, h=8, hk=2, hd=64, np=32, ps=16, mp=8, mq=0,
                 scale=0.125, ws=1 << 35, wsn=1 << 40, dt=_C.TX_BF16)
        a.update(kw)
        return self.lib.tx_flash_attn_paged(
            a["q"], self.st(*a["qs"]), a["kc"], self.st(*a["kcs"]), a["vc"], self.st(*a["vcs"]), a["o"], self.st(*a["os"]),
            a["cu"], a["kvl"], a["table"], a["ld"], a["t"], a["b"], a["h"], a["hk"], a["hd"], a["np"], a["ps"], a["mp"],
            a["mq"], a["scale"], 1, a["ws"], a["wsn"], a["dt"], None)


E, U = _C.TX_EINVAL, _C.TX_EUNSUPPORTED
SEQ_REFUSALS = [  # of every entry point
    (dict(q=None), E), (dict(cu=None), E), (dict(t=0), E), (dict(b=0), E), (dict(h=0), E), (dict(hk=0), E),
    (dict(hk=3), E), (dict(hd=0), E), (dict(dt=_C.TX_F32), U), (dict(q=FAKE + 2), U), (dict(qs=(516, 64)), U),
    (dict(qs=(512, -64)), E), (dict(t=1 << 25), U), (dict(h=1 << 16, hk=1 << 15), U), (dict(t=1 << 24, h=16), U),
    (dict(b=1 << 21), U), (dict(cu=FAKE + 1), U), (dict(t=64, h=1 << 14, hk=1 << 14, b=1 << 10), U),
]
PAGE_REFUSALS = [
    (dict(table=None), E), (dict(kvl=None), E), (dict(np=0), E), (dict(mp=0), E), (dict(ps=0), E), (dict(ps=4), U),
    (dict(ps=24), U), (dict(ps=1 << 16), U), (dict(ld=7), E), (dict(mp=1 << 27, ld=1 << 27), U), (dict(table=FAKE + 2), U),
    (dict(kcs=(2048, 1024, 60)), U), (dict(kcs=(1 << 31, 1024, 64)), U), (dict(vcs=(1 << 30, 1024, 1 << 24)), U), (dict(kcs=(2048, 1024, -64)), E), (dict(vcs=(2048, 512, 64)), E),
    (dict(kcs=(1024, 1024, 64)), E), (dict(kc=(1 << 33) + 8), U), (dict(vc=None), E),
]


@pytest.mark.parametrize("change,code", SEQ_REFUSALS + PAGE_REFUSALS + [
    (dict(steps=None), E), (dict(k=None), E), (dict(r=0), E), (dict(r=7), E), (dict(r=66), E), (dict(qo=None), E),
    (dict(hd=260, r=64), U), (dict(hd=512, r=64), U), (dict(amp=0.0), E), (dict(amp=math.nan), E), (dict(v=None), E),
    (dict(kc=None, vc=None), E),                                  # neither k_out nor a cache
    (dict(qo=FAKE + 1024), E), (dict(qo=FAKE, qos=(1024, 64)), E),  # over q, but not q itself
    (dict(qo=1 << 31), E),                                         # over k
    (dict(ko=FAKE), E), (dict(kc=1 << 31), E), (dict(vc=(1 << 33) + 1024), E), (dict(qos=(512, 0)), E),
    (dict(kos=(64, 64), ko=1 << 36), E), (dict(pos=FAKE + 4), U), (dict(steps=FAKE + 4), U),
])
def test_rotary_append_refusals(change, code):
    assert _Abi().rotary(**change) == code


@pytest.mark.parametrize("change,code", SEQ_REFUSALS + [
    (dict(k=None), E), (dict(v=None), E), (dict(o=None), E), (dict(hd=96), U), (dict(scale=0.0), E),
    (dict(scale=math.nan), E), (dict(scale=math.inf), E), (dict(os=(512, 32)), E), (dict(os=(256, 64)), E),
    (dict(o=FAKE), E), (dict(o=(1 << 30) + 128), E), (dict(o=1 << 31), E), (dict(ks=(1 << 24, 64)), U),
    (dict(vs=(1 << 24, 64)), U), (dict(o=(3 << 30) + 8), U),
])
def test_packed_attention_refusals(change, code):
    assert _Abi().packed(**change) == code


@pytest.mark.parametrize("change,code", SEQ_REFUSALS + PAGE_REFUSALS + [
    (dict(kc=None), E), (dict(o=None), E), (dict(hd=96), U), (dict(scale=-1.0), E), (dict(o=1 << 33), E),
    (dict(o=(1 << 34) + 256), E), (dict(o=FAKE + 16), E), (dict(os=(512, 8)), E), (dict(kvl=FAKE + 2), U),
])
def test_paged_attention_refusals(change, code):
    assert _Abi().paged(**change) == code


def test_paged_workspace_refusals():
    for bad in ((0, 1, 8, 2, 64, 16, 8), (1, 0, 8, 2, 64, 16, 8), (1, 1, 8, 3, 64, 16, 8), (1, 1, 8, 2, 96, 16, 8),
                (1, 1, 8, 2, 64, 12, 8), (1, 1, 8, 2, 64, 16, 0)):
        with pytest.raises(_C.TxError):
            _C.flash_attn_paged_workspace(*bad)
    assert _C.flash_attn_paged_workspace(4, 4, 8, 2, 64, 16, 8) >= 0


def _cpu_args():
    bf = torch.bfloat16
    return dict(q=torch.zeros(6, 8, 64, dtype=bf), k=torch.zeros(6, 2, 64, dtype=bf), v=torch.zeros(6, 2, 64, dtype=bf),
                kc=torch.zeros(5, 2, 16, 64, dtype=bf), vc=torch.zeros(5, 2, 16, 64, dtype=bf),
                table=torch.zeros(2, 3, dtype=torch.int32), cu=_i32([0, 2, 6], "cpu"), kvl=_i32([2, 4], "cpu"),
                steps=torch.zeros(32, dtype=torch.int64))


def test_wrappers_check_their_arguments_before_the_device():
    a = _cpu_args()
    with pytest.raises(ValueError, match="GPU tensors"):
        _C.flash_attn_packed(a["q"], a["k"], a["v"], a["cu"], 0.1, True)
    with pytest.raises(ValueError, match="GPU tensors"):
        _C.flash_attn_paged(a["q"], a["kc"], a["vc"], a["table"], a["cu"], a["kvl"], 0.1)
    with pytest.raises(ValueError, match="GPU tensors"):
        _C.rotary_append(a["q"], a["k"], a["v"], a["steps"], a["cu"])
    for bad, what in ((dict(q=a["q"][0]), r"q must be"), (dict(k=a["k"][:5]), "k must be"), (dict(k=a["k"].float()), "dtype"),
                      (dict(k=torch.zeros(6, 3, 64, dtype=torch.bfloat16)), "v must be"),
                      (dict(k=torch.zeros(6, 3, 64, dtype=torch.bfloat16), v=torch.zeros(6, 3, 64, dtype=torch.bfloat16)), "divide"),
                      (dict(cu=a["cu"].long()), "cu_seqlens"), (dict(cu=a["cu"][::2]), "cu_seqlens"),
                      (dict(q=a["q"].transpose(0, 2).contiguous().transpose(0, 2)), "contiguous in head_dim")):
        b = {**a, **bad}
        with pytest.raises(ValueError, match=what):
            _C.flash_attn_packed(b["q"], b["k"], b["v"], b["cu"], 0.1, True)
    for bad, what in ((dict(kc=a["kc"][0]), "k_cache"), (dict(vc=a["vc"][:4]), "k_cache"), (dict(kc=a["kc"].half()), "dtype"),
                      (dict(table=a["table"][:1]), "block_table"), (dict(table=a["table"].long()), "block_table"),
                      (dict(kvl=a["kvl"][:1]), "kv_lens"), (dict(kvl=a["kvl"].long()), "kv_lens"),
                      (dict(table=torch.zeros(3, 2, dtype=torch.int32).T), "rows must be contiguous")):
        b = {**a, **bad}
        with pytest.raises(ValueError, match=what):
            _C.flash_attn_paged(b["q"], b["kc"], b["vc"], b["table"], b["cu"], b["kvl"], 0.1)
        b["vc"] = b["vc"] if "kc" not in bad else a["vc"]
        with pytest.raises(ValueError, match=what):
            _C.rotary_append(b["q"], b["k"], b["v"], b["steps"], b["cu"], kv_lens=b["kvl"], block_table=b["table"],
                             k_cache=b["kc"], v_cache=b["vc"])
    for kw, what in ((dict(k_cache=a["kc"]), "a cache needs"), (dict(positions=torch.zeros(6, dtype=torch.int32)), "positions"),
                     (dict(q_out=a["q"][:5]), "q_out"), (dict(k_out=a["q"]), "k_out")):
        with pytest.raises(ValueError, match=what):
            _C.rotary_append(a["q"], a["k"], a["v"], a["steps"], a["cu"], **kw)
    with pytest.raises(ValueError, match="steps"):
        _C.rotary_append(a["q"], a["k"], a["v"], torch.zeros(33, dtype=torch.int64), a["cu"])
    with pytest.raises(ValueError, match="q_out without q"):
        _C.rotary_append(None, a["k"], a["v"], a["steps"], a["cu"], q_out=a["q"])


# ------------------------------------------------------------------ rotary
def _rotate(x, positions, steps, amplitude, interleaved, dtype):
    """The formula in 64 bits (angles from the integer steps), and its tolerance."""
    r = 2 * steps.shape[0]
    turns = torch.tensor([[((int(p) * int(s) + 2**63) % 2**64 - 2**63) / 2.0**64 for s in steps] for p in positions],
                         dtype=torch.float64, device=x.device).view(len(positions), 1, r // 2)
    c, s = torch.cos(2 * math.pi * turns) * amplitude, torch.sin(2 * math.pi * turns) * amplitude
    y, size = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    i1, i2 = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = x[..., i1].double(), x[..., i2].double()
    y[..., i1], y[..., i2] = a * c - b * s, b * c + a * s
    size[..., i1] = size[..., i2] = (a.abs() + b.abs()) * amplitude
    eps = torch.finfo(dtype).eps
    return y, eps / 2 * y.abs() + 2.0**-20 * size + (2.0**-25) * (size > 0)


ROTARY_CASES = [  # head dim, rotary, interleaved, q heads, kv heads, page, token-major cache
    (64, 64, False, 8, 8, 16, False), (64, 64, True, 8, 2, 8, True), (128, 128, False, 16, 4, 64, True),
    (128, 64, True, 4, 1, 32, False), (128, 96, False, 5, 5, 16, False), (64, 20, False, 6, 3, 8, False),
    (64, 20, True, 6, 3, 16, True), (8, 2, False, 1, 1, 8, False), (256, 256, True, 2, 1, 128, False),
    (120, 48, False, 3, 1, 16, False),
]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd,rotary,interleaved,h,hk,page,token_major", ROTARY_CASES)
def test_rotary_append(cuda, dtype, hd, rotary, interleaved, h, hk, page, token_major):
    log(f"rotary hd{hd} r{rotary} interleaved={interleaved} {h}/{hk} heads page {page} {dtype}")
    lens, new = [1, 37, 5, 64, 9], [1, 30, 0, 64, 4]
    rows, first, behind = sum(new), 2, 3
    t = first + rows + behind
    _, _, kc, vc, table = _paged(lens, hk, page, hd, dtype, cuda, 5, token_major, fill=7.0)
    kc0, vc0 = kc.clone(), vc.clone()
    qkv = _randn((t, h + 2 * hk, hd), dtype, cuda, 1)
    q, k, v = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
    steps, amplitude = _C.rotary_steps(rotary, scaling="ramp", factor=4.0, original_len=64, device=cuda)
    out = torch.full((t, h, hd), 3.0, dtype=dtype, device=cuda)
    k_out = torch.full((t, hk, hd), 3.0, dtype=dtype, device=cuda)
    cu, kvl = _cu(new, cuda, first), _i32(lens, cuda)
    got = _C.rotary_append(q, k, v, steps, cu, kv_lens=kvl, block_table=table, k_cache=kc, v_cache=vc, q_out=out,
                           k_out=k_out, interleaved=interleaved, amplitude=amplitude)
    assert got[0] is out and got[1] is k_out
    at = [list(range(n - m, n)) for n, m in zip(lens, new)]
    flat = [p for ps in at for p in ps]
    inner = slice(first, first + rows)
    for name, x, y in (("q", q, out), ("k", k, k_out)):
        want, tol = _rotate(x[inner], flat, steps.cpu(), amplitude, interleaved, dtype)
        _same(y[inner], want, tol, name)
        assert torch.equal(y[inner][..., rotary:], x[inner][..., rotary:])
        assert bool((y[:first] == 3).all()) and bool((y[first + rows:] == 3).all())
    row = first
    for b, ps in enumerate(at):
        for p in ps:
            pg = int(table[b, p // page])
            kc0[pg, :, p % page], vc0[pg, :, p % page] = k_out[row], v[row]
            row += 1
    assert torch.equal(kc, kc0) and torch.equal(vc, vc0)


@gpu
@pytest.mark.parametrize("interleaved,rotary", [(False, 64), (True, 64), (False, 20), (True, 20)])
def test_rotary_in_place_without_cache_and_far_positions(cuda, interleaved, rotary):
    dtype, new = torch.float16, [70, 1, 12]
    t = sum(new)
    steps, _ = _C.rotary_steps(rotary, device=cuda)
    buf = _randn((t, 10, 64), dtype, cuda, 3)
    q, k = buf[:, :8], buf[:, 8:]
    q0, k0 = q.clone(), k.clone()
    positions = torch.randint(-(10**6), 10**9, (t,), generator=_gen(4))
    positions[:3] = torch.tensor([0, 2**40 + 1, -(2**62)])
    got = _C.rotary_append(q, k, None, steps, _cu(new, cuda), positions=positions.to(cuda), q_out=q, k_out=k,
                           interleaved=interleaved)
    assert got[0].data_ptr() == q.data_ptr() and got[1].data_ptr() == k.data_ptr()
    for name, x0, x in (("q", q0, q), ("k", k0, k)):
        want, tol = _rotate(x0, positions.tolist(), steps.cpu(), 1.0, interleaved, dtype)
        _same(x, want, tol, name)
    # positions by default: 0, 1, .. of each sequence; keys alone
    _, k2 = _C.rotary_append(None, k0, None, steps, _cu(new, cuda), interleaved=interleaved)
    want, tol = _rotate(k0, [i for n in new for i in range(n)], steps.cpu(), 1.0, interleaved, dtype)
    _same(k2, want, tol, "k alone")


@gpu
def test_rotary_append_drops_what_has_no_place(cuda):
    """Rows before key 0, in pages outside the pool or behind the table are turned but not cached; nothing
    else of the cache changes."""
    dtype, page, hk = torch.bfloat16, 8, 2
    kc = torch.zeros(4, hk, page, 64, dtype=dtype, device=cuda)
    vc = torch.zeros_like(kc)
    table = _i32([[2, -1], [4, 1], [2**31 - 1, 3]], cuda)
    new, lens = [10, 12, 6], [7, 12, 19]  # 3 rows before key 0; page 4 of 4; keys 13..18, 16.. behind the table
    x = _randn((sum(new), 3 * hk, 64), dtype, cuda, 6) + 1.5
    steps, _ = _C.rotary_steps(64, device=cuda)
    q, _ = _C.rotary_append(x[:, :hk], x[:, hk:2 * hk], x[:, 2 * hk:], steps, _cu(new, cuda), kv_lens=_i32(lens, cuda),
                            block_table=table, k_cache=kc, v_cache=vc)
    pos = [i for n, m in zip(lens, new) for i in range(n - m, n)]
    want, tol = _rotate(x[:, :hk], pos, steps.cpu(), 1.0, False, dtype)
    _same(q, want, tol, "q")
    expect = torch.zeros_like(vc)
    row = 0
    for b, (n, m) in enumerate(zip(lens, new)):
        for p in range(n - m, n):
            pg = int(table[b, p // page]) if 0 <= p < 2 * page else -1
            if 0 <= pg < 4:
                expect[pg, :, p % page] = x[row, 2 * hk:]
            row += 1
    assert torch.equal(vc, expect)
    assert torch.equal((kc != 0).any(-1), (expect != 0).any(-1))  # the same slots hold keys (an element may be 0)


# ------------------------------------------------------------------ packed
PACKED_LENS = [[1], [0, 1, 0, 5, 0], [63, 64, 65], [130, 1, 300, 0, 2], [1000, 7, 129], [2, 513, 128, 31]]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("h,hk", [(8, 8), (8, 2), (6, 2), (5, 1), (16, 1)])
@pytest.mark.parametrize("causal", [False, True])
def test_packed_attention(cuda, dtype, hd, h, hk, causal):
    for lens in PACKED_LENS:
        log(f"packed {lens} hd{hd} heads {h}/{hk} causal={causal} {dtype}")
        first, behind = 3, 4
        t = first + sum(lens) + behind
        qkv = _randn((t, h + 2 * hk, hd), dtype, cuda, 11)
        qkv[:first], qkv[t - behind:] = math.nan, math.nan  # rows of no sequence
        q, k, v = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
        out = torch.full((t, h, hd), 3.0, dtype=dtype, device=cuda)
        got = _C.flash_attn_packed(q, k, v, _cu(lens, cuda, first), hd**-0.5, causal, out=out)
        assert got is out
        at = first
        for b, n in enumerate(lens):
            s = slice(at, at + n)
            want, tol = _attend(q[s], k[s], v[s], hd**-0.5, causal, dtype)
            _same(out[s], want, tol, f"sequence {b}")
            at += n
        assert bool((out[:first] == 3).all()) and bool((out[t - behind:] == 3).all())


@gpu
@pytest.mark.parametrize("hd,causal", [(64, True), (128, False)])
def test_packed_attention_heads_apart_and_large_scores(cuda, hd, causal):
    """Separate head-major tensors, an output with gaps, and scores far apart (a row's weight on few keys)."""
    dtype, n, h, hk = torch.bfloat16, 200, 4, 2
    q = _randn((h, n, hd), dtype, cuda, 21, 4.0).transpose(0, 1)
    k = _randn((hk, n, hd), dtype, cuda, 22, 4.0).transpose(0, 1)
    v = _randn((hk, n, hd), dtype, cuda, 23).transpose(0, 1)
    wide = torch.zeros(n, h + 1, hd, dtype=dtype, device=cuda)
    _C.flash_attn_packed(q, k, v, _cu([77, 123], cuda), 1.0, causal, out=wide[:, :h])
    for s in (slice(0, 77), slice(77, 200)):
        want, tol = _attend(q[s], k[s], v[s], 1.0, causal, dtype)
        _same(wide[s, :h], want, tol, "rows")
    assert bool((wide[:, h] == 0).all())


@gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("paged", [False, True])
def test_what_a_mask_hides_has_no_influence(cuda, hd, paged):
    """NaN and infinities in keys and values that come after a row."""
    dtype, n, h, hk = torch.float16, 150, 4, 2
    q, k, v = (_randn((n, x, hd), dtype, cuda, 30 + i) for i, x in enumerate((h, hk, hk)))
    for j, x in ((10, math.nan), (70, math.inf), (100, -math.inf), (149, math.nan)):
        k[j, 0, 5] = x
    for j, x in ((20, math.inf), (64, math.nan), (149, -math.inf)):
        v[j, 1, 7] = x
    if paged:
        _, _, kc, vc, table = _paged([n], hk, 16, hd, dtype, cuda, 33)
        for j in range(n):
            kc[table[0, j // 16].long(), :, j % 16], vc[table[0, j // 16].long(), :, j % 16] = k[j], v[j]
        got = _C.flash_attn_paged(q, kc, vc, table, _cu([n], cuda), _i32([n], cuda), hd**-0.5)
    else:
        got = _C.flash_attn_packed(q, k, v, _cu([n], cuda), hd**-0.5, True)
    # heads of K/V head 0 see the bad keys: finite up to key 9, then NaN or a finite choice of +inf / -inf scores
    clean_k = k.clone()
    clean_k[:, 0, 5] = torch.where(torch.isfinite(k[:, 0, 5]), k[:, 0, 5], torch.zeros_like(k[:, 0, 5]))
    want, tol = _attend(q, clean_k, v, hd**-0.5, True, dtype)
    _same(got[:10, :2], want[:10, :2], tol[:10, :2], "before the first bad key")
    assert bool(torch.isnan(got[10:, :2]).all())
    # of K/V head 1 only element 7 of the rows that see a bad value
    d = [i for i in range(hd) if i != 7]
    _same(got[:, 2:][..., d], want[:, 2:][..., d], tol[:, 2:][..., d], "other elements")
    _same(got[:20, 2:, 7], want[:20, 2:, 7], tol[:20, 2:, 7], "element 7 before")
    assert bool((got[20:64, 2:, 7] == math.inf).all()) and bool(torch.isnan(got[64:, 2:, 7]).all())


@gpu
@pytest.mark.parametrize("hd", [64, 128])
def test_rows_whose_scores_are_all_minus_infinity_are_nan(cuda, hd):
    """As torch.softmax gives, and as the other attention entry points do; rows without keys are 0."""
    dtype, big = torch.bfloat16, 3.0e38
    q = torch.full((3, 2, hd), big, dtype=dtype, device=cuda)
    k = torch.full((3, 2, hd), -big, dtype=dtype, device=cuda)
    v = _randn((3, 2, hd), dtype, cuda, 2)
    assert bool(torch.isnan(_C.flash_attn_packed(q, k, v, _cu([3], cuda), 1.0, True)).all())
    kc = k.transpose(0, 1).repeat(1, 3, 1)[None, :, :8].contiguous()
    vc = torch.zeros_like(kc)
    got = _C.flash_attn_paged(q, kc, vc, _i32([[0]], cuda), _cu([3], cuda), _i32([2], cuda), 1.0)
    assert bool((got[0] == 0).all()) and bool(torch.isnan(got[1:]).all())


# ------------------------------------------------------------------- paged
PAGED_CASES = [  # new tokens, keys of each sequence
    ([1], [1]), ([1], [513]), ([1, 1, 1, 1], [1, 64, 65, 1000]), ([1, 0, 1, 2, 1], [0, 5, 33, 2, 128]),
    ([3, 1, 5], [200, 31, 5]), ([17, 1], [17, 2100]), ([130, 1, 40, 64], [700, 90, 40, 1025]), ([9, 4], [3, 0]),
]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("h,hk", [(8, 8), (8, 2), (6, 2), (5, 1), (16, 1), (24, 1)])
@pytest.mark.parametrize("page,token_major", [(16, False), (8, True), (64, True), (256, False)])
def test_paged_attention(cuda, dtype, hd, h, hk, page, token_major):
    for i, (new, lens) in enumerate(PAGED_CASES):
        causal = i % 3 != 2
        log(f"paged {new} over {lens} hd{hd} heads {h}/{hk} page {page} causal={causal} {dtype}")
        ks, vs, kc, vc, table = _paged(lens, hk, page, hd, dtype, cuda, 40 + i, token_major)
        first, behind = 1, 2
        t = first + sum(new) + behind
        q = _randn((t, h, hd), dtype, cuda, 50 + i)
        out = torch.full_like(q, 3.0)
        _C.flash_attn_paged(q, kc, vc, table, _cu(new, cuda, first), _i32(lens, cuda), hd**-0.5, causal, out=out,
                            max_q_len=max(new) if i % 2 else 0)
        at = first
        for b, n in enumerate(new):
            s = slice(at, at + n)
            want, tol = _attend(q[s], ks[b], vs[b], hd**-0.5, causal, dtype)
            _same(out[s], want, tol, f"sequence {b}")
            at += n
        assert bool((out[:first] == 3).all()) and bool((out[t - behind:] == 3).all())


@gpu
@pytest.mark.parametrize("hd,h,hk,new,keys", [(128, 16, 4, 1, 20011), (64, 8, 8, 1, 9999), (128, 16, 2, 3, 12345),
                                              (64, 16, 2, 200, 8200), (128, 4, 4, 40, 16385), (128, 16, 4, 700, 5000)])
def test_paged_attention_long_rows(cuda, hd, h, hk, new, keys):
    """Rows whose keys are shared out over the card and joined."""
    dtype = torch.bfloat16
    ks, vs, kc, vc, table = _paged([keys, 70], hk, 64, hd, dtype, cuda, 60)
    q = _randn((new + 1, h, hd), dtype, cuda, 61)
    # a key that outweighs the others, in the middle and at the ends
    for j in (0, keys // 2, keys - new):
        x = q[:1, ::h // hk] * 1.5
        ks[0][j], pg = x[0], int(table[0, j // 64])
        kc[pg, :, j % 64] = x[0]
    got = _C.flash_attn_paged(q, kc, vc, table, _cu([new, 1], cuda), _i32([keys, 70], cuda), hd**-0.5, max_q_len=new)
    for b, s in ((0, slice(0, new)), (1, slice(new, new + 1))):
        want, tol = _attend(q[s], ks[b], vs[b], hd**-0.5, True, dtype)
        _same(got[s], want, tol, f"sequence {b}")


@gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,h,hk", [(1, 8, 2), (3, 4, 4), (60, 8, 2)])
def test_a_part_of_the_keys_without_a_finite_score_makes_the_row_nan(cuda, hd, new, h, hk):
    """Keys shared out over the card: one part's keys are all NaN (its largest score is no number), another's
    scores are all -inf (they weigh nothing)."""
    dtype, keys = torch.bfloat16, 4096 + new
    ks, vs, kc, vc, table = _paged([keys], hk, 256, hd, dtype, cuda, 65)
    q = _randn((new, h, hd), dtype, cuda, 66).abs()
    args = (table, _cu([new], cuda), _i32([keys], cuda), hd**-0.5)
    clean_k = kc.clone()
    kc[int(table[0, 2])] = -3.0e38  # 256 keys: q > 0, so every score is -inf
    ks[0][512:768] = -3.0e38
    got = _C.flash_attn_paged(q, kc, vc, *args)
    keep = [j for j in range(keys) if not 512 <= j < 768]
    want, tol = _attend(q, ks[0][keep], vs[0][keep], hd**-0.5, True, dtype)
    _same(got, want, tol, "a part that weighs nothing")
    for page in (0, 7, 15):
        kc = clean_k.clone()
        kc[int(table[0, page])] = math.nan
        assert bool(torch.isnan(_C.flash_attn_paged(q, kc, vc, *args)).all()), page
    kc = clean_k.clone()
    kc[int(table[0, 16]), :, new - 1] = math.nan  # the last key, of the last row alone
    got = _C.flash_attn_paged(q, kc, vc, *args)
    assert bool(torch.isnan(got[-1]).all()) and not bool(torch.isnan(got[:-1]).any())


@gpu
@pytest.mark.parametrize("hint", [1, 2, 3])
def test_paged_attention_with_a_bound_that_is_too_small(cuda, hint):
    """Slower, but right and within its workspace."""
    dtype, hd, h, hk = torch.float16, 64, 6, 2
    new, lens = [40, 1, 7, 200], [900, 300, 7, 1500]
    ks, vs, kc, vc, table = _paged(lens, hk, 16, hd, dtype, cuda, 68)
    q = _randn((sum(new), h, hd), dtype, cuda, 69)
    need = _C.flash_attn_paged_workspace(sum(new), len(new), h, hk, hd, 16, table.shape[1], hint)
    ws = torch.full((need + 64,), 2.0, device=cuda)
    got = _C.flash_attn_paged(q, kc, vc, table, _cu(new, cuda), _i32(lens, cuda), 0.125, max_q_len=hint, workspace=ws[:need])
    assert bool((ws[need:] == 2).all())
    at = 0
    for b, n in enumerate(new):
        want, tol = _attend(q[at:at + n], ks[b], vs[b], 0.125, True, dtype)
        _same(got[at:at + n], want, tol, f"sequence {b}")
        at += n


@gpu
@pytest.mark.parametrize("batch", [64, 65, 130])
def test_many_sequences(cuda, batch):
    """More than a wave holds at a time, in every operator."""
    dtype, hd, h, hk, page = torch.bfloat16, 64, 4, 2, 16
    new = [(7 * b) % 5 if b % 3 else 1 for b in range(batch)]
    new[batch // 2] = 150
    lens = [n + (37 * b) % 700 for b, n in enumerate(new)]
    ks, vs, kc, vc, table = _paged(lens, hk, page, hd, dtype, cuda, 170)
    x = _randn((sum(new), h + 2 * hk, hd), dtype, cuda, 171)
    q, k, v = x[:, :h], x[:, h:h + hk], x[:, h + hk:]
    cu, kvl = _cu(new, cuda), _i32(lens, cuda)
    packed = _C.flash_attn_packed(q, k, v, cu, 0.125, True)
    paged = _C.flash_attn_paged(q, kc, vc, table, cu, kvl, 0.125, max_q_len=150)
    steps, _ = _C.rotary_steps(hd, device=cuda)
    turned, _ = _C.rotary_append(q, k, v, steps, cu, kv_lens=kvl, block_table=table, k_cache=kc, v_cache=vc)
    at = 0
    for b, n in enumerate(new):
        s = slice(at, at + n)
        if n:
            want, tol = _attend(q[s], k[s], v[s], 0.125, True, dtype)
            _same(packed[s], want, tol, f"packed {b}")
            want, tol = _attend(q[s], ks[b], vs[b], 0.125, True, dtype)
            _same(paged[s], want, tol, f"paged {b}")
            want, tol = _rotate(q[s], list(range(lens[b] - n, lens[b])), steps.cpu(), 1.0, False, dtype)
            _same(turned[s], want, tol, f"turned {b}")
            last = lens[b] - 1
            assert torch.equal(vc[int(table[b, last // page]), :, last % page], v[at + n - 1])
        at += n


@gpu
@pytest.mark.parametrize("new", [1, 5, 90])
def test_paged_attention_of_a_sequence_does_not_depend_on_the_batch(cuda, new):
    dtype, hd, h, hk = torch.bfloat16, 128, 8, 2
    lens, news = [3000, 17, 2500, 900], [new, 1, 3, 200]
    ks, vs, kc, vc, table = _paged(lens, hk, 16, hd, dtype, cuda, 70)
    q = _randn((sum(news), h, hd), dtype, cuda, 71)
    both = _C.flash_attn_paged(q, kc, vc, table, _cu(news, cuda), _i32(lens, cuda), 0.1, max_q_len=max(news))
    alone = _C.flash_attn_paged(q[:new], kc, vc, table[:1], _cu([new], cuda), _i32([3000], cuda), 0.1, max_q_len=new)
    assert torch.equal(both[:new], alone)
    again = _C.flash_attn_paged(q, kc, vc, table, _cu(news, cuda), _i32(lens, cuda), 0.1, max_q_len=max(news))
    assert torch.equal(both, again)


@gpu
@pytest.mark.parametrize("new,h,hk", [(1, 8, 2), (3, 8, 8), (80, 8, 2)])
def test_paged_attention_pages_outside_the_pool(cuda, new, h, hk):
    """A page index the pool does not have, or keys the table has no page for, make the rows that need them
    NaN; nothing is read through it and no other row changes."""
    dtype, hd, page = torch.float16, 64, 16
    lens, news = [700, 300, 2000], [new, 1, new]
    ks, vs, kc, vc, table = _paged(lens, hk, page, hd, dtype, cuda, 80)
    q = _randn((sum(news), h, hd), dtype, cuda, 81)
    cu = _cu(news, cuda)
    good = _C.flash_attn_paged(q, kc, vc, table, cu, _i32(lens, cuda), 0.125, max_q_len=new)
    assert not bool(torch.isnan(good).any())
    hole = lens[0] - new + 1 if new > 1 else 5  # the last rows, or all of them, need this key
    hole = hole // page * page
    table[0, hole // page] = kc.shape[0]
    table[2, 1] = -(2**31)
    got = _C.flash_attn_paged(q, kc, vc, table, cu, _i32(lens, cuda), 0.125, max_q_len=new)
    need = torch.arange(lens[0] - new, lens[0], device=cuda) >= hole
    assert bool(torch.isnan(got[:new][need]).all()) and torch.equal(got[:new][~need], good[:new][~need])
    assert torch.equal(got[new:new + 1], good[new:new + 1]) and bool(torch.isnan(got[new + 1:]).all())
    # more keys than the table has pages for
    table2 = table[1:2, :4].contiguous()
    got = _C.flash_attn_paged(q[:1], kc, vc, table2, _cu([1], cuda), _i32([65], cuda), 0.125)
    assert bool(torch.isnan(got).all())


@gpu
def test_paged_attention_cache_beyond_32_bit_offsets(cuda):
    """Pages whose element offset passes 2^31, in a cache of 5 GB; and the append into them."""
    dtype, hd, hk, page = torch.bfloat16, 128, 4, 64
    pages = (1 << 31) // (hk * page * hd) + 40
    kc = torch.zeros(pages, hk, page, hd, dtype=dtype, device=cuda)
    vc = torch.zeros_like(kc)
    table = _i32([[pages - 1, pages - 3, 0, pages - 2]], cuda)
    n, h = 200, 8
    x = _randn((n, h + 2 * hk, hd), dtype, cuda, 90)
    steps, _ = _C.rotary_steps(hd, device=cuda)
    q, k = _C.rotary_append(x[:, :h], x[:, h:h + hk], x[:, h + hk:], steps, _cu([n], cuda), kv_lens=_i32([n], cuda),
                            block_table=table, k_cache=kc, v_cache=vc, k_out=torch.empty(n, hk, hd, dtype=dtype, device=cuda))
    want = _C.flash_attn_packed(q, k, x[:, h + hk:], _cu([n], cuda), 0.1, True)
    got = _C.flash_attn_paged(q, kc, vc, table, _cu([n], cuda), _i32([n], cuda), 0.1)
    ref, tol = _attend(q, k, x[:, h + hk:], 0.1, True, dtype)
    _same(want, ref, tol, "packed")
    _same(got, ref, tol, "paged")


@gpu
@pytest.mark.parametrize("starts", [[0, 9, 2, 20, 11, 30], [0, 40, 40, -5, 10**9, 30], [7, 3, 1, 0, 0, 0]])
def test_starts_that_do_not_ascend_stay_in_bounds(cuda, starts):
    """No result is promised for such starts but that nothing outside the rows and the slots named is written."""
    dtype, hd, h, hk, batch = torch.bfloat16, 64, 4, 2, 5
    _, _, kc, vc, table = _paged([600] * batch, hk, 16, hd, dtype, cuda, 150, fill=0.0)
    whole = torch.full((40, h, hd), 3.0, dtype=dtype, device=cuda)
    out, cu, kvl = whole[5:35], _i32(starts, cuda), _i32([600] * batch, cuda)
    x = _randn((30, h + 2 * hk, hd), dtype, cuda, 151)
    for max_q in (0, 1):
        ws = torch.full((_C.flash_attn_paged_workspace(30, batch, h, hk, hd, 16, table.shape[1], max_q) + 64,), 2.0,
                        device=cuda)
        _C.flash_attn_paged(x[:, :h], kc, vc, table, cu, kvl, 0.1, max_q_len=max_q, out=out, workspace=ws[:-64])
        assert bool((ws[-64:] == 2).all())
    _C.flash_attn_packed(x[:, :h], x[:, h:h + hk], x[:, h + hk:], cu, 0.1, True, out=out)
    steps, _ = _C.rotary_steps(hd, device=cuda)
    spare = [p for p in range(kc.shape[0]) if not bool((table == p).any())]
    _C.rotary_append(x[:, :h], x[:, h:h + hk], x[:, h + hk:], steps, cu, kv_lens=kvl, block_table=table, k_cache=kc,
                     v_cache=vc, q_out=out)
    torch.cuda.synchronize()
    assert bool((whole[:5] == 3).all()) and bool((whole[35:] == 3).all())
    assert bool((kc[spare] == 0).all()) and bool((vc[spare] == 0).all())


# ---------------------------------------------------------------- together
@gpu
@pytest.mark.parametrize("dtype,hd,h,hk,page", [(torch.bfloat16, 128, 8, 2, 16), (torch.float16, 64, 8, 8, 32)])
def test_prompts_chunks_and_single_tokens_in_turn(cuda, dtype, hd, h, hk, page):
    """Three sequences served: prompts packed, then a chunk of one beside single tokens, then single tokens;
    every step's rows against the attention of the whole sequences."""
    total, prompt = [190, 40, 77], [60, 33, 70]
    plan = [prompt, [90, 1, 1], [35, 1, 0], [1, 1, 1], [1, 1, 1], [1, 0, 1], [1, 1, 1], [1, 2, 2]]
    assert [sum(x) for x in zip(*plan)] == total
    xs = [_randn((n, h + 2 * hk, hd), dtype, cuda, 100 + b) for b, n in enumerate(total)]
    steps, _ = _C.rotary_steps(hd, device=cuda)
    pages = sum((n + page - 1) // page for n in total)
    kc = torch.full((pages, hk, page, hd), math.nan, dtype=dtype, device=cuda)
    vc = kc.clone()
    order = torch.randperm(pages, generator=_gen(3)).to(torch.int32)
    table = torch.full((3, 12 * 16 // page + 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(total):
        m = (n + page - 1) // page
        table[b, :m] = order[at:at + m]
        at += m
    table = table.to(cuda)
    want, tols = [], []
    for x, n in zip(xs, total):
        q, k = _C.rotary_append(x[:, :h], x[:, h:h + hk], None, steps, _cu([n], cuda))
        w, tol = _attend(q, k, x[:, h + hk:], hd**-0.5, True, dtype)
        want.append(w)
        tols.append(tol)
    done = [0, 0, 0]
    for i, new in enumerate(plan):
        x = torch.cat([x[d:d + n] for x, d, n in zip(xs, done, new)])
        now = [d + n for d, n in zip(done, new)]
        cu, kvl = _cu(new, cuda), _i32(now, cuda)
        k_out = torch.empty(x.shape[0], hk, hd, dtype=dtype, device=cuda) if i == 0 else None
        q, k = _C.rotary_append(x[:, :h], x[:, h:h + hk], x[:, h + hk:], steps, cu, kv_lens=kvl, block_table=table,
                                k_cache=kc, v_cache=vc, k_out=k_out)
        if i == 0:
            o = _C.flash_attn_packed(q, k, x[:, h + hk:], cu, hd**-0.5, True)
        else:
            o = _C.flash_attn_paged(q, kc, vc, table, cu, kvl, hd**-0.5, max_q_len=max(new))
        ref = torch.cat([w[d:n] for w, d, n in zip(want, done, now)])
        tol = torch.cat([w[d:n] for w, d, n in zip(tols, done, now)])
        _same(o, ref, tol, f"step {i}")
        done = now


@gpu
def test_one_captured_step_serves_other_lengths(cuda):
    """A captured append + attention, replayed after the lengths, pages and inputs changed, beside a second
    graph and eager calls; every replay equals the eager result."""
    dtype, hd, h, hk, page, batch = torch.bfloat16, 128, 8, 2, 16, 4
    lens = [700, 33, 1500, 260]
    steps, _ = _C.rotary_steps(hd, device=cuda)
    _, _, kc, vc, table = _paged([n + 40 for n in lens], hk, page, hd, dtype, cuda, 110, fill=0.0)
    cu = _cu([1] * batch, cuda)
    kvl = _i32(lens, cuda)
    x = _randn((batch, h + 2 * hk, hd), dtype, cuda, 111)

    def step():
        q, _ = _C.rotary_append(x[:, :h], x[:, h:h + hk], x[:, h + hk:], steps, cu, kv_lens=kvl, block_table=table,
                                k_cache=kc, v_cache=vc)
        return _C.flash_attn_paged(q, kc, vc, table, cu, kvl, hd**-0.5, max_q_len=1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for i in range(6):
        x.copy_(_randn(x.shape, dtype, cuda, 120 + i))
        kvl.copy_(_i32([n + i * (b + 1) for b, n in enumerate(lens)], cuda))
        graphs[i % 2].replay()
        got = outs[i % 2].clone()
        torch.cuda.synchronize()
        assert torch.equal(got, step()), i


@gpu
def test_recorded_launches_run_again(cuda):
    dtype, hd, h, hk = torch.bfloat16, 64, 4, 2
    ks, vs, kc, vc, table = _paged([900, 30], hk, 16, hd, dtype, cuda, 160)
    cu, kvl = _cu([2, 5], cuda), _i32([900, 30], cuda)
    x = _randn((7, h + 2 * hk, hd), dtype, cuda, 161)
    q, k, v = x[:, :h], x[:, h:h + hk], x[:, h + hk:]
    steps, _ = _C.rotary_steps(hd, device=cuda)
    with _C.record_launches() as calls:
        outs = [_C.rotary_append(q, k, None, steps, cu)[0], _C.flash_attn_packed(q, k, v, cu, 0.1, True),
                _C.flash_attn_paged(q, kc, vc, table, cu, kvl, 0.1)]
    assert [c.info["op"] for c in calls] == ["rotary_append", "flash_attn_packed", "flash_attn_paged"]
    want = [o.clone() for o in outs]
    for o in outs:
        o.zero_()
    for c in calls:
        c()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


@gpu
def test_calls_on_two_streams_at_once(cuda):
    dtype, hd, h, hk = torch.float16, 64, 8, 2
    ks, vs, kc, vc, table = _paged([5000, 400], hk, 32, hd, dtype, cuda, 130)
    cu, kvl = _cu([1, 6], cuda), _i32([5000, 400], cuda)
    qs = [_randn((7, h, hd), dtype, cuda, 131 + i) for i in range(2)]
    want = [_C.flash_attn_paged(q, kc, vc, table, cu, kvl, 0.125) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    outs = [[] for _ in qs]
    for _ in range(10):
        for q, s, o in zip(qs, streams, outs):
            with torch.cuda.stream(s):
                o.append(_C.flash_attn_paged(q, kc, vc, table, cu, kvl, 0.125))
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert all(torch.equal(w, x) for x in o)


@gpu
def test_nothing_to_do(cuda):
    bf = torch.bfloat16
    q, k = torch.empty(0, 8, 64, dtype=bf, device=cuda), torch.empty(0, 2, 64, dtype=bf, device=cuda)
    assert _C.flash_attn_packed(q, k, k, _cu([], cuda), 0.1, True).shape == (0, 8, 64)
    kc = torch.zeros(1, 2, 16, 64, dtype=bf, device=cuda)
    table = torch.zeros(2, 1, dtype=torch.int32, device=cuda)
    assert _C.flash_attn_paged(q, kc, kc.clone(), table, _cu([0, 0], cuda), _i32([0, 9], cuda), 0.1).shape == (0, 8, 64)
    # sequences that bring nothing, among rows of none
    q = torch.ones(3, 8, 64, dtype=bf, device=cuda)
    out = torch.full_like(q, 5.0)
    _C.flash_attn_paged(q, kc, kc.clone(), table, _cu([0, 0], cuda), _i32([0, 9], cuda), 0.1, out=out)
    assert bool((out == 5).all())
