"""Head norms with the append to 16- and 8-bit caches, attention over an 8-bit cache, attention of draft trees and
the move of their accepted path, each against its formula in 64 bits.

Tolerances, per element, from the roundings alone (eps = finfo(dtype).eps, half a step is eps / 2):

* norms, in fp32 (u = 2^-24): a mean over hd elements is off by at most (hd + 2) u A, A = mean |x|, so x - mu by
  that and u (|x| + A); the mean square by hd u of itself and, for the shifted mean, twice (hd + 2) u A / std; its
  root by half of that, and a few u for root, reciprocal and products.  With r = 1 / std of the formula all of it is
  below (2 hd + 16) u (1 + A r) of |weight| r (|x| + A), and u of the result for the bias.
* the turn: as in test_seq_ops, 2^-20 amplitude (|y1| + |y2|), and amplitude times the errors of y1 and y2.
* 16 bits: one rounding, eps / 2 of the result (fp16 below 2^-14: 2^-25).  8 bits: a code has 4 significant bits,
  2^-4 of the value and, where codes are subnormal, 2^-10 of the scale.
* attention: as in test_seq_ops, for the values that the cache stands for (exact in dtype).
"""

import math
import shutil
from fractions import Fraction

import pytest
import torch

from transformer_optimization_amd import _C
from _util import log
from test_seq_ops import E, FAKE, PAGE_REFUSALS, PAGED_CASES, SEQ_REFUSALS, U, _cu, _gen, _i32, _paged, _randn, _same

DTYPES = [torch.bfloat16, torch.float16]
gpu = pytest.mark.gpu
LOWEST = {torch.bfloat16: -117, torch.float16: -15}
TOP = {torch.bfloat16: 1.875 * 2.0**127, torch.float16: 61440.0}


# ------------------------------------------------------------------- oracles
def _scale_exponents(x, dtype):
    """Smallest e with every magnitude of the 32 within 448 * 2^e (x: finite, 64-bit, [..., hd])."""
    amax = x.unflatten(-1, (-1, 32)).abs().amax(-1).clamp(max=TOP[dtype])
    m, e = torch.frexp(amax)  # m in [1/2, 1)
    e = e - 9 + (m > 0.875).to(e.dtype)
    return torch.where(amax > 0, e, torch.full_like(e, LOWEST[dtype])).clamp(min=LOWEST[dtype])


def _codes(x, e, dtype):
    """The e4m3 values (64-bit) nearest to x / 2^e, ties to even."""
    y = x.clamp(-TOP[dtype], TOP[dtype]).unflatten(-1, (-1, 32)) / torch.exp2(e.double())[..., None]
    _, b = torch.frexp(y.abs().clamp(min=2.0**-6))
    step = torch.exp2((b - 4).double())
    return (torch.round(y / step) * step).flatten(-2)


def _stored(x, dtype, dev):
    """Codes and scale bytes of x [..., hd] as an 8-bit cache holds them, and the values they stand for, in dtype."""
    e = _scale_exponents(x.double(), dtype)
    c = _codes(x.double(), e, dtype)
    values = (c.unflatten(-1, (-1, 32)) * torch.exp2(e.double())[..., None]).flatten(-2)
    assert torch.equal(values.to(dtype).double(), values)  # exact in dtype
    return (c.float().to(torch.float8_e4m3fn).view(torch.uint8).to(dev), (e + 127).to(torch.uint8).to(dev),
            values.to(dtype).to(dev))


def _values(codes, scales):
    """64-bit values of a cache."""
    c = codes.view(torch.float8_e4m3fn).float().double().unflatten(-1, (-1, 32))
    s = scales.view(torch.uint8).double()
    return (c * torch.where(s == 255, torch.full_like(s, math.nan), torch.exp2(s - 127))[..., None]).flatten(-2)


def _paged8(lens, kv_heads, page, hd, dtype, dev, seed, token_major=False, spare=3, width=None):
    """As _paged, 8-bit: keys and values of each sequence (the values that are stored, in dtype), codes and scales
    whose unused slots are NaN (codes 0x7F, scales 255)."""
    counts = [(n + page - 1) // page for n in lens]
    pages = sum(counts) + spare
    order = torch.randperm(pages, generator=_gen(seed)).to(torch.int32)
    width = width or max(max(counts), 1)
    table = torch.full((len(lens), width), -7, dtype=torch.int32)
    table[:, 1::2] = 2**31 - 1
    made = []
    for n in (hd, hd // 32):
        shape = (pages, page, kv_heads, n) if token_major else (pages, kv_heads, page, n)
        made += [torch.full(shape, 0x7F if n == hd else 255, dtype=torch.uint8) for _ in range(2)]
    views = [c.transpose(1, 2) if token_major else c for c in made]
    sides, at = ([], []), 0
    for b, n in enumerate(lens):
        table[b, :counts[b]] = order[at:at + counts[b]]
        at += counts[b]
        for i in (0, 1):
            x = torch.randn(n, kv_heads, hd, generator=_gen(seed + 10 * b + i + 1))
            if i == 0:
                x[..., 3] *= 4  # a strong channel
            codes, scales, values = _stored(x, dtype, "cpu")
            for view, y in ((views[i], codes), (views[2 + i], scales)):
                for p in range(counts[b]):
                    part = y[p * page:(p + 1) * page]
                    view[int(table[b, p]), :, :part.shape[0]] = part.transpose(0, 1)
            sides[i].append(values.to(dev))
    made = [c.to(dev) for c in made]
    views = [c.transpose(1, 2) if token_major else c for c in made]
    return sides[0], sides[1], views[0].view(torch.float8_e4m3fn), views[2], views[1].view(torch.float8_e4m3fn), \
        views[3], table.to(dev)


def _attend(q, k, v, scale, seen, dtype):
    """64-bit attention of q [n, H, d] over k, v [m, Hk, d] where `seen` [n, m] says so; other keys are left out.
    Returns the result (0 for rows that see nothing) and its tolerance."""
    n, h, d = q.shape
    m, hk = k.shape[:2]
    out = torch.zeros(n, h, d, dtype=torch.float64, device=q.device)
    tol = torch.full_like(out, 2.0**-25)
    eps = torch.finfo(dtype).eps
    some = seen.any(1)
    for x in range(h if m else 0):
        qx, kx, vx = q[:, x].double(), k[:, x // (h // hk)].double(), v[:, x // (h // hk)].double()
        s = ((qx @ kx.T) * scale).masked_fill(~seen, -math.inf)
        size = ((qx.abs() @ kx.abs().T) * scale).masked_fill(~seen, 0.0)
        top = torch.where(some, s.amax(1), torch.zeros_like(s[:, 0]))[:, None]
        p = torch.where(seen, torch.exp(s - top), torch.zeros_like(s))
        total = torch.where(some, p.sum(1), torch.ones_like(p[:, 0]))[:, None]
        bad = ~torch.isfinite(vx)
        clean = vx.masked_fill(bad, 0.0)
        o, a = p @ clean / total, p @ clean.abs() / total
        out[:, x] = torch.where((seen.double() @ bad.double()) > 0, torch.full_like(o, math.nan), o)
        if dtype == torch.float16:
            a = a + 2.0**-25 / eps * (seen.double() @ clean.abs()) / total
        tol[:, x] += eps / 2 * o.abs() + a * (eps + 2 * (d + 8) * 2.0**-24 * size.amax(1, keepdim=True) + 2 * m * 2.0**-24)
    return out, tol


def _causal(n, m, dev):
    return torch.ones(n, m, dtype=torch.bool, device=dev).tril(m - n)


def _tree(n, seed, roots=1):
    """Parents of a random tree of n tokens, several of them possibly without one."""
    g = _gen(seed)
    return [-1 if i < roots else int(torch.randint(0, i, (1,), generator=g)) for i in range(n)]


def _tree_seen(parents, m, dev):
    """Which of m keys (the last ones the tokens of the tree) each token sees."""
    n = len(parents)
    seen = torch.zeros(n, m, dtype=torch.bool)
    seen[:, :max(m - n, 0)] = True
    for i in range(n):
        x = i
        while x >= 0:
            if m - n + x >= 0:
                seen[i, m - n + x] = True
            x = parents[x]
    return seen.to(dev)


# --------------------------------------------------------- refusals (CPU)
class _Abi:
    """The C entry points on made-up addresses, one argument changed at a time."""

    def __init__(self):
        import ctypes
        self.lib, self.ct, self.keep = _C.load_library(), ctypes, []

    def st(self, v):
        if v is None or v[0] is None:
            return None
        a = (self.ct.c_int64 * len(v))(*v)
        self.keep.append(a)
        return self.ct.addressof(a)

    def append(self, **kw):
        a = dict(q=FAKE, qs=(512, 64), qo=1 << 30, qos=(512, 64), k=1 << 31, ks=(128, 64), ko=None, kos=(128, 64),
                 v=3 << 30, vs=(128, 64), kc=1 << 33, kcs=(2048, 1024, 64), vc=1 << 34, vcs=(2048, 1024, 64),
                 ksc=None, kss=(64, 32, 2), vsc=None, vss=(64, 32, 2), qw=1 << 36, qb=None, kw=(1 << 36) + 4096, kb=None,
                 ph=0, pdt=_C.TX_BF16, norm=1, eps=1e-6, steps=FAKE, axis=None, pos=None, pld=64, axes=1, cu=FAKE,
                 kvl=FAKE, table=FAKE, ld=8, t=64, b=2, h=8, hk=2, hd=64, r=64, np=32, ps=16, mp=8, amp=1.0,
                 dt=_C.TX_BF16)
        a.update(kw)
        return self.lib.tx_norm_rotary_append(
            a["q"], self.st(a["qs"]), a["qo"], self.st(a["qos"]), a["k"], self.st(a["ks"]), a["ko"], self.st(a["kos"]),
            a["v"], self.st(a["vs"]), a["kc"], self.st(a["kcs"]), a["ksc"], self.st(a["kss"]), a["vc"], self.st(a["vcs"]),
            a["vsc"], self.st(a["vss"]), a["qw"], a["qb"], a["kw"], a["kb"], a["ph"], a["pdt"], a["norm"], a["eps"],
            a["steps"], a["axis"], a["pos"], a["pld"], a["axes"], a["cu"], a["kvl"], a["table"], a["ld"], a["t"], a["b"],
            a["h"], a["hk"], a["hd"], a["r"], a["np"], a["ps"], a["mp"], a["amp"], 0, a["dt"], None)

    def paged(self, tree=False, **kw):
        a = dict(q=FAKE, qs=(512, 64), kc=1 << 33, kcs=(2048, 1024, 64), vc=1 << 34, vcs=(2048, 1024, 64), ksc=1 << 36,
                 kss=(64, 32, 2), vsc=1 << 37, vss=(64, 32, 2), o=3 << 30, os=(512, 64), cu=FAKE, kvl=FAKE, table=FAKE,
                 ld=8, mask=1 << 38, mld=1, words=1, t=64, b=2, h=8, hk=2, hd=64, np=32, ps=16, mp=8, mq=0, scale=0.125,
                 ws=1 << 35, wsn=1 << 40, dt=_C.TX_BF16)
        a.update(kw)
        head = (a["q"], self.st(a["qs"]), a["kc"], self.st(a["kcs"]), a["ksc"], self.st(a["kss"]), a["vc"],
                self.st(a["vcs"]), a["vsc"], self.st(a["vss"]), a["o"], self.st(a["os"]), a["cu"], a["kvl"], a["table"],
                a["ld"])
        sizes = (a["t"], a["b"], a["h"], a["hk"], a["hd"], a["np"], a["ps"], a["mp"], a["mq"], a["scale"])
        if tree:
            return self.lib.tx_flash_attn_tree(*head, a["mask"], a["mld"], a["words"], *sizes, a["ws"], a["wsn"], a["dt"],
                                               None)
        return self.lib.tx_flash_attn_paged_mx8(*head, *sizes, 1, a["ws"], a["wsn"], a["dt"], None)

    def accept(self, **kw):
        a = dict(kc=1 << 33, kcs=(2048, 1024, 64), vc=1 << 34, vcs=(2048, 1024, 64), ksc=None, kss=(64, 32, 2), vsc=None,
                 vss=(64, 32, 2), cu=FAKE, kvl=FAKE, table=FAKE, ld=8, path=FAKE, pld=8, mpath=8, counts=FAKE, lens=1 << 30,
                 b=2, hk=2, hd=64, np=32, ps=16, mp=8, dt=_C.TX_BF16)
        a.update(kw)
        return self.lib.tx_cache_accept(
            a["kc"], self.st(a["kcs"]), a["ksc"], self.st(a["kss"]), a["vc"], self.st(a["vcs"]), a["vsc"],
            self.st(a["vss"]), a["cu"], a["kvl"], a["table"], a["ld"], a["path"], a["pld"], a["mpath"], a["counts"],
            a["lens"], a["b"], a["hk"], a["hd"], a["np"], a["ps"], a["mp"], a["dt"], None)


MX = dict(ksc=1 << 37, vsc=1 << 38)


@pytest.mark.parametrize("change,code", SEQ_REFUSALS + PAGE_REFUSALS + [
    (dict(steps=None), E), (dict(k=None), E), (dict(r=0), E), (dict(r=7), E), (dict(r=66), E), (dict(qo=None), E),
    (dict(hd=260, r=64), U), (dict(hd=512, r=64), U), (dict(amp=0.0), E), (dict(amp=math.nan), E), (dict(v=None), E),
    (dict(kc=None, vc=None), E), (dict(qo=FAKE + 1024), E), (dict(qo=FAKE, qos=(1024, 64)), E), (dict(qo=1 << 31), E),
    (dict(ko=FAKE), E), (dict(kc=1 << 31), E), (dict(vc=(1 << 33) + 1024), E), (dict(qos=(512, 0)), E),
    (dict(kos=(64, 64), ko=1 << 39), E), (dict(pos=FAKE + 4), U), (dict(steps=FAKE + 4), U), (dict(axis=FAKE + 2), U),
    (dict(norm=3), E), (dict(norm=-1), E), (dict(eps=-1.0), E), (dict(eps=math.nan), E), (dict(eps=math.inf), E),
    (dict(qb=1 << 37), E),                              # a shift without its norm
    (dict(norm=0), E),                                   # gains without a norm
    (dict(q=None, qo=None), E),                          # gains of a q that is not there
    (dict(qw=(1 << 36) + 8), U), (dict(pdt=_C.TX_F16), U), (dict(pdt=7), U),
    (dict(axes=0), E), (dict(axes=3, pos=1 << 39, pld=63), E), (dict(axes=1 << 17, pos=1 << 39), U),
    (dict(ksc=1 << 37), E), (dict(vsc=1 << 37), E), (dict(kc=None, vc=None, ko=1 << 39, **MX), E),
    (dict(hd=40, r=8, qs=(320, 40), qos=(320, 40), ks=(80, 40), vs=(80, 40), kcs=(1280, 640, 48), vcs=(1280, 640, 48), **MX), U),
    (dict(kcs=(2048, 1024, 72), **MX), U), (dict(kss=(64, 32, 1), **MX), E), (dict(kss=(64, 32, -2), **MX), E),
    (dict(kss=(1 << 31, 32, 2), **MX), U), (dict(ksc=1 << 37, vsc=(1 << 37) + 64), E), (dict(ksc=1 << 33, vsc=1 << 38), E),
    (dict(qo=1 << 36), E),                               # over the gains
    (dict(kc=FAKE & ~15), E),                            # over the table
])
def test_norm_rotary_append_refusals(change, code):
    assert _Abi().append(**change) == code


ATTENTION_REFUSALS = SEQ_REFUSALS + [c for c in PAGE_REFUSALS if "kcs" not in c[0] and "vcs" not in c[0]] + [
    (dict(kc=None), E), (dict(o=None), E), (dict(hd=96), U), (dict(scale=-1.0), E), (dict(o=1 << 33), E),
    (dict(o=(1 << 34) + 256), E), (dict(o=FAKE + 16), E), (dict(os=(512, 8)), E), (dict(kvl=FAKE + 2), U),
    (dict(kcs=(2048, 1024, 72)), U), (dict(kcs=(1 << 31, 1024, 64)), U), (dict(vcs=(1 << 30, 1024, 1 << 24)), U),
    (dict(kcs=(2048, 1024, -64)), E), (dict(vcs=(2048, 512, 64)), E), (dict(kcs=(1024, 1024, 64)), E),
    (dict(ksc=None), E), (dict(vsc=None), E), (dict(kss=(None,)), E), (dict(ksc=(1 << 36) + 1), U), (dict(kss=(65, 32, 2)), U),
    (dict(kss=(64, 32, 1)), U), (dict(vss=(64, 16, 2)), E), (dict(vss=(1 << 31, 32, 2)), U), (dict(o=1 << 36), E),
    (dict(wsn=0, mp=512, ld=512), E), (dict(ws=1 << 37, mp=512, ld=512), E), (dict(ws=1 << 33, mp=512, ld=512), E),
]


@pytest.mark.parametrize("change,code", ATTENTION_REFUSALS)
def test_paged_mx8_refusals(change, code):
    assert _Abi().paged(**change) == code


@pytest.mark.parametrize("change,code", ATTENTION_REFUSALS + [
    (dict(mask=None), E), (dict(words=0), E), (dict(mld=-1), E), (dict(words=2), E), (dict(mask=(1 << 38) + 4), U),
    (dict(words=1 << 25, mld=1 << 25), U), (dict(o=1 << 38), E), (dict(ws=1 << 38, mp=512, ld=512), E),
    (dict(ksc=None, vsc=None, kcs=(2048, 1024, 60)), U),
])
def test_tree_refusals(change, code):
    assert _Abi().paged(tree=True, **change) == code


@pytest.mark.parametrize("change,code", [c for c in PAGE_REFUSALS] + [
    (dict(cu=None), E), (dict(path=None), E), (dict(counts=None), E), (dict(lens=None), E), (dict(b=0), E), (dict(hk=0), E),
    (dict(hd=0), E), (dict(mpath=0), E), (dict(pld=7), E), (dict(path=FAKE + 2), U), (dict(counts=FAKE + 1), U),
    (dict(lens=FAKE), E), (dict(lens=(1 << 30) + 2), U), (dict(dt=_C.TX_F32), U), (dict(hd=260), U), (dict(ksc=1 << 37), E),
    (dict(kss=(64, 32, 1), **MX), E), (dict(hk=1 << 16), U), (dict(vc=(1 << 33) + 1024), E), (dict(lens=1 << 33), E),
])
def test_cache_accept_refusals(change, code):
    assert _Abi().accept(**change) == code


def _cpu_args():
    bf = torch.bfloat16
    kc, ks = _C.mx8_cache(5, 2, 16, 64)
    return dict(q=torch.zeros(6, 8, 64, dtype=bf), k=torch.zeros(6, 2, 64, dtype=bf), v=torch.zeros(6, 2, 64, dtype=bf),
                kc=kc, ks=ks, vc=kc.clone(), vs=ks.clone(), table=torch.zeros(2, 3, dtype=torch.int32),
                cu=_i32([0, 2, 6], "cpu"), kvl=_i32([2, 4], "cpu"), steps=torch.zeros(32, dtype=torch.int64),
                mask=torch.zeros(6, 1, dtype=torch.int64), path=torch.zeros(2, 4, dtype=torch.int32),
                counts=_i32([1, 2], "cpu"))


def test_wrappers_check_their_arguments_before_the_device():
    a = _cpu_args()

    def mx8(**kw):
        b = {**a, **kw}
        return _C.flash_attn_paged_mx8(b["q"], b["kc"], b["ks"], b["vc"], b["vs"], b["table"], b["cu"], b["kvl"], 0.1)

    def tree(**kw):
        b = {**a, **kw}
        return _C.flash_attn_tree(b["q"], b["kc"], b["vc"], b["table"], b["cu"], b["kvl"], b["mask"], 0.1,
                                  k_scales=b["ks"], v_scales=b["vs"])

    def accept(**kw):
        b = {**a, **kw}
        return _C.cache_accept(b["kc"], b["vc"], b["table"], b["cu"], b["kvl"], b["path"], b["counts"], k_scales=b["ks"],
                               v_scales=b["vs"])

    def append(**kw):
        b = {**a, **kw}
        more = {x: y for x, y in kw.items() if x not in a}
        return _C.norm_rotary_append(b["q"], b["k"], b["v"], b["steps"], b["cu"], kv_lens=b["kvl"], block_table=b["table"],
                                     k_cache=b["kc"], v_cache=b["vc"], k_scales=b["ks"], v_scales=b["vs"], **more)

    for call in (mx8, tree, accept, append):
        with pytest.raises(ValueError, match="GPU tensors"):
            call()
    bf = torch.bfloat16
    cache = ((dict(ks=a["ks"][:4]), "k_scales must be"), (dict(vs=a["vs"].view(torch.int8)), "uint8"),
             (dict(ks=None), "needs k_scales"), (dict(kc=torch.zeros(5, 2, 16, 64, dtype=bf)), "float8_e4m3fn"),
             (dict(table=a["table"][:1]), "block_table"), (dict(kvl=a["kvl"].long()), "kv_lens"),
             (dict(ks=a["ks"].view(torch.uint8).transpose(2, 3).contiguous().transpose(2, 3)), "contiguous in its last"))
    for call in (mx8, tree, accept, append):
        for bad, what in cache:
            with pytest.raises(ValueError, match=what):
                call(**bad)
    for bad, what in ((dict(mask=a["mask"][:5]), "tree_mask"), (dict(mask=a["mask"].int()), "tree_mask"),
                      (dict(mask=torch.zeros(2, 6, dtype=torch.int64).T), "rows must be contiguous"),
                      (dict(q=torch.zeros(6, 7, 64, dtype=bf)), "divide")):
        with pytest.raises(ValueError, match=what):
            tree(**bad)
    for bad, what in ((dict(path=a["path"][:1]), "path"), (dict(path=a["path"].long()), "path"),
                      (dict(path=torch.zeros(4, 2, dtype=torch.int32).T), "rows must be contiguous"),
                      (dict(counts=a["counts"][:1]), "counts"), (dict(cu=a["cu"].long()), "cu_seqlens")):
        with pytest.raises(ValueError, match=what):
            accept(**bad)
    w = torch.zeros(64, dtype=bf)
    for bad, what in ((dict(norm="l2"), "norm must be"), (dict(q_weight=w[:63]), "q_weight"), (dict(q_weight=w.half()), "q_weight"),
                      (dict(q_bias=w), "norm='rms'"), (dict(norm="none", k_weight=w), "norm='none'"),
                      (dict(q_weight=w, k_weight=w.float()), "alike"), (dict(q_weight=torch.zeros(8, 64, dtype=bf), k_weight=w), "alike"),
                      (dict(positions=torch.zeros(3, 6, dtype=torch.int64)), "pair_axis"),
                      (dict(positions=torch.zeros(5, dtype=torch.int64)), "positions"),
                      (dict(pair_axis=torch.zeros(31, dtype=torch.int32)), "pair_axis"), (dict(q=None, q_weight=w), "without q"),
                      (dict(kc=None, vc=None), "scales without"), (dict(v=None), "a cache needs")):
        with pytest.raises(ValueError, match=what):
            append(**bad)
    with pytest.raises(ValueError, match="multiple of 32"):
        _C.mx8_cache(1, 1, 16, 48)


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs the host C++ compiler")
def test_cut_of_a_call_by_its_totals(tmp_path):
    from test_seq_edges import _run_check
    _run_check(tmp_path, "cache_cut_check")


def test_cache_workspace_refusals():
    for bad in ((0, 1, 8, 2, 64, 16, 8), (1, 0, 8, 2, 64, 16, 8), (1, 1, 8, 3, 64, 16, 8), (1, 1, 8, 2, 96, 16, 8),
                (1, 1, 8, 2, 64, 12, 8), (1, 1, 8, 2, 64, 16, 0)):
        with pytest.raises(_C.TxError):
            _C.flash_attn_cache_workspace(*bad)
    assert _C.flash_attn_cache_workspace(4, 4, 8, 2, 64, 16, 8) >= 0


def test_tree_masks():
    m = _C.tree_masks([[-1, 0, 0, 2], [], [-1, -1]])
    assert m.tolist() == [[1], [3], [5], [13], [1], [2]]
    chain = _C.tree_masks([list(range(-1, 69))])
    assert chain.shape == (70, 2) and chain[63].tolist() == [-1, 0] and chain[69].tolist() == [-1, 63]
    assert _C.tree_masks([[-1]], words=3).tolist() == [[1, 0, 0]]
    for bad in ([[0]], [[-1, 1]], [[-2]]):
        with pytest.raises(ValueError):
            _C.tree_masks(bad)
    with pytest.raises(ValueError):
        _C.tree_masks([list(range(-1, 69))], words=1)


def test_the_oracle_s_quantiser_agrees_with_the_type():
    x = torch.randn(64, 64, generator=_gen(1)).double() * torch.exp2(torch.randint(-30, 10, (64, 64), generator=_gen(2)).double())
    for dtype in DTYPES:
        e = _scale_exponents(x, dtype)
        c = _codes(x, e, dtype)
        y = (x.unflatten(-1, (-1, 32)) / torch.exp2(e.double())[..., None]).flatten(-2)
        assert float(y.abs().max()) <= 448
        direct = y.float()
        same = direct.double() == y  # (a division by a power of two is exact unless it underflows)
        assert torch.equal(c[same], direct.to(torch.float8_e4m3fn).double()[same])


# ------------------------------------------------------------------ append
def _normed(x, norm, weight, bias, eps):
    """The norm in 64 bits, and its tolerance in fp32 arithmetic."""
    x, hd = x.double(), x.shape[-1]
    if norm == "none":
        return x, torch.zeros_like(x)
    a = x.abs().mean(-1, keepdim=True)
    y = x - x.mean(-1, keepdim=True) if norm == "layer" else x
    r = 1 / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
    w = weight.double() if weight is not None else torch.ones_like(x)
    y = y * r * w
    tol = (2 * hd + 16) * 2.0**-24 * (1 + a * r) * w.abs() * r * (x.abs() + a)
    if bias is not None:
        y = y + bias.double()
        tol = tol + 2.0**-24 * y.abs()
    return y, tol


def _turned(y, tol, positions, pair_axis, steps, amplitude, interleaved):
    """The turn of 64-bit heads [T, H, hd] by positions (lists per axis), and its tolerance."""
    r = 2 * len(steps)
    turns = [[((int(positions[a][t]) * int(s) + 2**63) % 2**64 - 2**63) / 2.0**64 for s, a in zip(steps, pair_axis)]
             for t in range(y.shape[0])]
    turns = torch.tensor(turns, dtype=torch.float64, device=y.device).view(y.shape[0], 1, r // 2)
    c, s = torch.cos(2 * math.pi * turns) * amplitude, torch.sin(2 * math.pi * turns) * amplitude
    out, err = y.clone(), tol.clone()
    i1, i2 = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = y[..., i1], y[..., i2]
    out[..., i1], out[..., i2] = a * c - b * s, b * c + a * s
    err[..., i1] = err[..., i2] = amplitude * (tol[..., i1] + tol[..., i2] + 2.0**-20 * (a.abs() + b.abs()))
    return out, err


def _check_stored(got, scales, want, tol, dtype, what):
    """Values of 8-bit rows [.., hd] against 64-bit ones: the scale is the smallest that holds the block (up to
    the error of its maximum), every value the nearest code."""
    e = scales.view(torch.uint8).double() - 127
    w, t = want.unflatten(-1, (-1, 32)), tol.unflatten(-1, (-1, 32))
    top, off = w.abs().amax(-1), t.amax(-1)
    assert bool((448 * torch.exp2(e) >= top - off).all()), what
    assert bool(((448 * torch.exp2(e - 1) <= top + off) | (e == LOWEST[dtype])).all()), what
    _same(got, want, tol * (1 + 2.0**-4) + 2.0**-4 * want.abs() + (torch.exp2(e - 10)[..., None] + 0 * w).flatten(-2), what)


APPEND_CASES = [  # hd, rotary, interleaved, q heads, kv heads, page, token-major, norm, per head, fp32 gains, axes, mx8
    (64, 64, False, 8, 8, 16, False, "rms", False, False, 1, False),
    (64, 64, True, 8, 2, 8, True, "layer", True, False, 2, True),
    (128, 128, False, 16, 4, 64, True, "rms", False, True, 3, True),
    (128, 64, True, 4, 1, 32, False, "layer", False, True, 3, False),
    (128, 96, False, 5, 5, 16, False, "rms", True, True, 1, True),
    (64, 20, False, 6, 3, 8, False, "layer", False, False, 2, True),
    (64, 20, True, 6, 3, 16, True, "none", False, False, 1, True),
    (96, 72, False, 4, 2, 16, False, "rms", False, False, 3, True),
    (96, 48, False, 4, 2, 16, True, "layer", True, False, 1, False),
    (8, 2, False, 1, 1, 8, False, "rms", False, False, 1, False),
    (256, 256, True, 2, 1, 128, False, "rms", True, False, 1, True),
    (256, 192, False, 2, 2, 16, False, "layer", False, False, 2, True),
    (120, 48, False, 3, 1, 16, False, "rms", False, False, 1, False),
    (32, 32, False, 3, 3, 8, False, "none", False, False, 2, True),
]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", APPEND_CASES, ids=lambda c: "-".join(str(x) for x in c))
def test_norm_rotary_append(cuda, dtype, case):
    hd, rotary, interleaved, h, hk, page, token_major, norm, per_head, f32, axes, mx = case
    log(f"norm append {case} {dtype}")
    lens, new = [1, 37, 5, 64, 9], [1, 30, 0, 64, 4]
    rows, first, behind = sum(new), 2, 3
    t = first + rows + behind
    if mx:
        _, _, kc, ks, vc, vs, table = _paged8(lens, hk, page, hd, dtype, cuda, 5, token_major)
    else:
        _, _, kc, vc, table = _paged(lens, hk, page, hd, dtype, cuda, 5, token_major, fill=7.0)
        ks = vs = None
    held = [x for x in (kc, vc, ks, vs) if x is not None]
    before = [x.view(torch.uint8).clone() if mx else x.clone() for x in held]
    qkv = _randn((t, h + 2 * hk, hd), dtype, cuda, 1)
    qkv[:, ::2] += 0.5
    q, k, v = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
    kind = torch.float32 if f32 else dtype
    par = {}
    for i, (x, n) in enumerate((("q", h), ("k", hk))):
        shape = (n, hd) if per_head else (hd,)
        if norm != "none":
            par[x + "_weight"] = (1 + 0.2 * torch.randn(shape, generator=_gen(7 + i))).to(cuda, kind)
        if norm == "layer":
            par[x + "_bias"] = (0.3 * torch.randn(shape, generator=_gen(9 + i))).to(cuda, kind)
    steps, amplitude = _C.rotary_steps(rotary, scaling="ramp", factor=4.0, original_len=64, device=cuda)
    at = [p for n, m in zip(lens, new) for p in range(n - m, n)]
    where = torch.randint(-50, 5000, (axes, t), generator=_gen(11))
    pair_axis = [(3 * i + 1) % axes for i in range(rotary // 2)]
    kw = {}
    if axes > 1:
        kw = dict(positions=where.to(cuda), pair_axis=_i32(pair_axis, cuda))
    positions = where[:, first:first + rows].tolist() if axes > 1 else [at]
    out = torch.full((t, h, hd), 3.0, dtype=dtype, device=cuda)
    k_out = torch.full((t, hk, hd), 3.0, dtype=dtype, device=cuda)
    got = _C.norm_rotary_append(q, k, v, steps, _cu(new, cuda, first), norm=norm, eps=1e-5, kv_lens=_i32(lens, cuda),
                                block_table=table, k_cache=kc, v_cache=vc, k_scales=ks, v_scales=vs, q_out=out,
                                k_out=k_out, interleaved=interleaved, amplitude=amplitude, **par, **kw)
    assert got[0] is out and got[1] is k_out
    inner = slice(first, first + rows)
    eps = torch.finfo(dtype).eps
    for name, x, y in (("q", q, out), ("k", k, k_out)):
        want, tol = _normed(x[inner], norm, par.get(name + "_weight"), par.get(name + "_bias"), 1e-5)
        want, tol = _turned(want, tol, positions, pair_axis, steps.tolist(), amplitude, interleaved)
        _same(y[inner], want, eps / 2 * want.abs() + (1 + eps) * tol + 2.0**-25, name)
        assert bool((y[:first] == 3).all()) and bool((y[first + rows:] == 3).all())
    # want, tol: k's.  The rows' slots hold them, nothing else changed.
    page_at = torch.tensor([int(table[b, p // page]) for b, (n, m) in enumerate(zip(lens, new)) for p in range(n - m, n)],
                           device=cuda)
    slot = torch.tensor(at, device=cuda) % page
    if mx:
        kv_ = _values(kc.view(torch.uint8)[page_at, :, slot], ks[page_at, :, slot])
        _check_stored(kv_, ks[page_at, :, slot], want, tol, dtype, "k stored")
        codes, scales, _ = _stored(v[inner], dtype, cuda)
        assert torch.equal(vs[page_at, :, slot], scales)
        assert torch.equal(vc.view(torch.uint8)[page_at, :, slot] & 0x7F, codes & 0x7F)  # (signs of 0 aside)
        assert torch.equal(_values(vc.view(torch.uint8)[page_at, :, slot], scales), _values(codes, scales))
    else:
        assert torch.equal(kc[page_at, :, slot], k_out[inner]) and torch.equal(vc[page_at, :, slot], v[inner])
    for x, old in zip(held, before):
        now = x.view(torch.uint8).clone() if mx else x.clone()
        now[page_at, :, slot] = old[page_at, :, slot]
        assert torch.equal(now, old)


@gpu
@pytest.mark.parametrize("interleaved,rotary", [(False, 64), (True, 64), (False, 20), (True, 20)])
@pytest.mark.parametrize("norm", ["rms", "layer", "none"])
def test_norm_rotary_in_place_and_without_a_cache(cuda, interleaved, rotary, norm):
    dtype, new = torch.float16, [70, 1, 12]
    t = sum(new)
    steps, _ = _C.rotary_steps(rotary, device=cuda)
    buf = _randn((t, 10, 64), dtype, cuda, 3)
    q, k = buf[:, :8], buf[:, 8:]
    q0, k0 = q.clone(), k.clone()
    positions = torch.randint(-(10**6), 10**9, (t,), generator=_gen(4))
    positions[:3] = torch.tensor([0, 2**40 + 1, -(2**62)])
    got = _C.norm_rotary_append(q, k, None, steps, _cu(new, cuda), norm=norm, positions=positions.to(cuda), q_out=q, k_out=k,
                                interleaved=interleaved)
    assert got[0].data_ptr() == q.data_ptr() and got[1].data_ptr() == k.data_ptr()
    for name, x0, x in (("q", q0, q), ("k", k0, k)):
        want, tol = _normed(x0, norm, None, None, 1e-6)
        want, tol = _turned(want, tol, [positions.tolist()], [0] * (rotary // 2), steps.tolist(), 1.0, interleaved)
        _same(x, want, 2.0**-11 * want.abs() + 1.001 * tol + 2.0**-25, name)
    # keys alone, at their places in the sequence
    _, k2 = _C.norm_rotary_append(None, k0, None, steps, _cu(new, cuda), norm=norm, interleaved=interleaved)
    want, tol = _normed(k0, norm, None, None, 1e-6)
    want, tol = _turned(want, tol, [[i for n in new for i in range(n)]], [0] * (rotary // 2), steps.tolist(), 1.0, interleaved)
    _same(k2, want, 2.0**-11 * want.abs() + 1.001 * tol + 2.0**-25, "k alone")


@gpu
def test_without_a_norm_the_append_is_rotary_append(cuda):
    """The same bits for one axis and a 16-bit cache (the same angles, products and roundings)."""
    dtype, hk, hd = torch.bfloat16, 2, 64
    x = _randn((50, 8, hd), dtype, cuda, 12)
    steps, _ = _C.rotary_steps(hd, device=cuda)
    res = []
    for f, kw in ((_C.rotary_append, {}), (_C.norm_rotary_append, {"norm": "none"})):
        _, _, kc, vc, table = _paged([30, 20], hk, 16, hd, dtype, cuda, 5, fill=0.0)
        q, _ = f(x[:, :4], x[:, 4:6], x[:, 6:], steps, _cu([30, 20], cuda), kv_lens=_i32([30, 20], cuda), block_table=table,
                 k_cache=kc, v_cache=vc, **kw)
        res.append((q, kc, vc))
    eps = 2.0**-7  # (a product may be fused with the sum on one side: a step where it is near a tie)
    for a, b in zip(*res):
        assert bool(((a.double() - b.double()).abs() <= eps * a.double().abs() + 1e-6).all())
    assert torch.equal(res[0][2], res[1][2])


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_what_an_8_bit_cache_holds(cuda, dtype):
    """Values of every size, blocks of zeros, the largest values, ties, and what is not finite."""
    hd, page = 64, 16
    big = float(torch.finfo(dtype).max)
    rows = [torch.zeros(hd), torch.full((hd,), big), torch.full((hd,), -big)]
    rows.append(torch.cat([torch.full((32,), 448.0), torch.full((32,), 449.0 if dtype == torch.float16 else 450.0)]))
    tiny = 2.0**-24 if dtype == torch.float16 else 2.0**-133
    rows.append(torch.arange(hd).float() * tiny)
    rows.append(torch.arange(hd).float() / 8 + 8)  # ties between codes
    rows.append(1.0 + torch.arange(hd).float() / 64)
    mixed = torch.randn(20, hd, generator=_gen(5)) * torch.exp2(torch.randint(-14, 15, (20, 1), generator=_gen(6)).float())
    wide = torch.randn(20, hd, generator=_gen(7)) * torch.exp2(torch.randint(-20, 2, (20, hd), generator=_gen(8)).float())
    odd = torch.randn(6, hd, generator=_gen(9))
    for i, x in enumerate((math.nan, math.inf, -math.inf, math.nan, math.inf, -math.inf)):
        odd[i, 7 * i] = x
        odd[i, 33] = x
    x = torch.cat([torch.stack(rows), mixed, wide, odd]).to(dtype)
    n = x.shape[0]
    pages = (n + page - 1) // page
    kc, ks = _C.mx8_cache(pages, 1, page, hd, device=cuda)
    vc, vs = _C.mx8_cache(pages, 1, page, hd, device=cuda)
    steps, _ = _C.rotary_steps(hd, device=cuda)
    dev = x.to(cuda)[:, None]
    _C.norm_rotary_append(None, dev, dev.clone(), steps, _cu([n], cuda), norm="none", kv_lens=_i32([n], cuda),
                          positions=torch.zeros(n, dtype=torch.int64, device=cuda),  # no turn
                          block_table=_i32([list(range(pages))], cuda), k_cache=kc, v_cache=vc, k_scales=ks, v_scales=vs)
    clean = torch.where(torch.isfinite(x), x, torch.zeros_like(x))
    codes, scales, values = _stored(clean, dtype, "cpu")
    bad = ~torch.isfinite(x)
    # an element turned by 0 with a partner that is not finite is not finite either (0 times it); v has no turn
    for name, c, s, lost in (("v", vc, vs, bad), ("k", kc, ks, bad | torch.cat([bad[:, 32:], bad[:, :32]], 1))):
        got = _values(c, s).transpose(1, 2).reshape(-1, hd)[:n].cpu()
        if name == "v":
            assert torch.equal(s.view(torch.uint8).transpose(1, 2).reshape(-1, 2)[:n].cpu(), scales)
        rows_ok = ~lost.any(1) if name == "k" else torch.ones(n, dtype=torch.bool)
        assert bool(torch.isnan(got[lost]).all()) and bool(torch.isfinite(got[~lost]).all())
        ok = ~lost & rows_ok[:, None]
        assert torch.equal(got[ok], values.double()[ok]), name


@gpu
@pytest.mark.parametrize("mx", [False, True])
def test_norm_rotary_append_drops_what_has_no_place(cuda, mx):
    dtype, page, hk = torch.bfloat16, 8, 2
    if mx:
        (kc, ks), (vc, vs) = (_C.mx8_cache(4, hk, page, 64, device=cuda) for _ in range(2))
    else:
        kc, ks, vs = torch.zeros(4, hk, page, 64, dtype=dtype, device=cuda), None, None
        vc = torch.zeros_like(kc)
    table = _i32([[2, -1], [4, 1], [2**31 - 1, 3]], cuda)
    new, lens = [10, 12, 6], [7, 12, 19]  # 3 rows before key 0; page 4 of 4; keys 13..18, 16.. behind the table
    x = _randn((sum(new), 3 * hk, 64), dtype, cuda, 6) + 1.5
    steps, _ = _C.rotary_steps(64, device=cuda)
    _C.norm_rotary_append(x[:, :hk], x[:, hk:2 * hk], x[:, 2 * hk:], steps, _cu(new, cuda), kv_lens=_i32(lens, cuda),
                          block_table=table, k_cache=kc, v_cache=vc, k_scales=ks, v_scales=vs)
    held = torch.zeros(4, page, dtype=torch.bool)
    for b, (n, m) in enumerate(zip(lens, new)):
        for p in range(n - m, n):
            pg = int(table[b, p // page]) if 0 <= p < 2 * page else -1
            if 0 <= pg < 4:
                held[pg, p % page] = True
    for c in [vc, kc] + ([ks, vs] if mx else []):
        some = (c.view(torch.uint8 if mx else torch.int16) != 0).any(-1).any(1).cpu()
        assert torch.equal(some, held)


# --------------------------------------------------------------- attention
def _cache(lens, hk, page, hd, dtype, dev, seed, mx, token_major=False, **kw):
    """(keys, values of each sequence; k, v caches; keyword arguments of their scales; table)"""
    if mx:
        k, v, kc, ks, vc, vs, table = _paged8(lens, hk, page, hd, dtype, dev, seed, token_major, **kw)
        return k, v, kc, vc, dict(k_scales=ks, v_scales=vs), table
    k, v, kc, vc, table = _paged(lens, hk, page, hd, dtype, dev, seed, token_major, **kw)
    return k, v, kc, vc, {}, table


def _mx8(q, kc, vc, sc, table, cu, kvl, scale, causal=True, **kw):
    return _C.flash_attn_paged_mx8(q, kc, sc["k_scales"], vc, sc["v_scales"], table, cu, kvl, scale, causal, **kw)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("h,hk", [(8, 8), (8, 2), (5, 1), (24, 1)])
@pytest.mark.parametrize("page,token_major", [(16, False), (8, True), (256, False)])
def test_paged_mx8(cuda, dtype, hd, h, hk, page, token_major):
    for i, (new, lens) in enumerate(PAGED_CASES):
        causal = i % 3 != 2
        log(f"mx8 {new} over {lens} hd{hd} heads {h}/{hk} page {page} causal={causal} {dtype}")
        ks, vs, kc, vc, sc, table = _cache(lens, hk, page, hd, dtype, cuda, 40 + i, True, token_major)
        first, behind = 1, 2
        t = first + sum(new) + behind
        q = _randn((t, h, hd), dtype, cuda, 50 + i)
        out = torch.full_like(q, 3.0)
        _mx8(q, kc, vc, sc, table, _cu(new, cuda, first), _i32(lens, cuda), hd**-0.5, causal, out=out,
             max_q_len=max(new) if i % 2 else 0)
        at = first
        for b, n in enumerate(new):
            s = slice(at, at + n)
            seen = _causal(n, lens[b], cuda) if causal else torch.ones(n, lens[b], dtype=torch.bool, device=cuda)
            want, tol = _attend(q[s], ks[b], vs[b], hd**-0.5, seen, dtype)
            _same(out[s], want, tol, f"sequence {b}")
            at += n
        assert bool((out[:first] == 3).all()) and bool((out[t - behind:] == 3).all())


@gpu
@pytest.mark.parametrize("hd,h,hk,new,keys", [(128, 16, 4, 1, 20011), (64, 8, 8, 1, 9999), (128, 16, 2, 3, 12345),
                                              (64, 16, 2, 200, 8200), (128, 4, 4, 40, 16385), (128, 16, 4, 700, 5000)])
def test_paged_mx8_long_rows(cuda, hd, h, hk, new, keys):
    """Rows whose keys are shared out over the card and joined, with a key that outweighs the others."""
    dtype = torch.bfloat16
    ks, vs, kc, vc, sc, table = _cache([keys, 70], hk, 64, hd, dtype, cuda, 60, True)
    q = _randn((new + 1, h, hd), dtype, cuda, 61)
    for j in (0, keys // 2, keys - new):
        codes, scales, values = _stored((q[:1, ::h // hk] * 1.5).cpu(), dtype, cuda)
        ks[0][j], pg = values[0], int(table[0, j // 64])
        kc.view(torch.uint8)[pg, :, j % 64], sc["k_scales"][pg, :, j % 64] = codes[0], scales[0]
    got = _mx8(q, kc, vc, sc, table, _cu([new, 1], cuda), _i32([keys, 70], cuda), hd**-0.5, max_q_len=new)
    for b, s in ((0, slice(0, new)), (1, slice(new, new + 1))):
        want, tol = _attend(q[s], ks[b], vs[b], hd**-0.5, _causal(s.stop - s.start, ks[b].shape[0], cuda), dtype)
        _same(got[s], want, tol, f"sequence {b}")


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [2, 40])
def test_scales_far_apart(cuda, dtype, new):
    """Keys and values whose scales span the type's range; e8m0 and uint8 scales alike."""
    hd, h, hk, n = 64, 4, 2, 300
    top = 8 if dtype == torch.float16 else 100
    ks, vs, kc, vc, sc, table = _cache([n], hk, 16, hd, dtype, cuda, 62, True)
    v = torch.randn(n, hk, hd, generator=_gen(63)) * torch.exp2(torch.randint(-top, top, (n, hk, 2), generator=_gen(64)).float()
                                                                .repeat_interleave(32, -1))
    codes, scales, values = _stored(v, dtype, cuda)
    for j in range(n):
        pg = int(table[0, j // 16])
        vc.view(torch.uint8)[pg, :, j % 16], sc["v_scales"][pg, :, j % 16] = codes[j], scales[j]
    q = _randn((new, h, hd), dtype, cuda, 65)
    args = (table, _cu([new], cuda), _i32([n], cuda), 0.125)
    got = _mx8(q, kc, vc, sc, *args)
    want, tol = _attend(q, ks[0], values, 0.125, _causal(new, n, cuda), dtype)
    _same(got, want, tol, "rows")
    e8 = {x: y.view(torch.float8_e8m0fnu) for x, y in sc.items()}
    assert torch.equal(got, _mx8(q, kc, vc, e8, *args))


TREE_CASES = [  # new tokens, keys of each sequence
    ([1], [1]), ([8], [1000]), ([4, 1, 16], [4, 1, 300]), ([43, 0, 7, 64], [500, 0, 129, 64]), ([65, 130], [900, 131]),
    ([3, 20], [2, 9]),  # more new tokens than keys
]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("h,hk", [(8, 8), (8, 2), (5, 1), (24, 1)])
@pytest.mark.parametrize("mx,page,token_major", [(False, 16, False), (True, 16, True), (False, 8, True), (True, 128, False)])
def test_tree_attention(cuda, dtype, hd, h, hk, mx, page, token_major):
    for i, (new, lens) in enumerate(TREE_CASES):
        log(f"tree {new} over {lens} hd{hd} heads {h}/{hk} page {page} mx8={mx} {dtype}")
        ks, vs, kc, vc, sc, table = _cache(lens, hk, page, hd, dtype, cuda, 70 + i, mx, token_major)
        first, behind = 1, 2
        t = first + sum(new) + behind
        trees = [_tree(n, 80 + b, roots=1 + b % 2) for b, n in enumerate(new)]
        words = (max(new) + 63) // 64 + i % 2
        mask = torch.full((t, words + 1), -1, dtype=torch.int64, device=cuda)[:, :words]  # rows with a gap
        mask[first:first + sum(new)] = _C.tree_masks(trees, words=words, device=cuda)
        q = _randn((t, h, hd), dtype, cuda, 90 + i)
        out = torch.full_like(q, 3.0)
        _C.flash_attn_tree(q, kc, vc, table, _cu(new, cuda, first), _i32(lens, cuda), mask, hd**-0.5, out=out,
                           max_q_len=max(new) if i % 2 else 0, **sc)
        at = first
        for b, n in enumerate(new):
            s = slice(at, at + n)
            want, tol = _attend(q[s], ks[b], vs[b], hd**-0.5, _tree_seen(trees[b], lens[b], cuda), dtype)
            _same(out[s], want, tol, f"sequence {b}")
            at += n
        assert bool((out[:first] == 3).all()) and bool((out[t - behind:] == 3).all())


@gpu
@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("hd,new,keys", [(64, 3, 9000), (128, 64, 20000), (128, 200, 4400)])
def test_tree_attention_long_rows(cuda, mx, hd, new, keys):
    dtype, h, hk = torch.bfloat16, 16, 4
    ks, vs, kc, vc, sc, table = _cache([keys, 30], hk, 64, hd, dtype, cuda, 100, mx)
    trees = [_tree(new, 101), _tree(5, 102)]
    q = _randn((new + 5, h, hd), dtype, cuda, 103)
    got = _C.flash_attn_tree(q, kc, vc, table, _cu([new, 5], cuda), _i32([keys, 30], cuda),
                             _C.tree_masks(trees, device=cuda), hd**-0.5, max_q_len=new, **sc)
    for b, s in ((0, slice(0, new)), (1, slice(new, new + 5))):
        want, tol = _attend(q[s], ks[b], vs[b], hd**-0.5, _tree_seen(trees[b], ks[b].shape[0], cuda), dtype)
        _same(got[s], want, tol, f"sequence {b}")


@gpu
@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [3, 40, 600])
def test_tree_rows_that_see_nothing_are_zero(cuda, mx, hd, n):
    """No key before the drafts and no bit: 0, whatever the keys hold; masks of any bits, words that end early."""
    dtype, h, hk = torch.float16, 4, 2
    ks, vs, kc, vc, sc, table = _cache([n], hk, 16, hd, dtype, cuda, 110, mx)
    words = min((n + 63) // 64, 2)  # of 600 tokens only the first 128 can be seen
    bits = torch.randint(-(2**63), 2**63 - 1, (n, words), generator=_gen(111))
    bits[::3] = 0
    q = _randn((n, h, hd), dtype, cuda, 112)
    got = _C.flash_attn_tree(q, kc, vc, table, _cu([n], cuda), _i32([n], cuda), bits.to(cuda), hd**-0.5, **sc)
    seen = torch.zeros(n, n, dtype=torch.bool)
    for j in range(min(n, 64 * words)):
        seen[:, j] = (bits[:, j // 64] >> (j % 64)) & 1 == 1
    want, tol = _attend(q, ks[0], vs[0], hd**-0.5, seen.to(cuda), dtype)
    _same(got, want, tol, "rows")
    assert bool((got[::3] == 0).all())
    for c in (kc, vc):
        (c.view(torch.uint8) if mx else c).fill_(0x7F if mx else math.nan)
    got = _C.flash_attn_tree(q, kc, vc, table, _cu([n], cuda), _i32([n], cuda), bits.to(cuda), hd**-0.5, **sc)
    some = seen.any(1).to(cuda)
    assert bool((got[~some] == 0).all()) and bool(torch.isnan(got[some]).all())


@gpu
@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,m", [(4, 5), (64, 64), (64, 700), (100, 4000)])
def test_what_a_tree_mask_hides_has_no_influence(cuda, mx, hd, n, m):
    """NaN and infinities in the drafts that a row does not see; what it sees makes it NaN."""
    dtype, h, hk = torch.bfloat16, 4, 2
    ks, vs, kc, vc, sc, table = _cache([m], hk, 16, hd, dtype, cuda, 120, mx)
    parents = _tree(n, 121)
    seen = _tree_seen(parents, m, cuda)
    q = _randn((n, h, hd), dtype, cuda, 122)
    args = (table, _cu([n], cuda), _i32([m], cuda), _C.tree_masks([parents], device=cuda), hd**-0.5)
    clean = _C.flash_attn_tree(q, kc, vc, *args, **sc)
    key, val = m - n + n // 2, m - n + (3 * n) // 4
    for c, j, x in ((kc, key, 0), (vc, val, 1)):
        pg, slot = int(table[0, j // 16]), j % 16
        if mx and x == 0:
            sc["k_scales"][pg, 0, slot, 1] = 255
        elif mx:
            c.view(torch.uint8)[pg, 1, slot, 7] = 0xFF
        else:
            c[pg, x, slot, 5 + 2 * x] = math.nan if x == 0 else math.inf
    got = _C.flash_attn_tree(q, kc, vc, *args, **sc)
    g = h // hk
    hit_k, hit_v = seen[:, key], seen[:, val]
    assert bool(torch.isfinite(clean).all()) and bool(torch.isnan(got[:, :g][hit_k]).all())
    d = [i for i in range(hd) if i != 7]
    # Not every bit: rows side by side renew the base that their weights are measured from together, and another base
    # rounds other weights up and down, each by half a step at most as before.
    # Rows that meet 0 times a value that is not finite are formed again, with weights that are rounded after the
    # division by their sum w_j / l, where the first pass rounds w_j and divides the sum of products.  Either way a
    # weight is off by half a step, eps / 2 of p_j, and the result is rounded once, so the tolerance is the same
    # (of its eps A for the weights the second half, for the sum, is not even used), but not every bit is.
    want, tol = _attend(q, ks[0], vs[0], hd**-0.5, seen, dtype)
    _same(got[:, :g][~hit_k], want[:, :g][~hit_k], tol[:, :g][~hit_k], "rows that do not see the key")
    _same(got[:, g:][~hit_v], want[:, g:][~hit_v], tol[:, g:][~hit_v], "rows that do not see it")
    _same(got[:, g:][..., d], want[:, g:][..., d], tol[:, g:][..., d], "other elements")
    assert bool((~torch.isfinite(got[:, g:, 7][hit_v])).all())


@gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [3, 150])
def test_hidden_nan_of_an_8_bit_cache_has_no_influence(cuda, hd, n):
    """Codes and scales that are NaN in keys after a row; what a row sees makes it NaN."""
    dtype, h, hk, m = torch.float16, 4, 2, 160
    ks, vs, kc, vc, sc, table = _cache([m], hk, 16, hd, dtype, cuda, 130, True)
    q = _randn((n, h, hd), dtype, cuda, 131)
    args = (table, _cu([n], cuda), _i32([m], cuda), hd**-0.5)
    clean = _mx8(q, kc, vc, sc, *args)
    last = m - 1
    pg, slot = int(table[0, last // 16]), last % 16
    sc["k_scales"][pg, 0, slot, 0] = 255
    vc.view(torch.uint8)[pg, 1, slot, 9] = 0x7F
    got = _mx8(q, kc, vc, sc, *args)
    assert bool(torch.isfinite(clean).all())
    # (within tolerance, not every bit, as above)
    want, tol = _attend(q, ks[0], vs[0], hd**-0.5, _causal(n, m, cuda), dtype)
    _same(got[:-1], want[:-1], tol[:-1], "rows before it")
    assert bool(torch.isnan(got[-1, :2]).all()) and bool(torch.isnan(got[-1, 2:, 9]).all())
    assert bool(torch.isfinite(got[-1, 2:, :9]).all())


@gpu
@pytest.mark.parametrize("tree,mx", [(False, True), (True, False), (True, True)])
@pytest.mark.parametrize("new,h,hk", [(1, 8, 2), (3, 8, 8), (80, 8, 2)])
def test_pages_outside_the_pool(cuda, tree, mx, new, h, hk):
    dtype, hd, page = torch.float16, 64, 16
    lens, news = [700, 300, 2000], [new, 1, new]
    ks, vs, kc, vc, sc, table = _cache(lens, hk, page, hd, dtype, cuda, 140, mx)
    q = _randn((sum(news), h, hd), dtype, cuda, 141)
    cu, mask = _cu(news, cuda), _C.tree_masks([list(range(-1, n - 1)) for n in news], device=cuda)

    def call(q, table, cu, lens, mask):
        if tree:
            return _C.flash_attn_tree(q, kc, vc, table, cu, _i32(lens, cuda), mask, 0.125, max_q_len=new, **sc)
        return _mx8(q, kc, vc, sc, table, cu, _i32(lens, cuda), 0.125, max_q_len=new)

    good = call(q, table, cu, lens, mask)
    assert not bool(torch.isnan(good).any())
    hole = lens[0] - new + 1 if new > 1 else 5  # the last rows, or all of them, need this key
    hole = hole // page * page
    table[0, hole // page] = kc.shape[0]
    table[2, 1] = -(2**31)
    got = call(q, table, cu, lens, mask)
    need = torch.arange(lens[0] - new, lens[0], device=cuda) >= hole
    assert bool(torch.isnan(got[:new][need]).all()) and torch.equal(got[:new][~need], good[:new][~need])
    assert torch.equal(got[new:new + 1], good[new:new + 1]) and bool(torch.isnan(got[new + 1:]).all())
    # more keys than the table has pages for
    got = call(q[:1], table[1:2, :4].contiguous(), _cu([1], cuda), [65], mask[:1])
    assert bool(torch.isnan(got).all())


@gpu
@pytest.mark.parametrize("mx", [False, True])
def test_a_tree_s_rows_do_not_need_the_pages_they_do_not_see(cuda, mx):
    """A draft without a page makes the rows that see it NaN, and no others."""
    dtype, hd, h, hk, page, n, m = torch.bfloat16, 128, 8, 2, 8, 40, 600
    ks, vs, kc, vc, sc, table = _cache([m], hk, page, hd, dtype, cuda, 145, mx)
    parents = [-1, 0, 1, 2] + [0] * 12 + [4 + i % 4 for i in range(24)]
    q = _randn((n, h, hd), dtype, cuda, 146)
    args = (_cu([n], cuda), _i32([m], cuda), _C.tree_masks([parents], device=cuda), hd**-0.5)
    table[0, (m - n + 8) // page] = -1  # drafts 8 .. 15
    got = _C.flash_attn_tree(q, kc, vc, table, *args, **sc)
    seen = _tree_seen(parents, m, cuda)
    lost = seen[:, m - n + 8:m - n + 16].any(1)
    assert bool(torch.isnan(got[lost]).all())
    want, tol = _attend(q, ks[0], vs[0], hd**-0.5, seen, dtype)
    _same(got[~lost], want[~lost], tol[~lost], "the other rows")


@gpu
@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("new", [1, 5, 90])
def test_a_sequence_does_not_depend_on_the_batch(cuda, mx, new):
    dtype, hd, h, hk = torch.bfloat16, 128, 8, 2
    lens, news = [3000, 17, 2500, 900], [new, 1, 3, 200]
    ks, vs, kc, vc, sc, table = _cache(lens, hk, 16, hd, dtype, cuda, 150, mx)
    q = _randn((sum(news), h, hd), dtype, cuda, 151)
    mask = _C.tree_masks([_tree(n, 152) for n in news], device=cuda)
    cu, kvl = _cu(news, cuda), _i32(lens, cuda)
    calls = [lambda q, table, cu, kvl, mask, most: _C.flash_attn_tree(q, kc, vc, table, cu, kvl, mask, 0.1, max_q_len=most, **sc)]
    if mx:
        calls.append(lambda q, table, cu, kvl, mask, most: _mx8(q, kc, vc, sc, table, cu, kvl, 0.1, max_q_len=most))
    for i, f in enumerate(calls):
        both = f(q, table, cu, kvl, mask, max(news))
        alone = f(q[:new], table[:1], _cu([new], cuda), _i32([3000], cuda), mask[:new], new)
        assert torch.equal(both, f(q, table, cu, kvl, mask, max(news)))
        if new * h // hk <= 16:
            assert torch.equal(both[:new], alone)
            continue
        # more rows: the keys are cut by the call's totals
        seen = _tree_seen(_tree(new, 152), 3000, cuda) if i == 0 else _causal(new, 3000, cuda)
        want, tol = _attend(q[:new], ks[0], vs[0], 0.1, seen, dtype)
        _same(both[:new], want, tol, "in the batch")
        _same(alone, want, tol, "alone")


@gpu
@pytest.mark.parametrize("hint", [1, 2, 3])
@pytest.mark.parametrize("mx", [False, True])
def test_a_bound_that_is_too_small_and_the_workspace(cuda, hint, mx):
    dtype, hd, h, hk = torch.float16, 64, 6, 2
    new, lens = [40, 1, 7, 200], [900, 300, 7, 1500]
    ks, vs, kc, vc, sc, table = _cache(lens, hk, 16, hd, dtype, cuda, 160, mx)
    q = _randn((sum(new), h, hd), dtype, cuda, 161)
    trees = [_tree(n, 162) for n in new]
    need = _C.flash_attn_cache_workspace(sum(new), len(new), h, hk, hd, 16, table.shape[1], hint)
    ws = torch.full((need + 64,), 2.0, device=cuda)
    got = _C.flash_attn_tree(q, kc, vc, table, _cu(new, cuda), _i32(lens, cuda), _C.tree_masks(trees, device=cuda), 0.125,
                             max_q_len=hint, workspace=ws[:need], **sc)
    assert bool((ws[need:] == 2).all())
    at = 0
    for b, n in enumerate(new):
        want, tol = _attend(q[at:at + n], ks[b], vs[b], 0.125, _tree_seen(trees[b], lens[b], cuda), dtype)
        _same(got[at:at + n], want, tol, f"sequence {b}")
        at += n


@gpu
@pytest.mark.parametrize("batch", [65, 130])
def test_many_sequences(cuda, batch):
    dtype, hd, h, hk, page = torch.bfloat16, 64, 4, 2, 16
    new = [(7 * b) % 5 if b % 3 else 1 for b in range(batch)]
    new[batch // 2] = 150
    lens = [n + (37 * b) % 700 for b, n in enumerate(new)]
    ks, vs, kc, vc, sc, table = _cache(lens, hk, page, hd, dtype, cuda, 170, True)
    q = _randn((sum(new), h, hd), dtype, cuda, 171)
    cu, kvl = _cu(new, cuda), _i32(lens, cuda)
    trees = [_tree(n, 172 + b) for b, n in enumerate(new)]
    paged = _mx8(q, kc, vc, sc, table, cu, kvl, 0.125, max_q_len=150)
    treed = _C.flash_attn_tree(q, kc, vc, table, cu, kvl, _C.tree_masks(trees, device=cuda), 0.125, max_q_len=150, **sc)
    at = 0
    for b, n in enumerate(new):
        s = slice(at, at + n)
        for got, seen in ((paged, _causal(n, lens[b], cuda)), (treed, _tree_seen(trees[b], lens[b], cuda))):
            want, tol = _attend(q[s], ks[b], vs[b], 0.125, seen, dtype)
            _same(got[s], want, tol, f"sequence {b}")
        at += n


@gpu
@pytest.mark.parametrize("starts", [[0, 9, 2, 20, 11, 30], [0, 40, 40, -5, 10**9, 30], [7, 3, 1, 0, 0, 0]])
def test_starts_that_do_not_ascend_stay_in_bounds(cuda, starts):
    """No result is promised for such starts but that nothing outside the rows and the slots named is written."""
    dtype, hd, h, hk, batch = torch.bfloat16, 64, 4, 2, 5
    _, _, kc, vc, sc, table = _cache([600] * batch, hk, 16, hd, dtype, cuda, 180, True)
    spare = [p for p in range(kc.shape[0]) if not bool((table == p).any())]
    whole = torch.full((40, h, hd), 3.0, dtype=dtype, device=cuda)
    out, cu, kvl = whole[5:35], _i32(starts, cuda), _i32([600] * batch, cuda)
    x = _randn((30, h + 2 * hk, hd), dtype, cuda, 181)
    mask = torch.full((30, 1), -1, dtype=torch.int64, device=cuda)
    for most in (0, 1):
        ws = torch.full((_C.flash_attn_cache_workspace(30, batch, h, hk, hd, 16, table.shape[1], most) + 64,), 2.0, device=cuda)
        _mx8(x[:, :h], kc, vc, sc, table, cu, kvl, 0.1, max_q_len=most, out=out, workspace=ws[:-64])
        _C.flash_attn_tree(x[:, :h], kc, vc, table, cu, kvl, mask, 0.1, max_q_len=most, out=out, workspace=ws[:-64], **sc)
        assert bool((ws[-64:] == 2).all())
    steps, _ = _C.rotary_steps(hd, device=cuda)
    _C.norm_rotary_append(x[:, :h], x[:, h:h + hk], x[:, h + hk:], steps, cu, kv_lens=kvl, block_table=table, k_cache=kc,
                          v_cache=vc, q_out=out, **sc)
    _C.cache_accept(kc, vc, table, cu, kvl, _i32([[0, 3, 9]] * batch, cuda), _i32([3] * batch, cuda), **sc)
    torch.cuda.synchronize()
    assert bool((whole[:5] == 3).all()) and bool((whole[35:] == 3).all())
    assert bool((kc.view(torch.uint8)[spare] == 0x7F).all()) and bool((sc["v_scales"][spare] == 255).all())


@gpu
def test_8_bit_cache_beyond_32_bit_offsets(cuda):
    """Pages whose byte offset passes 2^32: appended, read, and moved."""
    dtype, hd, hk, page = torch.bfloat16, 128, 4, 64
    pages = (1 << 32) // (hk * page * hd) + 40
    kc, ks = _C.mx8_cache(pages, hk, page, hd, device=cuda)
    vc, vs = _C.mx8_cache(pages, hk, page, hd, device=cuda)
    sc = dict(k_scales=ks, v_scales=vs)
    table = _i32([[pages - 1, pages - 3, 0, pages - 2]], cuda)
    n, h = 200, 8
    x = _randn((n, h + 2 * hk, hd), dtype, cuda, 190)
    steps, _ = _C.rotary_steps(hd, device=cuda)
    cu, kvl = _cu([n], cuda), _i32([n], cuda)
    q, k = _C.norm_rotary_append(x[:, :h], x[:, h:h + hk], x[:, h + hk:], steps, cu, kv_lens=kvl, block_table=table,
                                 k_cache=kc, v_cache=vc, k_out=torch.empty(n, hk, hd, dtype=dtype, device=cuda), **sc)
    at = [(int(table[0, j // page]), j % page) for j in range(n)]
    kk, vv = (torch.stack([_values(c[p, :, s], e.view(torch.uint8)[p, :, s]) for p, s in at]).to(dtype)
              for c, e in ((kc, ks), (vc, vs)))
    assert float((kk.double() - k.double()).norm() / k.double().norm()) < 2.0**-4
    got = _mx8(q, kc, vc, sc, table, cu, kvl, 0.1)
    ref, tol = _attend(q, kk, vv, 0.1, _causal(n, n, cuda), dtype)
    _same(got, ref, tol, "paged")
    few = _mx8(q[-2:], kc, vc, sc, table, _cu([2], cuda), kvl, 0.1)
    _same(few, ref[-2:], tol[-2:], "few rows")
    _C.cache_accept(kc, vc, table, _cu([150], cuda), kvl, _i32([[0, 60, 149]], cuda), _i32([3], cuda), **sc)
    for i, j in ((51, 110), (52, 199)):
        (p, s), want = at[i], vv[j]
        assert torch.equal(_values(vc[p, :, s], vs.view(torch.uint8)[p, :, s]).to(dtype), want)


# ------------------------------------------------------------------ accept
@gpu
@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("hd,hk,page,token_major", [(64, 2, 16, False), (128, 3, 8, True), (96, 24, 32, False), (256, 1, 8, False)])
def test_cache_accept(cuda, mx, hd, hk, page, token_major):
    """Paths that overlap what they move over, paths longer than are read at once, identities, none accepted."""
    dtype = torch.float16
    lens, new = [40, 5, 100, 9, 64, 3], [12, 5, 64, 4, 0, 1]
    paths = [[2, 3, 7, 8, 11], [0, 1, 2, 3, 4], [1] + list(range(3, 64, 2)), [], [], [0]]
    _, _, kc, vc, sc, table = _cache(lens, hk, page, hd, dtype, cuda, 200, mx, token_major)
    held = [kc.view(torch.uint8), vc.view(torch.uint8), *sc.values()] if mx else [kc, vc]
    want = [x.clone() for x in held]
    longest = max(len(p) for p in paths)
    for b, p in enumerate(paths):
        for x, y in zip(held, want):
            for i, f in enumerate(p):
                a, z = lens[b] - new[b] + f, lens[b] - new[b] + i
                y[int(table[b, z // page]), :, z % page] = x[int(table[b, a // page]), :, a % page]
    path = torch.full((len(lens), longest + 2), 1 << 30, dtype=torch.int32)
    for b, p in enumerate(paths):
        path[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
    got = _C.cache_accept(kc, vc, table, _cu(new, cuda, 3), _i32(lens, cuda), path.to(cuda)[:, :longest + 1],
                          _i32([len(p) for p in paths], cuda), **sc)
    assert got.tolist() == [n - m + len(p) for n, m, p in zip(lens, new, paths)]
    for x, y in zip(held, want):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))  # (bits: NaN among them)


@gpu
@pytest.mark.parametrize("mx", [False, True])
def test_cache_accept_stays_in_bounds(cuda, mx):
    """Indices outside the new tokens, counts below 0 or above them, keys before 0 and pages outside the pool."""
    dtype, hd, hk, page = torch.bfloat16, 64, 2, 8
    lens, new = [20, 20, 3, 40], [6, 6, 9, 6]
    _, _, kc, vc, sc, table = _cache(lens, hk, page, hd, dtype, cuda, 210, mx)
    table[1, 2] = kc.shape[0]            # keys 16.. of sequence 1
    table[3] = table[3, :1].clone()      # (a pool's page twice: never reached)
    table[3, 4:] = -1                    # keys 32.. of sequence 3
    held = [kc.view(torch.uint8), vc.view(torch.uint8), *sc.values()] if mx else [kc, vc]
    before = [x.clone() for x in held]
    path = _i32([[-1, 6, 2**31 - 1, -(2**31), 5], [0, 4, 5, 5, 5], [7, 7, 7, 7, 7], [1, 2, 3, 4, 5]], cuda)
    lens_out = torch.full((4,), -9, dtype=torch.int32, device=cuda)
    got = _C.cache_accept(kc, vc, table, _cu(new, cuda), _i32(lens, cuda), path, _i32([100, 5, 2, -3], cuda),
                          lens_out=lens_out, **sc)
    assert got is lens_out and got.tolist() == [19, 19, -4, 34]
    # sequence 0: key 14 + 4 <- key 14 + 5; sequence 1: keys 15, 18 and 19 have none; sequence 2: base -6, to before 0
    want = [x.clone() for x in before]
    for x, y in zip(before, want):
        y[int(table[0, 2]), :, 2] = x[int(table[0, 2]), :, 3]
    for x, y in zip(held, want):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


# ---------------------------------------------------------------- together
def _serve(cuda, dtype, hd, h, hk, page, mx, capture=False):
    """Prompts appended with norms, drafts appended at their depth, attended as trees, a path of them accepted, and
    the next step's single tokens after it; every step's rows against attention over the tokens that are left."""
    prompt, batch = [60, 7, 33], 3
    steps, _ = _C.rotary_steps(hd, device=cuda)
    w = {"q_weight": (1 + 0.1 * torch.randn(hd, generator=_gen(1))).to(cuda, dtype),
         "k_weight": (1 + 0.1 * torch.randn(hd, generator=_gen(2))).to(cuda, dtype)}
    width = 256 // page
    table = torch.randperm(batch * width, generator=_gen(3)).to(torch.int32).view(batch, width).to(cuda)
    pages = batch * width
    if mx:
        (kc, ks), (vc, vs) = (_C.mx8_cache(pages, hk, page, hd, device=cuda) for _ in range(2))
        sc = dict(k_scales=ks, v_scales=vs)
    else:
        kc = torch.full((pages, hk, page, hd), math.nan, dtype=dtype, device=cuda)
        vc, sc = kc.clone(), {}
    keys, vals = [[] for _ in range(batch)], [[] for _ in range(batch)]  # as stored, of the tokens that are left
    lens = [0] * batch

    def stored(b, j):
        p, s = int(table[b, j // page]), j % page
        if mx:
            return tuple(_values(c[p, :, s], e.view(torch.uint8)[p, :, s]).to(dtype) for c, e in ((kc, ks), (vc, vs)))
        return kc[p, :, s].clone(), vc[p, :, s].clone()

    def step(new, trees, seed):
        nonlocal lens
        x = _randn((sum(new), h + 2 * hk, hd), dtype, cuda, seed)
        now = [n + m for n, m in zip(lens, new)]
        cu, kvl = _cu(new, cuda), _i32(now, cuda)
        depth = []
        for b, (n, m) in enumerate(zip(lens, new)):
            d = []
            for i in range(m):
                d.append(i if trees is None else (0 if trees[b][i] < 0 else d[trees[b][i]] + 1))
            depth += [n + y for y in d]
        q, _ = _C.norm_rotary_append(x[:, :h], x[:, h:h + hk], x[:, h + hk:], steps, cu, kv_lens=kvl,
                                     positions=torch.tensor(depth, device=cuda), block_table=table, k_cache=kc, v_cache=vc,
                                     **w, **sc)
        if trees is not None:
            o = _C.flash_attn_tree(q, kc, vc, table, cu, kvl, _C.tree_masks(trees, device=cuda), hd**-0.5,
                                   max_q_len=max(new), **sc)
        elif mx:
            o = _mx8(q, kc, vc, sc, table, cu, kvl, hd**-0.5, max_q_len=max(new))
        else:
            o = _C.flash_attn_paged(q, kc, vc, table, cu, kvl, hd**-0.5, max_q_len=max(new))
        at = 0
        for b, m in enumerate(new):
            fresh = [stored(b, j) for j in range(lens[b], now[b])]
            k = torch.stack(keys[b] + [f[0] for f in fresh]) if keys[b] or fresh else None
            v = torch.stack(vals[b] + [f[1] for f in fresh])
            seen = _causal(m, now[b], cuda) if trees is None else _tree_seen(trees[b], now[b], cuda)
            want, tol = _attend(q[at:at + m], k, v, hd**-0.5, seen, dtype)
            _same(o[at:at + m], want, tol, f"sequence {b}")
            at += m
            if trees is None:
                keys[b] += [f[0] for f in fresh]
                vals[b] += [f[1] for f in fresh]
        if trees is None:
            lens = now
            return
        paths = []
        for b, t in enumerate(trees):
            path, i = [], len(t) - 1 - b % 2
            while i >= 0:
                path.append(i)
                i = t[i]
            path.reverse()
            paths.append(path)
            fresh = [stored(b, lens[b] + i) for i in path]
            keys[b] += [f[0] for f in fresh]
            vals[b] += [f[1] for f in fresh]
        most = max(len(p) for p in paths)
        left = _C.cache_accept(kc, vc, table, cu, kvl, _i32([p + [-1] * (most - len(p)) for p in paths], cuda),
                               _i32([len(p) for p in paths], cuda), **sc)
        lens = [n + len(p) for n, p in zip(lens, paths)]
        assert left.tolist() == lens

    step(prompt, None, 300)
    for i in range(3):
        new = [9, 17 + i, 4]
        step(new, [_tree(n, 310 + 10 * i + b) for b, n in enumerate(new)], 320 + i)
        step([1, 1, 1], None, 330 + i)


@gpu
@pytest.mark.parametrize("dtype,hd,h,hk,page,mx", [(torch.bfloat16, 128, 8, 2, 16, True), (torch.float16, 64, 8, 8, 32, True),
                                                   (torch.float16, 128, 6, 3, 8, False), (torch.bfloat16, 64, 4, 1, 64, False)])
def test_drafting_in_turn(cuda, dtype, hd, h, hk, page, mx):
    _serve(cuda, dtype, hd, h, hk, page, mx)


@gpu
@pytest.mark.parametrize("mx", [False, True])
def test_one_captured_step_serves_other_lengths(cuda, mx):
    """A captured append, tree attention, accept and single-token attention, replayed after lengths, trees and inputs
    changed, beside a second graph of the same workspace and eager calls; every replay equals the eager result."""
    dtype, hd, h, hk, page, batch, n = torch.bfloat16, 128, 8, 2, 16, 3, 20
    lens = [700, 33, 1500]
    steps, _ = _C.rotary_steps(hd, device=cuda)
    _, _, kc, vc, sc, table = _cache([m + 60 for m in lens], hk, page, hd, dtype, cuda, 220, mx)
    held = [kc.view(torch.uint8), vc.view(torch.uint8), *sc.values()] if mx else [kc, vc]
    for x in held:
        x.fill_(0x20 if mx else 0.5)
    start = [x.clone() for x in held]
    cu, cu1 = _cu([n] * batch, cuda), _cu([1] * batch, cuda)
    kvl, path, counts = _i32(lens, cuda), torch.zeros(batch, 4, dtype=torch.int32, device=cuda), _i32([1] * batch, cuda)
    x = _randn((batch * n, h + 2 * hk, hd), dtype, cuda, 221)
    mask = torch.zeros(batch * n, 1, dtype=torch.int64, device=cuda)
    need = [f(t, batch, h, hk, hd, page, table.shape[1], m) for t, m in ((batch * n, n), (batch, 1))
            for f in (_C.flash_attn_cache_workspace, _C.flash_attn_paged_workspace)]
    ws = torch.empty(max(need), device=cuda)

    def step():
        q, _ = _C.norm_rotary_append(x[:, :h], x[:, h:h + hk], x[:, h + hk:], steps, cu, kv_lens=kvl, block_table=table,
                                     k_cache=kc, v_cache=vc, **sc)
        o = _C.flash_attn_tree(q, kc, vc, table, cu, kvl, mask, hd**-0.5, max_q_len=n, workspace=ws, **sc)
        left = _C.cache_accept(kc, vc, table, cu, kvl, path, counts, **sc)
        if mx:
            one = _mx8(q[:batch], kc, vc, sc, table, cu1, left, hd**-0.5, max_q_len=1, workspace=ws)
        else:
            one = _C.flash_attn_paged(q[:batch], kc, vc, table, cu1, left, hd**-0.5, max_q_len=1, workspace=ws)
        return o, left, one

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
        x.copy_(_randn(x.shape, dtype, cuda, 230 + i))
        kvl.copy_(_i32([m + i * (b + 1) + n for b, m in enumerate(lens)], cuda))
        mask.copy_(_C.tree_masks([_tree(n, 240 + i + b) for b in range(batch)], device=cuda))
        path.copy_(_i32([[0, 1, 5 + i, 10 + b] for b in range(batch)], cuda))
        counts.copy_(_i32([1 + (i + b) % 4 for b in range(batch)], cuda))
        res = []
        for run in (lambda: (graphs[i % 2].replay(), outs[i % 2])[1], step):
            for y, z in zip(held, start):
                y.copy_(z)
            got = [y.clone() for y in run()] + [y.clone() for y in held]
            torch.cuda.synchronize()
            res.append(got)
        for a, b in zip(*res):
            assert torch.equal(a, b), i


@gpu
def test_calls_on_two_streams_at_once_and_recorded(cuda):
    dtype, hd, h, hk = torch.float16, 64, 8, 2
    ks, vs, kc, vc, sc, table = _cache([5000, 400], hk, 32, hd, dtype, cuda, 250, True)
    cu, kvl = _cu([1, 6], cuda), _i32([5000, 400], cuda)
    mask = _C.tree_masks([_tree(1, 1), _tree(6, 2)], device=cuda)
    qs = [_randn((7, h, hd), dtype, cuda, 251 + i) for i in range(2)]
    calls = [lambda q: _mx8(q, kc, vc, sc, table, cu, kvl, 0.125),
             lambda q: _C.flash_attn_tree(q, kc, vc, table, cu, kvl, mask, 0.125, **sc)]
    want = [f(q) for f, q in zip(calls, qs)]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in qs], [[], []]
    for _ in range(10):
        for f, q, s, o in zip(calls, qs, streams, outs):
            with torch.cuda.stream(s):
                o.append(f(q))
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert all(torch.equal(w, x) for x in o)
    steps, _ = _C.rotary_steps(hd, device=cuda)
    with _C.record_launches() as made:
        res = [calls[0](qs[0]), calls[1](qs[0]), _C.norm_rotary_append(qs[0], qs[1][:, :2], None, steps, cu)[0]]
        lens = _C.cache_accept(kc, vc, table, cu, kvl, _i32([[0], [0]], cuda), _i32([1, 1], cuda), **sc)
    assert [c.info["op"] for c in made] == ["flash_attn_paged_mx8", "flash_attn_tree", "norm_rotary_append", "cache_accept"]
    want = [o.clone() for o in res]
    for o in res:
        o.zero_()
    for c in made:
        c()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(res, want)) and lens.tolist() == [5000, 395]


@gpu
def test_nothing_to_do(cuda):
    bf = torch.bfloat16
    kc, ks = _C.mx8_cache(1, 2, 16, 64, device=cuda)
    vc, vs = _C.mx8_cache(1, 2, 16, 64, device=cuda)
    sc = dict(k_scales=ks, v_scales=vs)
    table = torch.zeros(2, 1, dtype=torch.int32, device=cuda)
    cu, kvl = _cu([0, 0], cuda), _i32([0, 9], cuda)
    q = torch.empty(0, 8, 64, dtype=bf, device=cuda)
    none = torch.empty(0, 1, dtype=torch.int64, device=cuda)
    assert _mx8(q, kc, vc, sc, table, cu, kvl, 0.1).shape == (0, 8, 64)
    assert _C.flash_attn_tree(q, kc, vc, table, cu, kvl, none, 0.1, **sc).shape == (0, 8, 64)
    # sequences that bring nothing, among rows of none
    q = torch.ones(3, 8, 64, dtype=bf, device=cuda)
    out = torch.full_like(q, 5.0)
    _mx8(q, kc, vc, sc, table, cu, kvl, 0.1, out=out)
    _C.flash_attn_tree(q, kc, vc, table, cu, kvl, torch.zeros(3, 1, dtype=torch.int64, device=cuda), 0.1, out=out, **sc)
    assert bool((out == 5).all())
    assert _C.cache_accept(kc, vc, table, cu, kvl, torch.zeros(2, 1, dtype=torch.int32, device=cuda), _i32([1, 1], cuda),
                           **sc).tolist() == [0, 9]
    assert _C.cache_accept(kc, vc, table[:0], _cu([], cuda), kvl[:0], torch.zeros(0, 1, dtype=torch.int32, device=cuda), kvl[:0],
                           **sc).shape == (0,)


@gpu
def test_numbers_of_any_kind_and_axes_that_are_not_there(cuda):
    dtype, hd = torch.float16, 64
    _, _, kc, vc, sc, table = _cache([70], 2, 16, hd, dtype, cuda, 260, True)
    q = _randn((3, 4, hd), dtype, cuda, 261)
    args = (table, _cu([3], cuda), _i32([70], cuda))
    mask = _C.tree_masks([[-1, 0, 0]], device=cuda)
    for one in (torch.tensor(0.125), Fraction(1, 8)):
        assert torch.equal(_mx8(q, kc, vc, sc, *args, one), _mx8(q, kc, vc, sc, *args, 0.125))
        assert torch.equal(_C.flash_attn_tree(q, kc, vc, *args, mask, one, **sc), _C.flash_attn_tree(q, kc, vc, *args, mask, 0.125, **sc))
    steps, _ = _C.rotary_steps(hd, device=cuda)
    pos = torch.tensor([[5, 6, 7], [100, 2, 9]], dtype=torch.int64, device=cuda)

    def turned(axes, **kw):
        return _C.norm_rotary_append(q, q[:, :2], None, steps, _cu([3], cuda), positions=pos, pair_axis=_i32(axes, cuda), **kw)

    want = turned([0] * 16 + [1] * 16, eps=0.5, amplitude=0.25)
    for kw in (dict(eps=torch.tensor(0.5), amplitude=torch.tensor(0.25)), dict(eps=Fraction(1, 2), amplitude=Fraction(1, 4))):
        got = turned([-7] * 15 + [-(2**31), 2**31 - 1] + [2] * 15, **kw)  # cut to the axes that there are
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@gpu
@pytest.mark.parametrize("mx", [False, True])
def test_an_accepted_token_named_twice(cuda, mx):
    """Slots that no move has written yet may be read again: both places get it."""
    dtype, hd, n, last = torch.bfloat16, 64, 12, 40
    _, _, kc, vc, sc, table = _cache([last], 2, 16, hd, dtype, cuda, 270, mx)
    at = lambda c, j: c.view(torch.uint8)[int(table[0, j // 16]), :, j % 16].clone()  # noqa: E731
    path = [3, 3, 9, 9, 9, 5, 6, 7, 11, 11]
    held = [kc, vc, *sc.values()]
    old = [[at(c, j) for j in range(last)] for c in held]
    lens = _C.cache_accept(kc, vc, table, _cu([n], cuda), _i32([last], cuda), _i32([path], cuda), _i32([len(path)], cuda), **sc)
    assert lens.tolist() == [last - n + len(path)]
    for c, was in zip(held, old):
        for j in range(last):
            i = j - (last - n)
            assert torch.equal(at(c, j), was[last - n + path[i]] if 0 <= i < len(path) else was[j]), j
