"""Edges of attention over packed sequences and over a paged cache: rows without keys, values that are not
finite, very long caches, workspaces.  Oracle and tolerances of finite elements are test_seq_ops's."""

import math

import shutil

import pytest
import torch

from transformer_optimization_amd import _C
from _util import log
from test_limits import _run_check
from test_seq_ops import _Abi, _attend, _cu, _i32, _paged, _randn, _same

DTYPES = [torch.bfloat16, torch.float16]
gpu = pytest.mark.gpu


# -------------------------------------------------------- rows without keys
@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("h,hk,new,keys", [(2, 2, 4, 1), (4, 4, 9, 3), (8, 2, 40, 25), (6, 2, 150, 70), (4, 1, 1100, 1030)])
def test_a_row_that_sees_no_key_is_zero_whatever_the_keys_hold(cuda, dtype, hd, h, hk, new, keys):
    """Fewer keys than new tokens: the first rows see none.  Keys and values of the later rows are not finite;
    the last shape's keys are shared out over the card."""
    ks, vs, kc, vc, table = _paged([keys], hk, 16, hd, dtype, cuda, 200)
    q = _randn((new, h, hd), dtype, cuda, 201)
    args = (table, _cu([new], cuda), _i32([keys], cuda), hd**-0.5)
    clean = _C.flash_attn_paged(q, kc, vc, *args)
    for cache, what in ((vc, math.nan), (vc, math.inf), (kc, math.nan)):
        good = cache.clone()
        for j in {0, keys // 2, keys - 1}:
            cache[int(table[0, j // 16]), :, j % 16] = what
        got = _C.flash_attn_paged(q, kc, vc, *args)
        log(f"no keys: {new} rows over {keys}, {h}/{hk} hd{hd} {dtype} {what}")
        assert bool((got[:new - keys] == 0).all())
        assert not bool(torch.isfinite(got[new - keys:]).any())
        cache.copy_(good)
    assert torch.equal(_C.flash_attn_paged(q, kc, vc, *args), clean)


# ------------------------------------------------ values that are not finite
def _ieee(q, k, v, scale, causal, dtype):
    """The formula in 64 bits with IEEE arithmetic over the keys that a row sees: an infinity stays one unless it meets
    its opposite, a weight of 0 (a score of -inf) or a NaN.  The tolerance of finite elements as _attend's, over the
    finite products."""
    n, h, d = q.shape
    m, hk = k.shape[:2]
    out = torch.zeros(n, h, d, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    eps = torch.finfo(dtype).eps
    seen = torch.ones(n, m, dtype=torch.bool, device=q.device)
    if causal:
        seen = seen.tril(m - n)
    for x in range(h):
        qx, kx, vx = q[:, x].double(), k[:, x // (h // hk)].double(), v[:, x // (h // hk)].double()
        products = torch.stack([(qx[i] * kx).sum(1) for i in range(n)]) if n * m < 1 << 16 else qx @ kx.T
        s = torch.where(seen, products * scale, torch.full_like(products, -math.inf))
        top = s.amax(1, keepdim=True)  # NaN where any is
        p = torch.where(seen, torch.exp(s - top), torch.zeros_like(s))
        total = torch.where(seen.any(1), p.sum(1), torch.ones_like(p[:, 0]))[:, None]
        finite = torch.isfinite(vx)
        clean = vx.masked_fill(~finite, 0.0)
        o = (p / total) @ clean
        # what each bad key adds, key by key
        for j in (~finite).any(1).nonzero().flatten().tolist():
            o = o + torch.where(seen[:, j, None], p[:, j, None] * vx[j].masked_fill(finite[j], 0.0), torch.zeros_like(o))
        o = torch.where(seen.any(1)[:, None], o, torch.zeros_like(o))
        size = torch.where(seen, (qx.abs() @ kx.abs().nan_to_num(0.0, 0.0, 0.0).T) * scale, torch.zeros_like(s))
        big = size.nan_to_num(0.0, 0.0, 0.0).amax(1, keepdim=True)
        a = (p / total).nan_to_num(0.0) @ clean.abs()
        if dtype == torch.float16:
            a = a + 2.0**-25 / eps * (seen.double() @ clean.abs()) / total.nan_to_num(1.0)
        out[:, x] = o
        tol[:, x] = eps / 2 * o.abs() + a * (eps + 2 * (d + 8) * 2.0**-24 * big + 2 * m * 2.0**-24) + 2.0**-25
    return out, tol


def _strictly_same(got, want, tol, what):
    """NaN where the formula gives NaN, the same infinities, and finite elements within their tolerance."""
    got = got.double()
    for name, f in (("NaN", torch.isnan), ("+inf", torch.isposinf), ("-inf", torch.isneginf)):
        g, w = f(got), f(want)
        assert torch.equal(g, w), f"{what}: {name} at {int((g & ~w).sum())} more and {int((w & ~g).sum())} fewer elements"
    ok = torch.isfinite(want)
    over = ((got - want).abs() - tol)[ok]
    log(f"  {what}: {int((~ok).sum())} of {ok.numel()} not finite, largest excess {float(over.max()) if over.numel() else 0:.3e}")
    assert not over.numel() or float(over.max()) <= 0, what


def _spoil(x, seed, count, values):
    """`count` elements of x [n, heads, hd] at random places, and one in each of the first and last row."""
    n, h, d = x.shape
    at = torch.randint(0, n * h * d, (count,), generator=torch.Generator("cpu").manual_seed(seed)).tolist()
    at += [3, n * h * d - 1]
    for i, j in enumerate(at):
        x.view(-1)[j] = values[i % len(values)]


SPOILS = [  # bad elements of v, of k, whether of q
    ((1, [math.nan]), None, False), ((3, [math.inf]), None, False), ((40, [math.inf, -math.inf, math.nan, math.inf]), None, False),
    (None, (2, [math.nan]), False), (None, (3, [math.inf, -math.inf]), False),
    ((6, [-math.inf, math.inf]), (2, [-math.inf]), False), (None, None, True), ((2, [math.inf]), None, True),
]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("h,hk", [(4, 4), (4, 1), (6, 2)])
@pytest.mark.parametrize("causal", [False, True])
def test_packed_attention_of_values_that_are_not_finite(cuda, dtype, hd, h, hk, causal):
    for i, (vs, ks, in_q) in enumerate(SPOILS):
        for lens in ([150], [5, 1, 90], [333]):
            t = sum(lens)
            q, k, v = (_randn((t, x, hd), dtype, cuda, 220 + i) for i, x in enumerate((h, hk, hk)))
            if vs:
                _spoil(v, i, *vs)
            if ks:
                _spoil(k, i + 50, *ks)
            if in_q:
                q[t // 2, 0, 1], q[t - 1, h - 1, 0] = math.nan, math.inf
            got = _C.flash_attn_packed(q, k, v, _cu(lens, cuda), hd**-0.5, causal)
            at = 0
            for n in lens:
                r = slice(at, at + n)
                want, tol = _ieee(q[r], k[r], v[r], hd**-0.5, causal, dtype)
                _strictly_same(got[r], want, tol, f"{i}: {n} of {lens}, {h}/{hk} hd{hd} {dtype}")
                at += n


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("h,hk,new,keys", [(4, 2, 1, 90), (4, 2, 3, 400), (4, 2, 7, 5000), (4, 1, 1, 9000), (4, 2, 40, 300),
                                           (4, 1, 60, 5000), (2, 2, 150, 150), (6, 2, 5, 3)])
def test_paged_attention_of_values_that_are_not_finite(cuda, dtype, hd, h, hk, new, keys):
    """Few rows and tiles, keys whole and in parts, fewer keys than tokens."""
    for i, (vs, ks, in_q) in enumerate(SPOILS):
        k, v, kc, vc, table = _paged([keys], hk, 16, hd, dtype, cuda, 230 + i)
        k, v = k[0], v[0]
        q = _randn((new, h, hd), dtype, cuda, 231)
        if vs:
            _spoil(v, i, *vs)
        if ks:
            _spoil(k, i + 50, *ks)
        if in_q:
            q[new // 2, 0, 1], q[new - 1, h - 1, 0] = math.nan, math.inf
        j = torch.arange(keys, device=cuda)
        for c, x in ((kc, k), (vc, v)):
            c[table[0, j // 16].long(), :, j % 16] = x
        for causal in (True, False):
            got = _C.flash_attn_paged(q, kc, vc, table, _cu([new], cuda), _i32([keys], cuda), hd**-0.5, causal)
            want, tol = _ieee(q, k, v, hd**-0.5, causal, dtype)
            _strictly_same(got, want, tol, f"{i}: {new} over {keys}, {h}/{hk} hd{hd} causal={causal} {dtype}")


@gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,keys", [(1, 40), (3, 5000), (200, 200), (40, 5000)])
def test_values_near_the_end_of_the_range_do_not_overflow(cuda, hd, new, keys):
    """bf16 values whose sums, weighted but not yet normalised, pass fp32's range."""
    dtype, h, hk = torch.bfloat16, 4, 2
    k, v, kc, vc, table = _paged([keys], hk, 16, hd, dtype, cuda, 240)
    v[0].copy_((v[0].float().abs().clamp(max=1) * 0.5 + 2.5) * 1e38)
    j = torch.arange(keys, device=cuda)
    vc[table[0, j // 16].long(), :, j % 16] = v[0]
    q = _randn((new, h, hd), dtype, cuda, 241)
    want, tol = _ieee(q, k[0], v[0], hd**-0.5, True, dtype)
    got = _C.flash_attn_paged(q, kc, vc, table, _cu([new], cuda), _i32([keys], cuda), hd**-0.5)
    _strictly_same(got, want, tol, f"paged {new} over {keys} hd{hd}")
    if new == keys:
        got = _C.flash_attn_packed(q, k[0], v[0], _cu([new], cuda), hd**-0.5, True)
        _strictly_same(got, want, tol, f"packed {new} hd{hd}")


@gpu
@pytest.mark.parametrize("hd", [64, 128])
def test_an_infinity_with_a_weight_too_small_for_16_bits_is_seen(cuda, hd):
    """Weights from 2^-8 to 2^-80 of the largest (below 2^-40 they round to 0 in fp16): the elements are infinite all
    the same, in one token's rows and in a tile's."""
    dtype, n = torch.float16, 100
    k = torch.zeros(n, 1, hd, dtype=dtype, device=cuda)
    k[:, 0, 0] = torch.arange(n, device=cuda) * 0.5
    v = _randn((n, 1, hd), dtype, cuda, 270)
    v[20:60:5, 0, 7] = math.inf
    v[30, 0, 9] = -math.inf
    q = torch.zeros(n, 4, hd, dtype=dtype, device=cuda)
    q[..., 0] = 1.0
    want, tol = _ieee(q, k, v, 1.0, True, dtype)
    assert bool(torch.isinf(want[:, :, 7]).any()) and not bool(torch.isnan(want).any())
    _strictly_same(_C.flash_attn_packed(q, k, v, _cu([n], cuda), 1.0, True), want, tol, "packed")
    kc, vc = (torch.zeros(7, 1, 16, hd, dtype=dtype, device=cuda) for _ in range(2))
    kc.view(-1, hd)[:n], vc.view(-1, hd)[:n] = k[:, 0], v[:, 0]
    table = torch.arange(7, dtype=torch.int32, device=cuda)[None]
    for new in (1, 3, n):
        got = _C.flash_attn_paged(q[n - new:], kc, vc, table, _cu([new], cuda), _i32([n], cuda), 1.0)
        _strictly_same(got, want[n - new:], tol[n - new:], f"paged {new}")


@gpu
def test_captured_calls_meet_values_that_are_not_finite(cuda):
    """Graphs captured over finite values, replayed over others: every replay equals the eager call."""
    dtype, hd, h, hk, n = torch.bfloat16, 128, 8, 2, 1500
    q, k, v = (_randn((n, x, hd), dtype, cuda, 280 + i) for i, x in enumerate((h, hk, hk)))
    _, _, kc, vc, table = _paged([n], hk, 16, hd, dtype, cuda, 283)
    cu, cu1, cu90, kvl = _cu([n], cuda), _cu([1], cuda), _cu([90], cuda), _i32([n], cuda)

    def step():
        return [_C.flash_attn_packed(q, k, v, cu, hd**-0.5, True),
                _C.flash_attn_paged(q[-1:], kc, vc, table, cu1, kvl, hd**-0.5, max_q_len=1),
                _C.flash_attn_paged(q[-90:], kc, vc, table, cu90, kvl, hd**-0.5)]

    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step()
    for i, (what, at) in enumerate(((0.5, 3), (math.inf, 3), (math.nan, n - 1), (-math.inf, n - 2), (1.0, 7))):
        for c in (v, k) if i % 2 else (v,):
            c[at, 0, 11] = what
        vc[table[0, at // 16].long(), 0, at % 16, 5] = what
        g.replay()
        torch.cuda.synchronize()
        for got, want in zip(outs, step()):
            assert torch.equal(got.view(torch.int16), want.view(torch.int16)), i


def _time_us(fn):
    for _ in range(3):
        fn()
    times = []
    for _ in range(7):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        fn()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) * 1e3)
    return min(times)


@gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("where", ["v first", "k first", "v last", "k last", "q"])
def test_rows_that_are_not_finite_take_about_the_time_of_others(cuda, hd, where):
    """One bad element: of the first token, which most rows see (twice a clean call's time at most, and 50 us for what
    launches of these sizes vary by), or of the last one's.  That is hidden from rows of a few waves, each of which goes
    through all keys by itself, for two groups of rows: n / 64 looks of hd / 8 loads, then n / 32 steps of 5 hd / 8 (hd / 2
    of values, hd / 8 of keys and q).  Each look and step waits 1 us for a few dependent loads at most, and its loads
    take 32 ns each (64 addresses at 2 a ns): (2 n / 64) (1 + hd / 8 * 0.032) + (2 n / 32) (1 + 5 hd / 8 * 0.032) us more
    than a clean call, 0.7 ms at head dim 64 and 1.1 at 128 (one row after another: 16 to 22)."""
    dtype, n, h, hk = torch.float16, 4096, 8, 2
    q, k, v = (_randn((n, x, hd), dtype, cuda, 250 + i) for i, x in enumerate((h, hk, hk)))
    _, _, kc, vc, table = _paged([n], hk, 16, hd, dtype, cuda, 253)
    j = torch.arange(n, device=cuda)

    def fill():
        for c, x in ((kc, k), (vc, v)):
            c[table[0, j // 16].long(), :, j % 16] = x

    fill()
    cu, kvl = _cu([n], cuda), _i32([n], cuda)
    calls = {"packed": lambda: _C.flash_attn_packed(q, k, v, cu, hd**-0.5, True),
             "packed, all visible": lambda: _C.flash_attn_packed(q, k, v, cu, hd**-0.5, False),
             "chunk": lambda: _C.flash_attn_paged(q[-300:], kc, vc, table, _cu300, kvl, hd**-0.5),
             "token": lambda: _C.flash_attn_paged(q[-1:], kc, vc, table, _cu1, kvl, hd**-0.5, max_q_len=1)}
    _cu300, _cu1 = _cu([300], cuda), _cu([1], cuda)
    clean = {name: _time_us(f) for name, f in calls.items()}
    x = {"v": v, "k": k, "q": q}[where[0]]
    x[0 if where.endswith("first") else n - 1, 0, 5] = math.nan if x is q else math.inf
    fill()
    walk = 2 * n / 64 * (1 + hd / 8 * 0.032) + 2 * n / 32 * (1 + 5 * hd / 8 * 0.032)
    took = {name: _time_us(f) for name, f in calls.items()}
    for name in calls:
        log(f"  {where} hd{hd} {name}: {clean[name]:.1f} us clean, {took[name]:.1f} us")
    for name in calls:
        assert took[name] <= (2 * clean[name] + 50 if where.endswith("first") else clean[name] + walk), name


# -------------------------------------------------- as many parts as there are
@pytest.mark.skipif(shutil.which("g++") is None, reason="needs the host C++ compiler")
def test_cut_of_a_paged_call(tmp_path):
    _run_check(tmp_path, "seq_cut_check")


@gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("h,new,keys", [(16, 2, 200000), (24, 1, 200000), (8, 4, 262144), (64, 2, 131584), (16, 1, 300001),
                                        (16, 9, 270000)])
def test_one_kv_head_over_a_very_long_cache(cuda, hd, h, new, keys):
    """One K/V head alone on the card: its keys go out in as many parts as the join takes, whatever their
    number; most of the weight lies on a key of a late part."""
    dtype, page = torch.bfloat16, 256
    ks, vs, kc, vc, table = _paged([keys], 1, page, hd, dtype, cuda, 210)
    q = _randn((new, h, hd), dtype, cuda, 211)
    for j in (0, keys * 3 // 4, keys - new - 3):
        x = q[:1, j % h] * 1.5
        ks[0][j] = x[0]
        kc[int(table[0, j // page]), :, j % page] = x[0]
    got = _C.flash_attn_paged(q, kc, vc, table, _cu([new], cuda), _i32([keys], cuda), hd**-0.5, max_q_len=new)
    want, tol = _attend(q, ks[0], vs[0], hd**-0.5, True, dtype)
    _same(got, want, tol, f"{new} tokens, {h}/1 heads, {keys} keys, hd{hd}")


# -------------------------------------------------------------- workspaces
@pytest.mark.skipif(shutil.which("g++") is None, reason="needs the host C++ compiler")
def test_spans_among_blocks(tmp_path):
    _run_check(tmp_path, "seq_spans_check")


@pytest.mark.parametrize("ws", [
    5 << 20, (5 << 20) + 63 * 1024, (5 << 20) - 16,     # q, its last row, just before it
    1 << 33, (1 << 33) + 31 * 4096, 1 << 34,            # the caches
    6 << 20, (6 << 20) - 16, 7 << 20, 8 << 20, (8 << 20) + 4 * 64,  # starts, lengths, the table and its last row
    3 << 30, 16 + (3 << 30),                            # the output
])
def test_a_workspace_may_not_be_an_argument(ws):
    sizes = dict(np=32, ps=16, mp=64, ld=64)
    assert _C.flash_attn_paged_workspace(64, 2, 8, 2, 64, 16, 64) > 4
    assert _Abi().paged(q=5 << 20, cu=6 << 20, kvl=7 << 20, table=8 << 20, ws=ws, **sizes) == _C.TX_EINVAL


@gpu
@pytest.mark.parametrize("hd,h,hk,new,lens", [
    (128, 16, 4, [1] * 20 + [150], [3000] * 21), (64, 8, 8, [1] * 9 + [300, 40], [5000] * 11), (128, 8, 1, [17], [40000]),
    (64, 16, 1, [2, 1, 9], [30000, 70, 9000]), (128, 4, 4, [1, 1, 1], [9000, 1, 700]), (64, 6, 2, [5, 6, 40], [2000, 2000, 2000]),
])
@pytest.mark.parametrize("hint", [False, True])
def test_a_call_stays_within_the_workspace_it_asks_for(cuda, hd, h, hk, new, lens, hint):
    dtype, page = torch.bfloat16, 64
    ks, vs, kc, vc, table = _paged(lens, hk, page, hd, dtype, cuda, 260)
    q = _randn((sum(new), h, hd), dtype, cuda, 261)
    most = max(new) if hint else 0
    need = _C.flash_attn_paged_workspace(sum(new), len(new), h, hk, hd, page, table.shape[1], most)
    ws = torch.full((need + 4096,), 2.0, device=cuda)
    got = _C.flash_attn_paged(q, kc, vc, table, _cu(new, cuda), _i32(lens, cuda), hd**-0.5, max_q_len=most,
                              workspace=ws[:need])
    assert bool((ws[need:] == 2).all())
    at = 0
    for b, n in enumerate(new):
        want, tol = _attend(q[at:at + n], ks[b], vs[b], hd**-0.5, True, dtype)
        _same(got[at:at + n], want, tol, f"sequence {b}")
        at += n
