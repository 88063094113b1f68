"""The operators of serving a causal stack, as a program calls them, and their plain forms.

* ``append``: rotary positions on the new tokens' q and k, and their k and v written into a paged
  cache (``_C.rotary_append``);
* ``packed``: attention over whole prompts of different lengths, packed without padding, with grouped
  heads (``_C.flash_attn_packed``);
* ``paged``: attention of each sequence's new tokens, one or a chunk, over its paged cache
  (``_C.flash_attn_paged``).

With ``own`` false ``run`` computes the operator from elementary torch operations in 32 bits (angles in
64), so it needs nothing of this package.  Head counts and head dims follow ``workloads.WORKLOADS`` and
``workloads.SUITE_FULL`` (8 heads of 64, 16 of 64, 16 of 128), with fewer K/V heads where they are
shared; q, k and v are N(0, 1).
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # One token of one sequence (small_fp16's heads): the smallest call there is.
        dict(name="append_token_fp16", op="append", batch=1, longest=65, least=1.0, new=1, heads=8, kv_heads=8,
             head_dim=64, rotary=64, interleaved=False, scaling="none", far=0, page=16, mix=1, dtype="fp16"),
        # One token each of a batch of long-running streams: their positions ran on far past the pages they
        # still hold; part of each head turns, frequencies scaled by parts, pairs interleaved.
        dict(name="append_batch_bf16", op="append", batch=96, longest=1024, least=0.3, new=1, heads=16, kv_heads=4,
             head_dim=128, rotary=64, interleaved=True, scaling="ramp", far=100000, page=16, mix=2, dtype="bf16"),
        # Whole prompts of different lengths on their way into the cache (c4's heads).
        dict(name="append_prompt_bf16", op="append", batch=7, longest=4096, least=0.2, new=4096, heads=16, kv_heads=4,
             head_dim=128, rotary=128, interleaved=False, scaling="base", far=0, page=64, mix=3, dtype="bf16"),
        # The suite's padded batch without its padding, both directions visible.
        dict(name="packed_short_fp16", op="packed", batch=8, longest=128, least=0.4, heads=8, kv_heads=8, head_dim=64,
             causal=False, mix=4, dtype="fp16"),
        # Prompts of odd lengths at c3's heads, four query heads to a K/V head.
        dict(name="packed_ragged_bf16", op="packed", batch=16, longest=1021, least=0.05, heads=16, kv_heads=4,
             head_dim=64, causal=True, mix=5, dtype="bf16"),
        # A few long prompts at c4's heads and length.
        dict(name="packed_long_fp16", op="packed", batch=3, longest=8192, least=0.3, heads=16, kv_heads=2, head_dim=128,
             causal=True, mix=6, dtype="fp16"),
        # One very long prompt: the largest call.
        dict(name="packed_largest_bf16", op="packed", batch=1, longest=32768, least=1.0, heads=16, kv_heads=4,
             head_dim=128, causal=True, mix=7, dtype="bf16"),
        # One token of one sequence over a cache of c4's length: latency, and few rows to fill the card with.
        dict(name="decode_single_bf16", op="paged", batch=1, longest=8192, least=1.0, new=1, chunks=1, heads=16,
             kv_heads=4, head_dim=128, causal=True, page=16, mix=8, dtype="bf16"),
        # A batch of short streams, every head with keys of its own (the suite's heads).
        dict(name="decode_batch_fp16", op="paged", batch=32, longest=2047, least=0.02, new=1, chunks=1, heads=8,
             kv_heads=8, head_dim=64, causal=True, page=16, mix=9, dtype="fp16"),
        # A full serving batch over long caches: the cache is read at the card's rate or it is not.
        dict(name="decode_large_bf16", op="paged", batch=64, longest=30000, least=0.1, new=1, chunks=1, heads=16,
             kv_heads=4, head_dim=128, causal=True, page=16, mix=10, dtype="bf16"),
        # The next chunk of one long prompt over what the cache holds of it.
        dict(name="chunk_long_bf16", op="paged", batch=1, longest=32768, least=1.0, new=512, chunks=1, heads=16,
             kv_heads=4, head_dim=128, causal=True, page=64, mix=11, dtype="bf16"),
        # One step of continuous batching: a chunk of one prompt among the single tokens of the others.
        dict(name="chunk_mixed_fp16", op="paged", batch=24, longest=6000, least=0.1, new=333, chunks=1, heads=16,
             kv_heads=2, head_dim=64, causal=True, page=32, mix=12, dtype="fp16"),
    ]


def _log(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "append", "packed", "packed", "packed", "paged", "paged", "paged", "paged"])
    dtype = rng.choice(["bf16", "fp16"])
    head_dim = rng.choice([64, 128])
    heads = rng.choice([8, 16])
    kv_heads = rng.choice([h for h in (1, 2, 4, 8, 16) if h <= heads])
    mix = rng.randint(100, 1 << 20)
    page = rng.choice([8, 16, 32, 64, 128])
    least = rng.choice([0.02, 0.3, 1.0])
    if op == "append":
        prompt = rng.random() < 0.5
        longest = _log(rng, 1, 4096 if prompt else 1024)
        return dict(op=op, batch=_log(rng, 1, 7 if prompt else 96), longest=longest, least=least,
                    new=_log(rng, 1, longest) if prompt else 1, heads=heads, kv_heads=min(kv_heads, 4),
                    head_dim=head_dim, rotary=rng.choice([head_dim, head_dim, head_dim // 2, 3 * head_dim // 4, 20]),
                    interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "base", "ramp"]),
                    far=rng.choice([0, 0, _log(rng, 1000, 1000000)]), page=page, mix=mix, dtype=dtype)
    if op == "packed":
        longest = _log(rng, 1, 16384)
        return dict(op=op, batch=_log(rng, 1, max(1, min(64, 32768 // longest))), longest=longest, least=least,
                    heads=heads, kv_heads=kv_heads, head_dim=head_dim, causal=rng.random() < 0.7, mix=mix, dtype=dtype)
    if rng.random() < 0.5:  # single tokens, or the few that a draft proposes
        longest = _log(rng, 1, 30000)
        batch = _log(rng, 1, max(1, min(64, 900000 // (longest * kv_heads) + 1)))
        return dict(op=op, batch=batch, longest=longest, least=least, new=rng.choice([1, 1, 1, 2, 5]), chunks=batch,
                    heads=heads, kv_heads=kv_heads, head_dim=head_dim, causal=True, page=page, mix=mix, dtype=dtype)
    longest = _log(rng, 16, 32768)
    batch = _log(rng, 1, max(1, min(32, 98304 // longest)))
    return dict(op=op, batch=batch, longest=longest, least=least, new=_log(rng, 1, min(longest, 1024)),
                chunks=rng.randint(1, min(batch, 4)), heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                causal=rng.random() < 0.8, page=page, mix=mix, dtype=dtype)


# ------------------------------------------------------------------ shapes
def _lengths(case):
    """Tokens of each sequence, the new ones included: the longest one first, the others spread evenly over
    [least * longest, longest], by the case alone."""
    rng = random.Random(case["mix"])
    lo = max(1, int(round(case["longest"] * case["least"])))
    lens = [rng.randint(lo, case["longest"]) for _ in range(case["batch"])]
    lens[0] = case["longest"]
    return lens


def _new(case):
    """New tokens of each sequence (the query rows)."""
    lens = _lengths(case)
    if case["op"] == "packed":
        return lens
    if case["op"] == "append":
        return [min(n, case["new"]) for n in lens]
    # the first ``chunks`` sequences bring a chunk, the others one token
    return [min(n, case["new"] if i < case["chunks"] else 1) for i, n in enumerate(lens)]


def _starts(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return at


def _pairs(case):
    """Admissible (query token, key) pairs of one head."""
    total = 0
    for n, new in zip(_lengths(case), _new(case)):
        total += new * n - (new * (new - 1) // 2 if case["causal"] else 0)
    return total


def work(case):
    t = sum(_new(case))
    h, hk, hd = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "append":
        # q, k, v read and written once; four products and two sums a pair
        return {"bytes": 2 * 2 * t * (h + 2 * hk) * hd, "flops": 3 * t * (h + hk) * case["rotary"]}
    keys = t if case["op"] == "packed" else sum(_lengths(case))
    return {"bytes": 2 * 2 * hd * (t * h + keys * hk), "flops": 4 * hd * h * _pairs(case)}


# ------------------------------------------------------------------ inputs
def _frequencies(case):
    """Angle per position of each pair (a list of floats), and the factor of the turned values."""
    r, base, factor, trained = case["rotary"], 10000.0, 8.0, 4096
    if case["scaling"] == "base":
        base *= factor ** (r / (r - 2))
    freq = [base ** (-2.0 * i / r) for i in range(r // 2)]
    if case["scaling"] == "linear":
        freq = [f / factor for f in freq]
    if case["scaling"] == "ramp":
        keep = [min(1.0, max(0.0, (trained * f / (2 * math.pi) - 1.0) / 31.0)) for f in freq]
        freq = [f * (w + (1 - w) / factor) for f, w in zip(freq, keep)]
        return freq, 0.1 * math.log(factor) + 1.0
    return freq, 1.0


def _rows(gen, rows, cols, dtype):
    return torch.randn((rows, cols), generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _pages(case, gen, dtype):
    """A pool that just holds the sequences, its pages dealt out in random order; the table's unused entries
    are -1."""
    ps = case["page"]
    counts = [(n + ps - 1) // ps for n in _lengths(case)]
    order = torch.randperm(sum(counts), generator=gen, device="cuda").to(torch.int32)
    table = torch.full((case["batch"], max(counts)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at:at + n]
        at += n
    shape = (sum(counts), case["kv_heads"], ps, case["head_dim"])
    pool = []
    for _ in range(2):
        t = torch.empty(shape, dtype=dtype, device="cuda")
        for part in t.split(1 << 14):
            part.copy_(torch.randn(part.shape, generator=gen, device="cuda", dtype=torch.float32))
        pool.append(t)
    return table, pool[0], pool[1]


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    h, hk, hd = case["heads"], case["kv_heads"], case["head_dim"]
    lens, new = _lengths(case), _new(case)
    t = sum(new)
    st = {"case": case, "lens": lens, "new": new, "at": _starts(new)}
    st["cu"] = torch.tensor(st["at"], dtype=torch.int32, device="cuda")
    st["kv_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    # q, k and v are column views of one projection's output, as a GEMM leaves them
    qkv = _rows(gen, t, (h + 2 * hk) * hd, dtype).view(t, h + 2 * hk, hd)
    st["q"], st["k"], st["v"] = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
    if case["op"] == "append":
        far = 0
        if case["far"]:
            far = torch.randint(0, case["far"], (case["batch"],), generator=gen, device="cuda")
            far = torch.repeat_interleave(far, torch.tensor(new, device="cuda"))
        within = [torch.arange(n - m, n, device="cuda") for n, m in zip(lens, new)]
        st["slots"] = torch.cat(within)
        st["positions"] = st["slots"] + far
        freq, st["amplitude"] = _frequencies(case)
        st["freq"] = torch.tensor(freq, dtype=torch.float64, device="cuda")
        st["table"], st["k_cache"], st["v_cache"] = _pages(case, gen, dtype)
        st["owner"] = torch.repeat_interleave(torch.arange(case["batch"], device="cuda"),
                                              torch.tensor(new, device="cuda"))
        if own:
            from transformer_optimization_amd import _C
            st["steps"], st["amplitude"] = _C.rotary_steps(
                case["rotary"], 10000.0, scaling=case["scaling"], factor=8.0, original_len=4096,
                device=torch.device("cuda"))
    elif case["op"] == "paged":
        st["table"], st["k_cache"], st["v_cache"] = _pages(case, gen, dtype)
    return st


# ------------------------------------------------------------------- calls
def run(st):
    case = st["case"]
    if own:
        return _run_own(case, st)
    if case["op"] == "append":
        return _plain_append(case, st)
    return _plain_attention(case, st)


def _run_own(case, st):
    from transformer_optimization_amd import _C
    scale = case["head_dim"] ** -0.5
    if case["op"] == "append":
        q, _ = _C.rotary_append(st["q"], st["k"], st["v"], st["steps"], st["cu"], kv_lens=st["kv_lens"],
                                positions=st["positions"], block_table=st["table"], k_cache=st["k_cache"],
                                v_cache=st["v_cache"], interleaved=case["interleaved"], amplitude=st["amplitude"])
        return q, st["k_cache"], st["v_cache"]
    if case["op"] == "packed":
        return _C.flash_attn_packed(st["q"], st["k"], st["v"], st["cu"], scale, case["causal"])
    return _C.flash_attn_paged(st["q"], st["k_cache"], st["v_cache"], st["table"], st["cu"], st["kv_lens"], scale,
                               case["causal"], max_q_len=max(st["new"]))


def _turn(x, cos, sin, rotary, interleaved):
    x = x.float()
    out = x.clone()
    if interleaved:
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        out[..., 0:rotary:2] = a * cos - b * sin
        out[..., 1:rotary:2] = b * cos + a * sin
    else:
        half = rotary // 2
        a, b = x[..., :half], x[..., half:rotary]
        out[..., :half] = a * cos - b * sin
        out[..., half:rotary] = b * cos + a * sin
    return out


def _plain_append(case, st):
    dtype = st["q"].dtype
    angle = st["positions"].double()[:, None] * st["freq"]
    cos = (torch.cos(angle) * st["amplitude"]).float()[:, None]
    sin = (torch.sin(angle) * st["amplitude"]).float()[:, None]
    q = _turn(st["q"], cos, sin, case["rotary"], case["interleaved"]).to(dtype)
    k = _turn(st["k"], cos, sin, case["rotary"], case["interleaved"]).to(dtype)
    ps = case["page"]
    pages = st["table"][st["owner"], st["slots"] // ps].long()
    st["k_cache"][pages, :, st["slots"] % ps] = k
    st["v_cache"][pages, :, st["slots"] % ps] = st["v"]
    return q, st["k_cache"], st["v_cache"]


def _keys(case, st, b):
    """K and V of sequence b as fp32 [kv_heads, n, head_dim]."""
    n = st["lens"][b]
    if case["op"] == "packed":
        rows = slice(st["at"][b], st["at"][b + 1])
        return st["k"][rows].float().transpose(0, 1), st["v"][rows].float().transpose(0, 1)
    pages = st["table"][b, :(n + case["page"] - 1) // case["page"]].long()
    both = []
    for cache in (st["k_cache"], st["v_cache"]):
        x = cache[pages].transpose(0, 1).reshape(case["kv_heads"], -1, case["head_dim"])
        both.append(x[:, :n].float())
    return both


def _plain_attention(case, st):
    h, hk, hd = case["heads"], case["kv_heads"], case["head_dim"]
    group, scale = h // hk, hd ** -0.5
    out = torch.empty((st["at"][-1], h, hd), dtype=st["q"].dtype, device=st["q"].device)
    for b, (n, new) in enumerate(zip(st["lens"], st["new"])):
        k, v = _keys(case, st, b)
        k = k.transpose(1, 2).contiguous()
        step = max(1, (1 << 28) // (h * n))  # about 2^28 scores at a time
        for i in range(0, new, step):
            rows = min(step, new - i)
            q = st["q"][st["at"][b] + i:st["at"][b] + i + rows].float()
            q = q.reshape(rows, hk, group, hd).permute(1, 2, 0, 3).reshape(hk, group * rows, hd)
            s = torch.matmul(q, k).mul_(scale)
            if case["causal"]:
                last = torch.arange(n - new + i, n - new + i + rows, device=s.device)
                hidden = torch.arange(n, device=s.device)[None, :] > last[:, None]
                s.view(hk, group, rows, n).masked_fill_(hidden, float("-inf"))
            s -= s.amax(-1, keepdim=True)
            s.exp_()
            s /= s.sum(-1, keepdim=True)
            o = torch.matmul(s, v).view(hk, group, rows, hd).permute(2, 0, 1, 3).reshape(rows, h, hd)
            out[st["at"][b] + i:st["at"][b] + i + rows] = o.to(out.dtype)
    return out


# ------------------------------------------------------- results in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, st)
    return _exact_attention(case, st)


def _exact_append(case, st):
    """The turn as a product of complex numbers."""
    freq, amplitude = _frequencies(case)
    r, ps = case["rotary"], case["page"]
    angle = torch.outer(st["positions"].double(), torch.tensor(freq, dtype=torch.float64, device="cuda"))
    turn = torch.polar(torch.full_like(angle, amplitude), angle)[:, None, :]

    def turned(x):
        x = x.double()
        head, rest = x[..., :r], x[..., r:]
        pairs = head.unflatten(-1, (r // 2, 2)) if case["interleaved"] else head.unflatten(-1, (2, r // 2)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        z = z if case["interleaved"] else z.transpose(-1, -2)
        return torch.cat([z.flatten(-2), rest], -1)

    caches = []
    for cache, x in ((st["k_cache"], turned(st["k"])), (st["v_cache"], st["v"].double())):
        tokens = cache.double().transpose(1, 2).flatten(0, 1)  # one row of heads to a slot of the pool
        for b, n in enumerate(st["lens"]):
            slot = torch.arange(n - st["new"][b], n, device="cuda")
            place = st["table"][b].long().repeat_interleave(ps)[slot] * ps + slot % ps
            tokens[place] = x[st["at"][b]:st["at"][b + 1]]
        caches.append(tokens.unflatten(0, (-1, ps)).transpose(1, 2))
    return turned(st["q"]), caches[0], caches[1]


def _exact_attention(case, st):
    """Head by head: weights from the scores' log-sum-exp, on blocks of rows."""
    h, hk, hd = case["heads"], case["kv_heads"], case["head_dim"]
    out = torch.empty((st["at"][-1], h, hd), dtype=torch.float64, device="cuda")
    for b, (n, new) in enumerate(zip(st["lens"], st["new"])):
        if case["op"] == "paged":
            place = st["table"][b].long().repeat_interleave(case["page"])[:n] * case["page"]
            place += torch.arange(n, device="cuda") % case["page"]
        for head in range(h):
            if case["op"] == "paged":
                key, value = (c[:, head // (h // hk)].reshape(-1, hd)[place].double() for c in (st["k_cache"], st["v_cache"]))
            else:
                key, value = (x[st["at"][b]:st["at"][b + 1], head // (h // hk)].double() for x in (st["k"], st["v"]))
            for i in range(0, new, 4096):
                j = min(new, i + 4096)
                seen = n - new + j if case["causal"] else n
                s = (st["q"][st["at"][b] + i:st["at"][b] + j, head].double() / math.sqrt(hd)) @ key[:seen].T
                if case["causal"]:
                    future = torch.ones((j - i, seen), dtype=torch.bool, device="cuda").triu(n - new + i + 1)
                    s[future] = -math.inf
                out[st["at"][b] + i:st["at"][b] + j, head] = torch.exp(s - torch.logsumexp(s, 1, keepdim=True)) @ value[:seen]
    return out
