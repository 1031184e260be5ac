"""Cases of the 8-bit paged K/V cache: writing tokens into it, reading it back, attending over it.

The cache holds E4M3 codes in pages of P tokens, [pages, Hk, P, 128] for K and for V, and one
power-of-two fp32 scale per page and head, [pages, Hk]; a value is code * scale.  A table
[B, W] names each sequence's pages in order (-1: none).  The three operators:

append     count[b] new tokens of sequence b go to positions start[b], start[b] + 1, ...  Per
           page and head the scale is the smallest 2^e (-120 <= e <= 119) with max |x| <= 448 * 2^e
           over every token written since the page was empty; tokens already in a page whose
           scale grows are rounded again to the new one.
read       the values of positions 0 .. max_len - 1 in bf16, zero past a sequence's length.
attention  softmax attention of q [B, Sq, Hq, 128] over the cached keys, query i of sequence b
           at position lens[b] - q_lens[b] + i, optionally causal, optionally within a band.

A case fixes the lengths; the seed draws the values and which pages a sequence has.
"""
import math

import torch

own = False

D = 128
E_MIN, E_MAX = -120, 119


# ------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one sequence's next token, the page half full: the latency of the smallest write
        dict(name="append_one_token", op="append", B=1, S=1, start=250, low=1.0, Hk=8, P=64),
        # a batch of sequences of every length writes its next token; small pages
        dict(name="append_token_batch", op="append", B=48, S=1, start=4095, low=0.0, Hk=8, P=16),
        # the condition's K / V of 16 sequences (256 encoder tokens), as one fused projection gives them
        dict(name="append_condition", op="append", B=16, S=256, start=0, low=1.0, Hk=8, P=64),
        # long prompts behind a short ragged prefix, odd counts
        dict(name="append_prompt", op="append", B=3, S=8191, start=37, low=0.3, Hk=8, P=128),
        # the condition read back into bf16
        dict(name="read_condition", op="read", B=16, L=256, low=1.0, Hk=8, P=64),
        # long ragged sequences read back
        dict(name="read_long", op="read", B=4, L=30001, low=0.5, Hk=8, P=32),
        # one query token over a short cache: the latency of the smallest attention
        dict(name="token_short", op="attention", B=1, Sq=1, L=750, low=1.0, Hq=16, Hk=8, P=64, causal=True, window=-1,
             ragged_q=False),
        # a serving batch, one token each, ragged lengths up to 8192
        dict(name="token_batch", op="attention", B=48, Sq=1, L=8192, low=0.1, Hq=32, Hk=8, P=64, causal=True,
             window=-1, ragged_q=False),
        # few tokens (a speculative or chunked step) over a very long cache
        dict(name="tokens_long", op="attention", B=2, Sq=5, L=100001, low=0.7, Hq=16, Hk=8, P=128, causal=True,
             window=-1, ragged_q=False),
        # the DiT's cross attention: 750 latent tokens over 256 cached encoder tokens
        dict(name="cross_condition", op="attention", B=16, Sq=750, L=256, low=1.0, Hq=16, Hk=8, P=64, causal=False,
             window=-1, ragged_q=False),
        # a whole prompt over its own freshly written keys
        dict(name="prompt_causal", op="attention", B=1, Sq=6001, L=6001, low=1.0, Hq=16, Hk=8, P=64, causal=True,
             window=-1, ragged_q=False),
        # chunks of ragged prompts within a sliding window of a long cache
        dict(name="chunk_window", op="attention", B=4, Sq=517, L=20000, low=0.2, Hq=16, Hk=4, P=32, causal=True,
             window=1024, ragged_q=True),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed ranges, at most as much work as the largest listed ones."""
    op = rng.choice(["append", "read", "attention", "attention"])
    P, Hk, low = rng.choice([16, 32, 64, 128]), rng.choice([1, 2, 4, 8]), rng.choice([0.0, 0.3, 0.7, 1.0])
    if op == "append":
        S = _spread(rng, 1, 8192)
        return dict(op=op, B=_spread(rng, 1, max(1, min(64, 24576 // S))), S=S, start=_spread(rng, 1, 4096) - 1, low=low,
                    Hk=Hk, P=P)
    if op == "read":
        L = _spread(rng, 1, 30000)
        return dict(op=op, B=_spread(rng, 1, max(1, min(64, 120000 // L))), L=L, low=low, Hk=Hk, P=P)
    G = rng.choice([1, 2, 3, 4, 7, 8])
    causal, window = rng.choice([True, True, False]), rng.choice([-1, -1, 128, 1000])
    if rng.random() < 0.5:  # single tokens and a few
        L, Sq = _spread(rng, 16, 100000), rng.choice([1, 1, 1, 2, 3, 5, 9])
        B = _spread(rng, 1, max(1, min(64, 200000 // L)))
    else:                   # prompts and chunks
        Sq = _spread(rng, 10, 4096)
        L = _spread(rng, 64, max(64, min(20000, 36000000 // (2 * G * Sq))))
        B = _spread(rng, 1, max(1, min(16, 36000000 // (Sq * L * max(1, G // 2)))))
    return dict(op=op, B=B, Sq=Sq, L=L, low=low, Hq=G * Hk, Hk=Hk, P=P, causal=causal, window=window,
                ragged_q=bool(Sq > 1 and rng.random() < 0.5))


def _ragged(top, low, B):
    """B lengths from `top` down towards low * top, in steps."""
    return [top - int(top * (1.0 - low) * b / B) for b in range(B)]


def _start_count(case):
    start = _ragged(case["start"], case["low"], case["B"])
    count = [max(1, case["S"] - (case["S"] // 3) * b // max(1, case["B"])) for b in range(case["B"])]
    return start, count


def _q_lens(case):
    B, Sq = case["B"], case["Sq"]
    return [max(1, Sq - (Sq // 2) * b // B) for b in range(B)] if case["ragged_q"] else [Sq] * B


# ------------------------------------------------------------------------------------ inputs

def _scale_of(amax):
    """The smallest power of two s with amax <= 448 s, its exponent within [E_MIN, E_MAX]: with
    amax = m 2^x, 1/2 <= m < 1, and 448 = 7/8 * 2^9."""
    m, x = torch.frexp(amax)
    e = torch.where(amax > 0, x - 9 + (m > 0.875).to(x.dtype), torch.full_like(x, E_MIN)).clamp(E_MIN, E_MAX)
    return torch.ldexp(torch.ones_like(amax), e)


def _filled(pages, Hk, P, g, outliers):
    """A cache half as earlier writes left it: N(0, 1) values, larger in some channels and pages."""
    x = torch.randn(pages, Hk, P, D, generator=g, device="cuda")
    x *= torch.exp(0.7 * torch.randn(pages, Hk, 1, 1, generator=g, device="cuda"))
    if outliers:
        x[..., 7::61] *= 6.0
    s = _scale_of(x.abs().amax((2, 3)))
    x /= s[:, :, None, None]
    return x.clamp(-448, 448).to(torch.float8_e4m3fn), s


def _table(lens, P, g):
    """Pages for sequences of these lengths, in an order of the seed's: table int32 [B, W], pages."""
    need = [-(-n // P) for n in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    at = torch.arange(max(1, max(need)), device="cuda")
    n = torch.tensor(need, device="cuda")
    first = torch.cumsum(n, 0) - n
    table = order[(first[:, None] + at[None, :]).clamp(max=pages - 1)]
    return torch.where(at[None, :] < n[:, None], table, torch.full_like(table, -1)).contiguous(), pages


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 11)
    B, Hk, P, op = case["B"], case["Hk"], case["P"], case["op"]
    st = dict(case)
    if op == "append":
        start, count = _start_count(case)
        lens = [a + b for a, b in zip(start, count)]
        st["start_t"], st["count_t"] = _int32(start), _int32(count)
        # k and v are the two halves of one projection's output rows
        kv = torch.randn(B * case["S"], 2 * Hk * D, generator=g, device="cuda")
        kv *= torch.exp(0.7 * torch.randn(B * case["S"], 1, generator=g, device="cuda"))
        kv = kv.to(torch.bfloat16).view(B, case["S"], 2, Hk, D)
        st["k_new"], st["v_new"] = kv[:, :, 0], kv[:, :, 1]
    else:
        lens = _ragged(case["L"], case["low"], B)
        st["lens_t"] = _int32(lens)
    st["table"], pages = _table(lens, P, g)
    st["k"], st["k_scale"] = _filled(pages, Hk, P, g, True)
    st["v"], st["v_scale"] = _filled(pages, Hk, P, g, False)
    if op == "attention":
        st["q"] = torch.randn(B, case["Sq"], case["Hq"], D, generator=g, device="cuda").to(torch.bfloat16)
        st["q_lens_t"] = _int32(_q_lens(case)) if case["ragged_q"] else None
    return st


# ------------------------------------------------------------------------------------ plain forms

def _append_half(codes, scale, new, table, start, count):
    B, S, Hk, _ = new.shape
    P, W = codes.shape[2], table.shape[1]
    t = torch.arange((S - 1) // P + 2, device=new.device)
    first, end = start // P, start + count
    page = first[:, None] + t                                         # [B, T] pages in their sequences' order
    page = torch.where(page * P < end[:, None], page, first[:, None])  # past the last: the first one again
    pid = table.gather(1, page.clamp(max=W - 1).long()).long()         # [B, T]
    pos = page[:, :, None] * P + torch.arange(P, device=new.device)    # [B, T, P]
    is_old = (pos < start[:, None, None])[:, :, None, :, None]
    is_new = ((pos >= start[:, None, None]) & (pos < end[:, None, None]))[:, :, None, :, None]
    row = (pos - start[:, None, None]).clamp(0, S - 1).long()
    x = new.float()[torch.arange(B, device=new.device)[:, None, None], row].permute(0, 1, 3, 2, 4)  # [B, T, Hk, P, D]
    old, s_old = codes[pid], scale[pid]                                # [B, T, Hk, P, D], [B, T, Hk]
    finite = torch.where(is_new & torch.isfinite(x), x.abs(), torch.zeros_like(x))
    s = _scale_of(finite.amax((3, 4)))
    s = torch.where((page * P < start[:, None])[:, :, None], torch.maximum(s, s_old), s)
    x = (x / s[..., None, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    kept = (old.float() * (s_old / s)[..., None, None]).to(torch.float8_e4m3fn)
    bits = torch.where(is_new, x.view(torch.uint8),
                       torch.where(is_old, kept.view(torch.uint8), old.view(torch.uint8)))
    codes.view(torch.uint8)[pid] = bits
    scale[pid] = s


def _values(codes, scale, table):
    """fp32 values of every position that the table covers, [B, Hk, W * P, D]."""
    pid = table.clamp(min=0).long()
    x = codes[pid].float() * scale[pid][..., None, None]
    B, W, Hk, P, _ = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(B, Hk, W * P, D)


def _read_half(codes, scale, st):
    x = _values(codes, scale, st["table"])[:, :, :st["L"]].transpose(1, 2)
    inside = torch.arange(st["L"], device=x.device)[None, :] < st["lens_t"][:, None]
    return torch.where(inside[:, :, None, None], x, torch.zeros_like(x)).to(torch.bfloat16)


def _visible(st, n_keys, dev):
    """[B, Sq, n_keys]: which keys a query sees."""
    lens = st["lens_t"].long()[:, None, None]
    ql = (st["q_lens_t"].long()[:, None, None] if st["q_lens_t"] is not None else torch.full_like(lens, st["Sq"]))
    i = torch.arange(st["Sq"], device=dev)[None, :, None]
    j = torch.arange(n_keys, device=dev)[None, None, :]
    pos = lens - ql + i
    see = (j < lens) & (i < ql)
    if st["causal"]:
        see = see & (j <= pos)
    if st["window"] >= 0:
        see = see & ((pos - j).abs() <= st["window"])
    return see


def _attention(st):
    q = st["q"].float()
    B, Sq, Hq, _ = q.shape
    Hk = st["Hk"]
    G = Hq // Hk
    k, v = _values(st["k"], st["k_scale"], st["table"]), _values(st["v"], st["v_scale"], st["table"])
    n = k.shape[2]
    v = torch.where((torch.arange(n, device=q.device)[None, :] < st["lens_t"][:, None])[:, None, :, None], v,
                    torch.zeros_like(v))
    qg = q.view(B, Sq, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * Sq, D)
    s = ((qg @ k.transpose(-1, -2)) * D ** -0.5).view(B, Hk, G, Sq, n)
    s = s.masked_fill(~_visible(st, n, q.device)[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    l = p.sum(-1, keepdim=True)
    p = p / torch.where(l > 0, l, torch.ones_like(l))
    o = p.view(B, Hk, G * Sq, n) @ v
    return o.view(B, Hk, G, Sq, D).permute(0, 3, 1, 2, 4).reshape(B, Sq, Hq, D).to(torch.bfloat16)


def run(st):
    if own:
        return _run_own(st)
    if st["op"] == "append":
        _append_half(st["k"], st["k_scale"], st["k_new"], st["table"], st["start_t"], st["count_t"])
        _append_half(st["v"], st["v_scale"], st["v_new"], st["table"], st["start_t"], st["count_t"])
        return st["k"], st["v"], st["k_scale"], st["v_scale"]
    if st["op"] == "read":
        return _read_half(st["k"], st["k_scale"], st), _read_half(st["v"], st["v_scale"], st)
    return _attention(st)


def _run_own(st):
    from demon_b200 import kvcache
    cache = st.get("cache")
    if cache is None:  # the handle around the cache's buffers, which a program keeps
        cache = st["cache"] = kvcache.KVCache(st["k"], st["v"], st["k_scale"], st["v_scale"])
    if st["op"] == "append":
        kvcache.append(cache, st["k_new"], st["v_new"], st["table"], st["start_t"], st["count_t"])
        return cache.k, cache.v, cache.k_scale, cache.v_scale
    if st["op"] == "read":
        return kvcache.read(cache, st["table"], st["lens_t"], st["L"])
    return kvcache.attention(st["q"], cache, st["table"], st["lens_t"], causal=st["causal"],
                             window=None if st["window"] < 0 else st["window"], q_lens=st["q_lens_t"])


# ------------------------------------------------------------------------------------ work

def work(case):
    B, Hk, P, op = case["B"], case["Hk"], case["P"], case["op"]
    if op == "append":
        start, count = _start_count(case)
        touched = sum((a + c - 1) // P - a // P + 1 for a, c in zip(start, count))
        return {"bytes": 2 * Hk * (sum(count) * D * 3 + touched * 4) + 8 * B, "flops": 0}
    lens = _ragged(case["L"], case["low"], B)
    held = 2 * Hk * sum(n * D + -(-n // P) * 4 for n in lens)
    if op == "read":
        return {"bytes": held + 2 * Hk * B * case["L"] * D * 2, "flops": 0}
    keys = pairs = 0
    for n, nq in zip(lens, _q_lens(case)):
        lo, hi = n, 0  # the keys that any query sees
        for i in range(nq):
            pos = n - nq + i
            a, b = 0, n - 1
            if case["causal"]:
                b = min(b, pos)
            if case["window"] >= 0:
                a, b = max(a, pos - case["window"]), min(b, pos + case["window"])
            if b >= a:
                pairs += b - a + 1
                lo, hi = min(lo, a), max(hi, b + 1)
        keys += max(0, hi - lo)
    rows = B * case["Sq"] * case["Hq"]
    return {"bytes": 2 * Hk * keys * (D + 4 / P) + 2 * rows * D * 2, "flops": 4 * D * pairs * case["Hq"]}


# ------------------------------------------------------------------------------------ in 64 bits

def _e4m3(x):
    """The nearest E4M3 value (ties to even, at most 448) of float64 x, by arithmetic: the spacing
    is 2^(e - 3) for 2^e <= |x| < 2^(e + 1), and 2^-9 below 2^-6."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def _exact_append(codes, scale, new, table, start, count):
    codes, scale, new = codes.double(), scale.double(), new.double()
    P, Hk = codes.shape[2], codes.shape[1]
    for b, (a, c) in enumerate(zip(start, count)):
        pages = torch.arange(a // P, (a + c - 1) // P + 1, device=codes.device)
        pid = table[b, pages].long()
        n = len(pages) * P
        block = codes[pid].transpose(1, 2).reshape(n, Hk, D)             # [tokens, Hk, D]
        before = a - int(pages[0]) * P
        fresh = torch.zeros(n, Hk, D, dtype=torch.float64, device=codes.device)
        fresh[before:before + c] = new[b, :c]
        amax = fresh.abs().view(len(pages), P, Hk, D).amax((1, 3))       # [pages, Hk]
        e = torch.ceil(torch.log2(amax.clamp(min=448.0 * 2.0 ** -200) / 448.0))
        e = torch.where(amax <= 448.0 * torch.exp2(e - 1), e - 1, e)     # log2 next to a power of two
        e = torch.where(amax > 448.0 * torch.exp2(e), e + 1, e).clamp(E_MIN, E_MAX)
        if before:
            e[0] = torch.maximum(e[0], torch.log2(scale[pid[0]]).round())
        s = torch.exp2(e).repeat_interleave(P, 0)[:, :, None]            # [tokens, Hk, 1]
        if before:
            block[:before] = _e4m3(block[:before] * scale[pid[0]][None, :, None] / s[:before])
        block[before:before + c] = _e4m3(fresh[before:before + c] / s[before:before + c])
        codes[pid] = block.view(len(pages), P, Hk, D).transpose(1, 2)
        scale[pid] = torch.exp2(e)
    return codes, scale


def _exact_values(codes, scale, row, n):
    """float64 values of the first n positions of one sequence, [Hk, n, D]."""
    P = codes.shape[2]
    pid = row[:-(-n // P)].long()
    x = codes[pid].double() * scale[pid].double()[:, :, None, None]
    return x.transpose(0, 1).reshape(codes.shape[1], -1, D)[:, :n]


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "append":
        start, count = _start_count(case)
        k, ks = _exact_append(st["k"], st["k_scale"], st["k_new"], st["table"], start, count)
        v, vs = _exact_append(st["v"], st["v_scale"], st["v_new"], st["table"], start, count)
        return k, v, ks, vs
    lens = _ragged(case["L"], case["low"], case["B"])
    if case["op"] == "read":
        out = []
        for codes, scale in ((st["k"], st["k_scale"]), (st["v"], st["v_scale"])):
            x = torch.zeros(case["B"], case["L"], case["Hk"], D, dtype=torch.float64, device="cuda")
            for b, n in enumerate(lens):
                x[b, :n] = _exact_values(codes, scale, st["table"][b], n).transpose(0, 1)
            out.append(x)
        return tuple(out)
    o = torch.zeros(case["B"], case["Sq"], case["Hq"], D, dtype=torch.float64, device="cuda")
    G = case["Hq"] // case["Hk"]
    for b, (n, nq) in enumerate(zip(lens, _q_lens(case))):
        k = _exact_values(st["k"], st["k_scale"], st["table"][b], n)
        v = _exact_values(st["v"], st["v_scale"], st["table"][b], n)
        pos = torch.arange(n - nq, n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None, :]
        hide = torch.zeros(nq, n, dtype=torch.bool, device="cuda")
        if case["causal"]:
            hide |= j > pos
        if case["window"] >= 0:
            hide |= (j - pos).abs() > case["window"]
        none = hide.all(1)
        for h in range(case["Hq"]):
            s = st["q"][b, :nq, h].double() @ k[h // G].T / math.sqrt(D)
            p = torch.softmax(s.masked_fill(hide, -math.inf), -1)
            o[b, :nq, h] = torch.where(none[:, None], 0.0, p) @ v[h // G]
    return o
