"""GPU parity of the paged 8-bit K/V cache against its definition in 64 bits (kv_reference.py).

append and read are exact: codes, scales and bf16 values must be equal bit for bit (a scale is a
power of two and a value has four significant bits).  attention is compared element by element
with the bound derived in kv_reference.attention: half a step of bf16 for the output, half a step
of f16 for the probabilities, fp32 sums.
"""
import os

import pytest
import torch

import kv_reference as R

pytestmark = pytest.mark.gpu

BAD_ARG = 0x2


def ok():
    from demon_b200 import _native as nat
    torch.cuda.synchronize()
    assert nat.device_status() == (0, 0)


def make_table(lens, P, dev, seed, extra=2, width=None):
    """Random distinct pages for sequences of these capacities: (device table, nested lists, pages)."""
    need = [-(-n // P) for n in lens]
    pages = sum(need) + extra
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    W = width or max(1, max(need))
    rows, at = [], 0
    for n in need:
        rows.append(order[at:at + n] + [-1] * (W - n))
        at += n
    return torch.tensor(rows, dtype=torch.int32, device=dev), rows, pages


def i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def filled(lens, P, heads, dev, seed, spread=1.0, k_scale_by=None, v_scale_by=None):
    """A cache holding random values at these lengths, its twin, and the table."""
    from demon_b200 import kvcache
    table, rows, pages = make_table(lens, P, dev, seed)
    cache = kvcache.KVCache.empty(pages, heads, P, dev)
    ref = R.RefCache(pages, heads, P, dev)
    g = torch.Generator().manual_seed(seed + 1)
    S = max(1, max(lens))
    x = [torch.randn(len(lens), S, heads, 128, generator=g).to(dev) * spread for _ in range(2)]
    for i, by in enumerate((k_scale_by, v_scale_by)):
        if by is not None:
            x[i] = x[i] * by(torch.arange(S, device=dev)).view(1, S, 1, 1)
    k, v = (t.to(torch.bfloat16) for t in x)
    kvcache.append(cache, k, v, table, i32([0] * len(lens), dev), i32(lens, dev))
    ref.append(k, v, rows, [0] * len(lens), lens)
    return cache, ref, table, rows


def same_cache(cache, ref, rows, lens):
    """Codes of every held position, scales of every held page, bit for bit."""
    for kv, (c, s) in enumerate(((cache.k, cache.k_scale), (cache.v, cache.v_scale))):
        P = ref.P
        for row, n in zip(rows, lens):
            for i in range(-(-n // P)):
                m = min(P, n - i * P)
                got, want = c[row[i], :, :m].double(), ref.codes[kv, row[i], :, :m]
                assert torch.equal(torch.nan_to_num(got, nan=999.0), torch.nan_to_num(want, nan=999.0))
                assert torch.equal(s[row[i]].double(), torch.exp2(ref.exp[kv, row[i]].double()))


# ------------------------------------------------------------------------------------ append

@pytest.mark.parametrize("P", [16, 32, 64, 128])
@pytest.mark.parametrize("heads", [1, 3, 8])
def test_append_matches_definition_over_several_writes(cuda, P, heads):
    """Prompts, then odd chunks, then single tokens, growing amplitudes: the scales of partly
    filled pages grow and their codes are rounded again; counts of zero write nothing."""
    from demon_b200 import kvcache
    B = 3
    caps = [2 * P + 5, 7 * P, 3 * P - 1]
    table, rows, pages = make_table(caps, P, cuda, P + heads)
    cache, ref = kvcache.KVCache.empty(pages, heads, P, cuda), R.RefCache(pages, heads, P, cuda)
    g = torch.Generator().manual_seed(P)
    start = [0, 0, 0]
    for step, (S, count) in enumerate([(P + 3, [P + 3, 1, P // 2]), (7, [0, 7, 5]), (1, [1, 1, 0]), (1, [1, 1, 1]),
                                       (P - 3, [P - 3, P - 3, 1])]):
        k, v = (torch.randn(B, S, heads, 128, generator=g).mul(3.0 ** step * 0.01).to(torch.bfloat16).to(cuda)
                for _ in range(2))
        kvcache.append(cache, k, v, table, i32(start, cuda), i32(count, cuda))
        ref.append(k, v, rows, start, count)
        start = [a + b for a, b in zip(start, count)]
        same_cache(cache, ref, rows, start)
    ok()


def test_append_reads_strided_halves_of_one_projection(cuda):
    """k and v as the two halves of a [B * L, 2 * heads * 128] projection, without count."""
    from demon_b200 import kvcache
    B, S, heads, P = 2, 77, 4, 32
    kv = torch.randn(B * S, 2 * heads * 128, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(cuda)
    ld = kv.stride(0)
    k = kv.as_strided((B, S, heads, 128), (S * ld, ld, 128, 1))
    v = kv.as_strided((B, S, heads, 128), (S * ld, ld, 128, 1), heads * 128)
    table, rows, pages = make_table([S, S], P, cuda, 4)
    cache, ref = kvcache.KVCache.empty(pages, heads, P, cuda), R.RefCache(pages, heads, P, cuda)
    kvcache.append(cache, k, v, table, i32([0, 0], cuda))
    ref.append(k, v, rows, [0, 0], [S, S])
    same_cache(cache, ref, rows, [S, S])
    # head-major inputs [B, heads, S, 128], transposed by strides only
    kt, vt = k.transpose(1, 2).contiguous().transpose(1, 2), v.transpose(1, 2).contiguous().transpose(1, 2)
    again = kvcache.KVCache.empty(pages, heads, P, cuda)
    kvcache.append(again, kt, vt, table, i32([0, 0], cuda))
    assert torch.equal(again.k.view(torch.uint8), cache.k.view(torch.uint8))
    ok()


def test_append_extreme_values(cuda):
    """Zeros, the smallest and largest magnitudes, infinities and NaN, and every boundary of the
    scale rule (448 * 2^e and its bf16 neighbours; above 448 * 2^119 values saturate)."""
    from demon_b200 import kvcache
    P, heads = 16, 2
    edge = [0.0, 448.0, 450.0, 446.0, 2.0 ** -133, 3.3895e38, -3.3895e38, 2.0 ** -120, 1.75 * 2.0 ** 100, 1.7578125 * 2.0 ** 100,
            float("inf"), float("-inf"), float("nan"), -0.0, 1e-30, 65504.0]
    n = len(edge)
    x = torch.zeros(1, n * P, heads, 128)
    for i, a in enumerate(edge):   # one page each: the edge value, small company, and zeros
        x[0, i * P + 3, 0, 5] = a
        x[0, i * P:(i + 1) * P, 1, :] = a
        if a not in (0.0,):
            x[0, i * P + 4, 0, :64] = torch.randn(64, generator=torch.Generator().manual_seed(i)) * 0.5
    x = x.to(torch.bfloat16).to(cuda)
    table, rows, pages = make_table([n * P], P, cuda, 9)
    cache, ref = kvcache.KVCache.empty(pages, heads, P, cuda), R.RefCache(pages, heads, P, cuda)
    kvcache.append(cache, x, -x, table, i32([0], cuda))
    ref.append(x, -x, rows, [0], [n * P])
    same_cache(cache, ref, rows, [n * P])
    k, v = kvcache.read(cache, table, i32([n * P], cuda), n * P)
    for kv, got in enumerate((k, v)):
        want = ref.values(kv, rows[0], n * P).transpose(0, 1)
        assert torch.equal(torch.nan_to_num(got[0].double(), nan=123.0), torch.nan_to_num(want, nan=123.0))
    ok()


def test_append_leaves_other_tokens_and_pages_alone(cuda):
    from demon_b200 import kvcache
    cache, ref, table, rows = filled([50, 20], 16, 2, cuda, 5)
    before = cache.k.view(torch.uint8).clone()
    x = torch.full((2, 4, 2, 128), 1e-3, dtype=torch.bfloat16, device=cuda)     # below the page's scale
    kvcache.append(cache, x, x, table, i32([30, 0], cuda), i32([2, 0], cuda))
    after = cache.k.view(torch.uint8)
    changed = (after != before).flatten(1).any(1).nonzero().flatten().tolist()
    assert changed in ([], [rows[0][1]])
    page_b, page_a = before[rows[0][1]], after[rows[0][1]]
    assert torch.equal(page_b[:, :14], page_a[:, :14])                           # tokens 16 .. 29
    ref.append(x, x, rows, [30, 0], [2, 0])
    same_cache(cache, ref, rows, [32, 20])
    ok()


def test_append_again_changes_nothing(cuda):
    from demon_b200 import kvcache
    cache, _, table, _ = filled([37], 32, 2, cuda, 6)
    x = torch.randn(1, 9, 2, 128, generator=torch.Generator().manual_seed(1)).mul(40).to(torch.bfloat16).to(cuda)
    kvcache.append(cache, x, x, table, i32([20], cuda))
    one = [t.view(torch.uint8).clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    kvcache.append(cache, x, x, table, i32([20], cuda))
    two = [t.view(torch.uint8) for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    assert all(torch.equal(a, b) for a, b in zip(one, two))


# ------------------------------------------------------------------------------------ read

@pytest.mark.parametrize("P,heads", [(16, 1), (32, 8), (64, 3), (128, 2)])
def test_read_gives_the_values_and_zeros_behind(cuda, P, heads):
    from demon_b200 import kvcache
    lens = [0, 1, P, 2 * P + 3, 5 * P - 1]
    cache, ref, table, rows = filled(lens, P, heads, cuda, P)
    for max_len in (max(lens), 1, P + 2, max(lens) + 40):
        held = [min(n, max_len) for n in lens]
        k, v = kvcache.read(cache, table, i32(lens, cuda), max_len)
        for kv, got in enumerate((k, v)):
            for b, n in enumerate(held):
                assert torch.equal(got[b, :n].double(), ref.values(kv, rows[b], lens[b])[:, :n].transpose(0, 1))
                assert not bool(got[b, n:].any())
    ok()


def test_read_into_strided_outputs(cuda):
    from demon_b200 import kvcache
    lens, heads = [40, 7], 2
    cache, _, table, _ = filled(lens, 16, heads, cuda, 8)
    want = kvcache.read(cache, table, i32(lens, cuda), 40)
    both = torch.full((2, 43, 3, 2, heads, 128), 7.0, dtype=torch.bfloat16, device=cuda)
    out = (both[:, :40, 0, 0], both[:, :40, 1, 1])
    got = kvcache.read(cache, table, i32(lens, cuda), 40, out=out)
    assert got[0].data_ptr() == out[0].data_ptr()
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    assert bool((both[:, 40:] == 7).all()) and bool((both[:, :, 2] == 7).all())
    ok()


# ------------------------------------------------------------------------------------ attention

def check_attention(cuda, cache, ref, rows, table, lens, q, q_lens=None, causal=False, window=None, scale=None,
                    label="", **kw):
    """The call as it is, then through each of the two kernels (few rows, tensor cores)."""
    chosen = os.environ.get("DEMON_KV_ATTENTION", "")
    for name in [n for n in ("small", "tc", "") if n != chosen] + [chosen]:
        os.environ["DEMON_KV_ATTENTION"] = name
        o = check_one(cuda, cache, ref, rows, table, lens, q, q_lens, causal, window, scale, f"{name} {label}", **kw)
    return o


@pytest.fixture(autouse=True)
def _no_choice_left():
    yield
    os.environ.pop("DEMON_KV_ATTENTION", None)


@pytest.fixture(params=["", "small", "tc"])
def which(request):
    """The attention kernel as the call chooses it, and each of the two."""
    os.environ["DEMON_KV_ATTENTION"] = request.param
    return request.param


def check_one(cuda, cache, ref, rows, table, lens, q, q_lens, causal, window, scale, label, **kw):
    from demon_b200 import kvcache
    o = kvcache.attention(q, cache, table, i32(lens, cuda), causal=causal, window=window, scale=scale,
                          q_lens=None if q_lens is None else i32(q_lens, cuda), **kw)
    sc = 128 ** -0.5 if scale is None else scale
    for b, n in enumerate(lens):
        nq = q.shape[1] if q_lens is None else q_lens[b]
        k, v = ref.values(0, rows[b], n), ref.values(1, rows[b], n)
        want, own = R.attention(q[b].double(), k, v, nq, causal, window, sc)
        got = o[b].double()
        assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{label} b={b}: NaN elsewhere"
        err = torch.where(torch.isnan(want), torch.zeros_like(want), (got - want).abs())
        room = torch.where(torch.isnan(want), torch.ones_like(want), R.error_bound(want, own))
        worst = float((err / room).max()) if err.numel() else 0.0
        assert worst <= 1.0, f"{label} b={b}: {worst:.3f} of the allowed error"
        assert not bool(got[nq:].any())
    ok()
    return o


def queries(B, Sq, Hq, dev, seed, by=1.0):
    return (torch.randn(B, Sq, Hq, 128, generator=torch.Generator().manual_seed(seed)) * by).to(torch.bfloat16).to(dev)


@pytest.mark.parametrize("P", [16, 32, 64, 128])
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (16, 8), (6, 2), (7, 1), (16, 1), (40, 2)])
def test_single_tokens(cuda, P, Hq, Hk):
    lens = [0, 1, 15, P, P + 1, 63, 64, 65, 700]
    cache, ref, table, rows = filled(lens, P, Hk, cuda, P + Hq)
    q = queries(len(lens), 1, Hq, cuda, Hq)
    check_attention(cuda, cache, ref, rows, table, lens, q, causal=True, label=f"P={P} {Hq}/{Hk}")


@pytest.mark.parametrize("causal,window", [(True, None), (False, None), (True, 0), (True, 37), (False, 20), (True, 5000)])
@pytest.mark.parametrize("Sq,Hq,Hk,P", [(2, 16, 8, 64), (5, 8, 1, 16), (17, 6, 2, 32), (40, 4, 4, 128), (130, 4, 2, 64),
                                        (300, 2, 1, 16), (129, 3, 1, 64), (257, 8, 1, 32)])
def test_chunks_masks_and_ragged_batches(cuda, causal, window, Sq, Hq, Hk, P):
    """Fewer keys than queries (rows that see nothing), no keys, ragged queries, odd lengths."""
    lens = [0, 1, Sq - 1, Sq, 333, 64]
    q_lens = [Sq, Sq, Sq, 1, max(1, Sq // 2), 0]
    cache, ref, table, rows = filled(lens, P, Hk, cuda, Sq + P)
    q = queries(len(lens), Sq, Hq, cuda, Sq)
    check_attention(cuda, cache, ref, rows, table, lens, q, None, causal, window, label="all rows")
    check_attention(cuda, cache, ref, rows, table, lens, q, q_lens, causal, window, label="ragged")


@pytest.mark.parametrize("Sq,Hq,Hk", [(1, 8, 2), (3, 8, 2), (200, 4, 2)])
def test_long_caches(cuda, Sq, Hq, Hk):
    lens = [5000, 4097, 128]
    cache, ref, table, rows = filled(lens, 64, Hk, cuda, 77)
    check_attention(cuda, cache, ref, rows, table, lens, queries(3, Sq, Hq, cuda, 5), causal=True)
    check_attention(cuda, cache, ref, rows, table, lens, queries(3, Sq, Hq, cuda, 5), causal=True, window=1000)


@pytest.mark.parametrize("Sq", [1, 9, 150])
def test_growing_maxima_and_large_scores(cuda, Sq):
    """Later keys dominate (the running maximum moves in every tile), scores of some hundreds."""
    cache, ref, table, rows = filled([640], 32, 1, cuda, 3, k_scale_by=lambda t: 0.1 + t / 80.0)
    check_attention(cuda, cache, ref, rows, table, [640], queries(1, Sq, 4, cuda, 4, 4.0), causal=False)


@pytest.mark.parametrize("Sq", [1, 9, 150])
@pytest.mark.parametrize("step", [3, 11, 40, -3, -11, -40])
def test_page_scales_far_apart(cuda, Sq, step):
    """V's scale rises or falls by 2^step from page to page (up to 2^80 in all)."""
    n_pages = max(2, 80 // abs(step))
    n = 16 * n_pages
    by = lambda t: torch.exp2((t // 16).double() * step).float()   # noqa: E731
    cache, ref, table, rows = filled([n], 16, 1, cuda, 21, v_scale_by=by)
    check_attention(cuda, cache, ref, rows, table, [n], queries(1, Sq, 2, cuda, 4), causal=True)


@pytest.mark.parametrize("Sq", [1, 6, 160])
@pytest.mark.parametrize("q_by,k_by,v_by", [(1e30, 1e-30, 1e-38), (1e-30, 1e30, 1e37), (1e-38, 1.0, 1.0), (0.0, 1.0, 1.0)])
def test_extreme_magnitudes(cuda, Sq, q_by, k_by, v_by):
    cache, ref, table, rows = filled([150], 32, 1, cuda, 31, k_scale_by=lambda t: torch.full_like(t, k_by, dtype=torch.float32),
                                     v_scale_by=lambda t: torch.full_like(t, v_by, dtype=torch.float32))
    check_attention(cuda, cache, ref, rows, table, [150], queries(1, Sq, 2, cuda, 4, q_by), causal=True)


@pytest.mark.parametrize("Sq", [1, 5, 24, 140])
def test_nan_reaches_only_the_rows_that_see_it(cuda, Sq):
    """NaN codes past the length (stale pages), in keys hidden by the causal mask or the band,
    and in keys that some rows see: V's NaN marks its channel, K's its whole row."""
    lens = [200, 200 - 7, 64]
    cache, ref, table, rows = filled([208, 208, 64], 16, 2, cuda, 41)
    for kv, t in enumerate((cache.k, cache.v)):
        for row, n in zip(rows, lens):
            for page in range(len([r for r in row if r >= 0])):
                for tok in range(16):
                    if page * 16 + tok >= n:
                        t.view(torch.uint8)[row[page], :, tok] = 0x7F     # stale: never seen
    def poison(kv, b, tok, ch):
        (cache.k, cache.v)[kv].view(torch.uint8)[rows[b][tok // 16], 1, tok % 16, ch] = 0xFF
        ref.codes[kv, rows[b][tok // 16], 1, tok % 16, ch] = float("nan")
    poison(1, 0, 199, 77)       # the last key: seen by the last row alone (causal)
    poison(1, 0, 150, 3)
    poison(0, 1, 192, 0)        # a key whose score is NaN
    poison(1, 2, 10, 127)
    q = queries(3, Sq, 4, cuda, Sq)
    for causal, window in ((True, None), (True, 30), (False, 25), (False, None)):
        check_attention(cuda, cache, ref, rows, table, lens, q, None, causal, window, label=f"{causal} {window}")


def test_strided_queries_and_outputs(cuda, which):
    from demon_b200 import kvcache
    lens = [90, 33]
    cache, ref, table, rows = filled(lens, 32, 2, cuda, 51)
    for Sq in (1, 3, 140):
        wide = torch.randn(2, Sq + 3, 3, 5, 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(cuda)
        q = wide[:, 1:Sq + 1, 1, :4]
        buf = torch.full((2, Sq + 2, 2, 6, 128), 9.0, dtype=torch.bfloat16, device=cuda)
        out = buf[:, 1:Sq + 1, 0, 1:5]
        want = check_attention(cuda, cache, ref, rows, table, lens, q.contiguous(), causal=True)
        got = kvcache.attention(q, cache, table, i32(lens, cuda), causal=True, out=out)
        assert got.data_ptr() == out.data_ptr() and torch.equal(out, want)
        rest = buf.clone()
        rest[:, 1:Sq + 1, 0, 1:5] = 9.0
        assert bool((rest == 9).all())
        same = kvcache.attention(q[:1].expand(2, -1, -1, -1), cache, table, i32(lens, cuda), causal=True)   # broadcast
        assert torch.equal(same, kvcache.attention(q[:1].repeat(2, 1, 1, 1), cache, table, i32(lens, cuda), causal=True))
        qt = q.contiguous().transpose(1, 2).contiguous().transpose(1, 2)          # head-major
        assert torch.equal(kvcache.attention(qt, cache, table, i32(lens, cuda), causal=True), want)


def test_shared_pages(cuda):
    """Two sequences over the same condition pages, a third with its own."""
    cache, ref, table, rows = filled([100, 60], 32, 2, cuda, 61)
    t3, r3 = torch.stack([table[0], table[0], table[1]]), [rows[0], rows[0], rows[1]]
    q = queries(3, 20, 4, cuda, 1)
    check_attention(cuda, cache, ref, r3, t3, [100, 70, 60], q)


def test_pages_beyond_32_bit_offsets(cuda, which):
    """Codes that lie past 2^32 bytes of the buffers."""
    from demon_b200 import kvcache
    P, heads = 128, 8
    pages = (1 << 32) // (P * heads * 128) + 64
    codes = [torch.empty(pages, heads, P, 128, dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.full((pages, heads), 2.0 ** -120, device=cuda) for _ in range(2)]
    cache = kvcache.KVCache(*codes, *scales)
    small, ref, _, rows = filled([300], P, heads, cuda, 71)
    moved = [pages - 1 - i for i in range(3)]
    table = i32([moved], cuda)
    k, v = kvcache.read(small, i32([rows[0][:3]], cuda), i32([300], cuda), 300)
    kvcache.append(cache, k, v, table, i32([0], cuda))
    k2, v2 = kvcache.read(cache, table, i32([300], cuda), 300)
    assert torch.equal(k, k2) and torch.equal(v, v2)
    # the same codes in low pages (values read back and written again may take a smaller scale:
    # the largest of a page can have been rounded down to 448 * 2^(e - 1))
    twin, low = kvcache.KVCache.empty(4, heads, P, cuda), i32([[2, 0, 3]], cuda)
    kvcache.append(twin, k, v, low, i32([0], cuda))
    for Sq in (1, 150):
        q = queries(1, Sq, 16, cuda, 2)
        o = kvcache.attention(q, cache, table, i32([300], cuda), causal=True)
        assert torch.equal(o, kvcache.attention(q, twin, low, i32([300], cuda), causal=True))
    ok()


# ------------------------------------------------------------------------------------ as it is used

def test_a_sequence_grows_token_by_token_and_graphs_replay(cuda):
    """Prompt, then tokens one at a time through one captured graph (append + attention) whose
    lengths and inputs change between replays; equal to the eager calls, bit for bit."""
    from demon_b200 import kvcache
    heads, Hq, P, B = 2, 4, 16, 2
    table, rows, pages = make_table([90, 90], P, cuda, 81)
    g = torch.Generator().manual_seed(5)
    prompt = [torch.randn(B, 40, heads, 128, generator=g).to(torch.bfloat16).to(cuda) for _ in range(2)]
    steps = [[torch.randn(B, 1, n, 128, generator=g).mul(1 + t / 5).to(torch.bfloat16).to(cuda) for n in (heads, heads, Hq)]
             for t in range(40)]
    out = []
    for graphed in (False, True):
        cache, ref = kvcache.KVCache.empty(pages, heads, P, cuda), R.RefCache(pages, heads, P, cuda)
        start, lens = i32([0, 0], cuda), i32([40, 31], cuda)
        kvcache.append(cache, *prompt, table, start, lens)
        ref.append(*prompt, rows, [0, 0], [40, 31])
        k, v, q = (t.clone() for t in steps[0])
        pos = lens.clone()

        def step():
            kvcache.append(cache, k, v, table, pos)
            return kvcache.attention(q, cache, table, pos + 1, causal=True)
        got = []
        if graphed:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                keep = [t.view(torch.uint8).clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
                step()
                for t, u in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), keep):
                    t.view(torch.uint8).copy_(u)
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                o = step()
        for t, (kk, vv, qq) in enumerate(steps):
            k.copy_(kk), v.copy_(vv), q.copy_(qq)
            if graphed:
                graph.replay()
            else:
                o = step()
            got.append(o.clone())
            pos += 1
        out.append(torch.stack(got))
        for t, (kk, vv, _) in enumerate(steps):
            ref.append(kk, vv, rows, [40 + t, 31 + t], [1, 1])
        same_cache(cache, ref, rows, [80, 71])
        check_attention(cuda, cache, ref, rows, table, [80, 71], steps[-1][2], causal=True)
    assert torch.equal(out[0], out[1])
    ok()


def test_calls_on_other_streams(cuda, which):
    """An explicit stream, and two streams at once over one cache, equal the plain call."""
    from demon_b200 import kvcache
    cache, _, table, _ = filled([3000, 2000], 64, 2, cuda, 91)
    lens = i32([3000, 2000], cuda)
    q = queries(2, 1, 4, cuda, 1)
    q2 = queries(2, 200, 4, cuda, 2)
    want, want2 = kvcache.attention(q, cache, table, lens, causal=True), kvcache.attention(q2, cache, table, lens, causal=True)
    kv = kvcache.read(cache, table, lens, 3000)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(10):
        got.append((kvcache.attention(q, cache, table, lens, causal=True, stream=a),
                    kvcache.attention(q2, cache, table, lens, causal=True, stream=b),
                    kvcache.read(cache, table, lens, 3000, stream=a)))
    torch.cuda.synchronize()
    for x, y, z in got:
        assert torch.equal(x, want) and torch.equal(y, want2) and torch.equal(z[0], kv[0]) and torch.equal(z[1], kv[1])
    ok()


def test_repeated_calls_give_equal_bits(cuda, which):
    from demon_b200 import kvcache
    cache, _, table, _ = filled([4000, 100, 999], 32, 2, cuda, 92)
    lens = i32([4000, 100, 999], cuda)
    for Sq in (1, 4, 70, 300):
        q = queries(3, Sq, 8, cuda, Sq)
        first = kvcache.attention(q, cache, table, lens, causal=True)
        for _ in range(5):
            assert torch.equal(kvcache.attention(q, cache, table, lens, causal=True), first)


# ------------------------------------------------------------------------------------ refusals

def test_bad_device_values_are_reported_and_harmless(cuda, which):
    """Page ids, lengths and starts out of range (checked on the CPU in test_kvcache.py): the
    status word says so, other sequences are right, nothing else is written."""
    from demon_b200 import _native as nat
    from demon_b200 import kvcache
    lens = [60, 60, 60]
    cache, ref, table, rows = filled(lens, 16, 2, cuda, 95)
    before = cache.k.view(torch.uint8).clone()
    x = torch.randn(3, 4, 2, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(cuda)
    for bad in ([62, -1, 1 << 30], [61, 2147483647, -2147483648]):      # past the table's 64 positions
        kvcache.append(cache, x, x, table, i32(bad, cuda))
        torch.cuda.synchronize()
        assert nat.device_status()[0] == BAD_ARG
    for count in ([5, -1, 2147483647],):
        kvcache.append(cache, x, x, table, i32([0, 0, 0], cuda), i32(count, cuda))
        torch.cuda.synchronize()
        assert nat.device_status()[0] == BAD_ARG
    assert torch.equal(cache.k.view(torch.uint8), before)
    hurt = table.clone()
    hurt[1, 1], hurt[2, 0] = 1 << 20, -5
    kvcache.append(cache, x, x, hurt, i32([60, 20, 2], cuda), i32([0, 4, 4], cuda))
    torch.cuda.synchronize()
    assert nat.device_status()[0] == BAD_ARG and torch.equal(cache.k.view(torch.uint8), before)
    k, _ = kvcache.read(cache, hurt, i32([60, 60, 99999], cuda), 60)
    torch.cuda.synchronize()
    assert nat.device_status()[0] == BAD_ARG
    assert torch.equal(k[0].double(), ref.values(0, rows[0], 60).transpose(0, 1))
    assert not bool(k[1, 16:32].any()) and bool(k[1, :16].any()) and not bool(k[2, :16].any())
    good = kvcache.attention(queries(3, 1, 4, cuda, 1), cache, table, i32(lens, cuda))
    for Sq in (1, 140):
        q = queries(3, Sq, 4, cuda, 1)
        good = kvcache.attention(q, cache, table, i32(lens, cuda))
        got = kvcache.attention(q, cache, hurt, i32([60, 60, -3], cuda))
        torch.cuda.synchronize()
        assert nat.device_status()[0] == BAD_ARG
        assert torch.equal(got[0], good[0]) and not bool(got[2].any())
        # a page that is not there is a page that no query sees
        left = R.RefCache(1, 2, 16, cuda)
        k1, v1 = (torch.cat([ref.values(kv, rows[1], 60)[:, :16], ref.values(kv, rows[1], 60)[:, 32:]], 1) for kv in (0, 1))
        want, own = R.attention(q[1].double(), k1, v1, Sq, False, None, 128 ** -0.5)
        assert bool(((got[1].double() - want).abs() <= R.error_bound(want, own)).all())
        del left
    ok()


def test_refusals(cuda):
    from demon_b200 import _native as nat
    from demon_b200 import kvcache
    cache, _, table, _ = filled([40, 40], 16, 2, cuda, 96)
    lens = i32([40, 40], cuda)
    q = queries(2, 1, 4, cuda, 1)
    x = queries(2, 3, 2, cuda, 1)
    with pytest.raises(nat.DemonError, match="multiple of the kv heads"):
        kvcache.attention(queries(2, 1, 3, cuda, 1), cache, table, lens)
    with pytest.raises(nat.DemonError, match="window"):
        kvcache.attention(q, cache, table, lens, window=-2)
    with pytest.raises(nat.DemonError, match="scale"):
        kvcache.attention(q, cache, table, lens, scale=0.0)
    with pytest.raises(ValueError, match="bf16"):
        kvcache.attention(q.half(), cache, table, lens)
    with pytest.raises(ValueError, match="int32"):
        kvcache.attention(q, cache, table, lens.long())
    with pytest.raises(ValueError, match="int32"):
        kvcache.attention(q, cache, table.long(), lens)
    with pytest.raises(ValueError, match="table"):
        kvcache.attention(q, cache, table[:1], lens)
    with pytest.raises(ValueError, match="head_dim"):
        kvcache.attention(q[..., :64], cache, table, lens)
    with pytest.raises(ValueError, match="out"):
        kvcache.attention(q, cache, table, lens, out=q[:, :, :2])
    with pytest.raises(ValueError, match="cuda"):
        kvcache.attention(q.cpu(), cache, table, lens)
    with pytest.raises(ValueError, match="overlap"):
        kvcache.attention(q, cache, table, lens, out=q[:1].clone().expand(2, -1, -1, -1))
    odd = torch.zeros(2, 1, 4, 132, dtype=torch.bfloat16, device=cuda)[..., :128]
    with pytest.raises(nat.DemonError, match="multiples of 8"):
        kvcache.attention(odd, cache, table, lens)
    shifted = torch.zeros(2 * 4 * 128 + 8, dtype=torch.bfloat16, device=cuda)[4:4 + 2 * 4 * 128].view(2, 1, 4, 128)
    with pytest.raises(nat.DemonError, match="aligned"):
        kvcache.attention(shifted, cache, table, lens)
    with pytest.raises(ValueError, match="heads"):
        kvcache.append(cache, x[:, :, :1], x[:, :, :1], table, lens)
    with pytest.raises(ValueError, match="start"):
        kvcache.append(cache, x, x, table, lens[:1])
    with pytest.raises(ValueError, match="count"):
        kvcache.append(cache, x, x, table, lens, lens.float())
    with pytest.raises(ValueError, match="equal"):
        kvcache.append(cache, x, x[:, :2], table, lens)
    with pytest.raises(ValueError, match="lens"):
        kvcache.read(cache, table, lens[:1], 40)
    with pytest.raises(ValueError, match="out k"):
        kvcache.read(cache, table, lens, 40, out=(x, x))
    with pytest.raises(nat.DemonError, match="overlap"):
        same = torch.empty(1, 40, 2, 128, dtype=torch.bfloat16, device=cuda).expand(2, 40, 2, 128)
        kvcache.read(cache, table, lens, 40, out=(same, same))
    ok()


def test_empty_calls(cuda, which):
    """No sequences, no tokens, no queries, no table columns."""
    from demon_b200 import kvcache
    cache, _, table, _ = filled([40, 40], 16, 2, cuda, 97)
    none = torch.empty(0, table.shape[1], dtype=torch.int32, device=cuda)
    e = torch.empty(0, dtype=torch.int32, device=cuda)
    lens = i32([40, 40], cuda)
    assert kvcache.attention(queries(0, 1, 4, cuda, 1), cache, none, e).shape == (0, 1, 4, 128)
    assert kvcache.attention(queries(2, 0, 4, cuda, 1), cache, table, lens).shape == (2, 0, 4, 128)
    kvcache.append(cache, queries(0, 3, 2, cuda, 1), queries(0, 3, 2, cuda, 1), none, e)
    kvcache.append(cache, queries(2, 0, 2, cuda, 1), queries(2, 0, 2, cuda, 1), table, lens)
    assert kvcache.read(cache, none, e, 5)[0].shape == (0, 5, 2, 128)
    assert kvcache.read(cache, table, lens, 0)[0].shape == (2, 0, 2, 128)
    thin = torch.empty(2, 0, dtype=torch.int32, device=cuda)
    for Sq in (1, 140):
        assert not bool(kvcache.attention(queries(2, Sq, 4, cuda, 1), cache, thin, i32([0, 0], cuda)).any())
    assert not bool(kvcache.read(cache, thin, i32([0, 0], cuda), 9)[0].any())
    ok()


def test_the_cache_keeps_the_tensors_it_checked(cuda):
    import dataclasses
    cache, _, _, _ = filled([40], 16, 2, cuda, 98)
    for name in ("k", "v", "k_scale", "v_scale"):
        with pytest.raises(dataclasses.FrozenInstanceError):
            setattr(cache, name, getattr(cache, name).clone())


def test_read_refuses_one_output_for_both(cuda):
    from demon_b200 import _native as nat
    from demon_b200 import kvcache
    cache, _, table, _ = filled([40], 16, 2, cuda, 99)
    x = torch.empty(1, 40, 2, 128, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(nat.DemonError, match="overlap"):
        kvcache.read(cache, table, i32([40], cuda), 40, out=(x, x))


def test_output_in_place_of_the_queries(cuda, which):
    from demon_b200 import kvcache
    lens, nq = [700, 90, 0], [1.0, 0.5, 1.0]
    cache, _, table, _ = filled(lens, 32, 2, cuda, 100)
    for Sq in (1, 3, 40, 300):
        q = queries(3, Sq, 6, cuda, Sq)
        n = i32([max(1, int(Sq * f)) for f in nq], cuda)
        want = kvcache.attention(q, cache, table, i32(lens, cuda), causal=True, q_lens=n)
        kvcache.attention(q, cache, table, i32(lens, cuda), causal=True, q_lens=n, out=q)
        assert torch.equal(q, want)
    ok()


def test_broadcast_queries_on_another_stream(cuda, which):
    """The copy of broadcast queries belongs to the call's stream, whatever the current one does."""
    from demon_b200 import kvcache
    cache, _, table, _ = filled([300, 200], 64, 2, cuda, 101)
    lens, s = i32([300, 200], cuda), torch.cuda.Stream()
    for Sq in (2, 200):
        q = queries(1, Sq, 4, cuda, Sq)
        want = kvcache.attention(q.repeat(2, 1, 1, 1), cache, table, lens)
        torch.cuda.synchronize()
        torch.cuda._sleep(100_000_000)   # some 50 ms
        got = kvcache.attention(q.expand(2, -1, -1, -1), cache, table, lens, stream=s)
        s.synchronize()
        assert torch.equal(got, want)
        torch.cuda.synchronize()
    ok()


def test_condition_rows_by_a_device_index(cuda):
    """An index held on the device is not looked at from the host; out of range it names no page."""
    from demon_b200 import _native as nat
    from demon_b200 import kvcache
    from demon_b200.dit import CrossCache
    cache, _, table, _ = filled([60, 50], 16, 2, cuda, 102)
    kv = CrossCache(cache, table, i32([60, 50], cuda))
    q = queries(4, 2, 4, cuda, 1)
    for index in ([1, 0, 0, 1], [1, 2, -1, 0]):
        r = kv.rows(torch.tensor(index, device=cuda))
        o = kvcache.attention(q, r.cache, r.table, r.lens)
        bits, _ = nat.device_status()
        assert (bits != 0) == any(i not in (0, 1) for i in index)
        for b, i in enumerate(index):
            if i in (0, 1):
                one = kvcache.attention(q[b:b + 1], cache, table[i:i + 1], kv.lens[i:i + 1])
                assert torch.equal(o[b:b + 1], one)
            else:
                assert not bool(o[b].any())
    ok()


def test_a_call_of_several_seconds(cuda):
    """300,000 queries of 16 heads over 2^20 keys (some 3 s): no wait gives up on a long call.

    The table names 8 pages again and again, so that every row equals the row over these 8 pages.
    Tolerance: two bf16 outputs (2^-9 each, relative); the long call adds 2^16 matrix instructions
    of 16 keys into an fp32 accumulator, each dropping at most 2^-23 of sum p |v|, and 2^13 tile
    sums of 2^-24 into the softmax sum.
    """
    from demon_b200 import kvcache
    cache, ref, table, rows = filled([1024], 128, 1, cuda, 103)
    q = queries(1, 500, 16, cuda, 5).repeat(1, 600, 1, 1)
    long = table[:, :8].repeat(1, 1024).contiguous()
    o = kvcache.attention(q, cache, long, i32([1 << 20], cuda))
    want = kvcache.attention(q[:, :500], cache, table, i32([1024], cuda)).double()
    ok()
    own = float(ref.values(1, rows[0], 1024).double().abs().max())
    for i in (0, 77_500, 299_500):
        err = (o[:, i:i + 500].double() - want).abs()
        assert bool((err <= (2.0 ** -8 + 2.0 ** -11) * want.abs() + 2.0 ** -7 * own).all())


def attention_args(q, cache, table, lens, out, causal, window=-1, q_lens=None):
    from demon_b200 import _native as nat
    from demon_b200 import kvcache
    B, Sq, Hq, _ = q.shape
    return nat.DemonKvAttnArgs.from_buffer_copy(kvcache._ATTN.pack(
        *cache._c, q.data_ptr(), *q.stride()[:3], out.data_ptr(), *out.stride()[:3], table.data_ptr(), table.stride(0),
        lens.data_ptr(), 0 if q_lens is None else q_lens.data_ptr(), B, Sq, Hq, table.shape[1], int(causal), window,
        128 ** -0.5, 0, 0, 0))


# rows of 8, 16 and (by the environment) 32 per unit; few enough units for a workspace
@pytest.mark.parametrize("Sq,Hq,Hk,P,lens", [(1, 8, 2, 64, [20_001, 17_000]), (1, 1, 1, 16, [40_000]), (5, 4, 2, 128, [33_000, 0]),
                                             (3, 12, 3, 32, [16_500]), (10, 6, 2, 64, [30_000]), (64, 1, 1, 16, [17_000])])
def test_keys_split_over_a_workspace(cuda, Sq, Hq, Hk, P, lens):
    from demon_b200 import _native as nat
    cache, ref, table, rows = filled(lens, P, Hk, cuda, 104, v_scale_by=lambda i: torch.exp2((i // 2500 % 3).float() * -9))
    q = queries(len(lens), Sq, Hq, cuda, Sq)
    for causal, window, q_lens in ((True, None, None), (False, None, [(Sq + 1) // 2] * len(lens)), (True, 9000, None), (False, 90, None)):
        check_attention(cuda, cache, ref, rows, table, lens, q, q_lens, causal, window, label=f"{causal} {window}")
    # with a workspace of any contents, and without one
    lib, n = nat.load(), i32(lens, cuda)
    os.environ["DEMON_KV_ATTENTION"] = "small"
    want = check_one(cuda, cache, ref, rows, table, lens, q, None, True, None, None, "chosen")
    out = torch.empty_like(q)
    args = attention_args(q, cache, table, n, out, True)
    size = lib.demon_kv_attention_workspace(bytes(args))
    assert size > 0
    room = torch.full((size + 64,), 255, dtype=torch.uint8, device=cuda)
    args.workspace, args.workspace_bytes = room.data_ptr(), size
    nat.check(lib.demon_kv_attention(bytes(args), nat.stream_ptr()))
    assert torch.equal(out, want) and bool((room[size:] == 255).all())
    args.workspace_bytes = size - 1
    with pytest.raises(nat.DemonError, match="workspace"):
        nat.check(lib.demon_kv_attention(bytes(args), nat.stream_ptr()))
    args.workspace, args.workspace_bytes = room.data_ptr() + 8, size
    with pytest.raises(nat.DemonError, match="aligned"):
        nat.check(lib.demon_kv_attention(bytes(args), nat.stream_ptr()))
    args.workspace = None
    out.fill_(3)
    nat.check(lib.demon_kv_attention(bytes(args), nat.stream_ptr()))
    for b, L in enumerate(lens):
        k, v = ref.values(0, rows[b], L), ref.values(1, rows[b], L)
        exact, own = R.attention(q[b].double(), k, v, Sq, True, None, 128 ** -0.5)
        assert bool(((out[b].double() - exact).abs() <= R.error_bound(exact, own)).all())
    ok()


def test_nan_across_a_workspace_and_graphs_with_one(cuda):
    """A NaN score or value met by one part reaches the whole row; captured calls keep workspaces of their own."""
    from demon_b200 import kvcache
    lens = [24_000]
    cache, ref, table, rows = filled(lens, 64, 2, cuda, 105)
    for kv, pos, d in ((0, 12_345, 7), (1, 20_000, 100)):
        page, at = rows[0][pos // 64], pos % 64
        (cache.k if kv == 0 else cache.v).view(torch.uint8)[page, kv, at, d] = 0x7F
        ref.codes[kv, page, kv, at, d] = torch.nan
    for Sq in (1, 6):
        q = queries(1, Sq, 4, cuda, Sq)
        for causal, window in ((True, None), (True, 3000), (True, 300)):
            check_attention(cuda, cache, ref, rows, table, lens, q, None, causal, window)
    n, q = i32(lens, cuda), queries(1, 1, 4, cuda, 9)
    side, graphs, outs = torch.cuda.Stream(), [], []
    for window in (2000, None):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(kvcache.attention(q, cache, table, n, causal=True, window=window))
        graphs.append(g)
    want = [kvcache.attention(q, cache, table, n, causal=True, window=w) for w in (2000, None)]
    torch.cuda.synchronize()
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o.view(torch.int16), w.view(torch.int16))
    ok()


@pytest.mark.parametrize("Sq,Hq,Hk", [(1, 100, 1), (3, 128, 1), (2, 130, 1), (1, 200, 1), (40, 65, 1)])
def test_many_query_heads_per_kv_head(cuda, Sq, Hq, Hk):
    lens = [300, 77]
    cache, ref, table, rows = filled(lens, 32, Hk, cuda, 106)
    check_attention(cuda, cache, ref, rows, table, lens, queries(2, Sq, Hq, cuda, Sq), causal=True)


@pytest.mark.parametrize("Sq,Hq,Hk,P,lens", [(40, 4, 2, 64, [5000, 3100]), (130, 8, 1, 16, [4000]), (300, 2, 2, 128, [9000, 0]),
                                             (70, 3, 1, 32, [1300]), (33, 100, 1, 64, [2200])])
def test_blocks_of_rows_split_over_a_workspace(cuda, Sq, Hq, Hk, P, lens):
    """The tensor-core kernel with few blocks: parts of their keys, some of which a row does not see."""
    from demon_b200 import _native as nat
    cache, ref, table, rows = filled(lens, P, Hk, cuda, 107, v_scale_by=lambda i: torch.exp2((i // 700 % 3).float() * -11))
    page = rows[0][1000 // P]
    cache.v.view(torch.uint8)[page, 0, 1000 % P, 5] = 0xFF      # one NaN of V, one of K
    ref.codes[1, page, 0, 1000 % P, 5] = torch.nan
    q = queries(len(lens), Sq, Hq, cuda, Sq)
    for causal, window, q_lens in ((True, None, None), (False, None, [Sq - 7] * len(lens)), (True, 700, None), (False, 2000, None)):
        check_attention(cuda, cache, ref, rows, table, lens, q, q_lens, causal, window, label=f"{causal} {window}")
    page = rows[0][1100 // P]
    cache.k.view(torch.uint8)[page, 0, 1100 % P, 50] = 0x7F
    ref.codes[0, page, 0, 1100 % P, 50] = torch.nan
    for causal, window in ((True, None), (True, 150)):
        check_attention(cuda, cache, ref, rows, table, lens, q, None, causal, window, label=f"NaN {causal} {window}")
    os.environ["DEMON_KV_ATTENTION"] = "tc"
    n, out = i32(lens, cuda), torch.empty_like(q)
    args = attention_args(q, cache, table, n, out, True)
    size = nat.load().demon_kv_attention_workspace(bytes(args))
    assert size > 0
    want = check_one(cuda, cache, ref, rows, table, lens, q, None, True, None, None, "chosen")
    room = torch.full((size + 64,), 255, dtype=torch.uint8, device=cuda)
    args.workspace, args.workspace_bytes = room.data_ptr(), size
    nat.check(nat.load().demon_kv_attention(bytes(args), nat.stream_ptr()))
    assert torch.equal(out.view(torch.int16), want.view(torch.int16)) and bool((room[size:] == 255).all())
    args.workspace = None
    nat.check(nat.load().demon_kv_attention(bytes(args), nat.stream_ptr()))
    ok()
    args.workspace, args.workspace_bytes = room.data_ptr(), size - 1
    with pytest.raises(nat.DemonError, match="workspace"):
        nat.check(nat.load().demon_kv_attention(bytes(args), nat.stream_ptr()))


@pytest.mark.parametrize("lens,Sq,q_lens", [([257] + [0] * 88 + [130], 200, None),                     # long runs of sequences without keys
                                            ([70, 0, 0] * 40, 150, None),
                                            ([90] * 60, 300, [1 + (b % 7 == 0) * 299 for b in range(60)]),   # and of blocks without queries
                                            ([400] * 5 + [0] * 120 + [300], 130, [129] * 126)])
def test_runs_of_empty_blocks(cuda, lens, Sq, q_lens):
    """More blocks than SMs, most of them without keys or queries, between others that have them."""
    cache, ref, table, rows = filled(lens, 32, 8, cuda, 108)
    q = queries(len(lens), Sq, 16, cuda, Sq)
    for causal, window in ((False, None), (True, None), (True, 20)):
        check_attention(cuda, cache, ref, rows, table, lens, q, q_lens, causal, window, label=f"{causal} {window}")


@pytest.mark.parametrize("lens,q_lens", [([3000, 0, 0, 0, 0, 0, 2000], None), ([2600] * 6, [1, 1, 200, 1, 1, 70])])
def test_parts_and_empty_blocks(cuda, lens, q_lens):
    cache, ref, table, rows = filled(lens, 64, 1, cuda, 109)
    q = queries(len(lens), 200, 2, cuda, 3)
    for causal, window in ((False, None), (True, None), (True, 900)):
        check_attention(cuda, cache, ref, rows, table, lens, q, q_lens, causal, window, label=f"{causal} {window}")


def test_copies_of_a_cache_are_caches_of_their_own(cuda):
    import copy
    import pickle

    from demon_b200 import kvcache
    cache, _, table, _ = filled([40], 16, 2, cuda, 110)
    lens = i32([40], cuda)
    k, v = kvcache.read(cache, table, lens, 40)
    for other in (copy.deepcopy(cache), pickle.loads(pickle.dumps(cache))):
        kvcache.append(cache, -k, -v, table, i32([0], cuda))
        same = kvcache.read(other, table, lens, 40)
        assert torch.equal(same[0], k) and torch.equal(same[1], v)
        kvcache.append(cache, k, v, table, i32([0], cuda))
        assert torch.equal(kvcache.read(cache, table, lens, 40)[0], k)
    ok()


# 128 rows of a tile are not a multiple of these heads: the rows behind them hold what shared memory held
@pytest.mark.parametrize("G", [3, 5, 6, 7, 12, 100])
def test_rows_that_no_token_has_change_nothing(cuda, G):
    """Equal bits whatever ran on the SMs before, in the blocks' own rows and behind a workspace."""
    from demon_b200 import kvcache
    os.environ["DEMON_KV_ATTENTION"] = "tc"
    cache, ref, table, rows = filled([864, 400, 3000], 16, 2, cuda, 120)
    other, _, table2, _ = filled([500] * 40, 16, 2, cuda, 121)
    lens, q = i32([864, 400, 3000], cuda), queries(3, 59, 2 * G, cuda, G)
    first = check_one(cuda, cache, ref, rows, table, [864, 400, 3000], q, None, True, None, None, f"G={G}")
    short = kvcache.attention(q, cache, table[:, :55].contiguous(), lens.clamp(max=880), causal=True)
    for by in (1e38, 1e-3, 1e20):
        kvcache.attention(queries(40, 260, 4, cuda, 9, by), other, table2, i32([500] * 40, cuda))
        assert torch.equal(kvcache.attention(q, cache, table, lens, causal=True), first), by
        assert torch.equal(kvcache.attention(q, cache, table[:, :55].contiguous(), lens.clamp(max=880), causal=True), short), by
    ok()


def test_a_second_part_on_an_sm(cuda):
    """The tensor-core kernel with more parts of blocks than SMs: a CTA takes several, of different blocks."""
    from demon_b200 import _native as nat
    lens, Sq, Hq, Hk = [9640, 5000, 9000, 0, 7001], 87, 24, 8
    cache, ref, table, rows = filled(lens, 64, Hk, cuda, 118, v_scale_by=lambda i: torch.exp2((i // 1700 % 3).float() * -7))
    q = queries(len(lens), Sq, Hq, cuda, 5)
    os.environ["DEMON_KV_ATTENTION"] = "tc"
    args = attention_args(q, cache, table, i32(lens, cuda), q, True)
    tokens, blocks = 2 * (128 // 3), 2 * len(lens) * Hk
    parts, rest = divmod(nat.load().demon_kv_attention_workspace(bytes(args)), blocks * tokens * 3 * (128 + 4) * 4)
    assert rest == 0 and parts * blocks > 148 and parts * blocks % 148 > 0
    for causal, window, q_lens in ((True, None, None), (False, None, [Sq, 1, 70, 3, 0]), (True, 6000, None)):
        first = check_one(cuda, cache, ref, rows, table, lens, q, q_lens, causal, window, None, f"{causal} {window}")
        assert torch.equal(first, check_one(cuda, cache, ref, rows, table, lens, q, q_lens, causal, window, None, "again"))


# ------------------------------------------------------------------------- values far from one

def held(k, v, lens, P, dev, seed):
    """A cache holding k / v [B, S, heads, 128] at these lengths, its twin, and the table."""
    from demon_b200 import kvcache
    table, rows, pages = make_table([k.shape[1]] * len(lens), P, dev, seed)
    cache, ref = kvcache.KVCache.empty(pages, k.shape[2], P, dev), R.RefCache(pages, k.shape[2], P, dev)
    k, v = k.to(torch.bfloat16).to(dev), v.to(torch.bfloat16).to(dev)
    kvcache.append(cache, k, v, table, i32([0] * len(lens), dev), i32(lens, dev))
    ref.append(k, v, rows, [0] * len(lens), lens)
    return cache, ref, table, rows


@pytest.mark.parametrize("signs", [False, True])
@pytest.mark.parametrize("Sq,Hq,Hk,P,lens", [(300, 2, 2, 128, [9000, 4100]), (40, 8, 2, 64, [5000]), (70, 1, 1, 16, [1300]),
                                             (1, 8, 2, 64, [20_001, 17_000]), (10, 6, 2, 32, [30_000])])
def test_large_values_in_parts(cuda, Sq, Hq, Hk, P, lens, signs):
    """V of 5e37 to 2e38 over keys whose parts are joined: no partial sum leaves fp32, which ends at 3.4e38."""
    g = torch.Generator().manual_seed(Sq)
    k = torch.randn(len(lens), max(lens), Hk, 128, generator=g)
    v = (1 + 3 * torch.rand(k.shape, generator=g)) * 5e37
    if signs:  # by channel: what overflows does not meet its opposite
        v = v * (1 - 2 * (torch.arange(128) % 2))
    cache, ref, table, rows = held(k, v, lens, P, cuda, 111)
    q = queries(len(lens), Sq, Hq, cuda, Sq)
    for causal, window in ((True, None), (False, 9000)):
        check_attention(cuda, cache, ref, rows, table, lens, q, None, causal, window, label=f"{causal} {window}")


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int16, torch.int32])
def test_condition_rows_by_a_device_index_of_other_types(cuda, dtype):
    from demon_b200.dit import CrossCache
    cache, _, table, _ = filled([60, 50, 40], 16, 2, cuda, 122)
    kv = CrossCache(cache, table, i32([60, 50, 40], cuda))
    for index in ([1, 1, 1], [0, 1, 1], [2, 0]):
        for where in (cuda, "cpu"):
            r = kv.rows(torch.tensor(index, dtype=dtype, device=where))
            assert torch.equal(r.table, table[torch.tensor(index, device=cuda)]) and r.lens.tolist() == [60 - 10 * i for i in index]


def test_condition_rows_of_no_conditions_by_a_device_index(cuda):
    """Every index is out of range: zeros, and reported, also where the first condition has no tokens."""
    from demon_b200 import _native as nat
    from demon_b200 import kvcache
    from demon_b200.dit import CrossCache
    cache, _, table, _ = filled([60], 16, 2, cuda, 123)
    index, q = torch.tensor([0, 1], device=cuda), queries(2, 2, 4, cuda, 1)
    for kv in (CrossCache(cache, table[:0], i32([], cuda)), CrossCache(cache, table[:0, :0], i32([], cuda)),
               CrossCache(cache, table, i32([0], cuda))):
        r = kv.rows(index)
        assert not bool(kvcache.attention(q, r.cache, r.table, r.lens).any())
        assert nat.device_status()[0] == BAD_ARG
        assert kv.rows(index[:0]).table.shape[0] == 0
    ok()


def check_seen(cuda, cache, ref, rows, table, lens, q, causal, window):
    """Through both kernels, with the allowed error of each row from the keys that it sees alone."""
    from demon_b200 import kvcache
    for name in ("small", "tc"):
        os.environ["DEMON_KV_ATTENTION"] = name
        o = kvcache.attention(q, cache, table, i32(lens, cuda), causal=causal, window=window)
        for b, n in enumerate(lens):
            k, v = ref.values(0, rows[b], n), ref.values(1, rows[b], n)
            pid = torch.tensor(rows[b][:-(-n // ref.P)], device=cuda)
            unit = torch.exp2(ref.exp[1][pid].double()).repeat_interleave(ref.P, 0)[:n].T
            want, _ = R.attention(q[b].double(), k, v, q.shape[1], causal, window, 128 ** -0.5)
            room = R.error_bound(want, R.seen_bound(q[b].double(), k, v, unit, q.shape[1], causal, window, 128 ** -0.5))
            err = (o[b].double() - want).abs()
            assert bool((err <= room).all()), f"{name} {causal} {window} b={b}: {float((err / room).nan_to_num(nan=9e9).max()):.3f}"
    ok()


@pytest.mark.parametrize("Sq,Hq,Hk,P,lens", [(40, 2, 1, 16, [200, 77]), (5, 3, 1, 16, [66, 34]), (150, 4, 2, 32, [300, 64]),
                                             (9, 1, 1, 16, [9000]), (33, 2, 2, 64, [9100]),
                                             (4, 2, 1, 16, [70, 18]), (8, 1, 1, 32, [9000, 40])])
@pytest.mark.parametrize("low,high", [(-120, 110), (110, -120), (-60, 70), (-3, 4)])
def test_scales_of_pages_that_a_row_does_not_see(cuda, Sq, Hq, Hk, P, lens, low, high):
    """V around 2^low before the middle of the rows' last positions and 2^high from there: a row's result
    has the precision of the pages that it sees, whatever the scales of those that its neighbours see."""
    g = torch.Generator().manual_seed(Sq)
    n = max(lens)
    k, v = (torch.randn(len(lens), n, Hk, 128, generator=g) for _ in range(2))
    for b, L in enumerate(lens):
        turn = (L - min(Sq, L) // 2) // P * P
        v[b] *= torch.exp2(torch.where(torch.arange(n) < turn, low, high).double()).float()[:, None, None]
    cache, ref, table, rows = held(k, v, lens, P, cuda, 112)
    q = queries(len(lens), Sq, Hq, cuda, Sq)
    for causal, window in ((True, None), (True, 11), (False, 3), (False, 20)):
        check_seen(cuda, cache, ref, rows, table, lens, q, causal, window)


@pytest.mark.parametrize("Sq", [1, 9, 150])
@pytest.mark.parametrize("step", [3, 11, 40, -3, -11, -40])
def test_page_scales_far_apart_row_by_row(cuda, Sq, step):
    """V's scale rises or falls by 2^step from page to page, each row held to what it sees."""
    n = 16 * max(2, 80 // abs(step))
    g = torch.Generator().manual_seed(113)
    k, v = (torch.randn(1, n, 1, 128, generator=g) for _ in range(2))
    v = v * torch.exp2((torch.arange(n) // 16).double() * step).float()[None, :, None, None]
    cache, ref, table, rows = held(k, v, [n], 16, cuda, 113)
    for causal, window in ((True, None), (False, 17)):
        check_seen(cuda, cache, ref, rows, table, [n], queries(1, Sq, 2, cuda, 4), causal, window)


@pytest.mark.parametrize("Sq", [1, 5, 150])
@pytest.mark.parametrize("big", [1e38, 3e30])
def test_a_page_scale_from_keys_that_are_not_seen(cuda, Sq, big):
    """Zero keys in a page whose scale comes from keys behind the length: the scores are zero, not 0 * inf."""
    g = torch.Generator().manual_seed(Sq)
    k, v = torch.zeros(1, 48, 1, 128), torch.randn(1, 48, 1, 128, generator=g)
    k[:, 40:] = big
    cache, ref, table, rows = held(k, v, [48], 16, cuda, 114)
    q = torch.full((1, Sq, 2, 128), big, dtype=torch.bfloat16, device=cuda)
    check_attention(cuda, cache, ref, rows, table, [40], q)


# long tables of few blocks: with a workspace the tensor-core kernel's parts are the faster choice
@pytest.mark.parametrize("Sq,Hq,Hk,L", [(64, 8, 1, 20_000), (40, 16, 8, 12_000), (130, 4, 2, 16_000)])
def test_the_kernel_without_a_workspace_is_chosen_for_that(cuda, Sq, Hq, Hk, L):
    """A C caller without a workspace is not sent to a kernel that is only faster with one."""
    from demon_b200 import _native as nat
    cache, ref, table, rows = filled([L], 128, Hk, cuda, 115)
    q, n, got = queries(1, Sq, Hq, cuda, Sq), i32([L], cuda), {}
    for name in ("", "small", "tc"):
        os.environ["DEMON_KV_ATTENTION"] = name
        got[name] = torch.full_like(q, 3)
        args = attention_args(q, cache, table, n, got[name], False)
        nat.check(nat.load().demon_kv_attention(bytes(args), nat.stream_ptr()))
        want, own = R.attention(q[0].double(), ref.values(0, rows[0], L), ref.values(1, rows[0], L), Sq, False, None, 128 ** -0.5)
        assert bool(((got[name][0].double() - want).abs() <= R.error_bound(want, own)).all())
    os.environ["DEMON_KV_ATTENTION"] = ""
    assert nat.load().demon_kv_attention_workspace(bytes(args)) > 0
    assert not torch.equal(got["small"], got["tc"]) and torch.equal(got[""], got["small"])
    ok()


@pytest.mark.parametrize("window", [-1, -2, -(1 << 40)])
def test_a_negative_window_is_refused(cuda, window):
    """None is no band; a negative one is a mistake, -1 (which means none in the C struct) as much as others."""
    from demon_b200 import _native as nat
    from demon_b200 import kvcache
    cache, _, table, _ = filled([40], 16, 2, cuda, 116)
    with pytest.raises(nat.DemonError, match="window"):
        kvcache.attention(queries(1, 1, 4, cuda, 1), cache, table, i32([40], cuda), window=window)


def test_append_refuses_one_buffer_for_k_and_v(cuda):
    """K and V may be one buffer for reading and attention, but not to write both into."""
    from demon_b200 import _native as nat
    from demon_b200 import kvcache
    cache, _, table, _ = filled([40], 16, 2, cuda, 117)
    x = queries(1, 3, 2, cuda, 1)
    for one in (kvcache.KVCache(cache.k, cache.k, cache.k_scale, cache.k_scale),
                kvcache.KVCache(cache.k, cache.v, cache.k_scale, cache.k_scale)):
        with pytest.raises(nat.DemonError, match="one buffer"):
            kvcache.append(one, x, x, table, i32([5], cuda))
    ok()


def test_a_cache_without_pages(cuda, which):
    """No page at all: nothing to append to, zeros read, rows that see no key."""
    from demon_b200 import _native as nat
    from demon_b200 import kvcache
    cache = kvcache.KVCache.empty(0, 2, 16, cuda)
    table, zero, one = i32([[-1, -1]], cuda), i32([0], cuda), i32([1], cuda)
    x = queries(1, 3, 2, cuda, 1)
    kvcache.append(cache, x, x, table, zero, zero)
    for Sq in (1, 140):
        assert not bool(kvcache.attention(queries(1, Sq, 4, cuda, 1), cache, table, zero).any())
    assert not bool(kvcache.read(cache, table, zero, 9)[0].any())
    ok()
    kvcache.append(cache, x, x, table, zero, one)
    for Sq in (1, 140):
        assert not bool(kvcache.attention(queries(1, Sq, 4, cuda, 1), cache, table, one).any())
    torch.cuda.synchronize()
    assert nat.device_status()[0] == BAD_ARG


@pytest.mark.parametrize("Sq,Hq,Hk,P,lens", [(40, 4, 2, 64, [5000, 3100]), (130, 8, 1, 16, [4000]), (300, 2, 2, 128, [9000, 0]),
                                             (70, 3, 1, 32, [1300]), (33, 100, 1, 64, [2200])])
def test_blocks_of_rows_without_a_workspace(cuda, Sq, Hq, Hk, P, lens):
    """The tensor-core kernel over whole key ranges where it would take parts with a workspace."""
    from demon_b200 import _native as nat
    cache, ref, table, rows = filled(lens, P, Hk, cuda, 119)
    q, n = queries(len(lens), Sq, Hq, cuda, Sq), i32(lens, cuda)
    os.environ["DEMON_KV_ATTENTION"] = "tc"
    out = torch.full_like(q, 3)
    args = attention_args(q, cache, table, n, out, True)
    assert nat.load().demon_kv_attention_workspace(bytes(args)) > 0
    nat.check(nat.load().demon_kv_attention(bytes(args), nat.stream_ptr()))
    for b, L in enumerate(lens):
        k, v = ref.values(0, rows[b], L), ref.values(1, rows[b], L)
        exact, own = R.attention(q[b].double(), k, v, Sq, True, None, 128 ** -0.5)
        assert bool(((out[b].double() - exact).abs() <= R.error_bound(exact, own)).all())
    ok()


@pytest.mark.parametrize("Sq,Hq", [(1, 16), (12, 2), (20_000, 16)])
def test_values_over_a_million_keys(cuda, Sq, Hq, which):
    """V of 1 + noise, so that an output is near 1 and the tolerance below means something: the table
    names 8 pages again and again, and every row equals the row over these 8 pages.

    Tolerance: two bf16 outputs, 2^-8 each at most; f16 probabilities 2^-11 of sum p |v| twice; the long
    call adds at most 2^16 matrix instructions of 16 keys into an fp32 accumulator, each dropping at most
    2^-23 of sum p |v|, and as many fp32 additions into the softmax sum (2^-24 each).
    """
    from demon_b200 import kvcache
    if Sq == 20_000 and which == "small":
        pytest.skip("the few-row kernel takes minutes for that many rows")
    table, rows, pages = make_table([1024], 128, cuda, 124)
    g = torch.Generator().manual_seed(124)
    cache, ref = kvcache.KVCache.empty(pages, 1, 128, cuda), R.RefCache(pages, 1, 128, cuda)
    k, v = torch.randn(1, 1024, 1, 128, generator=g), 1 + 0.25 * torch.randn(1, 1024, 1, 128, generator=g)
    k, v = k.to(torch.bfloat16).to(cuda), v.to(torch.bfloat16).to(cuda)
    kvcache.append(cache, k, v, table, i32([0], cuda))
    ref.append(k, v, rows, [0], [1024])
    q = queries(1, min(Sq, 500), Hq, cuda, 5)
    long = table[:, :8].repeat(1, 1024).contiguous()
    o = kvcache.attention(q.repeat(1, -(-Sq // 500), 1, 1), cache, long, i32([1 << 20], cuda))
    want, _ = R.attention(q[0].double(), ref.values(0, rows[0], 1024), ref.values(1, rows[0], 1024), q.shape[1], False, None, 128 ** -0.5)
    ok()
    mass, _ = R.attention(q[0].double(), ref.values(0, rows[0], 1024), ref.values(1, rows[0], 1024).abs(), q.shape[1], False, None,
                          128 ** -0.5)
    room = 2.0 ** -8 * want.abs() + (2.0 ** -10 + 2.0 ** 16 * (2.0 ** -23 + 2.0 ** -24)) * mass
    for i in range(0, Sq, 500 * 13):
        assert bool(((o[0, i:i + 500].double() - want[:o.shape[1] - i]).abs() <= room[:o.shape[1] - i]).all()), i
