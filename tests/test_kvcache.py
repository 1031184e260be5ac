"""CPU checks of the paged 8-bit K/V cache: the index arithmetic its kernels use (csrc/kv_index.h,
compiled here as plain C++), the Python side's refusals, and the 64-bit reference of the GPU tests
against exhaustive E4M3 tables."""
import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from kv_reference import RefCache, attention, e4m3, need_exp

ROOT = Path(__file__).resolve().parent.parent

HARNESS = r"""
#include "kv_index.h"
using namespace demon::kv;
extern "C" {
int span(int start, int count, int S, int cap, int* out) {
  Span s = append_span(start, count, S, cap);
  out[0] = s.start; out[1] = s.count;
  return s.bad;
}
int pages_of(int S, int P) { return append_pages(S, P); }
int page(const int32_t* row, int W, int i, long long pages) { return page_id(row, W, i, pages); }
int len_of(int len, int cap, int* bad) { bool b = false; int r = clamp_len(len, cap, &b); *bad = b; return r; }
void keys(int i0, int i1, int len, int nq, int causal, int window, int* out) {
  Keys k = visible(i0, i1, len, nq, causal != 0, window);
  out[0] = k.lo; out[1] = k.hi; out[2] = k.lo_all; out[3] = k.hi_all;
}
}
"""


@pytest.fixture(scope="module")
def index(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv_index")
    (d / "h.cpp").write_text(HARNESS)
    so = d / "h.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined",
                    "-fno-sanitize-recover=undefined", "-static-libubsan", "-shared", "-fPIC",
                    "-I", str(ROOT / "demon_b200" / "csrc"), str(d / "h.cpp"), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    lib.page.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_int, ctypes.c_longlong]
    return lib


def test_append_span_refuses_what_leaves_the_table(index):
    out = (ctypes.c_int * 2)()
    top = 1 << 30
    for start, count, S, cap, bad in [
        (0, 4, 4, 64, 0), (60, 4, 4, 64, 0), (64, 0, 4, 64, 0), (0, 0, 0, 0, 0), (top - 1, 1, 1, top, 0),
        (61, 4, 4, 64, 1), (-1, 2, 4, 64, 1), (0, -1, 4, 64, 1), (0, 5, 4, 64, 1), (65, 0, 4, 64, 1),
        (2147483647, 1, 1, top, 1), (2147483647, 2147483647, 2147483647, top, 1), (-2147483648, 1, 1, top, 1),
    ]:
        assert index.span(start, count, S, cap, out) == bad, (start, count, S, cap)
        assert (out[0], out[1]) == ((0, 0) if bad else (start, count))


def test_append_pages_covers_every_alignment(index):
    for P in (16, 32, 64, 128):
        for S in list(range(1, 300)) + [4095, 4096, 4097]:
            worst = max((s + S - 1) // P - s // P + 1 for s in range(P))
            assert index.pages_of(S, P) == worst
    assert index.pages_of(1 << 30, 16) == (1 << 26) + 1


def test_page_id_never_leaves_the_table_or_the_cache(index):
    row = (ctypes.c_int32 * 5)(3, -1, 7, 8, 2147483647)
    got = [index.page(row, 5, i, 8) for i in (-2147483648, -1, 0, 1, 2, 3, 4, 5, 2147483647)]
    assert got == [-1, -1, 3, -1, 7, -1, -1, -1, -1]


def test_lengths_are_clamped_and_reported(index):
    bad = ctypes.c_int()
    for n, cap, want, b in [(0, 0, 0, 0), (5, 64, 5, 0), (64, 64, 64, 0), (65, 64, 64, 1), (-1, 64, 0, 1),
                            (2147483647, 64, 64, 1), (-2147483648, 64, 0, 1)]:
        assert index.len_of(n, cap, ctypes.byref(bad)) == want and bad.value == b


def test_visible_ranges_match_enumeration(index):
    out = (ctypes.c_int * 4)()
    for n in (0, 1, 5, 12):
        for nq in (1, 3, 7, 15):
            for causal in (0, 1):
                for window in (-1, 0, 2, 9, (1 << 30) - 2):
                    for i0 in range(nq):
                        for i1 in range(i0, nq):
                            sets = []
                            for i in range(i0, i1 + 1):
                                pos = n - nq + i
                                sets.append({j for j in range(n) if (not causal or j <= pos)
                                             and (window < 0 or abs(pos - j) <= window)})
                            index.keys(i0, i1, n, nq, causal, window, out)
                            lo, hi, lo_all, hi_all = out
                            some, every = set.union(*sets), set.intersection(*sets)
                            assert some <= set(range(lo, hi)), (n, nq, causal, window, i0, i1)
                            assert set(range(lo_all, hi_all)) & set(range(n)) == every
                            assert 0 <= lo <= hi <= n and hi_all <= n


def test_visible_at_the_largest_sizes(index):
    """Nothing overflows at the limits (the harness traps signed overflow)."""
    out = (ctypes.c_int * 4)()
    top = 1 << 30
    index.keys(0, top - 1, top, top, 1, top - 2, out)
    assert (out[0], out[1]) == (0, top)
    index.keys(top - 1, top - 1, 0, top, 0, top - 2, out)
    index.keys(0, 0, 0, top, 1, top - 2, out)
    assert out[0] == out[1]


def test_reference_rounding_is_e4m3s():
    """Every E4M3 value is kept, and every midpoint goes to the even neighbour."""
    codes = torch.arange(0, 0x7F, dtype=torch.uint8)
    vals = codes.view(torch.float8_e4m3fn).double()
    assert torch.equal(e4m3(vals), vals) and torch.equal(e4m3(-vals), -vals)
    mid = (vals[:-1] + vals[1:]) / 2
    want = torch.where((codes[:-1] & 1) == 0, vals[:-1], vals[1:])
    assert torch.equal(e4m3(mid), want)
    assert float(e4m3(torch.tensor([1e300], dtype=torch.float64))) == 448.0
    x = torch.randn(20000, dtype=torch.float64).mul(30).to(torch.bfloat16)
    assert torch.equal(e4m3(x.double()).float(), x.float().to(torch.float8_e4m3fn).float())


def test_reference_exponent():
    assert [need_exp(a) for a in (0.0, 448.0, 448.1, 224.0, 224.5, 1e-40)] == [-120, 0, 1, -1, 0, -120]
    assert need_exp(3.3895e38) == 119


def test_reference_append_once_equals_token_by_token_scales():
    """The scale does not depend on how the tokens were split over appends."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(1, 40, 2, 128, generator=g).to(torch.bfloat16) * torch.linspace(0.1, 9, 40).view(1, 40, 1, 1).bfloat16()
    one, many = RefCache(3, 2, 16), RefCache(3, 2, 16)
    one.append(x, x, [[2, 0, 1]], [0], [40])
    for t in range(40):
        many.append(x[:, t:t + 1], x[:, t:t + 1], [[2, 0, 1]], [t], [1])
    assert torch.equal(one.exp, many.exp)
    # rounded once or again to a grown scale: at most half a step of the subnormal codes more
    assert float((one.codes - many.codes).abs().max()) <= 2.0 ** -9


def test_reference_attention_hides_by_selection():
    q = torch.randn(3, 2, 128, dtype=torch.float64)
    k, v = torch.randn(1, 3, 128, dtype=torch.float64), torch.randn(1, 3, 128, dtype=torch.float64)
    k[0, 2], v[0, 2, 5] = torch.nan, torch.nan
    o, _ = attention(q, k, v, 3, True, None, 0.1)
    assert bool(torch.isfinite(o[:2]).all()) and bool(torch.isnan(o[2]).all())


def test_cache_refuses_what_is_not_a_cuda_e4m3_cache():
    from demon_b200.kvcache import KVCache
    codes = torch.zeros(2, 1, 16, 128, dtype=torch.uint8).view(torch.float8_e4m3fn)
    s = torch.ones(2, 1)
    with pytest.raises(ValueError, match="CUDA"):
        KVCache(codes, codes, s, s)
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        KVCache(codes.view(torch.uint8), codes, s, s)
    with pytest.raises(ValueError, match="page_size"):
        KVCache(codes[:, :, :8].contiguous(), codes[:, :, :8].contiguous(), s, s)
    with pytest.raises(ValueError, match="k_scale"):
        KVCache(codes, codes, s.double(), s)
    with pytest.raises(ValueError, match="contiguous"):
        two = torch.cat([codes, codes], 1)
        KVCache(two.transpose(0, 1), two, s, s)


def test_struct_layouts_match_and_entry_points_refuse_without_a_gpu():
    from demon_b200 import _build, _native as nat
    _build.build()
    lib = nat.load()                       # checks the struct sizes
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    for fn, args in ((lib.demon_kv_append, nat.DemonKvAppendArgs()), (lib.demon_kv_read, nat.DemonKvReadArgs()),
                     (lib.demon_kv_attention, nat.DemonKvAttnArgs())):
        assert fn(bytes(args), None) != nat.DEMON_OK and nat.last_error()


def test_a_stream_of_another_device_is_refused():
    from types import SimpleNamespace

    from demon_b200.kvcache import _launch
    with pytest.raises(ValueError, match="stream is on cuda:1"):
        _launch(0, SimpleNamespace(device_index=1))


def test_rows_of_a_condition_cache_refuses_what_is_not_a_condition():
    from demon_b200.dit import CrossCache
    kv = CrossCache(None, torch.arange(6, dtype=torch.int32).view(3, 2), torch.tensor([5, 6, 7], dtype=torch.int32))
    got = kv.rows([2, 0, 0, 2])
    assert got.table.tolist() == [[4, 5], [0, 1], [0, 1], [4, 5]] and got.lens.tolist() == [7, 5, 5, 7]
    assert got.table.is_contiguous() and got.table.dtype == got.lens.dtype == torch.int32
    assert kv.rows(torch.tensor([1])).lens.tolist() == [6]
    assert kv.rows(torch.zeros(0, dtype=torch.int64)).table.shape == (0, 2)
    for bad in ([3], [0, -1], torch.tensor([0, 7])):
        with pytest.raises(IndexError, match="out of range"):
            kv.rows(bad)
    for bad in (1, [[0]], [0.5], torch.tensor([True, False, True])):
        with pytest.raises(ValueError, match="index"):
            kv.rows(bad)


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64, torch.uint16])
def test_rows_takes_every_integer_type_for_numbers(dtype):
    """torch takes a uint8 index for a mask; here it numbers conditions like any other."""
    from demon_b200.dit import CrossCache
    kv = CrossCache(None, torch.arange(6, dtype=torch.int32).view(3, 2), torch.tensor([5, 6, 7], dtype=torch.int32))
    for index in ([1, 1, 1], [0, 1, 1], [2, 0], [1, 0, 1, 2]):
        got = kv.rows(torch.tensor(index, dtype=dtype))
        assert got.table.tolist() == [[2 * i, 2 * i + 1] for i in index] and got.lens.tolist() == [5 + i for i in index]
    with pytest.raises(ValueError, match="index"):
        kv.rows(torch.tensor([1j]))


@pytest.mark.parametrize("n,W", [(3, 2), (1, 1), (0, 2), (0, 0)])
def test_rows_by_an_unread_index_never_leaves_the_conditions(n, W):
    """What a device index does, on the CPU: out of range is one token without a page, of no conditions too."""
    from demon_b200.dit import CrossCache
    table = torch.arange(n * W, dtype=torch.int32).view(n, W)
    kv = CrossCache(None, table, torch.zeros(n, dtype=torch.int32))     # (conditions without tokens: still reported)
    index = [-1, 0, n - 1, n, n + 7, -(1 << 40), 1 << 40]
    got = kv._chosen(torch.tensor(index))
    for row, length, i in zip(got.table.tolist(), got.lens.tolist(), index):
        assert (row, length) == ((table[i].tolist(), 0) if 0 <= i < n else ([-1] * W, 1))
    assert got.table.dtype == got.lens.dtype == torch.int32 and got.table.is_contiguous()
    assert kv._chosen(torch.zeros(0, dtype=torch.int64)).table.shape == (0, W)


def test_rows_of_an_empty_list():
    from demon_b200.dit import CrossCache
    kv = CrossCache(None, torch.arange(6, dtype=torch.int32).view(3, 2), torch.tensor([5, 6, 7], dtype=torch.int32))
    for none in ([], ()):
        got = kv.rows(none)
        assert got.table.shape == (0, 2) and got.lens.shape == (0,)
    with pytest.raises(ValueError, match="index"):
        kv.rows([[]])


@pytest.mark.parametrize("window", [-1, -2, -(1 << 40)])
def test_a_negative_window_is_refused(window):
    from types import SimpleNamespace

    from demon_b200 import _native as nat
    from demon_b200.kvcache import attention
    with pytest.raises(nat.DemonError, match="window"):
        attention(torch.zeros(1, 1, 1, 128), SimpleNamespace(_index=0), None, None, window=window)


def _attention_args(B, Sq, Hq, Hk, W, P, window=-1):
    """An argument block of these sizes; the planner looks at no buffer (only that there are some)."""
    from demon_b200 import _native as nat
    a = nat.DemonKvAttnArgs(B=B, Sq=Sq, Hq=Hq, W=W, window=window, causal=1, scale=0.1, q=16, o=16, table=16, ld_table=W, lens=16)
    a.cache = nat.DemonKvCache(k=16, v=16, k_scale=16, v_scale=16, pages=1, heads=Hk, page_size=P, head_dim=128)
    return bytes(a)


def test_workspaces_of_every_size_of_call():
    """Where the Python call does not ask for a workspace the planner would use none, and none exceeds 160 MB."""
    from demon_b200 import _build, _native as nat
    _build.build()
    size = nat.load().demon_kv_attention_workspace
    used = most = 0
    for Hk, G in ((1, 1), (8, 2), (4, 3), (2, 7), (1, 16), (8, 8), (1, 128), (1, 130)):
        for B in (1, 2, 3, 5, 9, 16, 18, 40, 73, 147):
            for Sq in (1, 2, 3, 5, 8, 16, 17, 33, 64, 100, 200, 500, 1000, 4000):
                few = Sq * G <= 16
                for keys in (16, 128, 512, 896, 912, 1024, 2048, 8128, 8192, 9600, 20000, 100000, 1 << 20):
                    for window in (-1, 500, 6000, 50000):
                        n = size(_attention_args(B, Sq, Hk * G, Hk, keys // 16, 16, window))
                        assert n >= 0 and (n == 0 or keys > (8_128 if few else 896)), (Hk, G, B, Sq, keys, window)
                        used, most = used + (n > 0), max(most, n)
    assert used > 1000 and 2 ** 26 < most <= 160_000_000
