"""The quantised K/V cache (append, read) and the attention over it against a
plain 64-bit implementation.  Stored values are exact; the attention's
tolerance is derived in decoder_reference.attention_tolerance."""
import ctypes

import numpy as np
import pytest
import torch

from iconnx_b200 import IcxError, _lib, kv_cache
from iconnx_b200.kv_cache import (KvCache, gpu_kv_cache_append, gpu_kv_cache_attention,
                                  gpu_kv_cache_read)
from tests import decoder_reference as ref

DEV = "cuda:0"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def f64(t):
    return t.detach().cpu().double().numpy()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def ends(counts):
    return [0, *np.cumsum(counts).tolist()]


def status():
    v = ctypes.c_int(0)
    assert _lib.load().icx_device_status(0, ctypes.byref(v)) == 0
    return v.value


class Case:
    """A pool filled with whole sequences of given lengths, pages in random order."""

    def __init__(self, lens, kv_heads=2, dim=64, bits=4, group=64, page=16, dtype=torch.float32, seed=0,
                 spread=1.0, width_extra=1):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.page = lens, page
        need = [-(-n // page) for n in lens]
        pool = sum(need) + 2
        perm = torch.randperm(pool, generator=g).tolist()
        table = torch.full((len(lens), max(need, default=0) + width_extra), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            for i in range(n):
                table[b, i] = perm.pop()
        self.table = table.to(DEV)
        self.cache = KvCache(pool, page, kv_heads, dim, bits, group, DEV)
        shape = (sum(lens), kv_heads, dim)
        self.k = (torch.randn(shape, generator=g) * spread + torch.randn(kv_heads, dim, generator=g)).to(dtype)
        self.v = torch.randn(shape, generator=g).to(dtype)
        gpu_kv_cache_append(self.cache, self.k.to(DEV), self.v.to(DEV), self.table, i32(lens), i32(ends(lens)))
        self.kv = [ref.cached_values(f64(x), bits, group) for x in (self.k, self.v)]

    def sequence(self, b):
        e = ends(self.lens)
        return [x[e[b]:e[b + 1]] for x in self.kv]


# ---------------------------------------------------------------- refusals
def c_args(**over):
    cache = dict(k_codes=16, v_codes=16, k_params=16, v_params=16, pages=4, page_size=16, kv_heads=2,
                 head_dim=64, bits=4, group=32)
    where = dict(d_page_table=16, d_seq_lens=16, d_cu_tokens=None, tokens=3, batch=3, table_width=4)
    for k, v in over.items():
        (cache if k in cache else where)[k] = v
    return _lib.KvCacheArg(*cache.values()), _lib.KvTokensArg(*where.values())


@pytest.mark.parametrize("over,text", [
    (dict(bits=5), b"bits"), (dict(head_dim=80), b"head_dim"), (dict(group=16), b"group"),
    (dict(page_size=24), b"page_size"), (dict(page_size=8), b"page_size"), (dict(page_size=2048), b"page_size"),
    (dict(kv_heads=0), b"kv_heads"), (dict(pages=-1), b"pages"), (dict(batch=-1), b"batch"),
    (dict(tokens=4), b"one token per sequence"), (dict(d_seq_lens=None), b"null index"),
    (dict(k_codes=None), b"null cache"), (dict(v_params=24), b"aligned"),
    (dict(table_width=1 << 28), b"2\\^31")])
def test_refusals_before_any_launch(over, text):
    import re
    L = _lib.load()
    p = ctypes.c_void_p(64)
    c, w = c_args(**over)
    for rc in (L.icx_kv_cache_append(None, ctypes.byref(c), ctypes.byref(w), p, p, 3, 64, 64, 64, 64, None, None),
               L.icx_kv_cache_read(None, ctypes.byref(c), ctypes.byref(w), 3, p, p),
               L.icx_kv_cache_attention(None, ctypes.byref(c), ctypes.byref(w), p, 3, 2, 128, 64, 1.0, p, None, 0)):
        assert rc == -1
        assert re.search(text, L.icx_last_error()), L.icx_last_error()


@pytest.mark.parametrize("page", [16, 64, 1024])
def test_page_tables_whose_last_positions_pass_32_bits_are_refused(page):
    L, p = _lib.load(), ctypes.c_void_p(64)
    for width in ((1 << 31) // page, (1 << 31) // page - 1, ((1 << 31) - 4096) // page + 1):
        c, w = (ctypes.byref(a) for a in c_args(page_size=page, table_width=width))
        for rc in (L.icx_kv_cache_append(None, c, w, p, p, 3, 64, 64, 64, 64, None, None),
                   L.icx_kv_cache_read(None, c, w, 3, p, p),
                   L.icx_kv_cache_attention(None, c, w, p, 3, 2, 128, 64, 1.0, p, None, 0)):
            assert rc == -1 and b"2^31 - 4096" in L.icx_last_error()
    # the widest table, of an empty call
    c, w = (ctypes.byref(a) for a in c_args(page_size=page, table_width=((1 << 31) - 4096) // page, tokens=0, batch=0))
    assert L.icx_kv_cache_read(None, c, w, 3, p, p) == 0


def test_operand_refusals_before_any_launch():
    L = _lib.load()
    p = ctypes.c_void_p(64)
    c, w = (ctypes.byref(a) for a in c_args())
    assert L.icx_kv_cache_append(None, None, w, p, p, 3, 1, 1, 1, 1, None, None) == -1
    assert L.icx_kv_cache_append(None, c, w, p, p, 0, 1, 1, 1, 1, None, None) == -1
    assert L.icx_kv_cache_append(None, c, w, None, p, 3, 1, 1, 1, 1, None, None) == -1
    assert L.icx_kv_cache_append(None, c, w, p, p, 3, -1, 1, 1, 1, None, None) == -1
    assert L.icx_kv_cache_append(None, c, w, p, p, 3, 1, 1, 1, 1, ctypes.c_void_p(8), None) == -1
    assert L.icx_kv_cache_read(None, c, w, 2, p, p) == -1
    assert L.icx_kv_cache_read(None, c, w, 3, ctypes.c_void_p(4), p) == -1
    for kw in (dict(t=1), dict(h=3), dict(h=0), dict(stride=-1), dict(scale=float("nan")), dict(q=None),
               dict(out=None)):
        a = dict(t=3, h=4, stride=64, scale=1.0, q=p, out=p) | kw
        assert L.icx_kv_cache_attention(None, c, w, a["q"], a["t"], a["h"], a["stride"], 64, a["scale"], a["out"],
                                        p, 1 << 30) == -1, kw
    with pytest.raises(IcxError, match="CUDA device"):
        KvCache(4, 16, 2, 64, device="cpu")
    for kw in (dict(bits=2), dict(head_dim=96), dict(group=128), dict(page_size=20), dict(kv_heads=0), dict(pages=-1)):
        with pytest.raises(IcxError):
            KvCache(**(dict(pages=4, page_size=16, kv_heads=2, head_dim=64) | kw))


@pytest.mark.parametrize("name", ["k_codes", "v_codes", "k_params", "v_params"])
def test_buffers_of_a_pool_cannot_be_replaced(name):
    """The calls keep their addresses: another tensor would not be used, and the
    one it replaces would be freed under them."""
    cache = object.__new__(KvCache)
    with pytest.raises(AttributeError):
        setattr(cache, name, torch.zeros(1))


@pytest.mark.gpu
def test_restored_pool_reads_the_same():
    c = Case([50, 20], seed=41)
    args = c.table, i32(c.lens), i32(ends(c.lens))
    want = gpu_kv_cache_read(c.cache, *args, tokens=70)
    other = KvCache(c.cache.pages, 16, 2, 64, 4, 64, DEV)
    for name in ("k_codes", "v_codes", "k_params", "v_params"):
        getattr(other, name).copy_(getattr(c.cache, name))
    got = gpu_kv_cache_read(other, *args, tokens=70)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_python_refusals():
    c = KvCache(4, 16, 2, 64, device=DEV)
    k = torch.zeros(2, 2, 64, device=DEV)
    table, lens = i32([[0], [1]]), i32([1, 1])
    gpu_kv_cache_append(c, k, k, table, lens)
    for a in ((k[:, :1], k, table, lens), (k, k.half(), table, lens), (k, k[:1], table, lens),
              (k.cpu(), k, table, lens), (k, k, table.long(), lens), (k, k, table, lens[:1]),
              (k, k, table[:1], lens[:1]), (k, k, table, lens, i32([0, 2])), (k.int(), k.int(), table, lens)):
        with pytest.raises(IcxError):
            gpu_kv_cache_append(c, *a)
    with pytest.raises(IcxError, match="tokens is needed"):
        gpu_kv_cache_read(c, table, lens, i32([0, 1, 2]))
    for kw in (dict(tokens=3), dict(dtype=torch.int8), dict(out=(k, k[:1])), dict(out=(k, k.half()))):
        with pytest.raises(IcxError):
            gpu_kv_cache_read(c, table, lens, **kw)
    q = torch.zeros(2, 4, 64, device=DEV)
    for a, kw in (((q[:, :3], table, lens), {}), ((q[..., :32], table, lens), {}), ((q[:1], table, lens), {}),
                  ((q, table, lens), dict(scale=float("inf"))), ((q, table, lens), dict(out=q.half())),
                  ((q.double(), table, lens), {})):
        with pytest.raises(IcxError):
            gpu_kv_cache_attention(c, *a, **kw)


# --------------------------------------------------------- append and read
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,bits,group,page", [(64, 4, 32, 16), (64, 8, 64, 32), (128, 4, 64, 16), (128, 8, 32, 64),
                                                 (256, 4, 32, 16), (256, 8, 64, 1024), (128, 4, 32, 128)])
def test_append_then_read_is_exact(dim, bits, group, page, dtype):
    lens = [1, 37, 16, 0, 65]
    c = Case(lens, 3, dim, bits, group, page, dtype, seed=dim + bits)
    got = gpu_kv_cache_read(c.cache, c.table, i32(lens), i32(ends(lens)), tokens=sum(lens))
    for g, want in zip(got, c.kv):
        # c * s + lo rounds once in f32
        np.testing.assert_array_equal(f64(g), want.astype(np.float32).astype(np.float64))
    # the newest tokens alone, in their own type
    news = [1, 5, 0, 0, 17]
    got = gpu_kv_cache_read(c.cache, c.table, i32(lens), i32(ends(news)), tokens=sum(news), dtype=dtype)
    for x, g in zip(c.kv, got):
        e = ends(lens)
        want = np.concatenate([x[e[b + 1] - n:e[b + 1]] for b, n in enumerate(news)])
        assert torch.equal(g.cpu(), torch.from_numpy(want).float().to(dtype))
    assert status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
def test_append_values_strides_and_positions(bits):
    """Packed QKV rows appended step by step equal one append of the whole."""
    H, D, page = 2, 128, 16
    lens = [21, 40]
    whole = Case(lens, H, D, bits, 64, page, torch.bfloat16, seed=4)
    c = KvCache(whole.cache.pages, page, H, D, bits, 64, DEV)
    done = [0, 0]
    while done != lens:
        news = [min(n - d, s) for n, d, s in zip(lens, done, (1, 7))]
        e = ends(lens)
        at = torch.cat([torch.arange(e[b] + done[b], e[b] + done[b] + n) for b, n in enumerate(news)])
        packed = torch.zeros(len(at), 3 * H * D + 3, dtype=torch.bfloat16, device=DEV)
        qkv = packed[:, 1:1 + 3 * H * D].view(len(at), 3 * H, D)   # rows off any alignment
        qkv[:, H:2 * H], qkv[:, 2 * H:] = whole.k[at].to(DEV), whole.v[at].to(DEV)
        done = [d + n for d, n in zip(done, news)]
        vals = gpu_kv_cache_append(c, qkv[:, H:2 * H], qkv[:, 2 * H:], whole.table, i32(done), i32(ends(news)),
                                   return_values=True)
        for got, x in zip(vals, whole.kv):
            assert torch.equal(got.cpu(), torch.from_numpy(x[at.numpy()]).float().bfloat16())
    for a, b in ((c.k_codes, whole.cache.k_codes), (c.v_codes, whole.cache.v_codes),
                 (c.k_params, whole.cache.k_params), (c.v_params, whole.cache.v_params)):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
def test_append_special_groups(bits):
    """Constant groups, ties, subnormal and huge ranges, NaN and infinities."""
    D, H, rows = 128, 1, 16
    g = torch.Generator().manual_seed(2)
    x = torch.randn(rows, H, D, generator=g)
    top = torch.finfo(torch.float32).max
    x[0] = 0
    x[1] = 0.1
    x[2] = -3.25
    x[3, 0, :64], x[3, 0, 64:] = torch.arange(64) * 0.5, torch.arange(64) * -0.25
    x[4] *= 1e-39
    x[5] *= 1e38
    x[6, 0, 3], x[6, 0, 4] = top, -top
    x[7, 0, 70] = float("nan")
    x[8, 0, 1] = float("inf")
    x[9, 0, 127] = float("-inf")
    x[10] = 1 + torch.arange(D) * 2.0 ** -23
    x[11] = -top
    x[12, 0] = torch.arange(D) * 2.0 ** -149
    x[13, 0, :64] = torch.arange(64) * 7.5 - 3   # exact halves of the step
    x[14] = 2.0 ** -133
    cache = KvCache(1, 16, H, D, bits, 64, DEV)
    vals = gpu_kv_cache_append(cache, x.to(DEV), x.to(DEV), i32([[0]]), i32([rows]), i32([0, rows]), return_values=True)
    want = ref.cached_values(f64(x), bits, 64).astype(np.float32)
    read = gpu_kv_cache_read(cache, i32([[0]]), i32([rows]), i32([0, rows]), tokens=rows)
    for got in (*vals, *read):
        np.testing.assert_array_equal(got.cpu().numpy(), want)


@pytest.mark.gpu
def test_rows_and_pages_that_are_not_named_stay():
    c = Case([20, 33], seed=1)
    before = [t.clone() for t in (c.cache.k_codes, c.cache.v_codes, c.cache.k_params, c.cache.v_params)]
    k = torch.randn(9, 2, 64, device=DEV)
    # rows 0, 1 and 7, 8 lie outside cu_tokens; sequence 0 has none; positions before 0 are skipped
    for lens, cu in (([20, 2], [2, 2, 7]), ([0, 0], [0, 4, 9])):
        gpu_kv_cache_append(c.cache, k, k, c.table, i32(lens), i32(cu))
        out = [torch.full((9, 2, 64), 5.0, device=DEV) for _ in range(2)]
        gpu_kv_cache_read(c.cache, c.table, i32(lens), i32(cu), tokens=9, out=out)
        stored = range(5, 7) if lens[1] else range(0)
        for o in out:
            for r in range(9):
                assert (o[r] == 5.0).all() != (r in stored)
    after = (c.cache.k_codes, c.cache.v_codes, c.cache.k_params, c.cache.v_params)
    page = int(c.table[1, 0])
    for a, b in zip(before, after):
        changed = (a != b).flatten(3).any(-1)          # [pages, heads, token]
        changed[page, :, :2] = False
        assert not changed.any()
    assert status() == 0


@pytest.mark.gpu
def test_unusable_pages_are_skipped_and_noted():
    c = Case([40, 40], seed=3)
    table = c.table.clone()
    table[0, 1] = -1
    table[1, 2] = c.cache.pages
    lens = i32([40, 40])
    k = torch.randn(80, 2, 64, device=DEV)
    before = c.cache.k_codes.clone()
    out = [torch.full((80, 2, 64), 5.0, device=DEV) for _ in range(2)]
    gpu_kv_cache_read(c.cache, table, lens, i32([0, 40, 80]), tokens=80, out=out)
    assert status() == _lib.ICX_DEVICE_BAD_PAGE
    for o in out:
        left = (o == 5.0).flatten(1).all(1).cpu()
        want = torch.zeros(80, dtype=torch.bool)
        want[16:32] = True
        want[72:80] = True
        assert torch.equal(left, want)
    gpu_kv_cache_append(c.cache, k, k, table, lens, i32([0, 40, 80]))
    assert status() == _lib.ICX_DEVICE_BAD_PAGE
    assert torch.equal(before[c.table[0, 1].long()], c.cache.k_codes[c.table[0, 1].long()])
    # a sequence longer than its row of the table
    gpu_kv_cache_read(c.cache, c.table[:, :1], lens, i32([0, 40, 80]), tokens=80, out=out)
    assert status() == _lib.ICX_DEVICE_BAD_PAGE
    # attention: the positions without a page take no part
    q = torch.randn(2, 2, 64, device=DEV)
    got = f64(gpu_kv_cache_attention(c.cache, q, table, lens))
    assert status() == _lib.ICX_DEVICE_BAD_PAGE
    kv = gpu_kv_cache_read(c.cache, c.table, lens, i32([0, 40, 80]), tokens=80)
    for b, gone in ((0, range(16, 32)), (1, range(32, 40))):
        keep = [40 * b + p for p in range(40) if p not in gone]
        kb, vb = (f64(x)[keep] for x in kv)
        want = ref.attention(f64(q[b:b + 1]), kb, vb, 0.125)
        tol = ref.attention_tolerance(f64(q[b:b + 1]), kb, vb, 0.125, torch.float32, want)
        assert (np.abs(got[b] - want[0]) <= tol[0]).all()


@pytest.mark.gpu
def test_a_bad_page_does_not_hide_a_wait_that_gave_up():
    L, timeout = _lib.load(), 0x1ff
    c = KvCache(4, 16, 2, 64, device=DEV)
    k = torch.zeros(1, 2, 64, device=DEV)

    def bad_page():
        gpu_kv_cache_append(c, k, k, i32([[-1]]), i32([1]))

    def wait():   # a bounded wait that nothing ends, 1 ms
        assert L.icx_selftest_bounded_wait(torch.cuda.current_stream(DEV).cuda_stream, 1_000_000) == 0

    status()
    for steps, want in (((bad_page,), _lib.ICX_DEVICE_BAD_PAGE), ((bad_page, wait), timeout), ((wait, bad_page), timeout),
                        ((bad_page, wait, bad_page), timeout)):
        for step in steps:
            step()
        torch.cuda.synchronize()
        assert status() == want
        assert status() == 0


# --------------------------------------------------------------- attention
def check_attention(c, news, q_heads, dtype, scale=None, seed=0, q_scale=1.0, pad=0):
    lens, D = c.lens, c.cache.head_dim
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(sum(news) + pad, q_heads, D, generator=g) * q_scale).to(dtype)
    cu = None if all(n == 1 for n in news) and not pad else i32(ends(news))
    out = torch.full((sum(news) + pad, q_heads, D), 7.0, dtype=dtype, device=DEV)
    got = gpu_kv_cache_attention(c.cache, q.to(DEV), c.table, i32(lens), cu, scale, out=out)
    assert got is out
    e = ends(news)
    s = D ** -0.5 if scale is None else scale
    for b, n in enumerate(news):
        if n == 0:
            continue
        k, v = c.sequence(b)
        qb = f64(q[e[b]:e[b + 1]])
        o = f64(out[e[b]:e[b + 1]])
        want = ref.attention(qb, k, v, s)
        if lens[b] == 0:
            assert (o == 0).all()
            continue
        tol = ref.attention_tolerance(qb, k, v, s, dtype, want)
        assert (np.abs(o - want) <= tol).all(), (b, np.abs(o - want).max(), tol.min())
    assert (out[sum(news):] == 7.0).all()
    assert status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim,group,heads,share", [(64, 32, 3, 1), (64, 64, 1, 8), (128, 64, 2, 4), (128, 32, 1, 7),
                                                   (256, 64, 1, 3), (256, 32, 2, 2)])
def test_attention_one_token(dim, group, heads, share, bits, dtype):
    lens = [1, 2, 15, 16, 17, 130, 0, 300]
    c = Case(lens, heads, dim, bits, group, 16, dtype, seed=dim + share)
    check_attention(c, [1] * len(lens), heads * share, dtype, seed=share)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,bits,share,news", [(128, 4, 4, [3, 1, 0, 16]), (64, 8, 1, [40, 7, 1, 100]),
                                                 (128, 4, 2, [200, 64, 33, 129]), (256, 4, 5, [9, 30, 2, 70]),
                                                 (128, 8, 16, [5, 1, 1, 21]), (64, 4, 3, [200, 180, 5, 129])])
def test_attention_several_tokens(dim, bits, share, news, dtype):
    lens = [200, 180, 33, 129]
    c = Case(lens, 2, dim, bits, 32 if dim == 64 else 64, 32, dtype, seed=dim + share)
    check_attention(c, news, 2 * share, dtype, seed=share, pad=3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_many_short_sequences(dtype):
    """More row tiles than CTAs at once, each within one warp."""
    lens = [(37 * b) % 61 for b in range(160)]
    c = Case(lens, 2, 128, 8, 64, 16, dtype, seed=31, width_extra=0)
    check_attention(c, [1] * 160, 4, dtype, seed=6)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,bits", [(64, 4), (64, 8), (128, 4), (256, 8)])
def test_attention_row_tile_per_cta(dim, bits, dtype):
    """Row tiles whose positions the warps of one CTA share: from none and one up."""
    lens = [440, 0, 1, 17, 130, 300]
    c = Case(lens, 2, dim, bits, 32, 16, dtype, seed=32 + dim)
    check_attention(c, [1] * 6, 6, dtype, seed=7)
    check_attention(c, [3, 0, 1, 5, 2, 9], 10, dtype, seed=8, pad=2)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 64, 1024])
def test_attention_long_and_ragged(page):
    """Long sequences beside short ones: work split over the positions and joined."""
    lens = [5000, 3, 1029, 0, 2048]
    c = Case(lens, 1, 128, 4, 64, page, torch.float32, seed=page)
    check_attention(c, [1] * 5, 4, torch.float32, seed=1)
    check_attention(c, [3, 1, 2, 0, 1], 4, torch.float32, seed=2)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_many_rows(dim):
    """Long runs of new tokens, with and without a cached prefix."""
    lens = [700, 257, 300]
    c = Case(lens, 2, dim, 4, 64, 64, torch.bfloat16, seed=dim)
    check_attention(c, [300, 257, 1], 8, torch.bfloat16, seed=3, pad=5)
    c = Case(lens, 1, dim, 8, 32, 16, torch.float32, seed=dim + 1)
    check_attention(c, [130, 200, 300], 3, torch.float32, seed=4)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,bits,share", [(64, 4, 2), (64, 8, 4), (128, 4, 8), (128, 8, 1)])
def test_attention_prompt_chunks(dim, bits, share, dtype):
    """Prompt chunks in the 16-bit types: tiles that end inside a page, chunks of
    every alignment, a sequence whose first rows see almost nothing."""
    lens = [129, 64, 200, 1, 333]
    c = Case(lens, 2, dim, bits, 64, 16, dtype, seed=dim + bits)
    check_attention(c, [129, 63, 70, 1, 130], 2 * share, dtype, seed=share, pad=2)
    check_attention(c, [129, 64, 200, 1, 333], 2 * share, dtype, -0.05, seed=share + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompt_chunks_with_missing_pages_and_nan(dtype):
    """Rows meet neither the positions of a missing page nor a NaN they do not see."""
    c = Case([150], 1, 128, 4, 64, 16, dtype, seed=21)
    q = torch.randn(100, 4, 128).to(dtype)
    lens, cu = i32([150]), i32([0, 100])
    table = c.table.clone()
    table[0, 2] = -1
    out = f64(gpu_kv_cache_attention(c.cache, q.to(DEV), table, lens, cu))
    assert status() == _lib.ICX_DEVICE_BAD_PAGE
    keep = [p for p in range(150) if not 32 <= p < 48]
    k, v = (x[keep] for x in c.sequence(0))
    want = ref.attention(f64(q), k, v, 128 ** -0.5)
    tol = ref.attention_tolerance(f64(q), k, v, 128 ** -0.5, dtype, want)
    assert (np.abs(out - want) <= tol).all()
    # position 120's V is NaN in the first group: rows from 70 on, dimensions 0..63
    bad = c.v[120:121].clone()
    bad[..., 5] = float("nan")
    gpu_kv_cache_append(c.cache, c.k[120:121].to(DEV), bad.to(DEV), c.table, i32([121]), i32([0, 1]))
    out = gpu_kv_cache_attention(c.cache, q.to(DEV), c.table, lens, cu)
    nan = out.isnan()
    assert nan[70:, :, :64].all() and not nan[:70].any() and not nan[..., 64:].any()
    # and with a NaN K, every dimension of the rows that see it
    gpu_kv_cache_append(c.cache, bad.to(DEV), c.v[120:121].to(DEV), c.table, i32([121]), i32([0, 1]))
    nan = gpu_kv_cache_attention(c.cache, q.to(DEV), c.table, lens, cu).isnan()
    assert nan[70:].all() and not nan[:70].any()
    assert status() == 0


@pytest.mark.gpu
def test_prompt_chunk_values_of_unequal_size():
    """V groups and K scales of very different sizes in one prompt chunk."""
    c = Case([300], 1, 128, 4, 64, 16, torch.bfloat16, seed=22)
    k = (c.k * torch.linspace(0.1, 2.0, 300)[:, None, None]).bfloat16()
    v = (c.v * torch.pow(10.0, torch.arange(300) % 5 - 4.0)[:, None, None]).bfloat16()
    gpu_kv_cache_append(c.cache, k.to(DEV), v.to(DEV), c.table, i32([300]), i32([0, 300]))
    c.kv = [ref.cached_values(f64(x), 4, 64) for x in (k, v)]
    check_attention(c, [200], 4, torch.bfloat16, seed=8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompt_output_of_small_weights(dtype):
    """One position holds nearly all the weight and no value; what the others
    (2^-20 of its weight each) give is as exact as an output should be."""
    n, D = 600, 64
    c = Case([n], 1, D, 8, 64, 16, dtype, seed=26)
    g = torch.Generator().manual_seed(27)
    k = torch.randn(n, 1, D, generator=g) * 0.01
    v = 1.0 + 0.1 * torch.rand(n, 1, D, generator=g)
    k[0], v[0] = 1.0, 0.0
    k, v = k.to(dtype), v.to(dtype)
    gpu_kv_cache_append(c.cache, k.to(DEV), v.to(DEV), c.table, i32([n]), i32([0, n]))
    kc, vc = (ref.cached_values(f64(x), 8, 64) for x in (k, v))
    q = (torch.full((80, 2, D), 20 * np.log(2.0) / (D * D ** -0.5)) + 0.01 * torch.randn(80, 2, D, generator=g)).to(dtype)
    out = f64(gpu_kv_cache_attention(c.cache, q.to(DEV), c.table, i32([n]), i32([0, 80])))
    want = ref.attention(f64(q), kc, vc, D ** -0.5)
    assert 1e-4 < want.min() and want.max() < 1e-3
    # every value is positive, so relative errors do not grow in the sum: the
    # output's half step (f16: in its subnormals' 2^-25 besides), a weight and a
    # value to f16 (2^-12 each), K and q as there is nothing to cancel: |S| 2^-11
    tol = np.abs(want) * (torch.finfo(dtype).eps / 2 + 2 * 2.0 ** -12 + 14 * 2.0 ** -11) + 2.0 ** -25
    assert (np.abs(out - want) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
def test_prompt_rows_beside_much_larger_values_they_do_not_see(bits):
    """A position 2^18 times as large as the others leaves the rows before it as exact."""
    c = Case([180], 1, 128, bits, 64, 16, torch.bfloat16, seed=24)
    v = c.v.clone()
    v[150] *= 2.0 ** 18
    gpu_kv_cache_append(c.cache, c.k.to(DEV), v.to(DEV), c.table, i32([180]), i32([0, 180]))
    c.kv[1] = ref.cached_values(f64(v), bits, 64)
    check_attention(c, [130], 4, torch.bfloat16, seed=9)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,bits,share", [(64, 8, 4), (128, 4, 4), (128, 8, 8)])
def test_prompt_chunks_on_long_prefixes(dim, bits, share, dtype):
    """Few rows and many positions, which are read in shares: some shares of the
    shorter sequences hold nothing, and the first rows of one see few positions."""
    lens = [2900, 70, 0, 1000]
    c = Case(lens, 2, dim, bits, 64, 16, dtype, seed=dim + bits + 1, width_extra=60)
    check_attention(c, [65, 70, 0, 129], 2 * share, dtype, seed=share + 2, pad=1)
    check_attention(c, [20, 20, 0, 300], 2 * share, dtype, seed=share + 3, q_scale=6.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompt_shares_with_missing_pages_and_nan(dtype):
    c = Case([2000], 1, 128, 4, 64, 16, dtype, seed=25)
    q = torch.randn(100, 4, 128).to(dtype)
    lens, cu = i32([2000]), i32([0, 100])
    table = c.table.clone()
    table[0, 3:90] = -1     # more than the first share
    out = f64(gpu_kv_cache_attention(c.cache, q.to(DEV), table, lens, cu))
    assert status() == _lib.ICX_DEVICE_BAD_PAGE
    k, v = (np.delete(x, np.s_[48:1440], 0) for x in c.sequence(0))
    want = ref.attention(f64(q), k, v, 128 ** -0.5)
    tol = ref.attention_tolerance(f64(q), k, v, 128 ** -0.5, dtype, want)
    assert (np.abs(out - want) <= tol).all()
    out = gpu_kv_cache_attention(c.cache, q.to(DEV), torch.full_like(table, -1), lens, cu)
    assert status() == _lib.ICX_DEVICE_BAD_PAGE and (out == 0).all()
    bad = c.v[1950:1951].clone()
    bad[..., 70] = float("nan")
    gpu_kv_cache_append(c.cache, c.k[1950:1951].to(DEV), bad.to(DEV), c.table, i32([1951]), i32([0, 1]))
    nan = gpu_kv_cache_attention(c.cache, q.to(DEV), c.table, lens, cu).isnan()
    assert nan[50:, :, 64:].all() and not nan[:50].any() and not nan[..., :64].any()
    assert status() == 0


def bounded_attention(q, k, v, scale, dtype, operand, parts=None):
    """(want, bound of |out - want|) of q [n, heads, D], the last n of k, v [len,
    kv_heads, D], all f64 on the GPU.  With r the half step of the operands that K,
    V and the weights pass through (f16: 2^-11; 0 where they keep f32's bits) and
    32-bit sums of D products, a score is off by e = (r + D 2^-24) sum |q k| scale
    and its weight by exp(e) - 1; a weight and a value are off by r, an exponential
    by 2^-20, and n weighted values in 32 bits by n 2^-24 of their largest sum
    (parts: what is summed in a value's place, where that is larger: its scaled
    code and its group's low end, with weights split at 2^-22)."""
    n, hq, D = q.shape
    length, hk = k.shape[:2]
    q, k, v = q.transpose(0, 1), *(x.transpose(0, 1).repeat_interleave(hq // hk, 0) for x in (k, v))
    s = q @ k.transpose(1, 2) * scale
    last = torch.arange(length - n, length, device=q.device)[:, None]
    s.masked_fill_(torch.arange(length, device=q.device) > last, -torch.inf)
    p = torch.softmax(s, -1)
    want = p @ v
    e = torch.expm1((operand + D * 2.0 ** -24) * (q.abs() @ k.abs().transpose(1, 2)) * abs(scale))
    e = p * (e + operand + 2.0 ** -20)
    off = e.sum(-1, keepdim=True)
    assert off.max() < 0.5
    far = p @ v.abs() * (operand + length * 2.0 ** -24)
    if parts is not None:
        far += p @ parts.transpose(0, 1).repeat_interleave(hq // hk, 0) * (2.0 ** -22 + length * 2.0 ** -24)
    tol = (e @ v.abs() + off * want.abs() + far) / (1 - off) + v.abs().max() * length * 2.0 ** -39
    want, tol = (x.transpose(0, 1).cpu().numpy() for x in (want, tol))
    return want, ref.rounding(want, tol, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,bits,tokens", [(64, 4, 1200), (64, 8, 1217), (128, 4, 1217), (128, 8, 1200)])
def test_prompt_rows_that_fill_the_gpu(dim, bits, tokens, dtype):
    """Enough rows for 256 per CTA in bf16 (the last ones over and under 128), whose
    scores grow along the positions: every 32 tokens (128 rows) at another rate, so
    that the reference moves in every tile of some rows and late and seldom in the
    rows beside them."""
    heads, share, page, prefix = 8, 4, 16, 150
    lens, news = [tokens + prefix, 70], [tokens, 20]
    g = torch.Generator(DEV).manual_seed(dim + bits)
    cache = KvCache(100, page, heads, dim, bits, 64, DEV)
    need = -(-lens[0] // page)
    order = torch.randperm(100, generator=g, device=DEV).int()
    table = torch.full((2, need), -1, dtype=torch.int32, device=DEV)
    table[0], table[1, :5] = order[:need], order[need:need + 5]
    k, v = torch.randn(2, sum(lens), heads, dim, generator=g, device=DEV)
    k[:lens[0], :, 0] = torch.linspace(0, 10, lens[0], device=DEV)[:, None]
    gpu_kv_cache_append(cache, k.to(dtype), v.to(dtype), table, i32(lens), i32(ends(lens)))
    kc, vc = (x.double() for x in gpu_kv_cache_read(cache, table, i32(lens), i32(ends(lens)), tokens=sum(lens)))
    # powers of two of weight over the whole sequence: 200, 40, -90 (the first position leads), 10
    rate = torch.tensor([200.0, 40.0, -90.0, 10.0], device=DEV) * np.log(2.0) * dim ** 0.5 / 10
    q = 0.5 * torch.randn(sum(news), heads * share, dim, generator=g, device=DEV)
    q[:tokens, :, 0] = rate[torch.arange(tokens, device=DEV) // 32 % 4][:, None]
    q = q.to(dtype)
    out = gpu_kv_cache_attention(cache, q, table, i32(lens), i32(ends(news)))
    for _ in range(8):
        assert torch.equal(gpu_kv_cache_attention(cache, q, table, i32(lens), i32(ends(news))), out)
    for a, n, la, ln in ((0, news[0], 0, lens[0]), (news[0], news[1], lens[0], lens[1])):
        want, tol = bounded_attention(q[a:a + n].double(), kc[la:la + ln], vc[la:la + ln], dim ** -0.5, dtype,
                                      2.0 ** -11 if dtype == torch.bfloat16 else 0.0)
        off = np.abs(f64(out[a:a + n]) - want)
        assert (off <= tol).all(), (off / tol).max()
    assert status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompt_rows_that_fill_the_gpu_with_missing_pages_and_nan(dtype):
    tokens, heads, share, dim, page = 1200, 8, 4, 64, 32
    g = torch.Generator(DEV).manual_seed(51)
    need = -(-tokens // page)
    cache = KvCache(need, page, heads, dim, 8, 64, DEV)
    table = torch.randperm(need, generator=g, device=DEV).int()[None]
    lens, cu = i32([tokens]), i32([0, tokens])
    k, v = (x.to(dtype) for x in torch.randn(2, tokens, heads, dim, generator=g, device=DEV))
    v[700, 3, 9] = float("nan")    # rows from 700 on, K/V head 3
    k[900, 5, 1] = float("inf")    # rows from 900 on, K/V head 5
    gpu_kv_cache_append(cache, k, v, table, lens, cu)
    kc, vc = (x.double() for x in gpu_kv_cache_read(cache, table, lens, cu, tokens=tokens))
    q = torch.randn(tokens, heads * share, dim, generator=g, device=DEV).to(dtype)
    gone = table.clone()
    gone[0, 3:5], gone[0, 20] = -1, need
    out = gpu_kv_cache_attention(cache, q, gone, lens, cu)
    assert status() == _lib.ICX_DEVICE_BAD_PAGE
    nan = torch.zeros(out.shape, dtype=torch.bool, device=DEV)
    nan[700:, 3 * share:4 * share] = True
    nan[900:, 5 * share:6 * share] = True
    assert torch.equal(out.isnan(), nan)
    # the missing positions as zero weight: K that no row can prefer
    mask = torch.zeros(tokens, device=DEV, dtype=torch.bool)
    mask[96:160], mask[640:672] = True, True
    keep = torch.arange(tokens, device=DEV)[~mask]
    for row in (95, 96, 130, 160, 641, 699, 1199):   # each row over what it sees
        seen = keep[keep <= row]
        fine = [h for h in range(heads * share) if not nan[row, h, 0]]
        kr, vr = (x[seen].repeat_interleave(share, 1)[:, fine] for x in (kc, vc))
        want, tol = bounded_attention(q[row:row + 1, fine].double(), kr, vr, dim ** -0.5, dtype, 2.0 ** -11)
        assert (np.abs(f64(out[row:row + 1, fine]) - want) <= tol).all(), row


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompt_chunks_captured_and_replayed_with_other_lengths(dtype):
    """Few rows on a wide table (positions in shares) and many rows."""
    for tokens, width, batch in ((130, 120, 2), (1300, 90, 2)):
        heads, share, dim, page = 8, 4, 64, 16
        g = torch.Generator(DEV).manual_seed(tokens)
        pool = width * batch
        cache = KvCache(pool, page, heads, dim, 4, 64, DEV)
        table = torch.randperm(pool, generator=g, device=DEV).int().view(batch, width)
        full = i32([width * page] * batch)
        k, v = (x.to(dtype) for x in torch.randn(2, pool * page, heads, dim, generator=g, device=DEV))
        gpu_kv_cache_append(cache, k, v, table, full, i32(ends([width * page] * batch)))
        q = torch.randn(tokens, heads * share, dim, generator=g, device=DEV).to(dtype)
        lens, cu = i32([0] * batch), i32([0] * (batch + 1))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = gpu_kv_cache_attention(cache, q, table, lens, cu)
        half = tokens // 2
        for ln, c in (([width * page, half], [0, half, tokens]), ([half + 1, 5], [0, 1, 6]),
                      ([tokens - 3, width * page], [0, tokens - 2, tokens]), ([0, 0], [0, half, tokens]),
                      ([1, width * page], [0, 0, tokens])):
            lens.copy_(i32(ln))
            cu.copy_(i32(c))
            out.fill_(3.0)
            graph.replay()
            want = gpu_kv_cache_attention(cache, q, table, lens, cu, out=torch.full_like(out, 3.0))
            assert torch.equal(out, want), (tokens, ln, c)
            assert (out[c[-1]:] == 3.0).all()
    assert status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,bits,group", [(64, 8, 64), (128, 4, 64), (128, 8, 32), (256, 8, 64)])
def test_attention_beside_a_strong_dimension(dim, bits, group, dtype):
    """One dimension of -50 in each group of V: the group's low end is far from the
    other values, which keep their bits all the same."""
    lens, heads, share = [40, 7, 33], 2, 3
    g = torch.Generator(DEV).manual_seed(dim + bits)
    cache = KvCache(16, 16, heads, dim, bits, group, DEV)
    table = torch.randperm(16, generator=g, device=DEV).int()[:9].view(3, 3)
    k, v = torch.randn(2, sum(lens), heads, dim, generator=g, device=DEV)
    v[..., 5::group] = -50
    gpu_kv_cache_append(cache, k.to(dtype), v.to(dtype), table, i32(lens), i32(ends(lens)))
    kc, vc = (x.double() for x in gpu_kv_cache_read(cache, table, i32(lens), i32(ends(lens)), tokens=sum(lens)))
    low = vc.unflatten(-1, (-1, group)).amin(-1).repeat_interleave(group, -1)
    for news in ([1, 1, 1], [5, 7, 2]):
        q = (2 * torch.randn(sum(news), heads * share, dim, generator=g, device=DEV)).to(dtype)
        out = gpu_kv_cache_attention(cache, q, table, i32(lens), i32(ends(news)))
        for b, n in enumerate(news):
            a, la, le = ends(news)[b], ends(lens)[b], ends(lens)[b + 1]
            want, tol = bounded_attention(q[a:a + n].double(), kc[la:le], vc[la:le], dim ** -0.5, dtype, 0.0,
                                          low[la:le].abs() + (vc - low)[la:le])
            off = np.abs(f64(out[a:a + n]) - want)
            assert (off <= tol).all(), (off / tol).max()
    assert status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,bits,group,news,batch", [(64, 4, 64, 1, 600), (128, 8, 32, 1, 300), (64, 8, 64, 9, 100),
                                                       (256, 4, 64, 1, 300), (256, 8, 64, 1, 300)])
def test_attention_sums_of_long_sequences(dim, bits, group, news, batch, dtype):
    """Many sequences over the pages of one: a warp's share is thousands of positions."""
    check_long_sums(dim, bits, group, news, batch, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,bits", [(64, 4), (64, 8), (128, 4), (128, 8)])
def test_prompt_sums_of_long_sequences(dim, bits, dtype):
    """Enough rows that each reads its thousands of positions in one share."""
    check_long_sums(dim, bits, 64, 400, 12, dtype, 2.0 ** -11 if dtype == torch.bfloat16 else 0.0)


def check_long_sums(dim, bits, group, news, batch, dtype, operand=0.0):
    """Values around zero whose average is small beside them: matrix units cut what
    falls off the end of a sum, always towards zero, so that one sum over all the
    positions would drift by its number of products."""
    length, heads, share, page = 12000, 4, 4, 64
    g = torch.Generator(DEV).manual_seed(dim + bits)
    need = -(-length // page)
    cache = KvCache(need, page, heads, dim, bits, group, DEV)
    table = torch.randperm(need, generator=g, device=DEV).int()[None]
    k, v = torch.randn(2, length, heads, dim, generator=g, device=DEV)
    gpu_kv_cache_append(cache, k.to(dtype), v.to(dtype), table, i32([length]), i32([0, length]))
    kc, vc = (x.double() for x in gpu_kv_cache_read(cache, table, i32([length]), i32([0, length]), tokens=length))
    q = torch.randn(batch * news, heads * share, dim, generator=g, device=DEV).to(dtype)
    out = gpu_kv_cache_attention(cache, q, table.expand(batch, -1), i32([length] * batch),
                                 i32(ends([news] * batch)))
    low = vc.unflatten(-1, (-1, group)).amin(-1).repeat_interleave(group, -1)
    parts = (low.abs() + (vc - low)).mean(0).amax()
    drift = []
    for b in range(0, batch, 7):
        want, tol = bounded_attention(q[b * news:(b + 1) * news].double(), kc, vc, dim ** -0.5, dtype, operand,
                                      low.abs() + (vc - low))
        off = f64(out[b * news:(b + 1) * news]) - want
        assert (np.abs(off) <= tol).all(), (np.abs(off) / tol).max()
        drift.append(off.mean())
    # At most 64 products (32 steps of two parts; 8 tiles of 64 positions in two
    # parts) in a piece, each cutting up to 2^-23 of the piece's sum and so 2^-24 of
    # it on average over its growth (which the last of them sees whole: 64 2^-24),
    # and rounding errors, which have no side: half a step of outputs up to 2^-2 (of
    # 2^-24 parts in f32), averaged
    n = len(drift) * news * heads * share * dim
    side = max(2.0 ** -2 * ref.HALF_STEP[dtype], parts.item() * length ** 0.5 * 2.0 ** -24)
    limit = 64 * 2.0 ** -24 * parts.item() + 5 * side / n ** 0.5
    assert abs(np.mean(drift)) <= limit, (np.mean(drift), limit)
    assert status() == 0


@pytest.mark.gpu
def test_attention_scales_and_strong_scores():
    """Scores of order 100 (one position takes all), scale 0, negative scale, tiny and huge q."""
    for spread, q_scale, scale in ((4.0, 4.0, 0.5), (1.0, 1.0, 0.0), (1.0, 1.0, -0.3), (1.0, 1e-6, None),
                                   (1e-3, 3e4, 1e-3), (1.0, 300.0, 1.0)):
        c = Case([77, 400], 2, 128, 8, 64, 16, torch.float32, seed=11, spread=spread)
        check_attention(c, [1, 1], 4, torch.float32, scale, seed=5, q_scale=q_scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("prompt,others", [(400, 63), (1500, 40)])
def test_attention_of_a_prompt_beside_decoding_sequences(prompt, others, dtype):
    """One call for a prompt chunk and sequences of one token: of 6 and of 38 tokens on
    average, so that with four query heads for a K/V head the one takes the kernel for
    few rows and the other, in 16 bits, that for prompts."""
    heads, share, dim, page = 2, 4, 128, 32
    g = torch.Generator(DEV).manual_seed(prompt)
    lens = [(prompt + 300) if b == others // 2 else 1 + (b * 97) % 900 for b in range(others + 1)]
    news = [prompt if b == others // 2 else 1 for b in range(others + 1)]
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need), generator=g, device=DEV).int()
    table = torch.full((others + 1, max(need)), -1, dtype=torch.int32, device=DEV)
    for b, n in enumerate(need):
        table[b, :n] = order[ends(need)[b]:ends(need)[b + 1]]
    cache = KvCache(sum(need), page, heads, dim, 4, 64, DEV)
    k, v = torch.randn(2, sum(lens), heads, dim, generator=g, device=DEV)
    gpu_kv_cache_append(cache, k.to(dtype), v.to(dtype), table, i32(lens), i32(ends(lens)))
    kc, vc = (x.double() for x in gpu_kv_cache_read(cache, table, i32(lens), i32(ends(lens)), tokens=sum(lens)))
    low = vc.unflatten(-1, (-1, 64)).amin(-1).repeat_interleave(64, -1)
    q = torch.randn(sum(news), heads * share, dim, generator=g, device=DEV).to(dtype)
    out = gpu_kv_cache_attention(cache, q, table, i32(lens), i32(ends(news)))
    rounded = dtype == torch.bfloat16 and sum(news) // (others + 1) * share >= 64
    for b, n in enumerate(news):
        a, la, le = ends(news)[b], ends(lens)[b], ends(lens)[b + 1]
        want, tol = bounded_attention(q[a:a + n].double(), kc[la:le], vc[la:le], dim ** -0.5, dtype,
                                      2.0 ** -11 if rounded else 0.0, low[la:le].abs() + (vc - low)[la:le])
        off = np.abs(f64(out[a:a + n]) - want)
        assert (off <= tol).all(), (b, (off / tol).max())
    assert status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("q_scale,scale", [(1.0, 1e-44), (1e-30, 1e-25)])
def test_attention_of_scores_that_vanish(q_scale, scale, dtype):
    """A scale and queries so small that their product is below f32: the average
    of the positions that a row sees."""
    c = Case([77, 400, 3], 2, 128, 4, 64, 16, dtype, seed=34)
    check_attention(c, [1, 1, 1], 4, dtype, scale, seed=5, q_scale=q_scale)
    check_attention(c, [70, 130, 3], 4, dtype, scale, seed=6, q_scale=q_scale)


@pytest.mark.gpu
def test_attention_values_of_unequal_size():
    """Values whose groups differ by many orders of magnitude, token by token."""
    c = Case([90], 1, 128, 4, 64, 16, torch.float32, seed=12)
    k = c.k.to(DEV)
    v = (c.v * torch.pow(10.0, torch.arange(90) % 13 - 6.0)[:, None, None]).to(DEV)
    gpu_kv_cache_append(c.cache, k, v, c.table, i32([90]), i32([0, 90]))
    c.kv[1] = ref.cached_values(f64(v), 4, 64)
    check_attention(c, [1], 4, torch.float32, seed=6)
    check_attention(c, [80], 2, torch.float32, seed=7)


@pytest.mark.gpu
def test_attention_ignores_what_lies_behind():
    """NaN in unused rows of pages, and in other sequences, reaches nobody."""
    c = Case([21, 30, 260], 2, 128, 4, 64, 16, torch.bfloat16, seed=13)
    nan = torch.full((64, 2, 128), float("nan"), device=DEV, dtype=torch.bfloat16)
    lens = i32(c.lens)
    for b, n in enumerate(c.lens):   # fill the tail of each last page
        tail = -n % 16
        table = c.table[b:b + 1]
        if tail:
            gpu_kv_cache_append(c.cache, nan[:tail], nan[:tail], table, i32([n + tail]), i32([0, tail]))
    check_attention(c, [1, 1, 1], 8, torch.bfloat16, seed=1)
    check_attention(c, [5, 30, 250], 8, torch.bfloat16, seed=2)
    # a NaN inside a sequence does reach that sequence's later rows, and them alone
    gpu_kv_cache_append(c.cache, nan[:1], nan[:1], c.table[1:2], i32([30]), i32([0, 1]))
    out = gpu_kv_cache_attention(c.cache, torch.randn(32, 8, 128, device=DEV, dtype=torch.bfloat16), c.table, lens,
                                 i32([0, 1, 31, 32]))
    bad = out.isnan().flatten(1)
    assert bad[30].all() and not bad[:30].any() and not bad[31].any()


@pytest.mark.gpu
def test_attention_strided_queries_and_more_new_tokens_than_positions():
    c = Case([10, 50], 2, 64, 8, 32, 16, torch.float16, seed=14)
    packed = torch.randn(60, 12, 64, device=DEV).half()
    q = packed[:, 4:8]
    got = gpu_kv_cache_attention(c.cache, q, c.table, i32([10, 50]), i32([0, 30, 60]))
    want = gpu_kv_cache_attention(c.cache, q.contiguous(), c.table, i32([10, 50]), i32([0, 30, 60]))
    assert torch.equal(got, want)
    assert (got[:20] == 0).all() and (got[20:] != 0).flatten(1).any(1).all()
    part = gpu_kv_cache_attention(c.cache, q[20:30], c.table[:1], i32([10]), i32([0, 10]))
    np.testing.assert_allclose(f64(part), f64(got[20:30]), atol=2e-3)
    every_other = gpu_kv_cache_attention(c.cache, packed[::2, ::3], c.table[1:], i32([50]), i32([0, 30]))
    want = gpu_kv_cache_attention(c.cache, packed[::2, ::3].contiguous(), c.table[1:], i32([50]), i32([0, 30]))
    assert torch.equal(every_other, want)


@pytest.mark.gpu
def test_empty_calls():
    c = KvCache(0, 16, 2, 64, device=DEV)
    none = torch.zeros(0, 2, 64, device=DEV)
    table, lens = torch.zeros(0, 4, dtype=torch.int32, device=DEV), i32([])
    assert gpu_kv_cache_append(c, none, none, table, lens) is None
    assert gpu_kv_cache_read(c, table, lens)[0].shape == (0, 2, 64)
    assert gpu_kv_cache_attention(c, none, table, lens).shape == (0, 2, 64)
    # a batch without positions in an empty pool
    table, lens = torch.zeros(3, 0, dtype=torch.int32, device=DEV), i32([0, 0, 0])
    out = gpu_kv_cache_attention(c, torch.ones(3, 2, 64, device=DEV), table, lens)
    assert (out == 0).all()
    assert status() == 0


@pytest.mark.gpu
def test_same_call_twice_is_equal_and_streams_agree():
    c = Case([3000, 70, 900], 2, 128, 4, 64, 32, torch.float32, seed=15)
    q = torch.randn(3, 8, 128, device=DEV)
    lens = i32(c.lens)
    want = gpu_kv_cache_attention(c.cache, q, c.table, lens)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(DEV) for _ in range(3)]
    outs = []
    for i in range(9):
        with torch.cuda.stream(streams[i % 3]):
            outs.append(gpu_kv_cache_attention(c.cache, q, c.table, lens))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, want)


@pytest.mark.gpu
def test_decode_steps_captured_in_graphs():
    """Two captured decode steps (append and attention) of different batches, replayed
    in turn and with other lengths, against eager calls."""
    H, D, page = 2, 64, 16
    cache = KvCache(40, page, H, D, 4, 32, DEV)
    eager = KvCache(40, page, H, D, 4, 32, DEV)
    tables = [i32(np.arange(20).reshape(2, 10)), i32(np.arange(20, 40).reshape(4, 5))]
    g = torch.Generator(DEV).manual_seed(3)
    graphs = []
    for table in tables:
        b = table.shape[0]
        lens = torch.ones(b, dtype=torch.int32, device=DEV)
        x = [torch.randn(b, H, D, generator=g, device=DEV) for _ in range(3)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            gpu_kv_cache_append(cache, x[0], x[1], table, lens)
            out = gpu_kv_cache_attention(cache, x[2], table, lens)
        graphs.append((graph, lens, x, out, table))
    for step in range(60):
        for graph, lens, x, out, table in graphs:
            lens.fill_(step + 1)
            for t in x:
                t.normal_(generator=g)
            graph.replay()
            gpu_kv_cache_append(eager, x[0], x[1], table, lens)
            want = gpu_kv_cache_attention(eager, x[2], table, lens)
            torch.cuda.synchronize()
            assert torch.equal(out, want), step
    assert torch.equal(cache.k_codes, eager.k_codes) and torch.equal(cache.v_params, eager.v_params)


@pytest.mark.gpu
def test_far_pages():
    """A pool whose later pages start beyond 2^31 bytes, and rows beyond 2^31 codes."""
    D, H, page = 256, 4, 256
    pages = (1 << 31) // (page * H * D) + 40
    cache = KvCache(pages, page, H, D, 8, 64, DEV)
    k = torch.randn(300, H, D, device=DEV)
    v = torch.randn(300, H, D, device=DEV)
    near, far = i32([[0, 1]]), i32([[pages - 1, pages - 2]])
    lens, cu = i32([300]), i32([0, 300])
    for table in (near, far):
        gpu_kv_cache_append(cache, k, v, table, lens, cu)
    a, b = (gpu_kv_cache_read(cache, t, lens, cu, tokens=300) for t in (near, far))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    q = torch.randn(1, 2 * H, D, device=DEV)
    assert torch.equal(gpu_kv_cache_attention(cache, q, near, lens), gpu_kv_cache_attention(cache, q, far, lens))
