"""The paged key-value cache (bmo_k_paged_*, bmo_jetson_b200/paged.py) against
plain implementations: the plan against an integer simulation, the append
against the oracle's RoPE and gguf-py's Q4_0 quantiser, the attention against
its formula in 64 bits.

Attention tolerance.  Both parts of a query element keep it to 2^-22 relative,
as do both parts of a weight; the sum over head_dim adds at most a few 2^-23
of sum |q k|.  With D = scale * max_j sum_d |q_d k_jd| a score is off by at most
d = 2^-20 D, a weight by a factor 1 + d + 2^-20, the quotient by twice that,
so an output by (2 d + 2^-19) max |v|: checked element by element, plus half
a unit of the output's type.  lse is off by at most d + 2^-19 + 2^-22 |lse|."""
import math

import numpy as np
import pytest
from gguf import GGMLQuantizationType, quants

from oracle import oracle as orc

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from bmo_jetson_b200 import engine, paged  # noqa: E402

DEV = torch.device("cuda:0")
HALF_UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)


def pack(x):
    """Q4_0 planes of float rows: nibble bytes [..., hd / 2], fp16 scales [..., hd / 32]."""
    hd = x.shape[-1]
    blocks = quants.quantize(np.ascontiguousarray(x.reshape(-1, 32)), GGMLQuantizationType.Q4_0)
    return (blocks[:, 2:].reshape(x.shape[:-1] + (hd // 2,)),
            blocks[:, :2].copy().view(np.float16).reshape(x.shape[:-1] + (hd // 32,)))


def unpack(nib, scale):
    b = nib.reshape(nib.shape[:-1] + (nib.shape[-1] // 16, 16)).astype(np.int64)
    n = np.concatenate([b & 15, b >> 4], -1) - 8
    return (n * scale.astype(np.float64)[..., None]).reshape(nib.shape[:-1] + (2 * nib.shape[-1],))


class Case:
    """A cache with random rows for requests of the given lengths; slots that no
    request holds, and pages before a window, hold NaN or are not in the table."""

    def __init__(self, lens, kv_heads, hd, ps, kv="f16", window=0, layers=1, seed=0, std=1.0, spare=3):
        rng = np.random.default_rng(seed)
        self.lens, self.kv_heads, self.hd, self.ps, self.kv, self.window = list(lens), kv_heads, hd, ps, kv, window
        first = [max(0, n - window) // ps if window else 0 for n in lens]
        last = [-(-n // ps) for n in lens]
        n_pages = sum(b - a for a, b in zip(first, last)) + spare
        order = rng.permutation(n_pages)
        table = np.full((len(lens), max(last + [1])), -1, np.int64)
        used = 0
        held = np.zeros((n_pages, ps), bool)
        for r, (a, b) in enumerate(zip(first, last)):
            table[r, a:b] = order[used:used + b - a]
            used += b - a
            for p in range(a * ps, lens[r]):
                held[table[r, p // ps], p % ps] = True
        self.table = table
        shape = (layers, n_pages, kv_heads, ps, hd)
        self.k, self.v = (rng.normal(0, std, shape).astype(np.float32) for _ in range(2))
        free = np.concatenate([order[used:], order[:used]])
        book = paged.PageBook(i32(table), i32(lens), i32(free), i32([0, n_pages - used, 0, 0]), page_size=ps, window=window)
        hole = ~np.broadcast_to(held[None, :, None, :, None], shape)
        if kv == "f16":
            self.k, self.v = self.k.astype(np.float16), self.v.astype(np.float16)
            self.k[hole] = self.v[hole] = np.nan
            self.cache = paged.PagedKV(book, torch.from_numpy(self.k).to(DEV), torch.from_numpy(self.v).to(DEV))
        else:
            (kn, ks), (vn, vs) = pack(self.k), pack(self.v)
            ks[hole[..., :hd // 32]] = vs[hole[..., :hd // 32]] = np.nan
            self.k, self.v = unpack(kn, ks), unpack(vn, vs)
            t = [torch.from_numpy(x).to(DEV) for x in (kn, vn, ks, vs)]
            self.cache = paged.PagedKV(book, t[0], t[1], k_scale=t[2], v_scale=t[3])

    def rows(self, x, layer, req, lo, hi):
        p = np.arange(lo, hi)
        page = self.table[req, p // self.ps]
        y = np.zeros((hi - lo, self.kv_heads, self.hd))
        y[page >= 0] = x[layer, page[page >= 0], :, (p % self.ps)[page >= 0]].astype(np.float64)
        return y, page >= 0

    def attention(self, q, layer=0, reqs=None, lens=None, scale=None):
        """(out, lse, bound on the score error) in 64 bits."""
        q = np.asarray(q, np.float64)
        n, heads, hd = q.shape
        scale = scale or 1.0 / math.sqrt(hd)
        out, lse, off = np.zeros(q.shape), np.full((n, heads), -np.inf), np.zeros((n, heads))
        for i in range(n):
            r = i if reqs is None else int(reqs[i])
            ln = self.lens[r] if lens is None else int(lens[i])
            lo = max(0, ln - self.window) if self.window else 0
            if ln <= lo:
                continue
            (k, there), (v, _) = self.rows(self.k, layer, r, lo, ln), self.rows(self.v, layer, r, lo, ln)
            k, v = k[there], v[there]
            if not len(k):
                continue
            for h in range(heads):
                g = h // (heads // self.kv_heads)
                s = scale * (k[:, g] @ q[i, h])
                off[i, h] = 2.0 ** -20 * scale * np.max(np.abs(k[:, g]) @ np.abs(q[i, h]))
                m = s.max()
                p = np.exp(s - m)
                lse[i, h] = m + np.log(p.sum())
                out[i, h] = (p / p.sum()) @ v[:, g]
        return out, lse, off


def close(got, lse, want, vmax, dtype=torch.float32):
    out, want_lse, off = want
    got, lse = got.double().cpu().numpy(), lse.double().cpu().numpy()
    tol = (2 * off[..., None] + 2.0 ** -19) * vmax + HALF_UNIT[dtype] * np.abs(out) + 2.0 ** -25
    assert np.isfinite(got).all()
    worst = np.max(np.abs(got - out) / tol, initial=0.0)
    assert worst <= 1.0, f"output off by {worst:.2f} of its bound"
    np.testing.assert_array_equal(np.isinf(lse), np.isinf(want_lse))
    fin = np.isfinite(want_lse)
    bound = off + 2.0 ** -19 + 2.0 ** -22 * np.abs(np.where(fin, want_lse, 0))
    assert (np.abs(lse[fin] - want_lse[fin]) <= bound[fin]).all()


def attend(c, heads, dtype=torch.float32, seed=1, layer=0, qstd=1.0, reqs=None, lens=None, scale=0.0):
    n = len(c.lens) if reqs is None else len(reqs)
    q = (torch.from_numpy(np.random.default_rng(seed).normal(0, qstd, (n, heads, c.hd)).astype(np.float32))
         .to(dtype).to(DEV))
    out, lse = torch.full_like(q, float("nan")), torch.full((n, heads), float("nan"), device=DEV)
    status = i32([0])
    c.cache.attention(layer, q, out, lse=lse, scale=scale, status=status, rows=None if reqs is None else i32(reqs),
                      row_lens=None if lens is None else i32(lens))
    return q, out, lse, int(status.item())


def vmax(c):
    return float(np.nanmax(np.abs(c.v.astype(np.float64)), initial=0.0))


def check(c, heads, dtype=torch.float32, **kw):
    q, out, lse, status = attend(c, heads, dtype, **kw)
    kw2 = {n: kw[n] for n in ("reqs", "lens", "layer") if n in kw}
    if kw.get("scale"):
        kw2["scale"] = kw["scale"]
    close(out, lse, c.attention(q.double().cpu().numpy(), **kw2), vmax(c), dtype)
    assert status == 0


# ---------------------------------------------------------------- attention

RAGGED = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 100, 127, 129, 255, 300]


@pytest.mark.parametrize("kv", ["f16", "q4_0"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("ps", [1, 3, 8, 16, 24, 64, 500])
def test_attention_page_sizes(kv, hd, ps):
    check(Case(RAGGED, 2, hd, ps, kv, seed=ps), 2)


@pytest.mark.parametrize("kv", ["f16", "q4_0"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("group,kv_heads", [(1, 3), (2, 2), (3, 2), (4, 1), (5, 2), (8, 2), (12, 1), (32, 1)])
def test_attention_shared_key_heads(kv, hd, group, kv_heads):
    check(Case([0, 1, 40, 333], kv_heads, hd, 16, kv, seed=group), group * kv_heads)


@pytest.mark.parametrize("kv", ["f16", "q4_0"])
@pytest.mark.parametrize("window", [1, 7, 16, 50, 64, 299, 1000])
def test_attention_window(kv, window):
    """Pages before the window are not in the table; slots past the length hold NaN."""
    check(Case(RAGGED, 2, 128, 24, kv, window=window, seed=window), 4)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kv", ["f16", "q4_0"])
def test_attention_types(kv, dtype):
    check(Case([5, 77, 0, 400], 2, 128, 16, kv), 8, dtype)
    check(Case([5, 77, 0, 400], 2, 64, 16, kv), 2, dtype, scale=0.3)


@pytest.mark.parametrize("kv", ["f16", "q4_0"])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 1), (32, 32)])
def test_attention_split_over_many_ctas(kv, heads, kv_heads):
    """Rows long enough to be cut across CTAs, beside short and empty ones; two layers."""
    c = Case([0, 9000, 1, 2500, 0], kv_heads, 128, 16, kv, layers=2, seed=heads)
    check(c, heads, layer=1)
    check(c, heads, layer=0, dtype=torch.bfloat16)


def test_attention_many_rows():
    rng = np.random.default_rng(4)
    check(Case(rng.integers(0, 40, 700), 1, 64, 16, "f16"), 2)


@pytest.mark.parametrize("kv", ["f16", "q4_0"])
@pytest.mark.parametrize("rows,kv_heads,longest", [(1, 1, 3000), (1, 32, 600), (13, 4, 90), (27, 4, 700), (55, 4, 300),
                                                   (75, 2, 40), (200, 2, 70), (40, 16, 130)])
def test_attention_shares_of_the_gpu(kv, rows, kv_heads, longest):
    """Numbers of heads and lengths at which a head is given a cluster of 8, 4 or
    2 CTAs, a CTA, or a part of the line of tiles."""
    lens = np.random.default_rng(rows).integers(0, longest + 1, rows)
    lens[0] = longest
    check(Case(lens, kv_heads, 64, 16, kv, seed=rows), kv_heads)
    check(Case(lens, kv_heads, 128, 20, kv, seed=rows + 1, window=longest // 2 + 1), kv_heads)


@pytest.mark.parametrize("kv", ["f16", "q4_0"])
def test_attention_several_tokens_of_a_request(kv):
    c = Case([50, 7, 130], 2, 128, 16, kv, window=64)
    check(c, 2, reqs=[2, 2, 2, 0, 1, 0, 2], lens=[128, 129, 130, 50, 0, 49, 128])


@pytest.mark.parametrize("kv", ["f16", "q4_0"])
@pytest.mark.parametrize("qstd,std", [(1e6, 1e-3), (1e-6, 1.0), (30.0, 3.0), (1e-30, 1.0), (1.0, 1e-4), (0.1, 3000.0)])
def test_attention_magnitudes(kv, qstd, std):
    """Queries beyond fp16's range, flat and one-hot weights, small and large values."""
    check(Case([1, 64, 700], 2, 128, 16, kv, std=std, seed=3), 2, qstd=qstd)


def test_attention_growing_scores():
    """Each position outscores the ones before it by more than the weights' range, and the reverse."""
    for sign in (1.0, -1.0):
        c = Case([600], 1, 64, 16)
        k = c.cache.k
        ramp = torch.zeros(600, dtype=torch.float64)
        for p in range(600):
            ramp[p] = sign * 0.1 * p
        for p in range(600):
            k[0, int(c.table[0, p // 16]), 0, p % 16] = ramp[p].half()
        c.k = k.cpu().numpy()
        q = torch.full((1, 2, 64), 3.0, device=DEV)
        out, lse = torch.empty_like(q), torch.empty((1, 2), device=DEV)
        c.cache.attention(0, q, out, lse=lse)
        close(out, lse, c.attention(q.cpu().numpy()), vmax(c))


def test_attention_nan_stays_in_its_row():
    c = Case([40, 40], 2, 128, 16)
    q = torch.randn(2, 2, 128, device=DEV)
    want = torch.empty_like(q)
    c.cache.attention(0, q, want)
    q[0, 1, 5] = float("nan")
    out = torch.empty_like(q)
    c.cache.attention(0, q, out)
    assert torch.isnan(out[0, 1]).all()
    assert torch.equal(out[0, 0], want[0, 0]) and torch.equal(out[1], want[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("off,extra", [(0, 0), (1, 3), (4, 4), (2, 1)])
def test_attention_strides(dtype, off, extra):
    """Queries and outputs as parts of wider, unaligned rows; what surrounds them stays."""
    c = Case([3, 70, 200], 2, 128, 16)
    n, h, hd = 3, 4, 128
    wide = torch.randn(n, h * hd + off + extra, device=DEV).to(dtype)
    q = wide[:, off:off + h * hd].unflatten(1, (h, hd))
    wide_out = torch.full_like(wide, 7.0)
    out = wide_out[:, off:off + h * hd].unflatten(1, (h, hd))
    lse = torch.empty(n, h, device=DEV)
    c.cache.attention(0, q, out, lse=lse)
    close(out, lse, c.attention(q.double().cpu().numpy()), vmax(c), dtype)
    assert (wide_out[:, :off] == 7).all() and (wide_out[:, off + h * hd:] == 7).all()


@pytest.mark.parametrize("kv", ["f16", "q4_0"])
def test_attention_bad_indices_are_left_out(kv):
    """Pages outside the cache, requests and lengths out of range: reported, nothing read."""
    c = Case([64, 64, 64], 1, 64, 16, kv)
    table = c.cache.book.table
    table[0, 1] = 10 ** 6
    table[0, 2] = -1
    table[1] = -5
    c.table[0, 1:3] = -1
    c.table[1] = -1
    q, out, lse, status = attend(c, 2)
    assert status == paged.BAD_INDEX
    close(out, lse, c.attention(q.cpu().numpy()), vmax(c))
    assert (out[1] == 0).all() and torch.isinf(lse[1]).all()
    q, out, lse, status = attend(c, 2, reqs=[2, 3, -1, 2], lens=[64, 5, 5, -7])
    assert status == paged.BAD_INDEX
    assert (out[1:] == 0).all() and (out[0] != 0).any()
    q, out, lse, status = attend(c, 2, reqs=[2], lens=[10 ** 6])  # clamped to the table's row
    assert status == paged.BAD_INDEX
    close(out, lse, c.attention(q.cpu().numpy(), reqs=[2], lens=[64]), vmax(c))


def test_attention_repeats_and_streams():
    """The same bits from call to call, on another stream, from a graph, and with scratch that other shapes used."""
    c = Case([0, 1, 5000, 77], 4, 128, 16)
    q = torch.randn(4, 16, 128, device=DEV)
    a, b = torch.empty_like(q), torch.empty_like(q)
    c.cache.attention(0, q, a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.cache.attention(0, q[:2], b[:2])
        c.cache.attention(0, q, b)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, b)
    b.zero_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.cache.attention(0, q, b)
    for _ in range(3):
        b.zero_()
        g.replay()
        assert torch.equal(a, b)


def test_attention_cache_beyond_32_bits():
    """Pages past 2^32 elements of a layer."""
    ps, hd, n_pages = 64, 128, (1 << 32) // (64 * 128) + 40
    k = torch.empty((1, n_pages, 1, ps, hd), dtype=torch.float16, device=DEV)
    v = torch.empty_like(k)
    n = 2000
    pages = torch.arange(n_pages - 1, n_pages - 33, -1)
    pages[3] = 0
    k[0, pages], v[0, pages] = (torch.randn((32, 1, ps, hd), device=DEV).half() for _ in range(2))
    book = paged.PageBook(pages[None].int().to(DEV), i32([n]), i32(np.zeros(n_pages)), i32([0, 0, 0, 0]), page_size=ps)
    cache = paged.PagedKV(book, k, v)
    q = torch.randn(1, 1, hd, device=DEV)
    out = torch.empty_like(q)
    cache.attention(0, q, out)
    kk, vv = (x[0, pages].reshape(-1, hd)[:n].double() for x in (k, v))
    s = (kk @ q[0, 0].double()) / math.sqrt(hd)
    want = torch.softmax(s, 0) @ vv
    assert (out[0, 0].double() - want).abs().max() < 2.0 ** -15
    # the append and the read reach them too
    slot = (pages[:5].int() * ps + 7).to(DEV)
    kn, vn = (torch.randn(5, 1, hd, device=DEV) for _ in range(2))
    cache.append(0, kn, vn, slot)
    ko, vo = torch.empty_like(kn), torch.empty_like(vn)
    cache.read(0, slot, ko, vo)
    assert torch.equal(ko, kn.half().float()) and torch.equal(vo, vn.half().float())
    assert torch.equal(k[0, pages[4], 0, 7], kn[4, 0].half())


# ---------------------------------------------------------------- append, read

def rope(x, pos, theta):
    """The oracle's interleaved RoPE of rows [n, heads, hd]."""
    n, heads, hd = x.shape
    return np.stack([np.asarray(orc.rope(np.ascontiguousarray(x[i]).reshape(-1), heads, hd, int(p), theta)).reshape(heads, hd)
                     for i, p in enumerate(pos)])


@pytest.mark.parametrize("kv", ["f16", "q4_0"])
@pytest.mark.parametrize("hd,heads,kv_heads,ps", [(128, 32, 32, 16), (64, 8, 2, 24), (128, 7, 1, 1), (64, 3, 3, 100)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_append_and_read(kv, hd, heads, kv_heads, ps, dtype):
    n, pages = 37, 60
    rng = np.random.default_rng(hd + heads)
    book = paged.PageBook.empty(2, pages, ps, 8)
    cache = paged.PagedKV.empty(book, 2, kv_heads, hd, engine.KV_F16 if kv == "f16" else engine.KV_Q4_0)
    qkv = torch.from_numpy(rng.normal(0, 1, (n, (heads + 2 * kv_heads) * hd)).astype(np.float32)).to(dtype).to(DEV)
    qkv[3, heads * hd:(heads + kv_heads) * hd] = 0
    q = qkv[:, :heads * hd].unflatten(1, (heads, hd))
    k = qkv[:, heads * hd:(heads + kv_heads) * hd].unflatten(1, (kv_heads, hd))
    v = qkv[:, (heads + kv_heads) * hd:].unflatten(1, (kv_heads, hd))
    pos = rng.integers(0, 5000, n)
    slots = rng.permutation(pages * ps)[:n]
    slots[5] = -1
    q_out = torch.empty((n, heads, hd), dtype=dtype, device=DEV)
    cache.append(1, k, v, i32(slots), pos=i32(pos), q=q, q_out=q_out, theta=10000.0)
    k32, v32, q32 = (x.float().cpu().numpy() for x in (k, v, q))
    kr, qr = rope(k32, pos, 10000.0), rope(q32, pos, 10000.0)
    assert torch.equal(q_out, torch.from_numpy(qr).to(dtype).to(DEV))
    out = [torch.empty((n, kv_heads, hd), dtype=torch.float32, device=DEV) for _ in range(2)]
    cache.read(1, i32(slots), *out)
    for got, want in zip(out, (kr, v32)):
        if kv == "f16":
            w = want.astype(np.float16).astype(np.float32)
        else:
            w = unpack(*pack(want)).astype(np.float32)
        w[5] = 0
        np.testing.assert_array_equal(got.cpu().numpy(), w)
    # nothing else was written, in this layer or the other
    held = torch.zeros(pages * ps, dtype=torch.bool, device=DEV)
    held[i32(slots[slots >= 0]).long()] = True
    for t in (cache.k, cache.v) + ((cache.k_scale, cache.v_scale) if kv != "f16" else ()):
        assert not t[0].any()
        by_slot = t[1].transpose(1, 2).reshape(pages * ps, -1)
        assert not by_slot[~held].any()
    # the stored bytes are ggml's blocks
    if kv != "f16":
        nib, sc = pack(v32)
        for i in (0, n - 1):
            page, at = divmod(int(slots[i]), ps)
            np.testing.assert_array_equal(cache.v[1, page, :, at].cpu().numpy(), nib[i])
            np.testing.assert_array_equal(cache.v_scale[1, page, :, at].cpu().numpy().view(np.uint16), sc[i].view(np.uint16))
    half = [torch.empty((n, kv_heads, hd), dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    cache.read(1, i32(slots), *half)
    assert torch.equal(half[0], out[0].bfloat16()) and torch.equal(half[1], out[1].bfloat16())


def test_append_in_place_without_rope_and_unaligned():
    book = paged.PageBook.empty(1, 4, 16, 4)
    cache = paged.PagedKV.empty(book, 1, 2, 64)
    wide = torch.randn(3, 3 * 128 + 5, device=DEV)
    q, k, v = (wide[:, 1 + 128 * i:129 + 128 * i].unflatten(1, (2, 64)) for i in range(3))
    q0, k0 = q.cpu().numpy().copy(), k.cpu().numpy().copy()
    cache.append(0, k, v, i32([0, 1, 2]))
    ko, vo = (torch.empty((3, 2, 64), dtype=torch.float16, device=DEV) for _ in range(2))
    cache.read(0, i32([0, 1, 2]), ko, vo)
    assert torch.equal(ko, k.half()) and torch.equal(vo, v.half())
    cache.append(0, k, v, i32([3, 4, 63]), pos=i32([0, 1, 2999]), q=q, q_out=q, theta=500.0)
    np.testing.assert_array_equal(q.cpu().numpy(), rope(q0, [0, 1, 2999], 500.0))
    cache.read(0, i32([3, 4, 63]), ko, vo)
    np.testing.assert_array_equal(ko.cpu().numpy(), rope(k0, [0, 1, 2999], 500.0).astype(np.float16))


@pytest.mark.parametrize("kv_type", [0, 1])
def test_append_and_read_bad_slots(kv_type):
    book = paged.PageBook.empty(1, 3, 16, 4)
    cache = paged.PagedKV.empty(book, 1, 1, 64, kv_type)
    k = torch.randn(3, 1, 64, device=DEV)
    status = i32([0])
    cache.append(0, k, k, i32([-1, 5, -1]), status=status)
    assert status.item() == 0
    cache.append(0, k, k, i32([48, 6, -2]), status=status)
    assert status.item() == paged.BAD_INDEX
    status.zero_()
    ko, vo = torch.full_like(k, 9.0), torch.full_like(k, 9.0)
    cache.read(0, i32([48, 6, -1]), ko, vo, status=status)
    assert status.item() == paged.BAD_INDEX
    assert not ko[0].any() and not ko[2].any() and not vo[0].any() and ko[1].any()
    cache.append(0, k[:0], k[:0], i32([]))
    cache.read(0, i32([]), ko[:0], vo[:0])


def test_pages_are_rings():
    """A page of one layer is a ring of page_size slots: bmo_k_decode_attention
    over it gives the paged attention's result up to fp32 rounding."""
    c = Case([32], 4, 128, 32)
    q = torch.randn(1, 4, 128, device=DEV)
    out = torch.empty_like(q)
    c.cache.attention(0, q, out)
    page = int(c.table[0, 0])
    kc, vc = c.cache.k[0, page].clone(), c.cache.v[0, page].clone()
    k, v = kc[:, 31].float().contiguous(), vc[:, 31].float().contiguous()
    ring, pos = torch.empty_like(out), i32([31])
    rc = engine.lib().bmo_k_decode_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), kc.data_ptr(), vc.data_ptr(), None,
                                             None, ring.data_ptr(), 128, 4, 4, 32, pos.data_ptr(), 0, 0,
                                             torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    assert (out - ring).abs().max() < 2.0 ** -15


# ---------------------------------------------------------------- plan

class Book:
    """The plan's rules on Python integers."""

    def __init__(self, n_req, n_pages, ps, blocks, window):
        self.ps, self.blocks, self.window, self.n_pages = ps, blocks, window, n_pages
        self.lens = [0] * n_req
        self.table = {}
        self.free = list(range(n_pages))

    def first(self, n):
        return max(0, n - self.window) // self.ps if self.window else 0

    def step(self, new, max_tokens):
        ps = self.ps
        after = [0 if n < 0 else a + n for a, n in zip(self.lens, new)]
        take = [0 if n < 0 else -(-(a + n) // ps) + (-a // ps) for a, n in zip(self.lens, new)]
        bad = 0
        if any(a > self.blocks * ps for a in after):
            bad |= paged.TABLE_FULL
        elif sum(take) > len(self.free):
            bad |= paged.NO_PAGES
        if not bad & paged.TABLE_FULL and sum(max(0, n) for n in new) > max_tokens:
            bad |= paged.NO_ROOM
        if bad:
            return bad, [], [0] * (len(new) + 1)
        for r, t in enumerate(take):
            have = -(-self.lens[r] // ps)
            for b in range(have, have + t):
                self.table[r, b] = self.free.pop(0)
        tokens, offsets = [], [0]
        for r, n in enumerate(new):
            for p in range(self.lens[r], self.lens[r] + max(0, n)):
                tokens.append((self.table[r, p // ps] * ps + p % ps, p, r))
            offsets.append(len(tokens))
        for r, n in enumerate(new):
            stop = -(-self.lens[r] // ps) if n < 0 else self.first(after[r])
            self.free += [self.table[r, b] for b in range(self.first(self.lens[r]), stop)]
        self.lens = after
        return 0, tokens, offsets


@pytest.mark.parametrize("n_req,ps,window,most", [(1, 16, 0, 3), (5, 16, 40, 60), (64, 1, 0, 2), (64, 24, 500, 90),
                                                  (1500, 8, 20, 4), (2100, 16, 0, 1), (7, 16, 100, 2500)])
@pytest.mark.parametrize("in_place", [True, False])
def test_plan_steps(n_req, ps, window, most, in_place):
    rng = np.random.default_rng(n_req + ps)
    blocks, max_tokens = 400, max(2 * n_req, n_req * most)
    n_pages = n_req * (window // ps + 4 + 2 * most // ps) + 300
    sim = Book(n_req, n_pages, ps, blocks, window)
    book = paged.PageBook.empty(n_req, n_pages, ps, blocks, window=window)
    slot, pos, req = (torch.empty(max_tokens, dtype=torch.int32, device=DEV) for _ in range(3))
    offsets = torch.empty(n_req + 1, dtype=torch.int32, device=DEV)
    served = refused = 0
    for step in range(12):
        new = rng.integers(0, most + 1, n_req)
        new[rng.random(n_req) < 0.15] = -1
        lens_out, state_out = (None, None) if in_place else (torch.empty_like(book.lens), torch.empty_like(book.state))
        book.plan(i32(new), slot, pos, req, offsets, lens_out=lens_out, state_out=state_out)
        if not in_place:
            book.lens.copy_(lens_out)
            book.state.copy_(state_out)
        before = list(sim.free)
        bad, tokens, offs = sim.step([int(x) for x in new], max_tokens)
        served, refused = served + (not bad), refused + bool(bad)
        head, count, status, total = book.state.tolist()
        assert (status, total, count) == (bad, len(tokens), len(sim.free)), step
        ring = book.free.tolist()
        assert [ring[(head + i) % n_pages] for i in range(count)] == sim.free
        if bad:
            assert sim.free == before
        assert book.lens.tolist() == sim.lens and offsets.tolist() == offs
        want = np.full((3, max_tokens), -1)
        if tokens:
            want[:, :len(tokens)] = np.array(tokens).T
        np.testing.assert_array_equal(torch.stack([slot, pos, req]).cpu().numpy(), want)
        t = book.table.cpu().numpy()
        for r in range(n_req):
            for b in range(sim.first(sim.lens[r]), -(-sim.lens[r] // ps)):
                assert t[r, b] == sim.table[r, b]
    assert served >= 3


def test_plan_refusals():
    ps, n_pages = 16, 6
    slot, pos, req = (torch.empty(50, dtype=torch.int32, device=DEV) for _ in range(3))
    offsets = torch.empty(3, dtype=torch.int32, device=DEV)
    book = paged.PageBook.empty(2, n_pages, ps, 3)

    def plan(new):
        book.plan(i32(new), slot, pos, req, offsets)
        return book.state[2].item(), book.state[3].item()

    assert plan([20, 17]) == (0, 37)
    keep = [x.clone() for x in (book.table, book.lens, book.free)]
    for new, bits in (([29, 0], paged.TABLE_FULL), ([2 ** 31 - 1, 0], paged.TABLE_FULL), ([28, 23], paged.NO_ROOM)):
        got, total = plan(new)
        assert got == bits and total == 0, (new, got)
        assert all(torch.equal(a, b) for a, b in zip(keep, (book.table, book.lens, book.free)))
        assert (slot == -1).all() and not offsets.any()
    assert plan([28, 16])[0] == 0 and book.state[1].item() == 0
    assert plan([-1, -1]) == (0, 0)
    # pages given back in a step are free from the next one on
    assert book.state[1].item() == n_pages
    assert plan([48, 2]) == (0, 50)
    book2 = paged.PageBook.empty(2, 3, ps, 3)
    book2.plan(i32([40, 0]), slot, pos, req, offsets)
    book2.plan(i32([-1, 1]), slot, pos, req, offsets)
    assert book2.state.tolist()[2:] == [paged.NO_PAGES, 0] and book2.lens.tolist() == [40, 0]
    # inconsistent input: reported, nothing done
    book2.lens[0] = -3
    book2.plan(i32([0, 0]), slot, pos, req, offsets)
    assert book2.state[2].item() == paged.BAD_INDEX and book2.lens.tolist() == [-3, 0]
    book2.lens[0] = 40
    book2.state[1] = 77
    book2.plan(i32([0, 0]), slot, pos, req, offsets)
    assert book2.state[2].item() == paged.BAD_INDEX


def test_plan_without_positions():
    """No room asked for, nothing appended; ended requests that hold nothing."""
    book = paged.PageBook.empty(3, 2, 16, 1)
    none = i32([])
    offsets = torch.empty(4, dtype=torch.int32, device=DEV)
    book.plan(i32([0, -1, 0]), none, none, none, offsets)
    assert book.state.tolist() == [0, 2, 0, 0] and not offsets.any()


# ---------------------------------------------------------------- refusals of the binding

def test_binding_refusals():
    c = Case([5, 6], 2, 64, 16)
    q = torch.randn(2, 4, 64, device=DEV)
    out = torch.empty_like(q)
    for bad in (lambda: c.cache.attention(0, q.double(), out), lambda: c.cache.attention(0, q, out.half()),
                lambda: c.cache.attention(0, q[:, :, :32], out[:, :, :32]),
                lambda: c.cache.attention(0, q.transpose(1, 2).contiguous().transpose(1, 2), out),
                lambda: c.cache.attention(0, q, out, lse=torch.empty(2, 4, device=DEV).half()),
                lambda: c.cache.attention(0, q, out, rows=torch.zeros(2, dtype=torch.int64, device=DEV)),
                lambda: c.cache.attention(0, q[:, :3], out[:, :3]),  # 3 query heads of 2 key heads
                lambda: c.cache.append(0, q[:, :2], q[:, :1], i32([0, 1])),
                lambda: c.cache.read(0, i32([0]), q, q),
                lambda: paged.PagedKV(c.cache.book, c.cache.k[:, :1], c.cache.v[:, :1]),
                lambda: paged.PagedKV(c.cache.book, c.cache.k, c.cache.v.float())):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: c.cache.attention(1, q, out), lambda: c.cache.attention(-1, q, out),
                lambda: c.cache.attention(0, q.repeat(2, 1, 1), out.repeat(2, 1, 1)),  # more rows than requests
                lambda: c.cache.attention(0, q, out, scale=float("nan")),
                lambda: c.cache.append(0, q[:, :2], q[:, :2], i32([0, 1]), theta=10000.0),  # no positions
                lambda: c.cache.append(0, q[:, :2], q[:, :2], i32([0, 1]), theta=-1.0),
                lambda: c.cache.append(7, q[:, :2], q[:, :2], i32([0, 1]))):
        with pytest.raises(RuntimeError):
            bad()
