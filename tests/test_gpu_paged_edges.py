"""The paged cache (bmo_k_paged_*, bmo_jetson_b200/paged.py) where its calls meet
what they rarely meet: a plan made again, lengths beyond a request's, infinite
rows, weights and scales of very different sizes, refused frames."""
import copy
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from bmo_jetson_b200 import engine, paged  # noqa: E402
from tests import test_gpu_paged as base  # noqa: E402

DEV, i32 = base.DEV, base.i32


# ---------------------------------------------------------------- a plan made again

class Steps:
    """A book on the GPU and the plan's rules on integers, step by step."""

    def __init__(self, n_req, n_pages, ps, blocks, window, max_tokens):
        self.sim = base.Book(n_req, n_pages, ps, blocks, window)
        self.book = paged.PageBook.empty(n_req, n_pages, ps, blocks, window=window)
        self.max_tokens = max_tokens
        self.lists = [torch.empty(max_tokens, dtype=torch.int32, device=DEV) for _ in range(3)]
        self.offsets = torch.empty(n_req + 1, dtype=torch.int32, device=DEV)
        self.lens, self.state = torch.empty_like(self.book.lens), torch.empty_like(self.book.state)

    def plan(self, new):
        """Plans into separate lengths and state; everything that the call has written."""
        b = self.book
        b.plan(i32(new), *self.lists, self.offsets, lens_out=self.lens, state_out=self.state)
        return [t.clone() for t in (b.table, b.free, self.lens, self.state, self.offsets, *self.lists)]

    def adopt(self):
        self.book.lens.copy_(self.lens)
        self.book.state.copy_(self.state)

    def check(self, new, got, sim=None):
        """What plan() gave against the rules, applied to a copy of the books' common past."""
        sim = sim or copy.deepcopy(self.sim)
        bad, tokens, offs = sim.step([int(x) for x in new], self.max_tokens)
        table, free, lens, state, offsets, *lists = got
        head, count, status, total = state.tolist()
        assert (status, total, count) == (bad, len(tokens), len(sim.free))
        n_pages, ring, t = sim.n_pages, free.tolist(), table.cpu().numpy()
        assert [ring[(head + i) % n_pages] for i in range(count)] == sim.free
        assert lens.tolist() == sim.lens and offsets.tolist() == offs
        want = np.full((3, self.max_tokens), -1)
        if tokens:
            want[:, :len(tokens)] = np.array(tokens).T
        np.testing.assert_array_equal(torch.stack(lists).cpu().numpy(), want)
        for r, n in enumerate(sim.lens):
            for b in range(sim.first(n), -(-n // sim.ps)):
                assert t[r, b] == sim.table[r, b]
        return sim


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


# requests, pages, page size, window, the two steps, room of the lists; pages
# are given back past the ring's end, over the entries that the step takes
REPEATED = {
    "a position or two each": (3, 9, 1, 1, [2, 2, 2], [2, 0, 1], 8),
    "histories": (5, 100, 4, 6, [50, 0, 33, 0, 90], [7, 99, 0, 1, 60], 300),
    "histories, long lists": (5, 100, 4, 6, [50, 0, 33, 0, 90], [7, 99, 0, 1, 60], 9000),
    "many requests": (1500, 9000, 2, 3, [9] * 1500, [3, 0, 11] * 500, 14000),
}


@pytest.mark.parametrize("case", REPEATED)
@pytest.mark.parametrize("before", [0, 3])
def test_plan_can_be_made_again(case, before):
    """From the same lengths and state a plan gives the same, and one that was
    dropped leaves no trace in the next, whatever that one appends."""
    n_req, n_pages, ps, window, first, second, most = REPEATED[case]
    s = Steps(n_req, n_pages, ps, 120, window, most)
    for k in range(before):  # the ring's first free entry moves on
        new = [(r + k) % 3 for r in range(n_req)]
        s.sim = s.check(new, s.plan(new))
        s.adopt()
    got = s.plan(first)
    s.check(first, got)
    assert int(s.book.state[1]) + given_back(s.sim, first) > n_pages  # it does wrap
    assert same(s.plan(first), got)
    got = s.plan(second)
    s.check(second, got)
    assert same(s.plan(second), got)
    too_much = [10 ** 6] + [0] * (n_req - 1)
    refused = s.plan(too_much)
    assert refused[3][2].item() == paged.TABLE_FULL and same(refused[:2], got[:2])
    assert same(s.plan(second), got)
    again = s.plan(first)
    s.sim = s.check(first, again)
    s.adopt()
    for k in range(3):  # and the book goes on from the one that was kept
        new = [-1 if r == k else (r + k) % 2 for r in range(n_req)]
        s.sim = s.check(new, s.plan(new))
        s.adopt()


def given_back(sim, new):
    sim = copy.deepcopy(sim)
    count = len(sim.free)
    take = sum(-(-(a + n) // sim.ps) + (-a // sim.ps) for a, n in zip(sim.lens, new))
    assert sim.step(list(new), 1 << 30)[0] == 0
    return len(sim.free) - (count - take)


def test_plan_after_the_ring_was_rewritten():
    """A ring that the caller has filled anew is taken as it is."""
    n_req, n_pages, ps, window, first, second, most = REPEATED["histories"]
    s = Steps(n_req, n_pages, ps, 120, window, most)
    s.plan(first)
    order = list(range(n_pages - 1, -1, -1))
    s.book.free.copy_(i32(order))
    s.sim.free = order
    s.check(second, s.plan(second))


@pytest.mark.parametrize("n_req,ps,window,most", [(1500, 8, 20, 12), (2100, 16, 0, 9)])
def test_plan_of_many_requests_with_long_lists(n_req, ps, window, most):
    rng = np.random.default_rng(n_req)
    s = Steps(n_req, n_req * (window // ps + 8) + 400, ps, 40, window, n_req * most)
    for _ in range(6):
        new = rng.integers(0, most + 1, n_req)
        new[rng.random(n_req) < 0.15] = -1
        s.sim = s.check(new, s.plan(new))
        s.adopt()


# ---------------------------------------------------------------- lengths beyond a request's

@pytest.mark.parametrize("kv", ["f16", "q4_0"])
@pytest.mark.parametrize("window", [0, 8])
def test_attention_row_len_above_the_requests(kv, window):
    """A row length that the table's row has room for and the request does not hold:
    reported, and the row attends to what the request holds, not to a page of another's."""
    c = base.Case([20, 64], 1, 64, 16, kv, window=window)
    c.cache.book.table[0, 2] = int(c.table[1, 3])  # stale: another request has the page now
    q, out, lse, status = base.attend(c, 2, reqs=[0, 1, 0], lens=[40, 64, 20])
    assert status == paged.BAD_INDEX
    base.close(out, lse, c.attention(q.cpu().numpy(), reqs=[0, 1, 0], lens=[20, 64, 20]), base.vmax(c))
    q, out, lse, status = base.attend(c, 2, reqs=[0, 1, 0], lens=[20, 64, 19])
    assert status == 0


# ---------------------------------------------------------------- infinite rows

class Rows:
    """One request on pages of 16 in order, its rows as given: k, v [positions, kv_heads, hd].
    Q4_0: packed, then `edit(codes and scales of k, of v)` may change them."""

    def __init__(self, k, v, kv="f16", edit=None, more=(), window=0):
        n, kv_heads, hd = k.shape
        pages = -(-n // 16)
        lens = [n] + list(more)

        def paged_rows(x):  # [1, page, head, slot, row]
            y = np.zeros((pages * 16,) + x.shape[1:], x.dtype)
            y[:n] = x
            return np.ascontiguousarray(y.reshape(pages, 16, *x.shape[1:]).transpose(0, 2, 1, 3)[None])

        table = np.tile(np.arange(pages), (len(lens), 1))
        book = paged.PageBook(i32(table), i32(lens), i32(np.arange(pages)), i32([0, 0, 0, 0]), page_size=16, window=window)
        self.kv_heads, self.hd, self.window, self.lens = kv_heads, hd, window, lens
        if kv == "f16":
            k, v = k.astype(np.float16), v.astype(np.float16)
            self.k, self.v = k.astype(np.float64), v.astype(np.float64)
            self.k_scale = np.ones(k.shape[:2] + (hd // 32,))
            self.cache = paged.PagedKV(book, *(torch.from_numpy(paged_rows(x)).to(DEV) for x in (k, v)))
        else:
            (kn, ks), (vn, vs) = base.pack(k.astype(np.float32)), base.pack(v.astype(np.float32))
            if edit:
                edit((kn, ks), (vn, vs))
            with np.errstate(invalid="ignore"):
                self.k, self.v = base.unpack(kn, np.ones_like(ks)), base.unpack(vn, vs)
            self.k_scale = ks.astype(np.float64)
            t = [torch.from_numpy(paged_rows(x)).to(DEV) for x in (kn, vn, ks, vs)]
            self.cache = paged.PagedKV(book, t[0], t[1], k_scale=t[2], v_scale=t[3])

    def run(self, q, rows=None):
        out = torch.full_like(q, 7.0)
        lse = torch.full(q.shape[:2], 7.0, device=DEV)
        self.cache.attention(0, q, out, lse=lse, rows=rows)
        return out.double().cpu().numpy(), lse.double().cpu().numpy()

    def want(self, q, n=None):
        """(out, lse, largest score error) of one row in 64 bits; products of zero and infinity are NaN.
        A block of 32 of a key counts as its scale times the sum of its codes' products."""
        q = np.asarray(q.double().cpu().numpy())
        n = self.lens[0] if n is None else n
        lo = max(0, n - self.window) if self.window else 0
        k, ks, v = self.k[lo:n], self.k_scale[lo:n], self.v[lo:n]
        heads = q.shape[0]
        out, lse, off = np.zeros((heads, self.hd)), np.zeros(heads), np.zeros(heads)
        with np.errstate(invalid="ignore", over="ignore"):
            for h in range(heads):
                g = h // (heads // self.kv_heads)
                s = ((k[:, g] * q[h]).reshape(len(k), -1, 32).sum(-1) * ks[:, g]).sum(-1) / math.sqrt(self.hd)
                a = (np.abs(k[:, g] * q[h]).reshape(len(k), -1, 32).sum(-1) * np.abs(ks[:, g])).sum(-1)
                off[h] = 2.0 ** -20 * np.max(a[np.isfinite(a)], initial=0.0) / math.sqrt(self.hd)
                p = np.exp(s - s.max())
                lse[h] = s.max() + np.log(p.sum())
                out[h] = (p[:, None] * v[:, g])[p != 0].sum(0) / p.sum()
        return out, lse, off


def check_edges(got, want, vmax, dtype=torch.float32):
    (out, lse), (want_out, want_lse, off) = got, want
    np.testing.assert_array_equal(np.isnan(out), np.isnan(want_out))
    there = ~np.isnan(want_out)
    np.testing.assert_array_equal(np.isinf(out[there]), np.isinf(want_out[there]))
    inf = np.isinf(want_out)
    np.testing.assert_array_equal(out[inf], want_out[inf])
    fin = np.isfinite(want_out)
    tol = (2 * off[:, None] + 2.0 ** -19) * vmax + base.HALF_UNIT[dtype] * np.abs(np.where(fin, want_out, 0)) + 2.0 ** -25
    assert (np.abs(out[fin] - want_out[fin]) <= tol[fin]).all()
    ok = np.isfinite(want_lse)
    assert not np.isfinite(lse[~ok]).any()
    bound = off + 2.0 ** -19 + 2.0 ** -22 * np.abs(np.where(ok, want_lse, 0))
    assert (np.abs(lse[ok] - want_lse[ok]) <= bound[ok]).all()


def finite_max(x):
    return float(np.max(np.abs(x[np.isfinite(x)])))


# positions, key heads, query heads, head_dim, window: a CTA or a cluster a head, parts of heads joined, shared heads
SHAPES = [(1, 1, 1, 64, 0), (40, 2, 2, 128, 0), (700, 3, 12, 128, 300), (700, 1, 5, 64, 0), (9000, 1, 2, 128, 0),
          (2500, 2, 24, 64, 0)]


@pytest.mark.parametrize("n,kv_heads,heads,hd,window", SHAPES[1:])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_attention_infinite_f16_keys(n, kv_heads, heads, hd, window, dtype):
    """A key of -inf score has weight 0; heads that give it the score +inf, or meet a zero, are NaN."""
    rng = np.random.default_rng(n + heads)
    k, v = (rng.normal(0, 1, (n, kv_heads, hd)) for _ in range(2))
    q = rng.normal(0, 1, (heads, hd))
    for at in {n - 1, max(0, n - 20), n // 2}:
        d = rng.integers(0, hd)
        k[at, :, d] = np.inf
        q[:, d] = -np.abs(q[:, d]) - 0.1
        if at == n // 2:
            q[-1, d] *= -1
    q = torch.from_numpy(q.astype(np.float32)).to(dtype).to(DEV)
    r = Rows(k, v, window=window)
    out, lse = r.run(q[None])
    want = r.want(q)
    assert np.isfinite(want[0][:-1]).all()
    check_edges((out[0], lse[0]), want, finite_max(r.v), dtype)


@pytest.mark.parametrize("n,kv_heads,heads,hd,window", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_infinite_f16_values(n, kv_heads, heads, hd, window, dtype):
    """An infinite value makes its element infinite, two of opposite signs make it NaN, the others stay."""
    rng = np.random.default_rng(n + heads)
    k, v = (rng.normal(0, 1, (n, kv_heads, hd)) for _ in range(2))
    v[n - 1, :, 3] = np.inf
    v[max(0, n - 9), 0, 40] = -np.inf
    if n > 1:
        v[n - 1, -1, 17], v[n - 2, -1, 17] = np.inf, -np.inf
    q = torch.from_numpy(rng.normal(0, 1, (heads, hd)).astype(np.float32)).to(dtype).to(DEV)
    r = Rows(k, v, window=window)
    out, lse = r.run(q[None])
    check_edges((out[0], lse[0]), r.want(q), finite_max(r.v), dtype)


@pytest.mark.parametrize("n,kv_heads,heads,hd,window", SHAPES)
def test_attention_infinite_q4_scales(n, kv_heads, heads, hd, window):
    rng = np.random.default_rng(n + heads)
    k, v = (rng.normal(0, 1, (n, kv_heads, hd)) for _ in range(2))
    q = rng.normal(0, 1, (heads, hd))
    q[:, 32:64] = np.abs(q[:, 32:64]) + 0.1
    q = torch.from_numpy(q.astype(np.float32)).to(DEV)

    def value(_, vals):
        vals[1][n - 1, :, 1] = np.inf

    def key_low(keys, _):  # every element -8 * inf: the score is -inf
        keys[0][n - 1, :, 16:32] = 0
        keys[1][n - 1, :, 1] = np.inf

    def key_any(keys, _):  # a block counts by the sign of its sum
        keys[1][n - 1, :, 0] = np.inf

    for edit in (value, key_low, key_any):
        r = Rows(k, v, "q4_0", edit, window=window)
        out, lse = r.run(q[None])
        want = r.want(q)
        if edit is not value and n == 1:
            continue  # a lone key of score -inf: nothing to attend to
        check_edges((out[0], lse[0]), want, finite_max(r.v))


def test_attention_over_rows_that_append_made_infinite():
    """Keys past fp16's range are stored as infinities."""
    cache = paged.PagedKV.empty(paged.PageBook.empty(1, 4, 16, 4), 1, 1, 64)
    k = torch.randn(20, 1, 64, device=DEV)
    k[7, 0, 5] = 1e5
    v = torch.randn(20, 1, 64, device=DEV)
    cache.append(0, k, v, i32(np.arange(20)))
    cache.book.table[0, :2] = i32([0, 1])
    cache.book.lens[0] = 20
    q = torch.randn(1, 2, 64, device=DEV)
    q[0, :, 5] = -0.25
    out = torch.empty_like(q)
    cache.attention(0, q, out)
    left = [i for i in range(20) if i != 7]
    kk, vv = k.half().double()[left, 0], v.half().double()[left, 0]
    want = torch.softmax(q[0].double() @ kk.T / 8, -1) @ vv
    assert (out[0].double() - want).abs().max() < 2.0 ** -15


# ---------------------------------------------------------------- weights, scales and queries of very different sizes
#
# Both parts of a factor x = hi + lo / 2^11 keep it to 2^-22 relative, and to
# 2^-36 absolute where that is more (lo's last bit, 2^-24, halved and divided by
# 2^11).  A weight is held times 2^7 or more over the largest of its piece, so
# n weights are off by n 2^-43 of the largest besides; with Q4_0 scales, which
# are brought below 1 by a power of two up to 4 times the largest, codes up
# to 8, by n 2^-42 of the largest |v|.

@pytest.mark.parametrize("kv", ["f16", "q4_0"])
@pytest.mark.parametrize("rows,bits", [(1, 32.0), (2048, 32.0), (2048, 28.5), (1, 36.0)])
def test_attention_many_small_weights(kv, rows, bits):
    """One position 2^bits above 65535 others of equal weight, a warp walking few of them or all.
    Scores are exact but for two roundings of some 36 (2^-18 of a weight)."""
    n, hd = 65536, 64
    k, v = np.zeros((n, 1, hd)), np.ones((n, 1, hd))
    k[0, 0, 0], v[0] = 8.0, 0.0
    r = Rows(k, v, kv)
    assert (r.k * r.k_scale[..., :1] == k).all() and (r.v == v).all()
    q = torch.zeros(rows, 1, hd, device=DEV)
    q[:, 0, 0] = bits * math.log(2.0)  # scale 1 / 8
    out, _ = r.run(q, rows=i32(np.zeros(rows)))
    p = math.exp(-float(q[0, 0, 0]))
    want = (n - 1) * p / (1 + (n - 1) * p)
    assert np.max(np.abs(out - want)) <= 2.0 ** -16 * want + n * 2.0 ** -42


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("group", [1, 2, 4])
def test_attention_q4_blocks_of_unequal_scales(hd, group):
    """Each block of 32 elements is as exact as its own values ask for."""
    n = 40
    rng = np.random.default_rng(hd + group)
    k, v = (rng.normal(0, 1, (n, 2, hd)) for _ in range(2))
    v[:, :, :32] *= 2.0 ** 9
    v[:, :, 32:64] *= 2.0 ** -11
    r = Rows(k, v, "q4_0")
    q = torch.from_numpy(rng.normal(0, 0.01, (2 * group, hd)).astype(np.float32)).to(DEV)
    (out, _), (want, _, off) = r.run(q[None]), r.want(q)
    top = np.abs(r.v).max()
    for b in range(hd // 32):
        e = slice(32 * b, 32 * b + 32)
        vmax = np.abs(r.v[:, :, e]).max()
        tol = (2 * off[:, None] + 2.0 ** -19) * vmax + n * 2.0 ** -42 * top
        assert (np.abs(out[0] - want)[:, e] <= tol).all(), b


@pytest.mark.parametrize("kv", ["f16", "q4_0"])
@pytest.mark.parametrize("heads", [1, 4, 8])
def test_attention_query_with_one_large_element(kv, heads):
    """A query element 2^24 times the others, whose keys are 0: the others keep their bits.
    2^-46 of the large one, over 128 elements, is below the bound of 2^-20 sum |q k|."""
    rng = np.random.default_rng(heads)
    k, v = (rng.normal(0, 1, (3, 1, 128)) for _ in range(2))
    k[:, :, 0] = 0
    q = rng.normal(0, 1, (heads, 128))
    q[:, 0] = 2.0 ** 24
    r = Rows(k, v, kv)
    q = torch.from_numpy(q.astype(np.float32)).to(DEV)
    out, lse = r.run(q[None])
    check_edges((out[0], lse[0]), r.want(q), finite_max(r.v))


# ---------------------------------------------------------------- arguments

def test_append_with_queries_names_theta():
    book = paged.PageBook.empty(1, 4, 16, 4)
    cache = paged.PagedKV.empty(book, 1, 1, 64)
    x = torch.randn(2, 1, 64, device=DEV)
    with pytest.raises(ValueError, match="theta"):
        cache.append(0, x, x, i32([0, 1]), pos=i32([0, 1]), q=x, q_out=x)
    with pytest.raises(ValueError, match="q_out"):
        cache.append(0, x, x, i32([0, 1]), pos=i32([0, 1]), q_out=x, theta=1e4)


@pytest.mark.parametrize("value", [1e-50, -1e-60])
def test_scale_and_theta_below_fp32(value):
    """What fp32 rounds to 0 is not taken for 0, which means 1 / sqrt(head_dim), or no rotation."""
    c = base.Case([5], 1, 64, 16)
    q = torch.randn(1, 1, 64, device=DEV)
    with pytest.raises(ValueError, match="scale"):
        c.cache.attention(0, q, torch.empty_like(q), scale=value)
    with pytest.raises(ValueError, match="theta"):
        c.cache.append(0, q, q, i32([0]), pos=i32([0]), theta=value)


@pytest.mark.parametrize("kw", [dict(page_size=2 ** 32 + 16), dict(page_size=16, window=2 ** 32), dict(page_size=0),
                                dict(page_size=65537), dict(page_size=16, window=-1)])
def test_book_sizes_out_of_range(kw):
    with pytest.raises(ValueError):
        paged.PageBook(i32([[-1]]), i32([0]), i32([0]), i32([0, 1, 0, 0]), **kw)


# ---------------------------------------------------------------- a pair of CTAs a head

@pytest.mark.parametrize("kv,hd,group", [("f16", 128, 8), ("f16", 64, 8), ("f16", 128, 1), ("q4_0", 128, 2), ("q4_0", 64, 4)])
@pytest.mark.parametrize("ps", [16, 20])
def test_attention_pairs_of_ctas(kv, hd, group, ps):
    """48 to 80 key heads of up to 380 positions: two CTAs each, of which a short row leaves one idle."""
    for rows, n in ((6, 380), (10, 250)):
        lens = [n, 0, 1, n // 3] + [n] * (rows - 4)
        base.check(base.Case(lens, 8, hd, ps, kv, seed=rows, window=n), 8 * group)


def test_plan_without_undo():
    """The undo buffer may be left out: plans that are adopted are served as before."""
    n_req, n_pages, ps, window, first, second, most = REPEATED["histories"]
    s = Steps(n_req, n_pages, ps, 120, window, most)
    s.book._c.undo = None
    for new in (first, [-1] * n_req, second, [1, 0, -1, 1, 1], [3, 50, 9, 0, 0]):
        s.sim = s.check(new, s.plan(new))
        s.adopt()
