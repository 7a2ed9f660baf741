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
