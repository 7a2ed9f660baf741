"""The paged-sessions example: a small stack of layers over the paged cache,
with sessions that join, idle, end and are replaced.  Every layer's attention
is compared with bmo_k_decode_attention over a ring of the session's own that
is given the same projection rows.

Bound: rows are stored bit for bit alike (test_gpu_paged.py), so the two differ
by the paged kernel's arithmetic: (2 d + 2^-19) max |v| with d = 2^-20 scale
sum |q k| (test_gpu_paged.py).  The projections give scale sum |q k| below 14,
so 2^-15 max |v|."""
import numpy as np
import pytest
from gguf import GGMLQuantizationType, quants

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from bmo_jetson_b200 import engine  # noqa: E402
from bmo_jetson_b200.examples import paged_sessions as ex  # noqa: E402
from oracle import oracle as orc  # noqa: E402

DEV = torch.device("cuda:0")
DIM, HEADS, KV_HEADS, HD, FFN, LAYERS, CTX = 256, 4, 2, 64, 512, 2, 64


def layers():
    rng = np.random.default_rng(3)

    def matrix(rows, cols, f=0):
        w = rng.normal(0, 0.06, (rows, cols)).astype(np.float32)
        b = np.ascontiguousarray(quants.quantize(w, GGMLQuantizationType.Q4_0))
        return ex.Matrix(torch.from_numpy(b.reshape(-1)).to(DEV), rows, cols, f)

    def gamma():
        return torch.from_numpy((1 + 0.1 * rng.normal(0, 1, DIM)).astype(np.float32)).to(DEV)

    kv = KV_HEADS * HD
    return [ex.Layer(gamma(), matrix(DIM + 2 * kv, DIM), matrix(DIM, DIM), gamma(), matrix(2 * FFN, DIM, FFN),
                     matrix(DIM, FFN)) for _ in range(LAYERS)]


class Rings:
    """An fp16 or Q4_0 ring of CTX slots for each session and all layers."""

    def __init__(self, n_req, kv_type):
        self.kv_type = kv_type
        n = LAYERS * KV_HEADS * CTX * HD
        self.pos = [0] * n_req
        if kv_type == engine.KV_F16:
            self.planes = [[torch.zeros(n, dtype=torch.float16, device=DEV) for _ in range(2)] + [None, None] for _ in range(n_req)]
        else:
            self.planes = [[torch.zeros(n // 2, dtype=torch.uint8, device=DEV) for _ in range(2)] +
                           [torch.zeros(n // 32, dtype=torch.float16, device=DEV) for _ in range(2)] for _ in range(n_req)]

    def attend(self, r, layer, qkv):
        """(attention of session r's projection row at its position, largest |v| of its ring)."""
        q_dim, kv = HEADS * HD, KV_HEADS * HD
        p = self.pos[r]
        v = qkv[q_dim + kv:].copy()
        if p == 0:  # a ring whose window is one position returns v as it is given, a page as it is stored
            v = v.astype(np.float16).astype(np.float32) if self.kv_type == engine.KV_F16 else \
                orc.dequantize_q4_0(orc.quantize_q4_0(v.reshape(-1, 32)).reshape(-1, 18), v.size).reshape(-1)
        q, k, v = (torch.from_numpy(np.ascontiguousarray(t, np.float32)).to(DEV) for t in (
            orc.rope(qkv[:q_dim], HEADS, HD, p), orc.rope(qkv[q_dim:q_dim + kv], KV_HEADS, HD, p), v))
        pos = torch.tensor([p], dtype=torch.int32, device=DEV)
        out = torch.empty(q_dim, device=DEV)
        ptr = [None if t is None else t.data_ptr() for t in self.planes[r]]
        rc = engine.lib().bmo_k_decode_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), *ptr, out.data_ptr(), HD, HEADS,
                                                 KV_HEADS, CTX, pos.data_ptr(), layer, self.kv_type,
                                                 torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        torch.cuda.synchronize()
        return out


class Compared(ex.PagedSessions):
    """The example's sessions, each attention beside the ring's."""

    def attend(self, i, qkv, slot, pos, req):
        before = qkv.cpu().numpy()
        a = super().attend(i, qkv, slot, pos, req)
        self.vmax = max(self.vmax, float(np.abs(before[:, (HEADS + KV_HEADS) * HD:]).max()))
        assert pos.tolist() == [self.rings.pos[r] for r in req.tolist()]
        for j, r in enumerate(req.tolist()):
            worst = float((a[j] - self.rings.attend(r, i, before[j])).abs().max())
            assert worst <= 2.0 ** -15 * self.vmax, (i, r, worst)
            self.checked += 1
        return a


@pytest.mark.parametrize("kv_type", [engine.KV_F16, engine.KV_Q4_0])
@pytest.mark.parametrize("page_size", [16, 10])
def test_paged_sessions_match_rings(kv_type, page_size):
    n_req = 3
    pages = n_req * (CTX // page_size + 2)
    s = Compared(layers(), HEADS, KV_HEADS, HD, n_req, pages, page_size, max_len=400, window=CTX, kv_type=kv_type)
    s.rings, s.vmax, s.checked = Rings(n_req, kv_type), 0.0, 0
    rng = np.random.default_rng(page_size)
    for f in range(90):
        new = [1, 1 if f % 3 else 0, 1 if f > 20 else 0]
        if f == 50:
            new[0] = -1
        live = [r for r in range(n_req) if new[r] > 0]
        y = s.frame(torch.from_numpy(rng.normal(0, 1, (len(live), DIM)).astype(np.float32)).to(DEV), new)
        assert torch.isfinite(y).all() and s.refused() == 0
        for r in range(n_req):
            s.rings.pos[r] = 0 if new[r] < 0 else s.rings.pos[r] + new[r]
    assert s.book.lens.tolist() == [39, 60, 69] and s.checked == LAYERS * (89 + 60 + 69)
    assert int(s.book.state[1]) == pages - sum(-(-n // page_size) - max(0, n - CTX) // page_size for n in (39, 60, 69))


def test_paged_sessions_out_of_pages():
    """A frame that the pool cannot serve is refused as a whole and reported."""
    stack = layers()
    s = ex.PagedSessions(stack, HEADS, KV_HEADS, HD, 2, 1, 16, max_len=64)
    s.book.plan(torch.tensor([1, 1], dtype=torch.int32, device=DEV), *(t for t in s.lists), s.offsets)
    assert s.refused() != 0 and s.book.lens.tolist() == [0, 0] and (s.lists[0] == -1).all()


def test_example_command():
    assert ex.main(["--sessions", "5", "--frames", "30", "--layers", "2", "--dim", "256", "--heads", "4", "--kv-heads", "2",
                    "--ffn", "512", "--window", "40", "--kv", "f16"]) == 0
