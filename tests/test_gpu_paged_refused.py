"""The paged-sessions example where a frame cannot be served, or is asked for wrongly."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from bmo_jetson_b200 import paged  # noqa: E402
from bmo_jetson_b200.examples import paged_sessions as ex  # noqa: E402
from tests.test_gpu_paged_sessions import DEV, DIM, HD, HEADS, KV_HEADS, layers  # noqa: E402


def test_refused_frame_is_seen_afterwards():
    """A frame that was refused gives NaN rows and stays in refused() after frames that were served."""
    s = ex.PagedSessions(layers(), HEADS, KV_HEADS, HD, 2, 1, 16, max_len=64)
    x = torch.randn(2, DIM, device=DEV)
    assert torch.isnan(s.frame(x, [1, 1])).all()  # two pages, one there
    assert torch.isfinite(s.frame(x[:1], [1, 0])).all()
    assert s.refused() == paged.NO_PAGES and s.refused() == 0
    assert torch.isfinite(s.frame(x[:1], [1, 0])).all() and s.refused() == 0
    assert s.book.lens.tolist() == [2, 0]


def test_frame_takes_a_position_a_session():
    s = ex.PagedSessions(layers(), HEADS, KV_HEADS, HD, 2, 4, 16, max_len=64)
    x = torch.randn(2, DIM, device=DEV)
    for new in ([2, 0], [1], [1, 1, 1]):
        with pytest.raises(ValueError):
            s.frame(x, new)
    with pytest.raises(ValueError):
        s.frame(x, [1, 0])
    assert s.refused() == 0 and s.book.lens.tolist() == [0, 0]


def test_example_command_without_a_window():
    assert ex.main(["--sessions", "3", "--frames", "40", "--layers", "1", "--dim", "128", "--heads", "2", "--kv-heads", "1",
                    "--ffn", "256", "--window", "0"]) == 0
