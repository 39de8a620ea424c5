"""Page bounds, selection of pages and shared prefixes where a call has just no room, numbers are at the end of their range, or offsets cannot be.  Bounds and lists are exact and
compared for equality; attention is held against 64 bits with the tolerance of test_gpu_attention.py."""
import pytest

from test_gpu_attention import backend  # noqa: F401
from test_gpu_select import run_select

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pages,tokens", [(5, 24), (100, 1), (400, 24), (500, 1), (1500, 1), (1500, 8), (5000, 1), (5000, 8), (9000, 1), (9000, 8)])
def test_select_no_room_between(backend, pages, tokens):
    """Lists that have room for the pages at their ends and for none of those between: on every way that a selection goes."""
    for first, recent in ((0, 0), (1, 16)):
        width = first + (recent + tokens + 14) // 16 + 1
        rest = 16 - (recent + tokens - 2) % 16  # of a context in its last page, so that the ends are as many pages as they can be
        lens = [16 * pages + rest, 700, 0]
        run_select(backend, lens, [tokens, 1, tokens], 8, 2, 64, 16, width, first, recent, tree=True, repeat=2)
    run_select(backend, [16 * pages + 3] * (40 if pages <= 400 else 2), [1] * (40 if pages <= 400 else 2), 4, 4, 128, 16, 1, 0, 0)
