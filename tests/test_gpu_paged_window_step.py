"""Serving through a sliding window with the pages behind it given back before every step:
from the first new token's position less window - 1 on, rows are still seen."""
import numpy as np
import pytest

from test_gpu_paged_more_step import PR, Server

pytestmark = pytest.mark.gpu


class Windowed(Server):
    def __init__(self, qk, t, type, window, **kw):
        super().__init__(qk, t, type, **kw)
        self.window = window

    def resize(self, lengths):
        """Of a step's rows those that some new token sees, and the new ones."""
        begins = [len(x) - (self.window - 1) for x in self.rows[0]]
        self.qk.pages_resize(self.pool, self.i32(lengths), begins=self.i32(begins), missing=self.missing, workspace=self.ws)
        assert int(self.missing) == 0
        table = self.pool.page_table.cpu().numpy()
        for r, (begin, n) in enumerate(zip(begins, lengths)):
            if n >= 0:
                held = np.flatnonzero(table[r] >= 0)
                assert held.tolist() == list(range(max(begin, 0) // PR, -(-n // PR)))


@pytest.mark.parametrize("type", ["I4", "F16"])
@pytest.mark.parametrize("window", [1, 16, 17, 40, 64])
def test_chunks_and_tokens_through_a_window(qk, torch_gpu, type, window):
    """The pool holds less than the sequences' whole contexts: 3 rows of 20 entries, 36 pages."""
    rng = np.random.default_rng(window)
    s = Windowed(qk, torch_gpu, getattr(qk, type), window, rows=3, pages=36, stride=20)
    s.step(rng, [(0, 70), (1, 33)], window=window)
    for counts in ([(0, 1), (1, 1)], [(0, 50), (1, 3), (2, 90)], [(2, 1), (0, 17)], [(1, 100), (0, 16), (2, 1)],
                   [(0, 100), (1, 1)], [(2, 95), (1, 64)], [(0, 1), (1, 1), (2, 1)]):
        s.step(rng, counts, window=window)
    assert sum(len(x) for x in s.rows[0]) > 36 * PR
