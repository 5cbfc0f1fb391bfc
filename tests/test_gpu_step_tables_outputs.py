"""What the outputs of step_tables keep alive."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_small_outputs_do_not_hold_the_tables(hcu, dev):
    """free_head goes from step to step, and lengths or slots may be kept: none of them holds the step's tables alive."""
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)
    t = hcu.step_tables(i(4, 64), i(4), i(4), torch.ones_like(i(4)), i(8), i(1), 4, 4096)
    for k in ("lengths", "positions", "token_loc", "loc", "free_head"):
        x = getattr(t, k)
        assert x.untyped_storage().nbytes() <= 1024, k
    assert t.page_table_size_1.untyped_storage().nbytes() >= 4 * 4096 * 4
