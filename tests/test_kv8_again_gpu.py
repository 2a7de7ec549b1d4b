"""A step's page tables asked for again."""

import pytest
import torch

from test_kv8_gpu import fine, ints, run_tables, status, tables_case  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [20, 60, 1500])
def test_rows_that_began_anew_asked_for_again(status, rows):  # noqa: F811
    """With their lengths and marks cleared the step takes nothing more and says the same; as they are, their pages go back and come again."""
    from oxr_inference_b200 import ops

    case = tables_case(rows, 16, 30, rows, most_new=60, fresh=0.5)
    lengths, held, table, free, new, anew = case
    assert sum(f and q > 32 for f, q in zip(anew, new)) > 1
    state, first = run_tables(case, 16, sum(new), status)
    fine(status)
    before = [s.clone() for s in state]
    cleared = ints([0 if f else n for f, n in zip(anew, lengths)])
    again = ops.step_pages(cleared, *state[1:], ints(new), ints([0] * rows), page_size=16, tokens=sum(new), status=status)
    fine(status)
    assert all(torch.equal(a, b) for a, b in zip(state[1:], before[1:])) and all(torch.equal(a, b) for a, b in zip(first, again))
    # asked for as it was: the same lengths, positions and numbers of pages, on pages that no row shares with another
    anew_again = ops.step_pages(*state, ints(new), ints(anew), page_size=16, tokens=sum(new), status=status)
    fine(status)
    for a, b in zip(first[1:], anew_again[1:]):
        assert torch.equal(a, b)
    assert torch.equal(state[1], before[1]) and torch.equal(state[4], before[4])
    pages = [p for row, h in zip(state[2].tolist(), state[1].tolist()) for p in row[:h]] + state[3].tolist()[:int(state[4])]
    assert len(set(pages)) == len(pages)
