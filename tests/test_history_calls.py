"""CPU: what the event-history modules and entries do with arguments at the edge of
what they document."""
import torch


def test_last_row_of_an_empty_history_is_zero_whatever_its_neighbours_hold():
    from fast_b200.history import HistoryEncoder
    rows = torch.tensor([[1.0, 2.0], [3.0, 4.0], [float("inf"), float("nan")], [5.0, 6.0]], requires_grad=True)
    starts = torch.tensor([0, 0, 3, 3, 4, 4])
    out = HistoryEncoder.last(rows, starts)
    assert torch.equal(out[[0, 2, 4]], torch.zeros(3, 2)) and torch.equal(out[3], rows[3])
    assert bool(torch.isinf(out[1, 0])) and bool(torch.isnan(out[1, 1]))
    # an empty history hands no gradient to the row in front of it
    grad, = torch.autograd.grad(out[[0, 2, 4]].sum() + out[3].sum(), rows)
    assert torch.equal(grad, torch.tensor([[0.0, 0.0], [0.0, 0.0], [0.0, 0.0], [1.0, 1.0]]))


def test_last_rows_stay_inside_the_rows():
    """starts beyond the rows are clamped to them, as the operators do, and not left to an index out of range."""
    from fast_b200.history import HistoryEncoder
    rows = torch.arange(8.0).view(4, 2)
    assert torch.equal(HistoryEncoder.last(rows, torch.tensor([0, 2, 9, 9, 12])), torch.stack([rows[1], rows[3], *torch.zeros(2, 2)]))
    assert torch.equal(HistoryEncoder.last(rows, torch.tensor([-3, -1, 4])), torch.stack([torch.zeros(2), rows[3]]))
