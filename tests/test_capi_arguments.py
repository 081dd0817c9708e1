"""What the binding makes of tensors before a call: no GPU needed."""
import pytest

torch = pytest.importorskip("torch")
from wavenet_amd import capi


def test_strides_of_tensors_that_are_not_contiguous():
    big = torch.zeros(10, 40)
    lies = capi._strided
    v = big[:, 3:11]                                       # rows with gaps
    assert lies(v, 10, 40, 8, 1) and lies(v, 4, 40, 5, 1)
    assert not lies(v, 10, 8, 8, 1) and not lies(v, 11, 40, 8, 1) and not lies(v, 10, 40, 9, 1)
    v = big[:, ::2]                                        # and gaps in them
    assert lies(v, 10, 40, 20, 2) and not lies(v, 10, 20, 20, 1) and not lies(v, 10, 40, 20, 1)
    v = big.t()                                            # column by column
    assert lies(v, 40, 1, 10, 40) and not lies(v, 40, 10, 10, 1)
    assert lies(v, 10, 40, 40, 1)                          # the same values as they lie in memory
    assert lies(big[:, 5], 10, 40, 1, 1) and not lies(big[:, 5], 10, 1, 1, 1)
    assert lies(big[:, 5], 1, 10, 10, 40) and not lies(big[:, 5], 1, 10, 10, 1)
    v = torch.zeros(6, 5, 8)[:, 1:]                        # examples of 4 columns, 8 samples each, out of 5
    assert lies(v, 6, 40, 32, 1) and not lies(v, 6, 32, 32, 1) and not lies(v, 6, 40, 33, 1)
    v = torch.zeros(6, 5, 8)[::2]                          # a dimension more than the rows
    assert lies(v, 5, 8, 8, 1) and lies(v, 3, 80, 40, 1)
    v = torch.zeros(1, 8).expand(4, 8)                     # one row four times
    assert not lies(v, 4, 8, 8, 1)


def test_tables_whose_rows_are_out_of_step():
    wide = capi._out_of_step
    t = torch.zeros
    assert wide(t(6, 3), 12, (2, 1)) and wide(t(6, 4), 12, (2, 1)) and wide(t(6, 5), 6 * 3, (3, 1))
    assert wide(t(6, 3, 4), 6 * 2 * 4, (8, 4)) and wide(t(6, 2, 5), 6 * 2 * 4, (8, 4))
    # rows to spare, one row, no rows, other shapes of the very table
    for x in (t(6, 2), t(7, 2), t(12), t(20), t(1, 20), t(3, 4), t(12, 1), t(14, 1)):
        assert not wide(x, 12, (2, 1))
    for x in (t(6, 2, 4), t(12, 4), t(6, 8), t(15, 4), t(48), t(50)):
        assert not wide(x, 48, (8, 4))
