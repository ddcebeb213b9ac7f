"""Attention over the 8-bit cache where its definition is easiest to lose: windows as long as an int."""
import pytest
import torch

from tests.test_gpu_attention import FORMS, attend64, compare, make, queries, run

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


# -- windows -------------------------------------------------------------------------

@pytest.mark.parametrize("rows,width,spare", FORMS)
def test_windows_as_long_as_an_int(gpu, rows, width, spare):
    """A window longer than every sequence hides nothing, also from sequences with rows before their first token."""
    lengths = [max(1, rows // 2), 0, rows + 20, min(5, rows)]
    cache, table = make(gpu, lengths, 1, 16, 64, seed=90)
    q, starts = queries(4 * rows, 2, 64, BF16, gpu, seed=90), [i * rows for i in range(5)]
    want, bound = attend64(q, cache, table, lengths, starts, 0.125, True, 0)
    all_of_it = run(q, cache, table, lengths, starts, gpu, width, spare)
    compare(all_of_it, want, bound)
    for window in (2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - rows, 2 ** 30):
        assert torch.equal(run(q, cache, table, lengths, starts, gpu, width, spare, window=window), all_of_it)
