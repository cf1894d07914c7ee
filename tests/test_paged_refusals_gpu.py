"""GPU checks of what the paged operators' binding turns down."""
import pytest
import torch

from scope_b200 import paged
from test_paged_gpu import BF, DEV, table_of

pytestmark = pytest.mark.gpu


def test_an_argument_whose_truth_raises_is_an_error():
    x = torch.ones(4, 2, 32, dtype=BF, device=DEV)
    pos, table = torch.zeros(4, dtype=torch.int32, device=DEV), table_of(8, 32)
    with pytest.raises(RuntimeError, match="ambiguous"):
        paged.rope(x, pos, table, inverse=torch.tensor([0, 1]))
    assert torch.equal(paged.rope(x, pos, table, inverse=torch.tensor(1)), paged.rope(x, pos, table, inverse=True))
