"""Host side of the paged serving operators: workspaces, page lists and sizes at their limits (no GPU needed)."""
import pytest

from conftest import pkg


@pytest.mark.parametrize("heads,dim", [(1, 8), (4, 64), (32, 128), (64, 256)])
def test_workspace_does_not_depend_on_the_number_of_sequences(heads, dim):
    """What a workspace holds, and where, is the same for every batch, so that batches can follow one another in it."""
    P = pkg()
    assert len({P.paged_attn_workspace(n, heads, dim) for n in (1, 2, 63, 512, 65535)}) == 1
