"""Host side of the paged serving operators: workspaces, page lists and sizes at their limits (no GPU needed)."""
import pytest

from conftest import pkg


@pytest.mark.parametrize("heads,dim", [(1, 8), (4, 64), (32, 128), (64, 256)])
def test_workspace_does_not_depend_on_the_number_of_sequences(heads, dim):
    """What a workspace holds, and where, is the same for every batch, so that batches can follow one another in it."""
    P = pkg()
    assert len({P.paged_attn_workspace(n, heads, dim) for n in (1, 2, 63, 512, 65535)}) == 1


A = 1 << 20  # an aligned address that nothing reads: every call below is refused before a launch


def _refused(code, kv, src, dst, layers=1, stride=0):
    P = pkg()
    with pytest.raises(P.MllmError) as e:
        P.copy_pages_device(kv, src, dst, layers, stride)
    assert e.value.code == code and "mllm_copy_pages" in str(e.value)


PAGE = 2 * 16 * 64  # elements of a page below


@pytest.mark.parametrize("layers,page_stride,stride", [
    (2, PAGE, PAGE),                      # a layer's page i is the next layer's page i - 1
    (2, PAGE, 7 * PAGE),                  # the last page of a layer is the first of the next
    (3, 2 * PAGE, PAGE),                  # room for two layers within a page's stride, not for three
    (2, 2 * PAGE, 15 * PAGE - 4),         # one 16-byte piece short of the last page
    (2, 2 * PAGE, PAGE + 4)])
def test_copy_pages_refuses_layers_that_overlap(layers, page_stride, stride):
    """Copies run in no order, so no page of a layer may be part of another layer's."""
    kv = pkg().paged_kv(A, A, "f32", 8, 16, 2, 64, (page_stride, 16 * 64, 64))
    _refused(-3, kv, [0], [1], layers, stride)
