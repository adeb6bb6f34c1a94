"""examples/paged_sampling.py where pages, positions or ids run out: a step that cannot be made changes nothing."""
import pytest

from conftest import pkg
from test_gpu_paged_example import _example

pytestmark = pytest.mark.gpu


def test_a_step_without_enough_pages_changes_nothing(cuda_ok):
    """Two of three sequences would have room: after the failure all have their length, and go on as if it had not been."""
    import torch
    P, E = pkg(), _example()
    data = P.synthetic_pgw("tiny-llama", 6)
    prompt = P.seeded_prompt(8, 512, 4)
    ids = torch.tensor([3, 4, 5], device="cuda")
    logits = []
    for short in (False, True):
        model = E.PagedDecoder(data, 10, 4, "f32", 3)
        first, _ = model.read(prompt)
        seqs = [first] + [model.pages.fork(first) for _ in range(2)]
        if short:
            taken = model.pages.new()
            model.pages.grow(taken, 6 * 4)  # leaves two pages for three sequences
            with pytest.raises(MemoryError):
                model.step(seqs, ids)
            assert [model.pages.length(s) for s in seqs] == [8] * 3 and model.pages.free_pages == 2
            model.pages.free(taken)
        logits.append(model.step(seqs, ids))
    assert torch.equal(*logits)
