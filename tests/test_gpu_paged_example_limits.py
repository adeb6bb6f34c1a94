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


def test_a_step_past_the_last_position_is_refused(cuda_ok):
    import torch
    P, E = pkg(), _example()
    model = E.PagedDecoder(P.synthetic_pgw("tiny-llama", 6), 60, 16, "f32", 2)
    most = model.cfg["maxSeqLen"]
    a, b = model.pages.new(), model.pages.new()
    model.pages.grow(a, most)
    model.pages.grow(b, 1)
    with pytest.raises(ValueError):
        model.step([b, a], torch.tensor([1, 2], device="cuda"))
    assert [model.pages.length(s) for s in (a, b)] == [most, 1]
    assert torch.isfinite(model.step([b], torch.tensor([1], device="cuda"))).all()


def test_a_prompt_is_checked_before_it_is_read(cuda_ok):
    P, E = pkg(), _example()
    model = E.PagedDecoder(P.synthetic_pgw("tiny-llama", 6), 60, 16, "f32", 2)
    for prompt in ([], [1, 2, -1], [1] * (model.cfg["maxSeqLen"] + 1)):
        with pytest.raises(ValueError):
            model.read(prompt)
    assert model.pages.free_pages == 60
