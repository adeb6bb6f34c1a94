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


@pytest.mark.parametrize("bad", [-1, 512, 2**31 - 1, -600])
def test_an_id_that_is_none_shows_in_its_own_sequence(bad, cuda_ok):
    """What a row with no token to draw gives (-1), or an id past the vocabulary: NaN for that sequence alone."""
    import torch
    P, E = pkg(), _example()
    model = E.PagedDecoder(P.synthetic_pgw("tiny-llama", 6), 60, 4, "f32", 3)
    first, _ = model.read(P.seeded_prompt(6, 512, 4))
    seqs = [first] + [model.pages.fork(first) for _ in range(2)]
    twins = [model.pages.fork(first) for _ in range(3)]
    logits = model.step(seqs, torch.tensor([7, bad, 9], device="cuda"))
    want = model.step(twins, torch.tensor([7, 8, 9], device="cuda"))
    assert torch.isnan(logits[1]).all() and torch.equal(logits[[0, 2]], want[[0, 2]])
    ids, lp = E.sample(logits, torch.full((3,), 0.5, device="cuda"), temperature=0.0)
    assert ids[1] == -1 and (ids[[0, 2]] >= 0).all()
    logits, want = model.step(seqs, ids), model.step(twins, torch.stack([ids[0], ids[0], ids[2]]))
    assert torch.isnan(logits[1]).all() and torch.equal(logits[[0, 2]], want[[0, 2]])


def test_pages_are_given_back_where_they_run_out(cuda_ok):
    P, E = pkg(), _example()
    model = E.PagedDecoder(P.synthetic_pgw("tiny-llama", 6), 6, 4, "f32", 3)
    with pytest.raises(MemoryError):
        model.read(P.seeded_prompt(25, 512, 1))
    assert model.pages.free_pages == 6
    with pytest.raises(MemoryError):
        E.continuations(model, P.seeded_prompt(8, 512, 1), 3, 12, temperature=0.5)
    assert model.pages.free_pages == 6
    ids, _ = E.continuations(model, P.seeded_prompt(8, 512, 1), 3, 4, temperature=0.5)
    assert ids.shape == (3, 4) and model.pages.free_pages == 6
