"""The paged serving operators together, as examples/paged_sampling.py runs them, against the engine that
decodes one contiguous sequence (CudaPetitGPT.generate): greedy ids are equal, with and without forks, on
pages that are shared, copied before a write and moved by a compaction."""
import importlib.util
import os

import numpy as np
import pytest

from conftest import ROOT, pkg

pytestmark = pytest.mark.gpu


def _example():
    spec = importlib.util.spec_from_file_location("paged_sampling", os.path.join(ROOT, "examples", "paged_sampling.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("page_len", [3, 16])
def test_greedy_forks_follow_the_engine(page_len, cuda_ok):
    P, E = pkg(), _example()
    data = P.synthetic_pgw("tiny-llama", 3)
    eng = P.CudaPetitGPT(data)
    prompt = P.seeded_prompt(21, 512, 1)
    want = eng.generate(prompt, maxNewTokens=24, eosId=-1)["generatedIds"]
    eng.destroy()
    model = E.PagedDecoder(data, 60, page_len, "f32", 3)
    ids, logprobs = E.continuations(model, prompt, 3, 24, temperature=0.0)
    assert ids.tolist() == [want] * 3
    assert (logprobs == 0).all()  # the only token kept
    assert model.pages.free_pages == 60  # everything was given back


def test_forks_diverge_and_survive_a_compaction(cuda_ok):
    """Forks that continue with other ids each follow the sequence that has those ids alone; pages move in between."""
    import torch
    P, E = pkg(), _example()
    data = P.synthetic_pgw("tiny-llama", 5)
    model = E.PagedDecoder(data, 80, 4, "f32", 4)
    prompt = P.seeded_prompt(10, 512, 2)
    holes, _ = model.read(prompt[:7])
    first, logits = model.read(prompt)
    seqs = [first] + [model.pages.fork(first) for _ in range(2)]
    shared = model.pages.pages(first)
    extra = np.random.default_rng(0).integers(0, 512, (3, 9))
    for i in range(9):
        logits = model.step(seqs, torch.from_numpy(extra[:, i]).cuda())
        if i == 4:
            model.pages.free(holes)
            model.copy(model.pages.compact())
            assert max(p for s in seqs for p in model.pages.pages(s)) < 80 - model.pages.free_pages
    assert len(shared) == 3
    for row, s in zip(extra, range(3)):
        alone, one = model.read(np.concatenate([prompt, row]))
        # the same products and sums in the same order, but for the batch's row count in the matrix products
        assert (one[0] - logits[s]).abs().max() <= 1e-3 * one.abs().max()
        model.pages.free(alone)


def test_sampled_ids_come_from_the_kept_tokens(cuda_ok):
    """A 16-bit cache and sampling settings: every id is among the row's top_k of the logits it was drawn from."""
    import torch
    P, E = pkg(), _example()
    model = E.PagedDecoder(P.synthetic_pgw("tiny-llama", 4), 40, 8, "bf16", 4)
    s, logits = model.read(P.seeded_prompt(9, 512, 3))
    seqs = [s] + [model.pages.fork(s) for _ in range(3)]
    logits = logits.expand(4, -1).contiguous()
    gen = torch.Generator(device="cuda").manual_seed(1)
    for _ in range(6):
        ids, lp = E.sample(logits, torch.rand(4, generator=gen, device="cuda"), temperature=0.9, top_k=5)
        top = logits.topk(5, -1)
        assert ((top.indices == ids[:, None]).sum(-1) == 1).all()
        ref = torch.log_softmax(top.values.double() / 0.9, -1)[top.indices == ids[:, None]]
        assert (lp - ref).abs().max() < 1e-5
        logits = model.step(seqs, ids)
