"""Page copies over layers that lie one after another with room between them, and side by side within a page's stride."""
import numpy as np
import pytest

from conftest import pkg
from test_gpu_paged import _torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", ["f32", "bf16"])
@pytest.mark.parametrize("side_by_side", [False, True])
def test_copy_pages_layer_layouts(cache, side_by_side, cuda_ok):
    import torch
    P = pkg()
    layers, pages, page, hk, dim, n = 5, 40, 16, 3, 64, 18
    size = hk * page * dim
    big = [torch.randn(pages * layers * (size + 8) + 64, device="cuda").to(_torch(cache)) for _ in range(2)]
    page_stride, layer_stride = (layers * (size + 8), size + 8) if side_by_side else (size + 8, pages * (size + 8))
    view = lambda t: t.as_strided((layers, pages, size), (layer_stride, page_stride, 1))
    want = [t.clone() for t in big]
    order = np.random.default_rng(n).permutation(pages)
    src, dst = order[:n], order[n: 2 * n]
    for w in want:
        view(w)[:, torch.from_numpy(dst.copy()).cuda()] = view(w)[:, torch.from_numpy(src.copy()).cuda()].clone()
    kv = P.paged_kv(big[0].data_ptr(), big[1].data_ptr(), cache, pages, page, hk, dim, (page_stride, page * dim, dim))
    P.copy_pages_device(kv, src, dst, layers, layer_stride)
    torch.cuda.synchronize()
    for w, t in zip(want, big):
        assert torch.equal(w, t)
