"""One workspace for calls of many shapes, one after another, as a batch grows and shrinks: every call gives the
bits that it gives with a workspace of its own."""
import numpy as np
import pytest

from conftest import pkg
from test_gpu_paged import Pool, _check_attention, _torch

pytestmark = pytest.mark.gpu


def _call(pool, act, heads, ws, q):
    import torch
    P = pkg()
    b = len(pool.lens)
    out = torch.full_like(q, 7.0)
    lse = torch.full((b, heads), 7.0, device="cuda")
    P.paged_attn_device(pool.kv, act, q.data_ptr(), q.stride(0), b, heads, pool.d_len.data_ptr(), pool.d_table.data_ptr(),
                        pool.d_table.stride(0), pool.dim ** -0.5, out.data_ptr(), out.stride(0), ws.data_ptr(), ws.numel(),
                        lse.data_ptr())
    torch.cuda.synchronize()
    return torch.cat([out.float().flatten(), lse.flatten()])


def test_one_workspace_through_calls_of_many_shapes(cuda_ok):
    """A long sequence in more than 32 parts (joined in two steps), then batches of more and fewer sequences, other
    head counts, head sizes and types, then the same again."""
    import torch
    P = pkg()
    shapes = [("f16", "f16", [60003], 8, 4, 128), ("f16", "f16", [60003] + [100] * 63, 8, 4, 128), ("f16", "f16", [700] * 301, 2, 1, 64),
              ("bf16", "bf16", [9001, 0, 50], 1, 16, 64), ("f32", "f32", [5000, 1, 4097], 2, 3, 256),
              ("f32", "bf16", [3000] + [200] * 200, 3, 3, 96), ("bf16", "bf16", [50000], 1, 9, 128), ("f16", "f16", [1], 1, 1, 8)]
    calls = []
    for i, (act, cache, lens, hk, rep, dim) in enumerate(shapes):
        pool = Pool(lens, 64, hk, dim, cache, seed=i)
        q = torch.randn(len(lens), hk * rep * dim, generator=torch.Generator("cuda").manual_seed(i), device="cuda").to(_torch(act))
        own = torch.zeros(P.paged_attn_workspace(len(lens), hk * rep, dim), dtype=torch.uint8, device="cuda")
        calls.append((pool, act, hk * rep, q, _call(pool, act, hk * rep, own, q)))
        assert not (calls[-1][4] == 7.0).all()
    room = max(P.paged_attn_workspace(len(p.lens), h, p.dim) for p, _, h, _, _ in calls)
    ws = torch.zeros(room, dtype=torch.uint8, device="cuda")
    order = list(range(len(calls))) + [1, 0, 2, 0, 6, 1, 3, 5, 4, 7, 1] + np.random.default_rng(0).integers(0, len(calls), 40).tolist()
    for at, i in enumerate(order):
        pool, act, heads, q, want = calls[i]
        assert torch.equal(_call(pool, act, heads, ws, q), want), (at, i)


def test_calls_that_share_a_workspace_are_right(cuda_ok):
    """The shapes of the test above that are joined in two steps, against 64 bits."""
    _check_attention(Pool([20003] + [100] * 9, 64, 2, 64, "f16", seed=1), "f16", 4, 64 ** -0.5)
    _check_attention(Pool([50000], 64, 1, 128, "bf16", seed=2), "bf16", 9, 128 ** -0.5)
