"""Precision of the paged attention where most of a row's weights are small, against 64 bits.

Bounds are relative to the sum of the row's own terms, A = sum p |v|, not to the largest value.  With
u = 2^-24 (half an f32 ulp), D the head size and n the length:
- a score is off by at most ds = (D + 4) u scale sum |q k|, which enters through the weight and through the sum;
- each of the n positions adds one rounding to a sum and, when the maximum moves, up to one to its factor: (2 n + 32) u;
- weights of 16-bit queries have two terms of the cache's type: 2^-16 of a weight in bf16, 2^-22 in f16; f32 queries
  over f16 have two as well, and 2^-22 as well;
- f16 ends at 2^-24, which is 2^-39 of the largest weight or query element where those are scaled to 2^15: half
  of that, 2^-40, for each position, or each element (a row of queries is scaled to between 2^14 and 2^15, which
  may double its share: ds holds that many times over);
- the output is rounded once: half an ulp of it, for f16 at least half of 2^-24.
"""
import math

import numpy as np
import pytest

from test_gpu_paged import HALF, KINDS, U, Pool, _attend, _torch

pytestmark = pytest.mark.gpu
TERMS = {("f32", "f32"): 0.0, ("f16", "f16"): 2.0 ** -22, ("bf16", "bf16"): 2.0 ** -16, ("f32", "bf16"): 0.0,
         ("f32", "f16"): 2.0 ** -22}


def _put(pool, which, seq, rows):
    """rows [kv head][n][dim] become the keys (0) or values (1) of a sequence."""
    import torch
    rows = torch.from_numpy(rows.astype(np.float32)).cuda().to(_torch(pool.cache))
    for p0 in range(0, rows.shape[1], pool.page):
        m = min(pool.page, rows.shape[1] - p0)
        pool.full[which][pool.table[seq, p0 // pool.page], :, :m] = rows[:, p0: p0 + m]


def _compare(pool, act, heads, scale, q):
    q, out, lse = _attend(pool, act, heads, scale, q=q)
    floor = 2.0 ** -40 if pool.cache == "f16" else 0.0
    for s, n in enumerate(pool.lens):
        k, v = pool.rows(0, s, n), pool.rows(1, s, n)
        for h in range(heads):
            hk = h // (heads // pool.hk)
            x = scale * (k[hk] @ q[s, h])
            e = np.exp(x - x.max())
            p = e / e.sum()
            ref, ref_l = p @ v[hk], x.max() + math.log(e.sum())
            ds = (pool.dim + 4) * U * (abs(scale) * np.abs(k[hk]) @ np.abs(q[s, h])).max()
            if act == "f32":
                ds += floor * np.abs(q[s, h]).max() * (abs(scale) * np.abs(k[hk]).sum(-1)).max()
            tol = (2 * ds + (2 * n + 32) * U + TERMS[act, pool.cache]) * (p @ np.abs(v[hk])) + n * floor * np.abs(v[hk]).max()
            tol += HALF[act] * np.abs(ref) + (2.0 ** -25 if act == "f16" else 0.0)
            worst = (np.abs(out[s, h] - ref) / np.maximum(tol, 1e-300)).max()
            assert worst <= 1, (s, h, n, worst)
            assert abs(lse[s, h] - ref_l) <= ds + (2 * n + 32) * U + 4 * U * abs(ref_l), (s, h, n, lse[s, h], ref_l)


@pytest.mark.parametrize("act,cache", KINDS)
@pytest.mark.parametrize("nats", [12, 15, 17, 18, 20, 22, 30])
def test_attention_beside_one_strong_position(act, cache, nats, cuda_ok):
    """One position `nats` above all others holds nothing: what comes out is the others' share alone."""
    rng = np.random.default_rng(nats)
    lens = [33, 40, 500, 3000]
    pool = Pool(lens, 16, 2, 64, cache, seed=nats)
    q = 0.5 * rng.standard_normal((len(lens), 6, 64))
    q[:, :, 0] = 8.0
    for s, n in enumerate(lens):
        k, v = 0.25 * rng.standard_normal((2, n, 64)), 8192 * rng.uniform(0.5, 1.5, (2, n, 64))
        strong = [0, 3, 7, n - 1][s]
        k[:, :, 0] = 0.0
        k[:, strong, 0] = nats  # scale q k = nats
        v[:, strong] = 0.0
        _put(pool, 0, s, k)
        _put(pool, 1, s, v)
    _compare(pool, act, 6, 0.125, q.astype(np.float32))


@pytest.mark.parametrize("act,cache", KINDS)
@pytest.mark.parametrize("dim,hk,rep", [(64, 2, 3), (64, 1, 12), (96, 2, 4), (128, 1, 16), (256, 2, 2)])
def test_attention_keeps_the_bits_of_its_weights(act, cache, dim, hk, rep, cuda_ok):
    """Values that nearly cancel: the roundings of the weights are not hidden by the output's own."""
    pool = Pool([7, 10, 24, 60], 16, hk, dim, cache, seed=dim + rep)
    q = np.random.default_rng(rep).standard_normal((4, hk * rep, dim)).astype(np.float32)
    _compare(pool, act, hk * rep, dim ** -0.5, q)


@pytest.mark.parametrize("act,cache", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_queries_with_one_large_element(act, cache, dim, cuda_ok):
    """The large element meets keys of 0, so the scores hang on elements 2^-17 of it and less."""
    rng = np.random.default_rng(dim)
    lens = [20, 300]
    pool = Pool(lens, 16, 2, dim, cache, seed=dim)
    q = 2.0 ** -17 * rng.uniform(0.25, 1.0, (2, 6, dim)) * rng.choice([-1, 1], (2, 6, dim))
    q[:, :, 5] = 1.0
    for s, n in enumerate(lens):
        k = 4096 * rng.standard_normal((2, n, dim))
        k[:, :, 5] = 0.0
        _put(pool, 0, s, k)
    _compare(pool, act, 6, 4.0, q.astype(np.float32))
