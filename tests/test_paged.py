"""Host side of the paged serving operators: the page bookkeeping, the rotation tables, and the refusals,
which come before any launch (no GPU needed)."""
import ctypes
import math
import random

import numpy as np
import pytest

from conftest import pkg


def test_pages_grow_fork_free_and_compact_like_a_list_of_tokens():
    """Random operations against plain lists: a pool of cells moved only by the returned copies holds what
    every sequence wrote."""
    P = pkg()
    rng = random.Random(7)
    for page_len in (1, 3, 16):
        t = P.PageTable(40, page_len)
        cells = np.full((40, page_len), -1)
        want, mark = {}, 0
        for _ in range(600):
            op = rng.choice(["new", "grow", "grow", "grow", "fork", "free", "compact"])
            if op == "new":
                want[t.new()] = []
            elif op == "grow" and want:
                s, n = rng.choice(list(want)), rng.randint(0, 2 * page_len + 1)
                free, pages = t.free_pages, t.pages(s)
                try:
                    src, dst = t.grow(s, n)
                except MemoryError:
                    assert (t.free_pages, t.pages(s), t.length(s)) == (free, pages, len(want[s]))
                    continue
                cells[dst] = cells[src]
                for p in range(len(want[s]), len(want[s]) + n):
                    cells[t.pages(s)[p // page_len], p % page_len] = mark
                    want[s].append(mark)
                    mark += 1
            elif op == "fork" and want:
                s = rng.choice(list(want))
                want[t.fork(s)] = list(want[s])
            elif op == "free" and len(want) > 3:
                s = rng.choice(list(want))
                t.free(s)
                del want[s]
            elif op == "compact":
                src, dst = t.compact()
                assert not set(src) & set(dst) and len(src) == len(dst)
                cells[dst] = cells[src]
                used = {p for s in want for p in t.pages(s)}
                assert used == set(range(len(used))) and t.free_pages == 40 - len(used)
            for s, ids in want.items():
                assert t.length(s) == len(ids)
                assert [cells[t.pages(s)[p // page_len], p % page_len] for p in range(len(ids))] == ids
        table = t.table(list(want), 40)
        assert table.dtype == np.int32 and all((r[len(t.pages(s)):] == -1).all() for r, s in zip(table, want))
        for s in list(want):
            t.free(s)
        assert t.free_pages == 40


def test_table_refuses_a_sequence_wider_than_asked():
    t = pkg().PageTable(4, 2)
    s = t.new()
    t.grow(s, 5)
    with pytest.raises(ValueError):
        t.table([s], 2)
    with pytest.raises(ValueError):
        t.grow(s, -1)
    with pytest.raises(ValueError):
        pkg().PageTable(0, 2)


def test_rope_tables():
    P = pkg()
    cs, sn = P.rope_tables(50, 8, 10000.0)
    assert cs.shape == sn.shape == (50, 4) and cs.dtype == np.float32
    for i in range(4):
        f = np.float32(10000.0 ** (-2 * i / 8))
        np.testing.assert_array_equal(cs[:, i], np.cos(np.arange(50) * np.float64(f)).astype(np.float32))
    # every frequency divided by 4: position 4 n turns as far as n did
    c4, s4 = P.rope_tables(50, 8, 10000.0, factor=4.0)
    np.testing.assert_allclose(c4[::4][:12], cs[:12], atol=1e-6)
    # blended: the fastest frequency stays, the slowest is divided
    cb, _ = P.rope_tables(50, 8, 10000.0, factor=4.0, low=1.0, high=4.0, original=64)
    np.testing.assert_array_equal(cb[:, 0], cs[:, 0])
    np.testing.assert_array_equal(cb[:, 3], c4[:, 3])
    assert P.rope_tables(3, 0)[0].shape == (3, 0)


A = 1 << 20  # an aligned address that nothing reads: every call below is refused before a launch


def _kv(**change):
    kv = pkg().paged_kv(A, A, "f32", 8, 16, 2, 64)
    for name, v in change.items():
        setattr(kv, name, v)
    return kv


BAD_KV = [(dict(dtype=3), -2), (dict(dtype=9), -2), (dict(k=None), -3), (dict(v=None), -3), (dict(k=A + 4), -3),
          (dict(head_dim=12), -2), (dict(head_dim=264), -2), (dict(head_dim=0), -2), (dict(n_pages=0), -3),
          (dict(page_len=0), -3), (dict(n_kv_heads=0), -3), (dict(pos_stride=63), -3), (dict(pos_stride=66), -3),
          (dict(head_stride=0), -3), (dict(page_stride=-64), -3)]


@pytest.mark.parametrize("change,code", BAD_KV)
def test_pool_descriptors_are_checked_by_every_operator(change, code):
    P = pkg()
    kv = _kv(**change)
    calls = [lambda: P.rope_append_device(kv, "f32", A, 512, 4, 4, 0, A, A, 4, 8, A, A, 100, 64, A, 256),
             lambda: P.paged_attn_device(kv, "f32", A, 256, 4, 4, A, A, 8, 0.125, A, 256, A, 1 << 30),
             lambda: P.copy_pages_device(kv, [0], [1])]
    for call in calls:
        with pytest.raises(P.MllmError) as e:
            call()
        assert e.value.code == code and "paged cache" in str(e.value)


def _rope(**change):
    a = dict(kv=_kv(), dtype="f32", qkv_ptr=A, row_stride=512, n_tok=4, n_heads=4, seq_ptr=0, pos_ptr=A, table_ptr=A, n_seq=4,
             table_stride=8, cos_ptr=A, sin_ptr=A, n_pos=100, rope_dim=64, q_ptr=A, q_stride=256)
    return pkg().rope_append_device(**(a | change))


@pytest.mark.parametrize("change,code", [
    (dict(dtype="f16"), -2), (dict(dtype="q8"), -2), (dict(n_tok=-1), -3), (dict(n_heads=0), -3), (dict(n_seq=0), -3),
    (dict(table_stride=0), -3), (dict(qkv_ptr=0), -3), (dict(pos_ptr=0), -3), (dict(table_ptr=0), -3), (dict(q_ptr=0), -3),
    (dict(q_gain_ptr=A), -3), (dict(k_gain_ptr=A), -3), (dict(rope_dim=63), -3), (dict(rope_dim=66), -3), (dict(rope_dim=-2), -3),
    (dict(cos_ptr=0), -3), (dict(n_pos=0), -3), (dict(row_stride=508), -3), (dict(q_stride=252), -3), (dict(row_stride=514), -3),
    (dict(q_ptr=A + 8), -3)])
def test_rope_append_refuses(change, code):
    with pytest.raises(pkg().MllmError) as e:
        _rope(**change)
    assert e.value.code == code and "mllm_rope_append" in str(e.value)


def _attn(**change):
    a = dict(kv=_kv(), dtype="f32", q_ptr=A, q_stride=256, n_seq=4, n_heads=4, len_ptr=A, table_ptr=A, table_stride=8, scale=0.125,
             out_ptr=A, out_stride=256, ws_ptr=A, ws_bytes=1 << 40)
    return pkg().paged_attn_device(**(a | change))


@pytest.mark.parametrize("change,code", [
    (dict(dtype="bf16"), -2), (dict(dtype="q4"), -2), (dict(n_seq=-1), -3), (dict(n_seq=65536), -3), (dict(n_heads=0), -3),
    (dict(n_heads=5), -2), (dict(n_heads=130, q_stride=8320, out_stride=8320), -2), (dict(q_ptr=0), -3), (dict(len_ptr=0), -3),
    (dict(table_ptr=0), -3), (dict(out_ptr=0), -3), (dict(table_stride=0), -3), (dict(q_stride=252), -3), (dict(out_stride=258), -3),
    (dict(out_ptr=A + 4), -3), (dict(ws_ptr=0), -3), (dict(ws_ptr=A + 8), -3), (dict(ws_bytes=0), -3)])
def test_paged_attn_refuses(change, code):
    with pytest.raises(pkg().MllmError) as e:
        _attn(**change)
    assert e.value.code == code and "mllm_paged_attn" in str(e.value)


def test_paged_attn_workspace_needs_no_device():
    P = pkg()
    assert P.paged_attn_workspace(1, 4, 64) > 0
    assert P.paged_attn_workspace(300, 4, 64) >= P.paged_attn_workspace(2, 4, 64)
    for bad in ((0, 4, 64), (1, 0, 64), (1, 4, 0), (1, 4, 264)):
        assert P.paged_attn_workspace(*bad) == 0


@pytest.mark.parametrize("src,dst,layers,stride,code", [
    ([0], [8], 1, 0, -3), ([-1], [0], 1, 0, -3), ([0, 1], [2, 2], 1, 0, -3), ([0, 1], [1, 2], 1, 0, -3), ([3], [3], 1, 0, -3),
    ([0], [1], 0, 0, -3), ([0], [1], 2, 100, -3), ([0], [1], 2, 16 * 2 * 64 + 1, -3), ([0], [1], 70000, 1 << 20, -3)])
def test_copy_pages_refuses(src, dst, layers, stride, code):
    with pytest.raises(pkg().MllmError) as e:
        pkg().copy_pages_device(_kv(), src, dst, layers, stride)
    assert e.value.code == code and "mllm_copy_pages" in str(e.value)


def test_copy_pages_refuses_gaps_and_uneven_lists():
    P = pkg()
    with pytest.raises(P.MllmError) as e:
        P.copy_pages_device(_kv(pos_stride=68), [0], [1])
    assert e.value.code == -2
    with pytest.raises(ValueError):
        P.copy_pages_device(_kv(), [0, 1], [2])


def _sample(**change):
    a = dict(dtype="f32", logits_ptr=A, row_stride=100, rows=2, vocab=100, u_ptr=A, id_ptr=A)
    return pkg().sample_device(**(a | change))


@pytest.mark.parametrize("change,code", [
    (dict(dtype="q8"), -2), (dict(rows=-1), -3), (dict(vocab=0), -3), (dict(row_stride=99), -3), (dict(u_ptr=0), -3), (dict(id_ptr=0), -3),
    (dict(logits_ptr=0), -3), (dict(logits_ptr=A + 2), -3), (dict(vocab=524289, row_stride=524289), -2)])
def test_sample_refuses(change, code):
    with pytest.raises(pkg().MllmError) as e:
        _sample(**change)
    assert e.value.code == code and "mllm_sample" in str(e.value)


def test_empty_calls_are_fine_without_a_device():
    """No rows: nothing is launched."""
    P = pkg()
    _rope(n_tok=0)
    _attn(n_seq=0)
    _sample(rows=0)
    P.copy_pages_device(_kv(), [], [])


def test_null_descriptor():
    P = pkg()
    L = P.load_library()
    assert L.mllm_copy_pages(None, 1, 0, None, None, 0, None) == -3
    assert b"null descriptor" in L.mllm_last_error(None)
    assert L.mllm_copy_pages(ctypes.byref(_kv()), 1, 0, None, None, 1, None) == -3
