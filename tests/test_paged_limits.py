"""Host side of the paged serving operators: workspaces, page lists and sizes at their limits (no GPU needed)."""
import subprocess
import sys

import numpy as np
import pytest

from conftest import ROOT, pkg


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


LIMITED = """
import ctypes, importlib, resource, sys
sys.path.insert(0, %r)
P = importlib.import_module("microllm-lab_b200")
L = P.load_library()
kv = P.paged_kv(1 << 20, 1 << 20, "f32", 2**31 - 1, 1, 1, 8)
now = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (now + (256 << 20), now + (256 << 20)))
for n in (1, 30, 64):  # every destination but the last is another page; the last is written twice, or read as well
    src, dst = (ctypes.c_int * n)(*range(n)), (ctypes.c_int * n)(*range(1000, 1000 + n))
    for bad in (0, 1000)[: n]:
        dst[n - 1] = bad
        rc = L.mllm_copy_pages(ctypes.byref(kv), 1, 0, ctypes.addressof(src), ctypes.addressof(dst), n, None)
        assert rc == -3 and b"written twice" in L.mllm_last_error(None), (n, bad, rc, L.mllm_last_error(None))
"""


def test_copy_pages_of_a_few_pages_does_not_depend_on_the_pool():
    """A pool of 2^31 - 1 pages: the check of one page's copy takes no memory for all of them."""
    r = subprocess.run([sys.executable, "-c", LIMITED % ROOT], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("n", [2, 64, 65, 300])
def test_copy_pages_finds_a_conflict_wherever_it_is(n):
    """A destination that is also the first, the last or a middle source or destination, in short and long lists."""
    kv = pkg().paged_kv(A, A, "f32", 4096, 16, 2, 64)
    src, dst = [(7 * i) % 2048 for i in range(n)], [2048 + (5 * i) % 2048 for i in range(n)]
    for at in (0, n // 2, n - 1):
        for other in (0, n // 2, n - 1):
            bad = list(dst)
            bad[at] = src[other]
            _refused(-3, kv, src, bad)
            if at != other:
                bad[at] = dst[other]
                _refused(-3, kv, src, bad)
    for outside in (-1, 4096):
        _refused(-3, kv, src[:-1] + [outside], dst)
        _refused(-3, kv, src, [outside] + dst[1:])


@pytest.mark.parametrize("heads,page_len,dim", [(2**31 - 1, 2**31 - 1, 8), (2**31 - 1, 2**31 - 1, 256), (1 << 30, 1 << 30, 16),
                                                (1, 2**31 - 1, 8), (1 << 20, 1 << 8, 8)])
def test_copy_pages_refuses_pages_whose_size_passes_64_bits(heads, page_len, dim):
    kv = pkg().paged_kv(A, A, "f32", 8, page_len, heads, dim, (1 << 62, page_len * dim, dim))
    _refused(-2, kv, [0], [1])


@pytest.mark.parametrize("heads", [2**31 - 2, 2**30, 2**30 - 1])
def test_rope_append_refuses_rows_of_too_many_heads(heads):
    """A row's heads are counted, two rounds ahead, in 31 bits."""
    P = pkg()
    kv = P.paged_kv(A, A, "f32", 8, 16, 1, 8)
    with pytest.raises(P.MllmError) as e:
        P.rope_append_device(kv, "f32", A, 1 << 40, 1, heads, 0, A, A, 1, 8, A, A, 100, 8, A, 1 << 40)
    assert e.value.code == -3 and "2^30 heads" in str(e.value)


def test_paged_attn_refuses_rows_of_too_many_elements():
    """A row's elements are counted in 31 bits where a sequence is empty."""
    P = pkg()
    kv = P.paged_kv(A, A, "f32", 8, 16, 1 << 25, 8)
    for heads in (1 << 28, 1 << 30):
        with pytest.raises(P.MllmError) as e:
            P.paged_attn_device(kv, "f32", A, 1 << 40, 4, heads, A, A, 8, 0.125, A, 1 << 40, A, 1 << 40)
        assert e.value.code == -2 and "2^30 elements" in str(e.value)


@pytest.mark.parametrize("ids", [np.array([1 << 32]), np.array([-(1 << 32)]), np.array([(1 << 32) + 1]), [2.5], np.array([1.0]), ["1"], [None],
                                 np.array([1 << 63], np.uint64), np.array([True])])
def test_copy_pages_takes_page_ids_as_they_are(ids):
    """Ids that are no 32-bit numbers are refused, not rounded or cut to some other page's."""
    for src, dst in ((ids, [3]), ([3], ids)):
        with pytest.raises((ValueError, TypeError, OverflowError)):
            pkg().copy_pages_device(pkg().paged_kv(A, A, "f32", 8, 16, 2, 64), src, dst)


def test_copy_pages_takes_ids_of_any_whole_type():
    """A conflict that the library finds shows that the ids came through."""
    kv = pkg().paged_kv(A, A, "f32", 8, 16, 2, 64)
    for ids in ([5], (5,), np.array([5]), np.array([5], np.uint8), np.array([5], np.uint64), np.array([0, 5, 0, 6])[1::2]):
        _refused(-3, kv, ids, ids)
    pkg().copy_pages_device(kv, [], [])


def test_sequences_grow_together_or_not_at_all():
    P = pkg()
    t = P.PageTable(8, 4)
    a = t.new()
    t.grow(a, 6)  # two pages, the second half full
    b, c = t.fork(a), t.fork(a)
    assert t.grow_all([a, b, c], 0) == ([], []) and t.free_pages == 6
    last = t.pages(a)[-1]
    src, dst = t.grow_all([a, b, c])  # two copies: the third may write the shared page itself
    assert src == [last, last] and t.pages(c)[-1] == last and [t.pages(s)[-1] for s in (a, b)] == dst and t.free_pages == 4
    assert [t.length(s) for s in (a, b, c)] == [7, 7, 7]
    assert t.grow_all([a, b, c]) == ([], [])  # eight positions in two pages each
    d = t.new()
    t.grow(d, 7)  # two of the four left
    before = [(t.length(s), t.pages(s)) for s in (a, b, c, d)]
    with pytest.raises(MemoryError):
        t.grow_all([d, a, b, c])  # one position is there in d's page, three pages are wanted, two are free
    with pytest.raises(ValueError):
        t.grow_all([d, d])
    with pytest.raises(ValueError):
        t.grow_all([d], -1)
    with pytest.raises(KeyError):
        t.grow_all([d, 99])
    assert [(t.length(s), t.pages(s)) for s in (a, b, c, d)] == before and t.free_pages == 2
    assert t.grow_all([d, a, b]) == ([], []) and t.free_pages == 0
    assert t.grow_all([]) == ([], [])


def test_sequences_that_share_a_page_outside_the_list_copy_it():
    P = pkg()
    t = P.PageTable(5, 4)
    a = t.new()
    t.grow(a, 2)
    b, c = t.fork(a), t.fork(a)
    src, dst = t.grow_all([b, c])  # a keeps the page
    assert src == [t.pages(a)[0]] * 2 and dst == [t.pages(b)[0], t.pages(c)[0]] and len({*dst, src[0]}) == 3
