"""Page calls whose new state lies in the memory of the old one: refused, and nothing changed;
in place, array by array, as anywhere else."""
import sys

import pytest
import torch

import heteromm_b200 as hmm
from heteromm_b200._abi import HMM_ERR_INVALID, HmmError
from test_serve_pages_gpu import dev, ints, same, state

pytestmark = pytest.mark.gpu


def test_new_state_over_the_old_one(cuda):
    m = state(3, 6, 40, 8, 4, 25)
    t, r, l, k, v = dev(m, cuda)
    buf = torch.cat([t.flatten(), r, l, torch.zeros(80, dtype=torch.int32, device=cuda)])
    t = buf[:48].view(6, 8)
    r, l = buf[48:88], buf[88:94]
    before = buf.clone()
    seqs = ints([1], cuda)
    for out in ((buf[8:56].view(6, 8), r, l), (t, buf[50:90], l), (t, r, buf[87:93]), (t, r, buf[90:96])):
        with pytest.raises(HmmError) as e:
            hmm.paged_free(t, r, l, seqs, out=out)
        assert e.value.status == HMM_ERR_INVALID
        with pytest.raises(HmmError):
            hmm.paged_grow(t, r, l, ints([1] * 6, cuda), 4, out=out)
    with pytest.raises(HmmError):
        hmm.paged_grow(t, r, l, buf[100:106], 4, out=(t, r, buf[100:106]))
    assert torch.equal(buf, before)


@pytest.mark.parametrize("which", range(8))
def test_some_arrays_in_place(cuda, which):
    """Any of the three in place beside new ones."""
    m = state(3, 6, 60, 12, 4, 25)
    t, r, l, _, _ = dev(m, cuda)
    out = tuple(x if which >> i & 1 else torch.full_like(x, 77) for i, x in enumerate((t, r, l)))
    m.free([1, 4])
    got = hmm.paged_free(t, r, l, ints([1, 4], cuda), out=out)
    same(m, *got)
    m.grow([3, 0, 9, 1, 5, 2])
    out = tuple(x if which >> i & 1 else torch.full_like(x, 77) for i, x in enumerate(got))
    same(m, *hmm.paged_grow(*got, ints([3, 0, 9, 1, 5, 2], cuda), 4, out=out))


def test_lengths_that_double_in_place(cuda):
    m = state(3, 6, 120, 16, 4, 25)
    t, r, l, _, _ = dev(m, cuda)
    m.grow(m.kv.copy())
    same(m, *hmm.paged_grow(t, r, l, l, 4, out=(t, r, l)))


def test_a_refused_out_is_given_back(cuda):
    """Refusals keep no reference to the tensors of `out`."""
    m = state(3, 6, 40, 8, 4, 25)
    t, r, l, k, v = dev(m, cuda)
    bad = (torch.empty_like(t), torch.empty_like(r), l[:3])
    before = [sys.getrefcount(x) for x in bad]
    for out in (bad, list(bad), bad[:2], bad + bad[:1]):
        for _ in range(5):
            with pytest.raises(ValueError):
                hmm.paged_free(t, r, l, ints([1], cuda), out=out)
            with pytest.raises(ValueError):
                hmm.paged_grow(t, r, l, ints([1] * 6, cuda), 4, out=out)
            with pytest.raises(ValueError):
                hmm.paged_compact(t, r, k, v, out=(bad[0], bad[2]))
    del out
    assert [sys.getrefcount(x) for x in bad] == before
    good = tuple(torch.empty_like(x) for x in (t, r, l))
    before = [sys.getrefcount(x) for x in good]
    got = hmm.paged_free(t, r, l, ints([1], cuda), out=good)
    assert all(a is b for a, b in zip(got, good))
    del got
    assert [sys.getrefcount(x) for x in good] == before
