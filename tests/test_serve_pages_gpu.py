"""Page management (copy, free, fork, grow, compact) against a plain Python model of the
state: everything here is integers and bytes, so everything is equal."""
import numpy as np
import pytest
import torch

import heteromm_b200 as hmm
from heteromm_b200._abi import HMM_ERR_BOUNDS, HMM_ERR_OOM, HmmError
from heteromm_b200.paged import check_status

pytestmark = pytest.mark.gpu


class Model:
    """The rules in plain Python, on numpy arrays."""

    def __init__(self, table, refs, kv, pages, pt):
        self.table, self.refs, self.kv = table.copy(), refs.copy(), kv.copy()
        self.pages, self.pt = pages.copy(), pt

    def lowest(self):
        return int(np.nonzero(self.refs == 0)[0][0])

    def free(self, seqs):
        for s in sorted(set(int(x) for x in seqs)):
            for e in self.table[s]:
                if e >= 0:
                    self.refs[e] -= 1
            self.table[s] = -1
            self.kv[s] = 0

    def fork(self, src, dst):
        for a, b in zip(src, dst):
            full, part = divmod(int(self.kv[a]), self.pt)
            new = self.table[a].copy()
            new[full:] = -1
            for e in new[:full]:
                if e >= 0:
                    self.refs[e] += 1
            if part and self.table[a][full] >= 0:
                p = self.lowest()
                self.refs[p] = 1
                self.pages[p] = self.pages[self.table[a][full]]
                new[full] = p
            self.table[b] = new
            self.kv[b] = self.kv[a]

    def grow(self, n_new):
        for s, n in enumerate(n_new):
            if n:
                for i in range(self.kv[s] // self.pt, -(-(self.kv[s] + n) // self.pt)):
                    if self.table[s, i] < 0:
                        p = self.lowest()
                        self.refs[p] = 1
                        self.table[s, i] = p
            self.kv[s] += n

    def compact(self):
        live = int((self.refs != 0).sum())
        movers = [p for p in range(live, len(self.refs)) if self.refs[p]]
        holes = [p for p in range(live) if not self.refs[p]]
        to = np.arange(len(self.refs))
        for a, b in zip(movers, holes):
            to[a] = b
            self.pages[b] = self.pages[a]
            self.refs[b], self.refs[a] = self.refs[a], 0
        held = self.table >= 0
        self.table[held] = to[self.table[held]]
        return live


def state(seed, n_seq, n_pages, pps, pt, kv_max, empty=0, page_words=8):
    """A model of random rows over shuffled pages; the last `empty` rows hold nothing."""
    r = np.random.RandomState(seed)
    kv = r.randint(0, kv_max + 1, n_seq).astype(np.int32)
    kv[n_seq - empty:] = 0
    table = np.full((n_seq, pps), -1, np.int32)
    refs = np.zeros(n_pages, np.int32)
    perm = r.permutation(n_pages)
    at = 0
    for s in range(n_seq):
        n = -(-kv[s] // pt)
        table[s, :n] = perm[at:at + n]
        refs[perm[at:at + n]] = 1
        at += n
    return Model(table, refs, kv, r.randint(-30000, 30000, (n_pages, 1, 1, page_words)).astype(np.int16), pt)


def dev(m, cuda):
    """(table, refs, kv, k_pages, v_pages) on the device; V is K plus one."""
    k = torch.from_numpy(m.pages).to(cuda)
    return (torch.from_numpy(m.table).to(cuda), torch.from_numpy(m.refs).to(cuda),
            torch.from_numpy(m.kv).to(cuda), k, k + 1)


def ints(x, cuda):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=cuda)


def same(m, table, refs, kv=None, k=None, v=None):
    assert np.array_equal(table.cpu().numpy(), m.table)
    assert np.array_equal(refs.cpu().numpy(), m.refs)
    if kv is not None:
        assert np.array_equal(kv.cpu().numpy(), m.kv)
    if k is not None:
        assert np.array_equal(k.cpu().numpy(), m.pages)
        assert np.array_equal(v.cpu().numpy(), m.pages + 1)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n_seq,n_pages,pps,pt,kv_max", [
    (1, 4, 3, 4, 9), (7, 200, 20, 5, 70), (40, 1024, 30, 8, 150), (9, 5000, 300, 1, 290),
    (300, 9000, 40, 16, 400)])
def test_sequence_of_calls(cuda, n_seq, n_pages, pps, pt, kv_max, in_place):
    """Free, fork, grow, compact and again: as a server runs them."""
    m = state(n_seq, n_seq, n_pages, pps, pt, kv_max, empty=n_seq // 3)
    t, r, l, k, v = dev(m, cuda)
    rng = np.random.RandomState(1)

    def out(*a):
        return a if in_place else None

    for step in range(3):
        done = rng.choice(n_seq, max(1, n_seq // 5)).astype(np.int32)      # some twice
        m.free(done)
        old = (t.clone(), r.clone(), l.clone())
        t2, r2, l2 = hmm.paged_free(t, r, l, ints(done, cuda), out=out(t, r, l))
        same(m, t2, r2, l2)
        if in_place:
            assert t2 is t and r2 is r and l2 is l
        else:
            assert torch.equal(t, old[0]) and torch.equal(r, old[1]) and torch.equal(l, old[2])
        t, r, l = t2, r2, l2
        empty = [s for s in range(n_seq) if (m.table[s] < 0).all() and m.kv[s] == 0]
        held = [s for s in range(n_seq) if s not in empty]
        if held and empty:
            src = rng.choice(held, len(empty))
            m.fork(src, empty)
            t, r, l = fork_with_pt(t, r, l, ints(src, cuda), ints(empty, cuda), k, v, pt, out(t, r, l))
            same(m, t, r, l)
        n_new = [int(min(rng.randint(0, 2 * pt + 2), pps * pt - m.kv[s])) for s in range(n_seq)]
        m.grow(n_new)
        t, r, l = hmm.paged_grow(t, r, l, ints(n_new, cuda), pt, out=out(t, r, l))
        same(m, t, r, l, k, v)
        live = m.compact()
        t, r, n = hmm.paged_compact(t, r, k, v, out=out(t, r))
        assert n.item() == live
        same(m, t, r, l, k, v)


def fork_with_pt(t, r, l, src, dst, k, v, pt, out):
    """The model's pages are [n_pages, 1, 1, words]; the calls read page_tokens off the
    page arrays, so these views give them pt rows."""
    words = k.shape[-1]
    big = [torch.empty((k.shape[0], 1, pt, words), dtype=k.dtype, device=k.device) for _ in range(2)]
    for b, x in zip(big, (k, v)):
        b.copy_(x.expand(-1, -1, pt, -1))
    res = hmm.paged_fork(t, r, l, src, dst, big[0], big[1], out=out)
    for b, x in zip(big, (k, v)):
        assert torch.equal(b[:, :, :1].expand(-1, -1, pt, -1), b)   # whole pages were copied
        x.copy_(b[:, :, :1])
    return res


@pytest.mark.parametrize("shape", [(40, 2, 16, 128), (40, 1, 5, 8), (3, 40, 4, 24, 80), (64, 8, 64, 128)])
@pytest.mark.parametrize("kind", ["dense", "token-major", "interleaved"])
def test_copy_pages(cuda, shape, kind):
    if len(shape) == 5 and kind != "dense":
        pytest.skip("one layout is enough with layers")
    g = torch.Generator(device=cuda).manual_seed(3)
    if kind == "interleaved":
        both = torch.randint(-30000, 30000, (shape[0], 2, *shape[1:]), generator=g, device=cuda, dtype=torch.int16)
        k, v = both[:, 0], both[:, 1]
    else:
        k = torch.randint(-30000, 30000, shape, generator=g, device=cuda, dtype=torch.int16)
        v = torch.randint(-30000, 30000, shape, generator=g, device=cuda, dtype=torch.int16)
        if kind == "token-major":
            k, v = k.transpose(1, 2).contiguous().transpose(1, 2), v.transpose(1, 2).contiguous().transpose(1, 2)
    n_pages = shape[1] if len(shape) == 5 else shape[0]
    perm = np.random.RandomState(0).permutation(n_pages)
    src = np.array([perm[0], perm[0], -1, perm[1], perm[2], perm[3]])
    dst = np.array([perm[10], perm[11], perm[12], perm[13], -5, perm[3]])    # one pair is a page on itself
    ek, ev = k.clone(), v.clone()
    sel = (slice(None),) if len(shape) == 5 else ()
    for a, b in zip(src, dst):
        if a >= 0 and b >= 0:
            ek[sel + (int(b),)] = ek[sel + (int(a),)]
            ev[sel + (int(b),)] = ev[sel + (int(a),)]
    hmm.paged_copy_pages(k, v, ints(src, cuda), ints(dst, cuda))
    assert torch.equal(k, ek) and torch.equal(v, ev)
    hmm.paged_copy_pages(k, v, ints([], cuda), ints([], cuda))


@pytest.mark.parametrize("src,dst", [([1, 2], [5, 5]), ([1, 5], [5, 6]), ([1], [400]), ([400], [1]),
                                     ([1, 5], [2, 2])])
def test_copy_refuses(cuda, src, dst):
    k = torch.arange(400 * 8, dtype=torch.int16, device=cuda).reshape(400, 1, 1, 8)
    v = k + 1
    k0 = k.clone()
    with pytest.raises(HmmError) as e:
        hmm.paged_copy_pages(k, v, ints(src, cuda), ints(dst, cuda))
    assert e.value.status == HMM_ERR_BOUNDS
    assert torch.equal(k, k0)


def test_copy_many_pages(cuda):
    """More pages than one pass of the validation's bitmap (1.5 Mi), and a conflict behind it."""
    n = 1 << 21
    k = torch.arange(n, dtype=torch.int32, device=cuda).view(torch.int16).reshape(n, 1, 1, 2).repeat(1, 1, 1, 4)
    v = k.clone()
    src = torch.arange(0, 3000, dtype=torch.int32, device=cuda)
    dst = n - 1 - src
    e = k.clone()
    e[dst.long()] = e[src.long()]
    hmm.paged_copy_pages(k, v, src, dst)
    assert torch.equal(k, e) and torch.equal(v, e)
    dst[7] = dst[8]
    with pytest.raises(HmmError):
        hmm.paged_copy_pages(k, v, src, dst)
    assert torch.equal(k, e)


@pytest.mark.parametrize("in_place", [False, True])
def test_refusals_change_nothing(cuda, in_place):
    m = state(5, 6, 30, 10, 4, 17, empty=2)
    m.kv[0], m.table[0] = 5, -1
    m.refs[:] = 0
    m.table[:4] = -1
    m.table[0, :2] = [3, 9]
    m.table[1, :1] = [4]
    m.refs[[3, 4, 9]] = 1
    m.kv[:4] = [5, 3, 0, 0]

    def check(want, call):
        t, r, l, k, v = dev(m, cuda)
        with pytest.raises(HmmError) as e:
            call(t, r, l, k.expand(-1, -1, 4, -1).contiguous(), v.expand(-1, -1, 4, -1).contiguous(),
                 (t, r, l) if in_place else None)
        assert e.value.status == want
        same(m, t, r, l)
        # the same with a status: the new state equals the old one
        out = tuple(torch.empty_like(x) for x in (t, r, l)) if not in_place else (t, r, l)
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        call(t, r, l, k.expand(-1, -1, 4, -1).contiguous(), v.expand(-1, -1, 4, -1).contiguous(), out, status)
        same(m, *out)
        with pytest.raises(HmmError):
            check_status(status)

    def fork(src, dst):
        return lambda t, r, l, k, v, out, status=None: hmm.paged_fork(
            t, r, l, ints(src, cuda), ints(dst, cuda), k, v, out=out, status=status)

    def grow(n):
        return lambda t, r, l, k, v, out, status=None: hmm.paged_grow(
            t, r, l, ints(n, cuda), 4, out=out, status=status)

    def free(s):
        return lambda t, r, l, k, v, out, status=None: hmm.paged_free(
            t, r, l, ints(s, cuda), out=out, status=status)

    check(HMM_ERR_BOUNDS, fork([0], [1]))             # the row holds pages
    check(HMM_ERR_BOUNDS, fork([0, 1], [4, 4]))       # twice
    check(HMM_ERR_BOUNDS, fork([0], [6]))
    check(HMM_ERR_BOUNDS, fork([-1], [4]))
    check(HMM_ERR_BOUNDS, fork([0, 4], [4, 5]))       # a source that is a destination
    check(HMM_ERR_BOUNDS, grow([0, 0, 0, 0, 0, -1]))
    check(HMM_ERR_BOUNDS, grow([36, 0, 0, 0, 0, 0]))  # 41 tokens, 40 slots
    check(HMM_ERR_OOM, grow([35, 37, 40, 1, 0, 0]))   # 8 + 9 + 10 + 1 pages, 27 free
    check(HMM_ERR_BOUNDS, free([0, 6]))
    check(HMM_ERR_BOUNDS, free([-1]))


def test_grow_to_the_last_page_and_one_more(cuda):
    m = state(5, 3, 27, 12, 4, 20)
    free = int((m.refs == 0).sum())
    room = [int(-m.kv[s] % 4) for s in range(3)]
    for extra, ok in ((0, True), (1, False)):
        t, r, l, _, _ = dev(m, cuda)
        n, left = [0, 0, 0], free + extra
        for s in range(3):
            take = min(left, 12 - int(-(-m.kv[s] // 4)))
            n[s] = room[s] + 4 * take
            left -= take
        assert left == 0
        if ok:
            e = state(5, 3, 27, 12, 4, 20)
            e.grow(n)
            same(e, *hmm.paged_grow(t, r, l, ints(n, cuda), 4))
            assert (e.refs > 0).all()
        else:
            with pytest.raises(HmmError) as err:
                hmm.paged_grow(t, r, l, ints(n, cuda), 4)
            assert err.value.status == HMM_ERR_OOM


def test_free_shared_and_bad_entries(cuda):
    t = ints([[0, 1, -1], [0, 2, -1], [7, -1, 99]], cuda)
    r = ints([2, 1, 1, 0, 0, 0, 0, 0], cuda)
    l = ints([8, 8, 4], cuda)
    t2, r2, l2 = hmm.paged_free(t, r, l, ints([0], cuda))
    assert r2.tolist() == [1, 0, 1, 0, 0, 0, 0, 0] and l2.tolist() == [0, 8, 4]
    assert t2.tolist() == [[-1, -1, -1], [0, 2, -1], [7, -1, 99]]
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    t2, r2, l2 = hmm.paged_free(t, r, l, ints([2, 1], cuda), status=status)
    assert status.item() == 1 and r2.tolist() == [1, 1, 0, 0, 0, 0, 0, 0]   # no reference below 0


@pytest.mark.parametrize("live", ["none", "all", "first", "last", "shared"])
@pytest.mark.parametrize("n_pages", [1, 31, 1024, 1025, 5000])
def test_compact_ends(cuda, n_pages, live):
    n_live = {"none": 0, "all": n_pages, "first": (n_pages + 1) // 2, "last": (n_pages + 1) // 2, "shared": (n_pages + 2) // 3}[live]
    ids = np.arange(n_pages)[n_pages - n_live:] if live == "last" else np.arange(n_live) if live != "shared" else \
        np.random.RandomState(2).permutation(n_pages)[:n_live]
    refs = np.zeros(n_pages, np.int32)
    refs[ids] = 1 + np.arange(len(ids)) % 3
    table = np.full((3, n_pages + 1), -1, np.int32)
    table[0, :len(ids)] = ids
    table[2, 1:len(ids) + 1] = ids[::-1]
    pages = np.random.RandomState(3).randint(-30000, 30000, (n_pages, 2, 3, 8)).astype(np.int16)
    m = Model(table, refs, np.zeros(3, np.int32), pages, 3)
    t, r, _, k, v = dev(m, cuda)
    n = m.compact()
    t2, r2, c = hmm.paged_compact(t, r, k, v)
    assert c.item() == n == n_live
    same(m, t2, r2)
    assert np.array_equal(k.cpu().numpy()[:n], m.pages[:n])
    assert np.array_equal(v.cpu().numpy()[:n], m.pages[:n] + 1)


def test_compact_flags_a_row_that_holds_a_free_page(cuda):
    k = torch.zeros((6, 1, 1, 8), dtype=torch.int16, device=cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    t, r, n = hmm.paged_compact(ints([[5, 1, 77]], cuda), ints([0, 0, 0, 0, 0, 1], cuda), k, k.clone(), status=status)
    assert t.tolist() == [[0, 1, 77]] and r.tolist() == [1, 0, 0, 0, 0, 0] and n.item() == 1
    assert status.item() == 1


def test_layers_fork_and_compact(cuda):
    """The state's pages are moved in every layer."""
    k = torch.randint(-9, 9, (3, 8, 2, 4, 16), dtype=torch.int16, device=cuda)
    v = torch.randint(-9, 9, (3, 8, 2, 4, 16), dtype=torch.int16, device=cuda)
    t, r, l = ints([[6, 2], [-1, -1]], cuda), ints([0, 0, 1, 0, 0, 0, 1, 0], cuda), ints([7, 0], cuda)
    ek, ev = k.clone(), v.clone()
    t, r, l = hmm.paged_fork(t, r, l, ints([0], cuda), ints([1], cuda), k, v)
    ek[:, 0], ev[:, 0] = ek[:, 2], ev[:, 2]
    assert t.tolist() == [[6, 2], [6, 0]] and r.tolist() == [1, 0, 1, 0, 0, 0, 2, 0] and l.tolist() == [7, 7]
    assert torch.equal(k, ek) and torch.equal(v, ev)
    t, r, n = hmm.paged_compact(t, r, k, v)
    ek[:, 1], ev[:, 1] = ek[:, 6], ev[:, 6]
    assert t.tolist() == [[1, 2], [1, 0]] and r.tolist() == [1, 2, 1, 0, 0, 0, 0, 0] and n.item() == 3
    assert torch.equal(k[:, :3], ek[:, :3]) and torch.equal(v[:, :3], ev[:, :3])


def test_captured_in_place_step(cuda):
    """Free, fork and grow captured once and replayed: two steps of a server."""
    m = state(8, 12, 400, 20, 4, 60, empty=3)
    t, r, l, k, v = dev(m, cuda)
    k4, v4 = (x.expand(-1, -1, 4, -1).contiguous() for x in (k, v))
    done, src, dst = ints([9, 10], cuda), ints([0, 3], cuda), ints([9, 10], cuda)
    n_new = ints([3] * 12, cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)

    def step():
        hmm.paged_free(t, r, l, done, out=(t, r, l), status=status)
        hmm.paged_fork(t, r, l, src, dst, k4, v4, out=(t, r, l), status=status)
        hmm.paged_grow(t, r, l, n_new, 4, out=(t, r, l), status=status)

    def model():
        m.free([9, 10])
        m.fork([0, 3], [9, 10])
        m.grow([3] * 12)

    step()
    model()
    same(m, t, r, l)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for _ in range(3):
        g.replay()
        model()
        same(m, t, r, l)
    check_status(status)
    assert np.array_equal(k4[:, :, 0].cpu().numpy(), m.pages[:, :, 0])
