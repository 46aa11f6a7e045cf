"""The page operations on the GPU against the host model (tests/_paged.py),
whole states and contents compared, and a run of them with the paged append,
step and decode as a server uses them."""
import numpy as np
import pytest

import b200attn
import oracle
from _gpu import Graph, bits, dev, host
from _paged import Pages, assert_within, attend64, rows_of
from _util import MAX_ABS, REL_L2, max_abs, rel_l2, seeded_f16

pytestmark = pytest.mark.gpu


def _sync():
    import torch
    torch.cuda.synchronize()


def _error_word():
    _sync()
    w = b200attn.lib().b2_device_error_word()
    assert b200attn.lib().b2_clear_device_error_word() == 0
    return w


_kept = []   # arguments of calls on other streams live until the end


def _i32(x):
    _kept.append(dev(np.asarray(x, np.int32)))
    return _kept[-1]


class Device:
    """The model's state on the device, and the operations' calls on it."""

    def __init__(self, m, by_page=False):
        import torch
        self.m = m
        planes, pages, elems = m.pool.shape
        self.by_page = by_page
        if by_page:       # a page's planes together
            self.pool = dev(np.ascontiguousarray(m.pool.transpose(1, 0, 2)))
            strides = elems, planes * elems
        else:
            self.pool = dev(m.pool)
            strides = 0, 0
        self.where = (self.pool, planes, strides[0], pages, strides[1], elems)
        self.table, self.len, self.ref = dev(m.table), dev(m.len), dev(m.ref)
        self.status = torch.full((2,), -9, dtype=torch.int32, device="cuda")
        n = b200attn.kv_pages_workspace_bytes(pages)
        self.ws = (torch.zeros(n, dtype=torch.uint8, device="cuda"), n)
        self.rows, self.stride = m.table.shape
        self.stream = None

    def seqs(self):
        return self.table, self.stride, self.rows, self.m.ps, self.where[3], self.len, self.ref

    def truncate(self, seqs, new=None):
        b200attn.launch_kv_pages_truncate(*self.seqs(), _i32(seqs), None if new is None else _i32(new), len(seqs),
                                          self.status, *self.ws, stream=self.stream)
        return self.done()[0]

    def fork(self, parents, children, n=None):
        b200attn.launch_kv_pages_fork(*self.seqs(), _i32(parents), _i32(children), None if n is None else _i32(n),
                                      len(parents), self.status, *self.ws, stream=self.stream)
        return self.done()[0]

    def extend(self, seqs, take):
        import torch
        first = torch.full((len(seqs) + 1,), -77, dtype=torch.int32, device="cuda")
        s = self.seqs()
        b200attn.launch_kv_pages_extend(*self.where, *s[:4], *s[5:], _i32(seqs), _i32(take), len(seqs), first,
                                        self.status, *self.ws, stream=self.stream)
        st, need = self.done()
        first = host(first)
        assert first[-1] == -77
        return st, need, first[:-1]

    def compact(self, apart=False):
        import torch
        table = torch.empty_like(self.table) if apart else self.table
        ref = torch.full_like(self.ref, -3) if apart else self.ref
        b200attn.launch_kv_pages_compact(*self.where, self.table, table, self.stride, self.rows, self.m.ps, self.len,
                                         self.ref, ref, self.status, *self.ws, stream=self.stream)
        self.table, self.ref = table, ref
        st, n = self.done()
        assert st == b200attn.PAGES_OK
        return n

    def done(self):
        _sync()
        return host(self.status).tolist()

    def contents(self):
        x = host(self.pool)
        return x.transpose(1, 0, 2) if self.by_page else x

    def same(self):
        np.testing.assert_array_equal(host(self.len), self.m.len)
        np.testing.assert_array_equal(host(self.ref), self.m.ref)
        np.testing.assert_array_equal(host(self.table), self.m.table)
        np.testing.assert_array_equal(bits(self.contents()), bits(self.m.pool))


def _model(planes, pages, ps, row, rows, stride, seed=1):
    return Pages(seeded_f16((planes, pages, ps * row), seed), rows, stride, ps)


@pytest.mark.parametrize("pages,ps,row,by_page", [(40, 4, 8, False), (300, 16, 128, True), (9000, 1, 8, False)])
def test_random_operations(cuda, pages, ps, row, by_page):
    """Long random sequences of operations, refused ones among them: the whole state after each."""
    rows, stride = 12, min(pages, 40)
    m = _model(3, pages, ps, row, rows, stride)
    d = Device(m, by_page)
    rng = np.random.default_rng(2)
    seen = set()
    for _ in range(120):
        op = rng.choice(["extend", "extend", "truncate", "fork", "fork", "compact"])
        n = int(rng.integers(1, 6))
        seqs = rng.permutation(rows)[:n].tolist()
        if rng.random() < 0.15:
            seqs.append(int(rng.choice([-1, -3, seqs[0], rows])))
        if op == "extend":
            take = rng.integers(0, 3 * ps + 3, len(seqs)).tolist()
            want = m.extend(seqs, take)
            got = d.extend(seqs, take)
            assert got[0] == want[0] and (want[1] is None or got[1] == want[1])
            np.testing.assert_array_equal(got[2], want[2])
            seen.add((op, want[0]))
        elif op == "truncate":
            whole = rng.random() < 0.3
            new = None if whole else [int(rng.integers(0, (m.len[s] if 0 <= s < rows else 5) + 1)) for s in seqs]
            if new and rng.random() < 0.1:
                new[0] += 10000
            want = m.truncate(seqs, new)
            assert d.truncate(seqs, new) == want
            seen.add((op, want))
        elif op == "fork":
            pair = rng.permutation(rows)
            empty = [s for s in pair.tolist() if m.len[s] == 0][:2]
            if not empty:
                continue
            par = [int(rng.integers(0, rows)) for _ in empty]
            ln = None if rng.random() < 0.4 else [int(rng.integers(0, m.len[p] + 2)) for p in par]
            want = m.fork(par, empty, ln)
            assert d.fork(par, empty, ln) == want
            seen.add((op, want))
        else:
            assert d.compact(apart=bool(rng.integers(2))) == m.compact()
        d.same()
    assert {("extend", m.OK), ("truncate", m.OK), ("fork", m.OK), ("truncate", m.BAD), ("fork", m.BAD)} <= seen
    assert _error_word() == 0


def test_too_few_pages_changes_nothing(cuda):
    m = _model(2, 10, 4, 8, 4, 10)
    d = Device(m)
    assert d.extend([0, 1], [9, 20])[0] == m.extend([0, 1], [9, 20])[0] == m.OK
    d.same()                                             # 8 pages of 10
    st, need, first = d.extend([2, 3], [4, 9])
    assert (st, need) == (m.SHORT, 4) and np.all(first == -1)
    d.same()
    assert d.extend([2, 3], [4, 4])[0] == m.extend([2, 3], [4, 4])[0] == m.OK
    d.same()
    assert d.extend([0], [4])[:2] == (m.SHORT, 1)
    d.same()


def test_all_holders_of_a_shared_page(cuda):
    """Of the holders that extend together the first keeps the page; while another holds it, all copy."""
    m = _model(2, 30, 8, 8, 6, 4)
    d = Device(m)
    for s in (m, d):
        s.extend([0], [13])
        s.fork([0, 0, 0], [1, 2, 3])
    d.same()
    assert d.extend([3, 1], [1, 2])[:2] == tuple(m.extend([3, 1], [1, 2])[:2]) == (0, 2)
    d.same()
    assert d.extend([2, 0], [0, 1])[:2] == tuple(m.extend([2, 0], [0, 1])[:2]) == (0, 1)   # nothing for 2: it still holds it
    d.same()
    assert d.extend([2], [1])[:2] == tuple(m.extend([2], [1])[:2]) == (0, 0)               # alone now
    d.same()
    for s in (m, d):
        s.fork([1, 1], [4, 5], [12, 9])
    assert d.extend([5, 4, 1], [1, 1, 1])[:2] == tuple(m.extend([5, 4, 1], [1, 1, 1])[:2]) == (0, 2)
    d.same()
    m.check()


def test_a_thousand_items(cuda):
    """The most items a call takes, all sharing pages, and long rows."""
    rows = 1024
    m = _model(1, 6000, 2, 8, rows + 1, 700)
    d = Device(m)
    assert d.extend([rows], [1001])[0] == m.extend([rows], [1001])[0] == m.OK
    kids = list(range(rows))
    cut = [1 + (i * 37) % 1001 for i in kids]
    assert d.fork([rows] * rows, kids, cut) == m.fork([rows] * rows, kids, cut) == m.OK
    d.same()
    take = [1 + i % 5 for i in kids]
    got, want = d.extend(kids, take), m.extend(kids, take)
    assert got[:2] == want[:2] and want[0] == m.OK
    np.testing.assert_array_equal(got[2], want[2])
    d.same()
    half = kids[::2]
    assert d.truncate(half) == m.truncate(half) == m.OK
    assert d.compact() == m.compact()
    d.same()
    m.check()


def test_more_pages_at_once_than_fit_on_chip(cuda):
    """One call that takes, and one that gives back, many thousand pages; copies among them."""
    m = _model(1, 20000, 2, 8, 5, 9000)
    d = Device(m)
    for s in (m, d):
        s.extend([4], [3])
        s.fork([4, 4], [1, 3])
    for seqs, take in (([0, 1, 2], [5, 14001, 1]), ([3, 4, 2], [9999, 1, 0])):
        got, want = d.extend(seqs, take), m.extend(seqs, take)
        assert got[:2] == want[:2] and want[0] == m.OK
        d.same()
    assert d.truncate([1, 3], [7, 0]) == m.truncate([1, 3], [7, 0]) == m.OK
    d.same()
    assert d.fork([1, 1], [3, 2]) == m.fork([1, 1], [3, 2])
    d.same()
    assert d.compact() == m.compact()
    d.same()
    m.check()


def test_huge_requests_are_short_not_wrapped(cuda):
    m = _model(1, 16, 1, 8, 5, 1 << 20)
    d = Device(m)
    for take in ([1 << 20] * 4, [1 << 20, 3, 3, 3], [(1 << 20) + 1, 0, 0, 0], [2**31 - 1] * 4):
        assert d.extend([0, 1, 2, 3], take)[0] == m.extend([0, 1, 2, 3], take)[0] != m.OK
        d.same()


@pytest.mark.parametrize("planes,pages,elems,by_page", [(72, 60, 8192, False), (5, 33, 40, False), (2, 100, 2048, True),
                                                        (1, 50, 8, False)])
def test_copy(cuda, planes, pages, elems, by_page):
    m = Pages(seeded_f16((planes, pages, elems), 3), 1, 1, 1)
    d = Device(m, by_page)
    rng = np.random.default_rng(4)
    perm = rng.permutation(pages)
    n = pages // 2
    b200attn.launch_kv_pages_copy(*d.where, _i32(perm[:n]), _i32(perm[n:2 * n]), n)
    _sync()
    m.pool[:, perm[n:2 * n]] = m.pool[:, perm[:n]]
    d.same()
    assert _error_word() == 0


def test_copy_of_the_same_page_twice_and_of_clashing_ones(cuda):
    m = Pages(seeded_f16((3, 20, 4096), 5), 1, 1, 1)
    d = Device(m)
    src, dst = [1, 2, 3, 4, 9, 3], [10, 10, 11, 4, 12, 10]     # page 10 three times: the last counts; 4 onto itself
    b200attn.launch_kv_pages_copy(*d.where, _i32(src), _i32(dst), 6)
    assert _error_word() == 0
    for s, t in zip(src, dst):
        m.pool[:, t] = m.pool[:, s]
    d.same()
    # 5 -> 6 while 6 -> 7: the copy onto a source is left out; so are pages the pool has not
    b200attn.launch_kv_pages_copy(*d.where, _i32([5, 6, 20, 8, -1]), _i32([6, 7, 13, 2**31 - 1, 14]), 5)
    assert _error_word() == 4
    m.pool[:, 7] = m.pool[:, 6]
    d.same()


def test_copies_that_are_none_hide_no_other(cuda):
    """A page copied onto itself, or from outside the pool, after a copy to it: that copy stands."""
    m = Pages(seeded_f16((2, 20, 2048), 6), 1, 1, 1)
    d = Device(m)
    b200attn.launch_kv_pages_copy(*d.where, _i32([1, 10]), _i32([10, 10]), 2)
    assert _error_word() == 0
    m.pool[:, 10] = m.pool[:, 1]
    d.same()
    b200attn.launch_kv_pages_copy(*d.where, _i32([2, 20, 3, -1, 4]), _i32([11, 11, 12, 12, 12]), 5)
    assert _error_word() == 4
    m.pool[:, 11] = m.pool[:, 2]
    m.pool[:, 12] = m.pool[:, 4]
    d.same()


def test_tables_that_lie_are_flagged_not_followed(cuda):
    """Bad page numbers and counts that are already 0: the error bit, no access outside."""
    m = _model(1, 12, 4, 8, 4, 6)
    d = Device(m)
    d.extend([0, 1], [16, 8])
    d.table[0, 1] = 12
    d.table[0, 2] = -7
    assert d.truncate([0], [2]) == m.OK and _error_word() == 4
    d.ref.zero_()
    assert d.truncate([1]) == m.OK and _error_word() == 4
    assert np.all(host(d.ref) == 0)
    d = Device(m)
    d.extend([0], [10])
    d.table[0, 0], d.table[0, 2] = 99, 99
    assert d.fork([0], [1]) == m.OK and _error_word() == 4
    assert d.extend([1], [1])[0] == m.BAD                # its last page is none
    d.compact()
    assert _error_word() == 4


def test_a_last_page_without_a_reference_is_not_extended(cuda):
    m = _model(1, 12, 4, 8, 4, 6)
    d = Device(m)
    d.extend([0, 1], [6, 4])
    g = int(host(d.table)[0, 1])
    d.ref[g] = 0
    before = host(d.table).copy(), host(d.len).copy(), host(d.ref).copy()
    assert d.extend([1, 0], [3, 1])[0] == m.BAD
    for got, want in zip((d.table, d.len, d.ref), before):
        np.testing.assert_array_equal(host(got), want)


def test_the_pages_taken_do_not_wrap(cuda):
    """1024 sequences that take 2^21 pages each: 2^31 of them."""
    import torch
    n = 1 << 21
    m = Pages(np.zeros((1, 1, 8), np.float16), 1, 1, 1)
    d = Device(m)
    table = torch.empty((1024, n), dtype=torch.int32, device="cuda")
    length, ref = (torch.zeros(k, dtype=torch.int32, device="cuda") for k in (1024, n))
    pool = torch.zeros(n * 8, dtype=torch.float16, device="cuda")
    size = b200attn.kv_pages_workspace_bytes(n)
    ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
    b200attn.launch_kv_pages_extend(pool, 1, 0, n, 0, 8, table, n, 1024, 1, length, ref, _i32(range(1024)),
                                    _i32([n] * 1024), 1024, None, d.status, ws, size)
    _sync()
    assert host(d.status).tolist() == [m.SHORT, 2 ** 31 - 1]
    assert not length.any() and not ref.any()


def test_the_pages_taken_are_counted_when_they_are_too_many(cuda):
    """Whatever one item asks for, up to a table's width: the count is that of the call."""
    m = _model(1, 16, 1, 8, 5, 1 << 20)
    d = Device(m)
    for seqs, take in (([0], [17]), ([0], [16]), ([1], [1]), ([0, 1, 2], [1, 17, 40]), ([3, 1], [1 << 20, 0]),
                       ([4, 3, 2, 1], [1 << 20, 1 << 20, (1 << 20) - 5, 3])):
        got, want = d.extend(seqs, take), m.extend(seqs, take)
        assert got[:2] == want[:2]
        np.testing.assert_array_equal(got[2], want[2])
        d.same()
    # a copied last page counts too
    m = _model(1, 3, 4, 8, 3, 8)
    d = Device(m)
    for s in (m, d):
        s.extend([0], [6])
        s.fork([0], [1])
    assert d.extend([1], [20])[:2] == m.extend([1], [20])[:2] == (m.SHORT, 6)
    d.same()


def test_copies_that_other_ctas_gave_up_are_made(cuda):
    """The workspace as CTAs leave it whose wait for the plan ran out: they are counted, beside the CTAs
    that are done, and a word that stands too early has the others copy nothing. The pages are copied
    all the same, and the workspace is as new."""
    import torch
    m = _model(72, 80, 4, 2048, 20, 4)
    d = Device(m)
    for s in (m, d):
        s.extend([0], [10])
        s.fork([0] * 19, list(range(1, 20)))
    head = d.ws[0][:16].view(torch.int32)        # finished, word, moves, unused
    head.copy_(_i32([1 << 16, 1, 0, 0]))
    _sync()
    kids = list(range(1, 20))
    assert d.extend(kids, [1] * 19)[:2] == m.extend(kids, [1] * 19)[:2] == (m.OK, 19)
    d.same()
    assert host(head).tolist() == [0] * 4 and _error_word() == 0
    for s in (m, d):
        s.truncate(kids, [9] * 19)
        s.truncate([0])
        s.fork([1], [0])
    assert d.extend([0], [1])[:2] == m.extend([0], [1])[:2]
    d.same()
    assert host(head).tolist() == [0] * 4


def test_on_another_stream_and_captured(cuda):
    """A scheduler's step (drop, fork, extend) captured once, replayed with other items in the same buffers."""
    import torch
    m = _model(4, 64, 8, 16, 8, 6)
    d = Device(m)
    for s in (m, d):
        s.extend([0, 1], [21, 30])
    drop, new, par, kid, ext, take = (torch.zeros(4, dtype=torch.int32, device="cuda") for _ in range(6))
    first = torch.zeros(4, dtype=torch.int32, device="cuda")
    g = Graph()
    s = d.seqs()
    with g:
        b200attn.launch_kv_pages_truncate(*s, drop, new, 4, d.status, *d.ws, stream=g.stream)
        b200attn.launch_kv_pages_fork(*s, par, kid, None, 4, d.status, *d.ws, stream=g.stream)
        b200attn.launch_kv_pages_extend(*d.where, *s[:4], *s[5:], ext, take, 4, first, d.status, *d.ws, stream=g.stream)
    rounds = [([-1] * 4, [0] * 4, [0, 1, -1, 0], [2, 3, 4, 5], [0, 2, 5, 3], [1, 2, 3, 1]),
              ([2, 5, -1, 0], [21, 0, 0, 9], [3, 0, 3, -1], [5, 6, 7, 1], [3, 5, 6, 7], [9, 1, 1, 1]),
              ([7, 6, 5, 3], [0, 0, 0, 2], [2, 2, 2, 2], [5, 6, 7, -1], [2, 5, 6, 7], [4, 4, 4, 4])]
    for r in rounds:
        for buf, x in zip((drop, new, par, kid, ext, take), r):
            buf.copy_(_i32(x))
        _sync()
        g.launch()
        assert m.truncate(r[0], r[1]) == m.OK and m.fork(r[2], r[3]) == m.OK
        st, _, want = m.extend(r[4], r[5])
        assert st == m.OK and host(d.status)[0] == m.OK
        np.testing.assert_array_equal(host(first), want)
        d.same()
        m.check()
    g.close()
    assert _error_word() == 0


def test_two_streams_at_once(cuda):
    """Operations on two caches on two streams, interleaved."""
    import torch
    made = []
    for k in range(2):
        m = _model(6, 80, 8, 128, 10, 10, seed=90 + k)
        d = Device(m)
        d.stream = torch.cuda.Stream()
        made.append((m, d))
    torch.cuda.synchronize()
    for r in range(12):
        for k, (m, d) in enumerate(made):
            seqs = [(r + i + k) % 10 for i in range(3)]
            for s in (m, d):
                s.truncate(seqs[2:])
                s.fork(seqs[:1], seqs[2:])
            d.done = lambda: [0, 0]                      # no waiting between the calls
            d.extend(seqs, [3, 5, 2])
            m.extend(seqs, [3, 5, 2])
            del d.done
    torch.cuda.synchronize()
    for m, d in made:
        d.same()
        m.check()
    assert _error_word() == 0


def test_two_streams_without_waiting(cuda):
    """Rounds of truncate, fork and extend of two caches, queued on two streams with nothing between
    them that waits: whole states and every call's positions against the model."""
    import torch
    rounds, made = 20, []
    for k in range(2):
        m = _model(36, 400, 8, 512, 40, 10, seed=93 + k)
        d = Device(m)
        d.stream = torch.cuda.Stream()
        plan = []
        for r in range(rounds):
            seqs = [(3 * r + i + k) % 40 for i in range(30)]
            take = [1 + (r + i) % 5 for i in range(30)]
            drop, kids = seqs[15:], seqs[15:]
            parents = [seqs[i % 15] for i in range(15)]
            first = torch.full((30,), -77, dtype=torch.int32, device="cuda")
            plan.append(([_i32(x) for x in (drop, parents, kids, seqs, take)], first, (drop, parents, kids, seqs, take)))
        made.append((m, d, plan))
    _sync()
    for r in range(rounds):
        for m, d, plan in made:
            (drop, parents, kids, seqs, take), first, _ = plan[r]
            s = d.seqs()
            b200attn.launch_kv_pages_truncate(*s, drop, None, 15, d.status, *d.ws, stream=d.stream)
            b200attn.launch_kv_pages_fork(*s, parents, kids, None, 15, d.status, *d.ws, stream=d.stream)
            b200attn.launch_kv_pages_extend(*d.where, *s[:4], *s[5:], seqs, take, 30, first, d.status, *d.ws,
                                            stream=d.stream)
    _sync()
    copies = 0
    for m, d, plan in made:
        for _, first, (drop, parents, kids, seqs, take) in plan:
            assert m.truncate(drop) == m.fork(parents, kids) == m.OK
            before = m.ref.copy()
            st, _, want = m.extend(seqs, take)
            assert st == m.OK
            copies += int((m.ref < before).sum())     # pages that lost a holder to its copy
            np.testing.assert_array_equal(host(first), want)
        d.same()
        m.check()
    assert copies > 100 and _error_word() == 0


def test_a_served_batch(cuda):
    """Prompts appended, forked into beams, decoded a few steps over two layers through pages,
    rolled back, compacted and decoded on: each output against 64-bit attention of the rows
    that the sequence has by then."""
    import torch
    layers, H, KVH, d, ps, pages, rows, stride = 2, 16, 4, 128, 16, 60, 6, 12
    kv, wide, theta, cap = KVH * d, (H + 2 * KVH) * d, 5.0e6, 12 * 16
    m = Pages(np.zeros((2 * layers, pages, ps * kv), np.float16), rows, stride, ps)
    c = Device(m)
    planes = [c.pool[i].view(pages, ps, kv) for i in range(2 * layers)]
    cos, sin = b200attn.rope_tables_host(cap, d, theta)
    dcos, dsin = dev(cos), dev(sin)
    text = [[] for _ in range(rows)]      # rows a sequence holds: per layer (k, v)
    serial = [70]

    def fresh(n):
        serial[0] += 1
        return seeded_f16((layers, n, wide), serial[0])

    def row(x, layer, t, pos):
        q, k = x[layer, t, :H * d].copy()[None], x[layer, t, H * d:H * d + kv].copy()[None]
        if layer == 0:       # layer 1 has no rotation
            oracle.rope_and_store_kv(q, k, None, None, None, cos, sin, 1, H, KVH, d, H * d, kv, pos, True)
        return q[0], (k[0], x[layer, t, H * d + kv:])

    def check_rows():
        for s in range(rows):
            assert m.len[s] == len(text[s])
            for layer in range(layers):
                for i in range(2):
                    got = rows_of(host(planes[2 * layer + i]), host(c.table)[s], len(text[s]), ps)
                    want = np.array([t[layer][i] for t in text[s]], np.float16).reshape(len(text[s]), kv)
                    np.testing.assert_array_equal(bits(got), bits(want))

    def prompts(seqs, lens):
        assert c.extend(seqs, lens)[0] == m.extend(seqs, lens)[0] == m.OK
        who = np.concatenate([np.full(n, s) for s, n in zip(seqs, lens)])
        pos = np.concatenate([np.arange(n) for n in lens])
        x = fresh(len(who))
        for layer in range(layers):
            b = dev(x[layer])
            b200attn.launch_rope_and_store_kv_paged(
                b, b[:, H * d:], b[:, H * d + kv:], planes[2 * layer], planes[2 * layer + 1], 0, pages, ps, c.table,
                stride, rows, _i32(who), dcos, dsin, cap, len(who), H, KVH, d, wide, wide, _i32(pos), layer == 0)
        _sync()
        for t, (s, p) in enumerate(zip(who, pos)):
            text[s].append([row(x, layer, t, p)[1] for layer in range(layers)])

    def step(seqs):
        n = len(seqs)
        st, _, first = c.extend(seqs, [0 if s < 0 else 1 for s in seqs])
        assert st == m.extend(seqs, [0 if s < 0 else 1 for s in seqs])[0] == m.OK
        x, size = fresh(n), b200attn.decode_paged_workspace_bytes(n, H, KVH, d)
        ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
        out = torch.empty((layers, n, H * d), dtype=torch.float16, device="cuda")
        ds, dp = _i32(seqs), _i32(first)
        for layer in range(layers):
            b = dev(x[layer])
            b200attn.launch_decode_step_paged_fused(
                b, wide, b[:, H * d:], b[:, H * d + kv:], wide, planes[2 * layer], planes[2 * layer + 1], 0, pages, ps,
                c.table, stride, rows, ds, dcos, dsin, cap, layer == 0, dp, out[layer], 0, n, H, KVH, d, ws, size)
        _sync()
        for b, s in enumerate(seqs):
            if s < 0:
                assert np.all(host(out)[:, b] == 0)
                continue
            text[s].append([row(x, layer, b, first[b])[1] for layer in range(layers)])
            for layer in range(layers):
                k = np.array([t[layer][0] for t in text[s]]).reshape(-1, KVH, d)
                v = np.array([t[layer][1] for t in text[s]]).reshape(-1, KVH, d)
                want, bound = attend64(row(x, layer, b, first[b])[0].reshape(H, d), k, v, H, KVH)
                assert_within(host(out)[layer, b].reshape(H, d), want, bound)

    prompts([0, 1], [37, 100])
    step([1, 0])
    assert c.fork([0, 1, 0], [2, 3, 4], [38, 64, 16]) == m.fork([0, 1, 0], [2, 3, 4], [38, 64, 16]) == m.OK
    text[2], text[3], text[4] = text[0][:38], text[1][:64], text[0][:16]
    step([0, -1, 2, 3, 4])
    step([4, 2, 1])
    assert c.truncate([1, 0], [90, 0]) == m.truncate([1, 0], [90, 0]) == m.OK
    del text[1][90:]
    text[0] = []
    step([1, 2])
    check_rows()
    assert c.compact() == m.compact()
    check_rows()
    prompts([5, 0], [50, 3])
    step([0, 1, 2, 3, 4, 5])
    check_rows()
    assert _error_word() == 0


@pytest.mark.parametrize("rotate", [True, False])
def test_prompts_attended_and_continued(cuda, rotate):
    """The way of a prompt into pages: Q and K rotated in place, stored as they are, attended from the rows;
    then a chunk that continues one, attended an entry a row. The pages hold what the rotating append stores."""
    import torch
    H, KVH, d, ps, pages, rows, stride, cap = 16, 4, 128, 16, 60, 3, 20, 320
    kv, wide = KVH * d, (H + 2 * KVH) * d
    cos, sin = b200attn.rope_tables_host(cap, d, 5.0e6)
    dcos, dsin = dev(cos), dev(sin)
    c = b200attn.PagedKVCache(1, pages, ps, KVH, d, rows, stride)
    seqs, lens = [2, 0], [200, 37]
    x = seeded_f16((sum(lens), wide), 60)
    qkv = dev(x)
    out = torch.empty((sum(lens), H * d), dtype=torch.float16, device="cuda")
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    who, at = np.repeat(seqs, lens), np.concatenate([np.arange(n) for n in lens])
    c.extend(_i32(seqs), _i32(lens), pos)
    starts = [0, lens[0]]
    if rotate:
        for a, n in zip(starts, lens):
            b200attn.launch_rope(qkv[a:], qkv[a:, H * d:], dcos, dsin, n, H, KVH, d, wide, wide, 0)
    b200attn.launch_rope_and_store_kv_paged(None, qkv[:, H * d:], qkv[:, H * d + kv:], *c.pages(0), _i32(who), None, None,
                                            0, sum(lens), 0, KVH, d, 0, wide, _i32(at), False)
    for a, n in zip(starts, lens):
        b200attn.launch_causal_attention_prefill(qkv[a:], qkv[a:, H * d:], qkv[a:, H * d + kv:], out[a:], n, H, KVH, d,
                                                 wide, wide)
    assert c.check() == 13 + 3 and pos.tolist() == [0, 0]
    # the same rows through the rotating append
    other = b200attn.PagedKVCache(1, pages, ps, KVH, d, rows, stride)
    other.buffer.copy_(c.buffer)
    other.get_k_pages(0)[:16].zero_()
    y = dev(x)
    b200attn.launch_rope_and_store_kv_paged(y, y[:, H * d:], y[:, H * d + kv:], *other.pages(0)[:5], c.page_table, stride,
                                            rows, _i32(who), dcos, dsin, cap, sum(lens), H, KVH, d, wide, wide, _i32(at),
                                            rotate)
    _sync()
    table = host(c.page_table)
    kp, vp = (host(p) for p in (c.get_k_pages(0), c.get_v_pages(0)))
    for s, n in zip(seqs, lens):
        np.testing.assert_array_equal(bits(rows_of(kp, table[s], n, ps)),
                                      bits(rows_of(host(other.get_k_pages(0)), table[s], n, ps)))
    np.testing.assert_array_equal(bits(host(y)[:, :H * d]), bits(host(qkv)[:, :H * d]))
    q = host(qkv)[:, :H * d].reshape(-1, H, d)
    for a, s, n in zip(starts, seqs, lens):
        k, v = (rows_of(p, table[s], n, ps).reshape(n, KVH, d) for p in (kp, vp))
        want = np.array([attend64(q[a + t], k[:t + 1], v[:t + 1], H, KVH)[0] for t in range(n)]).reshape(n, -1)
        got = host(out)[a:a + n]
        assert max_abs(got, want) <= MAX_ABS and rel_l2(got, want) <= REL_L2
    # nine more rows of sequence 2
    n, old = 9, 200
    z = seeded_f16((n, wide), 61)
    qkv = dev(z)
    c.extend(_i32([2]), _i32([n]), pos)
    assert c.check() == 1 and pos.tolist()[0] == old
    b200attn.launch_rope_and_store_kv_paged(qkv, qkv[:, H * d:], qkv[:, H * d + kv:], *c.pages(0), _i32([2] * n), dcos, dsin,
                                            cap, n, H, KVH, d, wide, wide, _i32(range(old, old + n)), rotate)
    size = b200attn.decode_paged_workspace_bytes(n, H, KVH, d)
    b200attn.launch_causal_attention_decode_paged(qkv, wide, *c.pages(0), _i32([2] * n), _i32(range(old, old + n)), 1, out,
                                                  0, n, H, KVH, d, torch.zeros(size, dtype=torch.uint8, device="cuda"), size)
    _sync()
    table = host(c.page_table)
    k, v = (rows_of(host(p), table[2], old + n, ps).reshape(-1, KVH, d) for p in (c.get_k_pages(0), c.get_v_pages(0)))
    for t in range(n):
        want, bound = attend64(host(qkv)[t, :H * d].reshape(H, d), k[:old + t + 1], v[:old + t + 1], H, KVH)
        assert_within(host(out)[t].reshape(H, d), want, bound)
    assert _error_word() == 0
