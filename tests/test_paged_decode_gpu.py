"""Decode attention, the decode step and the append over a paged KV cache on
the GPU, against 64-bit attention (tests/_paged.py has the bound and where it
comes from) and the oracle's RoPE rows, bit for bit."""
import numpy as np
import pytest

import b200attn
import oracle
from _gpu import Graph, bits, dev, host
from _paged import assert_within, attend64, attend64_wide, rows_of
from _util import seeded_f16

pytestmark = pytest.mark.gpu
THETA = 5.0e6


def _sync():
    import torch
    torch.cuda.synchronize()


def _error_word():
    _sync()
    w = b200attn.lib().b2_device_error_word()
    assert b200attn.lib().b2_clear_device_error_word() == 0
    return w


class Cache:
    """Host pools with NaN wherever no token lies, a shuffled table, and their device copies."""

    def __init__(self, lens, kvh, d, ps, seed, stride=None, interleaved=False, rows=None, q_std=1.0):
        rng = np.random.default_rng(seed)
        held = [-(-n // ps) for n in lens]
        self.lens, self.kvh, self.d, self.ps = lens, kvh, d, ps
        self.stride = stride or max(1, max(held))
        self.rows = rows or len(lens)
        self.pages = sum(held) + 3
        perm = rng.permutation(self.pages)
        # entries past a sequence's pages are never read: numbers no pool has
        self.table = np.full((self.rows, self.stride), 0x7ffffff0, np.int32)
        kv = kvh * d
        self.k = np.full((self.pages, ps, kv), np.nan, np.float16)
        self.v = self.k.copy()
        at = 0
        for b, n in enumerate(lens):
            mine = perm[at:at + held[b]]
            at += held[b]
            self.table[b, :held[b]] = mine
            for pool, s in ((self.k, 1), (self.v, 2)):
                x = seeded_f16((n, kv), seed * 1000 + b * 10 + s)
                for j in range(held[b]):
                    part = x[j * ps:(j + 1) * ps]
                    pool[mine[j], :len(part)] = part
        self.interleaved = interleaved
        if interleaved:   # [page][K | V]
            self.dev = dev(np.stack([self.k, self.v], 1))
            self.dk, self.dv = self.dev[:, 0], self.dev[:, 1]
            self.page_stride = 2 * ps * kv
        else:
            self.dk, self.dv = dev(self.k), dev(self.v)
            self.page_stride = 0
        self.dtable = dev(self.table)

    def rows_k(self, b, n):
        return rows_of(self.k, self.table[b], n, self.ps).reshape(n, self.kvh, self.d)

    def rows_v(self, b, n):
        return rows_of(self.v, self.table[b], n, self.ps).reshape(n, self.kvh, self.d)

    def args(self):
        return (self.dk, self.dv, self.page_stride, self.pages, self.ps, self.dtable, self.stride, self.rows)


def _ws(n, H, KVH, d):
    import torch
    size = b200attn.decode_paged_workspace_bytes(n, H, KVH, d)
    return torch.zeros(size, dtype=torch.uint8, device="cuda"), size


def _decode(c, q, H, seqs=None, lens=None, bias=0, q_stride=0, out_stride=0, ws=None, stream=None):
    import torch
    n = len(lens if lens is not None else c.lens)
    lens = np.asarray(c.lens if lens is None else lens, np.int32) - bias
    dq = q if isinstance(q, torch.Tensor) else dev(q)
    width = out_stride or H * c.d
    out = torch.full((n + 1, width), -7.0, dtype=torch.float16, device="cuda")
    dl, ds = dev(lens), None if seqs is None else dev(np.asarray(seqs, np.int32))
    ws = ws or _ws(n, H, c.kvh, c.d)
    _sync()
    b200attn.launch_causal_attention_decode_paged(dq, q_stride, *c.args(), ds, dl, bias, out, out_stride, n, H, c.kvh,
                                                  c.d, *ws, stream=stream)
    _sync()
    out = host(out)
    assert np.all(out[n] == -7) and np.all(out[:, H * c.d:] == -7)   # rows and columns behind: as they were
    return out[:n, :H * c.d].reshape(n, H, c.d)


def _check(got, c, q, H, seqs=None, lens=None):
    lens = c.lens if lens is None else lens
    for b, n in enumerate(lens):
        s = b if seqs is None else seqs[b]
        if n <= 0 or not 0 <= s < c.rows:
            assert np.all(got[b] == 0)
            continue
        want, bound = attend64(q[b].reshape(H, c.d), c.rows_k(s, n), c.rows_v(s, n), H, c.kvh)
        assert_within(got[b], want, bound)


@pytest.mark.parametrize("H,KVH", [(16, 4), (4, 1), (8, 2), (32, 8), (8, 8), (24, 8), (7, 1), (32, 4), (20, 4), (16, 2),
                                   (8, 1), (64, 8), (4, 4), (2, 2), (1, 1)])
@pytest.mark.parametrize("ps", [16, 64, 5])
def test_lengths_at_every_edge(cuda, H, KVH, ps):
    lens = [1, 0, 2, 15, 16, 17, ps, ps + 1, 4 * ps - 1, 255, 256, 257, 0, 700, 1543]
    c = Cache(lens, KVH, 128, ps, 3)
    q = seeded_f16((len(lens), H * 128), 4, 1.5)
    _check(_decode(c, q, H), c, q, H)
    assert _error_word() == 0


@pytest.mark.parametrize("ps", [1, 2, 8, 24, 32, 48, 100, 128, 256, 1000])
def test_page_sizes(cuda, ps):
    lens = [ps, 3 * ps + 1, 1, 333]
    c = Cache(lens, 4, 128, ps, 5)
    q = seeded_f16((4, 2048), 6)
    _check(_decode(c, q, 16), c, q, 16)


@pytest.mark.parametrize("H,KVH,d", [(9, 3, 64), (12, 1, 128), (40, 4, 128), (5, 5, 80), (4, 2, 256), (6, 2, 8), (16, 16, 64),
                                     (20, 4, 24)])
def test_other_head_layouts(cuda, H, KVH, d):
    lens = [1, 40, 0, 513]
    c = Cache(lens, KVH, d, 16, 7)
    q = seeded_f16((4, H * d), 8)
    _check(_decode(c, q, H), c, q, H)


@pytest.mark.parametrize("n,H,KVH", [(1, 16, 4), (1, 4, 1), (2, 32, 8), (1, 32, 4), (1, 16, 2), (2, 64, 8), (1, 8, 1)])
def test_long_sequences(cuda, n, H, KVH):
    lens = [40001, 17][:n]
    c = Cache(lens, KVH, 128, 32, 9)
    q = seeded_f16((n, H * 128), 10, 2.0)
    _check(_decode(c, q, H), c, q, H)
    assert _error_word() == 0


@pytest.mark.parametrize("n,H,KVH", [(300, 4, 1), (1024, 4, 1), (1100, 4, 1), (1024, 16, 4), (1024, 16, 2), (700, 32, 8)])
def test_many_short_sequences(cuda, n, H, KVH):
    rng = np.random.default_rng(11)
    lens = rng.integers(0, 60, n).tolist()
    c = Cache(lens, KVH, 128, 16, 12)
    q = seeded_f16((n, H * 128), 13)
    _check(_decode(c, q, H), c, q, H)
    assert _error_word() == 0


@pytest.mark.parametrize("H,KVH,d", [(16, 4, 128), (6, 3, 64)])
def test_entries_by_table_row_strides_and_bias(cuda, H, KVH, d):
    """Entries name their table rows: idle ones, some twice with different lengths
    (drafted tokens), Q inside wider rows, K and V of a page side by side."""
    c = Cache([100, 0, 517, 33], KVH, d, 16, 14, stride=40, interleaved=True)
    seqs = [2, -1, 2, 3, 0, 4, 1, 2, 1 << 30]
    lens = [517, 9, 516, 33, 100, 12, 0, 515, 3]
    wide = H * d + 2 * KVH * d
    rows = seeded_f16((len(seqs), wide), 15)
    got = _decode(c, rows, H, seqs=seqs, lens=lens, bias=1, q_stride=wide, out_stride=H * d + 64)
    _check(got, c, rows[:, :H * d], H, seqs=seqs, lens=lens)
    assert _error_word() == 0


@pytest.mark.parametrize("H,KVH,d", [(16, 4, 128), (4, 1, 128), (6, 3, 64)])
def test_lengths_beyond_the_table_are_its_capacity(cuda, H, KVH, d):
    c = Cache([64, 64], KVH, d, 16, 16)
    q = seeded_f16((2, H * d), 17)
    got = _decode(c, q, H, lens=[2**31 - 1, -(2**31)])
    _check(got[:1], c, q, H, lens=[64])
    assert np.all(got[1] == 0) and _error_word() == 0


@pytest.mark.parametrize("H,KVH,d", [(16, 4, 128), (4, 1, 128), (6, 3, 64)])
def test_pages_outside_the_pool_are_left_out_and_flagged(cuda, H, KVH, d):
    ps = 16
    c = Cache([100, 50, 20], KVH, d, ps, 18)
    for b, j, page in ((0, 2, -1), (0, 6, c.pages), (1, 1, 0x7fffffff), (2, 0, -5), (2, 1, c.pages)):
        c.table[b, j] = page
    c.dtable = dev(c.table)
    q = seeded_f16((3, H * d), 19)
    got = _decode(c, q, H)
    assert _error_word() == 4
    for b, n in enumerate(c.lens):
        keep = [t for t in range(n) if 0 <= c.table[b, t // ps] < c.pages]
        if not keep:
            assert np.all(got[b] == 0)
            continue
        at = c.table[b][np.array(keep) // ps], np.array(keep) % ps
        want, bound = attend64(q[b].reshape(H, d), c.k[at].reshape(-1, KVH, d), c.v[at].reshape(-1, KVH, d), H, KVH)
        assert_within(got[b], want, bound)


def test_offsets_past_32_bits(cuda):
    """A pool whose last pages lie past 2^32 elements, K and V in one allocation."""
    import torch
    ps, KVH, H, d = 16, 4, 16, 128
    stride = 1 << 26                                    # elements between pages
    pages = 66
    pool = torch.empty(pages * stride + 2 * ps * KVH * d, dtype=torch.float16, device="cuda")
    c = Cache([45], KVH, d, ps, 20)
    order = [65, 0, 64]
    for g, to in zip(c.table[0], order):
        for at, src in ((0, c.k), (ps * KVH * d, c.v)):
            pool[to * stride + at:][:ps * KVH * d] = dev(src[g]).flatten()
    q = seeded_f16((1, H * d), 21)
    c.dk, c.dv, c.page_stride = pool, pool[ps * KVH * d:], stride
    want, bound = attend64(q[0].reshape(H, d), c.rows_k(0, 45), c.rows_v(0, 45), H, KVH)
    c.table, c.pages, c.dtable = np.array([order], np.int32), pages, dev(np.array([order], np.int32))
    assert_within(_decode(c, q, H)[0], want, bound)
    # and a row appended there
    kn, vn = seeded_f16((1, KVH * d), 22), seeded_f16((1, KVH * d), 23)
    out = torch.empty((1, H * d), dtype=torch.float16, device="cuda")
    b200attn.launch_decode_step_paged_fused(dev(q), 0, dev(kn), dev(vn), 0, *c.args(), None, None, None, 0, False,
                                            dev(np.array([45], np.int32)), out, 0, 1, H, KVH, d, *_ws(1, H, KVH, d))
    _sync()
    at = 64 * stride + 13 * KVH * d
    np.testing.assert_array_equal(bits(host(pool[at:at + KVH * d])), bits(kn[0]))
    np.testing.assert_array_equal(bits(host(pool[at + ps * KVH * d:][:KVH * d])), bits(vn[0]))
    assert _error_word() == 0


@pytest.mark.parametrize("H,KVH,d", [(16, 4, 128), (4, 1, 128), (6, 3, 64)])
def test_a_batch_without_tokens(cuda, H, KVH, d):
    c = Cache([16, 16], KVH, d, 16, 70)
    q = seeded_f16((5, H * d), 71)
    got = _decode(c, q, H, seqs=[0, -1, 1, 0, -7], lens=[0, 40, -3, 0, 1])
    assert np.all(got == 0) and _error_word() == 0


def test_output_rows_off_four_bytes(cuda):
    """An odd output stride or address takes the other kernel: the same values within the bound."""
    import torch
    c = Cache([300, 17], 4, 128, 16, 72)
    q = seeded_f16((2, 2048), 73)
    _check(_decode(c, q, 16, out_stride=2049), c, q, 16)
    out = torch.zeros(2 * 2048 + 1, dtype=torch.float16, device="cuda")
    b200attn.launch_causal_attention_decode_paged(dev(q), 0, *c.args(), None, dev(np.array(c.lens, np.int32)), 0,
                                                  out[1:], 0, 2, 16, 4, 128, *_ws(2, 16, 4, 128))
    _sync()
    assert host(out)[0] == 0
    _check(host(out)[1:].reshape(2, 16, 128), c, q, 16)


def test_two_streams_at_once(cuda):
    """Steps of two caches on two streams, workspaces of their own: each as alone."""
    import torch
    H, KVH, d = 16, 4, 128
    rng = np.random.default_rng(74)
    made = []
    for k in range(2):
        lens = rng.integers(1, 3000, 20).tolist()
        c = Cache(lens, KVH, d, 16, 75 + k)
        q, kn, vn = seeded_f16((20, H * d), 77 + k), seeded_f16((20, KVH * d), 79 + k), seeded_f16((20, KVH * d), 81 + k)
        made.append((c, [dev(x) for x in (q, kn, vn)], dev(np.array(lens, np.int32) - 1), _ws(20, H, KVH, d),
                     torch.empty((20, H * d), dtype=torch.float16, device="cuda"), torch.cuda.Stream()))

    def go(m, stream):
        c, (q, kn, vn), pos, ws, out, _ = m
        b200attn.launch_decode_step_paged_fused(q, 0, kn, vn, 0, *c.args(), None, None, None, 0, False, pos, out, 0, 20,
                                                H, KVH, d, *ws, stream=stream)

    _sync()
    alone = []
    for m in made:
        go(m, None)
        _sync()
        alone.append(m[4].clone())
        m[4].zero_()
    _sync()
    for _ in range(20):
        for m in made:
            go(m, m[5])
    _sync()
    for m, want in zip(made, alone):
        np.testing.assert_array_equal(bits(host(m[4])), bits(host(want)))
    assert _error_word() == 0


@pytest.mark.parametrize("scale", [0.0, 20.0])
def test_flat_and_peaked_scores(cuda, scale):
    c = Cache([1000, 3], 4, 128, 16, 24)
    q = (seeded_f16((2, 2048), 25) * np.float16(scale)).astype(np.float16)
    _check(_decode(c, q, 16), c, q, 16)


@pytest.mark.parametrize("H,KVH,d", [(16, 4, 128), (4, 1, 128), (16, 2, 128), (32, 8, 128), (7, 1, 128), (12, 1, 128), (6, 3, 64)])
def test_weights_keep_more_than_16_bits(cuda, H, KVH, d):
    """Outputs far below the rows they are made of show the weights' rounding."""
    lens = [2, 3, 5, 16, 33, 1000]
    c = Cache(lens, KVH, d, 16, 90)
    q = seeded_f16((len(lens), H * d), 91, 0.1)
    got = _decode(c, q, H)
    for b, n in enumerate(lens):
        assert_within(got[b], *attend64_wide(q[b].reshape(H, d), c.rows_k(b, n), c.rows_v(b, n), H, KVH))


@pytest.mark.parametrize("H,KVH", [(16, 4), (4, 1), (32, 8)])
def test_many_small_weights_beside_a_large_one(cuda, H, KVH):
    """2,000 tokens that weigh 2^-26 of the first, whose V row is 0: their sum is the output.
    200 such sequences, so that a warp meets all tokens of one."""
    import torch
    n, B, d = 2000, 200, 128
    c = Cache([n] * B, KVH, d, 16, 92)
    c.k[:], c.v[:] = 0, 1
    q = np.zeros((B, H, d), np.float16)
    q[:, :, 0] = 8
    for b in range(B):
        c.k[c.table[b, 0], 0], c.v[c.table[b, 0], 0] = 25.5, 0
    c.dk.copy_(torch.from_numpy(c.k))
    c.dv.copy_(torch.from_numpy(c.v))
    got = _decode(c, q.reshape(B, -1), H)
    want, bound = attend64_wide(q[0], c.rows_k(0, n), c.rows_v(0, n), H, KVH)
    assert want.min() > 2.0 ** -16 > 16 * bound.max()
    for b in range(B):
        assert_within(got[b], want, bound)


def _formula(c, b, n, q, H):
    """softmax(q k / sqrt(d)) v of sequence b's first n rows in 64 bits, infinities and NaN as they come."""
    k, v, g = c.rows_k(b, n).astype(np.float64), c.rows_v(b, n).astype(np.float64), H // c.kvh
    q, out = q.reshape(H, c.d).astype(np.float64), np.zeros((H, c.d))
    with np.errstate(all="ignore"):
        for h in range(H):
            s = k[:, h // g] @ q[h] / np.sqrt(c.d)
            p = np.exp(s - s.max())
            out[h] = (p / p.sum()) @ v[:, h // g]
    return out


@pytest.mark.parametrize("H,KVH,d", [(16, 4, 128), (4, 1, 128), (32, 8, 128), (12, 1, 128), (6, 3, 64), (3, 3, 64)])
@pytest.mark.parametrize("where", [[0], range(16), range(40, 72), [399]])
def test_infinities_in_k(cuda, H, KVH, d, where):
    """A score of -infinity weighs nothing, wherever its tokens lie; one of +infinity has no softmax."""
    n = 400
    c = Cache([n, 17], KVH, d, 16, 94)
    for t in where:
        c.k[c.table[0, t // 16], t % 16].reshape(KVH, d)[:, 3] = np.inf
    c.dk.copy_(dev(c.k))
    q = seeded_f16((2, H * d), 95)
    got, want = _decode(c, q, H), _formula(c, 0, n, q[0], H)
    gone = np.isnan(want)
    assert gone.any() and not gone.all()
    np.testing.assert_array_equal(np.isnan(got[0]), gone)
    # the heads that keep a softmax keep its values: those of the other tokens
    keep = np.setdiff1d(np.arange(n), np.array(where))
    exact, bound = attend64(q[0].reshape(H, d), c.rows_k(0, n)[keep], c.rows_v(0, n)[keep], H, KVH)
    fine = ~gone.any(1)
    assert_within(got[0][fine], exact[fine], bound[fine])
    _check(got[1:], c, q[1:], H, seqs=[1], lens=[17])


@pytest.mark.parametrize("H,KVH,d", [(16, 4, 128), (4, 1, 128), (32, 8, 128), (12, 1, 128), (6, 3, 64), (3, 3, 64)])
def test_nan_in_a_query_reaches_its_output(cuda, H, KVH, d):
    """All scores of a head are then NaN: so is its output, and no other head's."""
    lens = [40, 700, 1, 0]
    c = Cache(lens, KVH, d, 16, 96)
    q = seeded_f16((4, H * d), 97)
    nan = [(0, 0), (1, H - 1), (2, H // 2), (3, 0)]
    for b, h in nan:
        q[b, h * d + 5] = np.nan
    got = _decode(c, q, H)
    for b, h in nan[:3]:
        assert np.all(np.isnan(got[b, h]))
        rest = np.arange(H) != h
        clean = np.nan_to_num(q[b].reshape(H, d))
        want, bound = attend64(clean, c.rows_k(b, lens[b]), c.rows_v(b, lens[b]), H, KVH)
        assert_within(got[b][rest], want[rest], bound[rest])
    assert np.all(got[3] == 0)


def test_repeated_calls_share_a_workspace(cuda):
    """Calls of different lengths on one workspace, on a stream of their own, give what each gives alone."""
    import torch
    lens = [5000, 1, 300, 0]
    c = Cache(lens, 4, 128, 16, 26)
    q = seeded_f16((4, 2048), 27)
    st = torch.cuda.Stream()
    ws = _ws(4, 16, 4, 128)
    first = _decode(c, q, 16, ws=ws, stream=st)
    short = _decode(c, q, 16, lens=[10, 1, 2, 0], ws=ws, stream=st)
    again = _decode(c, q, 16, ws=ws, stream=st)
    np.testing.assert_array_equal(bits(first), bits(again))
    _check(first, c, q, 16)
    _check(short, c, q, 16, lens=[10, 1, 2, 0])


# ---- the append --------------------------------------------------------------------

def _rotated(q, k, cos, sin, pos, H, KVH, d):
    """The oracle's rotation of one row at a position."""
    q, k = q.copy()[None], k.copy()[None]
    oracle.rope_and_store_kv(q, k, None, None, None, cos, sin, 1, H, KVH, d, H * d, KVH * d, pos, True)
    return q[0], k[0]


@pytest.mark.parametrize("H,KVH,d,ps", [(16, 4, 128, 16), (4, 1, 128, 5), (6, 3, 64, 48), (3, 1, 34, 7), (0, 2, 32, 16)])
@pytest.mark.parametrize("rotate", [True, False])
@pytest.mark.parametrize("odd", [False, True])
def test_append(cuda, H, KVH, d, ps, rotate, odd):
    """Rows of three sequences in any order, among them padding, rows past the capacity
    and past the tables; everything else in the pools stays as it was."""
    stride, rope_rows = 6, 4 * ps
    kv, wide = KVH * d, (H + 2 * KVH) * d + (3 if odd else 0)   # odd: rows off 16 bytes
    c = Cache([6 * ps] * 3, KVH, d, ps, 30, stride=stride)
    rng = np.random.default_rng(31)
    place = [(s, p) for s in range(3) for p in rng.permutation(6 * ps)[:13].tolist()]
    rng.shuffle(place)
    place += [(-1, 3), (1, -2), (0, 6 * ps), (2, 2**31 - 1), (3, 0)]
    T = len(place)
    qkv = seeded_f16((T, wide), 32)
    cos, sin = b200attn.rope_tables_host(rope_rows, d, THETA)
    dq = dev(qkv)
    flat = dq.view(-1)
    b200attn.launch_rope_and_store_kv_paged(
        flat if H else None, flat[H * d:], flat[H * d + kv:], *c.args(), dev(np.array([s for s, _ in place], np.int32)),
        dev(cos) if rotate else None, dev(sin) if rotate else None, rope_rows if rotate else 0, T, H, KVH, d, wide, wide,
        dev(np.array([p for _, p in place], np.int32)), rotate)
    want_q, k, v = qkv.copy(), c.k.copy(), c.v.copy()
    late = False
    for t, (s, p) in enumerate(place):
        if not 0 <= s < 3 or not 0 <= p < stride * ps:
            continue
        kr, vr = qkv[t, H * d:H * d + kv], qkv[t, H * d + kv:H * d + 2 * kv]
        if rotate:
            if p >= rope_rows:
                late = True
                continue
            if H:
                want_q[t, :H * d], kr = _rotated(qkv[t, :H * d], kr, cos, sin, p, H, KVH, d)
            else:
                _, kr = _rotated(kr, kr, cos, sin, p, KVH, KVH, d)
        k[c.table[s, p // ps], p % ps] = kr
        v[c.table[s, p // ps], p % ps] = vr
    assert _error_word() == (2 if late else 0)
    np.testing.assert_array_equal(bits(host(dq)), bits(want_q))
    np.testing.assert_array_equal(bits(host(c.dk)), bits(k))
    np.testing.assert_array_equal(bits(host(c.dv)), bits(v))


def test_append_flags_bad_pages_and_keeps_the_rest(cuda):
    c = Cache([32, 32], 4, 128, 16, 33)
    c.table[0, 1], c.table[1, 0] = -1, c.pages
    c.dtable = dev(c.table)
    kn, vn = seeded_f16((4, 512), 34), seeded_f16((4, 512), 35)
    b200attn.launch_rope_and_store_kv_paged(
        None, dev(kn), dev(vn), *c.args(), dev(np.array([0, 0, 1, 1], np.int32)), None, None, 0, 4, 0, 4, 128, 0, 0,
        dev(np.array([3, 20, 5, 30], np.int32)), False)
    assert _error_word() == 4
    k = c.k.copy()
    k[c.table[0, 0], 3], k[c.table[1, 1], 14] = kn[0], kn[3]
    np.testing.assert_array_equal(bits(host(c.dk)), bits(k))


def test_append_of_a_prompt_equals_the_contiguous_append(cuda):
    """A prompt's rows through pages and through the contiguous cache: the same bits."""
    import torch
    S, H, KVH, d, ps = 777, 16, 4, 128, 64
    c = Cache([S], KVH, d, ps, 36)
    cos, sin = (dev(x) for x in b200attn.rope_tables_host(S + 10, d, THETA))
    wide = (H + 2 * KVH) * d
    a = dev(seeded_f16((S, wide), 37))
    b = a.clone()
    kc, vc = (torch.zeros((S + 10, KVH * d), dtype=torch.float16, device="cuda") for _ in range(2))
    b200attn.launch_rope_and_store_kv(a, a[:, H * d:], a[:, H * d + KVH * d:], kc, vc, cos, sin, S, H, KVH, d, wide,
                                      wide, 0, True)
    b200attn.launch_rope_and_store_kv_paged(
        b, b[:, H * d:], b[:, H * d + KVH * d:], *c.args(), dev(np.zeros(S, np.int32)), cos, sin, S + 10, S, H, KVH, d,
        wide, wide, dev(np.arange(S, dtype=np.int32)), True)
    _sync()
    np.testing.assert_array_equal(bits(host(a)), bits(host(b)))
    c.k, c.v = host(c.dk), host(c.dv)
    np.testing.assert_array_equal(bits(c.rows_k(0, S).reshape(S, -1)), bits(host(kc)[:S]))
    np.testing.assert_array_equal(bits(c.rows_v(0, S).reshape(S, -1)), bits(host(vc)[:S]))


# ---- the step ------------------------------------------------------------------------

def _step(c, q, kn, vn, pos, H, rotate, rope_rows, seqs=None, ws=None, append=True, stream=None):
    import torch
    n = len(pos)
    out = torch.full((n + 1, H * c.d), -7.0, dtype=torch.float16, device="cuda")
    cos, sin = b200attn.rope_tables_host(max(rope_rows, 1), c.d, THETA) if rotate else (None, None)
    dq = dev(q)
    b200attn.launch_decode_step_paged_fused(
        dq, q.shape[1], dev(kn) if append else None, dev(vn) if append else None, kn.shape[1], *c.args(),
        None if seqs is None else dev(np.asarray(seqs, np.int32)), dev(cos) if rotate else None,
        dev(sin) if rotate else None, rope_rows if rotate else 0, rotate, dev(np.asarray(pos, np.int32)), out, 0, n, H,
        c.kvh, c.d, *(ws or _ws(n, H, c.kvh, c.d)), stream=stream)
    _sync()
    np.testing.assert_array_equal(bits(host(dq)), bits(q))   # Q is read, never written
    assert np.all(host(out)[n] == -7)
    return host(out)[:n].reshape(n, H, c.d)


@pytest.mark.parametrize("H,KVH,d,ps", [(16, 4, 128, 16), (4, 1, 128, 16), (8, 2, 128, 5), (32, 8, 128, 64), (7, 1, 128, 24),
                                        (6, 3, 64, 16)])
@pytest.mark.parametrize("rotate", [True, False])
def test_step(cuda, H, KVH, d, ps, rotate):
    """New rows at page starts, page ends and mid-page; the pools change there and nowhere else."""
    lens = [1, 2, 16, 17, ps, ps + 1, 4 * ps, 300, 1200]
    c = Cache(lens, KVH, d, ps, 40)
    n, rope_rows = len(lens), 1300
    pos = [x - 1 for x in lens]
    q, kn, vn = seeded_f16((n, H * d), 41, 1.5), seeded_f16((n, KVH * d), 42), seeded_f16((n, KVH * d), 43)
    got = _step(c, q, kn, vn, pos, H, rotate, rope_rows)
    assert _error_word() == 0
    cos, sin = b200attn.rope_tables_host(rope_rows, d, THETA)
    for b, p in enumerate(pos):
        qr, kr = _rotated(q[b], kn[b], cos, sin, p, H, KVH, d) if rotate else (q[b], kn[b])
        at = c.table[b, p // ps], p % ps
        c.k[at], c.v[at] = kr, vn[b]
        want, bound = attend64(qr.reshape(H, d), c.rows_k(b, p + 1), c.rows_v(b, p + 1), H, KVH)
        assert_within(got[b], want, bound)
    np.testing.assert_array_equal(bits(host(c.dk)), bits(c.k))
    np.testing.assert_array_equal(bits(host(c.dv)), bits(c.v))


@pytest.mark.parametrize("H,KVH,d", [(16, 4, 128), (4, 1, 128), (6, 3, 64)])
@pytest.mark.parametrize("rotate", [True, False])
def test_step_equals_append_then_decode(cuda, H, KVH, d, rotate):
    rng = np.random.default_rng(44)
    lens = rng.integers(1, 900, 11).tolist()
    n, rope_rows = len(lens), 1000
    pos = [x - 1 for x in lens]
    q, kn, vn = seeded_f16((n, H * d), 45), seeded_f16((n, KVH * d), 46), seeded_f16((n, KVH * d), 47)
    a, b = Cache(lens, KVH, d, 16, 48), Cache(lens, KVH, d, 16, 48)
    one = _step(a, q, kn, vn, pos, H, rotate, rope_rows)
    cos, sin = (dev(x) for x in b200attn.rope_tables_host(rope_rows, d, THETA))
    dq = dev(q)
    b200attn.launch_rope_and_store_kv_paged(dq, dev(kn), dev(vn), *b.args(), None, cos, sin, rope_rows, n, H, KVH, d, 0,
                                            0, dev(np.array(pos, np.int32)), rotate)
    two = _decode(b, dq, H, lens=lens, bias=1)
    np.testing.assert_array_equal(bits(one), bits(two))
    np.testing.assert_array_equal(bits(host(a.dk)), bits(host(b.dk)))
    np.testing.assert_array_equal(bits(host(a.dv)), bits(host(b.dv)))


@pytest.mark.parametrize("H,KVH,d", [(16, 4, 128), (4, 1, 128), (6, 3, 64)])
def test_step_idle_entries_capacity_and_late_positions(cuda, H, KVH, d):
    ps = 16
    c = Cache([64, 40, 64, 64], KVH, d, ps, 50)
    n, rope_rows = 6, 50
    seqs, pos = [0, -1, 1, 2, 3, 1], [49, 7, 39, 55, 64, -1]   # fine, idle, fine, past the tables, past the capacity, idle
    q, kn, vn = seeded_f16((n, H * d), 51), seeded_f16((n, KVH * d), 52), seeded_f16((n, KVH * d), 53)
    before = c.k.copy(), c.v.copy()
    got = _step(c, q, kn, vn, pos, H, True, rope_rows, seqs=seqs)
    assert _error_word() == 2
    cos, sin = b200attn.rope_tables_host(rope_rows, d, THETA)
    q = q.copy()
    for b in (0, 2):
        q[b], kr = _rotated(q[b], kn[b], cos, sin, pos[b], H, KVH, d)
        at = c.table[seqs[b], pos[b] // ps], pos[b] % ps
        c.k[at], c.v[at] = kr, vn[b]
    np.testing.assert_array_equal(bits(host(c.dk)), bits(c.k))
    np.testing.assert_array_equal(bits(host(c.dv)), bits(c.v))
    _check(got, c, q, H, seqs=seqs, lens=[50, 0, 40, 56, 64, 0])
    assert not np.array_equal(bits(before[0]), bits(c.k))
    # nothing appended: the pools stay, the rows there are attended
    c.dk.copy_(dev(before[0]))
    c.dv.copy_(dev(before[1]))
    c.k, c.v = before
    got = _step(c, q, kn, vn, [30], H, False, 0, append=False)
    _check(got, c, q, H, lens=[31])
    np.testing.assert_array_equal(bits(host(c.dk)), bits(c.k))


def test_step_captured_and_replayed(cuda):
    """One captured step and position advance, replayed: each token's output and row."""
    import torch
    H, KVH, d, ps, n, steps = 16, 4, 128, 16, 3, 20
    start = [14, 0, 31]
    c = Cache([s + steps for s in start], KVH, d, ps, 60)
    wide = (H + 2 * KVH) * d
    cos, sin = b200attn.rope_tables_host(64, d, THETA)
    dcos, dsin = dev(cos), dev(sin)
    row = torch.empty((n, wide), dtype=torch.float16, device="cuda")
    out = torch.empty((n, H * d), dtype=torch.float16, device="cuda")
    pos = dev(np.array(start, np.int32))
    ws = _ws(n, H, KVH, d)
    g = Graph()
    with g:
        b200attn.launch_decode_step_paged_fused(row, wide, row[:, H * d:], row[:, H * d + KVH * d:], wide, *c.args(),
                                                None, dcos, dsin, 64, True, pos, out, 0, n, H, KVH, d, *ws,
                                                stream=g.stream)
        for b in range(n):
            b200attn.advance_position(pos[b:], 1, stream=g.stream)
    for i in range(steps):
        x = seeded_f16((n, wide), 61 + i)
        row.copy_(dev(x))
        _sync()
        g.launch()
        for b in range(n):
            p = start[b] + i
            qr, kr = _rotated(x[b, :H * d], x[b, H * d:H * d + KVH * d], cos, sin, p, H, KVH, d)
            at = c.table[b, p // ps], p % ps
            c.k[at], c.v[at] = kr, x[b, H * d + KVH * d:]
            want, bound = attend64(qr.reshape(H, d), c.rows_k(b, p + 1), c.rows_v(b, p + 1), H, KVH)
            assert_within(host(out)[b].reshape(H, d), want, bound)
    g.close()
    np.testing.assert_array_equal(bits(host(c.dk)), bits(c.k))
    assert _error_word() == 0
