"""The paged cache without a GPU: the entry points' refusals (all before the
first CUDA call) and the host model that the GPU tests hold the kernels to."""
import os
import subprocess

import numpy as np
import pytest

import b200attn
from _paged import Pages, attend64, rows_of
from _util import ROOT

F = 0x1000


def _decode(L, **o):
    a = dict(q=F, qs=0, k=F, v=F, ps=0, np_=100, sz=16, tab=F, ts=32, tr=8, seqs=None, ln=F, bias=0, out=F, os_=0, B=8,
             H=16, KVH=4, d=128, w=F, wb=1 << 30)
    a.update(o)
    return L.b2_launch_causal_attention_decode_paged(
        a["q"], a["qs"], a["k"], a["v"], a["ps"], a["np_"], a["sz"], a["tab"], a["ts"], a["tr"], a["seqs"], a["ln"],
        a["bias"], a["out"], a["os_"], a["B"], a["H"], a["KVH"], a["d"], a["w"], a["wb"], None)


def _step(L, **o):
    a = dict(q=F, qs=0, kn=F, vn=F, kns=0, k=F, v=F, ps=0, np_=100, sz=16, tab=F, ts=32, tr=8, seqs=None, cos=F, sin=F,
             rows=512, rot=True, pos=F, out=F, os_=0, B=8, H=16, KVH=4, d=128, w=F, wb=1 << 30)
    a.update(o)
    return L.b2_launch_decode_step_paged_fused(
        a["q"], a["qs"], a["kn"], a["vn"], a["kns"], a["k"], a["v"], a["ps"], a["np_"], a["sz"], a["tab"], a["ts"],
        a["tr"], a["seqs"], a["cos"], a["sin"], a["rows"], a["rot"], a["pos"], a["out"], a["os_"], a["B"], a["H"],
        a["KVH"], a["d"], a["w"], a["wb"], None)


def _append(L, **o):
    a = dict(q=F, kn=F, vn=F, k=F, v=F, ps=0, np_=100, sz=16, tab=F, ts=32, tr=8, seqs=None, cos=F, sin=F, rows=512,
             T=8, H=16, KVH=4, d=128, qs=0, ks=0, pos=F, rot=True)
    a.update(o)
    return L.b2_launch_rope_and_store_kv_paged(
        a["q"], a["kn"], a["vn"], a["k"], a["v"], a["ps"], a["np_"], a["sz"], a["tab"], a["ts"], a["tr"], a["seqs"],
        a["cos"], a["sin"], a["rows"], a["T"], a["H"], a["KVH"], a["d"], a["qs"], a["ks"], a["pos"], a["rot"], None)


@pytest.mark.parametrize("call", [_decode, _step])
def test_decode_and_step_refusals(call):
    L = b200attn.lib()
    assert call(L, B=0) == 1 and call(L, KVH=0) == 1 and call(L, KVH=3) == 1 and call(L, d=0) == 1
    assert call(L, H=0) == 1
    for name in ("q", "k", "v", "tab", "out", "w"):
        assert call(L, **{name: None}) == -1, name
    assert call(L, np_=0) == -1 and call(L, sz=0) == -1 and call(L, ts=0) == -1 and call(L, tr=0) == -1
    assert call(L, tr=7) == -1                                    # entries without a table row ...
    assert call(L, tr=7, seqs=F, wb=0) == -5                      # ... unless d_seqs names them
    assert call(L, ps=16 * 512 - 8) == -1                         # pages overlap
    assert call(L, qs=2040) == -1 and call(L, os_=2040) == -1     # rows overlap
    assert call(L, d=12) == -2 and call(L, d=264) == -2 and call(L, B=65536, tr=70000) == -2
    assert call(L, np_=1 << 31) == -2 and call(L, sz=1 << 31, ps=1 << 45) == -2
    assert call(L, k=F + 2) == -3 and call(L, q=F + 8) == -3 and call(L, qs=2052) == -3 and call(L, w=F + 8) == -3
    assert call(L, ps=16 * 512 + 4) == -3
    need = b200attn.decode_paged_workspace_bytes(8, 16, 4)
    assert need > 0 and call(L, wb=need - 1) == -5
    with pytest.raises(b200attn.B2Error):
        b200attn.launch_causal_attention_decode_paged(None, 0, F, F, 0, 1, 16, F, 1, 1, None, F, 0, F, 0, 1, 16, 4,
                                                      128, F, 1 << 30)


def test_step_refusals():
    L = b200attn.lib()
    assert _step(L, pos=None) == -1 and _step(L, cos=None) == -1 and _step(L, rows=0) == -1
    assert _step(L, vn=None) == -1 and _step(L, kn=None) == -1
    assert _step(L, kns=504) == -1
    assert _step(L, kn=F + 4) == -3 and _step(L, kns=516) == -3 and _step(L, cos=F + 2) == -3
    assert _step(L, d=72) == -2                                   # halves of a head in whole 16-byte pieces
    # without rotation none of its inputs is needed: this gets as far as the workspace
    assert _step(L, rot=False, cos=None, sin=None, rows=0, d=72, wb=0) == -5
    assert _step(L, kn=None, vn=None, wb=0) == -5


def test_append_refusals():
    L = b200attn.lib()
    assert _append(L, T=0) == 1 and _append(L, KVH=0) == 1 and _append(L, d=0) == 1
    for name in ("q", "kn", "vn", "k", "v", "tab", "cos", "sin", "pos"):
        assert _append(L, **{name: None}) == -1, name
    assert _append(L, d=127) == -1 and _append(L, rows=0) == -1 and _append(L, tr=7) == -1
    assert _append(L, ks=504) == -1 and _append(L, qs=2040) == -1 and _append(L, ps=8) == -1
    assert _append(L, T=1 << 31, tr=1 << 30, seqs=F) == -2 and _append(L, d=1 << 16) == -2
    assert _append(L, H=0, q=None, T=0) == 1


def test_workspace_sizes():
    by = b200attn.decode_paged_workspace_bytes
    for args in ((1, 16, 4), (64, 16, 4), (256, 4, 1), (1024, 32, 8), (7, 12, 3), (65535, 2, 2)):
        n = by(*args)
        assert n > 0 and n % 256 == 0 and n < 2 << 30, args
    assert by(0, 16, 4) == 0 and by(8, 16, 3) == 0 and by(8, 16, 0) == 0 and by(65536, 16, 4) == 0
    assert by(8, 16, 4, 512) == 0
    assert b200attn.kv_pages_workspace_bytes(0) == 0 and b200attn.kv_pages_workspace_bytes((1 << 21) + 1) == 0
    assert b200attn.kv_pages_workspace_bytes(1000) >= 10000


def test_page_operation_refusals():
    L = b200attn.lib()
    pool = (F, 2, 0, 100, 0, 2048)
    seqs = (F, 8, 4, 16, 100, F, F)
    ws = (F, F, 1 << 20, None)
    assert L.b2_launch_kv_pages_copy(*pool, F, F, 0, None) == 1
    assert L.b2_launch_kv_pages_copy(*pool, None, F, 1, None) == -1
    assert L.b2_launch_kv_pages_copy(None, *pool[1:], F, F, 1, None) == -1
    assert L.b2_launch_kv_pages_copy(*pool, F, F, 4097, None) == -2
    assert L.b2_launch_kv_pages_copy(F, 2, 0, 100, 0, 2044, F, F, 1, None) == -3
    assert L.b2_launch_kv_pages_copy(F + 8, *pool[1:], F, F, 1, None) == -3
    assert L.b2_launch_kv_pages_copy(F, 2, 2048 * 99, 100, 0, 2048, F, F, 1, None) == -1      # planes overlap
    assert L.b2_launch_kv_pages_copy(F, 2, 1024, 100, 4096, 2048, F, F, 1, None) == -1
    assert L.b2_launch_kv_pages_copy(F, 2, 0, (1 << 21) + 1, 0, 2048, F, F, 1, None) == -2
    for n, want in ((0, 1), (1025, -2)):
        assert L.b2_launch_kv_pages_truncate(*seqs, F, F, n, *ws) == want
        assert L.b2_launch_kv_pages_fork(*seqs, F, F, None, n, *ws) == want
        assert L.b2_launch_kv_pages_extend(*pool, *seqs[:4], *seqs[5:], F, F, n, None, *ws) == want
    assert L.b2_launch_kv_pages_truncate(F, (1 << 21) + 1, *seqs[2:], F, F, 1, *ws) == -2
    assert L.b2_launch_kv_pages_truncate(*seqs, None, F, 1, *ws) == -1
    assert L.b2_launch_kv_pages_fork(*seqs, F, None, None, 1, *ws) == -1
    assert L.b2_launch_kv_pages_extend(*pool, *seqs[:4], *seqs[5:], F, None, 1, None, *ws) == -1
    for k in (0, 1, 2, 3, 4, 5, 6):
        bad = list(seqs)
        bad[k] = 0 if k in (1, 2, 3, 4) else None
        assert L.b2_launch_kv_pages_truncate(*bad, F, F, 1, *ws) == -1, k
    small = (F, F, 16, None)
    assert L.b2_launch_kv_pages_truncate(*seqs, F, F, 1, *small) == -5
    assert L.b2_launch_kv_pages_fork(*seqs, F, F, None, 1, *small) == -5
    assert L.b2_launch_kv_pages_truncate(*seqs, F, F, 1, F, None, 1 << 20, None) == -1
    assert L.b2_launch_kv_pages_truncate(*seqs, F, F, 1, F, F + 2, 1 << 20, None) == -3
    c = (*pool, F, F, 8, 4, 16, F, F, F)
    assert L.b2_launch_kv_pages_compact(*c, F, F, 16, None) == -5
    assert L.b2_launch_kv_pages_compact(*c[:7], None, *c[8:], F, F, 1 << 20, None) == -1


def test_host_model_keeps_its_invariants():
    """Random operations on the model: counts match the tables, contents follow the sequences."""
    rng = np.random.default_rng(5)
    ps, rows, stride, pages = 4, 9, 6, 40
    m = Pages(np.zeros((2, pages, ps), np.int64), rows, stride, ps)
    text = [[] for _ in range(rows)]
    serial = 1
    for _ in range(300):
        op = rng.integers(4)
        if op == 0:
            seqs = rng.permutation(rows)[:3].tolist() + [-1]
            take = rng.integers(0, 6, 4).tolist()
            st, need, first = m.extend(seqs, take)
            if st == m.OK:
                for s, t, f in zip(seqs, take, first):
                    if s < 0:
                        continue
                    assert f == len(text[s])
                    for j in range(f, f + t):
                        m.pool[:, m.table[s, j // ps], j % ps] = serial
                        text[s].append(serial)
                        serial += 1
        elif op == 1:
            seqs = rng.permutation(rows)[:2].tolist()
            new = [int(rng.integers(0, m.len[s] + 1)) for s in seqs]
            assert m.truncate(seqs, new) == m.OK
            for s, n in zip(seqs, new):
                del text[s][n:]
        elif op == 2:
            p, c = rng.permutation(rows)[:2].tolist()
            n = int(rng.integers(0, m.len[p] + 1))
            if m.fork([p], [c], [n]) == m.OK:
                text[c] = text[p][:n]
            else:
                assert text[c]
        else:
            m.compact()
            assert np.all(m.ref[:int((m.ref > 0).sum())] > 0)
        m.check()
        for s in range(rows):
            assert rows_of(m.pool[1], m.table[s], len(text[s]), ps).tolist() == text[s]
    assert m.extend([0, 0], [1, 1])[0] == m.BAD and m.extend([rows], [1])[0] == m.BAD
    assert m.truncate([0], [stride * ps + 1]) == m.BAD


def test_attend64_known_answer():
    q = np.zeros((2, 4))
    v = np.arange(12, dtype=float).reshape(3, 1, 4)
    o, b = attend64(q, np.ones((3, 1, 4)), v, 2, 1)
    np.testing.assert_allclose(o, np.tile(v.mean(0), (2, 1)))
    assert np.all(b > 0) and np.all(b < 0.02)


SLOT_PAIR = r"""
#include <cstdio>
#include "slot_pair.h"
// A producer of rows, each one copy and then some stages, that gives up before any of its
// waits: every copy that is issued and not given back is among those that it then waits for.
int main() {
    for (int give_up = 0; give_up < 60; ++give_up) {
        b2::SlotPair q;
        int phases[2] = {0, 0}, waits = 0, copies = 0;   // phases: copies into each slot
        bool on = true;
        for (int row = 0; row < 7 && on; ++row) {
            if (q.in_use() && waits++ == give_up) break;
            // the phase that is waited for is the slot's last one
            if (q.in_use() && q.free_parity() != unsigned(phases[q.next()] - 1) % 2) return 1;
            ++phases[q.begin()];
            ++copies;
            for (int stage = 0; stage < 3 && on; ++stage) if (waits++ == give_up) on = false;
        }
        if (q.issued() != unsigned(copies)) return 2;
        int pending = 0;
        for (uint32_t j = q.oldest(); j < q.issued(); ++j, ++pending)
            if (b2::SlotPair::slot(j) != j % 2 || b2::SlotPair::parity(j) != (j / 2) % 2) return 3;
        if (pending != (copies < 2 ? copies : 2)) return 4;
    }
    return 0;
}
"""


def test_copies_in_flight_are_counted_as_they_are_issued(tmp_path):
    """The producer of the tiled decode leaves its loop only with its copies into shared memory done:
    the count behind that wait is what gives a copy its slot."""
    csrc = os.path.join(ROOT, "llm-inference_b200", "csrc")
    exe = str(tmp_path / "slots")
    res = subprocess.run(["g++", "-std=c++17", "-x", "c++", "-", "-o", exe, f"-I{csrc}"], input=SLOT_PAIR,
                         capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    assert subprocess.run([exe]).returncode == 0
