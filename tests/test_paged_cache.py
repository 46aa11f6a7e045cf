"""PagedKVCache: its layout and refusals on the CPU, its operations on the GPU
against the host model, and the C++ class of the same name."""
import os
import subprocess

import numpy as np
import pytest

import b200attn
from _paged import Pages, assert_within, attend64, rows_of
from _util import ROOT, seeded_f16


def test_layout():
    c = b200attn.PagedKVCache(3, 10, 16, 4, 8, 5, 7, device="cpu")
    base, plane = c.buffer.data_ptr(), 10 * 16 * 32 * 2
    for layer in range(3):
        assert c.get_k_pages(layer).data_ptr() == base + 2 * layer * plane
        assert c.get_v_pages(layer).data_ptr() == base + (2 * layer + 1) * plane
        assert c.get_k_pages(layer).shape == (10, 16, 32)
    k, v, stride, pages, ps, table, width, rows = c.pages(1)
    assert (stride, pages, ps, width, rows) == (0, 10, 16, 7, 5) and table is c.page_table
    assert c.page_table.eq(-1).all() and c.seq_len.eq(0).all() and c.ref_count.eq(0).all()
    with pytest.raises(ValueError):
        b200attn.PagedKVCache(1, (1 << 21) + 1, 1, 1, 8, 1, 1, device="meta")
    with pytest.raises(ValueError):      # host tensors are refused before anything is launched
        c.extend(c.seq_len, c.seq_len)
    assert c.check() == 0
    c.status[0] = 1
    with pytest.raises(MemoryError):
        c.check()
    c.status[0] = 2
    with pytest.raises(ValueError):
        c.check()


def _short_wide_and_strided(ints):
    import torch
    return ints([1]), ints([1, 2]).to(torch.int64), ints([1, 0, 2, 0])[::2]


def _refuses_arrays(c, ints):
    two = ints([0, 1])
    for bad in _short_wide_and_strided(ints):
        for call in (lambda: c.extend(two, bad), lambda: c.extend(two, two, bad), lambda: c.truncate(two, bad),
                     lambda: c.fork(two, bad), lambda: c.fork(two, two, bad), lambda: c.copy_pages(two, bad)):
            with pytest.raises(ValueError, match="contiguous int32"):
                call()
    for bad in _short_wide_and_strided(ints)[1:]:
        for call in (lambda: c.extend(bad, two), lambda: c.truncate(bad), lambda: c.fork(bad, two),
                     lambda: c.copy_pages(bad, two)):
            with pytest.raises(ValueError, match="contiguous int32"):
                call()


def test_arrays_that_the_kernels_would_misread_are_refused():
    import torch
    _refuses_arrays(b200attn.PagedKVCache(1, 4, 16, 1, 8, 2, 2, device="cpu"),
                    lambda x: torch.tensor(x, dtype=torch.int32))


@pytest.mark.gpu
def test_arrays_and_devices_are_checked_on_the_gpu(cuda, monkeypatch):
    import torch
    c = b200attn.PagedKVCache(1, 4, 16, 1, 8, 2, 2)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")
    _refuses_arrays(c, ints)
    with pytest.raises(ValueError, match="contiguous int32"):
        c.extend(ints([0, 1]), torch.tensor([1, 1], dtype=torch.int32))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    for call in (c.compact, lambda: c.truncate(ints([0])), lambda: c.copy_pages(ints([0]), ints([1]))):
        with pytest.raises(ValueError, match="current device"):
            call()
    assert c.page_table.eq(-1).all() and c.seq_len.eq(0).all() and c.ref_count.eq(0).all()


def test_native_calls_refuse_what_they_cannot_pass():
    import torch
    f = b200attn.launch_kv_pages_copy
    host = torch.zeros(8, dtype=torch.int32)
    with pytest.raises(ValueError):
        f(0x1000, 1, 0, 1, 0, 8, host, 0x1000, 1)
    with pytest.raises(TypeError):
        f(0x1000, 1, 0, 1, 0, 8, "pages", 0x1000, 1)
    with pytest.raises(TypeError):
        f(0x1000, 1.5, 0, 1, 0, 8, 0x1000, 0x1000, 1)
    with pytest.raises(OverflowError):
        f(0x1000, -1, 0, 1, 0, 8, 0x1000, 0x1000, 1)
    with pytest.raises(AttributeError):
        f(0x1000, 1, 0, 1, 0, 8, 0x1000, 0x1000, 1, stream="default")
    f(0x1000, 1, 0, 1, 0, 8, 0x1000, 0x1000, 0)           # nothing to do


class _Elsewhere:
    """A tensor of a device that is not the current one, as far as a call looks at it."""
    is_cuda = True

    def get_device(self):
        return 63

    def data_ptr(self):
        return 0x1000


def test_native_calls_refuse_tensors_of_another_device():
    """With no items, so that nothing runs either way."""
    a, x = 0x1000, _Elsewhere()
    for call in (lambda: b200attn.launch_kv_pages_copy(a, 1, 0, 1, 0, 8, a, x, 0),
                 lambda: b200attn.launch_kv_pages_truncate(x, 1, 1, 1, 1, a, a, a, a, 0, a, a, 0),
                 lambda: b200attn.launch_rope_and_store_kv_paged(x, a, a, a, a, 0, 1, 1, a, 1, 1, a, a, a, 1, 0, 1, 1, 8, 0,
                                                                 0, a, True),
                 lambda: b200attn.launch_causal_attention_decode_paged(a, 0, a, x, 0, 1, 1, a, 1, 1, a, a, 0, a, 0, 0, 1, 1,
                                                                       8, a, 0)):
        with pytest.raises(ValueError, match="device 63"):
            call()


@pytest.mark.gpu
def test_native_calls_on_the_current_device(cuda):
    import torch
    t = torch.zeros(8, dtype=torch.int32, device="cuda")
    assert b200attn.lib().b2_current_device() == torch.cuda.current_device() == t.get_device()
    b200attn.launch_kv_pages_copy(t, 1, 0, 1, 0, 8, t, t, 0)
    test_native_calls_refuse_tensors_of_another_device()


def test_cpp_class_compiles():
    src = ('#include "b200attn/paged_kv_cache.hpp"\n'
           'int main() { return sizeof(b200attn::PagedKVCache) == 0 || &b200attn::PagedKVCache::compact == nullptr; }\n')
    res = subprocess.run(["g++", "-std=c++20", "-fsyntax-only", "-x", "c++", "-", f"-I{ROOT}/include",
                          "-I/usr/local/cuda/include"], input=src, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    assert os.path.exists(os.path.join(ROOT, "include", "b200attn", "paged_kv_cache.hpp"))


CPP_USE = r"""
#include <cstdio>
#include <vector>
#include "b200attn/paged_kv_cache.hpp"

#define EXPECT(x) do { if (!(x)) { std::printf("failed: %s\n", #x); return 1; } } while (0)

int main() {
    cudaStream_t s;   // does not wait for the default stream
    B2_CUDA_CHECK(cudaStreamCreateWithFlags(&s, cudaStreamNonBlocking));
    const b2_stream_t st = reinterpret_cast<b2_stream_t>(s);
    int32_t* d;       // seqs, counts, positions, one source page, one destination
    B2_CUDA_CHECK(cudaMalloc(&d, 8 * sizeof(int32_t)));
    const int32_t args[8] = {2, 0, 20, 5, -9, -9, 0, 9};
    B2_CUDA_CHECK(cudaMemcpy(d, args, sizeof(args), cudaMemcpyHostToDevice));
    b200attn::PagedKVCache c({2, 300000, 16, 1, 8, 4, 4});
    EXPECT(c.extend(d, d + 2, 2, d + 4, st) == B2_OK);
    EXPECT(c.copy_pages(d + 6, d + 7, 1, st) == B2_OK);
    EXPECT(c.truncate(d, nullptr, 1, st) == B2_OK);
    EXPECT(c.compact(st) == B2_OK);
    B2_CUDA_CHECK(cudaStreamSynchronize(s));
    int32_t table[16], len[4], status[2], pos[2];
    B2_CUDA_CHECK(cudaMemcpy(table, c.page_table(), sizeof(table), cudaMemcpyDeviceToHost));
    B2_CUDA_CHECK(cudaMemcpy(len, c.seq_len(), sizeof(len), cudaMemcpyDeviceToHost));
    B2_CUDA_CHECK(cudaMemcpy(status, c.status(), sizeof(status), cudaMemcpyDeviceToHost));
    B2_CUDA_CHECK(cudaMemcpy(pos, d + 4, sizeof(pos), cudaMemcpyDeviceToHost));
    EXPECT(status[0] == B2_PAGES_OK && status[1] == 1 && pos[0] == 0 && pos[1] == 0);
    for (int i = 0; i < 4; ++i) EXPECT(len[i] == (i == 0 ? 5 : 0));
    for (int i = 0; i < 16; ++i) EXPECT(table[i] == (i == 0 ? 0 : -1));
    EXPECT(b2_device_error_word() == 0);
    B2_CUDA_CHECK(cudaFree(d));
    B2_CUDA_CHECK(cudaStreamDestroy(s));
    return 0;
}
"""


def _build_cpp_use(tmp_path):
    exe, lib = str(tmp_path / "use"), os.path.dirname(b200attn._lib.LIB_PATH)
    res = subprocess.run(["g++", "-std=c++20", "-x", "c++", "-", "-o", exe, f"-I{ROOT}/include",
                          "-I/usr/local/cuda/include", f"-L{lib}", "-lb200attn", f"-Wl,-rpath,{lib}",
                          "-L/usr/local/cuda/lib64", "-lcudart"], input=CPP_USE, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    return exe


def test_cpp_class_links(tmp_path):
    _build_cpp_use(tmp_path)


@pytest.mark.gpu
def test_cpp_class_on_a_non_blocking_stream(cuda, tmp_path):
    res = subprocess.run([_build_cpp_use(tmp_path)], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0, res.stdout + res.stderr


def _slow(stream, rounds=40):
    """Ordinary work on a stream: some 0.7 ms a round."""
    import torch
    with torch.cuda.stream(stream):
        a = torch.randn(8192, 8192, device="cuda", dtype=torch.bfloat16)
        for _ in range(rounds):
            a = (a @ a).clamp(-1, 1)
    return a


@pytest.mark.gpu
@pytest.mark.parametrize("default", [False, True])
def test_arrays_outlive_a_call_on_another_stream(cuda, default):
    """Arguments dropped while their operation still waits behind slow work on its stream: their
    memory is not given to the next tensors before."""
    import torch

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    warm = b200attn.PagedKVCache(1, 40, 16, 1, 8, 4, 8)     # loading a kernel may wait for the device
    for call in (warm.extend, warm.fork, warm.truncate, warm.copy_pages):
        call(ints([-1]), ints([-1]))
    b200attn.lib().b2_clear_device_error_word()
    c = b200attn.PagedKVCache(1, 40, 16, 1, 8, 4, 8)
    pos = ints([-5, -5])
    side = torch.cuda.default_stream() if default else torch.cuda.Stream()
    stream = None if default else side
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        # (nothing here waits for the side stream: values come by device copies and fills)
        zero, two, three, n0, n1 = (torch.full((1,), v, dtype=torch.int32, device="cuda") for v in (0, 2, 3, 20, 33))
        torch.cat([zero, two])                       # (its kernel is loaded)
        torch.cuda.current_stream().synchronize()
        keep = _slow(side, 300)
        c.extend(torch.cat([zero, two]), torch.cat([n0, n1]), pos, stream=stream)
        c.fork(torch.cat([two]), torch.cat([three]), torch.cat([n0]), stream=stream)
        c.truncate(torch.cat([zero]), torch.cat([three]), stream=stream)
        c.copy_pages(torch.cat([two]), torch.cat([n1]), stream=stream)
        gone = b200attn.PagedKVCache(1, 40, 16, 1, 8, 4, 8)
        gone.extend(zero, n0, stream=stream)
        at = {t.data_ptr() for t in (gone.buffer, gone.page_table, gone.seq_len, gone.ref_count, gone.status, gone._ws)}
        del gone
        others = [torch.full((k,), 1, dtype=torch.int32, device="cuda") for _ in range(16) for k in (1, 2)]
        again = b200attn.PagedKVCache(1, 40, 16, 1, 8, 4, 8)
        assert not at & {t.data_ptr() for t in (again.buffer, again.page_table, again.seq_len, again.ref_count, again.status,
                                                again._ws, *others)}
        torch.cuda.current_stream().synchronize()
        assert not side.query()                      # all of it was still to come
        assert c.check() == 0
    torch.cuda.synchronize()
    assert c.seq_len.tolist() == [3, 0, 33, 20] and pos.tolist() == [0, 0]
    assert torch.equal(c.buffer[:, 33].view(torch.int16), c.buffer[:, 2].view(torch.int16))
    del keep, others


@pytest.mark.gpu
def test_a_new_cache_is_written_before_it_is_used(cuda):
    """Made behind slow work on torch's stream: its table, lengths and counts stand when the constructor returns."""
    import torch
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        keep = _slow(side)
        c = b200attn.PagedKVCache(1, 4, 16, 1, 8, 2, 8)
        assert side.query()
    c.extend(c.seq_len[:1].clone(), torch.ones(1, dtype=torch.int32, device="cuda"), stream=None)
    assert c.check() == 1
    del keep


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["stream", "handle", "default", "graph"])
def test_check_waits_for_the_last_operation(cuda, how):
    """Queued behind slow work on a stream that torch's own does not wait for: its refusal is seen."""
    import torch
    from _gpu import Graph

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    c = b200attn.PagedKVCache(1, 4, 16, 1, 8, 2, 8)
    one, other, few, many, far = ints([0]), ints([1]), ints([3]), ints([100]), ints([1000])
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        if how == "graph":
            g = Graph()
            with g:
                c.extend(one, many, stream=g.stream)
            keep = _slow(g.stream)
            assert int(g.rt.cudaGraphLaunch(g.exec, g.stream.cuda_stream)[0]) == 0
            with pytest.raises(MemoryError, match="takes 7"):
                c.check(g.stream)
            g.close()
            return
        side = torch.cuda.default_stream() if how == "default" else torch.cuda.Stream()
        stream = {"stream": side, "handle": side.cuda_stream, "default": None}[how]
        keep = _slow(side)
        c.extend(one, many, stream=stream)
        c.truncate(one[:0], stream=torch.cuda.Stream())      # no items: not an operation
        with pytest.raises(MemoryError, match="takes 7"):
            c.check()
        keep = _slow(side)
        c.extend(other, few, stream=stream)
        assert c.check() == 1
        keep = _slow(side)
        c.truncate(one, many, stream=stream)
        with pytest.raises(ValueError, match="length out of range"):
            c.check()
        keep = _slow(side)
        c.extend(other, far, stream=stream)
        with pytest.raises(ValueError, match="without a reference"):
            c.check()
        keep = _slow(side)
        c.compact(stream=stream)
        assert c.check() == 1
    del keep


@pytest.mark.gpu
def test_operations(cuda):
    import torch

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    H, KVH, d, ps = 8, 2, 128, 16
    c = b200attn.PagedKVCache(2, 24, ps, KVH, d, 6, 8)
    c.buffer.zero_()
    m = Pages(np.zeros((4, 24, ps * KVH * d), np.float16), 6, 8, ps)
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")

    def same():
        torch.cuda.synchronize()
        for got, want in ((c.page_table, m.table), (c.seq_len, m.len), (c.ref_count, m.ref)):
            np.testing.assert_array_equal(got.cpu().numpy(), want)

    c.extend(ints([2, 0, -1]), ints([50, 7, 3]), pos)
    assert m.extend([2, 0, -1], [50, 7, 3])[0] == m.OK and c.check() == 5 and pos.tolist() == [0, 0, -1]
    c.fork(ints([2]), ints([1]), ints([33]))
    assert m.fork([2], [1], [33]) == m.OK
    c.check()
    same()
    c.extend(ints([1]), ints([1]), pos)
    m.extend([1], [1])
    c.check()
    same()
    # one layer's rows appended and attended through the class's pages
    kv = seeded_f16((34, 2 * KVH * d), 1)
    rows = torch.from_numpy(kv).cuda()
    b200attn.launch_rope_and_store_kv_paged(
        None, rows, rows[:, KVH * d:], *c.pages(1), ints([1] * 34), None, None, 0, 34, 0, KVH, d, 0, 2 * KVH * d,
        ints(list(range(34))), False)
    q = seeded_f16((1, H * d), 2)
    out = torch.empty((1, H * d), dtype=torch.float16, device="cuda")
    n = b200attn.decode_paged_workspace_bytes(1, H, KVH)
    b200attn.launch_causal_attention_decode_paged(
        torch.from_numpy(q).cuda(), 0, *c.pages(1), ints([1]), ints([34]), 0, out, 0, 1, H, KVH, d,
        torch.zeros(n, dtype=torch.uint8, device="cuda"), n)
    want, bound = attend64(q.reshape(H, d), kv[:, :KVH * d].reshape(34, KVH, d), kv[:, KVH * d:].reshape(34, KVH, d), H, KVH)
    assert_within(out.cpu().numpy().reshape(H, d), want, bound)
    c.truncate(ints([2]))
    m.truncate([2])
    c.check()
    c.copy_pages(ints([int(m.table[1, 0])]), ints([23]))
    torch.cuda.synchronize()
    assert torch.equal(c.buffer[:, 23], c.buffer[:, int(m.table[1, 0])])
    c.compact()
    assert c.check() == m.compact()
    same()
    got = rows_of(c.get_k_pages(1).cpu().numpy(), m.table[1], 34, ps)
    np.testing.assert_array_equal(got.view(np.uint16), np.ascontiguousarray(kv[:, :KVH * d]).view(np.uint16))
    c.extend(ints([0, 0]), ints([1, 1]))
    with pytest.raises(ValueError):
        c.check()
    c.extend(ints([0, 3, 4]), ints([100, 128, 128]))
    with pytest.raises(MemoryError):
        c.check()
    same()
    assert b200attn.lib().b2_device_error_word() == 0
