"""Attention with score rules, drafted trees and acceptance at the ends of what their calls allow: streams,
lengths, positions, counts and arguments that the tests beside this file do not reach."""
from __future__ import annotations

import copy

import numpy as np
import pytest

from test_scores import PAIR_HALF, Batch, compare, lineages


def of_streams(b, n):
    """Batch b's first n sequences, on the same cache."""
    c, rows = copy.copy(b), int(b.rows[:n].sum())
    c.cached, c.rows, c.streams, c.q, c.k, c.v = b.cached[:n], b.rows[:n], b.streams[:n], b.q[:rows], b.k[:rows], b.v[:rows]
    return c


@pytest.mark.gpu
@pytest.mark.parametrize("scored", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_first_token_calls_on_a_side_stream_beside_a_busy_default_stream(ptts, cuda, dtype, scored):
    """The merge counters of a cache's first token call, and of one with more rows, are zeros before its rows
    are cut and joined, whatever the default stream has to do. Bounds as for attend_scored's f32 outputs."""
    import torch
    side = torch.cuda.Stream()
    all43 = Batch(ptts, cuda, [5000, 3000, 700] + [900 + 9 * i for i in range(40)], [1] * 43, dtype=dtype, seed=2)
    a = torch.randn(8192, 8192, device=cuda).bfloat16()
    c = torch.empty_like(a)
    got = []
    for b in (of_streams(all43, 3), all43):
        out = torch.empty(len(b.q), 512, device=cuda)
        torch.cuda.synchronize()
        for _ in range(60):  # tens of milliseconds
            torch.mm(a, a, out=c)
        args = (b.kv, 0, b.q, b.k, b.v, b.streams, b.rows)
        ptts.attend_scored(*args, softcap=9.0, out=out, stream=side) if scored else ptts.attend(*args, out=out, stream=side)
        side.synchronize()
        got.append((out.clone(), *b.want(softcap=9.0 if scored else 0.0, half_p=PAIR_HALF)))
    all43.kv.check()
    for out, want, bound in got:
        compare(out, want, bound)


CALLS = {  # name: (cached, rows, tree)
    "tokens": ([5000, 40, 0, 300], [1, 1, 1, 1], False),
    "rows": ([5000, 40, 0, 300], [9, 2, 70, 64], False),
    "prompts": ([500, 40, 0, 300], [200, 129, 300, 7], False),
    "trees": ([5000, 40, 0, 300], [9, 64, 33, 1], True),
}


def attend(ptts, b, tree, **kw):
    args = (b.kv, 0, b.q, b.k, b.v, b.streams, b.rows)
    return ptts.attend_tree(*args, b.parents_dev, **kw) if tree else ptts.attend_scored(*args, **kw)


def device_lengths(b, lengths):
    """The lengths as a caller's replayed graph would leave them: the device's alone."""
    import torch
    torch.cuda.synchronize()
    b.kv.tensors(0)[2][torch.from_numpy(b.streams).long().to(b.cuda)] = torch.tensor(lengths, dtype=torch.int32, device=b.cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("host", [0, 3])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", list(CALLS))
def test_rows_go_by_the_devices_lengths(ptts, cuda, kind, dtype, host):
    """Lengths that moved on the device alone: the rows' places, spans and work are the device's."""
    cached, rows, tree = CALLS[kind]
    b = Batch(ptts, cuda, cached, rows, dtype=dtype, tree=tree, seed=31)
    b.kv.set_lengths(b.streams, [host] * len(cached))
    device_lengths(b, cached)
    out = attend(ptts, b, tree, softcap=20.0, slopes=b.slopes)
    b.kv.check()
    compare(out, *b.want(softcap=20.0, slopes=b.slopes, tree=tree, half_p=PAIR_HALF))
    b.check_rows(tree=tree)


@pytest.mark.gpu
@pytest.mark.parametrize("spans", [False, True])
@pytest.mark.parametrize("past", ["one", "most", "before", "least"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", list(CALLS))
def test_a_device_length_that_does_not_fit_refuses_its_sequence(ptts, cuda, kind, dtype, past, spans):
    """The last stream of the cache and another one: nothing written, zeros, the error word; the rest as ever."""
    import torch
    cached, rows, tree = CALLS[kind]
    b = Batch(ptts, cuda, cached, rows, dtype=dtype, tree=tree, seed=32, spare=0)
    refused = [int(np.argmax(b.streams)), (int(np.argmax(b.streams)) + 1) % 4]  # sequences
    lengths = list(cached)
    for i in refused:
        lengths[i] = {"one": b.capacity - rows[i] + 1, "most": 2 ** 31 - 1, "before": -1, "least": -2 ** 31}[past]
    device_lengths(b, lengths)
    before = [t.clone() for t in b.kv.tensors(0)[:2]]
    first = b.dev(np.zeros(sum(rows), np.int32)) if spans else None
    last = b.dev(np.full(sum(rows), 2 ** 31 - 1, np.int32)) if spans and not tree else None
    out = attend(ptts, b, tree, first=first, **({} if tree else {"last": last}))
    with pytest.raises(ptts.PttsError) as e:
        b.kv.check()
    assert e.value.code == ptts.ERR_DEVICE and "capacity" in e.value.msg and "bounds" not in e.value.msg
    offsets = np.r_[0, np.cumsum(rows)]
    keep = np.ones(sum(rows), bool)
    for i in refused:
        keep[offsets[i]:offsets[i + 1]] = False
        for t, old in zip(b.kv.tensors(0)[:2], before):
            st = int(b.streams[i])
            raw = torch.int16 if dtype == "bf16" else torch.int32
            assert torch.equal(t[st].contiguous().view(raw), old[st].contiguous().view(raw))
    assert (out[torch.from_numpy(~keep)] == 0).all()
    for t in b.kv.tensors(0)[:2]:
        t.copy_(torch.nan_to_num(t))  # so that the oracle has numbers in the refused streams
    kw = {} if last is None else {"first": first.cpu().numpy(), "last": last.cpu().numpy().astype(np.int64)}
    want, bound = b.want(tree=tree, half_p=PAIR_HALF, **kw)
    keep = torch.from_numpy(keep)
    compare(out[keep], want[keep], bound[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("by", [-1, 1, 2])
@pytest.mark.parametrize("times", [1, 60])
def test_accept_refuses_a_stream_whose_device_length_is_another(ptts, cuda, by, times):
    """Also where the device is ahead by just the path's length. `times` 60: a list too long for the parameters."""
    import torch
    n = 4 * times
    b = Batch(ptts, cuda, [10 + i % 7 for i in range(n)], [20] * n, layers=2, seed=33)
    for l in range(2):
        for t in b.kv.tensors(l)[:2]:
            t.copy_(torch.randn(t.shape, device=cuda))
    wrong = [i for i in range(n) if i % 4 == 1]
    lengths = np.array(b.cached)
    lengths[wrong] += by
    device_lengths(b, lengths)
    want = [[t.clone() for t in b.kv.tensors(l)[:2]] for l in range(2)]
    for i, (st, L) in enumerate(zip(b.streams, b.cached)):
        for layer in want if i not in wrong else []:
            for t in layer:
                t[int(st), int(L):int(L) + 2] = t[int(st), [int(L) + 3, int(L) + 7]]
    b.kv.accept(b.streams, [[3, 7]] * n)
    with pytest.raises(ptts.PttsError) as e:
        b.kv.check()
    assert e.value.code == ptts.ERR_DEVICE and "bounds" in e.value.msg
    for l in range(2):
        for t, w in zip(b.kv.tensors(l)[:2], want[l]):
            assert torch.equal(t, w)
    lengths[[i for i in range(n) if i not in wrong]] += 2
    got = b.kv.tensors(0)[2].cpu().numpy()[b.streams]
    np.testing.assert_array_equal(got, lengths)
    # Lengths set on both sides: the next acceptance goes through (the arrivals were left at zero).
    b.kv.set_lengths(b.streams, b.cached)
    b.kv.accept(b.streams, [[0]] * n)
    b.kv.check()
    np.testing.assert_array_equal(b.kv.tensors(0)[2].cpu().numpy()[b.streams], b.cached + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("cached,last", [(20, 9), (6000, 4000), (40000, 39000)])
def test_a_cut_row_far_below_every_score_is_joined(ptts, cuda, dtype, cached, last):
    """Slopes that put every key a row sees below -10^31: the nearest has all the weight, exactly, whether the
    row is one CTA's or cut among many. (Distances differ by 1e28 after f32's rounding of 2^-24 x 6e32.)"""
    import torch
    b = Batch(ptts, cuda, [cached, cached], [1, 1], dtype=dtype, seed=41)
    last = b.dev(np.full(2, last, np.int32))
    out = ptts.attend_scored(b.kv, 0, b.q, b.k, b.v, b.streams, b.rows, last=last, max_period=0.0,
                             slopes=torch.full((8,), 1e28, device=cuda))
    b.kv.check()
    vt = b.kv.tensors(0)[1]
    want = torch.stack([vt[int(st), int(last[0])].float().reshape(512) for st in b.streams])
    assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_an_infinite_value_in_a_tokens_last_key_is_infinite(ptts, cuda, dtype):
    """A token sees itself: an infinity in its value is one in its output, at every place in a chunk of keys."""
    import torch
    cached = list(range(0, 70)) + [700, 2501]
    b = Batch(ptts, cuda, cached, [1] * len(cached), dtype=dtype, seed=42)
    args = (b.kv, 0, b.q, b.k, b.v, b.streams, b.rows)
    clean = ptts.attend_scored(*args, softcap=30.0).reshape(-1, 8, 64).clone()
    b.v[:, :, 3], b.v[:, :, 60] = float("inf"), -float("inf")
    out = ptts.attend_scored(*args, softcap=30.0).reshape(-1, 8, 64)
    b.kv.check()
    rest = [d for d in range(64) if d not in (3, 60)]
    assert torch.equal(out[..., rest], clean[..., rest])
    assert (out[..., 3] == float("inf")).all() and (out[..., 60] == -float("inf")).all()


class Far:
    """One stream whose cached rows end past position 2^24, of which the last 300 and the call's `rows` hold
    numbers; the oracle reads those alone (no rotation, so only differences of positions count)."""

    def __init__(self, ptts, cuda, rows, dtype, tree):
        import torch
        self.start = 16_800_001 - 300
        self.kv = ptts.KvState(1, 1, 16_800_001 + rows, dtype=dtype)
        self.kv.set_lengths([0], [16_800_001])
        kt, vt, _ = self.kv.tensors(0)
        for t in (kt, vt):
            t[0, self.start:] = torch.randn(300 + rows, 8, 64, device=cuda).to(t.dtype)
        b = self.b = Batch(ptts, cuda, [300], [rows], dtype=dtype, tree=tree, spare=0, seed=43)
        b.kv.close()
        b.kv = self
        b.streams = np.zeros(1, np.int32)

    def tensors(self, layer):
        kt, vt, lt = self.kv.tensors(layer)
        return kt[:, self.start:], vt[:, self.start:], lt


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["rows", "trees", "prompts", "tokens", "f32 rows", "f32 trees"])
def test_a_distance_bias_past_2_24_positions(ptts, cuda, kind):
    """Distances of near keys are whole numbers however far both are from 0 (an f32 position past 2^24 is
    even). Bounds as in test_scores.py."""
    import torch
    tree, dtype = kind.endswith("trees"), "f32" if kind.startswith("f32") else "bf16"
    rows = {"tokens": 1, "prompts": 1500}.get(kind, 40)  # 1500: too many blocks for the rows kernel
    far = Far(ptts, cuda, rows, dtype, tree)
    b = far.b
    pos = 300 + (np.array(lineages(b.parents[0])[0]) if tree else np.arange(rows))
    first = (pos - 100).astype(np.int32)
    slopes = torch.tensor([0.5, 0.25, 1.0, 0.125, 0.75, 0.5, 2.0, 0.0625], device=cuda)
    for softcap in (0.0, 30.0):
        for out_dtype in ("bf16", "f32"):
            args = (far.kv, 0, b.q, b.k, b.v, [0], [rows])
            rules = dict(softcap=softcap, slopes=slopes, max_period=0.0)
            at = b.dev(first + np.int32(far.start))
            if tree:
                out = ptts.attend_tree(*args, b.parents_dev, first=at, out_dtype=out_dtype, **rules)
            else:
                out = ptts.attend_scored(*args, first=at, out_dtype=out_dtype, **rules)
            half_out, half_p = b.halves(out_dtype)
            compare(out, *b.want(first=first, tree=tree, half_out=half_out, half_p=half_p, **rules))
    far.kv.check()
    far.kv.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_hundreds_of_thousands_of_trees(ptts, cuda, dtype):
    """One-node trees on empty streams: each node's value, exactly. More than the plan's sum of costs can count
    is refused before anything changes (bf16; the f32 kernel counts no costs)."""
    import torch
    n = 900_000
    kv = ptts.KvState(1, n, 2, dtype=dtype)
    x = torch.randn(n, 8, 64, device=cuda).to(torch.bfloat16 if dtype == "bf16" else torch.float32)
    roots = torch.full((n,), -1, dtype=torch.int32, device=cuda)
    streams, one = np.arange(n, dtype=np.int32), np.ones(n, np.int32)
    out = torch.full((n, 512), 7.0, device=cuda)
    if dtype == "bf16":
        with pytest.raises(ptts.PttsError) as e:
            ptts.attend_tree(kv, 0, x, x, x, streams, one, roots, out=out)
        assert e.value.code == ptts.ERR_UNSUPPORTED
        assert (out == 7.0).all() and not kv.tensors(0)[1].any()
        n = 800_000
    ptts.attend_tree(kv, 0, x[:n], x[:n], x[:n], streams[:n], one[:n], roots[:n], out=out[:n])
    kv.check()
    assert torch.equal(out[:n].view(n, 8, 64), x[:n].float()) and torch.equal(kv.tensors(0)[1][:n, 0], x[:n])
    kv.close()


class AnyStream:
    cuda_stream = 0


def refused_by_python(ptts, word, f, *a):
    """Refused with `word` before the library is called (which would say that the handle is NULL)."""
    with pytest.raises(ptts.PttsError) as e:
        f(*a, stream=AnyStream)
    assert e.value.code == ptts.ERR_ARG and word in e.value.msg, e.value


def test_accept_takes_one_path_per_stream(ptts):
    """Streams of another rank or number than the paths: the library would read past the counts. On no device."""
    kv = object.__new__(ptts.KvState)
    kv._h, kv.device = None, 0
    for streams in (np.zeros((2, 2), np.int32), np.zeros((2, 1), np.int32), [[0, 1], [2, 3]], np.int32(3), [0], [0, 1, 2]):
        refused_by_python(ptts, "one path per stream", kv.accept, streams, [[0], [0, 1]])


def test_accepted_nodes_are_whole_numbers(ptts):
    """An index that is not a whole number ([0, 1.5]) is no node; whole ones of any size get to the library, which
    refuses those past 63 (and here says that the handle is NULL). On no device."""
    kv = object.__new__(ptts.KvState)
    kv._h, kv.device = None, 0
    for path in ([0, 1.5], [0.0], np.array([0.0, 1.0]), ["a"], [None], [[0, 1]], np.zeros((2, 2), np.int64), 5):
        refused_by_python(ptts, "node", kv.accept, [0], [path])
    for path in ([0, 64], [0, 300], [-1], [0, 2 ** 40], [0, 2 ** 70], [1, 0], np.array([0, 7], np.int64)):
        refused_by_python(ptts, "NULL", kv.accept, [0], [path])


@pytest.mark.gpu
def test_a_call_that_finds_no_memory_fails_alone(ptts, cuda):
    """The next call on another cache is not blamed for it."""
    with pytest.raises(ptts.PttsError) as e:
        ptts.KvState(1, 1, 400_000_000)  # 410 GB of keys
    assert "out of memory" in e.value.msg
    b = Batch(ptts, cuda, [5, 70], [1, 1], seed=44)
    b.kv.set_lengths(b.streams, b.cached)
    out = ptts.attend_scored(b.kv, 0, b.q, b.k, b.v, b.streams, b.rows)
    b.kv.check()
    compare(out, *b.want(half_p=PAIR_HALF))


GROW = r"""
#include <cstdio>
#include <cstdlib>
#include "host.h"
// A device of 100 bytes; a failed call's error stays until it is read.
static size_t used = 0, sizes[64];
static int allocations = 0;
static cudaError_t last = cudaSuccess;
extern "C" {
cudaError_t cudaMalloc(void** p, size_t n) {
    if (n > 100 - used) return last = cudaErrorMemoryAllocation;
    used += n;
    sizes[allocations] = n;
    *p = &sizes[allocations++];
    return cudaSuccess;
}
cudaError_t cudaFree(void* p) { used -= *static_cast<size_t*>(p); return cudaSuccess; }
cudaError_t cudaGetLastError(void) { cudaError_t e = last; last = cudaSuccess; return e; }
cudaError_t cudaDeviceSynchronize(void) { return cudaSuccess; }
const char* cudaGetErrorString(cudaError_t) { return "out of memory"; }
cudaError_t cudaMemsetAsync(void*, int, size_t, cudaStream_t) { return cudaSuccess; }
}
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
int main() {
    ptts::host::DevBuf b;
    CHECK(b.grow(3, 10) && b.bytes == 10 && allocations == 1);
    CHECK(b.grow(10, 10) && allocations == 1);
    CHECK(b.grow(11, 10) && b.bytes == 15 && used == 15);
    CHECK(b.grow(80, 10) && b.bytes == 80 && used == 80);
    CHECK(b.grow(90, 10) && b.bytes == 90 && used == 90);  // 120 are not there, 90 are
    CHECK(last == cudaSuccess);
    const int rc = ptts::host::guarded([&] { b.grow(101, 10); });
    CHECK(rc == PTTS_B200_ERR_CUDA && last == cudaSuccess && b.p == nullptr && b.bytes == 0 && used == 0);
    CHECK(b.grow(40, 10) && b.bytes == 40 && used == 40);
    return 0;
}
"""


def test_scratch_grows_to_what_is_needed_where_half_again_is_not_there(tmp_path):
    """The buffer's growth against a device of 100 bytes, on the CPU."""
    import os
    import shutil
    import subprocess
    from conftest import ROOT
    cxx = shutil.which("g++")
    nvcc = next((c for c in ("/usr/local/cuda/bin/nvcc", shutil.which("nvcc")) if c and os.path.exists(c)), None)
    if not cxx or not nvcc:
        pytest.skip("no C++ compiler or no CUDA headers")
    (tmp_path / "grow.cpp").write_text(GROW)
    dirs = [os.path.join(ROOT, "include"), os.path.join(ROOT, "xn-ptts_b200", "csrc"),
            os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc))), "include")]
    exe = str(tmp_path / "grow")
    r = subprocess.run([cxx, "-std=c++17", *[f"-I{d}" for d in dirs], str(tmp_path / "grow.cpp"), "-o", exe],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout
