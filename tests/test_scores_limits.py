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


# ---- views, outputs, caps, refusals -------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("heads", [8, 16])
def test_a_view_keeps_its_cache(ptts, cuda, heads, which):
    import gc
    import weakref
    kv = ptts.KvState(2, 3, 5, num_heads=heads)
    alive, view = weakref.ref(kv), kv.tensors(1)[which][1:]
    del kv
    gc.collect()
    assert alive() is not None
    view.fill_(3)
    assert (view == 3).all()
    del view
    gc.collect()
    assert alive() is None


@pytest.mark.gpu
@pytest.mark.parametrize("out_dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", list(CALLS))
def test_out_is_written_and_nothing_beside_it(ptts, cuda, kind, dtype, out_dtype):
    import torch
    cached, rows, tree = CALLS[kind]
    a, b = (Batch(ptts, cuda, cached, rows, dtype=dtype, tree=tree, seed=34) for _ in range(2))
    n = sum(rows)
    room = torch.full((n + 4, 512), 7.0, device=cuda, dtype=torch.bfloat16 if out_dtype == "bf16" else torch.float32)
    out = attend(ptts, a, tree, softcap=30.0, out=room[2:n + 2], out_dtype="f32")  # out's own type is what counts
    want = attend(ptts, b, tree, softcap=30.0, out_dtype=out_dtype)
    assert out.data_ptr() == room[2].data_ptr() and torch.equal(room[2:n + 2], want)
    assert (room[:2] == 7).all() and (room[n + 2:] == 7).all()
    a.kv.check(), b.kv.check()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1.0, 30.0])
@pytest.mark.parametrize("cap", [40.5, 50.0, 90.0, 128.0])
@pytest.mark.parametrize("out_dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", ["rows", "prompts", "trees"])
def test_caps_above_40_without_a_bias(ptts, cuda, kind, out_dtype, cap, scale):
    """Caps of the fast tanh that keep maxima, with scores far below the cap and past it. Bounds as in
    test_scores.py: its score term charges the cap 2^-16, above the fast tanh's 3.6e-6 (2^-18)."""
    cached, rows, tree = CALLS[kind]
    b = Batch(ptts, cuda, cached, rows, tree=tree, seed=35, scale=scale)
    out = attend(ptts, b, tree, softcap=cap, out_dtype=out_dtype)
    b.kv.check()
    half_out, half_p = b.halves(out_dtype)
    compare(out, *b.want(softcap=cap, tree=tree, half_out=half_out, half_p=half_p))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_each_refusal_leaves_every_bit(ptts, cuda, dtype):
    """After every refused call: the caches bit for bit, the lengths of both sides, the output."""
    import torch
    b = Batch(ptts, cuda, [5, 9, 0], [2, 1, 1], dtype=dtype, tree=True, seed=20, spare=3)
    st = [int(s) for s in b.streams]
    ring, window = sorted(set(range(6)) - set(st))[:2]
    b.kv.start_ring([ring])
    b.kv.set_window([window], 4)
    raw = torch.int16 if dtype == "bf16" else torch.int32
    bits = lambda: [t.contiguous().view(raw).clone() for t in b.kv.tensors(0)[:2]]  # noqa: E731
    before, lengths = bits(), b.kv.lengths().copy()
    out = torch.full((4, 512), 7.0, device=cuda)
    flat = torch.zeros(4 * 512 + 8, dtype=b.q.dtype, device=cuda)
    ints = torch.zeros(8, dtype=torch.int32, device=cuda)

    def scored(layer=0, q=b.q, k=b.k, v=b.v, streams=st, rows=(2, 1, 1), **kw):
        return ptts.attend_scored(b.kv, layer, q, k, v, streams, list(rows), **{"out": out, **kw})

    def tree(parents, streams=st, rows=(2, 1, 1), **kw):
        return ptts.attend_tree(b.kv, 0, b.q, b.k, b.v, streams, list(rows), parents, out=out, **kw)

    good = b.parents_dev
    calls = [lambda: scored(layer=1), lambda: scored(layer=-1), lambda: scored(streams=[st[0], st[0], st[1]]),
             lambda: scored(streams=[st[0], st[1], 6]), lambda: scored(streams=[st[0], st[1], -1]),
             lambda: scored(rows=(3, 1, 0)), lambda: scored(rows=(5, -1, 0)), lambda: scored(streams=st[:2]),
             lambda: scored(streams=[st[0], st[1], ring]), lambda: scored(streams=[st[0], st[1], window]),
             lambda: scored(k=b.k[:, :3].contiguous(), v=b.v[:, :3].contiguous()), lambda: scored(slopes=b.slopes[:4]),
             lambda: scored(first=ints[:4].long()), lambda: scored(last=ints[::2]), lambda: scored(first=ints[:3]),
             lambda: scored(out=out[:, ::2]), lambda: scored(out=out.half()), lambda: scored(out=out[:3]),
             lambda: scored(q=flat[1:1 + 4 * 512].view(4, 8, 64)), lambda: scored(v=flat[1:1 + 4 * 512].view(4, 8, 64)),
             lambda: scored(out=None, out_dtype="f16"), lambda: scored(slopes=b.slopes.cpu()),
             lambda: tree(None), lambda: tree(good[:3]), lambda: tree(good.long()), lambda: tree(good.cpu()),
             lambda: tree(good, streams=[st[0], st[0], st[1]]), lambda: tree(good, streams=[st[0], st[1], ring]),
             lambda: tree(good, softcap=-2.0), lambda: tree(good, max_period=0.5), lambda: tree(good, first=ints[:3])]
    calls += [lambda c=c: scored(softcap=c) for c in (-1.0, 1e-38, 1e38, float("nan"), float("inf"))]
    calls += [lambda p=p: scored(max_period=p) for p in (1.0, -3.0, float("nan"), float("inf"))]
    calls += [lambda s=s, p=p: b.kv.accept(s, p) for s, p in [
        ([st[0], st[0]], [[0], [0]]), ([st[0]], [[0], [0]]), ([6], [[0]]), ([-1], [[0]]), ([], []), ([st[1]], [[0, b.capacity - 9]]),
        ([st[0], ring], [[0], []]), ([window], [[0]]), ([st[0]], [list(range(65))])]]
    calls += [lambda p=p: b.kv.accept([st[1], st[0]], [[0], p]) for p in ([1, 1], [2, 1], [-1], [0, 64], [0, 1.5])]
    for i, call in enumerate(calls):
        with pytest.raises(ptts.PttsError):
            call()
        assert all(torch.equal(x, y) for x, y in zip(bits(), before)), i
        np.testing.assert_array_equal(b.kv.lengths(), lengths)
        np.testing.assert_array_equal(b.kv.tensors(0)[2].cpu().numpy(), lengths)
        assert (out == 7.0).all(), i
    b.kv.check()


# ---- f32 caches: scores and weights in f32 --------------------------------------------------------------

def small_windows(q, keys, vals, first, last):
    """Per row and head over its keys first..last (f64): out, sum_j w_j |v_j - out| (how far a change of the scores
    moves an element), sum_j w_j |v_j|, and R = sqrt(sum_d (q_d k_d)^2) / 8 of the row's largest (the size of a
    score's partial sums)."""
    import torch
    n, H = q.shape[:2]
    out, away, size, R = (torch.zeros(n, H, 64, dtype=torch.float64) for _ in range(4))
    for r in range(n):
        k, v = keys[first[r]:last[r] + 1].double(), vals[first[r]:last[r] + 1].double()
        x = q[r].double()[None] * k
        w = torch.softmax(x.sum(-1) / 8, 0)[..., None]
        out[r] = (w * v).sum(0)
        away[r] = (w * (v - out[r]).abs()).sum(0)
        size[r] = (w * v.abs()).sum(0)
        R[r] = (x * x).sum(-1).sqrt().amax(0)[:, None] / 8
    return out, away, size, R


def steps_off(got, out, away, size, R):
    """Root mean square of the errors in units of what f32 gives: a score is a sum of 64 products, each rounded
    to half a step (2^-24) of partial sums of size R, so 2^-24 sqrt(64) R at most in the mean; a weight's
    exponential (2 steps of 2^-23), the sums of a few weights and the quotient 2^-22; the output 2^-24."""
    unit = ((away * R * 2.0 ** -21) ** 2 + (size * 2.0 ** -22) ** 2 + (out * 2.0 ** -24) ** 2).sqrt()
    return (((got.double() - out) / unit) ** 2).mean().sqrt().item()


def pair(x):
    """x as two bf16 planes."""
    hi = x.bfloat16().float()
    return hi + (x - hi).bfloat16().float()


@pytest.mark.parametrize("scale,what", [(16.0, "q"), (0.02, "p")])
def test_the_measure_tells_f32_from_bf16_pairs(scale, what):
    """f32 arithmetic stays under 1 in the mean, a bf16 pair in place of q (large scores) or of the weights
    (scores near 0) does not: 2^-18 of a value against 2^-21 and 2^-22."""
    import torch
    g = torch.Generator().manual_seed(1)
    n = 200
    q, keys, vals = torch.randn(n, 8, 64, generator=g) * scale, *(torch.randn(n + 3, 8, 64, generator=g) for _ in range(2))
    first, last = np.arange(n), np.arange(n) + 3
    want = small_windows(q, keys, vals, first, last)

    def f32(q, p_of):
        out = torch.zeros(n, 8, 64)
        for r in range(n):
            s = torch.einsum("hd,thd->th", q[r], keys[r:r + 4]) / 8
            e = torch.exp(s - s.amax(0))
            out[r] = torch.einsum("th,thd->hd", p_of(e), vals[r:r + 4]) / e.sum(0)[:, None]
        return steps_off(out, *want)

    assert f32(q, lambda p: p) < 0.7
    assert f32(pair(q) if what == "q" else q, pair if what == "p" else (lambda p: p)) > 1.4


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [16.0, 0.02])
@pytest.mark.parametrize("kind", ["tokens", "prompts", "trees"])
def test_f32_caches_hold_scores_and_weights_in_f32(ptts, cuda, kind, scale):
    """Windows of 4 keys, so that long sums do not hide what a pair of bf16s would lose; a tree of one chain is a
    prompt. Under 1 in the units of steps_off."""
    rows = {"tokens": [1] * 150, "prompts": [70, 33], "trees": [64, 40]}[kind]
    cached = [3 + 7 * i % 90 for i in range(len(rows))]
    b = Batch(ptts, cuda, cached, rows, dtype="f32", tree=kind == "trees", seed=36, scale=scale,
              parents=[list(range(-1, n - 1)) for n in rows])
    pos = np.concatenate(b.positions())
    out = attend(ptts, b, kind == "trees", first=b.dev((pos - 3).astype(np.int32)), max_period=0.0)
    b.kv.check()
    off, at = [], 0
    kt, vt, _ = b.kv.tensors(0)
    for st, L, n in zip(b.streams, b.cached, b.rows):
        p = np.arange(L, L + n)
        want = small_windows(b.q[at:at + n].cpu(), kt[int(st)].cpu(), vt[int(st)].cpu(), p - 3, p)
        off.append(steps_off(out[at:at + n].cpu().reshape(n, 8, 64), *want) ** 2 * n)
        at += n
    assert (sum(off) / at) ** 0.5 < 1.0


# ---- keys that a row does not see ---------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("what", [30.0, -1e3, float("inf"), float("nan")])
@pytest.mark.parametrize("rule", [{}, {"softcap": 30.0}, {"softcap": 50.0}, {"softcap": 50.0, "slopes": True}, {"softcap": 200.0},
                                  {"softcap": 0.5}], ids=str)
@pytest.mark.parametrize("dtype,out_dtype", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("kind", ["prompts", "rows", "tokens", "trees"])
def test_keys_that_a_row_does_not_see_change_no_bit_of_it(ptts, cuda, kind, dtype, out_dtype, rule, what):
    """Two documents in a stream (a tree: a node beside the others): the first one's keys and values, the call's
    own among them, and the slots behind the call's rows are replaced; the second one's rows keep their bits."""
    import torch
    cached, rows, tree = {"prompts": (200, 150, False), "rows": (3000, 40, False), "tokens": (900, 1, False),
                          "trees": (700, 30, True)}[kind]
    cut = {"prompts": 237, "rows": 3011, "tokens": 333, "trees": 411}[kind]  # where the second document begins
    parents = [[-1] + [0 if i < 8 else i - 7 for i in range(1, rows)]]  # node 5: its line is 5, 12, 19, 26
    outs = []
    for changed in (False, True):
        b = Batch(ptts, cuda, [cached], [rows], dtype=dtype, tree=tree, parents=parents, seed=51)
        line = {i for i, l in enumerate(lineages(parents[0])[1]) if 5 in l} if tree else set()
        pos = cached + (np.array(lineages(parents[0])[0]) if tree else np.arange(rows))
        if tree:
            keep, first = [i for i in range(rows) if i not in line], np.full(rows, cut)
        else:
            keep, first = [i for i in range(rows) if pos[i] >= cut], np.where(pos >= cut, cut, 0)
        kt, vt, _ = b.kv.tensors(0)
        st = int(b.streams[0])
        kt[st, cached:], vt[st, cached:] = 0.0, 0.0
        if changed:
            for t in (kt, vt):
                t[st, :min(cut, cached)] *= what
                t[st, cached + rows:] = what
            away = [5] if tree else [i for i in range(rows) if pos[i] < cut]
            for t in (b.k, b.v):
                t[away] *= what
        slopes = b.slopes if rule.get("slopes") else None
        args = dict(softcap=rule.get("softcap", 0.0), slopes=slopes, first=b.dev(first.astype(np.int32)), out_dtype=out_dtype)
        outs.append(attend(ptts, b, tree, **args)[keep].clone())
        b.kv.check()
    assert torch.isfinite(outs[0]).all() and torch.equal(outs[0], outs[1])


@pytest.mark.gpu
@pytest.mark.parametrize("size", [2.0 ** -35, 2.0 ** 70, 2.0 ** 100])
@pytest.mark.parametrize("cap,to", [(20.0, 1), (20.0, -1), (32.0, 1), (32.0, -1), (40.0, 1), (40.0, -1), (50.0, 1), (0.0, 1)])
@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("kind", ["rows", "prompts", "trees", "tokens"])
def test_values_of_any_size(ptts, cuda, kind, slopes, cap, to, size):
    """Values far from 1 beside scores at the cap (to: at its upper or lower end): finite, and in bounds relative to
    the values (test_scores.py's; its weights are relative too)."""
    import torch
    cached, rows, tree = CALLS[kind]
    b = Batch(ptts, cuda, cached, rows, tree=tree, seed=52)
    kt, vt, _ = b.kv.tensors(0)
    common = torch.randn(8, 64, device=cuda)  # in every q and key: scores of about `to` x 100
    b.q.copy_(b.q * 0.2 + common * 10), b.k.copy_(b.k * 0.2 + common * to)
    kt.copy_(kt * 0.2 + common * to), vt.mul_(size), b.v.mul_(size)
    rules = dict(softcap=cap, slopes=b.slopes if slopes else None, max_period=0.0)
    out = attend(ptts, b, tree, out_dtype="bf16", **rules)
    b.kv.check()
    want, bound = b.want(tree=tree, half_out=2.0 ** -8, half_p=2.0 ** -8, **rules)
    compare(out / size, want / size, bound / size)


@pytest.mark.gpu
@pytest.mark.parametrize("out_dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,tree", [(1, False), (1, True), (2, False), (2, True), (64, True), (130, False)])
def test_a_cache_of_one_stream_filled_by_one_call(ptts, cuda, rows, tree, dtype, out_dtype):
    """No slot beside the call's own rows; one-key rows give the key's value."""
    import torch
    kv = ptts.KvState(1, 1, rows, dtype=dtype)
    t = torch.bfloat16 if dtype == "bf16" else torch.float32
    q, k, v = (torch.randn(rows, 8, 64, device=cuda).to(t) for _ in range(3))
    args = (kv, 0, q, k, v, [0], [rows])
    rules = dict(softcap=30.0, slopes=torch.full((8,), 0.5, device=cuda), out_dtype=out_dtype)
    if tree:  # roots: each sees itself
        out = ptts.attend_tree(*args, torch.full((rows,), -1, dtype=torch.int32, device=cuda), **rules)
        assert torch.equal(out.view(rows, 8, 64), v.to(out.dtype))
    else:
        out = ptts.attend_scored(*args, **rules)
        # bf16 outputs of prompts: a weight rounded to bf16 (2^-8) over its sum in f32, then the output's rounding
        # (2^-8, of what that left). Else the weight is 1, exactly.
        slack = (1 + 2.0 ** -8) ** 2 - 1 if rows > 1 and dtype == out_dtype == "bf16" else 0.0
        want = v[0].to(out.dtype).double()
        assert ((out[0].view(8, 64).double() - want).abs() <= slack * want.abs()).all()
        assert torch.isfinite(out).all()
    kv.check()
    with pytest.raises(ptts.PttsError):
        kv.advance([0], [rows + 1])
    kv.accept([0], [list(range(min(rows, 64)))])
    kv.check()
    assert kv.lengths()[0] == min(rows, 64) and torch.equal(kv.tensors(0)[1][0].to(t), v)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,out_dtype", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("kind", list(CALLS))
def test_the_same_call_gives_the_same_bits(ptts, cuda, kind, dtype, out_dtype):
    import torch
    cached, rows, tree = CALLS[kind]
    b = Batch(ptts, cuda, [c + 2000 for c in cached], rows, dtype=dtype, tree=tree, seed=53)
    for rules in ({}, {"softcap": 30.0}, {"softcap": 50.0, "slopes": b.slopes}):
        outs = [attend(ptts, b, tree, out_dtype=out_dtype, **rules).clone() for _ in range(5)]
        assert all(torch.equal(o, outs[0]) for o in outs)
    b.kv.check()


@pytest.mark.gpu
def test_caches_on_streams_of_their_own_at_once(ptts, cuda):
    """Four caches, each with another kernel's call on its own stream, several times over without a wait: the bits
    of the same calls one after another."""
    import torch
    jobs = [(Batch(ptts, cuda, *CALLS[k][:2], dtype=dtype, tree=CALLS[k][2], seed=54 + i), CALLS[k][2])
            for i, (k, dtype) in enumerate([("prompts", "bf16"), ("trees", "bf16"), ("tokens", "bf16"), ("prompts", "f32")])]
    rules = dict(softcap=30.0, out_dtype="bf16")
    alone = [attend(ptts, b, tree, **rules) for b, tree in jobs]
    outs = [[torch.empty_like(a) for _ in range(20)] for a in alone]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for i in range(20):
        for (b, tree), s, o in zip(jobs, streams, outs):
            attend(ptts, b, tree, **{**rules, "out": o[i], "stream": s})
    torch.cuda.synchronize()
    for (b, _), a, o in zip(jobs, alone, outs):
        b.kv.check()
        assert all(torch.equal(x, a) for x in o)
