"""Attention with score rules (attend_scored), drafted trees (attend_tree) and their acceptance
(KvState.accept) against the definition in 64 bits.

The oracle reads the cache the call left (its own rows are checked apart, in `check_rows`), rotates
q by the f32 angles in f64, and bounds each output element by the roundings on its way:
    |out - want| <= A * (r_out + 2 (r_p + S r_s + r_e))
with A = sum_j w_j |v_j| (the largest a relative change of the weights can move the element), r_out
half a step of the output type, r_p half a step of the type the weights are held in for P.V, S r_s
the error of a score: S = max_j (sum_d |q_d k_jd| / 8 + |softcap| + |bias|) in log2 units, r_s half a
step of the q operand's hi/lo pair (2 bf16 planes: 2^-17, doubled for the keys' f32 products), and
r_e 2^-18 for the exponentials and the f32 sums of up to 2^5 tiles of 2^7 keys (2^-23 a step, 2^5
steps). The factor 2 is the quotient: the weights' sum moves as much as the weights. Half a step of
f32 (2^-24) is far below each and left to r_e.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

LOG2E = 1.4426950408889634
BF16_HALF, PAIR_HALF = 2.0 ** -8, 2.0 ** -16


# ---- the oracle --------------------------------------------------------------------------------

def inv_freq(max_period):
    return [np.float32(1) / np.float32(max_period ** (i / 32.0)) for i in range(32)]


def rotate64(x, pos, max_period):
    """x [n, heads, 64] (any float), rotated in f64 at the f32 angles."""
    import torch
    x = x.double()
    if not max_period:
        return x
    f = torch.tensor(np.array(inv_freq(max_period), np.float32), device=x.device)
    a = (pos.to(x.device).float()[:, None] * f[None]).double()[:, None]
    c, s = a.cos(), a.sin()
    e, o = x[..., 0::2], x[..., 1::2]
    return torch.stack((e * c - o * s, e * s + o * c), -1).flatten(-2)


def lineages(parents):
    depth, line = [], []
    for i, p in enumerate(parents):
        depth.append(0 if p < 0 else depth[p] + 1)
        line.append([i] + ([] if p < 0 else line[p]))
    return depth, line


class Batch:
    """A cache with random rows and NaN in every slot no row may read, and a call's inputs."""

    def __init__(self, ptts, cuda, cached, rows, *, heads=8, kv_heads=None, dtype="bf16", in_dtype=None, seed=0,
                 layers=1, spare=2, scale=2.0, tree=False, parents=None):
        import torch
        g = torch.Generator(device=cuda).manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.ptts, self.cuda, self.heads, self.dtype = ptts, cuda, heads, dtype
        self.cached, self.rows = np.array(cached, np.int32), np.array(rows, np.int32)
        S = len(cached) + spare
        self.streams = rng.permutation(S)[:len(cached)].astype(np.int32)
        self.capacity = int((self.cached + self.rows).max()) + 3
        self.kv = ptts.KvState(layers, S, self.capacity, num_heads=heads, dtype=dtype)
        for l in range(layers):
            for t in self.kv.tensors(l)[:2]:
                t.copy_(torch.randn(t.shape, generator=g, device=cuda))
                for st, L in zip(self.streams, self.cached):
                    t[st, L:] = float("nan")
        self.kv.set_lengths(self.streams, self.cached)
        n = int(self.rows.sum())
        t = torch.bfloat16 if (in_dtype or dtype) == "bf16" else torch.float32
        KVH = kv_heads or heads
        self.q = (torch.randn(n, heads, 64, generator=g, device=cuda) * scale).to(t)
        self.k, self.v = (torch.randn(n, KVH, 64, generator=g, device=cuda).to(t) for _ in range(2))
        self.slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], device=cuda)
        if tree:
            self.parents = parents or [[-1 if i == 0 or rng.random() < 0.1 else int(rng.integers(max(0, i - 9), i))
                                        for i in range(r)] for r in self.rows]
            self.parents_dev = torch.tensor(sum(self.parents, []), dtype=torch.int32, device=cuda)

    def positions(self):
        return [np.arange(L, L + n) for L, n in zip(self.cached, self.rows)]

    def spans(self, mask, seed=5):
        """(first, last) int32 arrays over all rows, or None."""
        rng = np.random.default_rng(seed)
        first, last = [], []
        for L, n in zip(self.cached, self.rows):
            p = np.arange(L, L + n)
            end = int(L + n)
            if mask == "causal":
                return None, None
            if mask == "prefix":
                pre = int(rng.integers(1, end + 1))
                first.append(np.zeros(n)), last.append(np.maximum(p, pre - 1))
            elif mask == "documents":
                cuts = np.unique(np.r_[0, rng.integers(0, end, 4)])
                f = cuts[np.searchsorted(cuts, p, side="right") - 1]
                f[n - n // 5:] = p[n - n // 5:] + 1  # padding rows see nothing
                first.append(f), last.append(p)
            elif mask == "window":
                first.append(p - int(rng.integers(1, end + 1)) + 1), last.append(p)
            elif mask == "wild":  # anything, past both ends and back to front
                first.append(rng.integers(-5, end + 5, n)), last.append(rng.integers(-5, end + 5, n))
            elif mask == "extremes":  # the type's ends
                first.append(np.full(n, -2 ** 31)), last.append(np.where(np.arange(n) % 2, 2 ** 31 - 1, -2 ** 31))
        return np.concatenate(first).astype(np.int32), np.concatenate(last).astype(np.int32)

    def dev(self, a):
        import torch
        return None if a is None else torch.from_numpy(a).to(self.cuda)

    def want(self, layer=0, *, first=None, last=None, softcap=0.0, slopes=None, max_period=10000.0, tree=False,
             half_out=0.0, half_p=0.0):
        """(out, bound) in f64 [rows, H * 64], from the cache as it is now."""
        import torch
        kt, vt, _ = self.kv.tensors(layer)
        outs, bounds, at = [], [], 0
        H = self.heads
        for i, (st, L, n) in enumerate(zip(self.streams, self.cached, self.rows)):
            mine = slice(at, at + n)
            end = int(L + n)
            j = torch.arange(end, device=self.cuda)
            if tree:
                depth, line = lineages(self.parents[i])
                pos = torch.tensor([int(L) + d for d in depth], device=self.cuda)
                where = torch.cat([j[:int(L)], pos])
                seen = torch.zeros(n, end, dtype=torch.bool)
                seen[:, :L] = True
                for r, ln in enumerate(line):
                    seen[r, [int(L) + a for a in ln]] = True
                seen = seen.to(self.cuda)
                if first is not None:
                    seen &= where[None] >= torch.from_numpy(first[mine]).to(self.cuda)[:, None]
            else:
                pos = torch.arange(int(L), end, device=self.cuda)
                where = j
                f = torch.from_numpy(first[mine].astype(np.int64)).to(self.cuda) if first is not None else torch.zeros_like(pos)
                t = torch.from_numpy(last[mine].astype(np.int64)).to(self.cuda) if last is not None else pos
                seen = (j[None] >= f[:, None]) & (j[None] <= t[:, None])
            q = rotate64(self.q[mine], pos, max_period)
            keys, vals = (c[int(st), :end].reshape(end, H, 64).double() for c in (kt, vt))
            any_seen = seen.any(0)
            keys, vals = (torch.where(any_seen[:, None, None], c, 0.0) for c in (keys, vals))
            u = torch.einsum("rhd,thd->hrt", q, keys) / 8
            size = torch.einsum("rhd,thd->hrt", q.abs(), keys.abs()) / 8
            if softcap:
                u = softcap * torch.tanh(u / softcap)
                size = size + softcap
            if slopes is not None:
                bias = slopes.double()[:, None, None] * (pos[:, None] - where[None]).abs().double()[None]
                u, size = u - bias, size + bias.abs()
            u = u.masked_fill(~seen[None], -math.inf)
            w = torch.exp(u - u.amax(-1, keepdim=True).clamp(min=-1e300))
            w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
            # a weight below 2^-30 of the sum moves nothing by its score's error
            S = torch.where(seen[None] & (w > 2.0 ** -30), size, 0.0).amax(-1) * LOG2E
            A = torch.einsum("hrt,thd->rhd", w, vals.abs())
            rel = half_out + 2 * (half_p + S * PAIR_HALF + 2.0 ** -18)
            outs.append(torch.einsum("hrt,thd->rhd", w, vals).reshape(n, H * 64))
            bounds.append((A * rel.T[..., None] + 1e-30).reshape(n, H * 64))
            at += n
        return torch.cat(outs), torch.cat(bounds)

    def check_rows(self, layer=0, *, max_period=10000.0, tree=False):
        """The call's own cache rows: v exactly (rounded once), k within half a step of the f64
        rotation plus the f32 rotation's own error (two products, a sum, sincosf's 2 steps: 2^-21)."""
        import torch
        kt, vt, _ = self.kv.tensors(layer)
        at, g = 0, self.heads // self.k.shape[1]
        half = BF16_HALF if self.dtype == "bf16" else 2.0 ** -24
        for i, (st, L, n) in enumerate(zip(self.streams, self.cached, self.rows)):
            pos = torch.arange(int(L), int(L + n), device=self.cuda)
            if tree:
                pos = torch.tensor([int(L) + d for d in lineages(self.parents[i])[0]], device=self.cuda)
            k = rotate64(self.k[at:at + n], pos, max_period).repeat_interleave(g, 1)
            v = self.v[at:at + n].repeat_interleave(g, 1)
            got_k, got_v = (c[int(st), int(L):int(L + n)].reshape(n, self.heads, 64) for c in (kt, vt))
            big = self.k[at:at + n].double().repeat_interleave(g, 1).reshape(n, self.heads, 32, 2).abs().sum(-1)
            big = big.repeat_interleave(2, -1)
            assert ((got_k.double() - k).abs() <= k.abs() * half + big * 2.0 ** -21 * (1 + half)).all()
            assert torch.equal(got_v, v.to(got_v.dtype))
            at += n

    def halves(self, out_dtype):
        """(r_out, r_p): bf16 outputs may hold the weights in bf16 for P.V, f32 ones in a hi/lo pair."""
        return (BF16_HALF, BF16_HALF) if out_dtype == "bf16" else (0.0, PAIR_HALF)


def compare(got, want, bound):
    import torch
    got = got.double()
    assert torch.isfinite(got).all()
    over = (got - want).abs() / bound
    assert over.max().item() <= 1.0, f"{over.max().item():.3f} of the bound at {int(over.argmax())}"


# ---- prompts and tokens --------------------------------------------------------------------------

SHAPES = {  # name: (cached, rows)
    "one_key": ([0], [1]),
    "tokens": ([0, 1, 31, 32, 33, 700, 2500], [1] * 7),
    "tokens_many": ([(i * 37) % 260 for i in range(301)], [1] * 301),
    "mixed": ([0, 5, 129, 600], [3, 1, 64, 17]),
    "short_rows_long_cache": ([4000, 1], [5, 63]),
    "prompt_tiles": ([0, 0, 7], [128, 129, 255]),
    "prompt_keys": ([0, 130, 1], [65, 300, 127]),
    "prompt_long": ([100], [1100]),
    "rows_over_long_cache": ([5000], [70]),
    "beside_a_prompt": ([6000, 3000, 0], [1, 40, 200]),
    "long_list": ([(i * 29) % 90 for i in range(400)], [1 + i % 2 for i in range(400)]),
}
RULES = {
    "plain": {},
    "cap": {"softcap": 20.0},
    "small_cap": {"softcap": 0.5},
    "big_cap": {"softcap": 3e4},
    "bias": {"slopes": True, "max_period": 0.0},
    "cap_bias": {"softcap": 50.0, "slopes": True},
    "cap_rising_bias": {"softcap": 30.0, "slopes": -0.25},
    "rising_bias": {"slopes": -1.0},
}


def call(b, rule, mask="causal", out_dtype="f32", layer=0, **kw):
    first, last = b.spans(mask)
    args = dict(rule)
    times = float(args.pop("slopes", 0.0))
    slopes = b.slopes * times if times else None
    out = b.ptts.attend_scored(b.kv, layer, b.q, b.k, b.v, b.streams, b.rows, first=b.dev(first), last=b.dev(last),
                               slopes=slopes, out_dtype=out_dtype, **args, **kw)
    half_out, half_p = b.halves(out_dtype)
    want, bound = b.want(layer, first=first, last=last, slopes=slopes, half_out=half_out, half_p=half_p, **args)
    return out, want, bound


@pytest.mark.gpu
@pytest.mark.parametrize("rule", list(RULES))
@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("dtype,out_dtype", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
def test_scored_rules_and_lengths(ptts, cuda, shape, rule, dtype, out_dtype):
    b = Batch(ptts, cuda, *SHAPES[shape], dtype=dtype, seed=len(shape) + len(rule))
    out, want, bound = call(b, RULES[rule], out_dtype=out_dtype)
    b.kv.check()
    compare(out, want, bound)
    b.check_rows(max_period=RULES[rule].get("max_period", 10000.0))


@pytest.mark.gpu
@pytest.mark.parametrize("mask", ["prefix", "documents", "window", "wild", "extremes"])
@pytest.mark.parametrize("shape", ["tokens", "mixed", "short_rows_long_cache", "prompt_tiles", "prompt_keys", "prompt_long",
                                   "beside_a_prompt"])
@pytest.mark.parametrize("dtype,rule", [("bf16", "plain"), ("bf16", "cap"), ("bf16", "bias"), ("bf16", "cap_bias"),
                                        ("bf16", "cap_rising_bias"), ("f32", "cap_bias")])
def test_scored_spans(ptts, cuda, shape, mask, dtype, rule):
    b = Batch(ptts, cuda, *SHAPES[shape], dtype=dtype, seed=len(shape) * 7 + len(mask))
    out, want, bound = call(b, RULES[rule], mask, out_dtype=dtype)
    b.kv.check()
    compare(out, want, bound)
    first, last = b.spans(mask)
    end = np.concatenate([np.full(n, L + n - 1) for L, n in zip(b.cached, b.rows)])
    empty = np.maximum(first, 0) > np.minimum(last, end)
    assert (out.float().cpu().numpy()[empty] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads", [(8, 1), (8, 2), (16, 16), (16, 4), (24, 8)])
@pytest.mark.parametrize("shape", ["tokens", "mixed", "prompt_keys", "beside_a_prompt"])
@pytest.mark.parametrize("dtype,in_dtype", [("bf16", "f32"), ("f32", "bf16"), ("bf16", "bf16")])
def test_scored_heads_and_types(ptts, cuda, shape, heads, kv_heads, dtype, in_dtype):
    b = Batch(ptts, cuda, *SHAPES[shape], heads=heads, kv_heads=kv_heads, dtype=dtype, in_dtype=in_dtype, seed=heads)
    out, want, bound = call(b, RULES["cap_bias"], "window", out_dtype="bf16")
    b.kv.check()
    compare(out, want, bound)
    b.check_rows()


@pytest.mark.gpu
def test_without_rules_it_is_attend(ptts, cuda):
    """No rules: attend's values in the cache bit for bit, its keys but for the last step of a rotation (sine
    and cosine rounded once here, sincosf's there: 2 f32 steps, at most one bf16 step, 2^-7), and its
    outputs within the same bound."""
    import torch
    for shape in ("tokens", "mixed", "prompt_keys"):
        a, b = (Batch(ptts, cuda, *SHAPES[shape], seed=3) for _ in range(2))
        out, want, bound = call(a, {})
        ref = ptts.attend(b.kv, 0, b.q, b.k, b.v, b.streams, b.rows)
        compare(out, want, bound)
        compare(ref, *b.want(half_p=PAIR_HALF))
        (ka, va, la), (kb, vb, lb) = a.kv.tensors(0), b.kv.tensors(0)
        assert torch.equal(torch.nan_to_num(va), torch.nan_to_num(vb)) and torch.equal(la, lb)
        x, y = torch.nan_to_num(ka).double(), torch.nan_to_num(kb).double()
        assert ((x - y).abs() <= 2.0 ** -7 * x.abs() + 2.0 ** -20).all()
        a.check_rows(), b.check_rows()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", ["tokens", "mixed", "prompt_keys", "rows_over_long_cache"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_bad_values_stay_with_the_rows_that_see_them(ptts, cuda, shape, bad, dtype):
    """A key and value that some rows of a tile see and others do not: not finite there, exact here."""
    import torch
    b = Batch(ptts, cuda, *SHAPES[shape], dtype=dtype, seed=9)
    first, last = b.spans("window", seed=2)
    kt, vt, _ = b.kv.tensors(0)
    clean = b.ptts.attend_scored(b.kv, 0, b.q, b.k, b.v, b.streams, b.rows, first=b.dev(first), last=b.dev(last),
                                 out_dtype=dtype)
    marks = []
    for st, L in zip(b.streams, b.cached):
        m = int(L) // 2
        if L:
            vt[int(st), m, ..., 3] = bad
            vt[int(st), m, ..., 60] = -bad
        marks.append(m if L else -1)
    out = b.ptts.attend_scored(b.kv, 0, b.q, b.k, b.v, b.streams, b.rows, first=b.dev(first), last=b.dev(last),
                               out_dtype=dtype)
    b.kv.check()
    mark = torch.tensor(np.repeat(marks, b.rows), device=cuda)
    sees = (mark >= 0) & (mark >= b.dev(first)) & (mark <= b.dev(last))
    dims = out.reshape(len(out), 8, 64)
    assert torch.equal(out[~sees], clean[~sees])
    touched = dims[sees][:, :, [3, 60]]
    assert not torch.isfinite(touched).any()
    rest = [d for d in range(64) if d not in (3, 60)]
    same = (dims[sees][:, :, rest] - clean.reshape(len(out), 8, 64)[sees][:, :, rest]).float()
    assert torch.isfinite(same).all() and same.abs().max().item() == 0.0 if sees.any() else True


@pytest.mark.gpu
def test_large_scores_and_one_sided_weights(ptts, cuda):
    """Scores in the thousands: one key takes all; and equal scores: the mean of the values."""
    import torch
    b = Batch(ptts, cuda, [40, 300], [1, 90], seed=4, scale=400.0)
    out, want, bound = call(b, {}, out_dtype="bf16")
    compare(out, want, bound)
    b = Batch(ptts, cuda, [40, 300], [1, 90], seed=4)
    b.q.zero_()
    out, want, bound = call(b, {}, out_dtype="bf16")
    compare(out, want, bound)


@pytest.mark.gpu
def test_calls_in_a_row_on_another_stream_and_other_layers(ptts, cuda):
    """Calls without a wait between them, on a side stream, growing and shrinking, two layers."""
    import torch
    side = torch.cuda.Stream()
    b = Batch(ptts, cuda, [60, 0, 700], [1, 1, 1], layers=2, seed=6)
    c = Batch(ptts, cuda, [60, 0, 700], [40, 200, 3], layers=2, seed=7)
    side.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(3):
        for layer in (1, 0):
            got.append((b, layer, ptts.attend_scored(b.kv, layer, b.q, b.k, b.v, b.streams, b.rows, softcap=9.0, stream=side)))
            got.append((c, layer, ptts.attend_scored(c.kv, layer, c.q, c.k, c.v, c.streams, c.rows, softcap=9.0, stream=side)))
    torch.cuda.synchronize()
    for x, layer, out in got:
        want, bound = x.want(layer, softcap=9.0, half_p=PAIR_HALF)
        compare(out, want, bound)


# ---- trees -----------------------------------------------------------------------------------------

TREES = {
    "one_node": ([0], [1]),
    "empty_cache": ([0, 0], [64, 7]),
    "batch": ([3, 64, 200, 31, 1000], [16, 17, 64, 1, 33]),
    "long": ([6000, 50], [48, 20]),
    "many": ([(i * 53) % 300 for i in range(260)], [1 + (i * 7) % 64 for i in range(260)]),
    "uneven": ([0, 3000, 1, 2500, 5, 1800] * 7, [64, 1, 33, 64, 2, 17] * 7),
}


@pytest.mark.gpu
@pytest.mark.parametrize("rule", ["plain", "cap", "bias", "cap_bias", "cap_rising_bias"])
@pytest.mark.parametrize("shape", list(TREES))
@pytest.mark.parametrize("dtype,out_dtype", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("windowed", [False, True])
def test_tree(ptts, cuda, shape, rule, dtype, out_dtype, windowed):
    b = Batch(ptts, cuda, *TREES[shape], dtype=dtype, seed=len(shape), tree=True)
    args = dict(RULES[rule])
    times = float(args.pop("slopes", 0.0))
    slopes = b.slopes * times if times else None
    first = None
    if windowed:  # a window of w positions before each node, from none of the cache to all of it
        w = np.repeat([1 + (7 * i) % (int(L) + 9) for i, L in enumerate(b.cached)], b.rows)
        pos = np.concatenate([[L + d for d in lineages(p)[0]] for L, p in zip(b.cached, b.parents)])
        first = (pos - w + 1).astype(np.int32)
    out = ptts.attend_tree(b.kv, 0, b.q, b.k, b.v, b.streams, b.rows, b.parents_dev, first=b.dev(first), slopes=slopes,
                           out_dtype=out_dtype, **args)
    b.kv.check()
    half_out, half_p = b.halves(out_dtype)
    want, bound = b.want(first=first, slopes=slopes, tree=True, half_out=half_out, half_p=half_p, **args)
    compare(out, want, bound)
    b.check_rows(max_period=args.get("max_period", 10000.0), tree=True)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (16, 4)])
def test_tree_heads(ptts, cuda, heads, kv_heads):
    b = Batch(ptts, cuda, *TREES["batch"], heads=heads, kv_heads=kv_heads, tree=True, seed=2)
    out = ptts.attend_tree(b.kv, 0, b.q, b.k, b.v, b.streams, b.rows, b.parents_dev, softcap=30.0, out_dtype="bf16")
    want, bound = b.want(softcap=30.0, tree=True, half_out=BF16_HALF, half_p=BF16_HALF)
    compare(out, want, bound)
    b.check_rows(tree=True)


@pytest.mark.gpu
def test_a_chain_is_a_prompt_and_siblings_do_not_see_each_other(ptts, cuda):
    import torch
    rows = [20, 64]
    chain = [list(range(-1, n - 1)) for n in rows]
    a = Batch(ptts, cuda, [9, 130], rows, tree=True, parents=chain, seed=1)
    b = Batch(ptts, cuda, [9, 130], rows, seed=1)
    x = ptts.attend_tree(a.kv, 0, a.q, a.k, a.v, a.streams, a.rows, a.parents_dev)
    y = ptts.attend_scored(b.kv, 0, b.q, b.k, b.v, b.streams, b.rows)
    want, bound = b.want(half_p=PAIR_HALF)
    compare(x, want, bound)
    compare(y, want, bound)
    # All roots, one of them NaN: the others keep their bits.
    roots = [[-1] * n for n in rows]
    c = Batch(ptts, cuda, [9, 130], rows, tree=True, parents=roots, seed=1)
    clean = ptts.attend_tree(c.kv, 0, c.q, c.k, c.v, c.streams, c.rows, c.parents_dev)
    c.k[5], c.v[5] = float("nan"), float("nan")
    out = ptts.attend_tree(c.kv, 0, c.q, c.k, c.v, c.streams, c.rows, c.parents_dev)
    others = [i for i in range(sum(rows)) if i != 5]
    assert torch.equal(out[others], clean[others]) and torch.isnan(out[5]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [-2, 3, 2 ** 31 - 1, -2 ** 31])
def test_a_bad_parent_refuses_its_tree_alone(ptts, cuda, bad):
    import torch
    b = Batch(ptts, cuda, [10, 20, 30], [4, 5, 6], tree=True, seed=8)
    b.parents_dev[4 + 3] = bad  # node 3 of the second tree
    before = [t.clone() for t in b.kv.tensors(0)[:2]]
    out = ptts.attend_tree(b.kv, 0, b.q, b.k, b.v, b.streams, b.rows, b.parents_dev)
    with pytest.raises(ptts.PttsError) as e:
        b.kv.check()
    assert e.value.code == ptts.ERR_DEVICE and "bounds" in e.value.msg
    b.kv.check()
    assert (out[4:9] == 0).all()
    for t, old in zip(b.kv.tensors(0)[:2], before):
        assert torch.equal(torch.nan_to_num(t[int(b.streams[1])]), torch.nan_to_num(old[int(b.streams[1])]))
    vt = b.kv.tensors(0)[1]
    vt[int(b.streams[1]), 20:25] = 0  # so that the oracle of the others has numbers there
    want, bound = b.want(tree=True, half_p=PAIR_HALF)
    keep = [i for i in range(15) if not 4 <= i < 9]
    compare(out[keep], want[keep], bound[keep])


# ---- acceptance -------------------------------------------------------------------------------------

PATHS = [[], [0], [0, 1, 2], [3], [0, 2, 3], [1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11], [0, 5, 6, 7, 20, 21, 40, 63],
         list(range(64)), list(range(0, 64, 2))]


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [8, 16])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("times", [1, 40])
def test_accept_moves_rows_and_nothing_else(ptts, cuda, heads, dtype, times):
    """Overlapping moves too; `times` 40: a list too long for the launch's parameters."""
    import torch
    n = len(PATHS) * times
    b = Batch(ptts, cuda, [(5 * i) % 23 for i in range(n)], [64] * n, heads=heads, dtype=dtype, layers=3, seed=12)
    paths = [PATHS[i % len(PATHS)] for i in range(n)]
    for l in range(3):
        for t in b.kv.tensors(l)[:2]:
            t.copy_(torch.randn(t.shape, device=cuda))
    want = [[t.clone() for t in b.kv.tensors(l)[:2]] for l in range(3)]
    for st, L, p in zip(b.streams, b.cached, paths):
        for layer in want:
            for t in layer:
                t[int(st), int(L):int(L) + len(p)] = t[int(st), [int(L) + i for i in p]]
    b.kv.accept(b.streams, paths)
    b.kv.check()
    for l in range(3):
        for t, w in zip(b.kv.tensors(l)[:2], want[l]):
            assert torch.equal(t, w)
    lengths = np.zeros(n + 2, np.int32)
    lengths[b.streams] = b.cached + [len(p) for p in paths]
    np.testing.assert_array_equal(b.kv.lengths(), lengths)
    np.testing.assert_array_equal(b.kv.tensors(0)[2].cpu().numpy(), lengths)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,dtype", [(8, "bf16"), (16, "bf16"), (8, "f32")])
def test_draft_accept_and_go_on_equals_one_row_at_a_time(ptts, cuda, heads, dtype):
    """Two layers: draft a tree, keep a path, take one more row; against the path fed row by row."""
    import torch
    cached, rows = [11, 200], [12, 40]
    b = Batch(ptts, cuda, cached, rows, heads=heads, dtype=dtype, layers=2, tree=True, seed=14)
    c = Batch(ptts, cuda, cached, rows, heads=heads, dtype=dtype, layers=2, tree=True, seed=14)
    paths = []
    for p in b.parents:
        node, path = max(range(len(p)), key=lambda i: len(lineages(p)[1][i])), []
        while node >= 0:
            path.insert(0, node)
            node = p[node]
        paths.append(path)
    starts = [0, rows[0]]
    for layer in range(2):
        tree_out = ptts.attend_tree(b.kv, layer, b.q, b.k, b.v, b.streams, b.rows, b.parents_dev, softcap=25.0)
    b.kv.accept(b.streams, paths)
    for s, (st, path, at) in enumerate(zip(c.streams, paths, starts)):
        for node in path:
            r = slice(at + node, at + node + 1)
            for layer in range(2):
                one = ptts.attend_scored(c.kv, layer, c.q[r], c.k[r], c.v[r], [st], [1], softcap=25.0)
            # both within 2^-14 of the definition's weights, bounded as in the module's docstring
            assert (tree_out[r] - one).abs().max().item() <= 2.0 ** -10
            c.kv.advance([st], [1])
    np.testing.assert_array_equal(b.kv.lengths(), c.kv.lengths())
    for layer in range(2):
        for x, y in zip(b.kv.tensors(layer)[:2], c.kv.tensors(layer)[:2]):
            for st in b.streams:
                n = int(b.kv.lengths()[st])
                assert torch.equal(x[int(st), :n], y[int(st), :n])
    q, k, v = (t[:2].contiguous() for t in (b.q, b.k, b.v))
    x = ptts.attend(b.kv, 1, q, k, v, b.streams, [1, 1])
    y = ptts.attend(c.kv, 1, q, k, v, c.streams, [1, 1])
    assert torch.equal(x, y)
    b.kv.check(), c.kv.check()


# ---- large offsets --------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", ["tokens", "prompts", "trees"])
def test_offsets_past_32_bits(ptts, cuda, kind, dtype):
    """Five streams of over a million slots: the last one's rows lie past 2^32 bytes (and 2^31 elements) of
    the cache, and the long stream's own keys past 2^30. Its weights' sum has 2^9 f32 steps (the parts'
    chunks and their joining, at most 2^8 of either): 2^-15 in place of the module's 2^-18."""
    import torch
    rows = {"tokens": [1] * 5, "prompts": [5, 200, 70, 1, 33], "trees": [9, 64, 1, 33, 17]}[kind]
    b = Batch(ptts, cuda, [1_100_000, 700, 0, 40, 900], rows, dtype=dtype, spare=0, seed=21, tree=kind == "trees")
    assert 4 * b.capacity * 512 > 2 ** 31
    args = dict(softcap=20.0, slopes=b.slopes)
    if kind == "trees":
        out = ptts.attend_tree(b.kv, 0, b.q, b.k, b.v, b.streams, b.rows, b.parents_dev, **args)
    else:
        out = ptts.attend_scored(b.kv, 0, b.q, b.k, b.v, b.streams, b.rows, **args)
    b.kv.check()
    want, bound = b.want(tree=kind == "trees", half_p=PAIR_HALF + 2.0 ** -15, **args)
    compare(out, want, bound)
    b.check_rows(tree=kind == "trees")
    if kind != "trees":
        return
    kt, vt, _ = b.kv.tensors(0)
    paths = [sorted(lineages(p)[1][-1]) for p in b.parents]
    kept = [[t[int(st), [int(L) + i for i in p]].clone() for t in (kt, vt)] for st, L, p in zip(b.streams, b.cached, paths)]
    b.kv.accept(b.streams, paths)
    for st, L, p, rows in zip(b.streams, b.cached, paths, kept):
        for t, r in zip((kt, vt), rows):
            assert torch.equal(t[int(st), int(L):int(L) + len(p)], r)


# ---- refusals ---------------------------------------------------------------------------------------

def test_null_handles_are_refused_without_a_device(ptts):
    lib = ptts.lib()
    one = (ctypes.c_int32 * 1)(1)
    rules = ptts.Scores()
    assert lib.ptts_b200_attend_scored(None, 0, None, None, None, 1, 8, one, one, 1, 1e4, ctypes.byref(rules), None, 0, None) == ptts.ERR_ARG
    assert lib.ptts_b200_attend_tree(None, 0, None, None, None, 1, 8, one, one, 1, None, 1e4, None, None, 0, None) == ptts.ERR_ARG
    assert lib.ptts_b200_kv_accept(None, one, one, one, 1, None) == ptts.ERR_ARG
    assert "kv is NULL" in lib.ptts_b200_last_error().decode()


def test_python_checks_come_before_the_library(ptts):
    """Shapes, types and devices are refused on CPU tensors, with no device in the machine."""
    import torch

    class Kv:  # what the checks read
        num_heads, head_dim, device, handle = 8, 64, 0, None

    q = torch.zeros(2, 8, 64)
    for bad in [dict(k=torch.zeros(2, 8, 64, dtype=torch.bfloat16)), dict(q=torch.zeros(3, 8, 64)),
                dict(q=torch.zeros(2, 8, 32)), dict(v=torch.zeros(2, 4, 64)), dict(rows=[1, 1]),
                dict(q=torch.zeros(2, 8, 64, dtype=torch.float16), k=torch.zeros(2, 8, 64, dtype=torch.float16),
                     v=torch.zeros(2, 8, 64, dtype=torch.float16)),
                dict(q=torch.zeros(8, 2, 64).transpose(0, 1)), {}]:
        a = dict(q=q, k=q, v=q, rows=[2])
        a.update(bad)
        with pytest.raises(ptts.PttsError) as e:
            ptts.attend_scored(Kv, 0, a["q"], a["k"], a["v"], [0], a["rows"])
        assert e.value.code == ptts.ERR_ARG
    with pytest.raises(ptts.PttsError):
        ptts._rule_tensor(Kv, torch.zeros(8, dtype=torch.float64), "slopes", torch.float32, 8)
    with pytest.raises(ptts.PttsError):
        ptts._rule_tensor(Kv, torch.zeros(7), "slopes", torch.float32, 8)
    with pytest.raises(ptts.PttsError):
        ptts._rule_tensor(Kv, torch.zeros(8), "slopes", torch.float32, 8)  # not on the cache's device


@pytest.mark.gpu
def test_refusals_change_nothing(ptts, cuda):
    import torch
    b = Batch(ptts, cuda, [5, 9, 0], [2, 1, 1], tree=True, seed=20, spare=3)
    st = [int(s) for s in b.streams]
    others = sorted(set(range(6)) - set(st))
    b.kv.start_ring(others[:1])
    b.kv.set_window(others[1:2], 4)
    before = [torch.nan_to_num(t) for t in b.kv.tensors(0)[:2]]
    lengths = b.kv.lengths().copy()

    def refused(code, f, *a, **k):
        with pytest.raises(ptts.PttsError) as e:
            f(*a, **k)
        assert e.value.code == code, e.value

    def scored(**k):
        a = dict(layer=0, q=b.q, k=b.k, v=b.v, streams=st, rows=[2, 1, 1])
        rest = {n: k.pop(n) for n in list(k) if n not in a}
        a.update(k)
        return ptts.attend_scored(b.kv, a["layer"], a["q"], a["k"], a["v"], a["streams"], a["rows"], **rest)

    refused(ptts.ERR_ARG, scored, layer=1)
    refused(ptts.ERR_ARG, scored, streams=[st[0], st[0], st[1]])
    refused(ptts.ERR_ARG, scored, streams=[st[0], st[1], 6])
    refused(ptts.ERR_ARG, scored, rows=[3, 1, 0])
    refused(ptts.ERR_UNSUPPORTED, scored, streams=[st[0], st[1], others[0]])
    refused(ptts.ERR_UNSUPPORTED, scored, streams=[st[0], st[1], others[1]])
    for cap in (-1.0, 1e-38, 1e38, float("nan"), float("inf")):
        refused(ptts.ERR_ARG, scored, softcap=cap)
    for period in (1.0, -3.0, float("nan"), float("inf")):
        refused(ptts.ERR_ARG, scored, max_period=period)
    refused(ptts.ERR_ARG, scored, k=b.k[:, :3].contiguous(), v=b.v[:, :3].contiguous())
    refused(ptts.ERR_ARG, scored, slopes=b.slopes[:4])
    refused(ptts.ERR_ARG, scored, first=torch.zeros(4, dtype=torch.int64, device=cuda))
    refused(ptts.ERR_ARG, scored, last=torch.zeros(8, dtype=torch.int32, device=cuda)[::2])
    refused(ptts.ERR_ARG, scored, out=torch.empty(4, 512, device=cuda)[:, ::2])
    refused(ptts.ERR_ARG, scored, out=torch.empty(4, 512, dtype=torch.float16, device=cuda))
    flat = torch.zeros(4 * 512 + 8, dtype=torch.bfloat16, device=cuda)
    refused(ptts.ERR_ARG, scored, q=flat[1:1 + 4 * 512].view(4, 8, 64))
    full = Batch(ptts, cuda, [5], [2], seed=1)
    full.kv.set_lengths(full.streams, [full.capacity - 1])
    refused(ptts.ERR_CAPACITY, ptts.attend_scored, full.kv, 0, full.q, full.k, full.v, full.streams, [2])
    refused(ptts.ERR_ARG, ptts.attend_tree, b.kv, 0, b.q, b.k, b.v, st, [2, 1, 1], None)
    refused(ptts.ERR_ARG, ptts.attend_tree, b.kv, 0, b.q, b.k, b.v, st, [2, 1, 1], b.parents_dev[:3])
    big = Batch(ptts, cuda, [0], [65], seed=1)
    refused(ptts.ERR_UNSUPPORTED, ptts.attend_tree, big.kv, 0, big.q, big.k, big.v, big.streams, [65],
            torch.full((65,), -1, dtype=torch.int32, device=cuda))
    refused(ptts.ERR_ARG, b.kv.accept, [st[0], st[0]], [[0], [0]])
    refused(ptts.ERR_ARG, b.kv.accept, [st[0]], [[0], [0]])
    refused(ptts.ERR_ARG, b.kv.accept, [6], [[0]])
    refused(ptts.ERR_ARG, b.kv.accept, [], [])
    for path in ([1, 1], [2, 1], [-1], [0, 64]):
        refused(ptts.ERR_ARG, b.kv.accept, [st[1], st[0]], [[0], path])
    refused(ptts.ERR_CAPACITY, b.kv.accept, [st[1]], [[0, b.capacity - 9]])
    refused(ptts.ERR_UNSUPPORTED, b.kv.accept, [st[0], others[0]], [[0], []])
    refused(ptts.ERR_UNSUPPORTED, b.kv.accept, [others[1]], [[0]])
    graph = torch.cuda.CUDAGraph()
    scored()  # workspaces are there: the capture alone is refused
    before = [torch.nan_to_num(t) for t in b.kv.tensors(0)[:2]]
    side = torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        refused(ptts.ERR_STATE, scored)
        refused(ptts.ERR_STATE, b.kv.accept, [st[0]], [[0]])
    b.kv.check()
    np.testing.assert_array_equal(b.kv.lengths(), lengths)
    for t, old in zip(b.kv.tensors(0)[:2], before):
        assert torch.equal(torch.nan_to_num(t), old)
