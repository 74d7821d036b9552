"""Cases of the attention operators with score rules, drafted trees and their acceptance.

Three entry points of the package are measured: `attend_scored` (prompts, and one token per
stream), `attend_tree` and `KvState.accept`. The plain forms below are the same operators in
elementary torch operations, f32 throughout and rounded once at the end.

An attention row at position p of a stream sees the positions first..last of it (0..p where a
call gives neither). With scores s_j = q . k_j / sqrt(64) over the rotated q and keys:
    t_j = softcap * tanh(s_j / softcap)   (s_j where there is no softcap)
    u_j = t_j - slopes[head] * |p - j|    (t_j where there are no slopes)
    out = sum_j exp(u_j) v_j / sum_j exp(u_j); zeros where a row sees nothing.
The call's own rows go into the cache first, rounded to its type. The rotation (interleaved pairs)
turns pair i by the f32 product of the position and the f32 1 / max_period^(i/32); max_period 0: none.
A drafted tree's node sees its stream's cached rows, its ancestors and itself, at position
length + depth; node i's row is stored at slot length + i. Accepting a path moves its rows to the
slots behind the cached ones, in every layer, and the stream grows by the path's length.
"""
import math
import random

import torch

own = False

D = 64


# ---- the cases -----------------------------------------------------------------------------

def _case(name, op, **kw):
    c = {"name": name, "op": op, "streams": 1, "heads": 8, "kv_heads": 8, "dtype": "bf16", "layers": 1, "cached_lo": 0,
         "cached_hi": 0, "rows_lo": 1, "rows_hi": 1, "softcap": 0.0, "slopes": False, "mask": "causal",
         "max_period": 10000.0, "sizes": 1}
    c.update(kw)
    return c


def listed():
    return [
        # A session's first call: a short text prompt whose rows all see the voice prefix.
        _case("prompt_prefix_short", "prompt", rows_lo=77, rows_hi=77, cached_lo=33, cached_hi=33, mask="prefix", sizes=11),
        # A server's prompt batch: several utterances packed per stream, capped scores, padding rows at the ends.
        _case("prompt_documents_batch", "prompt", streams=96, rows_lo=200, rows_hi=900, mask="documents", softcap=30.0,
              sizes=12),
        # Long prompts with a distance bias in place of the rotation, 16 heads sharing 4 key heads.
        _case("prompt_long_bias", "prompt", streams=4, heads=16, kv_heads=4, rows_lo=3900, rows_hi=4096, slopes=True,
              max_period=0.0, sizes=13),
        # The f32 cache, every rule at once, odd sizes.
        _case("prompt_f32", "prompt", streams=5, dtype="f32", rows_lo=65, rows_hi=301, cached_lo=0, cached_hi=130,
              mask="documents", softcap=50.0, slopes=True, sizes=14),
        # One session generating: a frame's single row, f32 as the single-stream configuration has it.
        _case("token_single_f32", "token", dtype="f32", cached_lo=511, cached_hi=511, softcap=30.0, sizes=21),
        # The ragged decode batch with capped scores.
        _case("token_ragged_batch", "token", streams=256, cached_lo=64, cached_hi=2048, softcap=30.0, sizes=22),
        # Few streams, long caches, a distance bias: the long axis has to be split.
        _case("token_long_bias", "token", streams=6, cached_lo=30000, cached_hi=65000, slopes=True, max_period=0.0,
              sizes=23),
        # One session drafting a small tree.
        _case("tree_single", "tree", cached_lo=300, cached_hi=300, rows_lo=13, rows_hi=13, sizes=31),
        # A batch of sessions, each with its own tree.
        _case("tree_batch", "tree", streams=128, cached_lo=64, cached_hi=2048, rows_lo=8, rows_hi=64, softcap=30.0,
              sizes=32),
        # Full trees over long caches.
        _case("tree_long", "tree", streams=4, cached_lo=20000, cached_hi=33000, rows_lo=60, rows_hi=64, sizes=33),
        # One session's accepted path, 6 layers.
        _case("accept_single", "accept", layers=6, cached_lo=300, cached_hi=300, rows_lo=40, rows_hi=40, sizes=41),
        # A batch's accepted paths, 9 layers.
        _case("accept_batch", "accept", streams=512, layers=9, cached_lo=32, cached_hi=440, rows_lo=30, rows_hi=64,
              sizes=42),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("prompt", "prompt", "token", "token", "tree", "tree", "accept"))
    heads = rng.choice((8, 8, 16))
    kw = {"heads": heads, "kv_heads": rng.choice((heads, heads, heads // 4, 1)), "sizes": rng.randrange(1 << 20),
          "dtype": rng.choice(("bf16", "bf16", "bf16", "f32"))}
    if op != "accept":
        kw["softcap"] = rng.choice((0.0, 0.0, 15.0, 30.0, 50.0))
        kw["slopes"] = rng.random() < 0.4
        kw["max_period"] = rng.choice((0.0, 10000.0)) if kw["slopes"] else 10000.0
    f32 = kw["dtype"] == "f32"
    if op == "prompt":
        kw["mask"] = rng.choice(("causal", "prefix", "documents", "window"))
        rows = _log(rng, 2, 700 if f32 else 3000)
        cached = rng.choice((0, _log(rng, 1, 400 if f32 else 1500)))
        # scores of all heads: at most the largest listed case's
        most = (1 << 24 if f32 else 1 << 27) // (heads // 8)
        streams = max(1, min(_log(rng, 1, 64), most // (rows * (rows + cached))))
        kw.update(streams=streams, rows_lo=max(1, rows // 2), rows_hi=rows, cached_lo=cached // 2, cached_hi=cached)
    elif op == "token":
        kw["mask"] = rng.choice(("causal", "causal", "window"))
        cached = _log(rng, 1, 60000)
        streams = max(1, min(_log(rng, 1, 300), 260000 // cached // (heads // 8) // (2 if f32 else 1)))
        kw.update(streams=streams, cached_lo=cached // 3, cached_hi=cached)
    elif op == "tree":
        rows = _log(rng, 2, 64)
        cached = _log(rng, 1, 2000 if f32 else 30000)
        streams = max(1, min(_log(rng, 1, 128), (8000 if f32 else 120000) // cached // (heads // 8)))
        kw.update(streams=streams, cached_lo=cached // 3, cached_hi=cached, rows_lo=max(1, rows // 2), rows_hi=rows)
    else:
        rows = _log(rng, 4, 64)
        cached = _log(rng, 1, 1000)
        layers = rng.randint(1, 9)
        streams = max(1, min(_log(rng, 1, 400), 1500000 // ((cached + rows) * layers * (heads // 8) * (2 if f32 else 1))))
        kw.update(streams=streams, layers=layers, cached_lo=cached // 2, cached_hi=cached, rows_lo=max(2, rows // 2),
                  rows_hi=rows)
    return {k: v for k, v in _case("", op, **kw).items() if k != "name"}


# ---- sizes and plans: plain lists, from the case alone --------------------------------------

def _tree(rng, n):
    """Parents of n drafted nodes, in order; several roots now and then."""
    return [-1 if i == 0 or rng.random() < 0.05 else rng.randrange(max(0, i - 12), i) for i in range(n)]


def _path(rng, n):
    """An accepted path of a tree of n nodes: rising node indexes, each its own place in the path or
    past its end (a tree laid out level by level), so that accepting it again changes nothing."""
    count = rng.randint(0, min(8, n))
    stay = rng.randint(0, count)
    free = list(range(count, n))
    if len(free) < count - stay:
        return list(range(count))
    return list(range(stay)) + sorted(rng.sample(free, count - stay))


def _sizes(case):
    rng = random.Random(case["sizes"])
    S = case["streams"]
    streams = list(range(S))
    rng.shuffle(streams)
    cached = [rng.randint(case["cached_lo"], case["cached_hi"]) for _ in streams]
    rows = [rng.randint(case["rows_lo"], case["rows_hi"]) for _ in streams]
    first, last, parents, paths = None, None, None, None
    if case["op"] in ("prompt", "token") and case["mask"] != "causal":
        first, last = [], []
        for L, n in zip(cached, rows):
            pos = range(L, L + n)
            if case["mask"] == "prefix":  # the prefix sees itself whole; the rest is causal
                prefix = rng.randint(1, max(1, (L + n) * 2 // 3))
                first += [0] * n
                last += [max(p, prefix - 1) for p in pos]
            elif case["mask"] == "documents":  # causal inside its document; the last rows are padding
                cuts = sorted({0} | {rng.randint(0, L + n - 1) for _ in range(rng.randint(0, 5))})
                pad = rng.randint(0, n // 8)
                first += [p + 1 if p >= L + n - pad else max(c for c in cuts if c <= p) for p in pos]
                last += list(pos)
            else:
                w = rng.randint(1, L + n)
                first += [max(0, p - w + 1) for p in pos]
                last += list(pos)
    if case["op"] == "tree":
        parents = [_tree(rng, n) for n in rows]
    if case["op"] == "accept":
        paths = [_path(rng, n) for n in rows]
    return {"streams": streams, "cached": cached, "rows": rows, "first": first, "last": last, "parents": parents,
            "paths": paths, "capacity": max(L + n for L, n in zip(cached, rows)) + rng.randint(0, 9)}


def work(case):
    z = _sizes(case)
    H, KVH, e = case["heads"], case["kv_heads"], 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "accept":
        moved = sum(i != j for p in z["paths"] for j, i in enumerate(p))
        return {"bytes": 2 * 2 * case["layers"] * moved * H * D * e + 8 * len(z["streams"]), "flops": 0}
    pairs, read, at = 0, 0, 0
    for n, (L, rows) in enumerate(zip(z["cached"], z["rows"])):
        if case["op"] == "tree":
            depth = []
            for p in z["parents"][n]:
                depth.append(0 if p < 0 else depth[p] + 1)
            pairs += rows * L + sum(d + 1 for d in depth)
            read += L
        else:
            f = z["first"][at:at + rows] if z["first"] else [0] * rows
            t = z["last"][at:at + rows] if z["last"] else list(range(L, L + rows))
            pairs += sum(max(0, b - a + 1) for a, b in zip(f, t))
            seen = [a for a, b in zip(f, t) if a <= b]
            read += max(0, L - min(seen)) if seen else 0  # cached rows; the call's own come with the call
        at += rows
    rows = sum(z["rows"])
    # cached K and V, q, the call's k and v, the cache rows written, the output
    return {"bytes": e * D * (2 * read * H + rows * (H + 2 * KVH) + 2 * rows * H + rows * H), "flops": 4 * D * H * pairs}


# ---- inputs ---------------------------------------------------------------------------------

def _inv_freq(max_period):
    """1 / max_period^(i/32), the power and the quotient rounded to f32; None: no rotation."""
    if not max_period:
        return None
    power = torch.pow(torch.tensor(max_period, dtype=torch.float64), torch.arange(D // 2, dtype=torch.float64) / (D // 2))
    return (1.0 / power.float()).cuda()


def _inputs(case, seed, z):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    H, KVH, S, G = case["heads"], case["kv_heads"], case["streams"], case["heads"] // 8

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dt)

    # One block per 8 heads, as the framework's cache has it, seen as [streams, capacity, (groups,) 8, 64].
    blocks = [[normal(G, S, z["capacity"], 8, D) for _ in range(2)] for _ in range(case["layers"])]
    caches = [[b[0] if G == 1 else b.permute(1, 2, 0, 3, 4) for b in kv] for kv in blocks]
    lengths = torch.zeros(S, dtype=torch.int32, device="cuda")
    lengths[torch.tensor(z["streams"], device="cuda")] = torch.tensor(z["cached"], dtype=torch.int32, device="cuda")
    x = {"caches": caches, "lengths": lengths}
    if case["op"] != "accept":
        N = sum(z["rows"])
        x["q"], x["k"], x["v"] = normal(N, H, D) * 2, normal(N, KVH, D), normal(N, KVH, D)
        x["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device="cuda") if case["slopes"] else None
        for name in ("first", "last"):
            x[name] = torch.tensor(z[name], dtype=torch.int32, device="cuda") if z[name] else None
        if case["op"] == "tree":
            x["parents"] = torch.tensor(sum(z["parents"], []), dtype=torch.int32, device="cuda")
    return x


def prepare(case, seed):
    z = _sizes(case)
    x = _inputs(case, seed, z)
    s = {"case": case, **z, **x}
    if own:
        import numpy as np
        from __graft_entry__ import load_package
        pkg = load_package()
        kv = pkg.KvState(case["layers"], case["streams"], z["capacity"], num_heads=case["heads"], dtype=case["dtype"])
        views = [kv.tensors(layer) for layer in range(case["layers"])]
        for (kt, vt, _), (k0, v0) in zip(views, x["caches"]):
            kt.copy_(k0)
            vt.copy_(v0)
        kv.set_lengths(z["streams"], z["cached"])
        s.update(pkg=pkg, kv=kv, caches=[[kt, vt] for kt, vt, _ in views], lengths=views[0][2],
                 streams=np.array(z["streams"], np.int32), rows=np.array(z["rows"], np.int32),
                 cached=np.array(z["cached"], np.int32))
        # Rows of streams' caches are made above and copied once; later calls are ordered after them.
        torch.cuda.synchronize()
        return s
    # What a program with this batch keeps beside its inputs: row -> (sequence, place), as index tensors.
    dev = {"device": "cuda"}
    s["stream_idx"] = torch.tensor(z["streams"], **dev)
    s["cached_idx"] = torch.tensor(z["cached"], **dev)
    if case["op"] == "accept":
        moves = [(st, L + i, L + j) for st, L, p in zip(z["streams"], z["cached"], z["paths"]) for j, i in enumerate(p)]
        s["move_stream"], s["move_from"], s["move_to"] = (torch.tensor([m[i] for m in moves], dtype=torch.long, **dev) for i in range(3))
        s["new_lengths"] = torch.tensor([L + len(p) for L, p in zip(z["cached"], z["paths"])], dtype=torch.int32, **dev)
        return s
    s["row_seq"] = torch.tensor([i for i, n in enumerate(z["rows"]) for _ in range(n)], **dev)
    s["row_at"] = torch.tensor([j for n in z["rows"] for j in range(n)], **dev)
    s["inv_freq"] = _inv_freq(case["max_period"])
    return s


# ---- the plain forms --------------------------------------------------------------------------

def _rotate(x, pos, inv_freq):
    """x [n, heads, 64] f32, interleaved pairs, by the f32 angle pos * inv_freq."""
    if inv_freq is None:
        return x
    angle = (pos.float()[:, None] * inv_freq[None, :]).double()
    c, s = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)


def _padded(s, x, fill=0):
    """[rows, ...] -> [sequences, most rows, ...]."""
    y = torch.full((len(s["rows"]), max(s["rows"])) + x.shape[1:], fill, dtype=x.dtype, device=x.device)
    y[s["row_seq"], s["row_at"]] = x
    return y


def _attend(s):
    case = s["case"]
    H, KVH, S, cap = case["heads"], case["kv_heads"], len(s["rows"]), s["capacity"]
    row_seq, row_at = s["row_seq"], s["row_at"]
    stream, base = s["stream_idx"][row_seq], s["cached_idx"][row_seq]
    slot = base + row_at
    live = _padded(s, torch.ones_like(row_at, dtype=torch.bool))
    R, T = live.shape[1], max(L + n for L, n in zip(s["cached"], s["rows"]))
    if case["op"] == "tree":
        parent = _padded(s, s["parents"].long(), -1)
        up = torch.zeros(S, R, R + 1, device="cuda").scatter_(2, torch.where(parent < 0, R, parent)[..., None], 1.0)[..., :R]
        lineage = torch.linalg.matrix_power(up + torch.eye(R, device="cuda"), 64) > 0  # itself and its ancestors
        depth = lineage.sum(-1) - 1
        pos = base + depth[row_seq, row_at]
    else:
        pos = slot
    group = H // KVH
    q = _rotate(s["q"].float(), pos, s["inv_freq"])
    k = _rotate(s["k"].float(), pos, s["inv_freq"]).repeat_interleave(group, 1)
    v = s["v"].float().repeat_interleave(group, 1)
    kc, vc = s["caches"][0]
    shape = kc.shape[2:]
    kc[stream, slot] = k.to(kc.dtype).reshape(-1, *shape)
    vc[stream, slot] = v.to(vc.dtype).reshape(-1, *shape)
    keys = kc[s["stream_idx"], :T].reshape(S, T, H, D).permute(0, 2, 3, 1).float()
    vals = vc[s["stream_idx"], :T].reshape(S, T, H, D).permute(0, 2, 1, 3).float()
    j = torch.arange(T, device="cuda")
    row_pos = _padded(s, pos)
    key_pos = j.expand(S, T)
    if case["op"] == "tree":
        at = j[None, :] - s["cached_idx"][:, None]  # a drafted key's node, negative for cached keys
        node = at.clamp(0, R - 1)
        among = lineage.gather(2, node[:, None, :].expand(S, R, T))
        seen = (at < 0)[:, None, :] | (among & (at < R)[:, None, :])
        key_pos = torch.where(at < 0, j[None, :], s["cached_idx"][:, None] + depth.gather(1, node))
    else:
        last = _padded(s, s["last"].long() if s["last"] is not None else slot)
        seen = j[None, None, :] <= last[:, :, None]
        if s["first"] is not None:
            seen &= j[None, None, :] >= _padded(s, s["first"].long())[:, :, None]
    seen = (seen & live[:, :, None])[:, None]
    u = torch.matmul(_padded(s, q).permute(0, 2, 1, 3), keys) / math.sqrt(D)
    if case["softcap"]:
        u = torch.tanh(u / case["softcap"]) * case["softcap"]
    if s["slopes"] is not None:
        apart = (row_pos[:, :, None] - key_pos[:, None, :]).abs().float()
        u = u - s["slopes"][None, :, None, None] * apart[:, None]
    u = torch.where(seen, u, -math.inf)
    top = u.amax(-1, keepdim=True)
    p = torch.exp(u - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, vals) / torch.where(total == 0, 1.0, total)
    out = o.permute(0, 2, 1, 3)[row_seq, row_at].reshape(-1, H * D).to(kc.dtype)
    return [out, kc, vc]


def _accept(s):
    for kc, vc in s["caches"]:
        kc[s["move_stream"], s["move_to"]] = kc[s["move_stream"], s["move_from"]]
        vc[s["move_stream"], s["move_to"]] = vc[s["move_stream"], s["move_from"]]
    s["lengths"][s["stream_idx"]] = s["new_lengths"]
    return [s["lengths"], s["caches"]]


def run(state):
    s = state
    case = s["case"]
    if not own:
        return _accept(s) if case["op"] == "accept" else _attend(s)
    if case["op"] == "accept":
        # Back to the step before the acceptance (as a program does that verifies again), then the call.
        s["kv"].set_lengths(s["streams"], s["cached"])
        s["kv"].accept(s["streams"], s["paths"])
        return [s["lengths"], s["caches"]]
    rules = {"softcap": case["softcap"], "slopes": s["slopes"], "max_period": case["max_period"], "out_dtype": case["dtype"]}
    if case["op"] == "tree":
        out = s["pkg"].attend_tree(s["kv"], 0, s["q"], s["k"], s["v"], s["streams"], s["rows"], s["parents"], **rules)
    else:
        out = s["pkg"].attend_scored(s["kv"], 0, s["q"], s["k"], s["v"], s["streams"], s["rows"], first=s["first"],
                                     last=s["last"], **rules)
    return [out, *s["caches"][0]]


# ---- the definition in 64 bits, sequence by sequence --------------------------------------------

def exact(case, seed):
    z = _sizes(case)
    x = _inputs(case, seed, z)
    if case["op"] == "accept":
        lengths = x["lengths"].clone()
        caches = [[c.clone() for c in kv] for kv in x["caches"]]
        for st, L, path in zip(z["streams"], z["cached"], z["paths"]):
            lengths[st] = L + len(path)
            if not path:
                continue
            take = torch.tensor([L + i for i in path], device="cuda")
            for new, old in zip(caches, x["caches"]):
                for a, b in zip(new, old):
                    a[st, L:L + len(path)] = b[st, take]
        return [lengths, caches]
    H, KVH, dt = case["heads"], case["kv_heads"], x["q"].dtype
    kc, vc = x["caches"][0]
    kd, vd = kc.double(), vc.double()
    out = torch.zeros(sum(z["rows"]), H * D, dtype=torch.float64, device="cuda")
    freq = [1.0 / torch.tensor(case["max_period"] ** (i / 32.0)) for i in range(32)] if case["max_period"] else None
    at = 0
    for n, (st, L, rows) in enumerate(zip(z["streams"], z["cached"], z["rows"])):
        mine = slice(at, at + rows)
        if case["op"] == "tree":
            depth, lines = [], []
            for i, p in enumerate(z["parents"][n]):
                depth.append(0 if p < 0 else depth[p] + 1)
                lines.append([i] + (lines[p] if p >= 0 else []))
            pos = torch.tensor([L + d for d in depth], device="cuda")
            where = torch.cat([torch.arange(L, device="cuda"), pos])
            seen = torch.zeros(rows, L + rows, dtype=torch.bool)
            seen[:, :L] = True
            for i, line in enumerate(lines):
                seen[i, [L + a for a in line]] = True
            seen = seen.cuda()
        else:
            pos = torch.arange(L, L + rows, device="cuda")
            where = torch.arange(L + rows, device="cuda")
            a = x["first"][mine].long() if x["first"] is not None else torch.zeros_like(pos)
            b = x["last"][mine].long() if x["last"] is not None else pos
            seen = (where[None] >= a[:, None]) & (where[None] <= b[:, None])
        q, k, v = (x[name][mine].double() for name in ("q", "k", "v"))
        if freq is not None:  # the angle is the f32 product, its sine and cosine are exact
            turn = (pos.float()[:, None] * torch.tensor(freq, dtype=torch.float32, device="cuda")).double()
            turn = torch.polar(torch.ones_like(turn), turn)[:, None]
            q, k = (torch.view_as_real(torch.view_as_complex(t.reshape(rows, -1, 32, 2)) * turn).reshape(rows, -1, D) for t in (q, k))
        k, v = (t[:, [h * KVH // H for h in range(H)]].reshape(rows, *kc.shape[2:]) for t in (k, v))
        kd[st, L:L + rows], vd[st, L:L + rows] = k.to(dt).double(), v.to(dt).double()
        keys, vals = (c[st, :L + rows].reshape(L + rows, H, D) for c in (kd, vd))
        u = torch.einsum("rhd,thd->hrt", q, keys) / 8.0
        if case["softcap"]:
            u = case["softcap"] * torch.tanh(u / case["softcap"])
        if x["slopes"] is not None:
            u = u - x["slopes"].double()[:, None, None] * (pos[:, None] - where[None]).abs().double()[None]
        u = u.masked_fill(~seen[None], -math.inf)
        w = torch.exp(u - u.amax(-1, keepdim=True).clamp(min=-1e300))
        w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
        out[mine] = torch.einsum("hrt,thd->rhd", w, vals).reshape(rows, H * D)
        at += rows
    return [out, kd, vd]
