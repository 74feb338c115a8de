"""Operators around a paged K/V cache, each in its plain form and as the library's call: rotary positions with several
axes, the append of new tokens, attention of the newest tokens, and the eviction of the tokens that got the least
attention.

The cache is a pool of pages, ``[pages, page_size, heads_k, head_dim]``; a row of the block table names a sequence's
pages in order. Accumulated attention weights lie beside it, ``[pages, heads_k, page_size]`` in fp32.

* ``rotary``: queries and keys turned by positions of several axes (time, height, width), forward, and in training with
  the gradients.
* ``append``: a step's queries and keys are turned, keys and values go to their pages.
* ``attend``: attention of the newest tokens over their sequences' pages; with ``mass`` each key's weights, summed over
  the heads of its group, are added to what it has got so far.
* ``evict``: every kv head of a sequence longer than the budget keeps its newest tokens and those of the others that got
  the most weight, in order, on pages of their own.
"""
import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _case(**kw):
    case = {"kind": "attend", "batch": 1, "heads": 32, "heads_k": 8, "seqlen": 1, "keys": 1024, "head_dim": 128, "dtype": "bf16",
            "page": 64, "ragged": False, "window": -1, "softcap": 0.0, "mass": False, "budget": 0, "recent": 0, "train": False,
            "sections": "16,24,24", "interleaved_axes": False, "interleaved_pairs": False}
    case.update(kw)
    return case


def listed():
    return [
        # A picture in front of a prompt, one user, heads whose last third is not turned. Launch and host latency.
        _case(name="rotary_image_s577_fp16", kind="rotary", heads=16, heads_k=4, seqlen=577, head_dim=96, dtype="fp16",
              sections="8,12,12", interleaved_pairs=True),
        # Training on ragged text and pictures: odd length, axes in turns.
        _case(name="rotary_train_b2_s4093", kind="rotary", batch=2, heads=16, heads_k=16, seqlen=4093, sections="24,20,20",
              interleaved_axes=True, train=True),
        # Training on long videos.
        _case(name="rotary_train_b4_s8192", kind="rotary", batch=4, seqlen=8192, train=True),
        # One new token of one user. Latency is all there is.
        _case(name="append_b1", kind="append", keys=8192, page=16),
        # A step of many users, uneven lengths, widest heads.
        _case(name="append_b64_d256_fp16", kind="append", batch=64, heads=16, heads_k=4, head_dim=256, keys=1021, page=32, dtype="fp16",
              ragged=True, sections="128", interleaved_pairs=True),
        # A chunk of a prompt goes into the cache behind what is there.
        _case(name="append_chunk_s4001", kind="append", batch=2, seqlen=4001, keys=1500, ragged=True),
        # Decoding for one user against 8k tokens on small pages.
        _case(name="attend_b1_k8192", keys=8192, page=16),
        # Decoding for a batch of users, uneven lengths, an odd page size.
        _case(name="attend_b32_k4093_fp16", batch=32, keys=4093, page=48, dtype="fp16", ragged=True),
        # Decoding that keeps account of the weights, capped scores.
        _case(name="attend_mass_b16_k16384", batch=16, keys=16384, heads=16, heads_k=4, ragged=True, mass=True, softcap=30.0),
        # Four drafted tokens of one user against a very long cache on large pages: the largest case.
        _case(name="attend_s4_k131072", seqlen=4, heads=64, heads_k=8, keys=131072, page=256),
        # A few users' caches go back to half.
        _case(name="evict_b2_k4096", kind="evict", batch=2, keys=4096, budget=2048, recent=256, page=16),
        # Many users' long caches, uneven lengths, some of them below the budget.
        _case(name="evict_b16_k16384", kind="evict", batch=16, keys=16384, budget=6000, recent=500, ragged=True, heads=16, heads_k=4),
    ]


def _log_int(rng, lo, hi):
    """An integer whose logarithm is spread evenly over [lo, hi]; odd as often as even."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("rotary", "append", "attend", "attend", "attend", "evict"))
    head_dim = rng.choice((64, 96, 128, 128, 128, 192, 256))
    pairs = rng.choice((head_dim // 2, head_dim // 2, head_dim // 4))
    third = pairs // 3
    heads_k, group = rng.choice(((1, 12), (2, 8), (4, 1), (4, 4), (8, 4), (8, 8), (12, 1), (16, 1)))
    case = _case(kind=kind, heads=heads_k * group, heads_k=heads_k, head_dim=head_dim, dtype=rng.choice(("bf16", "bf16", "fp16")),
                 page=rng.choice((16, 16, 32, 48, 64, 64, 100, 128, 256)), ragged=rng.random() < 0.7,
                 sections=rng.choice(("%d,%d,%d" % (pairs - 2 * third, third, third), "%d" % pairs)),
                 interleaved_axes=rng.random() < 0.5, interleaved_pairs=rng.random() < 0.3)
    token = heads_k * head_dim * 4  # bytes of a token's keys and values
    if kind == "rotary":
        tokens = _log_int(rng, 64, min(32768, 2 ** 27 // ((heads_k + case["heads"]) * head_dim)))
        batch = min(rng.choice((1, 1, 2, 4)), tokens)
        return {**case, "batch": batch, "seqlen": tokens // batch, "train": rng.random() < 0.5}
    batch = _log_int(rng, 1, 64)
    most = min(131072, 2 ** 29 // (token * batch))
    if kind == "append":
        return {**case, "batch": batch, "keys": _log_int(rng, 16, min(most, 4096)), "seqlen": rng.choice((1, 1, 3, _log_int(rng, 2, 8192 // batch)))}
    keys = _log_int(rng, 64, most)
    if kind == "evict":
        budget = max(16, int(keys * rng.uniform(0.1, 0.9)))
        return {**case, "batch": batch, "keys": keys, "budget": budget, "recent": int(budget * rng.choice((0.0, 0.1, 0.5)))}
    return {**case, "batch": batch, "keys": keys, "seqlen": rng.choice((1, 1, 1, 2, 5)), "window": rng.choice((-1, -1, -1, keys // 2)),
            "softcap": rng.choice((0.0, 0.0, 30.0)), "mass": rng.random() < 0.4}


def _lengths(case):
    """Tokens that each sequence has in the cache: the longest first, the others between an eighth of it and all of it."""
    rng = random.Random("%d %d" % (case["batch"], case["keys"]))
    most = case["keys"]
    return [most] + [rng.randint(max(1, most // 8), most) if case["ragged"] else most for _ in range(case["batch"] - 1)]


def _sections(case):
    return tuple(int(x) for x in case["sections"].split(","))


def _axis_of_pair(case):
    """Which axis's position turns a pair. In turns, the axes behind the first get every n-th pair until theirs are used up."""
    sections = _sections(case)
    n, pairs = len(sections), sum(sections)
    if case["interleaved_axes"]:
        return [i % n if i < n * sections[i % n] else 0 for i in range(pairs)]
    return [a for a, s in enumerate(sections) for _ in range(s)]


def _package():
    path = os.path.join(os.getcwd(), "kernels-community-rs_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import flash_attn2_b200

    return flash_attn2_b200


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    b, s, h, hk, d, page = (case[x] for x in ("batch", "seqlen", "heads", "heads_k", "head_dim", "page"))

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype)

    st = dict(case)
    if case["kind"] != "evict":
        st["q"] = normal(b, s, h, d)
    if case["kind"] in ("rotary", "append"):
        st["k"] = normal(b, s, hk, d)
        axis = _axis_of_pair(case)
        st["sections"] = _sections(case)
        st["axis"] = torch.tensor(axis, device="cuda")
        # Base 1e6, as for long contexts; pictures of 24 x 24 behind some text.
        st["inv_freq"] = 1e6 ** (-torch.arange(len(axis), device="cuda", dtype=torch.float32) / len(axis))
        start = torch.randint(0, 100000, (b, 1), generator=g, device="cuda")
        i = torch.arange(s, device="cuda").expand(b, s)
        grid = torch.stack([start + i // 576, start + i // 24 % 24, start + i % 24])
        st["positions"] = (grid if len(st["sections"]) == 3 else (start + i)[None]).contiguous()
    if case["kind"] == "rotary":
        if case["train"]:
            st["q"].requires_grad_()
            st["k"].requires_grad_()
            st["grads"] = normal(b, s, h, d), normal(b, s, hk, d)
        return st

    lengths = _lengths(case)
    new = s if case["kind"] == "append" else 0
    pages = [-(-(n + new) // page) for n in lengths]
    kept = [-(-min(n, case["budget"]) // page) for n in lengths] if case["kind"] == "evict" else [0] * b
    total = sum(pages) + sum(kept)
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)

    def table(counts, first):
        """Rows of the block table: each sequence's pages, -1 behind them."""
        width = torch.arange(max(counts), device="cuda")
        n = torch.tensor(counts, device="cuda")
        at = (first + n.cumsum(0) - n)[:, None] + width
        return torch.where(width < n[:, None], order[at.clamp(max=total - 1)], -1)

    st["block_table"] = table(pages, 0)
    st["seqlens"] = torch.tensor(lengths, device="cuda", dtype=torch.int32)
    st["k_cache"], st["v_cache"] = normal(total, page, hk, d), normal(total, page, hk, d)
    if case["kind"] == "append":
        st["v"] = normal(b, s, hk, d)
    if case["kind"] == "evict":
        st["dst_table"] = table(kept, sum(pages))
    if case["kind"] == "evict" or case["mass"]:
        # Weights are heavy-tailed, and some tokens have got none at all.
        w = torch.randn(total, hk, page, generator=g, device="cuda")
        st["attn_mass"] = torch.where(w < -0.5, 0.0, torch.exp(2.5 * w))
    return st


def _rotated(x, st):
    """x [B, S, H, D] turned by st's positions, in fp32 with angles in fp64."""
    angle = st["positions"].double()[st["axis"]].permute(1, 2, 0) * st["inv_freq"].double()
    cos, sin = (t.float()[:, :, None] for t in (angle.cos(), angle.sin()))
    n = cos.shape[-1]
    x = x.float()
    turned, rest = x[..., : 2 * n], x[..., 2 * n:]
    if st["interleaved_pairs"]:
        x0, x1 = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([x0 * cos - x1 * sin, x1 * cos + x0 * sin], -1).flatten(-2)
    else:
        x0, x1 = turned[..., :n], turned[..., n:]
        turned = torch.cat([x0 * cos - x1 * sin, x1 * cos + x0 * sin], -1)
    return torch.cat([turned, rest], -1)


def _plain_append(st):
    dtype = st["q"].dtype
    s, page = st["seqlen"], st["page"]
    slot = st["seqlens"].long()[:, None] + torch.arange(s, device="cuda")
    where = torch.gather(st["block_table"].long(), 1, slot // page), slot % page
    st["k_cache"][where] = _rotated(st["k"], st).to(dtype)
    st["v_cache"][where] = st["v"]
    return {"q": _rotated(st["q"], st).to(dtype), "k_cache": st["k_cache"], "v_cache": st["v_cache"]}


def _plain_attend(st):
    b, s, h, hk, d, page = (st[x] for x in ("batch", "seqlen", "heads", "heads_k", "head_dim", "page"))
    table = st["block_table"].long().clamp(min=0)
    keys = table.shape[1] * page
    col = torch.arange(keys, device="cuda")
    length = st["seqlens"].long()[:, None]
    row = length - s + torch.arange(s, device="cuda")  # where in the sequence each query stands
    seen = (col <= row[..., None]) & (col < length[..., None])
    if st["window"] >= 0:
        seen &= col >= row[..., None] - st["window"]
    k = st["k_cache"][table].view(b, keys, hk, d).float().permute(0, 2, 3, 1)
    v = st["v_cache"][table].view(b, keys, hk, d).float().permute(0, 2, 1, 3)
    v = torch.where((col < length)[:, None, :, None], v, 0.0)
    q = st["q"].float().view(b, s, hk, h // hk, d).permute(0, 2, 1, 3, 4).reshape(b, hk, s * (h // hk), d)
    x = torch.matmul(q, k) / math.sqrt(d)
    if st["softcap"] > 0:
        x = st["softcap"] * torch.tanh(x / st["softcap"])
    x = x.view(b, hk, s, h // hk, keys).masked_fill(~seen[:, None, :, None], -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(b, hk, -1, keys), v).view(b, hk, s, h // hk, d) / total.clamp(min=1e-30)
    lse = torch.where(total > 0, top + torch.log(total), math.inf).squeeze(-1)
    got = {"out": out.permute(0, 2, 1, 3, 4).reshape(b, s, h, d).to(st["q"].dtype), "lse": lse.permute(0, 1, 3, 2).reshape(b, h, s)}
    if st["mass"]:
        weight = (p / total.clamp(min=1e-30)).sum((2, 3))  # [B, Hk, keys]
        pages = table[:, col // page][:, None].expand(b, hk, keys)
        st["attn_mass"].index_put_((pages, torch.arange(hk, device="cuda")[:, None].expand(b, hk, keys), (col % page).expand(b, hk, keys)),
                                   weight, accumulate=True)
        got["mass"] = st["attn_mass"]
    return got


def _plain_evict(st):
    b, hk, page, budget = (st[x] for x in ("batch", "heads_k", "page", "budget"))
    table, to = st["block_table"].long().clamp(min=0), st["dst_table"].long()
    keys = table.shape[1] * page
    col = torch.arange(keys, device="cuda")
    length = st["seqlens"].long()[:, None]
    worth = st["attn_mass"][table].permute(0, 2, 1, 3).reshape(b, hk, keys)
    worth = torch.where((col >= length - st["recent"])[:, None], math.inf, worth)
    worth = torch.where((col >= length)[:, None], -math.inf, worth)
    best = torch.sort(worth, dim=-1, descending=True, stable=True).indices[..., :budget]
    n = length.clamp(max=budget)
    j = torch.arange(best.shape[-1], device="cuda")
    there = (j < n)[:, None].expand(best.shape)
    kept = torch.where(there, best, keys).sort(-1).values
    # A shorter sequence's places behind its last row write its first row once more.
    at, j = torch.where(there, kept, kept[..., :1]), torch.where(there, j, 0)
    to_page, to_row = to[:, None].expand(b, hk, -1).gather(2, j // page), j % page
    head = torch.arange(hk, device="cuda")[:, None].expand(kept.shape)
    from_page, from_row = table[:, None].expand(b, hk, -1).gather(2, at // page), at % page
    for cache in (st["k_cache"], st["v_cache"]):
        cache[to_page, to_row, head] = cache[from_page, from_row, head]
    st["attn_mass"][to_page, head, to_row] = st["attn_mass"][from_page, head, from_row]
    kept = torch.where(there, kept, -1)
    if kept.shape[-1] < budget:
        kept = torch.cat([kept, kept.new_full((b, hk, budget - kept.shape[-1]), -1)], -1)
    return {"seqlens": n[:, 0].int(), "kept": kept.int(), "k_cache": st["k_cache"], "v_cache": st["v_cache"], "mass": st["attn_mass"]}


def run(st):
    kind = st["kind"]
    if own:
        fa2 = _package()
        turns = dict(interleaved_axes=st["interleaved_axes"], interleaved_pairs=st["interleaved_pairs"])
    if kind == "rotary":
        if own:
            q, k = fa2.rotary_axes_func(st["q"], st["k"], st["positions"], st["inv_freq"], st["sections"], **turns)
        else:
            q, k = (_rotated(st[x], st).to(st[x].dtype) for x in ("q", "k"))
        got = {"q": q, "k": k}
        if st["train"]:
            got["dq"], got["dk"] = torch.autograd.grad((q, k), (st["q"], st["k"]), st["grads"])
        return got
    if kind == "append":
        if not own:
            return _plain_append(st)
        q = fa2.paged_append(st["q"], st["k"], st["v"], st["k_cache"], st["v_cache"], st["block_table"], st["seqlens"],
                             st["positions"], st["inv_freq"], st["sections"], **turns)
        return {"q": q, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}
    if kind == "attend":
        if not own:
            return _plain_attend(st)
        out, lse = fa2.paged_fwd(st["q"], st["k_cache"], st["v_cache"], st["block_table"], st["seqlens"],
                                 attn_mass=st["attn_mass"] if st["mass"] else None, window_size_left=st["window"],
                                 softcap=st["softcap"], max_seqlen_k=st["keys"])
        return {"out": out, "lse": lse, "mass": st["attn_mass"]} if st["mass"] else {"out": out, "lse": lse}
    if not own:
        return _plain_evict(st)
    seqlens, kept = fa2.paged_evict(st["k_cache"], st["v_cache"], st["attn_mass"], st["block_table"], st["seqlens"],
                                    st["dst_table"], st["budget"], recent=st["recent"])
    return {"seqlens": seqlens, "kept": kept, "k_cache": st["k_cache"], "v_cache": st["v_cache"], "mass": st["attn_mass"]}


def work(case):
    b, s, h, hk, d = (case[x] for x in ("batch", "seqlen", "heads", "heads_k", "head_dim"))
    lengths = _lengths(case)
    if case["kind"] in ("rotary", "append"):
        elements = b * s * (h + hk) * d
        passes = 2 if case["train"] else 1
        tables = b * s * len(_sections(case)) * 8
        values = b * s * hk * d if case["kind"] == "append" else 0
        return {"bytes": passes * (4 * elements + tables) + 4 * values, "flops": passes * 3 * elements}
    if case["kind"] == "attend":
        seen = [min(n, case["window"] + s) if case["window"] >= 0 else n for n in lengths]
        mass = 8 * hk * sum(seen) if case["mass"] else 0
        return {"bytes": 4 * hk * d * sum(seen) + 4 * b * s * h * d + 4 * b * s * h + mass, "flops": 4 * s * h * d * sum(seen)}
    kept = sum(min(n, case["budget"]) for n in lengths)
    # Weights are read, the kept rows of keys and values are read and written, with their weights and their places.
    return {"bytes": 4 * hk * sum(lengths) + 8 * hk * d * kept + 4 * hk * kept + 4 * hk * b * case["budget"], "flops": hk * sum(lengths)}


def _exact_turn(x, st):
    """By complex products: each pair is a number, its angle's point on the circle the factor."""
    angle = torch.stack([st["positions"][a].double() * f for a, f in zip(st["axis"].tolist(), st["inv_freq"].double().tolist())], -1)
    point = torch.polar(torch.ones_like(angle), angle)[:, :, None]
    n = point.shape[-1]
    x = x.detach().double()
    places = torch.arange(2 * n, device="cuda").view((n, 2) if st["interleaved_pairs"] else (2, n))
    first, second = places.unbind(1 if st["interleaved_pairs"] else 0)
    z = torch.complex(x[..., first], x[..., second])
    out = []
    for factor in (point, point.conj()):
        y = x.clone()
        y[..., first], y[..., second] = (z * factor).real, (z * factor).imag
        out.append(y)
    return out


def exact(case, seed):
    st = prepare(case, seed)
    kind, page = case["kind"], case["page"]
    if kind in ("rotary", "append"):
        got = {"q": _exact_turn(st["q"], st)[0], "k": _exact_turn(st["k"], st)[0]}
        if kind == "rotary":
            if case["train"]:
                got["dq"], got["dk"] = (_exact_turn(t, st)[1] for t in st["grads"])
            return got
        k_cache, v_cache = st["k_cache"].double(), st["v_cache"].double()
        for i, (n, pages) in enumerate(zip(_lengths(case), st["block_table"].long())):
            slot = torch.arange(n, n + case["seqlen"], device="cuda")
            k_cache[pages[slot // page], slot % page] = got["k"][i]
            v_cache[pages[slot // page], slot % page] = st["v"][i].double()
        return {"q": got["q"], "k_cache": k_cache, "v_cache": v_cache}
    hk, group, s = case["heads_k"], case["heads"] // case["heads_k"], case["seqlen"]
    mass = st["attn_mass"].double() if "attn_mass" in st else None
    if kind == "attend":
        out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
        lse = torch.full((case["batch"], case["heads"], s), math.inf, dtype=torch.float64, device="cuda")
        for i, n in enumerate(_lengths(case)):
            pages = st["block_table"][i, : -(-n // page)].long()
            k, v = (st[x][pages].flatten(0, 1)[:n].double() for x in ("k_cache", "v_cache"))
            weight = torch.zeros(n, hk, dtype=torch.float64, device="cuda")
            for t in range(s):
                hi = n - s + t + 1
                lo = max(0, hi - 1 - case["window"]) if case["window"] >= 0 else 0
                if hi <= 0:
                    continue
                q = st["q"][i, t].double().view(hk, group, -1)
                x = torch.einsum("hgd,nhd->hgn", q, k[lo:hi]) * case["head_dim"] ** -0.5
                if case["softcap"] > 0:
                    x = case["softcap"] * torch.tanh(x / case["softcap"])
                z = torch.logsumexp(x, -1)
                p = torch.exp(x - z[..., None])
                out[i, t] = torch.einsum("hgn,nhd->hgd", p, v[lo:hi]).flatten(0, 1)
                lse[i, :, t] = z.flatten()
                weight[lo:hi] += p.sum(1).T
            if mass is not None:
                padded = torch.zeros(len(pages) * page, hk, dtype=torch.float64, device="cuda")
                padded[:n] = weight
                mass[pages] += padded.view(len(pages), page, hk).transpose(1, 2)
        return {"out": out, "lse": lse, "mass": mass} if case["mass"] else {"out": out, "lse": lse}
    k_cache, v_cache = st["k_cache"].clone(), st["v_cache"].clone()
    budget, recent = case["budget"], case["recent"]
    kept = torch.full((case["batch"], hk, budget), -1, dtype=torch.int32, device="cuda")
    lengths = _lengths(case)
    for i, n in enumerate(lengths):
        pages, to = st["block_table"][i].long(), st["dst_table"][i].long()
        for head in range(hk):
            at = torch.arange(n, device="cuda")
            if n > budget:
                worth = st["attn_mass"][pages[at // page], head, at % page][: n - recent]
                # The most weight first, of equal ones the earliest: two stable sorts of one list.
                first = torch.sort(-worth.double(), stable=True).indices[: budget - recent]
                at = torch.cat([first.sort().values, at[n - recent:]])
            kept[i, head, : len(at)] = at.int()
            j = torch.arange(len(at), device="cuda")
            put, take = (to[j // page], j % page, head), (pages[at // page], at % page, head)
            k_cache[put], v_cache[put] = st["k_cache"][take], st["v_cache"][take]
            mass[to[j // page], head, j % page] = st["attn_mass"][pages[at // page], head, at % page].double()
    return {"seqlens": torch.tensor([min(n, budget) for n in lengths], device="cuda", dtype=torch.int32), "kept": kept,
            "k_cache": k_cache, "v_cache": v_cache, "mass": mass}
