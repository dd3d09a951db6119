"""Cases and plain forms of the operators that keep a paged KV cache to a budget.

Three operators of the serving path are measured here: the per-head norm of
queries and keys with the rotation and the append to the cache
(``qk_norm_rope_kv_append``), the decode attention that also adds to every
cached token the attention weight it got (``attention_decode_scored``), and
the eviction of the tokens with the least weight (``kv_evict``). ``run`` makes
one pass through one of them: in its plain form, in elementary torch
operations, or, with ``own`` set, by the framework's entry points.
"""
import math

import numpy as np
import torch

own = False
_device = "cuda"
_PAGE = 16
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_EPS = 1e-5


# ------------------------------------------------------------------ cases
def listed():
    def append(name, tokens, q, kv, dim, rot, dtype, track, decode):
        return dict(name=name, op="append", tokens=tokens, q_heads=q, kv_heads=kv, dim=dim, rot=rot, dtype=dtype,
                    track=track, decode=decode)

    def scored(name, requests, queries, length, low, q, kv, dim, dtype):
        return dict(name=name, op="scored", requests=requests, queries=queries, len=length, low=low, q_heads=q,
                    kv_heads=kv, dim=dim, dtype=dtype)

    def evict(name, requests, length, low, budget, recent, sink, kv, dim, dtype, steady):
        return dict(name=name, op="evict", requests=requests, len=length, low=low, budget=budget, recent=recent,
                    sink=sink, kv_heads=kv, dim=dim, dtype=dtype, steady=steady)

    return [
        # one decode token of the 8B architecture's heads: launch latency
        append("append-1", 1, 32, 8, 128, 128, "bf16", True, True),
        # a chunk of a prompt, half of each 64-wide head rotated, fp16
        append("append-1000-fp16-d64", 1000, 16, 4, 64, 32, "fp16", False, False),
        # a full prefill step of 4096 tokens and one decode row, tracked slots
        append("append-4097", 4097, 32, 8, 128, 128, "bf16", True, False),
        # one request with a short context: latency
        scored("scored-1x700", 1, 1, 700, 700, 32, 8, 128, "bf16"),
        # the serving benchmark's batch: 64 requests of 1536 to 1664 tokens
        scored("scored-64x1664", 64, 1, 1664, 1536, 32, 8, 128, "bf16"),
        # long contexts, eight query heads to a KV head
        scored("scored-8x32768", 8, 1, 32768, 20000, 64, 8, 128, "bf16"),
        # all sixteen query heads on one KV head of 64, fp16, from empty rows to 5000 tokens
        scored("scored-24x5000-fp16-d64", 24, 1, 5000, 0, 16, 1, 64, "fp16"),
        # the last 16 queries of prompts, which give their tokens their first weights
        scored("scored-4x1500-window", 4, 16, 1500, 900, 32, 8, 128, "bf16"),
        # one request that went a page over its budget: latency
        evict("evict-1x528", 1, 528, 528, 512, 64, 4, 8, 128, "bf16", True),
        # a decode batch trimmed back to its budget every 64 tokens
        evict("evict-64x2112", 64, 2112, 2049, 2048, 256, 4, 8, 128, "bf16", True),
        # long prompts cut to a quarter after prefill
        evict("evict-16x8192", 16, 8192, 6000, 2048, 512, 4, 8, 128, "bf16", False),
        # one long prompt, a single 64-wide KV head, fp16
        evict("evict-1x30001-fp16-d64", 1, 30001, 30001, 8192, 1024, 0, 1, 64, "fp16", False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["append", "scored", "evict"])
    dim = rng.choice([64, 128])
    dtype = rng.choice(["bf16", "fp16"])
    kv = rng.choice([1, 2, 4, 8])
    if op == "append":
        return dict(op=op, tokens=_log(rng, 1, 4097), q_heads=kv * rng.choice([1, 2, 4]), kv_heads=kv, dim=dim,
                    rot=rng.choice([dim // 2, dim]), dtype=dtype, track=rng.random() < 0.5, decode=rng.random() < 0.5)
    if op == "scored":
        queries = rng.choice([1, 1, 1, 2, 5, 16])
        length = _log(rng, 16, 32768 if queries == 1 else 2000)
        requests = min(_log(rng, 1, 128), max(1, 200000 // (length * queries)))
        return dict(op=op, requests=requests, queries=queries, len=length, low=rng.randint(0, length),
                    q_heads=kv * rng.choice([1, 3, 4, 8]), kv_heads=kv, dim=dim, dtype=dtype)
    length = _log(rng, 100, 30001)
    budget = max(16, int(length * rng.choice([0.25, 0.5, 0.9, 0.98])))
    return dict(op=op, requests=min(_log(rng, 1, 64), max(1, 110000 // length)), len=length,
                low=rng.randint(budget // 2, length), budget=budget, recent=rng.randint(0, budget // 2),
                sink=rng.choice([0, 4]), kv_heads=kv, dim=dim, dtype=dtype, steady=rng.random() < 0.5)


def _lens(case):
    """Lengths of a batch, spread evenly from ``low`` to ``len`` (the first row has ``len``)."""
    n = case["requests"]
    return [case["len"] - int((case["len"] - case["low"]) * ((i * 0.618033988749895) % 1.0) + 0.5) if i else case["len"]
            for i in range(n)]


def _over(case):
    return [n for n in _lens(case) if n > case["budget"]]


def work(case):
    e, D = 2, case["dim"]
    kv = case["kv_heads"]
    if case["op"] == "append":
        T, q = case["tokens"], case["q_heads"]
        track = 8 * T * kv if case["track"] else 0
        return {"bytes": 2 * T * (q + 2 * kv) * D * e + T * (case["rot"] * 4 + 8) + track,
                "flops": T * (q + kv) * (4 * D + 3 * case["rot"])}
    if case["op"] == "scored":
        total, R, Q, q = sum(_lens(case)), case["requests"], case["queries"], case["q_heads"]
        pages = sum(-(-n // _PAGE) for n in _lens(case))
        return {"bytes": total * kv * (2 * D * e + 8) + 2 * R * Q * q * D * e + 4 * R * Q * q + 4 * pages,
                "flops": 4 * D * q * Q * total}
    b, recent, sink = case["budget"], case["recent"], case["sink"]
    read = moved = 0
    for n in _over(case):
        read += n
        late = min(recent, n - b)  # protected tokens behind the budget; of the others an even share is kept
        moved += late + (n - b - late) * max(0, b - recent - sink) / max(1, n - recent - sink)
    return {"bytes": kv * (8 * read + moved * (4 * D * e + 16)) + 4 * read / _PAGE, "flops": kv * read}


# ------------------------------------------------------------------ inputs
def _pages(lens, gen, spare=3):
    """A block table over shuffled pages, and the number of pages: the last is in no request."""
    need = [max(1, -(-n // _PAGE)) for n in lens]
    count = sum(need) + spare
    order = torch.randperm(count - 1, generator=gen, device=_device).to(torch.int32)
    at = torch.tensor([0] + need, device=_device).cumsum(0)
    col = torch.arange(max(need), device=_device)
    row = at[:-1, None] + col[None, :]
    inside = col[None, :] < torch.tensor(need, device=_device)[:, None]
    table = order[row.clamp(max=count - 2)]
    return torch.where(inside, table, torch.zeros_like(table)).contiguous(), count


def _randn(gen, dtype, *shape):
    return torch.randn(*shape, generator=gen, device=_device, dtype=torch.float32).to(dtype)


def _cache(gen, dtype, pages, kv, dim):
    k = torch.empty(pages, kv, _PAGE, dim, dtype=dtype, device=_device).normal_(generator=gen)
    return k, torch.empty_like(k).normal_(generator=gen)


def _rope_table(rot, max_pos=16384):
    inv = 500000.0 ** (-torch.arange(0, rot // 2, dtype=torch.float64, device=_device) * 2.0 / rot)
    ang = torch.arange(max_pos, dtype=torch.float64, device=_device)[:, None] * inv[None, :]
    return torch.stack([ang.cos(), ang.sin()], dim=-1).to(torch.float32).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device=_device).manual_seed(seed)
    dtype, kv, D = _DTYPES[case["dtype"]], case["kv_heads"], case["dim"]
    st = dict(case)
    if case["op"] == "append":
        T, q = case["tokens"], case["q_heads"]
        pages = (T if case["decode"] else -(-T // _PAGE)) + 5
        st["qkv"] = _randn(gen, dtype, T, (q + 2 * kv) * D) * 2
        st["qw"], st["kw"] = (1 + 0.2 * _randn(gen, torch.float32, D)).to(dtype), (1 + 0.2 * _randn(gen, torch.float32, D)).to(dtype)
        st["table"] = _rope_table(case["rot"])
        order = torch.randperm(pages - 1, generator=gen, device=_device)
        t = torch.arange(T, device=_device)
        if case["decode"]:  # a token of each of T requests: any page, any position
            st["pos"] = torch.randint(0, 8192, (T,), generator=gen, device=_device).to(torch.int32)
            st["slot"] = (order[:T] * _PAGE + st["pos"] % _PAGE).to(torch.int32)
            if T > 8:
                st["slot"][-1] = -1  # a padding row of the step's batch size
        else:  # a chunk of one prompt
            st["pos"] = (t + 160).to(torch.int32)
            st["slot"] = (order[t // _PAGE] * _PAGE + t % _PAGE).to(torch.int32)
        st["k"], st["v"] = _cache(gen, dtype, pages, kv, D)
        st["q"] = torch.empty(T, q, D, dtype=dtype, device=_device)
        st["scores"] = torch.rand(pages, kv, _PAGE, generator=gen, device=_device) if case["track"] else None
        st["positions"] = torch.full((pages, kv, _PAGE), -1, dtype=torch.int32, device=_device) if case["track"] else None
        return st
    lens = _lens(case)
    st["bt"], pages = _pages(lens, gen)
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device=_device)
    st["k"], st["v"] = _cache(gen, dtype, pages, kv, D)
    if case["op"] == "scored":
        R, Q, q = case["requests"], case["queries"], case["q_heads"]
        st["q"] = _randn(gen, dtype, R, Q, q, D) * 1.5
        st["out"] = torch.empty_like(st["q"])
        st["lse"] = torch.empty(R, Q, q, dtype=torch.float32, device=_device)
        st["scores"] = torch.rand(pages, kv, _PAGE, generator=gen, device=_device)
        return st
    # eviction: weights spread over decades, some tokens never attended to
    R, b = case["requests"], case["budget"]
    j = torch.arange(max(lens), device=_device)
    if case["steady"]:  # tokens that earlier evictions left in any order, then the new ones
        older = torch.rand(R, kv, b, generator=gen, device=_device).argsort(-1) * 3
        pos = torch.cat([older, (2 * b + j[b:]).expand(R, kv, -1)], -1)[:, :, :j.numel()]
        last = torch.clamp(st["lens"], min=b) + 2 * b - 1
    else:  # a prompt as prefill wrote it
        pos = j.expand(R, kv, -1)
        last = st["lens"] - 1
    score = torch.exp(2.0 * torch.randn(R, kv, j.numel(), generator=gen, device=_device))
    score = score * (torch.rand(R, kv, j.numel(), generator=gen, device=_device) > 0.1)
    st["last"] = last.to(torch.int32)
    fresh = torch.zeros(2, pages, kv, _PAGE, dtype=torch.int32, device=_device)
    at = _slot_index(st, j.numel())
    fresh[1].view(torch.float32).view(-1)[at.reshape(-1)] = score.reshape(-1)
    fresh[0].view(-1)[at.reshape(-1)] = pos.reshape(-1).to(torch.int32)
    fresh[:, -1] = 0
    st["fresh"], st["track"] = fresh, fresh.clone()
    st["positions"], st["scores"] = st["track"][0], st["track"][1].view(torch.float32)
    return st


def _slot_index(st, n):
    """[R, Hkv, n] flat index of each cached token in a [pages, Hkv, page] tensor; the last page behind a row's end."""
    kv, pages = st["k"].shape[1], st["k"].shape[0]
    j = torch.arange(n, device=st["k"].device)
    page = st["bt"].long()[:, j // _PAGE]
    page = torch.where(j[None, :] < st["lens"][:, None], page, torch.full_like(page, pages - 1))
    h = torch.arange(kv, device=page.device)
    return (page[:, None, :] * kv + h[None, :, None]) * _PAGE + (j % _PAGE)


# ------------------------------------------------------------------ one pass
def run(state):
    return {"append": _append, "scored": _scored, "evict": _evict}[state["op"]](state)


def _append(st):
    q_heads, kv = st["q_heads"], st["kv_heads"]
    if own:
        from sched_pass_b200 import ops
        ops.qk_norm_rope_kv_append(st["qkv"], st["qw"], st["kw"], _EPS, st["pos"], st["slot"], st["table"], st["q"],
                                   st["k"], st["v"], q_heads, kv, scores=st["scores"], positions=st["positions"])
    else:
        T, D, half = st["tokens"], st["dim"], st["rot"] // 2
        x = st["qkv"].view(T, q_heads + 2 * kv, D)
        qk = x[:, :q_heads + kv].float()
        w = torch.cat([st["qw"].float().expand(q_heads, D), st["kw"].float().expand(kv, D)])
        y = qk * torch.rsqrt((qk * qk).mean(-1, keepdim=True) + _EPS) * w
        cs = st["table"][st["pos"].long()]
        c, s = cs[:, None, :, 0], cs[:, None, :, 1]
        a, b = y[..., :half], y[..., half:2 * half]
        y = torch.cat([a * c - b * s, b * c + a * s, y[..., 2 * half:]], -1).to(st["k"].dtype)
        st["q"].copy_(y[:, :q_heads])
        # rows without a slot write the last page, which no request has, its own values
        slot, none = st["slot"].long(), (st["slot"] < 0)
        page = torch.where(none, torch.full_like(slot, st["k"].shape[0] - 1), slot // _PAGE)
        off = torch.where(none, torch.zeros_like(slot), slot % _PAGE)
        keep = none[:, None, None]
        st["k"][page, :, off] = torch.where(keep, st["k"][page, :, off], y[:, q_heads:])
        st["v"][page, :, off] = torch.where(keep, st["v"][page, :, off], x[:, q_heads + kv:])
        if st["track"]:
            st["scores"][page, :, off] = torch.where(none[:, None], st["scores"][page, :, off], torch.zeros_like(st["scores"][page, :, off]))
            st["positions"][page, :, off] = torch.where(none[:, None], st["positions"][page, :, off], st["pos"][:, None].expand(T, kv))
    out = {"q": st["q"], "k": st["k"], "v": st["v"]}
    if st["track"]:
        out["scores"], out["positions"] = st["scores"], st["positions"]
    return out


def _scored(st):
    scale = 1.0 / math.sqrt(st["dim"])
    if own:
        from sched_pass_b200 import ops
        ops.attention_decode_scored(st["q"], st["out"], st["k"], st["v"], st["bt"], st["lens"], scale, st["scores"],
                                    lse=st["lse"], max_len=st["len"])
        return {"out": st["out"], "lse": st["lse"], "scores": st["scores"]}
    R, Q, Hq, D = st["q"].shape
    kv, n = st["kv_heads"], st["bt"].shape[1] * _PAGE
    g = Hq // kv
    bt = st["bt"].long()
    k = st["k"][bt].permute(0, 2, 1, 3, 4).reshape(R, kv, n, D).float()
    v = st["v"][bt].permute(0, 2, 1, 3, 4).reshape(R, kv, n, D).float()
    q = st["q"].float().view(R, Q, kv, g, D).permute(0, 2, 1, 3, 4).reshape(R, kv, Q * g, D)
    s = (q @ k.transpose(-1, -2)) * scale
    j = torch.arange(n, device=s.device)
    limit = st["lens"][:, None] - (Q - 1 - torch.arange(Q, device=s.device))[None, :]      # [R, Q]
    limit = limit.repeat_interleave(g, 1)[:, None, :, None]
    s = torch.where(j < limit, s, torch.full_like(s, -math.inf))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    lse = torch.where(total > 0, top + torch.log(total), torch.full_like(total, -math.inf))
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    o = (p @ v).view(R, kv, Q, g, D).permute(0, 2, 1, 3, 4).reshape(R, Q, Hq, D)
    st["out"].copy_(o)
    st["lse"].copy_(lse.view(R, kv, Q, g).permute(0, 2, 1, 3).reshape(R, Q, Hq))
    st["scores"].view(-1).index_add_(0, _slot_index(st, n).reshape(-1), p.sum(2).reshape(-1))
    return {"out": st["out"], "lse": st["lse"], "scores": st["scores"]}


def _evict(st):
    # the weights that the tokens have by now: attention has added to them since the last pass
    st["track"].copy_(st["fresh"])
    b, recent, sink = st["budget"], st["recent"], st["sink"]
    if own:
        from sched_pass_b200 import ops
        lens = ops.kv_evict(st["k"], st["v"], st["scores"], st["positions"], st["bt"], st["lens"], st["last"], b,
                            recent, sink=sink, max_len=st["len"])
        return {"k": st["k"], "v": st["v"], "scores": st["scores"], "positions": st["positions"], "lens": lens}
    R, kv, n, D = st["requests"], st["kv_heads"], st["bt"].shape[1] * _PAGE, st["dim"]
    at = _slot_index(st, n)
    score, pos = st["scores"].reshape(-1)[at], st["positions"].reshape(-1)[at]
    j = torch.arange(n, device=at.device).expand(R, kv, n)
    inside = j < st["lens"][:, None, None]
    kept_anyway = (pos > (st["last"] - recent)[:, None, None]) | (pos < sink)
    key = torch.where(kept_anyway, torch.full_like(score, 3e38), torch.nan_to_num(score, nan=-3e38))
    key = torch.where(inside, key, torch.full_like(key, -math.inf))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    keep = torch.zeros_like(key, dtype=torch.bool).scatter_(-1, order[..., :b], True) & inside
    hole, mover = ~keep & inside & (j < b), keep & (j >= b)
    # the i-th mover goes to the i-th hole, both in the order of the slots
    spare = torch.full_like(j, n)
    of_rank = torch.zeros(R, kv, n + 1, dtype=torch.int64, device=at.device)
    of_rank.scatter_(-1, torch.where(mover, mover.cumsum(-1) - 1, spare), j)
    src = torch.where(hole, of_rank.gather(-1, hole.cumsum(-1).clamp(min=1) - 1), j)[..., :b]
    # slots that keep their token write it back to themselves
    to, frm = at[..., :src.shape[-1]].reshape(-1), at.gather(-1, src).reshape(-1)
    # rows are [pages, Hkv, page]-ordered, so a slot's flat index is its row of K and V
    for x in (st["k"].view(-1, D), st["v"].view(-1, D), st["scores"].view(-1), st["positions"].view(-1)):
        x[to] = x[frm]
    lens = torch.clamp(st["lens"], max=b)
    return {"k": st["k"], "v": st["v"], "scores": st["scores"], "positions": st["positions"], "lens": lens}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    k, v, D, kv = st["k"].double(), st["v"].double(), case["dim"], case["kv_heads"]
    if case["op"] == "append":
        T, nq, rot = case["tokens"], case["q_heads"], case["rot"]
        heads = st["qkv"].double().reshape(T, -1, D)
        norm = heads / torch.sqrt(heads.pow(2).sum(-1, keepdim=True) / D + _EPS)
        norm[:, :nq] *= st["qw"].double()
        norm[:, nq:] *= st["kw"].double()
        turn = torch.view_as_complex(st["table"].double())[st["pos"].long()][:, None, :]
        z = torch.complex(norm[..., :rot // 2], norm[..., rot // 2:rot]) * turn
        full = torch.cat([z.real, z.imag, norm[..., rot:]], -1)
        used = (st["slot"] >= 0).nonzero()[:, 0]
        page, off = (st["slot"].long()[used] // _PAGE), (st["slot"].long()[used] % _PAGE)
        k[page, :, off] = full[used, nq:nq + kv]
        v[page, :, off] = heads[used, nq + kv:]
        out = {"q": full[:, :nq].contiguous(), "k": k, "v": v}
        if case["track"]:
            scores, positions = st["scores"].double(), st["positions"].clone()
            scores[page, :, off] = 0.0
            positions[page, :, off] = st["pos"][used][:, None].expand(-1, kv)
            out["scores"], out["positions"] = scores, positions
        return out
    lens = _lens(case)
    if case["op"] == "scored":
        R, Q, Hq, _ = st["q"].shape
        g = Hq // kv
        out = torch.zeros(R, Q, Hq, D, dtype=torch.float64, device=k.device)
        lse = torch.full((R, Q, Hq), -math.inf, dtype=torch.float64, device=k.device)
        scores = st["scores"].double()
        for r, n in enumerate(lens):
            pages = st["bt"][r, :-(-n // _PAGE)].long()
            weight = torch.zeros(kv, pages.numel() * _PAGE, dtype=torch.float64, device=k.device)
            keys = k[pages].transpose(0, 1).flatten(1, 2)
            vals = v[pages].transpose(0, 1).flatten(1, 2)
            for i in range(Q):
                seen = n - (Q - 1 - i)
                if seen <= 0:
                    continue
                one = st["q"][r, i].double().view(kv, g, D)
                logit = torch.einsum("hgd,hnd->hgn", one, keys[:, :seen]) / math.sqrt(D)
                z = torch.logsumexp(logit, -1)
                p = torch.exp(logit - z[..., None])
                out[r, i] = torch.einsum("hgn,hnd->hgd", p, vals[:, :seen]).reshape(Hq, D)
                lse[r, i] = z.reshape(-1)
                weight[:, :seen] += p.sum(1)
            scores[pages] += weight.view(kv, -1, _PAGE).transpose(0, 1)
        return {"out": out, "lse": lse, "scores": scores}
    # eviction: only whole rows move, so the values themselves are exact
    b, recent, sink = case["budget"], case["recent"], case["sink"]
    scores, positions = st["scores"].cpu().numpy().astype(np.float64), st["positions"].cpu().numpy().copy()
    table, last = st["bt"].cpu().numpy(), st["last"].cpu().numpy()
    to, frm = [], []
    for r, n in enumerate(lens):
        if n <= b:
            continue
        slots = np.arange(n)
        for h in range(kv):
            row = (table[r, slots // _PAGE].astype(np.int64) * kv + h) * _PAGE + slots % _PAGE
            at = positions.reshape(-1)[row]
            safe = (at > last[r] - recent) | (at < sink)
            best = np.lexsort((slots, -scores.reshape(-1)[row], ~safe))[:b]
            kept = np.zeros(n, bool)
            kept[best] = True
            frm.append(row[b:][kept[b:]])
            to.append(row[:b][~kept[:b]])
    if to:
        to, frm = np.concatenate(to), np.concatenate(frm)
        scores.reshape(-1)[to] = scores.reshape(-1)[frm]
        positions.reshape(-1)[to] = positions.reshape(-1)[frm]
        dst, src = torch.from_numpy(to).to(k.device), torch.from_numpy(frm).to(k.device)
        k.view(-1, D)[dst] = k.view(-1, D)[src]
        v.view(-1, D)[dst] = v.view(-1, D)[src]
    return {"k": k, "v": v, "scores": torch.from_numpy(scores).to(k.device),
            "positions": torch.from_numpy(positions).to(k.device), "lens": torch.clamp(st["lens"], max=b)}
