"""Cases of the bounded K/V cache's operators: attention that keeps, beside its
result, how much weight every cached key has received (chunks of prompt tokens and
single tokens), the choice of the keys that stay when a cache is cut to a budget, and
the closing of the gaps in its pages.

`run` computes them in plain torch operations, or, with `own`, by kaito_amd.ops.
"""
import math

import torch

own = False

PAGE = 16                 # keys of a page
E4M3 = torch.float8_e4m3fn

# (query heads, key/value heads, head size) of the catalog's models
LAYOUTS = {
    "32/8x128": (32, 8, 128),
    "28/4x128": (28, 4, 128),     # groups of 7
    "32/32x64": (32, 32, 64),     # a key/value head for each query head
    "64/8x64": (64, 8, 64),       # groups of 8, with sinks
    "8/4x256": (8, 4, 256),
}


def listed():
    return [
        # a short suffix behind a cached prefix, as when a few drafted tokens are
        # checked: the launches count
        dict(name="chunk few", op="chunk", layout="32/8x128", batch=2, chunk_lo=5,
             chunk_hi=16, past_lo=130, past_hi=400, fp8=False, sinks=False),
        # chunked prefill of eight prompts of unlike lengths
        dict(name="chunk ragged", op="chunk", layout="32/8x128", batch=8, chunk_lo=97,
             chunk_hi=1000, past_lo=0, past_hi=4001, fp8=False, sinks=False),
        # a chunk of one long prompt
        dict(name="chunk long", op="chunk", layout="32/8x128", batch=1, chunk_lo=2048,
             chunk_hi=2048, past_lo=14336, past_hi=14336, fp8=False, sinks=False),
        # 8-bit pages, heads of 64 and sinks
        dict(name="chunk fp8 sinks", op="chunk", layout="64/8x64", batch=4, chunk_lo=333,
             chunk_hi=1200, past_lo=100, past_hi=6000, fp8=True, sinks=True),
        # one user's next token
        dict(name="token one", op="token", layout="32/8x128", batch=1, past_lo=216,
             past_hi=216, fp8=False, sinks=False),
        # a full decode step with caches of up to 4096 keys
        dict(name="token batch", op="token", layout="32/8x128", batch=64, past_lo=1500,
             past_hi=4095, fp8=False, sinks=False),
        # few users with long 8-bit caches
        dict(name="token long fp8", op="token", layout="64/8x64", batch=16, past_lo=8000,
             past_hi=16000, fp8=True, sinks=True),
        # many short conversations, heads of 256
        dict(name="token many", op="token", layout="8/4x256", batch=256, past_lo=30,
             past_hi=1000, fp8=False, sinks=False),
        # caches a little above their budget, as a server cuts them
        dict(name="choose batch", op="choose", kv_heads=8, batch=64, len_lo=4100,
             len_hi=4352, budget=4096, recent=512),
        # long prompts, cut to half after their prefill
        dict(name="choose long", op="choose", kv_heads=8, batch=4, len_lo=20000,
             len_hi=32768, budget=16384, recent=1024),
        # the pages behind such choices: a few short caches, and a whole batch
        dict(name="close few", op="close", layout="32/8x128", batch=4, len_lo=400,
             len_hi=700, budget=512, recent=64),
        dict(name="close batch", op="close", layout="32/8x128", batch=64, len_lo=4100,
             len_hi=4352, budget=4096, recent=512),
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["chunk", "token", "choose", "close"])
    layout = rng.choice(sorted(LAYOUTS))
    QH, KH, D = LAYOUTS[layout]
    if op == "chunk":
        batch = size(1, 8)
        hi = size(4, 2048 // batch)
        past = size(16, 14000) if batch < 3 else size(16, 4000)
        return dict(op=op, layout=layout, batch=batch, chunk_lo=rng.randint(1, hi),
                    chunk_hi=hi, past_lo=rng.randint(0, past), past_hi=past,
                    fp8=rng.random() < 0.3, sinks=rng.random() < 0.3)
    if op == "token":
        batch = size(1, 256)
        past = size(16, min(16000, 260000 * 1024 // (batch * KH * D)))
        return dict(op=op, layout=layout, batch=batch, past_lo=rng.randint(0, past),
                    past_hi=past, fp8=rng.random() < 0.3, sinks=rng.random() < 0.3)
    batch = size(1, 64)
    budget = size(64, min(16384, 262144 // batch))
    most = budget + size(1, budget)
    more = dict(kv_heads=KH) if op == "choose" else dict(layout=layout)
    if op == "close":
        budget = min(budget, 260000 * 1024 // (batch * KH * D))
        most = min(most, 2 * budget)
    return dict(op=op, batch=batch, len_lo=rng.randint(budget // 2, most), len_hi=most,
                budget=budget, recent=rng.randint(0, budget // 2), **more)


def spread(lo, hi, n):
    """n lengths between lo and hi, the last one hi; the same for every seed."""
    return [lo + int((hi - lo) * ((i + 1) * 0.6180339887 % 1.0)) for i in range(n - 1)] + [hi]


def lengths(case):
    """(new tokens, keys) of every sequence of a case."""
    n = case["batch"]
    if case["op"] in ("choose", "close"):
        return [0] * n, spread(case["len_lo"], case["len_hi"], n)
    new = spread(case["chunk_lo"], case["chunk_hi"], n) if case["op"] == "chunk" else [1] * n
    return new, [p + c for p, c in zip(spread(case["past_lo"], case["past_hi"], n), new)]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    new, lens = lengths(case)
    B, KH = case["batch"], case["kv_heads"] if case["op"] == "choose" else LAYOUTS[case["layout"]][1]
    pages = [-(-n // PAGE) for n in lens]
    total = sum(pages)
    # pages of a pool in no order; one spare page stands behind every table's end
    pool = torch.randperm(total, generator=gen, device=dev, dtype=torch.int32).tolist()
    tables = torch.full((B, max(pages)), total, dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        tables[b, :n] = torch.tensor(pool[at:at + n], dtype=torch.int32)
        at += n
    s = dict(op=case["op"], tables=tables.to(dev),
             lens=torch.tensor(lens, dtype=torch.int32, device=dev))
    # what the keys have received so far: little for most, much for a few; the new
    # tokens' slots hold what their last user left
    s["weights"] = torch.rand(total + 1, KH, PAGE, generator=gen, device=dev) ** 4 * 10
    if case["op"] == "choose":
        s.update(budget=case["budget"], recent=case["recent"])
        return s
    QH, KH, D = LAYOUTS[case["layout"]]

    def cache():
        return torch.randn(total + 1, KH, PAGE, D, generator=gen, device=dev, dtype=torch.bfloat16)

    s.update(k=cache(), v=cache())
    if case["op"] == "close":
        s["kept"], s["kept_lens"] = choose(s["weights"], s["tables"], s["lens"],
                                           case["budget"], case["recent"])
        return s
    if case["fp8"]:
        s["k"], s["v"] = (t.to(E4M3).view(torch.uint8) for t in (s["k"], s["v"]))
    T = sum(new)
    # scores with a spread of two: a few keys of a row carry most of its weight
    s["q"] = torch.randn(T, QH, D, generator=gen, device=dev).mul_(2).to(torch.bfloat16)
    s["scale"] = D ** -0.5
    s["sinks"] = torch.randn(QH, generator=gen, device=dev) if case["sinks"] else None
    if case["op"] == "chunk":
        cu = torch.zeros(B + 1, dtype=torch.int32)
        cu[1:] = torch.tensor(new).cumsum(0)
        s.update(cu=cu.to(dev), most=max(new), tiles=None)
        # 64-row query tiles of the step, the ones with the most keys first
        tiles = [(-(lens[b] - new[b] + i), b, i) for b in range(B) for i in range(0, new[b], 64)]
        s["tiles"] = tuple(torch.tensor([t[j] for t in sorted(tiles)], dtype=torch.int32, device=dev)
                           for j in (1, 2))
    else:
        s.update(cu=torch.arange(B + 1, dtype=torch.int32, device=dev), most=1)
    return s


# ---- plain forms

def rows_of(cache, tables):
    """The cache's rows of every sequence, in 32 bits: [B, KH, keys, D]."""
    x = cache.view(E4M3) if cache.dtype == torch.uint8 else cache
    x = x[tables.long()].float()                    # [B, pages, KH, PAGE, D]
    return x.transpose(1, 2).flatten(2, 3)


def attend(q, k_cache, v_cache, weights, cu, most, lens, tables, scale, sinks):
    """Causal attention of each sequence's newest tokens over its pages; adds every
    key's weights to `weights`, where the new tokens' keys begin anew."""
    k, v = rows_of(k_cache, tables), rows_of(v_cache, tables)
    B, KH, L, D = k.shape
    QH = q.size(1)
    G = QH // KH
    n = (cu[1:] - cu[:-1]).long()
    i = torch.arange(most, device=q.device)
    real = i < n[:, None]                                          # [B, most]
    at = torch.where(real, cu[:-1, None].long() + i, 0)
    x = q[at].float().view(B, most, KH, G, D).permute(0, 2, 3, 1, 4)
    s = (x.reshape(B, KH, G * most, D) @ k.transpose(2, 3)).view(B, KH, G, most, L) * scale
    j = torch.arange(L, device=q.device)
    past = (lens.long() - n)[:, None]
    seen = (j <= (past + i)[:, :, None]) & real[:, :, None]        # [B, most, L]
    s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp_min(-1e30)
    if sinks is not None:
        sink = sinks.float().view(KH, G, 1, 1)
        top = torch.maximum(top, sink)
    p = (s - top).exp_()
    den = p.sum(-1, keepdim=True)
    if sinks is not None:
        den = den + (sink - top).exp()
    p /= den.clamp_min(1e-30)
    o = (p.reshape(B, KH, G * most, L) @ v).view(B, KH, G, most, D)
    out = torch.empty_like(q)
    o = o.permute(0, 3, 1, 2, 4).reshape(B * most, QH, D).to(q.dtype)
    # row i of sequence b is token cu[b] + i: the tokens in order, from the padded rows
    t = torch.arange(q.size(0), device=q.device)
    b = torch.searchsorted(cu[1:].long(), t, right=True)
    out.copy_(o[b * most + t - cu[:-1].long()[b]])
    w = p.sum((2, 3)).view(B, KH, L // PAGE, PAGE).transpose(1, 2)  # [B, pages, KH, PAGE]
    old = weights[tables.long()]
    j = j.view(1, L // PAGE, 1, PAGE)
    first, end = past.view(B, 1, 1, 1), lens.view(B, 1, 1, 1)
    weights[tables.long()] = torch.where(j < first, old + w, torch.where(j < end, w, old))
    return out, weights


def choose(weights, tables, lens, budget, recent):
    """The keys that stay: the newest `recent` and, of the others, those with the most
    weight over all heads. Returns their places [B, budget] in order (-1 behind the
    last) and how many they are."""
    w = weights[tables.long()].double().sum(2).float().flatten(1)   # [B, keys]
    j = torch.arange(w.size(1), device=w.device)
    end = lens.long()[:, None]
    w = torch.where(j >= end - recent, math.inf, w)
    w = torch.where(j < end, w, -1.0)
    order = w.sort(dim=1, descending=True, stable=True).indices[:, :budget]
    if order.size(1) < budget:
        order = torch.nn.functional.pad(order, (0, budget - order.size(1)))
    n = lens.clamp_max(budget)
    none = 1 << 30
    order = torch.where(torch.arange(budget, device=w.device) < n[:, None], order, none)
    order = order.sort(dim=1).values
    return torch.where(order < none, order, -1).int(), n


def close(k_cache, v_cache, weights, tables, kept, kept_lens):
    """Key kept[b, i] goes to place i of its sequence's pages, in all three arrays."""
    i = torch.arange(kept.size(1), device=kept.device).expand_as(kept)
    i = i[:, :tables.size(1) * PAGE]
    src = torch.where(i < kept_lens[:, None], kept[:, :i.size(1)].long(), i)
    t = tables.long()
    to, of = t.gather(1, i // PAGE), t.gather(1, src // PAGE)
    for x in (k_cache, v_cache, weights):
        x[to, :, i % PAGE] = x[of, :, src % PAGE]
    return k_cache, v_cache, weights


def run(s):
    if own:
        from kaito_amd import ops
        if s["op"] == "chunk":
            out = ops.context_attention_weights(
                s["q"], s["k"], s["v"], s["weights"], s["cu"], s["lens"], s["tables"],
                s["scale"], sinks=s["sinks"], tiles=s["tiles"])
            return out, s["weights"]
        if s["op"] == "token":
            out = ops.paged_attention_weights(
                s["q"], s["k"], s["v"], s["weights"], s["tables"], s["lens"], s["scale"],
                sinks=s["sinks"])
            return out, s["weights"]
        if s["op"] == "choose":
            return ops.heavy_keys(s["weights"], s["tables"], s["lens"], s["budget"], s["recent"])
        ops.compact_pages(s["k"], s["v"], s["weights"], s["tables"], s["kept"], s["kept_lens"])
        return s["k"], s["v"], s["weights"]
    if s["op"] in ("chunk", "token"):
        return attend(s["q"], s["k"], s["v"], s["weights"], s["cu"], s["most"], s["lens"],
                      s["tables"], s["scale"], s["sinks"])
    if s["op"] == "choose":
        return choose(s["weights"], s["tables"], s["lens"], s["budget"], s["recent"])
    return close(s["k"], s["v"], s["weights"], s["tables"], s["kept"], s["kept_lens"])


def work(case):
    new, lens = lengths(case)
    if case["op"] == "choose":
        kept = sum(min(n, case["budget"]) for n in lens)
        return dict(bytes=4 * (sum(lens) * case["kv_heads"] + kept), flops=sum(lens) * case["kv_heads"])
    QH, KH, D = LAYOUTS[case["layout"]]
    if case["op"] == "close":
        # nearly every kept key of a cache above its budget changes place
        moved = sum(case["budget"] for n in lens if n > case["budget"])
        return dict(bytes=2 * moved * KH * (2 * D * 2 + 4) + 4 * moved, flops=0)
    elem = 1 if case["fp8"] else 2
    pairs = sum(c * (n - c) + c * (c + 1) // 2 for c, n in zip(new, lens))
    past = sum(n - c for c, n in zip(new, lens))
    return dict(bytes=2 * 2 * sum(new) * QH * D + sum(lens) * KH * 2 * D * elem
                + 4 * KH * (past + sum(lens)), flops=4 * pairs * QH * D)


def exact(case, seed):
    """From the definitions in 64 bits, sequence by sequence."""
    if case["op"] == "choose":
        return None                       # whole numbers
    s = prepare(case, seed)
    weights = s["weights"].double()

    def pages(cache, b, n):
        x = cache.view(E4M3) if cache.dtype == torch.uint8 else cache
        slot = torch.arange(n, device=x.device)
        return x[s["tables"][b].long()[slot // PAGE], :, slot % PAGE].double()   # [n, KH, D]

    if case["op"] == "close":
        caches = [s["k"].double(), s["v"].double(), weights]
        for b, n in enumerate(s["kept_lens"].tolist()):
            place = torch.arange(n, device=weights.device)
            src, t = s["kept"][b, :n].long(), s["tables"][b].long()
            for x in caches:
                moved = x[t[src // PAGE], :, src % PAGE]
                x[t[place // PAGE], :, place % PAGE] = moved
        return tuple(caches)
    cu, lens = s["cu"].tolist(), s["lens"].tolist()
    QH, KH, D = LAYOUTS[case["layout"]]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=weights.device)
    for b, n in enumerate(lens):
        k, v = pages(s["k"], b, n), pages(s["v"], b, n)
        m = cu[b + 1] - cu[b]
        slot = torch.arange(n, device=k.device)
        t = s["tables"][b].long()[slot // PAGE]
        later = slot[None, :] > torch.arange(n - m, n, device=k.device)[:, None]
        mass = torch.zeros(n, KH, dtype=torch.float64, device=k.device)
        for h in range(QH):
            g = h // (QH // KH)
            z = s["q"][cu[b]:cu[b + 1], h].double() @ k[:, g].t() * s["scale"]
            z[later] = -math.inf
            if s["sinks"] is not None:
                z = torch.cat([z, s["sinks"][h].double().expand(m, 1)], 1)
            p = torch.softmax(z, 1)[:, :n]
            out[cu[b]:cu[b + 1], h] = p @ v[:, g]
            mass[:, g] += p.sum(0)
        before = weights[t, :, slot % PAGE]
        before[n - m:] = 0
        weights[t, :, slot % PAGE] = before + mass
    return out, weights
