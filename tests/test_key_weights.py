"""A cache kept to a budget: attention that keeps what every key receives, the
choice of the keys that stay and the closing of the gaps, against plain loops in 64
bits.

Tolerances. Outputs are bf16: half a step is 2^-8 of the value. Chunks' weights go
into the product with V as bf16, which adds 2^-8 of sum p |v|; single tokens' go in
whole. A score is a sum of D products in f32, off by at most (D + 2) 2^-24 of the
sum of their sizes, twice that for a weight (its own and its row's sum), and e4m3
and bf16 operands are exact. A key's entry is a sum of such weights and its old
value, each step of which rounds to 2^-24; 2^-20 of it covers the exponential, the
reciprocal and up to a few thousand additions of a random sign."""
import math

import pytest
import torch

from kaito_amd import ops

CPU_OR_GPU = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
PAGE = 16


def _pages(lens, KH, D, fp8=False, width=None, seed=0):
    """Caches and tables of sequences of `lens` keys, in pages of no order; what
    no sequence owns holds NaN (in e4m3 0x7f is one)."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // PAGE) for n in lens]
    width = max(width or 0, max(need + [1]))
    perm = torch.randperm(sum(need) + 2, generator=g).int()
    tables = torch.full((len(lens), width), int(perm[-1]), dtype=torch.int32)
    shape = (len(perm), KH, PAGE, D)
    k, v = (torch.full(shape, math.nan) for _ in range(2))
    w = torch.full(shape[:3], math.nan)
    at = 0
    for b, n in enumerate(lens):
        tables[b, :need[b]] = perm[at:at + need[b]]
        at += need[b]
        for i in range(0, n, PAGE):
            p, m = tables[b, i // PAGE], min(PAGE, n - i)
            k[p, :, :m] = torch.randn(KH, m, D, generator=g)
            v[p, :, :m] = torch.randn(KH, m, D, generator=g)
            w[p, :, :m] = torch.rand(KH, m, generator=g) ** 3 * 5
    if fp8:
        k, v = (t.to(torch.float8_e4m3fn).view(torch.uint8) for t in (k, v))
    else:
        k, v = k.bfloat16(), v.bfloat16()
    return k, v, w, tables


def _f64(cache):
    x = cache.cpu()
    return (x.view(torch.float8_e4m3fn) if x.dtype == torch.uint8 else x).double()


def _oracle(q, k, v, w, new, lens, tables, scale, sinks):
    """(output, its tolerance without its own rounding, weights, their
    tolerance) in 64 bits."""
    k, v, q, w = _f64(k), _f64(v), q.cpu().double(), w.cpu().double()
    KH, D = k.size(1), k.size(3)
    G = q.size(1) // KH
    out, near = torch.zeros_like(q), torch.zeros_like(q)
    off = torch.zeros_like(w)
    at = 0
    for b, (n, L) in enumerate(zip(new, lens)):
        if n == 0 or L == 0:
            at += n
            continue
        j = torch.arange(L)
        p = tables[b].cpu().long()[j // PAGE]
        kb, vb = k[p, :, j % PAGE], v[p, :, j % PAGE]              # [L, KH, D]
        later = j > torch.arange(L - n, L)[:, None]
        gain, gain_off = torch.zeros(L, KH).double(), torch.zeros(L, KH).double()
        for h in range(G * KH):
            x = q[at:at + n, h]
            s = (x @ kb[:, h // G].T * scale).masked_fill(later, -math.inf)
            top = s.amax(1, keepdim=True)
            if sinks is not None:
                top = top.maximum(sinks[h].double())
            e = (s - top).exp()
            den = e.sum(1, keepdim=True)
            if sinks is not None:
                den = den + (sinks[h].double() - top).exp()
            e = e / den
            out[at:at + n, h] = e @ vb[:, h // G]
            near[at:at + n, h] = e @ vb[:, h // G].abs()
            gain[:, h // G] += e.sum(0)
            size = (x.abs() @ kb[:, h // G].abs().T).amax(1) * abs(scale)
            rel = 2 * (D + 2) * 2.0 ** -24 * size + 2.0 ** -20
            gain_off[:, h // G] += (e * rel[:, None]).sum(0)
        old = w[p, :, j % PAGE]
        old[L - n:] = 0
        w[p, :, j % PAGE] = old + gain
        off[p, :, j % PAGE] = gain_off + (old + gain) * 2.0 ** -20
        at += n
    return out, near, w, off


def _run(dev, layout, new, past, fp8=False, sinks=False, width=None, token=False,
         seed=0):
    QH, KH, D = layout
    lens = [a + b for a, b in zip(new, past)]
    k, v, w, tables = _pages(lens, KH, D, fp8, width, seed)
    for b, (n, L) in enumerate(zip(new, lens)):    # what the slot's last user left
        for j in range(L - n, L):
            w[tables[b, j // PAGE], :, j % PAGE] = (math.nan, 3e38)[j % 2]
    g = torch.Generator().manual_seed(seed + 1)
    # rows cut from a fused projection
    q = torch.randn(sum(new), QH * D + 64, generator=g).mul(2).bfloat16().to(dev)
    q = q[:, :QH * D].unflatten(1, (QH, D))
    s = torch.randn(QH, generator=g) if sinks else None
    scale = D ** -0.5
    want, near, want_w, off = _oracle(q, k, v, w, new, lens, tables, scale, s)
    k, v, got_w, tables, lens_t = (
        t.to(dev) for t in (k, v, w, tables, torch.tensor(lens, dtype=torch.int32)))
    s = s.to(dev) if sinks else None
    if token:
        out = ops.paged_attention_weights(q, k, v, got_w, tables, lens_t, scale, s)
    else:
        cu = torch.tensor([0] + new).cumsum(0).int().to(dev)
        out = ops.context_attention_weights(q, k, v, got_w, cu, lens_t, tables,
                                            scale, s)
    out, got_w = out.cpu().double(), got_w.cpu().double()
    bf16 = 2.0 ** -8
    room = bf16 * want.abs() + (near * (2.0 ** -14 if token else bf16)) + 2.0 ** -20
    assert ((out - want).abs() <= room).all(), ((out - want).abs() - room).max()
    live = off > 0
    assert ((got_w - want_w).abs() <= off)[live].all()
    # nothing else has changed
    assert torch.equal(got_w[~live].float().view(torch.int32),
                       w[~live].view(torch.int32))


LAYOUTS = [(4, 1, 64), (8, 1, 64), (2, 2, 64), (8, 2, 128), (7, 1, 128),
           (3, 3, 128), (4, 2, 256), (4, 1, 256)]


@pytest.mark.parametrize("dev", CPU_OR_GPU)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("fp8", [False, True])
def test_chunks(dev, layout, fp8):
    """Edges of the 32- and 64-row tiles, of pages and of 64 and 256 keys;
    prompts whole and behind a past, and a sequence without rows."""
    _run(dev, layout, [1, 0, 17, 64, 33, 65, 5], [0, 40, 0, 1, 223, 191, 252],
         fp8=fp8, sinks=not fp8, width=24)


@pytest.mark.parametrize("dev", CPU_OR_GPU)
@pytest.mark.parametrize("layout", [(8, 2, 128), (5, 1, 128), (2, 1, 256)])
def test_long_chunks(dev, layout):
    _run(dev, layout, [300, 129], [700, 0], sinks=True, seed=3)


@pytest.mark.gpu
def test_chunk_over_many_keys():
    _run("cuda", (4, 1, 128), [70], [9000])
    _run("cuda", (16, 2, 64), [1030], [3], fp8=True)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", [(8, 2, 64), (8, 2, 128), (7, 1, 128),
                                    (2, 2, 256)])
@pytest.mark.parametrize("sinks", [False, True])
def test_few_rows_over_many_keys(layout, sinks):
    """Keys shared out over workgroups; shares that a sequence does not reach."""
    _run("cuda", layout, [5, 1, 70, 0, 33], [5000, 0, 130, 900, 2049], fp8=sinks,
         sinks=sinks, seed=7)
    _run("cuda", layout, [3], [13], sinks=sinks, width=600)


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [2, 63, 64, 65])
def test_many_chunks(seqs):
    """Sequences by the lengths of their chunks, equal ones among them; enough
    keys for workgroups of 256."""
    _run("cuda", (4, 2, 64), [(7 * i) % 13 for i in range(seqs)],
         [(31 * i) % 97 for i in range(seqs)], width=900 // seqs * 8, seed=seqs)


@pytest.mark.parametrize("dev", CPU_OR_GPU)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("fp8", [False, True])
def test_tokens(dev, layout, fp8):
    lens = [1, 15, 16, 17, 31, 32, 33, 0, 64, 65, 127, 129, 300]
    new = [1] * len(lens)
    _run(dev, layout, new, [n - 1 for n in lens], fp8=fp8, sinks=not fp8,
         token=True)


@pytest.mark.gpu
@pytest.mark.parametrize("D,KH,lens,width", [
    (128, 8, [40, 200, 7] * 11, 13),          # pairs beyond a workgroup per CU
    (128, 2, [1900, 33, 0, 2047], 128),       # few pairs, a long table: splits
    (128, 1, [5000], 700), (256, 1, [700, 3], 200),
    (64, 8, [17], 4096),                      # splits that are all but one empty
    (64, 8, [30, 5, 64, 70] * 40, 5),
    (128, 8, [64] * 140, 4),                  # two waves per pair
])
@pytest.mark.parametrize("fp8", [False, True])
def test_token_launch_rules(D, KH, lens, width, fp8):
    _run("cuda", (4 * KH, KH, D), [1] * len(lens), [n - 1 for n in lens], fp8=fp8,
         sinks=fp8, width=width, token=True)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", [(7, 1, 128), (16, 2, 128), (4, 4, 64),
                                    (3, 1, 128)])
def test_tokens_of_other_groups_in_splits(layout):
    _run("cuda", layout, [1] * 4, [2499, 8, 1300, 0], sinks=True, width=260,
         token=True, seed=9)


@pytest.mark.parametrize("dev", CPU_OR_GPU)
@pytest.mark.parametrize("scale", [0.0, -0.125])
def test_scales_that_are_not_positive(dev, scale):
    """Every visible key alike, and the least alike first."""
    new, past = [40, 3], [300, 0]
    lens = [a + b for a, b in zip(new, past)]
    k, v, w, tables = _pages(lens, 2, 64)
    q = torch.randn(43, 4, 64).bfloat16()
    want, near, want_w, off = _oracle(q, k, v, w, new, lens, tables, scale, None)
    cu = torch.tensor([0, 40, 43], dtype=torch.int32)
    got = w.to(dev)
    out = ops.context_attention_weights(
        q.to(dev), k.to(dev), v.to(dev), got, cu.to(dev),
        torch.tensor(lens, dtype=torch.int32).to(dev), tables.to(dev), scale)
    err = (out.cpu().double() - want).abs()
    assert (err <= 2.0 ** -8 * (want.abs() + near) + 2.0 ** -20).all()
    assert ((got.cpu().double() - want_w).abs() <= off)[off > 0].all()


@pytest.mark.gpu
def test_scores_without_a_weight():
    """Keys whose scores are minus infinity receive nothing, and a row that has
    no other key changes no entry."""
    k, v, w, t = _pages([20, 4], 1, 64)
    v[v.isnan()] = 0
    q = torch.ones(2, 1, 64).bfloat16()
    k[t[0, 0], :, 3] = -3e38                  # -3e38 * 64 ones
    k[t[1, 0], :, :4] = -3e38
    lens = torch.tensor([20, 4], dtype=torch.int32)
    args = [x.to("cuda") for x in (q, k, v)]
    for op in (ops.paged_attention_weights, ops.context_attention_weights):
        got = w.to("cuda")
        more = (torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"),) \
            if op is ops.context_attention_weights else ()
        rows = (t.to("cuda"), lens.to("cuda"))
        op(*args, got, *more, *(rows[::-1] if more else rows), 1.0)
        got = got.cpu()
        assert got[t[0, 0], 0, 3] == w[t[0, 0], 0, 3]
        assert torch.equal(got[t[1, 0], 0, :3], w[t[1, 0], 0, :3])
        assert got[t[1, 0], 0, 3] == 0        # its own key: anew, and nothing


def _heavy(w, tables, lens, budget, recent):
    """The rule, key by key."""
    kept = torch.full((len(lens), budget), -1, dtype=torch.int32)
    for b, L in enumerate(lens):
        places = list(range(L))
        if L > budget:
            total = [float(w[tables[b, j // PAGE], :, j % PAGE].double().sum()
                           .float()) for j in range(L - recent)]
            order = sorted(range(L - recent), key=lambda j: (
                -math.inf if math.isnan(total[j]) else -total[j], j))
            places = sorted(order[:budget - recent]) + places[L - recent:]
        kept[b, :len(places)] = torch.tensor(places, dtype=torch.int32)
    return kept


@pytest.mark.parametrize("dev", CPU_OR_GPU)
@pytest.mark.parametrize("budget,recent", [(1, 0), (1, 1), (64, 0), (64, 64),
                                           (100, 37), (257, 16), (600, 5)])
@pytest.mark.parametrize("kind", ["spread", "equal", "few", "zero", "signs"])
def test_heavy_keys(dev, budget, recent, kind):
    lens = [0, 1, 63, 64, 65, 100, 101, 258, 513]
    _, _, w, tables = _pages(lens, 3, 64, width=40)
    w = torch.nan_to_num(w, 7.)
    if kind == "equal":
        w.fill_(0.3)
    if kind == "few":                      # many ties of three values
        w = (w * 0.5).floor()
    if kind == "zero":
        w = w * 0 * torch.where(torch.rand(w.shape) < 0.5, 1., -1.)
    if kind == "signs":
        w = torch.where(torch.rand(w.shape) < 0.5, w, -w)
        w[tables[8, 0], 0, 3] = math.nan
        w[tables[8, 1], 1, 4] = math.inf
        w[tables[8, 1], 1, 5] = -math.inf
    kept, n = ops.heavy_keys(w.to(dev), tables.to(dev),
                             torch.tensor(lens, dtype=torch.int32, device=dev),
                             budget, recent)
    assert torch.equal(kept.cpu(), _heavy(w, tables, lens, budget, recent))
    assert n.tolist() == [min(L, budget) for L in lens]


@pytest.mark.parametrize("dev", CPU_OR_GPU)
def test_heavy_keys_of_many_heads(dev):
    """More kv heads than a short cache's choice sums by itself."""
    lens = [700, 33]
    _, _, w, tables = _pages(lens, 20, 64)
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    kept, _ = ops.heavy_keys(w.to(dev), tables.to(dev), n, 200, 10)
    assert torch.equal(kept.cpu(), _heavy(w, tables, lens, 200, 10))


@pytest.mark.parametrize("dev", CPU_OR_GPU)
def test_nothing_to_do(dev):
    """No sequences; tables without pages; no new rows at all."""
    k, v, w, tables = (t.to(dev) for t in _pages([40], 2, 64))
    before = [t.clone() for t in (k, v, w)]
    q = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device=dev)
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    zero = torch.zeros(1, dtype=torch.int32, device=dev)
    nothing = zero.new_zeros(0, 3)
    assert ops.paged_attention_weights(q, k, v, w, nothing, none,
                                       1.0).shape == q.shape
    assert ops.context_attention_weights(q, k, v, w, zero, none, nothing,
                                         1.0).shape == q.shape
    cu = torch.zeros(2, dtype=torch.int32, device=dev)
    assert ops.context_attention_weights(q, k, v, w, cu, zero + 40, tables,
                                         1.0).shape == q.shape
    kept, n = ops.heavy_keys(w, nothing, none, 8, 2)
    assert kept.shape == (0, 8) and n.shape == (0,)
    ops.compact_pages(k, v, w, nothing, kept, n)
    # a row whose table has no pages
    one = torch.ones(1, 4, 64, dtype=torch.bfloat16, device=dev)
    empty = zero.new_zeros(1, 0)
    assert (ops.paged_attention_weights(one, k, v, w, empty, zero, 1.0)
            == 0).all()
    kept, n = ops.heavy_keys(w, empty, zero, 8, 2)
    assert (kept == -1).all() and n.tolist() == [0]
    ops.compact_pages(k, v, w, empty, kept, n)
    for a, b in zip((k, v, w), before):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("lens,budget,recent", [([40000, 39999], 20000, 100),
                                                ([70001], 1000, 999),
                                                ([70001], 65537, 0)])
def test_heavy_keys_of_long_caches(lens, budget, recent):
    _, _, w, tables = _pages([1], 2, 64)
    pages = -(-max(lens) // PAGE)
    w = torch.rand(pages * len(lens), 2, PAGE)
    w[::3] = 0.5                           # ties among them
    tables = torch.randperm(len(w)).int().view(len(lens), pages)
    kept, n = ops.heavy_keys(w.cuda(), tables.cuda(),
                             torch.tensor(lens, dtype=torch.int32).cuda(), budget,
                             recent)
    assert torch.equal(kept.cpu(), _heavy(w, tables, lens, budget, recent))
    assert n.tolist() == [budget] * len(lens)


def _close(k, v, w, tables, kept, lens):
    for b, n in enumerate(lens):
        for x in (k, v, w):
            rows = [x[tables[b, j // PAGE], :, j % PAGE].clone()
                    for j in kept[b, :n].tolist()]
            for i, row in enumerate(rows):
                x[tables[b, i // PAGE], :, i % PAGE] = row


@pytest.mark.parametrize("dev", CPU_OR_GPU)
@pytest.mark.parametrize("KH,D,fp8", [(1, 32, False), (2, 64, False), (3, 64, True),
                                      (2, 128, False), (1, 256, True),
                                      (2, 256, False)])
def test_compact_pages(dev, KH, D, fp8):
    """Bit for bit, the places behind the kept ones among them."""
    lens = [500, 0, 1, 17, 300, 64]
    k, v, w, tables = _pages(lens, KH, D, fp8, width=33)
    kept = torch.full((6, 260), -1, dtype=torch.int32)
    g = torch.Generator().manual_seed(5)
    stay = [260, 0, 1, 9, 259, 64]
    for b, (n, L) in enumerate(zip(stay, lens)):
        kept[b, :n] = torch.randperm(L, generator=g)[:n].sort().values.int()
    kept[4, :259] = torch.arange(41, 300).int()         # all move by 41
    got = [t.to(dev) for t in (k, v, w)]
    ops.compact_pages(*got, tables.to(dev), kept.to(dev),
                      torch.tensor(stay, dtype=torch.int32, device=dev))
    _close(k, v, w, tables, kept, stay)
    for a, b in zip(got, (k, v, w)):
        assert torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("dev", CPU_OR_GPU)
def test_compact_pages_of_no_page(dev):
    """Places and pages that are none are left out: nothing is read or written
    for them."""
    k, v, w, tables = _pages([100], 1, 64)
    kept = torch.tensor([[-1, 2, 7, 5000, 60, 99]], dtype=torch.int32)
    tables[0, 3] = 1 << 20                               # of key 60
    tables[0, 6] = -5                                    # of key 99
    got = [t.to(dev) for t in (k, v, w)]
    ops.compact_pages(*got, tables.to(dev), kept.to(dev),
                      torch.tensor([6], dtype=torch.int32, device=dev))
    for x in (k, v, w):
        rows = x[tables[0, 0], :, [2, 7]].clone()
        x[tables[0, 0], :, [1, 2]] = rows
    for a, b in zip(got, (k, v, w)):
        assert torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("dev", CPU_OR_GPU)
def test_refusals(dev):
    k, v, w, t = (x.to(dev) for x in _pages([40], 2, 64))
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16, device=dev)
    n = torch.tensor([40], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 1], dtype=torch.int32, device=dev)
    kept = torch.zeros(1, 8, dtype=torch.int32, device=dev)

    def refused(f, *args):
        with pytest.raises((ValueError, RuntimeError)):
            f(*args)

    token, chunk = ops.paged_attention_weights, ops.context_attention_weights
    for bad in (w[:1], w.double(), w[:, :1], w.transpose(0, 1), w[:, :, :8]):
        refused(token, q, k, v, bad, t, n, 1.0)
        refused(chunk, q, k, v, bad, cu, n, t, 1.0)
        refused(ops.compact_pages, k, v, bad, t, kept, n)
    for bad in (q[:, :3], q[..., :32], q[0], torch.zeros(2, 4, 64).to(q)):
        refused(token, bad, k, v, w, t, n, 1.0)
    refused(chunk, q[:, :3], k, v, w, cu, n, t, 1.0)
    refused(token, q, k, v[:, :, :, :32], w, t, n, 1.0)
    refused(token, q, k, v.view(torch.uint8), w, t, n, 1.0)
    refused(token, q, k, v, w, t.long(), n, 1.0)
    refused(token, q, k, v, w, t, n.long(), 1.0)
    refused(token, q, k, v, w, t, n[:0], 1.0)
    refused(chunk, q, k, v, w, cu[:1], n, t, 1.0)
    refused(chunk, q, k, v, w, cu.long(), n, t, 1.0)
    for budget, recent in ((0, 0), (8, 9), (8, -1), (-4, -4)):
        refused(ops.heavy_keys, w, t, n, budget, recent)
    refused(ops.heavy_keys, w, t, n[:0], 8, 0)
    refused(ops.compact_pages, k, v, w, t, kept.long(), n)
    refused(ops.compact_pages, k, v, w, t, kept[:0], n)
    refused(ops.compact_pages, k.transpose(2, 3), v, w, t, kept, n)
    if dev == "cuda":
        refused(token, q.float(), k, v, w, t, n, 1.0)
        refused(token, q, k, v, w, t.cpu(), n, 1.0)
        refused(token, q, k, v, w, t, n, 1.0, torch.zeros(3, device=dev))
        refused(ops.heavy_keys, w, t, n.cpu(), 8, 0)
        refused(ops.compact_pages, k, k, w, t, kept, n)


@pytest.mark.gpu
def test_pages_far_behind():
    """Pages whose rows lie beyond 2^31 elements of the caches."""
    KH, D, far = 8, 128, 139000
    k, v = (torch.empty(far + 40, KH, PAGE, D, dtype=torch.bfloat16,
                        device="cuda") for _ in range(2))
    w = torch.empty(far + 40, KH, PAGE, device="cuda")
    small = _pages([300, 80], KH, D, width=19)
    pages = torch.arange(far, far + small[0].size(0))
    for x, y in zip((k, v, w), small):
        x[pages.cuda()] = y.cuda()
    tables = (small[3].long() + far).int().cuda()
    lens = torch.tensor([300, 80], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 16, D).bfloat16().cuda()
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    want, near, want_w, off = _oracle(q, *small[:3], [1, 1], [300, 80], small[3],
                                      D ** -0.5, None)
    for op in ("paged", "context"):
        w[pages.cuda()] = small[2].cuda()
        out = ops.paged_attention_weights(q, k, v, w, tables, lens, D ** -0.5) \
            if op == "paged" else ops.context_attention_weights(
                q, k, v, w, cu, lens, tables, D ** -0.5)
        err = (out.cpu().double() - want).abs()
        assert (err <= 2.0 ** -8 * (want.abs() + near) + 2.0 ** -20).all()
        got = w[pages.cuda()].cpu().double()
        assert ((got - want_w).abs() <= off)[off > 0].all()
    kept, n = ops.heavy_keys(w, tables, lens, 64, 16)
    assert torch.equal(kept.cpu(), _heavy(got.float(), small[3], [300, 80], 64, 16))
    ops.compact_pages(k, v, w, tables, kept, n)
    ref = [t.clone() for t in small[:2]] + [got.float()]
    _close(*ref, small[3], kept.cpu(), n.tolist())
    for x, y in zip((k, v, w), ref):
        x = x[pages.cuda()].cpu()
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def _append(k, v, tables, lens, rows_k, rows_v):
    """One new key a sequence, behind its last."""
    b = torch.arange(len(lens), device=k.device)
    page = tables[b, lens.long() // PAGE].long()
    k[page, :, lens.long() % PAGE] = rows_k
    v[page, :, lens.long() % PAGE] = rows_v


@pytest.mark.parametrize("dev", CPU_OR_GPU)
def test_a_cache_kept_to_its_budget(dev):
    """Two prompts in chunks, then tokens, their caches cut every eight of them:
    every output and all weights against 64 bits over the keys that are left."""
    QH, KH, D, budget, recent = 4, 2, 64, 48, 16
    scale = D ** -0.5
    g = torch.Generator().manual_seed(2)
    tables = torch.randperm(16, generator=g).int().view(2, 8)
    # weights of rows that no one has written: a new key's must not count
    k, v = (torch.full((16, KH, PAGE, D), math.nan).bfloat16() for _ in range(2))
    w = torch.full((16, KH, PAGE), math.nan)
    k, v, w, tables = (t.to(dev) for t in (k, v, w, tables))
    lens = torch.zeros(2, dtype=torch.int32, device=dev)

    def step(new):
        """`new` rows of each sequence through the operator and the oracle."""
        nonlocal lens
        T = sum(new)
        q, rk, rv = (torch.randn(T, n, D, generator=g).bfloat16().to(dev)
                     for n in (QH, KH, KH))
        at = 0
        for b, n in enumerate(new):
            for i in range(n):
                _append(k, v, tables[b:b + 1], lens[b:b + 1] + i, rk[at:at + 1],
                        rv[at:at + 1])
                at += 1
        lens = lens + torch.tensor(new, dtype=torch.int32, device=dev)
        want, near, want_w, off = _oracle(q, k, v, w, new, lens.tolist(),
                                          tables, scale, None)
        if max(new) == 1:
            out = ops.paged_attention_weights(q, k, v, w, tables, lens, scale)
        else:
            cu = torch.tensor([0] + new).cumsum(0).int().to(dev)
            out = ops.context_attention_weights(q, k, v, w, cu, lens, tables,
                                                scale)
        err = (out.cpu().double() - want).abs()
        assert (err <= 2.0 ** -8 * (want.abs() + near) + 2.0 ** -20).all()
        live = off > 0
        assert ((w.cpu().double() - want_w).abs() <= off)[live].all()

    step([40, 23])
    step([30, 9])
    for cut in range(3):
        for _ in range(8):
            step([1, 1])
        kept, n = ops.heavy_keys(w, tables, lens, budget, recent)
        want = _heavy(w.cpu(), tables.cpu(), lens.tolist(), budget, recent)
        assert torch.equal(kept.cpu(), want)
        ref = [t.cpu().clone() for t in (k, v, w)]
        _close(*ref, tables.cpu(), want, n.tolist())
        ops.compact_pages(k, v, w, tables, kept, n)
        for x, y in zip((k, v, w), ref):
            assert torch.equal(x.cpu().view(torch.uint8), y.view(torch.uint8))
        lens = n
        assert lens.tolist() == [48, min(48, 40 + 8 * cut)]


@pytest.mark.gpu
def test_replayed_from_graphs():
    """Both attentions, the choice and the closing captured, two graphs of one
    memory pool; eager work and other replays in between."""
    KH, D = 2, 128
    lens = [600, 33, 0, 2100]              # splits, and a padding row
    k, v, w, tables = (t.cuda() for t in _pages(lens, KH, D, width=160, seed=4))
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    new = [3, 33, 0, 70]
    cu = torch.tensor([0] + new).cumsum(0).int().cuda()
    tiles = ops.build_query_tiles(new, "cuda")
    q1 = torch.randn(4, 8, D).bfloat16().cuda()
    q2 = torch.randn(106, 8, D).bfloat16().cuda()

    def token(k, v, w):
        return ops.paged_attention_weights(q1, k, v, w, tables, n, 0.1)

    def cut(k, v, w):
        out = ops.context_attention_weights(q2, k, v, w, cu, n, tables, 0.1,
                                            tiles=tiles)
        kept, left = ops.heavy_keys(w, tables, n, 500, 100)
        ops.compact_pages(k, v, w, tables, kept, left)
        return out, kept, left

    eager = [t.clone() for t in (k, v, w)]
    scratch = [t.clone() for t in eager]
    token(*scratch), cut(*scratch)         # loaded before the capture
    torch.cuda.synchronize()
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        got1 = token(k, v, w)
    with torch.cuda.graph(second, pool=first.pool()):
        got2 = cut(k, v, w)
    for t, e in zip((k, v, w), eager):
        t.copy_(e)
    for _ in range(4):
        first.replay()
        want = token(*eager)
        assert torch.equal(got1, want)
        torch.cuda.synchronize()
        second.replay()
        want = cut(*eager)
        for a, b in zip(got2, want):
            assert torch.equal(a, b)
        for t, e in zip((k, v, w), eager):
            assert torch.equal(t.view(torch.uint8), e.view(torch.uint8))


@pytest.mark.gpu
def test_on_another_stream():
    KH, D, lens = 2, 64, [1500, 40]
    k, v, w, tables = (t.cuda() for t in _pages(lens, KH, D))
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    q = torch.randn(2, 8, D).bfloat16().cuda()

    def run(k, v, w):
        out = ops.paged_attention_weights(q, k, v, w, tables, n, 0.1)
        kept, left = ops.heavy_keys(w, tables, n, 300, 20)
        ops.compact_pages(k, v, w, tables, kept, left)
        return out, kept, left

    want_state = [t.clone() for t in (k, v, w)]
    want = run(*want_state)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)      # the other stream is far ahead
        got = run(k, v, w)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip([*got, k, v, w], [*want, *want_state]):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.gpu
def test_strided_arguments():
    """Tables, lengths and choices cut from larger arrays; q of odd strides."""
    KH, D, lens = 1, 64, [200, 90]
    k, v, w, tables = (t.cuda() for t in _pages(lens, KH, D))
    wide = torch.zeros(4, 30, dtype=torch.int32).cuda()
    wide[::2, 3:3 + tables.size(1)] = tables
    cut = wide[::2, 3:3 + tables.size(1)]
    n = torch.tensor([200, 7, 90, 7], dtype=torch.int32).cuda()[::2]
    x = torch.randn(2, 3 * D + 1, 2).bfloat16().cuda()
    q = x[:, 1:1 + 2 * D].transpose(1, 2).reshape(2, 2, 2 * D)[:, :, ::2]
    assert not cut.is_contiguous() and not n.is_contiguous()
    a, b = w.clone(), w.clone()
    assert torch.equal(
        ops.paged_attention_weights(q, k, v, a, cut, n, 0.1),
        ops.paged_attention_weights(q.contiguous(), k, v, b, tables,
                                    n.contiguous(), 0.1))
    assert torch.equal(a.view(torch.int32), b.view(torch.int32))
    kept, left = ops.heavy_keys(a, cut, n, 50, 5)
    want = ops.heavy_keys(b, tables, n.contiguous(), 50, 5)
    assert torch.equal(kept, want[0]) and torch.equal(left, want[1])
    other = [t.clone() for t in (k, v, b)]
    every = torch.full((2, 100), -7, dtype=torch.int32).cuda()
    every[:, ::2] = kept
    ops.compact_pages(k, v, a, cut, every[:, ::2], left)
    ops.compact_pages(*other, tables, kept, left)
    for s, t in zip((k, v, a), other):
        assert torch.equal(s.view(torch.uint8), t.view(torch.uint8))


@pytest.mark.parametrize("dev", CPU_OR_GPU)
@pytest.mark.parametrize("D,fp8", [(64, True), (128, False), (256, False)])
@pytest.mark.parametrize("width,said", [
    (None, 40),             # keys in one share
    (64, 40),               # in several
    (800, 40),              # and workgroups of 256 keys
    (2, 4000),              # a table that ends before the keys do
    (0, 40)])               # and one without pages
@pytest.mark.parametrize("sinks", [False, True])
def test_rows_that_see_no_key(dev, D, fp8, width, said, sinks):
    """More rows than keys, and rows of a sequence without any: zeros where a row
    sees nothing, the rest as ever."""
    QH, KH, new = 2, 1, [200, 9, 1]
    held = said if width is None or width > 2 else width * PAGE
    lens = [held, 0, min(held, 1)]
    k, v, w, tables = _pages(lens, KH, D, fp8, width)
    if width == 0:
        tables = tables[:, :0]
    g = torch.Generator().manual_seed(4)
    q = torch.randn(sum(new), QH, D, generator=g).bfloat16()
    scale = D ** -0.5
    sink = torch.randn(QH, generator=g) if sinks else None
    live = torch.cat([torch.arange(n) >= n - m for n, m in zip(new, lens)])
    want, near, want_w, off = _oracle(q[live], k, v, w, lens, lens, tables, scale,
                                      sink)
    q = q.to(dev)
    got, cu, lens = (t.to(dev) for t in (
        w, torch.tensor([0] + new).cumsum(0).int(),
        torch.tensor([said] + lens[1:], dtype=torch.int32)))
    k, v, tables = (t.to(dev) for t in (k, v, tables))
    if sinks:
        sink = sink.to(dev)
    # what is taken next: the output and, for several shares, theirs
    old = [torch.full(q.shape, math.nan, dtype=q.dtype, device=dev),
           torch.full((2 << 20,), math.nan, device=dev)]
    del old
    out = ops.context_attention_weights(q, k, v, got, cu, lens, tables, scale,
                                        sink)
    out, got = out.cpu().double(), got.cpu().double()
    assert (out[~live] == 0).all()
    err = (out[live] - want).abs()
    assert (err <= 2.0 ** -8 * (want.abs() + near) + 2.0 ** -20).all()
    assert ((got - want_w).abs() <= off)[off > 0].all()
    assert torch.equal(got[off == 0].float().view(torch.int32),
                       w[off == 0].view(torch.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("width", [None, 64, 300])
def test_rows_behind_the_last_sequence(width):
    """Rows of a padded step that belong to no sequence stay as they were, in one
    share of the keys and in several."""
    k, v, w, tables = (t.cuda() for t in _pages([40], 1, 128, width=width))
    q = torch.randn(20, 2, 128).bfloat16().cuda()
    cu = torch.tensor([0, 7], dtype=torch.int32).cuda()
    lens = torch.tensor([40], dtype=torch.int32).cuda()
    own = ops.context_attention_weights(q[:7], k, v, w.clone(), cu, lens, tables, 0.1)
    seq, base = ops.build_query_tiles([7], "cuda")
    out = torch.full_like(q, 7.)
    ops._K.context_attention_weights(out, q, k, v, w, seq, base, cu, lens, tables,
                                     0.1, torch.empty(0, device="cuda"))
    assert torch.equal(out[:7], own) and (out[7:] == 7).all()


@pytest.mark.parametrize("dev", CPU_OR_GPU)
@pytest.mark.parametrize("layout", [(8, 2, 64), (7, 1, 128), (4, 2, 256)])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("width", [None, 240, 3200])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_scores_that_are_no_number(dev, layout, fp8, width, bad):
    """A row and head with such a score comes out as no number, and so do the entries
    of the keys that it sees; all others are as ever. The first sequence has it in a
    query, the last in a key whose share of the keys has scores far below the row's
    largest."""
    QH, KH, D = layout
    G, scale = QH // KH, D ** -0.5
    new, lens = [6, 3, 2], [66, 10, 952]
    k, v, w, tables = _pages(lens, KH, D, fp8, width)
    g = torch.Generator().manual_seed(8)
    q = torch.randn(sum(new), QH, D, generator=g).bfloat16()

    def put(cache, j, x):               # into the last sequence's key j, kv head 0
        x = torch.tensor(x)
        cache[tables[2, j // PAGE], 0, j % PAGE, 5] = \
            x.to(torch.float8_e4m3fn).view(torch.uint8) if fp8 else x.bfloat16()

    q[9:, :, 5] = 64.
    put(k, 900, 448.)
    # in 64 bits without what is no number
    put(k, 3, 0.)
    want, near, want_w, off = _oracle(q, k, v, w, new, lens, tables, scale, None)
    put(k, 3, math.nan if fp8 else bad)         # e4m3 has no infinity
    q[1, 0, 3] = math.nan
    live = torch.ones(sum(new), QH, dtype=torch.bool)
    live[1, 0] = False
    live[9:, :G] = False

    def seen(*n):                       # kv head 0's first keys of a sequence
        keys = torch.zeros(w.shape, dtype=torch.bool)
        for b, m in zip((0, 2), n):
            j = torch.arange(m)
            keys[tables[b, j // PAGE].long(), 0, j % PAGE] = True
        return keys

    k, v, q, tables = (t.to(dev) for t in (k, v, q, tables))
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    cu = torch.tensor([0] + new).cumsum(0).int().to(dev)
    got = w.to(dev)
    out = ops.context_attention_weights(q, k, v, got, cu, n, tables, scale)
    out, got = out.cpu().double(), got.cpu().double()
    assert out[~live].isnan().all()
    err = (out - want).abs()
    assert (err <= 2.0 ** -8 * (want.abs() + near) + 2.0 ** -20)[live].all()
    keys = seen(62, 952)
    assert got[keys].isnan().all()
    other = (off > 0) & ~keys
    assert ((got - want_w).abs() <= off)[other].all()
    # single tokens: these rows of the three sequences
    rows = [1, 6, 10]
    got = w.to(dev)
    out = ops.paged_attention_weights(q[rows], k, v, got, tables, n, scale)
    out, got = out.cpu(), got.cpu()
    assert torch.equal(out.isnan(), ~live[rows, :, None].expand_as(out))
    keys = seen(66, 952)
    assert got[keys].isnan().all()
    assert not got[(off > 0) & ~keys].isnan().any()


# workgroups of 256 keys (128 with 256 dims) from 96 on: whole prompts, whose
# workgroups begin inside the chunk, at rows that are no multiple of a tile's positions
@pytest.mark.gpu
@pytest.mark.parametrize("G", [1, 4, 7])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("shared", [True, False])
def test_whole_prompts(G, D, fp8, shared):
    """shared: one kv head and a wide table, the first pass in shares of the keys."""
    if shared:
        _run("cuda", (G, 1, D), [701, 333], [0, 37], fp8=fp8, sinks=fp8, width=800,
             seed=G)
    else:
        _run("cuda", (8 * G, 8, D), [389, 97, 300, 520, 1], [0, 0, 25, 3, 600],
             fp8=fp8, sinks=not fp8, seed=G)


@pytest.mark.gpu
def test_many_tiles_of_rows():
    """Every place of the three buffers of rows, many times over."""
    _run("cuda", (8, 1, 128), [2100], [130], width=3200, seed=5)
    _run("cuda", (5, 1, 64), [1500, 700], [0, 0], fp8=True, width=1700, seed=6)


# tables of 2049 to 8192 keys, whose totals the choosing launch makes by itself, and of
# up to 32768, which stay in registers; as many keys to choose among as whole rows of
# 1024 threads, one less and one more
@pytest.mark.gpu
@pytest.mark.parametrize("lens,budget,recent", [
    ([2049, 1500, 2048], 1024, 1),
    ([4352, 4225, 4096], 4096, 512),
    ([8192, 8191, 5121], 5000, 1000),
    ([8193, 8192, 9], 100, 0),
    ([5120 + 64, 5119 + 64, 5121 + 64], 2000, 64),
    ([20000, 16384 + 300, 12289 + 300], 9000, 300),
    ([32768, 32767, 28673], 16384, 1024),
])
@pytest.mark.parametrize("kind", ["spread", "ties", "equal"])
def test_heavy_keys_of_ordinary_caches(lens, budget, recent, kind):
    pages = -(-max(lens) // PAGE)
    g = torch.Generator().manual_seed(11)
    w = torch.rand(pages * len(lens), 8, PAGE, generator=g) ** 4 * 10
    if kind == "ties":
        w = (w * 2).floor()
        w[::3] = 0.5
    elif kind == "equal":
        w.fill_(0.25)
    tables = torch.randperm(len(w), generator=g).int().view(len(lens), pages)
    kept, n = ops.heavy_keys(w.cuda(), tables.cuda(),
                             torch.tensor(lens, dtype=torch.int32).cuda(), budget,
                             recent)
    assert torch.equal(kept.cpu(), _heavy(w, tables, lens, budget, recent))
    assert n.tolist() == [min(L, budget) for L in lens]


# rows of 64, 128, 256 and 512 bytes, moved whole where there are workgroups enough
@pytest.mark.gpu
@pytest.mark.parametrize("D,fp8", [(64, True), (64, False), (128, True),
                                   (128, False), (256, True), (256, False)])
def test_compact_pages_of_a_batch(D, fp8):
    B, KH = 64, 8
    lens = [300 - 3 * b for b in range(B)]
    k, v, w, tables = _pages(lens, KH, D, fp8)
    stay = [min(n, 150 + b) for b, n in enumerate(lens)]
    kept = torch.full((B, 220), -1, dtype=torch.int32)
    g = torch.Generator().manual_seed(6)
    for b, (n, L) in enumerate(zip(stay, lens)):
        kept[b, :n] = torch.randperm(L, generator=g)[:n].sort().values.int()
    got = [t.cuda() for t in (k, v, w)]
    ops.compact_pages(*got, tables.cuda(), kept.cuda(),
                      torch.tensor(stay, dtype=torch.int32).cuda())
    _close(k, v, w, tables, kept, stay)
    for a, b in zip(got, (k, v, w)):
        assert torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("layout", [(8, 2, 64), (32, 8, 128), (8, 4, 256)])
def test_outputs_of_the_plain_operators(layout, fp8):
    """Keeping weights changes no output where the keys are not shared out
    otherwise: the same bits as context_attention and paged_attention."""
    QH, KH, D = layout
    new, lens = [300, 1, 200, 77] * 24, [310, 40, 200, 700] * 24
    k, v, w, tables = (t.cuda() for t in _pages(lens, KH, D, fp8))
    q = torch.randn(sum(new), QH, D).bfloat16().cuda()
    cu = torch.tensor([0] + new).cumsum(0).int().cuda()
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    scale = D ** -0.5
    got = ops.context_attention_weights(q, k, v, w.clone(), cu, n, tables, scale)
    assert torch.equal(got, ops.context_attention(q, k, v, cu, n, tables, scale))
    x = q[:len(lens)]
    got = ops.paged_attention_weights(x, k, v, w.clone(), tables, n, scale)
    assert torch.equal(got, ops.paged_attention(x, k, v, tables, n, scale))
