"""Serving with caches kept to a budget (EngineConfig.kv_budget): the engine
against a replay of the same model whose attention keeps plain lists of keys per
sequence and layer, and cuts them by the rule, key by key."""
import dataclasses

import pytest
import torch

from kaito_amd import ops
from kaito_amd.engine import EngineConfig, LLMEngine, SamplingParams
from kaito_amd.models import get_model_config
from kaito_amd.models.llama import AttnMetadata, LlamaAttention
from kaito_amd.parallel.state import init_parallel

SP = SamplingParams(max_tokens=60, ignore_eos=True)


@pytest.fixture(autouse=True)
def _parallel():
    init_parallel(1)


def _cfg(**kw):
    base = dict(model=get_model_config("tiny-llama-test"), device="cpu",
                max_num_seqs=8, num_gpu_blocks=64, enforce_eager=True,
                max_model_len=256, kv_budget=32, kv_budget_recent=8,
                kv_budget_slack=8)
    base.update(kw)
    return EngineConfig(**base)


class _Lists:
    """One sequence's keys, values and received weights, per layer."""

    def __init__(self, cfg):
        self.cfg, self.layers = cfg, {}

    def attend(self, attn, qkv, positions, kv_cache, meta, cos_sin, *_):
        q, k, v = qkv.split([attn.q_size, attn.kv_size, attn.kv_size], dim=-1)
        q, k = ops.rotary_embedding(positions, q.clone(), k.clone(),
                                    attn.head_dim, cos_sin)
        D, T = attn.head_dim, qkv.size(0)
        k, v = (t.reshape(T, attn.num_kv_heads, D) for t in (k, v))
        if attn.layer_idx in self.layers:
            K, V, W = self.layers[attn.layer_idx]
            k, v = torch.cat([K, k]), torch.cat([V, v])
            W = torch.cat([W, W.new_zeros(T, W.size(1))])
        else:
            W = torch.zeros(T, attn.num_kv_heads)
        L, G = k.size(0), attn.num_heads // attn.num_kv_heads
        x = q.reshape(T, attn.num_heads, D).float().transpose(0, 1)
        kx, vx = (t.float().repeat_interleave(G, 1).transpose(0, 1)
                  for t in (k, v))
        s = x @ kx.transpose(1, 2) * attn.scale
        later = torch.arange(L) > torch.arange(L - T, L)[:, None]
        p = s.masked_fill(later, float("-inf")).softmax(-1)
        W = W + p.unflatten(0, (-1, G)).sum((1, 2)).T
        self.layers[attn.layer_idx] = (k, v, W)
        out = (p @ vx).transpose(0, 1).to(qkv.dtype)
        return attn.o_proj(out.reshape(T, -1))

    def cut(self):
        c = self.cfg
        for i, (k, v, w) in self.layers.items():
            L = k.size(0)
            if L <= c.kv_budget + c.kv_budget_slack:
                continue
            total = w.double().sum(1).float()[:L - c.kv_budget_recent].tolist()
            order = sorted(range(len(total)), key=lambda j: (-total[j], j))
            stay = sorted(order[:c.kv_budget - c.kv_budget_recent]) \
                + list(range(L - c.kv_budget_recent, L))
            self.layers[i] = (k[stay], v[stay], w[stay])


def _replayed(eng, prompt, n, monkeypatch, chunk=10 ** 9):
    """n greedy tokens of a sequence by itself."""
    lists, model = _Lists(eng.cfg), eng.runner.model
    with monkeypatch.context() as m:
        m.setattr(LlamaAttention, "attend",
                  lambda attn, *a: lists.attend(attn, *a))
        toks, at = list(prompt), 0
        while len(toks) < len(prompt) + n:
            end = min(at + chunk, len(toks))
            ids = torch.tensor(toks[at:end])
            T = end - at
            meta = AttnMetadata(
                is_prefill=True, slot_mapping=torch.full((T,), -1),
                cu_seqlens=torch.tensor([0, T], dtype=torch.int32),
                max_seqlen=T)
            hidden = model(ids, torch.arange(at, end),
                           [None] * model.num_local_layers, meta)
            at = end
            if at == len(toks):
                toks.append(int(model.compute_logits(hidden[-1:]).argmax(-1)))
            lists.cut()
    return toks[len(prompt):]


def test_a_budget_that_holds_everything_changes_nothing():
    prompts = [list(range(5, 45)), [3, 5, 7]]
    want = LLMEngine(_cfg(kv_budget=None)).generate(prompts, SP)
    got = LLMEngine(_cfg(kv_budget=200)).generate(prompts, SP)
    for a, b in zip(want, got):
        assert a.output_token_ids == b.output_token_ids and b.evicted == 0


@pytest.mark.parametrize("prompt", [[3, 14, 15], list(range(7, 39)),
                                    list(range(10, 110))])
def test_cut_caches_match_plain_lists(prompt, monkeypatch):
    eng = LLMEngine(_cfg())
    out = eng.generate([prompt], SP)[0]
    assert out.evicted > 0
    assert out.output_token_ids == _replayed(eng, prompt, 60, monkeypatch)
    assert eng.pool.num_free == eng.pool.num_blocks


def test_batches_chunks_and_joins(monkeypatch):
    """Sequences that are cut at different steps, a long prompt in chunks
    (cut between them too) and one that joins later."""
    eng = LLMEngine(_cfg(max_num_batched_tokens=24))
    prompts = [list(range(10, 100)), list(range(30, 50)), [9, 8, 7, 6]]
    ids = [eng.add_request(p, SP) for p in prompts[:2]]
    for _ in range(9):
        eng.step()
    ids.append(eng.add_request(prompts[2], SP))
    most = 0
    while eng.has_unfinished():
        eng.step()
        most = max([most] + [len(s.block_table) for s in eng.scheduler.running])
    # 32 + 8 keys and the one that comes
    assert most <= -(-42 // 16)
    assert eng.seqs[ids[0]].output_token_ids == _replayed(
        eng, prompts[0], 60, monkeypatch, chunk=24)
    for i in (1, 2):
        assert eng.seqs[ids[i]].output_token_ids == _replayed(
            eng, prompts[i], 60, monkeypatch)
    assert eng.pool.num_free == eng.pool.num_blocks


def test_preempted_sequences_begin_anew():
    """A pool that runs dry: victims lose their cuts with their caches, and
    every sequence ends with all of its tokens and the pages given back."""
    eng = LLMEngine(_cfg(num_gpu_blocks=7, max_num_seqs=4, max_model_len=96))
    ids = [eng.add_request(list(range(a, a + 14)), SP) for a in (10, 30, 50)]
    for _ in range(500):
        if not eng.has_unfinished():
            break
        eng.step()
    assert any(eng.seqs[i].epoch > 0 for i in ids)
    assert all(len(eng.seqs[i].output_token_ids) == 60 for i in ids)
    assert eng.pool.num_free == eng.pool.num_blocks


@pytest.mark.parametrize("kw", [
    dict(kv_budget=0), dict(kv_budget_recent=33), dict(kv_budget_slack=-1),
    dict(kv_budget_recent=-1), dict(enable_mixed_batch=True),
    dict(model=get_model_config("tiny-deepseek-test")),
    dict(model=dataclasses.replace(get_model_config("tiny-llama-test"),
                                   sliding_window=32,
                                   sliding_window_pattern="all"))])
def test_refused(kw):
    with pytest.raises(ValueError):
        LLMEngine(_cfg(**kw))


def test_transferred_keys_have_received_nothing():
    from kaito_amd.engine.kv_transfer import extract_kv, inject_kv
    a, b = LLMEngine(_cfg()), LLMEngine(_cfg())
    for w in b.runner.key_weights:
        w.fill_(7.)
    pages = b.pool.allocate(2)
    layers = extract_kv(a.runner.kv_caches, a.pool.allocate(2), 20, 16)
    inject_kv(b.runner.kv_caches, pages, layers, 16, b.runner.key_weights)
    for w in b.runner.key_weights:
        assert (w[pages] == 0).all() and (w.sum() > 0)


def test_what_a_budget_turns_off():
    eng = LLMEngine(_cfg(enable_prefix_caching=True, kv_offload=True))
    assert not hasattr(eng.pool, "match_prefix") and eng.kv_offload is None


@pytest.mark.gpu
@pytest.mark.parametrize("eager", [True, False])
@pytest.mark.parametrize("dtype", ["auto", "fp8"])
def test_serving_on_the_gpu(eager, dtype):
    """With graphs and without: the same tokens, and those of an engine
    without a budget while nothing is cut."""
    kw = dict(device="cuda", enforce_eager=eager, kv_cache_dtype=dtype,
              graph_batch_sizes=(1, 2, 4), max_num_seqs=4)
    prompts = [list(range(10, 100)), [3, 5, 7, 11]]
    eng = LLMEngine(_cfg(**kw)).capture_graphs()
    got = eng.generate(prompts, SP)
    assert all(s.evicted > 0 for s in got)
    assert eng.pool.num_free == eng.pool.num_blocks
    again = LLMEngine(_cfg(**dict(kw, enforce_eager=True))).generate(prompts, SP)
    for a, b in zip(got, again):
        assert a.output_token_ids == b.output_token_ids
    short = SamplingParams(max_tokens=20, ignore_eos=True)
    wide = LLMEngine(_cfg(**dict(kw, kv_budget=200))).capture_graphs()
    for s in wide.generate(prompts, short):
        assert s.evicted == 0 and len(s.output_token_ids) == 20


def test_transferred_sequences_are_cut_before_they_decode():
    """100 keys that come from an engine without a budget: none has received
    anything, so that the newest and the first ones stay."""
    from kaito_amd.engine.kv_transfer import extract_kv, inject_kv
    from kaito_amd.engine.sequence import SeqStatus
    prompt, sp = list(range(10, 110)), SamplingParams(max_tokens=30,
                                                      ignore_eos=True)
    pre, dec = LLMEngine(_cfg(kv_budget=None)), LLMEngine(_cfg())
    src = pre.seqs[pre.add_request(prompt, sp)]
    pre.step()
    layers = extract_kv(pre.runner.kv_caches, src.block_table, 100, 16)
    seq = dec.seqs[dec.add_request(prompt, sp)]
    dec.scheduler.waiting.remove(seq)
    seq.block_table = dec.pool.allocate(dec.pool.blocks_needed(102))
    inject_kv(dec.runner.kv_caches, seq.block_table, layers, 16,
              dec.runner.key_weights)
    seq.output_token_ids = list(src.output_token_ids)
    seq.sched_len, seq.status = 101, SeqStatus.RUNNING
    dec.scheduler.running.append(seq)
    while dec.has_unfinished():
        dec.step()
    assert seq.evicted > 0 and len(seq.output_token_ids) == 30
    assert dec.pool.num_free == dec.pool.num_blocks

    lists, model = _Lists(dec.cfg), dec.runner.model
    with pytest.MonkeyPatch.context() as m:
        m.setattr(LlamaAttention, "attend",
                  lambda attn, *a: lists.attend(attn, *a))
        toks, at = list(prompt), 0
        while len(toks) < 130:
            T = len(toks) - at
            meta = AttnMetadata(
                is_prefill=True, slot_mapping=torch.full((T,), -1),
                cu_seqlens=torch.tensor([0, T], dtype=torch.int32),
                max_seqlen=T)
            hidden = model(torch.tensor(toks[at:]), torch.arange(at, len(toks)),
                           [None] * model.num_local_layers, meta)
            at = len(toks)
            toks.append(int(model.compute_logits(hidden[-1:]).argmax(-1)))
            if T == 100:
                for i, (k, v, w) in lists.layers.items():
                    lists.layers[i] = (k, v, torch.zeros_like(w))
            lists.cut()
    assert seq.output_token_ids == toks[100:]


def _drained(eng, steps=3000):
    for _ in range(steps):
        if not eng.has_unfinished():
            return True
        eng.step()
        tables = [s.block_table for s in eng.seqs.values()]
        pages = [p for t in tables for p in t]
        assert len(set(pages)) == len(pages)
        assert len(pages) + eng.pool.num_free == eng.pool.num_blocks
    return False


def test_a_preempted_sequence_comes_back(monkeypatch):
    """102 tokens in three of six pages: preempted there, all of its tokens would
    need seven. It is computed anew in chunks, cut between them, and what waits
    behind it has its turn."""
    eng = LLMEngine(_cfg(num_gpu_blocks=6, kv_budget=16, kv_budget_slack=32,
                         max_num_seqs=4))
    prompt = [(7 * i) % 90 + 5 for i in range(71)]
    long = eng.seqs[eng.add_request(prompt, SP)]
    while long.num_tokens < 102:
        eng.step()
    assert long.evicted > 0
    others = [eng.add_request([5 + i, 9, 40], SP) for i in range(2)]
    # the pool runs dry: what a younger sequence's growth does
    eng.flush()
    taken = eng.pool.allocate(eng.pool.num_free)
    for _ in range(40):
        if long.epoch:
            break
        eng.step()
    assert long.epoch > 0
    eng.pool.free(taken)
    assert _drained(eng)
    for i in (long.seq_id, *others):
        assert len(eng.seqs[i].output_token_ids) == 60
    assert eng.pool.num_free == 6


@pytest.mark.parametrize("seed", range(24))
def test_small_pools_end(seed):
    """Random budgets, slacks beyond the pool, chunks and arrivals: every request
    ends with all of its tokens."""
    import random
    rng = random.Random(seed)
    blocks = rng.randint(3, 9)
    budget = rng.randint(4, min(60, blocks * 16 - 2))
    eng = LLMEngine(_cfg(
        num_gpu_blocks=blocks, kv_budget=budget,
        kv_budget_recent=rng.randint(0, budget),
        kv_budget_slack=rng.choice([0, 8, 32, 100]), max_num_seqs=4,
        max_num_batched_tokens=rng.choice([16, 40, 8192])))
    want = {}
    for _ in range(rng.randint(2, 6)):
        n = rng.choice([1, 5, 30, 90, 150])
        most = rng.choice([1, 12, 60])
        sid = eng.add_request([rng.randint(3, 90) for _ in range(n)],
                              SamplingParams(max_tokens=most, ignore_eos=True))
        want[sid] = most
        for _ in range(rng.choice([0, 3, 20])):
            eng.step()
    assert _drained(eng)
    for sid, most in want.items():
        assert len(eng.seqs[sid].output_token_ids) == most


def test_a_prompt_takes_the_pages_of_a_budget_and_a_chunk(monkeypatch):
    """150 tokens in chunks of 24 through eight pages, the result that of a pool
    which would hold them all."""
    prompt = [(11 * i) % 90 + 4 for i in range(150)]
    small = LLMEngine(_cfg(num_gpu_blocks=8, max_num_batched_tokens=24))
    sid = small.add_request(prompt, SP)
    small.step()
    # 32 + 8 keys, 24 more and the next token
    assert len(small.seqs[sid].block_table) == -(-65 // 16)
    assert _drained(small)
    assert small.seqs[sid].output_token_ids == _replayed(
        small, prompt, 60, monkeypatch, chunk=24)


def test_a_pool_below_the_budget_is_refused():
    with pytest.raises(ValueError):
        LLMEngine(_cfg(num_gpu_blocks=2))
    LLMEngine(_cfg(num_gpu_blocks=2, max_model_len=32))      # nothing is cut


@pytest.mark.parametrize("n", [29, 30, 31])
def test_a_sequence_that_fills_a_pool_of_no_budget_is_not_cut(n):
    eng = LLMEngine(_cfg(num_gpu_blocks=2, max_model_len=32, kv_budget=40))
    out = eng.generate([list(range(5, 5 + n))], SP)[0]
    want = LLMEngine(_cfg(kv_budget=None, max_model_len=32)).generate(
        [list(range(5, 5 + n))], SP)[0]
    assert out.evicted == 0 and out.output_token_ids == want.output_token_ids
    assert eng.pool.num_free == 2


def _tp_worker(rank, world, port):
    import os
    os.environ.update({
        "MASTER_ADDR": "127.0.0.1", "MASTER_PORT": str(port),
        "WORLD_SIZE": str(world), "RANK": str(rank), "LOCAL_RANK": str(rank)})
    from kaito_amd.parallel import one_shot
    from kaito_amd.parallel import state as ps
    init_parallel(world, backend="gloo")
    try:
        eng = LLMEngine(_cfg(tensor_parallel_size=world))
        run = eng.runner
        g = torch.Generator().manual_seed(3)
        tables, lens = [[5, 9, 2, 7], [1, 0, 3]], [60, 41]
        ref = []
        for i, ((k, v), w) in enumerate(zip(run.kv_caches, run.key_weights)):
            own = w.size(1)
            # every rank draws all heads and keeps its own
            full = torch.rand(w.size(0), own * world, 16, generator=g)
            full[:, 0] *= 3             # heads that matter more than others
            w.copy_(full[:, rank * own:(rank + 1) * own])
            for x in (k, v):
                x.copy_(torch.randn(x.shape, generator=g))
            t = torch.tensor([r + [0] * (4 - len(r)) for r in tables]).int()
            kept, n = ops.heavy_keys(full, t, torch.tensor(lens).int(), 32, 8)
            want = [x.clone() for x in (k, v, w)]
            ops.compact_pages(*want, t, kept, n)
            ref.append(want)
        run.cut_caches(tables, lens, 32, 8)
        for (k, v), w, want in zip(run.kv_caches, run.key_weights, ref):
            for x, y in zip((k, v, w), want):
                assert torch.equal(x, y), "other keys than all heads' weights"
    finally:
        one_shot.deactivate()
        ps.destroy()


@pytest.mark.parametrize("world", [2])
def test_ranks_keep_the_same_keys(world):
    """Tensor-parallel ranks cut to the keys that all of their heads together
    gave the most weight."""
    import torch.multiprocessing as mp
    mp.start_processes(_tp_worker, args=(world, 29683), nprocs=world, join=True,
                       start_method="spawn")


def test_explicit_steps_are_cut(monkeypatch):
    """Two requests in portions that the caller composes, cut between them: the
    logits of plain lists, and no more pages than a budget, its slack and a
    portion need."""
    eng = LLMEngine(_cfg())
    toks = [[(7 * i) % 90 + 4 for i in range(140)],
            [(5 * i) % 80 + 9 for i in range(70)]]
    sizes = [[30, 1, 1, 40, 9, 1, 50, 1, 1, 6], [1, 1, 20, 1, 30, 1, 1, 1, 1, 13]]
    got = [[], []]
    for a, b in zip(*sizes):
        for i, n in enumerate((a, b)):
            at = len(eng.seqs[i].prompt_token_ids) if i in eng.seqs else 0
            eng.extend_request(i, toks[i][at:at + n])
        out = eng.step_explicit([(0, a), (1, b)], [(0, a - 1), (1, b - 1)])
        for i in (0, 1):
            got[i].append(out[i])
            seq = eng.seqs[i]
            assert seq.prefilled_len - seq.evicted <= 40
            assert len(seq.block_table) <= -(-(41 + 50) // 16)
    model = eng.runner.model
    for i in (0, 1):
        assert eng.seqs[i].evicted > 0
        lists, at = _Lists(eng.cfg), 0
        for n, row in zip(sizes[i], got[i]):
            with monkeypatch.context() as m:
                m.setattr(LlamaAttention, "attend",
                          lambda attn, *a: lists.attend(attn, *a))
                meta = AttnMetadata(
                    is_prefill=True, slot_mapping=torch.full((n,), -1),
                    cu_seqlens=torch.tensor([0, n], dtype=torch.int32),
                    max_seqlen=n)
                hidden = model(torch.tensor(toks[i][at:at + n]),
                               torch.arange(at, at + n),
                               [None] * model.num_local_layers, meta)
            at += n
            want = model.compute_logits(hidden[-1:]).float()[0]
            # bf16 hidden states of other batch sizes round otherwise here and there
            assert torch.allclose(row, want, atol=0.05, rtol=0.05)
            lists.cut()
    for i in (0, 1):
        eng.release(i)
    assert eng.pool.num_free == eng.pool.num_blocks


@pytest.mark.gpu
def test_a_cut_does_not_wait_for_the_stream():
    """A cut and the decode step that is built anew behind it, whose tokens are
    still under way, are issued while the stream is busy."""
    eng = LLMEngine(_cfg(device="cuda"))
    seqs = [eng.seqs[eng.add_request(list(range(a, a + 39)), SP)]
            for a in (10, 30)]
    for _ in range(2):
        eng.step()
    run, pend = eng.runner, eng._pending
    assert pend is not None and not seqs[0].evicted

    def launch():
        run.cut_caches([s.block_table for s in seqs], [40, 40], 32, 8)
        run.execute_decode(seqs, pend.tokens, (pend.tokens, pend.index))

    launch()                            # what the first launch loads
    torch.cuda.synchronize()
    done = torch.cuda.Event()
    torch.cuda._sleep(2_000_000_000)
    done.record()
    launch()
    assert not done.query()
    torch.cuda.synchronize()


def test_the_pool_leaves_room_for_scores(monkeypatch):
    """Pages take what is left beside the scores of the widest decode step."""
    eng = LLMEngine(_cfg(max_num_seqs=64, max_model_len=4096, kv_budget=1000))
    run, m = eng.runner, eng.cfg.model
    eng.cfg.num_gpu_blocks, run.is_gpu = None, True
    mem = 30 << 20
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda *_: (mem, mem))
    n = run.profile_and_allocate_kv()
    page = m.num_layers * m.num_kv_heads * 16 * (2 * 2 * m.head_dim + 4)
    scores = 64 * m.num_heads * (1008 + 32) * 4
    room = int(mem * eng.cfg.gpu_memory_utilization) - scores
    assert 16 < n < 64 * 256 and room - 2 * page < n * page <= room


def test_cut_sequences_are_not_extracted():
    from kaito_amd.engine.kv_transfer import extract_kv
    eng = LLMEngine(_cfg(kv_budget_slack=16))
    seq = eng.seqs[eng.add_request(list(range(5, 54)), SP)]     # 49 keys
    eng.step()
    assert seq.evicted > 0
    with pytest.raises(ValueError):
        extract_kv(eng.runner.kv_caches, seq.block_table, 49, 16)


@pytest.mark.gpu
@pytest.mark.parametrize("eager", [True, False])
@pytest.mark.parametrize("dtype", ["auto", "fp8"])
def test_a_budget_that_holds_everything_on_the_gpu(eager, dtype):
    """The tokens of an engine without a budget, prompts in one chunk and in
    several. With 8-bit pages in several only: a whole prompt without a budget
    attends to its keys ahead of their rounding, with one to what the pages hold."""
    prompts = [list(range(10, 100)), [3, 5, 7, 11], list(range(40, 71))]
    sp = SamplingParams(max_tokens=40, ignore_eos=True)
    for chunk in (8192, 32) if dtype == "auto" else (32,):
        kw = dict(device="cuda", enforce_eager=eager, kv_cache_dtype=dtype,
                  graph_batch_sizes=(1, 2, 4), max_num_seqs=4,
                  max_num_batched_tokens=chunk)
        want = LLMEngine(_cfg(**dict(kw, kv_budget=None))).capture_graphs()
        got = LLMEngine(_cfg(**dict(kw, kv_budget=200))).capture_graphs()
        for a, b in zip(want.generate(prompts, sp), got.generate(prompts, sp)):
            assert a.output_token_ids == b.output_token_ids and b.evicted == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["auto", "fp8"])
def test_every_call_of_a_served_batch(dtype, monkeypatch):
    """Every attention, choice and closing that the engine asks for, cuts at
    unlike steps among them, against 64 bits over what the pages held; and every
    sequence's tables and lengths against its positions and its cuts."""
    import test_key_weights as kw
    eng = LLMEngine(_cfg(device="cuda", kv_cache_dtype=dtype, max_num_seqs=4,
                         max_num_batched_tokens=48))
    calls = dict.fromkeys(("chunk", "token", "choose", "close"), 0)
    real = {n: getattr(ops, n) for n in (
        "context_attention_weights", "paged_attention_weights", "heavy_keys",
        "compact_pages")}

    def check(out, q, k, v, w, before, new, lens, tables, scale, sinks):
        want, near, want_w, off = kw._oracle(
            q, k, v, before, new, lens, tables,
            scale, None if sinks is None else sinks.cpu())
        err = (out.cpu().double() - want).abs()
        assert (err <= 2.0 ** -8 * (want.abs() + near) + 2.0 ** -20).all()
        live = off > 0
        now = w.cpu()
        assert ((now.double() - want_w).abs() <= off)[live].all()
        assert torch.equal(now[~live], before[~live])

    def chunk(q, k, v, w, cu, lens, tables, scale, sinks=None, tiles=None):
        calls["chunk"] += 1
        before = w.cpu()
        out = real["context_attention_weights"](q, k, v, w, cu, lens, tables,
                                                scale, sinks, tiles)
        check(out, q, k, v, w, before, (cu[1:] - cu[:-1]).tolist(), lens.tolist(),
              tables, scale, sinks)
        return out

    def token(q, k, v, w, tables, lens, scale, sinks=None):
        calls["token"] += 1
        before = w.cpu()
        out = real["paged_attention_weights"](q, k, v, w, tables, lens, scale, sinks)
        seqs = eng.scheduler.running[:len(q)]
        assert lens.tolist() == [s.sched_tokens - s.evicted for s in seqs]
        for s, row in zip(seqs, tables.tolist()):
            assert row[:len(s.block_table)] == s.block_table
        check(out, q, k, v, w, before, [1] * len(q), lens.tolist(), tables, scale,
              sinks)
        return out

    def choose(w, tables, lens, budget, recent):
        calls["choose"] += 1
        kept, n = real["heavy_keys"](w, tables, lens, budget, recent)
        assert torch.equal(kept.cpu(), kw._heavy(w.cpu(), tables.cpu(),
                                                 lens.tolist(), budget, recent))
        return kept, n

    def close(k, v, w, tables, kept, n):
        calls["close"] += 1
        ref = [t.cpu() for t in (k, v, w)]
        real["compact_pages"](k, v, w, tables, kept, n)
        kw._close(*ref, tables.cpu(), kept.cpu(), n.tolist())
        for a, b in zip((k, v, w), ref):
            assert torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8))

    for name, f in zip(real, (chunk, token, choose, close)):
        monkeypatch.setattr(ops, name, f)
    ids = [eng.add_request(list(range(a, a + n)), SP)
           for a, n in ((10, 90), (30, 20), (50, 35))]
    while eng.has_unfinished():
        eng.step()
    layers = eng.cfg.model.num_layers
    assert all(eng.seqs[i].evicted > 0 for i in ids)
    # the three are cut at different steps, and the long prompt between its chunks
    assert calls["choose"] == calls["close"] >= 8 * layers
    assert calls["chunk"] >= 3 * layers and calls["token"] >= 59 * layers
    assert eng.pool.num_free == eng.pool.num_blocks
