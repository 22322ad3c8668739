"""Beam search through the models' caches: every kind of cache against a search that computes all sequences anew with the training model, the
cache's lines and pages, and the runner with its graphs."""
import dataclasses
import importlib
import math
import weakref

import pytest
import torch

from neuronx_distributed_llama3_2_b200.inference import BeamLines, InferenceConfig, InferenceRunner, KVCache, LlamaInferenceModel
from neuronx_distributed_llama3_2_b200.models import LlamaForCausalLM, tiny_llama
from conftest import run_distributed
from test_beam_search import DEVICES, _Request
import test_beam_search as units

INF = math.inf


def _models(monkeypatch, **kw):
    torch.manual_seed(0)
    cfg = tiny_llama(sequence_parallel_enabled=False)
    train = LlamaForCausalLM(cfg)
    with torch.no_grad():          # peaked enough that beams differ, with an end that is met now and then
        train.lm_head.weight.mul_(6.0)
    inf = LlamaInferenceModel(tiny_llama(sequence_parallel_enabled=False), InferenceConfig(max_context_length=32, seq_len=64, page_size=8, **kw))
    inf.load_state_dict(train.state_dict())
    return cfg, train, inf


def _searched(logits_of, prompt, W, steps, eos, penalty, early):
    """The sequences and scores of a search that starts over for every beam and step; ``logits_of(sequences) -> [n, V]``."""
    r = _Request(W, penalty, early)
    for _ in range(steps):
        if r.done:
            break
        live = [(i, s, h) for i, (s, h) in enumerate(r.beams) if s > -INF]
        logp = torch.log_softmax(logits_of([prompt + h for _, _, h in live]).double(), -1)
        cands = [(units._fp32(s + lp), i, v) for (i, s, _), row in zip(live, logp.tolist()) for v, lp in enumerate(row)]
        cands.sort(key=lambda c: (-c[0], c[1], c[2]))
        r.step(cands[:2 * W])
    n = len(r.beams[0][1])
    return r.finish(n)


def _train_logits(train):
    def logits_of(seqs):
        with torch.no_grad():
            return train(torch.tensor(seqs)).transpose(0, 1)[:, -1]
    return logits_of


@pytest.mark.parametrize("kind", ["contiguous", "paged", "pool", "continuous"])
@pytest.mark.parametrize("W,steps,penalty,early", [(1, 6, 1.0, False), (3, 12, 1.0, False), (4, 10, 0.3, True), (5, 7, 2.0, False)])
def test_beams_equal_a_search_without_a_cache(monkeypatch, kind, W, steps, penalty, early):
    monkeypatch.setattr(units, "EOS", 17)
    cache = {"contiguous": {}, "paged": dict(paged_kv=True), "pool": dict(paged_kv=True, num_kv_pages=60),
             "continuous": dict(paged_kv=True, num_kv_pages=60, is_continuous_batching=True)}[kind]
    cfg, train, inf = _models(monkeypatch, batch_size=2, max_batch_size=2 * W + 1, **cache)
    with torch.no_grad():
        train.lm_head.weight[17] *= 1.3
        inf.lm_head.weight[17] *= 1.3
    prompts = torch.randint(20, cfg.vocab_size, (2, 17))
    mask = torch.ones_like(prompts)
    mask[1, 8:] = 0                      # a prompt that ends with a page, one that does not
    ended = 0
    for again in range(2):               # lines that an earlier search has left
        out, scores = inf.generate_beams(prompts, mask, num_beams=W, max_new_tokens=steps, eos_token_id=17, length_penalty=penalty, early_stopping=early,
                                         num_return_sequences=W, return_scores=True)
        for b in range(2):
            L = int(mask[b].sum())
            want = _searched(_train_logits(train), prompts[b, :L].tolist(), W, steps, 17, penalty, early)
            for i, (s, h) in enumerate(want):
                row = out[b * W + i]
                assert row[:L].tolist() == prompts[b, :L].tolist() and row[L:L + len(h)].tolist() == h, (b, i)
                assert int((row[L + len(h):] != 0).sum()) == 0
                assert abs(float(scores[b * W + i]) - s) <= 1e-4 * abs(s)          # fp32 logits of two orders of summation, sums of a dozen
                ended += h[-1] == 17
        prompts = prompts.flip(0)
        mask = mask.flip(0)
    assert inf.kv_cache.pool is None or inf.kv_cache.pool.num_free > 0


def test_one_token_prompts_and_no_end(monkeypatch):
    monkeypatch.setattr(units, "EOS", -5)
    cfg, train, inf = _models(monkeypatch, batch_size=1, max_batch_size=3)
    prompt = torch.tensor([[77]])
    out = inf.generate_beams(prompt, num_beams=3, max_new_tokens=5)
    assert out[0].tolist() == [77] + _searched(_train_logits(train), [77], 3, 5, -5, 1.0, False)[0][1]
    greedy = inf.generate_beams(prompt, num_beams=1, max_new_tokens=5)
    assert torch.equal(greedy, inf.generate(prompt, max_new_tokens=5))


def test_generation_refused(monkeypatch):
    cfg, train, inf = _models(monkeypatch, batch_size=1, max_batch_size=4)
    ids = torch.randint(1, 100, (2, 10))
    for kw in (dict(num_beams=3), dict(num_beams=2, max_new_tokens=56), dict(num_beams=2, num_return_sequences=3), dict(num_beams=0),
               dict(num_beams=2, attention_mask=torch.zeros_like(ids)), dict(num_beams=2, max_new_tokens=0)):
        with pytest.raises(ValueError):
            inf.generate_beams(ids, **kw)
    with pytest.raises(ValueError):
        InferenceConfig(num_beams=33)


def test_rows_of_beams_need_cache_lines():
    for kw in (dict(batch_size=2, max_batch_size=2), dict(batch_size=1, tkg_batch_size=8, max_batch_size=4), dict(batch_size=1, max_batch_size=3)):
        with pytest.raises(ValueError):
            InferenceConfig(num_beams=4, **kw)          # the graph of a step would write behind the cache
    assert InferenceConfig(num_beams=4, batch_size=2, max_batch_size=8).tkg_batch_size == 8


def test_a_search_does_not_sample():
    with pytest.raises(ValueError):
        InferenceConfig(num_beams=2, do_sample=True, top_k=5)
    assert InferenceConfig(num_beams=1, do_sample=True, top_k=5).do_sample


def test_the_search_has_the_last_fields_of_a_configuration():
    names = [f.name for f in dataclasses.fields(InferenceConfig)]
    assert names[-5:] == ["pad_token_id", "eos_token_id", "num_beams", "length_penalty", "early_stopping"]


@pytest.mark.parametrize("cache", [{}, dict(paged_kv=True), dict(paged_kv=True, num_kv_pages=8)])
def test_a_cache_of_one_token_is_refused(cache):
    # a prompt of one token is computed as two, the second of which has no row there
    model = LlamaInferenceModel(tiny_llama(sequence_parallel_enabled=False), InferenceConfig(max_context_length=1, seq_len=1, max_batch_size=3, page_size=1, **cache))
    with pytest.raises(ValueError):
        model.generate_beams(torch.tensor([[5]]), num_beams=3, max_new_tokens=1)


# recurrent state, short convolutions, latent columns and layers that share keys next to plain keys and values
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("family,pages", [("rasodra", None), ("rasodra", 90), ("gogalix", None), ("gogalix", 90)])
def test_beams_of_recurrent_families(monkeypatch, family, pages, dev):
    monkeypatch.setattr(units, "EOS", 3)
    F = importlib.import_module(f"test_{family}")
    W, steps, cfg = 4, 9, F.config()
    model, sd = F.build(cfg, dev, torch.float32, lines=2 * W, paged=pages is not None, pages=pages)
    other, _ = F.build(cfg, dev, torch.float32, lines=W, sd=sd)

    def logits_of(seqs):
        ids = torch.tensor(seqs, device=dev)
        pos = torch.arange(ids.shape[1], device=dev).expand_as(ids)
        return other.forward_infer(ids, pos, return_logits=True, sample=False)[1].float().cpu()

    prompts = torch.tensor([F.tokens_of(cfg, 14, 1), F.tokens_of(cfg, 14, 2)], device=dev)
    mask = torch.ones_like(prompts)
    mask[0, 11:] = 0
    out, scores = model.generate_beams(prompts, mask, num_beams=W, max_new_tokens=steps, eos_token_id=3, num_return_sequences=W, return_scores=True)
    for b in range(2):
        L = int(mask[b].sum())
        for i, (s, h) in enumerate(_searched(logits_of, prompts[b, :L].tolist(), W, steps, 3, 1.0, False)):
            assert out[b * W + i, L:L + len(h)].tolist() == h, (b, i)
            assert abs(float(scores[b * W + i]) - s) <= 2e-3 * abs(s)          # the families' own bound between prompts and single tokens


@pytest.mark.parametrize("paged", [False, True])
def test_the_runner_searches_with_its_buckets(monkeypatch, paged):
    monkeypatch.setattr(units, "EOS", 17)
    cfg, train, _ = _models(monkeypatch, batch_size=1)
    with torch.no_grad():
        train.lm_head.weight[17] *= 1.3
    W, extra = 3, dict(paged_kv=True, page_size=8, num_kv_pages=80) if paged else {}
    ic = InferenceConfig(batch_size=2, num_beams=W, max_context_length=16, seq_len=48, buckets=[8, 16], eos_token_id=17, length_penalty=0.8, **extra)
    assert ic.tkg_batch_size == 6 and ic.max_batch_size == 6
    r = InferenceRunner(tiny_llama(sequence_parallel_enabled=False), ic, checkpoint_loader=train.state_dict, device=torch.device("cpu"))
    r.trace()
    for B, T in ((2, 11), (1, 5), (2, 8)):
        prompts = torch.randint(20, cfg.vocab_size, (B, T))
        out, scores = r.generate_beams(prompts, max_new_tokens=9, num_return_sequences=2, return_scores=True)
        assert torch.equal(r.generate(prompts, max_new_tokens=9), out[::2])
        for b in range(B):
            want = _searched(_train_logits(train), prompts[b].tolist(), W, 9, 17, 0.8, False)
            for i in range(2):
                h = want[i][1]
                assert out[b * 2 + i, T:T + len(h)].tolist() == h and abs(float(scores[b * 2 + i]) - want[i][0]) <= 1e-4 * abs(want[i][0])
    with pytest.raises(ValueError):
        r.generate_beams(torch.ones(3, 8, dtype=torch.long), max_new_tokens=4)
    with pytest.raises(ValueError):
        r.generate_beams(torch.ones(1, 8, dtype=torch.long), max_new_tokens=42)


@pytest.mark.parametrize("W,penalty", [(2, 1.0), (4, 0.0), (4, 0.6)])
def test_sequences_equal_those_of_transformers(W, penalty):
    transformers = pytest.importorskip("transformers")
    from neuronx_distributed_llama3_2_b200.inference import BeamSearch

    torch.manual_seed(0)
    model = transformers.LlamaForCausalLM(transformers.LlamaConfig(
        vocab_size=60, hidden_size=32, intermediate_size=64, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, eos_token_id=5,
        pad_token_id=0, bos_token_id=1)).eval().double()
    with torch.no_grad():
        model.lm_head.weight.mul_(40.0)
        model.lm_head.weight[5] *= 1.1
        for seed in range(6):
            ids = torch.randint(6, 60, (1, 7), generator=torch.Generator().manual_seed(seed))
            ref = model.generate(ids, num_beams=W, max_new_tokens=14, do_sample=False, length_penalty=penalty, early_stopping=False,
                                 num_return_sequences=W)[:, 7:].tolist()
            ref = [r[:r.index(5) + 1] if 5 in r else r for r in ref]
            s = BeamSearch(1, W, 14, eos_token_id=5, length_penalty=penalty)
            hist = [ids[0].tolist()] * W
            for t in range(14):
                if s.finished():
                    break
                tokens, parents = s.advance(model(torch.tensor(hist if t else hist[:1])).logits[:, -1].float())
                hist = [hist[p] + [v] for v, p in zip(tokens[0].tolist(), parents[0].tolist())]
            tokens, lengths, _ = s.finish()
            assert [tokens[0, i, :n].tolist() for i, n in enumerate(lengths[0].tolist())] == ref, seed


def _tp_worker(rank, world):
    from neuronx_distributed_llama3_2_b200.inference import _mock_parallel_state
    from neuronx_distributed_llama3_2_b200.parallel import parallel_state as ps

    kw = dict(max_context_length=16, seq_len=48, buckets=[16], num_beams=3, eos_token_id=17, use_cuda_graphs=False)
    with _mock_parallel_state(1, 0):          # one process, before the groups exist
        torch.manual_seed(0)
        train = LlamaForCausalLM(tiny_llama(sequence_parallel_enabled=False))
        with torch.no_grad():
            train.lm_head.weight.mul_(6.0)
        sd = {k: v.clone() for k, v in train.state_dict().items()}
        prompts = torch.randint(20, 512, (2, 13), generator=torch.Generator().manual_seed(5))
        ref = LlamaInferenceModel(tiny_llama(sequence_parallel_enabled=False), InferenceConfig(batch_size=2, **kw))
        ref.load_state_dict(sd)
        want, want_scores = ref.generate_beams(prompts, num_beams=3, max_new_tokens=12, eos_token_id=17, num_return_sequences=3, return_scores=True)
        ps.set_tensor_model_parallel_size(None)
        ps.set_tensor_model_parallel_rank(None)
    ps.initialize_model_parallel(tensor_model_parallel_size=2)
    for extra in ({}, dict(paged_kv=True, page_size=8, num_kv_pages=40)):
        r = InferenceRunner(tiny_llama(sequence_parallel_enabled=False), InferenceConfig(batch_size=2, tp_degree=2, **kw, **extra),
                            checkpoint_loader=lambda: sd, device=torch.device("cpu"))
        r.trace()
        got, scores = r.generate_beams(prompts, max_new_tokens=12, num_return_sequences=3, return_scores=True)
        assert torch.equal(got, want), (rank, got, want)
        assert bool(((scores - want_scores).abs() <= 1e-4 * want_scores.abs()).all())


def test_lines_that_no_beam_has_keep_their_pages():
    torch.manual_seed(0)
    train = LlamaForCausalLM(tiny_llama(sequence_parallel_enabled=False))
    ic = InferenceConfig(batch_size=2, num_beams=2, max_batch_size=6, max_context_length=16, seq_len=32, buckets=[16], paged_kv=True, page_size=8, num_kv_pages=40)
    r = InferenceRunner(tiny_llama(sequence_parallel_enabled=False), ic, checkpoint_loader=train.state_dict, device=torch.device("cpu"))
    r.trace()
    cache = r.model.kv_cache
    cache.reserve(5, 11)
    pages = cache.pool.block_row(5)[0][:2]
    for t in cache._tensors():
        t[pages] = 3.0
    for B in (2, 1):
        r.generate_beams(torch.randint(1, 500, (B, 9)), max_new_tokens=6)
    assert cache.pool.line_tokens(5) == 11 and cache.pool.block_row(5)[0][:2] == pages
    assert all(bool((t[pages] == 3.0).all()) for t in cache._tensors())


def test_two_ranks_search_like_one():
    run_distributed(_tp_worker, 2)


# ---- lines and pages of a cache ---------------------------------------------------------------------------------------

def _filled(cache, g):
    for t in cache._tensors() + cache._state_tensors():
        t.copy_(torch.randint(-99, 99, t.shape, generator=g).to(t))


def _line(cache, i, line, n):
    """Rows ``[0, n)`` of a line of layer ``i``, keys and values."""
    out = []
    for t in cache.layer(i):
        if cache.paged:
            pages = cache.block_table[line].long()
            out.append(t[pages].permute(1, 0, 2, 3).reshape(t.shape[1], -1, t.shape[3])[:, :n].clone())
        else:
            out.append(t[line, :, :n].clone())
    return out


SPECS = [(2, 8, 8), (1, 12, 6, "columns"), None, (2, 8, 4, "heads", 3), (2, 8, 8)]


def _cache(kind, device, lines=6, **kw):
    paged = {"contiguous": {}, "paged": dict(paged=True, page_size=4), "pool": dict(paged=True, page_size=4, num_pages=40)}[kind]
    return KVCache(5, lines, 0, 24, 0, dtype=torch.float32, device=device, layer_specs=SPECS, share_from={4: 0},
                   state_specs={2: {"S": (2, 3, 4), "n": (5,)}}, **{**paged, **kw})


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["contiguous", "paged", "pool"])
def test_lines_of_a_search(device, kind):
    g = torch.Generator().manual_seed(3)
    cache, W, lengths = _cache(kind, device), 3, [7, 8]
    if kind == "pool":
        for b in range(2):
            cache.reserve(b * W, 12)
    _filled(cache, g)
    layers = [0, 1, 3, 4]
    before = {(i, b): _line(cache, i, b * W, lengths[b]) for i in layers for b in range(2)}
    states = {k: v.clone() for k, v in cache.state(2).items()}
    lines = cache.beams(lengths, W, 10)
    assert isinstance(lines, BeamLines) and lines.start.tolist() == lengths
    for i in layers:
        for line in range(2 * W):
            assert all(torch.equal(a, b) for a, b in zip(_line(cache, i, line, lengths[line // W]), before[i, line // W])), (i, line)
    for k, v in cache.state(2).items():
        assert torch.equal(v, states[k][[0, 0, 0, 3, 3, 3]])
    if kind == "pool":
        assert cache.pool.private_from(0, 6) == [4, 4, 4, 8, 8, 8]          # a page of one prompt is shared, both of the other
        assert cache.pool.num_free == 40 - (1 + 3 * 4) - (2 + 3 * 3)
    # rows behind the prompts, a value a line
    for t in cache._state_tensors():
        t.copy_(torch.arange(6.0).reshape([6] + [1] * (t.dim() - 1)).expand_as(t))
    for line in range(2 * W):
        for pos in range(lengths[line // W], lengths[line // W] + 4):
            for t in cache._tensors():
                if cache.paged:
                    t[int(cache.block_table[line, pos // 4]), :, pos % 4] = line * 100 + pos
                else:
                    t[line, :, pos] = line * 100 + pos
    end = torch.tensor([n + 4 for n in lengths], device=device)
    for parents in ([[0, 0, 2], [2, 1, 1]], [[1, 2, 0], [1, 0, 0]]):
        had = {(i, line): _line(cache, i, line, 12) for i in layers for line in range(6)}
        state = [t.clone() for t in cache._state_tensors()]
        lines.reorder(torch.tensor(parents, device=device), end)
        for line in range(6):
            b, frm = line // W, line // W * W + parents[line // W][line % W]
            n = lengths[b]
            for i in layers:
                for now, own, new in zip(_line(cache, i, line, 12), had[i, line], had[i, frm]):
                    assert torch.equal(now[:, :n], own[:, :n]) and torch.equal(now[:, n:n + 4], new[:, n:n + 4]) and torch.equal(now[:, n + 4:], own[:, n + 4:])
            assert all(torch.equal(t[line], s[frm]) for t, s in zip(cache._state_tensors(), state))
    lines.reorder(torch.tensor([[0, 1, 1], [0, 1, 2]], device=device))          # as far as there is room
    if kind == "pool":
        cache.free(5)
        cache.fork(4, 5)
        with pytest.raises(ValueError):
            lines.reorder(torch.tensor([[0, 1, 2]] * 2, device=device), end)
        with pytest.raises(ValueError):
            cache.reorder_lines(torch.tensor([[0, 1, 2]] * 2, device=device))
    for args in (([7, 8, 9], 3), ([7], 0), ([], 3), ([25], 2), ([20], 2, 5), ([-1], 2)):
        with pytest.raises(ValueError):
            cache.beams(*args)


@pytest.mark.parametrize("device", DEVICES)
def test_a_prompt_that_ends_in_a_page_of_another_line(device):
    cache = _cache("pool", device, lines=6)
    cache.reserve(0, 8)
    cache.reserve(2, 8)
    cache.fork_lines(0, [4])
    _filled(cache, torch.Generator().manual_seed(6))
    other = {i: _line(cache, i, 4, 8) for i in (0, 1, 3)}
    lines = cache.beams([6, 8], 2, 4)          # rows 6 and 7 are written again
    assert all(at <= n for at, n in zip(cache.pool.private_from(0, 4), (6, 6, 8, 8)))
    for line in range(4):
        for i in (0, 1, 3):
            assert all(torch.equal(a, b[:, :6]) for a, b in zip(_line(cache, i, line, 6), other[i])) or line > 1
        for pos in range(6 if line < 2 else 8, 10):
            for t in cache._tensors():
                t[int(cache.block_table[line, pos // 4]), :, pos % 4] = 100 * line + pos
    lines.reorder(torch.tensor([[1, 1], [0, 0]], device=device), torch.tensor([10, 10], device=device))
    for i in (0, 1, 3):
        assert all(torch.equal(a, b) for a, b in zip(_line(cache, i, 4, 8), other[i]))
        for line in range(4):
            for now, had in zip(_line(cache, i, line, 10), other[i]):
                first, frm = (6, 1) if line < 2 else (8, 2)
                assert torch.equal(now[:, first:], (100.0 * frm + torch.arange(first, 10, device=device))[None, :, None].expand_as(now[:, first:]))
                assert line > 1 or torch.equal(now[:, :6], had[:, :6])


@pytest.mark.parametrize("pages", [6, 7, 9, 11, 13])
def test_beams_that_a_pool_has_no_pages_for_leave_the_prompts_alone(pages):
    cache = _cache("pool", None, num_pages=pages)
    cache.reserve(0, 7)
    cache.reserve(3, 8)
    _filled(cache, torch.Generator().manual_seed(8))
    had = [_line(cache, 0, line, n) for line, n in ((0, 7), (3, 8))]
    with pytest.raises(MemoryError):
        cache.beams([7, 8], 3, 12)
    assert cache.pool.num_free == pages - 4 and [cache.pool.line_tokens(line) for line in range(6)] == [7, 0, 0, 8, 0, 0]
    for rows, (line, n) in zip(had, ((0, 7), (3, 8))):
        assert all(torch.equal(a, b) for a, b in zip(_line(cache, 0, line, n), rows))


@pytest.mark.parametrize("device", DEVICES)
def test_pages_of_a_pool_fork_compact_and_move(device):
    g = torch.Generator().manual_seed(4)
    cache = _cache("pool", device, lines=8)
    for line, n in ((0, 10), (1, 24), (2, 3), (3, 17)):
        cache.reserve(line, n)
    _filled(cache, g)
    cache.fork_lines(0, [4, 5, 6])
    held = {(i, line): _line(cache, i, line, n) for i in (0, 1, 3) for line, n in ((0, 10), (3, 17), (4, 10), (5, 10), (6, 10))}
    for (i, line), rows in held.items():
        if line > 3:
            assert all(torch.equal(a, b) for a, b in zip(rows, held[i, 0]))
    cache.free(1), cache.free(2)
    used = 40 - cache.pool.num_free
    assert cache.compact() == used and used == 2 + 4 + 5
    assert max(max(cache.pool.block_row(line)[0][:cache.pool.block_row(line)[1]], default=0) for line in range(8)) == used - 1
    for (i, line), rows in held.items():
        assert all(torch.equal(a, b) for a, b in zip(_line(cache, i, line, rows[0].shape[1]), rows)), (i, line)
    assert cache.compact() == used          # nothing to do
    cache.prepare_write(0, 9)
    cache.prepare_write(4, 0)
    assert not cache.pool.page_shared(4, 0) and all(torch.equal(a, b) for a, b in zip(_line(cache, 0, 4, 10), held[0, 4]))
    with pytest.raises(MemoryError):
        cache.resize_pool(5)
    for pages in (used + 1, 30, 50):
        cache.resize_pool(pages)
        assert cache.pool.num_pages == pages == cache.k[0].shape[0] and cache.pool.num_free == pages - used - 1
        for (i, line), rows in held.items():
            assert all(torch.equal(a, b) for a, b in zip(_line(cache, i, line, rows[0].shape[1]), rows)), (i, line)
        assert cache.v[1].data_ptr() == cache.k[1].data_ptr()          # columns of the same rows
    # more forks than there are pages: none of them is left half made
    small = _cache("pool", device, lines=8, num_pages=6)
    small.reserve(0, 15)
    with pytest.raises(MemoryError):
        small.fork_lines(0, [1, 2, 3])
    assert small.pool.num_free == 2 and all(small.pool.block_row(line)[1] == 0 for line in (1, 2, 3))
    small.fork_lines(0, [1, 2])
    with pytest.raises(AssertionError):
        _cache("contiguous", device).copy_pages([0], [1])


@pytest.mark.parametrize("pages", [12, 40, 60])
def test_a_resized_pool_lets_the_old_tensors_go(monkeypatch, pages):
    cache = _cache("pool", None)
    cache.reserve(0, 10)
    cache.fork_lines(0, [1, 2])
    held = [weakref.ref(t) for t in cache._tensors()]
    alive, resized = [], KVCache._resized

    def counted(t, num_pages, used):
        new = resized(t, num_pages, used)
        alive.append(sum(r() is not None for r in held))
        return new

    monkeypatch.setattr(KVCache, "_resized", staticmethod(counted))
    cache.resize_pool(pages)
    assert not any(r() is not None for r in held)
    assert alive == list(range(len(held), 0, -1))          # one after the other
    cache.fork_lines(0, [3])
    assert cache.tensors.cache[0].shape[0] == pages


@pytest.mark.parametrize("pages", [12, 60])
@pytest.mark.parametrize("at", range(5))
def test_a_pool_that_could_not_be_resized_names_no_page_that_is_not_there(monkeypatch, pages, at):
    cache = _cache("pool", None)
    cache.reserve(1, 3), cache.reserve(0, 10), cache.free(1)
    _filled(cache, torch.Generator().manual_seed(2))
    layers = (0, 1, 3, 4)
    held = {i: _line(cache, i, 0, 10) for i in layers}
    calls, resized = [], KVCache._resized

    def failing(t, num_pages, used):
        calls.append(t)
        if len(calls) == at + 1:
            raise torch.OutOfMemoryError("no room")
        return resized(t, num_pages, used)

    def check():
        assert cache.pool.num_pages <= min(t.shape[0] for t in cache._tensors())
        assert cache.pool.num_free == cache.pool.num_pages - 3
        for i in layers:
            assert all(torch.equal(a, b) for a, b in zip(_line(cache, i, 0, 10), held[i]))
            k, v = cache.layer(i)
            assert (v._base is None) == (i != 1) and k.shape[0] >= cache.pool.num_pages <= v.shape[0]

    monkeypatch.setattr(KVCache, "_resized", staticmethod(failing))
    with pytest.raises(torch.OutOfMemoryError):
        cache.resize_pool(pages)
    check()
    cache.reserve(2, 24)
    cache.fork_lines(0, [3])          # the kernels' layout copes with pools of two sizes
    cache.free(2), cache.free(3)
    monkeypatch.setattr(KVCache, "_resized", staticmethod(resized))
    cache.resize_pool(pages)
    check()
    assert cache.pool.num_pages == pages == max(t.shape[0] for t in cache._tensors())


@pytest.mark.gpu
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("W", [2, 5])
def test_captured_graphs_and_eager_steps_agree(paged, W):
    """The runner with graphs and the model without: the same kernels on the same rows, hence the same sequences."""
    torch.manual_seed(1)
    cfg = tiny_llama(sequence_parallel_enabled=False, torch_dtype=torch.bfloat16, hidden_size=512, head_dim=64)
    extra = dict(paged_kv=True, page_size=16, num_kv_pages=64) if paged else {}
    ic = InferenceConfig(batch_size=2, num_beams=W, max_context_length=32, seq_len=64, buckets=[32], eos_token_id=11, **extra)
    train = LlamaForCausalLM(cfg, device=torch.device("cuda"))
    with torch.no_grad():
        train.lm_head.weight.mul_(6.0)
    sd = {k: v.clone() for k, v in train.state_dict().items()}
    r = InferenceRunner(cfg, ic, checkpoint_loader=lambda: sd, device=torch.device("cuda"))
    r.trace()
    prompts = torch.randint(20, cfg.vocab_size, (2, 32), device="cuda")
    out, scores = r.generate_beams(prompts, max_new_tokens=20, num_return_sequences=W, return_scores=True)
    again = r.generate(prompts, max_new_tokens=20)
    eager, eager_scores = r.model.generate_beams(prompts, num_beams=W, max_new_tokens=20, eos_token_id=11, num_return_sequences=W, return_scores=True)
    assert torch.equal(out, eager) and torch.equal(scores, eager_scores) and torch.equal(again, out[::W])
    assert bool((scores.view(2, W).diff(dim=1) <= 0).all())
    # what a sequence's tokens are worth, from one pass over it: bf16 keys, values and logits, sums of 20
    seq = out[0]
    n = int((seq[32:] != 0).sum())
    n = 20 if 11 not in seq[32:].tolist() else seq[32:].tolist().index(11) + 1
    with torch.no_grad():
        logits = train(seq[None]).transpose(0, 1)[0].float()
    logp = torch.log_softmax(logits, -1)[31:31 + n].gather(1, seq[32:32 + n, None]).sum()
    assert abs(float(logp) / n - float(scores[0])) <= 0.1
    r.close()
