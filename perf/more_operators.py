"""What beam search over the key/value cache is timed on: the choice of the best continuations over beams and vocabulary, the step
that keeps the beams' books, the sequences at the end, the reordering of cache lines and recurrent states by their parents, and
copies of pages for lines that fork or move.

Sizes come from this repository's configurations (Llama 1B / 8B, Mixtral, DBRX and BERT vocabularies and cache shapes, recurrent
states of the hybrid families) or are generic.  ``prepare`` makes inputs from the seed alone; ``run`` with ``own`` false is each
operator's definition in elementary torch operations, with ``own`` true the framework's call; ``exact`` restates the computed
numbers in float64.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def listed():
    return [
        # the first step after the prompt, four beams to be: one row of the 1B model's vocabulary, where launches count
        {"name": "select_first_step", "kind": "select", "groups": 1, "beams": 1, "vocab": 128256, "n": 8, "dtype": "bf16", "mask": "none"},
        # every later step of one request with four beams
        {"name": "select_one_request", "kind": "select", "groups": 1, "beams": 4, "vocab": 128256, "n": 8, "dtype": "bf16", "mask": "none"},
        # constrained decoding with an encoder's vocabulary, an odd number of tokens: most of them are left out
        {"name": "select_constrained", "kind": "select", "groups": 12, "beams": 5, "vocab": 30522, "n": 10, "dtype": "fp32", "mask": "inf"},
        # a batch of 32 requests with eight beams each over the 1B / 8B vocabulary
        {"name": "select_batch", "kind": "select", "groups": 32, "beams": 8, "vocab": 128256, "n": 16, "dtype": "bf16", "mask": "none"},
        # the books of one request
        {"name": "advance_one_request", "kind": "advance", "groups": 1, "beams": 4, "steps": 256, "step": 100, "mix": 1},
        # the books of a large batch
        {"name": "advance_batch", "kind": "advance", "groups": 256, "beams": 16, "steps": 128, "step": 77, "mix": 2},
        # the sequences of one short answer
        {"name": "finish_one_request", "kind": "finish", "groups": 1, "beams": 4, "step": 48, "mix": 3},
        # the sequences of a batch of long answers
        {"name": "finish_batch", "kind": "finish", "groups": 64, "beams": 8, "step": 2000, "mix": 4},
        # one request of the 1B model, 300 tokens behind its prompt
        {"name": "reorder_one_request", "kind": "reorder", "layers": 16, "groups": 1, "beams": 4, "heads": 8, "rows": 1024, "dim": 64,
         "states": 0, "state": 0, "longest": 300, "dtype": "bf16", "mix": 5},
        # a batch of hybrid layers: the 1B model's cache shape and a recurrent state of 8 heads of 128 x 64 per line in every second layer
        {"name": "reorder_batch_hybrid", "kind": "reorder", "layers": 16, "groups": 4, "beams": 8, "heads": 8, "rows": 1024, "dim": 64,
         "states": 8, "state": 65536, "longest": 900, "dtype": "bf16", "mix": 6},
        # four lines fork: the part of their last page that is in use, in every layer of the 1B model
        {"name": "pages_fork", "kind": "pages", "layers": 16, "heads": 8, "page": 128, "dim": 64, "pages": 64, "moves": 4, "partial": True,
         "dtype": "bf16", "mix": 7},
        # a pool of the 8B model's shape is compacted
        {"name": "pages_compact", "kind": "pages", "layers": 8, "heads": 8, "page": 128, "dim": 128, "pages": 300, "moves": 120,
         "partial": False, "dtype": "bf16", "mix": 8},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _costs(case):
    return work(case)["bytes"]


def _state_bytes(case):
    """What a case holds, for the kinds whose tensors are larger than what moves."""
    if case["kind"] == "reorder":
        lines = case["groups"] * case["beams"]
        size = DTYPES[case["dtype"]].itemsize
        return lines * (2 * case["layers"] * case["heads"] * case["rows"] * case["dim"] * size + 4 * case["states"] * case["state"])
    if case["kind"] == "pages":
        return 2 * case["layers"] * case["pages"] * case["heads"] * case["page"] * case["dim"] * DTYPES[case["dtype"]].itemsize
    return 0


def draw(rng):
    kind = rng.choice(["select", "select", "advance", "finish", "reorder", "reorder", "pages"])
    of_kind = [c for c in listed() if c["kind"] == kind]
    most, held = max(_costs(c) for c in of_kind), max(_state_bytes(c) for c in of_kind)
    while True:
        mix = rng.randrange(1 << 30)
        if kind == "select":
            beams = rng.choice([1, 2, 3, 4, 5, 8, 12, 16, 24, 32])
            case = {"groups": _spread(rng, 1, 64), "beams": beams, "vocab": _spread(rng, 500, 262144), "n": min(64, 2 * beams),
                    "dtype": rng.choice(["bf16", "fp16", "fp32"]), "mask": rng.choice(["none", "none", "inf", "lowest"])}
        elif kind in ("advance", "finish"):
            step = _spread(rng, 1, 2000)
            case = {"groups": _spread(rng, 1, 256), "beams": rng.randint(1, 32), "step": step, "mix": mix}
            if kind == "advance":
                case["steps"] = step + rng.randint(1, 64)
        elif kind == "reorder":
            rows = _spread(rng, 16, 2048)
            case = {"layers": _spread(rng, 1, 32), "groups": _spread(rng, 1, 16), "beams": rng.choice([2, 3, 4, 5, 8, 16, 32]),
                    "heads": rng.choice([1, 2, 3, 8]), "rows": rows, "dim": rng.choice([40, 64, 80, 128]),
                    "states": rng.choice([0, 0, 1, 6]), "state": _spread(rng, 16, 65536), "longest": rng.randint(1, rows),
                    "dtype": rng.choice(["bf16", "fp16", "fp32"]), "mix": mix}
        else:
            pages = _spread(rng, 4, 400)
            case = {"layers": _spread(rng, 1, 32), "heads": rng.choice([1, 2, 3, 8]), "page": rng.choice([16, 32, 64, 128]),
                    "dim": rng.choice([40, 64, 80, 128]), "pages": pages, "moves": rng.randint(1, pages // 2), "partial": rng.random() < 0.5,
                    "dtype": rng.choice(["bf16", "fp16", "fp32"]), "mix": mix}
        case["kind"] = kind
        if _costs(case) <= most and _state_bytes(case) <= held:
            return case


# ---- what a step of a search looks like -------------------------------------------------------------------------------

def parents_of(case):
    """Per group: the line that each line continues.  A beam that survives stays where it is and the others take copies, which is
    how the books place them, so no line that is read is written."""
    rng, out = random.Random(case["mix"]), []
    for _ in range(case["groups"]):
        W = case["beams"]
        alive = sorted(rng.sample(range(W), max(1, round(W * rng.uniform(0.3, 0.8)))))
        out.append([w if w in alive else rng.choice(alive) for w in range(W)])
    return out


def ranges_of(case):
    """Per group: the first and the end row of what follows its prompt."""
    rng, out = random.Random(case["mix"] + 1), []
    for _ in range(case["groups"]):
        n = max(1, min(case["rows"], round(case["longest"] * rng.uniform(0.8, 1.0))))
        start = rng.randint(0, case["rows"] - n)
        out.append((start, start + n))
    return out


def moves_of(case):
    """Pages that are copied, the free pages that they go to, and how many rows of each are in use."""
    rng = random.Random(case["mix"])
    some = rng.sample(range(case["pages"]), 2 * case["moves"])
    rows = [rng.randint(1, case["page"]) if case["partial"] else case["page"] for _ in range(case["moves"])]
    return some[:case["moves"]], some[case["moves"]:], rows


def work(case):
    if case["kind"] == "select":
        n = case["groups"] * case["beams"] * case["vocab"]
        return {"bytes": n * DTYPES[case["dtype"]].itemsize + case["groups"] * (4 * case["beams"] + 20 * case["n"]), "flops": 4 * n}
    if case["kind"] == "advance":
        n = case["groups"] * case["beams"]
        # candidates 2 x 20, scores, the pool in and out, tokens, parents, a row of the history
        return {"bytes": n * (40 + 4 + 4 + 24 + 16 + 8) + 2 * case["groups"], "flops": 8 * n * case["beams"]}
    if case["kind"] == "finish":
        n = case["groups"] * case["beams"]
        return {"bytes": n * case["step"] * (8 + 8) + n * 32, "flops": 2 * n * case["step"]}
    size = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "reorder":
        total = 0
        for p, (lo, hi) in zip(parents_of(case), ranges_of(case)):
            lines = sum(a != w for w, a in enumerate(p)) + len({a for w, a in enumerate(p) if a != w})
            total += lines * ((hi - lo) * case["heads"] * case["dim"] * size * 2 * case["layers"] + 4 * case["state"] * case["states"])
        return {"bytes": total + 8 * case["groups"] * case["beams"], "flops": 0}
    return {"bytes": 2 * 2 * case["layers"] * sum(moves_of(case)[2]) * case["heads"] * case["dim"] * size, "flops": 0}


EOS, PAD = 2, 0


def _candidates(case, rng, groups, W, N):
    """Sorted candidates as a search meets them: per beam at most one that ends, scores of neighbours a few tenths apart."""
    gap = rng.exponential(0.3, (groups, N)).astype(np.float32)
    scores = -(rng.uniform(5.0, 60.0, (groups, 1)).astype(np.float32) + np.cumsum(gap, 1, dtype=np.float32))
    beams = rng.integers(0, W, (groups, N))
    tokens = rng.permuted(np.broadcast_to(np.arange(3, 3 + 40 * N), (groups, 40 * N)), axis=1)[:, :N].copy()
    for b in range(groups):
        seen = set()
        for r in np.flatnonzero(rng.random(N) < 0.3):
            if beams[b, r] not in seen:
                seen.add(beams[b, r])
                tokens[b, r] = EOS
    return scores, beams, tokens


def _books(case, rng, groups, W, step):
    """A pool that is partly filled, sorted; some requests are over."""
    held = rng.integers(0, W + 1, groups)
    scores = -np.sort(rng.uniform(0.5, 9.0, (groups, W)).astype(np.float32), 1)
    empty = np.arange(W)[None] >= held[:, None]
    scores[empty] = -np.inf
    lengths = rng.integers(1, max(2, step + 1), (groups, W)).astype(np.int32)
    slots = rng.integers(0, W, (groups, W)).astype(np.int32)
    lengths[empty], slots[empty] = 0, 0
    done = (held == W) & (rng.random(groups) < 0.5)
    return scores, lengths, slots, done


def _laid_out(cache, states=()):
    """A program's cache is laid out for the kernels once."""
    if not own:
        return None
    from neuronx_distributed_llama3_2_b200.ops.kv_lines import CacheTensors

    return CacheTensors(cache, states)


def prepare(case, seed):
    dev = _device()
    g = torch.Generator(device=dev).manual_seed(seed)
    kind = case["kind"]
    if kind == "select":
        dtype = DTYPES[case["dtype"]]
        B, W, V, n = case["groups"], case["beams"], case["vocab"], case["n"]
        x = torch.randn(B * W, V, generator=g, device=dev) * 2.5
        if dtype == torch.float32:
            x += torch.randn(1, V, generator=g, device=dev)
        x = x.to(dtype)
        if case["mask"] != "none":
            allowed = torch.rand(B * W, V, generator=g, device=dev) < 0.1
            allowed[:, : n] = True
            x.masked_fill_(~allowed, -math.inf if case["mask"] == "inf" else torch.finfo(dtype).min)
        scores = -torch.sort(torch.rand(B, W, generator=g, device=dev) * 4.0 + 10.0, dim=1).values
        return {"case": case, "logits": x.view(B, W, V), "scores": scores}
    if kind in ("advance", "finish"):
        rng = np.random.default_rng([seed, case["mix"]])
        B, W, step = case["groups"], case["beams"], case["step"]
        T = case["steps"] if kind == "advance" else step

        def put(a):
            return torch.from_numpy(np.ascontiguousarray(a)).to(dev)

        pool = tuple(put(a) for a in _books(case, rng, B, W, step))
        running = put(-np.sort(rng.uniform(3.0, 70.0, (B, W)).astype(np.float32), 1))
        history = (put(rng.integers(3, 30000, (T, B, W)).astype(np.int32)), put(rng.integers(0, W, (T, B, W)).astype(np.int32)))
        state = {"case": case, "pool": pool, "running": running, "history": history, "penalty": 0.9}
        if kind == "advance":
            state["candidates"] = tuple(put(a) for a in _candidates(case, rng, B, W, 2 * W))
        return state
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dtype):
        out = torch.empty(shape, dtype=dtype, device=dev)
        return out.normal_(generator=g)

    if kind == "reorder":
        lines = case["groups"] * case["beams"]
        cache = [normal(lines, case["heads"], case["rows"], case["dim"]) for _ in range(2 * case["layers"])]
        states = [normal(lines, case["state"], dtype=torch.float32) for _ in range(case["states"])]
        lo, hi = zip(*ranges_of(case))
        return {"case": case, "cache": cache, "states": states, "laid_out": _laid_out(cache, states), "lo": lo, "hi": hi,
                "parents": torch.tensor(parents_of(case), device=dev), "start": torch.tensor(lo, device=dev), "end": torch.tensor(hi, device=dev)}
    cache = [normal(case["pages"], case["heads"], case["page"], case["dim"]) for _ in range(2 * case["layers"])]
    src, dst, rows = (torch.tensor(a, device=dev) for a in moves_of(case))
    return {"case": case, "cache": cache, "laid_out": _laid_out(cache), "src": src, "dst": dst, "rows": rows if case["partial"] else None, "counts": moves_of(case)[2]}


# ---- the plain forms --------------------------------------------------------------------------------------------------

def _plain_select(s):
    """Log-probabilities in 64 bits: sums of near scores decide between candidates of different beams."""
    x, n = s["logits"].double(), s["case"]["n"]
    top = x.amax(-1, keepdim=True)
    x = x - (top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))) + s["scores"].double()[..., None]
    flat = x.flatten(1)
    kth = torch.topk(flat, n, dim=1).values[:, -1:]
    # everything above the n-th value, then its ties from the lowest index on
    above, tied = flat > kth, flat == kth
    take = above | (tied & (tied.cumsum(1) <= n - above.sum(1, keepdim=True)))
    at = take.nonzero()[:, 1].view(-1, n)
    score = flat.gather(1, at)
    order = torch.sort(score, dim=1, descending=True, stable=True).indices
    at, score = at.gather(1, order), score.gather(1, order)
    V = s["case"]["vocab"]
    return {"scores": score.float(), "beams": at // V, "tokens": at % V}


def _merge(W, *pairs):
    """The best ``W`` of entries side by side, of equals the first; places without an entry are zero."""
    score = torch.cat([p[0] for p in pairs], 1)
    order = torch.sort(score, dim=1, descending=True, stable=True).indices[:, :W]
    score = score.gather(1, order)
    rest = [torch.cat(cols, 1).gather(1, order) for cols in zip(*(p[1:] for p in pairs))]
    return [score] + [torch.where(score > -math.inf, r, torch.zeros_like(r)) for r in rest]


def _plain_advance(s):
    case, (scores, beams, tokens), step = s["case"], s["candidates"], s["case"]["step"]
    B, W, N = case["groups"], case["beams"], scores.shape[1]
    dev = scores.device
    pool_scores, pool_lengths, pool_slots, done = s["pool"]
    norm = torch.full((1, 1), (step + 1) ** s["penalty"], dtype=torch.float32, device=dev)
    over = (tokens == EOS) & (torch.arange(N, device=dev) < W) & (scores > -math.inf)
    new = _merge(W, (pool_scores, pool_lengths, pool_slots),
                 (torch.where(over, scores / norm, -math.inf), torch.full_like(beams, step + 1, dtype=torch.int32), beams.int()))
    goes_on = tokens != EOS
    pick = torch.sort((~goes_on).int(), dim=1, stable=True).indices[:, :W]
    valid = goes_on.gather(1, pick)
    score = torch.where(valid, scores.gather(1, pick), -math.inf)
    parent, token = beams.gather(1, pick), torch.where(valid, tokens.gather(1, pick), PAD)
    # the best child of a beam stays in its line, the others go to the lines that nobody continues, in order
    same = (parent[:, :, None] == parent[:, None, :]) & valid[:, None, :]
    stays = valid & ~(same & torch.ones(W, W, dtype=torch.bool, device=dev).tril(-1)).any(-1)
    taken = ((torch.arange(W, device=dev)[None, :, None] == parent[:, None, :]) & stays[:, None, :]).any(-1)
    free = torch.sort(taken.int(), dim=1, stable=True).indices
    slot = torch.where(stays, parent, free.gather(1, ((~stays).cumsum(1) - 1).clamp(min=0)))
    parent = torch.where(valid, parent, slot)

    def place(x):
        return torch.empty_like(x).scatter_(1, slot, x)

    was = done[:, None]
    running = torch.where(was, s["running"], place(score))
    next_tokens = torch.where(was, PAD, place(token))
    parents = torch.where(was, torch.arange(W, device=dev)[None], place(parent))
    out_pool = [torch.where(was, a, b) for a, b in zip((pool_scores, pool_lengths, pool_slots), new)]
    is_done = done | ((out_pool[0][:, -1] > -math.inf) & (out_pool[0][:, -1:] >= running.amax(1, keepdim=True) / norm)[:, 0])
    s["history"][0][step] = next_tokens.int()
    s["history"][1][step] = parents.int()
    return {"scores": running, "tokens": next_tokens, "parents": parents, "pool": out_pool, "done": is_done,
            "history": [h[step] for h in s["history"]]}


def _plain_finish(s):
    case, step = s["case"], s["case"]["step"]
    B, W = case["groups"], case["beams"]
    pool_scores, pool_lengths, pool_slots, done = s["pool"]
    dev = done.device
    norm = torch.full((1, 1), step ** s["penalty"], dtype=torch.float32, device=dev)
    score, length, slot, ended = _merge(
        W, (pool_scores, pool_lengths, pool_slots, torch.ones(B, W, dtype=torch.int32, device=dev)),
        (torch.where(done[:, None], -math.inf, s["running"] / norm), torch.full((B, W), step, dtype=torch.int32, device=dev),
         torch.arange(W, dtype=torch.int32, device=dev).expand(B, W), torch.zeros(B, W, dtype=torch.int32, device=dev)))
    tokens = torch.full((B, W, step), PAD, dtype=torch.int64, device=dev)
    slot, ended = slot.long(), ended.bool()
    for t in range(step - 1, -1, -1):
        last = ended & (length - 1 == t)
        inside = (length > t) & ~last
        tokens[:, :, t] = torch.where(last, EOS, torch.where(inside, s["history"][0][t].gather(1, slot), PAD))
        slot = torch.where(inside, s["history"][1][t].gather(1, slot).long(), slot)
    return {"tokens": tokens, "lengths": length.long(), "scores": score}


def _plain_reorder(s):
    W = s["case"]["beams"]
    lines = s["parents"] + W * torch.arange(s["case"]["groups"], device=s["parents"].device)[:, None]
    for t in s["cache"]:
        for b, (lo, hi) in enumerate(zip(s["lo"], s["hi"])):
            t[b * W:(b + 1) * W, :, lo:hi] = t[:, :, lo:hi].index_select(0, lines[b])
    for t in s["states"]:
        t.copy_(t.index_select(0, lines.flatten()))
    return {"cache": s["cache"], "states": s["states"]}


def _plain_pages(s):
    if s["rows"] is not None:
        used = torch.arange(s["case"]["page"], device=s["src"].device)[None, None, :, None] < s["rows"][:, None, None, None]
    for t in s["cache"]:
        new = t.index_select(0, s["src"])
        if s["rows"] is not None:
            new = torch.where(used, new, t.index_select(0, s["dst"]))
        t[s["dst"]] = new
    return {"cache": s["cache"]}


# ---- the framework's calls --------------------------------------------------------------------------------------------

def _own_select(s):
    from neuronx_distributed_llama3_2_b200.ops.beam_search import beam_select

    scores, beams, tokens = beam_select(s["logits"], s["scores"], s["case"]["n"])
    return {"scores": scores, "beams": beams, "tokens": tokens}


def _own_advance(s):
    from neuronx_distributed_llama3_2_b200.ops.beam_search import BeamHistory, BeamPool, beam_advance

    step = s["case"]["step"]
    running, tokens, parents, pool = beam_advance(s["candidates"], s["running"], BeamPool(*s["pool"]), BeamHistory(*s["history"]), step,
                                                  eos_token_id=EOS, pad_token_id=PAD, length_penalty=s["penalty"])
    return {"scores": running, "tokens": tokens, "parents": parents, "pool": [pool.scores, pool.lengths, pool.slots], "done": pool.done,
            "history": [h[step] for h in s["history"]]}


def _own_finish(s):
    from neuronx_distributed_llama3_2_b200.ops.beam_search import BeamHistory, BeamPool, beam_finish

    tokens, lengths, scores = beam_finish(s["running"], BeamPool(*s["pool"]), BeamHistory(*s["history"]), s["case"]["step"],
                                          eos_token_id=EOS, pad_token_id=PAD, length_penalty=s["penalty"])
    return {"tokens": tokens, "lengths": lengths, "scores": scores}


def _own_reorder(s):
    from neuronx_distributed_llama3_2_b200.ops.kv_lines import reorder_lines_

    reorder_lines_(s["laid_out"] or _laid_out(s["cache"], s["states"]), s["parents"], s["start"], s["end"])
    return {"cache": s["cache"], "states": s["states"]}


def _own_pages(s):
    from neuronx_distributed_llama3_2_b200.ops.kv_lines import copy_pages_

    copy_pages_(s["laid_out"] or _laid_out(s["cache"]), s["src"], s["dst"], rows=s["rows"])
    return {"cache": s["cache"]}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"select": _own_select, "advance": _own_advance, "finish": _own_finish, "reorder": _own_reorder, "pages": _own_pages}[kind](state)
    return {"select": _plain_select, "advance": _plain_advance, "finish": _plain_finish, "reorder": _plain_reorder, "pages": _plain_pages}[kind](state)


# ---- in 64 bits -------------------------------------------------------------------------------------------------------

def _exact_select(case, s):
    """Row by row with numpy: only the best of a row can be among the best of its group."""
    n, V = case["n"], case["vocab"]
    out = [[], [], []]
    scores = s["scores"].cpu().double().numpy()
    for b in range(case["groups"]):
        found = []
        for w in range(case["beams"]):
            x = s["logits"][b, w].cpu().float().numpy().astype(np.float64)
            base = scores[b, w] - np.logaddexp.reduce(x[np.argsort(x)]) if V < 2000 else scores[b, w] - x.max() - math.log(np.exp(x - x.max()).sum())
            floor = np.partition(x, V - n)[V - n] if V > n else -math.inf
            best = np.flatnonzero(x >= floor)
            best = best[np.argsort(-x[best], kind="stable")][:n]
            found += [(-(base + x[v]), w * V + int(v)) for v in best]
        found.sort()
        for at, col in ((0, [-f for f, _ in found[:n]]), (1, [i // V for _, i in found[:n]]), (2, [i % V for _, i in found[:n]])):
            out[at].append(col)
    dev = s["scores"].device
    return {"scores": torch.tensor(out[0], dtype=torch.float64, device=dev), "beams": torch.tensor(out[1], device=dev),
            "tokens": torch.tensor(out[2], device=dev)}


def _exact_advance(case, s):
    """Request by request, as lists.  Only the pool's scores are computed numbers."""
    step, W = case["step"], case["beams"]
    norm = float(step + 1) ** s["penalty"]
    cand = [t.cpu().tolist() for t in s["candidates"]]
    pool = [t.cpu().tolist() for t in s["pool"]]
    running = s["running"].cpu().tolist()
    scores, kept = [], []
    for b in range(case["groups"]):
        if pool[3][b]:
            scores.append(pool[0][b])
            kept.append(running[b])
            continue
        entries, line, children = list(pool[0][b]), [-math.inf] * W, []
        for r, (x, p, token) in enumerate(zip(*(c[b] for c in cand))):
            if token == EOS:
                if r < W and x > -math.inf:
                    entries.append(x / norm)
            elif len(children) < W:
                children.append((x, p))
        scores.append(sorted(entries, reverse=True)[:W])
        parents = [p for _, p in children]
        free = iter([w for w in range(W) if w not in parents])
        for i, (x, p) in enumerate(children):
            line[p if p not in parents[:i] else next(free)] = x
        kept.append(line)
    dev = s["running"].device
    return {"scores": torch.tensor(kept, dtype=torch.float64, device=dev), "tokens": None, "parents": None,
            "pool": [torch.tensor(scores, dtype=torch.float64, device=dev), None, None], "done": None, "history": [None, None]}


def _exact_finish(case, s):
    norm = float(case["step"]) ** s["penalty"]
    pool, done = s["pool"][0].cpu().double(), s["pool"][3].cpu()
    running = (s["running"].cpu().double() / norm).masked_fill(done[:, None], -math.inf)
    best = np.sort(torch.cat([pool, running], 1).numpy(), axis=1)[:, ::-1][:, :case["beams"]]
    return {"tokens": None, "lengths": None, "scores": torch.from_numpy(best.copy()).to(s["running"].device)}


def exact(case, seed):
    if case["kind"] in ("reorder", "pages"):
        return None          # copies: nothing is computed
    s = prepare(case, seed)
    return {"select": _exact_select, "advance": _exact_advance, "finish": _exact_finish}[case["kind"]](case, s)
