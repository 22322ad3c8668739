"""The operators of beam search and of cache lines and pages: against definitions in 64 bits and plain lists, on the CPU (torch forms) and on the
GPU (kernels), and what they refuse."""
import itertools
import math
import random
from pathlib import Path

import pytest
import torch

from neuronx_distributed_llama3_2_b200.ops import beam_search as bs
from neuronx_distributed_llama3_2_b200.ops import kv_lines as kl

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
INF = math.inf


# ---- the candidates ---------------------------------------------------------------------------------------------------

def _select_oracle(logits, scores, n):
    """All candidates as a sorted list, in 64 bits."""
    B, W = scores.shape
    V = logits.shape[-1]
    rows = logits.reshape(B, W, V).double().cpu()
    out = []
    for b in range(B):
        found = []
        for w in range(W):
            x = rows[b, w]
            s = float(scores[b, w])
            usable = not bool(x.isnan().any()) and not bool((x == INF).any()) and bool((x > -INF).any()) and s > -INF
            lse = float(torch.logsumexp(x, 0)) if usable else 0.0
            found += [(-(s + (v - lse)) if usable and v > -INF else INF, w * V + i) for i, v in enumerate(x.tolist())]
        found.sort()
        out.append(found[:n])
    return (torch.tensor([[-f for f, _ in r] for r in out], dtype=torch.float64), torch.tensor([[i // V for _, i in r] for r in out]),
            torch.tensor([[i % V for _, i in r] for r in out]))


def _check_select(logits, scores, n):
    got = bs.beam_select(logits, scores, n)
    ref = _select_oracle(logits, scores, n)
    assert got[0].dtype == torch.float32 and got[1].dtype == got[2].dtype == torch.int64
    assert torch.equal(got[1].cpu(), ref[1]) and torch.equal(got[2].cpu(), ref[2])
    g, r = got[0].cpu().double(), ref[0]
    low = r.float() == -INF          # nothing, or below what fp32 holds
    assert torch.equal(g == -INF, low)
    fine = ~low
    # exponentials of 2^-21 and sums of 2^-21 relative move log-sum-exp by no more than 2^-20; the result is rounded to fp32 once
    assert ((g - r).abs()[fine] <= 2.0 ** -20 + 2.0 ** -24 * r.abs()[fine]).all()


# rows that end inside a vector and inside a chunk, one token, more candidates than a chunk or a row has, and both chunk lengths
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,W,V,n", [(1, 1, 1, 1), (2, 3, 1, 3), (1, 4, 7, 8), (3, 2, 63, 64), (1, 1, 2048, 8), (2, 4, 2049, 8), (2, 5, 5003, 10), (1, 32, 700, 64),
                                     (1, 1, 40001, 64), (3, 1, 8191, 2), (40, 8, 257, 16)])
def test_candidates(device, dtype, B, W, V, n):
    g = torch.Generator().manual_seed(V + n)
    logits = (torch.randn(B, W, V, generator=g) * 3).to(dtype).to(device)
    scores = (-torch.rand(B, W, generator=g) * 20).to(device)
    _check_select(logits, scores, n)
    _check_select(logits.reshape(B * W, V), scores, n)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [301, 4099, 9000])
def test_candidates_of_masked_rows(device, dtype, V):
    g = torch.Generator().manual_seed(V)
    B, W, n = 9, 4, 12
    low = torch.finfo(dtype).min
    x = (torch.randn(B, W, V, generator=g) * 2).to(dtype)
    scores = -torch.rand(B, W, generator=g) * 5
    x[0, :, 5:] = -INF                        # fewer than n a beam, more than n a group
    x[1, :, 2:] = -INF                        # fewer than n a group: the rest are -inf from the lowest index on
    x[2, 1:] = -INF                           # beams without a token
    x[3] = -INF                               # a group without one
    x[4, :, 3:] = low                         # the type's lowest value: ties, from the lowest index on
    x[5] = 0.0                                # all equal
    x[5, 2, V // 2] = -0.0                    # which is equal too
    x[6, 0, 7], x[6, 1, V - 1] = math.nan, INF        # beams that are left out
    scores[7, 1:] = -INF                      # the first step: one beam that counts
    scores[8, 0], scores[8, 2] = math.nan, -INF
    _check_select(x.to(device), scores.to(device), n)


@pytest.mark.parametrize("device", DEVICES)
def test_candidates_of_equal_beams_and_equal_logits(device):
    g = torch.Generator().manual_seed(5)
    row = torch.randn(6000, generator=g).bfloat16()
    x = row.repeat(2, 4, 1)                   # four equal beams: the lower beam first
    x[1] = torch.randint(0, 3, (4, 6000), generator=g).bfloat16()          # three values: thousands of ties
    _check_select(x.to(device), torch.full((2, 4), -1.5, device=device), 8)
    _check_select(x.to(device), torch.tensor([[-1.5, -1.5, -2.0, -1.5]] * 2, device=device), 64)


# rows that start at different places of 16 bytes: what they add up to does not depend on it
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V,n", [(301, 8), (5003, 8), (5003, 64), (30522, 10), (128257, 16)])
def test_candidates_of_equal_beams_at_any_alignment(device, dtype, V, n):
    g = torch.Generator().manual_seed(V)
    B, W = (24, 8) if device == "cuda" else (2, 8)
    for pitch in (V, V + 1, V + 3):
        row = (torch.randn(B, 1, V, generator=g) * 2.5).to(dtype)
        wide = torch.randn(B, W, pitch, generator=g).to(dtype)
        wide[:, :, pitch - V:] = row
        x = wide.to(device)[:, :, pitch - V:]
        scores, beams, tokens = (t.cpu() for t in bs.beam_select(x, torch.full((B, W), -1.5, device=device), n))
        # the first token of all beams from the lowest on, then the second
        order = torch.sort(row[:, 0].float(), dim=1, descending=True, stable=True)
        for b in range(B):
            values, at = order.values[b].tolist(), order.indices[b].tolist()
            want, i = [], 0
            while len(want) < n:               # tokens of one logit: beam by beam, the lower tokens first
                j = i
                while j < V and values[j] == values[i]:
                    j += 1
                want += [(w, v) for w in range(W) for v in at[i:j]]
                i = j
            assert list(zip(beams[b].tolist(), tokens[b].tolist())) == want[:n], b
            assert len(set(scores[b, :W].tolist())) == 1


@pytest.mark.parametrize("device", DEVICES)
def test_candidates_of_rising_and_large_logits(device):
    x = torch.arange(5000, dtype=torch.float32).flip(0).repeat(1, 2, 1) * 1e-3
    x[0, 1] += 1e4
    _check_select(x.to(device), torch.tensor([[-3.0, -2.0]], device=device), 16)
    big = torch.full((1, 2, 600), -3e38)
    big[0, 0, 10], big[0, 1, 20] = 3e38, 2e38
    _check_select(big.to(device), torch.tensor([[-1.0, -2.0]], device=device), 4)


@pytest.mark.parametrize("device", DEVICES)
def test_candidates_of_strided_and_misaligned_logits(device):
    g = torch.Generator().manual_seed(3)
    for dtype in (torch.float32, torch.bfloat16):
        wide = torch.randn(2 * 3, 5010, generator=g).to(dtype).to(device)
        scores = (-torch.rand(2, 3, generator=g)).to(device)
        for lo, hi in ((0, 5000), (1, 5002), (3, 4100), (7, 5010)):
            _check_select(wide[:, lo:hi], scores, 6)                                     # a padded vocabulary's rows
            _check_select(wide.view(2, 3, -1)[:, :, lo:hi], scores, 6)
        _check_select(wide.view(3, 2, -1).transpose(0, 1), scores, 6)                    # beams not side by side
        _check_select(wide[:, :5000].t().contiguous().t(), scores, 6)                    # tokens not side by side
        _check_select(wide.view(2, 3, -1), scores.t().contiguous().t(), 6)


# pieces of a row with a value a thread in one warp and nothing behind it, and more candidates wanted than that warp has threads
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n", [33, 48, 64])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_more_candidates_than_the_threads_of_a_short_piece(device, dtype, n):
    g = torch.Generator().manual_seed(n)
    per = 16 // dtype.itemsize                # values of 16 bytes
    short = [32 * per - i for i in (0, 1, per - 1)]
    for V in (*short, 31 * per, 33 * per, 512 * per + 32 * per, 12 * 512 * per + 32 * per):
        lo = V - min(V, 32 * per)             # all that is allowed lies in the last piece
        wide = torch.randn(3, V + per, generator=g).to(dtype)
        wide[:, :lo] = -INF
        wide[1, lo:] = 0.0                    # one high value in 16 bytes
        wide[1, lo::per] = 10.0
        for at in range(per if V in short else 1):
            x = wide[:, at:at + V].to(device)
            _check_select(x, torch.zeros(3, 1, device=device), n)
    for W in (17, 32):                        # a first step with rows for all beams
        x = (torch.randn(2, W, 32 * per, generator=g) * 3).to(dtype)
        x[:, 0] = 0.0
        x[:, 0, per - 1::per] = 5.0
        scores = torch.full((2, W), -INF)
        scores[:, 0] = 0.0
        _check_select(x.to(device), scores.to(device), n)


# rows whose first round tells nothing about the others, and rounds with more values than are ranked easily; several rounds a row, one or many
# chunks of it, few and many entries to join
@pytest.mark.gpu
@pytest.mark.parametrize("B,W,V,n", [(2, 4, 40000, 8), (1, 32, 70001, 64), (300, 1, 17001, 3), (150, 2, 60003, 48), (3, 8, 131000, 16), (200, 4, 9001, 8)])
@pytest.mark.parametrize("kind", ["rising", "falling", "few values", "equal", "a stretch is masked", "a stretch is lowest", "few are allowed", "a plateau"])
def test_candidates_of_rows_unlike_a_sample(B, W, V, n, kind):
    g = torch.Generator(device="cuda").manual_seed(V + n)
    dtype = [torch.bfloat16, torch.float32, torch.float16][(V + n) % 3]
    low = torch.finfo(dtype).min
    x = torch.randn(B * W, V, generator=g, device="cuda") * 3
    lo, hi = V // 5, V - V // 9
    if kind in ("rising", "falling"):
        x = x.sort(1, descending=kind == "falling").values
    elif kind == "few values":
        x = torch.randint(0, 5, x.shape, generator=g, device="cuda").float()
    elif kind == "equal":
        x.zero_()
    x = x.to(dtype)
    if kind == "a stretch is masked":
        x[:, lo:hi] = -INF
        x[::3, :hi] = -INF
    elif kind == "a stretch is lowest":
        x[:, :hi] = low
    elif kind == "few are allowed":
        x.masked_fill_(torch.rand(x.shape, generator=g, device="cuda") > 5 / V, low)
    elif kind == "a plateau":
        x[:, lo:hi] = 9.0
    scores = -torch.rand(B, W, generator=g, device="cuda") * 4
    x = x.view(B, W, V)
    total = scores.double()[..., None] + (x.double() - torch.logsumexp(x.double(), -1, keepdim=True))
    want, at = torch.sort(total.flatten(1), dim=1, descending=True, stable=True)
    got, beams, tokens = bs.beam_select(x, scores, n)
    # where scores of two beams are nearer than log-sum-exp is good to (2^-20 as above), either may be first
    far = (want[:, :n] - total.flatten(1).gather(1, beams * V + tokens)).abs() > 2.0 ** -20 + 2.0 ** -50 * want[:, :n].abs()
    assert not bool((far & (want[:, :n] > -INF)).any())
    assert bool((at[:, :n] == beams * V + tokens).float().mean() > 0.99) and all(len(set(r)) == n for r in (beams * V + tokens).tolist())
    fine = want[:, :n].float() > -INF
    assert torch.equal(fine, got > -INF)
    assert bool(((got.double() - want[:, :n]).abs() <= 2.0 ** -20 + 2.0 ** -24 * want[:, :n].abs())[fine].all())


# one beam: its logits decide, so every place is known
@pytest.mark.gpu
@pytest.mark.parametrize("B,V,n", [(2, 40000, 8), (300, 17001, 64), (1, 262147, 64), (200, 9001, 16), (900, 1003, 33)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_candidates_of_one_beam_unlike_a_sample(B, V, n, dtype):
    g = torch.Generator(device="cuda").manual_seed(V + n)
    low, lo, hi = torch.finfo(dtype).min, V // 5, V - V // 9
    x = torch.randn(B, V, generator=g, device="cuda") * 3
    rows = {"rising": x.sort(1).values, "falling": x.sort(1, descending=True).values, "few values": torch.randint(0, 5, x.shape, generator=g, device="cuda").float(),
            "equal": torch.zeros_like(x), "a plateau": x.clone(), "masked": x.clone(), "lowest": x.clone(), "few": x.clone()}
    rows["a plateau"][:, lo:hi] = 9.0
    rows = {k: v.to(dtype) for k, v in rows.items()}
    rows["masked"][:, lo:hi] = -INF
    rows["masked"][::3, :hi] = -INF
    rows["lowest"][:, :hi] = low
    rows["few"].masked_fill_(torch.rand(x.shape, generator=g, device="cuda") > 5 / V, low)
    for kind, logits in rows.items():
        got, beams, tokens = bs.beam_select(logits, torch.full((B, 1), -2.0, device="cuda"), n)
        assert torch.equal(tokens, torch.sort(logits.float(), dim=1, descending=True, stable=True).indices[:, :n]) and not bool(beams.any()), kind
        assert not bool((got == -INF).any()) or kind in ("lowest", "few", "masked"), kind


# The scores are such that the results are near zero: what is left is the error of log-sum-exp.  Exponentials are good to 2^-22; the argument of one d below
# the maximum to half a step of d log2(e), which is 2^-20.5 at 12 and counts by the weight of such terms, at most a half beside the maximum's own (hence
# 2^-21.5); forty additions with the signs of chance to 2^-22.  Together less than 2^-20.
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [500, 5003, 30522, 128256, 262144])
def test_log_sum_exp_of_a_beam(V, dtype):
    g = torch.Generator(device="cuda").manual_seed(V)
    B = min(256, 2 ** 25 // V)
    rows = [torch.randn(B, V, generator=g, device="cuda") * s for s in (0.1, 1.0, 2.5, 6.0)]
    for f in (0.25, 1.0, 4.0):                 # one high value, the others together a part of its weight
        x = (-math.log(V * f) - torch.rand(B, 1, generator=g, device="cuda")).repeat(1, V)
        x[:, V // 3] = 0.0
        rows.append(x)
    for x in rows:
        x = x.to(dtype)
        lse, top = torch.logsumexp(x.double(), -1), x.amax(-1).double()
        scores = (lse - top).float()
        got = bs.beam_select(x, scores[:, None], 1)[0].double()[:, 0]
        assert bool(((got - (scores.double() + (top - lse))).abs() <= 2.0 ** -20).all())


def test_candidates_refused():
    x, s = torch.randn(2, 3, 50), torch.zeros(2, 3)
    for logits, scores, n in ((x, s, 0), (x, s, 65), (x, s, 151), (x, s.double(), 4), (x, s[0], 4), (x[:, :2], s, 4), (x.reshape(-1), s, 4), (x.long(), s, 4),
                              (torch.randn(1, 33, 50), torch.zeros(1, 33), 4), (torch.randn(1, 0, 50), torch.zeros(1, 0), 4),
                              (torch.randn(2, 3, 0), s, 4), (torch.randn(1, 1, 3), torch.zeros(1, 1), 4)):
        with pytest.raises(ValueError):
            bs.beam_select(logits, scores, n)
    empty = bs.beam_select(torch.randn(0, 3, 50), torch.zeros(0, 3), 4)
    assert [tuple(t.shape) for t in empty] == [(0, 4)] * 3


@pytest.mark.gpu
def test_candidates_refused_on_the_gpu():
    x, s = torch.randn(1, 2, 50, device="cuda"), torch.zeros(1, 2, device="cuda")
    for logits, scores in ((x.double(), s), (x, s.cpu()), (x.cpu(), s)):
        with pytest.raises(ValueError):
            bs.beam_select(logits, scores, 4)
    empty = bs.beam_select(x[:0], s[:0], 4)
    assert [tuple(t.shape) for t in empty] == [(0, 4)] * 3


# ---- the books --------------------------------------------------------------------------------------------------------

EOS, PAD = 2, 0


def _fp32(x):
    return torch.tensor(x, dtype=torch.float32).item()


class _Request:
    """One request as lists of tokens: what the tensors have to come to."""

    def __init__(self, W, penalty, early):
        self.W, self.penalty, self.early = W, penalty, early
        self.beams = [(0.0, [])] + [(-INF, [])] * (W - 1)
        self.pool, self.done = [], False

    def step(self, cands):
        """cands: (score, line, token), the best first."""
        if self.done:
            self.beams = [(s, h + [PAD]) for s, h in self.beams]
            return
        n = len(self.beams[0][1]) + 1
        norm = torch.tensor(float(n) ** self.penalty, dtype=torch.float32)
        going = [c for c in cands if c[2] != EOS][:self.W]
        for r, (s, line, token) in enumerate(cands):
            if token == EOS and r < self.W and s > -INF:
                self.pool.append((float(torch.tensor(s, dtype=torch.float32) / norm), self.beams[line][1] + [EOS]))
        self.pool = sorted(self.pool, key=lambda p: -p[0])[:self.W]          # stable: the older first
        lines, seen, late = [None] * self.W, set(), []
        for s, line, token in going:
            child = (s, self.beams[line][1] + [token])
            if line in seen:
                late.append(child)
            else:
                seen.add(line)
                lines[line] = child
        for i in range(self.W):
            if lines[i] is None:
                lines[i] = late.pop(0) if late else (-INF, [PAD] * n)
        self.beams = lines
        if len(self.pool) == self.W:
            best = max(torch.tensor(s, dtype=torch.float32) / norm for s, _ in self.beams)
            self.done = self.early or self.pool[-1][0] >= float(best)

    def finish(self, step):
        found = list(self.pool)
        if not self.done:
            norm = torch.tensor(float(step) ** self.penalty, dtype=torch.float32)
            found += [(float(torch.tensor(s, dtype=torch.float32) / norm), h) for s, h in self.beams if s > -INF]
        return sorted(found, key=lambda p: -p[0])[:self.W]


def _random_candidates(rng, W, N, ends):
    """The best first, distinct (line, token) pairs, at most one that ends a line."""
    pairs = rng.sample([(w, t) for w in range(W) for t in range(3, 3 + 2 * N)], N)
    ending = {}
    out, s = [], -rng.random() * 3
    for r, (line, token) in enumerate(pairs):
        if rng.random() < ends and line not in ending:
            ending[line] = token = EOS
        out.append((_fp32(s), line, token))
        s -= rng.choice([0.0, rng.random()])          # equal scores too
    return out


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("W,steps,penalty,early,ends", [(1, 9, 1.0, False, 0.3), (2, 17, 0.7, True, 0.2), (3, 33, -0.5, False, 0.15), (4, 40, 1.0, False, 0.1),
                                                        (8, 100, 2.0, False, 0.02), (17, 70, 0.0, True, 0.05), (32, 31, 1.0, False, 0.03)])
def test_books_and_sequences(device, W, steps, penalty, early, ends):
    B, N = 5, min(64, 2 * W)
    rng = random.Random(W * 100 + steps)
    kw = dict(eos_token_id=EOS, pad_token_id=PAD, length_penalty=penalty)
    requests = [_Request(W, penalty, early) for _ in range(B)]
    pool, history = bs.new_beam_pool(B, W, device), bs.new_beam_history(steps, B, W, device)
    scores = torch.tensor([[0.0] + [-INF] * (W - 1)] * B, device=device)
    for t in range(steps):
        cands = [_random_candidates(rng, 1 if t == 0 else W, N, ends * (b + 1) / 2) for b in range(B)]
        cols = [torch.tensor([[c[i] for c in row] for row in cands], device=device) for i in range(3)]
        before = [p.clone() for p in pool]
        scores, tokens, parents, new = bs.beam_advance((cols[0].float(), cols[1], cols[2]), scores, pool, history, t, early_stopping=early, **kw)
        assert all(torch.equal(a, b) for a, b in zip(before, pool))          # what goes in stays
        pool = new
        for r, c in zip(requests, cands):
            r.step(c)
        assert scores.tolist() == [[s for s, _ in r.beams] for r in requests]
        assert tokens.tolist() == [[h[-1] for _, h in r.beams] for r in requests]
        assert pool.done.tolist() == [r.done for r in requests]
        assert pool.scores.tolist() == [[s for s, _ in r.pool] + [-INF] * (W - len(r.pool)) for r in requests]
        assert pool.lengths.tolist() == [[len(h) for _, h in r.pool] + [0] * (W - len(r.pool)) for r in requests]
        p = parents.cpu()
        assert torch.equal(p.gather(1, p), p)          # no line that is read is written
        if t in (0, 1, steps // 2, steps - 1):
            seqs, lengths, best = bs.beam_finish(scores, pool, history, t + 1, **kw)
            want = [r.finish(t + 1) for r in requests]
            assert best.tolist() == [[s for s, _ in w] + [-INF] * (W - len(w)) for w in want]
            assert lengths.tolist() == [[len(h) for _, h in w] + [0] * (W - len(w)) for w in want]
            assert seqs.tolist() == [[h + [PAD] * (t + 1 - len(h)) for _, h in w] + [[PAD] * (t + 1)] * (W - len(w)) for w in want]


@pytest.mark.parametrize("device", DEVICES)
def test_books_with_few_candidates_and_without_an_end(device):
    def run(cands, W, **kw):
        cols = [torch.tensor([[c[i] for c in cands]], device=device) for i in range(3)]
        pool, history = bs.new_beam_pool(1, W, device), bs.new_beam_history(2, 1, W, device)
        return bs.beam_advance((cols[0].float(), cols[1], cols[2]), torch.zeros(1, W, device=device), pool, history, 1, **kw), history

    (scores, tokens, parents, pool), history = run([(-1.0, 2, 9), (-2.0, 2, EOS), (-3.0, 2, 8)], 4, eos_token_id=EOS, pad_token_id=7)
    assert scores.tolist() == [[-3.0, -INF, -1.0, -INF]] and tokens.tolist() == [[8, 7, 9, 7]] and parents.tolist() == [[2, 1, 2, 3]]
    assert pool.scores.tolist() == [[-1.0, -INF, -INF, -INF]] and pool.slots.tolist() == [[2, 0, 0, 0]] and pool.lengths.tolist() == [[2, 0, 0, 0]]
    assert history.tokens[1].tolist() == [[8, 7, 9, 7]] and history.tokens[0].tolist() == [[0] * 4]
    (scores, tokens, parents, pool), _ = run([(-1.0, 0, 9), (-2.0, 1, EOS), (-INF, 1, 8)], 2)
    assert tokens.tolist() == [[9, EOS]] and not bool(pool.done) and pool.scores.tolist() == [[-INF, -INF]]
    (_, _, _, pool), _ = run([(-1.0, 0, EOS), (-INF, 1, EOS), (-2.0, 1, 5)], 2, eos_token_id=EOS)          # a candidate of -inf does not end
    assert pool.scores.tolist() == [[-0.5, -INF]]


def test_books_refused():
    B, W, N = 2, 3, 6
    good = dict(c=(torch.zeros(B, N), torch.zeros(B, N, dtype=torch.int64), torch.zeros(B, N, dtype=torch.int64)), s=torch.zeros(B, W),
                p=bs.new_beam_pool(B, W), h=bs.new_beam_history(4, B, W), t=1)

    def call(kw=None, **over):
        a = {**good, **over}
        return bs.beam_advance(a["c"], a["s"], a["p"], a["h"], a["t"], **(kw or {}))

    call()
    for over in (dict(t=4), dict(t=-1), dict(s=torch.zeros(B, 4)), dict(s=torch.zeros(B, W).double()), dict(p=bs.new_beam_pool(B, 4)),
                 dict(h=bs.new_beam_history(4, 1, W)), dict(c=(good["c"][0].double(), *good["c"][1:])), dict(c=(good["c"][0][:, :4], *good["c"][1:])),
                 dict(c=tuple(torch.zeros(B, 65, dtype=t.dtype) for t in good["c"])), dict(kw=dict(length_penalty=1e4)), dict(kw=dict(eos_token_id=2 ** 31)),
                 dict(kw=dict(pad_token_id=2 ** 40))):
        with pytest.raises(ValueError):
            call(**over)
    for step in (0, 5):
        with pytest.raises(ValueError):
            bs.beam_finish(good["s"], good["p"], good["h"], step)
    with pytest.raises(ValueError):
        bs.beam_finish(good["s"], bs.new_beam_pool(B, 4), good["h"], 1)


@pytest.mark.parametrize("device", DEVICES)
def test_sequences_of_a_long_history_with_any_parents(device):
    g = torch.Generator().manual_seed(11)
    for B, W, T in ((1, 1, 1), (2, 5, 515), (3, 32, 1030)):
        history = bs.BeamHistory(torch.randint(3, 999, (T + 3, B, W), generator=g).int(), torch.randint(0, W, (T + 3, B, W), generator=g).int())
        held = torch.arange(W) < W // 2
        pool = bs.BeamPool(torch.where(held, -torch.arange(W).float() * 2, -INF).repeat(B, 1), torch.where(held, torch.randint(1, T + 1, (B, W), generator=g), 0).int(),
                           torch.where(held, torch.randint(0, W, (B, W), generator=g), 0).int(), torch.zeros(B, dtype=torch.bool))
        scores = -(torch.arange(W).float() * 2 + 1).repeat(B, 1) * T
        want, lens = [], []
        for b in range(B):
            found = [(float(pool.scores[b, i]), int(pool.lengths[b, i]) - 2, int(pool.slots[b, i]), [EOS]) for i in range(W) if held[i]]
            found += [(float(scores[b, w] / T), T - 1, w, []) for w in range(W)]
            rows = []
            for _, t, line, tail in sorted(found, key=lambda f: -f[0])[:W]:
                seq = list(tail)
                while t >= 0:
                    seq.insert(0, int(history.tokens[t, b, line]))
                    line, t = int(history.parents[t, b, line]), t - 1
                rows.append(seq)
            want.append([r + [PAD] * (T - len(r)) for r in rows])
            lens.append([len(r) for r in rows])
        put = lambda x: type(x)(*[t.to(device) for t in x])          # noqa: E731
        tokens, lengths, _ = bs.beam_finish(scores.to(device), put(pool), put(history), T, eos_token_id=EOS, pad_token_id=PAD)
        assert lengths.tolist() == lens and tokens.tolist() == want


# one CTA a request and clusters of them, spans whose tokens do not fit shared memory, and spans that do not fit at all
@pytest.mark.gpu
@pytest.mark.parametrize("B,W,T", [(200, 3, 301), (40, 8, 1999), (1, 32, 5603), (1, 32, 27001), (3, 1, 4097), (1, 7, 127), (2, 9, 128), (1, 2, 16)])
def test_sequences_of_many_steps(B, W, T):
    g = torch.Generator().manual_seed(T)
    history = bs.BeamHistory(torch.randint(3, 9999, (T, B, W), generator=g).int(), torch.randint(0, W, (T, B, W), generator=g).int())
    held = torch.rand(B, W, generator=g).sort(1, descending=True).values < 0.5
    held = held.flip(1)
    scores, running = (-torch.rand(2, B, W, generator=g).sort(-1).values).unbind(0)
    pool = bs.BeamPool(torch.where(held, scores, -INF), torch.where(held, torch.randint(1, T + 1, (B, W), generator=g), 0).int(),
                       torch.where(held, torch.randint(0, W, (B, W), generator=g), 0).int(), torch.rand(B, generator=g) < 0.3)
    kw = dict(eos_token_id=EOS, pad_token_id=PAD, length_penalty=0.5)
    want = bs.beam_finish(running * T ** 0.5, pool, history, T, **kw)
    put = lambda x: type(x)(*[t.cuda() for t in x])          # noqa: E731
    got = bs.beam_finish((running * T ** 0.5).cuda(), put(pool), put(history), T, **kw)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))


def test_a_cluster_waits_for_its_blocks_before_it_stores_into_them():
    """Another block's shared memory may be written once that block is known to run."""
    source = (Path(bs.__file__).parents[2] / "csrc" / "beam_search.cu").read_text()
    body = source[source.index("beam_finish_kernel("):source.index("finish_span(")]
    arrive, wait, store = (body.index(s) for s in ("cluster_arrive()", "cluster_wait()", "store_of_rank("))
    assert arrive < body.index("hist_parent[at]") < wait < store          # said at the start, waited for where it is needed
    assert body.rindex("cluster_arrive()") > body.rindex("store_of_rank(")


# clusters of two, four and eight blocks whose last has the fewest steps, launches behind each other
@pytest.mark.gpu
@pytest.mark.parametrize("B,W,T", [(148, 3, 129), (74, 5, 257), (37, 8, 513), (1, 32, 1025), (5, 1, 1031), (20, 4, 700)])
def test_sequences_of_uneven_spans(B, W, T):
    g = torch.Generator().manual_seed(T)
    history = bs.BeamHistory(torch.randint(3, 9999, (T, B, W), generator=g).int(), torch.randint(0, W, (T, B, W), generator=g).int())
    pool, running = bs.new_beam_pool(B, W), -torch.rand(B, W, generator=g).sort(-1).values
    want = bs.beam_finish(running, pool, history, T, length_penalty=0.0)
    put = lambda x: type(x)(*[t.cuda() for t in x])          # noqa: E731
    args = running.cuda(), put(pool), put(history), T
    for got in [bs.beam_finish(*args, length_penalty=0.0) for _ in range(20)]:
        assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))


# ---- lines and pages --------------------------------------------------------------------------------------------------

def _values(shape, dtype, g, device):
    n = math.prod(shape)
    return torch.randint(-120, 120, (max(n, 1),), generator=g)[:n].reshape(shape).to(dtype).to(device)


def _reordered(t, parents, lo, hi):
    out = t.clone()
    W = len(parents[0])
    for b, p in enumerate(parents):
        for w, x in enumerate(p):
            if 0 <= x < W:
                if t.dim() == 4 and lo is not None:
                    a, e = max(lo[b], 0), min(hi[b], t.shape[2])
                    if e > a:
                        out[b * W + w, :, a:e] = t[b * W + x, :, a:e]
                else:
                    out[b * W + w] = t[b * W + x]
    return out


MAPS = [[0], [0, 0], [1, 0], [2, 0, 1], [0, 0, 0, 0], [1, 2, 3, 0], [3, 3, 0, 1], [1, 0, 3, 2], [0, 1, 2, 3], [-1, 9, 0, 0], [4, 0, 0, 2, 3, 6, 5, 6]]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("p", MAPS + [32], ids=str)
def test_lines_continue_any_lines(device, p):
    g = torch.Generator().manual_seed(len(p) if isinstance(p, list) else p)
    W = len(p) if isinstance(p, list) else p
    B = 3
    parents = [p, list(range(W)), torch.randint(0, W, (W,), generator=g).tolist()] if isinstance(p, list) else [
        torch.randperm(W, generator=g).tolist(), torch.randint(0, W, (W,), generator=g).tolist(), [W - 1] * W]
    # heads and sizes that differ, odd ones, one byte a value; more lines than the groups have
    cache = [_values(s, d, g, device) for s, d in (((B * W + 2, 2, 9, 8), torch.bfloat16), ((B * W, 2, 9, 8), torch.bfloat16), ((B * W, 3, 9, 5), torch.float32),
                                                   ((B * W, 1, 9, 3), torch.float16), ((B * W, 2, 9, 3), torch.int8))]
    states = [_values((B * W, 4, 5), torch.float32, g, device), _values((B * W + 1, 3), torch.int8, g, device), _values((B * W,), torch.float32, g, device)]
    ids = torch.tensor(parents, device=device)
    for lo, hi in ((None, None), ([0, 2, 9], [9, 5, 9]), ([-3, 4, 0], [1, 4, 99]), ([5, 0, 8], [4, 0, 9])):
        want = [_reordered(t, parents, lo, hi) for t in cache] + [_reordered(t, parents, None, None) for t in states]
        got = [t.clone() for t in cache], [t.clone() for t in states]
        kw = {} if lo is None else dict(start=torch.tensor(lo, device=device), end=torch.tensor(hi, device=device, dtype=torch.int32))
        kl.reorder_lines_(got[0], ids, states=got[1], **kw)
        assert all(torch.equal(a, b) for a, b in zip(got[0] + got[1], want))
    got = [t.clone() for t in cache]
    only = torch.tensor([3, 8, 1], device=device)
    kl.reorder_lines_(got, ids.int(), only)
    assert all(torch.equal(a, _reordered(t, parents, only.tolist(), [9] * 3)) for a, t in zip(got, cache))


@pytest.mark.parametrize("device", DEVICES)
def test_lines_of_strided_caches_and_many_tensors(device):
    g = torch.Generator().manual_seed(0)
    parents = [[1, 1, 0], [2, 0, 1]]
    ids = torch.tensor(parents, device=device)
    both = _values((6, 2, 4, 16, 8), torch.bfloat16, g, device)          # keys and values side by side in a line
    want = torch.stack([_reordered(both[:, i], parents, [3, 0], [10, 16]) for i in range(2)], dim=1)
    handle = kl.CacheTensors([both[:, 0], both[:, 1]])
    kl.reorder_lines_(handle, ids, torch.tensor([3, 0], device=device), torch.tensor([10, 16], device=device))
    assert torch.equal(both, want)
    many = [_values((6, 1, 2, 4), torch.float32, g, device) for _ in range(300)]          # more than a launch takes
    want = [_reordered(t, parents, None, None) for t in many]
    handle = kl.CacheTensors(many[1:])
    kl.reorder_lines_(handle, ids)
    kl.reorder_lines_([many[0]], ids)
    assert all(torch.equal(a, b) for a, b in zip(many, want))
    moved = many[5].clone()
    many[5].data = moved          # a tensor that is given other storage is still the cache's
    want = _reordered(moved, parents, None, None)
    kl.reorder_lines_(handle, ids)
    assert torch.equal(many[5], want)
    kl.reorder_lines_(handle, ids[:0])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("page", [1, 4, 7])
def test_lines_in_pages(device, page):
    g = torch.Generator().manual_seed(page)
    B, W, per, H, D = 2, 4, 5, 3, 8
    S = page * per
    pages = torch.randperm(B * W * per + 3, generator=g)[:B * W * per].reshape(B * W, per).int()
    pool = [_values((B * W * per + 3, H, page, D), torch.bfloat16, g, device) for _ in range(2)]
    parents = [[3, 0, 0, 2], [1, 2, 0, 0]]
    lo, hi = [1, page], [S - 1, S]

    def lines(t):
        return t[pages.long()].permute(0, 2, 1, 3, 4).reshape(B * W, H, S, D)

    want = [_reordered(lines(t.cpu()), parents, lo, hi) for t in pool]
    others = [i for i in range(B * W * per + 3) if i not in set(pages.flatten().tolist())]
    spare = [t[others].clone() for t in pool]
    kl.reorder_lines_(pool, torch.tensor(parents, device=device), torch.tensor(lo, device=device), torch.tensor(hi, device=device),
                      block_table=pages.to(device), page_size=page)
    assert all(torch.equal(lines(t.cpu()), w) and torch.equal(t[others], s) for t, w, s in zip(pool, want, spare))
    bad = pages.clone()
    bad[1, 2], bad[0, 3] = -1, 10 ** 6          # pages that there are not: passed by
    kl.reorder_lines_(pool, torch.tensor([[0, 0, 1, 0], [0, 1, 2, 3]], device=device), block_table=bad.to(device), page_size=page)


@pytest.mark.parametrize("device", DEVICES)
def test_copies_of_pages(device):
    g = torch.Generator().manual_seed(7)
    pool = [_values(s, d, g, device) for s, d in (((40, 2, 6, 8), torch.bfloat16), ((40, 2, 6, 8), torch.bfloat16), ((40, 3, 6, 5), torch.float32),
                                                  ((41, 1, 6, 3), torch.int8))]
    some = torch.randperm(40, generator=g).tolist()
    for n, rows in ((1, None), (20, None), (13, [0, 1, 2, 3, 4, 5, 6, 7, -1, 2, 5, 6, 1])):
        src, dst = some[:n], some[20:20 + n]
        want = [t.clone() for t in pool]
        for t in want:
            for i, (a, b) in enumerate(zip(src, dst)):
                k = t.shape[2] if rows is None else max(0, min(rows[i], t.shape[2]))
                t[b, :, :k] = t[a, :, :k]
        for form in (list, lambda x: torch.tensor(x, device=device), lambda x: torch.tensor(x, device=device, dtype=torch.int32)):
            got = [t.clone() for t in pool]
            kl.copy_pages_(got, form(src), form(dst), rows=None if rows is None else form(rows))
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = [t.clone() for t in pool]
    kl.copy_pages_(got, torch.tensor([3, -1, 5, 10 ** 9], device=device), torch.tensor([3, 4, 40 + 1, 6], device=device))          # pairs that are passed by
    kl.copy_pages_(got, [], [])
    assert all(torch.equal(a, b) for a, b in zip(got, pool))


def test_lines_and_pages_refused():
    t = torch.zeros(8, 2, 4, 8)
    ids = torch.zeros(2, 4, dtype=torch.int64)
    for cache, parents, kw in (([t], ids.float(), {}), ([t], ids[0], {}), ([t], torch.zeros(3, 4, dtype=torch.int64), {}), ([t], torch.zeros(1, 33, dtype=torch.int64), {}),
                               ([t], torch.zeros(8, 0, dtype=torch.int64), {}), ([t], ids, dict(start=torch.zeros(3, dtype=torch.int64))),
                               ([t], ids, dict(end=torch.zeros(2))), ([t], ids, dict(states=[torch.zeros(7, 3)])), ([t[..., :4]], ids, {}), ([t[0]], ids, {}),
                               ([t.transpose(2, 3)], ids, {}), ([t, t], ids, {}), ([t[:1].expand(8, 2, 4, 8)], ids, {}), ([], ids, {}),
                               ([t], ids, dict(states=[torch.zeros(8, 3, 4).transpose(1, 2)])),
                               ([t], ids, dict(block_table=torch.zeros(8, 3, dtype=torch.int64), page_size=4)),
                               ([t], ids, dict(block_table=torch.zeros(8, 3, dtype=torch.int32), page_size=5)),
                               ([t], ids, dict(block_table=torch.zeros(7, 3, dtype=torch.int32), page_size=4))):
        with pytest.raises(ValueError):
            kl.reorder_lines_(cache, parents, **kw)
    for src, dst, kw in (([0], [8], {}), ([-1], [2], {}), ([0, 1], [2, 2], {}), ([0, 1], [1, 2], {}), ([0], [1, 2], {}), ([0], [1], dict(rows=[1, 2])),
                         (torch.zeros(1), [3], {}), (torch.zeros(1, 1, dtype=torch.int64), [3], {})):
        with pytest.raises(ValueError):
            kl.copy_pages_([t], src, dst, **kw)


@pytest.mark.gpu
def test_a_search_step_is_captured_and_replayed():
    g = torch.Generator(device="cuda").manual_seed(1)
    B, W, V, T, S = 3, 4, 5003, 12, 24
    logits = torch.empty(B, W, V, device="cuda", dtype=torch.bfloat16)
    scores = torch.empty(B, W, device="cuda")
    cache, state = torch.empty(B * W, 2, S, 8, device="cuda"), torch.empty(B * W, 5, device="cuda")
    start, end = torch.tensor([0, 3, 9], device="cuda"), torch.tensor([S, 9, 9], device="cuda")

    def step():
        cand = bs.beam_select(logits, scores, 2 * W)
        out = bs.beam_advance(cand, scores, pool, history, 3, eos_token_id=EOS)
        kl.reorder_lines_([cache], out[2], start, end, states=[state])
        return cand, out, bs.beam_finish(out[0], out[3], history, 4, eos_token_id=EOS)

    graphs = []
    for _ in range(2):
        pool, history = bs.new_beam_pool(B, W, "cuda"), bs.new_beam_history(T, B, W, "cuda")
        logits.normal_(generator=g), scores.zero_(), cache.normal_(generator=g), state.normal_(generator=g)
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out, pool, history))
    for graph, out, pool, history in graphs * 2:
        logits.normal_(generator=g), scores.copy_(-torch.rand(B, W, generator=g, device="cuda"))
        cache.normal_(generator=g), state.normal_(generator=g)
        saved = cache.clone(), state.clone()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (*out[0], *out[1][:3], *out[1][3], *out[2], cache, state)]
        cache.copy_(saved[0]), state.copy_(saved[1])
        now = step()
        assert all(torch.equal(a, b) for a, b in zip(got, (*now[0], *now[1][:3], *now[1][3], *now[2], cache, state)))


@pytest.mark.gpu
def test_a_search_step_runs_on_the_stream_that_is_current():
    torch.manual_seed(0)
    x, s = torch.randn(2, 4, 30000, device="cuda"), -torch.rand(2, 4, device="cuda")
    cache = torch.randn(8, 2, 64, 64, device="cuda")
    want = bs.beam_select(x, s, 8)
    p = torch.tensor([[1, 0, 0, 2], [3, 3, 3, 3]], device="cuda")
    ref = _reordered(cache, p.tolist(), None, None)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        y = x + 0.0
        got = bs.beam_select(y, s, 8)
        kl.reorder_lines_([cache], p)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(cache, ref)


@pytest.mark.gpu
def test_results_do_not_change_from_call_to_call():
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randint(0, 9, (6, 8, 50000), generator=g, device="cuda").bfloat16()
    s = -torch.rand(6, 8, generator=g, device="cuda")
    first = bs.beam_select(x, s, 32)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, bs.beam_select(x, s, 32)))
