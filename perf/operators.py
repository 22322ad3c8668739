"""What a training step on packed samples is timed on: attention over sequences of different lengths laid end to end, the
balance loss of a mixture's routers with its counts, and dropout whose mask is drawn again instead of kept.

Sizes come from this repository's configurations (Llama 1B / 8B and BERT-large heads, Mixtral's and DBRX's routers, adapters
in front of a layer's width).  ``prepare`` makes inputs from the seed alone; ``run`` with ``own`` false is each operator's
formula in elementary torch operations, with ``own`` true the framework's call; ``exact`` restates the formulas in float64.
"""
import itertools
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SCORES = 1 << 29          # scores that the plain forms hold at a time
FORWARD_PAIRS, BACKWARD_PAIRS = 4, 10      # flops per pair, head and channel


def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def listed():
    return [
        # scoring three short answers with the 1B model: one call of a hundred tokens, where launches count
        {"name": "packed_few_short", "kind": "packed", "heads": 32, "kv_heads": 8, "dim": 64, "tokens": 96, "sequences": 3,
         "spread": 20.0, "mix": 1, "behind": 0, "causal": True, "backward": False},
        # one layer of instruction tuning of the 1B model: two dozen samples fill a row of 8192 tokens
        {"name": "packed_finetune_1b", "kind": "packed", "heads": 32, "kv_heads": 8, "dim": 64, "tokens": 8192,
         "sequences": 24, "spread": 40.0, "mix": 2, "behind": 71, "causal": True, "backward": True},
        # one layer of continued training of the 8B model: a few long documents in 16384 tokens
        {"name": "packed_documents_8b", "kind": "packed", "heads": 32, "kv_heads": 8, "dim": 128, "tokens": 16384,
         "sequences": 4, "spread": 6.0, "mix": 3, "behind": 0, "causal": True, "backward": True},
        # the prompts of a batch in one call, without gradients: the 8B model, one of them is most of 32768 tokens
        {"name": "packed_prompts_8b", "kind": "packed", "heads": 32, "kv_heads": 8, "dim": 128, "tokens": 32768,
         "sequences": 7, "spread": 30.0, "mix": 4, "behind": 0, "causal": True, "backward": False},
        # BERT-large without padding: sentences of up to a few hundred tokens, every token sees its whole sentence
        {"name": "packed_bert_large", "kind": "packed", "heads": 16, "kv_heads": 16, "dim": 64, "tokens": 24576,
         "sequences": 120, "spread": 12.0, "mix": 5, "behind": 301, "causal": False, "backward": True},
        # the router of one layer on a handful of tokens
        {"name": "balance_one_layer", "kind": "balance", "layers": 1, "rows": 130, "experts": 8, "top": 2, "dtype": "fp32",
         "masked": False},
        # all routers of an 8x7B step, padding rows left out
        {"name": "balance_mixtral", "kind": "balance", "layers": 32, "rows": 8192, "experts": 8, "top": 2, "dtype": "bf16",
         "masked": True},
        # all routers of a DBRX step: sixteen experts, four a token
        {"name": "balance_dbrx", "kind": "balance", "layers": 40, "rows": 8192, "experts": 16, "top": 4, "dtype": "fp32",
         "masked": False},
        # fine-grained experts, an odd number of rows
        {"name": "balance_many_experts", "kind": "balance", "layers": 6, "rows": 40007, "experts": 128, "top": 8,
         "dtype": "fp32", "masked": False},
        # in front of an adapter of the 1B model, a few short samples
        {"name": "dropout_adapter_short", "kind": "dropout", "rows": 96, "cols": 2048, "p": 0.05, "dtype": "bf16",
         "residual": False},
        # in front of an adapter of the 8B model, a whole packed row
        {"name": "dropout_adapter_8b", "kind": "dropout", "rows": 8192, "cols": 4096, "p": 0.1, "dtype": "bf16",
         "residual": False},
        # an encoder's residual branch in fp32, a ragged number of tokens
        {"name": "dropout_residual", "kind": "dropout", "rows": 24275, "cols": 1024, "p": 0.1, "dtype": "fp32",
         "residual": True},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _costs(case):
    w = work(case)
    return w["bytes"] / 6.5e12 + w["flops"] / 1.6e15


def draw(rng):
    kind = rng.choice(["packed", "packed", "balance", "dropout"])
    most = max(_costs(c) for c in listed() if c["kind"] == kind)
    while True:
        if kind == "packed":
            heads, kv_heads, dim = rng.choice([(32, 8, 64), (32, 8, 128), (16, 16, 64), (8, 2, 128), (12, 1, 64), (5, 5, 128), (64, 8, 128)])
            tokens = _spread(rng, 33, 32768)
            n = max(1, min(tokens, _spread(rng, 1, 200)))
            case = {"heads": heads, "kv_heads": kv_heads, "dim": dim, "tokens": tokens, "sequences": n,
                    "spread": float(_spread(rng, 1, 60)), "mix": rng.randrange(1 << 30),
                    "behind": rng.choice([0, rng.randrange(0, 1 + tokens // 8)]), "causal": rng.random() < 0.75,
                    "backward": rng.random() < 0.6}
        elif kind == "balance":
            experts = _spread(rng, 2, 384)
            case = {"layers": _spread(rng, 1, 40), "rows": _spread(rng, 1, 16384), "experts": experts,
                    "top": rng.randint(1, min(8, experts)), "dtype": rng.choice(["fp32", "bf16", "fp16"]),
                    "masked": rng.random() < 0.5}
        else:
            case = {"rows": _spread(rng, 1, 32768), "cols": _spread(rng, 8, 16384), "p": rng.choice([0.05, 0.1, 0.5, rng.uniform(0.01, 0.9)]),
                    "dtype": rng.choice(["bf16", "fp16", "fp32"]), "residual": rng.random() < 0.4}
        case["kind"] = kind
        if _costs(case) <= most:
            return case


def lengths(case):
    """The sequences' lengths: ``sequences`` numbers spread over a factor of ``spread``, some of them none, that sum to the
    tokens that are not behind the last sequence."""
    rng = random.Random(case["mix"])
    share = [math.exp(rng.uniform(0.0, math.log(max(case["spread"], 1.0)))) for _ in range(case["sequences"])]
    total = case["tokens"] - case["behind"]
    out = [int(total * s / sum(share)) for s in share]
    out[rng.randrange(len(out))] += total - sum(out)
    return out


def _pairs(case):
    return sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lengths(case))


def work(case):
    if case["kind"] == "packed":
        T, H, G, D = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        per = _pairs(case) * H * D
        if not case["backward"]:
            return {"bytes": 2 * T * D * (2 * H + 2 * G), "flops": FORWARD_PAIRS * per}
        return {"bytes": 2 * T * D * (4 * H + 4 * G), "flops": (FORWARD_PAIRS + BACKWARD_PAIRS) * per}
    size = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "balance":
        n = case["layers"] * case["rows"] * case["experts"]
        return {"bytes": 2 * n * size, "flops": 20 * n}
    n = case["rows"] * case["cols"]
    return {"bytes": n * size * (5 if case["residual"] else 4), "flops": 4 * n}


def prepare(case, seed):
    dev = _device()
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=g, device=dev).to(dtype)

    if case["kind"] == "packed":
        T, H, G, D, back = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["backward"]
        qkv = normal(T, H + 2 * G, D)          # one projection's output: the heads side by side
        ends = torch.tensor([0] + lengths(case)).cumsum(0).to(torch.int32)
        q, k, v = (qkv[:, a:b].detach().requires_grad_(back) for a, b in ((0, H), (H, H + G), (H + G, H + 2 * G)))
        return {"case": case, "q": q, "k": k, "v": v, "ends": ends.to(dev), "lengths": lengths(case),
                "do": normal(T, H, D) if back else None}
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "balance":
        E, R = case["experts"], case["rows"]
        lean = torch.randn(E, generator=g, device=dev)          # some experts are preferred
        logits = [(1.5 * torch.randn(R, E, generator=g, device=dev) + lean).to(dtype).requires_grad_() for _ in range(case["layers"])]
        mask = torch.rand(R, generator=g, device=dev) < 0.85 if case["masked"] else None
        # gradients in fp16 come with a loss scale
        scale = 2.0 ** round(math.log2(case["layers"] * R)) if dtype == torch.float16 else 1.0
        return {"case": case, "logits": logits, "mask": mask, "coef": torch.full((), 0.02 * scale, device=dev)}
    shape = (case["rows"], case["cols"])
    return {"case": case, "x": normal(*shape, dtype=dtype).requires_grad_(), "dy": normal(*shape, dtype=dtype),
            "residual": normal(*shape, dtype=dtype) if case["residual"] else None,
            "seed": random.Random(seed).getrandbits(62), "offset": seed % 1000003}


# ---- the plain forms --------------------------------------------------------------------------------------------------

def _pieces(s):
    """(first row, rows, first key head, key heads) of pieces whose scores fit, from the lengths that a program has."""
    G, per = s["case"]["kv_heads"], s["case"]["heads"] // s["case"]["kv_heads"]
    starts = [0, *itertools.accumulate(s["lengths"])]
    step = [max(1, min(G, SCORES // max(1, per * n * n))) for n in s["lengths"]]
    return [(a, n, g, min(c, G - g)) for a, n, c in zip(starts, s["lengths"], step) if n for g in range(0, G, c)]


def _plain_packed(s):
    case, q, k, v, do = s["case"], s["q"].detach(), s["k"].detach(), s["v"].detach(), s["do"]
    per, scale = case["heads"] // case["kv_heads"], 1.0 / math.sqrt(case["dim"])
    o = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    dq, dk, dv = (torch.zeros(x.shape, dtype=x.dtype, device=x.device) for x in (q, k, v)) if case["backward"] else (None,) * 3

    def heads(x, a, n, h, count):              # [kv heads, rows per kv head and query head, D] in fp32
        return x[a:a + n, h:h + count].float().transpose(0, 1)

    for a, n, g, c in _pieces(s):
        qf = heads(q, a, n, g * per, c * per).reshape(c, per * n, -1)
        kf, vf = heads(k, a, n, g, c), heads(v, a, n, g, c)
        p = qf @ kf.transpose(1, 2) * scale
        if case["causal"]:
            p.view(c, per, n, n).masked_fill_(torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1), -math.inf)
        p = torch.exp(p - p.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        of = p @ vf
        o[a:a + n, g * per:(g + c) * per] = of.view(c * per, n, -1).transpose(0, 1).to(o.dtype)
        if case["backward"]:
            df = heads(do, a, n, g * per, c * per).reshape(c, per * n, -1)
            dv[a:a + n, g:g + c] = (p.transpose(1, 2) @ df).transpose(0, 1).to(dv.dtype)
            ds = p * (df @ vf.transpose(1, 2) - (df * of).sum(-1, keepdim=True)) * scale
            dq[a:a + n, g * per:(g + c) * per] = (ds @ kf).view(c * per, n, -1).transpose(0, 1).to(dq.dtype)
            dk[a:a + n, g:g + c] = (ds.transpose(1, 2) @ qf).transpose(0, 1).to(dk.dtype)
    return {"o": o, "dq": dq, "dk": dk, "dv": dv} if case["backward"] else {"o": o}


def _plain_balance(s):
    E, k = s["case"]["experts"], s["case"]["top"]
    x = torch.cat([t.detach() for t in s["logits"]]).float()
    rows = s["mask"].repeat(len(s["logits"])) if s["mask"] is not None else torch.ones(x.shape[0], dtype=torch.bool, device=x.device)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True) * rows[:, None]
    chosen = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :k]          # ties: the lowest expert
    counts = ((chosen[:, :, None] == torch.arange(E, device=x.device)) & rows[:, None, None]).sum((0, 1))
    n = rows.sum().clamp(min=1).float()
    f = counts.float() / n
    loss = (f * (p.sum(0, dtype=torch.float64).float() / n)).sum() * (E / k)
    dx = p * (f - (p * f).sum(-1, keepdim=True)) * (s["coef"] * (E / k) / n)
    dx = dx.to(s["logits"][0].dtype)
    return {"loss": loss, "counts": counts, "dlogits": list(dx.split(s["case"]["rows"]))}


def _words(n, seed, offset, device):
    """The first ``n`` words of Philox4x32-7 under the key ``seed``, four to a counter (element // 4, offset)."""
    low = 0xFFFFFFFF
    i = torch.arange((n + 3) // 4, dtype=torch.int64, device=device)
    c = [i & low, i >> 32, torch.full_like(i, offset & low), torch.full_like(i, offset >> 32)]
    key = (seed & low, seed >> 32)
    for r in range(7):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57          # products of 64 bits, which may wrap into the sign
        c = [(b >> 32 & low) ^ c[1] ^ (key[0] + r * 0x9E3779B9 & low), b & low, (a >> 32 & low) ^ c[3] ^ (key[1] + r * 0xBB67AE85 & low), a & low]
    return torch.stack(c, dim=1).view(-1)[:n]


def _plain_dropout(s):
    x, p = s["x"].detach(), s["case"]["p"]
    keep = (_words(x.numel(), s["seed"], s["offset"], x.device) >= int(p * 2 ** 32)).view(x.shape)
    scale = 1.0 / (1.0 - p)
    y = torch.where(keep, x.float() * scale, 0.0)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"y": y.to(x.dtype), "dx": torch.where(keep, s["dy"].float() * scale, 0.0).to(x.dtype)}


# ---- the framework's calls --------------------------------------------------------------------------------------------

def _own_packed(s):
    from neuronx_distributed_llama3_2_b200.ops.attention import flash_attn_packed_func

    o = flash_attn_packed_func(s["q"], s["k"], s["v"], s["ends"], causal=s["case"]["causal"])
    if not s["case"]["backward"]:
        return {"o": o}
    dq, dk, dv = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])
    return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}


def _own_balance(s):
    from neuronx_distributed_llama3_2_b200.modules.moe import load_balancing_loss_func

    loss, counts = load_balancing_loss_func(s["logits"], s["case"]["experts"], s["case"]["top"], mask=s["mask"], return_counts=True)
    return {"loss": loss.detach(), "counts": counts, "dlogits": list(torch.autograd.grad(loss, s["logits"], s["coef"]))}


def _own_dropout(s):
    from neuronx_distributed_llama3_2_b200.ops.dropout import dropout

    y = dropout(s["x"], s["case"]["p"], s["seed"], s["offset"], residual=s["residual"])
    return {"y": y.detach(), "dx": torch.autograd.grad(y, s["x"], s["dy"])[0]}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"packed": _own_packed, "balance": _own_balance, "dropout": _own_dropout}[kind](state)
    return {"packed": _plain_packed, "balance": _plain_balance, "dropout": _plain_dropout}[kind](state)


# ---- in 64 bits -------------------------------------------------------------------------------------------------------

def _exact_packed(case, s):
    """Query rows in blocks, one head at a time, from log-sum-exp."""
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    if case["backward"] and _pairs(case) * H * D > 1.5e12 or _pairs(case) * H * D > 4e12 or H * case["sequences"] > 8000:
        return None
    q, k, v = (s[x].detach().double() for x in "qkv")
    do = s["do"].double() if case["backward"] else None
    o, dq, dk, dv = (torch.zeros_like(x) for x in (q, q, k, v))
    begin = 0
    for n in lengths(case):
        for h in range(H if n else 0):
            g = h * G // H
            rows = slice(begin, begin + n)
            kk, vv = k[rows, g], v[rows, g]
            for at in range(0, n, 4096):
                end = min(n, at + 4096)
                seen = end if case["causal"] else n
                block = slice(begin + at, begin + end)
                score = torch.einsum("id,jd->ij", q[block, h], kk[:seen]) / math.sqrt(D)
                if case["causal"]:
                    i, j = torch.arange(at, end, device=q.device), torch.arange(seen, device=q.device)
                    score = torch.where(j[None] <= i[:, None], score, -math.inf)
                weight = torch.exp(score - torch.logsumexp(score, 1, keepdim=True))
                o[block, h] = torch.einsum("ij,jd->id", weight, vv[:seen])
                if case["backward"]:
                    dv[begin:begin + seen, g] += torch.einsum("ij,id->jd", weight, do[block, h])
                    back = torch.einsum("id,jd->ij", do[block, h], vv[:seen])
                    back = weight * (back - (weight * back).sum(1, keepdim=True)) / math.sqrt(D)
                    dq[block, h] = torch.einsum("ij,jd->id", back, kk[:seen])
                    dk[begin:begin + seen, g] += torch.einsum("ij,id->jd", back, q[block, h])
        begin += n
    return {"o": o, "dq": dq, "dk": dk, "dv": dv} if case["backward"] else {"o": o}


def _exact_balance(case, s):
    E, k = case["experts"], case["top"]
    keep = s["mask"].double() if s["mask"] is not None else torch.ones(case["rows"], dtype=torch.float64, device=s["coef"].device)
    n = max(1.0, float(keep.sum()) * case["layers"])
    soft = [torch.softmax(t.detach().double(), -1) for t in s["logits"]]
    hits = torch.zeros(E, dtype=torch.float64, device=keep.device)
    for t in s["logits"]:
        left = t.detach().double()
        for _ in range(k):
            best = left.argmax(-1)          # ties: the lowest expert
            best = (left == left.gather(1, best[:, None])).int().argmax(-1)
            hits.index_add_(0, best, keep)
            left = left.scatter(1, best[:, None], -math.inf)
    mean = sum((p * keep[:, None]).sum(0) for p in soft) / n
    share = hits / n
    loss = E / k * torch.dot(share, mean)
    grads = [float(s["coef"]) * E / (k * n) * p * keep[:, None] * (share - (p @ share)[:, None]) for p in soft]
    return {"loss": loss, "counts": None, "dlogits": grads}


def _exact_dropout(case, s):
    """The generator by products of 16-bit halves; the values in float64."""
    x, p = s["x"].detach(), case["p"]
    half = 0xFFFF

    def product(m, c):          # (high word, low word) of m * c
        m1, m0, c1, c0 = m >> 16, m & half, c >> 16, c & half
        mid = m1 * c0 + (m0 * c0 >> 16)
        cross = m0 * c1 + (mid & half)
        return m1 * c1 + (mid >> 16) + (cross >> 16), (cross & half) << 16 | m0 * c0 & half

    n = x.numel()
    at = torch.arange(-(-n // 4), device=x.device)
    a, b, c, d = at % 2 ** 32, at // 2 ** 32, torch.zeros_like(at) + s["offset"] % 2 ** 32, torch.zeros_like(at) + s["offset"] // 2 ** 32
    k0, k1 = s["seed"] % 2 ** 32, s["seed"] // 2 ** 32
    for _ in range(7):
        (h0, l0), (h1, l1) = product(0xD2511F53, a), product(0xCD9E8D57, c)
        a, b, c, d = h1 ^ b ^ k0, l1, h0 ^ d ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) % 2 ** 32, (k1 + 0xBB67AE85) % 2 ** 32
    drop = torch.stack([a, b, c, d], -1).flatten()[:n].view(x.shape) < math.floor(p * 2.0 ** 32)
    y = x.double() / (1.0 - p)
    y = y.masked_fill(drop, 0.0)
    if s["residual"] is not None:
        y = y + s["residual"].double()
    return {"y": y, "dx": (s["dy"].double() / (1.0 - p)).masked_fill(drop, 0.0)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"packed": _exact_packed, "balance": _exact_balance, "dropout": _exact_dropout}[case["kind"]](case, s)
