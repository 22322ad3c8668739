"""The load-balancing loss, its counts and its gradient against float64."""
import math

import pytest
import torch

from neuronx_distributed_llama3_2_b200.modules.moe import load_balancing_loss_func

BF16, FP16, FP32 = 2.0 ** -8, 2.0 ** -11, 2.0 ** -24


def oracle(logits, E, k, mask=None, coef=1.0):
    x = torch.cat([t.detach().reshape(-1, E) for t in logits]).double()
    keep = torch.ones(x.shape[0], dtype=torch.bool, device=x.device) if mask is None else mask.reshape(-1).bool().repeat(len(logits))
    p = torch.softmax(x, -1)[keep]
    counts = torch.zeros(E, dtype=torch.int64, device=x.device)
    left = torch.where(torch.isnan(x), math.inf, x)[keep]
    for _ in range(k):
        best = (left == left.amax(-1, keepdim=True)).int().argmax(-1)
        counts += torch.bincount(best, minlength=E)
        left = left.scatter(1, best[:, None], float("-inf"))
    n = max(1, int(keep.sum()))
    f, P = counts.double() / n, p.sum(0) / n
    dx = torch.zeros_like(x)
    dx[keep] = coef * E / (k * n) * p * (f - (p * f).sum(-1, keepdim=True))
    return E / k * (f * P).sum(), counts, dx


def _logits(layers, rows, E, dtype, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed + E)
    lean = torch.randn(E, generator=g, device=device)
    return [(1.5 * torch.randn(rows, E, generator=g, device=device) + lean).to(dtype) for _ in range(layers)]


def _check(logits, E, k, mask, coef=1.0):
    leaves = [t.detach().requires_grad_() for t in logits]
    loss, counts = load_balancing_loss_func(leaves, E, k, mask=mask, return_counts=True)
    assert loss.dtype == torch.float32 and counts.dtype == torch.int64 and not counts.requires_grad
    grads = torch.autograd.grad(loss, leaves, torch.full((), coef, device=loss.device))
    want_loss, want_counts, want = oracle(logits, E, k, mask, coef)
    assert torch.equal(counts, want_counts)
    # probabilities: an exponential, a sum of E terms and a product, 2^-24 each; the loss also sums over the rows in fp32, a few hundred
    # a thread
    assert abs(loss.double() - want_loss) <= FP32 * (8 + E / 8 + 256) * want_loss
    got = torch.cat([x.reshape(-1, E) for x in grads]).double()
    step = {torch.float32: 0.0, torch.bfloat16: BF16, torch.float16: FP16}[logits[0].dtype]
    # f - sum p f loses what the two have in common: relative to the larger of them, not to their difference
    top = want_counts.max().double() / max(1, int(want_counts.sum()) // k)
    x = torch.cat([t.reshape(-1, E) for t in logits]).double()
    scale = abs(coef) * E / k / max(1, int(want_counts.sum()) // k) * torch.softmax(x, -1) * top
    tiny = 2.0 ** -25 if logits[0].dtype == torch.float16 else 1e-38          # half of fp16's smallest step
    assert ((got - want).abs() <= step * want.abs() + FP32 * (24 + E / 4) * scale * 4 + tiny).all()
    return loss, counts, grads


@pytest.mark.parametrize("E,k", [(1, 1), (2, 1), (5, 5), (8, 2), (16, 4)])
@pytest.mark.parametrize("masked", [False, True])
def test_torch_path(E, k, masked):
    logits = _logits(3, 17, E, torch.float32, "cpu")
    mask = (torch.arange(17) % 3 > 0) if masked else None
    _check(logits, E, k, mask)


def test_gradient_is_a_difference():
    logits = [t.double() for t in _logits(2, 7, 5, torch.float64, "cpu")]
    g = torch.Generator().manual_seed(3)
    mask = torch.tensor([1, 1, 0, 1, 0, 1, 1])
    d = [torch.randn(7, 5, generator=g, dtype=torch.float64) for _ in logits]
    _, counts, dx = oracle(logits, 5, 2, mask)
    ahead, back = ([t + s * 1e-6 * e for t, e in zip(logits, d)] for s in (1, -1))
    assert torch.equal(oracle(ahead, 5, 2, mask)[1], counts) and torch.equal(oracle(back, 5, 2, mask)[1], counts)
    slope = (oracle(ahead, 5, 2, mask)[0] - oracle(back, 5, 2, mask)[0]) / 2e-6
    assert abs(slope - (dx * torch.cat(d)).sum()) <= 1e-8          # central difference: 1e-12, and 1e-16 / 1e-6 of rounding


def test_no_rows_and_refusals():
    x = torch.randn(4, 8, requires_grad=True)
    loss, counts = load_balancing_loss_func([x, None], 8, 2, mask=torch.zeros(4), return_counts=True)
    assert loss.item() == 0.0 and not counts.any() and not torch.autograd.grad(loss, x)[0].any()
    for bad in (dict(router_logits=[], num_experts=8, top_k=2), dict(router_logits=x, num_experts=8, top_k=9),
                dict(router_logits=x, num_experts=8, top_k=0), dict(router_logits=x, num_experts=5, top_k=2),
                dict(router_logits=[x, x[:3]], num_experts=8, top_k=2, mask=torch.ones(4))):
        with pytest.raises(ValueError):
            load_balancing_loss_func(**bad)


@pytest.mark.gpu
@pytest.mark.parametrize("E,k", [(1, 1), (2, 1), (3, 2), (8, 2), (8, 8), (9, 3), (16, 4), (31, 6), (64, 8), (100, 7), (128, 8), (129, 2),
                                 (256, 8), (300, 4), (512, 10), (1000, 3), (1024, 16)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_kernel(E, k, dtype):
    for layers, rows, masked in ((1, 1, False), (3, 130, True), (2, 1037, False)):
        logits = _logits(layers, rows, E, dtype, "cuda", seed=rows)
        mask = (torch.rand(rows, generator=torch.Generator().manual_seed(E)) < 0.7).cuda() if masked else None
        _check(logits, E, k, mask, coef=0.02 * layers * rows)


@pytest.mark.gpu
def test_kernel_of_many_layers_and_rows():
    _check(_logits(100, 77, 8, torch.bfloat16, "cuda"), 8, 2, None)
    _check(_logits(129, 5, 8, torch.float32, "cuda"), 8, 2, None)          # more tensors than one launch takes: torch
    _check(_logits(1, 300001, 16, torch.float32, "cuda"), 16, 4, torch.arange(300001, device="cuda") < 299990)
    uneven = [t for n in (0, 3, 1000, 1) for t in _logits(1, n, 8, torch.float32, "cuda")]
    _check(uneven, 8, 2, None)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("layers", [1, 3])
def test_no_rows_at_all(layers, device):
    logits = [torch.zeros(0, 8, device=device, requires_grad=True) for _ in range(layers)]
    for mask in (None, torch.zeros(0, dtype=torch.bool, device=device)):
        loss, counts = load_balancing_loss_func(logits, 8, 2, mask=mask, return_counts=True)
        grads = torch.autograd.grad(loss, logits)
        assert loss.item() == 0.0 and not counts.any() and all(g.shape == (0, 8) for g in grads)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("fill", [math.nan, math.inf, -math.inf])
def test_rows_left_out_hold_anything(fill, device):
    logits = [t.to(device) for t in _logits(2, 30, 8, torch.float32, "cpu")]
    mask = torch.arange(30, device=device) % 4 > 0
    leaves = [[x.clone().requires_grad_() for x in logits] for _ in range(2)]
    with torch.no_grad():
        for x in leaves[1]:
            x[~mask] = fill
    clean, dirty = (load_balancing_loss_func(x, 8, 2, mask=mask, return_counts=True) for x in leaves)
    assert torch.equal(clean[0], dirty[0]) and torch.equal(clean[1], dirty[1])
    for create in (False, True):
        for a, b in zip(*(torch.autograd.grad(out[0], x, create_graph=create, retain_graph=True) for out, x in zip((clean, dirty), leaves))):
            assert torch.equal(a, b) and not b[~mask].any()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("E", [8, 200])
def test_small_probabilities(E, device):
    """Gradients of experts far below the largest logit, whose differences from it are exact in fp32."""
    x = torch.full((5, E), -50.0)
    x[:, 0] = 0.0
    x[:, 1:5] = torch.tensor([-11.3125, -29.59375, -58.71875, -83.03125])
    leaf = x.to(device).requires_grad_()
    (grad,) = torch.autograd.grad(load_balancing_loss_func(leaf, E, 1), leaf)
    want = oracle([x], E, 1)[2]
    # the exponential, 2 units in the last place (4 half steps), its sum, the division, two products, the share and the rows' sum
    # p f, whose one large term is 1: less than 16 half steps
    assert ((grad.double().cpu() - want).abs() <= 16 * FP32 * want.abs())[:, 1:].all()


@pytest.mark.gpu
def test_kernel_reads_views():
    g = torch.Generator(device="cuda").manual_seed(0)
    wide = torch.randn(50, 3, 24, generator=g, device="cuda")
    odd = torch.randn(50 * 3 * 8 + 1, generator=g, device="cuda")[1:].view(50, 3, 8)
    for x in (wide[..., 8:16], wide[..., ::3], odd, wide[:1, :, :8].expand(50, 3, 8), wide[:, :1, :8].expand(50, 3, 8)):
        _check([x], 8, 2, None)
        _check([x, odd], 8, 2, torch.arange(300, device="cuda")[::2] % 4 < 3)


@pytest.mark.gpu
def test_ties_and_special_values():
    inf, nan = float("inf"), float("nan")
    x = torch.tensor([[0.0, -0.0, 0.0, 0.0], [-inf, -inf, 1.0, -inf], [2.0, 2.0, 1.0, 2.0], [-1.0, -1.0, -inf, -1.0], [1e-40, 0.0, -1e-40, 0.0]])
    _, counts = load_balancing_loss_func(x.cuda(), 4, 2, return_counts=True)
    # row 2 has one finite logit: the second is the lowest expert of the infinite ones
    assert counts.tolist() == [5, 4, 1, 0] and counts.tolist() == load_balancing_loss_func(x, 4, 2, return_counts=True)[1].tolist()
    for row in ([0.0, nan, 1.0, 2.0], [inf, 0.0, 1.0, 2.0], [-inf] * 4):
        y = torch.cat([x, torch.tensor([row])])
        for mask in (None, torch.tensor([1, 1, 1, 1, 1, 0])):
            got = load_balancing_loss_func(y.cuda(), 4, 2, mask=None if mask is None else mask.cuda(), return_counts=True)
            want = load_balancing_loss_func(y, 4, 2, mask=mask, return_counts=True)
            assert torch.equal(got[1].cpu(), want[1]) and got[0].isnan().item() == want[0].isnan().item() == (mask is None)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):          # a NaN of either sign is the largest
        row = torch.tensor([1.0, nan, 2.0, -nan]).copysign(torch.tensor([1.0, 1.0, 1.0, -1.0])).to(dtype)
        assert load_balancing_loss_func(row[None].cuda(), 4, 2, return_counts=True)[1].tolist() == [0, 1, 0, 1]
    leaf = torch.cat([x, torch.full((1, 4), nan)]).cuda().requires_grad_()
    loss = load_balancing_loss_func(leaf, 4, 2, mask=torch.tensor([1, 1, 1, 1, 1, 0], device="cuda"))
    (grad,) = torch.autograd.grad(loss, leaf)
    assert grad.isfinite().all() and not grad[5].any()


@pytest.mark.gpu
def test_same_bits_twice_captured_and_on_another_stream():
    logits = [t.requires_grad_() for t in _logits(4, 3000, 8, torch.float32, "cuda")]

    def step():
        loss, counts = load_balancing_loss_func(logits, 8, 2, return_counts=True)
        return [loss.detach(), counts, *torch.autograd.grad(loss, logits)]

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = step()
    graph.replay()
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)
    with torch.no_grad():
        logits[2].mul_(-1.0)
    graph.replay()
    for a, c in zip(step(), third):
        assert torch.equal(a, c)


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["checkpoint", "on the host"])
def test_saved_logits_that_move(how):
    """What the backward pass reads is computed again, or copied back, and lies elsewhere than in the forward pass."""
    from torch.utils.checkpoint import checkpoint

    weight = torch.randn(16, 8, generator=torch.Generator().manual_seed(2)).cuda().requires_grad_()
    hidden = [torch.randn(200, 16, generator=torch.Generator().manual_seed(i)).cuda() for i in range(3)]

    def loss():
        return load_balancing_loss_func([h @ weight for h in hidden], 8, 2)

    def again():
        if how == "checkpoint":
            return checkpoint(loss, use_reentrant=False)
        with torch.autograd.graph.save_on_cpu():
            return loss()

    (want,) = torch.autograd.grad(loss(), weight)
    out = again()
    trash = [torch.full((200, 8), math.nan, device="cuda") for _ in range(64)]          # where the logits were
    (got,) = torch.autograd.grad(out, weight)
    assert torch.equal(got, want)
    del trash


@pytest.mark.gpu
def test_logits_written_behind_the_loss():
    leaf = _logits(1, 200, 8, torch.float32, "cuda")[0].requires_grad_()
    for x in (leaf, leaf * 1.0):
        loss = load_balancing_loss_func(x, 8, 2)
        with torch.no_grad():
            x.mul_(2.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(loss, leaf)


@pytest.mark.gpu
def test_memory_goes_with_the_last_pass():
    """A loss that the program keeps does not hold the logits beyond the passes through its graph."""
    for again in (False, True):
        leaf = torch.randn(8, 8, device="cuda", requires_grad=True)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        loss = load_balancing_loss_func(torch.ones(1 << 20, 8, device="cuda") @ leaf, 8, 2)
        if again:
            torch.autograd.grad(loss, leaf, retain_graph=True)
            assert torch.cuda.memory_allocated() - before >= 32 << 20
        torch.autograd.grad(loss, leaf)
        assert torch.cuda.memory_allocated() - before < 1 << 20


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["other data", "smaller data", "data on the host", "hooks of the node", "a view moved"])
def test_saved_logits_that_get_other_storage(how):
    """The gradient is that of the logits as the loss saw them, wherever they lie by then."""
    for leaf in (False,) if how == "data on the host" else (True, False):          # torch refuses a leaf that went to another device
        logits = [t.requires_grad_() for t in _logits(3, 200, 8, torch.float32, "cuda", seed=5)]
        seen = logits if leaf else [t * 1.0 for t in logits]
        (want,) = torch.autograd.grad(load_balancing_loss_func(seen, 8, 2), logits[1], retain_graph=True)
        mask = torch.arange(200, device="cuda") % 7 > 0
        (want_masked,) = torch.autograd.grad(load_balancing_loss_func(seen, 8, 2, mask=mask), logits[1], retain_graph=True)
        loss, masked = load_balancing_loss_func(seen, 8, 2), load_balancing_loss_func(seen, 8, 2, mask=mask)
        if how == "hooks of the node":
            kept = []
            for out in (loss, masked):
                for saved in out.grad_fn._raw_saved_tensors[2:]:
                    saved.register_hooks(lambda t: kept.append(t.cpu()) or len(kept) - 1, lambda i: kept[i].cuda())
        else:
            for t in seen:
                t.data = {"other data": lambda: torch.full_like(t, math.nan), "smaller data": lambda: t.data[:1, :1].clone(), "data on the host": lambda: t.data.cpu(),
                          "a view moved": lambda: torch.full((200, 16), math.nan, device="cuda")[:, ::2]}[how]()
        trash = [torch.full((200, 8), math.nan, device="cuda") for _ in range(64)]          # where the logits were
        for _ in range(2):          # the graph is kept
            for out, same in ((loss, want), (masked, want_masked)):
                (got,) = torch.autograd.grad(out, logits[1], retain_graph=True)
                assert torch.equal(got, same)
        del trash


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("masked", [False, True])
def test_other_derivatives(masked, device):
    """Second derivatives, forward mode and torch.func, against the formulas in float64."""
    import torch.autograd.forward_ad as fw

    E, k, layers, rows = 8, 2, 3, 50
    logits = [t.to(device) for t in _logits(layers, rows, E, torch.float32, "cpu")]
    v = [t.to(device) for t in _logits(layers, rows, E, torch.float32, "cpu", seed=7)]
    mask = (torch.arange(rows, device=device) % 3 > 0) if masked else None

    def loss_of(*x):
        return load_balancing_loss_func(list(x), E, k, mask=mask)

    _, counts, dx = oracle(logits, E, k, mask)
    n = int(counts.sum()) // k
    p = torch.softmax(torch.cat(logits).double(), -1) * (1.0 if mask is None else mask.repeat(layers)[:, None])
    f, t = counts.double() / n, torch.cat(v).double()
    dp = p * (t - (p * t).sum(-1, keepdim=True))
    second = E / (k * n) * (dp * (f - (p * f).sum(-1, keepdim=True)) - p * (dp * f).sum(-1, keepdim=True))
    # a softmax and three more products and sums over E, 2^-24 each, of terms that are no larger than these
    size = E / (k * n) * (p * (t.abs() + (p * t.abs()).sum(-1, keepdim=True))) * f.max() * 4
    leaves = [x.clone().requires_grad_() for x in logits]
    first = torch.autograd.grad(loss_of(*leaves), leaves, create_graph=True)
    again = torch.autograd.grad(sum((a * b).sum() for a, b in zip(first, v)), leaves)
    assert ((torch.cat(again).double() - second).abs() <= 2.0 ** -24 * (24 + 3 * E) * (size + size.mean(-1, keepdim=True))).all()
    slope = (dx * t).sum()
    # rows of E products, then some hundred sums
    near = 2.0 ** -24 * (24 + 4 * E) * (E / (k * n) * (p * t.abs()).sum() * f.max() * 4)
    with fw.dual_level():
        _, tangent = fw.unpack_dual(loss_of(*[fw.make_dual(x, y) for x, y in zip(logits, v)]))
    assert abs(tangent.double() - slope) <= near
    assert abs(torch.func.jvp(loss_of, tuple(logits), tuple(v))[1].double() - slope) <= near
    grads = torch.func.grad(loss_of, argnums=tuple(range(layers)))(*logits)
    for a, b, c in zip(grads, first, torch.autograd.grad(loss_of(*leaves), leaves)):
        assert (a - b).abs().max() <= 2.0 ** -24 * (24 + E) * 4 * a.abs().max() and (b - c).abs().max() <= 2.0 ** -24 * (24 + E) * 4 * c.abs().max()
    only = torch.autograd.grad(loss_of(logits[0], leaves[1], logits[2]), leaves[1], create_graph=True)[0]
    assert only.requires_grad and torch.equal(only, first[1])


@pytest.mark.gpu
def test_part_of_the_layers_needs_gradients():
    a, b = _logits(2, 40, 8, torch.float32, "cuda")
    a.requires_grad_()
    loss = load_balancing_loss_func([b, a], 8, 2)
    loss.backward()
    assert (a.grad.double() - oracle([b, a], 8, 2)[2][40:]).abs().max() <= 1e-7
