"""Dropout from the counter-based generator: its words, its mask in every layout and type, its gradient, its refusals."""
import math

import pytest
import torch

from neuronx_distributed_llama3_2_b200.ops.dropout import Dropout, dropout, dropout_keep, philox_words

STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def test_generator_gives_the_published_words():
    # the known answers that the authors publish with Philox4x32, for counter and key of zeros, seven and ten rounds
    assert philox_words(4, 0, 0).tolist() == [0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48]
    assert philox_words(4, 0, 0, rounds=10).tolist() == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]

    def words(c, k, rounds=7):          # in Python's integers
        c, k = list(c), list(k)
        for _ in range(rounds):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [b >> 32 ^ c[1] ^ k[0], b % 2 ** 32, a >> 32 ^ c[3] ^ k[1], a % 2 ** 32]
            k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
        return c

    for seed, offset in ((0, 0), (2 ** 64 - 1, 2 ** 64 - 1), (0x0123456789ABCDEF, 0x89ABCDEF01234567)):
        want = [w for i in range(3) for w in words((i, 0, offset % 2 ** 32, offset >> 32), (seed % 2 ** 32, seed >> 32))]
        assert philox_words(11, seed, offset).tolist() == want[:11]


def test_share_kept_and_independence():
    n, p = 1 << 20, 0.3
    a, b = dropout_keep((n,), p, 1, 0), dropout_keep((n,), p, 1, 1)
    sigma = math.sqrt(p * (1 - p) / n)
    assert abs(a.double().mean() - (1 - p)) <= 5 * sigma
    both = (a & b).double().mean()
    assert abs(both - (1 - p) ** 2) <= 5 * math.sqrt((1 - p) ** 2 * (1 - (1 - p) ** 2) / n)


def _check(x, p, seed, offset=0, residual=None, state=None):
    leaf = x.detach().requires_grad_()
    res = None if residual is None else residual.detach().requires_grad_()
    g = torch.Generator(device=x.device).manual_seed(1)
    dy = torch.randn(x.shape, generator=g, device=x.device).to(x.dtype)
    y = dropout(leaf, p, seed if state is None else state, offset, residual=res)
    grads = torch.autograd.grad(y, [leaf] + ([] if res is None else [res]), dy)
    keep = dropout_keep(x.shape, p, seed, offset, x.device)
    want = torch.where(keep, x.double() / (1 - p), 0.0) + (0.0 if residual is None else residual.double())
    # fp32 for the scale and the product (twice half a step), one rounding of the result; fp16 ends at steps of 2^-24
    near = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    slack = 3 * 2.0 ** -24 * (x.double().abs() / (1 - p) + want.abs())
    assert ((y.double() - want).abs() <= STEP[x.dtype] * want.abs() + slack + near).all()
    back = torch.where(keep, dy.double() / (1 - p), 0.0)
    assert ((grads[0].double() - back).abs() <= (STEP[x.dtype] + 3 * 2.0 ** -24) * back.abs() + near).all()
    assert torch.equal(y.eq(0) | keep, torch.ones_like(keep)) or residual is not None
    if res is not None:
        assert torch.equal(grads[1], dy)
    return y


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1,), (3,), (7, 13), (2, 3, 8)])
def test_torch_path(dtype, shape):
    x = torch.randn(shape, generator=torch.Generator().manual_seed(0)).to(dtype)
    _check(x, 0.3, 77, 5)
    _check(x, 0.9, 2 ** 63 + 9, 0, residual=x.flip(0))
    _check(x, 0.5, 3, 7, state=torch.tensor([3]))


def test_edges():
    x = torch.tensor([1.0, float("nan"), float("inf"), -2.0], requires_grad=True)
    assert dropout(x, 0.0) is x and dropout(x, 0.7, training=False) is x
    y = dropout(x, 1.0, residual=torch.ones(4))
    assert y.tolist() == [1.0] * 4 and not torch.autograd.grad(y.sum(), x)[0].any()
    many = torch.full((1000,), float("nan"))
    keep = dropout_keep((1000,), 0.5, 4)
    assert torch.equal(dropout(many, 0.5, 4).isnan(), keep)
    assert dropout(torch.empty(0, 5), 0.5, 1).shape == (0, 5)
    state = torch.tensor([4, 3])
    assert torch.equal(dropout(torch.ones(1000), 0.5, state, 2), dropout(torch.ones(1000), 0.5, 4, 5))


@pytest.mark.parametrize("kw", [dict(p=-0.1), dict(p=1.5), dict(p=float("nan")), dict(residual=torch.zeros(3)), dict(seed=torch.tensor([1.0])),
                                dict(residual=torch.zeros(4, dtype=torch.float16)), dict(seed=torch.zeros(3, dtype=torch.int64))])
def test_refusals(kw):
    with pytest.raises(ValueError):
        dropout(torch.zeros(4), **{"p": 0.5, **kw})
    with pytest.raises(ValueError):
        dropout(torch.zeros(4, dtype=torch.int64), 0.5)


def test_module_draws_from_the_cpu_generator_and_checkpoints():
    from torch.utils.checkpoint import checkpoint

    m = Dropout(0.5)
    x = torch.ones(4096, requires_grad=True)
    torch.manual_seed(3)
    a, b = m(x), m(x)
    assert not torch.equal(a, b)
    torch.manual_seed(3)
    assert torch.equal(m(x), a)
    y = checkpoint(lambda t: m(t) * t, x, use_reentrant=False)
    (grad,) = torch.autograd.grad(y.sum(), x)
    assert torch.equal(grad, 2 * y)          # the mask of the repeated call is the first call's
    assert m.eval()(x) is x


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_checkpointed_with_a_seed_tensor(device):
    """Counted on behind the backward pass, or a copy that stays: both are the numbers that the first call read."""
    from torch.utils.checkpoint import checkpoint

    x = torch.ones(4096, device=device, requires_grad=True)
    state = torch.tensor([5, 0], device=device)
    for step in range(3):
        y = checkpoint(lambda t: dropout(t, 0.5, state, 7) * t, x, use_reentrant=False)
        (grad,) = torch.autograd.grad(y.sum(), x)
        keep = dropout_keep((4096,), 0.5, 5, 7 + step, device)
        assert torch.equal(y != 0, keep) and torch.equal(grad, 2 * y)
        state[1] += 1
    for step in range(3, 6):
        now = state.clone()
        y = checkpoint(lambda t: dropout(t, 0.5, now, 7) * t, x, use_reentrant=False)
        state[1] += 1
        (grad,) = torch.autograd.grad(y.sum(), x)
        assert torch.equal(y != 0, dropout_keep((4096,), 0.5, 5, 7 + step, device)) and torch.equal(grad, 2 * y)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 7, 8, 9, 4095, 4096, 4097, 8192 * 3 + 1, 1 << 20])
def test_kernel(dtype, n):
    x = torch.randn(n, generator=torch.Generator(device="cuda").manual_seed(n), device="cuda").to(dtype)
    y = _check(x, 0.3, 2 ** 64 - 5, 2 ** 40 + n)
    assert torch.equal(y, dropout(x.cpu(), 0.3, 2 ** 64 - 5, 2 ** 40 + n).cuda())
    _check(x, 0.75, n, 0, residual=x.flip(0))
    _check(x, 1 - 2.0 ** -20, n)
    _check(x, 2.0 ** -33, n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_kernel_layouts(dtype):
    g = torch.Generator(device="cuda").manual_seed(0)
    base = torch.randn(64 * 37 * 9 + 1, generator=g, device="cuda").to(dtype)
    odd = base[1:].view(64, 37, 9)
    for x in (odd, odd.transpose(0, 2), odd[:, ::2], odd[..., :1].expand(64, 37, 5)):
        y = _check(x, 0.4, 11, residual=base[:x.numel()].view(x.shape))
        assert torch.equal(dropout(x, 0.4, 11), dropout(x.contiguous(), 0.4, 11))
    nan = torch.full((5000,), float("nan"), device="cuda", dtype=dtype)
    assert torch.equal(dropout(nan, 0.5, 4).isnan(), dropout_keep((5000,), 0.5, 4, device="cuda"))
    ones = torch.ones(5000, device="cuda", dtype=dtype)
    assert torch.equal(dropout(nan, 0.5, 4, residual=ones).isnan(), dropout_keep((5000,), 0.5, 4, device="cuda"))


@pytest.mark.gpu
def test_counters_above_32_bits():
    n = (1 << 32) + 4096 + 3          # 4 GB of bf16 and more: element numbers and bytes pass 32 bits
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    y = dropout(x, 0.5, 9)
    for first in (0, (1 << 31) - 2048, (1 << 32) - 2048, n - 4096):
        first -= first % 4
        i = torch.arange(first // 4, first // 4 + 1024, device="cuda")
        # the words of those counters, by the generator's own function on a shifted counter
        part = torch.stack([_words_at(int(c), 9) for c in i[:: 64].tolist()]).view(-1)
        at = (i[::64, None] * 4 + torch.arange(4, device="cuda")).view(-1)
        inside = at < n
        assert torch.equal(y[at[inside]] > 0, (part.cuda() >= 2 ** 31)[inside])


def _words_at(counter, seed):
    c, k = [counter % 2 ** 32, counter >> 32, 0, 0], [seed, 0]
    for _ in range(7):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [b >> 32 ^ c[1] ^ k[0], b % 2 ** 32, a >> 32 ^ c[3] ^ k[1], a % 2 ** 32]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return torch.tensor(c)


@pytest.mark.gpu
def test_captured_with_a_state_on_the_device():
    x = torch.randn(3000, device="cuda", generator=torch.Generator(device="cuda").manual_seed(0)).requires_grad_()
    state = torch.tensor([21, 0], device="cuda")

    def step():
        y = dropout(x, 0.5, state, 4)
        state[1] += 1                                  # counted on before the backward pass: that one uses what this call used
        return y, torch.autograd.grad(y, x, torch.ones_like(y))[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = step()
    for turn in range(3):
        offset = 4 + int(state[1])
        graph.replay()
        keep = dropout_keep((3000,), 0.5, 21, offset, "cuda")
        assert torch.equal(dx, keep.float() * 2) and torch.equal(y, torch.where(keep, x * 2, 0.0))
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            dropout(x, 0.5)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_forward_mode_and_func(device):
    """A tangent is dropped where its element is, and torch.func's transforms see what autograd does."""
    import torch.autograd.forward_ad as fw

    g = torch.Generator().manual_seed(0)
    x, t, r, rt = (torch.randn(300, generator=g).to(device) for _ in range(4))
    keep = dropout_keep((300,), 0.25, 9, 2, device)
    slope = torch.where(keep, 1.0 / 0.75, 0.0)
    state = torch.tensor([9, 2], device=device)
    for kw in (dict(seed=9, offset=2), dict(seed=state)):
        for residual, rest in ((None, None), (r, None), (r, rt)):
            with fw.dual_level(), torch.no_grad():
                dual = fw.make_dual(x, t)
                add = residual if rest is None else fw.make_dual(residual, rest)
                y, tangent = fw.unpack_dual(dropout(dual, 0.25, residual=add, **kw))
            # the kernel rounds a product and its sum with the residual once, torch each: the product's half step, and one of either sum
            want = dropout(x, 0.25, residual=residual, **kw)
            assert ((y - want).abs() <= 2.0 ** -24 * (1.0001 * x.abs() / 0.75 + y.abs() + want.abs())).all()
            # a product of fp32 and a sum
            assert (tangent - (slope * t + (0.0 if rest is None else rest))).abs().max() <= 2.0 ** -22 * 8
    with fw.dual_level():
        assert fw.unpack_dual(dropout(x, 0.25, 9, 2, residual=fw.make_dual(r, rt))).tangent.equal(rt)
        assert fw.unpack_dual(dropout(x, 0.25, 9, 2)).tangent is None
    grad = torch.func.grad(lambda z: (dropout(z, 0.25, 9, 2) * t).sum())(x)
    assert (grad - slope * t).abs().max() <= 2.0 ** -22 * 8
    assert torch.equal(torch.func.jvp(lambda z: dropout(z, 0.25, 9, 2), (x,), (torch.ones_like(x),))[1] != 0, keep)


@pytest.mark.gpu
def test_float64_on_the_gpu():
    x = torch.randn(100, device="cuda", dtype=torch.float64)
    assert torch.equal(dropout(x, 0.5, 4) != 0, dropout_keep((100,), 0.5, 4, device="cuda"))
