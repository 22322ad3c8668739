"""Attention over packed sequences on the tensor cores against float64, with bounds that count the roundings."""
import pytest
import torch

from packed_oracle import check, packed

pytestmark = pytest.mark.gpu


def _inputs(T, H, G, D, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + T)
    qkv = torch.randn(T, H + 2 * G, D, generator=g, device="cuda").mul_(scale).bfloat16()
    do = torch.randn(T, H, D, generator=g, device="cuda").bfloat16()
    return qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:], do


def _run(q, k, v, do, ends, causal, dtype=torch.int32, scale=None):
    from neuronx_distributed_llama3_2_b200.ops.attention import flash_attn_packed_func

    q, k, v = (x.detach().requires_grad_() for x in (q, k, v))
    cu = ends if isinstance(ends, torch.Tensor) else torch.tensor(ends, dtype=dtype, device="cuda")
    o = flash_attn_packed_func(q, k, v, cu, softmax_scale=scale, causal=causal)
    return dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, (q, k, v), do)), o=o.detach())


def _ends(lens, first=0):
    out = [first]
    for n in lens:
        out.append(out[-1] + n)
    return out


# boundaries on and beside the tiles of 64 and 128 rows, one token, empty sequences, rows ahead of the first and behind the last
BATCHES = [([1], 0, 1), ([1, 1, 1], 0, 3), ([64], 0, 64), ([65, 63, 128], 0, 256), ([127, 1, 0, 129, 300, 0], 0, 557), ([256, 384], 0, 700),
           ([5, 200, 33], 7, 400), ([], 0, 130), ([0, 0], 3, 5), ([1000, 37, 2, 513], 129, 1700)]


def test_plan_lists_every_tile_once():
    from neuronx_distributed_llama3_2_b200.ops.packed_attention import PackedSequences

    g = torch.Generator().manual_seed(0)
    long = torch.randint(0, 3, (5000,), generator=g).tolist()
    for lens, first, T in BATCHES + [(long, 0, sum(long) + 200), ([600000, 70], 0, 600200)]:
        for dtype in (torch.int32, torch.int64):
            for causal in (True, False):
                ends = _ends(lens, first)
                size = 256 if causal == (dtype is torch.int32) else 128
                lists, entries, columns = PackedSequences(torch.tensor(ends, dtype=dtype, device="cuda"), T).plan(causal, size)
                rows = lists[:entries].tolist()
                want, pad = set(), 0
                for a, b in zip(ends, ends[1:]):
                    want |= {(a, b - a, t, pad) for t in range(-(-(b - a) // size))}
                    pad += (b - a + 3) // 4 * 4
                tiles = [tuple(r) for r in rows if r[1]]
                assert set(tiles) == want and len(tiles) == len(want) and pad + 64 <= columns
                assert all(r[1] for r in rows[:len(tiles)])
                weight = [min(t[2] + 1 if causal else -(-t[1] // size), 4096) for t in tiles]
                assert weight == sorted(weight, reverse=True)
                outside = [r for a, n, t, _ in rows if not n for r in range(a, a + t)]
                assert sorted(outside) == [r for r in range(T) if r < first or r >= ends[-1]]


def test_plan_brings_wrong_boundaries_back():
    from neuronx_distributed_llama3_2_b200.ops.packed_attention import PackedSequences

    cu = torch.tensor([-5, 40, 30, 2 ** 31 + 10, 90], dtype=torch.int64, device="cuda")
    lists, entries, _ = PackedSequences(cu, 100).plan(True)
    tiles = sorted(tuple(r) for r in lists[:entries].tolist() if r[1])
    assert tiles == [(0, 40, 0, 0), (40, 60, 0, 40)]


@pytest.mark.parametrize("H,G,D", [(4, 2, 64), (2, 2, 128), (6, 1, 64), (3, 1, 128)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,first,T", BATCHES)
def test_matches_float64(lens, first, T, causal, H, G, D):
    q, k, v, do = _inputs(T, H, G, D)
    ends = _ends(lens, first)
    got = _run(q, k, v, do, ends, causal, torch.int64 if T % 2 else torch.int32)
    want = packed(q, k, v, ends, causal, do)
    for name in ("o", "dq", "dk", "dv"):
        check(got[name], want, name)
    outside = [r for r in range(T) if r < first or r >= ends[-1]]
    assert all(got[n][outside].eq(0).all() for n in got)


# one K/V block per CTA and several CTAs per block, long walks, many query heads over one key head
@pytest.mark.parametrize("lens,H,G,D,causal", [([2500, 1200], 4, 1, 128, True), ([4100], 2, 1, 64, True), ([700] * 40, 8, 8, 64, False),
                                               ([1, 2, 3] * 200, 4, 4, 128, True), ([129] * 90 + [2048], 8, 2, 128, True)])
def test_long_and_many(lens, H, G, D, causal):
    T = sum(lens) + 11
    q, k, v, do = _inputs(T, H, G, D)
    got, want = _run(q, k, v, do, _ends(lens), causal), packed(q, k, v, _ends(lens), causal, do)
    for name in got:
        check(got[name], want, name)


# long stretches of no sequence: so many entries that every CTA has several of them in a row behind its items, whose last value tiles are
# whole or cut
@pytest.mark.parametrize("lens,first,T", [([3400], 0, 8192), ([100], 0, 8192), ([8000], 0, 16384), ([3192], 5000, 8192), ([300, 1664], 3000, 9000),
                                          ([2000, 128], 4000, 12000)])
@pytest.mark.parametrize("H,G,D,causal", [(32, 8, 64, True), (32, 8, 128, False), (12, 12, 64, False), (9, 3, 128, True)])
def test_long_gaps(lens, first, T, H, G, D, causal):
    q, k, v, do = _inputs(T, H, G, D)
    ends = _ends(lens, first)
    inside = slice(first, ends[-1])
    for x in (q, k, v, do):                          # what lies between is nobody's
        x[:first], x[ends[-1]:] = float("nan"), float("nan")
    got = _run(q, k, v, do, ends, causal)
    want = packed(*(x[inside] for x in (q, k, v)), [e - first for e in ends], causal, do[inside])
    for name in got:
        check(got[name][inside], want, name)
        assert not got[name][:first].any() and not got[name][ends[-1]:].any()


@pytest.mark.parametrize("lens,first,T,H,G,D,causal", [([300, 130], 7, 600, 4, 2, 64, True), ([2500], 100, 2700, 4, 1, 128, True),
                                                       ([60] * 80, 0, 5000, 3, 1, 64, False), ([700] * 20, 500, 16000, 8, 4, 128, False)])
def test_waits_that_run_out(lens, first, T, H, G, D, causal):
    """A call whose waits give up at once leaves NaN in every sequence and zeros outside, the next call fails, and those behind it are sound."""
    from neuronx_distributed_llama3_2_b200.ops import packed_attention as pa

    q, k, v, do = _inputs(T, H, G, D)
    ends = _ends(lens, first)
    p = pa.PackedSequences(torch.tensor(ends, device="cuda"), T)
    scale = D ** -0.5
    inside = slice(first, ends[-1])
    grads = [torch.full(x.shape, 7.0, dtype=x.dtype, device="cuda") for x in (q, k, v)]

    def all_nan(*xs):
        return all(x[inside].isnan().all() and not x[:first].any() and not x[ends[-1]:].any() for x in xs)

    assert not pa.gave_up()
    o, lse, rest = pa._forward(q, k, v, p, scale, causal, True)
    assert not pa.gave_up() and o.isfinite().all()
    lost, lost_lse, lost_rest = pa._forward(q, k, v, p, scale, causal, True, wait_tries=0)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="gave up"):
        pa._forward(q, k, v, p, scale, causal, True)
    assert all_nan(lost)
    pa._backward(q, k, v, lost, lost_lse, lost_rest, do, *grads, p.plan(causal), p.count, scale, causal)
    assert all_nan(*grads) and not pa.gave_up()
    pa._backward(q, k, v, o, lse, rest, do, *grads, p.plan(causal), p.count, scale, causal, wait_tries=0)
    torch.cuda.synchronize()
    assert all_nan(*grads)
    with pytest.raises(RuntimeError, match="gave up"):
        pa._backward(q, k, v, o, lse, rest, do, *grads, p.plan(causal), p.count, scale, causal)
    pa._forward(q, k, v, p, scale, causal, True, wait_tries=0)
    assert pa.gave_up() and not pa.gave_up()
    got, want = _run(q, k, v, do, ends, causal), packed(q, k, v, ends, causal, do)
    for name in got:
        check(got[name], want, name)


# scores that rise along the keys (the running maximum moves in every tile) and scores that leave one weight
@pytest.mark.parametrize("scale", [0.01, 1.0, None])
def test_scales(scale):
    q, k, v, do = _inputs(777, 4, 2, 64, scale=2.0)
    k = (k.float() * torch.linspace(0.1, 3.0, 777, device="cuda")[:, None, None]).bfloat16()
    ends = [0, 300, 777]
    got, want = _run(q, k, v, do, ends, True, scale=scale), packed(q, k, v, ends, True, do, scale)
    check(got["o"], want, "o")
    # scores are up to 1000 here, so their fp32 error is up to 2^-14 and more of a weight: gradients by norm, four roundings
    for n in ("dq", "dk", "dv"):
        assert (got[n].double() - want[n][0]).norm() <= 4 * 2.0 ** -8 * want[n][0].norm()


@pytest.mark.parametrize("scale", [0.0, -0.0, -0.125, -1.0, 2.0 ** -126])
@pytest.mark.parametrize("causal,D", [(True, 64), (False, 128)])
def test_scales_that_are_not_positive(scale, causal, D):
    q, k, v, do = _inputs(400, 4, 2, D)
    ends = [0, 150, 390]
    got, want = _run(q, k, v, do, ends, causal, scale=scale), packed(q, k, v, ends, causal, do, scale)
    bounds = packed(-q, k, v, ends, causal, do, -scale) if scale < 0.0 else want          # bounds of the same sums, with the scale's size
    for name in got:
        check(got[name], {name: (want[name][0], bounds[name][1])}, name)
    from neuronx_distributed_llama3_2_b200.ops import packed_attention as pa

    p = pa.PackedSequences(torch.tensor(ends, device="cuda"), 400)
    for bad in (0.0, -1.0, float("nan"), float("inf"), 2.0 ** -130):
        with pytest.raises(RuntimeError, match="scale"):
            pa._forward(q, k, v, p, bad, causal, False)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128])
def test_sequences_do_not_touch(causal, D):
    """What one sequence holds, infinities and NaN among it, leaves every other sequence's results as they are, bit by bit where
    nothing is summed in an order that is not fixed."""
    lens, T = [100, 130, 70, 1, 250], 600
    q, k, v, do = (x.contiguous() for x in _inputs(T, 4, 2, D))
    ends = _ends(lens)
    clean = _run(q, k, v, do, ends, causal)
    for bad, fill in ((1, float("nan")), (2, float("inf")), (3, float("nan")), (5, float("nan"))):
        rows = slice(ends[bad], ends[bad + 1] if bad < 5 else T)
        dirty = [x.clone() for x in (q, k, v, do)]
        for x in dirty:
            x[rows] = fill
        got = _run(*dirty, ends, causal)
        keep = torch.ones(T, dtype=torch.bool, device="cuda")
        if bad < 5:
            keep[rows] = False
        assert torch.equal(got["o"][keep], clean["o"][keep])
        for n in ("dq", "dk", "dv"):
            assert got[n][keep].isfinite().all()
            # the same sums in another order: at most one step of bf16
            assert ((got[n] - clean[n])[keep].abs() <= 2 * 2.0 ** -8 * clean[n][keep].abs() + 1e-6).all()


def test_strides_and_a_second_stream():
    T, H, G, D = 333, 4, 2, 128
    q, k, v, do = _inputs(T, H, G, D)
    ends = [0, 50, 333]
    want = packed(q, k, v, ends, True, do)
    head_first = q.permute(1, 0, 2).contiguous().permute(1, 0, 2)
    odd = torch.empty(T * G * D + 1, dtype=torch.bfloat16, device="cuda")[1:].view(T, G, D).copy_(k)          # 2 bytes off a boundary
    wide = torch.empty(T, G, 2 * D, dtype=torch.bfloat16, device="cuda")[..., ::2].copy_(v)                    # no unit stride
    late = do.transpose(0, 1).contiguous().transpose(0, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(head_first, odd, wide, late, ends, True)
    torch.cuda.current_stream().wait_stream(side)
    for name in got:
        check(got[name], want, name)
    grad = torch.ones((), dtype=torch.bfloat16, device="cuda").expand(T, H, D)                     # a sum's gradient has no strides
    got, want = _run(q, k, v, grad, ends, True), packed(q, k, v, ends, True, grad)
    for name in got:
        check(got[name], want, name)


def test_rows_further_apart_than_32_bits():
    """Queries and the results' gradients as views of a row store of 2.4e9 elements."""
    T, H, G, D = 300, 4, 2, 64
    q, k, v, do = _inputs(T, H, G, D)
    store = torch.empty((T, 8 << 20), dtype=torch.bfloat16, device="cuda")
    views = [store[:, at:at + H * D].view(T, H, D) for at in (0, 1 << 22)]
    for view, x in zip(views, (q, do)):
        view.copy_(x)
    ends = [0, 130, 290]
    want = packed(q, k, v, ends, True, do)
    got = _run(views[0], k, v, views[1], ends, True)
    for name in got:
        check(got[name], want, name)


def test_one_list_for_several_calls_and_no_gradients():
    from neuronx_distributed_llama3_2_b200.ops.attention import flash_attn_packed_func
    from neuronx_distributed_llama3_2_b200.ops.packed_attention import PackedSequences

    ends = [0, 90, 400]
    p = PackedSequences(torch.tensor(ends, device="cuda"), 400)
    for seed in (0, 1):
        q, k, v, _ = _inputs(400, 4, 2, 64, seed)
        for causal in (True, False):
            with torch.no_grad():
                o = flash_attn_packed_func(q, k, v, p, causal=causal)
            check(o, packed(q, k, v, ends, causal), "o")
            check(flash_attn_packed_func(q, k, v, p, causal=causal), packed(q, k, v, ends, causal), "o")


def test_captured_step_follows_new_lengths():
    from neuronx_distributed_llama3_2_b200.ops.attention import flash_attn_packed_func

    T = 640
    q, k, v, do = (x.contiguous() for x in _inputs(T, 4, 2, 64))
    cu = torch.tensor([0, 100, 640], dtype=torch.int32, device="cuda")
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]

    def step():
        o = flash_attn_packed_func(*leaves, cu)
        return (o, *torch.autograd.grad(o, leaves, do))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for ends in ([0, 100, 640], [0, 333, 334], [7, 7, 600]):
        cu.copy_(torch.tensor(ends))
        graph.replay()
        want = packed(q, k, v, ends, True, do)
        for name, x in zip(("o", "dq", "dk", "dv"), out):
            check(x, want, name)


@pytest.mark.parametrize("G", [2, 4])
def test_two_graphs_and_two_streams_of_one_object(G):
    """Each capture and each stream makes its own lists: those of a graph that is gone are nobody else's."""
    from neuronx_distributed_llama3_2_b200.ops import attention, rope
    from neuronx_distributed_llama3_2_b200.ops.packed_attention import PackedSequences

    T, ends = 700, [0, 300, 301, 690]
    q, k, v, do = (x.contiguous() for x in _inputs(T, 4, G, 64))
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    qkv = torch.cat([q, k, v], 1)
    cos, sin = rope.build_rope_cache(T, 64, 10000.0, None, device="cuda")
    p = PackedSequences(torch.tensor(ends, device="cuda"), T)
    want = packed(q, k, v, ends, True, do)

    def step():
        o = attention.flash_attn_packed_func(*leaves, p)
        return (o.detach(), *torch.autograd.grad(o, leaves, do), attention.rope_flash_attn_packed_func(qkv, cos, sin, 4, G, p))

    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    graph, out = graphs.pop(1)
    graphs.clear()                                              # the first one's memory goes back
    torch.cuda.empty_cache()
    trash = [torch.full((1 << 20,), 0x7f, dtype=torch.uint8, device="cuda") for _ in range(8)]
    graph.replay()
    turned = step()[-1]                                         # eager, behind the captures
    streams = [torch.cuda.Stream() for _ in range(2)]
    late = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for s in streams:                                           # at the same time
        with torch.cuda.stream(s):
            late.append(step())
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for results in (out, *late):
        for name, x in zip(("o", "dq", "dk", "dv"), results):
            check(x, want, name)
        assert torch.equal(results[-1], turned)
    del trash


def test_graphs_whose_lists_the_object_let_go():
    """Earlier graphs of one object are replayed behind later captures, follow new lengths, and their memory goes back with them."""
    from neuronx_distributed_llama3_2_b200.ops.attention import flash_attn_packed_func
    from neuronx_distributed_llama3_2_b200.ops.packed_attention import PackedSequences

    T = 500
    q, k, v, _ = (x.contiguous() for x in _inputs(T, 4, 2, 64))
    cu = torch.tensor([0, 100, 500], dtype=torch.int32, device="cuda")
    p = PackedSequences(cu, T)
    flash_attn_packed_func(q, k, v, p)
    graphs = []
    for _ in range(4):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = flash_attn_packed_func(q, k, v, p)
        graphs.append((graph, out))
    assert len(p._plans) <= 2          # one list without a capture, one of the last
    trash = [torch.full((T, 4), 1 << 20, dtype=torch.int32, device="cuda") for _ in range(64)]
    for ends in ([0, 100, 500], [0, 333, 334], [7, 7, 480]):
        cu.copy_(torch.tensor(ends))
        want = packed(q, k, v, ends, True)
        for graph, out in graphs[::-1]:
            out.fill_(float("nan"))
            graph.replay()
            check(out, want, "o")
    del trash


def test_backward_has_the_lists_of_its_forward():
    """Boundaries that are overwritten before the backward pass, with heads that take other lists there."""
    from neuronx_distributed_llama3_2_b200.ops.attention import flash_attn_packed_func

    T, ends = 640, [0, 100, 640]
    q, k, v, do = (x.contiguous() for x in _inputs(T, 4, 4, 64))
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    cu = torch.tensor(ends, device="cuda")
    o = flash_attn_packed_func(*leaves, cu)
    cu.fill_(640)
    want = packed(q, k, v, ends, True, do)
    for name, x in zip(("o", "dq", "dk", "dv"), (o.detach(), *torch.autograd.grad(o, leaves, do))):
        check(x, want, name)


@pytest.mark.parametrize("D", [64, 128])
def test_delta_is_not_of_the_rounded_result(D):
    """Two tokens that see one another, queries of zero: weights of one half, score gradients of d and -d.  With keys of ones dQ is the sum
    of the two, each rounded, so it is zero unless Delta's error e moves them apart: that takes a border between two numbers of bf16,
    2^-8 |d| apart, inside 2 e.  With Delta of the rounded result e is some 2^-9 |o| |dO| and most elements are not zero; with what the
    rounding took (to 2^-8 of it) and fp32 sums less than one in fifty moves."""
    T, H = 512, 4
    _, _, v, do = _inputs(T, H, H, D)
    q, k = torch.zeros_like(v), torch.ones_like(v)
    got = _run(q, k, v, do, list(range(0, T + 1, 2)), False)
    assert (got["dq"] != 0).any(-1).float().mean() <= 0.1


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_what_rounding_took_is_kept_by_sequence(D, causal):
    """As above in a long row with few sequences, some of them long or empty; what is kept for it grows with the sequences, not the row."""
    from neuronx_distributed_llama3_2_b200.ops import packed_attention as pa

    lens, H = [2] * 40 + [0, 5000, 0, 300] + [2] * 40 + [0], 4
    T = sum(lens) + 9000
    ends = _ends(lens, 200)
    _, _, v, do = _inputs(T, H, H, D)
    q, k = torch.zeros_like(v), torch.ones_like(v)
    p = pa.PackedSequences(torch.tensor(ends, device="cuda"), T)
    _, _, rest = pa._forward(q, k, v, p, D ** -0.5, causal, True)
    assert rest.numel() == H * 128 * len(lens) * D < H * T * D
    dq = _run(q, k, v, do, torch.tensor(ends, device="cuda"), causal)["dq"]
    # causal: the first token sees itself alone, and its score gradient is fp32's rounding; the second has the two of one half
    pairs = [a + i for a, n in zip(ends, lens) if n == 2 for i in range(causal, 2)]
    assert (dq[pairs] != 0).any(-1).float().mean() <= 0.1


@pytest.mark.parametrize("how", ["checkpoint", "on the host"])
def test_saved_tensors_that_move(how):
    from torch.utils.checkpoint import checkpoint
    from neuronx_distributed_llama3_2_b200.ops.attention import flash_attn_packed_func

    T, ends = 300, [0, 120, 290]
    q, k, v, do = _inputs(T, 4, 2, 64)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    cu = torch.tensor(ends, device="cuda")

    def attend():
        return flash_attn_packed_func(*(x * 1.0 for x in leaves), cu)

    if how == "checkpoint":
        o = checkpoint(attend, use_reentrant=False)
    else:
        with torch.autograd.graph.save_on_cpu():
            o = attend()
    trash = [torch.full((T, 4, 64), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(32)]
    want = packed(q, k, v, ends, True, do)
    for name, x in zip(("o", "dq", "dk", "dv"), (o.detach(), *torch.autograd.grad(o, leaves, do))):
        check(x, want, name)
    del trash


def test_saved_tensors_that_do_not_fit_are_refused():
    """Tensors that got other data behind the forward pass: no kernel reads beyond what they have now."""
    from neuronx_distributed_llama3_2_b200.ops.attention import flash_attn_packed_func

    T, ends = 300, [0, 120, 290]
    q, k, v, do = (x.contiguous() for x in _inputs(T, 4, 2, 64))
    cu = torch.tensor(ends, device="cuda")
    for at in range(3):
        for other in (lambda x: x[:7].clone(), lambda x: x[:, :1].clone(), lambda x: x[..., :32].clone(), lambda x: x.float(), lambda x: x.cpu()):
            leaves = [x.clone().requires_grad_() for x in (q, k, v)]
            args = [x * 1.0 for x in leaves]
            o = flash_attn_packed_func(*args, cu)
            args[at].data = other(args[at].data)
            with pytest.raises(RuntimeError, match="have become"):
                torch.autograd.grad(o, leaves, do)


def test_entry_points_refuse_what_is_missing():
    import ctypes as c

    from neuronx_distributed_llama3_2_b200.ops import _lib

    x = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda" if torch.cuda.is_available() else "cpu")
    lib, at = _lib.lib(), c.c_void_p(x.data_ptr() + (-x.data_ptr() & 15))
    nothing, n = c.c_void_p(None), c.c_longlong
    plan = [at, c.c_int(0), c.c_int(1), n(100), c.c_int(1), c.c_int(128), at, at, at, nothing]
    for i in (0, 6, 7, 8):
        assert lib.nxd_packed_plan(*[nothing if j == i else a for j, a in enumerate(plan)]) == -1 and b"missing" in lib.nxd_last_error()
    strides = (n * 16)(*([64] * 16))
    sizes = lambda rows, columns: (n(rows), c.c_int(2), n(columns), n(100))                 # noqa: E731
    tail = (c.c_int(1), c.c_int(1), c.c_int(64), c.c_float(1.0), c.c_int(1), c.c_int(-1), nothing)
    for which, rows in ((nothing, 128), (at, 64)):
        assert lib.nxd_packed_attn_fwd(at, at, at, at, at, at, strides, at, which, *sizes(rows, 192), *tail) == -1
        assert b"rows of what" in lib.nxd_last_error()
        assert lib.nxd_packed_attn_bwd(at, at, at, at, at, at, at, at, at, nothing, at, at, at, strides, at, which, *sizes(rows, 192), c.c_int(1),
                                       *tail) == -1
        assert b"rows of what" in lib.nxd_last_error()


def test_tables_shorter_than_the_row():
    """Rotation tables as long as the longest sequence are enough, and a sequence that is longer reads no further."""
    from neuronx_distributed_llama3_2_b200.ops import attention, rope

    T, D = 400, 64
    qkv = torch.randn(T, 8, D, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").bfloat16()
    cos, sin = rope.build_rope_cache(T, D, 10000.0, None, device="cuda")
    cu = torch.tensor([0, 200, 400], device="cuda")
    whole = attention.rope_flash_attn_packed_func(qkv, cos, sin, 4, 2, cu)
    assert torch.equal(whole, attention.rope_flash_attn_packed_func(qkv, cos[:200], sin[:200], 4, 2, cu))
    short = attention.rope_flash_attn_packed_func(qkv, cos[:150], sin[:150], 4, 2, cu)
    assert short.isfinite().all() and torch.equal(short[:150], whole[:150])


@pytest.mark.parametrize("D", [64, 128])
def test_rotation_and_attention(D):
    from neuronx_distributed_llama3_2_b200.ops import attention, rope

    T, H, G, ends = 500, 4, 2, [0, 1, 200, 470]
    g = torch.Generator(device="cuda").manual_seed(D)
    qkv = torch.randn(T, H + 2 * G, D, generator=g, device="cuda").bfloat16().requires_grad_()
    do = torch.randn(T, H, D, generator=g, device="cuda").bfloat16()
    cos, sin = rope.build_rope_cache(T, D, 10000.0, None, device="cuda")
    o = attention.rope_flash_attn_packed_func(qkv, cos, sin, H, G, torch.tensor(ends, device="cuda"))
    (grad,) = torch.autograd.grad(o, qkv, do)
    positions = torch.cat([torch.arange(b - a, device="cuda") for a, b in zip([0] + ends, ends + [T])])
    turn = lambda x, back: rope.rope_ref(x, cos.double(), sin.double(), H + G, 1, 1, positions, inverse=back)     # noqa: E731
    r = turn(qkv.detach().double(), False)
    want = packed(r[:, :H], r[:, H:H + G], r[:, H + G:], ends, True, do)
    back = turn(torch.cat([want[n][0] for n in ("dq", "dk", "dv")], 1), True)
    # roundings to bf16, 2^-8 of a value each: forward the rotated heads, the weights and the result; backward also the score gradients,
    # the three gradients, and their rotation back
    assert (o.double() - want["o"][0]).norm() <= 3 * 2.0 ** -8 * want["o"][0].norm()
    assert (grad.double() - back).norm() <= 6 * 2.0 ** -8 * back.norm()
    assert not o[470:].any() and not grad[470:].any()


def test_forward_mode_is_refused():
    """Not taken as a call without derivatives, with autograd on and off."""
    import torch.autograd.forward_ad as fw
    from neuronx_distributed_llama3_2_b200.ops.attention import flash_attn_packed_func

    q, k, v, _ = _inputs(100, 4, 2, 64)
    cu = torch.tensor([0, 60, 100], device="cuda")
    with fw.dual_level():
        for on in (True, False):
            for at in range(3):
                args = [fw.make_dual(x, torch.ones_like(x)) if i == at else x for i, x in enumerate((q, k, v))]
                with torch.set_grad_enabled(on), pytest.raises((NotImplementedError, RuntimeError), match="jvp"):
                    flash_attn_packed_func(*args, cu)
        assert flash_attn_packed_func(q, k, v, cu).isfinite().all()
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: flash_attn_packed_func(x, k, v, cu), (q,), (q,))


def test_other_types_take_one_sequence_after_the_other():
    q, k, v, do = (x.float() for x in _inputs(130, 4, 2, 64))
    ends = [0, 60, 120]
    got, want = _run(q, k, v, do, ends, True), packed(q, k, v, ends, True, do)
    for name in got:          # at most 60 products, 2^-24 each, numbers below 8
        assert (got[name].double() - want[name][0]).abs().max() <= 2.0 ** -24 * 60 * 64
