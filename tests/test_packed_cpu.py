"""Attention over packed sequences without a GPU: the formula's gradients, the path of other types, refusals."""
import pytest
import torch

from packed_oracle import packed

from neuronx_distributed_llama3_2_b200.ops import attention
from neuronx_distributed_llama3_2_b200.ops.packed_attention import PackedSequences


def _inputs(T, H, G, D, dtype=torch.float64):
    g = torch.Generator().manual_seed(T)
    return [torch.randn(T, h, D, generator=g, dtype=torch.float64).to(dtype) for h in (H, G, G, H)]


@pytest.mark.parametrize("causal", [True, False])
def test_oracle_gradients_are_differences(causal):
    q, k, v, do = _inputs(9, 4, 2, 8)
    ends, step = [0, 1, 1, 6, 8], 1e-6
    want = packed(q, k, v, ends, causal, do)
    g = torch.Generator().manual_seed(1)
    for i, name in enumerate(("dq", "dk", "dv")):
        d = torch.randn(*(q, k, v)[i].shape, generator=g, dtype=torch.float64)
        ahead, back = ([x + s * step * d if j == i else x for j, x in enumerate((q, k, v))] for s in (1, -1))
        slope = ((packed(*ahead, ends, causal)["o"][0] - packed(*back, ends, causal)["o"][0]) * do).sum() / (2 * step)
        # central difference: error step^2 in the third derivative (about 1e-12 here) and 1e-16 / step of rounding, sums of ~100 terms
        assert abs(slope - (want[name][0] * d).sum()) <= 1e-7


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("ends", [[0, 9], [0, 1, 1, 6, 8], [2, 3, 7], [0], [4, 4]])
def test_fp32_path(ends, causal):
    q, k, v, do = (x.requires_grad_() for x in _inputs(9, 4, 2, 8, torch.float32))
    o = attention.flash_attn_packed_func(q, k, v, torch.tensor(ends), causal=causal)
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, (q, k, v), do)), o=o)
    want = packed(q, k, v, ends, causal, do.detach())
    for name, x in got.items():          # sums of at most 9 products of numbers below 4, a softmax in between: 2^-24 each
        assert (x.double() - want[name][0]).abs().max() <= 2.0 ** -24 * 9 * 64


def test_positions_start_again():
    p = PackedSequences(torch.tensor([1, 4, 4, 6], dtype=torch.int32), 8)
    assert p.positions().tolist() == [0, 0, 1, 2, 0, 1, 0, 0]
    assert p.inside().tolist() == [False] + [True] * 5 + [False] * 2
    assert p.last_tokens().tolist() == [True, False, False, True, False, True, True, True]


def test_rotation_restarts_in_every_sequence():
    from neuronx_distributed_llama3_2_b200.ops.rope import build_rope_cache

    g = torch.Generator().manual_seed(0)
    qkv = torch.randn(11, 8, 16, generator=g)
    cos, sin = build_rope_cache(11, 16, 10000.0)
    o = attention.rope_flash_attn_packed_func(qkv, cos, sin, 4, 2, torch.tensor([0, 5, 11]))
    for a, b in ((0, 5), (5, 11)):
        alone = attention.rope_flash_attn_func(qkv[a:b, None], cos, sin, 4, 2)[0].transpose(0, 1)
        assert torch.equal(o[a:b], alone)


@pytest.mark.parametrize("cu", [torch.tensor([0, 5, 3]), torch.tensor([-1, 4]), torch.tensor([0, 10]), torch.tensor([0.0, 4.0]),
                                torch.tensor([[0, 4]]), torch.tensor([], dtype=torch.int32)])
def test_bad_boundaries_are_refused(cu):
    q, k, v, _ = _inputs(9, 4, 2, 8, torch.float32)
    with pytest.raises(ValueError):
        attention.flash_attn_packed_func(q, k, v, cu)


def test_bad_tensors_are_refused():
    q, k, v, _ = _inputs(9, 4, 2, 8, torch.float32)
    cu = torch.tensor([0, 9])
    for bad in ((q[:, :3], k, v), (q[:8], k, v), (q, k, v[:, :1]), (q[..., :4], k, v), (q[0], k, v), (q.double(), k, v),
                (q, k[:, :0], v[:, :0]), (q[:0], k[:0], v[:0])):
        with pytest.raises(ValueError):
            attention.flash_attn_packed_func(*bad, cu)
    with pytest.raises(ValueError):
        attention.flash_attn_packed_func(q, k, v, PackedSequences(torch.tensor([0, 4]), 8))
    with pytest.raises(ValueError):
        attention.rope_flash_attn_packed_func(q, None, None, 2, 2, cu)


@pytest.mark.parametrize("scale", [0.0, -0.5, -2.0])
def test_scales_that_are_not_positive(scale):
    q, k, v, do = (x.requires_grad_() for x in _inputs(9, 4, 2, 8, torch.float32))
    o = attention.flash_attn_packed_func(q, k, v, torch.tensor([0, 4, 9]), softmax_scale=scale)
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, (q, k, v), do)), o=o)
    want = packed(q, k, v, [0, 4, 9], True, do.detach(), scale)
    for name, x in got.items():          # as in the test of the fp32 path, with scores up to six times as large
        assert (x.double() - want[name][0]).abs().max() <= 2.0 ** -24 * 9 * 64 * 6


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 1e-39, 3e38, 1e300])
def test_bad_scales_are_refused(scale):
    q, k, v, _ = _inputs(9, 4, 2, 8, torch.float32)
    with pytest.raises(ValueError):
        attention.flash_attn_packed_func(q, k, v, torch.tensor([0, 9]), softmax_scale=scale)


def test_captures_that_are_over_are_let_go(monkeypatch):
    """A long-lived object keeps what the last capture of each stream made, and what the streams share without one."""
    import weakref

    p = PackedSequences(torch.tensor([0, 4, 9]), 9)
    here = {"at": (1, 0)}
    monkeypatch.setattr(p, "_here", lambda: here["at"])
    eager = p.positions()
    made = []
    for capture in range(1, 20):
        for stream in (1, 2):
            here["at"] = (stream, capture)
            x = p.positions()
            assert x is p.positions() and x.tolist() == eager.tolist() and x is not eager
            made.append(weakref.ref(x))
            del x
    assert sum(r() is not None for r in made) == 2 and all(r() is not None for r in made[-2:])
    here["at"] = (1, 0)
    assert p.positions() is eager


def test_bad_tables_are_refused():
    qkv, cu = torch.randn(9, 8, 16), torch.tensor([0, 4, 9])
    table = torch.ones(9, 8)
    short, half, odd = torch.ones(4, 8), table.half(), torch.ones(9, 4)
    for cos, sin in ((odd, odd), (table, short), (half, half), (short, short), (table[:0], table[:0])):
        with pytest.raises(ValueError):
            attention.rope_flash_attn_packed_func(qkv, cos, sin, 4, 2, cu)
    attention.rope_flash_attn_packed_func(qkv, table[:5], table[:5], 4, 2, cu)


def test_first_tokens():
    assert PackedSequences(torch.tensor([1, 4, 4, 6]), 8).first_tokens().tolist() == [1, 4, 4]
    assert PackedSequences(torch.tensor([0, 8, 8]), 8).first_tokens().tolist() == [0, 7]
    assert PackedSequences(torch.tensor([3]), 8).first_tokens().tolist() == []
