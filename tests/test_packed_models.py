"""Models on packed rows: samples end to end give what they give one by one, and attention, LoRA dropout and the balance loss work
together in one training step."""
import json
import math
import os
import subprocess
import sys

import pytest
import torch

from packed_oracle import check, packed as packed_attention
from neuronx_distributed_llama3_2_b200 import models as M
from neuronx_distributed_llama3_2_b200.models.bert import BertForPreTraining, tiny_bert
from neuronx_distributed_llama3_2_b200.modules.lora import LoraConfig, get_lora_model
from neuronx_distributed_llama3_2_b200.modules.moe import load_balancing_loss_func
from neuronx_distributed_llama3_2_b200.ops import attention, dropout
from neuronx_distributed_llama3_2_b200.ops.packed_attention import PackedSequences
from neuronx_distributed_llama3_2_b200.utils import data

ENDS, ROW = [0, 7, 8, 8, 30], 33            # a sample of one token, an empty one, three columns of padding
# Two orders of the same fp32 sums: about 40 operations from the ids to a gradient and back, sums of up to 512 products (whose error
# grows as their square root, 23), 2^-24 each.
FP32 = 40 * 23 * 2.0 ** -24


def _near(a, b, what):
    assert (a - b).abs().max() <= FP32 * max(b.abs().max().item(), 1e-3), (what, (a - b).abs().max().item(), b.abs().max().item())


def _grads(model):
    out = {n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None}
    model.zero_grad(set_to_none=True)
    return out


def _compare(got, want):
    assert got.keys() == want.keys()
    for n in want:
        _near(got[n], want[n], n)


@pytest.mark.parametrize("ckpt", [False, True])
@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
def test_llama_row_of_samples(ckpt, wide):
    torch.manual_seed(3)
    model = M.LlamaForCausalLM(M.tiny_llama(activation_checkpointing=ckpt)).train()
    ids = torch.randint(0, 512, (1, ROW))
    labels = torch.where(torch.rand(1, ROW) < 0.2, -100, ids)
    cu = torch.tensor(ENDS, dtype=wide)
    loss = model(ids, labels, cu_seqlens=cu)
    loss.backward()
    got = _grads(model)
    total, count = 0.0, 0
    for a, b in zip(ENDS, ENDS[1:]):
        if b > a + 1:
            n = int((labels[0, a + 1:b] >= 0).sum())
            total, count = total + model(ids[:, a:b], labels[:, a:b]) * n, count + n
    (total / count).backward()
    _near(loss, (total / count).detach(), "loss")
    _compare(got, _grads(model))
    logits = model(ids, cu_seqlens=PackedSequences(cu, ROW))
    for a, b in zip(ENDS, ENDS[1:]):
        if b > a:
            _near(logits[a:b], model(ids[:, a:b]), "logits")


@pytest.mark.parametrize("make,config", [(M.MixtralForCausalLM, M.tiny_mixtral), (M.DbrxForCausalLM, M.tiny_dbrx)])
def test_experts_row_of_samples(make, config):
    torch.manual_seed(4)
    cfg = config(capacity_factor=None)
    model = make(cfg).train()
    seen = []
    for layer in model.layers:
        layer.register_forward_hook(lambda m, i, o: seen.append(o[2]))
    ids = torch.randint(0, cfg.vocab_size, (1, ROW))
    loss = model(ids, ids, cu_seqlens=torch.tensor(ENDS))
    loss.backward()
    got = _grads(model)
    seen.clear()
    total, count = 0.0, 0
    for a, b in zip(ENDS, ENDS[1:]):
        if b > a:
            total = total + model.loss_fn(model(ids[:, a:b]), ids[:, a:b]) * (b - a - 1)
            count += b - a - 1
    layers = len(model.layers)
    joined = [torch.cat([t.reshape(-1, cfg.num_local_experts) for t in seen[i::layers]]) for i in range(layers)]
    want = total / count + cfg.router_aux_loss_coef * load_balancing_loss_func(joined, cfg.num_local_experts, cfg.num_experts_per_tok)
    want.backward()
    _near(loss, want.detach(), "loss")
    _compare(got, _grads(model))


def test_bert_row_of_sentences():
    torch.manual_seed(5)
    model = BertForPreTraining(tiny_bert()).train()
    ends = [0, 9, 10, 30]
    ids, types = torch.randint(0, 512, (1, ROW)), torch.randint(0, 2, (1, ROW))
    labels = torch.where(torch.rand(1, ROW) < 0.5, ids, -100)
    labels[:, 30:] = -100
    nsp = torch.tensor([1, 0, 1])
    loss = model(ids, types, labels=labels, next_sentence_label=nsp, cu_seqlens=torch.tensor(ends))
    loss.backward()
    got = _grads(model)
    total, count, pairs = 0.0, int((labels >= 0).sum()), []
    for s, (a, b) in enumerate(zip(ends, ends[1:])):
        n = int((labels[:, a:b] >= 0).sum())
        total = total + model(ids[:, a:b], types[:, a:b], labels=labels[:, a:b]) * n
        pairs.append(model(ids[:, a:b], types[:, a:b])[1])
    want = total / count + torch.nn.functional.cross_entropy(torch.cat(pairs), nsp)
    want.backward()
    _near(loss, want.detach(), "loss")
    _compare(got, _grads(model))


def test_dropout_of_a_checkpoint_file_stays_unread():
    from neuronx_distributed_llama3_2_b200.models.llama import config_from_json

    cfg = config_from_json(type(tiny_bert()), {"hidden_size": 128, "hidden_dropout_prob": 0.1, "attention_probs_dropout_prob": 0.1})
    assert cfg.residual_dropout == 0.0 and cfg.hidden_size == 128


def test_bert_hidden_dropout():
    cfg = tiny_bert(residual_dropout=0.3)
    torch.manual_seed(6)
    model = BertForPreTraining(cfg)
    torch.manual_seed(6)
    plain = BertForPreTraining(tiny_bert())
    ids = torch.randint(0, 512, (2, 16))
    assert torch.equal(model.eval()(ids)[0], plain.eval()(ids)[0])
    model.train()
    torch.manual_seed(7)
    one = model(ids, labels=ids)
    torch.manual_seed(7)
    assert torch.equal(one, model(ids, labels=ids)) and not torch.equal(one, model(ids, labels=ids))
    torch.manual_seed(7)
    one.backward()
    want = _grads(model)
    cfg.activation_checkpointing = True                  # the repeated forward pass draws the same masks
    torch.manual_seed(7)
    model(ids, labels=ids).backward()
    got = _grads(model)
    for n in want:
        assert torch.equal(got[n], want[n]), n


@pytest.mark.parametrize("family", ["llama", "mixtral", "bert"])
def test_pipelines_trace_models_without_packed_rows(family):
    from neuronx_distributed_llama3_2_b200.models.bert import BertLayer
    from neuronx_distributed_llama3_2_b200.models.llama import LlamaDecoderLayer
    from neuronx_distributed_llama3_2_b200.models.mixtral import MixtralDecoderLayer
    from neuronx_distributed_llama3_2_b200.pipeline.model import NxDPPModel
    from neuronx_distributed_llama3_2_b200.pipeline.trace import trace_model

    make, config, layer = {"llama": (M.LlamaForCausalLM, M.tiny_llama, LlamaDecoderLayer), "bert": (BertForPreTraining, tiny_bert, BertLayer),
                           "mixtral": (M.MixtralForCausalLM, M.tiny_mixtral, MixtralDecoderLayer)}[family]
    torch.manual_seed(1)
    model = make(config())
    ids = torch.randint(0, 512, (1, 8))
    want = model(ids, labels=ids)
    everything = trace_model(model, leaf_modules=[layer])                  # as inputs, but those that have to be named
    if family != "bert":                                                    # whose graph then takes a mask and token types
        assert torch.equal(everything(ids, labels=ids), want)
    traced = trace_model(model, input_names=["input_ids", "labels"], leaf_modules=[layer])
    assert torch.equal(traced(input_ids=ids, labels=ids), want)
    with pytest.raises(NotImplementedError):
        trace_model(model, input_names=["input_ids", "labels", "cu_seqlens"], leaf_modules=[layer])
    pipe = NxDPPModel.__new__(NxDPPModel)
    torch.nn.Module.__init__(pipe)
    pipe.original_torch_module, pipe.input_names, pipe.num_microbatches = model, None, 1
    with pytest.raises(ValueError, match="cu_seqlens"):
        pipe._split_microbatches({"input_ids": ids, "cu_seqlens": torch.tensor([0, 8])})
    assert pipe._split_microbatches({"input_ids": ids, "cu_seqlens": None})[0]["input_ids"] is not None


def test_models_refuse():
    llama, bert = M.LlamaForCausalLM(M.tiny_llama()), BertForPreTraining(tiny_bert())
    cu, two, one = torch.tensor([0, 8]), torch.zeros(2, 8, dtype=torch.long), torch.zeros(1, 8, dtype=torch.long)
    with pytest.raises(ValueError, match="one row"):
        llama(two, cu_seqlens=cu)
    with pytest.raises(ValueError, match="packed in 8 rows"):
        llama(one[:, :6], cu_seqlens=PackedSequences(cu, 8))
    with pytest.raises(ValueError, match="rise"):
        llama(one, cu_seqlens=torch.tensor([0, 9]))
    with pytest.raises(ValueError, match="padding mask"):
        bert(one, attention_mask=torch.ones_like(one), cu_seqlens=cu)


class _Samples(torch.utils.data.Dataset):
    def __init__(self, lengths, seq_len):
        self.rows = [{"input_ids": torch.cat([torch.arange(n) + 100 * i, torch.zeros(seq_len - n, dtype=torch.long)]),
                      "labels": torch.cat([torch.arange(n) + 100 * i, torch.full((seq_len - n,), -100)]),
                      "attention_mask": (torch.arange(seq_len) < n).long()} for i, n in enumerate(lengths)]

    def __len__(self):
        return len(self.rows)

    def __getitem__(self, i):
        return self.rows[i]


def test_packed_samples():
    rows = data.PackedSamples(_Samples([5, 3, 4, 8, 1], 8), 8)
    assert [rows[i]["cu_seqlens"].tolist() for i in range(len(rows))] == [[0, 5, 8], [0, 4], [0, 8], [0, 1]]
    assert rows[0]["input_ids"].tolist() == [0, 1, 2, 3, 4, 100, 101, 102] and rows[1]["labels"].tolist() == [200, 201, 202, 203] + [-100] * 4
    mixed = data.PackedSamples(_Samples([5, 3, 4, 8, 1], 8), 8, shuffle=True, seed=1)
    assert sorted(i for r in mixed.rows for i in r) == [0, 1, 2, 3, 4]
    with pytest.raises(ValueError, match="8 tokens"):
        data.PackedSamples(_Samples([8], 8), 7)


def test_finetune_example_runs_on_packed_rows(tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    (tmp_path / "model").mkdir()
    (tmp_path / "data").mkdir()
    json.dump(dict(vocab_size=256, hidden_size=64, intermediate_size=128, num_hidden_layers=1, num_attention_heads=4, num_key_value_heads=2,
                   max_position_embeddings=512, rope_theta=1e4, tie_word_embeddings=False), open(tmp_path / "model" / "config.json", "w"))
    with open(tmp_path / "data" / "train.jsonl", "w") as f:
        for i in range(24):
            f.write(json.dumps({"instruction": f"say {i}", "input": "", "output": "x" * (1 + 7 * i % 50)}) + "\n")
    out = subprocess.run([sys.executable, os.path.join(root, "examples", "training", "tp_llama_finetune.py"), "--model_path",
                          str(tmp_path / "model" / "config.json"), "--data_dir", str(tmp_path / "data"), "--batch_size", "2", "--seq_len",
                          "256", "--max_steps", "2", "--pack", "1", "--counter_dropout", "1", "--lora_dropout", "0.1"],
                         capture_output=True, text=True, timeout=600, env={**os.environ, "CUDA_VISIBLE_DEVICES": ""}, cwd=tmp_path)
    assert out.returncode == 0, out.stdout[-2000:] + out.stderr[-2000:]


def _two_ranks(rank, world, sp):
    from test_llama_tp_cpu import _shard_from_full, _solo

    cu = torch.tensor([0, 7, 8, 8, 30])
    ids = torch.randint(0, 512, (1, 32), generator=torch.Generator().manual_seed(1))
    torch.manual_seed(3)
    with _solo():
        full = M.LlamaForCausalLM(M.tiny_llama(sequence_parallel_enabled=False))
        want = full(ids, ids, cu_seqlens=cu)
    model = M.LlamaForCausalLM(M.tiny_llama(sequence_parallel_enabled=sp))
    _shard_from_full(full, model, world, rank)
    got = model(ids, ids, cu_seqlens=cu)
    got.backward()
    assert abs(got - want) <= FP32 * want, (got, want)
    # a rank with a part of the input draws a mask of its own
    lora = _lora(model)
    offsets = {n.split(".")[-2]: m.offset for n, m in lora.named_modules() if isinstance(m, dropout.Dropout)}
    assert offsets == {"qkv_proj": rank if sp else 0, "o_proj": rank}, offsets
    # the first token of every sentence, wherever its row lives
    bert = BertForPreTraining(tiny_bert(sequence_parallel_enabled=sp))
    hidden = torch.arange(32.0).view(32, 1, 1).expand(32, 1, 128)
    mine = hidden.chunk(world)[rank] if sp else hidden
    packed = PackedSequences(torch.tensor([0, 7, 20, 32]), 32)
    assert bert._cls_token(mine.contiguous(), packed)[:, 0].tolist() == [0.0, 7.0, 20.0]


@pytest.mark.parametrize("sp", [False, True])
def test_two_ranks(sp):
    from conftest import run_distributed

    run_distributed(_two_ranks_entry, 2, sp)


def _two_ranks_entry(rank, world, sp):
    from neuronx_distributed_llama3_2_b200.parallel import parallel_state as ps

    if not ps.model_parallel_is_initialized():
        ps.initialize_model_parallel(tensor_model_parallel_size=world)
    _two_ranks(rank, world, sp)



def _two_ranks_gradients(rank, world, family, sp):
    from test_llama_tp_cpu import _shard_from_full, _solo
    from neuronx_distributed_llama3_2_b200.parallel import parallel_state as ps
    from neuronx_distributed_llama3_2_b200.parallel.grads import allreduce_sequence_parallel_gradients

    if not ps.model_parallel_is_initialized():
        ps.initialize_model_parallel(tensor_model_parallel_size=world)
    # every rank of a tensor-parallel group adds the balance loss's gradient to the routers' sum, with and without packed rows: left out
    make, config, kw = {"llama": (M.LlamaForCausalLM, M.tiny_llama, {}), "bert": (BertForPreTraining, tiny_bert, {}),
                        "mixtral": (M.MixtralForCausalLM, M.tiny_mixtral, {"capacity_factor": None, "router_aux_loss_coef": 0.0})}[family]
    g = torch.Generator().manual_seed(1)
    ends, row = [0, 7, 8, 20, 30], 32
    ids = torch.randint(0, 512, (1, row), generator=g)
    batch = {"input_ids": ids, "labels": ids, "cu_seqlens": torch.tensor(ends)}
    if family == "bert":
        labels = torch.where(torch.rand(1, row, generator=g) < 0.5, ids, -100)
        labels[:, ends[-1]:] = -100
        batch.update(labels=labels, token_type_ids=torch.randint(0, 2, (1, row), generator=g), next_sentence_label=torch.tensor([1, 0, 1, 1]))
    torch.manual_seed(3)
    with _solo():
        full = make(config(sequence_parallel_enabled=False, **kw)).train()
        want = full(**batch)
        want.backward()
    model = make(config(sequence_parallel_enabled=sp, **kw)).train()
    _shard_from_full(full, model, world, rank)
    got = model(**batch)
    got.backward()
    if sp:
        allreduce_sequence_parallel_gradients(list(model.parameters()))
    assert abs(got - want) <= FP32 * abs(want), (got, want)
    grads = {n: p.grad for n, p in model.named_parameters()}
    with torch.no_grad():          # the whole model's gradients, cut as its weights are
        for p in full.parameters():
            p.copy_(p.grad)
    _shard_from_full(full, model, world, rank)
    for n, p in model.named_parameters():
        _near(grads[n], p.detach(), n)


@pytest.mark.parametrize("family", ["llama", "mixtral", "bert"])
@pytest.mark.parametrize("sp", [False, True])
def test_two_ranks_gradients(family, sp):
    from conftest import run_distributed

    run_distributed(_two_ranks_gradients, 2, family, sp)


# -- on the GPU --------------------------------------------------------------------------------------------------------------
GPU_ENDS, GPU_ROW = [0, 130, 131, 131, 448, 700], 768


def _lora(model, p=0.1):
    model = get_lora_model(model, LoraConfig(enable_lora=True, lora_rank=8, lora_alpha=8, lora_dropout=p, counter_dropout=True,
                                             target_modules=["qkv_proj", "o_proj"]))
    gen = torch.Generator().manual_seed(9)
    with torch.no_grad():
        for n, w in model.named_parameters():
            if "lora_B" in n:
                w.copy_(torch.randn(w.shape, generator=gen) * 0.05)
    return model.train()


def test_lora_counter_dropout_on_a_packed_row():
    """The path without kernels: same seeds, same masks, in and outside of checkpointing."""
    grads = []
    for ckpt in (False, True):
        torch.manual_seed(8)
        model = _lora(M.LlamaForCausalLM(M.tiny_llama(activation_checkpointing=ckpt)))
        assert sum(isinstance(m, dropout.Dropout) for m in model.modules()) == 4
        ids = torch.randint(0, 512, (1, ROW), generator=torch.Generator().manual_seed(1))
        torch.manual_seed(11)
        model(ids, ids, cu_seqlens=torch.tensor(ENDS)).backward()
        grads.append(_grads(model))
    for n in grads[0]:
        assert "lora_" in n and grads[0][n].abs().max() > 0 and torch.equal(grads[0][n], grads[1][n]), n


@pytest.mark.gpu
@pytest.mark.parametrize("head_dim,kv", [(64, 2), (128, 1)])
def test_llama_lora_step_follows_fp32(head_dim, kv):
    """A fine-tuning step in bf16 on the kernels against the same step in fp32 without them, with the same dropout masks."""
    cfg = dict(hidden_size=256, head_dim=head_dim, num_attention_heads=4, num_key_value_heads=kv, max_position_embeddings=1024)
    ids = torch.randint(0, 512, (1, GPU_ROW), generator=torch.Generator().manual_seed(1))
    runs = []
    for dev, dt in (("cpu", torch.float32), ("cuda", torch.bfloat16)):
        torch.manual_seed(8)
        # the adapters are drawn in bf16 for both: another type draws other numbers
        model = _lora(M.LlamaForCausalLM(M.tiny_llama(**cfg)).bfloat16()).to(dev, dt)
        torch.manual_seed(11)
        loss = model(ids.to(dev), ids.to(dev), cu_seqlens=torch.tensor(GPU_ENDS, device=dev))
        loss.backward()
        runs.append((loss.detach().double().cpu(), {n: g.double().cpu() for n, g in _grads(model).items()}))
    # two layers of about 10 rounded tensors each way: 40 roundings of half a step of bf16 between the ids and a gradient
    bound = 40 * 2.0 ** -8
    assert abs(runs[0][0] - runs[1][0]) <= bound * runs[0][0]
    for n, want in runs[0][1].items():
        assert (runs[1][1][n] - want).norm() <= bound * want.norm(), (n, ((runs[1][1][n] - want).norm() / want.norm()).item())


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [4, 2])
def test_bert_step_follows_fp32(heads):
    """A pre-training step on a row of sentences in bf16 on the kernels against fp32 without them, with the same dropout masks."""
    ends, g = [0, 130, 131, 448, 700], torch.Generator().manual_seed(1)
    ids, types = torch.randint(0, 512, (1, GPU_ROW), generator=g), torch.randint(0, 2, (1, GPU_ROW), generator=g)
    labels = torch.where(torch.rand(1, GPU_ROW, generator=g) < 0.3, ids, -100)
    labels[:, ends[-1]:] = -100
    runs = []
    for dev, dt in (("cpu", torch.float32), ("cuda", torch.bfloat16)):
        torch.manual_seed(8)
        cfg = tiny_bert(hidden_size=256, num_attention_heads=heads, max_position_embeddings=512, residual_dropout=0.1)
        model = BertForPreTraining(cfg).bfloat16().to(dev, dt).train()
        torch.manual_seed(11)
        loss = model(ids.to(dev), types.to(dev), labels=labels.to(dev), next_sentence_label=torch.tensor([1, 0, 1, 1], device=dev),
                     cu_seqlens=torch.tensor(ends, device=dev))
        loss.backward()
        runs.append((loss.detach().double().cpu(), {n: g.double().cpu() for n, g in _grads(model).items()}))
    # about 10 rounded tensors a layer each way, 40 roundings of half a step of bf16 between the ids and a gradient
    bound = 40 * 2.0 ** -8
    assert abs(runs[0][0] - runs[1][0]) <= bound * runs[0][0]
    for n, want in runs[0][1].items():
        # a bias behind which nothing changes with it (of keys: the softmax does not see it) has a gradient of roundings alone
        if not n.endswith("query_key_value.bias"):
            assert (runs[1][1][n] - want).norm() <= bound * want.norm(), (n, ((runs[1][1][n] - want).norm() / want.norm()).item())


@pytest.mark.gpu
@pytest.mark.parametrize("ckpt", [False, True])
def test_experts_step_runs_all_operators(ckpt, monkeypatch):
    """One step of a model with experts and LoRA on a packed row: what each operator returned, against float64 of what it was given."""
    torch.manual_seed(8)
    cfg = M.tiny_mixtral(hidden_size=256, head_dim=64, capacity_factor=None, torch_dtype=torch.bfloat16, activation_checkpointing=ckpt,
                         max_position_embeddings=1024)
    model = _lora(M.MixtralForCausalLM(cfg, device=torch.device("cuda"))).cuda()
    calls = {"attention": [], "dropout": [], "balance": []}

    def tap(module, name, key):
        inner = getattr(module, name)

        def outer(*a, **kw):
            out = inner(*a, **kw)
            calls[key].append((a, out))
            return out
        monkeypatch.setattr(module, name, outer)

    from neuronx_distributed_llama3_2_b200.models import mixtral

    tap(attention, "rope_flash_attn_packed_func", "attention")
    tap(dropout, "dropout", "dropout")
    tap(mixtral, "load_balancing_loss_func", "balance")
    ids = torch.randint(0, 512, (1, GPU_ROW), generator=torch.Generator().manual_seed(1)).cuda()
    model(ids, ids, cu_seqlens=torch.tensor(GPU_ENDS, device="cuda")).backward()
    grads = _grads(model)
    trained = [n for n, p in model.named_parameters() if p.requires_grad]
    assert sorted(grads) == sorted(trained)
    assert all(torch.isfinite(g).all() and g.abs().max() > 0 for g in grads.values())
    times = 2 if ckpt else 1
    assert len(calls["attention"]) == 2 * times and len(calls["dropout"]) == 4 * times and len(calls["balance"]) == 1
    for (qkv, cos, sin, nq, nkv, seqs), o in calls["attention"]:
        x, pos = qkv.detach().double().cpu(), seqs.positions().long().cpu()
        c, s = (t.double().cpu()[pos][:, None] for t in (cos, sin))
        half = qkv.shape[-1] // 2
        rot = torch.cat([x[..., :half] * c - x[..., half:] * s, x[..., half:] * c + x[..., :half] * s], -1)
        q, k, v = rot[:, :nq], rot[:, nq:nq + nkv], x[:, nq + nkv:]
        want = packed_attention(q, k, v, GPU_ENDS, True)
        # rotated queries and keys are rounded once: a score is off by 2 x 2^-8 sum |q k| at most, a weight by the factor e^(2 that)
        for a, b in zip(GPU_ENDS, GPU_ENDS[1:]):
            for h in range(nq if b > a else 0):
                g = h // (nq // nkv)
                size = (q[a:b, h].abs() @ k[a:b, g].abs().T).amax(-1, keepdim=True) / math.sqrt(2 * half)
                want["o"][1][a:b, h] += torch.expm1(2 * 2 * 2.0 ** -8 * size) * v[a:b, g].abs().max()
        check(o.detach().cpu(), want, "o")
    for (x, p, *_), y in calls["dropout"]:
        kept = y != 0
        share = kept.float().sum() / (x != 0).sum()
        assert abs(share - (1 - p)) <= 6 * math.sqrt(p * (1 - p) / x.numel())
        want = x.double() / (1 - p)
        assert ((y.double() - want).abs()[kept] <= (2.0 ** -8 + 2.0 ** -22) * want.abs()[kept]).all()
    (logits, E, top, inside), loss = calls["balance"][0]
    rows = torch.stack([t.detach().double().reshape(-1, E)[inside] for t in logits]).reshape(-1, E)
    share = torch.nn.functional.one_hot(rows.topk(top, -1).indices, E).sum(1).double().mean(0)
    want = E / top * (share * torch.softmax(rows, -1).mean(0)).sum()
    assert inside.sum() == GPU_ENDS[-1] and abs(loss.double() - want) <= 2.0 ** -12 * want
