# Copyright 2026. Licensed under the Apache License, Version 2.0.
"""BERT on packed batches: packed attention, layer norm and counter-based
dropout together, as a model runs them."""

import copy

import pytest
import torch

from bluefog_amd import models


def _tiny_bert(dropout=0.0):
    torch.manual_seed(3)
    return models.BertForMaskedLM(
        models.BertConfig(vocab_size=97, hidden_size=64, num_hidden_layers=2, num_attention_heads=4,
                          intermediate_size=128, max_position_embeddings=40, dropout=dropout)
    )


def _packed_batch(device):
    lengths = [7, 40, 1, 0, 23]
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(0, 97, (sum(lengths) + 3,), generator=g)
    labels = torch.where(torch.rand(ids.shape, generator=g) < 0.3, ids, -100)
    labels[sum(lengths):] = -100
    cu = torch.tensor([0] + lengths).cumsum(0).to(torch.int32)
    return lengths, ids.to(device), labels.to(device), cu


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_bert_packed_matches_its_sequences_alone(device):
    """Logits, loss and gradients of a packed batch against the dense model on
    each sequence by itself, in 64 bits. The packed run is 32-bit: two blocks of
    sums of at most 128 terms around values of size 1 keep six digits of the
    largest."""
    model = _tiny_bert().to(device)
    lengths, ids, labels, cu = _packed_batch(device)
    exact = copy.deepcopy(model).cpu().double()
    logits, at = [], 0
    for n in lengths:
        if n:
            logits.append(exact(ids[None, at:at + n].cpu())[0])
        at += n
    logits = torch.cat(logits)
    loss = torch.nn.functional.cross_entropy(logits, labels[:at].cpu(), ignore_index=-100)
    loss.backward()
    got = model(ids, cu_seqlens=cu)
    assert (got[:at].cpu().double() - logits).abs().max() < 1e-5 * logits.abs().max()
    got = model(ids, labels=labels, cu_seqlens=cu)
    assert abs(got.item() - loss.item()) < 1e-5 * loss.item()
    got.backward()
    for a, b in zip(model.parameters(), exact.parameters()):
        assert (a.grad.cpu().double() - b.grad).abs().max() <= 2e-5 * b.grad.abs().max() + 1e-9


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_bert_packed_dropout(device):
    """Masks follow torch's seed; evaluation has none; every gradient is there."""
    model = _tiny_bert(0.2).to(device)
    lengths, ids, labels, cu = _packed_batch(device)
    used = slice(0, sum(lengths))

    def run():
        torch.manual_seed(11)
        return model(ids, cu_seqlens=cu.to(device))[used]

    first = run()
    assert torch.equal(first, run())
    assert not torch.equal(first, model(ids, cu_seqlens=cu)[used])
    loss = model(ids, labels=labels, cu_seqlens=cu)
    loss.backward()
    assert all(torch.isfinite(p.grad).all() for p in model.parameters())
    model.eval()
    quiet = model(ids, cu_seqlens=cu)[used]
    assert torch.equal(quiet, model(ids, cu_seqlens=cu)[used])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_bert_packed_half_precision(dtype):
    """Under autocast the residual stream is 32-bit under half-precision
    branches; a model of that type runs as well. Both stay within the type's
    roundings of the 32-bit run: u = eps / 2 of values of size 4 at each of
    eight roundings of the two blocks and the head, whose width of 64 makes the
    errors of independent terms add up like their root, and a factor of 4."""
    model = _tiny_bert().cuda().eval()
    lengths, ids, _, cu = _packed_batch("cuda")
    used = slice(0, sum(lengths))
    with torch.no_grad():
        want = model(ids, cu_seqlens=cu)[used]
        with torch.autocast("cuda", dtype=dtype):
            a = model(ids, cu_seqlens=cu)[used]
        b = copy.deepcopy(model).to(dtype)(ids, cu_seqlens=cu)[used]
    bound = torch.finfo(dtype).eps / 2 * 4 * 8 * 4
    assert (a.float() - want).abs().max() < bound and (b.float() - want).abs().max() < bound


@pytest.mark.gpu
def test_bert_packed_in_a_captured_step():
    """A captured training step against the eager one, with new tokens, labels
    and lengths at every replay."""
    model = _tiny_bert().cuda()
    lengths, ids, labels, cu = _packed_batch("cuda")
    cu = cu.cuda()
    params = list(model.parameters())

    def step():
        loss = model(ids, labels=labels, cu_seqlens=cu)
        return [loss.detach(), *torch.autograd.grad(loss, params)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for n in range(4):
        ids.copy_(torch.randint(0, 97, ids.shape))
        labels.copy_(torch.where(torch.rand(ids.shape) < 0.5, torch.randint(0, 97, ids.shape), -100))
        cu.copy_(torch.tensor([0, 3 + n, 30, 30, 55, 60 + n]))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in got]
        # the library's sums over the embeddings' rows have no fixed order
        for a, b in zip(replayed, step()):
            assert (a - b).abs().max() <= 1e-5 * b.abs().max() + 1e-8


def test_bert_packed_refusals():
    model = _tiny_bert()
    ids = torch.zeros(50, dtype=torch.int64)

    def refused(match, ids, cu):
        with pytest.raises(ValueError, match=match):
            model(ids, cu_seqlens=cu)

    def ends(*v):
        return torch.tensor(v, dtype=torch.int32)

    refused("one row", ids[None], ends(0, 50))
    refused("int32", ids, ends(0, 30).long())
    refused("rise", ids, ends(0, 51))
    refused("rise", ids, ends(0, 20, 10))
    refused("rise", ids, ends(1, 20))
    refused("does not fit", ids, ends(0, 41))


@pytest.mark.gpu
def test_bert_packed_tokens_in_front_of_the_first_sequence():
    """Bounds on the GPU are not checked: those that start late leave what is in
    front of them without meaning, and the sequence as it is."""
    model = _tiny_bert().cuda().eval()
    ids = torch.randint(0, 97, (60,), generator=torch.Generator().manual_seed(2)).cuda()
    with torch.no_grad():
        got = model(ids, cu_seqlens=torch.tensor([13, 50], dtype=torch.int32, device="cuda"))[13:50]
        alone = model(ids[13:50], cu_seqlens=torch.tensor([0, 37], dtype=torch.int32))
    assert (got - alone).abs().max() < 1e-5 * alone.abs().max()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_bert_packed_modes_and_rates_of_its_modules(device):
    """A module in evaluation, or with a probability of its own, drops what it
    says, not what the model was made with."""
    model = _tiny_bert(0.2).to(device)
    lengths, ids, _, cu = _packed_batch(device)
    used = slice(0, sum(lengths))

    def run():
        torch.manual_seed(7)
        return model(ids, cu_seqlens=cu)[used]

    quiet = model.eval()(ids, cu_seqlens=cu)[used]
    model.train()
    dropped = run()
    for part in (model.embeddings, model.layers):
        part.eval()
    assert torch.equal(run(), quiet)
    model.train()
    for m in model.modules():
        if isinstance(m, torch.nn.Dropout):
            m.p = 0.0
        if hasattr(m, "dropout_p"):
            m.dropout_p = 0.0
    assert torch.equal(run(), quiet)
    model.layers[1].dropout.p = 0.5
    half = run()
    assert not torch.equal(half, quiet) and not torch.equal(half, dropped)
    model.layers[1].dropout = torch.nn.Identity()
    assert torch.equal(run(), quiet)
    model.layers[1].dropout = torch.nn.Dropout1d(0.1)
    with pytest.raises(TypeError, match="Dropout1d"):
        run()


def test_bert_packed_calls_its_modules():
    """Hooks of every module run, but for those of nn.Dropout, and what a hook
    returns takes part."""
    model = _tiny_bert(0.2)
    _, ids, _, cu = _packed_batch("cpu")
    called = []
    for name, m in model.named_modules():
        m.register_forward_hook(lambda m, args, out, name=name: called.append(name))
    model(ids, cu_seqlens=cu)
    idle = {n for n, m in model.named_modules() if isinstance(m, (torch.nn.Dropout, torch.nn.ModuleList))}
    # the position table's and the types' modules are called too
    assert set(called) == {n for n, _ in model.named_modules()} - idle
    model.eval()
    before = model(ids, cu_seqlens=cu)
    model.layers[0].norm1.register_forward_hook(lambda m, args, out: out * 2)
    assert not torch.equal(model(ids, cu_seqlens=cu), before)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_bert_packed_without_the_fused_norm(device, monkeypatch):
    """BLUEFOG_FUSED_LN=0 takes the norm operator out of the packed path; the
    masks are the same. Both norms are 32-bit sums of 64 terms."""
    from bluefog_amd.ops import transformer

    model = _tiny_bert(0.2).to(device)
    lengths, ids, _, cu = _packed_batch(device)
    used = slice(0, sum(lengths))

    def run():
        torch.manual_seed(7)
        return model(ids, cu_seqlens=cu)[used]

    want = run()
    monkeypatch.setenv("BLUEFOG_FUSED_LN", "0")
    monkeypatch.setattr(transformer, "layer_norm", None)
    assert (run() - want).abs().max() < 1e-5 * want.abs().max()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_bert_packed_empty_batch(device):
    model = _tiny_bert(0.1).to(device)
    out = model(torch.zeros(0, dtype=torch.int64, device=device), cu_seqlens=torch.zeros(1, dtype=torch.int32))
    assert out.shape == (0, 97)
    out.sum().backward()
    assert all(not p.grad.any() for p in model.parameters() if p.grad is not None)


def _attentive_bert():
    """Attention outweighs the residual: its weights are ten times as large, so
    that scores have a size of 2 and its branch one of 2 beside a residual of 1."""
    model = _tiny_bert().eval()
    with torch.no_grad():
        for layer in model.layers:
            for part in (layer.attn.qkv, layer.attn.out):
                part.weight *= 10
    return model


def _off(got, want):
    return float((got.double().cpu() - want).norm() / want.norm())


def _half_bound(dtype):
    """The relative error of the logits: 8 roundings in each of two blocks and one
    of the head, each of u = eps / 2 of its value at most, add up like their root;
    norms, softmax and the larger weights pass on at most 4 times as much."""
    return torch.finfo(dtype).eps / 2 * 17 ** 0.5 * 4


@pytest.mark.parametrize("mistake", ["no attention", "causal"])
def test_bert_packed_half_precision_bound_tells(mistake, monkeypatch):
    """An attention that gives nothing, or that is causal, is far outside of it."""
    from bluefog_amd.ops import transformer

    model = _attentive_bert().double()
    lengths, ids, _, cu = _packed_batch("cpu")
    used, right = slice(0, sum(lengths)), transformer.packed_attention
    with torch.no_grad():
        want = model(ids, cu_seqlens=cu)[used]
        monkeypatch.setattr(transformer, "packed_attention", lambda q, *a, **kw: (
            torch.zeros_like(q) if mistake == "no attention" else right(q, *a, **kw, causal=True)))
        off = _off(model(ids, cu_seqlens=cu)[used], want)
    assert off > 4 * _half_bound(torch.bfloat16)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_bert_packed_half_precision_where_attention_counts(device, dtype):
    model = _attentive_bert()
    lengths, ids, _, cu = _packed_batch(device)
    used = slice(0, sum(lengths))
    with torch.no_grad():
        want = copy.deepcopy(model).double()(ids.cpu(), cu_seqlens=cu)[used]
        model = model.to(device)
        with torch.autocast(device, dtype=dtype):
            a = model(ids, cu_seqlens=cu)[used]
        rounded = model.to(dtype)
        b = rounded(ids, cu_seqlens=cu)[used]
        # weights of the type are other weights: they have a result of their own
        want_b = copy.deepcopy(rounded).cpu().double()(ids.cpu(), cu_seqlens=cu)[used]
    assert _off(a, want) < _half_bound(dtype) and _off(b, want_b) < _half_bound(dtype)


@pytest.mark.gpu
def test_bert_packed_captured_dropout():
    """A captured step draws new masks at every replay, the same ones in its
    forward and backward pass: replayed from torch's seed it repeats the eager
    step."""
    model = _tiny_bert(0.3).cuda()
    _, ids, labels, cu = _packed_batch("cuda")
    cu, params = cu.cuda(), list(model.parameters())

    def step():
        loss = model(ids, labels=labels, cu_seqlens=cu)
        return [loss.detach(), *torch.autograd.grad(loss, params)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    losses = []
    for n in range(4):
        torch.manual_seed(20 + n)
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in got]
        losses.append(replayed[0].item())
        torch.manual_seed(20 + n)
        # the library's sums over the embeddings' rows have no fixed order
        for a, b in zip(replayed, step()):
            assert (a - b).abs().max() <= 1e-5 * b.abs().max() + 1e-8
    assert len(set(losses)) == 4
