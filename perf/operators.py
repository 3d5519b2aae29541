# Copyright 2026. Licensed under the Apache License, Version 2.0.
"""Timing cases of the transformer training operators.

Three operators that a transformer block trains with, on batches whose
sequences lie one behind the other without padding:

- ``attention``: softmax(q k^T * scale) v inside each sequence, causal or
  not, with grouped key/value heads and dropout on the probabilities;
- ``layer_norm``: the norm over the last dimension of x, or of
  residual + dropout(x), with the gradients of weight and bias;
- ``dropout``: y = x * keep / (1 - p).

The dropout masks come from Philox4x32 with 7 rounds (Salmon, Moraes, Dror,
Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011), 16 bits to an
element, so a mask is a function of (seed, offset, position) alone.

``run`` computes a case in elementary torch operations where ``own`` is
false, and with ``bluefog_amd``'s operators where it is true.
"""

import math
import random

import torch

own = False

_TYPES = {
    "float32": torch.float32,
    "float16": torch.float16,
    "bfloat16": torch.bfloat16,
}
_M32 = 0xFFFFFFFF


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------


def _attention(dtype, heads, kv_heads, dim, seqs, longest, mix, spare, causal, p, train):
    return dict(op="attention", dtype=dtype, heads=heads, kv_heads=kv_heads,
                dim=dim, seqs=seqs, longest=longest, mix=mix, spare=spare,
                causal=causal, p=p, train=train)


def _layer_norm(dtype, residual, weights, rows, width, bias, p, train):
    return dict(op="layer_norm", dtype=dtype, residual=residual,
                weights=weights, rows=rows, width=width, bias=bias, p=p,
                train=train)


def _dropout(dtype, rows, width, p):
    return dict(op="dropout", dtype=dtype, rows=rows, width=width, p=p)


def listed():
    bf16, fp16, fp32 = "bfloat16", "float16", "float32"
    return [
        # the BERT-base benchmark's batch (64 sequences of up to 512 tokens,
        # 12 heads of 64), packed, a training step of one block's attention
        dict(_attention(bf16, 12, 12, 64, 64, 512, 5, 0, False, 0.1, True), name="attention bert bf16"),
        # the same model in the framework's default type, a small batch, no dropout
        dict(_attention(fp32, 12, 12, 64, 8, 512, 7, 0, False, 0.0, True), name="attention bert fp32"),
        # long prompts read once by a model with shared key/value heads
        dict(_attention(bf16, 32, 8, 128, 2, 8192, 3, 0, True, 0.0, False), name="attention prompt bf16"),
        # a training step on long causal sequences with shared heads
        dict(_attention(bf16, 16, 4, 128, 6, 4096, 9, 0, True, 0.0, True), name="attention causal bf16"),
        # a handful of short sentences: launch latency counts
        dict(_attention(fp16, 12, 12, 64, 3, 40, 2, 0, False, 0.0, True), name="attention short fp16"),
        # an odd head size and length, rows behind the last sequence
        dict(_attention(fp16, 10, 2, 80, 5, 1023, 4, 77, True, 0.1, True), name="attention odd fp16"),
        # the join behind each half of a BERT block: residual + dropout, then the norm
        dict(_layer_norm(bf16, bf16, fp32, 32768, 768, True, 0.1, True), name="norm join bf16"),
        # a plain norm of a few tokens
        dict(_layer_norm(fp32, "", fp32, 37, 768, True, 0.0, True), name="norm short fp32"),
        # a wide model, norm in front of a block, weights in the model's type
        dict(_layer_norm(bf16, "", bf16, 8192, 8192, True, 0.0, True), name="norm wide bf16"),
        # an odd width without bias, a 32-bit residual stream under half inputs
        dict(_layer_norm(fp16, fp32, fp32, 5001, 1001, False, 0.2, True), name="norm odd fp16"),
        # the dropout behind the embeddings, forward and backward
        dict(_dropout(bf16, 32768, 768, 0.1), name="dropout bert bf16"),
        # an odd small tensor
        dict(_dropout(fp32, 53, 333, 0.25), name="dropout small fp32"),
    ]


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    dtype = rng.choice(("bfloat16", "float16", "float32"))
    what = rng.random()
    if what < 0.5:
        kv_heads = rng.choice((1, 2, 3, 4, 8, 12))
        heads = kv_heads * rng.choice([g for g in (1, 1, 2, 3, 4, 8) if g * kv_heads <= 32])
        dim = rng.choice((64, 64, 128, 128, 32, 40, 57, 80, 96, 112))
        longest = _log(rng, 1, 4096)
        seqs = _log(rng, 1, 64)
        # the plain form holds seqs * heads * longest^2 scores
        while seqs > 1 and (seqs * heads * longest ** 2 > 1 << 30 or seqs * longest > 32768):
            seqs -= 1
        train = rng.random() < 0.75
        return _attention(dtype, heads, kv_heads, dim, seqs, longest,
                          rng.randrange(1, 1000), rng.choice((0, 0, rng.randrange(1, 200))),
                          rng.random() < 0.5, rng.choice((0.0, 0.0, 0.1, 0.3)), train)
    if what < 0.8:
        width = _log(rng, 33, 10000)
        rows = _log(rng, 1, max(1, min(32768, (1 << 25) // width)))
        residual = rng.choice(("", dtype, "float32"))
        p = rng.choice((0.0, 0.1, 0.3))
        return _layer_norm(dtype, residual, rng.choice(("float32", dtype)),
                           rows, width, rng.random() < 0.7, p, rng.random() < 0.75)
    width = _log(rng, 33, 10000)
    rows = _log(rng, 1, max(1, min(32768, (1 << 25) // width)))
    return _dropout(dtype, rows, width, round(rng.uniform(0.05, 0.5), 3))


def _lengths(case):
    """Sequence lengths of a packed batch: the first is the longest, the
    others spread over the range, one in sixteen of them empty."""
    rng = random.Random(case["mix"])
    n = [case["longest"]]
    for _ in range(case["seqs"] - 1):
        n.append(0 if rng.random() < 1 / 16 else rng.randint(1, case["longest"]))
    return n


def _pairs(case):
    """Pairs of a query and a key that it sees, in one head."""
    if case["causal"]:
        return sum(n * (n + 1) // 2 for n in _lengths(case))
    return sum(n * n for n in _lengths(case))


def work(case):
    size = {"float32": 4, "float16": 2, "bfloat16": 2, "": 0}
    e = size[case["dtype"]]
    if case["op"] == "attention":
        rows = sum(_lengths(case)) + case["spare"]
        wide, narrow = rows * case["heads"] * case["dim"], rows * case["kv_heads"] * case["dim"]
        # q, k, v and the output; their gradients
        moved = e * (2 * wide + 2 * narrow)
        flops = 4 * _pairs(case) * case["heads"] * case["dim"]
        if case["train"]:
            moved, flops = 2 * moved, 3.5 * flops
        return {"bytes": moved, "flops": flops}
    n = case["rows"] * case["width"]
    if case["op"] == "layer_norm":
        r = size[case["residual"]]
        o = r or e
        moved = n * (e + r + o)
        per_column = size[case["weights"]] * (2 if case["bias"] else 1) * case["width"]
        if case["train"]:
            moved, per_column = moved + n * (o + e + r), 2 * per_column
        return {"bytes": moved + per_column, "flops": (20 if case["train"] else 8) * n}
    return {"bytes": 4 * n * e, "flops": 2 * n}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    dtype = _TYPES[case["dtype"]]
    s = {"case": case, "seed": torch.randint(0, 1 << 62, (1,), generator=g, device="cuda"),
         "offset": 1 + seed % 1000}
    if case["op"] == "attention":
        lengths = _lengths(case)
        ends = torch.tensor([0] + lengths).cumsum(0)
        rows = int(ends[-1]) + case["spare"]
        h, kv, d = case["heads"], case["kv_heads"], case["dim"]
        # one projection's output, as a model has it: q, k and v side by side
        qkv = normal(rows, h + 2 * kv, d)
        qkv[:, :h] *= 2
        qkv = qkv.to(dtype)
        s.update(cu_seqlens=ends.to(torch.int32).cuda(), longest=max(lengths),
                 q=qkv[:, :h], k=qkv[:, h:h + kv], v=qkv[:, h + kv:])
        if case["train"]:
            for name in ("q", "k", "v"):
                s[name].requires_grad_()
            s["dout"] = normal(rows, h, d).to(dtype)
        return s
    rows, width = case["rows"], case["width"]
    # some channels of a trained model's activations are far larger than the rest
    x = normal(rows, width) * (1 + 4 * (normal(width) > 2)) + 0.3 * normal(width)
    s["x"] = x.to(dtype)
    out = dtype
    if case["op"] == "layer_norm":
        weights = _TYPES[case["weights"]]
        s["weight"] = (1 + 0.2 * normal(width)).to(weights)
        s["bias"] = (0.2 * normal(width)).to(weights) if case["bias"] else None
        s["residual"] = None
        if case["residual"]:
            out = _TYPES[case["residual"]]
            s["residual"] = normal(rows, width).to(out)
    if case.get("train", True):
        for name in ("x", "weight", "bias", "residual"):
            if s.get(name) is not None:
                s[name].requires_grad_()
        s["dout"] = normal(rows, width).to(out)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"attention": _plain_attention, "layer_norm": _plain_layer_norm,
                "dropout": _plain_dropout}[state["case"]["op"]](state)


def _run_own(s):
    import bluefog_amd as bf

    c = s["case"]
    if c["op"] == "attention":
        leaves = {"dq": s["q"], "dk": s["k"], "dv": s["v"]}
        out = bf.packed_attention(s["q"], s["k"], s["v"], s["cu_seqlens"], causal=c["causal"],
                                  dropout_p=c["p"], seed=s["seed"], offset=s["offset"])
    elif c["op"] == "layer_norm":
        leaves = {"dx": s["x"], "dweight": s["weight"], "dbias": s["bias"], "dresidual": s["residual"]}
        out = bf.layer_norm(s["x"], s["weight"], s["bias"], residual=s["residual"],
                            dropout_p=c["p"], seed=s["seed"], offset=s["offset"])
    else:
        leaves = {"dx": s["x"]}
        out = bf.counter_dropout(s["x"], c["p"], s["seed"], offset=s["offset"])
    if not c.get("train", True):
        return {"out": out}
    leaves = {name: t for name, t in leaves.items() if t is not None}
    grads = torch.autograd.grad(out, list(leaves.values()), s["dout"])
    return {"out": out.detach(), **dict(zip(leaves, grads))}


def _philox(c0, c1, c2, c3, seed):
    """Philox4x32-7 on 64-bit tensors that hold 32-bit words; [..., 8] halves."""
    k0, k1 = seed & _M32, (seed >> 32) & _M32
    for _ in range(7):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (((b >> 32) & _M32) ^ c1 ^ k0, b & _M32,
                          ((a >> 32) & _M32) ^ c3 ^ k1, a & _M32)
        k0, k1 = (k0 + 0x9E3779B9) & _M32, (k1 + 0xBB67AE85) & _M32
    words = torch.stack(torch.broadcast_tensors(c0, c1, c2, c3), -1)
    return torch.stack((words & 0xFFFF, words >> 16), -1).flatten(-2)


def _threshold(p):
    return min(65535, int(p * 65536 + 0.5))


def _scaled_keep(halves, p):
    t = _threshold(p)
    return (halves >= t) * (65536 / (65536 - t))


def _flat_keep(s, shape):
    n = math.prod(shape)
    block = torch.arange((n + 7) // 8, device="cuda")
    zero = torch.zeros_like(block)
    halves = _philox(block & _M32, block >> 32, zero, zero + s["offset"], s["seed"])
    return _scaled_keep(halves.flatten()[:n].view(shape), s["case"]["p"])


def _plain_attention(s):
    c = s["case"]
    h, kv, d, longest = c["heads"], c["kv_heads"], c["dim"], s["longest"]
    scale = 1 / math.sqrt(d)
    start, end = s["cu_seqlens"][:-1].long(), s["cu_seqlens"][1:].long()
    pos = torch.arange(longest, device="cuda")
    valid = pos < (end - start)[:, None]
    row = torch.where(valid, start[:, None] + pos, 0)

    def padded(x, heads):
        x = torch.where(valid[:, :, None, None], x[row].float(), 0.0)
        return x.repeat_interleave(h // heads, 2).transpose(1, 2).contiguous()

    def packed(x, heads, like):
        x = x.view(-1, heads, h // heads, longest, d).sum(2).transpose(1, 2)
        out = torch.zeros(like.shape, device="cuda")
        out[row[valid]] = x[valid]
        return out.to(like.dtype)

    q, k, v = padded(s["q"], h), padded(s["k"], kv), padded(s["v"], kv)
    seen = valid[:, None, None, :]
    if c["causal"]:
        seen = seen & (pos[None, :] <= pos[:, None])
    score = torch.matmul(q, k.transpose(2, 3).contiguous())
    score.mul_(scale).masked_fill_(~seen, -1e30)
    score.sub_(score.amax(3, keepdim=True)).exp_()
    score.masked_fill_(~seen, 0.0)
    prob = score.div_(score.sum(3, keepdim=True).clamp_min_(1e-30))
    keep = None
    if c["p"]:
        group = torch.arange(2 * ((longest + 15) // 16), device="cuda")
        halves = _philox(group, row[:, None, :, None], torch.arange(h, device="cuda")[:, None, None],
                         torch.full_like(group, s["offset"]), s["seed"])
        # a group of eight: keys 0-3 and 8-11 of sixteen, or 4-7 and 12-15
        halves = halves.unflatten(4, (2, 4)).unflatten(3, (-1, 2)).transpose(4, 5)
        keep = _scaled_keep(halves.flatten(3)[..., :longest], c["p"])
    dropped = prob if keep is None else prob * keep
    out = torch.matmul(dropped, v)
    if not c["train"]:
        return {"out": packed(out, h, s["q"])}
    dout = padded(s["dout"], h)
    dv = torch.matmul(dropped.transpose(2, 3).contiguous(), dout)
    dprob = torch.matmul(dout, v.transpose(2, 3).contiguous())
    if keep is not None:
        dprob.mul_(keep)
    dscore = dprob.sub_((prob * dprob).sum(3, keepdim=True)).mul_(prob).mul_(scale)
    dq = torch.matmul(dscore, k)
    dk = torch.matmul(dscore.transpose(2, 3).contiguous(), q)
    return {"out": packed(out, h, s["q"]), "dq": packed(dq, h, s["q"]),
            "dk": packed(dk, kv, s["k"]), "dv": packed(dv, kv, s["v"])}


def _plain_layer_norm(s):
    c = s["case"]
    x, w = s["x"].float(), s["weight"].float()
    keep = _flat_keep(s, x.shape) if c["p"] else None
    z = x if keep is None else x * keep
    if s["residual"] is not None:
        z = z + s["residual"].float()
    z = z - z.mean(1, keepdim=True)
    rstd = torch.rsqrt(z.square().mean(1, keepdim=True) + 1e-5)
    xhat = z * rstd
    y = xhat * w
    if s["bias"] is not None:
        y = y + s["bias"].float()
    kind = s["x"].dtype if s["residual"] is None else s["residual"].dtype
    out = {"out": y.to(kind)}
    if not c["train"]:
        return out
    dy = s["dout"].float()
    out["dweight"] = (dy * xhat).sum(0).to(s["weight"].dtype)
    if s["bias"] is not None:
        out["dbias"] = dy.sum(0).to(s["bias"].dtype)
    g = dy * w
    dz = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    out["dx"] = (dz if keep is None else dz * keep).to(s["x"].dtype)
    if s["residual"] is not None:
        out["dresidual"] = dz.to(kind)
    return out


def _plain_dropout(s):
    keep = _flat_keep(s, s["x"].shape)
    return {"out": (s["x"].float() * keep).to(s["x"].dtype),
            "dx": (s["dout"].float() * keep).to(s["x"].dtype)}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------


def _exact_bits(counter, key):
    """The generator once more, on products of 16-bit halves that no word
    overflows. ``counter``: four equally shaped tensors; returns a list of
    the eight halves."""

    def multiply(a, m):
        low, high = (a & 0xFFFF) * m, (a >> 16) * m
        whole = (low >> 16) + high  # the product without its lowest 16 bits
        return whole >> 16, ((whole & 0xFFFF) << 16) | (low & 0xFFFF)

    c = list(counter)
    for i in range(7):
        ha, la = multiply(c[0], 0xD2511F53)
        hb, lb = multiply(c[2], 0xCD9E8D57)
        ka, kb = (key % 2 ** 32 + i * 0x9E3779B9) % 2 ** 32, (key // 2 ** 32 + i * 0xBB67AE85) % 2 ** 32
        c = [hb ^ c[1] ^ ka, lb, ha ^ c[3] ^ kb, la]
    return [half for w in c for half in (w % 65536, w // 65536)]


def _exact_keep(halves, p):
    t = min(65535, math.floor(p * 65536 + 0.5))
    return torch.where(halves < t, 0.0, 65536 / (65536 - t)).double()


def _exact_flat(shape, key, offset, p):
    i = torch.arange(math.prod(shape), device="cuda")
    at = torch.arange((i.numel() + 7) // 8, device="cuda")
    all8 = torch.stack(_exact_bits([at % 2 ** 32, at // 2 ** 32, at * 0, at * 0 + offset], key))
    return _exact_keep(all8[i % 8, i // 8], p).view(shape)


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        key = int(s["seed"])
        if case["op"] == "attention":
            return _exact_attention(case, s, key)
        x = s["x"].double()
        keep = _exact_flat(x.shape, key, s["offset"], case["p"]) if case["p"] else torch.ones_like(x)
        if case["op"] == "dropout":
            return {"out": x * keep, "dx": s["dout"].double() * keep}
        z = x * keep + (0 if s["residual"] is None else s["residual"].double())
        n = z.shape[1]
        mean = z.sum(1) / n
        sigma = torch.sqrt(((z - mean[:, None]) ** 2).sum(1) / n + 1e-5)
        unit = (z - mean[:, None]) / sigma[:, None]
        w = s["weight"].double()
        got = {"out": unit * w + (0 if s["bias"] is None else s["bias"].double())}
        if case["train"]:
            dy = s["dout"].double()
            got["dweight"] = torch.einsum("rc,rc->c", dy, unit)
            if s["bias"] is not None:
                got["dbias"] = dy.sum(0)
            dunit = dy * w
            along = (dunit * unit).sum(1) / n
            dz = (dunit - dunit.sum(1)[:, None] / n - unit * along[:, None]) / sigma[:, None]
            got["dx"] = dz * keep
            if s["residual"] is not None:
                got["dresidual"] = dz
        return got


def _exact_attention(case, s, key):
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    got = {"out": torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")}
    if case["train"]:
        for name in ("q", "k", "v"):
            got["d" + name] = torch.zeros(s[name].shape, dtype=torch.float64, device="cuda")
    at = 0
    for n in _lengths(case):
        rows = slice(at, at + n)
        i = torch.arange(n, device="cuda")
        group = (i // 16) * 2 + i % 8 // 4
        half = i % 16 // 8 * 4 + i % 4
        for head in range(h if n else 0):
            shared = head // (h // kv)
            q, k, v = s["q"][rows, head].double(), s["k"][rows, shared].double(), s["v"][rows, shared].double()
            score = q @ k.T.contiguous() / d ** 0.5
            if case["causal"]:
                score = torch.where(i[None, :] > i[:, None], -math.inf, score)
            prob = torch.softmax(score, 1)
            keep = 1.0
            if case["p"]:
                count = torch.arange(int(group.max()) + 1, device="cuda").expand(n, -1)
                row = (at + i)[:, None].expand_as(count)
                all8 = torch.stack(_exact_bits([count, row, torch.full_like(count, head), torch.full_like(count, s["offset"])], key))
                keep = _exact_keep(all8[half, :, group].T, case["p"])
            got["out"][rows, head] = (prob * keep) @ v
            if case["train"]:
                do = s["dout"][rows, head].double()
                got["dv"][rows, shared] += (prob * keep).T.contiguous() @ do
                dprob = (do @ v.T.contiguous()) * keep
                dscore = prob * (dprob - (dprob * prob).sum(1, keepdim=True)) / d ** 0.5
                got["dq"][rows, head] = dscore @ k
                got["dk"][rows, shared] += dscore.T.contiguous() @ q
        at += n
    return got
