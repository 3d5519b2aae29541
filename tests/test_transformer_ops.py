# Copyright 2026. Licensed under the Apache License, Version 2.0.
"""Packed attention, layer norm and counter-based dropout against plain 64-bit
implementations, on the CPU and on the GPU.

Tolerances are bounds, elementwise, worked out by ``attention_oracle`` and
``norm_oracle`` next to the values: every rounding to the storage type costs at
most u = finfo(type).eps / 2 of the rounded value, every 32-bit sum of n terms
at most n * 2**-24 of the sum of their magnitudes, an exponential 8 * 2**-24 of
its value beside the error of its argument."""

import math

import numpy as np
import pytest
import torch

import bluefog_amd as bf
from bluefog_amd.ops import hip_ext

F32 = 2.0 ** -24
LEAST = 2.0 ** -126


def rounding(dtype, value):
    """Half a step of the type at each value: f16 keeps steps of 2**-24 below
    2**-14, the others their relative precision down to LEAST."""
    least = 2.0 ** -25 if dtype == torch.float16 else LEAST
    return (torch.finfo(dtype).eps / 2 * value.abs()).clamp_min(least)
TYPES = [torch.float32, torch.float16, torch.bfloat16]
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


# ---------------------------------------------------------------------------
# oracles
# ---------------------------------------------------------------------------


def philox(c0, c1, c2, c3, key, rounds=7):
    """Philox4x32 on numpy; [..., 4] words."""
    c = [np.asarray(x, dtype=np.uint64) for x in np.broadcast_arrays(c0, c1, c2, c3)]
    m = np.uint64(0xFFFFFFFF)
    k0, k1 = key & 0xFFFFFFFF, (key >> 32) & 0xFFFFFFFF
    for i in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        ka = np.uint64((k0 + i * 0x9E3779B9) & 0xFFFFFFFF)
        kb = np.uint64((k1 + i * 0xBB67AE85) & 0xFFFFFFFF)
        s = np.uint64(32)
        c = [(b >> s) ^ c[1] ^ ka, b & m, (a >> s) ^ c[3] ^ kb, a & m]
    return np.stack(c, -1)


def keep_of(words, which, p):
    """Factor of the element with 16-bit value number ``which`` of its call."""
    word = np.take_along_axis(words, (which // 2)[..., None], -1)[..., 0]
    value = np.where(which % 2, word >> np.uint64(16), word & np.uint64(0xFFFF)).astype(np.int64)
    t = min(65535, math.floor(p * 65536 + 0.5))
    return torch.from_numpy(np.where(value >= t, 65536 / (65536 - t), 0.0))


def flat_keep(shape, p, key, offset):
    if not p:
        return torch.ones(shape, dtype=torch.float64)
    i = np.arange(math.prod(shape)).reshape(shape)
    return keep_of(philox(i // 8 % 2 ** 32, i // 8 // 2 ** 32, 0, offset, key), i % 8, p)


def attention_keep(heads, begin, n, p, key, offset):
    if not p:
        return torch.ones(heads, n, n, dtype=torch.float64)
    h, i, j = np.ogrid[:heads, :n, :n]
    h, i, j = np.broadcast_arrays(h, i, j)
    words = philox(j // 16 * 2 + j // 4 % 2, begin + i, h, offset, key)
    return keep_of(words, j // 8 % 2 * 4 + j % 4, p)


def attention_oracle(q, k, v, dout, ends, causal, scale, p, key, offset):
    """{name: (value, bound on the error)} in 64 bits, for inputs as given."""
    u = torch.finfo(q.dtype).eps / 2
    heads, group, d = q.shape[1], q.shape[1] // k.shape[1], q.shape[2]
    want = {"out": q, "dq": q, "dk": k, "dv": v}
    want = {n: [torch.zeros(t.shape, dtype=torch.float64) for _ in range(2)] for n, t in want.items()}
    wide = [x.detach().cpu().double().transpose(0, 1) for x in (q, k, v, dout)]
    for begin, end in zip(ends, ends[1:]):
        n = end - begin
        if not n:
            continue
        rows = slice(begin, end)
        Q, K, V, G = (x[:, rows] for x in wide)
        K, V = K.repeat_interleave(group, 0), V.repeat_interleave(group, 0)
        seen = torch.ones(n, n, dtype=torch.bool)
        if causal:
            seen = seen.tril()
        S = (Q @ K.transpose(1, 2)) * scale
        P = torch.softmax(S.masked_fill(~seen, -math.inf), 2)
        # error of a score: a sum of d products and the roundings of scaling;
        # P's relative error: twice the row's largest (numerator, denominator),
        # the sum of n terms and the exponentials
        magnitude = (Q.abs() @ K.abs().transpose(1, 2)) * scale
        es = (d + 4) * F32 * magnitude.masked_fill(~seen, 0).amax(2, keepdim=True)
        eP = 2 * es + (n + 16) * F32
        M = attention_keep(heads, begin, n, p, key, offset)
        D = P * M
        O = D @ V
        # D is rounded to the type in front of the product; half-precision
        # values below 2**-14 keep 2**-25 of the largest
        tiny = 2.0 ** -25 * n if q.dtype == torch.float16 else 0.0
        spread = D @ V.abs()
        big = M.amax() * V.abs().amax(1, keepdim=True)
        put(want["out"], rows, O, (eP + u + n * F32) * spread + tiny * big + rounding(q.dtype, O))
        dD = G @ V.transpose(1, 2)
        dP = dD * M
        delta = (P * dP).sum(2, keepdim=True)
        # delta comes from the rounded output
        e_delta = (G.abs() * ((eP + u + n * F32) * spread + tiny * big + rounding(q.dtype, O))).sum(2, keepdim=True)
        e_delta = e_delta + d * F32 * (G.abs() * O.abs()).sum(2, keepdim=True)
        e_dP = (d + 4) * F32 * (G.abs() @ V.abs().transpose(1, 2)) * M
        dS = P * (dP - delta)
        e_dS = P * (e_dP + e_delta) + (eP + u + 4 * F32) * P * (dP.abs() + delta.abs())
        alone = seen.sum(1) == 1
        # a probability below the smallest normal number may count as 0
        e_dS = e_dS + LEAST * (dP.abs() + delta.abs())
        e_dS[:, alone] = 0  # one key: dS is 0 by definition
        floor = 2.0 ** -24 if q.dtype == torch.float16 else 0.0  # of the largest dS
        e_dS = e_dS + floor * dS.abs().amax() * ~alone[:, None]
        put(want["dq"], rows, dS @ K * scale, (e_dS @ K.abs() + n * F32 * (dS.abs() @ K.abs())) * scale
            + rounding(q.dtype, dS @ K * scale))
        m = n * group
        for name, left, e_left, right, f in (
            ("dk", dS, e_dS, Q, scale), ("dv", D, (eP + u) * D + (tiny + LEAST) * M.amax(), G, 1.0)):
            value = (left.transpose(1, 2) @ right) * f
            bound = (e_left.transpose(1, 2) @ right.abs() + m * F32 * (left.abs().transpose(1, 2) @ right.abs())) * f
            value, bound = (x.unflatten(0, (-1, group)).sum(1) for x in (value, bound))
            put(want[name], rows, value, bound + rounding(q.dtype, value))
    return want


def put(pair, rows, value, bound):
    pair[0][rows], pair[1][rows] = value.transpose(0, 1), bound.transpose(0, 1)


def norm_oracle(x, r, weight, bias, dout, eps, p, key, offset):
    kind = x.dtype if r is None else r.dtype
    X, G = (t.detach().cpu().double().flatten(0, -2) for t in (x, dout))
    rows, n = X.shape
    M = flat_keep(X.shape, p, key, offset)
    R = torch.zeros_like(X) if r is None else r.detach().cpu().double().flatten(0, -2)
    W = torch.ones(n).double() if weight is None else weight.detach().cpu().double()
    B = torch.zeros(n).double() if bias is None else bias.detach().cpu().double()
    Z = X * M + R
    # a row's values, and so their mean, are off by this much; the sums run
    # over at most n / 64 terms in a lane and a tree of 16 levels
    terms = n / 64 + 32
    e_z = terms * F32 * (X.abs() * M + R.abs()).amax(1, keepdim=True)
    C = Z - Z.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(C.square().mean(1, keepdim=True) + eps)
    H = C * rstd
    # rstd depends on C's error by at most its share, and on the sum's rounding
    e_h = e_z * rstd * (1 + H.abs()) + terms * F32 * H.abs()
    Y = H * W + B
    e_y = e_h * W.abs() + 4 * F32 * (H * W).abs() + F32 * Y.abs() + rounding(kind, Y)
    g = G * W
    m1, m2 = g.mean(1, keepdim=True), (g * H).mean(1, keepdim=True)
    dZ = rstd * (g - m1 - H * m2)
    size = rstd * (g.abs() + g.abs().mean(1, keepdim=True) + H.abs() * (g * H).abs().mean(1, keepdim=True))
    e_rstd = e_z * rstd + terms * F32
    e_dz = size * (terms * F32 + e_rstd) + rstd * (
        e_h * m2.abs() + H.abs() * (g.abs() * e_h).mean(1, keepdim=True))
    want = {"out": (Y, e_y), "dx": (dZ * M, e_dz * M + 2 * F32 * dZ.abs() * M + rounding(x.dtype, dZ * M))}
    if r is not None:
        want["dresidual"] = (dZ, e_dz + rounding(kind, dZ))
    if weight is not None:
        dW = (G * H).sum(0)
        want["dweight"] = (dW, (G.abs() * e_h).sum(0) + (rows + 8) * F32 * (G * H).abs().sum(0) + rounding(weight.dtype, dW))
    if bias is not None:
        want["dbias"] = (G.sum(0), (rows + 8) * F32 * G.abs().sum(0) + rounding(bias.dtype, G.sum(0)))
    return want


def close(got, want):
    assert got.keys() == want.keys()
    for name, (value, bound) in want.items():
        x = got[name].detach().cpu().double().reshape(value.shape)
        off = (x - value).abs()
        bad = ~(off <= bound)
        assert not bad.any(), (
            f"{name}: {int(bad.sum())} of {bad.numel()} values are off, the worst by "
            f"{(off / bound.clamp_min(1e-300))[bad].max():.3g} times its bound"
        )


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------


def ends_of(lengths, device):
    return torch.tensor([0] + list(lengths)).cumsum(0).to(torch.int32).to(device)


def attention_inputs(lengths, heads, kv_heads, dim, dtype, device, spare=0, seed=0, factor=1.0):
    g = torch.Generator().manual_seed(seed)
    rows = sum(lengths) + spare
    qkv = torch.randn(rows, heads + 2 * kv_heads, dim, generator=g) * factor
    qkv = qkv.to(dtype).to(device)
    dout = torch.randn(rows, heads, dim, generator=g).to(dtype).to(device)
    return (*(t.detach().requires_grad_() for t in qkv.split([heads, kv_heads, kv_heads], 1)), dout)


def attention(q, k, v, dout, cu, **kw):
    out = bf.packed_attention(q, k, v, cu, **kw)
    assert out.is_contiguous() and out.shape == q.shape and out.dtype == q.dtype
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), dout)
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def attention_agrees(device, dtype, lengths, heads=2, kv_heads=1, dim=64, causal=False, scale=None,
                     p=0.0, spare=0, seed=0, factor=1.0, key=(5 << 33) + 77, offset=9):
    q, k, v, dout = attention_inputs(lengths, heads, kv_heads, dim, dtype, device, spare, seed, factor)
    cu = ends_of(lengths, device)
    kw = dict(causal=causal, dropout_p=p, seed=key, offset=offset)
    got = attention(q, k, v, dout, cu, **kw) if scale is None else attention(q, k, v, dout, cu, scale=scale, **kw)
    want = attention_oracle(q, k, v, dout, cu.tolist(), causal, scale or dim ** -0.5, p, key, offset)
    close(got, want)
    with torch.no_grad():  # the pass without a graph gives the same
        again = bf.packed_attention(q, k, v, cu, **kw, **({} if scale is None else {"scale": scale}))
    assert torch.equal(again, got["out"])


LENGTHS = [
    (3,) * 70, (40, 0, 1) * 40, (1,) * 300,  # more sequences than lanes
    (1,), (2,), (1, 1, 1), (17,), (31, 33), (0, 5, 0, 0, 64, 0), (127, 1, 129), (200, 3), (65, 63, 2, 130),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths", LENGTHS)
def test_attention_lengths(device, dtype, causal, lengths):
    attention_agrees(device, dtype, lengths, causal=causal, spare=len(lengths) % 3)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [1, 7, 16, 32, 40, 57, 64, 65, 72, 80, 96, 100, 112, 127, 128])
def test_attention_dims(device, dtype, dim):
    attention_agrees(device, dtype, (70, 19), dim=dim, causal=dim % 2 == 0, seed=dim)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 4), (6, 2), (8, 1), (12, 12), (15, 3)])
def test_attention_heads(device, dtype, heads, kv_heads):
    attention_agrees(device, dtype, (40, 61), heads, kv_heads, causal=heads % 2 == 0, seed=heads)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("p", [0.1, 0.5, 0.99999])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_dropout(device, dtype, causal, p, dim):
    attention_agrees(device, dtype, (75, 1, 40), 4, 2, dim, causal=causal, p=p, spare=3)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_long(device, dtype):
    attention_agrees(device, dtype, (1000, 300), 2, 1, 64, causal=True, p=0.1)
    attention_agrees(device, dtype, (777,), 1, 1, 128, scale=0.3)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_large_scores(device, dtype):
    """Scores of hundreds: the running maximum carries the softmax."""
    attention_agrees(device, dtype, (150,), 2, 2, 64, causal=True, factor=6.0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_rows_behind_the_last_sequence(device, dtype):
    """They are zero and reach nothing, whatever they hold."""
    q, k, v, dout = attention_inputs((30, 5), 4, 2, 64, dtype, device, spare=70)
    cu = ends_of((30, 5), device)
    clean = attention(q, k, v, dout, cu, causal=True)
    for bad in (math.nan, math.inf):
        for t in (q, k, v, dout):
            t.detach()[35:] = bad
        got = attention(q, k, v, dout, cu, causal=True)
        for name in clean:
            assert torch.equal(got[name], clean[name])
            assert not got[name][35:].any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_attention_bad_values_stay_in_their_sequence(device, dtype, bad):
    lengths = (20, 33, 9)
    q, k, v, dout = attention_inputs(lengths, 2, 1, 64, dtype, device)
    cu = ends_of(lengths, device)
    clean = attention(q, k, v, dout, cu)
    for t in (q, k, v, dout):
        t.detach()[20:53] = bad
    got = attention(q, k, v, dout, cu)
    for name in clean:
        for rows in (slice(0, 20), slice(53, 62)):
            assert torch.equal(got[name][rows], clean[name][rows])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attention_causal_rows_do_not_see_later_values(device, dtype, bad):
    """A later key or value that is not a number leaves earlier rows alone."""
    if device == "cpu":
        pytest.skip("a masked probability of 0 times such a value is no number in the torch products")
    for n, at in ((50, 37), (300, 150), (300, 299)):
        q, k, v, dout = attention_inputs((n,), 2, 2, 64, dtype, device)
        cu = ends_of((n,), device)
        with torch.no_grad():
            clean = bf.packed_attention(q, k, v, cu, causal=True)
            k[at], v[at] = bad, bad
            got = bf.packed_attention(q, k, v, cu, causal=True)
        assert torch.equal(got[:at], clean[:at])
        assert not torch.isfinite(got[at:]).any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_one_key_has_no_score_gradient(device, dtype):
    """A row that sees one key has probability 1: dq and dk are exactly 0."""
    lengths = (1, 1, 1, 1)
    q, k, v, dout = attention_inputs(lengths, 4, 2, 80, dtype, device)
    got = attention(q, k, v, dout, ends_of(lengths, device), dropout_p=0.2, seed=3)
    assert not got["dq"].any() and not got["dk"].any() and got["dv"].any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_small_and_large_gradients(device, dtype):
    """dO far from 1: no intermediate leaves its type's range. The factors are
    powers of two, so the gradients scale by them up to what the type's own
    range takes from dO and the results."""
    lengths = (90, 40)
    q, k, v, dout = attention_inputs(lengths, 4, 2, 64, dtype, device)
    cu = ends_of(lengths, device)
    for f in (2.0 ** 9, 2.0 ** -9):
        scaled = dout * f
        got = attention(q, k, v, scaled, cu, causal=True)
        want = attention_oracle(q, k, v, scaled, cu.tolist(), True, 0.125, 0.0, 0, 0)
        close(got, want)


@pytest.mark.parametrize("device", DEVICES)
def test_attention_strides(device):
    """Slices, swapped dimensions, broadcast heads, a misaligned start."""
    dtype, lengths = torch.bfloat16, (21, 44)
    cu = ends_of(lengths, device)
    n, h, d = 65, 4, 64
    g = torch.Generator().manual_seed(1)
    base = torch.randn(n * h * d * 8, generator=g).to(dtype).to(device)
    views = [
        base[: n * h * d * 3].view(n, 3, h, d).unbind(1),
        base[: n * h * d * 3].view(3, h, n, d).transpose(1, 2).unbind(0),
        base[: n * h * d * 3].view(3, n, d, h).transpose(2, 3).unbind(0),
        [x[:, :, 1:65] for x in base[: n * h * (d + 3) * 3].view(3, n, h, d + 3).unbind(0)],
        [base[i: i + n * d].view(n, 1, d).expand(n, h, d) for i in (0, 3, 8)],
        [x[::2] for x in base[: n * 2 * h * d * 3].view(3, n * 2, h, d).unbind(0)],
    ]
    for q, k, v in views:
        q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
        dout = torch.randn(d, h, n, generator=g).to(dtype).to(device).permute(2, 1, 0)
        got = attention(q, k, v, dout, cu, causal=True)
        dense = [t.detach().contiguous().requires_grad_() for t in (q, k, v)]
        want = attention(*dense, dout.contiguous(), cu, causal=True)
        for name in want:
            assert torch.equal(got[name], want[name])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim", [40, 64, 57])
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_dense_and_misaligned(device, dtype, dim):
    """Dense tensors, the output's gradient too, that start between 16-byte
    places: the same bits as aligned ones."""
    near = attention_inputs((21, 150), 4, 2, dim, dtype, device)
    cu = ends_of((21, 150), device)
    moved = []
    for t in near:
        flat = torch.empty(t.numel() + 1, dtype=dtype, device=device)
        flat[1:] = t.detach().flatten()
        moved.append(flat[1:].view(t.shape).requires_grad_())
        assert moved[-1].is_contiguous() and moved[-1].data_ptr() % 16
    got, want = (attention(*t[:3], t[3].detach(), cu, causal=True) for t in (moved, near))
    for name in want:
        assert torch.equal(got[name], want[name])


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [57, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("apart", [1 << 22, (1 << 22) + 8])
def test_attention_rows_far_apart(dtype, dim, apart):
    """Rows 2**22 values apart, the widest that is read in place, and more, of
    a sequence that spans over 2**32 bytes: the same bits as dense rows."""
    n = 1100 if dtype == torch.bfloat16 else 300
    base = torch.empty(n * apart, dtype=dtype, device="cuda")
    far = [base.as_strided((n, 1, dim), (apart, dim, 1), 128 * i).requires_grad_() for i in range(4)]
    near = attention_inputs((n,), 1, 1, dim, dtype, "cuda")
    with torch.no_grad():
        for a, b in zip(far, near):
            a.copy_(b)
    cu = ends_of((n,), "cuda")
    got, want = (attention(*t[:3], t[3].detach(), cu, causal=True) for t in (far, near))
    for name in want:
        assert torch.equal(got[name], want[name])


@pytest.mark.parametrize("device", DEVICES)
def test_attention_gradient_of_a_sum(device):
    """An expanded upstream gradient, and leaves that need none."""
    q, k, v, _ = attention_inputs((33, 7), 4, 2, 64, torch.float32, device)
    cu = ends_of((33, 7), device)
    ones = torch.ones_like(q)
    want = attention(q, k, v, ones, cu)
    out = bf.packed_attention(q, k, v, cu)
    got = torch.autograd.grad(out.sum(), (q, k, v))
    for a, b in zip(got, (want["dq"], want["dk"], want["dv"])):
        assert torch.equal(a, b)
    for leaves in ((q,), (k,), (v,), (q, v)):
        frozen = [t if any(t is x for x in leaves) else t.detach() for t in (q, k, v)]
        got = torch.autograd.grad(bf.packed_attention(*frozen, cu).sum(), leaves)
        for t, a in zip(leaves, got):
            assert torch.equal(a, want[{id(q): "dq", id(k): "dk", id(v): "dv"}[id(t)]])


@pytest.mark.parametrize("device", DEVICES)
def test_attention_twice_through_one_graph(device):
    """A kept graph gives the same gradients again; a wide batch of thousands
    of sequences is found row by row."""
    q, k, v, dout = attention_inputs((33, 7), 4, 2, 64, torch.bfloat16, device)
    out = bf.packed_attention(q, k, v, ends_of((33, 7), device), causal=True, dropout_p=0.1, seed=5)
    first = torch.autograd.grad(out, (q, k, v), dout, retain_graph=True)
    for a, b in zip(first, torch.autograd.grad(out, (q, k, v), dout)):
        assert torch.equal(a, b)
    lengths = [n % 3 for n in range(5000)]
    x = torch.randn(sum(lengths), 1, 8, device=device)
    ones = bf.packed_attention(torch.zeros_like(x), x, x, ends_of(lengths, device))
    # equal scores: the mean of a sequence's rows (its one or two), exactly
    row = torch.arange(len(x), device=device)
    pair = torch.where(row % 3 == 0, row, torch.where(row % 3 == 1, row + 1, row - 1))
    assert torch.allclose(ones, (x + x[pair.clamp_max(len(x) - 1)]) / 2, rtol=0, atol=2.0 ** -22)


@pytest.mark.parametrize("device", DEVICES)
def test_attention_nothing_to_do(device):
    cu0, cu = ends_of((), device), ends_of((0, 0), device)
    for c in (cu0, cu):
        for rows in (0, 3):
            q, k, v, dout = attention_inputs((rows,), 2, 1, 32, torch.float16, device)
            got = attention(q, k, v, dout, c)
            assert all(not t.any() for t in got.values())


def test_attention_gradient_by_differences():
    q, k, v, _ = attention_inputs((5, 1, 3), 4, 2, 3, torch.float64, "cpu", spare=2)
    cu = ends_of((5, 1, 3), "cpu")
    for causal in (False, True):
        assert torch.autograd.gradcheck(
            lambda *t: bf.packed_attention(*t, cu, causal=causal, dropout_p=0.3, seed=11), (q, k, v))


@pytest.mark.gpu
@pytest.mark.parametrize("p", [0.0, 0.2])
def test_attention_gradient_by_differences_gpu(p):
    """Along a random direction, in 32 bits: the difference quotient of a sum
    of about 4000 values of size 1 with step 2**-7 carries the roundings of
    that sum (2**-24 * 4000 * 2**7 = 0.03) and the step's third-order term
    (2**-14 of a derivative of the order of 100)."""
    q, k, v, dout = attention_inputs((40, 23), 2, 1, 32, torch.float32, "cuda")
    cu = ends_of((40, 23), "cuda")
    kw = dict(causal=True, dropout_p=p, seed=21)
    got = attention(q, k, v, dout, cu, **kw)
    g = torch.Generator().manual_seed(4)
    steps = [torch.randn(t.shape, generator=g).cuda() * 2.0 ** -7 for t in (q, k, v)]
    with torch.no_grad():
        up, down = (
            (bf.packed_attention(*(t + s * e for t, e in zip((q, k, v), steps)), cu, **kw).double()
             * dout.double()).sum() for s in (1, -1))
        along = sum((got[n].double() * e.double()).sum() for n, e in zip(("dq", "dk", "dv"), steps))
    assert abs((up - down) / 2 - along) * 2 ** 7 < 0.03 + 0.03


def refused(kind, match, f, *args, **kw):
    with pytest.raises(kind, match=match):
        f(*args, **kw)


@pytest.mark.parametrize("device", DEVICES)
def test_attention_refusals(device):
    q, k, v, _ = attention_inputs((8,), 4, 2, 16, torch.float32, device)
    cu, f = ends_of((8,), device), bf.packed_attention
    refused(ValueError, "tokens, heads, dim", f, q[0], k, v, cu)
    refused(TypeError, "one type", f, q, k.half(), v, cu)
    refused(ValueError, "do not match", f, q, k, v[:7], cu)
    refused(ValueError, "do not match", f, q, k[..., :8], v[..., :8], cu)
    refused(ValueError, "multiple", f, q[:, :3], k, v, cu)
    refused(ValueError, "multiple", f, q[:, :0], k, v, cu)
    refused(ValueError, "multiple", f, q[:, :1].expand(8, 65536, 16), k[:, :1], v[:, :1], cu)
    refused(ValueError, "too many", f, q, k, v, cu[:1].expand((1 << 24) + 1).contiguous())
    wide = torch.zeros(2, 1, 129, device=device)
    refused(ValueError, "1 to 128", f, wide, wide, wide, ends_of((2,), device))
    refused(TypeError, "int32", f, q, k, v, cu.long())
    refused(ValueError, "dense vector", f, q, k, v, cu[None])
    refused(ValueError, "scale", f, q, k, v, cu, scale=0.0)
    refused(ValueError, "scale", f, q, k, v, cu, scale=math.nan)
    for p in (-0.1, 1.0, math.nan):
        refused(ValueError, "probability", f, q, k, v, cu, dropout_p=p, seed=1)
    refused(ValueError, "offset", f, q, k, v, cu, dropout_p=0.1, seed=1, offset=1 << 32)
    refused(ValueError, "offset", f, q, k, v, cu, dropout_p=0.1, seed=1, offset=-1)
    refused(ValueError, "seed", f, q, k, v, cu, dropout_p=0.1, seed=torch.zeros(2, dtype=torch.int64, device=device))
    refused(ValueError, "seed", f, q, k, v, cu, dropout_p=0.1, seed=1.5)
    refused(ValueError, "64 bits", f, q, k, v, cu, dropout_p=0.1, seed=1 << 63)
    whole = torch.zeros(8, 1, 16, dtype=torch.int32, device=device)
    refused(TypeError, "f16", f, whole, whole, whole, cu)


def test_attention_refuses_bad_bounds_on_the_cpu():
    q, k, v, _ = attention_inputs((8,), 1, 1, 16, torch.float32, "cpu")
    for ends in ([1, 8], [0, 9], [0, 5, 3], [0, -1]):
        refused(ValueError, "rise", bf.packed_attention, q, k, v, torch.tensor(ends, dtype=torch.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("ends", [[0, 300, 0, 300, 0, 300], [-(1 << 31), (1 << 31) - 1]])
def test_attention_bad_bounds_are_cut_on_the_gpu(ends, causal):
    """Bounds that overlap or leave the tensors give what their part inside gives,
    up to roundings: their number decides over the slices of the sums."""
    inputs = attention_inputs((300,), 2, 2, 64, torch.bfloat16, "cuda")
    got = attention(*inputs, torch.tensor(ends, dtype=torch.int32, device="cuda"), causal=causal)
    close(got, attention_oracle(*inputs, [0, 300], causal, 0.125, 0.0, 0, 0))


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    q, k, v, dout = attention_inputs((8,), 2, 1, 16, torch.float32, "cuda")
    x = torch.randn(4, 16, device="cuda", requires_grad=True)
    for out, leaf in ((bf.packed_attention(q, k, v, ends_of((8,), "cuda")), q), (bf.layer_norm(x), x),
                      (bf.counter_dropout(x, 0.1, 1), x)):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(out.sum(), leaf, create_graph=True)


# ---------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------


def norm_inputs(shape, dtype, device, residual=None, weights=torch.float32, bias=True, seed=0, shift=0.0):
    g = torch.Generator().manual_seed(seed)

    def t(shape, kind, f=1.0, plus=0.0):
        return (torch.randn(shape, generator=g) * f + plus).to(kind).to(device).requires_grad_()

    x = t(shape, dtype, 2.0, shift)
    w = None if weights is None else t(shape[-1:], weights, 0.3, 1.0)
    b = t(shape[-1:], weights or torch.float32) if bias else None
    r = None if residual is None else t(shape, residual, 1.0, shift)
    dout = t(shape, residual or dtype).detach()
    return x, r, w, b, dout


def norm(x, r, w, b, dout, eps=1e-5, **kw):
    out = bf.layer_norm(x, w, b, eps, residual=r, **kw)
    assert out.is_contiguous() and out.shape == x.shape and out.dtype == (x if r is None else r).dtype
    leaves = {"dx": x, "dresidual": r, "dweight": w, "dbias": b}
    leaves = {n: t for n, t in leaves.items() if t is not None}
    got = dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), dout)))
    for n, t in leaves.items():
        assert got[n].shape == t.shape and got[n].dtype == t.dtype
    return {"out": out, **got}


def norm_agrees(device, dtype, shape, eps=1e-5, p=0.0, key=(1 << 40) + 5, offset=2, **kw):
    x, r, w, b, dout = norm_inputs(shape, dtype, device, **kw)
    got = norm(x, r, w, b, dout, eps, dropout_p=p, seed=key, offset=offset)
    close(got, norm_oracle(x, r, w, b, dout, eps, p, key, offset))
    with torch.no_grad():
        again = bf.layer_norm(x, w, b, eps, residual=r, dropout_p=p, seed=key, offset=offset)
    assert torch.equal(again, got["out"])


WIDTHS = [1, 2, 3, 8, 63, 64, 65, 200, 256, 257, 768, 1000, 1001, 1024, 2048, 2051, 4096, 5000, 8192, 8200, 12289, 16384,
          20000, 40001]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_norm_widths(device, dtype, width):
    norm_agrees(device, dtype, (5, width), seed=width)
    norm_agrees(device, dtype, (3, width), residual=dtype, weights=dtype, p=0.25, seed=width)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 2, 7, 64, 300, 2500])
def test_norm_rows(device, dtype, rows):
    norm_agrees(device, dtype, (rows, 96), residual=dtype, seed=rows)
    norm_agrees(device, dtype, (rows, 130), bias=False, seed=rows)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("width", [1, 3, 5, 7])
def test_norm_narrow_rows(device, width):
    norm_agrees(device, torch.float32, (40000, width), residual=torch.float32, p=0.1, seed=width)
    norm_agrees(device, torch.bfloat16, (700, width), weights=torch.bfloat16, seed=width)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("residual", [None, "same", torch.float32])
@pytest.mark.parametrize("weights", [None, "same", torch.float32])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("p", [0.0, 0.1])
def test_norm_variants(device, dtype, residual, weights, bias, p):
    norm_agrees(device, dtype, (2, 9, 136), residual=dtype if residual == "same" else residual,
                weights=dtype if weights == "same" else weights, bias=bias, p=p)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("width", [96, 777, 9000])
def test_norm_values_far_from_zero(device, width):
    """A row's spread is small beside its mean: the deviations are summed, not
    the squares."""
    norm_agrees(device, torch.float32, (4, width), shift=1000.0)


@pytest.mark.parametrize("device", DEVICES)
def test_norm_constant_rows(device):
    """The variance is 0: eps alone carries the root, 0 gives no number."""
    x = torch.full((3, 320), 2.5, device=device)
    assert not bf.layer_norm(x).any()
    assert torch.isnan(bf.layer_norm(x, eps=0.0)).all()


@pytest.mark.parametrize("device", DEVICES)
def test_norm_strides(device):
    g = torch.Generator().manual_seed(2)
    base = torch.randn(6, 4, 3, 160, generator=g).to(device)
    w = torch.randn(320, generator=g).to(device)[::2]
    cases = [base[:, :, 1], base[:, 1], base.transpose(0, 1), base[0, 0, 0], base[..., 3:103], base[:, :1, 0],
             base[0, :, :, 0].t(), base[:1].expand(5, 4, 3, 160), base[::2, 1:3]]
    for x in cases:
        weight = w[: x.shape[-1]]
        for r in (None, x.flip(0)):
            dense = norm(*(t if t is None else t.contiguous().requires_grad_() for t in (x, r, weight, weight)),
                         torch.ones(x.shape, device=device), dropout_p=0.2, seed=4)
            t = [None if t is None else t.detach().requires_grad_() for t in (x, r, weight, weight)]
            got = norm(*t, torch.ones((), device=device).expand(x.shape), dropout_p=0.2, seed=4)
            for name in dense:
                assert torch.equal(got[name], dense[name]), (name, x.shape)


@pytest.mark.parametrize("device", DEVICES)
def test_norm_single_leaves(device):
    """Only what needs a gradient gets one, with the same values."""
    x, r, w, b, dout = norm_inputs((11, 96), torch.float16, device, residual=torch.float16)
    for p in (0.0, 0.3):
        whole = norm(x, r, w, b, dout, dropout_p=p, seed=1)
        for name, leaf in (("dx", x), ("dresidual", r), ("dweight", w), ("dbias", b)):
            x1, r1, w1, b1 = (t if t is leaf else t.detach() for t in (x, r, w, b))
            out = bf.layer_norm(x1, w1, b1, residual=r1, dropout_p=p, seed=1)
            assert torch.equal(torch.autograd.grad(out, leaf, dout)[0], whole[name])


@pytest.mark.parametrize("device", DEVICES)
def test_norm_no_rows(device):
    x, _, w, b, dout = norm_inputs((0, 64), torch.float32, device)
    got = norm(x, None, w, b, dout)
    assert got["out"].shape == (0, 64) and not got["dweight"].any() and not got["dbias"].any()


def test_norm_gradient_by_differences():
    g = torch.Generator().manual_seed(0)
    x, r = (torch.randn(3, 7, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(2))
    w, b = (torch.randn(7, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(2))
    assert torch.autograd.gradcheck(
        lambda x, r, w, b: bf.layer_norm(x, w, b, residual=r, dropout_p=0.3, seed=6), (x, r, w, b))


@pytest.mark.parametrize("device", DEVICES)
def test_norm_refusals(device):
    x = torch.zeros(4, 16, device=device)
    w, f = torch.ones(16, device=device), bf.layer_norm
    refused(ValueError, "last dimension", f, x[0, 0])
    refused(ValueError, "last dimension", f, x[:, :0])
    refused(ValueError, "last dimension", f, x[:, :1].expand(4, (1 << 26) + 1))
    refused(ValueError, "vectors", f, x, w[:8])
    refused(ValueError, "vectors", f, x, w, x)
    refused(TypeError, "f32 or of the input's type", f, x, w.half())
    refused(TypeError, "one type", f, x.half(), w.half(), w)
    refused(ValueError, "input's shape", f, x, w, residual=x[:2])
    refused(TypeError, "f32 or of the input's type", f, x, w, residual=x.half())
    refused(ValueError, "eps", f, x, w, eps=-1.0)
    refused(ValueError, "eps", f, x, w, eps=math.inf)
    refused(ValueError, "probability", f, x, w, dropout_p=1.0, seed=1)
    refused(TypeError, "f16", f, x.int())


# ---------------------------------------------------------------------------
# dropout
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (3, 5), (255,), (64, 65), (3, 1001), (2, 3, 4, 5), (40000,)])
@pytest.mark.parametrize("p", [0.1, 0.75])
def test_dropout(device, dtype, shape, p):
    """Forward and backward are x and dy times the factors of the definition,
    rounded once: the product of two 32-bit numbers is rounded to 32 bits and
    then to the type."""
    g = torch.Generator().manual_seed(len(shape))
    x, dy = (torch.randn(shape, generator=g).to(dtype).to(device) for _ in range(2))
    x.requires_grad_()
    key, offset = (7 << 35) + 123456789, 4000000000
    y = bf.counter_dropout(x, p, key, offset=offset)
    assert y.dtype == dtype and y.shape == x.shape
    dx, = torch.autograd.grad(y, x, dy)
    keep = flat_keep(shape, p, key, offset)
    for got, t in ((y, x), (dx, dy)):
        want = t.detach().cpu().double() * keep
        off = (got.detach().cpu().double() - want).abs()
        assert (off <= rounding(dtype, want) + 2 * F32 * want.abs()).all()
        assert torch.equal(got.cpu() == 0, (keep == 0) | (t.detach().cpu() == 0))


@pytest.mark.parametrize("device", DEVICES)
def test_dropout_drops_what_it_should(device):
    """Of n elements np are dropped, within six standard deviations; seeds,
    offsets and places give other masks; a dropped NaN is 0."""
    n, p = 1 << 18, 0.3
    x = torch.ones(n, device=device)
    masks = [bf.counter_dropout(x, p, s, offset=o) == 0 for s, o in ((1, 0), (2, 0), (1, 1), (1 << 32, 0), (-1, 0))]
    for m in masks:
        assert abs(float(m.double().sum()) - n * p) < 6 * math.sqrt(n * p * (1 - p))
    for i, a in enumerate(masks):
        for b in masks[:i]:
            agree = p * p + (1 - p) ** 2
            same = float((a == b).double().sum())
            assert abs(same - n * agree) < 6 * math.sqrt(n * agree * (1 - agree))
    bad = bf.counter_dropout(torch.full((n,), math.nan, device=device), p, 1)
    assert torch.equal(bad == 0, masks[0]) and torch.equal(torch.isnan(bad), ~masks[0])
    assert torch.equal(bf.counter_dropout(x, 0.0, 1), x)
    assert torch.equal(bf.counter_dropout(x, 1e-6, 1), x)  # below 2**-17


@pytest.mark.parametrize("device", DEVICES)
def test_dropout_seeds(device):
    """An int, a tensor and torch's generator as the source."""
    x = torch.ones(1000, device=device)
    seed = torch.tensor([-5 - (3 << 40)], device=device)
    a = bf.counter_dropout(x, 0.5, seed, offset=3)
    assert torch.equal(a, bf.counter_dropout(x, 0.5, int(seed), offset=3))
    torch.manual_seed(1)
    b, c = bf.counter_dropout(x, 0.5), bf.counter_dropout(x, 0.5)
    assert not torch.equal(b, c)
    torch.manual_seed(1)
    assert torch.equal(b, bf.counter_dropout(x, 0.5))


@pytest.mark.parametrize("device", DEVICES)
def test_dropout_strides_and_emptiness(device):
    x = torch.arange(1.0, 61.0, device=device).view(3, 4, 5)
    for t in (x.transpose(0, 2), x[:, 1:], x[:1].expand(6, 4, 5), x[..., 2], x[:0]):
        assert torch.equal(bf.counter_dropout(t, 0.4, 8), bf.counter_dropout(t.contiguous(), 0.4, 8))


@pytest.mark.parametrize("device", DEVICES)
def test_dropout_refusals(device):
    x = torch.zeros(4, device=device)
    for p in (-0.1, 1.0, math.nan):
        refused(ValueError, "probability", bf.counter_dropout, x, p, 1)
    refused(ValueError, "offset", bf.counter_dropout, x, 0.1, 1, 1 << 32)
    refused(TypeError, "f16", bf.counter_dropout, x.int(), 0.1, 1)


# ---------------------------------------------------------------------------
# streams, graphs, repeatability
# ---------------------------------------------------------------------------


def all_three(q, k, v, dout, cu, x, r, w, b, dy, seed):
    got = attention(q, k, v, dout, cu, causal=True, dropout_p=0.1, seed=seed, offset=1)
    got.update({"n" + n: t for n, t in norm(x, r, w, b, dy, dropout_p=0.1, seed=seed, offset=2).items()})
    y = bf.counter_dropout(x, 0.1, seed, offset=3)
    got["y"], got["ydx"] = y, torch.autograd.grad(y, x, dy)[0]
    return [t.detach() for t in got.values()]


def all_inputs(seed):
    q, k, v, dout = attention_inputs((150, 70, 9), 6, 2, 64, torch.bfloat16, "cuda", spare=4, seed=seed)
    x, r, w, b, dy = norm_inputs((300, 768), torch.bfloat16, "cuda", residual=torch.bfloat16, seed=seed)
    return q, k, v, dout, ends_of((150, 70, 9), "cuda"), x, r, w, b, dy, torch.tensor([seed + 99], device="cuda")


@pytest.mark.gpu
def test_results_repeat():
    """Every bit, however often."""
    inputs = all_inputs(0)
    first = all_three(*inputs)
    for _ in range(5):
        for a, b in zip(all_three(*inputs), first):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_on_another_stream():
    want = all_three(*all_inputs(1))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = all_three(*all_inputs(1))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_two_streams_at_once():
    inputs = [all_inputs(2), all_inputs(3)]
    want = [all_three(*i) for i in inputs]
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for n, side in enumerate(sides):
            with torch.cuda.stream(side):
                got[n].append(all_three(*inputs[n]))
    torch.cuda.synchronize()
    for n in range(2):
        for run in got[n]:
            for a, b in zip(run, want[n]):
                assert torch.equal(a, b)


@pytest.mark.gpu
def test_in_captured_graphs():
    """Forward and backward in a graph, replayed with new inputs and a new
    seed between eager work; two graphs share nothing."""
    torch.cuda.synchronize()
    static = [all_inputs(4), all_inputs(5)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in static:
            all_three(*s)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for s in static:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(all_three(*s))
        graphs.append(graph)
    for step in range(4):
        fresh = [all_inputs(10 + 2 * step), all_inputs(11 + 2 * step)]
        want = [all_three(*f) for f in fresh]
        with torch.no_grad():
            for s, f in zip(static, fresh):
                for a, b in zip(s, f):
                    a.copy_(b)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for got, w in zip(outs, want):
            for a, b in zip(got, w):
                assert torch.equal(a, b)


@pytest.mark.gpu
def test_torch_code_on_the_gpu(monkeypatch):
    """Without the extension: an error, or the torch code when that is asked for,
    with the same masks."""
    q, k, v, dout = attention_inputs((9, 40), 4, 2, 16, torch.float32, "cuda", spare=3)
    cu, x = ends_of((9, 40), "cuda"), torch.randn(5, 24, device="cuda", requires_grad=True)
    kw = dict(dropout_p=0.3, seed=5, offset=2)

    def results():
        y = bf.counter_dropout(x, 0.3, 5, 2)
        got = attention(q, k, v, dout, cu, causal=True, **kw)
        return {**got, "y": y, "norm": bf.layer_norm(x, residual=x, **kw)}

    native = results()
    monkeypatch.setattr(hip_ext, "_C", None)
    with pytest.raises(RuntimeError, match="requires the native HIP"):
        results()
    monkeypatch.setenv("BLUEFOG_ALLOW_TORCH_FALLBACK", "1")
    want = attention_oracle(q, k, v, dout, cu.tolist(), True, 0.25, 0.3, 5, 2)
    plain = results()
    close({n: plain[n] for n in want}, want)
    close({n: native[n] for n in want}, want)
    assert torch.equal(native["y"], plain["y"])
    # both in 32 bits: sums of 24 values below 16 move the mean by 24 F32 * 16 at most and 1 / sigma (above 0.5
    # of values of size 1) by 26 F32 of itself, of results below 5
    torch.testing.assert_close(native["norm"], plain["norm"], rtol=0, atol=2 * (2 * 24 * 16 + 5 * 26) * F32)


# ---------------------------------------------------------------------------
# torch's other ways to call a function
# ---------------------------------------------------------------------------


def calls_of_all(device, dtype=torch.float32):
    """[(function of tensors, those tensors)], every differentiable argument among them."""
    q, k, v, _ = (t.detach() for t in attention_inputs((5, 9), 4, 2, 16, dtype, device))
    x, r, w, b, _ = (t.detach() for t in norm_inputs((6, 24), dtype, device, residual=dtype, weights=dtype))
    cu, kw = ends_of((5, 9), device), dict(dropout_p=0.3, seed=5, offset=2)
    return [
        (lambda q, k, v: bf.packed_attention(q, k, v, cu, causal=True, **kw), (q, k, v)),
        (lambda x, r, w, b: bf.layer_norm(x, w, b, residual=r, **kw), (x, r, w, b)),
        (lambda x: bf.counter_dropout(x, 0.3, 5, 2), (x,)),
    ]


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(3))
def test_forward_mode_is_refused_on_the_gpu(which):
    """The kernels take no tangents along: an argument that carries one is refused,
    whether or not it requires a gradient, in the backward pass too."""
    from torch.autograd import forward_ad

    f, args = calls_of_all("cuda")[which]
    leaf = args[0].clone().requires_grad_()
    with forward_ad.dual_level():
        for i, t in enumerate(args):
            for needs in (False, True):
                dual = forward_ad.make_dual(t.clone().requires_grad_(needs), torch.ones_like(t))
                refused(NotImplementedError, "forward-mode", f, *args[:i], dual, *args[i + 1:])
                with torch.no_grad():
                    refused(NotImplementedError, "forward-mode", f, *args[:i], dual, *args[i + 1:])
        out = f(leaf, *args[1:])
        dual = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
        refused(NotImplementedError, "forward-mode", torch.autograd.grad, out, leaf, dual)


@pytest.mark.parametrize("which", range(3))
def test_forward_mode_on_the_cpu(which):
    """The torch code's tangents against J t from two backward passes, in 64 bits:
    sums of at most 40 terms of size below 100."""
    from torch.autograd import forward_ad

    f, args = calls_of_all("cpu", torch.float64)[which]
    g = torch.Generator().manual_seed(8)
    along = tuple(torch.randn(t.shape, generator=g, dtype=t.dtype) for t in args)
    with forward_ad.dual_level():
        got = forward_ad.unpack_dual(f(*(forward_ad.make_dual(t, e) for t, e in zip(args, along)))).tangent
    _, want = torch.autograd.functional.jvp(f, args, along)
    torch.testing.assert_close(got, want, rtol=0, atol=40 * 100 * 2.0 ** -52)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", range(3))
def test_traced(device, which):
    """A trace holds the operator, not the memory of its first result: new inputs
    give what the function gives, gradients too."""
    f, args = calls_of_all(device)[which]
    traced = torch.jit.trace(f, args)
    if device == "cuda":
        assert "bluefog_amd::" in str(traced.graph)
    for factor in (1.0, -2.0, 0.5):
        new = [(t * factor).requires_grad_() for t in args]
        got, want = traced(*new), f(*new)
        assert torch.equal(got, want)
        for a, b in zip(torch.autograd.grad(got.sum(), new), torch.autograd.grad(want.sum(), new)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("device", DEVICES)
def test_traced_seed(device):
    """A seed that is a tensor is an input of the trace."""
    x, seed = torch.ones(1000, device=device), torch.tensor([3], device=device)
    if device == "cpu":
        pytest.skip("the torch code reads the seed on the host: a trace keeps its value")
    traced = torch.jit.trace(lambda x, s: bf.counter_dropout(x, 0.5, s), (x, seed))
    for s in (3, 4):
        assert torch.equal(traced(x, seed.fill_(s)), bf.counter_dropout(x, 0.5, s))


def test_fake_tensors_are_refused():
    """They say that they are on a GPU and have no memory: a kernel would read
    address 0. Nothing is launched, so this runs without a GPU as well."""
    from torch._subclasses import FakeTensorMode

    if not hip_ext.has_extension():
        pytest.skip("the native extension is not built")
    with FakeTensorMode():
        q, x = torch.empty(8, 2, 16, device="cuda"), torch.empty(4, 24, device="cuda")
        cu, seed = torch.empty(2, dtype=torch.int32, device="cuda"), torch.empty(1, dtype=torch.int64, device="cuda")
        for needs in (False, True):
            q.requires_grad_(needs)
            x.requires_grad_(needs)
            refused(NotImplementedError, "memory", bf.packed_attention, q, q, q, cu)
            refused(NotImplementedError, "memory", bf.packed_attention, q, q, q, cu, dropout_p=0.1, seed=seed)
            refused(NotImplementedError, "memory", bf.layer_norm, x, residual=x)
            refused(NotImplementedError, "memory", bf.counter_dropout, x, 0.1, seed)


@pytest.mark.gpu
def test_tensors_without_memory_are_refused():
    """Inputs and gradients whose storage was freed, and results that a mode
    makes fake, in both directions."""
    from torch._subclasses import FakeTensorMode

    def freed(t):
        t = t.clone()
        t.untyped_storage().resize_(0)
        assert t.data_ptr() == 0
        return t

    for f, args in calls_of_all("cuda"):
        for i, t in enumerate(args):
            refused(NotImplementedError, "memory", f, *args[:i], freed(t), *args[i + 1:])
        with FakeTensorMode(allow_non_fake_inputs=True):
            refused(NotImplementedError, "memory", f, *args)
        leaf = args[0].clone().requires_grad_()
        out = f(leaf, *args[1:])
        refused(NotImplementedError, "memory", torch.autograd.grad, out, leaf, freed(torch.ones_like(out)))


@pytest.mark.gpu
def test_mapped_over_a_dimension():
    """torch.vmap runs the operator slice by slice, and differentiates through it."""
    x = torch.randn(3, 4, 32, device="cuda")
    w = torch.rand(32, device="cuda", requires_grad=True)
    assert torch.equal(torch.vmap(lambda t: bf.counter_dropout(t, 0.3, 5))(x),
                       torch.stack([bf.counter_dropout(t, 0.3, 5) for t in x]))
    got, want = torch.vmap(lambda t: bf.layer_norm(t, w))(x), bf.layer_norm(x, w)
    assert torch.equal(got, want)
    a, b = (torch.autograd.grad(y.sum(), w)[0] for y in (got, want))
    # sums of 12 terms of size below 8 in another order
    assert (a - b).abs().max() <= 2 * 12 * 12 * 8 * F32


# ---------------------------------------------------------------------------
# many sequences
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_many_sequences(device, dtype, causal):
    """Over a thousand, some of several tiles, empty ones among them."""
    g = torch.Generator().manual_seed(6)
    lengths = torch.tensor([0, 0, 1, 2, 3, 17, 140])[torch.randint(0, 7, (1100,), generator=g)].tolist()
    lengths[500] = 300
    attention_agrees(device, dtype, lengths, 12, 4, 16, causal=causal, spare=150)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
def test_attention_very_many_sequences(causal):
    """2**17 of one token: the output is v, and the gradients are 0 and dO."""
    n = 1 << 17
    q, k, v, dout = attention_inputs((n,), 12, 12, 8, torch.float16, "cuda")
    cu = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    got = attention(q, k, v, dout, cu, causal=causal)
    assert torch.equal(got["out"], v) and torch.equal(got["dv"], dout)
    assert not got["dq"].any() and not got["dk"].any()


def test_attention_refuses_more_tiles_than_a_launch_holds():
    """Before the forward pass, also where only the backward pass has no room
    for them. Fake tensors: nothing is launched."""
    from torch._subclasses import FakeTensorMode

    if not hip_ext.has_extension():
        pytest.skip("the native extension is not built")
    with FakeTensorMode():
        def call(sequences, heads, dim, dtype, needs=False, tokens=8):
            q = torch.empty(tokens, heads, dim, dtype=dtype, device="cuda", requires_grad=needs)
            bf.packed_attention(q, q, q, torch.empty(sequences + 1, dtype=torch.int32, device="cuda"))

        refused(ValueError, "too many", call, 1 << 23, 2, 64, torch.float32)
        refused(ValueError, "too many", call, 1 << 18, 64, 64, torch.bfloat16)
        refused(ValueError, "too many", call, 1 << 23, 1, 128, torch.bfloat16, True)
        refused(ValueError, "too many", call, 0, 128, 8, torch.float16, tokens=1 << 24)
        # these have room: they reach the next refusal
        refused(NotImplementedError, "memory", call, 1 << 23, 1, 128, torch.bfloat16)
        refused(NotImplementedError, "memory", call, 1 << 23, 1, 128, torch.float32, True)
        refused(NotImplementedError, "memory", call, (1 << 24) - 9, 1, 64, torch.float16, True)
        refused(NotImplementedError, "memory", call, (1 << 24) - 1, 65535, 64, torch.float16, tokens=0)


# ---------------------------------------------------------------------------
# values that are infinite or no number
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [40, 64, 128, 57])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_attention_infinite_values(device, dtype, causal, dim, p):
    """An infinite v is infinite in every row that sees its key with a
    probability above 0, wherever the key lies; no number if the probability is
    dropped or another such v is of the other sign; nothing to rows that do not
    see it, and to other columns. The rest keeps its bits on the GPU, where the
    sums are the same; on the CPU it has the roundings of a sum of n terms."""
    if device == "cpu" and dim != 40:
        pytest.skip("the torch code does not depend on the head size")
    n = 700 if device == "cuda" else 70
    for lengths, bad in [((150, 40), [(140, 3, math.inf), (149, 5, -math.inf), (160, 7, math.inf)]),
                         ((150, 40), [(2, 0, math.inf), (70, 0, -math.inf), (189, 6, -math.inf), (100, 1, math.nan)]),
                         ((n,), [(n - 10, 1, math.inf), (31, 2, -math.inf), (n - 1, 4, math.inf)])]:
        q, k, v, _ = attention_inputs(lengths, 2, 1, dim, dtype, device)
        cu, kw = ends_of(lengths, device), dict(causal=causal, dropout_p=p, seed=3)
        with torch.no_grad():
            clean_v = v.detach().clone()
            for row, column, value in bad:
                v[row, 0, column], clean_v[row, 0, column] = value, 0
            clean = bf.packed_attention(q, k, clean_v, cu, **kw).cpu()
            got = bf.packed_attention(q, k, v, cu, **kw).cpu()
        want = clean.double()
        ends = cu.tolist()
        for row, column, value in bad:
            begin, end = next((a, b) for a, b in zip(ends, ends[1:]) if a <= row < b)
            keep = attention_keep(2, begin, end - begin, p, 3, 0)[:, :, row - begin] > 0
            for i in range(row if causal else begin, end):
                for h in range(2):
                    want[i, h, column] += value if keep[h, i - begin] else math.nan
        fine = torch.isfinite(want)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got[~fine].double().nan_to_num(7.0), want[~fine].nan_to_num(7.0))
        off = (got.double() - want)[fine].abs()
        if device == "cuda":
            assert not off.any()
        else:
            size = v[torch.isfinite(v)].abs().max().item() / (1 - p)
            assert (off <= 2 * (max(lengths) + 16) * F32 * size + 2 * rounding(dtype, want[fine])).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
def test_attention_infinite_value_of_small_probability(device, dtype, causal):
    """A probability of e**-25, which f16 does not hold, is above 0; one whose score
    is -inf is 0."""
    n = 90
    q, k, v, _ = (t.detach() for t in attention_inputs((n,), 1, 1, 64, dtype, device))
    q[:, 0, 0], k[:, 0, 0], k[4, 0] = 20.0, 0.0, 0.0
    k[4, 0, 0] = -10.0  # the score of key 4: -200 / 8; the others' are of size 1
    v[4, 0, 9] = math.inf
    got = bf.packed_attention(q, k, v, ends_of((n,), device), causal=causal)
    first = 4 if causal else 0
    assert (got[first:, 0, 9] == math.inf).all() and torch.isfinite(got[:first]).all()
    k[4, 0, 0] = -math.inf
    got = bf.packed_attention(q, k, v, ends_of((n,), device), causal=causal)
    assert torch.isnan(got[first:, 0, 9]).all() and torch.isfinite(got[:first]).all()
    assert torch.isfinite(got[first:, 0, :9]).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attention_causal_rows_ignore_later_values(device, dtype, bad):
    """A later key or value that is not a number leaves earlier rows alone, on the
    CPU too; there the last bits may differ, since rows are summed one by one."""
    for n, at in ((50, 37), (300, 150)):
        q, k, v, _ = (t.detach() for t in attention_inputs((n,), 2, 2, 64, dtype, device))
        cu = ends_of((n,), device)
        clean = bf.packed_attention(q, k, v, cu, causal=True)
        size = v.abs().max().item()
        k[at], v[at] = bad, bad
        got = bf.packed_attention(q, k, v, cu, causal=True)
        off = (got[:at].cpu().double() - clean[:at].cpu().double()).abs()
        assert (off <= 2 * (n + 16) * F32 * size + 2 * rounding(dtype, clean[:at].cpu().double())).all()
        assert not torch.isfinite(got[at:]).any()


@pytest.mark.parametrize("device", DEVICES)
def test_numbers_that_leave_32_bits_are_refused(device):
    """A scale or an eps that is 0 or infinite as the kernels hold it."""
    q, k, v, _ = attention_inputs((8,), 1, 1, 16, torch.float32, device)
    cu, x = ends_of((8,), device), torch.ones(3, 16, device=device)
    for scale in (1e-60, 1e39):
        refused(ValueError, "scale", bf.packed_attention, q, k, v, cu, scale=scale)
    for eps in (1e-60, 1e39):
        refused(ValueError, "eps", bf.layer_norm, x, eps=eps)
    if device == "cpu":  # 64-bit tensors hold them
        wide = [t.double() for t in (q, k, v)]
        assert torch.isfinite(bf.packed_attention(*wide, cu, scale=1e-60)).all()
        assert not bf.layer_norm(x.double(), eps=1e-60).any()


# ---------------------------------------------------------------------------
# how exact half-precision gradients are
# ---------------------------------------------------------------------------


def times_the_last_rounding(got, exact, dtype):
    """The error's size as a multiple of what rounding the exact result costs."""
    own = exact.to(dtype).double() - exact
    return float((got.detach().cpu().double() - exact).norm() / own.norm())


def exact_gradients(q, k, v, dout, causal, rounded=None):
    """out, dq, dk, dv in 64 bits for one sequence. ``rounded``: a mistake that
    is planted, 'dS' rounded to the type in front of its products (f16: times a
    power of two that keeps a row's largest near the type's), or 'delta' from
    the rounded output."""
    Q, K, V, G = (t.detach().cpu().double().transpose(0, 1) for t in (q, k, v, dout))
    group, scale = Q.shape[0] // K.shape[0], Q.shape[2] ** -0.5
    K, V = K.repeat_interleave(group, 0), V.repeat_interleave(group, 0)
    S = Q @ K.transpose(1, 2) * scale
    if causal:
        S = S.masked_fill(~torch.ones(S.shape[1:], dtype=torch.bool).tril(), -math.inf)
    P = torch.softmax(S, 2)
    O = P @ V
    delta = (G * (O.to(q.dtype).double() if rounded == "delta" else O)).sum(2, keepdim=True)
    dS = P * (G @ V.transpose(1, 2) - delta)
    if rounded == "dS":
        power = 2.0 ** -torch.frexp(dS.abs().amax(2, keepdim=True).clamp_min(1e-30)).exponent
        dS = (dS * power).to(q.dtype).double() / power
    shared = [t.unflatten(0, (-1, group)).sum(1) for t in (dS.transpose(1, 2) @ Q * scale, P.transpose(1, 2) @ G)]
    return {n: t.transpose(0, 1) for n, t in zip(("out", "dq", "dk", "dv"), (O, dS @ K * scale, *shared))}


# Queries and keys of size 2: scores of 2 * 2 * sqrt(dim) / sqrt(dim) = 4 let softmax
# pick keys that lie along the query. Those have a common part, and delta's error,
# which goes into all dS of a row at once, moves dq by it.
EXACT = [(1200, 4, 2, 64, False), (1200, 4, 2, 64, True), (900, 4, 1, 128, True), (900, 2, 2, 128, False), (500, 6, 2, 80, True)]
# 1: nothing but the last rounding. A rounding more, of a value of the same relative
# precision in every term of a sum with signs at random, adds as much again: sqrt(2).
# dS carries what its rounding took, so dq and dk stay below that; P is rounded
# once in front of out and dv, and nothing else is: below sqrt(3), two more.
MOST_TIMES = {"dq": 1.3, "dk": 1.3, "out": 1.5, "dv": 1.5}


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", EXACT)
def test_attention_is_as_exact_as_its_last_rounding(device, dtype, case):
    n, heads, kv_heads, dim, causal = case
    q, k, v, dout = attention_inputs((n,), heads, kv_heads, dim, dtype, device, seed=n, factor=2.0)
    got = attention(q, k, v, dout, ends_of((n,), device), causal=causal)
    exact = exact_gradients(q, k, v, dout, causal)
    times = {name: times_the_last_rounding(got[name], exact[name], dtype) for name in exact}
    assert all(times[name] < MOST_TIMES[name] for name in times), times


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", EXACT)
def test_a_rounding_more_is_found(dtype, case):
    """The bounds of the test above tell: dS rounded once, or delta from the
    rounded output, leaves dq and dk outside."""
    n, heads, kv_heads, dim, causal = case
    q, k, v, dout = attention_inputs((n,), heads, kv_heads, dim, dtype, "cpu", seed=n, factor=2.0)
    exact = exact_gradients(q, k, v, dout, causal)
    for mistake in ("dS", "delta"):
        off = exact_gradients(q, k, v, dout, causal, mistake)
        times = {m: times_the_last_rounding(off[m].to(dtype), exact[m], dtype) for m in ("dq", "dk")}
        assert all(times[m] > MOST_TIMES[m] for m in times), (mistake, times)


# ---------------------------------------------------------------------------
# norms of more rows than a launch has workgroups for at once
# ---------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,width", [(16400 + 3, 96), (8200 + 3, 1001), (4200, 2051), (2100, 4096), (1100, 5000),
                                        (1030, 8192), (600, 12289), (1030, 16385), (70, 40001), (9000, 5)])
def test_norm_takes_row_after_row(dtype, rows, width):
    """A workgroup has 4 rows at once up to a width of 1024 and 1 above; 8192 rows
    are under way in the forward pass then (4096 in the backward pass), 2048 (1024)
    up to 4096 columns, 1024 (512) up to 8192 and 512 (256) beyond, in the wide
    kernels 64 for the sums over rows: every workgroup here takes more than one,
    some one more than others."""
    norm_agrees("cuda", dtype, (rows, width), seed=width)
    norm_agrees("cuda", dtype, (rows, width), residual=dtype, weights=dtype, p=0.2, seed=width + 1)


@pytest.mark.gpu
def test_many_sequences_in_captured_graphs():
    """The table of the tiles is made anew at every replay, from the bounds of
    that replay; two graphs' tables are their own."""
    g = torch.Generator().manual_seed(3)

    def bounds(most):
        ends = torch.randint(0, most + 1, (150,), generator=g).sort().values
        ends[0] = 0
        return ends.to(torch.int32).cuda()

    static = [(*attention_inputs((n,), 4, 2, 64, torch.bfloat16, "cuda", seed=n), bounds(n)) for n in (900, 2000)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in static:
            attention(*s, causal=True)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for s in static:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(attention(*s, causal=True))
        graphs.append(graph)
    for _ in range(4):
        for s in static:
            s[4].copy_(bounds(len(s[0])))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for s, out in zip(static, outs):
            for name, t in attention(*s, causal=True).items():
                assert torch.equal(out[name], t)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("causal", [False, True])
def test_attention_mapped_over_a_dimension(device, causal):
    """torch.vmap over heads of batches of their own: slice by slice on the GPU;
    batched products on the CPU, whose sums of at most 9 terms may have
    another order."""
    g = torch.Generator().manual_seed(9)
    q = torch.randn(3, 14, 2, 8, generator=g).to(device)
    cu = ends_of((5, 9), device)
    got = torch.vmap(lambda t: bf.packed_attention(t, t, t, cu, causal=causal))(q)
    want = torch.stack([bf.packed_attention(t, t, t, cu, causal=causal) for t in q])
    assert (got - want).abs().max() <= (0 if device == "cuda" else 64 * F32 * float(q.abs().max()))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", range(5))
def test_negated_views(device, which):
    """The imaginary part of a conjugate is a view whose values are the memory's
    times -1: as an argument and as an upstream gradient. Its last dimension
    counts as dense where it has one value."""
    def negated(t):
        view = torch.imag(torch.complex(torch.zeros_like(t), -t).conj())
        assert view.is_neg() and torch.equal(view, t)
        return view

    calls = calls_of_all(device)
    q, k, v, _ = (t.detach() for t in attention_inputs((5, 9), 4, 2, 1, torch.float32, device))
    cu = ends_of((5, 9), device)
    calls.append((lambda q, k, v: bf.packed_attention(q, k, v, cu), (q, k, v)))
    x, r, w, b, _ = (t.detach() for t in norm_inputs((6, 1), torch.float32, device, residual=torch.float32))
    calls.append((lambda x, r, w, b: bf.layer_norm(x, w, b, residual=r), (x, r, w, b)))
    f, args = calls[which]
    leaves = [t.clone().requires_grad_() for t in args]
    want = f(*leaves)
    up = torch.randn(want.shape, generator=torch.Generator().manual_seed(1)).to(device)
    want_grads = torch.autograd.grad(want, leaves, up)
    views = [negated(t).detach().requires_grad_() for t in args]
    got = f(*views)
    assert torch.equal(got, want)
    for g, w in zip(torch.autograd.grad(got, views, negated(up)), want_grads):
        assert torch.equal(g, w)


@pytest.mark.parametrize("device", DEVICES)
def test_in_inference_mode(device):
    for f, args in calls_of_all(device):
        with torch.inference_mode():
            got = f(*args)
        assert torch.equal(got, f(*args))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [16, 7])
def test_saved_tensors_in_another_layout(dim):
    """Hooks that keep what the forward pass saves, and bring it back with its
    values but other strides, give the same gradients."""
    device = "cuda"
    q, k, v, dout = attention_inputs((70,) + (3,) * 80, 4, 2, dim, torch.bfloat16, device)
    cu = ends_of((70,) + (3,) * 80, device)
    x, r, w, b, dy = norm_inputs((6, 24), torch.bfloat16, device, residual=torch.bfloat16)
    kw = dict(dropout_p=0.2, seed=torch.tensor([3], device=device))

    def results():
        return [bf.packed_attention(q, k, v, cu, **kw), bf.layer_norm(x, w, b, residual=r, **kw)]

    def grads(outs):
        return [*torch.autograd.grad(outs[0], (q, k, v), dout), *torch.autograd.grad(outs[1], (x, r, w, b), dy)]

    want = grads(results())
    apart = []

    def unpack(t):
        t = torch.stack([t, t + 1], -1)[..., 0]
        apart.append(t.dim() and t.stride(-1) == 2)
        return t

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), unpack):
        outs = results()
    for g, t in zip(grads(outs), want):
        assert torch.equal(g, t)
    assert any(apart)


def test_dropout_refuses_more_than_a_launch_holds():
    """With what it is, before anything runs. Fake tensors: nothing is launched."""
    from torch._subclasses import FakeTensorMode

    if not hip_ext.has_extension():
        pytest.skip("the native extension is not built")
    with FakeTensorMode():
        x = torch.empty((1 << 35) - 2048, dtype=torch.float16, device="cuda")
        refused(NotImplementedError, "memory", bf.counter_dropout, x, 0.1, 1)
        x = torch.empty((1 << 35) - 2047, dtype=torch.float16, device="cuda")
        refused(ValueError, "at most", bf.counter_dropout, x, 0.1, 1)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
def test_attention_many_sequences_with_dropout(device, dtype, causal):
    """Their masks go by the packed row, whichever way its sequence is found."""
    lengths = [n % 7 for n in range(100)] + [135, 20]
    attention_agrees(device, dtype, lengths, 4, 2, 32, causal=causal, p=0.2, spare=3)
