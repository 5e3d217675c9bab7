"""GPU tests of the reading operators (libartread.so through its C ABI) against plain implementations in 64
bits, at the sizes and masks where they can go wrong.

Tolerances.  U[t] = finfo(t).eps / 2 is the relative error of one rounding to t; U32 that of a 32-bit step.
Every bound below counts the roundings the operators make: inputs are exact, sums and statistics are 32 bits,
the weights P and their gradients dS are rounded once to the inputs' type before the second product, results
once more.  A 32-bit sum of n terms is off by at most n * U32 * sum|term| in any order."""
import math
import threading

import numpy as np
import pytest
import torch

from art_amd import reader as rd
from art_amd import token_store as ts

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
U = {t: torch.finfo(t).eps / 2 for t in (F16, BF16, F32)}
U32 = U[F32]
TINY = {t: torch.finfo(t).smallest_normal * torch.finfo(t).eps for t in (F16, BF16, F32)}  # one subnormal step


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def within(got, want, bound):
    """|got - want| <= bound everywhere, infinities and NaN equal."""
    got, want = got.detach().double(), want.detach().double()
    assert got.shape == want.shape
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got))
    off = torch.where(fine, (got - want).abs() - bound, torch.full_like(want, -1.0))
    assert float(off.max()) <= 0, "off by %.3g more than the bound" % float(off.max())


# ---- embedding ------------------------------------------------------------------------------------
def embed_case(n, length, vocab, dim, dtype, seed, token_dtype=torch.int32, base=0, zipf=True):
    g = gen(seed)
    if zipf:
        tokens = (torch.rand((n, length), device="cuda", generator=g) * math.log(vocab + 1)).exp().long() - 1
        tokens.clamp_(0, vocab - 1)
    else:
        tokens = torch.randint(0, vocab, (n, length), device="cuda", generator=g)
    tokens = (tokens + base).to(token_dtype)
    lengths = torch.randint(-1, length + 2, (n,), device="cuda", generator=g, dtype=torch.int32)
    table = torch.randn((vocab, dim), device="cuda", generator=g).to(dtype)
    return tokens, lengths, table


def valid_of(tokens, lengths, vocab, base=0):
    inside = torch.arange(tokens.shape[-1], device="cuda") < lengths[..., None]
    return inside & (tokens >= base) & (tokens.long() - base < vocab)


def embed_ref(tokens, lengths, table, scale, base=0):
    ok = valid_of(tokens, lengths, table.shape[0], base)
    rows = table.double()[torch.where(ok, tokens.long() - base, 0)] * scale
    return torch.where(ok[..., None], rows, 0.0)


def grad_ref(grad, tokens, lengths, vocab, scale, base=0):
    """(64-bit gradient, sum of absolute terms, number of terms)"""
    ok = valid_of(tokens, lengths, vocab, base).flatten()
    key, rows = (tokens.long() - base).flatten()[ok], grad.double().flatten(0, -2)[ok]
    out = [torch.zeros((vocab, grad.shape[-1]), dtype=torch.float64, device="cuda").index_add_(0, key, x) * abs(scale)
           for x in (rows, rows.abs())]
    return out[0] * (1 if scale >= 0 else -1), out[1], torch.bincount(key, minlength=vocab)[:, None]


def grad_bound(want, total, count, dtype):
    return U[dtype] * want.abs() + (1 + U[dtype]) * (count + 3) * U32 * total + TINY[dtype]


SIZES = [(1, 1, 1, 8), (1, 24, 30522, 768), (3, 5, 7, 1), (5, 1, 50, 77), (2, 300, 11, 64), (67, 61, 28996, 1000),
         (64, 129, 300, 2056), (33, 40, 512, 256), (9, 17, 513, 255), (9, 17, 513, 770), (1, 4097, 40, 16), (3, 7001, 900, 18), (700, 13, 300000, 24)]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("n,length,vocab,dim", SIZES)
def test_embed_and_gradient(n, length, vocab, dim, dtype):
    tokens, lengths, table = embed_case(n, length, vocab, dim, dtype, seed=n + dim)
    scale = 1.7320507764816284  # a 32-bit value
    got = rd.embed_tokens(tokens, table, lengths, scale=scale)
    want = embed_ref(tokens, lengths, table, scale)
    assert got.dtype == dtype and got.shape == (n, length, dim)
    within(got, want, (U[dtype] + 2 * U32) * want.abs() + TINY[dtype])
    grad = torch.randn((n, length, dim), device="cuda", generator=gen(dim)).to(dtype)
    d = rd.embed_tokens_grad(grad, tokens, vocab, lengths, scale=scale)
    assert d.dtype == dtype
    ref = grad_ref(grad, tokens, lengths, vocab, scale)
    within(d, ref[0], grad_bound(*ref, dtype))
    assert torch.equal(d, rd.embed_tokens_grad(grad, tokens, vocab, lengths, scale=scale))


@pytest.mark.parametrize("token_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("out", [F16, BF16, F32])
def test_embed_types_from_a_32_bit_table(out, token_dtype):
    tokens, lengths, table = embed_case(9, 31, 257, 40, F32, 3, token_dtype)
    got = rd.embed_tokens(tokens, table, lengths, scale=0.5, out_dtype=out)
    within(got, embed_ref(tokens, lengths, table, 0.5), U[out] * embed_ref(tokens, lengths, table, 0.5).abs() + TINY[out])
    grad = torch.randn((9, 31, 40), device="cuda", generator=gen(4)).to(out)
    d = rd.embed_tokens_grad(grad, tokens, 257, lengths, scale=0.5, dtype=F32)
    assert d.dtype == F32
    ref = grad_ref(grad, tokens, lengths, 257, 0.5)
    within(d, ref[0], grad_bound(*ref, F32))
    table.requires_grad_()
    y = rd.embed_tokens(tokens, table, lengths, scale=0.5, out_dtype=out)
    assert torch.equal(y, got) and torch.equal(torch.autograd.grad(y, table, grad)[0], d)


def test_embed_shard_of_a_vocabulary_and_far_tokens():
    """Shards add up to the whole; tokens outside, the ends of int64 among them, give zeros and no gradient."""
    tokens, lengths, table = embed_case(20, 33, 100, 16, BF16, 5, torch.int64)
    tokens[0, :4] = torch.tensor([-1, 100, 2**63 - 1, -2**63], device="cuda")
    lengths[0] = 33
    whole = rd.embed_tokens(tokens, table, lengths)
    parts = [rd.embed_tokens(tokens, table[lo:hi], lengths, vocab_base=lo) for lo, hi in ((0, 37), (37, 100))]
    assert torch.equal(whole, parts[0] + parts[1]) and int(whole[0, :4].count_nonzero()) == 0
    assert torch.equal(whole, embed_ref(tokens, lengths, table, 1.0).to(BF16))
    grad = torch.randn((20, 33, 16), device="cuda", generator=gen(6)).to(BF16)
    d = rd.embed_tokens_grad(grad, tokens, 100, lengths)
    parts = [rd.embed_tokens_grad(grad, tokens, hi - lo, lengths, vocab_base=lo) for lo, hi in ((0, 37), (37, 100))]
    assert torch.equal(d, torch.cat(parts))
    ref = grad_ref(grad, tokens, lengths, 100, 1.0)
    within(d, ref[0], grad_bound(*ref, BF16))
    far = rd.embed_tokens(tokens, table, lengths, vocab_base=-2**63)
    assert int(far[0, 3].count_nonzero()) == 16 and int(far.count_nonzero()) == 16


def test_embed_layouts_and_empty_batches():
    tokens, lengths, table = embed_case(6, 10, 50, 64, F16, 7)
    want = embed_ref(tokens, lengths, table, 1.0).to(F16)
    padded = torch.full((50, 72), float("nan"), device="cuda", dtype=F16)
    padded[:, :64] = table
    assert torch.equal(rd.embed_tokens(tokens, padded[:, :64], lengths), want)
    shifted = torch.empty((50 * 64 + 1,), device="cuda", dtype=F16)[1:].view(50, 64).copy_(table)
    assert torch.equal(rd.embed_tokens(tokens, shifted, lengths), want)
    wide = torch.full((12, 20), 7, device="cuda", dtype=torch.int32)
    wide[::2, ::2] = tokens
    assert torch.equal(rd.embed_tokens(wide[::2, ::2], table, lengths), want)
    assert torch.equal(rd.embed_tokens(tokens.view(2, 3, 10), table, lengths.view(2, 3)), want.view(2, 3, 10, 64))
    assert torch.equal(rd.embed_tokens(tokens, table), embed_ref(tokens, torch.full_like(lengths, 10), table, 1.0).to(F16))
    assert rd.embed_tokens(tokens[:0], table, lengths[:0]).shape == (0, 10, 64)
    assert rd.embed_tokens(tokens[:, :0], table, lengths).shape == (6, 0, 64)
    empty = rd.embed_tokens_grad(torch.ones((6, 0, 64), device="cuda", dtype=F16), tokens[:, :0], 50, lengths)
    assert empty.shape == (50, 64) and int(empty.count_nonzero()) == 0
    none = rd.embed_tokens_grad(torch.ones((6, 10, 64), device="cuda", dtype=F16), tokens, 50, torch.zeros_like(lengths))
    assert int(none.count_nonzero()) == 0
    grad = torch.randn((6, 64, 10), device="cuda", generator=gen(8)).to(F16).transpose(1, 2)  # not contiguous
    assert torch.equal(rd.embed_tokens_grad(grad, tokens, 50, lengths),
                       rd.embed_tokens_grad(grad.contiguous(), tokens, 50, lengths))
    odd = torch.empty((6 * 10 * 64 + 1,), device="cuda", dtype=F16)[1:].view(6, 10, 64).copy_(grad)  # misaligned
    ref = grad_ref(grad, tokens, lengths, 50, 1.0)
    within(rd.embed_tokens_grad(odd, tokens, 50, lengths), ref[0], grad_bound(*ref, F16))


@pytest.mark.parametrize("n,length,vocab", [(40, 512, 30522), (40, 512, 1), (1, 65536, 3), (300, 256, 600000)])
def test_embed_gradient_runs_that_cross_workers(n, length, vocab):
    """Tokens repeated over many workers of the sum, and rows of NaN behind the lengths that must not count."""
    dim = 32
    tokens, lengths, _ = embed_case(n, length, vocab, 1, F32, 11)
    if n == 1:
        lengths[0] = length - 3
    grad = torch.randn((n, length, dim), device="cuda", generator=gen(12))
    grad[~valid_of(tokens, lengths, vocab)] = float("nan")
    d = rd.embed_tokens_grad(grad, tokens, vocab, lengths)
    ref = grad_ref(torch.nan_to_num(grad), tokens, lengths, vocab, 1.0)
    within(d, ref[0], grad_bound(*ref, F32))
    assert torch.equal(d, rd.embed_tokens_grad(grad, tokens, vocab, lengths))


def test_embed_gradient_against_differences():
    """The lookup is linear: its difference along a direction is the gradient's product with it."""
    tokens, lengths, table = embed_case(8, 20, 40, 24, F32, 13)
    grad = torch.randn((8, 20, 24), device="cuda", generator=gen(14))
    step = torch.randn((40, 24), device="cuda", generator=gen(15), dtype=torch.float64)
    d = rd.embed_tokens_grad(grad, tokens, 40, lengths, scale=3.0)
    ref = grad_ref(grad, tokens, lengths, 40, 3.0)
    h = 0.5
    plus, minus = (embed_ref(tokens, lengths, table.double() + x * step, 3.0) for x in (h, -h))
    diff = ((plus - minus) * grad.double()).sum() / (2 * h)
    assert abs(float((d.double() * step).sum() - diff)) <= float((grad_bound(*ref, F32) * step.abs()).sum()) + 1e-9


# ---- attention ------------------------------------------------------------------------------------
def attend_case(batch, rows, passages, length, heads, kv_heads, dim, dtype, seed, q_std=2.0):
    g = gen(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(shape, device="cuda", generator=g) * std).to(dtype)

    q = normal(batch, rows, heads, dim, std=q_std)
    k, v = normal(batch, passages, length, kv_heads, dim), normal(batch, passages, length, kv_heads, dim)
    lengths = torch.randint(-1, length + 2, (batch, passages), device="cuda", generator=g, dtype=torch.int32)
    return q, k, v, lengths, normal(batch, rows, heads, dim)


def attend_ref(q, k, v, lengths, grad=None, scale=None):
    """64-bit results and, beside each, the bound of what the kernels may be off by."""
    t = q.dtype
    u, tiny = U[t], TINY[t]
    batch, rows, heads, dim = q.shape
    if k.dim() == 4:
        k, v = k[:, None], v[:, None]
    _, passages, length, kv_heads, _ = k.shape
    share, keys = heads // kv_heads, passages * length
    scale = dim ** -0.5 if scale is None else scale
    if lengths is None:
        lengths = torch.full((batch, passages), length, device="cuda", dtype=torch.int32)
    inside = (torch.arange(length, device="cuda") < lengths.view(batch, passages)[..., None]).view(batch, 1, 1, keys)

    def rows_of(x):
        return x.double().view(batch, rows, kv_heads, share, dim).transpose(1, 2).reshape(batch, kv_heads, -1, dim)

    def states_of(x):
        x = torch.where(inside.view(batch, keys, 1, 1), x.reshape(batch, keys, kv_heads, dim).double(), 0.0)
        return x.transpose(1, 2).contiguous()

    def rows_back(x):
        return x.view(batch, kv_heads, rows, share, dim).transpose(1, 2).reshape(batch, rows, heads, dim)

    def states_back(x):
        return x.transpose(1, 2).reshape(batch, passages, length, kv_heads, dim)

    Q, K, V = rows_of(q), states_of(k), states_of(v)
    s = torch.matmul(Q, K.transpose(2, 3)) * scale
    s = s.masked_fill(~inside, -math.inf)
    top = s.amax(3, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(3, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    lse = (top + torch.log(total)).squeeze(3).view(batch, kv_heads, rows, share).transpose(2, 3).reshape(batch, heads, rows)
    out = torch.matmul(p, V)
    # a score is a 32-bit sum of dim products, scaled; exp2 and its argument, below 2^8, are off by 2^-14 * U32-ish
    # steps: 2^8 * 2 * U32 covers the argument's rounding, 4 * U32 the function's
    ds = (dim + 4) * U32 * abs(scale) * torch.matmul(Q.abs(), K.abs().transpose(2, 3)).amax(3, keepdim=True)
    ds = ds + 520 * U32
    n_keys = inside.sum(3, keepdim=True)
    # weights keep a power of two beside them: what a subnormal one loses; exp2 gives zero for what 32 bits hold as a
    # subnormal, below 2^-126, and a product takes subnormal operands as zero
    flush = 2.0 ** -126
    floor = max(TINY[t] * 2.0 ** -9, flush)
    pv = torch.matmul(p, V.abs())
    v_max = V.abs().amax((2, 3), keepdim=True)
    # weights: u, their scores' error in numerator and sum: 2 ds, the 32-bit sums of numerator and weights
    weight = u + 2 * ds + 2 * (n_keys + 8) * U32
    out_bound = weight * pv * (1 + u) + u * out.abs() + n_keys * floor * v_max + tiny
    res = {"out": (rows_back(out), rows_back(out_bound)),
           "lse": (lse, (ds + (n_keys + 8) * U32).squeeze(3).view(batch, kv_heads, rows, share).transpose(2, 3)
                   .reshape(batch, heads, rows) + 4 * U32 * torch.nan_to_num(lse, neginf=0.0).abs())}
    if grad is None:
        return res
    G = rows_of(grad)
    dv = torch.matmul(p.transpose(2, 3), G)
    dp = torch.matmul(G, V.transpose(2, 3))
    delta = (G * out).sum(3, keepdim=True)
    dS = p * (dp - delta)
    lse_off = ds + (n_keys + 8) * U32 + 6 * U32 * torch.nan_to_num(top, neginf=0.0).abs()
    p_off = 2 * ds + lse_off                                # relative, of a weight made from the stored lse
    # dp and delta: 32-bit sums of dim products; delta takes out as it is off before its rounding, the two roundings
    # of out and rest leave u * u
    gv = torch.matmul(G.abs(), V.abs().transpose(2, 3))
    delta_off = (G.abs() * (out_bound - u * out.abs() + (u * u + (dim + 1) * U32) * out.abs())).sum(3, keepdim=True)
    # a weight that was flushed is off by flush times its factor, a dS that was by flush
    dS_off = dS.abs() * (u + p_off) + p * (dim * U32 * gv + delta_off) * (1 + u + p_off) + flush * ((dp - delta).abs() + 1) * inside
    n_rows = rows * share
    small = TINY[t] * 2.0 ** -9 * dS.abs().amax((2, 3), keepdim=True) / max(torch.finfo(t).smallest_normal, 2.0 ** -14)
    a = abs(scale)
    dq = scale * torch.matmul(dS, K)
    dk = scale * torch.matmul(dS.transpose(2, 3), Q)
    dq_bound = a * torch.matmul(dS_off + (n_keys + 8) * U32 * dS.abs() + small * inside, K.abs()) + u * dq.abs() + tiny
    dk_bound = a * torch.matmul((dS_off + (n_rows + 8) * U32 * dS.abs() + small * inside).transpose(2, 3), Q.abs()) + u * dk.abs() + tiny
    dv_bound = torch.matmul((p * (u + p_off + (n_rows + 8) * U32) + floor * inside).transpose(2, 3), G.abs()) * (1 + u) + u * dv.abs() + tiny
    res.update(dq=(rows_back(dq), rows_back(dq_bound)), dk=(states_back(dk), states_back(dk_bound)),
               dv=(states_back(dv), states_back(dv_bound)))
    return res


def check_attend(q, k, v, lengths, grad=None, scale=None):
    ref = attend_ref(q, k, v, lengths, grad, scale)
    out, saved = rd.cross_attention(q, k, v, lengths, scale=scale, return_saved=True)
    lse = saved[0]
    assert out.dtype == q.dtype and out.shape == q.shape and out.is_contiguous()
    within(out, *ref["out"])
    within(lse, *ref["lse"])
    assert torch.equal(out, rd.cross_attention(q, k, v, lengths, scale=scale))
    assert torch.equal(lse, rd.cross_attention(q, k, v, lengths, scale=scale, return_lse=True)[1])
    if grad is None:
        return
    got = rd.cross_attention_grad(grad, q, k, v, out, saved, lengths, scale)
    for name, x, like in zip(("dq", "dk", "dv"), got, (q, k, v)):
        assert x.dtype == q.dtype and x.shape == like.shape and x.is_contiguous()
        within(x.view(ref[name][0].shape), *ref[name])
    again = rd.cross_attention_grad(grad, q, k, v, out, saved, lengths, scale)
    assert all(torch.equal(x, y) for x, y in zip(got, again))
    leaves = [x.detach().clone().requires_grad_() for x in (q, k, v)]
    y = rd.cross_attention(*leaves, lengths, scale=scale)
    assert torch.equal(y, out)
    assert all(torch.equal(x, y) for x, y in zip(got, torch.autograd.grad(y, leaves, grad)))


SHAPES = [
    (1, 1, 1, 1, 1, 1, 8), (1, 1, 1, 128, 12, 12, 64), (2, 1, 7, 65, 8, 2, 128), (3, 2, 3, 5, 4, 4, 32),
    (2, 31, 1, 64, 3, 3, 64), (2, 32, 4, 33, 4, 1, 128), (1, 33, 5, 63, 6, 2, 80), (2, 64, 2, 129, 2, 2, 40),
    (1, 65, 3, 100, 2, 1, 128), (1, 127, 1, 1, 3, 3, 64), (1, 130, 2, 300, 2, 2, 96), (1, 257, 3, 77, 4, 2, 128),
    (5, 16, 1, 16, 16, 2, 64), (2, 3, 40, 3, 5, 5, 72), (1, 17, 1, 700, 1, 1, 120), (4, 1, 32, 200, 4, 4, 64),
    (9, 4, 2, 20, 24, 3, 16), (1, 300, 1, 513, 2, 2, 64), (3, 40, 100, 7, 4, 2, 64), (2, 200, 70, 1, 3, 3, 128),
    (1, 70, 33, 32, 2, 1, 40), (2, 5, 300, 31, 2, 2, 128), (4, 100, 9, 13, 2, 2, 64),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attention_and_gradient(shape, dtype):
    q, k, v, lengths, grad = attend_case(*shape, dtype, seed=sum(shape))
    check_attend(q, k, v, lengths, grad)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_without_lengths_and_with_other_scales(dtype):
    q, k, v, _, grad = attend_case(2, 19, 3, 40, 4, 2, 64, dtype, 21)
    check_attend(q, k, v, None, grad)
    for scale in (0.0, -0.2, 1.0):
        check_attend(q, k, v, None, grad, scale)
    one = attend_case(3, 9, 1, 50, 2, 2, 32, dtype, 22)
    q, k, v, lengths, grad = one
    check_attend(q, k[:, 0], v[:, 0], lengths[:, 0], grad)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", [1, 40, 200])
def test_attention_what_lies_behind_the_lengths_is_never_used(rows, dtype):
    q, k, v, _, grad = attend_case(3, rows, 4, 70, 4, 2, 64, dtype, 23)
    lengths = torch.tensor([[0, 1, 64, 69], [-1, 0, 0, -5], [70, 33, 0, 1000]], device="cuda", dtype=torch.int32)
    want = attend_ref(q, k, v, lengths, grad)
    inside = torch.arange(70, device="cuda") < lengths[..., None]
    for junk in (float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).min):
        k[~inside], v[~inside] = junk, junk
        out, saved = rd.cross_attention(q, k, v, lengths, return_saved=True)
        lse = saved[0]
        within(out, *want["out"])
        within(lse, *want["lse"])
        assert int(out[1].count_nonzero()) == 0 and bool((lse[1] == -math.inf).all())
        got = rd.cross_attention_grad(grad, q, k, v, out, saved, lengths)
        for name, x in zip(("dq", "dk", "dv"), got):
            within(x, *want[name])
        assert int(got[0][1].count_nonzero()) == 0
        assert int(got[1][~inside].count_nonzero()) == 0 and int(got[2][~inside].count_nonzero()) == 0


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_layouts(dtype):
    """Any strides give the contiguous layout's bits."""
    q, k, v, lengths, grad = attend_case(2, 34, 3, 50, 4, 2, 64, dtype, 25)
    out, saved = rd.cross_attention(q, k, v, lengths, return_saved=True)
    want = rd.cross_attention_grad(grad, q, k, v, out, saved, lengths)

    def same(q, k, v, lengths, grad):
        o, l = rd.cross_attention(q, k, v, lengths, return_saved=True)
        assert torch.equal(o, out) and torch.equal(l[0], saved[0]) and torch.equal(l[1], saved[1])
        got = rd.cross_attention_grad(grad, q, k, v, o, l, lengths)
        assert all(torch.equal(x, y) for x, y in zip(got, want))

    heads_first = [x.transpose(-2, -3).contiguous().transpose(-2, -3) for x in (q, k, v, grad)]
    same(heads_first[0], heads_first[1], heads_first[2], lengths, heads_first[3])
    packed = torch.full((2, 3, 50, 2, 3, 64), float("nan"), device="cuda", dtype=dtype)
    packed[..., 0, :], packed[..., 2, :] = k, v
    same(q, packed[..., 0, :], packed[..., 2, :], lengths, grad)
    odd = [torch.empty((x.numel() + 1,), device="cuda", dtype=dtype)[1:].view(x.shape).copy_(x) for x in (q, k, v, grad)]
    same(odd[0], odd[1], odd[2], lengths, odd[3])
    inner = [x.transpose(-1, -2).contiguous().transpose(-1, -2) for x in (q, k, v, grad)]
    same(inner[0], inner[1], inner[2], lengths, inner[3])
    wide = torch.zeros((4, 6), device="cuda", dtype=torch.int32)
    wide[::2, ::2] = lengths
    same(q, k, v, wide[::2, ::2], grad)


# heads that share a key head in numbers that divide a tile's rows and in others; the last tile of rows is short
SHARED = [(2, 50, 3, 70, 6, 2, 128), (1, 40, 2, 130, 16, 1, 64), (1, 12, 2, 100, 32, 1, 128), (2, 30, 3, 70, 8, 1, 128),
          (1, 70, 2, 90, 10, 2, 64), (1, 192, 2, 64, 4, 4, 128)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("shape", SHARED, ids=str)
def test_attention_shared_heads_in_strided_rows(shape, dtype):
    """Many rows of shared heads, whose queries and gradients lie in wider tensors."""
    q, k, v, lengths, grad = attend_case(*shape, dtype, seed=37)
    check_attend(q, k, v, lengths, grad)
    out, saved = rd.cross_attention(q, k, v, lengths, return_saved=True)
    want = rd.cross_attention_grad(grad, q, k, v, out, saved, lengths)
    batch, rows, passages, length, heads, kv_heads, dim = shape

    def inside(x, pad):
        wide = torch.full((*x.shape[:-2], x.shape[-2] + pad, dim + 8 * pad), float("nan"), device="cuda", dtype=dtype)
        wide[..., 1:1 + x.shape[-2], 8:8 + dim] = x
        return wide[..., 1:1 + x.shape[-2], 8:8 + dim]

    qs, ks, vs, gs = inside(q, 2), inside(k, 3), inside(v, 4), inside(grad, 5)
    o, l = rd.cross_attention(qs, ks, vs, lengths, return_saved=True)
    assert torch.equal(o, out) and torch.equal(l[0], saved[0])
    got = rd.cross_attention_grad(gs, qs, ks, vs, o, l, lengths)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("rows,dim", [(1, 128), (20, 64), (70, 128), (130, 64), (40, 128)])
@pytest.mark.parametrize("passages,length", [(150, 40), (129, 63), (70, 70), (200, 33), (1100, 33)])
def test_attention_many_passages(passages, length, rows, dim):
    """More passages than are looked at together, most of them empty for one batch entry, one behind the other and with
    gaps between them."""
    q, k, v, lengths, grad = attend_case(3, rows, passages, length, 2, 1, dim, BF16, seed=passages + rows)
    lengths[0, 3:passages - 2] = 0
    lengths[1] = 0
    lengths[1, -1] = 1
    check_attend(q, k, v, lengths, grad)
    gaps = [torch.full((3, passages, length + 2, 1, dim), float("nan"), device="cuda", dtype=BF16) for _ in range(2)]
    for wide, x in zip(gaps, (k, v)):
        wide[:, :, 1:-1] = x
    check_attend(q, gaps[0][:, :, 1:-1], gaps[1][:, :, 1:-1], lengths, grad)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", [1, 40, 200])
@pytest.mark.parametrize("step", [0.002, 0.03, -0.03, 2.0])
def test_attention_scores_that_rise_along_the_keys(step, rows, dtype):
    """Maxima that creep up by less than a factor of two a tile, by some, by many, and that fall."""
    q, k, v, lengths, grad = attend_case(2, rows, 3, 230, 2, 1, 64, dtype, 39, q_std=0.5)
    q[..., 0] = 8.0
    k[..., 0] = (torch.arange(690, device="cuda").view(3, 230, 1) * step).to(dtype)
    check_attend(q, k, v, lengths, grad)
    alone = rd.cross_attention(q[:, :1], k, v, lengths)
    if rows == 1:
        assert torch.equal(alone, rd.cross_attention(q, k, v, lengths))


def test_attention_broadcast_states():
    """States shared by a batch through expand: the gradient adds up over it."""
    q, k, v, _, grad = attend_case(4, 20, 2, 30, 2, 2, 64, BF16, 27)
    lengths = torch.tensor([[30, 7]], device="cuda", dtype=torch.int32)
    leaves = [k[:1].clone().requires_grad_(), v[:1].clone().requires_grad_()]
    out_g = out = rd.cross_attention(q, leaves[0].expand(4, -1, -1, -1, -1), leaves[1].expand(4, -1, -1, -1, -1),
                             lengths.expand(4, 2))
    ref = attend_ref(q, k[:1].expand(4, -1, -1, -1, -1), v[:1].expand(4, -1, -1, -1, -1), lengths.expand(4, 2), grad)
    within(out.detach(), *ref["out"])
    for x, name in zip(torch.autograd.grad(out_g, leaves, grad), ("dk", "dv")):
        want, bound = (y.sum(0, keepdim=True) for y in ref[name])
        within(x, want, bound + 4 * U[BF16] * ref[name][0].abs().sum(0, keepdim=True))  # torch rounds while it adds four
    # the same answers read as further rows of one batch entry
    rows = rd.cross_attention(q.reshape(1, 80, 2, 64), k[:1], v[:1], lengths)
    within(rows.view(q.shape), *ref["out"])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("std", [1e-6, 3e3])
def test_attention_gradients_of_small_and_large_losses(std, dtype):
    """Gradients of a mean over many tokens, or of a scaled loss: the weights' gradients keep their precision."""
    q, k, v, lengths, grad = attend_case(2, 40, 8, 100, 2, 1, 64, dtype, 29, q_std=0.3)
    big = (grad.float() * (std if dtype == BF16 else max(std, 1e-4) if std < 1 else 100.0)).to(dtype)
    check_attend(q, k, v, lengths, big)
    # rows of very different size beside each other
    big[:, ::2] *= 2.0 ** -8
    check_attend(q, k, v, lengths, big)


def test_attention_large_scores():
    """One key far above the rest, and scores that would overflow an exponential."""
    q, k, v, lengths, grad = attend_case(2, 33, 2, 90, 2, 2, 64, BF16, 31, q_std=30.0)
    k[0, 0, 3] *= 20
    check_attend(q, k, v, None, None)
    out = rd.cross_attention(q, k, v, None)
    assert bool(torch.isfinite(out).all())


def test_attention_gradient_against_differences():
    """The kernels' gradients along a direction against central differences of the 64-bit formula."""
    q, k, v, lengths, grad = attend_case(2, 12, 3, 20, 4, 2, 32, F16, 33, q_std=1.0)
    ref = attend_ref(q, k, v, lengths, grad)
    out, saved = rd.cross_attention(q, k, v, lengths, return_saved=True)
    got = rd.cross_attention_grad(grad, q, k, v, out, saved, lengths)
    h = 1e-4
    for i, name in enumerate(("dq", "dk", "dv")):
        args = [x.double() for x in (q, k, v)]
        step = torch.randn(args[i].shape, device="cuda", generator=gen(34 + i), dtype=torch.float64)
        ends = []
        for sign in (h, -h):
            moved = list(args)
            moved[i] = args[i] + sign * step
            ends.append((plain_64(*moved, lengths) * grad.double()).sum())
        diff = float((ends[0] - ends[1]) / (2 * h))
        size = float((ref[name][0].abs() * step.abs()).sum())
        off = abs(float((got[i].double().view(step.shape) * step).sum()) - diff)
        assert off <= float((ref[name][1] * step.abs()).sum()) + 1e-6 * size, name  # h^2 of the differences themselves


def plain_64(q, k, v, lengths):
    batch, rows, heads, dim = q.shape
    share = heads // k.shape[3]
    out = torch.zeros_like(q)
    for b in range(batch):
        inside = torch.arange(k.shape[2], device="cuda") < lengths[b][:, None]
        if not bool(inside.any()):
            continue
        for h in range(heads):
            kk, vv = k[b, :, :, h // share][inside], v[b, :, :, h // share][inside]
            out[b, :, h] = torch.softmax(q[b, :, h] @ kk.T * dim ** -0.5, 1) @ vv
    return out


def test_attention_empty_shapes():
    q, k, v, lengths, grad = attend_case(2, 3, 2, 5, 2, 2, 16, F16, 37)
    assert rd.cross_attention(q[:0], k[:0], v[:0], lengths[:0]).shape == (0, 3, 2, 16)
    assert rd.cross_attention(q[:, :0], k, v, lengths).shape == (2, 0, 2, 16)
    for kk, ll in ((k[:, :0], lengths[:, :0]), (k[:, :, :0], lengths)):
        out, saved = rd.cross_attention(q, kk, kk, ll, return_saved=True)
        assert int(out.count_nonzero()) == 0 and bool((saved[0] == -math.inf).all())
        got = rd.cross_attention_grad(grad, q, kk, kk, out, saved, ll)
        assert got[0].shape == q.shape and got[1].shape == kk.shape and int(got[0].count_nonzero()) == 0
    out, saved = rd.cross_attention(q[:, :0], k, v, lengths, return_saved=True)
    got = rd.cross_attention_grad(grad[:, :0], q[:, :0], k, v, out, saved, lengths)
    assert all(int(x.count_nonzero()) == 0 for x in got) and got[1].shape == k.shape


@pytest.mark.parametrize("rows", [1, 70])
def test_attention_offsets_past_32_bits(rows):
    """Passages that start past 2^31 elements of the state tensors: all short but the last."""
    passages, length, heads, dim = 33, 1 << 16, 8, 128
    g = gen(39)
    states = torch.zeros((1, passages, length, heads, dim), device="cuda", dtype=BF16)
    assert states.numel() > 1 << 31
    q = torch.randn((1, rows, heads, dim), device="cuda", generator=g).to(BF16)
    lengths = torch.zeros((1, passages), device="cuda", dtype=torch.int32)
    lengths[0, -1], lengths[0, 0] = 100, 3
    for p, n in ((0, 3), (passages - 1, 100)):
        states[0, p, :n] = torch.randn((n, heads, dim), device="cuda", generator=g).to(BF16)
    small = torch.zeros((1, 2, 100, heads, dim), device="cuda", dtype=BF16)
    small[0, 0, :3], small[0, 1] = states[0, 0, :3], states[0, -1, :100]
    short = torch.tensor([[3, 100]], device="cuda", dtype=torch.int32)
    ref = attend_ref(q, small, small, short)
    within(rd.cross_attention(q, states, states, lengths), *ref["out"])
    # one long passage: rows of a cache far behind its start
    flat = states.view(1, 1, passages * length, heads, dim)
    kv = flat[:, :, -100:]
    within(rd.cross_attention(q, kv, kv), *attend_ref(q, kv, kv, None)["out"])
    full = torch.full((1, 1), passages * length, device="cuda", dtype=torch.int32)
    out, lse = rd.cross_attention(q, flat, flat, full, return_lse=True)  # zeros but for 103 rows
    s = torch.einsum("rhd,jhd->hrj", q[0].double(), torch.cat([small[0, 0, :3], small[0, 1]]).double()) * dim ** -0.5
    zeros = passages * length - 103
    want = torch.logsumexp(torch.cat([s, torch.full((heads, rows, 1), math.log(zeros), device="cuda", dtype=torch.float64)], 2), 2)
    # a sum of 2.2 million terms: the kernels add them in tiles, a few thousand 32-bit steps one after another
    within(lse[0], want, 1e-3 * torch.ones_like(want))


@pytest.mark.parametrize("rows", [1, 48])
def test_attention_streams_threads_and_graphs(rows):
    q, k, v, lengths, grad = attend_case(8, rows, 16, 90, 4, 2, 64, BF16, 41)
    out, saved = rd.cross_attention(q, k, v, lengths, return_saved=True)
    want = (out,) + rd.cross_attention_grad(grad, q, k, v, out, saved, lengths)
    torch.cuda.synchronize()

    def both():
        o, l = rd.cross_attention(q, k, v, lengths, return_saved=True)
        return (o,) + rd.cross_attention_grad(grad, q, k, v, o, l, lengths)

    # two threads, a stream each, at once
    results, failed = {}, []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                results[i] = [both() for _ in range(5)]
            stream.synchronize()
        except Exception as e:  # pragma: no cover
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for got in results.values():
        for one in got:
            assert all(torch.equal(x, y) for x, y in zip(one, want))
    # two graphs, captured one after the other and replayed with the eager call between
    graphs = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = both()
        graphs.append((graph, held))
    for seed in (1, 2, 3):
        q.copy_(torch.randn(q.shape, device="cuda", generator=gen(seed)).to(BF16))
        lengths.copy_(torch.randint(0, 91, lengths.shape, device="cuda", generator=gen(seed), dtype=torch.int32))
        now = both()
        torch.cuda.synchronize()
        for graph, held in graphs:
            for x in held:
                x.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(held, now))


def test_embed_streams_and_graphs():
    tokens, lengths, table = embed_case(64, 100, 5000, 64, F16, 43)
    grad = torch.randn((64, 100, 64), device="cuda", generator=gen(44)).to(F16)

    def both():
        return rd.embed_tokens(tokens, table, lengths), rd.embed_tokens_grad(grad, tokens, 5000, lengths)

    want = both()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append([both() for _ in range(3)])
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for per in got for one in per for x, y in zip(one, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for seed in (5, 6, 7):
        tokens.copy_(torch.randint(-2, 5100, tokens.shape, device="cuda", generator=gen(seed), dtype=torch.int32))
        now = both()
        torch.cuda.synchronize()
        for x in held:
            x.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(held, now))


# ---- together -------------------------------------------------------------------------------------
def test_reading_what_a_search_found(tmp_path):
    """ids -> tokens -> embeddings -> states of the passages -> the question's attention -> gradients of the table,
    on the store's own path, against the same chain in 64 bits."""
    rng = np.random.Generator(np.random.PCG64(51))
    vocab, heads, dim, top = 300, 4, 32, 6
    items = [rng.integers(0, vocab, size=int(n)) for n in rng.integers(0, 40, size=50)]
    ts.write_mmap_dataset(str(tmp_path / "docs"), items, dtype=np.uint16)
    store = ts.DeviceTokenStore(ts.MMapTokenDataset(str(tmp_path / "docs")), device=0)
    ids = torch.from_numpy(rng.integers(1, 51, size=(3, top)).astype(np.int32)).cuda()
    ids[0, 2] = 99  # not in the store
    g = gen(52)
    table = (torch.randn((vocab, heads * dim), device="cuda", generator=g)).to(BF16).requires_grad_()
    q = torch.randn((3, 10, heads, dim), device="cuda", generator=g).to(BF16).requires_grad_()
    grad = torch.randn(q.shape, device="cuda", generator=g).to(BF16)
    states, lens = store.embed(ids, table, scale=0.5)
    tokens, lens2 = store.gather(ids)
    assert torch.equal(lens, lens2) and int(lens[0, 2]) == -1
    assert torch.equal(states, rd.embed_tokens(tokens, table, lens, scale=0.5))
    assert int(states[0, 2].count_nonzero()) == 0
    kv = states.view(3, top, -1, heads, dim)
    out = rd.cross_attention(q, kv, kv, lens)
    d_table, d_q = torch.autograd.grad(out, (table, q), grad)
    ref = attend_ref(q.detach(), kv.detach(), kv.detach(), lens, grad)
    within(out, *ref["out"])
    within(d_q, *ref["dq"])
    d_states = ref["dk"][0] + ref["dv"][0]
    off = ref["dk"][1] + ref["dv"][1]
    off = off + U[BF16] * (d_states.abs() + off)  # autograd adds the two in their type
    flat = d_states.reshape(3, top, -1, heads * dim), off.reshape(3, top, -1, heads * dim)
    want, total, count = grad_ref(flat[0], tokens, lens, vocab, 0.5)
    more = grad_ref(flat[1], tokens, lens, vocab, 0.5)[1]
    within(d_table, want, more * (1 + U[BF16]) + grad_bound(want, total, count, BF16))
    with pytest.raises(ValueError):
        store.embed(ids, table.detach().cpu())
    store.close()


def test_gpu_refusals():
    q, k, v, lengths, grad = attend_case(2, 3, 2, 5, 2, 2, 16, F16, 53)
    for change in (dict(key=k.cpu()), dict(lengths=lengths.cpu()), dict(value=v.cpu()), dict(query=q.cpu())):
        args = dict(query=q, key=k, value=v, lengths=lengths)
        args.update(change)
        with pytest.raises(ValueError):
            rd.cross_attention(**args)
    tokens, lens, table = embed_case(2, 3, 5, 8, F16, 54)
    with pytest.raises(ValueError):
        rd.embed_tokens(tokens.cpu(), table, lens)
    with pytest.raises(ValueError):
        rd.embed_tokens(tokens, table, lens.cpu())
    with pytest.raises(ValueError):
        rd.embed_tokens_grad(torch.zeros((2, 3, 8), device="cuda", dtype=F16), tokens.cpu(), 5)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", [2, 25, 60])
@pytest.mark.parametrize("dim", range(8, 129, 8))
def test_attention_gradient_of_few_rows_at_every_head_size(dim, rows, dtype):
    """Columns behind the head size are cleared in LDS before the first tile comes to it, which is whole for one batch
    entry, part of a tile for another and empty for a third."""
    q, k, v, lengths, grad = attend_case(3, rows, 6, 70, 2, 2, dim, dtype, seed=dim + rows)
    lengths[0], lengths[1, ::2], lengths[2, 0] = 70, 5, 0
    check_attend(q, k, v, lengths, grad)
    check_attend(q, k, v, None, grad)


def test_forward_mode_is_refused_in_the_backward_pass_too():
    """Forward over reverse: the tangent of the result's gradient."""
    q, k, v, lengths, grad = attend_case(2, 3, 2, 5, 2, 2, 16, F16, 55)
    tokens, lens, table = embed_case(3, 5, 11, 8, F32, 56)
    forward_ad = torch.autograd.forward_ad
    calls = [(lambda x: rd.cross_attention(x, k, v, lengths), q, grad),
             (lambda x: rd.embed_tokens(tokens, x, lens), table, torch.ones((3, 5, 8), device="cuda"))]
    for call, leaf, weight in calls:
        leaf.requires_grad_()
        y = call(leaf)
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(weight, torch.ones_like(weight))
            with pytest.raises(NotImplementedError):
                torch.autograd.grad(y, leaf, dual)
            with pytest.raises(NotImplementedError):
                call(forward_ad.make_dual(leaf, torch.ones_like(leaf)))
        assert torch.autograd.grad(call(leaf), leaf, weight)[0].shape == leaf.shape


# ---- rows, layouts, values and sizes that stand alone ---------------------------------------------------
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", [2, 40, 200])
def test_attention_a_row_depends_on_itself_alone(rows, dtype):
    """One row kept while its neighbours, their maxima and their gradients change: its bits stay."""
    q, k, v, lengths, grad = attend_case(2, rows, 3, 90, 2, 1, 64, dtype, 57)
    k[..., 0] = (torch.arange(270, device="cuda").view(3, 90, 1) * 0.03).to(dtype)   # maxima that rise along the keys
    keep = rows // 2
    results = []
    for seed, std in ((1, 0.1), (2, 4.0)):
        other = (torch.randn(q.shape, device="cuda", generator=gen(seed)) * std).to(dtype)
        other[:, keep] = q[:, keep]
        g = (torch.randn(q.shape, device="cuda", generator=gen(seed + 10)) * std).to(dtype)
        g[:, keep] = grad[:, keep]
        out, saved = rd.cross_attention(other, k, v, lengths, return_saved=True)
        results.append((out[:, keep], saved[0][:, :, keep], saved[1][:, keep],
                        rd.cross_attention_grad(g, other, k, v, out, saved, lengths)[0][:, keep]))
    assert all(torch.equal(x, y) for x, y in zip(*results))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,dim", [(1, 64), (40, 64), (200, 64), (20, 128), (50, 128), (200, 128), (70, 40)])
@pytest.mark.parametrize("length,with_lengths", [(1, True), (7, True), (31, True), (32, True), (7, False), (50, False)])
def test_attention_short_passages_one_behind_the_other_and_with_gaps(length, with_lengths, rows, dim, dtype):
    """Passages that lie one behind the other may share tiles, those with gaps between them cannot: the same results
    within the same bounds, though not the same bits."""
    q, k, v, lengths, grad = attend_case(2, rows, 20, length, 2, 1, dim, dtype, seed=58 + length)
    lengths = lengths if with_lengths else None
    check_attend(q, k, v, lengths, grad)
    gaps = [torch.full((2, 20, length + 3, 1, dim), float("nan"), device="cuda", dtype=dtype) for _ in range(2)]
    for wide, x in zip(gaps, (k, v)):
        wide[:, :, 1:1 + length] = x
    k, v = gaps[0][:, :, 1:1 + length], gaps[1][:, :, 1:1 + length]
    ref = attend_ref(q, k, v, lengths, grad)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]   # no copies: those would close the gaps
    out = rd.cross_attention(*leaves, lengths)
    within(out, *ref["out"])
    within(rd.cross_attention(q, k, v, lengths, return_lse=True)[1], *ref["lse"])
    got = torch.autograd.grad(out, leaves, grad)
    for name, x in zip(("dq", "dk", "dv"), got):
        within(x, *ref[name])
    held, saved = rd.cross_attention(q, k, v, lengths, return_saved=True)
    assert torch.equal(held, out)
    again = rd.cross_attention_grad(grad, q, k, v, held, saved, lengths)
    assert all(torch.equal(x, y) for x, y in zip(got, again))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("std", [30.0, 120.0])
@pytest.mark.parametrize("rows", [1, 40, 200])
def test_attention_gradients_of_large_scores(rows, std, dtype):
    """Weights made anew from a log-sum of hundreds: its 32 bits are what their precision hangs on."""
    q, k, v, lengths, grad = attend_case(2, rows, 2, 90, 2, 2, 64, dtype, 59, q_std=std)
    check_attend(q, k, v, lengths, grad)
    check_attend(q, k, v, None, grad)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", [1, 40, 200])
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_attention_infinities_and_nan_among_valid_values(value, rows, dtype):
    """One element of one valid state's value: its column of its key head's rows has it, nothing else changes, and the
    gradients that need it have none for that head."""
    q, k, v, _, grad = attend_case(3, rows, 4, 70, 4, 2, 64, dtype, 60, q_std=0.3)
    lengths = torch.tensor([[70, 9, 0, 33], [70, 9, 0, 33], [1, 2, 3, 64]], device="cuda", dtype=torch.int32)
    clean, saved = rd.cross_attention(q, k, v, lengths, return_saved=True)
    grads = rd.cross_attention_grad(grad, q, k, v, clean, saved, lengths)
    v[1, 3, 20, 1, 5] = value   # read by heads 2 and 3
    out, saved2 = rd.cross_attention(q, k, v, lengths, return_saved=True)
    got = rd.cross_attention_grad(grad, q, k, v, out, saved2, lengths)
    hit = torch.zeros(q.shape, dtype=torch.bool, device="cuda")
    hit[1, :, 2:, 5] = True
    same = torch.isnan(out[hit]) if math.isnan(value) else out[hit] == value
    assert bool(same.all()) and torch.equal(out[~hit], clean[~hit]) and torch.equal(saved2[0], saved[0])
    rows_hit = torch.zeros(q.shape, dtype=torch.bool, device="cuda")
    rows_hit[1, :, 2:] = True
    inside = (torch.arange(70, device="cuda") < lengths[..., None])[..., None, None].expand(k.shape)
    states_hit = torch.zeros(k.shape, dtype=torch.bool, device="cuda")
    states_hit[1, :, :, 1] = True
    states_hit &= inside
    assert bool(torch.isnan(got[0][rows_hit]).all()) and torch.equal(got[0][~rows_hit], grads[0][~rows_hit])
    assert bool(torch.isnan(got[1][states_hit]).all()) and torch.equal(got[1][~states_hit], grads[1][~states_hit])
    assert torch.equal(got[2], grads[2])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", [1, 40, 200])
def test_attention_infinities_among_valid_keys(rows, dtype):
    """An infinite element of a key: rows whose score it makes -inf do without that key, those it makes inf have NaN."""
    q, k, v, _, grad = attend_case(3, rows, 2, 70, 2, 1, 64, dtype, 61, q_std=0.5)
    lengths = torch.tensor([[70, 34], [70, 34], [70, 34]], device="cuda", dtype=torch.int32)
    q[0, ..., 3], q[1, ..., 3], q[2, ..., 3] = -1.0, 1.0, 0.5
    k[:2, 1, 33, 0, 3] = float("inf")
    shorter = torch.tensor([[70, 33], [70, 33], [70, 34]], device="cuda", dtype=torch.int32)
    want = attend_ref(q, torch.where(torch.isinf(k), 0.0, k), v, shorter, grad)   # that key is behind the length there
    out, saved = rd.cross_attention(q, k, v, lengths, return_saved=True)
    got = rd.cross_attention_grad(grad, q, k, v, out, saved, lengths)
    fine = [0, 2]
    within(out[fine], *(x[fine] for x in want["out"]))
    within(saved[0][fine], *(x[fine] for x in want["lse"]))
    assert bool(torch.isnan(out[1]).all()) and bool(torch.isnan(saved[0][1]).all())
    assert all(bool(torch.isnan(x[1]).all()) for x in (got[0], got[1][:, :1, :34], got[2][:, :1, :34]))
    within(got[1][fine], *(x[fine] for x in want["dk"]))
    within(got[2][fine], *(x[fine] for x in want["dv"]))
    others = [d for d in range(64) if d != 3]   # 0 * inf in that column of the rows' gradients
    assert bool(torch.isnan(got[0][0, ..., 3]).all())
    within(got[0][fine][..., others], *(x[fine][..., others] for x in want["dq"]))
    within(got[0][2], *(x[2] for x in want["dq"]))


@pytest.mark.parametrize("rows", [1, 70])
def test_attention_gradient_offsets_past_32_bits(rows):
    """States and gradients of more than 2^31 elements, a few of them valid at both ends."""
    passages, length, heads, dim = 33, 1 << 16, 8, 128
    g = gen(62)
    states = torch.zeros((1, passages, length, heads, dim), device="cuda", dtype=BF16)
    assert states.numel() > 1 << 31
    q, grad = (torch.randn((1, rows, heads, dim), device="cuda", generator=g).to(BF16) for _ in range(2))
    lengths = torch.zeros((1, passages), device="cuda", dtype=torch.int32)
    ends = ((0, 3), (passages - 1, 100))
    small = torch.zeros((1, 2, 100, heads, dim), device="cuda", dtype=BF16)
    for i, (p, n) in enumerate(ends):
        lengths[0, p] = n
        states[0, p, :n] = small[0, i, :n] = torch.randn((n, heads, dim), device="cuda", generator=g).to(BF16)
    ref = attend_ref(q, small, small, torch.tensor([[3, 100]], device="cuda", dtype=torch.int32), grad)
    out, saved = rd.cross_attention(q, states, states, lengths, return_saved=True)
    got = rd.cross_attention_grad(grad, q, states, states, out, saved, lengths)
    within(out, *ref["out"])
    within(got[0], *ref["dq"])
    for x, name in zip(got[1:], ("dk", "dv")):
        for i, (p, n) in enumerate(ends):
            within(x[0, p, :n], *(y[0, i, :n] for y in ref[name]))
            x[0, p, :n] = 0
        assert int(x.count_nonzero()) == 0


def test_embed_and_gradient_past_32_bits():
    """Results and gradients of more than 2^31 elements, and a table of as many."""
    n, length, dim, vocab = 2100, 1000, 1024, 50
    tokens, lengths, table = embed_case(n, length, vocab, dim, BF16, 63)
    lengths[-1] = length
    out = rd.embed_tokens(tokens, table, lengths)
    assert out.numel() > 1 << 31
    for i in (0, n // 2, n - 1):
        assert torch.equal(out[i], embed_ref(tokens[i:i + 1], lengths[i:i + 1], table, 1.0)[0].to(BF16))
    few = torch.where(torch.arange(n, device="cuda") % 300 == 299, lengths, 0).int()   # the last row is one of them
    assert int(few[-1]) == length
    d = rd.embed_tokens_grad(out, tokens, vocab, few)
    some = torch.arange(299, n, 300, device="cuda")
    ref = grad_ref(out[some], tokens[some], few[some], vocab, 1.0)
    within(d, ref[0], grad_bound(*ref, BF16))
    del out
    vocab = 2_200_000
    big = torch.zeros((vocab, dim), device="cuda", dtype=BF16)
    big[-1], big[7] = 3.0, 2.0
    ids = torch.tensor([[vocab - 1, 7, 0, vocab - 2]], device="cuda", dtype=torch.int64)
    assert rd.embed_tokens(ids, big)[0, :, -1].tolist() == [3.0, 2.0, 0.0, 0.0]
    d = rd.embed_tokens_grad(torch.ones((1, 4, dim), device="cuda", dtype=BF16), ids, vocab)
    assert int(d.count_nonzero()) == 4 * dim and bool((d[ids[0]] == 1.0).all())


@pytest.mark.parametrize("out", [F32, BF16])
def test_embed_large_batches_of_a_32_bit_table(out):
    tokens, lengths, table = embed_case(1200, 256, 30522, 768, F32, 64)
    got = rd.embed_tokens(tokens, table, lengths, out_dtype=out)
    step = 200
    for i in range(0, 1200, step):
        want = embed_ref(tokens[i:i + step], lengths[i:i + step], table, 1.0).to(out)
        assert torch.equal(got[i:i + step], want)
    d = rd.embed_tokens_grad(got, tokens, 30522, lengths, dtype=F32)
    ref = grad_ref(got, tokens, lengths, 30522, 1.0)
    within(d, ref[0], grad_bound(*ref, F32))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", [1, 40, 200])
@pytest.mark.parametrize("dim", [40, 64, 80, 128])
def test_attention_a_row_whose_scores_are_all_minus_infinity(dim, rows, dtype):
    """An infinite element of one query that meets negative elements alone: its row has no weight, and the others'
    gradients stay what they are (but for dK's column of that element, 0 * inf)."""
    q, k, v, lengths, grad = attend_case(2, rows, 3, 70, 2, 2, dim, dtype, 65)
    k[..., 3] = -k[..., 3].abs() - 0.5
    lengths[0] = torch.tensor([70, 33, 0], device="cuda", dtype=torch.int32)
    row = rows - 1
    alone = q.clone()
    alone[0, row, 1] = 0
    weight = grad.clone()
    weight[0, row, 1] = 0
    ref = attend_ref(alone, k, v, lengths, weight)   # a row of zeros with no gradient adds nothing to dK and dV
    q[0, row, 1, 3] = float("inf")
    out, saved = rd.cross_attention(q, k, v, lengths, return_saved=True)
    got = rd.cross_attention_grad(grad, q, k, v, out, saved, lengths)
    assert int(out[0, row, 1].count_nonzero()) == 0 and float(saved[0][0, 1, row]) == -math.inf
    assert int(got[0][0, row, 1].count_nonzero()) == 0
    others = torch.ones((2, rows, 2), dtype=torch.bool, device="cuda")
    others[0, row, 1] = False
    within(out[others], *(x[others] for x in ref["out"]))
    within(got[0][others], *(x[others] for x in ref["dq"]))
    within(got[2], *ref["dv"])
    columns = torch.ones(k.shape, dtype=torch.bool, device="cuda")
    columns[0, :, :, 1, 3] = False
    within(got[1][columns], *(x[columns] for x in ref["dk"]))
    inside = torch.arange(70, device="cuda") < lengths[0][:, None]
    assert bool(torch.isnan(got[1][0, :, :, 1, 3][inside]).all()) and int(got[1][0, :, :, 1, 3][~inside].count_nonzero()) == 0


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", [1, 20, 40, 64, 200])
@pytest.mark.parametrize("dim", [64, 80, 128])
def test_attention_an_infinite_gradient_of_the_last_row(dim, rows, dtype):
    """dV takes the infinity in its column, with its sign, and keeps the others; rows that are not there add nothing."""
    q, k, v, lengths, grad = attend_case(2, rows, 3, 70, 4, 2, dim, dtype, 66, q_std=0.3)
    lengths[0] = torch.tensor([70, 33, 0], device="cuda", dtype=torch.int32)
    ref = attend_ref(q, k, v, lengths, grad)
    out, saved = rd.cross_attention(q, k, v, lengths, return_saved=True)
    clean = rd.cross_attention_grad(grad, q, k, v, out, saved, lengths)
    inside = torch.arange(70, device="cuda") < lengths[0][:, None]
    for value in (math.inf, -math.inf):
        grad[0, -1, 3, 9] = value
        got = rd.cross_attention_grad(grad, q, k, v, out, saved, lengths)
        assert bool((got[2][0, :, :, 1, 9][inside] == value).all())
        others = torch.ones(k.shape, dtype=torch.bool, device="cuda")
        others[0, :, :, 1, 9] = False
        assert torch.equal(got[2][others], clean[2][others])
        within(got[2][others], *(x[others] for x in ref["dv"]))
        rows_left = torch.ones(q.shape, dtype=torch.bool, device="cuda")
        rows_left[0, -1, 3] = False
        assert torch.equal(got[0][rows_left], clean[0][rows_left]) and not bool(torch.isfinite(got[0][~rows_left]).any())
        assert torch.equal(got[1][:, :, :, 0], clean[1][:, :, :, 0]) and torch.equal(got[1][1], clean[1][1])
