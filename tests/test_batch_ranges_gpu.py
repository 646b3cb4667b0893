"""The batch entries at the ends of their types' ranges, against the 64-bit statements of batch_ref:
logits masked by large negative numbers, cached rows of any finite size, rows of zeros."""
from __future__ import annotations

import pytest
import torch

import batch_ref as R
from test_batch_gpu import attention_case, attention_want, check_rows, gen, lens_tensor, logprob_want, near

pytestmark = pytest.mark.gpu


# ----------------------------------------------------------------------------- log probabilities

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R_,V", [(300, 4097), (4, 65537), (40, 50021), (3, 700)])  # one CTA a row, and up to eight
@pytest.mark.parametrize("mask", ["lowest", -1e38, -1e37, -1e30])
def test_rows_masked_by_a_large_negative_number(dc, cuda, dtype, R_, V, mask):
    """All but a few logits masked: threads, warps and whole CTAs see nothing but the mask, and their sums
    then join an ordinary maximum."""
    low = torch.finfo(dtype).min if mask == "lowest" else mask
    x = torch.full((R_, V), low, device=cuda, dtype=dtype)
    g = gen(101, cuda)
    few = torch.randint(0, V, (R_, 9), generator=g, device=cuda)
    few[0] = torch.arange(9, device=cuda)          # a run at the row's front, and one at its end
    few[1] = torch.arange(V - 9, V, device=cuda)
    x.scatter_(1, few, (3 * torch.randn(R_, 9, generator=g, device=cuda)).to(dtype))
    tokens = torch.stack([few[:, 3], torch.full((R_,), V // 2, device=cuda)], 1).to(torch.int32)
    got = dc.logprobs(x, tokens, top=5)
    torch.cuda.synchronize()
    given, ent, ids, best, _, lp = logprob_want(x, tokens, 5)
    assert torch.equal(got["top_ids"].long(), ids)
    assert near(got["logprobs"], given) and near(got["top_logprobs"], best)
    assert near(got["entropy"], ent, 2.0 ** -16 * (lp.exp() * lp).abs().sum(-1))


# ----------------------------------------------------------------------------- quantisation

@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("kind", ["normal", "signs", "constant", "wide", "one"])
def test_groups_of_the_largest_numbers(dc, cuda, bits, kind):
    """Finite groups whose edge times 2^bits - 1, or whose range, passes fp32's."""
    x = torch.rand(1, 2, 6, 128, generator=gen(105, cuda), device=cuda)
    x = {"normal": 1e37 * torch.randn(x.shape, generator=gen(106, cuda), device=cuda), "signs": torch.sign(x - 0.5) * 2e38,
         "constant": 0 * x - 3e38, "wide": x * 3.3e38 - (x > 0.5) * 3.3e38, "one": x}[kind]
    if kind == "one":  # one group of a row, beside ordinary ones
        x[0, 0, :, 64:] *= 2e37
    x = x.to(torch.bfloat16)
    assert x.isfinite().all()
    cache = dc.KVCache(1, 2, 8, 128, bits, 32, cuda)
    dc.stack_kv_write(cache, x, x, starts=lens_tensor([1], cuda))
    k, v = dc.stack_kv_read(cache, 6, starts=lens_tensor([1], cuda))
    torch.cuda.synchronize()
    assert dc.device_error() == 0 and torch.equal(k, v)
    want = R.values(R.quantise(x.double(), bits, 32), bits, 32)
    assert torch.equal(k.double(), want.to(torch.bfloat16).double())


# ----------------------------------------------------------------------------- attention

def stored(size, shape, bits, group, seed, dev):
    """Cache rows whose values are about `size` (a number, or one per row): random codes, scales and
    biases, not held to the smallest step that the write rule keeps."""
    g = gen(seed, dev)
    *lead, d = shape
    size = torch.as_tensor(size, dtype=torch.float64, device=dev)
    words = torch.randint(-2 ** 31, 2 ** 31, (*lead, d * bits // 32), generator=g, device=dev).to(torch.int32)
    r = lambda: torch.rand(*lead, d // group, generator=g, device=dev).double()  # noqa: E731
    scale = (0.5 + r()) * size / (2 ** bits - 1)
    return words, scale.to(torch.bfloat16), (-(0.25 + 0.5 * r()) * size).to(torch.bfloat16)


def put(part, new):
    for t, n in zip(part, new):
        if t is not None:
            t.copy_(n)


QUANT = [(8, 64, 128), (4, 32, 128), (8, 128, 256), (4, 64, 64)]


@pytest.mark.parametrize("bits,group,d", QUANT)
@pytest.mark.parametrize("size", [1e29, 1e32, 1e35, 1e37])
@pytest.mark.parametrize("tree", [False, True])
def test_finite_rows_of_any_size_that_a_token_does_not_see(dc, cuda, bits, group, d, size, tree):
    """The last block rows' k and v, finite but large, reach the tokens that see them alone."""
    case = (2, 6, 8, 2, d, bits, group, [125, 30], 20)
    S, T = case[:2]
    q, gate, cache, prefix, _ = attention_case(dc, cuda, case, seed=111)
    parents = torch.tensor([[-1, 0, 0, 1, 2, 2]] * 2, dtype=torch.int32) if tree else None
    want, tol = attention_want(q, gate, cache, prefix, parents, case, d ** -0.5)
    for b, n in enumerate(case[7]):
        for part, s in ((cache.k, 1), (cache.v, 2)):
            big = stored(size, (2, 1, d), bits, group, 113 + s, cuda)
            for t, x in zip(part, big):
                t[b, :, n + T - 1:n + T] = x
    out = dc.stack_attn_decode_batch(q, cache, lens_tensor(case[7], cuda), d ** -0.5, gate=gate, prefix=prefix,
                                     prefix_len=20, parents=None if parents is None else parents.to(cuda))
    torch.cuda.synchronize()
    assert dc.device_error() == 0
    good = torch.ones(S * T, dtype=torch.bool, device=cuda)
    good[[T - 1, 2 * T - 1]] = False
    check_rows(out[good], want[good], tol[good])


@pytest.mark.parametrize("bits,group,d", QUANT)
@pytest.mark.parametrize("size", [1e-25, 1e-15, 1e15, 1e29, 1e32, 1e35, 1e37])
def test_values_of_any_finite_size(dc, cuda, bits, group, d, size):
    case = (2, 3, 4, 2, d, bits, group, [40, 300], 130)
    q, gate, cache, prefix, _ = attention_case(dc, cuda, case, seed=121)
    for c, s in ((cache, 5), (prefix, 6)):
        put(c.v, stored(size, (c.sequences, 2, c.max_len, d), bits, group, s, cuda))
    out = dc.stack_attn_decode_batch(q, cache, lens_tensor(case[7], cuda), d ** -0.5, prefix=prefix, prefix_len=130)
    want, tol = attention_want(q, None, cache, prefix, None, case, d ** -0.5)
    check_rows(out, want, tol)


@pytest.mark.parametrize("bits,group,d", QUANT)
@pytest.mark.parametrize("size,q_size", [(1e32, 1e-31), (1e36, 3e-35), (1e-25, 1e25), (1e-30, 1e33)])
def test_keys_and_queries_of_any_finite_size(dc, cuda, bits, group, d, size, q_size):
    case = (2, 3, 4, 2, d, bits, group, [40, 300], 130)
    q, gate, cache, prefix, _ = attention_case(dc, cuda, case, seed=131, q_std=q_size)
    for c, s in ((cache, 7), (prefix, 8)):
        put(c.k, stored(size, (c.sequences, 2, c.max_len, d), bits, group, s, cuda))
    scale = d ** -0.5 / (size * q_size)
    out = dc.stack_attn_decode_batch(q, cache, lens_tensor(case[7], cuda), scale, prefix=prefix, prefix_len=130)
    want, tol = attention_want(q, None, cache, prefix, None, case, scale)
    check_rows(out, want, tol)


@pytest.mark.parametrize("bits,group,d", QUANT)
@pytest.mark.parametrize("size", [1e-20, 1e-12, 1e-10, 1e-8, 1.0, 1e15])
def test_values_beside_rows_of_zeros(dc, cuda, bits, group, d, size):
    """Rows whose codes, scales and biases are all zero take their share of the weight, and the others keep their bits."""
    case = (2, 3, 4, 2, d, bits, group, [40, 300], 130)
    q, gate, cache, prefix, _ = attention_case(dc, cuda, case, seed=141)
    for c, s in ((cache, 9), (prefix, 10)):
        put(c.v, stored(size, (c.sequences, 2, c.max_len, d), bits, group, s, cuda))
        for t in c.v:
            t[:, :, ::3] = 0
    out = dc.stack_attn_decode_batch(q, cache, lens_tensor(case[7], cuda), d ** -0.5, prefix=prefix, prefix_len=130)
    want, tol = attention_want(q, None, cache, prefix, None, case, d ** -0.5)
    check_rows(out, want, tol)


@pytest.mark.parametrize("bits,group,d", QUANT)
@pytest.mark.parametrize("small,large", [(1e-10, 1e10), (1e-20, 1e12), (1.0, 1e30)])
def test_values_of_very_different_sizes(dc, cuda, bits, group, d, small, large):
    """Every other row is large: the small ones count in the denominator alone, in full."""
    case = (2, 3, 4, 2, d, bits, group, [40, 300], 130)
    q, gate, cache, prefix, _ = attention_case(dc, cuda, case, seed=151)
    for c, s in ((cache, 11), (prefix, 12)):
        size = torch.tensor([small, large], dtype=torch.float64).repeat((c.max_len + 1) // 2)[:c.max_len, None]
        put(c.v, stored(size, (c.sequences, 2, c.max_len, d), bits, group, s, cuda))
    out = dc.stack_attn_decode_batch(q, cache, lens_tensor(case[7], cuda), d ** -0.5, prefix=prefix, prefix_len=130)
    want, tol = attention_want(q, None, cache, prefix, None, case, d ** -0.5)
    check_rows(out, want, tol)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("size", [1e-30, 1e-20, 1e33, 1e35, 1e36, 1e37])
def test_bf16_values_of_any_size(dc, cuda, d, size):
    """The sum of p V before its division stays in range wherever the plain sum of exp(s - max) V does."""
    case = (2, 3, 4, 2, d, 16, 0, [40, 300], 130)
    q, gate, cache, prefix, _ = attention_case(dc, cuda, case, seed=161)
    for c, s in ((cache, 13), (prefix, 14)):
        c.v[0].copy_(size * (torch.rand(c.v[0].shape, generator=gen(s, cuda), device=cuda) - 0.5))
    out = dc.stack_attn_decode_batch(q, cache, lens_tensor(case[7], cuda), d ** -0.5, prefix=prefix, prefix_len=130)
    want, tol = attention_want(q, None, cache, prefix, None, case, d ** -0.5)
    check_rows(out, want, tol)
