"""The batch entries at the ends of their types' ranges, against 64-bit statements."""
from __future__ import annotations

import pytest
import torch

import batch_ref as R
from test_batch_gpu import gen, lens_tensor, logprob_want, near

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
