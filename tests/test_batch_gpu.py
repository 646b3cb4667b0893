"""The batch entries against their 64-bit statements (batch_ref): sizes where tiles, groups and
splits end, trees, ragged and absent sequences, values that a token must not see, strides,
streams, graphs, and the three entries run one after another as a verify round runs them."""
from __future__ import annotations

import math
from dataclasses import replace

import pytest
import torch

import batch_ref as R

pytestmark = pytest.mark.gpu
NAN = float("nan")


def gen(seed, dev):
    return torch.Generator(device=dev).manual_seed(seed)


def lens_tensor(lens, dev):
    return torch.tensor(lens, dtype=torch.int32, device=dev)


def fill(dc, dev, S, hkv, max_len, d, bits, group, seed, std=1.0):
    """A cache of random rows, quantised by the 64-bit rule."""
    g = gen(seed, dev)
    k, v = (R.quantise(std * torch.randn(S, hkv, max_len, d, generator=g, device=dev).to(torch.bfloat16), bits, group or 32)
            for _ in range(2))
    return dc.KVCache.of(k, v, bits, group)


def poison(cache, seq, rows):
    """Cache rows of a sequence become NaN (bf16 values, or scales and biases)."""
    for part in (cache.k, cache.v):
        for t in (part if cache.bits != 16 else part[:1]):
            if t.dtype == torch.bfloat16:
                t[seq, :, rows] = NAN
            else:
                t[seq, :, rows] = -1


# ----------------------------------------------------------------------------- prep

PREP = [
    # S, T, hq, hkv, d, bits, group, rot, lens, position0
    (1, 1, 1, 1, 64, 16, 0, 64, [0], 0),
    (1, 8, 24, 4, 256, 8, 64, 64, [1024], 0),
    (3, 5, 6, 2, 128, 4, 32, 128, [0, 7, 2], 1_000_003),
    (2, 33, 4, 4, 64, 8, 32, 64, [5, 0], 9),
    (4, 1, 8, 1, 256, 4, 128, 192, [3, -1, 0, 40], 100),
    (2, 3, 5, 1, 64, 4, 64, 0, [1, 2], 0),
    (1, 300, 2, 1, 128, 8, 128, 64, [0], 131072),
    (2, 2, 2, 2, 256, 16, 0, 256, [-1, 11], 2 ** 30),
    (1, 7, 2, 2, 128, 4, 64, 64, [0], 0),
]


@pytest.mark.parametrize("case", PREP, ids=str)
@pytest.mark.parametrize("tree", [False, True])
def test_prep_writes_what_the_formula_says(dc, cuda, case, tree):
    S, T, hq, hkv, d, bits, group, rot, lens, pos0 = case
    if tree and T > 32:
        pytest.skip("trees have at most 32 rows")
    eps, theta, max_len = 1e-6, 1e4, max(lens) + T + 3
    g = gen(1, cuda)
    ld = (2 * hq + 2 * hkv) * d + 24
    qkv = (torch.randn(S * T, ld, generator=g, device=cuda) * 3).to(torch.bfloat16)
    before = qkv.clone()
    qn, kn = (torch.randn(d, generator=g, device=cuda).to(torch.bfloat16) for _ in range(2))
    cache = fill(dc, cuda, S, hkv, max_len, d, bits, group, 2)
    old = [t.clone() for t in cache.k + cache.v if t is not None]
    parents = None
    if tree:
        parents = torch.tensor([[-1] + [int(torch.randint(0, t, (1,), generator=torch.Generator().manual_seed(97 * b + t)))
                                        for t in range(1, T)] for b in range(S)], dtype=torch.int32)
    q_out = torch.full((S * T, hq * d + 8), 7.0, dtype=torch.bfloat16, device=cuda)
    dc.stack_attn_prep_batch(qkv, qn, kn, cache, lens_tensor(lens, cuda), hq, rot, eps, theta, q_out=q_out, position0=pos0,
                             parents=None if parents is None else parents.to(cuda))
    torch.cuda.synchronize()
    assert dc.device_error() == 0 and torch.equal(qkv, before)
    assert (q_out[:, hq * d:] == 7).all()
    new = [t for t in cache.k + cache.v if t is not None]
    for b, n in enumerate(lens):
        rows = slice(b * T, (b + 1) * T)
        keep = [i for i in range(max_len) if n < 0 or not n <= i < n + T]
        for o, t in zip(old, new):  # every other row as it was
            assert torch.equal(o[b][:, keep], t[b][:, keep])
        if n < 0:
            assert (q_out[rows] == 7).all()
            continue
        depth, _ = R.depths(None if parents is None else parents[b].tolist(), T)
        pos = torch.tensor(depth, device=cuda) + (pos0 + n)
        x = qkv[rows, :(2 * hq + 2 * hkv) * d].reshape(T, -1, d)
        q = R.norm_rope(x[:, :hq], qn, pos, rot, eps, theta)
        tol = R.NORM * q.abs().amax(-1, keepdim=True)
        assert ((q_out[rows, :hq * d].reshape(T, hq, d).double() - q).abs() <= R.BF16 * q.abs() + 2 * tol).all()
        k = R.norm_rope(x[:, 2 * hq:2 * hq + hkv], kn, pos, rot, eps, theta)
        for part, want in ((cache.k, k), (cache.v, x[:, 2 * hq + hkv:].double())):
            want = want.transpose(0, 1)
            stored = tuple(None if t is None else t[b][:, n:n + T] for t in part)
            got = R.values(stored, bits, group)
            off = R.NORM * want.abs().amax(-1, keepdim=True) if part is cache.k else torch.zeros_like(want[..., :1])
            if bits == 16:
                assert ((got - want).abs() <= R.BF16 * want.abs() + 2 * off).all()
                continue
            # the nearest value that the stored scale and bias offer, up to the error of the normalised value
            s, z = (t.double().repeat_interleave(group, -1) for t in stored[1:])
            best = torch.round((want - z) / s).clamp(0, 2 ** bits - 1) * s + z
            assert ((got - want).abs() <= (best - want).abs() + 4 * off).all()
            # scale and bias of the rule: a bf16 rounding, and for the scale the code of zero (one of 2^bits - 1 over 2)
            rs, rb = (t.double() for t in R.quantise(want, bits, group)[1:])
            assert ((stored[2].double() - rb).abs() <= 2 * R.BF16 * rb.abs() + 4 * off).all()
            assert ((stored[1].double() / rs).abs() - 1).abs().max() <= 2.0 / (2 ** bits - 1) + 2 * R.BF16


def test_prep_in_place_and_a_length_past_the_end(dc, cuda):
    g = gen(3, cuda)
    qkv = torch.randn(6, 8 * 64, generator=g, device=cuda).to(torch.bfloat16)
    w = torch.ones(64, dtype=torch.bfloat16, device=cuda)
    a, b = (fill(dc, cuda, 3, 2, 10, 64, 8, 64, 4) for _ in range(2))
    lens = lens_tensor([8, 9, 0], cuda)  # the middle block would end at row 11 of 10
    apart = torch.full((6, 128), 5.0, dtype=torch.bfloat16, device=cuda)
    dc.stack_attn_prep_batch(qkv, w, w, a, lens, 2, 64, 1e-6, 1e4, q_out=apart)
    assert dc.device_error() == dc.DEVERR_POSITION
    assert (apart[2:4] == 5).all() and not (apart[[0, 1, 4, 5]] == 5).all()
    inside = qkv.clone()
    dc.stack_attn_prep_batch(inside, w, w, b, lens, 2, 64, 1e-6, 1e4, q_out=inside)
    assert dc.device_error() == dc.DEVERR_POSITION
    assert torch.equal(inside[[0, 1, 4, 5], :128], apart[[0, 1, 4, 5]])
    assert torch.equal(inside[2:4], qkv[2:4]) and torch.equal(inside[:, 128:], qkv[:, 128:])
    for x, y, z in zip(a.k + a.v, b.k + b.v, fill(dc, cuda, 3, 2, 10, 64, 8, 64, 4).k * 2):
        assert torch.equal(x, y)
    assert torch.equal(a.k[0][1], fill(dc, cuda, 3, 2, 10, 64, 8, 64, 4).k[0][1])


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("kind", ["zeros", "constant", "tiny", "symmetric", "inf", "nan", "huge"])
def test_groups_at_the_edge_of_the_rule(dc, cuda, bits, kind):
    x = torch.randn(1, 1, 4, 128, generator=gen(5, cuda), device=cuda)
    one = {"zeros": 0 * x, "constant": 0 * x - 1.375, "tiny": x * 1e-9, "symmetric": torch.sign(x) * 2.5, "inf": x.clone(),
           "nan": x.clone(), "huge": x * 1e30}[kind]
    if kind in ("inf", "nan"):
        one[0, 0, 1, 70] = math.inf if kind == "inf" else NAN
    one = one.to(torch.bfloat16)
    cache = dc.KVCache(1, 1, 9, 128, bits, 64, cuda)
    dc.stack_kv_write(cache, one, one, starts=lens_tensor([5], cuda))
    k, v = dc.stack_kv_read(cache, 4, starts=lens_tensor([5], cuda))
    torch.cuda.synchronize()
    assert dc.device_error() == 0 and torch.equal(k.view(torch.int16), v.view(torch.int16))
    want = R.values(R.quantise(one.double(), bits, 64), bits, 64)
    bad = torch.zeros_like(one, dtype=torch.bool)
    if kind in ("inf", "nan"):
        bad[0, 0, 1, 64:] = True
        assert k[bad].isnan().all()
    assert torch.equal(k[~bad].double(), want.to(torch.bfloat16)[~bad].double())
    assert not cache.k[0][0, 0, :5].any()


@pytest.mark.parametrize("bits,group,d", [(16, 0, 64), (8, 32, 256), (4, 64, 64), (4, 128, 128), (8, 64, 128)])
def test_write_and_read_back(dc, cuda, bits, group, d):
    S, hkv, max_len, rows = 4, 3, 50, 17
    g = gen(6, cuda)
    k, v = (torch.randn(S, hkv, rows, d, generator=g, device=cuda).to(torch.bfloat16) for _ in range(2))
    cache, starts = dc.KVCache(S, hkv, max_len, d, bits, group, cuda), [33, 0, -1, 34]  # the last one ends at row 51
    dc.stack_kv_write(cache, k, v, starts=lens_tensor(starts, cuda))
    assert dc.device_error() == dc.DEVERR_POSITION
    back = [torch.full_like(k, 9.0) for _ in range(2)]
    dc.stack_kv_read(cache, rows, starts=lens_tensor(starts, cuda), k=back[0], v=back[1])
    assert dc.device_error() == dc.DEVERR_POSITION
    for x, part, got in ((k, cache.k, back[0]), (v, cache.v, back[1])):
        want = R.values(R.quantise(x.double(), bits, group), bits, group).to(torch.bfloat16)
        assert torch.equal(got[:2], want[:2]) and (got[2:] == 9).all()
        assert not part[0][2:].any()
    whole, _ = dc.stack_kv_read(cache, max_len)
    assert torch.equal(whole[0, :, 33:], back[0][0])


@pytest.mark.parametrize("bits,group,d", [(16, 0, 256), (8, 64, 128), (4, 32, 64)])
def test_compact_moves_the_paths(dc, cuda, bits, group, d):
    S, hkv, max_len, stride = 5, 2, 40, 8
    cache = fill(dc, cuda, S, hkv, max_len, d, bits, group, 8)
    old = [None if t is None else t.clone() for t in cache.k + cache.v]
    lens, counts = [3, 30, -1, 10, 10], [4, 3, 2, 0, 2]
    rows = torch.zeros(S, stride, dtype=torch.int32)
    rows[0, :4] = torch.tensor([0, 2, 3, 7])
    rows[1, :3] = torch.tensor([0, 1, 9])
    rows[4, :2] = torch.tensor([0, 31])  # row 41 of 40: refused
    dc.stack_kv_compact_batch(cache, lens_tensor(lens, cuda), rows.to(cuda), lens_tensor(counts, cuda))
    assert dc.device_error() == dc.DEVERR_POSITION
    for o, t in zip(old, cache.k + cache.v):
        if o is None:
            continue
        want = o.clone()
        for b in (0, 1):
            src = [lens[b] + int(r) for r in rows[b, :counts[b]]]
            want[b][:, lens[b]:lens[b] + counts[b]] = o[b][:, src]
        assert torch.equal(t, want)


# ----------------------------------------------------------------------------- attention

ATTN = [
    # S, T, hq, hkv, d, bits, group, lens, prefix_len
    (1, 1, 1, 1, 64, 16, 0, [0], 0),
    (1, 1, 1, 1, 64, 4, 64, [0], 1),
    (1, 8, 24, 4, 256, 8, 64, [1024], 0),
    (3, 2, 6, 2, 128, 16, 0, [126, 127, 128], 0),
    (4, 1, 8, 1, 256, 4, 128, [255, -1, 0, 700], 129),
    (2, 4, 10, 2, 64, 8, 32, [0, 3], 127),
    (5, 3, 7, 1, 128, 4, 32, [1, 2, 3, 4, 900], 128),
    (2, 40, 12, 2, 128, 16, 0, [100, 0], 300),
    (1, 200, 8, 2, 256, 8, 64, [70], 0),
    (1, 130, 2, 2, 64, 4, 64, [500], 5),
    (40, 1, 6, 2, 64, 8, 64, [11 * i for i in range(40)], 1000),
    (2, 3, 34, 2, 128, 8, 128, [513, 60], 257),
    (1, 5, 4, 4, 128, 16, 0, [3000], 0),
    (9, 16, 8, 1, 256, 16, 0, [64 * i for i in range(9)], 640),
]


def attention_case(dc, dev, case, tree=False, seed=11, spoil=False, q_std=1.0):
    S, T, hq, hkv, d, bits, group, lens, P = case
    g = gen(seed, dev)
    cache = fill(dc, dev, S, hkv, max(lens) + T + 5, d, bits, group, seed + 1)
    prefix = fill(dc, dev, 1, hkv, P + 3, d, bits, group, seed + 2) if P else None
    if spoil:  # rows that nothing may see
        for b, n in enumerate(lens):
            poison(cache, b, slice(max(n, -T) + T, None))
        if P:
            poison(prefix, 0, slice(P, None))
    q, gate = ((s * torch.randn(S * T, hq * d + 16, generator=g, device=dev)).to(torch.bfloat16)[:, 8:8 + hq * d]
               for s in (q_std, 1.0))
    parents = None
    if tree:
        parents = torch.tensor([[-1] + [int(torch.randint(0, t, (1,), generator=torch.Generator().manual_seed(31 * b + t)))
                                        for t in range(1, T)] for b in range(S)], dtype=torch.int32)
    return q, gate, cache, prefix, parents


def attention_want(q, gate, cache, prefix, parents, case, scale):
    """Reference output and tolerance per row, NaN rows for sequences that take no part."""
    S, T, hq, hkv, d, bits, group, lens, P = case
    eps_kv, eps_p = (0.0, R.BF16) if bits == 16 else (R.FP16, R.FP16)
    ks, vs = R.values(cache.k, bits, group), R.values(cache.v, bits, group)
    if P:
        pk, pv = R.values(prefix.k, bits, group)[0, :, :P], R.values(prefix.v, bits, group)[0, :, :P]
    out = torch.full((S, T, hq, d), NAN, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    G = hq // hkv
    for b, n in enumerate(lens):
        if n < 0:
            continue
        _, block = R.depths(None if parents is None else parents[b].tolist(), T)
        seen = torch.cat([torch.ones(T, P + n, dtype=torch.bool), block], 1).to(q.device)
        for h in range(hkv):
            k, v = ks[b, h, :n + T], vs[b, h, :n + T]
            if P:
                k, v = torch.cat([pk[h], k]), torch.cat([pv[h], v])
            for gq in range(G):
                j = h * G + gq
                o, t = R.attention(q[b * T:(b + 1) * T, j * d:(j + 1) * d], k, v, seen, scale, eps_kv, eps_p)
                out[b, :, j], tol[b, :, j] = o, t
    out, tol = out.reshape(S * T, -1), tol.reshape(S * T, -1)
    if gate is not None:
        sg = torch.sigmoid(gate.double())
        out, tol = out * sg, tol * sg
    return out, R.BF16 * out.abs() * (1 + 2.0 ** -10) + tol * (1 + R.BF16) + 2.0 ** -130


def check_rows(got, want, tol, sentinel=None):
    live = ~want.isnan()
    assert got[live].isfinite().all()
    over = ((got.double() - want).abs() - tol)[live]
    assert over.numel() == 0 or over.max() <= 0, f"off by up to {over.max():.3g} more than allowed"
    if sentinel is not None:
        assert (got[~live] == sentinel).all()


@pytest.mark.parametrize("case", ATTN, ids=str)
@pytest.mark.parametrize("tree", [False, True])
def test_attention_is_the_formula(dc, cuda, case, tree):
    S, T, hq, hkv, d, bits, group, lens, P = case
    if tree and T > 32:
        pytest.skip("trees have at most 32 rows")
    q, gate, cache, prefix, parents = attention_case(dc, cuda, case, tree, spoil=True)
    gate = gate if S != 2 else None
    out = torch.full((S * T, hq * d), 3.0, dtype=torch.bfloat16, device=cuda)
    dc.stack_attn_decode_batch(q, cache, lens_tensor(lens, cuda), d ** -0.5, out=out, gate=gate, prefix=prefix,
                               prefix_len=P, parents=None if parents is None else parents.to(cuda))
    torch.cuda.synchronize()
    assert dc.device_error() == 0
    want, tol = attention_want(q, gate, cache, prefix, parents, case, d ** -0.5)
    check_rows(out, want, tol, 3.0)


@pytest.mark.parametrize("case", [ATTN[2], ATTN[4], ATTN[7], ATTN[9]], ids=str)
def test_attention_with_sharp_scores(dc, cuda, case):
    """Scores of a few hundred: one key has all the weight, and running maxima move late."""
    q, gate, cache, prefix, _ = attention_case(dc, cuda, case, seed=21, q_std=24.0)
    out = dc.stack_attn_decode_batch(q, cache, lens_tensor(case[7], cuda), 1.0, gate=gate, prefix=prefix,
                                     prefix_len=case[8])
    want, tol = attention_want(q, gate, cache, prefix, None, case, 1.0)
    check_rows(out, want, tol)


@pytest.mark.parametrize("bits,group", [(16, 0), (8, 64), (4, 32)])
@pytest.mark.parametrize("size", [1e-6, 3e4])
def test_attention_over_values_of_unusual_size(dc, cuda, bits, group, size):
    case = (2, 3, 4, 2, 128, bits, group, [40, 300], 130)
    q, gate, cache, prefix, _ = attention_case(dc, cuda, case, seed=31)
    for c, s in ((cache, 5), (prefix, 6)):
        big = (size * torch.randn(c.sequences, c.kv_heads, c.max_len, 128, generator=gen(s, cuda), device=cuda))
        for t, n in zip(c.v, R.quantise(big.to(torch.bfloat16).double(), bits, group)):
            if t is not None:
                t.copy_(n)
    out = dc.stack_attn_decode_batch(q, cache, lens_tensor(case[7], cuda), 128 ** -0.5, prefix=prefix, prefix_len=130)
    want, tol = attention_want(q, None, cache, prefix, None, case, 128 ** -0.5)
    check_rows(out, want, tol)


@pytest.mark.parametrize("bits,group", [(16, 0), (8, 64), (4, 32)])
@pytest.mark.parametrize("what", [NAN, math.inf])
@pytest.mark.parametrize("tree", [False, True])
def test_a_row_that_a_token_does_not_see_does_not_reach_it(dc, cuda, bits, group, what, tree):
    """The last block row's k and v, not finite, reach that row's own output alone."""
    case = (2, 6, 8, 2, 128, bits, group, [125, 30], 20)
    S, T = case[:2]
    q, gate, cache, prefix, _ = attention_case(dc, cuda, case, seed=41)
    parents = torch.tensor([[-1, 0, 0, 1, 2, 2]] * 2, dtype=torch.int32) if tree else None
    want, tol = attention_want(q, gate, cache, prefix, parents, case, 128 ** -0.5)
    for b, n in enumerate(case[7]):
        for part in (cache.k, cache.v):
            for t in (part[:1] if bits == 16 else part[1:]):
                t[b, :, n + T - 1] = what
    q[T - 1] = what  # and a q row that is not finite spoils itself alone
    out = dc.stack_attn_decode_batch(q, cache, lens_tensor(case[7], cuda), 128 ** -0.5, gate=gate, prefix=prefix,
                                     prefix_len=20, parents=None if parents is None else parents.to(cuda))
    torch.cuda.synchronize()
    good = torch.ones(S * T, dtype=torch.bool, device=cuda)
    good[[T - 1, 2 * T - 1]] = False
    check_rows(out[good], want[good], tol[good])
    assert not out[~good].isfinite().any()


def test_a_length_past_the_end_is_refused(dc, cuda):
    case = (3, 4, 4, 2, 64, 8, 64, [5, 0, 9], 0)
    q, gate, cache, _, _ = attention_case(dc, cuda, case)
    lens = [5, cache.max_len - 3, 9]
    out = torch.full((12, 256), 3.0, dtype=torch.bfloat16, device=cuda)
    dc.stack_attn_decode_batch(q, cache, lens_tensor(lens, cuda), 0.125, out=out)
    assert dc.device_error() == dc.DEVERR_POSITION
    want, tol = attention_want(q, None, cache, None, None, case[:7] + ([5, -1, 9], 0), 0.125)
    check_rows(out, want, tol, 3.0)


def test_attention_is_the_same_every_time(dc, cuda):
    case = ATTN[10]
    q, gate, cache, prefix, _ = attention_case(dc, cuda, case)
    f = lambda: dc.stack_attn_decode_batch(q, cache, lens_tensor(case[7], cuda), 0.125, gate=gate,  # noqa: E731
                                           prefix=prefix, prefix_len=case[8])
    first = f()
    for _ in range(5):
        assert torch.equal(f(), first)


@pytest.mark.parametrize("case", [
    (2, 509, 16, 2, 128, 8, 32, [7000, 3100], 0), (1, 8, 24, 4, 256, 8, 64, [20000], 0), (3, 2, 24, 4, 256, 4, 32, [9000, 4000, 1], 700),
    (2, 40, 24, 4, 256, 8, 32, [5000, 100], 0), (4, 16, 8, 1, 64, 4, 32, [3000, 10, 8000, 400], 2000),
    (2, 100, 8, 2, 256, 16, 0, [6000, 50], 1000), (9, 3, 16, 2, 128, 4, 128, [1000 * i for i in range(9)], 5000),
], ids=str)
def test_long_runs_of_tiles_back_to_back(dc, cuda, case):
    """Many tiles per CTA, calls that follow each other without a pause, and every call the same bits:
    what a slot reused too early or a wait for the wrong phase would change."""
    q, gate, cache, prefix, _ = attention_case(dc, cuda, case, seed=71)
    lens = lens_tensor(case[7], cuda)
    f = lambda: dc.stack_attn_decode_batch(q, cache, lens, case[4] ** -0.5, gate=gate, prefix=prefix,  # noqa: E731
                                           prefix_len=case[8])
    outs = [f() for _ in range(40)]
    torch.cuda.synchronize()
    assert dc.device_error() == 0
    assert all(torch.equal(o, outs[0]) for o in outs)
    want, tol = attention_want(q, gate, cache, prefix, None, case, case[4] ** -0.5)
    check_rows(outs[0], want, tol)


def test_an_offset_past_32_bits(dc, cuda):
    """The last rows of a cache of 5 GB: element offsets pass 2^32."""
    hkv, d, max_len = 2, 256, 4_200_000
    cache = dc.KVCache(2, hkv, max_len, d, 8, 128, cuda)
    n, T = max_len - 2, 2
    lens = lens_tensor([-1, n], cuda)
    # every cached row is one row: the answer is that row's value, plus the block's two rows
    g = gen(51, cuda)
    row = torch.randn(1, hkv, 1, d, generator=g, device=cuda).to(torch.bfloat16)
    part = R.quantise(row.double(), 8, 128)
    for cache_part in (cache.k, cache.v):
        for t, p in zip(cache_part, part):
            t[1] = p[0]
    qkv = torch.randn(4, (2 * 2 + 2 * hkv) * d, generator=g, device=cuda).to(torch.bfloat16)
    w = torch.ones(d, dtype=torch.bfloat16, device=cuda)
    q = dc.stack_attn_prep_batch(qkv, w, w, cache, lens, 2, 64, 1e-6, 1e4)
    k, v = dc.stack_kv_read(cache, T, starts=lens)
    out = dc.stack_attn_decode_batch(q, cache, lens, 0.5)
    torch.cuda.synchronize()
    assert dc.device_error() == 0
    x = qkv.view(4, -1, d)[2:]
    assert torch.equal(v[1].transpose(0, 1).double(),
                       R.values(R.quantise(x[:, 2 * 2 + hkv:].double(), 8, 128), 8, 128).to(torch.bfloat16).double())
    kv, vv = R.values(tuple(t[1:, :, n:] for t in cache.k), 8, 128), R.values(tuple(t[1:, :, n:] for t in cache.v), 8, 128)
    base = R.values(part, 8, 128)
    for h in range(hkv):
        for t in range(T):
            qr = q[2 + t, h * d:(h + 1) * d].double()
            s = torch.cat([(qr @ base[0, h, 0] * 0.5 + math.log(n))[None], kv[0, h, :t + 1] @ qr * 0.5])
            want = torch.softmax(s, 0) @ torch.cat([base[0, h], vv[0, h, :t + 1]])
            # weights off by e^(2 delta), delta = 2^-11 0.5 sum |q||k| < 2^-11 256; all weight is on equal rows
            far = (R.BF16 + 2 * R.FP16 + 2.0 ** -12) * want.abs().max() + math.expm1(2 * R.FP16 * 0.5 * float(
                (qr.abs() @ base[0, h, 0].abs()).item())) * vv.abs().max()
            assert ((out[2 + t, h * d:(h + 1) * d].double() - want).abs() <= far).all()


# ----------------------------------------------------------------------------- streams, graphs, devices

def test_two_graphs_and_another_stream(dc, cuda):
    """Two captured calls replayed at once on two streams, at lengths that move between replays."""
    calls = []
    for i, case in enumerate((ATTN[10], ATTN[7])):
        q, gate, cache, prefix, _ = attention_case(dc, cuda, case, seed=61 + i)
        lens, stream = lens_tensor(case[7], cuda), torch.cuda.Stream()
        torch.cuda.synchronize()
        f = lambda q=q, gate=gate, cache=cache, prefix=prefix, lens=lens, P=case[8], d=case[4]: \
            dc.stack_attn_decode_batch(q, cache, lens, d ** -0.5, gate=gate, prefix=prefix, prefix_len=P)  # noqa: E731
        f()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            out = f()
        calls.append((graph, stream, out, case, lens, (q, gate, cache, prefix)))
    for shift in (0, 3, 1):
        torch.cuda.synchronize()
        for _, _, _, case, lens, _ in calls:
            lens.copy_(lens_tensor([max(n - shift, 0) for n in case[7]], cuda))
        torch.cuda.synchronize()
        for _ in range(3):
            for graph, stream, *_ in calls:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for _, _, out, case, lens, state in calls:
            moved = case[:7] + ([max(n - shift, 0) for n in case[7]], case[8])
            want, tol = attention_want(*state, None, moved, case[4] ** -0.5)
            check_rows(out, want, tol)
    del calls


def test_a_stream_that_is_not_the_current_one(dc, cuda):
    case = ATTN[6]
    q, gate, cache, prefix, _ = attention_case(dc, cuda, case)
    lens, other = lens_tensor(case[7], cuda), torch.cuda.Stream()
    want = dc.stack_attn_decode_batch(q, cache, lens, 0.1, gate=gate, prefix=prefix, prefix_len=case[8])
    logits = torch.randn(9, 1001, device=cuda)
    lp = dc.logprobs(logits, top=3)
    torch.cuda.synchronize()
    got = dc.stack_attn_decode_batch(q, cache, lens, 0.1, gate=gate, prefix=prefix, prefix_len=case[8], stream=other)
    lq = dc.logprobs(logits, top=3, stream=other)
    other.synchronize()
    assert torch.equal(got, want) and all(torch.equal(lp[k], lq[k]) for k in lp)


# ----------------------------------------------------------------------------- log probabilities

def logprob_want(x, tokens, top):
    x = x.double()
    lp = torch.log_softmax(x, -1)
    ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
    ent = -(lp.exp() * lp).nan_to_num(0.0).sum(-1)
    given = torch.where(tokens < 0, 0.0, lp.gather(1, tokens.long().clamp(min=0)))
    return given, ent, ids, lp.gather(1, ids), x.amax(-1, keepdim=True) - torch.logsumexp(x, -1, keepdim=True), lp


# An exponential is off by 2^-22 relative plus 2^-23 of its argument's size, which weighs at most
# |y| e^y; sums of up to 2^18 values in pieces add 2^-18 at most.  So log l is off by 2^-17, an
# entropy's second term by 2^-17 of its size, and a difference adds a rounding of its terms.
def near(got, want, extra=0.0):
    same = torch.isinf(want) & (got == want)
    return (same | ((got.double() - want).abs() <= 2.0 ** -17 + 2.0 ** -17 * want.abs().nan_to_num(0, 0, 0) + extra)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R_,V,pad,off,n,top", [
    (1, 1, 0, 0, 1, 1), (3, 2, 1, 0, 2, 2), (2, 31, 0, 1, 1, 31), (5, 33, 3, 1, 4, 32), (7, 1000, 0, 3, 1, 0),
    (4, 1023, 5, 1, 3, 20), (1, 248320, 0, 0, 1, 20), (9, 65537, 7, 5, 2, 5), (300, 4097, 0, 0, 1, 8), (150, 511, 1, 0, 1, 3),
    (40, 50021, 3, 0, 1, 32),
])
@pytest.mark.parametrize("kind", ["random", "ties", "sorted", "masked"])
def test_logprobs(dc, cuda, dtype, R_, V, pad, off, n, top, kind):
    g = gen(71, cuda)
    x = torch.randn(R_, V + pad + off, generator=g, device=cuda) * 4
    if kind == "ties":
        x = torch.round(x / 4)
    elif kind == "sorted":
        x = torch.sort(x, dim=1).values if R_ % 2 else torch.sort(x, dim=1, descending=True).values
    elif kind == "masked":
        x = torch.where(torch.rand(x.shape, generator=g, device=cuda) < 0.9, -math.inf, x)
        x[:, off + V // 2] = 1.0
    x = x.to(dtype)[:, off:off + V]
    tokens = torch.randint(0, V, (R_, n), generator=g, device=cuda, dtype=torch.int32)
    tokens[0, 0] = -1
    got = dc.logprobs(x, tokens, top=top)
    torch.cuda.synchronize()
    given, ent, ids, best, _, lp = logprob_want(x, tokens, top)
    assert torch.equal(got["top_ids"].long(), ids)
    assert near(got["logprobs"], given) and near(got["top_logprobs"], best)
    size = (lp.exp() * lp).nan_to_num(0.0).abs().sum(-1)
    assert near(got["entropy"], ent, 2.0 ** -16 * size)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_without_a_distribution(dc, cuda, dtype):
    x = torch.randn(6, 3001, generator=gen(81, cuda), device=cuda).to(dtype)
    x[0, 2999] = NAN
    x[1, 17] = math.inf
    x[2] = -math.inf
    x[3, 5:] = -math.inf
    x[4] = torch.finfo(dtype).min
    tokens = torch.tensor([[1, -1, 3001], [1, -1, 0], [1, -1, 0], [4000, 2, 7], [0, 3000, -2], [3000, 2, 2 ** 31 - 1]],
                          dtype=torch.int32, device=cuda)
    got = dc.logprobs(x, tokens, top=4)
    torch.cuda.synchronize()
    for r in range(3):
        assert got["entropy"][r].isnan() and (got["top_ids"][r] == -1).all() and got["top_logprobs"][r].isnan().all()
        assert got["logprobs"][r, 0].isnan() and got["logprobs"][r, 1] == 0
    assert got["logprobs"][0, 2].isnan() and got["logprobs"][3, 0].isnan() and got["logprobs"][5, 2].isnan()
    lp = torch.log_softmax(x[3:].double(), -1)
    assert got["logprobs"][3, 2] == -math.inf and near(got["logprobs"][3, 1], lp[0, 2])
    assert near(got["logprobs"][4, :2], lp[1, [0, 3000]]) and got["logprobs"][4, 2] == 0
    assert got["top_ids"][4].tolist() == [0, 1, 2, 3] and near(got["entropy"][4], torch.tensor(math.log(3001), device=cuda))


def test_logprobs_outputs_that_are_left_out(dc, cuda):
    x = torch.randn(3, 500, device=cuda)
    whole = dc.logprobs(x, torch.zeros(3, 1, dtype=torch.int32, device=cuda), top=2)
    few = dc.logprobs(x)
    assert few["logprobs"].shape == (3, 0) and few["top_ids"].shape == (3, 0)
    assert torch.equal(few["entropy"], whole["entropy"])
    assert dc.logprobs(x[:0], top=2)["entropy"].shape == (0,)
    with pytest.raises(dc.DFlashError):
        dc.logprobs(x[:1].expand(3, 500))


# ----------------------------------------------------------------------------- together

@pytest.mark.parametrize("bits", [16, 8, 4])
def test_a_batch_prefills_a_prefix_and_decodes(dc, cuda, bits):
    """A prompt becomes the shared prefix; two sequences then extend it in blocks, one of them
    as a tree whose path is compacted; every step against the formula on the cache's own values."""
    hq, hkv, d, group, P = 6, 2, 128, 0 if bits == 16 else 64, 150
    g = gen(91, cuda)
    w = torch.ones(d, dtype=torch.bfloat16, device=cuda)
    rows = lambda n: torch.randn(n, (2 * hq + 2 * hkv) * d, generator=g, device=cuda).to(torch.bfloat16)  # noqa: E731
    prefix = dc.KVCache(1, hkv, P, d, bits, group or 64, cuda)
    zero = lens_tensor([0], cuda)
    x = rows(P)
    q = dc.stack_attn_prep_batch(x, w, w, prefix, zero, hq, 64, 1e-6, 1e4)
    out = dc.stack_attn_decode_batch(q, prefix, zero, d ** -0.5, gate=x[:, hq * d:2 * hq * d])
    case = (1, P, hq, hkv, d, bits, group, [0], 0)
    want, tol = attention_want(q, x[:, hq * d:2 * hq * d], prefix, None, None, case, d ** -0.5)
    check_rows(out, want, tol)
    cache, lens = dc.KVCache(2, hkv, 64, d, bits, group or 64, cuda), [0, 0]
    parents = torch.tensor([[-1, 0, 0, 1, 2], [-1, 0, 1, 2, 3]], dtype=torch.int32)
    for step in range(3):
        x, at = rows(10), lens_tensor(lens, cuda)
        q = dc.stack_attn_prep_batch(x, w, w, cache, at, hq, 64, 1e-6, 1e4, position0=P, parents=parents.to(cuda))
        gate = x[:, hq * d:2 * hq * d]
        out = dc.stack_attn_decode_batch(q, cache, at, d ** -0.5, gate=gate, prefix=prefix, parents=parents.to(cuda))
        want, tol = attention_want(q, gate, cache, prefix, parents, (2, 5, hq, hkv, d, bits, group, lens, P), d ** -0.5)
        check_rows(out, want, tol)
        path, count = torch.tensor([[0, 2, 4], [0, 1, 0]], dtype=torch.int32), [3, 2]
        moved = dc.stack_kv_read(cache, 5, starts=at)
        dc.stack_kv_compact_batch(cache, at, path.to(cuda), lens_tensor(count, cuda))
        kept = dc.stack_kv_read(cache, 3, starts=at)
        for a, b in zip(moved, kept):
            assert torch.equal(b[0], a[0][:, [0, 2, 4]]) and torch.equal(b[1][:, :2], a[1][:, :2])
        lens = [lens[0] + 3, lens[1] + 2]
    assert dc.device_error() == 0


@pytest.mark.parametrize("bits,bar", [(16, 2e-2), (8, 3e-2)])
@pytest.mark.parametrize("tree", [False, True])
def test_the_stack_over_a_batch_cache(dc, cuda, bits, bar, tree):
    """VerifyStack(kv_bits=...) against the stack over bf16 caches that hold the same tokens (what the
    quantised ones read back as): the block's own rows alone are quantised on top, in 8 bits by
    half a step, 2^-9 of a group's range (about 1e-2 of a value), in one of the four layers."""
    import verify_stack as vs
    cfg = vs.TINY
    caches = replace(cfg, block=24)
    plan = vs.shard_plan(cfg, 0, 1)
    weights = vs.build_rank_weights(cfg, plan, 0, cuda)
    new = vs.VerifyStack(cfg, device=cuda, weights=weights, state=vs.build_rank_state(caches, plan, 0, cuda), tree=tree,
                         kv_bits=bits)
    state = vs.build_rank_state(caches, plan, 0, cuda)
    for S, N in zip(state["layers"], new.state["layers"]):
        if "cache" in N:
            assert N["cache"].bits == bits and "cache_k" not in N
            k, v = dc.stack_kv_read(N["cache"], N["cache"].max_len)
            S["cache_k"].copy_(k[0])
            S["cache_v"].copy_(v[0])
    old = vs.VerifyStack(cfg, device=cuda, weights=weights, state=state, tree=tree)
    hidden = vs.make_block(cfg, 0, cuda)
    close = lambda a, b: ((a.float() - b.float()).abs().max() / b.float().abs().max()).item()  # noqa: E731
    rows = [0, 2, 5] if tree else [0, 1, 2]
    if tree:
        for s in (new, old):
            s.set_tree([-1, 0, 0, 1, 2, 2, 4, 5])
    proposals = torch.zeros(cfg.block - 1, dtype=torch.int32, device=cuda)
    graph = new.capture(hidden, proposals)
    for _ in range(2):
        graph.replay()
        old.verify(hidden, proposals)
        torch.cuda.synchronize()
        assert close(new.out, old.out) <= bar
        tokens = new.tokens.view(-1, 1).clone()
        lp = new.logprobs(tokens, top=1)
        assert torch.equal(lp["top_ids"][:, 0], new.tokens)  # the LM head's argmax is the likeliest token
        assert torch.equal(lp["top_logprobs"], lp["logprobs"])
        for s in (new, old):
            s.commit(rows)
            s.advance(3)
    del graph
    assert dc.device_error() == 0
    with pytest.raises(ValueError):
        new.advance(100)


@pytest.mark.parametrize("bits,group,bar", [(4, 64, 0.18), (4, 32, 0.18), (8, 32, 3e-2)])
def test_the_stack_over_smaller_caches_and_groups(dc, cuda, bits, group, bar):
    """As above with 4 bits, whose half step is 16 times that of 8 (2e-2 + 16 (3e-2 - 2e-2)), and groups of 32."""
    import verify_stack as vs
    cfg = vs.TINY
    caches = replace(cfg, block=24)
    plan = vs.shard_plan(cfg, 0, 1)
    weights = vs.build_rank_weights(cfg, plan, 0, cuda)
    new = vs.VerifyStack(cfg, device=cuda, weights=weights, state=vs.build_rank_state(caches, plan, 0, cuda), kv_bits=bits,
                         kv_group=group)
    state = vs.build_rank_state(caches, plan, 0, cuda)
    for S, N in zip(state["layers"], new.state["layers"]):
        if "cache" in N:
            assert (N["cache"].bits, N["cache"].group) == (bits, group)
            k, v = dc.stack_kv_read(N["cache"], N["cache"].max_len)
            S["cache_k"].copy_(k[0])
            S["cache_v"].copy_(v[0])
    old = vs.VerifyStack(cfg, device=cuda, weights=weights, state=state)
    hidden = vs.make_block(cfg, 0, cuda)
    for _ in range(2):
        a, b = new.forward(hidden).float(), old.forward(hidden).float()
        assert (a - b).abs().max() <= bar * b.abs().max()
        for s in (new, old):
            s.commit([0, 1, 2])
            s.advance(3)
    assert dc.device_error() == 0
