"""Log probabilities, entropy and alternatives of rows of logits against plain 64-bit forms."""
import math

import pytest
import torch

import plain_tree

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def score(x, ids, top, entropy=True):
    from rocml_b200 import kernels
    n, m = ids.shape
    out = dict(logprobs=torch.full((n, m), 9.0, device=DEV), entropy=torch.full((n,), 9.0, device=DEV) if entropy else None,
               top_logprobs=torch.full((n, top), 9.0, device=DEV) if top else None,
               top_ids=torch.full((n, top), 9, dtype=torch.int32, device=DEV) if top else None)
    kernels.token_logprobs(x, ids.to(DEV), **out)
    return out["logprobs"].cpu(), None if not entropy else out["entropy"].cpu(), out["top_logprobs"], out["top_ids"]


def close(got, want, what):
    """The sum of exponentials is 32-bit: terms to 2^-20 of themselves (exponents up to about 100 in base 2, to 2^-24 of themselves, and the
    special-function unit's 2^-22), fewer than 2^-20 more for adding up: 2e-6 on a logarithm, and a result's own rounding.  The entropy is two such
    parts, the second a sum of terms of one sign times up to log V (< 13): 4e-5."""
    got, want = got.double().cpu(), want.double()
    same = torch.isfinite(want)
    assert torch.equal(got[~same], want[~same]), what
    err = (got[same] - want[same]).abs()
    tol = (4e-5 if what == "entropy" else 3e-6) + 2 ** -23 * want[same].abs()
    assert (err <= tol).all(), (what, err.max().item())


def check(x, ids, top, **kw):
    got = score(x, ids, top, **kw)
    want = plain_tree.logprobs(x.cpu(), ids, top)
    close(got[0], want[0], "given")
    if got[1] is not None:
        close(got[1], want[1], "entropy")
    if top:
        assert torch.equal(got[3].cpu(), want[3])
        close(got[2], want[2], "top")


def logits(n, V, seed, dtype=torch.float32, spread=3.0, pad=0, shift=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.zeros((n * (V + pad) + shift + 64,), dtype=dtype)
    rows = x[shift:shift + n * (V + pad)].view(n, V + pad)
    rows.copy_((torch.randn((n, V + pad), generator=g) * spread).to(dtype))
    return x.to(DEV)[shift:shift + n * (V + pad)].view(n, V + pad)[:, :V]


def tokens(n, m, V, seed):
    return torch.randint(0, V, (n, m), generator=torch.Generator().manual_seed(seed)).int()


@pytest.mark.parametrize("n,V", [(1, 151936), (3, 32003), (1, 1), (5, 2), (2, 31), (40, 33), (7, 4096), (300, 5001), (9, 70001)])
@pytest.mark.parametrize("top", [0, 1, 5, 32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_logprobs(n, V, top, dtype):
    check(logits(n, V, n + V, dtype), tokens(n, 2, V, 1), min(top, V))


@pytest.mark.parametrize("pad,shift", [(0, 1), (1, 0), (2, 3), (5, 7), (64, 0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_logprobs_rows_off_every_boundary(pad, shift, dtype):
    """What lies between the rows is not theirs: it holds NaN."""
    x = logits(6, 3001, pad, dtype, pad=pad, shift=shift)
    whole = x.as_strided((6, 3001 + pad), (3001 + pad, 1), x.storage_offset())
    whole[:, 3001:] = float("nan")
    check(x, tokens(6, 3, 3001, 2), 9)


def test_token_logprobs_of_equal_and_ordered_values():
    """Ties go to the lowest id, wherever equal values lie; rows in ascending and descending order; -0 is 0."""
    V = 20000
    x = torch.zeros((6, V))
    x[1] = torch.arange(V).float() * 1e-3
    x[2] = -x[1]
    x[3, ::2] = -0.0
    x[4] = (torch.arange(V) % 7).float()
    x[5, 4096:] = 1.0
    check(x.to(DEV), tokens(6, 1, V, 3), 32)
    check(x.to(DEV)[:1].repeat(400, 1), tokens(400, 1, V, 4), 20)


def test_token_logprobs_of_rows_with_few_possible_tokens():
    """-inf is a token that cannot be: a handful left, one left, none left."""
    V = 50257
    x = torch.full((5, V), -math.inf)
    x[0, [5, 40000, 50256]] = torch.tensor([1.0, 2.0, -30.0])
    x[1, 777] = -4.0
    x[3] = torch.randn(V, generator=torch.Generator().manual_seed(1))
    x[3, ::3] = -math.inf
    x[4, 0] = 0.0
    ids = torch.tensor([[5, 6], [777, 0], [3, 4], [1, 3], [0, V - 1]], dtype=torch.int32)
    check(x.to(DEV), ids, 20)
    check(x.to(DEV).bfloat16(), ids, 20)


def test_token_logprobs_of_nearly_certain_and_of_huge_logits():
    x = torch.randn((4, 9000), generator=torch.Generator().manual_seed(2))
    x[0, 17] = 40.0
    x[1] = x[1] * 30 + 1e4
    x[2] = x[2] * 1e3 - 3e4
    x[3, 5] = 80.0
    x[3, 6] = 79.5
    ids = torch.tensor([[17], [0], [1], [6]], dtype=torch.int32)
    got = score(x.to(DEV), ids, 3)
    want = plain_tree.logprobs(x, ids, 3)
    # (exponents in base 2 of up to 1e5: 2^-24 of that is the error of a term's exponent, and so of the logarithm, relative to the terms that matter)
    for g, w in zip(got[:2], want[:2]):
        assert ((g.double() - w).abs() <= 2e-2 * (w.abs() > 100) + 2e-2 * (x.abs().amax(1) > 1e3).double().reshape(-1, *[1] * (w.dim() - 1)) + 4e-5 + 2 ** -23 * w.abs()).all()
    assert torch.equal(got[3].cpu(), want[3])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_logprobs_of_bad_rows_and_ids(dtype):
    """A NaN or +inf spoils its own row only; ids outside the vocabulary cannot be."""
    x = logits(4, 3000, 5, dtype)
    x[1, 2999] = float("nan")
    x[2, 0] = math.inf
    ids = torch.tensor([[-1, 3000, 5]] * 4, dtype=torch.int32)
    lp, ent, tl, ti = score(x, ids, 4)
    want = plain_tree.logprobs(x.cpu()[[0, 3]], ids[[0, 3]], 4)
    close(lp[[0, 3]], want[0], "given")
    assert torch.isneginf(lp[:, :2]).all()
    assert torch.isnan(lp[1:3, 2]).all() and torch.isnan(ent[1:3]).all() and torch.isfinite(ent[[0, 3]]).all()
    assert ((ti >= -1) & (ti < 3000)).all()


def test_token_logprobs_parts_that_are_not_asked_for():
    from rocml_b200 import kernels
    x = logits(3, 999, 6)
    want = plain_tree.logprobs(x.cpu(), tokens(3, 1, 999, 1), 2)
    ent = torch.zeros(3, device=DEV)
    kernels.token_logprobs(x, None, None, ent)
    close(ent, want[1], "entropy")
    tl, ti = torch.zeros((3, 2), device=DEV), torch.zeros((3, 2), dtype=torch.int32, device=DEV)
    kernels.token_logprobs(x, None, None, None, tl, ti)
    close(tl, want[2], "top")
    kernels.token_logprobs(x[:0], None, None, ent[:0])
    check(x, tokens(3, 70, 999, 7), 0, entropy=False)


def test_token_logprobs_twice_captured_and_past_32_bit_offsets():
    from rocml_b200 import kernels
    x = logits(33, 30011, 8)
    ids = tokens(33, 1, 30011, 9)
    a, b = score(x, ids, 8), score(x, ids, 8)
    assert all(torch.equal(p.cpu(), q.cpu()) for p, q in zip(a, b))
    out = [torch.zeros((33, 1), device=DEV), torch.zeros(33, device=DEV), torch.zeros((33, 8), device=DEV), torch.zeros((33, 8), dtype=torch.int32, device=DEV)]
    dev_ids = ids.to(DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kernels.token_logprobs(x, dev_ids, *out)
    graph.replay()
    assert all(torch.equal(p.cpu(), q.cpu()) for p, q in zip(a, out))
    for n, V, top in ((64, 151936, 20), (300, 32003, 8), (1, 151936, 32)):           # one block a row and clusters, the same bits every time
        y, first = logits(n, V, n), None
        for _ in range(60):
            got = [t.cpu() for t in score(y, tokens(n, 1, V, 2), top)]
            first = first or got
            assert all(torch.equal(p, q) for p, q in zip(first, got))
    big = torch.empty(2 ** 31 + 2 ** 20, dtype=torch.bfloat16, device=DEV)
    rows = big.as_strided((2, 30011), (2 ** 31 + 5, 1))
    rows.copy_(x[:2].bfloat16())
    check(rows, ids[:2], 8)


@pytest.mark.parametrize("V,top", [(2, 1), (33, 4), (9001, 0), (50257, 20), (151936, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gap", [4.0, 14.0, 24.0])
def test_token_logprobs_of_nearly_certain_tokens_are_relative(V, top, dtype, gap):
    """What a nearly certain token's probability lacks is the other tokens' share, and that is held to its own size.  A term's exponent d (in base 2, not
    below -70: what lies lower is less than 2^-20 of the share) is rounded twice and multiplied by a log2 e that is 1.4e-8 off: 70 ln 2 (2^-23 + 1.4e-8) =
    6.5e-6 of the term.  The special-function unit gives 2^-22 for the term and for each of some 20 raised maxima: 5e-6.  Chunks of 16: 1e-6.  Together
    1.3e-5, and the results' own roundings."""
    g = torch.Generator().manual_seed(V + int(gap))
    x = (torch.randn((6, V), generator=g) * 2).to(dtype)
    at = torch.tensor([0, V - 1, V // 2, V // 3, min(V - 1, 8), min(V - 1, 1000)])
    x[torch.arange(6), at] = (x.float().amax(1) + gap).to(dtype)
    d = x.double() - x.double().amax(1, keepdim=True)
    others = torch.where(torch.arange(V) == at[:, None], 0.0, d.exp())
    log_s = torch.log1p(others.sum(1))
    want = -log_s[:, None], log_s - (others * d).sum(1) / (1 + others.sum(1))
    for rows in (slice(0, 6), slice(2, 3)):
        got = score(x.to(DEV)[rows], at[rows, None].int(), top)
        for a, b in ((got[0], want[0][rows]), (got[1], want[1][rows])):
            a, b = a.double().cpu(), b.double()
            assert ((a - b).abs() <= 1.5e-5 * b.abs()).all(), ((a - b).abs() / b.abs()).max().item()
        if top:
            assert torch.equal(got[2].cpu()[:, 0], got[0][:, 0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_logprobs_of_the_types_lowest_and_highest_values(dtype):
    V = 4099
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    x = torch.full((5, V), low, dtype=dtype)
    x[1, 7], x[2, [7, 4098]], x[3, 0] = high, 0.0, -math.inf
    x[4] = torch.randn(V, generator=torch.Generator().manual_seed(1)).to(dtype)
    x[4, 1::2] = low
    ids = torch.tensor([[0, V - 1], [7, 8], [7, 4098], [1, 0], [2, 3]], dtype=torch.int32)
    got = score(x.to(DEV), ids, 2)
    a = math.log(V)
    want = torch.tensor([[-a, -a], [0.0, -math.inf], [-math.log(2), -math.log(2)], [-math.log(V - 1), -math.inf]], dtype=torch.float64)
    lp = got[0].double()
    for r, c in ((0, 0), (0, 1), (1, 0), (2, 0), (2, 1), (3, 0), (3, 1)):
        close(lp[r, c].reshape(1), want[r, c].reshape(1), "given")
    close(got[1][:4], torch.tensor([a, 0.0, math.log(2), math.log(V - 1)], dtype=torch.float64), "entropy")
    # a difference past the type's range, or just short of it: not above the lowest value
    assert lp[1, 1] <= low and lp[4, 1] <= 0.99 * low
    rest = plain_tree.logprobs(x[4:, ::2].contiguous(), torch.tensor([[1]], dtype=torch.int32), 2)
    close(got[0][4:, :1], rest[0], "given")
    close(got[1][4:], rest[1], "entropy")
    assert got[3].tolist()[0] == [0, 1] and got[3].tolist()[2] == [7, 4098]
