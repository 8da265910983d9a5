"""K11 on the GPU where a filter's border or the random number meets a sum of weights exactly, where the
tokens must not depend on the rows beside them, and with more rows than a launch takes.

Equal logits have equal weights, so n of them (the rest -inf) have the sums j / n of all, whatever their
value: the expected tokens follow in whole numbers, and no tolerance is needed for them.  logprob is
-ln of the kept tokens' number: fp32's half step of the log, and 2^-50 for the quotient of two sums
that are n and 1 times the same weight."""

import math

import pytest
import torch

from .test_gpu_sample import BF, DEV, F32, K, check, draw

pytestmark = pytest.mark.gpu

VOCABS = [14, 64, 65, 1000, 4096, 4097, 30011, 131072]


def equal_rows(seed, rows, vocab, n, dtype, below=float("-inf")):
    """rows of n equal logits, of another value and at other places in each; places, ascending."""
    g = torch.Generator().manual_seed(seed)
    value = (torch.randn(rows, generator=g) * 6).to(dtype)
    at = torch.stack([torch.randperm(vocab, generator=g)[:n].sort().values for _ in range(rows)])
    x = (value[:, None].float() + below).to(dtype).expand(rows, vocab).contiguous()
    x.scatter_(1, at, value[:, None].expand(rows, n))
    heat = 0.3 + 2 * torch.rand(rows, generator=g)
    return x, at, heat, torch.rand(rows, generator=g)


def expect(token, lp, at, u, kept):
    """The tokens of rows whose first kept[r] of at[r] are kept, at equal weights."""
    for r in range(at.shape[0]):
        n = int(kept[r])
        j = min(int(float(u[r]) * n), n - 1)   # u n is exact: 24 bits and a power of two or a few
        assert int(token[r]) == int(at[r, j]), (r, n, float(u[r]))
        want = -math.log(n)
        assert abs(float(lp[r]) - want) <= (2.0 ** -24 + 2.0 ** -50) * abs(want), (r, n, float(lp[r]))


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("vocab,n", [(v, n) for v in VOCABS for n in (2, 4, 12, 64, 512, 8192) if n <= v])
def test_shares_that_meet_a_sum(dtype, vocab, n):
    """top-p of a quarter, a half and three quarters of n equal tokens keeps just as many."""
    rows = 24
    for q in (1, 2, 3):
        if n * q % 4:
            continue
        x, at, heat, u = equal_rows(100 * vocab + 10 * n + q, rows, vocab, n, dtype)
        p, kept = torch.full((rows,), q / 4), [n * q // 4] * rows
        token, lp = draw(x, u, top_p=p)
        expect(token, lp, at, u, kept)
        token, lp = draw(x, u, top_p=p, temperature=heat)
        expect(token, lp, at, u, kept)
        # of what top-k leaves, with other tokens below them in the row
        x, at, heat, u = equal_rows(100 * vocab + 10 * n + q, rows, vocab, n, dtype, below=-1.0)
        k = torch.full((rows,), n).int()
        if n < 4:
            continue   # a top_k of 2 and a share of a half are a row's first token: above
        token, lp = draw(x, u, top_k=k, top_p=p, temperature=heat)
        expect(token, lp, at, u, kept)
        # min-p between the two values: the shares are of the whole row, which p leaves as it is
        token, lp = draw(x, u, min_p=torch.full((rows,), 0.99), temperature=heat)
        expect(token, lp, at, u, [n] * rows)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("heat", [1e20, 1e30, float("inf")])
def test_temperatures_that_make_all_weights_equal(dtype, vocab, heat):
    """Weights differ by less than 2^-60, and the ones that are kept are the largest: a share of a quarter,
    a half or three quarters keeps as many of them."""
    g = torch.Generator().manual_seed(vocab)
    rows = 12
    x = (torch.randn(rows, vocab, generator=g) * 4).to(dtype)
    x[:, ::5] = -x[:, ::5].abs()
    u = torch.rand(rows, generator=g)
    n = vocab // 4 * 4
    x[:, n:] = float("-inf")
    order = x.float().sort(dim=1, descending=True, stable=True).indices
    for q in (1, 2, 3, 4):
        m = n * q // 4
        at = order[:, :m].sort(1).values
        p = torch.full((rows,), q / 4)
        token, lp = draw(x, u, top_p=p, temperature=torch.full((rows,), heat))
        for r in range(rows):
            # u m is exact in 64 bits (24 and 17 of them)
            assert int(token[r]) == int(at[r, int(float(u[r]) * m)]), (q, r)
            assert abs(float(lp[r]) + math.log(m)) <= (2.0 ** -24 + 2.0 ** -50) * math.log(m), (q, r)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("vocab,n", [(v, n) for v in VOCABS for n in (2, 4, 64, 8192) if n <= v])
def test_random_numbers_that_meet_a_sum(dtype, vocab, n):
    """u = j / n: the sum up to token j - 1 is not above it, that up to token j is."""
    rows = 24
    x, at, heat, _ = equal_rows(vocab + n, rows, vocab, n, dtype)
    u = (torch.arange(rows) * 37 % n).float() / n
    token, lp = draw(x, u)
    expect(token, lp, at, u, [n] * rows)
    token, lp = draw(x, u, temperature=heat)
    expect(token, lp, at, u, [n] * rows)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("vocab", [4097, 30011, 131072])
def test_a_row_alone_and_among_others(dtype, vocab):
    """The rows of a call are cut in parts by their number; the tokens are the same, also where the random
    number meets a sum."""
    g = torch.Generator().manual_seed(vocab)
    total = 150
    x = (torch.randn(total, vocab, generator=g) * 2.5).to(dtype)
    u = torch.rand(total, generator=g)
    half = torch.arange(total // 2)          # two equal tokens, at a half
    x[half] = float("-inf")
    value = (torch.randn(len(half), generator=g) * 6).to(dtype)
    first = torch.randint(0, 200, (len(half),), generator=g)
    second = first + torch.randint(1, vocab - 200, (len(half),), generator=g)
    x[half, first], x[half, second] = value, value
    u[half] = 0.5
    x, p = x.to(DEV), torch.full((total,), 0.97)
    for f in (dict(), dict(top_p=p)):
        token, lp = draw(x, u, **f)
        assert token[half].tolist() == second.tolist()
        assert bool((lp[half] == -torch.tensor(math.log(2.0))).all())
        for rows in (1, 3, 8, 40, 64):
            for r0 in range(0, total, rows if rows > 3 else 10):
                part = slice(r0, r0 + rows)
                few, few_lp = draw(x[part], u[part], **{n: v[part] for n, v in f.items()})
                assert torch.equal(few, token[part]), (rows, r0)
                assert torch.equal(few_lp, lp[part]), (rows, r0)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("have", [9, 60, 900, 4000])
def test_a_row_with_nothing_behind_it(dtype, have):
    """Tokens of -inf behind a row, so that another kernel takes it, change nothing."""
    g = torch.Generator().manual_seed(have)
    rows = 48
    x = (torch.randn(rows, have, generator=g) * 2.5).to(dtype)
    x[::3] = x[::3, :1]                       # rows of equal logits
    u, p = torch.rand(rows, generator=g), 0.25 * torch.randint(1, 4, (rows,), generator=g)
    k, m = torch.randint(2, have + 1, (rows,), generator=g).int(), 0.2 * torch.rand(rows, generator=g)
    u[::2] = (u[::2] * 16).floor() / 16
    heat = 0.4 + torch.rand(rows, generator=g)
    for f in (dict(), dict(top_p=p), dict(top_k=k, top_p=p), dict(temperature=heat, top_p=p, min_p=m)):
        token, lp = draw(x, u, **f)
        for vocab in (64, 65, 1000, 4096, 4097, 30011):
            if vocab < have:
                continue
            wide = torch.full((rows, vocab), float("-inf"), dtype=dtype)
            wide[:, :have] = x
            again, again_lp = draw(wide, u, **f)
            assert torch.equal(again, token), (vocab, f)
            assert torch.equal(again_lp, lp), (vocab, f)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("vocab", [4097, 30011, 131072])
def test_long_rows_with_values_that_are_not_finite(dtype, vocab):
    inf, nan = float("inf"), float("nan")
    g = torch.Generator().manual_seed(vocab)
    x = (torch.randn(12, vocab, generator=g) * 2.5).to(dtype)
    u = torch.rand(12, generator=g)
    last = vocab - 1
    x[0], x[1], x[2] = -inf, nan, -inf
    x[2, last] = -3e38
    x[3, ::2] = -inf
    x[4, ::3] = nan
    x[5, 7], x[5, last] = inf, inf            # of two parts, both parts' largest
    x[6] = -inf
    x[6, 5], x[6, last - 3] = nan, 0.25
    x[7, 4000] = 3e38
    x[8] = -inf
    x[8, 3], x[8, last] = 0.0, -0.0           # equal, whatever their sign
    x[9, :4090] = -inf                        # a part of nothing
    x[10, last] = inf
    x[11] = -inf
    x[11, [1, 4090, last]] = inf
    u[5], u[8], u[11] = 0.5, 0.5, 0.25
    token, lp = draw(x, u)
    assert token[0] == 0 and token[1] == 0 and lp[0] == -inf and lp[1] == -inf
    assert token[2] == last and token[6] == last - 3 and token[7] == 4000 and token[10] == last
    assert bool((lp[[2, 6, 7, 10]] == 0).all())
    assert token[5] == last and token[8] == last and token[11] == 1
    assert float(lp[11]) == pytest.approx(-math.log(3), abs=2.0 ** -23)
    keep = [3, 4, 9]
    check(x[keep], u[keep])
    check(x[keep], u[keep], top_k=torch.full((3,), 50).int(), top_p=torch.full((3,), 0.9))
    check(x[keep], u[keep], min_p=torch.full((3,), 0.05))
    token, lp = draw(x, u, top_p=[0.5] * 12)
    assert token[5] == 7 and lp[5] == 0 and token[8] == 3 and lp[8] == 0
    first = [0, 0] + [int(torch.where(torch.isnan(r), -inf, r.float()).argmax()) for r in x[2:]]
    for f in (dict(temperature=[0.0] * 12), dict(top_k=[1] * 12), dict(min_p=[1.5] * 12)):
        token, lp = draw(x, u, **f)
        assert token.tolist() == first and bool((lp[2:] == 0).all())


@pytest.mark.parametrize("vocab", [4097, 30011])
def test_long_rows_at_the_ends_of_the_random_numbers(vocab):
    x = torch.randn(6, vocab, generator=torch.Generator().manual_seed(1)) * 2.5
    x[:, 0], x[:, -1] = 8.0, 8.0
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, -1.0, float("nan"), 2.0])
    token, _ = draw(x, u)
    assert token.tolist() == [0, vocab - 1, vocab - 1, 0, 0, vocab - 1]


@pytest.mark.parametrize("rows,vocab", [(2 ** 22 + 5, 65), (2 ** 26 + 9, 2)])
def test_more_rows_than_a_launch_takes(rows, vocab):
    """2^32 threads and more, a grid's limit: a block of 1,024 a row, a wave of 64 a row."""
    x = torch.zeros(rows, vocab, dtype=BF, device=DEV)
    want = torch.arange(rows, device=DEV) * 40503 % vocab
    x.scatter_(1, want[:, None], 50.0)
    token = torch.full((rows,), -5, dtype=torch.int64, device=DEV)
    u = torch.full((rows,), 0.5, device=DEV)
    K().sample_tokens(x, u, token, top_p=u)
    assert torch.equal(token, want)


def test_more_parts_than_a_launch_takes():
    """Rows above 4,096 tokens, a block of 1,024 threads for each part of them."""
    rows, vocab = 2 ** 22 + 3, 4104
    if torch.cuda.mem_get_info()[0] < 100 * 2 ** 30:
        pytest.skip("needs 100 GB of free memory")
    row = torch.zeros(1, vocab, dtype=BF, device=DEV)
    row[0, 4100] = 50.0
    x = row.expand(rows, vocab).contiguous()
    x[-2:, 4100], x[-2:, 7] = 0.0, 50.0
    token = torch.full((rows,), -5, dtype=torch.int64, device=DEV)
    K().sample_tokens(x, torch.full((rows,), 0.5, device=DEV), token)
    assert bool((token[:-2] == 4100).all()) and bool((token[-2:] == 7).all())
