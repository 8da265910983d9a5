"""K11 on the GPU where a filter's border meets a sum of weights exactly.

Equal logits have equal weights, so n of them (the rest -inf) have the sums j / n of all, whatever their
value: the expected tokens follow in whole numbers, and no tolerance is needed for them.  logprob is
-ln of the kept tokens' number: fp32's half step of the log, and 2^-50 for the quotient of two sums
that are n and 1 times the same weight."""

import math

import pytest
import torch

from .test_gpu_sample import BF, F32, draw

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
