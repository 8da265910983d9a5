"""K11 on the GPU (sampling with temperature, top-k, top-p and min-p at given random numbers) against
the definition in 64 bits on the CPU.

Tokens have to be equal wherever the random number lies further from a border of the sums than what
the sums can be off: weights to 2^-45 of the largest each, at most 2^20 of them of which a row's sum is
at least one, and 64-bit arithmetic: below 1e-7 for the sizes here.  The filters' borders are exact but
for such sums, and no input here lies nearer.  logprob: fp32's half step of the log, and 1e-6 for the
sums."""

import math

import pytest
import torch

from .paged_ref import sampled

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
NEAR = 1e-7


def K():
    from mdlarc_scale_amd import kernels

    return kernels


def draw(x, u, logprob=True, **filters):
    """token and logprob of the kernel; filters by name, a number a row."""
    rows = x.shape[0]
    token = torch.full((rows,), -5, dtype=torch.int64, device=DEV)
    lp = torch.full((rows,), 9.0, device=DEV) if logprob else None
    kinds = dict(temperature=F32, top_k=torch.int32, top_p=F32, min_p=F32)
    args = {n: torch.tensor(v, dtype=kinds[n], device=DEV) if not torch.is_tensor(v)
            else v.to(DEV) for n, v in filters.items()}
    K().sample_tokens(x.to(DEV) if not x.is_cuda else x, u.to(DEV), token, logprob_out=lp, **args)
    torch.cuda.synchronize()
    return token.cpu(), None if lp is None else lp.cpu()


def check(x, u, **filters):
    token, lp = draw(x, u, **filters)
    names = list(filters)
    for r in range(x.shape[0]):
        f = {}
        for n in names:
            t = torch.as_tensor(filters[n])[r]
            f[n] = int(t) if n == "top_k" else float(t.float())
        want, share, near = sampled(x[r].float(), float(u[r]), **f)
        if near > NEAR:
            assert int(token[r]) == want, (r, f, int(token[r]), want, near)
            if share == float("-inf"):
                assert lp[r] == share
            else:
                assert abs(float(lp[r]) - share) <= 1e-6 + 2.0 ** -24 * abs(share), (r, f)
        else:
            assert 0 <= int(token[r]) < x.shape[1]


def rows_of(seed, rows, vocab, dtype, std=2.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=g) * std).to(dtype)
    return x, torch.rand(rows, generator=g), g


VOCABS = [1, 2, 14, 63, 64, 65, 100, 1000, 1023, 4099, 32003, 131072]


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("vocab", VOCABS)
def test_filters(dtype, vocab):
    rows = 24
    x, u, g = rows_of(vocab, rows, vocab, dtype)
    check(x, u)
    heat = 0.3 + torch.rand(rows, generator=g)
    k = torch.randint(1, min(vocab, 900) + 1, (rows,), generator=g).int()
    p, m = 0.2 + 0.79 * torch.rand(rows, generator=g), 0.1 * torch.rand(rows, generator=g)
    check(x, u, temperature=heat)
    check(x, u, top_k=k)
    check(x, u, top_p=p)
    check(x, u, min_p=m)
    check(x, u, temperature=heat, top_k=k, top_p=p, min_p=m)
    check(x, u, temperature=heat, top_k=k, top_p=p)
    check(x, u, top_k=k, min_p=5 * m)
    check(x, u, top_p=p, min_p=5 * m)
    # each filter off in some rows
    k[::3], p[1::3], m[2::3], heat[5::7] = 0, 1.0, 0.0, 0.0
    check(x, u, temperature=heat, top_k=k, top_p=p, min_p=m)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("vocab", [14, 5000, 70001])
@pytest.mark.parametrize("values", [1, 2, 5])
def test_many_equal_logits(dtype, vocab, values):
    """Borders inside thousands of equal logits: the lowest indexes are kept."""
    g = torch.Generator().manual_seed(vocab + values)
    rows = 12
    x = (torch.randint(0, values, (rows, vocab), generator=g).float() * 0.7).to(dtype)
    u = torch.rand(rows, generator=g)
    k = torch.randint(2, vocab + 3, (rows,), generator=g).int()
    p = 0.05 + 0.9 * torch.rand(rows, generator=g)
    check(x, u, top_k=k)
    check(x, u, top_p=p)
    check(x, u, top_k=k, top_p=p)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("vocab", [300, 1025, 2500, 4096, 4097, 30011])
@pytest.mark.parametrize("std", [0.0, 1e-4, 0.01, 0.3])
def test_borders_among_close_logits(dtype, vocab, std):
    """Thousands of tokens within a hundredth of an octave, or equal, in rows of every kind."""
    rows = 10
    x, u, g = rows_of(vocab + int(1e4 * std), rows, vocab, dtype, std=std)
    k = torch.randint(2, vocab + 1, (rows,), generator=g).int()
    p, m = 0.05 + 0.9 * torch.rand(rows, generator=g), 0.5 + 0.5 * torch.rand(rows, generator=g)
    check(x, u, top_k=k)
    check(x, u, top_p=p)
    check(x, u, min_p=m)
    check(x, u, top_k=k, top_p=p)
    check(x - 50, u, top_k=k, top_p=p, min_p=m)


@pytest.mark.parametrize("vocab", [500, 4096, 30011])
def test_shares_next_to_one_and_weights_below_the_sums(vocab):
    """Low temperatures leave most weights below 2^-43; top-p and min-p among them."""
    rows = 16
    x, u, g = rows_of(vocab + 3, rows, vocab, F32)
    heat = 0.02 + 0.2 * torch.rand(rows, generator=g)
    p = 1 - 2.0 ** -torch.randint(10, 25, (rows,), generator=g).float()
    m = 2.0 ** -(60 * torch.rand(rows, generator=g))
    check(x, u, temperature=heat, top_p=p)
    check(x, u, temperature=heat, min_p=m)
    check(x, u, temperature=heat, top_p=p, min_p=m)
    check(x, u, temperature=heat, top_p=p, top_k=torch.full((rows,), vocab - 1, dtype=torch.int32))


@pytest.mark.parametrize("vocab", [14, 64, 65, 3001])
def test_masked_rows_and_values_that_are_not_finite(vocab):
    inf, nan = float("inf"), float("nan")
    x, u, _ = rows_of(3, 9, vocab, F32)
    x[0] = -inf
    x[1] = nan
    x[2, :] = -inf
    x[2, vocab - 1] = -3e38
    x[3, ::2] = -inf
    x[4, ::3] = nan
    x[5, 7], x[5, 9] = inf, inf
    x[6] = -inf
    x[6, 5], x[6, 6] = nan, 0.25
    x[7, 3] = 3e38
    x[8, 4], x[8, 6] = -0.0, 0.0
    x[8, :4] = -9.0
    token, lp = draw(x, u)
    assert token[0] == 0 and token[1] == 0 and lp[0] == -inf and lp[1] == -inf
    assert token[2] == vocab - 1 and lp[2] == 0
    assert token[5] in (7, 9) and abs(float(lp[5]) + math.log(2)) < 1e-6
    assert token[6] == 6 and lp[6] == 0 and token[7] == 3
    keep = [3, 4, 8]
    check(x[keep], u[keep])
    check(x[keep], u[keep], top_k=torch.full((3,), 5).int(), top_p=torch.full((3,), 0.9))
    # greedy: the first of equal ones, through every way of asking for it
    for f in (dict(temperature=[0.0] * 9), dict(temperature=[-1.0] * 9), dict(top_k=[1] * 9),
              dict(temperature=[nan] * 9), dict(top_p=[0.0] * 9), dict(min_p=[1.5] * 9)):
        token, lp = draw(x, u, **f)
        assert token.tolist() == [0, 0] + [int(torch.where(torch.isnan(r), -inf, r).argmax())
                                           for r in x[2:]]
        assert bool((lp[2:] == 0).all())


def test_the_longest_rows():
    vocab, rows = 2 ** 20, 3
    x, u, g = rows_of(77, rows, vocab, BF)
    p, m = 0.3 + 0.6 * torch.rand(rows, generator=g), 0.01 * torch.rand(rows, generator=g)
    k = torch.randint(2000, 9000, (rows,), generator=g).int()
    check(x, u)
    check(x, u, top_p=p)
    check(x, u, top_k=k, top_p=p)
    check(x, u, top_p=p, min_p=m)


@pytest.mark.parametrize("rows,vocab", [(70001, 14), (70001, 65), (5003, 4100)])
def test_many_rows(rows, vocab):
    """Copies of four rows, whose tokens are checked."""
    x, u, g = rows_of(5, 4, vocab, F32)
    p, m = 0.3 + 0.6 * torch.rand(4, generator=g), 0.05 * torch.rand(4, generator=g)
    check(x, u, top_p=p, min_p=m)
    few, few_lp = draw(x, u, top_p=p, min_p=m)
    i = torch.arange(rows) % 4
    token, lp = draw(x.to(DEV)[i.to(DEV)], u[i], top_p=p[i], min_p=m[i])
    assert torch.equal(token, few[i]) and torch.equal(lp, few_lp[i])


@pytest.mark.parametrize("vocab", [14, 900, 30011])
def test_filters_that_are_none(vocab):
    """Numbers that switch a filter off, NaN among them, and a workspace of the caller's."""
    nan, inf = float("nan"), float("inf")
    x, u, _ = rows_of(vocab, 4, vocab, F32)
    plain, lp = draw(x, u)
    for f in (dict(top_k=[0, -1, -2 ** 31, vocab]), dict(top_p=[1.0, 7.0, inf, nan]),
              dict(min_p=[0.0, -1.0, -inf, nan]), dict(top_k=[2 ** 31 - 1] * 4)):
        token, lp2 = draw(x, u, **f)
        assert torch.equal(token, plain) and torch.equal(lp, lp2), f
    token = torch.zeros(4, dtype=torch.int64, device=DEV)
    ws = torch.empty(K().sample_workspace_bytes(4, vocab), dtype=torch.uint8, device=DEV)
    K().sample_tokens(x.to(DEV), u.to(DEV), token, workspace=ws)
    assert torch.equal(token.cpu(), plain)
    if vocab > 4096:
        with pytest.raises(RuntimeError, match="workspace"):
            K().sample_tokens(x.to(DEV), u.to(DEV), token, workspace=ws[:-8])


@pytest.mark.parametrize("vocab", [14, 900])
def test_random_numbers_at_the_ends(vocab):
    x, _, _ = rows_of(8, 6, vocab, F32)
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, -1.0, float("nan"), 2.0])
    token, _ = draw(x, u)
    assert token.tolist() == [0, vocab - 1, vocab - 1, 0, 0, vocab - 1]
    token, _ = draw(x, u, temperature=[1e-38, 1e-45, 0.01, 3e38, float("inf"), 1.0])
    assert token[:2].tolist() == [int(r.argmax()) for r in x[:2]] and token[3] == 0


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("vocab,ld,skip", [(1001, 1004, 1), (9, 11, 1), (70, 77, 5), (5003, 5003, 0)])
def test_strided_and_odd_rows(dtype, vocab, ld, skip):
    wide, u, _ = rows_of(5, 33, ld + 8, dtype)
    wide = wide.to(DEV)[:, :ld].contiguous()
    x = wide[:, skip:skip + vocab] if skip + vocab <= ld else wide[:, :vocab]
    p = torch.full((33,), 0.9)
    token, _ = draw(x, u, top_p=p)
    again, _ = draw(x.contiguous(), u, top_p=p)
    assert torch.equal(token, again)
    for r in range(33):
        want, _, near = sampled(x[r].float().cpu(), float(u[r]), top_p=float(p[r]))
        assert near <= NEAR or int(token[r]) == want


def test_frequencies_follow_the_shares():
    """One row many times, at evenly spread numbers: each token as often as its share says."""
    g = torch.Generator().manual_seed(1)
    row = torch.randn(300, generator=g) * 2
    n = 4096
    u = (torch.arange(n) + 0.5) / n
    token, _ = draw(row.expand(n, 300).contiguous(), u)
    share = torch.softmax(row.double(), 0)
    count = torch.bincount(token, minlength=300).double()
    assert bool(((count - n * share).abs() <= 1 + 1e-6).all())


@pytest.mark.parametrize("vocab", [14, 2000, 9000])
def test_graph_streams_and_no_logprob(vocab):
    """Captured calls (a long row's takes its workspace from the capture's pool) replayed with other
    data between eager calls, two of them side by side."""
    x, u, _ = rows_of(9, 40, vocab, F32)
    xd, ud = x.to(DEV), u.to(DEV)
    token, p = torch.zeros(40, dtype=torch.int64, device=DEV), torch.full((40,), 0.7, device=DEV)
    call = lambda: K().sample_tokens(xd, ud, token, top_p=p)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    other, u3, _ = rows_of(10, 40, vocab, F32)
    other, u3, token3 = other.to(DEV), u3.to(DEV), torch.zeros_like(token)
    graph3 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph3):
        K().sample_tokens(other, u3, token3, top_p=p)
    want3, _ = draw(other, u3, logprob=False, top_p=p)
    for step in range(3):
        x2, u2, _ = rows_of(50 + step, 40, vocab, F32)
        xd.copy_(x2)
        ud.copy_(u2)
        token.fill_(-1)
        token3.fill_(-1)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            graph3.replay()
        torch.cuda.synchronize()
        want, _ = draw(x2, u2, logprob=False, top_p=p)
        assert torch.equal(token.cpu(), want) and torch.equal(token3.cpu(), want3)
    K().sample_tokens(xd[:0], ud[:0], token[:0])
