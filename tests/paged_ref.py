"""Plain forms of paged caches and of sampling for the tests: 4-bit pages, pools, the order of tokens.
CPU, float64."""

import math

import torch

BF, F32 = torch.bfloat16, torch.float32
E2M1 = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def power_of(x):
    """The power of two of each 32 channels of x [.., D]: the smallest 2^k, -100 <= k <= 125, by which
    all magnitudes are below 7."""
    top = x.double().abs().unflatten(-1, (-1, 32)).amax(-1)
    k = torch.full(top.shape, -100, dtype=torch.int64)
    for n in range(-100, 125):
        k = torch.where(top >= 7.0 * 2.0 ** n, n + 1, k)
    return k


def to_fp4(x):
    """Codes uint8 [.., D / 2] and powers uint8 [.., D / 32] of x [.., D] (fp32 or wider)."""
    finite = torch.isfinite(x).unflatten(-1, (-1, 32)).all(-1)
    x = torch.where(finite[..., None], x.double().unflatten(-1, (-1, 32)), 0.0)
    k = power_of(x.flatten(-2))
    v = x.abs() * torch.pow(torch.tensor(2.0, dtype=torch.float64), -k)[..., None]
    # the nearest number, of two as near the one with the even code
    far = (v[..., None] - E2M1).abs()
    code = torch.where(far == far.amin(-1, keepdim=True),
                       torch.tensor([0, 9, 2, 11, 4, 13, 6, 15]), 99).amin(-1) % 8
    code = (code + 8 * torch.signbit(x)).flatten(-2).to(torch.uint8)
    scale = torch.where(finite, k + 127, 255).to(torch.uint8)
    return code[..., 0::2] | code[..., 1::2] << 4, scale


def from_fp4(codes, scale):
    """float64 [.., D]; NaN where a power is 255."""
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    value = E2M1[code & 7] * (1 - 2 * (code >> 3)).double()
    power = torch.pow(torch.tensor(2.0, dtype=torch.float64), scale.double() - 127)
    power = torch.where(scale == 255, float("nan"), power)
    return (value.unflatten(-1, (-1, 32)) * power[..., None]).flatten(-2)


def page_table(counts, width, n_pages, g):
    """Each sequence's first counts[s] pages anywhere in a pool, the entries behind them -1."""
    order = torch.randperm(n_pages, generator=g)[:sum(counts)].int()
    table = torch.full((len(counts), width), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(counts):
        table[s, :n] = order[at:at + n]
        at += n
    return table


def to_pool(rows, table, n_pages, page, fill):
    """rows [n_seq, kv, slots, ..] in a pool [n_pages, kv, page, ..]; the rest is `fill`."""
    pool = torch.full((n_pages, rows.shape[1], page, *rows.shape[3:]), fill, dtype=rows.dtype)
    for s in range(rows.shape[0]):
        for i in range(-(-rows.shape[2] // page)):
            if i < table.shape[1] and table[s, i] >= 0:
                part = rows[s, :, i * page:(i + 1) * page]
                pool[table[s, i], :, :part.shape[1]] = part
    return pool


# ---- sampling ----------------------------------------------------------------------------------

def kept_tokens(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Tokens that the filters leave, in the order of tokens, and their weights (largest 1)."""
    x = torch.where(torch.isnan(x), float("-inf"), x.double())
    order = torch.sort(x, descending=True, stable=True).indices
    if x[order[0]] == float("-inf"):
        return order[:1], torch.zeros(1, dtype=torch.float64)
    if not temperature > 0 or top_k == 1 or top_p <= 0 or min_p > 1:
        return order[:1], torch.ones(1, dtype=torch.float64)
    z = (x[order] - x[order[0]]) / temperature
    z[x[order] == x[order[0]]] = 0.0
    w = torch.exp(z)
    n = min(top_k, len(w)) if top_k > 0 else len(w)
    order, w = order[:n], w[:n]
    if top_p < 1:
        n = max(1, int((w.cumsum(0) - w < top_p * w.sum()).sum()))
        order, w = order[:n], w[:n]
    keep = w >= min_p
    return order[keep], w[keep]


def sampled(x, u, **filters):
    """Token, log of its share, and how near u is to a border of the sums (of all: 1)."""
    order, w = kept_tokens(x, **filters)
    if w.sum() == 0:
        return 0, float("-inf"), 1.0
    by_index = order.argsort()
    order, w = order[by_index], w[by_index] / w.sum()
    sums = w.cumsum(0)
    at = min(int((sums <= u * sums[-1]).sum()), len(w) - 1)
    edges = (sums / sums[-1] - u).abs()[:-1]
    return int(order[at]), math.log(float(w[at])), float(edges.min()) if len(edges) else 1.0
