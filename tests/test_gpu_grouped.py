"""K7 and K8 on the GPU (per-head norms with the rotation, attention with grouped key / value heads,
decode attention of rows that share a prefix) through mdlarc_scale_amd.kernels, against plain
implementations in 64 bits on the CPU.

Tolerances are bounds on what the roundings can add, element by element.  With w the softmax weights
and A = sum_j w_j |v_j|:
  * a score is off by at most ds = 2 D 2^-23 max_j sum_d |q_d k_jd| (D fp32 additions, partial sums
    that also hold the reference maximum), a weight by a factor 1 +- ln 2 ds 2, numerator and
    denominator together twice that;
  * bf16 rounds each weight by at most 2^-8 relative, in the numerator and in the sum: 2 2^-8 A;
  * the sums of n terms, their rescales and merges and v_exp_f32 add at most (n + 64) 2^-23 A;
  * the result is rounded once, by 2^-8 (bf16) or 2^-24 (fp32) relative.
"""

import math

import pytest
import torch

from mdlarc_scale_amd.transformer import LOG2E, RotaryEmbedding3D

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
HALF_STEP = {BF: 2.0 ** -8, F32: 2.0 ** -24}


def K():
    from mdlarc_scale_amd import kernels

    return kernels


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rand(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g) * std


# ---- references --------------------------------------------------------------------------------

def _attend(q, k, v, limit):
    """q [rows, D], k / v [keys, D], row r sees keys < limit[r] (a list): outputs and bounds'
    ingredients, all in float64."""
    q, k, v = q.double(), k.double(), v.double()
    out = torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64)
    mass, ds = torch.zeros_like(out), torch.zeros(q.shape[0], 1, dtype=torch.float64)
    for r, n in enumerate(limit):
        if n <= 0:
            continue
        s = k[:n] @ q[r]
        w = torch.exp2(s - s.max())
        w = w / w.sum()
        out[r], mass[r] = w @ v[:n], w @ v[:n].abs()
        ds[r] = 2 * q.shape[1] * 2.0 ** -23 * (k[:n].abs() @ q[r].abs()).max()
    return out, mass, ds


def _bound(ref, mass, ds, n, dtype, half_step=None):
    rounding = HALF_STEP[dtype] if half_step is None else half_step
    weights = 2 * HALF_STEP[BF] if dtype == BF else 0.0
    return (rounding * ref.abs() +
            (weights + 4 * math.log(2.0) * ds + (n + 64) * 2.0 ** -23) * mass * (1 + rounding) +
            1e-30)


def _check(got, ref, bound, what=""):
    got = got.double().cpu()
    assert not torch.isnan(got).any(), f"{what}: NaN"
    ratio = (got - ref).abs() / bound
    assert bool((ratio <= 1).all()), f"{what}: {ratio.max().item():.2f} of the bound"


class Grouped:
    """A packed batch: n queries and `past` cached keys of each sequence, `tail` rows of no
    sequence."""

    def __init__(self, seed, dtype, D, heads, kv, n, past, tail=0, spare=9, std=1.0):
        g = _gen(seed)
        self.n, self.keys = n, [a + b for a, b in zip(n, past)]
        self.tokens = sum(n) + tail
        self.D, self.heads, self.kv, self.dtype = D, heads, kv, dtype
        self.offset = [sum(n[:i]) for i in range(len(n) + 1)]
        slots = max(self.keys) + spare
        self.q = _rand(g, self.tokens, heads, D, std=std * LOG2E / math.sqrt(D)).to(dtype)
        self.k = _rand(g, len(n), kv, slots, D, std=std).to(dtype)
        self.v = _rand(g, len(n), kv, slots, D).to(dtype)

    def reference(self, causal=True, keys=None):
        """Outputs and bound of every row of a sequence ([tokens, heads, D]; NaN elsewhere)."""
        ref = torch.full((self.tokens, self.heads, self.D), float("nan"), dtype=torch.float64)
        bound = torch.zeros_like(ref)
        r = self.heads // self.kv
        for b, n in enumerate(self.n):
            total = self.keys[b] if keys is None else keys[b]
            limit = [total - n + i + 1 if causal else total for i in range(n)]
            a = self.offset[b]
            for h in range(self.heads):
                o, mass, ds = _attend(self.q[a:a + n, h], self.k[b, h // r], self.v[b, h // r],
                                      limit)
                ref[a:a + n, h] = o
                bound[a:a + n, h] = _bound(o, mass, ds, total, self.dtype)
        return ref, bound

    def run(self, causal=True, keys=None, workspace=True, max_q=None, out=None, **form):
        kern = K()
        q, k, v = self.q.to(DEV), self.k.to(DEV), self.v.to(DEV)
        max_q = max(self.n) if max_q is None else max_q
        ws = None
        if workspace:
            ws = torch.full((kern.attn_grouped_workspace_bytes(q, k, max_q) // 4,), float("nan"),
                            device=DEV)
        if out is None:
            out = torch.full_like(q, 7.0)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
        kern.attn_grouped(q, k, v, i32(self.offset), i32(self.keys if keys is None else keys),
                          max_q, out, causal=causal, workspace=ws, **form)
        torch.cuda.synchronize()
        return out

    def check(self, what, causal=True, keys=None, **kw):
        ref, bound = self.reference(causal, keys)
        out = self.run(causal, keys, **kw)
        end = self.offset[-1]
        _check(out[:end], ref[:end], bound[:end], what)
        assert bool((out[end:] == 7.0).all()), f"{what}: rows of no sequence were written"


# ---- K8: packed sequences ----------------------------------------------------------------------

SHAPES = [(BF, 64, 12, 12), (BF, 64, 12, 4), (BF, 128, 5, 1), (BF, 128, 16, 2), (F32, 64, 6, 3),
          (F32, 128, 4, 2), (F32, 64, 16, 1)]
BATCHES = {
    "one": ([1], [0]),
    "one_of_many_keys": ([1, 1, 1], [0, 31, 700]),
    "edges": ([31, 32, 33, 63, 64, 65], [0, 0, 0, 0, 0, 0]),
    "ragged": ([7, 0, 1, 129, 0, 200], [0, 5, 127, 33, 0, 3]),
    "chunk": ([5, 40], [513, 70]),
}


@pytest.mark.parametrize("dtype,D,heads,kv", SHAPES)
@pytest.mark.parametrize("batch", BATCHES)
def test_grouped(dtype, D, heads, kv, batch):
    n, past = BATCHES[batch]
    c = Grouped(len(batch) + D + heads, dtype, D, heads, kv, n, past, tail=3)
    c.check("causal")
    c.check("whole", causal=False)


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (F32, 64), (F32, 128)])
def test_grouped_tall_blocks(dtype, D):
    """Enough rows for the launch of 128-row blocks, with a last tile that is not full."""
    c = Grouped(3, dtype, D, 16, 16, [150, 300, 77, 5, 290, 33, 128, 257], [0] * 8, tail=2)
    c.check("tall")
    c.check("tall, whole", causal=False)


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (F32, 64), (F32, 128)])
def test_grouped_tall_blocks_in_parts(dtype, D):
    """A few hundred rows behind thousands of keys."""
    c = Grouped(13, dtype, D, 8, 2, [40, 17, 0, 3], [3000, 2950, 2000, 1], tail=1)
    assert K().attn_grouped_workspace_bytes(c.q.to(DEV), c.k.to(DEV), 40) > 0
    c.check("parts")
    c.check("no workspace", workspace=False)


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (F32, 64), (F32, 128)])
def test_grouped_many_heads_to_one(dtype, D):
    """More query heads to a key / value head than rows in a tile, and a number that divides none."""
    c = Grouped(14, dtype, D, 161, 1, [3, 2], [40, 0], tail=1)
    c.check("161 heads")
    c.check("161 heads, no workspace", workspace=False)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_grouped_parts_and_no_workspace(dtype):
    """Few rows and many keys: cut into parts with a workspace, whole without, equal calls equal."""
    c = Grouped(4, dtype, 64, 8, 2, [3, 1], [2100, 1030], tail=1)
    assert K().attn_grouped_workspace_bytes(c.q.to(DEV), c.k.to(DEV), 3) > 0
    c.check("parts")
    c.check("no workspace", workspace=False)
    assert torch.equal(c.run(), c.run())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("workspace", [True, False])
def test_grouped_rows_that_see_nothing(dtype, workspace):
    """Fewer keys than queries, and none: zeros there."""
    c = Grouped(5, dtype, 64, 4, 2, [40, 3, 70, 1], [0, 0, 0, 0])
    keys = [10, 0, 69, 0]
    c.check("causal", keys=keys, workspace=workspace)
    c.check("whole", causal=False, keys=keys, workspace=workspace)
    out = c.run(keys=keys, workspace=workspace)
    assert bool((out[:30] == 0).all()) and bool((out[40:43] == 0).all())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_grouped_large_scores(dtype):
    """Scores of some hundreds: weights underflow, the reference maximum moves often."""
    c = Grouped(6, dtype, 128, 4, 2, [90, 33], [50, 0], std=9.0)
    c.check("large")


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("workspace", [True, False])
def test_grouped_values_that_are_not_finite(dtype, D, bad, workspace):
    """Values behind the keys, and in slots that only later queries see, reach nobody else."""
    c = Grouped(7, dtype, D, 6, 2, [70, 45], [0, 20])
    ref, bound = c.reference()
    at = 50                                     # slot of query 50 of sequence 0, 30 of sequence 1
    for t in (c.k, c.v):
        for b, n in enumerate(c.keys):
            t[b, :, n:] = bad
    c.v[:, 0, at, 3] = bad                      # one channel of a value
    c.k[:, 1, at] = float("nan")                # a whole key
    out = c.run(workspace=workspace).double().cpu()
    lo0, lo1 = 50, 70 + 30                      # the first rows that see the slot
    hit = torch.zeros(c.offset[-1], dtype=torch.bool)
    hit[lo0:70] = True
    hit[lo1:] = True
    _check(out[~hit], ref[~hit], bound[~hit], "rows before")
    _check(out[hit][:, :3, :3], ref[hit][:, :3, :3], bound[hit][:, :3, :3], "other channels")
    _check(out[hit][:, :3, 4:], ref[hit][:, :3, 4:], bound[hit][:, :3, 4:], "other channels")
    got = out[hit][:, :3, 3]
    assert bool(torch.isnan(got).all() if math.isnan(bad) else (got == bad).all())
    assert bool(torch.isnan(out[hit][:, 3:]).all())


def test_grouped_too_many_queries_stay():
    """Queries past max_q are not computed, in either launch form."""
    c = Grouped(8, BF, 64, 4, 2, [40, 9], [0, 300])
    ref, bound = c.reference()
    for workspace in (True, False):
        out = c.run(max_q=9, workspace=workspace)
        _check(out[:9], ref[:9], bound[:9], "first rows")
        _check(out[40:], ref[40:], bound[40:], "second sequence")
        assert bool((out[9:40] == 7.0).all())


@pytest.mark.parametrize("max_q", [2 ** 31, 2 ** 32, 2 ** 32 + 1])
def test_grouped_bound_above_the_rows(max_q):
    Grouped(61, BF, 64, 4, 2, [3, 40, 1], [900, 0, 1500], tail=2).check("bound", max_q=max_q)


@pytest.mark.parametrize("max_q", [-1, -2 ** 32, -2 ** 32 + 5])
def test_grouped_bound_below_zero_is_refused(max_q):
    with pytest.raises((RuntimeError, ValueError)):
        Grouped(62, BF, 64, 4, 2, [3], [9]).run(max_q=max_q)


def test_grouped_lengths_out_of_range_are_clamped():
    c = Grouped(9, F32, 64, 4, 2, [5, 6], [10, 0])
    slots = c.k.shape[2]
    c.offset = [-3, 5, 99]
    out = c.run(keys=[slots + 50, -4], max_q=8)
    c.offset, c.n = [0, 5, 11], [5, 6]
    ref, bound = c.reference(keys=[slots, 0])
    _check(out, ref, bound, "clamped")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("tiled", [False, True])
@pytest.mark.parametrize("past", [0, 2200])
def test_grouped_split_output(dtype, tiled, past):
    """The split output carries the value to 2^-16: hi + lo against the plain one's arithmetic."""
    c = Grouped(10, dtype, 64, 4, 2, [3, 18], [past, past], tail=2)
    ref, bound = c.reference()
    width, rows = c.heads * c.D, c.tokens
    pad = -(-rows // 16) * 16 if tiled else rows
    out = torch.full((pad, 2 * width), 3.0, dtype=BF, device=DEV)
    got = c.run(out=out, split=True, tiled=tiled).float().cpu()
    if tiled:
        got = K().untile_matrix(out, rows, 2 * width).float().cpu()
    got = got[:rows]
    value = (got[:, :width] + got[:, width:]).view(rows, c.heads, c.D)
    end = c.offset[-1]
    # hi + lo is within 2^-8 2^-8 of the fp32 value
    extra = 2.0 ** -16 * ref.abs() - (HALF_STEP[BF] * ref.abs() if dtype == BF else 0)
    _check(value[:end], ref[:end], (bound + extra)[:end], "split")
    assert bool((got[end:] == 3.0).all())


def test_grouped_far_offsets():
    """K and V of more than 2^31 elements, and a head whose slots pass 2^31 bytes."""
    D, kv, slots = 128, 2, 4_200_000
    k = torch.empty(2, kv, slots, D, dtype=BF, device=DEV)
    v = torch.empty(2, kv, slots, D, dtype=BF, device=DEV)
    assert k.numel() > 2 ** 31
    c = Grouped(11, BF, D, 4, kv, [3, 5], [60, 80])
    n = c.k.shape[2]
    k[:, :, :n], v[:, :, :n] = c.k.to(DEV), c.v.to(DEV)
    q, out = c.q.to(DEV), torch.zeros_like(c.q, device=DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    K().attn_grouped(q, k, v, i32(c.offset), i32(c.keys), 5, out)
    ref, bound = c.reference()
    _check(out, ref, bound, "far rows")
    # one query over every slot of the last head: all keys equal, so the mean of the values
    k[1, 1], v[1, 1] = 0, 0
    v[1, 1, -4096:] = 1
    q1 = q[:1, 2:].contiguous()
    out1 = torch.zeros_like(q1)
    ws = torch.empty(K().attn_grouped_workspace_bytes(q1, k[1:, 1:], 1) // 4, device=DEV)
    K().attn_grouped(q1, k[1:, 1:], v[1:, 1:], i32([0, 1]), i32([slots]), 1, out1, workspace=ws)
    want = torch.full_like(out1, 4096 / slots, dtype=torch.float64).cpu()
    # sums of equal weights: 4.2 million of them, in fp32 and in the parts' order
    _check(out1, want, want * (2.0 ** -8 + 2.0 ** -10), "every slot")


def test_grouped_graph_and_streams():
    """Captured once, replayed with other data and lengths between eager work; another stream."""
    kern = K()
    c = Grouped(12, BF, 64, 8, 2, [3, 40, 1], [900, 0, 1500], tail=2)
    q, k, v = c.q.to(DEV), c.k.to(DEV), c.v.to(DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    off, lens, out = i32(c.offset), i32(c.keys), torch.full_like(q, 7.0)
    ws = torch.empty(kern.attn_grouped_workspace_bytes(q, k, 40) // 4, device=DEV)
    args = (q, k, v, off, lens, 40, out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kern.attn_grouped(*args, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    ref, bound = c.reference()
    _check(out[:44], ref[:44], bound[:44], "other stream")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kern.attn_grouped(*args, workspace=ws)
    for keys in ([903, 40, 1501], [3, 25, 700], [0, 40, 1]):
        lens.copy_(i32(keys))
        q.copy_(torch.randn_like(q) * 0.2)
        out.fill_(7.0)
        want = torch.full_like(out, 7.0)
        kern.attn_grouped(q, k, v, off, lens, 40, want, workspace=torch.empty_like(ws))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        torch.randn(1000, device=DEV).sum().item()


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("batch", ["flat", "tall"])
def test_grouped_one_buffer_for_keys_and_values(dtype, D, batch):
    """Keys that are the values too (one cache given for both), in either block form."""
    if batch == "flat":
        c = Grouped(71, dtype, D, 6, 2, [33, 1, 9], [40, 300, 0], tail=1)
    else:
        c = Grouped(72, dtype, D, 16, 16, [150, 300, 77, 5, 290, 33, 128, 257], [0] * 8)
    c.v = c.k
    ref, bound = c.reference()
    kern = K()
    q, cache, out = c.q.to(DEV), c.k.to(DEV), torch.full_like(c.q, 7.0, device=DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    kern.attn_grouped(q, cache, cache, i32(c.offset), i32(c.keys), max(c.n), out)
    end = c.offset[-1]
    _check(out[:end], ref[:end], bound[:end], batch)


FAINT = {"flat": (2, 3, 90), "tall": (90, 300, 300), "parts": (1, 1, 2300),
         "tall parts": (1, 140, 2300)}


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("form", FAINT)
@pytest.mark.parametrize("heavy", ["first", "last"])
def test_grouped_keeps_fp32_weights_below_the_normal_range(form, D, heavy):
    """A weight of 2^-130 is a denormal fp32 number, and counts: times a value of 2^100 it is 2^-30.
    The key of weight 1 comes before the others (their weights are formed so) or behind them (their
    sum is rescaled, or joined, by 2^-130)."""
    seqs, n, slots = FAINT[form]
    q = torch.zeros(seqs * n, 1, D, device=DEV)
    q[..., 0] = 1.0                                   # the score is the key's first channel
    kc, vc = torch.zeros(2, seqs, 1, slots, D, device=DEV).unbind()
    kc[..., 0], vc[..., 5] = -130.0, 2.0 ** 100
    one = 0 if heavy == "first" else slots - 1
    kc[:, :, one, 0], vc[:, :, one, 5] = 0.0, 0.0
    out = torch.full_like(q, 7.0)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    ws = torch.empty(K().attn_grouped_workspace_bytes(q, kc, n) // 4, device=DEV)
    assert (ws.numel() > 0) == ("parts" in form)
    K().attn_grouped(q, kc, vc, i32([n * s for s in range(seqs + 1)]), i32([slots] * seqs), n, out,
                     causal=False, workspace=ws)
    # whole numbers of 2^-30, and a sum of weights that rounds to 1
    assert bool((out[..., 5] == (slots - 1) * 2.0 ** -30).all())
    assert bool((out[..., :5] == 0).all()) and bool((out[..., 6:] == 0).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_grouped_faint_fp32_weights_beside_values_that_are_not_finite(bad):
    """A value that only later queries see does not reach the sums of weights of 2^-130."""
    q = torch.zeros(70, 1, 64, device=DEV)
    q[..., 0] = 1.0
    kc, vc = torch.zeros(2, 1, 1, 90, 64, device=DEV).unbind()
    kc[..., 0], vc[..., 5] = -130.0, 2.0 ** 100
    kc[:, :, 0, 0], vc[:, :, 0, 5] = 0.0, 0.0
    vc[:, :, 41, 5] = vc[:, :, 70:] = kc[:, :, 70:] = bad
    out = torch.full_like(q, 7.0)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    K().attn_grouped(q, kc, vc, i32([0, 70]), i32([70]), 70, out)
    assert bool((out[:41, 0, 5] == torch.arange(41, device=DEV) * 2.0 ** -30).all())
    assert not bool(out[41:, 0, 5].isfinite().any())
    assert bool((out[..., :5] == 0).all()) and bool((out[..., 6:] == 0).all())


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("tokens,slots", [(300, 337), (200, 255), (130, 140)])
def test_grouped_a_workspace_that_is_not_used_changes_nothing(dtype, D, tokens, slots):
    """Where a call needs no workspace (keys too few to be cut), the one that a program keeps for its
    other calls gives the bits of none."""
    if dtype == F32:
        tokens, slots = tokens // 2, slots // 2
    c = Grouped(81, dtype, D, 12, 4, [tokens], [0], spare=slots - tokens)
    q, k, v = c.q.to(DEV), c.k.to(DEV), c.v.to(DEV)
    assert k.shape[2] == slots and K().attn_grouped_workspace_bytes(q, k, tokens) == 0
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    out = []
    for ws in (None, torch.empty(1 << 20, device=DEV)):
        out.append(torch.full_like(q, 7.0))
        K().attn_grouped(q, k, v, i32([0, tokens]), i32([tokens]), tokens, out[-1], workspace=ws)
    ref, bound = c.reference()
    _check(out[0], ref, bound, "no workspace")
    _check(out[1], ref, bound, "workspace")
    assert torch.equal(out[0], out[1])


def _whole_reference(c):
    """Grouped.reference, causal, by matrix products in float64 on the GPU (long sequences)."""
    ref = torch.zeros(c.tokens, c.heads, c.D, dtype=torch.float64, device=DEV)
    bound = torch.zeros_like(ref)
    r = c.heads // c.kv
    for b, (n, keys) in enumerate(zip(c.n, c.keys)):
        a = c.offset[b]
        unseen = torch.arange(keys, device=DEV)[None] > \
            keys - n + torch.arange(n, device=DEV)[:, None]
        for h in range(c.heads):
            q = c.q[a:a + n, h].to(DEV).double()
            k, v = (t[b, h // r, :keys].to(DEV).double() for t in (c.k, c.v))
            kt = k.t().contiguous()
            s = (q @ kt).masked_fill(unseen, float("-inf"))
            w = torch.softmax(s * math.log(2.0), -1)
            ds = (q.abs() @ kt.abs()).masked_fill(unseen, 0.0).amax(-1, keepdim=True)
            ref[a:a + n, h] = w @ v
            bound[a:a + n, h] = _bound(ref[a:a + n, h], w @ v.abs(), 2 * c.D * 2.0 ** -23 * ds, keys,
                                       c.dtype)
    return ref.cpu(), bound.cpu()


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("blocks,seqs,heads,kv,longest", [
    (511, 7, 4, 1, 2331), (512, 4, 8, 1, 2047), (513, 9, 12, 3, 607), (546, 13, 12, 3, 447),
    (1053, 13, 9, 3, 1150)])
def test_grouped_order_of_many_tall_blocks(dtype, D, blocks, seqs, heads, kv, longest):
    """Launches around two blocks for each of the 256 CUs and above, whose second 256 blocks run
    backwards and whose pairs of sequence and head move over the XCDs from the sixth tile on: every
    row is some block's, once."""
    n = [longest - 37 * (b % 5) for b in range(seqs)]
    c = Grouped(blocks, dtype, D, heads, kv, n, [0] * seqs, tail=2)
    assert blocks == seqs * kv * -(-longest * heads // kv // 128)
    ref, bound = _whole_reference(c)
    out = c.run()
    end = c.offset[-1]
    _check(out[:end], ref[:end], bound[:end], blocks)
    assert bool((out[end:] == 7.0).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("tiled", [False, True])
@pytest.mark.parametrize("form", ["flat", "parts", "tall", "tall parts"])
def test_grouped_split_output_of_each_block_form(dtype, D, tiled, form):
    n, past, heads, kv = {"flat": ([3, 18], [0, 0], 4, 2), "parts": ([3, 1], [2200, 1900], 4, 2),
                          "tall": ([150, 300, 77, 5, 290, 33, 128, 257], [0] * 8, 16, 16),
                          "tall parts": ([40, 17], [3000, 2950], 8, 2)}[form]
    c = Grouped(91, dtype, D, heads, kv, n, past, tail=2)
    ws = K().attn_grouped_workspace_bytes(c.q.to(DEV), c.k.to(DEV), max(n))
    assert (ws > 0) == ("parts" in form)
    ref, bound = _whole_reference(c)
    width, rows = heads * D, c.tokens
    pad = -(-rows // 16) * 16 if tiled else rows
    out = torch.full((pad, 2 * width), 3.0, dtype=BF, device=DEV)
    got = c.run(out=out, split=True, tiled=tiled)
    got = (K().untile_matrix(out, rows, 2 * width) if tiled else got)[:rows].double().cpu()
    value = (got[:, :width] + got[:, width:]).view(rows, heads, D)
    end = c.offset[-1]
    # hi + lo is within 2^-8 2^-8 of the fp32 value
    extra = 2.0 ** -16 * ref.abs() - (HALF_STEP[BF] * ref.abs() if dtype == BF else 0)
    _check(value[:end], ref[:end], (bound + extra)[:end], form)
    assert bool((got[end:] == 3.0).all())


@pytest.mark.parametrize("tiled", [None, True])
def test_grouped_far_rows(tiled):
    """q and out of more than 2^31 elements: the last rows, and one in the middle."""
    D, heads, tokens = 128, 256, 66_000
    q = torch.zeros(tokens, heads, D, dtype=BF, device=DEV)
    assert q.numel() > 2 ** 31
    c = Grouped(97, BF, D, heads, 1, [3], [60])
    at = [30_000, 65_998, 65_999]                       # rows that get the queries of c
    q[at] = c.q.to(DEV)
    k, v = c.k.to(DEV), c.v.to(DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    width = heads * D
    out = torch.zeros(tokens, 2 * width if tiled else width, dtype=BF, device=DEV)
    K().attn_grouped(q, k, v, i32([0, tokens]), i32([63]), tokens, out, causal=False,
                     split=bool(tiled), tiled=bool(tiled))
    ref, bound = c.reference(causal=False)
    if tiled:
        first = [(a // 16) * 16 for a in at]             # blocks of sixteen rows
        got = torch.stack([K().untile_matrix(out.view(-1)[2 * f * width:2 * (f + 16) * width], 16,
                                             2 * width)[a - f] for f, a in zip(first, at)]).double()
        got = (got[:, :width] + got[:, width:]).view(3, heads, D)
        bound = bound + 2.0 ** -16 * ref.abs()
    else:
        got = out.view(tokens, heads, D)[at]
    _check(got, ref, bound, "far rows")
    # a query of zeros sees every key alike: the mean of the values
    if not tiled:
        want = c.v[0, 0, :63].double().mean(0).expand(heads, D)
        mass = c.v[0, 0, :63].double().abs().mean(0)
        _check(out.view(tokens, heads, D)[65_997], want,
               2.0 ** -8 * want.abs() + (63 + 64) * 2.0 ** -23 * mass * 1.01, "mean")


def test_grouped_calls_at_once():
    """Two streams, a workspace each, and two captured graphs replayed side by side."""
    kern = K()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    calls = []
    for seed in (98, 99):
        c = Grouped(seed, BF, 128, 8, 2, [3, 40, 1], [2900, 10, 1500])
        q, k, v = c.q.to(DEV), c.k.to(DEV), c.v.to(DEV)
        ws = torch.empty(kern.attn_grouped_workspace_bytes(q, k, 40) // 4, device=DEV)
        assert ws.numel() > 0
        calls.append((c, torch.cuda.Stream(), ws, (q, k, v, i32(c.offset), i32(c.keys), 40,
                                                   torch.full_like(q, 7.0))))
    refs = [c.reference() for c, _, _, _ in calls]
    torch.cuda.synchronize()

    def check(what):
        torch.cuda.synchronize()
        for (ref, bound), (_, _, _, a) in zip(refs, calls):
            _check(a[6], ref, bound, what)
            a[6].fill_(7.0)
        torch.cuda.synchronize()
    for _ in range(4):
        for _, side, ws, a in calls:
            with torch.cuda.stream(side):
                kern.attn_grouped(*a, workspace=ws)
    check("streams")
    graphs = []
    for _, side, ws, a in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            kern.attn_grouped(*a, workspace=ws)
    for step in range(3):
        for g, (_, side, _, _) in zip(graphs, calls):
            with torch.cuda.stream(side):
                g.replay()
        check(f"graphs, replay {step}")


# ---- K8: shared prefixes -----------------------------------------------------------------------

class Shared:
    def __init__(self, seed, dtype, D, heads, kv, edges, prefix, own):
        g = _gen(seed)
        self.edges, self.prefix, self.own = edges, prefix, own
        self.dtype, self.D, self.heads, self.kv = dtype, D, heads, kv
        b = len(own)
        self.q = _rand(g, b, heads, D, std=LOG2E / math.sqrt(D)).to(dtype)
        self.pk = _rand(g, len(prefix), kv, max(prefix) + 5, D).to(dtype)
        self.pv = _rand(g, len(prefix), kv, max(prefix) + 5, D).to(dtype)
        self.k = _rand(g, b, kv, max(own) + 3, D).to(dtype)
        self.v = _rand(g, b, kv, max(own) + 3, D).to(dtype)

    def reference(self, max_rows=None):
        ref = torch.zeros(len(self.own), self.heads, self.D, dtype=torch.float64)
        bound = torch.zeros_like(ref)
        r = self.heads // self.kv
        for b, n in enumerate(self.own):
            group = [g for g in range(len(self.prefix)) if self.edges[g] <= b < self.edges[g + 1]]
            if group and max_rows is not None and b - self.edges[group[0]] >= max_rows:
                group = []
            for h in range(self.heads):
                k, v = self.k[b, h // r, :n], self.v[b, h // r, :n]
                if group:
                    p = self.prefix[group[0]]
                    k = torch.cat([self.pk[group[0], h // r, :p], k])
                    v = torch.cat([self.pv[group[0], h // r, :p], v])
                o, mass, ds = _attend(self.q[b:b + 1, h], k, v, [len(k)])
                ref[b, h], bound[b, h] = o[0], _bound(o, mass, ds, len(k), self.dtype)[0]
        return ref, bound

    def args(self, max_rows=None):
        kern = K()
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
        q, pk, pv, k, v = (t.to(DEV) for t in (self.q, self.pk, self.pv, self.k, self.v))
        if max_rows is None:
            max_rows = max(b - a for a, b in zip(self.edges, self.edges[1:]))
        ws = torch.full((kern.attn_decode_shared_workspace_bytes(q, pk, k, max_rows) // 4,),
                        float("nan"), device=DEV)
        return [q, pk, pv, i32(self.edges), i32(self.prefix), max_rows, k, v, i32(self.own),
                torch.full_like(q, 7.0), ws]

    def run(self, max_rows=None, **form):
        a = self.args(max_rows)
        K().attn_decode_shared(*a, **form)
        torch.cuda.synchronize()
        return a[9]


GROUPS = {
    "one": ([0, 1], [300], [5]),
    "samples": ([0, 9], [731], [1, 40, 2, 33, 64, 65, 7, 128, 9]),
    "many": ([0, 70], [600], [1 + 3 * i for i in range(70)]),
    "groups": ([0, 4, 4, 5, 11], [130, 64, 1, 1000], [3, 0, 9, 200, 31, 1, 1, 2, 0, 5, 300]),
    "outside": ([2, 5, 7], [257, 40], [10, 20, 30, 0, 50, 60, 70, 0, 90]),
    "no_prefix": ([0, 3], [0], [0, 1, 170]),
}


@pytest.mark.parametrize("dtype,D,heads,kv", SHAPES)
@pytest.mark.parametrize("groups", GROUPS)
def test_shared(dtype, D, heads, kv, groups):
    if groups == "no_prefix":
        c = Shared(1, dtype, D, heads, kv, *GROUPS[groups])
        c.prefix = [0]
    else:
        c = Shared(len(groups) + D, dtype, D, heads, kv, *GROUPS[groups])
    ref, bound = c.reference()
    _check(c.run(), ref, bound, groups)


def test_shared_long_prefix_in_parts():
    c = Shared(2, BF, 128, 8, 2, [0, 3, 6], [5000, 3333], [1, 700, 2, 90, 1, 1])
    ref, bound = c.reference()
    _check(c.run(), ref, bound, "parts")
    assert torch.equal(c.run(), c.run())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_shared_tall_prefix(dtype):
    """Enough rows and keys for the prefixes' launch of 128-row blocks, in parts."""
    c = Shared(8, dtype, 128, 16, 4, [0, 31, 37], [9001, 130], [(7 * i) % 40 for i in range(40)])
    ref, bound = c.reference()
    _check(c.run(), ref, bound, "tall")


@pytest.mark.parametrize("n", [64, 65, 300])
def test_shared_many_prefixes(n):
    """A prefix for every other row, the rows between in none of them or in their neighbour's."""
    g = _gen(n)
    sizes = torch.randint(0, 3, (n,), generator=g).tolist()
    edges = [1 + sum(sizes[:i]) for i in range(n + 1)]
    c = Shared(9, BF, 64, 2, 1, edges, [1 + 5 * i % 40 for i in range(n)],
               [i % 9 for i in range(edges[-1] + 2)])
    ref, bound = c.reference()
    _check(c.run(), ref, bound, "prefixes")


def test_shared_rows_past_max_rows_have_no_prefix():
    c = Shared(3, F32, 64, 4, 2, [0, 6], [200], [5, 6, 7, 8, 9, 10])
    ref, bound = c.reference(max_rows=4)
    _check(c.run(max_rows=4), ref, bound, "max_rows")


@pytest.mark.parametrize("max_rows", [2 ** 31, 2 ** 32, 2 ** 32 + 1])
def test_shared_bound_above_the_rows(max_rows):
    c = Shared(63, BF, 64, 4, 2, [0, 3, 5], [70, 33], [9, 40, 5, 64, 7])
    ref, bound = c.reference()
    _check(c.run(max_rows=max_rows), ref, bound, "bound")


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_shared_slots_behind_the_ends(bad):
    """Whatever stands behind a prefix or a row's own slots is not read into a result."""
    c = Shared(4, BF, 64, 6, 3, [0, 2, 5], [70, 33], [1, 40, 0, 64, 7])
    ref, bound = c.reference()
    for t, lens in ((c.pk, c.prefix), (c.pv, c.prefix), (c.k, c.own), (c.v, c.own)):
        for b, n in enumerate(lens):
            t[b, :, n:] = bad
    _check(c.run(), ref, bound, "behind")


def test_shared_values_that_are_not_finite_stay_in_their_rows():
    c = Shared(5, BF, 64, 4, 2, [0, 3, 5], [70, 33], [9, 40, 5, 64, 7])
    ref, bound = c.reference()
    c.v[1, 1, 39, 2] = float("inf")              # the last own slot of row 1, kv head 1
    c.pv[1, 0, 32, 5] = float("nan")             # the last slot of prefix 1, kv head 0
    out = c.run().double().cpu()
    hit = torch.zeros_like(ref, dtype=torch.bool)
    hit[1, 2:, 2] = True
    hit[3:, :2, 5] = True
    _check(torch.where(hit, ref, out), ref, bound, "others")
    assert bool((out[1, 2:, 2] == float("inf")).all()) and bool(torch.isnan(out[3:, :2, 5]).all())


@pytest.mark.parametrize("tiled", [False, True])
def test_shared_split_output(tiled):
    c = Shared(6, F32, 64, 4, 2, [0, 3], [300], [9, 40, 5])
    ref, bound = c.reference()
    a = c.args()
    rows, width = 3, c.heads * c.D
    a[9] = torch.zeros(16 if tiled else rows, 2 * width, dtype=BF, device=DEV)
    K().attn_decode_shared(*a, split=True, tiled=tiled)
    got = K().untile_matrix(a[9], rows, 2 * width) if tiled else a[9]
    got = got.float().cpu()
    value = (got[:, :width] + got[:, width:]).view(rows, c.heads, c.D)
    _check(value, ref, bound + 2.0 ** -16 * ref.abs(), "split")


def test_shared_graph():
    kern = K()
    c = Shared(7, BF, 64, 12, 4, [0, 5, 8], [700, 90], [9, 40, 5, 1, 1, 2, 30, 77])
    a = c.args()
    kern.attn_decode_shared(*a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kern.attn_decode_shared(*a)
    for step in range(3):
        a[8].add_(1)
        a[0].copy_(torch.randn_like(a[0]) * 0.2)
        a[9].fill_(7.0)
        b = list(a)
        b[9], b[10] = torch.full_like(a[9], 7.0), torch.empty_like(a[10])
        kern.attn_decode_shared(*b)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a[9], b[9]), step
        torch.randn(1000, device=DEV).sum().item()


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (F32, 64), (F32, 128)])
def test_shared_one_buffer_for_keys_and_values(dtype, D):
    c = Shared(73, dtype, D, 6, 2, [0, 3, 5], [170, 33], [9, 40, 5, 64, 7])
    c.pv, c.v = c.pk, c.k
    ref, bound = c.reference()
    a = c.args()
    a[2], a[7] = a[1], a[6]
    K().attn_decode_shared(*a)
    _check(a[9], ref, bound, "one buffer")


@pytest.mark.parametrize("heavy", ["first", "last"])
def test_shared_keeps_fp32_weights_below_the_normal_range(heavy):
    """The same over a prefix and the row's own keys: the key of weight 1 is one or the other's."""
    q = torch.zeros(3, 1, 64, device=DEV)
    q[..., 0] = 1.0
    pk, pv = torch.zeros(2, 1, 1, 500, 64, device=DEV).unbind()
    kc, vc = torch.zeros(2, 3, 1, 70, 64, device=DEV).unbind()
    for k, v in ((pk, pv), (kc, vc)):
        k[..., 0], v[..., 5] = -130.0, 2.0 ** 100
    k, v = (pk, pv) if heavy == "first" else (kc, vc)
    k[:, :, 3, 0], v[:, :, 3, 5] = 0.0, 0.0
    out = torch.full_like(q, 7.0)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    ws = torch.empty(K().attn_decode_shared_workspace_bytes(q, pk, kc, 3) // 4, device=DEV)
    K().attn_decode_shared(q, pk, pv, i32([0, 3]), i32([500]), 3, kc, vc, i32([70, 9, 40]), out, ws)
    want = torch.tensor([569.0, 508.0, 539.0], device=DEV) * 2.0 ** -30
    assert bool((out[:, 0, 5] == want).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("tiled", [False, True])
def test_shared_split_output_of_each_type(dtype, D, tiled):
    c = Shared(92, dtype, D, 6, 2, [0, 3, 7], [300, 77], [9, 40, 5, 1, 70, 2, 130, 6])
    ref, bound = c.reference()
    a = c.args()
    rows, width = 8, c.heads * D
    a[9] = torch.zeros(16 if tiled else rows, 2 * width, dtype=BF, device=DEV)
    K().attn_decode_shared(*a, split=True, tiled=tiled)
    got = (K().untile_matrix(a[9], rows, 2 * width) if tiled else a[9]).double().cpu()
    value = (got[:, :width] + got[:, width:]).view(rows, c.heads, D)
    extra = 2.0 ** -16 * ref.abs() - (HALF_STEP[BF] * ref.abs() if dtype == BF else 0)
    _check(value, ref, bound + extra, "split")


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("heads,kv", [(80, 2), (33, 1), (161, 1)])
def test_shared_many_heads_to_one(dtype, D, heads, kv):
    """More query heads to a key / value head than rows in a flat tile: the rows' own keys run in tall
    blocks too."""
    c = Shared(93, dtype, D, heads, kv, [0, 5, 7], [2500, 60], [1, 300, 2, 0, 129, 90, 64, 200])
    ref, bound = c.reference()
    _check(c.run(), ref, bound, f"{heads} heads on {kv}")


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("heads", [4, 80])
def test_shared_values_that_are_not_finite_of_each_type(dtype, D, bad, heads):
    """In slots behind the ends, in a value of the prefix's or a row's own, in a key of either."""
    c = Shared(94, dtype, D, heads, 2, [0, 3, 6], [700, 33], [9, 40, 5, 64, 0, 150, 7])
    ref, bound = c.reference()
    for t, lens in ((c.pk, c.prefix), (c.pv, c.prefix), (c.k, c.own), (c.v, c.own)):
        for b, n in enumerate(lens):
            t[b, :, n:] = bad
    half = heads // 2
    c.v[1, 1, 39, 2] = bad                       # the last own slot of row 1, second kv head
    c.pv[1, 0, 32, 5] = bad                      # the last slot of prefix 1, first kv head
    c.k[6, 0, 3] = float("nan")                  # a whole own key of row 6
    c.pk[0, 0, 100] = float("nan")               # a whole key of prefix 0
    out = c.run().double().cpu()
    hit = torch.zeros_like(ref, dtype=torch.bool)
    hit[1, half:, 2] = hit[3:6, :half, 5] = True
    hit[6, :half] = hit[:3, :half] = True
    _check(torch.where(hit, ref, out), ref, bound, "others")
    for got in (out[1, half:, 2], out[3:6, :half, 5]):
        assert bool(got.isnan().all() if math.isnan(bad) else (got == bad).all())
    assert bool(out[6, :half].isnan().all()) and bool(out[:3, :half].isnan().all())


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (F32, 64), (F32, 128)])
def test_caches_with_many_more_slots_than_keys(dtype, D):
    """Caches that hold a whole output ahead: plans for their slots, most parts without a key."""
    c = Shared(95, dtype, D, 8, 2, [0, 3, 6], [70, 1], [1, 0, 5, 64, 2, 9, 33])

    def wide(t, n):
        return torch.cat([t, torch.full((*t.shape[:2], n, D), float("nan"), dtype=dtype)], 2)

    c.pk, c.pv, c.k, c.v = wide(c.pk, 9000), wide(c.pv, 9000), wide(c.k, 4096), wide(c.v, 4096)
    ref, bound = c.reference()
    _check(c.run(), ref, bound, "shared")
    for n, past in (([1, 1, 1], [0, 40, 129]), ([40, 7, 0], [0, 300, 0])):
        g = Grouped(96, dtype, D, 8, 2, n, past, tail=1)
        g.k, g.v = wide(g.k, 9000), wide(g.v, 9000)
        g.check("parts")
        g.check("no workspace", workspace=False)


def test_shared_another_stream():
    c = Shared(100, F32, 64, 4, 2, [0, 3, 5], [700, 33], [9, 40, 5, 64, 7])
    a = c.args()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K().attn_decode_shared(*a)
    torch.cuda.current_stream().wait_stream(side)
    ref, bound = c.reference()
    _check(a[9], ref, bound, "other stream")


# ---- K7 ----------------------------------------------------------------------------------------

def _rope(D, sizes=(32, 32, 8)):
    rope = RotaryEmbedding3D(D, *sizes)
    return rope.device_table(torch.device("cpu")), (*sizes, rope.px, rope.py, rope.pz)


def _line(D, longest):
    ang = torch.arange(longest, dtype=torch.float64)[:, None] * (
        10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2)))
    return torch.cat([ang.cos().reshape(-1), ang.sin().reshape(-1)]).float(), (longest, 1, 1,
                                                                             D // 2, 0, 0)


def _qk_norm_reference(qkv, rstd, pos, tab, geom, gq, gk, eps, heads, kv, D, q_scale):
    """q, k, v in float64 and the bound of each before its own rounding."""
    y = qkv.double().view(qkv.shape[0], heads + 2 * kv, D)
    if rstd is not None:
        y = y * rstd.double()[:, None, None]
    n = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
    cos, sin, at = [], [], 0
    for axis in range(3):
        size, pairs = geom[axis], geom[3 + axis]
        i = pos[:, axis].clamp(0, size - 1)
        cos.append(tab[at:at + size * pairs].double().view(size, pairs)[i])
        sin.append(tab[at + size * pairs:at + 2 * size * pairs].double().view(size, pairs)[i])
        at += 2 * size * pairs
    cos, sin = torch.cat(cos, 1)[:, None], torch.cat(sin, 1)[:, None]

    def turned(t, gain, scale):
        t = t * gain.double()
        a, b = t[..., 0::2], t[..., 1::2]
        out = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2) * scale
        size = torch.stack(((a * cos).abs() + (b * sin).abs(), (b * cos).abs() + (a * sin).abs()),
                           -1).flatten(-2) * scale
        # y, its square sum (12 additions), rsqrt, two products, the rotation, the scale: under 32
        # roundings of 2^-24 each
        return out, size * 32 * 2.0 ** -24
    q, k = turned(n[:, :heads], gq, q_scale), turned(n[:, heads:heads + kv], gk, 1.0)
    v = y[:, heads + kv:]
    return q, k, (v, v.abs() * 2.0 ** -23)


@pytest.mark.parametrize("source,dtype", [(F32, BF), (F32, F32), (BF, BF), (BF, F32)])
@pytest.mark.parametrize("D,heads,kv", [(64, 12, 12), (64, 3, 1), (128, 10, 5), (128, 16, 1)])
@pytest.mark.parametrize("rows", [1, 37, 700])
def test_qk_norm(source, dtype, D, heads, kv, rows):
    g = _gen(rows + D + heads)
    batch, slots = 5, 211
    wide = _rand(g, rows, (heads + 2 * kv) * D + 24, std=3.0).to(source)
    qkv = wide[:, 8:8 + (heads + 2 * kv) * D]              # strided rows
    rstd = None if rows == 37 else torch.rand(rows, generator=g) + 0.3
    pos = torch.randint(-2, 40, (rows, 3), generator=g)    # some beyond the table: clamped
    tab, geom = _line(D, 300) if kv == 1 else _rope(D)
    gq, gk = 1 + 0.2 * _rand(g, D), 1 + 0.2 * _rand(g, D)
    where = torch.randperm(batch * slots, generator=g)[:rows]
    row, slot = (where // slots).int(), (where % slots).int()
    if rows > 3:                                           # outside the cache: not written
        slot[0], slot[1], row[2], row[3] = -1, slots, batch, -1
    q_scale, eps = LOG2E / math.sqrt(D), 1e-5
    q_ref, k_ref, v_ref = _qk_norm_reference(qkv, rstd, pos, tab, geom, gq, gk, eps, heads, kv, D,
                                             q_scale)
    q = torch.full((rows, heads, D), 7.0, dtype=dtype, device=DEV)
    kc = torch.full((batch, kv, slots, D), 7.0, dtype=dtype, device=DEV)
    vc = torch.full_like(kc, 7.0)
    dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    K().qk_norm_rope_cache(dev(wide)[:, 8:8 + (heads + 2 * kv) * D], dev(rstd), dev(pos), dev(tab),
                           geom, dev(gq), dev(gk), eps, dev(row), dev(slot), q_scale, q, kc, vc)
    half = HALF_STEP[dtype]
    _check(q, q_ref[0], q_ref[1] * (1 + half) + half * q_ref[0].abs() + 1e-30, "q")
    kept = ((slot >= 0) & (slot < slots) & (row >= 0) & (row < batch)).nonzero()[:, 0]
    for got, (ref, err), name in ((kc, k_ref, "k"), (vc, v_ref, "v")):
        got = got.cpu()
        taken = got[row[kept].long(), :, slot[kept].long()]
        _check(taken, ref[kept], err[kept] * (1 + half) + half * ref[kept].abs() + 1e-30, name)
        got[row[kept].long(), :, slot[kept].long()] = 7.0
        assert bool((got == 7.0).all()), f"{name}: a slot of no token was written"


def test_qk_norm_streaming_rows_and_far_slots():
    """A batch past the streaming size, into a cache of more than 2^31 elements."""
    g = _gen(5)
    D, heads, kv, rows, slots = 128, 8, 2, 12000, 4_300_000
    kc = torch.empty(2, kv, slots, D, dtype=BF, device=DEV)
    vc = torch.empty_like(kc)
    assert kc.numel() > 2 ** 31 and rows * (heads + 2 * kv) * D * 4 > 2 ** 26
    qkv = _rand(g, rows, (heads + 2 * kv) * D)
    pos = torch.randint(0, 30, (rows, 3), generator=g)
    tab, geom = _rope(D)
    gq, gk = torch.ones(D), torch.ones(D)
    row, slot = (torch.arange(rows) % 2).int(), (slots - 1 - torch.arange(rows)).int()
    q = torch.empty(rows, heads, D, dtype=BF, device=DEV)
    K().qk_norm_rope_cache(qkv.to(DEV), None, pos.to(DEV), tab.to(DEV), geom, gq.to(DEV),
                           gk.to(DEV), 1e-5, row.to(DEV), slot.to(DEV), 0.5, q, kc, vc)
    q_ref, k_ref, v_ref = _qk_norm_reference(qkv, None, pos, tab, geom, gq, gk, 1e-5, heads, kv, D,
                                             0.5)
    half = HALF_STEP[BF]
    row, slot = row.long().to(DEV), slot.long().to(DEV)
    for got, (ref, err) in ((q, q_ref), (kc[row, :, slot], k_ref), (vc[row, :, slot], v_ref)):
        _check(got, ref, err * (1 + half) + half * ref.abs() + 1e-30)


def test_qk_norm_refuses_a_cache_without_rows():
    """q_out is written for every token, in the cache or not, so a call that would leave it as it was
    is an error; one without tokens has nothing to write."""
    D, heads, kv = 64, 4, 2
    tab, geom = _rope(D)
    ones = torch.ones(D, device=DEV)
    for rows in (3, 0):
        qkv = torch.zeros(rows, (heads + 2 * kv) * D, device=DEV)
        pos = torch.zeros(rows, 3, dtype=torch.int64, device=DEV)
        at = torch.zeros(rows, dtype=torch.int32, device=DEV)
        q = torch.full((rows, heads, D), 7.0, device=DEV)
        cache = torch.zeros(0, kv, 8, D, device=DEV)
        args = (qkv, None, pos, tab.to(DEV), geom, ones, ones, 1e-5, at, at, 1.0, q, cache,
                torch.zeros_like(cache))
        if rows:
            with pytest.raises(ValueError, match="batch"):
                K().qk_norm_rope_cache(*args)
        else:
            K().qk_norm_rope_cache(*args)


def test_qk_norm_far_rows():
    """qkv and q_out of more than 2^31 elements."""
    D, heads, kv, rows = 128, 256, 1, 66_000
    g = _gen(101)
    tab, geom = _rope(D)
    gain = torch.ones(D)
    last = _rand(g, 4, (heads + 2 * kv) * D).to(BF)
    qkv = torch.ones(rows, (heads + 2 * kv) * D, dtype=BF, device=DEV)
    qkv[-4:] = last.to(DEV)
    pos = torch.randint(0, 30, (rows, 3), generator=g)
    slot = torch.arange(rows).int()
    q = torch.empty(rows, heads, D, dtype=BF, device=DEV)
    assert q.numel() > 2 ** 31
    kc, vc = torch.zeros(2, 1, kv, rows, D, dtype=BF, device=DEV).unbind()
    K().qk_norm_rope_cache(qkv, None, pos.to(DEV), tab.to(DEV), geom, gain.to(DEV), gain.to(DEV),
                           1e-5, torch.zeros(rows, dtype=torch.int32, device=DEV), slot.to(DEV), 0.5,
                           q, kc, vc)
    refs = _qk_norm_reference(last, None, pos[-4:], tab, geom, gain, gain, 1e-5, heads, kv, D, 0.5)
    half = HALF_STEP[BF]
    for got, (ref, err) in zip((q[-4:], kc[0, :, -4:].transpose(0, 1), vc[0, :, -4:].transpose(0, 1)),
                               refs):
        _check(got, ref, err * (1 + half) + half * ref.abs() + 1e-30)


def test_qk_norm_graph_and_streams():
    """Captured once, replayed with other tokens and slots between eager work; another stream."""
    kern = K()
    D, heads, kv, rows, slots = 64, 6, 2, 16, 50
    g = _gen(102)
    tab, geom = _rope(D)
    ones = torch.ones(D, device=DEV)
    qkv = _rand(g, rows, (heads + 2 * kv) * D).to(DEV)
    pos = torch.randint(0, 30, (rows, 3), generator=g).to(DEV)
    row = torch.arange(rows, dtype=torch.int32, device=DEV)
    slot = torch.full_like(row, 3)
    new = lambda: (torch.full((rows, heads, D), 7.0, dtype=BF, device=DEV),  # noqa: E731
                   *torch.zeros(2, rows, kv, slots, D, dtype=BF, device=DEV).unbind())
    tab = tab.to(DEV)
    run = lambda o: kern.qk_norm_rope_cache(qkv, None, pos, tab, geom, ones, ones, 1e-5, row, slot,  # noqa: E731
                                            0.2, *o)
    a, b = new(), new()
    run(a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(b)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(a)
    for step in range(3):
        qkv.copy_(torch.randn_like(qkv))
        pos.add_(1)
        slot.add_(7)
        run(b)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(a, b)), step
        torch.randn(1000, device=DEV).sum().item()


# ---- together ----------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, F32])
def test_prompts_then_samples(dtype):
    """Two prompts through K7 and K8, then three decode steps of their samples behind them, the
    outputs through the out projection (K5): against the same in 64 bits."""
    kern = K()
    D, heads, kv, prompts, samples = 64, 6, 2, [40, 75], [2, 3]
    width, d = (heads + 2 * kv) * D, heads * D
    g = _gen(21)
    tab, geom = _line(D, 200)
    gq, gk = 1 + 0.1 * _rand(g, D), 1 + 0.1 * _rand(g, D)
    qs = LOG2E / math.sqrt(D)
    w = (_rand(g, d, d) / math.sqrt(d)).to(BF)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    dev = lambda t: t.to(DEV)  # noqa: E731
    new = lambda *s: torch.zeros(*s, dtype=dtype, device=DEV)  # noqa: E731

    def norm(qkv, slot, row, kc, vc):
        pos = torch.zeros(len(slot), 3, dtype=torch.int64)
        pos[:, 0] = torch.tensor(slot)
        q = new(len(slot), heads, D)
        return pos, q, lambda at: kern.qk_norm_rope_cache(
            dev(qkv), None, dev(pos), dev(tab), geom, dev(gq), dev(gk), 1e-5, i32(row), i32(at), qs,
            q, kc, vc)

    def project(out, rows):
        x = torch.zeros(kern.tile_rows(rows), d, device=DEV)
        kern.gemm_split_residual(out, kern.tile_matrix(dev(w)), x, None, rows, d, d)
        return kern.untile_f32(x.reshape(-1), rows, d).cpu()

    def close(got, parts):
        """Through the projection: each output's bound times |W|, and K5's own 2^-15."""
        ref = torch.cat([p[0] for p in parts]).view(-1, d)
        bound = torch.cat([p[1] for p in parts]).view(-1, d) + 2.0 ** -16 * ref.abs()
        wd = w.double()
        _check(got, ref @ wd.T, bound @ wd.abs().T + 2.0 ** -15 * ref.abs() @ wd.abs().T, "step")

    tokens = sum(prompts)
    pk, pv = new(2, kv, 80, D), new(2, kv, 80, D)
    qkv = _rand(g, tokens, width)
    slot = [i for n in prompts for i in range(n)]
    row = [b for b, n in enumerate(prompts) for _ in range(n)]
    _, q, go = norm(qkv, slot, row, pk, pv)
    go(slot)
    out = torch.zeros(kern.tile_rows(tokens), 2 * d, dtype=BF, device=DEV)
    ws = torch.empty(kern.attn_grouped_workspace_bytes(q, pk, max(prompts)) // 4, device=DEV)
    kern.attn_grouped(q, pk, pv, i32([0, 40, 115]), i32(prompts), max(prompts), out, workspace=ws,
                      split=True, tiled=True)

    def attend(q, k, v, limit):
        r = heads // kv
        o = [_attend(q[:, h].cpu(), k[h // r].cpu(), v[h // r].cpu(), limit) for h in range(heads)]
        n = max(limit)
        return (torch.stack([x[0] for x in o], 1),
                torch.stack([_bound(*x, n, dtype, half_step=0.0) for x in o], 1))
    close(project(out, tokens), [attend(q[:40], pk[0], pv[0], list(range(1, 41))),
                                 attend(q[40:], pk[1], pv[1], list(range(1, 76)))])

    batch, own = 5, []
    kc, vc = new(batch, kv, 8, D), new(batch, kv, 8, D)
    lens = torch.zeros(batch, dtype=torch.int32, device=DEV)
    group = [0, 0, 1, 1, 1]
    for step in range(3):
        at = [prompts[p] + step for p in group]
        _, q, go = norm(_rand(g, batch, width), at, list(range(batch)), kc, vc)
        go([step] * batch)
        lens += 1
        out = torch.zeros(16, 2 * d, dtype=BF, device=DEV)
        ws = torch.empty(kern.attn_decode_shared_workspace_bytes(q, pk, kc, 3) // 4, device=DEV)
        kern.attn_decode_shared(q, pk, pv, i32([0, 2, 5]), i32(prompts), 3, kc, vc, lens, out, ws,
                                split=True, tiled=True)
        parts = []
        for b in range(batch):
            p, n = group[b], prompts[group[b]]
            k = torch.cat([pk[p, :, :n], kc[b, :, :step + 1]], 1)
            v = torch.cat([pv[p, :, :n], vc[b, :, :step + 1]], 1)
            parts.append(attend(q[b:b + 1], k, v, [n + step + 1]))
        close(project(out, batch), parts)
