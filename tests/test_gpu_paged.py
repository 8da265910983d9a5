"""K9 and K10 on the GPU (append to paged caches, slots read back, attention over pages in bf16, fp32
and 4 bits) through mdlarc_scale_amd.kernels, against plain implementations in 64 bits on the CPU.

Tolerances are those of the contiguous forms (test_gpu_grouped.py): the pages change where a value
lies, and a 4-bit number times its power is exact in bf16 and fp32, so references take the values that
the pages hold.  What is written in 4 bits is compared exactly: the fp32 values in front of the
quantisation come from the reference's own arithmetic with the kernel's roundings."""

import math

import pytest
import torch

from mdlarc_scale_amd.transformer import LOG2E

from .paged_ref import from_fp4, page_table, to_fp4, to_pool
from .test_gpu_grouped import (BATCHES, BF, DEV, F32, HALF_STEP, K, Grouped, _attend, _bound, _check,
                               _gen, _line, _qk_norm_reference, _rand, _rope)

pytestmark = pytest.mark.gpu

U8 = torch.uint8


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class Paged(Grouped):
    """A packed batch whose keys and values lie in pages.  Pages of no sequence, slots behind the keys
    and table entries behind the last page hold what must not be seen."""

    def __init__(self, seed, dtype, D, heads, kv, n, past, page=16, fp4=False, spare=3, extra=2,
                 **kw):
        super().__init__(seed, dtype, D, heads, kv, n, past, **kw)
        g = _gen(seed + 1)
        self.page, self.fp4 = page, fp4
        counts = [-(-k // page) for k in self.keys]
        self.n_pages = sum(counts) + spare
        self.table = page_table(counts, max(counts) + extra, self.n_pages, g)
        if fp4:
            kc, self.k = self._four(self.k, dtype)
            vc, self.v = self._four(self.v, dtype)
            self.codes = kc, vc

    @staticmethod
    def _four(t, dtype):
        codes, scale = to_fp4(t.float())
        return (codes, scale), from_fp4(codes, scale).to(dtype)

    def pools(self):
        """k, v and their scales on the GPU, NaN wherever no sequence has a key."""
        def pool(rows, fill):
            rows = rows.clone()
            for s, n in enumerate(self.keys):
                rows[s, :, n:] = fill
            return to_pool(rows, self.table, self.n_pages, self.page, fill).to(DEV)
        if self.fp4:
            (kc, ks), (vc, vs) = self.codes
            return pool(kc, 0x35), pool(vc, 0x53), pool(ks, 255), pool(vs, 255)
        return pool(self.k, float("nan")), pool(self.v, float("nan")), None, None

    def run(self, causal=True, keys=None, workspace=True, max_q=None, out=None, table=None,
            pools=None, **form):
        kern = K()
        k, v, ks, vs = self.pools() if pools is None else pools
        table = self.table.to(DEV) if table is None else table
        q = self.q.to(DEV)
        max_q = max(self.n) if max_q is None else max_q
        ws = None
        if workspace:
            ws = torch.full((kern.attn_paged_workspace_bytes(q, k, table, max_q) // 4,),
                            float("nan"), device=DEV)
        if out is None:
            out = torch.full_like(q, 7.0)
        kern.attn_paged(q, k, v, table, i32(self.offset), i32(self.keys if keys is None else keys),
                        max_q, out, causal=causal, workspace=ws, k_scale=ks, v_scale=vs, **form)
        torch.cuda.synchronize()
        return out


FORMS = [(BF, 64, 12, 4, False), (BF, 128, 5, 1, False), (F32, 64, 6, 3, False),
         (F32, 128, 4, 2, False), (BF, 64, 12, 12, True), (BF, 128, 16, 2, True),
         (F32, 64, 16, 1, True), (F32, 128, 4, 2, True)]


@pytest.mark.parametrize("dtype,D,heads,kv,fp4", FORMS)
@pytest.mark.parametrize("batch", BATCHES)
def test_paged(dtype, D, heads, kv, fp4, batch):
    n, past = BATCHES[batch]
    page = {"one": 16, "edges": 48, "ragged": 32, "chunk": 16}.get(batch, 64)
    c = Paged(len(batch) + D + heads, dtype, D, heads, kv, n, past, page=page, fp4=fp4, tail=3)
    c.check("causal")
    c.check("whole", causal=False)


@pytest.mark.parametrize("dtype,D,heads,kv,fp4", FORMS)
def test_paged_tall_blocks(dtype, D, heads, kv, fp4):
    """Enough rows for blocks of 128, uncut; then a few hundred rows behind thousands of keys, in
    parts: more pages than the 64 whose numbers a wave holds."""
    c = Paged(3, dtype, D, 16, 16, [150, 300, 77, 5, 290, 33, 128, 257], [0] * 8, page=48, fp4=fp4,
              tail=2)
    c.check("tall")
    c = Paged(13, dtype, D, 8, 2, [40, 17, 0, 3], [3000, 2950, 2000, 1], fp4=fp4, tail=1)
    assert K().attn_paged_workspace_bytes(c.q.to(DEV), c.pools()[0], c.table, 40) > 0
    c.check("parts")
    c.check("no workspace", workspace=False)


@pytest.mark.parametrize("dtype,D,heads,kv,fp4", FORMS)
def test_paged_single_tokens(dtype, D, heads, kv, fp4):
    """A decode step: rows of very different lengths, one and none among them, wide table."""
    keys = [0, 1, 15, 16, 17, 31, 33, 1023, 1024, 1025, 2047, 4099]
    c = Paged(5, dtype, D, heads, kv, [1] * len(keys), [max(k - 1, 0) for k in keys], fp4=fp4,
              extra=70)
    c.keys = keys
    c.check("parts")
    c.check("no workspace", workspace=False)
    assert torch.equal(c.run(), c.run())


@pytest.mark.parametrize("dtype,D,heads,kv,fp4", FORMS)
@pytest.mark.parametrize("keys", [[9001], [5, 130, 0], [2600, 1, 900, 4000, 77, 31]])
@pytest.mark.parametrize("extra", [0, 600])
def test_paged_single_tokens_in_many_parts(dtype, D, heads, kv, fp4, keys, extra):
    """Few rows behind keys that are cut into as many parts as there are; a wide table leaves most of
    them empty."""
    c = Paged(19, dtype, D, heads, kv, [1] * len(keys), [max(k - 1, 0) for k in keys], fp4=fp4,
              extra=extra)
    c.keys = keys
    c.check("many parts")
    assert torch.equal(c.run(), c.run())


@pytest.mark.parametrize("dtype,D,fp4", [(BF, 64, False), (F32, 64, False), (F32, 128, False),
                                         (BF, 64, True), (BF, 128, True), (F32, 128, True)])
@pytest.mark.parametrize("causal", [True, False])
def test_paged_first_queries_alone(dtype, D, fp4, causal):
    """max_q 1 where sequences have more queries: the first of each sees what it would see among
    them, the others stay as they were."""
    c = Paged(15, dtype, D, 8, 2, [3, 1, 40, 0, 2], [500, 1700, 3, 0, 0], fp4=fp4)
    ref, bound = c.reference(causal)
    for workspace in (True, False):
        out = c.run(max_q=1, causal=causal, workspace=workspace)
        first = [0, 3, 4, 44]
        _check(out[first], ref[first], bound[first], "first queries")
        rest = [i for i in range(c.tokens) if i not in first]
        assert bool((out[rest] == 7.0).all())
    # fewer keys than queries: the first sees none
    keys = [2, 0, 12, 0, 1]
    out = c.run(max_q=1, keys=keys)
    assert bool((out[[0, 3, 4, 44]] == 0).all())


@pytest.mark.parametrize("dtype,D,fp4", [(F32, 64, False), (F32, 128, False), (BF, 64, True),
                                         (BF, 128, True), (F32, 64, True), (F32, 128, True)])
@pytest.mark.parametrize("heads,kv", [(16, 1), (17, 1), (7, 7), (15, 5)])
def test_paged_single_tokens_of_many_heads(dtype, D, fp4, heads, kv):
    """16 heads to a key / value head fill the rows of a block, 17 take the other tiles; large scores
    move the reference often."""
    c = Paged(17, dtype, D, heads, kv, [1] * 5, [700, 0, 63, 64, 1500], fp4=fp4, std=4.0)
    c.check("many heads")
    c.check("whole", workspace=False)


@pytest.mark.parametrize("dtype,fp4", [(BF, False), (F32, False), (BF, True), (F32, True)])
@pytest.mark.parametrize("workspace", [True, False])
def test_paged_rows_that_see_nothing(dtype, fp4, workspace):
    c = Paged(5, dtype, 64, 4, 2, [40, 3, 70, 1], [0, 0, 0, 0], fp4=fp4)
    keys = [10, 0, 69, 0]
    c.check("causal", keys=keys, workspace=workspace)
    c.check("whole", causal=False, keys=keys, workspace=workspace)
    out = c.run(keys=keys, workspace=workspace)
    assert bool((out[:30] == 0).all()) and bool((out[40:43] == 0).all())


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("n,past", [([70, 45, 1], [0, 20, 1500]), ([200] * 9, [0] * 9)])
def test_paged_gives_the_bits_of_the_contiguous_form(dtype, D, n, past):
    """With as many slots, the same work in the same order."""
    c = Paged(31, dtype, D, 16, 4, n, past, page=32, extra=0, spare=0)
    slots = c.table.shape[1] * 32
    k = torch.zeros(len(n), 4, slots, D, dtype=dtype)
    v = torch.zeros_like(k)
    for s, m in enumerate(c.keys):
        k[s, :, :m], v[s, :, :m] = c.k[s, :, :m], c.v[s, :, :m]
    q, k, v = c.q.to(DEV), k.to(DEV), v.to(DEV)
    out = torch.full_like(q, 7.0)
    ws = torch.empty(K().attn_grouped_workspace_bytes(q, k, max(n)) // 4, device=DEV)
    K().attn_grouped(q, k, v, i32(c.offset), i32(c.keys), max(n), out, workspace=ws)
    assert torch.equal(c.run(), out)


@pytest.mark.parametrize("dtype,D,fp4", [(BF, 64, False), (BF, 128, False), (F32, 64, False),
                                         (BF, 64, True), (BF, 128, True), (F32, 128, True)])
@pytest.mark.parametrize("workspace", [True, False])
def test_paged_values_that_are_not_finite(dtype, D, fp4, workspace):
    """A value in a slot that only later queries see reaches nobody else.  (In 4 bits NaN comes by 32
    channels; slots behind the keys are NaN in every test here.)"""
    c = Paged(7, dtype, D, 6, 2, [70, 45], [0, 20], fp4=fp4)
    ref, bound = c.reference()
    at = 50
    if fp4:
        c.codes[1][1][:, 0, at, 0] = 255           # channels 0..31 of a value
        c.codes[0][1][:, 1, at] = 255              # a whole key
        gone = 32
    else:
        c.v[:, 0, at, 0] = float("nan")
        c.k[:, 1, at] = float("nan")
        gone = 1
    out = c.run(workspace=workspace).double().cpu()
    hit = torch.zeros(c.offset[-1], dtype=torch.bool)
    hit[50:70] = True
    hit[70 + 30:] = True
    _check(out[~hit], ref[~hit], bound[~hit], "rows before")
    _check(out[hit][:, :3, gone:], ref[hit][:, :3, gone:], bound[hit][:, :3, gone:], "others")
    assert bool(torch.isnan(out[hit][:, :3, :gone]).all())
    assert bool(torch.isnan(out[hit][:, 3:]).all())


@pytest.mark.parametrize("dtype,fp4", [(BF, False), (F32, False), (BF, True)])
@pytest.mark.parametrize("number", [-1, 10 ** 6, 2 ** 31 - 1, -2 ** 31])
@pytest.mark.parametrize("workspace", [True, False])
def test_paged_numbers_outside_the_pool(dtype, fp4, number, workspace):
    """Rows that see such a page are NaN; other sequences are as they were, and so is a sequence that
    has such a number only behind its keys."""
    c = Paged(8, dtype, 64, 4, 2, [3, 40, 1, 2], [900, 0, 1700, 33], fp4=fp4)
    ref, bound = c.reference()
    table = c.table.clone()
    table[0, 40] = number
    table[2, 2] = number
    table[3, 3:] = number
    out = c.run(workspace=workspace, table=table.to(DEV)).double().cpu()
    assert bool(torch.isnan(out[:3]).all()) and bool(torch.isnan(out[43]).all())
    for rows in (slice(3, 43), slice(44, 46)):
        _check(out[rows], ref[rows], bound[rows], "the others")


def test_paged_strided_table_and_shared_pages():
    """A table cut to its first columns, and two sequences with the pages of one prefix."""
    c = Paged(9, BF, 64, 4, 2, [1, 1], [200, 200], page=64, extra=60)
    wide = c.table.to(DEV)
    c.check("narrow", table=wide[:, :4])
    c.table[1, :3] = c.table[0, :3]
    c.k[1, :, :192], c.v[1, :, :192] = c.k[0, :, :192], c.v[0, :, :192]
    c.check("shared")
    one = Paged(10, BF, 64, 4, 2, [2], [64], page=16, extra=0)
    one.check("one row of another table", table=one.table.to(DEV).expand(3, -1)[:1])


@pytest.mark.parametrize("fp4", [False, True])
def test_paged_lengths_out_of_range_are_clamped(fp4):
    c = Paged(11, F32, 64, 4, 2, [5, 6], [22, 0], page=16, fp4=fp4, extra=0, spare=0)
    slots = c.table.shape[1] * 16
    c.keys = [slots, 0]
    c.table = torch.arange(c.table.numel(), dtype=torch.int32).view(c.table.shape)
    c.n_pages = c.table.numel()
    pad = slots - c.k.shape[2]
    if fp4:
        assert pad <= 0
    ref_off, c.offset = c.offset, [-3, 5, 99]
    c.keys = [min(slots, c.k.shape[2]), 0]
    pools = c.pools()
    out = c.run(keys=[slots + 50, -4], max_q=8, pools=pools)
    c.offset = ref_off
    ref, bound = c.reference(keys=[slots, 0])
    _check(out, ref, bound, "clamped")


@pytest.mark.parametrize("dtype,fp4", [(BF, False), (F32, False), (BF, True), (F32, True)])
@pytest.mark.parametrize("tiled", [False, True])
@pytest.mark.parametrize("past", [0, 2200])
def test_paged_split_output(dtype, fp4, tiled, past):
    c = Paged(10, dtype, 64, 4, 2, [3, 18], [past, past], fp4=fp4, tail=2)
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
    extra = 2.0 ** -16 * ref.abs() - (HALF_STEP[BF] * ref.abs() if dtype == BF else 0)
    _check(value[:end], ref[:end], (bound + extra)[:end], "split")
    assert bool((got[end:] == 3.0).all())


@pytest.mark.parametrize("fp4", [False, True])
def test_paged_far_pages(fp4):
    """Pages behind 2^31 elements of a pool."""
    D, kv, page = 128, 2, 64
    c = Paged(12, BF, D, 4, kv, [3, 1], [60, 300], page=page, fp4=fp4)
    n = 2 ** 31 // (kv * page * (D // 2 if fp4 else D)) + 40
    small = c.pools()
    big = []
    for t in small:
        if t is None:
            big.append(None)
            continue
        far = torch.empty(n, *t.shape[1:], dtype=t.dtype, device=DEV)
        far[n - len(t):] = t
        big.append(far)
    assert big[0].numel() > 2 ** 31
    table = torch.where(c.table >= 0, c.table + n - len(small[0]), -1).int()
    ref, bound = c.reference()
    for workspace in (True, False):
        out = c.run(workspace=workspace, table=table.to(DEV), pools=big)
        _check(out, ref, bound, "far pages")
    # written and read there
    row, slot = i32([0, 1]), i32([5, 299])
    qkv = _rand(_gen(1), 2, (4 + 2 * kv) * D).to(DEV)
    tab, geom = _line(D, 400)
    pos = torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    q = torch.empty(2, 4, D, dtype=BF, device=DEV)
    K().rope_cache_paged(qkv, None, pos, tab.to(DEV), geom, row, slot, table.to(DEV), 1.0, q,
                         *big[:2], k_scale=big[2], v_scale=big[3])
    kr, vr = (torch.zeros(2, kv, 1, D, dtype=BF, device=DEV) for _ in range(2))
    K().paged_rows(*big[:2], table.to(DEV), slot, i32([1, 1]), kr, vr, k_scale=big[2],
                   v_scale=big[3])
    want = qkv.cpu().view(2, -1, D)
    for got, t in ((kr, want[:, 4:4 + kv]), (vr, want[:, 4 + kv:])):
        t = from_fp4(*to_fp4(t)).to(BF) if fp4 else t.to(BF)
        assert torch.equal(got[:, :, 0].cpu(), t)


@pytest.mark.parametrize("fp4", [False, True])
def test_paged_graphs_and_streams(fp4):
    """Two captured calls with workspaces of their own, replayed in turn and at once with other data
    and lengths between eager work, on other streams."""
    kern, table_w = K(), 130
    cs = [Paged(20 + i, BF, 64, 8, 2, [1, 1, 1], [900, 0, 1500], fp4=fp4, extra=table_w)
          for i in range(2)]
    runs, held = [], []   # `held`: what the graphs read lives as long as they do
    for c in cs:
        k, v, ks, vs = c.pools()
        q, out, table = c.q.to(DEV), torch.full_like(c.q, 7.0, device=DEV), c.table.to(DEV)
        ws = torch.empty(kern.attn_paged_workspace_bytes(q, k, table, 1) // 4, device=DEV)
        off, lens = i32(c.offset), i32(c.keys)
        call = (lambda q=q, k=k, v=v, ks=ks, vs=vs, table=table, off=off, lens=lens, out=out, ws=ws:
                kern.attn_paged(q, k, v, table, off, lens, 1, out, workspace=ws, k_scale=ks,
                                v_scale=vs))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        runs.append((c, graph, out, lens, side))
        held.append(call)
    for step in range(3):
        for c, graph, out, lens, side in runs:
            if step == 1:
                c.keys = [500, 1, 1499]
                lens.copy_(i32(c.keys))
            out.fill_(7.0)
        torch.cuda.synchronize()
        for c, graph, out, lens, side in runs:
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        for c, graph, out, lens, side in runs:
            ref, bound = c.reference()
            _check(out, ref, bound, f"replay {step}")


def test_paged_too_many_queries_and_no_tokens():
    c = Paged(8, BF, 64, 4, 2, [40, 9], [0, 300])
    ref, bound = c.reference()
    for workspace in (True, False):
        out = c.run(max_q=9, workspace=workspace)
        _check(out[:9], ref[:9], bound[:9], "first rows")
        assert bool((out[9:40] == 7.0).all())
    k, v, _, _ = c.pools()
    none = torch.zeros(0, 4, 64, dtype=BF, device=DEV)
    K().attn_paged(none, k, v, c.table.to(DEV), i32([0, 0, 0]), i32([1, 1]), 1, none)
    K().attn_paged(c.q.to(DEV), k, v, c.table.to(DEV)[:0], i32([0]), i32([]), 1,
                   torch.zeros_like(c.q, device=DEV))


# ---- K9 ----------------------------------------------------------------------------------------

def _rotated(qkv, rstd, pos, tab, geom, heads, kv, D):
    """q, k, v [rows, .., D] in fp32 with the kernel's roundings: the factor, then a multiply-add on a
    rounded product (in 64 bits the product of two fp32 numbers is exact, and the sum is too unless
    its terms lie 2^29 apart)."""
    y = qkv.float().view(len(qkv), heads + 2 * kv, D)
    if rstd is not None:
        y = y * rstd[:, None, None]
    cos, sin, at = [], [], 0
    for axis in range(3):
        size, pairs = geom[axis], geom[3 + axis]
        i = pos[:, axis].clamp(0, size - 1)
        cos.append(tab[at:at + size * pairs].view(size, pairs)[i])
        sin.append(tab[at + size * pairs:at + 2 * size * pairs].view(size, pairs)[i])
        at += 2 * size * pairs
    cos, sin = torch.cat(cos, 1)[:, None], torch.cat(sin, 1)[:, None]
    a, b = y[:, :heads + kv, 0::2], y[:, :heads + kv, 1::2]
    t = torch.stack((a.double() * cos.double() - (b * sin).double(),
                     b.double() * cos.double() + (a * sin).double()), -1).float().flatten(-2)
    return t[:, :heads], t[:, heads:], y[:, heads + kv:]


def _tokens(g, rows, n_seq, slots):
    where = torch.randperm(n_seq * slots, generator=g)[:rows]
    return (where // slots).int(), (where % slots).int()


@pytest.mark.parametrize("source,dtype,fp4", [(F32, BF, False), (F32, F32, False), (BF, BF, False),
                                              (BF, F32, False), (F32, BF, True), (F32, F32, True),
                                              (BF, BF, True), (BF, F32, True)])
@pytest.mark.parametrize("D,heads,kv", [(64, 12, 12), (64, 3, 1), (128, 10, 5), (128, 16, 1)])
@pytest.mark.parametrize("rows", [1, 37, 700])
def test_append(source, dtype, fp4, D, heads, kv, rows):
    """Written and read back: values, slots of no token, and tokens with nowhere to go."""
    g = _gen(rows + D + heads)
    n_seq, page = 5, 48
    width = 5
    slots, n_pages = width * page, n_seq * width + 2
    wide = _rand(g, rows, (heads + 2 * kv) * D + 24, std=3.0).to(source)
    qkv = wide[:, 8:8 + (heads + 2 * kv) * D]
    rstd = None if rows == 37 else torch.rand(rows, generator=g) + 0.3
    pos = torch.randint(-2, 40, (rows, 3), generator=g)
    tab, geom = _line(D, 300) if kv == 1 else _rope(D)
    norm = not fp4 and rows != 37
    gains = (1 + 0.2 * _rand(g, D), 1 + 0.2 * _rand(g, D)) if norm else (None, None)
    row, slot = _tokens(g, rows, n_seq, slots)
    table = page_table([width] * n_seq, width, n_pages, g)
    table[1, 2], table[2, 0], table[3, 4] = -1, n_pages, 2 ** 31 - 1
    if rows > 3:
        slot[0], slot[1], row[2], row[3] = -1, slots, n_seq, -1
    q_scale = LOG2E / math.sqrt(D)
    dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    q = torch.full((rows, heads, D), 7.0, dtype=dtype, device=DEV)
    shape = (n_pages, kv, page)
    if fp4:
        pools = [torch.full((*shape, D // 2), 0x77, dtype=U8, device=DEV) for _ in range(2)]
        scales = [torch.full((*shape, D // 32), 130, dtype=U8, device=DEV) for _ in range(2)]
    else:
        pools = [torch.full((*shape, D), 7.0, dtype=dtype, device=DEV) for _ in range(2)]
        scales = [None, None]
    K().rope_cache_paged(dev(wide)[:, 8:8 + (heads + 2 * kv) * D], dev(rstd), dev(pos), dev(tab),
                         geom, dev(row), dev(slot), dev(table), q_scale, q, *pools,
                         k_scale=scales[0], v_scale=scales[1], q_gamma=dev(gains[0]),
                         k_gamma=dev(gains[1]))
    kept = ((slot >= 0) & (slot < slots) & (row >= 0) & (row < n_seq))
    number = table[row.clamp(0, n_seq - 1).long(), slot.clamp(0, slots - 1).long() // page]
    kept &= (number >= 0) & (number < n_pages)
    number, at = number[kept].long(), slot[kept].long() % page
    half = HALF_STEP[dtype]
    if norm:
        refs = _qk_norm_reference(qkv, rstd, pos, tab, geom, *gains, 1e-5, heads, kv, D, q_scale)
    else:
        t = _rotated(qkv, rstd, pos, tab, geom, heads, kv, D)
        refs = [(x.double(), torch.zeros_like(x, dtype=torch.float64)) for x in t]
        refs[0] = (refs[0][0] * q_scale, refs[0][0].abs() * q_scale * 2.0 ** -23)
    _check(q, refs[0][0], refs[0][1] * (1 + half) + half * refs[0][0].abs() + 1e-30, "q")
    for pool, scale, (ref, err) in zip(pools, scales, refs[1:]):
        pool = pool.cpu()
        if fp4:
            scale = scale.cpu()
            codes, power = to_fp4(ref[kept].float())
            assert torch.equal(scale[number, :, at], power)
            assert torch.equal(pool[number, :, at], codes)
            scale[number, :, at] = 130
            assert bool((scale == 130).all())
            pool[number, :, at] = 0x77
            assert bool((pool == 0x77).all())
            continue
        _check(pool[number, :, at], ref[kept], err[kept] * (1 + half) + half * ref[kept].abs() +
               1e-30, "pages")
        pool[number, :, at] = 7.0
        assert bool((pool == 7.0).all()), "a slot of no token was written"


def test_append_gives_the_bits_of_the_contiguous_form():
    """With norms K7's, without (64 dims) K2's: the arithmetic is the same."""
    g = _gen(4)
    D, heads, rows, page = 64, 6, 90, 16
    tab, geom = _rope(D)
    dev = lambda t: t.to(DEV)  # noqa: E731
    row, slot = _tokens(g, rows, 3, 64)
    table = page_table([4] * 3, 4, 12, g)
    pos, rstd = torch.randint(0, 30, (rows, 3), generator=g), torch.rand(rows, generator=g) + 0.5
    for kv, gains in ((2, (1 + 0.2 * _rand(g, D), 1 + 0.2 * _rand(g, D))), (6, None)):
        qkv = _rand(g, rows, (heads + 2 * kv) * D)
        q = [torch.zeros(rows, heads, D, dtype=BF, device=DEV) for _ in range(2)]
        cache = [torch.zeros(3, kv, 64, D, dtype=BF, device=DEV) for _ in range(2)]
        pools = [torch.zeros(12, kv, page, D, dtype=BF, device=DEV) for _ in range(2)]
        extra = {}
        if gains:
            K().qk_norm_rope_cache(dev(qkv), dev(rstd), dev(pos), dev(tab), geom, dev(gains[0]),
                                   dev(gains[1]), 1e-5, dev(row), dev(slot), 0.3, q[0], *cache)
            extra = dict(q_gamma=dev(gains[0]), k_gamma=dev(gains[1]), eps=1e-5)
        else:
            K().qkv_rope_cache_packed(dev(qkv), dev(rstd), dev(pos), dev(tab), geom, dev(row),
                                      dev(slot), heads, 0.3, q[0], *cache)
        K().rope_cache_paged(dev(qkv), dev(rstd), dev(pos), dev(tab), geom, dev(row), dev(slot),
                             dev(table), 0.3, q[1], *pools, **extra)
        assert torch.equal(q[0].view(-1), q[1].view(-1))
        rows_out = [torch.zeros_like(c) for c in cache]
        K().paged_rows(*pools, dev(table), i32([0] * 3), i32([64] * 3), *rows_out)
        assert torch.equal(rows_out[0], cache[0]) and torch.equal(rows_out[1], cache[1])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D,heads,kv", [(64, 12, 4), (128, 10, 5)])
def test_append_fp4_with_norms(dtype, D, heads, kv):
    """Normed heads in 4 bits: within half a step of the formula's values, by a power that is the
    formula's but where its largest value lies at a border of two."""
    g = _gen(D + kv)
    rows, page, n_seq = 150, 32, 3
    qkv = _rand(g, rows, (heads + 2 * kv) * D, std=3.0)
    rstd = torch.rand(rows, generator=g) + 0.3
    pos = torch.randint(0, 30, (rows, 3), generator=g)
    tab, geom = _rope(D)
    gains = 1 + 0.2 * _rand(g, D), 1 + 0.2 * _rand(g, D)
    row, slot = _tokens(g, rows, n_seq, 64)
    table = page_table([2] * n_seq, 2, 6, g)
    dev = lambda t: t.to(DEV)  # noqa: E731
    pools = [torch.zeros(6, kv, page, D // 2, dtype=U8, device=DEV) for _ in range(2)]
    scales = [torch.zeros(6, kv, page, D // 32, dtype=U8, device=DEV) for _ in range(2)]
    q = torch.zeros(rows, heads, D, dtype=dtype, device=DEV)
    K().rope_cache_paged(dev(qkv), dev(rstd), dev(pos), dev(tab), geom, dev(row), dev(slot),
                         dev(table), 0.5, q, *pools, k_scale=scales[0], v_scale=scales[1],
                         q_gamma=dev(gains[0]), k_gamma=dev(gains[1]))
    refs = _qk_norm_reference(qkv, rstd, pos, tab, geom, *gains, 1e-5, heads, kv, D, 0.5)
    half = HALF_STEP[dtype]
    _check(q, refs[0][0], refs[0][1] * (1 + half) + half * refs[0][0].abs() + 1e-30, "q")
    number, at = table[row.long(), slot.long() // page].long(), slot.long() % page
    for pool, scale, (ref, err) in zip(pools, scales, refs[1:]):
        codes, power = pool.cpu()[number, :, at], scale.cpu()[number, :, at]
        step = torch.pow(2.0, power.double() - 127).repeat_interleave(32, -1)
        size = ref.abs() / step
        _check(from_fp4(codes, power), ref,
               err + step * torch.where(size < 2, 0.25, torch.where(size < 4, 0.5, 1.0)) *
               (1 + 2.0 ** -20), "pages")
        top = ref.unflatten(-1, (-1, 32)).abs().amax(-1) / torch.pow(2.0, power.double() - 127)
        assert bool(((top < 7 * (1 + 2.0 ** -18)) & (top > 3.5 * (1 - 2.0 ** -18))).all())


@pytest.mark.parametrize("source", [F32, BF])
def test_append_fp4_edges(source):
    """Borders between numbers, groups of zeros, the smallest and largest powers, and values that are
    not finite, which make their 32 channels NaN and no others."""
    D, kv, page = 64, 1, 16
    rows = []
    ticks = torch.tensor([0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, 6.875, -0.25, -0.75, -1.25, -1.75,
                          -2.5, -3.5, -5, -6.5, 0.2422, 0.2578, 0.74, 0.76, 1.23, 1.27, 1.73, 1.77,
                          2.47, 2.53, 3.45, 3.55, 4.9, 5.1])
    for k in (0, -20, 31, -98, -101, -126, 100, 124, 125):
        rows.append(torch.cat([ticks * 2.0 ** k, torch.zeros(32)]))
    rows.append(torch.cat([-torch.zeros(32), torch.full((32,), 7.0)]))
    rows.append(torch.cat([torch.full((32,), 3.3e38), torch.full((32,), -1e-45)]))
    for bad in (float("nan"), float("inf"), float("-inf")):
        t = torch.cat([ticks, ticks / 3])
        t[40] = bad
        rows.append(t)
    v = torch.stack(rows).to(source)
    n = len(v)
    qkv = torch.cat([torch.zeros(n, D), v.float(), v.float()], 1).to(source)
    tab, geom = _line(D, 4)
    pos = torch.zeros(n, 3, dtype=torch.int64)     # no rotation: cos 1, sin 0
    pools = [torch.zeros(1, kv, page, D // 2, dtype=U8, device=DEV) for _ in range(2)]
    scales = [torch.zeros(1, kv, page, D // 32, dtype=U8, device=DEV) for _ in range(2)]
    q = torch.zeros(n, 1, D, dtype=BF, device=DEV)
    K().rope_cache_paged(qkv.to(DEV), None, pos.to(DEV), tab.to(DEV), geom, i32([0] * n),
                         i32(list(range(n))), i32([[0]]), 1.0, q, *pools, k_scale=scales[0],
                         v_scale=scales[1])
    codes, power = to_fp4(v.float())
    good = power != 255
    for i in range(2):
        assert torch.equal(scales[i][0, 0, :n].cpu()[:, good.all(0)], power[:, good.all(0)])
        got, want = pools[i][0, 0, :n].cpu(), codes
        rot = i == 0 and not bool(torch.isfinite(v).all())
        same = torch.isfinite(v.float()).all(1) if rot else torch.ones(n, dtype=torch.bool)
        assert torch.equal(scales[i][0, 0, :n].cpu()[same], power[same])
        # a zero's sign: the rotation makes -0 a 0
        assert torch.equal(from_fp4(got, power)[same].nan_to_num(9e9),
                           from_fp4(want, power)[same].nan_to_num(9e9))
    out = [torch.zeros(1, kv, page, D, dtype=F32, device=DEV) for _ in range(2)]
    K().paged_rows(*pools, i32([[0]]), i32([0]), i32([n]), *out, k_scale=scales[0],
                   v_scale=scales[1])
    assert torch.equal(out[1][0, 0, :n].cpu().double().nan_to_num(9e9),
                       from_fp4(codes, power).nan_to_num(9e9))
    assert bool(torch.isnan(out[0][0, 0, n - 3:n, 32:]).all())
    assert bool(torch.isfinite(out[0][0, 0, n - 3:n, :32]).all())


@pytest.mark.parametrize("dtype,fp4", [(BF, False), (F32, False), (BF, True), (F32, True)])
@pytest.mark.parametrize("D,page,run", [(64, 16, 1), (64, 48, 333), (128, 64, 90), (128, 16, 1100)])
def test_rows(dtype, fp4, D, page, run):
    """Runs that start anywhere, are longer than the rows, are empty, reach outside the table or lie
    in pages that are not there: such rows stay."""
    c = Paged(6, dtype, D, 3, 3, [1] * 6, [0, 5, 700, 1300, 64, 200], page=page, fp4=fp4)
    g = _gen(run)
    slots = c.table.shape[1] * page
    k, v, ks, vs = c.pools()
    start = [0, 3, 650, -7, slots - 2, 100]
    count = [1, 0, run + 5, run, 9, -3]
    table = c.table.clone()
    table[2, 650 // page] = 10 ** 6
    c.keys = [slots] * 6
    out = [torch.full((6, 3, run, D), 7.0, dtype=dtype, device=DEV) for _ in range(2)]
    K().paged_rows(k, v, table.to(DEV), i32(start), i32(count), *out, k_scale=ks, v_scale=vs)
    for pool, scale, got in ((k, ks, out[0]), (v, vs, out[1])):
        pool, want = pool.cpu(), torch.full((6, 3, run, D), 7.0, dtype=dtype)
        if fp4:
            pool = from_fp4(pool, scale.cpu()).to(dtype)
        for s in range(6):
            for i in range(min(count[s], run)):
                j = start[s] + i
                if 0 <= j < slots and 0 <= table[s, j // page] < len(pool):
                    want[s, :, i] = pool[table[s, j // page], :, j % page]
        assert torch.equal(got.cpu().double().nan_to_num(9e9), want.double().nan_to_num(9e9))
    assert g is not None


# ---- together ----------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,fp4", [(BF, False), (F32, False), (BF, True), (F32, True)])
def test_prompts_then_sampled_steps(dtype, fp4):
    """Two prompts into pages, then sampled decode steps captured in a graph: append, attention, the
    tokens' logits, the next token.  The rows take a page on the way.  Against the same in 64 bits on
    the values that the pages hold, and against eager steps, bit for bit."""
    kern = K()
    D, heads, kv, page, prompts, steps, vocab = 64, 6, 2, 16, [40, 75], 9, 300
    width, d = (heads + 2 * kv) * D, heads * D
    g = _gen(21)
    tab, geom = (t.to(DEV) if torch.is_tensor(t) else t for t in _line(D, 200))
    qs = LOG2E / math.sqrt(D)
    embed, head = _rand(g, vocab, width).to(DEV), (_rand(g, vocab, d) / 3).to(DEV)
    n_pages, tokens = 20, sum(prompts)
    table = page_table([7, 7], 7, n_pages, g).to(DEV)
    wide = D // 2 if fp4 else D
    kind = U8 if fp4 else dtype
    uniform = torch.rand(steps, 2, generator=g).to(DEV)
    prompt = torch.randint(0, vocab, (tokens,), generator=g).to(DEV)

    def serve(graphed):
        pools = [torch.zeros(n_pages, kv, page, wide, dtype=kind, device=DEV) for _ in range(2)]
        scales = ([torch.zeros(n_pages, kv, page, 2, dtype=U8, device=DEV) for _ in range(2)]
                  if fp4 else [None, None])
        more = dict(k_scale=scales[0], v_scale=scales[1])
        slot = torch.cat([torch.arange(n) for n in prompts])
        row = torch.repeat_interleave(torch.arange(2), torch.tensor(prompts))
        pos = torch.zeros(tokens, 3, dtype=torch.int64)
        pos[:, 0] = slot
        q = torch.zeros(tokens, heads, D, dtype=dtype, device=DEV)
        out = torch.zeros_like(q)
        ws = torch.empty(kern.attn_paged_workspace_bytes(q, pools[0], table, 75) // 4, device=DEV)
        kern.rope_cache_paged(embed[prompt], None, pos.to(DEV), tab, geom, row.int().to(DEV),
                              slot.int().to(DEV), table, qs, q, *pools, **more)
        kern.attn_paged(q, *pools, table, i32([0, 40, 115]), i32(prompts), 75, out, workspace=ws,
                        **more)
        seen = [(q.clone(), out.clone())]
        # the step's state, all on the device
        token = torch.zeros(2, dtype=torch.int64, device=DEV)
        logp = torch.zeros(2, device=DEV)
        lens, u = i32(prompts), torch.zeros(2, device=DEV)
        at, pos1 = i32(prompts), torch.zeros(2, 3, dtype=torch.int64, device=DEV)
        q1 = torch.zeros(2, heads, D, dtype=dtype, device=DEV)
        out1, rows1, off1 = torch.zeros_like(q1), i32([0, 1]), i32([0, 1, 2])
        ws1 = torch.empty(kern.attn_paged_workspace_bytes(q1, pools[0], table, 1) // 4, device=DEV)
        heat, k, p = torch.full((2,), 0.9, device=DEV), i32([40, 0]), torch.tensor(
            [0.95, 0.8], device=DEV)

        def choose(x):
            kern.sample_tokens((x.float().view(2, d)[:, None] * head).sum(-1), u, token, heat, k, p,
                               logprob_out=logp)

        def step():
            kern.rope_cache_paged(embed[token], None, pos1, tab, geom, rows1, at, table, qs, q1,
                                  *pools, **more)
            lens.add_(1)
            kern.attn_paged(q1, *pools, table, off1, lens, 1, out1, workspace=ws1, **more)
            choose(out1)
            at.add_(1)
            pos1[:, 0].add_(1)

        pos1[:, 0] = at
        u.copy_(uniform[0])
        choose(out[[39, 114]])
        if graphed:
            # warm-up on copies of nothing: a step that lands behind the rows' keys, then undone
            keep = [t.clone() for t in (*pools, token, lens, at, pos1)]
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
            torch.cuda.current_stream().wait_stream(side)
            for t, old in zip((*pools, token, lens, at, pos1), keep):
                t.copy_(old)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        for i in range(1, steps):
            u.copy_(uniform[i])
            before = token.clone()
            graph.replay() if graphed else step()
            torch.cuda.synchronize()
            seen.append((q1.clone(), out1.clone(), before, token.clone(), logp.clone()))
        full = [torch.zeros(2, kv, 112, D, dtype=dtype, device=DEV) for _ in range(2)]
        kern.paged_rows(*pools, table, i32([0, 0]), lens, *full, **more)
        return seen, full, lens.tolist()

    eager, (k, v), lens = serve(False)
    again, (k2, v2), _ = serve(True)
    assert torch.equal(k, k2) and torch.equal(v, v2)
    for a, b in zip(eager, again):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert lens == [n + steps - 1 for n in prompts]

    def attend(q, b, limit):
        r = heads // kv
        o = [_attend(q[:, h].cpu(), k[b, h // r].cpu(), v[b, h // r].cpu(), limit)
             for h in range(heads)]
        return (torch.stack([x[0] for x in o], 1),
                torch.stack([_bound(*x, max(limit), dtype) for x in o], 1))
    q, out = eager[0]
    for b, (a, e) in enumerate(((0, 40), (40, 115))):
        _check(out[a:e], *attend(q[a:e], b, list(range(1, e - a + 1))), "prompt")
    for i, (q, out, before, token, logp) in enumerate(eager[1:], 1):
        for b in range(2):
            _check(out[b:b + 1], *attend(q[b:b + 1], b, [prompts[b] + i]), "step")
    assert len({tuple(s[3].tolist()) for s in eager[1:]}) > 2
