"""The operators of a paged cache and of sampling, as measurable cases.

Four operators, each through the entry points that a program calls:

  write   ``kernels.rope_cache_paged``: the split of the qkv projection, the rotation by the token's
          position (and the heads' RMS norms, where a layer has them) and the append of keys and
          values to the pages of their sequences, in bf16, fp32 or 4 bits.
  read    ``kernels.paged_rows``: a run of each sequence's slots out of its pages, as rows.
  attend  ``kernels.attn_paged``: attention of packed sequences (single tokens, continuations, whole
          prompts) over their pages.
  sample  ``kernels.sample_tokens``: a token a row from logits, with temperature, top-k, top-p and
          min-p, from given random numbers.

Formats are the framework's: q carries the softmax scale times log2(e), so weights are powers of
two.  Pages are [pages, kv heads, slots of a page, head dim]; slot j of sequence s is slot j % P of
page table[s, j / P].  4-bit pages hold e2m1 numbers, two to a byte (the even channel in the low
half), times a power of two for 32 channels (e8m0 bytes): the smallest power by which every
magnitude of the 32 is below 7.
"""

import math

import torch

own = False   # True: the framework's kernels; False: the same from elementary torch operations

LOG2E = 1.4426950408889634
EPS = 1e-5
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
WIDTH = {"bf16": 2, "f32": 4, "fp4": 17 / 32}   # bytes of a value
SPARE_PAGES = 5                                  # of a pool, in no sequence


def listed():
    return [
        # a decode step of 16 rows, 12 heads on 4 kv heads: a handful of kilobytes, all latency
        dict(name="write_step", op="write", source="f32", pages="bf16", dtype="bf16", head_dim=64,
             heads=12, kv_heads=4, batch=16, longest=1, spread=0.0, past=811, page=16, axes="grid",
             norm=False),
        # a batch of 64 ragged prompts into 4-bit pages, and what the pages then hold of them
        dict(name="write_fp4", op="write", source="f32", pages="fp4", dtype="bf16", head_dim=64,
             heads=12, kv_heads=12, batch=64, longest=731, spread=0.3, past=0, page=32, axes="grid",
             norm=False),
        # long prompts of a wide model whose heads are normed: bf16 projection output
        dict(name="write_long", op="write", source="bf16", pages="bf16", dtype="bf16", head_dim=128,
             heads=32, kv_heads=8, batch=8, longest=5203, spread=0.1, past=0, page=64, axes="line",
             norm=True),
        # one prompt's keys and values for samples that share them
        dict(name="read_prompt", op="read", pages="bf16", dtype="bf16", head_dim=64, kv_heads=12,
             batch=1, longest=731, spread=0.0, past=0, page=16),
        # long contexts leave their 4-bit pages
        dict(name="read_fp4", op="read", pages="fp4", dtype="bf16", head_dim=128, kv_heads=8,
             batch=24, longest=16381, spread=0.5, past=3, page=64),
        # a decode step of 16 rows of an fp32 model
        dict(name="attend_f32", op="attend", pages="f32", dtype="f32", head_dim=64, heads=12,
             kv_heads=4, batch=16, longest=1, spread=0.3, past=1203, page=16, tail=0),
        # four long prompts of a wide model
        dict(name="attend_prompts", op="attend", pages="bf16", dtype="bf16", head_dim=128, heads=32,
             kv_heads=8, batch=4, longest=4096, spread=0.2, past=0, page=32, tail=5),
        # three short continuations of a cached context: few queries, many keys
        dict(name="attend_fp4_few", op="attend", pages="fp4", dtype="bf16", head_dim=128, heads=32,
             kv_heads=8, batch=3, longest=17, spread=0.5, past=4099, page=16, tail=0),
        # a decode step of 256 rows, heads of their own, late in the output
        dict(name="attend_fp4_batch", op="attend", pages="fp4", dtype="bf16", head_dim=64, heads=16,
             kv_heads=16, batch=256, longest=1, spread=0.4, past=2663, page=64, tail=0),
        # a decode step of 64 long contexts of a wide model
        dict(name="attend_fp4_long", op="attend", pages="fp4", dtype="bf16", head_dim=128, heads=32,
             kv_heads=8, batch=64, longest=1, spread=0.5, past=32749, page=64, tail=0),
        # sampled decoding of 256 rows with the ARC vocabulary
        dict(name="sample_head", op="sample", dtype="f32", batch=256, vocab=14),
        # 64 rows of a language model's vocabulary
        dict(name="sample_wide", op="sample", dtype="f32", batch=64, vocab=131072),
    ]


# a drawn case's most: those of the largest listed case of its operator
MOST = {"write": {"bytes": 9.9e8}, "read": {"bytes": 1.55e9}, "attend": {"bytes": 1.72e9,
        "flops": 4.7e11}, "sample": {"bytes": 3.36e7}}


def _log(rng, lo, hi):
    return round(math.exp(rng.uniform(math.log(lo), math.log(hi))))


def draw(rng):
    while True:
        op = rng.choice(["write", "write", "read", "attend", "attend", "attend", "sample"])
        if op == "sample":
            case = dict(op=op, dtype=rng.choice(["f32", "bf16"]), batch=_log(rng, 1, 512),
                        vocab=_log(rng, 14, 200000))
            if work(case)["bytes"] <= MOST[op]["bytes"]:
                return case
            continue
        kv_heads = rng.choice([1, 2, 3, 4, 5, 8, 12])
        pages = rng.choice(["bf16", "f32", "fp4", "fp4"])
        case = dict(op=op, pages=pages, dtype=pages if pages != "fp4" else
                    rng.choice(["bf16", "bf16", "f32"]), head_dim=rng.choice([64, 128]),
                    kv_heads=kv_heads, page=rng.choice([16, 16, 32, 48, 64, 128]),
                    spread=round(rng.uniform(0.0, 0.9), 2))
        if op != "read":
            case["heads"] = kv_heads * rng.choice([1, 1, 2, 3, 4, 5, 8, 16])
        if op == "write":
            case.update(source=rng.choice(["f32", "bf16"]), axes=rng.choice(["grid", "line"]),
                        batch=_log(rng, 1, 256), longest=_log(rng, 1, 8000),
                        past=rng.choice([0, _log(rng, 1, 4000)]),
                        norm=pages != "fp4" and rng.choice([False, True]))
        elif op == "read":
            case.update(batch=_log(rng, 1, 256), longest=_log(rng, 1, 20000),
                        past=rng.choice([0, _log(rng, 1, 4000)]))
        elif rng.choice([True, False]):
            case.update(batch=_log(rng, 1, 256), longest=1, past=_log(rng, 1, 33000), tail=0)
        else:
            case.update(batch=_log(rng, 1, 64), longest=_log(rng, 1, 4096),
                        past=rng.choice([0, 0, _log(rng, 1, 20000)]), tail=rng.choice([0, 0, 7]))
        w = work(case)
        if all(w[k] <= most for k, most in MOST[op].items()) and _dense(case) <= 9e9 and (
                op != "attend" or case["dtype"] == "bf16" or w["flops"] <= 1e10):
            return case


# ---- sizes -------------------------------------------------------------------------------------

def _lengths(n, longest, spread, least):
    """n lengths: the first is the longest, the others lie at or below it."""
    return [max(least, longest - int(spread * longest * math.fmod(0.618034 * b, 1.0)))
            for b in range(n)]


def _sequences(case):
    """New tokens and cached slots (the new ones among them) of each sequence."""
    n = _lengths(case["batch"], case["longest"], case["spread"], 1)
    past = _lengths(case["batch"], case["past"], case["spread"], 0)
    return n, [p + q for p, q in zip(past, n)]


def _dense(case):
    """Bytes of a state's pages in fp32 (that many slots for every sequence), and of the scores."""
    slots = case["batch"] * (case["longest"] + case["past"] + 64)
    scores = slots * case["longest"] * case["heads"] if case["op"] == "attend" else 0
    return max(4 * slots * case["kv_heads"] * case["head_dim"], 4 * scores)


def work(case):
    if case["op"] == "sample":
        return {"bytes": case["batch"] * (case["vocab"] * WIDTH[case["dtype"]] + 32),
                "flops": 4 * case["batch"] * case["vocab"]}
    n, keys = _sequences(case)
    kv, d, rows = case["kv_heads"], case["head_dim"], sum(n)
    w, held = WIDTH[case["dtype"]], WIDTH[case["pages"]]
    if case["op"] == "write":
        h = case["heads"]
        back = 2 * kv * (held + w) if case["pages"] == "fp4" else 0
        return {"bytes": rows * d * ((h + 2 * kv) * WIDTH[case["source"]] + h * w +
                                     2 * kv * held + back) + rows * (4 + 24 + 8),
                "flops": 8 * rows * (h + kv) * d}
    if case["op"] == "read":
        return {"bytes": 2 * rows * kv * d * (held + w), "flops": 2 * rows * kv * d}
    h = case["heads"]
    pairs = sum(q * (k - q) + q * (q + 1) / 2 for q, k in zip(n, keys))
    return {"bytes": 2 * rows * h * d * w + 2 * sum(keys) * kv * d * held,
            "flops": 4 * d * h * pairs}


# ---- 4 bits ------------------------------------------------------------------------------------

def _power(n):
    """2^n in fp32 for whole numbers -126 .. 127, exactly."""
    return ((n.int() + 127) << 23).view(torch.float32)


def _quantised(x):
    """Codes [.., D / 2] and powers [.., D / 32] of fp32 or fp64 rows [.., D] of finite values."""
    x = x.unflatten(-1, (-1, 32))
    m, e = torch.frexp(x.abs().amax(-1))
    power = torch.where(m < 0.875, e - 3, e - 2)            # 7 2^power is 0.875 2^(power + 3)
    power = torch.where(m == 0, -100, power).clamp(-100, 125)
    v = x.abs() * _power(-power)[..., None].to(x.dtype)
    code = ((v > 0.25).to(torch.uint8) + (v >= 0.75) + (v > 1.25) + (v >= 1.75) + (v > 2.5) +
            (v >= 3.5) + (v > 5) + 8 * torch.signbit(x)).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, (power + 127).to(torch.uint8)


def _values(codes, scale):
    """fp32 [.., D] of codes and powers."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
    table = torch.cat([table, -table])
    pair = torch.stack([table[(codes & 15).long()], table[(codes >> 4).long()]], -1).flatten(-2)
    return (pair.unflatten(-1, (-1, 32)) * _power(scale.int() - 127)[..., None]).flatten(-2)


# ---- inputs ------------------------------------------------------------------------------------

def _axes(case, longest):
    """Positions and rotation pairs of the x, y and z axes."""
    pairs = case["head_dim"] // 2
    if case["axes"] == "line":
        return (longest, 1, 1), (pairs, 0, 0)
    third = pairs // 3
    return (32, 32, 8), (third, third, pairs - 2 * third)


def _rope_table(sizes, pairs):
    """fp32 [cos_x|sin_x|cos_y|sin_y|cos_z|sin_z], the framework's rotation table."""
    parts = []
    for n, p in zip(sizes, pairs):
        freq = 10000.0 ** (-torch.arange(p, dtype=torch.float64, device="cuda") / max(p, 1))
        angle = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * freq
        parts += [angle.cos().reshape(-1), angle.sin().reshape(-1)]
    return torch.cat(parts).float()


def prepare(case, seed):
    """Inputs, pages and host lengths that a serving program holds at the call."""
    g = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0, dtype=torch.float32):
        t = torch.empty(*shape, dtype=torch.float32, device="cuda")
        return t.normal_(mean, std, generator=g).to(dtype)

    def uniform(n, lo, hi):
        return lo + (hi - lo) * torch.rand(n, device="cuda", generator=g)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    if case["op"] == "sample":
        b, vocab = case["batch"], case["vocab"]
        # what a head gives: a few likely tokens, a long tail, two tokens that are not allowed
        logits = normal(b, vocab, std=2.5)
        logits[:, 11:13] = float("-inf")
        kind = torch.randint(0, 4, (4, b), device="cuda", generator=g)
        return dict(case=case, logits=logits.to(TYPES[case["dtype"]]),
                    uniform=torch.rand(b, device="cuda", generator=g),
                    # a quarter of the rows without each of the filters, a few greedy
                    temperature=torch.where((kind[0] == 0) & (kind[1] == 0), 0.0,
                                            uniform(b, 0.4, 1.5)),
                    top_k=torch.where(kind[1] == 1, 0, torch.randint(
                        1, min(vocab, 1000) + 1, (b,), device="cuda", generator=g)).int(),
                    top_p=torch.where(kind[2] == 1, 1.0, uniform(b, 0.3, 0.99)),
                    min_p=torch.where(kind[3] == 1, 0.0, uniform(b, 0.0, 0.1)),
                    token=torch.zeros(b, dtype=torch.int64, device="cuda"),
                    logprob=torch.zeros(b, device="cuda"))

    n, keys = _sequences(case)
    kv, d, page = case["kv_heads"], case["head_dim"], case["page"]
    dt, rows = TYPES[case["dtype"]], sum(n)
    # each sequence's pages lie anywhere in the pool; entries that it has not reached are -1
    counts = torch.tensor([-(-k // page) for k in keys], device="cuda")
    used = int(counts.sum())
    order = torch.randperm(used + SPARE_PAGES, device="cuda", generator=g)[:used].int()
    table = torch.full((len(n), int(counts.max()) + 2), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(table.shape[1], device="cuda")[None] < counts[:, None]] = order
    s = dict(case=case, table=table, n=n, keys=keys, k_scale=None, v_scale=None)
    for name, std in (("k", 1.0), ("v", 0.7)):
        pool = normal(used + SPARE_PAGES, kv, page, d, std=std)
        if case["pages"] == "fp4":
            s[name], s[name + "_scale"] = _quantised(pool)
        else:
            s[name] = pool.to(TYPES[case["pages"]])
        del pool
    if case["op"] == "attend":
        h, tokens = case["heads"], rows + case["tail"]
        s.update(q=normal(tokens, h, d, std=LOG2E / math.sqrt(d), dtype=dt), kv_len=ints(keys),
                 offset=ints([sum(n[:i]) for i in range(len(n) + 1)]),
                 out=torch.zeros(tokens, h, d, dtype=dt, device="cuda"))
        if own:
            from mdlarc_scale_amd import kernels as K
            s["ws"] = torch.empty(K.attn_paged_workspace_bytes(s["q"], s["k"], table, max(n)) // 4,
                                  device="cuda")
        return s
    s.update(start=ints([k - q for q, k in zip(n, keys)]), count=ints(n),
             k_rows=torch.zeros(len(n), kv, max(n), d, dtype=dt, device="cuda"),
             v_rows=torch.zeros(len(n), kv, max(n), d, dtype=dt, device="cuda"))
    if case["op"] == "read":
        return s
    h = case["heads"]
    sizes, pairs = _axes(case, max(keys) + 1)
    slot = torch.cat([torch.arange(k - q, k) for q, k in zip(n, keys)])
    if case["axes"] == "line":
        pos = torch.stack([slot, 0 * slot, 0 * slot], 1).cuda()
    else:
        pos = torch.stack([torch.randint(0, m, (rows,), device="cuda", generator=g)
                           for m in (31, 30, 5)], 1)
    gain = (lambda: normal(d, std=0.1, mean=1.0)) if case["norm"] else (lambda: None)
    s.update(qkv=normal(rows, (h + 2 * kv) * d, dtype=TYPES[case["source"]]), pos=pos,
             rstd=normal(rows, std=0.1, mean=1.0).abs(), tab=_rope_table(sizes, pairs),
             sizes=sizes, pairs=pairs, gq=gain(), gk=gain(), slot=slot.int().cuda(),
             row=torch.repeat_interleave(torch.arange(len(n)), torch.tensor(n)).int().cuda(),
             q_scale=LOG2E / math.sqrt(d), q=torch.zeros(rows, h, d, dtype=dt, device="cuda"))
    return s


# ---- one pass ----------------------------------------------------------------------------------

def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        return {"write": _plain_write, "read": _plain_read, "attend": _plain_attend,
                "sample": _plain_sample}[op](s)
    from mdlarc_scale_amd import kernels as K
    if op == "sample":
        K.sample_tokens(s["logits"], s["uniform"], s["token"], s["temperature"], s["top_k"],
                        s["top_p"], s["min_p"], logprob_out=s["logprob"])
        return s["token"], s["logprob"]
    if op == "attend":
        K.attn_paged(s["q"], s["k"], s["v"], s["table"], s["offset"], s["kv_len"], max(s["n"]),
                     s["out"], workspace=s["ws"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        return s["out"]
    if op == "write":
        K.rope_cache_paged(s["qkv"], s["rstd"], s["pos"], s["tab"], s["sizes"] + s["pairs"],
                           s["row"], s["slot"], s["table"], s["q_scale"], s["q"], s["k"], s["v"],
                           k_scale=s["k_scale"], v_scale=s["v_scale"], q_gamma=s["gq"],
                           k_gamma=s["gk"], eps=EPS)
        if s["k_scale"] is None:
            return s["q"], s["k"], s["v"]
    K.paged_rows(s["k"], s["v"], s["table"], s["start"], s["count"], s["k_rows"], s["v_rows"],
                 k_scale=s["k_scale"], v_scale=s["v_scale"])
    return (s["q"], s["k_rows"], s["v_rows"]) if op == "write" else (s["k_rows"], s["v_rows"])


def _places(s):
    """Page and slot in it of each slot of the runs, and which of them there are: [rows, run]."""
    page, j = s["case"]["page"], torch.arange(max(s["n"]), device="cuda")[None]
    slot = s["start"][:, None].long() + j
    there = j < s["count"][:, None]
    at = (slot // page).clamp(max=s["table"].shape[1] - 1)
    return s["table"].long().gather(1, at).clamp(min=0), slot % page, there


def _plain_read(s):
    number, at, there = _places(s)
    for name in ("k", "v"):
        scale, rows = s[name + "_scale"], s[name + "_rows"]
        got = s[name][number, :, at]                                     # [rows, run, kv, D]
        if scale is not None:
            got = _values(got, scale[number, :, at])
        got = got.to(rows.dtype).transpose(1, 2)
        rows.copy_(torch.where(there[:, None, :, None], got, rows))
    return s["k_rows"], s["v_rows"]


def _angles(s):
    """cos and sin of each token's pairs, [rows, 1, pairs]."""
    cos, sin, at = [], [], 0
    for axis, (n, p) in enumerate(zip(s["sizes"], s["pairs"])):
        i = s["pos"][:, axis].clamp(0, n - 1)
        cos.append(s["tab"][at:at + n * p].view(n, p)[i])
        sin.append(s["tab"][at + n * p:at + 2 * n * p].view(n, p)[i])
        at += 2 * n * p
    return torch.cat(cos, 1)[:, None], torch.cat(sin, 1)[:, None]


def _plain_write(s):
    case = s["case"]
    h, kv, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    y = s["qkv"].float().view(-1, h + 2 * kv, d) * s["rstd"][:, None, None]
    cos, sin = _angles(s)

    def rotated(t, gain):
        if gain is not None:
            t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS) * gain
        a, b = t[..., 0::2], t[..., 1::2]
        # a multiply-add on a rounded product, each rounded once: exact in 64 bits, which keeps
        # values next to a border of two 4-bit numbers on their side
        wide = lambda u: u.double()  # noqa: E731
        return torch.stack((wide(a) * wide(cos) - wide(b * sin),
                            wide(b) * wide(cos) + wide(a * sin)), -1).float().flatten(-2)

    s["q"].copy_(rotated(y[:, :h], s["gq"]) * s["q_scale"])
    number = s["table"][s["row"].long(), s["slot"].long() // page].long()
    at = s["slot"].long() % page
    for name, t in (("k", rotated(y[:, h:h + kv], s["gk"])), ("v", y[:, h + kv:])):
        if s["k_scale"] is None:
            s[name][number, :, at] = t.to(s[name].dtype)
        else:
            codes, scale = _quantised(t)
            s[name][number, :, at] = codes
            s[name + "_scale"][number, :, at] = scale
    return (s["q"], s["k"], s["v"]) if s["k_scale"] is None else (s["q"],) + _plain_read(s)


def _plain_attend(s):
    case = s["case"]
    h, kv, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    b, r, width = case["batch"], h // kv, -(-max(s["keys"]) // page)
    table = s["table"][:, :width].long().clamp(min=0)

    def dense(name):                                                    # [b, kv, keys, d] in fp32
        t = s[name][table]
        t = t.float() if s[name + "_scale"] is None else _values(t, s[name + "_scale"][table])
        return t.transpose(1, 2).reshape(b, kv, width * page, d)

    n = s["offset"].diff().long()
    i, j = torch.arange(max(s["n"]), device="cuda"), torch.arange(width * page, device="cuda")
    there = i[None] < n[:, None]                                        # [b, queries]
    token = (s["offset"][:-1, None].long() + i).clamp(max=len(s["q"]) - 1)
    q = s["q"][token].float().view(b, -1, kv, r, d).transpose(1, 2).reshape(b, kv, -1, d)
    last = s["kv_len"][:, None] - n[:, None] + i                        # the last key of a query
    seen = (j <= last[..., None]) & there[..., None]                    # [b, queries, keys]
    scores = torch.matmul(q, dense("k").transpose(2, 3).contiguous()).view(b, kv, -1, r, len(j))
    scores = torch.where(seen[:, None, :, None], scores, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    scores = torch.exp2(scores - torch.where(top == float("-inf"), 0.0, top))
    total = scores.sum(-1, keepdim=True)
    values = torch.where((j < s["kv_len"][:, None])[:, None, :, None], dense("v"), 0.0)
    o = torch.matmul(scores.view(b, kv, -1, len(j)), values).view(b, kv, -1, r, d)
    o = (o / torch.where(total == 0, 1.0, total)).transpose(1, 2).reshape(b, -1, h, d)
    s["out"][token[there]] = o[there].to(s["out"].dtype)
    return s["out"]


def _plain_sample(s):
    # borders between kept and dropped tokens, and between one token and the next: 64 bits
    greedy = s["temperature"] <= 0
    z = s["logits"].double() / torch.where(greedy, 1.0, s["temperature"].double())[:, None]
    vocab = z.shape[1]
    k = torch.where(greedy, 1, torch.where(s["top_k"] <= 0, vocab, s["top_k"]).long())
    z, order = torch.sort(z, dim=-1, descending=True, stable=True)          # ties: lowest index first
    w = torch.exp(z - z[:, :1])
    w = torch.where(torch.arange(vocab, device="cuda") < k[:, None], w, 0.0)
    before = w.cumsum(-1) - w
    nucleus = before < s["top_p"].double()[:, None] * w.sum(-1, keepdim=True)
    nucleus |= (s["top_p"] >= 1)[:, None]
    nucleus[:, 0] = True
    w = torch.where(nucleus & (w >= s["min_p"].double()[:, None]), w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)
    total = w.cumsum(-1)
    token = (total <= s["uniform"].double()[:, None] * total[:, -1:]).sum(-1)
    s["token"].copy_(token)
    s["logprob"].copy_(torch.log(w.gather(1, token[:, None])[:, 0] / total[:, -1]))
    return s["token"], s["logprob"]


# ---- the definition in 64 bits -----------------------------------------------------------------

def _slots(s, name, b, first, last):
    """Slots first .. last - 1 of sequence b in float64, [kv, slots, D]."""
    page = s["case"]["page"]
    slots = torch.arange(first, last, device="cuda")
    number = s["table"][b].long()[slots // page]
    t = s[name][number, :, slots % page].transpose(0, 1)
    if s[name + "_scale"] is None:
        return t.double()
    power = s[name + "_scale"][number, :, slots % page].transpose(0, 1).double() - 127
    code = torch.stack((t & 15, t >> 4), -1).flatten(-2).double()
    size = code % 8
    # 0, 1/2, 1, 3/2, then (1 or 3/2) times 2 and 4
    size = torch.where(size < 4, size / 2, (2 + size % 2) * torch.exp2(size // 2 - 2))
    size = torch.where(code >= 8, -size, size)
    return size * torch.exp2(power).repeat_interleave(32, -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        got = []
        for b in range(case["batch"]):
            z = s["logits"][b].double()
            if s["temperature"][b] <= 0:
                got.append(0.0)
                continue
            z = z / s["temperature"][b].double()
            k, p = int(s["top_k"][b]), float(s["top_p"][b].double())
            kept = torch.sort(z, descending=True, stable=True).indices
            kept = kept[:k] if k > 0 else kept
            if p < 1:
                kept = kept[:1 + int((torch.softmax(z[kept], 0).cumsum(0) < p).sum())]
            kept = kept[z[kept] - z[kept[0]] >= torch.log(s["min_p"][b].double())]
            share = torch.log_softmax(z[kept.sort().values], 0)
            at = int((share.exp().cumsum(0) <= s["uniform"][b].double()).sum())
            got.append(float(share[min(at, len(share) - 1)]))
        return None, torch.tensor(got, dtype=torch.float64, device="cuda")
    kv, d = case["kv_heads"], case["head_dim"]
    if case["op"] == "read":
        k, v = s["k_rows"].double(), s["v_rows"].double()
        for b, (n, last) in enumerate(zip(s["n"], s["keys"])):
            k[b, :, :n], v[b, :, :n] = (_slots(s, name, b, last - n, last) for name in "kv")
        return k, v
    h = case["heads"]
    if case["op"] == "write":
        x = s["qkv"].double() * s["rstd"].double()[:, None]
        x = x.view(len(x), h + 2 * kv, d)
        table, turn, at = s["tab"].double(), [], 0
        for i, (n, p) in enumerate(zip(s["sizes"], s["pairs"])):
            c, sn = table[at:at + 2 * n * p].view(2, n, p).unbind(0)
            turn.append(torch.complex(c, sn)[s["pos"][:, i]])
            at += 2 * n * p
        heads = x[:, :h + kv]
        if case["norm"]:
            gain = torch.cat([s["gq"].double().expand(h, d), s["gk"].double().expand(kv, d)])
            heads = heads * (heads.square().sum(-1, keepdim=True) / d + EPS).rsqrt() * gain
        heads = torch.view_as_complex(heads.unflatten(-1, (d // 2, 2)).contiguous())
        heads = torch.view_as_real(heads * torch.cat(turn, -1).unsqueeze(1)).flatten(-2)
        q = heads[:, :h] * s["q_scale"]
        if case["pages"] == "fp4":
            return q, None, None
        k, v = s["k"].double(), s["v"].double()
        number = s["table"][s["row"].long(), s["slot"].long() // case["page"]].long()
        k[number, :, s["slot"].long() % case["page"]] = heads[:, h:]
        v[number, :, s["slot"].long() % case["page"]] = x[:, h + kv:]
        return q, k, v
    out = s["out"].double()
    for b, (n, keys) in enumerate(zip(s["n"], s["keys"])):
        k, v = _slots(s, "k", b, 0, keys), _slots(s, "v", b, 0, keys)
        a = int(s["offset"][b])
        for head in range(kv):
            q = s["q"][a:a + n, head * (h // kv):(head + 1) * (h // kv)].double()
            e = torch.matmul(q, k[head].t().contiguous()) * math.log(2.0)      # [n, r, keys]
            ahead = torch.arange(keys, device="cuda") > torch.arange(
                keys - n, keys, device="cuda")[:, None]
            e.masked_fill_(ahead[:, None], float("-inf"))
            out[a:a + n, head * (h // kv):(head + 1) * (h // kv)] = torch.softmax(e, -1) @ v[head]
    return out
