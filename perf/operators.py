"""The attention operators of layers with grouped key / value heads, as measurable cases.

Three operators, each through the entry point that a program calls:

  qk_norm  ``kernels.qk_norm_rope_cache``: RMS norms of each query and key head, the rotation by
           the token's position, the split of the qkv projection and the write into the cache.
  grouped  ``kernels.attn_grouped``: attention of packed sequences of different lengths over their
           cache rows, causal, several query heads to a key / value head; a sequence may continue a
           context that is in the cache already.
  shared   ``kernels.attn_decode_shared``: one token a row, rows of a group behind one common
           prefix (the samples of a prompt), then the slots that a row wrote itself.

Formats are the framework's: q carries the softmax scale times log2(e), so weights are powers of
two; caches are [rows, kv heads, slots, head dim]; a packed list holds the tokens of all sequences
one behind the other.  Positions are (column, row, layer) of an ARC grid or plain token indexes.
"""

import math

import torch

own = False   # True: the framework's kernels; False: the same from elementary torch operations

LOG2E = 1.4426950408889634
EPS = 1e-5
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
WIDTH = {"bf16": 2, "f32": 4}


def listed():
    return [
        # sampling step of 16 rows, 12 heads on 4 kv heads: a handful of kilobytes, all latency
        dict(name="qk_norm_step", op="qk_norm", source="f32", dtype="bf16", head_dim=64, heads=12,
             kv_heads=4, batch=16, longest=1, spread=0.0, past=811, axes="grid"),
        # a batch of 64 ragged prompts in fp32 (the fp32 form's cache)
        dict(name="qk_norm_f32", op="qk_norm", source="f32", dtype="f32", head_dim=64, heads=12,
             kv_heads=12, batch=64, longest=731, spread=0.3, past=0, axes="grid"),
        # long prompts of a wide model: bf16 projection output, plain positions
        dict(name="qk_norm_long", op="qk_norm", source="bf16", dtype="bf16", head_dim=128,
             heads=32, kv_heads=8, batch=8, longest=5203, spread=0.1, past=0, axes="line"),
        # three short continuations of a cached context: few queries, many keys
        dict(name="grouped_few", op="grouped", dtype="bf16", head_dim=128, heads=32, kv_heads=8,
             batch=3, longest=17, spread=0.9, past=4099, tail=0),
        # a chunk of 16 augmentations' prompts
        dict(name="grouped_chunk", op="grouped", dtype="bf16", head_dim=64, heads=12, kv_heads=4,
             batch=16, longest=1203, spread=0.3, past=0, tail=5),
        # the same in fp32, as many kv heads as heads
        dict(name="grouped_f32", op="grouped", dtype="f32", head_dim=64, heads=12, kv_heads=12,
             batch=16, longest=811, spread=0.3, past=0, tail=0),
        # two long prompts of a wide model
        dict(name="grouped_long", op="grouped", dtype="bf16", head_dim=128, heads=32, kv_heads=8,
             batch=2, longest=8192, spread=0.2, past=0, tail=0),
        # eight samples of one task's prompt, heads of their own
        dict(name="shared_few", op="shared", dtype="bf16", head_dim=64, heads=12, kv_heads=12,
             batch=8, prefixes=1, prefix=731, new=57, spread=0.2),
        # fp32 samples of two prompts
        dict(name="shared_f32", op="shared", dtype="f32", head_dim=64, heads=12, kv_heads=4,
             batch=16, prefixes=2, prefix=1203, new=120, spread=0.3),
        # 256 samples of five prompts of different lengths, late in the output
        dict(name="shared_batch", op="shared", dtype="bf16", head_dim=64, heads=16, kv_heads=16,
             batch=256, prefixes=5, prefix=1763, new=900, spread=0.75),
        # 64 samples behind one long context of a wide model
        dict(name="shared_long", op="shared", dtype="bf16", head_dim=128, heads=32, kv_heads=8,
             batch=64, prefixes=1, prefix=32749, new=333, spread=0.5),
    ]


# a drawn case's most: those of the largest listed case of its operator
MOST = {"qk_norm": {"bytes": 9.5e8}, "grouped": {"flops": 9.7e11}, "shared": {"bytes": 6.1e8}}


def _log(rng, lo, hi):
    return round(math.exp(rng.uniform(math.log(lo), math.log(hi))))


def draw(rng):
    while True:
        op = rng.choice(["qk_norm", "grouped", "grouped", "shared", "shared"])
        dtype = rng.choice(["bf16", "bf16", "f32"])
        kv_heads = rng.choice([1, 2, 3, 4, 5, 8, 12])
        case = dict(op=op, dtype=dtype, head_dim=rng.choice([64, 128]), kv_heads=kv_heads,
                    heads=kv_heads * rng.choice([1, 1, 2, 3, 4, 5, 8, 16]))
        if op == "qk_norm":
            case.update(source=rng.choice(["f32", "bf16"]), axes=rng.choice(["grid", "line"]),
                        batch=_log(rng, 1, 256), longest=_log(rng, 1, 8000),
                        past=rng.choice([0, _log(rng, 1, 4000)]))
        elif op == "grouped":
            case.update(batch=_log(rng, 1, 64), longest=_log(rng, 1, 8192),
                        past=rng.choice([0, 0, _log(rng, 1, 20000)]), tail=rng.choice([0, 0, 7]))
        else:
            case.update(batch=_log(rng, 1, 256), prefixes=_log(rng, 1, 8),
                        prefix=_log(rng, 1, 33000), new=_log(rng, 1, 1500))
            case["prefixes"] = min(case["prefixes"], case["batch"])
        case["spread"] = round(rng.uniform(0.0, 0.9), 2)
        w, held = work(case), _held(case)
        if all(w[k] <= most for k, most in MOST[op].items()) and held <= 8e9 and (
                dtype == "bf16" or w["flops"] <= 1e11):
            return case


# ---- sizes -------------------------------------------------------------------------------------

def _lengths(n, longest, spread, least):
    """n lengths: the first is the longest, the others lie at or below it."""
    return [max(least, longest - int(spread * longest * math.fmod(0.618034 * b, 1.0)))
            for b in range(n)]


def _shape(case):
    return case["heads"], case["kv_heads"], case["head_dim"], WIDTH[case["dtype"]]


def _sequences(case):
    """Queries and cached keys of each sequence."""
    n = _lengths(case["batch"], case["longest"], case["spread"], 1)
    past = _lengths(case["batch"], case["past"], case["spread"], 0)
    return n, [p + q for p, q in zip(past, n)]


def _groups(case):
    """First row of each group (and the end), prefix lengths, own lengths of the rows."""
    p, b = case["prefixes"], case["batch"]
    size = _lengths(p, 100, 0.6, 1)
    edges = [round(b * sum(size[:i]) / sum(size)) for i in range(p + 1)]
    return (edges, _lengths(p, case["prefix"], case["spread"], 1),
            _lengths(b, case["new"], case["spread"], 1))


def _slots(longest):
    return longest + 37


def _held(case):
    """Bytes of a state's caches, which the lengths fill in part."""
    _, kv, d, w = _shape(case)
    if case["op"] == "shared":
        return 2 * kv * d * w * (case["prefixes"] * _slots(case["prefix"]) +
                                 case["batch"] * _slots(case["new"]))
    return 2 * kv * d * w * case["batch"] * _slots(case["longest"] + case["past"])


def work(case):
    h, kv, d, w = _shape(case)
    if case["op"] == "qk_norm":
        rows = sum(_lengths(case["batch"], case["longest"], case["spread"], 1))
        values = rows * (h + 2 * kv) * d
        return {"bytes": values * (WIDTH[case["source"]] + w) + rows * (4 + 24 + 8),
                "flops": 8 * rows * (h + kv) * d}
    if case["op"] == "grouped":
        n, keys = _sequences(case)
        pairs = sum(q * (k - q) + q * (q + 1) / 2 for q, k in zip(n, keys))
        return {"bytes": (2 * sum(n) * h + 2 * sum(keys) * kv) * d * w,
                "flops": 4 * d * h * pairs}
    edges, prefix, new = _groups(case)
    rows = [b - a for a, b in zip(edges, edges[1:])]
    pairs = sum(r * p for r, p in zip(rows, prefix)) + sum(new)
    return {"bytes": (2 * case["batch"] * h + 2 * kv * (sum(prefix) + sum(new))) * d * w,
            "flops": 4 * d * h * pairs}


# ---- inputs ------------------------------------------------------------------------------------

def _axes(case, longest):
    """Positions and rotation pairs of the x, y and z axes."""
    pairs = case["head_dim"] // 2
    if case["axes"] == "line":
        return (longest, 1, 1), (pairs, 0, 0)
    third = pairs // 3
    return (32, 32, 8), (third, third, pairs - 2 * third)


def _table(sizes, pairs):
    """fp32 [cos_x|sin_x|cos_y|sin_y|cos_z|sin_z], the framework's rotation table."""
    parts = []
    for n, p in zip(sizes, pairs):
        freq = 10000.0 ** (-torch.arange(p, dtype=torch.float64, device="cuda") / max(p, 1))
        angle = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * freq
        parts += [angle.cos().reshape(-1), angle.sin().reshape(-1)]
    return torch.cat(parts).float()


def prepare(case, seed):
    """Inputs, buffers and host lengths that a serving program holds at the call."""
    g = torch.Generator("cuda").manual_seed(seed)
    h, kv, d, _ = _shape(case)
    dt = TYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, dtype=dt):
        t = torch.empty(*shape, dtype=torch.float32, device="cuda")
        return t.normal_(mean, std, generator=g).to(dtype)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    if case["op"] == "qk_norm":
        n, keys = _sequences(case)
        rows, slots = sum(n), _slots(case["longest"] + case["past"])
        sizes, pairs = _axes(case, slots)
        token_row = torch.repeat_interleave(torch.arange(len(n)), torch.tensor(n))
        slot = torch.cat([torch.arange(k - q, k) for q, k in zip(n, keys)])
        if case["axes"] == "line":
            pos = torch.stack([slot, 0 * slot, 0 * slot], 1).cuda()
        else:
            pos = torch.stack([torch.randint(0, m, (rows,), device="cuda", generator=g)
                               for m in (31, 30, 5)], 1)
        return dict(case=case, qkv=normal(rows, (h + 2 * kv) * d, dtype=TYPES[case["source"]]),
                    rstd=normal(rows, std=0.1, mean=1.0, dtype=torch.float32).abs(), pos=pos,
                    tab=_table(sizes, pairs), sizes=sizes, pairs=pairs,
                    gq=normal(d, std=0.1, mean=1.0, dtype=torch.float32),
                    gk=normal(d, std=0.1, mean=1.0, dtype=torch.float32),
                    row=token_row.int().cuda(), slot=slot.int().cuda(),
                    q_scale=LOG2E / math.sqrt(d),
                    q=torch.zeros(rows, h, d, dtype=dt, device="cuda"),
                    k=torch.zeros(len(n), kv, slots, d, dtype=dt, device="cuda"),
                    v=torch.zeros(len(n), kv, slots, d, dtype=dt, device="cuda"))
    if case["op"] == "grouped":
        n, keys = _sequences(case)
        rows, slots = sum(n) + case.get("tail", 0), _slots(case["longest"] + case["past"])
        state = dict(case=case, q=normal(rows, h, d, std=LOG2E / math.sqrt(d)),
                     k=normal(len(n), kv, slots, d), v=normal(len(n), kv, slots, d, std=0.7),
                     n=n, keys=keys, offset=ints([sum(n[:i]) for i in range(len(n) + 1)]),
                     kv_len=ints(keys), out=torch.zeros(rows, h, d, dtype=dt, device="cuda"))
        if own:
            from mdlarc_scale_amd import kernels as K
            state["ws"] = torch.empty(K.attn_grouped_workspace_bytes(
                state["q"], state["k"], max(n)) // 4, device="cuda")
        return state
    edges, prefix, new = _groups(case)
    b, rows = case["batch"], max(e - a for a, e in zip(edges, edges[1:]))
    p_slots, slots = _slots(case["prefix"]), _slots(case["new"])
    state = dict(case=case, q=normal(b, h, d, std=LOG2E / math.sqrt(d)), edges=edges,
                 prefix=prefix, new=new, max_rows=rows, offset=ints(edges),
                 pk=normal(len(prefix), kv, p_slots, d),
                 pv=normal(len(prefix), kv, p_slots, d, std=0.7), p_len=ints(prefix),
                 k=normal(b, kv, slots, d), v=normal(b, kv, slots, d, std=0.7), kv_len=ints(new),
                 out=torch.zeros(b, h, d, dtype=dt, device="cuda"))
    if own:
        from mdlarc_scale_amd import kernels as K
        state["ws"] = torch.empty(K.attn_decode_shared_workspace_bytes(
            state["q"], state["pk"], state["k"], rows) // 4, device="cuda")
    return state


# ---- one pass ----------------------------------------------------------------------------------

def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        return {"qk_norm": _plain_norm, "grouped": _plain_grouped, "shared": _plain_shared}[op](s)
    from mdlarc_scale_amd import kernels as K
    if op == "qk_norm":
        K.qk_norm_rope_cache(s["qkv"], s["rstd"], s["pos"], s["tab"], s["sizes"] + s["pairs"],
                             s["gq"], s["gk"], EPS, s["row"], s["slot"], s["q_scale"], s["q"],
                             s["k"], s["v"])
        return s["q"], s["k"], s["v"]
    if op == "grouped":
        K.attn_grouped(s["q"], s["k"], s["v"], s["offset"], s["kv_len"], max(s["n"]), s["out"],
                       workspace=s["ws"])
    else:
        K.attn_decode_shared(s["q"], s["pk"], s["pv"], s["offset"], s["p_len"], s["max_rows"],
                             s["k"], s["v"], s["kv_len"], s["out"], s["ws"])
    return s["out"]


def _angles(s):
    """cos and sin of each token's pairs, [rows, 1, pairs]."""
    cos, sin, at = [], [], 0
    for axis, (n, p) in enumerate(zip(s["sizes"], s["pairs"])):
        i = s["pos"][:, axis].clamp(0, n - 1)
        cos.append(s["tab"][at:at + n * p].view(n, p)[i])
        sin.append(s["tab"][at + n * p:at + 2 * n * p].view(n, p)[i])
        at += 2 * n * p
    return torch.cat(cos, 1)[:, None], torch.cat(sin, 1)[:, None]


def _plain_norm(s):
    h, kv, d, _ = _shape(s["case"])
    y = s["qkv"].float().view(-1, h + 2 * kv, d) * s["rstd"][:, None, None]
    cos, sin = _angles(s)

    def rotated(t, gain):
        t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS) * gain
        a, b = t[..., 0::2], t[..., 1::2]
        return torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)

    dt = s["q"].dtype
    s["q"].copy_((rotated(y[:, :h], s["gq"]) * s["q_scale"]).to(dt))
    row, slot = s["row"].long(), s["slot"].long()
    s["k"][row, :, slot] = rotated(y[:, h:h + kv], s["gk"]).to(dt)
    s["v"][row, :, slot] = y[:, h + kv:].to(dt)
    return s["q"], s["k"], s["v"]


def _weighted(scores, seen, v):
    """sum 2^s v / sum 2^s over the seen keys; zero where none is."""
    scores = torch.where(seen, scores, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    w = torch.exp2(scores - torch.where(top == float("-inf"), 0.0, top))
    total = w.sum(-1, keepdim=True)
    return (w @ v) / torch.where(total == 0, 1.0, total)


def _plain_grouped(s):
    h, kv, d, _ = _shape(s["case"])
    r, at = h // kv, 0
    for b, (n, keys) in enumerate(zip(s["n"], s["keys"])):
        seen = (torch.arange(keys, device="cuda")[None] <=
                keys - n + torch.arange(n, device="cuda")[:, None])
        seen = seen.repeat_interleave(r, 0)
        for j in range(kv):
            q = s["q"][at:at + n, j * r:(j + 1) * r].float().reshape(n * r, d)
            o = _weighted(q @ s["k"][b, j, :keys].float().T, seen, s["v"][b, j, :keys].float())
            s["out"][at:at + n, j * r:(j + 1) * r] = o.view(n, r, d).to(s["out"].dtype)
        at += n
    return s["out"]


def _plain_shared(s):
    h, kv, d, _ = _shape(s["case"])
    r, longest = h // kv, max(s["new"])
    mine = torch.arange(longest, device="cuda")[None] < s["kv_len"][:, None]
    for p, n in enumerate(s["prefix"]):
        a, e = s["edges"][p], s["edges"][p + 1]
        if a == e:
            continue
        for j in range(kv):
            q = s["q"][a:e, j * r:(j + 1) * r].float()                       # [rows, r, d]
            front = q.reshape(-1, d) @ s["pk"][p, j, :n].float().T
            keys = s["k"][a:e, j, :longest].float().transpose(1, 2).contiguous()
            back = torch.where(mine[a:e, None], q @ keys, float("-inf"))     # [rows, r, longest]
            front = front.view(e - a, r, n)
            top = torch.maximum(front.amax(-1, keepdim=True), back.amax(-1, keepdim=True))
            wf, wb = torch.exp2(front - top), torch.exp2(back - top)
            values = torch.where(mine[a:e, :, None], s["v"][a:e, j, :longest].float(), 0.0)
            o = (wf.view(-1, n) @ s["pv"][p, j, :n].float()).view(e - a, r, d) + wb @ values
            o = o / (wf.sum(-1, keepdim=True) + wb.sum(-1, keepdim=True))
            s["out"][a:e, j * r:(j + 1) * r] = o.to(s["out"].dtype)
    return s["out"]


# ---- the definition in 64 bits -----------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    h, kv, d, _ = _shape(case)
    if case["op"] == "qk_norm":
        x = s["qkv"].double() * s["rstd"].double()[:, None]
        x = x.view(len(x), h + 2 * kv, d)
        table, turn, at = s["tab"].double(), [], 0
        for i, (n, p) in enumerate(zip(s["sizes"], s["pairs"])):
            c, sn = table[at:at + 2 * n * p].view(2, n, p).unbind(0)
            turn.append(torch.complex(c, sn)[s["pos"][:, i]])
            at += 2 * n * p
        turn = torch.cat(turn, -1).unsqueeze(1)
        heads = x[:, :h + kv]
        gain = torch.cat([s["gq"].double().expand(h, d) * s["q_scale"],
                          s["gk"].double().expand(kv, d)])
        heads = heads * (heads.square().sum(-1, keepdim=True) / d + EPS).rsqrt() * gain
        heads = torch.view_as_complex(heads.unflatten(-1, (d // 2, 2)).contiguous()) * turn
        heads = torch.view_as_real(heads).flatten(-2)
        k, v = s["k"].double(), s["v"].double()
        k[s["row"].long(), :, s["slot"].long()] = heads[:, h:]
        v[s["row"].long(), :, s["slot"].long()] = x[:, h + kv:]
        return heads[:, :h].contiguous(), k, v
    out = s["out"].double()
    if case["op"] == "grouped":
        pieces = [(b, first, last) for b, (first, last) in enumerate(
            zip(s["offset"].tolist(), s["offset"].tolist()[1:]))]
        for b, first, last in pieces:
            n_keys = s["keys"][b]
            for head in range(h):
                k = s["k"][b, head * kv // h, :n_keys].double()
                v = s["v"][b, head * kv // h, :n_keys].double()
                for i in range(first, last, 2048):
                    q = s["q"][i:min(i + 2048, last), head].double()
                    e = q @ k.t()
                    ahead = n_keys - last + i + 1          # keys that row i sees
                    e.masked_fill_(torch.ones_like(e, dtype=torch.bool).triu_(ahead),
                                   float("-inf"))
                    out[i:i + len(q), head] = torch.softmax(e * math.log(2.0), -1) @ v
        return out
    for p, n in enumerate(s["prefix"]):
        for b in range(s["edges"][p], s["edges"][p + 1]):
            q = s["q"][b].double().view(kv, h // kv, d)
            k = torch.cat([s["pk"][p, :, :n], s["k"][b, :, :s["new"][b]]], 1).double()
            v = torch.cat([s["pv"][p, :, :n], s["v"][b, :, :s["new"][b]]], 1).double()
            e = torch.matmul(q, k.transpose(1, 2).contiguous()) * math.log(2.0)
            out[b] = torch.matmul(torch.softmax(e, -1), v).view(h, d)
    return out
