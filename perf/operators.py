"""Cases of the group-decode operators: what a decode step of several sequences over one prompt calls.

Four operators, in the order a step runs them:
  rotary     q/k norm, rotary positions with several axes, and the write of k/v into the page pool
  attention  decode attention of sequences that share the pages of a long prefix
  select     the best continuations over a group's beams and the vocabulary
  reorder    recurrent-state rows follow their beams

`run` computes each in a plain form (elementary torch operations in 32 bits) or, with
`own` set, through shellsmith_b200's public entry points.

The page pool is [num_pages, Hkv, 2, 16, D] bf16; the row of token t keeps its 16-byte chunk c
at chunk position c ^ (t & 7).
"""

import math

import torch

own = False

PAGE = 16
DEV = "cuda"


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One decode step of a small batch: latency counts. q and its gate leave one projection
        # (strided q), a quarter of the head rotates, three axes of positions.
        dict(name="rotary decode 8", op="rotary", tokens=8, q_heads=16, kv_heads=2, dim=256, rotary_dim=64,
             axes=3, interleaved=True, norm=True, gated=True, start=16384),
        # A full decode batch at the engine's batch limit, plain positions over the whole head.
        dict(name="rotary decode 256", op="rotary", tokens=256, q_heads=24, kv_heads=8, dim=128, rotary_dim=128,
             axes=1, interleaved=False, norm=False, gated=False, start=1000),
        # A long prompt with images, an odd token count, as packed prefill hands it over.
        dict(name="rotary prompt 16381", op="rotary", tokens=16381, q_heads=16, kv_heads=2, dim=256, rotary_dim=64,
             axes=3, interleaved=False, norm=True, gated=True, start=0),
        # Eight samples of one short prompt, just forked: latency counts.
        dict(name="attention 8 rows 2k", op="attention", groups=1, rows=8, prefix=2048, suffix=64, q_heads=16,
             kv_heads=2, dim=256),
        # The engine's batch of 64: eight prompts of about 16k tokens, eight samples of each.
        dict(name="attention 8x8 rows 16k", op="attention", groups=8, rows=8, prefix=16272, suffix=2048, q_heads=16,
             kv_heads=2, dim=256),
        # A common system prompt and tool list over a whole batch: many rows for each cached byte.
        dict(name="attention 128 rows 8k", op="attention", groups=1, rows=128, prefix=8208, suffix=1024, q_heads=16,
             kv_heads=2, dim=256),
        # Beams of three prompts on a model with narrower heads and more kv heads, odd sizes.
        dict(name="attention 3x5 rows 5k", op="attention", groups=3, rows=5, prefix=5104, suffix=777, q_heads=24,
             kv_heads=8, dim=128),
        # One request, four beams, a small vocabulary: latency counts.
        dict(name="select 1x4 32k", op="select", groups=1, beams=4, vocab=32768, n=8, dtype="bf16", finished=False),
        # A batch of requests with an odd vocabulary, fp32 logits, some beams finished.
        dict(name="select 8x5 50k fp32", op="select", groups=8, beams=5, vocab=50001, n=10, dtype="fp32",
             finished=True),
        # A large batch of beams over a large vocabulary: the logits exceed the L2 cache.
        dict(name="select 32x8 250k", op="select", groups=32, beams=8, vocab=250001, n=16, dtype="bf16",
             finished=True),
        # Four beams of one request change places: every GDN layer's fp32 state rows.
        dict(name="reorder 1x4 36 layers", op="reorder", layers=36, groups=1, beams=4, survivors=3, sources=1,
             heads=32, dtype="fp32"),
        # Four requests of eight beams, half of the beams die.
        dict(name="reorder 4x8 36 layers", op="reorder", layers=36, groups=4, beams=8, survivors=4, sources=3,
             heads=32, dtype="fp32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "attention", "attention", "select", "select", "reorder"])
    if op == "rotary":
        dim = rng.choice([64, 128, 256])
        kv = rng.choice([1, 2, 4, 8])
        rot = rng.choice([dim, dim // 2, dim // 4])
        axes = rng.choice([1, 3, 3])
        return dict(op=op, tokens=_log_int(rng, 1, 16381), q_heads=kv * rng.choice([1, 3, 4, 8 if kv < 4 else 2]),
                    kv_heads=kv, dim=dim, rotary_dim=rot, axes=axes, interleaved=axes == 3 and rng.random() < 0.5,
                    norm=rng.random() < 0.7, gated=rng.random() < 0.5, start=_log_int(rng, 1, 200000) - 1)
    if op == "attention":
        dim = rng.choice([64, 128, 128, 256, 256, 256])
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 3, 4, 6, 8]) if kv < 8 else kv * rng.choice([1, 3, 4])
        prefix = 16 * _log_int(rng, 4, 1024)
        suffix = _log_int(rng, 1, 2048)
        budget = 4_600_000 // ((prefix + suffix) * kv * dim // 128)  # sequences the largest case has room for
        batch = min(128, max(2, _log_int(rng, 2, max(3, budget))))
        groups = rng.choice([1, 1, 2, 3, 4, 8])
        rows = max(2, batch // groups)
        groups = max(1, min(groups, batch // rows))
        return dict(op=op, groups=groups, rows=rows, prefix=prefix, suffix=suffix, q_heads=heads, kv_heads=kv,
                    dim=dim)
    if op == "select":
        beams = rng.randint(1, 16)
        vocab = _log_int(rng, 1000, 250001)
        groups = _log_int(rng, 1, max(2, min(64, 48_000_000 // (beams * vocab))))
        return dict(op=op, groups=groups, beams=beams, vocab=vocab, n=rng.randint(1, 2 * beams),
                    dtype=rng.choice(["bf16", "bf16", "fp32"]), finished=rng.random() < 0.5)
    beams = rng.randint(2, 12)
    survivors = rng.randint(1, beams - 1)
    sources = rng.randint(1, min(survivors, beams - survivors))
    heads = rng.choice([4, 8, 16, 32])
    layers = rng.randint(1, 36)
    groups = _log_int(rng, 1, max(2, min(16, 36_864 // (layers * beams * heads))))
    return dict(op=op, layers=layers, groups=groups, beams=beams, survivors=survivors, sources=sources, heads=heads,
                dtype=rng.choice(["fp32", "fp32", "bf16"]))


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _rand(gen, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=gen, device=DEV, dtype=dtype)


def _sections(half, axes):
    """Frequency pairs of each axis: time gets what height and width leave (11, 11, 10 of 32)."""
    side = half // axes
    return [half - side * (axes - 1)] + [side] * (axes - 1)


def _axis_of_pair(half, sections, interleaved):
    """The position axis that turns each frequency pair."""
    axis = [0] * half
    if interleaved:  # pair i takes axis i mod A while that axis has pairs left, else axis 0
        for a in range(1, len(sections)):
            for i in range(a, min(half, len(sections) * sections[a]), len(sections)):
                axis[i] = a
    else:            # one run of pairs for each axis
        at = 0
        for a, n in enumerate(sections):
            axis[at:at + n] = [a] * n
            at += n
    return axis


def _prepare_rotary(c, gen):
    n, hq, hkv, d, rot = c["tokens"], c["q_heads"], c["kv_heads"], c["dim"], c["rotary_dim"]
    # q (and its gate, where there is one) and k | v leave two projections: views, not copies.
    q = _rand(gen, n, hq, 2 * d if c["gated"] else d)[..., :d]
    kv = _rand(gen, n, 2 * hkv, d)
    pages = -(-n // PAGE) + 16
    slots = torch.randperm(pages, generator=gen, device=DEV)[:-(-n // PAGE)]
    slots = (slots[:, None] * PAGE + torch.arange(PAGE, device=DEV)).reshape(-1)[:n].contiguous()
    time = c["start"] + torch.arange(n, device=DEV, dtype=torch.int32)
    if c["axes"] == 1:
        positions = time[None].contiguous()
    else:  # text and image tokens: the time axis runs on, height and width walk over a grid of patches
        positions = torch.stack([time, c["start"] + torch.randint(0, 64, (n,), generator=gen, device=DEV,
                                                                  dtype=torch.int32),
                                 c["start"] + torch.randint(0, 64, (n,), generator=gen, device=DEV,
                                                            dtype=torch.int32)])
    half = rot // 2
    sections = _sections(half, c["axes"])
    s = dict(q=q, k=kv[:, :hkv], v=kv[:, hkv:], slots=slots, positions=positions, eps=1e-6, rot=rot,
             pool=_rand(gen, pages, hkv, 2, PAGE, d),
             q_weight=1 + 0.2 * _rand(gen, d) if c["norm"] else None,
             k_weight=1 + 0.2 * _rand(gen, d) if c["norm"] else None,
             axis=torch.tensor(_axis_of_pair(half, sections, c["interleaved"]), device=DEV),
             inv_freq=torch.tensor([1e6 ** (-i / half) for i in range(half)], device=DEV, dtype=torch.float64))
    if own:
        from shellsmith_b200 import rotary
        s["plan"] = rotary.RotaryPlan(d, rot, base=1e6, sections=sections, interleaved=c["interleaved"], device=DEV)
    return s


def _prepare_attention(c, gen):
    groups, rows, d = c["groups"], c["rows"], c["dim"]
    B, pre = groups * rows, c["prefix"] // PAGE
    # Each sample has written between one token and `suffix` tokens of its own.
    own_len = torch.randint(1, c["suffix"] + 1, (B,), generator=torch.Generator().manual_seed(gen.initial_seed()))
    own_pages = -(-own_len // PAGE)
    width = pre + int(own_pages.max())
    total = groups * pre + int(own_pages.sum())
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(gen.initial_seed() + 1)).to(torch.int32)
    table = torch.zeros((B, width), dtype=torch.int32)
    table[:, :pre] = perm[:groups * pre].view(groups, 1, pre).expand(groups, rows, pre).reshape(B, pre)
    cell = torch.arange(width - pre)[None] < own_pages[:, None]
    table[:, pre:][cell] = perm[groups * pre:]
    ctx = (c["prefix"] + own_len).to(torch.int32)
    s = dict(q=_rand(gen, B, c["q_heads"], d), pool=_rand(gen, total, c["kv_heads"], 2, PAGE, d),
             table=table.to(DEV), ctx=ctx.to(DEV), scale=1 / math.sqrt(d))
    if own:
        from shellsmith_b200 import paged
        s["plan"] = paged.PrefixGroups([(range(g * rows, (g + 1) * rows), c["prefix"]) for g in range(groups)], B,
                                       c["q_heads"], c["kv_heads"], d, device=DEV)
        s["max_suffix"], s["total_suffix"] = int(own_pages.max()), int(own_pages.sum())
        s["workspace"] = paged.SharedPrefixWorkspace(device=DEV)
    return s


def _prepare_select(c, gen):
    g, k, v = c["groups"], c["beams"], c["vocab"]
    logits = _rand(gen, g, k, v, dtype=torch.float32).mul_(2.5)
    if c["dtype"] == "bf16":
        logits = logits.to(torch.bfloat16)
    scores = -5 - 2 * torch.rand((g, k), generator=gen, device=DEV).mul_(4).cumsum(1)
    done = torch.rand((g, k), generator=gen, device=DEV) < 0.2 if c["finished"] else None
    return dict(logits=logits, scores=scores, n=c["n"], finished=done, pad=2)


def _prepare_reorder(c, gen):
    g, k, kept, src = c["groups"], c["beams"], c["survivors"], c["sources"]
    cpu = torch.Generator().manual_seed(gen.initial_seed())
    parents = torch.empty((g, k), dtype=torch.int64)
    for i in range(g):  # `survivors` beams have children; the surplus falls to the first `sources` of them
        alive = torch.randperm(k, generator=cpu)[:kept]
        more = torch.cat([torch.arange(src), torch.randint(0, src, (k - kept - src,), generator=cpu)])
        parents[i] = torch.cat([alive, alive[more]])[torch.randperm(k, generator=cpu)]
    rows = g * k + 2
    state = _rand(gen, c["layers"], rows, c["heads"], 128, 128,
                  dtype=torch.float32 if c["dtype"] == "fp32" else torch.bfloat16)
    slots = torch.randperm(rows, generator=cpu)[:g * k].view(g, k)
    return dict(state=state, slots=slots.to(DEV, torch.int32), parents=parents.to(DEV, torch.int32))


def prepare(case, seed):
    make = dict(rotary=_prepare_rotary, attention=_prepare_attention, select=_prepare_select,
                reorder=_prepare_reorder)[case["op"]]
    return dict(make(case, _gen(seed)), op=case["op"])


# ------------------------------------------------------------------ plain forms
def _place(slots, dim):
    """Element offsets [n, D] of a token's row inside its (head, K|V) block, and its page."""
    token = slots % PAGE
    col = torch.arange(dim, device=slots.device)
    chunk = (col // 8)[None] ^ (token & 7)[:, None]
    return slots // PAGE, token, chunk * 8 + (col % 8)[None]


def _plain_turn(x, weight, cos, sin, rot, eps):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight.float()
    a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rot:]], -1).to(torch.bfloat16)


def _plain_rotary(s):
    angle = s["positions"][s["axis"]].t().float() * s["inv_freq"].float()        # [n, rot / 2]
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    q = _plain_turn(s["q"], s["q_weight"], cos, sin, s["rot"], s["eps"])
    k = _plain_turn(s["k"], s["k_weight"], cos, sin, s["rot"], s["eps"])
    pool = s["pool"]
    page, token, col = _place(s["slots"], pool.shape[-1])
    head = torch.arange(pool.shape[1], device=pool.device)
    at = (page[:, None, None], head[None, :, None])
    for which, x in ((0, k), (1, s["v"])):
        pool[at[0], at[1], which, token[:, None, None], col[:, None]] = x
    return dict(q=q, pool=pool)


def _plain_attention(s):
    pool, table, q = s["pool"], s["table"].long(), s["q"].float()
    B, hq, d = q.shape
    hkv = pool.shape[1]
    chunk = torch.arange(d // 8, device=pool.device)[None] ^ (torch.arange(PAGE, device=pool.device) & 7)[:, None]
    row = torch.arange(PAGE, device=pool.device)[:, None]
    rows = pool.view(-1, hkv, 2, PAGE, d // 8, 8)[:, :, :, row, chunk].view(-1, hkv, 2, PAGE, d)
    kv = rows[table].permute(3, 0, 2, 1, 4, 5).reshape(2, B, hkv, -1, d)         # [2, B, Hkv, T, D]
    x = torch.matmul(q.view(B, hkv, hq // hkv, d), kv[0].float().transpose(-1, -2)) * s["scale"]
    seen = torch.arange(x.shape[-1], device=x.device)[None] < s["ctx"][:, None]
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    p = (x - x.amax(-1, keepdim=True)).exp()
    out = torch.matmul(p / p.sum(-1, keepdim=True), kv[1].float())
    return out.reshape(B, hq, d).to(torch.bfloat16)


def _plain_select(s):
    x, scores = s["logits"].float(), s["scores"]
    B, K, V = x.shape
    z = x - x.amax(-1, keepdim=True)
    score = scores[..., None] + (z - z.exp().sum(-1, keepdim=True).log())
    if s["finished"] is not None:
        pad = torch.arange(V, device=x.device) == s["pad"]
        kept = torch.where(pad, scores[..., None], -math.inf)
        score = torch.where(s["finished"][..., None], kept, score)
    score = torch.where(score.isnan(), -math.inf, score).view(B, K * V) + 0.0
    # One whole number orders scores first and, among equal ones, the lower place first.
    bits = score.view(torch.int32)
    rank = torch.where(bits >= 0, bits, bits ^ 0x7fffffff).long()
    key = rank * (1 << 32) + ((1 << 32) - 1 - torch.arange(K * V, device=x.device))
    at = (1 << 32) - 1 - (key.topk(s["n"], dim=-1).values & 0xffffffff)
    return dict(scores=score.gather(1, at), parents=(at // V).int(), tokens=(at % V).int())


def _plain_reorder(s):
    state, slots, parents = s["state"], s["slots"].long(), s["parents"].long()
    K = slots.shape[1]
    same = parents[:, :, None] == parents[:, None, :]                            # child j, child i
    later = (same & torch.ones(K, K, device=same.device, dtype=torch.bool).tril(-1)).any(-1)
    beam = torch.arange(K, device=slots.device)
    dead = ~(parents[:, None, :] == beam[None, :, None]).any(-1)
    free = torch.argsort((~dead).long(), dim=1, stable=True)                     # dead beams first, ascending
    taken = free.gather(1, (later.long().cumsum(1) - 1).clamp(min=0))
    new = slots.gather(1, torch.where(later, taken, parents))
    source = torch.arange(state.shape[1], device=slots.device)
    source[new.view(-1)] = slots.gather(1, parents).view(-1)
    state.copy_(state.index_select(1, source))
    return dict(slots=new.int(), state=state)


_PLAIN = dict(rotary=_plain_rotary, attention=_plain_attention, select=_plain_select, reorder=_plain_reorder)


# ------------------------------------------------------------------ the framework's operators
def _own_rotary(s):
    from shellsmith_b200 import rotary
    q = rotary.rotary_append(s["q"], s["k"], s["v"], s["positions"], s["plan"], s["pool"], s["slots"],
                             q_weight=s["q_weight"], k_weight=s["k_weight"], eps=s["eps"])
    return dict(q=q, pool=s["pool"])


def _own_attention(s):
    from shellsmith_b200 import paged
    return paged.shared_prefix_attention(s["q"], s["pool"], s["table"], s["ctx"], s["scale"], s["plan"],
                                         max_suffix_pages=s["max_suffix"], total_suffix_pages=s["total_suffix"],
                                         workspace=s["workspace"])


def _own_select(s):
    from shellsmith_b200 import beam
    scores, parents, tokens = beam.beam_select(s["logits"], s["scores"], s["n"], finished=s["finished"],
                                               pad_token=s["pad"])
    return dict(scores=scores, parents=parents, tokens=tokens)


def _own_reorder(s):
    from shellsmith_b200 import beam
    return dict(slots=beam.reorder_rows([s["state"]], s["slots"], s["parents"]), state=s["state"])


_OWN = dict(rotary=_own_rotary, attention=_own_attention, select=_own_select, reorder=_own_reorder)


def run(state):
    return (_OWN if own else _PLAIN)[state["op"]](state)


# ------------------------------------------------------------------ work
def work(c):
    if c["op"] == "rotary":
        heads = c["q_heads"] + 2 * c["kv_heads"]
        return dict(bytes=c["tokens"] * (2 * heads * c["dim"] * 2 + 4 * c["axes"] + 8),
                    flops=c["tokens"] * heads * c["dim"] * 6)
    if c["op"] == "attention":
        B, mean = c["groups"] * c["rows"], (c["suffix"] + 1) / 2
        tokens = c["groups"] * c["prefix"] + B * mean                            # cached tokens, each once
        return dict(bytes=tokens * c["kv_heads"] * c["dim"] * 4 + 2 * B * c["q_heads"] * c["dim"] * 2,
                    flops=4 * B * c["q_heads"] * c["dim"] * (c["prefix"] + mean))
    if c["op"] == "select":
        n = c["groups"] * c["beams"] * c["vocab"]
        return dict(bytes=n * (2 if c["dtype"] == "bf16" else 4) + c["groups"] * c["n"] * 12, flops=4 * n)
    row = c["heads"] * 128 * 128 * (4 if c["dtype"] == "fp32" else 2)
    moved = c["sources"] + c["beams"] - c["survivors"]                           # rows read once, rows written
    return dict(bytes=c["layers"] * c["groups"] * moved * row, flops=0)


# ------------------------------------------------------------------ 64-bit results
def _exact_rotary(c, s):
    d, rot = c["dim"], c["rotary_dim"]
    half = rot // 2
    sections = _sections(half, c["axes"])
    names = []
    if c["interleaved"]:
        for i in range(half):
            a = i % c["axes"]
            names.append(a if i < c["axes"] * sections[a] else 0)
    else:
        names = [a for a, n in enumerate(sections) for _ in range(n)]
    turn = torch.stack([s["positions"][a].double() * 1e6 ** (-i / half) for i, a in enumerate(names)], 1)
    z = torch.polar(torch.ones_like(turn), turn)[:, None]

    def rotate(x, w):
        x = x.double()
        if w is not None:
            x = x / ((x ** 2).sum(-1, keepdim=True) / d + 1e-6).sqrt() * w.double()
        y = torch.complex(x[..., :half].contiguous(), x[..., half:rot].contiguous()) * z
        return torch.cat((y.real, y.imag, x[..., rot:]), -1)

    pool = s["pool"].double()
    order = torch.stack([torch.arange(d, device=DEV).view(-1, 8)[torch.arange(d // 8, device=DEV) ^ (t & 7)].view(-1)
                         for t in range(PAGE)])                                  # stored column -> logical column
    flat = pool.transpose(2, 3).transpose(1, 2).contiguous().view(-1, c["kv_heads"], 2, d)   # [slot, head, K|V, D]
    kv = torch.stack([rotate(s["k"], s["k_weight"]), s["v"].double()], 2)
    pick = order[s["slots"] % PAGE][:, None, None].expand_as(kv)
    flat[s["slots"]] = kv.gather(-1, pick)
    pool = flat.view(-1, PAGE, c["kv_heads"], 2, d).permute(0, 2, 3, 1, 4).contiguous()
    return dict(q=rotate(s["q"], s["q_weight"]), pool=pool)


def _exact_attention(c, s):
    d, hkv, group = c["dim"], c["kv_heads"], c["q_heads"] // c["kv_heads"]
    order = torch.stack([torch.arange(d, device=DEV).view(-1, 8)[torch.arange(d // 8, device=DEV) ^ (t & 7)].view(-1)
                         for t in range(PAGE)])
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    for b, n in enumerate(s["ctx"].tolist()):                                    # one sequence at a time
        pages = s["pool"][s["table"][b, :-(-n // PAGE)].long()].double()
        pages = pages.gather(-1, order.expand_as(pages))
        k, v = (pages[:, :, i].transpose(0, 1).reshape(hkv, -1, d)[:, :n] for i in (0, 1))
        x = torch.einsum("hgd,htd->hgt", s["q"][b].double().view(hkv, group, d), k) * s["scale"]
        out[b] = torch.einsum("hgt,htd->hgd", torch.softmax(x, -1), v).reshape(-1, d)
    return out


def _exact_select(c, s):
    best = []
    for g in range(c["groups"]):
        x = s["logits"][g].double()
        total = s["scores"][g].double()[:, None] + torch.log_softmax(x, -1)
        if s["finished"] is not None:
            for k in torch.nonzero(s["finished"][g]).view(-1).tolist():
                total[k] = -math.inf
                total[k, s["pad"]] = s["scores"][g, k].double()
        best.append(torch.sort(total.view(-1), descending=True).values[:c["n"]])
    return dict(scores=torch.stack(best), parents=None, tokens=None)


def _exact_reorder(c, s):
    slots, parents, state = s["slots"].tolist(), s["parents"].tolist(), s["state"].double()
    copies = []
    for mine, up in zip(slots, parents):
        free = [mine[b] for b in range(len(mine)) if b not in up]
        seen = set()
        for p in up:
            if p in seen:
                copies.append((mine[p], free.pop(0)))
            seen.add(p)
    for a, b in copies:
        state[:, b] = state[:, a]
    return dict(slots=None, state=state)


def exact(case, seed):
    s = prepare(case, seed)
    return dict(rotary=_exact_rotary, attention=_exact_attention, select=_exact_select,
                reorder=_exact_reorder)[case["op"]](case, s)
