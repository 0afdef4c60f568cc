"""What the operators of a speculative decoding step over shared prefixes are
measured on: the append with per-head norms of queries and keys, attention over
a cache whose prefix many sequences share, token probabilities, and the
verification of drafted tokens.

``run`` computes an operator in elementary torch operations, or, with ``own``
set, through the framework's public calls. Cases name sizes only; lengths and
token counts of a case follow from its sizes (``shape``), values from the seed.
"""

import itertools
import math
import random

import torch

own = False

D = 64        # head width
PAGE = 16     # tokens of a cache block
EPS = 1e-5
THETA = 10000.0


# ---- cases -------------------------------------------------------------------


def listed():
    return [
        # the prefix-reuse configuration: 64 requests over a 384-token system
        # prompt, a step in the middle of their answers
        dict(name="attend reuse 64x384 f32", op="attend", dtype="f32", hq=4, hkv=2, seqs=64, groups=1,
             prefix=384, own=128, count=1, ragged=False, rotate=True),
        # the smallest call: two requests, a short shared greeting (latency)
        dict(name="attend pair 2x48 f32", op="attend", dtype="f32", hq=4, hkv=2, seqs=2, groups=1,
             prefix=48, own=17, count=1, ragged=False, rotate=False),
        # batched serving of the wide model: a long system prompt, own turns
        dict(name="attend serve 128x4096 bf16", op="attend", dtype="bf16", hq=32, hkv=8, seqs=128, groups=1,
             prefix=4096, own=512, count=1, ragged=False, rotate=True),
        # drafted tokens of many requests over one long document
        dict(name="attend drafts 48x8192 bf16", op="attend", dtype="bf16", hq=32, hkv=8, seqs=48, groups=1,
             prefix=8192, own=251, count=6, ragged=True, rotate=False),
        # two documents, eight query heads a key head, drafts, f32 pages
        dict(name="attend documents 24x2048 f32", op="attend", dtype="f32", hq=16, hkv=2, seqs=24, groups=2,
             prefix=2048, own=701, count=4, ragged=True, rotate=True),
        # one token of one request (latency)
        dict(name="append token 1 f32", op="append", dtype="f32", hq=4, hkv=2, seqs=1, base=37, count=1,
             fused=False, rotate=True),
        # a decode step of a full batch of the wide model
        dict(name="append step 128 bf16", op="append", dtype="bf16", hq=32, hkv=8, seqs=128, base=70, count=1,
             fused=True, rotate=True),
        # a prompt chunk of the wide model, projections in one buffer
        dict(name="append prompt 8191 bf16", op="append", dtype="bf16", hq=32, hkv=8, seqs=1, base=0, count=8191,
             fused=True, rotate=True),
        # a decode step's rows at this repository's vocabulary
        dict(name="probabilities 64x8192", op="probabilities", rows=64, vocab=8192, masked=False),
        # drafted rows at a wide, odd vocabulary, some tokens banned
        dict(name="probabilities 320x100003", op="probabilities", rows=320, vocab=100003, masked=True),
        # four drafts a request at this repository's vocabulary
        dict(name="verify 64x4 8192", op="verify", seqs=64, drafts=4, ragged=True, vocab=8192, sampled=True),
        # one request, drafts without probabilities (prompt lookup), odd vocabulary
        dict(name="verify 1x3 32003", op="verify", seqs=1, drafts=3, ragged=False, vocab=32003, sampled=False),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    top = {}
    for c in listed():
        top[c["op"]] = max(top.get(c["op"], 0), _cost(c))
    top["verify"] = top["probabilities"]  # the rows it chooses from lie in memory alike
    while True:
        op = rng.choice(["attend", "attend", "append", "probabilities", "verify"])
        if op == "attend":
            hq, hkv = rng.choice([(4, 2), (32, 8), (8, 8), (16, 2), (8, 4), (2, 1)])
            groups = rng.choice([1, 1, 2, 3])
            case = dict(op=op, dtype=rng.choice(["f32", "bf16"]), hq=hq, hkv=hkv,
                        seqs=groups * _log(rng, 1, 96), groups=groups, prefix=PAGE * _log(rng, 1, 512),
                        own=_log(rng, 1, 2048), count=_log(rng, 1, 8), ragged=rng.random() < 0.5,
                        rotate=rng.random() < 0.5)
        elif op == "append":
            hq, hkv = rng.choice([(4, 2), (32, 8), (8, 8), (16, 2)])
            case = dict(op=op, dtype=rng.choice(["f32", "bf16"]), hq=hq, hkv=hkv)
            if rng.random() < 0.5:  # one prompt or prompt chunk
                case.update(seqs=1, base=rng.choice([0, rng.randrange(500)]), count=_log(rng, 1, 8000))
            else:  # a step of many sequences
                count = rng.randrange(1, 7)
                case.update(seqs=_log(rng, 2, 256), base=PAGE * rng.randrange(40) + rng.randrange(1, 10),
                            count=count)
            case.update(fused=rng.random() < 0.5, rotate=rng.random() < 0.8)
        elif op == "probabilities":
            case = dict(op=op, rows=_log(rng, 1, 512), vocab=_log(rng, 100, 130000), masked=rng.random() < 0.5)
        else:
            case = dict(op=op, seqs=_log(rng, 1, 160), drafts=_log(rng, 1, 8), ragged=rng.random() < 0.5,
                        vocab=_log(rng, 100, 130000), sampled=rng.random() < 0.7)
            if case["seqs"] * (case["drafts"] + 1) * case["vocab"] > 64_000_000:
                continue
        if _cost(case) <= top[op]:
            return case


def shape(case):
    """Lengths and token counts of a case, from its sizes alone."""
    r = random.Random("%s" % sorted((k, v) for k, v in case.items() if k != "name"))
    n = case.get("seqs", 0)
    if case["op"] == "attend":
        own_len = [r.randint(0, case["own"]) for _ in range(n)]  # cached tokens after the prefix
        counts = [r.randint(1, case["count"]) if case["ragged"] else case["count"] for _ in range(n)]
        return own_len, counts
    if case["op"] == "append":
        return [case["base"]] * n, [case["count"]] * n
    if case["op"] == "probabilities":
        n = min(case["rows"], 256)
        return None, [case["rows"] // n + (i < case["rows"] % n) for i in range(n)]
    return None, [1 + (r.randint(0, case["drafts"]) if case["ragged"] else case["drafts"]) for _ in range(n)]


def work(case):
    own_len, counts = shape(case)
    if case["op"] == "attend":
        s = 2 if case["dtype"] == "bf16" else 4
        keys = case["groups"] * case["prefix"] + sum(l + c for l, c in zip(own_len, counts))
        pairs = sum(c * (case["prefix"] + l) + c * (c + 1) // 2 for l, c in zip(own_len, counts))
        rows = sum(counts)
        return {"bytes": keys * case["hkv"] * D * 2 * s + 2 * rows * case["hq"] * D * 4,
                "flops": 4 * D * case["hq"] * pairs}
    if case["op"] == "append":
        t = sum(counts)
        s = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": t * ((2 * case["hq"] + 2 * case["hkv"]) * D * 4 + 2 * case["hkv"] * D * s + D * 4),
                "flops": t * (case["hq"] + case["hkv"]) * D * 8}
    if case["op"] == "probabilities":
        v = case["rows"] * case["vocab"]
        return {"bytes": 8 * v, "flops": 5 * v}
    # one row of the target's, and the draft's where a draft is rejected (about half)
    v = case["seqs"] * case["vocab"]
    return {"bytes": v * (6 if case["sampled"] else 4), "flops": 3 * v}


# ---- inputs ------------------------------------------------------------------


def _randn(g, *size):
    return torch.randn(size, generator=g, device="cuda", dtype=torch.float32)


def _rope_table(positions):
    """(cos, sin) [positions, 32]: angles are f32 products of the position and
    the f32 inverse frequency, as the cache's rotation defines them."""
    inv = torch.tensor([THETA ** (-2.0 * i / D) for i in range(D // 2)], dtype=torch.float64).float()
    angle = (torch.arange(positions, dtype=torch.float32)[:, None] * inv[None]).double()
    return angle.cos().cuda(), angle.sin().cuda()


def _offsets(counts):
    return list(itertools.accumulate(counts, initial=0))[:-1]


def _index(values):
    return torch.tensor(values, dtype=torch.int64, device="cuda")


def _package():
    import sys
    from pathlib import Path

    root = str(Path(__file__).resolve().parents[1] / "small-lm-rs_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import slmkv

    return slmkv


def _pool(case, context, blocks, seqs):
    slmkv = _package()
    return slmkv.KvPool(num_layers=1, num_query_heads=case.get("hq", 1), num_key_value_heads=case.get("hkv", 1),
                        context_length=context, rope_theta=THETA, num_blocks=blocks, max_sequences=seqs,
                        kv_dtype=slmkv.KV_BF16 if case.get("dtype") == "bf16" else slmkv.KV_F32)


def _rows_batch(counts):
    """An open batch of sequences that each add counts[i] token rows."""
    pool = _pool({}, max(counts), sum(-(-c // PAGE) for c in counts), len(counts))
    return pool, pool.begin([pool.allocate_kv_cache(max(counts)) for _ in counts], counts)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return {"attend": _prepare_attend, "append": _prepare_append, "probabilities": _prepare_probabilities,
            "verify": _prepare_verify}[case["op"]](case, g)


def _prepare_attend(case, g):
    own_len, counts = shape(case)
    n, groups, prefix, hkv, hq = case["seqs"], case["groups"], case["prefix"], case["hkv"], case["hq"]
    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    lens = [l + c for l, c in zip(own_len, counts)]
    lmax, cmax, rows = max(lens), max(counts), sum(counts)
    # keys after a norm and a rotation, values of a projection
    kp, vp = _randn(g, groups, prefix, hkv, D).to(dtype), _randn(g, groups, prefix, hkv, D).to(dtype)
    ks, vs = _randn(g, n, lmax, hkv, D).to(dtype), _randn(g, n, lmax, hkv, D).to(dtype)
    live = torch.arange(lmax, device="cuda")[None] < _index(lens)[:, None]
    ks, vs = ks * live[..., None, None], vs * live[..., None, None]
    q = _randn(g, rows, hq, D)
    off = _offsets(counts)
    s = dict(case=case, q=q, kp=kp, vp=vp, ks=ks, vs=vs, own_len=own_len, counts=counts, off=off)
    s["place"] = _index([i * cmax + j for i, c in enumerate(counts) for j in range(c)])
    s["last"] = _index([own_len[i] + j for i, c in enumerate(counts) for j in range(c)])  # own keys seen: 0..last
    s["last_pad"] = torch.full((n * cmax,), -1, dtype=torch.int64, device="cuda")
    s["last_pad"][s["place"]] = s["last"]
    s["cos"], s["sin"] = _rope_table(prefix + max(lens))
    s["pos"] = s["last"] + prefix
    if own:
        context = prefix + lmax
        blocks = groups * (prefix // PAGE) + sum(-(-x // PAGE) + 1 for x in lens) + 1
        pool = _pool(case, context, blocks, n)
        caches = [pool.allocate_kv_cache(context) for _ in range(n)]
        m = n // groups
        leaders = caches[::m]
        [c.append_layer(0, kp[j].float(), vp[j].float(), prefix) for j, c in enumerate(leaders)]
        [c.publish_prefix([1 + j] * prefix) for j, c in enumerate(leaders)]
        [c.attach_prefix([1 + i // m] * prefix) for i, c in enumerate(caches) if i % m]
        some = [i for i in range(n) if own_len[i]]
        if some:
            with pool.begin([caches[i] for i in some], [own_len[i] for i in some]) as b:
                b.append_layer(0, torch.cat([ks[i, :own_len[i]] for i in some]).float(),
                               torch.cat([vs[i, :own_len[i]] for i in some]).float(), rotate_keys=False)
        s["batch"] = pool.begin(caches, counts)
        s["batch"].append_layer(0, torch.cat([ks[i, own_len[i]:lens[i]] for i in range(n)]).float(),
                                torch.cat([vs[i, own_len[i]:lens[i]] for i in range(n)]).float(), rotate_keys=False)
        s["pool"], s["out"] = pool, torch.empty_like(q)
    return s


def _prepare_append(case, g):
    n, base, count, hq, hkv = case["seqs"], case["base"], case["count"], case["hq"], case["hkv"]
    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    t, context = n * count, base + count
    if case["fused"]:  # one projection's output holds the three side by side
        qkv = _randn(g, t, hq + 2 * hkv, D) * 1.7
        q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    else:
        q, k, v = _randn(g, t, hq, D) * 1.7, _randn(g, t, hkv, D) * 1.7, _randn(g, t, hkv, D) * 1.7
    pages = -(-context // PAGE)
    s = dict(case=case, q=q, k=k, v=v, q_norm=1 + 0.2 * _randn(g, D), k_norm=1 + 0.2 * _randn(g, D))
    s["pos"] = (torch.arange(t, device="cuda") % count) + base
    s["cos"], s["sin"] = _rope_table(context)
    if own:
        pool = _pool(case, context, n * pages, n)
        caches = [pool.allocate_kv_cache(context) for _ in range(n)]
        if base:
            with pool.begin(caches, base) as b:
                b.append_layer(0, _randn(g, n * base, hkv, D), _randn(g, n * base, hkv, D))
        plan = pool.step_plan(caches, count)
        b = plan.begin()
        table = _index([c.blocks() for c in caches])  # the same blocks at every begin
        b.rollback()
        s.update(pool=pool, plan=plan, q_out=torch.empty((t, hq, D), device="cuda"))
        s["k_pages"], s["v_pages"] = (x[0] for x in pool.storage())
    else:
        table = torch.arange(n * pages, device="cuda").view(n, pages)
        s["k_pages"] = torch.zeros((n * pages, hkv, PAGE, D), dtype=dtype, device="cuda")
        s["v_pages"] = torch.zeros_like(s["k_pages"])
    s["block"] = table[torch.arange(t, device="cuda") // count, s["pos"] // PAGE]
    s["slot"] = s["pos"] % PAGE
    return s


def _prepare_probabilities(case, g):
    _, counts = shape(case)
    rows, vocab = case["rows"], case["vocab"]
    logits = _randn(g, rows, vocab) * 2.5
    if case["masked"]:  # tokens that a grammar or a ban list forbids
        logits.masked_fill_(torch.rand((rows, vocab), generator=g, device="cuda") < 0.3, -math.inf)
        logits[:, 0] = 1.0
    # requests ask for greedy, cool, plain and warm sampling
    t = torch.tensor([0.0, 0.3, 0.8, 1.0, 1.0, 1.7], device="cuda")[torch.arange(rows, device="cuda") % 6]
    s = dict(case=case, logits=logits, temperatures=t.contiguous())
    if own:
        s["pool"], s["batch"] = _rows_batch(counts)
        s["out"] = torch.empty_like(logits)
    return s


def _prepare_verify(case, g):
    _, counts = shape(case)
    n, vocab, rows = case["seqs"], case["vocab"], sum(counts)
    off = _offsets(counts)
    logits = _randn(g, rows, vocab) * 2.5
    target = torch.softmax(logits, -1)
    at = _index([off[i] + j for i, c in enumerate(counts) for j in range(c - 1)])  # target row of each draft
    ids = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    draft = None
    if at.numel():
        # a smaller model's distribution, near the target's; without one, the
        # drafts are likely continuations
        near = torch.softmax(logits[at] + 0.8 * _randn(g, at.numel(), vocab), -1)
        ids[at + 1] = torch.multinomial(near, 1, generator=g)[:, 0].int()
        if case["sampled"]:
            draft = near
    u = torch.rand((rows,), generator=g, device="cuda")
    s = dict(case=case, target=target, draft=draft, ids=ids, u=u, at=at)
    kmax = max(counts) - 1
    s["place"] = _index([i * kmax + j for i, c in enumerate(counts) for j in range(c - 1)])
    s["off"], s["k"], s["kmax"] = _index(off), _index([c - 1 for c in counts]), kmax
    s["draft_off"] = _index([off[i] - i for i in range(n)])
    if own:
        s["pool"], s["batch"] = _rows_batch(counts)
        s["accepted"] = torch.empty(n, dtype=torch.int32, device="cuda")
        s["next"] = torch.empty(n, dtype=torch.int32, device="cuda")
    return s


# ---- one pass ----------------------------------------------------------------


def run(s):
    op = s["case"]["op"]
    if own:
        return {"attend": _own_attend, "append": _own_append, "probabilities": _own_probabilities,
                "verify": _own_verify}[op](s)
    return {"attend": _plain_attend, "append": _plain_append, "probabilities": _plain_probabilities,
            "verify": _plain_verify}[op](s)


def _own_attend(s):
    s["batch"].shared_prefix_attention(0, s["q"], s["out"], rotate_query=s["case"]["rotate"])
    return s["out"]


def _own_append(s):
    b = s["plan"].begin()
    b.append_layer_normed(0, s["q"], s["k"], s["v"], s["q_norm"], s["k_norm"], s["q_out"], epsilon=EPS,
                          rotate=s["case"]["rotate"])
    out = s["q_out"], s["k_pages"][s["block"], :, s["slot"]], s["v_pages"][s["block"], :, s["slot"]]
    b.rollback()  # the next pass appends the same positions again
    return out


def _own_probabilities(s):
    s["batch"].token_probabilities(s["logits"], s["out"], temperatures=s["temperatures"])
    return s["out"]


def _own_verify(s):
    s["batch"].verify_drafts(s["ids"], s["target"], s["draft"], s["u"], s["accepted"], s["next"])
    return s["accepted"], s["next"]


def _rotate(x, cos, sin):
    """Rotates the pairs (2i, 2i + 1) of x [rows, heads, 64] by cos/sin [rows, 32]."""
    a, b = x[..., 0::2], x[..., 1::2]
    c, n = cos[:, None], sin[:, None]
    return torch.stack((a * c - b * n, a * n + b * c), -1).flatten(-2)


def _plain_attend(s):
    case = s["case"]
    n, groups, hkv, hq = case["seqs"], case["groups"], case["hkv"], case["hq"]
    rep, m = hq // hkv, n // groups
    cmax = s["last_pad"].numel() // n
    q = s["q"]
    if case["rotate"]:
        q = _rotate(q, s["cos"][s["pos"]].float(), s["sin"][s["pos"]].float())
    pad = torch.zeros((n * cmax, hq, D), device="cuda")
    pad[s["place"]] = q / math.sqrt(D)
    pad = pad.view(n, cmax, hkv, rep, D).permute(0, 2, 1, 3, 4)  # [n, hkv, c, rep, D]
    ks, vs = (s[x].float().permute(0, 2, 1, 3) for x in ("ks", "vs"))
    kp, vp = (s[x].float().permute(0, 2, 1, 3) for x in ("kp", "vp"))
    # the prefix: all rows of a group against one copy of its keys
    shared = pad.view(groups, m, hkv, cmax, rep, D).permute(0, 2, 1, 3, 4, 5)
    sp = shared.reshape(groups, hkv, m * cmax * rep, D) @ kp.transpose(-1, -2)
    so = pad.reshape(n, hkv, cmax * rep, D) @ ks.transpose(-1, -2)
    seen = torch.arange(ks.shape[2], device="cuda")[None] <= s["last_pad"][:, None]
    seen = seen.view(n, 1, cmax, 1, -1).expand(n, 1, cmax, rep, seen.shape[-1]).reshape(n, 1, cmax * rep, -1)
    so = so.masked_fill(~seen, -math.inf)
    sp_max = sp.amax(-1).view(groups, hkv, m, cmax * rep).transpose(1, 2).reshape(n, hkv, cmax * rep)
    top = torch.maximum(sp_max, so.amax(-1))
    top_p = top.view(groups, m, hkv, cmax * rep).transpose(1, 2).reshape(groups, hkv, -1)
    sp = torch.exp(sp - top_p[..., None])
    so = torch.exp(so - top[..., None])
    op, lp = sp @ vp, sp.sum(-1)
    op = op.view(groups, hkv, m, cmax * rep, D).transpose(1, 2).reshape(n, hkv, cmax * rep, D)
    lp = lp.view(groups, hkv, m, cmax * rep).transpose(1, 2).reshape(n, hkv, cmax * rep)
    out = (op + so @ vs) / (lp + so.sum(-1))[..., None]
    out = out.view(n, hkv, cmax, rep, D).transpose(1, 2).reshape(n * cmax, hq, D)
    return out[s["place"]]


def _plain_append(s):
    def normed(x, w):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w

    q, k = normed(s["q"], s["q_norm"]), normed(s["k"], s["k_norm"])
    if s["case"]["rotate"]:
        cos, sin = s["cos"][s["pos"]].float(), s["sin"][s["pos"]].float()
        q, k = _rotate(q, cos, sin), _rotate(k, cos, sin)
    pages = s["k_pages"], s["v_pages"]
    pages[0][s["block"], :, s["slot"]] = k.to(pages[0].dtype)
    pages[1][s["block"], :, s["slot"]] = s["v"].to(pages[1].dtype)
    return q, pages[0][s["block"], :, s["slot"]], pages[1][s["block"], :, s["slot"]]


def _plain_probabilities(s):
    x, t = s["logits"], s["temperatures"][:, None]
    top, first = x.max(-1, keepdim=True)
    first = (x == top).to(torch.int8).argmax(-1, keepdim=True)  # the lowest index of the maximum
    e = torch.exp((x - top) / torch.where(t > 0, t, torch.ones_like(t)))
    p = e / e.sum(-1, keepdim=True)
    hot = torch.arange(x.shape[1], device="cuda")[None] == first
    return torch.where(t > 0, p, hot.float())


def _plain_verify(s):
    # in 64 bits: the drawn index lies next to a border of the running sum
    n, kmax = s["case"]["seqs"], s["kmax"]
    accepted = torch.zeros(n, dtype=torch.int64, device="cuda")
    if kmax:
        x = s["ids"][s["at"] + 1].long()
        p = s["target"][s["at"], x].double()
        q = 1.0 if s["draft"] is None else s["draft"].gather(1, x[:, None])[:, 0].double()
        ok = torch.zeros(n * kmax, dtype=torch.int64, device="cuda")
        ok[s["place"]] = (s["u"][s["at"]].double() * q < p).long()
        accepted = ok.view(n, kmax).cumprod(1).sum(1)
    row = s["off"] + accepted
    w = s["target"][row].double()
    if kmax and s["at"].numel():
        rejected = accepted < s["k"]
        if s["draft"] is None:
            token = s["ids"][torch.where(rejected, row + 1, row)].long()
            q = torch.where(torch.arange(w.shape[1], device="cuda")[None] == token[:, None], w, 0.0)
        else:
            q = s["draft"][torch.where(rejected, s["draft_off"] + accepted, 0)].double()
        rest = torch.where(rejected[:, None], (w - q).clamp_min(0), w)
        w = torch.where((rest.sum(1) > 0)[:, None], rest, w)
    run_sum = w.cumsum(1)
    # the last row of uniforms of a sequence draws its next token
    point = s["u"][s["off"] + s["k"]].double() * run_sum[:, -1]
    nxt = (run_sum > point[:, None]).to(torch.int8).argmax(1)
    return accepted.int(), nxt.int()


# ---- the definition in 64 bits -------------------------------------------------


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "attend":
        rep, m, prefix = case["hq"] // case["hkv"], case["seqs"] // case["groups"], case["prefix"]
        q = s["q"].double()
        if case["rotate"]:
            q = _turn(q, s["cos"][s["pos"]], s["sin"][s["pos"]])
        out = torch.empty_like(q)
        for i, (l, c, o) in enumerate(zip(s["own_len"], s["counts"], s["off"])):
            k = torch.cat((s["kp"][i // m], s["ks"][i, :l + c])).double().repeat_interleave(rep, 1)
            v = torch.cat((s["vp"][i // m], s["vs"][i, :l + c])).double().repeat_interleave(rep, 1)
            w = torch.einsum("chd,khd->hck", q[o:o + c], k) / 8
            ahead = torch.arange(prefix + l + c, device="cuda")[None] > (prefix + l + torch.arange(c, device="cuda"))[:, None]
            w = torch.softmax(w.masked_fill(ahead[None], -math.inf), -1)
            out[o:o + c] = torch.einsum("hck,khd->chd", w, v)
        return out
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "probabilities":
        x, t = s["logits"].double(), s["temperatures"].double()
        for i in range(x.shape[0]):
            if t[i] > 0:
                x[i] = (x[i] / t[i] - torch.logsumexp(x[i] / t[i], 0)).exp()
            else:
                hot = torch.nonzero(x[i] == x[i].max())[0, 0]
                x[i] = 0
                x[i, hot] = 1
        return x
    return None  # whole numbers


def _turn(x, cos, sin):
    """x as complex pairs, times cos + i sin."""
    z = torch.view_as_complex(x.reshape(*x.shape[:-1], D // 2, 2).contiguous())
    z = z * torch.complex(cos, sin)[:, None]
    return torch.view_as_real(z).flatten(-2)


def _exact_append(s):
    def unit(x, w):
        x = x.double()
        return x / ((x * x).sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()

    q, k, v = unit(s["q"], s["q_norm"]), unit(s["k"], s["k_norm"]), s["v"].double()
    if s["case"]["rotate"]:
        q, k = (_turn(x, s["cos"][s["pos"]], s["sin"][s["pos"]]) for x in (q, k))
    return q, k, v
