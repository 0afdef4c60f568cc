"""The operators of a speculative step beside its attention: the append with
per-head norms, token probabilities and the verification of drafts, each
against the definition in 64 bits, their refusals, and a run of them together
with the model."""

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
slmkv = pytest.importorskip("slmkv")

D = 64
THETA = 10000.0


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *size):
    return torch.randn(size, generator=g, device="cuda")


def make_pool(hq=4, hkv=2, context=128, seqs=4, dtype="f32", layers=1, blocks=None):
    return slmkv.KvPool(num_layers=layers, num_query_heads=hq, num_key_value_heads=hkv, context_length=context,
                        num_blocks=blocks or seqs * (context // 16 + 1), max_sequences=seqs,
                        kv_dtype=slmkv.KV_BF16 if dtype == "bf16" else slmkv.KV_F32)


# ---- append with per-head norms ------------------------------------------------


def normed_reference(x, w, eps, positions):
    """In 64 bits; the angle is the f32 product the rotation table holds."""
    x = x.double()
    y = x / ((x * x).sum(-1, keepdim=True) / D + eps).sqrt() * w.double()
    if positions is None:
        return y
    inv = torch.tensor([THETA ** (-2.0 * i / D) for i in range(D // 2)], dtype=torch.float64).float().cuda()
    angle = (positions.float()[:, None] * inv[None]).double()[:, None]
    a, b = y[..., 0::2], y[..., 1::2]
    return torch.stack((a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()), -1).flatten(-2)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hq,hkv", [(4, 2), (8, 8), (16, 2), (32, 8)])
@pytest.mark.parametrize("bases,counts", [([0], [1]), ([37], [1]), ([0, 15, 16, 40], [1, 1, 1, 1]),
                                          ([0, 3, 30, 17, 1], [33, 17, 1, 100, 16])])
@pytest.mark.parametrize("fused", [False, True])
def test_normed_append(dtype, hq, hkv, bases, counts, fused):
    g = gen(len(bases) + hq)
    pool = make_pool(hq, hkv, 160, len(bases), dtype, layers=2)
    pool.shuffle(3)
    caches = [pool.allocate_kv_cache(160) for _ in bases]
    for c, n in zip(caches, bases):
        for layer in range(2):
            if n:
                c.append_layer(layer, randn(g, n, hkv, D), randn(g, n, hkv, D), n)
    t = sum(counts)
    qkv = 3 * randn(g, t, hq + 2 * hkv, D)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    qn, kn = 1 + 0.3 * randn(g, D), 1 + 0.3 * randn(g, D)
    pos = torch.tensor([b + j for b, c in zip(bases, counts) for j in range(c)], device="cuda")
    q_out = torch.empty((t, hq, D), device="cuda")
    for layer, rotate in ((0, True), (1, False)):
        q_out.fill_(math.nan)
        if layer == 0:
            b = pool.begin(caches, counts)
        b.append_layer_normed(layer, q, k, v, qn, kn, q_out, epsilon=1e-4, rotate=rotate)
        want_q, want_k = (normed_reference(x, w, 1e-4, pos if rotate else None) for x, w in ((q, qn), (k, kn)))
        # f32: 64 squares summed, a root, three products and the rotation's two
        # products and sum, of values up to max |q|: below 16 roundings of 2^-24
        tol = 16 * 2.0**-24 * max(want_q.abs().max().item(), want_k.abs().max().item())
        assert (q_out.double() - want_q).abs().max().item() <= tol
        row = 0
        for c, base, n in zip(caches, bases, counts):
            got_k, got_v = c.layer_keys(layer)[base:], c.layer_values(layer)[base:]
            ref_k, ref_v = want_k[row:row + n], v[row:row + n].double()
            # a bf16 page rounds by half a step, 2^-8 of the value
            half = 2.0**-8 if dtype == "bf16" else 0.0
            assert ((got_k.double() - ref_k).abs() <= tol * (1 + half) + half * ref_k.abs()).all()
            if dtype == "bf16":
                assert torch.equal(got_v, v[row:row + n].to(torch.bfloat16).float())
            else:
                assert torch.equal(got_v, v[row:row + n])
            row += n
    b.end()
    assert [c.sequence_length() for c in caches] == [b + n for b, n in zip(bases, counts)]


def test_normed_append_in_place_zero_rows_and_storage():
    g = gen(1)
    pool = make_pool(blocks=16)
    cache = pool.allocate_kv_cache(64)
    q, k, v = randn(g, 20, 4, D), randn(g, 20, 2, D), randn(g, 20, 2, D)
    q[3, 1] = 0
    k[5, 0] = 0
    qn, kn = 1 + 0.3 * randn(g, D), 1 + 0.3 * randn(g, D)
    want = torch.empty_like(q)
    with pool.begin([cache], 20) as b:
        b.append_layer_normed(0, q, k, v, qn, kn, want)
        blocks = torch.tensor(cache.blocks(), device="cuda")
    assert torch.equal(want[3, 1], torch.zeros(D, device="cuda"))
    keys = cache.layer_keys(0)
    assert torch.equal(keys[5, 0], torch.zeros(D, device="cuda"))
    kp, vp = pool.storage()
    assert tuple(kp.shape) == (1, 16, 2, 16, D)
    at = torch.arange(20, device="cuda")
    assert torch.equal(kp[0][blocks[at // 16], :, at % 16], keys)
    assert torch.equal(vp[0][blocks[at // 16], :, at % 16], v)
    cache.clear()
    with pool.begin([cache], 20) as b:
        b.append_layer_normed(0, q, k, v, qn, kn, q)
    assert torch.equal(q, want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("which,value", [("k", math.nan), ("k", math.inf), ("v", math.nan), ("v", -math.inf),
                                         ("k", 1e25)])
def test_normed_append_non_finite_fails_its_sequence(dtype, which, value):
    """1e25: a square sum past f32."""
    g = gen(2)
    pool = make_pool(dtype=dtype)
    caches = [pool.allocate_kv_cache(64) for _ in range(3)]
    q, k, v = randn(g, 9, 4, D), randn(g, 9, 2, D), randn(g, 9, 2, D)
    (k if which == "k" else v)[4, 1, 7] = value
    one = torch.ones(D, device="cuda")
    b = pool.begin(caches, 3)
    b.append_layer_normed(0, q, k, v, one, one, torch.empty_like(q))
    assert b.end(raise_on_error=False) == [0, slmkv.ERR_NON_FINITE, 0]
    assert [c.sequence_length() for c in caches] == [3, 0, 3]
    assert all(torch.isfinite(x.float()).all() for x in pool.storage())


def test_normed_append_refusals():
    pool = make_pool()
    cache = pool.allocate_kv_cache(64)
    g = gen(3)
    q, k, v, w = randn(g, 2, 4, D), randn(g, 2, 2, D), randn(g, 2, 2, D), torch.ones(D, device="cuda")
    out = torch.empty_like(q)
    b = pool.begin([cache], 2)

    def refused(match=None, **kw):
        a = dict(layer=0, query=q, keys=k, values=v, query_norm=w, key_norm=w, query_out=out)
        a.update(kw)
        with pytest.raises(slmkv.InvalidInput, match=match):
            b.append_layer_normed(**a)

    refused("epsilon", epsilon=0.0)
    refused("epsilon", epsilon=math.nan)
    refused("epsilon", epsilon=math.inf)
    refused("outside 0..1", layer=1)
    refused(query=q.double())
    refused(keys=k[:1])
    refused(values=v.cpu())
    refused(query_norm=w[:32])
    refused(query=q.transpose(0, 1).contiguous().transpose(0, 1))  # heads not dense
    both = torch.empty(q.numel() + 4 * D, device="cuda")
    refused("overlap", query=both[:q.numel()].view(q.shape), query_out=both[4 * D:].view(q.shape))
    refused("overlap", query=both[:q.numel()].view(q.shape), query_out=both[:q.numel()].view(q.shape), keys=both[:2 * 2 * D].view(k.shape))
    refused("aligned", query_out=torch.empty(q.numel() + 1, device="cuda")[1:].view(q.shape))
    refused("strides", query=torch.empty((2, 4 * D + 1), device="cuda")[:, :4 * D].view(2, 4, D))
    assert cache.layer_sequence_length(0) == 0
    b.append_layer_normed(0, q, k, v, w, w, out)
    refused("already appended")
    b.end()
    assert slmkv.lib().slm_batch_append_layer_normed(None, 0, None, None, None, 0, 0, 0, None, None, 1e-5, 1,
                                                     None) == slmkv.ERR_INVALID_INPUT


# ---- token probabilities ---------------------------------------------------------


def rows_batch(counts):
    pool = make_pool(2, 1, max(counts), len(counts))
    return pool, pool.begin([pool.allocate_kv_cache(max(counts)) for _ in counts], counts)


def probabilities_reference(x, t):
    x = x.double()
    out = torch.zeros_like(x)
    for i in range(x.shape[0]):
        if t[i] == 0:
            out[i, int(np.argmax(x[i].cpu().numpy()))] = 1
        else:
            out[i] = torch.softmax((x[i] - x[i].max()) / float(t[i]), 0)
    return out


def check_probabilities(got, x, t):
    """An exponent z = (x - max) log2(e) / T carries two roundings of its own
    (2^-23 |z|) and the difference's, the power and the sum a few units of 2^-22,
    so a probability is off by (3 |z| 2^-24 + 8 * 2^-22) of itself, or it is below
    the least normal number."""
    want = probabilities_reference(x, t)
    z = (x.double().max(1, keepdim=True)[0] - x.double()) / t.double().clamp_min(1e-300)[:, None] * 1.4427
    tol = want * (3 * z.clamp_max(1000) * 2.0**-24 + 8 * 2.0**-22) + 2.0**-126
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("vocab", [1, 2, 3, 31, 33, 127, 1000, 4096, 8192, 8193, 16390, 50021, 131072, 140003, 300001])
@pytest.mark.parametrize("rows", [1, 7])
def test_probabilities(vocab, rows):
    g = gen(vocab)
    pool, b = rows_batch([1] * rows)
    x = 3 * randn(g, rows, vocab)
    x[torch.rand((rows, vocab), generator=g, device="cuda") < 0.2] = -math.inf
    x[:, vocab // 2] = 0.5
    t = torch.tensor([1.0, 0.0, 0.25, 2.0, 1e-3, 1e-30, 1e30], device="cuda")[:rows]
    out = torch.full_like(x, math.nan)
    b.token_probabilities(x, out, t)
    check_probabilities(out, x, t)
    if rows == 1:
        b.token_probabilities(x, out)  # no temperatures: 1
        check_probabilities(out, x, torch.ones(1, device="cuda"))
    b.rollback()


def test_probabilities_strides_rows_a_sequence_and_in_place():
    g = gen(5)
    pool, b = rows_batch([3, 1, 5])
    wide = randn(g, 9, 1003)
    t = torch.full((9,), 0.7, device="cuda")
    out = torch.empty((9, 1001), device="cuda")
    for start in (0, 1, 2):  # rows that start anywhere in a 16-byte line
        x = wide[:, start:start + 1001]
        b.token_probabilities(x, out, t)
        check_probabilities(out, x, t)
    shifted = torch.empty(9 * 1001 + 3, device="cuda")[3:].view(9, 1001)
    b.token_probabilities(wide[:, :1001], shifted, t)
    check_probabilities(shifted, wide[:, :1001], t)
    for vocab in (1001, 40_001):  # in place, one row a sequence
        x = randn(g, 3, vocab)
        keep = x.clone()
        b.token_probabilities(x, x, t[:3].contiguous())
        check_probabilities(x, keep, t[:3])
    assert b.end(raise_on_error=False) == [slmkv.ERR_INVALID_INPUT] * 3  # no layer was appended


def test_probabilities_ties_and_extremes():
    pool, b = rows_batch([1] * 5)
    x = torch.full((5, 70), -math.inf, device="cuda")
    x[0, [13, 14, 69]] = 2.0      # a tie: the first
    x[1, 41] = -3e38              # a single token left
    x[2, :] = 3e38                # equal at the type's edge
    x[3, 0], x[3, 1] = 3e38, -3e38
    x[4, :] = torch.finfo(torch.float32).min  # a mask of the lowest value on every token
    out = torch.empty_like(x)
    b.token_probabilities(x, out, torch.zeros(5, device="cuda"))
    assert out.argmax(1).tolist() == [13, 41, 0, 0, 0] and torch.equal(out.sum(1), torch.ones(5, device="cuda"))
    b.token_probabilities(x, out)
    want = torch.zeros_like(x)
    want[0, [13, 14, 69]] = 1 / 3
    want[1, 41] = want[3, 0] = 1
    want[2] = want[4] = 1 / 70
    assert (out - want).abs().max().item() <= 8 * 2.0**-22
    b.rollback()


@pytest.mark.parametrize("vocab", [70, 20_003])
def test_probabilities_bad_rows_fail_their_sequences(vocab):
    counts = [2, 1, 1, 2, 1, 1, 1]
    pool, b = rows_batch(counts)
    x, t = randn(gen(6), 9, vocab), torch.ones(9, device="cuda")
    x[1, vocab - 1] = math.nan
    x[3] = -math.inf
    x[4, 17] = math.inf
    t[6], t[7] = -1.0, math.nan
    out = torch.full_like(x, 7.0)
    b.token_probabilities(x, out, t)
    sums = out.sum(1).tolist()
    assert [round(s, 3) for s in sums] == [1, 0, 1, 0, 0, 1, 0, 0, 1]
    one = torch.zeros((1, 2, D), device="cuda")
    b.append_layer(0, torch.zeros((9, 1, D), device="cuda"), torch.zeros((9, 1, D), device="cuda"))
    bad = slmkv.ERR_NON_FINITE
    assert b.end(raise_on_error=False) == [bad, 0, bad, bad, bad, bad, 0]
    with pytest.raises(slmkv.InvalidInput, match="give no distribution"):
        pool2, b = rows_batch([1])
        b.append_layer(0, one[:, :1], one[:, :1])
        b.token_probabilities(torch.full((1, 5), math.nan, device="cuda"), torch.empty((1, 5), device="cuda"))
        b.end()


def test_probabilities_refusals():
    pool, b = rows_batch([2, 1])
    x = torch.zeros((3, 8), device="cuda")
    out = torch.empty_like(x)
    for bad in (dict(logits=x[:1], probabilities=out[:1]), dict(probabilities=out[:2]), dict(logits=x.t()),
                dict(logits=x.double()), dict(logits=x[0]), dict(temperatures=torch.ones(2, device="cuda")),
                dict(temperatures=torch.ones(3)), dict(probabilities=torch.empty((3, 16), device="cuda")[:, :8]),
                dict(logits=x[:, :0], probabilities=out[:, :0])):
        a = dict(logits=x, probabilities=out, temperatures=None)
        a.update(bad)
        with pytest.raises(slmkv.InvalidInput):
            b.token_probabilities(**a)
    flat = torch.zeros(100, device="cuda")
    with pytest.raises(slmkv.InvalidInput, match="overlap"):
        b.token_probabilities(flat[:24].view(3, 8), flat[8:32].view(3, 8))
    with pytest.raises(slmkv.InvalidInput, match="overlap"):
        b.token_probabilities(x, flat[:24].view(3, 8), temperatures=flat[5:8])
    b.rollback()


# ---- verification of drafts --------------------------------------------------------


def verify_reference(counts, ids, p, q, u):
    """The definition, value by value, in 64 bits."""
    accepted, tokens, row = [], [], 0
    p, u = p.double().cpu().numpy(), u.double().cpu().numpy()
    q = None if q is None else q.double().cpu().numpy()
    for i, c in enumerate(counts):
        k, a = c - 1, 0
        while a < k:
            x = ids[row + a + 1]
            if not u[row + a] * (1.0 if q is None else q[row - i + a, x]) < p[row + a, x]:
                break
            a += 1
        w = p[row + a]
        if a < k:
            rest = w.copy()
            if q is None:
                rest[ids[row + a + 1]] = 0
            else:
                rest = np.maximum(w - q[row - i + a], 0)
            if rest.sum() > 0:
                w = rest
        run = np.cumsum(w)
        over = np.nonzero(run > u[row + k] * run[-1])[0]
        accepted.append(a)
        tokens.append(int(over[0]) if len(over) else int(np.nonzero(w)[0][-1]))
        row += c
    return accepted, tokens


def run_verify(counts, ids, p, q, u, end=False):
    pool, b = rows_batch(counts)
    acc = torch.full((len(counts),), -7, dtype=torch.int32, device="cuda")
    nxt = torch.full_like(acc, -7)
    b.verify_drafts(ids, p, q, u, acc, nxt)
    status = None
    if end:
        z = torch.zeros((sum(counts), 1, D), device="cuda")
        b.append_layer(0, z, z)
        status = b.end(raise_on_error=False)
    else:
        b.rollback()
    return acc.tolist(), nxt.tolist(), status


@pytest.mark.parametrize("vocab", [1, 2, 33, 128, 129, 1000, 8192, 50021, 200_003])
@pytest.mark.parametrize("counts", [[1], [4], [1, 2, 7, 1, 3, 5], [3] * 40])
@pytest.mark.parametrize("sampled", [True, False])
def test_verify(vocab, counts, sampled):
    counts = counts[:max(1, 6_000_000 // (vocab * counts[0]))]
    g = gen(vocab + len(counts))
    t, n = sum(counts), len(counts)
    p = torch.softmax(2 * randn(g, t, vocab), -1)
    q = torch.softmax(2 * randn(g, t - n, vocab), -1) if sampled and t > n else None
    if q is not None:  # drafts worth accepting now and then
        rows = [r for i, c in enumerate(counts) for r in range(sum(counts[:i]), sum(counts[:i]) + c - 1)]
        q = 0.5 * q + 0.5 * p[rows]
    ids = torch.randint(0, vocab, (t,), generator=g, device="cuda", dtype=torch.int32)
    for seed in range(3):
        u = torch.rand((t,), generator=gen(seed), device="cuda")
        if seed == 2:
            u[::2] = 0.0
        acc, nxt, _ = run_verify(counts, ids, p, q, u)
        want = verify_reference(counts, ids.tolist(), p, q, u)
        assert (acc, nxt) == want


@pytest.mark.parametrize("vocab", [8, 5000])
def test_verify_borders(vocab):
    """Weights that are exact in any order: draws at, below and above a border;
    u at its ends; equal distributions; a draft that its own model gives zero."""
    def row(**at):
        r = torch.zeros(vocab)
        for i, x in at.items():
            r[int(i[1:])] = x
        return r

    top = 1 - 2.0**-24
    last = vocab - 1
    half = row(_1=0.5, **{f"_{last}": 0.5})
    cases = [
        # (p rows, q rows, drafts, uniforms, accepted, next)
        ([half], [], [], [0.5], 0, last),           # the running sum has to exceed u
        ([half], [], [], [0.49999997], 0, 1),
        ([half], [], [], [0.0], 0, 1),              # never a token of weight zero
        ([half], [], [], [top], 0, last),
        ([half], [], [], [1.0], 0, last),           # past the end
        ([half], [], [], [-1.0], 0, 1),
        ([half, row(_3=1.0)], [half], [1], [top, 0.3], 1, 3),          # equal: accepted
        ([half, row(_3=1.0)], [row(_1=1.0)], [1], [0.5, 0.9], 0, last),  # u q < p fails at equality
        ([half, row(_3=1.0)], [row(_1=1.0)], [1], [0.49999997, 0.9], 1, 3),
        ([half, row(_3=1.0)], [half], [2], [0.0, 0.2], 0, 1),          # p = q, the draft has neither: p itself
        ([half, half, row(_4=2.0)], [half, half], [1, last], [0.9, 0.9, 0.1], 2, 4),  # not normalised
        ([half, half, row(_4=1.0)], [half, row(_1=0.25, _2=0.75)], [1, 2], [0.9, 0.0, 0.3], 1, 1),
        ([half, half, row(_4=1.0)], [half, row(_1=0.25, _2=0.75)], [1, 2], [0.9, 0.0, 0.34], 1, last),
    ]
    for p, q, drafts, u, acc, nxt in cases:
        counts = [len(drafts) + 1]
        ids = torch.tensor([0] + drafts, dtype=torch.int32, device="cuda")
        got = run_verify(counts, ids, torch.stack(p).cuda(), torch.stack(q).cuda() if q else None,
                         torch.tensor(u, device="cuda"))
        assert got[:2] == ([acc], [nxt]), (drafts, u)
    # drafts chosen outright: accepted with p, else another token
    ids = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    p = torch.stack([half, row(_3=1.0)]).cuda()
    assert run_verify([2], ids, p, None, torch.tensor([0.49999997, 0.0], device="cuda"))[:2] == ([1], [3])
    assert run_verify([2], ids, p, None, torch.tensor([0.5, 0.0], device="cuda"))[:2] == ([0], [last])


def test_verify_bad_inputs_fail_their_sequences():
    vocab, counts = 300, [2] * 8
    g = gen(9)
    p = torch.softmax(randn(g, 16, vocab), -1)
    q = torch.softmax(randn(g, 8, vocab), -1)
    ids = torch.zeros(16, dtype=torch.int32, device="cuda")
    u = torch.full((16,), 0.999, device="cuda")
    q[:, 0] = 1.0  # token 0 is always rejected, so rows 2i and q row i are read
    ids[3] = vocab
    ids[5] = -1
    p[6, 200] = math.nan
    p[8] = 0
    p[10, 5] = -0.5
    q[6, 299] = math.inf
    p[15, 7] = math.nan  # not read: the draft before it is rejected
    acc, nxt, status = run_verify(counts, ids, p, q, u, end=True)
    bad, token = slmkv.ERR_NON_FINITE, slmkv.ERR_INVALID_INPUT
    assert status == [0, token, token, bad, bad, bad, bad, 0]
    assert [x for x, s in zip(nxt, status) if s] == [-1] * 6 and acc == [0] * 8
    assert nxt[0] >= 0 and nxt[7] >= 0


def test_verify_refusals():
    pool, b = rows_batch([2, 1])
    ids = torch.zeros(3, dtype=torch.int32, device="cuda")
    p, q, u = torch.ones((3, 8), device="cuda"), torch.ones((1, 8), device="cuda"), torch.zeros(3, device="cuda")
    acc, nxt = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    good = dict(token_ids=ids, target=p, draft=q, uniforms=u, accepted=acc, next_tokens=nxt)
    for bad in (dict(token_ids=ids.long()), dict(token_ids=ids[:2]), dict(target=p[:2]), dict(target=p[0]),
                dict(draft=p), dict(draft=q[:, :4]), dict(uniforms=u.double()), dict(accepted=acc[:1]),
                dict(next_tokens=nxt.cpu()), dict(target=torch.ones((8, 3), device="cuda").t())):
        with pytest.raises(slmkv.InvalidInput):
            b.verify_drafts(**{**good, **bad})
    fn = slmkv.lib().slm_batch_verify_drafts
    ptr = [x.data_ptr() for x in (ids, p, q, u, acc, nxt)]
    assert fn(b._h, 0, *ptr) == slmkv.ERR_INVALID_INPUT
    assert fn(b._h, 655361, *ptr) == slmkv.ERR_INVALID_INPUT
    assert fn(b._h, 8, *ptr[:5], None) == slmkv.ERR_INVALID_INPUT
    b.rollback()


def test_verify_uniforms_outside_their_range():
    """They count as the nearer end, for the drafts as for the draw."""
    p = torch.tensor([[0.0, 0.5, 0.5], [1.0, 0.0, 0.0]], device="cuda")
    q = torch.tensor([[0.25, 0.375, 0.375]], device="cuda")
    for draft, u, acc, nxt in ((0, -1.0, 0, 1),       # 0 < p fails: p = 0
                               (1, 2.0, 1, 0),        # q < p, though 2 q > p
                               (1, -math.inf, 1, 0), (1, math.inf, 1, 0), (0, math.inf, 0, 2),
                               (1, math.nan, 1, 0)):  # as 0
        ids = torch.tensor([0, draft], dtype=torch.int32, device="cuda")
        uniforms = torch.tensor([u, u], device="cuda")
        assert run_verify([2], ids, p, q, uniforms)[:2] == ([acc], [nxt]), (draft, u)


def test_outputs_over_inputs_are_refused():
    pool, b = rows_batch([2, 1])
    words = torch.zeros(64, dtype=torch.int32, device="cuda")
    floats = words.view(torch.float32)
    good = dict(token_ids=words[:3], target=floats[8:32].view(3, 8), draft=floats[32:40].view(1, 8),
                uniforms=floats[40:43], accepted=words[44:46], next_tokens=words[46:48])
    for bad in (dict(accepted=words[2:4]), dict(next_tokens=words[30:32]), dict(accepted=words[39:41]),
                dict(next_tokens=words[42:44]), dict(next_tokens=words[45:47])):
        with pytest.raises(slmkv.InvalidInput, match="overlap"):
            b.verify_drafts(**{**good, **bad})
    fn = slmkv.lib().slm_batch_token_probabilities
    assert fn(b._h, floats[:4].data_ptr(), 3, 2**30 + 1, 2**30 + 1, None, 4) == slmkv.ERR_INVALID_INPUT
    b.rollback()
    g = gen(4)
    pool = make_pool()
    q, k, v = randn(g, 2, 4, D), randn(g, 2, 2, D), randn(g, 2, 2, D)
    buf = torch.ones(q.numel() + D, device="cuda")
    b = pool.begin([pool.allocate_kv_cache(64)], 2)
    for at in (0, q.numel() - D):
        w = buf[at:at + D]
        for norms in ((w, buf[-D:]), (buf[-D:], w)):
            with pytest.raises(slmkv.InvalidInput, match="overlap"):
                b.append_layer_normed(0, q, k, v, *norms, buf[:-D].view(q.shape))
    b.rollback()


# ---- together ------------------------------------------------------------------


def test_a_layer_of_a_speculative_step():
    """Normed append and shared attention of drafted rows over a common prefix,
    against both in 64 bits."""
    g = gen(20)
    hq, hkv, prefix, n = 8, 2, 80, 5
    counts, own = [1, 4, 3, 6, 2], [0, 5, 16, 31, 40]
    pool = make_pool(hq, hkv, 200, n)
    caches = [pool.allocate_kv_cache(200) for _ in range(n)]
    qn, kn = 1 + 0.3 * randn(g, D), 1 + 0.3 * randn(g, D)

    def rows(t):
        return randn(g, t, hq, D), randn(g, t, hkv, D), randn(g, t, hkv, D)

    hist, shared = [], rows(prefix)
    with pool.begin(caches[:1], prefix) as b:
        b.append_layer_normed(0, *shared, qn, kn, torch.empty_like(shared[0]))
    caches[0].publish_prefix(list(range(prefix)))
    for c in caches[1:]:
        assert c.attach_prefix(list(range(prefix))) == prefix
    hist = [rows(m) for m in own]
    some = [i for i in range(n) if own[i]]
    q, k, v = (torch.cat([hist[i][j] for i in some]) for j in range(3))
    with pool.begin([caches[i] for i in some], [own[i] for i in some]) as b:
        b.append_layer_normed(0, q, k, v, qn, kn, torch.empty_like(q))
    new = rows(sum(counts))
    q_out, out = torch.empty_like(new[0]), torch.empty_like(new[0])
    with pool.begin(caches, counts) as b:
        b.append_layer_normed(0, *new, qn, kn, q_out)
        b.shared_prefix_attention(0, q_out, out, rotate_query=False)
    row = 0
    for i, c in enumerate(counts):
        at = torch.arange(prefix + own[i] + c, device="cuda")
        k = torch.cat((shared[1], hist[i][1], new[1][row:row + c]))
        v = torch.cat((shared[2], hist[i][2], new[2][row:row + c])).double().repeat_interleave(4, 1)
        k = normed_reference(k, kn, 1e-5, at).repeat_interleave(4, 1)
        q = normed_reference(new[0][row:row + c], qn, 1e-5, at[-c:])
        s = torch.einsum("chd,nhd->hcn", q, k) / 8
        s = s.masked_fill((at[None] > at[-c:, None])[None], -math.inf)
        want = torch.einsum("hcn,nhd->chd", torch.softmax(s, -1), v)
        # normed rows are off by 16 * 2^-24 of at most ~8 each: scores by 64 *
        # 2 * 8 * 8 * 2^-20 / 8 at the very most, values are up to 5
        assert (out[row:row + c].double() - want).abs().max().item() <= 5e-3
        assert (out[row:row + c].double() - want).square().mean().sqrt().item() <= 1e-5
        row += c


def small_model(context=256, seqs=4, vocab=517, layers=2):
    pool = make_pool(4, 2, context, seqs, layers=layers)
    rng = np.random.default_rng(3)
    shapes = slmkv.model_tensor_shapes(vocab_size=vocab, hidden_size=256, intermediate_size=512, num_layers=layers,
                                       kv_width=128)
    tensors = [np.ones(s, np.float32) if len(s) == 1 else (rng.standard_normal(s) * 0.08).astype(np.float32)
               for _, s in shapes]
    return pool, slmkv.Model(pool, vocab_size=vocab, intermediate_size=512, tensors=tensors)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def test_model_score_projects_every_row():
    pool, model = small_model()
    caches = [pool.allocate_kv_cache(100) for _ in range(3)]
    prompts = [[5, 9, 100, 2], [7], list(range(30))]
    counts = [len(p) for p in prompts]
    logits = torch.empty((sum(counts), 517), device="cuda")
    nxt = torch.empty(sum(counts), dtype=torch.int32, device="cuda")
    with pool.begin(caches, counts) as b:
        model.score(b, ints(sum(prompts, [])), logits, nxt)
    assert torch.equal(nxt.long(), logits.argmax(1))
    # the same rows one token at a time
    row = 0
    for p in prompts:
        c = pool.allocate_kv_cache(100)
        one, tok = torch.empty((1, 517), device="cuda"), torch.empty(1, dtype=torch.int32, device="cuda")
        for j, t in enumerate(p):
            with pool.begin([c], 1) as b:
                model.decode(b, ints([t]), one, tok)
            # the exact-order path: equal but for the head's order of summation
            assert (one[0] - logits[row + j]).abs().max().item() <= 1e-4
        row += len(p)
        c.free()
    model.close()


def test_greedy_speculation_generates_the_greedy_tokens():
    """Drafts of mixed quality at temperature 0 through score, probabilities and
    verification: the tokens are those of plain greedy decoding."""
    pool, model = small_model()
    vocab, want, n = 517, [], 3
    prompts = [[5, 9, 100, 2], [7, 7], list(range(40, 70))]
    for p in prompts:  # plain greedy decoding
        c, tok = pool.allocate_kv_cache(120), torch.empty(1, dtype=torch.int32, device="cuda")
        with pool.begin([c], len(p)) as b:
            model.prefill(b, ints(p), None, tok)
        got = [int(tok)]
        while len(got) < 24:
            with pool.begin([c], 1) as b:
                model.decode(b, ints(got[-1:]), None, tok)
            got.append(int(tok))
        want.append(got)
        c.free()
    rng = np.random.default_rng(1)
    caches = [pool.allocate_kv_cache(120) for _ in prompts]
    tok = torch.empty(n, dtype=torch.int32, device="cuda")
    with pool.begin(caches, [len(p) for p in prompts]) as b:
        model.prefill(b, ints(sum(prompts, [])), None, tok)
    got = [[t] for t in tok.tolist()]
    rounds = 0
    while min(map(len, got)) < 20:
        rows, counts = [], []
        for i in range(n):
            k = int(rng.integers(0, 4))
            draft = want[i][len(got[i]):len(got[i]) + k]
            if draft and rng.random() < 0.5:
                draft[int(rng.integers(len(draft)))] = int(rng.integers(vocab))  # a wrong one
            rows += [got[i][-1]] + draft
            counts.append(1 + len(draft))
        base = [c.sequence_length() for c in caches]
        t = sum(counts)
        logits = torch.empty((t, vocab), device="cuda")
        acc, nxt = torch.empty(n, dtype=torch.int32, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda")
        with pool.begin(caches, counts) as b:
            model.score(b, ints(rows), logits)
            b.token_probabilities(logits, logits, torch.zeros(t, device="cuda"))
            b.verify_drafts(ints(rows), logits, None, torch.rand(t, device="cuda"), acc, nxt)
        at = 0
        for i, a in enumerate(acc.tolist()):
            got[i] += rows[at + 1:at + 1 + a] + [nxt.tolist()[i]]
            at += counts[i]
        pool.truncate_many(caches, [x + 1 + a for x, a in zip(base, acc.tolist())])
        rounds += 1
        assert rounds < 40
        for i in range(n):
            m = min(len(got[i]), len(want[i]))
            assert got[i][:m] == want[i][:m]
            if len(got[i]) > 20:  # keep drafting from what is known
                got[i] = got[i][:20]
                pool.truncate_many([caches[i]], [len(prompts[i]) + 19])
    model.close()


def test_sampled_speculation_follows_the_targets_distribution():
    """First tokens drawn through drafts from another distribution have the
    target's frequencies: 20000 draws of 6 tokens, each count within 6 standard
    deviations of its expectation."""
    vocab, n = 6, 200
    g = gen(4)
    p = torch.softmax(randn(g, vocab), -1)
    q = torch.softmax(randn(g, vocab), -1)
    counts = [2] * n
    freq = np.zeros(vocab)
    pool, b = rows_batch(counts)
    target, draft = p.expand(2 * n, vocab).contiguous(), q.expand(n, vocab).contiguous()
    acc, nxt = torch.empty(n, dtype=torch.int32, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda")
    for _ in range(100):
        x = torch.multinomial(q, n, replacement=True, generator=g).int()
        ids = torch.stack((torch.zeros_like(x), x), 1).flatten().contiguous()
        b.verify_drafts(ids, target, draft, torch.rand((2 * n,), generator=g, device="cuda"), acc, nxt)
        first = torch.where(acc > 0, x, nxt)
        freq += np.bincount(first.cpu().numpy(), minlength=vocab)
    b.rollback()
    expect = p.cpu().numpy().astype(np.float64)
    sd = np.sqrt(20000 * expect * (1 - expect))
    assert (np.abs(freq - 20000 * expect) <= 6 * sd).all(), (freq, 20000 * expect)
