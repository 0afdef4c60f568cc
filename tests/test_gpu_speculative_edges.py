"""The speculative step's operators at the ends of what their calls allow:
vocabularies beyond a cluster's shared memory, temperatures at the ends of f32,
probabilities that are none at accepted drafts, captured calls that are refused
or dropped, and the model's scores on each of its projection paths."""

import gc
import math

import numpy as np
import pytest

import oracle as O

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
slmkv = pytest.importorskip("slmkv")

from test_gpu_model import parity_metrics, random_model  # noqa: E402
from test_gpu_speculative_step import (D, check_probabilities, gen, randn, rows_batch, run_verify,  # noqa: E402
                                       verify_reference)


# ---- token probabilities ---------------------------------------------------------


@pytest.mark.parametrize("vocab", [458_745, 458_752, 458_753, 458_761, 500_003, 1_000_001])
@pytest.mark.parametrize("rows,start", [(1, 0), (4, 1)])
def test_probabilities_of_rows_beyond_shared_memory(vocab, rows, start):
    g = gen(vocab)
    pool, b = rows_batch([1] * rows)
    wide = 3 * randn(g, rows, vocab + 3)
    wide[torch.rand(wide.shape, generator=g, device="cuda") < 0.2] = -math.inf
    wide[:, vocab // 2] = 0.5
    t = torch.tensor([1.0, 0.0, 0.25, 3e38], device="cuda")[:rows]
    x = wide[:, start:start + vocab]
    out = torch.full((rows, vocab), math.nan, device="cuda")
    b.token_probabilities(x, out, t)
    check_probabilities(out, x, t)
    here = x.clone()
    b.token_probabilities(here, here, t)  # in place
    check_probabilities(here, x, t)
    x[0, vocab - 1] = math.nan
    b.token_probabilities(x, out, t)
    assert not out[0].any() and (rows == 1 or out[1:].sum(1).sub(1).abs().max() < 1e-4)
    b.rollback()


@pytest.mark.parametrize("vocab", [300_001, 2**24 + 3])
def test_probabilities_of_many_equal_weights(vocab):
    """A sum of equal weights that are no power of two: each addition is rounded
    the same way, so a long chain of them in 32 bits would drift."""
    pool, b = rows_batch([1])
    x = torch.full((1, vocab), -0.3, device="cuda")
    x[0, 5] = 0.0
    b.token_probabilities(x, x)
    w = math.exp(float(np.float32(-0.3)))
    want = w / (1 + (vocab - 1) * w)
    # as check_probabilities: two roundings of an exponent of 0.43, a few of 2^-22
    tol = want * (2 * 2.0**-24 + 8 * 2.0**-22)
    assert abs(x[0, 0].item() - want) <= tol and abs(x[0, -1].item() - want) <= tol
    assert abs(x[0, 5].item() - want / w) <= tol / w
    b.rollback()


def test_probabilities_at_temperatures_near_the_ends_of_f32():
    """Logits at f32's ends differ by more than f32 holds, and a temperature as
    large makes that difference a small number again."""
    top = torch.finfo(torch.float32).max
    t = torch.tensor([1e38, 3e38, top, 1e37, 2.0**100, 1.0, 2.0**-126, 1e-37, 4.0], device="cuda")
    pool, b = rows_batch([1] * len(t))
    x = torch.full((len(t), 41), -3e38, device="cuda")
    x[:, 3], x[:, 4], x[:, 5], x[:, 6] = 3e38, 2.9e38, -top, top
    x[6] = torch.linspace(0, 40, 41, device="cuda") * 2.0**-126
    x[7] = torch.linspace(-20, 20, 41, device="cuda") * 1e-37
    x[8] = torch.linspace(-60, 60, 41, device="cuda")
    out = torch.empty_like(x)
    b.token_probabilities(x, out, t)
    check_probabilities(out, x, t)
    big = x.repeat(1, 400)  # a cluster a row, some slices without the maximum
    big[:, 41:] = torch.minimum(big[:, 41:], big[:, :1])
    out = torch.empty_like(big)
    b.token_probabilities(big, out, t)
    check_probabilities(out, big, t)
    b.rollback()


def test_temperatures_below_the_normal_numbers_count_as_the_least_normal_one():
    pool, b = rows_batch([1] * 3)
    x = (torch.arange(12, device="cuda") * 2.0**-127).repeat(3, 1)
    out = torch.empty_like(x)
    b.token_probabilities(x, out, torch.tensor([1e-45, 1e-40, 2.0**-126], device="cuda"))
    assert torch.equal(out[0], out[2]) and torch.equal(out[1], out[2])
    check_probabilities(out, x, torch.full((3,), 2.0**-126, device="cuda"))
    b.rollback()


# ---- verification ------------------------------------------------------------------


def test_verify_values_that_are_no_probabilities_fail_at_accepted_drafts():
    """What the acceptance of a draft reads has to be a probability, as the rows
    have to: else the sequence fails. Behind the first rejected draft nothing is
    read."""
    vocab, bad = 300, slmkv.ERR_NON_FINITE
    cases = [  # (p at the draft, q at the draft, status); u is 0.5
        (0.5, 0.25, 0), (math.inf, 0.25, bad), (0.5, -0.25, bad), (0.5, -math.inf, bad), (math.inf, math.inf, bad),
        (math.nan, 0.25, bad), (0.5, math.nan, bad), (-0.5, -2.0, bad), (0.5, math.inf, bad), (-0.0, -0.0, 0)]
    n = len(cases)
    p = torch.full((3 * n, vocab), 1 / 512, device="cuda")
    q = torch.full((2 * n, vocab), 1 / 512, device="cuda")
    ids = torch.tensor([0, 7, 9] * n, dtype=torch.int32, device="cuda")
    for i, (x, y, _) in enumerate(cases):
        p[3 * i, 7], q[2 * i, 7] = x, y
    u = torch.full((3 * n,), 0.5, device="cuda")
    acc, nxt, status = run_verify([3] * n, ids, p, q, u, end=True)
    assert status == [c[2] for c in cases]
    assert [a for a, s in zip(acc, status) if s == 0] == [2, 0]
    assert all((a, t) == (0, -1) for a, t, s in zip(acc, nxt, status) if s)
    # the second draft's values, the first one accepted or not
    for first, want in ((0.5, bad), (0.0, 0)):
        p[:], q[:] = 1 / 512, 1 / 512
        p[0::3, 7], p[1::3, 9] = first, math.inf
        _, _, status = run_verify([3] * n, ids, p, q, u, end=True)
        assert status == [want] * n
    # drafts chosen outright
    p[:] = 1 / 512
    p[0::3, 7], p[3, 7], p[6, 7] = 0.75, math.inf, math.nan
    _, _, status = run_verify([3] * n, ids, p, None, u, end=True)
    assert status == [0, bad, bad] + [0] * (n - 3)


@pytest.mark.parametrize("vocab,n", [(81_921, 300), (655_360, 80), (655_360, 1), (655_231, 3), (400_001, 150)])
def test_verify_wide_rows_of_many_sequences(vocab, n):
    """More tiles than a CTA's sums have room for, where the number of sequences
    alone asks for fewer CTAs a row; weights that are exact in any order."""
    g = gen(vocab + n)
    p = torch.zeros((n, vocab), device="cuda")
    at = torch.randint(0, vocab, (n, 40), generator=g, device="cuda")
    at[:, 0], at[:, 1] = 0, vocab - 1
    p.scatter_(1, at, torch.randint(1, 1000, at.shape, generator=g, device="cuda") / 1024.0)
    u = torch.rand((n,), generator=g, device="cuda")
    ids = torch.zeros(n, dtype=torch.int32, device="cuda")
    acc, nxt, _ = run_verify([1] * n, ids, p, None, u)
    assert acc == [0] * n
    for i in range(n):
        x = torch.unique(at[i]).cpu().numpy()  # ascending
        run = np.cumsum(p[i].cpu().numpy()[x].astype(np.float64))
        assert nxt[i] == x[np.nonzero(run > float(u[i]) * run[-1])[0][0]]


def test_verify_dense_rows_at_the_widest():
    g = gen(77)
    counts, vocab = [2, 1, 3], 655_360
    p, q = torch.softmax(2 * randn(g, 6, vocab), -1), torch.softmax(2 * randn(g, 3, vocab), -1)
    ids = torch.randint(0, vocab, (6,), generator=g, device="cuda", dtype=torch.int32)
    u = torch.rand((6,), generator=g, device="cuda")
    acc, nxt, _ = run_verify(counts, ids, p, q, u)
    assert (acc, nxt) == verify_reference(counts, ids.tolist(), p, q, u)


# ---- calls under capture -------------------------------------------------------------


def one_layer_pool(hq=4, hkv=2, seqs=3, context=128):
    pool = slmkv.KvPool(num_layers=1, num_query_heads=hq, num_key_value_heads=hkv, context_length=context,
                        num_blocks=40, max_sequences=seqs)
    pool.shuffle(3)
    return pool


def test_a_first_call_refused_under_capture_leaves_nothing_in_the_graph():
    """A decode step leaves its new block's table entry to the next call that
    reads the table: a refused call must not put it into a graph that is dropped."""
    g = gen(31)
    pool = one_layer_pool()
    cache = pool.allocate_kv_cache(128)
    k, v = randn(g, 16, 2, D), randn(g, 16, 2, D)
    cache.append_layer(0, k, v, 16)
    assert cache.blocks() != [0]
    q, nk, nv = randn(g, 1, 4, D), randn(g, 1, 2, D), randn(g, 1, 2, D)
    want, out = torch.empty_like(q), torch.empty_like(q)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        b = pool.begin([cache], 1)
        assert 0 not in cache.blocks()  # (an entry that was never written is 0)
        b.decode_layer(0, q, nk, nv, want)
        graph = torch.cuda.CUDAGraph()
        before = pool.launch_count()
        with torch.cuda.graph(graph, stream=stream):
            torch.ones(1, device="cuda")  # (a graph of something)
            with pytest.raises(slmkv.InvalidInput, match="captured"):
                b.shared_prefix_attention(0, q, out)
        assert pool.launch_count() == before
        del graph
        gc.collect()
        b.shared_prefix_attention(0, q, out)
        b.end()
    # both are f32 means of 17 values of N(0, 1)
    assert (out - want).abs().max().item() <= 2e-5


def test_a_captured_call_takes_no_other_sequences_table_entries():
    """Blocks that another sequence got meanwhile are no part of the graph: it
    may be dropped, or replayed when they are another's."""
    g = gen(32)
    pool = one_layer_pool()
    a, c, d = (pool.allocate_kv_cache(128) for _ in range(3))
    tokens = list(range(32))
    k, v = randn(g, 32, 2, D), randn(g, 32, 2, D)
    a.append_layer(0, k, v, 32)
    a.publish_prefix(tokens)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    q, nk, nv = randn(g, 2, 4, D), randn(g, 2, 2, D), randn(g, 2, 2, D)
    out = torch.empty_like(q)
    with torch.cuda.stream(stream):
        b = pool.begin([a], 2)
        b.append_layer(0, nk, nv)
        b.shared_prefix_attention(0, q, out)
        assert c.attach_prefix(tokens) == 32  # its table entries wait for a call that reads them
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            b.shared_prefix_attention(0, q, out)
        del graph
        gc.collect()
        b.end()
        assert 0 not in c.blocks()
        again = torch.empty_like(q)
        with pool.begin([c], 2) as b:
            b.append_layer(0, nk, nv)
            b.shared_prefix_attention(0, q, again)
    stream.synchronize()
    assert torch.equal(out, again)  # the same tokens, read alike


def test_a_captured_step_of_all_operators():
    """Appends, attention, probabilities and verification in one graph, replayed
    on new contents: the same as the calls themselves."""
    g = gen(35)
    n, hq, hkv, layers, vocab = 5, 8, 2, 3, 1001
    pool = slmkv.KvPool(num_layers=layers, num_query_heads=hq, num_key_value_heads=hkv, context_length=256,
                        num_blocks=100, max_sequences=n)
    caches = [pool.allocate_kv_cache(256) for _ in range(n)]
    lengths, counts = [30, 16, 1, 100, 64], [3, 1, 4, 2, 2]
    t = sum(counts)
    with pool.begin(caches, lengths) as b:
        for layer in range(layers):
            b.append_layer(layer, randn(g, sum(lengths), hkv, D), randn(g, sum(lengths), hkv, D))
    q, k, v, w = randn(g, t, hq, D), randn(g, t, hkv, D), randn(g, t, hkv, D), randn(g, D).abs() + 0.5
    turned, outs = torch.empty_like(q), [torch.empty_like(q) for _ in range(layers)]
    logits, temperatures = randn(g, t, vocab), torch.full((t,), 0.8, device="cuda")
    draft, u = torch.softmax(randn(g, t - n, vocab), -1), torch.rand((t,), generator=g, device="cuda")
    ids = torch.randint(0, vocab, (t,), generator=g, device="cuda", dtype=torch.int32)
    p, acc = torch.empty_like(logits), torch.empty(n, dtype=torch.int32, device="cuda")
    nxt = torch.empty_like(acc)

    def step(b, first):
        for layer in range(first, layers):
            b.append_layer_normed(layer, q, k, v, w, w, turned)
            b.shared_prefix_attention(layer, turned, outs[layer], rotate_query=False)
        b.token_probabilities(logits, p, temperatures)
        b.verify_drafts(ids, p, draft, u, acc, nxt)

    def results():
        return [x.clone() for x in (*outs[1:], p, acc, nxt)]

    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        b = pool.begin(caches, counts)
        b.append_layer_normed(0, q, k, v, w, w, turned)
        b.shared_prefix_attention(0, turned, outs[0], rotate_query=False)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step(b, 1)
        for x in (q, k, v, logits):
            x.copy_(randn(g, *x.shape))
        graph.replay()
        graph.replay()
        got = results()
        stream.synchronize()
        del graph
        assert b.end() == [0] * n
        pool.truncate_many(caches, lengths)
        with pool.begin(caches, counts) as b:
            step(b, 0)
        want = results()
    stream.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


# ---- streams -------------------------------------------------------------------------


def test_batches_on_streams_that_come_and_go():
    """Each step on a stream of its own, destroyed while its kernels may run;
    the joined parts' scratch passes from one to the next."""
    import ctypes

    cudart = ctypes.CDLL("libcudart.so.12")
    g = gen(33)
    pool = slmkv.KvPool(num_layers=1, num_query_heads=8, num_key_value_heads=2, context_length=1100, num_blocks=400,
                        max_sequences=64)
    caches = [pool.allocate_kv_cache(1100) for _ in range(64)]
    k, v = randn(g, 1024, 2, D), randn(g, 1024, 2, D)
    caches[0].append_layer(0, k, v, 1024)
    caches[0].publish_prefix([1] * 1024)
    for c in caches[1:]:
        c.attach_prefix([1] * 1024)
    q, nk, nv = randn(g, 64, 8, D), randn(g, 64, 2, D), randn(g, 64, 2, D)
    torch.cuda.synchronize()
    outs = []
    for _ in range(12):
        h = ctypes.c_void_p()
        assert cudart.cudaStreamCreateWithFlags(ctypes.byref(h), 1) == 0
        out = torch.empty_like(q)
        torch.cuda.synchronize()
        b = pool.begin(caches, 1, stream=torch.cuda.ExternalStream(h.value))
        b.append_layer(0, nk, nv)
        b.shared_prefix_attention(0, q, out)
        b.rollback()
        assert cudart.cudaStreamDestroy(h) == 0
        outs.append(out)
    torch.cuda.synchronize()
    assert all(torch.equal(outs[0], o) for o in outs[1:])


# ---- the model's scores ----------------------------------------------------------------


@pytest.mark.parametrize("kv_dtype", [slmkv.KV_F32, slmkv.KV_BF16])
@pytest.mark.parametrize("exact_rows,lengths", [
    (1024, [5, 1, 33]),            # the exact-order kernels
    (0, [5, 1, 33]),               # this library's row GEMMs, the split head
    (0, [17, 64, 100, 250]),       # the same, more rows than one tile
    (0, [200, 120, 1, 255]),       # cuBLAS, as many vocabulary rows
    (16, [1, 3, 7])])
def test_model_scores_of_every_row_on_each_projection_path(exact_rows, lengths, kv_dtype):
    """Every position's logits against the oracle's, by the thresholds that the
    model's other steps are held to on that path."""
    vocab, hq, hkv, inter, layers, ctx = 1024, 4, 2, 704, 2, 256
    hidden = hq * D
    tensors = random_model(7, vocab, hidden, hkv, inter, layers, scale=0.8 / np.sqrt(hidden))
    omodel = O.Model(dict(vocab_size=vocab, hidden_size=hidden, intermediate_size=inter, num_layers=layers,
                          num_query_heads=hq, num_key_value_heads=hkv, head_dimension=D, rms_norm_epsilon=1e-5,
                          rope_theta=10000.0, situ_beta_gate=4.0, situ_beta_up=25.0), tensors)
    pool = slmkv.KvPool(num_layers=layers, num_query_heads=hq, num_key_value_heads=hkv, context_length=ctx,
                        num_blocks=len(lengths) * (ctx // 16 + 1), max_sequences=len(lengths), kv_dtype=kv_dtype)
    pool.shuffle(5)
    model = slmkv.Model(pool, vocab_size=vocab, intermediate_size=inter, tensors=tensors)
    model.set_exact_rows(exact_rows)
    rng = np.random.default_rng(sum(lengths))
    prompts = [rng.integers(0, vocab, n).astype(np.uint32) for n in lengths]
    ref = np.concatenate([omodel.prefill(omodel.new_cache(ctx, quantize_bf16=kv_dtype == slmkv.KV_BF16), p,
                                         O.max_threads()) for p in prompts])
    t = sum(lengths)
    logits = torch.full((t, vocab), math.nan, device="cuda")
    nxt = torch.empty(t, dtype=torch.int32, device="cuda")
    caches = [pool.allocate_kv_cache(ctx) for _ in lengths]
    with pool.begin(caches, lengths) as b:
        model.score(b, torch.from_numpy(np.concatenate(prompts).astype(np.int32)).cuda(), logits, nxt)
    assert torch.equal(nxt.long(), logits.argmax(1))
    m = parity_metrics(logits.cpu().numpy(), ref)
    # (top1 of hundreds of rows may meet near ties: held by the errors instead)
    assert m["max_abs"] <= 0.1 and m["mean_abs"] <= 0.01 and m["rms"] <= 0.02 and m["cosine"] >= 0.9999, m
    if t <= exact_rows and kv_dtype == slmkv.KV_F32:
        assert m["max_abs"] <= 1e-4, m  # (a bf16 pool holds keys and values to 2^-9 that the oracle's prompts do not round)
    last = np.cumsum(lengths) - 1
    one = torch.empty((len(lengths), vocab), device="cuda")
    pool.truncate_many(caches, [0] * len(lengths))
    with pool.begin(caches, lengths) as b:
        model.prefill(b, torch.from_numpy(np.concatenate(prompts).astype(np.int32)).cuda(), one)
    # the same layers; the vocabulary projection of other row counts sums in
    # another order, or over split operands: 2^-14 of |x| |w| = 16 * 0.8 at most
    assert (one - logits[torch.from_numpy(last).cuda()]).abs().max().item() <= 16 * 0.8 * 1.3 * 2.0**-14
    model.close()


# ---- Python arguments ------------------------------------------------------------------


def test_layers_and_epsilon_of_numpy_types_are_taken():
    """As the batch's other calls take them."""
    g = gen(34)
    pool = slmkv.KvPool(num_layers=2, num_query_heads=4, num_key_value_heads=2, context_length=64, num_blocks=8,
                        max_sequences=1)
    cache = pool.allocate_kv_cache(64)
    q, k, v, w = randn(g, 2, 4, D), randn(g, 2, 2, D), randn(g, 2, 2, D), torch.ones(D, device="cuda")
    outs = [[torch.empty_like(q) for _ in range(2)] for _ in range(2)]
    with pool.begin([cache], 2) as b:
        for layer, i in ((0, 0), (np.int64(1), 1)):
            b.append_layer_normed(layer, q, k, v, w, w, outs[i][0], epsilon=np.float32(1e-5) if i else 1e-5)
            b.shared_prefix_attention(layer, outs[i][0], outs[i][1], rotate_query=False)
    assert all(torch.equal(a, c) for a, c in zip(*outs))
