"""Attention over caches that share prefixes (Batch.shared_prefix_attention)
against softmax attention in 64 bits on the same keys and values: trees of
shared blocks, lengths around block borders, drafted rows, long splits, both
pool types, and the calls it refuses."""

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
slmkv = pytest.importorskip("slmkv")

D = 64


class Forest:
    """Sequences whose cached tokens are paths of token lists: equal leading
    full blocks are attached from the prefix index, the rest appended."""

    def __init__(self, hq, hkv, paths, counts, dtype="f32", layers=1, seed=0, scale=1.0, context=None,
                 blocks=None):
        self.hq, self.hkv, self.counts, self.layers = hq, hkv, counts, layers
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)
        self.scale = scale
        lens = [len(p) + c for p, c in zip(paths, counts)]
        self.pool = slmkv.KvPool(
            num_layers=layers, num_query_heads=hq, num_key_value_heads=hkv,
            context_length=context or max(lens), num_blocks=blocks or sum(x // 16 + 2 for x in lens),
            max_sequences=len(paths), kv_dtype=slmkv.KV_BF16 if dtype == "bf16" else slmkv.KV_F32)
        self.pool.shuffle(seed)
        self.caches = [self.pool.allocate_kv_cache(context or max(lens)) for _ in paths]
        self.kv = {}  # (layer, token path) -> the cached k, v
        self.dtype = torch.bfloat16 if dtype == "bf16" else torch.float32
        for cache, path in zip(self.caches, paths):
            have = cache.attach_prefix(path) if path else 0
            for layer in range(layers):
                if len(path) > have:
                    k = torch.stack([self.value(layer, path[:i + 1])[0] for i in range(have, len(path))])
                    v = torch.stack([self.value(layer, path[:i + 1])[1] for i in range(have, len(path))])
                    cache.append_layer(layer, k, v, len(path) - have)
            if path:
                cache.publish_prefix(path)
        self.paths = paths
        self.reused = self.pool.stats()[1]

    def randn(self, *size):
        return torch.randn(size, generator=self.g, device="cuda") * self.scale

    def value(self, layer, path):
        key = (layer, tuple(path))
        if key not in self.kv:
            self.kv[key] = (self.randn(self.hkv, D), self.randn(self.hkv, D))
        return self.kv[key]

    def new_rows(self):
        t = sum(self.counts)
        return self.randn(t, self.hq, D), self.randn(t, self.hkv, D), self.randn(t, self.hkv, D)

    def cached(self, i, layer):
        if not self.paths[i]:
            return torch.empty((0, self.hkv, D), device="cuda"), torch.empty((0, self.hkv, D), device="cuda")
        got = [self.value(layer, self.paths[i][:j + 1]) for j in range(len(self.paths[i]))]
        return torch.stack([a for a, _ in got]), torch.stack([b for _, b in got])

    def reference(self, layer, q, k, v):
        """(out, bound on the kernel's error) in 64 bits."""
        out, tol, row = torch.empty_like(q, dtype=torch.float64), 0.0, 0
        rep = self.hq // self.hkv
        for i, c in enumerate(self.counts):
            ck, cv = self.cached(i, layer)
            kk = torch.cat((ck, k[row:row + c])).to(self.dtype).double().repeat_interleave(rep, 1)
            vv = torch.cat((cv, v[row:row + c])).to(self.dtype).double().repeat_interleave(rep, 1)
            qq = q[row:row + c].double()
            n = kk.shape[0]
            s = torch.einsum("chd,nhd->hcn", qq, kk) / 8
            ahead = torch.arange(n, device="cuda")[None] > (n - c + torch.arange(c, device="cuda"))[:, None]
            w = torch.softmax(s.masked_fill(ahead[None], -math.inf), -1)
            out[row:row + c] = torch.einsum("hcn,nhd->chd", w, vv)
            # A score is a sum of 64 exact products taken in f32 in at most 12
            # chained groups (24 for f32 pools), each cut at 2^-23 of the sum of
            # magnitudes, after a query scaled with one rounding; a weight is off
            # by that (in the exponent) and a few units of 2^-22 for the
            # exponential and the running rescales, on both the sum and the
            # products; the result is a mean of values.
            mag = (torch.einsum("chd,nhd->hcn", qq.abs(), kk.abs()) / 8).max().item()
            tol = max(tol, 2 * ((26 * mag) * 2.0**-23 + 16 * 2.0**-22) * vv.abs().max().item())
            row += c
        return out, tol

    def attend(self, batch, layer, rows, **kw):
        q, k, v = rows
        out = torch.empty_like(q)
        batch.append_layer(layer, k, v, rotate_keys=False)
        batch.shared_prefix_attention(layer, q, out, rotate_query=False, **kw)
        return out

    def check(self):
        rows = [self.new_rows() for _ in range(self.layers)]
        with self.pool.begin(self.caches, self.counts) as b:
            outs = [self.attend(b, layer, rows[layer]) for layer in range(self.layers)]
        for layer, (out, r) in enumerate(zip(outs, rows)):
            ref, tol = self.reference(layer, *r)
            err = (out.double() - ref).abs().max().item()
            assert err <= tol, (layer, err, tol)


def path(*runs):
    """A token path from (first token, length) runs."""
    return [t for first, n in runs for t in range(first, first + n)]


HEADS = [(4, 2), (8, 8), (8, 2), (8, 1)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_nothing_shared_lengths_around_block_borders(hq, hkv, dtype):
    lens = [0, 1, 14, 15, 16, 17, 31, 32, 33, 63, 64, 127, 128, 129]
    Forest(hq, hkv, [path((1000 * (i + 1), n)) for i, n in enumerate(lens)], [1] * len(lens), dtype).check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hq,hkv", HEADS)
@pytest.mark.parametrize("prefix", [16, 64, 80, 144, 400])
def test_one_prefix_for_all(hq, hkv, prefix, dtype):
    tails = [0, 1, 15, 16, 17, 40, 100]
    paths = [path((1, prefix), (1000 * (i + 1), n)) for i, n in enumerate(tails)]
    f = Forest(hq, hkv, paths, [1] * len(tails), dtype, seed=prefix)
    assert len({c.blocks()[0] for c in f.caches}) == 1  # it is shared
    f.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_drafted_rows(hq, hkv, dtype):
    """Up to 21 new tokens a sequence: several row tiles, each row its own mask."""
    counts = [1, 2, 5, 3, 8, 16, 17, 21]
    paths = [path((1, 96), (1000 * (i + 1), 7 * i)) for i in range(len(counts))]
    Forest(hq, hkv, paths, counts, dtype, layers=2, seed=3).check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_levels_of_sharing(dtype):
    """All share 64 tokens, groups share more, one group splits again; one
    sequence shares nothing, one only less than a useful run."""
    a = (1, 64)
    paths = [path(a, (100, 80), (10_000, 5)), path(a, (100, 80), (200, 160), (20_000, 33)),
             path(a, (100, 80), (200, 160), (30_000, 0)), path(a, (500, 96), (40_000, 1)),
             path(a, (500, 96), (50_000, 50)), path(a, (60_000, 3)), path((70_000, 90)),
             path(a, (100, 80), (200, 160), (600, 64), (80_000, 9)),
             path(a, (100, 80), (200, 160), (600, 64), (90_000, 16)), path(a[:1] + (32,), (95_000, 40))]
    order = [3, 0, 8, 6, 1, 5, 2, 7, 4, 9]  # members of a group not next to each other
    Forest(4, 2, [paths[i] for i in order], [1, 2, 1, 3, 1, 1, 4, 1, 2, 1], dtype, layers=2, seed=11).check()


@pytest.mark.parametrize("dtype,hq,hkv", [("f32", 4, 2), ("bf16", 8, 2)])
def test_many_sequences(dtype, hq, hkv):
    n = 150
    paths = [path((1, 160), (1000 * (i + 1), (37 * i) % 70)) for i in range(n)]
    Forest(hq, hkv, paths, [1 + i % 3 for i in range(n)], dtype, seed=5).check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hq,hkv,length,count", [(2, 2, 20_001, 1), (8, 1, 9_000, 5)])
def test_one_long_sequence_is_split(dtype, hq, hkv, length, count):
    """Bulk keys: the split runs of one sequence, joined."""
    g = torch.Generator(device="cuda")
    g.manual_seed(length)
    kd = torch.bfloat16 if dtype == "bf16" else torch.float32
    k = torch.randn((length + count, hkv, D), generator=g, device="cuda").to(kd)
    v = torch.randn((length + count, hkv, D), generator=g, device="cuda").to(kd)
    q = torch.randn((count, hq, D), generator=g, device="cuda")
    pool = slmkv.KvPool(num_layers=1, num_query_heads=hq, num_key_value_heads=hkv, context_length=length + count,
                        num_blocks=length // 16 + 2, max_sequences=1,
                        kv_dtype=slmkv.KV_BF16 if dtype == "bf16" else slmkv.KV_F32)
    pool.shuffle(7)
    cache = pool.allocate_kv_cache(length + count)
    cache.append_layer(0, k[:length].float(), v[:length].float(), length)
    out, again = torch.empty_like(q), torch.empty_like(q)
    with pool.begin([cache], count) as b:
        b.append_layer(0, k[length:].float(), v[length:].float(), rotate_keys=False)
        b.shared_prefix_attention(0, q, out, rotate_query=False)
        b.shared_prefix_attention(0, q, again, rotate_query=False)
    rep = hq // hkv
    kk, vv = k.double().repeat_interleave(rep, 1), v.double().repeat_interleave(rep, 1)
    s = torch.einsum("chd,nhd->hcn", q.double(), kk) / 8
    ahead = torch.arange(length + count, device="cuda")[None] > (length + torch.arange(count, device="cuda"))[:, None]
    ref = torch.einsum("hcn,nhd->chd", torch.softmax(s.masked_fill(ahead[None], -math.inf), -1), vv)
    # the mean of many values: as in Forest.reference
    mag = (torch.einsum("chd,nhd->hcn", q.double().abs(), kk.abs()) / 8).max().item()
    tol = 2 * ((26 * mag) * 2.0**-23 + 16 * 2.0**-22) * vv.abs().max().item()
    assert (out.double() - ref).abs().max().item() <= tol
    assert torch.equal(out, again)  # parts are joined in a fixed order


def test_rotated_queries_equal_the_prompt_attention():
    """rotate_query, and the same rows as prefill_attention on an f32 pool."""
    f = Forest(4, 2, [path((1, 64), (1000 * (i + 1), 9 * i)) for i in range(5)], [1, 4, 2, 1, 7], seed=2)
    q, k, v = f.new_rows()
    a, b_out = torch.empty_like(q), torch.empty_like(q)
    with f.pool.begin(f.caches, f.counts) as b:
        b.append_layer(0, k, v, rotate_keys=True)
        b.shared_prefix_attention(0, q, a)
        b.prefill_attention(0, q, b_out)
    # two f32 computations of means of N(0, 1) values: each within ~1e-5
    assert (a - b_out).abs().max().item() <= 2e-5


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_parts_with_far_apart_scores(dtype):
    """Scores of hundreds: one part of a row outweighs the others entirely."""
    f = Forest(4, 2, [path((1, 80), (1000 * (i + 1), 20 * i)) for i in range(4)], [2, 1, 3, 1], dtype, seed=9,
               scale=12.0)
    f.check()


def test_a_truncated_sequence_copies_the_shared_block_it_writes():
    f = Forest(4, 2, [path((1, 96), (5000, 3)), path((1, 96)), path((1, 96), (6000, 40))], [1, 1, 1], seed=4)
    f.caches[1].truncate_all(77)  # inside the fifth shared block
    f.paths[1] = f.paths[1][:77]
    f.check()


def test_a_bad_query_fails_its_sequence_alone():
    paths = [path((1, 64), (1000 * (i + 1), 20)) for i in range(3)]
    f = Forest(4, 2, paths, [2, 2, 2], seed=6)
    q, k, v = f.new_rows()
    ref, tol = f.reference(0, q, k, v)
    for bad in (float("nan"), float("inf")):
        q2, out = q.clone(), torch.empty_like(q)
        q2[2, 1, 5] = bad
        b = f.pool.begin(f.caches, f.counts)
        b.append_layer(0, k, v, rotate_keys=False)
        b.shared_prefix_attention(0, q2, out, rotate_query=False)
        status = b.end(raise_on_error=False)
        assert status == [0, slmkv.ERR_NON_FINITE, 0]
        good = [0, 1, 4, 5]
        assert (out[good].double() - ref[good]).abs().max().item() <= tol
        f.pool.truncate_many([f.caches[0], f.caches[2]], [84, 84])
    assert [c.sequence_length() for c in f.caches] == [84, 84, 84]


def test_batches_in_flight_and_growing_plans():
    """Several submitted steps, each with a plan of its own, the later ones
    larger; on a stream other than the default one."""
    stream = torch.cuda.Stream()
    paths = [path((1, 128), (1000 * (i + 1), 3 * i)) for i in range(40)]
    f = Forest(4, 2, paths, [1] * 40, seed=8, context=300, blocks=2000)
    torch.cuda.synchronize()
    steps, pending = [], []
    with torch.cuda.stream(stream):
        for n in (2, 5, 40, 11, 40):
            f.counts = [1 + (i + n) % 3 for i in range(n)]
            rows = f.new_rows()
            keep = (f.caches, f.paths)
            b = f.pool.begin(f.caches[:n], f.counts)
            out = f.attend(b, 0, rows)
            pending.append(b.submit())
            steps.append((n, list(f.counts), rows, out, [list(p) for p in f.paths[:n]]))
            row = 0
            for i in range(n):  # what the step appended is the next one's cache
                for j in range(f.counts[i]):
                    token = 10_000_000 + 1000 * len(steps) + row
                    f.paths[i] = f.paths[i] + [token]
                    f.kv[(0, tuple(f.paths[i]))] = (rows[1][row], rows[2][row])
                    row += 1
            f.caches, f.paths = keep[0], f.paths
        for b in pending:
            b.wait()
    stream.synchronize()
    for n, counts, rows, out, paths_then in steps:
        f.counts, f.paths = counts, paths_then
        ref, tol = f.reference(0, *rows)
        assert (out.double() - ref).abs().max().item() <= tol, n


def test_refusals():
    f = Forest(4, 2, [path((1, 20)), path((1, 20))], [1, 1])
    q, k, v = f.new_rows()
    out = torch.empty_like(q)
    b = f.pool.begin(f.caches, 1)
    with pytest.raises(slmkv.InvalidInput, match="must be appended"):
        b.shared_prefix_attention(0, q, out)
    b.append_layer(0, k, v)
    with pytest.raises(slmkv.InvalidInput, match="outside 0..1"):
        b.shared_prefix_attention(1, q, out)
    with pytest.raises(slmkv.InvalidInput, match="overlap"):
        b.shared_prefix_attention(0, q, q)
    for wrong in (out[:1], out.half(), out.cpu(), out.transpose(0, 1), torch.empty((2, 4, 128), device="cuda")[..., ::2]):
        with pytest.raises(slmkv.InvalidInput):
            b.shared_prefix_attention(0, q, wrong)
    flat = torch.empty(q.numel() + 1, device="cuda")[1:].view(q.shape)
    with pytest.raises(slmkv.InvalidInput, match="aligned"):
        b.shared_prefix_attention(0, q, flat)
    with pytest.raises(TypeError):
        b.shared_prefix_attention(0, None, out)
    b.shared_prefix_attention(0, q, out)
    b.end()
    assert slmkv.lib().slm_batch_shared_attention(None, 0, None, 0, None) == slmkv.ERR_INVALID_INPUT


def test_captured_and_replayed():
    """A batch's first call plans and is refused under capture; later ones are
    captured, and a replay reads the buffers' new contents."""
    f = Forest(8, 2, [path((1, 160), (50 * i, 9)) for i in range(2, 30)], [2] * 28, seed=12, dtype="bf16")
    stream = torch.cuda.Stream()
    q, k, v = f.new_rows()
    out, first = torch.empty_like(q), torch.empty_like(q)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        b = f.pool.begin(f.caches, f.counts)
        b.append_layer(0, k, v, rotate_keys=False)
        empty, graph = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(empty, stream=stream):
            torch.ones(1, device="cuda")  # (a graph of something)
            with pytest.raises(slmkv.InvalidInput, match="captured"):
                b.shared_prefix_attention(0, q, out, rotate_query=False)
        b.shared_prefix_attention(0, q, first, rotate_query=False)
        with torch.cuda.graph(graph, stream=stream):
            b.shared_prefix_attention(0, q, out, rotate_query=False)
        graph.replay()
        stream.synchronize()
        ref, tol = f.reference(0, q, k, v)
        assert torch.equal(out, first) and (out.double() - ref).abs().max().item() <= tol
        q.copy_(f.randn(*q.shape))
        graph.replay()
        stream.synchronize()
        ref, tol = f.reference(0, q, k, v)
        assert (out.double() - ref).abs().max().item() <= tol
        b.end()


def test_a_rolled_back_step_and_the_next_on_another_stream():
    """Both use the context's scratch for joined parts."""
    f = Forest(4, 2, [path((1, 640), (9000 * (i + 1), 5)) for i in range(32)], [1] * 32, seed=13)
    rows = f.new_rows()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for turn in range(4):
        with torch.cuda.stream(streams[turn % 2]):
            b = f.pool.begin(f.caches, f.counts)
            outs.append(f.attend(b, 0, rows))
            b.rollback()
    torch.cuda.synchronize()
    ref, tol = f.reference(0, *rows)
    for out in outs:
        assert (out.double() - ref).abs().max().item() <= tol


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hq,hkv", [(8, 1), (8, 2), (4, 2)])
@pytest.mark.parametrize("prefix", [1040, 1504])
def test_runs_on_the_tensor_cores(hq, hkv, prefix, dtype):
    """Enough rows and shared blocks for the 128-row tiles, whose last tile ends
    inside; drafts, so that rows end in a last row tile too."""
    n = 40
    Forest(hq, hkv, [path((1, prefix), (70 * i, 1 + i % 7)) for i in range(2, 2 + n)], [1 + i % 4 for i in range(n)],
           dtype, seed=prefix).check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_magnitudes_on_the_tensor_cores(dtype):
    """Blocks and rows of very different sizes: values from 1e-12 to 1e12 with
    a block of zeros, keys and queries whose product stays of order one."""
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    n, prefix, hq, hkv = 48, 1024, 8, 2
    f = Forest(hq, hkv, [path((1, prefix), (70 * i, 3)) for i in range(2, 2 + n)], [1] * n, dtype, seed=21)
    key, value = f.pool.storage()
    ids = torch.tensor(f.caches[0].blocks()[:prefix // 16], device="cuda", dtype=torch.long)
    for scale_k, size_v in ((1e-20, 1e12), (1e20, 1e-12), (1.0, 1.0)):
        k = torch.randn((prefix // 16, hkv, 16, D), generator=g, device="cuda") * scale_k
        v = torch.randn((prefix // 16, hkv, 16, D), generator=g, device="cuda") * size_v
        v[5:9] *= 1e-3
        v[9] = 0
        key[0, ids], value[0, ids] = k.to(key.dtype), v.to(value.dtype)
        k, v = key[0, ids].transpose(1, 2).reshape(prefix, hkv, D), value[0, ids].transpose(1, 2).reshape(prefix, hkv, D)
        for i in range(prefix):
            f.kv[(0, tuple(f.paths[0][:i + 1]))] = (k[i].float(), v[i].float())
        q, nk, nv = f.new_rows()
        q, nk, nv = q / scale_k, nk * scale_k, nv * size_v
        for p in f.paths:  # the few own cached tokens are zeros
            for j in range(prefix, len(p)):
                f.kv[(0, tuple(p[:j + 1]))] = (torch.zeros((hkv, D), device="cuda"),) * 2
        for i, c in enumerate(f.caches):
            last = c.blocks()[prefix // 16]
            key[0, last], value[0, last] = 0, 0
        with f.pool.begin(f.caches, f.counts) as b:
            out = f.attend(b, 0, (q, nk, nv))
        ref, tol = f.reference(0, q, nk, nv)
        assert (out.double() - ref).abs().max().item() <= tol, (scale_k, size_v)
        f.pool.truncate_many(f.caches, [prefix + 3] * n)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scores_far_from_zero_on_the_tensor_cores(dtype):
    """Scores of 2^30 and beyond, ties among them: one key for all tokens of the
    prefix, zeros for the others, so that every row is the mean of the one's or
    of the others' values."""
    n, prefix, hq, hkv = 48, 1024, 8, 2
    f = Forest(hq, hkv, [path((1, prefix), (70 * i, 3)) for i in range(2, 2 + n)], [1] * n, dtype, seed=22)
    key, _ = f.pool.storage()
    shared = torch.tensor(f.caches[0].blocks()[:prefix // 16], device="cuda", dtype=torch.long)
    for at in (2.0**15, -(2.0**15), 2.0**40, -(2.0**40)):
        key[0] = 0
        key[0, shared] = at
        for x in f.kv:
            f.kv[x] = (torch.full((hkv, D), at if len(x[1]) <= prefix else 0.0, device="cuda"), f.kv[x][1])
        q, nk, nv = f.new_rows()
        q, nk = torch.full_like(q, 2.0**14), torch.zeros_like(nk)
        with f.pool.begin(f.caches, f.counts) as b:
            out = f.attend(b, 0, (q, nk, nv))
        ref, _ = f.reference(0, q, nk, nv)
        # equal scores are equal whatever they are: a mean, of weights of one
        # size. At most 12 sums cut at 2^-23 a tile of 64, values in parts to
        # 2^-22, 16 tiles and their joins each rounded at 2^-24.
        vmax = max(x.abs().max().item() for _, x in f.kv.values())
        assert (out.double() - ref).abs().max().item() <= 32 * 2.0**-22 * max(vmax, nv.abs().max().item()), at
        f.pool.truncate_many(f.caches, [prefix + 3] * n)


def test_a_score_past_f32_fails_its_sequence_on_the_tensor_cores():
    n, prefix, hq, hkv = 48, 1024, 8, 2
    f = Forest(hq, hkv, [path((1, prefix), (70 * i, 3)) for i in range(2, 2 + n)], [1] * n, "f32", seed=23)
    key, _ = f.pool.storage()
    ids = f.caches[0].blocks()[:prefix // 16]
    key[0, ids[20], :, 3, 7] = 1e30
    q, nk, nv = f.new_rows()
    q[:, :, 7] = 0.5
    q[4, 2, 7] = 1e20
    q[9, 5, 1] = math.inf
    b = f.pool.begin(f.caches, f.counts)
    out = f.attend(b, 0, (q, nk, nv))
    status = b.end(raise_on_error=False)
    assert [i for i, s in enumerate(status) if s] == [4, 9]
    assert set(status) == {0, slmkv.ERR_NON_FINITE}
    good = [i for i in range(n) if i not in (4, 9)]
    assert torch.isfinite(out[good]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hq,hkv,lengths,counts", [
    (8, 2, [12_005], [6]),                                             # one long cache, drafts
    (8, 8, [0, 1600, 1601, 1615, 1616, 90], [17, 16, 16, 20, 33, 1]),  # one query head a key head; chunks
    (16, 2, [2500, 2511, 2047, 31], [5, 8, 3, 8])])
def test_long_caches_of_one_sequence(hq, hkv, lengths, counts, dtype):
    """Nothing shared, but many new rows a sequence: its cache is read for all of
    them, the rows' own blocks apart."""
    Forest(hq, hkv, [path((1000 * i, n)) if n else [] for i, n in enumerate(lengths, 1)], counts, dtype, seed=len(lengths)).check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_shared_and_long_runs_with_one_query_head(dtype):
    paths = [path((1, 1600), (9000 * i, 1300 + 7 * i)) for i in range(1, 4)]
    Forest(4, 4, paths, [40, 33, 1], dtype, seed=5).check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_an_outlying_channel_on_the_tensor_cores(dtype):
    """One channel of the keys 2^17 times the others, of the queries 2^-17 times:
    the others keep 2^-40 of the large ones at least, 2^-22 of their own size."""
    n, prefix, hq, hkv = 48, 1024, 8, 2
    f = Forest(hq, hkv, [path((1, prefix), (70 * i, 3)) for i in range(2, 2 + n)], [1] * n, dtype, seed=24)
    key, _ = f.pool.storage()
    key[0, ..., 7] *= 2.0**17  # exact in both types
    for x in f.kv:
        f.kv[x][0][:, 7] *= 2.0**17
    q, nk, nv = f.new_rows()
    q[:, :, 7] *= 2.0**-17
    nk[:, :, 7] *= 2.0**17
    with f.pool.begin(f.caches, f.counts) as b:
        out = f.attend(b, 0, (q, nk, nv))
    ref, tol = f.reference(0, q, nk, nv)
    assert (out.double() - ref).abs().max().item() <= tol
