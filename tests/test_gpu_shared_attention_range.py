"""The range of attention over shared prefixes where its many-row runs go to
the tensor cores (every call here is checked to take them): values and scores
of very different sizes within a tile, up to the ends of f32, against softmax
attention in 64 bits on what the pages hold, with a bound for every output."""

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
slmkv = pytest.importorskip("slmkv")

D, PAGE = 64, 16
HQ, HKV, N, PREFIX, TAIL = 8, 2, 72, 1024, 3


class Shared:
    """N sequences over one PREFIX-token run, TAIL cached tokens of their own
    (zeros unless written), ready for one new token each."""

    def __init__(self, dtype, seed, n=N, prefix=PREFIX):
        self.n, self.prefix = n, prefix
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)
        context = prefix + TAIL + 8
        self.pool = slmkv.KvPool(num_layers=1, num_query_heads=HQ, num_key_value_heads=HKV, context_length=context,
                                 num_blocks=prefix // PAGE + 2 * n, max_sequences=n,
                                 kv_dtype=slmkv.KV_BF16 if dtype == "bf16" else slmkv.KV_F32)
        self.pool.shuffle(seed)
        self.caches = [self.pool.allocate_kv_cache(context) for _ in range(n)]
        zeros = torch.zeros((prefix, HKV, D), device="cuda")
        self.caches[0].append_layer(0, zeros, zeros, prefix)
        self.caches[0].publish_prefix([1] * prefix)
        for c in self.caches[1:]:
            assert c.attach_prefix([1] * prefix) == prefix
        tail = torch.zeros((n * TAIL, HKV, D), device="cuda")
        with self.pool.begin(self.caches, TAIL) as b:
            b.append_layer(0, tail, tail, rotate_keys=False)
        self.key, self.value = (x[0] for x in self.pool.storage())
        self.ids = self.blocks(0)[:prefix // PAGE]

    def randn(self, *size):
        return torch.randn(size, generator=self.g, device="cuda")

    def blocks(self, i):
        return torch.tensor(self.caches[i].blocks(), device="cuda", dtype=torch.long)

    def write(self, k, v):
        """Keys and values of the shared run, [blocks, HKV, 16, D]."""
        self.key[self.ids], self.value[self.ids] = k.to(self.key.dtype), v.to(self.value.dtype)

    def shared_like(self):
        return self.randn(self.prefix // PAGE, HKV, PAGE, D), self.randn(self.prefix // PAGE, HKV, PAGE, D)

    def attend(self, q, k, v):
        """(outputs, status, pages' blocks of each sequence); back to the old lengths."""
        out = torch.empty_like(q)
        b = self.pool.begin(self.caches, 1)
        b.append_layer(0, k, v, rotate_keys=False)
        before = self.pool.launch_count()
        b.shared_prefix_attention(0, q, out, rotate_query=False)
        assert self.pool.launch_count() - before == 3  # tiles, the other runs, their joining
        blocks = [self.blocks(i) for i in range(self.n)]
        status = b.end(raise_on_error=False)
        for c, s in zip(self.caches, status):
            if s == 0:
                c.truncate_all(self.prefix + TAIL)
        return out, status, blocks

    def reference(self, q, blocks):
        """(out, bound for each output) in 64 bits. A score's error is that of
        at most 26 chained groups of products, each cut at 2^-23 of the sum of
        magnitudes; a weight is off by that in the exponent and by a few units of
        2^-22 for powers, parts and rescales. Weights and values in parts keep
        2^-40 of the largest product of a weight and a value of a tile's blocks
        (each rounded up to a power of two, two parts, 64 tokens: 2^-38 x 64)."""
        length = self.prefix + TAIL + 1
        out, bound = (torch.empty((self.n, HQ, D), dtype=torch.float64, device="cuda") for _ in range(2))
        for i, ids in enumerate(blocks):
            k, v = (x[ids].transpose(1, 2).reshape(-1, HKV, D)[:length].double().repeat_interleave(HQ // HKV, 1)
                    for x in (self.key, self.value))
            s = torch.einsum("hd,nhd->hn", q[i].double(), k) / 8
            mag = torch.einsum("hd,nhd->hn", q[i].double().abs(), k.abs()) / 8
            w = torch.softmax(s, -1)
            out[i] = torch.einsum("hn,nhd->hd", w, v)
            off = w * (26 * mag * 2.0**-23 + 16 * 2.0**-22)
            bound[i] = torch.einsum("hn,nhd->hd", off, v.abs()) + off.sum(-1, keepdim=True) * out[i].abs()
            pad = -length % PAGE
            wb = torch.nn.functional.pad(w, (0, pad)).view(HQ, -1, PAGE).amax(-1)
            vb = torch.nn.functional.pad(v.abs().amax(-1).t(), (0, pad)).view(HQ, -1, PAGE).amax(-1)
            bound[i] += 64 * 2.0**-38 * (wb * vb).sum(-1, keepdim=True) + 2.0**-140
        return out, bound

    def check(self, q, k, v):
        out, status, blocks = self.attend(q, k, v)
        assert status == [0] * self.n
        ref, bound = self.reference(q, blocks)
        over = ((out.double() - ref).abs() / bound).max().item()
        assert over <= 1, over


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("spread", [20, 30, 38, 45, 70])
def test_large_values_that_no_row_attends_to(spread, dtype):
    """Blocks of values 2^spread times their neighbours', under scores hundreds
    below: their size must not reach the outputs, wherever in a tile they lie."""
    f = Shared(dtype, spread)
    k, v = f.shared_like()
    k[..., 0] = 0
    large = [0, 5, 10, 15, 20, 21, 24, 25, 26, 27, 33, 34, 35, 63]
    k[large, ..., 0] = -512.0
    v[large] *= 2.0**spread
    f.write(0.5 * k, v)
    q, nk, nv = f.randn(N, HQ, D), f.randn(N, HKV, D), f.randn(N, HKV, D)
    q[..., 0], nk[..., 0] = 16.0, 0.0
    f.check(q, nk, nv)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("spread", [24, 44, 60])
def test_sizes_and_weights_that_balance(spread, dtype):
    """Blocks of small values under large weights beside large ones under small
    weights, so that both give as much to the outputs; and rows that see one or
    the other alone."""
    f = Shared(dtype, 100 + spread)
    k, v = f.shared_like()
    k[..., 0] = 0
    large = list(range(2, 64, 3))
    k[large, ..., 0] = -1.0
    v[large] *= 2.0**spread
    f.write(0.5 * k, v)
    q, nk, nv = f.randn(N, HQ, D), f.randn(N, HKV, D), f.randn(N, HKV, D)
    # q0 k0 / 8 = -spread ln 2, times 0.8 .. 1.2 by the row, and some rows far off
    q[..., 0] = 16 * spread * math.log(2) * (0.8 + 0.4 * torch.arange(N, device="cuda")[:, None] / N)
    q[::9, ..., 0] = 5000.0
    q[4::9, ..., 0] = -5000.0
    nk[..., 0] = 0
    f.check(q, nk, nv)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size", [1e30, 1e34, 1e35, 1e-30, 1e-36])
def test_values_near_the_ends_of_f32(size, dtype):
    """Sums of weights times values stay in f32's range: 1024 of 1e35 do."""
    f = Shared(dtype, 7)
    k, v = f.shared_like()
    f.write(0.5 * k, (1 + 0.1 * v) * size)
    q, nk, nv = f.randn(N, HQ, D), f.randn(N, HKV, D), (1 + 0.1 * f.randn(N, HKV, D)) * size
    f.check(0.25 * q, nk, nv)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("scale_k,size_v", [(1e-20, 1e12), (1e20, 1e-12), (1.0, 1.0), (1e-30, 1e-20)])
def test_magnitudes(scale_k, size_v, dtype):
    """Keys and queries of any size whose product stays of order one; a block of
    zeros and blocks of smaller values."""
    f = Shared(dtype, 8)
    k, v = f.shared_like()
    v[5:9] *= 1e-3
    v[9] = 0
    k[12] = 0
    f.write(k * scale_k, v * size_v)
    q, nk, nv = f.randn(N, HQ, D), f.randn(N, HKV, D), f.randn(N, HKV, D)
    f.check(q / scale_k, nk * scale_k, nv * size_v)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("at", [2.0**15, -(2.0**15), 2.0**40, -(2.0**40)])
def test_scores_far_from_zero(at, dtype):
    """Scores of 2^30 and beyond, all tokens of the run alike and zeros after
    it: rows are the mean of the one's or of the others' values."""
    f = Shared(dtype, 9)
    k, v = f.shared_like()
    f.write(torch.full_like(k, at), v)
    q = torch.full((N, HQ, D), 2.0**14, device="cuda")
    nk, nv = torch.zeros((N, HKV, D), device="cuda"), f.randn(N, HKV, D)
    out, status, blocks = f.attend(q, nk, nv)
    assert status == [0] * N
    ref, _ = f.reference(q, blocks)
    # equal scores are equal whatever they are: a mean, of weights of one size.
    # At most 12 sums cut at 2^-23 a tile of 64, values in parts to 2^-22, 16
    # tiles and their joins each rounded at 2^-24.
    top = max(f.value[f.ids].float().abs().max().item(), nv.abs().max().item())
    assert (out.double() - ref).abs().max().item() <= 32 * 2.0**-22 * top


def test_a_score_past_f32_fails_its_sequence():
    f = Shared("f32", 10)
    k, v = f.shared_like()
    k[20, :, 3, 7] = 1e30
    f.write(k, v)
    q, nk, nv = f.randn(N, HQ, D), f.randn(N, HKV, D), f.randn(N, HKV, D)
    q[:, :, 7] = 0.5
    q[4, 2, 7] = 1e20
    q[9, 5, 1] = math.inf
    q[30, 0, 63] = math.nan
    out, status, _ = f.attend(q, nk, nv)
    assert [i for i, s in enumerate(status) if s] == [4, 9, 30]
    assert set(status) == {0, slmkv.ERR_NON_FINITE}
    good = [i for i in range(N) if i not in (4, 9, 30)]
    assert torch.isfinite(out[good]).all()


def test_a_bad_query_fails_its_sequence_bf16():
    f = Shared("bf16", 11)
    f.write(*f.shared_like())
    q, nk, nv = f.randn(N, HQ, D), f.randn(N, HKV, D), f.randn(N, HKV, D)
    q[9, 5, 1] = math.inf
    q[30, 0, 63] = math.nan
    q[71, 7, 0] = -math.inf
    out, status, blocks = f.attend(q, nk, nv)
    bad = [9, 30, 71]
    assert [i for i, s in enumerate(status) if s] == bad
    good = [i for i in range(N) if i not in bad]
    ref, bound = f.reference(q.nan_to_num(0, 0, 0), blocks)
    assert ((out.double() - ref).abs() <= bound)[good].all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_an_outlying_channel(dtype):
    """One channel of the keys 2^17 times the others, of the queries 2^-17 times:
    the others keep 2^-40 of the large ones at least, 2^-22 of their own size."""
    f = Shared(dtype, 12)
    k, v = f.shared_like()
    k[..., 7] *= 2.0**17
    f.write(k, v)
    q, nk, nv = f.randn(N, HQ, D), f.randn(N, HKV, D), f.randn(N, HKV, D)
    q[:, :, 7] *= 2.0**-17
    nk[:, :, 7] *= 2.0**17
    f.check(q, nk, nv)
