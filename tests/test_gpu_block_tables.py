"""Block tables and copied blocks when several changes of one entry, or copies
that follow one another, are sent to the device together."""

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
slmkv = pytest.importorskip("slmkv")

D = 64


def rows(g, t, *heads):
    return tuple(torch.randn((t, h, D), generator=g, device="cuda") for h in heads)


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


@pytest.mark.parametrize("seed", range(4))
def test_attached_then_truncated_sequences_write_to_their_copies(seed):
    """An attached block's entry and that of the copy which a truncated sequence
    writes to, sent at once: the copy's holds."""
    g, n = gen(seed), 60
    pool = slmkv.KvPool(num_layers=1, num_query_heads=4, num_key_value_heads=2, context_length=300,
                        num_blocks=300, max_sequences=n + 1)
    pool.shuffle(seed)
    first = pool.allocate_kv_cache(300)
    k, v = rows(g, 256, 2, 2)
    first.append_layer(0, k, v, 256)
    first.publish_prefix(list(range(256)))
    caches = [pool.allocate_kv_cache(300) for _ in range(n)]
    for i, c in enumerate(caches):
        assert c.attach_prefix(list(range(256))) == 256
        c.truncate_all(20 + 3 * i)
    q, nk, nv = rows(g, 2 * n, 4, 2, 2)
    out, want = torch.empty_like(q), torch.empty_like(q)
    with pool.begin(caches, 2) as b:
        b.append_layer(0, nk, nv, rotate_keys=False)
        b.shared_prefix_attention(0, q, out, rotate_query=False)
    for i, c in enumerate(caches):
        m = 20 + 3 * i
        assert torch.equal(c.layer_keys(0), torch.cat((k[:m], nk[2 * i:2 * i + 2])))
        assert torch.equal(c.layer_values(0), torch.cat((v[:m], nv[2 * i:2 * i + 2])))
    assert torch.equal(first.layer_keys(0), k)


def test_blocks_given_back_and_replaced_between_decode_steps():
    """Decode steps leave table entries for later: a block that was given back by
    a truncation, its successor, and a slot's next owner are pending together."""
    g, n = gen(9), 40
    pool = slmkv.KvPool(num_layers=1, num_query_heads=4, num_key_value_heads=2, context_length=64, num_blocks=4 * n,
                        max_sequences=n)
    pool.shuffle(2)
    caches = [pool.allocate_kv_cache(64) for _ in range(n)]
    q, k, v = rows(g, 16 * n, 4, 2, 2)
    with pool.begin(caches, 16) as b:
        b.append_layer(0, k, v, rotate_keys=False)
    out = torch.empty((n, 4, D), device="cuda")
    for turn in range(3):  # a new block each time, in another order
        order = caches[turn:] + caches[:turn]
        q, nk, nv = rows(g, n, 4, 2, 2)
        with pool.begin(order, 1) as b:
            b.decode_layer(0, q, nk, nv, out)
        if turn < 2:
            pool.truncate_many(caches, [16] * n)
    for i, c in enumerate(caches):
        at = (i - 2) % n
        got = c.layer_values(0)
        assert torch.equal(got[:16], v[16 * i:16 * i + 16]) and torch.equal(got[16], nv[at]), i


def test_a_copys_source_that_becomes_another_copys_target():
    """A full pool: the block that one sequence copies, and gives up, is evicted
    from the index and taken for the other sequence's copy in the same step."""
    g = gen(5)
    pool = slmkv.KvPool(num_layers=2, num_query_heads=4, num_key_value_heads=2, context_length=64, num_blocks=5,
                        max_sequences=2)
    tokens = [list(range(32)), list(range(100, 132))]
    kv = [[rows(g, 32, 2, 2) for _ in range(2)] for _ in tokens]
    for t, layers in zip(tokens, kv):
        c = pool.allocate_kv_cache(64)
        for layer, (k, v) in enumerate(layers):
            c.append_layer(layer, k, v, 32)
        c.publish_prefix(t)
        c.free()
    caches = [pool.allocate_kv_cache(64) for _ in tokens]
    for c, t in zip(caches, tokens):
        assert c.attach_prefix(t) == 32
        c.truncate_all(24)  # writes go into the second block, which is copied first
    source = caches[0].blocks()[1]
    assert pool.stats()[0] == 1
    nk, nv = rows(g, 2, 2, 2)
    with pool.begin(caches, 1) as b:
        for layer in range(2):
            b.append_layer(layer, nk, nv, rotate_keys=False)
    assert caches[1].blocks()[1] == source  # the case that is meant
    for i, c in enumerate(caches):
        for layer in range(2):
            assert torch.equal(c.layer_keys(layer), torch.cat((kv[i][layer][0][:24], nk[i:i + 1])))
            assert torch.equal(c.layer_values(layer), torch.cat((kv[i][layer][1][:24], nv[i:i + 1])))


def test_a_refused_step_gives_back_blocks_that_changed_hands_in_it():
    """The pool runs out in the middle of a step's reservations: a sequence's
    shared block, which it was to copy, was evicted and taken by another one. It
    stays the first one's."""
    g = gen(6)
    pool = slmkv.KvPool(num_layers=1, num_query_heads=4, num_key_value_heads=2, context_length=64, num_blocks=2,
                        max_sequences=3)
    a, b, c = (pool.allocate_kv_cache(64) for _ in range(3))
    k, v = rows(g, 16, 2, 2)
    a.append_layer(0, k, v, 16)
    a.publish_prefix(list(range(16)))
    a.truncate_all(5)
    held = a.blocks()
    for step, counts in (([a, b, c], 1), ([a, b], [20, 1]), ([a], 30), ([a, b, c], 1)):
        with pytest.raises(slmkv.InvalidInput, match="no free block"):
            pool.begin(step, counts)
        assert a.blocks() == held and b.blocks() == c.blocks() == [] and pool.stats()[0] == 1
    nk, nv = rows(g, 2, 2, 2)
    with pool.begin([b, a], 1) as step:
        step.append_layer(0, nk, nv, rotate_keys=False)
    assert not set(a.blocks()) & set(b.blocks()) and pool.stats()[0] == 0
    assert torch.equal(a.layer_keys(0), torch.cat((k[:5], nk[1:]))) and torch.equal(b.layer_keys(0), nk[:1])
