"""A submitted step fails while a later one of the same sequence is open: the
open one is rolled back with it when it ends, the other sequences go on."""

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
slmkv = pytest.importorskip("slmkv")

D = 64


@pytest.mark.parametrize("later", [1, 2])
def test_an_open_step_is_rolled_back_with_the_failed_one_before_it(later):
    g = torch.Generator(device="cuda")
    g.manual_seed(1)

    def rows(t):
        return tuple(torch.randn((t, h, D), generator=g, device="cuda") for h in (4, 2, 2))

    pool = slmkv.KvPool(num_layers=1, num_query_heads=4, num_key_value_heads=2, context_length=64, num_blocks=32,
                        max_sequences=3)
    caches = [pool.allocate_kv_cache(64) for _ in range(3)]
    with pool.begin(caches, [15, 16, 17]) as b:
        b.append_layer(0, *rows(48)[1:])
    q, k, v = rows(3)
    v[1, 0, 3] = math.nan
    out = torch.empty_like(q)
    first = pool.begin(caches, 1)
    first.decode_layer(0, q, k, v, out)
    first.submit()
    held = caches[1:] if later == 1 else caches
    b = pool.begin(held, 2)  # planned on the first step's lengths
    with pytest.raises(slmkv.InvalidInput):
        first.wait()
    assert first.statuses == [0, slmkv.ERR_NON_FINITE, 0]
    q, k, v = rows(2 * len(held))
    b.append_layer(0, k, v)
    b.shared_prefix_attention(0, q, torch.empty_like(q))
    status = b.end(raise_on_error=False)
    assert status == ([slmkv.ERR_NON_FINITE, 0] if later == 1 else [0, slmkv.ERR_NON_FINITE, 0])
    assert [c.sequence_length() for c in caches] == [16 if later == 1 else 18, 16, 20]
    # the sequence goes on from the length before the failed step
    with pool.begin(caches, 1) as b:
        q, k, v = rows(3)
        b.append_layer(0, k, v)
    assert caches[1].sequence_length() == 17


@pytest.mark.parametrize("end", [True, False])
def test_the_open_steps_blocks_stay_its_own(end):
    """Another sequence that grows meanwhile must not get a block that the open
    step writes to."""
    g = torch.Generator(device="cuda")
    g.manual_seed(2)

    def rows(t, *heads):
        return tuple(torch.randn((t, h, D), generator=g, device="cuda") for h in heads)

    pool = slmkv.KvPool(num_layers=1, num_query_heads=4, num_key_value_heads=2, context_length=64, num_blocks=16,
                        max_sequences=3)
    bad, good, other = (pool.allocate_kv_cache(64) for _ in range(3))
    with pool.begin([bad, good], [40, 7]) as b:
        b.append_layer(0, *rows(47, 2, 2))
    free = pool.stats()[0]
    q, k, v = rows(18, 4, 2, 2)
    v[3, 1, 9] = math.inf
    first = pool.begin([bad, good], [17, 1])  # two more blocks of the failing sequence
    first.append_layer(0, k, v)
    first.submit()
    second = pool.begin([bad, good], [6, 2])
    with pytest.raises(slmkv.InvalidInput):
        first.wait()
    assert first.statuses == [slmkv.ERR_NON_FINITE, 0]
    k, v = rows(20, 2, 2)
    other.append_layer(0, k, v, 20, rotate_keys=False)
    assert not set(other.blocks()) & set(bad.blocks())
    q, nk, nv = rows(8, 4, 2, 2)
    out = torch.empty_like(q)
    second.append_layer(0, nk, nv)
    second.shared_prefix_attention(0, q, out)
    if end:
        assert second.end(raise_on_error=False) == [slmkv.ERR_NON_FINITE, 0]
    else:
        second.rollback()
    assert [c.sequence_length() for c in (bad, good, other)] == [40, 10 if end else 8, 20]
    assert torch.equal(other.layer_keys(0).view(20, 2, D), k) and torch.equal(other.layer_values(0).view(20, 2, D), v)
    assert torch.isfinite(out[6:]).all()
    assert pool.stats()[0] == free - 2  # what the failed steps held is free again
    with pool.begin([bad, other], 3) as b:
        b.append_layer(0, *rows(6, 2, 2))
    assert [c.sequence_length() for c in (bad, other)] == [43, 23]
