"""Batches whose split over the GPU has every form: more sequences than a kernel has
threads, sequences of many query tiles, items that begin, end and are cut inside
the shares.  Oracle and tolerances are those of test_block_cache_gpu.py."""
import pytest
import torch

from test_block_cache_gpu import _attend, _case, _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("most", [1, 70])
def test_more_sequences_than_threads(cuda, most):
    g = torch.Generator().manual_seed(most)
    lens = torch.randint(0, 90, (1300,), generator=g).tolist()
    new = [min(n, int(k)) for n, k in zip(lens, torch.randint(0, most + 1, (1300,), generator=g))]
    c = _case(most, lens, new, hq=4, hkv=1)
    _check(_attend(c, cuda), c)


@pytest.mark.parametrize("lens,new,hq,hkv", [
    ([3000], [3000], 4, 1), ([2200, 40, 1100], [2200, 40, 900], 8, 2), ([700] * 9, [700] * 9, 2, 2),
    ([9000], [100], 4, 1)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 5)])
def test_prompts_of_many_query_tiles(cuda, lens, new, hq, hkv, window, sinks):
    c = _case(sum(new) + hq, lens, new, hq=hq, hkv=hkv, bs=32)
    _check(_attend(c, cuda, window, sinks), c, window, sinks)


@pytest.mark.parametrize("new", [1, 4, 9])
@pytest.mark.parametrize("hkv", [1, 4])
def test_decoding_items_end_inside_shares(cuda, new, hkv):
    lens = [1200 + 37 * i % 900 for i in range(40)] + [5, 0, 6000]
    c = _case(new + hkv, lens, [min(new, n) for n in lens], hq=4 * hkv, hkv=hkv, bs=64)
    _check(_attend(c, cuda), c)


@pytest.mark.parametrize("total,new", [(500, 1), (500, 16), (40, 17), (1, 1), (0, 0), (700, 300)])
def test_one_sequence_below_its_bound(cuda, total, new):
    """max_qlen says that a sequence may have many queries; it has few."""
    c = _case(total + new, [total], [new], hq=8, hkv=2)
    if new:
        _check(_attend(c, cuda, max_qlen=300), c)
    else:
        assert _attend(c, cuda, max_qlen=300).shape[0] == 0


def test_batches_without_tokens(cuda):
    """Sequences that bring nothing to a call: nothing changes, nothing is taken."""
    import block_cache
    import speculative
    c = _case(3, [20, 0], [0, 0], hq=4, hkv=2)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    kc, vc = (c[k].view(torch.uint8).to(cuda).view(torch.float8_e4m3fn) for k in "kv")
    ks, vs = c["ks"].to(cuda), c["vs"].to(cuda)
    before = [t.view(torch.uint8).clone() for t in (kc, vc, ks, vs)]
    q = block_cache.append(torch.empty(0, 8 * 128, dtype=torch.bfloat16, device=cuda), torch.zeros(64, 128, device=cuda),
                           kc, vc, ks, vs, i32([0, 0, 0]), i32([20, 0]), i32(c["table"]))
    assert q.shape == (0, 4, 128)
    assert all(torch.equal(a, t.view(torch.uint8)) for a, t in zip(before, (kc, vc, ks, vs)))
    out, accepted = speculative.verify(torch.empty(0, 100, device=cuda), torch.empty(0, dtype=torch.int64, device=cuda),
                                       i32([0, 0, 0]), torch.empty(0, device=cuda), torch.ones(2, 100, device=cuda),
                                       num_accepted=torch.full((2,), 7, dtype=torch.int32, device=cuda))
    assert out.shape == (0,) and accepted.tolist() == [0, 0]
