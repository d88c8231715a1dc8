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
