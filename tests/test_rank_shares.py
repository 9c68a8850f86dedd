# SPDX-License-Identifier: Apache-2.0
"""More ranks than samples or batches: every rank draws the same number of batches, or a training run waits for ever."""
import pytest

from nvalchemi_toolkit_b200.data.datapipes import (DataLoader, FixedCompositionBatchSampler, InMemoryDataset, MultiDataset,
                                                   MultiDatasetSampler)
from tests.helpers import random_molecule


def _data(n):
    return InMemoryDataset([random_molecule(2, i) for i in range(n)])


@pytest.mark.parametrize("n,world", [(1, 2), (1, 3), (1, 8), (2, 5), (3, 7), (5, 4)])
def test_every_rank_has_its_share(n, world):
    shares = []
    for r in range(world):
        loader = DataLoader(_data(n), batch_size=1)
        loader.set_distributed(r, world)
        assert len(list(loader)) == len(loader)
        shares.append([i for b in loader._batches() for i in b])
    per = -(-n // world)
    assert [len(s) for s in shares] == [per] * world
    assert [shares[i % world][i // world] for i in range(per * world)] == [i % n for i in range(per * world)]
    multi = MultiDataset([_data(n), _data(n)])
    for make in (lambda r: MultiDatasetSampler(multi, num_samples=n, rank=r, world_size=world),
                 lambda r: FixedCompositionBatchSampler(multi, 2, num_batches=n, rank=r, world_size=world)):
        ranks = [make(r) for r in range(world)]
        assert [len(list(s)) for s in ranks] == [len(s) for s in ranks] == [per] * world
