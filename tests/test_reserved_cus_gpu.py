"""vn_config.replay_reserved_cus: the longest batched replays on CUs of their own, every other stream
of the engine on the rest (whole groups of 8, at most a quarter of the GPU).  Placement changes no
result: a long key's digest, a short key's, and a split counter, set and key beside them equal one
consumer's bit for bit (merging_digest.go:97-243), in two windows on the same streams."""
import numpy as np
import pytest

import oracle
import veneur_amd as V
from tests.util import PCT

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cus", [1, 16, 100_000])
def test_reserved_cus_change_no_result(cus):
    rng = np.random.default_rng(5)
    n = [600_001, 70_000, 500]  # batched, four-wave and one-wave replays
    slot = np.repeat(np.arange(3, dtype=np.uint32), n)
    slot = slot[rng.permutation(len(slot))]
    with V.Engine((2, 2, 4, 2), percentiles=PCT, max_batch_records=1 << 20, split_max_records=1 << 16,
                  replay_reserved_cus=cus) as e:
        for _ in range(2):
            vals = np.exp(rng.normal(3.0, 1.0, len(slot)))
            ones = np.ones(len(slot), np.float32)
            e.split_keys(0, np.array([1], np.uint32), np.array([0], np.uint32))
            e.split_keys(2, np.array([3], np.uint32), np.array([0], np.uint32))
            e.ingest_split(histos=(np.zeros(9000, np.uint32), vals[:9000], ones[:9000]))
            e.ingest(counters=(np.array([0, 1, 1], np.uint32), np.array([7.0, 2.0, 3.0]), ones[:3]),
                     histos=(slot, vals, ones),
                     set_hashes=(np.zeros(9000, np.uint32), vals[:9000].view(np.uint64)))
            f = e.flush()
            w = oracle.Worker(1, 1, 4, 1)
            w.histo(slot, vals, ones)
            w.histo(np.full(9000, 3, np.uint32), vals[:9000], ones[:9000])
            w.set_hashed(np.zeros(9000, np.uint32), vals[:9000].view(np.uint64))
            assert f.counter_slot.tolist() == [0, 1] and f.counter_value.tolist() == [7, 5]
            assert f.histo_slot.tolist() == [0, 1, 2, 3]
            for k in range(4):
                np.testing.assert_array_equal(f.histo_quantiles[k], [w.histo_quantile(k, p) for p in PCT])
            assert f.set_slot.tolist() == [0] and f.set_estimate.tolist() == [w.set_estimate(0)]
