"""Split keys on an engine with per-class record caps (vn_config.max_batch_class_records): the caps
hold the engine's own ingest batches, not the split records gathered to a key's owner, whose count
only vn_config.split_max_records bounds.  So a cap below the gathered records, or above the split
engine's own batch size, changes nothing: every digest and sketch is the single consumer's, bit for
bit (server.go:655 routes every record of a key to one worker)."""
import numpy as np
import pytest

import oracle
import veneur_amd as V
from tests.util import PCT

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("records,caps", [
    (1 << 20, (64, 64, 64, 64)),       # far fewer than the split records below
    (3 << 20, (0, 0, 3 << 20, 0)),     # more than the split engine's 2^21
    (3 << 20, (16, 0, 1 << 16, 3 << 20)),
])
def test_split_keys_with_class_record_caps(records, caps):
    rng = np.random.default_rng(21)
    n = 120_001
    keys = rng.integers(0, 2, n).astype(np.uint32)
    vals = np.exp(rng.normal(3.0, 1.0, n))
    rates = np.where(rng.random(n) < 0.1, np.float32(0.1), np.float32(1.0)).astype(np.float32)
    skeys = np.zeros(n, np.uint32)
    shash = rng.integers(0, 2**64 - 1, n, dtype=np.uint64)
    with V.Engine((4, 4, 4, 4), percentiles=PCT, max_batch_records=records, max_class_records=caps,
                  split_max_records=1 << 18) as e:
        e.split_keys(0, np.array([1], np.uint32), np.array([0], np.uint32))
        e.split_keys(2, np.array([1, 3], np.uint32), np.zeros(2, np.uint32))
        e.split_keys(3, np.array([2], np.uint32), np.array([0], np.uint32))
        e.ingest(counters=(np.array([1, 1], np.uint32), np.array([2.0, 3.0]), np.ones(2, np.float32)))
        for part in np.array_split(np.arange(n), 2):
            e.ingest_split(histos=(keys[part], vals[part], rates[part]), set_hashes=(skeys[part], shash[part]))
        f = e.flush()
    w = oracle.Worker(1, 1, 2, 1)
    w.histo(keys, vals, rates)
    w.set_hashed(skeys, shash)
    assert f.counter_value.tolist() == [5]
    assert f.histo_slot.tolist() == [1, 3] and f.set_slot.tolist() == [2]
    for k in range(2):
        np.testing.assert_array_equal(f.histo_quantiles[k], [w.histo_quantile(k, p) for p in PCT])
    assert f.set_estimate.tolist() == [w.set_estimate(0)]
