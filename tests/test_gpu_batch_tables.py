"""A batch's page table, tiers and lengths in the package's own integer arrays."""

import numpy as np
import pytest

from conftest import announce
from test_gpu_batch import Batch, MIXED
from test_gpu_kv_pages import mi, put

pytestmark = pytest.mark.gpu


def test_tables_as_device_indexes_of_their_words():
    d = mi().device
    rng = np.random.default_rng(0)
    batch = Batch(rng, [300, 33, 0, 97], 14, 2, 64, MIXED)
    pages = d.DeviceIndex(batch.table.view(np.int32))
    tiers = np.full(-(-batch.tiers.size // 4) * 4, 255, np.uint8)
    tiers[:batch.tiers.size] = batch.tiers.reshape(-1)
    out = d.empty(batch.q.size)
    announce("tables as indexes")
    d.attention_batch(put(batch.q), pages, d.DeviceIndex(tiers.view(np.int32)), batch.length_index,
                      out, 4, batch.max_pages, 14, 2, 64)
    batch.check(out.to_numpy().reshape(4, 14, 64), what="tables")
