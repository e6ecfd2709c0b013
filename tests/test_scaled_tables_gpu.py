"""Block tables whose entries name no page, over a cache of 8 bits."""

import pytest
import torch

from test_scaled_attention_gpu import Batch, close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("page", [64, 16])
def test_entries_that_name_no_page_count_as_the_last_one(dtype, page):
    """Entries outside the pages lead to the last of them, whatever they hold, in rows and in portions alike; requests with good tables are as ever."""
    batch = Batch(dtype, 2, 1, 64, page, [200, 10, 77], [1, 40, 30], seed=15)
    last = batch.planes[0].codes.shape[0] - 1
    good = batch.tables.clone()
    results = []
    for entries in ((last, last, last), (-7, 2**30, last + 1), (-(2**31), 2**31 - 1, -1)):
        batch.tables = good.clone()
        batch.tables[0, 1], batch.tables[1, 0], batch.tables[0, 2] = entries
        for options in (dict(short_rows=1, short_requests=1), dict(max_q_len=None), {}):
            results.append(batch.run(**options))
    for a, b in zip(results, results[3:]):
        assert torch.equal(a, b)
    batch.tables = good
    for got in results:
        close(got[41:], batch.want()[41:], batch)
