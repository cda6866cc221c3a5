"""Attention over shared prefixes and selected pages where a call is allowed and rare:
pages without a token left (tolerances: segment_helpers).

A prefix of up to 32 query rows per KV head takes the form without tiles, of up to 64 the
one with tiles of two waves' rows, of more the one of four."""

from __future__ import annotations

import pytest
import torch

from segment_helpers import Batch
from test_gpu_prefix import planned, run, spread

pytestmark = pytest.mark.gpu

# of 4 heads per KV head: 8 and 24 rows, 36, 80 and 160
FORMS = [2, 6, 9, 20, 40]


@pytest.mark.parametrize("requests", FORMS)
@pytest.mark.parametrize("left", [float("nan"), float("inf"), 65504.0])
def test_a_page_without_tokens_weighs_nothing(cuda, requests, left):
    """Whatever its scales are: lengths may move to 0, and such a page was never written."""
    print(f"no tokens {requests} {left}", flush=True)
    b = Batch(cuda, [(0, requests, 1000)], spread(requests, 17, 70), [0] * requests, 1, 4, scale=2.0 ** -13)
    decode = planned(b, cuda)
    b.prefix_last.zero_()
    b.last.zero_()
    out, lse = run(decode, b)
    b.check(out, lse)
    pages = torch.cat((b.prefix_ids[-1:], b.ids[(b.own_ptr[1:] - 1).long().to(cuda)])).long()
    for scale in b.scales:
        scale[pages] = left
    got, got_lse = run(decode, b)
    assert torch.equal(got, out) and torch.equal(got_lse, lse)
