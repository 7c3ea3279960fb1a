"""Log probabilities of given tokens: rows of many batches with few alternatives, and numbers at the edges, against plain 64-bit
arithmetic."""
from __future__ import annotations

import pytest
import torch

from cpi_b200.csrc import lib as K

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("top", [2, 3, 5, 8])
@pytest.mark.parametrize("rows,vocab", [(700, 40001), (64, 202048), (3, 300003)])
def test_the_best_of_rows_of_many_batches(rows, vocab, top, dtype):
    """Every batch that raises the bound does so while other warps raise the maxima: no number above it may be lost.  Alternatives are
    the row's own numbers, so they are equal, not near."""
    g = torch.Generator(device=DEV).manual_seed(vocab + top)
    x = (torch.randn(rows, vocab, generator=g, device=DEV) * 4).to(dtype)
    ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top].int()
    targets = ids.long()[:, -1:].contiguous()
    for _ in range(20):
        got = K.log_probs(x, targets, top=top)
        assert torch.equal(got.top_ids, ids)
        assert torch.equal(got.top_logprobs[:, -1], got.logprob[:, 0])
