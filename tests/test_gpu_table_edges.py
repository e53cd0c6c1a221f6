"""The operators over a table of embeddings where their contracts are easiest to break."""
import math

import pytest
import torch

from cuhnsw_b200 import table
from test_gpu_table import DEV, TYPES, gen, normal, plain_select

pytestmark = pytest.mark.gpu


# -- beams -----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype, v", [("f16", 50_257), ("bf16", 32_001), ("f32", 50_257), ("f32", 4099), ("f16", 1003), ("bf16", 7),
                                      ("f32", 8191), ("f16", 65_535)])
def test_equal_beams_are_ties_wherever_their_rows_begin(dtype, v):
  """The same scores give the same log of their sum, so the smaller beam comes first: with rows at every place of a 16-byte word."""
  s, b, keep = 2, 4, 13
  row = normal(v, v, dtype=TYPES[dtype], sigma=3.0)
  row[torch.rand(v, generator=gen(1), device=DEV) < 0.01] = -math.inf
  first = None
  for beam_stride in (v, v + 1, v + 3, (v + 15) // 8 * 8):
    for place in range(16 // row.element_size()):
      space = torch.full((place + s * b * beam_stride,), 100.0, dtype=row.dtype, device=DEV)  # (more than any score)
      scores = space[place:].view(s, b, beam_stride)[:, :, :v]
      scores.copy_(row.expand(s, b, v))
      totals, beams, ids = table.select_beams(scores, keep=keep)
      # a constant taken from all scores alike leaves their order
      _, want_beams, want_ids = plain_select(scores, None, keep, False)
      assert torch.equal(beams, want_beams) and torch.equal(ids, want_ids)
      first = totals if first is None else first
      assert torch.equal(totals, first) and torch.equal(totals[0], totals[1])
  exact = row.double() - torch.logsumexp(row.double(), 0)
  assert (first[0, 0].double() - exact.max()).abs() <= 2 ** -20 + 2 ** -24 * exact.max().abs()
