"""The operators over a table of embeddings where their contracts are easiest to break."""
import math

import pytest
import torch
from torch.autograd import forward_ad

from cuhnsw_b200 import table
from test_gpu_table import DEV, TYPES, check_select, gen, ids_of, normal, plain_codes, plain_pack, plain_select

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


@pytest.mark.parametrize("offset", [-1e30, 1e30, float(torch.finfo(torch.float32).min), math.inf, -1e9])
@pytest.mark.parametrize("b, v", [(1, 5), (1, 100), (3, 700), (1, 9000), (2, 40_003), (300, 40)])
def test_totals_that_do_not_tell_scores_apart(offset, b, v):
  """Where a beam's total is so large that a score changes nothing, its continuations are ties: the smaller ids come first."""
  place = torch.arange(v, device=DEV)
  for i, dtype in enumerate(TYPES.values()):
    for row in (place / 8, -place / 8, normal(v + i, v), (place % 7 == 3) * 1.0, normal(v, v) * 1e-20):
      scores = row.to(dtype).expand(2, b, v).clone()
      scores[:, :, v // 2] = -math.inf
      scores[1].masked_fill_(torch.rand((b, v), generator=gen(i), device=DEV) < 0.3, math.nan)
      totals = torch.full((2, b), offset, device=DEV)
      totals[1, b // 2] = -2e30  # one beam before or after the others
      for keep in (1, 4, 37, 256):
        # (every term is a double without rounding but for the total itself, which is the same rounding on both sides)
        check_select(scores, totals, keep, False)


def test_totals_that_tell_some_scores_apart():
  """Beams of all kinds side by side, and scores close enough to 0 to vanish beside an ordinary total."""
  g = gen(3)
  tiny = 10.0 ** (-30 * torch.rand((3, 5, 3000), generator=g, device=DEV))
  scores = torch.where(torch.rand(tiny.shape, generator=g, device=DEV) < 0.5, tiny, -tiny)
  scores[0, 0, ::3] = 0.0
  scores[0, 1, ::2] = -0.0
  for totals in ([-20.0, -20.5, -20.0, -19.75, -20.0], [-20.0] * 5, [0.0, -0.0, 0.0, 0.0, 0.0], [-1e-9] * 5, [3.0, 1e30, -1e30, 1e30, -math.inf],
                 [-1e8, -1e9, -1e8, -1e8, -1e9]):
    for keep in (1, 5, 60, 256):
      for dtype in TYPES.values():
        at = torch.tensor(totals, device=DEV).expand(3, 5).contiguous()
        check_select(scores.to(dtype), at, keep, False)
        check_select(scores[:, :, :70].to(dtype), at, keep, False)  # (fewer continuations than results of some beams)
  # steps that a total of 1e9 merges by the dozen, at every place of a long row
  scores = (torch.randint(0, 1000, (1, 3, 50_000), generator=g, device=DEV) * 1e-9).float()
  for totals in ([1e9, 1e9, 1e9], [1e6, 1e6 + 1, 1e6 + 1], [-30.0, -30.0, -30.0]):
    for keep in (1, 7, 100, 256):
      check_select(scores, torch.tensor([totals], device=DEV), keep, False)
  # with the scores normalised too: the total is the beam's alone
  scores = normal(5, 2, 3, 6000, dtype=torch.float16)
  for keep in (1, 9, 256):
    check_select(scores, torch.tensor([[1e30, 1e30, 1e25], [-1e30, -1e30, -1e30]], device=DEV), keep, True)


# -- 4 bits ----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, d, group", [(9, 32, 32), (20_000, 50, 32), (300, 200, 64), (8000, 256, 256), (40, 300, 512), (60, 700, 128),
                                         (50, 2048, 128), (33, 1500, 512)])
def test_what_is_not_finite_costs_its_group_alone(dtype, n, d, group):
  rows = normal(d, n, d, dtype=TYPES[dtype])
  groups = -(-d // group)
  bad = torch.zeros((n, groups * group), dtype=torch.bool, device=DEV)
  bad[:, :d] = torch.rand((n, d), generator=gen(1), device=DEV) < 1 / (4 * min(d, group))
  bad[0, 0] = bad[n - 1, d - 1] = True
  values = torch.tensor([math.nan, math.inf, -math.inf], device=DEV)[torch.randint(0, 3, (n, groups * group), generator=gen(2), device=DEV)]
  values[0, 0] = math.nan
  spoilt = torch.where(bad[:, :d], values[:, :d].to(rows.dtype), rows)
  clean = torch.where(bad[:, :d], 0.0, rows)
  got, want = table.pack_rows(spoilt, group), table.pack_rows(clean, group)
  lost = bad.view(n, groups, group).any(2)
  nan = (bad & values.isnan()).view(n, groups, group).any(2)
  assert torch.equal(got.scales[~lost], want.scales[~lost])
  assert got.scales[nan].isnan().all() and (got.scales[lost & ~nan] == math.inf).all()
  out = got.unpack()
  of = lambda mask: mask.repeat_interleave(group, 1)[:, :d]
  expected = torch.where(of(nan), math.nan, torch.where(of(lost), torch.where(bad[:, :d], values[:, :d], math.nan), want.unpack()))
  assert torch.equal(out.isnan(), expected.isnan()) and torch.equal(out.nan_to_num(1e30), expected.nan_to_num(1e30))
  # no product of another row is touched
  scores, fine = got.scores(rows[:3]), want.scores(rows[:3])
  assert torch.equal(scores[:, ~lost.any(1)], fine[:, ~lost.any(1)]) and not scores[:, lost.any(1)].isfinite().any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [249, 250, 256])
def test_pack_with_a_group_that_is_a_row(dtype, d):
  rows = normal(d, 6001, d, dtype=TYPES[dtype])  # (rows of 32 words, four at a time)
  rows[5, :] = 0
  packed = table.pack_rows(rows, 256)
  codes, scales = plain_pack(rows, 256)
  assert torch.equal(packed.scales, scales) and torch.equal(plain_codes(packed), codes.double())
  assert torch.equal(packed.unpack(), codes * scales.float())


def packed_of(seed, n, d, group, values=range(-8, 8)):
  """(packed rows with scales that are powers of two, the values that they stand for)"""
  codes = torch.randint(0, len(values), (n, -(-d // 32) * 32), generator=gen(seed), device=DEV)
  codes = torch.tensor(list(values), device=DEV)[codes] + 8
  word, nibble = places(d)
  raw = torch.zeros((n, codes.shape[1] // 8), dtype=torch.int64, device=DEV)  # words of eight codes
  raw.index_add_(1, word, codes << nibble)
  raw = torch.where(raw >= 1 << 31, raw - (1 << 32), raw).to(torch.int32)
  scales = 2.0 ** torch.randint(0, 4, (n, -(-d // group)), generator=gen(seed + 1), device=DEV)
  rows = table.PackedRows(raw.view(torch.uint8), scales.bfloat16(), d, group)
  return rows, (codes[:, :d] - 8).double() * scales.double().repeat_interleave(group, 1)[:, :d]


def places(d):
  """Of every dimension (and those behind the last one in its block): its word in a row and the bit that its code begins at."""
  dims = torch.arange(-(-d // 32) * 32, device=DEV)
  block, four = dims // 32, dims // 128
  m = torch.clamp(len(dims) // 32 - 4 * four, max=4)
  t, j, k = dims % 32 // 8, block - 4 * four, dims % 8
  return 16 * four + t * m + j, 4 * (k // 2 + 4 * (k % 2))


SCORES = [(1, 129, 32), (15, 130, 64), (300, 257, 128), (64, 512, 256), (2000, 960, 128), (70, 1030, 384), (40, 4100, 1024), (5000, 200, 32),
          (48, 8192, 64), (3, 20_000, 128), (2100, 16_500, 64), (17_000, 300, 32), (40_000, 260, 64), (3000, 5000, 32), (9000, 5000, 128)]


@pytest.mark.parametrize("n, d, group", SCORES + [(100, 50, 32), (33, 128, 128), (31, 96, 64)])
def test_fp32_queries_enter_with_all_their_bits(n, d, group):
  """A query of one whole number of 24 bits: each of its parts, and their sum, is exact, and so is the product with 0 and powers of two."""
  packed, rows = packed_of(n, n, d, group, (-8, -4, -2, -1, 0, 1, 2, 4))
  for nq in (1, 7, 8, 9, 20):
    dims = torch.randint(0, d, (nq,), generator=gen(nq), device=DEV)
    dims[0], dims[-1] = d - 1, d // 2
    number = torch.randint(1 << 22, 1 << 23, (nq,), generator=gen(nq + 1), device=DEV) * 2 + 1
    queries = torch.zeros((nq, d), device=DEV)
    queries[torch.arange(nq, device=DEV), dims] = torch.where(number % 3 == 0, -number, number).float()
    want = queries[torch.arange(nq, device=DEV), dims].double()[:, None] * rows[:, dims].t()
    assert torch.equal(packed.scores(queries).double(), want)


@pytest.mark.parametrize("n, d", [(40, 1), (40, 100), (500, 200), (20_000, 300), (100, 5000)])
def test_the_largest_and_smallest_fp32_queries(n, d):
  packed, rows = packed_of(n, n, d, 32, (-1, 0, 1))
  packed = table.PackedRows(packed.codes, torch.ones_like(packed.scales), d, 32)
  rows = rows.sign()
  top, least = torch.finfo(torch.float32).max, 2.0 ** -110
  numbers = [top, -top, 3.396e38, 3.39617e38, 3.3962e38, 3.3895e38, least, least * (1 + 2 ** -23), -least * (2 - 2 ** -23), 2.0 ** -133]
  queries = torch.zeros((len(numbers), d), device=DEV)
  queries[:, d - 1] = torch.tensor(numbers, device=DEV)
  want = queries[:, d - 1:].double() * rows[:, d - 1]
  assert torch.equal(packed.scores(queries).double(), want)
  for other in (math.inf, -math.inf, math.nan):
    queries[0, d - 1] = other
    scores = packed.scores(queries)
    # (times 0 it is a NaN)
    assert torch.equal(scores[0].isinf(), (rows[:, d - 1] != 0) & math.isinf(other)) and not scores[0].isfinite().any()
    assert torch.equal(scores[1:].double(), want[1:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, d, group", SCORES + [(100, 50, 32)])
def test_scores_of_whole_numbers_are_exact(dtype, n, d, group):
  """Every sum is a whole number below 2^24, in whatever order: nothing may be missing or counted twice."""
  packed, rows = packed_of(n, n, d, group)
  most = min(100, ((1 << 24) - 200) // (64 * d))
  for nq in (1, 5, 8, 17, 33):
    queries = torch.randint(-most, most + 1, (nq, d), generator=gen(nq), device=DEV).to(TYPES[dtype])
    bias = torch.randint(-100, 101, (n,), generator=gen(3), device=DEV).float() if nq % 2 else None
    want = queries.double() @ rows.t() + (0 if bias is None else bias.double())
    assert torch.equal(packed.scores(queries, bias).double(), want)


def test_scores_and_searches_beyond_32_bits():
  n = 70_000_000
  codes = torch.randint(0, 256, (n, 16), generator=gen(1), device=DEV, dtype=torch.uint8)
  packed = table.PackedRows(codes, torch.ones((n, 1), dtype=torch.bfloat16, device=DEV), 32, 32)
  queries = torch.randint(-3, 4, (32, 32), generator=gen(2), device=DEV).float()
  scores = packed.scores(queries)  # 2.2 G scores
  for first in (0, 67_108_860, n - 1000):
    part = table.PackedRows(codes[first:first + 1000], packed.scales[first:first + 1000], 32, 32)
    assert torch.equal(scores[:, first:first + 1000].double(), queries.double() @ part.unpack().double().t())
  nns, distances, found = packed.search(queries, 5)
  assert (found == 5).all()
  for q in (0, 30, 31):
    best = scores[q].topk(5).values
    assert torch.equal(-distances[q], best) and torch.equal(scores[q][nns[q].long()], best)
    for value in best.unique():  # the first places of each
      mine = nns[q][best == value].long()
      assert torch.equal(mine, (scores[q] == value).nonzero().view(-1)[:len(mine)])
  del scores, codes, packed
  n, d = 2_200_000, 4096  # 4.5 GB of codes
  codes = torch.randint(0, 256, (n, d // 2), generator=gen(3), device=DEV, dtype=torch.uint8)
  packed = table.PackedRows(codes, torch.ones((n, d // 128), dtype=torch.bfloat16, device=DEV), d, 128)
  for dtype in (torch.float32, torch.bfloat16):
    queries = torch.randint(-9, 10, (3, d), generator=gen(4), device=DEV).to(dtype)
    scores = packed.scores(queries)
    for first in (0, 1_048_570, 2_097_150, n - 100):
      part = table.PackedRows(codes[first:first + 100], packed.scales[first:first + 100], d, 128)
      assert torch.equal(scores[:, first:first + 100].double(), queries.double() @ part.unpack().double().t())


def test_packing_beyond_32_bits():
  n, d = 600_000, 4096  # 2.5 G values
  rows = torch.randn((n, d), dtype=torch.bfloat16, generator=gen(1), device=DEV)
  for group in (128, 512):
    packed = table.pack_rows(rows, group)
    out = packed.unpack(torch.bfloat16)
    for first in (0, 524_280, n - 16):
      part = table.pack_rows(rows[first:first + 16], group)
      assert torch.equal(packed.codes[first:first + 16], part.codes) and torch.equal(packed.scales[first:first + 16], part.scales)
      assert torch.equal(out[first:first + 16], part.unpack(torch.bfloat16))
    del packed, out


# -- gradient --------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype, out_type", [("f32", "f32"), ("bf16", "f32"), ("f16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("count, n, d, kind", [
  (2, 1, 1, "one"), (65, 1000, 96, "any"), (512, 5000, 500, "one"), (512, 5001, 100, "zipf"), (1025, 2, 257, "uniform"), (5000, 4097, 100, "zipf"),
  (6144, 3, 33, "uniform"), (6145, 3, 33, "uniform"), (16_385, 70_000, 48, "any"), (20_000, 3, 2049, "any"), (40_961, 100_000, 8, "uniform"),
  (50_000, 255, 66, "one"), (64_000, 9, 130, "blocks"), (120_003, 131_072, 40, "zipf"), (300_000, 5, 17, "uniform"), (1_000_000, 20, 7, "blocks")])
def test_gradients_of_whole_numbers_are_exact(dtype, out_type, count, n, d, kind):
  """Every sum is a whole number below 2^24, in whatever order: no token and no partial sum may be missing or counted twice."""
  if kind == "blocks":  # a few long rows, one after another, of which none ends where a chunk does
    ids = torch.arange(count, device=DEV) * n // (count + 3)
  else:
    ids = ids_of(count, count, n, kind)
  grad = torch.randint(-8, 9, (count, d), generator=gen(count), device=DEV).to(TYPES[dtype])
  there = (ids >= 0) & (ids < n)
  sums = torch.zeros((n, d), dtype=torch.float64, device=DEV).index_add_(0, ids.clamp(0, n - 1), grad.double() * there[:, None])
  out = torch.full((n, d), math.nan, dtype=TYPES[out_type], device=DEV)
  assert torch.equal(table.lookup_grad(grad, ids, n, 0.25, out=out), (sums * 0.25).to(out.dtype))
  before = torch.randint(-100, 101, (n, d), generator=gen(1), device=DEV).to(out.dtype)
  added = table.lookup_grad(grad, ids, n, -2.0, out=before.clone(), accumulate=True)
  assert torch.equal(added, (before.double() - 2 * sums).to(out.dtype))


@pytest.mark.parametrize("dtype, out_type", [("f32", "f32"), ("bf16", "f32"), ("f16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("count, n, d, kind", [
  (1, 2_000_000, 30, "one"), (17, 1, 1, "one"), (64, 60_000, 24, "zipf"), (65, 20_000, 1, "zipf"), (96, 3, 511, "uniform"), (100, 100_000, 50, "ascending"),
  (127, 300_000, 9, "empty"), (128, 5000, 500, "one"), (128, 5001, 512, "any"), (128, 1_000_003, 16, "any"), (128, 2_000_000, 100, "uniform"),
  (128, 40, 1024, "zipf"), (128, 2, 300, "blocks"), (129, 5001, 300, "zipf"), (129, 2, 7, "blocks")])
def test_gradients_of_few_whole_numbers_are_exact(dtype, out_type, count, n, d, kind):
  test_gradients_of_whole_numbers_are_exact(dtype, out_type, count, n, d, kind)


def test_gradients_beyond_32_bits():
  count, n, d = 600_000, 560_000, 4096  # 2.5 G values, and 2.3 G of the table
  grad = torch.randint(-8, 9, (count, d), generator=gen(1), device=DEV, dtype=torch.int8).to(torch.bfloat16)
  ids = ids_of(2, count, n, "uniform", torch.int32)
  ids[1000:200_000:7] = n - 1
  out = table.lookup_grad(grad, ids, n)
  for c in (0, 1, 2047, d - 1):
    sums = torch.zeros(n, dtype=torch.float64, device=DEV).index_add_(0, ids, grad[:, c].double())
    assert torch.equal(out[:, c], sums.to(torch.bfloat16))


# -- derivatives -----------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("recorded", [False, True])
def test_a_tangent_passes_through_a_lookup(dtype, recorded):
  rows = normal(1, 30, 12, dtype=TYPES[dtype]).requires_grad_(recorded)
  tangent = normal(2, 30, 12, dtype=TYPES[dtype])
  ids = torch.tensor([[3, -1, 29], [3, 30, 0]], device=DEV)
  with forward_ad.dual_level():
    for given in (rows, rows.t().contiguous().t()):
      out, out_tangent = forward_ad.unpack_dual(table.lookup(forward_ad.make_dual(given, tangent), ids, -1.5))
      assert torch.equal(out, table.lookup(rows.detach(), ids, -1.5)) and torch.equal(out_tangent, table.lookup(tangent, ids, -1.5))
      assert out.requires_grad == recorded
    assert forward_ad.unpack_dual(table.lookup(rows, ids)).tangent is None


def underived(x):
  """Results that depend on `x` [6, 32] through each operator without a derivative, by its name."""
  rows = normal(1, 40, 32)
  packed = table.pack_rows(rows, 32)
  ids, beams = torch.arange(6, device=DEV), torch.tensor([[1, 0, -1], [0, 1, 1]], dtype=torch.int32, device=DEV)
  with torch.no_grad():
    scales = packed.scales.clone()
  return {
    "PackedRows.scores": lambda: [packed.scores(x), packed.scores(rows[:3], bias=x.reshape(-1)[:40])],
    "PackedRows.search": lambda: [packed.search(x, 3)[1], packed.search(rows[:3], 3, bias=x.reshape(-1)[:40])[1]],
    "PackedRows.unpack": lambda: [table.PackedRows(packed.codes, scales * x[0, 0].to(scales.dtype), 32, 32).unpack()],
    "select_beams": lambda: [table.select_beams(x.view(2, 3, 32))[0], table.select_beams(rows[None, :6], x[:, 0].reshape(1, 6))[0]],
    "reorder": lambda: [table.reorder(x.view(2, 3, 32), beams), table.reorder([ids.view(2, 3), x.view(2, 3, 4, 8)], beams)[1]],
    "lookup_grad": lambda: [table.lookup_grad(x, ids, 9)],
  }


def test_derivatives_that_there_are_not_are_refused_where_they_are_asked_for():
  x = normal(3, 6, 32)
  plain = {name: call() for name, call in underived(x).items()}
  x.requires_grad_()
  for name, call in underived(x).items():
    for out, want in zip(call(), plain[name]):
      assert torch.equal(out, want) and out.requires_grad
      with pytest.raises(RuntimeError, match=f"derivative for {name} is not implemented"):
        (2 * out).sum().backward()
    with torch.no_grad():
      assert not any(out.requires_grad for out in call())
  assert x.grad is None
  nns, _, found = table.pack_rows(x, 32).search(x, 2)
  _, beams, ids = table.select_beams(x[None])
  assert not any(t.requires_grad for t in (nns, found, beams, ids, table.pack_rows(x, 32).scores(x.detach())))
  assert not table.reorder([beams, x[None]], torch.zeros((1, 2), dtype=torch.int32, device=DEV))[0].requires_grad
  with pytest.raises(RuntimeError, match="out cannot be given"):
    table.lookup_grad(x, torch.arange(6, device=DEV), 9, out=torch.zeros((9, 32), device=DEV))
  with torch.no_grad():
    table.lookup_grad(x, torch.arange(6, device=DEV), 9, out=torch.zeros((9, 32), device=DEV))
  with forward_ad.dual_level():
    for name, call in underived(forward_ad.make_dual(x.detach(), torch.ones_like(x))).items():
      with pytest.raises(RuntimeError, match=f"{name} has no derivative"):
        call()
