"""The operators over a table of embeddings against plain implementations in 64 bits.

Tolerances: a rounding to a type is off by at most finfo(type).eps / 2 of the value; a sum of m products in fp32 by at most
about m * 2^-24 times the sum of their magnitudes (2^-23 where the matrix instruction adds, which may cut instead of round)."""
import math
import subprocess
import sys
import threading
from pathlib import Path

import numpy as np
import pytest
import torch

from conftest import has_gpu
from cuhnsw_b200 import CuHNSW, table

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"


def half_step(t):
  return torch.finfo(t).eps / 2


def gen(seed):
  return torch.Generator(device=DEV).manual_seed(seed)


def normal(seed, *shape, dtype=torch.float32, sigma=1.0):
  return (torch.randn(shape, generator=gen(seed), device=DEV) * sigma).to(dtype)


def ids_of(seed, count, n, kind, dtype=torch.int64):
  g = gen(seed)
  if kind == "uniform":
    ids = torch.randint(0, n, (count,), generator=g, device=DEV)
  elif kind == "zipf":
    ids = torch.exp(torch.rand(count, generator=g, device=DEV).double() * math.log(n)).long().clamp(1, n) - 1
  elif kind == "one":
    ids = torch.full((count,), n - 1, device=DEV)
  elif kind == "empty":
    ids = torch.full((count,), -1, device=DEV)
  elif kind == "ascending":
    ids = torch.arange(count, device=DEV) % n
  else:  # empty slots of both kinds among them
    ids = torch.randint(-n // 4 - 1, n + n // 4 + 1, (count,), generator=g, device=DEV)
  return ids.to(dtype)


def plain_lookup(rows, ids, scale):
  there = (ids >= 0) & (ids < rows.shape[0])
  out = rows[ids.long().clamp(0, max(0, rows.shape[0] - 1))].float() * scale if rows.shape[0] else \
    torch.zeros(ids.shape + rows.shape[1:], device=rows.device)
  return torch.where(there.unsqueeze(-1), out, torch.zeros((), device=rows.device)).to(rows.dtype)


# -- lookup ----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [1, 2, 3, 8, 31, 50, 64, 100, 257, 960, 2048, 4099])
def test_lookup_equals_the_product_rounded_once(dtype, d):
  n = 301
  rows = normal(d, n, d, dtype=TYPES[dtype])
  for count, kind, id_type, scale in ((1, "uniform", torch.int64, 1.0), (7, "any", torch.int32, 3.3),
                                      (2000, "zipf", torch.int64, math.sqrt(d)), (5003, "any", torch.int32, 1.0)):
    ids = ids_of(count, count, n, kind, id_type)
    assert torch.equal(table.lookup(rows, ids, scale), plain_lookup(rows, ids, scale))


def test_lookup_shapes_strides_and_edges():
  wide = normal(1, 40, 100, dtype=torch.bfloat16)
  for rows in (wide[:, :50], wide[:, 1:34], wide[::3, 4:68], wide.t()[:40], wide[:1].expand(7, 100)):
    ids = ids_of(2, 24, rows.shape[0], "any").view(2, 3, 4)
    for i in (ids, ids.transpose(0, 2), ids[:, 1], ids[:, :0]):
      out = table.lookup(rows, i, 2.0)
      assert out.shape == i.shape + rows.shape[1:] and torch.equal(out, plain_lookup(rows, i, 2.0))
  assert torch.equal(table.lookup(wide, torch.tensor(3, device=DEV)), wide[3])
  assert table.lookup(wide[:, :0], ids).shape == ids.shape + (0,)
  assert not table.lookup(wide[:0], ids).any()
  far = torch.tensor([2 ** 40, -2 ** 40, 2 ** 31 + 1, 2, -2 ** 63, 2 ** 32 + 2], device=DEV)
  assert torch.equal(table.lookup(wide, far), plain_lookup(wide, far, 1.0))
  special = torch.tensor([[math.inf, -math.inf, math.nan, -0.0]], device=DEV)
  out = table.lookup(special, torch.zeros(1, dtype=torch.int64, device=DEV))
  assert torch.equal(out.view(torch.int32), special.view(torch.int32))


def test_lookup_offsets_beyond_32_bits():
  n, d = 1_200_000, 2048
  rows = torch.zeros((n, d), dtype=torch.bfloat16, device=DEV)  # 4.9 GB, 2.5 G values
  rows[:, 0] = torch.arange(n, device=DEV) % 251
  rows[:, -1] = torch.arange(n, device=DEV) % 241
  ids = torch.tensor([n - 1, 0, 1_048_576, 1_048_575, n - 2], device=DEV)
  out = table.lookup(rows, ids)
  assert torch.equal(out, rows[ids])


# -- gradient --------------------------------------------------------------------------------------------------------


def check_grad(grad, ids, n, scale, out, before=None):
  live = (ids >= 0) & (ids < n)
  at = ids.long()[live]
  exact = torch.zeros((n, grad.shape[1]), dtype=torch.float64, device=DEV).index_add_(0, at, grad[live].double())
  size = torch.zeros_like(exact).index_add_(0, at, grad[live].double().abs())
  most = torch.zeros(n, dtype=torch.float64, device=DEV).index_add_(0, at, torch.ones(len(at), dtype=torch.float64, device=DEV))
  exact, size = exact * scale, size * abs(scale)
  # one rounding per addition, one for the scale, and one of the sum with what was there
  slack = (most[:, None] + 2) * 2 ** -24 * size
  if before is not None:
    exact = exact + before.double()
    slack = slack + 2 ** -24 * exact.abs()
  slack = slack * 1.01 + half_step(out.dtype) * (exact.abs() + slack) + torch.finfo(out.dtype).tiny
  assert ((out.double() - exact).abs() <= slack).all()
  if before is None:
    assert not out[most == 0].any()
  else:
    assert torch.equal(out[most == 0], before[most == 0])


@pytest.mark.parametrize("dtype, out_type", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("count, n, d, kind", [
  (1, 5, 3, "uniform"), (2, 1, 1, "one"), (8, 1, 7, "any"), (9, 100, 64, "ascending"), (63, 7, 50, "zipf"), (64, 64, 33, "uniform"),
  (65, 1000, 96, "any"), (511, 300, 128, "zipf"), (1025, 2, 257, "uniform"), (5000, 4097, 100, "zipf"),
  (16384, 70_000, 48, "zipf"), (16385, 70_000, 48, "any"), (20_000, 3, 2049, "any"), (40_961, 1_000_000, 8, "uniform"),
  (50_000, 255, 66, "one"), (70_000, 256, 12, "empty"), (120_003, 131_072, 40, "zipf")])
def test_grad_against_64_bits(dtype, out_type, count, n, d, kind):
  grad = normal(count, count, d, dtype=TYPES[dtype])
  ids = ids_of(count + 1, count, n, kind, torch.int32 if count % 2 else torch.int64)
  out = torch.full((n, d), math.nan, dtype=TYPES[out_type], device=DEV)
  got = table.lookup_grad(grad, ids, n, 1.5, out=out)
  assert got is out
  check_grad(grad, ids, n, 1.5, out)
  before = normal(7, n, d, dtype=TYPES[out_type])
  added = table.lookup_grad(grad, ids, n, -0.5, out=before.clone(), accumulate=True)
  check_grad(grad, ids, n, -0.5, added, before)
  if dtype == out_type:  # the same bits every time
    assert torch.equal(table.lookup_grad(grad, ids, n, 1.5), out)


@pytest.mark.parametrize("dtype, out_type", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("count, n, d, kind", [
  (1, 1, 1, "one"), (32, 40, 5, "zipf"), (31, 3, 512, "any"), (32, 1, 511, "one"), (33, 200_000, 13, "any"), (256, 60_000, 24, "zipf"),
  (257, 20_000, 120, "zipf"), (512, 5000, 500, "one"), (512, 5001, 512, "zipf"), (511, 300_000, 9, "empty"), (512, 100_000, 50, "ascending"),
  (512, 1_000_003, 16, "any"), (500, 1500, 1021, "any"), (513, 5000, 500, "zipf")])
def test_grad_of_few_tokens(dtype, out_type, count, n, d, kind):
  grad = normal(count, count, d + 3, dtype=TYPES[dtype])[:, :d]
  ids = ids_of(count + 2, count, n, kind, torch.int32 if count % 2 else torch.int64)
  if ids.dtype == torch.int64 and count > 8:
    ids[3], ids[5] = -2 ** 63, 2 ** 63 - 1
  space = torch.full((n * d + 2,), 7.0, dtype=TYPES[out_type], device=DEV)
  out = space[1:-1].view(n, d)  # at an odd place, between values that stay
  table.lookup_grad(grad, ids, n, -2.5, out=out)
  assert space[0] == 7 and space[-1] == 7
  check_grad(grad, ids, n, -2.5, out)
  even = table.lookup_grad(grad.contiguous(), ids, n, -2.5, out=torch.full_like(out, math.nan))
  check_grad(grad, ids, n, -2.5, even)
  assert torch.equal(table.lookup_grad(grad.contiguous(), ids, n, -2.5, out=torch.full_like(out, math.nan)), even)


def test_grad_takes_any_layout():
  wide = normal(3, 500, 100)
  ids = ids_of(4, 500, 60, "any")
  for grad in (wide[:, :50], wide[:, 3:36], normal(5, 100, 500).t(), wide[:1].expand(500, 100),
               torch.ones((), device=DEV).expand(500, 100)):
    check_grad(grad, ids, 60, 2.0, table.lookup_grad(grad, ids, 60, 2.0))
  out = table.lookup_grad(wide.view(5, 100, 100), ids.view(5, 100), 60)
  assert torch.equal(out, table.lookup_grad(wide, ids, 60))
  # a dense output at an odd place
  space = torch.zeros(60 * 100 + 1, device=DEV)
  at = space[1:].view(60, 100)
  table.lookup_grad(wide, ids, 60, out=at)
  assert torch.equal(at, out) and space[0] == 0
  assert table.lookup_grad(wide[:0], ids[:0], 5).abs().sum() == 0
  assert table.lookup_grad(wide, ids, 0).shape == (0, 100)
  assert table.lookup_grad(wide[:, :0], ids, 4).shape == (4, 0)
  kept = torch.ones(5, 100, device=DEV)
  assert torch.equal(table.lookup_grad(wide[:0], ids[:0], 5, out=kept, accumulate=True), torch.ones_like(kept))


def test_grad_leaves_what_surrounds_its_output():
  for count in (300, 30_000):
    for d, dtype in ((50, torch.float32), (33, torch.bfloat16)):
      guard = torch.full((1002, d), 7.0, dtype=dtype, device=DEV)
      table.lookup_grad(normal(1, count, d, dtype=dtype), ids_of(2, count, 1000, "any"), 1000, out=guard[1:1001])
      assert (guard[0] == 7).all() and (guard[1001] == 7).all()


def test_grad_keeps_non_finite_values_in_their_rows():
  grad = normal(1, 400, 32)
  ids = ids_of(2, 400, 50, "uniform")
  grad[17, 3], grad[18, 4] = math.inf, math.nan
  out = table.lookup_grad(grad, ids, 50)
  bad = ~torch.isfinite(out)
  assert bad.sum() == 2 and bad[ids[17], 3] and bad[ids[18], 4]


@pytest.mark.parametrize("dtype", TYPES)
def test_autograd_is_the_formula(dtype):
  rows = normal(1, 90, 40, dtype=TYPES[dtype]).requires_grad_()
  ids = ids_of(2, 120, 90, "any").view(4, 30)
  weight = normal(3, 4, 30, 40, dtype=TYPES[dtype])
  (table.lookup(rows, ids, 2.5) * weight).sum().backward()
  assert torch.equal(rows.grad, table.lookup_grad(weight, ids, 90, 2.5))
  with torch.no_grad():
    assert not table.lookup(rows, ids).requires_grad
  out = table.lookup(rows, ids)
  grad, = torch.autograd.grad(out.sum(), rows)  # an expanded gradient
  counts = torch.bincount(ids[(ids >= 0) & (ids < 90)], minlength=90).to(TYPES[dtype])
  assert torch.equal(grad, counts[:, None].expand(90, 40))


def test_gradient_against_differences():
  rows = normal(1, 6, 5)
  ids = torch.tensor([[0, 3, 3], [5, -1, 3]], device=DEV)

  def loss(r):
    return (table.lookup(r, ids, 1.7).double() ** 2).sum()

  r = rows.clone().requires_grad_()
  loss(r).backward()
  step = 2.0 ** -6
  for i in range(6):
    for j in range(5):
      up, down = rows.clone(), rows.clone()
      up[i, j] += step
      down[i, j] -= step
      # of a quadratic function the central difference is the derivative; the values carry fp32 roundings: each of up to three
      # squares is off by 2 * 2^-24 of itself and the step by a rounding of the argument
      size = 3 * 1.7 ** 2 * (abs(rows[i, j].item()) + step) ** 2
      difference = (loss(up) - loss(down)).item() / (up[i, j] - down[i, j]).item()
      assert abs(difference - r.grad[i, j].item()) <= 8 * 2 ** -24 * size / (2 * step) + 2 ** -20 * abs(r.grad[i, j].item())


# -- 4 bits ----------------------------------------------------------------------------------------------------------


def plain_pack(rows, group):
  """codes - 8 and scales in the arithmetic that the format is defined in"""
  n, d = rows.shape
  groups = -(-d // group)
  padded = torch.nn.functional.pad(rows.float(), (0, groups * group - d)).view(n, groups, group)
  scales = (padded.abs().amax(2) * torch.tensor(1 / 7, dtype=torch.float32, device=DEV)).bfloat16()
  step = scales.float()[:, :, None]
  codes = torch.where(step > 0, (padded / step).round().clamp(-8, 7), torch.zeros_like(padded))
  return codes.view(n, -1)[:, :d], scales


def plain_codes(packed):
  """code - 8 of every dimension, taken from the documented places one by one"""
  d, blocks = packed.num_dims, -(-packed.num_dims // 32)
  raw = packed.codes.cpu().numpy()
  out = np.zeros((packed.num_rows, d), np.float64)
  for i in range(d):
    block, four = i // 32, i // 128
    m = min(4, blocks - 4 * four)
    t, j, k = i % 32 // 8, block - 4 * four, i % 8
    nibble = k // 2 + 4 * (k % 2)
    byte = raw[:, 64 * four + 4 * (t * m + j) + nibble // 2]
    out[:, i] = (byte >> 4 if nibble % 2 else byte & 15).astype(np.float64) - 8
  return torch.from_numpy(out).to(DEV)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [1, 7, 8, 31, 32, 33, 50, 64, 96, 100, 128, 129, 200, 256, 300, 511, 960, 1300])
@pytest.mark.parametrize("group", [32, 64, 128, 384, 512])
def test_pack_and_unpack(dtype, d, group):
  for n in (1, 37):
    rows = normal(d, n, d, dtype=TYPES[dtype], sigma=0.2)
    rows[n // 2, :40] = 0  # groups without a scale
    rows[0, -1] = 5.0
    packed = table.pack_rows(rows, group)
    codes, scales = plain_pack(rows, group)
    assert torch.equal(packed.scales, scales)
    assert torch.equal(plain_codes(packed), codes.double())
    values = codes * scales.float().repeat_interleave(group, 1)[:, :d]
    for to in TYPES.values():
      assert torch.equal(packed.unpack(to), values.to(to))


def test_pack_takes_any_layout():
  wide = normal(1, 50, 300)
  for rows in (wide[:, :100], wide[:, 1:50], wide[::2, 3:200], wide.t()[:200], wide[:1].expand(9, 300)):
    a, b = table.pack_rows(rows, 64), table.pack_rows(rows.contiguous(), 64)
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
  rows = normal(2, 100_000, 32)  # many groups: scales at the border of two bfloat16 values among them
  packed, (codes, scales) = table.pack_rows(rows, 32), plain_pack(rows, 32)
  assert torch.equal(packed.scales, scales) and torch.equal(packed.unpack(), codes * scales.float())
  empty = table.pack_rows(wide[:0], 32)
  assert empty.num_rows == 0 and empty.unpack().shape == (0, 300) and empty.scores(wide).shape == (50, 0)


def random_packed(seed, n, d, group):
  """All 16 codes, scales of both signs and several magnitudes, and other bits than 8 behind the last dimension"""
  codes = torch.randint(0, 256, (n, 16 * -(-d // 32)), generator=gen(seed), device=DEV).to(torch.uint8)
  scales = normal(seed + 1, n, -(-d // group), dtype=torch.bfloat16, sigma=0.1)
  scales[0] = 0
  return table.PackedRows(codes, scales, d, group)


def check_scores(packed, queries, bias, out):
  values = packed.unpack().double() if packed.num_rows else torch.zeros((0, packed.num_dims), dtype=torch.float64, device=DEV)
  x = queries.double()
  exact = x @ values.T
  size = x.abs() @ values.abs().T
  if bias is not None:
    exact, size = exact + bias.double(), size + bias.double().abs()
  # (code - 8) * scale itself is exact to 2^-24 in unpack()
  slack = (packed.num_dims + 16) * 2 ** -23 * size * 1.01 + torch.finfo(torch.float32).tiny
  assert out.dtype == torch.float32 and out.shape == exact.shape
  assert ((out.double() - exact).abs() <= slack).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, d, group", [
  (1, 1, 32), (15, 8, 32), (16, 33, 32), (17, 50, 64), (129, 64, 64), (200, 96, 32), (300, 128, 128), (1000, 130, 64),
  (333, 257, 128), (64, 512, 256), (2000, 960, 128), (70, 1030, 384), (40, 4100, 1024), (5000, 50, 32), (48, 8192, 64)])
def test_scores_against_64_bits(dtype, n, d, group):
  packed = random_packed(n + d, n, d, group)
  for nq in (1, 2, 3, 7, 8, 9, 16, 21, 32, 45):
    queries = normal(nq, nq, d, dtype=TYPES[dtype])
    bias = normal(5, n) if nq % 2 else None
    check_scores(packed, queries, bias, packed.scores(queries, bias))


def test_scores_of_many_rows_and_wide_rows():
  for n, d, group, nq, dtype in ((100_003, 50, 64, 5, "f32"), (60_000, 256, 32, 32, "bf16"), (3, 40_000, 128, 2, "f32"),
                                 (2100, 16_500, 64, 32, "f16"), (100, 20_000, 32, 33, "f32")):
    packed = random_packed(1, n, d, group)
    queries = normal(2, nq, d, dtype=TYPES[dtype])
    check_scores(packed, queries, None, packed.scores(queries))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n, d, group", [(16_384, 256, 128), (16_500, 257, 32), (20_001, 300, 64), (16_385, 520, 256), (17_000, 1100, 384),
                                         (40_007, 384, 32), (16_389, 2050, 64), (16_384, 4999, 128)])
def test_scores_of_many_queries(dtype, n, d, group):
  packed = random_packed(n + d, n, d, group)
  for nq in (9, 16, 17, 32, 33, 50):
    wide = normal(nq, nq, (d + 7) // 8 * 8, dtype=TYPES[dtype])  # rows at 16-byte boundaries
    bias = normal(5, n) if nq % 2 else None
    check_scores(packed, wide[:, :d], bias, packed.scores(wide[:, :d], bias))


def test_scores_layouts_and_values():
  packed = random_packed(3, 77, 100, 32)
  wide = normal(4, 60, 300)
  for queries in (wide[:, :100], wide[:, 7:107], wide[::5, 100:200], wide[:, ::3],
                  wide[:1, :100].expand(4, 100), wide[:0, :100]):
    check_scores(packed, queries, None, packed.scores(queries))
  # three parts of 8 bits hold an fp32 value: whole numbers below 2^24 times codes are exact in each product
  rows = table.PackedRows(torch.full((4, 16), 0x99, dtype=torch.uint8, device=DEV), torch.ones((4, 1), dtype=torch.bfloat16, device=DEV), 1, 32)
  x = torch.tensor([[float(2 ** 24 - 1)], [float(2 ** 23 + 1)], [2.0 ** -100], [3.0e38]], device=DEV)
  assert torch.equal(rows.scores(x), x.expand(4, 4))
  # what is not finite stays with its query
  for dtype in TYPES.values():
    x = normal(5, 9, 100, dtype=dtype)
    x[4, 50], x[6, 3] = math.inf, math.nan
    bad = ~torch.isfinite(packed.scores(x))
    assert not bad[[0, 1, 2, 3, 5, 7, 8]].any() and bad[6].all() and bad[4].any()


def test_scores_write_their_rows_only():
  packed = random_packed(3, 61, 96, 32)
  queries = normal(4, 5, 96)
  space = torch.full((7, 61), 3.0, device=DEV)
  from cuhnsw_b200.cuhnsw_bind import load_library
  rc = load_library().cuhnsw_scores4_device(packed.codes.data_ptr(), packed.scales.data_ptr(), 61, 96, 32, queries.data_ptr(), 96,
                                            0, 5, None, space[1].data_ptr(), torch.cuda.current_stream().cuda_stream)
  assert rc == 0
  assert (space[0] == 3).all() and (space[6] == 3).all() and torch.equal(space[1:6], packed.scores(queries))


def test_search_is_exhaustive_and_in_the_order_of_the_index():
  rows = normal(1, 3000, 64, dtype=torch.bfloat16)
  rows[100:200] = rows[300:400]  # equal distances: the smaller id first
  packed = table.pack_rows(rows, 32)
  queries = normal(2, 20, 64)
  for topk in (1, 10, 100, 256):
    nns, distances, found = packed.search(queries, topk)
    scores = packed.scores(queries)
    value, at = scores.sort(dim=1, descending=True, stable=True)
    assert torch.equal(nns.long(), at[:, :topk]) and torch.equal(distances, -value[:, :topk]) and (found == topk).all()
  few = table.pack_rows(rows[:5], 32)
  nns, distances, found = few.search(queries, 8)
  assert (found == 5).all() and (nns[:, 5:] == -1).all() and (distances[:, 5:] == math.inf).all()
  nns, distances, found = table.pack_rows(rows[:0], 32).search(queries, 3)
  assert (nns == -1).all() and (distances == math.inf).all() and (found == 0).all()


# -- beams -----------------------------------------------------------------------------------------------------------


def plain_select(scores, totals, keep, norm):
  s, b, v = scores.shape
  t = scores.double()
  if norm:
    t = t - torch.logsumexp(t, 2, keepdim=True)
  if totals is not None:
    t = t + totals.double()[:, :, None]
  t = torch.where(t > -math.inf, t, -math.inf).reshape(s, -1)
  value, at = t.sort(dim=1, descending=True, stable=True)
  if value.shape[1] < keep:
    value = torch.nn.functional.pad(value, (0, keep - value.shape[1]), value=-math.inf)
    at = torch.nn.functional.pad(at, (0, keep - at.shape[1]))
  value, at = value[:, :keep], at[:, :keep]
  lost = value == -math.inf
  return value, torch.where(lost, -1, at // v).int(), torch.where(lost, -1, at % v).int()


def check_select(scores, totals, keep, norm, got=None):
  value, beams, ids = plain_select(scores, totals, keep, norm)
  t, b, i = got or table.select_beams(scores, totals, keep, log_softmax=norm)
  assert torch.equal(b, beams) and torch.equal(i, ids)
  live = beams >= 0
  assert (t[~live] == -math.inf).all()
  # fp32 exponentials (2 units, and up to 2^-24 times the argument) in the sum, and the rounding of the total
  slack = (2 ** -20 if norm else 0) + 2 ** -24 * value[live].abs()
  assert ((t[live].double() - value[live]).abs() <= slack).all() or torch.equal(t[live], value[live].float())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("s, b, v, keep", [
  (1, 1, 1, 1), (1, 1, 5, 8), (3, 2, 31, 4), (2, 4, 1000, 8), (5, 3, 2047, 6), (1, 4, 2049, 64), (4, 1, 32_000, 256), (2, 8, 50_001, 16),
  (1, 16, 8193, 33), (20, 5, 4100, 10), (40, 8, 9000, 8), (1, 2, 151_000, 100)])
def test_select_against_64_bits(dtype, s, b, v, keep):
  scores = normal(v, s, b, v, dtype=TYPES[dtype], sigma=3.0)
  scores.masked_fill_(torch.rand((s, b, v), generator=gen(1), device=DEV) < 0.02, -math.inf)
  totals = -20 * torch.rand((s, b), generator=gen(2), device=DEV)
  check_select(scores, totals, keep, True)
  check_select(scores, totals, keep, False)
  check_select(scores, None, keep, True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pattern", ["equal", "few values", "rising", "falling", "steps of 256", "steps of 2048", "blocks"])
def test_select_with_ties_and_in_any_order(dtype, pattern):
  s, b, v = 2, 3, 20_000
  place = torch.arange(v, device=DEV)
  row = {"equal": torch.zeros(v, device=DEV), "few values": torch.randint(0, 3, (v,), generator=gen(1), device=DEV),
         "rising": place * (1 / 8), "falling": -place * (1 / 8), "steps of 256": (place % 256 == 5) * 1.0,
         "steps of 2048": (place % 2048 < 8) * (place / 2048).floor(), "blocks": (place // 700 % 5) * 1.0}[pattern]
  scores = row.to(TYPES[dtype]).expand(s, b, v).contiguous()
  totals = torch.tensor([[0.0, 0.0, 0.0], [-1.0, 0.0, 1.0]], device=DEV)
  for keep in (1, 4, 37, 256):
    # whole and binary fractions: every total is exact, ties are ties
    check_select(scores, totals, keep, False)
    check_select(scores[:, :1], totals[:, :1].contiguous(), keep, True)


def test_select_masks_infinities_and_nan():
  scores = normal(1, 6, 4, 3000)
  totals = torch.zeros(6, 4, device=DEV)
  totals[0] = -math.inf                                  # nothing is left of a sequence
  totals[1, :3] = -math.inf                              # one beam is
  scores[2] = -math.inf                                  # no id may follow
  scores[3, 1] = -math.inf                               # no id may follow one beam
  scores[3, 2] = torch.finfo(torch.float32).min          # a mask of the lowest value
  scores[4, 0, 17] = math.nan
  scores[5, 1, 100] = math.inf
  totals[4, 2] = math.nan
  for norm in (True, False):
    want = plain_select(scores, totals, 8, norm)
    got = table.select_beams(scores, totals, 8, log_softmax=norm)
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    check_select(scores[:4], totals[:4], 8, norm)
    assert (got[1][0] == -1).all() and (got[1][1] == 3).all() and (got[1][2] == -1).all()
  all_masked = torch.full((1, 2, 700), torch.finfo(torch.float32).min, device=DEV)
  check_select(all_masked, None, 5, True)
  only = torch.full((1, 2, 700), -math.inf, device=DEV)
  only[0, 1, 699] = -3.0
  check_select(only, None, 4, True)
  check_select(only, None, 4, False)


def test_select_layouts():
  base = normal(1, 4, 6, 3001)
  for scores in (base[:, ::2], base[::2, 1:], base[:, :, 1:2000], base[:, :, ::3], base.transpose(0, 1), base[:1].expand(3, 6, 3001),
                 normal(2, 30, 5, 4).permute(2, 1, 0)):
    check_select(scores, None, 7, True)
  got = table.select_beams(base, torch.zeros(4, 12, device=DEV)[:, ::2])
  check_select(base, None, 6, True, got)
  assert table.select_beams(base[:0], keep=2)[0].shape == (0, 2)
  empty = table.select_beams(base[:, :, :0], keep=2)
  assert (empty[0] == -math.inf).all() and (empty[1] == -1).all() and (empty[2] == -1).all()
  wide = normal(3, 1, 700, 40)  # more beams than threads
  check_select(wide, normal(4, 1, 700), 50, True)


def test_select_rows_beyond_32_bits():
  scores = torch.zeros((1, 70_000, 31_000), dtype=torch.float16, device=DEV)[:, ::5]  # 14 000 beams, 4.3 GB apart
  scores[0, 13_999, 30_999] = 2.0
  scores[0, 13_998, 5] = 1.0
  totals, beams, ids = table.select_beams(scores, keep=3, log_softmax=False)
  assert totals.tolist() == [[2.0, 1.0, 0.0]] and beams.tolist() == [[13_999, 13_998, 0]] and ids.tolist() == [[30_999, 5, 0]]


def plain_reorder(state, beams):
  at = beams.long().clamp(min=0)
  out = torch.stack([state[s][at[s]] for s in range(len(at))]) if len(at) else state[:, :0]
  return torch.where((beams >= 0).view(beams.shape + (1,) * (state.dim() - 2)), out, torch.zeros((), dtype=state.dtype, device=DEV))


def test_reorder():
  beams = torch.tensor([[2, 2, -1, 0], [1, 0, 0, 2], [-1, -1, 1, 1]], dtype=torch.int32, device=DEV)
  cache = normal(1, 3, 3, 4, 20, 16, dtype=torch.bfloat16)
  states = [cache, cache[:, :, :, :7], cache[:, :, :, 3:4], cache[:, :, 1:, 2:9, :5], cache.transpose(2, 3), cache.transpose(0, 1),
            torch.arange(9, device=DEV).view(3, 3), torch.arange(63, device=DEV).view(3, 3, 7).to(torch.uint8),
            torch.rand((3, 3, 1001), generator=gen(1), device=DEV) > 0.5, normal(2, 3, 3, 5).double(), cache[:, :, :0],
            normal(3, 3, 3, 33, dtype=torch.float16)[:, :, 1:], cache[:, :1].expand(3, 3, 4, 20, 16)]
  outs = table.reorder(states, beams)
  for state, out in zip(states, outs):
    assert out.shape == (3, 4) + state.shape[2:] and out.is_contiguous() and torch.equal(out, plain_reorder(state, beams))
  assert torch.equal(table.reorder(cache, beams), outs[0])
  many = [normal(i, 3, 3, i + 1) for i in range(70)]
  for state, out in zip(many, table.reorder(tuple(many), beams)):
    assert torch.equal(out, plain_reorder(state, beams))
  assert table.reorder([], beams) == []
  assert table.reorder(cache, beams[:, :0]).shape == (3, 0, 4, 20, 16)
  outside = torch.tensor([[3, 2 ** 31 - 1], [-2 ** 31, 0], [1, 7]], dtype=torch.int32, device=DEV)
  assert torch.equal(table.reorder(cache, outside), plain_reorder(cache, torch.where((outside < 0) | (outside > 2), -1, outside)))


# -- together --------------------------------------------------------------------------------------------------------


def step(rows, packed, tokens, totals, memory, keep):
  """One step of a small decoder over the table: its state mixes the last tokens' rows."""
  s, b = totals.shape
  memory = 0.5 * memory + table.lookup(rows, tokens, 4.0).float()
  scores = packed.scores(memory.view(s * b, -1)).view(s, b, -1)
  totals, beams, ids = table.select_beams(scores, totals, keep)
  return table.reorder(memory, beams), totals, beams, ids


def test_a_beam_search_over_the_table():
  rows = normal(1, 5000, 48, dtype=torch.bfloat16)
  packed = table.pack_rows(rows, 32)
  values = packed.unpack().double()
  s, b = 3, 4
  memory, totals = torch.zeros((s, b, 48), device=DEV), torch.full((s, b), -math.inf, device=DEV)
  totals[:, 0] = 0  # all beams start as one
  tokens = torch.tensor([[7] * b, [77] * b, [777] * b], dtype=torch.int32, device=DEV)
  for _ in range(5):
    plain = 0.5 * memory.double() + 4.0 * rows.double()[tokens.long()]
    scores = plain @ values.T
    want = plain_select(scores, totals, b, True)
    memory, totals, beams, tokens = step(rows, packed, tokens, totals, memory, b)
    assert torch.equal(beams, want[1]) and torch.equal(tokens, want[2])
    assert torch.allclose(totals.double(), want[0], rtol=0, atol=1e-3)
    assert torch.allclose(memory.double(), plain_reorder(plain, beams), rtol=2 ** -20, atol=2 ** -20)


def test_training_the_vectors_of_an_index():
  """Rows that a search found are pulled towards their queries; the changed table is indexed again."""
  base = normal(1, 2000, 32).cpu().numpy()
  index = CuHNSW({"dist_type": "l2", "py_log_level": 1, "c_log_level": 1})
  index.set_data(base)
  index.build()
  queries = normal(2, 50, 32)
  nns, before, _ = index.search_knn(queries.cpu().numpy(), 5, 64)
  rows = torch.from_numpy(base).to(DEV).requires_grad_()
  ids = torch.from_numpy(nns).to(DEV)
  loss = ((table.lookup(rows, ids) - queries[:, None]) ** 2).sum()
  loss.backward()
  exact = torch.zeros((2000, 32), dtype=torch.float64, device=DEV)
  exact.index_add_(0, ids.view(-1).long(), 2 * (rows.detach().double()[ids.long()] - queries.double()[:, None]).view(-1, 32))
  assert torch.allclose(rows.grad.double(), exact, rtol=1e-5, atol=1e-5)
  index.set_data((rows.detach() - 0.1 * rows.grad).cpu().numpy())
  index.build()
  packed = table.pack_rows(rows.detach(), 32)
  bias = -0.5 * (packed.unpack() ** 2).sum(1)
  near, _, found = packed.search(queries, 5, bias)
  exact_order = (queries.double()[:, None] - packed.unpack().double()).pow(2).sum(2).argsort(dim=1, stable=True)[:, :5]
  assert (found == 5).all() and (near.long() == exact_order).float().mean() > 0.99


def test_streams_and_graphs():
  rows = normal(1, 3000, 64, dtype=torch.bfloat16)
  packed = table.pack_rows(rows, 64)
  s, b = 4, 4
  tokens = ids_of(2, s * b, 3000, "uniform", torch.int32).view(s, b)
  memory, totals = normal(3, s, b, 64), normal(4, s, b)
  want = step(rows, packed, tokens, totals, memory, b)
  grad = normal(5, 700, 64)
  ids = ids_of(6, 700, 3000, "zipf")
  want_grad = table.lookup_grad(grad, ids, 3000)
  big = normal(7, 30_000, 64)
  big_ids = ids_of(8, 30_000, 3000, "zipf")
  want_big = table.lookup_grad(big, big_ids, 3000)
  torch.cuda.synchronize()
  side = torch.cuda.Stream()
  with torch.cuda.stream(side):
    got = step(rows, packed, tokens, totals, memory, b)
    got_grad = table.lookup_grad(grad, ids, 3000)
  side.synchronize()
  assert all(torch.equal(x, y) for x, y in zip(got, want)) and torch.equal(got_grad, want_grad)
  # two graphs at the same time on two streams: their workspaces are their own
  graphs, outs, pool = [], [], None
  for _ in range(2):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
      outs.append((step(rows, packed, tokens, totals, memory, b), table.lookup_grad(grad, ids, 3000),
                   table.lookup_grad(big, big_ids, 3000)))
    graphs.append(graph)
  other = torch.cuda.Stream()
  for _ in range(3):
    for state, gradient, big_gradient in outs:
      for t in state:
        t.zero_()
      gradient.zero_()
      big_gradient.zero_()
    torch.cuda.synchronize()
    for graph, stream in zip(graphs, (side, other)):
      with torch.cuda.stream(stream):
        graph.replay()
    torch.cuda.synchronize()
    for state, gradient, big_gradient in outs:
      assert all(torch.equal(x, y) for x, y in zip(state, want))
      assert torch.equal(gradient, want_grad) and torch.equal(big_gradient, want_big)
  # inputs change between replays
  tokens.add_(1).remainder_(3000)
  torch.cuda.synchronize()
  graphs[0].replay()
  torch.cuda.synchronize()
  assert all(torch.equal(x, y) for x, y in zip(outs[0][0], step(rows, packed, tokens, totals, memory, b)))


def test_a_captured_backward_pass():
  rows = normal(1, 500, 32).requires_grad_()
  ids = ids_of(2, 900, 500, "zipf")
  weight = normal(3, 900, 32)
  want, = torch.autograd.grad((table.lookup(rows, ids, 2.0) * weight).sum(), rows)
  side = torch.cuda.Stream()
  with torch.cuda.stream(side):
    torch.autograd.grad((table.lookup(rows, ids, 2.0) * weight).sum(), rows)
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    grad, = torch.autograd.grad((table.lookup(rows, ids, 2.0) * weight).sum(), rows)
  grad.zero_()
  graph.replay()
  torch.cuda.synchronize()
  assert torch.equal(grad, want)


@pytest.mark.skipif(not has_gpu() or torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_tensors_of_another_device():
  for device in ("cuda:1", "cuda:0"):
    rows = normal(1, 100, 40).to(device)
    ids = ids_of(2, 60, 100, "any").to(device)
    assert torch.equal(table.lookup(rows, ids).cpu(), plain_lookup(rows, ids, 1.0).cpu())
    packed = table.pack_rows(rows)
    check = packed.scores(rows[:3])
    assert check.device == rows.device and torch.cuda.current_device() == 0


def test_refusals():
  rows, ids = normal(1, 10, 8), torch.zeros(3, dtype=torch.int64, device=DEV)

  def refused(match, call):
    with pytest.raises(RuntimeError, match=match):
      call()

  refused("float32, float16 or bfloat16", lambda: table.lookup(rows.double(), ids))
  refused("two dimensions", lambda: table.lookup(rows[0], ids))
  refused("int32 or int64", lambda: table.lookup(rows, ids.float()))
  refused("int32 or int64", lambda: table.lookup(rows, ids.to(torch.int16)))
  refused("ids are on cpu", lambda: table.lookup(rows, ids.cpu()))
  grad = normal(2, 3, 8)
  refused("grad must be", lambda: table.lookup_grad(grad.double(), ids, 10))
  refused("grad of shape", lambda: table.lookup_grad(grad[:2], ids, 10))
  refused("grad of shape", lambda: table.lookup_grad(grad.view(1, 3, 8), ids, 10))
  refused("out of range", lambda: table.lookup_grad(grad, ids, -1))
  refused("accumulate needs an out", lambda: table.lookup_grad(grad, ids, 10, accumulate=True))
  refused("out must be a dense", lambda: table.lookup_grad(grad, ids, 10, out=torch.zeros(9, 8, device=DEV)))
  refused("out must be a dense", lambda: table.lookup_grad(grad, ids, 10, out=torch.zeros(8, 10, device=DEV).t()))
  refused("out must be a dense", lambda: table.lookup_grad(grad, ids, 10, out=torch.zeros(10, 8, device=DEV).half()))
  refused("out must be a dense", lambda: table.lookup_grad(grad, ids, 10, out=torch.zeros(10, 8)))
  refused("require a gradient", lambda: table.lookup_grad(grad, ids, 10, out=torch.zeros(10, 8, device=DEV).requires_grad_()))
  for group in (0, 16, 48, 96, 200, -32):
    refused("group must be", lambda g=group: table.pack_rows(rows, g))
  refused("two dimensions", lambda: table.pack_rows(rows[0]))
  refused("without dimensions", lambda: table.pack_rows(rows[:, :0]))
  packed = table.pack_rows(rows, 32)
  refused("codes must be", lambda: table.PackedRows(packed.codes[:, :8], packed.scales, 8, 32))
  refused("codes must be", lambda: table.PackedRows(packed.codes.int(), packed.scales, 8, 32))
  refused("codes must be", lambda: table.PackedRows(torch.zeros(161, dtype=torch.uint8, device=DEV)[1:].view(10, 16), packed.scales, 8, 32))
  refused("scales must be", lambda: table.PackedRows(packed.codes, packed.scales.float(), 8, 32))
  refused("scales must be", lambda: table.PackedRows(packed.codes, packed.scales[:5], 8, 32))
  refused("num_dims", lambda: table.PackedRows(packed.codes[:, :0], packed.scales[:, :0], 0, 32))
  refused("cannot unpack", lambda: packed.unpack(torch.float64))
  refused("queries have 7 dimensions", lambda: packed.scores(rows[:, :7]))
  refused("queries must be", lambda: packed.scores(rows.double()))
  refused("queries are on cpu|CUDA tensor", lambda: packed.scores(rows.cpu()))
  refused("bias must be", lambda: packed.scores(rows, bias=torch.zeros(9, device=DEV)))
  refused("bias must be", lambda: packed.scores(rows, bias=torch.zeros(10, device=DEV).half()))
  for topk in (0, 257, -1):
    refused("topk must be", lambda k=topk: packed.search(rows, k))
  scores = normal(3, 2, 3, 50)
  refused("scores must be", lambda: table.select_beams(scores.double()))
  refused("sequences, beams, vocabulary", lambda: table.select_beams(scores[0]))
  for keep in (0, 257, -1):
    refused("keep must be", lambda k=keep: table.select_beams(scores, keep=k))
  refused("totals must be", lambda: table.select_beams(scores, torch.zeros(2, 2, device=DEV)))
  refused("totals must be", lambda: table.select_beams(scores, torch.zeros(2, 3, device=DEV).double()))
  refused("totals must be", lambda: table.select_beams(scores, torch.zeros(2, 3)))
  beams = torch.zeros((2, 3), dtype=torch.int32, device=DEV)
  refused("beams must be", lambda: table.reorder(scores, beams.long()))
  refused("beams must be", lambda: table.reorder(scores, beams[0]))
  refused("a state must be", lambda: table.reorder(scores.cpu(), beams))
  refused("a state must be", lambda: table.reorder(scores[:, 0, 0], beams))
  refused("states of shapes", lambda: table.reorder([scores, scores[:, :2]], beams))
  refused("states of shapes", lambda: table.reorder(scores[:1], beams))


def test_values_that_are_negated_lazily():
  """torch.conj and .imag of it leave the sign to the next operator."""
  pair = torch.complex(normal(1, 40, 64), normal(2, 40, 64))
  rows = torch.conj(pair).imag
  assert rows.is_neg()
  plain = -pair.imag.contiguous()
  ids = ids_of(3, 90, 40, "outside")
  assert torch.equal(table.lookup(rows, ids), table.lookup(plain, ids))
  assert torch.equal(table.lookup_grad(rows, ids[:40], 50), table.lookup_grad(plain, ids[:40], 50))
  packed, want = table.pack_rows(rows, 32), table.pack_rows(plain, 32)
  assert torch.equal(packed.codes, want.codes) and torch.equal(packed.scales, want.scales)
  assert torch.equal(packed.scores(rows[:5]), packed.scores(plain[:5]))
  got, want = table.select_beams(rows[None], rows[None, :, 0], 9), table.select_beams(plain[None], plain[None, :, 0], 9)
  assert all(torch.equal(x, y) for x, y in zip(got, want))
  states, beams = torch.conj(pair)[None], torch.tensor([[7, -1, 39]], dtype=torch.int32, device=DEV)
  out = table.reorder(states, beams)[0]
  assert torch.equal(out[0], pair[7].conj()) and torch.equal(out[2], pair[39].conj()) and (out[1] == 0).all()
  with pytest.raises(RuntimeError, match="out must be a dense"):
    table.lookup_grad(plain, ids[:40], 40, out=rows)
  with pytest.raises(RuntimeError, match="negated"):
    table.lookup_grad(plain, ids[:40], 40, out=torch._neg_view(torch.zeros((40, 64), device=DEV)))


def test_an_output_that_others_use():
  grad, ids = normal(1, 30, 16), ids_of(2, 30, 20, "uniform")
  out, weight = torch.zeros((20, 16), device=DEV), torch.ones((20, 16), device=DEV, requires_grad=True)
  product = (weight * out).sum()  # keeps `out` for its backward pass
  table.lookup_grad(grad, ids, 20, out=out, accumulate=True)
  with pytest.raises(RuntimeError, match="modified by an inplace operation"):
    product.backward()
  both = torch.zeros((50, 16), device=DEV)
  for part in (both[:20], both[10:30], both[29:49]):
    with pytest.raises(RuntimeError, match="overlap"):
      table.lookup_grad(both[:30], ids, 20, out=part)
  assert (both == 0).all()
  both[:30] = grad
  assert torch.equal(table.lookup_grad(both[:30], ids, 20, out=both[30:]), table.lookup_grad(grad, ids, 20))
  own = torch.arange(20, device=DEV).view(torch.float32).view(20, 2)
  with pytest.raises(RuntimeError, match="overlap"):
    table.lookup_grad(grad[:20, :2], own.view(torch.int64).view(20), 20, out=own)


def test_results_that_memory_does_not_hold():
  rows = torch.zeros((1, 1 << 24), device=DEV)
  with pytest.raises(torch.OutOfMemoryError):
    table.lookup(rows, torch.zeros(1 << 16, dtype=torch.int64, device=DEV))
  assert (table.lookup(rows, torch.zeros(2, dtype=torch.int64, device=DEV)) == 0).all()


def test_a_search_in_parts():
  """More scores than are kept at a time.  All products and sums are whole numbers, exact in any order."""
  n, d, count = 1_200_000, 32, 1000
  codes = torch.randint(0, 256, (n, 16), generator=gen(1), device=DEV).to(torch.uint8)
  packed = table.PackedRows(codes, torch.ones((n, 1), dtype=torch.bfloat16, device=DEV), d, 32)
  queries = torch.randint(-3, 4, (count, d), generator=gen(2), device=DEV).float()
  bias = torch.randint(-5, 6, (n,), generator=gen(3), device=DEV).float()
  assert n * count > 1 << 30
  nns, distances, found = packed.search(queries, 7, bias)
  assert (found == 7).all()
  values = packed.unpack()
  for first in (0, 850, 990):  # (queries of two parts among them)
    scores = queries[first:first + 10].double() @ values.double().T + bias.double()
    order = (-scores).sort(dim=1, stable=True)
    assert torch.equal(nns[first:first + 10].long(), order.indices[:, :7])
    assert torch.equal(distances[first:first + 10].double(), order.values[:, :7])
  whole = [packed.search(queries[i:i + 500], 7, bias) for i in (0, 500)]
  assert torch.equal(nns, torch.cat([w[0] for w in whole])) and torch.equal(distances, torch.cat([w[1] for w in whole]))


def test_threads_on_streams_of_their_own():
  rows = normal(1, 4000, 96, dtype=torch.float16)
  packed = table.pack_rows(rows, 32)
  work = []
  for i in range(4):
    count = (9, 700, 9000, 30_000)[i]
    work.append((ids_of(10 + i, count, 4000, "zipf"), normal(20 + i, count, 96), normal(30 + i, 1 + 3 * i, 96)))
  def run(ids, grad, queries):
    gradient = table.lookup_grad(grad, ids, 4000)
    scores = packed.scores(queries)
    return gradient, scores, *packed.search(queries, 5), *table.select_beams(scores[None], keep=8), table.lookup(rows, ids, 2.0)
  want = [run(*w) for w in work]
  torch.cuda.synchronize()
  wrong, errors = [], []
  def repeat(i):
    try:
      with torch.cuda.stream(torch.cuda.Stream()):
        for _ in range(20):
          got = run(*work[i])
          if not all(torch.equal(x, y) for x, y in zip(got, want[i])):
            wrong.append(i)
    except Exception as e:  # (an exception in a thread would go unseen)
      errors.append(e)
  threads = [threading.Thread(target=repeat, args=(i,)) for i in range(4)]
  for t in threads:
    t.start()
  for t in threads:
    t.join()
  assert not errors and not wrong


def test_a_capture_without_a_call_before_it():
  """The first calls of a process are captured ones."""
  program = """
import torch
from cuhnsw_b200 import table
rows, grad = torch.randn(1000, 256, device="cuda"), torch.randn(20000, 256, device="cuda")
ids, queries = torch.randint(0, 1000, (20000,), device="cuda"), torch.randn(3, 256, device="cuda")
torch.cuda.synchronize()
def run():
  scores = table.pack_rows(rows).scores(queries)
  best = table.select_beams(scores[None], keep=5)
  return table.lookup(rows, ids), table.lookup_grad(grad, ids, 1000), scores, *best, table.reorder(scores[None], best[1])
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
  outs = run()
for t in outs: t.zero_()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(x, y) for x, y in zip(outs, run()))
assert torch.equal(outs[0], rows[ids])
"""
  done = subprocess.run([sys.executable, "-c", program], cwd=Path(__file__).resolve().parent.parent, timeout=300,
                        capture_output=True, text=True)
  assert done.returncode == 0, done.stderr[-2000:]
