"""The operators next to the index, as timed cases: rows of a table of embeddings looked up and their gradient, rows
packed into 4 bits, scores of all packed rows, and a beam search's selection over those scores.

A case is a dict of plain values; ``kind`` says which operator it is:

  kind    "lookup"  ``table.lookup``: rows of a table by number, scaled
          "grad"    ``table.lookup_grad``: the gradient of the whole table
          "pack"    ``table.pack_rows`` and back (``PackedRows.unpack``): the values that the 4 bits stand for
          "scores"  ``PackedRows.scores``: products of queries with all rows
          "beams"   ``table.select_beams`` and ``table.reorder``: the best continuations of all beams of a sequence
                    and their states put in that order
  n, d    rows of the table and their dimensions;  dtype  type of the rows, gradients, queries or scores
  tokens  numbers to look up;  ids  "zipf" (words of a text: the first rows are most of them) or "found" (results of
          a search: uniform, one slot in ten empty);  scale  the factor of a lookup
  group   dimensions that share a scale;  q  queries;  bias  whether a value per row is added
  s, b, k  sequences, beams per sequence and continuations kept of each sequence (n: the vocabulary);  norm  whether the
          scores are normalised over the vocabulary first;  heads, length  the states' shape: heads x length x 64
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZES = {"f32": 4, "f16": 2, "bf16": 2}
_HEAD = 64  # width of a head of the beams' states
_CHUNK = 1 << 26  # values made or unpacked at a time


def listed():
  return [
    # one step of eight sequences: each one's last token (latency)
    dict(name="lookup, 8 tokens", kind="lookup", dtype="bf16", n=32_000, d=2048, tokens=8, ids="zipf", scale=45.25),
    # the rows that a batch of searches found in the benchmark's corpus, 10 000 queries x 10
    dict(name="lookup, rows found", kind="lookup", dtype="f32", n=1_183_514, d=50, tokens=100_000, ids="found", scale=1.0),
    # a step's tokens of a small model in training (latency; most rows are not touched)
    dict(name="grad, 511 tokens", kind="grad", dtype="f32", n=32_000, d=256, tokens=511, ids="zipf", scale=16.0),
    # a training batch of 16 sequences of 1024 tokens against a large vocabulary
    dict(name="grad, 16384 tokens", kind="grad", dtype="bf16", n=131_072, d=4096, tokens=16_384, ids="zipf", scale=64.0),
    # fine-tuning the indexed vectors themselves on lists of neighbours: narrow rows, many of them
    dict(name="grad, 1000003 rows found", kind="grad", dtype="f32", n=1_183_514, d=50, tokens=1_000_003, ids="found", scale=1.0),
    # the benchmark's corpus of short vectors, packed and unpacked
    dict(name="pack, 50-d", kind="pack", dtype="f32", n=1_183_514, d=50, group=32),
    # a model's output table
    dict(name="pack, 2048-d", kind="pack", dtype="bf16", n=50_000, d=2048, group=128),
    # one query against a small table (latency)
    dict(name="scores, one query", kind="scores", dtype="bf16", n=32_000, d=1024, group=32, q=1, bias=False),
    # a few full-precision queries against the benchmark's corpus: exhaustive search, ragged rows
    dict(name="scores, 7 queries, 50-d", kind="scores", dtype="f32", n=1_183_514, d=50, group=64, q=7, bias=True),
    # a decoding step of 32 beams: a large vocabulary's scores
    dict(name="scores, 32 queries", kind="scores", dtype="f16", n=131_072, d=4096, group=128, q=32, bias=False),
    # one sequence of four beams (latency)
    dict(name="beams, 1 x 4", kind="beams", dtype="bf16", n=32_000, s=1, b=4, k=8, norm=True, heads=2, length=129),
    # a server's step: 32 sequences of eight beams, large vocabulary, states of 512 tokens
    dict(name="beams, 32 x 8", kind="beams", dtype="f32", n=131_072, s=32, b=8, k=8, norm=True, heads=8, length=512),
  ]


def _log_int(rng, low, high):
  return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
  kind = rng.choice(["lookup", "grad", "pack", "scores", "beams"])
  dtype = rng.choice(["f32", "f16", "bf16"])
  if kind == "beams":
    s, n = _log_int(rng, 1, 64), _log_int(rng, 1000, 151_000)
    b = _log_int(rng, 1, min(16, max(1, (1 << 25) // (s * n))))
    return dict(kind=kind, dtype=dtype, n=n, s=s, b=b, k=rng.choice([b, 2 * b, rng.randint(1, 64)]), norm=rng.random() < 0.7,
                heads=rng.randint(1, 8), length=_log_int(rng, 1, max(1, min(512, 16_384 // (s * b)))))
  if kind == "lookup":
    d, tokens = _log_int(rng, 8, 8192), _log_int(rng, 1, 131_072)
    n = _log_int(rng, 1000, min(1_200_000, (1 << 28) // d))
    return dict(kind=kind, dtype=dtype, n=n, d=d, tokens=max(1, min(tokens, (1 << 26) // d)), ids=rng.choice(["zipf", "found"]),
                scale=rng.choice([1.0, math.sqrt(d)]))
  if kind == "grad":
    d, tokens = _log_int(rng, 8, 8192), _log_int(rng, 1, 1_000_000)
    n = _log_int(rng, 1000, min(1_200_000, (1 << 28) // d))
    return dict(kind=kind, dtype=dtype, n=n, d=d, tokens=max(1, min(tokens, (1 << 26) // d)), ids=rng.choice(["zipf", "found"]),
                scale=rng.choice([1.0, math.sqrt(d)]))
  d = _log_int(rng, 8, 8192)
  group = rng.choice([32, 64, 128, 256])
  if kind == "pack":
    return dict(kind=kind, dtype=dtype, n=_log_int(rng, 1000, min(1_200_000, (1 << 26) // d)), d=d, group=group)
  n = _log_int(rng, 1000, min(1_200_000, (1 << 28) // d))
  return dict(kind=kind, dtype=dtype, n=n, d=d, group=group, q=_log_int(rng, 1, max(1, min(32, (1 << 26) // n))),
              bias=rng.random() < 0.5)


def _row_words(d):
  """(dimension of every nibble of a row's 32-bit words, lowest nibble first; a row's words): blocks of 32 dimensions, four
  to a part of the row (its last part has what is left); a part's word t*m + j of its m blocks holds dimensions 8*t .. 8*t + 7
  of block j, the even ones in nibbles 0 to 3, the odd ones in 4 to 7."""
  blocks = -(-d // 32)
  dims = []
  for first in range(0, blocks, 4):
    m = min(4, blocks - first)
    for t in range(4):
      for j in range(m):
        at = 32 * (first + j) + 8 * t
        dims += [at, at + 2, at + 4, at + 6, at + 1, at + 3, at + 5, at + 7]
  return np.array(dims, np.int64), 4 * blocks


def _quantise(rows, group):
  """Codes 0..15 as int64 [n, d] and their scales, bfloat16 [n, groups], of float32 rows."""
  n, d = rows.shape
  groups = -(-d // group)
  padded = torch.nn.functional.pad(rows, (0, groups * group - d)).view(n, groups, group)
  scales = (padded.abs().amax(2) / 7).to(torch.bfloat16)
  step = scales.float().unsqueeze(2)
  codes = torch.where(step > 0, (padded / step).round().clamp(-8, 7), torch.zeros_like(padded)) + 8
  return codes.view(n, groups * group)[:, :d].to(torch.int64), scales


def prepare(case, seed):
  dev = torch.device("cuda")
  gen = torch.Generator(device=dev).manual_seed(seed)
  kind, dtype, n = case["kind"], _DTYPES[case["dtype"]], case["n"]
  state = dict(case, group=case.get("group", 0), seed=seed)

  def normal(*shape, sigma=1.0, to=dtype):
    return torch.randn(shape, generator=gen, device=dev).mul_(sigma).to(to)

  def uniform(*shape):
    return torch.rand(shape, generator=gen, device=dev)

  if kind in ("lookup", "grad"):
    tokens, d = case["tokens"], case["d"]
    if case["ids"] == "zipf":
      # the r-th row about 1/r as often as the first, the rows in no order
      rank = torch.exp(uniform(tokens).double() * math.log(n)).long().clamp_(1, n) - 1
      ids = torch.randperm(n, generator=gen, device=dev)[rank]
    else:
      ids = torch.randint(0, n, (tokens,), generator=gen, device=dev).to(torch.int32)
      ids = torch.where(uniform(tokens) < 0.1, torch.full_like(ids, -1), ids)
    state["numbers"] = ids
    state["values"] = normal(n, d, sigma=1 / math.sqrt(d)) if kind == "lookup" else normal(tokens, d, sigma=1e-2)
  elif kind == "pack":
    state["values"] = normal(n, case["d"], sigma=1 / math.sqrt(case["d"]))
  elif kind == "scores":
    d, group = case["d"], case["group"]
    dims, words = _row_words(d)
    dims = torch.from_numpy(dims).to(dev)
    codes = torch.empty((n, 4 * words), dtype=torch.uint8, device=dev)
    scales = torch.empty((n, -(-d // group)), dtype=torch.bfloat16, device=dev)
    step = max(1, _CHUNK // (32 * -(-d // 32)))
    for lo in range(0, n, step):
      values, scales[lo:lo + step] = _quantise(normal(min(step, n - lo), d, sigma=1 / math.sqrt(d), to=torch.float32), group)
      values = torch.nn.functional.pad(values, (0, 8 * words - d), value=8)[:, dims].view(-1, 2)
      codes[lo:lo + step] = (values[:, 0] + 16 * values[:, 1]).to(torch.uint8).view(-1, 4 * words)
    state.update(codes=codes, scales=scales, queries=normal(case["q"], d), dims=dims)
    state["offset"] = normal(n, to=torch.float32) if case["bias"] else None
  else:
    s, b = case["s"], case["b"]
    logits = normal(s, b, n, sigma=3.0)
    logits.masked_fill_(uniform(s, b, n) < 0.01, -math.inf)  # tokens that may not follow
    state["logits"] = logits
    totals = -20 * uniform(s, b)
    state["totals"] = totals.masked_fill_(uniform(s, b) < 0.05, -math.inf)  # beams that have ended
    state["tokens"] = torch.randint(0, n, (s, b, case["length"]), generator=gen, device=dev).to(torch.int32)
    state["cache"] = normal(s, b, case["heads"], case["length"], _HEAD, to=torch.bfloat16)
  return state


def _own_run(state):
  from cuhnsw_b200 import table
  kind = state["kind"]
  if kind == "lookup":
    return table.lookup(state["values"], state["numbers"], state["scale"])
  if kind == "grad":
    return table.lookup_grad(state["values"], state["numbers"], state["n"], state["scale"])
  if kind == "pack":
    return table.pack_rows(state["values"], state["group"]).unpack()
  if kind == "scores":
    rows = table.PackedRows(state["codes"], state["scales"], state["d"], state["group"])
    return rows.scores(state["queries"], bias=state["offset"])
  totals, beams, ids = table.select_beams(state["logits"], state["totals"], state["k"], log_softmax=state["norm"])
  tokens, cache = table.reorder([state["tokens"], state["cache"]], beams)
  return {"totals": totals, "beams": beams, "ids": ids, "tokens": tokens, "cache": cache}


def run(state):
  if own:
    return _own_run(state)
  kind = state["kind"]
  if kind == "lookup":
    rows, ids = state["values"], state["numbers"].long()
    there = (ids >= 0) & (ids < rows.shape[0])
    out = rows[ids.clamp(0, rows.shape[0] - 1)].float() * state["scale"]
    return torch.where(there[:, None], out, torch.zeros_like(out)).to(rows.dtype)
  if kind == "grad":
    grad, ids, n = state["values"], state["numbers"].long(), state["n"]
    there = (ids >= 0) & (ids < n)
    out = torch.zeros((n, grad.shape[1]), device=grad.device)
    values = torch.where(there[:, None], grad.float(), torch.zeros((), device=grad.device))
    out.index_add_(0, ids.clamp(0, n - 1), values)
    return (out * state["scale"]).to(grad.dtype)
  if kind == "pack":
    codes, scales = _quantise(state["values"].float(), state["group"])
    return (codes - 8).float() * scales.float().repeat_interleave(state["group"], 1)[:, :codes.shape[1]]
  if kind == "scores":
    words = state["codes"].view(torch.int32)
    shifts = torch.arange(0, 32, 4, dtype=torch.int32, device=words.device)
    values = ((words.unsqueeze(2) >> shifts) & 15).view(words.shape[0], -1)
    place = torch.empty_like(state["dims"])
    place[state["dims"]] = torch.arange(len(place), device=place.device)
    rows = (values[:, place[:state["d"]]] - 8).float()
    rows *= state["scales"].float().repeat_interleave(state["group"], 1)[:, :state["d"]]
    out = state["queries"].float() @ rows.T
    return out if state["offset"] is None else out + state["offset"]
  # 64 bits: near a border the order of two totals would depend on the rounding of either
  totals = state["logits"].double()
  if state["norm"]:
    top = totals.amax(2, keepdim=True).clamp(min=torch.finfo(torch.float64).min)
    totals = totals - (top + (totals - top).exp().sum(2, keepdim=True).log())
  totals = (state["totals"].double().unsqueeze(2) + totals).view(state["s"], -1)
  totals = torch.where(totals.isnan(), -math.inf, totals)
  k = min(state["k"], totals.shape[1])
  border = totals.topk(k, 1).values[:, -1:]
  # of the totals at the border the lowest indices
  place = torch.arange(totals.shape[1], device=totals.device)
  rank = torch.where(totals > border, 2 * len(place) - place, torch.where(totals == border, len(place) - place, 0))
  best = rank.topk(k, 1).indices.sort(1).values
  values, order = totals.gather(1, best).sort(dim=1, descending=True, stable=True)
  best = best.gather(1, order)
  lost = values == -math.inf
  pad = (0, state["k"] - k)
  values = torch.nn.functional.pad(values, pad, value=-math.inf).float()
  beams = torch.nn.functional.pad(torch.where(lost, -1, best // state["n"]), pad, value=-1).to(torch.int32)
  ids = torch.nn.functional.pad(torch.where(lost, -1, best % state["n"]), pad, value=-1).to(torch.int32)
  # an empty slot's state is zeros
  at = beams.long().clamp(min=0)
  seq = torch.arange(state["s"], device=at.device)[:, None]
  there = beams >= 0
  tokens = state["tokens"][seq, at] * there[:, :, None]
  cache = torch.where(there[:, :, None, None, None], state["cache"][seq, at], torch.zeros((), dtype=torch.bfloat16, device=at.device))
  return {"totals": values, "beams": beams, "ids": ids, "tokens": tokens.to(torch.int32), "cache": cache}


def work(case):
  kind, n, size = case["kind"], case["n"], _SIZES[case["dtype"]]
  if kind in ("lookup", "grad"):
    tokens, d = case["tokens"], case["d"]
    numbers = tokens * (8 if case["ids"] == "zipf" else 4)
    if kind == "grad":
      live = tokens if case["ids"] == "zipf" else 0.9 * tokens
      return {"bytes": numbers + (live + n) * d * size, "flops": live * d + n * d}
    # a row that is asked for twice is read once
    if case["ids"] == "zipf":
      share = [math.log((r + 1) / r) / math.log(n) for r in range(1, min(n, 2000))]
      rest = 1 - sum(share)
      distinct = sum(1 - (1 - p) ** tokens for p in share)
      left = max(1, n - len(share))
      distinct += min(left, tokens * rest)
    else:
      distinct = n * (1 - (1 - 1 / n) ** (0.9 * tokens))
    return {"bytes": numbers + (distinct + tokens) * d * size, "flops": tokens * d}
  if kind == "beams":
    s, b, k = case["s"], case["b"], case["k"]
    state = case["length"] * (4 + 2 * _HEAD * case["heads"])
    return {"bytes": s * b * (n * size + 4) + 12 * s * k + s * (min(b, k) + k) * state, "flops": 3 * s * b * n}
  d = case["d"]
  packed = n * (d / 2 + 2 * -(-d // case["group"]))
  if kind == "pack":
    return {"bytes": n * d * (size + 4) + 2 * packed, "flops": 4 * n * d}
  q = case["q"]
  return {"bytes": packed + q * d * size + 4 * q * n + (4 * n if case["bias"] else 0), "flops": 2 * q * n * d}


def exact(case, seed):
  if "q" in case and case["q"] * case["n"] * case["d"] > 1 << 36:
    return None
  state = prepare(case, seed)
  kind, n = case["kind"], case["n"]
  if kind == "lookup":
    table = torch.cat([state["values"], torch.zeros_like(state["values"][:1])]).double()
    ids = state["numbers"].long()
    ids = torch.where((ids < 0) | (ids >= n), n, ids)
    return torch.index_select(table, 0, ids).mul_(case["scale"])
  if kind == "grad":
    ids = state["numbers"].long()
    keep = ((ids >= 0) & (ids < n)).nonzero().view(-1)
    order = keep[ids[keep].argsort(stable=True)]
    sums = torch.zeros((n, case["d"]), dtype=torch.float64, device=ids.device)
    rows, counts = ids[order].unique_consecutive(return_counts=True)
    at = torch.repeat_interleave(rows, counts)
    step = max(1, _CHUNK // case["d"])
    for lo in range(0, len(order), step):
      sums.index_put_((at[lo:lo + step],), state["values"][order[lo:lo + step]].double(), accumulate=True)
    return sums.mul_(case["scale"])
  if kind == "pack":
    values, group, d = state["values"], case["group"], case["d"]
    out = torch.empty(values.shape, dtype=torch.float64, device=values.device)
    for first in range(0, d, group):
      part = values[:, first:first + group].double()
      # a scale is a bfloat16 by definition, of the quotient in float32
      scale = (part.abs().amax(1, keepdim=True).float() / 7).to(torch.bfloat16).double()
      code = torch.round(part / scale.where(scale > 0, torch.ones_like(scale))).clamp(-8, 7)
      out[:, first:first + group] = code * scale
    return out
  if kind == "scores":
    d, group = case["d"], case["group"]
    out = torch.empty((case["q"], n), dtype=torch.float64, device="cuda")
    queries = state["queries"].double()
    words = state["codes"].shape[1] // 4
    dims, wanted = state["dims"].view(words, 8), 32 * -(-d // 32)
    step = max(1, _CHUNK // wanted)
    for lo in range(0, n, step):
      part = state["codes"][lo:lo + step].view(-1, words, 4)
      rows = torch.zeros((len(part), wanted), dtype=torch.float64, device="cuda")
      for byte in range(4):
        rows[:, dims[:, 2 * byte]] = (part[:, :, byte] & 15).double() - 8
        rows[:, dims[:, 2 * byte + 1]] = (part[:, :, byte] >> 4).double() - 8
      for g, first in enumerate(range(0, d, group)):
        rows[:, first:first + group] *= state["scales"][lo:lo + step, g:g + 1].double()
      out[:, lo:lo + step] = queries @ rows[:, :d].T
    if state["offset"] is not None:
      out += state["offset"].double()
    return out
  s, b, k = case["s"], case["b"], case["k"]
  outs = {"totals": torch.full((s, k), -math.inf, dtype=torch.float64, device="cuda"),
          "beams": torch.full((s, k), -1, dtype=torch.int32, device="cuda"),
          "ids": torch.full((s, k), -1, dtype=torch.int32, device="cuda"),
          "tokens": torch.zeros((s, k) + state["tokens"].shape[2:], dtype=torch.int32, device="cuda"),
          "cache": torch.zeros((s, k) + state["cache"].shape[2:], dtype=torch.float64, device="cuda")}
  for i in range(s):
    row = state["logits"][i].double()
    if case["norm"]:
      row = row - torch.logsumexp(row, 1, keepdim=True)
    row = (row + state["totals"][i].double()[:, None]).view(-1)
    row = torch.where(row > -math.inf, row, -math.inf)
    value, at = row.sort(dim=0, descending=True, stable=True)
    count = min(k, int((value > -math.inf).sum()))
    outs["totals"][i, :count] = value[:count]
    outs["beams"][i, :count] = (at[:count] // n).int()
    outs["ids"][i, :count] = (at[:count] % n).int()
    outs["tokens"][i, :count] = state["tokens"][i][at[:count] // n]
    outs["cache"][i, :count] = state["cache"][i][at[:count] // n].double()
  return outs
