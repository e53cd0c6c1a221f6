"""Operators over a table of embeddings, on torch tensors of one GPU.

An index answers with row numbers of a table of learned vectors.  A model that keeps its table in an index also needs,
next to the search:

* the rows themselves (``lookup``) and, in training, the gradient of the table (``lookup_grad``, or autograd);
* the table in 4 bits (``pack_rows``, ``PackedRows``): the scores of all rows, and the exhaustive search over them that an
  index approximates;
* a beam search's step over such scores (``select_beams``) and the beams' states in the new order (``reorder``).

Everything is enqueued on torch's current stream of the tensors' device and not waited for.  Arguments that do not fit raise
``RuntimeError`` before anything is launched; contents (row numbers, beam numbers) are never read on the host, numbers outside
the table stand for empty slots.  Captured into a CUDA graph, the calls allocate from the graph's pool, so that graphs do not share
workspaces.  Only ``lookup`` is differentiable.  The results of the others can be computed from tensors that require a gradient, but
their backward pass raises ``RuntimeError``, as does a call with a forward-mode tangent; row numbers, and rows in 4 bits, are constants.

The checks and the calls of the C ABI are compiled (csrc/table_torch.cpp).  No counterpart in the reference, which keeps its
vectors on the host (cuhnsw/pyhnsw.py:48-58 there).
"""
import torch

try:
  from cuhnsw_b200 import _table
except ImportError as err:
  raise ImportError("cuhnsw_b200/_table.so is missing or does not load: build it with `make -C cuhnsw_b200/csrc` "
                    f"(there is no other path): {err}") from err

MAX_KEEP = 256  # results per sequence of select_beams and PackedRows.search


# -- rows by number --------------------------------------------------------------------------------------------------


class _Lookup(torch.autograd.Function):

  @staticmethod
  def forward(ctx, rows, ids, scale):
    ctx.save_for_backward(ids)
    ctx.save_for_forward(ids)
    ctx.num_rows, ctx.scale = rows.shape[0], scale
    return _table.lookup(rows, ids, scale)

  @staticmethod
  @torch.autograd.function.once_differentiable
  def backward(ctx, grad):
    ids, = ctx.saved_tensors
    return _table.lookup_grad(grad, ids, ctx.num_rows, ctx.scale, None, False), None, None

  @staticmethod
  def jvp(ctx, rows, ids, scale):  # (the tangent of the rows; the others have none)
    return _table.lookup(rows, *ctx.saved_tensors, ctx.scale)


def lookup(rows, ids, scale=1.0):
  """``scale * rows[ids]``, the product in float32 rounded to the rows' type: a tensor of ``ids.shape + (num_dims,)``.

  rows: float32, float16 or bfloat16 ``[num_rows, num_dims]``, rows any distance apart; ids: int32 or int64 of any shape.  An id
  outside ``0 .. num_rows-1`` gives zeros and gets no gradient: the -1 of an empty result slot of a search, or the padding of a
  batch.  Differentiable in ``rows`` (once, backward or forward): see ``lookup_grad``.  The backward pass may be captured into a CUDA graph
  as torch's own may: not while an eager graph of the same leaf lives, which torch answers with an error."""
  if isinstance(rows, torch.Tensor) and (rows.requires_grad and torch.is_grad_enabled() or _table.tangent(rows)):
    return _Lookup.apply(rows, ids, scale)
  return _table.lookup(rows, ids, scale)


def lookup_grad(grad, ids, num_rows, scale=1.0, out=None, accumulate=False):
  """The gradient of ``lookup``'s rows: ``out[r] = scale * sum of grad[t] over all t with ids[t] == r``, for every row.

  grad: ``ids.shape + (num_dims,)``; the sums are taken in fp32 in a fixed order, and rounded
  once: the same call gives the same bits.  out: a dense ``[num_rows, num_dims]`` tensor of grad's type or of float32 (default: a
  new one of grad's type) that overlaps neither grad nor ids; with ``accumulate`` the gradient is added to what it holds, and
  rows without ids keep their bits."""
  return _table.lookup_grad(grad, ids, num_rows, scale, out, accumulate)


# -- rows in 4 bits --------------------------------------------------------------------------------------------------


def pack_rows(rows, group=64):
  """``PackedRows`` of a float32, float16 or bfloat16 ``[num_rows, num_dims]`` tensor: a code of 4 bits per value and a
  bfloat16 scale per ``group`` consecutive dimensions (32, 64 or a multiple of 128): the group's largest magnitude times float32(1/7),
  rounded, and codes that are the values over it, rounded.  A group with a NaN becomes NaN altogether; in one
  with an infinity the infinities stay and the rest becomes NaN."""
  codes, scales = _table.pack(rows, group)
  return PackedRows(codes, scales, rows.shape[1], group)


class PackedRows:
  """Rows in 4 bits: ``codes`` uint8 ``[num_rows, 16 * ceil(num_dims / 32)]`` and ``scales`` bfloat16
  ``[num_rows, ceil(num_dims / group)]``, in the layout that ``cuhnsw_pack4_device`` documents (include/cuhnsw_b200.h).  Both are
  plain tensors: a program may keep them in its own files and make the object of them again."""
  __slots__ = ("codes", "scales", "num_dims", "group")

  def __init__(self, codes, scales, num_dims, group):
    _table.check_packed(codes, scales, num_dims, group)
    self.codes, self.scales, self.num_dims, self.group = codes, scales, int(num_dims), int(group)

  def __repr__(self):
    return f"<PackedRows {self.num_rows} x {self.num_dims}, groups of {self.group}>"

  @property
  def num_rows(self):
    return self.codes.shape[0]

  @property
  def device(self):
    return self.codes.device

  def unpack(self, dtype=torch.float32):
    """The values that the codes stand for, ``[num_rows, num_dims]`` of ``dtype``."""
    return _table.unpack(self.codes, self.scales, self.num_dims, self.group, dtype)

  def scores(self, queries, bias=None):
    """Products of queries with all rows, float32 ``[num_queries, num_rows]``, plus ``bias`` (float32 ``[num_rows]``) if
    given.  queries: float32, float16 or bfloat16 ``[num_queries, num_dims]``.  Made for few queries (a step of a
    decoder, a search): the codes are read once for every 32 of them (8 in float32, fewer if the rows are long)."""
    return _table.scores(self.codes, self.scales, self.num_dims, self.group, queries, bias)

  def search(self, queries, topk, bias=None):
    """``CuHNSW.search_knn``'s triple from an exhaustive search of the dot metric over these rows: (nns int32 ``[Q, topk]``,
    distances float32 ``[Q, topk]``, found_cnt int32 ``[Q]``), rows ascending by (distance, id), empty slots -1 / +inf; CUDA
    tensors.  A distance is minus the score (``scores``; with ``bias`` = -|row|^2 / 2 the order is that of the l2
    metric).  topk up to 256.  The scores of as many queries as fill 4 GB, at least 32, are held at a time."""
    return _table.search(self.codes, self.scales, self.num_dims, self.group, queries, topk, bias)


# -- beam search -----------------------------------------------------------------------------------------------------


def select_beams(scores, totals=None, keep=None, log_softmax=True):
  """The ``keep`` best continuations of every sequence over its beams and the vocabulary: (totals float32, beams int32, ids
  int32), each ``[sequences, keep]``, in descending order of

      totals[s, b] + scores[s, b, v] - log(sum over u of exp(scores[s, b, u]))

  (without the last term if ``log_softmax`` is false); equal ones by smaller beam, then smaller id.  scores: float32, float16 or
  bfloat16 ``[sequences, beams, vocabulary]``; totals: float32 ``[sequences, beams]``, default zeros; keep: 1 to 256, default
  the number of beams.  A total of -inf or NaN is never chosen (a beam that has ended or an id that may not follow is -inf);
  slots that stay empty hold -inf, -1, -1.  Totals are compared in 64 bits.  The log's sum is one of float32 exponentials: within some
  3e-7, and the same for the same scores, so that equal beams are ties; totals of different beams closer than that may come in
  either order."""
  return _table.select_beams(scores, totals, keep, log_softmax)


def reorder(states, beams):
  """The states of the chosen beams: ``out[s, k] = state[s, beams[s, k]]``, zeros where ``beams`` holds -1.

  states: one CUDA tensor ``[sequences, beams, ...]`` or a list of them, of any type; beams: int32 ``[sequences, keep]``, as
  ``select_beams`` gives it.  Returns new dense tensors ``[sequences, keep, ...]``, in a list if a list was given; all of them
  in one launch (per 32).  A view of the part of a cache that is in use, such as ``cache[:, :, :, :length]``, is read where it
  lies."""
  return _table.reorder(states, beams)
