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
workspaces.  No counterpart in the reference, which keeps its vectors on the host (cuhnsw/pyhnsw.py:48-58 there).
"""
import ctypes

import torch

from cuhnsw_b200.cuhnsw_bind import load_library

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_ID_TYPES = {torch.int32: 0, torch.int64: 1}
_MOST_IDS = 2 ** 31 - 2
MAX_KEEP = 256  # results per sequence of select_beams and PackedRows.search


def _require(good, message):
  if not good:
    raise RuntimeError(message)


def _check(rc, name):
  if rc != 0:
    raise RuntimeError(f"{name} failed ({rc})")


def _is_matrix(t, name):
  _require(isinstance(t, torch.Tensor) and t.is_cuda, f"{name} must be a CUDA tensor")
  _require(t.dtype in _TYPES, f"{name} must be float32, float16 or bfloat16, not {t.dtype}")
  _require(t.dim() == 2, f"{name} must have two dimensions, not {t.dim()}")


def _row_major(t):
  """`t` with the values of a row next to each other (a copy where they are not)."""
  return t if t.stride(1) == 1 or t.shape[1] == 1 and t.stride(0) >= 0 else t.contiguous()


def _are_ids(ids, device):
  _require(isinstance(ids, torch.Tensor) and ids.dtype in _ID_TYPES, "ids must be an int32 or int64 tensor")
  _require(ids.device == device, f"ids are on {ids.device}, the rows on {device}")
  _require(ids.numel() <= _MOST_IDS, f"{ids.numel()} ids are too many")
  return ids if ids.is_contiguous() else ids.contiguous()


def _stream(device):
  return torch.cuda.current_stream(device).cuda_stream


class _OnDevice:
  """The tensors' device as the current one for the length of a call."""
  __slots__ = ("device", "before")

  def __init__(self, device):
    self.device = device.index

  def __enter__(self):
    self.before = torch.cuda.current_device()
    if self.before != self.device:
      torch.cuda.set_device(self.device)

  def __exit__(self, *_):
    if self.before != self.device:
      torch.cuda.set_device(self.before)


def _workspace(nbytes, device):
  return torch.empty(max(1, nbytes), dtype=torch.uint8, device=device)


# -- rows by number --------------------------------------------------------------------------------------------------


def _lookup(rows, ids, scale):
  rows = _row_major(rows)
  ids = _are_ids(ids, rows.device)
  out = torch.empty(ids.shape + rows.shape[1:], dtype=rows.dtype, device=rows.device)
  if out.numel():
    with _OnDevice(rows.device):
      _check(load_library().cuhnsw_lookup_device(
        rows.data_ptr(), rows.stride(0), rows.shape[0], rows.shape[1], _TYPES[rows.dtype], ids.data_ptr(),
        _ID_TYPES[ids.dtype], ids.numel(), scale, out.data_ptr(), _stream(rows.device)), "cuhnsw_lookup_device")
  return out


class _Lookup(torch.autograd.Function):

  @staticmethod
  def forward(ctx, rows, ids, scale):
    ctx.save_for_backward(ids)
    ctx.num_rows, ctx.scale = rows.shape[0], scale
    return _lookup(rows, ids, scale)

  @staticmethod
  @torch.autograd.function.once_differentiable
  def backward(ctx, grad):
    ids, = ctx.saved_tensors
    return lookup_grad(grad, ids, ctx.num_rows, ctx.scale), None, None


def lookup(rows, ids, scale=1.0):
  """``scale * rows[ids]``, rounded once to the rows' type: a tensor of ``ids.shape + (num_dims,)``.

  rows: float32, float16 or bfloat16 ``[num_rows, num_dims]``, rows any distance apart; ids: int32 or int64 of any shape.  An id
  outside ``0 .. num_rows-1`` gives zeros and gets no gradient: the -1 of an empty result slot of a search, or the padding of a
  batch.  Differentiable in ``rows`` (once): see ``lookup_grad``."""
  _is_matrix(rows, "rows")
  scale = float(scale)
  if rows.requires_grad and torch.is_grad_enabled():
    return _Lookup.apply(rows, _are_ids(ids, rows.device), scale)
  return _lookup(rows, ids, scale)


def lookup_grad(grad, ids, num_rows, scale=1.0, out=None, accumulate=False):
  """The gradient of ``lookup``'s rows: ``out[r] = scale * sum of grad[t] over all t with ids[t] == r``, for every row.

  grad: ``ids.shape + (num_dims,)``; the sums are taken in fp32 over the ids sorted by row, in a fixed order, and rounded
  once: the same call gives the same bits.  out: a dense ``[num_rows, num_dims]`` tensor of grad's type or of float32 (default: a new one of
  grad's type); with ``accumulate`` the gradient is added to what it holds, and rows without ids keep their bits."""
  _require(isinstance(grad, torch.Tensor) and grad.is_cuda and grad.dtype in _TYPES,
           "grad must be a float32, float16 or bfloat16 CUDA tensor")
  ids = _are_ids(ids, grad.device)
  _require(grad.dim() == ids.dim() + 1 and grad.shape[:-1] == ids.shape,
           f"grad of shape {tuple(grad.shape)} for ids of shape {tuple(ids.shape)}")
  num_rows, dims, device = int(num_rows), grad.shape[-1], grad.device
  _require(0 <= num_rows <= _MOST_IDS, f"{num_rows} rows are out of range")
  grad = _row_major(grad.reshape(ids.numel(), dims))
  if out is None:
    _require(not accumulate, "accumulate needs an out to add to")
    out = torch.empty((num_rows, dims), dtype=grad.dtype, device=device)
  else:
    _require(isinstance(out, torch.Tensor) and out.device == device and out.dtype in (grad.dtype, torch.float32) and
             out.shape == (num_rows, dims) and out.is_contiguous(),
             f"out must be a dense [{num_rows}, {dims}] tensor of {grad.dtype} or float32 on {device}")
    _require(not (out.requires_grad and torch.is_grad_enabled()), "out must not require a gradient")
  if out.numel():
    lib = load_library()
    with _OnDevice(device):
      nbytes = lib.cuhnsw_lookup_grad_workspace(ids.numel(), num_rows, dims)
      _require(nbytes >= 0, f"cuhnsw_lookup_grad_workspace failed ({nbytes})")
      space = _workspace(nbytes, device)
      _check(lib.cuhnsw_lookup_grad_device(
        grad.data_ptr(), grad.stride(0), _TYPES[grad.dtype], ids.data_ptr(), _ID_TYPES[ids.dtype], ids.numel(), num_rows,
        dims, float(scale), out.data_ptr(), _TYPES[out.dtype], int(bool(accumulate)), space.data_ptr(), _stream(device)),
        "cuhnsw_lookup_grad_device")
  return out


# -- rows in 4 bits --------------------------------------------------------------------------------------------------


def _check_group(group):
  group = int(group)
  _require(group in (32, 64) or group >= 128 and group % 128 == 0,
           f"group must be 32, 64 or a multiple of 128, not {group}")
  return group


def pack_rows(rows, group=64):
  """``PackedRows`` of a float32, float16 or bfloat16 ``[num_rows, num_dims]`` tensor of finite values: a code of 4 bits per
  value and a bfloat16 scale per ``group`` consecutive dimensions (32, 64 or a multiple of 128)."""
  _is_matrix(rows, "rows")
  group = _check_group(group)
  rows = _row_major(rows.detach())
  n, d = rows.shape
  _require(d >= 1, "rows without dimensions cannot be packed")
  codes = torch.empty((n, 16 * -(-d // 32)), dtype=torch.uint8, device=rows.device)
  scales = torch.empty((n, -(-d // group)), dtype=torch.bfloat16, device=rows.device)
  with _OnDevice(rows.device):
    _check(load_library().cuhnsw_pack4_device(
      rows.data_ptr(), rows.stride(0), _TYPES[rows.dtype], n, d, group, codes.data_ptr(), scales.data_ptr(),
      _stream(rows.device)), "cuhnsw_pack4_device")
  return PackedRows(codes, scales, d, group)


class PackedRows:
  """Rows in 4 bits: ``codes`` uint8 ``[num_rows, 16 * ceil(num_dims / 32)]`` and ``scales`` bfloat16
  ``[num_rows, ceil(num_dims / group)]``, in the layout that ``cuhnsw_pack4_device`` documents (include/cuhnsw_b200.h).  Both are
  plain tensors: a program may keep them in its own files and make the object of them again."""

  def __init__(self, codes, scales, num_dims, group):
    self.num_dims, self.group = int(num_dims), _check_group(group)
    _require(self.num_dims >= 1, "num_dims must be at least 1")
    _require(isinstance(codes, torch.Tensor) and codes.is_cuda and codes.dtype == torch.uint8 and codes.dim() == 2 and
             codes.shape[1] == 16 * -(-self.num_dims // 32) and codes.is_contiguous() and codes.data_ptr() % 16 == 0,
             f"codes must be a dense, 16-byte aligned uint8 CUDA tensor [num_rows, {16 * -(-self.num_dims // 32)}]")
    _require(isinstance(scales, torch.Tensor) and scales.device == codes.device and scales.dtype == torch.bfloat16 and
             scales.shape == (codes.shape[0], -(-self.num_dims // self.group)) and scales.is_contiguous(),
             f"scales must be a dense bfloat16 tensor [{codes.shape[0]}, {-(-self.num_dims // self.group)}] beside the codes")
    self.codes, self.scales = codes, scales

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
    _require(dtype in _TYPES, f"cannot unpack to {dtype}")
    out = torch.empty((self.num_rows, self.num_dims), dtype=dtype, device=self.device)
    with _OnDevice(self.device):
      _check(load_library().cuhnsw_unpack4_device(
        self.codes.data_ptr(), self.scales.data_ptr(), self.num_rows, self.num_dims, self.group, out.data_ptr(),
        _TYPES[dtype], _stream(self.device)), "cuhnsw_unpack4_device")
    return out

  def scores(self, queries, bias=None):
    """Products of queries with all rows, float32 ``[num_queries, num_rows]``, plus ``bias`` (float32 ``[num_rows]``) if
    given.  queries: float32, float16 or bfloat16 ``[num_queries, num_dims]``.  Made for few queries (a step of a
    decoder, a search): every 32 of them read the codes once."""
    _is_matrix(queries, "queries")
    _require(queries.device == self.device, f"queries are on {queries.device}, the rows on {self.device}")
    _require(queries.shape[1] == self.num_dims,
             f"queries have {queries.shape[1]} dimensions, the rows have {self.num_dims}")
    _require(queries.shape[0] <= 1 << 18, f"{queries.shape[0]} queries are too many")
    queries = _row_major(queries.detach())
    if bias is not None:
      _require(isinstance(bias, torch.Tensor) and bias.device == self.device and bias.dtype == torch.float32 and
               bias.shape == (self.num_rows,), f"bias must be a float32 tensor [{self.num_rows}] beside the rows")
      bias = bias.detach().contiguous()
    out = torch.empty((queries.shape[0], self.num_rows), dtype=torch.float32, device=self.device)
    with _OnDevice(self.device):
      _check(load_library().cuhnsw_scores4_device(
        self.codes.data_ptr(), self.scales.data_ptr(), self.num_rows, self.num_dims, self.group, queries.data_ptr(),
        queries.stride(0), _TYPES[queries.dtype], queries.shape[0], 0 if bias is None else bias.data_ptr(),
        out.data_ptr(), _stream(self.device)), "cuhnsw_scores4_device")
    return out

  def search(self, queries, topk, bias=None):
    """``CuHNSW.search_knn``'s triple from an exhaustive search of the dot metric over these rows: (nns int32 ``[Q, topk]``,
    distances float32 ``[Q, topk]``, found_cnt int32 ``[Q]``), rows ascending by (distance, id), empty slots -1 / +inf; CUDA
    tensors.  A distance is minus the score (``scores``; with ``bias`` = -|row|^2 / 2 the order is that of the l2
    metric).  topk up to 256."""
    scores = self.scores(queries, bias)
    count, device = scores.shape[0], self.device
    topk = _check_keep(topk, "topk")
    nns = torch.empty((count, topk), dtype=torch.int32, device=device)
    distances = torch.empty((count, topk), dtype=torch.float32, device=device)
    found = torch.empty((count,), dtype=torch.int32, device=device)
    if self.num_rows == 0:
      return nns.fill_(-1), distances.fill_(float("inf")), found.zero_()
    _select(scores.unsqueeze(1), None, topk, False, True, distances, None, nns, found)
    return nns, distances, found


# -- beam search -----------------------------------------------------------------------------------------------------


def _check_keep(keep, name):
  keep = int(keep)
  _require(1 <= keep <= MAX_KEEP, f"{name} must be 1 to {MAX_KEEP}, not {keep}")
  return keep


def _select(scores, totals, keep, log_softmax, negate, out_totals, out_beams, out_ids, out_found):
  sequences, beams, vocabulary = scores.shape
  device, lib = scores.device, load_library()
  with _OnDevice(device):
    nbytes = lib.cuhnsw_select_workspace(sequences, beams, vocabulary, keep)
    _require(nbytes >= 0, f"cuhnsw_select_workspace failed ({nbytes})")
    space = _workspace(nbytes, device)
    _check(lib.cuhnsw_select_device(
      scores.data_ptr(), scores.stride(0), scores.stride(1), _TYPES[scores.dtype],
      0 if totals is None else totals.data_ptr(), sequences, beams, vocabulary, keep, int(bool(log_softmax)), int(negate),
      out_totals.data_ptr(), 0 if out_beams is None else out_beams.data_ptr(), out_ids.data_ptr(),
      0 if out_found is None else out_found.data_ptr(), space.data_ptr(), _stream(device)), "cuhnsw_select_device")


def select_beams(scores, totals=None, keep=None, log_softmax=True):
  """The ``keep`` best continuations of every sequence over its beams and the vocabulary: (totals float32, beams int32, ids
  int32), each ``[sequences, keep]``, in descending order of

      totals[s, b] + scores[s, b, v] - log(sum over u of exp(scores[s, b, u]))

  (without the last term if ``log_softmax`` is false); equal ones by smaller beam, then smaller id.  scores: float32, float16 or
  bfloat16 ``[sequences, beams, vocabulary]``; totals: float32 ``[sequences, beams]``, default zeros; keep: 1 to 256, default
  the number of beams.  A total of -inf or NaN is never chosen (a beam that has ended or an id that may not follow is -inf);
  slots that stay empty hold -inf, -1, -1."""
  _require(isinstance(scores, torch.Tensor) and scores.is_cuda and scores.dtype in _TYPES,
           "scores must be a float32, float16 or bfloat16 CUDA tensor")
  _require(scores.dim() == 3, f"scores must be [sequences, beams, vocabulary], not {scores.dim()}-dimensional")
  sequences, beams, vocabulary = scores.shape
  keep = _check_keep(beams if keep is None else keep, "keep")
  _require(beams <= 16384, f"{beams} beams are too many")
  device = scores.device
  scores = scores.detach()
  if scores.stride(2) != 1 and vocabulary > 1:
    scores = scores.contiguous()
  if totals is not None:
    _require(isinstance(totals, torch.Tensor) and totals.device == device and totals.dtype == torch.float32 and
             totals.shape == (sequences, beams), f"totals must be a float32 tensor [{sequences}, {beams}] beside the scores")
    totals = totals.detach().contiguous()
  out = (torch.empty((sequences, keep), dtype=torch.float32, device=device),
         torch.empty((sequences, keep), dtype=torch.int32, device=device),
         torch.empty((sequences, keep), dtype=torch.int32, device=device))
  if scores.numel() == 0:
    return out[0].fill_(float("-inf")), out[1].fill_(-1), out[2].fill_(-1)
  _select(scores, totals, keep, log_softmax, False, *out, None)
  return out


class _State(ctypes.Structure):
  _fields_ = [("src", ctypes.c_void_p), ("dst", ctypes.c_void_p), ("seq_stride", ctypes.c_int64),
              ("beam_stride", ctypes.c_int64), ("segment_stride", ctypes.c_int64), ("segments", ctypes.c_int64),
              ("bytes", ctypes.c_int64)]


def _pieces(state):
  """(segments, values between them, values of each) of a state's rows, or None if they are not evenly spaced pieces."""
  each, segments, between = 1, 1, 0
  for size, stride in zip(reversed(state.shape[2:]), reversed(state.stride()[2:])):
    if size == 1:
      continue
    if segments == 1 and stride == each:
      each *= size
    elif segments == 1:
      segments, between = size, stride
    elif stride == segments * between:
      segments *= size
    else:
      return None
  return segments, between, each


def reorder(states, beams):
  """The states of the chosen beams: ``out[s, k] = state[s, beams[s, k]]``, zeros where ``beams`` holds -1.

  states: one CUDA tensor ``[sequences, beams, ...]`` or a list of them, of any type; beams: int32 ``[sequences, keep]``, as
  ``select_beams`` gives it.  Returns new dense tensors ``[sequences, keep, ...]``, in a list if a list was given; all of them
  in one launch (per 32).  A view of the part of a cache that is in use, such as ``cache[:, :, :, :length]``, is read where it
  lies."""
  several = isinstance(states, (list, tuple))
  inputs = list(states) if several else [states]
  _require(isinstance(beams, torch.Tensor) and beams.is_cuda and beams.dtype == torch.int32 and beams.dim() == 2,
           "beams must be an int32 CUDA tensor [sequences, keep]")
  beams = beams.contiguous()
  sequences, keep = beams.shape
  outs, table, kept = [], (_State * max(1, len(inputs)))(), []
  for i, state in enumerate(inputs):
    _require(isinstance(state, torch.Tensor) and state.device == beams.device and state.dim() >= 2,
             f"a state must be a tensor [sequences, beams, ...] on {beams.device}")
    _require(state.shape[:2] == (sequences, inputs[0].shape[1]),
             f"states of shapes {tuple(inputs[0].shape)} and {tuple(state.shape)} for {sequences} sequences")
    state = state.detach()
    pieces = _pieces(state)
    if pieces is None:
      state = state.contiguous()
      pieces = _pieces(state)
    kept.append(state)
    size = state.element_size()
    out = torch.empty((sequences, keep) + tuple(state.shape[2:]), dtype=state.dtype, device=state.device)
    segments, between, each = pieces
    empty = out.numel() == 0
    table[i] = _State(state.data_ptr(), out.data_ptr(), state.stride(0) * size, state.stride(1) * size, between * size,
                      0 if empty else segments, 0 if empty else each * size)
    outs.append(out)
  if inputs:
    with _OnDevice(beams.device):
      _check(load_library().cuhnsw_reorder_device(table, len(inputs), beams.data_ptr(), sequences, inputs[0].shape[1], keep,
                                                  _stream(beams.device)), "cuhnsw_reorder_device")
  return outs if several else outs[0]
