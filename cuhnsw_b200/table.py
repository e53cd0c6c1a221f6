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
import functools

import torch

from cuhnsw_b200.cuhnsw_bind import load_library

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_ID_TYPES = {torch.int32: 0, torch.int64: 1}
_MOST_IDS = 2 ** 31 - 2
MAX_KEEP = 256  # results per sequence of select_beams and PackedRows.search

# (A call of a few microseconds on the GPU should not take more than that on the host: checks build their messages only when
# they fail, and nothing is asked twice.)


def _refuse(message):
  raise RuntimeError(message)


def _is_matrix(t, name):
  if not isinstance(t, torch.Tensor) or not t.is_cuda:
    _refuse(f"{name} must be a CUDA tensor")
  if t.dtype not in _TYPES:
    _refuse(f"{name} must be float32, float16 or bfloat16, not {t.dtype}")
  if t.dim() != 2:
    _refuse(f"{name} must have two dimensions, not {t.dim()}")


def _row_major(t):
  """`t` with the values of a row next to each other (a copy where they are not)."""
  return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _are_ids(ids, device):
  if not isinstance(ids, torch.Tensor) or ids.dtype not in _ID_TYPES:
    _refuse("ids must be an int32 or int64 tensor")
  if ids.device != device:
    _refuse(f"ids are on {ids.device}, the rows on {device}")
  if ids.numel() > _MOST_IDS:
    _refuse(f"{ids.numel()} ids are too many")
  return ids if ids.is_contiguous() else ids.contiguous()


def _run(name, device, *args):
  """One entry point of the library on the current stream of `device`, which is the current device meanwhile."""
  index = device.index
  before = torch.cuda.current_device()
  entry = getattr(load_library(), name)
  if before == index:
    rc = entry(*args, _stream_of(index))
  else:
    with torch.cuda.device(index):
      rc = entry(*args, _stream_of(index))
  if rc != 0:
    _refuse(f"{name} failed ({rc})")


try:
  _stream_of = torch._C._cuda_getCurrentRawStream  # (a fraction of the time of the public call)
except AttributeError:
  def _stream_of(index):
    return torch.cuda.current_stream(index).cuda_stream


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(name, *sizes):
  nbytes = getattr(load_library(), name)(*sizes)
  if nbytes < 0:
    _refuse(f"{name} failed ({nbytes})")
  return max(1, nbytes)


# -- rows by number --------------------------------------------------------------------------------------------------


def _lookup(rows, ids, scale):
  device, (num_rows, dims) = rows.device, rows.shape
  rows, ids = _row_major(rows), _are_ids(ids, device)
  out = rows.new_empty(ids.shape + (dims,))
  count = ids.numel()
  if count and dims:
    _run("cuhnsw_lookup_device", device, rows.data_ptr(), rows.stride(0), num_rows, dims, _TYPES[rows.dtype], ids.data_ptr(),
         _ID_TYPES[ids.dtype], count, scale, out.data_ptr())
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
  if not isinstance(grad, torch.Tensor) or not grad.is_cuda or grad.dtype not in _TYPES:
    _refuse("grad must be a float32, float16 or bfloat16 CUDA tensor")
  device, dtype, num_rows = grad.device, grad.dtype, int(num_rows)
  ids = _are_ids(ids, device)
  if grad.dim() != ids.dim() + 1 or grad.shape[:-1] != ids.shape:
    _refuse(f"grad of shape {tuple(grad.shape)} for ids of shape {tuple(ids.shape)}")
  if not 0 <= num_rows <= _MOST_IDS:
    _refuse(f"{num_rows} rows are out of range")
  count, dims = ids.numel(), grad.shape[-1]
  grad = _row_major(grad if grad.dim() == 2 else grad.reshape(count, dims))
  if out is None:
    if accumulate:
      _refuse("accumulate needs an out to add to")
    out = grad.new_empty((num_rows, dims))
  elif not (isinstance(out, torch.Tensor) and out.device == device and out.dtype in (dtype, torch.float32) and
            out.shape == (num_rows, dims) and out.is_contiguous()):
    _refuse(f"out must be a dense [{num_rows}, {dims}] tensor of {dtype} or float32 on {device}")
  elif out.requires_grad and torch.is_grad_enabled():
    _refuse("out must not require a gradient")
  if num_rows and dims:
    space = torch.empty(_workspace_bytes("cuhnsw_lookup_grad_workspace", count, num_rows, dims), dtype=torch.uint8,
                        device=device)
    _run("cuhnsw_lookup_grad_device", device, grad.data_ptr(), grad.stride(0), _TYPES[dtype], ids.data_ptr(),
         _ID_TYPES[ids.dtype], count, num_rows, dims, scale, out.data_ptr(), _TYPES[out.dtype], 1 if accumulate else 0,
         space.data_ptr())
  return out


# -- rows in 4 bits --------------------------------------------------------------------------------------------------


def _check_group(group):
  group = int(group)
  if group not in (32, 64) and (group < 128 or group % 128 != 0):
    _refuse(f"group must be 32, 64 or a multiple of 128, not {group}")
  return group


def pack_rows(rows, group=64):
  """``PackedRows`` of a float32, float16 or bfloat16 ``[num_rows, num_dims]`` tensor of finite values: a code of 4 bits per
  value and a bfloat16 scale per ``group`` consecutive dimensions (32, 64 or a multiple of 128)."""
  _is_matrix(rows, "rows")
  group = _check_group(group)
  rows = _row_major(rows)
  device, (n, d) = rows.device, rows.shape
  if d < 1:
    _refuse("rows without dimensions cannot be packed")
  codes = torch.empty((n, 16 * -(-d // 32)), dtype=torch.uint8, device=device)
  scales = torch.empty((n, -(-d // group)), dtype=torch.bfloat16, device=device)
  _run("cuhnsw_pack4_device", device, rows.data_ptr(), rows.stride(0), _TYPES[rows.dtype], n, d, group, codes.data_ptr(),
       scales.data_ptr())
  return PackedRows(codes, scales, d, group)


class PackedRows:
  """Rows in 4 bits: ``codes`` uint8 ``[num_rows, 16 * ceil(num_dims / 32)]`` and ``scales`` bfloat16
  ``[num_rows, ceil(num_dims / group)]``, in the layout that ``cuhnsw_pack4_device`` documents (include/cuhnsw_b200.h).  Both are
  plain tensors: a program may keep them in its own files and make the object of them again."""
  __slots__ = ("codes", "scales", "num_rows", "num_dims", "group", "device")

  def __init__(self, codes, scales, num_dims, group):
    num_dims, group = int(num_dims), _check_group(group)
    if num_dims < 1:
      _refuse("num_dims must be at least 1")
    width, groups = 16 * -(-num_dims // 32), -(-num_dims // group)
    if not (isinstance(codes, torch.Tensor) and codes.is_cuda and codes.dtype == torch.uint8 and codes.dim() == 2 and
            codes.shape[1] == width and codes.is_contiguous() and codes.data_ptr() % 16 == 0):
      _refuse(f"codes must be a dense, 16-byte aligned uint8 CUDA tensor [num_rows, {width}]")
    if not (isinstance(scales, torch.Tensor) and scales.device == codes.device and scales.dtype == torch.bfloat16 and
            scales.shape == (codes.shape[0], groups) and scales.is_contiguous()):
      _refuse(f"scales must be a dense bfloat16 tensor [{codes.shape[0]}, {groups}] beside the codes")
    self.codes, self.scales, self.num_rows, self.device = codes, scales, codes.shape[0], codes.device
    self.num_dims, self.group = num_dims, group

  def __repr__(self):
    return f"<PackedRows {self.num_rows} x {self.num_dims}, groups of {self.group}>"

  def unpack(self, dtype=torch.float32):
    """The values that the codes stand for, ``[num_rows, num_dims]`` of ``dtype``."""
    if dtype not in _TYPES:
      _refuse(f"cannot unpack to {dtype}")
    out = torch.empty((self.num_rows, self.num_dims), dtype=dtype, device=self.device)
    _run("cuhnsw_unpack4_device", self.device, self.codes.data_ptr(), self.scales.data_ptr(), self.num_rows, self.num_dims,
         self.group, out.data_ptr(), _TYPES[dtype])
    return out

  def scores(self, queries, bias=None):
    """Products of queries with all rows, float32 ``[num_queries, num_rows]``, plus ``bias`` (float32 ``[num_rows]``) if
    given.  queries: float32, float16 or bfloat16 ``[num_queries, num_dims]``.  Made for few queries (a step of a
    decoder, a search): the codes are read once for every 32 of them (8 in float32, fewer if the rows are long)."""
    _is_matrix(queries, "queries")
    device = self.device
    if queries.device != device:
      _refuse(f"queries are on {queries.device}, the rows on {device}")
    count, dims = queries.shape
    if dims != self.num_dims:
      _refuse(f"queries have {dims} dimensions, the rows have {self.num_dims}")
    if count > 1 << 18:
      _refuse(f"{count} queries are too many")
    queries = _row_major(queries)
    if bias is not None:
      if not (isinstance(bias, torch.Tensor) and bias.device == device and bias.dtype == torch.float32 and
              bias.shape == (self.num_rows,)):
        _refuse(f"bias must be a float32 tensor [{self.num_rows}] beside the rows")
      bias = bias.contiguous()
    out = torch.empty((count, self.num_rows), dtype=torch.float32, device=device)
    _run("cuhnsw_scores4_device", device, self.codes.data_ptr(), self.scales.data_ptr(), self.num_rows, dims, self.group,
         queries.data_ptr(), queries.stride(0), _TYPES[queries.dtype], count, None if bias is None else bias.data_ptr(),
         out.data_ptr())
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
  if not 1 <= keep <= MAX_KEEP:
    _refuse(f"{name} must be 1 to {MAX_KEEP}, not {keep}")
  return keep


def _select(scores, totals, keep, log_softmax, negate, out_totals, out_beams, out_ids, out_found):
  device, (sequences, beams, vocabulary) = scores.device, scores.shape
  space = torch.empty(_workspace_bytes("cuhnsw_select_workspace", sequences, beams, vocabulary, keep), dtype=torch.uint8,
                      device=device)
  _run("cuhnsw_select_device", device, scores.data_ptr(), scores.stride(0), scores.stride(1), _TYPES[scores.dtype],
       None if totals is None else totals.data_ptr(), sequences, beams, vocabulary, keep, 1 if log_softmax else 0,
       1 if negate else 0, out_totals.data_ptr(), None if out_beams is None else out_beams.data_ptr(), out_ids.data_ptr(),
       None if out_found is None else out_found.data_ptr(), space.data_ptr())


def select_beams(scores, totals=None, keep=None, log_softmax=True):
  """The ``keep`` best continuations of every sequence over its beams and the vocabulary: (totals float32, beams int32, ids
  int32), each ``[sequences, keep]``, in descending order of

      totals[s, b] + scores[s, b, v] - log(sum over u of exp(scores[s, b, u]))

  (without the last term if ``log_softmax`` is false); equal ones by smaller beam, then smaller id.  scores: float32, float16 or
  bfloat16 ``[sequences, beams, vocabulary]``; totals: float32 ``[sequences, beams]``, default zeros; keep: 1 to 256, default
  the number of beams.  A total of -inf or NaN is never chosen (a beam that has ended or an id that may not follow is -inf);
  slots that stay empty hold -inf, -1, -1."""
  if not isinstance(scores, torch.Tensor) or not scores.is_cuda or scores.dtype not in _TYPES:
    _refuse("scores must be a float32, float16 or bfloat16 CUDA tensor")
  if scores.dim() != 3:
    _refuse(f"scores must be [sequences, beams, vocabulary], not {scores.dim()}-dimensional")
  device, (sequences, beams, vocabulary) = scores.device, scores.shape
  keep = _check_keep(beams if keep is None else keep, "keep")
  if beams > 16384:
    _refuse(f"{beams} beams are too many")
  if totals is not None:
    if not (isinstance(totals, torch.Tensor) and totals.device == device and totals.dtype == torch.float32 and
            totals.shape == (sequences, beams)):
      _refuse(f"totals must be a float32 tensor [{sequences}, {beams}] beside the scores")
    totals = totals.contiguous()
  if scores.stride(2) != 1 and vocabulary > 1:
    scores = scores.contiguous()
  out_totals = torch.empty((sequences, keep), dtype=torch.float32, device=device)
  out_beams, out_ids = torch.empty((2, sequences, keep), dtype=torch.int32, device=device).unbind()
  if sequences == 0 or beams == 0 or vocabulary == 0:
    return out_totals.fill_(float("-inf")), out_beams.fill_(-1), out_ids.fill_(-1)
  _select(scores, totals, keep, log_softmax, False, out_totals, out_beams, out_ids, None)
  return out_totals, out_beams, out_ids


_STATE_WORDS = 7  # cuhnsw_state: two addresses and five int64


def _pieces(state):
  """(segments, values between them, values of each) of a state's rows, or None if they are not evenly spaced pieces."""
  shape, strides = state.shape, state.stride()
  each, segments, between = 1, 1, 0
  for i in range(len(shape) - 1, 1, -1):
    size, stride = shape[i], strides[i]
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
  inputs = states if several else (states,)
  if not isinstance(beams, torch.Tensor) or not beams.is_cuda or beams.dtype != torch.int32 or beams.dim() != 2:
    _refuse("beams must be an int32 CUDA tensor [sequences, keep]")
  beams = beams.contiguous()
  device, (sequences, keep) = beams.device, beams.shape
  outs, words, copies, first = [], [], [], None
  for state in inputs:
    if not isinstance(state, torch.Tensor) or state.device != device or state.dim() < 2:
      _refuse(f"a state must be a tensor [sequences, beams, ...] on {device}")
    shape = state.shape
    first = shape if first is None else first
    if shape[0] != sequences or shape[1] != first[1]:
      _refuse(f"states of shapes {tuple(first)} and {tuple(shape)} for {sequences} sequences")
    pieces = _pieces(state)
    if pieces is None:
      state = state.contiguous()
      copies.append(state)
      pieces = _pieces(state)
    segments, between, each = pieces
    out = torch.empty((sequences, keep) + shape[2:], dtype=state.dtype, device=device)
    size, strides = state.element_size(), state.stride()
    words += (state.data_ptr(), out.data_ptr(), strides[0] * size, strides[1] * size, between * size,
              segments if each else 0, each * size)
    outs.append(out)
  if outs and sequences and keep:
    _run("cuhnsw_reorder_device", device, (ctypes.c_int64 * len(words))(*words), len(outs), beams.data_ptr(), sequences,
         first[1], keep)
  return outs if several else outs[0]
