"""The operators over a table of embeddings without a GPU: what the C ABI and the torch layer refuse, and the host's part of
the beams' states."""
import ctypes
import importlib.util
import re
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from conftest import has_gpu
from cuhnsw_b200 import _table, cuhnsw_bind, table

CSRC = Path(__file__).resolve().parent.parent / "cuhnsw_b200" / "csrc"
INVALID = -1
# addresses that are aligned but belong to nobody: a refused call must not touch them
A, ODD = 0x10000, 0x10001


def lib():
  return cuhnsw_bind.load_library()


def lookup(rows=A, stride=8, n=10, d=8, dtype=0, ids=A, ids64=0, count=4, scale=1.0, out=A):
  return lib().cuhnsw_lookup_device(rows, stride, n, d, dtype, ids, ids64, count, scale, out, None)


def grad(grad_=A, stride=8, dtype=1, ids=A, ids64=1, count=4, n=10, d=8, out=A, out_type=0, space=A):
  return lib().cuhnsw_lookup_grad_device(grad_, stride, dtype, ids, ids64, count, n, d, 1.0, out, out_type, 0, space, None)


def pack(rows=A, stride=64, dtype=2, n=3, d=64, group=32, codes=A, scales=A):
  return lib().cuhnsw_pack4_device(rows, stride, dtype, n, d, group, codes, scales, None)


def unpack(codes=A, scales=A, n=3, d=64, group=32, out=A, dtype=2):
  return lib().cuhnsw_unpack4_device(codes, scales, n, d, group, out, dtype, None)


def scores(codes=A, scales=A, n=3, d=64, group=32, queries=A, stride=64, dtype=0, nq=2, bias=None, out=A):
  return lib().cuhnsw_scores4_device(codes, scales, n, d, group, queries, stride, dtype, nq, bias, out, None)


def select(scores_=A, dtype=0, totals=None, s=2, b=3, v=100, keep=3, out=A, ids=A, space=A, seq=300, beam=100):
  return lib().cuhnsw_select_device(scores_, seq, beam, dtype, totals, s, b, v, keep, 1, 0, out, None, ids, None, space, None)


@pytest.mark.parametrize("call, bad", [
  (lookup, [dict(d=0), dict(d=(1 << 24) + 1), dict(n=-1), dict(n=2 ** 31 - 1), dict(dtype=3), dict(dtype=-1), dict(stride=-1),
            dict(count=-1), dict(count=2 ** 31 - 1), dict(rows=None), dict(ids=None), dict(out=None), dict(rows=ODD),
            dict(out=ODD), dict(ids=A + 2), dict(ids=A + 4, ids64=1)]),
  (grad, [dict(d=0), dict(n=-1), dict(dtype=3), dict(out_type=2), dict(stride=-1), dict(count=-1), dict(grad_=None),
          dict(ids=None), dict(out=None), dict(space=None), dict(space=A + 16), dict(grad_=ODD), dict(out=A + 2),
          dict(ids=A + 4)]),
  (pack, [dict(d=0), dict(n=-1), dict(dtype=3), dict(group=0), dict(group=16), dict(group=96), dict(group=-128),
          dict(group=200), dict(rows=None), dict(rows=ODD), dict(codes=None), dict(codes=A + 8), dict(scales=None),
          dict(scales=ODD), dict(stride=-1)]),
  (unpack, [dict(d=0), dict(n=-1), dict(dtype=3), dict(group=33), dict(codes=None), dict(codes=A + 4), dict(scales=None),
            dict(out=None), dict(out=ODD)]),
  (scores, [dict(d=0), dict(n=-1), dict(dtype=3), dict(group=48), dict(codes=A + 4), dict(scales=None), dict(queries=None),
            dict(queries=A + 2), dict(out=None), dict(out=A + 2), dict(bias=A + 2), dict(nq=-1), dict(nq=(1 << 18) + 1),
            dict(stride=-1)]),
  (select, [dict(s=-1), dict(b=0), dict(b=16385), dict(v=0), dict(v=2 ** 31 - 1), dict(keep=0), dict(keep=257), dict(dtype=5),
            dict(scores_=None), dict(scores_=ODD), dict(totals=A + 2), dict(out=None), dict(ids=None), dict(space=None),
            dict(space=A + 128), dict(seq=-1), dict(beam=-1)]),
])
def test_c_abi_refuses(call, bad):
  for arguments in bad:
    assert call(**arguments) == INVALID, arguments


def test_c_abi_has_nothing_to_do():
  """Empty work needs neither buffers nor a GPU."""
  assert lookup(count=0, rows=None, ids=None, out=None) == 0
  assert grad(n=0, out=None, space=None) == 0
  assert pack(n=0, rows=None, codes=None, scales=None) == 0
  assert unpack(n=0, codes=None, scales=None, out=None) == 0
  assert scores(nq=0, queries=None, out=None) == 0 and scores(n=0, codes=None, scales=None, out=None) == 0
  assert select(s=0, scores_=None, out=None, ids=None, space=None) == 0
  assert lib().cuhnsw_reorder_device(None, 0, None, 4, 2, 2, None) == 0


def state_of(src, dst, seq_stride, beam_stride, segment_stride, segments, bytes):
  return (ctypes.c_int64 * 7)(src or 0, dst or 0, seq_stride, beam_stride, segment_stride, segments, bytes)


def test_workspaces_and_states_are_checked():
  assert lib().cuhnsw_lookup_grad_workspace(-1, 10, 8) == INVALID
  assert lib().cuhnsw_lookup_grad_workspace(5, 10, 0) == INVALID
  assert lib().cuhnsw_lookup_grad_workspace(0, 10, 8) == 0
  few, many = (lib().cuhnsw_lookup_grad_workspace(t, 50_000, 64) for t in (1000, 100_000))
  assert 0 < few < many
  assert lib().cuhnsw_select_workspace(2, 3, 100, 0) == INVALID
  assert lib().cuhnsw_select_workspace(2, 3, 100, 5) >= 2 * 3 * 5 * 8
  good = dict(src=A, dst=A, seq_stride=64, beam_stride=32, segment_stride=0, segments=1, bytes=32)
  for bad in (dict(src=None), dict(dst=None), dict(segments=-1), dict(bytes=-4), dict(seq_stride=-1), dict(beam_stride=-1),
              dict(segment_stride=-1)):
    state = state_of(**dict(good, **bad))
    assert lib().cuhnsw_reorder_device(state, 1, A, 2, 2, 2, None) == INVALID, bad
  state = state_of(**good)
  assert lib().cuhnsw_reorder_device(state, 1, None, 2, 2, 2, None) == INVALID
  assert lib().cuhnsw_reorder_device(None, 1, A, 2, 2, 2, None) == INVALID
  assert lib().cuhnsw_reorder_device(state, -1, A, 2, 2, 2, None) == INVALID


def test_torch_layer_refuses_tensors_of_the_host():
  rows = torch.zeros(4, 8)
  for call in (lambda: table.lookup(rows, torch.zeros(2, dtype=torch.int64)), lambda: table.pack_rows(rows),
               lambda: table.lookup_grad(rows, torch.zeros(4, dtype=torch.int64), 4),
               lambda: table.PackedRows(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.bfloat16), 8, 32),
               lambda: table.select_beams(torch.zeros(1, 2, 8)),
               lambda: table.reorder(torch.zeros(1, 2, 8), torch.zeros(1, 2, dtype=torch.int32))):
    with pytest.raises(RuntimeError, match="CUDA tensor"):
      call()


@pytest.mark.parametrize("make, pieces", [
  (lambda: torch.zeros(2, 3, 4, 5), (1, 0, 20)),                    # dense
  (lambda: torch.zeros(2, 3, 4, 9, 5)[:, :, :, :6], (4, 45, 30)),   # the part of a cache that is in use
  (lambda: torch.zeros(2, 3, 4, 7, 9, 5)[:, :, :, :, :6], (28, 45, 30)),
  (lambda: torch.zeros(2, 3, 9)[:, :, ::2], (5, 2, 1)),
  (lambda: torch.zeros(2, 3), (1, 0, 1)),
  (lambda: torch.zeros(2, 3, 1, 1), (1, 0, 1)),
  (lambda: torch.zeros(2, 3, 4, 5).transpose(2, 3), None),          # not evenly spaced pieces in the order of the output
  (lambda: torch.zeros(2, 3, 6, 5)[:, :, ::2, ::2], None),
])
def test_pieces_of_a_state(make, pieces):
  got = _table.pieces(make())
  assert got == pieces or pieces is not None and pieces[0] == 1 and got == (1, 0, pieces[2])


def test_pieces_cover_a_state():
  """Reading piece by piece gives the values in the order of the dense output."""
  base = torch.arange(2 * 3 * 4 * 9 * 5).view(2, 3, 4, 9, 5)
  for view in (base, base[:, :, :, 2:7], base[:, :, 1:3], base[:, :, :, :, 3:4], base.transpose(0, 1), base[:, :, :, 4]):
    segments, between, each = _table.pieces(view)
    flat = base.view(-1)
    for s in range(view.shape[0]):
      for b in range(view.shape[1]):
        at = view[s, b].storage_offset()
        got = torch.cat([flat[at + i * between:at + i * between + each] for i in range(segments)])
        assert torch.equal(got, view[s, b].reshape(-1))


@pytest.mark.skipif(has_gpu(), reason="checks the failure mode of a machine without a GPU")
def test_fails_loudly_without_a_gpu():
  assert lookup() == -5 and pack() == -5 and select() == -5


def test_kernels_that_start_early_read_by_ordinary_loads():
  """Read-only loads are for data that nobody writes while the kernel lives, and these live before the launch ahead of them ends."""
  launchers = [f for f in CSRC.glob("*.cu") if "launch_early(" in f.read_text()]
  assert len(launchers) >= 4
  for f in launchers + [CSRC / "table_common.cuh", CSRC / "scores4.cuh"]:
    code = re.sub(r"//[^\n]*", "", f.read_text())
    assert not re.search(r"__ldg\b|ld\.global(\.\w+)*\.nc|__restrict__|tex1Dfetch", code), f.name


def test_the_library_builds_without_torch(tmp_path):
  """Only the torch layer needs torch's headers."""
  def wanted(python):
    done = subprocess.run(["make", "-n", "-B", "-C", str(CSRC), f"PYTHON={python}"], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stderr
    return done.stdout

  without = tmp_path / "python"
  without.write_text(f'#!/bin/sh\nexec {sys.executable} -S "$@"\n')  # (no installed packages)
  without.chmod(0o755)
  alone = wanted(without)
  assert "libcuhnsw_b200.so" in alone and "table.cu" in alone
  assert "table_torch" not in alone and "-o ../_table.so" not in alone and "_table.so, which only" in alone
  nothing = wanted("/nonexistent/python")
  assert "libcuhnsw_b200.so" in nothing and "table_torch" not in nothing
  if importlib.util.find_spec("torch"):
    assert "table_torch.cpp" in wanted(sys.executable)
