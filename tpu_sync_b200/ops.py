"""Tensor-level wrappers of the manager-free kernels of the C ABI.

These take torch CUDA tensors, build the small device-side descriptor tables
the kernels read, and launch on the current stream.  They are what the
manager, the weight synchronizer and the hand-off executor are made of, and
what the parity tests and the benchmark call directly.

The paged cache operators at the end (`PagedKV`, `kv_append`,
`paged_attention`, `shared_prefix_attention`) are what an engine runs between
those transfers, on the same storages: the write of new tokens into their
pages and the attention that reads the pages.
"""

from __future__ import annotations

import ctypes
import struct
from typing import List, Optional, Sequence, Tuple, Union

import numpy as np
import torch
from torch.autograd import forward_ad

from tpu_sync_b200 import _native


def _stream(stream: Optional[torch.cuda.Stream], device) -> ctypes.c_void_p:
  s = stream if stream is not None else torch.cuda.current_stream(device)
  return ctypes.c_void_p(s.cuda_stream)


def _nbytes(t: torch.Tensor) -> int:
  return t.numel() * t.element_size()


def _to_device_bytes(arr: ctypes.Array, device) -> torch.Tensor:
  raw = np.frombuffer(bytes(arr), dtype=np.uint8).copy()
  return torch.from_numpy(raw).to(device)


class StorageTable:
  """Device table of (layer, shard) storages for the block kernels.

  stage_off of storage s = sum of the (16-byte rounded) slot bytes of the
  storages before it, so a staging block is [storage 0 | storage 1 | ...].
  `slot_scale` = 0.5 lays out fp8 payload slots (half the bf16 bytes).
  """

  def __init__(self, storages: Sequence[torch.Tensor], fp8: bool = False):
    if not storages:
      raise ValueError("need at least one storage")
    self.storages = list(storages)
    self.device = self.storages[0].device
    n = len(self.storages)
    arr = (_native.BlockStorage * n)()
    off = 0
    self.block_bytes = []
    self.stage_offs = []
    for i, t in enumerate(self.storages):
      if not t.is_cuda or not t.is_contiguous():
        raise ValueError("storages must be contiguous CUDA tensors")
      if t.device != self.device:
        raise ValueError("all storages must live on one device")
      bb = _nbytes(t) // t.shape[0]
      arr[i].dev_ptr = t.data_ptr()
      arr[i].block_bytes = bb
      arr[i].dev_bytes = _nbytes(t)
      arr[i].stage_off = off
      self.block_bytes.append(bb)
      self.stage_offs.append(off)
      slot = bb // 2 if fp8 else bb
      off += (slot + 15) // 16 * 16
    self.scale_off = off if fp8 else 0
    if fp8:
      off += (4 * n + 15) // 16 * 16
    self.pitch = (off + 15) // 16 * 16
    self.fp8 = fp8
    self.d_table = _to_device_bytes(arr, self.device)
    self.n = n

  def new_staging(self, n_blocks: int) -> torch.Tensor:
    return torch.empty((n_blocks, self.pitch), dtype=torch.uint8, device=self.device)


def _keep(tensors, stream: Optional[torch.cuda.Stream]) -> None:
  """Keeps temporaries alive for kernels queued on a non-current stream."""
  if stream is not None:
    for t in tensors:
      t.record_stream(stream)


def _ids(ids, device) -> torch.Tensor:
  if isinstance(ids, torch.Tensor):
    t = ids.to(device=device, dtype=torch.int64).contiguous()
  else:
    t = torch.tensor(list(ids), dtype=torch.int64, device=device)
  return t


def kv_extract(table: StorageTable, ids, staging: torch.Tensor,
               err_flag: Optional[torch.Tensor] = None,
               stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
  """staging[k] <- block ids[k] of every storage (block-major)."""
  d_ids = _ids(ids, table.device)
  fn = _native.lib().ts_kv_extract_fp8 if table.fp8 else _native.lib().ts_kv_extract
  args = [table.device.index, ctypes.c_void_p(table.d_table.data_ptr()), table.n,
          ctypes.c_void_p(d_ids.data_ptr()), d_ids.numel(),
          ctypes.c_void_p(staging.data_ptr()), table.pitch]
  if table.fp8:
    args.append(table.scale_off)
  args += [ctypes.c_void_p(err_flag.data_ptr() if err_flag is not None else 0),
           _stream(stream, table.device)]
  _native.check(fn(*args), "kv_extract: ")
  _keep([d_ids], stream)
  return staging


def kv_insert(table: StorageTable, ids, staging: torch.Tensor,
              err_flag: Optional[torch.Tensor] = None,
              stream: Optional[torch.cuda.Stream] = None) -> None:
  """block ids[k] of every storage <- staging[k]."""
  d_ids = _ids(ids, table.device)
  fn = _native.lib().ts_kv_insert_fp8 if table.fp8 else _native.lib().ts_kv_insert
  args = [table.device.index, ctypes.c_void_p(table.d_table.data_ptr()), table.n,
          ctypes.c_void_p(d_ids.data_ptr()), d_ids.numel(),
          ctypes.c_void_p(staging.data_ptr()), table.pitch]
  if table.fp8:
    args.append(table.scale_off)
  args += [ctypes.c_void_p(err_flag.data_ptr() if err_flag is not None else 0),
           _stream(stream, table.device)]
  _native.check(fn(*args), "kv_insert: ")
  _keep([d_ids], stream)


_TORCH_TO_TS = {torch.uint8: _native.DTYPE_U8, torch.bfloat16: _native.DTYPE_BF16,
                torch.float32: _native.DTYPE_F32, torch.float16: _native.DTYPE_F16}


def _extent_bytes(x) -> Optional[int]:
  """Bytes a chunk endpoint holds when it knows its size (a tensor or a
  PeerBuffer), else None (a raw address)."""
  if isinstance(x, torch.Tensor):
    return x.numel() * x.element_size()
  if isinstance(x, (int, np.integer)):
    return None
  if hasattr(x, "nbytes"):
    return int(x.nbytes)
  return None


def _check_chunks(chunks, src_es: int, dst_es: int) -> None:
  """Every chunk stays inside its source and destination where their sizes
  are known: (offset + (count - 1) * stride + size) elements."""
  for i, (sp, dp, so, do, size, ss, ds, cnt) in enumerate(chunks):
    if size <= 0 or cnt <= 0:
      continue
    for name, obj, off, stride, es in (("source", sp, so, ss, src_es),
                                       ("destination", dp, do, ds, dst_es)):
      n = _extent_bytes(obj)
      if n is None:
        continue
      end = (off + (cnt - 1) * stride + size) * es if cnt > 1 else (off + size * cnt) * es
      if off < 0 or end > n:
        raise ValueError(f"chunk {i} ends past its {name}: byte {end} of {n}")


class ReshardProgram:
  """A list of strided chunks compiled for one launch of ts_reshard_copy.

  chunks: iterables (src_tensor, dst_tensor_or_ptr, src_off, dst_off, size,
  src_stride, dst_stride, count) in elements.  All sources must be on
  `device`; destinations may be local or peer-GPU addresses.
  """

  def __init__(self, chunks, src_dtype: torch.dtype, dst_dtype: torch.dtype,
               device: torch.device):
    self.device = torch.device(device)
    self.src_dtype = _TORCH_TO_TS[src_dtype]
    self.dst_dtype = _TORCH_TO_TS[dst_dtype]
    chunks = list(chunks)
    _check_chunks(chunks, torch.empty((), dtype=src_dtype).element_size(),
                  torch.empty((), dtype=dst_dtype).element_size())
    n = len(chunks)
    arr = (_native.ReshardChunk * max(n, 1))()
    for i, (sp, dp, so, do, size, ss, ds, cnt) in enumerate(chunks):
      arr[i].src_ptr = sp.data_ptr() if hasattr(sp, "data_ptr") else int(sp)
      arr[i].dst_ptr = dp.data_ptr() if hasattr(dp, "data_ptr") else int(dp)
      arr[i].src_off, arr[i].dst_off, arr[i].size = int(so), int(do), int(size)
      arr[i].src_stride, arr[i].dst_stride, arr[i].count = int(ss), int(ds), int(cnt)
    prefix = np.zeros(n + 1, dtype=np.int64)
    _native.check(_native.lib().ts_reshard_work_items(
        arr, n, self.src_dtype, self.dst_dtype,
        prefix.ctypes.data_as(_native.c_i64_p)), "reshard plan: ")
    self.n_chunks = n
    self.n_items = int(prefix[-1])
    self.d_chunks = _to_device_bytes(arr, self.device)
    self.d_prefix = torch.from_numpy(prefix).to(self.device)

  def launch(self, stream: Optional[torch.cuda.Stream] = None) -> None:
    _native.check(_native.lib().ts_reshard_copy(
        self.device.index, ctypes.c_void_p(self.d_chunks.data_ptr()),
        ctypes.c_void_p(self.d_prefix.data_ptr()), self.n_chunks, self.n_items,
        self.src_dtype, self.dst_dtype, _stream(stream, self.device)), "reshard: ")


def _pages(storages, geom: dict, given: Optional[int], side: str) -> int:
  """Pages every storage holds: `given`, else the smallest storage's bytes
  (tensors and PeerBuffers know theirs) over the page size."""
  if given is not None:
    return int(given)
  page = int(geom["block_tokens"]) * int(geom["heads"]) * int(geom["head_bytes"])
  sizes = []
  for x in storages:
    if isinstance(x, torch.Tensor):
      sizes.append(x.numel() * x.element_size())
    elif hasattr(x, "nbytes"):
      sizes.append(int(x.nbytes))
    else:
      raise ValueError(f"{side} storages given as raw addresses need {side}_pages")
  return min(sizes) // page


class ReshardCopyEngineProgram:
  """The same chunks as ReshardProgram, pushed by the copy engines: the cast
  to the destination dtype goes to a local staging buffer and each staged
  chunk moves with one cudaMemcpy2DAsync, `groups` groups pipelining the
  cast against the copies (ts_reshard_ce_*)."""

  def __init__(self, chunks, src_dtype: torch.dtype, dst_dtype: torch.dtype,
               device: torch.device, groups: int = 16):
    self.device = torch.device(device)
    chunks = list(chunks)
    _check_chunks(chunks, torch.empty((), dtype=src_dtype).element_size(),
                  torch.empty((), dtype=dst_dtype).element_size())
    arr = (_native.ReshardChunk * max(len(chunks), 1))()
    for i, (sp, dp, so, do, size, ss, ds, cnt) in enumerate(chunks):
      arr[i].src_ptr = sp.data_ptr() if hasattr(sp, "data_ptr") else int(sp)
      arr[i].dst_ptr = dp.data_ptr() if hasattr(dp, "data_ptr") else int(dp)
      arr[i].src_off, arr[i].dst_off, arr[i].size = int(so), int(do), int(size)
      arr[i].src_stride, arr[i].dst_stride, arr[i].count = int(ss), int(ds), int(cnt)
    h = ctypes.c_void_p()
    _native.check(_native.lib().ts_reshard_ce_create(
        self.device.index, arr, len(chunks), _TORCH_TO_TS[src_dtype], _TORCH_TO_TS[dst_dtype],
        int(groups), ctypes.byref(h)), "reshard (copy engines): ")
    self._h = h
    g, b, c = ctypes.c_int64(), ctypes.c_uint64(), ctypes.c_int64()
    _native.check(_native.lib().ts_reshard_ce_info(h, ctypes.byref(g), ctypes.byref(b),
                                                   ctypes.byref(c)))
    self.groups, self.staging_bytes, self.copies = g.value, b.value, c.value

  def launch(self, stream: Optional[torch.cuda.Stream] = None) -> None:
    _native.check(_native.lib().ts_reshard_ce_launch(self._h, _stream(stream, self.device)),
                  "reshard (copy engines): ")

  def close(self) -> None:
    if getattr(self, "_h", None):
      _native.lib().ts_reshard_ce_destroy(self._h)
      self._h = None

  def __del__(self):
    try:
      self.close()
    except Exception:
      pass


class PullSender:
  """Sender side of the staged-pull weight sync (ts_wpull_src_*): casts the
  fp32 `src` (a 1-D CUDA tensor, the shard as the receivers' chunks address
  it) into a bf16 staging of the same element layout in `groups` groups, and
  publishes each group in the /dev/shm mailbox `name` as soon as it is
  written.  `stage()` is one generation; it first waits until every attached
  receiver has pulled the previous one."""

  def __init__(self, name: str, src: torch.Tensor, groups: int = 16):
    if src.dtype != torch.float32 or not src.is_cuda or not src.is_contiguous():
      raise ValueError("PullSender needs a contiguous fp32 CUDA tensor")
    self.device = src.device
    self.name = name
    self._src = src  # kept alive: the cast kernels read it
    h = ctypes.c_void_p()
    _native.check(_native.lib().ts_wpull_src_create(
        self.device.index, name.encode(), ctypes.c_void_p(src.data_ptr()), src.numel(),
        int(groups), ctypes.byref(h)), "weight pull sender: ")
    self._h = h
    g, b = ctypes.c_int64(), ctypes.c_uint64()
    _native.check(_native.lib().ts_wpull_src_info(h, None, ctypes.byref(g), ctypes.byref(b), None))
    self.groups, self.staging_bytes = g.value, b.value

  def stage(self, stream: Optional[torch.cuda.Stream] = None, timeout_ms: int = 30000) -> None:
    _native.check(_native.lib().ts_wpull_src_stage(self._h, _stream(stream, self.device),
                                                   int(timeout_ms)), "weight pull sender: ")

  def wait(self, timeout_ms: int = 30000) -> None:
    _native.check(_native.lib().ts_wpull_src_wait(self._h, int(timeout_ms)),
                  "weight pull sender: ")

  @property
  def receivers(self) -> int:
    n = ctypes.c_int64()
    _native.check(_native.lib().ts_wpull_src_info(self._h, None, None, None, ctypes.byref(n)))
    return n.value

  def close(self) -> None:
    if getattr(self, "_h", None):
      _native.lib().ts_wpull_src_destroy(self._h)
      self._h = None

  def __del__(self):
    try:
      self.close()
    except Exception:
      pass


class PullReceiver:
  """Receiver side of the staged-pull weight sync (ts_wpull_dst_*).

  names: the senders' mailboxes.  chunks: iterables (sender_index,
  dst_tensor_or_ptr, src_off, dst_off, size, src_stride, dst_stride, count)
  in bf16 elements; the source is the sender's staging (its fp32 shard's
  element layout).  `pull()` launches every chunk's copy on `stream` as soon
  as the groups it reads are published, and returns once all are queued."""

  def __init__(self, names: Sequence[str], chunks, device: torch.device):
    self.device = torch.device(device)
    chunks = list(chunks)
    _check_chunks([(None,) + tuple(c[1:]) for c in chunks], 2, 2)
    arr = (_native.ReshardChunk * max(len(chunks), 1))()
    self._keep = []
    for i, (t, dp, so, do, size, ss, ds, cnt) in enumerate(chunks):
      arr[i].src_ptr = int(t)
      arr[i].dst_ptr = dp.data_ptr() if hasattr(dp, "data_ptr") else int(dp)
      if hasattr(dp, "data_ptr"):
        self._keep.append(dp)
      arr[i].src_off, arr[i].dst_off, arr[i].size = int(so), int(do), int(size)
      arr[i].src_stride, arr[i].dst_stride, arr[i].count = int(ss), int(ds), int(cnt)
    cnames = (ctypes.c_char_p * len(names))(*[n.encode() for n in names])
    h = ctypes.c_void_p()
    _native.check(_native.lib().ts_wpull_dst_create(
        self.device.index, cnames, len(names), arr, len(chunks), ctypes.byref(h)),
        "weight pull receiver: ")
    self._h = h
    lc, b = ctypes.c_int64(), ctypes.c_uint64()
    _native.check(_native.lib().ts_wpull_dst_info(h, None, ctypes.byref(lc), ctypes.byref(b)))
    self.launches, self.bytes = lc.value, b.value

  def pull(self, stream: Optional[torch.cuda.Stream] = None, timeout_ms: int = 30000) -> None:
    _native.check(_native.lib().ts_wpull_dst_pull(self._h, _stream(stream, self.device),
                                                  int(timeout_ms)), "weight pull receiver: ")

  def close(self) -> None:
    if getattr(self, "_h", None):
      _native.lib().ts_wpull_dst_destroy(self._h)
      self._h = None

  def __del__(self):
    try:
      self.close()
    except Exception:
      pass


def kv_relayout(src_storages: Sequence, dst_storages: Sequence, src_geom: dict,
                dst_geom: dict, src_table: torch.Tensor, dst_table: torch.Tensor,
                seq_tokens: int, device=None,
                stream: Optional[torch.cuda.Stream] = None, src_pages: Optional[int] = None,
                dst_pages: Optional[int] = None,
                err: Optional[torch.Tensor] = None) -> torch.Tensor:
  """Copies every token of every sequence between two page geometries.

  src_storages / dst_storages: tensors, PeerBuffers or raw device addresses
  (destinations may be peer-GPU addresses; raw addresses need src_pages /
  dst_pages, the pages each storage holds).  Geometries are dicts with
  block_tokens, heads, head_bytes, head_major.  Tables are int32
  [n_seqs, blocks_per_seq].  Table entries outside a storage's pages are
  skipped and flagged: returns the device int32 flag (`err`, or a new one),
  non-zero after the kernel ran if any entry was out of range.
  """
  device = torch.device(device) if device is not None else src_table.device
  n = len(src_storages)
  if len(dst_storages) != n:
    raise ValueError("source and destination storage counts differ")
  sp = _pages(src_storages, src_geom, src_pages, "src")
  dp = _pages(dst_storages, dst_geom, dst_pages, "dst")
  if err is None:
    err = torch.zeros(1, dtype=torch.int32, device=device)
  ptr = lambda x: x.data_ptr() if hasattr(x, "data_ptr") else int(x)
  d_src = torch.tensor([ptr(x) for x in src_storages], dtype=torch.int64,
                       device=device)
  d_dst = torch.tensor([ptr(x) for x in dst_storages], dtype=torch.int64,
                       device=device)
  sg = _native.PageGeometry(int(src_geom["block_tokens"]), int(src_geom["heads"]),
                            int(src_geom["head_bytes"]), int(src_geom["head_major"]), 0)
  dg = _native.PageGeometry(int(dst_geom["block_tokens"]), int(dst_geom["heads"]),
                            int(dst_geom["head_bytes"]), int(dst_geom["head_major"]), 0)
  st = src_table.to(device=device, dtype=torch.int32).contiguous()
  dt = dst_table.to(device=device, dtype=torch.int32).contiguous()
  _native.check(_native.lib().ts_kv_relayout(
      device.index, ctypes.c_void_p(d_src.data_ptr()), ctypes.c_void_p(d_dst.data_ptr()),
      n, sg, dg, ctypes.c_void_p(st.data_ptr()), st.shape[1],
      ctypes.c_void_p(dt.data_ptr()), dt.shape[1], st.shape[0], int(seq_tokens), sp, dp,
      ctypes.c_void_p(err.data_ptr()), _stream(stream, device)), "kv_relayout: ")
  _keep([d_src, d_dst, st, dt, err], stream)
  return err


_PAGE_DTYPES = {torch.bfloat16: _native.DTYPE_BF16, torch.float16: _native.DTYPE_F16}


class PagedKV:
  """One layer's K and V storages as the paged cache operators address them.

  k_pages / v_pages: bf16 or fp16 CUDA tensors [pages, block_tokens, heads,
  head_dim], or with `head_major` [pages, heads, block_tokens, head_dim] (the
  page orders of kv_relayout): the storages given to the manager, or strided
  views of a joint cache such as kv[:, 0] and kv[:, 1] of [pages, 2, ...].
  The last dimension is contiguous.  Like StorageTable it is built once and
  describes the memory; it keeps the tensors alive.
  """

  def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, head_major: bool = False):
    for t in (k_pages, v_pages):
      if not t.is_cuda or t.dim() != 4:
        raise ValueError("pages must be 4-dimensional CUDA tensors")
      if t.dtype not in _PAGE_DTYPES:
        raise ValueError(f"pages must be bfloat16 or float16, not {t.dtype}")
      if t.shape[3] > 1 and t.stride(3) != 1:
        raise ValueError("the last dimension of the pages must be contiguous")
    if (k_pages.shape, k_pages.dtype, k_pages.device) != (v_pages.shape, v_pages.dtype,
                                                          v_pages.device):
      raise ValueError("K and V pages must have one shape, dtype and device")
    if min(k_pages.shape[1:]) < 1:
      raise ValueError("pages need at least one token, head and element")
    if k_pages.requires_grad or v_pages.requires_grad:
      raise ValueError("pages must not require grad: they are written in place")
    self.k_pages, self.v_pages, self.head_major = k_pages, v_pages, bool(head_major)
    self.device, self.dtype = k_pages.device, k_pages.dtype
    tok, head = (2, 1) if head_major else (1, 2)
    self.pages, self.block_tokens = k_pages.shape[0], k_pages.shape[tok]
    self.heads, self.head_dim = k_pages.shape[head], k_pages.shape[3]
    # a dimension of one element is never stepped over: its stride says nothing
    strides = [t.stride(i) if t.shape[i] > 1 else 0 for t in (k_pages, v_pages)
               for i in (0, tok, head)]
    self._c = _native.PagedKvC(
        k_pages.data_ptr(), v_pages.data_ptr(), self.pages, self.block_tokens, self.heads,
        self.head_dim, *strides, _PAGE_DTYPES[self.dtype], 0)
    self._ref = ctypes.byref(self._c)
    self._index = self.device.index
    self._workspace = {}  # bytes of attention workspace by shapes


# The argument structures as bytes (one pack is cheaper than filling a ctypes
# structure field by field): ts_kv_append_args, ts_attention_args.
_APPEND_ARGS = struct.Struct("=22qifii")
_ATTENTION_ARGS = struct.Struct("=17qfi")


def _check_heads(kv: PagedKV, name: str, t: torch.Tensor, shape: Tuple[int, ...]) -> None:
  """Raises what is wrong with a tensor of heads."""
  if t.shape != shape:
    raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
  if t.dtype != kv.dtype or t.device != kv.device:
    raise ValueError(f"{name} must have the pages' dtype and device")
  if t.stride(-1) != 1 and shape[-1] > 1:
    raise ValueError(f"the last dimension of {name} must be contiguous")


def _check_index(kv: PagedKV, name: str, t: torch.Tensor, dtype: torch.dtype, dims: int,
                 length: Optional[int]) -> None:
  """The same for an index tensor, a table or a weight; `length`: of its first dimension."""
  if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.dim() != dims or (
      t.device != kv.device):
    raise ValueError(f"{name} must be a {dims}-dimensional {dtype} tensor on {kv.device}")
  if t.stride(-1) != 1 and t.shape[-1] > 1:
    raise ValueError(f"the last dimension of {name} must be contiguous")
  if length is not None and t.shape[0] != length:
    raise ValueError(f"{name} must hold {length} entries, got {list(t.shape)}")


def _weight_ok(t: torch.Tensor, dtype: torch.dtype, length: int, index: int) -> bool:
  return (t.shape == (length,) and t.dtype is dtype and t.get_device() == index and
          t.stride() == (1,))


def _no_grad_path() -> ValueError:
  return ValueError("an input requires grad: the paged cache operators have no backward pass")


def _refuse_tangents(kv: PagedKV, *tensors: Optional[torch.Tensor]) -> None:
  """The same for forward-mode derivatives (called only within a dual level)."""
  for t in (kv.k_pages, kv.v_pages, *tensors):
    if t is not None and forward_ad.unpack_dual(t).tangent is not None:
      raise ValueError("an input has a tangent: the paged cache operators have no derivatives")


def _flag(kv: PagedKV, err_flag: Optional[torch.Tensor]) -> int:
  if err_flag is None:
    return 0
  if err_flag.dtype != torch.int32 or err_flag.device != kv.device or err_flag.numel() < 1:
    raise ValueError("err_flag must be an int32 tensor on the pages' device")
  return err_flag.data_ptr()


def kv_append(kv: PagedKV, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,
              q: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
              cos_sin: Optional[torch.Tensor] = None, interleaved: bool = False,
              q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
              eps: float = 1e-6, q_out: Optional[torch.Tensor] = None,
              err_flag: Optional[torch.Tensor] = None,
              stream: Optional[torch.cuda.Stream] = None) -> Optional[torch.Tensor]:
  """Writes new tokens' keys and values into their pages; norms and rotates
  queries and keys on the way.  Returns the queries (None without `q`).

  k, v [tokens, heads, head_dim] and q [tokens, q_heads, head_dim] may be
  strided views of one projection's output.  slots: int64 [tokens], page *
  block_tokens + offset; negative for a padding token, which writes nothing.
  cos_sin: float32 [max_position, rotary], row p = the cosines, then the sines,
  of position p's rotary / 2 angles; rotates the first `rotary` elements of a
  head by row positions[t] (int64), pairs (i, i + rotary/2), or (2i, 2i+1) if
  `interleaved`.  q_weight / k_weight [head_dim] (the pages' dtype or float32)
  apply x * weight / sqrt(mean(x^2) + eps) to every query / key head before the
  rotation.  q_out is q itself, or shares no element with q, k and v (other
  columns of their buffer will do); its padding rows stay as they were (a new
  one has zeros there).

  The slots of one call are distinct: where two tokens name one slot, it is not
  defined which of them stays.  A slot past the pages or a position past
  cos_sin writes nothing for its token and sets err_flag (int32, on the device)
  to 1.
  """
  index, dtype, dim = kv._index, kv.dtype, kv.head_dim
  shape = k.shape
  if len(shape) != 3 or shape[1] != kv.heads or shape[2] != dim:
    raise ValueError(f"k must be [tokens, {kv.heads}, {dim}], got {list(shape)}")
  tokens = shape[0]
  ks, vs = k.stride(), v.stride()
  if (k.dtype is not dtype or v.dtype is not dtype or v.shape != shape or
      k.get_device() != index or v.get_device() != index or ks[2] != 1 or vs[2] != 1):
    _check_heads(kv, "k", k, shape)
    _check_heads(kv, "v", v, shape)
  if (slots.dtype is not torch.int64 or slots.shape != (tokens,) or
      slots.get_device() != index or slots.stride() != (1,)):
    _check_index(kv, "slots", slots, torch.int64, 1, tokens)
  table = places = rows = row_stride = rotary = 0
  if cos_sin is not None:
    if (not isinstance(positions, torch.Tensor) or positions.dtype is not torch.int64 or
        positions.shape != (tokens,) or positions.get_device() != index or
        positions.stride() != (1,)):
      _check_index(kv, "positions", positions, torch.int64, 1, tokens)
    if (cos_sin.dtype is not torch.float32 or cos_sin.dim() != 2 or
        cos_sin.get_device() != index or cos_sin.stride(1) != 1):
      _check_index(kv, "cos_sin", cos_sin, torch.float32, 2, None)
    rows, rotary = cos_sin.shape
    if rows == 0:
      raise ValueError("cos_sin has no rows")
    table, places = cos_sin.data_ptr(), positions.data_ptr()
    row_stride = cos_sin.stride(0) if rows > 1 else rotary
  elif interleaved or positions is not None:
    raise ValueError("positions and interleaved need cos_sin")
  wq = wk = weight_dtype = 0
  if q_weight is not None or k_weight is not None:
    w = q_weight if q_weight is not None else k_weight
    if w.dtype not in (dtype, torch.float32):
      raise ValueError("norm weights must be float32 or of the pages' dtype")
    if q_weight is not None:
      if q is None:
        raise ValueError("q_weight needs q")
      if not _weight_ok(q_weight, w.dtype, dim, index):
        _check_index(kv, "q_weight", q_weight, w.dtype, 1, dim)
      wq = q_weight.data_ptr()
    if k_weight is not None:
      if not _weight_ok(k_weight, w.dtype, dim, index):
        _check_index(kv, "k_weight", k_weight, w.dtype, 1, dim)
      wk = k_weight.data_ptr()
    weight_dtype = _TORCH_TO_TS[w.dtype]
  if torch.is_grad_enabled() and (
      k.requires_grad or v.requires_grad or (q is not None and q.requires_grad) or
      (q_out is not None and q_out.requires_grad) or
      (cos_sin is not None and cos_sin.requires_grad) or
      (q_weight is not None and q_weight.requires_grad) or
      (k_weight is not None and k_weight.requires_grad)):
    raise _no_grad_path()
  if forward_ad._current_level >= 0:
    _refuse_tangents(kv, k, v, q, q_out, cos_sin, q_weight, k_weight)
  q_ptr = out_ptr = heads = qt = qh = ot = oh = zero = 0
  if q is not None:
    heads = q.shape[1] if q.dim() == 3 else 0
    if heads == 0:
      raise ValueError(f"q must be [{tokens}, heads, {dim}], got {list(q.shape)}")
    shape = (tokens, heads, dim)
    qt, qh, last = q.stride()
    if (q.shape != shape or q.dtype is not dtype or q.get_device() != index or last != 1):
      _check_heads(kv, "q", q, shape)
    if q_out is None:
      if stream is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
      else:
        with torch.cuda.stream(stream):  # what a call allocates belongs to its stream
          q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
      ot, oh, zero = heads * dim, dim, 1
    else:
      _check_heads(kv, "q_out", q_out, shape)
      ot, oh, _ = q_out.stride()
    q_ptr, out_ptr = q.data_ptr(), q_out.data_ptr()
  elif q_out is not None:
    raise ValueError("q_out needs q")
  args = _APPEND_ARGS.pack(k.data_ptr(), v.data_ptr(), q_ptr, out_ptr, ks[0], ks[1], vs[0], vs[1],
                           qt, qh, ot, oh, tokens, heads, slots.data_ptr(), places, table, rows,
                           row_stride, rotary, wq, wk, weight_dtype, eps, bool(interleaved), zero)
  rc = _native.lib().ts_kv_append(index, kv._ref, args,
                                  0 if err_flag is None else _flag(kv, err_flag),
                                  torch._C._cuda_getCurrentRawStream(index)
                                  if stream is None else stream.cuda_stream)
  if rc:
    _native.check(rc, "kv_append: ")
  return q_out


def _attention(kv, q, block_table, seq_lens, prefix_table, prefix_len, scale, out, return_lse,
               err_flag, stream):
  shape = q.shape
  if len(shape) == 3:
    batch, q_heads, dim = shape
    new = 1
  elif len(shape) == 4:
    batch, new, q_heads, dim = shape
  else:
    raise ValueError("q must be [batch, q_heads, head_dim] or [batch, new_tokens, q_heads, "
                     "head_dim]")
  if dim != kv.head_dim or q_heads == 0:
    raise ValueError(f"q heads must have {kv.head_dim} elements")
  index, dtype, device = kv._index, kv.dtype, kv.device
  strides = q.stride()
  if q.dtype is not dtype or q.get_device() != index or strides[-1] != 1:
    _check_heads(kv, "q", q, shape)
  if (block_table.dtype is not torch.int32 or block_table.dim() != 2 or
      block_table.get_device() != index or block_table.shape[0] != batch or
      block_table.stride(1) != 1):
    _check_index(kv, "block_table", block_table, torch.int32, 2, batch)
  if (seq_lens.dtype is not torch.int32 or seq_lens.shape != (batch,) or
      seq_lens.get_device() != index or seq_lens.stride() != (1,)):
    _check_index(kv, "seq_lens", seq_lens, torch.int32, 1, batch)
  shared = blocks = length = length_ptr = 0
  if prefix_table is not None:
    if (prefix_table.dtype is not torch.int32 or prefix_table.dim() != 1 or
        prefix_table.get_device() != index or prefix_table.stride(0) != 1):
      _check_index(kv, "prefix_table", prefix_table, torch.int32, 1, None)
    shared, blocks = prefix_table.data_ptr(), prefix_table.shape[0]
    if isinstance(prefix_len, torch.Tensor):
      if prefix_len.dtype != torch.int32 or prefix_len.device != device or (
          prefix_len.numel() != 1):
        raise ValueError("prefix_len must be an int or one int32 on the pages' device")
      length_ptr, length = prefix_len.data_ptr(), 2**31 - 1
    else:
      length = prefix_len
      if not 0 <= length <= blocks * kv.block_tokens:
        raise ValueError(f"prefix_table does not hold {prefix_len} tokens")
  if out is not None:
    _check_heads(kv, "out", out, shape)
    if not out.is_contiguous():
      raise ValueError("out must be contiguous")
  if torch.is_grad_enabled() and (q.requires_grad or (out is not None and out.requires_grad)):
    raise _no_grad_path()
  if forward_ad._current_level >= 0:
    _refuse_tangents(kv, q, out)
  lib = _native.lib()

  # a dimension of one element is never stepped over: its stride says nothing
  tail = (strides[0] if batch > 1 else 0, strides[1] if new > 1 else 0,
          strides[-2] if q_heads > 1 else 0, batch, new, q_heads, block_table.data_ptr(),
          block_table.stride(0) if batch > 1 else 0, block_table.shape[1], seq_lens.data_ptr(),
          shared, blocks, length, length_ptr, dim ** -0.5 if scale is None else scale, 0)
  # the workspace's size follows from the shapes alone
  key = (batch, new, q_heads, blocks > 0)
  nbytes = kv._workspace.get(key)
  if nbytes is None:
    n = ctypes.c_uint64()
    _native.check(lib.ts_paged_attention_workspace(
        index, kv._ref, _ATTENTION_ARGS.pack(0, 0, 0, *tail), ctypes.byref(n)), "attention: ")
    nbytes = n.value
    if len(kv._workspace) >= 1024:
      kv._workspace.clear()
    kv._workspace[key] = nbytes
  lse = None
  if stream is None:
    if out is None:
      out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if return_lse:
      lse = q.new_empty(shape[:-1], dtype=torch.float32)
    work = torch.empty(nbytes, dtype=torch.uint8, device=device)
    raw = torch._C._cuda_getCurrentRawStream(index)
  else:
    with torch.cuda.stream(stream):  # what a call allocates belongs to its stream
      if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
      if return_lse:
        lse = q.new_empty(shape[:-1], dtype=torch.float32)
      work = torch.empty(nbytes, dtype=torch.uint8, device=device)
    raw = stream.cuda_stream
  args = _ATTENTION_ARGS.pack(q.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0,
                              *tail)
  rc = lib.ts_paged_attention(index, kv._ref, args, work.data_ptr(), nbytes,
                              0 if err_flag is None else _flag(kv, err_flag), raw)
  if rc:
    _native.check(rc, "attention: ")
  return (out, lse) if return_lse else out


def paged_attention(kv: PagedKV, q: torch.Tensor, block_table: torch.Tensor,
                    seq_lens: torch.Tensor, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None, return_lse: bool = False,
                    err_flag: Optional[torch.Tensor] = None,
                    stream: Optional[torch.cuda.Stream] = None
                    ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
  """Attention of each sequence's last tokens over its pages.

  q: [batch, q_heads, head_dim], or [batch, n, q_heads, head_dim] for the last
  n tokens of each sequence.  It is made for drafted tokens: a prompt is
  answered as well, but at tens of times what its products need (4096 tokens
  1.9 ms a layer).  Query head h reads KV head
  h / (q_heads / heads).  block_table: int32 [batch, max_blocks], the pages of
  a sequence in order; seq_lens: int32 [batch], its tokens in the cache, the
  new ones included.  Query j sees the first seq_len - n + 1 + j tokens; one
  that sees none gets zeros, and none depends on a token it does not see.  scale: default head_dim ** -0.5.  With
  return_lse also returns float32 log(sum(exp(scores))) per query head (-inf
  for a query that sees nothing).  head_dim is 64 or 128.

  Tokens of a table entry outside the pages are left out, a length is cut to
  what its table row holds, and either sets err_flag (int32, on the device) to
  1 (2: a kernel gave up waiting for its own loads, the result is not valid and
  the rows it worked on are NaN).
  Nothing is read back: lengths and tables may change between replays of a
  captured call.
  """
  return _attention(kv, q, block_table, seq_lens, None, 0, scale, out, return_lse, err_flag,
                    stream)


def shared_prefix_attention(kv: PagedKV, q: torch.Tensor, prefix_table: torch.Tensor,
                            prefix_len: Union[int, torch.Tensor], block_table: torch.Tensor,
                            seq_lens: torch.Tensor, scale: Optional[float] = None,
                            out: Optional[torch.Tensor] = None, return_lse: bool = False,
                            err_flag: Optional[torch.Tensor] = None,
                            stream: Optional[torch.cuda.Stream] = None
                            ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
  """paged_attention of a batch whose sequences continue one cached prefix.

  Every query sees the first prefix_len tokens of the pages prefix_table
  (int32 [blocks]), which are read once for the whole batch, and then its
  sequence's own tokens as in paged_attention: block_table and seq_lens count
  the tokens after the prefix (a sequence with none sees the prefix alone).
  prefix_len: an int, or one int32 on the device (cut to what the table holds,
  with err_flag set).  With a length on the device the kernels and their CTAs
  are chosen for all that the table holds: give a table about as long as the
  prefix.  Pages whose size is no multiple of 8 tokens keep a prefix of many
  rows off the tensor cores of the fifth generation (four times slower).
  """
  if prefix_table is None:
    raise ValueError("prefix_table is missing: paged_attention is the form without a prefix")
  return _attention(kv, q, block_table, seq_lens, prefix_table, prefix_len, scale, out,
                    return_lse, err_flag, stream)
