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

import contextlib
import ctypes
from typing import List, Optional, Sequence, Tuple, Union

import numpy as np
import torch

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


def _on(stream: Optional[torch.cuda.Stream]):
  """What a call allocates or converts belongs to the stream it runs on."""
  return contextlib.nullcontext() if stream is None else torch.cuda.stream(stream)


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
    self.k_pages, self.v_pages, self.head_major = k_pages, v_pages, bool(head_major)
    self.device, self.dtype = k_pages.device, k_pages.dtype
    tok, head = (2, 1) if head_major else (1, 2)
    self.pages, self.block_tokens = k_pages.shape[0], k_pages.shape[tok]
    self.heads, self.head_dim = k_pages.shape[head], k_pages.shape[3]
    self._c = _native.PagedKvC(
        k_pages.data_ptr(), v_pages.data_ptr(), self.pages, self.block_tokens, self.heads,
        self.head_dim, k_pages.stride(0), k_pages.stride(tok), k_pages.stride(head),
        v_pages.stride(0), v_pages.stride(tok), v_pages.stride(head),
        _PAGE_DTYPES[self.dtype], 0)
    self._ref = ctypes.byref(self._c)
    self._index = self.device.index


def _check_heads(kv: PagedKV, name: str, t: torch.Tensor, tokens: int, heads: Optional[int]):
  if t.dim() != 3 or t.shape[0] != tokens or t.shape[2] != kv.head_dim or (
      heads is not None and t.shape[1] != heads):
    raise ValueError(f"{name} must be [{tokens}, {heads or 'heads'}, {kv.head_dim}], got "
                     f"{list(t.shape)}")
  _check_like(kv, name, t)


def _check_like(kv: PagedKV, name: str, t: torch.Tensor):
  if t.dtype != kv.dtype or t.device != kv.device:
    raise ValueError(f"{name} must have the pages' dtype and device")
  if t.stride(-1) != 1 and t.shape[-1] > 1:
    raise ValueError(f"the last dimension of {name} must be contiguous")
  if t.requires_grad and torch.is_grad_enabled():
    raise ValueError(f"{name} requires grad: the paged cache operators have no backward pass")


def _check_index(name: str, t: torch.Tensor, dtype: torch.dtype, dims: int, device):
  if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.dim() != dims or t.device != device:
    raise ValueError(f"{name} must be a {dims}-dimensional {dtype} tensor on {device}")
  if t.stride(-1) != 1 and t.shape[-1] > 1:
    raise ValueError(f"the last dimension of {name} must be contiguous")


def _check_flag(kv: PagedKV, err_flag: Optional[torch.Tensor]) -> int:
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
  rotation.  q_out may be q itself; its padding rows stay as they were (a new
  one has zeros there).

  The slots of one call are distinct: where two tokens name one slot, it is not
  defined which of them stays.  A slot past the pages or a position past
  cos_sin writes nothing for its token and sets err_flag (int32, on the device)
  to 1.
  """
  tokens = k.shape[0] if k.dim() else 0
  _check_heads(kv, "k", k, tokens, kv.heads)
  _check_heads(kv, "v", v, tokens, kv.heads)
  _check_index("slots", slots, torch.int64, 1, kv.device)
  if slots.shape[0] != tokens:
    raise ValueError(f"slots must hold {tokens} entries")
  flag = _check_flag(kv, err_flag)
  a = _native.KvAppendArgs()
  a.k, a.v, a.slots, a.tokens = k.data_ptr(), v.data_ptr(), slots.data_ptr(), tokens
  a.k_token_stride, a.k_head_stride, _ = k.stride()
  a.v_token_stride, a.v_head_stride, _ = v.stride()
  if cos_sin is not None:
    _check_index("positions", positions, torch.int64, 1, kv.device)
    _check_index("cos_sin", cos_sin, torch.float32, 2, kv.device)
    if positions.shape[0] != tokens:
      raise ValueError(f"positions must hold {tokens} entries")
    a.positions, a.cos_sin = positions.data_ptr(), cos_sin.data_ptr()
    a.max_position, a.rotary = cos_sin.shape
    a.cos_sin_stride = cos_sin.stride(0) if a.max_position > 1 else a.rotary
    a.interleaved = bool(interleaved)
    if a.max_position == 0:
      raise ValueError("cos_sin has no rows")
  elif interleaved or positions is not None:
    raise ValueError("positions and interleaved need cos_sin")
  if q_weight is not None or k_weight is not None:
    w = q_weight if q_weight is not None else k_weight
    if w.dtype not in (kv.dtype, torch.float32):
      raise ValueError("norm weights must be float32 or of the pages' dtype")
    for name, t in (("q_weight", q_weight), ("k_weight", k_weight)):
      if t is None:
        continue
      _check_index(name, t, w.dtype, 1, kv.device)
      if t.shape[0] != kv.head_dim:
        raise ValueError(f"{name} must hold {kv.head_dim} entries")
      if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires grad: the paged cache operators have no backward pass")
    a.q_weight = q_weight.data_ptr() if q_weight is not None else 0
    a.k_weight = k_weight.data_ptr() if k_weight is not None else 0
    a.weight_dtype = _TORCH_TO_TS[w.dtype]
    a.eps = eps
    if q_weight is not None and q is None:
      raise ValueError("q_weight needs q")
  if q is not None:
    _check_heads(kv, "q", q, tokens, None)
    if q_out is None:
      with _on(stream):
        q_out = torch.empty(q.shape, dtype=kv.dtype, device=kv.device)
      a.zero_padding = 1
    else:
      _check_heads(kv, "q_out", q_out, tokens, q.shape[1])
    a.q, a.q_out, a.q_heads = q.data_ptr(), q_out.data_ptr(), q.shape[1]
    a.q_token_stride, a.q_head_stride, _ = q.stride()
    a.q_out_token_stride, a.q_out_head_stride, _ = q_out.stride()
    if a.q_heads == 0:
      raise ValueError("q needs at least one head")
  elif q_out is not None:
    raise ValueError("q_out needs q")
  _native.check(_native.lib().ts_kv_append(kv._index, kv._ref, ctypes.byref(a), flag,
                                           _stream(stream, kv.device)), "kv_append: ")
  return q_out


def _attention(kv, q, block_table, seq_lens, prefix_table, prefix_len, scale, out, return_lse,
               err_flag, stream):
  if q.dim() == 3:
    batch, q_heads, dim = q.shape
    new = 1
  elif q.dim() == 4:
    batch, new, q_heads, dim = q.shape
  else:
    raise ValueError("q must be [batch, q_heads, head_dim] or [batch, new_tokens, q_heads, "
                     "head_dim]")
  if dim != kv.head_dim or q_heads == 0:
    raise ValueError(f"q heads must have {kv.head_dim} elements")
  _check_like(kv, "q", q)
  _check_index("block_table", block_table, torch.int32, 2, kv.device)
  _check_index("seq_lens", seq_lens, torch.int32, 1, kv.device)
  if block_table.shape[0] != batch or seq_lens.shape[0] != batch:
    raise ValueError(f"block_table and seq_lens must hold {batch} sequences")
  flag = _check_flag(kv, err_flag)
  a = _native.AttentionArgs()
  a.q, a.batch, a.new_tokens, a.q_heads = q.data_ptr(), batch, new, q_heads
  strides = q.stride()
  # a dimension of one element is never stepped over: its stride says nothing
  a.q_batch_stride = strides[0] if batch > 1 else 0
  a.q_token_stride = strides[1] if new > 1 else 0
  a.q_head_stride = strides[-2] if q_heads > 1 else 0
  a.block_table, a.max_blocks = block_table.data_ptr(), block_table.shape[1]
  a.block_table_stride = block_table.stride(0) if batch > 1 else 0
  a.seq_lens = seq_lens.data_ptr()
  a.scale = dim ** -0.5 if scale is None else scale
  if prefix_table is not None:
    _check_index("prefix_table", prefix_table, torch.int32, 1, kv.device)
    a.prefix_table, a.prefix_blocks = prefix_table.data_ptr(), prefix_table.shape[0]
    if isinstance(prefix_len, torch.Tensor):
      if prefix_len.dtype != torch.int32 or prefix_len.device != kv.device or (
          prefix_len.numel() != 1):
        raise ValueError("prefix_len must be an int or one int32 on the pages' device")
      a.prefix_len_dev, a.prefix_len = prefix_len.data_ptr(), 2**31 - 1
    else:
      if not 0 <= prefix_len <= a.prefix_blocks * kv.block_tokens:
        raise ValueError(f"prefix_table does not hold {prefix_len} tokens")
      a.prefix_len = prefix_len
  if out is not None:
    _check_like(kv, "out", out)
    if out.shape != q.shape or not out.is_contiguous():
      raise ValueError("out must be contiguous and of q's shape")
  lib = _native.lib()
  nbytes = ctypes.c_uint64()
  _native.check(lib.ts_paged_attention_workspace(kv._index, kv._ref, ctypes.byref(a),
                                                 ctypes.byref(nbytes)), "attention: ")
  with _on(stream):
    if out is None:
      out = torch.empty(q.shape, dtype=kv.dtype, device=kv.device)
    lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=kv.device) if return_lse else None
    work = torch.empty(nbytes.value, dtype=torch.uint8, device=kv.device)
  a.out = out.data_ptr()
  if return_lse:
    a.lse = lse.data_ptr()
  _native.check(lib.ts_paged_attention(kv._index, kv._ref, ctypes.byref(a), work.data_ptr(),
                                       nbytes.value, flag, _stream(stream, kv.device)),
                "attention: ")
  return (out, lse) if return_lse else out


def paged_attention(kv: PagedKV, q: torch.Tensor, block_table: torch.Tensor,
                    seq_lens: torch.Tensor, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None, return_lse: bool = False,
                    err_flag: Optional[torch.Tensor] = None,
                    stream: Optional[torch.cuda.Stream] = None
                    ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
  """Attention of each sequence's last tokens over its pages.

  q: [batch, q_heads, head_dim], or [batch, n, q_heads, head_dim] for the last
  n tokens of each sequence (drafted tokens); query head h reads KV head
  h / (q_heads / heads).  block_table: int32 [batch, max_blocks], the pages of
  a sequence in order; seq_lens: int32 [batch], its tokens in the cache, the
  new ones included.  Query j sees the first seq_len - n + 1 + j tokens; one
  that sees none gets zeros.  scale: default head_dim ** -0.5.  With
  return_lse also returns float32 log(sum(exp(scores))) per query head (-inf
  for a query that sees nothing).  head_dim is 64 or 128.

  Tokens of a table entry outside the pages are left out, a length is cut to
  what its table row holds, and either sets err_flag (int32, on the device) to
  1.  Nothing is read back: lengths and tables may change between replays of a
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
  with err_flag set).
  """
  return _attention(kv, q, block_table, seq_lens, prefix_table, prefix_len, scale, out,
                    return_lse, err_flag, stream)
