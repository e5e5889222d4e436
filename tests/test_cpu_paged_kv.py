"""Refusals of the paged cache operators at the C entries and in the Python
wrappers, without a GPU: every case is an error before anything is launched,
so the addresses given here are never followed."""

import ctypes
import math

import pytest
import torch

from tpu_sync_b200 import _native, ops

BASE = 1 << 30  # an address that only range checks see


def kv(**over):
  c = _native.PagedKvC(BASE, 2 * BASE, 10, 16, 2, 128, 16 * 2 * 128, 2 * 128, 128,
                       16 * 2 * 128, 2 * 128, 128, _native.DTYPE_BF16, 0)
  for name, x in over.items():
    setattr(c, name, x)
  return c


def append_args(**over):
  a = _native.KvAppendArgs(
      k=4 * BASE, v=5 * BASE, q=6 * BASE, q_out=7 * BASE, k_token_stride=256, k_head_stride=128,
      v_token_stride=256, v_head_stride=128, q_token_stride=512, q_head_stride=128,
      q_out_token_stride=512, q_out_head_stride=128, tokens=3, q_heads=4, slots=8 * BASE,
      positions=9 * BASE, cos_sin=10 * BASE, max_position=50, cos_sin_stride=128, rotary=128,
      q_weight=11 * BASE, k_weight=12 * BASE, weight_dtype=_native.DTYPE_F32, eps=1e-6)
  for name, x in over.items():
    setattr(a, name, x)
  return a


def attention_args(**over):
  a = _native.AttentionArgs(
      q=4 * BASE, out=5 * BASE, lse=6 * BASE, q_batch_stride=512, q_token_stride=512,
      q_head_stride=128, batch=3, new_tokens=1, q_heads=4, block_table=7 * BASE,
      block_table_stride=8, max_blocks=8, seq_lens=8 * BASE, prefix_table=9 * BASE,
      prefix_blocks=4, prefix_len=60, prefix_len_dev=0, scale=0.1)
  for name, x in over.items():
    setattr(a, name, x)
  return a


def append(c, a):
  return _native.lib().ts_kv_append(0, ctypes.byref(c) if c else None,
                                    ctypes.byref(a) if a else None, None, None)


def attend(c, a, work=13 * BASE, nbytes=1 << 40):
  return _native.lib().ts_paged_attention(0, ctypes.byref(c) if c else None,
                                          ctypes.byref(a) if a else None, work, nbytes, None, None)


PAGES = [
    (dict(k_ptr=0), "null"), (dict(v_ptr=0), "null"), (dict(pages=-1), "positive"),
    (dict(block_tokens=0), "positive"), (dict(heads=0), "positive"),
    (dict(head_dim=0), "positive"), (dict(pages=2 ** 31), "too large"),
    (dict(heads=70000), "too large"), (dict(k_token_stride=128), "overlap"),
    (dict(v_page_stride=0), "overlap"), (dict(k_head_stride=64), "overlap"),
    (dict(v_token_stride=-256), "overlap"),
]


@pytest.mark.parametrize("over,word", PAGES, ids=str)
def test_pages_refused_by_both(over, word):
  for rc in (append(kv(**over), append_args()), attend(kv(**over), attention_args())):
    assert rc == _native.INVALID_ARGUMENT
    assert word in _native.last_error()


def test_other_dtypes_are_unimplemented():
  for dtype in (_native.DTYPE_F32, _native.DTYPE_U8, 9):
    assert append(kv(dtype=dtype), append_args()) == _native.UNIMPLEMENTED
    assert attend(kv(dtype=dtype), attention_args()) == _native.UNIMPLEMENTED


APPEND = [
    (dict(tokens=-1), "range"), (dict(tokens=2 ** 31), "range"), (dict(q_heads=-1), "range"),
    (dict(k=0), "null"), (dict(v=0), "null"), (dict(slots=0), "null"), (dict(q_out=0), "null"),
    (dict(q_heads=0), "null"), (dict(positions=0), "null"), (dict(rotary=0), "rotary"),
    (dict(rotary=63), "rotary"), (dict(rotary=130), "rotary"), (dict(cos_sin_stride=100), "rows"),
    (dict(max_position=-1), "rows"), (dict(weight_dtype=_native.DTYPE_F16), "weights"),
    (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"), (dict(k_token_stride=-1), "strides"),
    (dict(q_out_token_stride=0), "q_out strides"), (dict(q_out_head_stride=64), "q_out strides"),
    (dict(q_out=4 * BASE), "q itself"), (dict(q_out=6 * BASE + 2), "q itself"),
    (dict(q_out=BASE), "overlap the pages"), (dict(k=2 * BASE + 64), "overlap the pages"),
    (dict(v=BASE - 2), "overlap the pages"),
    (dict(q_out=6 * BASE, k=6 * BASE), "q itself"), (dict(q_out=6 * BASE, v=6 * BASE), "q itself"),
]


@pytest.mark.parametrize("over,word", APPEND, ids=str)
def test_append_refuses(over, word):
  assert append(kv(), append_args(**over)) == _native.INVALID_ARGUMENT
  assert word in _native.last_error()


def test_append_null_and_empty():
  assert append(None, append_args()) == _native.INVALID_ARGUMENT
  assert append(kv(), None) == _native.INVALID_ARGUMENT
  assert append(kv(), append_args(tokens=0, k=0)) == _native.OK


ATTENTION = [
    (dict(batch=-1), "non-negative"), (dict(new_tokens=-1), "non-negative"),
    (dict(q_heads=0), "non-negative"), (dict(max_blocks=-1), "non-negative"),
    (dict(prefix_blocks=-1), "non-negative"), (dict(prefix_len=-1), "non-negative"),
    (dict(q_heads=5), "multiple"), (dict(batch=1 << 25), "rows"),
    (dict(batch=1 << 20, new_tokens=1 << 10), "rows"), (dict(max_blocks=1 << 40), "too many"),
    (dict(prefix_blocks=1 << 28), "too many"), (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"), (dict(scale=math.inf), "scale"), (dict(scale=math.nan), "scale"),
    (dict(q=0), "null"), (dict(out=0), "null"), (dict(seq_lens=0), "null"),
    (dict(block_table=0), "null"), (dict(prefix_table=0), "null"),
    (dict(q_head_stride=132), "16 bytes"), (dict(q_batch_stride=-512), "16 bytes"),
    (dict(q=4 * BASE + 2), "aligned"), (dict(out=5 * BASE + 8), "aligned"),
    (dict(out=4 * BASE + 16), "overlaps"), (dict(out=BASE + 160), "overlaps"),
    (dict(out=2 * BASE), "overlaps"),
]


@pytest.mark.parametrize("over,word", ATTENTION, ids=str)
def test_attention_refuses(over, word):
  assert attend(kv(), attention_args(**over)) == _native.INVALID_ARGUMENT
  assert word in _native.last_error()


def test_attention_workspace_and_head_dim():
  n = ctypes.c_uint64()
  a = attention_args()
  fn = _native.lib().ts_paged_attention_workspace
  assert fn(0, ctypes.byref(kv()), ctypes.byref(a), ctypes.byref(n)) == _native.OK
  assert n.value > 0
  for work, nbytes in ((0, n.value), (13 * BASE + 4, n.value), (13 * BASE, n.value - 1)):
    assert attend(kv(), a, work, nbytes) == _native.INVALID_ARGUMENT
    assert "workspace" in _native.last_error()
  assert fn(0, ctypes.byref(kv()), ctypes.byref(a), None) == _native.INVALID_ARGUMENT
  assert fn(0, None, ctypes.byref(a), ctypes.byref(n)) == _native.INVALID_ARGUMENT
  assert fn(0, ctypes.byref(kv()), None, ctypes.byref(n)) == _native.INVALID_ARGUMENT
  odd = kv(head_dim=96)
  assert fn(0, ctypes.byref(odd), ctypes.byref(a), ctypes.byref(n)) == _native.UNIMPLEMENTED
  assert attend(odd, a) == _native.UNIMPLEMENTED
  assert attend(kv(k_ptr=BASE + 2), a) == _native.INVALID_ARGUMENT
  assert attend(kv(k_page_stride=16 * 2 * 128 + 4), a) == _native.INVALID_ARGUMENT
  # nothing to do is no error, and no address is looked at
  assert attend(kv(), attention_args(batch=0, q=0)) == _native.OK
  assert attend(kv(), attention_args(new_tokens=0, q=0)) == _native.OK


def test_packed_arguments_have_the_structures_layout():
  assert ops._APPEND_ARGS.size == ctypes.sizeof(_native.KvAppendArgs)
  assert ops._ATTENTION_ARGS.size == ctypes.sizeof(_native.AttentionArgs)
  for packer, cls in ((ops._APPEND_ARGS, _native.KvAppendArgs),
                      (ops._ATTENTION_ARGS, _native.AttentionArgs)):
    values = list(range(3, 3 + len(cls._fields_)))
    got = cls.from_buffer_copy(packer.pack(*values))
    assert [getattr(got, name) for name, _ in cls._fields_] == values


def test_wrappers_need_cuda_tensors():
  t = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16)
  with pytest.raises(ValueError, match="CUDA"):
    ops.PagedKV(t, t)


# Addresses that are not aligned to their elements would be misaligned accesses.
UNALIGNED_APPEND = [
    dict(k=4 * BASE + 1), dict(v=5 * BASE + 1), dict(q=6 * BASE + 1), dict(q_out=7 * BASE + 1),
    dict(slots=8 * BASE + 4), dict(positions=9 * BASE + 4), dict(cos_sin=10 * BASE + 2),
    dict(q_weight=11 * BASE + 2), dict(k_weight=12 * BASE + 2),
    dict(k_weight=12 * BASE + 1, weight_dtype=_native.DTYPE_BF16),
]
UNALIGNED_ATTENTION = [
    dict(lse=6 * BASE + 2), dict(block_table=7 * BASE + 1), dict(seq_lens=8 * BASE + 2),
    dict(prefix_table=9 * BASE + 2), dict(prefix_len_dev=10 * BASE + 3),
]


def test_unaligned_addresses_are_refused():
  for over in UNALIGNED_APPEND:
    assert append(kv(), append_args(**over)) == _native.INVALID_ARGUMENT, over
    assert "aligned" in _native.last_error()
  for over in UNALIGNED_ATTENTION:
    assert attend(kv(), attention_args(**over)) == _native.INVALID_ARGUMENT, over
    assert "aligned" in _native.last_error()
  for over in (dict(k_ptr=BASE + 1), dict(v_ptr=2 * BASE + 1)):
    for rc in (append(kv(**over), append_args()), attend(kv(**over), attention_args())):
      assert rc == _native.INVALID_ARGUMENT
      assert "aligned" in _native.last_error()
  lib, flag = _native.lib(), 13 * BASE + 2
  assert lib.ts_kv_append(0, ctypes.byref(kv()), ctypes.byref(append_args()), flag,
                          None) == _native.INVALID_ARGUMENT
  assert "aligned" in _native.last_error()
  assert lib.ts_paged_attention(0, ctypes.byref(kv()), ctypes.byref(attention_args()), 13 * BASE,
                                1 << 40, flag, None) == _native.INVALID_ARGUMENT
  assert "aligned" in _native.last_error()


# Queries rotated in place whose elements are also keys' or values' (reads of one
# race with writes of the other): by heads, by rows, by a part of a head.
SHARED_IN_PLACE = [
    dict(k=6 * BASE + 2 * 256, k_token_stride=512),             # heads 2 and 3 of q
    dict(v=6 * BASE + 2 * 384, v_token_stride=512),             # heads 3 and 4: one is q's
    dict(k=6 * BASE + 2 * 512),                                  # q's next row
    dict(v=6 * BASE + 2 * 511, v_token_stride=768, q_token_stride=768, q_out_token_stride=768),
    dict(k=6 * BASE - 2 * 255, k_token_stride=768, q_token_stride=768, q_out_token_stride=768),
    # heads of [token, head, 3, 128]: k one element too early
    dict(k=6 * BASE + 2 * 127, k_head_stride=384, k_token_stride=1536, q_head_stride=384,
         q_token_stride=1536, q_out_head_stride=384, q_out_token_stride=1536),
    # heads before tokens: k is q's last head and one more
    dict(k=6 * BASE + 2 * 3 * 384, k_head_stride=384, k_token_stride=128, q_head_stride=384,
         q_token_stride=128, q_out_head_stride=384, q_out_token_stride=128),
]


@pytest.mark.parametrize("over", SHARED_IN_PLACE, ids=str)
def test_in_place_queries_that_are_keys_or_values(over):
  assert append(kv(), append_args(q_out=6 * BASE, **over)) == _native.INVALID_ARGUMENT
  assert "q itself" in _native.last_error()


# K and V pages that share elements: the two scatters of an append would race.
SHARED_PAGES = [
    dict(v_ptr=BASE), dict(v_ptr=BASE + 2 * 128), dict(v_ptr=BASE + 2 * 16 * 256),
    dict(k_ptr=2 * BASE - 2 * (9 * 16 * 256 + 8 * 256)),
    # [pages, 2, 16, 2, 128] with V a token early
    dict(k_page_stride=8192, v_page_stride=8192, v_ptr=BASE + 2 * 15 * 256),
    # [pages, 16, 2, 2 x 128] with V an element early
    dict(v_ptr=BASE + 2 * 127, k_page_stride=8192, v_page_stride=8192, k_token_stride=512,
         v_token_stride=512, k_head_stride=256, v_head_stride=256),
]


@pytest.mark.parametrize("over", SHARED_PAGES, ids=str)
def test_append_refuses_pages_of_k_that_are_v(over):
  assert append(kv(**over), append_args()) == _native.INVALID_ARGUMENT
  assert "K and V pages overlap" in _native.last_error()


def test_strides_whose_products_pass_64_bits():
  """Overlaps hidden by a product that would wrap."""
  # 3 heads 2^62 apart: the span of 2^63 + 128 is past the token stride, wrapped it was negative
  over = dict(heads=3, k_head_stride=1 << 62, k_token_stride=(1 << 62) + 8, v_token_stride=384,
              v_page_stride=16 * 384, k_page_stride=(1 << 62) + 16)
  for rc in (append(kv(**over), append_args(q=0)),
             attend(kv(**over), attention_args(q_heads=3))):
    assert rc == _native.INVALID_ARGUMENT
    assert "page strides overlap" in _native.last_error()
  over = dict(q_heads=4, q_out_head_stride=1 << 62, q_out_token_stride=1 << 61)
  assert append(kv(), append_args(**over)) == _native.INVALID_ARGUMENT
  assert "q_out strides" in _native.last_error()
