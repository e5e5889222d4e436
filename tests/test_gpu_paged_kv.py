"""Paged cache operators against the formulas in 64 bits.

u = finfo(dtype).eps / 2 bounds one rounding to the pages' dtype.

kv_append rounds once: |got - want| <= u |want| + 2^-20 (|want| + max |x|),
with x the normed head: 32-bit products, sums and the reciprocal root are a
few steps of 2^-24 of the head's largest element.

Attention rounds every probability to the pages' dtype (relative u) before the
product with V, and the result (u): |got - want| <= u (A + |want|) + c A with
A = sum p_i |v_i|.  c = 2^-15 covers the 32-bit scores: |x| 2^-24 for each of
the few roundings of a score of up to |x| ~ 60 (products and sums of head_dim
terms, the scaling, the subtraction of the maximum).  fp16 probabilities
under 2^-14 are off by up to 2^-25 absolutely: + 2^-25 sum |v_i|.  lse is held
in 32 bits: 2^-15 absolutely by the same count.

Whatever the operators must not read (pages of no table, tokens past a length,
unused table entries) is NaN or out of range.
"""

import ctypes
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from tpu_sync_b200 import KVCacheManager, _native, ops

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
BF, FP = torch.bfloat16, torch.float16


def gen(seed):
  return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape, std=1.0, dtype=torch.float32):
  return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


# -- append -------------------------------------------------------------------


def rotation_table(positions, rotary, base=10000.0):
  f = base ** (-torch.arange(0, rotary, 2, device="cuda", dtype=torch.float64) / rotary)
  a = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * f
  return torch.cat([a.cos(), a.sin()], 1).float()


def want_head(x, w, eps, row, interleaved):
  """One batch of heads [t, h, d] in 64 bits; row [t, rotary] or None."""
  x = x.double()
  if w is not None:
    x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
  big = x.abs().amax(-1, keepdim=True)
  if row is not None:
    half = row.shape[1] // 2
    c, s = row.double()[:, None, :half], row.double()[:, None, half:]
    ia = torch.arange(half, device="cuda") * (2 if interleaved else 1)
    ib = ia + (1 if interleaved else half)
    y = x.clone()
    y[..., ia] = x[..., ia] * c - x[..., ib] * s
    y[..., ib] = x[..., ib] * c + x[..., ia] * s
    x = y
  return x, big


def close(got, want, big, dtype):
  tol = U[dtype] * want.abs() + 2.0 ** -20 * (want.abs() + big)
  return bool(((got.double() - want).abs() <= tol).all())


APPEND = [
    # tokens, q heads, kv heads, d, rotary, block tokens, head major, interleaved, norm, dtype
    (1, 32, 8, 128, 128, 16, False, False, False, BF),
    (7, 32, 8, 128, 128, 16, False, False, True, BF),
    (33, 8, 1, 128, 64, 64, True, False, True, FP),
    (19, 4, 2, 64, 64, 16, False, True, True, BF),
    (64, 5, 5, 64, 32, 8, True, True, False, FP),
    (5, 3, 1, 256, 256, 16, False, False, True, BF),
    (11, 2, 1, 256, 64, 1, False, True, True, FP),
    (9, 6, 2, 80, 80, 16, False, False, True, BF),    # no vector path: 80 elements
    (9, 6, 3, 96, 24, 3, True, False, True, FP),      # rotary / 2 not a multiple of 8
    (3, 1, 1, 2, 2, 5, False, False, False, BF),
    (4, 1, 1, 33, 32, 5, False, True, True, FP),      # odd head
    (300, 28, 4, 128, 128, 32, False, False, False, BF),
    (3000, 2, 2, 128, 128, 32, False, False, True, FP),
]


@pytest.mark.parametrize("case", APPEND, ids=str)
@pytest.mark.parametrize("packed", [True, False])
def test_append(cuda, case, packed):
  t, hq, hk, d, rotary, bt, major, inter, norm, dt = case
  g = gen(1)
  pages = t // bt + 5
  shape = (pages, hk, bt, d) if major else (pages, bt, hk, d)
  kp, vp = rand(g, *shape, dtype=dt), rand(g, *shape, dtype=dt)
  before = kp.clone(), vp.clone()
  if packed:
    qkv = rand(g, t, (hq + 2 * hk) * d, dtype=dt)
    q, k, v = (x.view(t, -1, d) for x in qkv.split([hq * d, hk * d, hk * d], 1))
  else:  # head-first projections: the token dimension is the inner stride
    q, k, v = (rand(g, h, t, d, dtype=dt).transpose(0, 1) for h in (hq, hk, hk))
  slots = torch.randperm(pages * bt, generator=g, device="cuda")[:t].clone()
  pad = torch.rand(t, generator=g, device="cuda") < 0.2
  slots[pad] = -1 - torch.arange(int(pad.sum()), device="cuda")
  table = rotation_table(500, rotary)
  pos = torch.randint(0, 500, (t,), generator=g, device="cuda")
  pos[pad] = -7  # a padding token's position is not looked at
  wq = rand(g, d, dtype=dt) if norm else None
  wk = rand(g, d, dtype=dt) if norm else None
  err = torch.zeros(1, dtype=torch.int32, device="cuda")
  got = ops.kv_append(ops.PagedKV(kp, vp, head_major=major), k, v, slots, q=q, positions=pos,
                      cos_sin=table, interleaved=inter, q_weight=wq, k_weight=wk, eps=1e-5,
                      err_flag=err)
  assert int(err) == 0
  live = slots >= 0
  row = table[pos[live]]
  want, big = want_head(q[live], wq, 1e-5, row, inter)
  assert close(got[live], want, big, dt)
  assert (got[~live] == 0).all()
  want, big = want_head(k[live], wk, 1e-5, row, inter)
  view = [x.transpose(1, 2) if major else x for x in (kp, vp, *before)]
  at = slots[live] // bt, slots[live] % bt
  assert close(view[0][at], want, big, dt)
  assert torch.equal(view[1][at], v[live])
  # nothing else in the pages was touched
  for now, was in ((view[0], view[2]), (view[1], view[3])):
    now, was = now.clone(), was.clone()
    now[at] = 0
    was[at] = 0
    assert torch.equal(now, was)


def test_append_plain_copy_and_single_norm(cuda):
  """Without a table or weights keys are copied bit for bit; either norm alone is allowed."""
  g = gen(2)
  kp, vp = torch.zeros(4, 16, 2, 64, dtype=BF, device="cuda"), torch.zeros(
      4, 16, 2, 64, dtype=BF, device="cuda")
  kv = ops.PagedKV(kp, vp)
  k, v, q = (rand(g, 10, h, 64, dtype=BF) for h in (2, 2, 6))
  slots = torch.arange(13, 23, device="cuda")
  assert ops.kv_append(kv, k, v, slots) is None
  assert torch.equal(kp.view(-1, 2, 64)[13:23], k) and torch.equal(vp.view(-1, 2, 64)[13:23], v)
  got = ops.kv_append(kv, k, v, slots, q=q)
  assert torch.equal(got, q)
  w = rand(g, 64)  # float32 weights
  got = ops.kv_append(kv, k, v, slots, q=q, q_weight=w, eps=0.0)
  assert close(got, *want_head(q, w, 0.0, None, False), BF)
  assert torch.equal(kp.view(-1, 2, 64)[13:23], k)
  ops.kv_append(kv, k, v, slots, k_weight=w)
  assert close(kp.view(-1, 2, 64)[13:23], *want_head(k, w, 1e-6, None, False), BF)


@pytest.mark.parametrize("d", [64, 72])
def test_append_in_place_padding_and_bad_places(cuda, d):
  """q_out = q; rows of padding, of slots past the pages and of positions past the table stay
  as they were; the last two raise the flag."""
  g = gen(3)
  kp, vp = (torch.zeros(3, 2, 16, d, dtype=FP, device="cuda") for _ in range(2))
  kv = ops.PagedKV(kp, vp, head_major=True)
  qkv = rand(g, 6, 8 * d, dtype=FP)
  q, k, v = (x.view(6, -1, d) for x in qkv.split([4 * d, 2 * d, 2 * d], 1))
  q0 = q.clone()
  table = rotation_table(40, 32)
  err = torch.zeros(1, dtype=torch.int32, device="cuda")
  slots = torch.tensor([5, -1, 47, 48, 9, 10], device="cuda")
  pos = torch.tensor([39, 3, 0, 1, 40, 2], device="cuda")
  got = ops.kv_append(kv, k, v, slots, q=q, positions=pos, cos_sin=table, q_out=q, err_flag=err)
  assert got is q and int(err) == 1
  good = [0, 2, 5]
  want, big = want_head(q0[good], None, 0, table[pos[good]], False)
  assert close(q[good], want, big, FP)
  assert torch.equal(q[[1, 3, 4]], q0[[1, 3, 4]])
  written = vp.transpose(1, 2).reshape(48, 2, d).abs().sum((1, 2)).nonzero()[:, 0].tolist()
  assert written == [5, 10, 47]
  err.zero_()
  ops.kv_append(kv, k, v, torch.tensor([2 ** 40, 1, 2, 3, 4, 2 ** 62], device="cuda"),
                err_flag=err)
  assert int(err) == 1


def test_append_no_tokens(cuda):
  kp = torch.zeros(2, 16, 2, 64, dtype=BF, device="cuda")
  kv = ops.PagedKV(kp, kp.clone())
  e = torch.zeros(0, 2, 64, dtype=BF, device="cuda")
  out = ops.kv_append(kv, e, e, torch.zeros(0, dtype=torch.int64, device="cuda"), q=e)
  assert out.shape == (0, 2, 64)


def test_append_joint_cache_and_unaligned_views(cuda):
  """K and V as views of one [pages, 2, ...] tensor; views that start at odd elements."""
  g = gen(4)
  joint = torch.zeros(5, 2, 16, 2, 64, dtype=BF, device="cuda")
  kv = ops.PagedKV(joint[:, 0], joint[:, 1])
  buf = rand(g, 9, 1 + 2 * 2 * 65, dtype=BF)
  k = buf[:, 1:131].view(9, 2, 65)[..., :64]
  v = buf[:, 131:].view(9, 2, 65)[..., 1:]
  slots = torch.tensor([0, 79, 3, 17, 40, 41, 42, 15, 16], device="cuda")
  ops.kv_append(kv, k, v, slots)
  assert torch.equal(joint[:, 0][slots // 16, slots % 16], k)
  assert torch.equal(joint[:, 1][slots // 16, slots % 16], v)


# -- attention ----------------------------------------------------------------


def build(seed, dt, hq, hk, d, bt, major, n, lens, prefix=None, std=2.0):
  """A poisoned pool, tables whose unused entries are out of range, and queries."""
  g = gen(seed)
  b = len(lens)
  need = [-(-max(l, 0) // bt) for l in lens]
  npre = -(-(prefix or 0) // bt)
  pages = sum(need) + npre + 3
  perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
  width = max(need + [0]) + 2
  table = torch.full((b, width), 2 ** 31 - 1, dtype=torch.int32, device="cuda")
  at = 0
  pools = [torch.full((pages, bt, hk, d), math.nan, dtype=dt, device="cuda") for _ in range(2)]
  own, shared = [], None

  def fill(ids, count):
    seqs = []
    for pool in pools:
      x = rand(g, len(ids) * bt, hk, d, dtype=dt)[:count]
      flat = torch.full((len(ids) * bt, hk, d), math.nan, dtype=dt, device="cuda")
      flat[:count] = x
      pool[ids.long()] = flat.view(len(ids), bt, hk, d)
      seqs.append(x.double())
    return seqs

  for i in range(b):
    ids = perm[at:at + need[i]]
    at += need[i]
    table[i, :need[i]] = ids
    own.append(fill(ids, max(lens[i], 0)))
  ptable = None
  if prefix is not None:
    ptable = perm[at:at + npre]
    shared = fill(ptable, prefix)
  if major:
    pools = [p.transpose(1, 2).contiguous() for p in pools]
  q = rand(g, b, n, hq, d, std=std, dtype=dt)
  lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
  return pools, table, lens_t, ptable, q, own, shared


def check(got, lse, q, own, shared, lens, hk, dt, scale=None):
  b, n, hq, d = q.shape
  g = hq // hk
  scale = d ** -0.5 if scale is None else scale
  got, lse = got.view(b, n, hq, d), lse.view(b, n, hq)
  for i in range(b):
    for j in range(n):
      seen = max(0, lens[i] - n + 1 + j)
      k, v = own[i][0][:seen], own[i][1][:seen]
      if shared is not None:
        k, v = torch.cat([shared[0], k]), torch.cat([shared[1], v])
      if k.shape[0] == 0:
        assert (got[i, j] == 0).all() and (lse[i, j] == -math.inf).all()
        continue
      x = torch.einsum("hgd,thd->hgt", q[i, j].double().view(hk, g, d), k) * scale
      want_lse = torch.logsumexp(x, -1).view(hq)
      p = torch.softmax(x, -1)
      want = torch.einsum("hgt,thd->hgd", p, v).reshape(hq, d)
      size = torch.einsum("hgt,thd->hgd", p, v.abs()).reshape(hq, d)
      tol = U[dt] * (size + want.abs()) + 2.0 ** -15 * size
      if dt == FP:
        tol += 2.0 ** -25 * v.abs().sum(0).repeat_interleave(g, 0)
      off = (got[i, j].double() - want).abs()
      assert bool((off <= tol).all()), (i, j, float((off / tol).max()))
      assert float((lse[i, j].double() - want_lse).abs().max()) <= 2.0 ** -15


ATTENTION = [
    # q heads, kv heads, d, block tokens, head major, new tokens, lengths
    (32, 8, 128, 16, False, 1, [1]),
    (32, 8, 128, 16, False, 1, [0, 1, 15, 16, 17, 63, 64, 65, 500]),
    (8, 1, 128, 64, False, 1, [1000, 0, 3]),
    (8, 8, 64, 16, True, 1, [129, 64, 2]),
    (12, 2, 64, 1, False, 1, [37, 0, 66]),
    (28, 4, 128, 48, True, 2, [1, 2, 48, 49, 200]),
    (8, 2, 128, 5, False, 3, [2, 0, 3, 77]),
    (16, 2, 64, 16, False, 5, [4, 5, 6, 300]),      # 40 rows: two 32-row tiles
    (32, 1, 128, 16, False, 1, [70, 700]),           # 32 rows
    (6, 2, 128, 128, True, 1, [300, 1]),
    (32, 8, 128, 16, False, 1, [20000]),
    (2, 1, 64, 16, False, 1, [(37 * i) % 90 for i in range(333)]),
]


@pytest.mark.parametrize("dt", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("case", ATTENTION, ids=str)
def test_paged_attention(cuda, case, dt):
  hq, hk, d, bt, major, n, lens = case
  pools, table, lens_t, _, q, own, _ = build(5, dt, hq, hk, d, bt, major, n, lens)
  err = torch.zeros(1, dtype=torch.int32, device="cuda")
  out, lse = ops.paged_attention(ops.PagedKV(*pools, head_major=major), q, table, lens_t,
                                 return_lse=True, err_flag=err)
  assert int(err) == 0
  check(out, lse, q, own, None, lens, hk, dt)
  if n == 1:  # the form for single tokens
    again = ops.paged_attention(ops.PagedKV(*pools, head_major=major), q[:, 0], table, lens_t)
    assert again.shape == (len(lens), hq, d) and torch.equal(again, out[:, 0])


PREFIX = [
    # q heads, kv heads, d, block tokens, head major, new tokens, prefix, lengths
    (32, 8, 128, 16, False, 1, 1000, [1, 60, 0, 7]),
    (8, 1, 128, 64, False, 3, 130, [3, 100, 1, 0, 65]),
    (4, 4, 64, 16, True, 1, 16, [5]),
    (6, 2, 128, 16, False, 1, 0, [5, 0]),
    (12, 2, 64, 5, False, 2, 77, [0, 1, 2, 90]),
    (32, 8, 128, 16, False, 1, 129, [(11 * i) % 70 for i in range(70)]),   # 280 rows per head
    (16, 1, 64, 32, False, 1, 3001, [(7 * i) % 40 for i in range(50)]),    # 800 rows per head
    (8, 2, 128, 128, True, 4, 515, [4 + i for i in range(17)]),
    (8, 2, 128, 256, False, 1, 700, [4 + i for i in range(70)]),
    (32, 8, 128, 16, False, 1, 6000, [17, 33]),
    # many rows and pages of other than a power of two tokens: loads of 8 and 16 tokens
    (8, 1, 128, 24, False, 1, 500, [3, 0, 25, 49, 7] * 4),
    (12, 1, 64, 48, True, 1, 1111, [48, 1, 0, 2, 95, 96, 97] * 2),
    (10, 1, 128, 136, False, 2, 300, [2, 137, 0, 5, 1] * 2),
    (40, 1, 128, 20, False, 1, 260, [21, 3, 0, 1]),     # 20 tokens: not in whole groups of 8
    # fewer rows, where the walk reads the prefix: 24, 40, 64 and 112 of them
    (24, 1, 128, 16, False, 1, 1023, [40]),
    (8, 1, 128, 32, False, 1, 700, [3, 0, 25, 49, 7]),
    (8, 2, 64, 24, True, 2, 301, [2, 137, 0, 5, 1, 9, 33, 4]),
    (16, 1, 64, 16, False, 1, 97, [48, 1, 0, 2, 95, 96, 97]),
    # rows times keys that pass the border: 20 x 30000
    (20, 1, 128, 16, False, 1, 30000, [40]),
]


@pytest.mark.parametrize("dt", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("case", PREFIX, ids=str)
def test_shared_prefix_attention(cuda, case, dt):
  hq, hk, d, bt, major, n, prefix, lens = case
  pools, table, lens_t, ptable, q, own, shared = build(6, dt, hq, hk, d, bt, major, n, lens,
                                                       prefix)
  kv = ops.PagedKV(*pools, head_major=major)
  err = torch.zeros(1, dtype=torch.int32, device="cuda")
  out, lse = ops.shared_prefix_attention(kv, q, ptable, prefix, table, lens_t, return_lse=True,
                                         err_flag=err)
  assert int(err) == 0
  check(out, lse, q, own, shared, lens, hk, dt)
  # the length as a device value gives the same bits (the host then goes by what the table
  # holds, less than a page more)
  dev = torch.tensor([prefix], dtype=torch.int32, device="cuda")
  again = ops.shared_prefix_attention(kv, q, ptable, dev, table, lens_t)
  assert torch.equal(again, out)


@pytest.mark.parametrize("lens", [[700, 64], [3] * 40], ids=["few", "many"])
@pytest.mark.parametrize("std", [0.0, 30.0])
def test_flat_and_sharp_scores(cuda, std, lens):
  """All scores equal, and scores of a few hundred (one key takes nearly all the weight)."""
  pools, table, lens_t, ptable, q, own, shared = build(7, BF, 8, 2, 128, 16, False, 1, lens, 300,
                                                       std=std)
  kv = ops.PagedKV(*pools)
  out, lse = ops.shared_prefix_attention(kv, q, ptable, 300, table, lens_t, return_lse=True,
                                         scale=0.05)
  x = 30 * 0.05 * math.sqrt(128) * 5  # largest score: its 32-bit roundings bound the weights
  for i in range(len(lens)):
    k = torch.cat([shared[0], own[i][0]])
    v = torch.cat([shared[1], own[i][1]])
    s = torch.einsum("hgd,thd->hgt", q[i, 0].double().view(2, 4, 128), k) * 0.05
    p = torch.softmax(s, -1)
    want = torch.einsum("hgt,thd->hgd", p, v).reshape(8, 128)
    size = torch.einsum("hgt,thd->hgd", p, v.abs()).reshape(8, 128)
    tol = 2.0 ** -8 * (size + want.abs()) + 16 * x * 2.0 ** -24 * size
    assert bool(((out[i, 0].double() - want).abs() <= tol).all())
    assert float((lse[i, 0].double() - torch.logsumexp(s, -1).view(8)).abs().max()) <= (
        16 * x * 2.0 ** -24)


def test_bad_pages_and_lengths(cuda):
  """Tokens of table entries outside the pages are left out and lengths are cut, with the flag;
  the rest of the answer is as without them."""
  lens = [100, 40]
  pools, table, lens_t, ptable, q, own, shared = build(8, BF, 8, 2, 128, 16, False, 1, lens, 64)
  kv = ops.PagedKV(*pools)
  err = torch.zeros(1, dtype=torch.int32, device="cuda")
  bad = table.clone()
  bad[0, 2] = -1
  bad[1, 1] = pools[0].shape[0]
  out, lse = ops.paged_attention(kv, q, bad, lens_t, return_lse=True, err_flag=err)
  assert int(err) == 1
  keep = [torch.cat([torch.arange(32), torch.arange(48, 100)]),
          torch.cat([torch.arange(16), torch.arange(32, 40)])]
  cut = [[x[i][keep[n]] for i in range(2)] for n, x in enumerate(own)]
  check(out, lse, q, cut, None, [84, 24], 2, BF)
  err.zero_()
  pbad = ptable.clone()
  pbad[3] = -5
  out, lse = ops.shared_prefix_attention(kv, q, pbad, 64, table, lens_t, return_lse=True,
                                         err_flag=err)
  assert int(err) == 1
  check(out, lse, q, own, [x[:48] for x in shared], lens, 2, BF)
  # lengths past the table, and negative ones
  err.zero_()
  narrow = table[:, :3].contiguous()
  out, lse = ops.paged_attention(kv, q, narrow, lens_t, return_lse=True, err_flag=err)
  assert int(err) == 1
  check(out, lse, q, [[x[:48] for x in own[0]], own[1]], None, [48, 40], 2, BF)
  err.zero_()
  neg = torch.tensor([-3, 40], dtype=torch.int32, device="cuda")
  out, lse = ops.paged_attention(kv, q, table, neg, return_lse=True, err_flag=err)
  assert int(err) == 1
  check(out, lse, q, own, None, [0, 40], 2, BF)
  err.zero_()
  long = torch.tensor([65], dtype=torch.int32, device="cuda")
  out, lse = ops.shared_prefix_attention(kv, q, ptable, long, table, lens_t, return_lse=True,
                                         err_flag=err)
  assert int(err) == 1
  check(out, lse, q, own, shared, lens, 2, BF)


@pytest.mark.parametrize("d,bt,dt", [(128, 16, BF), (64, 64, FP)])
def test_bad_pages_of_a_prefix_with_many_rows(cuda, d, bt, dt):
  """The same for the tensor-core form (many query rows): holes in any tile, the first one
  among them, a whole tile of holes, and a length past the table."""
  lens = [(5 * i) % 23 for i in range(80)]
  n = 1000
  pools, table, lens_t, ptable, q, own, shared = build(15, dt, 8, 2, d, bt, False, 1, lens, n)
  kv = ops.PagedKV(*pools)
  err = torch.zeros(1, dtype=torch.int32, device="cuda")
  holes = [0, 3] + list(range(128 // bt, 256 // bt)) + [ptable.shape[0] - 1]
  pbad = ptable.clone()
  pbad[torch.tensor(holes)] = torch.tensor([-1, 2 ** 31 - 1, -2 ** 31, pools[0].shape[0]] * 9,
                                           dtype=torch.int32)[:len(holes)].cuda()
  out, lse = ops.shared_prefix_attention(kv, q, pbad, n, table, lens_t, return_lse=True,
                                         err_flag=err)
  assert int(err) == 1
  keep = torch.tensor([i for i in range(n) if i // bt not in holes])
  check(out, lse, q, own, [x[keep.cuda()] for x in shared], lens, 2, dt)
  err.zero_()
  all_bad = torch.full_like(ptable, -1)
  out, lse = ops.shared_prefix_attention(kv, q, all_bad, n, table, lens_t, return_lse=True,
                                         err_flag=err)
  assert int(err) == 1
  check(out, lse, q, own, None, lens, 2, dt)
  err.zero_()
  long = torch.tensor([ptable.shape[0] * bt + 1], dtype=torch.int32, device="cuda")
  whole = ptable[:n // bt]
  out, lse = ops.shared_prefix_attention(kv, q, whole, long, table, lens_t, return_lse=True,
                                         err_flag=err)
  assert int(err) == 1
  check(out, lse, q, own, [x[:n // bt * bt] for x in shared], lens, 2, dt)


@pytest.mark.parametrize("prefix", [1, 127, 128, 129, 255, 1023, 20000])
def test_prefix_lengths_with_many_rows(cuda, prefix):
  """Tile ends, one key, and more tiles than CTAs; 130, 1040 and 5600 rows per KV head,
  so that one CTA also does many short units after one another."""
  err = torch.zeros(1, dtype=torch.int32, device="cuda")
  for hq, hk, count in ((13, 1, 10), (26, 1, 40), (8, 1, 700)):
    lens = [(3 * i) % 7 for i in range(count)]
    pools, table, lens_t, ptable, q, own, shared = build(prefix, BF, hq, hk, 128, 16, True, 1,
                                                         lens, prefix)
    out, lse = ops.shared_prefix_attention(ops.PagedKV(*pools, head_major=True), q, ptable, prefix,
                                           table, lens_t, return_lse=True, err_flag=err)
    assert int(err) == 0
    check(out, lse, q, own, shared, lens, hk, BF)


def test_no_sequences_and_no_blocks(cuda):
  pools, table, lens_t, ptable, q, own, shared = build(9, FP, 8, 2, 64, 16, False, 1, [20, 3], 40)
  kv = ops.PagedKV(*pools)
  e = ops.paged_attention(kv, q[:0], table[:0], lens_t[:0])
  assert e.shape == (0, 1, 8, 64)
  none = torch.zeros(2, 0, dtype=torch.int32, device="cuda")
  zero = torch.zeros(2, dtype=torch.int32, device="cuda")
  out, lse = ops.paged_attention(kv, q, none, zero, return_lse=True)
  check(out, lse, q, own, None, [0, 0], 2, FP)
  out, lse = ops.shared_prefix_attention(kv, q, ptable, 40, none, zero, return_lse=True)
  check(out, lse, q, own, shared, [0, 0], 2, FP)
  out, lse = ops.shared_prefix_attention(kv, q, none[0], 0, table, lens_t, return_lse=True)
  check(out, lse, q, own, None, [20, 3], 2, FP)


def test_strided_queries_tables_and_joint_cache(cuda):
  lens = [90, 17, 33]
  pools, table, lens_t, ptable, q, own, shared = build(10, BF, 8, 2, 128, 16, False, 2, lens, 50)
  joint = torch.stack(pools, 1)
  kv = ops.PagedKV(joint[:, 0], joint[:, 1])
  packed = torch.full((3, 2, 12, 128), math.nan, dtype=BF, device="cuda")
  packed[:, :, 2:10] = q
  wide = torch.full((3, table.shape[1] + 5), -9, dtype=torch.int32, device="cuda")
  wide[:, :table.shape[1]] = table
  out, lse = ops.shared_prefix_attention(kv, packed[:, :, 2:10], ptable, 50,
                                         wide[:, :table.shape[1]], lens_t, return_lse=True)
  check(out, lse, q, own, shared, lens, 2, BF)
  heads_first = q.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)
  given = torch.empty_like(q)
  got = ops.paged_attention(kv, heads_first, table, lens_t, out=given)
  assert got is given
  assert torch.equal(got, ops.paged_attention(ops.PagedKV(*pools), q, table, lens_t))


def test_far_pages(cuda):
  """Pages whose byte offsets pass 32 bits."""
  pages = 70000  # 70000 x 16 x 8 x 128 x 2 bytes = 2.3 GB and 1.15e9 elements per storage
  kp = torch.empty(pages, 16, 8, 256, dtype=BF, device="cuda")[..., :128]
  vp = torch.empty(pages, 16, 8, 256, dtype=BF, device="cuda")[..., :128]
  g = gen(11)
  kv = ops.PagedKV(kp, vp)
  k, v = rand(g, 40, 8, 128, dtype=BF), rand(g, 40, 8, 128, dtype=BF)
  table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32, device="cuda")
  slots = (table[0].long()[:, None] * 16 + torch.arange(16, device="cuda")).flatten()[:40]
  ops.kv_append(kv, k, v, slots)
  q = rand(g, 1, 1, 32, 128, dtype=BF)
  lens = torch.tensor([40], dtype=torch.int32, device="cuda")
  out, lse = ops.paged_attention(kv, q, table, lens, return_lse=True)
  check(out, lse, q, [[k.double(), v.double()]], None, [40], 8, BF)
  out, lse = ops.shared_prefix_attention(kv, q, table[0], 40, table, lens * 0, return_lse=True)
  check(out, lse, q, [[k[:0].double(), v[:0].double()]], [k.double(), v.double()], [0], 8, BF)
  for count in (9, 40):  # 36 and 160 rows per KV head
    many = rand(g, count, 1, 32, 128, dtype=BF)
    out, lse = ops.shared_prefix_attention(kv, many, table[0], 40, table.repeat(count, 1),
                                           lens.repeat(count) * 0, return_lse=True)
    check(out, lse, many, [[k[:0].double(), v[:0].double()]] * count, [k.double(), v.double()],
          [0] * count, 8, BF)


def test_other_stream_and_repeatable(cuda):
  """A call on a given stream is ordered there; the same call gives the same bits."""
  lens = [900, 64, 1, 333]
  pools, table, lens_t, ptable, q, own, shared = build(12, BF, 32, 8, 128, 16, False, 1, lens,
                                                       2000)
  kv = ops.PagedKV(*pools)
  want = ops.shared_prefix_attention(kv, q, ptable, 2000, table, lens_t)
  streams = [torch.cuda.Stream() for _ in range(3)]
  torch.cuda.synchronize()
  outs = []
  for i in range(12):  # calls in flight at once, each with a workspace of its own
    s = streams[i % 3]
    outs.append(ops.shared_prefix_attention(kv, q, ptable, 2000, table, lens_t, stream=s))
  torch.cuda.synchronize()
  assert all(torch.equal(o, want) for o in outs)
  s = streams[0]
  late = torch.zeros_like(q)
  s.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(s):
    torch.cuda._sleep(20_000_000)
    late.copy_(q)
  got = ops.shared_prefix_attention(kv, late, ptable, 2000, table, lens_t, stream=s)
  s.synchronize()
  assert torch.equal(got, want)


def test_calls_from_threads(cuda):
  """Calls of several threads at once, each on its own stream, give the bits of one alone."""
  import threading
  lens = [70, 0, 333] * 7
  pools, table, lens_t, ptable, q, own, shared = build(16, FP, 16, 2, 64, 16, False, 1, lens, 500)
  kv = ops.PagedKV(*pools)
  want = ops.shared_prefix_attention(kv, q, ptable, 500, table, lens_t)
  alone = ops.paged_attention(kv, q, table, lens_t)
  torch.cuda.synchronize()
  bad = []

  def work():
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
      for _ in range(30):
        a = ops.shared_prefix_attention(kv, q, ptable, 500, table, lens_t)
        b = ops.paged_attention(kv, q, table, lens_t)
        stream.synchronize()
        if not (torch.equal(a, want) and torch.equal(b, alone)):
          bad.append(1)

  threads = [threading.Thread(target=work) for _ in range(4)]
  for t in threads:
    t.start()
  for t in threads:
    t.join()
  assert not bad


def test_first_call_is_captured(cuda):
  """A process whose first call of each operator happens while its stream is captured."""
  code = """
import torch
from tpu_sync_b200 import ops
g = torch.Generator(device="cuda").manual_seed(1)
pages = torch.randn(40, 16, 2, 64, generator=g, device="cuda").half()
kv = ops.PagedKV(pages, pages.clone())
q = torch.randn(40, 8, 64, generator=g, device="cuda").half()
k = torch.randn(3, 2, 64, generator=g, device="cuda").half()
slots = torch.tensor([5, 6, 200], device="cuda")
table = torch.arange(40, device="cuda", dtype=torch.int32).view(40, 1)
lens = torch.full((40,), 9, device="cuda", dtype=torch.int32)
shared = torch.arange(2, device="cuda", dtype=torch.int32)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
  ops.kv_append(kv, k, k, slots)
  a = ops.paged_attention(kv, q, table, lens)
  b = ops.shared_prefix_attention(kv, q, shared, 30, table, lens)
graph.replay()
torch.cuda.synchronize()
assert torch.equal(kv.k_pages.view(-1, 2, 64)[slots], k)
assert torch.equal(a, ops.paged_attention(kv, q, table, lens))
assert torch.equal(b, ops.shared_prefix_attention(kv, q, shared, 30, table, lens))
"""
  root = Path(__file__).resolve().parents[1]
  r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True,
                     timeout=120)
  assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_other_device_than_the_current_one(cuda):
  pools, table, lens_t, ptable, q, own, shared = build(17, BF, 32, 8, 128, 16, False, 1, [90] * 40,
                                                       300)
  there = lambda t: t.to("cuda:1")
  kv = ops.PagedKV(*[there(p) for p in pools])
  out = ops.shared_prefix_attention(kv, there(q), there(ptable), 300, there(table), there(lens_t))
  assert out.device == torch.device("cuda:1")
  want = ops.shared_prefix_attention(ops.PagedKV(*pools), q, ptable, 300, table, lens_t)
  assert torch.equal(out.cpu(), want.cpu())


def test_two_graphs_with_new_lengths(cuda):
  """Captured calls replay with lengths, tables and queries changed in place; two graphs keep
  their workspaces apart."""
  lens = [300, 20, 64]
  pools, table, lens_t, ptable, q, own, shared = build(13, FP, 8, 2, 128, 16, False, 1, lens, 90)
  kv = ops.PagedKV(*pools)
  plen = torch.tensor([90], dtype=torch.int32, device="cuda")
  ops.shared_prefix_attention(kv, q, ptable, plen, table, lens_t, return_lse=True)
  torch.cuda.synchronize()
  graphs = []
  for _ in range(2):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
      got = ops.shared_prefix_attention(kv, q, ptable, plen, table, lens_t, return_lse=True)
    graphs.append((graph, got))
  for new, p in (([5, 20, 0], 33), ([299, 1, 63], 90), ([0, 0, 0], 0), ([300, 20, 64], 1)):
    lens_t.copy_(torch.tensor(new, dtype=torch.int32))
    plen.fill_(p)
    q.copy_(torch.randn_like(q))
    for graph, _ in graphs:
      graph.replay()
    torch.cuda.synchronize()
    for _, (out, lse) in graphs:
      check(out, lse, q, own, [x[:p] for x in shared], new, 2, FP)


def test_append_attend_offload_reload(cuda):
  """The operators as an engine runs them: a prompt is appended, attended to, offloaded to the
  host tier, its pages reused and the prefix reloaded elsewhere; two sequences then continue it
  with one token each, whose answers equal the definition on all tokens."""
  g = gen(14)
  hq, hk, d, bt, n = 8, 2, 128, 16, 75
  shape = (24, bt, hk, d)
  kp, vp = torch.zeros(shape, dtype=BF, device="cuda"), torch.zeros(shape, dtype=BF, device="cuda")
  kv = ops.PagedKV(kp, vp)
  mgr = KVCacheManager([[kp], [vp]], host_blocks_to_allocate=16)
  table = rotation_table(128, d)
  wq, wk = rand(g, d, dtype=BF), rand(g, d, dtype=BF)

  def step(tokens, at, slots):
    qkv = rand(g, tokens, (hq + 2 * hk) * d, dtype=BF)
    q, k, v = (x.view(tokens, -1, d) for x in qkv.split([hq * d, hk * d, hk * d], 1))
    pos = torch.arange(at, at + tokens, device="cuda")
    return ops.kv_append(kv, k, v, slots, q=q, positions=pos, cos_sin=table, q_weight=wq,
                         k_weight=wk)

  def read(pages, count):
    return [x[pages.long()].reshape(-1, hk, d)[:count].double() for x in (kp, vp)]

  first = torch.tensor([3, 9, 1, 20, 7], dtype=torch.int32, device="cuda")
  spread = (first.long()[:, None] * bt + torch.arange(bt, device="cuda")).flatten()
  q = step(n, 0, spread[:n])
  lens = torch.tensor([n], dtype=torch.int32, device="cuda")
  last = q[-1:].clone()
  before, lse = ops.paged_attention(kv, last, first[None], lens, return_lse=True)
  check(before, lse, last[None], [read(first, n)], None, [n], hk, BF)

  mgr.d2h(first.tolist(), [0, 1, 2, 3, 4]).Await()
  kp[first.long()] = math.nan
  vp[first.long()] = math.nan
  moved = torch.tensor([11, 2, 16, 5, 22], dtype=torch.int32, device="cuda")
  mgr.h2d([0, 1, 2, 3, 4], moved.tolist()).Await()
  assert torch.equal(ops.paged_attention(kv, last, moved[None], lens), before)

  # two sequences go on after 64 shared tokens (whole pages), one new token each
  tails = torch.tensor([[13], [14]], dtype=torch.int32, device="cuda")
  q = torch.cat([step(1, 64, tails[i].long() * bt) for i in range(2)])
  one = torch.tensor([1, 1], dtype=torch.int32, device="cuda")
  out, lse = ops.shared_prefix_attention(kv, q, moved, 64, tails, one, return_lse=True)
  check(out, lse, q[:, None], [read(tails[i], 1) for i in range(2)], read(moved, 64), [1, 1], hk,
        BF)
  whole = torch.cat([moved[:4].repeat(2, 1), tails], 1)
  same, lse2 = ops.paged_attention(kv, q, whole, one + 64, return_lse=True)
  # both forms hold the same bound, so they differ by at most twice it
  assert float((same.double() - out.double()).abs().max()) <= 4 * U[BF] * float(
      vp[whole.long().flatten()].abs().max())
  assert float((lse - lse2).abs().max()) <= 2.0 ** -14
  mgr.close()


def test_refusals_on_the_device(cuda):
  kp = torch.zeros(4, 16, 2, 128, dtype=BF, device="cuda")
  kv = ops.PagedKV(kp, kp.clone())
  q = torch.zeros(2, 8, 128, dtype=BF, device="cuda")
  table = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
  lens = torch.ones(2, dtype=torch.int32, device="cuda")
  ok = ops.paged_attention(kv, q, table, lens)
  assert ok.shape == q.shape
  bad = [
      dict(q=q.half()), dict(q=q[..., :64]), dict(q=q[:, :7]), dict(table=table.long()),
      dict(table=table[:1]), dict(lens=lens.long()), dict(lens=lens[:1]), dict(lens=lens.cpu()),
      dict(q=q.cpu()), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf),
      dict(scale=math.nan), dict(out=q), dict(out=torch.zeros(2, 8, 64, dtype=BF, device="cuda")),
      dict(q=torch.zeros(2, 8, 136, dtype=BF, device="cuda")[..., 1:129]),
      dict(q=torch.zeros(2, 8, 132, dtype=BF, device="cuda")[..., :128]),
      dict(out=kp.view(-1, 8, 128)[:2]), dict(q=q.clone().requires_grad_()),
      dict(err_flag=torch.zeros(1, dtype=torch.int64, device="cuda")),
  ]
  for b in bad:
    with pytest.raises((ValueError, _native.NativeError)):
      ops.paged_attention(kv, b.get("q", q), b.get("table", table), b.get("lens", lens),
                          scale=b.get("scale"), out=b.get("out"), err_flag=b.get("err_flag"))
  for args in ((table[0], 49), (table[0], -1), (table, 3), (table[0].long(), 3),
               (table[0], lens), (table[0], lens[:1].long())):
    with pytest.raises((ValueError, _native.NativeError)):
      ops.shared_prefix_attention(kv, q, args[0], args[1], table, lens)
  for pages in (torch.zeros(4, 16, 2, 96, dtype=BF, device="cuda"),):
    small = ops.PagedKV(pages, pages.clone())
    with pytest.raises(_native.NativeError) as e:
      ops.paged_attention(small, q[..., :96].contiguous(), table, lens)
    assert e.value.status == "UNIMPLEMENTED"
  k = torch.zeros(3, 2, 128, dtype=BF, device="cuda")
  q3 = torch.zeros(3, 8, 128, dtype=BF, device="cuda")
  slots = torch.arange(3, device="cuda")
  cs = torch.zeros(9, 128, device="cuda")
  w = torch.ones(128, device="cuda")
  bad = [
      dict(k=k[:2]), dict(v=k.half()), dict(slots=slots.int()), dict(slots=slots[:2]),
      dict(cos_sin=cs), dict(positions=slots), dict(interleaved=True),
      dict(positions=slots, cos_sin=cs.double()), dict(positions=slots, cos_sin=cs[:, :5]),
      dict(positions=slots, cos_sin=torch.zeros(9, 130, device="cuda")),
      dict(positions=slots[:2], cos_sin=cs), dict(positions=slots, cos_sin=cs[:0]),
      dict(q_weight=w), dict(q=q3, q_weight=w[:5]), dict(q=q3, q_weight=w.half()),
      dict(q=q3, q_weight=w, k_weight=w.bfloat16()), dict(q=q3[..., :64]), dict(q_out=q3),
      dict(q=q3, q_out=q3[:, :4]), dict(q=q3, q_out=q3[:1].expand(3, 8, 128)),
      dict(k=kp[0, :3]), dict(q=q3, q_weight=w, eps=-1.0), dict(q=q3, q_weight=w, eps=math.nan),
      dict(k=k.clone().requires_grad_()), dict(k_weight=w.clone().requires_grad_()),
      dict(positions=slots, cos_sin=cs.clone().requires_grad_()),
      dict(k=q3[:, :2], q=q3, q_out=q3),
  ]
  for b in bad:
    with pytest.raises((ValueError, _native.NativeError)):
      ops.kv_append(kv, b.pop("k", k), b.pop("v", k), b.pop("slots", slots), **b)
  with torch.no_grad():
    ops.kv_append(kv, k.clone().requires_grad_(), k, slots)
  for args in ((kp, kp.half()), (kp, kp[:3]), (kp.cpu(), kp.cpu()), (kp[0], kp[0]),
               (kp.float(), kp.float()), (kp.transpose(2, 3), kp.transpose(2, 3))):
    with pytest.raises(ValueError):
      ops.PagedKV(*args)
  with pytest.raises(ValueError):
    ops.PagedKV(kp.clone().requires_grad_(), kp)
  spread = kp[:1].expand(4, 16, 2, 128)
  with pytest.raises(_native.NativeError):
    ops.paged_attention(ops.PagedKV(spread, kp), q, table, lens)


# -- values that a row does not see --------------------------------------------


def poison(seed, pools, table, lens, own, n, bt, major):
  """Infinities and NaN in V of some of the last n tokens of each sequence: single elements, and
  the whole head vector of the last one.  Keeps the pages and the 64-bit copies alike."""
  g = torch.Generator().manual_seed(seed)
  v = pools[1].transpose(1, 2) if major else pools[1]
  for i, length in enumerate(lens):
    for t in range(max(0, length - n + 1), length):
      if t < length - 1 and torch.rand((), generator=g) < 0.5:
        continue
      value = (math.inf, -math.inf, math.nan)[(i + t) % 3]
      at = slice(None) if t == length - 1 and i % 2 else int(
          torch.randint(0, v.shape[3], (), generator=g))
      v[int(table[i, t // bt]), t % bt, :, at] = value
      own[i][1][t, :, at] = value


def check_seen(got, lse, q, own, shared, lens, hk, dt):
  """check() of rows whose own visible V may not be finite: those elements are not finite, all
  others keep the bound."""
  b, n, hq, d = q.shape
  g = hq // hk
  for i in range(b):
    for j in range(n):
      seen = max(0, lens[i] - n + 1 + j)
      k, v = own[i][0][:seen], own[i][1][:seen]
      if shared is not None:
        k, v = torch.cat([shared[0], k]), torch.cat([shared[1], v])
      if k.shape[0] == 0:
        assert (got[i, j] == 0).all() and (lse[i, j] == -math.inf).all(), (i, j)
        continue
      x = torch.einsum("hgd,thd->hgt", q[i, j].double().view(hk, g, d), k) * d ** -0.5
      p = torch.softmax(x, -1)
      fine = torch.isfinite(v).all(0).repeat_interleave(g, 0)  # [hq, d]
      v = torch.where(torch.isfinite(v), v, 0.0)
      want = torch.einsum("hgt,thd->hgd", p, v).reshape(hq, d)
      size = torch.einsum("hgt,thd->hgd", p, v.abs()).reshape(hq, d)
      tol = U[dt] * (size + want.abs()) + 2.0 ** -15 * size
      if dt == FP:
        tol += 2.0 ** -25 * v.abs().sum(0).repeat_interleave(g, 0)
      off = (got[i, j].double() - want).abs()
      assert bool((off <= tol)[fine].all()), (i, j)
      assert not bool(torch.isfinite(got[i, j])[~fine].any()), (i, j)
      assert float((lse[i, j].double() - torch.logsumexp(x, -1).view(hq)).abs().max()) <= 2.0 ** -15


UNSEEN = [
    # q heads, kv heads, d, block tokens, head major, new tokens, lengths: 4, 12, 24, 32 and 80
    # rows a KV head, pages that are loaded by TMA and others
    (4, 2, 128, 16, False, 2, [1, 2, 3, 16, 17, 64, 65, 300]),
    (4, 2, 64, 5, False, 2, [1, 2, 17, 64, 65]),
    (8, 2, 128, 64, True, 3, [0, 1, 2, 3, 18, 65, 130]),
    (8, 1, 64, 16, False, 3, [1, 3, 63, 64, 65, 66, 1000]),
    (8, 1, 128, 24, False, 3, [2, 66, 191]),
    (8, 2, 128, 16, False, 8, [3, 8, 20, 70, 135]),
    (4, 1, 64, 48, True, 8, [1, 7, 9, 100]),
    (2, 1, 128, 16, False, 40, [12, 40, 100]),
    (2, 1, 64, 3, False, 40, [39, 77]),
]


@pytest.mark.parametrize("dt", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("case", UNSEEN, ids=str)
def test_values_of_later_drafts_do_not_reach_earlier_ones(cuda, case, dt):
  hq, hk, d, bt, major, n, lens = case
  pools, table, lens_t, _, q, own, _ = build(21, dt, hq, hk, d, bt, major, n, lens)
  poison(22, pools, table, lens, own, n, bt, major)
  out, lse = ops.paged_attention(ops.PagedKV(*pools, head_major=major), q, table, lens_t,
                                 return_lse=True)
  check_seen(out, lse, q, own, None, lens, hk, dt)


@pytest.mark.parametrize("hq,hk,prefix,count", [(8, 2, 100, 5), (8, 1, 600, 30)],
                         ids=["few", "many"])
def test_values_of_later_drafts_behind_a_prefix(cuda, hq, hk, prefix, count):
  lens = [(13 * i) % 140 for i in range(count)]
  pools, table, lens_t, ptable, q, own, shared = build(23, BF, hq, hk, 128, 16, False, 3, lens,
                                                       prefix)
  poison(24, pools, table, lens, own, 3, 16, False)
  out, lse = ops.shared_prefix_attention(ops.PagedKV(*pools), q, ptable, prefix, table, lens_t,
                                         return_lse=True)
  check_seen(out, lse, q, own, shared, lens, hk, BF)


# -- the flag -------------------------------------------------------------------


def test_a_flag_of_two_stays(cuda):
  """2 (the result is not valid) is not lowered to 1 by anything that is left out later."""
  lens = [60] * 40
  pools, table, lens_t, ptable, q, own, shared = build(31, BF, 8, 1, 128, 16, False, 1, lens, 300)
  kv = ops.PagedKV(*pools)
  err = torch.full((1,), 2, dtype=torch.int32, device="cuda")
  k = torch.zeros(3, 1, 128, dtype=BF, device="cuda")
  ops.kv_append(kv, k, k, torch.tensor([2 ** 40, 2 ** 41, -1], device="cuda"), err_flag=err)
  assert int(err) == 2
  bad, short = table.clone(), table[:, :2].contiguous()
  bad[:, 1] = -1
  pbad = ptable.clone()
  pbad[::3] = 2 ** 31 - 1
  long = torch.tensor([10000], dtype=torch.int32, device="cuda")
  for t, p, n in ((bad, ptable, 300), (short, ptable, 300), (table, pbad, 300),
                  (table, ptable, long)):
    ops.paged_attention(kv, q, t, lens_t, err_flag=err)
    ops.shared_prefix_attention(kv, q[:3], p, n, t[:3], lens_t[:3], err_flag=err)  # by the walk
    ops.shared_prefix_attention(kv, q, p, n, t, lens_t, err_flag=err)
    assert int(err) == 2


def test_flag_in_mapped_host_memory(cuda):
  """The C entries take a flag in host memory that the device sees."""
  kp = torch.zeros(4, 16, 2, 64, dtype=BF, device="cuda")
  kv = ops.PagedKV(kp, kp.clone())
  k = torch.zeros(2, 2, 64, dtype=BF, device="cuda")
  slots = torch.tensor([1, 64], device="cuda")
  flag = torch.zeros(1, dtype=torch.int32).pin_memory()
  args = _native.KvAppendArgs(k=k.data_ptr(), v=k.data_ptr(), k_token_stride=128,
                              k_head_stride=64, v_token_stride=128, v_head_stride=64, tokens=2,
                              slots=slots.data_ptr())
  torch.cuda.synchronize()
  for was, now in ((0, 1), (2, 2)):
    flag[0] = was
    assert _native.lib().ts_kv_append(0, kv._ref, ctypes.byref(args), flag.data_ptr(),
                                      None) == _native.OK
    torch.cuda.synchronize()
    assert int(flag) == now


# -- queries written beside or over their projections --------------------------


@pytest.mark.parametrize("layout", ["rows", "heads", "grouped", "head first", "one token"])
@pytest.mark.parametrize("out", ["itself", "columns"])
def test_append_within_one_buffer(cuda, layout, out):
  """Parts of one projection in any order of its dimensions are apart: queries are rewritten in
  place, or into columns of their own, and keys and values are read as they were."""
  g = gen(41)
  t, h, d = (1 if layout == "one token" else 37), 4, 64
  if layout in ("rows", "one token"):  # [t, (q, k, v, out) of h heads]
    buf = rand(g, t, 4 * h, d, dtype=BF)
    q, k, v, spare = (buf[:, i * h:(i + 1) * h] for i in range(4))
  elif layout == "heads":  # [t, h, (q, k, v, out)]
    buf = rand(g, t, h, 4, d, dtype=BF)
    q, k, v, spare = (buf[:, :, i] for i in range(4))
  elif layout == "grouped":  # two query heads to a KV head, side by side in its group
    buf = rand(g, t, 2, 6, d, dtype=BF)
    q, k, v, spare = buf[:, :, 0], buf[:, :, 2], buf[:, :, 3], buf[:, :, 4]
  else:
    buf = rand(g, 4 * h, t, d, dtype=BF).transpose(0, 1)
    q, k, v, spare = (buf[:, i * h:(i + 1) * h] for i in range(4))
  kp = torch.zeros(4, 16, k.shape[1], d, dtype=BF, device="cuda")
  kv = ops.PagedKV(kp, torch.zeros_like(kp))
  slots = torch.randperm(64, generator=g, device="cuda")[:t]
  pos = torch.arange(t, device="cuda")
  table = rotation_table(t, d)
  q0, k0, v0 = q.clone(), k.clone(), v.clone()
  got = ops.kv_append(kv, k, v, slots, q=q, positions=pos, cos_sin=table,
                      q_out=q if out == "itself" else spare)
  want, big = want_head(q0, None, 0, table, False)
  assert close(got, want, big, BF)
  want, big = want_head(k0, None, 0, table, False)
  assert close(kp.view(64, -1, d)[slots], want, big, BF)
  assert torch.equal(kv.v_pages.view(64, -1, d)[slots], v0)
  assert torch.equal(k, k0) and torch.equal(v, v0)
  if out == "columns":
    assert torch.equal(q, q0)


@pytest.mark.parametrize("at", [0, 1, 2, 3])
def test_append_into_joint_caches(cuda, at):
  """K and V interleaved at any dimension of one tensor are apart; one tensor as both is
  refused by the append, and may be read by the attention."""
  g = gen(42)
  shape = [4, 16, 2, 64]
  joint = torch.zeros(*shape[:at], 2, *shape[at:], dtype=FP, device="cuda")
  kp, vp = joint.select(at, 0), joint.select(at, 1)
  k, v = rand(g, 9, 2, 64, dtype=FP), rand(g, 9, 2, 64, dtype=FP)
  slots = torch.randperm(64, generator=g, device="cuda")[:9]
  ops.kv_append(ops.PagedKV(kp, vp), k, v, slots)
  assert torch.equal(kp[slots // 16, slots % 16], k)
  assert torch.equal(vp[slots // 16, slots % 16], v)
  one = ops.PagedKV(kp, kp)
  with pytest.raises(_native.NativeError, match="overlap"):
    ops.kv_append(one, k, v, slots)
  if at == 1:
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    lens = torch.tensor([16], dtype=torch.int32, device="cuda")
    q = rand(g, 1, 1, 4, 64, dtype=FP)
    out, lse = ops.paged_attention(one, q, table, lens, return_lse=True)
    check(out, lse, q, [[kp[0].double(), kp[0].double()]], None, [16], 2, FP)


def test_a_prefix_is_not_dropped_unseen(cuda):
  """No table is refused; a length on the device beside a table without blocks is cut to none,
  with the flag."""
  pools, table, lens_t, ptable, q, own, shared = build(43, BF, 4, 2, 64, 16, False, 1, [20, 3], 40)
  kv = ops.PagedKV(*pools)
  want = ops.paged_attention(kv, q, table, lens_t)
  length = torch.zeros(1, dtype=torch.int32, device="cuda")
  err = torch.zeros(1, dtype=torch.int32, device="cuda")
  for n in (40, length):
    with pytest.raises(ValueError, match="prefix_table"):
      ops.shared_prefix_attention(kv, q, None, n, table, lens_t)
  for n in (0, 1, 2 ** 31 - 1, -1):
    length.fill_(n)
    err.zero_()
    out = ops.shared_prefix_attention(kv, q, ptable[:0], length, table, lens_t, err_flag=err)
    assert torch.equal(out, want) and int(err) == int(n != 0)
  with pytest.raises(ValueError, match="does not hold"):
    ops.shared_prefix_attention(kv, q, ptable[:0], 1, table, lens_t)


def test_no_pages(cuda):
  """Storages of no pages: every token is left out, with the flag."""
  kp = torch.zeros(0, 16, 2, 64, dtype=BF, device="cuda")
  kv = ops.PagedKV(kp, kp.clone())
  q = torch.ones(3, 2, 8, 64, dtype=BF, device="cuda")
  table = torch.zeros(3, 4, dtype=torch.int32, device="cuda")
  lens = torch.tensor([5, 0, 64], dtype=torch.int32, device="cuda")
  err = torch.zeros(1, dtype=torch.int32, device="cuda")
  for prefix in (None, 20):
    err.zero_()
    if prefix is None:
      out, lse = ops.paged_attention(kv, q, table, lens, return_lse=True, err_flag=err)
    else:
      out, lse = ops.shared_prefix_attention(kv, q, table[0], prefix, table, lens,
                                             return_lse=True, err_flag=err)
    assert (out == 0).all() and (lse == -math.inf).all() and int(err) == 1
  err.zero_()
  k = torch.ones(2, 2, 64, dtype=BF, device="cuda")
  got = ops.kv_append(kv, k, k, torch.tensor([0, -1], device="cuda"), q=q[0], err_flag=err)
  assert (got == 0).all() and int(err) == 1


def test_tangents_are_refused(cuda):
  """Forward-mode derivatives would be lost without a word."""
  from torch.autograd import forward_ad as fwd
  dual = lambda t: fwd.make_dual(t, torch.ones_like(t))
  kp = torch.zeros(4, 16, 2, 64, dtype=BF, device="cuda")
  kv = ops.PagedKV(kp, kp.clone())
  q = torch.zeros(2, 8, 64, dtype=BF, device="cuda")
  k = torch.zeros(2, 2, 64, dtype=BF, device="cuda")
  table = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
  lens = torch.ones(2, dtype=torch.int32, device="cuda")
  slots = torch.arange(2, device="cuda")
  cs, w = torch.zeros(9, 64, device="cuda"), torch.ones(64, device="cuda")
  with fwd.dual_level():
    for grad in (torch.enable_grad, torch.no_grad):
      with grad():
        for call in (lambda: ops.paged_attention(kv, dual(q), table, lens),
                     lambda: ops.shared_prefix_attention(kv, dual(q), table[0], 3, table, lens),
                     lambda: ops.paged_attention(ops.PagedKV(kp, dual(kp.clone())), q, table, lens),
                     lambda: ops.kv_append(kv, dual(k), k, slots),
                     lambda: ops.kv_append(kv, k, dual(k), slots),
                     lambda: ops.kv_append(kv, k, k, slots, q=dual(q)),
                     lambda: ops.kv_append(kv, k, k, slots, k_weight=dual(w)),
                     lambda: ops.kv_append(kv, k, k, slots, positions=slots, cos_sin=dual(cs))):
          with pytest.raises(ValueError, match="tangent"):
            call()
        ops.kv_append(kv, k, k, slots, q=q)  # without one they run
        ops.paged_attention(kv, q, table, lens)


# -- more than drafts, other streams, lengths far below the table's -------------


PROMPTS = [
    # q heads, kv heads, d, block tokens, head major, new tokens, prefix, lengths
    (8, 2, 128, 16, False, 6, None, [6, 3, 0, 100]),
    (32, 8, 128, 16, False, 20, None, [20, 90]),         # 80 rows a KV head: three row tiles
    (8, 2, 128, 16, False, 100, None, [100, 37, 0, 250]),
    (4, 1, 64, 64, True, 257, None, [257, 300]),
    (2, 1, 128, 5, False, 200, None, [200, 13]),
    (8, 2, 128, 16, False, 70, 200, [70, 3, 90]),        # the rest of a prompt behind a prefix
    (4, 2, 64, 16, False, 150, 1000, [150, 151]),
]


@pytest.mark.parametrize("dt", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("case", PROMPTS, ids=str)
def test_many_new_tokens(cuda, case, dt):
  hq, hk, d, bt, major, n, prefix, lens = case
  pools, table, lens_t, ptable, q, own, shared = build(51, dt, hq, hk, d, bt, major, n, lens,
                                                       prefix)
  kv = ops.PagedKV(*pools, head_major=major)
  if prefix is None:
    out, lse = ops.paged_attention(kv, q, table, lens_t, return_lse=True)
  else:
    out, lse = ops.shared_prefix_attention(kv, q, ptable, prefix, table, lens_t, return_lse=True)
  check(out, lse, q, own, shared, lens, hk, dt)


@pytest.mark.parametrize("hq,hk,count", [(8, 2, 33), (8, 1, 70)])
def test_replayed_prefix_lengths_far_below_the_table(cuda, hq, hk, count):
  """A captured call of many rows, planned by a table of 4096 tokens, replayed with any length:
  fewer units of work than CTAs were launched for, and none."""
  lens = [(7 * i) % 60 for i in range(count)]
  pools, table, lens_t, ptable, q, own, shared = build(52, BF, hq, hk, 128, 16, False, 1, lens,
                                                       4096)
  kv = ops.PagedKV(*pools)
  plen = torch.tensor([4096], dtype=torch.int32, device="cuda")
  err = torch.zeros(1, dtype=torch.int32, device="cuda")
  ops.shared_prefix_attention(kv, q, ptable, plen, table, lens_t, return_lse=True)
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out, lse = ops.shared_prefix_attention(kv, q, ptable, plen, table, lens_t, return_lse=True,
                                           err_flag=err)
  for p in (0, 1, 129, 4096, 127, 2000):
    for new in (lens, [0] * count, [x // 2 for x in lens]):
      lens_t.copy_(torch.tensor(new, dtype=torch.int32))
      plen.fill_(p)
      graph.replay()
      torch.cuda.synchronize()
      check(out, lse, q, own, [x[:p] for x in shared], new, hk, BF)
  assert int(err) == 0


@pytest.mark.parametrize("d", [64, 72])
def test_append_on_a_given_stream(cuda, d):
  """The append is ordered on the stream it is given, and allocates there."""
  g = gen(53)
  kp = torch.zeros(8, 16, 2, d, dtype=BF, device="cuda")
  kv = ops.PagedKV(kp, torch.zeros_like(kp))
  k, v, q = (rand(g, 50, h, d, dtype=BF) for h in (2, 2, 6))
  late = [torch.zeros_like(x) for x in (k, v, q)]
  slots = torch.randperm(128, generator=g, device="cuda")[:50]
  s = torch.cuda.Stream()
  s.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(s):
    torch.cuda._sleep(20_000_000)
    for to, x in zip(late, (k, v, q)):
      to.copy_(x)
  got = ops.kv_append(kv, late[0], late[1], slots, q=late[2], stream=s)
  s.synchronize()
  assert torch.equal(got, q)
  assert torch.equal(kp.view(128, 2, d)[slots], k)
  assert torch.equal(kv.v_pages.view(128, 2, d)[slots], v)


@pytest.mark.parametrize("hq,prefix,count", [(4, None, 3), (4, 300, 3), (8, 700, 40)],
                         ids=["own", "walked prefix", "many rows"])
def test_visible_values_that_are_not_finite(cuda, hq, prefix, count):
  """They reach exactly the rows and elements that the definition says: a NaN in K every element
  of its KV head's rows, an infinity in K the rows whose score becomes +infinity (at -infinity
  the key has no weight), one in V its element."""
  lens = [40 + i for i in range(count)]
  pools, table, lens_t, ptable, q, own, shared = build(54, BF, hq, 2, 128, 16, False, 1, lens,
                                                       prefix)
  kv = ops.PagedKV(*pools)

  def put(pool, i, t, head, e, value):  # sequence i, or the prefix: None
    pages, copy = (table[i], own[i]) if i is not None else (ptable, shared)
    pools[pool][int(pages[t // 16]), t % 16, head, e] = value
    copy[pool][t, head, e] = value

  where = None if prefix else 1
  put(0, 0, 5, 0, 3, math.nan)
  put(1, 1, 39, 1, 7, math.inf)
  put(0, 2, 17, 1, 11, math.inf)
  put(0, where, 30, 1, 100, -math.inf)
  put(1, where, 31, 0, 64, math.nan)
  if prefix is None:
    out, lse = ops.paged_attention(kv, q, table, lens_t, return_lse=True)
  else:
    out, lse = ops.shared_prefix_attention(kv, q, ptable, prefix, table, lens_t, return_lse=True)
  g = hq // 2
  for i in range(count):
    k, v = own[i]
    if prefix:
      k, v = torch.cat([shared[0], k]), torch.cat([shared[1], v])
    x = torch.einsum("hgd,thd->hgt", q[i, 0].double().view(2, g, 128), k) * 128 ** -0.5
    p = torch.softmax(x, -1)  # NaN where a score is NaN or +infinity
    fine = torch.isfinite(v).all(0)[:, None] & torch.isfinite(p).all(-1, keepdim=True)
    want = torch.einsum("hgt,thd->hgd", p, torch.where(torch.isfinite(v), v, 0.0))
    size = torch.einsum("hgt,thd->hgd", p, torch.where(torch.isfinite(v), v, 0.0).abs())
    tol = U[BF] * (size + want.abs()) + 2.0 ** -15 * size
    got = out[i, 0].double().view(2, g, 128)
    assert bool(((got - want).abs() <= tol)[fine].all()), i
    assert not bool(torch.isfinite(got)[~fine].any()), i
