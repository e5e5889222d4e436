"""Measured cases of the paged KV cache operators.

Three operators of ``tpu_sync_b200.ops`` on the paged storages that the
manager offloads and the hand-offs move:

* ``kv_append``: new tokens' keys and values into their pages, with the norm
  of every query and key head and the position rotation on the way;
* ``paged_attention``: the attention of each sequence's last tokens over its
  pages;
* ``shared_prefix_attention``: the same for a batch whose sequences continue
  one cached prefix (what a prefix-cache hit leaves in the pool).

``run`` computes them from elementary torch operations in 32 bits, or, with
``own`` set, makes the calls a serving engine makes of the package.
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_EPS = 1e-5


# -- cases --------------------------------------------------------------------


def _append(name, tokens, seqs, **kw):
  c = dict(name=name, op="append", dtype="bf16", tokens=tokens, seqs=seqs, q_heads=32, kv_heads=8,
           head_dim=128, rotary=128, block_tokens=16, head_major=False, norm=False,
           interleaved=False, padding=0, max_pos=8192)
  c.update(kw)
  return c


def _paged(name, batch, lo, hi, **kw):
  c = dict(name=name, op="paged", dtype="bf16", batch=batch, new_tokens=1, lo=lo, hi=hi, cap=8192,
           q_heads=32, kv_heads=8, head_dim=128, block_tokens=16, head_major=False, lse=False)
  c.update(kw)
  return c


def _prefix(name, batch, prefix, lo, hi, **kw):
  c = dict(name=name, op="prefix", dtype="bf16", batch=batch, new_tokens=1, prefix=prefix, lo=lo,
           hi=hi, cap=2048, q_heads=32, kv_heads=8, head_dim=128, block_tokens=16,
           head_major=False, lse=False)
  c.update(kw)
  return c


def listed():
  return [
      # one decode step of a small Llama-3-8B batch: latency alone
      _append("append step of 8", 8, 8),
      # one decode step of a large batch on a TP8 rank (8 query heads, 1 KV head, 64-token pages)
      _append("append step of 256, normed", 256, 256, dtype="fp16", q_heads=8, kv_heads=1,
              block_tokens=64, norm=True, max_pos=32768),
      # a full prompt batch of one layer, with the norms of queries and keys
      _append("append prompt of 8192, normed", 8192, 3, norm=True),
      # a ragged prompt batch padded to a bucket: half-width interleaved rotation, 64-wide heads,
      # head-major pages
      _append("append padded prompt of 1531", 1531, 7, dtype="fp16", head_dim=64, rotary=32,
              head_major=True, interleaved=True, padding=83),
      # one user's long conversation: latency, and one sequence for the whole GPU
      _paged("decode 1 x 8191", 1, 8191, 8191),
      # a ragged serving batch of Llama-3-8B
      _paged("decode 64 x 17..4096", 64, 17, 4096),
      # drafted tokens being checked: 4 queries per sequence, small heads, head-major 64-token pages
      _paged("decode 24 x 4 drafts x 5..2001", 24, 5, 2001, dtype="fp16", new_tokens=4,
             head_dim=64, block_tokens=64, head_major=True, lse=True),
      # the largest batch: long sequences, most of a pool read in one step
      _paged("decode 128 x 3001..8192", 128, 3001, 8192),
      # a few requests that share a system prompt and have just begun
      _prefix("prefix 1000 + 4 x 1..60", 4, 1000, 1, 60),
      # a serving batch behind one long document
      _prefix("prefix 8192 + 64 x 1..511", 64, 8192, 1, 511),
      # drafted tokens behind a prefix that ends inside a page, on a TP8 rank
      _prefix("prefix 16389 + 48 x 3 drafts x 3..700", 48, 16389, 3, 700, dtype="fp16",
              new_tokens=3, q_heads=8, kv_heads=1, block_tokens=64, lse=True),
      # the largest batch behind the longest prefix: bound by the matrix products
      _prefix("prefix 32768 + 256 x 1..1024", 256, 32768, 1, 1024),
  ]


def _log(rng, lo, hi):
  return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
  q_heads, kv_heads = rng.choice([(32, 8), (8, 1), (8, 8), (16, 2), (28, 4), (6, 2)])
  kw = dict(dtype=rng.choice(["bf16", "fp16"]), q_heads=q_heads, kv_heads=kv_heads,
            head_dim=rng.choice([64, 128]), block_tokens=rng.choice([16, 32, 64]),
            head_major=rng.random() < 0.3)
  op = rng.choice(["append", "paged", "prefix"])
  if op == "append":
    tokens = _log(rng, 1, 7000)
    seqs = tokens if rng.random() < 0.4 else max(1, min(tokens, _log(rng, 1, 64)))
    c = _append("", tokens, seqs, norm=rng.random() < 0.5, interleaved=rng.random() < 0.3,
                rotary=rng.choice([kw["head_dim"], kw["head_dim"] // 2]),
                padding=rng.choice([0, 0, tokens // 9]), **kw)
  elif op == "paged":
    hi = _log(rng, 1, 8192)
    batch = max(1, min(_log(rng, 1, 192), 600000 // hi))
    c = _paged("", batch, rng.randint(max(0, hi // 8), hi), hi, new_tokens=rng.choice([1, 1, 2, 5]),
               lse=rng.random() < 0.5, **kw)
  else:
    batch = _log(rng, 1, 192)
    hi = _log(rng, 1, 1024)
    c = _prefix("", batch, _log(rng, 64, 32000), rng.randint(0, hi), hi,
                new_tokens=rng.choice([1, 1, 2, 4]) if batch <= 64 else 1,
                lse=rng.random() < 0.5, **kw)
  del c["name"]
  return c


def _lens(case):
  """The lengths of a batch, spread evenly from lo to hi."""
  b, lo, hi = case["batch"], case["lo"], case["hi"]
  return [hi] if b == 1 else [lo + (hi - lo) * i // (b - 1) for i in range(b)]


def _pairs(case):
  """Query-position pairs of the own parts (one head), summed over the batch."""
  n = case["new_tokens"]
  return sum(max(0, l - n + 1 + j) for l in _lens(case) for j in range(n))


def work(case):
  d, hq, hk = case["head_dim"], case["q_heads"], case["kv_heads"]
  if case["op"] == "append":
    t = case["tokens"] - case["padding"]
    moved = 2 * 2 * t * (hq + 2 * hk) * d + 4 * t * case["rotary"] + 16 * case["tokens"]
    flops = t * (hq + hk) * (3 * case["rotary"] + (4 * d if case["norm"] else 0))
    return {"bytes": moved, "flops": flops}
  rows = case["batch"] * case["new_tokens"]
  tokens = sum(_lens(case)) + case.get("prefix", 0)
  pages = sum(-(-l // case["block_tokens"]) for l in _lens(case))
  pages += -(-case.get("prefix", 0) // case["block_tokens"])
  moved = 2 * 2 * tokens * hk * d + 2 * 2 * rows * hq * d + 4 * (pages + case["batch"])
  if case["lse"]:
    moved += 4 * rows * hq
  flops = 4 * hq * d * (_pairs(case) + rows * case.get("prefix", 0))
  return {"bytes": moved, "flops": flops}


# -- inputs -------------------------------------------------------------------


def _normal(shape, gen, dtype, std=1.0):
  return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * std).to(dtype)


def _pool(case, pages, gen):
  """K and V storages of one layer, drawn a slice at a time (no 32-bit copy of a large pool)."""
  bt, h, d = case["block_tokens"], case["kv_heads"], case["head_dim"]
  shape = (pages, h, bt, d) if case["head_major"] else (pages, bt, h, d)
  out = []
  for _ in range(2):
    t = torch.empty(shape, dtype=_DTYPES[case["dtype"]], device="cuda")
    step = max(1, (1 << 27) // (bt * h * d))
    for at in range(0, pages, step):
      t[at:at + step] = torch.randn((min(step, pages - at),) + shape[1:], generator=gen,
                                    device="cuda", dtype=torch.float32)
    out.append(t)
  return out


def _rotation_table(max_pos, rotary):
  """[max_pos, rotary] in 32 bits: the cosines of a position's angles, then the sines."""
  freq = 500000.0 ** (-torch.arange(0, rotary, 2, device="cuda", dtype=torch.float64) / rotary)
  ang = torch.arange(max_pos, device="cuda", dtype=torch.float64)[:, None] * freq[None]
  return torch.cat([ang.cos(), ang.sin()], dim=1).float()


def prepare(case, seed):
  gen = torch.Generator(device="cuda").manual_seed(seed)
  dt, d = _DTYPES[case["dtype"]], case["head_dim"]
  hq, hk, bt = case["q_heads"], case["kv_heads"], case["block_tokens"]
  s = {"case": case}
  if case["op"] == "append":
    t, seqs = case["tokens"], case["seqs"]
    live = t - case["padding"]
    # sequence i appends its share of the live tokens behind a history of its own
    share = [live // seqs + (i < live % seqs) for i in range(seqs)]
    counts = torch.tensor(share, device="cuda")
    first = torch.cumsum(counts, 0) - counts
    most = max(max(share), 1)
    start = (torch.rand(seqs, generator=gen, device="cuda") * (case["max_pos"] - most)).long()
    seq = torch.repeat_interleave(torch.arange(seqs, device="cuda"), counts, output_size=live)
    pos = start[seq] + torch.arange(live, device="cuda") - first[seq]
    page = pos // bt - start[seq] // bt
    per_seq = most // bt + 2
    pages = seqs * per_seq + 3
    perm = torch.randperm(pages, generator=gen, device="cuda")
    slots = perm[seq * per_seq + page] * bt + pos % bt
    pad = torch.full((case["padding"],), -1, device="cuda", dtype=torch.int64)
    s["slots"] = torch.cat([slots, pad])
    s["positions"] = torch.cat([pos, torch.zeros_like(pad)])
    s["k_pages"], s["v_pages"] = _pool(case, pages, gen)
    qkv = _normal((t, (hq + 2 * hk) * d), gen, dt)  # one projection's output, as engines have it
    q, k, v = qkv.split([hq * d, hk * d, hk * d], dim=1)
    s["q"], s["k"], s["v"] = q.view(t, hq, d), k.view(t, hk, d), v.view(t, hk, d)
    s["cos_sin"] = _rotation_table(case["max_pos"], case["rotary"])
    s["q_weight"] = (1 + _normal((d,), gen, torch.float32, 0.2)).to(dt) if case["norm"] else None
    s["k_weight"] = (1 + _normal((d,), gen, torch.float32, 0.2)).to(dt) if case["norm"] else None
  else:
    b, n = case["batch"], case["new_tokens"]
    lens = torch.tensor(_lens(case), device="cuda", dtype=torch.int32)
    s["seq_lens"] = lens[torch.randperm(b, generator=gen, device="cuda")]
    width = -(-max(case["cap"], case["hi"]) // bt)
    need = (s["seq_lens"].long() + bt - 1) // bt
    n_prefix = -(-case.get("prefix", 0) // bt)
    used = sum(-(-l // bt) for l in _lens(case))
    pages = used + n_prefix + 5
    perm = torch.randperm(pages, generator=gen, device="cuda")
    col = torch.arange(width, device="cuda")[None]
    at = (torch.cumsum(need, 0) - need)[:, None] + col
    table = torch.where(col < need[:, None], perm[at.clamp(max=pages - 1)], 0)
    s["block_table"] = table.to(torch.int32)
    s["k_pages"], s["v_pages"] = _pool(case, pages, gen)
    s["q"] = _normal((b, n, hq, d) if n > 1 else (b, hq, d), gen, dt, 2.0)
    s["longest"] = case["hi"]
    if case["op"] == "prefix":
      s["prefix_table"] = perm[used:used + n_prefix].to(torch.int32)
      s["prefix_len"] = case["prefix"]
  if own:
    from tpu_sync_b200 import ops
    s["kv"] = ops.PagedKV(s["k_pages"], s["v_pages"], head_major=case["head_major"])
  return s


# -- the operators ------------------------------------------------------------


def _rotate(x, cos, sin, rotary, interleaved):
  """x [tokens, heads, head_dim] in 32 bits; cos, sin [tokens, 1, rotary / 2]."""
  r = x[..., :rotary]
  if interleaved:
    a, b = r[..., 0::2], r[..., 1::2]
    r = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
  else:
    a, b = r[..., :rotary // 2], r[..., rotary // 2:]
    r = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
  return torch.cat([r, x[..., rotary:]], dim=-1)


def _norm(x, weight):
  return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS) * weight.float()


def _append_plain(s):
  c = s["case"]
  q, k = s["q"].float(), s["k"].float()
  if c["norm"]:
    q, k = _norm(q, s["q_weight"]), _norm(k, s["k_weight"])
  row = s["cos_sin"][s["positions"]][:, None]
  cos, sin = row[..., :c["rotary"] // 2], row[..., c["rotary"] // 2:]
  q = _rotate(q, cos, sin, c["rotary"], c["interleaved"])
  k = _rotate(k, cos, sin, c["rotary"], c["interleaved"])
  live = s["slots"] >= 0
  at = s["slots"][live]
  page, off = at // c["block_tokens"], at % c["block_tokens"]
  for pages, new in ((s["k_pages"], k), (s["v_pages"], s["v"])):
    view = pages.transpose(1, 2) if c["head_major"] else pages
    view[page, off] = new[live].to(pages.dtype)
  q_out = torch.where(live[:, None, None], q, 0.0).to(s["q"].dtype)
  return {"q": q_out, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _gather(pages, table, tokens, head_major):
  """[..., heads, tokens, head_dim] in 32 bits of the pages a table names."""
  x = pages[table.long()]  # [..., blocks, tokens, heads, dim] or [..., blocks, heads, tokens, dim]
  x = x.movedim(-3, -4) if head_major else x.movedim(-2, -4)
  return x.flatten(-3, -2)[..., :tokens, :].float()


def _parts(q, k, v, scale, visible):
  """Maximum, sum and weighted values of one key range; `visible` masks scores (None: all seen)."""
  scores = torch.matmul(q, k.transpose(-1, -2)) * scale
  if visible is not None:
    scores = scores.masked_fill(~visible, -math.inf)
  top = scores.amax(-1, keepdim=True)
  p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
  return top, p.sum(-1, keepdim=True), torch.matmul(p, v)


def _attention_plain(s):
  c = s["case"]
  b, n, hq, hk, d, bt = (c[x] for x in ("batch", "new_tokens", "q_heads", "kv_heads", "head_dim",
                                        "block_tokens"))
  g, scale = hq // hk, d ** -0.5
  longest = s["longest"]
  q = s["q"].float().view(b, n, hk, g, d).transpose(1, 2).reshape(b, hk, n * g, d)
  table = s["block_table"][:, :-(-longest // bt)]
  k = _gather(s["k_pages"], table, longest, c["head_major"])
  v = _gather(s["v_pages"], table, longest, c["head_major"])
  seen = s["seq_lens"].long()[:, None] - n + 1 + torch.arange(n, device=q.device)  # [b, n]
  seen = seen.repeat_interleave(g, dim=1)[:, None, :, None]
  visible = torch.arange(longest, device=q.device) < seen
  top, total, acc = _parts(q, k, v, scale, visible)
  if c["op"] == "prefix":
    del k, v
    k = _gather(s["k_pages"], s["prefix_table"], s["prefix_len"], c["head_major"])
    v = _gather(s["v_pages"], s["prefix_table"], s["prefix_len"], c["head_major"])
    rows = q.transpose(0, 1).reshape(hk, b * n * g, d)
    parts = _parts(rows, k, v, scale, None)
    top2, total2, acc2 = (x.view(hk, b, n * g, -1).transpose(0, 1) for x in parts)
    new = torch.maximum(top, top2)
    w1, w2 = torch.exp(top - new), torch.exp(top2 - new)
    top, total, acc = new, total * w1 + total2 * w2, acc * w1 + acc2 * w2
  out = torch.where(total > 0, acc / total, 0.0)
  out = out.view(b, hk, n, g, d).transpose(1, 2).reshape(s["q"].shape).to(s["q"].dtype)
  if not c["lse"]:
    return {"out": out}
  lse = torch.where(total > 0, top + torch.log(total), -math.inf)
  return {"out": out, "lse": lse.view(b, hk, n, g).transpose(1, 2).reshape(s["q"].shape[:-1])}


def run(state):
  s, c = state, state["case"]
  if not own:
    return _append_plain(s) if c["op"] == "append" else _attention_plain(s)
  from tpu_sync_b200 import ops
  if c["op"] == "append":
    q = ops.kv_append(s["kv"], s["k"], s["v"], s["slots"], q=s["q"], positions=s["positions"],
                      cos_sin=s["cos_sin"], interleaved=c["interleaved"], q_weight=s["q_weight"],
                      k_weight=s["k_weight"], eps=_EPS)
    return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
  if c["op"] == "paged":
    got = ops.paged_attention(s["kv"], s["q"], s["block_table"], s["seq_lens"],
                              return_lse=c["lse"])
  else:
    got = ops.shared_prefix_attention(s["kv"], s["q"], s["prefix_table"], s["prefix_len"],
                                      s["block_table"], s["seq_lens"], return_lse=c["lse"])
  return {"out": got[0], "lse": got[1]} if c["lse"] else {"out": got}


# -- the definitions in 64 bits -----------------------------------------------


def _exact_append(c, s):
  half, bt = c["rotary"] // 2, c["block_tokens"]
  i = torch.arange(half, device="cuda")
  first = 2 * i if c["interleaved"] else i
  second = 2 * i + 1 if c["interleaved"] else i + half
  angles = s["cos_sin"].double()[s["positions"]]
  turned = {}
  for name in ("q", "k"):
    x = s[name].double()
    if c["norm"]:
      x = s[name + "_weight"].double() * x / (x.pow(2).sum(-1, keepdim=True) / c["head_dim"]
                                              + _EPS).sqrt()
    z = torch.complex(x[..., first], x[..., second])
    z = z * torch.complex(angles[:, :half], angles[:, half:])[:, None]
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    turned[name] = y
  pages = {}
  for name, new in (("k_pages", turned["k"]), ("v_pages", s["v"].double())):
    flat = s[name].double()
    if c["head_major"]:
      flat = flat.transpose(1, 2).contiguous()
    flat = flat.reshape(-1, c["kv_heads"], c["head_dim"])
    keep = (s["slots"] >= 0).nonzero()[:, 0]
    flat[s["slots"][keep]] = new[keep]
    flat = flat.view(-1, bt, c["kv_heads"], c["head_dim"])
    pages[name] = flat.transpose(1, 2).contiguous() if c["head_major"] else flat
  turned["q"][s["slots"] < 0] = 0
  return {"q": turned["q"], **pages}


def _exact_attention(c, s):
  n, hk, d, bt = c["new_tokens"], c["kv_heads"], c["head_dim"], c["block_tokens"]
  q = s["q"].double().view(c["batch"], n, hk, -1, d)

  def tokens(pages, table, count):
    x = pages[table[:-(-count // bt)].long()].double()
    x = x.transpose(1, 2) if c["head_major"] else x
    return x.reshape(-1, hk, d)[:count]

  out, lse = torch.zeros_like(q), torch.full(q.shape[:-1], -math.inf, dtype=torch.float64,
                                             device="cuda")
  if c["op"] == "prefix":
    pk = tokens(s["k_pages"], s["prefix_table"], c["prefix"])
    pv = tokens(s["v_pages"], s["prefix_table"], c["prefix"])
  for b, length in enumerate(s["seq_lens"].tolist()):
    k = tokens(s["k_pages"], s["block_table"][b], length)
    v = tokens(s["v_pages"], s["block_table"][b], length)
    past = 0
    if c["op"] == "prefix":
      k, v, past = torch.cat([pk, k]), torch.cat([pv, v]), c["prefix"]
    for j in range(n):
      seen = past + max(0, length - n + 1 + j)
      if seen == 0:
        continue
      x = torch.einsum("hgd,thd->hgt", q[b, j], k[:seen]) / math.sqrt(d)
      lse[b, j] = torch.logsumexp(x, -1)
      out[b, j] = torch.einsum("hgt,thd->hgd", torch.softmax(x, -1), v[:seen])
  out, lse = out.view(s["q"].shape), lse.view(s["q"].shape[:-1])
  return {"out": out, "lse": lse} if c["lse"] else {"out": out}


def exact(case, seed):
  s = prepare(case, seed)
  return _exact_append(case, s) if case["op"] == "append" else _exact_attention(case, s)
