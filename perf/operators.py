"""Workloads of the batched decode step over a paged KV cache, one operator a pass.

A server decodes many sequences at once.  Their cache rows lie in pages of one
pool, a page table row per sequence; the projections run on 4-bit weights.  The
operators of such a step:

* "decode": attention of one new token per sequence over its pages;
* "append": RoPE of the new tokens' queries and keys, keys and values written to
  their page rows, for a batch of single tokens or for chunks of prompts;
* "pages": what happens to the pages between steps.  "step" drops the last
  candidates, forks candidates from their parents (pages are shared) and grows
  each by a few tokens (a shared last page is copied first, new pages are the
  lowest free ones); "compact" moves the used pages to the front of the pool;
* "w4": y = W x, or y = W x + residual, with 4-bit weights and a scale per group of
  columns, for one token or a few.

Formats.  A page holds `page` rows of kv_heads * head_dim fp16 values; the pool has
a K and a V plane per layer, [plane][pages][page rows].  Page tables are int32
[sequences][max pages]; entry j of a row is the page of the sequence's rows
j * page and on.  4-bit weights lie in tiles of 16 rows and 128 columns, uint32
[rows / 16][columns / 128][4 a][16 r][4 s]: word s of (a, r) has row r, columns 32 s +
8 a + 0..7 of the tile, column 2 i in bits 4 i and column 2 i + 1 in bits 16 + 4 i; a
code c stands for (c - 8) * scale; scales are fp16 [column groups][rows padded to 16].
"""
import functools
import math
import pathlib
import random
import sys

import numpy as np
import torch

own = False

HIDDEN = 2048
THETA = 5.0e6
# (query heads, KV heads, head dim): the model's own, then other grouped-query,
# multi-head and 64-dim layouts
MODEL = (16, 4, 128)
GROUPED_64 = (16, 4, 64)
OTHERS = ((16, 8, 128), (16, 16, 128), (8, 2, 128), GROUPED_64, (8, 8, 64), (32, 8, 64))
LAYERS = 36
VOCABULARY = 128256
INTERMEDIATE = 11008


@functools.cache
def _binding():
    path = str(pathlib.Path.cwd() / "llm-inference_amd" / "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    import attn_mi355x
    return attn_mi355x


def _layout(layout):
    heads, kv_heads, head_dim = layout
    return {"heads": heads, "kv_heads": kv_heads, "head_dim": head_dim}


def _decode(layout, seqs, low, high, page):
    """seqs sequences of low..high keys, their logarithms evenly spread."""
    return {"kind": "decode", **_layout(layout), "seqs": seqs, "low": low, "high": high, "page": page}


def _append(layout, seqs, tokens, page, rotate):
    """`tokens` new tokens over `seqs` sequences (tokens == seqs: one each)."""
    return {"kind": "append", **_layout(layout), "seqs": seqs, "tokens": tokens, "page": page,
            "rotate": rotate}


def _pages(op, layers, seqs, forks, high, page, pages):
    return {"kind": "pages", "op": op, "kv_heads": 4, "head_dim": 128, "layers": layers,
            "seqs": seqs, "forks": forks, "high": high, "page": page, "pages": pages}


def _w4(tokens, rows, columns, group, residual):
    return {"kind": "w4", "tokens": tokens, "rows": rows, "columns": columns, "group": group,
            "residual": residual}


def listed():
    return [
        # one user with a short chat: every launch is latency
        {"name": "decode_1x254", **_decode(MODEL, 1, 254, 254, 16)},
        # a middling batch of 64-dim heads, chats of all lengths
        {"name": "decode_d64_32", **_decode(GROUPED_64, 32, 20, 4096, 32)},
        # one user over a long document: the benchmark's headline length
        {"name": "decode_1x32768", **_decode(MODEL, 1, 32768, 32768, 64)},
        # a full server: short and long conversations in one batch
        {"name": "decode_64_ragged", **_decode(MODEL, 64, 100, 16384, 16)},
        # the new tokens of that batch
        {"name": "append_64", **_append(MODEL, 64, 64, 16, True)},
        # prompts that arrive together, cut into one chunk of tokens
        {"name": "append_2000", **_append(MODEL, 3, 2000, 16, True)},
        # four candidates of one answer, one token on
        {"name": "pages_step_4", **_pages("step", LAYERS, 2, 4, 500, 16, 256)},
        # a wide search: 256 candidates over 96 sequences
        {"name": "pages_step_256", **_pages("step", LAYERS, 96, 256, 600, 16, 4096)},
        # a pool of five gigabytes in which finished sequences left holes
        {"name": "pages_compact", **_pages("compact", LAYERS, 64, 0, 600, 16, 4096)},
        # the output projection of one token, added to the residual stream
        {"name": "w4_1_out", **_w4(1, HIDDEN, HIDDEN, 128, True)},
        # the logits of one token
        {"name": "w4_1_vocabulary", **_w4(1, VOCABULARY, HIDDEN, 128, False)},
        # the widest product of a layer for a batch of 33 tokens, fine groups
        {"name": "w4_33_down", **_w4(33, HIDDEN, INTERMEDIATE, 32, True)},
    ]


def _between(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("decode", "decode", "append", "pages", "w4", "w4"))
    layout = MODEL if rng.random() < 0.5 else rng.choice(OTHERS)
    page = rng.choice((8, 16, 16, 32, 64, 128)) if rng.random() < 0.8 else _between(rng, 1, 100)
    if kind == "decode":
        seqs = _between(rng, 1, 128)
        high = _between(rng, 4, max(4, min(32768, 200000 // seqs)))
        return _decode(layout, seqs, _between(rng, 1, high), high, page)
    if kind == "append":
        seqs = _between(rng, 1, 200)
        tokens = seqs if rng.random() < 0.5 else _between(rng, seqs, 2000)
        return _append(layout, seqs, tokens, page, rng.random() < 0.75)
    if kind == "pages":
        page = rng.choice((16, 32, 64)) if rng.random() < 0.8 else _between(rng, 2, 40)
        seqs, forks = _between(rng, 1, 64), _between(rng, 1, 128)
        high = _between(rng, 20, 600)
        pages = max(forks * 3 + seqs * (high // page + 2) * 2, 64)
        # 72 planes of 4096 pages of 16 rows at most
        layers = max(1, min(LAYERS, LAYERS * 16 * 4096 // (pages * page)))
        op = rng.choice(("step", "compact"))
        return _pages(op, _between(rng, 1, layers), seqs, forks if op == "step" else 0, high,
                      page, pages)
    tokens = 1 if rng.random() < 0.4 else _between(rng, 2, 64)
    rows, columns = _between(rng, 16, 12000), _between(rng, 32, 12000)
    if rng.random() < 0.6:
        rows, columns = rows // 16 * 16, columns // 32 * 32
    return _w4(tokens, rows, columns, rng.choice((32, 64, 128)), rng.random() < 0.5)


# ---------------------------------------------------------------- sizes of a case

def _lengths(case):
    """The sequences' lengths, from the case alone."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    if case["kind"] == "decode":
        got = [_between(rng, case["low"], case["high"]) for _ in range(case["seqs"])]
        got[-1] = case["high"]
        if case["seqs"] >= 16:  # a batch is padded to a fixed size: rows without a sequence
            got[0] = 0
        return got
    return [_between(rng, 1, case["high"]) for _ in range(case["seqs"])]


def _plan(case):
    """The whole numbers of a pages case, from the case alone: lengths, parents of the
    forks (-1: no fork in that row) and tokens each fork grows by."""
    rng = random.Random("plan" + repr(sorted((k, v) for k, v in case.items() if k != "name")))
    lens = _lengths(case)
    parents = [rng.randrange(case["seqs"]) if rng.random() < 0.95 else -1 for _ in range(case["forks"])]
    grow = [rng.choice((1, 1, 1, 2, 5, 0)) for _ in range(case["forks"])]
    return lens, parents, grow


def _moved_pages(case):
    """How many pages a pages case copies."""
    lens, parents, grow = _plan(case)
    if case["op"] == "compact":
        # used pages lie at random places: the expected number above the used count
        used = sum(-(-n // case["page"]) for n in lens)
        return used * (1 - used / case["pages"])
    return sum(1 for p, g in zip(parents, grow) if p >= 0 and g and lens[p] % case["page"])


def work(case):
    if case["kind"] == "decode":
        row = case["kv_heads"] * case["head_dim"] * 2
        keys, live = sum(_lengths(case)), sum(n > 0 for n in _lengths(case))
        q = case["heads"] * case["head_dim"] * 2
        table = 4 * sum(-(-n // case["page"]) for n in _lengths(case)) + 4 * case["seqs"]
        return {"bytes": keys * 2 * row + live * 2 * q + table,
                "flops": 4 * keys * case["heads"] * case["head_dim"]}
    if case["kind"] == "append":
        values = (case["heads"] + 2 * case["kv_heads"]) * case["head_dim"]
        return {"bytes": case["tokens"] * (2 * 2 * values + 2 * case["head_dim"] + 12),
                "flops": 3 * case["tokens"] * (case["heads"] + case["kv_heads"]) * case["head_dim"]}
    if case["kind"] == "pages":
        page = case["page"] * case["kv_heads"] * case["head_dim"] * 2 * 2 * case["layers"]
        return {"bytes": _moved_pages(case) * 2 * page + 4 * case["pages"], "flops": 0}
    rows, columns, tokens = case["rows"], case["columns"], case["tokens"]
    groups = -(-columns // case["group"])
    return {"bytes": rows * columns / 2 + 2 * rows * groups +
            2 * tokens * (columns + rows * (2 if case["residual"] else 1)),
            "flops": 2 * tokens * rows * columns}


# ---------------------------------------------------------------- inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(g, *shape, scale=1.0):
    x = torch.randn(*shape, generator=g, device="cuda", dtype=torch.float16)
    return x if scale == 1.0 else x.mul_(scale)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _table(lens, page, pages, columns, seed):
    """A page table whose pages lie at random places of the pool; unused entries -1."""
    order = np.random.RandomState(int(seed) % 2**32).permutation(pages)
    table = np.full((len(lens), columns), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(lens):
        k = -(-n // page)
        table[b, :k] = order[at:at + k]
        at += k
    return table


def _tables(rows, head_dim):
    """fp16 cos/sin [rows, head_dim / 2], angles in 64 bits."""
    half = head_dim // 2
    inverse = THETA ** (-torch.arange(half, dtype=torch.float64, device="cuda") * 2 / head_dim)
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * inverse[None]
    return angle.cos().half(), angle.sin().half()


def prepare(case, seed):
    return {"decode": _prepare_decode, "append": _prepare_append, "pages": _prepare_pages,
            "w4": _prepare_w4}[case["kind"]](case, seed)


def _prepare_decode(case, seed):
    g = _generator(seed)
    lens = _lengths(case)
    random.Random(int(seed)).shuffle(lens)
    page, B = case["page"], case["seqs"]
    heads, kv_heads, D = case["heads"], case["kv_heads"], case["head_dim"]
    columns = -(-max(lens) // page) + 1
    pages = sum(-(-n // page) for n in lens) + 3
    kv = _normal(g, 2, pages, page, kv_heads * D)
    s = {"case": case, "k": kv[0], "v": kv[1], "lens": _ints(lens),
         "table": torch.from_numpy(_table(lens, page, pages, columns, seed)).cuda(),
         "pages": pages, "columns": columns,
         # queries of trained heads reach larger scores than independent normals do
         "q": _normal(g, B, heads, D, scale=2.0),
         "out": _normal(g, B, heads, D)}
    if own:
        s["workspace"] = _binding().paged_decode_workspace(B, heads, kv_heads, D)
    return s


def _prepare_append(case, seed):
    g = _generator(seed)
    rng = random.Random(int(seed))
    B, T, page = case["seqs"], case["tokens"], case["page"]
    heads, kv_heads, D = case["heads"], case["kv_heads"], case["head_dim"]
    most = max(4096, 2 * T)
    count = [T // B + (b < T % B) for b in range(B)]
    start = [rng.randrange(0, most - n) for n in count]
    seq = [b for b in range(B) for _ in range(count[b])]
    pos = [start[b] + i for b in range(B) for i in range(count[b])]
    if T >= 16:  # a batch is padded to a fixed size
        pos[T // 3] = -1
    columns = -(-most // page)
    # only the pages that hold new tokens belong to this pool's part of the table
    held = sorted({(b, p // page) for b, p in zip(seq, pos) if p >= 0})
    pages = sum(-(-n // page) + 1 for n in count)
    order = np.random.RandomState(int(seed) % 2**32).permutation(pages)
    table = np.full((B, columns), -1, dtype=np.int32)
    for i, (b, j) in enumerate(held):
        table[b, j] = order[i]
    cos, sin = _tables(most, D)
    kv = _normal(g, 2, pages, page, kv_heads * D)
    return {"case": case, "qkv": _normal(g, T, (heads + 2 * kv_heads) * D), "k": kv[0], "v": kv[1],
            "q_out": _normal(g, T, heads, D), "cos": cos, "sin": sin, "most": most,
            "table": torch.from_numpy(table).cuda(), "pages": pages, "columns": columns,
            "positions": _ints(pos), "seqs": _ints(seq)}


def _prepare_pages(case, seed):
    g = _generator(seed)
    lens, parents, grow = _plan(case)
    page, pages = case["page"], case["pages"]
    columns = -(-(max(lens) + 8) // page)
    table = _table(lens, page, pages, columns, seed)
    held = table[table >= 0]
    count = np.zeros(pages, dtype=np.int32)
    count[held] = 1
    s = {"case": case, "columns": columns,
         "pool": _normal(g, 2 * case["layers"], pages, page * case["kv_heads"] * case["head_dim"]),
         "table": torch.from_numpy(table).cuda(), "lens": _ints(lens),
         "count": torch.from_numpy(count).cuda()}
    if case["op"] == "step":
        s.update(parents=_ints(parents), grow=_ints(grow),
                 table_b=torch.full((case["forks"], columns), -1, dtype=torch.int32, device="cuda"),
                 lens_b=torch.zeros(case["forks"], dtype=torch.int32, device="cuda"),
                 status=torch.zeros(2, dtype=torch.int32, device="cuda"))
        if own:
            s["workspace"] = _binding().pages_workspace(case["forks"], pages)
    else:
        s.update(table_b=torch.full_like(s["table"], -1), count_b=torch.zeros_like(s["count"]),
                 used=torch.zeros(1, dtype=torch.int32, device="cuda"))
        if own:
            s["workspace"] = _binding().pages_workspace(case["seqs"], pages)
    return s


def _prepare_w4(case, seed):
    g = _generator(seed)
    rows, columns, group, tokens = (case[k] for k in ("rows", "columns", "group", "tokens"))
    high, wide = -(-rows // 16) * 16, -(-columns // 128) * 128
    words, scales = [], []
    for r in range(0, high, 4096):  # in parts: a vocabulary's weights are large in fp16
        n = min(4096, high - r)
        w = torch.zeros(n, wide, device="cuda")
        live = min(n, rows - r)
        w[:live, :columns] = _normal(g, live, columns, scale=columns ** -0.5)
        groups = -(-columns // group)
        part = torch.nn.functional.pad(w[:, :columns], (0, groups * group - columns))
        part = part.view(n, groups, group)
        scale = (part.abs().amax(-1) / 7).half()
        step = scale.float().clamp(min=1e-12)[:, :, None]
        code = torch.zeros(n, wide, dtype=torch.int32, device="cuda") + 8
        code[:, :columns] = (torch.round(part / step).clamp(-8, 7).int() + 8).view(n, -1)[:, :columns]
        code = code.view(n // 16, 16, wide // 128, 4, 4, 4, 2)  # tile, r, tile, s, a, i, low/high
        code = code.permute(0, 2, 4, 1, 3, 6, 5).reshape(n // 16, wide // 128, 4, 16, 4, 8).long()
        word = (code << (4 * torch.arange(8, device="cuda"))).sum(-1)
        words.append(torch.where(word >= 2**31, word - 2**32, word).int())
        scales.append(scale.t())
    return {"case": case, "words": torch.cat(words), "scales": torch.cat(scales, 1).contiguous(),
            "x": _normal(g, tokens, columns), "residual": _normal(g, tokens, rows),
            "y": torch.empty(tokens, rows, dtype=torch.float16, device="cuda")}


# ---------------------------------------------------------------- one pass

def run(state):
    return {"decode": _run_decode, "append": _run_append, "pages": _run_pages,
            "w4": _run_w4}[state["case"]["kind"]](state)


def _run_decode(s):
    c = s["case"]
    B, page, heads, kv_heads, D = (c[k] for k in ("seqs", "page", "heads", "kv_heads", "head_dim"))
    if own:
        _binding().paged_decode(s["q"], s["k"], s["v"], s["out"], s["table"], s["lens"], B,
                                s["columns"], s["pages"], page, heads, kv_heads, D, s["workspace"])
        return s["out"]
    keys = s["columns"] * page
    where = s["table"].long().clamp(min=0)
    seen = torch.arange(keys, device="cuda")[None] < s["lens"][:, None]
    q = s["q"].float().view(B, kv_heads, heads // kv_heads, D)
    out = torch.empty(B, heads, D, device="cuda")
    most = max(1, (1 << 28) // (keys * kv_heads * D))
    for b in range(0, B, most):  # a few sequences at a time: a gigabyte of 32-bit keys
        part = slice(b, b + most)
        n = where[part].shape[0]
        k = s["k"][where[part]].view(n, keys, kv_heads, D).float().transpose(1, 2)
        score = torch.matmul(q[part], k.transpose(2, 3)) / math.sqrt(D)
        score = score.masked_fill(~seen[part][:, None, None], -math.inf)
        p = torch.exp(score - score.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        v = s["v"][where[part]].view(n, keys, kv_heads, D).float().transpose(1, 2)
        out[part] = torch.matmul(p, v).view(n, heads, D)
    live = (s["lens"] > 0)[:, None, None]  # rows without a sequence stay as they were
    return torch.where(live, out.half(), s["out"])


def _rotate(x, cos, sin):
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _run_append(s):
    c = s["case"]
    T, page, heads, kv_heads, D = (c[k] for k in ("tokens", "page", "heads", "kv_heads", "head_dim"))
    qd, kvd = heads * D, kv_heads * D
    if own:
        stride, at = qd + 2 * kvd, s["qkv"].data_ptr()
        _binding().paged_rope_store_kv(
            at, at + 2 * qd, at + 2 * (qd + kvd), s["k"], s["v"], s["cos"], s["sin"], s["table"],
            s["positions"], T, c["seqs"], s["columns"], s["pages"], page, s["most"], heads,
            kv_heads, D, stride, stride, c["rotate"], q_out=s["q_out"],
            seq_ids=None if T == c["seqs"] else s["seqs"])
        return [s["q_out"], s["k"], s["v"]]
    live = (s["positions"] >= 0).nonzero()[:, 0]
    pos = s["positions"][live].long()
    x = s["qkv"][live].float()
    q, k = x[:, :qd].view(-1, heads, D), x[:, qd:qd + kvd].view(-1, kv_heads, D)
    if c["rotate"]:
        cos, sin = s["cos"][pos].float()[:, None], s["sin"][pos].float()[:, None]
        q, k = _rotate(q, cos, sin), _rotate(k, cos, sin)
    row = s["table"][s["seqs"][live].long(), pos // page].long() * page + pos % page
    s["q_out"][live] = q.half()
    s["k"].view(-1, kvd)[row] = k.reshape(-1, kvd).half()
    s["v"].view(-1, kvd)[row] = s["qkv"][live, qd + kvd:]
    return [s["q_out"], s["k"], s["v"]]


def _run_pages(s):
    return _run_step(s) if s["case"]["op"] == "step" else _run_compact(s)


def _held(table, lens, page):
    """Truth table of a page table's used entries."""
    return torch.arange(table.shape[1], device="cuda")[None] < ((lens + page - 1) // page)[:, None]


def _run_step(s):
    c = s["case"]
    page, pages, layers = c["page"], c["pages"], c["layers"]
    A, lens, B, lens_b, count = s["table"], s["lens"], s["table_b"], s["lens_b"], s["count"]
    if own:
        binding = _binding()
        elements = page * c["kv_heads"] * c["head_dim"]
        binding.pages_free(B, lens_b, count, c["forks"], s["columns"], pages, page)
        binding.pages_fork(A, lens, B, lens_b, s["parents"], count, c["seqs"], c["forks"],
                           s["columns"], pages, page)
        binding.pages_grow(s["pool"], 2 * layers, elements, B, lens_b, s["grow"], count, s["status"],
                           c["forks"], s["columns"], pages, page, s["workspace"])
        return [B, lens_b, count, s["status"], s["pool"]]
    one = torch.ones((), dtype=torch.int32, device="cuda")
    # drop the last candidates
    gone = B[_held(B, lens_b, page)].long()
    count.index_put_((gone,), -one, accumulate=True)
    lens_b.zero_()
    # fork: a child's row names its parent's pages
    child = (s["parents"] >= 0).nonzero()[:, 0]
    parent = s["parents"][child].long()
    held = _held(A[parent], lens[parent], page)
    B[child] = torch.where(held, A[parent], B[child])
    lens_b[child] = lens[parent]
    count.index_put_((A[parent][held].long(),), one, accumulate=True)
    # grow: the last page of a child is copied if it is shared, new pages follow
    had, more = lens_b.long(), s["grow"].long()
    grows = (more > 0)
    last = (had - 1).clamp(min=0) // page
    tail = B.gather(1, last[:, None])[:, 0].long().clamp(min=0)
    copies = grows & (had % page > 0) & (count[tail] > 1)
    first = (had + page - 1) // page
    new = torch.where(grows, (had + more + page - 1) // page - first, 0)
    need = new + copies
    offset = need.cumsum(0) - need
    free = (count == 0).nonzero()[:, 0]
    row = copies.nonzero()[:, 0]
    source, target = tail[row], free[offset[row]]
    s["pool"][:, target] = s["pool"][:, source]
    count.index_put_((source,), -one, accumulate=True)
    B[row, last[row]] = target.int()
    r = torch.repeat_interleave(torch.arange(len(new), device="cuda"), new)
    i = torch.arange(len(r), device="cuda") - torch.repeat_interleave(new.cumsum(0) - new, new)
    fresh = free[offset[r] + copies[r] + i]
    B[r, first[r] + i] = fresh.int()
    count[target] = 1
    count[fresh] = 1
    lens_b.copy_(torch.where(grows, had + more, had))
    s["status"].zero_()
    return [B, lens_b, count, s["status"], s["pool"]]


def _run_compact(s):
    c = s["case"]
    page, pages, layers = c["page"], c["pages"], c["layers"]
    if own:
        _binding().pages_compact(s["pool"], 2 * layers, page * c["kv_heads"] * c["head_dim"],
                                 s["table"], s["lens"], s["count"], s["table_b"], s["count_b"],
                                 s["used"], c["seqs"], s["columns"], pages, page, s["workspace"])
        return [s["table_b"], s["count_b"], s["used"], s["pool"]]
    live = s["count"] > 0
    used = live.sum()
    number = torch.arange(pages, device="cuda")
    source = (live & (number >= used)).nonzero()[:, 0]
    target = (~live & (number < used)).nonzero()[:, 0]
    to = number.clone()
    to[source] = target
    s["pool"][:, target] = s["pool"][:, source]
    s["count_b"].copy_(s["count"])
    s["count_b"][target] = s["count"][source]
    s["count_b"][source] = 0
    held = _held(s["table"], s["lens"], page)
    s["table_b"].copy_(torch.where(held, to[s["table"].long().clamp(min=0)].int(), s["table_b"]))
    s["used"].fill_(used)
    return [s["table_b"], s["count_b"], s["used"], s["pool"]]


def _codes(words, rows, columns):
    """The codes [rows][columns] of packed words."""
    shift = 4 * torch.arange(8, device=words.device, dtype=torch.int32)
    code = (words[..., None] >> shift) & 15  # tile, tile, a, r, s, low/high i
    high, wide = words.shape[0] * 16, words.shape[1] * 128
    code = code.view(*words.shape, 2, 4).permute(0, 3, 1, 4, 2, 6, 5)
    return code.reshape(high, wide)[:rows, :columns]


def _run_w4(s):
    c = s["case"]
    rows, columns, group = c["rows"], c["columns"], c["group"]
    if own:
        _binding().w4_matvec(s["x"], s["y"], s["words"], s["scales"], c["tokens"], columns, rows,
                             group, residual=s["residual"] if c["residual"] else None)
        return s["y"]
    scale = s["scales"][:, :rows].t().float().repeat_interleave(group, 1)[:, :columns]
    w = (_codes(s["words"], rows, columns) - 8).float() * scale
    y = torch.matmul(s["x"].float(), w.t())
    if c["residual"]:
        y = y + s["residual"].float()
    return y.half()


# ---------------------------------------------------------------- in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"decode": _exact_decode, "append": _exact_append, "pages": _exact_pages,
            "w4": _exact_w4}[case["kind"]](s)


def _exact_decode(s):
    c = s["case"]
    page, heads, kv_heads, D = (c[k] for k in ("page", "heads", "kv_heads", "head_dim"))
    out = s["out"].double()
    table = s["table"].cpu().numpy()
    for b, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        number = torch.from_numpy(table[b, :-(-n // page)].astype(np.int64)).cuda()
        for g in range(kv_heads):
            k = s["k"][number].view(-1, kv_heads, D)[:n, g].double()
            v = s["v"][number].view(-1, kv_heads, D)[:n, g].double()
            mine = slice(g * (heads // kv_heads), (g + 1) * (heads // kv_heads))
            weight = torch.softmax(s["q"][b, mine].double() @ k.t() * D ** -0.5, -1)
            out[b, mine] = weight @ v
    return out


def _exact_append(s):
    c = s["case"]
    page, heads, kv_heads, D = (c[k] for k in ("page", "heads", "kv_heads", "head_dim"))
    half = D // 2
    qkv = s["qkv"].cpu().double().numpy().reshape(c["tokens"], heads + 2 * kv_heads, D)
    cos, sin = s["cos"].cpu().double().numpy(), s["sin"].cpu().double().numpy()
    q_out = s["q_out"].cpu().double().numpy()
    k, v = (s[x].cpu().double().numpy().reshape(-1, kv_heads, D) for x in ("k", "v"))
    table = s["table"].cpu().numpy()
    for t, (p, b) in enumerate(zip(s["positions"].tolist(), s["seqs"].tolist())):
        if p < 0:
            continue
        x = qkv[t].copy()
        if c["rotate"]:
            turned = x[:heads + kv_heads]
            low, high = turned[:, :half].copy(), turned[:, half:].copy()
            turned[:, :half] = low * cos[p] - high * sin[p]
            turned[:, half:] = high * cos[p] + low * sin[p]
        row = int(table[b, p // page]) * page + p % page
        q_out[t], k[row], v[row] = x[:heads], x[heads:heads + kv_heads], x[heads + kv_heads:]
    return [q_out, k.reshape(s["k"].shape), v.reshape(s["v"].shape)]


def _exact_pages(s):
    """Page by page, in plain loops."""
    c = s["case"]
    page = c["page"]
    lens, table, count = s["lens"].tolist(), s["table"].tolist(), s["count"].tolist()
    if c["op"] == "compact":
        used = sum(n > 0 for n in count)
        moves = dict(zip([p for p, n in enumerate(count) if n and p >= used],
                         [p for p, n in enumerate(count) if not n and p < used]))
        new = [[-1] * s["columns"] for _ in lens]
        for b, n in enumerate(lens):
            for j in range(-(-n // page)):
                new[b][j] = moves.get(table[b][j], table[b][j])
        for a, b in moves.items():
            count[b], count[a] = count[a], 0
            s["pool"][:, b] = s["pool"][:, a]
        return [np.array(new), np.array(count), np.array([used]), s["pool"]]
    parents, grow = s["parents"].tolist(), s["grow"].tolist()
    new, lens_b = [[-1] * s["columns"] for _ in parents], [0] * len(parents)
    for i, p in enumerate(parents):
        if p >= 0:
            lens_b[i] = lens[p]
            for j in range(-(-lens[p] // page)):
                new[i][j] = table[p][j]
                count[table[p][j]] += 1
    free = iter([p for p, n in enumerate(count) if n == 0])
    before, copies = list(count), []
    for i, g in enumerate(grow):
        n = lens_b[i]
        if g and n % page and before[new[i][n // page]] > 1:
            old, fresh = new[i][n // page], next(free)
            copies.append((old, fresh))
            count[old] -= 1
            count[fresh] = 1
            new[i][n // page] = fresh
        if g:
            for j in range(-(-n // page), -(-(n + g) // page)):
                new[i][j] = next(free)
                count[new[i][j]] = 1
            lens_b[i] = n + g
    for a, b in copies:
        s["pool"][:, b] = s["pool"][:, a]
    return [np.array(new), np.array(lens_b), np.array(count), np.array([0, 0]), s["pool"]]


def _exact_w4(s):
    c = s["case"]
    rows, columns, group, tokens = (c[k] for k in ("rows", "columns", "group", "tokens"))
    words, scales = s["words"], s["scales"].double()
    x = torch.zeros(tokens, words.shape[1] * 128, dtype=torch.float64, device="cuda")
    x[:, :columns] = s["x"]
    y = torch.zeros(tokens, words.shape[0], 16, dtype=torch.float64, device="cuda")
    for t in range(words.shape[1]):
        for step in range(4):
            for a in range(4):
                for i in range(8):
                    k = 128 * t + 32 * step + 8 * a + i
                    if k >= columns:
                        continue
                    bits = 4 * (i // 2) + 16 * (i % 2)
                    w = (((words[:, t, a, :, step] >> bits) & 15) - 8).double()
                    w = w * scales[k // group].view(-1, 16)
                    y += x[:, k, None, None] * w[None]
    y = y.view(tokens, -1)[:, :rows]
    return y + s["residual"].double() if c["residual"] else y
