"""A cache in pages that several sequences share, and trees of drafted tokens over it: the calls,
the same results from elementary torch operations, and from their definition in 64 bits.

``listed()`` are fixed sizes; ``draw(rng)`` gives further cases of the same ranges. A case's
"kind" selects the call:

* append:    rotary positions on q and k, and the keys' and values' append to the pages;
* step:      a decode step of every sequence: rotary positions, the append and the attention of
             one token each;
* attention: the attention of several tokens of each sequence over pages that hold them already:
             prompts, and the next parts of long prompts;
* tree:      a tree of drafted tokens for each sequence, from its parents: masks and depths,
             rotary positions by depth, the append and the attention by the masks;
* keep:      drafted tokens into every layer, the walk along the tree by the tokens the model chose,
             and the kept tokens' keys and values to their places.

The cache: keys and values [layers][pages][kv_heads][page_tokens][head_dim]; a table of page numbers,
a length and a range of rows for each sequence. The sequences' lengths follow from the case alone:
"past" is the longest, "skew" says how much shorter the others are (0: none).
"""
import ctypes
import math

import torch

own = False

THETA = 500000.0
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


# ---- the cases ------------------------------------------------------------------------

def _case(name, kind, sequences, tokens, past, skew, shape, fmt, page, layers=1):
    heads, kv_heads, head_dim = shape
    return {"name": name, "kind": kind, "sequences": sequences, "tokens": tokens, "past": past, "skew": skew, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "format": fmt, "page": page, "layers": layers}


def listed():
    return [
        # one token each of 16 chats (8 kv heads of 64) into half-size pages
        _case("append_step", "append", 16, 1, 1000, 1.0, (32, 8, 64), "bfloat16", 64),
        # five prompts of different lengths into empty pages, heads of 128
        _case("append_prompts", "append", 5, 1001, 0, 1.0, (32, 8, 128), "float32", 16),
        # a decode step of five short chats of a 0.5B decoder (2 kv heads), ...
        _case("step_chats", "step", 5, 1, 543, 1.0, (14, 2, 64), "float32", 16),
        # ... of 64 sequences up to 4096 tokens, heads of 128, ...
        _case("step_batch", "step", 64, 1, 4095, 1.0, (32, 8, 128), "bfloat16", 64),
        # ... and of one long context beside seven shorter ones
        _case("step_long", "step", 8, 1, 131000, 8.0, (32, 8, 64), "float16", 32),
        # one prompt of 1024 tokens
        _case("prompt", "attention", 1, 1024, 0, 0.0, (32, 8, 64), "float16", 32),
        # the next parts of four long prompts of different lengths, heads of 128
        _case("prompt_parts", "attention", 4, 301, 7000, 1.0, (32, 8, 128), "bfloat16", 64),
        # a prompt of odd length on the fp32 cache
        _case("prompt_full", "attention", 2, 777, 100, 1.0, (32, 8, 64), "float32", 64),
        # a small tree after 4000 tokens, one sequence
        _case("tree_one", "tree", 1, 15, 4000, 0.0, (32, 8, 64), "float32", 64),
        # trees of up to 64 tokens for 16 sequences, heads of 128
        _case("tree_batch", "tree", 16, 64, 3000, 1.0, (32, 8, 128), "bfloat16", 64),
        # what is kept of a small tree, two layers
        _case("keep_one", "keep", 1, 15, 300, 0.0, (32, 8, 64), "float32", 64, 2),
        # what is kept of 16 trees, eight layers
        _case("keep_batch", "keep", 16, 64, 500, 1.0, (32, 8, 128), "bfloat16", 32, 8),
    ]


SHAPES = [(32, 8, 64), (14, 2, 64), (32, 8, 128), (16, 16, 64), (8, 1, 128), (6, 6, 32), (8, 2, 256)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(["append", "step", "attention", "tree", "keep"], [15, 30, 20, 25, 10])[0]
    shape = rng.choice(SHAPES)
    heads, kv_heads, head_dim = shape
    fmt, page = rng.choice(list(TYPES)), rng.choice([16, 32, 64, 128, 256])
    skew = rng.choice([0.0, 1.0, 1.0, 3.0, 8.0])
    sequences, layers = _log(rng, 1, 64), 1
    if kind == "step":
        tokens, past = 1, _log(rng, 1, 131072) - 1
    elif kind == "append":
        tokens, past = rng.choice([1, _log(rng, 2, 1001)]), _log(rng, 1, 4096) - 1
    elif kind == "attention":
        tokens, past = _log(rng, 2, 1536), rng.choice([0, _log(rng, 1, 8192)])
    else:
        tokens, past = _log(rng, 2, 200), _log(rng, 1, 8192) - 1
        if kind == "keep":
            layers, past = rng.choice([1, 2, 4, 8]), min(past, 600)
    case = _case(None, kind, sequences, tokens, past, skew, shape, fmt, page, layers)
    del case["name"]
    while case["sequences"] > 1 and not _affordable(case):
        case["sequences"] = case["sequences"] // 2
    while not _affordable(case):
        case["past"], case["tokens"] = case["past"] * 2 // 3, max(1 if kind == "step" else 2, case["tokens"] * 2 // 3)
    return case


def _affordable(case):
    """No more than the largest listed cases, the plain form's padded work included."""
    b, t, past = case["sequences"], case["tokens"], case["past"]
    e = torch.tensor([], dtype=TYPES[case["format"]]).element_size()
    held = sum(_lengths(case)) * case["kv_heads"] * case["head_dim"] * e * case["layers"]
    padded = b * (past + t)
    if case["kind"] in ("append", "keep"):
        return b * t * (case["heads"] + case["kv_heads"]) * case["head_dim"] * case["layers"] < 42e6 and padded * case["kv_heads"] * case["head_dim"] * case["layers"] < 80e6
    return held < 300e6 and padded * case["kv_heads"] * case["head_dim"] < 5.4e8 and padded * t * case["heads"] < 3e8 and padded * t * case["heads"] * case["head_dim"] < 36e9


def _fraction(s, step):
    return s * step % 1.0


def _lengths(case):
    """What each sequence holds before the call, the first the most."""
    return [int(case["past"] * (1.0 - _fraction(s, 0.6180339887)) ** case["skew"]) for s in range(case["sequences"])]


def _counts(case):
    """The call's rows of each sequence."""
    least = 0.0 if case["skew"] == 0.0 else 0.6
    return [max(1, round(case["tokens"] * (1.0 - least * _fraction(s, 0.7548776662)))) for s in range(case["sequences"])]


# ---- what a program holds before the call ------------------------------------------------

def _generator(seed, part):
    return torch.Generator(device="cuda").manual_seed((seed * 7919 + part * 104729 + 1) % (1 << 62))


def _normal(seed, part, shape, std=1.0):
    return torch.randn(shape, generator=_generator(seed, part), device="cuda", dtype=torch.float32) * std


def _loud(seed, part, kv, d):
    """Some dims far larger than the others, as keys have them."""
    return 0.3 + _normal(seed, part, (kv, d)).abs().pow(3).clamp(max=4.0)


def _frequencies(d):
    return (1.0 / (THETA ** (torch.arange(0, d, 2, dtype=torch.float64) / d)).float()).float()


def _pools(case, seed, pages):
    """The pages' memory, as earlier calls left it."""
    kv, d = case["kv_heads"], case["head_dim"]
    out = []
    for part in (10, 20):
        x = torch.randn((case["layers"], pages, kv, case["page"], d), generator=_generator(seed, part), device="cuda", dtype=torch.float32)
        x *= _loud(seed, part + 1, kv, d)[:, None]
        out.append(x.to(TYPES[case["format"]]))
    return out


def _new_rows(case, seed, rows):
    """The new tokens' projections: q [rows x heads d], k and v [layers x rows x kv_heads d]."""
    h, kv, d, layers = case["heads"], case["kv_heads"], case["head_dim"], case["layers"]
    q = _normal(seed, 1, (rows, h * d))
    k, v = (_normal(seed, part, (layers, rows, kv, d)).mul_(_loud(seed, part + 9, kv, d)).view(layers, rows, kv * d) for part in (2, 12))
    return q, k, v


def _tree(case, seed, counts):
    """Each row's parent among its sequence's rows (-1: the first, which follows the text), its
    token, and the token that the model chose after it (often one of its children's)."""
    starts = torch.tensor([0] + counts).cumsum(0)
    rows = int(starts[-1])
    index = torch.cat([torch.arange(n) for n in counts]).cuda()
    first = torch.arange(rows, device="cuda") - index
    parents = (torch.rand(rows, generator=_generator(seed, 30), device="cuda") * index).long().clamp(max=(index - 1).clamp(min=0))
    tokens = torch.randint(0, 32000, (rows,), generator=_generator(seed, 31), device="cuda")
    taken = torch.where((torch.rand(rows, generator=_generator(seed, 32), device="cuda") < 0.6) & (index > 0), torch.arange(rows, device="cuda"), -1)
    best = torch.full((rows,), -1, device="cuda").scatter_reduce_(0, first + parents, taken, "amax")
    other = torch.randint(0, 32000, (rows,), generator=_generator(seed, 33), device="cuda")
    chosen = torch.where(best >= 0, tokens[best.clamp(min=0)], other)
    parents = torch.where(index == 0, -1, parents)
    return parents.int(), tokens.int(), chosen.int()


def prepare(case, seed):
    lengths, counts = _lengths(case), _counts(case)
    page, b = case["page"], case["sequences"]
    needed = [-(-(n + t) // page) for n, t in zip(lengths, counts)]
    pages, rows = sum(needed), sum(counts)
    order = torch.randperm(pages, generator=_generator(seed, 40), device="cuda").int().cpu().tolist()
    tables, at = [], 0
    for n in needed:  # a sequence's pages lie anywhere
        tables.append(order[at:at + n] + [0] * (max(needed) - n))
        at += n
    q, k, v = _new_rows(case, seed, rows)
    keys, values = _pools(case, seed, pages)
    state = {"case": case, "rows": rows, "most_rows": max(counts), "most_keys": max(n + t for n, t in zip(lengths, counts)), "pages": pages,
             "q": q, "k": k, "v": v, "keys": keys, "values": values, "context": torch.zeros_like(q), "frequencies": _frequencies(case["head_dim"]).cuda(),
             "tables": torch.tensor(tables, dtype=torch.int32, device="cuda"), "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"),
             "starts": torch.tensor([0] + counts, device="cuda").cumsum(0).int()}
    if case["kind"] in ("tree", "keep"):
        state["parents"], state["tokens"], state["chosen"] = _tree(case, seed, counts)
        words = -(-max(counts) // 32)
        state["depths"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
        state["masks"] = torch.zeros((rows, words), dtype=torch.int32, device="cuda")
        state["kept"] = torch.zeros((b, max(counts)), dtype=torch.int32, device="cuda")
        state["counts"], state["next"], state["after"] = torch.zeros((3, b), dtype=torch.int32, device="cuda")
    if own:  # the descriptors of that memory, which a program keeps beside it
        state["cache"], state["batch"] = _descriptors(state)
    torch.cuda.synchronize()
    return state


# ---- the framework's calls ----------------------------------------------------------------

def _descriptors(s):
    from kotensor_amd import _lib
    case = s["case"]
    c, b = _lib.PagedCache(), _lib.PagedBatch()
    c.keys, c.values = s["keys"].data_ptr(), s["values"].data_ptr()
    c.format = {"float32": _lib.KT_PAGED_F32, "float16": _lib.KT_PAGED_F16, "bfloat16": _lib.KT_PAGED_BF16}[case["format"]]
    c.layers, c.pages, c.kv_heads, c.page_tokens, c.head_dim = case["layers"], s["pages"], case["kv_heads"], case["page"], case["head_dim"]
    b.tables, b.lengths, b.starts = s["tables"].data_ptr(), s["lengths"].data_ptr(), s["starts"].data_ptr()
    b.table_stride, b.sequences, b.rows = s["tables"].shape[1], case["sequences"], s["rows"]
    b.most_rows, b.key_bound = s["most_rows"], s["most_keys"]
    if "masks" in s:
        b.depths, b.masks, b.mask_words = s["depths"].data_ptr(), s["masks"].data_ptr(), s["masks"].shape[1]
    return c, b


def _run_own(s):
    from kotensor_amd import _lib
    case, cache, batch = s["case"], ctypes.byref(s["cache"]), ctypes.byref(s["batch"])
    kind, heads = case["kind"], case["heads"]
    q, k, v, freq, context = (s[n].data_ptr() for n in ("q", "k", "v", "frequencies", "context"))
    if kind == "append":
        _lib.call("kt_rope_paged", q, k, v, heads, freq, cache, 0, batch, context, None)
        return {"q": s["context"], "keys": s["keys"], "values": s["values"]}
    if kind == "attention":
        _lib.call("kt_attention_paged", q, heads, cache, 0, batch, context, None)
        return s["context"]
    if kind in ("tree", "keep"):
        _lib.call("kt_tree_masks", s["parents"].data_ptr(), batch, s["depths"].data_ptr(), s["masks"].data_ptr(), None)
    if kind != "keep":
        _lib.call("kt_rope_attention_paged", q, k, v, freq, heads, cache, 0, batch, context, None)
        return {"context": s["context"], "keys": s["keys"], "values": s["values"]}
    layer_bytes = 4 * s["k"].shape[1] * s["k"].shape[2]
    for layer in range(case["layers"]):
        _lib.call("kt_rope_paged", None, k + layer * layer_bytes, v + layer * layer_bytes, heads, freq, cache, layer, batch, None, None)
    kept, counts = s["kept"].data_ptr(), s["counts"].data_ptr()
    _lib.call("kt_tree_accept", s["tokens"].data_ptr(), s["chosen"].data_ptr(), s["parents"].data_ptr(), batch, kept, s["kept"].shape[1], counts,
              s["next"].data_ptr(), None)
    _lib.call("kt_paged_keep", cache, batch, kept, s["kept"].shape[1], counts, s["after"].data_ptr(), None)
    return {n: s[n] for n in ("kept", "counts", "next", "after", "keys", "values")}


# ---- the plain form -----------------------------------------------------------------------

def _rotate(x, position, freq):
    """Rotary positions on x [.. rows x heads x d]: pairs (i, i + d / 2); angles, cosines and sines in 64 bits of the fp32 angle."""
    d = x.shape[-1]
    angle = (position.float()[:, None] * freq).double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[..., :d // 2], x[..., d // 2:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _places(s):
    """Each row's sequence, its index among the sequence's rows, and the rows of all sequences as [sequences x most_rows]."""
    starts = s["starts"].long()
    row = torch.arange(s["rows"], device=starts.device)
    sequence = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    square = (starts[:-1, None] + torch.arange(s["most_rows"], device=starts.device)).clamp(max=s["rows"] - 1)
    return sequence, row - starts[sequence], square


def _ancestors(s, square):
    """[sequences x most_rows x most_rows]: whether row i is row j or comes after it in the tree."""
    n, starts = s["most_rows"], s["starts"].long()
    inside = torch.arange(n, device=starts.device) < (starts[1:] - starts[:-1])[:, None]
    parent = torch.where(inside, s["parents"].long()[square], -1)
    reach = (parent[:, :, None] == torch.arange(n, device=starts.device)).float() + torch.eye(n, device=starts.device)
    for _ in range(max(1, (n - 1).bit_length())):
        reach = (torch.bmm(reach, reach) > 0).float()
    return reach > 0


def _store(s, k, slot, sequence):
    """Rows [layers x rows x kv x d] into the pages."""
    page = s["case"]["page"]
    number = s["tables"].long()[sequence, slot // page]
    for pool, x in ((s["keys"], k), (s["values"], s["v"].view(k.shape))):
        pool[:, number, :, slot % page] = x.transpose(0, 1).to(pool.dtype)


def _held(s, pool):
    """Layer 0's rows of every sequence as fp32 [sequences x kv x most_keys x d]."""
    case = s["case"]
    x = pool[0][s["tables"].long()].float().transpose(1, 2)
    return x.reshape(case["sequences"], case["kv_heads"], -1, case["head_dim"])[:, :, :s["most_keys"]].contiguous()


def _attend(s, q, sequence, index, square, seen):
    """Attention of q [rows x heads x d] over the pages; `seen`: [sequences x most_rows x most_rows] among the new rows, or None: those before."""
    case = s["case"]
    b, h, kv, d, n, total = case["sequences"], case["heads"], case["kv_heads"], case["head_dim"], s["most_rows"], s["most_keys"]
    keys, values = _held(s, s["keys"]), _held(s, s["values"])
    rows = q[square].view(b, n, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(b * kv, h // kv * n, d)
    scores = torch.bmm(rows, keys.view(b * kv, total, d).transpose(1, 2).contiguous()).view(b, h, n, total) / math.sqrt(d)
    new = torch.arange(total, device=q.device)[None, None] - s["lengths"].long()[:, None, None]  # a key's index among the new rows
    if seen is None:
        visible = new <= torch.arange(n, device=q.device)[:, None]
    else:
        visible = (new < 0) | (seen.gather(2, new.clamp(0, n - 1).expand(b, n, total)) & (new < n))
    scores.masked_fill_(~visible[:, None], float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = torch.bmm(p.view(b * kv, h // kv * n, total), values.view(b * kv, total, d))
    return out.view(b, h, n, d).transpose(1, 2)[sequence, index].reshape(s["rows"], h * d)


def _accept(s, index, square, seen):
    """The rows of each sequence that the walk keeps, in order (-1 behind them), how many, and the token after them."""
    n, starts = s["most_rows"], s["starts"].long()
    inside = torch.arange(n, device=starts.device) < (starts[1:] - starts[:-1])[:, None]
    parent, token, chosen = (s[x].long()[square] for x in ("parents", "tokens", "chosen"))
    parent = torch.where(inside, parent, -2)
    matches = token == chosen.gather(1, parent.clamp(min=0))
    earlier = (parent[:, :, None] == parent[:, None, :]) & (token[:, :, None] == token[:, None, :])
    earlier = (earlier & torch.ones((n, n), dtype=torch.bool, device=starts.device).tril(-1)).any(2)
    fine = (matches & ~earlier & (parent >= 0)) | (torch.arange(n, device=starts.device) == 0)
    kept = inside & ~(seen & ~fine[:, None, :]).any(2)
    counts = kept.sum(1)
    order = torch.where(kept, torch.arange(n, device=starts.device), n).sort(1)[0]
    last = order.gather(1, (counts - 1)[:, None])
    return torch.where(order < n, order, -1).int(), counts.int(), chosen.gather(1, last)[:, 0].int()


def _keep(s, kept, counts):
    """The kept rows of every layer to the places behind the text."""
    case, page = s["case"], s["case"]["page"]
    sequence, m = (kept >= 0).nonzero(as_tuple=True)
    tables, lengths = s["tables"].long(), s["lengths"].long()[sequence]
    source, target = lengths + kept[sequence, m].long(), lengths + m
    for pool in (s["keys"], s["values"]):
        pool[:, tables[sequence, target // page], :, target % page] = pool[:, tables[sequence, source // page], :, source % page]
    return s["lengths"] + counts


def run(state):
    if own:
        return _run_own(state)
    s, case = state, state["case"]
    rows, h, kv, d, layers = s["rows"], case["heads"], case["kv_heads"], case["head_dim"], case["layers"]
    sequence, index, square = _places(s)
    q = s["q"].view(rows, h, d)
    if case["kind"] == "attention":
        return _attend(s, q, sequence, index, square, None)
    seen = _ancestors(s, square) if "parents" in s else None
    slot = s["lengths"].long()[sequence] + index
    position = slot if seen is None else s["lengths"].long()[sequence] + seen[sequence, index].sum(1) - 1
    _store(s, _rotate(s["k"].view(layers, rows, kv, d), position, s["frequencies"]), slot, sequence)
    pools = {"keys": s["keys"], "values": s["values"]}
    if case["kind"] == "keep":
        kept, counts, following = _accept(s, index, square, seen)
        return {"kept": kept, "counts": counts, "next": following, "after": _keep(s, kept, counts), **pools}
    q = _rotate(q, position, s["frequencies"])
    if case["kind"] == "append":
        return {"q": q.reshape(rows, h * d), **pools}
    return {"context": _attend(s, q, sequence, index, square, seen), **pools}


# ---- what a pass cannot do without -----------------------------------------------------------

def work(case):
    h, kv, d, layers = (case[x] for x in ("heads", "kv_heads", "head_dim", "layers"))
    e = torch.tensor([], dtype=TYPES[case["format"]]).element_size()
    lengths, counts = _lengths(case), _counts(case)
    rows = sum(counts)
    append = 8.0 * rows * kv * d + 2.0 * e * rows * kv * d
    if case["kind"] == "append":
        return {"bytes": append + 8.0 * rows * h * d, "flops": 6.0 * rows * (h + kv) * d}
    if case["kind"] == "keep":  # (few rows move: as many as a tree is deep at most)
        return {"bytes": layers * append + 12.0 * rows, "flops": 6.0 * layers * rows * kv * d}
    attend = 2.0 * e * kv * d * (sum(lengths) + rows) + 8.0 * rows * h * d
    if case["kind"] == "tree":  # (a node of a random tree of n has about ln n above it)
        pairs = sum(n * (past + 1 + math.log(n)) for past, n in zip(lengths, counts))
    else:
        pairs = sum(n * past + n * (n + 1) // 2 for past, n in zip(lengths, counts))
    return {"bytes": attend + (0.0 if case["kind"] == "attention" else append), "flops": 4.0 * pairs * h * d}


# ---- the same from the definition, in 64 bits ---------------------------------------------------

def _exact_rotated(x, position, freq, steps):
    """Rotary positions in 64 bits; with `steps` rounded to fp32 as the operator defines a cached key."""
    half = x.shape[-1] // 2
    r = (lambda y: y.float().double()) if steps else (lambda y: y)
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    angle = (torch.tensor(position, device=x.device).float()[:, None] * freq).double()[:, None]
    c, s = r(torch.cos(angle)), r(torch.sin(angle))
    x = x.double()
    out[..., :half] = r(r(x[..., :half] * c) - r(x[..., half:] * s))
    out[..., half:] = r(r(x[..., :half] * s) + r(x[..., half:] * c))
    return out


def _exact_above(parents):
    """The rows above each row of one tree, itself last."""
    above = []
    for i, p in enumerate(parents):
        above.append((above[p] if 0 <= p < i else []) + [i])
    return above


def _exact_path(parents, tokens, chosen):
    path = [0]
    while True:
        follow = [i for i in range(path[-1] + 1, len(parents)) if parents[i] == path[-1] and tokens[i] == chosen[path[-1]]]
        if not follow:
            return path
        path.append(follow[0])


def exact(case, seed):
    layers, h, kv, d, page, kind = (case[x] for x in ("layers", "heads", "kv_heads", "head_dim", "page", "kind"))
    state = prepare(case, seed)
    lengths, counts, tables = _lengths(case), _counts(case), state["tables"].tolist()
    freq = state["frequencies"]
    # the pages as the call leaves them: `held` as numbers of their type, `pools` before that last rounding
    held, pools = (state["keys"], state["values"]), {}
    if kind != "attention":
        pools = {"keys": state["keys"].double(), "values": state["values"].double()}
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    tree = [state[x].tolist() for x in ("parents", "tokens", "chosen")] if "parents" in state else None
    context = torch.empty((state["rows"], h, d), dtype=torch.float64, device="cuda")
    rotated = torch.empty_like(context)
    kept = torch.full((case["sequences"], state["most_rows"]), -1, dtype=torch.int32)
    total, following = [], []
    for s, (past, n) in enumerate(zip(lengths, counts)):
        a, b = starts[s], starts[s + 1]
        q = state["q"][a:b].view(n, h, d)
        hidden = torch.ones((n, n), dtype=torch.bool).triu(1)
        position = [past + i for i in range(n)]
        if tree:
            above = _exact_above(tree[0][a:b])
            position = [past + len(x) - 1 for x in above]
            hidden = torch.ones((n, n), dtype=torch.bool)
            for i, x in enumerate(above):
                hidden[i, x] = False
        number = torch.tensor([tables[s][(past + i) // page] for i in range(n)], device="cuda")
        place = torch.tensor([(past + i) % page for i in range(n)], device="cuda")
        if kind != "attention":
            k = _exact_rotated(state["k"][:, a:b].view(layers, n, kv, d), position, freq, True)
            v = state["v"][:, a:b].view(layers, n, kv, d).double()
            for name, memory, x in (("keys", held[0], k), ("values", held[1], v)):
                pools[name][:, number, :, place] = x.transpose(0, 1)
                memory[:, number, :, place] = x.transpose(0, 1).float().to(memory.dtype)
            q = _exact_rotated(q, position, freq, False)
            rotated[a:b] = q
        if kind == "keep":
            path = _exact_path(*(x[a:b] for x in tree))
            kept[s, :len(path)] = torch.tensor(path, dtype=torch.int32)
            total.append(len(path))
            following.append(tree[2][a + path[-1]])
            for name in pools:
                rows = pools[name][:, number[path], :, place[path]].clone()
                pools[name][:, number[:len(path)], :, place[:len(path)]] = rows
        if kind in ("append", "keep"):
            continue
        where = torch.tensor(tables[s][:-(-(past + n) // page)], device="cuda")
        mine = [x[0][where].transpose(0, 1).reshape(kv, -1, d)[:, :past + n] for x in held]
        unseen = torch.cat([torch.zeros((n, past), dtype=torch.bool), hidden], 1).cuda()
        q = q.double()
        for g in range(kv):
            key, value = mine[0][g].double(), mine[1][g].double()
            for j in range(g * (h // kv), (g + 1) * (h // kv)):
                score = (q[:, j] @ key.t().contiguous()).div_(math.sqrt(d)).masked_fill_(unseen, -math.inf)
                context[a:b, j] = torch.softmax(score, 1) @ value
    if kind == "append":
        return {"q": rotated.view(-1, h * d), **pools}
    if kind == "keep":
        after = torch.tensor(lengths, dtype=torch.int32) + torch.tensor(total, dtype=torch.int32)
        return {"kept": kept, "counts": torch.tensor(total, dtype=torch.int32), "next": torch.tensor(following, dtype=torch.int32), "after": after, **pools}
    return context.view(-1, h * d) if kind == "attention" else {"context": context.view(-1, h * d), **pools}
