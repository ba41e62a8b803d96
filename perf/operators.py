"""The operators of a decode step that grow with the text, on a cache held in 8 bits, and the
control of the next token by the text so far: the calls, the same results from elementary
torch operations, and from their definition in 64 bits.

``listed()`` are fixed sizes; ``draw(rng)`` gives further cases of the same ranges. A case's
"kind" selects the call:

* append:    rotary positions on q and k, and the keys' and values' append to the cache, one
             token or a prompt; the values the touched blocks hold are read back;
* step:      a decode step's attention: rotary positions, the append and the attention of one
             token; the values of the block that received it are read back;
* attention: the attention of several tokens over a cache that holds them already: drafted
             tokens to be checked, a prompt, the next part of a long prompt;
* logits:    penalties for tokens of the text, biases and a grammar's mask, one row a sequence.

The cache: keys [kv_heads][slots][head_dim] codes; values [kv_heads][slots / 64][head_dim][64]
codes, the 64 tokens of a dim as [piece p][32 tokens h][quad u][token i] for token 32 h + 16 (p / 2) +
8 u + 4 (p % 2) + i; one scale for the keys and one for the values of each block of tokens and head;
and the open block's rows in fp32. Codes are int8 (stored + 128) or e4m3.
"""
import ctypes
import math

import torch

own = False

THETA = 500000.0
QMAX = {"int8": 127.0, "e4m3": 448.0}


# ---- the cases ------------------------------------------------------------------------

def _cache_case(name, kind, tokens, past, shape, fmt, block):
    heads, kv_heads, head_dim = shape
    return {"name": name, "kind": kind, "tokens": tokens, "past": past, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "format": fmt,
            "block": block}


def _logits_case(name, rows, n, history, bias, mask):
    return {"name": name, "kind": "logits", "rows": rows, "n": n, "history": history, "bias": bias, "mask": mask}


def listed():
    return [
        # one token's key and value into a short chat's cache (8 kv heads of 64)
        _cache_case("append_step", "append", 1, 200, (32, 8, 64), "int8", 64),
        # a 1024-token prompt into an empty cache
        _cache_case("append_prompt", "append", 1024, 0, (32, 8, 64), "int8", 64),
        # an odd prompt of a model with heads of 128, e4m3
        _cache_case("append_wide", "append", 1501, 0, (32, 8, 128), "e4m3", 32),
        # decode steps: early in a chat of a 0.5B decoder (2 kv heads), ...
        _cache_case("step_short", "step", 1, 543, (14, 2, 64), "int8", 32),
        # ... 8191 tokens into a context, ...
        _cache_case("step_8k", "step", 1, 8191, (32, 8, 64), "int8", 64),
        # ... and at the end of a 128k context with heads of 128
        _cache_case("step_128k", "step", 1, 131071, (32, 8, 128), "e4m3", 128),
        # seven drafted tokens checked at once, 4000 tokens into a context
        _cache_case("check_drafts", "attention", 7, 4000, (32, 8, 64), "e4m3", 64),
        # a 1024-token prompt
        _cache_case("prompt", "attention", 1024, 0, (32, 8, 64), "int8", 64),
        # the next 301 tokens of a long prompt, heads of 128
        _cache_case("prompt_part", "attention", 301, 7000, (32, 8, 128), "int8", 128),
        # one sequence's logits, a short text, no grammar
        _logits_case("logits_chat", 1, 32000, 300, 0, False),
        # 64 sequences against a large vocabulary, long texts, biases and a grammar's mask
        _logits_case("logits_batch", 64, 151936, 4096, 100, True),
        # few sequences, odd sizes, one bias
        _logits_case("logits_odd", 5, 49157, 1001, 1, True),
    ]


SHAPES = [(32, 8, 64), (14, 2, 64), (32, 8, 128), (16, 16, 64), (8, 1, 128), (6, 6, 32), (8, 2, 256)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(["append", "step", "attention", "logits"], [20, 30, 30, 20])[0]
    if kind == "logits":
        rows, n = _log(rng, 1, 64), _log(rng, 1000, 151936)
        return {"kind": kind, "rows": rows, "n": n, "history": _log(rng, 1, 4096), "bias": rng.choice([0, 1, _log(rng, 2, 300)]), "mask": rng.random() < 0.5}
    shape = rng.choice(SHAPES)
    heads, kv_heads, head_dim = shape
    fmt, block = rng.choice(["int8", "e4m3"]), rng.choice([32, 64, 128])
    if kind == "append":
        tokens = 1 if rng.random() < 0.4 else _log(rng, 2, 1501)
        past = _log(rng, 1, 8192) - 1
        if tokens > 1:  # a call that can be made again: its first block holds no earlier tokens
            past = rng.choice([0, past // block * block])
        if head_dim == 256:
            tokens = max(1, tokens // 2)
    elif kind == "step":
        tokens, past = 1, _log(rng, 1, 131072) - 1
        while kv_heads * head_dim * past > 8 * 128 * 131071:
            past //= 2
    else:
        tokens = _log(rng, 2, 1536)
        past = rng.choice([0, _log(rng, 1, 8192)])
        while tokens * (2 * past + tokens) * heads * head_dim > 301 * (14000 + 301) * 32 * 128:
            tokens, past = max(2, tokens * 2 // 3), past * 2 // 3
    case = _cache_case(None, kind, tokens, past, shape, fmt, block)
    del case["name"]
    return case


# ---- what a program holds before the call ------------------------------------------------

def _generator(seed, part):
    return torch.Generator(device="cuda").manual_seed((seed * 7919 + part * 104729 + 1) % (1 << 62))


def _normal(seed, part, shape, std=1.0):
    return torch.randn(shape, generator=_generator(seed, part), device="cuda", dtype=torch.float32) * std


def _slots(case):
    unit = max(64, case["block"])
    return -(-(case["past"] + case["tokens"]) // unit) * unit


def _rows(case, seed, part, count, new=0):
    """Keys or values of `count` tokens [kv_heads x count x head_dim] held already, or new ones: some
    dims far larger than the others, as keys have them, and stretches of different loudness."""
    kv, d = case["kv_heads"], case["head_dim"]
    x = _normal(seed, part + 5 * new, (kv, count, d))
    x *= 0.3 + _normal(seed, part + 1, (kv, 1, d)).abs().pow(3).clamp(max=4.0)
    return x * torch.exp(0.5 * _normal(seed, part + 2, (kv, -(-max(count, 1) // 100), 1))).repeat_interleave(100, 1)[:, :count]


def _divide(a, b):
    """The correctly rounded fp32 quotient."""
    return (a.double() / b).float()


def _encode(rows, block, fmt):
    """(codes as the values they hold [kv x blocks * block x d], scales [kv x blocks]) of fp32 rows [kv x count x d]."""
    kv, count, d = rows.shape
    blocks = -(-count // block)
    rows = torch.cat([rows, rows.new_zeros((kv, blocks * block - count, d))], 1).view(kv, blocks, block, d)
    scales = _divide(rows.abs().amax((2, 3)), QMAX[fmt]).clamp(min=2.0 ** -120)
    codes = rows * _divide(torch.ones_like(scales), scales)[:, :, None, None]
    if fmt == "int8":
        codes = codes.round().clamp(-127.0, 127.0)
    else:
        codes = codes.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).float()
    return codes.view(kv, blocks * block, d), scales


def _bytes(codes, fmt):
    return (codes + 128.0).to(torch.uint8) if fmt == "int8" else codes.to(torch.float8_e4m3fn).view(torch.uint8)


def _values_of(stored, fmt):
    return stored.float() - 128.0 if fmt == "int8" else stored.view(torch.float8_e4m3fn).float()


def _transpose_in(codes):
    """Values [kv x slots x d] in the order the cache holds them."""
    kv, slots, d = codes.shape
    return codes.view(kv, slots // 64, 2, 2, 2, 2, 4, d).permute(0, 1, 7, 3, 5, 2, 4, 6).contiguous()


def _transpose_out(stored, kv, slots, d):
    return stored.view(kv, slots // 64, d, 2, 2, 2, 2, 4).permute(0, 1, 5, 3, 6, 4, 7, 2).reshape(kv, slots, d)


def _frequencies(d):
    return (1.0 / (THETA ** (torch.arange(0, d, 2, dtype=torch.float64) / d)).float()).float()


def _memory(case, seed, count):
    """The cache's memory after `count` tokens, and the open block's rows."""
    kv, d, block, fmt, slots = case["kv_heads"], case["head_dim"], case["block"], case["format"], _slots(case)
    out = {}
    for name, part in (("keys", 10), ("values", 20)):
        codes = torch.zeros((kv, slots, d), device="cuda")
        scales = torch.zeros((kv, slots // block), device="cuda")
        open_rows = torch.zeros((kv, block, d), device="cuda")
        if count:
            rows = _rows(case, seed, part, count)
            held, s = _encode(rows, block, fmt)
            codes[:, :held.shape[1]], scales[:, :s.shape[1]] = held, s
            first = count // block * block
            open_rows[:, :count - first] = rows[:, first:]
        stored = _bytes(codes, fmt)
        out[name] = _transpose_in(stored) if name == "values" else stored
        out[name + "_scales"], out[name + "_open"] = scales, open_rows
    return out


def _tokens_in(case, seed):
    """The new tokens' projections q, k and v."""
    t, h, kv, d = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
    q = _normal(seed, 1, (t, h * d))
    k, v = (_rows(case, seed, part, t, 1).transpose(0, 1).reshape(t, kv * d).contiguous() for part in (10, 20))
    return q, k, v


def _logits_inputs(case, seed):
    rows, n, length = case["rows"], case["n"], case["history"]
    logits = _normal(seed, 1, (rows, n), 3.0)
    g = _generator(seed, 2)
    # a text's tokens: few are frequent, most occur once; some entries are padding
    history = (n * torch.rand((rows, length), generator=g, device="cuda").pow(6.0)).to(torch.int32).clamp(max=n - 1)
    history[torch.rand((rows, length), generator=g, device="cuda") < 0.02] = -1
    lengths = (length - (torch.rand(rows, generator=g, device="cuda") * length * 0.5).to(torch.int32)).to(torch.int32)
    starts = (lengths * 0.3).to(torch.int32)
    bias_tokens = torch.randint(0, n, (max(1, case["bias"]),), generator=g, device="cuda", dtype=torch.int32)
    bias_values = _normal(seed, 3, (max(1, case["bias"]),), 2.0)
    words = -(-n // 32)
    allowed = torch.randint(-2 ** 31, 2 ** 31 - 1, (rows, words), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
    if rows > 1:
        allowed[1] = 0  # a sequence whose grammar is at its end: nothing may follow
    return {"logits": logits, "history": history, "lengths": lengths, "starts": starts, "bias_tokens": bias_tokens, "bias_values": bias_values, "allowed": allowed}


REPETITION, FREQUENCY, PRESENCE = 1.3, 0.2, 0.5


def prepare(case, seed):
    if case["kind"] == "logits":
        state = {"case": case, **_logits_inputs(case, seed)}
        state["out"] = torch.empty_like(state["logits"])
    else:
        held = case["past"] + (case["tokens"] if case["kind"] == "attention" else 0)
        state = {"case": case, **_memory(case, seed, held)}
        state["q"], state["k"], state["v"] = _tokens_in(case, seed)
        state["position"] = torch.tensor([case["past"]], dtype=torch.int32, device="cuda")
        state["frequencies"] = _frequencies(case["head_dim"]).cuda()
        state["context"] = torch.empty_like(state["q"])
        first = case["past"] // case["block"] * case["block"]
        state["read"] = first, case["past"] + case["tokens"] - first
        state["rows"] = [torch.empty((case["kv_heads"], state["read"][1], case["head_dim"]), device="cuda") for _ in range(2)]
    if own:  # the descriptor of that memory, which a program keeps beside it
        state["handle"] = _handle(state)
    torch.cuda.synchronize()
    return state


# ---- the framework's calls ----------------------------------------------------------------

def _handle(s):
    from kotensor_amd import _lib
    case = s["case"]
    if case["kind"] == "logits":
        c = _lib.LogitsControls()
        c.history, c.history_length, c.output_start = s["history"].data_ptr(), s["lengths"].data_ptr(), s["starts"].data_ptr()
        c.history_stride = c.history_capacity = case["history"]
        c.repetition, c.frequency, c.presence = REPETITION, FREQUENCY, PRESENCE
        c.bias_count = case["bias"]
        c.bias_tokens, c.bias_values = s["bias_tokens"].data_ptr(), s["bias_values"].data_ptr()
        if case["mask"]:
            c.allowed, c.allowed_stride = s["allowed"].data_ptr(), s["allowed"].shape[1]
        return c
    c = _lib.KV8Cache()
    c.keys, c.values, c.key_scales, c.value_scales = (s[n].data_ptr() for n in ("keys", "values", "keys_scales", "values_scales"))
    c.key_rows, c.value_rows = s["keys_open"].data_ptr(), s["values_open"].data_ptr()
    c.format = {"int8": _lib.KT_KV8_INT8, "e4m3": _lib.KT_KV8_E4M3}[case["format"]]
    c.layers, c.kv_heads, c.max_seq, c.head_dim, c.block_tokens = 1, case["kv_heads"], case["past"] + case["tokens"], case["head_dim"], case["block"]
    return c


def _run_own(s):
    from kotensor_amd import _lib
    case, handle = s["case"], ctypes.byref(s["handle"])
    kind = case["kind"]
    if kind == "logits":
        _lib.call("kt_process_logits", s["logits"].data_ptr(), case["rows"], case["n"], case["n"], handle, s["out"].data_ptr(), case["n"], None)
        return s["out"]
    tokens, heads, q, position, context = case["tokens"], case["heads"], s["q"].data_ptr(), s["position"].data_ptr(), s["context"].data_ptr()
    if kind == "attention":
        _lib.call("kt_attention_kv8", q, tokens, position, case["past"] + tokens, handle, 0, heads, context, None)
        return s["context"]
    k, v, freq = s["k"].data_ptr(), s["v"].data_ptr(), s["frequencies"].data_ptr()
    if kind == "append":
        _lib.call("kt_rope_kv8", q, k, v, tokens, heads, freq, position, handle, 0, context, None)
    else:
        _lib.call("kt_rope_attention_kv8", q, k, v, freq, 1, position, case["past"] + 1, handle, 0, heads, context, None)
    _lib.call("kt_kv8_read", handle, 0, s["read"][0], s["read"][1], s["rows"][0].data_ptr(), s["rows"][1].data_ptr(), None)
    return {"q" if kind == "append" else "context": s["context"], "keys": s["rows"][0], "values": s["rows"][1]}


# ---- the plain form -----------------------------------------------------------------------

def _rotate(x, first, freq):
    """Rotary positions on x [T x heads x d]: pairs (i, i + d / 2); angles, cosines and sines in 64 bits of the fp32 angle."""
    t, _, d = x.shape
    angle = ((first.float() + torch.arange(t, device=x.device, dtype=torch.float32))[:, None] * freq).double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[..., :d // 2], x[..., d // 2:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _held(s):
    """The cache as fp32 keys and values [kv x slots x d]."""
    case = s["case"]
    kv, d, block, fmt, slots = case["kv_heads"], case["head_dim"], case["block"], case["format"], _slots(case)
    keys = _values_of(s["keys"].view(kv, slots, d), fmt)
    values = _values_of(_transpose_out(s["values"], kv, slots, d).contiguous(), fmt)
    return [x * s[n].repeat_interleave(block, 1)[..., None] for x, n in ((keys, "keys_scales"), (values, "values_scales"))]


def _appended(s):
    """What the blocks from the new tokens' first on hold after the append, as fp32 rows."""
    case = s["case"]
    t, kv, d, past = case["tokens"], case["kv_heads"], case["head_dim"], case["past"]
    k = _rotate(s["k"].view(t, kv, d), s["position"], s["frequencies"])
    out = []
    for name, new in (("keys", k), ("values", s["v"].view(t, kv, d))):
        rows = torch.cat([s[name + "_open"][:, :past % case["block"]], new.transpose(0, 1)], 1)
        codes, scales = _encode(rows, case["block"], case["format"])
        out.append((codes * scales.repeat_interleave(case["block"], 1)[..., None])[:, :rows.shape[1]])
    return out


def _attend(q, keys, values, past, heads):
    """Causal attention of q [T x heads x d] over fp32 keys and values [kv x n x d]."""
    t, _, d = q.shape
    kv, n = keys.shape[:2]
    group = heads // kv
    rows = q.view(t, kv, group, d).permute(1, 2, 0, 3).reshape(kv, group * t, d)
    scores = torch.bmm(rows, keys.transpose(1, 2).contiguous()).view(kv, group, t, n) / math.sqrt(d)
    if t > 1:
        scores.masked_fill_(torch.arange(n, device=q.device)[None] > past + torch.arange(t, device=q.device)[:, None], float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = torch.bmm(p.view(kv, group * t, n), values).view(kv, group, t, d)
    return out.permute(2, 0, 1, 3).reshape(t, heads * d)


def _process(s):
    case, x = s["case"], s["logits"]
    rows, n, length = case["rows"], case["n"], case["history"]
    at = torch.arange(length, device=x.device)[None]
    history = s["history"].long()
    counted = (at < s["lengths"][:, None]) & (history >= 0) & (history < n)
    seen, count = torch.zeros((2, rows, n), device=x.device)
    where = history.clamp(0, n - 1)
    seen.scatter_add_(1, where, counted.float())
    count.scatter_add_(1, where, (counted & (at >= s["starts"][:, None])).float())
    x = torch.where(seen > 0, torch.where(x > 0, x / REPETITION, x * REPETITION), x)
    x = x - (count * FREQUENCY + (count > 0).float() * PRESENCE)
    if case["bias"]:
        entry = torch.full((n,), -1, dtype=torch.int64, device=x.device)  # of a token given twice the later bias holds
        entry.scatter_reduce_(0, s["bias_tokens"].long(), torch.arange(case["bias"], device=x.device), "amax")
        x = x + torch.where(entry >= 0, s["bias_values"][entry.clamp(min=0)], 0.0)
    if case["mask"]:
        i = torch.arange(n, device=x.device)
        x = torch.where((s["allowed"][:, i // 32] >> (i % 32)) & 1 > 0, x, float("-inf"))
    return x


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    kind = case["kind"]
    if kind == "logits":
        return _process(state)
    t, heads, d, past = case["tokens"], case["heads"], case["head_dim"], case["past"]
    n = past + t
    if kind == "attention":
        keys, values = _held(state)
        return _attend(state["q"].view(t, heads, d), keys[:, :n].contiguous(), values[:, :n].contiguous(), past, heads)
    q = _rotate(state["q"].view(t, heads, d), state["position"], state["frequencies"])
    new_keys, new_values = _appended(state)
    if kind == "append":
        return {"q": q.reshape(t, heads * d), "keys": new_keys, "values": new_values}
    keys, values = _held(state)
    first = state["read"][0]
    keys = torch.cat([keys[:, :first], new_keys], 1)
    values = torch.cat([values[:, :first], new_values], 1)
    return {"context": _attend(q, keys, values, past, heads), "keys": new_keys, "values": new_values}


# ---- what a pass cannot do without -----------------------------------------------------------

def work(case):
    if case["kind"] == "logits":
        rows, n = case["rows"], case["n"]
        return {"bytes": rows * (8.0 * n + 4.0 * case["history"] + (n / 8.0 if case["mask"] else 0.0)) + 8.0 * case["bias"], "flops": 4.0 * rows * n}
    t, past, h, kv, d, block = (case[x] for x in ("tokens", "past", "heads", "kv_heads", "head_dim", "block"))
    held = past % block  # tokens of the open block
    append = 4.0 * (2 * t * h * d + 2 * t * kv * d) + 2.0 * t * kv * d + 8.0 * kv * d * (held + t)  # with the rows read back
    attend = 2.0 * kv * (past + t) * d + 8.0 * kv * (past + t) / block + 8.0 * t * h * d
    pairs = t * past + t * (t + 1) // 2
    if case["kind"] == "append":
        return {"bytes": append, "flops": 6.0 * t * (h + kv) * d}
    if case["kind"] == "attention":
        return {"bytes": attend, "flops": 4.0 * pairs * h * d}
    return {"bytes": attend + 4.0 * 2 * kv * d + 8.0 * kv * d * (held + 1), "flops": 4.0 * pairs * h * d}


# ---- the same from the definition, in 64 bits ---------------------------------------------------

def _nearest(y):
    """Whole numbers, ties to even."""
    lower = torch.floor(y)
    part = y - lower
    return lower + ((part > 0.5) | ((part == 0.5) & (lower.remainder(2) == 1))).double()


def _exact_rows(rows, fmt, block):
    """What a cache holds of fp32 rows [count x d] of one head; the format's own roundings (the
    scale, its reciprocal, their products with the rows, the codes) as it defines them."""
    count, d = rows.shape
    held, whole = [], count // block * block
    for part, size in ((rows[:whole], block), (rows[whole:], count - whole)):
        if part.shape[0] == 0:
            continue
        x = part.double().reshape(-1, size * d)
        s = (torch.maximum(x.max(1, keepdim=True)[0], -x.min(1, keepdim=True)[0]) / QMAX[fmt]).float().double().clamp(min=2.0 ** -120)
        y = (x * (1.0 / s).float().double()).float().double()
        if fmt == "int8":
            code = _nearest(y)
        else:  # three bits after the leading one, down to multiples of 2^-9
            step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
            code = torch.sign(y) * _nearest(y.abs() / step) * step
        held.append((code.clamp(-QMAX[fmt], QMAX[fmt]) * s).view(-1, d))
    return torch.cat(held)


def _exact_rotated(x, past, freq, steps):
    """Rotary positions in 64 bits; with `steps` rounded to fp32 as the operator defines a cached key."""
    t, heads, d = x.shape
    r = (lambda y: y.float().double()) if steps else (lambda y: y)
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    angle = (torch.arange(past, past + t, device=x.device).float()[:, None] * freq).double()[:, None]
    c, s = r(torch.cos(angle)), r(torch.sin(angle))
    x = x.double()
    out[..., :d // 2] = r(r(x[..., :d // 2] * c) - r(x[..., d // 2:] * s))
    out[..., d // 2:] = r(r(x[..., :d // 2] * s) + r(x[..., d // 2:] * c))
    return out


def _exact_context(q, keys, values, past, group):
    """q [T x heads x d] over what the cache holds [kv x n x d], all in 64 bits, a head at a time."""
    t, heads, d = q.shape
    out = torch.empty((t, heads, d), dtype=torch.float64, device=q.device)
    last = past + torch.arange(t, device=q.device)
    hidden = torch.arange(keys.shape[1], device=q.device)[None, :] > last[:, None]
    for h in range(heads):
        score = (q[:, h] @ keys[h // group].t().contiguous()).div_(math.sqrt(d)).masked_fill_(hidden, -math.inf)
        weight = torch.softmax(score, 1)
        out[:, h] = weight @ values[h // group]
    return out.view(t, heads * d)


def _exact_logits(case, seed):
    s = _logits_inputs(case, seed)
    out = s["logits"].double()
    lengths, starts = s["lengths"].tolist(), s["starts"].tolist()
    rows, n = out.shape
    biases = dict(zip(s["bias_tokens"].tolist(), s["bias_values"].double().tolist())) if case["bias"] else {}
    # the coefficients as the call takes them, in fp32
    repetition, frequency, presence = (float(torch.tensor(c, dtype=torch.float32)) for c in (REPETITION, FREQUENCY, PRESENCE))
    for r in range(rows):
        text = s["history"][r, :lengths[r]].long()
        tail = text[starts[r]:]
        seen = torch.unique(text[(text >= 0) & (text < n)])
        out[r, seen] = torch.where(out[r, seen] > 0, out[r, seen] / repetition, out[r, seen] * repetition)
        said, times = torch.unique(tail[(tail >= 0) & (tail < n)], return_counts=True)
        out[r, said] -= times.double() * frequency + presence
    for token, value in biases.items():
        out[:, token] += value
    if case["mask"]:
        bits = (s["allowed"][:, :, None] >> torch.arange(32, device=out.device, dtype=torch.int32)) & 1
        out[bits.reshape(rows, -1)[:, :n] == 0] = -math.inf
    return out


def exact(case, seed):
    if case["kind"] == "logits":
        return _exact_logits(case, seed)
    t, past, heads, kv, d, block, fmt = (case[x] for x in ("tokens", "past", "heads", "kv_heads", "head_dim", "block", "format"))
    q, k, v = _tokens_in(case, seed)
    freq = _frequencies(d).cuda()
    q = q.view(t, heads, d)
    if case["kind"] == "attention":
        held = [torch.stack([_exact_rows(r, fmt, block) for r in _rows(case, seed, part, past + t)]) for part in (10, 20)]
        return _exact_context(q.double(), held[0], held[1], past, heads // kv)
    k = _exact_rotated(k.view(t, kv, d), past, freq, True).float()
    new = [x.transpose(0, 1) for x in (k, v.view(t, kv, d))]
    first = past // block * block
    if case["kind"] == "append":
        old = [_rows(case, seed, part, past)[:, first:] if past else x[:, :0] for part, x in zip((10, 20), new)]
    else:
        old = [_rows(case, seed, part, past) if past else x[:, :0] for part, x in zip((10, 20), new)]
    held = [torch.stack([_exact_rows(torch.cat([o[h], x[h]]), fmt, block) for h in range(kv)]) for o, x in zip(old, new)]
    q = _exact_rotated(q, past, freq, False)
    if case["kind"] == "append":
        return {"q": q.reshape(t, heads * d), "keys": held[0], "values": held[1]}
    return {"context": _exact_context(q, held[0], held[1], past, heads // kv), "keys": held[0][:, first:], "values": held[1][:, first:]}
