"""Cases of the operators beside the packed linears of a decode step: the 8-bit key/value cache (append, attend) and the
log probabilities of tokens.  ``run`` computes a case either in plain torch operations or through the package."""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_TOP = {"int8": 127.0, "e4m3": 448.0}
_LEAST = 2.0 ** -60            # smallest absolute maximum that a block's scale is made of


# ---------------------------------------------------------------------------------------------------------------- cases

def _append(name, seqs, least_new, new, shortest, longest, kv_heads, dim, block, fmt, dtype):
    return {"name": name, "op": "append", "seqs": seqs, "least_new": least_new, "new": new, "shortest": shortest, "longest": longest,
            "kv_heads": kv_heads, "dim": dim, "block": block, "fmt": fmt, "dtype": dtype}


def _attend(name, seqs, least_new, new, shortest, longest, q_heads, kv_heads, dim, block, fmt, dtype, window=0):
    return {"name": name, "op": "attend", "seqs": seqs, "least_new": least_new, "new": new, "shortest": shortest,
            "longest": longest, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "block": block, "fmt": fmt,
            "dtype": dtype, "window": window}


def _logprobs(name, rows, vocab, dtype, top, masked):
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "dtype": dtype, "top": top, "masked": masked}


def listed():
    return [
        # a decode step of 64 sequences writes one token each into the cache of one layer (8 key heads of 128)
        _append("append_step", 64, 1, 1, 130, 4001, 8, 128, 64, "int8", "bf16"),
        # prompts of a batch, ragged, written for the first time or behind a cached prefix
        _append("append_prompts", 8, 700, 4096, 700, 5000, 8, 128, 64, "e4m3", "bf16"),
        # one user, a short conversation: 32 heads of 128 without sharing; latency counts
        _attend("attend_one", 1, 1, 1, 517, 517, 32, 32, 128, 64, "int8", "bf16"),
        # a serving batch of ragged lengths, eight query heads to a key head
        _attend("attend_batch", 64, 1, 1, 257, 8191, 64, 8, 128, 64, "int8", "bf16"),
        # one user with a very long context
        _attend("attend_long", 1, 1, 1, 131071, 131071, 64, 8, 128, 128, "e4m3", "bf16"),
        # a few drafted tokens of each sequence are checked at once; small heads, small blocks, a sliding window
        _attend("attend_draft", 16, 3, 5, 100, 4000, 32, 8, 64, 16, "e4m3", "fp16", 2048),
        # a prompt of one user from its first token, heads without sharing
        _attend("attend_prompt", 1, 2048, 2048, 2048, 2048, 32, 32, 128, 64, "int8", "bf16"),
        # a part of a long prompt behind 15000 tokens that are in the cache already
        _attend("attend_chunk", 1, 1024, 1024, 16384, 16384, 64, 8, 128, 128, "e4m3", "bf16"),
        # one sampled token whose alternatives are shown; latency counts
        _logprobs("logprobs_one", 1, 32000, "fp32", 5, 0.0),
        # the answers of a serving batch, constrained to a part of a large vocabulary
        _logprobs("logprobs_batch", 64, 131072, "bf16", 20, 0.3),
        # scoring a text (perplexity), a vocabulary of odd size, no alternatives
        _logprobs("logprobs_score", 2047, 32003, "bf16", 0, 0.0),
        # scoring with the strongest alternatives of every position
        _logprobs("logprobs_tops", 1024, 131072, "fp32", 8, 0.0),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1)) ))))


def draw(rng):
    kind = rng.choice(["append", "append", "step", "step", "step", "draft", "prompt", "prompt", "logprobs", "logprobs", "logprobs"])
    if kind == "logprobs":
        vocab = _log_int(rng, 4000, 131072)
        rows = _log_int(rng, 1, max(1, min(4096, 134000000 // vocab)))
        case = _logprobs("", rows, vocab, rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.choice([0, 1, 5, 8, 20]),
                         rng.choice([0.0, 0.0, 0.3, 0.95]))
        del case["name"]
        return case
    fmt, dtype = rng.choice(["int8", "e4m3"]), rng.choice(["bf16", "bf16", "fp16"])
    dim, block = rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 64, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 32])
    if kind == "append":
        new = _log_int(rng, 1, 4096)
        seqs = _log_int(rng, 1, max(1, min(128, 23000 * 8 * 128 // (new * kv_heads * dim))))
        longest = new + _log_int(rng, 1, 4096)
        case = _append("", seqs, rng.randint(max(1, new // 4), new), new, rng.randint(new, longest), longest, kv_heads, dim, block,
                       fmt, dtype)
    else:
        group = rng.choice([1, 3, 4, 8, 8, 16]) if kv_heads < 32 else 1
        window = rng.choice([0, 0, 0, 300, 2048])
        if kind == "prompt":
            longest = _log_int(rng, 200, 16384)
            # the plain form holds the scores of all pairs; no more of them than the largest listed prompt has
            new = _log_int(rng, 64, max(64, min(longest, 4096, 1000000000 // (longest * kv_heads * group))))
            new = min(new, longest)
            seqs = _log_int(rng, 1, max(1, min(8, 1000000000 // (longest * new * kv_heads * group))))
            least = rng.randint(max(1, new // 4), new)
        else:
            new = 1 if kind == "step" else rng.randint(2, 8)
            longest = _log_int(rng, 16, 131072)
            seqs = _log_int(rng, 1, max(1, min(128, 270000 * 8 * 128 // (longest * kv_heads * dim))))
            least = 1 if kind == "step" else rng.randint(1, new)
        shortest = rng.randint(max(new, longest // 20), longest) if longest >= new else new
        case = _attend("", seqs, least, new, min(shortest, max(longest, new)), max(longest, new), kv_heads * group, kv_heads, dim,
                       block, fmt, dtype, window)
    del case["name"]
    return case


def _spread(low, high, count):
    """`count` whole numbers from `high` down to `low`, evenly."""
    return [high - (high - low) * i // max(1, count - 1) for i in range(count)]


def _sequences(case):
    """(tokens held, new tokens) of each sequence; the seed only orders them."""
    return list(zip(_spread(case["shortest"], case["longest"], case["seqs"]), _spread(case["least_new"], case["new"], case["seqs"])))


def _pairs(length, new, window):
    """Visible (query, key) pairs of a sequence, and the keys that any of its queries sees."""
    first = length - new
    if not window:
        return new * first + new * (new + 1) // 2, length
    return sum(min(p + 1, window) for p in range(first, length)), min(length, new + window - 1)


def work(case):
    if case["op"] == "logprobs":
        size = 4 if case["dtype"] == "fp32" else 2
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (8 + 8 + case["top"] * 12), "flops": 6 * n}
    seqs = _sequences(case)
    if case["op"] == "append":
        size = 4 if case["dtype"] == "fp32" else 2
        new = sum(n for _, n in seqs) * case["kv_heads"] * case["dim"] * 2
        back = sum(min(length, _last(case)) for length, _ in seqs) * case["kv_heads"] * case["dim"] * 2
        return {"bytes": new * (size + 1) + back * (1 + 4), "flops": 4 * new + back}
    pairs = keys = 0
    for length, new in seqs:
        p, k = _pairs(length, new, case["window"])
        pairs, keys = pairs + p, keys + k
    rows = sum(n for _, n in seqs) * case["q_heads"] * case["dim"]
    return {"bytes": keys * case["kv_heads"] * case["dim"] * 2 + keys // case["block"] * case["kv_heads"] * 8 + rows * 4,
            "flops": 4 * pairs * case["q_heads"] * case["dim"]}


def _last(case):
    """Tokens that an append is read back for: the new ones and those that lie in a block with them."""
    return case["new"] + case["block"] - 1


# --------------------------------------------------------------------------------------------------------------- inputs

def _lay_keys(codes):
    """[..., T, D] codes -> the cache's order: groups of 16 tokens, in them chunks of 32 values, in them 16 bytes for each of
    8 x 4 places: the place (token / 4 % 4, token % 2, value / 8 % 4) holds 8 values of a token and of the one two behind it."""
    lead, (T, D) = codes.shape[:-2], codes.shape[-2:]
    n = len(lead)
    x = codes.reshape(*lead, T // 16, 4, 2, 2, D // 32, 4, 8)
    return x.permute(*range(n), n, n + 4, n + 1, n + 3, n + 5, n + 2, n + 6).reshape(*lead, T, D)


def _lay_values(codes):
    """The same for values: the place (value % 8, token / 4 % 4) holds 4 tokens of 4 values that are 8 apart."""
    lead, (T, D) = codes.shape[:-2], codes.shape[-2:]
    n = len(lead)
    x = codes.reshape(*lead, T // 16, 4, 4, D // 32, 4, 8)
    return x.permute(*range(n), n, n + 3, n + 5, n + 1, n + 4, n + 2).reshape(*lead, T, D)


def _keys_of(laid):
    lead, (T, D) = laid.shape[:-2], laid.shape[-2:]
    n = len(lead)
    x = laid.reshape(*lead, T // 16, D // 32, 4, 2, 4, 2, 8)
    return x.permute(*range(n), n, n + 2, n + 5, n + 3, n + 1, n + 4, n + 6).reshape(*lead, T, D)


def _values_of(laid):
    lead, (T, D) = laid.shape[:-2], laid.shape[-2:]
    n = len(lead)
    x = laid.reshape(*lead, T // 16, D // 32, 8, 4, 4, 4)
    return x.permute(*range(n), n, n + 3, n + 5, n + 1, n + 4, n + 2).reshape(*lead, T, D)


def _decode(codes, fmt):
    """uint8 codes -> fp32 values at scale 1."""
    return codes.view(torch.float8_e4m3fn).float() if fmt == "e4m3" else codes.float() - 128


def _encode(x, fmt):
    """fp32 values at scale 1 -> uint8 codes, to the nearest, ties to even."""
    x = torch.nan_to_num(x, nan=0.0, posinf=_TOP[fmt], neginf=-_TOP[fmt]).clamp(-_TOP[fmt], _TOP[fmt])
    return x.to(torch.float8_e4m3fn).view(torch.uint8) if fmt == "e4m3" else (torch.round(x) + 128).to(torch.uint8)


def _device():
    return "cuda" if torch.cuda.is_available() else "cpu"


def prepare(case, seed):
    dev = _device()
    g = torch.Generator(dev).manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g, device=dev)                                      # noqa: E731
    if case["op"] == "logprobs":
        # logits of a trained head: most tokens in a bell, a few far above it, some masked by a grammar
        rows, vocab, dtype = case["rows"], case["vocab"], _DTYPES[case["dtype"]]
        logits = normal(rows, vocab).mul_(2.0)
        peaks = torch.randint(0, vocab, (rows, 24), generator=g, device=dev)
        logits.scatter_add_(1, peaks, normal(rows, 24).abs().mul_(6.0))
        tokens = torch.where(torch.rand(rows, generator=g, device=dev) < 0.7, peaks[:, 0],
                             torch.randint(0, vocab, (rows,), generator=g, device=dev))
        if case["masked"]:
            banned = torch.rand(vocab, generator=g, device=dev) < case["masked"]
            banned[tokens] = False
            logits.masked_fill_(banned, -math.inf)
        return {"case": dict(case), "logits": logits.to(dtype), "tokens": tokens}
    # the pool has a fifth more blocks than the sequences hold, which lie in it in no order
    S, T, H, D, fmt = case["seqs"], case["block"], case["kv_heads"], case["dim"], case["fmt"]
    order = torch.randperm(S, generator=torch.Generator().manual_seed(seed)).tolist()
    seqs = [_sequences(case)[i] for i in order]
    width = -(-case["longest"] // T)
    held = [-(-length // T) for length, _ in seqs]
    blocks = sum(held) + sum(held) // 5 + 1
    free = torch.randperm(blocks, generator=g, device=dev).int()
    table = torch.zeros(S, width, dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(held):
        table[i, :n] = free[at:at + n]
        at += n
    starts = [0]
    for _, n in seqs:
        starts.append(starts[-1] + n)
    lengths = torch.tensor([length for length, _ in seqs], dtype=torch.int32, device=dev)
    state = {"case": dict(case), "table": table, "lengths": lengths, "starts": torch.tensor(starts, dtype=torch.int32, device=dev)}
    # keys have a few strong channels, values do not; blocks differ in size
    channels = torch.ones(H, 1, D, device=dev)
    channels[:, :, ::37] = 6.0
    dtype = _DTYPES[case["dtype"]]
    for what in ("keys", "values"):
        unit = {"keys": 8.0, "values": 32.0}[what] * (1.0 if fmt == "int8" else 3.5)      # codes of a key or value of 1
        codes = _encode(normal(blocks, H, T, D) * (channels if what == "keys" else 1.0) * unit, fmt)
        state[what] = (_lay_keys if what == "keys" else _lay_values)(codes).contiguous()
        state[what[:-1] + "_scales"] = (torch.rand(blocks, H, generator=g, device=dev) * 0.5 + 0.75) / unit
        del codes
    if case["op"] == "append":
        state["k"] = (normal(starts[-1], H, D) * channels[:, 0]).to(dtype)
        state["v"] = normal(starts[-1], H, D).to(dtype)
    else:
        state["q"] = (normal(starts[-1], case["q_heads"], D) * 2.0).to(dtype)
    return state


# ------------------------------------------------------------------------------------------------------- the plain forms

def _plain_append(s):
    """Blocks that receive tokens are gathered, decoded, given their new scales and written back whole."""
    c, table, lengths, starts = s["case"], s["table"], s["lengths"].long(), s["starts"].long()
    T, D, H, fmt = c["block"], c["dim"], c["kv_heads"], c["fmt"]
    dev = table.device
    new = starts[1:] - starts[:-1]
    first = lengths - new
    touched = -(-c["new"] // T) + 1
    index = (first // T)[:, None] + torch.arange(touched, device=dev)                    # [S, touched] blocks of a sequence
    position = index[:, :, None] * T + torch.arange(T, device=dev)                       # [S, touched, T]
    is_new = (position >= first[:, None, None]) & (position < lengths[:, None, None])
    is_old = position < first[:, None, None]
    row = (starts[:-1, None, None] + position - first[:, None, None]).clamp(0, s["k"].shape[0] - 1)
    hit = is_new.any(-1)
    at = table.long().gather(1, index.clamp(max=table.shape[1] - 1))[hit]                # the pool's blocks, each once
    is_new, is_old, row = is_new[hit][:, None, :, None], is_old[hit][:, None, :, None], row[hit]
    for what, x in (("keys", s["k"]), ("values", s["v"])):
        lay, of = (_lay_keys, _keys_of) if what == "keys" else (_lay_values, _values_of)
        scales = s[what[:-1] + "_scales"]
        x = x.float()[row].transpose(1, 2)                                               # [hit, H, T, D]
        size = torch.where(is_new & torch.isfinite(x), x.abs(), 0.0).amax((-1, -2)).clamp(min=_LEAST)
        had = is_old.any(-2).squeeze(-1)
        old = torch.where(had, scales[at], 0.0)
        scale = torch.maximum(old, size / torch.full_like(size, _TOP[fmt]))[..., None, None]
        before = of(s[what][at])
        codes = torch.where(is_new, _encode(x / scale, fmt),
                            torch.where(is_old & (scale > old[..., None, None]),
                                        _encode(_decode(before, fmt) * old[..., None, None] / scale, fmt), before))
        s[what][at] = lay(codes)
        scales[at] = scale[..., 0, 0]
    # what the last tokens stand for now
    last = _last(c)
    position = lengths[:, None] - last + torch.arange(last, device=dev)
    ok = position >= 0
    position = position.clamp(min=0)
    at = table.long().gather(1, position // T)
    found = []
    for what in ("keys", "values"):
        got = _decode(_at(s[what], at, position % T, what), fmt)
        got = got * s[what[:-1] + "_scales"][at][..., None]
        found.append(torch.where(ok[:, :, None, None], got, 0.0))
    return {"k": found[0], "v": found[1]}


def _at(laid, block, token, what):
    """Codes [S, n, H, D] of single tokens of blocks, by their places in the cache's order."""
    H, T, D = laid.shape[1:]
    d = torch.arange(D, device=laid.device)
    t = token[..., None]
    group, kk = t // 16, t % 16
    if what == "keys":
        place = (2 * (kk // 4) + kk % 2) * 4 + d % 32 // 8
        offset = group * 16 * D + d // 32 * 512 + place * 16 + kk // 2 % 2 * 8 + d % 8
    else:
        place = d % 8 * 4 + kk // 4
        offset = group * 16 * D + d // 32 * 512 + place * 16 + d % 32 // 8 * 4 + kk % 4
    base = (block[..., None] * H + torch.arange(H, device=laid.device)) * (T * D)
    return laid.reshape(-1)[base[..., None] + offset[:, :, None, :]]


def _plain_attend(s):
    """All sequences padded to the longest; scores of all pairs, masked, exponentials, products."""
    c, table, lengths, starts, q = s["case"], s["table"].long(), s["lengths"].long(), s["starts"].long(), s["q"]
    T, D, H, fmt, G = c["block"], c["dim"], c["kv_heads"], c["fmt"], c["q_heads"] // c["kv_heads"]
    S, dev, most = c["seqs"], table.device, c["new"]
    L = table.shape[1] * T

    def dense(what, of):
        x = _decode(of(s[what][table]), fmt) * s[what[:-1] + "_scales"][table][..., None, None]          # [S, width, H, T, D]
        return x.transpose(1, 2).reshape(S, H, L, D)

    new = starts[1:] - starts[:-1]
    j = torch.arange(most, device=dev)
    row = (starts[:-1, None] + j).clamp(max=q.shape[0] - 1)                                                # [S, most]
    qs = q.float()[row].reshape(S, most, H, G, D).permute(0, 2, 3, 1, 4).reshape(S, H, G * most, D)
    position = lengths[:, None] - new[:, None] + j
    key = torch.arange(L, device=dev)
    seen = (key <= position[..., None]) & (key < lengths[:, None, None]) & (j < new[:, None])[..., None]   # [S, most, L]
    if c["window"]:
        seen = seen & (key > position[..., None] - c["window"])
    scores = (qs @ dense("keys", _keys_of).transpose(-1, -2)).mul_(1 / math.sqrt(D)).view(S, H, G, most, L)
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(torch.isfinite(top), top, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(S, H, G * most, L) @ dense("values", _values_of)).view(S, H, G, most, D)
    out = out / torch.where(total > 0, total, 1.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(S, most, H * G, D)
    return out[j < new[:, None]].to(q.dtype)


def _plain_logprobs(s):
    x, k = s["logits"].float(), s["case"]["top"]
    m = x.amax(-1, keepdim=True)
    y = x - m
    e = y.exp()
    total = e.sum(-1, keepdim=True)
    log_total = total.log()
    entropy = log_total[:, 0] - torch.where(e > 0, e * y, 0.0).sum(-1) / total[:, 0]
    logprob = (y.gather(1, s["tokens"][:, None]) - log_total)[:, 0]
    out = {"logprob": logprob, "entropy": entropy}
    if k:
        # values in order as whole numbers, then the lowest index first
        bits = (x + 0.0).view(torch.int32).long()
        order = torch.where(bits >= 0, bits, -(bits & 0x7fffffff) - 1) << 32
        best = (order + (0x7fffffff - torch.arange(x.shape[1], device=x.device))).topk(k, -1).indices
        out["top_logprobs"] = y.gather(1, best) - log_total
        out["top_tokens"] = best
    return out


# ------------------------------------------------------------------------------------------------------------------ runs

def _cache(state):
    """The cache's handle, which a program makes once."""
    if "cache" not in state:
        from if_i_could_turn_back_time_b200 import KVCache
        state["cache"] = KVCache(state["keys"], state["values"], state["key_scales"], state["value_scales"], state["case"]["fmt"])
    return state["cache"]


def run(state):
    case = state["case"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "logprobs": _plain_logprobs}[case["op"]](state)
    if case["op"] == "logprobs":
        from if_i_could_turn_back_time_b200 import ops
        got = ops.token_logprobs(state["logits"], state["tokens"], top=case["top"])
        out = {"logprob": got.logprob, "entropy": got.entropy}
        if case["top"]:
            out.update(top_logprobs=got.top_logprobs, top_tokens=got.top_tokens)
        return out
    cache = _cache(state)
    if case["op"] == "append":
        cache.append(state["k"], state["v"], state["table"], state["lengths"], state["starts"], max_new=case["new"])
        k, v = cache.read(state["table"], state["lengths"], last=_last(case))
        return {"k": k, "v": v}
    return cache.attend(state["q"], state["table"], state["lengths"], state["starts"], max_new=case["new"], window=case["window"])


# --------------------------------------------------------------------------------------------------- the answer in 64 bits

def _e4m3_values():
    """What the 256 codes of e4m3 stand for, by the format's definition: four exponent bits with bias 7, three of mantissa."""
    got = []
    for code in range(256):
        e, m = code >> 3 & 15, code & 7
        size = math.ldexp(m, -9) if e == 0 else math.ldexp(8 + m, e - 10)
        got.append(-size if code & 128 else size)
    return torch.tensor(got, dtype=torch.float64)


def _exact_block(laid, fmt, what):
    """Natural-order values [H, T, D], in 64 bits, of blocks [H, T * D] in the cache's order, by the place of each."""
    H, T, D = laid.shape
    t, d = torch.arange(T, device=laid.device)[:, None], torch.arange(D, device=laid.device)[None]
    if what == "keys":
        place = 32 * (t % 16 // 4) + 16 * (t % 2) + 4 * (d % 32 // 8)      # in units of 4 bytes of the 512
        offset = t // 16 * (16 * D) + d // 32 * 512 + place * 4 + t % 4 // 2 * 8 + d % 8
    else:
        offset = t // 16 * (16 * D) + d // 32 * 512 + d % 8 * 64 + t % 16 // 4 * 16 + d % 32 // 8 * 4 + t % 4
    codes = laid.reshape(H, T * D)[:, offset.reshape(-1)].reshape(H, T, D).long()
    return _e4m3_values().to(laid.device)[codes] if fmt == "e4m3" else codes.double() - 128


def _exact_sequence(s, i, length, what, blocks=None):
    """[H, tokens, D] in 64 bits of a sequence's blocks."""
    T, fmt = s["case"]["block"], s["case"]["fmt"]
    ids = s["table"][i, :-(-length // T)].tolist() if blocks is None else blocks
    laid = s[what][ids]                                                    # [n, H, T, D]
    n, H, _, D = laid.shape
    flat = _exact_block(laid.reshape(n * H, T, D), fmt, what).reshape(n, H, T, D)
    flat = flat * s[what[:-1] + "_scales"][ids].double()[..., None, None]
    return flat.permute(1, 0, 2, 3).reshape(H, n * T, D)


def _nearest(x, fmt):
    """Values of the format nearest to x (64 bits), ties to the even code."""
    top = _TOP[fmt]
    x = x.clamp(-top, top)
    if fmt == "int8":
        return torch.round(x)
    size = x.abs().clamp(min=2.0 ** -6)
    step = torch.exp2(torch.floor(torch.log2(size)) - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "logprobs":
        out = {"logprob": [], "entropy": []} | ({"top_logprobs": [], "top_tokens": []} if c["top"] else {})
        for at in range(0, c["rows"], 64):
            x = s["logits"][at:at + 64].double()
            lse = torch.logsumexp(x, -1, keepdim=True)
            lp = x - lse
            out["logprob"].append(lp.gather(1, s["tokens"][at:at + 64, None])[:, 0])
            out["entropy"].append(torch.special.entr(lp.exp()).sum(-1))
            if c["top"]:
                out["top_logprobs"].append(lp.topk(c["top"], -1).values)
        return {k: torch.cat(v) if v else None for k, v in out.items()}
    lengths, starts = s["lengths"].tolist(), s["starts"].tolist()
    if c["op"] == "append":
        T, fmt, last, H, D = c["block"], c["fmt"], _last(c), c["kv_heads"], c["dim"]
        got = {}
        for name, what in (("k", "keys"), ("v", "values")):
            every = []
            for i, length in enumerate(lengths):
                new = starts[i + 1] - starts[i]
                first = length - new
                x = torch.zeros(H, -(-length // T) * T, D, dtype=torch.float64, device=s["k"].device)
                x[:, first:length] = s[name][starts[i]:starts[i + 1]].double().transpose(0, 1)
                ids, scales = s["table"][i, :-(-length // T)].long(), s[what[:-1] + "_scales"]
                n = len(ids)
                old = scales[ids].double().T                                                       # [H, n]
                b = torch.arange(n, device=x.device)
                had = b * T < first
                old = torch.where(had, old, 0.0)
                x = x.reshape(H, n, T, D)
                position = torch.arange(n * T, device=x.device).reshape(n, T)
                fresh = ((position >= first) & (position < length))[None, :, :, None]
                size = torch.where(fresh, x.abs(), 0.0).amax((2, 3)).clamp(min=_LEAST)
                scale = torch.where(fresh[..., 0].any(-1), torch.maximum(old, size / _TOP[fmt]), old)[..., None, None]
                unit = _exact_sequence({**s, what[:-1] + "_scales": torch.ones_like(scales)}, i, length, what).reshape(H, n, T, D)
                grown = scale > old[..., None, None]
                before = torch.where(grown, _nearest(unit * old[..., None, None] / torch.where(scale > 0, scale, 1.0), fmt), unit)
                x = torch.where(fresh, _nearest(x / torch.where(scale > 0, scale, 1.0), fmt), before) * scale
                x = x.reshape(H, n * T, D)[:, max(0, length - last):length].transpose(0, 1)
                every.append(torch.cat([x.new_zeros(last - x.shape[0], H, D), x]))
            got[name] = torch.stack(every)
        return got
    G = c["q_heads"] // c["kv_heads"]
    if sum(length * (starts[i + 1] - starts[i]) for i, length in enumerate(lengths)) * c["q_heads"] > 6e9:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for i, length in enumerate(lengths):
        keys, values = (_exact_sequence(s, i, length, what)[:, :length] for what in ("keys", "values"))
        new = starts[i + 1] - starts[i]
        position = torch.arange(length - new, length, device=out.device)[:, None]
        key = torch.arange(length, device=out.device)
        hidden = (key > position) | ((key <= position - c["window"]) if c["window"] else False)
        for h in range(c["q_heads"]):
            score = s["q"][starts[i]:starts[i + 1], h].double() @ keys[h // G].T / math.sqrt(c["dim"])
            out[starts[i]:starts[i + 1], h] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ values[h // G]
    return out
