"""Timed cases of serving from a paged KV cache that is held in 4 bits: quantising rows as they are written, reading them
back, and attention over the codes.

  append     the fused projection's rows of a step: Q rotated, K rotated and quantised, V quantised, into the pages of their
             sequences; the rows written are read back, so that a pass returns what they stand for
  read       the keys and values of whole sequences, or of their last tokens, out of the pages
  attention  new tokens of every sequence against its cache of codes: one token (decoding), a few (checking drafted tokens),
             hundreds (a prompt taken in pieces), and batches that mix them

A row of a KV head is cut into groups of 64 elements. A group is held as `low`, its least element, `step`, a fifteenth of its
range rounded up, both in the cache's type, and 4-bit codes: an element stands for low + code * step.

`listed()` gives fixed representatives; `draw()` gives further cases of the same ranges. With `own` false `run` computes the
operators from elementary torch operations, in 32 bits but for the rotation of what is quantised (64 bits: a code is a
decision next to a border); with `own` true it calls this package.
"""
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
# (query heads, KV heads): grouped forms of the benchmark and of the 28-head block, a narrow shard, plain multi-head
_HEADS = ((32, 8), (28, 4), (16, 4), (8, 2), (8, 8), (32, 32))
_PAGE_SIZES = (16, 32, 64, 128)
_THETA = 500000.0
_GROUP = 64

_MAX_KEYS = 64 * 17000 * 8 * 128        # key elements of one launch
_MAX_READ = 24 * 17000 * 8 * 128
_MAX_FLOPS = 4 * 128 * 32 * 4096 * 34816

_backend_of_process = None


def _backend():
    """One backend per process, as a program holds it."""
    global _backend_of_process
    if _backend_of_process is None:
        from vibe_compiler_b200.backend import B200TargetModelBackend
        _backend_of_process = B200TargetModelBackend(torch.cuda.current_device())
    return _backend_of_process


# ------------------------------------------------------------------ cases
def _case(name, op, sequences, single, new_min, new_max, keys_min, keys_max, heads, head_dim, dtype, page_size, mix, interleaved=False):
    """`single` of the sequences bring one token, the others new_min to new_max; keys_min to keys_max keys before them. A read
    with new_max 0 takes the sequences whole."""
    return {"name": name, "op": op, "sequences": sequences, "single": single, "new_min": new_min, "new_max": new_max,
            "keys_min": keys_min, "keys_max": keys_max, "q_heads": heads[0], "kv_heads": heads[1], "head_dim": head_dim,
            "dtype": dtype, "page_size": page_size, "interleaved": interleaved, "mix": mix}


def listed():
    return [
        # one decoding step of 33 sequences: their K and V rows go to 33 different pages
        _case("append_step", "append", 33, 33, 1, 1, 0, 20000, (28, 4), 128, "f16", 16, 1),
        # drafted tokens of 64 sequences, interleaved pairs, head dimension 64
        _case("append_drafts", "append", 64, 0, 2, 9, 0, 9000, (16, 4), 64, "bf16", 32, 2, True),
        # prompts of 7 sequences taken together, ragged
        _case("append_prompts", "append", 7, 0, 300, 4000, 0, 8000, (32, 8), 128, "bf16", 64, 3),
        # three short sequences handed over to another program
        _case("read_few", "read", 3, 0, 0, 0, 700, 2000, (28, 4), 128, "bf16", 16, 4),
        # long sequences handed over whole: bandwidth
        _case("read_long", "read", 24, 0, 0, 0, 2000, 32000, (32, 8), 128, "f16", 64, 5),
        # the smallest decoding batch: latency
        _case("attention_few", "attention", 3, 3, 1, 1, 700, 2000, (28, 4), 128, "bf16", 16, 6),
        # a full decoding batch over long caches: bandwidth
        _case("attention_decode", "attention", 64, 64, 1, 1, 2000, 32000, (32, 8), 128, "f16", 64, 7),
        # many sequences of moderate length, a KV head to each query head
        _case("attention_heads", "attention", 100, 100, 1, 1, 100, 4000, (8, 8), 128, "bf16", 32, 8),
        # drafted tokens of 17 sequences checked at once, head dimension 64
        _case("attention_drafts", "attention", 17, 0, 2, 9, 900, 9000, (16, 4), 64, "bf16", 32, 9),
        # a serving step: 40 sequences decode while pieces of 8 prompts are taken in
        _case("attention_mixed", "attention", 48, 40, 100, 512, 50, 8000, (32, 8), 128, "bf16", 32, 10),
        # a piece of one long prompt behind what is already cached: tensor pipe
        _case("attention_piece", "attention", 1, 0, 4096, 4096, 32768, 32768, (32, 8), 128, "bf16", 128, 11),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("append", "read", "attention", "attention"))
    mix = rng.randrange(1 << 30)
    while True:
        heads, head_dim, dtype, size = rng.choice(_HEADS), rng.choice((64, 128)), rng.choice(("bf16", "f16")), rng.choice(_PAGE_SIZES)
        sequences, keys = _log_int(rng, 1, 128), _log_int(rng, 128, 65536)
        width = heads[1] * head_dim
        if op == "append":
            high = _log_int(rng, 1, 4000)
            case = _case("", op, sequences, 0, rng.randint(1, high), high, 0, keys, heads, head_dim, dtype, size, mix, rng.random() < 0.5)
            if sequences * (high + keys) * width <= _MAX_KEYS // 4 and sequences * high <= 16384:
                break
        elif op == "read":
            high = rng.choice((0, _log_int(rng, 1, 2000)))
            case = _case("", op, sequences, 0, rng.randint(0, high), high, rng.randint(0, keys), keys, heads, head_dim, dtype, size, mix)
            new, lengths = _lengths(case)
            if sum(lengths) * width <= _MAX_READ and sum(new) > 0:
                break
        else:
            high = _log_int(rng, 1, 4096)
            single = sequences if high == 1 else rng.choice((0, 0, sequences // 2, sequences * 7 // 8))
            case = _case("", op, sequences, single, rng.randint(max(1, high // 8), high), high, rng.randint(0, keys), keys, heads, head_dim, dtype, size, mix)
            if sum(_lengths(case)[1]) * width <= _MAX_KEYS and work(case)["flops"] <= _MAX_FLOPS:
                break
    del case["name"]
    return case


def _lengths(case):
    """New tokens and keys (the new ones among them) of every sequence: the case's own, whatever the seed."""
    rng = random.Random(case["mix"])
    pairs = []
    for s in range(case["sequences"]):
        n = 1 if s < case["single"] else rng.randint(case["new_min"], case["new_max"])
        length = n + rng.randint(case["keys_min"], case["keys_max"])
        pairs.append((length if case["new_max"] == 0 else n, length))
    rng.shuffle(pairs)
    return [n for n, _ in pairs], [length for _, length in pairs]


# ------------------------------------------------------------------ inputs
def _quantised(x):
    """Rows x [..., head_dim] as (codes, uint8 [..., head_dim / 2], two to a byte, the even element in the low half; steps [..., groups, 2],
    (step, low) in x's type)."""
    dtype = x.dtype
    x = x.float().unflatten(-1, (-1, _GROUP))
    low, high = x.amin(-1), x.amax(-1)
    wanted = (high - low) / torch.full_like(low, 15.0)             # a true division: one by a number is a product with 1 / 15, rounded
    step = wanted.to(dtype)
    short = step.float() < wanted                                  # rounded up: fifteen steps reach the largest element
    step = (step.view(torch.int16) + short.to(torch.int16)).view(dtype)
    codes = torch.where(step[..., None] > 0, (x - low[..., None]) / step.float()[..., None], 0.0).round().clamp(max=15.0).to(torch.uint8)
    codes = codes.flatten(-2).unflatten(-1, (-1, 2))
    return codes[..., 0] | (codes[..., 1] << 4), torch.stack((step, low.to(dtype)), dim=-1)


def _decoded(codes, steps, dtype=torch.float32):
    """The values that codes and steps of _quantised stand for."""
    codes = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).unflatten(-1, (-1, _GROUP)).to(dtype)
    steps = steps.to(dtype)
    return (codes * steps[..., :1] + steps[..., 1:]).flatten(-2)


def _filled(pages, case, g, device):
    """Codes and steps of a cache of random rows; the heads lie outside the rows in memory. [pages, page_size, kv_heads, ...]"""
    size, heads, d, dtype = case["page_size"], case["kv_heads"], case["head_dim"], _DTYPES[case["dtype"]]
    codes = torch.empty(pages, heads, size, d // 2, dtype=torch.uint8, device=device)
    steps = torch.empty(pages, heads, size, d // _GROUP, 2, dtype=dtype, device=device)
    at_once = max(1, (1 << 27) // (size * heads * d))
    for first in range(0, pages, at_once):
        part = slice(first, min(pages, first + at_once))
        x = torch.randn(codes[part].shape[:3] + (d,), generator=g, device=device, dtype=dtype)
        codes[part], steps[part] = _quantised(x)
    return codes.transpose(1, 2), steps.transpose(1, 2)


def _place(lengths, page_size, pages, width, seed):
    """A page table with the sequences' pages anywhere in the pool; entries behind a sequence's pages are -1."""
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(lengths):
        count = -(-n // page_size)
        table[s, :count] = order[at:at + count].sort().values if s % 2 else order[at:at + count]
        at += count
    return table


def prepare(case, seed):
    device = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device="cuda").manual_seed(seed)
    new, lengths = _lengths(case)
    size, dtype, d = case["page_size"], _DTYPES[case["dtype"]], case["head_dim"]
    counts = [-(-n // size) for n in lengths]
    pages, tokens = sum(counts) + 7, sum(new)
    state = {"case": case, "new": new, "lengths": lengths, "tokens": tokens}
    state["k_codes"], state["k_steps"] = _filled(pages, case, g, device)
    state["v_codes"], state["v_steps"] = _filled(pages, case, g, device)
    state["page_table"] = _place(lengths, size, pages, max(counts) + 3, seed).to(device)
    state["key_lengths"] = torch.tensor(lengths, dtype=torch.int32, device=device)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    state["starts"] = starts
    state["query_starts"] = torch.tensor(starts, dtype=torch.int32, device=device)
    if case["op"] == "append":
        state["qkv"] = torch.randn(tokens, (case["q_heads"] + 2 * case["kv_heads"]) * d, generator=g, device=device, dtype=dtype)
        state["frequencies"] = _frequencies(d).to(device)
    if case["op"] == "attention":
        state["q"] = torch.randn(tokens, case["q_heads"], d, generator=g, device=device, dtype=dtype)
    if own:                                            # the handles, which a program keeps as long as what they stand for
        from vibe_compiler_b200.paged_cache import QuantizedCache, RotaryTable
        state["cache"] = QuantizedCache(state["k_codes"], state["k_steps"], state["v_codes"], state["v_steps"])
        state["rotary"] = RotaryTable(d, theta=_THETA)
    return state


def _frequencies(head_dim):
    return _THETA ** (-2.0 * torch.arange(head_dim // 2, dtype=torch.float64) / head_dim)


# ------------------------------------------------------------------ a pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    from vibe_compiler_b200.paged_cache import PagedBatch
    case, backend, cache = state["case"], _backend(), state["cache"]
    batch = PagedBatch(state["page_table"], state["key_lengths"], state["query_starts"], max_query=max(state["new"]))
    if case["op"] == "attention":
        return backend.attention_paged(state["q"], cache, batch, case["head_dim"] ** -0.5, causal=True)
    if case["op"] == "read":
        return backend.cache_read(cache, batch, state["tokens"])
    q = backend.rope_append(state["qkv"], cache, batch, state["rotary"], q_heads=case["q_heads"], interleaved=case["interleaved"])
    return (q, *backend.cache_read(cache, batch, state["tokens"]))


def _slots(state):
    """(position of every new token, its page, its row in the page)."""
    case, device = state["case"], state["page_table"].device
    counts = state["query_starts"][1:] - state["query_starts"][:-1]
    sequence = torch.repeat_interleave(torch.arange(case["sequences"], device=device), counts.long(), output_size=state["tokens"])
    tokens = torch.arange(state["tokens"], device=device)
    position = tokens - state["query_starts"].long()[sequence] + (state["key_lengths"] - counts).long()[sequence]
    page = state["page_table"][sequence, position // case["page_size"]].long()
    return position, page, position % case["page_size"]


def _rotated(x, angles, interleaved):
    """x [tokens, heads, head_dim], turned in its own precision; angles [tokens, pairs] in 64 bits."""
    cos, sin = angles.cos().to(x.dtype)[:, None], angles.sin().to(x.dtype)[:, None]
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else x.chunk(2, dim=-1)
    turned = (a * cos - b * sin, b * cos + a * sin)
    return torch.stack(turned, dim=-1).flatten(-2) if interleaved else torch.cat(turned, dim=-1)


def _rows(state, page, row):
    """K and V rows as they stand in the cache, in its type."""
    dtype = state["k_steps"].dtype
    return tuple(_decoded(state[x + "_codes"][page, row], state[x + "_steps"][page, row]).to(dtype) for x in "kv")


def _run_plain(state):
    case = state["case"]
    if case["op"] == "attention":
        return _attention(state)
    position, page, row = _slots(state)
    if case["op"] == "read":
        return _rows(state, page, row)
    hq, hk = case["q_heads"], case["kv_heads"]
    rows = state["qkv"].view(-1, hq + 2 * hk, case["head_dim"])
    angles = position.double()[:, None] * state["frequencies"]
    q = _rotated(rows[:, :hq].float(), angles, case["interleaved"]).to(rows.dtype)
    k = _rotated(rows[:, hq:hq + hk].double(), angles, case["interleaved"]).float().to(rows.dtype)
    state["k_codes"][page, row], state["k_steps"][page, row] = _quantised(k)
    state["v_codes"][page, row], state["v_steps"][page, row] = _quantised(rows[:, hq + hk:])
    return (q, *_rows(state, page, row))


def _attention(state):
    case = state["case"]
    hq, hk, d, size = case["q_heads"], case["kv_heads"], case["head_dim"], case["page_size"]
    group, scale = hq // hk, case["head_dim"] ** -0.5
    q_all = state["q"]
    out = torch.empty_like(q_all)
    for s, (n, length) in enumerate(zip(state["new"], state["lengths"])):
        pages = state["page_table"][s, :-(-length // size)].long()
        k = _decoded(state["k_codes"][pages], state["k_steps"][pages]).reshape(-1, hk, d)[:length].permute(1, 2, 0)       # [hk, d, keys]
        v = _decoded(state["v_codes"][pages], state["v_steps"][pages]).reshape(-1, hk, d)[:length].transpose(0, 1)        # [hk, keys, d]
        step = max(1, (1 << 27) // (hq * length))
        for first in range(0, n, step):
            count = min(step, n - first)
            at = state["starts"][s] + first
            q = q_all[at:at + count].float().view(count, hk, group, d).permute(1, 2, 0, 3).reshape(hk, group * count, d)
            scores = torch.matmul(q, k).mul_(scale).view(hk, group, count, length)
            last = torch.arange(first, first + count, device=k.device) + (length - n)
            if length - n + first + 1 < length:
                scores.masked_fill_(torch.arange(length, device=k.device)[None, :] > last[:, None], -math.inf)
            top = scores.amax(-1, keepdim=True)
            p = scores.sub_(top).exp_()
            total = p.sum(-1, keepdim=True)
            o = torch.matmul(p.view(hk, group * count, length), v).view(hk, group, count, d) / total
            out[at:at + count] = o.permute(2, 0, 1, 3).reshape(count, hq, d).to(out.dtype)
    return out


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    new, lengths = _lengths(case)
    d, hq, hk = case["head_dim"], case["q_heads"], case["kv_heads"]
    held = 2 * hk * (d // 2 + 4 * (d // _GROUP))                   # bytes of a token's K and V in the cache
    plain = 2 * hk * d * 2
    if case["op"] == "read":
        return {"bytes": sum(new) * (held + plain), "flops": sum(new) * 2 * hk * d * 2}
    if case["op"] == "append":                                     # the projection's row in, Q, the codes and the rows read back out
        return {"bytes": sum(new) * (2 * hq * d * 2 + 2 * plain + held), "flops": sum(new) * (3 * (hq + hk) * d + 2 * hk * d * 8)}
    pairs = sum(n * (length - n) + n * (n + 1) // 2 for n, length in zip(new, lengths))
    return {"bytes": sum(lengths) * held + 2 * sum(new) * hq * d * 2, "flops": 4 * d * hq * pairs}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    device, size = state["page_table"].device, case["page_size"]
    if case["op"] == "attention":
        return _exact_attention(state)
    positions = torch.cat([torch.arange(length - n, length) for n, length in zip(state["new"], state["lengths"])]).to(device)
    sequence = torch.cat([torch.full((n,), s) for s, n in enumerate(state["new"])]).to(device)
    pages, rows = state["page_table"][sequence, positions // size].long(), positions % size
    if case["op"] == "read":
        return tuple(_exact_values(state[x + "_codes"][pages, rows], state[x + "_steps"][pages, rows]) for x in "kv")
    d, hq, hk = case["head_dim"], case["q_heads"], case["kv_heads"]
    x = state["qkv"].view(-1, hq + 2 * hk, d)
    angle = positions.double()[:, None, None] * _frequencies(d).to(device)
    first, second = (slice(0, d, 2), slice(1, d, 2)) if case["interleaved"] else (slice(0, d // 2), slice(d // 2, d))
    turned = torch.empty(x.shape[0], hq + hk, d, dtype=torch.float64, device=device)
    z = torch.complex(x[:, :hq + hk, first].double(), x[:, :hq + hk, second].double()) * torch.polar(torch.ones_like(angle), angle)
    turned[..., first], turned[..., second] = z.real, z.imag
    k = turned[:, hq:].float().to(x.dtype)                         # what is quantised is a value of the type
    return turned[:, :hq], _exact_quantised(k), _exact_quantised(x[:, hq + hk:])


def _exact_quantised(x):
    """The values that x's codes stand for, group by group."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for at in range(0, x.shape[-1], _GROUP):
        part = x[..., at:at + _GROUP].double()
        low = part.min(-1, keepdim=True).values
        wanted = (part.max(-1, keepdim=True).values - low) / 15
        step = wanted.to(x.dtype)
        bits = step.view(torch.int16)
        step = torch.where(step.double() < wanted, (bits + 1).view(x.dtype), step).double()
        code = torch.where(step > 0, torch.round((part - low) / step), torch.zeros_like(part)).clamp(0, 15)
        out[..., at:at + _GROUP] = low + code * step
    return out


def _exact_values(codes, steps):
    out = torch.empty(codes.shape[:-1] + (2 * codes.shape[-1],), dtype=torch.float64, device=codes.device)
    out[..., 0::2], out[..., 1::2] = codes % 16, codes // 16
    for i in range(steps.shape[-2]):
        at = slice(i * _GROUP, (i + 1) * _GROUP)
        out[..., at] = steps[..., i, 1:].double() + out[..., at] * steps[..., i, :1].double()
    return out


def _exact_attention(state):
    """Head by head, over the keys that a row sees, with the log-sum-exp first."""
    case = state["case"]
    hq, hk, d, size = case["q_heads"], case["kv_heads"], case["head_dim"], case["page_size"]
    q = state["q"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for s, (n, length) in enumerate(zip(state["new"], state["lengths"])):
        keys = torch.arange(length, device=q.device)
        pages, rows = state["page_table"][s].long()[keys // size], keys % size
        tokens = torch.arange(n, device=q.device)
        for head in range(hk):
            k, v = (_exact_values(state[x + "_codes"][pages, rows, head], state[x + "_steps"][pages, rows, head]) for x in "kv")
            for first in range(0, n, 1024):
                part = slice(first, min(first + 1024, n))
                hidden = keys[None, :] > (length - n + tokens[part])[:, None]
                for h in range(head * (hq // hk), (head + 1) * (hq // hk)):
                    at = slice(state["starts"][s] + part.start, state["starts"][s] + part.stop)
                    scores = (q[at, h].double() @ k.T) / math.sqrt(d)
                    scores[hidden] = -math.inf
                    out[at, h] = (scores - torch.logsumexp(scores, -1)[:, None]).exp() @ v
    return out
