"""Timed cases of serving from a paged KV cache: rotary positions, cache writes, attention, and the pages themselves.

Four kinds of work:

  rope       rotary positions on rows of a projection, and their gradient: every token has a position of its own
  append     the same on the fused projection's rows, the new K and V rows written into the pages of their sequences
  attention  a chunk of new tokens of every sequence against its paged cache: one token (decoding), a few (checking drafted
             tokens), hundreds (a prompt taken in pieces), and batches that mix them
  pages      the cache's pages: room for the next tokens; a step of parallel sampling that frees some sequences, forks
             others into their place and copies what cannot be shared; moving all pages together

`listed()` gives fixed representatives; `draw()` gives further cases of the same ranges. With `own` false `run` computes
the operators from elementary torch operations in 32 bits (angles in 64); with `own` true it calls this package.
"""
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# (query heads, KV heads): grouped forms of the benchmark and of the 28-head block, a narrow shard, plain multi-head
_HEADS = ((32, 8), (28, 4), (16, 4), (8, 2), (8, 8), (32, 32))
_PAGE_SIZES = (16, 32, 64, 128)
_THETA = 500000.0
_SCALINGS = ("none", "linear", "base", "wavelength", "yarn")

_MAX_ROPE = 16384 * 40 * 128            # elements
_MAX_KEYS = 64 * 17000 * 8 * 128        # key elements of one launch
_MAX_FLOPS = 4 * 128 * 32 * 4096 * 34816
_MAX_POOL = 3 << 29                     # bytes of K and V in the pages cases

_backend_of_process = None


def _backend():
    """One backend per process, as a program holds it."""
    global _backend_of_process
    if _backend_of_process is None:
        from vibe_compiler_b200.backend import B200TargetModelBackend
        _backend_of_process = B200TargetModelBackend(torch.cuda.current_device())
    return _backend_of_process


# ------------------------------------------------------------------ cases
def _rope(name, tokens, heads, head_dim, rotary_dim, dtype, interleaved, backward, scaling, longest):
    return {"name": name, "op": "rope", "tokens": tokens, "heads": heads, "head_dim": head_dim, "rotary_dim": rotary_dim,
            "dtype": dtype, "interleaved": interleaved, "backward": backward, "scaling": scaling, "longest": longest}


def _append(name, sequences, new_min, new_max, longest, heads, head_dim, dtype, page_size, interleaved, scaling, mix):
    return {"name": name, "op": "append", "sequences": sequences, "new_min": new_min, "new_max": new_max, "keys_min": 0,
            "keys_max": longest, "q_heads": heads[0], "kv_heads": heads[1], "head_dim": head_dim, "dtype": dtype,
            "page_size": page_size, "interleaved": interleaved, "scaling": scaling, "mix": mix}


def _attention(name, sequences, single, new_min, new_max, keys_min, keys_max, heads, head_dim, dtype, page_size, mix):
    """`single` of the sequences bring one token, the others new_min to new_max; keys_min to keys_max keys before them."""
    return {"name": name, "op": "attention", "sequences": sequences, "single": single, "new_min": new_min, "new_max": new_max,
            "keys_min": keys_min, "keys_max": keys_max, "q_heads": heads[0], "kv_heads": heads[1], "head_dim": head_dim,
            "dtype": dtype, "page_size": page_size, "mix": mix}


def _pages(name, op, sequences, keys_max, page_size, layers, kv_heads, dtype, part, mix):
    """`part`: forked sequences of 16 (fork), live pages of 16 (compact)."""
    return {"name": name, "op": op, "sequences": sequences, "keys_max": keys_max, "page_size": page_size, "layers": layers,
            "kv_heads": kv_heads, "head_dim": 128, "dtype": dtype, "part": part, "mix": mix}


def listed():
    return [
        # q and k heads of one decoding step of 64 sequences: latency
        _rope("rope_step", 64, 40, 128, 128, "bf16", False, False, "wavelength", 100000),
        # gradient of the rotation over a batch of 8 x 2048 tokens, interleaved pairs, three quarters of the head
        _rope("rope_gradient", 16384, 40, 128, 96, "bf16", True, True, "yarn", 131072),
        # one decoding step of 33 sequences: their K and V rows go to 33 different pages
        _append("append_step", 33, 1, 1, 20000, (28, 4), 128, "f16", 16, False, "none", 1),
        # prompts of 7 sequences taken together, ragged
        _append("append_prompts", 7, 300, 4000, 30000, (32, 8), 128, "bf16", 64, False, "linear", 2),
        # the smallest decoding batch: latency
        _attention("attention_few", 3, 3, 1, 1, 700, 2000, (28, 4), 128, "bf16", 16, 3),
        # a full decoding batch over long caches: bandwidth
        _attention("attention_decode", 64, 64, 1, 1, 2000, 32000, (32, 8), 128, "f16", 64, 4),
        # drafted tokens of 17 sequences checked at once, head dimension 64
        _attention("attention_drafts", 17, 0, 2, 9, 900, 9000, (16, 4), 64, "bf16", 32, 5),
        # a serving step: 40 sequences decode while pieces of 8 prompts are taken in
        _attention("attention_mixed", 48, 40, 100, 512, 50, 8000, (32, 8), 128, "bf16", 32, 6),
        # a piece of one long prompt behind what is already cached: tensor pipe
        _attention("attention_piece", 1, 0, 4096, 4096, 32768, 32768, (32, 8), 128, "bf16", 128, 7),
        # room for the next token of 200 sequences: latency
        _pages("pages_room", "reserve", 200, 9000, 16, 0, 8, "bf16", 0, 8),
        # parallel sampling: 6 of 16 sequences make way for forks of others, over 4 layers' caches
        _pages("pages_fork", "fork", 64, 1500, 64, 4, 8, "bf16", 6, 9),
        # a pool of which 9 of 16 pages are in use is moved together, over 2 layers' caches
        _pages("pages_compact", "compact", 48, 8000, 64, 2, 4, "f16", 9, 10),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("rope", "append", "attention", "attention", "attention", "pages"))
    mix = rng.randrange(1 << 30)
    while True:
        if kind == "rope":
            head_dim = rng.choice((64, 128))
            case = _rope("", _log_int(rng, 1, 16384), rng.choice((1, 8, 10, 32, 36, 40)), head_dim,
                         rng.choice((head_dim, head_dim // 2, head_dim * 3 // 4)), rng.choice(("bf16", "f16", "f32")),
                         rng.random() < 0.5, rng.random() < 0.5, rng.choice(_SCALINGS), _log_int(rng, 2000, 1000000))
            if case["tokens"] * case["heads"] * head_dim * (2 if case["dtype"] == "f32" else 1) <= _MAX_ROPE:
                break
        elif kind == "append":
            high = _log_int(rng, 1, 4000)
            case = _append("", _log_int(rng, 1, 128), rng.randint(1, high), high, _log_int(rng, 100, 60000), rng.choice(_HEADS),
                           rng.choice((64, 128)), rng.choice(("bf16", "f16")), rng.choice(_PAGE_SIZES), rng.random() < 0.5,
                           rng.choice(_SCALINGS), mix)
            rows = case["sequences"] * (high + case["keys_max"]) * case["kv_heads"] * case["head_dim"]
            if rows <= _MAX_KEYS // 4 and case["sequences"] * high <= 16384:
                break
        elif kind == "attention":
            sequences = _log_int(rng, 1, 128)
            high = _log_int(rng, 1, 4096)
            single = sequences if high == 1 else rng.choice((0, 0, sequences // 2, sequences * 7 // 8))
            keys = _log_int(rng, 128, 65536)
            case = _attention("", sequences, single, rng.randint(max(1, high // 8), high), high, rng.randint(0, keys), keys,
                              rng.choice(_HEADS), rng.choice((64, 128)), rng.choice(("bf16", "f16")), rng.choice(_PAGE_SIZES), mix)
            new, lengths = _lengths(case)
            elements = sum(lengths) * case["kv_heads"] * case["head_dim"]
            if elements <= _MAX_KEYS and work(case)["flops"] <= _MAX_FLOPS:
                break
        else:
            op = rng.choice(("reserve", "fork", "compact"))
            case = _pages("", op, _log_int(rng, 16, 256), _log_int(rng, 300, 20000), rng.choice(_PAGE_SIZES), rng.randint(1, 8),
                          rng.choice((2, 4, 8)), rng.choice(("bf16", "f16")), rng.randint(1, 8) if op == "fork" else rng.randint(4, 13), mix)
            pages = _pool_pages(case)
            row_bytes = case["layers"] * case["kv_heads"] * case["head_dim"] * 4
            if op == "reserve" or pages * case["page_size"] * row_bytes <= _MAX_POOL:
                break
    del case["name"]
    return case


def _lengths(case):
    """New tokens and keys (the new ones among them) of every sequence: the case's own, whatever the seed."""
    rng = random.Random(case["mix"])
    single = case.get("single", 0)
    new, lengths = [], []
    for s in range(case["sequences"]):
        n = 1 if s < single else rng.randint(case["new_min"], case["new_max"])
        new.append(n)
        lengths.append(n + rng.randint(case["keys_min"], case["keys_max"]))
    order = list(range(case["sequences"]))
    rng.shuffle(order)
    return [new[i] for i in order], [lengths[i] for i in order]


def _held(case):
    """Tokens that each sequence of a pages case holds; of 16 in a row, one holds nothing."""
    rng = random.Random(case["mix"])
    return [0 if s % 16 == 15 else rng.randint(1, case["keys_max"]) for s in range(case["sequences"])]


def _pool_pages(case):
    used = sum(-(-n // case["page_size"]) for n in _held(case))
    if case["op"] == "compact":
        return max(used + 1, used * 16 // case["part"])
    return used + used // 4 + 2 * case["sequences"]


def _fork_lists(case):
    """(freed sequences, parents, children): the freed ones and the empty ones become children of sequences that stay."""
    rng = random.Random(case["mix"] + 1)
    held = _held(case)
    alive = [s for s, n in enumerate(held) if n > 0]
    count = max(1, min(len(alive) - 1, case["sequences"] * case["part"] // 16))
    freed = rng.sample(alive, count)
    gone = set(freed)
    stay = [s for s in alive if s not in gone]
    parents = [rng.choice(stay) for _ in freed]
    return freed, parents, list(freed)


# ------------------------------------------------------------------ inputs
def _frequencies(rotary_dim, scaling):
    """(angles per position of the pairs, magnitude), 64-bit: theta^(-2 i / R), scaled for contexts beyond the trained one."""
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    theta, factor, original = _THETA, 8.0, 8192
    if scaling == "base":
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    f = theta ** (-2.0 * i / rotary_dim)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "wavelength":                      # by how often a pair turns within the trained context
        turns = original * f / (2.0 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0.0, 1.0)
        return f * (keep + (1.0 - keep) / factor), 1.0
    if scaling == "yarn":                            # by the pair's index
        def pair(turns):
            return rotary_dim * math.log(original / (turns * 2.0 * math.pi)) / (2.0 * math.log(theta))
        low, high = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), rotary_dim - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        return f * ((1.0 - ramp) + ramp / factor), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _table(rotary_dim, scaling):
    from vibe_compiler_b200.paged_cache import RotaryTable
    if scaling == "none":
        return RotaryTable(rotary_dim, theta=_THETA)
    return RotaryTable(rotary_dim, theta=_THETA, scaling=scaling, factor=8.0, original_length=8192)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


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
    op, device = case["op"], torch.device("cuda", torch.cuda.current_device())
    g = _generator(seed)
    state = {"case": case}
    if op == "rope":
        rows = torch.randn(case["tokens"], case["heads"] + 2, case["head_dim"], generator=g, device=device, dtype=torch.float32).to(_DTYPES[case["dtype"]])
        state["x"] = rows[:, :case["heads"]]         # the rotated heads of wider rows
        state["positions"] = torch.randint(0, case["longest"], (case["tokens"],), generator=g, device=device)
        _with_table(state, case["rotary_dim"], case["scaling"])
        return state
    if op in ("append", "attention"):
        new, lengths = _lengths(case)
        size, dtype = case["page_size"], _DTYPES[case["dtype"]]
        counts = [-(-n // size) for n in lengths]
        pages = sum(counts) + 7
        tokens = sum(new)
        state["new"], state["lengths"] = new, lengths
        state["k"] = torch.randn(pages, size, case["kv_heads"], case["head_dim"], generator=g, device=device, dtype=dtype)
        state["v"] = torch.randn(pages, size, case["kv_heads"], case["head_dim"], generator=g, device=device, dtype=dtype)
        _with_caches(state, [(state["k"], state["v"])])
        state["page_table"] = _place(lengths, size, pages, max(counts) + 3, seed).to(device)
        state["key_lengths"] = torch.tensor(lengths, dtype=torch.int32, device=device)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        state["starts"] = starts
        state["query_starts"] = torch.tensor(starts, dtype=torch.int32, device=device)
        if op == "append":
            state["qkv"] = torch.randn(tokens, (case["q_heads"] + 2 * case["kv_heads"]) * case["head_dim"], generator=g, device=device, dtype=dtype)
            _with_table(state, case["head_dim"], case["scaling"])
        else:
            state["q"] = torch.randn(tokens, case["q_heads"], case["head_dim"], generator=g, device=device, dtype=dtype)
        return state
    held, pages, size = _held(case), _pool_pages(case), case["page_size"]
    width = -(-(case["keys_max"] + 2 * size) // size) + 2
    table = _place(held, size, pages, width, seed)
    refs = torch.zeros(pages, dtype=torch.int32)
    refs[table[table >= 0].long()] = 1
    state["table"], state["refs"] = table.to(device), refs.to(device)
    state["held"] = torch.tensor(held, dtype=torch.int32, device=device)
    if op == "reserve":
        state["wanted"] = state["held"] + 1
    if op == "fork":
        for name, values in zip(("freed", "parents", "children"), _fork_lists(case)):
            state[name] = torch.tensor(values, dtype=torch.int32, device=device)
    if op != "reserve":
        shape = (pages, size, case["kv_heads"], case["head_dim"])
        state["caches"] = [(torch.randn(shape, generator=g, device=device, dtype=_DTYPES[case["dtype"]]),
                            torch.randn(shape, generator=g, device=device, dtype=_DTYPES[case["dtype"]])) for _ in range(case["layers"])]
        _with_caches(state, state["caches"])
    return state


def _with_caches(state, pairs):
    """The caches' handles, which a program keeps as long as the caches."""
    if own:
        from vibe_compiler_b200.paged_cache import PagedCache
        state["handles"] = [PagedCache(k, v) for k, v in pairs]


def _with_table(state, rotary_dim, scaling):
    """The rotation's constants, which a program makes once."""
    if own:
        state["rotary"] = _table(rotary_dim, scaling)
    else:
        f, state["magnitude"] = _frequencies(rotary_dim, scaling)
        state["frequencies"] = f.cuda()


# ------------------------------------------------------------------ a pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    case, backend = state["case"], _backend()
    op = case["op"]
    if op == "rope":
        return backend.rope(state["x"], state["positions"], state["rotary"], interleaved=case["interleaved"], backward=case["backward"])
    if op in ("append", "attention"):
        from vibe_compiler_b200.paged_cache import PagedBatch
        cache = state["handles"][0]
        batch = PagedBatch(state["page_table"], state["key_lengths"], state["query_starts"], max_query=max(state["new"]))
        if op == "append":
            q = backend.rope_append(state["qkv"], cache, batch, state["rotary"], q_heads=case["q_heads"], interleaved=case["interleaved"])
            return q, state["k"], state["v"]
        lse = torch.empty(state["q"].shape[:2], dtype=torch.float32, device=state["q"].device)
        out = backend.attention_paged(state["q"], cache, batch, case["head_dim"] ** -0.5, causal=True, lse=lse)
        return out, lse
    size = case["page_size"]
    if op == "reserve":
        return backend.pages_reserve(state["table"], state["held"], state["refs"], state["wanted"], size)
    caches = state["handles"]
    if op == "fork":
        table, held, refs = backend.pages_free(state["table"], state["held"], state["refs"], state["freed"], size)
        table, held, refs, sources, destinations, result = backend.pages_fork(table, held, refs, state["parents"], state["children"], size)
        backend.pages_copy(caches, sources, destinations)
        return table, held, refs, result, state["caches"]
    table, refs, sources, destinations = backend.pages_compact(state["table"], state["held"], state["refs"], size)
    backend.pages_copy(caches, sources, destinations)
    return table, refs, state["caches"]


def _rotated(x, angles, magnitude, interleaved, backward):
    """x [tokens, heads, head_dim] in 32 bits, angles [tokens, pairs] in 64."""
    cos, sin = (magnitude * angles.cos()).float()[:, None], (magnitude * angles.sin()).float()[:, None]
    if backward:
        sin = -sin
    x = x.float()
    pairs = angles.shape[1]
    head, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = head[..., :pairs], head[..., pairs:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, rest), dim=-1)


def _slots(state):
    """(position of every new token, its page, its row in the page)."""
    case, device = state["case"], state["page_table"].device
    counts = state["query_starts"][1:] - state["query_starts"][:-1]
    sequence = torch.repeat_interleave(torch.arange(case["sequences"], device=device), counts.long(), output_size=state["starts"][-1])
    tokens = torch.arange(state["starts"][-1], device=device)
    position = tokens - state["query_starts"].long()[sequence] + (state["key_lengths"] - counts).long()[sequence]
    page = state["page_table"][sequence, position // case["page_size"]].long()
    return position, page, position % case["page_size"]


def _run_plain(state):
    case = state["case"]
    op = case["op"]
    if op == "rope":
        angles = state["positions"].double()[:, None] * state["frequencies"]
        return _rotated(state["x"], angles, state["magnitude"], case["interleaved"], case["backward"]).to(state["x"].dtype)
    if op == "append":
        hq, hk, d = case["q_heads"], case["kv_heads"], case["head_dim"]
        position, page, row = _slots(state)
        rows = state["qkv"].view(-1, hq + 2 * hk, d)
        angles = position.double()[:, None] * state["frequencies"]
        qk = _rotated(rows[:, :hq + hk], angles, state["magnitude"], case["interleaved"], False).to(rows.dtype)
        state["k"][page, row] = qk[:, hq:]
        state["v"][page, row] = rows[:, hq + hk:]
        return qk[:, :hq].contiguous(), state["k"], state["v"]
    if op == "attention":
        return _attention_in(state, torch.float32)
    return _pages_plain(state)


def _attention_in(state, dtype):
    case = state["case"]
    hq, hk, d, size = case["q_heads"], case["kv_heads"], case["head_dim"], case["page_size"]
    group, scale = hq // hk, case["head_dim"] ** -0.5
    q_all = state["q"]
    out = torch.empty_like(q_all) if dtype == torch.float32 else torch.empty(q_all.shape, dtype=dtype, device=q_all.device)
    lse = torch.empty(q_all.shape[:2], dtype=dtype, device=q_all.device)
    for s, (n, length) in enumerate(zip(state["new"], state["lengths"])):
        pages = state["page_table"][s, :-(-length // size)].long()
        k = state["k"][pages].reshape(-1, hk, d)[:length].to(dtype).permute(1, 2, 0)       # [hk, d, keys]
        v = state["v"][pages].reshape(-1, hk, d)[:length].to(dtype).transpose(0, 1)        # [hk, keys, d]
        step = max(1, (1 << 27) // (hq * length))
        for first in range(0, n, step):
            count = min(step, n - first)
            at = state["starts"][s] + first
            q = q_all[at:at + count].to(dtype).view(count, hk, group, d).permute(1, 2, 0, 3).reshape(hk, group * count, d)
            scores = torch.matmul(q, k).mul_(scale).view(hk, group, count, length)
            last = torch.arange(first, first + count, device=k.device) + (length - n)
            if length - n + first + 1 < length:
                scores.masked_fill_(torch.arange(length, device=k.device)[None, :] > last[:, None], -math.inf)
            top = scores.amax(-1, keepdim=True)
            p = scores.sub_(top).exp_()
            total = p.sum(-1, keepdim=True)
            o = torch.matmul(p.view(hk, group * count, length), v).view(hk, group, count, d) / total
            out[at:at + count] = o.permute(2, 0, 1, 3).reshape(count, hq, d).to(out.dtype)
            lse[at:at + count] = (top + total.log()).permute(2, 0, 1, 3).reshape(count, hq)
    return out, lse


def _free_pages(refs):
    return torch.nonzero(refs == 0).flatten().to(torch.int32)


def _reserved(table, held, refs, wanted, size):
    have, need = (held + size - 1) // size, (torch.maximum(held, wanted) + size - 1) // size
    extra = need - have
    free = _free_pages(refs)
    missing = (extra.sum() - free.numel()).clamp(min=0)
    if int(missing) > 0:
        return table.clone(), held.clone(), refs.clone(), missing.to(torch.int32).view(1)
    slot = torch.arange(table.shape[1], device=table.device)[None, :]
    fresh = (slot >= have[:, None]) & (slot < need[:, None])
    index = (torch.cumsum(extra, 0) - extra)[:, None] + slot - have[:, None]
    new = free[index.clamp(0, max(free.numel() - 1, 0)).long()]
    table = torch.where(fresh, new, table)
    refs = refs.clone()
    refs[table[fresh].long()] = 1
    return table, torch.maximum(held, wanted), refs, missing.to(torch.int32).view(1)


def _freed(table, held, refs, sequences, size):
    rows = sequences.long()
    listed_pages = table[rows]
    used = torch.arange(table.shape[1], device=table.device)[None, :] < ((held[rows] + size - 1) // size)[:, None]
    pages = listed_pages[used].long()
    refs = refs.index_add(0, pages, torch.full_like(pages, -1, dtype=torch.int32))
    table, held = table.clone(), held.clone()
    table[rows] = -1
    held[rows] = 0
    return table, held, refs


def _forked(table, held, refs, parents, children, size):
    p, c = parents.long(), children.long()
    full, partial = held[p] // size, held[p] % size != 0
    free = _free_pages(refs)
    take = torch.cumsum(partial.int(), 0) - partial.int()
    fresh = torch.where(partial, free[take.long().clamp(max=free.numel() - 1)], torch.full_like(parents, -1))
    slot = torch.arange(table.shape[1], device=table.device)[None, :]
    rows = table[p]
    sources = torch.where(partial, rows.gather(1, full.long().clamp(max=table.shape[1] - 1)[:, None]).flatten(), torch.full_like(parents, -1))
    shared = slot < full[:, None]
    new_rows = torch.where(shared, rows, torch.full_like(rows, -1))
    new_rows = torch.where((slot == full[:, None]) & partial[:, None], fresh[:, None], new_rows)
    pages = rows[shared].long()
    refs = refs.index_add(0, pages, torch.ones_like(pages, dtype=torch.int32))
    refs[fresh[partial].long()] = 1
    table, held = table.clone(), held.clone()
    table[c], held[c] = new_rows, held[p]
    return table, held, refs, sources, fresh


def _compacted(table, held, refs, size):
    live = int((refs > 0).sum())
    index = torch.arange(refs.numel(), device=refs.device)
    sources = index[(refs > 0) & (index >= live)]
    destinations = index[(refs == 0) & (index < live)]
    place = index.clone()
    place[sources] = destinations
    used = torch.arange(table.shape[1], device=table.device)[None, :] < ((held + size - 1) // size)[:, None]
    table = torch.where(used, place[table.clamp(min=0).long()].to(torch.int32), table)
    refs = refs.clone()
    refs[destinations] = refs[sources]
    refs[sources] = 0
    return table, refs, sources, destinations


def _pages_plain(state):
    case, size = state["case"], state["case"]["page_size"]
    if case["op"] == "reserve":
        return _reserved(state["table"], state["held"], state["refs"], state["wanted"], size)
    if case["op"] == "fork":
        table, held, refs = _freed(state["table"], state["held"], state["refs"], state["freed"], size)
        table, held, refs, sources, destinations = _forked(table, held, refs, state["parents"], state["children"], size)
        wanted = sources >= 0
        sources, destinations = sources[wanted].long(), destinations[wanted].long()
        for k, v in state["caches"]:
            k[destinations] = k[sources]
            v[destinations] = v[sources]
        return table, held, refs, torch.zeros(1, dtype=torch.int32, device=table.device), state["caches"]
    table, refs, sources, destinations = _compacted(state["table"], state["held"], state["refs"], size)
    for k, v in state["caches"]:
        k[destinations] = k[sources]
        v[destinations] = v[sources]
    return table, refs, state["caches"]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    width = 4 if case["dtype"] == "f32" else 2
    if op == "rope":
        elements = case["tokens"] * case["heads"] * case["head_dim"]
        return {"bytes": 2 * elements * width + 8 * case["tokens"], "flops": 3 * case["tokens"] * case["heads"] * case["rotary_dim"]}
    if op == "append":
        new, _ = _lengths(case)
        tokens, d = sum(new), case["head_dim"]
        rows = tokens * (case["q_heads"] + 2 * case["kv_heads"]) * d
        return {"bytes": 2 * rows * width, "flops": 3 * tokens * (case["q_heads"] + case["kv_heads"]) * d}
    if op == "attention":
        new, lengths = _lengths(case)
        d, hq, hk = case["head_dim"], case["q_heads"], case["kv_heads"]
        pairs = sum(n * (length - n) + n * (n + 1) // 2 for n, length in zip(new, lengths))
        return {"bytes": (2 * sum(lengths) * hk * d + 2 * sum(new) * hq * d) * width + 4 * sum(new) * hq, "flops": 4 * d * hq * pairs}
    held, pages, size = _held(case), _pool_pages(case), case["page_size"]
    used = sum(-(-n // size) for n in held)
    numbers = 4 * (2 * pages + 2 * used + 2 * len(held))       # reference counts, table entries in use and lengths, in and out
    page_bytes = 2 * 2 * size * case["kv_heads"] * case["head_dim"] * width * case["layers"]   # K and V, read and written
    if op == "reserve":
        return {"bytes": numbers, "flops": 0}
    if op == "fork":
        _, parents, _ = _fork_lists(case)
        moved = sum(1 for p in parents if held[p] % size)
        return {"bytes": 2 * numbers + moved * page_bytes, "flops": 0}
    return {"bytes": numbers + max(1, used * (pages - used) // pages) * page_bytes, "flops": 0}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    op = case["op"]
    if op in ("reserve", "fork", "compact"):
        return None                                   # whole numbers and copies
    state = prepare(case, seed)
    if op == "attention":
        return _exact_attention(state)
    if op == "rope":
        return _exact_rotation(state["x"], state["positions"], case["rotary_dim"], case)
    hq, hk = case["q_heads"], case["kv_heads"]
    rows = state["qkv"].view(-1, hq + 2 * hk, case["head_dim"])
    k, v = state["k"].double(), state["v"].double()
    positions = torch.empty(rows.shape[0], dtype=torch.int64)
    pages, offsets = torch.empty_like(positions), torch.empty_like(positions)
    table = state["page_table"].cpu()
    for s, (n, length) in enumerate(zip(state["new"], state["lengths"])):
        at = torch.arange(length - n, length)
        positions[state["starts"][s]:state["starts"][s + 1]] = at
        pages[state["starts"][s]:state["starts"][s + 1]] = table[s][at // case["page_size"]].long()
        offsets[state["starts"][s]:state["starts"][s + 1]] = at % case["page_size"]
    turned = _exact_rotation(rows[:, :hq + hk], positions.to(rows.device), case["head_dim"], dict(case, backward=False))
    k[pages, offsets] = turned[:, hq:]
    v[pages, offsets] = rows[:, hq + hk:].double()
    return turned[:, :hq], k, v


def _exact_rotation(x, positions, rotary_dim, case):
    """Pairs as complex numbers times magnitude * exp(+-i position f)."""
    f, magnitude = _frequencies(rotary_dim, case["scaling"])
    angle = positions.double()[:, None, None] * f.to(x.device)
    turn = torch.polar(torch.full_like(angle, magnitude), -angle if case["backward"] else angle)
    y = x.double().clone()
    half = rotary_dim // 2
    first, second = (slice(0, rotary_dim, 2), slice(1, rotary_dim, 2)) if case["interleaved"] else (slice(0, half), slice(half, rotary_dim))
    z = torch.complex(x[..., first].double(), x[..., second].double()) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_attention(state):
    """Head by head, over the keys that a row sees, with the log-sum-exp first."""
    case = state["case"]
    hq, hk, d, size = case["q_heads"], case["kv_heads"], case["head_dim"], case["page_size"]
    q = state["q"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    for s, (n, length) in enumerate(zip(state["new"], state["lengths"])):
        keys = torch.arange(length, device=q.device)
        pages, rows = state["page_table"][s].long()[keys // size], keys % size
        tokens = torch.arange(n, device=q.device)
        for head in range(hk):
            k, v = state["k"][pages, rows, head].double(), state["v"][pages, rows, head].double()
            for first in range(0, n, 1024):
                part = slice(first, min(first + 1024, n))
                hidden = keys[None, :] > (length - n + tokens[part])[:, None]
                for h in range(head * (hq // hk), (head + 1) * (hq // hk)):
                    at = slice(state["starts"][s] + part.start, state["starts"][s] + part.stop)
                    scores = (q[at, h].double() @ k.T) / math.sqrt(d)
                    scores[hidden] = -math.inf
                    lse[at, h] = torch.logsumexp(scores, -1)
                    out[at, h] = (scores - lse[at, h][:, None]).exp() @ v
    return out, lse
