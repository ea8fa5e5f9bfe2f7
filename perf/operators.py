"""The attention step's operators over a 4-bit cache: what is timed, in a plain form and through the package's plans.

Four operators that sit between the quantized qkv projection and the quantized output projection of a decoder layer:

* ``norm_rope``  RMS norm of every query and key head and the rotation by position (one or several axes), one pass;
* ``append``     the same pass with the keys and values going straight into the 4-bit paged cache;
* ``read``       the cache's tokens back as bf16 keys and values;
* ``attention``  attention of ragged query rows over the cache: single tokens, a few drafted tokens, whole prompts.

The cache.  A page holds ``page`` tokens (a multiple of 16) of every kv head: ``[heads_kv][page / 16]`` tiles of 18 * dim
bytes.  Each group of 64 channels of a token and head is held as codes c = 0..15 with a half-precision scale s and minimum
m, the value being s * c + m.  A tile is, in this order, with t the token (0..15) and d the channel:

* keys' codes, 8 * dim bytes: for d = 64 g + 16 c + 8 u + 2 b + n the nibble n (0 low) of byte
  ``(((h * 16 + t) * 4 + c) * w + g % w) * 8 + 4 * u + b`` with w = min(2, dim / 64) and h = g // w;
* values' codes, 8 * dim bytes: for d = 64 h + 16 j + 8 n + r and t = 8 e + 2 c + o the nibble n of byte
  ``h * 512 + (r * 4 + c) * 16 + 4 * j + 2 * o + e``;
* keys' (s, m) pairs [16][dim / 64], then values' pairs.
"""
import math
import random

import torch

own = False

GROUP = 64
F16_MAX = 65504.0
EPS = 1e-6


# ------------------------------------------------------------------------------------------------ cases
def _attention(name, batch, q_len, kv_len, heads_q, heads_kv, dim, page, ragged, window=0):
    return {"name": name, "op": "attention", "batch": batch, "q_len": q_len, "kv_len": kv_len, "heads_q": heads_q,
            "heads_kv": heads_kv, "dim": dim, "page": page, "ragged": ragged, "window": window}


def _tokens(name, op, tokens, heads_q, heads_kv, dim, page=0, axes=1, rot=0, interleaved=False):
    return {"name": name, "op": op, "tokens": tokens, "heads_q": heads_q, "heads_kv": heads_kv, "dim": dim, "page": page,
            "axes": axes, "rot": rot or dim, "interleaved": interleaved}


def listed():
    return [
        # one user, a short conversation: nothing but latency (the 8B-class layer whose qkv projection has 6144 columns)
        _attention("decode_one", 1, 1, 129, 32, 8, 128, 16, False),
        # a serving batch of that layer, every sequence of another length
        _attention("decode_batch", 64, 1, 4001, 32, 8, 128, 64, True),
        # two users with books in their context, on the 70B-class layer (8192 hidden, 64 heads)
        _attention("decode_long", 2, 1, 131071, 64, 8, 128, 64, False),
        # five drafted tokens checked at once
        _attention("verify", 16, 5, 6001, 40, 8, 128, 32, True),
        # a prompt
        _attention("prefill", 1, 4096, 4096, 32, 8, 128, 64, False),
        # chunks of three prompts over what is cached of them, wide heads, a sliding window
        _attention("prefill_chunks", 3, 2049, 9001, 16, 2, 256, 16, True, 4096),
        # one token's keys and values into the cache; and a long prompt's
        _tokens("append_one", "append", 1, 32, 8, 128, page=16),
        _tokens("append_prompt", "append", 8191, 64, 8, 128, page=64),
        # drafted tokens, narrow heads, half of the channels rotated in neighbouring pairs
        _tokens("norm_rope_few", "norm_rope", 5, 40, 8, 64, rot=32, interleaved=True),
        # images and video among text: time, height and width
        _tokens("norm_rope_image", "norm_rope", 4097, 28, 4, 128, axes=3),
        # a page's worth of a prefix, and a long one, handed on in bf16
        _tokens("read_few", "read", 100, 0, 8, 128, page=16),
        _tokens("read_prefix", "read", 65537, 0, 8, 128, page=64),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "append", "norm_rope", "read"])
    heads_q, heads_kv = rng.choice([(32, 8), (64, 8), (40, 8), (28, 4), (16, 2), (8, 1), (16, 16), (20, 4)])
    dim = rng.choice([64, 128, 128, 256])
    page = rng.choice([16, 32, 64, 128])
    if op == "attention":
        kind = rng.choice(["decode", "decode", "verify", "prefill"])
        ragged = rng.random() < 0.7
        window = rng.choice([0, 0, 0, 100, 1024])
        if kind == "prefill":
            batch = rng.choice([1, 1, 2, 4])
            cells = (1 << 37) // (4 * heads_q * dim * batch)  # of the scores, for one sequence
            q_len = _spread(rng, 33, int(cells**0.5))
            kv_len = q_len + rng.choice([0, 0, _spread(rng, 1, max(1, min(8000, cells // q_len - q_len)))])
        else:
            q_len = 1 if kind == "decode" else rng.randint(2, 8)
            batch = _spread(rng, 1, 128)
            kv_len = _spread(rng, q_len, min(65536, (1 << 21) // (batch * heads_kv * dim // 64)))
        case = _attention("", batch, q_len, kv_len, heads_q, heads_kv, dim, page, ragged, window)
    else:
        limit = {"append": 8191 * 64 * 128 // (heads_q * dim), "norm_rope": 8191 * 64 * 128 // (heads_q * dim),
                 "read": 65537 * 1024 // (heads_kv * dim)}[op]
        tokens = _spread(rng, 1, min(limit, 65537))
        axes, interleaved = rng.choice([1, 1, 2, 3]), rng.random() < 0.3
        rot = rng.choice([dim, dim, dim // 2])
        case = _tokens("", op, tokens, 0 if op == "read" else heads_q, heads_kv, dim, 0 if op == "norm_rope" else page,
                       axes, rot, interleaved)
    del case["name"]
    return case


def _lengths(case):
    """(query rows, cached tokens) of each sequence; the cached ones include the queries' own."""
    rng = random.Random("%(batch)d %(q_len)d %(kv_len)d" % case)
    got = []
    for i in range(case["batch"]):
        n, length = case["q_len"], case["kv_len"]
        if case["ragged"] and i:  # the first sequence has the full lengths
            n = n if n <= 8 else rng.randint(1, n)
            length = max(n, int(length * rng.uniform(0.1, 1.0)))
        got.append((n, length))
    return got


def work(case):
    d, kv = case["dim"], case["heads_kv"]
    token = kv * (d + d // GROUP * 8)  # bytes of one token's keys and values in the cache
    if case["op"] == "attention":
        rows = cells = cached = 0
        for n, length in _lengths(case):
            first = length - n  # keys before the first query row
            if case["window"]:
                w = case["window"]
                cells += sum(min(first + i + 1, w) for i in range(n))
                cached += min(length, w + n - 1)
            else:
                cells += n * first + n * (n + 1) // 2
                cached += length
            rows += n
        return {"bytes": cached * token + 2 * rows * case["heads_q"] * d * 2, "flops": 4 * cells * case["heads_q"] * d}
    t = case["tokens"]
    if case["op"] == "read":
        return {"bytes": t * (token + 2 * kv * d * 2), "flops": 2 * t * 2 * kv * d}
    table = t * (case["rot"] * 4 + 4 * case["axes"])
    if case["op"] == "append":  # q, k and v read, q and the cache written
        return {"bytes": t * ((2 * case["heads_q"] + 2 * kv) * d * 2 + token) + table, "flops": 12 * t * (case["heads_q"] + 2 * kv) * d}
    return {"bytes": t * 2 * (case["heads_q"] + kv) * d * 2 + table, "flops": 10 * t * (case["heads_q"] + kv) * d}


# ------------------------------------------------------------------------------------------------ the cache's form
def _quantize(x):
    """x [..., dim] in bf16 -> (codes, s, m): each step one rounding in 32 bits, s and m rounded to half precision."""
    x = x.float().unflatten(-1, (-1, GROUP))
    low, high = x.amin(-1), x.amax(-1)
    s = ((high - low) / 15.0).clamp(max=F16_MAX).half()
    m = low.clamp(-F16_MAX, F16_MAX).half()
    step = torch.where(s > 0, s.float(), torch.full_like(low, math.inf))  # a group of one value has codes 0
    codes = torch.round((x - m.float().unsqueeze(-1)) / step.unsqueeze(-1)).clamp(0, 15)
    return codes.flatten(-2), s, m


def _values(codes, s, m):
    return (codes.unflatten(-1, (-1, GROUP)) * s.float().unsqueeze(-1) + m.float().unsqueeze(-1)).flatten(-2)


def _tiles(kv, dead):
    """Tiles' bytes [..., 18 * dim] from keys and values [..., 16, dim] in bf16; tokens in `dead` get NaN scales."""
    parts, pairs = [], []
    for which, x in enumerate(kv):
        codes, s, m = _quantize(x)
        codes, d, lead = codes.to(torch.uint8), x.shape[-1], x.shape[:-2]
        w = min(2, d // GROUP)
        if which == 0:  # [t, h, gw, c, u, b, n] -> [h, t, c, gw, u, b]
            v = codes.reshape(*lead, 16, d // GROUP // w, w, 4, 2, 4, 2)
            v = v[..., 0] | (v[..., 1] << 4)
            k = len(lead)
            v = v.permute(*range(k), k + 1, k, k + 3, k + 2, k + 4, k + 5)
        else:  # [e, c, o, h, j, n, r] -> [h, r, c, j, o, e]
            v = codes.reshape(*lead, 2, 4, 2, d // 64, 4, 2, 8)
            v = v[..., 0, :] | (v[..., 1, :] << 4)
            k = len(lead)
            v = v.permute(*range(k), k + 3, k + 5, k + 1, k + 4, k + 2, k)
        parts.append(v.reshape(*lead, 8 * d))
        pair = torch.stack([s, m], -1)
        pair[dead] = float("nan")
        pairs.append(pair.reshape(*lead, -1).view(torch.uint8))
    return torch.cat(parts + pairs, -1)


def _untile(tiles, dim):
    """Keys and values [..., 16, dim] in 32 bits from tiles' bytes [..., 18 * dim]."""
    lead, k, w = tiles.shape[:-1], tiles.dim() - 1, min(2, dim // GROUP)
    keys, vals, pairs = tiles[..., : 8 * dim], tiles[..., 8 * dim : 16 * dim], tiles[..., 16 * dim :]
    nib = lambda v: torch.stack([v & 15, v >> 4], -1)  # noqa: E731
    keys = nib(keys.reshape(*lead, dim // GROUP // w, 16, 4, w, 2, 4)).permute(*range(k), k + 1, k, k + 3, k + 2, k + 4, k + 5, k + 6)
    vals = nib(vals.reshape(*lead, dim // 64, 8, 4, 4, 2, 2)).permute(*range(k), k + 5, k + 2, k + 4, k, k + 3, k + 6, k + 1)
    pairs = pairs.contiguous().view(torch.float16).reshape(*lead, 2, 16, dim // GROUP, 2)
    keys = _values(keys.reshape(*lead, 16, dim).float(), pairs[..., 0, :, :, 0], pairs[..., 0, :, :, 1])
    vals = _values(vals.reshape(*lead, 16, dim).float(), pairs[..., 1, :, :, 0], pairs[..., 1, :, :, 1])
    return keys, vals


# ------------------------------------------------------------------------------------------------ inputs
def _cache(case, lengths, gen):
    """A cache that holds sequences of these lengths on pages in no order, NaN in every place that no token has, and its page table."""
    page, d, kv = case["page"], case["dim"], case["heads_kv"]
    longest = max(max(lengths), 1)
    pages = [-(-n // page) for n in lengths]
    total, width = sum(pages) + 3, -(-longest // page)
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    cache = torch.full((total, kv, page // 16, 18 * d), 255, dtype=torch.uint8, device="cuda")
    table = torch.full((len(lengths), width), -1, dtype=torch.int32, device="cuda")
    # channels of their own size and offset, as keys have them after training; the first token draws attention and says little
    gain = 0.6 + torch.rand(kv, d, generator=gen, device="cuda")
    bias = 1.5 * torch.randn(kv, d, generator=gen, device="cuda") * (torch.rand(kv, d, generator=gen, device="cuda") < 0.1)
    at = 0
    for i, n in enumerate(lengths):
        if not n:
            continue
        tiles = -(-n // 16)
        k = torch.randn(tiles, kv, 16, d, generator=gen, device="cuda") * gain.unsqueeze(1) + bias.unsqueeze(1)
        v = torch.randn(tiles, kv, 16, d, generator=gen, device="cuda")
        k[0, :, 0] *= 1.5
        v[0, :, 0] *= 0.05
        dead = (torch.arange(tiles * 16, device="cuda") >= n).reshape(tiles, 1, 16).expand(tiles, kv, 16)
        made = _tiles((k.bfloat16(), v.bfloat16()), dead)
        table[i, : pages[i]] = order[at : at + pages[i]]
        at += pages[i]
        of = torch.arange(tiles, device="cuda")
        cache[table[i, of // (page // 16)].long(), :, of % (page // 16)] = made
    return cache.reshape(total, -1), table


def _axis_of_pair(case):
    """Which axis turns each pair of channels: a quarter of them by time and the rest by height and width, say."""
    pairs, axes = case["rot"] // 2, case["axes"]
    first = pairs if axes == 1 else pairs // 4
    return [0] * first + [1 + i * (axes - 1) // (pairs - first) for i in range(pairs - first)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    d, kv = case["dim"], case["heads_kv"]
    state = {"case": dict(case)}
    if case["op"] == "attention":
        lens = _lengths(case)
        state["cache"], state["page_table"] = _cache(case, [n for _, n in lens], gen)
        rows = sum(n for n, _ in lens)
        state["q"] = torch.randn(rows, case["heads_q"] * d, generator=gen, device="cuda").mul_(1.5).bfloat16()
        state["cu_q"] = torch.tensor([sum(n for n, _ in lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")
        state["kv_lens"] = torch.tensor([n for _, n in lens], dtype=torch.int32, device="cuda")
        state["out"] = torch.empty_like(state["q"])
        return state
    t = case["tokens"]
    if case["page"]:
        spare = case["page"] // 2 + 1 if case["op"] == "append" else 0  # what the sequence has already
        cache, table = _cache(case, [t + spare], gen)
        of = torch.arange(spare, t + spare, device="cuda")
        state["cache"] = cache
        state["slots"] = table[0, of // case["page"]].long() * case["page"] + of % case["page"]
        state["k_read"] = torch.empty(t, kv * d, dtype=torch.bfloat16, device="cuda")
        state["v_read"] = torch.empty(t, kv * d, dtype=torch.bfloat16, device="cuda")
    if case["op"] == "read":
        return state
    hq, rot = case["heads_q"], case["rot"]
    # the qkv projection's output: channels of their own size
    gain = torch.exp(0.5 * torch.randn((hq + 2 * kv) * d, generator=gen, device="cuda"))
    state["qkv"] = (torch.randn(t, (hq + 2 * kv) * d, generator=gen, device="cuda") * gain).bfloat16()
    state["q_weight"] = 1.0 + 0.3 * torch.randn(d, generator=gen, device="cuda")
    state["k_weight"] = 1.0 + 0.3 * torch.randn(d, generator=gen, device="cuda")
    longest = 16384
    angle = torch.arange(longest, device="cuda").double().unsqueeze(1) * 500000.0 ** (-torch.arange(rot // 2, device="cuda").double() / (rot // 2))
    state["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).float()
    start = torch.randint(0, longest // 2, (1,), generator=gen, device="cuda")
    line = start + torch.arange(t, device="cuda")
    places = [line, start + line // 40 % 97, start + line % 40][: case["axes"]]
    state["positions"] = (torch.stack(places) % longest).to(torch.int32)
    state["q_out"] = torch.empty(t, hq * d, dtype=torch.bfloat16, device="cuda")
    if case["op"] == "norm_rope":
        state["k_out"] = torch.empty(t, kv * d, dtype=torch.bfloat16, device="cuda")
    return state


# ------------------------------------------------------------------------------------------------ plain forms
def _norm_rope_plain(x, weight, state):
    """x [T, heads * dim] in bf16, normed and turned, in bf16.  The mean square is summed in 64 bits and rounded once, so that
    keys that lie next to a border of two codes fall on the same side whatever the order of the sum."""
    case = state["case"]
    d, rot = case["dim"], case["rot"]
    x = x.unflatten(-1, (-1, d))
    mean = (x.double().square().sum(-1, keepdim=True) / d).float()
    y = x.float() * (1.0 / torch.sqrt(mean + EPS)) * weight
    axis = torch.tensor(_axis_of_pair(case), device=x.device)
    where = state["positions"].long()[axis].T  # [T, pairs]
    pair = torch.arange(rot // 2, device=x.device)
    c, s = state["cos_sin"][where, pair].unsqueeze(1), state["cos_sin"][where, pair + rot // 2].unsqueeze(1)
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if case["interleaved"] else (y[..., : rot // 2], y[..., rot // 2 : rot])
    turned = torch.stack([a * c - b * s, b * c + a * s], -1 if case["interleaved"] else -2)
    return torch.cat([turned.flatten(-2), y[..., rot:]], -1).bfloat16()


def _attention_plain(state):
    case = state["case"]
    d, kv, page = case["dim"], case["heads_kv"], case["page"]
    batch, width = state["page_table"].shape
    most = case["q_len"]
    pages = state["cache"][state["page_table"].clamp(min=0).long()].reshape(batch, width, kv, page // 16, 18 * d)
    keys, vals = _untile(pages.transpose(2, 3), d)  # [batch, width, page / 16, kv, 16, d]
    keys, vals = (x.movedim(3, 1).reshape(batch, kv, width * page, d) for x in (keys, vals))
    live = torch.arange(width * page, device="cuda") < state["kv_lens"].unsqueeze(1)  # [batch, keys]
    keys, vals = (torch.where(live[:, None, :, None], x, torch.zeros_like(x)) for x in (keys, vals))
    n = state["cu_q"][1:] - state["cu_q"][:-1]
    row = torch.arange(most, device="cuda")
    there = row < n.unsqueeze(1)  # [batch, rows]
    at = (state["cu_q"][:-1].unsqueeze(1) + row).clamp(max=state["q"].shape[0] - 1).long()
    q = state["q"][at].float().unflatten(-1, (kv, -1, d)).movedim(1, 3)  # [batch, kv, group, rows, d]
    scores = (q.flatten(2, 3) @ keys.transpose(-1, -2)).unflatten(2, (-1, most)) * d**-0.5
    last = (state["kv_lens"] - n).unsqueeze(1) + row  # the last key that a row sees
    key = torch.arange(width * page, device="cuda")
    seen = (key <= last.unsqueeze(-1)) & live.unsqueeze(1)
    if case["window"]:
        seen = seen & (key > last.unsqueeze(-1) - case["window"])
    seen = seen[:, None, None]
    top = scores.masked_fill(~seen, -math.inf).amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(scores - top).masked_fill(~seen, 0.0)
    total = p.sum(-1, keepdim=True)
    out = (p.flatten(2, 3) @ vals).unflatten(2, (-1, most)) / torch.where(total > 0, total, torch.ones_like(total))
    out = out.movedim(3, 1).reshape(batch, most, -1)
    return out[there].bfloat16()


def _read_plain(state):
    case = state["case"]
    d, kv, page = case["dim"], case["heads_kv"], case["page"]
    at = state["slots"]
    tiles = state["cache"].reshape(-1, kv, page // 16, 18 * d)[at // page, :, at % page // 16]
    t = torch.arange(at.numel(), device="cuda")
    return [x[t, :, at % 16].reshape(at.numel(), kv * d).bfloat16() for x in _untile(tiles, d)]


def _columns(state):
    case = state["case"]
    a, b = case["heads_q"] * case["dim"], case["heads_kv"] * case["dim"]
    return state["qkv"][:, :a], state["qkv"][:, a : a + b], state["qkv"][:, a + b :]


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return _run_own(state, op)
    if op == "attention":
        return {"out": _attention_plain(state)}
    if op == "read":
        k, v = _read_plain(state)
        return {"k": k, "v": v}
    q, k, v = _columns(state)
    q, k = _norm_rope_plain(q, state["q_weight"], state), _norm_rope_plain(k, state["k_weight"], state)
    if op == "norm_rope":
        return {"q": q, "k": k}
    # what the cache then holds of these tokens
    k, v = (_values(*_quantize(x.unflatten(-1, (-1, state["case"]["dim"])))).flatten(-2).bfloat16() for x in (k, v))
    return {"q": q, "k": k, "v": v}


def _plan(state, op):
    """The plans, arguments and workspace that a program keeps beside its buffers, made on its first pass."""
    import baracuda_b200 as bq

    case = state["case"]
    layout = None
    if case["page"]:
        layout = bq.Kv4CacheDescriptor(state["cache"].shape[0], case["page"], case["heads_kv"], case["dim"])
    if op == "attention":
        plan = bq.Kv4AttentionPlan.select(None, bq.Kv4AttentionDescriptor(
            case["batch"], case["q_len"], case["kv_len"], case["heads_q"], layout, causal=True, window=case["window"]))
        args = bq.Kv4AttentionArgs(q=state["q"], cu_q=state["cu_q"], kv_lens=state["kv_lens"], page_table=state["page_table"],
                                   cache=state["cache"], out=state["out"])
        return plan, torch.empty(plan.workspace_size(), dtype=torch.uint8, device="cuda"), args
    read = None
    if case["page"]:
        read = (bq.Kv4ReadPlan.select(None, bq.Kv4ReadDescriptor(case["tokens"], layout)),
                bq.Kv4ReadArgs(cache=state["cache"], slots=state["slots"], k=state["k_read"], v=state["v_read"]))
    if op == "read":
        return read
    plan = bq.QkNormRopePlan.select(None, bq.QkNormRopeDescriptor(
        case["tokens"], case["heads_q"], case["heads_kv"], case["dim"], rot_dim=case["rot"], interleaved=case["interleaved"],
        axis_of_pair=tuple(_axis_of_pair(case)) if case["axes"] > 1 else None, eps=EPS, cache=layout))
    q, k, v = _columns(state)
    args = bq.QkNormRopeArgs(q=q, k=k, q_out=state["q_out"], cos_sin=state["cos_sin"], positions=state["positions"],
                             q_weight=state["q_weight"], k_weight=state["k_weight"], k_out=state.get("k_out"),
                             v=v if layout else None, cache=state.get("cache"), slots=state.get("slots"))
    by_head = {n: state[n].unflatten(-1, (-1, case["dim"])) for n in ("q_out", "k_out", "k_read") if n in state}
    return plan, args, read, by_head


def _run_own(state, op):
    kept = state.get("kept")
    if kept is None:
        kept = state["kept"] = _plan(state, op)
    if op == "attention":
        plan, workspace, args = kept
        plan.run(None, workspace, args)
        return {"out": state["out"]}
    if op == "read":
        kept[0].run(None, None, kept[1])
        return {"k": state["k_read"], "v": state["v_read"]}
    plan, args, read, by_head = kept
    plan.run(None, None, args)
    if op == "norm_rope":
        return {"q": by_head["q_out"], "k": by_head["k_out"]}
    read[0].run(None, None, read[1])  # what the cache then holds of these tokens
    return {"q": by_head["q_out"], "k": by_head["k_read"], "v": state["v_read"]}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _lookup(cache, slots, which, case):
    """[kv, tokens, dim] of keys (which 0) or values (1) at these slots, one byte looked up for each value by the format's formulas."""
    d, kv, page = case["dim"], case["heads_kv"], case["page"]
    flat = cache.reshape(cache.shape[0], kv, -1)
    of, t = slots % page // 16 * (18 * d), (slots % 16).unsqueeze(1)
    c = torch.arange(d, device=cache.device).unsqueeze(0)
    if which == 0:
        w = min(2, d // 64)
        g = c // 64
        byte = ((((g // w) * 16 + t) * 4 + c % 64 // 16) * w + g % w) * 8 + c % 16 // 8 * 4 + c % 8 // 2
        high = c % 2
    else:
        byte = 8 * d + c // 64 * 512 + (c % 8 * 4 + t % 8 // 2) * 16 + c % 64 // 16 * 4 + t % 2 * 2 + t // 8
        high = c % 16 // 8
    pair = 16 * d + which * (d // 64) * 64 + t * (d // 64) * 4 + torch.arange(d // 64, device=cache.device) * 4
    got = []
    for h in range(kv):
        rows = flat[slots // page, h]  # [tokens, bytes of a page's head]
        code = (rows.gather(1, of.unsqueeze(1) + byte) >> (4 * high).to(torch.uint8)) & 15
        four = rows.gather(1, (of.unsqueeze(1) + pair).repeat_interleave(4, 1) + torch.arange(4, device=cache.device).repeat(d // 64))
        sm = four.contiguous().view(torch.float16).double().reshape(-1, d // 64, 2).repeat_interleave(64, 1)
        got.append(code.double() * sm[..., 0] + sm[..., 1])
    return torch.stack(got)


def _norm_rope_exact(x, weight, state):
    case = state["case"]
    d, rot = case["dim"], case["rot"]
    x = x.double().reshape(x.shape[0], -1, d)
    x = x * (x.pow(2).mean(-1, keepdim=True) + EPS).pow(-0.5) * weight.double()
    z = x.clone()
    for i, axis in enumerate(_axis_of_pair(case)):
        one, two = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + rot // 2)
        turn = state["cos_sin"][state["positions"][axis].long()].double()
        c, s = turn[:, i, None], turn[:, i + rot // 2, None]
        z[..., one] = x[..., one] * c - x[..., two] * s
        z[..., two] = x[..., one] * s + x[..., two] * c
    return z


def _held_exact(x):
    """What the cache holds of x: rounded to bf16, then each group of 64 as 16 steps of a half-precision scale from a half-precision minimum."""
    x = x.to(torch.bfloat16).double()
    parts = []
    for part in x.split(64, -1):
        low, high = part.min(-1, keepdim=True)[0], part.max(-1, keepdim=True)[0]
        s = ((high - low) / 15).float().half().double()
        m = low.float().half().double()
        step = torch.where(s > 0, s, torch.ones_like(s))
        parts.append(m + s * torch.clamp(torch.round((part - m) / step), 0, 15))
    return torch.cat(parts, -1)


def exact(case, seed):
    state = prepare(case, seed)
    d, kv = case["dim"], case["heads_kv"]
    if case["op"] == "read":
        k, v = (_lookup(state["cache"], state["slots"], i, case).movedim(0, 1).reshape(case["tokens"], -1) for i in (0, 1))
        return {"k": k, "v": v}
    if case["op"] != "attention":
        q, k, v = _columns(state)
        q, k = _norm_rope_exact(q, state["q_weight"], state), _norm_rope_exact(k, state["k_weight"], state)
        if case["op"] == "append":
            k, v = _held_exact(k), _held_exact(v.reshape(-1, kv, d))
            return {"q": q.flatten(1), "k": k.flatten(1), "v": v.flatten(1)}
        return {"q": q.flatten(1), "k": k.flatten(1)}
    rows, at, page = [], 0, case["page"]
    for i, (n, length) in enumerate(_lengths(case)):
        first = max(0, length - n - case["window"] + 1) if case["window"] else 0
        place = torch.arange(first, length, device="cuda")
        slots = state["page_table"][i, place // page].long() * page + place % page
        out = torch.empty(n, case["heads_q"], d, dtype=torch.float64, device="cuda")
        keys, vals = (torch.cat([_lookup(state["cache"], s, w, case) for s in slots.split(16384)], 1) for w in (0, 1))
        q = state["q"][at : at + n].double().reshape(n, -1, d)
        last = length - n + torch.arange(n, device="cuda").unsqueeze(1)
        mask = place > last
        if case["window"]:
            mask = mask | (place <= last - case["window"])
        for h in range(case["heads_q"]):
            g = h // (case["heads_q"] // kv)
            out[:, h] = torch.softmax((q[:, h] @ keys[g].T / math.sqrt(d)).masked_fill_(mask, -math.inf), -1) @ vals[g]
        rows.append(out.flatten(1))
        at += n
    return {"out": torch.cat(rows)}
