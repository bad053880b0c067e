"""The operators of a cache in 8 bits and of trees of drafted tokens, as they are measured: their plain forms and the calls.

* write: rotation of queries and keys, keys and values quantised into the pages of an 8-bit cache (e4m3, one power of two for
  each token and kv head), and the written entries read back;
* attend: attention over such a cache, for single tokens, for portions of prompts, and for both beside each other;
* tree: attention of drafted tokens, each of which sees the context and its own ancestors, over a cache in 8 bits, in bfloat16
  or in float32;
* keep: what an accepted path of drafted tokens left in the cache is moved to the places of its positions, for all layers.

A case names the operator, the head layout, the page size, the type of the activations and of the cache, and how many tokens and
cached keys the requests have (`least` to `most`, spread evenly over the requests).
"""

import math

import torch

own = False

E4M3_TOP = 448.0
_ops = None


def _kernels():
    """The framework's kernels, constructed once as an engine does."""
    global _ops
    if _ops is None:
        from distie_amd.kernels.hip_ops import HipOps

        _ops = HipOps("cuda:0")
    return _ops


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    small = dict(heads=12, kv_heads=2, dim=128, page=16, act="bf16")            # the head layout of bench.py's 1.5b shape
    wide = dict(heads=28, kv_heads=4, dim=128, page=16, act="bf16")             # and of its 7b shape
    return [
        # one layer of a decode step of eight requests
        dict(small, name="write, 8 single tokens", op="write", requests=8, tokens=1, least=500, most=2048),
        # one layer of a step that brings two portions of prompts, the second behind what is cached
        dict(wide, name="write, 2 portions of 2,051", op="write", requests=2, tokens=2051, least=0, most=4099),
        # the lowest latency: one conversation
        dict(small, name="decode, 1 of 517 keys", op="attend", requests=1, tokens=1, least=516, most=516, window=0),
        # a serving batch whose requests differ in length
        dict(wide, name="decode, 64 of 1,050-3,150 keys", op="attend", requests=64, tokens=1, least=1050, most=3150, window=0),
        # long contexts, where the cache is what a step reads
        dict(wide, name="decode, 8 of 32,767 keys", op="attend", requests=8, tokens=1, least=32766, most=32766, window=0),
        # a portion of a prompt behind an earlier one
        dict(wide, name="portion of 2,048 behind 2,051", op="attend", requests=1, tokens=2048, least=2051, most=2051, window=0),
        # the float32 engine: short portions over a cache in 8 bits, a sliding window
        dict(small, name="float32, 6 of 37 tokens", op="attend", act="f32", requests=6, tokens=37, least=3, most=1500, window=1021),
        # one conversation with a small tree of drafted tokens, cache in bfloat16
        dict(small, name="tree of 7 over 300, bf16", op="tree", cache="bf16", requests=1, tokens=7, least=300, most=300, window=0),
        # a batch of conversations with trees of 61 drafted tokens over an 8-bit cache
        dict(wide, name="16 trees of 61, 8-bit", op="tree", cache="e4m3", requests=16, tokens=61, least=1001, most=4003, window=0),
        # wide trees of an offline draft over long contexts
        dict(wide, name="4 trees of 200, bf16", op="tree", cache="bf16", requests=4, tokens=200, least=9001, most=16001, window=0),
        # a few accepted tokens of one conversation, all layers of the 1.5b shape
        dict(small, name="keep, 1 path of 4", op="keep", cache="bf16", layers=28, requests=1, tokens=7, kept=4, least=300, most=300),
        # accepted paths of a batch
        dict(wide, name="keep, 32 paths of 9", op="keep", cache="bf16", layers=28, requests=32, tokens=61, kept=9, least=100, most=300),
    ]


def draw(rng):
    def over(low, high):                                    # spread over the logarithm
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    heads, kv_heads, dim = rng.choice([(12, 2, 128), (28, 4, 128), (40, 8, 128), (32, 8, 64), (14, 2, 64), (16, 16, 96), (8, 1, 256),
                                       (20, 4, 128), (24, 3, 64)])
    case = dict(op=rng.choice(["write", "attend", "attend", "attend", "tree", "tree", "keep"]), heads=heads, kv_heads=kv_heads, dim=dim,
                page=rng.choice([16, 16, 32, 64]), act=rng.choice(["bf16", "bf16", "bf16", "f32"]))
    if case["op"] == "write":
        case.update(requests=over(1, 64), least=rng.randrange(0, 900))
        case.update(tokens=over(1, 8192 // case["requests"]), most=case["least"] + over(1, 5000))
    elif case["op"] == "attend":
        single = rng.random() < 0.6
        case.update(requests=over(1, 96) if single else over(1, 8))
        case.update(tokens=1 if single else over(2, 2048 // case["requests"]))
        limit = 200000 // case["requests"] if single else 4000
        case["most"] = over(1, min(limit, 40000))
        case.update(least=rng.randrange(0, case["most"] + 1), window=rng.choice([0, 0, 0, rng.randrange(1, 4500)]))
    elif case["op"] == "tree":
        case.update(requests=over(1, 24), cache=rng.choice(["e4m3", "bf16"] if case["act"] == "bf16" else ["e4m3", "f32"]))
        case.update(tokens=over(1, min(256, 1024 // case["requests"])), most=over(1, 64000 // case["requests"]))
        case.update(least=rng.randrange(0, case["most"] + 1), window=rng.choice([0, 0, 0, rng.randrange(1, 4500)]))
    else:
        case.update(requests=over(1, 32), layers=over(2, 32), cache="f32" if case["act"] == "f32" else "bf16", tokens=over(2, 64))
        case.update(kept=rng.randrange(1, min(12, case["tokens"]) + 1), least=rng.randrange(0, 100), most=rng.randrange(100, 250))
    return case


def _past(case):
    """Cached keys of every request, in front of its new tokens: `least` to `most`, evenly spread and out of order."""
    n, low, span = case["requests"], case["least"], case["most"] - case["least"]
    spread = [low + (span * i // (n - 1) if n > 1 else span) for i in range(n)]
    return spread[::2] + spread[1::2][::-1]


def _pages(case):
    """Pages of every request, one to spare."""
    return [(p + case["tokens"]) // case["page"] + 1 for p in _past(case)]


def _seen(case):
    """(keys that the request's tokens see between them, pairs of token and key) over all requests."""
    window, n, keys, pairs = case["window"] or 1 << 40, case["tokens"], 0, 0
    for past in _past(case):
        if case["op"] == "tree":                            # at least the context and itself
            keys += min(past, window) + n
            pairs += n * (min(past, window) + 1)
        else:
            keys += past + n - max(0, past + 1 - window)
            pairs += sum(min(past + i + 1, window) for i in range(n))
    return keys, pairs


def work(case):
    act = 4 if case["act"] == "f32" else 2
    T, H, KH, D = case["requests"] * case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "write":                               # qkv in, q out, codes and powers out and in again, values out
        codes = T * 2 * KH * (D + 1)
        return {"bytes": T * ((2 * H + 2 * KH) * D * act + 2 * KH * D * 2) + 2 * codes, "flops": T * (H + KH) * D * 3}
    if case["op"] == "keep":
        moved = case["requests"] * case["kept"] * case["layers"] * 2 * KH * D
        return {"bytes": 2 * moved * (4 if case["cache"] == "f32" else 2), "flops": 0}
    keys, pairs = _seen(case)
    entry = {"e4m3": D + 1, "bf16": 2 * D, "f32": 4 * D}[case.get("cache", "e4m3")]
    return {"bytes": 2 * T * H * D * act + keys * 2 * KH * entry, "flops": 4 * pairs * H * D}


# --------------------------------------------------------------------------------------------------------------- inputs
def _quantise(x):
    """x float32 [..., D] -> (codes e4m3, uint8 powers [...]): the smallest power of two at which the row's largest value fits."""
    bits = x.abs().amax(-1).view(torch.int32)
    power = ((bits >> 23) - 135 + ((bits & 0x7FFFFF) > 0x600000)).clamp(-126, 127)
    codes = torch.ldexp(x, -power[..., None]).to(torch.float8_e4m3fn)
    return codes, (power + 127).to(torch.uint8)


def _values(codes, powers):
    return torch.ldexp(codes.float(), powers[..., None].to(torch.int32) - 127)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    host = torch.Generator().manual_seed(int(seed))
    act = torch.float32 if case["act"] == "f32" else torch.bfloat16
    B, n, P, H, KH, D = (case[k] for k in ("requests", "tokens", "page", "heads", "kv_heads", "dim"))
    past, pages = _past(case), _pages(case)
    width = max(pages)
    order = torch.randperm(sum(pages), generator=host, dtype=torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32)
    at = 0
    for b, count in enumerate(pages):
        table[b, :count] = order[at:at + count]
        at += count
    index = torch.tensor(past)[:, None] + torch.arange(n)[None]                  # place in the cache of every new token
    slots = table.gather(1, index // P).long() * P + index % P
    place = lambda t: t.to("cuda", torch.int32).contiguous()
    state = dict(
        case=case, table=place(table), slots=place(slots.view(-1)), positions=place(index.view(-1)),
        request=place(torch.arange(B)[:, None].expand(B, n).reshape(-1)), cu_q=place(torch.arange(B + 1) * n),
        kv_len=place(torch.tensor(past) + n), host_past=torch.tensor(past).numpy(), host_cu_q=(torch.arange(B + 1) * n).numpy(),
        max_kv=max(past) + n)
    randn = lambda *shape: torch.randn(shape, generator=gen, device="cuda")
    # keys have channels much larger than the rest, values have means, and tokens differ in size
    big = 1 + 3 * (torch.rand(KH, D, generator=gen, device="cuda") > 0.95)
    mean = 0.3 * randn(KH, D)
    if case["op"] == "write":
        x = randn(B * n, H + 2 * KH, D)
        x[:, H:H + KH] *= big
        x[:, H + KH:] = (x[:, H + KH:] + mean) * torch.exp(0.5 * randn(B * n, 1, 1))
        state["qkv"] = x.view(B * n, -1).to(act)
        state["inv_freq"] = (1000000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).float().cuda()
        state["k"] = torch.zeros(sum(pages), KH, P, D, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        state["v"] = torch.zeros(sum(pages), KH, D, P, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        state["k_scale"] = torch.ones(sum(pages), KH, P, dtype=torch.uint8, device="cuda")
        state["v_scale"] = torch.ones(sum(pages), KH, P, dtype=torch.uint8, device="cuda")
        return state
    layers = (case["layers"],) if case["op"] == "keep" else ()
    k = randn(*layers, sum(pages), KH, P, D) * big[:, None]
    v = (randn(*layers, sum(pages), KH, P, D) + mean[:, None]) * torch.exp(0.5 * randn(sum(pages), KH, P, 1))
    if case.get("cache", "e4m3") == "e4m3":
        codes, state["k_scale"] = _quantise(k)
        state["k"] = codes
        codes, state["v_scale"] = _quantise(v)
        state["v"] = codes.view(torch.uint8).transpose(-1, -2).contiguous().view(torch.float8_e4m3fn)
    else:
        kept = torch.float32 if case["cache"] == "f32" else torch.bfloat16
        state["k"], state["v"] = k.to(kept), v.to(kept).transpose(-1, -2).contiguous()
    if case["op"] == "keep":
        # an accepted path: the first drafted token and further ones in their order
        path = torch.rand(B, n - 1, generator=host).argsort(1)[:, :case["kept"] - 1].sort(1).values + 1
        state["path"] = place(torch.cat([torch.zeros(B, 1, dtype=path.dtype), path], 1))
        state["past"] = place(torch.tensor(past))
        return state
    state["q"] = (1.5 * randn(B * n, H * D)).to(act)
    state["scale"] = D ** -0.5
    if case["op"] == "tree":
        # drafted token 0 is the root; every other one hangs on an earlier one, mostly a near one
        sees = torch.zeros(B, n, n, dtype=torch.bool)
        depth = torch.zeros(B, n, dtype=torch.int64)
        rows = torch.arange(B)
        for i in range(n):
            if i:
                parent = (i - 1 - (torch.rand(B, generator=host) ** 2 * min(i, 8)).long()).clamp(min=0)
                sees[:, i] = sees[rows, parent]
                depth[:, i] = depth[rows, parent] + 1
            sees[:, i, i] = True
        words = -(-n // 64)
        bits = torch.nn.functional.pad(sees, (0, 64 * words - n)).view(B * n, words, 64).long()
        state["visible"] = (bits << torch.arange(64)).sum(-1).to("cuda").contiguous()
        state["positions"] = place((torch.tensor(past)[:, None] + depth).view(-1))
    return state


# ------------------------------------------------------------------------------------------------------------ one pass
def _meta(s, tree=None):
    from distie_amd.kernels.interface import BatchMeta, GroupMeta

    case = s["case"]
    return BatchMeta(num_tokens=case["requests"] * case["tokens"], num_requests=case["requests"], positions=s["positions"],
                     token_request=s["request"], cu_q=s["cu_q"], kv_len=s["kv_len"], state_slots=s["request"], max_q=case["tokens"],
                     max_kv=s["max_kv"], block_size=case["page"], groups=[GroupMeta(block_table=s["table"], slots=s["slots"])],
                     host_cu_q=s["host_cu_q"], host_past=s["host_past"], all_decode=case["tokens"] == 1 and tree is None, tree=tree)


def _cache(s):
    from distie_amd.kernels.interface import EightBitCache

    return EightBitCache(s["k"], s["v"], s["k_scale"], s["v_scale"]) if "k_scale" in s else (s["k"], s["v"])


def _run_own(s):
    ops, case = _kernels(), s["case"]
    H, KH, D, window = case["heads"], case["kv_heads"], case["dim"], case.get("window") or None
    if case["op"] == "write":
        cache = _cache(s)
        q = ops.rope_kv_write_e4m3(s["qkv"], _meta(s), 0, cache, s["inv_freq"], H, KH, D, True)
        k, v = ops.read_kv_e4m3(cache, s["slots"], torch.bfloat16)
        return {"q": q, "k": k, "v": v}
    if case["op"] == "attend":
        return ops.paged_attention_e4m3(s["q"], _meta(s), 0, _cache(s), H, KH, D, s["scale"], window)
    if case["op"] == "tree":
        return ops.tree_attention(s["q"], _meta(s, s["visible"]), 0, _cache(s), H, KH, D, s["scale"], window)
    ops.keep_drafted(s["k"], 3, s["table"], None, s["past"], s["path"])
    ops.keep_drafted(s["v"], 4, s["table"], None, s["past"], s["path"])
    return {"k": s["k"], "v": s["v"]}


def _plain_write(s):
    case = s["case"]
    H, KH, D, P = case["heads"], case["kv_heads"], case["dim"], case["page"]
    x = s["qkv"].float().view(-1, H + 2 * KH, D)
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[:, :H + KH, :D // 2], x[:, :H + KH, D // 2:]
    turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    page, at = s["slots"].long() // P, s["slots"].long() % P
    k, k_scale = _quantise(turned[:, H:])
    v, v_scale = _quantise(x[:, H + KH:])
    s["k"].view(torch.uint8)[page, :, at] = k.view(torch.uint8)
    s["v"].view(torch.uint8)[page, :, :, at] = v.view(torch.uint8)
    s["k_scale"][page, :, at] = k_scale
    s["v_scale"][page, :, at] = v_scale
    k = s["k"].view(torch.uint8)[page, :, at].view(torch.float8_e4m3fn)
    v = s["v"].view(torch.uint8)[page, :, :, at].view(torch.float8_e4m3fn)
    return {"q": turned[:, :H].reshape(-1, H * D).to(s["qkv"].dtype),
            "k": _values(k, s["k_scale"][page, :, at]).bfloat16(), "v": _values(v, s["v_scale"][page, :, at]).bfloat16()}


def _plain_keys(s, as_type):
    """The cached keys and values of every request in their order, [B, KH, L, D]."""
    table = s["table"].long().clamp(min=0)
    if "k_scale" in s:
        k = s["k"].view(torch.uint8)[table].view(torch.float8_e4m3fn).to(as_type)
        v = s["v"].view(torch.uint8)[table].view(torch.float8_e4m3fn).to(as_type)
        k = k * torch.ldexp(torch.ones((), device="cuda"), s["k_scale"][table].int() - 127).to(as_type)[..., None]
        v = v * torch.ldexp(torch.ones((), device="cuda"), s["v_scale"][table].int() - 127).to(as_type)[..., None, :]
    else:
        k, v = s["k"][table].to(as_type), s["v"][table].to(as_type)
    B, W, KH, P, D = k.shape
    return k.transpose(1, 2).reshape(B, KH, W * P, D), v.permute(0, 2, 1, 4, 3).reshape(B, KH, W * P, D)


def _plain_attend(s):
    case = s["case"]
    B, n, H, KH, D = (case[k] for k in ("requests", "tokens", "heads", "kv_heads", "dim"))
    k, v = _plain_keys(s, torch.float32)
    L = k.shape[2]
    key, position = torch.arange(L, device="cuda"), s["positions"].long().view(B, n, 1)
    past = s["kv_len"].long()[:, None, None] - n
    if case["op"] == "tree":
        bits = ((s["visible"][:, :, None] >> torch.arange(64, device="cuda")) & 1).bool().view(B, n, -1)[:, :, :n]
        drafted = (key - past).clamp(0, n - 1)
        seen = (key < past) | ((key < past + n) & bits.gather(2, drafted.expand(B, n, L)))
        key_position = torch.where(key < past, key, s["positions"].long().view(B, 1, n).gather(2, drafted.expand(B, 1, L)))
    else:
        seen, key_position = key <= position, key
    if case["window"]:
        seen = seen & (position - key_position < case["window"])
    q = s["q"].float().view(B, n, KH, H // KH, D).permute(0, 2, 1, 3, 4).reshape(B, KH, -1, D)
    score = torch.matmul(q, k.transpose(2, 3)).mul_(s["scale"]).view(B, KH, n, H // KH, L)
    score.masked_fill_(~seen.view(B, 1, n, 1, L), -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight.view(B, KH, -1, L), v).view(B, KH, n, H // KH, D)
    out = torch.where(total > 0, out / total, 0.0)
    return out.permute(0, 2, 1, 3, 4).reshape(B * n, H * D).to(s["q"].dtype)


def _plain_keep(s):
    case = s["case"]
    P, rows = case["page"], torch.arange(case["requests"], device="cuda")[:, None]
    source = s["past"].long()[:, None] + s["path"].long()
    target = s["past"].long()[:, None] + torch.arange(case["kept"], device="cuda")
    table = s["table"].long()
    from_page, to_page = table[rows, source // P], table[rows, target // P]
    s["k"][:, to_page, :, target % P] = s["k"][:, from_page, :, source % P]
    s["v"][:, to_page, :, :, target % P] = s["v"][:, from_page, :, :, source % P]
    return {"k": s["k"], "v": s["v"]}


def run(state):
    if own:
        return _run_own(state)
    return {"write": _plain_write, "attend": _plain_attend, "tree": _plain_attend, "keep": _plain_keep}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------- the definition, 64 bits
def _exact_codes(x):
    """Rows of float64 to the values that their codes stand for: 4 significant bits, nothing finer than 2^-9 of the power."""
    largest = x.abs().amax(-1, keepdim=True)
    power = torch.ceil(torch.log2(largest / E4M3_TOP)).clamp(-126, 127)
    power = torch.where(E4M3_TOP * torch.exp2(power - 1) >= largest, power - 1, power)          # (the logarithm rounds)
    power = torch.where(E4M3_TOP * torch.exp2(power) < largest, power + 1, power).clamp(-126, 127)
    y = x / torch.exp2(power)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step * torch.exp2(power)


def exact(case, seed):
    s = prepare(case, seed)
    B, n, H, KH, D, P = (case[k] for k in ("requests", "tokens", "heads", "kv_heads", "dim", "page"))
    if case["op"] == "write":
        x = s["qkv"].double().view(-1, H + 2 * KH, 2, D // 2)
        angle = (s["positions"].double()[:, None] * s["inv_freq"].double())[:, None]
        first = x[:, :, 0] * torch.cos(angle) - x[:, :, 1] * torch.sin(angle)
        second = x[:, :, 1] * torch.cos(angle) + x[:, :, 0] * torch.sin(angle)
        turned = torch.stack([first, second], 2).view(-1, H + 2 * KH, D)
        return {"q": turned[:, :H].reshape(-1, H * D), "k": _exact_codes(turned[:, H:H + KH]),
                "v": _exact_codes(x[:, H + KH:].reshape(-1, KH, D))}
    if case["op"] == "keep":
        k, v = s["k"].clone(), s["v"].clone()
        for b, (past, path) in enumerate(zip(s["past"].tolist(), s["path"].tolist())):
            for d, i in enumerate(path):
                there, here = (int(s["table"][b, (past + j) // P]) for j in (i, d))
                k[:, here, :, (past + d) % P] = s["k"][:, there, :, (past + i) % P]
                v[:, here, :, :, (past + d) % P] = s["v"][:, there, :, :, (past + i) % P]
        return {"k": k, "v": v}
    out = torch.empty(B * n, H, D, dtype=torch.float64, device="cuda")
    visible = s["visible"].cpu().tolist() if case["op"] == "tree" else None
    for b, past in enumerate(_past(case)):
        one = dict(s, table=s["table"][b:b + 1, :-(-(past + n) // P)])
        k, v = (t[0, :, :past + n] for t in _plain_keys(one, torch.float64))
        where = s["positions"][b * n:(b + 1) * n].long()
        of_key = torch.arange(past + n, device="cuda")
        if visible is None:
            sees = of_key <= where[:, None]
        else:
            of_key[past:] = where
            drafted = [[bool(visible[b * n + i][j // 64] >> (j % 64) & 1) for j in range(n)] for i in range(n)]
            sees = torch.cat([torch.ones(n, past, dtype=torch.bool), torch.tensor(drafted)], 1).cuda()
        if case["window"]:
            sees = sees & (of_key > where[:, None] - case["window"])
        for h in range(H):
            score = s["q"][b * n:(b + 1) * n, h * D:(h + 1) * D].double() @ k[h * KH // H].T * s["scale"]
            out[b * n:(b + 1) * n, h] = torch.softmax(score.masked_fill(~sees, -math.inf), -1).nan_to_num(0.0) @ v[h * KH // H]
    return out.view(B * n, H * D)
