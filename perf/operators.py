"""What an attention layer runs between its weight products, as cases that can be timed and compared: keys and values
appended to a paged 8-bit cache with the rotation of their positions, attention over that cache, and the norms around a
block with its gate and residual. Sizes are those of the products this library is timed on and generic ones.

`run` computes a case in its plain form (elementary torch operations in 32 bits), or, where `own` is set, through
dromos_b200.host. `exact` computes it again from the definitions in 64 bits.

The cache: pages of `page` tokens, codes [pages, kv_heads, page, dim] in E4M3 or INT8, one power-of-two scale per page
and head for keys and for values; a sequence's pages are listed in its row of the page table. A scale is the smallest
power of two that brings the largest magnitude of the page's tokens so far to 448 (INT8: 127) or less.
"""

import math
import random

import torch

own = False

TOP = {"fp8": 448.0, "int8": 127.0}
MOST_SCORES = 32 * 8192 * 8192 // 4  # query-key pairs of a drawn case, so that its plain form fits


def listed():
    return [
        # One sequence decodes one token: appended in the type of a decode step's product. Latency alone.
        {"name": "append_1", "op": "append", "type": "int8", "sequences": 1, "new": 1, "history": 700, "ragged": False, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "rotary": 128, "interleaved": False, "input": "f32", "far": 0},
        # A decode step of 64 sequences, at positions far into long contexts.
        {"name": "append_64", "op": "append", "type": "fp8", "sequences": 64, "new": 1, "history": 250, "ragged": True, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "rotary": 128, "interleaved": False, "input": "f32", "far": 1000000},
        # Prompts of three sequences, ragged, half of each head rotated in neighbouring pairs.
        {"name": "append_prompts", "op": "append", "type": "fp8", "sequences": 3, "new": 4001, "history": 90, "ragged": True, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "rotary": 64, "interleaved": True, "input": "bf16", "far": 0},
        # The rows of one decoded token between two blocks of width 4096.
        {"name": "norm_1", "op": "norm", "rows": 1, "width": 4096, "y": "f32", "h": "f32", "weight": "bf16", "post": True, "gate": "none"},
        # A decode batch, residual kept in bf16, a gate per token and channel.
        {"name": "norm_33", "op": "norm", "rows": 33, "width": 8192, "y": "f32", "h": "bf16", "weight": "bf16", "post": True, "gate": "token"},
        # A prompt's rows, residual in 32 bits, a learned gate per channel.
        {"name": "norm_4096", "op": "norm", "rows": 4096, "width": 8192, "y": "f32", "h": "f32", "weight": "f32", "post": True, "gate": "channel"},
        # One sequence decodes one token over four thousand cached ones.
        {"name": "decode_1", "op": "attention", "type": "fp8", "sequences": 1, "new": 1, "length": 4099, "ragged": False, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "window": 0, "q": "bf16"},
        # A decode batch over ragged contexts: the cache is what is read.
        {"name": "decode_64", "op": "attention", "type": "fp8", "sequences": 64, "new": 1, "length": 8192, "ragged": True, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "window": 0, "q": "bf16"},
        # Four drafted tokens per sequence, INT8, small pages, small heads, a window.
        {"name": "draft_8", "op": "attention", "type": "int8", "sequences": 8, "new": 4, "length": 6001, "ragged": True, "heads": 14, "kv_heads": 2, "dim": 64,
         "page": 16, "window": 4096, "q": "bf16"},
        # Wide heads, few of them, a decode batch.
        {"name": "decode_wide", "op": "attention", "type": "int8", "sequences": 24, "new": 1, "length": 5000, "ragged": True, "heads": 16, "kv_heads": 4, "dim": 256,
         "page": 32, "window": 0, "q": "bf16"},
        # A whole prompt at once: the products of its scores are what counts.
        {"name": "prompt_8192", "op": "attention", "type": "fp8", "sequences": 1, "new": 8192, "length": 8192, "ragged": False, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "window": 0, "q": "bf16"},
        # Pieces of four prompts over what is cached of them, ragged, INT8.
        {"name": "pieces_4", "op": "attention", "type": "int8", "sequences": 4, "new": 513, "length": 7000, "ragged": True, "heads": 16, "kv_heads": 2, "dim": 128,
         "page": 32, "window": 0, "q": "bf16"},
    ]


def spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["append", "norm", "attention", "attention"])
    if op == "norm":
        width = 8 * spread(rng, 64, 1024)
        return {"op": op, "rows": spread(rng, 1, 4096 * 8192 // width // 2), "width": width, "y": rng.choice(["f32", "bf16"]), "h": rng.choice(["f32", "bf16"]),
                "weight": rng.choice(["f32", "bf16"]), "post": rng.random() < 0.7, "gate": rng.choice(["none", "channel", "token"])}
    kv_heads, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256])
    case = {"op": op, "type": rng.choice(["fp8", "int8"]), "sequences": spread(rng, 1, 48), "new": 1, "ragged": rng.random() < 0.7,
            "heads": kv_heads * rng.choice([1, 2, 3, 4, 7, 8]), "kv_heads": kv_heads, "dim": dim, "page": rng.choice([16, 32, 64, 128])}
    if rng.random() < 0.5:
        case["new"] = spread(rng, 2, 2048)
        case["sequences"] = max(1, min(case["sequences"], 4096 // case["new"]))
    if op == "append":
        case |= {"history": spread(rng, 1, 500), "rotary": rng.choice([0, dim // 2, dim]), "interleaved": rng.random() < 0.5, "input": rng.choice(["f32", "bf16"]),
                 "far": rng.choice([0, 1000000])}
        return case
    case |= {"length": case["new"] + spread(rng, 1, 8192), "window": rng.choice([0, 0, spread(rng, 1, 4096)]), "q": rng.choice(["f32", "bf16"])}
    while case["sequences"] > 1 and (case["sequences"] * case["heads"] * case["new"] * case["length"] > MOST_SCORES
                                     or case["sequences"] * case["kv_heads"] * dim * case["length"] > 64 * 8 * 128 * 4096):
        case["sequences"] = (case["sequences"] + 1) // 2
    while case["heads"] * case["new"] * case["length"] > MOST_SCORES:
        case["length"] -= case["new"] // 2
        case["new"] -= case["new"] // 2
    return case


def spans(case):
    """New tokens and tokens in the cache (the new ones included) of each sequence."""
    rng = random.Random("%d %d %d" % (case["sequences"], case["new"], case.get("length", 0)))
    new = [case["new"] if i == 0 or not case["ragged"] else rng.randint((case["new"] + 1) // 2, case["new"]) for i in range(case["sequences"])]
    if case["op"] == "append":
        past = [case["history"] if i == 0 or not case["ragged"] else rng.randint(0, case["history"]) for i in range(case["sequences"])]
        return new, [n + p for n, p in zip(new, past)]
    total = [case["length"] if i == 0 or not case["ragged"] else rng.randint(max(n, case["length"] // 8), case["length"]) for i, n in enumerate(new)]
    return new, total


def work(case):
    if case["op"] == "norm":
        size = {"f32": 4, "bf16": 2}
        cells = case["rows"] * case["width"]
        gate = {"none": 0, "channel": case["width"], "token": cells}[case["gate"]]
        weights = case["width"] * (1 + case["post"])
        return {"bytes": cells * (size[case["y"]] + 2 * size[case["h"]] + 2) + 2 * gate + weights * size[case["weight"]], "flops": 10 * cells}
    new, total = spans(case)
    H, K, D = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        T, size = sum(new), {"f32": 4, "bf16": 2}[case["input"]]
        pages = sum((t - 1) // case["page"] - (t - n) // case["page"] + 1 for n, t in zip(new, total))
        return {"bytes": T * ((H + 2 * K) * D * size + H * D * 2 + 2 * K * D) + 8 * K * pages, "flops": T * ((H + K) * case["rotary"] * 3 + 4 * K * D)}
    keys = pairs = 0
    for n, t in zip(new, total):
        w = case["window"] or t
        keys += t - max(0, t - n - w + 1)
        first = t - n + 1  # keys that the first query could see, itself among them
        short = max(0, min(n, w - first + 1))  # queries that see every key before them
        pairs += short * first + short * (short - 1) // 2 + (n - short) * w
    T = sum(new)
    return {"bytes": 2 * K * D * keys + 8 * K * (keys // case["page"]) + T * H * D * (2 + {"f32": 4, "bf16": 2}[case["q"]]), "flops": 4 * D * H * pairs}


def dtype_of(name):
    return {"f32": torch.float32, "bf16": torch.bfloat16}[name]


def exponent(largest, kind):
    """The smallest power of two s with largest <= TOP * s, as its exponent."""
    m, e = torch.frexp(largest)  # largest = m 2^e, m in [0.5, 1); 448 = 0.875 2^9, 127 = (127 / 128) 2^7
    e = e - (9 if kind == "fp8" else 7) + (m > (0.875 if kind == "fp8" else 127 / 128)).to(e.dtype)
    return torch.where(largest == 0, torch.full_like(e, -100), e.clamp(-100, 120))


def encode(x, kind):
    """Values already divided by their scale, as codes in bytes."""
    if kind == "fp8":
        return x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    return x.clamp(-127, 127).round().to(torch.int8).view(torch.uint8)


def decode(codes, kind):
    return codes.view(torch.float8_e4m3fn if kind == "fp8" else torch.int8).float()


def stored(g, shape, kind):
    """A cache half filled by earlier tokens: codes and scales of normal values, some pages and heads louder than others."""
    x = torch.randn(shape, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(shape[:2], generator=g, device="cuda"))[:, :, None, None]
    scale = torch.ldexp(torch.ones(shape[:2], device="cuda"), exponent(x.abs().amax((2, 3)), kind))
    return encode(x / scale[:, :, None, None], kind), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    if case["op"] == "norm":
        T, C = case["rows"], case["width"]
        weight = dtype_of(case["weight"])
        state = {"case": case, "y": normal(T, C, dtype=dtype_of(case["y"]), scale=0.7), "h": normal(T, C, dtype=dtype_of(case["h"]), scale=2.0),
                 "pre": 1 + normal(C, dtype=weight, scale=0.1), "post": 1 + normal(C, dtype=weight, scale=0.1) if case["post"] else None,
                 "gate": {"none": None, "channel": (C,), "token": (T, C)}[case["gate"]], "residual_scale": 0.9, "block_scale": 1.5, "eps": 1e-6}
        if state["gate"] is not None:
            state["gate"] = normal(*state["gate"], dtype=torch.bfloat16)
        state["handle"] = handle(state) if own else None
        return state
    new, total = spans(case)
    S, T, H, K, D, P = case["sequences"], sum(new), case["heads"], case["kv_heads"], case["dim"], case["page"]
    most = max(-(-t // P) for t in total)
    pages = sum(-(-t // P) for t in total)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).cpu()
    table, at = torch.full((S, most), -1, dtype=torch.int32), 0
    for s, t in enumerate(total):
        n = -(-t // P)
        table[s, :n] = order[at:at + n]
        at += n
    starts = torch.tensor([sum(new[:s]) for s in range(S + 1)], dtype=torch.int32)
    k, k_scale = stored(g, (pages, K, P, D), case["type"])
    v, v_scale = stored(g, (pages, K, P, D), case["type"])
    state = {"case": case, "tokens": T, "most_new": max(new), "starts": starts.cuda(), "lengths": torch.tensor(total, dtype=torch.int32).cuda(), "pages": table.cuda(),
             "k": k, "v": v, "k_scale": k_scale, "v_scale": v_scale}
    if case["op"] == "append":
        rows = normal(T, (H + 2 * K) * D, dtype=dtype_of(case["input"]), scale=1.3)  # what the product of q, k and v wrote
        state |= {"q_in": rows[:, :H * D], "k_in": rows[:, H * D:(H + K) * D], "v_in": rows[:, (H + K) * D:]}
        state["frequencies"] = torch.pow(torch.tensor(500000.0, dtype=torch.float64), -torch.arange(0, case["rotary"], 2, dtype=torch.float64) / max(1, case["rotary"])).cuda()
        slots = torch.cat([torch.arange(t - n, t, dtype=torch.int32) for n, t in zip(new, total)])
        state["positions"] = (slots + case["far"]).cuda()
    else:
        state["q"] = normal(T, H * D, dtype=dtype_of(case["q"]), scale=2.0)
        state["scale"] = 1 / math.sqrt(D)
    state["handle"] = handle(state) if own else None
    return state


_library = None


def handle(state):
    """The objects a program keeps for these buffers."""
    global _library
    from dromos_b200 import abi, host

    if _library is None:
        _library = abi.Library()
    case = state["case"]
    if case["op"] == "norm":
        return host.NormResidual(_library, case["width"], pre=state["pre"], post=state["post"], residual_scale=state["residual_scale"], block_scale=state["block_scale"],
                                 gate_sigmoid=case["gate"] == "token", eps=state["eps"])
    wtype = {"fp8": abi.W_FP8, "int8": abi.W_INT8}[case["type"]]
    cache = host.KvCache(_library, wtype, state["k"], state["v"], state["k_scale"], state["v_scale"])
    batch = host.KvBatch(state["starts"], state["lengths"], state["pages"], tokens=state["tokens"], max_new=state["most_new"])
    if case["op"] == "append":
        return cache, batch, host.Rotary(state["frequencies"], interleaved=case["interleaved"]) if case["rotary"] else None
    return host.Attention(cache, case["heads"], scale=state["scale"], window=case["window"]), batch


def run(state):
    case = state["case"]
    if case["op"] == "norm":
        if own:
            return state["handle"](state["y"], state["h"], gate=state["gate"])
        return norm(state)
    if case["op"] == "append":
        if own:
            cache, batch, rotary = state["handle"]
            q = cache.append(batch, state["k_in"], state["v_in"], q=state["q_in"], rotary=rotary, positions=state["positions"])
        else:
            q = append(state)
        return q, held(state["k"], state["k_scale"], case), held(state["v"], state["v_scale"], case), state["k_scale"], state["v_scale"]
    if own:
        attention_, batch = state["handle"]
        return attention_(batch, state["q"])
    return attention(state)


def held(codes, scale, case):
    """The cache as the numbers it holds: E4M3 codes as such (their scales are outputs of their own); INT8 ones times their
    scale, which bf16 holds exactly."""
    if case["type"] == "fp8":
        return codes.view(torch.float8_e4m3fn)
    return codes.view(torch.int8) * scale.to(torch.bfloat16)[:, :, None, None]


def places(state):
    """Of each new token: its sequence, its slot there."""
    token = torch.arange(state["tokens"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(state["starts"], token, right=True) - 1
    return seq, state["lengths"][seq] - (state["starts"][seq + 1] - token)


def rotate(x, state):
    """x f32 [T, heads, dim], each pair turned by position * frequency."""
    r = state["case"]["rotary"]
    if not r:
        return x
    angle = state["positions"].double()[:, None, None] * state["frequencies"]
    c, s = angle.cos().float(), angle.sin().float()
    turned = x[..., :r]
    if state["case"]["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = turned[..., :r // 2], turned[..., r // 2:]
        turned = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((turned, x[..., r:]), -1)


def append(state):
    case = state["case"]
    K, D, P, kind = case["kv_heads"], case["dim"], case["page"], case["type"]
    seq, slot = places(state)
    page, offset = state["pages"][seq, slot // P].long(), slot % P
    pages = state["k"].shape[0]
    # tokens that a page held before: none where its first slot is among the new ones, and then its scale starts anew
    kept = torch.full((pages,), P, device="cuda").index_reduce_(0, page, offset.long(), "amin")
    touched = (kept < P)[:, None]
    rescaled = touched[..., None] & (torch.arange(P, device="cuda") < kept[:, None])[:, None]
    q = rotate(state["q_in"].float().reshape(-1, case["heads"], D), state)
    new_k = rotate(state["k_in"].float().reshape(-1, K, D), state)
    new_v = state["v_in"].float().reshape(-1, K, D)
    for x, codes, scale in ((new_k, state["k"], state["k_scale"]), (new_v, state["v"], state["v_scale"])):
        largest = torch.zeros(pages, K, device="cuda").index_reduce_(0, page, x.abs().amax(2), "amax")
        wanted = torch.ldexp(torch.ones_like(scale), exponent(largest, kind))
        now = torch.where(touched, torch.maximum(torch.where(kept[:, None] == 0, torch.zeros_like(scale), scale), wanted), scale)
        old = encode(decode(codes, kind) * (scale / now)[:, :, None, None], kind)
        codes.copy_(torch.where(rescaled[..., None], old, codes))
        codes[page, :, offset.long()] = encode(x / now[page][:, :, None], kind)
        scale.copy_(now)
    return q.to(torch.bfloat16).reshape(-1, case["heads"] * D)


def attention(state):
    case = state["case"]
    S, H, K, D, P, N = case["sequences"], case["heads"], case["kv_heads"], case["dim"], case["page"], state["most_new"]
    table = state["pages"].clamp(min=0).long()

    def gather(codes, scale):  # [S, K, L, D]
        x = decode(codes[table], case["type"]) * scale[table][..., None, None]
        return x.transpose(1, 2).reshape(S, K, -1, D)

    seq, slot = places(state)
    i = torch.arange(state["tokens"], device="cuda") - state["starts"][seq]
    q = torch.zeros(S, N, H, D, device="cuda")
    q[seq, i] = state["q"].float().reshape(-1, H, D) * state["scale"]
    q = q.reshape(S, N, K, H // K, D).permute(0, 2, 1, 3, 4).reshape(S, K, N * (H // K), D)
    scores = (q @ gather(state["k"], state["k_scale"]).transpose(2, 3)).view(S, K, N, H // K, -1)
    at = torch.arange(scores.shape[-1], device="cuda")
    last = (state["lengths"] - state["starts"][1:] + state["starts"][:-1])[:, None] + torch.arange(N, device="cuda")
    seen = at <= last[..., None]
    if case["window"]:
        seen &= at > last[..., None] - case["window"]
    seen &= (at < state["lengths"][:, None])[:, None]  # rows past a sequence's last new token are padding
    scores.masked_fill_(~seen[:, None, :, None], -math.inf)
    weights = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    values = torch.where((at < state["lengths"][:, None])[:, None, :, None], gather(state["v"], state["v_scale"]), 0.0)
    out = weights.view(S, K, N * (H // K), -1) @ values / weights.sum(-1).view(S, K, -1, 1)
    return out.view(S, K, N, H // K, D)[seq, :, i].to(torch.bfloat16).reshape(-1, H * D)


def norm(state):
    case, C = state["case"], state["case"]["width"]

    def normed(x, weight):
        return x * torch.rsqrt(x.square().sum(-1, keepdim=True) / C + state["eps"]) * weight.float()

    block = state["y"].float()
    if case["post"]:
        block = normed(block, state["post"])
    if case["gate"] == "channel":
        block = block * state["gate"].float()
    elif case["gate"] == "token":
        block = block / (1 + torch.exp(-state["gate"].float()))
    h = state["residual_scale"] * state["h"].float() + state["block_scale"] * block
    return h.to(state["h"].dtype), normed(h, state["pre"]).to(torch.bfloat16)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "norm":
        y, h, n = state["y"].double(), state["h"].double(), case["width"]
        if case["post"]:
            y = y / torch.sqrt((y * y).mean(1, keepdim=True) + state["eps"]) * state["post"].double()
        if case["gate"] != "none":
            gate = state["gate"].double()
            y = y * (torch.sigmoid(gate) if case["gate"] == "token" else gate)
        h = h * state["residual_scale"] + y * state["block_scale"]
        return h, h / torch.sqrt((h * h).sum(1, keepdim=True) / n + state["eps"]) * state["pre"].double()
    new, total = spans(case)
    D, K, P = case["dim"], case["kv_heads"], case["page"]
    G = case["heads"] // K
    if case["op"] == "append":
        T, r = sum(new), case["rotary"]
        turn = torch.polar(torch.ones(T, r // 2, dtype=torch.float64, device="cuda"), state["positions"].double()[:, None] * state["frequencies"][None]) if r else None

        def turned(x, heads):
            x = x.double().reshape(T, heads, D).clone()
            if r:
                first, second = (slice(0, r, 2), slice(1, r, 2)) if case["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
                z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn[:, None]
                x[..., first], x[..., second] = z.real, z.imag
            return x

        table, row = state["pages"].cpu().tolist(), 0
        for s, (n, t) in enumerate(zip(new, total)):
            keys = turned(state["k_in"], K) if s == 0 else keys
            for page in range((t - n) // P, (t - 1) // P + 1):
                lo, hi = max(t - n, page * P), min(t, page * P + P)
                at = slice(row + lo - (t - n), row + hi - (t - n))
                for x, codes, scale in ((keys, state["k"], state["k_scale"]), (state["v_in"].double().reshape(T, K, D), state["v"], state["v_scale"])):
                    p = table[s][page]
                    large = x[at].abs().amax((0, 2))
                    need = torch.ceil(torch.log2((large / TOP[case["type"]]).clamp(min=2.0 ** -100))).exp2()
                    was = scale[p].double()
                    now = need if lo == page * P else torch.maximum(was, need)
                    kept = codes[p, :, :lo - page * P]
                    kept.copy_(encode((decode(kept.contiguous(), case["type"]).double() * (was / now)[:, None, None]).float(), case["type"]))
                    codes[p, :, lo - page * P:hi - page * P] = encode((x[at] / now[None, :, None]).float(), case["type"]).transpose(0, 1)
                    scale[p] = now.float()
            row += n
        # which code a rotated key next to a border gets is not a matter of precision: keys have no exact codes
        v = decode(state["v"], case["type"]).double() * (1.0 if case["type"] == "fp8" else state["v_scale"].double()[:, :, None, None])
        return turned(state["q_in"], case["heads"]).reshape(T, -1), None, v, state["k_scale"].double(), state["v_scale"].double()
    out, row, table = torch.empty(sum(new), K, G, D, dtype=torch.float64, device="cuda"), 0, state["pages"].long()
    for s, (n, t) in enumerate(zip(new, total)):
        q = state["q"][row:row + n].double().view(n, K, G, D)
        own_pages = table[s, :-(-t // P)]
        slot, key = torch.arange(t - n, t, device="cuda")[:, None], torch.arange(t, device="cuda")[None]
        hidden = key > slot
        if case["window"]:
            hidden |= key <= slot - case["window"]
        for h in range(K):
            k, v = ((decode(c[own_pages, h], case["type"]).double() * x[own_pages, h].double()[:, None, None]).reshape(-1, D)[:t]
                    for c, x in ((state["k"], state["k_scale"]), (state["v"], state["v_scale"])))
            score = torch.einsum("ngd,td->gnt", q[:, h], k).mul_(state["scale"]).masked_fill_(hidden, -math.inf)
            out[row:row + n, h] = torch.einsum("gnt,td->ngd", torch.softmax(score, -1), v)
        row += n
    return out.reshape(sum(new), -1)
