"""Cases of the decode-step operators and their plain forms.

The operators are the steps around the windowed cache that a model's decode or
prompt pass takes: rotary positions of queries and keys, attention with a
sliding window and always-visible first tokens, and the choice of the next
token.  ``listed`` and ``draw`` name sizes, ``prepare`` makes what a program
holds before the call, ``run`` is one call, ``exact`` the same from the
definition in 64 bits.
"""

import math

import numpy as np
import torch

own = False  # True: run() calls the framework; False: the plain forms below

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
BYTES = {"float32": 4, "float16": 2, "bfloat16": 2}
HEADS = ((32, 8), (16, 8), (14, 2), (8, 8), (8, 1), (28, 4), (64, 8))  # query heads, kv heads


# -- the cases ---------------------------------------------------------------------

def listed():
    return [
        # one decode step's queries and keys of a few rows: the smallest call, latency only
        rotary("rotary decode 4 rows", 4, 1, 32, 8, 64, 64, False, "bfloat16", "none"),
        # a prompt of a long-context model (frequencies blended for long contexts)
        rotary("rotary prompt 4x8192", 4, 8192, 32, 8, 128, 128, False, "bfloat16", "blend"),
        # neighbouring pairs, a quarter of the head left as it is, odd length, far positions
        rotary("rotary pairs part of head", 3, 1013, 14, 2, 96, 72, True, "float16", "linear"),
        # one token of one short conversation over a small window
        window("window decode 1 row", 1, 1, 2048, 32, 8, 64, 1000, 4, "float16", "right"),
        # the decode batch of the repository's benchmark, each row at a length of its own
        window("window decode 16 rows", 16, 1, 32768, 32, 8, 64, 4096, 4, "float16", "right"),
        # prompts of one length
        window("window prompt 4x8192", 4, 8192, 8192, 32, 8, 64, 1024, 4, "bfloat16", "none"),
        # a long prompt
        window("window prompt 1x32768", 1, 32768, 32768, 32, 8, 128, 4096, 4, "bfloat16", "none"),
        # left-padded prompts of odd lengths, seven query heads to a kv head
        window("window padded prompts", 5, 777, 777, 14, 2, 64, 100, 3, "float16", "left"),
        # 32-bit tensors of small heads, a chunk behind a cache
        window("window chunk 32 bits", 2, 300, 1111, 8, 2, 32, 257, 5, "float32", "right"),
        # one row's next token, the usual three cuts
        sample("sample 1 row", 1, 32000, "float32", 0.8, 50, 0.95, 0.0),
        # a served batch with one nucleus for all rows
        sample("sample 128 rows nucleus", 128, 128256, "bfloat16", 0.7, 0, 0.9, 0.0),
        # every row with settings of its own, an odd vocabulary
        sample("sample 33 rows mixed", 33, 50001, "float32", -1.0, -1, -1.0, -1.0),
    ]


def rotary(name, batch, tokens, q_heads, kv_heads, head_dim, rotary_dim, interleaved, dtype, scaling):
    return dict(name=name, op="rotary", batch=batch, tokens=tokens, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim,
                rotary_dim=rotary_dim, interleaved=interleaved, dtype=dtype, scaling=scaling)


def window(name, batch, tokens, slots, q_heads, kv_heads, head_dim, span, sinks, dtype, padding):
    return dict(name=name, op="window", batch=batch, tokens=tokens, slots=slots, q_heads=q_heads, kv_heads=kv_heads,
                head_dim=head_dim, span=span, sinks=sinks, dtype=dtype, padding=padding)


def sample(name, batch, vocabulary, dtype, temperature, top_k, top_p, min_p):
    """A setting of -1 stands for one value for each row."""
    return dict(name=name, op="sample", batch=batch, vocabulary=vocabulary, dtype=dtype, temperature=temperature, top_k=top_k,
                top_p=top_p, min_p=min_p)


def spread(rng, low, high):
    """A whole number, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    which = rng.choice(("rotary", "window decode", "window prompt", "window prompt", "sample", "sample"))
    q_heads, kv_heads = rng.choice(HEADS)
    if which == "rotary":
        batch = spread(rng, 1, 32)
        head_dim = rng.choice((32, 64, 80, 96, 128))
        tokens = spread(rng, 1, max(1, 4 * 8192 * 128 * 40 // (batch * head_dim * (q_heads + kv_heads))))
        case = rotary("", batch, min(tokens, 32768), q_heads, kv_heads, head_dim, rng.choice((head_dim, head_dim, head_dim // 2, head_dim // 4 * 2)),
                      rng.random() < 0.5, rng.choice(tuple(DTYPES)), rng.choice(("none", "linear", "blend")))
    elif which == "window decode":
        batch = spread(rng, 1, 64)
        head_dim = rng.choice((32, 64, 64, 128, 128))
        slots = spread(rng, 1, min(65536, 16 * 32768 * 64 * 8 // (batch * head_dim * kv_heads)))
        case = window("", batch, 1, slots, q_heads, kv_heads, head_dim, spread(rng, 1, 16384), rng.choice((0, 1, 4, 7, 64)),
                      rng.choice(("float16", "bfloat16", "bfloat16", "float32")), "right")
    elif which == "window prompt":
        dtype = rng.choice(("float16", "bfloat16", "bfloat16", "float32"))
        head_dim = rng.choice((64, 128)) if dtype != "float32" else rng.choice((16, 32, 64, 128))
        batch = spread(rng, 1, 8)
        most = 16384 if dtype != "float32" else 1500
        slots = spread(rng, 2, max(2, min(most, 32768 * 4 // batch)))
        padding = rng.choice(("none", "left", "right"))
        tokens = slots if padding != "right" or rng.random() < 0.5 else rng.randint(1, slots)
        case = window("", batch, tokens, slots, q_heads, kv_heads, head_dim, spread(rng, 1, 4096), rng.choice((0, 1, 4, 7, 130)),
                      dtype, padding)
    else:
        batch = spread(rng, 1, 64)
        case = sample("", batch, spread(rng, 100, 128256), rng.choice(tuple(DTYPES)), rng.choice((0.0, 0.5, 0.7, 1.0, 1.3, -1.0)),
                      rng.choice((0, 0, 1, 20, 50, 1000, -1)), rng.choice((1.0, 1.0, 0.95, 0.9, 0.5, -1.0)), rng.choice((0.0, 0.0, 0.05, 0.2, -1.0)))
    del case["name"]
    return case


# -- what a program has in hand --------------------------------------------------------

def frequencies(case):
    """The rotary angle of one position for each pair of channels, in float32."""
    half = case["rotary_dim"] // 2
    f = 1.0 / 500000.0 ** (np.arange(half, dtype=np.float64) / max(1, half))
    if case["scaling"] == "linear":
        f = f / 4.0
    elif case["scaling"] == "blend":  # short waves stay, long ones are stretched eightfold, those between are blended
        turns = 8192 * f / (2 * math.pi)
        keep = np.clip((turns - 1.0) / 3.0, 0.0, 1.0)
        f = f * (keep + (1.0 - keep) / 8.0)
    return torch.from_numpy(f.astype(np.float32)).cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32 if dtype == torch.float32 else dtype)

    if case["op"] == "rotary":
        dtype, B, T, D = DTYPES[case["dtype"]], case["batch"], case["tokens"], case["head_dim"]
        # a projection's output is [batch, tokens, heads, channels]; attention code sees it transposed
        q = normal(B, T, case["q_heads"], D, dtype=dtype).transpose(1, 2)
        k = normal(B, T, case["kv_heads"], D, dtype=dtype).transpose(1, 2)
        far = 8192 if case["scaling"] == "none" else 1000000
        first = torch.randint(0, far, (B, 1), generator=g, device="cuda")
        return dict(case=case, q=q, k=k, positions=first + torch.arange(T, device="cuda"), inv_freq=frequencies(case),
                    scale=1.0 if case["scaling"] == "none" else 1.0 + 0.1 * math.log(8.0))
    if case["op"] == "window":
        dtype, B, T, S, D = DTYPES[case["dtype"]], case["batch"], case["tokens"], case["slots"], case["head_dim"]
        q = normal(B, T, case["q_heads"], D, dtype=dtype).transpose(1, 2)
        k, v = (normal(B, case["kv_heads"], S, D, dtype=dtype) for _ in range(2))
        starts = ends = query_slots = None
        if case["padding"] == "left":  # every row ends in the last slot and begins somewhere
            starts = torch.randint(0, S, (B,), generator=g, device="cuda", dtype=torch.int32) // 2
        elif case["padding"] == "right":  # every row begins in slot 0 and ends somewhere
            least = max(1, S - (T if T > 1 else S) // 2)  # half the queries at least are no padding
            ends = torch.randint(least, S + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
            if T > 1:  # a prompt or a chunk: the queries' slots are the same for all rows
                query_slots = torch.full((B,), S - T, device="cuda", dtype=torch.int32)
        return dict(case=case, q=q, k=k, v=v, starts=starts, ends=ends, query_slots=query_slots, scaling=D ** -0.5)
    B, V = case["batch"], case["vocabulary"]
    # a model's logits: most of the vocabulary in a wide bell, a few hundred candidates above it, rows of unlike sharpness
    x = torch.randn(B, V, generator=g, device="cuda") * 2.0
    lift = torch.rand(B, 1, generator=g, device="cuda") * 6.0
    few = max(1, min(V, 300))
    at = torch.randint(0, V, (B, few), generator=g, device="cuda")
    x.scatter_add_(1, at, lift + 3.0 * torch.rand(B, few, generator=g, device="cuda"))
    state = dict(case=case, logits=x.to(DTYPES[case["dtype"]]), uniform=torch.rand(B, generator=g, device="cuda"))

    def choices(setting, values, dtype):
        if setting != -1:
            return setting
        at = torch.randint(0, len(values), (B,), generator=g, device="cuda")
        return torch.tensor(values, device="cuda", dtype=dtype)[at]

    state["temperature"] = choices(case["temperature"], (0.0, 0.3, 0.7, 1.0, 1.5), torch.float32)
    state["top_k"] = choices(case["top_k"], (0, 1, 7, 50, 400, 5000), torch.int32)
    state["top_p"] = choices(case["top_p"], (1.0, 0.99, 0.9, 0.6), torch.float32)
    state["min_p"] = choices(case["min_p"], (0.0, 0.02, 0.1), torch.float32)
    return state


# -- one pass ----------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        import stickykv_b200 as skv
        if op == "rotary":
            return skv.apply_rotary(state["q"], state["k"], state["positions"], state["inv_freq"],
                                    interleaved=state["case"]["interleaved"], scale=state["scale"])
        if op == "window":
            return skv.sink_window_attention(state["q"], state["k"], state["v"], window=state["case"]["span"],
                                             sinks=state["case"]["sinks"], scaling=state["scaling"], starts=state["starts"],
                                             ends=state["ends"], query_slots=state["query_slots"])
        return skv.sample_tokens(state["logits"], state["uniform"], temperature=state["temperature"], top_k=state["top_k"],
                                 top_p=state["top_p"], min_p=state["min_p"])
    if op == "rotary":
        return plain_rotary(state)
    if op == "window":
        return plain_window(state)
    return plain_sample(state)


def plain_rotary(s):
    c = s["case"]
    angle = s["positions"].double()[:, None, :, None] * s["inv_freq"].double()
    cos, sin = (angle.cos() * s["scale"]).float(), (angle.sin() * s["scale"]).float()
    r, h = c["rotary_dim"], c["rotary_dim"] // 2
    outs = []
    for x in (s["q"], s["k"]):
        y = x.float()
        if c["interleaved"]:
            a, b = y[..., 0:r:2], y[..., 1:r:2]
            turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = y[..., :h], y[..., h:r]
            turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        outs.append(torch.cat((turned, y[..., r:]), -1).to(x.dtype))
    return tuple(outs)


def plain_window(s):
    c = s["case"]
    q, k, v = s["q"], s["k"].float(), s["v"].float()
    B, Hq, T, D = q.shape
    Hkv, S = k.shape[1], k.shape[2]
    w, n = c["span"], c["sinks"]
    dev = q.device
    zero = torch.zeros(B, dtype=torch.int64, device=dev)
    start = zero if s["starts"] is None else s["starts"].long()
    end = zero + S if s["ends"] is None else s["ends"].long()
    first = end - T if s["query_slots"] is None else s["query_slots"].long()
    shared = T > 1  # the queries' slots are then the same for all rows: first = S - T
    slot = torch.arange(S, device=dev)
    live = ((slot >= start[:, None]) & (slot < end[:, None]))[:, None, :, None]
    k, v = k.masked_fill(~live, 0.0), v.masked_fill(~live, 0.0)
    at = start[:, None] + torch.arange(n, device=dev)
    pick = at.clamp(max=S - 1)[:, None, :, None].expand(B, Hkv, n, D)
    k_sink, v_sink = k.gather(2, pick), v.gather(2, pick)
    step = max(1, min(512, T))
    parts = []
    for i in range(0, T, step):
        m = min(step, T - i)
        low, high = (max(0, S - T + i - w + 1), S - T + i + m) if shared else (0, S)
        p = (first[:, None] + torch.arange(i, i + m, device=dev))[:, None, None, :, None]
        j = torch.cat((at, slot[low:high].expand(B, -1)), 1)[:, None, None, None, :]
        st, en = start[:, None, None, None, None], end[:, None, None, None, None]
        seen = (j >= st) & (j <= p) & (p < en) & ((j - st < n) | (p - j < w))
        seen = seen & torch.cat((at < low, (slot[low:high] >= 0).expand(B, -1)), 1)[:, None, None, None, :]  # a first token inside the band counts once
        kk, vv = torch.cat((k_sink, k[:, :, low:high]), 2), torch.cat((v_sink, v[:, :, low:high]), 2)
        qq = q[:, :, i:i + m].float().reshape(B, Hkv, Hq // Hkv * m, D)
        score = (qq @ kk.transpose(2, 3)).view(B, Hkv, Hq // Hkv, m, -1) * s["scaling"]
        score = score.masked_fill(~seen, -math.inf)
        top = score.amax(-1, keepdim=True)
        e = torch.exp(score - top.masked_fill(top == -math.inf, 0.0))
        total = e.sum(-1, keepdim=True)
        e = e / total.masked_fill(total == 0.0, 1.0)
        o = e.view(B, Hkv, Hq // Hkv * m, -1) @ vv
        parts.append(o.view(B, Hq, m, D).transpose(1, 2).to(q.dtype))
    return torch.cat(parts, 1)


def plain_sample(s):
    x = s["logits"].double()
    x = x.masked_fill(x.isnan(), -math.inf)
    B, V = x.shape

    def each(setting, dtype):
        if torch.is_tensor(setting):
            return setting.to(dtype)[:, None]
        return torch.full((B, 1), setting, dtype=torch.float32, device=x.device).to(dtype)

    heat, k = each(s["temperature"], torch.float64), each(s["top_k"], torch.float64)
    p, floor = each(s["top_p"], torch.float64), each(s["min_p"], torch.float64)
    value, token = torch.sort(x, dim=1, descending=True, stable=True)
    top = value[:, :1]
    fall = torch.where(value == top, torch.zeros_like(value), value - top)
    weight = torch.exp(fall / torch.where(heat > 0, heat, torch.ones_like(heat)))
    rank = torch.arange(V, device=x.device)
    keep = (rank < torch.where(k > 0, k, k + V)) & ((heat > 0) | (rank < 1))
    weight = torch.where(keep, weight, torch.zeros_like(weight))
    before = weight.cumsum(1) - weight
    keep = keep & ((p >= 1) | (before < p * weight.sum(1, keepdim=True)) | (rank < 1)) & (weight >= floor)
    weight = torch.where(keep, weight, torch.zeros_like(weight))
    weight = torch.zeros_like(weight).scatter(1, token, weight)  # back into the vocabulary's order
    total = weight.cumsum(1)
    passed = (total > s["uniform"].double()[:, None] * total[:, -1:]) & (weight > 0)
    last = V - 1 - (weight > 0).flip(1).double().argmax(1)
    chosen = torch.where(passed.any(1), passed.double().argmax(1), last)
    return torch.where(top[:, 0] == -math.inf, torch.full_like(chosen, -1), chosen)


# -- what one pass cannot do without -------------------------------------------------------

def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "rotary":
        values = case["batch"] * case["tokens"] * (case["q_heads"] + case["kv_heads"]) * case["head_dim"]
        return {"bytes": 2 * values * e + 8 * case["batch"] * case["tokens"] + 2 * case["rotary_dim"], "flops": 3 * values}
    if case["op"] == "window":
        B, T, S, D = case["batch"], case["tokens"], case["slots"], case["head_dim"]
        w, n = case["span"], case["sinks"]
        # rows that are padded hold three quarters of the queries or, before one token, of the slots on average
        rows = 1.0 if case["padding"] == "none" else 0.75
        p = np.arange(S - T, S, dtype=np.float64) if T > 1 else np.array([rows * S - 1])
        pairs = float((np.minimum(p + 1, w) + np.clip(p + 1 - w, 0, n)).sum()) * (rows if T > 1 else 1.0)
        keys = min(S * rows, max(n + w + T - 1, 1))
        return {"bytes": e * B * D * (2 * case["kv_heads"] * keys + 2 * case["q_heads"] * T), "flops": 4.0 * B * case["q_heads"] * D * pairs}
    return {"bytes": case["batch"] * (case["vocabulary"] * e + 12), "flops": 2 * case["batch"] * case["vocabulary"]}


# -- the same from the definition, in 64 bits -------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return tuple(exact_rotary(case, s, x) for x in (s["q"], s["k"]))
    if case["op"] == "window":
        return exact_window(case, s)
    return exact_sample(case, s)


def exact_rotary(case, s, x):
    """Every pair of channels as one complex number, turned by its angle."""
    half = case["rotary_dim"] // 2
    index = torch.arange(case["rotary_dim"], device=x.device)
    first, second = (index[0::2], index[1::2]) if case["interleaved"] else (index[:half], index[half:])
    out = x.double().clone()
    turn = torch.polar(torch.full((), s["scale"], dtype=torch.float64, device=x.device).expand(x.shape[0], 1, x.shape[2], half).contiguous(),
                       (s["positions"].double().unsqueeze(-1) * s["inv_freq"].double()).unsqueeze(1))
    z = torch.complex(out[..., first], out[..., second]) * turn
    out[..., first], out[..., second] = z.real, z.imag
    return out


def exact_window(case, s):
    """Row by row and head by head, a block of queries against all slots at once."""
    q, k, v = s["q"], s["k"], s["v"]
    B, Hq, T, D = q.shape
    S, group = k.shape[2], Hq // k.shape[1]
    if B * Hq * T * S * D > 6e13:
        return None
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64, device=q.device)
    j = torch.arange(S, device=q.device)
    for b in range(B):
        start = 0 if s["starts"] is None else int(s["starts"][b])
        end = S if s["ends"] is None else int(s["ends"][b])
        first = end - T if s["query_slots"] is None else int(s["query_slots"][b])
        for h in range(k.shape[1]):
            keys, values = k[b, h, start:end].double(), v[b, h, start:end].double()
            slots = j[start:end]
            for i in range(0, T, 1024):
                p = first + torch.arange(i, min(T, i + 1024), device=q.device)
                sees = (slots[None] <= p[:, None]) & (p[:, None] < end) & ((slots[None] < start + case["sinks"]) | (slots[None] > p[:, None] - case["span"]))
                some = sees.any(1)
                if keys.shape[0] == 0:
                    continue
                for h2 in range(h * group, (h + 1) * group):
                    a = q[b, h2, i:i + 1024].double() @ keys.T * s["scaling"]
                    a = torch.where(sees, a, torch.full_like(a, -1e300))
                    o = torch.softmax(a, 1) @ values
                    out[b, i:i + 1024, h2] = torch.where(some[:, None], o, torch.zeros_like(o))
    return out


def exact_sample(case, s):
    x = s["logits"].double().cpu().numpy()
    u = s["uniform"].double().cpu().numpy()

    def each(setting):
        return setting.double().cpu().numpy() if torch.is_tensor(setting) else np.full(x.shape[0], np.float32(setting), dtype=np.float64)

    chosen = []
    for row, r, heat, k, p, floor in zip(x, u, each(s["temperature"]), each(s["top_k"]), each(s["top_p"]), each(s["min_p"])):
        order = np.argsort(-row, kind="stable")  # the largest first, of equal ones the lowest index
        if heat <= 0:
            chosen.append(int(order[0]))
            continue
        if k > 0:
            order = order[:int(k)]
        weight = np.exp((row[order] - row[order[0]]) / heat)
        if p < 1:
            order = order[:int(np.searchsorted(np.cumsum(weight), p * weight.sum(), side="left")) + 1]
            weight = weight[:len(order)]
        order = np.sort(order[weight >= floor])
        total = np.cumsum(np.exp((row[order] - row.max()) / heat))
        chosen.append(int(order[min(len(order) - 1, int(np.searchsorted(total, r * total[-1], side="right")))]))
    return torch.tensor(chosen, device="cuda")
