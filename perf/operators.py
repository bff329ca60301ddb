"""The packed key/value cache's operators, measured: rows written to a cache of
4-bit codes and read back, attention over such a cache, and attention through a
sliding window that keeps a few first positions in sight.

The cache holds, for each (slot, key/value head, position), `size` 4-bit codes
(two a byte, low nibble first) and one f16 scale for each 32 columns; a value
is (code - 8) * scale.  Row i of sequence s stands at position fill[s] + i of
its slot and sees the positions j <= fill[s] + i, with a window only those
with j > fill[s] + i - window or j < sinks.

`run` computes a case in its plain form with torch operations, or with the
framework's operators where `own` is true.
"""

import math
import random

import torch

own = False

GROUP = 32         # columns that share a scale
TILE = 64          # a cache holds a whole number of these positions a slot
SCALE_MOST = 8188.0  # largest scale: 8 of it is still an f16
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
BYTES = {"float32": 4, "float16": 2, "bfloat16": 2}


def _case(name, op, type, seqs, rows, depth, heads, kv, size, window=0, sinks=0, ragged=0):
    return {"name": name, "op": op, "type": type, "seqs": seqs, "rows": rows, "depth": depth, "heads": heads,
            "kv": kv, "size": size, "window": window, "sinks": sinks, "ragged": ragged}


def listed():
    return [
        # one session's step: a single token's rows written, then read back
        _case("store 1x1", "store", "float32", 1, 1, 1024, 8, 1, 256),
        # a round of 64 sessions' 4-lane blocks at their own positions
        _case("store 64x4", "store", "float32", 64, 4, 8192, 8, 1, 256, ragged=1),
        # prompts of several sequences in 16 bits, several key/value heads
        _case("store prompts", "store", "bfloat16", 6, 16384, 0, 32, 8, 128, ragged=2),
        # a long cache turned back into 16-bit rows, as for another engine
        _case("read 32768", "read", "float16", 1, 32768, 0, 8, 1, 256),
        # one session's decode step on a global layer after a 1024-id prompt
        _case("attend 1x1 at 1024", "attend", "float32", 1, 1, 1024, 8, 1, 256),
        # 64 sessions' 4-lane blocks, each at its own depth
        _case("attend 64x4", "attend", "bfloat16", 64, 4, 8192, 8, 1, 256, ragged=3),
        # one long stream's decode step, four query heads a key/value head
        _case("attend 1x1 at 131071", "attend", "bfloat16", 1, 1, 131071, 32, 8, 128),
        # a batch of whole prompts
        _case("attend prompts", "attend", "bfloat16", 3, 4096, 0, 8, 1, 256, ragged=4),
        # a prime chunk behind a long prompt, 512-wide heads
        _case("attend chunk 512 wide", "attend", "float16", 1, 512, 8192, 8, 1, 512),
        # many streams' single tokens on a sliding layer, far past its window
        _case("window 64x1", "attend", "bfloat16", 64, 1, 32000, 8, 1, 256, 512, 4, 5),
        # a whole long prompt on a sliding layer
        _case("window prompt 8192", "attend", "bfloat16", 1, 8192, 0, 8, 1, 256, 512, 4),
        # a session's prime chunk on a sliding layer, 32-bit rows
        _case("window chunk", "attend", "float32", 1, 511, 1537, 8, 1, 256, 512, 4),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    while True:
        op = rng.choice(["store", "read", "attend", "attend", "attend", "attend"])
        kv = rng.choice([1, 1, 2, 3, 4, 8])
        group = rng.choice([1, 2, 4, 5, 7, 8, 8, 16])
        case = {"op": op, "type": rng.choice(["float32", "float16", "bfloat16", "bfloat16"]), "kv": kv,
                "heads": kv * group, "size": rng.choice([32, 64, 96, 128, 128, 160, 256, 256, 320, 512]),
                "window": 0, "sinks": 0, "ragged": rng.randrange(1, 1000)}
        if op != "attend":
            case |= {"seqs": _log(rng, 1, 64), "rows": _log(rng, 1, 16384), "depth": rng.choice([0, _log(rng, 1, 8192)])}
        elif rng.random() < 0.5:  # single tokens and blocks
            case |= {"seqs": _log(rng, 1, 128), "rows": rng.choice([1, 1, 2, 4, 8, 16]), "depth": _log(rng, 1, 65536)}
        else:  # prompts and chunks
            case |= {"seqs": _log(rng, 1, 8), "rows": _log(rng, 17, 8192), "depth": rng.choice([0, _log(rng, 1, 16384)])}
        if op == "attend" and rng.random() < 0.4:
            case |= {"window": _log(rng, 1, 4096), "sinks": rng.choice([0, 1, 4, 4, 16, 100])}
        w = work(case)
        positions = case["seqs"] * kv * (case["depth"] + case["rows"])
        pairs = case["seqs"] * case["heads"] * case["rows"] * (case["depth"] + case["rows"])
        # no more than the largest listed case's work, nor more than the plain form's memory allows
        if w["bytes"] <= 1.5e8 and w["flops"] <= 1.3e11 and positions * case["size"] <= 3.0e8 and \
                (op != "attend" or pairs <= 6.0e8):
            return case


def _lengths(case):
    """Rows and first positions of each sequence; the first sequence has the most of both."""
    r = random.Random(case["ragged"])
    part = lambda most, least: most if not case["ragged"] else max(least, int(most * r.uniform(0.1, 1.0)))  # noqa: E731
    block = case["rows"] <= 16  # blocks have one length, prompts their own
    rows = [case["rows"] if s == 0 or block else part(case["rows"], 1) for s in range(case["seqs"])]
    fill = [case["depth"] if s == 0 else part(case["depth"], 0) for s in range(case["seqs"])]
    return rows, fill


def _sight(case, rows, fill):
    """(query row, position) pairs in sight, and the positions that any row sees, of one sequence."""
    if not case["window"]:
        return rows * fill + rows * (rows + 1) // 2, fill + rows
    w, sinks = case["window"], case["sinks"]
    pairs = 0
    for p in range(fill, fill + rows):
        low = max(0, p - w + 1)
        pairs += p + 1 - low + min(sinks, low)
    low = max(0, fill - w + 1)
    return pairs, fill + rows - low + min(sinks, low)


def work(case):
    rows, fill = _lengths(case)
    size, kv, heads, wide = case["size"], case["kv"], case["heads"], BYTES[case["type"]]
    packed = kv * (size // 2 + size // GROUP * 2) * 2  # key and value bytes of one position
    total = sum(rows)
    if case["op"] == "store":
        # rows in, codes out, codes in, rows out
        return {"bytes": total * (2 * packed + 4 * kv * size * wide), "flops": total * kv * size * 2 * 4}
    if case["op"] == "read":
        return {"bytes": total * (packed + 2 * kv * size * wide), "flops": total * kv * size * 2 * 2}
    seen = [_sight(case, n, f) for n, f in zip(rows, fill)]
    return {"bytes": sum(s for _, s in seen) * packed + 2 * total * heads * size * wide,
            "flops": 4 * size * heads * sum(p for p, _ in seen)}


def _pack(x):
    """Rows of 32-bit values to (codes two a byte, f16 scales)."""
    g = x.unflatten(-1, (-1, GROUP))
    scale = torch.clamp(g.abs().amax(-1) / 7.0, max=SCALE_MOST).to(torch.float16)
    step = scale.to(torch.float32).unsqueeze(-1)
    code = torch.clamp(torch.round(g / torch.where(step > 0, step, 1.0)), -8, 7)
    code = (torch.where(step > 0, code, 0.0) + 8).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def _unpack(codes, scales):
    """(codes, scales) to 32-bit rows."""
    n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).to(torch.float32) - 8.0
    return (n.unflatten(-1, (-1, GROUP)) * scales.to(torch.float32).unsqueeze(-1)).flatten(-2)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    rows, fill = _lengths(case)
    seqs, kv, size, total = case["seqs"], case["kv"], case["size"], sum(rows)
    positions = -(-(case["depth"] + case["rows"]) // TILE) * TILE
    kind = TYPES[case["type"]]
    # a few columns of a head run larger than the others, as keys' do after their norm and turn
    gain = torch.exp(0.5 * torch.randn(2, kv, 1, size, generator=g, device=dev))

    def side(which):
        codes = torch.empty(seqs, kv, positions, size // 2, dtype=torch.uint8, device=dev)
        scales = torch.empty(seqs, kv, positions, size // GROUP, dtype=torch.float16, device=dev)
        step = max(1, (1 << 26) // (kv * positions * size))
        for s in range(0, seqs, step):
            n = min(step, seqs - s)
            codes[s:s + n], scales[s:s + n] = _pack(
                torch.randn(n, kv, positions, size, generator=g, device=dev) * gain[which])
        return codes, scales

    state = {"op": case["op"], "rows_most": max(rows), "depth_most": case["depth"] + case["rows"],
             "window": case["window"], "sinks": case["sinks"], "scale": size ** -0.5, "kind": kind, "total": total}
    state["key_codes"], state["key_scales"] = side(0)
    state["value_codes"], state["value_scales"] = side(1)
    starts = [sum(rows[:s]) for s in range(seqs + 1)]
    state["starts"] = torch.tensor(starts, dtype=torch.int32, device=dev)
    state["fill"] = torch.tensor(fill, dtype=torch.int32, device=dev)
    # a server's sequences are in any of its slots
    state["slots"] = torch.randperm(seqs, generator=g, device=dev).to(torch.int32)
    if case["op"] == "attend":
        state["queries"] = torch.randn(total, case["heads"], size, generator=g, device=dev).to(kind)
    if case["op"] == "store":
        state["keys"] = (torch.randn(total, kv, size, generator=g, device=dev) * gain[0].transpose(0, 1)).to(kind)
        state["values"] = (torch.randn(total, kv, size, generator=g, device=dev) * gain[1].transpose(0, 1)).to(kind)
    return state


def _places(state):
    """Each row's sequence, its place in the sequence, its slot and its position."""
    starts, row = state["starts"].long(), torch.arange(state["total"], device=state["starts"].device)
    seq = torch.searchsorted(starts, row, right=True) - 1
    place = row - starts[seq]
    return seq, place, state["slots"].long()[seq], state["fill"].long()[seq] + place


def _plain_attend(state):
    dev = state["starts"].device
    starts, fill, slots = state["starts"].long(), state["fill"].long(), state["slots"].long()
    seqs, most, window, sinks = len(fill), state["rows_most"], state["window"], state["sinks"]
    kv, size = state["key_codes"].shape[1], state["queries"].shape[2]
    heads = state["queries"].shape[1]
    # the positions that matter: all of them, or the first few and those the window can reach
    if window and sinks + window + most - 1 < state["depth_most"]:
        near = (fill - window + 1).unsqueeze(1) + torch.arange(window + most - 1, device=dev)
        first = torch.arange(sinks, device=dev).expand(seqs, -1)
        place = torch.cat((first, torch.where(near >= sinks, near, -1)), 1)
    else:
        place = torch.arange(state["depth_most"], device=dev).expand(seqs, -1)
    at = place.clamp(min=0, max=state["key_codes"].shape[2] - 1)
    pick = (slots.view(-1, 1, 1), torch.arange(kv, device=dev).view(1, -1, 1), at.unsqueeze(1))
    keys = _unpack(state["key_codes"][pick], state["key_scales"][pick])
    values = _unpack(state["value_codes"][pick], state["value_scales"][pick])
    i = torch.arange(most, device=dev)
    row = (starts[:-1].unsqueeze(1) + i).clamp(max=state["total"] - 1)
    q = state["queries"].to(torch.float32)[row].unflatten(2, (kv, heads // kv))  # seq, row, kv, head, size
    q = q.permute(0, 2, 3, 1, 4).flatten(2, 3)
    score = torch.matmul(q, keys.transpose(2, 3)).unflatten(2, (heads // kv, most)) * state["scale"]
    p = (fill.unsqueeze(1) + i).unsqueeze(2)  # seq, row, 1
    j = place.unsqueeze(1)                    # seq, 1, position
    see = (j >= 0) & (j <= p)
    if window:
        see &= (j > p - window) | (j < sinks)
    score = score.masked_fill(~see.unsqueeze(1).unsqueeze(1), -math.inf)
    e = torch.exp(score - score.amax(-1, keepdim=True))
    out = torch.matmul(e.flatten(2, 3), values) / e.sum(-1).flatten(2, 3).unsqueeze(-1)
    out = out.unflatten(2, (heads // kv, most)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    seq, place, _, _ = _places(state)
    return out[seq, place].to(state["kind"])


def _plain_read(state):
    _, _, slot, position = _places(state)
    return (_unpack(state["key_codes"][slot, :, position], state["key_scales"][slot, :, position]).to(state["kind"]),
            _unpack(state["value_codes"][slot, :, position], state["value_scales"][slot, :, position]).to(state["kind"]))


def _plain_write(state):
    _, _, slot, position = _places(state)
    for side, rows in (("key", state["keys"]), ("value", state["values"])):
        codes, scales = _pack(rows.to(torch.float32))
        state[side + "_codes"][slot, :, position] = codes
        state[side + "_scales"][slot, :, position] = scales


def _cache(state):
    if "cache" not in state:
        import igllm_b200 as ig
        state["cache"] = ig.PackCache(state["key_codes"], state["key_scales"], state["value_codes"],
                                      state["value_scales"])
    return state["cache"]


def run(state):
    if own:
        cache = _cache(state)
        where = {"starts": state["starts"], "slots": state["slots"], "rows_most": state["rows_most"]}
        if state["op"] == "attend":
            return cache.attend(state["queries"], state["fill"], window=state["window"], sinks=state["sinks"],
                                scale=state["scale"], **where)
        if state["op"] == "store":
            cache.write(state["keys"], state["values"], state["fill"], **where)
        return cache.read(state["fill"], state["total"], state["kind"], **where)
    if state["op"] == "attend":
        return _plain_attend(state)
    if state["op"] == "store":
        _plain_write(state)
    return _plain_read(state)


def _exact_values(codes, scales):
    wide = torch.empty(*codes.shape[:-1], codes.shape[-1] * 2, dtype=torch.float64, device=codes.device)
    wide[..., 0::2] = (codes % 16).double() - 8
    wide[..., 1::2] = torch.div(codes, 16, rounding_mode="floor").double() - 8
    return wide * scales.double().repeat_interleave(GROUP, -1)


def _exact_stored(x):
    """What each value becomes once stored, in 64 bits."""
    x = x.double()
    big = x.unflatten(-1, (-1, GROUP)).abs().max(-1).values
    scale = (big / 7).clamp(max=SCALE_MOST).to(torch.float16).double().repeat_interleave(GROUP, -1)
    return torch.where(scale > 0, (x / scale).round().clamp(-8, 7) * scale, 0.0)


def exact(case, seed):
    state = prepare(case, seed)
    rows, fill = _lengths(case)
    if case["op"] == "store":
        return _exact_stored(state["keys"]), _exact_stored(state["values"])
    kc, ks, vc, vs = (state[n] for n in ("key_codes", "key_scales", "value_codes", "value_scales"))
    slots = state["slots"].tolist()
    group = case["heads"] // case["kv"]
    if case["op"] == "read":
        keys, values = [], []
        for s, n in enumerate(rows):
            at = slice(fill[s], fill[s] + n)
            keys.append(_exact_values(kc[slots[s], :, at], ks[slots[s], :, at]).transpose(0, 1))
            values.append(_exact_values(vc[slots[s], :, at], vs[slots[s], :, at]).transpose(0, 1))
        return torch.cat(keys), torch.cat(values)
    out = torch.empty(sum(rows), case["heads"], case["size"], dtype=torch.float64, device=kc.device)
    first = 0
    for s, n in enumerate(rows):
        end = fill[s] + n
        j = torch.arange(end, device=kc.device)
        for h in range(case["kv"]):
            k = _exact_values(kc[slots[s], h, :end], ks[slots[s], h, :end])
            v = _exact_values(vc[slots[s], h, :end], vs[slots[s], h, :end])
            for a in range(0, n, 1024):
                b = min(n, a + 1024)
                p = fill[s] + torch.arange(a, b, device=kc.device)
                hide = j[None, :] > p[:, None]
                if case["window"]:
                    hide |= (j[None, :] <= p[:, None] - case["window"]) & (j[None, :] >= case["sinks"])
                for c in range(h * group, (h + 1) * group):
                    q = state["queries"][first + a:first + b, c].double()
                    weight = torch.softmax((q @ k.T * case["size"] ** -0.5).masked_fill(hide, -math.inf), -1)
                    out[first + a:first + b, c] = weight @ v
        first += n
    return out
