"""Workloads of the 4-bit K/V cache operators: writing it, reading it back, and attending over it.

The cache holds pages of 64 tokens.  Per page and K/V head it has one record of 9216 bytes:
K codes [64][64 B], V codes [64][64 B], K scales [64][4] bf16, V scales [64][4] bf16.  A
group of 32 channels shares a scale s, the smallest number of five significant bits that is
at least max|x| / 7; a code is rint(x / s) in -7..7, held as code + 8 in a nibble.
"""
import math
import types

import numpy as np
import torch

own = False

D = 128        # head size
PAGE = 64      # tokens of a page
GROUP = 32     # channels that share a scale
RECORD = 9216  # bytes of one page of one K/V head
EPS = 1e-6


# ------------------------------------------------------------------------------- cases

def _case(name, kind, hq, hk, rows, ctx, window=0, sinks=0):
    """rows, ctx: "newest rows" and "tokens in the cache with them" of each sequence, as
    "n*count" terms joined by "+", so that a case stays a dict of plain values."""
    return {"name": name, "kind": kind, "hq": hq, "hk": hk, "rows": rows, "ctx": ctx, "window": window, "sinks": sinks}


def listed():
    return [
        # one token of one answer, 4B heads, right after a 320-token prefill: latency alone
        _case("write_one_token", "write", 32, 8, "1*1", "321*1"),
        # the prefix of one request (256 visual rows + 64 of text) put into the cache
        _case("write_prefix_320", "write", 32, 8, "320*1", "320*1"),
        # four long documents of images, 32B heads, ragged
        _case("write_four_long", "write", 64, 8, "2048*2+1999*1+1033*1", "2048*2+1999*1+4105*1"),
        # one token of one answer over a 320-token prefix: latency alone
        _case("decode_one_short", "attend", 32, 8, "1*1", "321*1"),
        # one answer over a very long context: the cache's bytes over all the machine
        _case("decode_one_long", "attend", 32, 8, "1*1", "131001*1"),
        # a full serving batch, ragged contexts
        _case("decode_batch_64", "attend", 32, 8, "1*64", "8192*16+5000*16+2049*16+777*16"),
        # 32B heads (eight queries to a K/V head)
        _case("decode_batch_32B", "attend", 64, 8, "1*16", "4096*8+3333*8"),
        # long streams that keep their first four tokens and a window of 4096
        _case("decode_window", "attend", 32, 8, "1*16", "30000*8+16384*8", 4096, 4),
        # a new question of 64 text rows over a cached image prefix
        _case("question_64_rows", "attend", 32, 8, "64*1", "2112*1"),
        # four requests go on by 512 rows over 8192 tokens, 32B heads
        _case("chunk_512_rows", "attend", 64, 8, "512*4", "8704*4"),
        # a few draft tokens, long chunks and a short sequence in one call, with a window, 2B heads
        _case("chunk_window_ragged", "attend", 16, 8, "3*2+300*3+1*1", "1000*2+9001*3+17*1", 1024, 64),
        # a decoding step of a layer: new rows into the cache, then attention over it
        _case("step_batch_16", "step", 32, 8, "1*16", "2048*8+1023*8"),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    hq, hk = rng.choice([(32, 8), (64, 8), (16, 8), (8, 8), (12, 4), (5, 1), (48, 4)])
    kind = rng.choice(["write", "attend", "attend", "attend", "step"])
    if kind == "write":
        batch = log_int(1, 16)
        rows = [log_int(1, max(2, 8192 // batch)) for _ in range(batch)]
        ctx = [r + rng.choice([0, log_int(1, 4000)]) for r in rows]
    elif rng.random() < 0.6 or kind == "step":
        batch = log_int(1, 48)
        rows = [1] * batch
        top = max(2, min(100000, 260000 // batch))
        ctx = [log_int(1, top) for _ in range(batch)]
    else:
        batch = log_int(1, 6)
        rows = [log_int(1, 480) for _ in range(batch)]
        ctx = [r + log_int(1, 8000) for r in rows]
    window, sinks = (log_int(1, 8192), rng.choice([0, 1, 4, 64, 100])) if rng.random() < 0.3 and kind != "write" else (0, 0)
    case = _case("", kind, hq, hk, "+".join("%d*1" % r for r in rows), "+".join("%d*1" % c for c in ctx), window, sinks)
    del case["name"]
    return case


def _ints(text):
    return [int(term.split("*")[0]) for term in text.split("+") for _ in range(int(term.split("*")[1]))]


# ------------------------------------------------------------------------------- the format, in torch

def _quantize(x):
    """[..., 128] fp64 -> (codes [..., 128] int, scales [..., 4] fp64)."""
    g = x.unflatten(-1, (D // GROUP, GROUP))
    top = g.abs().amax(-1) / 7.0
    frac, power = torch.frexp(top)
    scale = torch.ldexp(torch.ceil(frac * 32.0) / 32.0, power)
    codes = torch.where(scale[..., None] > 0, torch.round(g / scale[..., None]), 0.0).clamp(-7, 7)
    return codes.flatten(-2).to(torch.int8), scale


def _bytes(codes, is_v):
    """Codes [..., 128] of one token -> its 64 bytes (V: before the token's chunk swap)."""
    n = (codes + 8).to(torch.uint8)
    if is_v:  # chunk c of 8 bytes: channels c, 8 + c, 16 + c, ...
        n = n.unflatten(-1, (16, 8)).transpose(-1, -2)
    else:     # chunk t of 16 bytes: channels 32 j + 8 t .. + 7 for j = 0..3
        n = n.unflatten(-1, (4, 4, 8)).transpose(-2, -3)
    n = n.reshape(*codes.shape[:-1], 64, 2)
    return n[..., 0] | (n[..., 1] << 4)


def _pages_of(k, v):
    """K, V [pages, heads, 64, 128] fp32 -> records [pages, heads, 9216]."""
    (ck, sk), (cv, sv) = _quantize(k), _quantize(v)
    bv = _bytes(cv, True).unflatten(-1, (2, 32))
    swap = (torch.arange(PAGE, device=k.device) // 4 % 2 == 1)[:, None, None]
    bv = torch.where(swap, bv.flip(-2), bv)  # tokens 4..7 of eight hold their two halves the other way round
    lead = k.shape[:2]
    parts = [_bytes(ck, False).reshape(*lead, -1), bv.reshape(*lead, -1)]
    parts += [s.to(torch.bfloat16).contiguous().view(torch.uint8).reshape(*lead, -1) for s in (sk, sv)]
    return torch.cat(parts, -1)


def _half(pages, is_v):
    """Records [..., 9216] -> the K or V values [..., 64, 128] fp32 that they hold."""
    lead = pages.shape[:-1]
    raw = pages[..., 4096 * is_v:4096 * (is_v + 1)].reshape(*lead, PAGE, 64)
    if is_v:
        raw = raw.unflatten(-1, (2, 32))
        swap = (torch.arange(PAGE, device=pages.device) // 4 % 2 == 1)[:, None, None]
        raw = torch.where(swap, raw.flip(-2), raw).flatten(-2)
    n = torch.stack([raw & 15, raw >> 4], -1).flatten(-2)
    if is_v:
        n = n.unflatten(-1, (8, 16)).transpose(-1, -2).flatten(-2)
    else:
        n = n.unflatten(-1, (4, 4, 8)).transpose(-2, -3).flatten(-3)
    scale = pages[..., 8192 + 512 * is_v:8704 + 512 * is_v].contiguous().view(torch.bfloat16).reshape(*lead, PAGE, 4)
    return (n.float() - 8.0) * scale.float().repeat_interleave(GROUP, -1)


def _values(pages):
    return _half(pages, 0), _half(pages, 1)


# ------------------------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    hq, hk = case["hq"], case["hk"]
    rows, ctx = _ints(case["rows"]), _ints(case["ctx"])
    total, batch = sum(rows), len(rows)
    need = [-(-c // PAGE) for c in ctx]
    order = torch.randperm(sum(need) + 3, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(batch, max(need), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    # keys after norm and rotation have unit size with some strong channels; values are wider
    strong = 1.0 + 3.0 * (torch.rand(hk, 1, D, generator=g, device="cuda") > 0.95)
    pages = torch.empty(sum(need) + 3, hk, RECORD, dtype=torch.uint8, device="cuda")
    for p in range(0, pages.shape[0], 512):
        n = min(512, pages.shape[0] - p)
        k = torch.randn(n, hk, PAGE, D, generator=g, device="cuda") * strong
        v = torch.randn(n, hk, PAGE, D, generator=g, device="cuda") * 0.5
        pages[p:p + n] = _pages_of(k, v)
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    state = {
        "case": case, "pages": pages, "page_table": table, "scale": D ** -0.5, "max_rows": max(rows), "longest": max(ctx),
        "row_start": torch.tensor(starts, dtype=torch.int32, device="cuda"),
        "ctx_len": torch.tensor(ctx, dtype=torch.int32, device="cuda"),
    }
    if case["kind"] in ("write", "step"):
        state["qkv"] = torch.randn(total, (hq + 2 * hk) * D, generator=g, device="cuda").to(torch.bfloat16)
        for name in ("qn", "kn"):
            weight = (1.0 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(torch.bfloat16)
            state[name] = types.SimpleNamespace(weight=weight, variance_epsilon=EPS)
        spot = torch.cat([torch.arange(c - r, c) for r, c in zip(rows, ctx)]).double()
        angle = spot[:, None] * (5e6 ** -(torch.arange(64).double() / 64))[None, :]
        angle = torch.cat([angle, angle], -1)
        state["cos"], state["sin"] = (f(angle).to(torch.bfloat16).cuda() for f in (torch.cos, torch.sin))
    if case["kind"] == "attend":
        state["q"] = (torch.randn(hq, total, D, generator=g, device="cuda") * 1.5).to(torch.bfloat16)
    return state


# ------------------------------------------------------------------------------- the plain forms

def _rows_of(state, total):
    """Sequence and position in the context of each new row."""
    start = state["row_start"].long()
    t = torch.arange(total, device=start.device)
    seq = torch.searchsorted(start[1:], t, right=True)
    return seq, state["ctx_len"].long()[seq] - (start[seq + 1] - t)


def _plain_write(state):
    case, qkv = state["case"], state["qkv"]
    hq, hk, total = case["hq"], case["hk"], qkv.shape[0]
    x = qkv.view(total, hq + 2 * hk, D)
    cos, sin = state["cos"][:, None, :], state["sin"][:, None, :]

    def norm_and_turn(y, module, kind):
        y = y.to(kind)
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + module.variance_epsilon) * module.weight.to(kind)
        other = torch.cat([-y[..., 64:], y[..., :64]], -1)
        return y * cos.to(kind) + other * sin.to(kind)

    q = norm_and_turn(x[:, :hq], state["qn"], torch.float32).to(torch.bfloat16)
    # 64 bits: a key next to the border of two codes goes to the right one
    ck, sk = _quantize(norm_and_turn(x[:, hq:hq + hk], state["kn"], torch.float64))
    cv, sv = _quantize(x[:, hq + hk:].double())
    seq, spot = _rows_of(state, total)
    page = state["page_table"][seq, spot // PAGE].long()
    slot = spot % PAGE
    pages = state["pages"]
    head = torch.arange(hk, device=pages.device)[None, :, None]
    byte = torch.arange(64, device=pages.device)
    put = [(_bytes(ck, False), 64 * slot[:, None] + byte), (_bytes(cv, True), 4096 + 64 * slot[:, None] + (byte ^ (32 * (slot // 4 % 2))[:, None]))]
    put += [(s.to(torch.bfloat16).contiguous().view(torch.uint8), base + 8 * slot[:, None] + byte[:8]) for s, base in ((sk, 8192), (sv, 8704))]
    at = torch.cat([where for _, where in put], -1)[:, None, :]
    pages[page[:, None, None], head, at] = torch.cat([what for what, _ in put], -1)
    return q.transpose(0, 1).contiguous()


def _plain_read(state, total):
    seq, spot = _rows_of(state, total)
    k, v = _values(state["pages"][state["page_table"][seq, spot // PAGE].long()])  # [rows, heads, 64, 128]
    t = torch.arange(total, device=spot.device)
    return [y[t, :, spot % PAGE].transpose(0, 1).to(torch.bfloat16).contiguous() for y in (k, v)]


def _plain_attend(state, q):
    case = state["case"]
    hq, hk, total = case["hq"], case["hk"], q.shape[1]
    k, v = _values(state["pages"][state["page_table"].long()])  # [batch, pages, heads, 64, 128]
    k, v = (y.transpose(1, 2).flatten(2, 3) for y in (k, v))    # [batch, heads, tokens, 128]
    seq, spot = _rows_of(state, total)
    line = torch.arange(total, device=q.device) - state["row_start"].long()[seq]
    batch, rows = k.shape[0], state["max_rows"]
    wide = torch.zeros(batch, rows, hq, D, device=q.device)
    wide[seq, line] = q.transpose(0, 1).float()
    place = torch.full((batch, rows), -1, dtype=torch.long, device=q.device)
    place[seq, line] = spot
    wide = wide.view(batch, rows, hk, hq // hk, D).permute(0, 2, 3, 1, 4).flatten(2, 3)
    score = wide @ k.transpose(-1, -2) * state["scale"]
    key = torch.arange(k.shape[2], device=q.device)
    seen = key <= place[..., None]
    if case["window"]:
        seen &= (place[..., None] - key < case["window"]) | (key < case["sinks"])
    score.unflatten(2, (hq // hk, rows)).masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    weight = weight / weight.sum(-1, keepdim=True).clamp_min(1e-38)
    out = (weight @ v).unflatten(2, (hq // hk, rows)).permute(0, 3, 1, 2, 4).reshape(batch, rows, hq, D)
    return out[seq, line].to(torch.bfloat16)


def run(state):
    kind = state["case"]["kind"]
    if own:
        from fastforward_b200 import ops
        place = (state["page_table"], state["row_start"], state["ctx_len"])
    result = {}
    q = state.get("q")
    if kind in ("write", "step"):
        if own:
            q = ops.qk_pair_kv4(state["qkv"], state["qn"], state["kn"], state["cos"], state["sin"], state["pages"], *place)
            result["k"], result["v"] = ops.kv4_read(state["pages"], *place, q.shape[1])
        else:
            q = _plain_write(state)
            result["k"], result["v"] = _plain_read(state, q.shape[1])
        result["q"] = q
    if kind in ("attend", "step"):
        if own:
            case = state["case"]
            result["out"] = ops.attention_kv4(q, state["pages"], *place, state["scale"], window=case["window"],
                                              sinks=case["sinks"], max_rows=state["max_rows"])
        else:
            result["out"] = _plain_attend(state, q)
    return result


# ------------------------------------------------------------------------------- what a pass needs

def work(case):
    hq, hk = case["hq"], case["hk"]
    rows, ctx = _ints(case["rows"]), _ints(case["ctx"])
    total, moved, flops = sum(rows), 0, 0
    if case["kind"] in ("write", "step"):
        # qkv and the rotation in, queries and records out, and the new rows read back
        moved += total * ((hq + 2 * hk) * D * 2 + 2 * D * 2 + hq * D * 2 + hk * 144 + hk * (144 + 4 * D))
        flops += total * (hq + 2 * hk) * D * 8
    if case["kind"] in ("attend", "step"):
        window, sinks = case["window"], case["sinks"]
        pairs = keys = 0
        for r, c in zip(rows, ctx):
            if window:
                first = max(0, c - r - window + 1)
                keys += c - first + min(sinks, first)
                pairs += sum(min(p + 1, window) + min(sinks, max(0, p + 1 - window)) for p in range(c - r, c))
            else:
                keys += c
                pairs += r * (c - r) + r * (r + 1) // 2
        moved += keys * hk * 144 + total * hq * D * 4
        flops += pairs * hq * D * 4
    return {"bytes": moved, "flops": flops}


# ------------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    state = prepare(case, seed)
    hq, hk = case["hq"], case["hk"]
    rows, ctx = _ints(case["rows"]), _ints(case["ctx"])
    total = sum(rows)
    pairs = sum(r * c for r, c in zip(rows, ctx))
    if pairs * hq > 4e9:
        return None
    dev = state["pages"].device
    result = {}
    held = {}  # sequence -> newest K, V rows, as the cache holds them
    q64 = state["q"].double() if case["kind"] == "attend" else None
    starts = np.concatenate([[0], np.cumsum(rows)])
    if case["kind"] in ("write", "step"):
        x = state["qkv"].double().view(total, hq + 2 * hk, D).transpose(0, 1)
        turn_c, turn_s = state["cos"].double()[:, :64], state["sin"].double()[:, :64]

        def turned(y, module):
            y = y * torch.rsqrt(y.pow(2).sum(-1, keepdim=True) / D + module.variance_epsilon) * module.weight.double()
            a, b = y[..., :64], y[..., 64:]
            return torch.cat([a * turn_c - b * turn_s, b * turn_c + a * turn_s], -1)

        def held_as(y):
            parts = []
            for j in range(4):
                part = y[..., 32 * j:32 * j + 32]
                top = part.abs().max(-1, keepdim=True).values / 7
                power = torch.floor(torch.log2(top.clamp_min(1e-300))) - 4
                power = torch.where(torch.exp2(power + 5) <= top, power + 1, torch.where(torch.exp2(power + 4) > top, power - 1, power))
                s = torch.ceil(top / torch.exp2(power)) * torch.exp2(power)
                parts.append(torch.where(s > 0, torch.round(part / torch.where(s > 0, s, 1.0)), 0.0) * s)
            return torch.cat(parts, -1)

        q64 = turned(x[:hq], state["qn"])
        k64, v64 = held_as(turned(x[hq:hq + hk], state["kn"])), held_as(x[hq + hk:])
        result["k"], result["v"], result["q"] = k64, v64, q64
        for b in range(len(rows)):
            held[b] = (k64[:, starts[b]:starts[b + 1]], v64[:, starts[b]:starts[b + 1]])
        # the attention that follows takes the rounded queries
        q64 = q64.to(torch.bfloat16).double()
    if case["kind"] in ("attend", "step"):
        out = torch.zeros(total, hq, D, dtype=torch.float64, device=dev)
        digit = torch.arange(256, device=dev)
        look = torch.stack([digit % 16, digit // 16], -1).double() - 8.0
        for b, (r, c) in enumerate(zip(rows, ctx)):
            n = -(-c // PAGE)
            rec = state["pages"][state["page_table"][b, :n].long()].transpose(0, 1)  # [heads, pages, bytes]
            token = torch.arange(c, device=dev)
            chan = torch.arange(D, device=dev)
            kv = []
            for is_v in (0, 1):
                code = rec[..., 4096 * is_v:4096 * is_v + 4096].reshape(hk, n * PAGE, 64)[:, :c]
                if is_v:
                    chunk = (chan % 8)[None, :] ^ (4 * ((token // 4) % 2))[:, None]
                    byte, high = 8 * chunk + (chan // 8 // 2)[None, :], (chan // 8) % 2
                else:
                    byte = (16 * (chan % 32 // 8) + 4 * (chan // 32) + chan % 8 // 2)[None, :].expand(c, D)
                    high = chan % 2
                got = look[torch.gather(code, 2, byte[None].expand(hk, c, D)).long(), high[None, None, :].expand(hk, c, D)]
                s = rec[..., 8192 + 512 * is_v:8704 + 512 * is_v].contiguous().view(torch.bfloat16).reshape(hk, n * PAGE, 4)[:, :c]
                kv.append(got * s.double()[..., chan // 32])
            if b in held:
                kv[0][:, c - r:], kv[1][:, c - r:] = held[b]
            place = torch.arange(c - r, c, device=dev)[:, None]
            seen = token[None, :] <= place
            if case["window"]:
                seen = seen & ((place - token[None, :] < case["window"]) | (token[None, :] < case["sinks"]))
            for h in range(hq):
                score = q64[h, starts[b]:starts[b + 1]] @ kv[0][h // (hq // hk)].T * state["scale"]
                weight = torch.softmax(torch.where(seen, score, -math.inf), -1)
                out[starts[b]:starts[b + 1], h] = torch.where(seen.any(-1, keepdim=True), weight, 0.0) @ kv[1][h // (hq // hk)]
        result["out"] = out
    return result
