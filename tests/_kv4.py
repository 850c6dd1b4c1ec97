"""Plain formulas of the 4-bit K/V cache in 64 bits, on the CPU (test helper)."""
import math

import torch


def up5(x):
    """Smallest number of five significant bits >= x (x > 0)."""
    m, e = torch.frexp(x)
    return torch.ldexp(torch.ceil(m * 32), e - 5)


def quantize(x):
    """[..., 128] fp64 -> codes [..., 128], scales [..., 4]; values = code * scale."""
    groups = x.reshape(*x.shape[:-1], 4, 32)
    top = groups.abs().amax(-1)
    scale = torch.where(top > 0, up5(torch.where(top > 0, top, 1.0) / 7), 0.0)
    codes = torch.where(scale[..., None] > 0, torch.round(groups / torch.where(scale > 0, scale, 1.0)[..., None]), 0.0)
    assert codes.abs().max() <= 7
    return codes.reshape(x.shape), scale


def held(x):
    """What the cache holds of any x [..., 128] fp64: groups below 2^-100 as zeros, groups with a value
    that is not finite or reaches 2^127 as NaN."""
    top = x.abs().reshape(*x.shape[:-1], 4, 32).amax(-1).repeat_interleave(32, -1)  # a NaN stays one
    bad = ~(top < 2.0 ** 127)
    return values(*quantize(x.masked_fill(bad | (top < 2.0 ** -100), 0.0))).masked_fill(bad, float("nan"))


def values(codes, scale):
    return codes * scale.repeat_interleave(32, -1)


def _byte_index():
    """byte and shift of each channel's nibble: K, and V of tokens 0..3 of eight."""
    k = [(16 * (c % 32 // 8) + 4 * (c // 32) + c % 8 // 2, 4 * (c % 2)) for c in range(128)]
    v = [(8 * (c % 8) + c // 8 // 2, 4 * (c // 8 % 2)) for c in range(128)]
    return k, v


def pack_tokens(codes, scale, is_v, token):
    """Codes / scales [..., 128] / [..., 4] of tokens (index in the page) -> 64 bytes, 8 bytes."""
    out = torch.zeros(*codes.shape[:-1], 64, dtype=torch.int64)
    nib = (codes + 8).to(torch.int64)
    for c, (byte, shift) in enumerate(_byte_index()[1 if is_v else 0]):
        out[..., byte] |= nib[..., c] << shift
    if is_v:
        flipped = out.reshape(*out.shape[:-1], 2, 32).flip(-2).reshape(out.shape)
        out = torch.where((token % 8 >= 4)[..., None].expand(out.shape), flipped, out)
    return out.to(torch.uint8), scale.to(torch.bfloat16).contiguous().view(torch.uint8)


def pack(k, v):
    """K, V [pages, heads, 64, 128] -> records [pages, heads, 9216]."""
    token = torch.arange(64).expand(k.shape[:-1])
    parts, scales = [], []
    for is_v, x in enumerate((k, v)):
        b, s = pack_tokens(*quantize(x), is_v, token)
        parts.append(b.flatten(-2))
        scales.append(s.flatten(-2))
    return torch.cat(parts + scales, -1)


def unpack(pages):
    """Records -> K, V [pages, heads, 64, 128] fp64."""
    out = []
    for is_v in (0, 1):
        raw = pages[..., 4096 * is_v:4096 * is_v + 4096].reshape(*pages.shape[:-1], 64, 64).to(torch.int64)
        if is_v:
            flipped = raw.reshape(*raw.shape[:-1], 2, 32).flip(-2).reshape(raw.shape)
            raw = torch.where((torch.arange(64) % 8 >= 4)[:, None], flipped, raw)
        x = torch.stack([(raw[..., byte] >> shift) & 15 for byte, shift in _byte_index()[is_v]], -1).double() - 8
        s = pages[..., 8192 + 512 * is_v:8704 + 512 * is_v].contiguous().view(torch.bfloat16)
        out.append(values(x, s.reshape(*pages.shape[:-1], 64, 4).double()))
    return out


def poison(pages, table, lens):
    """Scales of every token that no sequence holds become NaN."""
    held = torch.zeros(pages.shape[0], 64, dtype=torch.bool)
    for b, n in enumerate(lens.tolist()):
        for j in range(n):
            held[table[b, j // 64], j % 64] = True
    sc = pages[..., 8192:].contiguous().view(torch.bfloat16).reshape(*pages.shape[:-1], 2, 64, 4).clone()
    sc[(~held)[:, None, None, :, None].expand(sc.shape)] = float("nan")
    out = pages.clone()
    out[..., 8192:] = sc.reshape(*pages.shape[:-1], 512).view(torch.uint8)
    return out


def _heads(qkv, hq, hk):
    return qkv.double().reshape(qkv.shape[0], hq + 2 * hk, 128).transpose(0, 1)


def norm_rotate(x, module, cos, sin):
    n = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + module.variance_epsilon) * module.weight.double()
    c, s = cos.double(), sin.double()
    a, b = n[..., :64], n[..., 64:]
    return torch.cat([a * c[:, :64] - b * s[:, :64], b * c[:, 64:] + a * s[:, 64:]], -1)


def norm_rotate_quantize(qkv, qn, kn, cos, sin, hq, hk):
    """Queries, and keys and values as the cache holds them: [heads, T, 128] fp64."""
    x = _heads(qkv, hq, hk)
    return (norm_rotate(x[:hq], qn, cos, sin), values(*quantize(norm_rotate(x[hq:hq + hk], kn, cos, sin))),
            values(*quantize(x[hq + hk:])))


def query_terms(qkv, qn, cos, sin, hq):
    """|n c| + |n' s| of each query value: what a relative error of the products scales with."""
    x = qkv.double().reshape(qkv.shape[0], -1, 128).transpose(0, 1)[:hq]
    n = (x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + qn.variance_epsilon) * qn.weight.double()).abs()
    return n * cos.double().abs() + torch.cat([n[..., 64:], n[..., :64]], -1) * sin.double().abs()


def positions(starts, lens, total):
    """[(sequence, position)] or None per row."""
    out = [None] * total
    for b in range(len(lens)):
        for t in range(int(starts[b]), int(starts[b + 1])):
            out[t] = (b, int(lens[b]) - (int(starts[b + 1]) - t))
    return out


def records(k, v, c):
    """The pages of test case c with rows k, v [heads, T, 128] (held values) in place."""
    pages = torch.zeros(c.pages.shape, dtype=torch.uint8)
    for is_v, x in enumerate((k, v)):
        codes, scale = quantize(x)  # requantising held values is exact up to the scale's choice
        raw = _heads(c.qkv, c.hq, c.hk)
        src = raw[c.hq + c.hk:] if is_v else norm_rotate(raw[c.hq:c.hq + c.hk], c.kn, c.cos, c.sin)
        codes, scale = quantize(src)
        for t, where in enumerate(positions(c.starts, c.lens, c.total)):
            if where is None:
                continue
            b, pos = where
            page, slot = int(c.table[b, pos // 64]), pos % 64
            byt, sc = pack_tokens(codes[:, t], scale[:, t], is_v, torch.full((c.hk,), slot))
            pages[page, :, 4096 * is_v + 64 * slot:4096 * is_v + 64 * slot + 64] = byt
            pages[page, :, 8192 + 512 * is_v + 8 * slot:8192 + 512 * is_v + 8 * slot + 8] = sc
    return pages


def held_mask(c):
    """Bytes of the pages that the rows of case c own."""
    mask = torch.zeros(c.pages.shape, dtype=torch.bool)
    for where in positions(c.starts, c.lens, c.total):
        if where is None:
            continue
        b, pos = where
        page, slot = int(c.table[b, pos // 64]), pos % 64
        for is_v in (0, 1):
            mask[page, :, 4096 * is_v + 64 * slot:4096 * is_v + 64 * slot + 64] = True
            mask[page, :, 8192 + 512 * is_v + 8 * slot:8192 + 512 * is_v + 8 * slot + 8] = True
    return mask


def attention(q, pages, table, starts, lens, scale, window, sinks):
    """o [T, HQ, 128] fp64 and how far a kernel may be off:
      - a probability (times V's scale) is rounded to bf16: 2^-8 of its term; exp2's
        approximation, the fp32 sums and the scale's product stay below 2^-15 of it;
      - K's codes may be multiplied with an offset, code + 8 <= 15, whose 8 sum(q) is taken off
        afterwards: the fp32 steps (two MMAs of 16 products and the subtraction, at most 2^-23 of
        the largest partial sum each, 2^-21 in all) move a score by at most
        2^-21 23 sum_group s_group sum|q|, a probability by that times |scale|, o by twice that;
      - V's codes may be multiplied with the offset too, sixteen keys at a time: two MMAs each add
        sixteen products to the sum, the second taking 8 p s off again.  An adder that lines its 17
        terms up with the largest and cuts each at 2^-23 of that is off by 17 2^-23 of the largest
        term, at most 15 sum(p s) over those keys (s: the scale of the value's group): 2^-22 255
        sum(p s) over all keys, also where every code is 0 and o with it;
      - the result is rounded to bf16: 2^-8 of itself."""
    hq, total, _ = q.shape
    hk = pages.shape[1]
    out = torch.zeros(total, hq, 128, dtype=torch.float64)
    limit = torch.full_like(out, 1e-30)
    for b in range(len(lens)):
        n, r0, r1 = int(lens[b]), int(starts[b]), int(starts[b + 1])
        if n == 0 or r1 == r0:
            continue
        k, v = (x.transpose(0, 1).reshape(hk, -1, 128)[:, :n] for x in unpack(pages[table[b, :-(-n // 64)].long()]))
        k, v = (x.repeat_interleave(hq // hk, 0) for x in (k, v))
        pos = torch.arange(n - (r1 - r0), n)[:, None]
        key = torch.arange(n)[None]
        seen = key <= pos
        if window:
            seen &= (pos - key < window) | (key < sinks)
        s = torch.where(seen, q[:, r0:r1].double() @ k.transpose(1, 2) * scale, -math.inf)
        p = torch.exp(s - torch.nan_to_num(s.amax(-1, keepdim=True), neginf=0.0))
        p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
        out[r0:r1] = (p @ v).transpose(0, 1)
        spread = (p @ v.abs()).transpose(0, 1)
        top = pages[table[b, :-(-n // 64)].long()][..., 8192:8704].contiguous().view(torch.bfloat16).double()
        top = top.reshape(-1, hk, 64, 4).transpose(0, 1).reshape(hk, -1, 4)[:, :n].amax(1).repeat_interleave(hq // hk, 0)
        mass = (q[:, r0:r1].double().abs().reshape(hq, -1, 4, 32).sum(-1) * top[:, None]).sum(-1).T[..., None]
        sv = pages[table[b, :-(-n // 64)].long()][..., 8704:].contiguous().view(torch.bfloat16).double()
        sv = sv.reshape(-1, hk, 64, 4).transpose(0, 1).reshape(hk, -1, 4)[:, :n].repeat_interleave(hq // hk, 0)
        limit[r0:r1] += 2.0 ** -22 * 255 * (p @ sv).transpose(0, 1).repeat_interleave(32, -1)
        shift = 2 * abs(scale) * 2.0 ** -21 * 23 * mass
        limit[r0:r1] += spread * (2.0 ** -8 + 2.0 ** -15) * 1.01 + (spread + out[r0:r1].abs()) * shift + out[r0:r1].abs() * 2.0 ** -8 * 1.01
    return out, limit
