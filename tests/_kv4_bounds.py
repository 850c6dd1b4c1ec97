"""The plain formula of attention over the 4-bit cache in 64 bits, with pages that are absent, and
bounds on what each kernel's arithmetic may be off by (test helper)."""
import math

import torch

from tests import _kv4 as ref

CUT = 2.0 ** -23  # a tensor core's adder lines 17 terms up with the largest and cuts each there


def attention(q, pages, table, starts, lens, scale, window=0, sinks=0, registers=True):
    """o [T, HQ, 128] fp64 and how far the kernel of up to 32 columns (`registers`) or that of more may
    be off.  Keys in pages whose id is outside the cache, or behind the table, are seen by nobody.
      - Both round a probability to bf16, the registers' kernel after multiplying it with V's scale:
        2^-8 of its term; exp2, the sums and the joins stay below 2^-15 of it.  The result rounds to
        bf16: 2^-8 of itself.
      - Scores, more columns: eight MMAs of 16 products, each cutting 17 terms at 2^-23 of the
        largest, which is at most sum |q k|: 136 2^-23 sum |q k|.
      - Scores, registers: codes carry an offset, code + 8 <= 15, whose 8 sum(q) is taken off again: per
        group of channels two MMAs and the subtraction, 2^-21 23 sum_group s_group sum |q| in all.
      - A probability below 2^-126 of the largest may be 0: exp2 has no subnormals.
      - A score off by e moves a probability by e of itself, the result by e (sum p |v| + |o|).
      - P V, more columns: eight MMAs a block of 128 keys, each cutting 17 terms at 2^-23 of the
        largest, at most sum p |v|: 136 2^-23 sum p |v| a block.
      - P V, registers: a fragment of 16 keys is two MMAs (codes with their offset, and the offset taken
        off), the largest of whose terms is at most what the sum holds so far plus 15 p s of its
        keys: 34 2^-23 (sum p |v| + 15 sum_fragment p s), or 34 of fp32's smallest steps, 2^-149, of a sum
        held 2^-69 too small.  A warp has at most two fragments of every fourth page, and the sums of its
        fragments add up to at most all keys'."""
    hq, total, _ = q.shape
    num, hk = pages.shape[:2]
    k_all, v_all = (x.transpose(1, 2) for x in ref.unpack(pages))  # [pages, 64, heads, 128]
    scales = pages[..., 8192:].contiguous().view(torch.bfloat16).double().reshape(num, hk, 2, 64, 4).permute(2, 0, 3, 1, 4)
    out = torch.zeros(total, hq, 128, dtype=torch.float64)
    limit = torch.full_like(out, 1e-30)
    for b in range(len(lens)):
        n, r0, r1 = int(lens[b]), int(starts[b]), int(starts[b + 1])
        held = min(n, table.shape[1] * 64)
        if held <= 0 or r1 == r0:
            continue
        key = torch.arange(held)
        page, slot = table[b, key // 64].long(), key % 64
        there = (page >= 0) & (page < num)
        page = page.clamp(0, num - 1)
        rep = hq // hk
        k, v, sk, sv = (x[page, slot].transpose(0, 1).repeat_interleave(rep, 0) for x in (k_all, v_all, *scales))
        k, v, sk, sv = (torch.where(there[None, :, None], x, 0.0) for x in (k, v, sk, sv))  # [HQ, keys, ..]
        pos = torch.arange(n - (r1 - r0), n)[:, None]
        seen = (key <= pos) & there
        if window:
            seen &= (pos - key < window) | (key < sinks)
        x = q[:, r0:r1].double()
        s = torch.where(seen, x @ k.transpose(1, 2) * scale, -math.inf)
        p = torch.exp(s - torch.nan_to_num(s.amax(-1, keepdim=True), neginf=0.0))
        p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
        o, spread = ((p @ y).transpose(0, 1) for y in (v, v.abs()))
        if registers:
            mass = torch.where(seen, x.abs().unflatten(-1, (4, 32)).sum(-1) @ sk.transpose(1, 2), 0.0)
            score = 2.0 ** -21 * 23 * abs(scale) * mass
            fragments = 2 * -(-(-(-held // 64)) // 4)
            product = 34 * fragments * 2.0 ** -80 + 34 * CUT * (fragments * spread + 15 * (p @ sv).transpose(0, 1).repeat_interleave(32, -1))
        else:
            score = 136 * CUT * abs(scale) * torch.where(seen, x.abs() @ k.abs().transpose(1, 2), 0.0)
            product = 136 * CUT * -(-held // 128) * spread
        product = product + 2.0 ** -126 * (seen.double() @ v.abs()).transpose(0, 1)
        off = score.amax(-1).transpose(0, 1)[..., None]
        limit[r0:r1] += spread * (2.0 ** -8 + 2.0 ** -15) + (spread + o.abs()) * off + product + o.abs() * 2.0 ** -8
        limit[r0:r1] *= 1.01  # products of these
        out[r0:r1] = o
    return out, limit
