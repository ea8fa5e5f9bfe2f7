"""The attention step over the 4-bit cache in 64 bits, from the formulas: what its tests compare with.  Works on any device."""
import math

import torch

F16 = torch.float16
# half a step of each type, relative to the value
HALF_BF16, HALF_F16, HALF_F32 = 2.0 ** -8, 2.0 ** -11, 2.0 ** -24


def byte_of(t, d, values, dim):
    """(byte, nibble) of channel d of token t (tensors) within its tile of 18 * dim bytes."""
    if values:
        h, j, n, r = d // 64, d % 64 // 16, d % 16 // 8, d % 8
        e, c, o = t // 8, t % 8 // 2, t % 2
        return 8 * dim + h * 512 + (r * 4 + c) * 16 + 4 * j + 2 * o + e, n
    w = min(2, dim // 64)
    g, c, u, b, n = d // 64, d % 64 // 16, d % 16 // 8, d % 8 // 2, d % 2
    return (((g // w * 16 + t) * 4 + c) * w + g % w) * 8 + 4 * u + b, n


def unpack(cache, page, heads, dim):
    """codes [2, slots, heads, dim], s and m [2, slots, heads, dim / 64] (float64) of a whole cache buffer [pages, >= page bytes]."""
    pages = cache.shape[0]
    tiles = cache[:, : heads * (page // 16) * 18 * dim].reshape(pages, heads, page // 16, 18 * dim)
    t = torch.arange(16, device=cache.device).unsqueeze(1)
    d = torch.arange(dim, device=cache.device).unsqueeze(0)
    codes, pairs = [], []
    for which in (0, 1):
        byte, nib = byte_of(t, d, which, dim)
        codes.append((tiles[..., byte.expand(16, dim)].long() >> (4 * nib)) & 15)
        at = 16 * dim + which * dim
        pairs.append(tiles[..., at : at + dim].contiguous().view(F16).reshape(pages, heads, page // 16, 16, dim // 64, 2).double())
    slots = lambda x: x.permute(0, 2, 3, 1, 4).reshape(pages * page, heads, -1)  # noqa: E731
    codes = torch.stack([slots(x).double() for x in codes])
    s = torch.stack([slots(x[..., 0]) for x in pairs])
    m = torch.stack([slots(x[..., 1]) for x in pairs])
    return codes, s, m


def quantize(x):
    """x [..., dim] bf16 -> (codes, s, m) float64, s and m rounded to f16 from f32 as the format says."""
    x = x.float().unflatten(-1, (-1, 64))
    low, high = x.amin(-1).clamp(-32768.0, 32768.0), x.amax(-1).clamp(-32768.0, 32768.0)
    s = ((high - low) / 15.0).half().double()
    m = low.half().double() + 0.0  # a zero minimum is +0
    codes = torch.round((x.double() - m.unsqueeze(-1)) / s.unsqueeze(-1)).clamp(0, 15)
    codes = torch.where((s > 0).unsqueeze(-1), codes, torch.zeros_like(codes))
    return codes.flatten(-2), s, m


def values(codes, s, m):
    return codes * s.repeat_interleave(64, -1) + m.repeat_interleave(64, -1)


def fill(cache, page, heads, dim, slots, k, v):
    """Writes tokens (k, v [n, heads, dim] bf16) into the cache buffer's bytes at `slots` (host loops over nothing but kinds)."""
    view = cache[:, : heads * (page // 16) * 18 * dim].reshape(cache.shape[0], heads, page // 16, 18 * dim)
    slots = slots.to(cache.device)
    pg, off = slots // page, slots % page
    head = torch.arange(heads, device=cache.device)
    for which, x in enumerate((k, v)):
        codes, s, m = quantize(x)
        codes = codes.to(torch.uint8)
        d = torch.arange(dim, device=cache.device)
        byte, nib = byte_of((off % 16)[:, None, None], d[None, None, :], which, dim)
        byte = byte.expand(len(slots), heads, dim)
        low = (nib == 0).expand_as(byte)
        index = (pg[:, None, None].expand_as(byte), head[None, :, None].expand_as(byte), (off // 16)[:, None, None].expand_as(byte), byte)
        pick = lambda sel: tuple(i[sel] for i in index)  # noqa: E731
        view[pick(low)] = codes[low]  # the low nibble's channel comes first, the other one shares its byte
        view[pick(~low)] |= codes[~low] << 4
        pair = torch.stack([s, m], -1).half().reshape(len(slots), heads, -1).view(torch.uint8)
        at = 16 * dim + which * dim + (off % 16)[:, None, None] * (dim // 16) + torch.arange(dim // 16, device=cache.device)
        at = at.expand(len(slots), heads, dim // 16)
        view[pg[:, None, None].expand_as(at), head[None, :, None].expand_as(at), (off // 16)[:, None, None].expand_as(at), at] = pair
    return cache


def norm_rope(x, heads, dim, weight, eps, cos_sin, positions, axis_of_pair, rot, interleaved):
    """x [tokens, heads * dim] -> (y, bound on what f32 steps and the last rounding to bf16 may change), both [tokens, heads, dim]."""
    y = x.double().reshape(x.shape[0], heads, dim)
    if weight is not None:
        y = y * (1.0 / torch.sqrt(y.square().mean(-1, keepdim=True) + eps)) * weight.double()
    size = y.abs()
    out, reach = y.clone(), size.clone()
    for i in range(rot // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        pos = positions.reshape(-1, positions.shape[-1])[axis_of_pair[i] if axis_of_pair is not None else 0].long()
        c, s = cos_sin[pos, i].double()[:, None], cos_sin[pos, i + rot // 2].double()[:, None]
        out[..., a] = y[..., a] * c - y[..., b] * s
        out[..., b] = y[..., b] * c + y[..., a] * s
        reach[..., a] = size[..., a] * c.abs() + size[..., b] * s.abs()
        reach[..., b] = size[..., b] * c.abs() + size[..., a] * s.abs()
    # f32: mean, + eps, sqrt, division, two products, then product and sum: 8 roundings of at most half a step each
    return out, HALF_BF16 * out.abs() + (1 + HALF_BF16) * 8 * HALF_F32 * reach + 1e-38


def attention(q, cu_q, kv_lens, page_table, cache, page, heads_kv, dim, scale, causal, window, rounded=True):
    """(out [rows, heads_q, dim], lse [rows, heads_q], bound on out, bound on lse) in float64.

    The bounds count, for every score and every output, the roundings that the operator makes:
      scores   products of f16 numbers are exact, their sum over dim channels and the sum with the minima's part are f32: at most
               (dim + 8) additions of at most one unit of 2^-23 of the sum of magnitudes; each operand is rounded to f16 at most
               once (2^-11), which is what `rounded` allows
      weights  exp2 in f32 (2^-21 with its argument's rounding), once to f16 (2^-11)
      outputs  f32 sums over n keys (2^-23 each, at most n + 64 of them, but no more than 2^-11 in all for n up to 4096),
               operands of the product rounded to f16 at most once, then bf16
    The sums of magnitudes are over s * c + |m|, since the two parts are added separately.
    """
    codes, s, m = unpack(cache, page, heads_kv, dim)
    rows, heads_q = q.shape[0], q.shape[1] // dim
    out = torch.zeros(rows, heads_q, dim, dtype=torch.float64, device=q.device)
    out_tol = torch.zeros_like(out)
    lse = torch.full((rows, heads_q), -math.inf, dtype=torch.float64, device=q.device)
    lse_tol = torch.zeros_like(lse)
    group = heads_q // heads_kv
    for b in range(len(kv_lens)):
        r0, r1, n_keys = int(cu_q[b]), int(cu_q[b + 1]), int(kv_lens[b])
        n = r1 - r0
        if n == 0 or n_keys == 0:
            continue
        place = torch.arange(n_keys, device=q.device)
        slots = page_table[b].long()[place // page] * page + place % page
        last = n_keys - n + torch.arange(n, device=q.device).unsqueeze(1)
        seen = torch.ones(n, n_keys, dtype=torch.bool, device=q.device)
        if causal:
            seen = seen & (place <= last)
        if window:
            seen = seen & (place > last - window)
        for h in range(heads_q):
            hk = h // group
            k = values(codes[0, slots, hk], s[0, slots, hk], m[0, slots, hk])
            v = values(codes[1, slots, hk], s[1, slots, hk], m[1, slots, hk])
            k_mag = values(codes[0, slots, hk], s[0, slots, hk], m[0, slots, hk].abs())
            v_mag = values(codes[1, slots, hk], s[1, slots, hk], m[1, slots, hk].abs())
            x = q[r0:r1].double().reshape(n, heads_q, dim)[:, h]
            score = (x @ k.T) * scale
            mag = (x.abs() @ k_mag.T) * abs(scale)
            off = mag * ((dim + 8) * 2.0 ** -23 + (2 * HALF_F16 if rounded else 0.0))  # of a score, in nats
            masked = score.masked_fill(~seen, -math.inf)
            some = seen.any(1)
            l = torch.logsumexp(masked, 1)
            p = torch.where(seen, torch.exp(masked - torch.where(some, l, torch.zeros_like(l))[:, None]), torch.zeros_like(score))
            worst = torch.where(seen, off, torch.zeros_like(off)).amax(1) + 2.0 ** -20
            out[r0:r1, h] = p @ v
            lse[r0:r1, h] = torch.where(some, l, torch.full_like(l, -math.inf))
            each = 2 * worst + 3 * HALF_F16 + min(2.0 ** -11, (n_keys + 64) * 2.0 ** -23)
            out_tol[r0:r1, h] = torch.expm1(each)[:, None] * (p @ v_mag) * (1 + HALF_BF16) + HALF_BF16 * out[r0:r1, h].abs() + 1e-30
            lse_tol[r0:r1, h] = worst + HALF_F16 * 2 + 2.0 ** -20 * (1 + l.abs().nan_to_num(posinf=0.0))
    return out, lse, out_tol, lse_tol
