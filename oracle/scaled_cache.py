"""The 8-bit cache with one scale for each (block, kv head), in 64 bits on the CPU: what the kernels' results are compared with.

Codes are kept as the numbers they are (int8 values, e4m3 values), tokens in a block's order: [blocks, tokens, heads, head_size]."""
import math

import torch

TOP = {"int8": 127.0, "fp8_e4m3": 448.0}


def codes_of(cache: torch.Tensor, kind: str) -> torch.Tensor:
    """[blocks, tokens, heads, head_size] numbers of a key cache (five axes) or a value cache (four)."""
    x = cache.view(torch.int8 if kind == "int8" else torch.float8_e4m3fn).double()
    if x.dim() == 5:
        return x.permute(0, 3, 1, 2, 4).flatten(3)
    return x.permute(0, 3, 1, 2)


def cache_of(codes: torch.Tensor, kind: str, keys: bool) -> torch.Tensor:
    """The inverse of ``codes_of``."""
    b, t, h, d = codes.shape
    x = codes.float().to(torch.int8 if kind == "int8" else torch.float8_e4m3fn).view(torch.uint8)
    if keys:
        return x.view(b, t, h, d // 16, 16).permute(0, 2, 3, 1, 4).contiguous()
    return x.permute(0, 2, 3, 1).contiguous()


def half_step(y: torch.Tensor, kind: str) -> torch.Tensor:
    """The furthest that the nearest code may be from y (within the codes' range)."""
    if kind == "int8":
        return torch.full_like(y, 0.5)
    place = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    return torch.exp2(place - 4)


def write(x, codes, scales, slots, kind):
    """What blocks hold after the tokens x [T, heads, D] went to their slots: (scales, values that each slot's code should stand
    for in units of the new scale [blocks, tokens, heads, D], blocks touched).  Values are not rounded to codes."""
    blocks, size = codes.shape[:2]
    x = x.double()
    want, new = codes.clone(), scales.double().clone()
    touched = set()
    for t, slot in enumerate(slots.tolist()):
        if 0 <= slot < blocks * size:
            touched.add(slot // size)
    for b in sorted(touched):
        there = {s % size: t for t, s in enumerate(slots.tolist()) if 0 <= s < blocks * size and s // size == b}
        some = torch.stack([x[t] for t in there.values()])
        finite = torch.where(torch.isfinite(some), some.abs(), 0.0)
        largest = finite.amax((0, 2))
        old = torch.zeros_like(new[b]) if 0 in there else new[b]
        now = torch.maximum(old, torch.where(largest < 2.0 ** -100, 0.0, largest / TOP[kind]))
        ratio = torch.where(now > 0, old / now.clamp(min=1e-300), 0.0)
        want[b] *= ratio[:, None]
        for o, t in there.items():
            y = torch.where(now[:, None] > 0, x[t] / now[:, None].clamp(min=1e-300), 0.0)
            want[b, o] = torch.nan_to_num(y, nan=0.0).clamp(-TOP[kind], TOP[kind])
        new[b] = now
    return new, want, sorted(touched)


def rows(codes, scales, table, length):
    """[length, heads, D] of a sequence: codes times scales; blocks that do not exist give zeros.  And which tokens exist."""
    blocks, size = codes.shape[:2]
    found, there = [], []
    for b in table.tolist()[:(length + size - 1) // size]:
        good = 0 <= b < blocks
        found.append(codes[b] * scales[b].double()[None, :, None] if good else torch.zeros_like(codes[0]))
        there.append(torch.full((size,), good))
    if not found:
        return codes.new_zeros(0, *codes.shape[2:]), torch.zeros(0, dtype=torch.bool)
    return torch.cat(found)[:length], torch.cat(there)[:length]


def attention(query, key_codes, value_codes, key_scales, value_scales, table, length, first, scale, kind, slopes=None, window=0):
    """query [rows, heads, D], row j at position first + j of a sequence of `length` tokens.  (out, bound): in 64 bits, and how far a
    kernel may be off that keeps scores, sums and weights in 32 bits and hands the second product its weights as halves:

      weights:  relative 2^-11 (a half's rounding); below a half's normal numbers 2^-25, where the largest product of weight and scale that
                the row sees stands at 2^7 or above, so 2^-32 of that one; and 2^-22 for exp2;
      scales:   they go into the exponent as logarithms, 4 roundings of numbers up to 32 and the largest of them, in numerator and sum;
      scores:   the D products and their sum, relative 2^-24 each of sum |q||k|, and three roundings of the score: d; a weight over the
                sum of weights is then off by 2 d;
      sums:     one rounding for each of T tokens, the running maximum's factors among them, of numerator and denominator.
    The rounding of the result itself comes on top."""
    n, heads, d = query.shape
    k, there = rows(key_codes, key_scales, table, length)
    v, _ = rows(value_codes, value_scales, table, length)
    group = heads // k.shape[1] if k.shape[1] else 1
    out = torch.zeros(n, heads, d, dtype=torch.float64)
    bound = torch.zeros_like(out)
    t = k.shape[0]
    if t == 0:
        return out, bound
    q = query.double()
    at = torch.arange(t)
    pos = first + torch.arange(n)
    see = there[None] & (at[None] <= pos[:, None])
    if window:
        see &= at[None] > pos[:, None] - window
    u32 = 2.0 ** -24
    pages = [b if 0 <= b < key_codes.shape[0] else 0 for b in table.tolist()[:(length + key_codes.shape[1] - 1) // key_codes.shape[1]]]
    scale_of = value_scales.double()[pages].repeat_interleave(key_codes.shape[1], 0)[:t]          # [tokens, kv heads]
    for h in range(heads):
        g = h // group
        kk, vv = torch.where(there[:, None], k[:, g], 0.0), torch.where(there[:, None], v[:, g], 0.0)
        x = (q[:, h] @ kk.T) * scale
        size = (q[:, h].abs() @ kk.abs().T) * abs(scale)
        if slopes is not None:
            bias = slopes[h].double() * (at[None] - pos[:, None])
            x, size = x + bias, size + bias.abs()
        off = torch.where(see, (d + 8) * u32 * size, 0.0).amax(1, keepdim=True)
        x = x.masked_fill(~see, -math.inf)
        w = torch.softmax(x, 1)
        w = torch.where(see.any(1, keepdim=True), w, 0.0)
        out[:, h] = w @ vv
        mass = w @ vv.abs()
        sv = torch.where(see, scale_of[:, g], 0.0)
        largest = (w * sv).amax(1, keepdim=True) * TOP[kind]
        powers = torch.where(sv > 0, sv, 1.0).log2().abs().amax(1, keepdim=True) + 32
        bound[:, h] = mass * (2.0 ** -11 + 2.0 ** -21 + 2 * off + 2.0 ** -21 * powers + 4 * t * u32) + t * 2.0 ** -32 * largest
    return out, bound
