"""The operators over a caller's paged cache in 64 bits, written from their definitions: what pages stand for, which keys a row sees, softmax over those alone."""
import math

import torch

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


class Heads:                     # what PagedKVCache asks of a configuration
    attention_type, is_mla, is_gqa = "gqa", False, True

    def __init__(self, kv_heads, dim): self.num_key_value_heads, self.gqa_head_dim = kv_heads, dim


DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}


def make_cache(kv_heads, dim, fmt, max_pages, page=16, layers=1, device="cuda"):
    from krasis_amd.kv_cache import PagedKVCache
    args = dict(kv_format=fmt) if fmt in ("mx8", "mx4") else dict(kv_dtype=DTYPES[fmt])
    return PagedKVCache(Heads(kv_heads, dim), layers, device, max_pages=max_pages, page_size=page, **args)


def pow2(e):
    """2^e, exact (a library's power may be off by a last bit); NaN where e is"""
    e = torch.as_tensor(e).double()
    x = ((e.nan_to_num() + 1023).long() << 52).view(torch.double)
    return torch.where(e.isnan(), torch.full_like(x, math.nan), x)


def nearest(x, fmt):
    """rows [..., dim] of bf16 / f16 as what a page of this format stands for, 64 bits; blocks of the microscaled formats with a NaN or an infinity become NaN"""
    if fmt in ("bf16", "f16"):
        return x.to(DTYPES[fmt]).double()
    x = x.double()
    mbits, least, top = (1, 0, 6.0) if fmt == "mx4" else (3, -6, 448.0)
    scale = torch.ones_like(x)
    if fmt in ("mx8", "mx4"):
        amax = x.abs().unflatten(-1, (-1, 32)).amax(-1)
        s = torch.full_like(amax, -100.0)
        for e in range(-100, 121):                   # the smallest s that holds the largest magnitude
            s = torch.where(amax > top * 2.0 ** e, torch.full_like(s, e + 1), s)
        s = torch.where(amax.isfinite(), s, torch.full_like(s, math.nan))
        scale = pow2(s).repeat_interleave(32, -1)
    y = x / scale
    exp = torch.frexp(y.abs().clamp(max=1e300))[1].double() - 1
    unit = pow2(exp.clamp(min=least) - mbits)
    y = torch.round(y / unit) * unit                 # torch.round: ties to even
    if fmt == "e4m3":
        y = torch.where(y.abs() <= top, y, torch.full_like(y, math.nan))
    return y * scale


def values(codes, scales, fmt):
    """pages' codes and scale bytes [..., dim or dim / 2], [..., dim / 32] as numbers"""
    if fmt in ("bf16", "f16"):
        return codes.double()
    if fmt == "mx4":
        table = torch.tensor(E2M1 + [-x for x in E2M1], dtype=torch.double, device=codes.device)
        x = table[torch.stack([codes & 15, codes >> 4], -1).long()].flatten(-2)
    else:
        x = codes.view(torch.float8_e4m3fn).double()
    if scales is None:
        return x
    s = torch.where(scales == 255, torch.full(scales.shape, math.nan, dtype=torch.double, device=scales.device), pow2(scales.double() - 127))
    return x * s.repeat_interleave(32, -1)


def stored_rows(cache, state, fmt, layer=0, length=None):
    """(k, v) [tokens, heads, dim] of a sequence in 64 bits, read with torch indexing"""
    n = state.seq_len if length is None else length
    pos = torch.arange(n, device=cache.k_cache.device)
    pages = torch.tensor(state.pages, device=pos.device)[pos // cache.page_size] if n else pos
    out = []
    for c, s in ((cache.k_cache, cache.k_scale), (cache.v_cache, cache.v_scale)):
        raw = c[layer].view(torch.uint8) if c.dtype == torch.float8_e4m3fn else c[layer]
        out.append(values(raw[pages, pos % cache.page_size], None if s is None else s[layer][pages, pos % cache.page_size], fmt))
    return out


def depths(parents):
    d = []
    for p in parents:
        d.append(0 if p < 0 else d[p] + 1)
    return d


def visible(before, count, window=0, first=0, parents=None):
    """[count, before + count]: which keys the new rows see"""
    n = before + count
    see = torch.zeros((count, n), dtype=torch.bool)
    at_q = list(range(before, n)) if parents is None else [before + d for d in depths(parents)]
    at_k = list(range(before)) + at_q
    for i in range(count):
        if parents is None:
            see[i, :before + i + 1] = True
        else:
            see[i, :before] = True
            j = i
            while j >= 0:
                see[i, before + j] = True
                j = parents[j]
    if window:
        q, k = torch.tensor(at_q, dtype=torch.long)[:, None], torch.tensor(at_k, dtype=torch.long)[None, :]
        see &= (q - k < window) | (k < first)
    return see


def attend(q, k, v, see, scale):
    """q [t, heads, dim], k / v [n, kv_heads, dim] in 64 bits: (out, weighted mean of |v|, largest sum of |q k| scale) [t, heads, ...].  Keys that a row does not see take no part."""
    t, heads, d = q.shape
    g = heads // k.shape[1]
    out, mean, size = torch.zeros_like(q), torch.zeros_like(q), torch.zeros((t, heads), dtype=torch.double, device=q.device)
    see = see.to(q.device)
    for h in range(heads):
        kh, vh = k[:, h // g], v[:, h // g]
        s = (q[:, h] @ kh.t().contiguous()) * scale
        s = torch.where(see, s, torch.full_like(s, -math.inf))
        p = torch.softmax(s, -1)
        if bool(kh.isfinite().all()) and bool(vh.isfinite().all()):
            out[:, h], mean[:, h] = p @ vh, p @ vh.abs()
        else:
            for i in range(t):                       # 0 times what is not finite is not 0: seen keys alone
                on = see[i]
                w = torch.softmax(s[i, on], 0)
                out[i, h], mean[i, h] = w @ vh[on], w @ vh[on].abs()
        size[:, h] = torch.where(see, (q[:, h].abs() @ kh.abs().t().contiguous()) * abs(scale), torch.zeros_like(s)).amax(-1)
    return out, mean, size


def tolerance(out, mean, size, dim, keys, dtype, weight_eps):
    """How far a result of 16 bits may be off: half a step of the type; the weights, of the sum of their |v|, by their own rounding (weight_eps), by what 32-bit sums of `dim` products
    leave in a score (both in a weight and in the denominator), and by 32-bit sums over the keys in pieces of at least eight."""
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0                     # half a step of f16's subnormal numbers
    w = weight_eps + 2 * (dim + 16) * 2.0 ** -24 * (size[..., None] + 1) + 2 * (keys / 8 + 64) * 2.0 ** -24
    return torch.finfo(dtype).eps / 2 * (out.abs() + w * mean) + w * mean + tiny
