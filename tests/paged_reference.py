"""Norm, rotation, store and attention over a paged key-value cache in 64 bits on the CPU, one row at a time, with bounds of
what fp32 sums and the roundings to 16 and 8 bits may differ by."""
import math

import torch


def eps_half(dt):
    return torch.finfo(dt).eps / 2


def rows_of(lens, start, T):
    """(row, sequence, position) of every row that belongs to a sequence."""
    out = []
    for b, L in enumerate(lens):
        r0, r1 = (b, b + 1) if start is None else (start[b], start[b + 1])
        for r in range(r0, min(r1, T)):
            out.append((r, b, L - (r1 - r0) + r - r0))
    return out


def page_of(table, b, j, size, pages):
    if j < 0 or j // size >= table.shape[1]:
        return None
    p = int(table[b, j // size])
    return p if 0 <= p < pages else None


def keys_of(cache, scale, table, b, n, h):
    """[n, D] fp64 and which of the first n keys of the sequence are there."""
    pages, _, size, D = cache.shape
    x, there = torch.zeros(n, D, dtype=torch.float64), torch.zeros(n, dtype=torch.bool)
    for j in range(n):
        p = page_of(table, b, j, size, pages)
        if p is None:
            continue
        there[j] = True
        x[j] = cache[p, h, j % size].double()
        if scale is not None:
            x[j] *= scale[p, h, j % size].double()
    return x, there


def attention(q, kc, vc, table, lens, start=None, scale=None, window=0, sinks=0, ks=None, vs=None):
    """(out, bound): out [T, H, D] fp64, rows of no sequence zero; bound: how far a kernel may be from it elementwise."""
    T, H, D = q.shape
    G = H // kc.shape[1]
    scale = D ** -0.5 if scale is None else scale
    out, bound = torch.zeros(T, H, D, dtype=torch.float64), torch.zeros(T, H, D, dtype=torch.float64)
    u = eps_half(q.dtype)
    # the probabilities' rounding: to q's type, or with an e4m3 cache to bf16 (two terms for fp16: 2^-16)
    up = u if ks is None else 2.0 ** -16 if q.dtype == torch.float16 else 2.0 ** -8
    kept = {}
    for r, b, p in rows_of(lens, start, T):
        n = max(0, min(lens[b], table.shape[1] * kc.shape[2]))
        for h in range(H):
            if (b, h // G) not in kept:
                kept[b, h // G] = keys_of(kc, ks, table, b, n, h // G), keys_of(vc, vs, table, b, n, h // G)
            (k, there), (v, _) = kept[b, h // G]
            j = torch.arange(n)
            seen = there & (j <= p)
            if window:
                seen &= (j > p - window) | (j < sinks)
            if not seen.any():
                continue
            k, v = k[seen], v[seen]
            x = q[r, h].double()
            s = scale * (k @ x)
            w = torch.softmax(s, 0)
            out[r, h] = w @ v
            # scores: D products and sums in fp32, and the scale's and the exponent's own roundings; twice (numerator, denominator)
            ds = float((abs(scale) * (k.abs() @ x.abs())).max()) * (D + 8) * 2.0 ** -24 + 2.0 ** -20
            mean = w @ v.abs()
            more = int(seen.sum()) * 2.0 ** -25 * float(v.abs().max()) if q.dtype == torch.float16 and ks is None else 0.0  # fp16 below its normals
            bound[r, h] = u * out[r, h].abs() + (up + 2 * ds + (int(seen.sum()) + 64) * 2.0 ** -23) * (1 + u) * mean + more + 2.0 ** -24
    return out, bound


def turned(x, w, eps, cos, sin, p, interleaved):
    """(y, how far fp32 may be from it) of one row [H, D]"""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    y = x.clone()
    off = x.abs()
    if cos is not None:
        half = cos.shape[1]
        c, s = cos[p].double(), sin[p].double()
        a, b = (x[:, 0:2 * half:2], x[:, 1:2 * half:2]) if interleaved else (x[:, :half], x[:, half:2 * half])
        na, nb = a * c - b * s, b * c + a * s
        oa = a.abs() + b.abs()
        if interleaved:
            y[:, 0:2 * half:2], y[:, 1:2 * half:2] = na, nb
            off[:, 0:2 * half:2] = off[:, 1:2 * half:2] = oa
        else:
            y[:, :half], y[:, half:2 * half] = na, nb
            off[:, :half] = off[:, half:2 * half] = oa
    # a sum of up to 256 squares over lanes (16 roundings), root, quotient, two products; two products and a sum
    return y, off * 32 * 2.0 ** -24


def make_pages(g, lens, size, spare=3):
    """A block table over shuffled pages: [B, P] with -1 behind a sequence's last page, and the number of pages."""
    need = [max(0, -(-n // size)) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(need + [1]) + 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pages


def make_cache(g, pages, heads, size, D, dt, e4m3, layout="heads"):
    """k, v, k_scale, v_scale; layout "heads": a head's keys of a page together, "keys": a key's heads together."""
    def one(mul):
        x = torch.randn(pages, heads, size, D, generator=g) * mul
        scale = None
        if e4m3:
            scale = x.abs().amax(-1) / 448
            x = (x / scale[..., None]).to(torch.float8_e4m3fn)
        else:
            x = x.to(dt)
        if layout == "keys":
            x = x.transpose(1, 2).contiguous().transpose(1, 2)
        return x, scale
    k, ks = one(1.5)
    v, vs = one(1.0)
    return k, v, ks, vs


def worst(y, ref, bound):
    """largest |y - ref| / bound (inf where y is not finite)"""
    d = (y.double().cpu() - ref).abs() / bound.clamp(min=1e-30)
    return math.inf if not torch.isfinite(d).all() else float(d.max()) if d.numel() else 0.0
