"""64-bit references of the operators around a layer's 8-bit products, and how far fp32 arithmetic may be from them.  Plain torch on the CPU."""
import math

import torch

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}  # a rounding, relative: half a step
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}  # and among the subnormal numbers
FLOOR = {torch.int8: 1e-5, torch.float8_e4m3fn: 448e-12}
MOST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def rounding(v, dtype):
    """Half a step of dtype at the values v."""
    return HALF[dtype] * v.abs() + TINY[dtype]


def to_codes(v, dtype):
    """64-bit quotients as codes (64-bit numbers)."""
    if dtype == torch.int8:
        return v.round().clamp(-127, 127)
    return v.clamp(-448, 448).float().to(dtype).double()


def code_half_step(v, dtype):
    """How far a code may be from the quotient v that it stands for."""
    return torch.full_like(v, 0.5) if dtype == torch.int8 else torch.maximum(v.abs() * 2.0 ** -4, torch.full_like(v, 2.0 ** -10))


def norm(x, weight, residual, eps):
    """h and n of add_rms_norm_quant."""
    h = x.double() + (0 if residual is None else residual.double())
    return h, h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()


# n in fp32: the sum of squares goes through chains of at most 64 additions of a lane, 6 across a wave and 16 across waves (half of their error
# counts, under the root), then the mean, eps, root (an ulp and a half), and two products: (86 / 2 + 8) half ulps of 2^-24 at most.
NORM_ERROR = 51 * 2.0 ** -24


def lora(y, x, a, b, adapters, start, scales):
    """(result, what fp32 sums and the two 16-bit halves of a x may add up to) in 64 bits."""
    T = x.shape[0]
    out, slack = y.double().clone(), torch.zeros(y.shape, dtype=torch.float64)
    rows = [(i, [i]) for i in range(T)] if start is None else [(i, list(range(start[i], start[i + 1]))) for i in range(len(start) - 1)]
    K, r = x.shape[1], a.shape[1]
    for i, mine in rows:
        s = int(adapters[i])
        if not mine or not 0 <= s < a.shape[0]:
            continue
        A, B, f = a[s].double(), b[s].double(), 1.0 if scales is None else float(scales[s].double())
        X = x[mine].double()
        v = X @ A.T
        out[mine] += f * (v @ B.T)
        # v: K additions of fp32; two halves: 2^-18 of a number in bf16, in fp16 (which ends at 2^-25) of the row's largest, the scale and
        # the power of two 2^-24 each; B v: 2 r additions
        dv = (K + 4) * 2.0 ** -24 * (X.abs() @ A.abs().T) + 2.0 ** -18 * v.abs().amax(-1, keepdim=True)
        slack[mine] += abs(f) * (dv @ B.abs().T + (2 * r + 4) * 2.0 ** -24 * (v.abs() @ B.abs().T))
    return out, slack


def route(logits, top, renormalize):
    """Chosen experts and their shares per token, as lists."""
    ids, shares = [], []
    for row in logits.double().tolist():
        order = sorted(range(len(row)), key=lambda i: (-row[i], i))[:top]
        best = row[order[0]]
        p = [0.0 if best == -math.inf else math.exp(row[i] - best) for i in order]
        total = sum(p) if renormalize else sum(math.exp(v - best) if best > -math.inf else 0.0 for v in row)
        ids.append(order)
        shares.append([v / total if total else 0.0 for v in p])
    return ids, shares


def moe(a, a_scale, logits, w13, s13, w2, s2, top, renormalize=True):
    """(y, how far fp32 arithmetic may be from it) in 64 bits.  Codes of h that lie nearer to the border between two than the fp32 h and scale
    are exact may be either: what that changes is part of the slack."""
    T, K = a.shape
    I = w2.shape[2]
    code = a.dtype
    y, slack = torch.zeros(T, K, dtype=torch.float64), torch.zeros(T, K, dtype=torch.float64)
    ids, shares = route(logits, top, renormalize)
    up = 2.0 ** -24
    for t in range(T):
        x = a[t].double()
        sa = float(a_scale[t if a_scale.numel() > 1 else 0].double())
        for e, c in zip(ids[t], shares[t]):
            if c == 0.0:
                continue
            W, S = w13[e].double(), s13[e].double()
            z, dz = W @ x, W.abs() @ x.abs() * ((K + 4) * up if code != torch.int8 else 0.0)
            z, dz = z * sa * S, dz * abs(sa) * S.abs()
            dz = dz + 4 * up * z.abs()  # the conversion, two scales, their product
            g, u, dg, du = z[:I], z[I:], dz[:I], dz[I:]
            sig = torch.sigmoid(g)
            h = g * sig * u
            # d(g sig)/dg <= 1.1; exp to two ulps, an addition, a division, a product
            dh = 1.1 * dg * u.abs() + (g * sig).abs() * du + dg * du + 8 * up * (1 + g.abs()) * h.abs()
            m = float(h.abs().max())
            dm = float(dh.max())
            s = max(m, FLOOR[code]) / MOST[code]
            ds = dm / MOST[code] / s + 3 * up  # relative
            v = h / s
            dv = dh / s + v.abs() * ds
            q = to_codes(v, code)
            lo, hi = to_codes(v - dv, code), to_codes(v + dv, code)
            either = torch.maximum((hi - q).abs(), (q - lo).abs())
            D, S2 = w2[e].double(), s2[e].double()
            part, sums = D @ q, D.abs() @ q.abs()
            y[t] += c * s * S2 * part
            # Up to sixteen waves of up to eight blocks share the experts' reductions: each wave's part of a sum (in int32 for int8) is converted,
            # multiplied by its scales and added in fp32 to what the wave has, then the waves' sums and the blocks' are added.  Running sums are no
            # larger than the magnitudes in them, so that is a rounding of the sum of magnitudes for the conversions, two for the products, one for each
            # addition on the longest way: `top` in a wave, 16 over the waves, 8 over the blocks.
            wrong = D.abs() @ either + part.abs() * (ds + 10 * up) + sums * up * (27 + top + (I if code != torch.int8 else 0))
            slack[t] += c * s * S2.abs() * wrong
    return y, slack
