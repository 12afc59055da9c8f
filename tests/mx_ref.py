"""The operators of a decoder block in microscaled types in 64 bits, on the CPU, from their definitions: no code
shared with the framework."""
import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
# Half the smallest subnormal: what rounding to the type may be off by below its normal range.
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
E4M3 = [(m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)) for e in range(16) for m in range(8)][:-1]


def quantized(x, format):
    """(codes as integers, scale bytes) of x [rows, K]: each block's exponent by trying them all, each value by looking for
    the nearest, the even code at a tie."""
    table = torch.tensor(E2M1 if format == "e2m1" else E4M3, dtype=torch.float64)
    x = x.double().unflatten(-1, (-1, 32))
    top = x.abs().amax(-1)
    e = torch.full(top.shape, 127, dtype=torch.long)
    for k in range(127, -128, -1):
        e[top <= table[-1] * 2.0 ** k] = k
    bad = ~torch.isfinite(x).all(-1)
    m = torch.where(bad[..., None], 0.0, x.abs() * torch.exp2(-e.double())[..., None])
    code = torch.zeros(m.shape, dtype=torch.long)
    for i in range(len(table) - 1):
        mid = (table[i] + table[i + 1]) / 2
        code += ((m > mid) | ((m == mid) & (i % 2 == 1))).long()
    sign = torch.signbit(x) & ~bad[..., None]
    code = code + sign * (8 if format == "e2m1" else 128)
    return code.flatten(-2), torch.where(bad, 255, e + 127)


def unpacked(codes):
    """Codes as integers, from the framework's storage."""
    codes = codes.cpu()
    if codes.dtype == torch.uint8:
        return torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    return codes.view(torch.uint8).long()


def packed(code, format):
    """The framework's storage of codes given as integers."""
    if format == "e2m1":
        c = code.unflatten(-1, (-1, 2))
        return (c[..., 0] | c[..., 1] << 4).to(torch.uint8)
    return code.to(torch.uint8).view(torch.float8_e4m3fn)


def values(mx):
    codes, scales = mx
    c = unpacked(codes)
    if codes.dtype == torch.uint8:
        t = torch.tensor(E2M1 + [-v for v in E2M1], dtype=torch.float64)
    else:
        t = torch.tensor(E4M3 + [float("nan")] + [-v for v in E4M3] + [float("nan")], dtype=torch.float64)
    s = scales.cpu().long()
    s = torch.where(s == 255, float("nan"), torch.exp2((s - 127).double()))
    return (t[c].unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def random_mx(seed, lead, K, format, lo=120, hi=131, device="cpu"):
    """Codes of all values (no NaN) and scales from a range of exponents."""
    g = torch.Generator().manual_seed(seed)
    top = 16 if format == "e2m1" else 256
    code = torch.randint(0, top, (*lead, K), generator=g)
    if format == "e4m3":
        code = torch.where(code % 128 == 127, code - 1, code)
    scales = torch.randint(lo, hi, (*lead, K // 32), generator=g).to(torch.uint8)
    return packed(code, format).to(device), scales.to(device)


def product_bound(x, w, dtype, format):
    """What a product of values x [M, K] and w [N, K] may be off by.

    f32 sums of instructions that add up to 128 exact products: (K / 32 + 16) additions, each off by 2^-23 of the sum of
    magnitudes so far (partial sums of waves and splits among them).  The 8-bit instruction loses up to 2^-11 of the largest
    product among its 128; f32 results do not use it.  Then a rounding to dtype."""
    K = x.shape[1]
    mag = x.abs() @ w.abs().t()
    y = (x @ w.t()).abs()
    b = (K / 32 + 16) * 2.0 ** -23 * mag
    if format == "e4m3" and dtype != torch.float32:
        for k in range(0, K, 128):
            xk, wk = x[:, k:k + 128].abs(), w[:, k:k + 128].abs()
            # of many results the largest factors stand for the largest product
            big = xk.shape[0] * wk.shape[0] > 10 ** 6
            b += 2.0 ** -11 * (xk.amax(-1)[:, None] * wk.amax(-1)[None] if big else (xk[:, None] * wk[None]).amax(-1))
    return b + UNIT[dtype] * (y + b) + TINY[dtype]


def rms_norm(x, weight, eps):
    x = x.double()
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    return y if weight is None else y * weight.double()


def rms_norm_gradient(dy, x, weight, dsum, eps):
    """(dx, dweight, and the sums of magnitudes that either adds up)."""
    x, dy = x.double(), dy.double()
    D = x.shape[-1]
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    g = dy if weight is None else dy * weight.double()
    ds = 0.0 if dsum is None else dsum.double()
    dx = r * g - r ** 3 * x * (g * x).sum(-1, keepdim=True) / D + ds
    mag = (r * g).abs() + r ** 3 * x.abs() * (g * x).abs().sum(-1, keepdim=True) / D + (0.0 if dsum is None else ds.abs())
    t = dy * x * r
    return dx, t.reshape(-1, D).sum(0), mag, t.abs().reshape(-1, D).sum(0)


def route(logits, k, scoring="softmax", bias=None, groups=1, kept=1, best=1, normalize=True, scale=1.0, active=None):
    """(ids, weights) row by row."""
    z = logits.double()
    s = torch.sigmoid(z) if scoring == "sigmoid" else torch.softmax(z, -1)
    T, E = z.shape
    size = E // groups
    ids, ws = torch.full((T, k), -1, dtype=torch.int32), torch.zeros(T, k, dtype=torch.float64)
    low = lambda v: float("-inf") if v != v else v  # noqa: E731
    for t in range(T):
        if active is not None and not active[t]:
            continue
        zt, st = z[t].tolist(), s[t].tolist()
        if scoring == "softmax" and all(v == float("-inf") for v in zt):
            st = [0.0] * E
        by = [st[e] + float(bias[e]) for e in range(E)] if bias is not None else zt
        allowed = range(E)
        if kept < groups:
            of = by if bias is not None or best == 1 else st
            score = [sum(sorted((low(v) for v in of[g * size:(g + 1) * size]), reverse=True)[:best]) for g in range(groups)]
            chosen = sorted(range(groups), key=lambda g: (-score[g], g))[:kept]
            allowed = [e for e in range(E) if e // size in chosen]
        # NaN after all others, the lowest expert first among equal ones
        order = sorted(allowed, key=lambda e: (by[e] != by[e], -by[e] if by[e] == by[e] else 0.0, e))[:k]
        w = torch.tensor([st[e] for e in order], dtype=torch.float64)
        if normalize:
            total = w.sum()
            w = torch.zeros_like(w) if total == 0 else w / total
        if scoring == "softmax" and any(v != v or v == float("inf") for v in zt):
            w = torch.full_like(w, float("nan"))
        ids[t], ws[t] = torch.tensor(order, dtype=torch.int32), w * scale
    return ids, ws


def plan(ids, E):
    flat = ids.flatten().tolist()
    lists = [[c for c, e in enumerate(flat) if e == x] for x in range(E)] + [[c for c, e in enumerate(flat) if not 0 <= e < E]]
    starts = [0]
    for rows in lists[:E]:
        starts.append(starts[-1] + len(rows))
    return torch.tensor(starts, dtype=torch.int32), torch.tensor([c for rows in lists for c in rows], dtype=torch.int32)


def route_gradient(dw, logits, ids, scoring, normalize, scale):
    """(dlogits, a bound of what their terms come to) by the chain rule through autograd in 64 bits."""
    z = logits.double().requires_grad_(True)
    s = torch.sigmoid(z) if scoring == "sigmoid" else torch.softmax(z, -1)
    live = (ids >= 0) & (ids < z.shape[1])
    p = torch.where(live, s.gather(1, ids.clamp(0, z.shape[1] - 1).long()), 0.0)
    total = p.sum(-1, keepdim=True)
    w = scale * (p / torch.where(total > 0, total, 1.0) if normalize else p)
    up = torch.where(live, dw.double(), 0.0)
    (w * up).sum().backward()
    with torch.no_grad():
        u = up.abs() * scale
        share = p / torch.where(total > 0, total, 1.0)
        if normalize:
            u = (u + (u * share).sum(-1, keepdim=True)) / torch.where(total > 0, total, 1.0)
        m = torch.zeros_like(s).scatter_add_(1, ids.clamp(0, z.shape[1] - 1).long(), torch.where(live, u, 0.0))
        mag = s * (m + (0.0 if scoring == "sigmoid" else (m * s).sum(-1, keepdim=True)))
    return z.grad, mag


def experts(x, w, ids, bias):
    """y [T, k, N] and the values that x's rows and the experts have."""
    xv, wv = values(x), values(w)
    T, k = ids.shape
    y = torch.zeros(T, k, wv.shape[1], dtype=torch.float64)
    for t in range(T):
        for j in range(k):
            e = int(ids[t, j])
            if 0 <= e < wv.shape[0]:
                y[t, j] = wv[e] @ (xv[t, j] if xv.dim() == 3 else xv[t]) + (0.0 if bias is None else bias[e].double())
    return y, xv, wv
