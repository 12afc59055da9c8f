"""The paged-cache operators in 64 bits, on the CPU, from their definitions: no code shared with the framework.

A Problem holds the tokens of every sequence in plain order; it lays them out in pages, with every place
that no token fills set to NaN and every table entry that names no page to one far out of range."""
import math

import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
# Half the smallest subnormal: what rounding to the type may be off by where the value is below its normal range.
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


def pieces(dtype):
    return 8 if dtype != torch.float32 else 4


def lay_out(k, v, pages, page):
    """k, v: lists of [length, heads, D] (CPU), pages: lists of page ids.  (k_cache, v_cache) of max page + 1."""
    dtype, (_, heads, D) = k[0].dtype, k[0].shape
    C = pieces(dtype)
    pool = max([p for ps in pages for p in ps], default=0) + 1
    kc = torch.full((pool, heads, page // 16, D // C, 16, C), float("nan"), dtype=dtype)
    vc = torch.full((pool, heads, page // C, D, C), float("nan"), dtype=dtype)
    for kb, vb, ps in zip(k, v, pages):
        for j in range(kb.shape[0]):
            p, s = ps[j // page], j % page
            kc[p, :, s // 16, :, s % 16] = kb[j].view(heads, D // C, C)
            vc[p, :, s // C, :, s % C] = vb[j]
    return kc, vc


class Problem:
    def __init__(self, seed, lens, heads, group, D, page=16, dtype=torch.bfloat16, std=1.5):
        """lens: (new, cached with them) of each sequence."""
        g = torch.Generator().manual_seed(seed)
        self.lens, self.heads, self.group, self.D, self.page, self.dtype = lens, heads, group, D, page, dtype
        rnd = lambda *s: (torch.randn(s, generator=g, dtype=torch.float32) * std).to(dtype)  # noqa: E731
        self.T = sum(n for n, _ in lens)
        self.q = rnd(self.T, heads * group, D)
        self.k = [rnd(L, heads, D) for _, L in lens]
        self.v = [rnd(L, heads, D) for _, L in lens]
        need = [-(-L // page) for _, L in lens]
        order = torch.randperm(sum(need) + 3, generator=g).tolist()
        self.pages, at = [], 0
        for n in need:
            self.pages.append(order[at:at + n])
            at += n
        self.pool = sum(need) + 3

    def starts(self):
        s = [0]
        for n, _ in self.lens:
            s.append(s[-1] + n)
        return s

    def batch(self, device="cuda", max_q=None, max_kv=None, width=0, junk=2 ** 30):
        import mlxq
        width = max(width, 1, *(len(p) for p in self.pages))
        rows = [p + [junk] * (width - len(p)) for p in self.pages]
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
        return mlxq.CacheBatch(i32(rows), i32(self.starts()), i32([L for _, L in self.lens]),
                               max(n for n, _ in self.lens) if max_q is None else max_q,
                               max(L for _, L in self.lens) if max_kv is None else max_kv)

    def cache(self, device="cuda"):
        kc, vc = lay_out(self.k, self.v, self.pages + [[self.pool - 1]], self.page)
        return kc.to(device), vc.to(device)


def attention(pr, scale=None, causal=True, window=0, softcap=0.0, prefix=None, slopes=None, sinks=None, roundoff=None):
    """(result, bound on a kernel's error) [T, Hq, D] in 64 bits.

    The bound, for unit roundoff u of the type: the result is rounded once (u |o|, or TINY below the normal range); 16-bit softmax weights are
    rounded (u A, A = sum w |v| / sum w); f32 scores, exponents and sums are off by e = 2^-24 (D S + 16 (1 + max |z|) + L / 4)
    relative, S the largest sum of |q_d k_d| scale of the row (a dot product of D terms in any order, the weight's exponent
    an absolute error of a score; a sum of L terms spread over at least four partial sums), twice (numerator and
    denominator): 2 e A.  fp16 weights below 2^-25 of the largest vanish, up to L 2^-25 max |v| in sum."""
    scale = 1 / math.sqrt(pr.D) if scale is None else scale
    out = torch.zeros(pr.T, pr.heads * pr.group, pr.D, dtype=torch.float64)
    tol = torch.zeros_like(out)
    t = 0
    u = UNIT[pr.dtype]
    for b, (n, L) in enumerate(pr.lens):
        for i in range(n):
            p = L - n + i
            hi = min(L, max(p + 1, int(prefix[b]) if prefix is not None else 0)) if causal else L
            lo = max(0, p + 1 - window) if window else 0
            for h in range(pr.heads * pr.group):
                if hi <= lo:
                    continue
                q = pr.q[t, h].double()
                k, v = (x[b][lo:hi, h // pr.group].double() for x in (pr.k, pr.v))
                z = (k @ q) * scale
                S = float((k.abs() @ q.abs()).max()) * scale
                if softcap:
                    z = softcap * torch.tanh(z / softcap)
                if slopes is not None:
                    z = z - float(slopes[h]) * (p - torch.arange(lo, hi)).abs()
                m = z.max() if sinks is None else max(z.max(), float(sinks[h]))
                w = torch.exp(z - m)
                total = w.sum() + (math.exp(float(sinks[h]) - m) if sinks is not None else 0.0)
                o, A = (w @ v) / total, (w @ v.abs()) / total
                e = 2.0 ** -24 * (pr.D * S + 16 * (1 + float(z.abs().max())) + (hi - lo) / 4)
                out[t, h] = o
                tol[t, h] = u * o.abs() + 2 * e * A + TINY[pr.dtype]
                if pr.dtype != torch.float32:
                    tol[t, h] += u * A * (1 + 2.0 ** -6)
                if pr.dtype == torch.float16:
                    tol[t, h] += (hi - lo) * 2.0 ** -25 * v.abs().max() / max(float(total), 1e-30) * float(torch.exp(z.max() - m))
            t += 1
    return out, tol


def rotated(x, positions, table, interleaved, inverse=False):
    """x [T, heads, D] turned, in 64 bits; NaN in the turned features for positions outside the table."""
    R = 2 * table.shape[1]
    y = x.double().clone()
    for t, p in enumerate(positions):
        for i in range(R // 2):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
            c, s = (table[p, i].double().tolist() if 0 <= p < table.shape[0] else (math.nan, math.nan))
            s = -s if inverse else s
            xa, xb = x[t, :, a].double(), x[t, :, b].double()
            y[t, :, a], y[t, :, b] = xa * c - xb * s, xb * c + xa * s
    return y


def rotation_bound(x, table, dtype):
    """|error| of a turned value: two products and a sum in f32, the result rounded once to the type."""
    m = x.double().abs().amax() * table.double().abs().amax()
    return float(m) * (2 * UNIT[dtype] + 4 * 2.0 ** -24)
