"""Plain forms of the cache and norm operators for the tests: the row quantiser in
32-bit operations (codes and scales must match it bit for bit), attention and
norm in 64 bits with bounds on the error of the kernels' arithmetic."""
import numpy as np
import torch

TOP = {"f8": 448.0, "i8": 127.0}
# unit roundoffs: half a step over the smallest value of a binade, so 2^-p with
# p significant bits (24 in 32 bits, 8 in bfloat16, 11 in float16)
U32 = 2.0 ** -24
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: U32}


def quantise(x, fmt):
    """(values of the codes as float32, scales) of rows of x (CPU float32), by the
    definition: a = max|x|; a < 2^-100: zeros; not finite: scale NaN, codes 0."""
    a = x.abs().amax(-1) if x.shape[-1] else torch.zeros(x.shape[:-1])
    a = torch.where(torch.isnan(x).any(-1), torch.tensor(float("nan")), a)
    fin = torch.isfinite(a)
    big = fin & (a >= 2.0 ** -100)
    safe = torch.where(big, a, torch.ones(()))
    scale = torch.where(big, safe / TOP[fmt], torch.zeros(()))
    inv = torch.where(big, torch.full_like(safe, TOP[fmt]) / safe, torch.zeros(()))  # a number / tensor rounds twice
    v = torch.where(big[..., None], x * inv[..., None], torch.zeros(()))
    code = v.round() if fmt == "i8" else v.to(torch.float8_e4m3fn).float()
    return code, torch.where(fin, scale, torch.tensor(float("nan")))


class Seqs:
    """A batch's layout on the host: starts, chunk lengths, page table."""

    def __init__(self, starts, lens, page, spare=2, seed=0, width=None):
        r = np.random.default_rng(seed)
        self.starts, self.lens, self.page = list(starts), list(lens), page
        need = [-(-(o + n) // page) for o, n in zip(starts, lens)]
        self.n_pages = sum(need) + spare
        ids = r.permutation(self.n_pages)
        self.table = np.full((len(need), max(need + [1]) if width is None else width), -1, np.int32)
        at = 0
        for s, p in enumerate(need):
            self.table[s, :p] = ids[at:at + p]
            at += p
        self.free = ids[at:]
        self.offsets = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        self.tokens = int(self.offsets[-1])

    def place(self, s, j):
        """(page, slot) of position j of sequence s; page -1: unmapped."""
        c = j // self.page
        p = self.table[s, c] if 0 <= c < self.table.shape[1] else -1
        return (int(p) if 0 <= p < self.n_pages else -1), j % self.page


def attention(sq, k, v, q, group, scale, window):
    """In 64 bits: (out, lse, bound of |out error| before its rounding, bound of
    |lse error|) given the cache's values k, v [pages, heads, page, dim] (numpy
    float64) and q [tokens, heads, dim].  p_unit: roundoff of the probabilities."""
    T, HQ, D = q.shape
    out, lse = np.zeros((T, HQ, D)), np.full((T, HQ), -np.inf)
    absv, slack, keys = np.zeros((T, HQ, D)), np.zeros((T, HQ)), np.zeros(T)
    for s, (o, n) in enumerate(zip(sq.starts, sq.lens)):
        where = [sq.place(s, j) for j in range(o + n)]
        mapped = np.array([p >= 0 for p, _ in where], bool)
        pg = np.array([max(p, 0) for p, _ in where], np.int64)
        sl = np.array([x for _, x in where], np.int64)
        ks, vs = k[pg, :, sl].copy(), v[pg, :, sl].copy()   # [L, H, D]
        ks[~mapped], vs[~mapped] = 0, 0
        for i in range(n):
            t, p = int(sq.offsets[s]) + i, o + i
            j = np.arange(o + n)
            see = mapped & (j <= p)
            if window:
                see &= j > p - window
            idx = np.nonzero(see)[0]
            keys[t] = idx.size
            if not idx.size:
                continue
            for h in range(HQ):
                kk, vv = ks[idx, h // group], vs[idx, h // group]
                e = scale * (kk @ q[t, h])
                m = e.max()
                w = np.exp(e - m)
                l = w.sum()
                out[t, h] = w @ vv / l
                lse[t, h] = m + np.log(l)
                absv[t, h] = w @ np.abs(vv) / l
                slack[t, h] = abs(scale) * (np.abs(kk) @ np.abs(q[t, h])).max()
    return out, lse, absv, slack, keys


def attention_bounds(out, lse, absv, slack, keys, D, p_unit, out_type, vmax):
    """Bounds on the kernels' error.  A score is a 32-bit dot of D exact products
    (error <= D U32 |q||k|, and a few roundings of scalings), so a weight is off by
    twice that (its own score and the maximum) relatively; weights are rounded
    once to p_unit before they meet the values, in 16-bit floats with a smallest
    step of 2^-32 of the largest weight; sums of n terms in 32 bits add n U32."""
    n = keys[:, None]
    rel = 2 * (D + 8) * U32 * slack + (n + 16) * U32
    b = absv * (p_unit * (1 + 2.0 ** -6) + rel)[..., None] + (n * vmax * 2.0 ** -32)[..., None]
    b = b + np.abs(out) * UNIT[out_type] * 1.01 + 2.0 ** -24
    return b, (D + 8) * U32 * slack + (n + 16) * U32 + 4 * U32 * (1 + np.abs(np.where(np.isfinite(lse), lse, 0)))


def norm(x, r, w, eps):
    """(h, y) in 64 bits."""
    h = x.double() + (0 if r is None else r.double())
    return h, h / torch.sqrt(h.pow(2).mean(-1, keepdim=True) + eps) * w.double()
