"""The paged E4M3 K/V cache restated in 64 bits for the tests: rounding, append, values and
attention, from their definitions, on any device, without the package."""
import torch

D = 128
E_MIN, E_MAX = -120, 119


def e4m3(x):
    """Nearest E4M3 value (ties to even) of float64 x, saturating at +-448; NaN stays NaN."""
    _, e = torch.frexp(torch.where(torch.isfinite(x), x, torch.ones_like(x)))
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def need_exp(amax):
    """Smallest e in [E_MIN, E_MAX] with amax <= 448 * 2^e, for one Python float."""
    e = E_MIN
    while e < E_MAX and amax > 448.0 * 2.0 ** e:
        e += 1
    return e


class RefCache:
    """A dense twin of a paged cache: float64 codes per page and exponents per page and head."""

    def __init__(self, pages, heads, P, device="cpu"):
        self.codes = torch.zeros(2, pages, heads, P, D, dtype=torch.float64, device=device)
        self.exp = torch.full((2, pages, heads), E_MIN, dtype=torch.int64, device=device)
        self.P = P

    def append(self, k, v, table, start, count):
        """k / v [B, S, heads, 128]; table, start, count nested lists."""
        P = self.P
        for kv, x in ((0, k), (1, v)):
            x = x.double()
            for b in range(x.shape[0]):
                for page in range(start[b] // P, (start[b] + count[b] + P - 1) // P):
                    lo, hi = max(start[b], page * P), min(start[b] + count[b], (page + 1) * P)
                    if hi <= lo:
                        continue
                    pid, n_old = table[b][page], max(0, start[b] - page * P)
                    new = x[b, lo - start[b]:hi - start[b]]                       # [n, heads, 128]
                    for h in range(x.shape[2]):
                        w = new[:, h]
                        fin = w[torch.isfinite(w)].abs()
                        e = need_exp(float(fin.max()) if fin.numel() else 0.0)
                        if n_old:
                            e_old = int(self.exp[kv, pid, h])
                            e = max(e, e_old)
                            c = self.codes[kv, pid, h, :n_old]
                            self.codes[kv, pid, h, :n_old] = e4m3(c * 2.0 ** (e_old - e))
                        self.exp[kv, pid, h] = e
                        at = lo - page * P
                        self.codes[kv, pid, h, at:at + hi - lo] = e4m3(w * 2.0 ** -e)

    def values(self, kv, row, n):
        """[heads, n, 128] float64 values of the first n positions of a table row."""
        pid = torch.tensor(row[:-(-n // self.P)], dtype=torch.int64, device=self.codes.device)
        x = self.codes[kv][pid] * torch.exp2(self.exp[kv][pid].double())[:, :, None, None]
        return x.transpose(0, 1).reshape(self.codes.shape[2], -1, D)[:, :n]


def attention(q, k, v, nq, causal, window, scale):
    """One sequence: q [Sq, Hq, 128] float64, k / v [heads, n, 128] float64; query i < nq at
    position n - nq + i.  Returns o [Sq, Hq, 128] and the per-element error scale of an fp32
    kernel with f16 probabilities (see error_bound)."""
    Sq, Hq, _ = q.shape
    Hk, n, _ = k.shape
    o = torch.zeros_like(q)
    bound = torch.zeros_like(q)
    if nq == 0 or n == 0:
        return o, bound
    pos = torch.arange(n - nq, n, device=q.device)[:, None]
    j = torch.arange(n, device=q.device)[None, :]
    hide = torch.zeros(nq, n, dtype=torch.bool, device=q.device)
    if causal:
        hide |= j > pos
    if window is not None:
        hide |= (j - pos).abs() > window
    dead = hide.all(1)[:, None]
    for h in range(Hq):
        kh, vh = k[h * Hk // Hq], v[h * Hk // Hq]
        s = (q[:nq, h] @ kh.T) * scale
        s = torch.where(hide, torch.full_like(s, -torch.inf), s)     # by selection: NaN keys stay hidden
        p = torch.softmax(s, -1)
        p = torch.where(dead, torch.zeros_like(p), p)
        # hidden keys are left out by selection too: 0 * NaN
        nan = torch.isnan(vh).any(1)
        if bool(nan.any()):
            clean = torch.nan_to_num(vh, nan=0.0)
            oh = p @ clean
            hit = (~hide).double() @ torch.isnan(vh).double() > 0
            oh = torch.where(hit, torch.full_like(oh, torch.nan), oh)
        else:
            clean, oh = vh, p @ vh
        o[:nq, h] = oh
        # dS: each score is a sum of 128 products held in fp32 (at most 2^-23 of the sum of
        # magnitudes per addition); hidden and NaN scores do not count
        mag = (q[:nq, h].abs() @ torch.nan_to_num(kh).abs().T) * scale
        ds = (2.0 ** -16 * torch.where(hide, torch.zeros_like(mag), mag)).amax(-1, keepdim=True)
        # probabilities: half a step of f16, 2^-11, of p; scores twice (numerator and sum);
        # fp32 sums over the keys and exp2 within 2^-13; p below 2^-28 of the largest within
        # 2^-31 (f16's subnormal half step, the page scale folded in up to 2^-8)
        bound[:nq, h] = (2.0 ** -11 + 2.0 ** -13 + 2 * ds) * (p @ clean.abs()) + 2.0 ** -31 * n * clean.abs().max()
    return o, bound


def error_bound(o, bound):
    """Largest allowed |kernel - o| for a bf16 output: half a step of bf16, 2^-8 of the value
    (2^-134 where bf16 is subnormal), and the kernel's own error."""
    return 2.0 ** -8 * (o.abs() + bound) + bound + 2.0 ** -134


def seen_bound(q, k, v, v_unit, nq, causal, window, scale):
    """The error that an attention kernel may make in fp32 with f16 probabilities, from the keys that
    each row sees alone: as in `attention`, with its last term by row.  v_unit [heads, n]: the scale
    of each key's V.  p below 2^-28 of the row's largest is off by half of f16's smallest step, which
    is 2^-31 of the largest weight at most (V's scales are folded into p down to 2^-8), and weighs a
    code of up to 448 in units of the largest V scale that the row sees."""
    Sq, Hq, _ = q.shape
    Hk, n, _ = k.shape
    bound = torch.zeros_like(q)
    if nq == 0 or n == 0:
        return bound
    pos = torch.arange(n - nq, n, device=q.device)[:, None]
    j = torch.arange(n, device=q.device)[None, :]
    see = torch.ones(nq, n, dtype=torch.bool, device=q.device)
    if causal:
        see &= j <= pos
    if window is not None:
        see &= (j - pos).abs() <= window
    zero = torch.zeros((), dtype=torch.float64, device=q.device)
    for h in range(Hq):
        kh, vh, unit = k[h * Hk // Hq], v[h * Hk // Hq], v_unit[h * Hk // Hq]
        s = torch.where(see, (q[:nq, h] @ kh.T) * scale, -torch.inf)
        p = torch.where(see.any(1)[:, None], torch.softmax(s, -1), zero)
        ds = torch.where(see, 2.0 ** -16 * (q[:nq, h].abs() @ kh.abs().T) * scale, zero).amax(-1, keepdim=True)
        top = torch.where(see, 448.0 * unit, zero).amax(-1, keepdim=True)
        bound[:nq, h] = (2.0 ** -11 + 2.0 ** -13 + 2 * ds) * (p @ vh.abs()) + 2.0 ** -31 * see.sum(-1, keepdim=True) * top
    return bound
