"""Plain 64-bit forms of the 4-bit cache operators, of the head norms with rotation and of packed causal attention, on the
CPU, for the tests to compare with."""
import torch

F64 = torch.float64
LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
BORDERS = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]           # a tie goes to the even code
SCALES = [m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)][:127]


def _round_to_grid(x, grid):
    """Index of the nearest grid value of every element of x >= 0, ties to the even index, the last one beyond the end."""
    g = torch.tensor(grid, dtype=F64)
    mid = (g[1:] + g[:-1]) / 2
    i = torch.bucketize(x, mid)                              # mid[i-1] < x <= mid[i]
    tie = (i < len(mid)) & (x == mid[i.clamp(max=len(mid) - 1)])
    return torch.where(tie & (i % 2 == 1), i + 1, i)


def quantise(x, g=1.0):
    """(codes [.., D], scale bytes [.., D/16]) of [.., D]."""
    b = x.to(F64).unflatten(-1, (-1, 16)) / g
    top = b.abs().amax(-1)
    finite = torch.isfinite(b).all(-1)
    scale = _round_to_grid(torch.where(finite, top, 0.0) / 6.0, SCALES)
    s = torch.tensor(SCALES, dtype=F64)[scale][..., None]
    ratio = torch.where((s > 0) & finite[..., None], b / s, 0.0)
    code = _round_to_grid(ratio.abs(), LEVELS) + 8 * (ratio < 0)
    return code.flatten(-2), torch.where(finite, scale, 127)


def values(codes, scales, g=1.0):
    """What codes [.., D] and scale bytes [.., D/16] stand for."""
    lv = torch.tensor(LEVELS + [-x for x in LEVELS], dtype=F64)[codes.long()]
    sc = torch.tensor(SCALES + [float("nan")], dtype=F64)[scales.long()]
    return lv * sc.repeat_interleave(16, -1) * g


def held(x, g=1.0):
    return values(*quantise(x, g), g)


def pack(k, v, gk=1.0, gv=1.0):
    """Pool rows [n, heads, 9 D / 8] of k and v [n, heads, D]."""
    (kc, ks), (vc, vs) = quantise(k, gk), quantise(v, gv)
    two = lambda c: c[..., 0::2] + 16 * c[..., 1::2]         # noqa: E731
    return torch.cat((two(kc), two(vc), ks, vs), -1).to(torch.uint8)


def unpack(pool, gk=1.0, gv=1.0):
    d = pool.shape[-1] * 8 // 9
    codes = torch.stack((pool[..., :d] & 15, pool[..., :d] >> 4), -1).flatten(-2)
    x = values(codes, pool[..., d:])
    return x[..., :d] * gk, x[..., d:] * gv


def rotate(x, positions, base, scale=1.0):
    """[n, heads, D] turned by the positions [n]."""
    d = x.shape[-1]
    freq = base ** (-torch.arange(0, d, 2, dtype=F64) / d) / scale
    ang = positions.to(F64)[:, None] * freq
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    lo, hi = x.to(F64).chunk(2, -1)
    return torch.cat((lo * c - hi * s, hi * c + lo * s), -1)


def norm(x, w, eps):
    x = x.to(F64)
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w.to(F64)


def attend(q, k, v, seen, sm_scale, cap=0.0):
    """q [nq, hq, D], k, v [nk, hkv, D], seen [nq, nk] -> outputs [nq, hq, D] and sum_j p_j |v_j|, which scales their
    rounding errors.  Keys that are not seen do not enter, whatever they hold; a row that sees nothing gives zeros."""
    nq, hq, d = q.shape
    group = hq // k.shape[1]
    out, mag = torch.zeros(nq, hq, d, dtype=F64), torch.zeros(nq, hq, d, dtype=F64)
    q, k, v = q.to(F64), k.to(F64), v.to(F64)
    for i in range(nq):
        at = seen[i].nonzero()[:, 0]
        if at.numel() == 0:
            continue
        for h in range(hq):
            s = k[at, h // group] @ q[i, h] * sm_scale
            if cap > 0:
                s = cap * torch.tanh(s / cap)
            p = torch.softmax(s, 0)
            out[i, h] = p @ v[at, h // group]
            mag[i, h] = p @ v[at, h // group].abs()
    return out, mag


def causal(lens, tokens):
    """seen [tokens, tokens] of packed sequences of these lengths."""
    seen = torch.zeros(tokens, tokens, dtype=torch.bool)
    a = 0
    for n in lens:
        seen[a:a + n, a:a + n] = torch.ones(n, n, dtype=torch.bool).tril()
        a += n
    return seen
