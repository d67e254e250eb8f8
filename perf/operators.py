"""Timed cases of the operators around a cache held in 4 bits: what one layer does with a prompt and with the tokens after it.

* ``norm``   -- RMS norm of every query and key head with the position rotation in the same pass (``norm_rotate``);
* ``cache``  -- key and value rows quantised into pool rows as they are written, and read back (``kv4_write``, ``kv4_read``);
* ``attend`` -- decode attention of a ragged batch over such pool rows (``kv4_attend``);
* ``prompt`` -- causal attention of packed prompts of different lengths, grouped heads (``prompt_attend``).

Head counts are those of the framework's two models (32 query and 8 KV heads, 28 and 4) and of their shards over
several ranks; head_dim is 128, or 64 as in the framework's tests.  Keys and values follow the benchmark's
distribution: N(0, 1) with four outlier channels times 8; pool rows are a random permutation, as a pool of page size 1
is after some time of serving.

The plain forms compute in 32 bits and round once; angles are products of whole positions with 64-bit frequencies, and the
quantiser compares in 64 bits, where its borders are exact.
"""
import math

import torch

own = False

HEADS = {                        # query heads, KV heads, rope base
    "llama": (32, 8, 5e5), "llama/4": (8, 2, 5e5), "llama/8": (4, 1, 5e5),
    "qwen": (28, 4, 1e6), "qwen/2": (14, 2, 1e6), "qwen/4": (7, 1, 1e6),
}
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
BLOCK = 16                       # elements of a head that share a scale
EPS = 1e-6                       # of the norm


def _case(name, op, heads, d=128, dtype="bf16", **more):
    return {"name": name, "op": op, "heads": heads, "d": d, "dtype": dtype, **more}


def listed():
    return [
        # one decoded token of one request, deep in a long context: latency alone
        _case("norm 1 token", "norm", "llama", tokens=1, first=130000),
        # the packed tokens of a prefill step
        _case("norm 8192 tokens", "norm", "llama", tokens=8192, first=0),
        # the new rows of a decode step of sixteen requests
        _case("cache 16 rows", "cache", "llama", rows=16, pool=65536),
        # the rows of a prompt, odd count
        _case("cache 16385 rows", "cache", "llama", rows=16385, pool=65536),
        # the list of a selection: 128 + 2048 + 512 rows of one request
        _case("attend 1 x 2688", "attend", "llama", batch=1, lo=2688, hi=2688),
        # ordinary serving: chats and documents of very different lengths, seven heads a group
        _case("attend 16 x 1000..32000", "attend", "qwen", batch=16, lo=1000, hi=32000),
        # one long document, all of it attended to
        _case("attend 1 x 131072", "attend", "llama", batch=1, lo=131072, hi=131072),
        # a loaded server of long documents
        _case("attend 4 x 100000..262144", "attend", "qwen", batch=4, lo=100000, hi=262144),
        # packed prompts of a continuous batch, the shortest a single token
        _case("prompt 9 x 1..2000", "prompt", "qwen", batch=9, lo=1, hi=2000),
        # one long prompt
        _case("prompt 1 x 8192", "prompt", "llama", batch=1, lo=8192, hi=8192),
        # a longer one on a quarter of the heads
        _case("prompt 1 x 16384", "prompt", "llama/4", batch=1, lo=16384, hi=16384),
        # the check mode in fp32
        _case("prompt 3 x 200..1500 fp32", "prompt", "llama/4", dtype="fp32", batch=3, lo=200, hi=1500),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "cache", "attend", "attend", "prompt", "prompt"])
    heads, d = rng.choice(sorted(HEADS)), rng.choice([128, 128, 128, 64])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    if op == "norm":
        c = _case("", op, heads, d, dtype, tokens=_log(rng, 1, 8192), first=rng.choice([0, rng.randrange(1000000)]))
    elif op == "cache":
        c = _case("", op, heads, d, dtype, rows=_log(rng, 1, 16385), pool=rng.choice([20000, 65536]))
    elif op == "attend":
        # at most half a million rows in all, an eighth of that in fp32
        most = 524288 if dtype == "bf16" else 65536
        batch = _log(rng, 1, 32)
        hi = _log(rng, 16, most // batch)
        c = _case("", op, heads, d, dtype, batch=batch, lo=_log(rng, 1, hi), hi=hi)
    else:
        hq = HEADS[heads][0]
        most = int(math.sqrt((2 ** 31 if dtype == "bf16" else 2 ** 25) / hq))   # tokens in all
        batch = _log(rng, 1, 16)
        hi = _log(rng, 16, most // batch)
        c = _case("", op, heads, d, dtype, batch=batch, lo=_log(rng, 1, hi), hi=hi)
    del c["name"]
    return c


def lengths(case):
    """Tokens of each request: spread over the logarithm, odd and even ones, the longest first."""
    lo, hi, b = case["lo"], case["hi"], case["batch"]
    return [max(lo, int(hi * (lo / hi) ** (i / max(1, b - 1)))) for i in range(b)]


def work(case):
    hq, hkv, _ = HEADS[case["heads"]]
    d, es = case["d"], TYPES[case["dtype"]].itemsize
    held = hkv * d * 9 // 8                                   # a pool row: K and V codes, K and V scales
    if case["op"] == "norm":
        t = case["tokens"]
        return {"bytes": t * (2 * hq + 3 * hkv) * d * es + 4 * t + 2 * d * es, "flops": t * (hq + hkv) * d * 7}
    if case["op"] == "cache":
        n = case["rows"]
        return {"bytes": n * (4 * hkv * d * es + 2 * held + 8), "flops": 2 * n * hkv * d * 4}
    lens = lengths(case)
    if case["op"] == "attend":
        n = sum(lens)
        return {"bytes": n * (held + 4) + 2 * len(lens) * hq * d * es, "flops": 4 * n * hq * d}
    n = sum(lens)
    return {"bytes": n * (2 * hq + 2 * hkv) * d * es, "flops": 4 * d * hq * sum(x * (x + 1) // 2 for x in lens)}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _rows(gen, n, heads, d, dtype, loud):
    """Rows of keys or values: N(0, 1), the ``loud`` channels of every head times 8."""
    x = torch.randn(n, heads, d, generator=gen, device="cuda")
    x[:, :, loud] *= 8.0
    return x.to(dtype)


def prepare(case, seed):
    hq, hkv, base = HEADS[case["heads"]]
    d, dtype = case["d"], TYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    loud = torch.randperm(d, generator=gen, device="cuda")[:4]
    st = {"case": case, "hq": hq, "hkv": hkv, "d": d, "dtype": dtype, "base": base, "sm_scale": d ** -0.5}
    if case["op"] == "norm":
        t = case["tokens"]
        qkv = torch.randn(t, (hq + 2 * hkv) * d, generator=gen, device="cuda").to(dtype)     # what the projection leaves
        st["q"] = qkv[:, : hq * d].view(t, hq, d)
        st["k"] = qkv[:, hq * d: (hq + hkv) * d].view(t, hkv, d)
        st["q_weight"] = (1.0 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(dtype)
        st["k_weight"] = (1.0 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(dtype)
        st["positions"] = torch.arange(case["first"], case["first"] + t, dtype=torch.int32, device="cuda")
    elif case["op"] == "cache":
        n = case["rows"]
        st["k"] = _rows(gen, n, hkv, d, dtype, loud)
        st["v"] = _rows(gen, n, hkv, d, dtype, loud[:0])
        st["rows"] = torch.randperm(case["pool"], generator=gen, device="cuda")[:n].int()
        st["pool"] = torch.zeros(case["pool"], hkv, d * 9 // 8, dtype=torch.uint8, device="cuda")
    elif case["op"] == "attend":
        lens = lengths(case)
        n, ctx = sum(lens) + 7, max(lens)
        # 4096 different tokens, quantised once; every pool row is one of them
        bank = _pack(_rows(gen, 4096, hkv, d, dtype, loud), _rows(gen, 4096, hkv, d, dtype, loud[:0]))
        st["pool"] = bank[torch.randint(4096, (n,), generator=gen, device="cuda")]
        perm = torch.randperm(n, generator=gen, device="cuda").int()
        at = torch.tensor([sum(lens[:i]) for i in range(len(lens))], device="cuda")
        pos = torch.arange(ctx, device="cuda")
        st["req_to_token"] = perm[torch.clamp(at[:, None] + pos[None, :], max=n - 1)].contiguous()
        st["req_pool_indices"] = torch.arange(len(lens), dtype=torch.int32, device="cuda")
        st["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        st["q"] = torch.randn(len(lens), hq * d, generator=gen, device="cuda").to(dtype)
    else:
        lens = lengths(case)
        t = sum(lens)
        st["q"] = torch.randn(t, hq, d, generator=gen, device="cuda").to(dtype)
        st["k"] = _rows(gen, t, hkv, d, dtype, loud)
        qkv = torch.randn(t, (hq + 2 * hkv) * d, generator=gen, device="cuda").to(dtype)
        st["v"] = qkv[:, (hq + hkv) * d:].view(t, hkv, d)                                     # where the projection left it
        st["cu_seqlens"] = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")
    return st


# ---------------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _levels(device):
    """What the 16 codes of a 4-bit float stand for: sign, two bits of exponent, one of mantissa."""
    up = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    return torch.tensor(up + [-x for x in up], dtype=torch.float32, device=device)


def _quantise(x):
    """(codes, scale bytes) of rows [n, heads, d]: per 16 elements a scale of 8 bits (4 of exponent, 3 of mantissa),
    the greatest magnitude over 6; codes are the nearest of the 16 levels, ties to the even code."""
    n, h, d = x.shape
    x = x.double().view(n, h, d // BLOCK, BLOCK)
    six = torch.full((1,), 6.0, dtype=torch.float64, device=x.device)      # a tensor: the product with 1/6 would miss ties
    scale = torch.clamp(x.abs().amax(-1) / six, max=448.0).float().to(torch.float8_e4m3fn)
    s = scale.double()[..., None]
    a = torch.where(s > 0, x.abs() / s, 0.0)
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int()
            + (a >= 3.5).int() + (a > 5.0).int())
    code = torch.where((x < 0) & (s > 0), code + 8, code).view(n, h, d)
    return code.to(torch.uint8), scale.view(torch.uint8)


def _pack(k, v):
    """Pool rows [n, heads, 9 d / 8] of keys and values: K codes, V codes (two a byte, the lower half first), K scales, V scales."""
    (kc, ks), (vc, vs) = _quantise(k), _quantise(v)
    return torch.cat((kc[..., 0::2] | (kc[..., 1::2] << 4), vc[..., 0::2] | (vc[..., 1::2] << 4), ks, vs), dim=-1)


def _unpack(held, d):
    """What pool rows [..., 9 d / 8] stand for, in 32 bits: K [..., d] and V [..., d]."""
    levels = _levels(held.device)
    codes = torch.stack((held[..., :d] & 15, held[..., :d] >> 4), dim=-1).flatten(-2).int()
    scales = held[..., d:].contiguous().view(torch.float8_e4m3fn).float()
    x = (levels[codes].unflatten(-1, (2 * d // BLOCK, BLOCK)) * scales[..., None]).flatten(-2)
    return x[..., :d], x[..., d:]


def _angles(positions, d, base):
    """cos, sin [n, d/2] of whole positions, the products taken in 64 bits."""
    freq = base ** (-torch.arange(0, d, 2, dtype=torch.float64, device=positions.device) / d)
    ang = positions.double()[:, None] * freq
    return ang.cos().float(), ang.sin().float()


def _turn(x, cos, sin):
    """Rotation of the pairs (i, i + d/2); cos and sin broadcast against [..., d/2]."""
    lo, hi = x.chunk(2, dim=-1)
    return torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), dim=-1)


def _plain_norm(st):
    def normed(x, w):
        x = x.float()
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    cos, sin = _angles(st["positions"], st["d"], st["base"])
    q, k = normed(st["q"], st["q_weight"]), normed(st["k"], st["k_weight"])
    cos, sin = cos[:, None], sin[:, None]
    return tuple(x.to(st["dtype"]) for x in (_turn(q, cos, sin), _turn(k, cos, sin), k))


def _plain_cache(st):
    rows = st["rows"].long()
    st["pool"][rows] = _pack(st["k"], st["v"])
    k, v = _unpack(st["pool"][rows], st["d"])
    return k.to(st["dtype"]), v.to(st["dtype"])


def _plain_attend(st):
    b, hq, hkv, d = st["q"].shape[0], st["hq"], st["hkv"], st["d"]
    ctx = st["req_to_token"].shape[1]
    rows = st["req_to_token"][st["req_pool_indices"].long()].long()
    pos = torch.arange(ctx, device=rows.device)
    cos, sin = _angles(pos, d, st["base"])
    k, v = _unpack(st["pool"][rows], d)                                       # [b, ctx, hkv, d]
    k = _turn(k, cos[None, :, None], sin[None, :, None])
    last = torch.clamp(st["seq_lens"].long() - 1, min=0)
    q = _turn(st["q"].float().view(b, hq, d), cos[last][:, None], sin[last][:, None])
    s = q.view(b, hkv, hq // hkv, d) @ k.permute(0, 2, 3, 1) * st["sm_scale"]
    s = s.masked_fill((pos[None] >= st["seq_lens"][:, None])[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = (p @ v.permute(0, 2, 1, 3)) / p.sum(-1, keepdim=True)
    return o.reshape(b, hq * d).to(st["dtype"])


def _plain_prompt(st):
    t, hq, d = st["q"].shape
    hkv = st["hkv"]
    i = torch.arange(t, device=st["q"].device)
    seq = (i[:, None] >= st["cu_seqlens"][None, 1:]).sum(-1)
    seen = (seq[:, None] == seq[None, :]) & (i[None, :] <= i[:, None])
    q = st["q"].float().view(t, hkv, hq // hkv, d).permute(1, 2, 0, 3).reshape(hkv, -1, d)
    s = (q @ st["k"].float().permute(1, 2, 0)).view(hkv, hq // hkv, t, t) * st["sm_scale"]
    s = s.masked_fill(~seen, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True)
    o = p.view(hkv, -1, t) @ st["v"].float().permute(1, 0, 2)
    o = o.view(hkv, hq // hkv, t, d) / total
    return o.permute(2, 0, 1, 3).reshape(t, hq, d).to(st["dtype"])


def run(st):
    op = st["case"]["op"]
    if own:
        from tokenselect_b200 import prompt, quant_cache
        if op == "norm":
            return prompt.norm_rotate(st["q"], st["k"], st["positions"], rope_base=st["base"], q_weight=st["q_weight"],
                                      k_weight=st["k_weight"], eps=EPS, with_plain_k=True)
        if op == "cache":
            quant_cache.kv4_write(st["pool"], st["k"], st["v"], st["rows"])
            return quant_cache.kv4_read(st["pool"], st["rows"], st["dtype"])
        if op == "attend":
            return quant_cache.kv4_attend(st["q"], st["pool"], st["req_to_token"], st["req_pool_indices"], st["seq_lens"],
                                          sm_scale=st["sm_scale"], rope_base=st["base"])
        return prompt.prompt_attend(st["q"], st["k"], st["v"], st["cu_seqlens"], sm_scale=st["sm_scale"])
    return {"norm": _plain_norm, "cache": _plain_cache, "attend": _plain_attend, "prompt": _plain_prompt}[op](st)


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    hq, hkv, d = st["hq"], st["hkv"], st["d"]
    group = hq // hkv
    f64 = torch.float64

    def spun(x, positions):
        """Rows [n, heads, d] as complex numbers (i, i + d/2), turned by position x base^(-2 i / d)."""
        theta = torch.exp(torch.arange(d // 2, dtype=f64, device="cuda") * (-2.0 * math.log(st["base"]) / d))
        turn = torch.polar(torch.ones((), dtype=f64, device="cuda"), positions.to(f64)[:, None] * theta)[:, None]
        z = torch.complex(x[..., : d // 2].to(f64).contiguous(), x[..., d // 2:].to(f64).contiguous()) * turn
        return torch.cat((z.real, z.imag), dim=-1)

    def held(raw):
        """The values of pool rows [n, heads, 9 d / 8], from the bits of their codes and scales."""
        bits = torch.empty(*raw.shape[:2], 2 * d, dtype=torch.int64, device="cuda")
        bits[..., 0::2], bits[..., 1::2] = (raw[..., :d] % 16).long(), (raw[..., :d] // 16).long()
        exp, man = (bits // 2) % 4, bits % 2
        mag = torch.where(exp == 0, 0.5 * man.to(f64), (1.0 + 0.5 * man.to(f64)) * 2.0 ** (exp.to(f64) - 1.0))
        val = torch.where(bits >= 8, -mag, mag)
        sc = raw[..., d:].long()
        e, m = (sc // 8) % 16, (sc % 8).to(f64)
        sc = torch.where(e == 0, m * 2.0 ** -9, (1.0 + m / 8.0) * 2.0 ** (e.to(f64) - 7.0))
        return (val[..., :d] * sc[..., : d // BLOCK].repeat_interleave(BLOCK, -1),
                val[..., d:] * sc[..., d // BLOCK:].repeat_interleave(BLOCK, -1))

    if case["op"] == "norm":
        def unit(x, w):
            x = x.to(f64)
            return x / (x.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt() * w.to(f64)
        q, k = unit(st["q"], st["q_weight"]), unit(st["k"], st["k_weight"])
        return spun(q, st["positions"]), spun(k, st["positions"]), k
    if case["op"] == "cache":
        grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=f64, device="cuda")
        scales = [m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)][:127]
        scales = torch.tensor(scales, dtype=f64, device="cuda")
        borders = (scales[1:] + scales[:-1]) / 2.0

        def kept(x):
            b = x.to(f64).reshape(*x.shape[:2], d // BLOCK, BLOCK)
            want = (b.abs().max(-1).values / torch.tensor([6.0], dtype=f64, device="cuda")).clamp(max=448.0)
            i = torch.bucketize(want, borders)                          # the nearest scale; on a border the one with an even code
            s = scales[torch.where((want == borders[i.clamp(max=125)]) & (i % 2 == 1), i + 1, i)].unsqueeze(-1)
            r = torch.where(s > 0, b / s, torch.zeros_like(b)).abs().clamp(max=6.0)
            # the nearest level: the spacing is 1/2 below 2, 1 below 4, 2 above; round() takes ties to even
            step = torch.where(r < 2.0, 0.5, torch.where(r < 4.0, 1.0, 2.0))
            near = torch.round(r / step) * step
            assert torch.isin(near.reshape(-1)[:4096], grid).all()
            return (torch.sign(b) * near * s).reshape(x.shape)
        return kept(st["k"]), kept(st["v"])
    if case["op"] == "attend":
        outs = []
        for b, n in enumerate(lengths(case)):
            k, v = held(st["pool"][st["req_to_token"][b, :n].long()])
            k = spun(k, torch.arange(n, device="cuda"))
            q = spun(st["q"][b].view(1, hq, d), torch.tensor([n - 1], device="cuda"))[0]
            o = [torch.softmax((k[:, h // group] @ q[h]) * st["sm_scale"], dim=-1) @ v[:, h // group] for h in range(hq)]
            outs.append(torch.cat(o))
        return torch.stack(outs)
    out = torch.empty(*st["q"].shape, dtype=f64, device="cuda")
    a = 0
    for n in lengths(case):
        late = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
        for h in range(hq):
            s = (st["q"][a:a + n, h].to(f64) @ st["k"][a:a + n, h // group].to(f64).T) * st["sm_scale"]
            s.masked_fill_(late, -math.inf)
            out[a:a + n, h] = torch.softmax(s, dim=-1) @ st["v"][a:a + n, h // group].to(f64)
        a += n
    return out
