"""Head norms with rotation, and causal attention of packed prompts, on the GPU against plain 64-bit forms.

Tolerances.  A rounding to a type t is off by eps(t)/2 relative to the value at most.
Norm and rotation: fp32 inside.  The sum of D squares is off by (D/8 + 4) 2^-24 relative, its root by half that, the two
products by 2^-24 each, cosine and sine (from a position of 64 bits) by 2^-22 and the pair's two products and sum by 2^-23 of
their magnitudes: within 4e-6 (|y_i| + |y_{i+D/2}|) beyond doubt; in bf16 the fast cosine and sine are off by 2^-20, 1e-6 more
each, and the output is rounded once: 2^-8 |y|.
Attention in bf16: the inputs' products are exact in fp32; a logit's sum of D of them is off by D 2^-24 of sum |q k| (<= 2000 scaled
here: not more than 2e-2 of a unit in the worst order, 20 times less in fact; 1e-3 in a weight is allowed), weights are rounded to
bf16 (2^-8 each, of both signs), the output once (2^-8): |do| <= 2^-8 |o| + (2^-8 + 1e-3) sum p |v|.
Attention in fp32: 2e-4 sum p |v| covers logits off by 60 * 20 * 2^-24 as in the 4-bit attention's tests.
"""
import pytest
import torch

from tests import operators_ref as ref
from tokenselect_b200 import prompt, quant_cache as qc

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _near(got, want, tol):
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), f"max error {err.max():.3e}, {float((err / tol.clamp(min=1e-30)).max()):.2f} of the bound"


def _norm_tol(want, plain, dtype):
    pair = plain.abs() + plain.abs().roll(plain.shape[-1] // 2, -1)
    return (6e-6 * pair + 2.0 ** -8 * want.abs()) if dtype == BF16 else 4e-6 * pair


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("hq,hkv,d,n,first", [(32, 8, 128, 1, 130000), (28, 4, 128, 33, 0), (7, 1, 64, 5, 999990), (3, 3, 64, 257, 7), (1, 1, 128, 1, 0)])
def test_norm_and_rotation(hq, hkv, d, n, first, dtype):
    g = torch.Generator().manual_seed(n)
    qkv = (torch.randn(n, (hq + 2 * hkv) * d, generator=g) * 3).to(dtype)
    qw, kw = (1 + 0.3 * torch.randn(2, d, generator=g)).to(dtype).unbind(0)
    pos = torch.arange(first, first + n, dtype=torch.int32)
    dev = qkv.cuda()
    q, k = dev[:, :hq * d].view(n, hq, d), dev[:, hq * d:(hq + hkv) * d].view(n, hkv, d)
    qn, kn = ref.norm(q.cpu(), qw, 1e-6), ref.norm(k.cpu(), kw, 1e-6)
    a, b, c = prompt.norm_rotate(q, k, pos.cuda(), 5e5, 2.0, qw.cuda(), kw.cuda(), with_plain_k=True)
    wq, wk = ref.rotate(qn, pos, 5e5, 2.0), ref.rotate(kn, pos, 5e5, 2.0)
    _near(a, wq, _norm_tol(wq, qn, dtype))
    _near(b, wk, _norm_tol(wk, kn, dtype))
    _near(c, kn, _norm_tol(kn, kn, dtype))
    a, b = prompt.norm_rotate(q, k, None, q_weight=qw.cuda(), k_weight=kw.cuda())            # a decode step's: norms alone
    _near(a, qn, _norm_tol(qn, qn, dtype))
    _near(b, kn, _norm_tol(kn, kn, dtype))
    a, b = prompt.norm_rotate(q, k, pos.cuda(), 5e5, k_weight=kw.cuda())                      # one norm; the other only turned
    wq, wk = ref.rotate(q.cpu(), pos, 5e5), ref.rotate(kn, pos, 5e5)
    _near(a, wq, _norm_tol(wq, q.cpu().double(), dtype))
    _near(b, wk, _norm_tol(wk, kn, dtype))


def test_norm_in_place_unaligned_and_empty():
    g = torch.Generator().manual_seed(5)
    q, k = torch.randn(9, 4, 128, generator=g).to(BF16), torch.randn(9, 2, 128, generator=g).to(BF16)
    pos = torch.randint(0, 1000, (9,), generator=g).int()
    want = prompt.norm_rotate(q.cuda(), k.cuda(), pos.cuda(), 1e4)
    for offset in (0, 1):
        put = lambda t: torch.cat((torch.zeros(offset, dtype=t.dtype), t.flatten())).cuda()[offset:].view(t.shape)     # noqa: E731
        qi, ki = put(q), put(k)
        prompt.norm_rotate(qi, ki, pos.cuda(), 1e4, q_out=qi, k_out=ki)
        assert torch.equal(qi, want[0]) and torch.equal(ki, want[1])
    a, b = prompt.norm_rotate(q.cuda()[:0], k.cuda()[:0], pos.cuda()[:0])
    assert a.shape == (0, 4, 128) and b.shape == (0, 2, 128)
    neg = torch.tensor([-3], dtype=torch.int32)                                               # a position below zero turns back
    a, _ = prompt.norm_rotate(q.cuda()[:1], k.cuda()[:1], neg.cuda(), 1e4)
    w = ref.rotate(q[:1], neg, 1e4)
    _near(a, w, _norm_tol(w, q[:1].double(), BF16))


# ---------------------------------------------------------------------------------------------------------------------
def _prompt_case(seed, hq, hkv, d, lens, dtype, spare=0):
    g = torch.Generator().manual_seed(seed)
    n = sum(lens) + spare
    q, k, v = (torch.randn(n, h, d, generator=g) for h in (hq, hkv, hkv))
    k[:, :, torch.randperm(d, generator=g)[:4]] *= 8.0
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)
    return q.to(dtype), k.to(dtype), v.to(dtype), cu


def _check_prompt(q, k, v, cu, lens, sm_scale, cap=0.0):
    n, hq, d = q.shape
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full((n, hq, d), 7.0, dtype=q.dtype, device="cuda")
    prompt.prompt_attend(q.cuda(), k.cuda(), v.cuda(), cu.cuda(), sm_scale, cap, out=out, status=status)
    assert int(status) == 0
    used = sum(lens)
    want, mag = ref.attend(q[:used], k[:used], v[:used], ref.causal(lens, used), sm_scale, cap)
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 1e-3) * mag if q.dtype == BF16 else 2e-4 * mag
    _near(out[:used], want, tol)
    assert bool((out[used:] == 7.0).all())
    return out


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("hq,hkv,d,lens", [
    (4, 1, 128, [1]), (4, 2, 128, [128]), (4, 2, 128, [129]), (2, 1, 128, [255, 1, 257]), (7, 1, 128, [300]), (4, 4, 64, [200]),
    (8, 2, 64, [1, 2, 3, 63, 64, 65, 0, 0, 127, 5]), (2, 2, 128, [0, 17, 0]), (2, 1, 128, [640]), (14, 2, 128, [31, 130]), (2, 1, 64, [513, 100]),
], ids=str)
def test_packed_prompts(hq, hkv, d, lens, dtype):
    _check_prompt(*_prompt_case(len(lens) + hq, hq, hkv, d, lens, dtype, spare=5), lens, d ** -0.5)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
def test_prompts_with_soft_cap(dtype):
    _check_prompt(*_prompt_case(3, 4, 2, 128, [200, 70], dtype), [200, 70], 0.3, cap=4.0)


@pytest.mark.parametrize("d", [64, 128])
def test_a_long_prompt_row_by_row(d):
    """Rows of a prompt of many key blocks, those at the blocks' edges among them."""
    lens, hq, hkv = [3001], 4, 2
    q, k, v, cu = _prompt_case(9, hq, hkv, d, lens, BF16)
    k[1500] *= 4.0                                                            # a maximum that comes late
    out = prompt.prompt_attend(q.cuda(), k.cuda(), v.cuda(), cu.cuda(), d ** -0.5)
    rows = torch.tensor([0, 1, 127, 128, 129, 255, 256, 511, 512, 1499, 1500, 1501, 2047, 2048, 2999, 3000])
    seen = torch.arange(3001)[None] <= rows[:, None]
    want, mag = ref.attend(q[rows], k, v, seen, d ** -0.5)
    _near(out[rows.cuda()], want, 2.0 ** -8 * want.abs() + (2.0 ** -8 + 1e-3) * mag)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
def test_many_short_prompts(dtype):
    lens = [(5 * i) % 19 for i in range(300)]
    _check_prompt(*_prompt_case(13, 4, 1, 64, lens, dtype), lens, 0.125)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_what_is_not_finite_reaches_only_the_tokens_that_attend_to_it(bad, dtype):
    """An infinite or undefined key or value in the middle of one sequence: earlier tokens of it, other heads and the other
    sequences give what they gave without it."""
    lens, hq, hkv, d = [100, 333, 60], 4, 2, 128
    q, k, v, cu = _prompt_case(17, hq, hkv, d, lens, dtype)
    at, head = 100 + 270, 1
    good = prompt.prompt_attend(q.cuda(), k.cuda(), v.cuda(), cu.cuda(), 0.1)
    for which in ("k", "v"):
        k2, v2 = k.clone(), v.clone()
        (k2 if which == "k" else v2)[at, head, 5] = bad
        out = prompt.prompt_attend(q.cuda(), k2.cuda(), v2.cuda(), cu.cuda(), 0.1)
        touched = torch.zeros(sum(lens), hq, dtype=torch.bool)
        touched[at:433, 2:] = True                                            # KV head 1's query heads
        assert bool(torch.isfinite(out.cpu()[~touched]).all())
        tol = 1e-5 if dtype == F32 else 2.0 ** -7 * 8
        assert (out.cpu()[~touched].float() - good.cpu()[~touched].float()).abs().max() <= tol
        if which == "v" or bad != bad:
            assert not bool(torch.isfinite(out.cpu()[touched][:, 5]).any())


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
def test_an_infinite_value_of_the_next_sequence_or_of_a_later_token(dtype):
    """The block of keys at a sequence's end holds the next sequence's first values, the one on the diagonal those of later
    tokens: neither reaches a token that does not attend to them, and a long run of undefined values keeps the call's waits."""
    lens, hq, hkv, d = [200, 700, 3], 4, 2, 128
    q, k, v, cu = _prompt_case(31, hq, hkv, d, lens, dtype)
    good = prompt.prompt_attend(q.cuda(), k.cuda(), v.cuda(), cu.cuda(), 0.1)
    tol = 1e-5 if dtype == F32 else 2.0 ** -7 * 8
    for first, last in ((200, 201), (900, 903), (250, 900), (0, 1)):
        v2 = v.clone()
        v2[first:last] = float("inf")
        v2[first:last, :, ::2] = float("nan")
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = prompt.prompt_attend(q.cuda(), k.cuda(), v2.cuda(), cu.cuda(), 0.1, status=status).cpu()
        clean = torch.ones(903, dtype=torch.bool)
        for a, n in ((0, 200), (200, 700), (900, 3)):
            if a <= first < a + n:
                clean[first:a + n] = False
        assert int(status) == 0 and bool(torch.isfinite(out[clean]).all())
        assert (out[clean].float() - good.cpu()[clean].float()).abs().max() <= tol
        assert not bool(torch.isfinite(out[~clean]).any())


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
def test_maxima_that_jump(dtype):
    """A key whose logit is far above all before it, by what O follows (2^55), and by more than it could hold (2^700); at the
    start, inside and at the end of a block of keys."""
    n, hq, hkv, d, scale = 600, 2, 1, 128, 0.5
    q, k, v, cu = _prompt_case(37, hq, hkv, d, [n], F32)
    u = torch.randn(d, generator=torch.Generator().manual_seed(3))
    u *= 11.3137 / u.norm()                                                   # |u|^2 = 128
    q = (u + 0.1 * q).to(dtype)
    for at, factor in ((150, 0.6), (128, 8.0), (255, 8.0), (40, 8.0), (383, 0.6)):
        k2 = 0.05 * k
        k2[at] = u * factor
        _check_prompt(q, k2.to(dtype), v.to(dtype), cu, [n], scale)


def test_slices_of_a_projection_and_other_strides():
    hq, hkv, d, lens = 4, 2, 128, [77, 200]
    n = sum(lens)
    qkv = torch.randn(n, (hq + 2 * hkv) * d + 64).to(BF16).cuda()
    q, k, v = (qkv[:, a * d:b * d].view(n, -1, d) for a, b in ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv)))
    cu = torch.tensor([0, 77, 277], dtype=torch.int32, device="cuda")
    assert torch.equal(prompt.prompt_attend(q, k, v, cu, 0.1), prompt.prompt_attend(q.contiguous(), k.contiguous(), v.contiguous(), cu, 0.1))


def test_bounds_that_make_no_sense_are_reported():
    q, k, v, _ = _prompt_case(19, 2, 1, 128, [100], BF16)
    args = q.cuda(), k.cuda(), v.cuda()
    for cu in ([0, 50, 300], [-5, 50], [30, 20, 60]):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        prompt.prompt_attend(*args, torch.tensor(cu, dtype=torch.int32, device="cuda"), 0.1, status=status)
        assert int(status) == 7, cu
    for dtype in (BF16, F32):
        e = [t[:0].to(dtype) for t in args]
        assert prompt.prompt_attend(*e, torch.zeros(3, dtype=torch.int32, device="cuda"), 0.1).shape == (0, 2, 128)
        out = torch.full_like(args[0].to(dtype), 3.0)
        prompt.prompt_attend(*[t.to(dtype) for t in args], torch.zeros(1, dtype=torch.int32, device="cuda"), 0.1, out=out)
        assert bool((out == 3.0).all())


def test_offsets_beyond_31_bits():
    """The last tokens of tensors of more than 2^31 elements."""
    t, hq, hkv, d, n = 530000, 32, 1, 128, 100
    assert t * hq * d > 1 << 31
    small = _prompt_case(41, hq, hkv, d, [n], BF16)
    big = []
    for x in small[:3]:
        y = torch.empty(t, x.shape[1], d, dtype=BF16, device="cuda")
        y[-n:] = x.cuda()
        big.append(y)
    cu = torch.tensor([t - n, t], dtype=torch.int32, device="cuda")
    out = prompt.prompt_attend(*big, cu, 0.1)[-n:]
    assert torch.equal(out, prompt.prompt_attend(*[x.cuda() for x in small[:3]], small[3].cuda(), 0.1))
    pos = torch.arange(t, dtype=torch.int32, device="cuda")
    a, b = prompt.norm_rotate(big[0], big[1], pos, 5e5, q_out=big[0], k_out=big[1])
    wq = ref.rotate(small[0][-2:], pos[-2:].cpu(), 5e5)
    _near(a[-2:], wq, _norm_tol(wq, small[0][-2:].double(), BF16))
    assert torch.equal(b[-n:], prompt.norm_rotate(small[0].cuda(), small[1].cuda(), pos[-n:].contiguous(), 5e5)[1])


def test_prompt_attention_in_graphs_and_on_streams():
    q, k, v, cu = (t.cuda() for t in _prompt_case(23, 8, 2, 128, [300, 200], BF16))
    want = prompt.prompt_attend(q, k, v, cu, 0.1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = prompt.norm_rotate(q, k, None)
        res = prompt.prompt_attend(a, b, v, cu, 0.1)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        outs = [prompt.prompt_attend(q, k, v, cu, 0.1) for _ in range(5)]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(res, want) and all(torch.equal(o, want) for o in outs)
    cu.copy_(torch.tensor([0, 10, 500], dtype=torch.int32))
    graph.replay()
    assert torch.equal(res, prompt.prompt_attend(q, k, v, cu, 0.1))


@pytest.mark.parametrize("d", [128, 64])
def test_prompts_and_decode_steps_over_a_4bit_cache(d):
    """The operators together, as a layer uses them: norm and rotate the packed prompts' projections, attend, keep the un-rotated
    keys and the values in 4 bits; then decode steps that append their own row and attend to all rows of their request."""
    hq, hkv, base, lens, steps, eps = 8, 2, 5e5, [130, 1, 45], 3, 1e-6
    g = torch.Generator().manual_seed(29)
    total, scale = sum(lens), d ** -0.5
    qkv = torch.randn(total, (hq + 2 * hkv) * d, generator=g).to(BF16)
    qw, kw = (1 + 0.2 * torch.randn(2, d, generator=g)).to(BF16).unbind(0)
    new = torch.randn(steps, len(lens), (hq + 2 * hkv) * d, generator=g).to(BF16)
    pool_rows = total + steps * len(lens) + 11
    perm = torch.randperm(pool_rows, generator=g).int()
    pos = torch.cat([torch.arange(m) for m in lens]).int()
    cu = torch.tensor([0, 130, 131, 176], dtype=torch.int32)

    def split(x):
        n = x.shape[0]
        return x[:, :hq * d].view(n, hq, d), x[:, hq * d:(hq + hkv) * d].view(n, hkv, d), x[:, (hq + hkv) * d:].view(n, hkv, d)

    pool = qc.kv4_pool(pool_rows, hkv, d)
    q, k, v = split(qkv.cuda())
    qr, kr, kp = prompt.norm_rotate(q, k, pos.cuda(), base, q_weight=qw.cuda(), k_weight=kw.cuda(), eps=eps, with_plain_k=True)
    out = prompt.prompt_attend(qr, kr, v, cu.cuda(), scale)
    rows = perm[:total]
    qc.kv4_write(pool, kp, v, rows.cuda())
    want, mag = ref.attend(qr.cpu(), kr.cpu(), v.cpu(), ref.causal(lens, total), scale)
    _near(out, want, 2.0 ** -8 * want.abs() + (2.0 ** -8 + 1e-3) * mag)
    rtt = torch.zeros(4, max(lens) + steps, dtype=torch.int32)
    slots, a = torch.tensor([2, 0, 3], dtype=torch.int32), 0
    for s, m in zip(slots.tolist(), lens):
        rtt[s, :m] = rows[a:a + m]
        a += m
    store = {int(r): (kp[i].cpu(), v[i].cpu()) for i, r in enumerate(rows)}
    table = rtt.cuda()
    for t in range(steps):
        loc = perm[total + t * 3: total + t * 3 + 3]
        now = torch.tensor(lens) + t + 1
        table[slots.long().cuda(), (now - 1).cuda()] = loc.cuda()
        q, k, v = split(new[t].cuda())
        qn, kn = prompt.norm_rotate(q, k, None, q_weight=qw.cuda(), k_weight=kw.cuda(), eps=eps)
        qc.kv4_write(pool, kn, v, loc.cuda())
        out = qc.kv4_attend(qn.view(3, hq * d), pool, table, slots.cuda(), now.int().cuda(), scale, base)
        for b in range(3):
            store[int(loc[b])] = (kn[b].cpu(), v[b].cpu())
            n = int(now[b])
            kk, vv = (torch.stack([store[int(r)][i] for r in table[slots[b], :n].cpu()]) for i in (0, 1))
            kh, vh = ref.held(kk), ref.held(vv)
            qq = ref.rotate(qn[b:b + 1].cpu(), torch.tensor([n - 1]), base)
            o, m = ref.attend(qq, ref.rotate(kh, torch.arange(n), base), vh, torch.ones(1, n, dtype=torch.bool), scale)
            pair = (kh.abs() + kh.abs().roll(d // 2, -1))[:, torch.arange(hq) // (hq // hkv)]
            e = 6 * 5 * 2.0 ** -11 * scale * ((qq * pair) ** 2).sum(-1).sqrt().amax(0)
            _near(out[b].view(1, hq, d), o, 2.0 ** -8 * o.abs() + (torch.exp(2 * e)[:, None] - 1 + 2.0 ** -10) * m)


def _matches(out, want, mag):
    """Finite where the 64-bit form is, and near it there."""
    out, fine = out.cpu().double(), torch.isfinite(want)
    assert torch.equal(torch.isfinite(out), fine), f"{int((torch.isfinite(out) != fine).sum())} elements finite that should not be, or not that should"
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 1e-3) * mag
    assert bool(((out - want).abs() <= tol)[fine].all())


@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("d", [64, 128])
def test_an_undefined_key_at_any_place_reaches_every_later_token(d, cap):
    """A NaN in a key makes every token from it on undefined, whatever its place in its block of keys and however many
    blocks later the token comes; earlier tokens, the other head and the other sequence do not see it."""
    lens, hq, hkv = [30, 520], 2, 2
    q, k, v, cu = _prompt_case(43, hq, hkv, d, lens, BF16)
    for at in (0, 1, 2, 3, 4, 5, 6, 7, 30, 95, 127, 134, 383):
        k2 = k.clone()
        k2[30 + at, 1, at % d] = float("nan")
        out = prompt.prompt_attend(q.cuda(), k2.cuda(), v.cuda(), cu.cuda(), 0.1, cap).cpu()
        seen = torch.zeros(550, hq, dtype=torch.bool)
        seen[30 + at:, 1] = True
        assert bool(torch.isfinite(out[~seen]).all()), at
        assert not bool(torch.isfinite(out[seen]).any()), (at, int(torch.isfinite(out[seen]).sum()))


@pytest.mark.parametrize("d", [64, 128])
def test_infinite_keys_give_what_the_softmax_gives(d):
    """An infinite key gives a logit of plus infinity (the softmax is undefined), of minus infinity (a weight of zero) or, where
    two infinities meet, none; a token all of whose logits are minus infinity has no softmax either."""
    n, hq, hkv = 400, 2, 1
    q, k, v, cu = _prompt_case(47, hq, hkv, d, [n], BF16)
    one, two, all_ = k.clone(), k.clone(), k.clone()
    one[6, 0, 5] = float("inf")
    two[7, 0, 5], two[7, 0, 6] = float("inf"), -float("inf")
    all_[:, 0, 5] = -float("inf")
    for k2 in (one, two, all_):
        out = prompt.prompt_attend(q.cuda(), k2.cuda(), v.cuda(), cu.cuda(), d ** -0.5)
        _matches(out, *ref.attend(q, k2, v, ref.causal([n], n), d ** -0.5))


@pytest.mark.parametrize("d", [64, 128])
def test_columns_that_become_undefined_one_after_the_other(d):
    """Values that are not finite, each in a column of its own, in the same block of keys and in later ones, before and behind
    the tokens of a block, with keys far above the others among them: every column of every token is finite where the tokens
    it sees are."""
    lens, hq, hkv = [700, 150], 4, 2
    q, k, v, cu = _prompt_case(53, hq, hkv, d, lens, BF16)
    k[260, 0] *= 40.0                                                         # logits that jump for some queries
    for at, col, x in ((10, 3, "nan"), (300, 7, "inf"), (390, 9, "-inf"), (391, 9, "inf"), (511, 3, "inf"), (512, 40, "nan"), (640, 11, "nan"), (699, 50, "inf"),
                       (701, 5, "nan"), (849, 6, "inf")):
        v[at, :, col] = float(x)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = prompt.prompt_attend(q.cuda(), k.cuda(), v.cuda(), cu.cuda(), 0.1, status=status)
    assert int(status) == 0
    _matches(out, *ref.attend(q, k, v, ref.causal(lens, 850), 0.1))


@pytest.mark.parametrize("columns", [slice(None), slice(5, 6)], ids=["all", "one"])
def test_an_early_undefined_value_does_not_hold_the_call_up(columns):
    """An undefined value at the start of a long prompt makes every later token undefined, with cause: no more than a block's
    tokens are computed again.  (One value after the other on a warp, they would take two hundred times the clean call's time.)"""
    n, hq, hkv, d = 16384, 8, 1, 128
    g = torch.Generator(device="cuda").manual_seed(5)
    q, k, v = (torch.randn(n, h, d, generator=g, device="cuda").to(BF16) for h in (hq, hkv, hkv))
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    v2 = v.clone()
    v2[3, :, columns] = float("nan")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    took = []
    for x in (v, v2):
        times = []
        for _ in range(4):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            out = prompt.prompt_attend(q, k, x, cu, d ** -0.5, status=status)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        took.append(min(times))
    bad = torch.zeros(n, hq, d, dtype=torch.bool, device="cuda")
    bad[3:, :, columns] = True
    assert int(status) == 0 and torch.equal(~torch.isfinite(out), bad)
    assert took[1] <= 10 * took[0], took


def _in_order(cu, tokens):
    """Bounds that give the sequences that are left of `cu`: each ends where it still does, behind all before it."""
    got, high = [], 0
    for x in cu:
        high = max(high, min(max(x, 0), tokens))
        got.append(high)
    return got


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
def test_sequences_of_bounds_out_of_order_share_no_token(dtype):
    """A bound below one before it, or outside the tokens, ends its sequence; the next one starts behind all before it, so no token
    is written twice and none of a sequence's tokens is left out.  Sequences by the dozen, over the edges of what a warp looks
    at together, among them."""
    g = torch.Generator().manual_seed(59)
    q, k, v, _ = _prompt_case(59, 4, 2, 64, [500], dtype)
    args = [t.cuda() for t in (q, k, v)]
    cases = [[0, 100, 50, 200], [0, 50, 900], [-5, 50, 500], [30, 20, 60], [0, 90, 10, 80, 200, 150, 300, 299, 500], [500, 0, 500], [100, 0, 100, 0, 500, 0, 500]]
    cases += [torch.randint(-50, 600, (n,), generator=g).tolist() for n in (33, 34, 70, 300)]
    ordered = torch.randint(0, 501, (300,), generator=g).sort()[0]
    for at in (31, 32, 33, 64, 200, 299):
        case = ordered.clone()
        case[at] = int(case[at - 1]) - 40
        cases.append(case.tolist())
    for case in cases:
        good = _in_order(case, 500)
        outs = []
        for cu in (case, good):
            status = torch.zeros(1, dtype=torch.int32, device="cuda")
            out = torch.full_like(args[0], 7.0)
            prompt.prompt_attend(*args, torch.tensor(cu, dtype=torch.int32, device="cuda"), 0.1, out=out, status=status)
            assert int(status) == (7 if cu != good else 0), case
            outs.append(out)
        assert torch.equal(outs[0], outs[1]), case
        assert bool((outs[0][:good[0]] == 7.0).all()) and bool((outs[0][good[-1]:] == 7.0).all()) and not bool((outs[0][good[0]:good[-1]] == 7.0).any())


@pytest.mark.parametrize("d", [64, 128])
def test_infinite_keys_in_fp32(d):
    """The check mode gives the same: undefined, a weight of zero, or no softmax at all."""
    n, hq, hkv = 200, 2, 1
    q, k, v, cu = _prompt_case(61, hq, hkv, d, [n], F32)
    one, two, all_ = k.clone(), k.clone(), k.clone()
    one[6, 0, 5] = float("inf")
    two[70, 0, 5], two[70, 0, 6] = float("inf"), -float("inf")
    all_[:, 0, 5] = -float("inf")
    for k2 in (one, two, all_):
        out = prompt.prompt_attend(q.cuda(), k2.cuda(), v.cuda(), cu.cuda(), d ** -0.5)
        _matches(out, *ref.attend(q, k2, v, ref.causal([n], n), d ** -0.5))


def test_a_captured_decode_step_over_a_4bit_cache():
    """Norm, rows written, attention and rows read back in one graph: a replay follows new contents of every input, and gives
    what the calls give one by one."""
    hq, hkv, d, base, batch = 8, 2, 128, 5e5, 3
    g = torch.Generator().manual_seed(71)
    qkv = torch.randn(batch, (hq + 2 * hkv) * d, generator=g).to(BF16).cuda()
    q, k, v = (qkv[:, a * d:b * d].view(batch, -1, d) for a, b in ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv)))
    w = torch.ones(d, dtype=BF16, device="cuda")
    start = torch.randint(0, 120, (200, hkv, qc.kv4_row_bytes(d)), dtype=torch.uint8, generator=g).cuda()      # (no NaN scale)
    table = torch.randperm(200, generator=g).int().view(1, 200).expand(batch, 200).cuda()
    loc, lens, slots = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([5, 6, 7], [17, 200, 33], [2, 0, 1]))

    def step(pool):
        qn, kn = prompt.norm_rotate(q, k, None, q_weight=w, k_weight=w)
        qc.kv4_write(pool, kn, v, loc)
        out = qc.kv4_attend(qn.view(batch, hq * d), pool, table, slots, lens, 0.1, base)
        return (out, *qc.kv4_read(pool, loc))

    step(start.clone())
    pool = start.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step(pool)
    for turn in range(3):
        qkv.copy_(torch.randn(qkv.shape, generator=g).to(BF16))
        loc.copy_(torch.tensor([9 + turn, 50 + turn, 80 + turn], dtype=torch.int32))
        lens.copy_(torch.tensor([1 + turn, 0, 190 + turn], dtype=torch.int32))
        pool.copy_(start)
        graph.replay()
        other = start.clone()
        assert all(torch.equal(a, b) for a, b in zip(res, step(other))) and torch.equal(pool, other)
