"""The 4-bit cache on the GPU: rows written and read back, and decode attention over them, against plain 64-bit forms.

Tolerances of the attention.  A rounding to a type t is off by eps(t)/2 relative to the value at most.
bf16: the output's own rounding, 2^-8 |o|.  The rotated query is rounded to fp16 once (2^-11), a rotated key's element is
made of two products of a value with a cosine or sine rounded to fp16, one of them rounded, and their rounded sum: at most
four roundings of 2^-11 of (|k_i| + |k_{i+D/2}|).  These 5 errors per element are independent of each other and of
the next element's, so a logit is off by e = 6 * 5 * 2^-11 * scale * sqrt(sum q^2 (|k_i| + |k_{i+D/2}|)^2) beyond doubt (six
times the sum in quadrature of worst cases); weights are off by a factor e^(2 e) and by their own fp16 rounding 2^-11, in
the sum and above it: |do| <= (e^(2 e) - 1 + 2^-10) * sum p |v|.
fp32: a logit's D products and sums and the rotations are each off by 2^-24 of sum |q k| (1 + sqrt D + 8 beyond doubt),
angles by 2^-23, the exponential by 2^-22: with sum |q k| scale <= 60 here e <= 60 * 20 * 2^-24 = 7.2e-5, so the weights are off by 1.5e-4
at most; the test's factor is 2e-4.
"""
import pytest
import torch

from tests import operators_ref as ref
from tokenselect_b200 import quant_cache as qc

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _rows(seed, n, heads, d, dtype, loud=4):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, heads, d, generator=g)
    x[:, :, torch.randperm(d, generator=g)[:loud]] *= 8.0
    return x.to(dtype)


@pytest.mark.parametrize("heads,d,n,dtype", [(8, 128, 1, BF16), (8, 128, 33, BF16), (4, 128, 257, F32), (1, 64, 65, BF16), (3, 64, 7, F32),
                                             (5, 128, 100, BF16)])
@pytest.mark.parametrize("gk,gv", [(1.0, 1.0), (0.25, 8.0)])
def test_rows_written_and_read_back_are_exact(heads, d, n, dtype, gk, gv):
    """Codes, scales and values are decided exactly, borders included; other rows of the pool stay as they were."""
    k, v = _rows(n, n, heads, d, dtype), _rows(n + 1, n, heads, d, dtype, 0) * 0.3
    v = v.to(dtype)
    # ties: values halfway between two levels of a block whose largest element fixes the scale at 1
    k[0, 0, :16] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, 0.0]) * gk
    v[0, 0, :16] = 0.0                                                        # an empty block
    pool = torch.randint(0, 256, (n + 50, heads, qc.kv4_row_bytes(d)), dtype=torch.uint8)
    rows = torch.randperm(n + 50)[:n].int()
    dev = pool.cuda()
    qc.kv4_write(dev, k.cuda(), v.cuda(), rows.cuda(), gk, gv)
    want = pool.clone()
    want[rows.long()] = ref.pack(k, v, gk, gv)
    got = dev.cpu()
    gk_, gv_ = ref.unpack(got[rows.long()], gk, gv)
    wk, wv = ref.unpack(want[rows.long()], gk, gv)
    assert torch.equal(gk_, wk) and torch.equal(gv_, wv)
    keep = torch.ones(n + 50, dtype=torch.bool)
    keep[rows.long()] = False
    assert torch.equal(got[keep], pool[keep])
    for out in (BF16, F32):
        rk, rv = qc.kv4_read(dev, rows.cuda(), out, gk, gv)
        assert torch.equal(rk.cpu().double(), wk) and torch.equal(rv.cpu().double(), wv)
    again = torch.zeros_like(dev)                                             # a row read back keeps its codes
    qc.kv4_write(again, rk, rv, rows.cuda(), gk, gv)
    ak, av = qc.kv4_read(again, rows.cuda(), F32, gk, gv)
    assert torch.equal(ak.cpu().double(), wk) and torch.equal(av.cpu().double(), wv)


def test_every_border_is_decided_exactly():
    """Every scale with every border of the codes times it, and the fp32 and bf16 values next to them on both sides."""
    for dtype in (F32, BF16):
        blocks = []
        for s in ref.SCALES[1:]:
            mids = torch.tensor(ref.BORDERS, dtype=F32) * s
            near = torch.cat((mids, torch.nextafter(mids, torch.zeros(())), torch.nextafter(mids, torch.full((), 1e9))))
            if dtype is BF16:
                b = mids.to(BF16)
                i = b.view(torch.int16)
                near = torch.cat((b, (i - 1).view(BF16), (i + 1).view(BF16))).float()
            for part in near.split(15):
                x = torch.zeros(16)
                x[0] = 6.0 * s
                x[1:1 + len(part)] = part
                blocks.append(x.to(dtype))
        # scales next to their own borders
        sc = torch.tensor(ref.SCALES, dtype=F32)
        mid = (sc[1:] + sc[:-1]) / 2 * 6.0
        for m in torch.cat((mid, torch.nextafter(mid, torch.zeros(())), torch.nextafter(mid, torch.full((), 1e9)), torch.tensor([2700.0, 1e9, 3e38, 1e-30]))):
            x = torch.randn(16) * m / 8
            x[3] = -m
            blocks.append(x.clamp(-m.abs(), m.abs()).to(dtype))
        n = len(blocks) // 8 * 8
        x = torch.stack(blocks[:n]).view(-1, 1, 128)
        pool = qc.kv4_pool(x.shape[0], 1, 128)
        rows = torch.arange(x.shape[0], dtype=torch.int32, device="cuda")
        qc.kv4_write(pool, x.cuda(), x.flip(0).contiguous().cuda(), rows)
        k, v = qc.kv4_read(pool, rows, F32)
        assert torch.equal(k.cpu().double(), ref.held(x)) and torch.equal(v.cpu().double(), ref.held(x.flip(0)))


def test_infinite_and_nan_blocks_read_back_as_nan():
    k = _rows(3, 4, 2, 128, BF16)
    v = k.clone()
    k[1, 0, 17], k[2, 1, 0], v[3, 1, 127] = float("inf"), float("nan"), -float("inf")
    pool, rows = qc.kv4_pool(4, 2, 128), torch.arange(4, dtype=torch.int32, device="cuda")
    qc.kv4_write(pool, k.cuda(), v.cuda(), rows)
    a, b = qc.kv4_read(pool, rows)
    assert torch.equal(a.isnan().cpu(), ref.held(k).isnan()) and torch.equal(b.isnan().cpu(), ref.held(v).isnan())
    assert int(a.isnan().sum()) == 32 and int(b.isnan().sum()) == 16
    assert torch.equal(torch.nan_to_num(a).cpu().double(), torch.nan_to_num(ref.held(k)))


def test_strided_and_unaligned_rows():
    """Slices of a fused projection's output, and rows that start at any element."""
    heads, d, n = 2, 128, 9
    for offset in (0, 1, 8):
        flat = torch.randn(n * 6 * heads * d + offset).to(BF16).cuda()[offset:]
        qkv = flat.view(n, 6 * heads * d)
        k, v = qkv[:, 2 * heads * d:3 * heads * d].view(n, heads, d), qkv[:, 3 * heads * d:4 * heads * d].view(n, heads, d)
        pool, rows = qc.kv4_pool(n, heads, d), torch.randperm(n).int().cuda()
        qc.kv4_write(pool, k, v, rows)
        big = torch.full((n, 3, heads, d), 7.0, dtype=BF16, device="cuda")
        qc.kv4_read(pool, rows, k=big[:, 0], v=big[:, 2])
        assert torch.equal(big[:, 0].cpu().double(), ref.held(k.cpu())) and torch.equal(big[:, 2].cpu().double(), ref.held(v.cpu()))
        assert bool((big[:, 1] == 7.0).all())


def test_rows_outside_the_pool_are_skipped_and_reported():
    heads, d = 2, 64
    k, v = _rows(5, 4, heads, d, BF16), _rows(6, 4, heads, d, BF16)
    rows = torch.tensor([2, -1, 10, 0], dtype=torch.int32).cuda()
    pool, status = qc.kv4_pool(10, heads, d), torch.zeros(1, dtype=torch.int32, device="cuda")
    qc.kv4_write(pool, k.cuda(), v.cuda(), rows, status=status)
    assert int(status) == 6
    status.zero_()
    a, b = qc.kv4_read(pool, rows, status=status)
    assert int(status) == 6
    ok = torch.tensor([True, False, False, True])
    assert torch.equal(a.cpu().double()[ok], ref.held(k)[ok]) and torch.equal(b.cpu().double()[ok], ref.held(v)[ok])
    assert not a[1:3].any() and not b[1:3].any() and not pool[[1, 3, 4, 5, 6, 7, 8, 9]].any()
    qc.kv4_write(pool, k.cuda()[:0], v.cuda()[:0], rows[:0])                  # nothing to do


# ---------------------------------------------------------------------------------------------------------------------
def _attend_case(seed, hq, hkv, d, lens, dtype, spare=3):
    g = torch.Generator().manual_seed(seed)
    n = sum(lens) + spare
    pool = ref.pack(_rows(seed + 1, n, hkv, d, dtype), _rows(seed + 2, n, hkv, d, dtype, 0))
    perm = torch.randperm(n, generator=g).int()
    ctx = max(max(lens), 1) + 5
    rtt = torch.full((len(lens) + 2, ctx), 10 ** 8, dtype=torch.int32)        # entries behind a request's end are never read
    slots = torch.randperm(len(lens) + 2, generator=g)[: len(lens)].int()
    a = 0
    for s, m in zip(slots.tolist(), lens):
        rtt[s, :m] = perm[a:a + m]
        a += m
    q = torch.randn(len(lens), hq * d, generator=g).to(dtype)
    return q, pool, rtt, slots, torch.tensor(lens, dtype=torch.int32)


def _attend_ref(q, pool, rtt, slots, lens, hq, sm_scale, base, scale=1.0, cap=0.0, gk=1.0, gv=1.0):
    """Outputs [batch, hq, D] and the bound of their error that the head of this file derives."""
    d = pool.shape[-1] * 8 // 9
    outs, tols = [], []
    group = hq // pool.shape[1]
    for b, n in enumerate(lens.tolist()):
        if n == 0:
            outs.append(torch.zeros(hq, d, dtype=ref.F64))
            tols.append(torch.zeros(hq, d, dtype=ref.F64))
            continue
        k, v = ref.unpack(pool[rtt[slots[b], :n].long()], gk, gv)
        kr = ref.rotate(k, torch.arange(n), base, scale)
        qr = ref.rotate(q[b].view(1, hq, d), torch.tensor([n - 1]), base, scale)
        o, mag = ref.attend(qr, kr, v, torch.ones(1, n, dtype=torch.bool), sm_scale, cap)
        if q.dtype == BF16:
            pair = (k.abs() + k.abs().roll(d // 2, -1))[:, torch.arange(hq) // group]          # [n, hq, D]
            e = 6 * 5 * 2.0 ** -11 * sm_scale * ((qr * pair) ** 2).sum(-1).sqrt().amax(0)       # [hq]
            tol = 2.0 ** -8 * o[0].abs() + (torch.exp(2 * e)[:, None] - 1 + 2.0 ** -10) * mag[0]
        else:
            tol = 2e-4 * mag[0]
        outs.append(o[0])
        tols.append(tol)
    return torch.stack(outs), torch.stack(tols)


def _check_attend(case, hq, sm_scale, base, **kw):
    q, pool, rtt, slots, lens = case
    names = {"scale": "rope_scale", "cap": "logit_cap", "gk": "k_scale", "gv": "v_scale"}
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = qc.kv4_attend(q.cuda(), pool.cuda(), rtt.cuda(), slots.cuda(), lens.cuda(), sm_scale, base, status=status,
                        **{names[k]: v for k, v in kw.items()})
    assert int(status) == 0
    want, tol = _attend_ref(q, pool, rtt, slots, lens, hq, sm_scale, base, **kw)
    err = (out.cpu().double().view_as(want) - want).abs()
    assert bool((err <= tol).all()), f"max error {err.max():.3e}, {float((err / tol.clamp(min=1e-30)).max()):.2f} of the bound"
    return out


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("hq,hkv,d,lens", [
    (32, 8, 128, [1]), (32, 8, 128, [700]), (28, 4, 128, [1, 2, 15, 16, 17, 31, 33, 64, 65, 127, 300]), (8, 1, 128, [129, 0, 1000]),
    (7, 1, 128, [513]), (4, 4, 128, [77, 200]), (6, 3, 128, [40, 5]), (8, 2, 64, [1, 16, 100, 333]), (3, 3, 64, [18]), (5, 1, 64, [64, 0, 0, 63]),
    (16, 16, 128, [90]), (40, 20, 64, [50, 3]), (9, 9, 64, [70, 5]), (11, 11, 128, [40, 90]), (12, 6, 64, [100]), (8, 1, 128, [3000, 17]),
    (5, 1, 64, [2500]), (14, 2, 128, [1500, 0, 700]),
], ids=str)
def test_attention_over_a_4bit_pool(hq, hkv, d, lens, dtype):
    _check_attend(_attend_case(hq + d + len(lens), hq, hkv, d, lens, dtype), hq, d ** -0.5, 5e5)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("kw", [{"cap": 5.0}, {"scale": 4.0}, {"gk": 0.25, "gv": 16.0}], ids=str)
def test_attention_options(kw, dtype):
    _check_attend(_attend_case(11, 8, 2, 128, [150, 31], dtype), 8, 128 ** -0.5, 1e4, **kw)


def test_attention_of_a_long_request_and_many_short_ones():
    """Pieces that hold many requests, and a request over many pieces."""
    _check_attend(_attend_case(21, 8, 2, 128, [9000] + [(7 * i) % 23 for i in range(300)], BF16), 8, 128 ** -0.5, 5e5)


@pytest.mark.parametrize("hq,hkv,d,lens", [(2, 1, 128, [150000]), (4, 2, 128, [70000, 50001]), (4, 2, 64, [110000]), (5, 5, 64, [60000]),
                                           (6, 3, 128, [40000, 40007])])
def test_rings_of_every_width_go_round(hq, hkv, d, lens):
    """Enough rows that every CTA fills its stages several times, however many a row's width leaves room for."""
    _check_attend(_attend_case(25, hq, hkv, d, lens, BF16), hq, d ** -0.5, 5e5)


def test_queries_of_any_size_and_alignment():
    """fp16 holds the rotated query whatever its size: it is scaled by a power of two."""
    case = list(_attend_case(31, 8, 2, 128, [100, 40], BF16))
    q = case[0]
    for factor in (1e-6, 1e4):
        scale = 128 ** -0.5 / factor
        case[0] = (q.float() * factor).to(BF16)
        _check_attend(case, 8, scale, 5e5)
    flat = torch.zeros(q.numel() + 1, dtype=BF16, device="cuda")
    flat[1:] = q.flatten().cuda()
    _, pool, rtt, slots, lens = case
    args = (pool.cuda(), rtt.cuda(), slots.cuda(), lens.cuda(), 128 ** -0.5, 5e5)
    odd = torch.zeros(q.numel() + 1, dtype=BF16, device="cuda")[1:].view(q.shape)
    qc.kv4_attend(flat[1:].view(q.shape), *args, out=odd)
    assert torch.equal(odd, qc.kv4_attend(q.cuda(), *args))


def test_bad_rows_lengths_and_slots_are_reported():
    hq, hkv, d = 8, 2, 128
    q, pool, rtt, slots, lens = _attend_case(41, hq, hkv, d, [50, 60, 70, 80], BF16)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    good = qc.kv4_attend(q.cuda(), pool.cuda(), rtt.cuda(), slots.cuda(), lens.cuda(), 0.1, 5e5)
    lens2, slots2 = lens.clone(), slots.clone()
    lens2[0], lens2[2], slots2[3] = -5, rtt.shape[1] + 1, 99
    out = qc.kv4_attend(q.cuda(), pool.cuda(), rtt.cuda(), slots2.cuda(), lens2.cuda(), 0.1, 5e5, status=status)
    assert int(status) == 7 and not out[[0, 2, 3]].any() and torch.equal(out[1], good[1])
    status.zero_()
    rtt2 = rtt.clone()
    rtt2[slots[1], 13], rtt2[slots[1], 59] = pool.shape[0], -7
    out = qc.kv4_attend(q.cuda(), pool.cuda(), rtt2.cuda(), slots.cuda(), lens.cuda(), 0.1, 5e5, status=status)
    assert int(status) == 6 and torch.equal(out[[0, 2, 3]], good[[0, 2, 3]])
    # a row outside the pool counts as zeros
    more = torch.cat((pool, torch.zeros_like(pool[:1])))
    rtt2[slots[1], 59] = pool.shape[0]
    want, tol = _attend_ref(q, more, rtt2, slots, lens, hq, 0.1, 5e5)
    assert bool(((out.cpu().double().view_as(want) - want).abs() <= tol).all())


def test_nan_stays_in_its_request_and_empty_batches_are_calls_like_any_other():
    hq, hkv, d = 8, 2, 128
    q, pool, rtt, slots, lens = _attend_case(51, hq, hkv, d, [50, 60], BF16)
    good = qc.kv4_attend(q.cuda(), pool.cuda(), rtt.cuda(), slots.cuda(), lens.cuda(), 0.1, 5e5)
    row = int(rtt[slots[0], 49])
    pool[row, 1, 128] = 0x7F                                                  # a K scale of head 1
    out = qc.kv4_attend(q.cuda(), pool.cuda(), rtt.cuda(), slots.cuda(), lens.cuda(), 0.1, 5e5)
    assert torch.equal(out[1], good[1]) and torch.equal(out[0, :512], good[0, :512]) and bool(out[0, 512:].isnan().all())
    empty = qc.kv4_attend(q.cuda()[:0], pool.cuda(), rtt.cuda(), slots.cuda()[:0], lens.cuda()[:0], 0.1, 5e5)
    assert empty.shape == (0, hq * d)


def test_selected_lists_are_attended_to_like_the_engine_does():
    """The row list that a selection leaves, over a 4-bit copy of the pool, against the bf16 attention over what it holds."""
    from oracle import synth
    from tests import gpu_util as gu
    hq, hkv, d, n_init, n_local, k = 8, 2, 128, 16, 64, 256
    eng = gu.make_engine(hq, hkv, d, n_init, n_local, k, 5e5, BF16, max_ctx=4096)
    case = synth.make_layer_case(71, 3000, hq, hkv, d, n_init, n_local, 5e5, dtype=BF16)
    q, kp, vp, rtt, ridx, lens = gu.case_tensors(case)
    pool = qc.kv4_pool(kp.shape[0], hkv, d)
    every = torch.arange(kp.shape[0], dtype=torch.int32, device="cuda")
    qc.kv4_write(pool, kp.cuda(), vp.cuda(), every)
    kd, vd = qc.kv4_read(pool, every)
    want, res = gu.run_gpu(eng, 0, q, kd.cpu(), vd.cpu(), rtt, ridx, lens)
    got = qc.kv4_attend(q.cuda(), pool, res["slots"].cuda(), torch.zeros(1, dtype=torch.int32, device="cuda"), res["count"].cuda(), d ** -0.5, 5e5)
    assert (got.float().cpu() - want.float()).abs().max().item() <= 2e-2      # the framework's tolerance between its attentions


def test_streams_graphs_and_workspaces():
    """Calls on two streams at once and two captured graphs replayed at once have workspaces of their own; a captured call
    follows new contents of its inputs, lengths included."""
    hq, hkv, d = 32, 8, 128
    a, b = _attend_case(61, hq, hkv, d, [900, 41], BF16), _attend_case(62, hq, hkv, d, [333, 1000], BF16)
    on = [[t.cuda() for t in c] for c in (a, b)]
    want = [qc.kv4_attend(*c, 0.1, 5e5) for c in on]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in on]
    outs = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(qc.kv4_attend(*on[i], 0.1, 5e5))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in (0, 1) for o in outs[i])
    graphs, res = [], []
    for i in (0, 1):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res.append(qc.kv4_attend(*on[i], 0.1, 5e5))
        graphs.append(g)
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                graphs[i].replay()
    torch.cuda.synchronize()
    assert torch.equal(res[0], want[0]) and torch.equal(res[1], want[1])
    on[0][4].copy_(torch.tensor([17, 0], dtype=torch.int32))
    on[0][0].mul_(0.5)
    graphs[0].replay()
    assert torch.equal(res[0], qc.kv4_attend(*on[0], 0.1, 5e5)) and not res[0][1].any()
    own = torch.empty(qc.kv4_attend_workspace(2, hq, d), dtype=torch.uint8, device="cuda")
    assert torch.equal(qc.kv4_attend(*on[1], 0.1, 5e5, workspace=own), want[1])


def test_offsets_beyond_32_bits():
    """Rows of a pool of more than 4 GiB, by their first and last row."""
    heads, d = 8, 128
    n = (1 << 32) // (heads * qc.kv4_row_bytes(d)) + 1000
    pool = qc.kv4_pool(n, heads, d)
    k, v = _rows(7, 5, heads, d, BF16), _rows(8, 5, heads, d, BF16)
    rows = torch.tensor([0, n - 1, n - 2, n // 2, n - 900], dtype=torch.int32)
    qc.kv4_write(pool, k.cuda(), v.cuda(), rows.cuda())
    a, b = qc.kv4_read(pool, rows.cuda())
    assert torch.equal(a.cpu().double(), ref.held(k)) and torch.equal(b.cpu().double(), ref.held(v))
    q = torch.randn(1, 32 * d).to(BF16)
    small = ref.pack(k, v)
    lens = torch.tensor([5], dtype=torch.int32)
    zero = torch.zeros(1, dtype=torch.int32)
    for dtype in (BF16, F32):
        out = qc.kv4_attend(q.to(dtype).cuda(), pool, rows[None].cuda(), zero.cuda(), lens.cuda(), d ** -0.5, 5e5)
        want, tol = _attend_ref(q.to(dtype), small, torch.arange(5)[None].int(), zero, lens, 32, d ** -0.5, 5e5)
        assert bool(((out.cpu().double().view_as(want) - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
def test_far_positions_turn_by_exact_angles(dtype):
    """A list of 300001 rows of which all but 64 hold zeros: the 64 must be turned as far as they are.  (An angle computed in
    fp32 would be off by up to 300000 * 2^-24 = 0.018, which moves logits of this size by more than the bound allows.)"""
    hq, hkv, d, n, scale = 4, 1, 128, 300001, 0.3
    k, v = _rows(9, 64, hkv, d, F32), _rows(10, 64, hkv, d, F32)
    pool = torch.cat((ref.pack(k, v), torch.zeros(1, hkv, qc.kv4_row_bytes(d), dtype=torch.uint8)))
    at = torch.cat((torch.randperm(n - 1, generator=torch.Generator().manual_seed(1))[:63], torch.tensor([n - 1])))
    table = torch.full((1, n), 64, dtype=torch.int32)
    table[0, at] = torch.arange(64, dtype=torch.int32)
    q = torch.randn(1, hq * d, generator=torch.Generator().manual_seed(2)).to(dtype)
    kh, vh = ref.unpack(pool[:64])
    kr, qr = ref.rotate(kh, at, 1e4), ref.rotate(q.view(1, hq, d), torch.tensor([n - 1]), 1e4)
    s = torch.einsum("hd,jd->hj", qr[0], kr[:, 0]) * scale
    top = s.amax(1, keepdim=True).clamp(min=0)
    w, rest = torch.exp(s - top), (n - 64) * torch.exp(-top)
    want = (w @ vh[:, 0]) / (w.sum(1, keepdim=True) + rest)
    mag = (w @ vh[:, 0].abs()) / (w.sum(1, keepdim=True) + rest)
    pair = (kh.abs() + kh.abs().roll(d // 2, -1))                            # [64, 1, D], broadcast over the heads
    if dtype == BF16:
        e = 6 * 5 * 2.0 ** -11 * scale * ((qr * pair) ** 2).sum(-1).sqrt().amax(0)[:, None]
        tol = 2.0 ** -8 * want.abs() + (torch.exp(2 * e) - 1 + 2.0 ** -10) * mag
    else:
        # logits reach sum |q k| scale <= 400 here: 400 * 20 * 2^-24 = 5e-4 beyond doubt, twice that in a weight
        tol = 1e-3 * mag
    out = qc.kv4_attend(q.cuda(), pool.cuda(), table.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda"),
                        torch.tensor([n], dtype=torch.int32, device="cuda"), scale, 1e4)
    err = (out.cpu().double().view_as(want) - want).abs()
    assert bool((err <= tol + 1e-12).all()), float((err / mag).max())


def test_a_workspace_apart_from_the_tensors():
    """A workspace that shares memory with the call's tensors is refused before a launch; the output may take the query's place."""
    import tokenselect_b200
    hq, hkv, d = 8, 2, 128
    q, pool, rtt, slots, lens = (t.cuda() for t in _attend_case(73, hq, hkv, d, [50, 300], BF16))
    need = qc.kv4_attend_workspace(2, hq, d)
    want = qc.kv4_attend(q, pool, rtt, slots, lens, 0.1, 5e5)
    both = torch.zeros(need + q.numel() * 2, dtype=torch.uint8, device="cuda")
    for at in (0, need - 64):
        inside = both[at:at + q.numel() * 2].view(BF16).view(q.shape)
        inside.copy_(q)
        for kw in ({"out": inside}, {}):
            with pytest.raises(tokenselect_b200.TokenSelectError):
                qc.kv4_attend(q if kw else inside, pool, rtt, slots, lens, 0.1, 5e5, workspace=both[:need], **kw)
    own = q.clone()
    assert qc.kv4_attend(own, pool, rtt, slots, lens, 0.1, 5e5, out=own, workspace=both[:need]) is own and torch.equal(own, want)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("cap", [0.0, 5.0])
def test_queries_of_zeros_and_the_smallest_pool_scale(cap, dtype):
    """A head of zeros attends to every row alike, whatever the pool's scale of K: the mean of its values.  So does one whose
    logits are too small for fp32."""
    hq, hkv, d = 8, 2, 128
    case = list(_attend_case(67, hq, hkv, d, [17, 40, 160], dtype))
    case[0].view(3, hq, d)[:, ::2] = 0.0
    case[0].view(3, hq, d)[:, 1] = 1e-36
    for gk in (2.0 ** -32, 2.0 ** -21, 1.0):
        _check_attend(case, hq, d ** -0.5, 5e5, cap=cap, gk=gk)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("g", [1.0, 2.0 ** -20, 2.0 ** 20])
def test_bytes_written_and_written_again(g, dtype):
    """The bytes of a pool row are those of the plain quantiser, the sign of an element that rounds to zero among them (a zero
    keeps its sign too).  Read back and written again, a block whose largest magnitude is above 10/512 of the pool's scale
    keeps its bytes; of a smaller one the values read back are written like any others."""
    gen = torch.Generator().manual_seed(3)
    n, heads, d = 96, 2, 128
    size = torch.logspace(-2.6, 3.3, n * heads * (d // 16)).view(n, heads, d // 16, 1)       # of a block: scales from 0 to the largest
    x = (torch.randn(n, heads, d // 16, 16, generator=gen) * size).flatten(-2)
    x[0, 0, :16] = torch.tensor([3.2, -1.0] + [0.0] * 14) * 2.0 ** -9
    x[1, 0, :16] = torch.tensor([9.5, -4.0, 0.1, -0.1] + [0.0] * 12) * 2.0 ** -9
    x[2, 0, :16] = torch.tensor([10.0, -10.0, 0.1, -0.1] + [0.0] * 12) * 2.0 ** -9
    x[3, 0, :16] = torch.tensor([1e32, -1e3] + [0.0] * 14)
    x = (x * g).to(dtype)
    y = x.flip(0).contiguous()
    rows = torch.arange(n, dtype=torch.int32, device="cuda")

    def written(k, v):
        pool = qc.kv4_pool(n, heads, d)
        qc.kv4_write(pool, k.cuda(), v.cuda(), rows, g, g)
        return pool

    pool = written(x, y)
    assert torch.equal(pool.cpu(), ref.pack(x, y, g, g))
    for out in (BF16, F32):
        k, v = qc.kv4_read(pool, rows, out, g, g)
        again = written(k, v).cpu()
        assert torch.equal(torch.stack(ref.unpack(again, g, g)), torch.stack((ref.held(k.cpu(), g), ref.held(v.cpu(), g))))
        kept = x.double().unflatten(-1, (-1, 16)).abs().amax(-1) > 10.0 / 512.0 * g              # [n, heads, blocks]
        code = lambda p: p[..., :d // 2].unflatten(-1, (-1, 8))                                  # noqa: E731
        scale = slice(d, d + d // 16)
        assert torch.equal(code(again)[kept], code(pool.cpu())[kept]) and torch.equal(again[..., scale][kept], pool.cpu()[..., scale][kept])
    zero = torch.zeros(n, heads, d)
    zero[:, :, 0], zero[:, :, 1::2] = 1.0, -0.0
    for top in (1.0, 2e31):                                                   # beyond 1e30 the quotients are taken another way
        zero[:, :, ::16] = top
        z = (zero * g).to(dtype)
        assert bool((written(z, z)[..., :d // 2] & 0xF0 == 0x80).all()), top


def test_type_of_what_is_read():
    """bf16 by default, what is asked for otherwise, and the given tensors' own; a type that contradicts them is refused."""
    pool, rows = qc.kv4_pool(4, 2, 64), torch.arange(3, dtype=torch.int32, device="cuda")
    given = torch.empty(3, 2, 64, dtype=F32, device="cuda")
    assert [t.dtype for t in qc.kv4_read(pool, rows)] == [BF16, BF16] and [t.dtype for t in qc.kv4_read(pool, rows, F32)] == [F32, F32]
    for kw in ({"k": given}, {"v": given}, {"k": given, "dtype": F32}):
        assert [t.dtype for t in qc.kv4_read(pool, rows, **kw)] == [F32, F32]
    for kw in ({"k": given}, {"v": given}):
        with pytest.raises(ValueError, match="dtype"):
            qc.kv4_read(pool, rows, BF16, **kw)


@pytest.mark.parametrize("octaves", [24.5, 25.5, 28.0])
def test_many_small_weights_beside_a_large_one(octaves):
    """Every 2000th row holds 2^24 to 2^28 times the weight of the rows behind it, and its value is 0: what the others add up to
    is not lost.  (Each CTA's rows begin with a large one.  Keys and queries lie in the slowest pair of a base so large that
    nothing turns.)"""
    heads, d, every, v1 = 8, 64, 2000, 3.0
    n = torch.cuda.get_device_properties(0).multi_processor_count * every
    k, v = torch.zeros(2, heads, d), torch.zeros(2, heads, d)
    k[0, :, d // 2 - 1], v[1] = 1.0, v1
    pool = ref.pack(k, v)                                                    # row 0: a large weight; row 1: a key of zeros
    kh, vh = ref.unpack(pool)
    table = (torch.arange(n) % every != 0).int()[None]
    q = torch.zeros(1, heads, d)
    q[:, :, d // 2 - 1] = 1.0
    scale = octaves * 0.6931471805599453 / float(kh[0, 0, d // 2 - 1])
    out = qc.kv4_attend(q.view(1, -1).to(BF16).cuda(), pool.cuda(), table.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda"),
                        torch.tensor([n], dtype=torch.int32, device="cuda"), scale, 1e30).cpu().double()
    small = (every - 1) * 2.0 ** -octaves
    want = small / (1.0 + small) * float(vh[1, 0, 0])
    e = torch.tensor(6 * 5 * 2.0 ** -11 * octaves * 0.6931471805599453)      # |q_i| = 1, scale |k_i| = the logit
    tol = want * (2.0 ** -8 + float(torch.exp(2 * e)) - 1 + 2.0 ** -10) + every * 2.0 ** -32 * v1
    assert float((out - want).abs().max()) <= tol, (want, float(out[0, 0]), tol)
