"""AdamW over many tensors (``ops.adamw_step``, ``strata_amd.optim.AdamW``) against its float64 oracle.

Tolerances count roundings of half a step (u = 2^-24 in fp32): a moment's b1 m + (1 - b1) c g has two
rounded constants, a rounded c, c g and two rounded operations, at most 8 u of b1 |m| + (1 - b1) |c g|
(v 10 u, its g enters twice).  The update rate m / (sqrt(v) r + eps) adds a rounded rate (3), sqrt (1),
product and sum (3) and quotient (2) and half of v's error: at most 24 u of its magnitude before
cancellation; p (1 - lr decay) - update two of |p| and one of the result.
"""

import math

import pytest
import torch

from oracle import optim as O
from strata_amd import ops
from strata_amd.optim import AdamW

pytestmark = pytest.mark.gpu
U = 2.0**-24
HP = dict(lr=3e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
SIZES = [1, 7, 255, 256, 257, 1000, 4096, 4097, 16384, 50001]


def _tensors(sizes, p_dtype, g_dtype, bits, master, seed, gpu, offset=0, zero=False):
    """Lists on the GPU; ``offset`` elements before each tensor in its allocation."""
    gen = torch.Generator().manual_seed(seed)

    def place(t):
        if not offset:
            return t.to(gpu)
        buf = torch.zeros(t.numel() + offset, dtype=t.dtype, device=gpu)
        buf[offset:] = t.to(gpu)
        return buf[offset:]

    out = dict(params=[], grads=[], exp_avgs=[], exp_avg_sqs=[], masters=[], exp_avg_scales=[], exp_avg_sq_scales=[])
    for n in sizes:
        p = torch.randn(n, generator=gen) * 0.05
        mag = torch.exp(2 * torch.randn(n, generator=gen))
        m, v = torch.randn(n, generator=gen) * 0.01 * mag, (torch.randn(n, generator=gen) * 0.02 * mag) ** 2
        if zero:
            m, v = torch.zeros(n), torch.zeros(n)
        g = torch.randn(n, generator=gen) * 0.03 * mag
        g[torch.rand(n, generator=gen) < 0.1] = 0.0
        out["params"].append(place(p.to(p_dtype)))
        out["grads"].append(place(g.to(g_dtype)))
        out["masters"].append(place(p) if master else None)
        if bits == 8:
            mc, ms, _ = O.pack(m.double(), True)
            vc, vs, _ = O.pack(v.double(), False)
            out["exp_avgs"].append(place(mc))
            out["exp_avg_sqs"].append(place(vc))
            out["exp_avg_scales"].append(ms.to(gpu))
            out["exp_avg_sq_scales"].append(vs.to(gpu))
        else:
            out["exp_avgs"].append(place(m))
            out["exp_avg_sqs"].append(place(v))
            out["exp_avg_scales"].append(None)
            out["exp_avg_sq_scales"].append(None)
    return out


def _check(ts, before, t, coef, hp=HP, lrs=None, wds=None):
    for i in range(len(ts["params"])):
        cpu = lambda k: before[k][i].cpu() if before[k][i] is not None else None  # noqa: E731
        p0, g, master = cpu("params"), cpu("grads").double(), cpu("masters")
        bits = 8 if before["exp_avgs"][i].dtype == torch.int8 else 32
        if bits == 8:
            m0, v0 = O.unpack(cpu("exp_avgs"), cpu("exp_avg_scales")), O.unpack(cpu("exp_avg_sqs"), cpu("exp_avg_sq_scales"))
        else:
            m0, v0 = cpu("exp_avgs").double(), cpu("exp_avg_sqs").double()
        base = (master if master is not None else p0).double()
        lr, wd = (lrs[i] if lrs else hp["lr"]), (wds[i] if wds else hp["weight_decay"])
        b1, b2 = hp["betas"]
        p, m, v = O.adamw(base, g, m0, v0, t, lr, hp["betas"], hp["eps"], wd, coef)
        big = lr / (1 - b1**t) * (b1 * m0.abs() + (1 - b1) * (g * coef).abs()) / ((v / (1 - b2**t)).sqrt() + hp["eps"])
        # a v under 2^-126 is rounded to a multiple of 2^-149: off by 2^-150, relative to v twice what its root is off by
        tol = U * (3 * base.abs() + 24 * big) + big * torch.where(v < 2.0**-126, 2.0**-150 / v.clamp_min(1e-300), 0.0) + 1e-44
        if master is not None:
            got = ts["masters"][i].cpu().double()
            assert ((got - p).abs() <= tol).all(), i
        got = ts["params"][i].cpu()
        half = 2.0**-8 if got.dtype == torch.bfloat16 else U
        assert ((got.double() - p).abs() <= tol + half * (p.abs() + tol)).all(), i
        if master is not None:  # the parameter is its master, rounded
            assert torch.equal(got, ts["masters"][i].cpu().to(torch.bfloat16)), i
        if bits == 8:
            for k, x, signed in (("exp_avg", m, True), ("exp_avg_sq", v, False)):
                codes, scale, border = O.pack(x, signed)
                gs = ts[k + "_scales"][i].cpu()
                assert ((gs - scale).abs() <= 2.0**-23 * scale).all(), (i, k)
                same = ts[k + "s"][i].cpu() == codes
                assert (same | (border < 1e-6)).all(), (i, k)  # beside a border the scale's own rounding decides
                assert int(same.sum()) >= 0.999 * same.numel(), (i, k)
        else:
            tm = 8 * U * (b1 * m0.abs() + (1 - b1) * (g * coef).abs()) + 1e-44
            assert ((ts["exp_avgs"][i].cpu().double() - m).abs() <= tm).all(), i
            assert ((ts["exp_avg_sqs"][i].cpu().double() - v).abs() <= 10 * U * v + 1e-44).all(), i


def _copy(ts):
    return {k: [None if t is None else t.clone() for t in x] for k, x in ts.items()}


@pytest.mark.parametrize("offset", [0, 1], ids=["aligned", "odd-start"])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("p_dtype,g_dtype,master", [
    (torch.float32, torch.float32, False), (torch.float32, torch.bfloat16, False), (torch.bfloat16, torch.bfloat16, False),
    (torch.bfloat16, torch.float32, False), (torch.bfloat16, torch.bfloat16, True), (torch.bfloat16, torch.float32, True)])
@pytest.mark.parametrize("clip", [None, 0.5])
def test_two_steps_match_the_oracle(gpu, p_dtype, g_dtype, master, bits, offset, clip):
    print(f"adamw {p_dtype} {g_dtype} master {master} bits {bits} offset {offset} clip {clip}", flush=True)
    ts = _tensors(SIZES, p_dtype, g_dtype, bits, master, 1, gpu, offset)
    step = torch.full((1,), 4, dtype=torch.int64, device=gpu)
    norm = O.global_norm([g.cpu() for g in ts["grads"]])
    for t in (5, 6):
        before = _copy(ts)
        got = ops.adamw_step(**ts, step=step, max_norm=clip, **HP)
        torch.cuda.synchronize()
        assert int(step) == t
        if clip:
            assert abs(float(got) - norm) <= 1e-12 * norm  # 64-bit sums of exact squares
        else:
            assert got is None
        _check(ts, before, t, min(1.0, clip / (norm + 1e-6)) if clip else 1.0)


def test_mixed_tensors_rates_and_many(gpu):
    """fp32 and bf16 parameters, both kinds of state and different rates in one call of more tensors
    than a launch takes, an empty one among them."""
    a = _tensors([5000, 33, 0, 8192], torch.bfloat16, torch.bfloat16, 8, True, 2, gpu)
    b = _tensors([n % 700 + 1 for n in range(37, 37 + 160 * 13, 13)], torch.float32, torch.float32, 32, False, 3, gpu)
    c = _tensors([777, 64], torch.bfloat16, torch.float32, 32, False, 4, gpu)
    ts = {k: a[k] + b[k] + c[k] for k in a}
    n = len(ts["params"])
    lrs, wds = [1e-3 * (1 + i % 3) for i in range(n)], [0.1 * (i % 2) for i in range(n)]
    hp = dict(HP, lr=lrs, weight_decay=wds)
    before = _copy(ts)
    step = torch.zeros(1, dtype=torch.int64, device=gpu)
    norm = ops.adamw_step(**ts, step=step, max_norm=2.0, **hp)
    want = O.global_norm([g.cpu() for g in before["grads"]])
    assert abs(float(norm) - want) <= 1e-12 * want
    _check(ts, before, 1, min(1.0, 2.0 / (want + 1e-6)), HP, lrs, wds)
    again = _copy(before)
    step.zero_()
    ops.adamw_step(**again, step=step, max_norm=2.0, **hp)
    for k in ts:  # the same bits on every call
        assert all(x is None or torch.equal(x, y) for x, y in zip(ts[k], again[k])), k


def test_first_steps_from_zero_states(gpu):
    for bits in (32, 8):
        ts = _tensors([3000, 5], torch.float32, torch.float32, bits, False, 5, gpu, zero=True)
        step = torch.zeros(1, dtype=torch.int64, device=gpu)
        for t in (1, 2, 3):
            before = _copy(ts)
            ops.adamw_step(**ts, step=step, **HP)
            _check(ts, before, t, 1.0)


@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_norm_that_is_not_finite_leaves_everything(gpu, bad):
    ts = _tensors([300, 5000], torch.bfloat16, torch.float32, 8, True, 6, gpu)
    ts["grads"][1][4321] = bad
    before = _copy(ts)
    step = torch.full((1,), 9, dtype=torch.int64, device=gpu)
    norm = ops.adamw_step(**ts, step=step, max_norm=1.0, **HP)
    assert not math.isfinite(float(norm)) and int(step) == 9
    for k in ts:
        assert all(x is None or torch.equal(x.nan_to_num(), y.nan_to_num()) for x, y in zip(ts[k], before[k])), k


def test_neighbours_in_memory_stay(gpu):
    """Tensors that are views of one buffer, with elements between them that are not theirs."""
    for bits in (32, 8):
        ts = _tensors([1000, 300], torch.bfloat16, torch.bfloat16, bits, False, 7, gpu)
        big = {k: torch.full((4000,), 3, dtype=ts[k][0].dtype, device=gpu) for k in ("params", "exp_avgs", "exp_avg_sqs")}
        for k, buf in big.items():
            for i, (a, n) in enumerate(((8, 1000), (1500, 300))):
                buf[a:a + n] = ts[k][i]
                ts[k][i] = buf[a:a + n]
        ops.adamw_step(**ts, step=torch.zeros(1, dtype=torch.int64, device=gpu), **HP)
        for buf in big.values():
            rest = torch.cat([buf[:8], buf[1008:1500], buf[1800:]])
            assert (rest == 3).all()


def test_step_replayed_from_a_graph(gpu):
    ts = _tensors([5000, 64, 300], torch.bfloat16, torch.bfloat16, 8, True, 8, gpu)
    want = _copy(ts)
    step, wstep = (torch.zeros(1, dtype=torch.int64, device=gpu) for _ in range(2))
    kw = dict(HP, max_norm=1.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        norm = ops.adamw_step(**ts, step=step, **kw)
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        wnorm = ops.adamw_step(**want, step=wstep, **kw)  # eager work between the replays
        torch.cuda.synchronize()
        assert int(step) == int(wstep) == i + 1 and float(norm) == float(wnorm)
        for k in ts:
            assert all(x is None or torch.equal(x, y) for x, y in zip(ts[k], want[k])), (i, k)


def test_another_stream(gpu):
    ts = _tensors([9000], torch.float32, torch.float32, 32, False, 9, gpu)
    before = _copy(ts)
    step = torch.zeros(1, dtype=torch.int64, device=gpu)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.adamw_step(**ts, step=step, max_norm=1.0, **HP)
    s.synchronize()
    norm = O.global_norm([g.cpu() for g in before["grads"]])
    _check(ts, before, 1, min(1.0, 1.0 / (norm + 1e-6)))


def test_state_values(gpu):
    for signed in (True, False):
        x = torch.randn(1000, dtype=torch.float64) * torch.exp(torch.randn(1000, dtype=torch.float64))
        codes, scale, _ = O.pack(x if signed else x * x, signed)
        got = torch.ops.strata_hip.adamw_state_values(codes.to(gpu), scale.to(gpu)).cpu().double()
        want = O.unpack(codes, scale)
        assert ((got - want).abs() <= U * want.abs()).all()  # 64 bits, rounded once


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_and_its_state_dict(gpu, bits):
    """Three steps of two optimizers, the second loaded from the first's state after two."""
    gen = torch.Generator().manual_seed(10)

    def model():
        torch.manual_seed(0)
        return torch.nn.Sequential(torch.nn.Linear(64, 96), torch.nn.Linear(96, 8)).to(gpu).bfloat16()

    grads = [[torch.randn(p.shape, generator=gen).to(gpu).bfloat16() for p in model().parameters()] for _ in range(3)]

    def step(opt, net, k):
        for p, g in zip(net.parameters(), grads[k]):
            p.grad = g.clone()
        opt.step()

    def make(net):
        ps = list(net.parameters())
        return AdamW([dict(params=ps[::2], weight_decay=0.1), dict(params=ps[1::2], weight_decay=0.0)], lr=1e-2,
                     state_bits=bits, max_norm=1.0, min_8bit=512)

    a = model()
    oa = make(a)
    for k in range(2):
        step(oa, a, k)
    b = model()
    b.load_state_dict(a.state_dict())
    ob = make(b)
    ob.load_state_dict(oa.state_dict())
    kinds = {s["exp_avg"].dtype for s in ob.state.values()}
    assert kinds == ({torch.int8, torch.float32} if bits == 8 else {torch.float32})
    assert all(s["master"].dtype == torch.float32 for s in ob.state.values())
    step(oa, a, 2)
    step(ob, b, 2)
    assert all(torch.equal(x, y) for x, y in zip(a.parameters(), b.parameters()))
    assert float(oa.grad_norm) == float(ob.grad_norm)
    if bits == 32:  # against torch's step on the master weights
        ref = model().float()
        ps = list(ref.parameters())
        oref = torch.optim.AdamW([dict(params=ps[::2], weight_decay=0.1), dict(params=ps[1::2], weight_decay=0.0)], lr=1e-2)
        for k in range(3):
            for p, g in zip(ps, grads[k]):
                p.grad = g.float()
            torch.nn.utils.clip_grad_norm_(ps, 1.0)
            oref.step()
        masters = [oa.state[p]["master"] for p in a.parameters()]
        for x, y in zip(masters, ps):  # three steps of lr at most 24 u each and |p| roundings, on both sides
            assert ((x - y).abs() <= 2 * 3 * U * (3 * y.abs() + 24 * 2e-2) + 1e-7).all()


def test_8bit_scales_half_way_between_two(gpu):
    """0.9 s + 0.1 g of the largest element often lies exactly between two fp32 scales: the 64-bit operations
    round in the formula's order, so scales and codes are those of the formula, all of them."""
    n = 256 * 4000
    ts = _tensors([n], torch.bfloat16, torch.bfloat16, 8, False, 11, gpu)
    before = _copy(ts)
    ops.adamw_step(**ts, step=torch.full((1,), 4, dtype=torch.int64, device=gpu), **HP)
    g = before["grads"][0].cpu().double()
    m0 = O.unpack(before["exp_avgs"][0].cpu(), before["exp_avg_scales"][0].cpu())
    v0 = O.unpack(before["exp_avg_sqs"][0].cpu(), before["exp_avg_sq_scales"][0].cpu())
    _, m, v = O.adamw(m0, g, m0, v0, 5, 1e-3, HP["betas"], 1e-8, 0.0)
    for k, x, signed in (("exp_avg", m, True), ("exp_avg_sq", v, False)):
        codes, scale, _ = O.pack(x, signed)
        assert (ts[k + "_scales"][0].cpu() != scale).sum() <= 4, k  # of 4000; ties of other codes than the largest
        assert (ts[k + "s"][0].cpu() != codes).sum() <= 1, k


@pytest.mark.parametrize("size,eps", [(1e-16, 1e-20), (1e-30, 1e-8)])
def test_8bit_codes_of_tiny_gradients(gpu, size, eps):
    """Blocks whose largest moment is so small that 65536 over it leaves fp32."""
    hp = dict(HP, eps=eps)
    ts = _tensors([3, 256, 1300], torch.float32, torch.float32, 8, False, 21, gpu, zero=True)
    ts["grads"] = [g * size for g in ts["grads"]]
    step = torch.zeros(1, dtype=torch.int64, device=gpu)
    before = _copy(ts)
    ops.adamw_step(**ts, step=step, **hp)
    _check(ts, before, 1, 1.0, hp)
    assert not any(ts["exp_avgs"][i][ts["grads"][i] == 0].any() for i in range(3))


@pytest.mark.parametrize("bits", [32, 8])
def test_offsets_past_32_bits(gpu, bits):
    """A tensor of 2^31 + 555 elements: its first and last ones against the oracle."""
    n = 2**31 + 555
    blocks = -(-n // 256)
    p, g = (torch.full((n,), v, dtype=torch.bfloat16, device=gpu) for v in (0.5, 0.25))
    ends = [slice(0, 300), slice(2**31 - 256, n)]
    gen = torch.Generator().manual_seed(12)
    for sl in ends:
        k = p[sl].numel()
        p[sl], g[sl] = torch.randn(k, generator=gen).to(gpu), torch.randn(k, generator=gen).to(gpu)
    dt = (torch.int8, torch.uint8) if bits == 8 else (torch.float32,) * 2
    ts = dict(params=[p], grads=[g], exp_avgs=[torch.zeros(n, dtype=dt[0], device=gpu)],
              exp_avg_sqs=[torch.zeros(n, dtype=dt[1], device=gpu)])
    if bits == 8:
        ts |= {k: [torch.zeros(blocks, device=gpu)] for k in ("exp_avg_scales", "exp_avg_sq_scales")}
    before = [(p[sl].cpu().double(), g[sl].cpu().double()) for sl in ends]
    step = torch.zeros(1, dtype=torch.int64, device=gpu)
    norm = ops.adamw_step(**ts, step=step, max_norm=1e9, **HP)
    rest = n - sum(b[1].numel() for b in before)
    want = math.sqrt(rest * 0.0625 + sum(float((b[1] ** 2).sum()) for b in before))
    assert abs(float(norm) - want) <= 1e-12 * want
    for sl, (p0, g0) in zip(ends, before):
        new, m, v = O.adamw(p0, g0, 0 * p0, 0 * p0, 1, HP["lr"], HP["betas"], HP["eps"], HP["weight_decay"])
        got = p[sl].cpu().double()
        assert ((got - new).abs() <= U * (3 * p0.abs() + 24 * HP["lr"]) + 2.0**-8 * new.abs()).all()
        if bits == 32:
            assert ((ts["exp_avgs"][0][sl].cpu().double() - m).abs() <= 8 * U * m.abs() + 1e-44).all()
    assert float(p[2**30]) == float(p[1000])


def test_refusals(gpu):
    """Kinds of moments that do not go together, sizes, layouts and places; nothing is changed by a refused call."""
    ts = _tensors([300, 512], torch.bfloat16, torch.float32, 32, True, 31, gpu)
    q8 = _tensors([300, 512], torch.bfloat16, torch.float32, 8, True, 31, gpu)
    step = torch.zeros(1, dtype=torch.int64, device=gpu)
    before = _copy(ts)
    mix = lambda k: [ts[k][0], q8[k][1]]  # noqa: E731
    for over, msg in (
            (dict(exp_avgs=q8["exp_avgs"]), "both be fp32"), (dict(exp_avgs=mix("exp_avgs")), "both be fp32"),
            (dict(exp_avg_scales=q8["exp_avg_scales"]), "scales"),
            (dict(exp_avgs=q8["exp_avgs"], exp_avg_sqs=q8["exp_avg_sqs"], exp_avg_scales=None), "scales"),
            (dict(exp_avgs=mix("exp_avgs"), exp_avg_sqs=mix("exp_avg_sqs"), exp_avg_scales=q8["exp_avg_scales"],
                  exp_avg_sq_scales=q8["exp_avg_sq_scales"]), "scales"),
            (dict(grads=ts["grads"][::-1]), "grads"), (dict(grads=[g.half() for g in ts["grads"]]), "grads"),
            (dict(exp_avg_sqs=[t.repeat(2)[::2] for t in ts["exp_avg_sqs"]]), "contiguous"),
            (dict(masters=[t.cpu() for t in ts["masters"]]), "step's GPU"), (dict(params=[t.float() for t in ts["params"]]), "masters"),
            (dict(grads=[ts["exp_avgs"][0], ts["grads"][1]]), "gradient overlaps"), (dict(lr=[1e-3]), "one entry")):
        with pytest.raises(ValueError, match=msg):
            ops.adamw_step(**{**ts, **HP, "step": step, **over})
    assert int(step) == 0
    for k in ts:
        assert all(x is None or torch.equal(x, y) for x, y in zip(ts[k], before[k])), k
    both = {k: mix(k) for k in ts}
    ops.adamw_step(**both, step=step, **HP)  # one of each kind in one call
    assert int(step) == 1


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("clip", [None, 0.7])
def test_counts_of_their_own(gpu, bits, clip):
    """Tensors of three counts in one call, one norm over all of them."""
    ts = _tensors(SIZES, torch.bfloat16, torch.float32, bits, True, 41, gpu)
    n = len(SIZES)
    kinds = [torch.full((1,), k, dtype=torch.int64, device=gpu) for k in (0, 7, 400)]
    steps = [kinds[i % 3] for i in range(n)]
    norm = O.global_norm([g.cpu() for g in ts["grads"]])
    for more in (1, 2):
        before = _copy(ts)
        got = ops.adamw_step(**ts, step=steps, max_norm=clip, **HP)
        assert [int(k) for k in kinds] == [more, 7 + more, 400 + more]
        assert got is None if clip is None else abs(float(got) - norm) <= 1e-12 * norm
        for k in range(3):
            part = lambda d: {c: x[k::3] for c, x in d.items()}  # noqa: E731
            _check(part(ts), part(before), int(kinds[k]), min(1.0, clip / (norm + 1e-6)) if clip else 1.0)


def test_more_counts_than_a_launch_takes(gpu):
    """A count for each of 1000 tensors, and a norm that is not finite: all stay."""
    ts = _tensors([3] * 1000, torch.float32, torch.float32, 32, False, 42, gpu)
    steps = list(torch.arange(1000, device=gpu).split(1))
    before = _copy(ts)
    norm = float(ops.adamw_step(**ts, step=steps, max_norm=1.0, **HP))
    assert torch.cat(steps).tolist() == list(range(1, 1001))
    for i in (0, 1, 447, 448, 449, 895, 896, 999):
        one = lambda d: {c: x[i:i + 1] for c, x in d.items()}  # noqa: E731
        _check(one(ts), one(before), i + 1, min(1.0, 1.0 / (norm + 1e-6)))
    ts["grads"][500][1] = math.nan
    before = _copy(ts)
    assert math.isnan(float(ops.adamw_step(**ts, step=steps, max_norm=1.0, **HP)))
    assert torch.cat(steps).tolist() == list(range(1, 1001))
    assert all(torch.equal(x, y) for x, y in zip(ts["params"], before["params"]))


def test_late_and_missing_parameters_as_torch(gpu):
    """Parameters without a gradient at first, for a while, and a group added later, against torch's step in 64 bits.
    8 steps, each off by at most 24 u of its size (up to 12 lr while the moments are young, the errors of
    the moments' up to 8 steps among them) and 3 u of |p|."""
    lr, gen = 1e-2, torch.Generator().manual_seed(43)
    start = [torch.randn(300, generator=gen) * 0.1 for _ in range(4)]
    ps = [torch.nn.Parameter(t.to(gpu)) for t in start]
    qs = [torch.nn.Parameter(t.double()) for t in start]
    ours, ref = AdamW(ps[:3], lr=lr, max_norm=3.0), torch.optim.AdamW(qs[:3], lr=lr)
    for k, which in enumerate(((0,), (0, 1), (0, 1), (0, 2), (0, 1, 2), (1,), (0, 1, 2, 3), (0, 1, 2, 3))):
        if k == 6:
            ours.add_param_group(dict(params=[ps[3]]))
            ref.add_param_group(dict(params=[qs[3]]))
        for i in range(4):
            g = torch.randn(300, generator=gen)
            ps[i].grad = g.to(gpu) if i in which else None
            qs[i].grad = g.double() if i in which else None
        torch.nn.utils.clip_grad_norm_([q for q in qs if q.grad is not None], 3.0)
        ours.step()
        ref.step()
        for i in range(4):
            tol = (k + 1) * U * (3 * qs[i].detach().abs() + 24 * 12 * lr * (k + 1))
            assert ((ps[i].detach().cpu().double() - qs[i].detach()).abs() <= tol).all(), (k, i)


def test_counts_replayed_from_a_graph(gpu):
    """A captured step of an optimizer with two counts, replayed between eager work, as the eager one."""
    gen = torch.Generator().manual_seed(44)
    start, grads = ([torch.randn(500, generator=gen) for _ in range(3)] for _ in range(2))

    def make():
        ps = [torch.nn.Parameter(t.to(gpu)) for t in start]
        opt = AdamW(ps, max_norm=1.0)
        for which in ((0, 2), (0, 1, 2)):
            for i, p in enumerate(ps):
                p.grad = grads[i].to(gpu) if i in which else None
            opt.step()
        return ps, opt

    (a, oa), (b, ob) = make(), make()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        oa.step()
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        ob.step()
        torch.cuda.synchronize()
        assert [int(oa.state[p]["step"]) for p in a] == [int(ob.state[p]["step"]) for p in b] == [3 + k, 2 + k, 3 + k]
        assert all(torch.equal(x, y) for x, y in zip(a, b)) and float(oa.grad_norm) == float(ob.grad_norm)
