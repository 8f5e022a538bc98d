"""Orthogonalised updates on the GPU (``ops.orthogonalize``, ``ops.muon_step``, ``optim.Muon``) against their float64 oracle.

The oracle gives, with each result, the norm of the error that the kernels' roundings make (``oracle.optim.orthogonalize``: each
rounding counted as half a step, independent and evenly spread; simulated with the kernels' roundings, the error is a
sixth to an eleventh of it with operands of one fp16, a 36th to a 370th with two: test_muon_operands_gpu has tight
bounds); the result's own rounding is half a step of its type.  The momentum is one rounded product, a rounded
constant each and a fused sum: 4 u of the two terms.  p (1 - lr decay) - rate o: a rounded constant, product, rate and
result, 3 u of |p| and 3 u of the update.
"""

import pytest
import torch

from oracle import optim as O
from strata_amd import modules, ops
from strata_amd.optim import AdamW, Muon, matrices

pytestmark = pytest.mark.gpu
U = 2.0**-24
F32, BF16 = torch.float32, torch.bfloat16


def _half(t):
    return 2.0**-8 if t.dtype == BF16 else U


def matrix(rows, cols, kind, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    if kind == "low":  # four directions alone
        return r(rows, 4) @ r(4, cols)
    x = r(rows, cols)
    if kind == "strong":
        x = x + r(rows, 4) @ r(4, cols)
    if kind == "rows":
        x = x * torch.exp(r(rows, 1))
    return x


def check(got, x, precise, **kw):
    """One matrix of the result, of x in its own type."""
    want, off = O.orthogonalize(x.double(), precise=precise or min(x.shape) <= 64, **kw)
    err = float((got.double() - want).norm())
    tol = off + _half(got) * float(want.norm())
    print(f"  off by {err / max(float(want.norm()), 1e-300):.2e}, at most {tol / max(float(want.norm()), 1e-300):.2e}", flush=True)
    assert err <= tol


SHAPES = [(1, 1), (1, 2), (1, 777), (500, 1), (2, 3), (63, 65), (64, 64), (65, 64), (100, 300), (128, 128), (129, 127), (130, 257),
          (192, 640), (513, 96), (300, 290), (64, 384), (300, 40), (64, 385), (128, 129), (65, 128), (66, 512)]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_matches_the_oracle(gpu, rows, cols, dtype):
    for kind in ("plain", "strong", "rows"):
        print(f"orthogonalize {rows} {cols} {dtype} {kind}", flush=True)
        x = matrix(rows, cols, kind, rows + cols).to(dtype)
        check(ops.orthogonalize(x.to(gpu)).cpu(), x, dtype == F32)


@pytest.mark.parametrize("dtype,precise", [(F32, False), (BF16, True)])
@pytest.mark.parametrize("rows,cols", [(5, 64), (192, 320), (140, 70)])
def test_precision_of_choice(gpu, rows, cols, dtype, precise):
    for kind in ("plain", "low"):
        x = matrix(rows, cols, kind, 7).to(dtype)
        check(ops.orthogonalize(x.to(gpu), precise=precise).cpu(), x, precise)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_stacks_strides_and_transposes(gpu, dtype):
    """A stack's matrices by themselves, the same bits as alone; views of other strides; the transpose's transpose."""
    x = torch.stack([matrix(70, 132, k, i) * 10.0 ** (3 * i - 6) for i, k in enumerate(("plain", "strong", "rows", "low", "plain"))])
    x = x.to(dtype).to(gpu)
    y = ops.orthogonalize(x)
    for i in range(5):
        check(y[i].cpu(), x[i].cpu(), dtype == F32)
        assert torch.equal(y[i], ops.orthogonalize(x[i]))
    assert torch.equal(ops.orthogonalize(x.mT), y.mT)
    wide = torch.zeros(5, 2, 70, 264, dtype=dtype, device=gpu)
    wide[:, 1, :, ::2] = x
    assert torch.equal(ops.orthogonalize(wide[:, 1, :, ::2]), y)
    assert torch.equal(ops.orthogonalize(x.view(5, 1, 70, 132)), y.view(5, 1, 70, 132))
    odd = torch.zeros(x.numel() + 1, dtype=dtype, device=gpu)[1:].view(x.shape)
    odd.copy_(x)
    assert torch.equal(ops.orthogonalize(odd), y)


@pytest.mark.parametrize("count,rows,cols,dtype", [(100, 130, 260, BF16), (70, 512, 600, BF16), (150, 260, 300, F32), (64, 513, 400, BF16),
                                                   (90, 384, 260, F32), (300, 64, 200, F32), (300, 100, 120, BF16)])
def test_many_matrices(gpu, count, rows, cols, dtype):
    """Enough of them for every tile of the products: each as alone, to the bit, and some against the oracle."""
    g = torch.Generator(device=gpu).manual_seed(count)
    x = (torch.randn(count, rows, cols, generator=g, device=gpu) * torch.exp(torch.randn(count, rows, 1, generator=g, device=gpu))).to(dtype)
    y = ops.orthogonalize(x)
    for i in (0, count // 2, count - 1):
        check(y[i].cpu(), x[i].cpu(), dtype == F32)
        assert torch.equal(y[i], ops.orthogonalize(x[i]))
    assert torch.equal(ops.orthogonalize(x), y)


@pytest.mark.parametrize("count,rows,cols", [(64000, 130, 256), (240000, 64, 128)])
def test_offsets_past_32_bits(gpu, count, rows, cols):
    """Stacks of nearly 2^31 elements, whose workspace has more: the first and last matrices as alone, to the bit."""
    x = torch.empty(count, rows, cols, dtype=BF16, device=gpu)
    g = torch.Generator(device=gpu).manual_seed(1)
    x.fill_(0.5)
    for i in (0, 1, count // 2, count - 1):
        x[i] = torch.randn(rows, cols, generator=g, device=gpu)
    y = ops.orthogonalize(x)
    for i in (0, 1, 2, count // 2, count - 1):
        assert torch.equal(y[i], ops.orthogonalize(x[i])), i
    check(y[count - 1].cpu(), x[count - 1].cpu(), False)


def test_steps_and_coefficients(gpu):
    x = matrix(90, 200, "plain", 3).float()
    for co in ((O.NEWTON_SCHULZ,) * 2, (O.NEWTON_SCHULZ,), (), ((4.0848, -6.8946, 2.9270), (3.9505, -6.3029, 2.6377), (3.7418, -5.5913, 2.3037)),
               ((1.5, -0.5, 0.0),) * 9):
        for precise in (True, False):
            y = ops.orthogonalize(x.to(gpu), co, precise=precise).cpu()
            check(y, x, precise, coefficients=co)
    assert torch.equal(ops.orthogonalize(x.to(gpu), steps=3), ops.orthogonalize(x.to(gpu), (O.NEWTON_SCHULZ,) * 3))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_zeros_and_values_that_are_not_finite(gpu, dtype):
    """A zero matrix stays zero, whatever eps; a value that is not finite makes its own matrix NaN and no other."""
    x = torch.stack([matrix(40, 72, "plain", i) for i in range(4)]).to(dtype).to(gpu)
    want = ops.orthogonalize(x)
    for bad in (float("inf"), float("nan"), -float("inf")):
        y = x.clone()
        y[1, 3, 70] = bad
        y[2] = 0
        for eps in (1e-7, 1e-308):
            got = ops.orthogonalize(y, eps=eps)
            assert got[1].isnan().all() and not got[2].any()
            assert torch.equal(got[0], want[0]) and torch.equal(got[3], want[3])


def test_magnitudes(gpu):
    """Matrices of tiny and huge values, which their norm brings back; below eps it is eps."""
    base = matrix(70, 90, "plain", 5)
    for size in (1e-36, 1e-20, 1e-3, 1e30):
        x = (base * size).float()
        check(ops.orthogonalize(x.to(gpu), eps=1e-45).cpu(), x, True, eps=1e-45)
    x = (base * 1e-9).float()  # a norm of 8e-8
    check(ops.orthogonalize(x.to(gpu)).cpu(), x, True)


def _tensors(specs, p_dtype, g_dtype, master, seed, gpu, offset=0):
    """Lists on the GPU for shapes; ``offset`` elements before each tensor in its allocation."""
    def place(t):
        buf = torch.zeros(t.numel() + offset, dtype=t.dtype, device=gpu)
        buf[offset:] = t.to(gpu).reshape(-1)
        return buf[offset:].view(t.shape)

    out = dict(params=[], grads=[], momentums=[], masters=[])
    for i, s in enumerate(specs):
        n = s[:-2].numel() if isinstance(s, torch.Size) else torch.Size(s[:-2]).numel()
        some = [torch.stack([matrix(*s[-2:], k, seed + 10 * i + j) for j in range(n)]).view(s) if n else torch.zeros(s)
                for k in ("plain", "strong", "rows")]
        out["params"].append(place((some[0] * 0.02).to(p_dtype)))
        out["grads"].append(place((some[1] * 1e-3).to(g_dtype)))
        out["momentums"].append(place((some[2] * 5e-4).float()))
        out["masters"].append(place((some[0] * 0.02).float()) if master else None)
    return out


HP = dict(lr=2e-2, momentum=0.95, weight_decay=0.1)


def _copy(ts):
    return {k: [None if t is None else t.clone() for t in x] for k, x in ts.items()}


def _check_step(ts, before, nesterov=True, adjust="original", precise=None, lrs=None, wds=None):
    for i in range(len(ts["params"])):
        if not ts["params"][i].numel():
            continue
        cpu = lambda d, k: None if d[k][i] is None else d[k][i].cpu().reshape(-1, *d[k][i].shape[-2:])  # noqa: E731
        p0, g, m0, w0 = (cpu(before, k) for k in ("params", "grads", "momentums", "masters"))
        p1, m1, w1 = cpu(ts, "params"), cpu(ts, "momentums"), cpu(ts, "masters")
        fine = (p0.dtype == F32 or w0 is not None) if precise is None else precise
        lr, wd = lrs[i] if lrs else HP["lr"], wds[i] if wds else HP["weight_decay"]
        for j in range(len(p0)):
            base = (p0 if w0 is None else w0)[j].double()
            p, m, off = O.muon(base, g[j].double(), m0[j].double(), lr, HP["momentum"], nesterov, wd, adjust, fine)
            tm = 4 * U * (0.95 * m0[j].abs() + 0.05 * g[j].float().abs()) + 1e-44
            assert ((m1[j].double() - m).abs() <= tm).all(), (i, j)
            own = 3 * U * (float(base.norm()) + float((p - base * (1 - lr * wd)).norm()))
            got = (p1 if w1 is None else w1)[j]
            err, tol = float((got.double() - p).norm()), off + own + _half(got) * float(p.norm())
            print(f"  {i} {j}: {err:.2e} of {tol:.2e}", flush=True)
            assert err <= tol, (i, j)
            if w1 is not None:
                assert torch.equal(p1[j], w1[j].to(BF16))


SPECS = [(96, 64), (64, 96), (3, 40, 72), (2, 2, 33, 31), (1, 65), (130, 1), (0, 4, 4), (4, 0), (128, 192), (20, 20)]


@pytest.mark.parametrize("offset", [0, 1], ids=["aligned", "odd-start"])
@pytest.mark.parametrize("p_dtype,g_dtype,master", [(F32, F32, False), (F32, BF16, False), (BF16, BF16, False), (BF16, F32, False),
                                                    (BF16, BF16, True), (BF16, F32, True)])
def test_steps_match_the_oracle(gpu, p_dtype, g_dtype, master, offset):
    print(f"muon {p_dtype} {g_dtype} master {master} offset {offset}", flush=True)
    for nesterov, adjust, precise in ((True, "match_rms_adamw", None), (False, "original", None), (True, "original", False)):
        ts = _tensors(SPECS, p_dtype, g_dtype, master, 1, gpu, offset)
        before = _copy(ts)
        assert ops.muon_step(**ts, **HP, nesterov=nesterov, adjust=adjust, precise=precise) is None
        _check_step(ts, before, nesterov, adjust, precise)
        assert all(torch.equal(a, b) for a, b in zip(ts["grads"], before["grads"]))


@pytest.mark.parametrize("big", [False, True], ids=["small", "with-large"])
def test_many_tensors_rates_and_types_in_one_call(gpu, big):
    """More tensors and more shapes than a launch takes; every matrix as in a call of its own, to the bit (small ones
    where all are small)."""
    a = _tensors([(k % 7 + 1, 3 * k + 1) for k in range(50)], F32, F32, False, 2, gpu)
    b = _tensors([(24, 40)] * 45, BF16, BF16, True, 3, gpu)
    c = _tensors([(40, 24), (24, 40), (70, 3)], BF16, F32, False, 4, gpu)
    sets = [a, b, c]
    if big:
        sets += [_tensors([(k % 5 + 1, 400 + 70 * k) for k in range(43)], F32, BF16, False, 5, gpu),
                 _tensors([(400, 70 + 66 * (k % 2)) for k in range(46)], BF16, F32, False, 6, gpu)]
    ts = {k: [t for s in sets for t in s[k]] for k in a}
    n = len(ts["params"])
    lrs, wds = [1e-2 * (1 + i % 3) for i in range(n)], [0.1 * (i % 2) for i in range(n)]
    before = _copy(ts)
    ops.muon_step(**ts, lr=lrs, weight_decay=wds, momentum=0.95)
    _check_step(ts, before, lrs=lrs, wds=wds)
    for i in (98, 100, 139, 140, 141, 185, 186) if big else (0, 3, 49, 50, 94, 95, 96, 97):
        one = {k: x[i:i + 1] for k, x in _copy(before).items()}
        ops.muon_step(**one, lr=lrs[i], weight_decay=wds[i], momentum=0.95)
        for k in one:
            assert one[k][0] is None or torch.equal(one[k][0], ts[k][i]), (i, k)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_slim_matrices_beside_others(gpu, dtype):
    """A shorter side of 65 to 128: a step of two launches in a call of such alone, of three beside wider ones, and the same bits."""
    specs = [(100, 400), (500, 70), (3, 128, 200), (2, 77, 1030), (128, 129), (64, 500), (700, 30)]
    ts = _tensors(specs, dtype, dtype, False, 21, gpu)
    wide = _tensors([(200, 330)], dtype, dtype, False, 22, gpu)
    both = {k: x + wide[k] for k, x in _copy(ts).items()}
    before = _copy(ts)
    ops.muon_step(**ts, **HP)
    ops.muon_step(**both, **HP)
    _check_step(ts, before)
    for k in ts:
        assert all(a is None or torch.equal(a, b) for a, b in zip(ts[k], both[k])), k
    for i in (0, 3):
        one = {k: x[i:i + 1] for k, x in before.items()}
        ops.muon_step(**one, **HP)
        assert torch.equal(one["params"][0], ts["params"][i])


def test_neighbours_in_memory_stay(gpu):
    """Tensors that are views of one buffer, with elements between them that are not theirs."""
    for shape in ((17, 31), (32, 40)):
        n = shape[0] * shape[1]
        ts = _tensors([shape, shape], BF16, BF16, True, 6, gpu)
        big = {k: torch.full((4000,), 3, dtype=ts[k][0].dtype, device=gpu) for k in ("params", "momentums", "masters")}
        for k, buf in big.items():
            for i, at in enumerate((8, 2000)):
                buf[at:at + n] = ts[k][i].reshape(-1)
                ts[k][i] = buf[at:at + n].view(shape)
        ops.muon_step(**ts, **HP)
        for buf in big.values():
            assert (torch.cat([buf[:8], buf[8 + n:2000], buf[2000 + n:]]) == 3).all()


def test_step_replayed_from_a_graph(gpu):
    ts = _tensors(SPECS, BF16, BF16, True, 8, gpu)
    want = _copy(ts)
    x = matrix(100, 130, "plain", 1).float().to(gpu)
    ops.orthogonalize(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.muon_step(**ts, **HP)
        y = ops.orthogonalize(x)
    for i in range(4):
        x.mul_(1.5).add_(0.01)
        graph.replay()
        torch.cuda.synchronize()
        ops.muon_step(**want, **HP)  # eager work between the replays
        assert torch.equal(y, ops.orthogonalize(x))
        torch.cuda.synchronize()
        for k in ts:
            assert all(a is None or torch.equal(a, b) for a, b in zip(ts[k], want[k])), (i, k)


def test_other_streams_at_once(gpu):
    """Two steps and two products on streams of their own, as one after the other."""
    sets = [_tensors(SPECS, F32, F32, False, 9 + i, gpu) for i in range(2)]
    xs = [matrix(200, 300, "plain", i).to(BF16).to(gpu) for i in range(2)]
    want = [_copy(s) for s in sets]
    for w in want:
        ops.muon_step(**w, **HP)
    wx = [ops.orthogonalize(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s, ts, x in zip(streams, sets, xs):
        with torch.cuda.stream(s):
            ops.muon_step(**ts, **HP)
            got.append(ops.orthogonalize(x))
    torch.cuda.synchronize()
    for ts, w, x, y in zip(sets, want, got, wx):
        assert torch.equal(x, y)
        for k in ts:
            assert all(a is None or torch.equal(a, b) for a, b in zip(ts[k], w[k])), k


def test_refusals(gpu):
    ts = _tensors([(12, 20), (20, 12)], BF16, F32, True, 31, gpu)
    before = _copy(ts)
    for over, msg in (
            (dict(grads=ts["grads"][::-1]), "grads"), (dict(grads=[g.half() for g in ts["grads"]]), "grads"),
            (dict(momentums=[t.cpu() for t in ts["momentums"]]), "GPU"), (dict(params=[t.float() for t in ts["params"]]), "masters"),
            (dict(grads=[ts["momentums"][0], ts["grads"][1]]), "gradient overlaps"), (dict(params=[ts["params"][0]] * 2, grads=[ts["grads"][0]] * 2,
             momentums=[t.view(12, 20) for t in ts["momentums"]], masters=[t.view(12, 20) for t in ts["masters"]]), "overlap"),
            (dict(lr=float("nan")), "finite"), (dict(lr=[1e-3]), "one entry")):
        with pytest.raises(ValueError, match=msg):
            ops.muon_step(**{**ts, **HP, **over})
    for k in ts:
        assert all(torch.equal(x, y) for x, y in zip(ts[k], before[k])), k


def test_optimizer_and_its_state_dict(gpu):
    """Three steps of two optimizers, the second loaded from the first's state after two, the first against the oracle."""
    gen = torch.Generator().manual_seed(10)

    def model():
        torch.manual_seed(0)
        return torch.nn.Sequential(torch.nn.Linear(64, 96, bias=False), torch.nn.Linear(96, 8, bias=False)).to(gpu).bfloat16()

    grads = [[torch.randn(p.shape, generator=gen).to(gpu).bfloat16() for p in model().parameters()] for _ in range(3)]

    def step(opt, net, k):
        for p, g in zip(net.parameters(), grads[k]):
            p.grad = g.clone()
        opt.step()

    def make(net):
        ps = list(net.parameters())
        return Muon([dict(params=ps[:1], weight_decay=0.1), dict(params=ps[1:], lr=2e-2)], lr=1e-2, weight_decay=0.0, adjust="match_rms_adamw")

    a = model()
    ref = [(p.detach().cpu().double(), torch.zeros(p.shape, dtype=torch.float64), 0.0) for p in a.parameters()]
    oa = make(a)
    for k in range(2):
        step(oa, a, k)
    b = model()
    b.load_state_dict(a.state_dict())
    ob = make(b)
    ob.load_state_dict(oa.state_dict())
    step(oa, a, 2)
    step(ob, b, 2)
    assert all(torch.equal(x, y) for x, y in zip(a.parameters(), b.parameters()))
    for i, p in enumerate(a.parameters()):
        w, m, tol = ref[i]
        for k in range(3):
            w, m, off = O.muon(w, grads[k][i].cpu().double(), m, (1e-2, 2e-2)[i], 0.95, True, (0.1, 0.0)[i], "match_rms_adamw", True)
            tol += off + 4 * U * float(w.norm())
        assert float((oa.state[p]["master"].cpu().double() - w).norm()) <= 1.5 * tol  # a step's roundings in the next one's momentum: 4 u of it
        assert torch.equal(p.detach(), oa.state[p]["master"].to(BF16))


def test_a_block_trained_with_its_losses_and_both_optimizers(gpu):
    """Routing, experts, the balance's losses, every gradient, Muon on the matrices and AdamW on the rest: the gradients
    are the task's plus the losses', and the steps take them."""
    torch.manual_seed(0)
    mlp = modules.ExpertMlp(64, 96, 4, 2).to(gpu).bfloat16()
    g = torch.Generator().manual_seed(4)
    x, dy = (torch.randn(2, 150, 64, generator=g).to(BF16).to(gpu) for _ in range(2))
    some, rest = matrices(mlp)
    assert len(some) == 3 and len(rest) == 2

    def backward(weight):
        mlp.zero_grad()
        with modules.RoutingLosses(per_sample=True) as routing:
            out = mlp(x)
        ((out * dy).sum() + weight * (routing.balance + 0.1 * routing.z)).backward()
        return {n: p.grad.clone() for n, p in mlp.named_parameters()}, routing

    plain, _ = backward(0.0)
    both, routing = backward(5.0)
    ((m, load),) = routing.load
    assert m is mlp and int(load.sum()) == 600
    assert torch.equal(plain["w1"], both["w1"]) and not torch.equal(plain["router.weight"], both["router.weight"])
    steps = [Muon(some, lr=1e-2, adjust="match_rms_adamw"), AdamW(rest, lr=1e-2)]
    before = {n: p.detach().clone() for n, p in mlp.named_parameters()}
    for s in steps:
        s.step()
    for n, p in mlp.named_parameters():
        assert torch.isfinite(p).all() and not torch.equal(p, before[n]), n
    for n, p in mlp.named_parameters():
        if n in ("b1", "b2"):
            continue
        w0 = before[n].cpu().double().reshape(-1, *p.shape[-2:])
        got = steps[0].state[p]["master"].cpu().double().reshape(w0.shape)
        for j in range(len(w0)):
            gr = both[n].cpu().double().reshape(w0.shape)[j]
            w, _, off = O.muon(w0[j], gr, torch.zeros_like(gr), 1e-2, 0.95, True, 0.1, "match_rms_adamw", True)
            assert float((got[j] - w).norm()) <= off + 5 * U * float(w.norm())
    # and the next step runs on what they left
    del routing
    backward(5.0)
    for s in steps:
        s.step()
    assert all(torch.isfinite(p).all() for p in mlp.parameters())
