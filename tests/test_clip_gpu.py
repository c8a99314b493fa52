"""The norm of all gradients and their clipping against 64 bits: tensors of every size and alignment, types, extremes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
SENTINEL = 31000.0
# A sum of eight squares in f32: each product and addition half a step, eight of them at most on one value; the rest is 64 bits. Half of that for
# the root, one rounding of the result.
NORM_TOL = (8 / 2 + 1) * 2.0 ** -24


def _flat(sizes, dtype, lead, std=1.0):
    """Tensors one behind the other from `lead` on in one vector full of sentinels."""
    whole = torch.full((lead + sum(sizes) + 40,), SENTINEL, device="cuda", dtype=dtype)
    part = whole[lead:lead + sum(sizes)]
    part.copy_((torch.randn(sum(sizes), device="cuda") * std).to(dtype))
    return list(part.split(sizes)), whole


def _norm(ts, scale=1.0):
    return abs(scale) * math.sqrt(sum(float(t.double().square().sum()) for t in ts))


def _check_out(out, ref, want_coef, scale):
    for o, r in zip(out, ref):
        want = r.double() * want_coef * scale
        # the coefficient to NORM_TOL and a rounding to f32, the product one rounding, the output's type half a step (or of its denormals)
        tol = want.abs() * (NORM_TOL + 3 * 2.0 ** -24 + torch.finfo(o.dtype).eps / 2) + torch.finfo(o.dtype).smallest_normal * torch.finfo(o.dtype).eps
        assert ((o.double() - want).abs() <= tol).all()


SIZES = [[1], [7], [8], [9, 1, 3], [4096], [4095, 4097, 0, 5], [100352, 128, 1280, 10], [333 * 517, 333, 2, 1, 1, 1], [1] * 300, [0, 0], [40000, 0, 12345], [3] * 700 + [5000]]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("lead", [0, 3])
def test_norm_and_clipping(sizes, dtype, lead):
    from oxidized_neural_orchestra_b200.ops.clip import clip_grads, grad_norm

    torch.manual_seed(len(sizes))
    ts, whole = _flat(sizes, dtype, lead)
    for scale in (1.0, -0.25):
        want = _norm(ts, scale)
        for max_norm in (want / 3 + 1e-3, want * 2 + 1.0, math.inf):
            c = min(1.0, max_norm / want) if want else 1.0
            norm, coef = torch.full((1,), -1.0, device="cuda"), torch.full((1,), -1.0, device="cuda")
            grad_norm(ts, norm, max_norm=max_norm, coef=coef, scale=scale)
            assert abs(norm.item() - want) <= NORM_TOL * want and abs(coef.item() - c) <= (NORM_TOL + 2.0 ** -24) * c
            for out_dtype, out_lead in ((F32, lead), (BF16, lead), (F16, 5), (dtype, 1)):
                out, ow = _flat(sizes, out_dtype, out_lead)
                n2, c2 = torch.empty(1, device="cuda"), torch.empty(1, device="cuda")
                clip_grads(ts, max_norm, scale=scale, norm=n2, coef=c2, out=out)
                assert torch.equal(n2, norm) and torch.equal(c2, coef)
                _check_out(out, ts, c, scale)
                assert (ow[:out_lead] == SENTINEL).all() and (ow[out_lead + sum(sizes):] == torch.tensor(SENTINEL, dtype=out_dtype)).all()
    before, at = [t.clone() for t in ts], whole.clone()
    n3 = torch.empty(1, device="cuda")
    clip_grads(ts, 1e30, norm=n3)      # nothing to clip: not a bit changes
    assert torch.equal(whole, at)
    limit = _norm(ts) / 2 + 1e-3
    clip_grads(ts, limit, scale=2.0)
    _check_out(ts, before, min(1.0, limit / (2 * _norm(before))) if _norm(before) else 1.0, 2.0)
    assert (whole[:lead] == SENTINEL).all() and (whole[lead + sum(sizes):] == torch.tensor(SENTINEL, dtype=dtype)).all()


def test_tensors_of_several_types_in_one_call():
    from oxidized_neural_orchestra_b200.ops.clip import clip_grads, grad_norm

    torch.manual_seed(1)
    ts = [torch.randn(37, 91, device="cuda"), torch.randn(5003, device="cuda").to(BF16), torch.randn(2, 3, 4, device="cuda").to(F16), torch.zeros(70000, device="cuda")]
    before, want = [t.clone() for t in ts], _norm(ts)
    norm = torch.empty((), device="cuda")
    grad_norm(ts, norm)
    assert abs(norm.item() - want) <= NORM_TOL * want
    clip_grads(ts, 2.5)
    _check_out(ts, before, 2.5 / want, 1.0)
    grad_norm([t for t in ts for _ in range(2)], norm)      # a tensor that is named twice counts twice
    assert abs(norm.item() - 2.5 * math.sqrt(2)) <= 2.0 ** -7
    grad_norm([], norm)
    assert norm.item() == 0.0


@pytest.mark.parametrize("value", [1e30, 3e38, 1e-30, 1.4e-45, 2e18, 1e-24])
def test_values_whose_squares_leave_f32(value):
    from oxidized_neural_orchestra_b200.ops.clip import clip_grads, grad_norm

    t = torch.full((10001,), value, device="cuda")
    t[::3] = 0.0
    t[1::7] *= 0.5 if value > 1e-44 else 1.0
    want, norm, coef = _norm([t]), torch.empty(1, device="cuda"), torch.empty(1, device="cuda")
    grad_norm([t], norm, max_norm=1.0, coef=coef)
    if want < 3.4e38:
        assert abs(norm.item() - want) <= max(NORM_TOL * want, 1.4e-45)
    else:
        assert norm.item() == math.inf
    assert abs(coef.item() - min(1.0, 1.0 / want)) <= max(2 * NORM_TOL * min(1.0, 1.0 / want), 1.4e-45)
    out = [torch.empty_like(t)]
    clip_grads([t], 1.0, out=out)
    if want > 1.0:
        # (a coefficient below the smallest normal f32 has fewer bits: a step of 2^-149 of it)
        c = 1.0 / want
        assert ((out[0].double() - t.double() * c).abs() <= (t.double() * c).abs() * 8 * 2.0 ** -24 + t.double().abs() * 2.0 ** -149).all()
    else:
        assert torch.equal(out[0], t)


def test_infinities_and_nan():
    from oxidized_neural_orchestra_b200.ops.clip import clip_grads, grad_norm

    for bad, norm_is, rest in ((math.inf, math.inf, 0.0), (math.nan, math.nan, math.nan)):
        t = torch.ones(5000, device="cuda")
        t[4321] = bad
        norm, coef = torch.empty(1, device="cuda"), torch.empty(1, device="cuda")
        grad_norm([t], norm, max_norm=1.0, coef=coef)
        assert torch.equal(norm.cpu(), torch.tensor([norm_is])) or norm.isnan().item() and math.isnan(norm_is)
        assert coef.item() == rest or math.isnan(rest) and coef.isnan().item()
        clip_grads([t], 1.0)
        assert t[4321].isnan().item() and (t[0].item() == rest or math.isnan(rest) and t[0].isnan().item())


def test_same_bits_on_streams_and_in_graphs():
    from oxidized_neural_orchestra_b200.ops.clip import clip_grads, clip_scratch

    torch.manual_seed(2)
    sets = []
    for sizes in ([123457, 1001, 77], [4000000]):
        ts, _ = _flat(sizes, F32, 3)
        sets.append((ts, [torch.empty_like(t) for t in ts], torch.empty(1, device="cuda")))
    call = lambda s, **kw: clip_grads(s[0], 1.0, out=s[1], norm=s[2], **kw)  # noqa: E731
    for s in sets:
        call(s)
    wanted = [([o.clone() for o in s[1]], s[2].clone()) for s in sets]
    same = lambda: all(torch.equal(s[2], w[1]) and all(torch.equal(a, b) for a, b in zip(s[1], w[0])) for s, w in zip(sets, wanted))  # noqa: E731

    def clear():
        for s in sets:
            s[2].fill_(-1)
            for o in s[1]:
                o.fill_(-1)
        torch.cuda.synchronize()

    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        clear()
        for s, st in zip(sets, streams):
            call(s, stream=st)
        torch.cuda.synchronize()
        assert same()
    graphs = []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(s)
        graphs.append(g)
    for _ in range(5):
        clear()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert same()
    clear()
    own = [torch.empty(clip_scratch(), device="cuda", dtype=torch.uint8) for _ in sets]
    for s, o in zip(sets, own):
        call(s, scratch=o)
    assert same()


@pytest.mark.parametrize("kind", ["sgd", "momentum", "adam"])
def test_optimizer_takes_the_coefficient(kind):
    """The step with the coefficient equals the step on gradients clipped beforehand, to the roundings of one more product."""
    from oxidized_neural_orchestra_b200.ops import elementwise as ew
    from oxidized_neural_orchestra_b200.ops.clip import clip_grads, grad_norm

    torch.manual_seed(9)
    n = 100003
    g, p0, m0, v0 = (torch.randn(n, device="cuda") * s for s in (1.0, 1.0, 0.1, 0.1))
    v0.square_()
    norm, coef, pows = torch.empty(1, device="cuda"), torch.empty(1, device="cuda"), torch.tensor([0.5, 0.9], device="cuda")
    hp = dict(kind=kind, lr=0.01, mu=0.9, b1=0.9, b2=0.999, eps=1e-8, adam_pows=pows)
    got = []
    for clipped in (False, True):
        p, m, v = p0.clone(), m0.clone(), v0.clone()
        if clipped:
            out = [torch.empty_like(g)]
            clip_grads([g], 1.5, scale=0.5, out=out)
            ew.optim_step(p, out[0], m=m, v=v, grad_coef=torch.ones(1, device="cuda"), **hp)
        else:
            grad_norm([g], norm, max_norm=1.5, coef=coef, scale=0.5)
            ew.optim_step(p, g, m=m, v=v, grad_scale=0.5, grad_coef=coef, **hp)
        got.append((p, m, v))
    if kind == "adam":      # v itself, of numbers where 1 - b2 counts: b2 v + (1 - b2) g^2 with the rounding of each part
        c = 1.5 / (0.5 * math.sqrt(float(g.double().square().sum())))
        parts = 0.999 * v0.double(), 0.001 * (0.5 * c * g.double()).square()
        assert ((got[0][2].double() - parts[0] - parts[1]).abs() <= 2.0 ** -24 * (3 * parts[0] + 24 * parts[1])).all()
        zero, m, v = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
        ew.optim_step(zero, g, m=m, v=v, grad_coef=torch.ones(1, device="cuda"), **hp)
        assert ((v.double() - 0.001 * g.double().square()).abs() <= 4 * 2.0 ** -24 * 0.001 * g.double().square() + 1e-44).all()
        assert ((m.double() - 0.1 * g.double()).abs() <= 3 * 2.0 ** -24 * 0.1 * g.double().abs() + 1e-44).all()
    want = 0.5 * math.sqrt(float(g.double().square().sum()))
    assert abs(norm.item() - want) <= NORM_TOL * want and abs(coef.item() - 1.5 / want) <= 2 * NORM_TOL * 1.5 / want
    for a, b, start in zip(got[0], got[1], (p0, m0, v0)):
        # four roundings of the gradient and the update's own few, relative to what is added up
        assert ((a - b).abs() <= 16 * 2.0 ** -24 * (start.abs() + b.abs() + 0.05)).all()


@pytest.mark.parametrize("dtype,out_dtype,total", [(BF16, F32, 17_000_011), (F16, F16, 17_000_011), (F32, BF16, 34_000_011), (F32, F32, 34_000_011)])
def test_many_values(dtype, out_dtype, total):
    """So many values that a thread has twice as many in flight: tensors of every alignment, groups that are not whole, a tensor shorter than one."""
    from oxidized_neural_orchestra_b200.ops.clip import clip_grads

    torch.manual_seed(3)
    sizes = [1, 5, 8191, 8193, 16384, 3, 1_000_003, total // 2]
    sizes.append(total - sum(sizes))
    ts, whole = _flat(sizes, dtype, 3)
    want = _norm(ts)
    out, ow = _flat(sizes, out_dtype, 3 if dtype == out_dtype else 6)
    norm, coef = torch.empty(1, device="cuda"), torch.empty(1, device="cuda")
    clip_grads(ts, want / 3, norm=norm, coef=coef, out=out)
    assert abs(norm.item() - want) <= NORM_TOL * want
    _check_out(out, ts, 1 / 3, 1.0)
    lead = 3 if dtype == out_dtype else 6
    assert (ow[:lead] == SENTINEL).all() and (ow[lead + total:] == torch.tensor(SENTINEL, dtype=out_dtype)).all()
    before = [t.clone() for t in ts]
    clip_grads(ts, want / 3)
    _check_out(ts, before, 1 / 3, 1.0)
    assert (whole[:3] == SENTINEL).all() and (whole[3 + total:] == torch.tensor(SENTINEL, dtype=dtype)).all()


@pytest.mark.parametrize("count", [31, 33, 300])
def test_many_tensors_of_several_types(count):
    """On both sides of the number of tensors that one cluster takes, and more than a launch takes."""
    from oxidized_neural_orchestra_b200.ops.clip import clip_grads, grad_norm

    torch.manual_seed(count)
    kinds = (F32, BF16, F16)
    ts = [torch.randn(1 + 37 * k % 1500, device="cuda").to(kinds[k % 3]) for k in range(count)]
    out = [torch.empty(t.numel(), device="cuda", dtype=kinds[(k // 3) % 3]) for k, t in enumerate(ts)]
    want = _norm(ts, 0.5)
    norm, n2, coef = (torch.empty(1, device="cuda") for _ in range(3))
    grad_norm(ts, norm, max_norm=want / 7, coef=coef, scale=0.5)
    clip_grads(ts, want / 7, scale=0.5, norm=n2, out=out)
    assert abs(norm.item() - want) <= NORM_TOL * want and torch.equal(norm, n2) and abs(coef.item() - 1 / 7) <= (NORM_TOL + 2.0 ** -24) / 7
    _check_out(out, ts, 1 / 7, 0.5)


@pytest.mark.parametrize("n", [1, 4096 * 16, 4096 * 32 - 3, 4096 * 32 - 2, 4096 * 32, 4096 * 32 + 1])
def test_sizes_around_what_one_cluster_takes(n):
    from oxidized_neural_orchestra_b200.ops.clip import clip_grads

    torch.manual_seed(5)
    for lead in (0, 3):
        ts, whole = _flat([n], BF16, lead)
        before, want, norm = [t.clone() for t in ts], _norm(ts), torch.empty(1, device="cuda")
        clip_grads(ts, want / 2, norm=norm)
        assert abs(norm.item() - want) <= NORM_TOL * want
        _check_out(ts, before, 0.5, 1.0)
        assert (whole[:lead] == SENTINEL).all() and (whole[lead + n:] == torch.tensor(SENTINEL, dtype=BF16)).all()


def _adam(p, g, m, v, pows, lr, b1, b2, eps, **kw):
    from oxidized_neural_orchestra_b200.ops import elementwise as ew

    ew.adam_tick(pows, b1, b2)
    ew.optim_step(p, g, kind="adam", lr=lr, b1=b1, b2=b2, eps=eps, m=m, v=v, adam_pows=pows, **kw)


@pytest.mark.parametrize("exact", [False, True])
def test_a_coefficient_of_one_is_no_other_step(exact):
    """Adam over several steps: the same bits with a coefficient of one as without, and both the 64-bit recurrence of the betas that were asked for."""
    torch.manual_seed(2)
    n, steps, lr, b1, b2, eps = 50003, 5, 1e-3, 0.9, 0.999, 1e-8
    gs = [torch.randn(n, device="cuda") for _ in range(steps)]
    p0, one, sets = torch.randn(n, device="cuda"), torch.ones(1, device="cuda"), []
    for kw in (dict(grad_coef=one, exact_betas=exact), dict(exact_betas=exact), dict(grad_coef=one) if exact else {}):
        p, m, v, pows, powers = p0.clone(), torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda"), torch.ones(2, device="cuda"), []
        for g in gs:
            _adam(p, g, m, v, pows, lr, b1, b2, eps, **kw)
            powers.append(pows.double())
        sets.append((p, m, v))
    assert all(torch.equal(a, b) for s in sets[1:] for a, b in zip(sets[0], s))
    if not exact:
        b1, b2 = (float(torch.tensor(b)) for b in (b1, b2))
    p, m, v, size = p0.double(), 0.0, 0.0, 0.0
    for g, t in zip(gs, powers):
        g = g.double()
        m, v, size = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g, b1 * size + (1 - b1) * g.abs()
        step = lr * torch.sqrt(1 - t[1]) / (1 - t[0])
        p = p - step * m / (v.sqrt() + eps)
        moved = step * size / (v.sqrt() + eps)
    # a step's moments: four roundings at most, relative to the parts that are added up; a step of p: theirs, ten of its own, one of p
    u = 2.0 ** -24
    assert ((sets[0][1].double() - m).abs() <= 4 * steps * u * size).all() and ((sets[0][2].double() - v).abs() <= 4 * steps * u * v).all()
    assert ((sets[0][0].double() - p).abs() <= steps * u * (p.abs() + 0.01) + steps * (8 * steps + 10) * u * moved.clamp_min(20 * lr)).all()


def test_the_weights_of_the_second_moment_add_up_to_one():
    """After 4000 steps the mean of v over many values is that of 64 bits: its roundings are of either sign, some 11 units on a value (half a step in each of the
    last thousand or so, at random) and a few thousandths of one on the mean. Weights of 1.0000129 would show as that."""
    torch.manual_seed(3)
    n, b1, b2 = 65536, 0.9, 0.999
    gs, one = [torch.randn(n, device="cuda") for _ in range(16)], torch.ones(1, device="cuda")
    p, m, v, pows = (torch.zeros(k, device="cuda") for k in (n, n, n, 2))
    want = torch.zeros(n, device="cuda", dtype=torch.float64)
    pows.fill_(0.5)
    squares = [g.double().square() for g in gs]
    for k in range(4000):
        _adam(p, gs[k % 16], m, v, pows, 1e-6, b1, b2, 1e-8, grad_coef=one)
        pows.fill_(0.5)
        want.mul_(b2).add_(squares[k % 16], alpha=1 - b2)
    assert abs(float((v.double() / want).mean()) - 1.0) <= 2.0 ** -20


def test_moments_that_left_the_range_stay_there():
    for exact in (False, True):
        p, m, v = torch.zeros(4, device="cuda"), torch.tensor([math.inf, -math.inf, 1.0, 0.0], device="cuda"), torch.tensor([1.0, 1.0, math.inf, 1.0], device="cuda")
        g, pows = torch.tensor([1.0, 1.0, 1.0, 1e25], device="cuda"), torch.tensor([0.5, 0.5], device="cuda")
        _adam(p, g, m, v, pows, 0.1, 0.9, 0.999, 1e-8, exact_betas=exact)
        assert m[:2].tolist() == [math.inf, -math.inf] and v[2:].tolist() == [math.inf, math.inf] and p[2:].tolist() == [0.0, 0.0]
