"""Log probabilities, entropy, alternatives, token loss and the logits' gradients against 64 bits, at the sizes, masks and values where they can go wrong."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
SENTINEL = -7.0e11
SIZES = [(1, 1), (3, 2), (5, 8), (2, 31), (40, 33), (300, 10), (7, 100), (37, 257), (19, 1000), (5, 1023), (6, 1025), (4, 2500), (9, 4097), (3, 10007), (5, 50257), (2, 128256), (2, 200003)]


def _logits(rows, vocab, dtype, ld=None, lead=0, std=3.0):
    ld = ld or vocab
    whole = torch.full((lead + rows * ld + 64,), SENTINEL, device="cuda", dtype=dtype)
    x = whole[lead:lead + rows * ld].view(rows, ld)[:, :vocab]
    x.copy_((torch.randn(rows, vocab, device="cuda") * std).to(dtype))
    return x, whole


def _ref(x, targets, vocab):
    """lp, logp, lse, entropy in 64 bits; rows that are not read zeros."""
    xd = x.double()
    empty = (xd == -math.inf).all(1)
    top = torch.where(empty, 0.0, xd.amax(1)).unsqueeze(1)
    log_z = torch.log(torch.exp(xd - top).sum(1, keepdim=True))
    lp, lse = (xd - top) - log_z, (top + log_z).squeeze(1)      # (a logarithm of the sum is lost beside a logit of 3e38, even in 64 bits)
    lp[empty] = -math.inf
    bad = (xd.isnan() | (xd == math.inf)).any(1)
    lp[bad], lse = math.nan, torch.where(bad, math.nan, lse)
    ent = -torch.where(lp > -math.inf, torch.exp(lp) * lp, torch.where(lp.isnan(), lp, 0.0)).sum(1)
    live = torch.ones(x.shape[0], dtype=torch.bool, device="cuda") if targets is None else (targets >= 0) & (targets < vocab)
    logp = lp.gather(1, targets.long().clamp(0, vocab - 1).unsqueeze(1)).squeeze(1) if targets is not None else None
    z = lambda v: torch.where(live, v, 0.0)  # noqa: E731
    return lp, None if logp is None else z(logp), z(lse), z(torch.where(empty, 0.0, ent)), live, empty


def _tol(vocab):
    # The sum of exponentials: at most V / 256 additions a thread and a tree, each half a step, and a term's own error (argument and
    # exponential, a few units weighted by exp(-d) d <= 0.4): V / 128 + 64 units of 2^-24, twice as much as that adds up to.
    return (vocab / 128 + 64) * 2.0 ** -24


def _near(got, ref, tol):
    f32 = ref.float()      # (differences of huge logits leave its range)
    assert torch.equal(got.isnan(), f32.isnan()) and torch.equal(got == -math.inf, f32 == -math.inf)
    ok = torch.isfinite(f32)
    assert torch.isfinite(got[ok]).all()
    assert ((got[ok].double() - ref[ok]).abs() <= tol * ref[ok].abs().clamp_min(1.0)).all(), (got[ok].double() - ref[ok]).abs().max()


def _top_ref(x, k, live):
    val, at = torch.sort(torch.where(x.isnan(), -math.inf, x.double() + 0.0), dim=1, descending=True, stable=True)
    there = (val[:, :k] > -math.inf) & live.unsqueeze(1)
    return torch.where(there, at[:, :k], -1).int(), there


def _check_forward(x, targets, k, ignore=-1):
    from oxidized_neural_orchestra_b200.ops.token_loss import token_logprobs

    rows, vocab = x.shape
    out = [torch.full((rows,), SENTINEL, device="cuda") for _ in range(3)]
    top = torch.full((rows, k), SENTINEL, device="cuda") if k else None
    tid = torch.full((rows, k), 77, device="cuda", dtype=torch.int32) if k else None
    token_logprobs(x, targets, logp=out[0] if targets is not None else None, lse=out[1], entropy=out[2], top_logp=top, top_id=tid, ignore_id=ignore)
    lp, logp, lse, ent, live, empty = _ref(x, targets, vocab)
    tol = _tol(vocab)
    if targets is not None:
        _near(out[0], logp, tol)
    _near(out[1], lse, tol)
    _near(out[2], ent, tol)
    if k:
        want, there = _top_ref(x, k, live)
        assert torch.equal(tid, want)
        val = torch.where(there, lp.gather(1, want.long().clamp_min(0)), -math.inf)
        bad = lp.isnan().any(1)
        assert top[bad.unsqueeze(1) & there].isnan().all()
        _near(top[~bad], val[~bad], tol)
    return out


def _check_loss(x, whole, targets, out_dtype, in_place=False):
    from oxidized_neural_orchestra_b200.ops.token_loss import token_loss

    rows, vocab = x.shape
    lp, logp, _, _, live, empty = _ref(x, targets, vocab)
    weight, scale = torch.rand(rows, device="cuda") + 0.5, 0.37
    got_logp = torch.empty(rows, device="cuda")
    if in_place:
        d, dw = x, whole
    else:
        ld = x.stride(0) if rows > 1 else vocab
        dw = torch.full((rows * ld + 72,), SENTINEL, device="cuda", dtype=out_dtype)
        d = dw[3:3 + rows * ld].view(rows, ld)[:, :vocab]
    token_loss(x, targets, out=d, logp=got_logp, weight=weight, scale=scale)
    p = torch.exp(lp)
    one = torch.zeros_like(p).scatter_(1, targets.long().clamp(0, vocab - 1).unsqueeze(1), 1.0)
    w = (scale * weight).double().unsqueeze(1)
    ref = w * (p - one)
    ref[~live | empty] = 0.0
    # w p: the sum's error, a few units of its own; the subtraction half a step of 1; then the output's type, half a step of the value.
    # (an exponential below the smallest normal f32 counts as zero)
    tol = w * (p.nan_to_num(0) + one) * _tol(vocab) + (torch.finfo(out_dtype).eps / 2) * ref.abs() * 1.01 + 1e-37
    assert torch.equal(d.isnan(), ref.isnan())
    ok = ~ref.isnan()
    assert ((d.double() - ref).abs()[ok] <= tol.nan_to_num(0)[ok]).all()
    _near(got_logp, logp, _tol(vocab))
    flags = torch.zeros_like(dw, dtype=torch.bool)
    flags.as_strided(d.shape, (d.stride(0), 1), d.storage_offset()).fill_(True)
    assert (dw[~flags] == torch.tensor(SENTINEL, dtype=dw.dtype)).all()


def _check_grad(x, targets, out_dtype, logp=True, entropy=True):
    from oxidized_neural_orchestra_b200.ops.token_loss import token_logprobs, token_logprobs_grad

    rows, vocab = x.shape
    lse, ent = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    token_logprobs(x, targets, lse=lse, entropy=ent)
    g, h = torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda")
    dw = torch.full((rows * vocab + 72,), SENTINEL, device="cuda", dtype=out_dtype)
    d = dw[5:5 + rows * vocab].view(rows, vocab)
    token_logprobs_grad(x, targets, lse=lse, out=d, d_logp=g if logp else None, entropy=ent if entropy else None, d_entropy=h if entropy else None)
    lp, _, rlse, H, live, empty = _ref(x, targets, vocab)
    p = torch.exp(lp)
    gd = g.double().unsqueeze(1) if logp else torch.zeros(rows, 1, device="cuda", dtype=torch.float64)
    hd = h.double().unsqueeze(1) if entropy else torch.zeros(rows, 1, device="cuda", dtype=torch.float64)
    one = torch.zeros_like(p)
    if targets is not None:
        one.scatter_(1, targets.long().clamp(0, vocab - 1).unsqueeze(1), 1.0)
    inner = torch.where(p > 0, lp + H.unsqueeze(1), torch.where(lp.isnan(), lp, 0.0))
    ref = gd * (one - p) - hd * p * inner
    ref[~live | empty] = 0.0
    # d = -p (g + h (lp + H)), so its error is (error of p) (g + h (lp + H)) + p h (error of lp + error of H). lse comes rounded to f32, half a step
    # of it, which is relative in p and absolute in lp (of 128 at most: beyond that the kernel takes the logits themselves); H has an absolute error of _tol max(1, H) (see _near: it is a difference of
    # numbers of size 1 where it is small), so h (lp + H) counts with at least h.
    size = p * (gd.abs() + hd.abs() * (inner.abs() + 2 * H.unsqueeze(1).clamp_min(1.0) + lp.clamp_min(-1e4).abs())) + one * gd.abs()
    tol = size * (_tol(vocab) + 2.0 ** -23 * rlse.abs().unsqueeze(1).nan_to_num(0, 0, 0).clamp_max(128.0)) + (torch.finfo(out_dtype).eps / 2) * ref.abs() * 1.01 + 1e-36
    assert torch.equal(d.isnan(), ref.isnan())
    ok = ~ref.isnan()
    assert ((d.double() - ref).abs()[ok] <= tol.nan_to_num(0)[ok]).all()
    assert (dw[:5] == torch.tensor(SENTINEL, dtype=out_dtype)).all() and (dw[5 + rows * vocab:] == torch.tensor(SENTINEL, dtype=out_dtype)).all()


@pytest.mark.parametrize("rows,vocab", SIZES)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_against_64_bits(rows, vocab, dtype):
    torch.manual_seed(vocab)
    for ld, lead in ((None, 0), (-(-vocab // 16) * 16, 0), (vocab + 5, 3)):
        x, whole = _logits(rows, vocab, dtype, ld, lead)
        targets = torch.randint(-1, vocab, (rows,), device="cuda", dtype=torch.int32 if lead else torch.int64)
        for k in sorted({0, 1, min(5, vocab), min(20, vocab), min(32, vocab)}):
            _check_forward(x, targets, k)
        _check_forward(x, None, min(3, vocab))
        for out_dtype in (F32, BF16):
            _check_loss(x, whole, targets, out_dtype)
            _check_grad(x, targets, out_dtype)
        _check_grad(x, targets, dtype, entropy=False)
        _check_grad(x, None, dtype, logp=False)
        _check_loss(x, whole, targets, dtype, in_place=True)


def _special(kind, x):
    rows, vocab = x.shape
    low = torch.finfo(x.dtype).min
    if kind == "equal":
        x.fill_(1.5)
    elif kind == "zeros of both signs":
        x.zero_()
        x[:, 1::2] = -0.0
    elif kind == "ascending":
        x.copy_(torch.linspace(-8, 8, vocab, device="cuda").expand(rows, vocab))
    elif kind == "descending":
        x.copy_(torch.linspace(8, -8, vocab, device="cuda").expand(rows, vocab))
    elif kind == "sawtooth":      # the large ones all at the same place of every group of 256 and of 2048
        x[:, ::256] += 9.0
        x[:, 8::2048] += 9.0
    elif kind == "few values":
        x.copy_((x / 2).round() * 2)
    elif kind == "one allowed":
        x.fill_(-math.inf)
        x[:, vocab // 2] = 3.0
    elif kind == "three allowed":
        keep = x[:, [0, vocab // 3, vocab - 1]].clone()
        x.fill_(-math.inf)
        x[:, [0, vocab // 3, vocab - 1]] = keep
    elif kind == "nothing allowed":
        x[::2] = -math.inf
    elif kind == "masked by the lowest value":
        x[:, ::2] = low
        x[0] = low
        x[1] = low
        x[1, vocab // 2] = 0.0
    elif kind == "huge":
        x.copy_((x.float() * 1e37).to(x.dtype))
        x[0, vocab // 2] = 3.3e38
        x[1] = 3.0e38
        x[2, 0] = -3.3e38
    elif kind == "far from zero":
        x += 1000.0
        x[1] -= 3000.0
    elif kind == "infinity":
        x[0, vocab - 1] = math.inf
        x[1, 0] = math.inf
        x[1, 1] = -math.inf
    elif kind == "nan":
        x[0, vocab - 1] = math.nan
        x[1, 0] = -math.nan
        x[2] = math.nan
        x[3] = -math.inf
        x[3, 2] = math.nan


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [10, 100, 1000, 1030, 5003, 60000])
@pytest.mark.parametrize("kind", ["equal", "zeros of both signs", "ascending", "descending", "sawtooth", "few values", "one allowed", "three allowed", "nothing allowed",
                                  "masked by the lowest value", "huge", "far from zero", "infinity", "nan"])
def test_rows_of_every_kind(kind, vocab, dtype):
    torch.manual_seed(7)
    x, whole = _logits(6, vocab, dtype, vocab + 3)
    _special(kind, x)
    targets = torch.tensor([0, vocab // 2, 1, -1, vocab - 1, vocab // 3], device="cuda")
    _check_forward(x, targets, min(20, vocab))
    _check_forward(x, None, min(7, vocab))
    _check_loss(x, whole, targets, BF16)
    _check_grad(x, targets, F32)
    _check_loss(x, whole, targets, dtype, in_place=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", [(2400, 1030), (2400, 2500), (2500, 7001), (2368, 4099), (700, 9000), (200, 30011), (3000, 64), (5000, 3), (601, 250)])
def test_many_rows_of_mixed_kinds(rows, vocab, dtype):
    """As many rows as take other forms than a few do (a warp to a row, several rows to a warp, one CTA to a row), extraordinary ones among them."""
    torch.manual_seed(rows)
    x, whole = _logits(rows, vocab, dtype, vocab + 1 if rows % 3 else None)
    kinds = ["equal", "ascending", "few values", "one allowed", "nothing allowed", "masked by the lowest value", "huge", "far from zero", "infinity", "nan"]
    for k, kind in enumerate(kinds):
        _special(kind, x[7 + 11 * k:13 + 11 * k])
    targets = torch.randint(-1, vocab, (rows,), device="cuda")
    for k in sorted({0, 1, min(5, vocab), min(20, vocab)}):
        _check_forward(x, targets, k)
    _check_grad(x, targets, dtype)
    _check_grad(x, None, BF16, logp=False)
    _check_loss(x, whole, targets, BF16)
    _check_loss(x, whole, targets, dtype, in_place=True)


def test_ignored_and_unknown_targets():
    from oxidized_neural_orchestra_b200.ops.token_loss import token_logprobs, token_logprobs_grad, token_loss

    x = torch.randn(6, 50, device="cuda")
    x[1], x[2] = math.nan, math.nan      # rows that are not read
    targets = torch.tensor([3, -100, -100, 4, 50, 2**33], device="cuda")
    logp, lse, d = torch.ones(6, device="cuda"), torch.ones(6, device="cuda"), torch.ones(6, 50, device="cuda")
    top, tid = torch.ones(6, 2, device="cuda"), torch.ones(6, 2, device="cuda", dtype=torch.int32)
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    token_logprobs(x[:4], targets[:4], logp=logp[:4], lse=lse[:4], top_logp=top[:4], top_id=tid[:4], ignore_id=-100, status=status)
    assert status.item() == 0 and (logp[1:3] == 0).all() and (lse[1:3] == 0).all() and (tid[1:3] == -1).all() and (top[1:3] == -math.inf).all()
    token_logprobs(x, targets, logp=logp, lse=lse, ignore_id=-100, status=status)
    assert status.item() != 0 and (logp[4:] == 0).all() and logp[0] < 0 and logp[3] < 0
    status.zero_()
    token_loss(x, targets, out=d, ignore_id=-100, status=status)
    assert status.item() != 0 and not d[[1, 2, 4, 5]].any() and d[[0, 3]].all()
    d.fill_(1.0)
    status.zero_()
    token_logprobs_grad(x, targets, lse=lse, d_logp=torch.ones(6, device="cuda"), out=d, ignore_id=-100, status=status)
    assert status.item() != 0 and not d[[1, 2, 4, 5]].any() and d[[0, 3]].all()
    status.zero_()
    token_logprobs(x[:1], targets[:1], logp=logp[:1], ignore_id=None, status=status)
    assert status.item() == 0
    token_logprobs(x[1:2], targets[1:2], logp=logp[:1], ignore_id=None, status=status)
    assert status.item() != 0
    token_logprobs(x[:0], targets[:0], logp=logp[:0])      # no rows


def test_gradients_against_differences():
    """Central differences of the 64-bit definitions at the f32 logits."""
    from oxidized_neural_orchestra_b200.ops.token_loss import token_logprobs, token_logprobs_grad, token_loss

    torch.manual_seed(3)
    rows, vocab, h = 4, 23, 1e-4
    x, targets = torch.randn(rows, vocab, device="cuda") * 2, torch.tensor([0, 22, 7, 7], device="cuda")
    g, ge, w = torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda"), torch.rand(rows, device="cuda")

    def both(x):
        lp = torch.log_softmax(x, 1)
        logp, ent = lp.gather(1, targets.unsqueeze(1)).squeeze(1), -(lp.exp() * lp).sum(1)
        return g.double() * logp + ge.double() * ent, -w.double() * logp * 0.5

    num = torch.zeros(2, rows, vocab, device="cuda", dtype=torch.float64)
    for j in range(vocab):
        e = torch.zeros(vocab, device="cuda", dtype=torch.float64)
        e[j] = h
        for k, (a, b) in enumerate(zip(both(x.double() + e), both(x.double() - e))):
            num[k, :, j] = (a - b) / (2 * h)
    lse, ent, d1, d2 = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"), torch.empty_like(x), torch.empty_like(x)
    token_logprobs(x, targets, lse=lse, entropy=ent)
    token_logprobs_grad(x, targets, lse=lse, entropy=ent, d_logp=g, d_entropy=ge, out=d1)
    token_loss(x, targets, out=d2, weight=w, scale=0.5)
    # third derivatives of these functions are below 10: h^2 / 6 of them, and 2 eps64 |f| / h from the subtraction; f32 results to 100 units
    tol = 10 * h * h / 6 + 1e-11 + 100 * 2.0 ** -24 * 10
    assert (d1.double() - num[0]).abs().max().item() <= tol and (d2.double() - num[1]).abs().max().item() <= tol


def test_same_bits_on_streams_and_in_graphs():
    from oxidized_neural_orchestra_b200.ops.token_loss import token_logprobs, token_logprobs_grad, token_loss

    torch.manual_seed(5)
    sets = []
    for vocab, dtype in ((50257, BF16), (1000, F32)):
        x = torch.randn(40, vocab, device="cuda").to(dtype)
        t = torch.randint(0, vocab, (40,), device="cuda")
        f = lambda *s: torch.empty(*s, device="cuda")  # noqa: E731
        sets.append((x, t, f(40), f(40), f(40), f(40, 20), torch.empty(40, 20, device="cuda", dtype=torch.int32), torch.empty_like(x), torch.empty_like(x)))

    def call(s, stream=None):
        x, t, logp, lse, ent, top, tid, d1, d2 = s
        token_logprobs(x, t, logp=logp, lse=lse, entropy=ent, top_logp=top, top_id=tid, stream=stream)
        token_logprobs_grad(x, t, lse=lse, entropy=ent, d_logp=logp, d_entropy=ent, out=d1, stream=stream)
        token_loss(x, t, out=d2, scale=1 / 40, stream=stream)

    for s in sets:
        call(s)
    wanted = [[v.clone() for v in s] for s in sets]
    same = lambda: all(torch.equal(a, b) for s, w in zip(sets, wanted) for a, b in zip(s, w))  # noqa: E731

    def clear():
        for s in sets:
            for v in s[2:]:
                v.fill_(-3)
        torch.cuda.synchronize()

    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        clear()
        for s, st in zip(sets, streams):
            call(s, st)
        torch.cuda.synchronize()
        assert same()
    graphs = []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(s)
        graphs.append(graph)
    for _ in range(4):
        clear()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert same()


def test_rows_far_into_a_large_matrix():
    """Rows that begin past 2^31 values."""
    from oxidized_neural_orchestra_b200.ops.token_loss import token_logprobs, token_loss

    rows, vocab = 17000, 131000
    x = torch.zeros(rows, vocab, device="cuda", dtype=BF16)
    x[rows - 1].copy_(torch.randn(vocab, device="cuda").to(BF16) * 3)
    t = torch.full((rows,), -1, device="cuda")
    t[0], t[rows - 1] = 5, vocab - 1
    logp, lse = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    token_logprobs(x, t, logp=logp, lse=lse)
    ref = torch.log_softmax(x[rows - 1].double(), 0)
    assert abs(logp[rows - 1].item() - ref[vocab - 1].item()) <= _tol(vocab) * 20 and abs(logp[0].item() + math.log(vocab)) <= _tol(vocab) * 12
    assert logp.count_nonzero().item() == 2
    token_loss(x, t, out=x)
    want = torch.exp(ref)
    want[vocab - 1] -= 1
    assert ((x[rows - 1].double() - want).abs() <= want.abs() * 2.0 ** -8 * 1.02 + _tol(vocab) * torch.exp(ref)).all() and not x[1:rows - 1].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [129, 255, 400, 509, 519, 640, 900, 1019, 1027, 2043, 2061])
def test_alternatives_of_rows_of_few_logits_a_warp(vocab, dtype):
    """Rows that fill one warp or several, or leave the last one with a few logits or none: all different, equal, of few values, all but three masked."""
    torch.manual_seed(vocab)
    for kind in ("as drawn", "equal", "few values", "three allowed"):
        for ld, lead in ((-(-vocab // 16) * 16, 0), (vocab + 5, 3)):
            x, _ = _logits(5, vocab, dtype, ld, lead)
            _special(kind, x)
            targets = torch.randint(-1, vocab, (5,), device="cuda")
            for k in (1, 5, 8, 9, 20, 32):
                _check_forward(x, targets, k)


def test_two_threads_with_rows_of_different_lengths():
    """One kernel with two sizes of its shared memory, launched from two threads of the host at once (a call into the library lets other threads run):
    neither takes the other's allowance away."""
    import ctypes as C
    import threading

    from oxidized_neural_orchestra_b200.ops import _lib
    from oxidized_neural_orchestra_b200.ops.token_loss import token_loss

    torch.manual_seed(11)
    lib, jobs, failed = _lib.load(), [], []
    for vocab in (200003, 70001):
        x, t = torch.randn(1, vocab, device="cuda"), torch.randint(0, vocab, (1,), device="cuda")
        want, got = torch.empty_like(x), torch.zeros_like(x)
        token_loss(x, t, out=want)
        jobs.append((x, t, want, got, torch.cuda.Stream()))
    torch.cuda.synchronize()

    def work(x, t, want, got, stream):
        vocab = x.shape[1]
        a = _lib.OnoTokens(x=x.data_ptr(), targets=t.data_ptr(), R=1, ld=vocab, ld_out=vocab, ignore_id=-1, V=vocab, targets64=1, out=got.data_ptr(), scale=1.0)
        for k in range(2000):
            rc = lib.ono_tokens(C.byref(a), stream.cuda_stream)
            if rc:
                failed.append((vocab, k, rc))
            if k % 200 == 199:
                stream.synchronize()

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    torch.cuda.synchronize()
    assert not failed, failed[:5]
    assert all(torch.equal(want, got) for _, _, want, got, _ in jobs)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", [(40, 3), (40, 10), (40, 100), (40, 1000), (3000, 2500), (40, 2500), (40, 10007), (40, 50257), (3, 128256)])
def test_log_probabilities_are_rounded_as_the_definition_has_them(rows, vocab, dtype):
    """Whole logits, one of them 40 or more above all others: lse is that one, and the others' log probabilities their distances from it, to the bit. (The
    others weigh less than 1e-12; the sum is 1 to the 2^-22 of an exponential and the rounding of its shift, which is taken off again, so that its logarithm
    is below 2^-21, less than half a step of a number from 16 on.)"""
    from oxidized_neural_orchestra_b200.ops.token_loss import token_logprobs, token_loss

    torch.manual_seed(vocab)
    most = torch.randint(20, 101, (rows,), device="cuda")
    least = torch.randint(40, 101, (rows, vocab), device="cuda")
    at = torch.randint(0, vocab, (rows,), device="cuda")
    least[torch.arange(rows, device="cuda"), at] = 0
    x = (most.unsqueeze(1) - least).to(dtype)
    targets = torch.randint(0, vocab, (rows,), device="cuda")
    targets = torch.where(targets == at, (at + 1) % vocab, targets)
    want = -least.gather(1, targets.unsqueeze(1)).squeeze(1).float()
    k = min(4, vocab)
    logp, lse, top, tid = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"), torch.empty(rows, k, device="cuda"), torch.empty(rows, k, device="cuda", dtype=torch.int32)
    for kw in (dict(), dict(entropy=torch.empty(rows, device="cuda")), dict(top_logp=top, top_id=tid)):
        token_logprobs(x, targets, logp=logp, lse=lse, **kw)
        assert torch.equal(lse, most.float()) and torch.equal(logp, want)
    assert torch.equal(top[:, 1:], -least.gather(1, tid[:, 1:].long()).float()) and torch.equal(tid[:, 0].long(), at)
    lse.zero_(), logp.zero_()
    token_loss(x, targets, out=torch.empty_like(x), logp=logp, lse=lse)
    assert torch.equal(lse, most.float()) and torch.equal(logp, want)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", [(64, 3), (64, 10), (64, 100), (64, 1000), (3000, 1100), (64, 2500), (64, 10007)])
def test_gradient_with_what_rounding_took_off_lse(rows, vocab, dtype):
    """Rows of equal logits, p = 1 / V, whose lse is from 64 to 128 and rounded by up to 3.8e-6. With lse_low none of that is left: two exponentials of 2^-22 (one
    in the sum), at most 22 additions and ten other roundings of half a step. (A thread has at most 16 logits an accumulator at these sizes.)"""
    from oxidized_neural_orchestra_b200.ops.token_loss import token_logprobs, token_logprobs_grad

    torch.manual_seed(vocab)
    c = (torch.rand(rows, 1, device="cuda") * 50 + 64).to(dtype)
    x = c.expand(rows, vocab).contiguous()
    targets = torch.randint(0, vocab, (rows,), device="cuda")
    lse, low, ent, g = (torch.empty(rows, device="cuda") for _ in range(4))
    g.normal_()
    tol = 2 * 2.0 ** -22 + 32 * 2.0 ** -24
    want = (torch.zeros(rows, vocab, device="cuda", dtype=torch.float64).scatter_(1, targets.unsqueeze(1), 1.0) - 1.0 / vocab) * g.double().unsqueeze(1)
    for kw in (dict(), dict(entropy=ent), dict(entropy=ent, top_logp=torch.empty(rows, 2, device="cuda"), top_id=torch.empty(rows, 2, device="cuda", dtype=torch.int32))):
        low.fill_(SENTINEL)
        token_logprobs(x, targets, lse=lse, lse_low=low, **kw)
        # (log2 e as f32 has it is 1.4e-8 off)
        assert ((lse.double() + low.double() - c.double().squeeze(1) - math.log(vocab)).abs() <= tol + 1.4e-8 * math.log(vocab)).all()
        assert (low.abs() <= 2.0 ** -18 + tol).all()
        d = torch.empty(rows, vocab, device="cuda")
        token_logprobs_grad(x, targets, lse=lse, lse_low=low, d_logp=g, out=d)
        assert ((d.double() - want).abs() <= g.double().abs().unsqueeze(1) * (tol / vocab + 2.0 ** -24 * (want != 0))).all()
        other = torch.ones(rows, vocab, device="cuda") * SENTINEL
        token_logprobs_grad(x, targets, lse=lse, lse_low=low, d_logp=g, entropy=ent, d_entropy=torch.zeros_like(g), out=other)
        assert torch.equal(other.isnan(), d.isnan()) and ((other - d).abs() <= 4 * 2.0 ** -24 * d.abs() + 2.0 ** -24 * g.abs().unsqueeze(1)).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", [(12, 50), (12, 1030), (2400, 1030), (12, 30011)])
def test_what_rounding_took_off_of_rows_of_every_kind(rows, vocab, dtype):
    """None where there is no sum or a gradient takes it again: the gradient is the one without it there, and within its bounds elsewhere."""
    from oxidized_neural_orchestra_b200.ops.token_loss import token_logprobs, token_logprobs_grad

    torch.manual_seed(vocab)
    x, _ = _logits(rows, vocab, dtype, vocab + 3)
    x[1] = -math.inf
    x[2], x[3] = torch.finfo(dtype).min, torch.finfo(dtype).max
    x[4, 0], x[5, 1] = math.nan, math.inf
    x[6] *= 1e30
    x[7] += 500.0
    targets = torch.randint(0, vocab, (rows,), device="cuda")
    targets[0] = -1
    lse, low, ent, g, h = (torch.full((rows,), SENTINEL, device="cuda") for _ in range(5))
    g.normal_(), h.normal_()
    token_logprobs(x, targets, lse=lse, lse_low=low, entropy=ent)
    assert (low[[0, 1, 2, 3, 6]] == 0).all() and low[[4, 5]].isnan().logical_or(low[[4, 5]] == 0).all()
    ok = torch.isfinite(lse)
    assert (low[ok].abs() <= 2.0 ** -23 * lse[ok].abs().clamp_min(1.0)).all()
    a, b = torch.empty(rows, vocab, device="cuda"), torch.empty(rows, vocab, device="cuda")
    token_logprobs_grad(x, targets, lse=lse, entropy=ent, d_logp=g, d_entropy=h, out=a)
    token_logprobs_grad(x, targets, lse=lse, lse_low=low, entropy=ent, d_logp=g, d_entropy=h, out=b)
    assert torch.equal(a[:8].isnan(), b[:8].isnan())
    again = [0, 1, 2, 3, 6, 7]
    assert torch.equal(a[again], b[again])
    _, _, rlse, H, _, _ = _ref(x, targets, vocab)
    size = g.abs() + h.abs() * (2 * H.clamp_min(1.0) + 30).float()
    rest = slice(8, None)
    assert ((a - b).abs()[rest] <= (size * 2.0 ** -22 * rlse.float().abs().clamp_min(1.0))[rest].unsqueeze(1)).all()


@pytest.mark.parametrize("vocab,dtype", [(210011, F32), (420013, BF16)])
def test_loss_of_rows_too_long_to_be_kept(vocab, dtype):
    """Rows that do not fit into the shared memory of a cluster: their logits are read again, in place as well, wherever rows and outputs begin."""
    torch.manual_seed(vocab)
    for ld, lead in ((vocab // 16 * 16 + 16, 0), (vocab + 2, 3)):
        x, whole = _logits(6, vocab, dtype, ld, lead)
        _special("huge", x)
        x[3] = -math.inf
        x[4, ::2] = torch.finfo(dtype).min
        targets = torch.tensor([vocab - 1, 7, vocab // 2, 0, 4, -1], device="cuda")
        for out_dtype in (F32, BF16):
            _check_loss(x, whole, targets, out_dtype)
        _check_loss(x, whole, targets, dtype, in_place=True)
        x.copy_((torch.randn(6, vocab, device="cuda") * 3).to(dtype))
        for out_dtype in (F32, BF16):
            _check_loss(x, whole, targets, out_dtype)
        _check_loss(x, whole, targets, dtype, in_place=True)
