"""What a model over tokens adds to this framework's training step, timed operator by operator.

``embed``: rows of a table looked up by token, scaled, and the table's gradient from the rows' (``dir`` "fwd", "bwd" or "both").
``logprobs``: log probabilities of given tokens with their entropy and the most likely alternatives; ``policy``: log probabilities and
entropy, then the logits' gradient from both of theirs; ``loss``: the token cross entropy with the logits' gradient in one call.
``clip``: the norm of all gradients of a network of dense layers, laid one behind the other in a flat vector as the engines lay them, and
the clipped gradients; ``step``: the norm, then an optimizer step on the flat vector that takes the clipping along.

``own`` False: elementary torch operations in 32 bits. True: the framework's kernels.
"""
import math

import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "i32": torch.int32, "i64": torch.int64}
PAD = -1
_ops = None


def _own():
    """The framework's modules, imported at the first call that is to use them."""
    global _ops
    if _ops is None:
        from oxidized_neural_orchestra_b200.ops import clip, elementwise, embedding, token_loss
        _ops = (embedding, token_loss, clip, elementwise)
    return _ops


def _embed(name, dir, n, vocab, width, table, out, ids, *, accumulate=False, padded=0.0, scale=1.0):
    return dict(name=name, op="embed", dir=dir, n=n, vocab=vocab, width=width, table=table, out=out, ids=ids, accumulate=accumulate,
                padded=padded, scale=scale)


def _tokens(name, op, rows, vocab, type, *, out="bf16", top=0, entropy=False, aligned=True, masked=False, padded=0.0, ids="i64"):
    return dict(name=name, op=op, rows=rows, vocab=vocab, type=type, out=out, top=top, entropy=entropy, aligned=aligned, masked=masked,
                padded=padded, ids=ids)


def listed():
    return [
        # the tokens of a few sequences at one step of decoding: latency
        _embed("embed_decode_8", "fwd", 8, 32000, 4096, "bf16", "bf16", "i64", scale=64.0),
        # a character model's padded batch: widths and counts that are no multiple of anything
        _embed("embed_ragged_333", "both", 333, 1003, 517, "f32", "f32", "i32", padded=0.1, scale=22.75),
        # a training batch of an ordinary model: lookup to bf16 rows, then the whole table's gradient
        _embed("embed_train_16k", "both", 16384, 50257, 1024, "f32", "bf16", "i64", padded=0.05, scale=32.0),
        # one of several large micro-batches: gradients added to those of the ones before (or to those of the head that shares the table)
        _embed("embed_grad_131k", "bwd", 131072, 128000, 2048, "f32", "bf16", "i64", accumulate=True),
        # four sequences at one step of decoding, with the twenty most likely tokens: latency
        _tokens("logprobs_decode_4", "logprobs", 4, 128256, "bf16", top=20, entropy=True),
        # scoring of given text in f32, rows that start anywhere, part of the vocabulary masked, some rows padding
        _tokens("logprobs_ragged_333", "logprobs", 333, 50257, "f32", top=5, entropy=True, aligned=False, masked=True, padded=0.1, ids="i32"),
        # a small vocabulary and many rows (characters, actions, classes): f32 logits of the last layer, bf16 deltas
        _tokens("loss_classes_16k", "loss", 16384, 1000, "f32", ids="i32"),
        # a training batch of an ordinary model: loss and gradient, some rows padding
        _tokens("loss_train_4k", "loss", 4096, 50257, "bf16", padded=0.05),
        # reinforcement learning on a large vocabulary: log probabilities and entropy, then the gradient from both
        _tokens("policy_4k_128k", "policy", 4096, 128256, "bf16", entropy=True),
        # the smallest network of the benchmark (784-128-10): latency
        dict(name="clip_mlp", op="clip", x=784, y=10, width=128, layers=1, grads="f32", out="f32", max_norm=1.0, scale=1.0),
        # a deep network with widths that leave every tensor of the flat vector at another alignment, clipped on the way to a 16-bit wire
        dict(name="clip_deep_1001", op="clip", x=517, y=333, width=1001, layers=96, grads="f32", out="bf16", max_norm=1.0, scale=0.125),
        # Adam on two layers of 8192 with their biases, with the bf16 shadow of the parameters
        dict(name="step_adam_134m", op="step", n=2 * 8193 * 8192, kind="adam", shadow=True, max_norm=1.0, scale=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "embed", "logprobs", "loss", "policy", "clip", "step"])
    if op == "embed":
        dir = rng.choice(["fwd", "bwd", "both"])
        n, vocab, width = _log(rng, 1, 131072), _log(rng, 100, 128256), _log(rng, 16, 4096)
        while n * width > 131072 * 2048:
            n //= 2
        while vocab * width > 128000 * 2048:
            vocab //= 2
        width = width // 64 * 64 if width > 200 and rng.random() < 0.5 else width
        return dict(op=op, dir=dir, n=n, vocab=vocab, width=width, table=rng.choice(["f32", "bf16"]), out=rng.choice(["f32", "bf16"]),
                    ids=rng.choice(["i32", "i64"]), accumulate=dir != "fwd" and rng.random() < 0.4, padded=rng.choice([0.0, 0.0, 0.1]),
                    scale=rng.choice([1.0, 0.125, 27.5]))
    if op in ("logprobs", "loss", "policy"):
        vocab, rows = _log(rng, 10, 128256), _log(rng, 1, 65536)
        while rows * vocab > (4096 * 128256 if op != "logprobs" else 1024 * 65536):
            rows = max(1, rows // 2)
        type = rng.choice(["f32", "bf16"])
        return dict(op=op, rows=rows, vocab=vocab, type=type, out=rng.choice([type, "bf16"]), entropy=op == "policy" or rng.random() < 0.5,
                    top=rng.choice([0, 1, 5, 20]) if op == "logprobs" else 0, aligned=rng.random() < 0.7, masked=rng.random() < 0.3,
                    padded=rng.choice([0.0, 0.1]), ids=rng.choice(["i32", "i64"]))
    if op == "clip":
        layers, width = _log(rng, 1, 96), _log(rng, 16, 2500)
        while layers * width * width > 100e6:
            layers = max(1, layers // 2)
        return dict(op=op, x=rng.choice([784, 517, 1024]), y=rng.choice([10, 333, 1000]), width=width, layers=layers,
                    grads=rng.choice(["f32", "bf16"]), out=rng.choice(["f32", "bf16"]), max_norm=rng.choice([0.5, 1.0, 1e9]),
                    scale=rng.choice([1.0, 0.25]))
    return dict(op=op, n=_log(rng, 1000, 130e6), kind=rng.choice(["sgd", "momentum", "adam"]), shadow=rng.random() < 0.5,
                max_norm=rng.choice([0.5, 1.0, 1e9]), scale=rng.choice([1.0, 0.25]))


# ------------------------------------------------------------------------------------------------------------------------------
def _token_ids(g, n, vocab, padded, dtype):
    """Tokens by Zipf's law (the k-th most frequent one in proportion to 1 / k), the frequent ones spread over the vocabulary."""
    rank = torch.exp(torch.rand(n, device="cuda", generator=g, dtype=torch.float64) * math.log(vocab)).long().clamp_(1, vocab) - 1
    ids = rank * 7919 % vocab
    if padded:
        ids[torch.rand(n, device="cuda", generator=g) < padded] = PAD
    return ids.to(dtype)


def _randn(g, *shape, dtype=torch.float32, std=1.0):
    t = torch.empty(*shape, device="cuda", dtype=dtype)
    return t.normal_(0.0, std, generator=g)


def _layer_sizes(c):
    feats = [c["x"]] + [c["width"]] * c["layers"] + [c["y"]]
    return [n for i, o in zip(feats, feats[1:]) for n in (i * o, o)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c, s = case, {"case": dict(case)}
    if c["op"] == "embed":
        n, v, w = c["n"], c["vocab"], c["width"]
        s["ids"] = _token_ids(g, n, v, c["padded"], DT[c["ids"]])
        if c["dir"] != "bwd":
            s["table"] = _randn(g, v, w, dtype=DT[c["table"]], std=0.02)
            s["out"] = torch.empty(n, w, device="cuda", dtype=DT[c["out"]])
        if c["dir"] != "fwd":
            s["d"] = _randn(g, n, w, dtype=DT[c["out"]], std=1e-3)
            s["grad"] = _randn(g, v, w, std=1e-3) if c["accumulate"] else torch.empty(v, w, device="cuda")
        return s
    if c["op"] in ("logprobs", "loss", "policy"):
        r, v = c["rows"], c["vocab"]
        ld = -(-v // 16) * 16 if c["aligned"] else v
        s["logits"] = _randn(g, r, ld, dtype=DT[c["type"]], std=2.5)[:, :v]
        s["targets"] = _token_ids(g, r, v, c["padded"], DT[c["ids"]])
        # a trained model: about half of the given tokens are the likely ones
        at = torch.arange(r, device="cuda")
        sure = (torch.rand(r, device="cuda", generator=g) < 0.5) * 10.0
        t = s["targets"].long().clamp_min(0)
        s["logits"][at, t] += sure.to(s["logits"].dtype)
        if c["masked"]:       # a third of the vocabulary is not allowed, except where it was said
            off = torch.rand(v, device="cuda", generator=g) < 0.33
            kept = s["logits"][at, t]
            s["logits"].masked_fill_(off, -math.inf)
            s["logits"][at, t] = kept
            if r >= 4:
                s["logits"][1].fill_(-math.inf)
        f = lambda *sh: torch.empty(*sh, device="cuda")  # noqa: E731
        s["logp"], s["lse"] = f(r), f(r)
        if c["entropy"]:
            s["entropy"] = f(r)
        if c["top"]:
            s["top"], s["top_logp"] = min(c["top"], v), f(r, min(c["top"], v))
            s["top_id"] = torch.empty(r, s["top"], device="cuda", dtype=torch.int32)
        if c["op"] != "logprobs":
            s["d"] = torch.empty(r, ld, device="cuda", dtype=DT[c["out"]])[:, :v]
            s["weight"] = torch.rand(r, device="cuda", generator=g) + 0.5
        if c["op"] == "policy":
            s["d_logp"] = _randn(g, r) / r
            s["d_entropy"] = torch.full((r,), -0.01 / r, device="cuda")
        return s
    if c["op"] == "clip":
        sizes = _layer_sizes(c)
        flat = _randn(g, sum(sizes), dtype=DT[c["grads"]], std=0.01)
        s["grads"] = list(flat.split(sizes))
        s["out"] = list(torch.empty(sum(sizes), device="cuda", dtype=DT[c["out"]]).split(sizes))
        s["norm"] = torch.empty(1, device="cuda")
        return s
    n = c["n"]
    s["p"], s["g"] = _randn(g, n, std=0.02), _randn(g, n, std=0.01)
    s["m"], s["v"] = _randn(g, n, std=1e-4), _randn(g, n, std=1e-4).square_()
    s["pows"] = torch.tensor([0.9 ** 5, 0.999 ** 5], device="cuda")
    s["p16"] = torch.empty(n, device="cuda", dtype=torch.bfloat16) if c["shadow"] else None
    s["norm"], s["coef"] = torch.empty(1, device="cuda"), torch.empty(1, device="cuda")
    return s


STEP = dict(lr=1e-3, mu=0.9, b1=0.9, b2=0.999, eps=1e-8)


def run(state):
    c = state["case"]
    return (_run_own if own else _run_plain)(c, state)


def _run_own(c, s):
    embedding, token_loss, clip, ew = _own()
    if c["op"] == "embed":
        if c["dir"] != "bwd":
            embedding.embedding(s["table"], s["ids"], s["out"], scale=c["scale"], padding_id=PAD)
        if c["dir"] != "fwd":
            embedding.embedding_grad(s["d"], s["ids"], s["grad"], scale=c["scale"], accumulate=c["accumulate"], padding_id=PAD)
        return {k: s[k] for k in ("out", "grad") if k in s}
    if c["op"] == "logprobs":
        token_loss.token_logprobs(s["logits"], s["targets"], logp=s["logp"], lse=s["lse"], entropy=s.get("entropy"),
                                  top_logp=s.get("top_logp"), top_id=s.get("top_id"), ignore_id=PAD)
        return {k: s[k] for k in ("logp", "lse", "entropy", "top_logp", "top_id") if k in s}
    if c["op"] == "policy":
        token_loss.token_logprobs(s["logits"], s["targets"], logp=s["logp"], lse=s["lse"], entropy=s["entropy"], ignore_id=PAD)
        token_loss.token_logprobs_grad(s["logits"], s["targets"], lse=s["lse"], entropy=s["entropy"], d_logp=s["d_logp"],
                                       d_entropy=s["d_entropy"], out=s["d"], ignore_id=PAD)
        return {k: s[k] for k in ("logp", "lse", "entropy", "d")}
    if c["op"] == "loss":
        token_loss.token_loss(s["logits"], s["targets"], out=s["d"], logp=s["logp"], weight=s["weight"], scale=1.0 / c["rows"], ignore_id=PAD)
        return {"logp": s["logp"], "d": s["d"]}
    if c["op"] == "clip":
        clip.clip_grads(s["grads"], c["max_norm"], scale=c["scale"], norm=s["norm"], out=s["out"])
        return {"norm": s["norm"], "out": s["out"][0]._base}
    clip.grad_norm([s["g"]], s["norm"], scale=c["scale"], max_norm=c["max_norm"], coef=s["coef"])
    if c["kind"] == "adam":
        ew.adam_tick(s["pows"], STEP["b1"], STEP["b2"])
    ew.optim_step(s["p"], s["g"], kind=c["kind"], m=s["m"], v=s["v"], adam_pows=s["pows"], p_bf16=s["p16"], grad_scale=c["scale"],
                  grad_coef=s["coef"], **STEP)
    return _step_outputs(c, s)


def _step_outputs(c, s):
    kept = ["norm", "p"] + (["m"] if c["kind"] != "sgd" else []) + (["v"] if c["kind"] == "adam" else []) + (["p16"] if c["shadow"] else [])
    return {k: s[k] for k in kept}


# ------------------------------------------------------------------------------------------------------------------------------
def _run_plain(c, s):
    if c["op"] == "embed":
        ids = s["ids"].long()
        known = ((ids >= 0) & (ids < c["vocab"])).unsqueeze(1)
        at = ids.clamp(0, c["vocab"] - 1)
        if c["dir"] != "bwd":
            s["out"].copy_(torch.where(known, s["table"][at].float() * c["scale"], 0.0))
        if c["dir"] != "fwd":
            if not c["accumulate"]:
                s["grad"].zero_()
            s["grad"].index_add_(0, at, torch.where(known, s["d"].float() * c["scale"], 0.0))
        return {k: s[k] for k in ("out", "grad") if k in s}
    if c["op"] == "clip":
        total = torch.stack([t.float().square().sum() for t in s["grads"]]).sum()
        s["norm"].copy_(total.sqrt() * c["scale"])
        f = torch.clamp(c["max_norm"] / s["norm"], max=1.0) * c["scale"]
        for o, t in zip(s["out"], s["grads"]):
            o.copy_(t.float() * f)
        return {"norm": s["norm"], "out": s["out"][0]._base}
    if c["op"] == "step":
        p, m, v, lr = s["p"], s["m"], s["v"], STEP["lr"]
        s["norm"].copy_(s["g"].square().sum().sqrt() * c["scale"])
        g = s["g"] * (torch.clamp(c["max_norm"] / s["norm"], max=1.0) * c["scale"])
        if c["kind"] == "sgd":
            p.sub_(lr * g)
        elif c["kind"] == "momentum":
            m.mul_(STEP["mu"]).add_(g)
            p.sub_(lr * m)
        else:
            s["pows"][0].mul_(STEP["b1"])
            s["pows"][1].mul_(STEP["b2"])
            step = lr * torch.sqrt(1.0 - s["pows"][1]) / (1.0 - s["pows"][0])
            m.mul_(STEP["b1"]).add_((1.0 - STEP["b1"]) * g)
            v.mul_(STEP["b2"]).add_((1.0 - STEP["b2"]) * g * g)
            p.sub_(step * m / (v.sqrt() + STEP["eps"]))
        if c["shadow"]:
            s["p16"].copy_(p)
        return _step_outputs(c, s)
    # the operators on logits: one softmax in 32 bits, from which everything else follows
    t = s["targets"].long()
    known = (t >= 0) & (t < c["vocab"])
    at = t.clamp(0, c["vocab"] - 1).unsqueeze(1)
    x = s["logits"].float()
    top = x.amax(1, keepdim=True)
    some = top > -math.inf              # a row of which the mask leaves something
    top = torch.where(some, top, 0.0)
    e = torch.exp(x - top)
    z = e.sum(1, keepdim=True)
    log_z = torch.log(torch.where(some, z, 1.0))
    of = lambda col, empty: torch.where(known, torch.where(some.squeeze(1), col.squeeze(1), empty), 0.0)  # noqa: E731
    s["lse"].copy_(of(top + log_z, -math.inf))
    s["logp"].copy_(of(x.gather(1, at) - top - log_z, -math.inf))
    if c["entropy"]:
        h = log_z - torch.where(e > 0, e * (x - top), 0.0).sum(1, keepdim=True) / torch.where(some, z, 1.0)
        s["entropy"].copy_(of(h, 0.0))
    if c["op"] == "logprobs":
        if c["top"]:
            val, place = torch.sort(x, dim=1, descending=True, stable=True)     # ties: the lowest index first
            val, place = val[:, :s["top"]], place[:, :s["top"]]
            there = known.unsqueeze(1) & (val > -math.inf)
            s["top_logp"].copy_(torch.where(there, val - top - log_z, -math.inf))
            s["top_id"].copy_(torch.where(there, place, -1))
        return {k: s[k] for k in ("logp", "lse", "entropy", "top_logp", "top_id") if k in s}
    p = e / torch.where(some, z, 1.0)
    live = known.unsqueeze(1) & some
    if c["op"] == "loss":
        d = p.scatter_add(1, at, torch.full_like(z, -1.0))
        d *= s["weight"].unsqueeze(1) / c["rows"]
        s["d"].copy_(torch.where(live, d, 0.0))
        return {"logp": s["logp"], "d": s["d"]}
    g, ge = s["d_logp"].unsqueeze(1), s["d_entropy"].unsqueeze(1)
    d = -p * (g + ge * (torch.where(p > 0, x - top - log_z, 0.0) + h))
    s["d"].copy_(torch.where(live, d.scatter_add(1, at, g), 0.0))
    return {k: s[k] for k in ("logp", "lse", "entropy", "d")}


# ------------------------------------------------------------------------------------------------------------------------------
def work(case):
    c = case
    size = lambda k: DT[c[k]].itemsize  # noqa: E731
    if c["op"] == "embed":
        n, v, w = c["n"], c["vocab"], c["width"]
        met = v * (1.0 - math.exp(-n / (v * max(1.0, math.log(v)))))       # rows met at least, by Zipf's law
        b = n * size("ids")
        if c["dir"] != "bwd":
            b += met * w * size("table") + n * w * size("out")
        if c["dir"] != "fwd":
            b += n * w * size("out") + (2 * met if c["accumulate"] else v) * w * 4
        return {"bytes": b, "flops": 2.0 * n * w}
    if c["op"] in ("logprobs", "loss", "policy"):
        cells = c["rows"] * c["vocab"]
        b = cells * (size("type") + (size("out") if c["op"] != "logprobs" else 0)) + c["rows"] * (12 + 8 * c["top"])
        return {"bytes": b, "flops": cells * {"logprobs": 5.0, "loss": 8.0, "policy": 12.0}[c["op"]]}
    if c["op"] == "clip":
        n = sum(_layer_sizes(c))
        return {"bytes": n * (size("grads") + size("out")), "flops": 3.0 * n}
    per = {"sgd": 12, "momentum": 20, "adam": 28}[c["kind"]] + (2 if c["shadow"] else 0)
    return {"bytes": float(per) * c["n"], "flops": 12.0 * c["n"]}


def exact(case, seed):
    """The definitions in 64 bits."""
    c, s = case, prepare(case, seed)
    if c["op"] == "embed":
        ids, got = s["ids"].long(), {}
        if c["dir"] != "bwd":
            rows = torch.zeros(c["n"], c["width"], device="cuda", dtype=torch.float64)
            rows[ids >= 0] = s["table"].index_select(0, ids[ids >= 0]).double() * c["scale"]
            got["out"] = rows
        if c["dir"] != "fwd":
            # sums over the runs of the sorted tokens, as differences of running sums
            grad = s["grad"].double() if c["accumulate"] else torch.zeros(c["vocab"], c["width"], device="cuda", dtype=torch.float64)
            key, order = torch.sort(ids)
            order, key = order[key >= 0], key[key >= 0]
            if key.numel():
                token, count = torch.unique_consecutive(key, return_counts=True)
                running = torch.cumsum(s["d"].double()[order], 0)[torch.cumsum(count, 0) - 1]
                running[1:] -= running[:-1].clone()
                grad[token] += running * c["scale"]
            got["grad"] = grad
        return got
    if c["op"] == "clip":
        flat = torch.cat([t.double() for t in s["grads"]])
        norm = torch.linalg.vector_norm(flat) * c["scale"]
        return {"norm": norm.reshape(1), "out": flat.mul_(c["scale"] * min(1.0, c["max_norm"] / float(norm)))}
    if c["op"] == "step":
        g, p, m, v = (s[k].double() for k in ("g", "p", "m", "v"))
        norm = torch.linalg.vector_norm(g) * c["scale"]
        g *= c["scale"] * min(1.0, c["max_norm"] / float(norm))
        if c["kind"] == "sgd":
            p -= STEP["lr"] * g
        elif c["kind"] == "momentum":
            m = STEP["mu"] * m + g
            p -= STEP["lr"] * m
        else:
            b1, b2 = STEP["b1"], STEP["b2"]
            b1t, b2t = float(s["pows"][0]) * b1, float(s["pows"][1]) * b2
            m = b1 * m + (1 - b1) * g
            v = b2 * v + (1 - b2) * g ** 2
            p -= STEP["lr"] * math.sqrt(1 - b2t) / (1 - b1t) * m / (torch.sqrt(v) + STEP["eps"])
        return _step_outputs(c, {"norm": norm.reshape(1), "p": p, "m": m, "v": v, "p16": p})
    if c["rows"] * c["vocab"] * 8 * 6 > 100e9:
        return None
    t, live = s["targets"].long(), s["targets"] >= 0
    lp = torch.log_softmax(s["logits"].double(), 1)
    empty = torch.isinf(s["logits"]).all(1)
    lp[empty] = -math.inf
    mine = lp.gather(1, t.clamp_min(0).unsqueeze(1)).squeeze(1)
    h = -torch.nansum(torch.exp(lp) * lp, 1)
    got = {"logp": torch.where(live, mine, 0.0), "lse": torch.where(live, torch.logsumexp(s["logits"].double(), 1), 0.0)}
    if c["entropy"]:
        got["entropy"] = torch.where(live, h, 0.0)
    if c["op"] == "logprobs":
        if c["top"]:
            got["top_logp"] = torch.where(live.unsqueeze(1), torch.topk(lp, s["top"], 1).values, -math.inf)
            got["top_id"] = None
        return got
    p = torch.exp(lp)
    one = torch.zeros_like(p)
    one.scatter_(1, t.clamp_min(0).unsqueeze(1), 1.0)
    dead = ~live | empty
    if c["op"] == "loss":
        d = (p - one) * (s["weight"].double() / c["rows"]).unsqueeze(1)
        d[dead] = 0.0
        return {"logp": got["logp"], "d": d}
    d = (one - p) * s["d_logp"].double().unsqueeze(1)
    d -= torch.nan_to_num(p * (lp + h.unsqueeze(1)), nan=0.0) * s["d_entropy"].double().unsqueeze(1)
    d[dead] = 0.0
    return {**got, "d": d}
