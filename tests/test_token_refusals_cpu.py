"""What the operators on tokens and gradients refuse, before anything is launched."""
import math

import pytest
import torch


def _e():
    return torch.zeros(5, 8), torch.zeros(3, dtype=torch.int64), torch.zeros(3, 8)


def test_embedding():
    from oxidized_neural_orchestra_b200.ops.embedding import embedding, embedding_grad

    t, i, o = _e()
    with pytest.raises(RuntimeError, match="CUDA"):
        embedding(t, i, o)
    with pytest.raises(RuntimeError, match="CUDA"):
        embedding_grad(o, i, t)
    for call in (embedding, lambda a, b, c: embedding_grad(c, b, a)):
        with pytest.raises(TypeError):
            call(t, i.float(), o)
        with pytest.raises(TypeError):
            call(t, i.to(torch.int16), o)
        with pytest.raises(ValueError):
            call(t, i[:2], o)
        with pytest.raises(ValueError):
            call(t, torch.zeros(6, dtype=torch.int64)[::2], o)
        with pytest.raises(ValueError):
            call(t, i, o[:, :7])
        with pytest.raises(ValueError):
            call(t.t().contiguous().t(), i, o)
        with pytest.raises(ValueError):
            call(t, i, o[0].expand(3, 8))
        with pytest.raises(TypeError):
            call(t.double(), i, o)
        with pytest.raises(TypeError):
            call(t, i, o.half())
    with pytest.raises(TypeError):
        embedding_grad(o, i, t.bfloat16())
    with pytest.raises(ValueError):
        embedding_grad(o, i, t, scratch=torch.zeros(100, 2)[:, 0])


def test_tokens():
    from oxidized_neural_orchestra_b200.ops.token_loss import token_logprobs, token_logprobs_grad, token_loss

    x, t, v = torch.zeros(3, 9), torch.zeros(3, dtype=torch.int64), torch.zeros(3)
    with pytest.raises(RuntimeError, match="CUDA"):
        token_logprobs(x, t, logp=v)
    with pytest.raises(RuntimeError, match="CUDA"):
        token_loss(x, t, out=torch.zeros(3, 9))
    with pytest.raises(RuntimeError, match="CUDA"):
        token_logprobs_grad(x, t, lse=v, d_logp=v, out=x)
    for bad in (dict(logp=torch.zeros(4)), dict(logp=v.double()), dict(logp=torch.zeros(6)[::2]), dict(lse=torch.zeros(3, 1)), dict(entropy=v.bfloat16()),
                dict(top_logp=torch.zeros(3, 10), top_id=torch.zeros(3, 10, dtype=torch.int32)), dict(top_logp=torch.zeros(2, 2), top_id=torch.zeros(2, 2, dtype=torch.int32)),
                dict(top_logp=torch.zeros(3, 2), top_id=torch.zeros(3, 3, dtype=torch.int32))):
        with pytest.raises((ValueError, RuntimeError)):
            token_logprobs(x, t, **bad)
    with pytest.raises(ValueError):
        token_logprobs(torch.zeros(3, 90), t, top_logp=torch.zeros(3, 33), top_id=torch.zeros(3, 33, dtype=torch.int32))
    for bad in (dict(top_logp=torch.zeros(3, 2)), dict(top_id=torch.zeros(3, 2, dtype=torch.int32)), dict(top_logp=torch.zeros(3, 2), top_id=torch.zeros(3, 2, dtype=torch.int64))):
        with pytest.raises(TypeError):
            token_logprobs(x, t, **bad)
    for targets, err in ((t.float(), TypeError), (t[:2], ValueError), (t.unsqueeze(1), ValueError), (torch.zeros(6, dtype=torch.int64)[::2], ValueError)):
        with pytest.raises(err):
            token_logprobs(x, targets, lse=v)
    with pytest.raises(ValueError):
        token_logprobs(x, None, logp=v)
    with pytest.raises(ValueError):
        token_loss(x, None, out=x)
    for logits, err in ((x.half(), TypeError), (x.t(), ValueError), (x[0], ValueError), (x[0].expand(3, 9), ValueError)):
        with pytest.raises(err):
            token_logprobs(logits, t, lse=v)
    for out, err in ((torch.zeros(3, 8), ValueError), (torch.zeros(3, 9).half(), TypeError), (torch.zeros(9, 3).t(), ValueError), (x.view(torch.bfloat16)[:, :9], ValueError)):
        with pytest.raises(err):
            token_loss(x, t, out=out)
        with pytest.raises(err):
            token_logprobs_grad(x, t, lse=v, d_logp=v, out=out)
    with pytest.raises(ValueError):
        token_logprobs_grad(x, t, lse=v, out=x)
    with pytest.raises(ValueError):
        token_logprobs_grad(x, None, lse=v, d_logp=v, out=x)
    with pytest.raises(ValueError):
        token_logprobs_grad(x, t, lse=v, d_entropy=v, out=x)
    with pytest.raises(ValueError):
        token_logprobs_grad(x, t, lse=v, d_logp=v, entropy=v, out=x)
    with pytest.raises(TypeError, match="status"):
        from oxidized_neural_orchestra_b200.ops._launch import status_ptr
        status_ptr(v)


def test_clip():
    from oxidized_neural_orchestra_b200.ops.clip import clip_grads, grad_norm

    g, n = [torch.zeros(4), torch.zeros(2, 3)], torch.zeros(1)
    with pytest.raises(RuntimeError, match="CUDA"):
        grad_norm(g, n)
    with pytest.raises(RuntimeError, match="CUDA"):
        clip_grads(g, 1.0)
    for max_norm in (0.0, -1.0, math.nan):
        with pytest.raises(ValueError):
            clip_grads(g, max_norm)
    for scale in (math.nan, math.inf):
        with pytest.raises(ValueError):
            grad_norm(g, n, scale=scale)
    for bad, err in (([torch.zeros(4, 4).t()], ValueError), ([torch.zeros(8)[::2]], ValueError), ([torch.zeros(4).double()], TypeError), ([torch.zeros(4).int()], TypeError)):
        with pytest.raises(err):
            grad_norm(bad, n)
    with pytest.raises(TypeError):
        grad_norm(torch.zeros(4), n)
    for out in ([torch.zeros(4)], [torch.zeros(4), torch.zeros(3, 3)], [g[0].view(torch.bfloat16)[:4], torch.zeros(2, 3)]):
        with pytest.raises(ValueError):
            clip_grads(g, 1.0, out=out)
    with pytest.raises(ValueError, match="one place"):
        clip_grads([g[0], g[0]], 1.0)


def test_sizes_and_ids_that_32_and_64_bits_do_not_hold():
    """Rows whose indexes would pass 32 bits within a block's stride of their end, and ids that a 64-bit integer would take for another."""
    from oxidized_neural_orchestra_b200.ops import _lib
    from oxidized_neural_orchestra_b200.ops.embedding import embedding, embedding_grad, embedding_grad_scratch
    from oxidized_neural_orchestra_b200.ops.token_loss import token_logprobs, token_logprobs_grad, token_loss

    def of(rows, width, dtype=torch.bfloat16):
        return torch.empty(rows, width, dtype=dtype, device="meta")

    top, ids, v = 2**31 - 2**16, torch.empty(1, dtype=torch.int64, device="meta"), torch.empty(1, device="meta")
    for size in (top + 1, 2**31 - 100, 2**31):
        for call in (lambda: embedding(of(1, size), ids, of(1, size)), lambda: embedding(of(size, 4), ids, of(1, 4)),
                     lambda: embedding_grad(of(1, size), ids, of(1, size, torch.float32)), lambda: embedding_grad(of(1, 4), ids, of(size, 4, torch.float32)),
                     lambda: token_logprobs(of(1, size), ids, logp=v), lambda: token_loss(of(1, size), ids, out=of(1, size)),
                     lambda: token_logprobs_grad(of(1, size), ids, lse=v, d_logp=v, out=of(1, size))):
            with pytest.raises(ValueError, match=str(top)):
                call()
    with pytest.raises(RuntimeError, match="CUDA"):
        token_logprobs(of(1, top), ids, logp=v)
    assert embedding_grad_scratch(1000, top, 4) > 0
    for vocab, width in ((top + 1, 4), (4, top + 1), (2**32 + 4, 4)):
        with pytest.raises(ValueError, match=str(top)):
            embedding_grad_scratch(1000, vocab, width)
    lib = _lib.load()
    assert lib.ono_embedding_grad_scratch(1000, top + 1, 4) == -1 and lib.ono_embedding_grad_scratch(1000, 4, top + 1) == -1
    assert lib.ono_tokens(_lib.C.byref(_lib.OnoTokens(16, 16, 1, 2**31 - 100, 0, -1, 2**31 - 100)), None) != 0
    x, t, w = torch.zeros(3, 9), torch.zeros(3, dtype=torch.int64), torch.zeros(3)
    for wide in (2**63, 2**64 - 1, -(2**63), -(2**64)):
        for call in (lambda: embedding(x, t, x, padding_id=wide), lambda: embedding_grad(x, t, x, padding_id=wide), lambda: token_logprobs(x, t, lse=w, ignore_id=wide),
                     lambda: token_loss(x, t, out=x, ignore_id=wide), lambda: token_logprobs_grad(x, t, lse=w, d_logp=w, out=x, ignore_id=wide)):
            with pytest.raises(ValueError, match="no id"):
                call()


def test_launches_go_to_the_tensors_device(monkeypatch):
    """The device of the tensors is the current one during a launch, whichever was, and the stream is that device's, or the one that was given."""
    from contextlib import contextmanager
    from types import SimpleNamespace

    from oxidized_neural_orchestra_b200.ops import _launch

    now, calls = [0], []

    @contextmanager
    def device(d):
        was, now[0] = now[0], d
        yield
        now[0] = was

    lib = SimpleNamespace(op=lambda *args: calls.append((now[0], *args)) or 0, bad=lambda *args: 7, ono_last_error=lambda: b"why")
    monkeypatch.setattr(_launch._lib, "load", lambda: lib)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: now[0], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 100 + d, raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)
    for at in (0, 1):
        t = SimpleNamespace(get_device=lambda at=at: at)
        _launch.launch(t, None, "op", "x")
        _launch.launch(t, SimpleNamespace(cuda_stream=5), "op", "x", "y")
        assert calls[-2:] == [(at, "x", 100 + at), (at, "x", "y", 5)] and now == [0]
        with pytest.raises(RuntimeError, match="bad.*why"):
            _launch.launch(t, None, "bad", "x")
    cuda = [SimpleNamespace(is_cuda=True, device=f"cuda:{d}", get_device=lambda d=d: d) for d in (0, 1)]
    _launch.one_device(cuda[1], None, cuda[1])
    with pytest.raises(ValueError, match="different devices"):
        _launch.one_device(cuda[0], None, cuda[1])


def test_powers_that_the_gpu_cannot_read():
    from oxidized_neural_orchestra_b200.ops import elementwise as ew

    with pytest.raises(RuntimeError, match="CUDA"):
        ew.adam_tick(torch.ones(2), 0.9, 0.999)


def test_what_rounding_took_off_lse():
    from oxidized_neural_orchestra_b200.ops.token_loss import token_logprobs, token_logprobs_grad

    x, t, v = torch.zeros(3, 9), torch.zeros(3, dtype=torch.int64), torch.zeros(3)
    with pytest.raises(ValueError, match="lse_low needs lse"):
        token_logprobs(x, t, logp=v, lse_low=v)
    with pytest.raises(RuntimeError, match="CUDA"):
        token_logprobs(x, t, lse=v, lse_low=v)
    for bad in (torch.zeros(4), v.double(), torch.zeros(6)[::2], torch.zeros(3, 1)):
        with pytest.raises((ValueError, RuntimeError)):
            token_logprobs(x, t, lse=v, lse_low=bad)
        with pytest.raises((ValueError, RuntimeError)):
            token_logprobs_grad(x, t, lse=v, lse_low=bad, d_logp=v, out=x)


def test_a_cluster_is_taken_only_where_there_is_room_for_it():
    """A device, or a part of one, that has no room for a cluster of 16 clips in two launches."""
    from oxidized_neural_orchestra_b200.ops import _lib

    one = _lib.load().ono_clip_one_launch
    assert one(4, 101770, 1) == 1 and one(32, 131072, 9) == 1
    assert one(4, 101770, 0) == 0 and one(33, 1000, 1) == 0 and one(4, 131073, 1) == 0


def test_one_row_in_place_whatever_its_pitch():
    """A single row has no next one: a view of it that says otherwise is the same place."""
    from oxidized_neural_orchestra_b200.ops.token_loss import token_logprobs_grad, token_loss

    buf, t, v = torch.zeros(1, 16), torch.zeros(1, dtype=torch.int64), torch.zeros(1)
    x, out = buf[:, :9], buf[0, :9].unsqueeze(0).as_strided((1, 9), (9, 1))
    assert x.stride(0) != out.stride(0)
    with pytest.raises(RuntimeError, match="CUDA"):      # (nothing else is wrong with it)
        token_loss(x, t, out=out)
    with pytest.raises(RuntimeError, match="CUDA"):
        token_logprobs_grad(x, t, lse=v, d_logp=v, out=out)


def test_scratch_for_many_tokens_does_for_fewer():
    """One tensor, of what the most tokens want, serves all calls: wherever shorter chunks or other tiles begin, and everywhere between."""
    import random

    from oxidized_neural_orchestra_b200.ops.embedding import embedding_grad_scratch

    rng = random.Random(1)
    edges = {1, 511, 512, 513, 2048, 2049, 131072, 131073, 262144, 262145, 1000000}
    for width in (1, 24, 128, 129, 517, 1024, 2048, 4096, 16384, 130000):
        tiles = (width + 127) // 128
        for L, warps in ((16, 32), (32, 32), (64, 64), (128, 128), (256, 128), (512, 128)):
            least = -(-warps * 148 // tiles) * L
            edges |= {least - L, least - 1, least, least + 1, least + L}
    edges = sorted(edges | {int(2 ** rng.uniform(0, 27)) for _ in range(300)})
    for width in (1, 24, 128, 129, 517, 1024, 2048, 4096, 16384, 130000):
        for vocab in (5, 50257):
            wanted = [embedding_grad_scratch(n, vocab, width) for n in edges if n > 0]
            assert wanted == sorted(wanted), width
