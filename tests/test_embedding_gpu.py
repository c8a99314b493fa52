"""Rows by token and the table's gradient against 64 bits: ids of every kind, runs of equal tokens at every edge of a chunk, odd sizes."""
import pytest
import torch

pytestmark = pytest.mark.gpu
SENTINEL = -7.0e11
F32, BF16 = torch.float32, torch.bfloat16


def _guarded(rows, cols, dtype, ld=None, lead=0):
    """[rows, cols] with `ld` values a row, `lead` values into an allocation full of sentinels."""
    ld = ld or cols
    whole = torch.full((lead + rows * ld + 64,), SENTINEL, device="cuda", dtype=dtype)
    return whole[lead:lead + rows * ld].view(rows, ld)[:, :cols], whole


def _untouched(view, whole):
    inside = torch.zeros_like(whole, dtype=torch.bool)
    off = view.storage_offset()
    for r in range(view.shape[0]):
        inside[off + r * view.stride(0):off + r * view.stride(0) + view.shape[1]] = True
    return bool((whole[~inside] == torch.tensor(SENTINEL, dtype=whole.dtype)).all())


@pytest.mark.parametrize("table_dtype", [F32, BF16])
@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("n,vocab,width,pad_ld,lead", [(1, 1, 1, 0, 0), (1, 50, 4096, 0, 0), (8, 320, 1024, 0, 0), (333, 1003, 517, 0, 1), (77, 11, 8, 8, 0),
                                                      (5, 9, 13, 3, 8), (1000, 130, 260, 4, 0), (64, 7, 1032, 24, 8), (9, 4, 5001, 0, 0)])
def test_lookup_is_exact(table_dtype, out_dtype, n, vocab, width, pad_ld, lead):
    from oxidized_neural_orchestra_b200.ops.embedding import embedding

    torch.manual_seed(n)
    table = torch.randn(lead + vocab * (width + pad_ld), device="cuda").to(table_dtype)[lead:].view(vocab, width + pad_ld)[:, :width]
    for ids_dtype, scale in ((torch.int32, 1.0), (torch.int64, 22.6)):
        ids = torch.randint(-1, vocab, (n,), device="cuda", dtype=ids_dtype)
        ids[0] = vocab - 1
        out, whole = _guarded(n, width, out_dtype, width + pad_ld, lead)
        status = torch.zeros(1, device="cuda", dtype=torch.int32)
        embedding(table, ids, out, scale=scale, status=status)
        ref = torch.where(ids.unsqueeze(1) >= 0, table[ids.long().clamp_min(0)].float() * scale, 0.0).to(out_dtype)
        assert torch.equal(out, ref) and _untouched(out, whole) and status.item() == 0


def test_lookup_of_ids_outside_the_table():
    from oxidized_neural_orchestra_b200.ops.embedding import embedding, embedding_grad

    table, d = torch.randn(10, 24, device="cuda"), torch.randn(6, 24, device="cuda")
    ids = torch.tensor([3, 10, -1, -5, 2**40, 9], device="cuda")
    for pad, bad in ((-1, True), (None, True)):
        status = torch.zeros(1, device="cuda", dtype=torch.int32)
        out = torch.full((6, 24), 5.0, device="cuda")
        embedding(table, ids, out, padding_id=pad, status=status)
        assert torch.equal(out[[0, 5]], table[[3, 9]]) and not out[1:5].any() and bool(status.item()) == bad
        grad, status = torch.full((10, 24), 3.0, device="cuda"), torch.zeros(1, device="cuda", dtype=torch.int32)
        embedding_grad(d, ids, grad, padding_id=pad, status=status)
        assert torch.equal(grad[[3, 9]], d[[0, 5]]) and grad.count_nonzero().item() == 48 and bool(status.item()) == bad
    # a token of the table may stand for padding; 32-bit ids do not see 2^32 + 3 as 3
    ids = torch.tensor([3, 4, 3], device="cuda", dtype=torch.int32)
    out, status = torch.ones(3, 24, device="cuda"), torch.zeros(1, device="cuda", dtype=torch.int32)
    embedding(table, ids, out, padding_id=3, status=status)
    assert torch.equal(out[1], table[4]) and not out[::2].any() and status.item() == 0
    grad = torch.full((10, 24), 3.0, device="cuda")
    embedding_grad(d[:3], ids, grad, padding_id=3, accumulate=True)
    assert torch.equal(grad[4], 3.0 + d[1]) and (grad[3] == 3.0).all()


def _check_grad(ids, vocab, width, d_dtype, *, accumulate=False, scale=1.0, pad_ld=0, lead=0):
    from oxidized_neural_orchestra_b200.ops.embedding import embedding_grad

    n = ids.numel()
    d = torch.randn(lead + n * (width + pad_ld), device="cuda").to(d_dtype)[lead:].view(n, width + pad_ld)[:, :width]
    grad, whole = _guarded(vocab, width, F32, width + pad_ld, lead)
    start = torch.randn(vocab, width, device="cuda") if accumulate else torch.zeros(vocab, width, device="cuda")
    if accumulate:
        grad.copy_(start)
    embedding_grad(d, ids, grad, scale=scale, accumulate=accumulate)
    known = (ids >= 0) & (ids < vocab)
    at, dd = ids[known].long(), d[known].double() * scale
    ref = start.double().index_add(0, at, dd)
    size = torch.zeros_like(ref).index_add(0, at, dd.abs())
    count = torch.bincount(at, minlength=vocab).double().unsqueeze(1)
    # f32 additions: each partial sum is off by half a step of at most the sum of the sizes; two more for the scale and the final addition
    tol = 2.0 ** -24 * ((count + 2) * size + ref.abs()) * 1.001
    assert ((grad.double() - ref).abs() <= tol).all()
    assert _untouched(grad, whole)
    again = start.clone()
    embedding_grad(d, ids, again, scale=scale, accumulate=accumulate)
    assert torch.equal(again, grad)


@pytest.mark.parametrize("d_dtype", [F32, BF16])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("n,vocab,width,pad_ld,lead", [(1, 1, 1, 0, 0), (1, 9, 40, 0, 0), (2, 2, 8, 0, 0), (63, 5, 12, 4, 0), (64, 3, 256, 0, 0), (65, 200, 257, 0, 1),
                                                      (128, 1, 24, 0, 0), (129, 1, 64, 0, 0), (333, 1003, 517, 0, 1), (1000, 511, 48, 16, 8), (1025, 512, 33, 0, 0),
                                                      (4096, 30, 96, 0, 0), (5000, 70000, 72, 0, 0), (20000, 300000, 16, 0, 0), (70001, 1300, 8, 0, 0)])
def test_gradient_of_random_tokens(d_dtype, accumulate, n, vocab, width, pad_ld, lead):
    torch.manual_seed(n + vocab)
    ids = torch.randint(-1, vocab, (n,), device="cuda", dtype=torch.int32 if n % 2 else torch.int64)
    _check_grad(ids, vocab, width, d_dtype, accumulate=accumulate, scale=1.0 if n % 3 else 0.37, pad_ld=pad_ld, lead=lead)


COUNTS = [[64, 64, 64], [63, 1, 64, 128], [1, 127, 65, 63], [200, 5, 300], [32, 96, 129, 127, 1, 1, 62], [64, 128, 192, 256], [1] * 63 + [66, 62, 130], [1000], [3, 1000, 3],
          [65, 64, 63, 128, 129, 500, 31, 33, 2], [2048, 4096, 7], [40] * 30, [255, 257, 1, 1, 510]]


@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: "-".join(map(str, c[:6])))
@pytest.mark.parametrize("width,d_dtype", [(40, BF16), (133, F32)])
def test_gradient_of_runs_at_the_edges_of_chunks(counts, width, d_dtype):
    torch.manual_seed(len(counts))
    ids = torch.repeat_interleave(torch.arange(len(counts), device="cuda") * 3, torch.tensor(counts, device="cuda"))
    for padded in (0, 37):      # (places without a token are sorted behind the others)
        mixed = torch.cat([ids, torch.full((padded,), -1, device="cuda")])[torch.randperm(ids.numel() + padded, device="cuda")]
        for accumulate in (False, True):
            _check_grad(mixed, 3 * len(counts), width, d_dtype, accumulate=accumulate)


@pytest.mark.parametrize("seed", range(12))
def test_gradient_of_drawn_runs(seed):
    g = torch.Generator().manual_seed(seed)
    kinds = torch.tensor([1, 1, 2, 30, 63, 64, 65, 127, 128, 129, 190, 400])
    counts = kinds[torch.randint(0, len(kinds), (40,), generator=g)].tolist()
    torch.manual_seed(seed)
    ids = torch.repeat_interleave(torch.arange(40), torch.tensor(counts))[torch.randperm(sum(counts), generator=g)].cuda()
    _check_grad(ids, 40, 24, BF16 if seed % 2 else F32, accumulate=seed % 3 == 0)


def test_gradient_without_tokens():
    from oxidized_neural_orchestra_b200.ops.embedding import embedding, embedding_grad

    for ids in (torch.zeros(0, device="cuda", dtype=torch.int64), torch.full((200,), -1, device="cuda")):
        n = ids.numel()
        grad = torch.ones(50, 20, device="cuda")
        embedding_grad(torch.randn(n, 20, device="cuda"), ids, grad, accumulate=True)
        assert (grad == 1.0).all()
        embedding_grad(torch.randn(n, 20, device="cuda"), ids, grad)
        assert not grad.any()
        out = torch.ones(n, 20, device="cuda")
        embedding(grad, ids, out)
        assert not out.any()


def test_far_rows_of_a_large_table():
    """Rows whose place in the table passes 2^32 bytes and 2^31 values."""
    from oxidized_neural_orchestra_b200.ops.embedding import embedding, embedding_grad

    vocab, width = 1_100_000, 2048
    table = torch.zeros(vocab, width, device="cuda", dtype=BF16)
    ids = torch.tensor([vocab - 1, 0, 1_050_001, vocab - 1], device="cuda")
    table[ids] = torch.randn(4, width, device="cuda").to(BF16)
    out = torch.empty(4, width, device="cuda", dtype=BF16)
    embedding(table, ids, out)
    assert torch.equal(out, table[ids])
    grad, d = torch.empty(vocab, width, device="cuda"), torch.randn(4, width, device="cuda")
    embedding_grad(d, ids, grad)
    assert torch.equal(grad[ids[1:3]], d[1:3]) and torch.equal(grad[vocab - 1], d[0] + d[3]) and grad.count_nonzero().item() == 3 * width


def test_on_two_streams_and_in_graphs():
    from oxidized_neural_orchestra_b200.ops.embedding import embedding, embedding_grad, embedding_grad_scratch

    torch.manual_seed(4)
    n, vocab, width = 3000, 700, 136
    sets = []
    for _ in range(2):
        ids = torch.randint(-1, vocab, (n,), device="cuda")
        sets.append((torch.randn(vocab, width, device="cuda"), ids, torch.randn(n, width, device="cuda"), torch.empty(n, width, device="cuda"),
                     torch.empty(vocab, width, device="cuda")))

    def call(s, **kw):
        embedding(s[0], s[1], s[3], scale=2.0, **kw)
        embedding_grad(s[2], s[1], s[4], **kw)

    wanted = []
    for s in sets:
        call(s)
        wanted.append((s[3].clone(), s[4].clone()))
    same = lambda: all(torch.equal(s[3], w[0]) and torch.equal(s[4], w[1]) for s, w in zip(sets, wanted))  # noqa: E731
    assert same()

    def clear():
        for s in sets:
            s[3].fill_(-1.0), s[4].fill_(-1.0)
        torch.cuda.synchronize()

    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        clear()
        for s, st in zip(sets, streams):
            call(s, stream=st)
        torch.cuda.synchronize()
        assert same()
    graphs = []
    for s in sets:      # each capture's scratch is its own: the two may run at once
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
    own = torch.empty(embedding_grad_scratch(n, vocab, width), device="cuda", dtype=torch.uint8)
    clear()
    embedding_grad(sets[0][2], sets[0][1], sets[0][4], scratch=own)
    assert torch.equal(sets[0][4], wanted[0][1])
    with pytest.raises(RuntimeError, match="scratch"):
        embedding_grad(sets[0][2], sets[0][1], sets[0][4], scratch=own[:-1])


@pytest.mark.parametrize("n,vocab", [(1, 100), (511, 22), (512, 21), (512, 22), (513, 600), (48, 2), (49, 2), (2048, 500), (2049, 500)])
@pytest.mark.parametrize("width,d_dtype,lead", [(40, BF16, 0), (33, BF16, 1), (133, F32, 3)])
def test_gradient_of_equal_tokens(n, vocab, width, d_dtype, lead):
    """All places of one token, or of two, on both sides of the sizes where another form begins."""
    torch.manual_seed(n)
    for ids in (torch.full((n,), vocab - 1, device="cuda"), torch.arange(n, device="cuda") % 2 * (vocab - 1)):
        for accumulate in (False, True):
            _check_grad(ids, vocab, width, d_dtype, accumulate=accumulate, lead=lead)
