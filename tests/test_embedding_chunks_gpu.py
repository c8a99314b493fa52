"""The table's gradient where a warp has more than a few places: chunks of every length that sizes lead to, runs of equal tokens at their edges, and so many places
that a CTA of the sort goes through its own in several batches."""
import pytest
import torch

from test_embedding_gpu import BF16, F32, _check_grad

pytestmark = pytest.mark.gpu


def _chunk(n, width):
    """Places that a warp adds up, by the rule in embedding.cu."""
    tiles, L = (width + 127) // 128, 512
    while L > 8 and n // L * tiles < (128 if L > 64 else 64 if L > 32 else 32) * 148:
        L //= 2
    return L


def _runs(L, least):
    """Runs that end one place ahead of a chunk's end, at it and behind it, fill none, one or several chunks, and are cut by a batch of 32; `least` places or more."""
    once = [L - 1, 1, L, L + 1, 2 * L - 1, 1, 2 * L, 2 * L + 1, 31, 33, 3 * L, 2, 5 * L + 3, 32, L // 2, L // 2, 1, 1]
    return once * -(-least // sum(once))


def _width(n, L, odd):
    """The least width, of whole tiles but for `odd`, that n places take chunks of L with."""
    tiles = next(t for t in range(1, 20000) if _chunk(n, 128 * t) >= L)
    assert _chunk(n, 128 * tiles - odd) == L
    return 128 * tiles - odd


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("d_dtype,odd,lead", [(BF16, 0, 0), (F32, 8, 0), (BF16, 3, 1), (F32, 125, 3)])
@pytest.mark.parametrize("L,least", [(16, 600), (16, 2100), (32, 600), (32, 5000), (64, 2100), (64, 9000), (128, 2100)])
def test_runs_at_the_edges_of_longer_chunks(L, least, d_dtype, odd, lead, accumulate):
    counts = _runs(L, least)
    torch.manual_seed(L + least)
    ids = torch.repeat_interleave(torch.arange(len(counts), device="cuda") * 2, torch.tensor(counts, device="cuda"))
    for padded in (0, 37):      # (places without a token are sorted behind the others)
        mixed = torch.cat([ids, torch.full((padded,), -1, device="cuda")])[torch.randperm(ids.numel() + padded, device="cuda")]
        width = _width(mixed.numel(), L, odd)
        _check_grad(mixed, 2 * len(counts), width, d_dtype, accumulate=accumulate, lead=lead)
        _check_grad(torch.randint(0, 2 * len(counts), mixed.shape, device="cuda", dtype=torch.int32), 2 * len(counts), width, d_dtype, accumulate=accumulate, scale=0.37, lead=lead)


@pytest.mark.parametrize("L,d_dtype", [(256, BF16), (512, BF16), (256, F32)])
def test_runs_at_the_edges_of_the_longest_chunks(L, d_dtype):
    counts = _runs(L, 2100)
    torch.manual_seed(L)
    ids = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), torch.tensor(counts, device="cuda"))
    ids = ids[torch.randperm(ids.numel(), device="cuda")]
    _check_grad(ids, len(counts), _width(ids.numel(), L, 0), d_dtype, accumulate=d_dtype == F32)


@pytest.mark.parametrize("vocab,n", [(v, n) for v in (300, 511, 512) for n in (131072, 131073, 131072 + 1500, 262144, 262145, 400003)] +
                         [(70000, 131073), (70000, 262144), (70000, 400003), (270000, 132572), (270000, 400003)])
def test_more_places_than_a_batch_to_each_warp_of_the_sort(vocab, n):
    """One to three passes; a CTA of the sort has one, two or four batches of the places, the last of them fewer."""
    torch.manual_seed(n % 1000 + vocab)
    for ids in (torch.randint(-1, vocab, (n,), device="cuda"), (torch.rand(n, device="cuda").pow(6) * vocab).to(torch.int32)):
        _check_grad(ids, vocab, 24, BF16 if n % 2 else F32, accumulate=vocab == 512)
