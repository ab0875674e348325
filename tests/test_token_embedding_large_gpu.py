"""The token table with the batches for which its kernels take their other forms:
four tokens a warp in the lookup, chunks of 32 sorted positions in the gradient,
tokens that cross many chunks.

Lookups: bit for bit, as in test_token_embedding_gpu.py.  Gradients: of whole
numbers from -8 to 8 times a power of two, so that every sum (310001 * 8 < 2^24)
and every product is exact in fp32 in any order, and a row that is lost, doubled
or added elsewhere shows however often its token occurs.  The result is the
int64 sum; in a bf16 table that sum rounded once."""
import numpy as np
import pytest
import torch

from gpu_helpers import assert_bits_equal, dev, host
from nntrain_b200.native import CudaBfp8Native, TokenEmbedding, scale_count
from test_token_embedding_gpu import some_tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,block,first", (("f32", 0, 0), ("bf16", 0, 0), ("bfp8", 32, 0), ("bfp8", 0, 0), ("bfp8", 96, 40),
                                              ("bfp8", 100, 3)))
@pytest.mark.parametrize("out_dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("count,width", ((9473, 256), (9474, 200), (9475, 33), (2371, 1000), (9476, 8), (3159, 771)))
def test_lookup_of_four_tokens_a_warp(cuda, kind, block, first, out_dtype, count, width):
    rng = np.random.default_rng(count + width)
    vocab = 515
    table = (rng.standard_normal((vocab, width)) * 0.02).astype(np.float32)
    tokens = some_tokens(rng, count, vocab, 0.2, "even")
    bad = rng.random(count) < 0.01
    tokens = np.where(bad, rng.choice([vocab, -2, 2 ** 40], count), tokens)
    scales = None
    if kind == "f32":
        values, d_table = table, dev(table)
    elif kind == "bf16":
        d_table = dev(table).to(torch.bfloat16)
        values = d_table.float().cpu().numpy()
    else:
        arena = np.concatenate([rng.standard_normal(first).astype(np.float32), table.ravel()])
        payload = torch.zeros(arena.size, dtype=torch.int8, device="cuda")
        scales = torch.zeros(scale_count(arena.size, block), device="cuda")
        CudaBfp8Native.block_encode(0, dev(arena), payload, scales, block)
        d_table = payload[first:].view(vocab, width)
        per_value = np.repeat(host(scales), block or arena.size)[:arena.size]
        values = (host(payload).astype(np.float32) * per_value)[first:].reshape(vocab, width)
    named = (tokens >= 0) & (tokens < vocab)
    scale = np.float32(1.7)
    want = np.where(named[:, None], values[np.where(named, tokens, 0)] * scale, np.float32(0)).astype(np.float32)
    want = torch.from_numpy(want).to(out_dtype).float().numpy()
    out = torch.full((count + 1, width), 9.0, dtype=out_dtype, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    TokenEmbedding.lookup(0, dev(tokens), d_table, out[:count], scale=float(scale), table_scales=scales, block_size=block,
                          first_value=first, token_status=status)
    torch.cuda.synchronize()
    assert_bits_equal(out[:count].float().cpu().numpy().ravel(), want.ravel(), "rows")
    assert int(status.item()) == 1 and (out[count] == 9.0).all()


def check_exactly(tokens, numbers, vocab, dout_dtype, table_dtype, tokens_dtype=torch.int64):
    """Written and added gradients of whole numbers against their int64 sums."""
    scale = 0.25
    sums = torch.zeros(vocab, numbers.shape[1], dtype=torch.int64, device="cuda")
    d_tokens = dev(tokens)
    named = d_tokens >= 0
    sums.index_add_(0, d_tokens[named], numbers[named].long())
    assert int(sums.abs().max()) < 1 << 24
    dout = numbers.to(dout_dtype)
    d_tokens = d_tokens.to(tokens_dtype)
    want = (sums.double() * scale).to(table_dtype)                       # exact in fp32, rounded once in bf16
    whole = torch.full((vocab, numbers.shape[1]), 9.0, dtype=table_dtype, device="cuda")
    TokenEmbedding.gradient(0, d_tokens, dout, whole, scale=scale)
    torch.cuda.synchronize()
    assert torch.equal(whole, want), rows_that_differ(whole, want)
    before = torch.arange(vocab, device="cuda").remainder(7).sub(3).to(table_dtype)[:, None].repeat(1, numbers.shape[1])
    added = before.clone()
    TokenEmbedding.gradient(0, d_tokens, dout, added, scale=scale, accumulate=True)
    torch.cuda.synchronize()
    want = (sums.double() * scale + before.double()).to(table_dtype)
    assert torch.equal(added, want), rows_that_differ(added, want)


def rows_that_differ(got, want):
    rows = (got != want).any(dim=1).nonzero().flatten().tolist()
    return f"{len(rows)} rows differ, the first of them {rows[:5]}"


def whole_numbers(count, width):
    g = torch.Generator(device="cuda").manual_seed(count + width)
    return torch.randint(-8, 9, (count, width), generator=g, device="cuda", dtype=torch.int8)


@pytest.mark.parametrize("law", ("text", "same", "ends", "even"))
@pytest.mark.parametrize("dout_dtype,table_dtype", ((torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                                    (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16)))
@pytest.mark.parametrize("count,vocab,width", (
    (310001, 900, 8), (310001, 900, 7), (160001, 5000, 264), (151553, 40, 300), (160001, 5001, 259),       # chunks of 32
    (70000, 300, 8), (4097, 100, 1000), (300001, 900, 4), (20000, 1250, 33), (2048, 2, 40), (540, 3, 771)))   # of 16
def test_sums_of_whole_numbers(cuda, law, dout_dtype, table_dtype, count, vocab, width):
    rng = np.random.default_rng(count + vocab)
    check_exactly(some_tokens(rng, count, vocab, 0.1, law), whole_numbers(count, width), vocab, dout_dtype, table_dtype)


@pytest.mark.parametrize("width", (8, 264))
@pytest.mark.parametrize("size", (16, 32))
def test_tokens_that_end_at_every_place_of_a_chunk(cuda, width, size):
    """Runs of one token after the other with lengths around one chunk, a few, the 16 from which a token is long, and
    the reach of the search for its last chunk; with a shift, so that they begin everywhere."""
    lengths = [1, 2, size - 1, size, size + 1, 2 * size, 3 * size - 1, 15 * size, 16 * size - 1, 16 * size, 16 * size + 1,
               17 * size, 17 * size + 1, 33 * size + 5, 34 * size, 65 * size - 1, 700 * size + 3]
    least = {(16, 8): 0, (16, 264): 0, (32, 8): 304_000, (32, 264): 152_000}[size, width]   # positions from which chunks are 32
    for shift in (0, 1, size // 2, size - 1):
        runs = [shift] + lengths * 2 if shift else lengths * 2
        rest = max(0, least - sum(runs))
        runs = runs + [37] * (-(-rest // 37))
        tokens = np.repeat(np.arange(len(runs)), runs)
        check_exactly(tokens, whole_numbers(len(tokens), width), len(runs) + 3, torch.float32, torch.float32, torch.int32)
