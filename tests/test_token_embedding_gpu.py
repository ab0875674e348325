"""The token table's lookup and gradient against numpy in 64 bits.

Tolerances, with e = 2^-24.  Lookup: the decode's product and the scale's, then
the output's rounding: bit for bit against the same products in numpy.
Gradient: a row's n terms are added in fp32, up to 32 positions, then the chunks'
partials, an eighth of them a warp: no term passes more than 32 + chunks + 8
additions, each off by e of at most the sum of the absolute terms; the scale
and the sum with what is there add 2 e, the output's rounding its half step."""
import numpy as np
import pytest
import torch

from gpu_helpers import assert_bits_equal, dev, host, misaligned
from nntrain_b200.native import CudaBfp8Native, TokenEmbedding, scale_count

pytestmark = pytest.mark.gpu

E = 2.0 ** -24


def to_f64(t):
    return t.detach().double().cpu().numpy()


def some_tokens(rng, count, vocab, padded=0.2, law="text"):
    if law == "text":
        t = np.floor(np.exp(rng.random(count) * np.log(vocab + 1.0)) - 1.0).astype(np.int64).clip(0, vocab - 1)
    elif law == "same":
        t = np.full(count, vocab // 2, dtype=np.int64)
    elif law == "ends":
        t = np.where(rng.random(count) < 0.5, 0, vocab - 1)
    else:
        t = rng.integers(0, vocab, count)
    return np.where(rng.random(count) < padded, -1, t)


# ---- lookup -------------------------------------------------------------------

@pytest.mark.parametrize("kind", ("f32", "bf16", "bfp8"))
@pytest.mark.parametrize("out_dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("count,vocab,width,block,first", (
    (1, 1, 1, 32, 0), (7, 50, 33, 32, 0), (64, 300, 512, 32, 0), (33, 300, 520, 0, 0), (5, 40, 1536, 128, 640), (9, 40, 96, 96, 5),
    (9, 40, 64, 32, 8), (300, 1000, 771, 771, 0), (3, 20, 5000, 64, 64)))
def test_lookup(cuda, kind, out_dtype, count, vocab, width, block, first):
    rng = np.random.default_rng(count + width)
    table = (rng.standard_normal((vocab, width)) * 0.02).astype(np.float32)
    tokens = some_tokens(rng, count, vocab)
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
        decoded = torch.zeros(arena.size, device="cuda")
        CudaBfp8Native.block_decode(0, payload, scales, decoded, block)
        values = host(decoded)[first:].reshape(vocab, width)
    scale = np.float32(np.sqrt(width))
    want = np.where((tokens >= 0)[:, None], values[tokens.clip(0)] * scale, np.float32(0)).astype(np.float32)
    want = torch.from_numpy(want).to(out_dtype).float().numpy()
    for dtype in (torch.int64, torch.int32):
        out = torch.full((count, width), 9.0, dtype=out_dtype, device="cuda")
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        TokenEmbedding.lookup(0, dev(tokens).to(dtype), d_table, out, scale=float(scale), table_scales=scales,
                              block_size=block if kind == "bfp8" else 0, first_value=first if kind == "bfp8" else 0,
                              token_status=status)
        torch.cuda.synchronize()
        assert_bits_equal(out.float().cpu().numpy().ravel(), want.ravel(), "rows")
        assert int(status.item()) == 0


@pytest.mark.parametrize("shift,extra", ((0, 8), (1, 3), (3, 0)))
def test_lookup_at_any_place_and_stride(cuda, shift, extra):
    rng = np.random.default_rng(1)
    vocab, width, count = 30, 64, 11
    base = dev(rng.standard_normal(vocab * width + 16).astype(np.float32))
    table = base[shift:shift + vocab * width].view(vocab, width)
    tokens = some_tokens(rng, count, vocab)
    rows = torch.full((count * (width + extra) + 8,), 7.0, device="cuda")
    out = rows[shift:shift + count * (width + extra)].view(count, width + extra)[:, :width]
    TokenEmbedding.lookup(0, dev(tokens), table, out, scale=0.5)
    torch.cuda.synchronize()
    want = np.where((tokens >= 0)[:, None], host(table)[tokens.clip(0)] * np.float32(0.5), 0).astype(np.float32)
    assert (host(out) == want).all()
    gaps = rows[shift:shift + count * (width + extra)].view(count, width + extra)[:, width:]
    assert (gaps == 7.0).all() and (rows[:shift] == 7.0).all() and (rows[shift + count * (width + extra):] == 7.0).all()


def test_tokens_outside_the_table_are_none_and_raise_the_status(cuda):
    table = torch.ones(10, 16, device="cuda")
    for bad in (-2, 10, 2 ** 40, -2 ** 62):
        status, out = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.full((3, 16), 9.0, device="cuda")
        TokenEmbedding.lookup(0, torch.tensor([3, bad, 0], device="cuda"), table, out, token_status=status)
        assert int(status.item()) == 1 and out[:, 0].tolist() == [1.0, 0.0, 1.0]
        gradient = torch.zeros(10, 16, device="cuda")
        status.zero_()
        TokenEmbedding.gradient(0, torch.tensor([3, bad, 0], device="cuda"), out + 1.0, gradient, token_status=status)
        assert int(status.item()) == 1 and gradient[:, 0].tolist() == [2.0, 0, 0, 2.0] + [0] * 6
    status.zero_()
    out = torch.full((2, 16), 9.0, device="cuda")
    TokenEmbedding.lookup(0, torch.tensor([3, 0], device="cuda"), table, out, padding_token=3, token_status=status)
    assert int(status.item()) == 0 and out[:, 0].tolist() == [0.0, 1.0]
    gradient = torch.full((10, 16), 5.0, device="cuda")
    TokenEmbedding.gradient(0, torch.tensor([3, 0], device="cuda"), out, gradient, padding_token=3, token_status=status)
    assert int(status.item()) == 0 and gradient[:, 0].tolist() == [1.0] + [0] * 9


def test_values_that_are_not_finite_stay_in_their_rows(cuda):
    table = torch.ones(4, 64, device="cuda")
    table[1] = float("nan")
    table[2] = float("inf")
    out = torch.zeros(4, 64, device="cuda")
    TokenEmbedding.lookup(0, torch.tensor([0, 1, 2, -1], device="cuda"), table, out, scale=2.0)
    assert (out[0] == 2.0).all() and out[1].isnan().all() and out[2].isinf().all() and not out[3].any()
    # a padded position's gradient is not read into any row
    dout = torch.ones(40, 64, device="cuda")
    dout[5] = float("nan")
    tokens = torch.arange(40, device="cuda") % 3
    tokens[5] = -1
    gradient = torch.zeros(4, 64, device="cuda")
    TokenEmbedding.gradient(0, tokens, dout, gradient)
    assert gradient.isfinite().all()


# ---- gradient -----------------------------------------------------------------

def check_gradient(tokens, dout, got, scale, vocab, before=None):
    d = to_f64(dout)
    width = d.shape[1]
    want, size = np.zeros((vocab, width)), np.zeros((vocab, width))
    valid = tokens >= 0
    np.add.at(want, tokens[valid], d[valid])
    np.add.at(size, tokens[valid], np.abs(d[valid]))
    counts = np.bincount(tokens[valid], minlength=vocab)
    want, size = want * scale, size * abs(scale)
    bound = (32 + counts / 16 + 8 + 3)[:, None] * E * size
    if before is not None:
        want = want + to_f64(before)
        bound = bound + E * (np.abs(want) + size) * (counts > 0)[:, None]
    if got.dtype == torch.bfloat16:
        bound = bound + np.abs(want) * 2.0 ** -8 * 1.01
    assert (np.abs(to_f64(got) - want) <= bound).all()


@pytest.mark.parametrize("count,vocab,width", (
    (1, 1, 1), (1, 300, 64), (31, 40, 33), (32, 40, 256), (33, 5, 264), (64, 7, 771), (1000, 513, 512), (5000, 70000, 40),
    (4097, 1000, 1000), (70000, 300, 8)))
@pytest.mark.parametrize("law", ("text", "same", "ends", "even"))
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
def test_gradient(cuda, count, vocab, width, law, dtype):
    rng = np.random.default_rng(count + vocab)
    tokens = some_tokens(rng, count, vocab, 0.1, law)
    dout = dev((rng.standard_normal((count, width)) * 1e-3).astype(np.float32)).to(dtype)
    d_tokens = dev(tokens)
    for table_dtype in (torch.float32, torch.bfloat16):
        got = torch.full((vocab, width), 9.0, dtype=table_dtype, device="cuda")
        TokenEmbedding.gradient(0, d_tokens, dout, got, scale=1.5)
        torch.cuda.synchronize()
        check_gradient(tokens, dout, got, 1.5, vocab)
        before = dev(rng.standard_normal((vocab, width)).astype(np.float32) * 1e-3).to(table_dtype)
        added = before.clone()
        TokenEmbedding.gradient(0, d_tokens.to(torch.int32), dout, added, scale=1.5, accumulate=True)
        torch.cuda.synchronize()
        check_gradient(tokens, dout, added, 1.5, vocab, before)
        unnamed = torch.ones(vocab, dtype=torch.bool)
        unnamed[torch.from_numpy(tokens[tokens >= 0])] = False
        assert not got.cpu()[unnamed].any() and torch.equal(added.cpu()[unnamed], before.cpu()[unnamed])


@pytest.mark.parametrize("vocab", (2, 511, 512, 513, 262143, 262144, 300000))
def test_every_number_of_passes_sorts(cuda, vocab):
    """The order shows in the bits: equal tokens are added as they occur."""
    rng = np.random.default_rng(vocab)
    count, width = 3000, 4
    tokens = some_tokens(rng, count, vocab, 0.05, "even")
    tokens[:3] = [vocab - 1, 0, vocab - 1]
    dout = (10.0 ** rng.uniform(-6, 6, (count, width))).astype(np.float32)
    got = torch.zeros(vocab, width, device="cuda")
    TokenEmbedding.gradient(0, dev(tokens), dev(dout), got)
    torch.cuda.synchronize()
    want = np.zeros((vocab, width), np.float32)
    if vocab > 1000:                                     # few repeats: chunks cut no long run, plain order
        order = np.argsort(tokens[tokens >= 0], kind="stable")
        t, d = tokens[tokens >= 0][order], dout[tokens >= 0][order]
        partial, at = np.zeros(width, np.float32), 0
        for i in range(len(t)):
            partial = (partial + d[i]).astype(np.float32)
            ends = i + 1 == len(t) or t[i + 1] != t[i]
            if ends or (i + 1) % 16 == 0:                # a chunk's border splits the sum
                want[t[i]] = partial if at == 0 else (want[t[i]] + partial).astype(np.float32)
                at = 0 if ends else 1
                partial = np.zeros(width, np.float32)
        assert_bits_equal(host(got).ravel(), want.ravel(), "rows")
    else:
        check_gradient(tokens, dev(dout), got, 1.0, vocab)


@pytest.mark.parametrize("vocab", (3, 1000, (1 << 21) - 1, 1 << 21, (1 << 21) + 7))
@pytest.mark.parametrize("count", (1, 2, 63, 64, 65, 500, 1024, 1025, 2047, 2048, 2049))
def test_small_sorts(cuda, vocab, count):
    """One CTA's sort at its borders, with 32- and 64-bit keys."""
    rng = np.random.default_rng(count)
    tokens = some_tokens(rng, count, vocab, 0.1, "even" if vocab > 1000 else "text")
    dout = dev(rng.standard_normal((count, 4)).astype(np.float32))
    before = torch.ones(vocab, 4, device="cuda")
    got = before.clone()
    TokenEmbedding.gradient(0, dev(tokens), dout, got, accumulate=True)
    whole = torch.full((vocab, 4), 9.0, device="cuda")
    TokenEmbedding.gradient(0, dev(tokens), dout, whole)
    torch.cuda.synchronize()
    check_gradient(tokens, dout, got, 1.0, vocab, before)
    check_gradient(tokens, dout, whole, 1.0, vocab)


@pytest.mark.parametrize("law", ("even", "text"))
@pytest.mark.parametrize("count", (8192, 8193, 32768, 32769, 65536, 65537, 131072, 131073, 300001))
def test_sorts_of_several_ctas(cuda, count, law):
    """The cluster's sizes, and stretches that fill a warp's registers, pass them and pass them twice."""
    rng = np.random.default_rng(count)
    vocab = 900
    tokens = some_tokens(rng, count, vocab, 0.03, law)
    dout = dev(rng.standard_normal((count, 4)).astype(np.float32))
    before = torch.ones(vocab, 4, device="cuda")
    added, whole = before.clone(), torch.full((vocab, 4), 9.0, device="cuda")
    TokenEmbedding.gradient(0, dev(tokens), dout, added, accumulate=True)
    TokenEmbedding.gradient(0, dev(tokens), dout, whole)
    torch.cuda.synchronize()
    check_gradient(tokens, dout, added, 1.0, vocab, before)
    check_gradient(tokens, dout, whole, 1.0, vocab)


@pytest.mark.parametrize("count,vocab,width", ((3000, 70000, 1024), (8192, 64000, 1024), (30000, 100_000, 1024),
                                               (140_000, 340_000, 1024)))
def test_zeros_beside_the_sort(cuda, count, vocab, width):
    """The sums do not depend on how the sort and the zeros share the machine: the bits of a gradient added to zeros."""
    generator = torch.Generator(device="cuda").manual_seed(count)
    tokens = torch.randint(-1, vocab, (count,), generator=generator, device="cuda")
    tokens[::7] = tokens[0]                              # one that crosses every chunk of its own
    dout = torch.randn(count, width, generator=generator, device="cuda", dtype=torch.bfloat16)
    whole, added = torch.full((vocab, width), 9.0, device="cuda"), torch.zeros(vocab, width, device="cuda")
    TokenEmbedding.gradient(0, tokens, dout, whole)
    TokenEmbedding.gradient(0, tokens, dout, added, accumulate=True)
    torch.cuda.synchronize()
    assert torch.equal(whole, added)
    assert not whole[~torch.zeros(vocab, dtype=torch.bool, device="cuda").index_fill_(0, tokens[tokens >= 0], True)].any()


@pytest.mark.parametrize("vocab,width", ((70000, 4), (300_000, 4), (1 << 28, 1)))
def test_one_bucket_takes_all(cuda, vocab, width):
    """Rows that agree in their low 9 bits: one, two and three passes over the others."""
    rng = np.random.default_rng(vocab)
    count = 5000
    rows = np.unique(np.concatenate([rng.integers(0, vocab // 512, 40), [0, vocab // 512 - 1]])) * 512
    tokens = rows[rng.integers(0, len(rows), count)]
    dout = rng.standard_normal((count, width)).astype(np.float32)
    got = torch.full((vocab, width), 9.0, device="cuda")
    TokenEmbedding.gradient(0, dev(tokens), dev(dout), got)
    torch.cuda.synchronize()
    want, size = np.zeros((len(rows), width)), np.zeros((len(rows), width))
    np.add.at(want, np.searchsorted(rows, tokens), dout.astype(np.float64))
    np.add.at(size, np.searchsorted(rows, tokens), np.abs(dout.astype(np.float64)))
    index = torch.from_numpy(rows).cuda()
    assert (np.abs(to_f64(got[index]) - want) <= (32 + count / 16 + 8 + 3) * E * size).all()
    got[index] = 0.0
    assert not got.any()


def test_same_inputs_same_bits(cuda):
    rng = np.random.default_rng(3)
    tokens, dout = dev(some_tokens(rng, 20000, 500)), dev(rng.standard_normal((20000, 264)).astype(np.float32))
    results = []
    for _ in range(5):
        got = torch.zeros(500, 264, device="cuda")
        TokenEmbedding.gradient(0, tokens, dout, got)
        results.append(got)
    torch.cuda.synchronize()
    assert all(torch.equal(results[0], r) for r in results[1:])


@pytest.mark.parametrize("width,shift", ((64, 1), (64, 4), (33, 0), (33, 3)))
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
def test_gradient_at_an_arena_offset(cuda, width, shift, dtype):
    rng = np.random.default_rng(4)
    count, vocab = 500, 90
    tokens = some_tokens(rng, count, vocab)
    rows = dev((rng.standard_normal((count, width + 5))).astype(np.float32))
    dout = rows[:, :width]
    arena = misaligned(vocab * width + 20, dtype, shift)
    arena.fill_(3.0)
    got = arena[10:10 + vocab * width].view(vocab, width)
    TokenEmbedding.gradient(0, dev(tokens), dout, got)
    torch.cuda.synchronize()
    check_gradient(tokens, dout, got, 1.0, vocab)
    assert (arena[:10] == 3.0).all() and (arena[10 + vocab * width:] == 3.0).all()


def test_no_tokens(cuda):
    table, out = torch.ones(40, 24, device="cuda"), torch.zeros(0, 24, device="cuda")
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    TokenEmbedding.lookup(0, none, table, out)
    TokenEmbedding.gradient(0, none, out, table, accumulate=True)
    assert (table == 1.0).all()
    TokenEmbedding.gradient(0, none, out, table)
    assert not table.any()
    table.fill_(1.0)
    for count in (70, 5000):
        table.fill_(1.0)
        TokenEmbedding.gradient(0, torch.full((count,), -1, device="cuda"), torch.ones(count, 24, device="cuda"), table)
        assert not table.any()


def test_offsets_beyond_32_bits(cuda):
    """A table of 2.2 G values: row offsets pass 2^31, byte offsets 2^32."""
    vocab, width = 270_000, 8192
    table = torch.zeros(vocab, width, dtype=torch.bfloat16, device="cuda")
    table[-1], table[-2] = 2.0, 3.0
    tokens = torch.tensor([vocab - 1, vocab - 2, 0, vocab - 1], device="cuda")
    out = torch.zeros(4, width, device="cuda")
    TokenEmbedding.lookup(0, tokens, table, out)
    assert (out == torch.tensor([2.0, 3.0, 0.0, 2.0], device="cuda")[:, None]).all()
    table.fill_(1.0)
    TokenEmbedding.gradient(0, tokens, out, table)
    torch.cuda.synchronize()
    assert (table[-1] == 4.0).all() and (table[-2] == 3.0).all()
    assert not table[:-2].any()


def test_gradient_against_differences(cuda):
    """sum(out * dout) is linear in the table: its difference over a step of 1 in
    one value is the gradient there, up to the roundings of both (1e-4 of sums of
    some thousand terms of size one)."""
    rng = np.random.default_rng(5)
    vocab, width, count = 6, 8, 200
    tokens, table = some_tokens(rng, count, vocab), rng.standard_normal((vocab, width)).astype(np.float32)
    dout = rng.standard_normal((count, width)).astype(np.float32)

    def f(t):
        out = torch.zeros(count, width, device="cuda")
        TokenEmbedding.lookup(0, dev(tokens), dev(t), out, scale=0.5)
        return float((out.double() * dev(dout).double()).sum())

    gradient = torch.zeros(vocab, width, device="cuda")
    TokenEmbedding.gradient(0, dev(tokens), dev(dout), gradient, scale=0.5)
    for v in range(vocab):
        for c in range(width):
            up = table.copy()
            up[v, c] += 1.0
            assert abs(f(up) - f(table) - host(gradient)[v, c]) <= 1e-4


def test_on_a_stream_of_its_own_and_replayed_from_two_graphs(cuda):
    rng = np.random.default_rng(6)
    count, vocab, width = 3000, 700, 264
    tokens = dev(some_tokens(rng, count, vocab))
    dout = dev(rng.standard_normal((count, width)).astype(np.float32))
    eager, side = torch.zeros(vocab, width, device="cuda"), torch.zeros(vocab, width, device="cuda")
    TokenEmbedding.gradient(0, tokens, dout, eager)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    TokenEmbedding.gradient(0, tokens, dout, side, stream=stream)
    stream.synchronize()
    recorded, graphs = [torch.zeros_like(eager) for _ in range(2)], []
    for out in recorded:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            TokenEmbedding.gradient(0, tokens, dout, out)
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(10):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for out in [side, *recorded]:
        assert torch.equal(out, eager)


def test_refusals(cuda):
    table, out = torch.zeros(10, 16, device="cuda"), torch.zeros(3, 16, device="cuda")
    tokens = torch.zeros(3, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="int32 or int64"):
        TokenEmbedding.lookup(0, tokens.float(), table, out)
    with pytest.raises(ValueError, match="contiguous"):
        TokenEmbedding.lookup(0, torch.zeros(3, 2, dtype=torch.int64, device="cuda").t(), table, out)
    with pytest.raises(ValueError, match="out has shape"):
        TokenEmbedding.lookup(0, tokens, table, out[:2])
    with pytest.raises(ValueError, match="expected \\(vocab, width\\)"):
        TokenEmbedding.lookup(0, tokens, table.view(-1), out)
    with pytest.raises(ValueError, match="encoded table"):
        TokenEmbedding.lookup(0, tokens, table.to(torch.int8), out)
    with pytest.raises(ValueError, match="needs 5"):
        TokenEmbedding.lookup(0, tokens, table.to(torch.int8), out, table_scales=torch.ones(4, device="cuda"), block_size=32)
    with pytest.raises(ValueError, match="needs 6"):
        TokenEmbedding.lookup(0, tokens, table.to(torch.int8), out, table_scales=torch.ones(5, device="cuda"), block_size=32,
                              first_value=1)
    with pytest.raises(ValueError, match="no scales"):
        TokenEmbedding.lookup(0, tokens, table, out, table_scales=torch.ones(4, device="cuda"))
    with pytest.raises(ValueError, match="table_gradient has type"):
        TokenEmbedding.gradient(0, tokens, out, table.to(torch.int8))
    with pytest.raises(ValueError, match="out_gradient has shape"):
        TokenEmbedding.gradient(0, tokens, out[:, :8], table)
    with pytest.raises(ValueError, match="workspace"):
        TokenEmbedding.gradient(0, tokens, out, table, workspace=torch.zeros(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError, match="token_status"):
        TokenEmbedding.lookup(0, tokens, table, out, token_status=torch.zeros(1, device="cuda"))


@pytest.mark.parametrize("count", (3000, 20000, 70000))
def test_recorded_sorts_of_several_ctas(cuda, count):
    """A cluster's sort in a graph, replayed on other tokens than it was recorded with."""
    rng = np.random.default_rng(count)
    vocab, width = 5000, 40
    dout = dev(rng.standard_normal((count, width)).astype(np.float32))
    tokens, got = torch.zeros(count, dtype=torch.int64, device="cuda"), torch.zeros(vocab, width, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        TokenEmbedding.gradient(0, tokens, dout, got, scale=0.5, accumulate=True)
    for law in ("text", "even"):
        other = some_tokens(rng, count, vocab, 0.1, law)
        tokens.copy_(torch.from_numpy(other))
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        check_gradient(other, dout, got, 0.5, vocab)
