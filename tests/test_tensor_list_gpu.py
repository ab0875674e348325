"""The norm and clip of a list of gradient tensors against numpy in 64 bits.

Tolerances.  A norm is a binary64 sum (relative error below 1e-12 at these
lengths) whose root is rounded to binary32 once: half a step, 2^-24.  The
coefficient adds the roundings of max_norm, of norm + 1e-6 and of the quotient
to the norm's: 4 x 2^-24.  Clipped values are the products of the device's own
coefficient, rounded once: bit for bit."""
import numpy as np
import pytest
import torch

from gpu_helpers import assert_bits_equal, dev, host, misaligned
from nntrain_b200.library import NativeCudaError
from nntrain_b200.native import CudaBfp8Native, GradientNorm, GradientTensorList, scale_count

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -24
FLT_MIN = np.float32(1.1754943508222875e-38)


def bf16_round(x: np.ndarray) -> np.ndarray:
    return torch.from_numpy(np.ascontiguousarray(x)).to(torch.bfloat16).float().numpy()


class Leaf:
    """One tensor of a list and what it stands for."""

    def __init__(self, rng, n, kind, block=0, offset=0, destination=None, sigma=1e-3):
        x = (rng.standard_normal(n) * sigma).astype(np.float32)
        self.kind, self.block, self.scales = kind, block, None
        if kind == "f32":
            self.tensor = misaligned(n, torch.float32, offset) if n else torch.zeros(0, device="cuda")
            self.tensor.copy_(torch.from_numpy(x))
            self.values = x.astype(np.float64)
        elif kind == "bf16":
            self.tensor = misaligned(n, torch.bfloat16, offset) if n else torch.zeros(0, dtype=torch.bfloat16, device="cuda")
            self.tensor.copy_(torch.from_numpy(x))
            self.values = bf16_round(x).astype(np.float64)
        else:
            self.tensor = misaligned(n, torch.int8, offset)
            self.scales = torch.zeros(scale_count(n, block), device="cuda")
            CudaBfp8Native.block_encode(0, dev(x), self.tensor, self.scales, block)
            per_value = np.repeat(host(self.scales), min(block, n) if block else n)[:n]
            self.values = host(self.tensor).astype(np.float64) * per_value.astype(np.float64)
        self.source = self.scales if kind == "bfp8" else self.tensor
        self.before = self.source.clone()
        self.to = None
        if destination is not None:
            self.to = misaligned(self.source.numel(), self.source.dtype, destination)

    def clipped(self, c: np.float32) -> np.ndarray:
        """What the clip makes of it, bit for bit."""
        before = self.before.float().cpu().numpy()
        if c == 1.0:
            return before
        product = (before * c).astype(np.float32)
        if self.kind == "bfp8":
            return np.maximum(product, FLT_MIN)
        return bf16_round(product) if self.kind == "bf16" else product


def as_list(leaves):
    return GradientTensorList(0, [v.tensor for v in leaves], [v.scales for v in leaves], [v.block for v in leaves],
                              [v.to for v in leaves])


def run(leaves, max_norm, apply=True, stream=None):
    plan = as_list(leaves)
    out, norms = torch.full((2,), -1.0, device="cuda"), torch.full((len(leaves),), -1.0, device="cuda")
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    GradientNorm.clip_tensors(0, plan, max_norm, out, norms, flag, apply=apply, stream=stream)
    torch.cuda.synchronize()
    return host(out), host(norms), int(flag.item())


def check(leaves, max_norm, out, norms, applied=True):
    squares = [float(np.dot(v.values, v.values)) for v in leaves]
    norm = np.sqrt(sum(squares))
    for got, want in zip(norms, np.sqrt(squares)):
        assert abs(got - want) <= want * HALF * 1.001
    assert abs(out[0] - norm) <= norm * HALF * 1.001
    want = max_norm / (norm + 1e-6) if out[0] > np.float32(max_norm) else 1.0
    assert abs(out[1] - want) <= want * 4 * HALF * 1.001
    for i, v in enumerate(leaves):
        got = v.to if v.to is not None and applied else v.source
        want = v.clipped(out[1]) if applied else v.before.float().cpu().numpy()
        assert_bits_equal(got.float().cpu().numpy(), want, f"tensor {i}")
        if v.to is not None or not applied:
            assert torch.equal(v.source, v.before), f"tensor {i} was written"


LENGTHS = (1, 3, 7, 31, 255, 4095, 4096, 4097, 8191, 12289, 70001)


@pytest.mark.parametrize("kind,block", (("f32", 0), ("bf16", 0), ("bfp8", 32), ("bfp8", 96), ("bfp8", 100), ("bfp8", 0)))
@pytest.mark.parametrize("max_norm", (1e-2, 1e3))
def test_every_kind_and_length_in_place(cuda, kind, block, max_norm):
    rng = np.random.default_rng(1)
    leaves = [Leaf(rng, n, kind, block, offset=i % 5) for i, n in enumerate(LENGTHS)]
    out, norms, flag = run(leaves, max_norm)
    assert flag == 0 and (out[1] < 1.0) == (max_norm < 1.0)
    check(leaves, max_norm, out, norms)


@pytest.mark.parametrize("kind,steps", (("f32", 4), ("bf16", 8)))
def test_every_shift_between_source_and_destination(cuda, kind, steps):
    rng = np.random.default_rng(2)
    leaves = [Leaf(rng, n, kind, offset=a, destination=b)
              for a in range(steps) for b in range(steps) for n in (1, 5, 17, 4096 + 13)]
    out, norms, flag = run(leaves, 1e-2)
    assert flag == 0
    check(leaves, 1e-2, out, norms)
    for v in leaves:                                   # nothing behind the destination's end is written
        base = v.to._base
        start = v.to.storage_offset()
        assert not base[:start].any() and not base[start + v.to.numel():].any()


def test_a_mixed_list_into_its_arenas(cuda):
    rng = np.random.default_rng(3)
    leaves = [Leaf(rng, int(n), kind, 32, offset=0, destination=i % 7, sigma=10.0 ** -(i % 5))
              for i, (n, kind) in enumerate(zip(rng.integers(1, 30000, 60), ["f32", "bf16", "bfp8"] * 20))]
    out, norms, flag = run(leaves, 1.0)
    assert flag == 0
    check(leaves, 1.0, out, norms)


def test_norm_alone_writes_no_tensor(cuda):
    rng = np.random.default_rng(4)
    leaves = [Leaf(rng, n, k, 32, destination=1) for n, k in ((5000, "f32"), (77, "bf16"), (640, "bfp8"))]
    out, norms, flag = run(leaves, 1e-3, apply=False)
    check(leaves, 1e-3, out, norms, applied=False)
    assert all(not v.to.any() for v in leaves)


def test_empty_tensors_and_an_empty_list(cuda):
    rng = np.random.default_rng(5)
    leaves = [Leaf(rng, 0, "f32"), Leaf(rng, 9, "f32"), Leaf(rng, 0, "bf16")]
    out, norms, flag = run(leaves, 1e-4)
    check(leaves, 1e-4, out, norms)
    out, norms, flag = run([Leaf(rng, 0, "f32")], 1.0)
    assert (out == [0.0, 1.0]).all() and norms[0] == 0.0 and flag == 0


def test_zero_gradients_stay_and_a_norm_at_the_border_is_not_clipped(cuda):
    zeros = torch.zeros(1000, device="cuda")
    out = torch.zeros(2, device="cuda")
    GradientNorm.clip_tensors(0, GradientTensorList(0, [zeros]), 1.0, out)
    assert host(out).tolist() == [0.0, 1.0]
    border = torch.full((4,), 0.5, device="cuda")      # norm exactly 1
    GradientNorm.clip_tensors(0, GradientTensorList(0, [border]), 1.0, out)
    assert host(out).tolist() == [1.0, 1.0] and (border == 0.5).all()


@pytest.mark.parametrize("bad", (np.nan, np.inf, -np.inf))
@pytest.mark.parametrize("kind", ("f32", "bf16"))
def test_a_value_that_is_not_finite_leaves_the_list_as_it_was(cuda, bad, kind):
    rng = np.random.default_rng(6)
    leaves = [Leaf(rng, 5001, "f32", destination=3), Leaf(rng, 333, kind), Leaf(rng, 640, "bfp8", 32)]
    leaves[1].tensor[100] = float(bad)
    leaves[1].before = leaves[1].tensor.clone()
    out, norms, flag = run(leaves, 1e-3)
    assert flag == 1 and out[1] == 1.0 and not np.isfinite(out[0])
    assert not np.isfinite(norms[1]) and np.isfinite(norms[[0, 2]]).all()
    assert torch.equal(leaves[0].to, leaves[0].before) and torch.equal(leaves[2].scales, leaves[2].before)
    view = torch.int32 if kind == "f32" else torch.int16
    assert torch.equal(leaves[1].tensor.view(view), leaves[1].before.view(view))


@pytest.mark.parametrize("bad", (float("nan"), float("inf"), 0.0, -1.0))
def test_a_scale_that_no_encoding_has_raises_the_flag(cuda, bad):
    rng = np.random.default_rng(7)
    leaves = [Leaf(rng, 640, "bfp8", 32), Leaf(rng, 50, "f32")]
    leaves[0].scales[7] = bad
    leaves[1].before = leaves[1].tensor.clone()
    out, _, flag = run(leaves, 1e-6)
    assert flag == 1 and out[1] == 1.0 and torch.equal(leaves[1].tensor, leaves[1].before)


def test_a_norm_beyond_binary32_is_not_finite(cuda):
    x = torch.full((4,), 3e38, device="cuda")
    out, flag = torch.zeros(2, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    GradientNorm.clip_tensors(0, GradientTensorList(0, [x]), 1.0, out, finite_status=flag)
    assert int(flag.item()) == 1 and host(out)[1] == 1.0 and (x == torch.tensor(3e38)).all()


def test_clipped_scales_do_not_fall_below_the_smallest_normal(cuda):
    payload = torch.full((64,), 127, dtype=torch.int8, device="cuda")
    scales = torch.tensor([1e30, 2e-38], device="cuda")
    out = torch.zeros(2, device="cuda")
    GradientNorm.clip_tensors(0, GradientTensorList(0, [payload], [scales], [32]), 1e-3, out)
    assert host(out)[1] < 1e-30 and host(scales)[1] == FLT_MIN


def test_same_list_same_bits(cuda):
    rng = np.random.default_rng(8)
    leaves = [Leaf(rng, n, "f32", destination=1) for n in (1_000_003, 5, 300_000)]
    plan, results = as_list(leaves), []
    for _ in range(5):
        out, norms = torch.zeros(2, device="cuda"), torch.zeros(3, device="cuda")
        GradientNorm.clip_tensors(0, plan, 0.1, out, norms)
        results.append((host(out).tobytes(), host(norms).tobytes(), leaves[0].to.clone()))
    for r in results[1:]:
        assert r[:2] == results[0][:2] and torch.equal(r[2], results[0][2])


@pytest.mark.parametrize("lengths", ((70_001, 5, 300), (9_000_000, 4096)))
def test_the_norm_alone_and_with_the_clip_has_the_same_bits(cuda, lengths):
    """Short lists are summed by the clip's blocks, long ones by a block of their own: one order."""
    rng = np.random.default_rng(10)
    plan, results = as_list([Leaf(rng, n, "f32") for n in lengths]), []
    for apply in (False, True):
        out, norms = torch.zeros(2, device="cuda"), torch.zeros(len(lengths), device="cuda")
        GradientNorm.clip_tensors(0, plan, 0.1, out, norms, apply=apply)
        results.append((host(out).tobytes(), host(norms).tobytes()))
    assert results[0] == results[1]


def test_a_list_longer_than_the_smallest_chunks(cuda):
    """300 M values: the longest chunks, over 12 000 of them, several for a finishing lane."""
    n = 300_000_001
    x = torch.full((n,), 2.0 ** -10, device="cuda")
    y = torch.full((1001,), 1.0, dtype=torch.bfloat16, device="cuda")
    plan = GradientTensorList(0, [x, y])
    assert plan.chunk_values == 24576 and plan.chunks > 12000
    out, norms = torch.zeros(2, device="cuda"), torch.zeros(2, device="cuda")
    GradientNorm.clip_tensors(0, plan, 1.0, out, norms)
    want = np.sqrt(n * 2.0 ** -20 + 1001)
    got = host(out)
    assert abs(got[0] - want) <= want * HALF * 1.001
    assert abs(host(norms)[0] - np.sqrt(n * 2.0 ** -20)) <= np.sqrt(n * 2.0 ** -20) * HALF * 1.001
    assert (x == float(np.float32(2.0 ** -10) * got[1])).all()


def test_on_a_stream_of_its_own_and_replayed_from_two_graphs(cuda):
    rng = np.random.default_rng(9)
    side = torch.cuda.Stream()
    lists = [[Leaf(rng, n, "f32", destination=1) for n in (70_001, 12)] for _ in range(2)]
    plans = [as_list(v) for v in lists]
    outs = [torch.zeros(2, device="cuda") for _ in plans]
    torch.cuda.synchronize()
    GradientNorm.clip_tensors(0, plans[0], 0.1, outs[0], stream=side)      # eager, another stream
    side.synchronize()
    first = host(outs[0]).copy()
    graphs = []
    for plan, out in zip(plans, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            GradientNorm.clip_tensors(0, plan, 0.1, out)
        graphs.append(graph)
    for v in lists[0] + lists[1]:
        v.to.zero_()
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):                                                       # both at once: their scratch is their own
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert (host(outs[0]) == first).all()
    for leaves, out in zip(lists, outs):
        c = host(out)[1]
        for i, v in enumerate(leaves):
            assert_bits_equal(host(v.to), v.clipped(c), f"tensor {i}")


def test_refusals(cuda):
    x, out = torch.zeros(10, device="cuda"), torch.zeros(2, device="cuda")
    with pytest.raises(ValueError, match="contiguous"):
        GradientTensorList(0, [torch.zeros(4, 4, device="cuda").t()[:2]])
    with pytest.raises(ValueError, match="float16"):
        GradientTensorList(0, [x.half()])
    with pytest.raises(ValueError, match="its scales"):
        GradientTensorList(0, [x.to(torch.int8)])
    with pytest.raises(ValueError, match="no scales"):
        GradientTensorList(0, [x], [x])
    with pytest.raises(ValueError, match="descriptor"):
        GradientTensorList(0, [x.to(torch.int8)], [torch.ones(2, device="cuda")], [10])
    with pytest.raises(ValueError, match="its type"):
        GradientTensorList(0, [x], destinations=[x.to(torch.bfloat16)])
    with pytest.raises(ValueError, match="its length"):
        GradientTensorList(0, [x], destinations=[torch.zeros(9, device="cuda")])
    base = torch.zeros(20, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        GradientTensorList(0, [base[:10]], destinations=[base[5:15]])
    with pytest.raises(ValueError, match="overlap"):
        GradientTensorList(0, [x, x])
    GradientTensorList(0, [x, x], destinations=[base[:10], base[10:]])
    plan = GradientTensorList(0, [x])
    with pytest.raises(ValueError, match="device"):
        GradientNorm.clip_tensors(1, plan, 1.0, out)
    for max_norm in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            GradientNorm.clip_tensors(0, plan, max_norm, out)
    with pytest.raises(ValueError, match="two values"):
        GradientNorm.clip_tensors(0, plan, 1.0, out[:1])
    with pytest.raises(ValueError, match="workspace"):
        GradientNorm.clip_tensors(0, plan, 1.0, out, workspace=torch.zeros(0, dtype=torch.float64, device="cuda"))
    with pytest.raises(ValueError, match="tensor_norms"):
        GradientNorm.clip_tensors(0, plan, 1.0, out, tensor_norms=torch.zeros(0, device="cuda"))
    assert issubclass(NativeCudaError, RuntimeError)


@pytest.mark.parametrize("current", (False, True))
def test_a_list_may_be_dropped_while_another_stream_works_on_it(cuda, current):
    """Neither its table nor the tensors that only it holds are handed out again before that stream has come past."""
    side = torch.cuda.Stream()
    rng = np.random.default_rng(11)
    values = rng.standard_normal(5000).astype(np.float32)
    x, to, out = dev(values), torch.zeros(5000, device="cuda"), torch.zeros(2, device="cuda")
    plan = GradientTensorList(0, [x], destinations=[to])
    torch.cuda.synchronize()
    held = [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in (plan.buffer, x)]
    sizes = [plan.buffer.numel(), x.numel() * 4]
    with torch.cuda.stream(side):
        torch.cuda._sleep(400_000_000)                 # some 0.2 s
        if current:
            GradientNorm.clip_tensors(0, plan, 0.1, out)
    if not current:
        GradientNorm.clip_tensors(0, plan, 0.1, out, stream=side)
    del plan, x
    later = [torch.empty(size, dtype=torch.uint8, device="cuda") for size in sizes for _ in range(200)]
    taken = [t.data_ptr() for t in later if any(a < t.data_ptr() + t.numel() and t.data_ptr() < b for a, b in held)]
    assert not side.query(), "the other stream was too fast to show anything"
    assert not taken
    for t in later:
        t.fill_(255)
    torch.cuda.synchronize()
    c = host(out)[1]
    assert c < 1.0
    assert_bits_equal(host(to), values * c, "clipped")
