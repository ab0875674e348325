"""The training operators called by several host threads at once, each with its
own stream, outputs and scratch: every call succeeds and leaves the bits of a
call made alone."""
import threading

import numpy as np
import pytest
import torch

from gpu_helpers import dev
from nntrain_b200.library import load
from nntrain_b200.native import GradientNorm, GradientTensorList, RmsNorm, TokenEmbedding

pytestmark = pytest.mark.gpu

EPS = 1e-6


def run_together(jobs):
    """Every job in a thread of its own, started together; their errors."""
    errors, start = [], threading.Barrier(len(jobs))

    def body(job):
        try:
            torch.cuda.set_device(0)
            start.wait()
            job()
        except Exception as e:                                       # reported by the test's own thread
            errors.append(repr(e))

    threads = [threading.Thread(target=body, args=(job,)) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return errors


def norm_gradient_inputs(width, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = 160
    h, dy = (torch.randn(rows, width, generator=g, device="cuda").to(dtype) for _ in range(2))
    return h, dy, torch.ones(width, device="cuda"), torch.rsqrt(h.float().square().mean(dim=1) + EPS)


@pytest.mark.parametrize("dtype,widths", ((torch.bfloat16, (4096, 3584)), (torch.float32, (2048, 1792))))
def test_norm_gradients_of_two_widths_of_one_kernel(cuda, dtype, widths):
    """Both widths run the same kernel with different amounts of shared memory.
    The library is called directly, so that the threads meet inside of it."""
    backward = load().nntrain_rms_norm_backward
    jobs, outputs, expected, statuses = [], [], [], []
    for seed, width in enumerate(widths):
        h, dy, w, i = norm_gradient_inputs(width, dtype, seed)
        want = torch.zeros_like(h), torch.zeros(width, device="cuda")
        RmsNorm.backward(0, dy, h, w, i, *want)
        got = torch.zeros_like(h), torch.zeros(width, device="cuda")
        stream, scratch = torch.cuda.Stream(), torch.zeros(len(h) * width * 4, dtype=torch.uint8, device="cuda")
        kind = 0 if dtype is torch.float32 else 1
        arguments = (0, kind, dy.data_ptr(), width, 0, 0, h.data_ptr(), width, w.data_ptr(), 0, i.data_ptr(), len(h), width,
                     got[0].data_ptr(), got[1].data_ptr(), 0, 0, scratch.data_ptr(), scratch.numel(), stream.cuda_stream)
        seen = set()

        def job(arguments=arguments, seen=seen, keep=(h, dy, w, i, scratch, stream)):
            for _ in range(20000):
                seen.add(backward(*arguments))

        jobs.append(job)
        outputs.append(got)
        expected.append(want)
        statuses.append(seen)
    torch.cuda.synchronize()
    assert run_together(jobs) == []
    assert statuses == [{0}, {0}]
    for got, want in zip(outputs, expected):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_every_operator_from_four_threads(cuda):
    rng = np.random.default_rng(1)
    rows, vocab = 3000, 700

    def inputs(width, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        return dict(x=torch.randn(rows, width, generator=g, device="cuda"), w=torch.rand(width, generator=g, device="cuda"),
                    table=torch.randn(vocab, width, generator=g, device="cuda"),
                    tokens=dev(rng.integers(-1, vocab, rows)), width=width)

    def outputs(s):
        width = s["width"]
        return dict(y=torch.zeros(rows, width, device="cuda"), payload=torch.zeros(rows, width, dtype=torch.int8, device="cuda"),
                    scales=torch.zeros(rows, device="cuda"), inverse=torch.zeros(rows, device="cuda"),
                    dx=torch.zeros(rows, width, device="cuda"), dw=torch.zeros(width, device="cuda"),
                    out=torch.zeros(rows, width, device="cuda"), dt=torch.zeros(vocab, width, device="cuda"),
                    clipped=torch.zeros(rows * width, device="cuda"), norm=torch.zeros(2, device="cuda"))

    def step(s, o, stream):
        RmsNorm.forward(0, s["x"], s["w"], EPS, y=o["y"], payload=o["payload"], scales=o["scales"], inverse_rms=o["inverse"],
                        stream=stream)
        RmsNorm.backward(0, o["y"], s["x"], s["w"], o["inverse"], o["dx"], o["dw"], stream=stream)
        TokenEmbedding.lookup(0, s["tokens"], s["table"], o["out"], scale=0.5, stream=stream)
        TokenEmbedding.gradient(0, s["tokens"], o["dx"], o["dt"], stream=stream)
        GradientNorm.clip_tensors(0, o["list"], 0.1, o["norm"], stream=stream)

    states = [inputs(width, seed) for seed, width in enumerate((1536, 771, 1024, 40))]
    expected, got = [outputs(s) for s in states], [outputs(s) for s in states]
    for s, results in zip(states + states, expected + got):
        results["list"] = GradientTensorList(0, [s["x"].view(-1)], destinations=[results["clipped"]])
    for s, o in zip(states, expected):
        step(s, o, None)
    streams = [torch.cuda.Stream() for _ in states]
    torch.cuda.synchronize()

    def job(s, o, stream):
        for _ in range(50):
            step(s, o, stream)

    assert run_together([lambda a=a: job(*a) for a in zip(states, got, streams)]) == []
    for o, e in zip(got, expected):
        for name in e:
            if name != "list":
                assert torch.equal(o[name], e[name]), name
